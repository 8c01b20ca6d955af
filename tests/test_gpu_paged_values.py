"""What attend makes of values and scales at the ends of their range, against 64-bit arithmetic: rows of zeros, rows
whose scales lie far apart, infinities and NaNs that are seen. Tolerances are those of test_gpu_paged (Case.exact): one
bf16 ulp, the logits' and weights' relative errors, and for an 8-bit cache fp16's floor, taken of the largest
*weighted* value row."""
import math

import pytest
import torch

from helpers import bf16_ulp
from test_gpu_paged import DEV, Case

pytestmark = pytest.mark.gpu


def _set_values(case, b, j, factor=None, zero=False):
    """Position j of sequence b, all heads: its value row times `factor` (by its scale, exactly), or zeros as append
    writes them (scale 1)."""
    page, slot = int(case.table[b, j // case.page]), j % case.page
    if zero:
        case.v.view(torch.uint8)[page, :, slot] = 0
        case.v_scale[page, :, slot] = 1.0
        case.v64[b, :, j] = 0.0
    else:
        case.v_scale[page, :, slot] *= factor
        case.v64[b, :, j] *= factor


def _set_keys(case, b, j, rows):
    """Position j of sequence b: its key rows (heads, D), of at most 448, as e4m3 with scale 1."""
    page, slot = int(case.table[b, j // case.page]), j % case.page
    x = rows.to(torch.float8_e4m3fn)
    case.k.view(torch.uint8)[page, :, slot] = x.view(torch.uint8).to(DEV)
    case.k_scale[page, :, slot] = 1.0
    case.k64[b, :, j] = x.double()


def _check(case, q, window=0, counts=None):
    from tbf16 import _ext
    dc = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=DEV)
    out = case.cache().attend(q, window=window, counts=dc).cpu().double()
    ref, tol, _, _ = case.exact(q, counts, window)
    err = (out - ref).abs()
    assert bool((err <= tol).all()), f"max excess {(err - tol).max().item():.3e}, {((err > tol).double().mean()):.3f} of all"
    assert _ext.device_status() == 0


@pytest.mark.parametrize("magnitude", [2.0 ** -8, 2.0 ** -16, 2.0 ** -24, 2.0 ** -60])
@pytest.mark.parametrize("D,Hq,T", [(64, 4, 1), (128, 16, 1), (256, 4, 4), (256, 64, 1)])
def test_zero_value_rows_leave_the_others_their_bits(magnitude, D, Hq, T):
    """A zero row has scale 1, however small the rows beside it are."""
    lens = [50, 400, 33]
    for zeros in ([0], [17, 18], [49, 300, 399]):
        case = Case(lens, 2, D, 16, 8, seed=D)
        for b, n in enumerate(lens):
            for j in range(n):
                _set_values(case, b, j, factor=magnitude)
            for j in zeros:
                if j < n:
                    _set_values(case, b, j, zero=True)
        _check(case, case.queries(Hq, T))


@pytest.mark.parametrize("ratio", [2.0 ** 12, 2.0 ** 20, 2.0 ** 30])
@pytest.mark.parametrize("light", ["first", "front", "middle", "last", "all but one", "every third"])
@pytest.mark.parametrize("D", [64, 256])
def test_large_rows_of_little_weight_leave_the_others_their_bits(ratio, light, D):
    """Keys that the first query row of a head hardly sees (their logits lie about 45 below) and whose value rows are
    `ratio` times as large; the second row, the negated query, sees little else."""
    lens = [300, 41]
    case = Case(lens, 2, D, 16, 8, seed=3, gain=0.25)
    q = case.queries(4, 1)
    q[:, 1::2] = -q[:, ::2]
    for b, n in enumerate(lens):
        at = {"first": [0], "front": range(40), "middle": [n // 2], "last": [n - 1], "all but one": range(n - 1),
              "every third": range(0, n, 3)}[light]
        for j in at:
            x = q[b, ::2, 0].cpu().double()
            _set_keys(case, b, j, (-45 * math.sqrt(D) * x / x.square().sum(-1, keepdim=True)).float())
            _set_values(case, b, j, factor=ratio)
    _check(case, q)
    if light != "all but one":
        _check(case, q, window=35)


def test_scales_of_either_sign():
    """A caller's scales need not be positive."""
    lens = [100, 17]
    case = Case(lens, 2, 128, 16, 8)
    for b, n in enumerate(lens):
        for j in range(n):
            if j % 3 != 1 or j < 16:
                _set_values(case, b, j, factor=-1.0)
    _check(case, case.queries(4, 1))
    _check(case, case.queries(4, 3))


@pytest.mark.parametrize("T,Hq", [(1, 2), (3, 8), (1, 16)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_visible_infinities_follow_the_formula(T, Hq, D):
    """A value of +-infinity that a row sees, wherever it lies, makes that output column +-infinity: every weight is
    positive. Both signs make it NaN, as a NaN does; the other columns keep their values."""
    lens = [50, 300]
    case = Case(lens, 1, D, 16)
    q = case.queries(Hq, T)
    bad = {5: [(3, math.inf)], 6: [(20, -math.inf)], 7: [(3, math.inf), (21, -math.inf)], 8: [(30, math.nan)],
           9: [(n - 1 - T, math.inf) for n in (50,)], 40: [(40, -math.inf), (41, -math.inf)]}
    for b in range(len(lens)):
        for col, rows in bad.items():
            for j, x in rows:
                case.v[case.table[b, j // 16], :, j % 16, col] = x
    got = case.cache().attend(q).cpu().double()
    ref, tol, _, _ = case.exact(q)  # of the finite values that were there
    fine = [c for c in range(D) if c not in bad]
    assert bool(((got - ref).abs() <= tol)[..., fine].all())
    for col, rows in bad.items():
        want = sum(x for _, x in rows)
        x = got[..., col]
        assert bool(x.isnan().all() if math.isnan(want) else (x == want).all()), (col, x)


@pytest.mark.parametrize("bits", [16, 8])
def test_nan_weights_stay_among_the_positions_a_row_sees(bits):
    """Totals: a row whose softmax is NaN makes the totals of what it sees NaN, and no other's."""
    case = Case([50, 70], 2, 64, 16, bits)

    def totals(q, window):
        w = torch.zeros(2, 2, case.cap, device=DEV)
        case.cache(weights=w).attend(q, window=window)
        return w.cpu()
    q = case.queries(4, 1)
    q[:, :, 0, 0] = float("nan")
    w = totals(q, 21)  # the window begins inside a block
    for b, n in enumerate(case.lens):
        assert w[b, :, n - 21:n].isnan().all() and not w[b, :, :n - 21].any() and not w[b, :, n:].any()
    q = case.queries(4, 2)
    q[:, :, 0, 0] = float("nan")  # the first of two new tokens, which does not see the second
    w = totals(q, 0)
    for b, n in enumerate(case.lens):
        assert w[b, :, :n - 1].isnan().all() and torch.isfinite(w[b, :, n - 1:]).all() and (w[b, :, n - 1] > 0).all()

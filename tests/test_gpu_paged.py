"""tbf16.PagedCache against plain 64-bit arithmetic: append, attend and compact at the sizes, masks and
layouts where they can go wrong, their refusals, and the three together.

Tolerances. attend: one bf16 ulp of the exact output, plus what the 32-bit logits and the rounding of the
softmax weights can move it by. A logit of D products summed in fp32 is off by at most (D + 8) 2^-24
sum|q k| * scale (call it d); a weight is then off by a factor exp(2 d), and is kept to 2^-16 (bf16 cache:
two bf16 parts) or 2^-11 (e4m3 cache: fp16) of itself, with an fp16 floor of 2^-25 of the largest weighted
row scale. So |out - exact| <= ulp + (2 d + r) sum p|v| + floor. weights: (2 d + 2^-18) p, plus the rounding
of each fp32 addition. append and compact: bit-equal."""
import itertools
import math

import pytest
import torch

from helpers import bf16_ulp

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Case:
    """Pools, a shuffled page table and lengths, with everything outside the cached rows poisoned."""

    def __init__(self, lens, Hkv, D, page, bits=16, seed=0, layout="hnd", poison=float("nan"), max_len=None, gain=1.0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.H, self.D, self.page, self.bits = list(lens), Hkv, D, page, bits
        B, per = len(lens), -(-max(1, max_len or max(lens)) // page)
        pages = B * per + 3
        self.cap = per * page
        self.table = torch.randperm(pages, generator=g)[:B * per].view(B, per).to(torch.int32)
        shape = (pages, Hkv, page, D) if layout == "hnd" else (pages, page, Hkv, D)
        fix = (lambda x: x) if layout == "hnd" else (lambda x: x.transpose(1, 2))
        self.k64, self.v64 = (torch.randn(B, Hkv, self.cap, D, generator=g, dtype=torch.float64) * gain for _ in range(2))
        self.k_scale = self.v_scale = None
        pools, scales = [], []
        for x in (self.k64, self.v64):
            x *= torch.exp2(torch.randint(-3, 4, (B, 1, self.cap, 1), generator=g).double() * 0.25)
            if bits == 16:
                x.copy_(x.bfloat16().double())
                pool = fix(torch.full(shape, poison, dtype=torch.bfloat16))
            else:
                inv = torch.exp2(torch.randint(-9, -5, (B, Hkv, self.cap), generator=g).double())
                q = (x / inv[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn)
                x.copy_(q.double() * inv[..., None])
                pool = fix(torch.full(shape, poison, dtype=torch.bfloat16).to(torch.float8_e4m3fn))
                scale = torch.full((pages, Hkv, page), poison)
                scales.append(scale)
            for b, n in enumerate(lens):
                for i in range(-(-n // page)):
                    m = min(page, n - i * page)
                    at = slice(i * page, i * page + m)
                    if bits == 16:
                        pool[self.table[b, i], :, :m] = x[b, :, at].bfloat16()
                    else:
                        pool.view(torch.uint8)[self.table[b, i], :, :m] = q[b, :, at].view(torch.uint8)
                        scale[self.table[b, i], :, :m] = inv[b, :, at].float()
            pools.append(pool)
        self.k, self.v = (x.to(DEV) if layout == "hnd" else x.transpose(1, 2).to(DEV).transpose(1, 2) for x in pools)
        if bits == 8:
            self.k_scale, self.v_scale = (x.to(DEV) for x in scales)
        self.dtable, self.dlens = self.table.to(DEV), torch.tensor(self.lens, dtype=torch.int32, device=DEV)

    def cache(self, **kw):
        import tbf16
        return tbf16.PagedCache.over(self.k, self.v, self.dtable, self.dlens, k_scale=self.k_scale, v_scale=self.v_scale, **kw)

    def queries(self, Hq, T, seed=1, gain=1.0):
        g = torch.Generator().manual_seed(seed)
        return (torch.randn(len(self.lens), T, Hq, self.D, generator=g) * gain).bfloat16().to(DEV).transpose(1, 2)

    def exact(self, q, counts=None, window=0, scale=None):
        """(out, tolerance, summed weights, their tolerance), sequence by sequence in 64 bits on the CPU."""
        q = q.cpu().double()
        B, Hq, T, D = q.shape
        g = Hq // self.H
        scale = 1.0 / math.sqrt(D) if scale is None else scale
        out, slack = torch.zeros(2, B, Hq, T, D, dtype=torch.float64).unbind(0)
        w, wtol = torch.zeros(2, B, self.H, self.cap, dtype=torch.float64).unbind(0)
        r = 2.0 ** -16 if self.bits == 16 else 2.0 ** -11
        for b, n in enumerate(self.lens):
            c = min(T, n) if counts is None else counts[b]
            for t in range(c):
                last = n - c + t
                first = max(0, last - window + 1) if window else 0
                if last < first:
                    continue
                k, v = self.k64[b, :, first:last + 1], self.v64[b, :, first:last + 1]
                qt = q[b, :, t].view(self.H, g, D)
                p = torch.softmax(torch.einsum("hgd,hnd->hgn", qt, k) * scale, -1)
                d = (D + 8) * 2.0 ** -24 * abs(scale) * torch.einsum("hgd,hnd->hgn", qt.abs(), k.abs()).amax(-1, keepdim=True)
                out[b, :, t] = torch.einsum("hgn,hnd->hgd", p, v).reshape(Hq, D)
                pv = torch.einsum("hgn,hnd->hgd", p, v.abs())
                floor = 0.0
                if self.bits == 8:
                    vmax = v.abs().amax(-1)[:, None]  # a row's scale is below its largest magnitude
                    floor = 2.0 ** -25 * (p * vmax).amax(-1, keepdim=True) * 256 * p.shape[-1]
                slack[b, :, t] = ((2 * d + r) * pv + floor).reshape(Hq, D)
                w[b, :, first:last + 1] += p.sum(1)
                wtol[b, :, first:last + 1] += ((2 * d + 2.0 ** -18) * p).sum(1)
        return out, bf16_ulp(out) + slack, w, wtol


def _ids(v):
    return "-".join(map(str, v)) if isinstance(v, (list, tuple)) else str(v)


def _check_attend(case, Hq, T=1, counts=None, window=0, scale=None, track=False, gain=1.0):
    from tbf16 import _ext
    q = case.queries(Hq, T, gain=gain)
    old = torch.rand(len(case.lens), case.H, case.cap, generator=torch.Generator().manual_seed(5))
    kw = dict(weights=old.to(DEV)) if track else {}
    cache = case.cache(**kw)
    dc = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=DEV)
    out = cache.attend(q, counts=dc, window=window, scale=scale)
    assert out.shape == q.shape and out.dtype == torch.bfloat16
    ref, tol, w, wtol = case.exact(q, counts, window, scale)
    err = (out.cpu().double() - ref).abs()
    assert bool((err <= tol).all()), f"max excess {(err - tol).max().item():.3e} of {tol.max().item():.3e}, nan {err.isnan().sum()}"
    if track:
        got = kw["weights"].cpu().double()
        bound = wtol + 2.0 ** -23 * (Hq // case.H * T + 1) * (old.double() + w)
        assert bool(((got - (old.double() + w)).abs() <= bound).all())
        again = old.to(DEV)
        cache2 = case.cache(weights=again)
        assert torch.equal(cache2.attend(q, counts=dc, window=window, scale=scale), out)  # same bits every time
        assert torch.equal(again, kw["weights"])
    assert _ext.device_status() == 0
    return out


# lengths around block, page and split boundaries; an empty sequence in the middle
LENS = [1, 0, 15, 16, 17, 31, 33, 64, 65, 127, 200, 513]


@pytest.mark.parametrize("D,bits,page", list(itertools.product([64, 128, 256], [16, 8], [16, 64])), ids=_ids)
def test_attend_lengths(D, bits, page):
    _check_attend(Case(LENS, 2, D, page, bits), Hq=8)


@pytest.mark.parametrize("Hq,Hkv,T", [(1, 1, 1), (4, 4, 1), (6, 2, 1), (20, 5, 1), (16, 1, 1), (24, 1, 1), (71, 1, 1),
                                      (8, 4, 2), (5, 1, 3), (32, 2, 4), (4, 2, 20)], ids=_ids)
@pytest.mark.parametrize("bits", [16, 8])
def test_attend_heads_and_tokens(Hq, Hkv, T, bits):
    lens = [max(n, T) if n else 0 for n in (0, 1, 50, 129, 300)]
    counts = [min(T, n) for n in lens]
    _check_attend(Case(lens, Hkv, 128, 32, bits, seed=Hq), Hq, T, counts)
    _check_attend(Case(lens, Hkv, 64, 16, bits, seed=Hq), Hq, T, counts, track=True)
    _check_attend(Case(lens, Hkv, 256, 128, bits, seed=Hq), Hq, T, counts)


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 64, 100, 511, 512, 1000])
@pytest.mark.parametrize("T,bits", [(1, 16), (3, 16), (1, 8)])
def test_attend_window(window, T, bits):
    lens = [T, 16, 17, 80, 129, 512, 513]
    _check_attend(Case(lens, 2, 128, 16, bits), 4, T, window=window)
    _check_attend(Case(lens, 2, 64, 64, bits), 8, T, window=window, track=True)


@pytest.mark.parametrize("bits", [16, 8])
def test_attend_counts_below_T(bits):
    """Fewer real tokens than T: the rest of a sequence's rows are zeros, and position counts from the end."""
    lens, counts = [5, 1, 40, 300, 0, 2], [3, 1, 0, 4, 0, 2]
    out = _check_attend(Case(lens, 2, 128, 16, bits), 6, 4, counts, track=True)
    for b, c in enumerate(counts):
        assert not out[b, :, c:].any()


@pytest.mark.parametrize("lens,Hkv,Hq,D,page,bits", [
    ([20011], 1, 8, 128, 16, 16), ([30000, 3, 9000], 2, 8, 64, 64, 16), ([17000], 4, 8, 256, 32, 16),
    ([40001], 1, 16, 128, 128, 8), ([9999, 20000], 2, 4, 256, 16, 8), ([50000], 2, 2, 64, 256, 8)], ids=_ids)
def test_attend_long(lens, Hkv, Hq, D, page, bits):
    """Long enough to be split over many blocks and joined."""
    _check_attend(Case(lens, Hkv, D, page, bits), Hq, track=True)


def test_attend_many_sequences():
    lens = [(i * 37) % 90 for i in range(300)]
    _check_attend(Case(lens, 2, 64, 16), 4, counts=[min(1, n) for n in lens])
    _check_attend(Case([7] * 1024, 1, 64, 16), 1)


@pytest.mark.parametrize("bits", [16, 8])
def test_attend_peaked_and_scaled(bits):
    """Logits far apart (one key takes all), a negative and a zero scale."""
    case = Case([300, 4000], 2, 128, 32, bits)
    _check_attend(case, 4, gain=30.0, track=True)
    _check_attend(case, 4, scale=-0.1)
    _check_attend(case, 4, scale=0.0)


@pytest.mark.parametrize("bits", [16, 8])
def test_attend_layouts(bits):
    """Pools in (page, slot, head, D) order, queries as a slice of a packed projection, and misaligned ones."""
    from tbf16 import _ext
    case = Case([100, 37], 4, 64, 16, bits, layout="nhd")
    assert case.k.stride(1) == 64
    _check_attend(case, 8)
    cache = case.cache()
    q = case.queries(8, 2)
    ref = cache.attend(q)
    packed = torch.randn(2, 2, 16 * 64 + 3, device=DEV).bfloat16()
    packed[..., :8 * 64] = q.transpose(1, 2).flatten(2)
    assert torch.equal(cache.attend(packed[..., :8 * 64].unflatten(-1, (8, 64)).transpose(1, 2)), ref)  # odd strides
    packed[..., 3:3 + 8 * 64] = q.transpose(1, 2).flatten(2)
    assert torch.equal(cache.attend(packed[..., 3:3 + 8 * 64].unflatten(-1, (8, 64)).transpose(1, 2)), ref)
    assert torch.equal(cache.attend(q.contiguous()), ref)
    one = Case([100], 4, 64, 16, bits)  # one sequence, one token: strides of a packed row that is no multiple of 8
    q1 = one.queries(8, 1)
    odd = torch.zeros(1, 1, 8 * 64 + 3, device=DEV, dtype=torch.bfloat16)
    odd[..., :8 * 64] = q1.transpose(1, 2).flatten(2)
    assert torch.equal(one.cache().attend(odd[..., :8 * 64].unflatten(-1, (8, 64)).transpose(1, 2)), one.cache().attend(q1))
    assert ref.transpose(1, 2).is_contiguous()  # (B, T, heads, D) memory for the output projection
    assert _ext.device_status() == 0


@pytest.mark.parametrize("poison", [float("nan"), float("inf"), -float("inf"), torch.finfo(torch.bfloat16).min])
def test_attend_ignores_what_is_masked(poison):
    """Slots past the length, pages of nobody, keys before the window: whatever they hold, nothing changes."""
    for bits, window in ((16, 0), (16, 20), (8, 0)):
        if bits == 8 and not math.isnan(poison):
            continue
        _check_attend(Case([33, 100, 18], 2, 64, 32, bits, poison=poison), 4, window=window)
    case = Case([60, 130], 2, 128, 16, poison=poison)
    want = case.cache().attend(case.queries(4, 1), window=40)
    for b, n in enumerate(case.lens):
        for j in range(n - 40):
            case.k[case.table[b, j // 16], :, j % 16] = poison
            case.v[case.table[b, j // 16], :, j % 16] = poison
    assert torch.equal(case.cache().attend(case.queries(4, 1), window=40), want)


@pytest.mark.parametrize("bits", [16, 8])
def test_attend_later_token_does_not_leak(bits):
    """A NaN or infinity in the value of a draft token reaches the tokens that see it, and no earlier one."""
    for bad in (float("nan"), float("inf")):
        if bits == 8 and bad != bad + 1 and math.isinf(bad):
            continue
        case = Case([40, 17], 2, 128, 16, bits)
        q = case.queries(4, 4)
        want = case.cache().attend(q)
        for b, n in enumerate(case.lens):
            page, slot = case.table[b, (n - 2) // 16], (n - 2) % 16
            if bits == 16:
                case.v[page, :, slot, 5] = bad
            else:
                case.v_scale[page, :, slot] = bad
        got = case.cache().attend(q)
        assert torch.equal(got[:, :, :2], want[:, :, :2])
        assert not torch.isfinite(got[:, :, 2:, 5].float()).any()
        if bits == 16:
            keep = [i for i in range(128) if i != 5]
            assert torch.equal(got[:, :, 2:, keep], want[:, :, 2:, keep])


def test_attend_visible_nan_and_inf_follow_the_formula():
    case = Case([50], 1, 64, 16)
    case.k[case.table[0, 1], 0, 3, 0] = float("nan")
    assert case.cache().attend(case.queries(2, 1)).isnan().all()


def test_attend_offsets_past_32_bits():
    """Pages at the far end of pools over 2^32 bytes and 2^31 elements."""
    pages, H, page, D = 70000, 4, 64, 128
    import tbf16
    k = torch.empty(pages, H, page, D, device=DEV, dtype=torch.bfloat16)
    v = torch.empty_like(k)
    assert k.numel() > 2 ** 31
    small = Case([200], H, D, page)
    far = torch.tensor([[pages - 1, pages - 3, 5, pages - 2]], dtype=torch.int32, device=DEV)
    for i in range(4):
        k[far[0, i]], v[far[0, i]] = small.k[small.table[0, i]], small.v[small.table[0, i]]
    cache = tbf16.PagedCache.over(k, v, far, small.dlens)
    q = small.queries(8, 1)
    assert torch.equal(cache.attend(q), small.cache().attend(q))
    new = torch.randn(1, H, 1, D, device=DEV).bfloat16()
    cache.append(new, -new)
    assert torch.equal(k[pages - 2, :, 199 - 192], new[0, :, 0]) and torch.equal(v[pages - 2, :, 199 - 192], -new[0, :, 0])


@pytest.mark.parametrize("D,bits", list(itertools.product([64, 128, 256], [16, 8])), ids=_ids)
@pytest.mark.parametrize("T,layout", [(1, "hnd"), (1, "nhd"), (37, "hnd"), (200, "nhd")])
def test_append(D, bits, T, layout):
    from tbf16 import _ext
    lens = [0, 1, T, T + 5, T + 64, 300]
    counts = [min(T, n) if i != 4 else min(T, n) // 2 for i, n in enumerate(lens)]
    case = Case(lens, 3, D, 16, bits, layout=layout, poison=0.5)
    g = torch.Generator().manual_seed(T)
    x = torch.randn(2, len(lens), T, 3, D, generator=g) * torch.exp2(torch.randint(-30, 30, (2, len(lens), T, 3, 1), generator=g))
    x[0, 5, 0, 0] = 0.0
    x[1, 5, 0, 1] = 1e-38
    x[1, 5, 0, 2, 1:] = 0.0
    x = x.bfloat16().to(DEV)
    before = [y.clone() if y is not None else None for y in (case.k, case.v, case.k_scale, case.v_scale)]
    pos = torch.full((len(lens), 3, case.cap), -7, dtype=torch.int32, device=DEV)
    seen = case.dlens + 1000
    case.cache(pos=pos, seen=seen).append(*(y.transpose(1, 2) for y in x),
                                         counts=torch.tensor(counts, dtype=torch.int32, device=DEV))
    want = [y.cpu() if y is not None else None for y in before]
    want_pos = torch.full_like(pos, -7).cpu()
    for b, (n, c) in enumerate(zip(lens, counts)):
        for t in range(c):
            j = n - c + t
            page, slot = case.table[b, j // 16], j % 16
            want_pos[b, :, j] = n + 1000 - c + t
            for i in range(2):
                row = x[i, b, t].cpu()
                if bits == 16:
                    want[i][page, :, slot] = row
                    continue
                m = row.double().abs().amax(-1)
                e = torch.frexp(m.clamp_min(2.0 ** -119)).exponent
                e = torch.where(m == 0, 8, e)
                scale = torch.ldexp(torch.ones(3, dtype=torch.float64), e - 8)
                want[2 + i][page, :, slot] = scale.float()
                want[i].view(torch.uint8)[page, :, slot] = (row.double() / scale[:, None]).float().to(torch.float8_e4m3fn).view(torch.uint8)
    for got, ref in zip((case.k, case.v, case.k_scale, case.v_scale), want):
        if ref is not None:
            as_int = (lambda y: y.view(torch.uint8)) if ref.dtype == torch.float8_e4m3fn else (lambda y: y)
            assert torch.equal(as_int(got.cpu()), as_int(ref))
    assert torch.equal(pos.cpu(), want_pos)
    assert _ext.device_status() == 0


def test_append_non_finite_rows_read_back_as_nan():
    case = Case([4], 2, 64, 16, 8, poison=0.0)
    x = torch.randn(1, 2, 4, 64, device=DEV).bfloat16()
    x[0, 0, 1, 7], x[0, 1, 2, 0] = float("inf"), float("nan")
    case.cache().append(x, x)
    page = int(case.table[0, 0])
    back = case.k[page].float() * case.k_scale[page][..., None]
    assert back[0, 1].isnan().all() and back[1, 2].isnan().all()
    ok = torch.ones(2, 16, dtype=torch.bool)
    ok[0, 1] = ok[1, 2] = False
    assert torch.isfinite(back[ok]).all()


def _plain_compact(case, w, pos, seen, keep, recent):
    """Per sequence and head in plain Python: (from, to) of every moved row, new weights and numbers."""
    B, H, cols = w.shape
    new_w, new_pos, moves = torch.zeros_like(w), torch.full_like(pos, -1), []
    for b, h in itertools.product(range(B), range(H)):
        n = case.lens[b]
        m = min(n, keep)

        def rank(i):
            x = float(w[b, h, i])
            if int(pos[b, h, i]) >= int(seen[b]) - recent:
                return (0, 0.0, i)
            return (1, 0.0, i) if math.isnan(x) else (2, -x, i)
        kept = set(sorted(range(n), key=rank)[:m])
        holes, loose = [i for i in range(m) if i not in kept], sorted(i for i in kept if i >= m)
        assert len(holes) == len(loose)
        src = list(range(m))
        for to, frm in zip(holes, loose):
            src[to] = frm
            moves.append((b, h, frm, to))
        new_w[b, h, :m], new_pos[b, h, :m] = w[b, h, src], pos[b, h, src]
    return new_w, new_pos, moves


@pytest.mark.parametrize("lens,keep,recent,kind", [
    ([0, 1, 31, 32, 33, 100, 257], 32, 8, "heavy"), ([300, 1000], 999, 0, "heavy"), ([300, 64], 1, 0, "heavy"),
    ([300, 64], 1, 1, "heavy"), ([500], 0, 0, "heavy"), ([500], 500, 10, "heavy"), ([700, 650], 600, 600, "heavy"),
    ([2500, 900], 800, 100, "ties"), ([5000], 2048, 16, "same"), ([400, 90], 77, 5, "odd"), ([5000, 33], 20, 15, "front"),
    ([20000, 70000], 9000, 128, "heavy"), ([70001], 60000, 0, "ties"), ([400001, 5], 399000, 7, "heavy")], ids=_ids)
@pytest.mark.parametrize("D,bits,page,layout", [(64, 16, 16, "hnd"), (128, 8, 64, "nhd"), (256, 16, 32, "nhd"), (64, 8, 16, "hnd")])
def test_compact(lens, keep, recent, kind, D, bits, page, layout):
    from tbf16 import _ext
    if max(lens) > 10000 and D == 256:
        D = 64
    H = 1 if max(lens) > 10000 else 3
    case = Case(lens, H, D, page, bits, layout=layout, poison=0.25)
    B, cols = len(lens), case.cap
    g = torch.Generator().manual_seed(keep)
    w = torch.exp(2 * torch.randn(B, H, cols, generator=g))
    if kind == "ties":
        w = torch.randint(0, 3, w.shape, generator=g).float()
    elif kind == "same":
        w = torch.full_like(w, 0.5)
    elif kind == "odd":  # every kind of value a weight could hold
        w = torch.randn(w.shape, generator=g)
        for i, x in enumerate((float("nan"), -float("nan"), float("inf"), -float("inf"), 0.0, -0.0, 1e-40, -1e-40)):
            w[..., i::11] = x
    elif kind == "front":
        w[..., :keep] += 1e6
    pos = torch.stack([torch.randperm(cols, generator=g) for _ in range(B * H)]).view(B, H, cols).to(torch.int32)
    for b, n in enumerate(lens):  # numbers 100..n + 99 in any order, as after earlier cuts
        for h in range(H):
            pos[b, h, :n] = torch.randperm(n, generator=g).to(torch.int32) + 100
    seen = torch.tensor(lens, dtype=torch.int32) + 100
    wd, pd = w.to(DEV), pos.to(DEV)
    cache = case.cache(weights=wd, pos=pd, seen=seen.to(DEV))
    state = [case.k, case.v] + ([case.k_scale, case.v_scale] if bits == 8 else [])
    as_int = lambda y: y.view(torch.uint8) if y.dtype == torch.float8_e4m3fn else y  # noqa: E731
    want = [as_int(y).cpu() for y in state]
    new_w, new_pos, moves = _plain_compact(case, w, pos, seen, keep, recent)
    if moves:
        b, h, frm, to = (torch.tensor(x) for x in zip(*moves))
        f, t = (case.table[b, frm // page].long(), h, frm % page), (case.table[b, to // page].long(), h, to % page)
        for y in want:
            y[t] = y[f]
    got_w, got_pos = cache.compact(keep, recent)
    assert torch.equal(got_w.cpu().view(torch.int32), new_w.view(torch.int32)) and torch.equal(got_pos.cpu(), new_pos)
    for y, ref in zip(state, want):
        assert torch.equal(as_int(y).cpu(), ref)
    assert torch.equal(wd.cpu().view(torch.int32), w.view(torch.int32)) and torch.equal(pd.cpu(), pos)  # inputs stay
    assert _ext.device_status() == 0


@pytest.mark.parametrize("cols", [49152, 49153])
def test_compact_of_many_items_with_long_slices(cols):
    """More items than half the SMs have no clusters: one CTA ranks all positions, as many as its shared memory
    holds, or (one more) a pair does. Every kept row is found by its number."""
    import tbf16
    from tbf16 import _ext
    B, page, keep, recent = 75, 64, 9000, 100
    lens = [cols, cols - 5] + [90] * (B - 2)
    need, cap = [-(-n // page) for n in lens], -(-cols // page)
    order = torch.randperm(sum(need), generator=torch.Generator().manual_seed(1)).to(torch.int32).split(need)
    table = torch.zeros(B, cap, dtype=torch.int32)
    for b, pages in enumerate(order):
        table[b, :need[b]] = pages
    g = torch.Generator(device=DEV).manual_seed(2)
    k, v = (torch.randn(sum(need), 1, page, 64, generator=g, device=DEV).bfloat16() for _ in range(2))
    w = torch.exp(torch.randn(B, 1, cap * page, generator=g, device=DEV))
    pos = torch.arange(cap * page, dtype=torch.int32, device=DEV).expand(B, 1, -1).contiguous()
    ints = dict(dtype=torch.int32, device=DEV)
    cache = tbf16.PagedCache.over(k, v, table.to(DEV), torch.tensor(lens, **ints), weights=w, pos=pos,
                                  seen=torch.tensor(lens, **ints))
    rows = lambda x, b, n: x[table[b].long().to(DEV), 0].reshape(-1, 64)[:n]  # noqa: E731
    old = [[rows(x, b, lens[b]).clone() for x in (k, v)] for b in range(3)]
    new_w, new_pos = cache.compact(keep, recent)
    for b in range(B):
        n, m = lens[b], min(lens[b], keep)
        rank = w[b, 0, :n].double()
        rank[n - recent if n > recent else 0:] = math.inf
        kept = torch.zeros(n, dtype=torch.bool, device=DEV)
        kept[torch.sort(rank, descending=True, stable=True).indices[:m]] = True
        number = new_pos[b, 0, :m].long()
        stay = torch.arange(m, device=DEV)
        assert torch.equal(number.sort().values, kept.nonzero()[:, 0])
        assert torch.equal(number[kept[:m]], stay[kept[:m]]) and bool((number[~kept[:m]].diff() > 0).all())
        assert torch.equal(new_w[b, 0, :m], w[b, 0, number]) and not new_w[b, 0, m:].any() and bool((new_pos[b, 0, m:] == -1).all())
        if b < len(old):
            assert all(torch.equal(rows(x, b, m), y[number]) for x, y in zip((k, v), old[b]))
    assert _ext.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("head_dim", [64, 80, 256])
def test_cache_decodes_like_attention_over_everything(dtype, head_dim):
    """Prompts of different lengths, then decoding with drafts, two layers: every output equals attention over
    the whole sequence, in 64 bits on the rows as the cache holds them."""
    import tbf16
    B, H, Hq, L = 3, 2, 6, 2
    cache = tbf16.PagedCache(B, H, head_dim, 200, layers=L, page_size=16, dtype=dtype, track=True)
    g = torch.Generator().manual_seed(9)
    past = [[[], []] for _ in range(L)]
    total = torch.zeros(L, B, H, cache.capacity, dtype=torch.float64)
    lens, steps = [0] * B, []
    for T, counts in ((70, [70, 1, 33]), (1, None), (1, None), (4, None), (1, [1, 0, 1]), (1, None)):
        real = counts or [T] * B
        cache.advance(real)
        dc = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=DEV)
        lens = [n + c for n, c in zip(lens, real)]
        steps.append(real)
        assert cache.lengths == lens
        for layer in range(L):
            k, v = (torch.randn(B, H, T, head_dim, generator=g).bfloat16() for _ in range(2))
            q = torch.randn(B, Hq, T, head_dim, generator=g).bfloat16()
            cache.append(k.to(DEV), v.to(DEV), layer, counts=dc)
            out = cache.attend(q.to(DEV), layer, counts=dc).cpu().double()
            for x, kept in zip((k, v), past[layer]):
                if dtype == torch.float8_e4m3fn:
                    e = torch.frexp(x.float().abs().amax(-1, keepdim=True)).exponent
                    x = torch.ldexp(torch.ldexp(x.float(), 8 - e).to(dtype).float(), e - 8)
                kept.append(x.double())
            for b in range(B):
                kk, vv = (torch.cat([x[b, :, :c[b]] for x, c in zip(kept, steps)], 1) for kept in past[layer])
                for t in range(real[b]):
                    n = lens[b] - real[b] + t + 1
                    s = torch.einsum("hgd,hnd->hgn", q[b, :, t].double().view(H, 3, head_dim), kk[:, :n]) / math.sqrt(head_dim)
                    p = torch.softmax(s, -1)
                    ref = torch.einsum("hgn,hnd->hgd", p, vv[:, :n]).reshape(Hq, head_dim)
                    total[layer, b, :, :n] += p.sum(1)
                    assert bool(((out[b, :, t] - ref).abs() <= bf16_ulp(ref) + 2.0 ** -10 * vv.abs().max()).all())
                assert not out[b, :, real[b]:].any()
    assert torch.allclose(cache.weights.cpu().double(), total, rtol=1e-4, atol=1e-5)
    assert torch.equal(cache.pos[0, 0, 0, :lens[0]].cpu(), torch.arange(lens[0], dtype=torch.int32))


def test_evict_then_decode():
    """After a cut the cache holds the heaviest positions and the newest tokens; attention goes on over exactly
    those, and freed pages serve other sequences."""
    import tbf16
    B, H, D, keep, recent = 2, 2, 64, 48, 16
    cache = tbf16.PagedCache(B, H, D, 400, layers=1, pages=2 * 25, page_size=16, track=True)
    g = torch.Generator().manual_seed(4)
    rows = [torch.randn(B, H, 400, D, generator=g).bfloat16() for _ in range(2)]
    q = torch.randn(B, 4, 400, D, generator=g).bfloat16()
    cache.advance([300, 90])
    counts = torch.tensor([300, 90], dtype=torch.int32, device=DEV)
    cache.append(*(x[:, :, :300].to(DEV) for x in rows), counts=counts)
    cache.attend(q[:, :, :300].to(DEV), counts=counts)
    w = cache.weights[0].cpu()
    cache.evict(keep, recent)
    assert cache.lengths == [48, 48] and len(cache.pool.free) == 50 - 6
    for b, n in enumerate((300, 90)):
        for h in range(H):
            order = sorted(range(n), key=lambda i: (i < n - recent, -float(w[b, h, i]), i))[:keep]
            assert sorted(cache.pos[0, b, h, :keep].tolist()) == sorted(order)
            assert not cache.weights[0, b, h, keep:].any()
    cache.advance(1)
    at = torch.tensor([300, 90])
    k1, v1 = (x[torch.arange(B), :, at][:, :, None] for x in rows)
    cache.append(k1.to(DEV), v1.to(DEV))
    out = cache.attend(q[torch.arange(B), :, at][:, :, None].to(DEV)).cpu().double()
    pos = cache.pos[0].cpu().long()
    assert pos[:, :, 48].tolist() == [[300, 300], [90, 90]]
    for b in range(B):
        for h in range(H):
            k, v = (x[b, h, pos[b, h, :49]].double() for x in rows)
            p = torch.softmax(q[b, 2 * h:2 * h + 2, at[b]].double() @ k.T / math.sqrt(D), -1)
            ref = p @ v
            assert bool(((out[b, 2 * h:2 * h + 2, 0] - ref).abs() <= bf16_ulp(ref) + 2.0 ** -15 * v.abs().max()).all())
    cache.release(0)
    assert cache.lengths == [0, 49] and not cache.weights[0, 0].any()


def test_captured_step_follows_lengths():
    """One captured append + attend, replayed while the cache grows past a page, equals the eager calls."""
    import tbf16
    B, H, D = 2, 2, 128
    a, b = (tbf16.PagedCache(B, H, D, 100, page_size=16, track=True) for _ in range(2))
    g = torch.Generator(device=DEV).manual_seed(2)
    k, v = (torch.randn(B, H, 1, D, device=DEV, generator=g).bfloat16() for _ in range(2))
    q = torch.randn(B, 4, 1, D, device=DEV, generator=g).bfloat16()
    for c in (a, b):
        c.advance([14, 3])
        fill = torch.Generator(device=DEV).manual_seed(3)
        rows = torch.randn(2, B, H, 14, D, device=DEV, generator=fill).bfloat16()
        c.append(*rows, counts=c.lens.clone())
    graph = torch.cuda.CUDAGraph()
    a.attend(q)  # warm
    a.weights.zero_()
    with torch.cuda.graph(graph):
        a.append(k, v)
        out = a.attend(q)
    for _ in range(40):
        for x in (k, v, q):
            x.normal_(generator=g)
        a.advance(1)
        graph.replay()
        b.advance(1)
        b.append(k, v)
        assert torch.equal(out, b.attend(q))
    assert torch.equal(a.weights, b.weights) and torch.equal(a.k, b.k) and torch.equal(a.pos, b.pos)


def test_streams_side_by_side():
    """The same cache read on two streams at once, with the results of one stream alone."""
    case = Case([9000, 5000], 1, 128, 64)
    cache = case.cache()
    qs = [case.queries(8, 1, seed=i) for i in range(8)]
    want = [cache.attend(q) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i, q in enumerate(qs):
        with torch.cuda.stream(streams[i % 2]):
            got.append(cache.attend(q))
    torch.cuda.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_page_outside_the_pool_is_reported():
    """A page number the pool does not have sets bit 8 of the status word; nothing outside the pool is touched."""
    from tbf16 import _ext
    case = Case([40, 40], 2, 64, 16, poison=0.0)
    good = case.cache().attend(case.queries(4, 1))
    x = torch.randn(2, 2, 1, 64, device=DEV).bfloat16()
    assert _ext.device_status() == 0
    for bad in (-1, case.k.shape[0], 2 ** 31 - 1):
        case.dtable[0, 2] = bad
        before = case.k.clone()
        assert torch.equal(case.cache().attend(case.queries(4, 1))[1], good[1])
        assert _ext.device_status() == 8
        case.cache().append(x, x)
        assert _ext.device_status() == 8
        before[case.table[1, 2], :, 39 % 16] = x[1, :, 0]
        assert torch.equal(case.k, before)
        case.k[case.table[1, 2], :, 39 % 16] = case.k64[1, :, 39].bfloat16().to(DEV)
        case.v[case.table[1, 2], :, 39 % 16] = case.v64[1, :, 39].bfloat16().to(DEV)
    case.dtable[0, 2] = int(case.table[0, 2])
    for lens in ([-1, 40], [case.cap + 1, 40]):  # lengths outside the table are held inside it
        case.dlens.copy_(torch.tensor(lens, dtype=torch.int32))
        assert torch.equal(case.cache().attend(case.queries(4, 1))[1], good[1])
        assert _ext.device_status() == 8


def test_refusals():
    import tbf16
    from tbf16 import _ext
    case = Case([20, 5], 2, 64, 16)
    cache = case.cache()
    q, kv = case.queries(4, 1), torch.randn(2, 2, 1, 64, device=DEV).bfloat16()

    def refused(fn, *args, **kw):
        with pytest.raises(RuntimeError):
            fn(*args, **kw)
    refused(cache.attend, q.float())
    refused(cache.attend, q.cpu())
    refused(cache.attend, q[:1])
    refused(cache.attend, q[:, :3])  # 3 query heads over 2
    refused(cache.attend, q[..., :32])
    refused(cache.attend, q[0])
    refused(cache.attend, q, window=-1)
    refused(cache.attend, q, scale=float("nan"))
    refused(cache.attend, q, counts=torch.ones(2, device=DEV))
    refused(cache.attend, q, counts=torch.ones(3, device=DEV, dtype=torch.int32))
    refused(cache.attend, q, counts=torch.ones(2, dtype=torch.int32))
    refused(cache.attend, q.clone().requires_grad_())
    refused(cache.append, kv, kv[:, :, :0])
    refused(cache.append, kv.float(), kv)
    refused(cache.append, kv[:, :1], kv[:, :1])
    refused(cache.compact, 4)  # no weights
    refused(cache.advance, 1)  # the caller's buffers
    refused(cache.evict, 4)
    refused(cache.release, 0)
    over = tbf16.PagedCache.over
    refused(over, case.k.float(), case.v.float(), case.dtable, case.dlens)
    refused(over, case.k, case.v[:-1], case.dtable, case.dlens)
    refused(over, case.k[..., :32], case.v[..., :32], case.dtable, case.dlens)
    refused(over, case.k[:, :, :12], case.v[:, :, :12], case.dtable, case.dlens)
    refused(over, case.k, case.v, case.dtable.long(), case.dlens)
    refused(over, case.k, case.v, case.dtable, case.dlens[:1])
    refused(over, case.k, case.v, case.dtable.cpu(), case.dlens)
    refused(over, case.k, case.v, case.dtable, case.dlens, k_scale=torch.ones(case.k.shape[:3], device=DEV))
    refused(over, case.k, case.v, case.dtable, case.dlens, weights=torch.zeros(2, 2, case.cap - 1, device=DEV))
    refused(over, case.k, case.v, case.dtable, case.dlens, pos=torch.zeros(2, 2, case.cap, device=DEV, dtype=torch.int32))
    refused(tbf16.PagedCache, 2, 2, 64, 64, page_size=24)
    refused(tbf16.PagedCache, 2000, 1, 64, 16, page_size=16)
    own = tbf16.PagedCache(2, 2, 64, 64, page_size=16, pages=3)
    refused(own.advance, [17, 17])
    refused(own.advance, [65, 0])
    # the C entry points refuse what the Python layer would not send them
    L, c = _ext.lib(), cache._layers[0]
    args = [c.ref, _ext.ptr(q), 256, 64, 256, 4, 1, None, 1.0, 0, _ext.ptr(q), 256, 64, 256, None, 0, 0, None, None, 0, None]
    for i, bad, status in ((0, None, 1), (1, None, 1), (1, q.data_ptr() + 2, 2), (2, -8, 1), (2, 4, 2), (5, 3, 1), (6, -1, 1),
                           (9, -1, 1)):
        assert L.tbf16_paged_attend(*(args[:i] + [bad] + args[i + 1:])) == status, (i, bad)
    s = _ext.PagedCacheStruct.from_buffer_copy(c.struct)
    for field, bad, status in (("D", 96, 6), ("page_size", 8, 6), ("batch", 1025, 1), ("pages", 0, 1), ("max_pages", 99, 1),
                               ("dtype", 1, 3), ("k", 0, 1), ("k", c.struct.k + 8, 2), ("k_sp", -16, 1), ("k_ss", 32, 1),
                               ("v_sh", 4, 2), ("table", 0, 1)):
        t = _ext.PagedCacheStruct.from_buffer_copy(s)
        setattr(t, field, bad)
        assert L.tbf16_paged_attend(*([_ext.ctypes.addressof(t)] + args[1:])) == status, field
        assert L.tbf16_paged_append(_ext.ctypes.addressof(t), _ext.ptr(kv), 128, 64, 64, _ext.ptr(kv), 128, 64, 64, 1, 64,
                                    None, None, 0, 0, None, None) == status, field
    assert _ext.device_status() == 0


def test_nothing_to_do():
    """No new tokens, no sequences that reach anything: no launch fails, nothing is written."""
    case = Case([0, 0], 2, 64, 16, poison=0.5, max_len=16)
    cache = case.cache(weights=torch.zeros(2, 2, 16, device=DEV))
    before = case.k.clone()
    assert not cache.attend(case.queries(4, 3)).any()
    assert cache.attend(case.queries(4, 0)).shape == (2, 4, 0, 64)
    none = torch.zeros(2, 2, 0, 64, device=DEV, dtype=torch.bfloat16)
    cache.append(none, none)
    assert torch.equal(case.k, before) and not cache.weights.any()

"""A paged key/value cache for token-by-token decoding, and the three operators that work on it.

    cache = tbf16.PagedCache(batch, kv_heads, head_dim, max_len, layers=L)     # bf16; dtype=torch.float8_e4m3fn
    cache.advance(T)                        # room for T new tokens of every sequence (or a count for each)
    cache.append(k, v, layer)               # k, v (B, kv_heads, T, head_dim): into the pages, by those counts
    out = cache.attend(q, layer)            # q (B, heads, T, head_dim): attention over everything cached
    cache.rewind(counts)                    # drafts that were not accepted: the newest tokens of each sequence go
    cache.evict(keep, recent)               # with track=True: cut every head to its heaviest positions

`append` writes bf16 rows as they are, or as e4m3 rows with an exact power-of-two scale from the row's
largest exponent (the same idea as the fp16 rows of the linears, at half the bytes). `attend` is the
attention of the newest token or few tokens (decode, draft verification) over the pages; with `track=True`
it also adds each cached position's attention weight to `cache.weights`. `evict` keeps, per head, the
positions with the largest weights and closes the holes in place (`compact` does one layer). Prompts take
tbf16.sdpa on the prompt's own k and v, after `append`; sdpa leaves no weights, so where a cut is to know a
prompt, `attend` on the queries of its last tokens starts them.

Everything a kernel reads that changes from step to step (page table, lengths) lives on the GPU, so a
decoding step can be captured in a CUDA graph and replayed after `advance`. No host synchronisation.
The reference has no counterpart: it leaves calls with few query rows to torch (tbf16/convert.py there).
"""
import ctypes

import torch

from ._ext import BF16, E4M3, PagedCacheStruct, check, lib, require_cuda

KERNEL_D = (64, 128, 256)  # row lengths of the cache; other head dims are zero-padded up
MAX_BATCH = 1024
_DTYPES = {torch.bfloat16: BF16, torch.float8_e4m3fn: E4M3}


def _kernel_dim(d):
    for D in KERNEL_D:
        if d <= D:
            return D
    raise RuntimeError(f"tbf16.PagedCache: head dims up to {KERNEL_D[-1]}, got {d}")


def _rows(x, name, B, H, d, device, width):
    """A bf16 (B, H, T, d) tensor as the kernels read it: 16-byte rows, contiguous last dimension, widened with zeros
    to `width` columns."""
    if x.dtype != torch.bfloat16 or x.device != device:
        require_cuda(x)
        raise RuntimeError(f"tbf16.PagedCache: {name} must be bf16 on {device}, got {x.dtype} on {x.device}")
    if x.dim() != 4 or x.shape[0] != B or (H and x.shape[1] != H) or x.shape[3] != d:
        raise RuntimeError(f"tbf16.PagedCache: {name} must be ({B}, {H or 'heads'}, T, {d}), got {tuple(x.shape)}")
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"tbf16.PagedCache: {name} requires grad; the cache is for inference (use torch.no_grad)")
    sb, sh, st, se = x.stride()
    if d != width:
        wide = x.new_zeros((*x.shape[:3], width))
        wide[..., :d] = x
        return wide
    if se != 1 or (sb | sh | st) & 7 or x.data_ptr() & 15:
        # clone: also rewrites odd strides of dimensions of one element, which count as contiguous
        x = x.clone(memory_format=torch.contiguous_format)
    return x


class _Layer:
    """One layer's buffers and their description for the library."""

    def __init__(self, k, v, k_scale, v_scale, table, lens, weights, pos, seen, fresh):
        self.k, self.v, self.k_scale, self.v_scale, self.weights, self.pos = k, v, k_scale, v_scale, weights, pos
        pages, heads, page_size, D = k.shape
        c = self.struct = PagedCacheStruct()
        c.k, c.v, c.table, c.lens = k.data_ptr(), v.data_ptr(), table.data_ptr(), lens.data_ptr()
        c.k_sp, c.k_sh, c.k_ss = k.stride()[:3]
        c.v_sp, c.v_sh, c.v_ss = v.stride()[:3]
        if k_scale is not None:
            c.k_scale, c.v_scale = k_scale.data_ptr(), v_scale.data_ptr()
            c.ks_sp, c.ks_sh = k_scale.stride()[:2]
            c.vs_sp, c.vs_sh = v_scale.stride()[:2]
        c.table_ld, c.batch, c.max_pages = table.stride(0), table.shape[0], table.shape[1]
        c.heads, c.D, c.page_size, c.pages, c.dtype = heads, D, page_size, pages, _DTYPES[k.dtype]
        c.fresh = None if fresh is None else fresh.data_ptr()
        self.ref, self.D = ctypes.addressof(c), D
        self.weight_args = (None, 0, 0) if weights is None else (weights.data_ptr(), *weights.stride()[:2])
        self.pos_args = (None, 0, 0, None) if pos is None else (pos.data_ptr(), *pos.stride()[:2], seen.data_ptr())


class PagePool:
    """Which pages belong to which sequence, on the host."""

    def __init__(self, batch, pages, page_size, max_len):
        self.page_size, self.max_len = page_size, max_len
        self.lengths, self.seen, self.fresh = [0] * batch, [0] * batch, [0] * batch  # fresh: of the last advance
        self.fixed = [0] * batch  # positions that an eviction has reordered: they cannot be rewound into
        self.owned = [[] for _ in range(batch)]
        self.free = list(range(pages - 1, -1, -1))

    def advance(self, counts) -> bool:
        """Adds counts tokens; takes the pages they need. Returns whether the table changed. Changes nothing
        when it raises."""
        counts = self._counts(counts, "advance")
        new = [n + c for n, c in zip(self.lengths, counts)]
        if max(new) > self.max_len:
            raise RuntimeError(f"tbf16.PagedCache.advance: a sequence would pass max_len = {self.max_len}")
        want = [max(0, -(-n // self.page_size) - len(own)) for n, own in zip(new, self.owned)]
        if sum(want) > len(self.free):
            raise RuntimeError(f"tbf16.PagedCache.advance: out of pages ({sum(want)} wanted, {len(self.free)} free)")
        for own, w in zip(self.owned, want):
            own.extend(self.free.pop() for _ in range(w))
        self.lengths, self.fresh = new, counts
        self.seen = [s + c for s, c in zip(self.seen, counts)]
        return any(want)

    def _counts(self, counts, what):
        batch = len(self.lengths)
        counts = [counts] * batch if isinstance(counts, int) else [int(c) for c in counts]
        if len(counts) != batch or min(counts) < 0:
            raise RuntimeError(f"tbf16.PagedCache.{what}: {batch} counts of at least 0 expected, got {counts}")
        return counts

    def rewind(self, counts):
        """Takes the newest counts tokens back, as if they had never come. Changes nothing when it raises."""
        counts = self._counts(counts, "rewind")
        for b, (n, c, least) in enumerate(zip(self.lengths, counts, self.fixed)):
            if c and n - c < least:
                raise RuntimeError(f"tbf16.PagedCache.rewind: sequence {b} can lose {n - least} tokens, not {c}")
        for b, c in enumerate(counts):
            self.cut(b, self.lengths[b] - c)
            self.seen[b] -= c
            self.fresh[b] = max(0, self.fresh[b] - c)

    def cut(self, sequence, length):
        """Shortens a sequence to at most `length` tokens and frees the pages past them."""
        own, n = self.owned[sequence], min(self.lengths[sequence], length)
        used = -(-n // self.page_size)
        self.free.extend(reversed(own[used:]))
        del own[used:]
        self.lengths[sequence] = n
        self.fresh[sequence] = min(self.fresh[sequence], n)

    def rows(self, width):
        """The page table: one row of `width` page numbers for each sequence, 0 past its pages."""
        return [own + [0] * (width - len(own)) for own in self.owned]


class PagedCache:
    """Keys and values of `batch` sequences in pages of `page_size` tokens, for `layers` layers.

    pages: pages in the pool of each layer, shared by the sequences (default: enough for every sequence at
    max_len). track=True keeps `weights` (fp32, attention weight summed over the queries so far) and `pos`
    (int32, the token's number in its sequence), both (layers, batch, kv_heads, capacity), for `evict`.

    lens / seen / table are device tensors: cached tokens, tokens ever appended, page numbers. Different streams may
    work on one cache if the caller orders their accesses."""

    def __init__(self, batch, kv_heads, head_dim, max_len, *, layers=1, pages=None, page_size=64,
                 dtype=torch.bfloat16, track=False, device="cuda"):
        if min(batch, kv_heads, head_dim, max_len, layers) < 1 or page_size < 1:
            raise RuntimeError("tbf16.PagedCache: batch, kv_heads, head_dim, max_len, layers and page_size must be positive")
        if dtype not in _DTYPES:
            raise RuntimeError(f"tbf16.PagedCache: dtype must be torch.bfloat16 or torch.float8_e4m3fn, got {dtype}")
        per = -(-max_len // page_size)
        pages = batch * per if pages is None else pages
        D = _kernel_dim(head_dim)
        dev = torch.device(device)
        raw = torch.bfloat16 if dtype == torch.bfloat16 else torch.uint8
        k, v = torch.zeros((2, layers, pages, kv_heads, page_size, D), device=dev, dtype=raw).view(dtype).unbind(0)
        ks = vs = None
        if dtype != torch.bfloat16:
            ks, vs = torch.ones((2, layers, pages, kv_heads, page_size), device=dev).unbind(0)
        ints = dict(device=dev, dtype=torch.int32)
        shape = (layers, batch, kv_heads, per * page_size)
        weights = torch.zeros(shape, device=dev) if track else None
        pos = torch.full(shape, -1, **ints) if track else None
        self._state = torch.zeros((3, batch), **ints)  # lens, seen, fresh
        lens, seen, fresh = self._state.unbind(0)
        self._init(k, v, ks, vs, torch.zeros((batch, per), **ints), lens, seen, weights, pos, head_dim, fresh)
        self.pool = PagePool(batch, pages, page_size, max_len)

    @classmethod
    def over(cls, k, v, table, lens, *, k_scale=None, v_scale=None, weights=None, pos=None, seen=None, head_dim=None):
        """A one-layer cache over the caller's buffers: pools (pages, kv_heads, page_size, D) with any
        16-byte strides, table (batch, max_pages) and lens (batch) int32; e4m3 pools take k_scale and v_scale
        (pages, kv_heads, page_size). weights / pos / seen as in the class. The caller manages pages, table and
        lens; `advance`, `rewind`, `release` and `evict` are for caches that own them."""
        self = cls.__new__(cls)
        up = lambda x: None if x is None else x.unsqueeze(0)  # noqa: E731
        self._init(up(k), up(v), up(k_scale), up(v_scale), table, lens, seen, up(weights), up(pos), head_dim or k.shape[-1])
        self.pool = None
        return self

    def _init(self, k, v, k_scale, v_scale, table, lens, seen, weights, pos, head_dim, fresh=None):
        require_cuda(k, v, table, lens, k_scale, v_scale, seen, weights, pos)
        if k.dtype not in _DTYPES or v.dtype != k.dtype:
            raise RuntimeError(f"tbf16.PagedCache: bf16 or e4m3 pools expected, got {k.dtype} and {v.dtype}")
        if k.dim() != 5 or k.shape != v.shape or k.shape[-1] not in KERNEL_D or k.stride(-1) != 1 or v.stride(-1) != 1:
            raise RuntimeError(f"tbf16.PagedCache: pools of (pages, heads, page_size, D in {KERNEL_D}) with contiguous "
                               f"rows expected, got {tuple(k.shape[1:])} and {tuple(v.shape[1:])}")
        L, _, heads, page_size, D = k.shape
        if page_size & (page_size - 1) or not 16 <= page_size <= 1024:
            raise RuntimeError(f"tbf16.PagedCache: page_size must be a power of two from 16 to 1024, got {page_size}")
        if not 1 <= head_dim <= D:
            raise RuntimeError(f"tbf16.PagedCache: head_dim {head_dim} does not fit rows of {D}")
        for x in (table, lens, seen, pos):
            if x is not None and x.dtype != torch.int32:
                raise RuntimeError(f"tbf16.PagedCache: table, lens, seen and pos are int32, got {x.dtype}")
        if table.dim() != 2 or table.stride(1) != 1 or lens.shape != table.shape[:1] or not lens.is_contiguous():
            raise RuntimeError("tbf16.PagedCache: table (batch, max_pages) and lens (batch) with contiguous last dimensions")
        if table.shape[0] > MAX_BATCH:
            raise RuntimeError(f"tbf16.PagedCache: up to {MAX_BATCH} sequences, got {table.shape[0]}")
        if (k.dtype != torch.bfloat16) != (k_scale is not None) or (k_scale is None) != (v_scale is None):
            raise RuntimeError("tbf16.PagedCache: k_scale and v_scale belong to e4m3 pools, and only to them")
        for x in (k_scale, v_scale):
            if x is not None and (x.dtype != torch.float32 or x.shape != k.shape[:4] or x.stride(-1) != 1):
                raise RuntimeError("tbf16.PagedCache: scales are fp32 (pages, heads, page_size)")
        B, cap = table.shape[0], table.shape[1] * page_size
        for x, dt in ((weights, torch.float32), (pos, torch.int32)):
            if x is not None and (x.dtype != dt or x.dim() != 4 or x.shape[:3] != (L, B, heads) or x.shape[3] < cap
                                  or x.stride(-1) != 1):
                raise RuntimeError(f"tbf16.PagedCache: weights (fp32) and pos (int32) are (batch, heads, at least {cap})")
        if weights is not None and pos is not None and weights.shape != pos.shape:
            raise RuntimeError(f"tbf16.PagedCache: weights {tuple(weights.shape[1:])} and pos {tuple(pos.shape[1:])} differ")
        if pos is not None and (seen is None or seen.shape != lens.shape or not seen.is_contiguous()):
            raise RuntimeError("tbf16.PagedCache: pos needs seen (batch)")
        self.device, self.batch, self.kv_heads, self.page_size, self.capacity = k.device, B, heads, page_size, cap
        if any(x is not None and x.device != k.device for x in (v, table, lens, seen, weights, pos, k_scale, v_scale)):
            raise RuntimeError("tbf16.PagedCache: all tensors on one device")
        self.head_dim, self.dtype, self.table, self.lens, self.seen = head_dim, k.dtype, table, lens, seen
        self.k, self.v, self.k_scale, self.v_scale, self.weights, self.pos = k, v, k_scale, v_scale, weights, pos
        pick = lambda x, i: None if x is None else x[i]  # noqa: E731
        self._layers = [_Layer(k[i], v[i], pick(k_scale, i), pick(v_scale, i), table, lens, pick(weights, i), pick(pos, i),
                               seen, fresh) for i in range(L)]
        self._sizes, self._buffers, self._lib = {}, {}, lib()

    # ------------------------------------------------------------------------------------------- host side

    def _owned(self, what) -> PagePool:
        if self.pool is None:
            raise RuntimeError(f"tbf16.PagedCache.{what}: this cache is over buffers that the caller manages")
        return self.pool

    def _stepping(self, what) -> PagePool:
        """The pool, for a call that changes it. Its upload would be recorded by a capture, with these lengths."""
        pool = self._owned(what)
        with torch.cuda.device(self.device):
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"tbf16.PagedCache.{what}: not inside a graph capture; call it before each replay")
        return pool

    @property
    def lengths(self):
        """The host's copy of lens."""
        return list(self._owned("lengths").lengths)

    def advance(self, counts):
        """Makes room for counts new tokens (an int for every sequence, or one int each): takes pages from the
        pool and raises lens and seen. Call it once a step, before `append` and `attend` of every layer, which take
        these counts unless they are given others."""
        self._upload(table=self._stepping("advance").advance(counts))

    def rewind(self, counts):
        """Takes back the newest tokens (an int for every sequence, or one int each), as after drafts that were not
        accepted: lens and seen fall, pages past them go back to the pool, their weights and token numbers are
        cleared. What their queries added to the weights of earlier positions stays. Tokens that an `evict` has
        reordered cannot be taken back."""
        pool = self._stepping("rewind")
        old = list(pool.lengths)
        pool.rewind(counts)
        if self.weights is not None:
            for b, (n, new) in enumerate(zip(old, pool.lengths)):
                if new < n:
                    self.weights[:, b, :, new:n] = 0
                    self.pos[:, b, :, new:n] = -1
        self._upload(table=False)

    def release(self, sequence):
        """Forgets a sequence: its slot is empty again and its pages go back to the pool."""
        pool = self._stepping("release")
        pool.cut(sequence, 0)
        pool.seen[sequence] = pool.fixed[sequence] = 0
        if self.weights is not None:
            self.weights[:, sequence] = 0
            self.pos[:, sequence] = -1
        self._upload(table=False)

    def _upload(self, table):
        """lens, seen, the new counts and, where it changed, the table to the GPU, in stream order and without waiting for it: from
        pinned memory that torch's allocator does not hand out again before the copy is done."""
        pinned = dict(dtype=torch.int32, pin_memory=True)
        self._state.copy_(torch.tensor([self.pool.lengths, self.pool.seen, self.pool.fresh], **pinned), non_blocking=True)
        if table:
            self.table.copy_(torch.tensor(self.pool.rows(self.table.shape[1]), **pinned), non_blocking=True)

    def _counts(self, counts):
        if counts is None:
            return None
        if (not isinstance(counts, torch.Tensor) or counts.dtype is not torch.int32 or counts.device != self.device
                or counts.dim() != 1 or counts.numel() != self.batch or not counts.is_contiguous()):
            raise RuntimeError(f"tbf16.PagedCache: counts must be a contiguous int32 ({self.batch},) tensor on {self.device}")
        return counts.data_ptr()

    def _elsewhere(self, call, *args):
        """A call made while another device is current: again, with the cache's current. The library's size queries, the
        question whether a capture is on, allocations and launches all go by that."""
        with torch.cuda.device(self.device):
            return call(*args)

    def _run(self, fn, what, *args):
        status = fn(*args)
        if status:
            check(status, what)

    def _scratch(self, stream, sync, size):
        """Device memory for one attend call: `sync` zeroed bytes, which the call leaves zero, then its workspace.
        One buffer for each stream, reused by the stream's next call. A captured call gets its own, zeroed in the
        graph, so that graphs share nothing with each other or with calls outside."""
        buf = None if torch._C._cuda_isCurrentStreamCapturing() else self._buffers.get(stream)
        if buf is None or buf.sync < sync or buf.numel() - buf.sync < size:
            buf = torch.empty(sync + size, device=self.device, dtype=torch.uint8)
            buf[:sync].zero_()
            buf.sync = sync  # its workspace starts there, also for calls that need less
            if not torch._C._cuda_isCurrentStreamCapturing():
                self._buffers[stream] = buf
        return buf

    # ------------------------------------------------------------------------------------------- operators

    def append(self, k, v, layer=0, counts=None):
        """Writes the newest rows of every sequence into the pages: k, v bf16 (B, kv_heads, T, head_dim), any
        strides. lens counts them already (`advance`). counts: int32 (B,) on the GPU, the tokens that are real
        in each sequence (the first ones of its T; default: those of the last `advance`, at most T; over a caller's
        buffers T, or lens where that is less)."""
        if torch._C._cuda_getDevice() != self.device.index:
            return self._elsewhere(self.append, k, v, layer, counts)
        c, d = self._layers[layer], self.head_dim
        k = _rows(k, "k", self.batch, self.kv_heads, d, self.device, d + -d % 8)
        v = _rows(v, "v", self.batch, self.kv_heads, d, self.device, d + -d % 8)
        if k.shape != v.shape:
            raise RuntimeError(f"tbf16.PagedCache.append: k {tuple(k.shape)} and v {tuple(v.shape)} differ")
        _, _, T, d = k.shape
        kb, kh, kt, _ = k.stride()
        vb, vh, vt, _ = v.stride()
        self._run(self._lib.tbf16_paged_append, "append", c.ref, k.data_ptr(), kb, kh, kt, v.data_ptr(), vb, vh, vt, T, d,
                  self._counts(counts), *c.pos_args, torch._C._cuda_getCurrentRawStream(self.device.index))

    def attend(self, q, layer=0, counts=None, scale=None, window=0):
        """Attention of the newest T tokens over the cache: q bf16 (B, heads, T, head_dim), heads a multiple of
        kv_heads -> bf16 of the same shape, over (B, T, heads, head_dim) memory as tbf16.sdpa returns it. counts as in
        `append`. Token t of a sequence sits at position lens - counts + t and sees the positions up to its own; window > 0: only
        the last `window` of them. Rows past counts, and rows that see nothing, are zeros. A tracking cache adds
        the attention weights to `weights`."""
        if torch._C._cuda_getDevice() != self.device.index:
            return self._elsewhere(self.attend, q, layer, counts, scale, window)
        c, d = self._layers[layer], self.head_dim
        # zero columns leave the logits unchanged and give zero output columns
        q = _rows(q, "q", self.batch, 0, d, self.device, c.D)
        B, Hq, T, D = q.shape
        if window < 0:
            raise RuntimeError("tbf16.PagedCache.attend: window must not be negative")
        sizes = self._sizes.get((Hq, T))
        if sizes is None:
            if Hq == 0 or Hq % self.kv_heads:
                raise RuntimeError(f"tbf16.PagedCache.attend: {Hq} query heads over {self.kv_heads} key/value heads")
            n = int(self._lib.tbf16_paged_attend_sync_size(c.ref, Hq, T))
            sizes = self._sizes[(Hq, T)] = ((n + 255) // 256 * 256,
                                            int(self._lib.tbf16_paged_attend_ws_size(c.ref, Hq, T, int(c.weights is not None))))
        sync, size = sizes
        row = Hq * D
        out = torch.empty_strided((B, Hq, T, D), (T * row, D, row, 1), device=self.device, dtype=torch.bfloat16)
        stream = torch._C._cuda_getCurrentRawStream(self.device.index)
        buf = self._scratch(stream, sync, size)
        ptr = buf.data_ptr()
        sb, sh, st, _ = q.stride()
        self._run(self._lib.tbf16_paged_attend, "attend", c.ref, q.data_ptr(), sb, sh, st, Hq, T, self._counts(counts),
                  d ** -0.5 if scale is None else float(scale), int(window), out.data_ptr(), T * row, D, row, *c.weight_args, ptr,
                  ptr + buf.sync, size, stream)
        return out[..., :d] if d != D else out

    def compact(self, keep, recent=0, layer=0):
        """Cuts one layer's sequences to their `keep` heaviest positions per head, the newest `recent` tokens
        first of all, and moves the kept rows that lie beyond `keep` into the holes. Returns (weights, pos) in
        the new order, 0 and -1 past the end; weights, pos and lens of the cache are left as they were, so that
        every layer sees the same lengths (`evict` does all layers and then takes over the results)."""
        if torch._C._cuda_getDevice() != self.device.index:
            return self._elsewhere(self.compact, keep, recent, layer)
        c = self._layers[layer]
        if c.weights is None or c.pos is None or self.seen is None:
            raise RuntimeError("tbf16.PagedCache.compact: needs a cache with weights, pos and seen (track=True)")
        if keep < 0 or recent < 0:
            raise RuntimeError("tbf16.PagedCache.compact: keep and recent must not be negative")
        cols = c.weights.shape[2]
        size = self._sizes.get(keep)
        if size is None:
            size = self._sizes[keep] = int(self._lib.tbf16_paged_compact_ws_size(c.ref, cols, keep))
        shape = c.weights.shape
        weights, pos = c.weights.new_empty(shape), c.pos.new_empty(shape)
        stream = torch._C._cuda_getCurrentRawStream(self.device.index)
        buf = self._scratch(stream, 0, size)
        self._run(self._lib.tbf16_paged_compact, "compact", c.ref, *c.weight_args, *c.pos_args[:3], cols, c.pos_args[3], keep,
                  recent, weights.data_ptr(), pos.data_ptr(), buf.data_ptr() + buf.sync, size, stream)
        return weights, pos

    def evict(self, keep, recent=0):
        """`compact` for every layer, then the lengths: sequences longer than keep are keep long from here on,
        and pages that hold nothing any more go back to the pool. Cached order is no longer token order
        (`pos` has the token numbers), so a `window` no longer means the newest tokens."""
        pool = self._stepping("evict")
        for i, c in enumerate(self._layers):
            weights, pos = self.compact(keep, recent, i)
            c.weights.copy_(weights)
            c.pos.copy_(pos)
        for b, n in enumerate(pool.lengths):
            if n > keep:
                pool.cut(b, keep)
                pool.fixed[b] = keep
        self._upload(table=False)

// Writing to a paged key/value cache (append) and cutting it to a budget (compact).
#include <cuda_fp8.h>

#include <algorithm>

#include "paged.cuh"

namespace tbf16_host {

int paged_view(const tbf16_paged_cache* c, tbf16::PagedView* v) {
  if (!c) return TBF16_ERR_INVALID;
  if (c->dtype != TBF16_BF16 && c->dtype != TBF16_E4M3) return TBF16_ERR_DTYPE;
  const bool e4m3 = c->dtype == TBF16_E4M3;
  if (!c->k || !c->v || !c->table || !c->lens || e4m3 != (c->k_scale != nullptr) || e4m3 != (c->v_scale != nullptr))
    return TBF16_ERR_INVALID;
  if (c->D != 64 && c->D != 128 && c->D != 256) return TBF16_ERR_UNSUPPORTED;
  if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1))) return TBF16_ERR_UNSUPPORTED;
  if (c->batch < 0 || c->batch > 1024 || c->heads < 1 || c->heads > 1024) return TBF16_ERR_INVALID;
  if (c->pages < 1 || c->pages > INT32_MAX || c->max_pages < 1 || c->table_ld < c->max_pages ||
      c->max_pages > INT32_MAX / 2 / c->page_size)
    return TBF16_ERR_INVALID;
  const int64_t item = e4m3 ? 1 : 2;
  const int64_t strides[6] = {c->k_sp, c->k_sh, c->k_ss, c->v_sp, c->v_sh, c->v_ss};
  for (int64_t s : strides)
    if (s < 0 || s > (INT64_C(1) << 39) / item) return TBF16_ERR_INVALID;
  for (int64_t s : strides)
    if (s * item % 16) return TBF16_ERR_ALIGN;
  if (c->k_ss < c->D || c->v_ss < c->D) return TBF16_ERR_INVALID;
  if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->k_scale) || !aligned16(c->v_scale)) return TBF16_ERR_ALIGN;
  if (e4m3)
    for (int64_t s : {c->ks_sp, c->ks_sh, c->vs_sp, c->vs_sh}) {
      if (s < 0) return TBF16_ERR_INVALID;
      if (s % 4) return TBF16_ERR_ALIGN;
    }
  const DeviceInfo* d = device_info();
  if (!d) return TBF16_ERR_DEVICE;
  v->k = static_cast<uint8_t*>(c->k);
  v->v = static_cast<uint8_t*>(c->v);
  v->k_scale = c->k_scale;
  v->v_scale = c->v_scale;
  v->table = c->table;
  v->lens = c->lens;
  v->k_sp = c->k_sp * item; v->k_sh = c->k_sh * item; v->k_ss = c->k_ss * item;
  v->v_sp = c->v_sp * item; v->v_sh = c->v_sh * item; v->v_ss = c->v_ss * item;
  v->ks_sp = c->ks_sp; v->ks_sh = c->ks_sh; v->vs_sp = c->vs_sp; v->vs_sh = c->vs_sh;
  v->table_ld = c->table_ld;
  v->pages = c->pages;
  v->batch = (int)c->batch;
  v->heads = (int)c->heads;
  v->page_shift = 0;
  while ((INT64_C(1) << v->page_shift) < c->page_size) ++v->page_shift;
  v->max_pages = (int)c->max_pages;
  v->cap = (int)(c->max_pages << v->page_shift);
  v->err = d->err;
  return TBF16_OK;
}

}  // namespace tbf16_host

namespace {
using namespace tbf16;

// ------------------------------------------------------------------ append

struct AppendParams {
  PagedView c;
  const __nv_bfloat16* src[2];  // k, v
  int64_t sb[2], sh[2], st[2];
  const int* counts;
  const int* seen;
  int* pos;
  int64_t pos_sb, pos_sh;
  int T, d8;       // d8: source row length in 8-element vectors
  int tp_log2;     // log2 of the tokens of a pass
  int tiles;       // blocks of a sequence, kAppendVectors passes of tokens each
  int block_heads; // heads of a block
};
constexpr int kAppendVectors = 4;  // rows that a thread has in flight

// Eight bf16 values times `scale` (a power of two: exact short of e4m3's range) rounded to nearest-even e4m3.
__device__ __forceinline__ uint2 e4m3x8(uint4 x, float scale) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    h[i] = __nv_cvt_float2_to_fp8x2(make_float2(bf16lo(w[i]) * scale, bf16hi(w[i]) * scale), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}

// A block copies the rows of some tokens and heads of one sequence to their slots; blockIdx.y picks keys or values.
// D / 8 lanes hold a row, 8 elements each; the 256 D / 8 rows of a pass are 2^tp_log2 tokens (one when decoding) x
// heads, and a thread goes through the heads with the same kAppendVectors tokens, so that page numbers and offsets
// are worked out once and a row costs two pointer steps (with both strides multiplied out for each row, the 8-bit
// form was bound by instructions: 163 a row, 37 us where this takes AAA). Bound by HBM: each row is read once and
// written once.
// An e4m3 row is scaled by 2^(8 - e), e the exponent (frexp) of its largest magnitude, which lands in
// [128, 256): half the format's range stays unused, none of its precision does, and nothing can saturate.
template <int D, bool E4M3>
__global__ void __launch_bounds__(256) append_kernel(const AppendParams p) {
  constexpr int LR = D / 8, V = kAppendVectors, ROWS = 256 / LR;
  const int kv = blockIdx.y, chunk = threadIdx.x % LR, row = threadIdx.x / LR;
  const int b = (int)(blockIdx.x / (unsigned)p.tiles), tp = 1 << p.tp_log2;
  const int t0 = (int)(blockIdx.x % (unsigned)p.tiles) * (V * tp) + (row & (tp - 1));
  const int h0 = blockIdx.z * p.block_heads + (row >> p.tp_log2), h1 = min(p.c.heads, (int)(blockIdx.z + 1) * p.block_heads);
  const int hp = ROWS >> p.tp_log2;
  pdl_launch_dependents();
  pdl_wait();
  const int len = paged_len(p.c, b), n = paged_count(p.c, p.counts, b, p.T, len);
  if (t0 - (row & (tp - 1)) >= n) return;
  const __nv_bfloat16* src[V];
  uint8_t* dst[V];
  float* scale[V];
  const int64_t sh = kv ? p.c.v_sh : p.c.k_sh, ssh = kv ? p.c.vs_sh : p.c.ks_sh;
  int live = 0;  // bit i: token i is there and its page is in the pool
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int t = t0 + i * tp, j = len - n + t, page = t < n ? paged_page(p.c, b, j) : -1, slot = paged_slot(p.c, j);
    live |= (page >= 0) << i;
    src[i] = p.src[kv] + b * p.sb[kv] + h0 * p.sh[kv] + t * p.st[kv] + chunk * 8;
    dst[i] = (kv ? p.c.v + page * p.c.v_sp + slot * p.c.v_ss : p.c.k + page * p.c.k_sp + slot * p.c.k_ss) + h0 * sh +
             chunk * (E4M3 ? 8 : 16);
    if (E4M3) scale[i] = (kv ? p.c.v_scale + page * p.c.vs_sp : p.c.k_scale + page * p.c.ks_sp) + h0 * ssh + slot;
    if (p.pos && page >= 0 && kv == 0 && chunk == 0)
      for (int h = h0; h < h1; h += hp) p.pos[b * p.pos_sb + h * p.pos_sh + j] = p.seen[b] - n + t;
  }
  const int passes = (h1 - (int)(blockIdx.z * p.block_heads) + hp - 1) / hp;
#pragma unroll 1
  for (int k = 0, h = h0; k < passes; ++k, h += hp) {
    if (h >= h1) live = 0;
    uint4 x[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      x[i] = make_uint4(0, 0, 0, 0);
      if (((live >> i) & 1) && chunk < p.d8) x[i] = __ldcs(reinterpret_cast<const uint4*>(src[i]));
      src[i] += hp * p.sh[kv];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (E4M3) {
        // the largest magnitude as bits, ordered like the values with infinity and NaN on top; two in a register
        unsigned m = 0;
        for (uint32_t w : {x[i].x, x[i].y, x[i].z, x[i].w}) m = __vmaxu2(m, w & 0x7fff7fffu);
#pragma unroll
        for (int o = LR / 2; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
        m = max(m << 16, m & 0xffff0000u);
        const bool finite = m < 0x7f800000u;
        // its frexp exponent; at least -118 (2^-119), so that 2^(8 - e) and 2^(e - 8) are normal: smaller rows round
        // to e4m3's subnormals
        const int e = m == 0 || !finite ? 8 : (int)(max(m, 8u << 23) >> 23) - 126;
        const uint2 y = e4m3x8(x[i], __uint_as_float((unsigned)(135 - e) << 23));
        if ((live >> i) & 1) {
          *reinterpret_cast<uint2*>(dst[i]) = y;
          if (chunk == 0) *scale[i] = __uint_as_float(finite ? (unsigned)(119 + e) << 23 : 0x7fc00000u);
        }
        scale[i] += hp * ssh;
      } else if ((live >> i) & 1) {
        *reinterpret_cast<uint4*>(dst[i]) = x[i];
      }
      dst[i] += hp * sh;
    }
  }
}

template <int D>
int launch_append(AppendParams& p, bool e4m3, cudaStream_t st) {
  constexpr int ROWS = 256 / (D / 8);
  p.tp_log2 = 0;
  while ((2 << p.tp_log2) <= std::min(p.T, ROWS)) ++p.tp_log2;
  const int tokens = kAppendVectors << p.tp_log2, hp = ROWS >> p.tp_log2, passes = (p.c.heads + hp - 1) / hp;
  p.tiles = (p.T + tokens - 1) / tokens;
  const int64_t blocks = (int64_t)p.c.batch * p.tiles;
  if (blocks > INT32_MAX) return TBF16_ERR_INVALID;
  // a block takes several passes of heads only while there are four blocks an SM all the same
  const int sms = tbf16_host::device_info()->sms;
  const int64_t k = std::max<int64_t>(1, std::min<int64_t>(passes, 2 * blocks * passes / (4 * sms)));
  p.block_heads = (int)k * hp;
  return tbf16_host::launch_pdl(e4m3 ? append_kernel<D, true> : append_kernel<D, false>,
                                dim3((unsigned)blocks, 2, (unsigned)((p.c.heads + p.block_heads - 1) / p.block_heads)), 256, 0,
                                st, p);
}

// ------------------------------------------------------------------ compact

struct CompactParams {
  PagedView c;
  const float* w;
  const int* pos;
  int64_t w_sb, w_sh, p_sb, p_sh;
  const int* seen;
  int cols, keep, recent, row16;  // row16: 16-byte chunks of a key or value row
  int scaled;
  float* w_out;
  int* pos_out;
  int2* moves;  // (from, to) for each (sequence, head): at most max_moves
  int max_moves;
};

// Rank of a position as an unsigned integer: protected ones above every weight, then weights in the order of
// their values (NaN on top, -0 equal to 0).
__device__ __forceinline__ uint32_t rank_key(float w, int pos, int protect_from) {
  if (pos >= protect_from) return 0xffffffffu;
  if (w != w) return 0xffc00000u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Exclusive prefix of v over the block's 32 warps (one value per warp, the same in all its lanes), and the total.
__device__ __forceinline__ int warp_prefix(int v, int* scratch, int& total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  int x = scratch[lane], own = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    const int y = __shfl_sync(0xffffffffu, x, i);
    own += i < warp ? y : 0;
    total += y;
  }
  __syncthreads();
  return own;
}

// One block per (sequence, head): the keep-th largest key by a radix select (four 8-bit digits, counted in
// shared memory), then two passes that number the holes and the rows that fill them, then the copies.
__global__ void __launch_bounds__(1024) compact_kernel(const CompactParams p) {
  __shared__ int hist[256];
  __shared__ int scratch[32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_need;
  const int b = blockIdx.x / p.c.heads, h = blockIdx.x % p.c.heads;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int n = min(paged_len(p.c, b), p.cols);
  const float* w = p.w + b * p.w_sb + h * p.w_sh;
  const int* pos = p.pos + b * p.p_sb + h * p.p_sh;
  const int64_t out = (int64_t)blockIdx.x * p.cols;
  const int left = min(n, p.keep);
  for (int i = left + tid; i < p.cols; i += 1024) {
    p.w_out[out + i] = 0.f;
    p.pos_out[out + i] = -1;
  }
  if (n <= p.keep) {
    for (int i = tid; i < n; i += 1024) {
      p.w_out[out + i] = w[i];
      p.pos_out[out + i] = pos[i];
    }
    return;
  }
  if (p.keep == 0) return;
  const int protect_from = p.seen[b] - p.recent;
  uint32_t prefix = 0;
  int need = p.keep;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += 1024) {
      const uint32_t key = rank_key(w[i], pos[i], protect_from);
      if (shift == 24 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int above = 0, d = 255;
      while (d > 0 && above + hist[d] < need) above += hist[d--];
      s_prefix = prefix | ((uint32_t)d << shift);
      s_need = need - above;
    }
    __syncthreads();
    prefix = s_prefix;
    need = s_need;
    __syncthreads();
  }
  // `need` of the positions whose key equals `prefix` are kept, the lowest first
  const int per = ((n + 31) / 32 + 31) / 32 * 32, first = warp * per, last = min(n, first + per);
  int ties = 0, total;
  for (int i = first + lane; i - lane < last; i += 32)
    ties += __popc(__ballot_sync(0xffffffffu, i < last && rank_key(w[i], pos[i], protect_from) == prefix));
  const int ties_before = warp_prefix(ties, scratch, total);
  int2* moves = p.moves + (int64_t)blockIdx.x * p.max_moves;
  int holes_before = 0, loose_before = 0, holes = 0, loose = 0, count = 0;
  for (int write = 0; write < 2; ++write) {
    int tie = ties_before;
    holes = loose = 0;
    for (int i = first + lane; i - lane < last; i += 32) {
      const bool in = i < last;
      const uint32_t key = in ? rank_key(w[i], pos[i], protect_from) : 0u;
      const unsigned eq = __ballot_sync(0xffffffffu, in && key == prefix);
      const bool kept = in && (key > prefix || (key == prefix && tie + __popc(eq & ((1u << lane) - 1)) < need));
      tie += __popc(eq);
      const unsigned hb = __ballot_sync(0xffffffffu, in && !kept && i < p.keep);
      const unsigned lb = __ballot_sync(0xffffffffu, kept && i >= p.keep);
      if (write) {
        if ((hb >> lane) & 1) moves[holes_before + holes + __popc(hb & ((1u << lane) - 1))].y = i;
        if ((lb >> lane) & 1) moves[loose_before + loose + __popc(lb & ((1u << lane) - 1))].x = i;
        if (kept && i < p.keep) {
          p.w_out[out + i] = w[i];
          p.pos_out[out + i] = pos[i];
        }
      }
      holes += __popc(hb);
      loose += __popc(lb);
    }
    if (!write) {
      holes_before = warp_prefix(holes, scratch, count);
      loose_before = warp_prefix(loose, scratch, total);
    }
  }
  __syncthreads();
  for (int m = warp; m < count; m += 32) {
    const int2 mv = moves[m];
    const int from = paged_page(p.c, b, mv.x), to = paged_page(p.c, b, mv.y);
    if (lane == 0) {
      p.w_out[out + mv.y] = w[mv.x];
      p.pos_out[out + mv.y] = pos[mv.x];
    }
    if (from < 0 || to < 0) continue;
    const int sf = paged_slot(p.c, mv.x), st = paged_slot(p.c, mv.y);
    for (int i = lane; i < 2 * p.row16; i += 32) {
      const bool v = i >= p.row16;
      const int64_t off = (v ? i - p.row16 : i) * 16;
      uint8_t* pool = v ? p.c.v + h * p.c.v_sh + off : p.c.k + h * p.c.k_sh + off;
      const int64_t sp = v ? p.c.v_sp : p.c.k_sp, ss = v ? p.c.v_ss : p.c.k_ss;
      *reinterpret_cast<uint4*>(pool + to * sp + st * ss) = *reinterpret_cast<const uint4*>(pool + from * sp + sf * ss);
    }
    if (p.scaled && lane < 2) {
      float* s = lane ? p.c.v_scale + h * p.c.vs_sh : p.c.k_scale + h * p.c.ks_sh;
      const int64_t sp = lane ? p.c.vs_sp : p.c.ks_sp;
      s[to * sp + st] = s[from * sp + sf];
    }
  }
}

}  // namespace

extern "C" int tbf16_paged_append(const tbf16_paged_cache* cache, const void* k, int64_t k_sb, int64_t k_sh,
                                  int64_t k_st, const void* v, int64_t v_sb, int64_t v_sh, int64_t v_st, int64_t T,
                                  int64_t d, const int32_t* counts, int32_t* pos, int64_t pos_sb, int64_t pos_sh,
                                  const int32_t* seen, void* stream) {
  if (int st = tbf16_host::require_sm100()) return st;
  AppendParams p;
  if (int st = tbf16_host::paged_view(cache, &p.c)) return st;
  if (T == 0 || cache->batch == 0) return TBF16_OK;
  if (!k || !v || T < 0 || d < 8 || d > cache->D || (pos && !seen)) return TBF16_ERR_INVALID;
  if (T > INT32_MAX / 2) return TBF16_ERR_INVALID;
  for (int64_t s : {k_sb, k_sh, k_st, v_sb, v_sh, v_st}) {
    if (s < 0) return TBF16_ERR_INVALID;
    if (s % 8) return TBF16_ERR_ALIGN;
  }
  if (d % 8 || !tbf16_host::aligned16(k) || !tbf16_host::aligned16(v)) return TBF16_ERR_ALIGN;
  p.src[0] = static_cast<const __nv_bfloat16*>(k);
  p.src[1] = static_cast<const __nv_bfloat16*>(v);
  p.sb[0] = k_sb; p.sh[0] = k_sh; p.st[0] = k_st;
  p.sb[1] = v_sb; p.sh[1] = v_sh; p.st[1] = v_st;
  p.counts = counts;
  p.seen = seen;
  p.pos = pos;
  p.pos_sb = pos_sb;
  p.pos_sh = pos_sh;
  p.T = (int)T;
  p.d8 = (int)(d / 8);
  auto st = static_cast<cudaStream_t>(stream);
  const bool e4m3 = cache->dtype == TBF16_E4M3;
  if (cache->D == 64) return launch_append<64>(p, e4m3, st);
  if (cache->D == 128) return launch_append<128>(p, e4m3, st);
  return launch_append<256>(p, e4m3, st);
}

namespace {
int64_t compact_max_moves(int64_t cols, int64_t keep) { return std::max<int64_t>(0, std::min(keep, cols - keep)); }
}  // namespace

extern "C" int64_t tbf16_paged_compact_ws_size(const tbf16_paged_cache* cache, int64_t cols, int64_t keep) {
  if (!cache || cache->batch < 0 || cache->heads < 1 || cols < 0 || keep < 0) return 0;
  return cache->batch * cache->heads * compact_max_moves(cols, keep) * (int64_t)sizeof(int2);
}

extern "C" int tbf16_paged_compact(const tbf16_paged_cache* cache, const float* weights, int64_t w_sb, int64_t w_sh,
                                   const int32_t* pos, int64_t pos_sb, int64_t pos_sh, int64_t cols,
                                   const int32_t* seen, int64_t keep, int64_t recent, float* weights_out,
                                   int32_t* pos_out, void* ws, int64_t ws_bytes, void* stream) {
  if (int st = tbf16_host::require_sm100()) return st;
  CompactParams p;
  if (int st = tbf16_host::paged_view(cache, &p.c)) return st;
  if (!weights || !pos || !seen || !weights_out || !pos_out || cols < 0 || cols > INT32_MAX || keep < 0 ||
      keep > INT32_MAX || recent < 0 || recent > INT32_MAX)
    return TBF16_ERR_INVALID;
  const int64_t need = tbf16_paged_compact_ws_size(cache, cols, keep);
  if (need > 0 && (!ws || ws_bytes < need)) return TBF16_ERR_INVALID;
  if (reinterpret_cast<uintptr_t>(ws) % sizeof(int2)) return TBF16_ERR_ALIGN;
  const int64_t items = cache->batch * cache->heads;
  if (items == 0 || cols == 0) return TBF16_OK;
  p.w = weights; p.w_sb = w_sb; p.w_sh = w_sh;
  p.pos = pos; p.p_sb = pos_sb; p.p_sh = pos_sh;
  p.seen = seen;
  p.cols = (int)cols;
  p.keep = (int)keep;
  p.recent = (int)recent;
  p.scaled = cache->dtype == TBF16_E4M3;
  p.row16 = (int)(cache->D * (p.scaled ? 1 : 2) / 16);
  p.w_out = weights_out;
  p.pos_out = pos_out;
  p.moves = static_cast<int2*>(ws);
  p.max_moves = (int)compact_max_moves(cols, keep);
  compact_kernel<<<(unsigned)items, 1024, 0, static_cast<cudaStream_t>(stream)>>>(p);
  return tbf16_host::check_launch();
}

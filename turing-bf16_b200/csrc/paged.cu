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
  v->fresh = c->fresh;
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
  int tiles;       // blocks of a sequence, V passes of tokens each
  int block_heads; // heads of a block
};
// What a thread has in flight: N vectors of each of V rows. (Four rows of bf16 take as long for prompts, and 3.5 us in place
// of 2.6 for one token of 64 sequences.)
template <int D_, bool E4M3_>
struct AppendTile {
  static constexpr int D = D_;
  static constexpr bool E4M3 = E4M3_;
  static constexpr int N = E4M3 ? 2 : 1, V = 2;
  static constexpr int LR = D / 8 / N, ROWS = 256 / LR;  // lanes of a row, rows of a pass
};

// Eight bf16 values times `scale` (a power of two: exact in bf16 as far as e4m3 tells the products from zero) rounded
// to nearest-even e4m3.
__device__ __forceinline__ uint2 e4m3x8(uint4 x, __nv_bfloat162 scale) {
  const uint32_t w[4] = {x.x, x.y, x.z, x.w};
  uint32_t h[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    h[i] = __nv_cvt_float2_to_fp8x2(__bfloat1622float2(__hmul2(reinterpret_cast<const __nv_bfloat162&>(w[i]), scale)),
                                    __NV_SATFINITE, __NV_E4M3);
  return make_uint2(h[0] | (h[1] << 16), h[2] | (h[3] << 16));
}

// A block copies the rows of some tokens and heads of one sequence to their slots; blockIdx.y picks keys or values.
// LR lanes hold a row, N vectors of 8 elements each; the ROWS rows of a pass are 2^tp_log2 tokens (one when decoding)
// x heads, and a thread goes through the heads with the same V tokens, so that page numbers and offsets are worked
// out once and a row costs two pointer steps. Bound by the latency of its loads: for prompts of 127 MB (6 x 4 heads
// of 256, up to 4096 tokens: 24.7 us, 0.79 of the copy rate) 39 warps an SM wait for them, with 0.39 of the issue
// slots used and the DRAM 0.41 busy (its writes stay in L2); the 8-bit form has more instructions (8 x 8 heads of 128
// elements: 23 us; 33 with one vector of each of four rows, whose maxima and scales take twice as many, 37 with both
// strides multiplied out for each row). Each row is read once and written once.
// An e4m3 row is scaled by 2^(8 - e), e the exponent (frexp) of its largest magnitude, which lands in
// [128, 256): half the format's range stays unused, none of its precision does, and nothing can saturate.
template <class A>
__global__ void __launch_bounds__(256) append_kernel(const AppendParams p) {
  constexpr int LR = A::LR, V = A::V, N = A::N, ROWS = A::ROWS;
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
             chunk * (A::E4M3 ? 8 : 16);
    if (A::E4M3) scale[i] = (kv ? p.c.v_scale + page * p.c.vs_sp : p.c.k_scale + page * p.c.ks_sp) + h0 * ssh + slot;
    if (p.pos && page >= 0 && kv == 0 && chunk == 0)
      for (int h = h0; h < h1; h += hp) p.pos[b * p.pos_sb + h * p.pos_sh + j] = p.seen[b] - n + t;
  }
  const int passes = (h1 - (int)(blockIdx.z * p.block_heads) + hp - 1) / hp;
#pragma unroll 1
  for (int k = 0, h = h0; k < passes; ++k, h += hp) {
    if (h >= h1) live = 0;
    uint4 x[V][N];
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
      for (int c = 0; c < N; ++c) {
        x[i][c] = make_uint4(0, 0, 0, 0);
        if (((live >> i) & 1) && chunk + c * LR < p.d8) x[i][c] = __ldcs(reinterpret_cast<const uint4*>(src[i]) + c * LR);
      }
      src[i] += hp * p.sh[kv];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (A::E4M3) {
        // the largest magnitude as bits, ordered like the values with infinity and NaN on top; two in a register
        unsigned m = 0;
#pragma unroll
        for (int c = 0; c < N; ++c)
          for (uint32_t w : {x[i][c].x, x[i][c].y, x[i][c].z, x[i][c].w}) m = __vmaxu2(m, w & 0x7fff7fffu);
#pragma unroll
        for (int o = LR / 2; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
        m = max(m << 16, m & 0xffff0000u);
        const bool finite = m < 0x7f800000u;
        // its frexp exponent; at least -118 (2^-119), so that 2^(8 - e) and 2^(e - 8) are normal: smaller rows round
        // to e4m3's subnormals
        const int e = m == 0 || !finite ? 8 : (int)(max(m, 8u << 23) >> 23) - 126;
        const __nv_bfloat162 up = __bfloat162bfloat162(__ushort_as_bfloat16((unsigned short)((135 - e) << 7)));
        if ((live >> i) & 1) {
#pragma unroll
          for (int c = 0; c < N; ++c) *(reinterpret_cast<uint2*>(dst[i]) + c * LR) = e4m3x8(x[i][c], up);
          if (chunk == 0) *scale[i] = __uint_as_float(finite ? (unsigned)(119 + e) << 23 : 0x7fc00000u);
        }
        scale[i] += hp * ssh;
      } else if ((live >> i) & 1) {
        *reinterpret_cast<uint4*>(dst[i]) = x[i][0];
      }
      dst[i] += hp * sh;
    }
  }
}

template <class A>
int launch_append(AppendParams& p, cudaStream_t st) {
  p.tp_log2 = 0;
  while ((2 << p.tp_log2) <= std::min(p.T, A::ROWS)) ++p.tp_log2;
  const int tokens = A::V << p.tp_log2, hp = A::ROWS >> p.tp_log2, passes = (p.c.heads + hp - 1) / hp;
  p.tiles = (p.T + tokens - 1) / tokens;
  const int64_t blocks = (int64_t)p.c.batch * p.tiles;
  if (blocks > INT32_MAX) return TBF16_ERR_INVALID;
  // a block takes several passes of heads only while there are four blocks an SM all the same
  const int sms = tbf16_host::device_info()->sms;
  const int64_t k = std::max<int64_t>(1, std::min<int64_t>(passes, 2 * blocks * passes / (4 * sms)));
  p.block_heads = (int)k * hp;
  return tbf16_host::launch_pdl(append_kernel<A>,
                                dim3((unsigned)blocks, 2, (unsigned)((p.c.heads + p.block_heads - 1) / p.block_heads)), 256, 0,
                                1, st, p);
}
template <int D>
int launch_append(AppendParams& p, bool e4m3, cudaStream_t st) {
  return e4m3 ? launch_append<AppendTile<D, true>>(p, st) : launch_append<AppendTile<D, false>>(p, st);
}

// ------------------------------------------------------------------ compact

// Which positions a (sequence, head) keeps, in two kernels: select_kernel ranks the positions by weight and lists
// the moves, move_kernel makes them. Moves go from positions at or beyond `keep` to positions below it, so no
// row is both read and written and all of them run at once, on the whole GPU however few the items are.
struct CompactParams {
  PagedView c;
  const float* w;
  const int* pos;
  int64_t w_sb, w_sh, p_sb, p_sh;
  const int* seen;
  int cols, keep, recent;
  int row16_log2;  // 16-byte chunks of a key or value row
  int scaled;
  int in_smem;     // a CTA's keys stay in shared memory
  int inline_moves;  // select_kernel makes the moves itself
  float* w_out;
  int* pos_out;
  int* counts;     // moves of each (sequence, head)
  int* moves;      // where they come from, then where they go: max_moves each, for each
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

constexpr int kSelThreads = 1024;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kDigitBits = 11;  // keys are ranked by digits of 11, 11 and 10 bits: the first is sign, exponent and two
constexpr int kBins = 1 << kDigitBits;  // bits of the weight, so that like weights still spread over several counters

static_assert(kSelWarps == 32 && kBins == 64 * kSelWarps, "a warp for each group of 64 bins, a lane for each group");

// Another CTA's copy of a shared variable.
__device__ __forceinline__ int ld_cluster(const int* x, int cta) {
  int y;
  asm volatile("ld.shared::cluster.b32 %0, [%1];" : "=r"(y) : "r"(mapa_u32(smem_u32(x), cta)) : "memory");
  return y;
}
__device__ __forceinline__ int2 ld_cluster2(const int* x, int cta) {
  int2 y;
  asm volatile("ld.shared::cluster.v2.b32 {%0, %1}, [%2];" : "=r"(y.x), "=r"(y.y) : "r"(mapa_u32(smem_u32(x), cta)) : "memory");
  return y;
}
// Inclusive sums over the lanes.
__device__ __forceinline__ int scan_lanes(int x) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if ((int)(threadIdx.x & 31) >= o) x += y;
  }
  return x;
}

// Exclusive prefix of four counts (the same in all lanes of a warp) over the warps of the cluster, in order of CTA and
// warp, and the totals.
__device__ __forceinline__ int4 add4(int4 a, int4 b) { return make_int4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }
__device__ __forceinline__ int4 warp_sum(int4 v) {
  return make_int4(__reduce_add_sync(0xffffffffu, v.x), __reduce_add_sync(0xffffffffu, v.y),
                   __reduce_add_sync(0xffffffffu, v.z), __reduce_add_sync(0xffffffffu, v.w));
}
__device__ __forceinline__ int4 cluster_scan(int4 v, int ctas, int rank, int4* warp_sums, int4* cta_sum, int4& total) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int4 zero = make_int4(0, 0, 0, 0);
  if (lane == 0) warp_sums[warp] = v;
  __syncthreads();
  const int4 x = lane < kSelWarps ? warp_sums[lane] : zero;
  int4 before = warp_sum(lane < warp ? x : zero);
  total = warp_sum(x);
  if (ctas > 1) {
    if (threadIdx.x == 0) *cta_sum = total;
    cluster_sync();
    int4 y = zero;
    if (lane < ctas)
      asm volatile("ld.shared::cluster.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(y.x), "=r"(y.y), "=r"(y.z), "=r"(y.w)
                   : "r"(mapa_u32(smem_u32(cta_sum), lane)));
    before = add4(before, warp_sum(lane < rank ? y : zero));
    total = warp_sum(y);
    cluster_sync();  // no CTA ends while its counts are read
  }
  return before;
}

// Makes moves m0, m0 + kMoveRows * stride, ... of an item: looks up the pages of kMoveRows moves, then streams the
// rows, 16 bytes a thread, V loads in flight, and last stores the moves' scales, weights and numbers, which come in
// meanwhile. 84000 moves of 512 bytes with 256 threads: 15 us with 128 rows and four loads; 16.4 with 64 and four, 17.6
// with 128 and eight, 19.7 with 64 and eight or 32 and four; copying them takes 13 at the HBM rate.
constexpr int kMoveRows = 128;
struct MoveScratch {
  int64_t from[2][kMoveRows], to[2][kMoveRows];  // byte offsets of keys, values; -1: not to be copied
};
template <int THREADS, int V>
__device__ __forceinline__ void move_rows(const CompactParams& p, int bh, int count, int m0, int stride, MoveScratch& s) {
  const int b = bh / p.c.heads, h = bh % p.c.heads, tid = threadIdx.x;
  const int chunk = tid & ((1 << p.row16_log2) - 1), value = (tid >> p.row16_log2) & 1;
  uint8_t* pool = (value ? p.c.v + h * p.c.v_sh : p.c.k + h * p.c.k_sh) + chunk * 16;
  const int row0 = tid >> (p.row16_log2 + 1), step = THREADS >> (p.row16_log2 + 1);  // rows of a pass
  for (m0 *= kMoveRows; m0 < count; m0 += stride * kMoveRows) {
    const int rows = min(kMoveRows, count - m0);
    // the move of this thread: its scales, weight and number are on their way while the rows move
    int2 mv = make_int2(0, 0);
    float weight = 0.f, ks = 0.f, vs = 0.f;
    int number = 0;
    int64_t ks_to = -1, vs_to = 0;
    if (tid < rows) {
      const int* moves = p.moves + (int64_t)bh * 2 * p.max_moves + m0 + tid;
      mv = make_int2(moves[0], moves[p.max_moves]);
      weight = p.w[b * p.w_sb + h * p.w_sh + mv.x];
      number = p.pos[b * p.p_sb + h * p.p_sh + mv.x];
      const int from = paged_page(p.c, b, mv.x), to = paged_page(p.c, b, mv.y);
      const int sf = paged_slot(p.c, mv.x), st = paged_slot(p.c, mv.y);
      const bool ok = from >= 0 && to >= 0;
      s.from[0][tid] = ok ? from * p.c.k_sp + sf * p.c.k_ss : -1;
      s.from[1][tid] = ok ? from * p.c.v_sp + sf * p.c.v_ss : -1;
      s.to[0][tid] = to * p.c.k_sp + st * p.c.k_ss;
      s.to[1][tid] = to * p.c.v_sp + st * p.c.v_ss;
      if (ok && p.scaled) {
        ks = p.c.k_scale[h * p.c.ks_sh + from * p.c.ks_sp + sf];
        vs = p.c.v_scale[h * p.c.vs_sh + from * p.c.vs_sp + sf];
        ks_to = h * p.c.ks_sh + to * p.c.ks_sp + st;
        vs_to = h * p.c.vs_sh + to * p.c.vs_sp + st;
      }
    }
    __syncthreads();
    for (int r0 = row0; r0 < rows; r0 += V * step) {
      uint4 x[V];
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const int r = r0 + k * step;
        const int64_t from = r < rows ? s.from[value][r] : -1;
        if (from >= 0) x[k] = *reinterpret_cast<const uint4*>(pool + from);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const int r = r0 + k * step;
        if (r < rows && s.from[value][r] >= 0) *reinterpret_cast<uint4*>(pool + s.to[value][r]) = x[k];
      }
    }
    if (tid < rows) {
      const int64_t out = (int64_t)bh * p.cols + mv.y;
      p.w_out[out] = weight;
      p.pos_out[out] = number;
      if (ks_to >= 0) {
        p.c.k_scale[ks_to] = ks;
        p.c.v_scale[vs_to] = vs;
      }
    }
    __syncthreads();
  }
}

// A cluster of 1 to 8 CTAs per (sequence, head), each with an equal slice of the positions, whose rank keys it keeps
// in shared memory. The keep-th largest key comes from a radix select over the slices' histograms (read through
// distributed shared memory); then every warp numbers its holes and the rows that fill them. Bound by the chain of its
// steps: with four items of 100001 positions on 32 CTAs it takes 20 us, 6 of them to read and rank, 7 for the three
// digits, 6 to count and list the moves.
__global__ void __launch_bounds__(kSelThreads) select_kernel(const CompactParams p) {
  extern __shared__ uint32_t keys[];
  __shared__ __align__(16) int hists[3][kBins];  // one for each digit: no pass waits until all have read the last one's
  __shared__ int groups[3][kSelWarps];
  __shared__ int4 scan_sums[kSelWarps], cta_sum;
  __shared__ int s_digit, s_need, s_equal;
  __shared__ MoveScratch scratch;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int ctas;
  asm("mov.u32 %0, %%cluster_nctaid.x;" : "=r"(ctas));
  const int rank = (int)cluster_ctarank(), bh = blockIdx.x / ctas, b = bh / p.c.heads, h = bh % p.c.heads;
  pdl_launch_dependents();
  pdl_wait();
  const int n = min(paged_len(p.c, b), p.cols), left = min(n, p.keep);
  const float* w = p.w + b * p.w_sb + h * p.w_sh;
  const int* pos = p.pos + b * p.p_sb + h * p.p_sh;
  float* w_out = p.w_out + (int64_t)bh * p.cols;
  int* pos_out = p.pos_out + (int64_t)bh * p.cols;
  for (int i = left + rank * kSelThreads + tid; i < p.cols; i += ctas * kSelThreads) {
    w_out[i] = 0.f;
    pos_out[i] = -1;
  }
  if (n <= p.keep || p.keep == 0) {  // the same in every CTA of the cluster
    for (int i = rank * kSelThreads + tid; i < left; i += ctas * kSelThreads) {
      w_out[i] = w[i];
      pos_out[i] = pos[i];
    }
    if (!p.inline_moves && rank == 0 && tid == 0) p.counts[bh] = 0;
    return;
  }
  const int protect_from = p.seen[b] - p.recent;
  // this CTA's slice, and this warp's part of it, both in order
  const int slice = (n + ctas - 1) / ctas, lo = min(n, rank * slice), hi = min(n, lo + slice);
  const int per = ((hi - lo + kSelWarps - 1) / kSelWarps + 31) & ~31, first = lo + warp * per, last = min(hi, first + per);
  auto key_at = [&](int i) { return p.in_smem ? keys[i - lo] : rank_key(w[i], pos[i], protect_from); };
  uint32_t prefix = 0;
  int need = p.keep;
  int equal = 0;  // positions whose key, as far as its digits are known, is the need-th largest
  int low = 32;   // bits of the keys that are not known
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bits = pass == 2 ? 10 : 11;
    int* hist = hists[pass];
    if (pass == 0) {
      for (int i = tid; i < 3 * kBins; i += kSelThreads) hists[0][i] = 0;
      __syncthreads();
      constexpr int V = 8;  // positions that a thread has in flight
      for (int i = lo + tid; i < hi; i += V * kSelThreads) {
        float x[V];
        int y[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const int j = i + k * kSelThreads;
          x[k] = j < hi ? w[j] : 0.f;
          y[k] = j < hi ? pos[j] : 0;
        }
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const int j = i + k * kSelThreads;
          if (j >= hi) break;
          const uint32_t key = rank_key(x[k], y[k], protect_from);
          if (p.in_smem) keys[j - lo] = key;
          if (j < p.keep) {  // holes among them get another weight and number with their row
            w_out[j] = x[k];
            pos_out[j] = y[k];
          }
          atomicAdd(&hist[key >> 21], 1);
        }
      }
    } else {
      constexpr int V = 4;
      for (int i = lo + tid; i < hi; i += V * kSelThreads) {
        uint32_t key[V];
#pragma unroll
        for (int k = 0; k < V; ++k) key[k] = i + k * kSelThreads < hi ? key_at(i + k * kSelThreads) : ~prefix;
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (((key[k] ^ prefix) >> (shift + bits)) == 0) atomicAdd(&hist[(key[k] >> shift) & ((1 << bits) - 1)], 1);
      }
    }
    // The bin in which the need-th key lies, the highest first. Every warp adds up one of 32 groups of 64 bins, then
    // warp 0 finds the group in the sums of all CTAs, and the bin in the group's counts: 320 bytes from each CTA (8 KB
    // from each, all bins at once, took 2.5 us of a pass where this takes 1.5).
    __syncthreads();
    const int2 pair = reinterpret_cast<const int2*>(hist)[tid];
    const int group_sum = __reduce_add_sync(0xffffffffu, pair.x + pair.y);
    if (lane == 0) groups[pass][warp] = group_sum;
    if (ctas > 1) cluster_sync();
    else __syncthreads();
    if (warp == 0) {
      int x = 0, a = 0, b = 0;  // lane 0: the highest group, then the highest two bins
#pragma unroll 8
      for (int c = 0; c < ctas; ++c) x += ld_cluster(&groups[pass][31 - lane], c);
      int above = scan_lanes(x) - x;
      const int at = 31 - (__ffs(__ballot_sync(0xffffffffu, above + x >= need)) - 1);  // the first that reaches `need`
      above = __shfl_sync(0xffffffffu, above, 31 - at);
#pragma unroll 8
      for (int c = 0; c < ctas; ++c) {
        const int2 y = ld_cluster2(&hist[64 * at + 62 - 2 * lane], c);
        a += y.y;
        b += y.x;
      }
      above += scan_lanes(a + b) - a - b;
      const int bin = 64 * at + 63 - 2 * lane;
      if (above < need && need <= above + a + b) {
        const bool second = need > above + a;
        s_digit = bin - second;
        s_need = need - above - (second ? a : 0);
        s_equal = second ? b : a;
      }
    }
    __syncthreads();
    prefix |= (uint32_t)s_digit << shift;
    need = s_need;
    equal = s_equal;
    low = shift;
    if (equal == need) break;  // all of them are kept, whatever their further digits: usual after two passes
  }
  prefix >>= low;
  // Positions with a larger key than `prefix` (without the unknown bits) are kept, and `need` of those with an equal one,
  // the lowest first. Four counts of what comes before a warp tell it the rest: those above and those at the cut, below
  // `keep` and from there on.
  const bool cut = equal != need;
  auto count = [&](int from, int to, int& above, int& at) {
    constexpr int V = 4;  // keys in flight
    for (int i = from + lane; i < to; i += 32 * V) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const int j = i + k * 32;
        const uint32_t key = j < to ? key_at(j) >> low : 0;
        above += key > prefix;
        at += j < to && key == prefix;
      }
    }
  };
  int4 mine4 = make_int4(0, 0, 0, 0), total;
  count(first, min(last, p.keep), mine4.x, mine4.y);
  count(max(first, p.keep), last, mine4.z, mine4.w);
  const int4 before = cluster_scan(warp_sum(mine4), ctas, rank, scan_sums, &cta_sum, total);
  const int moved = p.keep - total.x - min(need, total.y);
  int tie = before.y + before.w;
  int holes = min(first, p.keep) - before.x - min(need, before.y);
  int loose = before.z + min(need, tie) - min(need, before.y);
  int* from = p.moves + (int64_t)bh * 2 * p.max_moves;
  int* to = from + p.max_moves;
  const unsigned lane_below = (1u << lane) - 1;
  auto low_bits = [](int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1; };
  constexpr int V = 4;  // groups of 32 positions in flight
  for (int i0 = first; i0 < last; i0 += 32 * V) {
    uint32_t key[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const int i = i0 + k * 32 + lane;
      key[k] = i < last ? key_at(i) >> low : 0u;
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
      // the group as bits: positions that exist, are kept, lie below `keep`
      const int g = i0 + k * 32, i = g + lane;
      const unsigned in = low_bits(last - g), under = low_bits(p.keep - g);
      unsigned kept = __ballot_sync(0xffffffffu, key[k] >= prefix) & in;
      if (cut) {
        const unsigned eq = __ballot_sync(0xffffffffu, key[k] == prefix) & in;
        const bool over = ((eq >> lane) & 1) && tie + __popc(eq & lane_below) >= need;
        kept &= ~__ballot_sync(0xffffffffu, over);
        tie += __popc(eq);
      }
      if (under) {
        const unsigned hole = in & under & ~kept;
        if ((hole >> lane) & 1) to[holes + __popc(hole & lane_below)] = i;
        holes += __popc(hole);
      }
      const unsigned beyond = kept & ~under;
      if ((beyond >> lane) & 1) from[loose + __popc(beyond & lane_below)] = i;
      loose += __popc(beyond);
    }
  }
  if (p.inline_moves) {  // one CTA, few moves: made here
    __syncthreads();
    move_rows<kSelThreads, 4>(p, bh, moved, 0, 1, scratch);
  } else if (rank == 0 && tid == 0) {
    p.counts[bh] = moved;
  }
}

// Makes the listed moves; grid (items, splits of an item's moves).
__global__ void __launch_bounds__(256) move_kernel(const CompactParams p) {
  __shared__ MoveScratch scratch;
  pdl_launch_dependents();
  pdl_wait();
  move_rows<256, 4>(p, blockIdx.x, p.counts[blockIdx.x], blockIdx.y, gridDim.y, scratch);
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
  const int64_t items = cache->batch * cache->heads;
  return items * compact_max_moves(cols, keep) * 2 * (int64_t)sizeof(int) + (items + 3) / 4 * 4 * (int64_t)sizeof(int);
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
  if (!tbf16_host::aligned16(ws)) return TBF16_ERR_ALIGN;
  const int64_t items = cache->batch * cache->heads;
  if (items == 0 || cols == 0) return TBF16_OK;
  p.w = weights; p.w_sb = w_sb; p.w_sh = w_sh;
  p.pos = pos; p.p_sb = pos_sb; p.p_sh = pos_sh;
  p.seen = seen;
  p.cols = (int)cols;
  p.keep = (int)keep;
  p.recent = (int)recent;
  p.scaled = cache->dtype == TBF16_E4M3;
  p.row16_log2 = 0;
  while ((16 << p.row16_log2) < cache->D * (p.scaled ? 1 : 2)) ++p.row16_log2;
  p.w_out = weights_out;
  p.pos_out = pos_out;
  p.counts = static_cast<int*>(ws);
  p.moves = p.counts + (items + 3) / 4 * 4;
  p.max_moves = (int)compact_max_moves(cols, keep);
  // CTAs for an item: more while its slices are long and there are SMs for them. Whole calls with 1 / 2 / 4 / 8 CTAs:
  // 8 items of 36156 positions 46 / 36 / 32 / 26 us, of 9000 17.8 / 17.3 / 16.8 / 18.6, of 4200 13.9 / 14.1 / 14.3 / 14.4.
  // More CTAs than SMs do not pay: 64 items of 16000 57 / 54 / 63 / 87, 128 of 2112 9 / 22 / 41 / 73.
  const tbf16_host::DeviceInfo* dev = tbf16_host::device_info();
  const int sms = dev->sms;
  int ctas = 1;
  while (ctas < 8 && (cols + ctas - 1) / ctas > 4096 && items * ctas * 2 <= sms) ctas *= 2;
  constexpr int kMaxKeys = 48 * 1024;
  while (ctas < 8 && (cols + ctas - 1) / ctas > kMaxKeys) ctas *= 2;
  const int64_t slice = (cols + ctas - 1) / ctas;
  p.in_smem = slice <= kMaxKeys;
  p.inline_moves = ctas == 1 && p.max_moves <= kMoveRows;
  if (items * ctas > INT32_MAX) return TBF16_ERR_LAUNCH;
  static bool attr_done[64] = {false};
  if (!attr_done[dev->device & 63]) {
    if (cudaFuncSetAttribute(select_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxKeys * 4) != cudaSuccess) {
      cudaGetLastError();
      return TBF16_ERR_LAUNCH;
    }
    attr_done[dev->device & 63] = true;
  }
  auto st = static_cast<cudaStream_t>(stream);
  if (int rc = tbf16_host::launch_pdl(select_kernel, dim3((unsigned)(items * ctas)), kSelThreads,
                                      p.in_smem ? (size_t)slice * 4 : 0, (unsigned)ctas, st, p))
    return rc;
  if (p.inline_moves) return TBF16_OK;
  const int64_t blocks = (p.max_moves + kMoveRows - 1) / kMoveRows;
  const int64_t splits = std::max<int64_t>(1, std::min<int64_t>(blocks, 16 * sms / items));
  return tbf16_host::launch_pdl(move_kernel, dim3((unsigned)items, (unsigned)splits), 256, 0, 1, st, p);
}

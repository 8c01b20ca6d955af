// Attention of the newest tokens over a paged key/value cache.
#include <cuda_fp8.h>

#include "paged.cuh"

namespace {
using namespace tbf16;

struct AttendParams {
  PagedView c;
  const __nv_bfloat16* q;
  int64_t q_sb, q_sh, q_st;
  __nv_bfloat16* out;
  int64_t o_sb, o_sh, o_st;
  const int* counts;
  float* weights;
  int64_t w_sb, w_sh;
  int T, group, window;
  float scale_log2;
};

template <bool E4M3>
__device__ __forceinline__ float cached(const uint8_t* row, int i) {
  if (E4M3) return __half2float(__half(__nv_cvt_fp8_to_halfraw(row[i], __NV_E4M3)));
  return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(row)[i]);
}

// One block per (sequence, key/value head); its query rows one after another, 128 keys at a time with the
// running maximum and sum of an online softmax.
template <int D, bool E4M3>
__global__ void __launch_bounds__(128) attend_kernel(const AttendParams p) {
  __shared__ float q[D], prob[128], red[4];
  const int b = blockIdx.x / p.c.heads, h = blockIdx.x % p.c.heads, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int len = paged_len(p.c, b), n = paged_count(p.c, p.counts, b, p.T, len);
  for (int r = 0; r < p.T * p.group; ++r) {
    const int t = r / p.group, head = h * p.group + r % p.group;
    __syncthreads();
    for (int i = tid; i < D; i += 128)
      q[i] = __bfloat162float(p.q[b * p.q_sb + head * p.q_sh + t * p.q_st + i]) * p.scale_log2;
    const int last = t < n ? len - n + t : -1, first = p.window ? max(0, last - p.window + 1) : 0;
    float m = -INFINITY, l = 0.f, acc[(D + 127) / 128] = {};
    for (int pass = 0; pass < (p.weights ? 2 : 1); ++pass) {
      for (int j0 = first; j0 <= last; j0 += 128) {
        const int j = j0 + tid;
        float s = -INFINITY;
        __syncthreads();
        const int page = j <= last ? paged_page(p.c, b, j) : -1;
        const int slot = paged_slot(p.c, j);
        if (page >= 0) {
          const uint8_t* row = p.c.k + page * p.c.k_sp + h * p.c.k_sh + slot * p.c.k_ss;
          s = 0.f;
          for (int i = 0; i < D; ++i) s += q[i] * cached<E4M3>(row, i);
          if (E4M3) s *= p.c.k_scale[page * p.c.ks_sp + h * p.c.ks_sh + slot];
        }
        if (pass == 1) {
          if (page >= 0) p.weights[b * p.w_sb + h * p.w_sh + j] += exp2f(s - m) / l;
          continue;
        }
        float mx = warp_max(s);
        if (lane == 0) red[warp] = mx;
        __syncthreads();
        mx = fmaxf(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])), m);
        const float base = mx == -INFINITY ? 0.f : mx, fac = exp2f(m - base), pr = page >= 0 ? exp2f(s - base) : 0.f;
        m = mx;
        prob[tid] = pr;
        __syncthreads();
        l *= fac;
        for (int i = 0; i < 128; ++i) l += prob[i];
        for (int e = 0; e * 128 + tid < D; ++e) acc[e] *= fac;
        for (int i = 0; i < 128 && j0 + i <= last; ++i) {
          const int pg = paged_page(p.c, b, j0 + i);
          if (pg < 0) continue;
          const int sl = paged_slot(p.c, j0 + i);
          const float sv = E4M3 ? p.c.v_scale[pg * p.c.vs_sp + h * p.c.vs_sh + sl] : 1.f;
          const uint8_t* row = p.c.v + pg * p.c.v_sp + h * p.c.v_sh + sl * p.c.v_ss;
          for (int e = 0; e * 128 + tid < D; ++e) acc[e] += prob[i] * (cached<E4M3>(row, e * 128 + tid) * sv);
        }
      }
    }
    for (int e = 0; e * 128 + tid < D; ++e)
      p.out[b * p.o_sb + head * p.o_sh + t * p.o_st + e * 128 + tid] = __float2bfloat16(l == 0.f ? 0.f : acc[e] / l);
  }
}

template <int D>
void launch_attend(const AttendParams& p, bool e4m3, cudaStream_t st) {
  const unsigned grid = (unsigned)(p.c.batch * p.c.heads);
  if (e4m3) attend_kernel<D, true><<<grid, 128, 0, st>>>(p);
  else attend_kernel<D, false><<<grid, 128, 0, st>>>(p);
}

}  // namespace

extern "C" int64_t tbf16_paged_attend_ws_size(const tbf16_paged_cache* cache, int64_t Hq, int64_t T, int with_weights) {
  return 0;
}

extern "C" int64_t tbf16_paged_attend_sync_size(const tbf16_paged_cache* cache, int64_t Hq, int64_t T) { return 0; }

extern "C" int tbf16_paged_attend(const tbf16_paged_cache* cache, const void* q, int64_t q_sb, int64_t q_sh,
                                  int64_t q_st, int64_t Hq, int64_t T, const int32_t* counts, float scale,
                                  int64_t window, void* out, int64_t out_sb, int64_t out_sh, int64_t out_st,
                                  float* weights, int64_t w_sb, int64_t w_sh, void* sync, void* ws, int64_t ws_bytes,
                                  void* stream) {
  if (int st = tbf16_host::require_sm100()) return st;
  AttendParams p;
  if (int st = tbf16_host::paged_view(cache, &p.c)) return st;
  if (T == 0 || cache->batch == 0) return TBF16_OK;
  if (!q || !out || T < 0 || Hq < 1 || Hq % cache->heads || window < 0 || !(scale == scale)) return TBF16_ERR_INVALID;
  if (T > 4096 || Hq > 65536 || T * (Hq / cache->heads) > 65536) return TBF16_ERR_INVALID;
  for (int64_t s : {q_sb, q_sh, q_st, out_sb, out_sh, out_st}) {
    if (s < 0) return TBF16_ERR_INVALID;
    if (s % 8) return TBF16_ERR_ALIGN;
  }
  if (!tbf16_host::aligned16(q) || !tbf16_host::aligned16(out)) return TBF16_ERR_ALIGN;
  p.q = static_cast<const __nv_bfloat16*>(q);
  p.q_sb = q_sb; p.q_sh = q_sh; p.q_st = q_st;
  p.out = static_cast<__nv_bfloat16*>(out);
  p.o_sb = out_sb; p.o_sh = out_sh; p.o_st = out_st;
  p.counts = counts;
  p.weights = weights;
  p.w_sb = w_sb; p.w_sh = w_sh;
  p.T = (int)T;
  p.group = (int)(Hq / cache->heads);
  p.window = (int)(window > p.c.cap ? 0 : window);
  p.scale_log2 = scale * 1.4426950408889634f;
  const bool e4m3 = cache->dtype == TBF16_E4M3;
  auto st = static_cast<cudaStream_t>(stream);
  if (cache->D == 64) launch_attend<64>(p, e4m3, st);
  else if (cache->D == 128) launch_attend<128>(p, e4m3, st);
  else launch_attend<256>(p, e4m3, st);
  return tbf16_host::check_launch();
}

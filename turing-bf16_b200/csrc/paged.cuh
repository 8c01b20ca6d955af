// The paged key/value cache as the kernels see it, and the lookups they share. Layout and limits:
// tbf16_paged_cache in include/tbf16_sm100.h.
#pragma once
#include "common.cuh"

namespace tbf16 {

struct PagedView {
  uint8_t* k;  // rows of D bf16 or e4m3 values; strides below in bytes
  uint8_t* v;
  float* k_scale;  // e4m3: inverse row scales; strides in floats
  float* v_scale;
  const int* table;
  const int* lens;
  const int* fresh;
  int64_t k_sp, k_sh, k_ss, v_sp, v_sh, v_ss, ks_sp, ks_sh, vs_sp, vs_sh, table_ld;
  int64_t pages;
  int batch, heads, page_shift, max_pages, cap;  // cap = max_pages << page_shift, below 2^31
  unsigned int* err;
};

// Cached tokens of sequence b, held inside [0, cap].
__device__ __forceinline__ int paged_len(const PagedView& c, int b) {
  const int n = c.lens[b];
  if (n < 0 || n > c.cap) atomicOr(c.err, kErrPage);
  return min(max(n, 0), c.cap);
}
// New tokens of sequence b, held inside [0, min(T, len)] (counts null: that many, or the cache's own count if less).
__device__ __forceinline__ int paged_count(const PagedView& c, const int* counts, int b, int T, int len) {
  const int n = counts ? counts[b] : c.fresh ? min(c.fresh[b], min(T, len)) : min(T, len);
  if (n < 0 || n > T || n > len) atomicOr(c.err, kErrPage);
  return min(max(n, 0), min(T, len));
}
// Page that holds position j of sequence b, or -1 (with the error bit set) for a number outside the pool.
__device__ __forceinline__ int paged_page(const PagedView& c, int b, int j) {
  const int id = c.table[b * c.table_ld + (j >> c.page_shift)];
  if (id >= 0 && id < c.pages) return id;
  atomicOr(c.err, kErrPage);
  return -1;
}
__device__ __forceinline__ int paged_slot(const PagedView& c, int j) { return j & ((1 << c.page_shift) - 1); }

}  // namespace tbf16

namespace tbf16_host {
// Checks a tbf16_paged_cache and fills the device view; TBF16_OK or the status to return.
int paged_view(const tbf16_paged_cache* cache, tbf16::PagedView* view);

// A launch that may be set up while the kernel before it in the stream ends (the kernels wait for it themselves), in
// clusters of `cluster` CTAs.
template <class... Params, class... Args>
int launch_pdl(void (*kernel)(Params...), dim3 grid, unsigned threads, size_t smem, unsigned cluster, cudaStream_t st,
               const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, kernel, args...) != cudaSuccess) {
    cudaGetLastError();
    return TBF16_ERR_LAUNCH;
  }
  return TBF16_OK;
}
}  // namespace tbf16_host

// interim
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>

#include "bf16x8.cuh"
#include "host_common.h"
#include "paged_attention.h"
#include "ptx_sm100.cuh"
#include "warp_reduce.cuh"

namespace l3ci {
namespace {

template <int D>
__global__ void __launch_bounds__(128) paged_attention_row_kernel(const PagedParams pp) {
  pdl_begin();
  const l3ci_paged_attention_args& p = pp.a;
  const float scale_log2e = pp.scale_log2e;
  const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const long long row = item / p.Hq;
  const int hq = (int)(item % p.Hq), h = hq / (p.Hq / p.Hkv);
  if (row >= p.rows) return;
  int b = 0, n = p.T;
  long long t = 0;
  if (p.starts) {
    int hit = -1;
    for (int i = lane; i < p.B; i += 32)
      if (p.starts[i] <= row && row < p.starts[i + 1]) hit = i;
    hit = __reduce_max_sync(kFullMask, hit);
    if (hit < 0) return;
    b = hit;
    t = row - p.starts[b];
    n = p.starts[b + 1] - p.starts[b];
  } else {
    b = (int)(row / p.T);
    t = row % p.T;
  }
  if ((long long)n * pp.R < pp.min_rows || n < 0) return;
  const long long cap = (long long)p.max_pages * p.page_size;
  const long long len = min(max((long long)p.seq_lens[b], 0LL), cap);
  const long long seen = len - n + t + 1;
  constexpr int E = D / 32;
  const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(p.q) + (p.starts ? row * p.q_st : b * p.q_sb + t * p.q_st) + hq * p.q_sh + lane * E;
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out) + (p.starts ? row * p.o_st : b * p.o_sb + t * p.o_st) + hq * p.o_sh + lane * E;
  float x[E], o[E] = {};
  for (int i = 0; i < E; ++i) x[i] = __bfloat162float(q[i]);
  float m = -INFINITY, l = 0.f;
  for (long long j = 0; j < seen; ++j) {
    const int page = p.page_table[b * p.table_st + j / p.page_size];
    const bool there = page >= 0 && page < p.pages;
    const long long at = page * p.cache_sp + j % p.page_size * p.cache_st + h * D + lane * E;
    float s = 0.f;
    for (int i = 0; i < E; ++i) s += x[i] * (there ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.cache_k)[at + i]) : 0.f);
    s = group_sum<32>(s) * scale_log2e;
    const float mn = fmaxf(m, s), mu = mn == -INFINITY ? 0.f : mn, a = exp2f(m - mu), e = exp2f(s - mu);
    l = l * a + e;
    for (int i = 0; i < E; ++i) o[i] = o[i] * a + e * (there ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.cache_v)[at + i]) : 0.f);
    m = mn;
  }
  for (int i = 0; i < E; ++i) out[i] = __float2bfloat16_rn(seen > 0 ? o[i] / l : 0.f);
}


}  // namespace

size_t paged_chunks_scratch_bytes(const PagedParams& p) { return 0; }
int paged_chunks_launch(const PagedParams& p, void* scratch, cudaStream_t stream) {
  const dim3 grid((unsigned)((p.a.rows * p.a.Hq + 3) / 4));
  if (p.a.D == 64) L3CI_LAUNCH("paged_attention_row_kernel", paged_attention_row_kernel<64>, grid, dim3(128), 0, stream, p);
  else L3CI_LAUNCH("paged_attention_row_kernel", paged_attention_row_kernel<128>, grid, dim3(128), 0, stream, p);
  return L3CI_OK;
}

}  // namespace l3ci

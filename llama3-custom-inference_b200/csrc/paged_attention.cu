// Attention of new tokens over a paged cache (include/l3ci_b200.h, l3ci_paged_attention).  A warp per query row: lanes hold the row, keys one
// after the other, running maximum and sum of the softmax.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>

#include "bf16x8.cuh"
#include "host_common.h"
#include "ptx_sm100.cuh"
#include "warp_reduce.cuh"

namespace l3ci {
namespace {

template <int D>
__global__ void __launch_bounds__(128) paged_attention_row_kernel(const l3ci_paged_attention_args p, float scale_log2e) {
  pdl_begin();
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

// The arguments of a call, checked; kNothing: there is nothing to do.
constexpr int kNothing = -1;
int check(const l3ci_paged_attention_args* a) {
  if (!a) return fail(L3CI_ERR_INVALID, "paged_attention: null arguments");
  if (a->B < 0 || a->Hq <= 0 || a->Hkv <= 0 || a->page_size <= 0 || a->max_pages < 0 || a->pages < 0 || (a->starts ? a->rows < 0 : a->T < 0))
    return fail(L3CI_ERR_INVALID, "paged_attention: B=%d T=%d rows=%lld heads %d, %d, pages of %d", a->B, a->T, (long long)a->rows, a->Hq, a->Hkv, a->page_size);
  if (a->D != 64 && a->D != 128) return fail(L3CI_ERR_UNSUPPORTED, "Unsupported head size for paged_attention kernel: %d", a->D);
  if (a->Hq % a->Hkv || a->Hq / a->Hkv > 16) return fail(L3CI_ERR_UNSUPPORTED, "Unsupported QKV head ratio for paged_attention kernel: %d/%d", a->Hq, a->Hkv);
  if (a->page_size % 16) return fail(L3CI_ERR_UNSUPPORTED, "paged_attention: pages of %d tokens, not a multiple of 16", a->page_size);
  const long long rows = a->starts ? a->rows : (long long)a->B * a->T;
  if (rows == 0 || a->B == 0) return kNothing;
  if (!a->q || !a->cache_k || !a->cache_v || !a->out || !a->page_table || !a->seq_lens) return fail(L3CI_ERR_INVALID, "paged_attention: null pointer");
  if (!aligned16(a->q) || !aligned16(a->out) || !aligned16(a->cache_k) || !aligned16(a->cache_v) || a->q_sb % 8 || a->q_st % 8 || a->q_sh % 8 || a->o_sb % 8 ||
      a->o_st % 8 || a->o_sh % 8 || a->cache_sp % 8 || a->cache_st % 8)
    return fail(L3CI_ERR_ALIGNMENT, "paged_attention: rows must start on 16 bytes");
  if (rows > 0x7fffffffLL || (long long)a->max_pages * a->page_size > 0x7fffffffLL || a->pages > 0x7fffffffLL)
    return fail(L3CI_ERR_INVALID, "paged_attention: %lld rows, %lld keys a sequence", rows, (long long)a->max_pages * a->page_size);
  return L3CI_OK;
}

}  // namespace
}  // namespace l3ci

extern "C" size_t l3ci_paged_attention_scratch_bytes(const l3ci_paged_attention_args* a) {
  (void)a;
  return 0;
}

extern "C" int l3ci_paged_attention(const l3ci_paged_attention_args* args) {
  using namespace l3ci;
  clear_error();
  if (int st = check(args)) return st == kNothing ? L3CI_OK : st;
  l3ci_paged_attention_args a = *args;
  if (!a.starts) a.rows = (long long)a.B * a.T;
  const float scale_log2e = (a.scale > 0.f ? a.scale : 1.0f / sqrtf((float)a.D)) * 1.4426950408889634f;
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(a.stream);
  const dim3 grid((unsigned)((a.rows * a.Hq + 3) / 4));
  if (a.D == 64) L3CI_LAUNCH("paged_attention_row_kernel", paged_attention_row_kernel<64>, grid, dim3(128), 0, stream, a, scale_log2e);
  else L3CI_LAUNCH("paged_attention_row_kernel", paged_attention_row_kernel<128>, grid, dim3(128), 0, stream, a, scale_log2e);
  return L3CI_OK;
}

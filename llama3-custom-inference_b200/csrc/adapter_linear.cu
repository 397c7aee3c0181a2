// Low-rank adapters beside a shared projection (include/l3ci_b200.h, l3ci_adapter_linear).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "bf16x8.cuh"
#include "host_common.h"
#include "linear_rows.h"
#include "ptx_sm100.cuh"
#include "warp_reduce.cuh"

namespace l3ci {
namespace {

// z[r, j] = scales[i] x[r] . a[i, j], i = index[r]; 0 without an adapter.  A warp per (r, j).
__global__ void __launch_bounds__(128) adapter_shrink_kernel(const l3ci_adapter_linear_args p, float* z) {
  pdl_wait();                // (before the next kernel may start: it reads x and w at once)
  pdl_launch_dependents();
  const long long item = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  const long long r = item / p.rank;
  if (r >= p.rows) return;
  const int j = (int)(item % p.rank), i = p.index[r];
  float s = 0.f;
  if (i >= 0 && i < p.adapters) {
    const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(p.x) + r * p.x_st;
    const __nv_bfloat16* a = static_cast<const __nv_bfloat16*>(p.a) + ((long long)i * p.rank + j) * p.K;
    for (int k = lane * 8; k < p.K; k += 256) {
      float u[8], v[8];
      unpack8(*reinterpret_cast<const uint4*>(x + k), u);
      unpack8(*reinterpret_cast<const uint4*>(a + k), v);
#pragma unroll
      for (int e = 0; e < 8; ++e) s = fmaf(u[e], v[e], s);
    }
    s = group_sum<32>(s) * (p.scales ? p.scales[i] : 1.f);
  }
  if (lane == 0) z[item] = s;
}

// A tile of 64 x 64 outputs: the shared product and the adapters' part.
__global__ void __launch_bounds__(256) adapter_expand_kernel(const l3ci_adapter_linear_args p, const float* z) {
  __shared__ float xs[64][17], ws[64][17];
  pdl_begin();
  const long long r0 = (long long)blockIdx.y * 64;
  const int n0 = blockIdx.x * 64, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < p.K; k0 += 16) {
    for (int e = threadIdx.x; e < 64 * 16; e += 256) {
      const int y = e >> 4, k = k0 + (e & 15);
      xs[y][e & 15] = r0 + y < p.rows && k < p.K ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.x)[(r0 + y) * p.x_st + k]) : 0.f;
      ws[y][e & 15] = n0 + y < p.N && k < p.K ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.w)[(long long)(n0 + y) * p.K + k]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 16; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xs[ty * 4 + i][k], ws[tx * 4 + j][k], acc[i][j]);
    __syncthreads();
  }
  for (int i = 0; i < 4; ++i) {
    const long long r = r0 + ty * 4 + i;
    if (r >= p.rows) break;
    const int ad = p.index[r];
    for (int j = 0; j < 4; ++j) {
      const int n = n0 + tx * 4 + j;
      if (n >= p.N) break;
      float y = acc[i][j];
      if (ad >= 0 && ad < p.adapters)
        for (int k = 0; k < p.rank; ++k) y = fmaf(z[r * p.rank + k], __bfloat162float(static_cast<const __nv_bfloat16*>(p.b)[((long long)ad * p.N + n) * p.rank + k]), y);
      static_cast<__nv_bfloat16*>(p.out)[r * p.out_st + n] = __float2bfloat16_rn(y);
    }
  }
}

// The arguments of a call, checked; kNothing: there is nothing to do.
constexpr int kNothing = -1;
int check(const l3ci_adapter_linear_args* a) {
  if (!a) return fail(L3CI_ERR_INVALID, "adapter_linear: null arguments");
  if (a->rows < 0 || a->rows > INT32_MAX || a->K <= 0 || a->N < 0 || a->rank <= 0 || a->adapters < 0)
    return fail(L3CI_ERR_INVALID, "adapter_linear: rows=%lld K=%d N=%d, %d adapters of rank %d", (long long)a->rows, a->K, a->N, a->adapters, a->rank);
  if (a->rank % 8 || a->rank > L3CI_ADAPTER_MAX_RANK)
    return fail(L3CI_ERR_UNSUPPORTED, "adapter_linear: rank %d is not a multiple of 8 up to %d", a->rank, L3CI_ADAPTER_MAX_RANK);
  if (a->rows == 0 || a->N == 0) return kNothing;
  if (!a->x || !a->w || !a->out || !a->index || (a->adapters && (!a->a || !a->b))) return fail(L3CI_ERR_INVALID, "adapter_linear: null pointer");
  if (a->K % 8 || a->N % 8 || a->x_st % 8 || a->out_st % 8 || !aligned16(a->x) || !aligned16(a->w) || !aligned16(a->a) || !aligned16(a->b) || !aligned16(a->out))
    return fail(L3CI_ERR_ALIGNMENT, "adapter_linear: rows must be whole 16-byte vectors");
  if (a->rows > 1 && (a->x_st <= 0 || a->out_st < a->N)) return fail(L3CI_ERR_INVALID, "adapter_linear: rows without a stride of their own");
  return L3CI_OK;
}

}  // namespace
}  // namespace l3ci

extern "C" size_t l3ci_adapter_linear_scratch_bytes(const l3ci_adapter_linear_args* a) {
  const int st = l3ci::check(a);
  l3ci::clear_error();
  return st ? 0 : (size_t)a->rows * a->rank * 4;
}

extern "C" int l3ci_adapter_linear(const l3ci_adapter_linear_args* a) {
  using namespace l3ci;
  clear_error();
  if (int st = check(a)) return st == kNothing ? L3CI_OK : st;
  const size_t need = (size_t)a->rows * a->rank * 4;
  if (!a->scratch || a->scratch_bytes < need || !aligned16(a->scratch)) return fail(L3CI_ERR_SCRATCH, "adapter_linear: %zu bytes of scratch, %zu are needed", a->scratch_bytes, need);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(a->stream);
  float* z = static_cast<float*>(a->scratch);
  L3CI_LAUNCH("adapter_shrink_kernel", adapter_shrink_kernel, dim3((unsigned)((a->rows * a->rank + 3) / 4)), dim3(128), 0, stream, *a, z);
  if (a->rows <= L3CI_LINEAR_MAX_ROWS) {
    l3ci_linear_args l = {};
    l.x = a->x; l.w = a->w; l.out = a->out; l.status = a->status;
    l.rows = a->rows; l.x_st = a->rows > 1 ? a->x_st : a->K; l.out_st = a->out_st;
    l.K = a->K; l.N = a->N; l.groups = 1;
    l.stream = a->stream;
    return adapter_rows_launch(&l, AdapterRows{z, a->index, static_cast<const __nv_bfloat16*>(a->b), a->rank, a->adapters});
  }
  L3CI_LAUNCH("adapter_expand_kernel", adapter_expand_kernel, dim3((unsigned)((a->N + 63) / 64), (unsigned)((a->rows + 63) / 64)), dim3(256), 0, stream, *a, (const float*)z);
  return L3CI_OK;
}

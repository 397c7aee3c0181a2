// Low-rank adapters beside a shared projection (include/l3ci_b200.h, l3ci_adapter_linear).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "bf16x8.cuh"
#include "host_common.h"
#include "linear_many.h"
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

// The same of many rows, on the tensor cores: 32 rows of x a CTA, warps share the columns of K and add up at the end.  A dot product does not
// ask in which order its terms come: a lane takes 8 neighbouring columns, 16 bytes, of a row of x and of a row of a, which are the operands of two
// products.  Of every adapter among the 32 rows all rows' products are computed and its own rows' kept.
// CTAs behind these list the adapters among every 256 rows (linear_many.h).
constexpr int kShrinkRows = 32, kShrinkWarps = 8, kShrinkRanks = 32;   // ranks at a time: four products wide

__global__ void __launch_bounds__(32 * kShrinkWarps) adapter_shrink_many_kernel(const l3ci_adapter_linear_args p, float* z, int* lists, int blocks) {
  __shared__ float parts[kShrinkWarps][kShrinkRows][kShrinkRanks + 1];
  __shared__ int ids[kAdapterTile];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  auto id_of = [&](long long row) {
    const int id = row < p.rows ? __ldg(p.index + row) : -1;
    return id >= 0 && id < p.adapters ? id : -1;
  };
  if ((int)blockIdx.x >= blocks) {       // ---- a list ----
    const int t = threadIdx.x, tile = blockIdx.x - blocks;
    ids[t] = id_of((long long)tile * kAdapterTile + t);
    __syncthreads();
    bool first = ids[t] >= 0;            // the first row of its adapter
    for (int i = 0; i < t && first; ++i) first = ids[i] != ids[t];
    int* counts = reinterpret_cast<int*>(parts);
    const unsigned mask = __ballot_sync(kFullMask, first);
    if (lane == 0) counts[warp] = __popc(mask);
    __syncthreads();
    int at = __popc(mask & ((1u << lane) - 1)), all = 0;
    for (int w = 0; w < kShrinkWarps; ++w) {
      if (w < warp) at += counts[w];
      all += counts[w];
    }
    int* list = lists + (long long)tile * kAdapterList;
    if (first) list[1 + at] = ids[t];
    if (t == 0) list[0] = all;
    return;
  }
  const long long row0 = (long long)blockIdx.x * kShrinkRows;
  if (threadIdx.x < kShrinkRows) ids[threadIdx.x] = id_of(row0 + threadIdx.x);
  __syncthreads();
  const int mine = ids[lane];
  unsigned left = __ballot_sync(kFullMask, mine >= 0);     // rows whose adapters are still to come
  const __nv_bfloat16* x[4];                               // rows gid, gid + 8, + 16, + 24 (the last row for those behind it)
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const long long row = row0 + gid + 8 * i;
    x[i] = static_cast<const __nv_bfloat16*>(p.x) + (row < p.rows ? row : p.rows - 1) * p.x_st + tig * 8;
  }
  while (left) {
    const int id = __shfl_sync(kFullMask, mine, __ffs(left) - 1);
    const unsigned here = __ballot_sync(kFullMask, mine == id);
    left &= ~here;
    const float scale = p.scales ? __ldg(p.scales + id) : 1.f;
    for (int j0 = 0; j0 < p.rank; j0 += kShrinkRanks) {
      const int tiles = min(p.rank - j0, kShrinkRanks) / 8;
      const __nv_bfloat16* a = static_cast<const __nv_bfloat16*>(p.a) + ((long long)id * p.rank + j0 + gid) * p.K + tig * 8;
      float acc[2][4][4] = {};
#pragma unroll 2
      for (int k = warp * 32; k < p.K; k += kShrinkWarps * 32) {
        const bool in = k + tig * 8 < p.K;                 // (K is a multiple of 8)
        uint4 xv[4], av[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) xv[i] = in ? __ldg(reinterpret_cast<const uint4*>(x[i] + k)) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int n = 0; n < 4; ++n) av[n] = in && n < tiles ? __ldg(reinterpret_cast<const uint4*>(a + (long long)n * 8 * p.K + k)) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            mma_bf16(acc[m][n], xv[2 * m].x, xv[2 * m + 1].x, xv[2 * m].y, xv[2 * m + 1].y, av[n].x, av[n].y);
            mma_bf16(acc[m][n], xv[2 * m].z, xv[2 * m + 1].z, xv[2 * m].w, xv[2 * m + 1].w, av[n].z, av[n].w);
          }
      }
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) parts[warp][m * 16 + gid + (e >> 1) * 8][n * 8 + 2 * tig + (e & 1)] = acc[m][n][e];
      __syncthreads();
      for (int i = threadIdx.x; i < kShrinkRows * tiles * 8; i += 32 * kShrinkWarps) {
        const int r = i / (tiles * 8), j = i % (tiles * 8);
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < kShrinkWarps; ++w) s += parts[w][r][j];
        if ((here >> r) & 1) z[(row0 + r) * p.rank + j0 + j] = s * scale;
      }
      __syncthreads();
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

namespace l3ci {
namespace {

// Scratch: z, then the lists of many rows.
size_t z_bytes(const l3ci_adapter_linear_args* a) { return ((size_t)a->rows * a->rank * 4 + 15) / 16 * 16; }
size_t scratch_of(const l3ci_adapter_linear_args* a) {
  const size_t tiles = ((size_t)a->rows + kAdapterTile - 1) / kAdapterTile;
  return z_bytes(a) + (a->rows > L3CI_LINEAR_MAX_ROWS ? tiles * kAdapterList * 4 : 0);
}

}  // namespace
}  // namespace l3ci

extern "C" size_t l3ci_adapter_linear_scratch_bytes(const l3ci_adapter_linear_args* a) {
  const int st = l3ci::check(a);
  l3ci::clear_error();
  return st ? 0 : l3ci::scratch_of(a);
}

extern "C" int l3ci_adapter_linear(const l3ci_adapter_linear_args* a) {
  using namespace l3ci;
  clear_error();
  if (int st = check(a)) return st == kNothing ? L3CI_OK : st;
  const size_t need = scratch_of(a);
  if (!a->scratch || a->scratch_bytes < need || !aligned16(a->scratch)) return fail(L3CI_ERR_SCRATCH, "adapter_linear: %zu bytes of scratch, %zu are needed", a->scratch_bytes, need);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(a->stream);
  float* z = static_cast<float*>(a->scratch);
  l3ci_linear_args l = {};
  l.x = a->x; l.w = a->w; l.out = a->out; l.status = a->status;
  l.rows = a->rows; l.x_st = a->rows > 1 ? a->x_st : a->K; l.out_st = a->out_st;
  l.K = a->K; l.N = a->N; l.groups = 1;
  l.stream = a->stream;
  const __nv_bfloat16* b = static_cast<const __nv_bfloat16*>(a->b);
  if (a->rows <= L3CI_LINEAR_MAX_ROWS) {
    L3CI_LAUNCH("adapter_shrink_kernel", adapter_shrink_kernel, dim3((unsigned)((a->rows * a->rank + 3) / 4)), dim3(128), 0, stream, *a, z);
    return adapter_rows_launch(&l, AdapterRows{z, a->index, b, a->rank, a->adapters});
  }
  int* lists = reinterpret_cast<int*>(static_cast<uint8_t*>(a->scratch) + z_bytes(a));
  const long long blocks = (a->rows + kShrinkRows - 1) / kShrinkRows, tiles = (a->rows + kAdapterTile - 1) / kAdapterTile;
  L3CI_LAUNCH("adapter_shrink_many_kernel", adapter_shrink_many_kernel, dim3((unsigned)(blocks + tiles)), dim3(32 * kShrinkWarps), 0, stream, *a, z, lists, (int)blocks);
  return adapter_many_launch(&l, AdapterMany{z, a->index, b, lists, a->rank, a->adapters});
}

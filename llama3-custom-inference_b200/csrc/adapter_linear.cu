// Low-rank adapters beside a shared projection (include/l3ci_b200.h, l3ci_adapter_linear): y = x w^T + z b^T, z = s x a^T by the adapters of the rows.
// Two launches: z (fp32, in scratch), then the shared product with z b^T in its fp32 sums, one rounding at the end.
// Few rows (linear_rows.cu) are bound by the bytes of w, which the second launch reads, with x, while the first computes z: z b^T is multiply-adds
// of the output warps, a row of b a thread, under the stream of w.  Many rows (linear_many.cu) are bound by the tensor cores, and read nothing before z
// is complete: z b^T is two more products of a tile, z as the sum of two
// bf16 (kept to 2^-16), for each adapter of the tile's rows in turn with the others' rows masked out of the instruction, not multiplied by zero.
// (A value of b that is infinite meets both halves of z there, and may give NaN where z b is infinite.)
// Measured on a B200, calls one behind the other with changing weights: 8 rows of as many adapters of rank 16, 2048 -> 8192 10.1 us (34 MB of w: 3.3 TB/s; the
// kernel alone 9.0); 64 rows of 8 adapters of rank 32, 8192 -> 2048 16.6, of 64 adapters 33 (a
// library's product alone 10.4 and 14.6); 6001 rows of 6 adapters of rank 16, 2048 -> 8192 154 us in rows of 40 calls, 178 in long runs, at the power limit,
// of which z takes 15 and the product 133 to 142 (1510 to 1420 TFLOP/s).
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

__device__ __forceinline__ int adapter_of(const l3ci_adapter_linear_args& p, long long row) {
  const int id = row < p.rows ? __ldg(p.index + row) : -1;
  return id >= 0 && id < p.adapters ? id : -1;
}

// The list of the adapters among 256 rows (linear_many.h), by all threads of a CTA of THREADS.
template <int THREADS>
__device__ void adapter_list(const l3ci_adapter_linear_args& p, int* list, int tile) {
  __shared__ int ids[kAdapterTile], counts[kAdapterTile / 32];
  constexpr int kRounds = kAdapterTile / THREADS;
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 0; k < kRounds; ++k) ids[k * THREADS + threadIdx.x] = adapter_of(p, (long long)tile * kAdapterTile + k * THREADS + threadIdx.x);
  __syncthreads();
  bool first[kRounds];                   // the first row of its adapter
  unsigned mask[kRounds];
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int t = k * THREADS + threadIdx.x;
    first[k] = ids[t] >= 0;
    for (int i = 0; i < t && first[k]; ++i) first[k] = ids[i] != ids[t];
    mask[k] = __ballot_sync(kFullMask, first[k]);
    if (lane == 0) counts[t / 32] = __popc(mask[k]);
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kRounds; ++k) {
    const int t = k * THREADS + threadIdx.x;
    int at = __popc(mask[k] & ((1u << lane) - 1)), all = 0;
    for (int w = 0; w < kAdapterTile / 32; ++w) {
      if (w < t / 32) at += counts[w];
      all += counts[w];
    }
    if (t == 0) list[0] = all;
    if (!first[k]) continue;
    int* entry = list + kAdapterHead + at * kAdapterEntry;
    entry[0] = ids[t];
    for (int w = 0; w < kAdapterTile / 32; ++w) {
      unsigned others = 0;
      for (int i = 0; i < 32; ++i) others |= (unsigned)(ids[w * 32 + i] != ids[t]) << i;
      entry[4 + w] = (int)others;
    }
  }
}

// z[r, j] = scales[i] x[r] . a[i, j], i = index[r]; 0 without an adapter.  A CTA per row and kDots ranks, whose warps share the columns of K: a row of
// x is read once for kDots rows of a, and a warp has all of its loads under way at once (a warp per r and j took 6.2 us for 64 rows of 8192
// columns and rank 32, and slowed the product's weights, which stream meanwhile, by as much).
constexpr int kDots = 4, kDotWarps = 4;
constexpr int kDotRows = 512;   // up to which a row of a is read for every token (from L2) rather than for 32 at a time by few CTAs

__global__ void __launch_bounds__(32 * kDotWarps) adapter_shrink_kernel(const l3ci_adapter_linear_args p, float* z, int* lists) {
  __shared__ float parts[kDotWarps][kDots];
  pdl_wait();                // (before the next kernel may start: it reads x and w at once)
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = blockIdx.x, j0 = blockIdx.y * kDots;
  if (r >= p.rows) {         // (CTAs behind the rows, where the product is that of many rows)
    if (j0 == 0) adapter_list<32 * kDotWarps>(p, lists + (r - p.rows) * kAdapterList, r - (int)p.rows);
    return;
  }
  const int i = adapter_of(p, r);
  const bool has = i >= 0;
  float s[kDots] = {};
  if (has) {
    const __nv_bfloat16* x = static_cast<const __nv_bfloat16*>(p.x) + r * p.x_st;
    const __nv_bfloat16* a = static_cast<const __nv_bfloat16*>(p.a) + ((long long)i * p.rank + j0) * p.K;
#pragma unroll 4
    for (int k = (warp * 32 + lane) * 8; k < p.K; k += kDotWarps * 256) {
      const uint4 xv = __ldg(reinterpret_cast<const uint4*>(x + k));
      uint4 av[kDots];
#pragma unroll
      for (int j = 0; j < kDots; ++j) av[j] = __ldg(reinterpret_cast<const uint4*>(a + (long long)j * p.K + k));
      float u[8], v[8];
      unpack8(xv, u);
#pragma unroll
      for (int j = 0; j < kDots; ++j) {
        unpack8(av[j], v);
#pragma unroll
        for (int e = 0; e < 8; ++e) s[j] = fmaf(u[e], v[e], s[j]);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < kDots; ++j) {
    s[j] = group_sum<32>(s[j]);
    if (lane == 0) parts[warp][j] = s[j];
  }
  __syncthreads();
  if (threadIdx.x < kDots) {
    float y = 0.f;
    for (int w = 0; w < kDotWarps; ++w) y += parts[w][threadIdx.x];
    z[(long long)r * p.rank + j0 + threadIdx.x] = has ? y * (p.scales ? __ldg(p.scales + i) : 1.f) : 0.f;
  }
}

// The same of many rows, on the tensor cores: 32 rows of x a CTA, warps share the columns of K and add up at the end.  A dot product does not
// ask in which order its terms come: a lane takes 8 neighbouring columns, 16 bytes, of a row of x and of a row of a, which are the operands of two
// products.  Of every adapter among the 32 rows all rows' products are computed and its own rows' kept.
// blockIdx.y: the ranks.  CTAs behind these make the lists.
constexpr int kShrinkRows = 32, kShrinkWarps = 8;

// NT: products of 8 ranks side by side.  (Two CTAs an SM: 6001 rows are then one wave.  16 warps at 128 registers, one CTA an SM, took 17.5 us for
// them at K = 2048, rank 16.)
template <int NT>
__global__ void __launch_bounds__(32 * kShrinkWarps, 2) adapter_shrink_many_kernel(const l3ci_adapter_linear_args p, float* z, int* lists, int blocks) {
  constexpr int kShrinkRanks = 8 * NT;   // ranks at a time
  __shared__ float parts[kShrinkWarps][kShrinkRows][kShrinkRanks + 1];
  __shared__ int ids[kShrinkRows];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  if ((int)blockIdx.x >= blocks) {
    if (blockIdx.y == 0) adapter_list<32 * kShrinkWarps>(p, lists + (long long)(blockIdx.x - blocks) * kAdapterList, blockIdx.x - blocks);
    return;
  }
  const long long row0 = (long long)blockIdx.x * kShrinkRows;
  if (threadIdx.x < kShrinkRows) ids[threadIdx.x] = adapter_of(p, row0 + threadIdx.x);
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
    {
      const int j0 = blockIdx.y * kShrinkRanks;
      const int tiles = min(p.rank - j0, kShrinkRanks) / 8;
      const __nv_bfloat16* a = static_cast<const __nv_bfloat16*>(p.a) + ((long long)id * p.rank + j0 + gid) * p.K + tig * 8;
      float acc[2][NT][4] = {};
      constexpr int kAhead = NT > 2 ? 2 : 4;
#pragma unroll kAhead
      for (int k = warp * 32; k < p.K; k += kShrinkWarps * 32) {
        const bool in = k + tig * 8 < p.K;                 // (K is a multiple of 8)
        uint4 xv[4], av[NT];
#pragma unroll
        for (int i = 0; i < 4; ++i) xv[i] = in ? __ldg(reinterpret_cast<const uint4*>(x[i] + k)) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int n = 0; n < NT; ++n) av[n] = in && n < tiles ? __ldg(reinterpret_cast<const uint4*>(a + (long long)n * 8 * p.K + k)) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            mma_bf16(acc[m][n], xv[2 * m].x, xv[2 * m + 1].x, xv[2 * m].y, xv[2 * m + 1].y, av[n].x, av[n].y);
            mma_bf16(acc[m][n], xv[2 * m].z, xv[2 * m + 1].z, xv[2 * m].w, xv[2 * m + 1].w, av[n].z, av[n].w);
          }
      }
#pragma unroll
      for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n)
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

// Whether the call goes to the product of few rows (64 at a time, weights on the wide side of the tensor cores, low-rank parts in multiply-adds) or to
// that of many (tiles of 256 x 256 over pairs of SMs).  Estimates in us, fits to both sides on a B200, e.g. rank 16, 2 adapters, few and many: rows 128,
// 2048 -> 8192 19 and 27, 512 62 and 27; 8192 -> 2048 rows 512 35 and 72; 4096 -> 4096 rows 256 21 and 42, 512 39 and 42; rank 64, 8
// adapters: 2048 -> 8192 rows 128 41 and 55, 256 105 and 42.  They know nothing of how many adapters a tile of rows has, which costs the product of
// many rows a stage each: 256 rows, 2048 -> 8192, rank 16 of 1, 8, 64, 256 adapters 21, 36, 57, 163 us.
bool few_rows(const l3ci_adapter_linear_args* a) {
  const int sms = sm_count() > 0 ? sm_count() : 148;
  const long long groups = (a->rows + L3CI_LINEAR_MAX_ROWS - 1) / L3CI_LINEAR_MAX_ROWS;
  const long long tiles = (a->rows + kAdapterTile - 1) / kAdapterTile * ((a->N + 255) / 256), pairs = sms / 2 > 0 ? sms / 2 : 1;
  const double few = 9.0 + 7.7e-8 * groups * a->N * a->K + 7e-7 * a->rows * a->N * a->rank;
  const double many = 11.0 + 0.0076 * a->K * ((tiles + pairs - 1) / pairs);
  return few <= many;
}

// Scratch: z, then the lists of many rows.
size_t z_bytes(const l3ci_adapter_linear_args* a) { return ((size_t)a->rows * a->rank * 4 + 15) / 16 * 16; }
size_t scratch_of(const l3ci_adapter_linear_args* a) {
  const size_t tiles = ((size_t)a->rows + kAdapterTile - 1) / kAdapterTile;
  return z_bytes(a) + (few_rows(a) ? 0 : tiles * kAdapterList * 4);
}

}  // namespace
}  // namespace l3ci

extern "C" size_t l3ci_adapter_linear_scratch_bytes(const l3ci_adapter_linear_args* a) {
  const int st = l3ci::check(a);
  l3ci::clear_error();
  return st ? 0 : l3ci::scratch_of(a);
}

extern "C" int l3ci_adapter_linear_kernel_choice(const l3ci_adapter_linear_args* a) {
  const int st = l3ci::check(a);
  l3ci::clear_error();
  return st ? -1 : l3ci::few_rows(a) ? 0 : 1;
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
  const bool few = few_rows(a);
  const long long blocks = (a->rows + kShrinkRows - 1) / kShrinkRows, tiles = few ? 0 : (a->rows + kAdapterTile - 1) / kAdapterTile;
  int* lists = reinterpret_cast<int*>(static_cast<uint8_t*>(a->scratch) + z_bytes(a));
  if (a->rows <= kDotRows) {
    L3CI_LAUNCH("adapter_shrink_kernel", adapter_shrink_kernel, dim3((unsigned)(a->rows + tiles), (unsigned)(a->rank / kDots)), dim3(32 * kDotWarps), 0, stream, *a, z, lists);
  } else {
    auto shrink = [&](auto kernel, int ranks) -> int {
      const dim3 grid((unsigned)(blocks + tiles), (unsigned)((a->rank + ranks - 1) / ranks));
      L3CI_LAUNCH("adapter_shrink_many_kernel", kernel, grid, dim3(32 * kShrinkWarps), 0, stream, *a, z, lists, (int)blocks);
      return L3CI_OK;
    };
    if (int st = a->rank <= 8 ? shrink(adapter_shrink_many_kernel<1>, 8) : a->rank <= 16 ? shrink(adapter_shrink_many_kernel<2>, 16) : shrink(adapter_shrink_many_kernel<4>, 32)) return st;
  }
  if (few) return adapter_rows_launch(&l, AdapterRows{z, a->index, b, a->rank, a->adapters});
  return adapter_many_launch(&l, AdapterMany{z, b, lists, a->rank, a->adapters, a->status});
}

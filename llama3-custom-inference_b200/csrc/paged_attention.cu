// Attention of new tokens over a paged cache (include/l3ci_b200.h, l3ci_paged_attention), sequences of few query rows (decode steps):
// bound by the bytes of the cache.  Chunks of many rows are paged_attention_tc.cu's.
//
// A unit is a sequence's KV head with the at most 16 query rows (tokens x heads) that share its keys; its keys are cut into tiles of 4 KB of
// K and 4 KB of V, and the tiles of all units, one behind the other, are dealt in equal runs to all warps of the device.  Lengths are known to
// the device alone, so every CTA adds them up for itself (a scan over the sequences); no mix of lengths leaves an SM idle, and none needs a host
// that knows them.  A warp streams its run through a ring of three tiles of its own (16-byte asynchronous copies into the 128-byte-swizzled
// layout that ldmatrix reads) without a word to the others: what stands at a run's ends is part of a unit and goes to scratch as running
// maximum, sum and fp32 products, which a second small launch merges; a unit that lies within a run is written at once.  Scratch holds nothing
// from one call to the next, so that calls and captured graphs share nothing.  (A counter per unit, with which the last part could merge in the same
// launch, would have to be cleared by a launch as well.)
// A token's place comes from the table: a lane holds the place of every 16 tokens of the next 512, asked for one block ahead.
// The arithmetic of a tile is that of flash_decode_small.cu: S^T = K Q^T and O^T += V^T P^T on mma.sync.m16n8k16, keys on the rows of a
// tile, query rows on its 8 columns, twice where there are more than 8.  p is rounded to bf16 for the second product (tensor cores take
// bf16 operands; a weight is off by at most 2^-8 of it), everything else is fp32.
// Measured on a B200: 16 sequences of 3500 to 8000 keys, 64 query on 8 KV heads of 128, pages of 16, 384 MB: 63.4 us, 6.05 TB/s, and 5.2 for the
// merge (eight parts at a time; one after the other 8); a sequence of 131072 keys, 32 on 8 heads, 537 MB: 83.6 us, 6.4 TB/s, and 7.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>

#include <type_traits>

#include "bf16x8.cuh"
#include "flash_decode_plan.h"
#include "host_common.h"
#include "paged_attention.h"
#include "ptx_sm100.cuh"
#include "warp_reduce.cuh"

namespace l3ci {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = 32 * kWarps;
constexpr int kSlots = 3;            // tiles in flight per warp
constexpr int kTileBytes = 8192;     // K then V
constexpr int kFewRows = 16;
constexpr int kMergeThreads = kThreads;   // (it counts the columns as the first kernel does)

constexpr size_t rows_smem(int B) { return 1024 + (size_t)kWarps * kSlots * kTileBytes + (size_t)(B + 1) * 4; }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid, uint64_t policy) {
  const int bytes = valid ? 16 : 0;  // 0: the 16 bytes are zero-filled
  asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2, %3;" ::"r"(dst), "l"(src), "r"(bytes), "l"(policy)
               : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ bool no_number(uint32_t bf16) { return (bf16 & 0x7f80u) == 0x7f80u; }   // NaN or infinite
__device__ __forceinline__ bool no_numbers(const uint4& v) {
  auto any = [](uint32_t w) { return no_number(w) || no_number(w >> 16); };
  return any(v.x) || any(v.y) || any(v.z) || any(v.w);
}

// Parts that `total` columns are dealt to.
__device__ __forceinline__ int parts_of(int total, int max_parts) { return min(total, max_parts); }

// Where a part of a unit goes: two records per warp, 0 for a unit that began in an earlier one, 1 for one that begins here.
template <int D, int NB>
__device__ __forceinline__ float* record_of(const PagedParams& p, int part, bool begins) {
  return p.records + (long long)(2 * part + (begins ? 1 : 0)) * (8 * NB * (D + 2));   // o[row][D], m[row], l[row]
}

// Columns of the deal before every sequence, pref[0 .. B], by all threads of the CTA (kThreads).
template <int D>
__device__ __forceinline__ void count_columns(const PagedParams& p, int* pref) {
  __shared__ int warp_sums[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  auto columns = [&](int b) {
    const PagedSeq s = paged_seq(p, b);
    return s.n > 0 ? p.a.Hkv * fd_tiles(s.len, fd_tile_tokens(D)) : 0;
  };
  const int each = (p.a.B + kThreads - 1) / kThreads, b0 = min((int)threadIdx.x * each, p.a.B), b1 = min(b0 + each, p.a.B);
  int mine = 0;
  for (int b = b0; b < b1; ++b) {
    const int c = columns(b);
    pref[b + 1] = c;
    mine += c;
  }
  int upto = mine;
#pragma unroll
  for (int d = 1; d < 32; d *= 2) {
    const int other = __shfl_up_sync(kFullMask, upto, d);
    if (lane >= d) upto += other;
  }
  if (lane == 31) warp_sums[warp] = upto;
  if (threadIdx.x == 0) pref[0] = 0;
  __syncthreads();
  int before = upto - mine;
  for (int w = 0; w < warp; ++w) before += warp_sums[w];
  for (int b = b0; b < b1; ++b) pref[b + 1] = before += pref[b + 1];
  __syncthreads();
}

// One warp's walk over the tiles of its run.
struct Cursor {
  int b, h, tile, tiles;
};

template <int D, int NB>
__global__ void __launch_bounds__(kThreads, 1) paged_rows_kernel(const PagedParams p) {
  constexpr int kTile = fd_tile_tokens(D);             // tokens per tile
  constexpr int kHalves = D / 64;
  constexpr int kBoxBytes = kTile * 128;               // one 64-column half of a tile
  constexpr int KS = D / 16, MB = kTile / 16, MT = D / 16;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  int* pref = reinterpret_cast<int*>(smem + kWarps * kSlots * kTileBytes);
  const l3ci_paged_attention_args& a = p.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gid = lane >> 2, tig = lane & 3;
  pdl_wait();                // (in this order: the chunk kernel and the merge behind read what the kernels before have written, without a wait of their own)
  pdl_launch_dependents();

  count_columns<D>(p, pref);
  const int total = pref[a.B];
  const int parts = parts_of(total, p.max_parts), part = warp * (int)gridDim.x + (int)blockIdx.x;   // (few parts: one per SM)
  if (part >= parts) return;
  const int begin = fd_range_begin(part, total, parts), end = fd_range_begin(part + 1, total, parts);

  auto enter = [&](Cursor& c, int b) {   // the first sequence from b on with columns
    while (b < a.B && pref[b + 1] == pref[b]) ++b;
    c.b = b;
    if (b < a.B) c.tiles = (pref[b + 1] - pref[b]) / a.Hkv;
  };
  auto seek = [&](int col) {
    int lo = 0, hi = a.B;                // largest b with pref[b] <= col (of equal ones the last, which has the columns)
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (pref[mid] <= col) lo = mid; else hi = mid;
    }
    Cursor c;
    c.b = lo;
    c.tiles = (pref[lo + 1] - pref[lo]) / a.Hkv;
    const int local = col - pref[lo];
    c.h = local / c.tiles;
    c.tile = local - c.h * c.tiles;
    return c;
  };
  auto advance = [&](Cursor& c) {
    if (++c.tile < c.tiles) return;
    c.tile = 0;
    if (++c.h < a.Hkv) return;
    c.h = 0;
    enter(c, c.b + 1);
  };

  // ---- copies: the fetching cursor runs kSlots tiles ahead ----
  const uint64_t policy = l2_evict_first_policy();
  const __nv_bfloat16* kc = static_cast<const __nv_bfloat16*>(a.cache_k);
  const __nv_bfloat16* vc = static_cast<const __nv_bfloat16*>(a.cache_v);
  const uint32_t buf0 = smem_u32(smem) + warp * kSlots * kTileBytes;
  const int r0 = lane >> 3, c8 = lane & 7;
  const long long row4 = 4 * a.cache_st;
  const uint32_t d_even = r0 * 128 + ((c8 ^ r0) << 4), d_odd = r0 * 128 + ((c8 ^ r0 ^ 4) << 4);   // (see flash_decode_small.cu)
  constexpr int kGran = MB;              // 16-token places of a tile
  Cursor f = seek(begin);
  int f_b = -1, f_block = -1, f_len = 0;
  long long place = -1;                  // this lane's 16 tokens of the block of 32 places: elements before them, -1: not there
  int ahead = -1;                        // the page of this lane's 16 tokens of the next block
  auto page_of = [&](int b, int block) { // (places behind the sequence's end are not looked up)
    const int token = (block * 32 + lane) * 16;
    return token < f_len ? __ldg(a.page_table + b * a.table_st + token / a.page_size) : -1;
  };
  auto fetch = [&](bool on, int slot) {
    if (on) {
      const int g0 = f.tile * kGran;
      if (f.b != f_b || g0 / 32 != f_block) {
        const bool next = f.b == f_b && g0 / 32 == f_block + 1;
        if (f.b != f_b) f_len = paged_seq(p, f.b).len;
        f_b = f.b;
        f_block = g0 / 32;
        const int page = next ? ahead : page_of(f_b, f_block);
        const int token = (f_block * 32 + lane) * 16;
        place = page >= 0 && page < a.pages ? page * a.cache_sp + (token % a.page_size) * a.cache_st : -1;
        ahead = page_of(f_b, f_block + 1);
      }
      const uint32_t dst = buf0 + slot * kTileBytes;
#pragma unroll
      for (int g = 0; g < kGran; ++g) {
        const long long at = __shfl_sync(kFullMask, place, (g0 + g) & 31);
        const long long off = at + f.h * D + r0 * a.cache_st + c8 * 8;
        const __nv_bfloat16* kp = kc + off;
        const __nv_bfloat16* vp = vc + off;
        const int left = at >= 0 ? f_len - (g0 + g) * 16 - r0 : 0;   // this lane's rows that are there: 4 j < left
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t d = dst + (g * 4 + j) * 512 + ((j & 1) ? d_odd : d_even);
          const bool ok = 4 * j < left;
#pragma unroll
          for (int h = 0; h < kHalves; ++h) {
            cp_async16(d + h * kBoxBytes, ok ? kp + h * 64 : kc, ok, policy);
            cp_async16(d + (kHalves + h) * kBoxBytes, ok ? vp + h * 64 : vc, ok, policy);
          }
          kp += row4;
          vp += row4;
        }
      }
      advance(f);
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < kSlots; ++i) fetch(begin + i < end, i);

  const int mat = lane >> 3, r8 = lane & 7;
  const uint32_t k_row_off = (r8 + 8 * (mat & 1)) * 128, k_x = (mat >> 1) ^ r8;
  const uint32_t v_row_off = (r8 + 8 * (mat >> 1)) * 128, v_x = (mat & 1) ^ r8;
  uint32_t qb[NB][KS][2];
  float o[NB][MT][4], m_run[NB][2], l_run[NB][2];
  int limit[NB][2], rows = 0, first_limit = 0, len = 0, n = 0;   // limit: last key of this lane's query rows
  bool fresh = true, begins = true;
  Cursor c = seek(begin);

  for (int col = begin; col < end; ++col) {
    if (fresh) {     // ---- a unit's query rows ----
      fresh = false;
      begins = c.tile == 0;
      const PagedSeq s = paged_seq(p, c.b);
      n = s.n;
      len = s.len;
      rows = n * p.R;
      first_limit = len - n;
      const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(a.q) + paged_row0(p, c.b, a.q_sb, a.q_st) + (long long)(c.h * p.R) * a.q_sh;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const int row = nb * 8 + gid, t = row / p.R;
        const __nv_bfloat16* qp = q + t * a.q_st + (row - t * p.R) * a.q_sh;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          qb[nb][ks][0] = row < rows ? ld_global_u32(qp + ks * 16 + 2 * tig) : 0u;
          qb[nb][ks][1] = row < rows ? ld_global_u32(qp + ks * 16 + 2 * tig + 8) : 0u;
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          limit[nb][j] = first_limit + min((nb * 8 + 2 * tig + j) / p.R, n - 1);
          m_run[nb][j] = -INFINITY;
          l_run[nb][j] = 0.f;
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) o[nb][mt][0] = o[nb][mt][1] = o[nb][mt][2] = o[nb][mt][3] = 0.f;
      }
    }
    const int slot = (col - begin) % kSlots;
    cp_async_wait<kSlots - 1>();
    __syncwarp();
    const uint32_t kb = buf0 + slot * kTileBytes, vb = kb + kHalves * kBoxBytes;
    const int tok0 = c.tile * kTile;
    // ---- S^T = K Q^T (several accumulators per score: a chain of KS dependent products is 20 cycles each) ----
    constexpr int kAcc = MB == 1 && NB == 1 ? 4 : 2;
    float sp[kAcc][NB][MB][4];
#pragma unroll
    for (int x = 0; x < kAcc; ++x)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) sp[x][nb][mb][0] = sp[x][nb][mb][1] = sp[x][nb][mb][2] = sp[x][nb][mb][3] = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        uint32_t a0, a1, a2, a3;
        ldsm_x4(kb + (ks >> 2) * kBoxBytes + mb * 2048 + k_row_off + (((2u * (ks & 3)) ^ k_x) << 4), a0, a1, a2, a3);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) mma_bf16(sp[ks % kAcc][nb][mb], a0, a1, a2, a3, qb[nb][ks][0], qb[nb][ks][1]);
      }
    const bool cut = tok0 + kTile > first_limit + 1;   // some row does not see all keys of the tile
    uint32_t pb[NB][MB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float s[MB][4];
#pragma unroll
      for (int mb = 0; mb < MB; ++mb)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float acc = sp[0][nb][mb][e];
#pragma unroll
          for (int x = 1; x < kAcc; ++x) acc += sp[x][nb][mb][e];
          s[mb][e] = acc;
        }
      if (cut) {
#pragma unroll
        for (int mb = 0; mb < MB; ++mb)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (tok0 + mb * 16 + gid + (e >> 1) * 8 > limit[nb][e & 1]) s[mb][e] = -INFINITY;
      }
      // ---- running softmax in the log2 domain; reductions over the 8 lanes of a column pair ----
      float alpha[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float mx = -INFINITY;
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) mx = fmaxf(mx, fmaxf(s[mb][j], s[mb][2 + j]));
        mx = fmaxf(mx, __shfl_xor_sync(kFullMask, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(kFullMask, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(kFullMask, mx, 16)) * p.scale_log2e;
        const float mn = fmaxf(m_run[nb][j], mx);
        const float mu = mn == -INFINITY ? 0.f : mn;
        alpha[j] = fast_exp2(m_run[nb][j] - mu);
        m_run[nb][j] = mn;
        float ps = 0.f;
#pragma unroll
        for (int mb = 0; mb < MB; ++mb) {
          s[mb][j] = fast_exp2(fmaf(s[mb][j], p.scale_log2e, -mu));
          s[mb][2 + j] = fast_exp2(fmaf(s[mb][2 + j], p.scale_log2e, -mu));
          ps += s[mb][j] + s[mb][2 + j];
        }
        l_run[nb][j] = fmaf(l_run[nb][j], alpha[j], ps);
      }
#pragma unroll
      for (int mb = 0; mb < MB; ++mb) {
        pb[nb][mb][0] = movmatrix_trans(pack_bf16x2(s[mb][0], s[mb][1]));
        pb[nb][mb][1] = movmatrix_trans(pack_bf16x2(s[mb][2], s[mb][3]));
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        o[nb][mt][0] *= alpha[0]; o[nb][mt][1] *= alpha[1];
        o[nb][mt][2] *= alpha[0]; o[nb][mt][3] *= alpha[1];
      }
    }
    // A value that is no number meets a weight of 0 in the rows that do not see its key, and 0 times it is no number either: such values are
    // taken out of the tile and added to the rows that see them.  Only tiles in which the rows of several tokens see different keys.
    if (cut && n > 1) {
      bool odd = false;
#pragma unroll
      for (int i = 0; i < kTileBytes / 2 / 512; ++i) {
        uint4 v;
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(vb + i * 512 + lane * 16) : "memory");
        odd |= no_numbers(v);
      }
      if (__any_sync(kFullMask, odd)) {
        auto value_at = [&](int j, int d) { return vb + (d >> 6) * kBoxBytes + j * 128 + ((((d & 63) >> 3) ^ (j & 7)) << 4) + (d & 7) * 2; };
#pragma unroll 1
        for (int j = 0; j < kTile; ++j)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              uint16_t w;
              asm volatile("ld.shared.u16 %0, [%1];" : "=h"(w) : "r"(value_at(j, 16 * mt + gid + 8 * e)) : "memory");
              if (no_number(w))
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                  for (int i = 0; i < 2; ++i)
                    if (tok0 + j <= limit[nb][i]) o[nb][mt][2 * e + i] += __uint_as_float((uint32_t)w << 16);
            }
        __syncwarp();
        for (int i = lane; i < kTile * D; i += 32) {
          const uint32_t at = value_at(i / D, i % D);
          uint16_t w;
          asm volatile("ld.shared.u16 %0, [%1];" : "=h"(w) : "r"(at) : "memory");
          if (no_number(w)) asm volatile("st.shared.u16 [%0], %1;" ::"r"(at), "h"((uint16_t)0) : "memory");
        }
        __syncwarp();
      }
    }
    // ---- O^T += V^T P^T ----
#pragma unroll
    for (int kk = 0; kk < MB; ++kk)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        uint32_t a0, a1, a2, a3;
        ldsm_x4_trans(vb + (mt >> 2) * kBoxBytes + kk * 2048 + v_row_off + (((2u * (mt & 3)) ^ v_x) << 4), a0, a1, a2, a3);
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) mma_bf16(o[nb][mt], a0, a1, a2, a3, pb[nb][kk][0], pb[nb][kk][1]);
      }
    __syncwarp();
    fetch(col + kSlots < end, slot);

    const bool last = c.tile == c.tiles - 1;
    if (last || col == end - 1) {     // ---- the unit ends, or this warp's part of it ----
      fresh = true;
      const bool whole = begins && last;
      float* rec = whole ? nullptr : record_of<D, NB>(p, part, begins);
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + paged_row0(p, c.b, a.o_sb, a.o_st) + (long long)(c.h * p.R) * a.o_sh;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          l_run[nb][j] += __shfl_xor_sync(kFullMask, l_run[nb][j], 4);
          l_run[nb][j] += __shfl_xor_sync(kFullMask, l_run[nb][j], 8);
          l_run[nb][j] += __shfl_xor_sync(kFullMask, l_run[nb][j], 16);
        }
        if (whole) {
          const float i0 = l_run[nb][0] == 0.f ? 0.f : 1.f / l_run[nb][0], i1 = l_run[nb][1] == 0.f ? 0.f : 1.f / l_run[nb][1];
          // neighbouring columns lie 4 lanes apart: even ones take row 2 tig, odd ones row 2 tig + 1
          const int row = nb * 8 + 2 * tig + (gid & 1), t = row / p.R;
          __nv_bfloat16* to = out + t * a.o_st + (row - t * p.R) * a.o_sh + (gid & ~1);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float x = o[nb][mt][2 * e] * i0, y = o[nb][mt][2 * e + 1] * i1;
              const float other = __shfl_xor_sync(kFullMask, (gid & 1) ? x : y, 4);
              if (row < rows) *reinterpret_cast<uint32_t*>(to + 16 * mt + 8 * e) = (gid & 1) ? pack_bf16x2(other, y) : pack_bf16x2(x, other);
            }
        } else {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const int row = nb * 8 + 2 * tig + j;
            if (row >= rows) continue;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              rec[row * D + 16 * mt + gid] = o[nb][mt][j];
              rec[row * D + 16 * mt + gid + 8] = o[nb][mt][2 + j];
            }
            if (gid == 0) {
              rec[8 * NB * D + row] = m_run[nb][j];
              rec[8 * NB * (D + 1) + row] = l_run[nb][j];
            }
          }
        }
      }
    }
    advance(c);
  }
  cp_async_wait<0>();
}

// Merges the parts of the units of few rows that were cut.  D / 4 lanes per query row and group of parts, `groups` (a power of two) groups of parts
// per row.
template <int D, int NB>
__device__ __forceinline__ void merge_rows(const PagedParams& p, const int* pref, int groups, int row_slots, int cta) {
  constexpr int kTile = fd_tile_tokens(D), kLanes = D / 4, kSets = kMergeThreads / kLanes;
  __shared__ float4 sums[kSets][kLanes];
  __shared__ float2 stats[kSets];
  const l3ci_paged_attention_args& a = p.a;
  const int set = threadIdx.x / kLanes, lane = threadIdx.x % kLanes, group = set & (groups - 1);
  const long long item = (long long)cta * (kSets / groups) + set / groups;
  const long long unit = item / row_slots;
  const int row = (int)(item - unit * row_slots), b = (int)(unit / a.Hkv), h = (int)(unit - (long long)b * a.Hkv);
  bool live = b < a.B;
  const PagedSeq s = live ? paged_seq(p, b) : PagedSeq{0, 0};
  live = live && row < s.n * p.R;
  int first = 0, last = 0, parts = 1, total = 0;
  if (live) {
    const int tiles = fd_tiles(s.len, kTile), begin = pref[b] + h * tiles;
    total = pref[a.B];
    parts = parts_of(total, p.max_parts);
    first = fd_cta_of(begin, total, parts);
    last = fd_cta_of(begin + tiles - 1, total, parts);
    live = last > first;
  }
  float m = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  if (live) {
    constexpr int kAtOnce = 8;
    for (int p0 = first + group; p0 <= last; p0 += groups * kAtOnce) {
      float mv[kAtOnce], lv[kAtOnce];
      float4 ov[kAtOnce];
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        const int part = p0 + i * groups;
        mv[i] = -INFINITY;
        lv[i] = 0.f;
        ov[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (part <= last) {
          const float* rec = record_of<D, NB>(p, part, part == first);
          ov[i] = __ldcg(reinterpret_cast<const float4*>(rec + row * D) + lane);
          mv[i] = __ldcg(rec + 8 * NB * D + row);
          lv[i] = __ldcg(rec + 8 * NB * (D + 1) + row);
        }
      }
      float mn = m;
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) mn = fmaxf(mn, mv[i]);
      const float mu = mn == -INFINITY ? 0.f : mn, w0 = fast_exp2(m - mu);
      l *= w0;
      acc.x *= w0; acc.y *= w0; acc.z *= w0; acc.w *= w0;
      m = mn;
#pragma unroll
      for (int i = 0; i < kAtOnce; ++i) {
        if (p0 + i * groups > last) break;
        const float w = fast_exp2(mv[i] - mu);
        l = fmaf(lv[i], w, l);
        acc.x = fmaf(ov[i].x, w, acc.x);
        acc.y = fmaf(ov[i].y, w, acc.y);
        acc.z = fmaf(ov[i].z, w, acc.z);
        acc.w = fmaf(ov[i].w, w, acc.w);
      }
    }
  }
  if (groups > 1) {
    sums[set][lane] = acc;
    if (lane == 0) stats[set] = make_float2(m, l);
    __syncthreads();
    if (group != 0) return;
    float mn = -INFINITY;
    for (int g = 0; g < groups; ++g) mn = fmaxf(mn, stats[set + g].x);
    const float mu = mn == -INFINITY ? 0.f : mn;
    l = 0.f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int g = 0; g < groups; ++g) {
      const float w = fast_exp2(stats[set + g].x - mu);
      const float4 v = sums[set + g][lane];
      l = fmaf(stats[set + g].y, w, l);
      acc.x = fmaf(v.x, w, acc.x);
      acc.y = fmaf(v.y, w, acc.y);
      acc.z = fmaf(v.z, w, acc.z);
      acc.w = fmaf(v.w, w, acc.w);
    }
  }
  if (!live) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int t = row / p.R;
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + paged_row0(p, b, a.o_sb, a.o_st) + t * a.o_st + (long long)(h * p.R + row - t * p.R) * a.o_sh;
  *reinterpret_cast<uint2*>(out + lane * 4) = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
}

// Puts the parts of a cut unit of a chunk together: kShares CTAs for every part of the deal, each with a share of the unit's rows and columns.
constexpr int kMergeItems = 4;       // float4 a thread merges
template <int D>
constexpr int kShares = 2 * kChunkRows * (D / 4) / (kMergeThreads * kMergeItems);

template <int D>
__device__ __forceinline__ void merge_chunk(const ChunkParams& cp, int cta) {
  const PagedParams& p = cp.p;
  const l3ci_paged_attention_args& a = p.a;
  const int4 c0 = __ldcg(reinterpret_cast<const int4*>(cp.cuts + cta / kShares<D> + 1)), c1 = __ldcg(reinterpret_cast<const int4*>(cp.cuts + cta / kShares<D> + 1) + 1);
  const int b = c0.x, h = c0.y, m = c0.z, first = c0.w, parts = c1.x;
  if (parts < 2) return;
  const PagedSeq s = paged_seq(p, b);
  const int t_unit = m * 2 * cp.tile_tokens;
  const long long row0 = paged_row0(p, b, a.o_sb, a.o_st);
  // neighbouring lanes: 8 rows of 4 vectors each (runs of 128 bytes of a part, of 32 bytes of the result)
  constexpr int kPerRow = D / 4;
#pragma unroll 1
  for (int i = 0; i < kMergeItems; ++i) {
    const int item = (cta % kShares<D> * kMergeItems + i) * kMergeThreads + threadIdx.x;
    const int in8 = item & 31, rest = item >> 5;
    const int vec = (rest % (kPerRow / 4)) * 4 + (in8 >> 3), row = rest / (kPerRow / 4) * 8 + (in8 & 7);   // row: 0 .. 255
    const int e = row / kChunkRows, t = (row % kChunkRows) / p.R, token = t_unit + e * cp.tile_tokens + t;
    if (t >= cp.tile_tokens || token >= s.n) continue;
    float mx = -INFINITY, l = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int kAtOnce = 4;
    for (int p0 = 0; p0 < parts; p0 += kAtOnce) {
      float mv[kAtOnce], lv[kAtOnce];
      float4 ov[kAtOnce];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        mv[k] = -INFINITY;
        lv[k] = 0.f;
        ov[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (p0 + k < parts) {
          const float* rec = chunk_part_of<D>(p, first + p0 + k, p0 + k == 0);
          ov[k] = __ldcg(reinterpret_cast<const float4*>(rec) + vec * (2 * kChunkRows) + row);
          mv[k] = __ldcg(rec + 2 * kChunkRows * D + row);
          lv[k] = __ldcg(rec + 2 * kChunkRows * (D + 1) + row);
        }
      }
      float mn = mx;
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) mn = fmaxf(mn, mv[k]);
      const float mu = mn == -INFINITY ? 0.f : mn, w0 = fast_exp2(mx - mu);
      l *= w0;
      acc.x *= w0; acc.y *= w0; acc.z *= w0; acc.w *= w0;
      mx = mn;
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        if (p0 + k >= parts) break;
        const float w = fast_exp2(mv[k] - mu);
        l = fmaf(lv[k], w, l);
        acc.x = fmaf(ov[k].x, w, acc.x);
        acc.y = fmaf(ov[k].y, w, acc.y);
        acc.z = fmaf(ov[k].z, w, acc.z);
        acc.w = fmaf(ov[k].w, w, acc.w);
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + row0 + token * a.o_st + (long long)(h * p.R + row % kChunkRows - t * p.R) * a.o_sh;
    *reinterpret_cast<uint2*>(out + vec * 4) = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
  }
}

// NB 0: no sequences of few rows.  The first rows_ctas CTAs are theirs.
template <int D, int NB>
__global__ void __launch_bounds__(kMergeThreads) paged_merge_kernel(const PagedParams p, int groups, int row_slots, int rows_ctas, const ChunkParams cp) {
  extern __shared__ int merge_pref[];
  // (the lengths were complete before the first kernel of the call let the next one start)
  const bool rows = NB > 0 && (int)blockIdx.x < rows_ctas;
  if (rows) count_columns<D>(p, merge_pref);
  pdl_wait();
  pdl_launch_dependents();
  if constexpr (NB > 0)
    if (rows) return merge_rows<D, NB>(p, merge_pref, groups, row_slots, blockIdx.x);
  merge_chunk<D>(cp, blockIdx.x - rows_ctas);
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
  // (columns of a sequence, 16 keys of a head each, are counted in 32 bits)
  if (rows > 0x7fffffffLL || a->pages > 0x7fffffffLL || (long long)a->max_pages * a->page_size > (1LL << 30) / (a->Hkv < 16 ? 16 : a->Hkv) * 16)
    return fail(L3CI_ERR_INVALID, "paged_attention: %lld rows, %lld keys a sequence", rows, (long long)a->max_pages * a->page_size);
  if ((a->starts ? a->rows : a->T) * (a->Hq / a->Hkv) > kFewRows && paged_chunk_columns(a) >= 0x7fffffffLL)
    return fail(L3CI_ERR_INVALID, "paged_attention: %lld rows over up to %lld keys are too many for one call", rows, (long long)a->max_pages * a->page_size);
  return L3CI_OK;
}

}  // namespace

// ---- host ----
namespace {

// How a launch over sequences of few rows is laid out.
struct RowsPlan {
  int NB, ctas, max_parts, row_slots;
  size_t bytes;                  // of scratch
};

RowsPlan rows_plan(const PagedParams& p) {
  RowsPlan r;
  const l3ci_paged_attention_args& a = p.a;
  const int sms = sm_count() > 0 ? sm_count() : 148;
  const long long rows = a.starts ? a.rows * p.R : (long long)a.T * p.R;     // of one sequence at most
  r.row_slots = (int)(rows < p.max_rows ? rows : p.max_rows);
  r.NB = r.row_slots <= 8 ? 1 : 2;
  const long long columns = (long long)a.B * a.Hkv * fd_tiles(p.cap, fd_tile_tokens(a.D));
  r.max_parts = (int)(columns < (long long)sms * kWarps ? columns : (long long)sms * kWarps);
  r.ctas = r.max_parts < sms ? r.max_parts : sms;
  r.bytes = (size_t)r.max_parts * 2 * 8 * r.NB * (a.D + 2) * 4;
  return r;
}

// The sequences of few rows (NB 0: none) and of many of one launch, and the merge.
template <int D, int NB>
int launch(PagedParams p, const RowsPlan& r, bool many, void* scratch, cudaStream_t stream) {
  int groups = 1;
  long long rows_ctas = 0;
  ChunkParams cp = {};
  if constexpr (NB > 0) {
    p.min_rows = 1;
    p.max_rows = kFewRows;
    p.records = static_cast<float*>(scratch);
    p.max_parts = r.max_parts;
    static bool configured[64] = {false};
    int dev = 0;
    L3CI_CUDA_TRY(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64 || !configured[dev]) {
      L3CI_CUDA_TRY(cudaFuncSetAttribute(paged_rows_kernel<D, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)rows_smem(kPagedMaxSeqs)));
      if (dev >= 0 && dev < 64) configured[dev] = true;
    }
    L3CI_LAUNCH("paged_rows_kernel", paged_rows_kernel<D, NB>, dim3((unsigned)r.ctas), dim3(kThreads), rows_smem(p.a.B), stream, p);
    // up to eight parts a group of lanes (four: twice the CTAs, two waves of them, 16 sequences of 8 KV heads of 8 query heads 8.2 us instead of 5.2)
    const long long units = (long long)p.a.B * p.a.Hkv, each = r.max_parts / units;
    constexpr int kSets = kMergeThreads / (D / 4);
    while (groups < kSets && each > 8 * groups) groups *= 2;
    rows_ctas = (units * r.row_slots + kSets / groups - 1) / (kSets / groups);
  }
  long long chunk_ctas = 0;
  if (many) {
    PagedParams c = p;
    c.min_rows = kFewRows + 1;
    c.max_rows = INT32_MAX;
    // (its own part of the scratch: where both kernels run, the second does not wait for the first)
    if (int st = paged_chunks_launch(c, static_cast<uint8_t*>(scratch) + (NB > 0 ? r.bytes : 0), NB > 0, stream, &cp)) return st;
    chunk_ctas = (long long)(cp.p.max_parts - 1) * kShares<D>;
  }
  if (rows_ctas + chunk_ctas > 0)
    L3CI_LAUNCH("paged_merge_kernel", paged_merge_kernel<D, NB>, dim3((unsigned)(rows_ctas + chunk_ctas)), dim3(kMergeThreads), NB > 0 ? (size_t)(p.a.B + 1) * 4 : 0, stream, p, groups, r.row_slots, (int)rows_ctas, cp);
  return L3CI_OK;
}

PagedParams params_of(const l3ci_paged_attention_args* a) {
  PagedParams p = {};
  p.a = *a;
  if (!a->starts) p.a.rows = (long long)a->B * a->T;
  p.R = a->Hq / a->Hkv;
  p.cap = a->max_pages * a->page_size;
  p.scale_log2e = (a->scale > 0.f ? a->scale : 1.0f / sqrtf((float)a->D)) * 1.4426950408889634f;
  return p;
}

// Sequences per launch: as many as fit the kernels' shared memory and whose columns can be counted in 32 bits.
int seqs_per_launch(const PagedParams& p) {
  const long long each = (long long)p.a.Hkv * fd_tiles(p.cap, 16);
  const long long fit = 0x7fffffffLL / each;
  return (int)(fit < kPagedMaxSeqs ? fit : kPagedMaxSeqs);
}

// Which kernels a call of these sizes may need: sequences of up to kFewRows query rows, and of more.
void kernels_of(const PagedParams& p, bool* few, bool* many) {
  const long long rows = (p.a.starts ? p.a.rows : p.a.T) * p.R;
  *few = p.a.starts ? true : rows <= kFewRows;
  *many = rows > kFewRows;
}

size_t scratch_of(PagedParams p) {
  const int most = seqs_per_launch(p);
  if (p.a.B > most) p.a.B = most;
  bool few, many;
  kernels_of(p, &few, &many);
  size_t bytes = 0;
  if (few) {
    p.max_rows = kFewRows;
    bytes = rows_plan(p).bytes;
  }
  return bytes + (many ? paged_chunks_scratch_bytes(p) : 0);
}

}  // namespace
}  // namespace l3ci

extern "C" size_t l3ci_paged_attention_scratch_bytes(const l3ci_paged_attention_args* a) {
  using namespace l3ci;
  const int st = check(a);
  clear_error();
  return st ? 0 : scratch_of(params_of(a));
}

extern "C" int l3ci_paged_attention(const l3ci_paged_attention_args* a) {
  using namespace l3ci;
  clear_error();
  if (int st = check(a)) return st == kNothing ? L3CI_OK : st;
  PagedParams p = params_of(a);
  const size_t need = scratch_of(p);
  if (need && (!a->scratch || a->scratch_bytes < need || !aligned16(a->scratch)))
    return fail(L3CI_ERR_SCRATCH, "paged_attention: %zu bytes of scratch, %zu are needed", a->scratch_bytes, need);
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(a->stream);
  bool few, many;
  kernels_of(p, &few, &many);
  const int most = seqs_per_launch(p);
  for (int b0 = 0; b0 < a->B; b0 += most) {
    p.a.B = a->B - b0 < most ? a->B - b0 : most;
    p.a.page_table = a->page_table + b0 * a->table_st;
    p.a.seq_lens = a->seq_lens + b0;
    if (a->starts) {
      p.a.starts = a->starts + b0;
    } else {
      p.a.q = static_cast<const __nv_bfloat16*>(a->q) + b0 * a->q_sb;
      p.a.out = static_cast<__nv_bfloat16*>(a->out) + b0 * a->o_sb;
      p.a.rows = (long long)p.a.B * p.a.T;
    }
    p.max_rows = kFewRows;
    const RowsPlan r = few ? rows_plan(p) : RowsPlan{};
    auto go = [&](auto d) {
      constexpr int D = decltype(d)::value;
      return r.NB == 0 ? launch<D, 0>(p, r, many, a->scratch, stream) : r.NB == 1 ? launch<D, 1>(p, r, many, a->scratch, stream) : launch<D, 2>(p, r, many, a->scratch, stream);
    };
    if (int st = a->D == 64 ? go(std::integral_constant<int, 64>{}) : go(std::integral_constant<int, 128>{})) return st;
  }
  return L3CI_OK;
}

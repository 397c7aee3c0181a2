// Attention of new tokens over a paged cache (include/l3ci_b200.h, l3ci_paged_attention), sequences of more than a few query rows: chunks of
// prompts.  Bound by the tensor cores (4 D operations per query row and key) and by the instructions of the softmax between the two products.
//
// The same pipeline as prefill_tc_persist_kernel (prefill_attention_tc.cu): tcgen05 products with accumulators in tensor memory, a producer
// warp, an MMA warp, two softmax groups, an output group.  What differs:
//   * a tile of 128 query rows is 128 / R tokens by the R query heads of a KV head, so that K and V are read once for all of them, whatever R is
//     (two tiles, e = 0 and 1, share them: a unit);
//   * keys come page by page: a tile of 128 keys is filled by copies of as many tokens as lie together in every page (a power of two from 16),
//     each lane of the producer with its own page;
//   * tiles of keys of all units are dealt in equal runs to the CTAs, by lengths that the device alone knows; a unit that a run's end cuts goes to
//     scratch as maximum, sum and fp32 products, and paged_merge_kernel puts the parts together;
//   * what lies behind a sequence's end in its last page, and values that some rows of a tile must not see, may be no numbers, and a
//     weight of 0 does not stop them: two guard warps look through V tiles at the diagonal and the end, under the first product and the softmax
//     of the same tile, take such values out, and the output group adds them to the rows that see them.
// Measured on a B200, rows of 40 calls, merge included: 2 x 512 tokens of 16500 keys, 32 query on 8 KV heads of 128, 241 us, 1130 TFLOP/s (284, 960, in long
// runs, at the power limit), heads of 64 192, 711; a prompt of
// 4096 tokens, heads of 128 157 us, 876, of 64 115, 600 (a head of 64 has half the products to the same exponentials).  A tile of keys takes
// 3650 cycles (heads of 128), of which a warp's softmax is 2030 (its exponentials alone 1450 for the 1024 that they cannot do without) and
// the wait for the products between 1240; the tensor cores need 2050 and the exponentials of both groups as much.  For heads of 64 the weights
// in a place of their own, so that the next scores come under the exponentials: both groups then take theirs at once, 234 us instead of 227 (of 202
// with the first half of the weights multiplied ahead).
// Scores read from tensor memory twice by loops of 32 keys instead of once: 3 to 10 % slower.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>

#include "bf16x8.cuh"
#include "flash_decode_plan.h"
#include "host_common.h"
#include "paged_attention.h"
#include "ptx_sm100.cuh"
#include "tcgen05.cuh"
#include "tensor_map.h"
#include "warp_reduce.cuh"

namespace l3ci {
namespace {

// Where a wait that ran out is recorded by calls without a status word of their own, until l3ci_paged_attention_poll reads it.
__device__ int g_wait_status = 0;

constexpr int kRows = kChunkRows;   // query rows of a tile (M of the products)
constexpr int kKeys = 128;     // keys of a tile
constexpr int kStages = 2;
constexpr int kSoftmaxWarps = 8;
constexpr int kThreads = 32 * (4 + kSoftmaxWarps + 4);
constexpr int kReaders = 1 + 2 + kSoftmaxWarps + 4;            // warps that read the segments
constexpr int kRegsLow = 56, kRegsHigh = 192, kRegsOut = 72;   // of the producer's, the softmax and the output warpgroups
static_assert(4 * kRegsLow + kSoftmaxWarps * kRegsHigh + 4 * kRegsOut <= 16 * 128, "register re-deal");
constexpr uint32_t kTmemCols = 512;                            // S_0, S_1 (128 columns each), O_0, O_1 (D columns each)
constexpr int kSegments = 8;   // of the ring (the guards are at most three ahead of the output: one-tile segments, two in the ring of V, one on its way out)
// Columns that a tile counts in the deal, and a unit beside its tiles: its start and its end.
constexpr int kTileCost = 2;
constexpr int unit_cost(int D) { return D == 128 ? 3 : 1; }

// Keys that the tokens of block m (2 * tile_tokens tokens) of a sequence see, in tiles; at least one.
__device__ __forceinline__ int unit_tiles(const PagedSeq& s, int m, int block) {
  const int seen = s.len - s.n + min(s.n, (m + 1) * block);
  return seen <= 0 ? 1 : (seen + kKeys - 1) / kKeys;
}

// What a CTA does next: tiles [j0, j1) of a unit's keys; j1 0: nothing is left.  The producer walks through the deal and leaves these in a ring for
// the other warps, whose code has to be short.
struct Segment {
  int j0, j1, ne;      // ne: tiles of rows, 1 or 2
  int limit;           // last key that the unit's first token sees
  int len, b, h;
  int t0, n, row;      // the unit's first token, the sequence's tokens, its row in packed tensors
  int whole, pad;
};

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
paged_chunk_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap,
                   const __grid_constant__ ChunkParams cp) {
  // Whether the product of the first half of a tile's weights with their values starts under the exponentials of the second.  (Heads of 64 and of 128, 2 x 512
  // tokens of 16500 keys: 227 us to 202, 243 either way and 1 % more at the power limit.)
  constexpr bool kHalfWeights = D == 64;
  constexpr int kHalves = D / 64;
  constexpr int kBoxBytes = 128 * 128;             // 128 rows of 128 bytes
  constexpr int kTileBytes = kHalves * kBoxBytes;  // a Q, K or V tile
  constexpr int kSPitch = 64 + 16;                 // staging row: 32 output columns + padding
  const PagedParams& p = cp.p;
  const l3ci_paged_attention_args& a = p.a;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t q_smem = smem_u32(smem);
  const uint32_t k_smem = q_smem + 2 * kTileBytes;             // [kStages]
  const uint32_t v_smem = k_smem + kStages * kTileBytes;       // [kStages]
  uint8_t* stage_all = smem + (2 + 2 * kStages) * kTileBytes;  // [2 tiles][128 rows][kSPitch]
  uint64_t* bars = reinterpret_cast<uint64_t*>(stage_all + 2 * kRows * kSPitch);
  // as in prefill_tc_persist_kernel; V_OK: the guard warps have been through the tile, if it is one of theirs
  // (they arrive on V_EMPTY too, so that they never miss a phase of V_FULL)
  enum { Q_FULL = 0, K_FULL = 1, K_EMPTY = 3, V_FULL = 5, V_EMPTY = 7, S_FULL = 9, O_FULL = 11, Q_EMPTY = 13, V_OK = 14, P_FULL = 16, L_FULL = 18, O_READ = 20, P_HALF = 22,
         SEG_FULL = 24, SEG_EMPTY = SEG_FULL + kSegments, N_BARS = SEG_EMPTY + kSegments };
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + N_BARS);
  int* odd = reinterpret_cast<int*>(bars + N_BARS + 1);            // [kSegments]: one more than the number of the last segment of which values were taken out
  int* sums = odd + kSegments;                                            // [16 warps]
  float* stat = reinterpret_cast<float*>(sums + 16);               // [2 tiles][128 rows][l, m_ref]
  Segment* segs = reinterpret_cast<Segment*>(stat + 4 * kRows);    // [kSegments]
  int* pref = reinterpret_cast<int*>(segs + kSegments);            // [B + 1]
  const uint32_t bar0 = smem_u32(bars);
  auto bar = [&](int i) { return bar0 + 8u * i; };
  auto wait = [&](uint32_t at, uint32_t parity) { return mbar_wait_bounded_lo(at, parity, cp.wait_ns); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < N_BARS; ++i)
      mbar_init(bar(i), i >= SEG_EMPTY ? kReaders : i >= SEG_FULL ? 1 : i >= P_FULL ? kSoftmaxWarps / 2 : i >= V_OK ? 2 : i == V_EMPTY || i == V_EMPTY + 1 ? 3 : 1);
    for (int i = 0; i < kSegments; ++i) odd[i] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&qmap)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&kmap)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&vmap)) : "memory");
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), kTmemCols);
    tmem_relinquish();
  }
  if (!cp.follows) pdl_wait();
  // ---- columns of the deal before every sequence ----
  // (The host has seen that the rows of the call, each counted once, stay below 2^31.  `starts` that do not ascend may name rows again and again: a sum that
  // gets there stays there, and nothing is done.)
  constexpr int kMost = 0x7fffffff;
  auto add = [](int x, int y) { return (int)min((unsigned)x + (unsigned)y, (unsigned)kMost); };
  constexpr int kUnitCost = unit_cost(D);
  const int block = 2 * cp.tile_tokens;
  auto columns_of_head = [&](const PagedSeq& s) {
    int sum = 0;
    for (int m = 0; m * block < s.n; ++m) sum += kUnitCost + kTileCost * unit_tiles(s, m, block);
    return sum;
  };
  {
    const int each = (a.B + kThreads - 1) / kThreads, b0 = min((int)threadIdx.x * each, a.B), b1 = min(b0 + each, a.B);
    int mine = 0;
    for (int b = b0; b < b1; ++b) {
      const int c = a.Hkv * columns_of_head(paged_seq(p, b));
      pref[b + 1] = c;
      mine = add(mine, c);
    }
    int upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
      const int other = __shfl_up_sync(kFullMask, upto, d);
      if (lane >= d) upto = add(upto, other);
    }
    if (lane == 31) sums[warp] = upto;
    if (threadIdx.x == 0) pref[0] = 0;
    __syncthreads();
    int before = upto - mine;
    for (int w = 0; w < warp; ++w) before = add(before, sums[w]);
    for (int b = b0; b < b1; ++b) pref[b + 1] = before = add(before, pref[b + 1]);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();   // (behind pdl_wait, here or in paged_rows_kernel: the merge reads lengths and starts before its own)
  const uint32_t tmem = *tmem_slot;
  const uint32_t t_s[2] = {tmem, tmem + 128u};
  const uint32_t t_o[2] = {tmem + 256u, tmem + 256u + (uint32_t)D};
  const int total = pref[a.B] == kMost ? 0 : pref[a.B], parts = max(min(total / kTileCost, p.max_parts), 1), part = blockIdx.x;   // (no run between two tiles' first columns)
  const int begin = total > 0 && part < parts ? fd_range_begin(part, total, parts) : 0, end = total > 0 && part < parts ? fd_range_begin(part + 1, total, parts) : 0;

  // the next segment; false: the wait for it ran out
  auto take = [&](int k) {
    __syncwarp();
    if (k > 0 && lane == 0) mbar_arrive(bar(SEG_EMPTY + (k - 1) % kSegments));
    return wait(bar(SEG_FULL + k % kSegments), (k / kSegments) & 1);
  };
  auto cut_tile = [&](int j, int limit) { return j * kKeys + kKeys - 1 > limit; };    // some row does not see all keys
  bool ok = true;
  int fill = 0;        // tiles of keys so far: stage and phase of the rings follow
  int segments = 0;

  if (warp == 0) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsLow));
    // ---- producer: deals the segments; lane 0 copies the query rows, every lane the tokens of its own copies ----
    struct Unit { int b, h, m, n, len, first, tiles; };   // first: its first column
    auto unit_at = [&](int col) {                         // the unit that holds a column
      int lo = 0, hi = a.B;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (pref[mid] <= col) lo = mid; else hi = mid;
      }
      Unit u;
      u.b = lo;
      const PagedSeq s = paged_seq(p, lo);
      u.n = s.n;
      u.len = s.len;
      const int per_head = (pref[lo + 1] - pref[lo]) / a.Hkv, local = col - pref[lo];
      u.h = local / per_head;
      int before = u.h * per_head;
      for (u.m = 0;; ++u.m) {
        u.tiles = unit_tiles(s, u.m, block);
        if (before + kUnitCost + kTileCost * u.tiles > local) break;
        before += kUnitCost + kTileCost * u.tiles;
      }
      u.first = pref[lo] + before;
      return u;
    };
    auto next_unit = [&](Unit& u) {
      u.first += kUnitCost + kTileCost * u.tiles;
      if (++u.m * block >= u.n) {
        u.m = 0;
        if (++u.h == a.Hkv) {
          u.h = 0;
          do ++u.b; while (u.b < a.B && pref[u.b + 1] == pref[u.b]);
          if (u.b >= a.B) return;
          const PagedSeq s = paged_seq(p, u.b);
          u.n = s.n;
          u.len = s.len;
        }
      }
      u.tiles = unit_tiles(PagedSeq{u.n, u.len}, u.m, block);
    };
    // (a tile is dealt with its first column)
    auto tiles_from = [&](const Unit& u, int col) { return max(col - u.first - kUnitCost + kTileCost - 1, 0) / kTileCost; };
    Unit u = {}, held = {};
    int col = begin;
    bool on = begin < end, waits = false, last = false;    // the run's first unit's part is still to come; it is at work
    if (on) {
      u = unit_at(begin);
      if (tiles_from(u, begin) == u.tiles) next_unit(u);
      on = u.first + kUnitCost < end && tiles_from(u, end) > tiles_from(u, begin);
    }
    if (lane == 0) {      // what the merge has to know of a unit that this run begins in the middle of
      ChunkCut cut = {};
      if (on && u.first + kUnitCost < begin) {
        cut.first = fd_cta_of(u.first + kUnitCost, total, parts);
        if (cut.first == part - 1) {
          cut.b = u.b;
          cut.h = u.h;
          cut.m = u.m;
          cut.parts = fd_cta_of(u.first + kUnitCost + kTileCost * (u.tiles - 1), total, parts) - cut.first + 1;
        }
      }
      cp.cuts[part] = cut;
    }
    // Such a part is taken last: the runs of one head then start at its first keys together and go through them side by side, and K and V come
    // from memory about once (in the order of the deal they came six times: 907 MB instead of 135 for 2 x 512 tokens of 16500 keys).
    if (on && u.first + kUnitCost < begin && u.first + 2 * kUnitCost + kTileCost * u.tiles < end) {
      held = u;
      waits = true;
      next_unit(u);
      col = u.first;
    }
    const uint64_t policy = l2_evict_first_policy();
    const int copies = kKeys / cp.box;                      // per half of a tile
    for (;; ++segments) {
      const int slot = segments % kSegments;
      if (segments >= kSegments && !wait(bar(SEG_EMPTY + slot), (segments / kSegments - 1) & 1)) { ok = false; break; }
      const int j0 = tiles_from(u, col), j1 = on ? min(u.tiles, tiles_from(u, end)) : 0;
      const int row = a.starts && on ? __ldg(a.starts + u.b) : 0;
      const bool two = (u.m * 2 + 1) * cp.tile_tokens < u.n;
      if (lane == 0) {
        segs[slot] = Segment{j0, j1, two ? 2 : 1, u.len - u.n + u.m * block, u.len, u.b, u.h, u.m * block, u.n, row, j0 == 0 && j1 == u.tiles, 0};
        mbar_arrive(bar(SEG_FULL + slot));
      }
      if (!on) break;
      auto page_of = [&](int j) {                          // of this lane's tokens of tile j; one past the last: nothing is there
        const int token = j * kKeys + lane * cp.box;
        const int page = lane < copies && token < u.len ? __ldg(a.page_table + u.b * a.table_st + token / a.page_size) : -1;
        return page >= 0 && page < a.pages ? page : (int)a.pages;
      };
      int page = page_of(j0);
      for (int j = j0; j < j1 && ok; ++j, ++fill) {
        const int s = fill % kStages, off = (j * kKeys + lane * cp.box) % a.page_size;
        const int ahead = page_of(j + 1);
        const uint32_t par = ((fill / kStages) - 1) & 1;
        auto load = [&](const CUtensorMap& map, uint32_t to, uint32_t full) {
          if (lane == 0) mbar_expect_tx(full, kTileBytes);
          __syncwarp();
          if (lane < copies)
#pragma unroll
            for (int h = 0; h < kHalves; ++h) tma_load_4d(to + s * kTileBytes + h * kBoxBytes + lane * cp.box * 128, &map, full, h * 64, off, u.h, page, policy);
        };
        if (fill >= kStages && !wait(bar(K_EMPTY + s), par)) { ok = false; break; }
        load(kmap, k_smem, bar(K_FULL + s));
        if (j == j0) {     // (behind the first keys, whose place is free before the last unit's scores are done)
          if (segments > 0 && !wait(bar(Q_EMPTY), (segments - 1) & 1)) { ok = false; break; }
          if (lane == 0) {
            const int tiles = two ? 2 : 1;
            mbar_expect_tx(bar(Q_FULL), tiles * kHalves * cp.tile_tokens * p.R * 128);
            for (int e = 0; e < tiles; ++e)
#pragma unroll
              for (int h = 0; h < kHalves; ++h)
                tma_load_4d(q_smem + e * kTileBytes + h * kBoxBytes, &qmap, bar(Q_FULL), h * 64, u.h * p.R, row + u.m * block + e * cp.tile_tokens, a.starts ? 0 : u.b, policy);
          }
        }
        if (fill >= kStages && !wait(bar(V_EMPTY + s), par)) { ok = false; break; }
        load(vmap, v_smem, bar(V_FULL + s));
        page = ahead;
      }
      if (!ok) break;
      on = false;
      if (!last) {                       // to the unit behind it, or to the part that waits
        if (j1 == u.tiles) {
          next_unit(u);
          col = u.first;
          on = u.first + kUnitCost < end;
        }
        if (!on && waits) {
          u = held;
          col = begin;
          on = last = true;
          waits = false;
        }
      }
    }
  } else if (warp == 1) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsLow));
    // ---- MMA issue: all lanes run the code, one issues the instructions; what all lanes agree on comes out of a shuffle, so that the compiler knows it too
    // (elect_one).  With `lane == 0` and plain registers this warp bounded the kernel: 2 x 512 tokens of 16500 keys of 32 heads of 128 took 283 us
    // instead of 243 (short runs; 960 and 1120 TFLOP/s), a prompt of 4096 tokens of heads of 64 142 instead of 130 ----
    constexpr uint32_t idesc_qk = instr_desc(kRows, kKeys, false);
    constexpr uint32_t idesc_pv = instr_desc(kRows, D, true);
    const uint32_t elected = elect_one();
    auto alike = [](uint32_t v) { return __shfl_sync(kFullMask, v, 0); };
    // the lower halves of the operands' descriptors; the upper ones are all alike
    const uint32_t q_desc = (uint32_t)smem_desc(q_smem, 16, 1024), k_desc = (uint32_t)smem_desc(k_smem, 16, 1024), v_desc = (uint32_t)smem_desc(v_smem, kBoxBytes, 1024);
    auto desc = [](uint32_t low) { return (uint64_t)low | (smem_desc(0, 0, 1024) & 0xffffffff00000000ull); };
    // One loop over the tiles of all segments, a round ahead with the scores: a unit's first scores follow the last product of the one before at
    // once, and there is one place for each product's code (what is unrolled further falls out of the instruction cache that the warp shares with
    // the softmax: with both tiles of rows and both stages unrolled a tile of keys took 3.3 us instead of 2.7).
    uint32_t p_phase = 0, o_phase = 0, o_used = 0, guarded = 0;   // phases of P_FULL, O_READ and V_OK, a bit for each; whether O_e has been used
    ok = take(0);
    int nj = segs[0].j0, nj1 = ok ? segs[0].j1 : 0, nne = segs[0].ne, nlimit = segs[0].limit;   // the tile whose scores come
    bool on = nj1 > 0;
    int j = 0, ne = 0, limit = 0;                                 // the tile whose values come: the one before; ne 0: none
    bool first = true, nfirst = true;
    for (fill = -1; (on || ne > 0) && ok; ++fill) {
      const int s = fill & (kStages - 1), ns = (fill + 1) & (kStages - 1);
      if (ne > 0) {
        if (!wait(bar(V_FULL + s), (fill / kStages) & 1)) { ok = false; break; }
        if (cut_tile(j, limit)) {
          if (!wait(bar(V_OK + s), (guarded >> s) & 1)) { ok = false; break; }
          guarded ^= 1u << s;
        }
      }
#pragma unroll 1
      for (int e = 0; e < 2; ++e) {
        const uint32_t s_at = alike(tmem + 128u * e), o_at = alike(tmem + 256u + (uint32_t)D * e);
        if (e < ne) {
          // O_e += P_e V once P_e is in tensor memory, on a segment's first tile once the last segment's O_e has been read; then at
          // once the next scores, which go where P_e lay
          if (!wait(bar((kHalfWeights ? P_HALF : P_FULL) + e), (p_phase >> e) & 1)) { ok = false; break; }
          if (first) {
            if ((o_used >> e) & 1) {
              if (!wait(bar(O_READ + e), (o_phase >> e) & 1)) { ok = false; break; }
              o_phase ^= 1u << e;
            }
            o_used |= 1u << e;
          }
          tc_fence_after();
          const uint32_t vd = alike(v_desc + s * (kTileBytes >> 4));
          constexpr int kFirst = kKeys / 16 / (kHalfWeights ? 2 : 1);
          if (elected) {
#pragma unroll
            for (int kk = 0; kk < kFirst; ++kk) mma_ts(o_at, s_at + kk * 8, desc(vd + kk * 128), idesc_pv, (!first || kk > 0) ? 1u : 0u, 1u);
          }
          __syncwarp();
          if constexpr (kHalfWeights) {
            if (!wait(bar(P_FULL + e), (p_phase >> e) & 1)) { ok = false; break; }
            tc_fence_after();
          }
          p_phase ^= 1u << e;
          if (elected) {
#pragma unroll
            for (int kk = kFirst; kk < kKeys / 16; ++kk) mma_ts(o_at, s_at + kk * 8, desc(vd + kk * 128), idesc_pv, 1u, 1u);
            tc_commit(bar(O_FULL + e), 1u);
            if (e == ne - 1) tc_commit(bar(V_EMPTY + s), 1u);
          }
          __syncwarp();
        }
        if (on && e < nne) {
          if (e == 0) {
            if (!wait(bar(K_FULL + ns), ((fill + 1) / kStages) & 1)) { ok = false; break; }
            if (nfirst && !wait(bar(Q_FULL), segments & 1)) { ok = false; break; }
            tc_fence_after();
          }
          const uint32_t qd = alike(q_desc + e * (kTileBytes >> 4)), kd = alike(k_desc + ns * (kTileBytes >> 4));
          if (elected) {
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {
              const uint32_t step = ((ks >> 2) * kBoxBytes + (ks & 3) * 32) / 16;
              mma_ss(s_at, desc(qd + step), desc(kd + step), idesc_qk, ks > 0, 1u);
            }
            tc_commit(bar(S_FULL + e), 1u);
            if (e == nne - 1) {
              tc_commit(bar(K_EMPTY + ns), 1u);
              if (nj + 1 == nj1) tc_commit(bar(Q_EMPTY), 1u);
            }
          }
          __syncwarp();
        }
      }
      // a round on
      j = nj;
      ne = on ? nne : 0;
      limit = nlimit;
      first = nfirst;
      nfirst = false;
      if (on && ++nj == nj1) {
        if (!take(++segments)) { ok = false; break; }
        const Segment& g = segs[segments % kSegments];
        nj1 = g.j1;
        on = nj1 > 0;
        nfirst = true;
        nj = g.j0;
        nne = g.ne;
        nlimit = g.limit;
      }
    }
  } else if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsLow));
    // ---- guards: a key's values a thread, tiles at the diagonal and the end only ----
    for (; ok; ++segments) {
      if (!take(segments)) { ok = false; break; }
      const Segment& g = segs[segments % kSegments];
      const int j1 = g.j1, limit = g.limit, len = g.len;
      if (j1 == 0) break;
      for (int j = g.j0; j < j1 && ok; ++j, ++fill) {
        const int s = fill % kStages;
        if (!wait(bar(V_FULL + s), (fill / kStages) & 1)) { ok = false; break; }
        if (!cut_tile(j, limit)) {
          if (lane == 0) mbar_arrive(bar(V_EMPTY + s));
          continue;
        }
        bool any = false;
#pragma unroll 1
        for (int r = max(limit + 1 - j * kKeys, 0) + (warp - 2) * 32 + lane; r < kKeys; r += 64) {   // (keys up to `limit` all rows see)
          const bool behind = j * kKeys + r >= len;
#pragma unroll 1
          for (int c = 0; c < kHalves * 8; ++c) {      // (short loops here and in the output: unrolled code comes from memory every time)
            const uint32_t at = v_smem + s * kTileBytes + (c >> 3) * kBoxBytes + r * 128 + (((c & 7) ^ (r & 7)) << 4);
            uint32_t w[4];
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
            bool write = behind;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              if (behind) w[x] = 0;
              if ((w[x] & 0x7f80u) == 0x7f80u) { w[x] &= 0xffff0000u; write = any = true; }
              if ((w[x] & 0x7f800000u) == 0x7f800000u) { w[x] &= 0xffffu; write = any = true; }
            }
            if (write) asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
          }
        }
        if (any) odd[segments % kSegments] = segments + 1;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(bar(V_OK + s));
          mbar_arrive(bar(V_EMPTY + s));
        }
      }
    }
  } else if (warp < 4 + kSoftmaxWarps) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsHigh));
    // ---- softmax: group e = tile e of the unit's rows, a thread a row ----
    const int q4 = warp & 3, e = (warp - 4) >> 2, r = q4 * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(q4 * 32) << 16;
    const uint32_t ts = t_s[e] + lane_addr, to = t_o[e] + lane_addr;
    constexpr float kLazy = 8.f;                   // log2 of how far the running maximum may outgrow m_ref
    const int token = r / p.R;                     // of the tile
    int g = 0, mine = 0;                           // tiles and segments of this group so far
    for (; ok; ++segments) {
      if (!take(segments)) { ok = false; break; }
      const Segment& s = segs[segments % kSegments];
      const int j0 = s.j0, j1 = s.j1;
      if (j1 == 0) break;
      if (e < s.ne) {
        const int limit0 = s.limit + e * cp.tile_tokens;
        const int limit = token < cp.tile_tokens ? min(limit0 + token, s.len - 1) : -1;   // last key this row may see
        float m_ref = -INFINITY, l_run = 0.f;
        for (int j = j0; j < j1 && ok; ++j, ++g) {
          if (!wait(bar(S_FULL + e), g & 1)) { ok = false; break; }
          tc_fence_after();
          uint32_t x[4][32];
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld32(ts + c * 32, x[c]);
          tc_wait_ld();
          if (__builtin_expect(cut_tile(j, limit0), 0)) {
            const int left = limit - j * kKeys;                    // last key of the tile that this row sees
#pragma unroll
            for (int c = 0; c < 4; ++c)
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (c * 32 + i > left) x[c][i] = 0xff800000u;      // -inf
          }
          float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 32; i += 2)
              mx4[(i >> 1) & 3] = fmax3(mx4[(i >> 1) & 3], __uint_as_float(x[c][i]), __uint_as_float(x[c][i + 1]));
          const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * p.scale_log2e;
          // the reference maximum moves (and this warp's rows of O_e are rescaled) only when some row needs it
          if (__any_sync(kFullMask, mx > m_ref + kLazy)) {
            const float m_new = fmaxf(m_ref, mx);
            const float alpha = m_new == -INFINITY ? 1.f : fast_exp2(m_ref - m_new);
            if (j > j0) {
              if (!wait(bar(O_FULL + e), (g - 1) & 1)) { ok = false; break; }
              tc_fence_after();
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
                uint32_t y[32];
                tmem_ld32(to + c * 32, y);
                tc_wait_ld();
                uint32_t lo[16], hi[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  lo[i] = __float_as_uint(__uint_as_float(y[i]) * alpha);
                  hi[i] = __float_as_uint(__uint_as_float(y[16 + i]) * alpha);
                }
                tmem_st16(to + c * 32, lo);
                tmem_st16(to + c * 32 + 16, hi);
              }
              l_run *= alpha;
            }
            m_ref = m_new;
          }
          const float mu = m_ref == -INFINITY ? 0.f : m_ref;
          const unsigned long long scale2 = f2_packf(p.scale_log2e, p.scale_log2e), nmu2 = f2_packf(-mu, -mu);
          unsigned long long ps2[4] = {0ull, 0ull, 0ull, 0ull};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            uint32_t pk[16];
            unsigned long long t2[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) t2[i] = f2_fma(f2_pack(x[c][2 * i], x[c][2 * i + 1]), scale2, nmu2);
            float pe[32];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float x0, x1;
              f2_unpack(t2[i], x0, x1);
              pe[2 * i] = fast_exp2(x0);
              pe[2 * i + 1] = fast_exp2(x1);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              ps2[i & 3] = f2_add(ps2[i & 3], f2_packf(pe[2 * i], pe[2 * i + 1]));
              pk[i] = pack_bf16x2(pe[2 * i], pe[2 * i + 1]);
            }
            tmem_st16(ts + c * 16, pk);                // P: 64 packed columns over the first 64 of S
            if (kHalfWeights && c == 1) {
              tc_wait_st();
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(bar(P_HALF + e));
            }
          }
          {
            float a0, a1, b0, b1;
            f2_unpack(f2_add(ps2[0], ps2[1]), a0, a1);
            f2_unpack(f2_add(ps2[2], ps2[3]), b0, b1);
            l_run += (a0 + a1) + (b0 + b1);
          }
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(P_FULL + e));
        }
        if (!ok) break;
        // the row's sums go to the output group, which has read the last segment's before it arrived on O_READ
        if (mine > 0 && !wait(bar(O_READ + e), (mine - 1) & 1)) { ok = false; break; }
        *reinterpret_cast<float2*>(stat + (e * kRows + r) * 2) = make_float2(l_run, m_ref);
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(L_FULL + e));
        ++mine;
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOut));
    // ---- output: a thread a row of one tile after the other.  No barrier among the four warps: each finds out for itself when a wait has run out, and the
    // others would stand at it for good ----
    const int q4 = warp & 3, r = q4 * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(q4 * 32) << 16;
    int g[2] = {0, 0}, mine[2] = {0, 0};
    const int over_r = (65535 + p.R) / p.R;        // x * over_r >> 16 is x / R for the rows of a tile
    for (; ok; ++segments) {
      if (!take(segments)) { ok = false; break; }
      const Segment& s = segs[segments % kSegments];
      const int j0 = s.j0, j1 = s.j1, ne = s.ne;
      if (j1 == 0) break;
      const bool whole = s.whole != 0;
      const long long row0 = a.starts ? s.row * a.o_st : s.b * a.o_sb;
      for (int e = 0; e < ne && ok; ++e) {
        if (!wait(bar(L_FULL + e), mine[e] & 1)) { ok = false; break; }
        const float2 lm = *reinterpret_cast<const float2*>(stat + (e * kRows + r) * 2);
        g[e] += j1 - j0;
        if (!wait(bar(O_FULL + e), (g[e] - 1) & 1)) { ok = false; break; }   // the segment's last product
        tc_fence_after();
        const int t0 = s.t0 + e * cp.tile_tokens, tokens = min(cp.tile_tokens, s.n - t0);   // tokens of the tile
        const bool taken = *reinterpret_cast<volatile int*>(odd + segments % kSegments) == segments + 1;
        const float inv = lm.x == 0.f ? 0.f : 1.f / lm.x;
        float* rec = chunk_part_of<D>(p, part, j0 == 0);
        const uint32_t to = t_o[e] + lane_addr;
        if (__builtin_expect(taken, 0)) {
          // values that the guards took out, for the rows that see them: from the cache, key by key, into O_e (a call with such values is lost anyway)
          const int upto = r < tokens * p.R ? min(min(s.limit + e * cp.tile_tokens + r / p.R, s.len - 1), j1 * kKeys - 1) : -1;
#pragma unroll 1
          for (int c = 0; c < D; c += 16) {
            uint32_t y[16];
            tmem_ld16(to + c, y);
            tc_wait_ld();
#pragma unroll 1
            for (int key = max(max(j0 * kKeys, s.limit + 1), 0); key <= upto; ++key) {
              const int page = __ldg(a.page_table + s.b * a.table_st + key / a.page_size);
              if (page < 0 || page >= a.pages) continue;
              const uint16_t* v = static_cast<const uint16_t*>(a.cache_v) + page * a.cache_sp + key % a.page_size * a.cache_st + s.h * D + c;
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const uint32_t w = __ldg(v + i);
                if ((w & 0x7f80u) == 0x7f80u) y[i] = __float_as_uint(__uint_as_float(y[i]) + __uint_as_float(w << 16));
              }
            }
            __syncwarp();
            tmem_st16(to + c, y);
            tc_wait_st();
          }
        }
        auto read = [&]() {                                   // O_e and the row's sums are in registers: they may take the next segment's
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(O_READ + e));
        };
        if (whole) {
          // 64 columns at a time through the warp's own staging rows: a thread holds one row, a store is to touch few
          uint8_t* stage = stage_all + q4 * (2 * kRows * kSPitch / 4);
          constexpr int kPitch = 128 + 16;
          static_assert(32 * kPitch <= 2 * kRows * kSPitch / 4, "staging rows of a warp");
          __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + row0 + (long long)(s.h * p.R) * a.o_sh + (lane & 7) * 8;
#pragma unroll 1
          for (int h = 0; h < kHalves; ++h) {
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t y[16];
              tmem_ld16(to + h * 64 + c * 16, y);
              tc_wait_ld();
              float f[8];
#pragma unroll
              for (int v = 0; v < 2; ++v) {
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(y[8 * v + i]) * inv;
                *reinterpret_cast<uint4*>(stage + lane * kPitch + c * 32 + v * 16) = pack8(f);
              }
            }
            if (h == kHalves - 1) read();
            __syncwarp();
#pragma unroll 1
            for (int i = 0; i < 8; ++i) {
              const int row = i * 4 + (lane >> 3), t = (q4 * 32 + row) * over_r >> 16;
              if (t < tokens)
                *reinterpret_cast<uint4*>(out + (t0 + t) * a.o_st + (q4 * 32 + row - t * p.R) * a.o_sh + h * 64) =
                    *reinterpret_cast<const uint4*>(stage + row * kPitch + (lane & 7) * 16);
            }
            __syncwarp();
          }
        } else {
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            uint32_t y[16];
            tmem_ld16(to + c * 16, y);
            tc_wait_ld();
            if (c == D / 16 - 1) read();
#pragma unroll
            for (int q = 0; q < 4; ++q)
              *reinterpret_cast<uint4*>(rec + ((long long)(c * 4 + q) * (2 * kRows) + e * kRows + r) * 4) = make_uint4(y[4 * q], y[4 * q + 1], y[4 * q + 2], y[4 * q + 3]);
          }
          rec[2 * kRows * D + e * kRows + r] = lm.y;
          rec[2 * kRows * (D + 1) + e * kRows + r] = lm.x;
        }
        ++mine[e];
      }
    }
  }
  if (!ok && lane == 0) atomicExch(a.status ? a.status : &g_wait_status, (int)L3CI_ERR_DEVICE_WAIT);
  if (cp.follows) pdl_wait();              // (the merge behind counts on both kernels)
  __syncwarp();
  tc_fence_before();
  // a wait ran out: the copies and the products still under way end before the shared and the tensor memory are given back (or their own waits run out too)
  if (__syncthreads_or(!ok) && (threadIdx.x == 0 || warp == 1)) {
    if (threadIdx.x == 0) {
      if (segments > 0 || fill > 0) (void)mbar_wait_bounded_one(bar(Q_FULL), segments & 1, cp.wait_ns);
      for (int f = max(fill - kStages, 0); f <= fill; ++f) {
        (void)mbar_wait_bounded_one(bar(K_FULL + f % kStages), (f / kStages) & 1, cp.wait_ns);
        (void)mbar_wait_bounded_one(bar(V_FULL + f % kStages), (f / kStages) & 1, cp.wait_ns);
      }
    } else if (elect_one()) {              // (the lane that issued the products, on a barrier that nobody has to do with any more)
      const uint32_t at = bar(SEG_EMPTY);
      asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(at) : "memory");
      mbar_init(at, 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      tc_commit(at, 1u);
      (void)mbar_wait_bounded_one(at, 0, cp.wait_ns);
    }
  }
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, kTmemCols);
}

// ---- host ----
size_t chunk_smem(int D, int B) {
  const size_t tile = (size_t)(D / 64) * 128 * 128;
  return 1024 + 6 * tile + 2 * kRows * 80 + (25 + 2 * kSegments) * 8 + (kSegments + 16) * 4 + 4 * kRows * 4 + kSegments * sizeof(Segment) + (size_t)(B + 1) * 4;
}

int chunk_parts(const PagedParams& p) {
  const int sms = sm_count() > 0 ? sm_count() : 148;
  const long long columns = paged_chunk_columns(&p.a);
  return (int)(columns < sms ? columns : sms);
}

int chunk_maps(const ChunkParams& cp, CUtensorMap* qmap, CUtensorMap* kmap, CUtensorMap* vmap) {
  auto enc = tensor_map_encoder();
  if (!enc) return fail(L3CI_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  const l3ci_paged_attention_args& a = cp.p.a;
  const cuuint64_t row = (cuuint64_t)a.D * 2;
  const cuuint32_t one[4] = {1u, 1u, 1u, 1u};
  {
    const long long T = a.starts ? a.rows : a.T, B = a.starts ? 1 : a.B;
    // (a dimension of extent 1 may carry any stride in the caller's view; a valid one then)
    const cuuint64_t dims[4] = {(cuuint64_t)a.D, (cuuint64_t)a.Hq, (cuuint64_t)T, (cuuint64_t)B};
    const cuuint64_t strides[3] = {a.Hq > 1 ? (cuuint64_t)a.q_sh * 2 : row, T > 1 ? (cuuint64_t)a.q_st * 2 : row, B > 1 ? (cuuint64_t)a.q_sb * 2 : row};
    const cuuint32_t box[4] = {64u, (cuuint32_t)cp.p.R, (cuuint32_t)cp.tile_tokens, 1u};
    const CUresult r = enc(qmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(a.q), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                           CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(L3CI_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", (int)r);
  }
  const cuuint64_t dims[4] = {(cuuint64_t)a.D, (cuuint64_t)a.page_size, (cuuint64_t)a.Hkv, (cuuint64_t)a.pages};
  const cuuint64_t strides[3] = {(cuuint64_t)a.cache_st * 2, row, a.pages > 1 ? (cuuint64_t)a.cache_sp * 2 : row};
  const cuuint32_t box[4] = {64u, (cuuint32_t)cp.box, 1u, 1u};
  for (int i = 0; i < 2; ++i) {
    const CUresult r = enc(i ? vmap : kmap, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(i ? a.cache_v : a.cache_k), dims, strides, box, one,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           a.D == 128 ? CU_TENSOR_MAP_L2_PROMOTION_L2_256B : CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(L3CI_ERR_CUDA, "cuTensorMapEncodeTiled failed with %d", (int)r);
  }
  return L3CI_OK;
}

template <int D>
int chunk_launch(const ChunkParams& cp, cudaStream_t stream) {
  CUtensorMap qmap, kmap, vmap;
  if (int st = chunk_maps(cp, &qmap, &kmap, &vmap)) return st;
  static bool configured[64] = {false};
  int dev = 0;
  L3CI_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    L3CI_CUDA_TRY(cudaFuncSetAttribute(paged_chunk_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)chunk_smem(D, kPagedMaxSeqs)));
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  L3CI_LAUNCH("paged_chunk_kernel", paged_chunk_kernel<D>, dim3((unsigned)cp.p.max_parts), dim3(kThreads), chunk_smem(D, cp.p.a.B), stream, qmap, kmap, vmap, cp);
  return L3CI_OK;
}

}  // namespace

// (every block of every sequence a unit over all the keys that the table can hold)
long long paged_chunk_columns(const l3ci_paged_attention_args* a) {
  const long long rows = a->starts ? a->rows : (long long)a->B * a->T, block = 2 * (kRows / (a->Hq / a->Hkv));
  const long long seqs = a->B < kPagedMaxSeqs ? a->B : kPagedMaxSeqs;
  return (rows / block + seqs) * a->Hkv * (kTileCost * (((long long)a->max_pages * a->page_size + kKeys - 1) / kKeys + 1) + unit_cost(a->D));
}

size_t paged_chunks_scratch_bytes(const PagedParams& p) {
  const int parts = chunk_parts(p);
  return (size_t)parts * (sizeof(ChunkCut) + 2 * 4 * (size_t)(p.a.D == 64 ? chunk_part_floats(64) : chunk_part_floats(128)));
}

int paged_chunks_launch(const PagedParams& params, void* scratch, bool follows, cudaStream_t stream, ChunkParams* launched) {
  ChunkParams& cp = *launched;
  cp.p = params;
  cp.p.max_parts = chunk_parts(params);
  cp.cuts = static_cast<ChunkCut*>(scratch);
  cp.p.records = reinterpret_cast<float*>(cp.cuts + cp.p.max_parts);
  cp.tile_tokens = kRows / params.R;
  const int low = params.a.page_size & -params.a.page_size;    // tokens that lie together in every page: a power of two
  cp.box = low < kKeys ? low : kKeys;
  cp.follows = follows;
  const unsigned long long limit = device_wait_limit_ns(kWaitLimitNs);
  cp.wait_ns = limit < kWaitLimitLoNs ? (uint32_t)limit : kWaitLimitLoNs;
  return params.a.D == 64 ? chunk_launch<64>(cp, stream) : chunk_launch<128>(cp, stream);
}

}  // namespace l3ci

extern "C" int l3ci_paged_attention_poll(l3ci_stream_t stream_) {
  using namespace l3ci;
  clear_error();
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(stream_);
  void* word = nullptr;
  int status = 0;
  L3CI_CUDA_TRY(cudaGetSymbolAddress(&word, g_wait_status));
  L3CI_CUDA_TRY(cudaMemcpyAsync(&status, word, sizeof(int), cudaMemcpyDeviceToHost, stream));
  L3CI_CUDA_TRY(cudaStreamSynchronize(stream));
  if (status == 0) return L3CI_OK;
  L3CI_CUDA_TRY(cudaMemsetAsync(word, 0, sizeof(int), stream));
  L3CI_CUDA_TRY(cudaStreamSynchronize(stream));
  return fail(status, "paged_attention: a bounded wait ran out in an earlier launch");
}

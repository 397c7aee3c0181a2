// New tokens into a paged cache (include/l3ci_b200.h, l3ci_rot_embed_paged_kv_cache): one pass over the rows q|k|v of a fused projection
// norms every query and key head (optional), rotates them, and writes queries to their own rows, keys and values to the tokens' pages.
//
// Bound by the bytes of the rows, read once and written once.  One CTA per token: a thread owns one 16-byte vector of a head at a
// time and sits at the same place of all its heads, so that it loads the rotary table and the norms' weights once; a head's sum of
// squares is a shuffle over the lanes that hold it.  The row itself does not depend on where the token goes: its loads are asked for
// before the chain starts -> positions -> page table, which is most of what a decode step's call takes.  With norms the arithmetic is near the
// bytes' time as well (a warp has some 80 instructions a vector): the norms' weights go into the rotation, two floats an instruction.
// Measured on a B200: 24 sequences, 20 with chunks of up to 500 tokens, 64 + 2 x 8 heads of 128 with norms, 294 MB: 53.8 us, 5.5 TB/s (62.7 before
// those two); a prompt of 2001 tokens, 24 + 2 x 8 heads of 64 with norms, 20 MB mostly in L2: 5.2 us, one wave of CTAs; 64 single tokens of 32 + 2 x 8
// heads of 128: 2.4 us in a graph, 6.2 in calls from the host, whose time that is.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "bf16x8.cuh"
#include "host_common.h"
#include "ptx_sm100.cuh"
#include "rotate.cuh"
#include "tcgen05.cuh"
#include "warp_reduce.cuh"

namespace l3ci {
namespace {

constexpr int kBatch = 4;   // 16-byte loads of queries a thread has in flight

typedef unsigned long long f2;   // two floats

// What a vector's four pairs are multiplied with: (x, y) -> x (c w_x, s w_x) + y (-s w_y, c w_y), the norm's weights in the rotation.
struct Turn {
  f2 x[4], y[4];
};
__device__ __forceinline__ Turn turn_of(const float4& f0, const float4& f1, const uint4& weights) {
  float w[8];
  unpack8(weights, w);
  const float c[4] = {f0.x, f0.z, f1.x, f1.z}, s[4] = {f0.y, f0.w, f1.y, f1.w};
  Turn t;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    t.x[i] = f2_packf(c[i] * w[2 * i], s[i] * w[2 * i]);
    t.y[i] = f2_packf(-s[i] * w[2 * i + 1], c[i] * w[2 * i + 1]);
  }
  return t;
}
// A head's vector normed and rotated; LANES lanes hold the head.
template <int LANES>
__device__ __forceinline__ uint4 norm_rotate8(const uint4& v, const Turn& t, float over_d, float eps) {
  float a[8];
  unpack8(v, a);
  f2 ss = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f2 p = f2_packf(a[2 * i], a[2 * i + 1]);
    ss = f2_fma(p, p, ss);
  }
  float s0, s1;
  f2_unpack(ss, s0, s1);
  const float rs = rsqrtf(fmaf(group_sum<LANES>(s0 + s1), over_d, eps));
  const f2 rs2 = f2_packf(rs, rs);
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const f2 turned = f2_fma(f2_packf(a[2 * i], a[2 * i]), t.x[i], f2_mul(f2_packf(a[2 * i + 1], a[2 * i + 1]), t.y[i]));
    float x, y;
    f2_unpack(f2_mul(turned, rs2), x, y);
    o[i] = pack_bf16x2(x, y);
  }
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// LANES: lanes that hold a head, a power of two of at least D / 8 (those beyond it have nothing).
template <int LANES, bool NORM, int kBlock>
__global__ void __launch_bounds__(kBlock, (NORM ? 7 : 9) * 128 / kBlock)
rot_embed_paged_kv_cache_kernel(const l3ci_paged_rope_args p) {
  __shared__ int found;
  if (threadIdx.x == 0) found = -1;
  pdl_begin();
  const long long row = blockIdx.x;
  int b = p.starts ? 0 : (int)(row / p.T);
  long long t = p.starts ? 0 : row % p.T;
  const int vecs = p.D / kVecElems, vec = threadIdx.x % LANES, head0 = threadIdx.x / LANES;
  constexpr int kHeads = kBlock / LANES;                       // heads the CTA takes at a time
  const bool mine = vec < vecs;
  const __nv_bfloat16* in = static_cast<const __nv_bfloat16*>(p.qkv) + (p.starts ? row * p.qkv_st : b * p.qkv_sb + t * p.qkv_st) + vec * kVecElems;
  const __nv_bfloat16 *in_k = in + p.Hq * p.D, *in_v = in_k + p.Hkv * p.D;
  auto load = [&](const __nv_bfloat16* from, int h, int heads) { return mine && h < heads ? ld_stream16(from + h * p.D) : make_uint4(0, 0, 0, 0); };
  uint4 q[kBatch], k, v;
#pragma unroll
  for (int u = 0; u < kBatch; ++u) q[u] = load(in, head0 + u * kHeads, p.Hq);
  k = load(in_k, head0, p.Hkv);
  v = load(in_v, head0, p.Hkv);
  uint4 wq = make_uint4(0, 0, 0, 0), wk = wq;
  if (NORM && mine) {
    wq = __ldg(static_cast<const uint4*>(p.q_norm) + vec);
    wk = __ldg(static_cast<const uint4*>(p.k_norm) + vec);
  }
  if (p.starts) {
    __syncthreads();                                           // (found is set)
    for (int i = threadIdx.x; i < p.B; i += kBlock)
      if (__ldg(p.starts + i) <= row && row < __ldg(p.starts + i + 1)) found = i;
    __syncthreads();
    b = found;
    if (b < 0) return;                                         // a row of no sequence
    t = row - __ldg(p.starts + b);
  }
  const long long pos = (long long)__ldg(p.positions + b) + t;
  if (pos < 0 || pos >= p.freq_rows) return;
  const long long slot = pos / p.page_size;
  if (slot >= p.max_pages) return;
  const int page = __ldg(p.page_table + b * p.table_st + slot);
  if (page < 0 || page >= p.pages) return;
  float4 f0 = make_float4(0, 0, 0, 0), f1 = f0;
  if (mine) {
    const float* f = p.freq_table + pos * p.D + vec * kVecElems;
    f0 = __ldg(reinterpret_cast<const float4*>(f));
    f1 = __ldg(reinterpret_cast<const float4*>(f) + 1);
  }
  const float over_d = 1.f / (float)p.D;
  Turn turn;
  if (NORM) turn = turn_of(f0, f1, wq);
  auto turned = [&](const uint4& x) {
    if constexpr (NORM) return norm_rotate8<LANES>(x, turn, over_d, p.eps);
    else return rotate8(x, f0, f1);
  };
  __nv_bfloat16* qo = static_cast<__nv_bfloat16*>(p.q_out) + row * p.q_st + vec * kVecElems;
  const long long at = page * p.cache_sp + (pos - slot * p.page_size) * p.cache_st + vec * kVecElems;
  __nv_bfloat16* ko = static_cast<__nv_bfloat16*>(p.cache_k) + at;
  __nv_bfloat16* vo = static_cast<__nv_bfloat16*>(p.cache_v) + at;
  // (all lanes of a warp take every round: the shuffles of a norm want them)
  for (int h0 = 0; h0 < p.Hq; h0 += kHeads * kBatch) {
    if (h0 > 0)
#pragma unroll
      for (int u = 0; u < kBatch; ++u) q[u] = load(in, h0 + head0 + u * kHeads, p.Hq);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int h = h0 + head0 + u * kHeads;
      const uint4 r = turned(q[u]);
      if (mine && h < p.Hq) st_stream16(qo + h * p.D, r);
    }
  }
  if (NORM) turn = turn_of(f0, f1, wk);
  // (the cache rows are read again by the attention of the same step: plain stores)
  for (int h0 = 0; h0 < p.Hkv; h0 += kHeads) {
    const int h = h0 + head0;
    if (h0 > 0) {
      k = load(in_k, h, p.Hkv);
      v = load(in_v, h, p.Hkv);
    }
    const uint4 r = turned(k);
    if (mine && h < p.Hkv) {
      *reinterpret_cast<uint4*>(ko + h * p.D) = r;
      *reinterpret_cast<uint4*>(vo + h * p.D) = v;
    }
  }
}

}  // namespace
}  // namespace l3ci

extern "C" int l3ci_rot_embed_paged_kv_cache(const l3ci_paged_rope_args* a) {
  using namespace l3ci;
  clear_error();
  if (!a) return fail(L3CI_ERR_INVALID, "rot_embed_paged_kv_cache: null arguments");
  if (a->B < 0 || a->Hq <= 0 || a->Hkv <= 0 || a->D <= 0 || a->page_size <= 0 || a->max_pages < 0 || a->pages < 0 || a->freq_rows < 0 ||
      (a->starts ? a->rows < 0 : a->T < 0))
    return fail(L3CI_ERR_INVALID, "rot_embed_paged_kv_cache: B=%d T=%d rows=%lld heads %d, %d of %d, pages of %d", a->B, a->T, (long long)a->rows, a->Hq,
                a->Hkv, a->D, a->page_size);
  const long long rows = a->starts ? a->rows : (long long)a->B * a->T;
  if (rows == 0 || a->B == 0) return L3CI_OK;
  if (!a->qkv || !a->freq_table || !a->q_out || !a->cache_k || !a->cache_v || !a->page_table || !a->positions || !a->q_norm != !a->k_norm)
    return fail(L3CI_ERR_INVALID, "rot_embed_paged_kv_cache: null pointer");
  if (a->D % kVecElems || a->D > 256)
    return fail(L3CI_ERR_UNSUPPORTED, "rot_embed_paged_kv_cache: head size %d is not a multiple of 8 up to 256", a->D);
  if (!aligned16(a->qkv) || !aligned16(a->freq_table) || !aligned16(a->q_out) || !aligned16(a->cache_k) || !aligned16(a->cache_v) || !aligned16(a->q_norm) ||
      !aligned16(a->k_norm) || a->qkv_sb % kVecElems || a->qkv_st % kVecElems || a->q_st % kVecElems || a->cache_sp % kVecElems || a->cache_st % kVecElems)
    return fail(L3CI_ERR_ALIGNMENT, "rot_embed_paged_kv_cache: rows must start on 16 bytes");
  if (rows > 0x7fffffffLL || ((long long)a->Hq + 2LL * a->Hkv) * a->D > 0x7fffffffLL)
    return fail(L3CI_ERR_INVALID, "rot_embed_paged_kv_cache: tensor too large");
  if (rows > 1 && a->q_st < (long long)a->Hq * a->D) return fail(L3CI_ERR_INVALID, "rot_embed_paged_kv_cache: rows of the queries overlap");
  cudaStream_t stream = reinterpret_cast<cudaStream_t>(a->stream);
  auto go = [&](auto lanes, auto norm) -> int {
    constexpr int kLanes = decltype(lanes)::value;
    constexpr bool kNorm = decltype(norm)::value;
    auto in = [&](auto threads) -> int {
      constexpr int kBlock = decltype(threads)::value;
      L3CI_LAUNCH("rot_embed_paged_kv_cache_kernel", (rot_embed_paged_kv_cache_kernel<kLanes, kNorm, kBlock>), dim3((unsigned)rows), dim3(kBlock), 0, stream, *a);
      return L3CI_OK;
    };
    // The smallest CTA that asks for its whole row before it waits.  (Threads without a vector keep others off the SM: 2001 tokens of 24 + 2 x 8 heads of 64
    // with norms take 8.2 us by CTAs of 128, 5.2 by 64, 6.4 by 32; 6000 of 16 + 2 heads of 64 19.6, 11.6, 8.2; of 32 + 2 x 8 heads of 128 30.3, 29.2, 30.8,
    // a single token of these 3.0, 4.2, 6.5.)
    auto holds = [&](int threads) { return a->Hq * kLanes <= threads * kBatch && a->Hkv * kLanes <= threads; };
    if (holds(32)) return in(std::integral_constant<int, 32>{});
    if (holds(64)) return in(std::integral_constant<int, 64>{});
    // (where every CTA has an SM of its own: 64 tokens of 64 + 2 x 8 heads of 128 2.3 us instead of 3.0; 500 of them with norms 6.6 and 5.5)
    if (!holds(128) && holds(256) && rows <= sm_count()) return in(std::integral_constant<int, 256>{});
    return in(std::integral_constant<int, 128>{});
  };
  auto with = [&](auto lanes) { return a->q_norm ? go(lanes, std::true_type{}) : go(lanes, std::false_type{}); };
  if (a->D <= 64) return with(std::integral_constant<int, 8>{});
  if (a->D <= 128) return with(std::integral_constant<int, 16>{});
  return with(std::integral_constant<int, 32>{});
}

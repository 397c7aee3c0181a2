// What the kernels of attention over a paged cache share: the call, the sequences they take, and how work is dealt.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "host_common.h"

namespace l3ci {

// Sequences of one launch (more go in several): their prefix sums lie in shared memory.
constexpr int kPagedMaxSeqs = 2048;

struct PagedParams {
  l3ci_paged_attention_args a;
  int R;               // query heads of a KV head
  int cap;             // keys that a row of the table can hold
  int min_rows, max_rows;   // query rows (tokens x R) of the sequences that the launch takes
  int max_parts;       // CTAs or warps that work is dealt to
  float scale_log2e;
  float* records;      // scratch: partial results
};

struct PagedSeq {
  int n, len;          // new tokens, keys
};

#if defined(__CUDACC__)
// New tokens and keys of sequence b; no tokens where `starts` does not name rows of the call.
__device__ __forceinline__ PagedSeq paged_seq(const PagedParams& p, int b) {
  PagedSeq s;
  s.len = min(max(__ldg(p.a.seq_lens + b), 0), p.cap);
  s.n = p.a.T;
  if (p.a.starts) {
    const int r0 = __ldg(p.a.starts + b), r1 = __ldg(p.a.starts + b + 1);
    s.n = r0 >= 0 && r1 >= r0 && r1 <= p.a.rows ? r1 - r0 : 0;
  }
  const long long rows = (long long)s.n * p.R;
  if (rows < p.min_rows || rows > p.max_rows) s.n = 0;
  return s;
}
// Elements before the first new token of sequence b in a tensor of these strides.
__device__ __forceinline__ long long paged_row0(const PagedParams& p, int b, long long sb, long long st) {
  return p.a.starts ? __ldg(p.a.starts + b) * st : b * sb;
}
#endif

// Chunks of many rows (paged_attention_tc.cu): a unit is two tiles of 128 query rows of a KV head.
constexpr int kChunkRows = 128;
// The unit that part g of the deal begins in the middle of, written by its CTA for the merge; parts 0: none, or its first cut is another part's.
struct ChunkCut {
  int b, h, m, first, parts;
  int pad[3];
};
struct ChunkParams {
  PagedParams p;
  ChunkCut* cuts;
  int tile_tokens;   // tokens of a tile of query rows: 128 / R
  int box;           // tokens of a copy
  int follows;       // launched behind paged_rows_kernel of the same call, which has waited for the kernels before
  uint32_t wait_ns;  // bound of every wait
};
// Floats of a part: o[D / 4][256 rows][4], m[256], l[256].
constexpr long long chunk_part_floats(int D) { return 2 * kChunkRows * (D + 2); }
#if defined(__CUDACC__)
template <int D>
__device__ __forceinline__ float* chunk_part_of(const PagedParams& p, int part, bool begins) {
  return p.records + (2 * part + (begins ? 1 : 0)) * chunk_part_floats(D);
}
#endif

long long paged_chunk_columns(const l3ci_paged_attention_args* a);   // of the deal, at most
size_t paged_chunks_scratch_bytes(const PagedParams& p);
int paged_chunks_launch(const PagedParams& p, void* scratch, bool follows, cudaStream_t stream, ChunkParams* launched);

}  // namespace l3ci

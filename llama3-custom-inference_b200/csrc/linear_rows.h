// The product of few rows (linear_rows.cu) as other files of the library see it.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

#include "host_common.h"

namespace l3ci {

// Low-rank parts beside a product of few rows: out[t, :] += z[t, :] b[index[t]]^T, z fp32 [rows, rank], b bf16 [adapters, N, rank]; tokens whose
// index lies outside [0, adapters) have none.
struct AdapterRows {
  const float* z;
  const int32_t* index;
  const __nv_bfloat16* b;
  int rank, adapters;
};
// l3ci_linear of any number of rows (no activation, bf16) with these parts, one rounding.  The kernel ahead of it in the stream is to have
// waited for its own predecessors before it lets this one start, and to leave z, index, x and w complete.
int adapter_rows_launch(const l3ci_linear_args* a, const AdapterRows& low);

}  // namespace l3ci

// The product of many rows (linear_many.cu) as the others of the library see it.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

#include "host_common.h"

namespace l3ci {

// The device word where its waits that ran out are recorded (of the current device); null without a device.
int* linear_many_wait_status();

// Low-rank parts beside a product of many rows, as AdapterRows (linear_rows.h) beside one of few, and for every 256 rows a list of kAdapterList
// words: the number of adapters among them, then these.
constexpr int kAdapterTile = 256, kAdapterList = 1 + kAdapterTile;
struct AdapterMany {
  const float* z;
  const int32_t* index;
  const __nv_bfloat16* b;
  const int* lists;
  int rank, adapters;
};
// l3ci_linear_many (one group, no activation) with these parts, one rounding.
int adapter_many_launch(const l3ci_linear_args* a, const AdapterMany& low);

}  // namespace l3ci

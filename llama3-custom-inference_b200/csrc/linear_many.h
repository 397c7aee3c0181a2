// The product of many rows (linear_many.cu) as the others of the library see it.
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

#include "host_common.h"

namespace l3ci {

// The device word where its waits that ran out are recorded (of the current device); null without a device.
int* linear_many_wait_status();

// Low-rank parts beside a product of many rows, as AdapterRows (linear_rows.h) beside one of few, and for every 256 rows a list of kAdapterList words, on 16
// bytes: the number of adapters among them, then, from kAdapterHead on, an entry of kAdapterEntry words for each: its number at 0, and from 4 on a bit
// for each of the 256 rows that is NOT its own.  z of rows without an adapter may hold anything.
constexpr int kAdapterTile = 256, kAdapterHead = 4, kAdapterEntry = 12, kAdapterList = kAdapterHead + kAdapterTile * kAdapterEntry;
struct AdapterMany {
  const float* z;
  const __nv_bfloat16* b;
  const int* lists;
  int rank, adapters;
  int* status;         // where a wait that ran out is recorded; null: the library's word
};
// l3ci_linear_many (one group, no activation) with these parts, one rounding.
int adapter_many_launch(const l3ci_linear_args* a, const AdapterMany& low);

}  // namespace l3ci

// Rotation of interleaved pairs of bf16 vectors, shared by the rotary kernels of dense and paged caches.
#pragma once

#include "bf16x8.cuh"

namespace l3ci {

// One rotation, rounded exactly as the reference's compiled kernel rounds it: nvcc contracts each of
// `x*c - y*s` and `x*s + y*c` (custom_kernels/custom_kernels.cu:408,410) into a rounded product of the second
// term and a fused multiply-add of the first.  Written with explicit intrinsics so that the form does not depend
// on a file's compiler flags; outputs are bit-identical to the reference kernel's on the same inputs.
__device__ __forceinline__ void rotate_pair(float x, float y, float c, float s, float& xo, float& yo) {
  xo = __fmaf_rn(x, c, -__fmul_rn(y, s));
  yo = __fmaf_rn(x, s, __fmul_rn(y, c));
}

// Rotates the 8 bf16 of `v` with the table entries (f0, f1) = (c0,s0,c1,s1 | c2,s2,c3,s3).
__device__ __forceinline__ uint4 rotate8(const uint4& v, const float4& f0, const float4& f1) {
  float a[8], r[8];
  unpack8(v, a);
  rotate_pair(a[0], a[1], f0.x, f0.y, r[0], r[1]);
  rotate_pair(a[2], a[3], f0.z, f0.w, r[2], r[3]);
  rotate_pair(a[4], a[5], f1.x, f1.y, r[4], r[5]);
  rotate_pair(a[6], a[7], f1.z, f1.w, r[6], r[7]);
  return pack8(r);
}
__device__ __forceinline__ uint4 rotate8(const uint4& v, const float* __restrict__ freq8) {
  return rotate8(v, __ldg(reinterpret_cast<const float4*>(freq8)), __ldg(reinterpret_cast<const float4*>(freq8) + 1));
}

}  // namespace l3ci

// The transformer operators' host side: argument checks and launchers.
//
// The checks are host rules over the C structs of arthip.h (no GPU needed): each
// returns an empty text, or what is wrong. The launchers take checked arguments.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "../../include/arthip.h"

namespace arthip {

// One rotary frequency as the kernel reads it. Turns (radians / 2 pi) in fp64: the
// product with a 31-bit position is then reduced to its fraction without losing
// phase, at the cost of four fp64 operations a frequency and token.
struct RopeFreq {
  double turns;
  int32_t axis;
  int32_t pad;
};
static_assert(sizeof(RopeFreq) == 16, "the packed size is part of the C ABI");

std::string check_rope(const arthip_rope_args& a);
std::string check_attention(const arthip_attention_args& a);
std::string check_attention_shape(const arthip_attention_args& a);  // what attention_plan() relies on
std::string check_norm(const arthip_norm_args& a);

hipError_t launch_rope(const arthip_rope_args& a, hipStream_t s);
hipError_t launch_norm(const arthip_norm_args& a, hipStream_t s);
hipError_t launch_attention(const arthip_attention_args& a, hipStream_t s);

// Launches a grid of any size: launch(first, count) for runs of workgroups whose threads
// number fewer than 2^32, which is as many as HIP takes along a dimension.
template <class F>
hipError_t launch_parts(int64_t blocks, int threads, F launch) {
  const int64_t most = ((int64_t{1} << 32) - 1) / threads;
  for (int64_t first = 0; first < blocks; first += most) {
    const hipError_t e = launch(first, static_cast<unsigned>(std::min(most, blocks - first)));
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// How attention divides its work (attention.hip); of arguments whose shape is checked.
struct AttnPlan {
  int splits;         // ranges of the keys, each its own workgroup; joined by a second kernel
  int range;          // tiles of each
  size_t workspace;   // bytes
};
AttnPlan attention_plan(const arthip_attention_args& a);

}  // namespace arthip

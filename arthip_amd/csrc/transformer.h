// The transformer operators' host side: argument checks and launchers.
//
// The checks are host rules over the C structs of arthip.h (no GPU needed): each
// returns an empty text, or what is wrong. The launchers take checked arguments.
#pragma once

#include <hip/hip_runtime.h>

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

// How attention divides its work (attention.hip); of arguments whose shape is checked.
struct AttnPlan {
  int splits;         // ranges of the keys, each its own workgroup; joined by a second kernel
  int range;          // tiles of each
  size_t workspace;   // bytes
};
AttnPlan attention_plan(const arthip_attention_args& a);

}  // namespace arthip

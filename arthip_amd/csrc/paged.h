// The paged cache's host side: argument checks and launchers.
//
// The checks are host rules over the C structs of arthip.h (no GPU needed): each
// returns an empty text, or what is wrong. The launchers take checked arguments.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "../../include/arthip.h"

namespace arthip {

std::string check_cache_write(const arthip_cache_write_args& a);
std::string check_paged_attention(const arthip_paged_attention_args& a);
std::string check_paged_attention_shape(const arthip_paged_attention_args& a);  // what the plan relies on
std::string check_key_weights(const arthip_key_weights_args& a);
std::string check_key_weights_shape(const arthip_key_weights_args& a);
std::string check_cache_evict(const arthip_cache_evict_args& a);

hipError_t launch_cache_write(const arthip_cache_write_args& a, hipStream_t s);
hipError_t launch_paged_attention(const arthip_paged_attention_args& a, hipStream_t s);
hipError_t launch_key_weights(const arthip_key_weights_args& a, hipStream_t s);
hipError_t launch_cache_evict(const arthip_cache_evict_args& a, hipStream_t s);

// How paged attention divides its work (paged_attention.hip); of arguments whose shape is checked.
struct PagedPlan {
  bool one_wave;     // 32 rows a workgroup instead of 128
  int tile_tokens;   // new tokens of a row tile, with all heads of a key head
  int ranges;        // workgroups, each a range of the key tiles of all row tiles
  bool counted;      // a kernel of its own counts the tiles before each sequence
  size_t sums, stats, pieces, before;  // bytes of the workspace's parts, in this order
  size_t workspace() const { return sums + stats + pieces + before; }
};
PagedPlan paged_plan(const arthip_paged_attention_args& a);

// How the key weights are divided (key_weights.hip); of arguments whose shape is checked.
struct KeyWeightsPlan {
  int tiles;    // workgroups along the slots
  int splits;   // and along the rows, whose sums a second kernel joins
  int stream;   // few rows: slots of a workgroup (of one wave); 0: many
  size_t workspace;
};
KeyWeightsPlan key_weights_plan(const arthip_key_weights_args& a);

}  // namespace arthip

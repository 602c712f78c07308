// Device helpers of the paged cache: a sequence's rows and slots, a slot's place.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/arthip.h"
#include "wino_dev.h"

namespace arthip {

// A sequence: its new tokens' first row, their number, and its slots in use.
struct Sequence {
  int first, tokens, len;
  __device__ __forceinline__ int start() const { return len - tokens; }  // of the new tokens; may be negative
};

__device__ __forceinline__ int slots_of(const arthip_pages& p, int b) {
  return min(max(p.kv_len[b], 0), p.max_pages * p.page_size);
}

__device__ __forceinline__ Sequence sequence_of(const arthip_pages& p, int b) {
  Sequence s;
  s.len = slots_of(p, b);
  s.first = b;
  s.tokens = 1;
  if (p.q_offsets != nullptr) {
    s.first = min(max(p.q_offsets[b], 0), p.tokens);
    s.tokens = min(max(p.q_offsets[b + 1], s.first), p.tokens) - s.first;
  }
  return s;
}

// Element offset of a slot's row (head 0) in a pool of these strides (multiples of 8); -1 where its
// page is outside the pool. The slot is below max_pages * page_size.
__device__ __forceinline__ int64_t row_of(const arthip_pages& p, FastDiv by_page, const int32_t* pages, int slot,
                                          const int64_t* stride) {
  const int at = (int)fdiv((uint32_t)slot, by_page);
  const int page = pages[at];
  if ((uint32_t)page >= (uint32_t)p.pool_pages) return -1;
  return page * stride[0] + (slot - at * p.page_size) * stride[1];
}

}  // namespace arthip

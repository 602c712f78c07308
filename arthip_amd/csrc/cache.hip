// A paged cache's rows: new tokens into their slots (arthip_cache_write), and the
// eviction of the slots with little weight (arthip_cache_evict).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "launch.h"
#include "paged.h"
#include "paged_dev.h"
#include "token_dev.h"
#include "transformer.h"

namespace arthip {

namespace {

// -- writing ------------------------------------------------------------------------------

struct WriteArgs {
  arthip_cache_write_args c;
  int group;   // tokens of a workgroup
  int chunks;  // 16-byte chunks of a token's keys
  int head_chunks;
  FastDiv by_chunks, by_head_chunks, by_page;
};

constexpr int kOffsets = 1024;  // of the sequences that a workgroup keeps in LDS

// A thread moves 16 bytes of a token's keys and of its values. The token's sequence is found by
// halving among the offsets, which lie in LDS for up to 1023 sequences.
__global__ void __launch_bounds__(256) cache_write(WriteArgs a, int64_t first_block) {
  __shared__ int offsets[kOffsets];
  const arthip_pages& p = a.c.p;
  const bool near = p.q_offsets != nullptr && p.batch < kOffsets;
  if (near) {
    for (int i = threadIdx.x; i <= p.batch; i += 256) offsets[i] = p.q_offsets[i];
    lds_sync();
  }
  const int64_t t0 = (first_block + blockIdx.x) * a.group;
  const int tokens = (int)min((int64_t)a.group, p.tokens - t0);
  for (int i = threadIdx.x; i < tokens * a.chunks; i += 256) {
    const int of = (int)fdiv((uint32_t)i, a.by_chunks), chunk = i - of * a.chunks;
    const int token = (int)t0 + of;
    const int head = (int)fdiv((uint32_t)chunk, a.by_head_chunks), part = chunk - head * a.head_chunks;
    const u4 k = *reinterpret_cast<const u4*>(static_cast<const uint16_t*>(a.c.k) + token * a.c.k_stride[0] +
                                              head * a.c.k_stride[1] + part * 8);
    const u4 v = *reinterpret_cast<const u4*>(static_cast<const uint16_t*>(a.c.v) + token * a.c.v_stride[0] +
                                              head * a.c.v_stride[1] + part * 8);
    // The last sequence that begins at or before the token, if the token is one of its own.
    int b = token;
    if (p.q_offsets != nullptr) {
      int lo = 0, hi = p.batch;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        ((near ? offsets[mid] : p.q_offsets[mid]) <= token ? lo : hi) = mid;
      }
      b = lo;
    }
    const Sequence s = sequence_of(p, b);
    const int index = token - s.first, slot = s.start() + index;
    if (index < 0 || index >= s.tokens || slot < 0) continue;
    const int32_t* const pages = p.pages + b * p.pages_stride;
    if (a.c.positions != nullptr && part == 0 && slot < a.c.slots)
      a.c.positions[b * a.c.positions_stride[0] + head * a.c.positions_stride[1] + slot] = a.c.token_positions[token];
    const int64_t k_row = row_of(p, a.by_page, pages, slot, a.c.k_cache_stride);
    if (k_row == -1) continue;
    const int64_t v_row = row_of(p, a.by_page, pages, slot, a.c.v_cache_stride);
    *reinterpret_cast<u4*>(static_cast<uint16_t*>(a.c.k_cache) + k_row + head * a.c.k_cache_stride[2] + part * 8) = k;
    *reinterpret_cast<u4*>(static_cast<uint16_t*>(a.c.v_cache) + v_row + head * a.c.v_cache_stride[2] + part * 8) = v;
  }
}

// -- eviction -----------------------------------------------------------------------------

struct EvictArgs {
  arthip_cache_evict_args c;
  int head_chunks;
  FastDiv by_page, by_heads, by_head_chunks;
};

constexpr int kThreads = 1024;
constexpr int kMoves = 4096;    // slots listed in LDS at once
constexpr int kMovesHere = 256;  // up to this many the selecting workgroup moves the rows itself

// A weight as a number whose order is the weights': NaN is 0, less than -inf.
__device__ __forceinline__ uint32_t ordered(float w) {
  const uint32_t u = __builtin_bit_cast(uint32_t, w + 0.0f);  // -0 becomes 0
  return w != w ? 0u : u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Sum of x over the lanes up to this one, inside the vector unit: rows of 16, then across them.
__device__ __forceinline__ uint32_t up_to(uint32_t x) {
  auto add = [&](auto control, auto rows) __attribute__((always_inline)) {
    x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(control)::value, decltype(rows)::value, 0xf, false);
  };
  add(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{});
  add(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{});
  add(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{});
  add(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{});
  add(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});
  add(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});
  return x;
}

// Sum of x over the threads before this one, and over all (16 waves). Its halves are two sums.
__device__ __forceinline__ uint64_t scan(uint64_t x, uint64_t* box, uint64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t sum = up_to((uint32_t)x) | (uint64_t)up_to((uint32_t)(x >> 32)) << 32;
  lds_sync();  // the box has been read
  if (lane == 63) box[wave] = sum;
  lds_sync();
  uint64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kThreads / 64; ++w) {
    before += w < wave ? box[w] : 0;
    total += box[w];
  }
  return before + sum - x;
}

// 16 bytes of a slot's key and of its value to another slot.
__device__ __forceinline__ void move_chunk(const EvictArgs& a, const int32_t* pages, int head, int part, int from,
                                           int to) {
  const arthip_pages& p = a.c.p;
  const int64_t k_from = row_of(p, a.by_page, pages, from, a.c.k_cache_stride);
  const int64_t k_to = row_of(p, a.by_page, pages, to, a.c.k_cache_stride);
  if (k_from == -1 || k_to == -1) return;
  const int64_t v_from = row_of(p, a.by_page, pages, from, a.c.v_cache_stride);
  const int64_t v_to = row_of(p, a.by_page, pages, to, a.c.v_cache_stride);
  uint16_t* const k = static_cast<uint16_t*>(a.c.k_cache) + head * a.c.k_cache_stride[2] + part * 8;
  uint16_t* const v = static_cast<uint16_t*>(a.c.v_cache) + head * a.c.v_cache_stride[2] + part * 8;
  const u4 x = *reinterpret_cast<const u4*>(k + k_from), y = *reinterpret_cast<const u4*>(v + v_from);
  *reinterpret_cast<u4*>(k + k_to) = x;
  *reinterpret_cast<u4*>(v + v_to) = y;
}

// The slots of one key head of one sequence: a thread holds E of them in a row (E = 0: as many as
// there are, read again each time). The `keep`-th largest key is found bit by bit from the top: a
// candidate stands if at least `keep` keys reach it. Waves count with ballots, so that equal
// weights cost no more than others, as they would in a histogram's counters.
template <int E, bool HERE>
__global__ void __launch_bounds__(kThreads) evict_select(EvictArgs a) {
  __shared__ uint64_t box[kThreads / 64];
  __shared__ int counts[32];
  __shared__ int newest_box;
  __shared__ int list[kMoves];
  __shared__ int holes_at[HERE ? kMovesHere : 1];
  const arthip_pages& p = a.c.p;
  const int tid = threadIdx.x, lane = tid & 63;
  const int b = (int)fdiv(blockIdx.x, a.by_heads), head = (int)blockIdx.x - b * p.k_heads;
  const int n = min(slots_of(p, b), a.c.slots), keep = a.c.keep;
  const float* const w = a.c.weights + b * a.c.weights_stride[0] + head * a.c.weights_stride[1];
  const int32_t* const place =
      a.c.positions == nullptr ? nullptr : a.c.positions + b * a.c.positions_stride[0] + head * a.c.positions_stride[1];
  const int64_t at = blockIdx.x;
  float* const w_out = a.c.weights_out == nullptr ? nullptr : a.c.weights_out + at * a.c.slots;
  int32_t* const place_out = a.c.positions_out == nullptr ? nullptr : a.c.positions_out + at * a.c.slots;
  int32_t* const kept = a.c.kept + at * keep;
  const int used = min(n, keep);
  if (head == 0 && tid == 0 && a.c.new_len != nullptr) a.c.new_len[b] = used;
  for (int s = used + tid; s < a.c.slots; s += kThreads) {
    if (w_out != nullptr) w_out[s] = 0.0f;
    if (place_out != nullptr) place_out[s] = -1;
  }
  auto stays = [&](int s, int from) __attribute__((always_inline)) {
    kept[s] = from;
    if (w_out != nullptr) w_out[s] = w[from];
    if (place_out != nullptr) place_out[s] = place[from];
  };
  if (n <= keep) {
    for (int s = tid; s < keep; s += kThreads) {
      if (s < n)
        stays(s, s);
      else
        kept[s] = -1;
    }
    return;
  }

  const int each = E > 0 ? E : (n + kThreads - 1) / kThreads;
  const int first = tid * each;
  int newest = n - 1;
  if (place != nullptr) {
    if (tid == 0) newest_box = INT32_MIN;
    lds_sync();
    int top = INT32_MIN;
    for (int s = tid; s < n; s += kThreads) top = max(top, place[s]);
    atomicMax(&newest_box, top);
    lds_sync();
    newest = newest_box;
  }
  auto key_of = [&](int s) __attribute__((always_inline)) -> uint32_t {
    if (s >= n) return 0u;
    const int64_t t = place != nullptr ? place[s] : s;
    return t > (int64_t)newest - a.c.recent || t < a.c.first ? UINT32_MAX : ordered(w[s]);
  };
  uint32_t keys[E > 0 ? E : 1];
  if constexpr (E > 0) {
#pragma unroll
    for (int i = 0; i < E; ++i) keys[i] = key_of(first + i);
  }
  auto each_key = [&](auto f) __attribute__((always_inline)) {
    if constexpr (E > 0) {
#pragma unroll
      for (int i = 0; i < E; ++i) f(first + i, keys[i]);
    } else {
      for (int i = 0; i < each; ++i) f(first + i, key_of(first + i));
    }
  };

  // -- the keep-th largest key ---------------------------------------------------------
  if (tid < 32) counts[tid] = 0;
  lds_sync();
  uint32_t least = 0;
  int reach = n;  // keys of `least` or more
  for (int bit = 31; bit >= 0 && reach != keep; --bit) {
    const uint32_t candidate = least | 1u << bit;
    int count = 0;
    each_key([&](int, uint32_t key) { count += __popcll(__ballot(key >= candidate)); });
    if (lane == 0) atomicAdd(&counts[bit], count);
    lds_sync();
    const int all = counts[bit];
    if (all >= keep) {
      least = candidate;
      reach = all;
    }
  }
  // Of the equals of the least, the lowest slots make up for what the larger leave.
  int equals_before = 0, equals = 0;
  uint64_t total;
  const bool ties = reach != keep;
  if (ties) {
    uint64_t here = 0;
    each_key([&](int s, uint32_t key) { here += s < n && key == least; });
    equals_before = (int)scan(here, box, total);
    equals = keep - (reach - (int)total);
  }
  auto each_slot = [&](auto f) __attribute__((always_inline)) {
    int seen = equals_before;
    each_key([&](int s, uint32_t key) {
      bool stay = key >= least && s < n;
      if (ties && key == least && s < n) stay = seen++ < equals;
      f(s, stay);
    });
  };

  // -- holes below the budget and slots past it that stay, by their ranks -----------------
  uint64_t mine = 0;  // holes, and movers above them
  each_slot([&](int s, bool stay) {
    mine += s < keep && !stay ? 1 : 0;
    mine += s >= keep && stay ? uint64_t{1} << 32 : 0;
  });
  const uint64_t before = scan(mine, box, total);
  const int moves = (int)(uint32_t)total;
  each_slot([&](int s, bool stay) {
    if (s < keep && stay) stays(s, s);
  });
  for (int from = 0; from < moves; from += kMoves) {
    lds_sync();  // the list has been read
    int rank = (int)(before >> 32) - from;
    each_slot([&](int s, bool stay) {
      if (s < keep || !stay) return;
      if ((uint32_t)rank < (uint32_t)kMoves) list[rank] = s;
      ++rank;
    });
    lds_sync();
    rank = (int)(uint32_t)before - from;
    each_slot([&](int s, bool stay) {
      if (s >= keep || stay) return;
      if ((uint32_t)rank < (uint32_t)kMoves) {
        stays(s, list[rank]);
        if constexpr (HERE) holes_at[rank] = s;
      }
      ++rank;
    });
  }
  if constexpr (HERE) {
    lds_sync();
    const int32_t* const pages = p.pages + b * p.pages_stride;
    for (int i = tid; i < moves * a.head_chunks; i += kThreads) {
      const int m = (int)fdiv((uint32_t)i, a.by_head_chunks), part = i - m * a.head_chunks;
      move_chunk(a, pages, head, part, list[m], holes_at[m]);
    }
  }
}

// The rows that evict_select found to move: a thread 16 bytes of a slot's key and value. Rows come
// from slots past the budget and go to slots below it, so that no order is needed.
__global__ void __launch_bounds__(256) evict_move(EvictArgs a, int64_t first_block, int blocks) {
  const arthip_pages& p = a.c.p;
  const int64_t block = first_block + blockIdx.x, at = block / blocks;
  const int per = 256 / a.head_chunks;  // slots of a workgroup
  const int of = (int)fdiv(threadIdx.x, a.by_head_chunks), part = (int)threadIdx.x - of * a.head_chunks;
  const int s = (int)(block - at * blocks) * per + of;
  if (of >= per || s >= a.c.keep) return;
  const int from = a.c.kept[at * a.c.keep + s];
  if (from < 0 || from == s) return;
  const int b = (int)fdiv((uint32_t)at, a.by_heads), head = (int)at - b * p.k_heads;
  const int32_t* const pages = p.pages + b * p.pages_stride;
  move_chunk(a, pages, head, part, from, s);
}

template <int E>
void (*select_of(bool here))(EvictArgs) {
  return here ? evict_select<E, true> : evict_select<E, false>;
}

}  // namespace

hipError_t launch_cache_write(const arthip_cache_write_args& c, hipStream_t s) {
  if (c.p.batch == 0 || c.p.tokens == 0) return hipSuccess;
  WriteArgs a{};
  a.c = c;
  a.head_chunks = c.p.head_dim / 8;
  a.chunks = c.p.k_heads * a.head_chunks;
  a.group = std::max(1, 1024 / a.chunks);
  a.by_chunks = make_fastdiv((uint32_t)a.chunks);
  a.by_head_chunks = make_fastdiv((uint32_t)a.head_chunks);
  a.by_page = make_fastdiv((uint32_t)c.p.page_size);
  return launch_parts((c.p.tokens + (int64_t)a.group - 1) / a.group, 256, [&](int64_t first, unsigned count) {
    hipLaunchKernelGGL(cache_write, dim3(count), dim3(256), 0, s, a, first);
    return hipGetLastError();
  });
}

hipError_t launch_cache_evict(const arthip_cache_evict_args& c, hipStream_t s) {
  if (c.p.batch == 0) return hipSuccess;
  EvictArgs a{};
  a.c = c;
  a.head_chunks = c.p.head_dim / 8;
  a.by_page = make_fastdiv((uint32_t)c.p.page_size);
  a.by_heads = make_fastdiv((uint32_t)c.p.k_heads);
  a.by_head_chunks = make_fastdiv((uint32_t)a.head_chunks);
  const int64_t heads = (int64_t)c.p.batch * c.p.k_heads;
  const int most = std::min(c.keep, std::max(0, c.slots - c.keep));  // moves of a key head
  const bool here = most <= kMovesHere;
  const int each = (c.slots + kThreads - 1) / kThreads;
  const auto fn = each <= 4    ? select_of<4>(here)
                  : each <= 8  ? select_of<8>(here)
                  : each <= 16 ? select_of<16>(here)
                  : each <= 32 ? select_of<32>(here)
                               : select_of<0>(here);
  hipLaunchKernelGGL(fn, dim3((unsigned)heads), dim3(kThreads), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || here) return e;
  const int per = 256 / a.head_chunks;
  const int64_t blocks = ((int64_t)c.keep + per - 1) / per;
  return launch_parts(heads * blocks, 256, [&](int64_t first, unsigned count) {
    hipLaunchKernelGGL(evict_move, dim3(count), dim3(256), 0, s, a, first, (int)blocks);
    return hipGetLastError();
  });
}

}  // namespace arthip

// A paged cache's rows: new tokens into their slots (arthip_cache_write), and the
// eviction of the slots with little weight (arthip_cache_evict).

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "attention_dev.h"
#include "launch.h"
#include "paged.h"
#include "paged_dev.h"
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

constexpr int kWaves = 16;       // of the selecting workgroup
constexpr int kThreads = 64 * kWaves;
constexpr int kBins = 2048;      // 11 bits of a key at a time: 11, 11, 10
constexpr int kMoves = 8192;     // slots listed in LDS at once
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

// The slots of one key head of one sequence, by one workgroup. The `keep`-th largest key is found
// 11 bits at a time from a histogram of the keys that share the bits before; then each wave ranks
// the holes and the movers of a run of slots. Keys are read anew in every pass, 64 in a row a wave:
// they come from the L2 (32768 slots: some 1 us a pass).
template <bool HERE>
__global__ void __launch_bounds__(kThreads) evict_select(EvictArgs a) {
  __shared__ int bins[kBins];
  __shared__ int box[3][kWaves];
  __shared__ int found[3];
  __shared__ int list[HERE ? kMovesHere : kMoves];
  __shared__ int holes_at[HERE ? kMovesHere : 1];
  constexpr int kList = HERE ? kMovesHere : kMoves;
  const arthip_pages& p = a.c.p;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int b = (int)fdiv(blockIdx.x, a.by_heads), head = (int)blockIdx.x - b * p.k_heads;
  const int n = __builtin_amdgcn_readfirstlane(min(slots_of(p, b), a.c.slots)), keep = a.c.keep;
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

  int newest = n - 1;
  if (place != nullptr) {
    int top = INT32_MIN;
    for (int s = tid; s < n; s += kThreads) top = max(top, place[s]);
    top = over_wave(top, [](int x, int y) { return max(x, y); });
    if (lane == 0) box[0][wave] = top;
    lds_sync();
    newest = box[0][0];
    for (int i = 1; i < kWaves; ++i) newest = max(newest, box[0][i]);
  }
  auto key_of = [&](int s) __attribute__((always_inline)) -> uint32_t {
    const int64_t t = place != nullptr ? place[s] : s;
    const uint32_t u = ordered(w[s]);
    return t > (int64_t)newest - a.c.recent || t < a.c.first ? UINT32_MAX : u;
  };

  // -- the keep-th largest key ---------------------------------------------------------
  uint32_t least = 0;  // its bits so far
  int want = keep;     // it is the want-th largest of the keys that share them
  bool ties = false;   // of which not all stay
  for (int level = 0; level < 3; ++level) {
    const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, width = level == 2 ? 10 : 11;
    for (int i = tid; i < kBins; i += kThreads) bins[i] = 0;
    lds_sync();
    for (int s = tid; s < n; s += kThreads) {
      const uint32_t key = key_of(s);
      bool in = level == 0 || key >> (shift + width) == least >> (shift + width);
      const int bin = (int)(key >> shift) & ((1 << width) - 1);
      // Equal keys are common (weights of 0, protected slots) and would meet in one counter: two
      // of a wave's bins are counted by ballots.
#pragma unroll
      for (int round = 0; round < 2; ++round) {
        const uint64_t left = __ballot(in);
        if (left == 0) break;
        const int first = __builtin_amdgcn_readlane(bin, __builtin_ctzll(left));
        const bool same = in && bin == first;
        const int count = __popcll(__ballot(same));
        if (lane == (int)__builtin_ctzll(left)) atomicAdd(&bins[first], count);
        in = in && !same;
      }
      if (in) atomicAdd(&bins[bin], 1);
    }
    lds_sync();
    // Two bins a thread, the largest keys first: the bin in which the want-th key lies.
    const int top = kBins - 1 - 2 * tid;
    const int c0 = bins[top], c1 = bins[top - 1];
    const int sum = (int)up_to((uint32_t)(c0 + c1));
    if (lane == 63) box[level][wave] = sum;
    lds_sync();
    int before = sum - c0 - c1;
    for (int i = 0; i < wave; ++i) before += box[level][i];
    const bool here = before < want && want <= before + c0 + c1;
    if (here) {
      const bool second = want > before + c0;
      found[0] = top - (second ? 1 : 0);
      found[1] = want - before - (second ? c0 : 0);
      found[2] = second ? c1 : c0;
    }
    lds_sync();
    least |= (uint32_t)found[0] << shift;
    want = found[1];
    ties = found[2] != want;
    lds_sync();
    if (!ties) break;  // all keys from here on stay
  }

  // -- holes below the budget and slots past it that stay, by their ranks -----------------
  const int run = ((n + kWaves - 1) / kWaves + 63) & ~63;  // slots of a wave
  const int begin = min(wave * run, n), end = min(begin + run, n);
  auto all_waves = [&](int mine, int (&of)[kWaves], int& total) __attribute__((always_inline)) {
    if (lane == 0) of[wave] = mine;
    lds_sync();
    int before = 0;
    total = 0;
    for (int i = 0; i < kWaves; ++i) {
      before += i < wave ? of[i] : 0;
      total += of[i];
    }
    return before;
  };
  // Of the equals of the least, the lowest `want` slots stay.
  int equals_before = 0, total;
  if (ties) {
    int equals = 0;
    for (int s0 = begin; s0 < end; s0 += 64) {
      const int s = s0 + lane;
      equals += __popcll(__ballot(s < end && key_of(min(s, n - 1)) == least));
    }
    equals_before = all_waves(equals, box[0], total);
  }
  const uint64_t below = (uint64_t{1} << lane) - 1;
  auto each_slot = [&](auto f) __attribute__((always_inline)) {  // (slot, there is one, it stays)
    int seen = equals_before;
    for (int s0 = begin; s0 < end; s0 += 64) {
      const int s = s0 + lane;
      const uint32_t key = key_of(min(s, n - 1));
      bool stay = s < end && key >= least;
      if (ties) {
        const bool equal = s < end && key == least;
        const uint64_t mask = __ballot(equal);
        if (equal) stay = seen + __popcll(mask & below) < want;
        seen += __popcll(mask);
      }
      f(s, s < end, stay);
    }
  };
  int holes = 0, movers = 0;
  each_slot([&](int s, bool is, bool stay) {
    holes += __popcll(__ballot(is && s < keep && !stay));
    movers += __popcll(__ballot(is && s >= keep && stay));
  });
  const int holes_before = all_waves(holes, box[1], total);
  const int moves = total;
  const int movers_before = all_waves(movers, box[2], total);
  for (int from = 0; from == 0 || from < moves; from += kList) {
    if (movers > 0) {
      int rank = movers_before - from;
      each_slot([&](int s, bool is, bool stay) {
        const bool mover = is && s >= keep && stay;
        const uint64_t mask = __ballot(mover);
        const int mine = rank + __popcll(mask & below);
        if (mover && (uint32_t)mine < (uint32_t)kList) list[mine] = s;
        rank += __popcll(mask);
      });
    }
    lds_sync();
    int rank = holes_before - from;
    each_slot([&](int s, bool is, bool stay) {
      const bool hole = is && s < keep && !stay;
      const uint64_t mask = __ballot(hole);
      const int mine = rank + __popcll(mask & below);
      if (hole && (uint32_t)mine < (uint32_t)kList) {
        stays(s, list[mine]);
        if constexpr (HERE) holes_at[mine] = s;
      }
      if (from == 0 && is && s < keep && stay) stays(s, s);
      rank += __popcll(mask);
    });
    lds_sync();  // the list has been read
  }
  if constexpr (HERE) {
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
  hipLaunchKernelGGL(here ? evict_select<true> : evict_select<false>, dim3((unsigned)heads), dim3(kThreads), 0, s, a);
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

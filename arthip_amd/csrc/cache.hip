// A paged cache's rows: new tokens into their slots (arthip_cache_write), and the
// eviction of the slots with little weight (arthip_cache_evict).
//
// Writing is bound by HBM: 65280 tokens of 16 heads of 64, 535 MB in 107 us (5.0 TB/s). Eviction of 4
// caches of up to 32768 slots to 8192, 8 heads of 128, takes 87 us: 41 for the selection, by one
// workgroup a key head, whose passes over the keys wait for one another, and 46 for moving 180 MB.

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

// The slots of one key head of one sequence, by one workgroup. A wave holds the keys of a run of
// slots in registers, 64 slots in a row an instruction, E times (E = 0: more than fit, read anew in
// every pass). The `keep`-th largest key is found 11 bits at a time from a histogram of the keys that
// share the bits before; then each wave ranks the holes and the movers of its run.
template <int E, bool HERE>
__global__ void __launch_bounds__(kThreads) evict_select(EvictArgs a) {
  __shared__ int bins[3][kBins];
  __shared__ int box[5][kWaves];
  __shared__ int found[3][3];
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
  // (Where rows are moved by a kernel of their own, that one writes the weights and positions too.)
  auto stays = [&](int s, int from) __attribute__((always_inline)) {
    kept[s] = from;
    if (HERE && w_out != nullptr) w_out[s] = w[from];
    if (HERE && place_out != nullptr) place_out[s] = place[from];
  };
  auto rest = [&]() __attribute__((always_inline)) {  // what lies behind
    if constexpr (HERE)
      for (int s = used + tid; s < a.c.slots; s += kThreads) {
        if (w_out != nullptr) w_out[s] = 0.0f;
        if (place_out != nullptr) place_out[s] = -1;
      }
    for (int s = used + tid; s < keep; s += kThreads) kept[s] = -1;
  };
  if (n <= keep) {
    for (int s = tid; s < n; s += kThreads) stays(s, s);
    rest();
    return;
  }

  // -- the keys --------------------------------------------------------------------------
  const int each = (n + kThreads - 1) / kThreads;
  const int begin = min(wave * each * 64, n), end = min(begin + each * 64, n);  // the wave's slots
  uint32_t keys[E > 0 ? E : 1];
  int newest = n - 1;
  constexpr int kOnce = E == 4 ? 4 : E == 40 ? 20 : 8;  // 64 slots each whose addresses are known together
  // f(i, the lane's slot), i counting the wave's 64 slots in a row. (What is known of some of them is
  // kept from the others, or their addresses fill the registers.)
  auto each_run = [&](auto f) __attribute__((always_inline)) {
    if constexpr (E > 0) {
      int slot = begin + lane;
#pragma unroll
      for (int i = 0; i < E; ++i)
        if (i < each) {
          if (i % kOnce == 0) {
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("" : "+v"(slot));
          }
          f(i, slot + i % kOnce * 64);
          if (i % kOnce == kOnce - 1) slot += kOnce * 64;
        }
    }
  };
  for (int i = tid; i < 3 * kBins; i += kThreads) bins[0][i] = 0;
  // All weights' loads are in flight at once, and positions' where registers hold them (32 key heads of
  // 32768 slots: 42 us, eight at a time 52).
  constexpr bool kPlaces = E > 0 && E <= 16;
  int places[kPlaces ? E : 1];
  each_run([&](int i, int slot) __attribute__((always_inline)) {
    const int s = min(slot, n - 1);  // (past the run: the last slot's)
    keys[i] = __builtin_bit_cast(uint32_t, w[s]);
    if constexpr (kPlaces) places[i] = place != nullptr ? place[s] : s;
  });
  if (place != nullptr) {
    int top = INT32_MIN;
    if constexpr (kPlaces) {
      each_run([&](int i, int) __attribute__((always_inline)) { top = max(top, places[i]); });
    } else {
#pragma unroll 8
      for (int s = tid; s < n; s += kThreads) top = max(top, place[s]);
    }
    top = over_wave(top, [](int x, int y) { return max(x, y); });
    if (lane == 0) box[3][wave] = top;
  }
  lds_sync();
  if (place != nullptr) {
    newest = box[3][0];
    for (int i = 1; i < kWaves; ++i) newest = max(newest, box[3][i]);
  }
  auto key = [&](float weight, int64_t t) __attribute__((always_inline)) -> uint32_t {
    return t > (int64_t)newest - a.c.recent || t < a.c.first ? UINT32_MAX : ordered(weight);
  };
  each_run([&](int i, int slot) __attribute__((always_inline)) {
    const int s = min(slot, n - 1);
    const int t = kPlaces ? places[kPlaces ? i : 0] : place != nullptr ? place[s] : s;
    keys[i] = key(__builtin_bit_cast(float, keys[i]), t);
  });
  auto each_slot = [&](auto f) __attribute__((always_inline)) {  // (slot, there is one, its key)
    if constexpr (E > 0) {
      each_run([&](int i, int slot) __attribute__((always_inline)) { f(slot, slot < end, keys[i]); });
    } else {
      for (int s0 = begin; s0 < end; s0 += 64 * kOnce) {
        uint32_t x[kOnce];
#pragma unroll
        for (int i = 0; i < kOnce; ++i) {
          const int s = min(s0 + i * 64 + lane, n - 1);
          x[i] = key(w[s], place != nullptr ? place[s] : s);
        }
#pragma unroll
        for (int i = 0; i < kOnce; ++i) f(s0 + i * 64 + lane, s0 + i * 64 + lane < end, x[i]);
      }
    }
  };

  // -- the keep-th largest key ---------------------------------------------------------
  uint32_t least = 0;  // its bits so far
  int want = keep;     // it is the want-th largest of the keys that share them
  bool ties = false;   // of which not all stay
  for (int level = 0; level < 3; ++level) {
    const int shift = level == 0 ? 21 : level == 1 ? 10 : 0, width = level == 2 ? 10 : 11;
    int* const mine = bins[level];
    each_slot([&](int, bool is, uint32_t x) __attribute__((always_inline)) {
      const bool in = is && (level == 0 || x >> (shift + width) == least >> (shift + width));
      const int bin = (int)(x >> shift) & ((1 << width) - 1);
      const uint64_t mask = __ballot(in);
      if (mask == 0) return;
      // Equal keys (weights of 0, protected slots) would meet in one counter.
      const int first = __builtin_amdgcn_readlane(bin, __builtin_ctzll(mask));
      if (__ballot(in && bin != first) == 0) {
        if (lane == 0) atomicAdd(&mine[first], __popcll(mask));
      } else if (in) {
        atomicAdd(&mine[bin], 1);
      }
    });
    lds_sync();
    // Two bins a thread, the largest keys first: the bin in which the want-th key lies.
    const int top = kBins - 1 - 2 * tid;
    const int c0 = mine[top], c1 = mine[top - 1];
    const int sum = (int)up_to((uint32_t)(c0 + c1));
    if (lane == 63) box[level][wave] = sum;
    lds_sync();
    int before = sum - c0 - c1;
    for (int i = 0; i < wave; ++i) before += box[level][i];
    if (before < want && want <= before + c0 + c1) {
      const bool second = want > before + c0;
      found[level][0] = top - (second ? 1 : 0);
      found[level][1] = want - before - (second ? c0 : 0);
      found[level][2] = second ? c1 : c0;
    }
    lds_sync();
    least |= (uint32_t)found[level][0] << shift;
    want = found[level][1];
    ties = found[level][2] != want;
    if (!ties) break;  // all keys from here on stay
  }

  // -- holes below the budget and slots past it that stay, by their ranks -----------------
  // Of the equals of the least, the lowest `want` slots stay.
  int equals_before = 0;
  if (ties) {
    int equals = 0;
    each_slot([&](int, bool is, uint32_t x) { equals += __popcll(__ballot(is && x == least)); });
    if (lane == 0) box[4][wave] = equals;
    lds_sync();
    for (int i = 0; i < wave; ++i) equals_before += box[4][i];
  }
  const uint64_t below = (uint64_t{1} << lane) - 1;
  auto each_stay = [&](auto f) __attribute__((always_inline)) {  // (slot, there is one, it stays)
    int seen = equals_before;
    each_slot([&](int s, bool is, uint32_t x) __attribute__((always_inline)) {
      bool stay = is && x >= least;
      if (ties) {
        const bool equal = is && x == least;
        const uint64_t mask = __ballot(equal);
        if (equal) stay = seen + __popcll(mask & below) < want;
        seen += __popcll(mask);
      }
      f(s, is, stay);
    });
  };
  int holes = 0, movers = 0;
  each_stay([&](int s, bool is, bool stay) {
    holes += __popcll(__ballot(is && s < keep && !stay));
    movers += __popcll(__ballot(is && s >= keep && stay));
  });
  if (lane == 0) {
    box[0][wave] = holes;
    box[1][wave] = movers;
  }
  lds_sync();
  int holes_before = 0, movers_before = 0, moves = 0;
  for (int i = 0; i < kWaves; ++i) {
    holes_before += i < wave ? box[0][i] : 0;
    movers_before += i < wave ? box[1][i] : 0;
    moves += box[0][i];
  }
  for (int from = 0; from == 0 || from < moves; from += kList) {
    if (movers > 0) {
      int rank = movers_before - from;
      each_stay([&](int s, bool is, bool stay) __attribute__((always_inline)) {
        const bool mover = is && s >= keep && stay;
        const uint64_t mask = __ballot(mover);
        const int mine = rank + __popcll(mask & below);
        if (mover && (uint32_t)mine < (uint32_t)kList) list[mine] = s;
        rank += __popcll(mask);
      });
    }
    lds_sync();
    int rank = holes_before - from;
    each_stay([&](int s, bool is, bool stay) __attribute__((always_inline)) {
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
  rest();
}

// The rows that evict_select found to move: a thread 16 bytes of a slot's key and value. Rows come
// from slots past the budget and go to slots below it, so that no order is needed. The workgroups
// from `movers` on write the weights and positions.
constexpr int kSlots = 2048;  // of such a workgroup

__global__ void __launch_bounds__(256) evict_move(EvictArgs a, int64_t first_block, int blocks, int movers) {
  const arthip_pages& p = a.c.p;
  const int64_t block = first_block + blockIdx.x, at = block / blocks;
  const int index = (int)(block - at * blocks);
  const int b = (int)fdiv((uint32_t)at, a.by_heads), head = (int)at - b * p.k_heads;
  const int32_t* const kept = a.c.kept + at * a.c.keep;
  if (index >= movers) {
    const float* const w = a.c.weights + b * a.c.weights_stride[0] + head * a.c.weights_stride[1];
    const int s0 = (index - movers) * kSlots;
#pragma unroll
    for (int i = 0; i < kSlots; i += 256) {
      const int s = s0 + i + (int)threadIdx.x;
      if (s >= a.c.slots) return;
      const int from = s < a.c.keep ? kept[s] : -1;
      if (a.c.weights_out != nullptr) a.c.weights_out[at * a.c.slots + s] = from < 0 ? 0.0f : w[from];
      if (a.c.positions_out != nullptr)
        a.c.positions_out[at * a.c.slots + s] =
            from < 0 ? -1 : a.c.positions[b * a.c.positions_stride[0] + head * a.c.positions_stride[1] + from];
    }
    return;
  }
  const int per = 256 / a.head_chunks;  // slots of a workgroup
  const int of = (int)fdiv(threadIdx.x, a.by_head_chunks), part = (int)threadIdx.x - of * a.head_chunks;
  const int s = index * per + of;
  if (of >= per || s >= a.c.keep) return;
  const int from = kept[s];
  if (from < 0 || from == s) return;
  move_chunk(a, p.pages + b * p.pages_stride, head, part, from, s);
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
  // Registers hold the keys of 40 x 1024 slots beside what a pass needs (86 of 128). (32768 slots of 32 key
  // heads, keys in registers and read anew: 42 and 68 us; calls that cut 40960, 49152 and 65536 slots of 32
  // key heads to a quarter take 108, 174 and 241 us.)
  const auto fn = each <= 4    ? select_of<4>(here)
                  : each <= 16 ? select_of<16>(here)
                  : each <= 40 ? select_of<40>(here)
                               : select_of<0>(here);
  hipLaunchKernelGGL(fn, dim3((unsigned)heads), dim3(kThreads), 0, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || here) return e;
  const int per = 256 / a.head_chunks;
  const int movers = (c.keep + per - 1) / per;
  const int blocks = movers + (c.slots + kSlots - 1) / kSlots;
  return launch_parts(heads * blocks, 256, [&](int64_t first, unsigned count) {
    hipLaunchKernelGGL(evict_move, dim3(count), dim3(256), 0, s, a, first, blocks, movers);
    return hipGetLastError();
  });
}

}  // namespace arthip

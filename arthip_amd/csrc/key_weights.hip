// The attention weight that cached keys gather (arthip_key_weights): for each slot the sum of
// exp(score - lse) over the new tokens that see it and the query heads that share its key head.
//
// A workgroup owns a run of slots of one key head and takes all rows (token, head) that see them, so
// that nothing is added across workgroups but in a fixed order. S = Q K^T (v_mfma_f32_32x32x16): a
// lane holds 16 rows of ONE key, so that a weight is one multiply-add, one exponential and one
// addition to the lane's own sum; a row's lse is the same for a half's lanes and comes from LDS.
//
// Many rows (key_tile): each wave keeps its keys in registers, and the rows pass through LDS in
// tiles of 64, which four waves share. While one block of 32 rows goes through its exponentials, the
// next one's products are multiplied. Few rows (key_stream): the rows are kept instead, and a wave by
// itself streams the keys through a ring of tiles in LDS.
//
// Many rows are bound by their products and exponentials: 2 x 2000 tokens over up to 8192 keys, 32 heads
// of 128, 261 us (695 TFLOP/s; vector unit 45%, matrix unit 32% busy; cards differ, 244 to 261). Few rows by
// HBM: 16 tokens over up to 16384 keys of 8 heads, 279 MB in 74 us (3.7 TB/s).

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

// What the scores go through: nothing (the scale is in the exponent), a cap up to kCapSmall, or
// any cap and scale.
enum Shape { kPlain, kCap, kAny };

struct KeyArgs {
  arthip_key_weights_args c;
  int group;   // query heads of a key head
  int tiles;   // workgroups along the slots
  int splits;  // and along the rows
  int stream;  // slots of a workgroup with few rows
  FastDiv by_group, by_page, by_heads, by_tiles, by_splits;
  CapFit cap;
  float* part;  // [splits][batch * k_heads][slots], if splits > 1
};

constexpr int kRows = 64;  // of a tile
constexpr int kStarts = 4 * (kRows + 32) * 4;  // bytes of their exponents' starts in LDS
// Workgroups that many rows are divided into. (2 x 2000 tokens over up to 8192 keys: 32 heads of 128 with 1024,
// 2048, 4096: 272, 283, 282 us; 16 of 64 112, 98, 98.)
constexpr int kItems = 2048;
// And waves that few rows are. (16 tokens over up to 16384 keys with 2560, 5120, 10240: 87, 88, 90 us.)
constexpr int kStreams = 5120;

__device__ __forceinline__ float started(const KeyArgs& a, const Sequence& s, int b, int head, int slot) {
  if (slot >= s.start() || a.c.decay == 0.0f) return 0.0f;
  return a.c.decay * a.c.weights[b * a.c.weights_stride[0] + head * a.c.weights_stride[1] + slot];
}

// A score s of a block in the base of 2 or, plain ones, still to be scaled by `mul`.
template <Shape SHAPE, int KB>
__device__ __forceinline__ void transform(const KeyArgs& a, f16v (&s)[KB]) {
  if (SHAPE == kCap || (SHAPE == kAny && a.c.cap > 0)) {
    float far = 0.0f;
    if constexpr (SHAPE == kCap) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) far = fmaxf(far, fabsf(s[kb][r]));
    }
    if (SHAPE == kCap && !__any(!(far <= a.cap.reach))) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[kb][r] = cap_near(a.cap, s[kb][r]);
    } else {
      const float in = a.cap.in, out = a.cap.out;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float x = s[kb][r];
          const float e = __builtin_amdgcn_exp2f(x * in);
          const float y = __builtin_fmaf(-2.0f * out, __builtin_amdgcn_rcpf(e + 1.0f), out);
          s[kb][r] = SHAPE == kAny && fabsf(x) <= a.cap.reach ? cap_near(a.cap, x) : y;
        }
    }
  } else if constexpr (SHAPE == kAny) {
    const float unit = a.c.scale * kLog2e;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[kb][r] *= unit;
  }
}

// Rows [lo, hi) of a sequence's (token, head) that see a slot.
struct Rows {
  int lo, hi;
};
__device__ __forceinline__ Rows rows_of(const KeyArgs& a, const Sequence& s, int slot) {
  const int first = a.c.causal ? min(max(slot - s.start(), 0), s.tokens) : 0;
  const int64_t last = (int64_t)slot + a.c.left - s.start() + 1;
  const int end = a.c.left < 0 ? s.tokens : (int)min(max(last, (int64_t)first), (int64_t)s.tokens);
  return {first * a.group, end * a.group};
}

// What a row's exponents start from: -lse in the base of 2. A row that saw nothing (lse -inf), or none
// at all, weighs nothing.
__device__ __forceinline__ float start_of(const KeyArgs& a, const Sequence& s, int head, int row, int end) {
  if (row >= end) return -__builtin_inff();
  const int token = (int)fdiv((uint32_t)row, a.by_group), g = row - token * a.group;
  const float lse = a.c.lse[(int64_t)(s.first + token) * a.c.q_heads + head * a.group + g];
  return lse == -__builtin_inff() ? lse : -lse * kLog2e;
}

// A wave's own reads and writes of LDS so far are done.
__device__ __forceinline__ void lds_wave() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

// The sum of a lane's slot over the rows [from, to), by a wave from memory. A row whose start is -inf adds
// nothing, whatever it and the key hold, but a score that is not finite takes its weight to NaN: the
// kernels below find sums that became NaN once more by this, which leaves such rows out. (Asked
// of every block of rows there, it took the 2000-token pieces from 307 to 324 us.)
template <class T, int DP, Shape SHAPE>
__device__ __forceinline__ float apart(const KeyArgs& a, const Sequence& seq, int b, int head, int slot, int k1, int from,
                                       int to, float mul, float* starts) {
  using E = Elem<T>;
  using frag = typename E::frag;
  constexpr int KS = DP / 16;
  const arthip_pages& pg = a.c.p;
  const int lane = threadIdx.x & 63, n = lane & 31, half = lane >> 5;
  Rows mine = rows_of(a, seq, slot);
  if (slot >= k1) mine.hi = 0;
  const int64_t at = slot < k1 ? row_of(pg, a.by_page, pg.pages + b * pg.pages_stride, slot, a.c.k_cache_stride) : -1;
  const T* const key = static_cast<const T*>(a.c.k_cache) + at + head * a.c.k_cache_stride[2];
  float sum = 0.0f;
  for (int row0 = from; row0 < to; row0 += 32) {
    const int row = min(row0 + n, to - 1);
    const int token = (int)fdiv((uint32_t)row, a.by_group), g = row - token * a.group;
    const T* const query = static_cast<const T*>(a.c.q) + (int64_t)(seq.first + token) * a.c.q_stride[0] +
                           (int64_t)(head * a.group + g) * a.c.q_stride[1];
    f16v s[1] = {f16v{}};
#pragma unroll 1
    for (int ks = 0; ks < KS; ++ks) {
      const int d = ks * 16 + half * 8;
      const bool in = d < pg.head_dim;
      s[0] = E::mma(in ? *reinterpret_cast<const frag*>(query + d) : frag{},
                    in && at != -1 ? *reinterpret_cast<const frag*>(key + d) : frag{}, s[0]);
    }
    transform<SHAPE>(a, s);
    const float start = start_of(a, seq, head, row0 + n, to);
    lds_wave();  // the last rows' have been read
    if (half == 0) starts[n] = start;
    lds_wave();
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int of = 8 * (r / 4) + 4 * half + r % 4;
      const float base = starts[of], w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][r], mul, base));
      sum += row0 + of >= mine.lo && row0 + of < mine.hi && base != -__builtin_inff() ? w : 0.0f;
    }
  }
  return halves_sum(sum);
}

template <class T, int DP, int KB, Shape SHAPE>  // KB: blocks of 32 keys a wave
__global__ void __launch_bounds__(256, DP > 128 ? 1 : 2) key_tile(KeyArgs a) {
  using L = TileL<DP, kRows>;
  using E = Elem<T>;
  using frag = typename E::frag;
  constexpr int RB = L::RB, KS = DP / 16;
  constexpr int LOADS = L::kTile / 1024 / 4;  // of a wave
  constexpr int STEP = 1024 / RB;             // rows of a load
  constexpr uint32_t kOob = 0x80000000u;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  __shared__ __attribute__((aligned(16))) float starts[4][kRows];
  __shared__ float apart_starts[4][32];
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;

  const arthip_pages& pg = a.c.p;
  auto scalar = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  // Items go round the eight XCDs as they come: sequences differ in length. (Each XCD an eighth of them
  // in a row, which then share the queries: the calls above 277 for 283 us, 100 for 98.)
  const int item = (int)blockIdx.x;
  const int rest = (int)fdiv((uint32_t)item, a.by_splits), split = item - rest * a.splits;
  const int bh = (int)fdiv((uint32_t)rest, a.by_tiles), tile = rest - bh * a.tiles;
  const int b = (int)fdiv((uint32_t)bh, a.by_heads), head = bh - b * pg.k_heads;
  const int tid = threadIdx.x;
  const int wave = scalar(tid >> 6);
  const int lane = tid & 63;
  const int n = lane & 31;
  const int half = lane >> 5;

  Sequence seq = sequence_of(pg, b);
  seq.first = scalar(seq.first);
  seq.tokens = scalar(seq.tokens);
  seq.len = scalar(seq.len);
  const int k0 = tile * 128 * KB, k1 = min(k0 + 128 * KB, min(seq.len, a.c.slots));
  const int w0 = k0 + wave * 32 * KB;  // the wave's first key

  // -- the rows that see some of the keys ------------------------------------------------
  const int row0 = rows_of(a, seq, k0).lo, row_end = k1 > k0 ? max(rows_of(a, seq, k1 - 1).hi, row0) : row0;
  const int steps = (row_end - row0 + kRows - 1) / kRows;
  const int share = (steps + a.splits - 1) / a.splits;
  const int first = min(split * share, steps), last = min(first + share, steps);
  // Those that see the lane's keys; all of the wave's are seen by rows [whole_lo, whole_hi).
  Rows mine[KB];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    const int slot = w0 + 32 * kb + n;
    mine[kb] = rows_of(a, seq, slot);
    if (slot >= k1) mine[kb].hi = 0;
  }
  const int whole_lo = scalar(rows_of(a, seq, w0 + 32 * KB - 1).lo);
  const int whole_hi = scalar(w0 + 32 * KB <= k1 ? rows_of(a, seq, w0).hi : 0);

  // -- the keys ----------------------------------------------------------------------------
  frag k[KB][KS];
  {
    const int32_t* const pages = pg.pages + b * pg.pages_stride;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
      const int slot = w0 + 32 * kb + n;
      const int64_t row = slot < k1 && first < last ? row_of(pg, a.by_page, pages, slot, a.c.k_cache_stride) : -1;
      const T* const from = static_cast<const T*>(a.c.k_cache) + row + head * a.c.k_cache_stride[2];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int d = ks * 16 + half * 8;
        k[kb][ks] = row != -1 && d < pg.head_dim ? *reinterpret_cast<const frag*>(from + d) : frag{};
      }
    }
  }

  // -- staging -------------------------------------------------------------------------------
  const int l_row = lane * 16 / RB, chunk = lane * 16 % RB / 16;
  constexpr int BACK = 3 * 1024;  // what buffers begin before the rows, for the constants' sake
  // A lane's offset of load i in a tile that begins at row `from`, of token0.
  auto offset_of = [&](int i, int from, int token0) __attribute__((always_inline)) {
    const int of = wave * LOADS * STEP + l_row + i * STEP;  // the tile's row
    const int row = from + of;
    const int token = (int)fdiv((uint32_t)row, a.by_group), g = row - token * a.group;
    const int c = chunk ^ L::k_swizzle(of);
    return row < row_end && c * 8 < pg.head_dim
               ? (uint32_t)((token - token0) * (int)a.c.q_stride[0] + g * (int)a.c.q_stride[1] + c * 8) * 2 +
                     (BACK - i % 4 * 1024)
               : kOob;
  };
  // Tiles of whole tokens are alike but for the last.
  const bool alike = kRows % a.group == 0;
  uint32_t offset[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i) offset[i] = offset_of(i, row0, (int)fdiv((uint32_t)row0, a.by_group));
  auto stage = [&](int buf, int step) __attribute__((always_inline)) {
    const int from = row0 + step * kRows;
    const int token0 = scalar((int)fdiv((uint32_t)from, a.by_group));
    const char* const p = reinterpret_cast<const char*>(
        static_cast<const T*>(a.c.q) + (int64_t)(seq.first + token0) * a.c.q_stride[0] +
        (int64_t)head * a.group * a.c.q_stride[1]);
    const rsrc_t r = buffer_of(p - BACK, 0x7fffffffu);
    constexpr int N = LOADS < 4 ? LOADS : 4;
    if (!alike || from + kRows > row_end) {
#pragma unroll
      for (int i = 0; i < LOADS; ++i) offset[i] = offset_of(i, from, token0);
    }
#pragma unroll
    for (int i = 0; i < LOADS; i += N) {
      uint32_t at[N];
#pragma unroll
      for (int j = 0; j < N; ++j) at[j] = offset[i + j];
      load_lds16<N>(r, at, lds_base + buf * L::kTile + (wave * LOADS + i) * 1024);
    }
  };

  // -- the sums ------------------------------------------------------------------------------
  typedef __attribute__((address_space(3))) unsigned char lds_byte;
  typedef __attribute__((address_space(3))) const frag lds_frag;
  lds_byte* const lds0 = (lds_byte*)lds;
  const uint32_t q_lane = n * RB + (half ^ L::k_swizzle(n)) * 16;
  const float mul = SHAPE != kPlain ? 1.0f : a.c.scale * kLog2e;
  float sum[KB];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) sum[kb] = 0.0f;
  f16v even[KB], odd[KB];  // scores of blocks of 32 rows
  int pending = -1;        // first row of the one whose weights are still to be found (-1: none)
  // The weights of that block (scores s), which are summed, beside the products of block i of a tile.
  auto block = [&](bool more, int buf, int i, f16v (&s)[KB], f16v (&following)[KB]) __attribute__((always_inline)) {
    constexpr int N = KS * KB;
    lds_byte* const from = lds0 + buf * L::kTile + i * 32 * RB;
    frag q[KS];
    auto read = [&](int ks) __attribute__((always_inline)) { q[ks] = *(lds_frag*)(from + (q_lane ^ (ks * 32))); };
    auto product = [&](int j) __attribute__((always_inline)) {
      following[j % KB] = E::mma(q[j / KB], k[j % KB][j / KB], j < KB ? f16v{} : following[j % KB]);
    };
    const int step = (pending - row0) / kRows;
    const float* const start = starts[step & 3] + (pending - row0 - step * kRows) + 4 * half;
    float base[16];
    const bool has = pending >= 0;
    if (has) {
      transform<SHAPE>(a, s);
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f4 x = *reinterpret_cast<const f4*>(start + 8 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) base[4 * g + e] = x[e];
      }
    }
    if (has && more && pending >= whole_lo && pending + 32 <= whole_hi) {
      // A product, the operand of the second after it, and its share of the exponentials.
      constexpr int A = KS < 2 ? KS : 2;
#pragma unroll
      for (int ks = 0; ks < A; ++ks) read(ks);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        product(j);
        if (j % KB == 0 && j / KB + A < KS) read(j / KB + A);
#pragma unroll
        for (int e = j * 16 * KB / N; e < (j + 1) * 16 * KB / N; ++e)
          sum[e / 16] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[e / 16][e % 16], mul, base[e % 16]));
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
      if (has) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int row = pending + 8 * (r / 4) + 4 * half + r % 4;
            const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r], mul, base[r]));
            sum[kb] += row >= mine[kb].lo && row < mine[kb].hi ? w : 0.0f;
          }
      }
      if (!more) return;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) read(ks);
#pragma unroll
      for (int j = 0; j < N; ++j) product(j);
    }
  };

  if (first < last) {
    float next = 0.0f;
    if (wave == 0) starts[first & 3][lane] = start_of(a, seq, head, row0 + first * kRows + lane, row_end);
    stage(0, first);
    vm_wait();
    lds_sync();
    int buf = 0;
    for (int t = first; t < last; ++t) {
      if (t + 1 < last) {
        stage(buf ^ 1, t + 1);
        if (wave == 0) next = start_of(a, seq, head, row0 + (t + 1) * kRows + lane, row_end);
      }
      if (w0 < k1) {
        block(true, buf, 0, odd, even);
        pending = row0 + t * kRows;
        block(true, buf, 1, even, odd);
        pending += 32;
      }
      vm_wait();
      if (wave == 0) starts[(t + 1) & 3][lane] = next;
      lds_sync();
      buf ^= 1;
    }
    if (w0 < k1) block(false, 0, 0, odd, even);
  }

  // -- results -------------------------------------------------------------------------------
  bool odd_sum = false;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    sum[kb] = halves_sum(sum[kb]);
    odd_sum = odd_sum || sum[kb] != sum[kb];
  }
  if (__builtin_expect(__any(odd_sum), 0)) {
    for (int kb = 0; kb < KB; ++kb) {
      const float x = apart<T, DP, SHAPE>(a, seq, b, head, w0 + 32 * kb + n, k1, row0 + first * kRows,
                                          min(row0 + last * kRows, row_end), mul, apart_starts[wave]);
#pragma unroll
      for (int i = 0; i < KB; ++i) sum[i] = i == kb ? x : sum[i];
    }
  }
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    const float x = sum[kb];
    const int slot = w0 + 32 * kb + n;
    if (half != 0 || slot >= a.c.slots) continue;
    if (a.splits > 1) {
      a.part[((int64_t)split * pg.batch * pg.k_heads + bh) * a.c.slots + slot] = x;
    } else {
      float* const out = a.c.out + b * a.c.out_stride[0] + head * a.c.out_stride[1];
      out[slot] = slot < seq.len ? started(a, seq, b, head, slot) + x : 0.0f;
    }
  }
}

// Tiles of 32 keys in the ring of a wave, and keys of a workgroup at most (a lane holds the page of
// 16 of them).
constexpr int ring_of(int dp) { return dp > 128 ? 3 : 4; }
constexpr int kStream = 1024;

template <class T, int DP, Shape SHAPE>
__global__ void __launch_bounds__(64) key_stream(KeyArgs a) {
  using L = TileL<DP, 32>;
  using E = Elem<T>;
  using frag = typename E::frag;
  constexpr int RB = L::RB, KS = DP / 16, RING = ring_of(DP);
  constexpr int LOADS = L::kTile / 1024, STEP = 1024 / RB, GL = LOADS / 2;  // GL: loads of 16 keys
  constexpr uint32_t kOob = 0x80000000u;
  static_assert((RING - 1) * LOADS < 64, "loads that the counter holds");
  __shared__ __attribute__((aligned(16))) unsigned char lds[RING * L::kTile];
  __shared__ float sums[kStream];
  __shared__ __attribute__((aligned(16))) float starts[32];
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;
  const arthip_pages& pg = a.c.p;
  auto scalar = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  const int bh = (int)fdiv(blockIdx.x, a.by_tiles), chunk0 = (int)blockIdx.x - bh * a.tiles;
  const int b = (int)fdiv((uint32_t)bh, a.by_heads), head = bh - b * pg.k_heads;
  const int lane = threadIdx.x, n = lane & 31, half = lane >> 5;

  Sequence seq = sequence_of(pg, b);
  seq.first = scalar(seq.first);
  seq.tokens = scalar(seq.tokens);
  seq.len = scalar(seq.len);
  const int k0 = chunk0 * a.stream, k1 = min(k0 + a.stream, min(seq.len, a.c.slots));
  const int k_end = min(k0 + a.stream, a.c.slots);  // slots of the result
  const int row0 = rows_of(a, seq, k0).lo, row_end = k1 > k0 ? max(rows_of(a, seq, k1 - 1).hi, row0) : row0;
  const int tiles = k1 > k0 ? (k1 - k0 + 31) >> 5 : 0;

  if (row0 < row_end) {
    // Each lane the page of 16 keys.
    const int32_t* const pages = pg.pages + b * pg.pages_stride;
    const int of_lane = pages[min((int)fdiv((uint32_t)(k0 + 16 * lane), a.by_page), pg.max_pages - 1)];
    constexpr int BACK = 3 * 1024;
    const int l_row = lane * 16 / RB, chunk = lane * 16 % RB / 16;
    uint32_t offset[GL];
#pragma unroll
    for (int i = 0; i < GL; ++i) {
      const int c = chunk ^ L::k_swizzle(l_row + i * STEP);
      offset[i] = c * 8 < pg.head_dim
                      ? (uint32_t)((l_row + i * STEP) * (int)a.c.k_cache_stride[1] * 2 + c * 16 + BACK - i % 4 * 1024)
                      : kOob;
    }
    const uint64_t k_head = reinterpret_cast<uint64_t>(a.c.k_cache) + head * a.c.k_cache_stride[2] * 2 - BACK;
    auto stage = [&](int t) __attribute__((always_inline)) {
      const uint32_t to = lds_base + (uint32_t)(t % RING) * L::kTile;
      const int left = k1 - k0 - t * 32;  // keys past the length come as zeros
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const int slot = k0 + t * 32 + g * 16;
        const uint32_t page = (uint32_t)__builtin_amdgcn_readlane(of_lane, 2 * t + g);
        const uint32_t in = (uint32_t)(slot - (int)fdiv((uint32_t)slot, a.by_page) * pg.page_size);
        const uint64_t at = k_head + (uint64_t)page * (uint32_t)(a.c.k_cache_stride[0] * 2) +
                            in * (uint32_t)(a.c.k_cache_stride[1] * 2);
        const rsrc_t r = {(uint32_t)at, (uint32_t)(at >> 32) & 0xffffu,
                          page < (uint32_t)pg.pool_pages ? 0x7fffffffu : 0u, 0x00020000u};
        constexpr int N = GL < 4 ? GL : 4;
#pragma unroll
        for (int i = 0; i < GL; i += N) {
          uint32_t x[N];
#pragma unroll
          for (int j = 0; j < N; ++j)
            x[j] = left >= 32 || l_row + (g * GL + i + j) * STEP < left ? offset[i + j] : kOob;
          load_lds16<N>(r, x, to + (g * GL + i) * 1024);
        }
      }
    };
    typedef __attribute__((address_space(3))) unsigned char lds_byte;
    typedef __attribute__((address_space(3))) const frag lds_frag;
    lds_byte* const lds0 = (lds_byte*)lds;
    const uint32_t k_lane = n * RB + (half ^ L::k_swizzle(n)) * 16;
    const float mul = SHAPE != kPlain ? 1.0f : a.c.scale * kLog2e;

    uint64_t odd_sums = 0;
    for (int from = row0; from < row_end; from += 32) {
      // The rows: as the left operand in registers, what their exponents start from by way of LDS.
      frag q[KS];
      const int row = min(from + n, row_end - 1);
      const int token = (int)fdiv((uint32_t)row, a.by_group), g_head = row - token * a.group;
      const T* const qp = static_cast<const T*>(a.c.q) + (int64_t)(seq.first + token) * a.c.q_stride[0] +
                          (int64_t)(head * a.group + g_head) * a.c.q_stride[1];
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int d = ks * 16 + half * 8;
        q[ks] = d < pg.head_dim ? *reinterpret_cast<const frag*>(qp + d) : frag{};
      }
      const float mine = start_of(a, seq, head, from + n, row_end);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(q[ks]));  // loaded by here: the waits below count K's loads
      lds_sync();  // the last rows' have been used
      if (half == 0) starts[n] = mine;
      for (int t = 0; t < RING - 1; ++t)
        if (t < tiles) stage(t);
      lds_sync();
      float base[16];
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f4 x = *reinterpret_cast<const f4*>(starts + 8 * g + 4 * half);
#pragma unroll
        for (int e = 0; e < 4; ++e) base[4 * g + e] = x[e];
      }
      for (int t = 0; t < tiles; ++t) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the tile before has been read
        if (t + RING - 1 < tiles) {
          stage(t + RING - 1);
          asm volatile("s_waitcnt vmcnt(%0)" ::"n"((RING - 1) * LOADS) : "memory");
        } else {
          vm_wait();
        }
        lds_byte* const at = lds0 + t % RING * L::kTile;
        f16v s[1];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) s[0] = E::mma(q[ks], *(lds_frag*)(at + (k_lane ^ (ks * 32))), ks == 0 ? f16v{} : s[0]);
        transform<SHAPE>(a, s);
        const int slot = k0 + t * 32 + n;
        Rows seen = rows_of(a, seq, slot);
        if (slot >= k1) seen.hi = 0;
        float x = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int i = from + 8 * (r / 4) + 4 * half + r % 4;
          const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][r], mul, base[r]));
          x += i >= seen.lo && i < seen.hi ? w : 0.0f;
        }
        x = halves_sum(x);
        odd_sums |= __ballot(x != x);
        if (half == 0) sums[t * 32 + n] = from == row0 ? x : sums[t * 32 + n] + x;
      }
    }
    lds_sync();
    if (__builtin_expect(odd_sums != 0, 0)) {
      for (int t = 0; t < tiles; ++t) {
        const float x = apart<T, DP, SHAPE>(a, seq, b, head, k0 + t * 32 + n, k1, row0, row_end, mul, starts);
        if (half == 0) sums[t * 32 + n] = x;
      }
      lds_sync();
    }
  }
  float* const out = a.c.out + b * a.c.out_stride[0] + head * a.c.out_stride[1];
  for (int slot = k0 + lane; slot < k_end; slot += 64)
    out[slot] = slot < k1 ? started(a, seq, b, head, slot) + (row0 < row_end ? sums[slot - k0] : 0.0f) : 0.0f;
}

// The old weights and the sums of the ranges of rows, in order.
__global__ void __launch_bounds__(256) key_join(KeyArgs a, int64_t first_block, int64_t total) {
  const int64_t at = (first_block + blockIdx.x) * 256 + threadIdx.x;
  if (at >= total) return;
  const int bh = (int)(at / a.c.slots), slot = (int)(at - (int64_t)bh * a.c.slots);
  const int b = (int)fdiv((uint32_t)bh, a.by_heads), head = bh - b * a.c.p.k_heads;
  const Sequence s = sequence_of(a.c.p, b);
  float sum = 0.0f;
  if (slot < s.len) {
    sum = started(a, s, b, head, slot);
    for (int i = 0; i < a.splits; ++i) sum += a.part[i * total + at];
  }
  a.c.out[b * a.c.out_stride[0] + head * a.c.out_stride[1] + slot] = sum;
}

template <class T, int DP>
void (*pick(bool stream, Shape shape))(KeyArgs) {
  if (stream)
    return shape == kPlain ? key_stream<T, DP, kPlain> : shape == kCap ? key_stream<T, DP, kCap> : key_stream<T, DP, kAny>;
  return shape == kPlain ? key_tile<T, DP, 2, kPlain> : shape == kCap ? key_tile<T, DP, 2, kCap> : key_tile<T, DP, 2, kAny>;
}
template <class T>
void (*pick(int d, bool stream, Shape shape))(KeyArgs) {
  if (d <= 32) return pick<T, 32>(stream, shape);
  if (d <= 64) return pick<T, 64>(stream, shape);
  if (d <= 96) return pick<T, 96>(stream, shape);
  if (d <= 128) return pick<T, 128>(stream, shape);
  return pick<T, 256>(stream, shape);
}
int tile_bytes(int d) {
  return kRows * (d <= 32 ? 64 : d <= 64 ? 128 : d <= 128 ? 256 : 512);
}

}  // namespace

KeyWeightsPlan key_weights_plan(const arthip_key_weights_args& c) {
  KeyWeightsPlan p{1, 1, 0, 0};
  if (c.p.batch == 0 || c.slots == 0) return p;
  const int64_t rows = (int64_t)c.p.tokens * (c.q_heads / c.p.k_heads);
  const int64_t heads = (int64_t)c.p.batch * c.p.k_heads;
  if (rows <= 32 * c.p.batch) {
    // Few rows: enough workgroups of one wave for the chip, four times over as lengths differ.
    const int64_t tiles = (c.slots + 31) / 32;
    p.stream = 32 * (int)std::min<int64_t>(kStream / 32, std::max<int64_t>(1, heads * tiles / kStreams));
    p.tiles = (c.slots + p.stream - 1) / p.stream;
    return p;
  }
  p.tiles = (c.slots + 255) / 256;
  const int64_t items = heads * p.tiles;
  // Ranges of the rows: enough workgroups for the chip, of 512 rows at least.
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({(kItems + items - 1) / items, rows / c.p.batch / 512, 64}));
  if (p.splits > 1) p.workspace = (size_t)p.splits * heads * c.slots * sizeof(float);
  return p;
}

hipError_t launch_key_weights(const arthip_key_weights_args& c, hipStream_t s) {
  if (c.p.batch == 0 || c.slots == 0) return hipSuccess;
  const KeyWeightsPlan plan = key_weights_plan(c);
  KeyArgs a{};
  a.c = c;
  a.group = c.q_heads / c.p.k_heads;
  a.tiles = plan.tiles;
  a.stream = plan.stream;
  a.splits = plan.splits;
  const int64_t heads = (int64_t)c.p.batch * c.p.k_heads;
  const unsigned items = (unsigned)(heads * a.tiles * a.splits);
  a.by_group = make_fastdiv((uint32_t)a.group);
  a.by_page = make_fastdiv((uint32_t)c.p.page_size);
  a.by_heads = make_fastdiv((uint32_t)c.p.k_heads);
  a.by_tiles = make_fastdiv((uint32_t)a.tiles);
  a.by_splits = make_fastdiv((uint32_t)a.splits);
  if (c.cap > 0) a.cap = make_cap(c.cap, c.scale);
  a.part = static_cast<float*>(c.workspace);
  const Shape shape = c.cap > kCapSmall || !(c.scale > 0) ? kAny : c.cap > 0 ? kCap : kPlain;
  const auto fn = c.p.dtype == ARTHIP_TYPE_F16 ? pick<_Float16>(c.p.head_dim, plan.stream > 0, shape)
                                               : pick<__bf16>(c.p.head_dim, plan.stream > 0, shape);
  if (plan.stream > 0) {
    hipLaunchKernelGGL(fn, dim3(items), dim3(64), 0, s, a);
    return hipGetLastError();
  }
  const int bytes = 2 * tile_bytes(c.p.head_dim);
  hipError_t e = hipSuccess;
  if (bytes + kStarts > 65536)  // what a kernel may have without asking
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(fn, dim3(items), dim3(256), bytes, s, a);
  e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  const int64_t total = heads * c.slots;
  return launch_parts((total + 255) / 256, 256, [&](int64_t first, unsigned count) {
    hipLaunchKernelGGL(key_join, dim3(count), dim3(256), 0, s, a, first, total);
    return hipGetLastError();
  });
}

}  // namespace arthip

// Attention of new tokens over a paged cache (arthip_paged_attention).
//
// The query heads that share a key head are rows of one matrix. A row tile is as many whole
// tokens of a sequence as fit 32 rows a wave; a workgroup walks a row tile's keys in tiles
// that it stages in LDS. Both products are v_mfma_f32_32x32x16 with the keys of the first as
// rows, S^T = K Q^T: a lane holds 16 keys of ONE query, and the accumulator, packed to the
// element type, is the right operand of O^T += V^T P^T. Statistics are fp32 in the base of 2;
// P is rounded to the element type (it lies in [0, 2^10], fp16's in [0, 2^15]), its sum is taken
// before.
//
// Lengths are known on the device alone, and differ: one call holds prompts beside single
// tokens. So the work is divided there. The key tiles that the row tiles need, all sequences'
// in a row, are cut into equal ranges, one a workgroup; a range may end inside a row tile, whose
// parts a second kernel joins in a fixed order. Every wave finds its range's beginning from the
// lengths, a lane (or some) a sequence.
//
// Single tokens over long caches are bound by HBM: 16 over up to 16384 keys of 8 heads, 541 MB, 109 to 112
// us, of which the tiles take 102 to 108 (5.2 TB/s). Large calls are bound by products and exponentials, which
// share a SIMD's two or three waves: a prompt of 8192 with a window of 4096, 32 heads of 128, 467 us
// (884 TFLOP/s; matrix unit 48%, vector unit 40% busy), a frame of 8160 tokens over 40800, 12 heads of 64,
// 1230 us (832 TFLOP/s; 48% and 75%). (Cards differ: 444 to 482 us, 1123 to 1230.)

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "attention_dev.h"
#include "launch.h"
#include "paged.h"
#include "paged_dev.h"

namespace arthip {

namespace {

// What the scores go through: nothing (the scale is in the exponent), a cap up to kCapSmall, or
// any cap and scale.
enum Shape { kPlain, kCap, kAny };

struct PagedArgs {
  arthip_paged_attention_args c;
  int group;        // query heads of a key head
  int tile_tokens;  // tokens of a row tile
  int ranges;       // workgroups
  int lanes;        // that count one sequence's tiles together, if `before` is not there
  int few;          // 31 bits hold the units, times `ranges`
  FastDiv by_group, by_page, by_lanes, by_heads;
  CapFit cap;
  const int64_t* before;  // key tiles of the sequences before each [batch + 1], of all key heads
  // Parts of row tiles, two a range: the one that begins inside its tile, the one that ends inside.
  float* sums;    // [2 ranges][waves][padded D / 8][64 lanes][4] unscaled, as the lanes hold them
  float2* stats;  // [2 ranges][32 waves] of a row: maximum (base 2) and sum
  int4* pieces;   // [ranges] the row tile that begins in a range and ends in another: sequence, key head,
                  // tile, number of parts (0: none) and 2^16 times what the waves met
};

// Parts of row tiles in which a row met an infinity or NaN that it may not see: the one that begins
// inside its tile, the one that ends inside, whole row tiles.
constexpr int kHead = 1, kTail = 2, kWhole = 4;
constexpr int kMaxRanges = 1024, kAgain = 1 << 16;
// Workgroups that join. (16 single tokens with 512, 1024 and 2048: 113, 118, 124 us; prompts beside
// tokens 466, 471, 468.)
constexpr int kJoiners = 512;

constexpr int kStart = 2;
constexpr int kLeast = 4;  // units of a range, where there are that many

// Key tiles of a row tile: from `first` on, `count` of them. KT: log2 of the keys of one.
struct Span {
  int first, count;
};
template <int KT>
__device__ __forceinline__ Span span_of(const PagedArgs& a, const Sequence& s, int tile) {
  const int from = tile * a.tile_tokens, to = min(from + a.tile_tokens, s.tokens);
  const int lo = a.c.left < 0 ? 0 : min(max(s.start() + from - a.c.left, 0), s.len);
  const int hi = a.c.causal ? min(max(s.start() + to, 0), s.len) : s.len;
  const int first = lo >> KT;
  return {first, hi > lo ? ((hi + (1 << KT) - 1) >> KT) - first : 0};
}
// The units of a row tile: its key tiles, and before them kStart for what it takes to begin and end one.
template <int KT>
__device__ __forceinline__ int units_of(const PagedArgs& a, const Sequence& s, int tile) {
  return span_of<KT>(a, s, tile).count + kStart;
}
__device__ __forceinline__ int tiles_of(const PagedArgs& a, const Sequence& s) {
  return (s.tokens + a.tile_tokens - 1) / a.tile_tokens;
}

__device__ __forceinline__ int64_t shuffle(int64_t x, int lane) { return __shfl((long long)x, lane); }

// Where a unit lies.
struct Place {
  int b, head, tile, unit;  // unit: of the row tile's
};

// The row tile after a place's; false where there is none (which the units rule out, if no one changes
// the lengths meanwhile).
__device__ __forceinline__ bool next_tile(const PagedArgs& a, Sequence& s, Place& at) {
  at.unit = 0;
  if (++at.tile < tiles_of(a, s)) return true;
  at.tile = 0;
  if (++at.head < a.c.p.k_heads) return true;
  at.head = 0;
  do {
    if (++at.b >= a.c.p.batch) {
      at.b = a.c.p.batch - 1;
      return false;
    }
    s = sequence_of(a.c.p, at.b);
  } while (s.tokens == 0);
  return true;
}

// The units before each sequence, by one workgroup: a wave a sequence, then a running sum.
template <int KT>
__global__ void __launch_bounds__(1024) paged_count(PagedArgs a, int64_t* before) {
  __shared__ int64_t box[16];
  __shared__ int64_t carry;
  const arthip_pages& p = a.c.p;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (threadIdx.x == 0) {
    carry = 0;
    before[0] = 0;
  }
  for (int b0 = 0; b0 < p.batch; b0 += 1024) {
    // 16 waves, 64 sequences each; lane i keeps the i-th one's units.
    int64_t mine = 0;
    for (int i = 0; i < 64; ++i) {
      const int b = b0 + wave * 64 + i;
      if (b >= p.batch) break;
      const Sequence s = sequence_of(p, b);
      const int tiles = tiles_of(a, s);
      int64_t n = 0;
      for (int t = lane; t < tiles; t += 64) n += units_of<KT>(a, s, t);
#pragma unroll
      for (int step = 32; step > 0; step /= 2) n += shuffle(n, lane ^ step);
      if (lane == i) mine = n * p.k_heads;
    }
    int64_t sum = mine;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
      const int64_t y = shuffle(sum, max(lane - step, 0));
      sum += lane >= step ? y : 0;
    }
    lds_sync();
    if (lane == 63) box[wave] = sum;
    lds_sync();
    int64_t base = carry;
    for (int w = 0; w < wave; ++w) base += box[w];
    const int b = b0 + wave * 64 + lane;
    if (b < p.batch) before[b + 1] = base + sum;
    lds_sync();
    if (threadIdx.x == 1023) carry = base + sum;
    lds_sync();
  }
}

// A wave's view of the batch: units of each sequence (64 at most, `lanes` lanes each) or the
// counted ones. Where 31 bits hold all units times the ranges, sums and quotients are of 32 bits and
// stay in the vector unit.
template <int KT>
struct Finder {
  int64_t end;     // units of one key head up to the lane's share of its sequence
  uint32_t end32;  // the same, if they are few
  int64_t total;   // of all key heads
  Sequence mine;   // the lane's

  __device__ __forceinline__ void count(const PagedArgs& a, int lane) {
    const arthip_pages& p = a.c.p;
    if (a.before != nullptr) {
      total = a.before[p.batch];
      return;
    }
    const int b = (int)fdiv((uint32_t)lane, a.by_lanes), sub = lane - b * a.lanes;
    int64_t n = 0;
    mine = sequence_of(p, min(b, p.batch - 1));
    if (b < p.batch) {
      const int tiles = tiles_of(a, mine);
      for (int t = sub; t < tiles; t += a.lanes) n += units_of<KT>(a, mine, t);
    }
    if (a.few) {
      end32 = up_to((uint32_t)n);
      total = (int64_t)__builtin_amdgcn_readlane((int)end32, 63) * p.k_heads;
      return;
    }
    end = n;
#pragma unroll
    for (int step = 1; step < 64; step *= 2) {
      const int64_t y = shuffle(end, max(lane - step, 0));
      end += lane >= step ? y : 0;
    }
    total = shuffle(end, 63) * p.k_heads;
  }

  // The place of unit x, below `total` (uniform), and its sequence.
  __device__ __forceinline__ Place find(const PagedArgs& a, int64_t x, int lane, Sequence& s) const {
    auto scalar = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    auto from = [&](int v, int of) { return __builtin_amdgcn_readlane(v, scalar(of)); };
    const arthip_pages& p = a.c.p;
    Place at;
    if (a.before != nullptr) {
      int lo = 0, n = p.batch;  // the last sequence whose units begin at or before x
      while (n > 1) {
        const int step = (n + 63) >> 6;
        const bool in = lane * step < n && a.before[lo + min(lane * step, n - 1)] <= x;
        const int skip = (__popcll(__ballot(in)) - 1) * step;
        lo += skip;
        n = min(step, n - skip);
      }
      at.b = scalar(lo);
      const int64_t first = a.before[at.b], one = (a.before[at.b + 1] - first) / p.k_heads;
      s = sequence_of(p, at.b);
      at.head = scalar((int)((x - first) / one));
      x -= first + at.head * one;
    } else {
      // A sequence's key heads follow one another: its first unit is as many times the units of one
      // key head before it.
      const int of = a.few ? __popcll(__ballot(end32 <= fdiv((uint32_t)x, a.by_heads)))
                           : __popcll(__ballot(end <= x / p.k_heads));  // lanes before unit x's
      at.b = scalar(min((int)fdiv((uint32_t)of, a.by_lanes), p.batch - 1));
      const int first = at.b * a.lanes, last = first + a.lanes - 1;
      s = {from(mine.first, first), from(mine.tokens, first), from(mine.len, first)};
      if (a.few) {
        const uint32_t before = at.b > 0 ? (uint32_t)from((int)end32, first - 1) : 0u;
        const uint32_t one = (uint32_t)from((int)end32, last) - before, left = (uint32_t)x - before * (uint32_t)p.k_heads;
        at.head = scalar((int)(left / one));
        x = left - (uint32_t)at.head * one;
      } else {
        const int64_t before = at.b > 0 ? shuffle(end, first - 1) : 0, one = shuffle(end, last) - before;
        x -= before * p.k_heads;
        at.head = scalar((int)(x / one));
        x -= at.head * one;
      }
    }
    for (int t0 = 0;; t0 += 64) {
      const int t = t0 + lane;
      const uint32_t n = t < tiles_of(a, s) ? (uint32_t)units_of<KT>(a, s, t) : 0;
      const uint32_t sum = up_to(n), all = (uint32_t)from((int)sum, 63);
      if (x >= all && all > 0) {
        x -= all;
        continue;
      }
      const int of = min(__popcll(__ballot((int64_t)sum <= x)), 63);
      at.tile = scalar(t0 + of);
      at.unit = scalar((int)(x - ((uint32_t)from((int)sum, of) - (uint32_t)from((int)n, of))));
      return at;
    }
  }
};

__device__ __forceinline__ int ranges_of(const PagedArgs& a, int64_t total) {
  return total >= (int64_t)a.ranges * kLeast ? a.ranges : max((int)total / kLeast, total > 0 ? 1 : 0);
}

// One workgroup's range of the units: about as many as any other's. A cut that would leave only a
// little (a 32nd of a range, or four tiles) of a row tile on one side goes to that tile's end: two
// parts more cost more than they balance (256 tokens over 32765 keys: 147 us, 136 so).
struct Range {
  int64_t at, cut, slack;  // where it is, where it is cut off
  int64_t total;           // units of all ranges,
  int live;                // and their number
  Place place;
  Sequence seq;            // the place's

  // False where there is no range of this number.
  template <int KT>
  __device__ __forceinline__ bool begin(const PagedArgs& a, const Finder<KT>& finder, int ranges, int range, int lane) {
    auto scalar = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    total = finder.total;
    live = ranges;
    int64_t share;
    if (a.few) {
      const uint32_t all = (uint32_t)total, n = (uint32_t)live;
      at = (uint32_t)range * all / n;
      cut = (uint32_t)(range + 1) * all / n;
      share = all / n;
    } else {
      at = range * total / live;
      cut = (range + 1) * total / live;
      share = total / live;
    }
    slack = min(share >> 3, max(share >> 5, (int64_t)4));
    Sequence s;
    const Place p = finder.find(a, at, lane, s);
    place = {scalar(p.b), scalar(p.head), scalar(p.tile), scalar(p.unit)};
    seq = {scalar(s.first), scalar(s.tokens), scalar(s.len)};
    if (place.unit == 0) return true;
    const int left = units_of<KT>(a, seq, place.tile) - place.unit;
    if (place.unit <= slack) {
      at -= place.unit;
      place.unit = 0;
    } else if (left <= slack) {
      at += left;
      return next_tile(a, seq, place);
    }
    return true;
  }
  // Units to take of the row tile at hand, which has `units`.
  __device__ __forceinline__ int take(int units) const {
    const int64_t start = at - place.unit, end = start + units;
    if (cut >= end || (cut - start > slack && end - cut <= slack)) return units - place.unit;
    return cut - start <= slack ? 0 : (int)(cut - at);
  }
  // Whether the range ends with them.
  __device__ __forceinline__ bool last(int units) const { return cut <= at - place.unit + units; }
  // The range in which a row tile ends that has `units` and begins here.
  __device__ __forceinline__ int end_of(int units) const {
    return (int)(((at + units - slack) * live - 1) / total);
  }
};

template <class T, int DP, int KT, int NW, Shape SHAPE>
__global__ void __launch_bounds__(NW * 64, DP > 128 ? 1 : DP > 64 || (DP > 32 && SHAPE == kAny) ? 2 : 3)
    paged_tile(PagedArgs a) {
  using L = TileL<DP, KT>;
  using E = Elem<T>;
  using frag = typename E::frag;
  constexpr int LOG = KT == 64 ? 6 : 5;
  static_assert(1 << LOG == KT, "keys of a tile");
  constexpr int RB = L::RB, KB = KT / 32, KS = DP / 16, DB = DP / 32;
  constexpr int SEG = L::kTile / 1024;                 // loads of a tile, 1 KiB each
  constexpr int LOADS = (SEG + NW - 1) / NW;           // of a wave
  constexpr int STEP = 1024 / RB;                      // keys of a load
  constexpr int WK = LOADS * STEP;                     // keys that a wave loads: in one page each 16
  constexpr int NG = WK > 16 ? WK / 16 : 1;            // pages at most
  constexpr int GL = LOADS / NG;                       // loads of a page
  static_assert(SEG % NW == 0 && LOADS % NG == 0 && (WK <= 16 || WK % 16 == 0), "whole pages a wave");
  constexpr uint32_t kOob = 0x80000000u;
  constexpr bool kLazy = DP > 64;  // see follow()
  // A wave at its exponentials goes before one at its products where the vector unit has more to do
  // (heads of 64, 8160 over 40800: 1265 -> 1203 us; capped heads of 128 110 -> 106; plain ones 454 -> 472).
  constexpr bool kFirst = DP <= 64 || SHAPE != kPlain;
  // Two tiles a round of the walk: the next tile's scores need no copies (that frame 1212 -> 1169 us, prompts
  // beside single tokens 450 -> 438, in bf16 428 -> 414; one prompt 454 -> 452). Capped heads of 33 to 64 have
  // no registers for it: spilled ones in the walk cost more (4096 tokens, 16 heads of 64: two tiles 101 us,
  // one 90; 256 over 32765 keys 89 and 77; 8160 over 16320 without a mask 763 and 671).
  constexpr int kRound = NW == 4 && DP <= 128 && !(SHAPE == kCap && DP == 64) ? 2 : 1;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;
  constexpr int v_at = 2 * L::kTile;  // V's buffers

  const arthip_pages& pg = a.c.p;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  auto scalar = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  auto scalar64 = [&](int64_t x) {
    return (int64_t)((uint64_t)(uint32_t)scalar((int)x) | (uint64_t)(uint32_t)scalar((int)(x >> 32)) << 32);
  };

  // -- the workgroup's range ---------------------------------------------------------
  // Workgroups go round the eight XCDs: each takes an eighth of the ranges in a row, as row tiles
  // of one key head share K and V.
  Finder<LOG> finder;
  finder.count(a, tid & 63);
  const int live = scalar(ranges_of(a, finder.total));
  const int per = (live + 7) >> 3;
  const int range = ((int)blockIdx.x & 7) * per + ((int)blockIdx.x >> 3);
  if ((int)blockIdx.x >= live && tid == 0) a.pieces[blockIdx.x] = int4{};  // no such range
  if (((int)blockIdx.x >> 3) >= per || range >= live) return;
  Range r;
  if (!r.begin(a, finder, live, range, tid & 63)) {
    if (tid == 0) a.pieces[range] = int4{};
    return;
  }
  r.total = scalar64(r.total);
  r.slack = scalar64(r.slack);
  r.at = scalar64(r.at);
  r.cut = scalar64(r.cut);
  Place place = {scalar(r.place.b), scalar(r.place.head), scalar(r.place.tile), scalar(r.place.unit)};
  Sequence seq = {scalar(r.seq.first), scalar(r.seq.tokens), scalar(r.seq.len)};
  int odd = 0;  // what the wave met
  // The last of a range: the row tile that it shares with later ones, if any.
  auto finish = [&](int4 piece) __attribute__((always_inline)) {
    if constexpr (NW > 1) {
      int* const flag = reinterpret_cast<int*>(lds);
      lds_sync();
      if ((tid & 63) == 0) flag[wave] = odd;
      lds_sync();
      odd = 0;
      for (int i = 0; i < NW; ++i) odd |= flag[i];
    }
    piece.w |= odd << 16;
    if (tid == 0) a.pieces[range] = piece;
  };

  while (true) {
    // -- the lane's part -----------------------------------------------------------------
    // (Found again for every row tile: what would be kept across them is registers that the walk
    // needs. Spilled ones come back by loads that wait for the tiles' own.)
    int lane = tid & 63;
    asm volatile("" : "+v"(lane));
    const int n = lane & 31;     // its row of the wave's 32
    const int half = lane >> 5;  // which keys and values of it
    const int my_token = (int)fdiv((uint32_t)(wave * 32 + n), a.by_group);  // of the row tile
    const int g_head = wave * 32 + n - my_token * a.group;
    const float mul = SHAPE != kPlain ? 1.0f : a.c.scale * kLog2e;
    const int s_row = (wave * LOADS * 1024 + lane * 16) / RB;  // tile's key of the wave's first load
    const int s_chunk = lane * 16 % RB / 16;
    const int l_row = lane * 16 / RB;  // the same of the load's keys
    // A lane's offsets of a page's loads. (Less what an instruction's constant adds to both addresses:
    // buffers begin BACK before the rows.)
    constexpr int BACK = 3 * 1024;
    uint32_t k_off[GL], v_off[GL];
#pragma unroll
    for (int i = 0; i < GL; ++i) {
      auto offset = [&](int chunk, int64_t stride) __attribute__((always_inline)) {
        return chunk * 8 < pg.head_dim
                   ? (uint32_t)((l_row + i * STEP) * (int)stride * 2 + chunk * 16 + BACK - i % 4 * 1024)
                   : kOob;
      };
      k_off[i] = offset(s_chunk ^ L::k_swizzle(s_row + i * STEP), a.c.k_cache_stride[1]);
      v_off[i] = offset(s_chunk ^ L::v_swizzle(s_row + i * STEP), a.c.v_cache_stride[1]);
    }
    typedef __attribute__((address_space(3))) unsigned char lds_byte;
    typedef __attribute__((address_space(3))) const frag lds_frag;
    typedef __attribute__((address_space(3))) s4 lds_s4;
    lds_byte* const lds0 = (lds_byte*)lds;
    const uint32_t k_lane = n * RB + (half ^ L::k_swizzle(n)) * 16;
    const int v_row = 4 * half + (lane & 15) / 4;
    const uint32_t v_lane =
        v_row * RB + ((((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) ^ L::v_swizzle(v_row)) * 16 + (lane & 1) * 8;

    // -- a row tile, or a part of it ----------------------------------------------------
    const int token0 = place.tile * a.tile_tokens;
    const int rows = min(a.tile_tokens, seq.tokens - token0) * a.group;  // of the row tile
    const Span span = span_of<LOG>(a, seq, place.tile);
    const int units = span.count + kStart;
    r.place.unit = place.unit;
    const int take = r.take(units);
    const bool last = r.last(units);
    if (take == 0) {
      finish(int4{});
      return;
    }
    const int begin = span.first + max(place.unit - kStart, 0), end = span.first + max(place.unit + take - kStart, 0);
    const int32_t* const pages = pg.pages + place.b * pg.pages_stride;
    const int kv_len = seq.len, start = seq.start();
    // Keys [lo, hi) that a token sees.
    auto low = [&](int token) __attribute__((always_inline)) -> int {
      return a.c.left < 0 ? 0 : min(max(start + token - a.c.left, 0), kv_len);
    };
    auto high = [&](int token) __attribute__((always_inline)) -> int {
      return a.c.causal ? min(max(start + token + 1, 0), kv_len) : kv_len;
    };
    const bool real = wave * 32 + n < rows, w_real = wave * 32 < rows;
    const int token = token0 + (real ? my_token : 0);
    const int head = place.head * a.group + (real ? g_head : 0);
    const int lo = low(token), hi = high(token);
    // The wave's rows all see [w_lo_max, w_hi_min).
    const int t_first = token0 + (int)fdiv((uint32_t)min(wave * 32, rows - 1), a.by_group);
    const int t_last = token0 + (int)fdiv((uint32_t)min(wave * 32 + 31, rows - 1), a.by_group);
    const int w_lo_max = low(t_last), w_hi_min = high(t_first);

    frag q[KS];
    {
      const T* const qp = static_cast<const T*>(a.c.q) + (seq.first + token) * a.c.q_stride[0] + head * a.c.q_stride[1];
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        const int d = s * 16 + half * 8;
        q[s] = real && d < pg.head_dim ? *reinterpret_cast<const frag*>(qp + d) : frag{};
      }
    }
    f16v o[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i) o[i] = f16v{};
    float m = -__builtin_inff(), l = 0.0f;

    // -- staging -------------------------------------------------------------------------
    // Where each 16 keys that the wave loads of a tile lie: their page, then their bytes in the pools
    // from the head on, less BACK, and the buffers' size (0 outside the pool: zeros). (Slots past the
    // length are not read, whatever their page.)
    struct Spot {
      int page[NG];
      uint64_t k[NG], v[NG];
      uint32_t size[NG];
    };
    const uint64_t k_head = reinterpret_cast<uint64_t>(a.c.k_cache) + place.head * a.c.k_cache_stride[2] * 2 - BACK;
    const uint64_t v_head = reinterpret_cast<uint64_t>(a.c.v_cache) + place.head * a.c.v_cache_stride[2] * 2 - BACK;
    auto ask = [&](Spot& x, int tile) __attribute__((always_inline)) {
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const int slot = tile * KT + wave * WK + g * 16;
        x.page[g] = pages[min((int)fdiv((uint32_t)slot, a.by_page), pg.max_pages - 1)];
      }
    };
    auto settle = [&](Spot& x, int tile) __attribute__((always_inline)) {  // after the wait for the loads
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        asm volatile("" : "+v"(x.page[g]));
        const uint32_t page = (uint32_t)scalar(x.page[g]);
        const int slot = tile * KT + wave * WK + g * 16;
        const uint32_t in = (uint32_t)(slot - (int)fdiv((uint32_t)slot, a.by_page) * pg.page_size);
        x.k[g] = k_head + (uint64_t)page * (uint32_t)(a.c.k_cache_stride[0] * 2) + in * (uint32_t)(a.c.k_cache_stride[1] * 2);
        x.v[g] = v_head + (uint64_t)page * (uint32_t)(a.c.v_cache_stride[0] * 2) + in * (uint32_t)(a.c.v_cache_stride[1] * 2);
        x.size[g] = page < (uint32_t)pg.pool_pages ? 0x7fffffffu : 0u;
      }
    };
    auto stage = [&](const uint64_t (&from)[NG], const uint32_t (&size)[NG], const uint32_t (&offset)[GL], int tile,
                     uint32_t to) __attribute__((always_inline)) {
      const int left = kv_len - tile * KT;  // keys past the length come as zeros
      const uint32_t to_wave = to + wave * LOADS * 1024;
      constexpr int N = GL < 4 ? GL : 4;
      static_assert(GL % N == 0, "whole blocks of loads");
      auto loads = [&](auto all) __attribute__((always_inline)) {
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          const rsrc_t r = {(uint32_t)from[g], (uint32_t)(from[g] >> 32) & 0xffffu, size[g], 0x00020000u};
#pragma unroll
          for (int i = 0; i < GL; i += N) {
            uint32_t at_lane[N];
#pragma unroll
            for (int j = 0; j < N; ++j)
              at_lane[j] = decltype(all)::value || s_row + (g * GL + i + j) * STEP < left ? offset[i + j] : kOob;
            load_lds16<N>(r, at_lane, to_wave + (g * GL + i) * 1024);
          }
        }
      };
      if (left >= KT)
        loads(std::true_type{});
      else
        loads(std::false_type{});
    };
    auto stage_k = [&](int buf, int tile, const Spot& in) __attribute__((always_inline)) {
      stage(in.k, in.size, k_off, tile, lds_base + buf * L::kTile);
    };
    auto stage_v = [&](int buf, int tile, const Spot& in) __attribute__((always_inline)) {
      stage(in.v, in.size, v_off, tile, lds_base + v_at + buf * L::kTile);
    };

    // -- the products --------------------------------------------------------------------
    f16v s[kRound][KB];  // scores of a tile, and of the next, key block by key block
    int u = 0;           // the tile's
    auto scores = [&](int buf, f16v (&x)[KB]) __attribute__((always_inline)) {
      lds_byte* const from = lds0 + buf * L::kTile;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        lds_byte* const k = from + (k_lane ^ (ks * 32));
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) x[kb] = E::mma(*(lds_frag*)(k + kb * 32 * RB), q[ks], ks == 0 ? f16v{} : x[kb]);
      }
    };
    auto v_frag = [&](lds_byte* from, int kk) __attribute__((always_inline)) -> frag {  // 32 values of 16 keys
      const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(from + kk * 16 * RB));
      const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(from + kk * 16 * RB + 8 * RB));
      return __builtin_bit_cast(frag, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
    };
    auto values = [&](int buf, const frag (&p)[KT / 16]) __attribute__((always_inline)) {
      lds_byte* const from = lds0 + v_at + buf * L::kTile;
      lds_byte* v[DB];
#pragma unroll
      for (int db = 0; db < DB; ++db) v[db] = from + (v_lane ^ (db * 64));
#pragma unroll
      for (int kk = 0; kk < KT / 16; ++kk)
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] = E::mma(v_frag(v[db], kk), p[kk], o[db]);
    };

    // -- scores to weights -----------------------------------------------------------------
    // The scores in the base of 2 or, plain ones, still to be scaled by `mul`; hidden ones -inf.
    auto ready = [&](int k0, bool partial) __attribute__((always_inline)) {
      const int key0 = k0 + 4 * half;  // key of element r of block kb: key0 + 32 kb + 8 (r / 4) + r % 4
      if (SHAPE == kCap || (SHAPE == kAny && a.c.cap > 0)) {
        float far = 0.0f;
        if constexpr (SHAPE == kCap) {
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) far = fmaxf(far, fabsf(s[u][kb][r]));
        }
        if (SHAPE == kCap && !__any(!(far <= a.cap.reach))) {
          // Small scores: six plain operations where the exponential and the reciprocal take a
          // quarter of the rate each.
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[u][kb][r] = cap_near(a.cap, s[u][kb][r]);
        } else {
          // Off by some 2^-22 of the cap; large caps choose score by score.
          const float in = a.cap.in, out = a.cap.out;
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const float x = s[u][kb][r];
              const float e = __builtin_amdgcn_exp2f(x * in);
              const float y = __builtin_fmaf(-2.0f * out, __builtin_amdgcn_rcpf(e + 1.0f), out);
              s[u][kb][r] = SHAPE == kAny && fabsf(x) <= a.cap.reach ? cap_near(a.cap, x) : y;
            }
        }
      } else if constexpr (SHAPE == kAny) {
        const float unit = a.c.scale * kLog2e;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[u][kb][r] *= unit;
      }
      if (partial) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int key = key0 + 32 * kb + 8 * (r / 4) + r % 4;
            s[u][kb][r] = key >= lo && key < hi ? s[u][kb][r] : -__builtin_inff();
          }
      }
    };
    auto largest = [&]() __attribute__((always_inline)) {
      float top = s[u][0][0];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[u][kb][r]);
      return halves_max(top);
    };
    // A row's base is a score near its largest so far; this makes it the largest. Where that has not
    // grown by more than 2^8 or so nothing is rescaled. Heads above 64 take no maximum to see whether
    // it has: the weights' sum tells (also of a row that has seen nothing yet, whose base of -inf makes
    // it infinite or NaN), and they are found again. (Prompts beside single tokens 462 -> 448 us;
    // narrower heads have no registers for it.)
    auto follow = [&]() __attribute__((always_inline)) {
      const float next = fmaxf(m, largest());
      // A row that has seen nothing yet has no sums to keep (next may be -inf as well).
      const float f = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((m - next) * mul);
      m = next;
      l *= f;
#pragma unroll
      for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] *= f;
    };
    // The weights of the scores against a row's base, packed; their sum.
    auto weight = [&](int e, float base, float& sum, float (&w)[8], frag (&p)[KT / 16]) __attribute__((always_inline)) {
      const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][e / 16][e % 16], mul, -base));
      sum += x;
      w[e % 8] = x;
      if (e % 8 == 7) {
        typedef float f8 __attribute__((ext_vector_type(8)));
        p[e / 8] = __builtin_convertvector(f8{w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]}, frag);
      }
    };

    // -- the walk ------------------------------------------------------------------------
    // One barrier a tile. While the weights of tile t are found, the scores of tile t + 1 are
    // multiplied, in one run of instructions: a product takes the matrix unit 32 clocks, in which the
    // wave's exponentials go on. Then t's values are multiplied. K of tile t + 2 and V of tile t + 1
    // are on their way meanwhile to the buffers that the last barrier freed, and the page of the tile
    // after them is asked for.
    lds_sync();  // the last row tile has been used
    if (begin < end) {
      Spot here, next, then;
      ask(here, begin);
      ask(next, min(begin + 1, end - 1));
      ask(then, min(begin + 2, end - 1));
      settle(here, begin);
      stage_k(0, begin, here);
      settle(next, begin + 1);
      if (begin + 1 < end) stage_k(1, begin + 1, next);
      stage_v(0, begin, here);
      vm_wait();
      settle(then, begin + 2);
      lds_sync();
      if (w_real) scores(0, s[0]);
      lds_sync();  // K's first buffer has been used
      for (int t0 = begin; t0 < end; t0 += kRound) {
#pragma unroll
        for (u = 0; u < kRound; ++u) {
          const int t = t0 + u, buf = kRound > 1 ? u : (t - begin) & 1, k0 = t * KT;
          if (u > 0 && t >= end) break;
          if (t + 2 < end) stage_k(buf, t + 2, then);
          if (t + 1 < end) stage_v(buf ^ 1, t + 1, next);
          next = then;
          ask(then, min(t + 3, end - 1));
          if (w_real) {
            ready(k0, !(k0 >= w_lo_max && k0 + KT <= w_hi_min));
            if constexpr (!kLazy) {
              if (__any((largest() - m) * mul > 8.0f)) follow();
            }
            // fp16's weights are raised to the top of its range, so that small ones, of which a long
            // walk adds up many, keep their digits down to 2^-21 of a row's largest and are 0 below 2^-32.
            float base = (!kLazy && m == -__builtin_inff() ? 0.0f : m * mul) - E::kRaise;
            f16v following[KB];
            frag p[KT / 16];
            float w[8], sum = 0.0f;
            if constexpr (kFirst) __builtin_amdgcn_s_setprio(1);
            {
              // A product, the operand of the fourth after it, and its share of the exponentials.
              constexpr int N = KS * KB, A = N < 4 ? N : 4;
              lds_byte* const from = lds0 + (buf ^ 1) * L::kTile;
              frag k[N];
              auto read = [&](int i) __attribute__((always_inline)) {
                k[i] = *(lds_frag*)(from + (k_lane ^ (i / KB * 32)) + i % KB * 32 * RB);
              };
#pragma unroll
              for (int i = 0; i < A; ++i) read(i);
#pragma unroll
              for (int i = 0; i < N; ++i) {
                following[i % KB] = E::mma(k[i], q[i / KB], i < KB ? f16v{} : following[i % KB]);
                if (i + A < N) read(i + A);
#pragma unroll
                for (int e = i * 16 * KB / N; e < (i + 1) * 16 * KB / N; ++e) weight(e, base, sum, w, p);
                __builtin_amdgcn_sched_barrier(0);
              }
            }
            if constexpr (kFirst) __builtin_amdgcn_s_setprio(0);
            if (kLazy && __any(!(sum <= E::kMost))) {
              follow();
              base = (m == -__builtin_inff() ? 0.0f : m * mul) - E::kRaise;
              sum = 0.0f;
#pragma unroll
              for (int e = 0; e < 16 * KB; ++e) {
                weight(e, base, sum, w, p);
                if (e % 8 == 7) __builtin_amdgcn_sched_barrier(0);  // or registers run out
              }
            }
            l += sum;  // this half's keys; the halves are added at the end
            values(buf, p);
            ahead<KT / 16 * DB, 2>();
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) s[kRound - 1 - u][kb] = following[kb];
          }
          vm_wait();
          settle(then, t + 3);
          lds_sync();
        }
      }
    }

    // Rows that do not see all of a tile weigh some of V by 0, which infinities and NaN survive. Where
    // the sums are not finite, such tiles are looked over, and those row tiles that met one are found
    // anew by the joining kernel.
    float rest = 0.0f;
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) rest = __builtin_fmaf(o[i][r], 0.0f, rest);
    if (__builtin_expect(__any(rest != 0.0f), 0)) {
      bool found = false;
      for (int t = begin; t < end; ++t) {
        if (!w_real || (t * KT >= w_lo_max && t * KT + KT <= w_hi_min)) continue;
        for (int i = lane; i < KT * (DP / 8); i += 64) {
          const int slot = t * KT + i / (DP / 8), d = i % (DP / 8) * 8;
          if (slot >= kv_len || d >= pg.head_dim) continue;
          const int64_t row = row_of(pg, a.by_page, pages, slot, a.c.v_cache_stride);
          if (row == -1) continue;
          const frag x = *reinterpret_cast<const frag*>(static_cast<const T*>(a.c.v_cache) + row +
                                                        place.head * a.c.v_cache_stride[2] + d);
#pragma unroll
          for (int e = 0; e < 8; ++e) found = found || !(fabsf((float)x[e]) < __builtin_inff());
        }
      }
      if (__any(found)) odd |= take == units ? kWhole : place.unit == 0 ? kTail : kHead;
    }

    // -- results -------------------------------------------------------------------------
    l = halves_sum(l);
    if (take < units) {
      if (real) {
        const int64_t part = 2 * range + (place.unit == 0 ? 1 : 0);
        f4* const sums = reinterpret_cast<f4*>(a.sums) + (part * NW + wave) * (DP / 8) * 64 + lane;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            if (db * 32 + 8 * g < pg.head_dim)
              sums[(db * 4 + g) * 64] = f4{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]};
        if (half == 0) a.stats[(part * NW + wave) * 32 + n] = float2{m * mul - E::kRaise, l};
      }
    } else {
      const float scale = l == 0.0f ? 0.0f : 1.0f / l;
      T* const op = static_cast<T*>(a.c.out) + (seq.first + token) * a.c.out_stride[0] + head * a.c.out_stride[1];
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int g = 0; g < 4; g += 2) {
          // A lane holds four values of every eight; the halves trade so that each stores
          // eight in a row.
          uint32_t w[2][2];
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              typedef float f2 __attribute__((ext_vector_type(2)));
              typedef T t2 __attribute__((ext_vector_type(2)));
              const f2 pair = {in_range<T>(o[db][4 * (g + e) + 2 * j] * scale),
                               in_range<T>(o[db][4 * (g + e) + 2 * j + 1] * scale)};
              w[e][j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, t2));
            }
          const u2 x = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
          const u2 y = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
          const int d = db * 32 + 8 * (g + half);
          if (real && d < pg.head_dim) *reinterpret_cast<u4*>(op + d) = u4{x[0], y[0], x[1], y[1]};
        }
      if (a.c.lse && real && half == 0)
        a.c.lse[(int64_t)(seq.first + token) * a.c.q_heads + head] =
            (m * mul - E::kRaise + __builtin_amdgcn_logf(l)) * kLn2;
    }
    if (last) {
      finish({place.b, place.head, place.tile,
              place.unit == 0 && take < units ? r.end_of(units) - range + 1 : 0});
      return;
    }
    r.at += take;
    next_tile(a, seq, place);
    place = {scalar(place.b), scalar(place.head), scalar(place.tile), 0};
    seq = {scalar(seq.first), scalar(seq.tokens), scalar(seq.len)};
  }
}

// One row by itself, from the definition: the rows of a workgroup's share of a row tile one after the
// other, each key added only to the rows that see it (an infinity whatever its weight).
template <class T>
__device__ __forceinline__ void rows_apart(const PagedArgs& a, int b, int kh, int tile, int index, int wide,
                                           float* weight, float* box) {
  const arthip_pages& pg = a.c.p;
  const Sequence seq = sequence_of(pg, b);
  const int32_t* const pages = pg.pages + b * pg.pages_stride;
  const int token0 = tile * a.tile_tokens, rows = min(a.tile_tokens, seq.tokens - token0) * a.group;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  for (int row = index; row < rows; row += wide) {
    const int of = (int)fdiv((uint32_t)row, a.by_group), token = token0 + of;
    const int head = kh * a.group + row - of * a.group, place = seq.start() + token;
    const int lo = a.c.left < 0 ? 0 : min(max(place - a.c.left, 0), seq.len);
    const int hi = a.c.causal ? min(max(place + 1, 0), seq.len) : seq.len;
    const T* const q = static_cast<const T*>(a.c.q) + (seq.first + token) * a.c.q_stride[0] + head * a.c.q_stride[1];
    auto score = [&](int slot) {  // in the base of 2
      const int64_t at = row_of(pg, a.by_page, pages, slot, a.c.k_cache_stride);
      float x = 0.0f;
      if (at != -1) {
        const T* const k = static_cast<const T*>(a.c.k_cache) + at + kh * a.c.k_cache_stride[2];
        for (int d = 0; d < pg.head_dim; ++d) x = __builtin_fmaf((float)q[d], (float)k[d], x);
      }
      if (!(a.c.cap > 0)) return x * (a.c.scale * kLog2e);
      if (fabsf(x) <= a.cap.reach) return cap_near(a.cap, x);
      const float e = __builtin_amdgcn_exp2f(x * a.cap.in);
      return __builtin_fmaf(-2.0f * a.cap.out, __builtin_amdgcn_rcpf(e + 1.0f), a.cap.out);
    };
    auto over_all = [&](float x, auto f) {
      x = over_wave(x, f);
      lds_sync();
      if (lane == 0) box[wave] = x;
      lds_sync();
      return f(f(box[0], box[1]), f(box[2], box[3]));
    };
    float top = -__builtin_inff();
    for (int slot = lo + tid; slot < hi; slot += 256) top = fmaxf(top, score(slot));
    top = over_all(top, [](float x, float y) { return fmaxf(x, y); });
    const float base = top == -__builtin_inff() ? 0.0f : top;
    float l = 0.0f, o = 0.0f;  // o: value tid of the head
    for (int slot0 = lo; slot0 < hi; slot0 += 256) {
      const int n = min(256, hi - slot0);
      lds_sync();
      if (tid < n) {
        const float w = __builtin_amdgcn_exp2f(score(slot0 + tid) - base);
        weight[tid] = w;
        l += w;
      }
      lds_sync();
      if (tid < pg.head_dim)
        for (int i = 0; i < n; ++i) {
          const int64_t at = row_of(pg, a.by_page, pages, slot0 + i, a.c.v_cache_stride);
          if (at == -1) continue;
          const float x = (float)static_cast<const T*>(a.c.v_cache)[at + kh * a.c.v_cache_stride[2] + tid];
          const float w = weight[i];
          o += w == 0.0f && !(fabsf(x) < __builtin_inff()) ? x : w * x;
        }
    }
    l = over_all(l, [](float x, float y) { return x + y; });
    T* const op = static_cast<T*>(a.c.out) + (seq.first + token) * a.c.out_stride[0] + head * a.c.out_stride[1];
    if (tid < pg.head_dim) op[tid] = to_elem<T>(in_range<T>(l == 0.0f ? 0.0f : o * (1.0f / l)));
    if (a.c.lse && tid == 0)
      a.c.lse[(int64_t)(seq.first + token) * a.c.q_heads + head] = (top + __builtin_amdgcn_logf(l)) * kLn2;
  }
}

// A workgroup's share of a job of the joining kernel: the parts of the row tile that begins in a range,
// in their order, four values of a row a thread; where there are fewer of these than threads, several
// threads take an item's parts in turn. What costs time is that loads wait: four items a thread, two
// parts of each at a time, are in flight (prompts 456 -> 449 us against one item a thread).
template <class T, int DP, int KT, int NW>
__device__ void join_one(const PagedArgs& a, int job, int index, int wide, f4* sums, float2* stats, int* met) {
  const arthip_pages& pg = a.c.p;
  const int range = job & ~kAgain, tid = threadIdx.x;
  if (__builtin_expect((job & kAgain) != 0, 0)) {
    // All whole row tiles of the range, once more.
    const int lane = tid & 63;
    Finder<KT> finder;
    finder.count(a, lane);
    Range r;
    bool on = r.begin(a, finder, ranges_of(a, finder.total), range, lane);
    while (on) {
      const int units = units_of<KT>(a, r.seq, r.place.tile);
      if (r.take(units) == units)
        rows_apart<T>(a, r.place.b, r.place.head, r.place.tile, index, wide, reinterpret_cast<float*>(sums),
                      reinterpret_cast<float*>(stats));
      if (r.last(units)) break;
      r.at += units - r.place.unit;
      on = next_tile(a, r.seq, r.place);
    }
    return;
  }
  const int4 piece = a.pieces[range];
  const int parts = piece.w & 0xffff;
  lds_sync();  // the last job is done
  if (tid == 0) *met = piece.w >> 16 & kTail;
  lds_sync();
  for (int s = 1 + tid; s < parts; s += 256)
    if (a.pieces[range + s].w >> 16 & kHead) *met = kHead;
  const Sequence seq = sequence_of(pg, piece.x);
  const int token0 = piece.z * a.tile_tokens;
  const int rows = min(a.tile_tokens, seq.tokens - token0) * a.group;
  // Items: four values of a row, the rows of a quad one after the other, as they lie in the parts, or
  // 8 rows of 8 quads, so that out is written 64 bytes at a time.
  const bool blocks = rows % 8 == 0 && pg.head_dim % 32 == 0;
  const int items = rows * (pg.head_dim / 4);
  const int share = (items + wide - 1) / wide;
  const int first = index * share, last = min(first + share, items);
  const int steps = max(min(256 / max(share, 1), parts), 1);  // threads of an item
  const int at_once = 256 / steps, step = tid / at_once;
  lds_sync();
  if (__builtin_expect(*met != 0, 0)) {
    lds_sync();
    rows_apart<T>(a, piece.x, piece.y, piece.z, index, wide, reinterpret_cast<float*>(sums), reinterpret_cast<float*>(stats));
    return;
  }
  // COUNT items a thread and ONCE parts of each at a time, all in flight.
  auto join = [&](auto count, auto once) __attribute__((always_inline)) {
    constexpr int COUNT = decltype(count)::value, ONCE = decltype(once)::value;
    for (int item0 = first; item0 < last; item0 += COUNT * at_once) {
      int row[COUNT], quad[COUNT];
      float top[COUNT], l[COUNT];
      f4 o[COUNT];
      bool in[COUNT];
      const f4* sums_at[COUNT];
      const float2* stats_at[COUNT];
#pragma unroll
      for (int c = 0; c < COUNT; ++c) {
        const int item = min(item0 + c * at_once + tid - step * at_once, last - 1);
        in[c] = item0 + c * at_once + tid - step * at_once < last && step < steps;
        if (blocks) {
          const int block = item >> 6, quads = block / (rows / 8);
          row[c] = (block - quads * (rows / 8)) * 8 + (item & 7);
          quad[c] = quads * 8 + (item >> 3 & 7);
        } else {
          quad[c] = item / rows;
          row[c] = item - quad[c] * rows;
        }
        const int wave = NW == 1 ? 0 : row[c] >> 5, n = row[c] & 31;
        sums_at[c] = reinterpret_cast<const f4*>(a.sums) + wave * (DP / 8) * 64 + (quad[c] >> 1) * 64 +
                     (quad[c] & 1) * 32 + n;
        stats_at[c] = a.stats + wave * 32 + n;
        top[c] = -__builtin_inff();
        l[c] = 0.0f;
        o[c] = f4{};
      }
      auto merge = [&](int c, float2 st, f4 x) __attribute__((always_inline)) {
        const float next = fmaxf(top[c], st.x), base = next == -__builtin_inff() ? 0.0f : next;
        const float f = __builtin_amdgcn_exp2f(top[c] - base), w = __builtin_amdgcn_exp2f(st.x - base);
        top[c] = next;
        l[c] = l[c] * f + st.y * w;
        // (A part that weighs nothing beside another has a factor of 0, which infinities and NaN survive, as they
        // do in the walk: its rows see them. Parts that hold some of what a row does not see are not joined.)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[c][e] = o[c][e] * f + x[e] * w;
      };
      if (step < steps) {
        for (int s0 = step; s0 < parts; s0 += ONCE * steps) {
          f4 x[COUNT][ONCE];
          float2 st[COUNT][ONCE];
#pragma unroll
          for (int i = 0; i < ONCE; ++i) {
            const int s = min(s0 + i * steps, parts - 1);
            // The first part is one that ends inside its tile, the others begin inside.
            const int64_t part = 2 * (range + s) + (s == 0 ? 1 : 0);
#pragma unroll
            for (int c = 0; c < COUNT; ++c) {
              x[c][i] = sums_at[c][part * NW * (DP / 8) * 64];
              st[c][i] = stats_at[c][part * NW * 32];
            }
          }
#pragma unroll
          for (int i = 0; i < ONCE; ++i)
            if (s0 + i * steps < parts)
#pragma unroll
              for (int c = 0; c < COUNT; ++c) merge(c, st[c][i], x[c][i]);
        }
      }
      if (COUNT == 1 && steps > 1) {
        stats[tid] = float2{top[0], l[0]};
        sums[tid] = o[0];
        lds_sync();
        if (in[0] && step == 0)
          for (int s = 1; s < steps; ++s) merge(0, stats[tid + s * at_once], sums[tid + s * at_once]);
      }
#pragma unroll
      for (int c = 0; c < COUNT; ++c) {
        if (!in[c] || step != 0) continue;
        const int of = (int)fdiv((uint32_t)row[c], a.by_group);
        const int64_t token = seq.first + token0 + of;
        const int head = piece.y * a.group + row[c] - of * a.group;
        const float scale = l[c] == 0.0f ? 0.0f : 1.0f / l[c];
        T* const op = static_cast<T*>(a.c.out) + token * a.c.out_stride[0] + head * a.c.out_stride[1];
        typedef T t4 __attribute__((ext_vector_type(4)));
#pragma unroll
        for (int e = 0; e < 4; ++e) o[c][e] = in_range<T>(o[c][e] * scale);
        *reinterpret_cast<t4*>(op + 4 * quad[c]) = __builtin_convertvector(o[c], t4);
        if (a.c.lse && quad[c] == 0) a.c.lse[token * a.c.q_heads + head] = (top[c] + __builtin_amdgcn_logf(l[c])) * kLn2;
      }
      if (COUNT == 1 && steps > 1) lds_sync();  // the sums have been read
    }
  };
  using std::integral_constant;
  if (share > 256)  // (steps is 1)
    join(integral_constant<int, 4>{}, integral_constant<int, 2>{});
  else if (parts <= 2 * steps)
    join(integral_constant<int, 1>{}, integral_constant<int, 2>{});
  else
    join(integral_constant<int, 1>{}, integral_constant<int, 8>{});
}

// Joins the parts of row tiles that several ranges share.
template <class T, int DP, int KT, int NW>
__global__ void __launch_bounds__(256) paged_join(PagedArgs a) {
  __shared__ f4 sums[256];
  __shared__ float2 stats[256];
  __shared__ int met;
  __shared__ int box[4];
  __shared__ int list[2 * kMaxRanges];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // The ranges in which such a row tile begins, and those with whole row tiles to find anew.
  constexpr int kEach = kMaxRanges / 256;
  int mine[2 * kEach], count = 0;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int range = tid * kEach + i, w = range < a.ranges ? a.pieces[range].w : 0;
    mine[2 * i] = (w & 0xffff) != 0 ? range : -1;
    mine[2 * i + 1] = (w >> 16 & kWhole) != 0 ? range | kAgain : -1;
    count += (mine[2 * i] >= 0) + (mine[2 * i + 1] >= 0);
  }
  const int sum = (int)up_to((uint32_t)count);
  if (lane == 63) box[wave] = sum;
  lds_sync();
  int jobs = 0, at = sum - count;
  for (int i = 0; i < 4; ++i) {
    at += i < wave ? box[i] : 0;
    jobs += box[i];
  }
  if (jobs == 0) return;
#pragma unroll
  for (int i = 0; i < 2 * kEach; ++i)
    if (mine[i] >= 0) list[at++] = mine[i];
  lds_sync();
  // Workgroups of a job; and the job and share of this one.
  const int wide = min(max((int)gridDim.x / jobs, 1), 16);
  for (int job = blockIdx.x; job < jobs * wide; job += gridDim.x)
    join_one<T, DP, KT, NW>(a, list[job / wide], job % wide, wide, sums, stats, &met);
}

struct TilePick {
  void (*fn)(PagedArgs);
  void (*join)(PagedArgs);
  void (*count)(PagedArgs, int64_t*);
  int threads;
  int bytes;  // of LDS
};

template <class T, int DP, int KT, int NW>
TilePick pick(Shape shape) {
  constexpr int LOG = KT == 64 ? 6 : 5;
  return {shape == kPlain ? paged_tile<T, DP, KT, NW, kPlain>
          : shape == kCap ? paged_tile<T, DP, KT, NW, kCap>
                          : paged_tile<T, DP, KT, NW, kAny>,
          paged_join<T, DP, LOG, NW>, paged_count<LOG>, NW * 64, 4 * TileL<DP, KT>::kTile};
}

// Values of a head, padded.
int padded(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : d <= 96 ? 96 : d <= 128 ? 128 : 256; }

template <class T>
TilePick pick(int d, bool one_wave, Shape shape) {
  switch (padded(d)) {
    case 32: return one_wave ? pick<T, 32, 32, 1>(shape) : pick<T, 32, 64, 4>(shape);
    case 64: return one_wave ? pick<T, 64, 32, 1>(shape) : pick<T, 64, 64, 4>(shape);
    case 96: return one_wave ? pick<T, 96, 32, 1>(shape) : pick<T, 96, 64, 4>(shape);
    case 128: return one_wave ? pick<T, 128, 32, 1>(shape) : pick<T, 128, 64, 4>(shape);
    default: return one_wave ? pick<T, 256, 32, 1>(shape) : pick<T, 256, 32, 4>(shape);
  }
}

}  // namespace

PagedPlan paged_plan(const arthip_paged_attention_args& c) {
  PagedPlan p{};
  if (c.p.batch == 0 || c.p.tokens == 0 || c.q_heads == 0) return p;
  const int group = c.q_heads / c.p.k_heads;
  const int64_t rows = (int64_t)c.p.tokens * group;
  p.one_wave = group <= 32 && rows <= (int64_t)32 * c.p.batch;
  const int tile = p.one_wave ? 32 : 128;
  p.tile_tokens = tile / group;
  p.ranges = c.p.head_dim > 128 ? (p.one_wave ? 512 : 256) : p.one_wave ? 1024 : c.p.head_dim <= 64 ? 768 : 512;
  p.counted = c.p.batch > 64;
  const size_t rows_kept = (size_t)2 * p.ranges * tile;
  p.sums = rows_kept * padded(c.p.head_dim) * sizeof(float);
  p.stats = rows_kept * sizeof(float2);
  p.pieces = (size_t)p.ranges * sizeof(int4);
  p.before = p.counted ? ((size_t)c.p.batch + 1) * sizeof(int64_t) : 0;
  return p;
}

hipError_t launch_paged_attention(const arthip_paged_attention_args& c, hipStream_t s) {
  if (c.p.batch == 0 || c.p.tokens == 0 || c.q_heads == 0) return hipSuccess;
  const PagedPlan plan = paged_plan(c);
  PagedArgs a{};
  a.c = c;
  a.group = c.q_heads / c.p.k_heads;
  a.tile_tokens = plan.tile_tokens;
  a.ranges = plan.ranges;
  a.lanes = 64;
  while (a.lanes * c.p.batch > 64 && a.lanes > 1) a.lanes /= 2;
  a.by_group = make_fastdiv((uint32_t)a.group);
  a.by_page = make_fastdiv((uint32_t)c.p.page_size);
  a.by_lanes = make_fastdiv((uint32_t)a.lanes);
  a.by_heads = make_fastdiv((uint32_t)c.p.k_heads);
  const int64_t tiles = ((int64_t)c.p.tokens / a.tile_tokens + 1) * c.p.batch;  // whatever q_offsets hold
  const int64_t units = ((int64_t)c.p.max_pages * c.p.page_size + 31) / 32 + 1 + kStart;
  a.few = tiles < INT32_MAX / units / c.p.k_heads / a.ranges;
  if (c.cap > 0) a.cap = make_cap(c.cap, c.scale);
  char* at = static_cast<char*>(c.workspace);
  a.sums = reinterpret_cast<float*>(at);
  a.stats = reinterpret_cast<float2*>(at += plan.sums);
  a.pieces = reinterpret_cast<int4*>(at += plan.stats);
  int64_t* const before = reinterpret_cast<int64_t*>(at += plan.pieces);
  const bool f16 = c.p.dtype == ARTHIP_TYPE_F16;
  const Shape shape = c.cap > kCapSmall || !(c.scale > 0) ? kAny : c.cap > 0 ? kCap : kPlain;
  const TilePick k =
      f16 ? pick<_Float16>(c.p.head_dim, plan.one_wave, shape) : pick<__bf16>(c.p.head_dim, plan.one_wave, shape);
  if (plan.counted) {
    a.before = before;
    hipLaunchKernelGGL(k.count, dim3(1), dim3(1024), 0, s, a, before);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(k.fn, dim3((unsigned)a.ranges), dim3((unsigned)k.threads), k.bytes, s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k.join, dim3(kJoiners), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace arthip

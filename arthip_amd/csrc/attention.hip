// Attention over strided tokens (arthip_attention): softmax(score + mask) V in one
// pass over the keys, with capped scores, a bias over the distance, windows,
// prefixes, documents and ragged lengths.
//
// The query heads that share a key head are rows of one matrix: row r of a key head
// is token r / G, head r % G of its G heads. A workgroup takes 32 rows a wave and
// walks the keys in tiles that it stages in LDS for all its waves. Both products are
// v_mfma_f32_32x32x16 with the keys of the first as rows, S^T = K Q^T: a lane then
// holds 16 keys of ONE query in its accumulator, so that the running maximum and sum
// need one exchange between the wave's halves a tile, the rescale of the output is
// one factor a lane, and the accumulator, packed to the element type, already is the
// right operand of O^T += V^T P^T. (The order of the keys inside a product is free:
// V's rows are fetched in the accumulator's order, by transposing LDS reads.)
//
// Statistics are fp32 in the base of 2. P is rounded to the element type for the
// second product (it lies in [0, 2^8], fp16's in [0, 2^15], see weights()); its sum is taken
// before the rounding. fp16 and bf16 run alike: 8192 x 8192 keys, 32 heads of 128: 1125 us, 977
// TFLOP/s, 79% of a large library product; heads of 64: 664 us. No unit is full there (vector
// 41%, matrix 42% busy; 59% and 35% with heads of 64): a wave's products and its exponentials
// follow one another, and two or three waves a SIMD cover only part of that. One token over
// 16384 keys: 4.8 TB/s.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <limits>
#include <type_traits>

#include "launch.h"
#include "token_dev.h"
#include "transformer.h"

namespace arthip {

namespace {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// tanh x / x by powers of x^2, up to x = 0.6.
constexpr double kTanh[5] = {0.9999999283998549, -0.33332323371192635, 0.13310358022610624, -0.05210962448570825,
                             0.015486690367999443};
// Up to this cap an error of 2^-22 caps is 2^-16 of a score, far below the rounding of the
// weights; above it small scores take a form of their own wherever they are. (Both forms for every
// score: causal 8192 with 32 heads of 128, scores beyond the cap, 740 -> 1069 us.)
constexpr float kCapSmall = 64.0f;

struct AttnArgs {
  arthip_attention_args c;
  int group;      // query heads of a key head
  int rows;       // rows of a key head: q_tokens * group
  int row_tiles;  // workgroups along the rows
  int splits;     // workgroups along the keys
  int range;      // tiles of each but the last
  int items;      // batch * k_heads * row_tiles * splits
  int table_lds;  // the tables of a key head's rows are kept in LDS
  int table_bytes;  // and take these
  int wide;       // keys further apart than 32-bit offsets reach
  FastDiv by_group, by_k_heads, by_row_tiles, by_splits, by_rows;
  float cap_reach;  // |q.k| up to which the polynomial of the capped scores holds
  float cap_fit[5];
  float cap_in, cap_out;  // 2 log2(e) scale / cap and log2(e) cap
  const int2* doc_ranges;  // smallest and largest document of each tile, [batch, or 1][doc_tiles]
  int doc_tiles, doc_tile;  // tiles of a sequence, keys of a tile
  float* part;    // [splits][batch * k_heads * rows][D] unscaled sums, if splits > 1
  float* stat;    // [splits][batch * k_heads * rows][2] maximum (base 2) and sum
};

template <class T>
struct Elem;
template <>
struct Elem<_Float16> {
  typedef h8 frag;
  static constexpr float kZero = 0x1p-25f;  // numbers of 0 and more up to here round to 0
  static constexpr float kRaise = 7.0f;     // weights are up to 2^(8 + 7), see weights()
  static __device__ __forceinline__ f16v mma(h8 a, h8 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Elem<__bf16> {
  typedef b8 frag;
  static constexpr float kZero = 0.0f;  // as the exponential's are 2^-126 or more, or 0
  static constexpr float kRaise = 0.0f;
  static __device__ __forceinline__ f16v mma(b8 a, b8 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

// The two halves' values of a lane's x. (The results are copied before they are cast:
// a bit cast of a vector's element takes element 0, whichever is named.)
__device__ __forceinline__ void halves(float x, float& low, float& high) {
  const uint32_t a = __builtin_bit_cast(uint32_t, x);
  const u2 r = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  const uint32_t r0 = r[0], r1 = r[1];
  low = __builtin_bit_cast(float, r0);
  high = __builtin_bit_cast(float, r1);
}
// f over the values of a wave, the same in every lane: quads, half rows, rows of 16, then
// halves, inside the vector unit. (A shuffle is an LDS instruction, which the compiler may
// move between a barrier and the wait before it.)
template <class X, class F>
__device__ __forceinline__ X over_wave(X x, F f) {
  auto dpp = [&](auto control) __attribute__((always_inline)) {
    const int y = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(control)::value, 0xf, 0xf, true);
    x = f(x, __builtin_bit_cast(X, y));
  };
  dpp(std::integral_constant<int, 0xb1>{});
  dpp(std::integral_constant<int, 0x4e>{});
  dpp(std::integral_constant<int, 0x141>{});
  dpp(std::integral_constant<int, 0x140>{});
  uint32_t u = __builtin_bit_cast(uint32_t, x);
  const u2 r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t r0 = r[0], r1 = r[1];
  x = f(__builtin_bit_cast(X, r0), __builtin_bit_cast(X, r1));
  u = __builtin_bit_cast(uint32_t, x);
  const u2 h = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t h0 = h[0], h1 = h[1];
  return f(__builtin_bit_cast(X, h0), __builtin_bit_cast(X, h1));
}
__device__ __forceinline__ int wave_min(int x) { return over_wave(x, [](int a, int b) { return min(a, b); }); }
__device__ __forceinline__ int wave_max(int x) { return over_wave(x, [](int a, int b) { return max(a, b); }); }

__device__ __forceinline__ float halves_max(float x) {
  float a, b;
  halves(x, a, b);
  return fmaxf(a, b);
}
__device__ __forceinline__ float halves_sum(float x) {
  float a, b;
  halves(x, a, b);
  return a + b;
}

// LDS of a workgroup: two buffers of K tiles and of V tiles, written by loads that go
// to LDS without passing registers. Such a load puts a wave's 64 x 16 bytes in a row,
// so rows cannot be padded; their 16-byte chunks are permuted instead, by an exclusive
// or with bits of the row, so that the 16 rows of a K operand, and the four rows of a
// transposed V read, lie on different banks. The permutation is in the addresses that
// the lanes load from.
template <int DP, int KT>  // values of a head, padded; keys of a tile
struct TileL {
  static constexpr int RB = DP <= 32 ? 64 : DP <= 64 ? 128 : DP <= 128 ? 256 : 512;  // bytes of a row
  static constexpr int kTile = KT * RB;
  static constexpr int kChunk = 1024;  // tiles whose documents are looked over at once
  // After two K tiles and two V tiles:
  static constexpr int kRange = 0;                   // int32 [2][16] documents of the waves
  static constexpr int kDoc = kRange + 2 * 16 * 4;   // int32 [2][64]
  static constexpr int kCode = kDoc + 2 * 64 * 4;    // int32 [2][64]
  static constexpr int kAny = kCode + 2 * 64 * 4;    // bit a tile: some key of a row's document
  static constexpr int kTable = kAny + kChunk / 8;   // fp32 [group][table_len], if it fits
  // and after that, with documents, int2 a tile: its range of them
  static constexpr int kBytes = 4 * kTile + kTable;
  static __device__ __forceinline__ int k_swizzle(int row) {
    return RB == 64 ? (row >> 2) & 3 : RB == 128 ? (row >> 1) & 7 : RB == 256 ? row & 15 : row & 7;
  }
  static __device__ __forceinline__ int v_swizzle(int row) {
    return RB == 64 ? 0 : RB == 128 ? ((row >> 1) & 1) << 2 : (row & 3) << 2;
  }
};

constexpr int kTableBytes = 16384;  // of the tables that a workgroup keeps in LDS

typedef uint32_t rsrc_t __attribute__((ext_vector_type(4)));

// A buffer of up to `bytes` bytes from p (uniform).
__device__ __forceinline__ rsrc_t buffer_of(const void* p, uint32_t bytes) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)a);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));
  return rsrc_t{lo, hi & 0xffffu, bytes, 0x00020000u};
}

// Loads from the buffer to LDS, 16 (4) bytes a lane, lane after lane from `to` on: N
// loads to consecutive KiB. An instruction's constant goes to both addresses, so that M0
// is set once; the caller's `base` of load i has to take those i KiB out. Offsets past the buffer bring zeros. The compiler does not
// see these loads (its own would make every later LDS read wait for them): vm_wait()
// stands between them and their use. Nor does it see that they read scalar registers,
// which a vector instruction (a lane read back from a spill, a first lane) may have
// written just before: that takes five wait states, the s_nop.
template <int N>
__device__ __forceinline__ void load_lds16(rsrc_t from, const uint32_t (&at)[N], const uint32_t (&base)[N],
                                           uint32_t to) {
  static_assert(N == 1 || N == 2 || N == 4, "KiB that the constant reaches");
  if constexpr (N == 1)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %2, %1, %3 offen lds"
                 :
                 : "s"(to), "s"(from), "v"(at[0]), "s"(base[0])
                 : "memory");
  else if constexpr (N == 2)
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %2, %1, %4 offen lds\n\t"
        "buffer_load_dwordx4 %3, %1, %5 offen offset:1024 lds"
        :
        : "s"(to), "s"(from), "v"(at[0]), "v"(at[1]), "s"(base[0]), "s"(base[1])
        : "memory");
  else
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %2, %1, %6 offen lds\n\t"
        "buffer_load_dwordx4 %3, %1, %7 offen offset:1024 lds\n\t"
        "buffer_load_dwordx4 %4, %1, %8 offen offset:2048 lds\n\t"
        "buffer_load_dwordx4 %5, %1, %9 offen offset:3072 lds"
        :
        : "s"(to), "s"(from), "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3]), "s"(base[0]), "s"(base[1]),
          "s"(base[2]), "s"(base[3])
        : "memory");
}
__device__ __forceinline__ void load_lds4(rsrc_t from, uint32_t at, uint32_t base, uint32_t to) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dword %1, %2, %3 offen lds"
               :
               : "s"(to), "v"(at), "s"(from), "s"(base)
               : "memory");
}
__device__ __forceinline__ void vm_wait() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// The order of a block of N products with R LDS reads each: the reads run four products
// ahead, so that their latency (some 64 to 128 clocks) passes behind the matrix unit.
// Left to itself the compiler reads an operand right before its product.
template <int N, int R>
__device__ __forceinline__ void ahead() {
  constexpr int A = N < 4 ? N : 4;
  __builtin_amdgcn_sched_group_barrier(0x100, A * R, 0);
#pragma unroll
  for (int i = 0; i < N - A; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, A, 0);
}

// What the scores go through: nothing (the scale is in the exponent), a cap up to kCapSmall,
// any of such a cap, slopes, table and a scale that turns their order, or the same with a
// larger cap.
enum Shape { kPlain, kCap, kAny, kLarge };

// cap tanh(x / cap) in the base of 2 of a score x up to 0.6 caps.
__device__ __forceinline__ float cap_near(const AttnArgs& a, float x) {
  const float z = x * x;
  float t = __builtin_fmaf(a.cap_fit[4], z, a.cap_fit[3]);
  t = __builtin_fmaf(t, z, a.cap_fit[2]);
  t = __builtin_fmaf(t, z, a.cap_fit[1]);
  t = __builtin_fmaf(t, z, a.cap_fit[0]);
  return x * t;
}

// A table's entry in the base of 2. Only -inf hides: the least finite numbers, which masks are made
// of, stay finite.
__device__ __forceinline__ float entry_of(float e) {
  const float x = e * kLog2e;
  return x == -__builtin_inff() && e != -__builtin_inff() ? -__FLT_MAX__ : x;
}

// A mean of finite values stays in their type's range: the weights' rounding (2^-11) can take one of
// fp16's largest numbers out of it.
template <class T>
__device__ __forceinline__ float in_range(float x) {
  if constexpr (std::is_same_v<T, _Float16>)
    return fabsf(x) < __builtin_inff() ? __builtin_amdgcn_fmed3f(x, -65504.0f, 65504.0f) : x;
  return x;
}

// SHARED: the waves of a workgroup hold the same (up to) 32 rows and divide each
// tile's keys; otherwise each holds 32 rows of its own and takes all keys.
template <class T, int DP, int KT, int NW, bool SHARED, Shape SHAPE>
__global__ void __launch_bounds__(NW * 64, DP > 128 ? 1 : DP > 64 || (DP > 32 && SHAPE >= kAny) ? 2 : 3)
    attention_tile(AttnArgs a) {
  using L = TileL<DP, KT>;
  using E = Elem<T>;
  using frag = typename E::frag;
  constexpr int RB = L::RB, KW = SHARED ? KT / NW : KT, KB = KW / 32, KS = DP / 16, DB = DP / 32;
  constexpr int ROWS = SHARED ? 32 : 32 * NW;
  constexpr int SEG = L::kTile / 1024;                // loads of a tile, 1 KiB each
  constexpr int LOADS = (SEG + NW - 1) / NW;          // of a wave
  constexpr uint32_t kOob = 0x80000000u;
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;
  constexpr int v_at = 2 * L::kTile;  // V's buffers
  unsigned char* const more = lds + 2 * v_at;  // what follows them
  const uint32_t more_base = lds_base + 2 * v_at;

  // Workgroups go round the eight XCDs. Row tiles of one key head share K and V: each XCD
  // takes an eighth of them in order (even for causal rows where batch times key heads is a
  // multiple of 8; one key head alone gives the busiest XCD 1.87 times the mean). A single row
  // tile shares nothing: its items go round as they come, one further each round, so that no
  // XCD gets all the first (long) ranges.
  const int bid = (int)blockIdx.x, per = (int)gridDim.x >> 3;
  const int item = a.row_tiles == 1 ? (bid & ~7) + ((bid + (bid >> 3)) & 7) : (bid & 7) * per + (bid >> 3);
  if (item >= a.items) return;
  const int ranges = (int)fdiv((uint32_t)item, a.by_splits);
  const int split = item - ranges * a.splits;
  const int bh = (int)fdiv((uint32_t)ranges, a.by_row_tiles);
  const int row_tile = a.row_tiles - 1 - (ranges - bh * a.row_tiles);  // causal: the longest first
  const int b = (int)fdiv((uint32_t)bh, a.by_k_heads);
  const int kh = bh - b * a.c.k_heads;

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int n = lane & 31;     // the lane's row of the wave's 32
  const int half = lane >> 5;  // which keys and values of it

  // -- rows ------------------------------------------------------------------------
  auto token_of = [&](int row) __attribute__((always_inline)) { return (int)fdiv((uint32_t)row, a.by_group); };
  auto scalar = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  const int kv_len = scalar(a.c.kv_len ? min(max(a.c.kv_len[b], 0), a.c.k_tokens) : a.c.k_tokens);
  const int q_start = scalar(a.c.q_start ? a.c.q_start[b] : a.c.k_tokens - a.c.q_tokens);
  const int pre = scalar(a.c.prefix ? min(max(a.c.prefix[b], 0), kv_len) : 0);
  // Keys [lo, hi) that a window leaves to a token (and those below pre).
  auto low = [&](int token) __attribute__((always_inline)) -> int {
    if (a.c.left < 0) return 0;
    const int64_t p = (int64_t)q_start + token - a.c.left;
    return p < 0 ? 0 : p > kv_len ? kv_len : (int)p;
  };
  auto high = [&](int token) __attribute__((always_inline)) -> int {
    if (a.c.right < 0) return kv_len;
    const int64_t p = (int64_t)q_start + token + a.c.right + 1;
    return p < 0 ? 0 : p > kv_len ? kv_len : (int)p;
  };
  const int first_row = row_tile * ROWS;
  const int last_row = min(first_row + ROWS, a.rows) - 1;
  const int w_row = first_row + (SHARED ? 0 : wave * 32);  // the wave's first
  const int wk = SHARED ? wave * KW : 0;                   // and its first key of a tile
  const int row = w_row + n;
  const bool real = row <= last_row;
  const int token = token_of(min(row, last_row));
  const int g_head = min(row, last_row) - token * a.group;
  const int head = kh * a.group + g_head;
  const int lo = low(token), hi = high(token);
  // The wave's and the workgroup's rows together: all see [lo_max, hi_min), some see
  // [lo_min, hi_max). Positions grow with the row.
  const int wr0 = min(w_row, last_row), wr1 = min(wr0 + 31, last_row);
  const int w_lo_min = low(token_of(wr0)), w_lo_max = low(token_of(wr1));
  const int w_hi_min = high(token_of(wr0)), w_hi_max = high(token_of(wr1));
  const bool w_real = w_row <= last_row;
  const int g_lo_min = low(token_of(first_row)), g_hi_max = high(token_of(last_row));

  frag q[KS];
  {
    const T* const qp = static_cast<const T*>(a.c.q) + b * a.c.q_stride[0] + token * a.c.q_stride[1] +
                        head * a.c.q_stride[2];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const int d = s * 16 + half * 8;
      q[s] = real && d < a.c.head_dim ? *reinterpret_cast<const frag*>(qp + d) : frag{};
    }
  }

  // -- score transforms --------------------------------------------------------------
  // Without cap and bias the scale goes into the exponent's multiply-add.
  const float mul = SHAPE != kPlain ? 1.0f : a.c.scale * kLog2e;
  const float slope = SHAPE >= kAny && a.c.slopes ? a.c.slopes[head] * kLog2e : 0.0f;
  const int cq = SHAPE >= kAny && a.c.code_q ? a.c.code_q[b * a.c.code_q_stride + token] : q_start + token;
  const float* const table = SHAPE >= kAny && a.c.table ? a.c.table : nullptr;
  const int32_t* const code_k = SHAPE >= kAny && a.c.code_k ? a.c.code_k + b * a.c.code_k_stride : nullptr;
  const int dq = a.c.doc_q ? a.c.doc_q[b * a.c.doc_q_stride + token] : 0;
  const int32_t* const doc_k = a.c.doc_k ? a.c.doc_k + b * a.c.doc_k_stride : nullptr;
  // The table has an entry of -inf; one that is not in LDS may (to read it whole costs a
  // workgroup more than its tiles: one token over 777 keys and 32768 entries 278 us for 17).
  bool hides = table && !a.table_lds;
  auto load_table = [&]() __attribute__((always_inline)) {
    float* const t = reinterpret_cast<float*>(more + L::kTable);
    const int len = a.group * a.c.table_len;  // kTableBytes bound it
    const float* const from = table + (int64_t)kh * len;
    bool h = false;
    for (int i = tid; i < len; i += NW * 64) {
      const float e = from[i];
      t[i] = entry_of(e);
      h = h || e == -__builtin_inff();
    }
    int* const flag = reinterpret_cast<int*>(more + L::kRange);
    const int found = __any(h);
    if (lane == 0) flag[wave] = found;
    lds_sync();
    int all = 0;
    for (int i = 0; i < NW; ++i) all |= flag[i];
    hides = scalar(all) != 0;
  };

  // -- the tiles: those of the prefix, then those of the windows ----------------------
  const int pre_tiles = (pre + KT - 1) / KT;
  const int win_first = max(g_lo_min / KT, pre_tiles);
  const int win_end = g_hi_max > g_lo_min ? (g_hi_max + KT - 1) / KT : 0;
  const int count = pre_tiles + max(win_end - win_first, 0);
  const int begin = min(split * a.range, count);
  const int end = split == a.splits - 1 ? count : min(begin + a.range, count);
  auto tile_of = [&](int i) __attribute__((always_inline)) { return i < pre_tiles ? i : i - pre_tiles + win_first; };

  // Documents: the range of a wave's rows, and of the workgroup's.
  uint64_t* const any = reinterpret_cast<uint64_t*>(more + L::kAny);
  int2* const tile_docs = reinterpret_cast<int2*>(more + L::kTable + a.table_bytes);
  const int2* const doc_ranges =
      doc_k ? a.doc_ranges + (a.c.doc_k_stride == 0 ? 0 : (int64_t)b * a.doc_tiles) : nullptr;
  int w_dmin = dq, w_dmax = dq, dmin = 0, dmax = 0;
  if (doc_k) {
    int* const range = reinterpret_cast<int*>(more + L::kRange);
    w_dmin = scalar(wave_min(dq));  // a lane past the last row repeats it
    w_dmax = scalar(wave_max(dq));
    lds_sync();
    if (lane == 0) {
      range[wave] = w_dmin;
      range[16 + wave] = w_dmax;
    }
    lds_sync();
    dmin = range[0];
    dmax = range[16];
    for (int i = 1; i < NW; ++i) {
      dmin = min(dmin, range[i]);
      dmax = max(dmax, range[16 + i]);
    }
  }

  f16v o[DB];
#pragma unroll
  for (int i = 0; i < DB; ++i) o[i] = f16v{};
  float m = -__builtin_inff(), l = 0.0f;

  // -- staging -------------------------------------------------------------------------
  const T* const kp = static_cast<const T*>(a.c.k) + b * a.c.k_stride[0] + kh * a.c.k_stride[2];
  const T* const vp = static_cast<const T*>(a.c.v) + b * a.c.v_stride[0] + kh * a.c.v_stride[2];
  const int s_row = (wave * LOADS * 1024 + lane * 16) / RB;  // of the wave's first load; the others follow
  const int s_chunk = lane * 16 % RB / 16;
  const int64_t ks2 = a.c.k_stride[1] * 2, vs2 = a.c.v_stride[1] * 2;  // bytes
  constexpr int STEP = 1024 / RB;  // rows of a load
  // K's permutation comes round after 16 rows (8 of 512 bytes), V's after 4.
  constexpr int KP = (RB == 512 ? 8 : 16) / STEP < LOADS ? (RB == 512 ? 8 : 16) / STEP : LOADS;
  constexpr int VP = 4 / STEP < 1 ? 1 : 4 / STEP < LOADS ? 4 / STEP : LOADS;
  uint32_t k_off[KP], v_off[VP];  // a lane's offsets, but for the rows between its loads
  auto offset_of = [&](int chunk, int64_t stride) __attribute__((always_inline)) {
    return chunk * 8 < a.c.head_dim ? (uint32_t)(s_row * (int)stride + chunk * 16) : kOob;
  };
#pragma unroll
  for (int i = 0; i < KP; ++i) k_off[i] = offset_of(s_chunk ^ L::k_swizzle(s_row + i * STEP), ks2);
#pragma unroll
  for (int i = 0; i < VP; ++i) v_off[i] = offset_of(s_chunk ^ L::v_swizzle(s_row + i * STEP), vs2);
  constexpr int BACK = 3 * 1024;  // what buffers begin before the tile, for the constants' sake
  auto stage = [&](const T* from, int64_t stride, auto offset, auto swizzle, int tile, uint32_t to)
      __attribute__((always_inline)) {
    if (SEG % NW != 0 && wave * LOADS >= SEG) return;
    const char* const p = reinterpret_cast<const char*>(from) + (int64_t)tile * KT * stride;
    const int left = kv_len - tile * KT;  // keys past the length come as zeros
    const uint32_t to_wave = to + wave * LOADS * 1024;
    if (__builtin_expect(!a.wide, 1)) {
      constexpr int N = LOADS < 4 ? LOADS : 4;
      static_assert(LOADS % N == 0, "whole blocks of loads");
      const rsrc_t r = buffer_of(p - BACK, 0x7fffffffu);
#pragma unroll
      for (int i = 0; i < LOADS; i += N) {
        uint32_t at[N], base[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
          base[j] = (i + j) * STEP * (uint32_t)stride + (BACK - j * 1024);
          at[j] = left >= KT || s_row + (i + j) * STEP < left ? offset(i + j) : kOob;
        }
        load_lds16<N>(r, at, base, to_wave + i * 1024);
      }
    } else {
      // 32-bit offsets would wrap: a buffer of its own for every key.
#pragma unroll 1
      for (int i = 0; i < LOADS; ++i) {
        const int row = s_row + i * STEP;
        const int chunk = s_chunk ^ swizzle(row);
        const uint32_t at[1] = {chunk * 8 < a.c.head_dim && row < left ? chunk * 16u : kOob}, base[1] = {0};
#pragma unroll 1
        for (int k = 0; k < STEP; ++k) {
          const int key = (wave * LOADS + i) * STEP + k;
          const rsrc_t far = buffer_of(p + key * stride, 0x7fffffffu);
          if (row == key) load_lds16<1>(far, at, base, to_wave + i * 1024);
        }
      }
    }
  };
  auto stage_k = [&](int buf, int tile) __attribute__((always_inline)) {
    stage(kp, ks2, [&](int i) { return k_off[i % KP]; }, L::k_swizzle, tile, lds_base + buf * L::kTile);
    // The tile's documents and codes, those past the length as zeros. (From the tile on: an offset
    // from the first key would pass 32 bits in the longest caches.)
    if (doc_k && wave == 0)
      load_lds4(buffer_of(doc_k + (int64_t)tile * KT, (uint32_t)min(kv_len - tile * KT, KT) * 4), lane * 4, 0,
                more_base + L::kDoc + buf * 256);
    if (code_k && wave == NW - 1)
      load_lds4(buffer_of(code_k + (int64_t)tile * KT, (uint32_t)min(kv_len - tile * KT, KT) * 4), lane * 4, 0,
                more_base + L::kCode + buf * 256);
  };
  auto stage_v = [&](int buf, int tile) __attribute__((always_inline)) {
    stage(vp, vs2, [&](int i) { return v_off[i % VP]; }, L::v_swizzle, tile, lds_base + v_at + buf * L::kTile);
  };

  // -- the products --------------------------------------------------------------------
  // Operands come from a lane's base plus constants; the permutation, an exclusive or
  // with the lane's bits, leaves one base for each K step and each block of V values.
  typedef __attribute__((address_space(3))) unsigned char lds_byte;
  typedef __attribute__((address_space(3))) const frag lds_frag;
  typedef __attribute__((address_space(3))) s4 lds_s4;
  lds_byte* const lds0 = (lds_byte*)lds;
  const uint32_t k_lane = (wk + n) * RB + (half ^ L::k_swizzle(n)) * 16;
  const int v_row = 4 * half + (lane & 15) / 4;
  const uint32_t v_lane =
      (wk + v_row) * RB + ((((lane >> 4) & 1) * 2 + ((lane & 3) >> 1)) ^ L::v_swizzle(v_row)) * 16 + (lane & 1) * 8;

  f16v s[KB];        // scores of the current tile, key block by key block
  frag p[KW / 16];   // weights of the previous tile
  auto scores = [&](int buf) __attribute__((always_inline)) {
    lds_byte* const at = lds0 + buf * L::kTile;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      lds_byte* const k = at + (k_lane ^ (ks * 32));
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) s[kb] = E::mma(*(lds_frag*)(k + kb * 32 * RB), q[ks], ks == 0 ? f16v{} : s[kb]);
    }
    ahead<KS * KB, 1>();
  };
  auto v_frag = [&](lds_byte* at, int kk) __attribute__((always_inline)) -> frag {  // 32 values of 16 keys (block kk)
    const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + kk * 16 * RB));
    const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(at + kk * 16 * RB + 8 * RB));
    return __builtin_bit_cast(frag, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  bool odd = false;  // a tile that a row does not see whole holds an infinity or NaN in V
  auto values = [&](int buf, bool look) __attribute__((always_inline)) {
    lds_byte* const at = lds0 + v_at + buf * L::kTile;
    lds_byte* v[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) v[db] = at + (v_lane ^ (db * 64));
    if (look) {
      // Rows that do not see all of this tile weigh some of V by 0, which infinities and
      // NaN survive: 0 times the tile tells whether it has any.
      f16v z = f16v{};
#pragma unroll
      for (int kk = 0; kk < KW / 16; ++kk)
#pragma unroll
        for (int db = 0; db < DB; ++db) z = E::mma(v_frag(v[db], kk), frag{}, z);
      float t = 0.0f;
#pragma unroll
      for (int r = 0; r < 16; ++r) t += z[r];
      odd = odd || t != 0.0f;
    }
#pragma unroll
    for (int kk = 0; kk < KW / 16; ++kk)
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] = E::mma(v_frag(v[db], kk), p[kk], o[db]);
    ahead<KW / 16 * DB, 2>();
  };
  // The same key by key, each added only to the rows that see it. (Weights that round to 0 are -0
  // there, as an infinity or NaN counts with any weight; those of hidden keys are +0.)
  auto values_apart = [&](int buf) __attribute__((always_inline)) {
    lds_byte* const at = lds0 + v_at + buf * L::kTile;
#pragma unroll
    for (int kk = 0; kk < KW / 16; ++kk)
#pragma unroll 1
      for (int key = 0; key < 16; ++key) {
        const int of = (key >> 2) & 1, j = (key & 3) | ((key >> 1) & 4);  // its half and element
        u4 keep;
#pragma unroll
        for (int e = 0; e < 4; ++e) keep[e] = half != of || j >> 1 != e ? 0u : j & 1 ? 0xffff0000u : 0x0000ffffu;
        const u4 one = __builtin_bit_cast(u4, p[kk]) & keep;
        const float sees = halves_max((one[0] | one[1] | one[2] | one[3]) != 0 ? 1.0f : 0.0f);
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const u4 x = __builtin_bit_cast(u4, v_frag(at + (v_lane ^ (db * 64)), kk)) & keep;
          const f16v c = E::mma(__builtin_bit_cast(frag, x), __builtin_bit_cast(frag, one), f16v{});
#pragma unroll
          for (int r = 0; r < 16; ++r) o[db][r] += sees != 0.0f ? c[r] : 0.0f;
        }
      }
  };

  // -- scores to weights -----------------------------------------------------------------
  auto weights = [&](auto apart, int buf, int k0, bool partial, int t_dmin, int t_dmax) __attribute__((always_inline)) {
    const int key0 = k0 + 4 * half;  // key of element r of block kb: key0 + 32 kb + 8 (r / 4) + r % 4
    const float unit = a.c.cap > 0 ? 1.0f : a.c.scale * kLog2e;  // what scores are still to be scaled by
    if (SHAPE == kCap || SHAPE == kLarge || (SHAPE == kAny && a.c.cap > 0)) {
      float far = 0.0f;
      if constexpr (SHAPE != kAny) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) far = fmaxf(far, fabsf(s[kb][r]));
      }
      if (SHAPE != kAny && !__any(!(far <= a.cap_reach))) {
        // x = score / cap below 0.6: tanh x / x as a polynomial of x^2 (Chebyshev fit, off by
        // less than 8e-8), six plain operations where the exponential and the reciprocal
        // take a quarter of the rate each.
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[kb][r] = cap_near(a, s[kb][r]);
      } else {
        // cap tanh x = cap - 2 cap / (exp(2 x) + 1), in the base of 2, off by some 2^-22 of the cap.
        const float in = a.cap_in, out = a.cap_out;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float x = s[kb][r];
            const float e = __builtin_amdgcn_exp2f(x * in);
            const float y = __builtin_fmaf(-2.0f * out, __builtin_amdgcn_rcpf(e + 1.0f), out);
            s[kb][r] = SHAPE == kLarge && fabsf(x) <= a.cap_reach ? cap_near(a, x) : y;
          }
      }
    }
    if constexpr (SHAPE >= kAny) {
      // The loops below are whole loops a branch: a uniform branch inside would be taken
      // for every score.
      const int4* const codes = reinterpret_cast<const int4*>(more + L::kCode + buf * 256 + wk * 4) + half;
      auto bias = [&](auto coded, int from, auto add) __attribute__((always_inline)) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            int4 c{};
            if constexpr (decltype(coded)::value) c = codes[8 * kb + 2 * g];
            const int ck[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
              s[kb][4 * g + e] =
                  add(s[kb][4 * g + e], decltype(coded)::value ? from - ck[e] : from - key0 - (32 * kb + 8 * g + e));
          }
      };
      if (a.c.slopes) {
        auto add = [&](float x, int diff) __attribute__((always_inline)) {
          return __builtin_fmaf(x, unit, -slope * fabsf((float)diff));
        };
        if (code_k)
          bias(std::true_type{}, cq, add);
        else {
          const float first = (float)(cq - key0);
#pragma unroll
          for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              s[kb][r] = __builtin_fmaf(s[kb][r], unit, -slope * fabsf(first - (float)(32 * kb + 8 * (r / 4) + r % 4)));
        }
      }
      if (table) {
        const float by = a.c.slopes ? 1.0f : unit;
        const int last = a.c.table_len - 1, zero = a.c.table_zero;
        if (a.table_lds) {
          // Entries in the base of 2.
          const float* const t = reinterpret_cast<const float*>(more + L::kTable) + g_head * a.c.table_len;
          auto add = [&](float x, int diff) __attribute__((always_inline)) {
            return __builtin_fmaf(x, by, t[min(max(diff, 0), last)]);
          };
          auto add_hidden = [&](float x, int diff) __attribute__((always_inline)) {
            const float entry = t[min(max(diff, 0), last)];
            const float sum = __builtin_fmaf(x, by, entry);
            return entry == -__builtin_inff() ? entry : sum;
          };
          if (hides)
            code_k ? bias(std::true_type{}, cq + zero, add_hidden) : bias(std::false_type{}, cq + zero, add_hidden);
          else
            code_k ? bias(std::true_type{}, cq + zero, add) : bias(std::false_type{}, cq + zero, add);
        } else {
          const float* const t = table + (int64_t)head * a.c.table_len;
          auto add = [&](float x, int diff) __attribute__((always_inline)) {
            const float entry = entry_of(t[min(max(diff, 0), last)]);
            const float sum = __builtin_fmaf(x, by, entry);
            return entry == -__builtin_inff() ? entry : sum;
          };
          code_k ? bias(std::true_type{}, cq + zero, add) : bias(std::false_type{}, cq + zero, add);
        }
      }
      if (!a.c.slopes && !table && unit != 1.0f) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[kb][r] *= unit;
      }
    }
    if (partial) {
      const bool whole = k0 + KW <= pre || (k0 >= w_lo_max && k0 + KW <= w_hi_min);
      if (!whole) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int key = key0 + 32 * kb + 8 * (r / 4) + r % 4;
            s[kb][r] = (key >= lo && key < hi) || key < pre ? s[kb][r] : -__builtin_inff();
          }
      }
      if (doc_k && t_dmin == t_dmax) {
        const float away = t_dmin == dq ? 0.0f : 1.0f;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[kb][r] = away != 0.0f ? -__builtin_inff() : s[kb][r];
      } else if (doc_k) {
        const int4* const docs = reinterpret_cast<const int4*>(more + L::kDoc + buf * 256 + wk * 4) + half;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const int4 d = docs[8 * kb + 2 * g];
            s[kb][4 * g] = d.x == dq ? s[kb][4 * g] : -__builtin_inff();
            s[kb][4 * g + 1] = d.y == dq ? s[kb][4 * g + 1] : -__builtin_inff();
            s[kb][4 * g + 2] = d.z == dq ? s[kb][4 * g + 2] : -__builtin_inff();
            s[kb][4 * g + 3] = d.w == dq ? s[kb][4 * g + 3] : -__builtin_inff();
          }
      }
    }

    float top = s[0][0];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[kb][r]);
    top = halves_max(top);
    // The base of a row's exponents follows its largest score only where that has grown
    // by more than 2^8: until then weights are at most 256, and nothing is rescaled.
    if (__any((top - m) * mul > 8.0f)) {
      const float next = fmaxf(m, top);
      // A row that has seen nothing yet has no sums to keep (next may be -inf as well).
      const float f = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((m - next) * mul);
      m = next;
      l *= f;
#pragma unroll
      for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] *= f;
    }
    // fp16's weights are raised to the top of its range, so that small ones, of which a long
    // walk adds up many, keep their digits down to 2^-21 of a row's largest and are 0 below 2^-32.
    const float base = (m == -__builtin_inff() ? 0.0f : m * mul) - E::kRaise;
    float sum = 0.0f;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float x = s[kb][r], w = __builtin_amdgcn_exp2f(__builtin_fmaf(x, mul, -base));
        sum += w;
        s[kb][r] = decltype(apart)::value && w <= E::kZero && x != -__builtin_inff() ? -0.0f : w;
      }
    l += sum;  // this half's keys; the halves are added at the end
#pragma unroll
    for (int kk = 0; kk < KW / 16; ++kk) {
      const f16v x = s[kk / 2];
      p[kk] = kk & 1
                  ? __builtin_convertvector(__builtin_shufflevector(x, x, 8, 9, 10, 11, 12, 13, 14, 15), frag)
                  : __builtin_convertvector(__builtin_shufflevector(x, x, 0, 1, 2, 3, 4, 5, 6, 7), frag);
    }
  };

  // -- the walk ------------------------------------------------------------------------
  // One barrier a tile. While tile t's scores and the previous tile's values are
  // multiplied, K of the next tile and V of this one are on their way to the buffers
  // that the last barrier freed. (Three buffers, two tiles' loads on their way, were no
  // faster anywhere, and take the LDS of a second workgroup.)
  auto walk = [&](auto apart) __attribute__((always_inline)) {
    const int chunk = doc_k ? L::kChunk : max(end - begin, 1);
    for (int c0 = begin; c0 < end; c0 += chunk) {
      const int c1 = min(end, c0 + chunk);
      lds_sync();  // the last chunk's tiles and bits have been used
      if (doc_k) {
        // Tiles whose documents cannot be a row's are not read: a lane looks at the range
        // of one tile, a wave at 64.
        for (int w = wave; w < (c1 - c0 + 63) / 64; w += NW) {
          const int at = c0 + w * 64 + lane;
          const int2 r = at < c1 ? doc_ranges[tile_of(at)] : int2{INT32_MAX, INT32_MIN};
          tile_docs[w * 64 + lane] = r;
          const uint64_t in = __ballot(r.y >= dmin && r.x <= dmax);
          if (lane == 0) any[w] = in;
        }
        lds_sync();
      }
      auto next = [&](int i) __attribute__((always_inline)) {
        if (doc_k)
          while (i < c1) {
            const uint64_t left = any[(i - c0) >> 6] >> ((i - c0) & 63);
            if (left != 0) {
              i += __builtin_ctzll(left);
              break;
            }
            i = c0 + (((i - c0) >> 6) + 1) * 64;
          }
        return scalar(min(i, c1));
      };
      int i = next(c0);
      const bool nothing = i >= c1;
      if (!nothing) stage_k(0, tile_of(i));
      if (table && a.table_lds && !decltype(apart)::value && c0 == begin) load_table();
      if (nothing) continue;
      vm_wait();
      lds_sync();
      int buf = 0;
      bool has = false, look = false;  // weights of the previous tile; some row sees not all of it
      while (true) {
        const bool live = i < c1;
        const int tile = tile_of(i), k0 = tile * KT + wk, k1 = k0 + KW;
        bool seen = false, partial = false;
        int t_dmin = w_dmin, t_dmax = w_dmin, following = i;
        if (live) {
          if (doc_k) {
            const int2 r = tile_docs[i - c0];
            t_dmin = scalar(r.x);
            t_dmax = scalar(r.y);
          }
          following = next(i + 1);
          if (following < c1) stage_k(buf ^ 1, tile_of(following));
          stage_v(buf, tile);
          seen = w_real && (k0 < pre || (k0 < w_hi_max && k1 > w_lo_min)) &&
                 (!doc_k || (t_dmax >= w_dmin && t_dmin <= w_dmax));
          partial = !(k1 <= pre || (k0 >= w_lo_max && k1 <= w_hi_min)) ||
                    (doc_k && !(t_dmin == t_dmax && w_dmin == w_dmax));
        }
        if (seen) scores(buf);
        if (has) {
          if constexpr (decltype(apart)::value)
            values_apart(buf ^ 1);
          else
            values(buf ^ 1, look);
        }
        if (!live) break;
        if (seen) weights(apart, buf, k0, partial, t_dmin, t_dmax);
        has = seen;
        look = partial || hides;
        vm_wait();
        lds_sync();
        i = following;
        buf ^= 1;
      }
    }
  };
  walk(std::false_type{});
  // A workgroup that met such a tile starts over and takes the keys one by one. (Rarely, and so it
  // is called: this and `wide` hold scalar registers against the loop otherwise, 465 us for 450
  // in windows.)
  {
    int* const flag = reinterpret_cast<int*>(more + L::kRange);
    lds_sync();
    if (lane == 0) flag[wave] = 0;
    if (odd) flag[wave] = 1;
    lds_sync();
    int again = 0;
    for (int i = 0; i < NW; ++i) again |= flag[i];
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(again) != 0, 0)) {
#pragma unroll
      for (int i = 0; i < DB; ++i) o[i] = f16v{};
      m = -__builtin_inff();
      l = 0.0f;
      walk(std::true_type{});
    }
  }

  // -- results -------------------------------------------------------------------------
  l = halves_sum(l);
  if constexpr (SHARED) {
    // The other waves hand their sums to the first, one after the other.
    float* const box = reinterpret_cast<float*>(lds);
    for (int w = 1; w < NW; ++w) {
      lds_sync();  // the tiles, and the last wave's sums, have been used
      if (wave == w) {
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<f4*>(box + ((i * 4 + g) * 64 + lane) * 4) =
                f4{o[i][4 * g], o[i][4 * g + 1], o[i][4 * g + 2], o[i][4 * g + 3]};
        box[DB * 1024 + lane] = m;
        box[DB * 1024 + 64 + lane] = l;
      }
      lds_sync();
      if (wave == 0) {
        const float m2 = box[DB * 1024 + lane], next = fmaxf(m, m2);
        const float f1 = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((m - next) * mul);
        const float f2 = m2 == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f((m2 - next) * mul);
        m = next;
        l = l * f1 + box[DB * 1024 + 64 + lane] * f2;
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const f4 x = *reinterpret_cast<const f4*>(box + ((i * 4 + g) * 64 + lane) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][4 * g + e] = o[i][4 * g + e] * f1 + x[e] * f2;
          }
      }
    }
    if (wave != 0) return;
  }
  if (a.splits > 1) {
    if (!real) return;
    // A range without keys leaves no sums; the join weighs it by 0 and does not use them.
    const int64_t at = ((int64_t)split * a.c.batch * a.c.k_heads + bh) * a.rows + row;
    float* const p = a.part + at * a.c.head_dim;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = db * 32 + 8 * g + 4 * half;
        if (begin < end && d < a.c.head_dim)
          *reinterpret_cast<f4*>(p + d) = f4{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]};
      }
    if (half == 0) {
      a.stat[2 * at] = m * mul - E::kRaise;
      a.stat[2 * at + 1] = l;
    }
    return;
  }
  const float scale = l == 0.0f ? 0.0f : 1.0f / l;
  T* const op = static_cast<T*>(a.c.out) + b * a.c.out_stride[0] + token * a.c.out_stride[1] +
                head * a.c.out_stride[2];
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
      if (real && d < a.c.head_dim) *reinterpret_cast<u4*>(op + d) = u4{x[0], y[0], x[1], y[1]};
    }
  if (a.c.lse && real && half == 0)
    a.c.lse[((int64_t)b * a.c.q_heads + head) * a.c.q_tokens + token] =
        (m * mul - E::kRaise + __builtin_amdgcn_logf(l)) * kLn2;
}

// Smallest and largest document of each tile of keys: a wave a tile. (Looked over by
// every workgroup instead, the documents of 16384 keys took each some 30 us.)
__global__ void __launch_bounds__(256) attention_docs(AttnArgs a, int2* out, int64_t first_block, int64_t total) {
  const int64_t at = (first_block + blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (at >= total) return;
  const int lane = threadIdx.x & 63;
  const int64_t b = at / a.doc_tiles, first = (at - b * a.doc_tiles) * a.doc_tile;
  int lo = INT32_MAX, hi = INT32_MIN;
  if (lane < a.doc_tile && first + lane < a.c.k_tokens)
    lo = hi = a.c.doc_k[b * a.c.doc_k_stride + first + lane];
  lo = wave_min(lo);
  hi = wave_max(hi);
  if (lane == 0) out[at] = int2{lo, hi};
}

// Joins the ranges of the keys, a workgroup a row: four values a thread, so that D / 4
// threads read a range's sums and 1024 / D ranges are read at once. Sums are added in a
// fixed order.
template <class T>
__global__ void __launch_bounds__(256) attention_join(AttnArgs a) {
  __shared__ float weight[64];
  __shared__ f4 sums[256];
  const int64_t total = (int64_t)a.c.batch * a.c.k_heads * a.rows;
  const int64_t at = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 63;
  const int D = a.c.head_dim, quads = D / 4, steps = 256 / quads;
  const int step = tid / quads, quad = tid - step * quads;
  // Every wave looks at the statistics of all ranges (at most 64), a lane each.
  const bool in = lane < a.splits;
  const float2 st = in ? *reinterpret_cast<const float2*>(a.stat + 2 * (lane * total + at))
                       : float2{-__builtin_inff(), 0.0f};
  f4 o = f4{};
  const float* const p = a.part + at * D + 4 * quad;
  const float top = over_wave(st.x, [](float a, float b) { return fmaxf(a, b); });
  const float base = top == -__builtin_inff() ? 0.0f : top;
  const float w = in ? __builtin_amdgcn_exp2f(st.x - base) : 0.0f;
  const float l = over_wave(w * st.y, [](float a, float b) { return a + b; });
  if (tid < 64) weight[tid] = w;
  lds_sync();
  if (step < steps) {
#pragma unroll 4
    for (int s = step; s < a.splits; s += steps) {
      const float ws = weight[s];
      const f4 x = *reinterpret_cast<const f4*>(p + s * total * D);
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = ws != 0.0f ? __builtin_fmaf(ws, x[e], o[e]) : o[e];
    }
    sums[tid] = o;
  }
  lds_sync();
  const int64_t bh = at / a.rows;
  const int row = (int)(at - bh * a.rows);
  const int b = (int)fdiv((uint32_t)bh, a.by_k_heads), kh = (int)(bh - (int64_t)b * a.c.k_heads);
  const int token = (int)fdiv((uint32_t)row, a.by_group), head = kh * a.group + row - token * a.group;
  if (tid < quads) {
    const int n = min(steps, a.splits);
    for (int s = 1; s < n; ++s) o += sums[s * quads + tid];
    const float scale = l == 0.0f ? 0.0f : 1.0f / l;
    T* const op = static_cast<T*>(a.c.out) + b * a.c.out_stride[0] + token * a.c.out_stride[1] +
                  head * a.c.out_stride[2];
    typedef T t4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = in_range<T>(o[e] * scale);
    *reinterpret_cast<t4*>(op + 4 * tid) = __builtin_convertvector(o, t4);
  }
  if (a.c.lse && tid == 0)
    a.c.lse[((int64_t)b * a.c.q_heads + head) * a.c.q_tokens + token] =
        (top + __builtin_amdgcn_logf(l)) * kLn2;
}

// The same for up to eight ranges of many rows: D / 4 threads a row, which read its ranges
// one after the other. (A workgroup a row took 41 us for 30740 rows of 80 in four ranges.)
template <class T>
__global__ void __launch_bounds__(256) attention_join_few(AttnArgs a) {
  const int64_t total = (int64_t)a.c.batch * a.c.k_heads * a.rows;
  const int D = a.c.head_dim, quads = D / 4, rows = 256 / quads;
  const int slot = threadIdx.x / quads, quad = threadIdx.x - slot * quads;
  const int64_t at = (int64_t)blockIdx.x * rows + slot;
  if (slot >= rows || at >= total) return;
  float2 st[8];
  f4 x[8];
  float top = -__builtin_inff();
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    if (s >= a.splits) break;
    st[s] = *reinterpret_cast<const float2*>(a.stat + 2 * (s * total + at));
    x[s] = *reinterpret_cast<const f4*>(a.part + (s * total + at) * D + 4 * quad);
  }
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    if (s >= a.splits) break;
    top = fmaxf(top, st[s].x);
  }
  const float base = top == -__builtin_inff() ? 0.0f : top;
  float l = 0.0f;
  f4 o = f4{};
#pragma unroll
  for (int s = 0; s < 8; ++s) {
    if (s >= a.splits) break;
    const float w = __builtin_amdgcn_exp2f(st[s].x - base);
    l = __builtin_fmaf(w, st[s].y, l);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = w != 0.0f ? __builtin_fmaf(w, x[s][e], o[e]) : o[e];
  }
  const uint32_t bh = fdiv((uint32_t)at, a.by_rows);
  const int row = (int)at - (int)bh * a.rows;
  const int b = (int)fdiv(bh, a.by_k_heads), kh = (int)bh - b * a.c.k_heads;
  const int token = (int)fdiv((uint32_t)row, a.by_group), head = kh * a.group + row - token * a.group;
  const float scale = l == 0.0f ? 0.0f : 1.0f / l;
  T* const op = static_cast<T*>(a.c.out) + b * a.c.out_stride[0] + token * a.c.out_stride[1] +
                head * a.c.out_stride[2];
  typedef T t4 __attribute__((ext_vector_type(4)));
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = in_range<T>(o[e] * scale);
  *reinterpret_cast<t4*>(op + 4 * quad) = __builtin_convertvector(o, t4);
  if (a.c.lse && quad == 0)
    a.c.lse[((int64_t)b * a.c.q_heads + head) * a.c.q_tokens + token] =
        (top + __builtin_amdgcn_logf(l)) * kLn2;
}

struct TilePick {
  void (*fn)(AttnArgs);
  int threads;
  int bytes;  // of LDS
  int chunk;  // tiles whose documents' ranges it keeps
};

template <class T, int DP, int KT, int NW, bool SHARED>
TilePick pick(Shape shape) {
  return {shape == kPlain ? attention_tile<T, DP, KT, NW, SHARED, kPlain>
          : shape == kCap ? attention_tile<T, DP, KT, NW, SHARED, kCap>
          : shape == kAny ? attention_tile<T, DP, KT, NW, SHARED, kAny>
                          : attention_tile<T, DP, KT, NW, SHARED, kLarge>,
          NW * 64, TileL<DP, KT>::kBytes, TileL<DP, KT>::kChunk};
}

template <class T>
TilePick pick(int d, bool shared, Shape shape) {
  if (shared) {
    if (d <= 32) return pick<T, 32, 32, 1, true>(shape);
    if (d <= 64) return pick<T, 64, 32, 1, true>(shape);
    if (d <= 96) return pick<T, 96, 32, 1, true>(shape);
    if (d <= 128) return pick<T, 128, 32, 1, true>(shape);
    return pick<T, 256, 64, 2, true>(shape);
  }
  if (d <= 32) return pick<T, 32, 64, 4, false>(shape);
  if (d <= 64) return pick<T, 64, 64, 4, false>(shape);
  if (d <= 96) return pick<T, 96, 64, 4, false>(shape);
  if (d <= 128) return pick<T, 128, 64, 4, false>(shape);
  return pick<T, 256, 32, 4, false>(shape);
}

// Up to 32 rows are one wave's, or above heads of 128 two waves', which divide the keys; of more rows
// each of four waves takes 32.
bool shared_rows(const arthip_attention_args& c) {
  return (int64_t)c.q_tokens * (c.q_heads / c.k_heads) <= 32;
}
int tile_rows(const arthip_attention_args& c) { return shared_rows(c) ? 32 : 128; }
int tile_keys(const arthip_attention_args& c) { return (c.head_dim > 128) == shared_rows(c) ? 64 : 32; }

}  // namespace

AttnPlan attention_plan(const arthip_attention_args& c) {
  AttnPlan p{1, 1, 0};
  if (c.batch == 0 || c.q_tokens == 0 || c.q_heads == 0) return p;
  const int64_t rows = (int64_t)c.q_tokens * (c.q_heads / c.k_heads);
  const int per = tile_rows(c), kt = tile_keys(c);
  const int64_t row_tiles = (rows + per - 1) / per;
  const int64_t items = (int64_t)c.batch * c.k_heads * row_tiles;
  // Tiles that a row tile can need at most: a window on both sides bounds them.
  int64_t tiles = (c.k_tokens + kt - 1) / kt;
  if (c.left >= 0 && c.right >= 0 && c.prefix == nullptr)
    tiles = std::min<int64_t>(tiles, ((int64_t)c.left + c.right + std::min<int64_t>(c.q_tokens, per)) / kt + 2);
  // Ranges: enough workgroups for the chip (one-wave workgroups fit a CU four at a time,
  // those of four waves two), of at least four tiles. From half of that number on walks of 32
  // tiles or more are divided where the halves take fewer turns of the chip than half of the
  // whole ones', by the workgroups that it holds at once: with four waves two a CU, three for
  // heads of up to 64 (with a bias 32), one above 128. Whole and halved, us:
  //   four waves, heads of 128: 256 items 32 tiles 65, 56; 260 items 70, 87, 64 tiles 131, 150
  //   heads of 64: 300 items 64 tiles 95, 79; 400 items 95, 114. Of 256: 260 items 287, 248; 400 288, 331
  //   one wave, heads of 128: 512 items 32 tiles 51, 49; 520 items 52, 68. Of 64: 640 items 64 tiles
  //   73, 70; 704 items 79, 83. Of 32: 640 items 64 tiles 55, 59, 128 tiles 125, 112
  const bool shared = shared_rows(c);
  const int64_t want = shared ? 1024 : 512;
  const bool biased = c.slopes != nullptr || c.table != nullptr || c.cap > kCapSmall;
  const bool five = c.head_dim == 64 || (c.head_dim <= 32 && tiles >= 128);
  const int64_t slots = c.head_dim > 128 ? 256
                        : shared         ? (five ? 1280 : 1024)
                                         : (c.head_dim <= (biased ? 32 : 64) ? 768 : 512);
  const bool halve = tiles >= 32 && (2 * items + slots - 1) / slots < 2 * ((items + slots - 1) / slots);
  if (items < want / 2 || (items < want && halve))
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({(want + items - 1) / items, tiles / 4, 64}));
  p.range = (int)std::max<int64_t>(1, (tiles + p.splits - 1) / p.splits);
  if (p.splits > 1)
    p.workspace = (size_t)p.splits * c.batch * c.k_heads * rows * (c.head_dim + 2) * sizeof(float);
  if (c.doc_k != nullptr) {
    const int64_t n = (c.k_tokens + tile_keys(c) - 1) / tile_keys(c);
    p.workspace += (size_t)(c.doc_k_stride == 0 ? 1 : c.batch) * n * sizeof(int2);
  }
  return p;
}

hipError_t launch_attention(const arthip_attention_args& c, hipStream_t s) {
  if (c.batch == 0 || c.q_tokens == 0 || c.q_heads == 0) return hipSuccess;
  AttnArgs a{};
  a.c = c;
  if (c.k_tokens == 0)  // nothing to compare: one side of a pair may be missing
    a.c.doc_q = a.c.doc_k = a.c.code_q = a.c.code_k = nullptr;
  a.group = c.q_heads / c.k_heads;
  a.rows = c.q_tokens * a.group;
  const bool shared = shared_rows(c);
  a.row_tiles = (a.rows + tile_rows(c) - 1) / tile_rows(c);
  const AttnPlan plan = attention_plan(c);
  a.splits = plan.splits;
  a.range = plan.range;
  a.items = c.batch * c.k_heads * a.row_tiles * a.splits;
  a.by_group = make_fastdiv((uint32_t)a.group);
  a.by_k_heads = make_fastdiv((uint32_t)c.k_heads);
  a.by_row_tiles = make_fastdiv((uint32_t)a.row_tiles);
  a.by_splits = make_fastdiv((uint32_t)a.splits);
  a.by_rows = make_fastdiv((uint32_t)a.rows);
  const int64_t total = (int64_t)c.batch * c.k_heads * a.rows;
  a.part = static_cast<float*>(c.workspace);
  if (a.splits > 1) a.stat = a.part + a.splits * total * c.head_dim;
  const bool f16 = c.dtype == ARTHIP_TYPE_F16;
  const Shape shape = c.cap > kCapSmall                                                  ? kLarge
                      : c.slopes != nullptr || c.table != nullptr || !(c.scale > 0) ? kAny
                      : c.cap > 0                                                   ? kCap
                                                                                    : kPlain;
  const TilePick k = f16 ? pick<_Float16>(c.head_dim, shared, shape) : pick<__bf16>(c.head_dim, shared, shape);
  if (c.cap > 0) {
    // A cap near 0 takes these past their type's end: a coefficient that is no number leaves
    // all scores to the other form, squares stay below infinity (as 0 times it is NaN), and a
    // score of 0 meets a finite factor. One above 1e30 changes no score below 4e26.
    constexpr double top = std::numeric_limits<float>::max();
    const double cap = std::min<double>(c.cap, 1e30), r = c.scale / cap;
    bool fits = true;
    for (int i = 0; i < 5; ++i) {
      a.cap_fit[i] = (float)(kTanh[i] * std::pow(r, 2 * i) * c.scale * kLog2e);
      fits = fits && std::isfinite(a.cap_fit[i]);
    }
    a.cap_reach = fits ? (float)std::min(0.6 / std::fabs(r), 1e19) : -1.0f;
    a.cap_in = (float)std::min(std::max(2.0 * kLog2e * r, -top), top);
    a.cap_out = (float)(kLog2e * cap);
  }
  if (a.c.doc_k != nullptr) {
    a.doc_tile = tile_keys(c);
    a.doc_tiles = (c.k_tokens + a.doc_tile - 1) / a.doc_tile;
    int2* const ranges = reinterpret_cast<int2*>(a.splits > 1 ? a.stat + 2 * a.splits * total : a.part);
    const int64_t n = (int64_t)(c.doc_k_stride == 0 ? 1 : c.batch) * a.doc_tiles;
    a.doc_ranges = ranges;
    const hipError_t e = launch_parts((n + 3) / 4, 256, [&](int64_t first, unsigned count) {
      hipLaunchKernelGGL(attention_docs, dim3(count), dim3(256), 0, s, a, ranges, first, n);
      return hipGetLastError();
    });
    if (e != hipSuccess) return e;
  }
  const int64_t table = c.table == nullptr ? 0 : (int64_t)a.group * c.table_len * 4;
  a.table_lds = table <= kTableBytes;
  // Offsets of a tile's keys from its first one have 31 bits.
  const int64_t far = std::max(std::abs(c.k_stride[1]), std::abs(c.v_stride[1]));
  a.wide = c.k_stride[1] < 0 || c.v_stride[1] < 0 || far * 2 * 64 + 512 > INT32_MAX;
  a.table_bytes = a.table_lds ? (int)(table + 7) / 8 * 8 : 0;
  const int bytes = k.bytes + a.table_bytes + (a.c.doc_k != nullptr ? k.chunk * 8 : 0);
  hipError_t e = hipSuccess;
  if (bytes > 65536)  // what a kernel may have without asking
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(k.fn), hipFuncAttributeMaxDynamicSharedMemorySize,
                            bytes);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k.fn, dim3((unsigned)((a.items + 7) / 8 * 8)), dim3((unsigned)k.threads), bytes, s, a);
  e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  if (a.splits <= 8 && total >= 512) {
    const int rows = 256 / (c.head_dim / 4);
    hipLaunchKernelGGL(f16 ? attention_join_few<_Float16> : attention_join_few<__bf16>,
                       dim3((unsigned)((total + rows - 1) / rows)), dim3(256), 0, s, a);
    return hipGetLastError();
  }
  hipLaunchKernelGGL(f16 ? attention_join<_Float16> : attention_join<__bf16>,
                     dim3((unsigned)total), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace arthip

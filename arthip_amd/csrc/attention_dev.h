// Device helpers of the attention kernels: matrix products of 32 x 32 x 16 by element
// type, exchanges inside a wave, tiles of keys and values in LDS and the loads that bring
// them there, capped scores.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <limits>
#include <type_traits>

#include "token_dev.h"

namespace arthip {

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

// A cap on scores, cap tanh(scale x / cap), in the base of 2: as a polynomial of x up to `reach`, as
// cap - 2 cap / (exp(2 scale x / cap) + 1) with the factors `in` and `out` elsewhere.
struct CapFit {
  float reach;
  float fit[5];
  float in, out;
};

// A score x up to 0.6 caps.
__device__ __forceinline__ float cap_near(const CapFit& c, float x) {
  const float z = x * x;
  float t = __builtin_fmaf(c.fit[4], z, c.fit[3]);
  t = __builtin_fmaf(t, z, c.fit[2]);
  t = __builtin_fmaf(t, z, c.fit[1]);
  t = __builtin_fmaf(t, z, c.fit[0]);
  return x * t;
}

// The factors for a cap above 0.
inline CapFit make_cap(float given, float scale) {
  CapFit c;
  // A cap near 0 takes these past their type's end: a coefficient that is no number leaves
  // all scores to the other form, squares stay below infinity (as 0 times it is NaN), and a
  // score of 0 meets a finite factor. One above 1e30 changes no score below 4e26.
  constexpr double top = std::numeric_limits<float>::max();
  const double cap = std::min<double>(given, 1e30), r = scale / cap;
  bool fits = true;
  for (int i = 0; i < 5; ++i) {
    c.fit[i] = (float)(kTanh[i] * std::pow(r, 2 * i) * scale * kLog2e);
    fits = fits && std::isfinite(c.fit[i]);
  }
  c.reach = fits ? (float)std::min(0.6 / std::fabs(r), 1e19) : -1.0f;
  c.in = (float)std::min(std::max(2.0 * kLog2e * r, -top), top);
  c.out = (float)(kLog2e * cap);
  return c;
}

template <class T>
struct Elem;
template <>
struct Elem<_Float16> {
  typedef h8 frag;
  static constexpr float kZero = 0x1p-25f;  // numbers of 0 and more up to here round to 0
  // The power of 2 that weights are raised by, so that small ones, of which a long walk adds up many, keep
  // their digits: those of a row's base are 2^7, and as a base is kept up to 2^8 below the row's largest
  // score, weights are up to 2^15.
  static constexpr float kRaise = 7.0f;
  static constexpr float kMost = 0x1p+15f;  // sum of weights that each are numbers of the type
  static __device__ __forceinline__ f16v mma(h8 a, h8 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Elem<__bf16> {
  typedef b8 frag;
  static constexpr float kZero = 0.0f;  // as the exponential's are 2^-126 or more, or 0
  static constexpr float kRaise = 0.0f;
  static constexpr float kMost = 0x1p+10f;  // values up to 2^-10 of the type's largest stay finite
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
// The same with everything but the buffer's address in the lanes' offsets.
template <int N>
__device__ __forceinline__ void load_lds16(rsrc_t from, const uint32_t (&at)[N], uint32_t to) {
  static_assert(N == 1 || N == 2 || N == 4, "KiB that the constant reaches");
  if constexpr (N == 1)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %2, %1, 0 offen lds"
                 :
                 : "s"(to), "s"(from), "v"(at[0])
                 : "memory");
  else if constexpr (N == 2)
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %2, %1, 0 offen lds\n\t"
        "buffer_load_dwordx4 %3, %1, 0 offen offset:1024 lds"
        :
        : "s"(to), "s"(from), "v"(at[0]), "v"(at[1])
        : "memory");
  else
    asm volatile(
        "s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %2, %1, 0 offen lds\n\t"
        "buffer_load_dwordx4 %3, %1, 0 offen offset:1024 lds\n\t"
        "buffer_load_dwordx4 %4, %1, 0 offen offset:2048 lds\n\t"
        "buffer_load_dwordx4 %5, %1, 0 offen offset:3072 lds"
        :
        : "s"(to), "s"(from), "v"(at[0]), "v"(at[1]), "v"(at[2]), "v"(at[3])
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

// A mean of finite values stays in their type's range: the weights' rounding (2^-11) can take one of
// fp16's largest numbers out of it.
template <class T>
__device__ __forceinline__ float in_range(float x) {
  if constexpr (std::is_same_v<T, _Float16>)
    return fabsf(x) < __builtin_inff() ? __builtin_amdgcn_fmed3f(x, -65504.0f, 65504.0f) : x;
  return x;
}

}  // namespace arthip

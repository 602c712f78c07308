// The attention weight that cached keys gather (arthip_key_weights): for each slot the sum of
// exp(score - lse) over the new tokens that see it and the query heads that share its key head.
//
// A workgroup owns a run of slots of one key head and walks all rows (token, head) that see them, so
// that nothing is added across workgroups but in a fixed order. Each wave keeps its keys in
// registers as the left operand of S^T = K Q^T (v_mfma_f32_32x32x16); the rows pass through LDS in
// tiles of 64, which all waves share. A lane's accumulator holds 16 keys of one row, whose lse is
// one number a lane: a weight is one multiply-add, one exponential and one addition to the key's
// own sum, and sums meet across the lanes once, at the end.

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
  int items;   // all workgroups
  FastDiv by_group, by_page, by_heads, by_tiles, by_splits;
  CapFit cap;
  float* part;  // [splits][batch * k_heads][slots], if splits > 1
};

constexpr int kRows = 64;  // of a tile

__device__ __forceinline__ float started(const KeyArgs& a, const Sequence& s, int b, int head, int slot) {
  if (slot >= s.start() || a.c.decay == 0.0f) return 0.0f;
  return a.c.decay * a.c.weights[b * a.c.weights_stride[0] + head * a.c.weights_stride[1] + slot];
}

// Sum of x over the 32 lanes of a half, in each of them.
__device__ __forceinline__ float half_sum(float x) {
  auto dpp = [&](auto control) __attribute__((always_inline)) {
    const int y = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(control)::value, 0xf, 0xf, true);
    x += __builtin_bit_cast(float, y);
  };
  dpp(std::integral_constant<int, 0xb1>{});
  dpp(std::integral_constant<int, 0x4e>{});
  dpp(std::integral_constant<int, 0x141>{});
  dpp(std::integral_constant<int, 0x140>{});
  const uint32_t u = __builtin_bit_cast(uint32_t, x);
  const u2 r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t r0 = r[0], r1 = r[1];
  return __builtin_bit_cast(float, r0) + __builtin_bit_cast(float, r1);
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
  const uint32_t lds_base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char*)lds;

  const arthip_pages& pg = a.c.p;
  auto scalar = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  // Each XCD takes an eighth of the items in a row: those of one key head share the queries.
  const int bid = (int)blockIdx.x, per = (int)gridDim.x >> 3;
  const int item = (bid & 7) * per + (bid >> 3);
  if (item >= a.items) return;
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
  const int start = seq.start();
  const int k0 = tile * 128 * KB, k1 = min(k0 + 128 * KB, min(seq.len, a.c.slots));
  const int w0 = k0 + wave * 32 * KB;  // the wave's first key

  // -- the rows that see some of the keys ------------------------------------------------
  const int t_lo = a.c.causal ? min(max(k0 - start, 0), seq.tokens) : 0;
  const int t_hi = a.c.left < 0 ? seq.tokens : (int)min(max((int64_t)k1 + a.c.left - start, (int64_t)t_lo), (int64_t)seq.tokens);
  const int all = k1 > k0 ? (t_hi - t_lo) * a.group : 0;
  const int steps = (all + kRows - 1) / kRows;
  const int share = (steps + a.splits - 1) / a.splits;
  const int first = min(split * share, steps), last = min(first + share, steps);
  const int row0 = t_lo * a.group, row_end = row0 + all;

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
  auto stage = [&](int buf, int step) __attribute__((always_inline)) {
    const int from = row0 + step * kRows;
    const int token0 = scalar((int)fdiv((uint32_t)from, a.by_group));
    const char* const p = reinterpret_cast<const char*>(
        static_cast<const T*>(a.c.q) + (int64_t)(seq.first + token0) * a.c.q_stride[0] +
        (int64_t)head * a.group * a.c.q_stride[1]);
    const rsrc_t r = buffer_of(p - BACK, 0x7fffffffu);
    constexpr int N = LOADS < 4 ? LOADS : 4;
#pragma unroll
    for (int i = 0; i < LOADS; i += N) {
      uint32_t at[N], base[N];
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int of = wave * LOADS * STEP + l_row + (i + j) * STEP;  // the tile's row
        const int row = from + of;
        const int token = (int)fdiv((uint32_t)row, a.by_group), g = row - token * a.group;
        const int c = chunk ^ L::k_swizzle(of);
        base[j] = BACK - j * 1024;
        at[j] = row < row_end && c * 8 < pg.head_dim
                    ? (uint32_t)((token - token0) * (int)a.c.q_stride[0] + g * (int)a.c.q_stride[1] + c * 8) * 2
                    : kOob;
      }
      load_lds16<N>(r, at, base, lds_base + buf * L::kTile + (wave * LOADS + i) * 1024);
    }
  };
  // A lane's rows of a tile, one of each 32: -lse in the base of 2, and the token's position. (Rows past
  // the last: their weights are 0.)
  struct Rows {
    float base[2];
  };
  auto bases = [&](int step) __attribute__((always_inline)) {
    Rows r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = row0 + step * kRows + 32 * i + n;
      const int token = (int)fdiv((uint32_t)row, a.by_group), g = row - token * a.group;
      r.base[i] = row < row_end ? a.c.lse[(int64_t)(seq.first + token) * a.c.q_heads + head * a.group + g]
                                : -__builtin_inff();
    }
    return r;
  };

  // -- the sums ------------------------------------------------------------------------------
  typedef __attribute__((address_space(3))) unsigned char lds_byte;
  typedef __attribute__((address_space(3))) const frag lds_frag;
  lds_byte* const lds0 = (lds_byte*)lds;
  const uint32_t q_lane = n * RB + (half ^ L::k_swizzle(n)) * 16;
  const float mul = SHAPE != kPlain ? 1.0f : a.c.scale * kLog2e;
  f16v sum[KB];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) sum[kb] = f16v{};

  auto block = [&](int buf, int i, int row, float lse) __attribute__((always_inline)) {
    lds_byte* const from = lds0 + buf * L::kTile + i * 32 * RB;
    f16v s[KB];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const frag q = *(lds_frag*)(from + (q_lane ^ (ks * 32)));
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) s[kb] = E::mma(k[kb][ks], q, ks == 0 ? f16v{} : s[kb]);
    }
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
    // A row that saw nothing (lse -inf) weighs nothing.
    const float base = lse == -__builtin_inff() ? lse : -lse * kLog2e;
    const int t0 = (int)fdiv((uint32_t)row, a.by_group);
    const int t1 = (int)fdiv((uint32_t)min(row + 31, row_end - 1), a.by_group);
    const bool whole = row + 32 <= row_end && w0 + 32 * KB <= k1 && (!a.c.causal || w0 + 32 * KB <= start + t0 + 1) &&
                       (a.c.left < 0 || w0 >= start + t1 - a.c.left);
    if (whole) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) sum[kb][r] += __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r], mul, base));
    } else {
      const int place = start + (int)fdiv((uint32_t)(row + n), a.by_group);
      const int lo = a.c.left < 0 ? 0 : max(place - a.c.left, 0);
      const int hi = row + n >= row_end || lse == -__builtin_inff() ? 0 : a.c.causal ? min(place + 1, k1) : k1;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int key = w0 + 32 * kb + 8 * (r / 4) + 4 * half + r % 4;
          const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r], mul, base));
          sum[kb][r] += key >= lo && key < hi ? w : 0.0f;
        }
    }
  };

  if (first < last) {
    Rows here = bases(first), next = here;
    stage(0, first);
    vm_wait();
    lds_sync();
    int buf = 0;
    for (int t = first; t < last; ++t) {
      if (t + 1 < last) {
        stage(buf ^ 1, t + 1);
        next = bases(t + 1);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int row = row0 + t * kRows + 32 * i;
        if (row < row_end && w0 < k1) block(buf, i, row, here.base[i]);
      }
      vm_wait();
      lds_sync();
      here = next;
      buf ^= 1;
    }
  }

  // -- results -------------------------------------------------------------------------------
  // Key 32 kb + 8 (r / 4) + 4 half + r % 4 goes to lane 16 kb + r of its half.
  float mine = 0.0f;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float x = half_sum(sum[kb][r]);
      if (n == 16 * kb + r) mine = x;
    }
  const int r = n & 15, slot = w0 + 32 * (n >> 4) + 8 * (r / 4) + 4 * half + r % 4;
  if ((n >> 4) >= KB || slot >= a.c.slots) return;
  if (a.splits > 1) {
    a.part[((int64_t)split * pg.batch * pg.k_heads + bh) * a.c.slots + slot] = mine;
    return;
  }
  float* const out = a.c.out + b * a.c.out_stride[0] + head * a.c.out_stride[1];
  out[slot] = slot < seq.len ? started(a, seq, b, head, slot) + mine : 0.0f;
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

template <class T, int DP, int KB>
void (*pick(Shape shape))(KeyArgs) {
  return shape == kPlain ? key_tile<T, DP, KB, kPlain> : shape == kCap ? key_tile<T, DP, KB, kCap> : key_tile<T, DP, KB, kAny>;
}
template <class T, int DP>
void (*pick(int blocks, Shape shape))(KeyArgs) {
  return blocks == 2 ? pick<T, DP, 2>(shape) : pick<T, DP, 1>(shape);
}
template <class T>
void (*pick(int d, int blocks, Shape shape))(KeyArgs) {
  if (d <= 32) return pick<T, 32>(blocks, shape);
  if (d <= 64) return pick<T, 64>(blocks, shape);
  if (d <= 96) return pick<T, 96>(blocks, shape);
  if (d <= 128) return pick<T, 128>(blocks, shape);
  return pick<T, 256>(blocks, shape);
}
int tile_bytes(int d) {
  return kRows * (d <= 32 ? 64 : d <= 64 ? 128 : d <= 128 ? 256 : 512);
}

}  // namespace

KeyWeightsPlan key_weights_plan(const arthip_key_weights_args& c) {
  KeyWeightsPlan p{1, 1, 0};
  if (c.p.batch == 0 || c.slots == 0) return p;
  const int64_t rows = (int64_t)c.p.tokens * (c.q_heads / c.p.k_heads);
  const int64_t heads = (int64_t)c.p.batch * c.p.k_heads;
  p.blocks = rows > 64 * c.p.batch ? 2 : 1;
  const int64_t items = heads * ((c.slots + 128 * p.blocks - 1) / (128 * p.blocks));
  // Ranges of the rows: enough workgroups for the chip, of 512 rows at least.
  p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({(2048 + items - 1) / items, rows / c.p.batch / 512, 64}));
  if (p.splits > 1) p.workspace = (size_t)p.splits * heads * c.slots * sizeof(float);
  return p;
}

hipError_t launch_key_weights(const arthip_key_weights_args& c, hipStream_t s) {
  if (c.p.batch == 0 || c.slots == 0) return hipSuccess;
  const KeyWeightsPlan plan = key_weights_plan(c);
  KeyArgs a{};
  a.c = c;
  a.group = c.q_heads / c.p.k_heads;
  a.tiles = (c.slots + 128 * plan.blocks - 1) / (128 * plan.blocks);
  a.splits = plan.splits;
  const int64_t heads = (int64_t)c.p.batch * c.p.k_heads;
  a.items = (int)(heads * a.tiles * a.splits);
  a.by_group = make_fastdiv((uint32_t)a.group);
  a.by_page = make_fastdiv((uint32_t)c.p.page_size);
  a.by_heads = make_fastdiv((uint32_t)c.p.k_heads);
  a.by_tiles = make_fastdiv((uint32_t)a.tiles);
  a.by_splits = make_fastdiv((uint32_t)a.splits);
  if (c.cap > 0) a.cap = make_cap(c.cap, c.scale);
  a.part = static_cast<float*>(c.workspace);
  const Shape shape = c.cap > kCapSmall || !(c.scale > 0) ? kAny : c.cap > 0 ? kCap : kPlain;
  const auto fn = c.p.dtype == ARTHIP_TYPE_F16 ? pick<_Float16>(c.p.head_dim, plan.blocks, shape)
                                               : pick<__bf16>(c.p.head_dim, plan.blocks, shape);
  hipLaunchKernelGGL(fn, dim3((unsigned)((a.items + 7) / 8 * 8)), dim3(256), 2 * tile_bytes(c.p.head_dim), s, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  const int64_t total = heads * c.slots;
  return launch_parts((total + 255) / 256, 256, [&](int64_t first, unsigned count) {
    hipLaunchKernelGGL(key_join, dim3(count), dim3(256), 0, s, a, first, total);
    return hipGetLastError();
  });
}

}  // namespace arthip

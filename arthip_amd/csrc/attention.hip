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
// second product (it lies in [0, 1]); its sum is taken before the rounding.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "launch.h"
#include "token_dev.h"
#include "transformer.h"

namespace arthip {

namespace {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kFar = 1 << 30;

struct AttnArgs {
  arthip_attention_args c;
  int group;      // query heads of a key head
  int rows;       // rows of a key head: q_tokens * group
  int row_tiles;  // workgroups along the rows
  int splits;     // workgroups along the keys
  int items;      // batch * k_heads * row_tiles * splits
  float* part;    // [splits][batch * k_heads * rows][D] unscaled sums, if splits > 1
  float* stat;    // [splits][batch * k_heads * rows][2] maximum (base 2) and sum
};

template <class T>
struct Elem;
template <>
struct Elem<_Float16> {
  typedef h8 frag;
  static constexpr uint32_t kExp = 0x7c007c00u;
  static __device__ __forceinline__ f16v mma(h8 a, h8 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Elem<__bf16> {
  typedef b8 frag;
  static constexpr uint32_t kExp = 0x7f807f80u;
  static __device__ __forceinline__ f16v mma(b8 a, b8 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

// Whether a half-word of x is an infinity or NaN of T.
template <class T>
__device__ __forceinline__ bool nonfinite(uint32_t x) {
  constexpr uint32_t lo = Elem<T>::kExp & 0xffffu, hi = Elem<T>::kExp & 0xffff0000u;
  return (x & lo) == lo || (x & hi) == hi;
}

// The two halves' values of a lane's x. (The results are copied before they are cast:
// a bit cast of a vector's element takes element 0, whichever is named.)
__device__ __forceinline__ void halves(float x, float& low, float& high) {
  const uint32_t a = __builtin_bit_cast(uint32_t, x);
  const u2 r = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  const uint32_t r0 = r[0], r1 = r[1];
  low = __builtin_bit_cast(float, r0);
  high = __builtin_bit_cast(float, r1);
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

// LDS of a workgroup. Rows of K are padded by 16 bytes, rows of V to 64 bytes modulo
// 256: the 32 rows of a K operand, and the four rows of a transposed V read, start on
// different banks, and every address is a lane's base plus a constant.
template <int DP>
struct TileL {
  static constexpr int KT = DP > 128 ? 32 : 64;  // keys of a tile
  static constexpr int KS = DP * 2 + 16;
  static constexpr int VS = DP == 64 ? 192 : DP >= 128 ? DP * 2 + 64 : DP * 2;
  static constexpr int kChunk = 2048;            // tiles whose documents are looked over at once
  static constexpr int kV = 2 * KT * KS;
  static constexpr int kDoc = kV + 2 * KT * VS;  // int32 [2][KT]
  static constexpr int kCode = kDoc + 2 * KT * 4;
  static constexpr int kAny = kCode + 2 * KT * 4;     // bit a tile: some key of a row's document
  static constexpr int kWhole = kAny + kChunk / 8;    // bit a tile: all keys, all rows of one
  static constexpr int kMisc = kWhole + kChunk / 8;   // int32 [2] bad tile, [2][16] documents' range
  static constexpr int kBytes = kMisc + (2 + 32) * 4;
};

template <class T, int DP, int NW>
__global__ void __launch_bounds__(NW * 64, DP > 128 ? 1 : 2) attention_tile(AttnArgs a) {
  using L = TileL<DP>;
  using E = Elem<T>;
  using frag = typename E::frag;
  constexpr int KT = L::KT, NT = NW * 64, KB = KT / 32, KS = DP / 16, DB = DP / 32;
  constexpr int CH = DP / 8;                          // 16-byte chunks of a key
  constexpr int LOADS = (KT * CH + NT - 1) / NT;      // chunks of a tile a thread moves
  extern __shared__ __attribute__((aligned(16))) unsigned char lds[];

  const int per = (int)gridDim.x >> 3;
  int item = ((int)blockIdx.x & 7) * per + ((int)blockIdx.x >> 3);  // one XCD: neighbours share K, V
  if (item >= a.items) return;
  const int split = item % a.splits;
  item /= a.splits;
  const int row_tile = a.row_tiles - 1 - item % a.row_tiles;  // causal: the longest first
  const int bh = item / a.row_tiles;
  const int b = bh / a.c.k_heads;
  const int kh = bh - b * a.c.k_heads;

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int n = lane & 31;     // the lane's row of the wave's 32
  const int half = lane >> 5;  // which keys and values of it

  // -- rows ------------------------------------------------------------------------
  const int kv_len = a.c.kv_len ? min(max(a.c.kv_len[b], 0), a.c.k_tokens) : a.c.k_tokens;
  const int q_start = a.c.q_start ? min(max(a.c.q_start[b], -kFar), kFar) : a.c.k_tokens - a.c.q_tokens;
  const int pre = a.c.prefix ? min(max(a.c.prefix[b], 0), kv_len) : 0;
  // Keys [lo, hi) that a window leaves to a token (and those below pre).
  auto low = [&](int token) -> int {
    if (a.c.left < 0) return 0;
    const int64_t p = (int64_t)q_start + token - a.c.left;
    return p < 0 ? 0 : p > kv_len ? kv_len : (int)p;
  };
  auto high = [&](int token) -> int {
    if (a.c.right < 0) return kv_len;
    const int64_t p = (int64_t)q_start + token + a.c.right + 1;
    return p < 0 ? 0 : p > kv_len ? kv_len : (int)p;
  };
  const int first_row = row_tile * 32 * NW;
  const int last_row = min(first_row + 32 * NW, a.rows) - 1;
  const int row = first_row + wave * 32 + n;
  const bool real = row <= last_row;
  const int token = min(row, last_row) / a.group;
  const int head = kh * a.group + min(row, last_row) - token * a.group;
  const int lo = low(token), hi = high(token);
  // The wave's and the workgroup's rows together: all see [lo_max, hi_min), some see
  // [lo_min, hi_max). Positions grow with the row.
  const int wr0 = min(first_row + wave * 32, last_row), wr1 = min(wr0 + 31, last_row);
  const int w_lo_min = low(wr0 / a.group), w_lo_max = low(wr1 / a.group);
  const int w_hi_min = high(wr0 / a.group), w_hi_max = high(wr1 / a.group);
  const bool w_real = first_row + wave * 32 <= last_row;
  const int g_lo_min = low(first_row / a.group), g_lo_max = low(last_row / a.group);
  const int g_hi_min = high(first_row / a.group), g_hi_max = high(last_row / a.group);

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
  const bool shaped = a.c.cap > 0 || a.c.slopes || a.c.table || !(a.c.scale > 0);
  const float mul = shaped ? 1.0f : a.c.scale * kLog2e;
  const float slope = a.c.slopes ? a.c.slopes[head] * kLog2e : 0.0f;
  const int cq = a.c.code_q ? a.c.code_q[b * a.c.code_q_stride + token] : q_start + token;
  const float* const table = a.c.table ? a.c.table + (int64_t)head * a.c.table_len : nullptr;
  const int dq = a.c.doc_q ? a.c.doc_q[b * a.c.doc_q_stride + token] : 0;
  const int32_t* const doc_k = a.c.doc_k ? a.c.doc_k + b * a.c.doc_k_stride : nullptr;
  const int32_t* const code_k = a.c.code_k ? a.c.code_k + b * a.c.code_k_stride : nullptr;

  // -- the tiles: those of the prefix, then those of the windows ----------------------
  const int pre_tiles = (pre + KT - 1) / KT;
  const int win_first = max(g_lo_min / KT, pre_tiles);
  const int win_end = g_hi_max > g_lo_min ? (g_hi_max + KT - 1) / KT : 0;
  const int count = pre_tiles + max(win_end - win_first, 0);
  const int begin = (int)((int64_t)count * split / a.splits);
  const int end = (int)((int64_t)count * (split + 1) / a.splits);
  auto tile_of = [&](int i) { return i < pre_tiles ? i : i - pre_tiles + win_first; };

  uint32_t* const any = reinterpret_cast<uint32_t*>(lds + L::kAny);
  uint32_t* const whole = reinterpret_cast<uint32_t*>(lds + L::kWhole);
  int* const bad = reinterpret_cast<int*>(lds + L::kMisc);
  int* const range = bad + 2;
  int dmin = 0, dmax = 0;
  if (tid < 2) bad[tid] = -1;
  if (doc_k) {
    int lo_d = dq, hi_d = dq;  // a lane past the last row repeats it
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      lo_d = min(lo_d, __shfl_xor(lo_d, o));
      hi_d = max(hi_d, __shfl_xor(hi_d, o));
    }
    if (lane == 0) {
      range[wave] = lo_d;
      range[16 + wave] = hi_d;
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
  u4 kr[LOADS], vr[LOADS];
  int doc_r = 0, code_r = 0;
  auto fetch = [&](int tile) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int c = tid + i * NT;
      const int64_t key = (int64_t)tile * KT + c / CH;
      const int d = c % CH * 8;
      // Keys past the length and values past the head read nothing and are zeros.
      const bool in = c < KT * CH && key < kv_len && d < a.c.head_dim;
      kr[i] = in ? *reinterpret_cast<const u4*>(kp + key * a.c.k_stride[1] + d) : u4{};
      vr[i] = in ? *reinterpret_cast<const u4*>(vp + key * a.c.v_stride[1] + d) : u4{};
    }
    if (tid < KT) {
      const int64_t key = (int64_t)tile * KT + tid;
      if (doc_k) doc_r = key < kv_len ? doc_k[key] : 0;
      if (code_k) code_r = key < kv_len ? code_k[key] : 0;
    }
  };
  auto stage = [&](int buf, int tile, bool partial) {
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int c = tid + i * NT;
      if (KT * CH % NT != 0 && c >= KT * CH) break;
      *reinterpret_cast<u4*>(lds + buf * KT * L::KS + c / CH * L::KS + c % CH * 16) = kr[i];
      *reinterpret_cast<u4*>(lds + L::kV + buf * KT * L::VS + c / CH * L::VS + c % CH * 16) = vr[i];
      // A value that is not finite, in a tile that some row does not see whole: the
      // products below would carry it into rows that do not see it.
      if (partial && (nonfinite<T>(vr[i][0]) || nonfinite<T>(vr[i][1]) || nonfinite<T>(vr[i][2]) ||
                      nonfinite<T>(vr[i][3])))
        bad[buf] = tile;
    }
    if (tid < KT) {
      if (doc_k) reinterpret_cast<int*>(lds + L::kDoc)[buf * KT + tid] = doc_r;
      if (code_k) reinterpret_cast<int*>(lds + L::kCode)[buf * KT + tid] = code_r;
    }
  };

  // -- one tile ------------------------------------------------------------------------
  const unsigned char* const k_lane = lds + n * L::KS + half * 16;
  const unsigned char* const v_lane =
      lds + L::kV + (4 * half + (lane & 15) / 4) * L::VS + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
  auto v_frag = [&](int buf, int db, int kk) -> frag {  // 32 values (block db) of 16 keys (block kk)
    typedef __attribute__((address_space(3))) s4 lds_s4;
    const unsigned char* const p = v_lane + buf * KT * L::VS + kk * 16 * L::VS + db * 64;
    const s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p));
    const s4 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + 8 * L::VS));
    return __builtin_bit_cast(frag, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
  };
  auto compute = [&](int buf, int tile, bool one_doc) {
    const int k0 = tile * KT;
    const int k1 = k0 + KT;
    const bool seen = k0 < pre || (k0 < w_hi_max && k1 > w_lo_min);
    if (!w_real || !seen) return;
    const bool inside = k1 <= pre || (k0 >= w_lo_max && k1 <= w_hi_min);
    const bool partial = !inside || !one_doc;

    f16v s[KB];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) s[kb] = f16v{};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const frag k = *reinterpret_cast<const frag*>(k_lane + buf * KT * L::KS + kb * 32 * L::KS + ks * 32);
        s[kb] = E::mma(k, q[ks], s[kb]);
      }

    const int key0 = k0 + 4 * half;  // key of element r of block kb: key0 + 32 kb + 8 (r / 4) + r % 4
    if (shaped) {
      if (a.c.cap > 0) {
        // cap tanh(x / cap) = cap - 2 cap / (exp(2 x / cap) + 1), in the base of 2
        const float in = 2.0f * kLog2e * a.c.scale / a.c.cap, out = kLog2e * a.c.cap;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float e = __builtin_amdgcn_exp2f(s[kb][r] * in);
            s[kb][r] = __builtin_fmaf(-2.0f * out, __builtin_amdgcn_rcpf(e + 1.0f), out);
          }
      } else {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[kb][r] *= a.c.scale * kLog2e;
      }
      if (a.c.slopes || table) {
        const int* const codes = reinterpret_cast<const int*>(lds + L::kCode) + buf * KT + 4 * half;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int off = 32 * kb + 8 * (r / 4) + r % 4;
            const int diff = cq - (code_k ? codes[off] : key0 + off);
            if (a.c.slopes) s[kb][r] = __builtin_fmaf(-slope, fabsf((float)diff), s[kb][r]);
            if (table) {
              const int64_t e = (int64_t)diff + a.c.table_zero;
              const int at = e < 0 ? 0 : e >= a.c.table_len ? a.c.table_len - 1 : (int)e;
              const float entry = table[at];
              s[kb][r] = entry == -__builtin_inff() ? entry : __builtin_fmaf(entry, kLog2e, s[kb][r]);
            }
          }
      }
    }
    if (partial) {
      const int* const docs = reinterpret_cast<const int*>(lds + L::kDoc) + buf * KT + 4 * half;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int off = 32 * kb + 8 * (r / 4) + r % 4;
          const int key = key0 + off;
          bool sees = (key >= lo && key < hi) || key < pre;
          if (doc_k) sees = sees && docs[off] == dq;
          s[kb][r] = sees ? s[kb][r] : -__builtin_inff();
        }
    }

    float top = m;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, s[kb][r]);
    top = halves_max(top);
    // A row that has seen nothing yet keeps -inf; its exponents are taken about 0.
    const float base = top == -__builtin_inff() ? 0.0f : top * mul;
    const float keep = __builtin_amdgcn_exp2f(__builtin_fmaf(m, mul, -base));
    m = top;
    float sum = 0.0f;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[kb][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r], mul, -base));
        sum += s[kb][r];
      }
    l = __builtin_fmaf(l, keep, sum);  // this half's keys; the halves are added at the end
    if (__any(keep != 1.0f)) {
#pragma unroll
      for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[i][r] *= keep;
    }

    auto p_frag = [&](int kk) -> frag {
      const f16v x = s[kk / 2];
      return kk & 1 ? __builtin_convertvector(__builtin_shufflevector(x, x, 8, 9, 10, 11, 12, 13, 14, 15), frag)
                    : __builtin_convertvector(__builtin_shufflevector(x, x, 0, 1, 2, 3, 4, 5, 6, 7), frag);
    };
    if ((partial || table) && __builtin_amdgcn_readfirstlane(bad[buf]) == tile) {
      // Infinities and NaN of V apart from its finite values: how many of each sign
      // the row weighs, NaN as both.
#pragma unroll 1
      for (int kk = 0; kk < KT / 16; ++kk) {
        frag p = frag{}, one = frag{};
#pragma unroll
        for (int e = 0; e < KT / 16; ++e)
          if (e == kk) {
            p = p_frag(e);
#pragma unroll
            for (int j = 0; j < 8; ++j) one[j] = to_elem<T>(s[e / 2][8 * (e & 1) + j] != 0.0f ? 1.0f : 0.0f);
          }
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const frag v = v_frag(buf, db, kk);
          frag fin, up, down;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float x = static_cast<float>(v[j]);
            const bool ok = __builtin_isfinite(x);
            fin[j] = ok ? v[j] : to_elem<T>(0.0f);
            up[j] = to_elem<T>(!ok && !(x < 0.0f) ? 1.0f : 0.0f);
            down[j] = to_elem<T>(!ok && !(x > 0.0f) ? 1.0f : 0.0f);
          }
          o[db] = E::mma(fin, p, o[db]);
          const f16v nu = E::mma(up, one, f16v{}), nd = E::mma(down, one, f16v{});
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            if (nu[r] > 0.0f) o[db][r] += __builtin_inff();
            if (nd[r] > 0.0f) o[db][r] -= __builtin_inff();
          }
        }
      }
      return;
    }
#pragma unroll
    for (int kk = 0; kk < KT / 16; ++kk) {
      const frag p = p_frag(kk);
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] = E::mma(v_frag(buf, db, kk), p, o[db]);
    }
  };

  // -- the walk ------------------------------------------------------------------------
  // Two buffers and one barrier a tile: a wave writes a buffer only after the barrier
  // that follows every wave's last use of it.
  const int chunk = doc_k ? L::kChunk : max(end - begin, 1);
  for (int c0 = begin; c0 < end; c0 += chunk) {
    const int c1 = min(end, c0 + chunk);
    if (doc_k) {
      // Tiles whose documents cannot be a row's are not read. A wave looks over 64 / KT
      // .. one tile at a time; a word of the bit sets has one writer.
      lds_sync();
      for (int w = wave; w < (c1 - c0 + 31) / 32; w += NW) {
        uint32_t some = 0, all = 0;
        for (int i = 0; i < 32 && c0 + w * 32 + i < c1; ++i) {
          const int64_t key = (int64_t)tile_of(c0 + w * 32 + i) * KT + (lane & (KT - 1));
          const bool in = key < kv_len;
          const int d = in ? doc_k[key] : 0;
          if (__any(in && d >= dmin && d <= dmax)) some |= 1u << i;
          if (__all(in && d == dmin && d == dmax)) all |= 1u << i;
        }
        if (lane == 0) {
          any[w] = some;
          whole[w] = all;
        }
      }
      lds_sync();
    }
    auto next = [&](int i) {
      if (doc_k)
        while (i < c1 && !(any[(i - c0) >> 5] >> ((i - c0) & 31) & 1)) ++i;
      return __builtin_amdgcn_readfirstlane(i);
    };
    auto one_doc = [&](int i) {
      return !doc_k || __builtin_amdgcn_readfirstlane(whole[(i - c0) >> 5] >> ((i - c0) & 31) & 1) != 0;
    };
    int i = next(c0);
    int buf = 0;
    if (i < c1) fetch(tile_of(i));
    lds_sync();  // the last chunk's tiles have been used
    while (i < c1) {
      const int tile = tile_of(i);
      const bool od = one_doc(i);
      const int k0 = tile * KT;
      const bool inside = k0 + KT <= pre || (k0 >= g_lo_max && k0 + KT <= g_hi_min);
      stage(buf, tile, !inside || !od || table != nullptr);
      const int following = next(i + 1);
      lds_sync();
      if (following < c1) fetch(tile_of(following));
      compute(buf, tile, od);
      i = following;
      buf ^= 1;
    }
  }

  // -- results -------------------------------------------------------------------------
  l = halves_sum(l);
  if (a.splits > 1) {
    if (!real) return;
    const int64_t at = ((int64_t)split * a.c.batch * a.c.k_heads + bh) * a.rows + row;
    float* const p = a.part + at * a.c.head_dim;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = db * 32 + 8 * g + 4 * half;
        if (d < a.c.head_dim)
          *reinterpret_cast<f4*>(p + d) = f4{o[db][4 * g], o[db][4 * g + 1], o[db][4 * g + 2], o[db][4 * g + 3]};
      }
    if (half == 0) {
      a.stat[2 * at] = m * mul;
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
          const f2 pair = {o[db][4 * (g + e) + 2 * j] * scale, o[db][4 * (g + e) + 2 * j + 1] * scale};
          w[e][j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(pair, t2));
        }
      const u2 x = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
      const u2 y = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
      const int d = db * 32 + 8 * (g + half);
      if (real && d < a.c.head_dim) *reinterpret_cast<u4*>(op + d) = u4{x[0], y[0], x[1], y[1]};
    }
  if (a.c.lse && real && half == 0)
    a.c.lse[((int64_t)b * a.c.q_heads + head) * a.c.q_tokens + token] =
        (m * mul + __builtin_amdgcn_logf(l)) * kLn2;
}

// Joins the ranges of the keys: a wave a row.
template <class T>
__global__ void __launch_bounds__(256) attention_join(AttnArgs a) {
  const int64_t total = (int64_t)a.c.batch * a.c.k_heads * a.rows;
  const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= total) return;
  const int lane = threadIdx.x & 63;
  const int D = a.c.head_dim;
  float top = -__builtin_inff();
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, a.stat[2 * (s * total + at)]);
  const float base = top == -__builtin_inff() ? 0.0f : top;
  float l = 0.0f, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int s = 0; s < a.splits; ++s) {
    const float w = __builtin_amdgcn_exp2f(a.stat[2 * (s * total + at)] - base);
    l = __builtin_fmaf(w, a.stat[2 * (s * total + at) + 1], l);
    const float* const p = a.part + (s * total + at) * D;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (lane + 64 * i < D) o[i] = __builtin_fmaf(w, p[lane + 64 * i], o[i]);
  }
  const int64_t bh = at / a.rows;
  const int row = (int)(at - bh * a.rows);
  const int b = (int)(bh / a.c.k_heads), kh = (int)(bh - (int64_t)b * a.c.k_heads);
  const int token = row / a.group, head = kh * a.group + row % a.group;
  const float scale = l == 0.0f ? 0.0f : 1.0f / l;
  T* const op = static_cast<T*>(a.c.out) + b * a.c.out_stride[0] + token * a.c.out_stride[1] +
                head * a.c.out_stride[2];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (lane + 64 * i < D) op[lane + 64 * i] = to_elem<T>(o[i] * scale);
  if (a.c.lse && lane == 0)
    a.c.lse[((int64_t)b * a.c.q_heads + head) * a.c.q_tokens + token] =
        (top + __builtin_amdgcn_logf(l)) * kLn2;
}

struct TilePick {
  void (*fn)(AttnArgs);
  int bytes;
};

template <class T, int DP, int NW>
TilePick pick() {
  return {attention_tile<T, DP, NW>, TileL<DP>::kBytes};
}

template <class T, int NW>
TilePick pick_dim(int d) {
  if (d <= 32) return pick<T, 32, NW>();
  if (d <= 64) return pick<T, 64, NW>();
  if (d <= 96) return pick<T, 96, NW>();
  if (d <= 128) return pick<T, 128, NW>();
  return pick<T, 256, 4>();
}

int waves_of(const arthip_attention_args& c) {
  const int64_t rows = (int64_t)c.q_tokens * (c.q_heads / c.k_heads);
  return rows > 128 && c.head_dim <= 128 ? 8 : 4;
}

}  // namespace

AttnPlan attention_plan(const arthip_attention_args& c) {
  AttnPlan p{1, 0};
  if (c.batch == 0 || c.q_tokens == 0 || c.q_heads == 0) return p;
  const int64_t rows = (int64_t)c.q_tokens * (c.q_heads / c.k_heads);
  const int per = 32 * waves_of(c);
  const int64_t items = (int64_t)c.batch * c.k_heads * ((rows + per - 1) / per);
  const int64_t tiles = (c.k_tokens + 63) / 64;
  if (items < 256) p.splits = (int)std::max<int64_t>(1, std::min<int64_t>({512 / items, tiles / 4, 64}));
  if (p.splits > 1)
    p.workspace = (size_t)p.splits * c.batch * c.k_heads * rows * (c.head_dim + 2) * sizeof(float);
  return p;
}

hipError_t launch_attention(const arthip_attention_args& c, hipStream_t s) {
  if (c.batch == 0 || c.q_tokens == 0 || c.q_heads == 0) return hipSuccess;
  AttnArgs a{};
  a.c = c;
  a.group = c.q_heads / c.k_heads;
  a.rows = c.q_tokens * a.group;
  const int nw = waves_of(c);
  a.row_tiles = (a.rows + 32 * nw - 1) / (32 * nw);
  a.splits = attention_plan(c).splits;
  a.items = c.batch * c.k_heads * a.row_tiles * a.splits;
  const int64_t total = (int64_t)c.batch * c.k_heads * a.rows;
  a.part = static_cast<float*>(c.workspace);
  if (a.splits > 1) a.stat = a.part + a.splits * total * c.head_dim;
  const bool f16 = c.dtype == ARTHIP_TYPE_F16;
  const TilePick k = nw == 8 ? (f16 ? pick_dim<_Float16, 8>(c.head_dim) : pick_dim<__bf16, 8>(c.head_dim))
                             : (f16 ? pick_dim<_Float16, 4>(c.head_dim) : pick_dim<__bf16, 4>(c.head_dim));
  hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(k.fn),
                                     hipFuncAttributeMaxDynamicSharedMemorySize, k.bytes);
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(k.fn, dim3((unsigned)((a.items + 7) / 8 * 8)), dim3(64 * nw), k.bytes, s, a);
  e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  hipLaunchKernelGGL(f16 ? attention_join<_Float16> : attention_join<__bf16>,
                     dim3((unsigned)((total + 3) / 4)), dim3(256), 0, s, a);
  return hipGetLastError();
}

}  // namespace arthip

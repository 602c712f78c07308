// Rotary positions with several axes (arthip_rope_axes): queries and keys of a token
// in one launch.
//
// A thread owns one unit of a head, V frequencies and their 2 V values, at one token:
// it computes the V angles once and turns that unit of every head of its group. Units
// are contiguous (pairs (2f, 2f + 1)) or two runs half a head apart (pairs (f, f + n)),
// so that neighbouring threads read neighbouring memory either way. Values past the
// turned ones are units without angles, copied.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "launch.h"
#include "token_dev.h"
#include "transformer.h"

namespace arthip {

namespace {

constexpr int kRopeThreads = 256;
constexpr int kRopeBatch = 4;            // heads that a thread loads at once
constexpr int64_t kRopeFill = 512 * 1024;  // threads that fill the chip twice over

struct RopeArgs {
  arthip_rope_args c;
  int units;      // of a head: the turned ones first, then copies
  int turned;     // units that turn
  int groups;     // threads of a token and unit, heads dealt out in turn
  int per_token;  // units * groups
  int per_block;  // tokens of a workgroup
  int64_t first;  // token of the launch
};

// sin and cos of 2 pi x, |x| <= 1/2. The nearest quarter turn comes off exactly, the
// rest, |y| <= 1/8, goes through the Taylor polynomials of degree 9 and 10, whose
// next terms are below 2e-9 there; the quarter picks and signs the results.
__device__ __forceinline__ void sincos_turns(float x, float& s, float& c) {
  const float quarter = __builtin_rintf(4.0f * x);
  const float y = __builtin_fmaf(-0.25f, quarter, x);
  const int k = static_cast<int>(quarter);
  const float z = y * y;
  float ps = 42.058693944897655f;  // (2 pi)^9 / 9!
  ps = __builtin_fmaf(ps, z, -76.70585975306136f);
  ps = __builtin_fmaf(ps, z, 81.60524927607504f);
  ps = __builtin_fmaf(ps, z, -41.341702240399755f);
  ps = __builtin_fmaf(ps, z, 6.283185307179586f);
  ps *= y;
  float pc = -26.42625678337438f;  // (2 pi)^10 / 10!
  pc = __builtin_fmaf(pc, z, 60.24464137187666f);
  pc = __builtin_fmaf(pc, z, -85.45681720669373f);
  pc = __builtin_fmaf(pc, z, 64.93939402266829f);
  pc = __builtin_fmaf(pc, z, -19.739208802178716f);
  pc = __builtin_fmaf(pc, z, 1.0f);
  const float a = (k & 1) ? pc : ps;
  const float b = (k & 1) ? ps : pc;
  s = (k & 2) ? -a : a;
  c = ((k + 1) & 2) ? -b : b;
}

template <class T, int V, bool PAIRS>
__global__ void __launch_bounds__(kRopeThreads) rope_axes(RopeArgs a) {
  const int tid = threadIdx.x;
  const int slot = tid / a.per_token;
  const int rest = tid - slot * a.per_token;
  const int group = rest / a.units;
  const int unit = rest - group * a.units;
  const int64_t token = a.first + static_cast<int64_t>(blockIdx.x) * a.per_block + slot;
  if (slot >= a.per_block || token >= static_cast<int64_t>(a.c.batch) * a.c.tokens) return;
  const uint32_t b = static_cast<uint32_t>(token) / static_cast<uint32_t>(a.c.tokens);
  const uint32_t t = static_cast<uint32_t>(token) - b * static_cast<uint32_t>(a.c.tokens);

  const bool turn = unit < a.turned;
  // The two runs of V values of this unit.
  const int first = PAIRS || !turn ? 2 * V * unit : V * unit;
  const int second = PAIRS || !turn ? first + V : first + a.c.n_freq;

  float sn[V], cs[V];
  if (turn) {
    const RopeFreq* const fr = static_cast<const RopeFreq*>(a.c.packed) + unit * V;
    const int32_t* const pos = a.c.pos + b * a.c.pos_stride[1] + t * a.c.pos_stride[2];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const double turns = static_cast<double>(pos[fr[i].axis * a.c.pos_stride[0]]) * fr[i].turns;
      sincos_turns(static_cast<float>(turns - __builtin_rint(turns)), sn[i], cs[i]);
      if (a.c.inverse) sn[i] = -sn[i];
    }
  }

  const T* const q = static_cast<const T*>(a.c.q) + b * a.c.q_stride[0] + t * a.c.q_stride[1];
  const T* const k = static_cast<const T*>(a.c.k) + b * a.c.k_stride[0] + t * a.c.k_stride[1];
  T* const qo = static_cast<T*>(a.c.q_out) + b * a.c.q_out_stride[0] + t * a.c.q_out_stride[1];
  T* const ko = static_cast<T*>(a.c.k_out) + b * a.c.k_out_stride[0] + t * a.c.k_out_stride[1];
  const int heads = a.c.q_heads + a.c.k_heads;
  // Heads in batches: all loads of a batch, then its turns and stores.
  for (int head = group; head < heads; head += kRopeBatch * a.groups) {
    float x[kRopeBatch][V], y[kRopeBatch][V];
    T* out[kRopeBatch];
#pragma unroll
    for (int j = 0; j < kRopeBatch; ++j) {
      const int hj = head + j * a.groups;
      if (hj >= heads) break;
      const bool is_q = hj < a.c.q_heads;
      const int h = is_q ? hj : hj - a.c.q_heads;
      const T* const in = is_q ? q + h * a.c.q_stride[2] : k + h * a.c.k_stride[2];
      out[j] = is_q ? qo + h * a.c.q_out_stride[2] : ko + h * a.c.k_out_stride[2];
      load_chunk<T, V>(in + first, x[j]);
      load_chunk<T, V>(in + second, y[j]);
    }
#pragma unroll
    for (int j = 0; j < kRopeBatch; ++j) {
      if (head + j * a.groups >= heads) break;
      if (turn) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          // Pairs (2f, 2f + 1) are neighbours in the unit's 2 V values, x then y.
          float& u = PAIRS ? (2 * i < V ? x[j][2 * i % V] : y[j][2 * i % V]) : x[j][i];
          float& w = PAIRS ? (2 * i + 1 < V ? x[j][(2 * i + 1) % V] : y[j][(2 * i + 1) % V]) : y[j][i];
          const float u0 = u, w0 = w;
          u = u0 * cs[i] - w0 * sn[i];
          w = w0 * cs[i] + u0 * sn[i];
        }
      }
      store_chunk<T, V>(out[j] + first, x[j]);
      store_chunk<T, V>(out[j] + second, y[j]);
    }
  }
}

template <class T, int V>
void (*rope_kernel(bool pairs))(RopeArgs) {
  return pairs ? rope_axes<T, V, true> : rope_axes<T, V, false>;
}

template <class T>
void (*rope_kernel(int v, bool pairs))(RopeArgs) {
  switch (v) {
    case 8: return rope_kernel<T, 8>(pairs);
    case 4: return rope_kernel<T, 4>(pairs);
    case 2: return rope_kernel<T, 2>(pairs);
    default: return rope_kernel<T, 1>(pairs);
  }
}

}  // namespace

hipError_t launch_rope(const arthip_rope_args& c, hipStream_t s) {
  const int heads = c.q_heads + c.k_heads;
  if (c.batch == 0 || c.tokens == 0 || heads == 0) return hipSuccess;
  RopeArgs a{};
  a.c = c;
  // In place, values that do not turn stay where they are.
  const bool in_place = (c.q_heads == 0 || c.q == c.q_out) && (c.k_heads == 0 || c.k == c.k_out);
  const int copied = in_place ? 0 : c.head_dim - 2 * c.n_freq;
  int v = c.dtype == ARTHIP_TYPE_F32 ? 4 : 8;
  while (c.n_freq % v != 0 || copied % (2 * v) != 0) v /= 2;
  a.turned = c.n_freq / v;
  a.units = a.turned + copied / (2 * v);
  const int64_t tokens = static_cast<int64_t>(c.batch) * c.tokens;
  // A thread for every head where threads are few; where they fill the chip anyway, one
  // for up to four heads, which shares the angles among them.
  a.groups = heads;
  while (a.groups * kRopeBatch > heads && tokens * a.units * (a.groups / 2) >= kRopeFill) a.groups = (a.groups + 1) / 2;
  a.groups = std::min(a.groups, kRopeThreads / a.units);
  a.per_token = a.units * a.groups;
  a.per_block = kRopeThreads / a.per_token;
  const int64_t blocks = (tokens + a.per_block - 1) / a.per_block;
  void (*fn)(RopeArgs) = c.dtype == ARTHIP_TYPE_F16    ? rope_kernel<_Float16>(v, c.pairs != 0)
                         : c.dtype == ARTHIP_TYPE_BF16 ? rope_kernel<__bf16>(v, c.pairs != 0)
                                                       : rope_kernel<float>(v, c.pairs != 0);
  return launch_parts(blocks, kRopeThreads, [&](int64_t first, unsigned count) {
    a.first = first * a.per_block;
    hipLaunchKernelGGL(fn, dim3(count), dim3(kRopeThreads), 0, s, a);
    return hipGetLastError();
  });
}

}  // namespace arthip

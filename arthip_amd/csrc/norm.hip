// The norms around a block's gated residual (arthip_gated_norm) in one pass: y and
// the residual are read once, the new residual and the next block's input written
// once, and what lies between stays in registers.
//
// A row (one token) belongs to R threads, R a multiple of the wave; each holds N
// chunks of eight channels of the row in fp32. Statistics take two steps (mean, then
// the squares about it), so that a large mean costs no digits. 65280 x 1024 in fp16, two
// layer norms, tanh gate and modulation (535 MB): 122 us, 4.4 TB/s, the vector unit 77% busy
// and waves waiting 68% of their cycles, for memory and for one another at the four sums. Rows
// taken in turn with the weights kept in registers or LDS were slower (180 to 270 us for 143):
// fewer waves. Above 16384 channels (four chunks a thread) 18 to 40 registers spill.

#include <hip/hip_runtime.h>

#include <cstdint>

#include "launch.h"
#include "token_dev.h"
#include "transformer.h"

namespace arthip {

namespace {

constexpr int kNormVec = 8;

struct NormArgs {
  arthip_norm_args c;
  int row_threads;  // threads of a row: 64, 128, .. 1024
  int rows;         // rows of a workgroup
  int64_t first;    // row of the launch
  float inv_c;
  FastDiv by_tokens;
};

// Sum over a wave, the same in every lane: exchanges between lanes inside the vector unit
// (quads, half rows, rows of 16, then halves), a few clocks each where a shuffle through
// the LDS path takes its whole latency.
template <int DPP>
__device__ __forceinline__ float add_dpp(float x) {
  return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), DPP, 0xf, 0xf, true));
}
__device__ __forceinline__ float wave_sum(float x) {
  x = add_dpp<0xb1>(x);   // lanes 1 0 3 2
  x = add_dpp<0x4e>(x);   // lanes 2 3 0 1
  x = add_dpp<0x141>(x);  // half rows mirrored
  x = add_dpp<0x140>(x);  // rows mirrored
  uint32_t u = __builtin_bit_cast(uint32_t, x);
  const u2 r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  const uint32_t r0 = r[0], r1 = r[1];
  x = __builtin_bit_cast(float, r0) + __builtin_bit_cast(float, r1);
  u = __builtin_bit_cast(uint32_t, x);
  const u2 h = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  const uint32_t h0 = h[0], h1 = h[1];
  return __builtin_bit_cast(float, h0) + __builtin_bit_cast(float, h1);
}

// Sum over the row's threads. Every thread of the workgroup calls it the same number
// of times; `part` holds two sets of one value a wave, used in turn, so that one
// barrier a sum is enough.
struct RowSum {
  float* part;
  int wave, first, waves, turn;
  __device__ __forceinline__ float operator()(float x) {
    x = wave_sum(x);
    if (waves == 1) return x;
    float* const p = part + turn * 16;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) p[wave] = x;
    lds_sync();
    float s = 0.0f;
    for (int i = 0; i < waves; ++i) s += p[first + i];
    return s;
  }
};

// The channels of a thread. Its last chunk, where it would reach past the row, ends with
// the row instead and repeats `skip` channels of the chunk before it: read and written
// whole, with the same values, and left out of the sums (all eight where the thread has
// no chunk).
template <int N>
struct Chans {
  int at[N], skip[N];
};

// A thread's channels of a row. Rows of fewer than eight go value by value.
template <bool FULL, class T, int N>
__device__ __forceinline__ void load_rows(const T* p, const Chans<N>& c, int C, float (&x)[N][kNormVec]) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (!FULL && c.skip[n] >= kNormVec) {
#pragma unroll
      for (int i = 0; i < kNormVec; ++i) x[n][i] = 0.0f;
    } else if (FULL || C >= kNormVec) {
      load_chunk<T, kNormVec>(p + c.at[n], x[n]);
    } else {
#pragma unroll
      for (int i = 0; i < kNormVec; ++i) x[n][i] = i >= c.skip[n] ? static_cast<float>(p[c.at[n] + i]) : 0.0f;
    }
  }
}
template <bool FULL, class T, int N>
__device__ __forceinline__ void store_rows(T* p, const Chans<N>& c, int C, const float (&x)[N][kNormVec]) {
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (!FULL && c.skip[n] >= kNormVec) continue;
    if (FULL || C >= kNormVec) {
      store_chunk<T, kNormVec>(p + c.at[n], x[n]);
    } else {
#pragma unroll
      for (int i = 0; i < kNormVec; ++i)
        if (i >= c.skip[n]) p[c.at[n] + i] = to_elem<T>(x[n][i]);
    }
  }
}

// Sum of f over a thread's channels.
template <bool FULL, int N, class F>
__device__ __forceinline__ float add_up(const float (&x)[N][kNormVec], const Chans<N>& c, F f) {
  float t = 0.0f;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (FULL || !__any(c.skip[n] > 0)) {
#pragma unroll
      for (int i = 0; i < kNormVec; ++i) t = f(x[n][i], t);
    } else {
#pragma unroll
      for (int i = 0; i < kNormVec; ++i) t = i >= c.skip[n] ? f(x[n][i], t) : t;
    }
  }
  return t;
}

template <bool FULL, int N>
__device__ __forceinline__ void normalize(float (&x)[N][kNormVec], const Chans<N>& c, const NormArgs& a, int kind,
                                          const float* weight, const float* bias, RowSum& sum) {
  if (kind == ARTHIP_NORM_NONE) return;
  if (kind == ARTHIP_NORM_LAYER) {
    const float mean = sum(add_up<FULL>(x, c, [](float v, float t) { return t + v; })) * a.inv_c;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < kNormVec; ++i) x[n][i] -= mean;
  }
  const float squares = add_up<FULL>(x, c, [](float v, float t) { return __builtin_fmaf(v, v, t); });
  const float r = 1.0f / __builtin_sqrtf(sum(squares) * a.inv_c + a.c.eps);
  float w[N][kNormVec];
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < kNormVec; ++i) x[n][i] *= r;
  if (weight) {
    load_rows<FULL>(weight, c, a.c.channels, w);
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < kNormVec; ++i) x[n][i] *= w[n][i];
  }
  if (bias) {
    load_rows<FULL>(bias, c, a.c.channels, w);
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < kNormVec; ++i) x[n][i] += w[n][i];
  }
}

// tanh without branches: near 0, where 1 - 2 / (exp(2 x) + 1) has no digits left, x times
// a polynomial of x^2 (a Chebyshev fit up to 0.6, off by less than 8e-8).
__device__ __forceinline__ float tanh_of(float x) {
  const float z = x * x;
  float p = 0.01548669f;
  p = __builtin_fmaf(p, z, -0.05210962f);
  p = __builtin_fmaf(p, z, 0.13310358f);
  p = __builtin_fmaf(p, z, -0.33332323f);
  p = __builtin_fmaf(p, z, 0.99999993f);
  const float far = 1.0f - 2.0f * __builtin_amdgcn_rcpf(__expf(2.0f * x) + 1.0f);
  return fabsf(x) < 0.6f ? x * p : far;
}

__device__ __forceinline__ void gates(float (&g)[kNormVec], int act) {
  if (act == ARTHIP_GATE_TANH) {
#pragma unroll
    for (int i = 0; i < kNormVec; ++i) g[i] = tanh_of(g[i]);
  } else if (act != ARTHIP_GATE_NONE) {
#pragma unroll
    for (int i = 0; i < kNormVec; ++i) {
      const float s = 1.0f / (1.0f + __expf(-g[i]));
      g[i] = act == ARTHIP_GATE_SILU ? g[i] * s : s;
    }
  }
}

// FULL: every thread's chunks are whole, as where the channels are a power of two from
// 512 on; the checks of the other kind are a third of the vector work.
template <class T, class TR, int N, bool FULL>
__global__ void __launch_bounds__(1024) gated_norm(NormArgs a) {
  __shared__ float part[32];
  const int tid = threadIdx.x;
  const int slot = tid / a.row_threads;
  const int lane = tid - slot * a.row_threads;
  const int64_t total = static_cast<int64_t>(a.c.batch) * a.c.tokens;
  const int64_t index = a.first + static_cast<int64_t>(blockIdx.x) * a.rows + slot;
  const bool real = index < total;
  // A slot past the last row computes the last one again, so that every thread meets
  // every barrier, and writes nothing.
  const uint32_t row = static_cast<uint32_t>(real ? index : total - 1);
  const uint32_t b = fdiv(row, a.by_tokens);
  const uint32_t t = row - b * static_cast<uint32_t>(a.c.tokens);
  const int C = a.c.channels;
  RowSum sum{part, tid >> 6, slot * (a.row_threads >> 6), a.row_threads >> 6, 0};
  auto at = [&](const int64_t (&stride)[2]) { return b * stride[0] + t * stride[1]; };

  Chans<N> c;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int first = (n * a.row_threads + lane) * kNormVec;
    c.skip[n] = FULL ? 0 : min(max(first + kNormVec - C, 0), kNormVec);
    // Below 0 where a row has fewer than eight channels: the values skipped are not touched.
    c.at[n] = first - c.skip[n];
  }
  float r[N][kNormVec], y[N][kNormVec];
  load_rows<FULL>(static_cast<const TR*>(a.c.residual) + at(a.c.residual_stride), c, C, r);
  // In place, no thread may write channels that another one has yet to read.
  if (!FULL && sum.waves > 1) lds_sync();
  if (a.c.y) {
    load_rows<FULL>(static_cast<const T*>(a.c.y) + at(a.c.y_stride), c, C, y);
    float g[N][kNormVec];
    if (a.c.gate) {
      load_rows<FULL>(static_cast<const T*>(a.c.gate) + at(a.c.gate_stride), c, C, g);
#pragma unroll
      for (int n = 0; n < N; ++n) gates(g[n], a.c.gate_act);
    } else {
      float one[kNormVec];
#pragma unroll
      for (int i = 0; i < kNormVec; ++i) one[i] = 1.0f;
      gates(one, a.c.gate_act);
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int i = 0; i < kNormVec; ++i) g[n][i] = one[0];
    }
    normalize<FULL>(y, c, a, a.c.post, a.c.post_weight, a.c.post_bias, sum);
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < kNormVec; ++i)
        r[n][i] = __builtin_fmaf(a.c.branch_scale * g[n][i], y[n][i], a.c.residual_scale * r[n][i]);
  } else {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < kNormVec; ++i) r[n][i] *= a.c.residual_scale;
  }
  if (a.c.residual_out && real)
    store_rows<FULL>(static_cast<TR*>(a.c.residual_out) + at(a.c.residual_out_stride), c, C, r);
  if (!a.c.h) return;
  normalize<FULL>(r, c, a, a.c.pre, a.c.pre_weight, a.c.pre_bias, sum);
  if (a.c.mod_scale) {
    float m[N][kNormVec];
    load_rows<FULL>(static_cast<const T*>(a.c.mod_scale) + at(a.c.mod_scale_stride), c, C, m);
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < kNormVec; ++i) r[n][i] = __builtin_fmaf(r[n][i], m[n][i], r[n][i]);
  }
  if (a.c.mod_shift) {
    float m[N][kNormVec];
    load_rows<FULL>(static_cast<const T*>(a.c.mod_shift) + at(a.c.mod_shift_stride), c, C, m);
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < kNormVec; ++i) r[n][i] += m[n][i];
  }
  if (real) store_rows<FULL>(static_cast<T*>(a.c.h) + at(a.c.h_stride), c, C, r);
}

template <class T, class TR, bool FULL>
void (*norm_kernel(int n))(NormArgs) {
  return n == 1 ? gated_norm<T, TR, 1, FULL> : n == 2 ? gated_norm<T, TR, 2, FULL> : gated_norm<T, TR, 4, FULL>;
}

template <class T, class TR>
void (*norm_kernel(int n, bool full))(NormArgs) {
  return full ? norm_kernel<T, TR, true>(n) : norm_kernel<T, TR, false>(n);
}

}  // namespace

hipError_t launch_norm(const arthip_norm_args& c, hipStream_t s) {
  if (c.batch == 0 || c.tokens == 0) return hipSuccess;
  NormArgs a{};
  a.c = c;
  a.inv_c = 1.0f / static_cast<float>(c.channels);
  a.by_tokens = make_fastdiv((uint32_t)c.tokens);
  const int chunks = (c.channels + kNormVec - 1) / kNormVec;
  a.row_threads = 64;
  while (a.row_threads < 1024 && a.row_threads * 2 < chunks) a.row_threads *= 2;
  const int n = (chunks + a.row_threads - 1) / a.row_threads;
  const int held = n == 3 ? 4 : n;  // chunks a thread holds
  const bool full = c.channels == a.row_threads * held * kNormVec;
  a.rows = a.row_threads < 256 ? 256 / a.row_threads : 1;
  const int64_t total = static_cast<int64_t>(c.batch) * c.tokens;
  if (total < a.rows) a.rows = 1;
  const int64_t blocks = (total + a.rows - 1) / a.rows;
  const bool wide = c.residual_dtype == ARTHIP_TYPE_F32;
  void (*fn)(NormArgs) =
      c.dtype == ARTHIP_TYPE_F32   ? norm_kernel<float, float>(n, full)
      : c.dtype == ARTHIP_TYPE_F16 ? (wide ? norm_kernel<_Float16, float>(n, full) : norm_kernel<_Float16, _Float16>(n, full))
                                   : (wide ? norm_kernel<__bf16, float>(n, full) : norm_kernel<__bf16, __bf16>(n, full));
  const int threads = a.rows * a.row_threads;
  return launch_parts(blocks, threads, [&](int64_t first, unsigned count) {
    a.first = first * a.rows;
    hipLaunchKernelGGL(fn, dim3(count), dim3((unsigned)threads), 0, s, a);
    return hipGetLastError();
  });
}

}  // namespace arthip

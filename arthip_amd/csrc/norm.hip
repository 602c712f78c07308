// The norms around a block's gated residual (arthip_gated_norm) in one pass: y and
// the residual are read once, the new residual and the next block's input written
// once, and what lies between stays in registers.
//
// A row (one token) belongs to R threads, R a multiple of the wave; each holds N
// chunks of eight channels of the row in fp32. Statistics take two steps (mean, then
// the squares about it), so that a large mean costs no digits.

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
  float inv_c;
};

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o);
  return x;
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

template <int N>
__device__ __forceinline__ void normalize(float (&x)[N][kNormVec], const bool (&live)[N],
                                          const int (&chan)[N], const NormArgs& a, int kind,
                                          const float* weight, const float* bias, RowSum& sum) {
  if (kind == ARTHIP_NORM_NONE) return;
  const int C = a.c.channels;
  if (kind == ARTHIP_NORM_LAYER) {
    float t = 0.0f;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < kNormVec; ++i) t += x[n][i];
    const float mean = sum(t) * a.inv_c;
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < kNormVec; ++i)
        x[n][i] = live[n] && chan[n] + i < C ? x[n][i] - mean : 0.0f;
  }
  float t = 0.0f;
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < kNormVec; ++i) t = __builtin_fmaf(x[n][i], x[n][i], t);
  const float r = 1.0f / __builtin_sqrtf(sum(t) * a.inv_c + a.c.eps);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (!live[n]) continue;
    const int left = C - chan[n];
    float w[kNormVec], b[kNormVec];
#pragma unroll
    for (int i = 0; i < kNormVec; ++i) {
      w[i] = 1.0f;
      b[i] = 0.0f;
    }
    if (left >= kNormVec) {
      if (weight) load_chunk<float, kNormVec>(weight + chan[n], w);
      if (bias) load_chunk<float, kNormVec>(bias + chan[n], b);
    } else {
      for (int i = 0; i < kNormVec; ++i) {
        if (weight && i < left) w[i] = weight[chan[n] + i];
        if (bias && i < left) b[i] = bias[chan[n] + i];
      }
    }
#pragma unroll
    for (int i = 0; i < kNormVec; ++i) x[n][i] = __builtin_fmaf(x[n][i] * r, w[i], b[i]);
  }
}

// Eight channels of a row, or the `left` ones that it still has (zeros after them).
template <class T>
__device__ __forceinline__ void load_row(const T* p, int left, float (&x)[kNormVec]) {
  if (left >= kNormVec) {
    load_chunk<T, kNormVec>(p, x);
  } else {
#pragma unroll
    for (int i = 0; i < kNormVec; ++i) x[i] = i < left ? static_cast<float>(p[i]) : 0.0f;
  }
}

template <class T>
__device__ __forceinline__ void store_row(T* p, int left, const float (&x)[kNormVec]) {
  if (left >= kNormVec) {
    store_chunk<T, kNormVec>(p, x);
  } else {
#pragma unroll
    for (int i = 0; i < kNormVec; ++i)
      if (i < left) p[i] = to_elem<T>(x[i]);
  }
}

__device__ __forceinline__ float gate_of(float g, int act) {
  switch (act) {
    case ARTHIP_GATE_SIGMOID: return 1.0f / (1.0f + __expf(-g));
    case ARTHIP_GATE_TANH: return tanhf(g);
    case ARTHIP_GATE_SILU: return g / (1.0f + __expf(-g));
    default: return g;
  }
}

template <class T, class TR, int N>
__global__ void __launch_bounds__(1024) gated_norm(NormArgs a) {
  __shared__ float part[32];
  const int tid = threadIdx.x;
  const int slot = tid / a.row_threads;
  const int lane = tid - slot * a.row_threads;
  const int64_t total = static_cast<int64_t>(a.c.batch) * a.c.tokens;
  const int64_t index = static_cast<int64_t>(blockIdx.x) * a.rows + slot;
  const bool real = index < total;
  // A slot past the last row computes the last one again, so that every thread meets
  // every barrier, and writes nothing.
  const uint32_t row = static_cast<uint32_t>(real ? index : total - 1);
  const uint32_t b = row / static_cast<uint32_t>(a.c.tokens);
  const uint32_t t = row - b * static_cast<uint32_t>(a.c.tokens);
  const int C = a.c.channels;
  RowSum sum{part, tid >> 6, slot * (a.row_threads >> 6), a.row_threads >> 6, 0};

  auto at = [&](const int64_t (&stride)[2]) { return b * stride[0] + t * stride[1]; };

  bool live[N];
  int chan[N];
  float r[N][kNormVec], y[N][kNormVec];
  const TR* const res = static_cast<const TR*>(a.c.residual) + at(a.c.residual_stride);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    chan[n] = (n * a.row_threads + lane) * kNormVec;
    live[n] = chan[n] < C;
#pragma unroll
    for (int i = 0; i < kNormVec; ++i) r[n][i] = y[n][i] = 0.0f;
    if (live[n]) load_row(res + chan[n], C - chan[n], r[n]);
  }
  if (a.c.y) {
    const T* const yp = static_cast<const T*>(a.c.y) + at(a.c.y_stride);
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (live[n]) load_row(yp + chan[n], C - chan[n], y[n]);
    normalize<N>(y, live, chan, a, a.c.post, a.c.post_weight, a.c.post_bias, sum);
    const T* const gp = a.c.gate ? static_cast<const T*>(a.c.gate) + at(a.c.gate_stride) : nullptr;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if (!live[n]) continue;
      float g[kNormVec];
      if (gp) {
        load_row(gp + chan[n], C - chan[n], g);
#pragma unroll
        for (int i = 0; i < kNormVec; ++i) g[i] = gate_of(g[i], a.c.gate_act);
      } else {
#pragma unroll
        for (int i = 0; i < kNormVec; ++i) g[i] = 1.0f;
      }
#pragma unroll
      for (int i = 0; i < kNormVec; ++i)
        r[n][i] = chan[n] + i < C ? __builtin_fmaf(a.c.branch_scale * g[i], y[n][i],
                                                   a.c.residual_scale * r[n][i])
                                  : 0.0f;
    }
  } else {
#pragma unroll
    for (int n = 0; n < N; ++n)
#pragma unroll
      for (int i = 0; i < kNormVec; ++i) r[n][i] *= a.c.residual_scale;
  }
  if (a.c.residual_out && real) {
    TR* const out = static_cast<TR*>(a.c.residual_out) + at(a.c.residual_out_stride);
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (live[n]) store_row(out + chan[n], C - chan[n], r[n]);
  }
  if (!a.c.h) return;
  normalize<N>(r, live, chan, a, a.c.pre, a.c.pre_weight, a.c.pre_bias, sum);
  const T* const sp =
      a.c.mod_scale ? static_cast<const T*>(a.c.mod_scale) + at(a.c.mod_scale_stride) : nullptr;
  const T* const fp =
      a.c.mod_shift ? static_cast<const T*>(a.c.mod_shift) + at(a.c.mod_shift_stride) : nullptr;
  T* const h = static_cast<T*>(a.c.h) + at(a.c.h_stride);
#pragma unroll
  for (int n = 0; n < N; ++n) {
    if (!live[n]) continue;
    float m[kNormVec];
    if (sp) {
      load_row(sp + chan[n], C - chan[n], m);
#pragma unroll
      for (int i = 0; i < kNormVec; ++i) r[n][i] = __builtin_fmaf(r[n][i], m[i], r[n][i]);
    }
    if (fp) {
      load_row(fp + chan[n], C - chan[n], m);
#pragma unroll
      for (int i = 0; i < kNormVec; ++i) r[n][i] += m[i];
    }
    if (real) store_row(h + chan[n], C - chan[n], r[n]);
  }
}

template <class T, class TR>
void (*norm_kernel(int n))(NormArgs) {
  return n == 1 ? gated_norm<T, TR, 1> : n == 2 ? gated_norm<T, TR, 2> : gated_norm<T, TR, 4>;
}

}  // namespace

hipError_t launch_norm(const arthip_norm_args& c, hipStream_t s) {
  if (c.batch == 0 || c.tokens == 0) return hipSuccess;
  NormArgs a{};
  a.c = c;
  a.inv_c = 1.0f / static_cast<float>(c.channels);
  const int chunks = (c.channels + kNormVec - 1) / kNormVec;
  a.row_threads = 64;
  while (a.row_threads < 1024 && a.row_threads * 2 < chunks) a.row_threads *= 2;
  const int n = (chunks + a.row_threads - 1) / a.row_threads;
  a.rows = a.row_threads < 256 ? 256 / a.row_threads : 1;
  const int64_t total = static_cast<int64_t>(c.batch) * c.tokens;
  if (total < a.rows) a.rows = 1;
  const int64_t blocks = (total + a.rows - 1) / a.rows;
  const bool wide = c.residual_dtype == ARTHIP_TYPE_F32;
  void (*fn)(NormArgs) =
      c.dtype == ARTHIP_TYPE_F32   ? norm_kernel<float, float>(n)
      : c.dtype == ARTHIP_TYPE_F16 ? (wide ? norm_kernel<_Float16, float>(n) : norm_kernel<_Float16, _Float16>(n))
                                   : (wide ? norm_kernel<__bf16, float>(n) : norm_kernel<__bf16, __bf16>(n));
  hipLaunchKernelGGL(fn, dim3((unsigned)blocks), dim3((unsigned)(a.rows * a.row_threads)), 0, s, a);
  return hipGetLastError();
}

}  // namespace arthip

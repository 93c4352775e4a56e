// Shared pieces of the vocabulary objectives (objectives.cu, top_logits.cu, preference.cu): logits
// rows of bf16, fp16 or fp32 with any row stride, the softcap, and (max, sum) statistics.
#pragma once

#include <cuda_fp16.h>

#include "act.cuh"
#include "common.cuh"
#include "objectives.h"

namespace me {

template <>
ME_DEVICE float to_f<__half>(__half x) { return __half2float(x); }
template <>
ME_DEVICE __half from_f<__half>(float x) { return __float2half_rn(x); }

// One 16-byte vector of logits.
template <typename T>
union Vec16 {
  static constexpr int kN = 16 / sizeof(T);
  uint4 u;
  T h[16 / sizeof(T)];
};

// z = c tanh(x / c), or x without a cap (cap <= 0).
ME_DEVICE float softcap(float x, float cap) { return cap > 0.f ? cap * tanhf(x / cap) : x; }
// dz/dx, from z.
ME_DEVICE float softcap_slope(float z, float cap) {
  if (cap <= 0.f) return 1.f;
  const float t = z / cap;
  return 1.f - t * t;
}

// A logits matrix and its rows' stride in elements.
template <typename T>
struct Rows {
  T* base;
  int64_t stride;
  ME_DEVICE T* row(int64_t r) const { return base + r * stride; }
};

// Calls f(j, x_j) for every column of a row of V logits, the block's threads in turn: single
// elements up to the first 16-byte boundary and after the last one, 16-byte vectors between.
template <typename T, typename F>
ME_DEVICE void for_row(const T* row, int64_t V, F&& f) {
  constexpr int kN = Vec16<T>::kN;
  int64_t head = ((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T);
  if (head > V) head = V;
  for (int64_t j = threadIdx.x; j < head; j += blockDim.x) f(j, to_f<T>(row[j]));
  const int64_t nvec = (V - head) / kN;
  const uint4* body = reinterpret_cast<const uint4*>(row + head);
  for (int64_t i = threadIdx.x; i < nvec; i += blockDim.x) {
    Vec16<T> v;
    v.u = body[i];
#pragma unroll
    for (int e = 0; e < kN; ++e) f(head + i * kN + e, to_f<T>(v.h[e]));
  }
  for (int64_t j = head + nvec * kN + threadIdx.x; j < V; j += blockDim.x) f(j, to_f<T>(row[j]));
}

// Running (m, s): s = sum exp(y - m), m the largest y so far. A NaN or +inf makes s NaN.
struct MaxSum {
  float m = -INFINITY, s = 0.f;
  ME_DEVICE void add(float y) {
    if (y > m) {
      s = s * exp2_fast((m - y) * kLog2e) + exp2_fast(y - y);  // + 1, or NaN for y = inf
      m = y;
    } else if (y != -INFINITY) {  // y NaN: s becomes NaN
      s += exp2_fast((y - m) * kLog2e);
    }
  }
  ME_DEVICE void merge(float m2, float s2) {
    if (m2 == -INFINITY) {
      s += s2;  // 0, or NaN
    } else if (m == -INFINITY) {
      s += s2;
      m = m2;
    } else {
      const float mx = fmaxf(m, m2);
      s = s * exp2_fast((m - mx) * kLog2e) + s2 * exp2_fast((m2 - mx) * kLog2e);
      m = mx;
    }
  }
};

// Over the whole block, the same for all threads; `scratch` holds 64 floats.
ME_DEVICE MaxSum block_merge(MaxSum a, float* scratch) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, a.m, o), s2 = __shfl_xor_sync(0xffffffffu, a.s, o);
    a.merge(m2, s2);
  }
  __syncthreads();
  if (lane == 0) {
    scratch[wid] = a.m;
    scratch[32 + wid] = a.s;
  }
  __syncthreads();
  MaxSum r;
  if (lane < nw) {
    r.m = scratch[lane];
    r.s = scratch[32 + lane];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, r.m, o), s2 = __shfl_xor_sync(0xffffffffu, r.s, o);
    r.merge(m2, s2);
  }
  return r;
}

// SMs of the current device (one kind of GPU is built for).
inline int objective_sms() {
  static int n = [] {
    int dev = 0, c = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&c, cudaDevAttrMultiProcessorCount, dev);
    return c;
  }();
  return n;
}

template <typename T>
Rows<const T> rows_in(const Logits& x) {
  return {static_cast<const T*>(x.data), x.stride};
}
template <typename T>
Rows<T> rows_out(const Gradient& g) {
  return {static_cast<T*>(g.data), g.stride};
}

#define ME_LOGITS_DISPATCH(TYPE, ...)      \
  if ((TYPE) == LogitType::kBF16) {        \
    using T = __nv_bfloat16;               \
    __VA_ARGS__;                           \
  } else if ((TYPE) == LogitType::kF16) {  \
    using T = __half;                      \
    __VA_ARGS__;                           \
  } else {                                 \
    using T = float;                       \
    __VA_ARGS__;                           \
  }

}  // namespace me

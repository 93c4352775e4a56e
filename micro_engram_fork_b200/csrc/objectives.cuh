// Shared pieces of the vocabulary objectives (objectives.cu, top_logits.cu, preference.cu): logits
// rows of bf16, fp16 or fp32 with any row stride, the softcap, and (max, sum) statistics.
#pragma once

#include <cuda_fp16.h>

#include <string.h>

#include <type_traits>

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

// z = c tanh(x / c), or x without a cap (cap <= 0): the accurate form of single elements. For |x| <= c a
// polynomial in which x enters unrounded (relative error 5e-9 before rounding); tanhf, times c, would be
// off by 1e-6 at z = 15 on average.
ME_DEVICE float softcap(float x, float cap) {
  if (!(cap > 0.f)) return x;
  const float u = x / cap;
  if (!(fabsf(u) <= 1.f)) return cap * tanhf(u);
  const float w = u * u;
  float q = fmaf(-0.000358452002f, w, 0.00230136459f);
  q = fmaf(q, w, -0.00794610642f);
  q = fmaf(q, w, 0.0214866576f);
  q = fmaf(q, w, -0.0538798027f);
  q = fmaf(q, w, 0.133323446f);
  q = fmaf(q, w, -0.333332954f);
  return fmaf(x * w, q, x);
}
// dz/dx, from z.
ME_DEVICE float softcap_slope(float z, float cap) {
  if (cap <= 0.f) return 1.f;
  const float t = z / cap;
  return 1.f - t * t;
}

// ---------------------------------------------------------------- two fp32 numbers an instruction
typedef unsigned long long f32x2;

ME_DEVICE f32x2 pack2(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
ME_DEVICE f32x2 both2(float a) { return pack2(a, a); }
ME_DEVICE float2 unpack2(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
ME_DEVICE f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
ME_DEVICE f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
ME_DEVICE f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// A 16-byte vector of logits as pairs, and back (one rounding).
template <typename T>
ME_DEVICE void to_pairs(uint4 v, f32x2 (&p)[Vec16<T>::kN / 2]) {
  if constexpr (sizeof(T) == 4) {
    p[0] = pack2(__uint_as_float(v.x), __uint_as_float(v.y));
    p[1] = pack2(__uint_as_float(v.z), __uint_as_float(v.w));
  } else {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        p[i] = pack2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
      } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        p[i] = pack2(f.x, f.y);
      }
    }
  }
}
template <typename T>
ME_DEVICE uint4 from_pairs(const f32x2 (&p)[Vec16<T>::kN / 2]) {
  uint32_t w[4];
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 f = unpack2(p[i]);
      w[2 * i] = __float_as_uint(f.x);
      w[2 * i + 1] = __float_as_uint(f.y);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2(p[i]);
      if constexpr (std::is_same_v<T, __nv_bfloat16>) {
        const __nv_bfloat162 h = __float22bfloat162_rn(f);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __half2 h = __float22half2_rn(f);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// The running largest of a thread's logits (a NaN beside numbers is passed over). 16-bit types: two lanes in one
// register.
template <typename T>
struct MaxOf {
  using T2 = std::conditional_t<std::is_same_v<T, __nv_bfloat16>, __nv_bfloat162,
                                std::conditional_t<std::is_same_v<T, __half>, __half2, float>>;
  T2 m;
  ME_DEVICE MaxOf() { clear(); }
  ME_DEVICE void clear() {
    if constexpr (sizeof(T) == 4) m = -INFINITY;
    else m = T2(from_f<T>(-INFINITY), from_f<T>(-INFINITY));
  }
  ME_DEVICE void add(uint4 v) {
    if constexpr (sizeof(T) == 4) {
      m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)),
                         fmaxf(__uint_as_float(v.z), __uint_as_float(v.w))));
    } else {
      const T2 a = *reinterpret_cast<T2*>(&v.x), b = *reinterpret_cast<T2*>(&v.y), c = *reinterpret_cast<T2*>(&v.z),
               d = *reinterpret_cast<T2*>(&v.w);
      m = __hmax2(m, __hmax2(__hmax2(a, b), __hmax2(c, d)));
    }
  }
  ME_DEVICE float value() const {
    if constexpr (sizeof(T) == 4) return m;
    else return fmaxf(to_f<T>(m.x), to_f<T>(m.y));
  }
};

// How raw logits become exponents: z = softcap(x), y = z / tau.
//
// c tanh(x / c) is evaluated on the FMA pipe, as x P(v), v = x^2, P the minimax polynomial of tanh(u) / u in
// u^2 (Remez exchange on tanh itself; the coefficients carry the powers of 1 / c^2): one for
// |x| <= c / 2, where most logits lie, one for |x| <= c. (By exponential and reciprocal it
// would be two results of the special function unit, which gives 16 a clock on an SM and has the
// softmax's exponential to do. A packed FMA takes two issue slots on sm_100, so what counts is operations:
// the short polynomial saves two of about thirteen a logit.)
struct Scale {
  float cap, limit, inv_temp, slope;  // limit: c^2, or -1 (no polynomial for this cap); slope = -1 / c^2
  float twice;                        // 2 log2 e / c
  // 16-bit logits: P log2 e / tau (relative error 6e-8 and 2e-8), for sums
  f32x2 sum_full[7], sum_short[5];
  // 16-bit logits: P to 7e-7, for gradients that are rounded to 16 bits
  f32x2 z_full[6], z_short[4];
  // 32-bit logits, and vectors with a logit beyond the cap: Q of P = 1 + v Q, so that x enters unrounded
  f32x2 q_full[6], q_short[4];
};

template <int kN>
ME_DEVICE f32x2 horner2(const f32x2 (&c)[kN], f32x2 v) {
  f32x2 p = fma2(c[kN - 1], v, c[kN - 2]);
#pragma unroll
  for (int i = kN - 3; i >= 0; --i) p = fma2(p, v, c[i]);
  return p;
}

inline Scale make_scale(float cap, float temp) {
  // Q of tanh(u) = u (1 + u^2 Q(u^2)): on |u| <= 1 and <= 1/2, and the shorter ones for gradients
  static const double kFull[6] = {-0.333329868, 0.133264089, -0.0534987079, 0.0203597599, -0.00625933984, 0.00105826482};
  static const double kShort[4] = {-0.333331439, 0.13325879, -0.0530454943, 0.0172414915};
  static const double kFull16[5] = {-0.333302797, 0.132884903, -0.0517682859, 0.0169064092, -0.00312657789};
  static const double kShort16[3] = {-0.333281593, 0.132053597, -0.0447506447};
  Scale s = {};
  s.cap = cap;
  s.inv_temp = (float)(1.0 / (double)temp);
  if (!(cap > 0.f)) return s;
  const double r = 1.0 / ((double)cap * cap), k = 1.4426950408889634 / (double)temp;
  s.slope = (float)-r;
  s.twice = (float)(2.0 * 1.4426950408889634 / (double)cap);
  // (c^12 has to be an fp32 number; other caps take tanhf)
  s.limit = cap > 4e-3f && cap < 400.f ? cap * cap : -1.f;
  if (s.limit < 0.f) return s;
  auto twice = [](double v) {
    const float f = (float)v;
    uint32_t bits;
    memcpy(&bits, &f, 4);
    return (f32x2)bits << 32 | bits;
  };
  auto fill_p = [&](f32x2* to, const double* q, int n, double scale) {  // scale (1 + v Q)
    to[0] = twice(scale);
    double p = scale * r;
    for (int i = 0; i < n; ++i, p *= r) to[i + 1] = twice(q[i] * p);
  };
  auto fill_q = [&](f32x2* to, const double* q, int n) {
    double p = r;
    for (int i = 0; i < n; ++i, p *= r) to[i] = twice(q[i] * p);
  };
  fill_p(s.sum_full, kFull, 6, k);
  fill_p(s.sum_short, kShort, 4, k);
  fill_p(s.z_full, kFull16, 5, 1.0);
  fill_p(s.z_short, kShort16, 3, 1.0);
  fill_q(s.q_full, kFull, 6);
  fill_q(s.q_short, kShort, 4);
  return s;
}

// z of kV vectors (kExponent false), or the exponents z log2 e / tau - shift (true). `whole`: every lane of the
// warp is here.
template <typename T, bool kExponent, bool kWhole, int kV>
ME_DEVICE void vec_softcap(const uint4 (&x)[kV], const Scale& sc, float shift, f32x2 (&z)[kV][Vec16<T>::kN / 2]) {
  constexpr int kP = Vec16<T>::kN / 2;
  const float k = sc.inv_temp * kLog2e;
  float top = 0.f;
#pragma unroll
  for (int u = 0; u < kV; ++u) {
    to_pairs<T>(x[u], z[u]);
#pragma unroll
    for (int p = 0; p < kP; ++p) {
      const float2 v = unpack2(mul2(z[u][p], z[u][p]));
      asm("max.f32 %0, %0, %1, %2;" : "+f"(top) : "f"(v.x), "f"(v.y));  // a NaN is passed over, and stays in x
    }
  }
  auto all = [&](auto&& f) {
#pragma unroll
    for (int u = 0; u < kV; ++u)
#pragma unroll
      for (int p = 0; p < kP; ++p) z[u][p] = f(z[u][p]);
  };
  auto poly = [&](const auto& sum, const auto& low, const auto& q) {
    all([&](f32x2 a) {
      const f32x2 v = mul2(a, a);
      if constexpr (sizeof(T) == 4) {
        const f32x2 r = fma2(mul2(a, v), horner2(q, v), a);
        return kExponent ? fma2(r, both2(k), both2(-shift)) : r;
      } else {
        return kExponent ? fma2(a, horner2(sum, v), both2(-shift)) : mul2(a, horner2(low, v));
      }
    });
  };
  // (the warp takes the short polynomial together: a divided warp would pay for both)
  if (kWhole && __all_sync(0xffffffffu, top <= 0.25f * sc.limit)) {
    poly(sc.sum_short, sc.z_short, sc.q_short);
  } else if (top <= sc.limit) {
    poly(sc.sum_full, sc.z_full, sc.q_full);
  } else if (sc.limit > 0.f) {
    // Some logit is beyond the cap: there c (1 - 2 / (e^(2 |u|) + 1)) by the special function unit, whose error the
    // small second term scales down (to 2e-6 at c = 30); the polynomial for the others.
    all([&](f32x2 a) {
      const f32x2 v = mul2(a, a);
      const float2 f = unpack2(a), near = unpack2(fma2(mul2(a, v), horner2(sc.q_full, v), a));
      float r[2] = {near.x, near.y};
#pragma unroll
      for (int l = 0; l < 2; ++l) {
        const float x = l ? f.y : f.x, size = fabsf(x);
        const float t = fmaf(-2.f, rcp_fast(exp2_fast(size * sc.twice) + 1.f), 1.f);
        if (size > sc.cap) r[l] = copysignf(sc.cap * t, x);
      }
      const f32x2 z2 = pack2(r[0], r[1]);
      return kExponent ? fma2(z2, both2(k), both2(-shift)) : z2;
    });
  } else {
#pragma unroll
    for (int u = 0; u < kV; ++u) {
#pragma unroll 1
      for (int i = 0; i < kP; ++i) {
        // (a loop that is not unrolled would index the pairs in local memory: rotate them instead)
        const float2 f = unpack2(z[u][0]);
        float a = softcap(f.x, sc.cap), b = softcap(f.y, sc.cap);
        if (kExponent) {
          a = fmaf(a, k, -shift);
          b = fmaf(b, k, -shift);
        }
#pragma unroll
        for (int o = 0; o + 1 < kP; ++o) z[u][o] = z[u][o + 1];
        z[u][kP - 1] = pack2(a, b);
      }
    }
  }
}

// e^d of a pair, -87 <= d <= 88: the argument is reduced as in Cody and Waite, "Software Manual for the Elementary
// Functions" (1980), chapter 6: n = d / ln 2 rounded to a whole number, r = d - n ln 2, e^d = 2^n e^r. An FMA forms
// d - n ln 2 with one rounding, at the size of r, so the first of their two constants is enough: what fp32 leaves out
// of ln 2 (1.9e-9) moves e^d by 3e-8 at d = -10. e^r is ex2 of r log2 e, |r| <= 0.35, and 2^n goes onto the exponent.
// (ex2 of d log2 e itself carries that product's rounding, up to 5e-7 at d = -10, into a sum of many terms.) A NaN gives
// a NaN or 3e38: either way the sum that it enters is out of range.
ME_DEVICE f32x2 exp_pair(f32x2 d) {
  const float kWhole = 12582912.f;  // 1.5 * 2^23: the fp32 numbers around it are the whole ones
  const float kLn2 = 0.693147180559945309f;
  const f32x2 t = fma2(d, both2(kLog2e), both2(kWhole));  // n + 1.5 * 2^23: n stands in the low bits
  const f32x2 r = fma2(add2(t, both2(-kWhole)), both2(-kLn2), d);
  const float2 g = unpack2(mul2(r, both2(kLog2e))), n = unpack2(t);
  return pack2(__uint_as_float(__float_as_uint(exp2_fast(g.x)) + (__float_as_uint(n.x) << 23)),
               __uint_as_float(__float_as_uint(exp2_fast(g.y)) + (__float_as_uint(n.y) << 23)));
}
// max(a, b) that keeps a NaN
ME_DEVICE float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

constexpr int kThreads = 256;  // of every block that walks a row

// A logits matrix and its rows' stride in elements.
template <typename T>
struct Rows {
  T* base;
  int64_t stride;
  ME_DEVICE T* row(int64_t r) const { return base + r * stride; }
};

// A block's share of one row: 16-byte vectors [begin, end) from `head` on, and for the row's first and
// last block the elements ahead of the first 16-byte boundary and after the last one. (V is at most kMaxColumns.)
template <typename T>
struct Slice {
  static constexpr int kN = Vec16<T>::kN;
  const T* row;
  int V, head, body_end;  // columns [head, body_end) are vectors
  int begin, end;         // of them, this block's
  bool first, last;

  // the row's blocks are 2^lg_ranks
  ME_DEVICE Slice(const T* row_, int V_, int rank, int lg_ranks) : row(row_), V(V_) {
    head = (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(T);
    head = min(head, V);
    const int nvec = (V - head) / kN, per = (nvec + (1 << lg_ranks) - 1) >> lg_ranks;
    body_end = head + nvec * kN;
    begin = (int)min((long long)nvec, (long long)rank * per);
    end = min(nvec - begin, per) + begin;
    first = rank == 0;
    last = rank == (1 << lg_ranks) - 1;
  }
  // This thread's vectors: how many, the i-th one's number in the row, where the first one is.
  ME_DEVICE int count() const { return (end - begin + kThreads - 1 - (int)threadIdx.x) / kThreads; }
  ME_DEVICE int vec(int i) const { return begin + threadIdx.x + i * kThreads; }
  ME_DEVICE const uint4* mine() const { return reinterpret_cast<const uint4*>(row + head) + begin + threadIdx.x; }
  ME_DEVICE int column(int v) const { return head + v * kN; }
  // The block's single columns, one a thread: -1 for the threads that have none.
  ME_DEVICE int single() const {
    const int t = threadIdx.x;
    if (first && t < head) return t;
    if (last && t >= 16 && t - 16 < V - body_end) return body_end + t - 16;
    return -1;
  }
  // Whether a column is this block's.
  ME_DEVICE bool holds(int j) const {
    if (j < head) return first;
    if (j >= body_end) return last;
    const int v = (j - head) / kN;
    return v >= begin && v < end;
  }
};

// Running (m, s): s = sum exp(y - m), m the largest y so far. A NaN or +inf makes s NaN.
struct MaxSum {
  float m = -INFINITY, s = 0.f;
  ME_DEVICE void add(float y) {
    if (y > m) {
      s = s * expf(m - y) + expf(y - y);  // + 1, or NaN for y = inf
      m = y;
    } else if (y != -INFINITY) {  // y NaN: s becomes NaN
      s += expf(y - m);
    }
  }
  ME_DEVICE void merge(MaxSum o) {
    if (o.m == -INFINITY) {
      s += o.s;  // 0, or NaN
    } else if (m == -INFINITY) {
      s += o.s;
      m = o.m;
    } else {
      const float mx = fmaxf(m, o.m);
      s = s * expf(m - mx) + o.s * expf(o.m - mx);
      m = mx;
    }
  }
};

// No column is left out.
struct KeepAll {
  ME_DEVICE uint32_t operator()(int) const { return 0; }
  ME_DEVICE bool column(int) const { return false; }
};

// ---------------------------------------------------------------- a thread's vectors, read ahead
// Each thread copies its own vectors of a slice into its own places of a ring in shared memory,
// kDepth ahead of use (cp.async: no registers are held, no other thread waits): 256 threads keep 32 KB in
// flight a block, four blocks an SM 128 KB, three times what the memory's latency asks for.
constexpr int kDepth = 8;
constexpr int kFirst = 4;  // vectors that the reference of a sum is taken from

struct Ring {
  uint4 v[kDepth][kThreads];
};

ME_DEVICE void copy_async(uint4* to, const uint4* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to)), "l"(from)
               : "memory");
}
ME_DEVICE void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
ME_DEVICE void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory");
}

// first(n, v): the thread's n first vectors (at most kFirst) are there; f(v, i): the array v of vectors from
// the thread's i-th on, two of them while the whole warp is in the loop (kWhole), else one. `src`: its first one,
// the others follow kStep (+-kThreads) apart. Every thread of the block calls it, those without a vector too.
template <int kStep = kThreads, typename First, typename F>
ME_DEVICE void stream(const uint4* src, int count, Ring& ring, First&& first, F&& f) {
  const int tid = threadIdx.x;
  uint4* mine = &ring.v[0][tid];
#pragma unroll
  for (int d = 0; d < kDepth; ++d) {
    if (d < count) copy_async(mine + d * kThreads, src + d * kStep);
    if (d & 1) copy_commit();
  }
  copy_wait<(kDepth - kFirst) / 2>();
  {
    uint4 v[kFirst];
#pragma unroll
    for (int u = 0; u < kFirst; ++u) v[u] = mine[u * kThreads];
    first(min(count, kFirst), v);
  }
  const uint4* next = src + kDepth * kStep;
  const int whole = __shfl_sync(0xffffffffu, count, 31);  // the warp's last lane has the fewest
  int i = 0;
  for (; i + 2 * kDepth <= whole; i += kDepth, next += kDepth * kStep) {
#pragma unroll
    for (int s = 0; s < kDepth; s += 2) {
      copy_wait<kDepth / 2 - 1>();
      const uint4 v[2] = {mine[s * kThreads], mine[(s + 1) * kThreads]};
      f(v, i + s, std::true_type());
      copy_async(mine + s * kThreads, next + s * kStep);
      copy_async(mine + (s + 1) * kThreads, next + (s + 1) * kStep);
      copy_commit();
    }
  }
  // the last vectors: pairs as long as the whole warp has them
#pragma unroll 1
  for (; i + 2 <= whole; i += 2) {
    copy_wait<kDepth / 2 - 1>();
    uint4* at = mine + i % kDepth * kThreads;
    const uint4 v[2] = {at[0], at[kThreads]};
    f(v, i, std::true_type());
#pragma unroll
    for (int u = 0; u < 2; ++u)
      if (i + u + kDepth < count) copy_async(at + u * kThreads, src + (i + u + kDepth) * kStep);
    copy_commit();
  }
#pragma unroll 1
  for (; i < count; i += 2) {
    copy_wait<kDepth / 2 - 1>();
#pragma unroll 1
    for (int u = 0; u < 2 && i + u < count; ++u) {
      const uint4 v[1] = {mine[(i + u) % kDepth * kThreads]};
      f(v, i + u, std::false_type());
    }
    copy_commit();
  }
}

// This thread's share of sum exp(y - m) over a slice. `drop(vec)`: a mask of the vector's elements
// that are left out (`drop.column(j)` for a single column).
//
// One pass with a fixed reference: the largest z of the thread's first vectors, so no running maximum
// is carried. A share that this does not suit (a sum out of range, a NaN or +inf anywhere) is added again element by element with a running maximum.
//
// With a softcap the exponential is ex2 of the difference times log2 e / tau (an argument's rounding
// moves a term by 1e-6 at c / tau = 30 and 3e-6 at most, and the softcap's own rounding is as large); without one exp_pair(),
// since nothing else is rounded then.
// watch(x, i): sees the thread's vectors from the i-th on, one or two at a time, in order.
struct WatchNothing {
  template <typename X>
  ME_DEVICE void operator()(const X&, int) const {}
};
template <typename T, bool kCap, typename Drop, typename Watch = WatchNothing>
ME_DEVICE MaxSum slice_sum(const Slice<T>& sl, const Scale& sc, const Drop& drop, Ring& ring, Watch&& watch = Watch()) {
  constexpr int kN = Vec16<T>::kN, kP = kN / 2;
  MaxSum out;
  const int count = sl.count();
  MaxOf<T> big;
  float sum0 = 0.f, sum1 = 0.f;
  const float k = sc.inv_temp * kLog2e;
  float ref = 0.f, shift = 0.f;  // the reference; the same, or the rounded ref k
  stream(
      sl.mine(), count, ring,
      [&](int n, const uint4(&v)[kFirst]) {
        MaxOf<T> top;
#pragma unroll
        for (int u = 0; u < kFirst; ++u)
          if (u < n) top.add(v[u]);
        // (masked columns only, -inf or the type's lowest: 0 suits the others as well as any)
        const float lowest = std::is_same_v<T, __half> ? -65504.f : -1e38f;
        ref = kCap ? softcap(top.value(), sc.cap) : top.value() > lowest ? top.value() * sc.inv_temp : 0.f;
        shift = kCap ? ref * k : ref;
      },
      [&](const auto& x, int i, auto whole) {
        constexpr int kV = sizeof(x) / sizeof(uint4);
        f32x2 y[kV][kP];
        watch(x, i);
        if constexpr (kCap) {
          vec_softcap<T, true, decltype(whole)::value>(x, sc, shift, y);
        } else {
#pragma unroll
          for (int u = 0; u < kV; ++u) {
            to_pairs<T>(x[u], y[u]);
            big.add(x[u]);
          }
        }
#pragma unroll
        for (int u = 0; u < kV; ++u) {
          if (!std::is_same_v<Drop, KeepAll>) {
            const uint32_t out_mask = drop(sl.vec(i + u));
            if (out_mask) {
              const float gone = kCap ? -200.f : -INFINITY;
#pragma unroll
              for (int p = 0; p < kP; ++p) {
                float2 f = unpack2(y[u][p]);
                if (out_mask >> (2 * p) & 1) f.x = gone;
                if (out_mask >> (2 * p) & 2) f.y = gone;
                y[u][p] = pack2(f.x, f.y);
              }
            }
          }
#pragma unroll
          for (int p = 0; p < kP; ++p) {
            float2 d = unpack2(kCap ? y[u][p] : fma2(y[u][p], both2(sc.inv_temp), both2(-shift)));
            if constexpr (!kCap) {
              d.x = max_nan(d.x, -87.f);
              d.y = max_nan(d.y, -87.f);
            }
            if constexpr (kCap) {
              d.x = exp2_fast(d.x);
              d.y = exp2_fast(d.y);
            } else {
              d = unpack2(exp_pair(pack2(d.x, d.y)));
            }
            sum0 += d.x;
            sum1 += d.y;
          }
        }
      });
  const float s = sum0 + sum1;
  // exp_pair's range; ex2 leaves its own with an infinity, which the sum shows. (Not the largest exponent that the cap
  // allows: that sent every row with 2 cap / tau near 160 to the slow form, 122 -> 801 us for top logits of 1024 x 262144.)
  const bool in_range = kCap || big.value() * sc.inv_temp - ref < 80.f;
  if (count > 0 && s > 1e-20f && s < 1e37f && in_range) {  // (masked columns add 2e-38 each)
    // (m is rounded: what separates it from the shift that was taken goes into s)
    out.m = kCap ? ref * sc.inv_temp : ref;
    out.s = kCap ? s * exp2_fast((float)(shift - 1.4426950408889634 * out.m)) : s;
    // A reference far below the largest: a gradient's coefficient over s has to stay a normal number, so m takes the
    // whole part of log s (the exponential is of an exact argument; m's own rounding goes into s).
    if (out.s > 1e12f) {
      const float up = rintf(logf(out.s));
      const double m = (double)out.m + up;
      out.m = (float)m;
      out.s *= expf(-up) * (1.f + (float)(m - out.m));
    }
  } else {
    for (int i = 0; i < count; ++i) {
      const uint32_t out_mask = drop(sl.vec(i));
      for (int e = 0; e < kN; ++e)
        if (!(out_mask >> e & 1)) out.add(softcap(to_f<T>(sl.row[sl.column(sl.vec(i)) + e]), sc.cap) * sc.inv_temp);
    }
  }
  const int j = sl.single();
  if (j >= 0 && !drop.column(j)) out.add(softcap(to_f<T>(sl.row[j]), sc.cap) * sc.inv_temp);
  return out;
}

// The warp's (m, s), the same for every lane: one exponential a lane.
ME_DEVICE MaxSum warp_merge(MaxSum a) {
  MaxSum r;
  r.m = warp_max(a.m);
  // (m = -inf: s is 0 or NaN)
  r.s = warp_sum(a.m == -INFINITY ? a.s : a.s * expf(a.m - r.m));
  return r;
}

// ---------------------------------------------------------------- thread-block clusters
// (.aligned: the lanes of a warp have to execute them together, whatever divergent code came before)
ME_DEVICE void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
ME_DEVICE void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A pair in the shared memory of the cluster's block `rank`, at the place that `p` has in this one.
ME_DEVICE float2 cluster_load(const float2* p, uint32_t rank) {
  uint32_t a = (uint32_t)__cvta_generic_to_shared(p), b;
  float2 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"(a), "r"(rank));
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(b) : "memory");
  return v;
}

constexpr int kWarps = kThreads / 32;

// A row's (m, s) from its threads', the same bits for every thread of the cluster: the warps' pairs are
// exchanged behind one barrier. Where there is more than one block, row_done() has to follow before
// the block leaves (others may still read its pairs).
ME_DEVICE MaxSum row_merge(MaxSum a, float2* part, int lg_ranks) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  a = warp_merge(a);
  if (lane == 0) part[wid] = make_float2(a.m, a.s);
  MaxSum r;
  if (lg_ranks == 0) {
    __syncthreads();
    if (lane < kWarps) {
      r.m = part[lane].x;
      r.s = part[lane].y;
    }
  } else {
    cluster_arrive();
    cluster_wait();
    for (int i = lane; i < kWarps << lg_ranks; i += 32) {
      const float2 o = cluster_load(part + i % kWarps, i / kWarps);
      MaxSum b;
      b.m = o.x;
      b.s = o.y;
      r.merge(b);
    }
    cluster_arrive();
  }
  return warp_merge(r);
}
ME_DEVICE void row_done(int lg_ranks) {
  if (lg_ranks > 0) cluster_wait();
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

// Launches `kernel` on `grid` blocks of kThreads in clusters of `cluster`.
template <typename... Params, typename... Args>
cudaError_t launch_cluster(void (*kernel)(Params...), int64_t grid, int cluster, int smem, cudaStream_t stream,
                           Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, Params(args)...);
}

inline int ilog2(int c) {
  int l = 0;
  while (1 << l < c) ++l;
  return l;
}

// Blocks a row: enough for `per_sm` on each SM, while a block keeps two vectors a thread. (2048 rows of 262144 bf16
// logits, summed by 1 / 2 / 4 / 8 blocks a row: 207 / 217 / 233 / 259 us; 5 rows by 1 / 8: 31 / 9 us. Four blocks
// an SM instead of two: 515 x 100003 distilled in 97 instead of 102 us, 301 x 50001 preferred in 29 instead of 31.)
inline int ranks_for(int64_t N, int64_t V, int per_sm = 4) {
  int c = 1;
  while (c < 8 && N * c < per_sm * objective_sms() && V / (2 * c) >= 4096) c *= 2;
  return c;
}
// The same for the backward pass alone, whose blocks do not wait for one another: as many as leave a thread 16
// vectors (the preference step with 1024 of 2048 rows of 262144 trained, by 1 / 2 / 4 / 8: 397 / 385 / 372 / 366 us).
inline int ranks_for_gradient(const Logits& x) {
  const int64_t vecs = x.V * (x.type == LogitType::kF32 ? 4 : 2) / 16;
  int c = ranks_for(x.N, x.V);
  while (c < 8 && vecs / (2 * c) >= 16 * kThreads) c *= 2;
  return c;
}

// And for value and gradient in one kernel, which reads a row twice. More blocks a row: fewer rows in flight, so that the
// second read finds them in L2; but what a block does once a row counts for more. 16-bit logits with a softcap are
// bound by arithmetic: two where a thread keeps 32 vectors then (1024 x 262144 by 1 / 2 / 4 / 8: 277 / 262 / 264 /
// 298 us; 100000: 116 / 118 / 145 / 185). The others by memory: until the rows in flight take 64 MB, while a thread
// keeps 16 vectors (bf16 without a cap, 262144: 258 / 254 / 238 / 219, 100000: 103 / 95 / 113 / 150; fp32, 262144:
// 505 / 503 / 488 / 460, 100000: 204 / 197 / 178 / 226).
inline int ranks_for_both(const Logits& x) {
  const int64_t row = x.V * (x.type == LogitType::kF32 ? 4 : 2), vecs = row / 16;
  int c = ranks_for(x.N, x.V);
  if (x.cap > 0.f && x.type != LogitType::kF32) return c == 1 && vecs / 2 >= 32 * kThreads ? 2 : c;
  while (c < 8 && 4 * objective_sms() / c * row > (64 << 20) && vecs / (2 * c) >= 16 * kThreads) c *= 2;
  return c;
}

// Lets a kernel have more than 48 KB of shared memory, the ring and `bytes` at the launch.
template <typename K>
void allow_smem(K* kernel, int bytes) {
  if (bytes > (8 << 10)) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
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

#define ME_CAP_DISPATCH(CAP, ...)        \
  if ((CAP) > 0.f) {                     \
    constexpr bool kCap = true;          \
    __VA_ARGS__;                         \
  } else {                               \
    constexpr bool kCap = false;         \
    __VA_ARGS__;                         \
  }

}  // namespace me

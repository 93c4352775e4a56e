// Objectives over the vocabulary: token log-probabilities and distillation from a teacher's top
// logits, value and gradient, over rows of logits x [N, V] (sm_100a).
//
// z = c tanh(x / c) (or x), y = z / tau, lse = log sum_j exp(y_j), p_j = exp(y_j - lse).
//   log-probability   lp = z_t - lse                        d lp / d x_j = ([j = t] - p_j) z'_j
//   distillation      L = w tau^2 [sum_k q_k (log q_k - log p_k) + q_r (log q_r - log p_r)]
//                     dL / d x_j = w tau z'_j [p_j rho_j - sum_{k: id_k = j} q_k]
// with q the teacher's probabilities of its entries: renormalised over them (then q_r = 0 and
// rho = 1), or exp(t_k / tau - lse_T) with everything else as one class of its own: q_r = 1 - sum q
// (0 where the entries sum to more than 1), p_r = the student's probability outside the entries,
// rho_j = M - [j no entry] q_r / p_r, M = sum q + q_r. For the columns that are no entry
// p_j rho_j = exp(y_j - m') c' with m' their largest y and c' = M exp(m' - lse) - q_r / sum exp(y - m'):
// one exponential, and no overflow where the student's rest is tiny.
// Each row's statistics (m, s), lse = m + log s, are kept in fp32; sums have a fixed order.
#include "objectives.cuh"

#include <algorithm>

using namespace me;

namespace {

constexpr int kThreads = 512;
constexpr int kBloom = 32768;  // bits of the filter that says which vectors may hold a teacher entry

// A row of the teacher's records in shared memory.
struct Teacher {
  int id[kMaxTop];       // < 0: an unused entry
  float t[kMaxTop];      // t_k / tau
  float q[kMaxTop];      // probability
  float x[kMaxTop];      // the student's raw logit
  uint32_t bloom[kBloom / 32];
  float m, log_s;        // log q_k = (t_k - m) - log_s
  float q_rest;          // the rest's probability
  float mass;            // sum q + q_rest
};

// Loads row r's entries: ids outside [0, V) are unused, q from the temperature-scaled logits.
template <typename T>
ME_DEVICE void load_teacher(Teacher& te, const TeacherArgs& a, int64_t r, const T* row, int64_t V, float inv_temp,
                            float* scratch) {
  MaxSum ms;
  for (int k = threadIdx.x; k < a.k; k += blockDim.x) {
    const int64_t id = a.ids[r * a.k + k];
    const bool used = id >= 0 && id < V;
    te.id[k] = used ? (int)id : -1;
    te.t[k] = used ? a.top[r * a.k + k] * inv_temp : -INFINITY;
    te.x[k] = used ? to_f<T>(row[id]) : 0.f;
    if (used) ms.add(te.t[k]);
  }
  if (a.lse) {
    for (int i = threadIdx.x; i < kBloom / 32; i += blockDim.x) te.bloom[i] = 0;
  }
  ms = block_merge(ms, scratch);
  const float m = a.lse ? a.lse[r] : ms.m, log_s = a.lse ? 0.f : logf(ms.s), inv_s = a.lse ? 1.f : 1.f / ms.s;
  float sum = 0.f, used = 0.f;
  for (int k = threadIdx.x; k < a.k; k += blockDim.x) {
    const float q = te.t[k] == -INFINITY ? 0.f : expf(te.t[k] - m) * inv_s;
    te.q[k] = q;
    sum += q;
    if (te.id[k] >= 0) used += 1.f;
    if (a.lse && te.id[k] >= 0) {
      const int b = (te.id[k] >> 3) & (kBloom - 1);
      atomicOr(&te.bloom[b >> 5], 1u << (b & 31));
    }
  }
  const float2 both = block_sum2(sum, used, scratch);
  if (threadIdx.x == 0) {
    te.m = m;
    te.log_s = log_s;
    // no rest where the entries are the whole vocabulary: 1 - sum is rounding then
    te.q_rest = a.lse && both.y < (float)V ? fmaxf(0.f, 1.f - both.x) : 0.f;
    te.mass = a.lse ? both.x + te.q_rest : 1.f;
  }
  __syncthreads();
}

ME_DEVICE bool is_entry(const Teacher& te, int k, int64_t j) {
  const int b = (int)(j >> 3) & (kBloom - 1);
  if (!((te.bloom[b >> 5] >> (b & 31)) & 1)) return false;
  for (int i = 0; i < k; ++i)
    if (te.id[i] == (int)j) return true;
  return false;
}

// ------------------------------------------------------------------------------------ forward
template <typename T>
__global__ void __launch_bounds__(kThreads) logprob_fwd_kernel(Rows<const T> x, int64_t N, int64_t V,
                                                               const int64_t* __restrict__ target, float cap,
                                                               float* __restrict__ logp, float2* __restrict__ stats) {
  __shared__ float scratch[64];
  for (int64_t r = blockIdx.x; r < N; r += gridDim.x) {
    const int64_t t = target[r];
    if (t == kIgnoreToken) {
      if (threadIdx.x == 0) {
        logp[r] = 0.f;
        stats[r] = make_float2(0.f, 1.f);
      }
      continue;
    }
    const T* row = x.row(r);
    MaxSum a;
    for_row<T>(row, V, [&](int64_t, float v) { a.add(softcap(v, cap)); });
    a = block_merge(a, scratch);
    if (threadIdx.x == 0) {
      logp[r] = t >= 0 && t < V ? softcap(to_f<T>(row[t]), cap) - a.m - logf(a.s) : NAN;
      stats[r] = make_float2(a.m, a.s);
    }
  }
}

// stats: m, s (-1: a row without gradient), m', c'; without teacher_lse m' = m, c' = 1 / s
template <typename T>
__global__ void __launch_bounds__(kThreads) distill_fwd_kernel(Rows<const T> x, int64_t N, int64_t V, TeacherArgs ta,
                                                               float cap, float* __restrict__ loss,
                                                               float4* __restrict__ stats) {
  __shared__ Teacher te;
  __shared__ float scratch[64];
  const float temp = ta.temp, inv_temp = 1.f / temp;
  for (int64_t r = blockIdx.x; r < N; r += gridDim.x) {
    const float w = ta.weight ? ta.weight[r] : 1.f;
    if (w == 0.f) {
      if (threadIdx.x == 0) {
        loss[r] = 0.f;
        stats[r] = make_float4(0.f, -1.f, 0.f, 0.f);
      }
      continue;
    }
    const T* row = x.row(r);
    load_teacher<T>(te, ta, r, row, V, inv_temp, scratch);
    MaxSum a, rest;
    for_row<T>(row, V, [&](int64_t j, float v) {
      const float y = softcap(v, cap) * inv_temp;
      if (ta.lse && is_entry(te, ta.k, j)) a.add(y);
      else rest.add(y);
    });
    a = block_merge(a, scratch);
    rest = block_merge(rest, scratch);
    a.merge(rest.m, rest.s);
    const float log_s = logf(a.s);
    float sum = 0.f, used = 0.f;
    for (int k = threadIdx.x; k < ta.k; k += blockDim.x) {
      const float q = te.q[k];
      if (q != 0.f) {
        // maxima first: what is left to round is of the size of the difference
        const float y = softcap(te.x[k], cap) * inv_temp;
        sum += q * (((te.t[k] - te.m) - (y - a.m)) + (log_s - te.log_s));
      }
      if (q != 0.f) used += 1.f;
    }
    const float2 both = block_sum2(sum, used, scratch);
    if (threadIdx.x == 0) {
      float kl = both.x, m1 = a.m, c1 = 1.f / a.s;
      if (ta.lse) {
        const float log_rest = rest.m == -INFINITY ? -INFINITY : rest.m - a.m + (logf(rest.s) - log_s);
        if (te.q_rest > 0.f) kl += te.q_rest * (logf(te.q_rest) - log_rest);
        const bool some = rest.m != -INFINITY;
        m1 = some ? rest.m : 0.f;
        c1 = some ? te.mass * (expf(rest.m - a.m) / a.s) - te.q_rest / rest.s : 0.f * a.s;
      } else if (both.y == 0.f) {  // no entry: nothing to match
        kl = 0.f;
        a.s = -1.f;
      }
      loss[r] = w * temp * temp * kl;
      stats[r] = make_float4(a.m, a.s, m1, c1);
    }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------ backward
template <typename T, typename F>
ME_DEVICE void write_row(const T* row, T* out, int64_t V, F&& f) {
  for (int64_t j = threadIdx.x; j < V; j += blockDim.x) out[j] = from_f<T>(f(j, to_f<T>(row[j])));
}

template <typename T>
ME_DEVICE void zero_row(T* out, int64_t V) {
  for (int64_t j = threadIdx.x; j < V; j += blockDim.x) out[j] = from_f<T>(0.f);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) logprob_bwd_kernel(Rows<const T> x, Rows<T> out, int64_t N, int64_t V,
                                                               const int64_t* __restrict__ target, float cap,
                                                               const float2* __restrict__ stats,
                                                               const float* __restrict__ g) {
  for (int64_t r = blockIdx.x; r < N; r += gridDim.x) {
    const int64_t t = target[r];
    T* o = out.row(r);
    if (t == kIgnoreToken) {
      zero_row<T>(o, V);
      continue;
    }
    const float2 ms = stats[r];
    const float c = t >= 0 && t < V ? g[r] : NAN, inv_s = 1.f / ms.y;
    write_row<T>(x.row(r), o, V, [&](int64_t j, float v) {
      const float z = softcap(v, cap);
      const float p = exp2_fast((z - ms.x) * kLog2e) * inv_s;
      return c * ((j == t ? 1.f : 0.f) - p) * softcap_slope(z, cap);
    });
  }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) distill_bwd_kernel(Rows<const T> x, Rows<T> out, int64_t N, int64_t V,
                                                               TeacherArgs ta, float cap,
                                                               const float4* __restrict__ stats,
                                                               const float* __restrict__ g) {
  __shared__ Teacher te;
  __shared__ float scratch[64];
  const float temp = ta.temp, inv_temp = 1.f / temp;
  for (int64_t r = blockIdx.x; r < N; r += gridDim.x) {
    const float w = ta.weight ? ta.weight[r] : 1.f;
    const float4 st = stats[r];
    T* o = out.row(r);
    if (st.y == -1.f) {
      zero_row<T>(o, V);
      continue;
    }
    const T* row = x.row(r);
    load_teacher<T>(te, ta, r, row, V, inv_temp, scratch);
    const float c = w * temp * (g ? g[r] : 1.f), inv_s = 1.f / st.y;
    write_row<T>(row, o, V, [&](int64_t, float v) {
      const float z = softcap(v, cap);
      return c * st.w * exp2_fast((z * inv_temp - st.z) * kLog2e) * softcap_slope(z, cap);
    });
    __syncthreads();  // the entries' own columns are written again
    for (int k = threadIdx.x; k < ta.k; k += blockDim.x) {
      const int id = te.id[k];
      if (id < 0) continue;
      float q = 0.f;
      bool first = true;
      for (int i = 0; i < ta.k; ++i) {
        if (te.id[i] != id) continue;
        first = first && i >= k;
        q += te.q[i];
      }
      if (!first) continue;
      const float z = softcap(te.x[k], cap);
      const float p = exp2_fast((z * inv_temp - st.x) * kLog2e) * inv_s;
      o[id] = from_f<T>(c * (p * te.mass - q) * softcap_slope(z, cap));
    }
    __syncthreads();
  }
}

int grid_of(int64_t N) { return (int)std::min<int64_t>(N, (int64_t)objective_sms() * 4); }

}  // namespace

namespace me {

void launch_logprob_fwd(const Logits& x, const int64_t* target, float* logp, float2* stats, cudaStream_t stream) {
  ME_LOGITS_DISPATCH(x.type, logprob_fwd_kernel<T><<<grid_of(x.N), kThreads, 0, stream>>>(
                                 rows_in<T>(x), x.N, x.V, target, x.cap, logp, stats));
}

void launch_logprob_bwd(const Logits& x, const int64_t* target, const float2* stats, const float* g, Gradient out,
                        cudaStream_t stream) {
  ME_LOGITS_DISPATCH(x.type, logprob_bwd_kernel<T><<<grid_of(x.N), kThreads, 0, stream>>>(
                                 rows_in<T>(x), rows_out<T>(out), x.N, x.V, target, x.cap, stats, g));
}

void launch_distill_fwd(const Logits& x, const TeacherArgs& teacher, float* loss, float4* stats, cudaStream_t stream) {
  ME_LOGITS_DISPATCH(x.type, distill_fwd_kernel<T><<<grid_of(x.N), kThreads, 0, stream>>>(
                                 rows_in<T>(x), x.N, x.V, teacher, x.cap, loss, stats));
}

void launch_distill_bwd(const Logits& x, const TeacherArgs& teacher, const float4* stats, const float* g, Gradient out,
                        cudaStream_t stream) {
  ME_LOGITS_DISPATCH(x.type, distill_bwd_kernel<T><<<grid_of(x.N), kThreads, 0, stream>>>(
                                 rows_in<T>(x), rows_out<T>(out), x.N, x.V, teacher, x.cap, stats, g));
}

}  // namespace me

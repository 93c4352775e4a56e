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

static_assert(kThreads >= kMaxTop, "one teacher entry a thread");
constexpr int kFilter = 16384;  // bits of the filter that says which vectors may hold a teacher entry

struct Shared {
  Ring ring;
  float scratch[64];
  float part[2];  // this block's (m, s), read by the cluster's other blocks
};

// The row's (m, s) from its blocks' (all threads of all blocks get the same); `s` may be NaN.
ME_DEVICE MaxSum cluster_merge(const float* part, int ranks) {
  const int lane = threadIdx.x & 31;
  MaxSum a;
  if (lane < ranks) {
    a.m = cluster_load(part, lane);
    a.s = cluster_load(part + 1, lane);
  }
  MaxSum r;
  r.m = warp_max(a.m);
  r.s = warp_sum(a.m == -INFINITY ? a.s : a.s * expf(a.m - r.m));
  return r;
}

// Adds a row's exponentials over its cluster, the same result for every thread. Ends after a cluster
// arrival: cluster_wait() has to follow before the block leaves (its `part` may still be read).
template <typename T, bool kCap, typename Drop>
ME_DEVICE MaxSum row_sum(const Slice<T>& sl, const Scale& sc, const Drop& drop, Shared& sh, int ranks) {
  MaxSum a = block_merge(slice_sum<T, kCap>(sl, sc, drop, sh.ring), sh.scratch);
  if (ranks == 1) return a;
  if (threadIdx.x == 0) {
    sh.part[0] = a.m;
    sh.part[1] = a.s;
  }
  cluster_arrive();
  cluster_wait();
  a = cluster_merge(sh.part, ranks);
  cluster_arrive();
  return a;
}
ME_DEVICE void row_done(int ranks) {
  if (ranks > 1) cluster_wait();
}

// ------------------------------------------------------------------------------------ gradient of a slice
// out_j = coef exp(y_j - m) z'_j for the block's columns, in 16-byte stores where the two rows are
// aligned alike.
template <typename T, bool kCap>
ME_DEVICE void write_slice(const Slice<T>& sl, T* out, const Scale& sc, float m, float coef, Ring& ring) {
  constexpr int kN = Vec16<T>::kN, kP = kN / 2;
  const bool aligned = (reinterpret_cast<uintptr_t>(out + sl.head) & 15) == 0;
  // coef (1 - (z / c)^2) is one FMA with the coefficient inside
  const float coef_slope = coef * sc.slope;
  stream(
      sl.mine(), sl.count(), ring, [](int, auto&) {},
      [&](const auto& x, int i, auto whole) {
        constexpr int kV = sizeof(x) / sizeof(uint4);
        f32x2 z[kV][kP];
        if constexpr (kCap) {
          vec_softcap<T, false, decltype(whole)::value>(x, sc, 0.f, z);
        } else {
#pragma unroll
          for (int u = 0; u < kV; ++u) to_pairs<T>(x[u], z[u]);
        }
#pragma unroll
        for (int u = 0; u < kV; ++u) {
#pragma unroll
          for (int p = 0; p < kP; ++p) {
            const f32x2 zp = z[u][p];
            const float2 a = unpack2(mul2(fma2(zp, both2(sc.inv_temp), both2(-m)), both2(kLog2e)));
            const f32x2 e = pack2(exp2_fast(a.x), exp2_fast(a.y));
            z[u][p] = mul2(e, kCap ? fma2(mul2(zp, both2(coef_slope)), zp, both2(coef)) : both2(coef));
          }
          Vec16<T> r;
          r.u = from_pairs<T>(z[u]);
          const int64_t at = sl.vec(i + u);
          if (aligned) {
            reinterpret_cast<uint4*>(out + sl.head)[at] = r.u;
          } else {
#pragma unroll
            for (int e = 0; e < kN; ++e) out[sl.column(at) + e] = r.h[e];
          }
        }
      });
  const int64_t j = sl.single();
  if (j >= 0) {
    const float z = softcap(to_f<T>(sl.row[j]), sc.cap);
    out[j] = from_f<T>(coef * exp2_fast((z * sc.inv_temp - m) * kLog2e) * softcap_slope(z, sc.cap));
  }
}

template <typename T>
ME_DEVICE void zero_slice(const Slice<T>& sl, T* out) {
  const int64_t head = ((16 - (reinterpret_cast<uintptr_t>(out) & 15)) & 15) / sizeof(T);
  if (head == sl.head || sl.begin >= sl.end) {
    for (int64_t i = sl.begin + threadIdx.x; i < sl.end; i += blockDim.x)
      reinterpret_cast<uint4*>(out + sl.head)[i] = make_uint4(0, 0, 0, 0);
  } else {
    for (int64_t j = sl.column(sl.begin) + threadIdx.x; j < sl.column(sl.end); j += blockDim.x)
      out[j] = from_f<T>(0.f);
  }
  const int64_t j = sl.single();
  if (j >= 0) out[j] = from_f<T>(0.f);
}

// ------------------------------------------------------------------------------------ log-probabilities
template <typename T, bool kCap>
__global__ void __launch_bounds__(kThreads, 4) logprob_fwd_kernel(Rows<const T> x, int64_t V, int ranks,
                                                                  const int64_t* __restrict__ target, Scale sc,
                                                                  float* __restrict__ logp,
                                                                  float2* __restrict__ stats) {
  __shared__ Shared sh;
  const int64_t r = blockIdx.x / ranks;
  const int rank = blockIdx.x % ranks;
  const int64_t t = target[r];
  if (t == kIgnoreToken) {
    if (threadIdx.x == 0 && rank == 0) {
      logp[r] = 0.f;
      stats[r] = make_float2(0.f, 1.f);
    }
    return;
  }
  const Slice<T> sl(x.row(r), V, rank, ranks);
  const float xt = t >= 0 && t < V ? to_f<T>(sl.row[t]) : NAN;
  const MaxSum a = row_sum<T, kCap>(sl, sc, KeepAll(), sh, ranks);
  if (threadIdx.x == 0 && rank == 0) {
    logp[r] = softcap(xt, sc.cap) - a.m - logf(a.s);
    stats[r] = make_float2(a.m, a.s);
  }
  row_done(ranks);
}

// Rows are taken last to first: where the forward pass just went over them, the last ones are in L2.
template <typename T, bool kCap>
__global__ void __launch_bounds__(kThreads, 4) logprob_bwd_kernel(Rows<const T> x, Rows<T> out, int64_t N, int64_t V,
                                                                  int ranks, const int64_t* __restrict__ target,
                                                                  Scale sc, const float2* __restrict__ stats,
                                                                  const float* __restrict__ g) {
  __shared__ Ring ring;
  const int64_t r = N - 1 - blockIdx.x / ranks;
  const int rank = blockIdx.x % ranks;
  const int64_t t = target[r];
  const Slice<T> sl(x.row(r), V, rank, ranks);
  T* o = out.row(r);
  if (t == kIgnoreToken) {
    zero_slice<T>(sl, o);
    return;
  }
  const bool valid = t >= 0 && t < V, mine = valid && sl.holds(t) && threadIdx.x == 0;
  const float2 ms = stats[r];
  const float c = valid ? g[r] : NAN;
  const float xt = mine ? to_f<T>(sl.row[t]) : 0.f;
  __syncthreads();  // read before the row may be written in place
  write_slice<T, kCap>(sl, o, sc, ms.x, -c / ms.y, ring);
  __syncthreads();  // the target's column is written again
  if (mine) {
    const float z = softcap(xt, sc.cap);
    o[t] = from_f<T>(c * (1.f - expf(z - ms.x) / ms.y) * softcap_slope(z, sc.cap));
  }
}

// ------------------------------------------------------------------------------------ distillation
struct Entries {
  int id[kMaxTop];    // < 0: an unused entry
  float q[kMaxTop];   // probability
};

// A thread's entry of the row's teacher.
struct Entry {
  int id = -1;
  float t = -INFINITY;  // t_k / tau
  float x = 0.f;        // the student's raw logit
  float q = 0.f;        // probability; log q = (t - m) - log_s
  bool first = false;   // no earlier entry has this id
  float q_id = 0.f;     // sum of q over the entries with this id
};
struct TeacherRow {
  float m, log_s;
  float mass;    // sum of q, and of the rest's
  float q_rest;  // the rest's probability
  bool any;      // an entry with q != 0
};

template <typename T>
ME_DEVICE Entry load_entry(const TeacherArgs& a, int64_t r, const T* row, int64_t V, float inv_temp, Entries& en) {
  Entry e;
  if (threadIdx.x < a.k) {
    const int64_t id = a.ids[r * a.k + threadIdx.x];
    if (id >= 0 && id < V) {
      e.id = (int)id;
      e.t = a.top[r * a.k + threadIdx.x] * inv_temp;
      e.x = to_f<T>(row[id]);
    }
  }
  en.id[threadIdx.x] = e.id;
  return e;
}

// Probabilities of the entries; `tail`: all other tokens are one more class.
ME_DEVICE TeacherRow finish_entries(Entry& e, const TeacherArgs& a, int64_t r, int64_t V, bool tail, Entries& en,
                                    float* scratch) {
  TeacherRow te;
  te.m = tail ? a.lse[r] : block_max(e.t, scratch);
  e.q = e.t == -INFINITY ? 0.f : expf(e.t - te.m);
  if (!tail) {
    const float s = block_sum(e.q, scratch);
    e.q = e.q == 0.f ? 0.f : e.q / s;
    te.log_s = logf(s);
  } else {
    te.log_s = 0.f;
  }
  en.q[threadIdx.x] = e.q;
  const float2 sums = block_sum2(e.q, e.id >= 0 ? 1.f : 0.f, scratch);  // (its barriers publish en)
  te.any = __syncthreads_or(e.q != 0.f);
  // no rest where the entries are the whole vocabulary: 1 - sum is rounding then
  te.q_rest = tail && sums.y < (float)V ? fmaxf(0.f, 1.f - sums.x) : 0.f;
  te.mass = tail ? sums.x + te.q_rest : 1.f;
  if (e.id >= 0) {
    e.first = true;
    for (int i = 0; i < a.k; ++i) {
      if (en.id[i] != e.id) continue;
      e.first = e.first && i >= (int)threadIdx.x;
      e.q_id += en.q[i];
    }
  }
  return te;
}

// Leaves the teacher's entries out of a sum. A bit of the filter is set for each vector that holds
// one (and stands for every 16384th vector); such a vector is compared with the list.
template <typename T>
struct DropEntries {
  const uint32_t* filter;
  const Entries* en;
  int k;
  int64_t head;
  ME_DEVICE uint32_t operator()(int64_t vec) const {
    constexpr int kN = Vec16<T>::kN;
    const uint32_t b = (uint32_t)vec & (kFilter - 1);
    if (!(filter[b >> 5] >> (b & 31) & 1)) return 0;
    const int j0 = (int)(head + vec * kN);
    uint32_t mask = 0;
    for (int i = 0; i < k; ++i) {
      const uint32_t d = (uint32_t)(en->id[i] - j0);
      if (d < (uint32_t)kN) mask |= 1u << d;  // an unused entry is negative: never within
    }
    return mask;
  }
  ME_DEVICE bool column(int64_t j) const {
    for (int i = 0; i < k; ++i)
      if (en->id[i] == (int)j) return true;
    return false;
  }
};

// The entries' own columns, after the slice was written without them.
template <typename T>
ME_DEVICE void write_entry(const Slice<T>& sl, T* out, const Entry& e, const Scale& sc, float c, float m, float inv_s,
                           float mass) {
  if (!e.first || !sl.holds(e.id)) return;
  const float z = softcap(e.x, sc.cap);
  out[e.id] = from_f<T>(c * (expf(z * sc.inv_temp - m) * inv_s * mass - e.q_id) * softcap_slope(z, sc.cap));
}

// One cluster a row. Value (and the statistics that the backward pass starts from: m, s (-1: a row
// without gradient), m', c'; without a rest m' = m, c' = 1 / s), or with kGrad value and gradient:
// the slice is read again, from L2, once the cluster has the row's sum.
template <typename T, bool kCap, bool kTail, bool kGrad>
__global__ void __launch_bounds__(kThreads, 4) distill_kernel(Rows<const T> x, Rows<T> out, int64_t V, int ranks,
                                                              TeacherArgs ta, Scale sc, float* __restrict__ loss,
                                                              float4* __restrict__ stats) {
  __shared__ Shared sh;
  __shared__ Entries en;
  __shared__ uint32_t filter[kTail ? kFilter / 32 : 1];
  const int64_t r = blockIdx.x / ranks;
  const int rank = blockIdx.x % ranks;
  const Slice<T> sl(x.row(r), V, rank, ranks);
  T* o = kGrad ? out.row(r) : nullptr;
  const float w = ta.weight ? ta.weight[r] : 1.f;
  const bool writer = threadIdx.x == 0 && rank == 0;
  if (w == 0.f) {
    if (writer) loss[r] = 0.f;
    if (writer && !kGrad) stats[r] = make_float4(0.f, -1.f, 0.f, 0.f);
    if (kGrad) zero_slice<T>(sl, o);
    return;
  }
  Entry e = load_entry<T>(ta, r, sl.row, V, sc.inv_temp, en);
  MaxSum a;
  if constexpr (kTail) {
    for (int i = threadIdx.x; i < kFilter / 32; i += kThreads) filter[i] = 0;
    __syncthreads();
    if (e.id >= sl.head && e.id < sl.body_end) {
      const uint32_t b = (uint32_t)((e.id - sl.head) / Vec16<T>::kN) & (kFilter - 1);
      atomicOr(&filter[b >> 5], 1u << (b & 31));
    }
    __syncthreads();
    a = row_sum<T, kCap>(sl, sc, DropEntries<T>{filter, &en, ta.k, sl.head}, sh, ranks);
  } else {
    a = row_sum<T, kCap>(sl, sc, KeepAll(), sh, ranks);
  }
  const TeacherRow te = finish_entries(e, ta, r, V, kTail, en, sh.scratch);
  const float y = softcap(e.x, sc.cap) * sc.inv_temp;
  const MaxSum rest = a;
  if constexpr (kTail) {
    MaxSum own;
    own.m = block_max(e.first ? y : -INFINITY, sh.scratch);
    own.s = block_sum(e.first && y != -INFINITY ? expf(y - own.m) : 0.f, sh.scratch);
    a.merge(own);
  }
  const float log_s = logf(a.s);
  float kl = 0.f;
  // maxima first: what is left to round is of the size of the difference
  if (e.q != 0.f) kl = e.q * (((e.t - te.m) - (y - a.m)) + (log_s - te.log_s));
  kl = block_sum(kl, sh.scratch);
  float m1 = a.m, c1 = 1.f / a.s;
  if constexpr (kTail) {
    const bool some = rest.m != -INFINITY;
    const float share = some ? expf(rest.m - a.m) : 0.f, p_rest = share * (rest.s / a.s);
    // (a rest that fp32 cannot hold: by its logarithm)
    const float log_rest = p_rest > 1e-30f ? logf(p_rest) : some ? rest.m - a.m + (logf(rest.s) - log_s) : -INFINITY;
    if (te.q_rest > 0.f) kl += te.q_rest * (logf(te.q_rest) - log_rest);
    m1 = some ? rest.m : 0.f;
    c1 = some ? te.mass * (share / a.s) - te.q_rest / rest.s : 0.f * log_s;
  }
  const bool nothing = !kTail && !te.any;  // no entry: nothing to match
  if (writer) {
    loss[r] = nothing ? 0.f : w * ta.temp * ta.temp * kl;
    if (!kGrad) stats[r] = make_float4(a.m, nothing ? -1.f : a.s, m1, c1);
  }
  if constexpr (kGrad) {
    if (nothing) {
      zero_slice<T>(sl, o);
    } else {
      const float c = w * ta.temp;
      write_slice<T, kCap>(sl, o, sc, m1, c * c1, sh.ring);
      __syncthreads();
      write_entry<T>(sl, o, e, sc, c, a.m, 1.f / a.s, te.mass);
    }
  }
  row_done(ranks);
}

template <typename T, bool kCap>
__global__ void __launch_bounds__(kThreads, 4) distill_bwd_kernel(Rows<const T> x, Rows<T> out, int64_t N, int64_t V,
                                                                  int ranks, TeacherArgs ta, Scale sc,
                                                                  const float4* __restrict__ stats,
                                                                  const float* __restrict__ g) {
  __shared__ Shared sh;
  __shared__ Entries en;
  const int64_t r = N - 1 - blockIdx.x / ranks;  // last to first, as above
  const Slice<T> sl(x.row(r), V, blockIdx.x % ranks, ranks);
  T* o = out.row(r);
  const float4 st = stats[r];
  if (st.y == -1.f) {
    zero_slice<T>(sl, o);
    return;
  }
  Entry e = load_entry<T>(ta, r, sl.row, V, sc.inv_temp, en);
  const TeacherRow te = finish_entries(e, ta, r, V, ta.lse != nullptr, en, sh.scratch);
  const float c = (ta.weight ? ta.weight[r] : 1.f) * ta.temp * g[r];
  write_slice<T, kCap>(sl, o, sc, st.z, c * st.w, sh.ring);
  __syncthreads();
  write_entry<T>(sl, o, e, sc, c, st.x, 1.f / st.y, te.mass);
}

// ------------------------------------------------------------------------------------ launches
// Blocks a row: enough for two on each SM, while a block keeps two vectors a thread.
int ranks_for(int64_t N, int64_t V, int at_least = 1) {
  static const int fix = getenv("RNK") ? atoi(getenv("RNK")) : 0;
  if (fix) return fix;
  int c = at_least;
  while (c < 8 && N * c < 2 * objective_sms() && V / (2 * c) >= 4096) c *= 2;
  return c;
}

// Blocks a row where the row is read twice: the rows in flight (four blocks an SM) have to stay in L2
// between the two passes; 40 of its 126 MB are given to them.
int ranks_for_two_passes(const Logits& x) {
  static const int l2_rows = getenv("L2R") ? atoi(getenv("L2R")) : 40;
  const int64_t row = x.V * (x.type == LogitType::kF32 ? 4 : 2);
  int c = 1;
  while (c < 8 && 4 * objective_sms() / c * row > ((int64_t)l2_rows << 20)) c *= 2;
  return ranks_for(x.N, x.V, c);
}

}  // namespace

namespace me {

#define ME_CAP_DISPATCH(CAP, ...)        \
  if ((CAP) > 0.f) {                     \
    constexpr bool kCap = true;          \
    __VA_ARGS__;                         \
  } else {                               \
    constexpr bool kCap = false;         \
    __VA_ARGS__;                         \
  }

void launch_logprob_fwd(const Logits& x, const int64_t* target, float* logp, float2* stats, cudaStream_t stream) {
  const int ranks = ranks_for(x.N, x.V);
  ME_LOGITS_DISPATCH(x.type, ME_CAP_DISPATCH(x.cap, launch_cluster(logprob_fwd_kernel<T, kCap>, x.N * ranks, kThreads,
                                                                   ranks, stream, rows_in<T>(x), x.V, ranks, target,
                                                                   make_scale(x.cap, 1.f), logp, stats)));
}

void launch_logprob_bwd(const Logits& x, const int64_t* target, const float2* stats, const float* g, Gradient out,
                        cudaStream_t stream) {
  const int ranks = ranks_for(x.N, x.V);
  ME_LOGITS_DISPATCH(
      x.type, ME_CAP_DISPATCH(x.cap, logprob_bwd_kernel<T, kCap><<<(unsigned)(x.N * ranks), kThreads, 0, stream>>>(
                                         rows_in<T>(x), rows_out<T>(out), x.N, x.V, ranks, target, make_scale(x.cap, 1.f),
                                         stats, g)));
}

void launch_distill_fwd(const Logits& x, const TeacherArgs& te, float* loss, float4* stats, cudaStream_t stream) {
  const int ranks = ranks_for(x.N, x.V);
  ME_LOGITS_DISPATCH(x.type, ME_CAP_DISPATCH(x.cap, {
    auto* kernel = te.lse ? distill_kernel<T, kCap, true, false> : distill_kernel<T, kCap, false, false>;
    launch_cluster(kernel, x.N * ranks, kThreads, ranks, stream, rows_in<T>(x), Rows<T>{}, x.V, ranks, te,
                   make_scale(x.cap, te.temp), loss, stats);
  }));
}

void launch_distill_grad(const Logits& x, const TeacherArgs& te, float* loss, Gradient out, cudaStream_t stream) {
  const int ranks = ranks_for_two_passes(x);
  ME_LOGITS_DISPATCH(x.type, ME_CAP_DISPATCH(x.cap, {
    auto* kernel = te.lse ? distill_kernel<T, kCap, true, true> : distill_kernel<T, kCap, false, true>;
    launch_cluster(kernel, x.N * ranks, kThreads, ranks, stream, rows_in<T>(x), rows_out<T>(out), x.V, ranks, te,
                   make_scale(x.cap, te.temp), loss, (float4*)nullptr);
  }));
}

void launch_distill_bwd(const Logits& x, const TeacherArgs& te, const float4* stats, const float* g, Gradient out,
                        cudaStream_t stream) {
  const int ranks = ranks_for(x.N, x.V);
  ME_LOGITS_DISPATCH(
      x.type, ME_CAP_DISPATCH(x.cap, distill_bwd_kernel<T, kCap><<<(unsigned)(x.N * ranks), kThreads, 0, stream>>>(
                                         rows_in<T>(x), rows_out<T>(out), x.N, x.V, ranks, te, make_scale(x.cap, te.temp),
                                         stats, g)));
}

}  // namespace me

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

// ------------------------------------------------------------------------------------ gradient of a slice
// out_j = coef exp(y_j - m) z'_j for the block's columns, in 16-byte stores where the two rows are
// aligned alike. The slice is walked from its end: what a sum has just read last is in L2.
template <typename T, bool kCap, bool kAligned>
ME_DEVICE void write_vectors(const Slice<T>& sl, T* out, const Scale& sc, float m, float coef, Ring& ring) {
  constexpr int kN = Vec16<T>::kN, kP = kN / 2;
  // coef (1 - (z / c)^2) is one FMA with the coefficient inside
  const float coef_slope = coef * sc.slope, k = sc.inv_temp * kLog2e, shift = m * kLog2e;
  const int last = max(sl.count() - 1, 0);
  T* mine = out + sl.column(sl.vec(last));
  stream<-kThreads>(
      sl.mine() + last * kThreads, sl.count(), ring, [](int, auto&) {},
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
            // (a 16-bit result is rounded at 2^-9 or 2^-12, a 32-bit z under a softcap at up to 1e-6: the exponent's
            // rounding, 2e-6, may stay)
            float2 a;
            if constexpr (sizeof(T) == 4) a = unpack2(fma2(zp, both2(sc.inv_temp), both2(-m)));
            else a = unpack2(fma2(zp, both2(k), both2(-shift)));
            f32x2 e;
            if constexpr (sizeof(T) == 4 && !kCap) {
              const float2 r = unpack2(exp_pair(pack2(a.x, a.y)));  // down to e^-87; 0 below, for masked columns too
              e = pack2(a.x < -87.f ? 0.f : r.x, a.y < -87.f ? 0.f : r.y);
            } else if constexpr (sizeof(T) == 4) {
              a = unpack2(mul2(pack2(a.x, a.y), both2(kLog2e)));
              e = pack2(exp2_fast(a.x), exp2_fast(a.y));
            } else {
              e = pack2(exp2_fast(a.x), exp2_fast(a.y));
            }
            z[u][p] = mul2(e, kCap ? fma2(mul2(zp, both2(coef_slope)), zp, both2(coef)) : both2(coef));
          }
          Vec16<T> r;
          r.u = from_pairs<T>(z[u]);
          T* at = mine - (i + u) * (kThreads * kN);
          if constexpr (kAligned) {
            *reinterpret_cast<uint4*>(at) = r.u;
          } else {
#pragma unroll
            for (int e = 0; e < kN; ++e) at[e] = r.h[e];
          }
        }
      });
}
template <typename T, bool kCap>
ME_DEVICE void write_slice(const Slice<T>& sl, T* out, const Scale& sc, float m, float coef, Ring& ring) {
  if (m == -INFINITY) coef = NAN;  // nothing but masked columns (every other NaN of a row is in coef already)
  if ((reinterpret_cast<uintptr_t>(out + sl.head) & 15) == 0) write_vectors<T, kCap, true>(sl, out, sc, m, coef, ring);
  else write_vectors<T, kCap, false>(sl, out, sc, m, coef, ring);
  const int j = sl.single();
  if (j >= 0) {
    const float z = softcap(to_f<T>(sl.row[j]), sc.cap), y = z * sc.inv_temp - m;
    const float e = sizeof(T) == 4 ? expf(y) : exp2_fast(y * kLog2e);
    out[j] = from_f<T>(coef * e * softcap_slope(z, sc.cap));
  }
}

template <typename T>
ME_DEVICE void zero_slice(const Slice<T>& sl, T* out) {
  const int64_t head = ((16 - (reinterpret_cast<uintptr_t>(out) & 15)) & 15) / sizeof(T);
  if (head == sl.head || sl.begin >= sl.end) {
    for (int i = sl.begin + threadIdx.x; i < sl.end; i += kThreads)
      reinterpret_cast<uint4*>(out + sl.head)[i] = make_uint4(0, 0, 0, 0);
  } else {
    for (int j = sl.column(sl.begin) + threadIdx.x; j < sl.column(sl.end); j += kThreads)
      out[j] = from_f<T>(0.f);
  }
  const int j = sl.single();
  if (j >= 0) out[j] = from_f<T>(0.f);
}

// ------------------------------------------------------------------------------------ log-probabilities
// One cluster a row, one walk. Bound by issue slots under a softcap (97 for 8 logits a thread): 2048 x 262144 bf16,
// softcap 30, 204 us, 0.80 of the copy rate with every row counted; fp32 without one runs at the copy rate.
template <typename T, bool kCap>
__global__ void __launch_bounds__(kThreads, 4) logprob_fwd_kernel(Rows<const T> x, int V, int lg_ranks,
                                                                  const int64_t* __restrict__ target, Scale sc,
                                                                  float* __restrict__ logp,
                                                                  float2* __restrict__ stats) {
  __shared__ Ring ring;
  __shared__ float2 part[kWarps];
  const int64_t r = (blockIdx.x >> lg_ranks);
  const int rank = blockIdx.x & ((1 << lg_ranks) - 1);
  const int64_t t = target[r];
  if (t == kIgnoreToken) {
    if (threadIdx.x == 0 && rank == 0) {
      logp[r] = 0.f;
      stats[r] = make_float2(0.f, 1.f);
    }
    return;
  }
  const Slice<T> sl(x.row(r), V, rank, lg_ranks);
  const float xt = t >= 0 && t < V ? to_f<T>(sl.row[t]) : NAN;
  const MaxSum a = row_merge(
      slice_sum<T, kCap>(sl, sc, KeepAll(), ring), part, lg_ranks);
  if (threadIdx.x == 0 && rank == 0) {
    logp[r] = softcap(xt, sc.cap) - a.m - logf(a.s);
    stats[r] = make_float2(a.m, a.s);
  }
  row_done(lg_ranks);
}

// Rows are taken last to first: where the forward pass just went over them, the last ones are in L2. Bound by memory, one
// read and one write of a logit: 0.75 of the DRAM's peak for 1184 x 262144 bf16 with half of the rows trained.
template <typename T, bool kCap>
__global__ void __launch_bounds__(kThreads, 4) logprob_bwd_kernel(Rows<const T> x, Rows<T> out, int64_t N, int V,
                                                                  int lg_ranks, const int64_t* __restrict__ target,
                                                                  Scale sc, const float2* __restrict__ stats,
                                                                  const float* __restrict__ g, int64_t g_step) {
  __shared__ Ring ring;
  const int64_t r = N - 1 - (blockIdx.x >> lg_ranks);
  const int rank = blockIdx.x & ((1 << lg_ranks) - 1);
  const int64_t t = target[r];
  const Slice<T> sl(x.row(r), V, rank, lg_ranks);
  T* o = out.row(r);
  if (t == kIgnoreToken) {
    zero_slice<T>(sl, o);
    return;
  }
  const bool valid = t >= 0 && t < V, mine = valid && sl.holds((int)t) && threadIdx.x == 0;
  const float2 ms = stats[r];
  const float c = valid ? g[r * g_step] : NAN;
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
// A teacher's entry, and what the student's side of its column needs.
struct Entry {
  int id;       // -1: unused, or an earlier entry has the same id
  float q;      // the probability of all entries with this id
  float y;      // the student's y
  float slope;  // z'
};
static_assert(sizeof(Entry) == sizeof(float4));

// What a row's loss needs of the teacher.
struct TeacherRow {
  float b;       // sum q [log q - (y - y_ref)]: with it the divergence is b + sum q [log s + (m - y_ref)]
  float sum_q;
  float q_rest;  // with a rest: its probability
  float mass;    // sum of q and q_rest
  float y_ref;   // the entries' largest y
  float s;       // sum exp(y - y_ref) over the entries (each id once)
  float any;     // 1: an entry has q != 0
  float pad;
};
static_assert(sizeof(TeacherRow) == kTeacherRowBytes && sizeof(Entry) == kEntryBytes);

// One warp a row of the teacher's records: probabilities, repeated ids, the student's logits there. It
// runs ahead of the kernels that walk the logits, which then wait for nothing but the logits (with this
// in their blocks, eight to a row, the chain ids -> logits -> sums took half of a block's time).
template <typename T>
__global__ void __launch_bounds__(kThreads) teacher_kernel(Rows<const T> x, int64_t N, int V, TeacherArgs a, Scale sc,
                                                           Entry* __restrict__ entries, TeacherRow* __restrict__ rows) {
  constexpr int kSeen = 8192;  // bits
  __shared__ int ids[kWarps][kMaxTop], firsts[kWarps][kMaxTop];
  __shared__ float qs[kWarps][kMaxTop], sums[kWarps][kMaxTop];
  __shared__ uint32_t seen_bits[kWarps][kSeen / 32];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int64_t r = (int64_t)blockIdx.x * kWarps + wid;
  if (r >= N || (a.weight && a.weight[r] == 0.f)) return;
  const bool tail = a.lse != nullptr;
  const T* row = x.row(r);
  int* id = ids[wid];
  float* qr = qs[wid];
  float t[kMaxTop / 32], y[kMaxTop / 32], slope[kMaxTop / 32];
  float m = -INFINITY, y_ref = -INFINITY;
#pragma unroll
  for (int i = 0; i < kMaxTop / 32; ++i) {
    const int k = lane + 32 * i;
    t[i] = -INFINITY;
    y[i] = slope[i] = 0.f;
    if (k >= a.k) continue;
    const int64_t j = a.ids[r * a.k + k];
    const bool there = j >= 0 && j < V;  // other ids are unused entries
    id[k] = there ? (int)j : -1;
    if (!there) continue;
    t[i] = a.top[r * a.k + k] * sc.inv_temp;
    const float z = softcap(to_f<T>(row[j]), sc.cap);
    y[i] = z * sc.inv_temp;
    slope[i] = softcap_slope(z, sc.cap);
    m = fmaxf(m, t[i]);
    y_ref = fmaxf(y_ref, y[i]);
  }
  m = tail ? a.lse[r] : warp_max(m);
  y_ref = warp_max(y_ref);
  if (y_ref == -INFINITY) y_ref = 0.f;
  float q[kMaxTop / 32];
  float sum = 0.f;
  bool any = false;
#pragma unroll
  for (int i = 0; i < kMaxTop / 32; ++i) {
    q[i] = t[i] == -INFINITY ? 0.f : expf(t[i] - m);
    sum += q[i];
    any = any || q[i] != 0.f;
  }
  sum = warp_sum(sum);
  any = __any_sync(0xffffffffu, any);
  const float inv = tail || !any ? 1.f : 1.f / sum, log_s = tail ? 0.f : logf(sum);
#pragma unroll
  for (int i = 0; i < kMaxTop / 32; ++i) {
    const int k = lane + 32 * i;
    q[i] *= inv;
    if (k < a.k) qr[k] = q[i];
  }
  if (!tail && any) sum = 1.f;
  // Repeated ids: a bit that is set already (by one of 8192 ids, so seldom by another id) asks for a look at the
  // list; the first entry with an id stands for all of them.
  uint32_t* seen = seen_bits[wid];
  int* first = firsts[wid];
  float* q_id = sums[wid];
  for (int i = lane; i < kSeen / 32; i += 32) seen[i] = 0;
#pragma unroll
  for (int i = 0; i < kMaxTop / 32; ++i) {
    const int k = lane + 32 * i;
    if (k < a.k) {
      first[k] = id[k];
      q_id[k] = q[i];
    }
  }
  __syncwarp();
  for (int k0 = 0; k0 < a.k; k0 += 32) {
    const int k = k0 + lane;
    bool again = false;
    if (k < a.k && id[k] >= 0) {
      const int bit = id[k] & (kSeen - 1);
      again = atomicOr(&seen[bit >> 5], 1u << (bit & 31)) >> (bit & 31) & 1;
    }
    for (uint32_t look = __ballot_sync(0xffffffffu, again); look; look &= look - 1) {
      const int same = id[k0 + __ffs(look) - 1];
      int one = a.k;
      float total = 0.f;
      for (int o = lane; o < a.k; o += 32) {
        if (id[o] != same) continue;
        one = min(one, o);
        total += qr[o];
      }
      one = __reduce_min_sync(0xffffffffu, one);
      total = warp_sum(total);
      for (int o = lane; o < a.k; o += 32)
        if (id[o] == same && o != one) first[o] = -1;
      if (lane == 0) q_id[one] = total;
      __syncwarp();
    }
  }
  __syncwarp();
  // what the loss needs, by ids: q log q of an id's whole probability
  float b = 0.f, s = 0.f, used = 0.f;
#pragma unroll
  for (int i = 0; i < kMaxTop / 32; ++i) {
    const int k = lane + 32 * i;
    if (k >= a.k) continue;
    const float q_all = q_id[k];
    Entry e = {first[k], q_all, y[i], slope[i]};
    reinterpret_cast<float4*>(entries)[r * a.k + k] = *reinterpret_cast<float4*>(&e);
    if (first[k] < 0) continue;
    s += y[i] == -INFINITY ? 0.f : expf(y[i] - y_ref);
    used += 1.f;
    if (q_all == 0.f) continue;
    // maxima first: what is left to round is of the size of the difference
    const float log_q = q_all == q[i] ? (t[i] - m) - log_s : logf(q_all);
    b += y[i] == -INFINITY ? INFINITY : q_all * (log_q - (y[i] - y_ref));
  }
  b = warp_sum(b);
  s = warp_sum(s);
  used = warp_sum(used);
  if (lane == 0) {
    // no rest where the entries are the whole vocabulary: 1 - sum is rounding then
    const float q_rest = tail && used < (float)V ? fmaxf(0.f, 1.f - sum) : 0.f;
    rows[r] = {b, sum, q_rest, tail ? sum + q_rest : 1.f, y_ref, s, any ? 1.f : 0.f, 0.f};
  }
}

// Leaves the teacher's entries out of a sum: a byte for each of the block's vectors says which of its elements are
// entries. (A filter with one bit for several vectors and a look at the list made the sum take 2.3 times as long.)
// A slice of more vectors than there are bytes shares them, and looks at the list behind a byte that is set.
constexpr int kMostMasks = 32768;
template <typename T>
struct DropEntries {
  const uint8_t* mask;
  const int* id;
  int k, head, begin;
  bool exact;
  ME_DEVICE uint32_t operator()(int vec) const {
    constexpr int kN = Vec16<T>::kN;
    uint32_t m = mask[vec - begin & kMostMasks - 1];
    if (m == 0 || exact) return m;
    m = 0;
    const int j0 = head + vec * kN;
    for (int i = 0; i < k; ++i) {
      const uint32_t d = (uint32_t)(id[i] - j0);
      if (id[i] >= 0 && d < (uint32_t)kN) m |= 1u << d;
    }
    return m;
  }
  ME_DEVICE bool column(int j) const {
    for (int i = 0; i < k; ++i)
      if (id[i] == j) return true;
    return false;
  }
};
// Its bytes, for a slice of n vectors.
ME_HOST_DEVICE int mask_bytes(int n) { return ((n < kMostMasks ? n : kMostMasks) + 15) / 16 * 16; }

// The student's side of a row, from the sum over its columns (with a rest: over those that are no entry).
struct Student {
  MaxSum all;
  float log_s;
  float m1, c1;      // p_j rho_j = c1 exp(y_j - m1) for the columns that are no entry
  float log_p_rest;
};
template <bool kTail>
ME_DEVICE Student finish_student(MaxSum a, const TeacherRow& te) {
  Student st;
  const MaxSum rest = a;
  if (kTail) {
    MaxSum own;
    own.m = te.s == 0.f ? -INFINITY : te.y_ref;
    own.s = te.s;
    a.merge(own);
  }
  st.all = a;
  st.log_s = logf(a.s);
  st.m1 = a.m;
  st.c1 = 1.f / a.s;
  st.log_p_rest = 0.f;
  if (kTail) {
    const bool some = rest.m != -INFINITY;
    const float share = some ? expf(rest.m - a.m) : 0.f, p_rest = share * (rest.s / a.s);
    // (a rest that fp32 cannot hold: by its logarithm)
    st.log_p_rest = p_rest > 1e-30f ? logf(p_rest) : some ? rest.m - a.m + (logf(rest.s) - st.log_s) : -INFINITY;
    st.m1 = some ? rest.m : 0.f;
    st.c1 = some ? te.mass * (share / a.s) - te.q_rest / rest.s : 0.f * st.log_s;
  }
  return st;
}

// The row's divergence.
ME_DEVICE float divergence(const TeacherRow& te, const Student& st) {
  float kl = te.b + te.sum_q * (st.log_s + (st.all.m - te.y_ref));
  if (te.q_rest > 0.f) kl += te.q_rest * (logf(te.q_rest) - st.log_p_rest);
  return kl;
}

// A thread's entry of the row (k is at most a block's threads).
static_assert(kThreads >= kMaxTop);
ME_DEVICE Entry load_entry(const Entry* entries, int64_t r, int k) {
  Entry e = {-1, 0.f, 0.f, 0.f};
  if (threadIdx.x < k) *reinterpret_cast<float4*>(&e) = reinterpret_cast<const float4*>(entries)[r * k + threadIdx.x];
  return e;
}
// The entries' own columns, after the slice was written without them.
template <typename T>
ME_DEVICE void write_entry(const Slice<T>& sl, T* out, const Entry& e, float c, float m, float inv_s, float mass) {
  if (e.id >= 0 && sl.holds(e.id)) out[e.id] = from_f<T>(c * (expf(e.y - m) * inv_s * mass - e.q) * e.slope);
}

// One cluster a row. Value, and the statistics that the backward pass starts from: m, s (-1: a row without
// gradient), m', c'; or with kGrad value and gradient: the slice is read again once the cluster has the
// row's sum, from L2 where the rows in flight fit there (1024 x 262144 bf16: 262 us with a softcap, where they do not,
// for 164 us of one read and one write; 219 us without one).
template <typename T, bool kCap, bool kTail, bool kGrad>
__global__ void __launch_bounds__(kThreads, 4)
    distill_kernel(Rows<const T> x, Rows<T> out, int V, int lg_ranks, int k, const float* __restrict__ weight,
                   float temp, const Entry* __restrict__ entries, const TeacherRow* __restrict__ rows, Scale sc,
                   float* __restrict__ loss, float4* __restrict__ stats) {
  __shared__ Ring ring;
  __shared__ float2 part[kWarps];
  __shared__ int ids[kTail ? kMaxTop : 1];
  extern __shared__ uint4 masks[];  // with a rest
  const int64_t r = blockIdx.x >> lg_ranks;
  const int rank = blockIdx.x & ((1 << lg_ranks) - 1);
  const Slice<T> sl(x.row(r), V, rank, lg_ranks);
  T* o = kGrad ? out.row(r) : nullptr;
  const float w = weight ? weight[r] : 1.f;
  const bool writer = threadIdx.x == 0 && rank == 0;
  if (w == 0.f) {
    if (writer) loss[r] = 0.f;
    if (writer && !kGrad) stats[r] = make_float4(0.f, -1.f, 0.f, 0.f);
    if (kGrad) zero_slice<T>(sl, o);
    return;
  }
  MaxSum a;
  if constexpr (kTail) {
    const Entry e = load_entry(entries, r, k);
    const int vecs = sl.end - sl.begin;
    for (int i = threadIdx.x; i < mask_bytes(vecs) / 16; i += kThreads) masks[i] = make_uint4(0, 0, 0, 0);
    if (threadIdx.x < k) ids[threadIdx.x] = e.id;
    __syncthreads();
    if (e.id >= sl.head && e.id < sl.body_end) {
      constexpr int kN = Vec16<T>::kN;
      const int v = (e.id - sl.head) / kN - sl.begin, at = v & kMostMasks - 1;
      if (v >= 0 && v < vecs)
        atomicOr(reinterpret_cast<uint32_t*>(masks) + at / 4, 1u << (at % 4 * 8 + (e.id - sl.head) % kN));
    }
    __syncthreads();
    const DropEntries<T> drop = {reinterpret_cast<const uint8_t*>(masks), ids, k, sl.head, sl.begin, vecs <= kMostMasks};
    a = slice_sum<T, kCap>(sl, sc, drop, ring);
  } else {
    a = slice_sum<T, kCap>(sl, sc, KeepAll(), ring);
  }
  const TeacherRow te = rows[r];
  const Student st = finish_student<kTail>(row_merge(a, part, lg_ranks), te);
  const bool nothing = !kTail && te.any == 0.f;  // no entry: nothing to match
  if (writer) {
    loss[r] = nothing ? 0.f : w * temp * temp * divergence(te, st);
    if (!kGrad) stats[r] = make_float4(st.all.m, nothing ? -1.f : st.all.s, st.m1, st.c1);
  }
  if constexpr (kGrad) {
    if (nothing) {
      zero_slice<T>(sl, o);
    } else {
      const float c = w * temp;
      write_slice<T, kCap>(sl, o, sc, st.m1, c * st.c1, ring);
      __syncthreads();
      write_entry<T>(sl, o, load_entry(entries, r, k), c, st.all.m, 1.f / st.all.s, te.mass);
    }
  }
  row_done(lg_ranks);
}

template <typename T, bool kCap>
__global__ void __launch_bounds__(kThreads, 4)
    distill_bwd_kernel(Rows<const T> x, Rows<T> out, int64_t N, int V, int lg_ranks, int k,
                       const float* __restrict__ weight, float temp, const Entry* __restrict__ entries,
                       const TeacherRow* __restrict__ rows, Scale sc, const float4* __restrict__ stats,
                       const float* __restrict__ g, int64_t g_step) {
  __shared__ Ring ring;
  const int64_t r = N - 1 - (blockIdx.x >> lg_ranks);  // last to first, as above
  const Slice<T> sl(x.row(r), V, blockIdx.x & ((1 << lg_ranks) - 1), lg_ranks);
  T* o = out.row(r);
  const float4 st = stats[r];
  if (st.y == -1.f) {
    zero_slice<T>(sl, o);
    return;
  }
  const Entry e = load_entry(entries, r, k);
  const float c = (weight ? weight[r] : 1.f) * temp * g[r * g_step];
  write_slice<T, kCap>(sl, o, sc, st.z, c * st.w, ring);
  __syncthreads();
  write_entry<T>(sl, o, e, c, st.x, 1.f / st.y, rows[r].mass);
}

// ------------------------------------------------------------------------------------ launches
// Dynamic shared memory of distill_kernel: DropEntries' bytes.
int masks_for(const Logits& x, const TeacherArgs& te, int ranks) {
  if (!te.lse) return 0;
  const int64_t vecs = x.V * (x.type == LogitType::kF32 ? 4 : 2) / 16;
  return mask_bytes((int)((vecs + ranks - 1) / ranks));
}

}  // namespace

namespace me {

void launch_logprob_fwd(const Logits& x, const int64_t* target, float* logp, float2* stats, cudaStream_t stream) {
  const int ranks = ranks_for(x.N, x.V);
  ME_LOGITS_DISPATCH(x.type, ME_CAP_DISPATCH(x.cap, launch_cluster(logprob_fwd_kernel<T, kCap>, x.N * ranks, ranks, 0,
                                                                   stream, rows_in<T>(x), x.V, ilog2(ranks), target,
                                                                   make_scale(x.cap, 1.f), logp, stats)));
}

void launch_logprob_bwd(const Logits& x, const int64_t* target, const float2* stats, RowValues g, Gradient out,
                        cudaStream_t stream) {
  const int ranks = ranks_for_gradient(x);
  ME_LOGITS_DISPATCH(
      x.type, ME_CAP_DISPATCH(x.cap, logprob_bwd_kernel<T, kCap><<<(unsigned)(x.N * ranks), kThreads, 0, stream>>>(
                                         rows_in<T>(x), rows_out<T>(out), x.N, (int)x.V, ilog2(ranks), target,
                                         make_scale(x.cap, 1.f), stats, g.data, g.step)));
}

void launch_teacher(const Logits& x, const TeacherArgs& te, void* entries, void* rows, cudaStream_t stream) {
  ME_LOGITS_DISPATCH(x.type, teacher_kernel<T><<<(unsigned)((x.N + kWarps - 1) / kWarps), kThreads, 0, stream>>>(
                                 rows_in<T>(x), x.N, (int)x.V, te, make_scale(x.cap, te.temp),
                                 static_cast<Entry*>(entries), static_cast<TeacherRow*>(rows)));
}

void launch_distill_fwd(const Logits& x, const TeacherArgs& te, const void* entries, const void* rows, float* loss,
                        float4* stats, cudaStream_t stream) {
  const int ranks = ranks_for(x.N, x.V);
  ME_LOGITS_DISPATCH(x.type, ME_CAP_DISPATCH(x.cap, {
    auto* kernel = te.lse ? distill_kernel<T, kCap, true, false> : distill_kernel<T, kCap, false, false>;
    const int smem = masks_for(x, te, ranks);
    allow_smem(kernel, smem);
    launch_cluster(kernel, x.N * ranks, ranks, smem, stream, rows_in<T>(x), Rows<T>{}, x.V, ilog2(ranks), te.k, te.weight,
                   te.temp, static_cast<const Entry*>(entries), static_cast<const TeacherRow*>(rows),
                   make_scale(x.cap, te.temp), loss, stats);
  }));
}

void launch_distill_grad(const Logits& x, const TeacherArgs& te, const void* entries, const void* rows, float* loss,
                         Gradient out, cudaStream_t stream) {
  const int ranks = ranks_for_both(x);
  ME_LOGITS_DISPATCH(x.type, ME_CAP_DISPATCH(x.cap, {
    auto* kernel = te.lse ? distill_kernel<T, kCap, true, true> : distill_kernel<T, kCap, false, true>;
    const int smem = masks_for(x, te, ranks);
    allow_smem(kernel, smem);
    launch_cluster(kernel, x.N * ranks, ranks, smem, stream, rows_in<T>(x), rows_out<T>(out), x.V, ilog2(ranks), te.k,
                   te.weight, te.temp, static_cast<const Entry*>(entries), static_cast<const TeacherRow*>(rows),
                   make_scale(x.cap, te.temp), loss, (float4*)nullptr);
  }));
}

void launch_distill_bwd(const Logits& x, const TeacherArgs& te, const void* entries, const void* rows,
                        const float4* stats, RowValues g, Gradient out, cudaStream_t stream) {
  const int ranks = ranks_for_gradient(x);
  ME_LOGITS_DISPATCH(
      x.type, ME_CAP_DISPATCH(x.cap, distill_bwd_kernel<T, kCap><<<(unsigned)(x.N * ranks), kThreads, 0, stream>>>(
                                         rows_in<T>(x), rows_out<T>(out), x.N, (int)x.V, ilog2(ranks), te.k, te.weight,
                                         te.temp, static_cast<const Entry*>(entries),
                                         static_cast<const TeacherRow*>(rows), make_scale(x.cap, te.temp), stats, g.data, g.step)));
}

}  // namespace me

// The k largest logits of each row with their ids, and the row's log-sum-exp (sm_100a): what a
// teacher records for a student that is trained on its top logits.
//
// Rows are ordered by the raw logit x (the softcap z = c tanh(x / c) is monotone), equal logits by
// the lower id, NaN above +inf. lse = log sum_j exp(z_j / tau).
//
// One pass over the row gives the sum of exponentials and the largest logit of each of some
// thousand groups of columns. The k-th largest group maximum is a lower bound of the k-th largest logit
// (k groups hold one each that is as large), so only the groups that reach it are read again, about k of
// them, and their logits above the bound, a little more than k, are ranked by counting. Where that
// does not end in few candidates (many equal logits, few columns, a NaN), the row's first block finds the
// exact k-th logit by radix selection, some passes over the row.
#include "objectives.cuh"

#include <algorithm>

using namespace me;

namespace {

constexpr int kMaxGroups = 16;  // of a thread and of the threads with its number in the row's other blocks
constexpr int kHits = 512;      // groups that are read again
constexpr int kFound = 1024;    // candidates

// A number that orders as the logits do: larger logit, larger key. -0 and +0 share one, NaN is on top.
ME_DEVICE uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
ME_DEVICE float key_value(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);  // (NaN for NaN's)
}

// key, then the lower column
ME_DEVICE uint64_t candidate(uint32_t key, int col) { return (uint64_t)key << 32 | (uint32_t)~col; }

struct Work {
  union {
    Ring ring;
    struct {
      uint64_t found[kFound];
      int hits[kHits];
    } pick;
    struct {
      int hist[256];
      uint64_t found[kMaxTop];
      int warp_sum[kWarps];
      uint32_t prefix;
      int need, count;
    } exact;
  };
};

// Ranks n candidates, all different, and writes the k largest.
ME_DEVICE void write_ranked(const uint64_t* found, int n, int k, float cap, float* values, int64_t* ids) {
  for (int c = threadIdx.x; c < n; c += kThreads) {
    const uint64_t mine = found[c];
    int rank = 0;
    for (int o = 0; o < n; ++o) rank += found[o] > mine;
    if (rank < k) {
      values[rank] = softcap(key_value((uint32_t)(mine >> 32)), cap);
      ids[rank] = (int)~(uint32_t)mine;
    }
  }
}

// One block, any row: the k-th largest key, eight bits a pass, then all larger ones and the lowest columns
// among its equals.
template <typename T>
ME_DEVICE void exact_top(const T* row, int V, int k, float cap, Work& work, float* values, int64_t* ids) {
  auto& w = work.exact;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  __syncthreads();
  if (threadIdx.x == 0) {
    w.prefix = 0;
    w.need = k;
    w.count = 0;
  }
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += kThreads) w.hist[i] = 0;
    __syncthreads();
    const uint32_t want = w.prefix, mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
    for (int j0 = 0; j0 < V; j0 += kThreads) {
      const int j = j0 + threadIdx.x;
      const uint32_t q = j < V ? order_key(to_f<T>(row[j])) : 0u;
      const bool in = j < V && (q & mask) == want;
      const uint32_t bin = q >> shift & 255;
      // (equal logits meet in one bin: one atomic for the lanes that share theirs)
      const uint32_t same = __match_any_sync(0xffffffffu, in ? bin : 256u);
      if (in && lane == __ffs(same) - 1) atomicAdd(&w.hist[bin], __popc(same));
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int left = w.need, b = 255;
      while (b > 0 && w.hist[b] < left) left -= w.hist[b--];
      w.need = left;
      w.prefix |= (uint32_t)b << shift;
    }
    __syncthreads();
  }
  const uint32_t kth = w.prefix;
  for (int j = threadIdx.x; j < V; j += kThreads) {
    const uint32_t q = order_key(to_f<T>(row[j]));
    if (q > kth) w.found[atomicAdd(&w.count, 1)] = candidate(q, j);  // fewer than k of them
  }
  __syncthreads();
  int have = w.count, left = w.need;
  for (int j0 = 0; left > 0 && j0 < V; j0 += kThreads) {
    const int j = j0 + threadIdx.x;
    const bool eq = j < V && order_key(to_f<T>(row[j])) == kth;
    const uint32_t votes = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) w.warp_sum[wid] = __popc(votes);
    __syncthreads();
    int before = __popc(votes & ((1u << lane) - 1)), total = 0;
    for (int i = 0; i < kWarps; ++i) {
      if (i < wid) before += w.warp_sum[i];
      total += w.warp_sum[i];
    }
    if (eq && before < left) w.found[have + before] = candidate(kth, j);
    const int taken = min(total, left);
    have += taken;
    left -= taken;
    __syncthreads();
  }
  __syncthreads();
  write_ranked(w.found, k, k, cap, values, ids);
}

ME_DEVICE uint32_t cluster_at(const void* p, uint32_t rank) {
  uint32_t b;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(b) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(rank));
  return b;
}

// Adds a candidate to the list of the row's first block; those past its end are only counted.
ME_DEVICE void push(Work& work, int* count, uint64_t c) {
  uint32_t at;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(at) : "r"(cluster_at(count, 0)) : "memory");
  if (at < kFound)
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(cluster_at(&work.pick.found[at], 0)), "l"(c) : "memory");
}

// The largest v (its low 16 bits 0) that at least k of the keys reach, 0 if there are fewer: two bits a step.
ME_DEVICE uint32_t kth_bound(const uint32_t (&keys)[kMaxGroups], int n, int k, uint32_t (*counts)[kWarps][2]) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  uint32_t bound = 0;
#pragma unroll 1
  for (int bit = 30, turn = 0; bit >= 16; bit -= 2, turn ^= 1) {
    const uint32_t v1 = bound | 1u << bit, v2 = bound | 2u << bit, v3 = bound | 3u << bit;
    uint32_t c12 = 0, c3 = 0;  // (a count is 4096 at most)
#pragma unroll
    for (int i = 0; i < kMaxGroups; ++i) {
      if (i >= n) break;
      c12 += (keys[i] >= v1 ? 1u : 0u) + (keys[i] >= v2 ? 1u << 16 : 0u);
      c3 += keys[i] >= v3 ? 1u : 0u;
    }
    c12 = __reduce_add_sync(0xffffffffu, c12);
    c3 = __reduce_add_sync(0xffffffffu, c3);
    if (lane == 0) {
      counts[turn][wid][0] = c12;
      counts[turn][wid][1] = c3;
    }
    __syncthreads();
    c12 = c3 = 0;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) {
      c12 += counts[turn][i][0];
      c3 += counts[turn][i][1];
    }
    if (c3 >= (uint32_t)k) bound = v3;
    else if (c12 >> 16 >= (uint32_t)k) bound = v2;
    else if ((c12 & 0xffff) >= (uint32_t)k) bound = v1;
  }
  return bound;
}

// One cluster a row. A thread's groups are 2^lg_group of its vectors each.
template <typename T, bool kCap>
__global__ void __launch_bounds__(kThreads, 4)
    top_kernel(Rows<const T> x, int V, int lg_ranks, int k, int lg_group, int groups, Scale sc,
               float* __restrict__ values, int64_t* __restrict__ ids, float* __restrict__ lse) {
  extern __shared__ uint4 dynamic[];
  __shared__ float2 part[kWarps];
  __shared__ uint32_t counts[2][kWarps][2];
  __shared__ int found, hits;
  Work& work = *reinterpret_cast<Work*>(dynamic);
  uint32_t* top = reinterpret_cast<uint32_t*>(dynamic + sizeof(Work) / sizeof(uint4));  // [groups][thread]
  const int64_t r = blockIdx.x >> lg_ranks;
  const int rank = blockIdx.x & ((1 << lg_ranks) - 1);
  const Slice<T> sl(x.row(r), V, rank, lg_ranks);
  if (threadIdx.x == 0) found = hits = 0;
  float best = -INFINITY;
  const int group = 1 << lg_group, count = sl.count();
  MaxSum a = slice_sum<T, kCap>(
      sl, sc, KeepAll(), work.ring,
      [&](uint4 v, int i) {
        best = fmaxf(best, vec_max<T, false>(v));
        if ((i + 1 & group - 1) == 0) {
          top[(i >> lg_group) * kThreads + threadIdx.x] = order_key(best);
          best = -INFINITY;
        }
      });
  if (count & group - 1) top[(count >> lg_group) * kThreads + threadIdx.x] = order_key(best);
  for (int g = (count + group - 1) >> lg_group; g < groups; ++g) top[g * kThreads + threadIdx.x] = 0;
  a = row_merge(a, part, lg_ranks);  // (behind its barrier the blocks' groups are there)
  const bool lead = rank == 0;
  if (lead && threadIdx.x == 0) lse[r] = a.m + logf(a.s);
  values += r * k;
  ids += r * k;
  if (a.s != a.s) {  // a NaN or +inf: the same for the whole cluster
    row_done(lg_ranks);
    if (lead) exact_top<T>(sl.row, V, k, sc.cap, work, values, ids);
    return;
  }
  uint32_t keys[kMaxGroups];
  const int n = groups << lg_ranks;
#pragma unroll
  for (int i = 0; i < kMaxGroups; ++i) {
    keys[i] = 0;
    if (i >= n) continue;
    const uint32_t* mine = &top[(i >> lg_ranks) * kThreads + threadIdx.x];
    if (lg_ranks == 0) {
      keys[i] = *mine;
    } else {
      asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(keys[i]) : "r"(cluster_at(mine, i & ((1 << lg_ranks) - 1))));
    }
  }
  const uint32_t bound = kth_bound(keys, n, k, counts);
  for (int g = 0; g < groups; ++g) {
    if (top[g * kThreads + threadIdx.x] < bound || g << lg_group >= count) continue;
    const int at = atomicAdd(&hits, 1);
    if (at < kHits) work.pick.hits[at] = g * kThreads + threadIdx.x;
  }
  __syncthreads();
  const int todo = min(hits, kHits) << lg_group;
  if (hits <= kHits) {
    for (int i = threadIdx.x; i < todo; i += kThreads) {
      const int h = work.pick.hits[i >> lg_group];
      const int vec = sl.begin + (h & kThreads - 1) + ((h / kThreads << lg_group) + (i & group - 1)) * kThreads;
      if (vec >= sl.end) continue;
      Vec16<T> v;
      v.u = *reinterpret_cast<const uint4*>(sl.row + sl.column(vec));
#pragma unroll
      for (int e = 0; e < Vec16<T>::kN; ++e) {
        const uint32_t q = order_key(to_f<T>(v.h[e]));
        if (q >= bound) push(work, &found, candidate(q, sl.column(vec) + e));
      }
    }
    const int j = sl.single();
    if (j >= 0) {
      const uint32_t q = order_key(to_f<T>(sl.row[j]));
      if (q >= bound) push(work, &found, candidate(q, j));
    }
  } else if (threadIdx.x == 0) {  // too many: more candidates than there is room for
    asm volatile("red.shared::cluster.add.u32 [%0], %1;" ::"r"(cluster_at(&found, 0)), "r"(kFound + 1) : "memory");
  }
  __syncthreads();
  row_done(lg_ranks);
  if (lg_ranks > 0) {
    cluster_arrive();
    cluster_wait();
  }
  if (!lead) return;
  const int n_found = found;
  if (n_found >= k && n_found <= kFound) write_ranked(work.pick.found, n_found, k, sc.cap, values, ids);
  else exact_top<T>(sl.row, V, k, sc.cap, work, values, ids);
}

}  // namespace

namespace me {

void launch_top_logits(const Logits& x, int k, float temp, float* values, int64_t* ids, float* lse,
                       cudaStream_t stream) {
  const int ranks = ranks_for(x.N, x.V), lg_ranks = ilog2(ranks);
  // Groups of up to eight vectors, as long as there are eight times as many of them as logits asked
  // for (then about 1.07 k logits reach the bound); more vectors where a thread would have too many groups.
  const int64_t vecs = (x.V * (x.type == LogitType::kF32 ? 4 : 2) + 15) / 16;
  const int per_thread = (int)(((vecs + ranks - 1) / ranks + kThreads - 1) / kThreads);
  int lg_group = 0;
  while (lg_group < 3 && vecs >> (lg_group + 1) >= 8 * k) ++lg_group;
  while (((per_thread + (1 << lg_group) - 1) >> lg_group) << lg_ranks > kMaxGroups) ++lg_group;
  const int groups = (per_thread + (1 << lg_group) - 1) >> lg_group;
  const int smem = sizeof(Work) + groups * kThreads * 4;
  ME_LOGITS_DISPATCH(x.type, ME_CAP_DISPATCH(x.cap, {
    allow_smem(top_kernel<T, kCap>, smem);
    launch_cluster(top_kernel<T, kCap>, x.N * ranks, ranks, smem, stream, rows_in<T>(x), x.V, lg_ranks, k, lg_group,
                   groups, make_scale(x.cap, temp), values, ids, lse);
  }));
}

}  // namespace me

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
// exact k-th logit by radix selection, some passes over the row. 2048 x 262144 bf16, softcap 30, k 64: 268 us (one
// read takes 164 us at the copy rate). Three quarters of the issue slots are taken (the sum's 97 for 8 logits a thread, 12
// for the maxima); the selection, which follows a row's walk, and three blocks an SM instead of four leave the rest.
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

// A lower bound of the k-th largest of the row's group maxima: at least k of them reach it, and few more than that
// (2 k + 64, or as many as are equal). Each thread brings the largest of its groups; 256 threads reach the smallest of
// those, so the k-th largest lies between it and the largest key. A histogram of 256 steps over that range tells the
// step that it is in, a second one over that step where too many lie there.
struct Bound {
  uint32_t ends[kWarps][2];
  int hist[256];
  int bin, above, count;
};
static_assert(kMaxTop <= kThreads);
ME_DEVICE uint32_t kth_bound(const uint32_t (&keys)[kMaxGroups], int n, int k, Bound& w) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  uint32_t high = 0;
#pragma unroll
  for (int i = 0; i < kMaxGroups; ++i) high = max(high, keys[i]);  // (those past n are 0)
  uint32_t low = __reduce_min_sync(0xffffffffu, high);
  high = __reduce_max_sync(0xffffffffu, high);
  if (lane == 0) {
    w.ends[wid][0] = low;
    w.ends[wid][1] = high;
  }
  w.hist[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWarps; ++i) {
    low = min(low, w.ends[i][0]);
    high = max(high, w.ends[i][1]);
  }
  for (int left = k;;) {
    const int shift = max(24 - __clz(high - low | 1u), 0);  // (high - low) >> shift <= 255
#pragma unroll
    for (int i = 0; i < kMaxGroups; ++i)
      if (i < n && keys[i] >= low && keys[i] <= high) atomicAdd(&w.hist[keys[i] - low >> shift], 1);
    __syncthreads();
    if (wid == 0) {
      int mine[8], sum = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += mine[i] = w.hist[lane * 8 + i];
      int from = sum;  // of this lane's steps and the higher lanes'
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_down_sync(0xffffffffu, from, o);
        if (lane + o < 32) from += v;
      }
      const uint32_t enough = __ballot_sync(0xffffffffu, from >= left);
      if (lane == 31 - __clz(enough | 1u)) {
        int above = from - sum, bin = 7;
        while (bin > 0 && above + mine[7] < left) {  // (the steps from the top; rotated, not indexed)
          above += mine[7];
#pragma unroll
          for (int i = 7; i > 0; --i) mine[i] = mine[i - 1];
          --bin;
        }
        w.bin = lane * 8 + bin;
        w.above = above;
        w.count = mine[7];
      }
    }
    __syncthreads();
    low += (uint32_t)w.bin << shift;
    if (shift == 0 || k - left + w.above + w.count <= 2 * k + 64) return low;
    left -= w.above;
    high = min(high, low + (1u << shift) - 1);
    __syncthreads();
    w.hist[threadIdx.x] = 0;
    __syncthreads();
  }
}

// One cluster a row. A thread's groups are 2^lg_group of its vectors each. (Three blocks an SM where the softcap's
// polynomial on 16-bit vectors wants more than 64 registers: 263 instead of 292 us for 2048 x 262144.)
template <typename T, bool kCap>
__global__ void __launch_bounds__(kThreads, kCap && sizeof(T) == 2 ? 3 : 4)
    top_kernel(Rows<const T> x, int V, int lg_ranks, int k, int lg_group, int groups, Scale sc,
               float* __restrict__ values, int64_t* __restrict__ ids, float* __restrict__ lse) {
  extern __shared__ uint4 dynamic[];
  __shared__ float2 part[kWarps];
  __shared__ Bound select;
  __shared__ int found, hits;
  Work& work = *reinterpret_cast<Work*>(dynamic);
  uint32_t* top = reinterpret_cast<uint32_t*>(dynamic + sizeof(Work) / sizeof(uint4));  // [groups][thread]
  const int64_t r = blockIdx.x >> lg_ranks;
  const int rank = blockIdx.x & ((1 << lg_ranks) - 1);
  const Slice<T> sl(x.row(r), V, rank, lg_ranks);
  if (threadIdx.x == 0) found = hits = 0;
  MaxOf<T> best;
  const int group = 1 << lg_group, count = sl.count();
  MaxSum a = slice_sum<T, kCap>(sl, sc, KeepAll(), work.ring, [&](const auto& v, int i) {
    constexpr int kV = sizeof(v) / sizeof(uint4);
#pragma unroll
    for (int u = 0; u < kV; ++u) best.add(v[u]);
    if ((i + kV & group - 1) == 0) {
      top[(i >> lg_group) * kThreads + threadIdx.x] = order_key(best.value());
      best.clear();
    }
  });
  if (count & group - 1) top[(count >> lg_group) * kThreads + threadIdx.x] = order_key(best.value());
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
  const uint32_t bound = kth_bound(keys, n, k, select);
  const float least = key_value(bound);  // (a NaN where there are too few groups: no candidates then)
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
        const float f = to_f<T>(v.h[e]);
        if (f >= least) push(work, &found, candidate(order_key(f), sl.column(vec) + e));
      }
    }
    const int j = sl.single();
    if (j >= 0) {
      const float f = to_f<T>(sl.row[j]);
      if (f >= least) push(work, &found, candidate(order_key(f), j));
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
  // (two blocks an SM: each block of a row selects over all its groups; 333 x 50001 with four: 40 instead of 31 us)
  const int ranks = ranks_for(x.N, x.V, 2), lg_ranks = ilog2(ranks);
  // Groups of two to eight vectors (they are seen by twos), eight as long as there are eight times as many of them
  // as logits asked for (then about 1.07 k logits reach the bound); more where a thread would have too many groups.
  const int64_t vecs = (x.V * (x.type == LogitType::kF32 ? 4 : 2) + 15) / 16;
  const int per_thread = (int)(((vecs + ranks - 1) / ranks + kThreads - 1) / kThreads);
  int lg_group = 1;
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

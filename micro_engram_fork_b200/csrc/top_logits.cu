// The k largest logits of each row with their ids, and the row's log-sum-exp (sm_100a): what a
// teacher records for a student that is trained on its top logits.
//
// Rows are ordered by the raw logit x (the softcap z = c tanh(x / c) is monotone), equal logits by
// the lower id, NaN above +inf. lse = log sum_j exp(z_j / tau).
#include "objectives.cuh"

#include <algorithm>

using namespace me;

namespace {

constexpr int kTopThreads = 512;

// A number that orders as the logits do: larger logit, larger key. -0 and +0 share one, NaN is on top.
ME_DEVICE uint32_t order_key(float x) {
  if (x != x) return 0xffffffffu;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
template <typename T, typename F>
ME_DEVICE void for_row(const T* row, int64_t V, F&& f) {
  for (int64_t j = threadIdx.x; j < V; j += blockDim.x) f(j, to_f<T>(row[j]));
}
ME_DEVICE MaxSum block_merge(MaxSum a, float* scratch) {
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, nw = blockDim.x >> 5;
  a = warp_merge(a);
  __syncthreads();
  if (lane == 0) scratch[wid] = a.m, scratch[32 + wid] = a.s;
  __syncthreads();
  MaxSum r;
  if (lane < nw) r.m = scratch[lane], r.s = scratch[32 + lane];
  return warp_merge(r);
}
// Radix selection, eight bits of the key a pass over the row: the exact k-th largest key, then every
// larger one and the lowest ids among its equals, ranked by counting.
template <typename T>
__global__ void __launch_bounds__(kTopThreads) top_logits_kernel(Rows<const T> x, int64_t N, int64_t V, int k, float cap,
                                                              float inv_temp, float* __restrict__ values,
                                                              int64_t* __restrict__ ids, float* __restrict__ lse) {
  __shared__ float scratch[64];
  __shared__ int hist[256];
  __shared__ uint32_t key[kMaxTop];
  __shared__ int col[kMaxTop];
  __shared__ int count, need, warp_sum_[kTopThreads / 32];
  __shared__ uint32_t prefix;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  for (int64_t r = blockIdx.x; r < N; r += gridDim.x) {
    const T* row = x.row(r);
    MaxSum a;
    for_row<T>(row, V, [&](int64_t, float v) { a.add(softcap(v, cap) * inv_temp); });
    a = block_merge(a, scratch);
    if (threadIdx.x == 0) {
      lse[r] = a.m + logf(a.s);
      prefix = 0;
      need = k;
      count = 0;
    }
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = threadIdx.x; i < 256; i += blockDim.x) hist[i] = 0;
      __syncthreads();
      const uint32_t want = prefix, mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
      for_row<T>(row, V, [&](int64_t, float v) {
        const uint32_t q = order_key(v);
        if ((q & mask) == want) atomicAdd(&hist[(q >> shift) & 255], 1);
      });
      __syncthreads();
      if (threadIdx.x == 0) {
        int left = need, b = 255;
        while (b > 0 && hist[b] < left) left -= hist[b--];
        need = left;
        prefix |= (uint32_t)b << shift;
      }
      __syncthreads();
    }
    const uint32_t kth = prefix;
    for_row<T>(row, V, [&](int64_t j, float v) {
      const uint32_t q = order_key(v);
      if (q > kth) {
        const int at = atomicAdd(&count, 1);
        key[at] = q;
        col[at] = (int)j;
      }
    });
    __syncthreads();
    int have = count, left = need;  // `left` equals of the k-th, the lowest ids first
    for (int64_t j0 = 0; left > 0 && j0 < V; j0 += blockDim.x) {
      const int64_t j = j0 + threadIdx.x;
      const bool eq = j < V && order_key(to_f<T>(row[j])) == kth;
      const uint32_t votes = __ballot_sync(0xffffffffu, eq);
      if (lane == 0) warp_sum_[wid] = __popc(votes);
      __syncthreads();
      int before = __popc(votes & ((1u << lane) - 1)), total = 0;
      for (int w = 0; w < kTopThreads / 32; ++w) {
        if (w < wid) before += warp_sum_[w];
        total += warp_sum_[w];
      }
      if (eq && before < left) {
        key[have + before] = kth;
        col[have + before] = (int)j;
      }
      have += min(total, left);
      left -= min(total, left);
      __syncthreads();
    }
    __syncthreads();
    for (int i = threadIdx.x; i < k; i += blockDim.x) {
      int rank = 0;
      for (int o = 0; o < k; ++o) rank += key[o] > key[i] || (key[o] == key[i] && col[o] < col[i]);
      values[r * k + rank] = softcap(to_f<T>(row[col[i]]), cap);
      ids[r * k + rank] = col[i];
    }
    __syncthreads();
  }
}

}  // namespace

namespace me {

void launch_top_logits(const Logits& x, int k, float temp, float* values, int64_t* ids, float* lse,
                       cudaStream_t stream) {
  const int grid = (int)std::min<int64_t>(x.N, (int64_t)objective_sms() * 4);
  ME_LOGITS_DISPATCH(x.type, top_logits_kernel<T><<<grid, kTopThreads, 0, stream>>>(rows_in<T>(x), x.N, x.V, k, x.cap,
                                                                                 1.f / temp, values, ids, lse));
}

}  // namespace me

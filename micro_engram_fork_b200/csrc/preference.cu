// Paired preference loss over packed sequences (sm_100a).
//
// 2P sequences, chosen and rejected in turn, packed over T tokens with offsets cu [2P + 1]. With
// r_s = sum over the tokens of s of (log-probability - the reference policy's), h = r_c - r_r:
//   sigmoid  L = -(1 - e) log sigma(beta h) - e log sigma(-beta h)    dL/dh = beta (e - sigma(-beta h))
//   hinge    L = max(0, 1 - beta h)                                   dL/dh = -beta [beta h < 1]
//   ipo      L = (h - 1 / (2 beta))^2                                 dL/dh = 2 (h - 1 / (2 beta))
// and dL / d logp_t = +-dL/dh for the tokens of the chosen / rejected sequence.
//
// One block a pair: it adds its two sequences (fp32, fixed order) and writes their tokens' gradient, so that value and
// gradient are one launch. Bound by the launch: 4 pairs over 6000 tokens, 9 us a call, of which the host takes 8. (A
// block reads all offsets ahead of its pair's, so that malformed ones cost no launch of their own: nothing for hundreds of
// pairs, 29 us for 4096, 164 us for 16384.)
#include "objectives.cuh"

using namespace me;

namespace {

constexpr int kPairThreads = 1024;  // at most: a block has 256 for short sequences

// log(1 + e^v) without overflow
ME_DEVICE float softplus(float v) { return fmaxf(v, 0.f) + log1pf(expf(-fabsf(v))); }

// A pair's offsets [a, b) and [b, c): `cu` is read as its running maximum, clamped to [0, T], so every token lies
// in one sequence, or ahead of the first or after the last one (those get no gradient), whatever it holds.
struct Bounds {
  int64_t a, b, c;
};
template <typename I>
ME_DEVICE Bounds pair_bounds(const I* cu, int64_t p, int64_t T) {
  __shared__ long long bound[4];  // the running maximum ahead of this pair, its three offsets
  long long top = 0;
  for (int64_t i = threadIdx.x; i < 2 * p; i += blockDim.x) top = max(top, (long long)cu[i]);
  if (threadIdx.x < 4) bound[threadIdx.x] = 0;
  __syncthreads();
  if (top > 0) atomicMax(&bound[0], top);
  __syncthreads();
  if (threadIdx.x == 0) {
    long long at = bound[0];
    for (int i = 0; i < 3; ++i) {
      at = max(at, (long long)cu[2 * p + i]);
      bound[1 + i] = min(at, (long long)T);
    }
  }
  __syncthreads();
  return {bound[1], bound[2], bound[3]};
}

template <typename I>
__global__ void __launch_bounds__(kPairThreads) preference_scale_kernel(const float* __restrict__ grad,
                                                                        const float* __restrict__ g,
                                                                        const I* __restrict__ cu, int64_t T,
                                                                        int64_t pairs, float* __restrict__ out) {
  const int64_t p = blockIdx.x;
  const Bounds s = pair_bounds(cu, p, T);
  const float c = g[p];
  for (int64_t t = s.a + threadIdx.x; t < s.c; t += blockDim.x) out[t] = grad[t] * c;
  if (p == 0)
    for (int64_t t = threadIdx.x; t < s.a; t += blockDim.x) out[t] = 0.f;
  if (p == pairs - 1)
    for (int64_t t = s.c + threadIdx.x; t < T; t += blockDim.x) out[t] = 0.f;
}

template <typename I>
__global__ void __launch_bounds__(kPairThreads) preference_kernel(
    const float* __restrict__ logp, const float* __restrict__ ref, const int64_t* __restrict__ target, int64_t T,
    const I* __restrict__ cu, int64_t pairs, int kind, float beta, float smooth, float scale,
    float* __restrict__ loss, float2* __restrict__ rewards, float* __restrict__ grad) {
  __shared__ float scratch[64];
  const int64_t p = blockIdx.x;
  const Bounds s = pair_bounds(cu, p, T);
  const int64_t a = s.a, b = s.b, c = s.c;
  auto ratio = [&](int64_t t) {
    if (target && target[t] == kIgnoreToken) return 0.f;
    return logp[t] - (ref ? ref[t] : 0.f);
  };
  float rc = 0.f, rr = 0.f;
#pragma unroll 8
  for (int64_t t = a + threadIdx.x; t < b; t += blockDim.x) rc += ratio(t);
#pragma unroll 8
  for (int64_t t = b + threadIdx.x; t < c; t += blockDim.x) rr += ratio(t);
  const float2 sums = block_sum2(rc, rr, scratch);
  const float h = sums.x - sums.y, u = beta * h;
  float l, d;
  if (kind == 0) {
    l = (1.f - smooth) * softplus(-u);
    if (smooth > 0.f) l += smooth * softplus(u);  // (0 times infinity where the rejected answer is impossible)
    d = beta * (smooth - 1.f / (1.f + expf(u)));
  } else if (kind == 1) {
    l = u < 1.f ? 1.f - u : (u == u ? 0.f : u);
    d = u < 1.f ? -beta : (u == u ? 0.f : u);
  } else {
    const float e = h - 0.5f / beta;
    l = e * e;
    d = 2.f * e;
  }
  if (threadIdx.x == 0) {
    loss[p] = l;
    rewards[p] = make_float2(beta * sums.x, beta * sums.y);
  }
  d *= scale;
  for (int64_t t = a + threadIdx.x; t < b; t += blockDim.x) grad[t] = d;
  for (int64_t t = b + threadIdx.x; t < c; t += blockDim.x) grad[t] = -d;
  if (p == 0)
    for (int64_t t = threadIdx.x; t < a; t += blockDim.x) grad[t] = 0.f;
  if (p == pairs - 1)
    for (int64_t t = c + threadIdx.x; t < T; t += blockDim.x) grad[t] = 0.f;
}

// Threads of a pair's block: all of them where a thread would have more than four tokens.
int pair_threads(int64_t tokens, int64_t pairs) { return tokens / pairs > 4 * 256 ? kPairThreads : 256; }

}  // namespace

namespace me {

void launch_preference(const PairArgs& a, float* loss, float2* rewards, float* grad, cudaStream_t stream) {
  const int threads = pair_threads(a.tokens, a.pairs);
  auto launch = [&](auto* cu) {
    preference_kernel<<<(unsigned)a.pairs, threads, 0, stream>>>(a.logp, a.ref, a.target, a.tokens, cu, a.pairs, a.kind,
                                                                  a.beta, a.smooth, a.scale, loss, rewards, grad);
  };
  if (a.cu64) launch(static_cast<const int64_t*>(a.cu));
  else launch(static_cast<const int*>(a.cu));
}

void launch_preference_scale(const float* grad, const float* g, const void* cu, bool cu64, int64_t tokens, int64_t pairs,
                             float* out, cudaStream_t stream) {
  auto launch = [&](auto* offsets) {
    preference_scale_kernel<<<(unsigned)pairs, pair_threads(tokens, pairs), 0, stream>>>(grad, g, offsets, tokens, pairs, out);
  };
  if (cu64) launch(static_cast<const int64_t*>(cu));
  else launch(static_cast<const int*>(cu));
}

}  // namespace me

// Appending new tokens to a paged cache: the fused q/k/v projection's heads are normalised, q and k rotated by their
// position, k and v written into their pages and q beside them, in one pass over the projection.
//
//   y = x / sqrt(mean(x^2) + eps) * w,  (a, b) -> (a cos - b sin, b cos + a sin)  of the halves a, b of y,
//
// all in 32 bits and rounded once. The angle p * f of a far position keeps no fraction in 32 bits (p = 100000: steps of
// 0.008): the product and its whole turns are taken in 64 bits, sine and cosine of the rest in 32.
//
// Bound: memory. Each element is read once and written once. A lane holds 8 elements of each half of a head in two 16-byte
// loads, so dim / 16 lanes share a head and a warp works on 512 / dim heads of one token; it keeps them for all tokens of its
// block, with its heads' weights in registers, and reads the block's table of sines from shared memory.
//
// Measured: 8192 new tokens of a sliding layer (32 q, 16 + 16 kv heads of 256; 537 MB) 102 us, 0.81 of the copy rate (half of the issue slots:
// 40 operations an element pair with its unpacking and packing). Small calls are the host's: one token 8.2 us, its kernel 3.3.
#include <algorithm>

#include "paged.cuh"

namespace me {
namespace {
using namespace paged;

constexpr int kThreads = 256, kWarps = 8, kResident = 3;  // blocks an SM: 64 to 80 registers
constexpr float kPrologue = 1.5f;  // (0.7 and 3: the same but for 8192 tokens at dim 512, 125 us with 0.7 and 115 with the others)

// Tokens of a block at most; the table of sines is this many times dim / 2 pairs.
template <int D>
constexpr int kTokens = D == 512 ? 8 : 16;

struct Place {
  int b, pos;  // b < 0: no sequence's token
  int64_t k, v;  // offset of its head 0 in the pages, < 0: no page
};

template <int D>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(AppendArgs a, int tokens_a_block, int plog) {
  constexpr int HALF = D / 2, L = D / 16, HPW = 32 / L;  // lanes a head, heads a warp
  constexpr int TB = kTokens<D>;
  __shared__ float4 table[TB * HALF / 2];  // [token][chunk of 2][lane]: (cos, sin) of two elements
  __shared__ Place place[TB];
  const PagedBatch& p = a.batch;
  const int hq = a.q_heads, hk = a.cache.heads, heads = hq + 2 * hk;
  const int n0 = blockIdx.x * tokens_a_block, n = min(tokens_a_block, p.tokens - n0);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l = lane % L;

  // where each token goes: every thread looks whether its sequences have any of them
  for (int i = threadIdx.x; i < n; i += kThreads) place[i] = {-1, 0, -1, -1};
  __syncthreads();
  for (int b = threadIdx.x; b < p.seqs; b += kThreads) {
    const Sequence s = sequence_of(p, b);
    for (int t = max(s.first, n0); t < min(s.first + s.count, n0 + n); ++t)
      if (s.context + t - s.first >= 0) place[t - n0].b = b, place[t - n0].pos = s.context + t - s.first;
  }
  __syncthreads();
  if (threadIdx.x < n && place[threadIdx.x].b >= 0) {
    Place& at = place[threadIdx.x];
    const int id = page_at(p, a.cache.pages, at.b, at.pos >> plog);
    const int64_t row = (int64_t)(at.pos & (a.cache.page - 1)) * D;
    if (id >= 0) at.k = id * a.cache.k_stride + row, at.v = id * a.cache.v_stride + row;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < n * HALF; i += kThreads) {
    const int t = i / HALF, j = i % HALF;
    // in turns: position * f / (2 pi), without its whole part
    double turns = (double)place[t].pos * ((double)a.inv_freq[j] * 0.15915494309189533577);
    turns -= rint(turns);
    float sn, cs;
    sincospif(2.f * (float)turns, &sn, &cs);
    float* at = reinterpret_cast<float*>(&table[t * (HALF / 2) + (j % 8) / 2 * L + j / 8]) + (j & 1) * 2;
    at[0] = cs, at[1] = sn;
  }
  __syncthreads();

  // A warp takes a group of heads; with fewer groups than warps several warps share one and take its tokens in turn.
  const int groups = (heads + HPW - 1) / HPW, sharing = max(kWarps / groups, 1);
  for (int g = sharing > 1 ? warp % groups : blockIdx.y * kWarps + warp; g < groups; g += gridDim.y * kWarps) {
    const int h = g * HPW + lane / L, t0 = sharing > 1 ? warp / groups : 0;
    const bool live = h < heads;
    const bool is_q = h < hq, is_v = h >= hq + hk;
    const int src_h = !live ? 0 : (a.kv_shared && is_v) ? h - hk : h;
    float wl[8], wh[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) wl[e] = wh[e] = 1.f;
    if (!is_v) {
      const float* w = is_q ? a.q_w : a.k_w;
#pragma unroll
      for (int e = 0; e < 8; ++e) wl[e] = w[l * 8 + e], wh[e] = w[HALF + l * 8 + e];
    }
    const bf16* src = reinterpret_cast<const bf16*>(a.qkv) + (int64_t)n0 * a.qkv_stride + (int64_t)src_h * D + l * 8;
    BF16x8 lo, hi, next_lo, next_hi;
    auto read = [&](int t, BF16x8& x, BF16x8& y) {
      x.u = *reinterpret_cast<const uint4*>(src + t * a.qkv_stride);
      y.u = *reinterpret_cast<const uint4*>(src + t * a.qkv_stride + HALF);
    };
    if (sharing > 1 && t0 >= sharing) break;  // (a warp left over)
    if (t0 < n) read(t0, next_lo, next_hi);
    for (int t = t0; t < n; t += sharing) {
      lo.u = next_lo.u, hi.u = next_hi.u;
      if (t + sharing < n) read(t + sharing, next_lo, next_hi);  // on its way while this one is worked on
      float xl[8], xh[8], ss = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        xl[e] = bf2f(lo.h[e]), xh[e] = bf2f(hi.h[e]);
        ss += xl[e] * xl[e] + xh[e] * xh[e];
      }
#pragma unroll
      for (int o = 1; o < L; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float rs = rsqrtf(ss / D + a.eps);
      const float4* tab = table + t * (HALF / 2) + l;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float4 cs = tab[c * L];
        float yl0 = xl[2 * c] * rs * wl[2 * c], yh0 = xh[2 * c] * rs * wh[2 * c];
        float yl1 = xl[2 * c + 1] * rs * wl[2 * c + 1], yh1 = xh[2 * c + 1] * rs * wh[2 * c + 1];
        if (!is_v) {
          const float a0 = yl0, a1 = yl1;
          yl0 = a0 * cs.x - yh0 * cs.y, yh0 = yh0 * cs.x + a0 * cs.y;
          yl1 = a1 * cs.z - yh1 * cs.w, yh1 = yh1 * cs.z + a1 * cs.w;
        }
        lo.h2[c] = __floats2bfloat162_rn(yl0, yl1);
        hi.h2[c] = __floats2bfloat162_rn(yh0, yh1);
      }
      const Place at = place[t];
      bf16* dst = nullptr;
      if (is_q) {
        dst = reinterpret_cast<bf16*>(a.q) + ((int64_t)(n0 + t) * hq + h) * D;
        if (at.b < 0) lo.u = hi.u = make_uint4(0, 0, 0, 0);  // a row of no sequence
      } else if (live && at.k >= 0) {
        dst = is_v ? reinterpret_cast<bf16*>(a.cache.v) + at.v + ((int64_t)(h - hq - hk) * D << plog)
                   : reinterpret_cast<bf16*>(a.cache.k) + at.k + ((int64_t)(h - hq) * D << plog);
      }
      if (dst != nullptr) {
        *reinterpret_cast<uint4*>(dst + l * 8) = lo.u;
        *reinterpret_cast<uint4*>(dst + HALF + l * 8) = hi.u;
      }
    }
    if (sharing > 1) break;
  }
}

template <int D>
void launch(const AppendArgs& a, int sms, cudaStream_t stream) {
  const int heads = a.q_heads + 2 * a.cache.heads, groups = (heads + 512 / D - 1) / (512 / D);
  // Tokens a block: its prologue takes about as long as kPrologue tokens, and blocks run in waves of `resident`, so the fewest
  // (waves x (tokens + prologue)). With fewer blocks than a wave the heads are split too. (Powers of two that left four blocks an SM, which
  // took a second or third wave for little: 2048 tokens 43 us, 33 now; 1000 of a global layer 41 and 29; 8192 109 and 102.)
  const int resident = kResident * sms;
  int tb = 1;
  float least = 1e30f;
  for (int n = 1; n <= kTokens<D>; ++n) {
    const int64_t blocks = ((int64_t)a.batch.tokens + n - 1) / n;
    const float cost = (float)((blocks + resident - 1) / resident) * (n + kPrologue);
    if (cost < least) least = cost, tb = n;
  }
  const int blocks = (a.batch.tokens + tb - 1) / tb;
  const int most = (groups + kWarps - 1) / kWarps;
  const int split = std::min(most, std::max(1, resident / blocks));
  int plog = 0;
  while ((1 << plog) < a.cache.page) ++plog;
  paged_append_kernel<D><<<dim3(blocks, split), kThreads, 0, stream>>>(a, tb, plog);
}

}  // namespace

void launch_paged_append(const AppendArgs& a, int sms, cudaStream_t stream) {
  switch (a.cache.dim) {
    case 64: return launch<64>(a, sms, stream);
    case 128: return launch<128>(a, sms, stream);
    case 256: return launch<256>(a, sms, stream);
    default: return launch<512>(a, sms, stream);
  }
}

}  // namespace me

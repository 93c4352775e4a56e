// What the kernels of the paged cache share: a sequence's place in the batch, looking a place up in the list of all
// work, bounds of keys. Lengths, offsets and page numbers come from device memory that no host check has seen, so all of
// them are brought into range here: a token outside its batch is not read, a page outside the cache is no page.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"
#include "paged.h"

namespace me {
namespace paged {

using bf16 = __nv_bfloat16;

// Positions are below 2^31: the host refuses tables that name more.
struct Sequence {
  int first, count;  // its new tokens
  int context;       // its tokens in the cache before them (negative: its length is below count)
};

ME_DEVICE Sequence sequence_of(const PagedBatch& p, int b) {
  const int s = min(max(p.cu[b], 0), p.tokens);
  const int e = min(max(p.cu[b + 1], s), p.tokens);
  return {s, e - s, max(p.lens[b], 0) - (e - s)};
}

// Keys [lo, hi) that any of the new tokens i0 .. i1 of a sequence sees and that its table has room for.
struct Keys {
  int lo, hi;
};
ME_DEVICE Keys keys_of(const PagedBatch& p, int page, const Sequence& s, int i0, int i1, int window) {
  const int room = p.width * page;
  const int hi = min(max(s.context + i1 + 1, 0), room);
  const int lo = window > 0 ? max(max(s.context + i0, 0) - window + 1, 0) : 0;  // (in this order nothing passes 32 bits)
  return {min(lo, hi), hi};
}

// The page at column `col` of sequence b's row, -1 where there is none.
ME_DEVICE int page_at(const PagedBatch& p, int pages, int b, int col) {
  if (col < 0 || col >= p.width) return -1;
  const int id = p.table[b * p.table_stride + col];
  return id >= 0 && id < pages ? id : -1;
}

// Work of all sequences in one line: `count(b)` units each. total() and find() are called by all NT threads of the block.
template <int NT>
struct WorkLine {
  static constexpr int W = NT / 32;
  struct Shared {
    int64_t warp[W];
    int64_t before;
    int b;
  };
  Shared& sh;
  int64_t mine = 0, upto = 0;  // of the last chunk of sequences that was scanned

  ME_DEVICE explicit WorkLine(Shared& s) : sh(s) {}

  // The sum over the block; upto: over this thread's and those before it.
  ME_DEVICE int64_t scan(int64_t v) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    mine = upto = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    __syncthreads();
    if (lane == 31) sh.warp[warp] = upto;
    __syncthreads();
    int64_t all = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if (i < warp) upto += sh.warp[i];
      all += sh.warp[i];
    }
    return all;
  }

  template <class Count>
  ME_DEVICE int64_t total(int seqs, Count count) {
    int64_t sum = 0;
    for (int c = 0; c < seqs; c += NT) sum += scan(c + (int)threadIdx.x < seqs ? count(c + threadIdx.x) : 0);
    return sum;
  }
  // The sequence that unit x lies in, and the units before it. x is below the total.
  template <class Count>
  ME_DEVICE int find(int seqs, Count count, int64_t x, int64_t& before) {
    int64_t base = 0;
    for (int c = 0; c < seqs; c += NT) {
      int64_t all;
      if (seqs <= NT) all = INT64_MAX;  // total() has just scanned them
      else all = scan(c + (int)threadIdx.x < seqs ? count(c + threadIdx.x) : 0);
      const int64_t b0 = base + upto - mine;
      if (x >= b0 && x < base + upto) sh.before = b0, sh.b = c + threadIdx.x;
      if (seqs <= NT || x < base + all) break;
      base += all;
    }
    __syncthreads();
    before = sh.before;
    const int b = sh.b;
    __syncthreads();
    return b;
  }
};

// ------------------------------------------------------------------------------- attention
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
// A running maximum (in log2 units) moves only when a score is this far above it: p stays below 2^8.
constexpr float kSlack = 8.f;

ME_DEVICE float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// A part's sum (of terms below its own maximum) next to the whole's maximum.
ME_DEVICE float share(float2 max_sum, float top) {
  return max_sum.y == 0.f || max_sum.x == -INFINITY ? max_sum.y : max_sum.y * ex2(max_sum.x - top);
}
ME_DEVICE uint32_t pack2(float a, float b) {
  const __nv_bfloat162 x = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&x);
}

// The rows of no sequence: a log-sum-exp of -inf, and zeros (a caller's own output is left as it is).
template <int D>
ME_DEVICE void clear_rest(const PagedAttentionArgs& a, int threads) {
  const PagedBatch& p = a.batch;
  const int head = p.seqs ? min(max(p.cu[0], 0), p.tokens) : p.tokens;
  const int tail = p.seqs ? min(max(p.cu[p.seqs], head), p.tokens) : p.tokens;
  for (int64_t i = (int64_t)blockIdx.x * threads + threadIdx.x; i < (int64_t)(head + p.tokens - tail) * a.q_heads;
       i += (int64_t)gridDim.x * threads) {
    const int h = (int)(i % a.q_heads), n = (int)(i / a.q_heads), t = n < head ? n : n - head + tail;
    a.lse[(int64_t)h * p.tokens + t] = -INFINITY;
    if (!a.clear_rest) continue;
    bf16* o = reinterpret_cast<bf16*>(a.o) + t * a.o_token + h * a.o_head;
    for (int c = 0; c < D; c += 8) *reinterpret_cast<uint4*>(o + c) = make_uint4(0, 0, 0, 0);
  }
}

}  // namespace paged
}  // namespace me

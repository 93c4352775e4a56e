// Attention of new tokens over a paged cache.
//
// Rows (token, query head) of a sequence whose query heads share a key head read the same keys, so a unit of
// work is (sequence, key head, 8 or 16 of those rows) over blocks of 64 keys. One new token a sequence, 2 to 8 query heads a key head: two
// products of 2 to 8 rows with each 2-byte element, far below what the tensor cores need to be busy; the keys' and values' way
// from memory is the bound, and everything here is for keeping loads in flight:
//
//   * All units' blocks are one line, cut into as many equal pieces as blocks fit on the GPU (two on an SM): whatever the
//     lengths, every SM reads the same number of bytes. A piece that begins or ends inside a unit leaves (max, sum, output) of its part
//     in the workspace, and a second kernel joins them; it is launched beside the first one's end (programmatic
//     dependent launch).
//   * A warp works alone: its own 16 keys of each block, its own ring of shared memory (24 KB, cp.async, rows outside the
//     range and pages that are none filled with zeros), its own running maximum and sum. The 4 warps meet at a unit's end.
//   * Keys are the M side of mma.m16n8k16 and 8 rows its N side: S^T = K Q^T, O^T += V^T P^T. The rows of S^T become the
//     B operand of the second product through movmatrix, without shared memory. P goes as two bf16 terms (its value rounded and
//     what the rounding left, relative error 2^-17), which the idle tensor cores give for nothing: the output is as exact as its own
//     rounding.
//
// Measured, single tokens: 128 sequences of 30 to 9000 tokens in a sliding layer (window 1024, 16 heads of 256; 2.0 GB) 307-324 us, 0.94-1.0 of the copy
// rate; 64 of 100 to 16000 in a global one (4 heads of 512; 4.5 GB) 745-762 us, 0.91-0.94; one over 131072 (1.07 GB) 196-200 us, 0.82-0.84 (ramp, two partial
// blocks each piece, the join: 25-30 us); one sliding sequence (16 MB) 14 us, two launches one after another.
#include <algorithm>

#include "paged.cuh"

namespace me {
namespace {
using namespace paged;

ME_DEVICE uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
// 16 bytes global -> shared; `bytes` 0: zeros, nothing is read.
ME_DEVICE void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
ME_DEVICE void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
ME_DEVICE void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
ME_DEVICE void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
ME_DEVICE void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
ME_DEVICE uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
ME_DEVICE void mma16n8k16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// ------------------------------------------------------------------------------- few rows a key head
constexpr int kWarps = 4, kTile = 16, kBlock = kWarps * kTile, kThreads = kWarps * 32;

// NT: sets of 8 rows that go through the keys together. Two of them where a sequence has more than 8 rows and its O fits the registers (up
// to dim 256): the keys are read once and not twice (64 sequences of 5 new tokens in a sliding layer: 345 -> 222 us, 8 tokens: 239; at
// the copy rate 165). Where no sequence has more than 8 rows one set is enough: two would cost registers and empty products.
template <int D, int NT>
struct Cfg {
  static constexpr int ROWS = 8 * NT;
  static constexpr int UC = D < 256 ? D : 256;  // columns of a unit of the ring
  static constexpr int UNIT = kTile * UC * 2;
  static constexpr int PARTS = D / UC;          // units a tile of K
  static constexpr int RING = 24 * 1024 / UNIT;
  static constexpr int PITCH = D + 4;           // floats of a row where the warps meet: no bank conflicts
  static constexpr int SMEM = kWarps * RING * UNIT;
  static_assert(kWarps * ROWS * PITCH * 4 <= SMEM, "the warps meet in the ring");
  static_assert(2 * (SMEM + 2048) <= 227 * 1024, "two blocks an SM");
};

struct RowsArgs {
  PagedAttentionArgs a;
  float* part_o;   // [slots][rows][D]
  float2* part_ml; // [slots][rows] (maximum, sum)
  int rows;        // of a unit
  int pieces;      // blocks of the grid
  int plog;
  int most_rows;   // sequences with more rows are the tensor cores' (paged_tiles.cu)
};

struct UnitsOf {
  int tiles;   // row tiles of the sequence
  int blocks;  // blocks of 64 keys of each
};
ME_DEVICE UnitsOf units_of(const RowsArgs& args, int b, const Sequence& s) {
  const PagedAttentionArgs& a = args.a;
  const int group = a.q_heads / a.cache.heads;
  if (s.count == 0 || (int64_t)s.count * group > args.most_rows) return {0, 0};
  const Keys k = keys_of(a.batch, a.cache.page, s, 0, s.count - 1, a.window);
  return {(s.count * group + args.rows - 1) / args.rows, max((k.hi + kBlock - 1) / kBlock - k.lo / kBlock, 1)};
}

// The line of blocks in pieces of the same length, the first `rest` of them one longer.
struct Cut {
  int64_t total;
  int pieces;
  int64_t each;
  int rest;
  ME_DEVICE Cut(int64_t blocks, int most) : total(blocks), pieces((int)min((int64_t)most, blocks)) {
    if (pieces == 0) each = 0, rest = 0;
    else if (total <= UINT32_MAX) each = (uint32_t)total / (uint32_t)pieces, rest = (uint32_t)total % (uint32_t)pieces;
    else each = total / pieces, rest = (int)(total % pieces);
  }
  ME_DEVICE int64_t start(int i) const { return i * each + min(i, rest); }
  ME_DEVICE int owner(int64_t x) const {  // the piece that block x lies in
    const int64_t longer = rest * (each + 1), in = x < longer ? x : x - longer, by = x < longer ? each + 1 : each;
    const int n = in <= UINT32_MAX && by <= UINT32_MAX ? (int)((uint32_t)in / (uint32_t)by) : (int)(in / by);
    return x < longer ? n : rest + n;
  }
};

template <int D, int NT>
__global__ void __launch_bounds__(kThreads, 2) paged_rows_kernel(const RowsArgs args) {
  using C = Cfg<D, NT>;
  constexpr int kRows = C::ROWS;
  extern __shared__ __align__(128) uint8_t ring[];
  __shared__ WorkLine<kThreads>::Shared line_shared;
  __shared__ float2 warp_ml[kWarps][kRows];
  const PagedAttentionArgs& a = args.a;
  const PagedBatch& p = a.batch;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int hk = a.cache.heads, group = a.q_heads / hk, plog = args.plog;
  const int g = lane >> 2, t4 = lane & 3;  // a fragment's row and column pair
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  clear_rest<D>(a, kThreads);

  auto count = [&](int b) -> int64_t {
    const UnitsOf u = units_of(args, b, sequence_of(p, b));
    return (int64_t)u.tiles * hk * u.blocks;
  };
  WorkLine<kThreads> line(line_shared);
  const Cut cut(line.total(p.seqs, count), args.pieces);
  if (blockIdx.x >= cut.pieces) return;
  const int64_t x0 = cut.start(blockIdx.x), x1 = cut.start(blockIdx.x + 1);
  int64_t x = x0, before;
  int b = line.find(p.seqs, count, x, before);

  const uint32_t my_ring = smem_u32(ring) + warp * (C::RING * C::UNIT);
  constexpr int CPR = C::UC / 8, RPP = 32 / CPR;  // 16-byte chunks a row, rows a pass of the warp
  const int c_row = lane / CPR, c_col = lane % CPR;
  const int l_row = (lane & 7) + ((lane >> 3) & 1) * 8;

  while (x < x1) {
    const Sequence s = sequence_of(p, b);
    const UnitsOf u = units_of(args, b, s);
    const int64_t in_seq = x - before;
    if (in_seq >= (int64_t)u.tiles * hk * u.blocks) {  // on to the next sequence that has any
      before += (int64_t)u.tiles * hk * u.blocks;
      ++b;
      continue;
    }
    const int unit = (int)(in_seq / u.blocks), first_block = (int)(in_seq % u.blocks);
    const int blocks = (int)min((int64_t)(u.blocks - first_block), x1 - x);
    const int tile = unit % u.tiles, kv = unit / u.tiles;  // a head's row tiles lie together: their keys meet in L2
    const int r0 = tile * kRows, rows = min(kRows, s.count * group - r0);
    const Keys keys = keys_of(p, a.cache.page, s, r0 / group, (r0 + rows - 1) / group, a.window);
    const int seq_lo = keys_of(p, a.cache.page, s, 0, s.count - 1, a.window).lo;
    const int start = (seq_lo / kBlock + first_block) * kBlock + warp * kTile;  // this warp's first key; a tile a block

    // this lane's two rows of each S^T: their last and first keys
    int last[2 * NT], from[2 * NT];
#pragma unroll
    for (int e = 0; e < 2 * NT; ++e) {
      const int r = r0 + e / 2 * 8 + 2 * t4 + e % 2, pos = s.context + r / group;
      last[e] = r < r0 + rows ? pos : -1;
      from[e] = a.window > 0 ? max(pos, 0) - a.window + 1 : 0;
    }
    const int all_last = s.context + r0 / group;
    const int all_from = a.window > 0 ? max(s.context + (r0 + rows - 1) / group, 0) - a.window + 1 : 0;

    uint32_t qf[NT][D / 16][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = r0 + n * 8 + g;
      const bf16* q = reinterpret_cast<const bf16*>(a.q) + (int64_t)(s.first + r / group) * a.q_token + (kv * group + r % group) * a.q_head + 2 * t4;
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        qf[n][k][0] = n * 8 + g < rows ? *reinterpret_cast<const uint32_t*>(q + k * 16) : 0u;
        qf[n][k][1] = n * 8 + g < rows ? *reinterpret_cast<const uint32_t*>(q + k * 16 + 8) : 0u;
      }
    }
    const bf16* kbase = reinterpret_cast<const bf16*>(a.cache.k) + ((int64_t)kv * D << plog);
    const bf16* vbase = reinterpret_cast<const bf16*>(a.cache.v) + ((int64_t)kv * D << plog);

    int ids = -1;        // pages of the 32 tiles around the one that is loaded next, one a lane
    uint32_t there = 0;  // bit j % 32: tile j has a page
    int slot_in = 0, slot_out = 0;
    auto issue = [&](int j, int part) {  // part of tile j: columns of K, then of V
      if (j < blocks) {
        if (part == 0) {
          if ((j & 31) == 0) {
            const int key = start + (j + lane) * kBlock;
            ids = j + lane < blocks && key < keys.hi && key + kTile > keys.lo ? page_at(p, a.cache.pages, b, key >> plog) : -1;
          }
          const int id = __shfl_sync(0xffffffffu, ids, j & 31);
          there = (there & ~(1u << (j & 31))) | ((id >= 0 ? 1u : 0u) << (j & 31));
        }
        const int id = __shfl_sync(0xffffffffu, ids, j & 31);
        const int key = start + j * kBlock;
        const bool is_v = part >= C::PARTS;
        const bf16* src = (is_v ? vbase : kbase) + (id < 0 ? 0 : id * (is_v ? a.cache.v_stride : a.cache.k_stride)) +
                          (int64_t)((key & (a.cache.page - 1)) + c_row) * D + (part % C::PARTS) * C::UC + c_col * 8;
        const uint32_t dst = my_ring + slot_in * C::UNIT;
#pragma unroll
        for (int i = 0; i < kTile / RPP; ++i) {
          const int row = i * RPP + c_row;
          const bool in = id >= 0 && key + row >= keys.lo && key + row < keys.hi;
          cp_async16(dst + row * (C::UC * 2) + ((c_col ^ (row & 7)) << 4), in ? src + i * RPP * D : kbase, in ? 16 : 0);
        }
        slot_in = slot_in + 1 == C::RING ? 0 : slot_in + 1;
      }
      cp_commit();
    };

    float acc[NT][D / 16][4];
    float m[2 * NT], sum[2 * NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int i = 0; i < D / 16; ++i) acc[n][i][0] = acc[n][i][1] = acc[n][i][2] = acc[n][i][3] = 0.f;
      m[2 * n] = m[2 * n + 1] = -INFINITY, sum[2 * n] = sum[2 * n + 1] = 0.f;
    }
    const float to_log2 = a.scale * kLog2e;

    constexpr int UPT = 2 * C::PARTS;
#pragma unroll
    for (int i = 0; i < C::RING; ++i) issue(i / UPT, i % UPT);
    for (int j = 0; j < blocks; ++j) {
      float sc[NT][2][4] = {};
      uint32_t ph[NT][2], pl[NT][2];
#pragma unroll
      for (int part = 0; part < UPT; ++part) {
        cp_wait<C::RING - 1>();
        __syncwarp();
        const uint32_t at = my_ring + slot_out * C::UNIT + l_row * (C::UC * 2);
        if (part < C::PARTS) {
#pragma unroll
          for (int k = 0; k < C::UC / 16; ++k) {
            uint32_t f[4];
            ldsm4(f, at + (((2 * k + (lane >> 4)) ^ (l_row & 7)) << 4));
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16n8k16(sc[n][k & 1], f, qf[n][part * (C::UC / 16) + k][0], qf[n][part * (C::UC / 16) + k][1]);
          }
        } else {
          if (part == C::PARTS) {  // the scores are whole: softmax
            const int key0 = start + j * kBlock, key = key0 + g;
            const bool page = (there >> (j & 31)) & 1;
            const bool open = page && key0 >= all_from && key0 + kTile - 1 <= all_last && key0 + kTile <= keys.hi;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              float v[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) v[e] = (sc[n][0][e] + sc[n][1][e]) * to_log2;
              if (!open) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const int at_key = key + (e >> 1) * 8;
                  if (!page || at_key > last[2 * n + (e & 1)] || at_key < from[2 * n + (e & 1)] || at_key >= keys.hi) v[e] = -INFINITY;
                }
              }
              float& m0 = m[2 * n];
              float& m1 = m[2 * n + 1];
              float mx[2] = {fmaxf(v[0], v[2]), fmaxf(v[1], v[3])};
#pragma unroll
              for (int o = 4; o < 32; o <<= 1) {
                mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], o));
                mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], o));
              }
              const bool up0 = mx[0] > m0 + kSlack, up1 = mx[1] > m1 + kSlack;  // -inf + slack = -inf: any score is above it
              if (__any_sync(0xffffffffu, up0 || up1)) {
                const float f0 = up0 ? ex2(m0 - mx[0]) : 1.f, f1 = up1 ? ex2(m1 - mx[1]) : 1.f;
                if (up0) m0 = mx[0];
                if (up1) m1 = mx[1];
                sum[2 * n] *= f0, sum[2 * n + 1] *= f1;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) acc[n][i][0] *= f0, acc[n][i][1] *= f1, acc[n][i][2] *= f0, acc[n][i][3] *= f1;
              }
              const float z0 = m0 == -INFINITY ? 0.f : m0, z1 = m1 == -INFINITY ? 0.f : m1;
              v[0] = ex2(v[0] - z0), v[1] = ex2(v[1] - z1), v[2] = ex2(v[2] - z0), v[3] = ex2(v[3] - z1);
              sum[2 * n] += v[0] + v[2], sum[2 * n + 1] += v[1] + v[3];
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const uint32_t h = pack2(v[2 * e], v[2 * e + 1]);
                const float h0 = __uint_as_float(h << 16), h1 = __uint_as_float(h & 0xffff0000u);
                ph[n][e] = transpose8x8(h);
                pl[n][e] = transpose8x8(pack2(v[2 * e] - h0, v[2 * e + 1] - h1));
              }
            }
          }
          // V^T: the transposed reads give dimensions as rows
          const uint32_t vat = my_ring + slot_out * C::UNIT + ((lane & 7) + (lane >> 4) * 8) * (C::UC * 2);
#pragma unroll
          for (int k = 0; k < C::UC / 16; ++k) {
            uint32_t f[4];
            ldsm4_t(f, vat + (((2 * k + ((lane >> 3) & 1)) ^ (lane & 7)) << 4));
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              mma16n8k16(acc[n][(part - C::PARTS) * (C::UC / 16) + k], f, ph[n][0], ph[n][1]);
              mma16n8k16(acc[n][(part - C::PARTS) * (C::UC / 16) + k], f, pl[n][0], pl[n][1]);
            }
          }
        }
        __syncwarp();
        slot_out = slot_out + 1 == C::RING ? 0 : slot_out + 1;
        issue(j + (part + C::RING) / UPT, (part + C::RING) % UPT);
      }
    }

    // ---- the four warps meet
#pragma unroll
    for (int e = 0; e < 2 * NT; ++e) {
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], o);
      if (g == 0) warp_ml[warp][e / 2 * 8 + 2 * t4 + e % 2] = make_float2(m[e], sum[e]);
    }
    cp_wait<0>();
    __syncthreads();
    float* meet = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float f[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, warp_ml[w][n * 8 + 2 * t4 + e].x);
        f[e] = m[2 * n + e] == -INFINITY ? 0.f : ex2(m[2 * n + e] - top);
      }
      float* out = meet + (warp * kRows + n * 8 + 2 * t4) * C::PITCH + g;
#pragma unroll
      for (int i = 0; i < D / 16; ++i) {
        out[i * 16] = acc[n][i][0] * f[0], out[C::PITCH + i * 16] = acc[n][i][1] * f[1];
        out[i * 16 + 8] = acc[n][i][2] * f[0], out[C::PITCH + i * 16 + 8] = acc[n][i][3] * f[1];
      }
    }
    __syncthreads();
    const bool whole = blocks == u.blocks;
    const int64_t slot = 2 * (int64_t)blockIdx.x + (x == x0 ? 0 : 1);
    for (int i = threadIdx.x; i < rows * (D / 4); i += kThreads) {
      const int r = i / (D / 4), c = i % (D / 4) * 4;
      float top = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) top = fmaxf(top, warp_ml[w][r].x);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) l += share(warp_ml[w][r], top);
      float4 o = *reinterpret_cast<const float4*>(meet + r * C::PITCH + c);
#pragma unroll
      for (int w = 1; w < kWarps; ++w) {
        const float4 y = *reinterpret_cast<const float4*>(meet + (w * kRows + r) * C::PITCH + c);
        o.x += y.x, o.y += y.y, o.z += y.z, o.w += y.w;
      }
      if (whole) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int t = s.first + (r0 + r) / group, h = kv * group + (r0 + r) % group;
        uint2 b4;
        b4.x = pack2(o.x * inv, o.y * inv), b4.y = pack2(o.z * inv, o.w * inv);
        *reinterpret_cast<uint2*>(reinterpret_cast<bf16*>(a.o) + t * a.o_token + h * a.o_head + c) = b4;
        if (c == 0) a.lse[(int64_t)h * p.tokens + t] = l == 0.f ? -INFINITY : (top + log2f(l)) * kLn2;
      } else {
        *reinterpret_cast<float4*>(args.part_o + (slot * kRows + r) * D + c) = o;
        if (c == 0) args.part_ml[slot * kRows + r] = make_float2(top, l);
      }
    }
    __syncthreads();  // the ring is free again
    x += blocks;
  }
}

// Joins the parts of units that were cut. A block finds the unit that its border between two pieces lies in; the blocks of a unit's borders share its
// rows, 128 columns at a time. Units of many parts: the block's warps take every eighth part of a task; of few: a task a warp.
constexpr int kJoinThreads = 256, kJoinWarps = 8;

template <int D>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const RowsArgs args) {
  constexpr int COLS = D < 128 ? D : 128, SETS = D / COLS;  // columns of a task
  __shared__ WorkLine<kJoinThreads>::Shared line_shared;
  __shared__ float4 meet[kJoinWarps][32];
  __shared__ float meet_l[kJoinWarps];
  const PagedAttentionArgs& a = args.a;
  const PagedBatch& p = a.batch;
  const int hk = a.cache.heads, group = a.q_heads / hk, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto blocks_of = [&](int b) -> int64_t {
    const UnitsOf u = units_of(args, b, sequence_of(p, b));
    return (int64_t)u.tiles * hk * u.blocks;
  };
  WorkLine<kJoinThreads> line(line_shared);
  const Cut cut(line.total(p.seqs, blocks_of), args.pieces);
  const int border = blockIdx.x + 1;
  if (border < cut.pieces) {
    const int64_t x = cut.start(border);  // the border is before block x of the line
    int64_t before;
    const int b = line.find(p.seqs, blocks_of, x, before);
    const Sequence s = sequence_of(p, b);
    const UnitsOf u = units_of(args, b, s);
    const int64_t in_seq = x - before;
    const int unit = in_seq <= UINT32_MAX ? (int)((uint32_t)in_seq / (uint32_t)u.blocks) : (int)(in_seq / u.blocks);
    const int64_t begin = before + (int64_t)unit * u.blocks;
    const int first = cut.owner(begin), count = cut.owner(begin + u.blocks - 1) - first + 1;  // the unit's pieces
    const int tile = unit % u.tiles, kv = unit / u.tiles, r0 = tile * args.rows, rows = min(args.rows, s.count * group - r0);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (x == begin) return;  // it separates two units
    const int borders = count - 1, mine = border - first - 1, tasks = rows * SETS;
    const bool split = 2 * borders >= tasks;  // all warps on one task
    for (int task = split ? mine : mine * kJoinWarps + warp; task < tasks; task += split ? borders : borders * kJoinWarps) {
      const int r = task % rows, c = task / rows * COLS + lane * 4;
      auto row_of = [&](int k) { return (2 * (int64_t)(first + k) + (cut.start(first + k) >= begin ? 0 : 1)) * args.rows + r; };
      float top = -INFINITY;
      for (int k = lane; k < count; k += 32) top = fmaxf(top, args.part_ml[row_of(k)].x);
      top = warp_max(top);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      float l = 0.f;
#pragma unroll 8
      for (int k = split ? warp : 0; k < count; k += split ? kJoinWarps : 1) {
        const float2 x = args.part_ml[row_of(k)];
        const float4 y = lane * 4 < COLS ? *reinterpret_cast<const float4*>(args.part_o + row_of(k) * D + c) : o;
        const float f = x.x == -INFINITY ? (x.y == 0.f ? 0.f : x.y) : ex2(x.x - top);  // (a NaN stays one)
        l += share(x, top);
        o.x += y.x * f, o.y += y.y * f, o.z += y.z * f, o.w += y.w * f;
      }
      if (split) {
        __syncthreads();
        meet[warp][lane] = o;
        if (lane == 0) meet_l[warp] = l;
        __syncthreads();
        if (warp != 0) continue;
#pragma unroll
        for (int w = 1; w < kJoinWarps; ++w) {
          const float4 y = meet[w][lane];
          o.x += y.x, o.y += y.y, o.z += y.z, o.w += y.w;
          l += meet_l[w];
        }
      }
      if (lane * 4 >= COLS) continue;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int t = s.first + (r0 + r) / group, h = kv * group + (r0 + r) % group;
      uint2 b4;
      b4.x = pack2(o.x * inv, o.y * inv), b4.y = pack2(o.z * inv, o.w * inv);
      *reinterpret_cast<uint2*>(reinterpret_cast<bf16*>(a.o) + t * a.o_token + h * a.o_head + c) = b4;
      if (c == 0) a.lse[(int64_t)h * p.tokens + t] = l == 0.f ? -INFINITY : (top + log2f(l)) * kLn2;
    }
  } else {
    asm volatile("griddepcontrol.wait;" ::: "memory");
  }
}

template <int D, int NT>
void launch_rows(const PagedAttentionArgs& a, int most_rows, void* workspace, int sms, cudaStream_t stream) {
  using C = Cfg<D, NT>;
  RowsArgs args;
  args.a = a;
  args.pieces = 2 * sms;
  args.part_o = static_cast<float*>(workspace);
  args.part_ml = reinterpret_cast<float2*>(args.part_o + (int64_t)2 * args.pieces * C::ROWS * D);
  args.rows = C::ROWS;
  args.plog = 0;
  while ((1 << args.plog) < a.cache.page) ++args.plog;
  args.most_rows = most_rows;
  cudaFuncSetAttribute(paged_rows_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  paged_rows_kernel<D, NT><<<args.pieces, kThreads, C::SMEM, stream>>>(args);
  // one block a border between two pieces
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(args.pieces - 1);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaLaunchKernelEx(&cfg, paged_join_kernel<D>, (const RowsArgs)args);
}

// Which kernel takes which sequence: up to kFewRows rows this file's, more the tensor cores', whose time hardly depends on the rows. 9 to 16 rows a
// sequence, this kernel | that one, us (500 and 5000 tokens in the cache; every number of sequences from 1 to 64 was measured in powers of 2):
//   sequences             1                  4                  16                 64
//   dim 64 (2 heads)      13|19    15|28     13|19    17|28     16|19    25|56     19|29    47|133
//   dim 128 (3)           12|19    17|29     13|20    21|32     18|21    38|83     25|40    94|197
//   dim 256 (4)           15|21    21|31     17|21    36|52     23|25    76|83     46|57   217|298
//   dim 256 (16, window)  17|21    21|26     25|25    35|35     50|57    72|92    129|157  214|281
//   dim 512 (4)           17|23    33|37     21|24    66|80     39|37   236|193   116|101  830|717
// Up to dim 256 this kernel is never slower by more than 2%. At dim 512, where it goes through the keys twice, it is from 8 sequences on
// (8: 27|27 and 133|100); that is not told apart.
constexpr int kFewRows = 16;
// With this many rows a sequence on average, or few sequences, the tensor cores' kernel takes all of them: what single tokens among them cost it more
// is mostly less than two launches. That kernel for all | both, us:
//   rows on average                      13 to 27         34 to 66         100 to 160       250 to 410
//   8 sequences, dim 128                 27|44 (19)       25|41            31|42            31|43
//   32 sequences, dim 128                35|47 (16)       36|43            39|45            41|59
//   8 sequences, dim 256, window 1024    105|90  73|85    88|98 105|85     106|112 150|121  100|216
//   32 sequences, dim 256, window 1024   145|150 148|165  149|170 155|223  163|173 215|215  301|309
//   8 sequences, dim 512                 97|93 (31)       83|87            111|121 179|150  249|276
//   32 sequences, dim 512                218|157 (25)     252|219 (54)     291|290          333|396 (206)
// (two pairs: few long runs second. The rule loses most where one chunk of 300 stands beside seven single tokens at dim 256: 143|78.) A chunk of 40 and one or
// two single tokens: 23-36|35-53 up to dim 256 with at most 5000 tokens each; at dim 512 27|46 over 500, 113|119 over 5000, 365|347 over 30000. Three
// single tokens whose max_q is not said take that kernel too: 62|58 us at dim 512 over 5000 (46 with max_q 1, by this kernel alone), 202|163 (147)
// over 30000. With more than kFewRows query heads a key head `both` has nothing for this file's kernel: 33 against 27 us (31 heads, 32 sequences).
constexpr int kMeanRows = 32, kFewSequences = 4;

enum Which { kRowsOnly, kTilesOnly, kBoth };
Which which(const PagedAttentionArgs& a) {
  const int64_t group = a.q_heads / a.cache.heads;
  if (a.max_q * group <= kFewRows) return kRowsOnly;
  return a.batch.seqs < kFewSequences || a.batch.tokens * group >= (int64_t)kMeanRows * a.batch.seqs ? kTilesOnly : kBoth;
}

// Sets of 8 rows a unit (see Cfg).
int sets_of(const PagedAttentionArgs& a) { return a.cache.dim <= 256 && (int64_t)a.max_q * (a.q_heads / a.cache.heads) > 8 ? 2 : 1; }

}  // namespace

int64_t paged_attention_workspace(const PagedAttentionArgs& a, int sms) {
  const int64_t rows = (int64_t)2 * 2 * sms * 8 * sets_of(a) * (a.cache.dim + 2) * 4;
  const Which w = which(a);
  return w == kRowsOnly ? rows : w == kTilesOnly ? paged_tiles_workspace(a) : std::max(rows, paged_tiles_workspace(a));
}

const char* launch_paged_attention(const PagedAttentionArgs& a, void* workspace, int sms, cudaStream_t stream) {
  const Which w = which(a);
  if (w != kTilesOnly) {
    const int most = w == kRowsOnly ? INT32_MAX : kFewRows;
    const bool two = sets_of(a) == 2;
    switch (a.cache.dim) {
      case 64: two ? launch_rows<64, 2>(a, most, workspace, sms, stream) : launch_rows<64, 1>(a, most, workspace, sms, stream); break;
      case 128: two ? launch_rows<128, 2>(a, most, workspace, sms, stream) : launch_rows<128, 1>(a, most, workspace, sms, stream); break;
      case 256: two ? launch_rows<256, 2>(a, most, workspace, sms, stream) : launch_rows<256, 1>(a, most, workspace, sms, stream); break;
      default: launch_rows<512, 1>(a, most, workspace, sms, stream);
    }
  }
  return w == kRowsOnly ? nullptr : launch_paged_tiles(a, w == kBoth ? kFewRows : 0, workspace, stream);
}

}  // namespace me

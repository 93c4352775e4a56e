// Attention of chunks of new tokens over a paged cache, on the tensor cores.
//
// Many rows a key head: S = Q K^T and O += P V are bound by the tensor cores, and next by the L2 cache, out of which every tile of
// rows reads its sequence's keys and values again. So two SMs work as one (cta_group::2): 256 rows (new token, query head of the
// key head's group) a pair, 128 of them in each SM's tensor memory, and each SM loads half of every block of 128 keys, which halves what
// both read. Per SM and block at dim 256: 64 KB of keys and values for 2048 clocks of the tensor core.
//
//   warps 0, 2 loads: rows of Q once a unit, and K; V (TMA, each through a ring of its own; a page is a run of rows of the tensor
//              map, a page that is none is an index past its last dimension, which reads zeros)
//   warp 1     issues the products (from the even SM): S of block j + 1 goes ahead of P V of block j, so that block j's
//              softmax has the time of two products
//   warp 3     finds the pair's next unit while the others are at work, two ahead
//   warps 4-7  softmax, a thread a row: 128 scores from tensor memory, running
//              maximum (O is rescaled only when it grows by more than 2^8), P rounded to bf16 (as what it is multiplied with is) and put
//              back over its scores, from where it is the A operand of P V; the sum is of the terms before that. At a unit's end:
//              O / sum to global memory. One warp a scheduler: what a block costs beside its exponentials is paid once, and nothing is
//              exchanged (two and four threads a row were slower)
//
// Tensor memory: O in columns 0-255, two S (P) buffers of 128. dim 512 has no room for both halves of O: a unit takes one half of the
// columns, and S is computed twice (3/2 of the operations).
// Rows of V that no row of the sequence may see (past its end, before its first window) can hold anything, and 0 * NaN is not 0: in blocks that have
// such rows the softmax threads wait for V themselves and put zeros there.
//
// Units (sequence, tile of rows, key head, half of the columns) are dealt to the pairs in turn, the longest of a sequence first. With few of them a
// sequence's keys are cut into chunks, whose (max, sum, O) a second kernel joins.
// Every wait is bounded: 2 s, 60 s where a whole unit may lie in between (one over 2^31 keys takes up to 40 s; a block that gives up ends these
// at once). Where one runs out the block gives up, frees tensor memory, counts itself in g_waits and returns.
//
// Measured: 2048 new tokens over 16048, 32 query heads on 4 of dim 512: 2.29 ms, 880 TFLOP/s of what has to be computed (0.53 of the measured
// bf16 rate; the tensor cores are 78% busy, a third of it with S a second time). 4096 new tokens under a window of 1024, 32 heads on 16 of dim 256: 198 us,
// 693 TFLOP/s (0.42; 182 us where calls on two caches take turns): a block takes 2950 clocks, of them the softmax 2450 (128 exponentials a thread
// at 8 clocks a warp's, two readings of the scores, the arrival), the rest the way of P to the products and of the next S back (two S buffers cover one of both); a unit of
// 10 blocks has 7000 clocks between its last softmax and the next unit's first (its last product 1800, O out 4700).
#include <cudaTypedefs.h>

#include <algorithm>
#include <mutex>
#include <type_traits>
#include <unordered_map>

#include "paged.cuh"
#include "tc_common.cuh"

namespace me {
namespace {
using namespace paged;
using namespace tc;

constexpr int kSoftWarps = 4, kFirstSoft = 4, kThreads = (kFirstSoft + kSoftWarps) * 32;
constexpr int BM = 128, BN = 128;     // rows an SM, keys a block
constexpr int kLeastBlocks = 8;       // of a chunk: below, its O costs more to write and join than its keys
constexpr int kDeals = 4;             // units a pair that cutting aims at
constexpr uint64_t kUnitLimit = 60000000000ull;

// QR: rows of Q an SM. 64 of them serve calls whose chunks are short (drafts): the product's other 64 rows are then what lies behind,
// and nobody looks at them; what Q leaves goes to the rings, which such calls need most, for they wait for memory.
template <int D, int QR>
struct Cfg {
  static constexpr int ROWS = QR;
  static constexpr int DV = D < 256 ? D : 256;       // columns of O a unit
  static constexpr int HALVES = D / DV;
  static constexpr int NV = D == 64 ? 128 : DV;      // columns of the P V product (dim 64: the odd SM's half is past the row, zeros)
  static constexpr int VC = NV / 2;                  // of them in this SM
  static constexpr int Q_BYTES = QR * D * 2;
  // a stage of K: this SM's 64 keys of a block x KC columns; of V: 128 keys x VC, one set of 64 keys after the other. (Stages of 16 KB, twice
  // as many: 10% slower, for a stage costs its loader and the products' warp some hundred clocks.)
  static constexpr int KC = D < 256 ? D : 256, K_STAGES = D / KC;
  static constexpr int K_BYTES = 64 * KC * 2, V_BYTES = BN * VC * 2;
  static constexpr int KR = D == 512 ? (QR == 64 ? 3 : 2) : D == 256 ? (QR == 64 ? 4 : 3) : 6;
  static constexpr int VR = D == 512 ? (QR == 64 ? 2 : 1) : D == 256 ? 2 : 6;  // stages
  static constexpr int K_OFF = Q_BYTES, V_OFF = K_OFF + KR * K_BYTES, BAR_OFF = V_OFF + VR * V_BYTES;
  static constexpr int SMEM = BAR_OFF + 640;
  static_assert(SMEM <= 232448, "shared memory");
  static_assert((2 * KR + 3 * VR + 15) * 8 <= 496, "barriers");
};
constexpr int kO = 0, kS = 256;  // columns of tensor memory

struct TilesArgs {
  PagedAttentionArgs a;
  float4* part_o;   // [slots][DV / 4][slot_rows]: a warp's rows lie together
  float2* part_ml;  // [slots][slot_rows]
  int slot_rows;    // a sequence with more rows is not cut, unless 256
  int group, tokens;  // query heads a key head, new tokens an SM
  int pairs;
  int plog;
  int least_rows;   // sequences with up to this many rows are others' work
};
// Blocks in which a wait ran out since the process began, and where the last of them waited: a device's own words, not an allocation that a captured
// graph could own. Nobody sets them back, so that every caller sees what ran out between two looks of its own.
__device__ int g_waits[2];
ME_DEVICE void count_wait(int where) {
  atomicAdd(&g_waits[0], 1);
  g_waits[1] = where;
}

// ------------------------------------------------------------------------------- units of work
struct UnitsOf {
  int tiles, chunks, per;  // tiles of rows, chunks of keys, blocks of a chunk
  int first, blocks;       // the sequence's blocks of keys
};
template <int D, int QR>
ME_DEVICE UnitsOf units_of(const TilesArgs& t, int b, const Sequence& s, int cut) {
  const PagedAttentionArgs& a = t.a;
  const int group = t.group, tokens = 2 * t.tokens;
  if (s.count == 0 || (int64_t)s.count * group <= t.least_rows) return {0, 1, 0, 0, 0};
  const Keys k = keys_of(a.batch, a.cache.page, s, 0, s.count - 1, a.window);
  UnitsOf u;
  u.tiles = (s.count + tokens - 1) / tokens;
  u.first = k.lo / BN;
  u.blocks = max((k.hi + BN - 1) / BN - u.first, 1);
  const bool whole = cut <= 0 || (t.slot_rows < 2 * QR && (int64_t)s.count * group > t.slot_rows);
  u.chunks = whole ? 1 : (u.blocks + cut - 1) / cut;
  u.per = (u.blocks + u.chunks - 1) / u.chunks;
  return u;
}

// Blocks a chunk, 0: no cutting. By a whole warp. Uncut, the last pair is done about after the mean of the blocks and, where units
// differ, most of the longest one; cut to about kDeals units a pair, after 1.15 times the mean and what four blocks take for the parts.
// At most 2 kDeals units a pair come of it: as many as there were (fewer than kDeals) and one for every `cut` blocks.
template <int D, int QR>
ME_DEVICE int cut_of(const TilesArgs& t) {
  const PagedBatch& p = t.a.batch;
  int64_t units = 0, blocks = 0;
  int most = 0;
#pragma unroll 4
  for (int b = threadIdx.x & 31; b < p.seqs; b += 32) {
    const UnitsOf u = units_of<D, QR>(t, b, sequence_of(p, b), 0);
    units += u.tiles, blocks += (int64_t)u.tiles * u.blocks;
    most = max(most, u.blocks);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    units += __shfl_xor_sync(0xffffffffu, units, o);
    blocks += __shfl_xor_sync(0xffffffffu, blocks, o);
  }
  most = __reduce_max_sync(0xffffffffu, most);
  const int each = t.a.cache.heads * Cfg<D, QR>::HALVES, aim = kDeals * t.pairs;
  units *= each, blocks *= each;
  if (units == 0 || units >= aim) return 0;
  const float mean = (float)blocks / t.pairs;
  const float uncut = blocks == units * most ? (float)((int)(units + t.pairs - 1) / t.pairs * most) : mean + 0.75f * most;
  if (uncut <= 1.15f * mean + 4.f) return 0;
  return max((int)((blocks + aim - 1) / aim), kLeastBlocks);
}

struct Unit {
  Sequence s;
  int b, tile, kv, half;
  int kb0, kb1;  // its blocks of keys, kb1 <= kb0: none
  int chunk, chunks;
};

// A warp's way along the units: 32 sequences at a time, a lane each.
template <int D, int QR>
struct Walk {
  const TilesArgs& t;
  int cut, c = 0;
  int64_t base = 0, mine = 0, upto = 0, all = 0;

  ME_DEVICE Walk(const TilesArgs& args, int cut_blocks) : t(args), cut(cut_blocks) { scan(); }
  ME_DEVICE void scan() {
    const PagedBatch& p = t.a.batch;
    const int lane = threadIdx.x & 31, b = c + lane;
    mine = 0;
    if (b < p.seqs) {
      const UnitsOf u = units_of<D, QR>(t, b, sequence_of(p, b), cut);
      mine = (int64_t)u.tiles * u.chunks * t.a.cache.heads * Cfg<D, QR>::HALVES;
    }
    upto = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += x;
    }
    all = __shfl_sync(0xffffffffu, upto, 31);
  }
  // Unit x (not below an earlier one's); false: there is none.
  ME_DEVICE bool at(int64_t x, Unit& out) {
    while (x >= base + all) {
      base += all;
      c += 32;
      if (c >= t.a.batch.seqs) return false;
      scan();
    }
    const uint32_t here = __ballot_sync(0xffffffffu, x - base < upto);
    const int src = __ffs(here) - 1;
    const int64_t before = base + __shfl_sync(0xffffffffu, upto - mine, src);
    const PagedAttentionArgs& a = t.a;
    out.b = c + src;
    out.s = sequence_of(a.batch, out.b);
    const UnitsOf u = units_of<D, QR>(t, out.b, out.s, cut);
    unsigned i = (unsigned)(x - before);  // (a sequence's units: the host checks that they fit)
    out.half = i % Cfg<D, QR>::HALVES, i /= Cfg<D, QR>::HALVES;
    out.kv = i % a.cache.heads, i /= a.cache.heads;
    out.chunk = i % u.chunks, out.chunks = u.chunks, i /= u.chunks;
    out.tile = u.tiles - 1 - (int)i;  // the last rows see the most keys
    const int tokens = 2 * t.tokens;
    const int i0 = out.tile * tokens, i1 = min(i0 + tokens, out.s.count) - 1;
    const Keys k = keys_of(a.batch, a.cache.page, out.s, i0, i1, a.window);
    out.kb0 = max(k.lo / BN, u.first + out.chunk * u.per);
    out.kb1 = min(k.hi <= k.lo ? 0 : (k.hi + BN - 1) / BN, u.first + (out.chunk + 1) * u.per);
    return true;
  }
};

// ------------------------------------------------------------------------------- instructions
// A load by the lanes of `issue`, into this SM's shared memory; `bar_cluster` may be the other's.
ME_DEVICE void tma_load_3d_pair_if(uint32_t dst, const CUtensorMap* map, uint32_t bar_cluster, int x, int y, int z, uint32_t issue) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %6, 0;\n\t"
      "@q cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];\n\t}" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster), "r"(x), "r"(y), "r"(z), "r"(issue)
      : "memory");
}
ME_DEVICE void tma_load_4d_pair_if(uint32_t dst, const CUtensorMap* map, uint32_t bar_cluster, int x, int y, int z, int w, uint32_t issue) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %7, 0;\n\t"
      "@q cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];\n\t}" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar_cluster), "r"(x), "r"(y), "r"(z), "r"(w), "r"(issue)
      : "memory");
}
// The pair's product and its commits, by the lanes of `issue` (one lane of the warp that goes along). Descriptors in halves: steps change the
// low one alone.
ME_DEVICE void umma_bf16_pair_if(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc, uint32_t accumulate, uint32_t issue) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "setp.ne.b32 q, %6, 0;\n\t"
      "@q tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %4, p;\n\t}" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate), "r"(issue));
}
// A (P) from tensor memory.
ME_DEVICE void umma_bf16_pair_ts_if(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t accumulate, uint32_t issue) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %3};\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "setp.ne.b32 q, %6, 0;\n\t"
      "@q tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], b, %4, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(accumulate), "r"(issue));
}
ME_DEVICE void umma_commit_pair_if(uint64_t* bar, uint32_t issue, uint16_t mask = 0x3) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %2, 0;\n\t"
      "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(smem_addr(bar)),
      "h"(mask), "r"(issue)
      : "memory");
}
// 32 columns of this warp's lanes, not yet there until tmem_wait_ld().
ME_DEVICE void tmem_issue_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
// The loads' results pass through here, so that no use of them moves ahead of the wait.
ME_DEVICE void tmem_wait_ld(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                 "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                 "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}
ME_DEVICE void tmem_issue_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
ME_DEVICE void tmem_wait_ld(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
ME_DEVICE void tmem_st16u(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
               "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
               "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
               : "memory");
}

ME_DEVICE void tmem_st32u(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
      "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]),
      "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]),
      "r"(v[31])
      : "memory");
}
// Arrive on a barrier of either SM of the pair. The release is this SM's alone: enough for what tensor memory holds, and without the
// wait for all earlier memory operations that one at cluster scope costs (1000 clocks a block).
ME_DEVICE void mbar_arrive_cta(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cta.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
ME_DEVICE void st_global32(void* p, const uint32_t* v) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
               "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// ------------------------------------------------------------------------------- the kernel
template <int D, int QR>
__global__ void __launch_bounds__(kThreads, 1)
    paged_tiles_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                       const __grid_constant__ TilesArgs args) {
  using C = Cfg<D, QR>;
  constexpr int KR = C::KR, VR = C::VR;
  extern __shared__ __align__(1024) uint8_t smem[];  // (no room to align it here: there is no other shared memory)
  uint8_t *sQ = smem, *sK = smem + C::K_OFF, *sV = smem + C::V_OFF;
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + C::BAR_OFF);  // [KR], the even SM's counts for both
  uint64_t* k_empty = k_full + KR;
  uint64_t* v_full = k_empty + KR;   // [VR], the even SM's
  uint64_t* v_empty = v_full + VR;
  uint64_t* v_here = v_empty + VR;   // [VR] V of a block whose rows are put right here
  uint64_t* q_full = v_here + VR;    // the even SM's
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;    // [2]
  uint64_t* p_full = s_full + 2;     // [2], the even SM's: the softmax warps of both
  uint64_t* pv_done = p_full + 2;    // [2]
  uint64_t* o_full = pv_done + 2;    // once a unit
  uint64_t* o_free = o_full + 1;     // the even SM's
  uint64_t* all_done = o_free + 1;
  uint64_t* next_full = all_done + 1;   // [2]
  uint64_t* next_empty = next_full + 2; // [2]
  int* next_unit = reinterpret_cast<int*>(smem + C::BAR_OFF + 496);  // [2][16]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::BAR_OFF + 624);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const PagedAttentionArgs& a = args.a;
  const PagedBatch& p = a.batch;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1;
  const int group = args.group, tokens = args.tokens;
  int* status = reinterpret_cast<int*>(smem + C::BAR_OFF + 632);  // what went wrong first in this block, and where
  if (smem_addr(smem) & 1023) {
    if (threadIdx.x == 0) count_wait(76);
    return;
  }

  if (threadIdx.x == 0) {
    for (int i = 0; i < KR; ++i) mbar_init(&k_full[i], 1), mbar_init(&k_empty[i], 1);
    for (int i = 0; i < VR; ++i) mbar_init(&v_full[i], 1), mbar_init(&v_empty[i], 1), mbar_init(&v_here[i], 1);
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < 2; ++i) mbar_init(&s_full[i], 1), mbar_init(&p_full[i], 2 * kSoftWarps), mbar_init(&pv_done[i], 1);
    mbar_init(o_full, 1);
    mbar_init(o_free, 2 * kSoftWarps);
    mbar_init(all_done, 1);
    for (int i = 0; i < 2; ++i) mbar_init(&next_full[i], 1), mbar_init(&next_empty[i], 2 + kSoftWarps + (leader ? 1 : 0));
    *abort = 0;
    status[0] = status[1] = 0;
    fence_barrier_init();
    prefetch_tmap(&tq);
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, 512);
  if (args.least_rows == 0) clear_rest<D>(a, kThreads);  // (else the kernel of few rows does)
  tc_fence_before();
  cluster_sync();
  tc_fence_after();
  constexpr uint32_t tmem = 0;  // all columns are this kernel's, so they begin at 0 (and addresses need no register)
  if (*tmem_slot != tmem) {
    if (threadIdx.x == 0) report(status, ME_ERR_ALIGN, 77), *abort = 1;
  }
  __syncthreads();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // The `it`-th unit of the pair, by warp 3; false: there is none, or a wait ran out. Whole warps; the numbers are the same in all lanes, and
  // pass a reduction so that they are known to be, and addresses and descriptors that come of them stay in uniform registers.
  auto uniform = [](int x) { return (int)__reduce_or_sync(0xffffffffu, (unsigned)x); };
  auto wait_u = [&](uint64_t* bar, int parity, int where, uint64_t limit_ns = 2000000000ull) {
    return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) || __all_sync(0xffffffffu, mbar_wait(bar, parity, status, where, abort, limit_ns));
  };
  Unit u;
  Keys seq;
  int unit_x = 0;
  bool whole = true;  // every page of the unit's keys is one
  auto take_unit = [&](int it, int where) {
    if (!wait_u(&next_full[it & 1], (it >> 1) & 1, where, kUnitLimit)) return false;
    const int mine = next_unit[(it & 1) * 16 + (lane & 15)];
    __syncwarp();
    if (lane == 0) mbar_arrive(&next_empty[it & 1]);
    auto field = [&](int i) { return uniform(__shfl_sync(0xffffffffu, mine, i)); };
    u.s = {field(1), field(2), field(3)};
    u.b = field(4), u.tile = field(5), u.kv = field(6), u.half = field(7);
    u.kb0 = field(8), u.kb1 = field(9), u.chunk = field(10), u.chunks = field(11);
    seq = {field(12), field(13)};
    unit_x = field(14), whole = field(15);
    return field(0) != 0;
  };

  // In a block with rows of V that may hold anything, V arrives at v_here and the softmax threads put zeros there.
  auto has_stale = [&](const Keys& seq, int kb) { return kb * BN < seq.lo || (kb + 1) * BN > seq.hi; };

  if (warp == 0 || warp == 2) {
    // ---------------------------------------------------------------- loads
    // (the whole warp goes along and its lane 0 issues, as for the products)
    const bool of_k = warp == 0;
    uint64_t *full = of_k ? k_full : v_full, *empty = of_k ? k_empty : v_empty;
    const int ring = of_k ? KR : VR;
    const uint32_t full_leader = mapa_shared(smem_addr(full), 0), q_leader = mapa_shared(smem_addr(q_full), 0);
    const uint32_t v_here_own = mapa_shared(smem_addr(v_here), rank), aQ = smem_addr(sQ), aK = smem_addr(sK), aV = smem_addr(sV);
    // rows of a load; pages of 64 and more: all columns of a stage at once
    const int box = min(a.cache.page, 64), page_mask = a.cache.page - 1;
    const uint32_t one = lane == 0;
    int st = 0, round = 0, g = 0;   // the ring's next stage; stages so far
    int live = 0;
    bool ok = true;
    auto free_stage = [&] {
      if (round > 0) ok = wait_u(&empty[st], (round - 1) & 1, of_k ? 50 : 53);
    };
    auto next_stage = [&] {
      ++g;
      if (++st == ring) st = 0, ++round;
    };
    for (int it = 0; ok && take_unit(it, of_k ? 54 : 55); ++it) {
      const int n = u.kb1 - u.kb0;
      if (n <= 0) continue;
      const int y0 = u.kv << args.plog;
      // The table's entries for four blocks, a lane for each 16 keys: read four blocks ahead and looked at when they are needed (a look at
      // once would wait for memory in every block, which held most SMs at 5000 to 6000 clocks a block). Runs of `box` keys that no new token sees
      // are none: their pages may be another's by now.
      auto pages_of = [&](int kb) {
        const int key = kb * BN + lane * 16, run = key & ~(box - 1);
        return run + box > seq.lo && run < seq.hi ? p.table[u.b * p.table_stride + (key >> args.plog)] : -1;  // (seq.hi is within the table's row)
      };
      // 64 keys from `in` of block kb, NC x 64 columns from chunk x on
      auto load64 = [&](uint32_t dst, const CUtensorMap* map, uint32_t bar, int kb, int in, int ids, int x, auto NC) {
        if (box == 64) {
          const int id = __shfl_sync(0xffffffffu, ids, (kb - u.kb0) % 4 * 8 + in / 16);
          tma_load_4d_pair_if(dst, map, bar, 0, y0 + ((kb * BN + in) & page_mask), x, id, one);
        } else {
          // small pages: their numbers first, so that the loads go out one after the other
          const int at = (kb - u.kb0) % 4 * 8 + in / 16, y = y0 + ((kb * BN + in) & page_mask);
          int id[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) id[i] = __shfl_sync(0xffffffffu, ids, at + i);
          if (box == 32) {
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int c = 0; c < decltype(NC)::value; ++c) tma_load_4d_pair_if(dst + c * (64 * 128) + i * (32 * 128), map, bar, 0, y, x + c, id[2 * i], one);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int c = 0; c < decltype(NC)::value; ++c) tma_load_4d_pair_if(dst + c * (64 * 128) + i * (16 * 128), map, bar, 0, y, x + c, id[i], one);
          }
        }
      };
      int raw = pages_of(u.kb0), ids = 0;
      for (int j = 0; j < n && ok; ++j) {
        const int kb = u.kb0 + j;
        if ((j & 3) == 0) {
          ids = raw >= 0 && raw < a.cache.pages ? raw : a.cache.pages;  // none: an index past the cache
          if (j + 4 < n) raw = pages_of(kb + 4);
        }
        if (of_k) {
#pragma unroll
          for (int c = 0; c < C::K_STAGES; ++c) {
            free_stage();
            if (!ok) break;
            if (leader && one) mbar_expect_tx(&full[st], 2 * C::K_BYTES);
            __syncwarp();
            load64(aK + st * C::K_BYTES, &tk, full_leader + st * 8, kb, (int)rank * 64, ids, c * (C::KC / 64), std::integral_constant<int, C::KC / 64>());
            next_stage();
          }
          if (j == 0 && ok) {  // Q, once the unit before is done with it
            if (live > 0) ok = wait_u(q_empty, (live - 1) & 1, 51);
            if (!ok) break;
            if (leader && one) mbar_expect_tx(q_full, 2 * (D / 64) * tokens * group * 128);
            __syncwarp();
#pragma unroll
            for (int c = 0; c < D / 64; ++c)
              tma_load_3d_pair_if(aQ + c * (C::ROWS * 128), &tq, q_leader, c * 64, u.kv * group, u.s.first + u.tile * 2 * tokens + (int)rank * tokens, one);
          }
        } else {
          const bool stale = has_stale(seq, kb);
          free_stage();
          if (!ok) break;
          if (one) {
            if (stale) mbar_expect_tx(&v_here[st], C::V_BYTES);
            if (leader && stale) mbar_arrive(&full[st]);
            if (leader && !stale) mbar_expect_tx(&full[st], 2 * C::V_BYTES);
          }
          __syncwarp();
#pragma unroll
          for (int c = 0; c < 2; ++c)
            load64(aV + st * C::V_BYTES + c * (C::V_BYTES / 2), &tv, stale ? v_here_own + st * 8 : full_leader + st * 8, kb, c * 64, ids,
                   (u.half * C::DV + (int)rank * C::VC) / 64, std::integral_constant<int, C::VC / 64>());
          next_stage();
        }
      }
      ++live;
    }
    // Every stage this SM filled is given back by the products that read it: then no copy is in flight.
    for (int i = max(0, g - ring); i < g; ++i) {
      if (*abort && !leader) break;
      mbar_wait(&empty[i % ring], (i / ring) & 1, status, 52, abort, 500000000ull);
    }
  } else if (warp == 1) {
    // ---------------------------------------------------------------- products
    // The whole warp goes along, so that descriptors stay in uniform registers; its lane 0 issues. (With lane 0 alone in here an
    // issue took 110 to 180 clocks, more than the product.)
    if (leader) {
      const uint32_t id_s = idesc_bf16(2 * BM, BN), id_o = idesc_bf16(2 * BM, C::NV, true);
      const uint32_t dQ = (uint32_t)desc_sw128(smem_addr(sQ)), dK = (uint32_t)desc_sw128(smem_addr(sK)), hi = (uint32_t)(desc_sw128(0) >> 32);
      const uint32_t dV = (uint32_t)desc_mn_sw128(smem_addr(sV), 64 * 128, 1024), hV = (uint32_t)(desc_mn_sw128(0, 64 * 128, 1024) >> 32);
      const uint32_t one = lane == 0;
      int kst = 0, kphase = 0, vst = 0, vphase = 0;  // the rings' next stages
      int gb = 0, live = 0;    // blocks, units so far
      bool ok = true;
      auto wait = [&](uint64_t* bar, int parity, int where) { ok = wait_u(bar, parity, where); };
      for (int it = 0; ok && take_unit(it, 66); ++it) {
        const int n = u.kb1 - u.kb0;
        if (n <= 0) continue;
        wait(q_full, live & 1, 60);
        for (int j = 0; j <= n && ok; ++j) {
          if (j < n) {
            const uint32_t to = kS + ((gb + j) & 1) * BN;
#pragma unroll 1
            for (int c = 0; c < C::K_STAGES; ++c) {
              wait(&k_full[kst], kphase, 63);
              if (!ok) break;
              tc_fence_after();
              const uint32_t dk = dK + (kst * C::K_BYTES >> 4), dq = dQ + (c * (C::KC / 64) * (C::ROWS * 128) >> 4);
#pragma unroll
              for (int k4 = 0; k4 < C::KC / 64; ++k4)
#pragma unroll
                for (int kk = 0; kk < 4; ++kk)
                  umma_bf16_pair_if(to, dq + ((k4 * (C::ROWS * 128) + kk * 32) >> 4), dk + ((k4 * (64 * 128) + kk * 32) >> 4), hi, id_s, (c | k4 | kk) != 0, one);
              umma_commit_pair_if(&k_empty[kst], one);
              if (++kst == KR) kst = 0, kphase ^= 1;
            }
            if (!ok) break;
            umma_commit_pair_if(&s_full[(gb + j) & 1], one);
            if (j == n - 1) umma_commit_pair_if(q_empty, one);
          }
          if (j > 0) {
            const int i = gb + j - 1;  // block of all
            if (j == 1 && live > 0) wait(o_free, (live - 1) & 1, 64);
            if (!ok) break;
            if (has_stale(seq, u.kb0 + j - 1))  // the other SM's shared memory was written
              ok = __all_sync(0xffffffffu, mbar_wait_cluster(&p_full[i & 1], (i >> 1) & 1, status, 61, abort));
            else if (ok)
              wait(&p_full[i & 1], (i >> 1) & 1, 61);
            if (!ok) break;
            wait(&v_full[vst], vphase, 62);
            if (!ok) break;
            tc_fence_after();
            const uint32_t dv = dV + (vst * C::V_BYTES >> 4), from_p = kS + (i & 1) * BN;
#pragma unroll
            for (int kk = 0; kk < BN / 16; ++kk)
              umma_bf16_pair_ts_if(kO, from_p + kk * 8, dv + (((kk / 4) * (C::V_BYTES / 2) + (kk & 3) * 2048) >> 4), hV, id_o, (j > 1 || kk > 0), one);
            umma_commit_pair_if(&v_empty[vst], one);
            if (++vst == VR) vst = 0, vphase ^= 1;
            if (!ok) break;
            umma_commit_pair_if(&pv_done[i & 1], one);
            if (j == n) umma_commit_pair_if(o_full, one);
          }
        }
        gb += n;
        ++live;
      }
      // every product has ended before tensor memory is freed
      umma_commit_pair_if(all_done, one, 0x1);
      if (one) mbar_wait(all_done, 0, status, 65, nullptr, 500000000ull);
      __syncwarp();
    }
  } else if (warp == 3) {
    // ---------------------------------------------------------------- units
    Walk<D, QR> walk(args, cut_of<D, QR>(args));
    Unit w = {};
    bool more = true;
    for (int it = 0; more; ++it) {
      const int64_t x = pair + (int64_t)it * args.pairs;
      more = __all_sync(0xffffffffu, walk.at(x, w));
      const Keys k = keys_of(p, a.cache.page, w.s, 0, w.s.count - 1, a.window);
      bool all = true;
      for (int kb = w.kb0 + lane / 8; more && kb < w.kb1; kb += 4) {  // a lane for 16 keys
        const int key = kb * BN + lane % 8 * 16;
        if (key + 15 >= k.lo && key < k.hi) all = all && page_at(p, a.cache.pages, w.b, key >> args.plog) >= 0;
      }
      all = __all_sync(0xffffffffu, all);
      if (it >= 2 && !wait_u(&next_empty[it & 1], ((it >> 1) - 1) & 1, 80, kUnitLimit)) break;
      int* to = next_unit + (it & 1) * 16;
      if (lane == 0) {
        to[0] = more, to[1] = w.s.first, to[2] = w.s.count, to[3] = w.s.context, to[4] = w.b, to[5] = w.tile, to[6] = w.kv, to[7] = w.half;
        to[8] = w.kb0, to[9] = w.kb1, to[10] = w.chunk, to[11] = w.chunks, to[12] = k.lo, to[13] = k.hi, to[14] = (int)x, to[15] = all;
        mbar_arrive(&next_full[it & 1]);
      }
      __syncwarp();
    }
  } else if (warp >= kFirstSoft) {
    // ---------------------------------------------------------------- softmax
    const int quarter = warp & 3, r = quarter * 32 + lane;  // row of the SM
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t p_leader = mapa_shared(smem_addr(p_full), 0), o_leader = mapa_shared(smem_addr(o_free), 0);
    const float to_log2 = a.scale * kLog2e;
    const int ti = r / group, head = r % group;
    // 32-byte stores of O where its rows allow them
    const bool wide = reinterpret_cast<uintptr_t>(a.o) % 32 == 0 && a.o_token % 16 == 0 && a.o_head % 16 == 0;
    int gb = 0, live = 0;   // blocks, units with any so far
    uint32_t v_phases = 0;  // bit i: parity of v_here[i]
    bool ok = true;
    for (int it = 0; ok && take_unit(it, 77); ++it) {
      const int n = max(u.kb1 - u.kb0, 0);
      const int token = u.tile * 2 * tokens + (int)rank * tokens + ti;  // of the sequence's new ones
      const bool mine = ti < tokens && token < u.s.count, any_mine = __any_sync(0xffffffffu, mine);
      const int last = mine ? min(u.s.context + token, seq.hi - 1) : -1;
      const int from = a.window > 0 ? max(u.s.context + token, 0) - a.window + 1 : 0;
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < n; ++j) {
        const int i = gb + j, kb = u.kb0 + j, key0 = kb * BN;
        const uint32_t at = lanes + kS + (i & 1) * BN;
        const bool stale = has_stale(seq, kb);
        float alpha = 1.f;
        if (!(ok = wait_u(&s_full[i & 1], (i >> 1) & 1, 70))) break;
        tc_fence_after();
        if (any_mine) {  // (rows of nothing: P may be what it is)
          uint32_t pages = 0xff;
          if (!whole) {
            const int key = key0 + (lane & 7) * 16;
            pages = __ballot_sync(0xffffffffu, lane < 8 && key + 15 >= seq.lo && key < seq.hi && page_at(p, a.cache.pages, u.b, key >> args.plog) >= 0);
          }
          const bool open = __all_sync(0xffffffffu, pages == 0xffu && ((key0 >= from && key0 + BN - 1 <= last) || !mine));
          auto scores = [&](int c, uint32_t(&s)[2][32]) {  // 64 of them from column c on
            tmem_issue_ld32(at + c, s[0]);
            tmem_issue_ld32(at + c + 32, s[1]);
            tmem_wait_ld(s[0]);
            tmem_wait_ld(s[1]);
          };
          // (Rolled loops: with 128 scores unrolled the roles' code together does not fit the instruction caches, and the SMs of a
          // full GPC took 4000 to 5000 clocks for what takes 1400.)
          float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll 1
          for (int c = 0; c < BN; c += 64) {
            uint32_t s[2][32];
            scores(c, s);
            if (!open) {  // -inf where the row does not see the key, put back for the second reading (masking twice: 500 clocks a block)
              // bits from .. last of these keys that have a page
              const int lo = min(max(from - key0 - c, 0), 64), hi = min(max(last + 1 - key0 - c, 0), 64);
              const uint64_t seen = (hi == 64 ? ~0ull : (1ull << hi) - 1) & ~(lo == 64 ? ~0ull : (1ull << lo) - 1);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const uint32_t two = pages >> (c / 16 + 2 * h);
                const uint32_t bits = (uint32_t)(seen >> (32 * h)) & ((two & 1 ? 0xffffu : 0u) | (two & 2 ? 0xffff0000u : 0u));
#pragma unroll
                for (int e = 0; e < 32; ++e)
                  if (!(bits & (1u << e))) s[h][e] = 0xff800000u;  // -inf
                tmem_st32u(at + c + 32 * h, s[h]);
              }
              tmem_st_wait();
            }
#pragma unroll
            for (int e = 0; e < 64; ++e) mx[e & 1] = fmaxf(mx[e & 1], __uint_as_float(s[e / 32][e % 32]));
          }
          const float top = fmaxf(mx[0], mx[1]) * to_log2;
          if (top > m + kSlack) {
            if (m != -INFINITY) alpha = ex2(m - top), l *= alpha;  // (before its first score a row's O is zero)
            m = top;
          }
          const float z = m == -INFINITY ? 0.f : m;
          float sum[2] = {0.f, 0.f};
#pragma unroll 1
          for (int c = 0; c < BN; c += 64) {
            uint32_t s[2][32], pk[32];
            scores(c, s);
#pragma unroll
            for (int e = 0; e < 64; e += 2) {
              const float p0 = ex2(fmaf(__uint_as_float(s[e / 32][e % 32]), to_log2, -z)), p1 = ex2(fmaf(__uint_as_float(s[e / 32][e % 32 + 1]), to_log2, -z));
              sum[0] += p0, sum[1] += p1;
              pk[e / 2] = pack2(p0, p1);
            }
            tmem_st32u(at + c / 2, pk);  // over scores of keys up to c + 63, which have been read
          }
          l += sum[0] + sum[1];
        }
        if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {  // O stands still once the product before has ended
          if (!(ok = wait_u(&pv_done[(i - 1) & 1], ((i - 1) >> 1) & 1, 71))) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < C::DV; c += 16) {
            uint32_t o[16];
            tmem_issue_ld16(lanes + kO + c, o);
            tmem_wait_ld(o);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st16u(lanes + kO + c, o);
          }
        }
        if (stale) {  // thread r: key r of the block, this SM's columns
          const int st = i % VR;
          if (!(ok = wait_u(&v_here[st], (v_phases >> st) & 1, 72))) break;
          v_phases ^= 1u << st;
          const int key = key0 + r;
          if (key < seq.lo || key >= seq.hi) {
#pragma unroll
            for (int c = 0; c < C::VC / 8; ++c)  // its 16-byte chunks; the warp's rows in different banks
              *reinterpret_cast<uint4*>(sV + st * C::V_BYTES + (r / 64) * (C::V_BYTES / 2) + (c / 8) * (64 * 128) + (r & 63) * 128 + ((c + r) & 7) * 16) =
                  make_uint4(0, 0, 0, 0);
          }
          fence_async_smem();
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          // P is in tensor memory, which the fences above order; what was written to shared memory has to be there for the other SM's eyes
          if (stale) mbar_arrive_cluster(p_leader + (i & 1) * 8);
          else mbar_arrive_cta(p_leader + (i & 1) * 8);
        }
      }
      // ---- the unit's end
      if (n > 0 && ok) ok = wait_u(o_full, live & 1, 73), ++live;
      if (!ok) break;
      tc_fence_after();
      const int t = u.s.first + token, h = u.kv * group + head;
      const int64_t slot = unit_x, row = (int64_t)(int)rank * tokens * group + r;
      auto release = [&] {  // O has been read: the next unit's products may go over it
        if (n == 0) return;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cta(o_leader);
      };
      if (!any_mine) {
        release();
      } else if (u.chunks > 1) {
        float4* dst = args.part_o + slot * (C::DV / 4) * args.slot_rows + row;
#pragma unroll 1
        for (int c = 0; c < C::DV; c += 32) {
          uint32_t o[32] = {};
          if (n > 0) {
            tmem_issue_ld32(lanes + kO + c, o);
            tmem_wait_ld(o);
          }
          if (c + 32 == C::DV) release();
          if (mine)
#pragma unroll
            for (int e = 0; e < 32; e += 4)
              dst[(int64_t)((c + e) / 4) * args.slot_rows] = make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]), __uint_as_float(o[e + 2]),
                                                                         __uint_as_float(o[e + 3]));
        }
        if (mine) args.part_ml[slot * args.slot_rows + row] = make_float2(m, l);
      } else {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        bf16* dst = reinterpret_cast<bf16*>(a.o) + t * a.o_token + h * a.o_head + u.half * C::DV;
#pragma unroll 1
        for (int c = 0; c < C::DV; c += 64) {
          uint32_t o[2][32] = {};
          if (n > 0) {
            tmem_issue_ld32(lanes + kO + c, o[0]);
            tmem_issue_ld32(lanes + kO + c + 32, o[1]);
            tmem_wait_ld(o[0]);
            tmem_wait_ld(o[1]);
          }
          if (c + 64 == C::DV) release();
          if (!mine) continue;
          uint32_t out[32];
#pragma unroll
          for (int e = 0; e < 64; e += 2) out[e / 2] = pack2(__uint_as_float(o[e / 32][e % 32]) * inv, __uint_as_float(o[e / 32][e % 32 + 1]) * inv);
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            if (wide) {
              st_global32(dst + c + e * 2, &out[e]);
            } else {
              *reinterpret_cast<uint4*>(dst + c + e * 2) = make_uint4(out[e], out[e + 1], out[e + 2], out[e + 3]);
              *reinterpret_cast<uint4*>(dst + c + e * 2 + 8) = make_uint4(out[e + 4], out[e + 5], out[e + 6], out[e + 7]);
            }
          }
        }
        if (mine) {
          if (u.half == 0) a.lse[(int64_t)h * p.tokens + t] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
        }
      }
      gb += n;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && status[0] != 0) count_wait(status[1]);
  __syncwarp();
  cluster_sync();  // both SMs are done with every product, copy and remote arrival
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// Joins the chunks of sequences that were cut: a block takes every gridDim.x-th (unit, 32 rows, 32 columns), its lanes a row and its warps 4
// columns each.
constexpr int kJoinThreads = 256;
template <int D, int QR>
__global__ void __launch_bounds__(kJoinThreads) paged_join_tiles_kernel(const __grid_constant__ TilesArgs args) {
  using C = Cfg<D, QR>;
  constexpr int SETS = C::DV / 32;
  const PagedAttentionArgs& a = args.a;
  const int steps = (args.slot_rows + 31) / 32, cut = cut_of<D, QR>(args);
  if (cut == 0) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  Walk<D, QR> walk(args, cut);
  Unit u;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = args.group, tokens = 2 * args.tokens;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  for (int i = blockIdx.x; walk.at(i / (steps * SETS), u); i += gridDim.x) {  // (units are few where any is cut)
    if (u.chunks == 1 || u.chunk != 0) continue;
    const int64_t x = i / (steps * SETS), stride = (int64_t)a.cache.heads * C::HALVES;  // between a tile's chunks
    const int set = i % SETS, i0 = u.tile * tokens, rows = min(tokens, u.s.count - i0) * group, r = i / SETS % steps * 32 + lane;
    if (r >= rows) continue;
    const float2* mls = args.part_ml + x * args.slot_rows + r;
    const int64_t ml_step = stride * args.slot_rows;
    float top = -INFINITY, l = 0.f;
#pragma unroll 8
    for (int k = 0; k < u.chunks; ++k) top = fmaxf(top, mls[k * ml_step].x);
    const int c = set * 8 + warp;  // of the columns, 4 at a time
    const float4* parts = args.part_o + (x * (C::DV / 4) + c) * args.slot_rows + r;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int k = 0; k < u.chunks; ++k) {
      const float2 ml = mls[k * ml_step];
      const float4 y = parts[k * ml_step * (C::DV / 4)];
      const float f = ml.x == -INFINITY ? (ml.y == 0.f ? 0.f : ml.y) : ex2(ml.x - top);  // (a NaN stays one)
      l += share(ml, top);
      o.x += y.x * f, o.y += y.y * f, o.z += y.z * f, o.w += y.w * f;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const int t = u.s.first + i0 + r / group, h = u.kv * group + r % group;
    uint2 b4;
    b4.x = pack2(o.x * inv, o.y * inv), b4.y = pack2(o.z * inv, o.w * inv);
    *reinterpret_cast<uint2*>(reinterpret_cast<bf16*>(a.o) + t * a.o_token + h * a.o_head + u.half * C::DV + c * 4) = b4;
    if (c == 0 && u.half == 0) a.lse[(int64_t)h * a.batch.tokens + t] = l == 0.f ? -INFINITY : (top + log2f(l)) * kLn2;
  }
}

// ------------------------------------------------------------------------------- host
PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = [] {
    cudaDriverEntryPointQueryResult q;
    void* f = nullptr;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess) f = nullptr;
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(f);
  }();
  return fn;
}

// bf16, a box of 64 elements of the first dimension, 128-byte swizzle. Strides in elements, of the dimensions from the second on.
template <int N>
bool make_map(CUtensorMap* map, const void* ptr, const int64_t (&dim)[N], const int64_t (&stride)[N - 1], const int (&box)[N - 1]) {
  cuuint64_t dims[N], strides[N - 1];
  cuuint32_t boxes[N] = {64}, one[N];
  for (int i = 0; i < N; ++i) dims[i] = dim[i], one[i] = 1;
  for (int i = 0; i + 1 < N; ++i) strides[i] = stride[i] * 2, boxes[i + 1] = box[i];
  return encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, N, const_cast<void*>(ptr), dims, strides, boxes, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int QR>
int resident_pairs() {
  static std::mutex mu;
  static std::unordered_map<int, int> known;
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lk(mu);
  auto it = known.find(dev);
  if (it != known.end()) return it->second;
  cudaFuncSetAttribute(paged_tiles_kernel<D, QR>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D, QR>::SMEM);
  int sms = 0, n = 0;
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 2, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.gridDim = dim3(sms & ~1);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Cfg<D, QR>::SMEM;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, paged_tiles_kernel<D, QR>, &cfg) != cudaSuccess || n <= 0) {
    (void)cudaGetLastError();
    n = sms / 2;
  }
  return known[dev] = n;
}

template <int D, int QR>
int slot_rows_of(const PagedAttentionArgs& a) {
  return (int)std::min<int64_t>(2 * QR, ((int64_t)a.max_q * (a.q_heads / a.cache.heads) + 7) / 8 * 8);
}
template <int D, int QR>
int64_t workspace(const PagedAttentionArgs& a) {
  return (int64_t)2 * kDeals * resident_pairs<D, QR>() * slot_rows_of<D, QR>(a) * (Cfg<D, QR>::DV + 2) * 4;
}

template <int D, int QR>
const char* launch(const PagedAttentionArgs& a, int least_rows, void* space, cudaStream_t stream) {
  using C = Cfg<D, QR>;
  if (encode_fn() == nullptr) return "cuTensorMapEncodeTiled is unavailable";
  TilesArgs args;
  args.a = a;
  args.pairs = resident_pairs<D, QR>();
  args.slot_rows = slot_rows_of<D, QR>(a);
  args.part_o = static_cast<float4*>(space);
  args.part_ml = reinterpret_cast<float2*>(args.part_o + (int64_t)2 * kDeals * args.pairs * args.slot_rows * (C::DV / 4));
  args.group = a.q_heads / a.cache.heads, args.tokens = QR / args.group;
  args.plog = 0;
  while ((1 << args.plog) < a.cache.page) ++args.plog;
  args.least_rows = least_rows;
  bind_primary_context();
  const int box = std::min(a.cache.page, 64);
  const int64_t rows = (int64_t)a.cache.heads * a.cache.page;
  // pages as [page][64 columns of the head][head, position][column]
  const int64_t dims[4] = {64, rows, D / 64, a.cache.pages};
  CUtensorMap tq, tk, tv;
  if (!make_map<3>(&tq, a.q, {D, a.q_heads, a.batch.tokens}, {a.q_head, a.q_token}, {args.group, args.tokens}) ||
      !make_map<4>(&tk, a.cache.k, dims, {D, 64, a.cache.k_stride}, {box, box == 64 ? C::KC / 64 : 1, 1}) ||
      !make_map<4>(&tv, a.cache.v, dims, {D, 64, a.cache.v_stride}, {box, box == 64 ? C::VC / 64 : 1, 1}))
    return "cuTensorMapEncodeTiled failed";
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 2, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.gridDim = dim3(2 * args.pairs);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, paged_tiles_kernel<D, QR>, tq, tk, tv, args);
  if (e != cudaSuccess) return cudaGetErrorString(e);
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(8 * args.pairs);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.dynamicSmemBytes = 0;
  e = cudaLaunchKernelEx(&cfg, paged_join_tiles_kernel<D, QR>, args);
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace

cudaError_t paged_waits(int (&words)[2], cudaStream_t stream) {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;  // (another thread's capture goes on)
  cudaThreadExchangeStreamCaptureMode(&mode);
  cudaError_t e = cudaMemcpyFromSymbolAsync(words, g_waits, sizeof words, 0, cudaMemcpyDeviceToHost, stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  cudaThreadExchangeStreamCaptureMode(&mode);
  return e;
}

namespace {
// Short chunks: a tile of 64 rows an SM holds them all. (Sharper: with more than 64 query heads a key head a token has no room there.)
bool few(const PagedAttentionArgs& a) {
  const int group = a.q_heads / a.cache.heads;
  return group <= 64 && (int64_t)a.max_q * group <= 64;
}
template <class F>
auto by_shape(const PagedAttentionArgs& a, F f) {
  using std::integral_constant;
  auto rows = [&](auto dim) { return few(a) ? f(dim, integral_constant<int, 64>()) : f(dim, integral_constant<int, 128>()); };
  switch (a.cache.dim) {
    case 64: return rows(integral_constant<int, 64>());
    case 128: return rows(integral_constant<int, 128>());
    case 256: return rows(integral_constant<int, 256>());
    default: return rows(integral_constant<int, 512>());
  }
}
}  // namespace

int64_t paged_tiles_workspace(const PagedAttentionArgs& a) {
  return by_shape(a, [&](auto d, auto rows) { return workspace<decltype(d)::value, decltype(rows)::value>(a); });
}

const char* launch_paged_tiles(const PagedAttentionArgs& a, int least_rows, void* space, cudaStream_t stream) {
  return by_shape(a, [&](auto d, auto rows) { return launch<decltype(d)::value, decltype(rows)::value>(a, least_rows, space, stream); });
}

}  // namespace me

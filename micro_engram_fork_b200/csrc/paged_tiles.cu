// Attention of chunks of new tokens over a paged cache, on the tensor cores.
//
// Many rows a key head: S = Q K^T and O += P V are bound by the tensor cores, and next by the L2 cache, out of which every tile of
// rows reads its sequence's keys and values again. So two SMs work as one (cta_group::2): 256 rows (new token, query head of the
// key head's group) a pair, 128 of them in each SM's tensor memory, and each SM loads half of every block of 128 keys, which halves what
// both read. Per SM and block at dim 256: 64 KB in 2048 clocks of the tensor core.
//
//   warps 0, 2 loads: rows of Q once a unit, and K; V (TMA, each through a ring of its own; a page is a run of rows of the tensor
//              map, a page that is none is an index past its last dimension, which reads zeros)
//   warp 1     issues the products (from the even SM): S of block j + 1 goes ahead of P V of block j, so that block j's
//              softmax has the time of two products
//   warp 3     finds the pair's next unit while the others are at work, two ahead
//   warps 4-11 softmax, two threads a row (a half of a block's keys each): 64 scores from tensor memory; p = 2^(s - m) by the
//              maximum m that the row's threads had agreed on a block before, for the maximum of this block comes round through shared
//              memory while they compute (a row that has none yet, or jumps by more than 2^60, waits for it). O is rescaled
//              only when m grows by more than 2^8. P is rounded to bf16 (as what it is multiplied with is) and put back over its scores, from where
//              it is the A operand of P V; the sum is of the terms before that. At a unit's end: O / sum to global memory
//
// Tensor memory: O in columns 0-255, two S (P) buffers of 128. dim 512 has no room for both halves of O: a unit takes one half of the
// columns, and S is computed twice (4/3 of the operations).
// Rows of V that no row of the sequence may see (past its end, before its first window) can hold anything, and 0 * NaN is not 0: in blocks that have
// such rows the softmax threads wait for V themselves and put zeros there.
//
// Units (sequence, tile of rows, key head, half of the columns) are dealt to the pairs in turn, the longest of a sequence first. With few of them a
// sequence's keys are cut into chunks, whose (max, sum, O) a second kernel joins.
// Every wait is bounded (2 s); a timeout records ME_ERR_TIMEOUT in the status word and the kernel frees tensor memory and returns.
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

constexpr int kParts = 2, kSoftWarps = 4 * kParts, kFirstSoft = 4, kThreads = (kFirstSoft + kSoftWarps) * 32;  // kParts softmax threads a row
constexpr int BM = 128, BN = 128;     // rows an SM, keys a block
constexpr int kLeastBlocks = 8;       // of a chunk: below, its O costs more to write and join than its keys
constexpr int kDeals = 4;             // units a pair that cutting aims at

template <int D>
struct Cfg {
  static constexpr int DV = D < 256 ? D : 256;       // columns of O a unit
  static constexpr int HALVES = D / DV;
  static constexpr int NV = D == 64 ? 128 : DV;      // columns of the P V product (dim 64: the odd SM's half is past the row, zeros)
  static constexpr int VC = NV / 2;                  // of them in this SM
  static constexpr int Q_BYTES = BM * D * 2;
  // a stage of K: this SM's 64 keys of a block x KC columns; of V: 128 keys x VC, one set of 64 keys after the other
  static constexpr int KC = D < 256 ? D : 256, K_STAGES = D / KC;
  static constexpr int K_BYTES = 64 * KC * 2, V_BYTES = BN * VC * 2;
  static constexpr int KR = D == 512 ? 2 : D == 256 ? 3 : 6, VR = D == 512 ? 1 : D == 256 ? 2 : 6;  // stages
  static constexpr int K_OFF = Q_BYTES, V_OFF = K_OFF + KR * K_BYTES, BAR_OFF = V_OFF + VR * V_BYTES;
  static constexpr int MEET_OFF = BAR_OFF + 640;   // [4 blocks][BM]: maxima; [kParts][BM]: sums
  static constexpr int SMEM = MEET_OFF + 4 * BM * 4;
  static_assert(SMEM <= 232448, "shared memory");
  static_assert((2 * KR + 3 * VR + 19) * 8 <= 496, "barriers");
};
constexpr int kO = 0, kS = 256;  // columns of tensor memory
constexpr float kJump = 60.f;   // a score this far above m (log2) does not wait for the next block

struct TilesArgs {
  PagedAttentionArgs a;
  float* part_o;    // [slots][slot_rows][DV]
  float2* part_ml;  // [slots][slot_rows]
  int slot_rows;    // a sequence with more rows is not cut, unless 256
  int pairs;
  int plog;
  int least_rows;   // sequences with up to this many rows are others' work
};
// The first wait that ran out (ME_ERR_TIMEOUT, where): a device's own word, not an allocation that a captured graph could own.
__device__ int g_status[2];

// ------------------------------------------------------------------------------- units of work
struct UnitsOf {
  int tiles, chunks, per;  // tiles of rows, chunks of keys, blocks of a chunk
  int first, blocks;       // the sequence's blocks of keys
};
template <int D>
ME_DEVICE UnitsOf units_of(const TilesArgs& t, int b, const Sequence& s, int cut) {
  const PagedAttentionArgs& a = t.a;
  const int group = a.q_heads / a.cache.heads, tokens = 2 * (BM / group);
  if (s.count == 0 || (int64_t)s.count * group <= t.least_rows) return {0, 1, 0, 0, 0};
  const Keys k = keys_of(a.batch, a.cache.page, s, 0, s.count - 1, a.window);
  UnitsOf u;
  u.tiles = (s.count + tokens - 1) / tokens;
  u.first = k.lo / BN;
  u.blocks = max((k.hi + BN - 1) / BN - u.first, 1);
  const bool whole = cut <= 0 || (t.slot_rows < 2 * BM && (int64_t)s.count * group > t.slot_rows);
  u.chunks = whole ? 1 : (u.blocks + cut - 1) / cut;
  u.per = (u.blocks + u.chunks - 1) / u.chunks;
  return u;
}

// Blocks a chunk that make about kDeals units a pair, 0: no cutting, where the units as they are keep four pairs of five busy. At most 2 kDeals
// units a pair come of it: as many as there were (fewer than kDeals) and one for every `cut` blocks.
template <int D, int NT>
ME_DEVICE int cut_of(const TilesArgs& t, typename WorkLine<NT>::Shared& sh, int64_t& units) {
  WorkLine<NT> line(sh);
  const PagedBatch& p = t.a.batch;
  const int each = t.a.cache.heads * Cfg<D>::HALVES;
  units = line.total(p.seqs, [&](int b) -> int64_t { return (int64_t)units_of<D>(t, b, sequence_of(p, b), 0).tiles * each; });
  const int64_t aim = (int64_t)kDeals * t.pairs;
  if (units == 0 || units >= aim) return 0;
  const int few = (int)units, deals = (few + t.pairs - 1) / t.pairs;
  if (few * 5 >= deals * t.pairs * 4) return 0;
  const int64_t blocks = line.total(p.seqs, [&](int b) -> int64_t {
    const UnitsOf u = units_of<D>(t, b, sequence_of(p, b), 0);
    return (int64_t)u.tiles * each * u.blocks;
  });
  return (int)max((blocks + aim - 1) / aim, (int64_t)kLeastBlocks);
}

struct Unit {
  Sequence s;
  int b, tile, kv, half;
  int kb0, kb1;  // its blocks of keys, kb1 <= kb0: none
  int chunk, chunks;
};

// A warp's way along the units: 32 sequences at a time, a lane each.
template <int D>
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
      const UnitsOf u = units_of<D>(t, b, sequence_of(p, b), cut);
      mine = (int64_t)u.tiles * u.chunks * t.a.cache.heads * Cfg<D>::HALVES;
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
    const UnitsOf u = units_of<D>(t, out.b, out.s, cut);
    unsigned i = (unsigned)(x - before);  // (a sequence's units: the host checks that they fit)
    out.half = i % Cfg<D>::HALVES, i /= Cfg<D>::HALVES;
    out.kv = i % a.cache.heads, i /= a.cache.heads;
    out.chunk = i % u.chunks, out.chunks = u.chunks, i /= u.chunks;
    out.tile = u.tiles - 1 - (int)i;  // the last rows see the most keys
    const int tokens = 2 * (BM / (a.q_heads / a.cache.heads));
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
// The order of floats as that of integers, and back.
ME_DEVICE int ordered(float x) {
  const int i = __float_as_int(x);
  return i ^ ((i >> 31) & 0x7fffffff);
}
ME_DEVICE float unordered(int i) { return __int_as_float(i ^ ((i >> 31) & 0x7fffffff)); }

// The pair's product and its commits, by the lanes of `issue` (one lane of the warp that goes along).
ME_DEVICE void umma_bf16_pair_if(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate, uint32_t issue) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(issue));
}
// A (P) from tensor memory.
ME_DEVICE void umma_bf16_pair_ts_if(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate, uint32_t issue) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(issue));
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
template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    paged_tiles_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                       const __grid_constant__ TilesArgs args) {
  using C = Cfg<D>;
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
  uint64_t* meet_bar = all_done + 1;  // [4] the warps of the same rows
  uint64_t* next_full = meet_bar + 4;   // [2]
  uint64_t* next_empty = next_full + 2; // [2]
  int* next_unit = reinterpret_cast<int*>(smem + C::BAR_OFF + 496);  // [2][16]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::BAR_OFF + 624);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  int* tops = reinterpret_cast<int*>(smem + C::MEET_OFF);       // [4][BM] ordered()
  float* sums = reinterpret_cast<float*>(smem + C::MEET_OFF);   // [kParts][BM]
  auto& line_shared = *reinterpret_cast<typename WorkLine<kThreads>::Shared*>(sQ);  // before Q comes

  const PagedAttentionArgs& a = args.a;
  const PagedBatch& p = a.batch;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1;
  const int group = a.q_heads / a.cache.heads, tokens = BM / group;  // new tokens an SM
  int* status = g_status;
  if (smem_addr(smem) & 1023) {
    report(status, ME_ERR_ALIGN, 76);
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
    for (int i = 0; i < 4; ++i) mbar_init(&meet_bar[i], kParts);
    for (int i = 0; i < 2; ++i) mbar_init(&next_full[i], 1), mbar_init(&next_empty[i], 2 + kSoftWarps + (leader ? 1 : 0));
    *abort = 0;
    fence_barrier_init();
    prefetch_tmap(&tq);
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
  }
  if (warp == 1) tmem_alloc_pair(tmem_slot, 512);
  for (int i = threadIdx.x; i < 4 * BM; i += kThreads) tops[i] = ordered(-INFINITY);
  if (args.least_rows == 0) clear_rest<D>(a, kThreads);  // (else the kernel of few rows does)
  int64_t units0;
  const int cut = cut_of<D, kThreads>(args, line_shared, units0);
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
  auto wait_u = [&](uint64_t* bar, int parity, int where) {
    return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) || __all_sync(0xffffffffu, mbar_wait(bar, parity, status, where, abort));
  };
  Unit u;
  Keys seq;
  int unit_x = 0;
  auto take_unit = [&](int it, int where) {
    if (!wait_u(&next_full[it & 1], (it >> 1) & 1, where)) return false;
    const int mine = next_unit[(it & 1) * 16 + (lane & 15)];
    __syncwarp();
    if (lane == 0) mbar_arrive(&next_empty[it & 1]);
    auto field = [&](int i) { return uniform(__shfl_sync(0xffffffffu, mine, i)); };
    u.s = {field(1), field(2), field(3)};
    u.b = field(4), u.tile = field(5), u.kv = field(6), u.half = field(7);
    u.kb0 = field(8), u.kb1 = field(9), u.chunk = field(10), u.chunks = field(11);
    seq = {field(12), field(13)};
    unit_x = field(14);
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
      // pages of a block, a lane for each 16 keys; an index past the cache where there is none
      auto pages_of = [&](int kb) {
        int id = -1;
        if (lane < 8) id = page_at(p, a.cache.pages, u.b, (kb * BN + lane * 16) >> args.plog);
        return id < 0 ? a.cache.pages : id;
      };
      // 64 keys from `in` of block kb, NC x 64 columns from chunk x on
      auto load64 = [&](uint32_t dst, const CUtensorMap* map, uint32_t bar, int kb, int in, int ids, int x, auto NC) {
        if (box == 64) {
          const int id = __shfl_sync(0xffffffffu, ids, in / 16);
          tma_load_4d_pair_if(dst, map, bar, 0, y0 + ((kb * BN + in) & page_mask), x, id, one);
        } else {
          for (int row = 0; row < 64; row += box) {
            const int id = __shfl_sync(0xffffffffu, ids, (in + row) / 16);
#pragma unroll
            for (int i = 0; i < decltype(NC)::value; ++i)
              tma_load_4d_pair_if(dst + i * (64 * 128) + row * 128, map, bar, 0, y0 + ((kb * BN + in + row) & page_mask), x + i, id, one);
          }
        }
      };
      int ids = pages_of(u.kb0);
      for (int j = 0; j < n && ok; ++j) {
        const int next = j + 1 < n ? pages_of(u.kb0 + j + 1) : 0, kb = u.kb0 + j;
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
              tma_load_3d_pair_if(aQ + c * (BM * 128), &tq, q_leader, c * 64, u.kv * group, u.s.first + u.tile * 2 * tokens + (int)rank * tokens, one);
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
        ids = next;
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
      const uint64_t dQ = desc_sw128(smem_addr(sQ)), dK = desc_sw128(smem_addr(sK)), dV = desc_mn_sw128(smem_addr(sV), 64 * 128, 1024);
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
#pragma unroll
            for (int c = 0; c < C::K_STAGES; ++c) {
              wait(&k_full[kst], kphase, 63);
              if (!ok) break;
              tc_fence_after();
              const uint64_t dk = dK + (kst * C::K_BYTES >> 4);
#pragma unroll
              for (int kk = 0; kk < C::KC / 16; ++kk)
                umma_bf16_pair_if(to, dQ + (((c * (C::KC / 64) + kk / 4) * (BM * 128) + (kk & 3) * 32) >> 4),
                                  dk + (((kk / 4) * (64 * 128) + (kk & 3) * 32) >> 4), id_s, (c | kk) != 0, one);
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
            const uint64_t dv = dV + (vst * C::V_BYTES >> 4);
#pragma unroll
            for (int kk = 0; kk < BN / 16; ++kk)
              umma_bf16_pair_ts_if(kO, kS + (i & 1) * BN + kk * 8, dv + (((kk / 4) * (C::V_BYTES / 2) + (kk & 3) * 2048) >> 4), id_o, (j > 1 || kk > 0), one);
            umma_commit_pair_if(&v_empty[vst], one);
            if (++vst == VR) vst = 0, vphase ^= 1;
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
    Walk<D> walk(args, cut);
    Unit w = {};
    bool more = true;
    for (int it = 0; more; ++it) {
      const int64_t x = pair + (int64_t)it * args.pairs;
      more = __all_sync(0xffffffffu, walk.at(x, w));
      const Keys k = keys_of(p, a.cache.page, w.s, 0, w.s.count - 1, a.window);
      if (it >= 2 && !wait_u(&next_empty[it & 1], ((it >> 1) - 1) & 1, 80)) break;
      int* to = next_unit + (it & 1) * 16;
      if (lane == 0) {
        to[0] = more, to[1] = w.s.first, to[2] = w.s.count, to[3] = w.s.context, to[4] = w.b, to[5] = w.tile, to[6] = w.kv, to[7] = w.half;
        to[8] = w.kb0, to[9] = w.kb1, to[10] = w.chunk, to[11] = w.chunks, to[12] = k.lo, to[13] = k.hi, to[14] = (int)x;
        mbar_arrive(&next_full[it & 1]);
      }
      __syncwarp();
    }
  } else if (warp >= kFirstSoft) {
    // ---------------------------------------------------------------- softmax
    const int quarter = warp & 3, part = (warp - kFirstSoft) >> 2, r = quarter * 32 + lane;  // part of a block's keys; row of the SM
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t p_leader = mapa_shared(smem_addr(p_full), 0), o_leader = mapa_shared(smem_addr(o_free), 0);
    constexpr int HB = BN / kParts;  // keys a thread
    const float to_log2 = a.scale * kLog2e;
    const int ti = r / group, head = r % group;
    // 32-byte stores of O where its rows allow them
    const bool wide = reinterpret_cast<uintptr_t>(a.o) % 32 == 0 && a.o_token % 16 == 0 && a.o_head % 16 == 0;
    int gb = 0, live = 0, met = 0;  // blocks, units with any, meetings so far
    uint32_t v_phases = 0;          // bit i: parity of v_here[i]
    bool ok = true;
    // The row's four warps meet: what each wrote before come_by() is there after meet().
    auto come_by = [&] {
      __syncwarp();
      if (lane == 0) mbar_arrive(&meet_bar[quarter]);
    };
    auto meet = [&] { ok = wait_u(&meet_bar[quarter], met & 1, 75), ++met; };
    // The sum of all parts' x, in the parts' order. (sums lies over tops: both are idle at a unit's end.)
    auto sum_up = [&](float x) {
      sums[part * BM + r] = x;
      come_by(), meet();
      const float all = sums[r] + sums[BM + r];
      come_by(), meet();
      return all;
    };
    for (int it = 0; ok && take_unit(it, 77); ++it) {
      const int n = max(u.kb1 - u.kb0, 0);
      const int token = u.tile * 2 * tokens + (int)rank * tokens + ti;  // of the sequence's new ones
      const bool mine = ti < tokens && token < u.s.count;
      const int last = mine ? min(u.s.context + token, seq.hi - 1) : -1;
      const int from = a.window > 0 ? u.s.context + token - a.window + 1 : 0;
      float m = -INFINITY, l = 0.f;  // l: this part's sum of p
      float alpha = 1.f;             // what O has to be rescaled by
      auto pages_of = [&](int kb) {  // bit i: keys 16 i of the four blocks from kb on have a page
        return __ballot_sync(0xffffffffu, page_at(p, a.cache.pages, u.b, (kb * BN + lane * 16) >> args.plog) >= 0);
      };
      uint32_t there = n > 0 ? pages_of(u.kb0) : 0, there_next = 0;
      for (int j = 0; j < n && ok; ++j) {
        const int i = gb + j, kb = u.kb0 + j, key0 = kb * BN + part * HB;
        if ((j & 3) == 0) {
          if (j > 0) there = there_next;
          if (j + 4 < n) there_next = pages_of(kb + 4);
        }
        const uint32_t pages = (there >> ((j & 3) * 8 + part * (HB / 16))) & 0xfu;
        const bool open = pages == 0xfu && ((key0 >= from && key0 + HB - 1 <= last) || !mine), all_open = __all_sync(0xffffffffu, open);
        if (!(ok = wait_u(&s_full[i & 1], (i >> 1) & 1, 70))) break;
        tc_fence_after();
        const uint32_t at = tmem + lanes + kS + (i & 1) * BN;
        float top = -INFINITY, sum[2];
        uint32_t pk[HB / 2];
        bool first = true;  // a second pass, from the scores again, for a row that jumps
#pragma unroll 1
        for (;;) {
          uint32_t s[HB];
          uint32_t(&low)[32] = reinterpret_cast<uint32_t(&)[32]>(s[0]), (&high)[32] = reinterpret_cast<uint32_t(&)[32]>(s[32]);
          tmem_issue_ld32(at + part * HB, low);
          tmem_issue_ld32(at + part * HB + 32, high);
          tmem_wait_ld(low);
          tmem_wait_ld(high);
          if (!all_open) {
#pragma unroll
            for (int c = 0; c < HB; c += 32) {
              // bits from .. last of these 32 keys that have a page
              const int lo = min(max(from - key0 - c, 0), 32), hi = min(max(last + 1 - key0 - c, 0), 32);
              uint32_t seen = (uint32_t)(((1ull << hi) - 1) & ~((1ull << lo) - 1));
              seen &= ((pages >> (c / 16)) & 1 ? 0xffffu : 0u) | ((pages >> (c / 16)) & 2 ? 0xffff0000u : 0u);
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (!(seen & (1u << e))) s[c + e] = 0xff800000u;  // -inf
            }
          }
          bool wait_here = !first;  // the maximum of this block has come round before the exponentials
          if (first) {
            first = false;
            float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int e = 0; e < HB; ++e) mx[e & 3] = fmaxf(mx[e & 3], __uint_as_float(s[e]));
            atomicMax(&tops[(i & 3) * BM + r], ordered(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]))));
            if (part == 0) tops[((i + 2) & 3) * BM + r] = ordered(-INFINITY);  // block i - 2's, which all have read: its P has been taken
            come_by();
            if (__any_sync(0xffffffffu, m == -INFINITY && mine)) {
              meet();
              if (!ok) break;
              top = unordered(tops[(i & 3) * BM + r]) * to_log2;
              if (m == -INFINITY) m = top;
              wait_here = true;
            }
          }
          const float z = m == -INFINITY ? 0.f : m;
          sum[0] = sum[1] = 0.f;
#pragma unroll
          for (int e = 0; e < HB; e += 2) {
            const float p0 = ex2(fmaf(__uint_as_float(s[e]), to_log2, -z)), p1 = ex2(fmaf(__uint_as_float(s[e + 1]), to_log2, -z));
            sum[0] += p0, sum[1] += p1;
            pk[e / 2] = pack2(p0, p1);
          }
          if (!wait_here) {
            meet();  // (and all have read their scores: P may go over them)
            if (!ok) break;
            top = unordered(tops[(i & 3) * BM + r]) * to_log2;
          }
          if (!__any_sync(0xffffffffu, top > m + kJump)) break;  // (the row's threads see the same numbers)
          if (top > m + kJump) {
            const float f = ex2(m - top);
            alpha *= f, l *= f;
            m = top;
          }
        }
        if (!ok) break;
        l += sum[0] + sum[1];
        tmem_st32u(at + part * (HB / 2), pk);
        if (__any_sync(0xffffffffu, alpha != 1.f) && j > 0) {  // O stands still once the product before has ended
          if (!(ok = wait_u(&pv_done[(i - 1) & 1], ((i - 1) >> 1) & 1, 71))) break;
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < C::DV / kParts; c += 16) {
            uint32_t o[16];
            const uint32_t col = tmem + lanes + kO + part * (C::DV / kParts) + c;
            tmem_issue_ld16(col, o);
            tmem_wait_ld(o);
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
            tmem_st16u(col, o);
          }
        }
        alpha = 1.f;
        if (top > m + kSlack) {  // from the next block on
          alpha = ex2(m - top);
          l *= alpha;
          m = top;
        }
        const bool stale = has_stale(seq, kb);
        if (stale) {  // row r: key r of the block, a part of this SM's columns
          const int st = i % VR;
          if (!(ok = wait_u(&v_here[st], (v_phases >> st) & 1, 72))) break;
          v_phases ^= 1u << st;
          const int key = kb * BN + r;
          if (key < seq.lo || key >= seq.hi) {
#pragma unroll
            for (int i8 = 0; i8 < C::VC / 8 / kParts; ++i8) {
              const int c = part * (C::VC / 8 / kParts) + i8;  // of its 16-byte chunks
              *reinterpret_cast<uint4*>(sV + st * C::V_BYTES + (r / 64) * (C::V_BYTES / 2) + (c / 8) * (64 * 128) + (r & 63) * 128 + (c & 7) * 16) =
                  make_uint4(0, 0, 0, 0);
            }
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
      float o_scale = 1.f;
      if (n > 0 && ok) {
        o_scale = alpha;  // a rescaling that no block was left for
        come_by(), meet();  // all have read the last maxima
        if (ok) l = sum_up(l);
        tops[part * BM + r] = tops[(part + 2) * BM + r] = ordered(-INFINITY);
        come_by();
        if (ok) meet();
        if (ok) ok = wait_u(o_full, live & 1, 73);
        ++live;
      }
      if (!ok) break;
      tc_fence_after();
      const float inv = u.chunks > 1 ? o_scale : l == 0.f ? 0.f : o_scale / l;  // (a part keeps its sum)
      const int t = u.s.first + token, h = u.kv * group + head;
      const int64_t slot = (int64_t)unit_x * args.slot_rows + (int)rank * tokens * group + r;
      constexpr int PC = C::DV / kParts, PS = PC < 32 ? PC : 32;  // this part's columns of O, and of a step
      const int col0 = part * PC;
      auto release = [&] {  // O has been read: the next unit's products may go over it
        if (n == 0) return;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_cta(o_leader);
      };
      if (u.chunks > 1) {
        float* dst = args.part_o + slot * C::DV + col0;
#pragma unroll 1
        for (int c = 0; c < PC; c += PS) {
          uint32_t o[32] = {};
          if (n > 0) {
            tmem_issue_ld32(tmem + lanes + kO + col0 + c, o);
            tmem_wait_ld(o);
          }
          if (mine)
#pragma unroll
            for (int e = 0; e < PS; e += 4)
              *reinterpret_cast<float4*>(dst + c + e) = make_float4(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv,
                                                                    __uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
        }
        if (mine && part == 0) args.part_ml[slot] = make_float2(m, l);
        release();
      } else {
        uint32_t out[PC / 2] = {};
        if (n > 0) {
#pragma unroll
          for (int c = 0; c < PC; c += PS) {
            uint32_t o[32];
            tmem_issue_ld32(tmem + lanes + kO + col0 + c, o);
            tmem_wait_ld(o);
#pragma unroll
            for (int e = 0; e < PS; e += 2) out[(c + e) / 2] = pack2(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv);
          }
        }
        release();
        if (mine) {
          bf16* dst = reinterpret_cast<bf16*>(a.o) + t * a.o_token + h * a.o_head + u.half * C::DV + col0;
#pragma unroll
          for (int e = 0; e < PC / 2; e += 8) {
            if (wide) {
              st_global32(dst + e * 2, &out[e]);
            } else {
              *reinterpret_cast<uint4*>(dst + e * 2) = make_uint4(out[e], out[e + 1], out[e + 2], out[e + 3]);
              *reinterpret_cast<uint4*>(dst + e * 2 + 8) = make_uint4(out[e + 4], out[e + 5], out[e + 6], out[e + 7]);
            }
          }
          if (u.half == 0 && part == 0) a.lse[(int64_t)h * p.tokens + t] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
        }
      }
      gb += n;
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // both SMs are done with every product, copy and remote arrival
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// Joins the chunks of sequences that were cut: a block takes every gridDim.x-th 32 rows of units.
constexpr int kJoinThreads = 256, kJoinRows = 32;
template <int D>
__global__ void __launch_bounds__(kJoinThreads) paged_join_tiles_kernel(const __grid_constant__ TilesArgs args) {
  using C = Cfg<D>;
  constexpr int PER = C::DV / 4, ROWS = kJoinThreads / PER, STEPS = 2 * BM / kJoinRows;
  __shared__ typename WorkLine<kJoinThreads>::Shared line_shared;
  const PagedAttentionArgs& a = args.a;
  int64_t units;
  const int cut = cut_of<D, kJoinThreads>(args, line_shared, units);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  if (cut == 0) return;
  const int group = a.q_heads / a.cache.heads, tokens = 2 * (BM / group);
  Walk<D> walk(args, cut);
  Unit u;
  for (int64_t i = blockIdx.x; walk.at(i / STEPS, u); i += gridDim.x) {
    if (u.chunks == 1 || u.chunk != 0) continue;
    const int64_t x = i / STEPS, stride = (int64_t)a.cache.heads * C::HALVES;  // between a tile's chunks
    const int i0 = u.tile * tokens, rows = min(tokens, u.s.count - i0) * group, r0 = (int)(i % STEPS) * kJoinRows;
    const int c = threadIdx.x % PER * 4;
    for (int r = r0 + threadIdx.x / PER; r < min(rows, r0 + kJoinRows); r += ROWS) {
      float top = -INFINITY, l = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int k = 0; k < u.chunks; ++k) {
        const int64_t slot = (x + k * stride) * args.slot_rows + r;
        const float2 ml = args.part_ml[slot];
        const float4 y = *reinterpret_cast<const float4*>(args.part_o + slot * C::DV + c);
        if (ml.x == -INFINITY && ml.y == 0.f) continue;
        const float up = fmaxf(top, ml.x);
        const float f0 = top == -INFINITY ? 0.f : ex2(top - up), f1 = ex2(ml.x - up);
        o.x = o.x * f0 + y.x * f1, o.y = o.y * f0 + y.y * f1, o.z = o.z * f0 + y.z * f1, o.w = o.w * f0 + y.w * f1;
        l = l * f0 + ml.y * f1;
        top = up;
      }
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const int t = u.s.first + i0 + r / group, h = u.kv * group + r % group;
      uint2 b4;
      b4.x = pack2(o.x * inv, o.y * inv), b4.y = pack2(o.z * inv, o.w * inv);
      *reinterpret_cast<uint2*>(reinterpret_cast<bf16*>(a.o) + t * a.o_token + h * a.o_head + u.half * C::DV + c) = b4;
      if (c == 0 && u.half == 0) a.lse[(int64_t)h * a.batch.tokens + t] = l == 0.f ? -INFINITY : (top + log2f(l)) * kLn2;
    }
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

template <int D>
int resident_pairs() {
  static std::mutex mu;
  static std::unordered_map<int, int> known;
  int dev = 0;
  cudaGetDevice(&dev);
  std::lock_guard<std::mutex> lk(mu);
  auto it = known.find(dev);
  if (it != known.end()) return it->second;
  cudaFuncSetAttribute(paged_tiles_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::SMEM);
  int sms = 0, n = 0;
  cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = 2, attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.gridDim = dim3(sms & ~1);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = Cfg<D>::SMEM;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, paged_tiles_kernel<D>, &cfg) != cudaSuccess || n <= 0) {
    (void)cudaGetLastError();
    n = sms / 2;
  }
  return known[dev] = n;
}

template <int D>
int slot_rows_of(const PagedAttentionArgs& a) {
  return (int)std::min<int64_t>(2 * BM, ((int64_t)a.max_q * (a.q_heads / a.cache.heads) + 7) / 8 * 8);
}
template <int D>
int64_t workspace(const PagedAttentionArgs& a) {
  return (int64_t)2 * kDeals * resident_pairs<D>() * slot_rows_of<D>(a) * (Cfg<D>::DV + 2) * 4;
}

template <int D>
const char* launch(const PagedAttentionArgs& a, int least_rows, void* space, cudaStream_t stream) {
  using C = Cfg<D>;
  if (encode_fn() == nullptr) return "cuTensorMapEncodeTiled is unavailable";
  TilesArgs args;
  args.a = a;
  args.pairs = resident_pairs<D>();
  args.slot_rows = slot_rows_of<D>(a);
  args.part_o = static_cast<float*>(space);
  args.part_ml = reinterpret_cast<float2*>(args.part_o + (int64_t)2 * kDeals * args.pairs * args.slot_rows * C::DV);
  args.plog = 0;
  while ((1 << args.plog) < a.cache.page) ++args.plog;
  args.least_rows = least_rows;
  bind_primary_context();
  const int group = a.q_heads / a.cache.heads, box = std::min(a.cache.page, 64);
  const int64_t rows = (int64_t)a.cache.heads * a.cache.page;
  // pages as [page][64 columns of the head][head, position][column]
  const int64_t dims[4] = {64, rows, D / 64, a.cache.pages};
  CUtensorMap tq, tk, tv;
  if (!make_map<3>(&tq, a.q, {D, a.q_heads, a.batch.tokens}, {a.q_head, a.q_token}, {group, BM / group}) ||
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
  cudaError_t e = cudaLaunchKernelEx(&cfg, paged_tiles_kernel<D>, tq, tk, tv, args);
  if (e != cudaSuccess) return cudaGetErrorString(e);
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(8 * args.pairs);
  cfg.blockDim = dim3(kJoinThreads);
  cfg.dynamicSmemBytes = 0;
  e = cudaLaunchKernelEx(&cfg, paged_join_tiles_kernel<D>, args);
  return e == cudaSuccess ? nullptr : cudaGetErrorString(e);
}

}  // namespace

int paged_status(int* detail) {
  int word[2] = {0, 0};
  cudaMemcpyFromSymbol(word, g_status, sizeof word);
  *detail = word[1];
  return word[0];
}

int64_t paged_tiles_workspace(const PagedAttentionArgs& a) {
  switch (a.cache.dim) {
    case 64: return workspace<64>(a);
    case 128: return workspace<128>(a);
    case 256: return workspace<256>(a);
    default: return workspace<512>(a);
  }
}

const char* launch_paged_tiles(const PagedAttentionArgs& a, int least_rows, void* space, cudaStream_t stream) {
  switch (a.cache.dim) {
    case 64: return launch<64>(a, least_rows, space, stream);
    case 128: return launch<128>(a, least_rows, space, stream);
    case 256: return launch<256>(a, least_rows, space, stream);
    default: return launch<512>(a, least_rows, space, stream);
  }
}

}  // namespace me

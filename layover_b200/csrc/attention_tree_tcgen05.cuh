// Attention for trees of drafts on the 5th-generation tensor cores: bfloat16, heads of 128 channels, pages of 8 .. 128 tokens.
//
// The work is a list of key tiles (128 keys of one key/value head for one tile of rows), sequence by sequence, and every block takes
// an equal, contiguous share of the list: a few segments, each a row tile and a range of its keys. Blocks stay for the whole
// launch, one an SM, so the loads of a segment run under the arithmetic and the stores of the one before. A row tile whose keys
// lie in several blocks' shares leaves maxima, sums and unnormalised outputs in scratch memory, two places a block (its first and its last
// segment), for `join_kernel`.
//
// A row tile holds 128 / group drafts with all their heads of the group, or, with ROWS2, twice as many. Two warpgroups of softmax
// have scores and an output accumulator of their own in tensor memory: they take the key tiles in turn, or, with ROWS2, a half of
// the rows each. Either way the products go through "turns" 0, 1, 2, ... of alternate warpgroups: O += P(t) V, then S(t + 2) = Q K^T,
// so that one warpgroup's softmax runs under the other's products. K and V come through a ring each,
// 16 bytes a thread (cp.async, two warps for either; a TMA copy of a page of 16 tokens takes 70 cycles whoever issues it, 1,150 for
// the 32 KB of a tile with pages of 16, and 1,430 are what a tile may take at the memory's rate). The weights overwrite their scores in tensor
// memory and are the A operand of the second product.
//
// Code that runs first is slow: a turn of softmax takes four times as long until its instructions have been fetched. So the warps run
// through parts of it each, on nothing, while the first loads are under way.
//
// The keys' and values' bytes bound it. Measured (one B200): 40 requests of 25 drafts after 400 .. 8,000 keys, 32 heads over 8, 150 us where calls
// follow one another in a graph over three sets of inputs (734 MB, 4.9 TB/s), 169 as single calls over many (4.3); 8 of 32 after 3,000 37 us (104 MB);
// 2 of 64 after 12,345, 16 over 4, 44 to 50 us (52 MB), 9 of them the join of 18 parts a row; 1 of 8 after 700 12.1 us. What is left is time in
// which nothing streams: about 4 us until a block's share is known and 4 more until its first scores, 4 to 6 at the border of two segments (partial
// tiles, results to be stored, instructions that run for the first time), and the join. The same by mma.sync, the rows' keys in chunks: 843, 202 and
// 167 us.
//
// The weights round to bfloat16 for the second product, as in the package's other kernels of the models that take drafts (the output is off by 0.0023
// of its size against 64 bits, 0.0017 with weights of 32 bits); their sum, the maxima and the outputs are held in 32 bits.
//
// Rows that the tree does not have cost nothing but the tensor cores' time: their warps only hand tiles on. A draft's values may hold what
// is not finite, and 0 x NaN is NaN also for rows that do not see the draft. A block whose outputs are not all finite therefore takes its share once
// more, carefully: in tiles of which a row may not see every key, zeros stand for values that are not finite, and who sees those gets their
// terms added afterwards. So who does not see them has the bits that he would have beside finite ones, and a call without them pays nothing: to look at
// the drafts' values in every call costs 4 of 38 us and 14 to 26 of 156 (8 x 32 and 40 requests), whichever warp does it, for what runs seldom waits for its
// instructions. With one draft of NaN a call that is waited for takes 122 us instead of 62 (8 x 32) and 537 instead of 194 (40 requests). (Its rows
// made again key by key: 10,100 and 21,800.)
#pragma once
#include <math.h>

#include <type_traits>

#include "attention_tree.cuh"
#include "tcgen05.cuh"

namespace {

__device__ int g_tree_error = 0;       // 0 = ok; which wait ran out otherwise: 1 ring, 2 queries, 3 keys, 4 values, 5 weights, 6 scores, 7 and 8 second product, 9 values that are looked at

namespace wide {

constexpr int ROWS = 128, KEYS = 128, DIM = 128;
constexpr int HALF_BYTES = 128 * 128;           // 64 channels of 128 rows
constexpr int TILE_BYTES = 2 * HALF_BYTES;
constexpr int STAGES = 2;                       // tiles of either ring
constexpr int LOADERS = 4;                      // warps that load: two K, two V, each 64 rows of a tile
constexpr int FIRST_SOFTMAX = 8;                // then one that issues the products, one for the borders and two of the careful pass, then two warpgroups of softmax
constexpr int THREADS = 32 * (FIRST_SOFTMAX + 8);
constexpr int FEW_REGS = 72, MANY_REGS = 184;   // of a thread of the first eight warps and of the others: 256 * (72 + 184) = 512 * 128, the launch's
constexpr int SEQ_CACHE = 512;                  // sequences whose lengths are kept there
// A pass's barriers: K's, then V's stages are full and empty; a segment's queries have come (two segments, or ROWS2: the first alone) and its last
// scores are made; a turn's scores are in tensor memory (two warpgroups), its weights are, and the output is rescaled, its second product is
// finished; a segment's products are finished, its outputs have been read, its maxima and sums are in shared memory; `start` and `known`
// are; in the careful pass, values that are still to be looked at have come (two halves of a tile, STAGES).
constexpr int FULL = 0, EMPTY = FULL + 2 * STAGES, Q_FULL = EMPTY + 2 * STAGES, Q_EMPTY = Q_FULL + 2, S_FULL = Q_EMPTY + 2, P_FULL = S_FULL + 2,
              PV_DONE = P_FULL + 2, O_FULL = PV_DONE + 2, O_EMPTY = O_FULL + 1, STATS_FULL = O_EMPTY + 1, STARTED = STATS_FULL + 1, LANDED = STARTED + 1,
              BARRIERS = LANDED + 2 * STAGES;
constexpr int SMEM_BYTES = (2 + 2 * STAGES) * TILE_BYTES + 1024 + (2 * BARRIERS + 8) * 8 + 2 * 2 * ROWS * 8 + SEQ_CACHE * 16;
constexpr float GROWTH = 8.0f;                  // the maximum that weights are relative to may lag by this, in log2 units
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Copies, barriers and arrivals by one elected lane of a whole warp with the same operands in every lane: as with the products (tcgen05.cuh),
// from inside a branch each copy would take 60 cycles and more.
__device__ __forceinline__ void load_queries(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n\t}"
      ::"r"(dst), "l"((uint64_t)map), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
}
__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint4 load_shared(uint32_t p) {
  uint4 w;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(p) : "memory");
  return w;
}
__device__ __forceinline__ void clear_shared(uint32_t p) { asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(p), "r"(0) : "memory"); }
// Rows [lo, hi) of a tile of values that are not finite become zeros, by a warp, half of it a row (all its pieces: their order does not matter).
__device__ __forceinline__ void clear_odd_rows(uint32_t tile, int lo, int hi) {
  const int lane = threadIdx.x & 31;
  const uint32_t at = tile + ((lane & 15) >> 3) * HALF_BYTES + (lane & 7) * 16;
#pragma unroll 1
  for (int r0 = lo; r0 < hi; r0 += 2) {
    const int r = r0 + (lane >> 4);
    const uint4 w = r < hi ? load_shared(at + r * 128) : make_uint4(0, 0, 0, 0);
    const unsigned odd = __ballot_sync(0xffffffffu, not_finite(w.x) || not_finite(w.y) || not_finite(w.z) || not_finite(w.w));
    if (odd >> (lane & 16) & 0xFFFFu) clear_shared(at + r * 128);
  }
}
template <int ID, int N> __device__ __forceinline__ void meet() { asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(N) : "memory"); }
template <int ID, int N> __device__ __forceinline__ bool meet_any(bool mine) {      // whether any of them says so
  uint32_t any;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbar.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(any) : "r"((uint32_t)mine), "n"(ID), "n"(N) : "memory");
  return any != 0;
}
// 16 bytes to shared memory; zeros where `bytes` is 0; an arrival on the barrier when all copies of this thread before it have landed
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy16_or_zeros(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void arrive_when_copied(uint32_t bar) { asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory"); }
template <int N> __device__ __forceinline__ void give_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void take_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) { asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)map) : "memory"); }
// 32 bytes of one thread: a whole sector of the L2
__device__ __forceinline__ void store32(void* p, const uint32_t (&w)[8]) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
// D (+)= A B with A (two bfloat16 of K a column) in tensor memory
__device__ __forceinline__ void umma_from_tmem(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void tmem_ld128(uint32_t taddr, float (&v)[128]) {      // two loads under one wait
  uint32_t r[128];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%128];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%64, %65, %66, %67, %68, %69, %70, %71, %72, %73, %74, %75, %76, %77, %78, %79, %80, %81, %82, %83, %84, %85, %86, %87, %88, %89, %90, %91, %92, %93, %94, %95, %96, %97, %98, %99, %100, %101, %102, %103, %104, %105, %106, %107, %108, %109, %110, %111, %112, %113, %114, %115, %116, %117, %118, %119, %120, %121, %122, %123, %124, %125, %126, %127}, [%129];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63]), "=r"(r[64]), "=r"(r[65]), "=r"(r[66]), "=r"(r[67]), "=r"(r[68]), "=r"(r[69]), "=r"(r[70]), "=r"(r[71]), "=r"(r[72]), "=r"(r[73]), "=r"(r[74]), "=r"(r[75]), "=r"(r[76]), "=r"(r[77]), "=r"(r[78]), "=r"(r[79]), "=r"(r[80]), "=r"(r[81]), "=r"(r[82]), "=r"(r[83]), "=r"(r[84]), "=r"(r[85]), "=r"(r[86]), "=r"(r[87]), "=r"(r[88]), "=r"(r[89]), "=r"(r[90]), "=r"(r[91]), "=r"(r[92]), "=r"(r[93]), "=r"(r[94]), "=r"(r[95]), "=r"(r[96]), "=r"(r[97]), "=r"(r[98]), "=r"(r[99]), "=r"(r[100]), "=r"(r[101]), "=r"(r[102]), "=r"(r[103]), "=r"(r[104]), "=r"(r[105]), "=r"(r[106]), "=r"(r[107]), "=r"(r[108]), "=r"(r[109]), "=r"(r[110]), "=r"(r[111]), "=r"(r[112]), "=r"(r[113]), "=r"(r[114]), "=r"(r[115]), "=r"(r[116]), "=r"(r[117]), "=r"(r[118]), "=r"(r[119]), "=r"(r[120]), "=r"(r[121]), "=r"(r[122]), "=r"(r[123]), "=r"(r[124]), "=r"(r[125]), "=r"(r[126]), "=r"(r[127])
      : "r"(taddr), "r"(taddr + 64) : "memory");
#pragma unroll
  for (int i = 0; i < 128; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_ld64(uint32_t taddr, float (&v)[64]) {
  uint32_t r[64];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(taddr) : "memory");
#pragma unroll
  for (int i = 0; i < 64; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
               ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                 "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ uint64_t desc_k_major(uint32_t addr) {       // rows of 128 bytes, groups of 8 rows 1024 bytes apart: Q and K
  return ((uint64_t)((1024u >> 4) | (1u << 14) | (2u << 29)) << 32) | (((addr >> 4) & 0x3FFFu) | (1u << 16));
}
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t addr) {      // the same bytes with the channels along N: V; its other half HALF_BYTES on
  return ((uint64_t)((1024u >> 4) | (1u << 14) | (2u << 29)) << 32) | (((addr >> 4) & 0x3FFFu) | ((uint32_t)(HALF_BYTES >> 4) << 16));
}
constexpr uint32_t IDESC_S = instr_desc(KEYS), IDESC_O = instr_desc(DIM) | (1u << 16);     // the second with B along N

template <int N>
__device__ __forceinline__ float row_max(const float (&s)[N]) {        // four chains side by side
  float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int e = 0; e < N; e += 4)
#pragma unroll
    for (int k = 0; k < 4; ++k) m[k] = fmaxf(m[k], s[e + k]);
  return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}

// A sequence's rows and keys, and how many units of work it is: a unit is a row tile of a key/value head.
struct Sequence {
  int first, n, held, ctx, key_lo;      // its first token, drafts, held tokens, keys, the first key that a row may see
  int row_tiles, tile_lo, tiles;        // row tiles; the first of its key tiles and how many there are (one at least)
};
template <bool ROWS2>
__device__ __forceinline__ Sequence find_sequence(const TreeArgs& a, int first, int end, int ctx) {
  Sequence s;
  s.first = first;
  s.n = min(end, a.tokens) - first;
  s.ctx = ctx;
  s.held = s.ctx - s.n;
  s.key_lo = a.window > 0 ? max(0, s.held - a.window + 1) : 0;
  const int drafts = a.tile_drafts * (ROWS2 ? 2 : 1);
  s.row_tiles = s.n <= 0 ? 0 : ROWS2 ? (min(s.n, a.max_nodes) + drafts - 1) / drafts : 1;      // one tile holds all drafts, but for ROWS2
  s.tile_lo = s.key_lo / KEYS;
  s.tiles = max(1, (s.ctx + KEYS - 1) / KEYS - s.tile_lo);
  return s;
}
template <bool ROWS2>
__device__ __forceinline__ Sequence find_sequence(const TreeArgs& a, const int4* known, int seq) {
  if (seq < SEQ_CACHE) {
    const int4 k = known[seq];
    return find_sequence<ROWS2>(a, k.x, k.y, k.z);
  }
  return find_sequence<ROWS2>(a, a.cu_q[seq], a.cu_q[seq + 1], a.ctx_len[seq]);
}

// The blocks' shares of `total` tiles: block b begins at total * b / blocks. No more blocks than tiles: a share is empty only where
// it stands behind the list.
__device__ __forceinline__ int share_begin(int total, int b, int blocks) {
  return total < 1 << 20 ? (int)((unsigned)total * (unsigned)b / (unsigned)blocks) : (int)((long)total * b / blocks);      // blocks: 1,024 at most
}
__device__ __forceinline__ int share_of(int total, int at, int blocks) { return (int)((((long)at + 1) * blocks - 1) / total); }

// A block's walk through its share, segment by segment; every role of the block makes the same walk. A segment is the key tiles
// [begin, begin + count) of a row tile, counted from tile_lo on.
template <bool ROWS2>
struct Walk {
  const int4* known;                    // the lengths of the first sequences
  int next_seq, offset, left;           // where the walk stands: in tiles of that sequence; tiles still to come
  Sequence s;
  int seq, head, row_tile, begin, count;
  __device__ __forceinline__ void begin_at(const TreeArgs& a, const int4* known_, int seq_, int offset_, int left_) {
    known = known_; next_seq = seq_; offset = offset_; left = left_;
    count = 0;
    if (left > 0) s = find_sequence<ROWS2>(a, known, next_seq);
  }
  __device__ __forceinline__ bool next(const TreeArgs& a) {
    if (left <= 0) return false;
    while (offset >= a.kv_heads * s.row_tiles * s.tiles) { offset = 0; s = find_sequence<ROWS2>(a, known, ++next_seq); }     // sequences without drafts have no tiles
    const int unit = offset / s.tiles;
    seq = next_seq; head = unit / s.row_tiles; row_tile = unit - head * s.row_tiles;
    begin = offset - unit * s.tiles;
    count = min(s.tiles - begin, left);
    offset += count; left -= count;
    return true;
  }
};

__device__ __forceinline__ float4 four_values(const void* rows, long row) {      // of 128 a row, a lane's
  const uint2 w = *reinterpret_cast<const uint2*>((const bf16*)rows + row * DIM + 4 * (threadIdx.x & 31));
  const float2 x = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w.x)), y = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w.y));
  return make_float4(x.x, x.y, y.x, y.y);
}
// Behind a careful pass, by the softmax warps: the values for which zeros stood are found once more, and who sees them gets their terms added,
// to what the segment's rows left in scratch memory or, where a row tile lies wholly in the block's share, to the output (whose finite channels so
// round twice). `bits`: four words a key tile, of MOST_LOOKS tiles at a time. Rows whose weights are not finite are NaN already.
constexpr int MOST_LOOKS = 4 * ROWS * 8 / 16;
template <bool ROWS2>
__device__ __forceinline__ void add_odd_values(const TreeArgs& a, const int4* known, const int* start, unsigned* bits, int warp) {
  constexpr int WARPS = 8;
  const int lane = threadIdx.x & 31, tile_drafts = a.tile_drafts * (ROWS2 ? 2 : 1);
  Walk<ROWS2> walk;
  walk.begin_at(a, known, start[0], start[1], start[2]);
  while (walk.next(a)) {
    const Sequence& s = walk.s;
    const int* table = a.block_table + (size_t)walk.seq * a.table_width;
    const int first_key = (s.tile_lo + walk.begin) * KEYS, draft0 = walk.row_tile * tile_drafts;
    const int rows = max(0, min(tile_drafts, min(s.n, a.max_nodes) - draft0)) * a.group;
    const bool split = walk.count < s.tiles;
    for (int begin = a.window > 0 ? 0 : max(0, s.held - first_key) / KEYS; begin < walk.count; begin += MOST_LOOKS) {
      const int tiles = min(MOST_LOOKS, walk.count - begin), base = first_key + begin * KEYS;
      meet<2, 32 * WARPS>();
      for (int i = threadIdx.x & (32 * WARPS - 1); i < 4 * tiles; i += 32 * WARPS) bits[i] = 0;
      meet<2, 32 * WARPS>();
#pragma unroll 4
      for (int j = (a.window > 0 ? max(0, s.key_lo - base) : max(0, s.held - base)) + warp; j < min(tiles * KEYS, s.ctx - base); j += WARPS) {
        const long at = key_row(a, table, base + j, walk.head);
        const uint2 v = at < 0 ? make_uint2(0, 0) : *reinterpret_cast<const uint2*>((const bf16*)a.v_pool + at * DIM + 4 * lane);
        if (__any_sync(0xffffffffu, not_finite(v.x) || not_finite(v.y)) && lane == 0) atomicOr(&bits[j >> 5], 1u << (j & 31));
      }
      meet<2, 32 * WARPS>();
      unsigned some = 0;
      for (int w = 0; w < 4 * tiles; ++w) some |= bits[w];
      if (!some) continue;
#pragma unroll 1
      for (int r = warp; r < rows; r += WARPS) {
        const int draft = r / a.group, member = r - draft * a.group, token = s.first + draft0 + draft, row_head = walk.head * a.group + member;
        const long row = (long)token * a.q_heads + row_head;
        const int local = ROWS2 && draft >= a.tile_drafts ? ROWS + (draft - a.tile_drafts) * a.group + member : r;
        const long place = ((long)2 * blockIdx.x + (walk.begin == 0 ? 1 : 0)) * (ROWS2 ? 2 * ROWS : ROWS) + local;
        const float2 of = split ? reinterpret_cast<const float2*>(a.partials + a.partial_stats)[place] : a.row_stats[row];
        if (!(of.y > 0.f)) continue;                       // it sees nothing here, or its weights are NaN
        const int oldest = a.window > 0 ? max(a.positions[token], s.held) - a.window + 1 : 0;
        const int* seen = a.tree + (size_t)token * a.tree_words;
        const float4 q = four_values(a.q, row);
        float4 more = make_float4(0.f, 0.f, 0.f, 0.f);
        bool any = false;
#pragma unroll 1
        for (int w = 0; w < 4 * tiles; ++w) {
          if (!bits[w]) continue;
          for (unsigned odd = bits[w] & seen_word(a.tree_words, seen, base + 32 * w, s.held, s.ctx, oldest); odd; odd &= odd - 1) {
            const long at = key_row(a, table, base + 32 * w + __ffs(odd) - 1, walk.head);       // it is there: its values were read
            const float4 k = four_values(a.k_pool, at), v = four_values(a.v_pool, at);
            float z = warp_sum(q.x * k.x + q.y * k.y + q.z * k.z + q.w * k.w);
            if (a.cap_in != 0.f) z = a.cap_out - __fdividef(2.f * a.cap_out, 1.f + fast_exp2(z * a.cap_in));
            const float weight = exp2f(z * a.scale_log2 - of.x) / (split ? 1.f : of.y);
            if (weight != 0.f) { more.x += weight * v.x; more.y += weight * v.y; more.z += weight * v.z; more.w += weight * v.w; }
            any = true;
          }
        }
        if (!any) continue;
        if (split) {
          float4* to = reinterpret_cast<float4*>(a.partials + place * DIM + 4 * lane);
          const float4 x = *to;
          *to = make_float4(x.x + more.x, x.y + more.y, x.z + more.z, x.w + more.w);
        } else {
          const float4 x = four_values(a.out, row);
          *reinterpret_cast<uint2*>((bf16*)a.out + row * DIM + 4 * lane) = make_uint2(pack_bf16(x.x + more.x, x.y + more.y), pack_bf16(x.z + more.z, x.w + more.w));
        }
      }
    }
  }
}

template <bool ROWS2>
__global__ void __launch_bounds__(THREADS, 1)
attention_tree_tcgen05_kernel(const __grid_constant__ CUtensorMap q_map, const __grid_constant__ TreeArgs a) {
  extern __shared__ uint8_t raw_smem[];
  uint8_t* q_s = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~(uintptr_t)1023);      // two tiles: of two segments, or of two halves
  uint8_t* ring = q_s + 2 * TILE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + 2 * STAGES * TILE_BYTES);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * BARRIERS);
  volatile uint32_t* flag = tmem_slot + 1;        // [0] a wait ran out, [1] an output is not finite
  int* start = const_cast<int*>(reinterpret_cast<volatile int*>(flag + 2));      // where the walk begins: sequence, tile of it, tiles
  float2* stats = reinterpret_cast<float2*>(bars + 2 * BARRIERS + 8);      // [2 segments][2 warpgroups][ROWS]
  int4* known = reinterpret_cast<int4*>(stats + 4 * ROWS);                  // first draft, end, keys and tiles of the first sequences

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  auto make_barriers = [&]() {
    for (int i = 0; i < 2 * STAGES; ++i) { mbar_init(&bars[FULL + i], 32 * LOADERS / 2); mbar_init(&bars[EMPTY + i], 1); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&bars[Q_FULL + i], 1); mbar_init(&bars[Q_EMPTY + i], 1); mbar_init(&bars[S_FULL + i], 1); mbar_init(&bars[P_FULL + i], 4); mbar_init(&bars[PV_DONE + i], 1);
    }
    mbar_init(&bars[O_FULL], 1); mbar_init(&bars[O_EMPTY], 8); mbar_init(&bars[STATS_FULL], 8); mbar_init(&bars[STARTED], 1);
  };
  auto publish_barriers = [&]() {
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
  };
  if (threadIdx.x == 32 * LOADERS) {
    make_barriers();
    flag[0] = 0; flag[1] = 0;
    prefetch_map(&q_map);
    publish_barriers();
  }
  __syncwarp();
  if (warp == LOADERS) tmem_alloc(tmem_slot, 512);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem_s = *tmem_slot, tmem_o = tmem_s + 256;      // two of 128 columns each
  const int group = a.group, drafts_tile = a.tile_drafts;      // drafts of 128 rows
  auto ran_out = [&](int code) { atomicCAS(&g_tree_error, 0, code); flag[0] = 1; return false; };
  bool ok = true;
  pdl_launch_dependents();
  // The end of the first pass, for all warps: whether there is a careful one, whose barriers they then turn to. (Each pass has code of its own: as one
  // loop the registers do not suffice.)
  auto careful_pass = [&]() {
    fence_before_sync();
    meet<1, THREADS>();
    fence_after_sync();
    if (flag[0] || !flag[1]) return false;
    bars += BARRIERS;
    if (threadIdx.x == 32 * LOADERS) {
      make_barriers();
      for (int i = 0; i < 2 * STAGES; ++i) mbar_init(&bars[LANDED + i], 32);
      publish_barriers();
    }
    meet<1, THREADS>();
    return true;
  };

  auto load_and_issue = [&](auto careful) {
    if (warp < LOADERS) {
      pdl_wait();
      if (warp == 0) {
        // ---------------- the list's length, then the sequence in which this block's share begins
        int total = 0;
        for (int base = 0; base < a.n_seqs; base += 64) {
          int first[2], end[2], ctx[2];                        // on their way at once
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int seq = min(base + 32 * i + lane, a.n_seqs - 1);
            first[i] = a.cu_q[seq]; end[i] = a.cu_q[seq + 1]; ctx[i] = a.ctx_len[seq];
          }
          int tiles = 0;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int seq = base + 32 * i + lane;
            if (seq < a.n_seqs) {
              const Sequence s = find_sequence<ROWS2>(a, first[i], end[i], ctx[i]);
              const int mine = a.kv_heads * s.row_tiles * s.tiles;
              if (seq < SEQ_CACHE) known[seq] = make_int4(first[i], end[i], ctx[i], mine);
              tiles += mine;
            }
          }
          total += __reduce_add_sync(0xffffffffu, tiles);
        }
        const int blocks = min((int)gridDim.x, total), b = min((int)blockIdx.x, blocks);
        const int from = b < blocks ? share_begin(total, b, blocks) : total, upto = b < blocks ? share_begin(total, b + 1, blocks) : total;
        if (lane == 0) { start[0] = start[1] = 0; start[2] = upto - from; }
        __syncwarp();
        int before = 0;
        for (int base = 0; base < a.n_seqs; base += 32) {
          const int i = base + lane;
          int tiles = 0;
          if (i < a.n_seqs) {
            if (i < SEQ_CACHE) {
              tiles = known[i].w;
            } else {
              const Sequence s = find_sequence<ROWS2>(a, known, i);
              tiles = a.kv_heads * s.row_tiles * s.tiles;
            }
          }
          int sum = tiles;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += other;
          }
          const int mine = before + sum - tiles;
          if (from >= mine && from < mine + tiles) { start[0] = i; start[1] = from - mine; }
          before += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (lane == 0) start[3] = total;
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[STARTED]);
      } else {
        ok = warp_wait(&bars[STARTED], 0) || ran_out(1);
      }
      // ---------------- K or V, and the first of these warps the queries
      const int n_tiles = ok ? start[2] : 0, values = warp >> 1, row0 = (warp & 1) * 64, page_shift = __ffs(a.page_tokens) - 1;
      const bf16* pool = (const bf16*)(values ? a.v_pool : a.k_pool);
      // a lane copies 16 bytes of rows 2 i + (lane >> 4) of each 8 of this warp's rows; `to` are their places in those 8, swizzled
      const uint32_t ring_at = smem_u32(ring) + values * STAGES * TILE_BYTES + ((lane & 15) >> 3) * HALF_BYTES + row0 * 128;
      uint32_t to[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) to[i] = (2 * i + (lane >> 4)) * 128 + (((lane & 7) ^ (2 * i + (lane >> 4))) << 4);
      const long lane_from = (lane >> 4) * DIM + (lane & 15) * 8;
      // Up to four tiles of a segment, whose pages are looked up together, four tiles ahead (a read from memory waits behind all copies
      // in flight): lane 8 j + i has the page of rows 8 i .. of tile j.
      struct Group { int page, key0, count, head, key_lo, ctx, draft, looked_at; } now, soon;
      Walk<ROWS2> ahead;
      ahead.begin_at(a, known, start[0], start[1], n_tiles);
      int tile = 0, segments = 0, taken = 0;
      auto next_group = [&](Group& g) {
        g.count = 0; g.draft = -1;
        if (tile == ahead.count) {
          if (!ahead.next(a)) return;
          tile = 0;
          g.draft = ahead.s.first + ahead.row_tile * (ROWS2 ? 2 : 1) * drafts_tile;      // a segment begins: its queries
        }
        g.count = min(4, ahead.count - tile); g.head = ahead.head; g.key0 = (ahead.s.tile_lo + ahead.begin + tile) * KEYS;
        g.key_lo = ahead.s.key_lo; g.ctx = ahead.s.ctx;
        g.looked_at = !careful || values == 0 ? 0x7fffffff : a.window > 0 ? 0 : ahead.s.held - KEYS + 1;      // tiles from here on
        const int key = g.key0 + (lane >> 3) * KEYS + row0 + (lane & 7) * 8, index = key >> page_shift;
        g.page = index < a.table_width && key < g.ctx ? a.block_table[(size_t)ahead.seq * a.table_width + index] : -1;
        tile += g.count;
      };
      next_group(now);
      while (ok && now.count > 0) {
        next_group(soon);
        if (warp == 0 && now.draft >= 0) {
          const int buf = ROWS2 ? 0 : segments & 1;
          ok = warp_wait(&bars[Q_EMPTY + buf], ((ROWS2 ? segments : segments >> 1) & 1) ^ 1) || ran_out(2);
          if (!ok) break;
          const uint32_t bar = smem_u32(&bars[Q_FULL + buf]);
          expect_bytes(bar, (uint32_t)(drafts_tile * group * 128) * (ROWS2 ? 4 : 2));
          const int head = warp_uniform(now.head * group), draft = warp_uniform(now.draft);
          for (int part = 0; part < (ROWS2 ? 2 : 1); ++part)
            for (int h = 0; h < 2; ++h)
              load_queries(smem_u32(q_s) + (ROWS2 ? part : buf) * TILE_BYTES + h * HALF_BYTES, &q_map, bar, h * 64, head, draft + part * drafts_tile);
          ++segments;
        }
        // the places in the pool of the rows that begin the eights; -1: the page is not there
        const int first = (unsigned)now.page < (unsigned)a.n_pages
                              ? (now.page * a.kv_heads + now.head) * a.page_tokens + ((row0 + (lane & 7) * 8) & (a.page_tokens - 1)) : -1;
        const unsigned there = __ballot_sync(0xffffffffu, first >= 0);
        for (int j = 0; j < now.count; ++j) {
          const int stage = taken % STAGES, key0 = now.key0 + j * KEYS;
          ok = warp_wait(&bars[EMPTY + values * STAGES + stage], ((taken / STAGES) & 1) ^ 1) || ran_out(1);
          if (!ok || flag[0]) { ok = false; break; }
          const uint32_t at = ring_at + stage * TILE_BYTES;
          if ((there >> (8 * j) & 0xFFu) == 0xFFu && key0 >= now.key_lo && key0 + KEYS <= now.ctx) {
#pragma unroll
            for (int g = 0; g < 8; ++g) {
              const bf16* from = pool + (long)__shfl_sync(0xffffffffu, first, 8 * j + g) * DIM + lane_from;
#pragma unroll
              for (int i = 0; i < 4; ++i) copy16(at + to[i] + g * 1024, from + 2 * i * DIM);
            }
          } else {
#pragma unroll 1
            for (int g = 0; g < 8; ++g) {
              const int row = __shfl_sync(0xffffffffu, first, 8 * j + g);
              const bf16* from = pool + (row < 0 ? 0 : (long)row * DIM + lane_from);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int key = key0 + row0 + g * 8 + 2 * i + (lane >> 4);
                const bool wanted = row >= 0 && key < now.ctx && key >= now.key_lo;
                copy16_or_zeros(at + to[i] + g * 1024, wanted ? from + 2 * i * DIM : pool, wanted ? 16 : 0);
              }
            }
          }
          arrive_when_copied(smem_u32(key0 < now.looked_at ? &bars[FULL + values * STAGES + stage] : &bars[LANDED + (warp & 1) * STAGES + stage]));
          ++taken;
        }
        now = soon;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp == LOADERS) {
      // ---------------- the products, turn by turn; the scores are two turns ahead
      pdl_wait();
      ok = warp_wait(&bars[STARTED], 0) || ran_out(2);
      const int n_tiles = ok ? start[2] : 0;
      Walk<ROWS2> ahead, walk;
      ahead.begin_at(a, known, start[0], start[1], n_tiles);
      walk.begin_at(a, known, start[0], start[1], n_tiles);
      const int turns = warp_uniform(n_tiles * (ROWS2 ? 2 : 1));
      int k_taken = 0, v_taken = 0, k_stage = 0, v_stage = 0;
      int a_left = 0, a_segment = -1, g_left = 0, g_turn = 0, g_segment = -1;
      // turn -2 and -1 have scores to be made and no second product: the loop holds each kind of product once
#pragma unroll 1
      for (int t = -2; t < turns && ok; ++t) {
        const int w = t & 1;
        if (t >= 0) {
          if (g_left == 0) {
            walk.next(a);
            g_left = warp_uniform(ROWS2 ? 2 * walk.count : walk.count);
            g_turn = 0;
            ++g_segment;
            if (g_segment > 0) ok = warp_wait(&bars[O_EMPTY], (g_segment - 1) & 1) || ran_out(8);
          }
          if (ok && (!ROWS2 || w == 0)) {
            v_stage = STAGES + v_taken % STAGES;
            ok = warp_wait(&bars[FULL + v_stage], (v_taken / STAGES) & 1) || ran_out(4);
            ++v_taken;
            fence_async_smem();                              // what cp.async wrote is read by the tensor cores
          }
          ok = ok && (warp_wait(&bars[P_FULL + w], (t >> 1) & 1) || ran_out(5));
          if (!ok) break;
          fence_after_sync();
          const uint32_t v_addr = smem_u32(ring + v_stage * TILE_BYTES);
#pragma unroll
          for (int ks = 0; ks < KEYS / 16; ++ks)            // 16 keys: 8 columns of weights, 16 rows of V
            umma_from_tmem(tmem_o + w * 128, tmem_s + w * 128 + ks * 8, desc_mn_major(v_addr + ks * 16 * 128), IDESC_O, (g_turn > 1 || ks > 0) ? 1u : 0u);
          umma_commit(&bars[PV_DONE + w]);
          if (!ROWS2 || w == 1) umma_commit(&bars[EMPTY + v_stage]);
          ++g_turn;
          if (--g_left == 0) umma_commit(&bars[O_FULL]);
        }
        if (t + 2 < turns) {
          if (a_left == 0) {
            ahead.next(a);
            a_left = warp_uniform(ROWS2 ? 2 * ahead.count : ahead.count);
            ++a_segment;
            ok = warp_wait(&bars[Q_FULL + (ROWS2 ? 0 : a_segment & 1)], (ROWS2 ? a_segment : a_segment >> 1) & 1) || ran_out(2);
          }
          if (ok && (!ROWS2 || w == 0)) {
            k_stage = k_taken % STAGES;
            ok = warp_wait(&bars[FULL + k_stage], (k_taken / STAGES) & 1) || ran_out(3);
            ++k_taken;
            fence_async_smem();
          }
          if (!ok) break;
          fence_after_sync();
          const uint32_t q_addr = smem_u32(q_s + (ROWS2 ? w : a_segment & 1) * TILE_BYTES), k_addr = smem_u32(ring + k_stage * TILE_BYTES);
#pragma unroll
          for (int ks = 0; ks < DIM / 16; ++ks) {
            const uint32_t off = (ks >> 2) * HALF_BYTES + (ks & 3) * 32;
            umma_bf16(tmem_s + w * 128, desc_k_major(q_addr + off), desc_k_major(k_addr + off), IDESC_S, ks > 0 ? 1u : 0u);
          }
          umma_commit(&bars[S_FULL + w]);
          if (!ROWS2 || w == 1) umma_commit(&bars[EMPTY + k_stage]);
          if (--a_left == 0) umma_commit(&bars[Q_EMPTY + (ROWS2 ? 0 : a_segment & 1)]);
        }
      }
    } else if (warp > LOADERS + 1) {
      // ---------------- the careful pass: values that may not be seen by all rows, each warp what one of the loading warps copied
      if (careful) {
        const int part = warp - LOADERS - 2, row0 = part * 64;
        ok = warp_wait(&bars[STARTED], 0) || ran_out(9);
        Walk<ROWS2> walk;
        walk.begin_at(a, known, start[0], start[1], ok ? start[2] : 0);
        int taken = 0;
        unsigned phases = 0;                                 // a bit a stage
        while (ok && walk.next(a)) {
          const int first_key = (walk.s.tile_lo + walk.begin) * KEYS;
          for (int j = a.window > 0 ? 0 : max(0, walk.s.held - first_key) / KEYS; j < walk.count && ok; ++j) {
            const int stage = (taken + j) % STAGES, key0 = first_key + j * KEYS;
            ok = warp_wait(&bars[LANDED + part * STAGES + stage], phases >> stage & 1u) || ran_out(9);
            phases ^= 1u << stage;
            const int from = a.window > 0 ? row0 : max(row0, walk.s.held - key0);      // without a window every row sees what is held
            clear_odd_rows(smem_u32(ring + (STAGES + stage) * TILE_BYTES), from, min(walk.s.ctx - key0, row0 + 64));
            fence_async_smem();                              // zeros are read by the tensor cores
            mbar_arrive(&bars[FULL + STAGES + stage]);              // for a lane of the loading warp
          }
          taken += walk.count;
        }
      }
    } else if (warp == LOADERS + 1) {
      // ---------------- for the kernel that joins: the row tile inside which this block's share begins, if it is the first that does
      pdl_wait();
      ok = warp_wait(&bars[STARTED], 0) || ran_out(2);
      Walk<ROWS2> walk;
      walk.begin_at(a, known, start[0], start[1], ok ? start[2] : 0);
      Border border = {};
      if (walk.next(a) && walk.begin > 0) {
        const int total = start[3], shares = min((int)gridDim.x, total), unit = share_begin(total, blockIdx.x, shares) - walk.begin;
        border.from = share_of(total, unit, shares);
        border.upto = share_of(total, unit + walk.s.tiles - 1, shares);
        if (border.from + 1 == (int)blockIdx.x) {
          border.draft = walk.row_tile * (ROWS2 ? 2 : 1) * drafts_tile;
          border.drafts = min(min(walk.s.n, a.max_nodes) - border.draft, (ROWS2 ? 2 : 1) * drafts_tile);
          border.seq = walk.seq; border.head = walk.head; border.token = walk.s.first + border.draft;
        }
      }
      if (lane == 0) a.borders[blockIdx.x] = border;
    }
  };
  auto softmax = [&](auto careful) {
    // ---------------- softmax: one row a thread
    const int wg = (warp - FIRST_SOFTMAX) >> 2, quarter = warp & 3, lane_row = quarter * 32 + lane;
    const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
    const uint32_t my_s = tmem_s + wg * 128 + lane_addr, my_o = tmem_o + wg * 128 + lane_addr;
    const float c = a.scale_log2;
    // Segment -1 is a turn on nothing, of which every warp goes through a part (masks and maximum, weights, rescaling and values, the
    // segment's end) and whose result nobody takes: their instructions are fetched side by side while the first loads are under way.
    Walk<ROWS2> g;
    g.begin_at(a, known, 0, 0, 0);
    g.begin = g.row_tile = g.head = g.seq = 0; g.s = Sequence{};
    int turn0 = 0, n_tiles = 0;                            // the segment's first turn; the block's tiles
    for (int k = careful ? 0 : -1; ok; ++k) {
      const bool dry = k < 0;
      if (k == 0) {
        pdl_wait();
        ok = mbar_wait(&bars[STARTED], 0) || ran_out(6);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        n_tiles = start[2];
        g.begin_at(a, known, start[0], start[1], n_tiles);
      }
      if (!dry && !g.next(a)) break;
      const int turns = dry ? 2 : ROWS2 ? 2 * g.count : g.count, held = dry ? 1 : g.s.held, ctx = dry ? KEYS - 1 : g.s.ctx, key_lo = dry ? 0 : g.s.key_lo;
      const int first_key = dry ? 0 : (g.s.tile_lo + g.begin) * KEYS, tree_words = dry ? 0 : a.tree_words;
      const int draft0 = dry ? 0 : (g.row_tile * (ROWS2 ? 2 : 1) + (ROWS2 ? wg : 0)) * drafts_tile;
      const int rows = dry ? ROWS : max(0, min(drafts_tile, min(g.s.n, a.max_nodes) - draft0)) * group;       // of this warpgroup
      const bool live = quarter * 32 < rows, valid = !dry && lane_row < rows;
      const int draft = lane_row / group, row_head = dry ? 0 : g.head * group + lane_row - draft * group;
      const int token = dry ? 0 : g.s.first + (valid ? draft0 + draft : 0);
      const int* bits = a.tree + (size_t)token * a.tree_words;
      const int oldest = a.window > 0 && !dry ? max(a.positions[token], held) - a.window + 1 : 0;
      // the words of the tree that the segment's last tile needs are under way until then
      const int last_key = first_key + (dry ? 0 : g.count - 1) * KEYS, last_draft = last_key - held, last_word = last_draft >> 5;
      uint32_t tree_bits[5];
#pragma unroll
      for (int i = 0; i < 5; ++i) {
        const int w = last_word + i;
        tree_bits[i] = w >= 0 && w < tree_words ? (uint32_t)bits[w] : 0u;
      }
      float m_ref = -INFINITY, l_sum = 0.f;
      const int t_first = turn0 + ((turn0 ^ wg) & 1);      // this warpgroup's first turn
      for (int t = t_first; t < turn0 + turns && ok; t += 2) {
        const int tile = ROWS2 ? (t - turn0) >> 1 : t - turn0, key0 = first_key + tile * KEYS, j = t >> 1;
        const bool masked = (key0 + KEYS > held || key0 < key_lo || a.window > 0) && (!dry || quarter == 0);
        uint32_t words[4];
        if (masked) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            words[i] = key0 == last_key ? seen_word(__funnelshift_r(tree_bits[i], tree_bits[i + 1], last_draft & 31), key0 + 32 * i, held, ctx, oldest)
                                        : seen_word(tree_words, bits, key0 + 32 * i, held, ctx, oldest);
        }
        // a warp without rows waits as well: the turn before has been handed on by all four by then
        ok = dry || mbar_wait(&bars[S_FULL + wg], j & 1) || ran_out(6);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        fence_after_sync();
        if (live) {
          float s[KEYS];
          float top = -INFINITY;
          tmem_ld128(my_s, s);
          if (!dry || quarter == 0) {
            if (a.cap_in != 0.f) {
#pragma unroll
              for (int e = 0; e < KEYS; ++e) s[e] = a.cap_out - __fdividef(2.f * a.cap_out, 1.f + fast_exp2(s[e] * a.cap_in));
            }
            if (masked) {
#pragma unroll
              for (int e = 0; e < KEYS; ++e)
                if (!(words[e >> 5] >> (e & 31) & 1u)) s[e] = -INFINITY;
            }
            top = row_max(s);
          }
          const bool grow = (top - m_ref) * c > GROWTH || (m_ref == -INFINITY && top > -INFINITY);
          const bool any_grow = __any_sync(0xffffffffu, grow);
          const float m_new = grow ? top : m_ref;
          const float factor = m_ref == -INFINITY ? 0.f : fast_exp2((m_ref - m_new) * c);
          const float neg_base = m_new == -INFINITY ? 0.f : -m_new * c;
          m_ref = m_new;
          if (!dry || quarter == 1) {
            float sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int part = 0; part < 4; ++part) {
              uint32_t w[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) {
                const float x = fast_exp2(fmaf(s[part * 32 + 2 * e], c, neg_base)), y = fast_exp2(fmaf(s[part * 32 + 2 * e + 1], c, neg_base));
                sums[e & 3] += x + y;
                w[e] = pack_bf16(x, y);
              }
              if (!dry) tmem_st16(my_s + part * 16, w);
            }
            l_sum = l_sum * factor + ((sums[0] + sums[1]) + (sums[2] + sums[3]));
          }
          if ((any_grow && t > t_first) || (dry && quarter == 2)) {
            ok = dry || mbar_wait(&bars[PV_DONE + wg], (j - 1) & 1) || ran_out(7);
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            fence_after_sync();
#pragma unroll 2
            for (int ch = 0; ch < DIM / 16; ++ch) {
              float v[16];
              uint32_t r[16];
              tmem_ld16(my_o + ch * 16, v);
#pragma unroll
              for (int e = 0; e < 16; ++e) r[e] = __float_as_uint(v[e] * factor);
              tmem_st16(my_o + ch * 16, r);
            }
          }
          tmem_wait_st();
        }
        fence_before_sync();
        __syncwarp();
        if (lane == 0 && !dry) mbar_arrive(&bars[P_FULL + wg]);
      }
      if (!ok) break;
      if (dry && quarter != 3) continue;

      // ---- the segment's result: with turns of both warpgroups each takes half the channels of both accumulators
      float2* pair = stats + (k & 1) * 2 * ROWS;
      const bool both = !ROWS2 && turns > 1;
      if (!dry) {
        pair[wg * ROWS + lane_row] = make_float2(m_ref, l_sum);
        __syncwarp();
        if (lane == 0) mbar_arrive(&bars[STATS_FULL]);
        ok = (mbar_wait(&bars[STATS_FULL], k & 1) || ran_out(7)) && (mbar_wait(&bars[O_FULL], k & 1) || ran_out(8));
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      }
      fence_after_sync();
      auto release = [&]() {                               // the accumulators may be written again
        fence_before_sync();
        __syncwarp();
        if (lane == 0 && !dry) mbar_arrive(&bars[O_EMPTY]);
      };
      // relative to one maximum: this warpgroup's accumulator by `mine`, the other's by `other`
      float mine = 1.f, other = 0.f;
      if (!ROWS2) {
        const float2 ml = pair[(wg ^ 1) * ROWS + lane_row];
        const float top = fmaxf(m_ref, ml.x), base = top == -INFINITY ? 0.f : top;
        mine = fast_exp2((m_ref - base) * c);
        other = fast_exp2((ml.x - base) * c);
        l_sum = l_sum * mine + ml.y * other;
        m_ref = top;
      }
      const bool split = g.count < g.s.tiles;
      const float m_log2 = m_ref * c;
      if (live) {
        float inv = 1.f;
        if (!split) {
          float total = l_sum, factor = 1.f, base = m_log2;
          if (a.sinks && valid) {
            const float sink = a.sinks[row_head] * LOG2E, top = fmaxf(m_log2, sink);
            base = top == -INFINITY ? 0.f : top;
            factor = fast_exp2(m_log2 - base);
            total = total * factor + fast_exp2(sink - base);
          }
          inv = total == 0.f ? 0.f : __fdividef(factor, total);
          if (careful && valid && (ROWS2 || wg == 0)) a.row_stats[(size_t)token * a.q_heads + row_head] = make_float2(base, total);
        }
        // 64 channels at a time: all of its own rows, or, where the rows are both warpgroups', half; `first_acc`: the accumulator of the
        // segment's first turn. The accumulators are free as soon as they lie in registers.
        const uint32_t first_acc = tmem_o + (ROWS2 ? wg : turn0 & 1) * 128 + lane_addr, second_acc = tmem_o + (~turn0 & 1) * 128 + lane_addr;
        const float by_first = (ROWS2 || (turn0 & 1) == wg ? mine : other) * inv, by_second = ((turn0 & 1) == wg ? other : mine) * inv;
        const long at = ((long)2 * blockIdx.x + (g.begin == 0 ? 1 : 0)) * (ROWS2 ? 2 * ROWS : ROWS) + (ROWS2 ? wg * ROWS : 0) + lane_row;
        float* part = a.partials + at * DIM;
        bf16* out = (bf16*)a.out + ((size_t)token * a.q_heads + row_head) * DIM;
#pragma unroll 1
        for (int half = ROWS2 ? 0 : wg; half < (ROWS2 ? 2 : wg + 1); ++half) {
          float v[64];
          tmem_ld64(first_acc + half * 64, v);
          if (both) {
            float x[64];
            tmem_ld64(second_acc + half * 64, x);
            if (!ROWS2) release();
#pragma unroll
            for (int e = 0; e < 64; ++e) v[e] = v[e] * by_first + x[e] * by_second;
          } else {
            if (!ROWS2 || half == 1) release();
#pragma unroll
            for (int e = 0; e < 64; ++e) v[e] *= by_first;
          }
          bool bad = false;                                // x - x is 0 for what is finite
          {
            float zero[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 64; ++e) zero[e & 3] += v[e] - v[e];
            bad = valid && !((zero[0] + zero[1]) + (zero[2] + zero[3]) == 0.f);
          }
          if (valid) {
            if (split) {
#pragma unroll
              for (int piece = 0; piece < 8; ++piece) {
                uint32_t w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = __float_as_uint(v[piece * 8 + e]);
                store32(part + half * 64 + piece * 8, w);
              }
            } else {
#pragma unroll
              for (int piece = 0; piece < 4; ++piece) {
                uint32_t w[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) w[e] = pack_bf16(v[piece * 16 + 2 * e], v[piece * 16 + 2 * e + 1]);
                store32(out + half * 64 + piece * 16, w);
              }
            }
          }
          if (bad) flag[1] = 1;
        }
        if (valid && split && (ROWS2 || wg == 0)) *reinterpret_cast<float2*>(a.partials + a.partial_stats + at * 2) = make_float2(m_log2, l_sum);
      } else {
        release();
      }
      if (!dry) turn0 += turns;
    }
  };
  if (warp < FIRST_SOFTMAX) {
    give_registers<FEW_REGS>();
    load_and_issue(std::false_type{});
    if (careful_pass()) load_and_issue(std::true_type{});
  } else {
    take_registers<MANY_REGS>();
    softmax(std::false_type{});
    if (careful_pass()) {
      softmax(std::true_type{});
      if (!meet_any<2, 256>(flag[0] != 0)) add_odd_values<ROWS2>(a, known, start, reinterpret_cast<unsigned*>(stats), warp - FIRST_SOFTMAX);
    }
  }

  // ---------------- teardown
  fence_before_sync();
  __syncthreads();
  if (flag[0]) {
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);     // let copies in flight land
    __syncthreads();
  }
  if (warp == LOADERS) {
    fence_after_sync();
    tmem_dealloc(tmem_s, 512);
  }
}

// The parts of the rows whose keys lie in several blocks' shares, in the order of the keys: eight lanes a row, 16 channels each.
constexpr int JOIN_THREADS = 256, JOIN_ROWS = JOIN_THREADS / 8;
template <bool ROWS2>
__global__ void __launch_bounds__(JOIN_THREADS, ROWS2 ? 2 : 4) join_kernel(const __grid_constant__ TreeArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  const Border border = a.borders[blockIdx.x];
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.y * JOIN_ROWS + (threadIdx.x >> 3), rows = border.drafts * a.group;
  if (rows > blockIdx.y * JOIN_ROWS) {
    const int draft = row / a.group, member = row - draft * a.group, row_head = border.head * a.group + member;
    const int local = min(ROWS2 && draft >= a.tile_drafts ? ROWS + (draft - a.tile_drafts) * a.group + member : row, (ROWS2 ? 2 * ROWS : ROWS) - 1);
    const int channel = 4 * (lane & 7);                    // and 32, 64, 96 behind it
    auto place = [&](int p) { return ((long)2 * p + (p == border.from ? 1 : 0)) * (ROWS2 ? 2 * ROWS : ROWS) + local; };
    const float2* stats = reinterpret_cast<const float2*>(a.partials + a.partial_stats);
    float top = a.sinks && row < rows ? a.sinks[row_head] * LOG2E : -INFINITY, total = a.sinks ? 1.f : 0.f;
    float4 sum[4] = {};
    // Parts on their way: tiles of 256 rows are few and have many (2 requests x 64 drafts after 12,345, us for two and four at once: 47.1, 45.6).
    constexpr int AT_ONCE = ROWS2 ? 4 : 2;
    for (int p0 = border.from; p0 <= border.upto; p0 += AT_ONCE) {
      float2 ml[AT_ONCE];
      float4 v[AT_ONCE][4];
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        const long at = place(min(p0 + j, border.upto));
        ml[j] = stats[at];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[j][i] = *reinterpret_cast<const float4*>(a.partials + at * DIM + channel + 32 * i);
        if (p0 + j > border.upto) ml[j].x = -INFINITY;
      }
      float m = top;
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) m = fmaxf(m, ml[j].x);
      const float base = m == -INFINITY ? 0.f : m, keep = exp2f(top - base);
      total *= keep;
#pragma unroll
      for (int i = 0; i < 4; ++i) { sum[i].x *= keep; sum[i].y *= keep; sum[i].z *= keep; sum[i].w *= keep; }
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        const float w = exp2f(ml[j].x - base);
        if (w == 0.f && ml[j].y == ml[j].y) continue;      // a part without a score that is a number has no maximum, and a sum of NaN
        total += w * ml[j].y;
#pragma unroll
        for (int i = 0; i < 4; ++i) { sum[i].x += w * v[j][i].x; sum[i].y += w * v[j][i].y; sum[i].z += w * v[j][i].z; sum[i].w += w * v[j][i].w; }
      }
      top = m;
    }
    if (row < rows) {
      const float inv = total == 0.f ? 0.f : 1.f / total;
      bf16* to = (bf16*)a.out + ((size_t)(border.token + draft) * a.q_heads + row_head) * DIM + channel;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<uint2*>(to + 32 * i) = make_uint2(pack_bf16(sum[i].x * inv, sum[i].y * inv), pack_bf16(sum[i].z * inv, sum[i].w * inv));
    }
  }
}

// The queries [tokens][q_heads][128]: 128 / group drafts with their heads of a group, 64 channels.
static bool query_map(CUtensorMap* map, const void* q, long tokens, int q_heads, int group) {
  auto encode = encode_fn();
  if (!encode) return false;
  cuuint64_t dims[3] = {DIM, (cuuint64_t)q_heads, (cuuint64_t)tokens}, strides[2] = {DIM * 2, (cuuint64_t)q_heads * DIM * 2};
  cuuint32_t box[3] = {64, (cuuint32_t)group, (cuuint32_t)(ROWS / group)}, elem[3] = {1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(q), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// scratch of `blocks` blocks, in floats: two places each of the partial outputs, their maxima and sums; the borders; the rows' maxima and sums
static long scratch_floats(int blocks, bool rows2, long rows) { return 2L * blocks * (rows2 ? 2 * ROWS : ROWS) * (DIM + 2) + 8L * blocks + 2 * rows; }

template <bool ROWS2>
int launch(TreeArgs a, int blocks, cudaStream_t stream) {
  CUtensorMap q_map;
  const int group = a.q_heads / a.kv_heads;
  if (!query_map(&q_map, a.q, a.tokens, a.q_heads, group)) return LB_ERR_SIZE;
  static LbPerDeviceOnce once;
  if (!once.run(LB_ALLOW_SMEM(attention_tree_tcgen05_kernel<ROWS2>, SMEM_BYTES))) return lb_last_error();
  const long slots = 2L * blocks * (ROWS2 ? 2 * ROWS : ROWS);
  a.partial_stats = slots * DIM;
  a.borders = reinterpret_cast<Border*>(a.partials + slots * (DIM + 2));
  a.row_stats = reinterpret_cast<float2*>(a.borders + blocks);
  a.group = group; a.tile_drafts = ROWS / group;
  int code = lb_launch(attention_tree_tcgen05_kernel<ROWS2>, blocks, THREADS, SMEM_BYTES, stream, q_map, a);
  if (code) return code;
  const int rows = min(a.max_nodes, a.tile_drafts * (ROWS2 ? 2 : 1)) * group;
  return lb_launch(join_kernel<ROWS2>, dim3(blocks, (rows + JOIN_ROWS - 1) / JOIN_ROWS), JOIN_THREADS, 0, stream, a);
}
}  // namespace wide
}  // namespace

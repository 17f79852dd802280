// Attention for trees of drafts on the 5th-generation tensor cores: bfloat16, heads of 128 channels, pages of 8 .. 128 tokens.
//
// A block takes up to 128 rows (draft * group + head of the group) of one key/value head and walks its chunk of the keys in tiles of
// 128, dealt in turn to two warpgroups: each has scores and an output accumulator of its own in tensor memory, so one tile's
// softmax runs under the other's products. K and V come page by page (TMA, one copy a lane) through one ring in the order in which the
// products use them: K0, K1, V0, K2, V1, K3, ... The weights overwrite their scores in tensor memory and are the A operand of the
// second product. At the end the two accumulators are joined in shared memory.
//
// Rows that the tree does not have cost nothing but the tensor cores' time: their warps only hand tiles on. What a draft's values
// hold that is not finite is zeroed in the tile and added at the end to the rows that see it.
#pragma once
#include <math.h>

#include "attention_tree.cuh"
#include "tcgen05.cuh"

namespace {

__device__ int g_tree_error = 0;       // 0 = ok; which wait ran out otherwise: 1 ring, 2 queries, 3 keys, 4 values, 5 weights, 6 scores, 7 and 8 second product

namespace wide {

constexpr int ROWS = 128, KEYS = 128, DIM = 128;
constexpr int HALF_BYTES = 128 * 128;           // 64 channels of 128 rows
constexpr int TILE_BYTES = 2 * HALF_BYTES;
constexpr int STAGES = 5;
constexpr int THREADS = 320;                    // warp 0 loads, warp 1 issues the products, warps 2-5 and 6-9 the softmax
constexpr int PAGE_CACHE = 2048;                // block-table entries kept in shared memory
constexpr int JOIN_STRIDE = DIM + 4;            // floats of a row that one warpgroup hands to the other
constexpr int SMEM_BYTES = (1 + STAGES) * TILE_BYTES + 1024 + 512 + PAGE_CACHE * 4;
constexpr float GROWTH = 8.0f;                  // the maximum that weights are relative to may lag by this, in log2 units
static_assert(ROWS * JOIN_STRIDE * 4 + ROWS * 8 <= STAGES * TILE_BYTES, "the joined rows lie in the ring");

__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void load_page(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(smem_u32(dst)), "l"((uint64_t)map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar)) : "memory");
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
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, "
      "%23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
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

// What the drafts' value rows that were zeroed add to 16 channels of a row: their weights anew, from the tensors.
__device__ __noinline__ void add_not_finite(const TreeArgs& a, const Unit& u, const int* table, int from, int upto, int row, int group, int oldest,
                                            float base, int channel, float (&v)[16]) {
  const bf16 *k_pool = (const bf16*)a.k_pool, *v_pool = (const bf16*)a.v_pool;
  const int token = u.first + row / group;
  const bf16* q = (const bf16*)a.q + ((size_t)token * a.q_heads + u.head * group + row % group) * DIM;
  const int* bits = a.tree + (size_t)token * a.tree_words;
  for (int key = max(from, u.held); key < upto; ++key) {
    if (!sees(a, bits, key, u.held, oldest)) continue;
    const long at = key_row(a, table, key, u.head);
    if (at < 0) continue;
    bool bad = false;
    for (int c = 0; c < DIM; c += 2) bad |= not_finite(*reinterpret_cast<const uint32_t*>(v_pool + at * DIM + c));
    if (!bad) continue;
    float s = 0.f;
    for (int c = 0; c < DIM; ++c) s += __bfloat162float(q[c]) * __bfloat162float(k_pool[at * DIM + c]);
    if (a.cap_in != 0.f) s = a.cap_out - __fdividef(2.f * a.cap_out, 1.f + fast_exp2(s * a.cap_in));
    const float w = fast_exp2(fmaf(s, a.scale_log2, -base));
    if (w == 0.f) continue;
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] += w * __bfloat162float(v_pool[at * DIM + channel + e]);
  }
}

__global__ void __launch_bounds__(THREADS, 1) attention_tree_tcgen05_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                                                                          const TreeArgs a) {
  extern __shared__ uint8_t raw_smem[];
  uint8_t* q_s = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~(uintptr_t)1023);
  uint8_t* ring = q_s + TILE_BYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + STAGES * TILE_BYTES);
  uint64_t* full = bars;              // [STAGES]
  uint64_t* empty = bars + STAGES;    // [STAGES]
  uint64_t* q_full = bars + 2 * STAGES;
  uint64_t* s_full = q_full + 1;      // [2 warpgroups] the scores of a tile are in tensor memory
  uint64_t* p_full = q_full + 3;      // [2] its weights are, and the output is rescaled
  uint64_t* pv_done = q_full + 5;     // [2] its second product is finished
  uint64_t* all_done = q_full + 7;    // every product is
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(q_full + 8);
  volatile uint32_t* flag = tmem_slot + 1;        // [0] a wait ran out, [1] a draft's values are not finite
  int* page_cache = reinterpret_cast<int*>(bars) + 128;

  pdl_launch_dependents();
  pdl_wait();
  const int seq = blockIdx.y / a.row_tiles;
  const Unit u = find_unit<KEYS>(a, ROWS, seq, blockIdx.y - seq * a.row_tiles, blockIdx.x, blockIdx.z, gridDim.z);
  if (u.rows <= 0 || (int)blockIdx.z >= u.chunks) return;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int group = a.q_heads / a.kv_heads, n_tiles = max(0, u.tile_end - u.tile_begin);
  const int* table = a.block_table + (size_t)seq * a.table_width;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
    mbar_init(q_full, 8);
    for (int i = 0; i < 2; ++i) { mbar_init(&s_full[i], 1); mbar_init(&p_full[i], 4); mbar_init(&pv_done[i], 1); }
    mbar_init(all_done, 1);
    flag[0] = 0; flag[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_async_smem();
  }
  if (warp == 1) tmem_alloc(tmem_slot, 512);
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  const uint32_t tmem_s = *tmem_slot, tmem_o = tmem_s + 256;      // two of 128 columns each
  auto ran_out = [&](int code) { atomicCAS(&g_tree_error, 0, code); flag[0] = 1; return false; };

  float m_ref = -INFINITY, l_sum = 0.f;
  const int wg = (warp - 2) >> 2, quarter = warp & 3, row_local = quarter * 32 + lane;
  const int row = u.row0 + row_local, token = u.first + min(row, u.n * group - 1) / group;
  const int* bits = a.tree + (size_t)token * a.tree_words;
  const int oldest = a.window > 0 ? max(a.positions[token], u.held) - a.window + 1 : 0;
  const uint32_t lane_addr = (uint32_t)(quarter * 32) << 16;
  bool ok = true;

  if (warp == 0) {
    // ---------------- K and V, page by page; pages that are not there lie behind the pool's last and read as zeros
    const int per_tile = KEYS / a.page_tokens, first_page = u.tile_begin * per_tile, last_page = min(a.table_width, (u.ctx + a.page_tokens - 1) / a.page_tokens);
    const int cached = min(n_tiles * per_tile, PAGE_CACHE);
    auto page_at = [&](int i) {
      const int page = i < last_page ? table[i] : -1;
      return (unsigned)page < (unsigned)a.n_pages ? page : a.n_pages;
    };
    for (int i = lane; i < cached; i += 32) page_cache[i] = page_at(first_page + i);
    __syncwarp();
    const int pg = lane >> 1, half = lane & 1;
    int count = 0;
    auto load = [&](int tile, const CUtensorMap* map) {
      const int stage = count % STAGES;
      if (!warp_wait(&empty[stage], ((count / STAGES) & 1) ^ 1)) return ran_out(1);
      if (flag[0]) return false;
      if (lane == 0) mbar_expect_tx(&full[stage], TILE_BYTES);
      __syncwarp();
      if (pg < per_tile) {
        const int local = tile * per_tile + pg, page = local < PAGE_CACHE ? page_cache[local] : page_at(first_page + local);
        load_page(ring + stage * TILE_BYTES + half * HALF_BYTES + pg * a.page_tokens * 128, map, &full[stage], half * 64, 0, u.head, page);
      }
      ++count;
      return true;
    };
    if (n_tiles > 0) ok = load(0, &k_map);
    if (ok && n_tiles > 1) ok = load(1, &k_map);
    for (int i = 0; i < n_tiles && ok; ++i) {
      ok = load(i, &v_map);
      if (ok && i + 2 < n_tiles) ok = load(i + 2, &k_map);
    }
  } else if (warp == 1) {
    // ---------------- the products, in the order of the ring
    const int tiles = warp_uniform(n_tiles);
    int count = 0;
    auto scores = [&](int i) {
      const int stage = count % STAGES, w = i & 1;
      if (!warp_wait(&full[stage], (count / STAGES) & 1)) return ran_out(3);
      fence_after_sync();
      const uint32_t q_addr = smem_u32(q_s), k_addr = smem_u32(ring + stage * TILE_BYTES);
#pragma unroll
      for (int ks = 0; ks < DIM / 16; ++ks) {
        const uint32_t off = (ks >> 2) * HALF_BYTES + (ks & 3) * 32;
        umma_bf16(tmem_s + w * 128, desc_k_major(q_addr + off), desc_k_major(k_addr + off), IDESC_S, ks > 0 ? 1u : 0u);
      }
      umma_commit(&s_full[w]);
      umma_commit(&empty[stage]);
      ++count;
      return true;
    };
    if (tiles > 0) ok = (warp_wait(q_full, 0) || ran_out(2)) && scores(0);
    if (ok && tiles > 1) ok = scores(1);
    for (int i = 0; i < tiles && ok; ++i) {
      const int stage = count % STAGES, w = i & 1;
      ok = (warp_wait(&full[stage], (count / STAGES) & 1) || ran_out(4)) && (warp_wait(&p_full[w], (i >> 1) & 1) || ran_out(5));
      if (!ok) break;
      fence_after_sync();
      const uint32_t v_addr = smem_u32(ring + stage * TILE_BYTES);
#pragma unroll
      for (int ks = 0; ks < KEYS / 16; ++ks)              // 16 keys: 8 columns of weights, 16 rows of V
        umma_from_tmem(tmem_o + w * 128, tmem_s + w * 128 + ks * 8, desc_mn_major(v_addr + ks * 16 * 128), IDESC_O, (i > 1 || ks > 0) ? 1u : 0u);
      umma_commit(&pv_done[w]);
      umma_commit(&empty[stage]);
      ++count;
      if (i + 2 < tiles) ok = scores(i + 2);
    }
    if (ok) umma_commit(all_done);
  } else {
    // ---------------- the queries, swizzled as the products read them; rows that are not there are zeros
    {
      const bf16* q = (const bf16*)a.q;
      const int t = threadIdx.x - 64;
      uint4 w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = (t + i * 256) >> 4, c = t & 15, at = u.row0 + r;
        w[i] = make_uint4(0, 0, 0, 0);
        if (r < u.rows) w[i] = *reinterpret_cast<const uint4*>(q + ((size_t)(u.first + at / group) * a.q_heads + u.head * group + at % group) * DIM + c * 8);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = (t + i * 256) >> 4, c = t & 15;
        *reinterpret_cast<uint4*>(q_s + (c >> 3) * HALF_BYTES + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = w[i];
      }
      fence_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);
    }
    // ---------------- softmax: one row a thread, every other tile a warpgroup
    const uint32_t my_s = tmem_s + wg * 128 + lane_addr, my_o = tmem_o + wg * 128 + lane_addr;
    const bool live = quarter * 32 < u.rows;              // whether this warp has a row at all
    const float c = a.scale_log2;
    for (int i = wg; i < n_tiles && ok; i += 2) {
      const int j = i >> 1, key0 = (u.tile_begin + i) * KEYS;
      // value rows of keys that are not there, or that nobody may see, may hold anything: zeroed, since 0 x NaN is NaN
      const bool drafts = key0 + KEYS > u.held, edge = drafts || key0 < u.key_lo;
      // a warp without rows waits as well: the tile before has been handed on by all four by then
      ok = mbar_wait(&s_full[wg], j & 1) || ran_out(6);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      fence_after_sync();
      if (live) {
        float s[KEYS];
#pragma unroll
        for (int part = 0; part < 4; ++part) {
          uint32_t raw[32];
          tmem_ld32(my_s + part * 32, raw);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 32; ++e) s[part * 32 + e] = __uint_as_float(raw[e]);
        }
        if (a.cap_in != 0.f) {
#pragma unroll
          for (int e = 0; e < KEYS; ++e) s[e] = a.cap_out - __fdividef(2.f * a.cap_out, 1.f + fast_exp2(s[e] * a.cap_in));
        }
        if (edge || a.window > 0) {
#pragma unroll
          for (int part = 0; part < 4; ++part) {
            const uint32_t word = seen_word(a, bits, key0 + part * 32, u.held, u.ctx, oldest);
#pragma unroll
            for (int e = 0; e < 32; ++e)
              if (!(word >> e & 1u)) s[part * 32 + e] = -INFINITY;
          }
        }
        const float top = row_max(s);
        const bool grow = (top - m_ref) * c > GROWTH || (m_ref == -INFINITY && top > -INFINITY);
        const bool any_grow = __any_sync(0xffffffffu, grow);
        const float m_new = grow ? top : m_ref;
        const float factor = m_ref == -INFINITY ? 0.f : fast_exp2((m_ref - m_new) * c);
        const float neg_base = m_new == -INFINITY ? 0.f : -m_new * c;
        float sums[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t w[KEYS / 2];
#pragma unroll
        for (int e = 0; e < KEYS / 2; ++e) {
          const float x = fast_exp2(fmaf(s[2 * e], c, neg_base)), y = fast_exp2(fmaf(s[2 * e + 1], c, neg_base));
          sums[e & 3] += x + y;
          w[e] = pack_bf16(x, y);
        }
        l_sum = l_sum * factor + ((sums[0] + sums[1]) + (sums[2] + sums[3]));
        m_ref = m_new;
#pragma unroll
        for (int part = 0; part < 4; ++part) {
          uint32_t piece[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) piece[e] = w[part * 16 + e];
          tmem_st16(my_s + part * 16, piece);
        }
        if (any_grow && j > 0) {
          ok = mbar_wait(&pv_done[wg], (j - 1) & 1) || ran_out(7);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          fence_after_sync();
#pragma unroll
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
      if (edge) {
        const int at = min(n_tiles, 2) + i + min(i, max(0, n_tiles - 2)), stage = at % STAGES;      // V(i)'s place in the ring's order
        ok = mbar_wait(&full[stage], (at / STAGES) & 1) || ran_out(4);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        const int key = key0 + row_local;
        uint8_t* v_row = ring + stage * TILE_BYTES + row_local * 128;
        bool zero = key >= u.ctx || key < u.key_lo;
        if (!zero && key >= u.held) {
          bool bad = false;
#pragma unroll
          for (int piece = 0; piece < 8; ++piece)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint4 x = *reinterpret_cast<const uint4*>(v_row + half * HALF_BYTES + piece * 16);
              bad |= not_finite(x.x) || not_finite(x.y) || not_finite(x.z) || not_finite(x.w);
            }
          if (bad) { zero = true; flag[1] = 1; }
        }
        if (zero) {
#pragma unroll
          for (int piece = 0; piece < 8; ++piece)
#pragma unroll
            for (int half = 0; half < 2; ++half) *reinterpret_cast<uint4*>(v_row + half * HALF_BYTES + piece * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_async_smem();
      }
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[wg]);
    }
    if (n_tiles > 0 && ok) {
      ok = mbar_wait(all_done, 0) || ran_out(8);
      ok = __all_sync(0xffffffffu, ok);
      fence_after_sync();
    }
  }

  // ---------------- the second warpgroup hands its accumulator over
  float* joined = reinterpret_cast<float*>(ring);
  float2* joined_stats = reinterpret_cast<float2*>(ring + ROWS * JOIN_STRIDE * 4);
  const bool softmax_warp = warp >= 2 && quarter * 32 < u.rows;
  if (softmax_warp && wg == 1 && n_tiles > 1 && ok) {
#pragma unroll
    for (int ch = 0; ch < DIM / 16; ++ch) {
      float v[16];
      tmem_ld16(tmem_o + 128 + lane_addr + ch * 16, v);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        *reinterpret_cast<float4*>(joined + row_local * JOIN_STRIDE + ch * 16 + e * 4) = make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
    }
    joined_stats[row_local] = make_float2(m_ref, l_sum);
  }
  __syncthreads();
  if (softmax_warp && wg == 0 && ok && !flag[0]) {
    const float c = a.scale_log2;
    float mine = 1.f, other = 0.f;
    if (n_tiles > 1) {
      const float2 ml = joined_stats[row_local];
      const float top = fmaxf(m_ref, ml.x), base = top == -INFINITY ? 0.f : top;
      mine = fast_exp2((m_ref - base) * c);
      other = fast_exp2((ml.x - base) * c);
      l_sum = l_sum * mine + ml.y * other;
      m_ref = top;
    }
    const bool valid = row_local < u.rows, split = u.chunks > 1, bad = flag[1];
    const float m_log2 = m_ref * c;
    float inv = 1.f;
    if (!split) {
      float total = l_sum, factor = 1.f;
      if (a.sinks) {
        const float sink = a.sinks[u.head * group + row % group] * LOG2E, top = fmaxf(m_log2, sink);
        factor = fast_exp2(m_log2 - top);
        total = total * factor + fast_exp2(sink - top);
      }
      inv = total == 0.f ? 0.f : factor / total;
    }
    const long at = (u.index * gridDim.z + blockIdx.z) * ROWS + row_local;
    bf16* out = (bf16*)a.out + ((size_t)token * a.q_heads + u.head * group + row % group) * DIM;
#pragma unroll 1
    for (int ch = 0; ch < DIM / 16; ++ch) {
      float v[16];
      __syncwarp();                                        // lanes without a row, or with drafts to add, come back together
      if (n_tiles > 0) {
        tmem_ld16(tmem_o + lane_addr + ch * 16, v);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = 0.f;
      }
      if (!valid) continue;
      if (n_tiles > 1) {
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = v[e] * mine + joined[row_local * JOIN_STRIDE + ch * 16 + e] * other;
      }
      if (bad) add_not_finite(a, u, table, u.tile_begin * KEYS, min(u.ctx, u.tile_end * KEYS), row, group, oldest, m_ref == -INFINITY ? 0.f : m_log2, ch * 16, v);
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] *= inv;
      if (split) {
        store_row16(a.partials + at * DIM + ch * 16, v);
      } else {
        store_row16(out + ch * 16, v);
      }
    }
    if (valid && split) *reinterpret_cast<float2*>(a.partials + a.partial_stats + at * 2) = make_float2(m_log2, l_sum);
  }

  // ---------------- teardown
  fence_before_sync();
  __syncthreads();
  if (flag[0]) {
    for (int i = 0; i < 2000; ++i) __nanosleep(1000);     // let copies in flight land
    __syncthreads();
  }
  if (warp == 1) {
    fence_after_sync();
    tmem_dealloc(tmem_s, 512);
  }
}

// A pool [pages][heads][page_tokens][128] of bfloat16: copies of one page's tokens of one head, 64 channels.
static bool pool_map(CUtensorMap* map, const void* pool, long pages, int heads, int page_tokens) {
  auto encode = encode_fn();
  if (!encode) return false;
  cuuint64_t dims[4] = {DIM, (cuuint64_t)page_tokens, (cuuint64_t)heads, (cuuint64_t)pages};
  cuuint64_t strides[3] = {DIM * 2, (cuuint64_t)page_tokens * DIM * 2, (cuuint64_t)heads * page_tokens * DIM * 2};
  cuuint32_t box[4] = {64, (cuuint32_t)page_tokens, 1, 1}, elem[4] = {1, 1, 1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(pool), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

static int launch(const TreeArgs& a, dim3 grid, cudaStream_t stream) {
  CUtensorMap k_map, v_map;
  if (!pool_map(&k_map, a.k_pool, a.n_pages, a.kv_heads, a.page_tokens) || !pool_map(&v_map, a.v_pool, a.n_pages, a.kv_heads, a.page_tokens)) return LB_ERR_SIZE;
  static LbPerDeviceOnce once;
  if (!once.run(LB_ALLOW_SMEM(attention_tree_tcgen05_kernel, SMEM_BYTES))) return lb_last_error();
  return lb_launch(attention_tree_tcgen05_kernel, grid, THREADS, SMEM_BYTES, stream, k_map, v_map, a);
}
}  // namespace wide
}  // namespace

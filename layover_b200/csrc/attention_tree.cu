// Attention for a tree of drafted tokens over the paged cache.
//
// A request holds `held` tokens and brings n drafts that form a tree: their keys and values lie behind the held ones,
// draft j at place held + j. Row t of draft i (one row per draft and query head) attends to
//
//   every held key j < held          (with a window: positions[t] - j < window)
//   the drafts j whose bit is set in tree[t]     (its ancestors and itself, as whoever drafted them says)
//
//   s_j = scale q.k_j,  or cap tanh(scale q.k_j / cap);   o = sum_j e^(s_j - m) v_j / (sum_j e^(s_j - m) + e^(sink - m))
//
// in one pass over the keys with a running maximum and sum in 32 bits. A row that sees no key is zero. The query heads of a
// key/value head and the drafts are the rows of one tile (row = draft * group + head of the group), so every key and value is read
// once for all of them. The reference has no drafts: it decodes one token a request and step (layover/engine.py:176-189).
//
// Blocks: (sequence x row tile x key/value head, the head fastest; chunk of the keys). Chunks have the same number of key tiles for every sequence, so
// blocks take equally long whatever the lengths, and one that lies behind its sequence's end leaves at once. Where there is more
// than one chunk each leaves its maxima, sums and unnormalised outputs in scratch memory of this call, and a second kernel joins them.
//
//   attention_tree_mma_kernel   bfloat16, mma.sync m16n8k16: RG groups of 16 rows, the four warps share a tile's 64 keys
//   attention_tree_f32_kernel   float32, FFMA: 8 x 16 threads, RT / 8 rows and 2 keys (dim / 16 channels) each
//
// The values of a draft may be anything (a draft whose arithmetic overflowed): what a row does not see must not reach it, and
// 0 x NaN is NaN. So in tiles that hold drafts, or held keys that lie behind the window of some row, value rows that are not finite are
// taken out of the product and added one by one to the rows that see them.
//
// The weights round to bfloat16 for the second product of the bfloat16 kernel (see attention_tree_tcgen05.cuh); all else is held in 32 bits.
//
// Bounds. bfloat16: the keys' and values' bytes and, with few keys, the time to start two launches and to reach a page through its
// table; 5 requests of 13 drafts behind a window of 1,024, 12 heads over 2 of 64 channels 16.5 us. 32 bits: 2 x rows x keys x dim FFMA a
// head, 11 us at the pipes' rate for 4 requests of 13 drafts after 900 keys, 32 heads over 8 of 128 (32 MB: 4.9 us), measured 63 us:
// three instructions are issued for every one of those (reads of shared memory, the weights doubled for two products an instruction),
// half of the cycles issue none (waits for shared memory and for sums before). Tiles of 64 keys, two blocks an SM: 74; one product an
// instruction before that 204.
#include <math.h>

#include <type_traits>

#include "attention_tree.cuh"
#include "attention_tree_tcgen05.cuh"
#include "common.cuh"

namespace {

constexpr int THREADS = 128;
constexpr int KEYS = 64;        // keys per tile
constexpr int PAD = 8;          // bf16 of padding per shared-memory row
__device__ __forceinline__ void cp_async16(void* dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(p));
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(p));
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Keys [tile * KEYS, + KEYS) of one head into rows of `stride` elements of T; what lies outside [key_lo, ctx) becomes zeros.
template <int KEYS, typename T>
__device__ __forceinline__ void load_tile(T* to, const T* __restrict__ pool, const TreeArgs& a, const Unit& u, const int* table, int tile, int stride) {
  constexpr int PER = 16 / (int)sizeof(T);
  const int pieces = a.dim / PER;
  int r = threadIdx.x / pieces, c = threadIdx.x - r * pieces;
  const int r_step = THREADS / pieces, c_step = THREADS - r_step * pieces;
  const int shift = (a.page_tokens & (a.page_tokens - 1)) == 0 ? __ffs(a.page_tokens) - 1 : -1;
#pragma unroll 4
  for (int i = threadIdx.x; i < KEYS * pieces; i += THREADS) {
    const int key = tile * KEYS + r;
    long row = -1;
    if (key >= u.key_lo && key < u.ctx) {
      const int index = shift >= 0 ? key >> shift : key / a.page_tokens;
      const int page = index < a.table_width ? table[index] : -1;
      if ((unsigned)page < (unsigned)a.n_pages) row = ((long)page * a.kv_heads + u.head) * a.page_tokens + (key - index * a.page_tokens);
    }
    cp_async16(to + r * stride + c * PER, pool + (row < 0 ? 0 : row * a.dim) + c * PER, row < 0 ? 0 : 16);
    r += r_step; c += c_step;
    if (c >= pieces) { c -= pieces; ++r; }
  }
}

// ------------------------------------------------------------------------------- bfloat16
// A warp owns 16 rows and 64 / KG keys of every tile (KG = 4 / RG warps share a row group's keys and are joined at the end).
template <int RG, int MAX_DIM>
__global__ void __launch_bounds__(THREADS, MAX_DIM == 128 ? 2 : 1) attention_tree_mma_kernel(const TreeArgs a) {
  constexpr int KG = 4 / RG, NT = KEYS / KG / 8, KSTEPS = MAX_DIM / 16, NT_O = MAX_DIM / 8, STAGES = 2;
  extern __shared__ __align__(16) uint8_t smem_raw[];
  __shared__ unsigned bad_rows[4];                         // per 16 keys of a tile that is looked at: value rows that are not finite
  __shared__ int hidden_s[4];                              // per warp: below it are held keys that a row does not see
  const int stride = a.dim + PAD, dk = a.dim >> 4;
  bf16* q_s = reinterpret_cast<bf16*>(smem_raw);           // [16 RG][stride]
  bf16* k_s = q_s + 16 * RG * stride;                      // [STAGES][KEYS][stride]
  bf16* v_s = k_s + STAGES * KEYS * stride;
  pdl_launch_dependents();
  pdl_wait();
  const int row_tile_of = blockIdx.x / a.kv_heads, seq = row_tile_of / a.row_tiles;
  const Unit u = find_unit<KEYS>(a, 16 * RG, seq, row_tile_of - seq * a.row_tiles, blockIdx.x - row_tile_of * a.kv_heads, blockIdx.y, gridDim.y);
  if (u.rows <= 0 || (int)blockIdx.y >= u.chunks) return;
  const int group = a.q_heads / a.kv_heads;
  const int* table = a.block_table + (size_t)seq * a.table_width;
  const bf16 *q = (const bf16*)a.q, *k_pool = (const bf16*)a.k_pool, *v_pool = (const bf16*)a.v_pool;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rg = warp % RG, kg = warp / RG;

  {
    const int pieces = a.dim >> 3;
    for (int i = threadIdx.x; i < 16 * RG * pieces; i += THREADS) {
      const int r = i / pieces, c = i - r * pieces, row = u.row0 + r;
      const bool live = r < u.rows;
      const long at = ((long)(u.first + (live ? row / group : 0)) * a.q_heads + u.head * group + (live ? row % group : 0)) * a.dim + c * 8;
      cp_async16(q_s + r * stride + c * 8, q + at, live ? 16 : 0);
    }
  }
  if (u.tile_begin < u.tile_end) {
    load_tile<KEYS>(k_s, k_pool, a, u, table, u.tile_begin, stride);
    load_tile<KEYS>(v_s, v_pool, a, u, table, u.tile_begin, stride);
  }
  cp_async_commit();

  // the two rows of this lane: their masks, and the oldest held key they see
  const int* bits[2];
  int oldest[2];
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int row = min(u.row0 + rg * 16 + g + 8 * r, u.n * group - 1), token = u.first + row / group;
    bits[r] = a.tree + (size_t)token * a.tree_words;
    oldest[r] = a.window > 0 ? max(a.positions[token], u.held) - a.window + 1 : 0;
  }
  if (a.window > 0) {
    const int most = __reduce_max_sync(0xffffffffu, max(oldest[0], oldest[1]));
    if (lane == 0) hidden_s[warp] = most;
  }
  uint32_t qf[KSTEPS][4];
  float o[NT_O][4];
#pragma unroll
  for (int n = 0; n < NT_O; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.f;
  float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
  // ldmatrix lane addresses: K rows by key, V rows by key with the channel pieces swapped in
  const int key_w = kg * NT * 8;                           // the warp's first key within a tile
  const uint32_t k_lane = smem_u32(k_s) + (uint32_t)((key_w + (lane >> 4) * 8 + (lane & 7)) * stride + ((lane >> 3) & 1) * 8) * 2;
  const uint32_t v_lane = smem_u32(v_s) + (uint32_t)((key_w + ((lane >> 3) & 1) * 8 + (lane & 7)) * stride + (lane >> 4) * 8) * 2;
  const uint32_t buf_bytes = (uint32_t)KEYS * stride * 2;

  for (int tile = u.tile_begin; tile < u.tile_end; ++tile) {
    const int buf = (tile - u.tile_begin) & 1;
    if (tile + 1 < u.tile_end) {
      load_tile<KEYS>(k_s + (buf ^ 1) * KEYS * stride, k_pool, a, u, table, tile + 1, stride);
      load_tile<KEYS>(v_s + (buf ^ 1) * KEYS * stride, v_pool, a, u, table, tile + 1, stride);
      cp_async_commit();
      cp_async_wait<1>();
    } else {
      cp_async_wait<0>();
    }
    __syncthreads();
    if (tile == u.tile_begin) {
#pragma unroll
      for (int k = 0; k < KSTEPS; ++k)
        if (k < dk) ldmatrix_x4(qf[k], smem_u32(q_s + (rg * 16 + (lane & 15)) * stride + k * 16 + (lane >> 4) * 8));
    }
    const int key0 = tile * KEYS;
    const bool drafts = key0 + KEYS > u.held;
    const int hidden = a.window > 0 ? max(max(hidden_s[0], hidden_s[1]), max(hidden_s[2], hidden_s[3])) : 0;
    const bool looked = drafts || key0 < hidden;
    if (looked) {                                          // two threads look at a value row
      bf16* row = v_s + buf * KEYS * stride + (threadIdx.x >> 1) * stride;
      bool bad = false;
      for (int c = (threadIdx.x & 1); c < a.dim >> 3; c += 2) {
        const uint4 w = *reinterpret_cast<const uint4*>(row + c * 8);
        bad |= not_finite(w.x) || not_finite(w.y) || not_finite(w.z) || not_finite(w.w);
      }
      const int key = key0 + (int)(threadIdx.x >> 1);
      const unsigned both = __ballot_sync(0xffffffffu, bad && (key >= u.held || key < hidden));
      unsigned rows = 0;
#pragma unroll
      for (int i = 0; i < 16; ++i) rows |= ((both >> (2 * i)) & 3u) ? 1u << i : 0u;
      if (rows >> (lane >> 1) & 1u)
        for (int c = (threadIdx.x & 1); c < a.dim >> 3; c += 2) *reinterpret_cast<uint4*>(row + c * 8) = make_uint4(0, 0, 0, 0);
      if (lane == 0) bad_rows[warp] = rows;
      __syncthreads();
    }

    // ---- scores
    float s[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
    for (int k = 0; k < KSTEPS; ++k) {
      if (k >= dk) break;
#pragma unroll
      for (int n = 0; n < NT; n += 2) {
        uint32_t b[4];
        ldmatrix_x4(b, k_lane + buf * buf_bytes + (uint32_t)(n * 8 * stride + k * 16) * 2);
        mma_bf16(s[n], qf[k], b[0], b[1]);
        mma_bf16(s[n + 1], qf[k], b[2], b[3]);
      }
    }
    if (a.cap_in != 0.f) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = a.cap_out - __fdividef(2.f * a.cap_out, 1.f + fast_exp2(s[n][e] * a.cap_in));
    }
    if (drafts || key0 < u.key_lo || a.window > 0) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + key_w + n * 8 + 2 * t + (e & 1);
          if (key >= u.ctx || !sees(a, bits[e >> 1], key, u.held, oldest[e >> 1])) s[n][e] = -INFINITY;
        }
    }
    // ---- weights
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      float top = -INFINITY;
#pragma unroll
      for (int n = 0; n < NT; ++n) top = fmaxf(top, fmaxf(s[n][2 * r], s[n][2 * r + 1]));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      top = fmaxf(top, m_run[r]);
      const float base = top == -INFINITY ? 0.f : top * a.scale_log2;
      const float alpha = fast_exp2(m_run[r] * a.scale_log2 - base);       // 0 as long as nothing was seen
      m_run[r] = top;
      float sum = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float w = fast_exp2(fmaf(s[n][2 * r + e], a.scale_log2, -base));
          s[n][2 * r + e] = w;
          sum += w;
        }
      l_run[r] = l_run[r] * alpha + sum;
#pragma unroll
      for (int n = 0; n < NT_O; ++n) { o[n][2 * r] *= alpha; o[n][2 * r + 1] *= alpha; }
    }
    // ---- outputs
#pragma unroll
    for (int k = 0; k < NT / 2; ++k) {                     // 16 keys a step
      const uint32_t p[4] = {pack_bf16(s[2 * k][0], s[2 * k][1]), pack_bf16(s[2 * k][2], s[2 * k][3]),
                             pack_bf16(s[2 * k + 1][0], s[2 * k + 1][1]), pack_bf16(s[2 * k + 1][2], s[2 * k + 1][3])};
#pragma unroll
      for (int n = 0; n < NT_O; n += 2) {
        if (n >= 2 * dk) break;
        uint32_t b[4];
        ldmatrix_x4_trans(b, v_lane + buf * buf_bytes + (uint32_t)(k * 16 * stride + n * 8) * 2);
        mma_bf16(o[n], p, b[0], b[1]);
        mma_bf16(o[n + 1], p, b[2], b[3]);
      }
    }
    if (looked && (bad_rows[0] | bad_rows[1] | bad_rows[2] | bad_rows[3])) {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        for (int i = 0; i < 8; ++i) {
          const int local = key_w + n * 8 + i;
          if (!(bad_rows[local >> 4] >> (local & 15) & 1u)) continue;
          const long from = key_row(a, table, key0 + local, u.head);       // its values were read: it is there
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const float w = __shfl_sync(0xffffffffu, i & 1 ? s[n][2 * r + 1] : s[n][2 * r], (lane & 28) | (i >> 1));
            if (w == 0.f || from < 0) continue;
#pragma unroll
            for (int c = 0; c < NT_O; ++c)
              if (c < 2 * dk) {
                const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(v_pool + from * a.dim + c * 8 + 2 * t));
                o[c][2 * r] += w * v.x;
                o[c][2 * r + 1] += w * v.y;
              }
          }
        }
      }
    }
    __syncthreads();                                       // the buffer is loaded anew by the next step
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 1);
    l_run[r] += __shfl_xor_sync(0xffffffffu, l_run[r], 2);
  }

  // ---- the warps that share a row group's keys are joined, in the order of their keys
  if (KG > 1) {
    float* parts = reinterpret_cast<float*>(k_s);          // [KG - 1][16 RG][dim + 2]: at most 48 rows in the room of 128 keys
    const int width = a.dim + 2;
    if (kg > 0) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float* to = parts + ((kg - 1) * 16 * RG + rg * 16 + g + 8 * r) * width;
#pragma unroll
        for (int n = 0; n < NT_O; ++n)
          if (n < 2 * dk) { to[n * 8 + 2 * t] = o[n][2 * r]; to[n * 8 + 2 * t + 1] = o[n][2 * r + 1]; }
        if (t == 0) { to[a.dim] = m_run[r]; to[a.dim + 1] = l_run[r]; }
      }
    }
    __syncthreads();
    if (kg > 0) return;
#pragma unroll
    for (int r = 0; r < 2; ++r) {
#pragma unroll
      for (int p = 0; p < KG - 1; ++p) {
        const float* from = parts + (p * 16 * RG + rg * 16 + g + 8 * r) * width;
        const float m = from[a.dim], top = fmaxf(m_run[r], m), base = top == -INFINITY ? 0.f : top * a.scale_log2;
        const float mine = fast_exp2(m_run[r] * a.scale_log2 - base), other = fast_exp2(m * a.scale_log2 - base);
        m_run[r] = top;
        l_run[r] = l_run[r] * mine + from[a.dim + 1] * other;
#pragma unroll
        for (int n = 0; n < NT_O; ++n)
          if (n < 2 * dk) {
            o[n][2 * r] = o[n][2 * r] * mine + from[n * 8 + 2 * t] * other;
            o[n][2 * r + 1] = o[n][2 * r + 1] * mine + from[n * 8 + 2 * t + 1] * other;
          }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int local = rg * 16 + g + 8 * r, row = u.row0 + local;
    if (local >= u.rows) continue;
    if (u.chunks > 1) {
      const long at = (u.index * gridDim.y + blockIdx.y) * (16 * RG) + local;
      float* to = a.partials + at * a.dim;
#pragma unroll
      for (int n = 0; n < NT_O; ++n)
        if (n < 2 * dk) *reinterpret_cast<float2*>(to + n * 8 + 2 * t) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
      if (t == 0) *reinterpret_cast<float2*>(a.partials + a.partial_stats + at * 2) = make_float2(m_run[r] * a.scale_log2, l_run[r]);
    } else {
      const int head = u.head * group + row % group;
      float total = l_run[r];
      float factor = 1.f;
      if (a.sinks) {                                       // the sink may be the largest of all, or -inf where nothing is seen either
        const float sink = a.sinks[head] * LOG2E, m = m_run[r] * a.scale_log2, top = fmaxf(m, sink), base = top == -INFINITY ? 0.f : top;
        factor = fast_exp2(m - base);
        total = total * factor + fast_exp2(sink - base);
      }
      const float inv = total == 0.f ? 0.f : factor / total;
      bf16* to = (bf16*)a.out + ((size_t)(u.first + row / group) * a.q_heads + head) * a.dim;
#pragma unroll
      for (int n = 0; n < NT_O; ++n)
        if (n < 2 * dk) *reinterpret_cast<uint32_t*>(to + n * 8 + 2 * t) = pack_bf16(o[n][2 * r] * inv, o[n][2 * r + 1] * inv);
    }
  }
}

// ------------------------------------------------------------------------------- float32
// Two products an instruction: (x, y) += (a, b) (c, d)
__device__ __forceinline__ void fma2(float2& x, float2 a, float2 b) {
  asm("{\n\t.reg .b64 p, q, r;\n\t"
      "mov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %5};\n\tmov.b64 r, {%0, %1};\n\t"
      "fma.rn.f32x2 r, p, q, r;\n\t"
      "mov.b64 {%0, %1}, r;\n\t}"
      : "+f"(x.x), "+f"(x.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
}

constexpr int F32_KEYS = 32;    // keys per tile: four blocks an SM have room for theirs
static_assert(F32_KEYS * 4 == THREADS, "four threads a value row");

// MAX_C: blocks of 64 channels of a head
template <int RT, int MAX_C>
__global__ void __launch_bounds__(THREADS, MAX_C == 2 ? 4 : 2) attention_tree_f32_kernel(const TreeArgs a) {
  constexpr int RPT = RT / 8, KEYS = F32_KEYS, KPT = KEYS / 16;      // rows and keys of a thread
  extern __shared__ __align__(16) float smem_f[];
  __shared__ unsigned bad_rows[4];
  __shared__ int hidden_s[4];
  const int stride = a.dim + 4;                            // rows 16 bytes apart modulo 128: eight rows' pieces lie in different banks
  float* q_s = smem_f;                                     // [RT][stride]
  float* k_s = q_s + RT * stride;                          // [KEYS][stride]
  float* v_s = k_s + KEYS * stride;                        // [KEYS][stride]
  float* p_s = v_s + KEYS * stride;                        // [RT][KEYS + 4]
  constexpr int P_STRIDE = KEYS + 4;
  pdl_launch_dependents();
  pdl_wait();
  const int row_tile_of = blockIdx.x / a.kv_heads, seq = row_tile_of / a.row_tiles;
  const Unit u = find_unit<KEYS>(a, RT, seq, row_tile_of - seq * a.row_tiles, blockIdx.x - row_tile_of * a.kv_heads, blockIdx.y, gridDim.y);
  if (u.rows <= 0 || (int)blockIdx.y >= u.chunks) return;
  const int group = a.q_heads / a.kv_heads;
  const int* table = a.block_table + (size_t)seq * a.table_width;
  const float *q = (const float*)a.q, *k_pool = (const float*)a.k_pool, *v_pool = (const float*)a.v_pool;
  const int ty = threadIdx.x >> 4, tx = threadIdx.x & 15;  // rows ty + 8 i, keys tx + 16 j, channels 64 c + 4 tx ..
  {
    const int pieces = a.dim >> 2;
    for (int i = threadIdx.x; i < RT * pieces; i += THREADS) {
      const int r = i / pieces, c = i - r * pieces, row = u.row0 + r;
      const bool live = r < u.rows;
      const long at = ((long)(u.first + (live ? row / group : 0)) * a.q_heads + u.head * group + (live ? row % group : 0)) * a.dim + c * 4;
      cp_async16(q_s + r * stride + c * 4, q + at, live ? 16 : 0);
    }
  }
  if (u.tile_begin < u.tile_end) load_tile<KEYS>(k_s, k_pool, a, u, table, u.tile_begin, stride);
  cp_async_commit();

  const int* bits[RPT];
  int oldest[RPT];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int row = min(u.row0 + ty + 8 * i, u.n * group - 1), token = u.first + row / group;
    bits[i] = a.tree + (size_t)token * a.tree_words;
    oldest[i] = a.window > 0 ? max(a.positions[token], u.held) - a.window + 1 : 0;
  }
  if (a.window > 0) {
    int most = oldest[0];
#pragma unroll
    for (int i = 1; i < RPT; ++i) most = max(most, oldest[i]);
    most = __reduce_max_sync(0xffffffffu, most);
    if ((threadIdx.x & 31) == 0) hidden_s[threadIdx.x >> 5] = most;
  }
  float2 o[RPT][MAX_C][2];
  float m_run[RPT], l_run[RPT];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    m_run[i] = -INFINITY; l_run[i] = 0.f;
#pragma unroll
    for (int c = 0; c < MAX_C; ++c) o[i][c][0] = o[i][c][1] = make_float2(0.f, 0.f);
  }
  for (int tile = u.tile_begin; tile < u.tile_end; ++tile) {
    load_tile<KEYS>(v_s, v_pool, a, u, table, tile, stride);
    cp_async_commit();
    cp_async_wait<1>();                                    // the keys; the values come under the first product
    __syncthreads();
    const int key0 = tile * KEYS;
    const bool drafts = key0 + KEYS > u.held;
    const bool looked = drafts || (a.window > 0 && key0 < max(max(hidden_s[0], hidden_s[1]), max(hidden_s[2], hidden_s[3])));
    float2 pairs[RPT][KPT];                                  // sums over the even and over the odd channels
#pragma unroll
    for (int i = 0; i < RPT; ++i)
#pragma unroll
      for (int j = 0; j < KPT; ++j) pairs[i][j] = make_float2(0.f, 0.f);
#pragma unroll 2
    for (int d = 0; d < a.dim; d += 4) {
      float4 kv[KPT];
#pragma unroll
      for (int j = 0; j < KPT; ++j) kv[j] = *reinterpret_cast<const float4*>(k_s + (tx + 16 * j) * stride + d);
      float4 qv[RPT];
#pragma unroll
      for (int i = 0; i < RPT; ++i) qv[i] = *reinterpret_cast<const float4*>(q_s + (ty + 8 * i) * stride + d);
#pragma unroll
      for (int i = 0; i < RPT; ++i)                        // a sum's two products stand apart: one waits for the other
#pragma unroll
        for (int j = 0; j < KPT; ++j) fma2(pairs[i][j], make_float2(qv[i].x, qv[i].y), make_float2(kv[j].x, kv[j].y));
#pragma unroll
      for (int i = 0; i < RPT; ++i)
#pragma unroll
        for (int j = 0; j < KPT; ++j) fma2(pairs[i][j], make_float2(qv[i].z, qv[i].w), make_float2(kv[j].z, kv[j].w));
    }
    float s[RPT][KPT];
#pragma unroll
    for (int i = 0; i < RPT; ++i)
#pragma unroll
      for (int j = 0; j < KPT; ++j) s[i][j] = pairs[i][j].x + pairs[i][j].y;
    const bool masked = drafts || key0 < u.key_lo || a.window > 0;
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      float top = -INFINITY;
#pragma unroll
      for (int j = 0; j < KPT; ++j) {
        const int key = key0 + tx + 16 * j;
        if (a.cap_in != 0.f) s[i][j] = a.cap_out * tanhf(s[i][j] / a.cap_out);
        if (masked && (key >= u.ctx || !sees(a, bits[i], key, u.held, oldest[i]))) s[i][j] = -INFINITY;
        top = fmaxf(top, s[i][j]);
      }
#pragma unroll
      for (int x = 1; x < 16; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
      top = fmaxf(top, m_run[i]);
      const float shift = top == -INFINITY ? 0.f : top;
      const float alpha = exp2f((m_run[i] - shift) * a.scale_log2);
      m_run[i] = top;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < KPT; ++j) {
        const float w = exp2f((s[i][j] - shift) * a.scale_log2);      // the difference first: a product of the maximum would round with its size
        p_s[(ty + 8 * i) * P_STRIDE + tx + 16 * j] = w;
        sum += w;
      }
      l_run[i] = l_run[i] * alpha + sum;
#pragma unroll
      for (int c = 0; c < MAX_C; ++c)
#pragma unroll
        for (int e = 0; e < 2; ++e) { o[i][c][e].x *= alpha; o[i][c][e].y *= alpha; }
    }
    cp_async_wait<0>();
    __syncthreads();                                       // values and weights are there, the keys are done with
    if (tile + 1 < u.tile_end) load_tile<KEYS>(k_s, k_pool, a, u, table, tile + 1, stride);
    cp_async_commit();
    if (looked) {
      const float* row = v_s + (threadIdx.x >> 2) * stride;                  // four threads look at a value row
      bool bad = false;
      for (int c = threadIdx.x & 3; c < a.dim >> 2; c += 4) {
        const float4 w = *reinterpret_cast<const float4*>(row + c * 4);
        bad |= !isfinite(w.x) || !isfinite(w.y) || !isfinite(w.z) || !isfinite(w.w);
      }
      const unsigned both = __ballot_sync(0xffffffffu, bad);
      if ((threadIdx.x & 31) == 0) bad_rows[threadIdx.x >> 5] = both;
      __syncthreads();
    }
    const bool any_bad = looked && (bad_rows[0] | bad_rows[1] | bad_rows[2] | bad_rows[3]);
    auto values = [&](auto some_bad) {
#pragma unroll 1
      for (int key = 0; key < KEYS; key += 4) {
        float4 w[RPT];
#pragma unroll
        for (int i = 0; i < RPT; ++i) w[i] = *reinterpret_cast<const float4*>(p_s + (ty + 8 * i) * P_STRIDE + key);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bool bad = some_bad && (bad_rows[(key + e) >> 3] >> (4 * ((key + e) & 7)) & 15u);
#pragma unroll
          for (int c = 0; c < MAX_C; ++c) {
            if (64 * c >= a.dim) break;                    // sums behind the last channel are of what lies there, and are not stored
            const float4 v = *reinterpret_cast<const float4*>(v_s + (key + e) * stride + 64 * c + 4 * tx);
#pragma unroll
            for (int i = 0; i < RPT; ++i) {
              const float p = e == 0 ? w[i].x : e == 1 ? w[i].y : e == 2 ? w[i].z : w[i].w;
              if (some_bad && bad && p == 0.f) continue;   // what a row does not see does not reach it
              fma2(o[i][c][0], make_float2(p, p), make_float2(v.x, v.y));
              fma2(o[i][c][1], make_float2(p, p), make_float2(v.z, v.w));
            }
          }
        }
      }
    };
    if (any_bad) values(std::true_type{}); else values(std::false_type{});
    __syncthreads();                                       // values and weights are done with
  }
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
#pragma unroll
    for (int x = 1; x < 16; x <<= 1) l_run[i] += __shfl_xor_sync(0xffffffffu, l_run[i], x);
    const int local = ty + 8 * i, row = u.row0 + local;
    if (local >= u.rows) continue;
    if (u.chunks > 1) {
      const long at = (u.index * gridDim.y + blockIdx.y) * RT + local;
#pragma unroll
      for (int c = 0; c < MAX_C; ++c)
        if (64 * c + 4 * tx < a.dim)
          *reinterpret_cast<float4*>(a.partials + at * a.dim + 64 * c + 4 * tx) = make_float4(o[i][c][0].x, o[i][c][0].y, o[i][c][1].x, o[i][c][1].y);
      if (tx == 0) *reinterpret_cast<float2*>(a.partials + a.partial_stats + at * 2) = make_float2(m_run[i] * a.scale_log2, l_run[i]);
    } else {
      const int head = u.head * group + row % group;
      float total = l_run[i], factor = 1.f;
      if (a.sinks) {
        const float sink = a.sinks[head] * LOG2E, m = m_run[i] * a.scale_log2, top = fmaxf(m, sink), base = top == -INFINITY ? 0.f : top;
        factor = exp2f(m - base);
        total = total * factor + exp2f(sink - base);
      }
      const float inv = total == 0.f ? 0.f : factor / total;
      float* to = (float*)a.out + ((size_t)(u.first + row / group) * a.q_heads + head) * a.dim;
#pragma unroll
      for (int c = 0; c < MAX_C; ++c)
        if (64 * c + 4 * tx < a.dim)
          *reinterpret_cast<float4*>(to + 64 * c + 4 * tx) = make_float4(o[i][c][0].x * inv, o[i][c][0].y * inv, o[i][c][1].x * inv, o[i][c][1].y * inv);
    }
  }
}

// ------------------------------------------------------------------------------- the chunks' results
// One warp per row: the chunks in order, relative to the largest of their maxima (kept in log2 units) and the sink.
template <typename T>
__global__ void __launch_bounds__(THREADS) attention_tree_join_kernel(const TreeArgs a, int tile_rows, int n_chunks) {
  pdl_launch_dependents();
  pdl_wait();
  const int row_tile_of = blockIdx.x / a.kv_heads, seq = row_tile_of / a.row_tiles;
  const Unit u = find_unit<sizeof(T) == 4 ? F32_KEYS : KEYS>(a, tile_rows, seq, row_tile_of - seq * a.row_tiles, blockIdx.x - row_tile_of * a.kv_heads, 0, n_chunks);
  const int local = blockIdx.y * (THREADS / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (local >= u.rows || u.chunks <= 1) return;
  const int group = a.q_heads / a.kv_heads, row = u.row0 + local, head = u.head * group + row % group;
  const long at = u.index * n_chunks * tile_rows + local;
  const float2* stats = reinterpret_cast<const float2*>(a.partials + a.partial_stats);
  float top = a.sinks ? a.sinks[head] * LOG2E : -INFINITY;
  const float sink = top;
  for (int c = lane; c < u.chunks; c += 32) top = fmaxf(top, stats[at + (long)c * tile_rows].x);
  top = warp_max(top);
  const float base = top == -INFINITY ? 0.f : top;
  float total = a.sinks ? exp2f(sink - base) : 0.f;
  constexpr int MAX_C = 2;                                 // 128 channels a step: head sizes up to 256
  float4 sum[MAX_C] = {};
  for (int c = 0; c < u.chunks; ++c) {
    const float2 ml = stats[at + (long)c * tile_rows];
    const float w = exp2f(ml.x - base);
    total += w * ml.y;
#pragma unroll
    for (int i = 0; i < MAX_C; ++i) {
      const int d = 128 * i + 4 * lane;
      if (d < a.dim) {
        const float4 v = *reinterpret_cast<const float4*>(a.partials + (at + (long)c * tile_rows) * a.dim + d);
        if (w != 0.f) { sum[i].x += w * v.x; sum[i].y += w * v.y; sum[i].z += w * v.z; sum[i].w += w * v.w; }
      }
    }
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  T* to = (T*)a.out + ((size_t)(u.first + row / group) * a.q_heads + head) * a.dim;
#pragma unroll
  for (int i = 0; i < MAX_C; ++i) {
    const int d = 128 * i + 4 * lane;
    if (d >= a.dim) break;
    Elem<T>::store(to + d, sum[i].x * inv); Elem<T>::store(to + d + 1, sum[i].y * inv);
    Elem<T>::store(to + d + 2, sum[i].z * inv); Elem<T>::store(to + d + 3, sum[i].w * inv);
  }
}

template <int RG, int MAX_DIM>
int launch_mma(const TreeArgs& a, dim3 grid, cudaStream_t stream) {
  const size_t smem = (size_t)(16 * RG + 4 * KEYS) * (a.dim + PAD) * sizeof(bf16);
  static LbPerDeviceOnce once;
  if (!once.run(LB_ALLOW_SMEM((attention_tree_mma_kernel<RG, MAX_DIM>), (16 * RG + 4 * KEYS) * (MAX_DIM + PAD) * sizeof(bf16)))) return lb_last_error();
  return lb_launch(attention_tree_mma_kernel<RG, MAX_DIM>, grid, THREADS, smem, stream, a);
}
template <int RT, int MAX_C>
int launch_f32_of(const TreeArgs& a, dim3 grid, cudaStream_t stream) {
  constexpr int KEYS = F32_KEYS;
  const size_t smem = ((size_t)(RT + 2 * KEYS) * (a.dim + 4) + RT * (KEYS + 4)) * sizeof(float);
  static LbPerDeviceOnce once;
  if (!once.run(LB_ALLOW_SMEM((attention_tree_f32_kernel<RT, MAX_C>), ((RT + 2 * KEYS) * (64 * MAX_C + 4) + RT * (KEYS + 4)) * sizeof(float)))) return lb_last_error();
  return lb_launch(attention_tree_f32_kernel<RT, MAX_C>, grid, THREADS, smem, stream, a);
}
template <int RT>
int launch_f32(const TreeArgs& a, dim3 grid, cudaStream_t stream) { return a.dim <= 128 ? launch_f32_of<RT, 2>(a, grid, stream) : launch_f32_of<RT, 4>(a, grid, stream); }
}  // namespace

// What the two entries below check alike.
static int check_tree(int dtype, const void* q, const void* k_pool, const void* v_pool, const void* out, int table_width, int n_pages, const int* positions,
                      int tree_words, int tokens, int q_heads, int kv_heads, int dim, int page_tokens, int window, float softcap, int max_nodes) {
  if (dtype != LB_F32 && dtype != LB_BF16) return LB_ERR_DTYPE;
  if (kv_heads <= 0 || q_heads <= 0 || q_heads % kv_heads || dim <= 0 || dim > 256 || dim % (dtype == LB_BF16 ? 16 : 4) || page_tokens <= 0 ||
      table_width <= 0 || n_pages <= 0 || tree_words <= 0 || window < 0 || softcap < 0.f || (window > 0 && !positions) || max_nodes <= 0 ||
      (long)max(max_nodes, tokens) * (q_heads / kv_heads) > 0x7fffffffL - 256)      // rows are counted in 32 bits
    return LB_ERR_SIZE;
  if (((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool | (uintptr_t)out) & 15) return LB_ERR_ALIGN;
  return 0;
}

// `tile_rows`: rows of a block (16, 32 or, in bfloat16, 64). `chunks` blocks of `chunk_tiles` tiles of 64 keys (float32: of 32) share a row tile's keys (the last takes
// what is left); with more than one, `partials` holds n_seqs * kv_heads * row_tiles * chunks * tile_rows * (dim + 2) floats.
LB_EXPORT int lb_attention_tree(int dtype, const void* q, const void* k_pool, const void* v_pool, void* out, const int* block_table, int table_width,
                                int n_pages, const int* cu_q, const int* ctx_len, const int* positions, const int* tree, int tree_words, int tokens,
                                int n_seqs, int q_heads, int kv_heads, int dim, int page_tokens, float scale, int window, const float* sinks,
                                float softcap, int max_nodes, int tile_rows, int row_tiles, int chunks, int chunk_tiles, float* partials,
                                long partial_floats, cudaStream_t stream) {
  if (tokens <= 0 || n_seqs <= 0) return 0;
  const int refused = check_tree(dtype, q, k_pool, v_pool, out, table_width, n_pages, positions, tree_words, tokens, q_heads, kv_heads, dim, page_tokens,
                                 window, softcap, max_nodes);
  if (refused) return refused;
  if (row_tiles <= 0 || chunks <= 0 || chunks > 65535 || chunk_tiles <= 0 || (double)n_seqs * row_tiles * kv_heads > 0x7fffffff ||
      (tile_rows != 16 && tile_rows != 32 && (tile_rows != 64 || dtype != LB_BF16)))
    return LB_ERR_SIZE;
  const long partial_rows = (long)n_seqs * kv_heads * row_tiles * chunks * tile_rows;
  if (chunks > 1 && (!partials || partial_floats < partial_rows * (dim + 2))) return LB_ERR_SIZE;
  if ((uintptr_t)partials & 15) return LB_ERR_ALIGN;
  TreeArgs a{q, k_pool, v_pool, out, block_table, table_width, n_pages, cu_q, ctx_len, positions, tree, tree_words, tokens, q_heads, kv_heads, dim,
             page_tokens, scale * LOG2E, 0.f, 0.f, window, sinks, row_tiles, chunk_tiles, chunks > 1 ? partials : nullptr, partial_rows * dim, n_seqs,
             max_nodes, 0, 0, nullptr, nullptr};
  if (softcap > 0.f) { a.cap_in = 2.f * LOG2E * scale / softcap; a.cap_out = softcap / scale; }
  const dim3 grid((unsigned)(n_seqs * row_tiles * kv_heads), chunks);
  int code;
  if (dtype == LB_F32) {
    code = tile_rows == 16 ? launch_f32<16>(a, grid, stream) : launch_f32<32>(a, grid, stream);
  } else if (dim <= 128) {
    code = tile_rows == 16 ? launch_mma<1, 128>(a, grid, stream) : tile_rows == 32 ? launch_mma<2, 128>(a, grid, stream) : launch_mma<4, 128>(a, grid, stream);
  } else {
    code = tile_rows == 16 ? launch_mma<1, 256>(a, grid, stream) : tile_rows == 32 ? launch_mma<2, 256>(a, grid, stream) : launch_mma<4, 256>(a, grid, stream);
  }
  if (code || chunks == 1) return code ? code : lb_last_error();
  const dim3 joined(grid.x, tile_rows / (THREADS / 32));
  code = dtype == LB_F32 ? lb_launch(attention_tree_join_kernel<float>, joined, THREADS, 0, stream, a, tile_rows, chunks)
                         : lb_launch(attention_tree_join_kernel<bf16>, joined, THREADS, 0, stream, a, tile_rows, chunks);
  return code ? code : lb_last_error();
}

// The tcgen05 kernel: bfloat16, heads of 128 channels, at most 128 query heads a key/value head, pages of 8 .. 128 tokens that divide 128. `blocks` blocks
// share the keys; `rows2`: tiles of twice 128 / group drafts. `scratch` holds wide::scratch_floats(blocks, rows2, tokens * q_heads) of them.
LB_EXPORT int lb_attention_tree_tcgen05(const void* q, const void* k_pool, const void* v_pool, void* out, const int* block_table, int table_width,
                                        int n_pages, const int* cu_q, const int* ctx_len, const int* positions, const int* tree, int tree_words,
                                        int tokens, int n_seqs, int q_heads, int kv_heads, int dim, int page_tokens, float scale, int window,
                                        const float* sinks, float softcap, int max_nodes, int blocks, int rows2, float* scratch, long floats,
                                        cudaStream_t stream) {
  if (tokens <= 0 || n_seqs <= 0) return 0;
  const int refused = check_tree(LB_BF16, q, k_pool, v_pool, out, table_width, n_pages, positions, tree_words, tokens, q_heads, kv_heads, dim, page_tokens,
                                 window, softcap, max_nodes);
  if (refused) return refused;
  // key tiles are counted in 32 bits too
  const double most_tiles = (double)n_seqs * kv_heads * (max_nodes / (128 / max(1, min(128, q_heads / kv_heads))) + 1) * ((double)table_width * page_tokens / 128 + 1);
  if (most_tiles > 0x7fffffff || dim != 128 || q_heads / kv_heads > 128 || page_tokens % 8 || 128 % page_tokens || blocks <= 0 || blocks > 1024 || !scratch ||
      floats < wide::scratch_floats(blocks, rows2 != 0, (long)tokens * q_heads))
    return LB_ERR_SIZE;
  if (((uintptr_t)scratch | (uintptr_t)out) & 31) return LB_ERR_ALIGN;
  TreeArgs a{q, k_pool, v_pool, out, block_table, table_width, n_pages, cu_q, ctx_len, positions, tree, tree_words, tokens, q_heads, kv_heads, dim,
             page_tokens, scale * LOG2E, 0.f, 0.f, window, sinks, 0, 0, scratch, 0, n_seqs, max_nodes, 0, 0, nullptr, nullptr};
  if (softcap > 0.f) { a.cap_in = 2.f * LOG2E * scale / softcap; a.cap_out = softcap / scale; }
  const int code = rows2 ? wide::launch<true>(a, blocks, stream) : wide::launch<false>(a, blocks, stream);
  return code ? code : lb_last_error();
}

LB_EXPORT void* lb_attention_tree_status_address() {
  void* address = nullptr;
  return cudaGetSymbolAddress(&address, g_tree_error) == cudaSuccess ? address : nullptr;
}
// What a bounded wait that ran out left, and clears it; synchronises.
LB_EXPORT int lb_attention_tree_status() {
  int code = 0;
  const int zero = 0;
  if (cudaMemcpyFromSymbol(&code, g_tree_error, sizeof(int)) != cudaSuccess) return -1;
  if (code) cudaMemcpyToSymbol(g_tree_error, &zero, sizeof(int));
  return code;
}

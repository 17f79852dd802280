// What the kernels of attention for trees of drafts share (attention_tree.cu, attention_tree_tcgen05.cuh): their arguments, what a
// block works on, which keys a row sees.
#pragma once
#include "common.cuh"

namespace {

constexpr float LOG2E = 1.4426950408889634f;

// A row tile whose keys lie in the shares of blocks `from` to `upto`; drafts 0: none.
struct Border { int from, upto, seq, head, token, draft, drafts, unused; };

struct TreeArgs {
  const void *q, *k_pool, *v_pool;
  void* out;
  const int* block_table;
  int table_width, n_pages;
  const int *cu_q, *ctx_len, *positions, *tree;
  int tree_words, tokens;
  int q_heads, kv_heads, dim, page_tokens;
  float scale_log2;             // scale * log2(e)
  float cap_in, cap_out;        // 2 log2(e) scale / cap and cap / scale; 0: no cap
  int window;
  const float* sinks;
  int row_tiles, chunk_tiles;   // row tiles of a sequence, key tiles of a block
  float* partials;              // [unit][chunk][rows][dim] outputs, then [unit][chunk][rows][2] maxima and sums; null: one chunk
  long partial_stats;           // where the second part begins, in floats
  int n_seqs, max_nodes;
  int group, tile_drafts;       // query heads of a key/value head; drafts of a tile of 128 rows (the tcgen05 kernel's)
  Border* borders;       // the tcgen05 kernel's, for the kernel that joins: per block
  float2* row_stats;            // its [tokens][q_heads], of its careful pass: a row's maximum, and the sum of its weights and the sink's relative to it
};

// What a block works on: its rows, and its share of the keys.
struct Unit {
  int seq, head, row0, rows;    // the sequence, the first row of its tile and how many of the tile's rows there are
  int first, n, held, ctx;      // its first token, drafts, held tokens, keys
  int key_lo;                   // no row sees a key below
  int tile_begin, tile_end, chunks;
  long index;                   // in the partial results
};

template <int KEYS>     // keys of a tile
__device__ __forceinline__ Unit find_unit(const TreeArgs& a, int tile_rows, int seq, int row_tile, int head, int chunk, int n_chunks) {
  Unit u;
  u.seq = seq; u.head = head;
  u.first = a.cu_q[seq];
  u.n = min(a.cu_q[seq + 1], a.tokens) - u.first;
  u.ctx = a.ctx_len[seq];
  u.held = u.ctx - u.n;
  const int group = a.q_heads / a.kv_heads;
  u.row0 = row_tile * tile_rows;
  u.rows = min(tile_rows, min(u.n, a.max_nodes) * group - u.row0);
  u.key_lo = a.window > 0 ? max(0, u.held - a.window + 1) : 0;      // the first draft's position is `held` at least
  const int tile_lo = u.key_lo / KEYS, tiles = (u.ctx + KEYS - 1) / KEYS - tile_lo;
  u.chunks = min(n_chunks, max(1, (tiles + a.chunk_tiles - 1) / a.chunk_tiles));
  u.tile_begin = tile_lo + chunk * a.chunk_tiles;
  u.tile_end = tile_lo + (chunk == n_chunks - 1 ? tiles : min(tiles, (chunk + 1) * a.chunk_tiles));
  u.index = ((long)seq * a.kv_heads + head) * a.row_tiles + row_tile;
  return u;
}

// Bit i: whether a row sees key key0 + i, 32 of them: `bits` are its drafts, `oldest` the first held key it sees.
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? ~0u : (1u << n) - 1u; }
__device__ __forceinline__ uint32_t seen_word(uint32_t drafts, int key0, int held, int ctx, int oldest) {      // `drafts`: the tree's bits from key0 on
  const uint32_t kept = below(held - key0);
  return ((drafts & ~kept) | (kept & ~below(oldest - key0))) & below(ctx - key0);
}
__device__ __forceinline__ uint32_t seen_word(int tree_words, const int* bits, int key0, int held, int ctx, int oldest) {
  const int j = key0 - held, w = j >> 5;                  // the first key's draft; negative for held ones
  const uint32_t lo = w >= 0 && w < tree_words ? (uint32_t)bits[w] : 0u, hi = w + 1 >= 0 && w + 1 < tree_words ? (uint32_t)bits[w + 1] : 0u;
  return seen_word(__funnelshift_r(lo, hi, j & 31), key0, held, ctx, oldest);
}

// Where key `key` of a sequence lies in its pool, in rows of one head's channels; -1 for a page that is not there.
__device__ __forceinline__ long key_row(const TreeArgs& a, const int* table, int key, int head) {
  const int index = key / a.page_tokens;
  if (index >= a.table_width) return -1;
  const int page = table[index];
  if ((unsigned)page >= (unsigned)a.n_pages) return -1;
  return ((long)page * a.kv_heads + head) * a.page_tokens + (key - index * a.page_tokens);
}

// Whether row `token` sees key `key`, `held` <= key < ctx or below: the tree decides among drafts, the window among held keys.
__device__ __forceinline__ bool sees(const TreeArgs& a, const int* bits, int key, int held, int oldest) {
  if (key < held) return key >= oldest;
  const int j = key - held;
  return (j >> 5) < a.tree_words && ((unsigned)bits[j >> 5] >> (j & 31)) & 1u;
}

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ bool not_finite(uint32_t two) {
  return (two & 0x7F800000u) == 0x7F800000u || (two & 0x00007F80u) == 0x00007F80u;
}
}  // namespace

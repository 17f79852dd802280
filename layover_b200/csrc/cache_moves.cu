// Moving what a cache holds: whole pages (or state slots) copied for a request that is forked, rows of accepted drafts
// moved to the places right behind what their request holds. In all layers of a pool at once. The reference neither forks nor
// drafts; its nearest relative moves blocks to and from the host (layover/kv/paged_cache.py).
//
// Both are bound by memory: every byte that moves is read once and written once. Measured (one B200): 56 pages of 72 planes, 216 MB in all, 38.5
// us (5.6 TB/s of 6.5), 24 states of 2 MB in 3 layers 42.3 us (5.9), the accepted rows of 64 requests, 55 MB, 18.5 us (3.0: rows of 256
// bytes in 72 x 8 places each), of one request 3.6 us.
//
// Neither kernel lets its dependents start early, and each thread's last act is to make its writes visible to the whole device: decode
// attention reads a cache's earlier keys ahead of its wait, which is sound only where no kernel that may still run writes them. So
// whatever is launched behind a move, or behind others that are, starts when the rows have been moved. (0.4 to 0.9 us a launch.)
#include "common.cuh"

namespace {

constexpr int THREADS = 256;
constexpr int MOST_BLOCKS = 512;    // of the compaction (64 sequences of 5 rows in 72 planes of 8 heads, us with 512, 1,024 and 2,048, without the fence at the end: 17.6, 18.8, 19.9)
constexpr int COPY_UNROLL = 4;      // vectors of a thread that are on their way at once

// pool [planes][pages][vecs of a page]: plane p's page dst[i] = its page src[i].
template <typename V>
__global__ void __launch_bounds__(THREADS) copy_pages_kernel(V* __restrict__ pool, const int* __restrict__ src, const int* __restrict__ dst,
                                                             int n_pages, long vecs) {
  pdl_wait();
  const int from = src[blockIdx.y], to = dst[blockIdx.y];
  if ((unsigned)from >= (unsigned)n_pages || (unsigned)to >= (unsigned)n_pages || from == to) return;
  V* plane = pool + (size_t)blockIdx.z * n_pages * vecs;
  const V* a = plane + (size_t)from * vecs;
  V* b = plane + (size_t)to * vecs;
  const long at = (long)blockIdx.x * (THREADS * COPY_UNROLL) + threadIdx.x;
  V v[COPY_UNROLL];
#pragma unroll
  for (int i = 0; i < COPY_UNROLL; ++i)
    if (at + i * THREADS < vecs) v[i] = a[at + i * THREADS];
#pragma unroll
  for (int i = 0; i < COPY_UNROLL; ++i)
    if (at + i * THREADS < vecs) b[at + i * THREADS] = v[i];
  __threadfence();
}

// pool [planes][pages][heads][page_tokens][vecs of a row]. Sequence s keeps its drafts picked[cu[s]] < picked[cu[s] + 1] < ...: the
// row at place first[s] + picked[cu[s] + i] goes to place first[s] + i. In place: a thread takes its own piece of the rows of one
// plane and head in order, `ROWS` loads before their stores, and a row that is still to be read lies at or behind the place that is written.
// What a row's places are comes from five reads one after the other, so a block finds them once for all the planes and heads that it takes.
constexpr int ROWS = 8;
template <typename V>
__global__ void __launch_bounds__(THREADS) compact_tokens_kernel(V* __restrict__ pool, const int* __restrict__ block_table, int table_width,
                                                                 const int* __restrict__ first, const int* __restrict__ picked,
                                                                 const int* __restrict__ cu, int n_picked, int n_pages, int heads, int page_tokens,
                                                                 int vecs, unsigned pieces) {
  __shared__ long from_s[ROWS], to_s[ROWS];
  pdl_wait();
  const int seq = blockIdx.y, lo = max(cu[seq], 0), n = min(cu[seq + 1], n_picked) - lo, held = first[seq];
  const int* table = block_table + (size_t)seq * table_width;
  for (int i0 = 0; i0 < n; i0 += ROWS) {
    __syncthreads();
    if (threadIdx.x < ROWS) {                              // the rows' places without plane, head and piece; -1: nothing to move
      const int i = i0 + threadIdx.x;
      long from = -1, to = -1;
      if (i < n) {
        const int p = picked[lo + i];
        const long a = (long)held + p, b = (long)held + i;
        if (p > i && held >= 0 && a / page_tokens < table_width) {
          const int page_a = table[a / page_tokens], page_b = table[b / page_tokens];
          if ((unsigned)page_a < (unsigned)n_pages && (unsigned)page_b < (unsigned)n_pages) {
            from = ((long)page_a * heads * page_tokens + a % page_tokens) * vecs;
            to = ((long)page_b * heads * page_tokens + b % page_tokens) * vecs;
          }
        }
      }
      from_s[threadIdx.x] = from; to_s[threadIdx.x] = to;
    }
    __syncthreads();
    for (unsigned piece = blockIdx.x * THREADS + threadIdx.x; piece < pieces; piece += gridDim.x * THREADS) {
      const unsigned unit = piece / (unsigned)vecs, plane_at = unit / (unsigned)heads;      // plane * heads + head
      V* plane = pool + ((size_t)plane_at * n_pages * heads + (unit - plane_at * heads)) * page_tokens * vecs + (piece - unit * vecs);
      V v[ROWS];
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
        if (from_s[i] >= 0) v[i] = plane[from_s[i]];
#pragma unroll
      for (int i = 0; i < ROWS; ++i)
        if (from_s[i] >= 0) plane[to_s[i]] = v[i];
    }
  }
  __threadfence();
}

// the widest vector that divides a row of `bytes` bytes and the pool's alignment
template <typename F>
int with_vector(long bytes, const void* base, F launch) {
  const uintptr_t odd = (uintptr_t)bytes | (uintptr_t)base;
  if (odd % 16 == 0) return launch(uint4{});
  if (odd % 8 == 0) return launch(uint2{});
  if (odd % 4 == 0) return launch((unsigned)0);
  if (odd % 2 == 0) return launch((unsigned short)0);
  return launch((unsigned char)0);
}
}  // namespace

LB_EXPORT int lb_copy_pages(void* pool, const int* src, const int* dst, int n_pairs, int planes, int n_pages, long page_bytes, cudaStream_t stream) {
  if (n_pairs <= 0 || planes <= 0 || page_bytes <= 0) return 0;
  if (n_pages <= 0 || n_pairs > 65535 || planes > 65535) return LB_ERR_SIZE;
  return with_vector(page_bytes, pool, [&](auto vec) {
    using V = decltype(vec);
    const long vecs = page_bytes / (long)sizeof(V), blocks = (vecs + THREADS * COPY_UNROLL - 1) / (THREADS * COPY_UNROLL);
    if (blocks > 0x7fffffffL) return (int)LB_ERR_SIZE;
    lb_launch(copy_pages_kernel<V>, dim3((unsigned)blocks, n_pairs, planes), THREADS, 0, stream, (V*)pool, src, dst, n_pages, vecs);
    return lb_last_error();
  });
}

LB_EXPORT int lb_compact_tokens(void* pool, const int* block_table, int table_width, const int* first, const int* picked, const int* cu, int n_picked,
                                int n_seqs, int planes, int n_pages, int heads, int page_tokens, long row_bytes, cudaStream_t stream) {
  if (n_seqs <= 0 || planes <= 0 || heads <= 0 || row_bytes <= 0) return 0;
  if (n_pages <= 0 || page_tokens <= 0 || table_width <= 0 || n_seqs > 65535) return LB_ERR_SIZE;
  return with_vector(row_bytes, pool, [&](auto vec) {
    using V = decltype(vec);
    const long vecs = row_bytes / (long)sizeof(V), pieces = (long)planes * heads * vecs;
    if (pieces > 0x7fffffffL) return (int)LB_ERR_SIZE;
    const long blocks = (pieces + THREADS - 1) / THREADS, each = (blocks * n_seqs + MOST_BLOCKS - 1) / MOST_BLOCKS;      // passes of a block
    lb_launch(compact_tokens_kernel<V>, dim3((unsigned)((blocks + each - 1) / each), n_seqs), THREADS, 0, stream, (V*)pool, block_table, table_width, first,
              picked, cu, n_picked, n_pages, heads, page_tokens, (int)vecs, (unsigned)pieces);
    return lb_last_error();
  });
}

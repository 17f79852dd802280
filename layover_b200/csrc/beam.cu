// Choosing the continuations of a request's beams: the `keep` best of beams x vocabulary by
//
//   score[b] + logit[b, v] - log sum_w exp(logit[b, w])
//
// ties to the lowest b * vocab + v. An ended beam is one candidate, itself with the padding token; a beam whose score is
// -inf, or whose logits have no finite sum of exponentials, is none. The reference samples greedily, one sequence a request
// (layover/engine.py:139-141,187).
//
// Two kernels. The first reads the logits once: a block takes a chunk of one row, piece by piece, and leaves the chunk's maximum and sum of
// exponentials and its `keep` best. Those are found by a threshold that `keep` values reach at least and few more: the keep-th largest of 64
// groups' own maxima in the first piece. What reaches it is collected, and ranked by counting when there is much of it (which gives
// a higher threshold) and at the end. Within a beam the order is that of the logits themselves, so no rounding is involved. The
// second kernel has one block a request: the beams' sums are joined in 64 bits, and of the chunks' lists the candidates are compared
// in 64 bits behind a threshold of the same kind, where two beams' tie only where the formula's do within 1e-7.
// Where more values reach a threshold than there is room for (many equal ones), the best are picked one by one.
#include <math.h>

#include "common.cuh"

namespace {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_KEEP = 32;
constexpr int MAX_BEAMS = 64;
constexpr int ROOM = 1024;          // values that reach the threshold: of random ones about 45 for 32
constexpr int NONE = 0x7fffffff;    // the index of what is not there
constexpr float LOG2E = 1.4426950408889634f;

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ bool before(T v, int i, T w, int j) { return v > w || (v == w && i < j); }

// The keep-th largest (keep <= 64) of the values of threads 0 .. 63 (ties: the lower thread first): the same for all threads. Where they
// are the largest of 64 groups of values, `keep` values reach it at least. `all` has room for them.
template <typename T>
__device__ __forceinline__ T kth_largest_of_64(T v, int keep, T* all, T* result) {
  if (threadIdx.x < 64) all[threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.x < 64) {
    int rank = 0;
#pragma unroll 16
    for (int t = 0; t < 64; ++t) rank += before(all[t], t, v, (int)threadIdx.x) ? 1 : 0;
    if (rank == keep - 1) *result = v;
  }
  __syncthreads();
  return *result;
}
// The best of what the threads offer: the same for all threads.
template <typename T>
__device__ __forceinline__ void block_best(T& v, int& i, T* values, int* indices) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const T ov = __shfl_xor_sync(0xffffffffu, v, o);
    const int oi = __shfl_xor_sync(0xffffffffu, i, o);
    if (before(ov, oi, v, i)) { v = ov; i = oi; }
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) { values[threadIdx.x >> 5] = v; indices[threadIdx.x >> 5] = i; }
  __syncthreads();
  v = values[0]; i = indices[0];
  for (int w = 1; w < WARPS; ++w)
    if (before(values[w], indices[w], v, i)) { v = values[w]; i = indices[w]; }
}

// stats [rows][chunks] (maximum, sum of exp(x - maximum)), lists [rows][chunks][keep] of (value, index), best first, (-inf, NONE) behind the last.
// A chunk is `pieces` of PIECE values.
constexpr int EACH = 16, PIECE = THREADS * EACH;
__global__ void __launch_bounds__(THREADS, 4) beam_chunk_kernel(const float* __restrict__ logits, long row_stride, int vocab, int keep, int pieces,
                                                                float2* __restrict__ stats, float2* __restrict__ lists) {
  __shared__ float values[ROOM], part[WARPS], part_sum[WARPS], threshold, spread[THREADS];
  __shared__ int indices[ROOM], count;
  pdl_launch_dependents();
  pdl_wait();
  const float* row = logits + (size_t)blockIdx.y * row_stride;
  const int begin = blockIdx.x * pieces * PIECE, end = min(vocab, begin + pieces * PIECE), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float next[EACH], m = -INFINITY, sum = 0.f, reach = -INFINITY;
#pragma unroll
  for (int j = 0; j < EACH; ++j) next[j] = begin + (int)threadIdx.x + j * THREADS < end ? row[begin + threadIdx.x + j * THREADS] : -INFINITY;
  if (threadIdx.x == 0) count = 0;
  for (int from = begin; from < end; from += PIECE) {
    const int lo = from + threadIdx.x;
    float x[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j) {                       // the next piece is on its way while this one is looked at
      x[j] = next[j];
      next[j] = lo + PIECE + j * THREADS < end ? row[lo + PIECE + j * THREADS] : -INFINITY;
    }
    float top = -INFINITY;                                 // of numbers: NaN is no maximum, but the sum becomes it
#pragma unroll
    for (int j = 0; j < EACH; ++j) top = fmaxf(top, x[j]);
    if (from == begin) {
      spread[threadIdx.x] = top;
      __syncthreads();
      float group = -INFINITY;
      if (threadIdx.x < 64) group = fmaxf(fmaxf(spread[threadIdx.x], spread[threadIdx.x + 64]), fmaxf(spread[threadIdx.x + 128], spread[threadIdx.x + 192]));
      reach = kth_largest_of_64(group, keep, values, &threshold);
    }
    const float rise = fmaxf(m, top), base = rise == -INFINITY ? 0.f : rise;
    sum *= fast_exp2((m - base) * LOG2E);
    m = rise;
#pragma unroll
    for (int j = 0; j < EACH; ++j) sum += fast_exp2((x[j] - base) * LOG2E);
    if (top >= reach) {
#pragma unroll
      for (int j = 0; j < EACH; ++j)
        if (x[j] >= reach && x[j] > -INFINITY) {
          const int at = atomicAdd(&count, 1);
          if (at < ROOM) { values[at] = x[j]; indices[at] = lo + j * THREADS; }
        }
    }
    __syncthreads();
    const int n = count;
    if (n > ROOM / 2 && n <= ROOM) {                       // the best of them, and a higher threshold
      float v[ROOM / THREADS];
      int i[ROOM / THREADS], rank[ROOM / THREADS];
#pragma unroll
      for (int c = 0; c < ROOM / THREADS; ++c) {
        rank[c] = NONE;
        if ((int)threadIdx.x + c * THREADS < n) {
          v[c] = values[threadIdx.x + c * THREADS]; i[c] = indices[threadIdx.x + c * THREADS];
          rank[c] = 0;
          for (int o = 0; o < n; ++o) rank[c] += before(values[o], indices[o], v[c], i[c]) ? 1 : 0;
        }
      }
      __syncthreads();
#pragma unroll
      for (int c = 0; c < ROOM / THREADS; ++c)
        if (rank[c] < keep) {
          values[rank[c]] = v[c]; indices[rank[c]] = i[c];
          if (rank[c] == keep - 1) threshold = v[c];
        }
      if (threadIdx.x == 0) count = keep;
      __syncthreads();
      reach = threshold;
    }
  }
  // the maximum and the sum of all threads
  float top = warp_max(m), base = top == -INFINITY ? 0.f : top;
  sum = warp_sum(sum * fast_exp2((m - base) * LOG2E));
  if (lane == 0) { part[warp] = top; part_sum[warp] = sum; }
  __syncthreads();
  const size_t at = (size_t)blockIdx.y * gridDim.x + blockIdx.x;
  if (threadIdx.x == 0) {
    for (int w = 1; w < WARPS; ++w) top = fmaxf(top, part[w]);
    base = top == -INFINITY ? 0.f : top;
    float all = 0.f;
    for (int w = 0; w < WARPS; ++w) all += part_sum[w] * fast_exp2((part[w] - base) * LOG2E);
    stats[at] = make_float2(top, all);
  }
  float2* list = lists + at * keep;
  const int n = count;
  if (n <= ROOM) {
    for (int c = threadIdx.x; c < n; c += THREADS) {
      const float v = values[c];
      const int i = indices[c];
      int rank = 0;
      for (int o = 0; o < n; ++o) rank += before(values[o], indices[o], v, i) ? 1 : 0;
      if (rank < keep) list[rank] = make_float2(v, __int_as_float(i));
    }
    if ((int)threadIdx.x >= n && (int)threadIdx.x < keep) list[threadIdx.x] = make_float2(-INFINITY, __int_as_float(NONE));
  } else {                                                 // one after the other: the best behind the one before
    float last = INFINITY;
    int last_index = -1;
    for (int k = 0; k < keep; ++k) {
      float v = -INFINITY;
      int i = NONE;
      for (int j = begin + threadIdx.x; j < end; j += THREADS) {
        const float y = row[j];
        if (y > -INFINITY && before(last, last_index, y, j) && before(y, j, v, i)) { v = y; i = j; }
      }
      block_best(v, i, part, indices);
      if (threadIdx.x == 0) list[k] = make_float2(v, __int_as_float(i));
      last = v; last_index = i;
    }
  }
}

__global__ void __launch_bounds__(THREADS) beam_join_kernel(const float* __restrict__ scores, const int* __restrict__ ended, int beams, int vocab, int keep,
                                                            int pad, int chunks, const float2* __restrict__ stats, const float2* __restrict__ lists,
                                                            float* __restrict__ next_scores, int* __restrict__ parents, int* __restrict__ tokens) {
  __shared__ double offsets[MAX_BEAMS];                    // what a beam's logits are raised by; its own score where it has ended; -inf: no beam
  __shared__ bool over[MAX_BEAMS];
  __shared__ double values[ROOM], part[WARPS], threshold;
  __shared__ double spread[THREADS];
  __shared__ int indices[ROOM], part_index[WARPS];
  __shared__ int count;
  pdl_launch_dependents();
  pdl_wait();
  const int request = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n_lists = beams * chunks;
  const float2* mine = lists + (size_t)request * n_lists * keep;
  for (int b = warp; b < beams; b += WARPS) {
    const size_t row = (size_t)request * beams + b;
    const float score = scores[row];
    const bool end = ended && ended[row];
    const float2* of = stats + row * chunks;
    float m = -INFINITY;
    for (int c = lane; c < chunks; c += 32) m = fmaxf(m, of[c].x);
    m = warp_max(m);
    double sum = 0.0;
    for (int c = lane; c < chunks; c += 32)
      if (of[c].y != 0.f) sum += (double)of[c].y * (double)expf(of[c].x - m);      // a chunk without a finite value has a sum of 0
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      double offset = (double)score - (double)m - log(sum);
      if (!(score > -INFINITY) || (!end && !isfinite(offset))) offset = -INFINITY;
      offsets[b] = end && score > -INFINITY ? (double)score : offset;
      over[b] = end;
    }
  }
  if (threadIdx.x == 0) count = 0;
  __syncthreads();
  // candidate c, of all lists' one after the other: an ended beam has one, in its first list
  const int n_candidates = n_lists * keep;
  auto candidate = [&](int c, double& v, int& i) {
    const int l = c / keep, b = l / chunks;
    v = -INFINITY; i = NONE;
    if (offsets[b] == -INFINITY) return;
    if (over[b]) {
      if (c == b * chunks * keep) { v = offsets[b]; i = b * vocab + pad; }
      return;
    }
    const float2 x = mine[c];
    if (x.x > -INFINITY) { v = offsets[b] + (double)x.x; i = b * vocab + __float_as_int(x.y); }
  };
  double best = -INFINITY;
  for (int c = threadIdx.x; c < n_candidates; c += THREADS) {
    double v;
    int i;
    candidate(c, v, i);
    if (v > best) best = v;
  }
  // groups of threads 64 apart: what is best of a list lies in different ones
  spread[threadIdx.x] = best;
  __syncthreads();
  if (threadIdx.x < 64) best = fmax(fmax(spread[threadIdx.x], spread[threadIdx.x + 64]), fmax(spread[threadIdx.x + 128], spread[threadIdx.x + 192]));
  const double reach = kth_largest_of_64(best, keep, values, &threshold);
  for (int c = threadIdx.x; c < n_candidates; c += THREADS) {
    double v;
    int i;
    candidate(c, v, i);
    if (v >= reach && i != NONE) {
      const int at = atomicAdd(&count, 1);
      if (at < ROOM) { values[at] = v; indices[at] = i; }
    }
  }
  __syncthreads();
  const int n = count;
  auto choose = [&](int k, double v, int i) {
    const size_t at = (size_t)request * keep + k;
    next_scores[at] = (float)v;
    parents[at] = i == NONE ? -1 : i / vocab;
    tokens[at] = i == NONE ? -1 : i % vocab;
  };
  if (n <= ROOM) {
    for (int c = threadIdx.x; c < n; c += THREADS) {
      const double v = values[c];
      const int i = indices[c];
      int rank = 0;
      for (int o = 0; o < n; ++o) rank += before(values[o], indices[o], v, i) ? 1 : 0;
      if (rank < keep) choose(rank, v, i);
    }
    if ((int)threadIdx.x >= n && (int)threadIdx.x < keep) choose(threadIdx.x, -INFINITY, NONE);
  } else {                                                 // one after the other
    double last = INFINITY;
    int last_index = -1;
    for (int k = 0; k < keep; ++k) {
      double v = -INFINITY;
      int i = NONE;
      for (int c = threadIdx.x; c < n_candidates; c += THREADS) {
        double w;
        int j;
        candidate(c, w, j);
        if (j != NONE && before(last, last_index, w, j) && before(w, j, v, i)) { v = w; i = j; }
      }
      block_best(v, i, part, part_index);
      if (threadIdx.x == 0) choose(k, v, i);
      last = v; last_index = i;
    }
  }
}
}  // namespace

// A block of the first kernel takes `pieces` of lb_beam_piece() values, chunks = ceil(vocab / (pieces * lb_beam_piece())). Scratch: rows * chunks * (2 + 2
// keep) words.
LB_EXPORT int lb_beam_piece() { return PIECE; }
LB_EXPORT int lb_beam_select(const float* logits, long row_stride, const float* scores, const int* ended, int requests, int beams, int vocab, int keep,
                             int pad, int pieces, void* scratch, long scratch_words, float* next_scores, int* parents, int* tokens, cudaStream_t stream) {
  if (requests <= 0) return 0;
  if (beams <= 0 || beams > MAX_BEAMS || keep <= 0 || keep > MAX_KEEP || vocab <= 0 || pieces <= 0 || pieces > 0x7fffffff / PIECE || pad < 0 || pad >= vocab ||
      (long)beams * vocab >= 0x7fffffffL - PIECE || (long)requests * beams > 65535)
    return LB_ERR_SIZE;
  const long rows = (long)requests * beams, chunks = (vocab + (long)PIECE * pieces - 1) / ((long)PIECE * pieces);
  if (scratch_words < rows * chunks * (2 + 2 * keep)) return LB_ERR_SIZE;
  if ((uintptr_t)scratch & 7) return LB_ERR_ALIGN;
  float2 *stats = (float2*)scratch, *lists = stats + rows * chunks;
  int code = lb_launch(beam_chunk_kernel, dim3((unsigned)chunks, (unsigned)rows), THREADS, 0, stream, logits, row_stride, vocab, keep, pieces, stats, lists);
  if (code) return code;
  code = lb_launch(beam_join_kernel, requests, THREADS, 0, stream, scores, ended, beams, vocab, keep, pad, (int)chunks, stats, lists, next_scores, parents, tokens);
  return code ? code : lb_last_error();
}

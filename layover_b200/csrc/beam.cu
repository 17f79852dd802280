// Choosing the continuations of a request's beams: the `keep` best of beams x vocabulary by
//
//   score[b] + logit[b, v] - log sum_w exp(logit[b, w])
//
// ties to the lowest b * vocab + v. An ended beam is one candidate, itself with the padding token; a beam whose score is
// -inf, or whose logits have no finite sum of exponentials, is none. The reference samples greedily, one sequence a request
// (layover/engine.py:139-141,187).
//
// Two kernels. The first reads the logits once: a block takes a chunk of one row, every thread keeps the maximum and sum of
// what it reads and every warp a sorted list of its best 32 in its lanes, which a value enters only if it is better than the last that
// counts; a warp's list is joined with the others' and left with the chunk's maximum and sum. Within a beam the order is that of
// the logits themselves, so no rounding is involved. The second has one block a request: the beams' sums are joined and the lists'
// candidates compared in 64 bits, in which two beams' candidates tie only where the formula's do within 1e-7.
#include <math.h>

#include "common.cuh"

namespace {

constexpr int THREADS = 256;
constexpr int WARPS = THREADS / 32;
constexpr int MAX_KEEP = 32;
constexpr int MAX_BEAMS = 64;
constexpr int UNROLL = 8;           // values of a thread that are on their way at once

__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The best candidates a warp has met, best first, one a lane; `keep` of them count.
template <typename T>
struct Best {
  T value;
  int index;
  __device__ __forceinline__ void clear() { value = -INFINITY; index = 0x7fffffff; }
  static __device__ __forceinline__ bool before(T v, int i, T w, int j) { return v > w || (v == w && i < j); }
  // one more candidate, the same in every lane
  __device__ __forceinline__ void insert(T v, int i) {
    const int lane = threadIdx.x & 31;
    const int place = __popc(__ballot_sync(0xffffffffu, before(value, index, v, i)));
    const T up_value = __shfl_up_sync(0xffffffffu, value, 1);
    const int up_index = __shfl_up_sync(0xffffffffu, index, 1);
    if (lane == place) { value = v; index = i; }
    if (lane > place) { value = up_value; index = up_index; }
  }
  // one candidate a lane; -inf is none
  __device__ __forceinline__ void offer(T v, int i, int keep) {
    const int lane = threadIdx.x & 31;
    T last = __shfl_sync(0xffffffffu, value, keep - 1);
    int last_index = __shfl_sync(0xffffffffu, index, keep - 1);
    unsigned waiting = __ballot_sync(0xffffffffu, v > (T)-INFINITY && before(v, i, last, last_index));
    while (waiting) {
      const int from = __ffs(waiting) - 1;
      insert(__shfl_sync(0xffffffffu, v, from), __shfl_sync(0xffffffffu, i, from));
      last = __shfl_sync(0xffffffffu, value, keep - 1);
      last_index = __shfl_sync(0xffffffffu, index, keep - 1);
      waiting = __ballot_sync(0xffffffffu, lane > from && (waiting >> lane & 1u) && before(v, i, last, last_index));
    }
  }
};

// stats [rows][chunks] (maximum, sum of exp(x - maximum)), list_values / list_index [rows][chunks][keep]
__global__ void __launch_bounds__(THREADS) beam_chunk_kernel(const float* __restrict__ logits, long row_stride, int vocab, int keep, int chunk,
                                                             float2* __restrict__ stats, float* __restrict__ list_values, int* __restrict__ list_index) {
  __shared__ float2 warp_stats[WARPS];
  __shared__ float value_s[WARPS][MAX_KEEP];
  __shared__ int index_s[WARPS][MAX_KEEP];
  pdl_launch_dependents();
  pdl_wait();
  const float* row = logits + (size_t)blockIdx.y * row_stride;
  const int lo = blockIdx.x * chunk, hi = min(vocab, lo + chunk);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float m = -INFINITY, sum = 0.f;
  Best<float> best;
  best.clear();
  for (int at = lo + warp * 32 * UNROLL; at < hi; at += THREADS * UNROLL) {
    float x[UNROLL];
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) x[i] = at + i * 32 + lane < hi ? row[at + i * 32 + lane] : -INFINITY;
    float top = m;
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) top = fmaxf(top, x[i]);
    const float base = top == -INFINITY ? 0.f : top;
    sum *= fast_exp2((m - base) * 1.4426950408889634f);
    m = top;
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) sum += fast_exp2((x[i] - base) * 1.4426950408889634f);
    const float last = __shfl_sync(0xffffffffu, best.value, keep - 1);
    if (__any_sync(0xffffffffu, top >= last)) {
#pragma unroll
      for (int i = 0; i < UNROLL; ++i) best.offer(x[i], at + i * 32 + lane, keep);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, m, o), os = __shfl_xor_sync(0xffffffffu, sum, o);
    const float top = fmaxf(m, om), base = top == -INFINITY ? 0.f : top;
    sum = sum * fast_exp2((m - base) * 1.4426950408889634f) + os * fast_exp2((om - base) * 1.4426950408889634f);
    m = top;
  }
  if (lane == 0) warp_stats[warp] = make_float2(m, sum);
  value_s[warp][lane] = best.value;
  index_s[warp][lane] = best.index;
  __syncthreads();
  if (warp == 0) {
    for (int w = 1; w < WARPS; ++w) best.offer(lane < keep ? value_s[w][lane] : -INFINITY, index_s[w][lane], keep);
    const size_t at = (size_t)blockIdx.y * gridDim.x + blockIdx.x;
    if (lane < keep) { list_values[at * keep + lane] = best.value; list_index[at * keep + lane] = best.index; }
    if (lane == 0) {
      float2 all = warp_stats[0];
      for (int w = 1; w < WARPS; ++w) {
        const float2 other = warp_stats[w];
        const float top = fmaxf(all.x, other.x), base = top == -INFINITY ? 0.f : top;
        all.y = all.y * expf(all.x - base) + other.y * expf(other.x - base);
        all.x = top;
      }
      stats[at] = all;
    }
  }
}

__global__ void __launch_bounds__(THREADS) beam_join_kernel(const float* __restrict__ scores, const int* __restrict__ ended, int beams, int vocab, int keep,
                                                            int pad, int chunks, const float2* __restrict__ stats, const float* __restrict__ list_values,
                                                            const int* __restrict__ list_index, float* __restrict__ next_scores,
                                                            int* __restrict__ parents, int* __restrict__ tokens) {
  __shared__ double value_s[WARPS][MAX_KEEP];
  __shared__ int index_s[WARPS][MAX_KEEP];
  pdl_launch_dependents();
  pdl_wait();
  const int request = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  Best<double> best;
  best.clear();
  for (int b = warp; b < beams; b += WARPS) {
    const size_t row = (size_t)request * beams + b;
    const float score = scores[row];
    if (!(score > -INFINITY)) continue;
    if (ended && ended[row]) {
      best.offer(lane == 0 ? (double)score : (double)-INFINITY, b * vocab + pad, keep);
      continue;
    }
    const float2* mine = stats + row * chunks;
    float m = -INFINITY;
    for (int c = lane; c < chunks; c += 32) m = fmaxf(m, mine[c].x);
    m = warp_max(m);
    double sum = 0.0;
    for (int c = lane; c < chunks; c += 32) {
      const float2 part = mine[c];
      if (part.y != 0.f) sum += (double)part.y * exp((double)part.x - (double)m);      // a chunk without a finite value has a sum of 0
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const double offset = (double)score - (double)m - log(sum);
    if (!isfinite(offset)) continue;
    for (int c0 = 0; c0 < chunks * keep; c0 += 32) {
      const int c = c0 + lane;
      const bool there = c < chunks * keep;
      const float logit = there ? list_values[row * chunks * keep + c] : -INFINITY;
      best.offer(offset + (double)logit, there && logit > -INFINITY ? b * vocab + list_index[row * chunks * keep + c] : 0x7fffffff, keep);
    }
  }
  value_s[warp][lane] = best.value;
  index_s[warp][lane] = best.index;
  __syncthreads();
  if (warp == 0) {
    for (int w = 1; w < WARPS; ++w) best.offer(lane < keep ? value_s[w][lane] : (double)-INFINITY, index_s[w][lane], keep);
    if (lane < keep) {
      const bool none = best.index == 0x7fffffff;
      const size_t at = (size_t)request * keep + lane;
      next_scores[at] = (float)best.value;
      parents[at] = none ? -1 : best.index / vocab;
      tokens[at] = none ? -1 : best.index % vocab;
    }
  }
}
}  // namespace

// The longest chunk of a row that a block of the first kernel takes is `chunk`; scratch: rows * chunks * (2 + 2 keep) words, chunks =
// ceil(vocab / chunk).
LB_EXPORT int lb_beam_select(const float* logits, long row_stride, const float* scores, const int* ended, int requests, int beams, int vocab, int keep,
                             int pad, int chunk, void* scratch, long scratch_words, float* next_scores, int* parents, int* tokens, cudaStream_t stream) {
  if (requests <= 0) return 0;
  if (beams <= 0 || beams > MAX_BEAMS || keep <= 0 || keep > MAX_KEEP || vocab <= 0 || chunk <= 0 || pad < 0 || pad >= vocab ||
      (long)beams * vocab >= 0x7fffffffL || (long)requests * beams > 65535)
    return LB_ERR_SIZE;
  const long rows = (long)requests * beams, chunks = (vocab + (long)chunk - 1) / chunk;
  if (scratch_words < rows * chunks * (2 + 2 * keep)) return LB_ERR_SIZE;
  if ((uintptr_t)scratch & 7) return LB_ERR_ALIGN;
  float2* stats = (float2*)scratch;
  float* values = (float*)scratch + rows * chunks * 2;
  int* index = (int*)(values + rows * chunks * keep);
  int code = lb_launch(beam_chunk_kernel, dim3((unsigned)chunks, (unsigned)rows), THREADS, 0, stream, logits, row_stride, vocab, keep, chunk, stats, values, index);
  if (code) return code;
  code = lb_launch(beam_join_kernel, requests, THREADS, 0, stream, scores, ended, beams, vocab, keep, pad, (int)chunks, stats, values, index, next_scores,
                   parents, tokens);
  return code ? code : lb_last_error();
}

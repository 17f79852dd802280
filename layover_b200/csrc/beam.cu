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
// groups' own maxima in the first piece. Every warp collects what reaches it by itself (a barrier a piece and a counter of the block cost 11 of
// 27 us at 128 rows of 151,936), keeps the best of it when it gets much, which gives a higher threshold, and at the end a threshold
// of the same kind, over the whole chunk, leaves a few to be ranked by counting. Within a beam the order is that of the logits
// themselves, so no rounding is involved. The second kernel has one block a request: the beams' sums are joined in 64 bits, and of the
// chunks' lists the candidates are compared in 64 bits behind a threshold of the same kind, where two beams' tie only where the formula's
// do within 1e-7; where more reach it than there is room for (many equal ones), the best are picked one by one.
//
// The logits' bytes bound it in theory. Measured (one B200): 128 rows of 151,936, a fifth of the beams ended, 16 kept 26 us, of them 18 to 20 the
// first kernel (3.3 TB/s of what it reads: a block's first piece, its thresholds and ranking run alone), 64 rows 14 us, 4 rows 8 us, two launches
// of about 4 that wait for memory twice.
#include <float.h>
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

// The best `keep` of the warp's `n` values (keep < n <= WARP_ROOM) are left in `found`, best first; the last of them.
constexpr int WARP_ROOM = 128;
__device__ __noinline__ float keep_best(const float* __restrict__ row, int* found, float* worth, int n, int keep) {
  const int lane = threadIdx.x & 31;
  float v[WARP_ROOM / 32];
  int i[WARP_ROOM / 32], rank[WARP_ROOM / 32];
  __syncwarp();
#pragma unroll
  for (int c = 0; c < WARP_ROOM / 32; ++c) {
    rank[c] = 0; i[c] = NONE; v[c] = -INFINITY;
    if (lane + 32 * c < n) {
      i[c] = found[lane + 32 * c]; v[c] = row[i[c]];
      worth[lane + 32 * c] = v[c];
    }
  }
  __syncwarp();
  for (int o = 0; o < n; ++o) {
    const float other = worth[o];
    const int index = found[o];
#pragma unroll
    for (int c = 0; c < WARP_ROOM / 32; ++c) rank[c] += before(other, index, v[c], i[c]) ? 1 : 0;
  }
  __syncwarp();
#pragma unroll
  for (int c = 0; c < WARP_ROOM / 32; ++c)
    if (lane + 32 * c < n && rank[c] < keep) { found[rank[c]] = i[c]; worth[rank[c]] = v[c]; }
  __syncwarp();
  return worth[keep - 1];
}

// A value that at least `keep` of the block's reach, found from the maxima of 64 groups of four threads: the keep-th largest of those, up to
// its last six bits, which make way for the group's number so that no two are equal. Not below the lowest finite number: -inf is no candidate.
__device__ __forceinline__ float reached_by(float top, int keep, int* keys, float* result) {
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const int bits = __float_as_int(top), key = bits ^ (bits >> 31 & 0x7fffffff);      // in the order of the numbers
  if ((threadIdx.x & 3) == 0) keys[threadIdx.x >> 2] = (key & ~63) | threadIdx.x >> 2;
  __syncthreads();
  if (threadIdx.x < 64) {
    const int mine = keys[threadIdx.x], low = mine & ~63;
    int rank = 0;
#pragma unroll
    for (int t = 0; t < 64; t += 4) {
      const int4 k = *reinterpret_cast<const int4*>(keys + t);
      rank += (k.x > mine ? 1 : 0) + (k.y > mine ? 1 : 0) + (k.z > mine ? 1 : 0) + (k.w > mine ? 1 : 0);
    }
    if (rank == keep - 1) *result = fmaxf(__int_as_float(low ^ (low >> 31 & 0x7fffffff)), -FLT_MAX);      // what is below -inf is NaN
  }
  __syncthreads();
  return *result;
}

// stats [rows][chunks] (maximum, sum of exp(x - maximum)), lists [rows][chunks][keep] of (value, index), best first, (-inf, NONE) behind the last.
// A chunk is `pieces` of PIECE values. Rows of beams that are not there or have ended are not read, and nothing is written for them.
constexpr int EACH = 14, PIECE = THREADS * EACH;
__global__ void __launch_bounds__(THREADS, 4) beam_chunk_kernel(const float* __restrict__ logits, long row_stride, const float* __restrict__ scores,
                                                                const int* __restrict__ ended, int vocab, int keep, int pieces, int chunks,
                                                                float2* __restrict__ stats, float2* __restrict__ lists) {
  __shared__ __align__(16) int keys[64];
  __shared__ float worth[WARPS][WARP_ROOM], part[WARPS], part_sum[WARPS], threshold, last_threshold;
  __shared__ float2 all_best[THREADS];
  __shared__ int found[WARPS][WARP_ROOM], total;
  pdl_launch_dependents();
  pdl_wait();
  const int row_at = blockIdx.x / chunks;
  const float* row = logits + (size_t)row_at * row_stride;
  const int begin = (blockIdx.x - row_at * chunks) * pieces * PIECE, end = min(vocab, begin + pieces * PIECE), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float next[EACH], m = -INFINITY, sum = 0.f, bar = -FLT_MAX;      // what does not reach `bar` is not among the best
  int held = 0;                                            // indices in `found` of this warp, in their order
  const bool wanted = scores[row_at] > -INFINITY && !(ended && ended[row_at]);
#pragma unroll
  for (int j = 0; j < EACH; ++j) next[j] = begin + (int)threadIdx.x + j * THREADS < end ? row[begin + threadIdx.x + j * THREADS] : -INFINITY;
  if (!wanted) return;                                     // the first piece was asked for all the same: the others would wait for this
  if (threadIdx.x == 0) total = 0;
  for (int from = begin; from < end; from += PIECE) {
    const int lo = from + threadIdx.x;
    float x[EACH];
#pragma unroll
    for (int j = 0; j < EACH; ++j) x[j] = next[j];
    const float* behind = row + lo + PIECE;                // the next piece is on its way while this one is looked at
    if (from + 2 * PIECE <= end) {
#pragma unroll
      for (int j = 0; j < EACH; ++j) next[j] = behind[j * THREADS];
    } else {
#pragma unroll
      for (int j = 0; j < EACH; ++j) next[j] = lo + PIECE + j * THREADS < end ? behind[j * THREADS] : -INFINITY;
    }
    float top = -INFINITY;                                 // of numbers: NaN is no maximum, but the sum becomes it
#pragma unroll
    for (int j = 0; j < EACH; ++j) top = fmaxf(top, x[j]);
    if (from == begin) bar = reached_by(top, keep, keys, &threshold);
    const float rise = fmaxf(m, top), base = rise == -INFINITY ? 0.f : rise;
    sum *= fast_exp2((m - base) * LOG2E);
    m = rise;
#pragma unroll
    for (int j = 0; j < EACH; ++j) sum += fast_exp2((x[j] - base) * LOG2E);
    unsigned hits = 0, any;
    if (top >= bar) {
#pragma unroll
      for (int j = 0; j < EACH; ++j) hits |= x[j] >= bar ? 1u << j : 0u;
    }
    for (any = __reduce_or_sync(0xffffffffu, hits); any; any &= any - 1) {      // in the order of the indices
      const int j = __ffs(any) - 1;
      const unsigned with = __ballot_sync(0xffffffffu, hits >> j & 1u);
      if (hits >> j & 1u) found[warp][held + __popc(with & ((1u << lane) - 1u))] = lo + j * THREADS;
      held += __popc(with);
      if (held > WARP_ROOM - 32) {                         // what comes behind and equals the last of the best is not among them
        bar = nextafterf(keep_best(row, found[warp], worth[warp], held, keep), INFINITY);
        held = keep;
        unsigned still = 0;
#pragma unroll
        for (int e = 0; e < EACH; ++e) still |= x[e] >= bar ? 1u << e : 0u;
        hits &= still;
        any &= __reduce_or_sync(0xffffffffu, hits) | (1u << j);
      }
    }
  }
  if (held > 32) {
    keep_best(row, found[warp], worth[warp], held, keep);
    held = keep;
  }
  // the maximum and the sum of all threads, and of what the warps hold that which reaches a threshold of the whole chunk
  int i = NONE;
  float v = -INFINITY;
  if (lane < held) { i = found[warp][lane]; v = row[i]; }
  const float top = warp_max(m), base = top == -INFINITY ? 0.f : top;
  sum = warp_sum(sum * fast_exp2((m - base) * LOG2E));
  if (lane == 0) { part[warp] = top; part_sum[warp] = sum; }
  bar = reached_by(m, keep, keys, &last_threshold);
  const unsigned with = __ballot_sync(0xffffffffu, v >= bar);
  int at = 0;
  if (lane == 0 && with) at = atomicAdd(&total, __popc(with));      // any order: they are ranked
  at = __shfl_sync(0xffffffffu, at, 0) + __popc(with & ((1u << lane) - 1u));
  if (v >= bar) all_best[at] = make_float2(v, __int_as_float(i));
  __syncthreads();
  const size_t chunk = blockIdx.x;
  float2* list = lists + chunk * keep;
  const int n = total;                                     // 32 of each warp at most
  if ((int)threadIdx.x < n) {
    const float2 mine = all_best[threadIdx.x];
    int rank = 0;
    for (int o = 0; o < n; ++o) {
      const float2 other = all_best[o];
      rank += before(other.x, __float_as_int(other.y), mine.x, __float_as_int(mine.y)) ? 1 : 0;
    }
    if (rank < keep) list[rank] = mine;
  } else if ((int)threadIdx.x < keep) {
    list[threadIdx.x] = make_float2(-INFINITY, __int_as_float(NONE));
  }
  if (warp == WARPS - 1) {
    const float mine = lane < WARPS ? part[lane] : -INFINITY, all = warp_max(mine), from = all == -INFINITY ? 0.f : all;
    const float sums = warp_sum(lane < WARPS ? part_sum[lane] * fast_exp2((mine - from) * LOG2E) : 0.f);
    if (lane == 0) stats[chunk] = make_float2(all, sums);
  }
}

__global__ void __launch_bounds__(THREADS) beam_join_kernel(const float* __restrict__ scores, const int* __restrict__ ended, int beams, int vocab, int keep,
                                                            int pad, int chunks, const float2* __restrict__ stats, const float2* __restrict__ lists,
                                                            float* __restrict__ next_scores, int* __restrict__ parents, int* __restrict__ tokens) {
  __shared__ double offsets[MAX_BEAMS];                    // what a beam's logits are raised by; its own score where it has ended; -inf: no beam
  __shared__ bool over[MAX_BEAMS];
  __shared__ double values[ROOM], part[WARPS];
  __shared__ __align__(16) int keys[64];
  __shared__ float threshold;
  __shared__ int indices[ROOM], part_index[WARPS];
  __shared__ int count;
  pdl_launch_dependents();
  pdl_wait();
  const int request = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, n_lists = beams * chunks;
  const float2* mine = lists + (size_t)request * n_lists * keep;
  // A thread's candidates, of all lists' one after the other; those of the four threads of a group lie 64 apart, so that what is best of a list is in
  // several groups. The first four are on their way while the sums are joined.
  const int n_candidates = n_lists * keep, at0 = (threadIdx.x & 3) * 64 + (threadIdx.x >> 2);
  constexpr int FIRST = 4;
  float2 held[FIRST];
#pragma unroll
  for (int k = 0; k < FIRST; ++k) held[k] = at0 + k * THREADS < n_candidates ? mine[at0 + k * THREADS] : make_float2(-INFINITY, 0.f);
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
  // candidate c, which the lists have as x: an ended beam has one, in its first list
  auto candidate = [&](int c, float2 x, double& v, int& i) {
    const int l = c / keep, b = l / chunks;
    v = -INFINITY; i = NONE;
    if (offsets[b] == -INFINITY) return;
    if (over[b]) {
      if (c == b * chunks * keep) { v = offsets[b]; i = b * vocab + pad; }
      return;
    }
    if (x.x > -INFINITY) { v = offsets[b] + (double)x.x; i = b * vocab + __float_as_int(x.y); }
  };
  auto all = [&](auto look) {
#pragma unroll
    for (int k = 0; k < FIRST; ++k) {
      double v;
      int i;
      if (at0 + k * THREADS >= n_candidates) return;
      candidate(at0 + k * THREADS, held[k], v, i);
      look(v, i);
    }
    for (int c = at0 + FIRST * THREADS; c < n_candidates; c += THREADS) {
      double v;
      int i;
      candidate(c, mine[c], v, i);
      look(v, i);
    }
  };
  double best = -INFINITY;
  all([&](double v, int) { best = v > best ? v : best; });
  // a value that `keep` candidates reach; the lowest one stands for none
  const float lowest = reached_by(__double2float_rd(best), keep, keys, &threshold);
  const double reach = lowest == -FLT_MAX ? -INFINITY : (double)lowest;
  if (best >= reach)
    all([&](double v, int i) {
      if (v >= reach && i != NONE) {
        const int at = atomicAdd(&count, 1);
        if (at < ROOM) { values[at] = v; indices[at] = i; }
      }
    });
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
      all([&](double w, int j) {
        if (j != NONE && before(last, last_index, w, j) && before(w, j, v, i)) { v = w; i = j; }
      });
      block_best(v, i, part, part_index);
      if (threadIdx.x == 0) choose(k, v, i);
      last = v; last_index = i;
    }
  }
}
}  // namespace

// A block of the first kernel takes `pieces` of PIECE values, chunks = ceil(vocab / (pieces * PIECE)). Scratch: rows * chunks * (2 + 2 keep) words.
LB_EXPORT int lb_beam_select(const float* logits, long row_stride, const float* scores, const int* ended, int requests, int beams, int vocab, int keep,
                             int pad, int pieces, void* scratch, long scratch_words, float* next_scores, int* parents, int* tokens, cudaStream_t stream) {
  if (requests <= 0) return 0;
  if (beams <= 0 || beams > MAX_BEAMS || keep <= 0 || keep > MAX_KEEP || vocab <= 0 || pieces <= 0 || pieces > 0x7fffffff / PIECE || pad < 0 || pad >= vocab ||
      (long)beams * vocab > 0x7fffffffL - (pieces + 2L) * PIECE)      // places, and the ends of chunks and of the pieces ahead, are counted in 32 bits
    return LB_ERR_SIZE;
  const long rows = (long)requests * beams, chunks = (vocab + (long)PIECE * pieces - 1) / ((long)PIECE * pieces);
  if (rows * chunks > 0x7fffffffL) return LB_ERR_SIZE;
  if (scratch_words < rows * chunks * (2 + 2 * keep)) return LB_ERR_SIZE;
  if ((uintptr_t)scratch & 7) return LB_ERR_ALIGN;
  float2 *stats = (float2*)scratch, *lists = stats + rows * chunks;
  int code = lb_launch(beam_chunk_kernel, dim3((unsigned)(rows * chunks)), THREADS, 0, stream, logits, row_stride, scores, ended, vocab, keep, pieces, (int)chunks, stats, lists);
  if (code) return code;
  code = lb_launch(beam_join_kernel, requests, THREADS, 0, stream, scores, ended, beams, vocab, keep, pad, (int)chunks, stats, lists, next_scores, parents, tokens);
  return code ? code : lb_last_error();
}

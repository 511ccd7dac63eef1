// Beam search: the choice of the next beams.
//
// Beam j of a sequence carries the score s_j (a sum of log probabilities); token v after it is worth
//     c(j, v) = s_j + x_jv - ln sum_u exp(x_ju)
// and the `width` largest of a sequence's beams x vocabulary are wanted in order, ties to the lowest j * V + v.  One pass over
// the logits does both halves: a block holds its stretch of a row in registers, takes the stretch's maximum and sum of
// exponentials, and lists the stretch's `width` largest logits (within a row the logits' order is the candidates').  A second
// kernel joins a sequence's stretches: the rows' log sums, then the `width` largest candidates of all lists, compared in 64
// bits, so that the order between two beams does not hang on the rounding of a sum.
// What is kept of a stretch must hold its `width` largest, and few more: with the k-th largest of every warp's 32 lane maxima,
// k = ceil(width / warps), at least `width` logits reach the smallest of the warps' values.  Whatever reaches it goes to a list
// in shared memory and is put in order by counting.  A list that overflows (rows of equal logits) is made by `width` rounds
// of a block maximum instead.
// Bound: the logits' bytes; about ten instructions a logit (one exponential) leave room for them.
#include <math.h>

#include "api.h"
#include "common.cuh"

namespace {

typedef unsigned long long u64;

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int MAX_WIDTH = 64, MAX_BEAMS = 64;
constexpr int CAP = 512;            // entries of a block's list

// Order of floats as order of unsigned numbers; -inf gives the smallest key that occurs.
__device__ __forceinline__ unsigned order_key(float v) {
  v += 0.0f;                          // -0 and +0 are equal
  const unsigned b = __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(unsigned k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
constexpr unsigned KEY_NONE = 0x007fffffu;    // order_key(-inf)

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void load(const float* p, float* x) {
    const float4 v = __ldcs(reinterpret_cast<const float4*>(p));
    x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
  }
};
template <> struct Vec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void load(const __nv_bfloat16* p, float* x) {
    const uint4 v = __ldcs(reinterpret_cast<const uint4*>(p));
    const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};

// One stretch of one row.  `stretch` numbers (a multiple of a vector); the stretch's aligned middle comes in vectors, the few
// numbers before and after it one by one (rows of an odd length start on no boundary).
// part_stat [row][stretches]: (maximum, sum of exponentials above it); part_key [row][stretches][width]: logits in descending
// order as (order of the value, ~token), 0 where there are no more.
template <typename T, int VECS>
__global__ void __launch_bounds__(THREADS, 2)
beam_stretch_kernel(const T* logits, long ld, int vocab, int stretch, int width, double2* __restrict__ part_stat, u64* __restrict__ part_key) {
  constexpr int N = Vec<T>::N;
  __shared__ unsigned s_kth[WARPS];
  __shared__ float s_max[WARPS];
  __shared__ double s_sum[WARPS];
  __shared__ u64 s_list[CAP];
  __shared__ u64 s_best[WARPS];
  __shared__ int s_count;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int part = blockIdx.x, row = blockIdx.y;
  if (tid == 0) s_count = 0;
  gi::pdl_prologue();

  const T* x_row = logits + (size_t)row * ld;
  const int lo = part * stretch, hi = min(vocab, lo + stretch);
  // the first 16-byte boundary at or after the stretch's start, and the last one at or before its end
  const int lead = (int)((16 - ((uintptr_t)(x_row + lo) & 15)) & 15) / (int)sizeof(T);
  const int mid_lo = min(hi, lo + lead), vecs = (hi - mid_lo) / N, mid_hi = mid_lo + vecs * N;
  const int loose = (mid_lo - lo) + (hi - mid_hi);

  float x[VECS * N + 1];
#pragma unroll
  for (int i = 0; i < VECS; ++i) {
    const int v = i * THREADS + tid;
    if (v < vecs) {
      Vec<T>::load(x_row + mid_lo + v * N, x + i * N);
    } else {
#pragma unroll
      for (int e = 0; e < N; ++e) x[i * N + e] = -INFINITY;
    }
  }
  const int loose_at = tid < mid_lo - lo ? lo + tid : mid_hi + (tid - (mid_lo - lo));
  x[VECS * N] = tid < loose ? gi::ldf(x_row + loose_at) : -INFINITY;
  auto token_of = [&](int i) { return i < VECS * N ? mid_lo + ((i / N) * THREADS + tid) * N + i % N : loose_at; };

  float mine = -INFINITY;
#pragma unroll
  for (int i = 0; i <= VECS * N; ++i) {
    x[i] = fmaxf(x[i], -INFINITY);          // what is no number counts as -inf
    mine = fmaxf(mine, x[i]);
  }
  // the k-th largest of the warp's lane maxima
  const int k = (width + WARPS - 1) / WARPS;
  unsigned key = order_key(mine), kth = 0, warp_key = 0;
  for (int r = 0; r < k; ++r) {
    kth = __reduce_max_sync(0xffffffffu, key);
    if (r == 0) warp_key = kth;
    const unsigned who = __ballot_sync(0xffffffffu, key == kth);
    if (lane == __ffs(who) - 1) key = 0;
  }
  if (lane == 0) {
    s_kth[warp] = kth;
    s_max[warp] = key_value(warp_key);
  }
  __syncthreads();
  float top = s_max[0];
  unsigned bar = s_kth[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) {
    top = fmaxf(top, s_max[w]);
    bar = min(bar, s_kth[w]);
  }
  const float floor_ = key_value(max(bar, KEY_NONE));
  // the sum of exponentials: in 32 bits over a thread's numbers, in 64 from there on
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
  const float base = top > -INFINITY ? top : 0.f;
#pragma unroll
  for (int i = 0; i <= VECS * N; ++i) {
    sum[i & 3] += ex2((x[i] - base) * 1.4426950408889634f);
    if (x[i] >= floor_ && x[i] > -INFINITY) {
      const int at = atomicAdd(&s_count, 1);
      if (at < CAP) s_list[at] = ((u64)order_key(x[i]) << 32) | (u64)(~(unsigned)token_of(i));
    }
  }
  double total = (double)sum[0] + sum[1] + ((double)sum[2] + sum[3]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) s_sum[warp] = total;
  __syncthreads();
  const size_t at_part = (size_t)row * gridDim.x + part;
  if (tid == 0) {
    double t = 0.0;
    for (int w = 0; w < WARPS; ++w) t += s_sum[w];
    part_stat[at_part] = make_double2((double)top, t);
  }
  u64* out = part_key + at_part * width;
  const int count = s_count;
  if (count <= CAP) {
    for (int i = tid; i < count; i += THREADS) {
      const u64 own = s_list[i];
      int place = 0;
      for (int o = 0; o < count; ++o) place += s_list[o] > own ? 1 : 0;      // no two are alike
      if (place < width) out[place] = own;
    }
    for (int i = count + tid; i < width; i += THREADS) out[i] = 0;
    return;
  }
  u64 last = ~(u64)0;
  for (int r = 0; r < width; ++r) {
    u64 best = 0;
#pragma unroll
    for (int i = 0; i <= VECS * N; ++i) {
      const u64 own = x[i] > -INFINITY ? ((u64)order_key(x[i]) << 32) | (u64)(~(unsigned)token_of(i)) : 0;
      if (own < last && own > best) best = own;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const u64 other = __shfl_xor_sync(0xffffffffu, best, o);
      best = other > best ? other : best;
    }
    if (lane == 0) s_best[warp] = best;
    __syncthreads();
    best = s_best[0];
#pragma unroll
    for (int w = 1; w < WARPS; ++w) best = s_best[w] > best ? s_best[w] : best;
    __syncthreads();
    if (tid == 0) out[r] = best;
    last = best;
  }
}

// A candidate of the join: worth more, or as much and earlier among beams x vocabulary.
struct Candidate {
  double c;
  long at;
  __device__ __forceinline__ bool before(const Candidate& o) const { return c > o.c || (c == o.c && at < o.at); }
};

// One block joins a sequence's lists (`beams` x `parts`, each in descending order).
__global__ void __launch_bounds__(THREADS)
beam_join_kernel(const float* scores, const double2* part_stat, const u64* part_key, int beams, int parts, int width, int vocab,
                 float* __restrict__ out_scores, int* __restrict__ out_parents, int* __restrict__ out_tokens) {
  extern __shared__ double s_base[];              // [beams], then every list's first candidate [beams * parts]
  __shared__ Candidate s_list[CAP];
  __shared__ Candidate s_best[WARPS];
  __shared__ int s_count;
  __shared__ double s_floor;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int seq = blockIdx.x, lists = beams * parts;
  double* s_head = s_base + beams;
  if (tid == 0) {
    s_count = 0;
    s_floor = -INFINITY;
  }
  gi::pdl_prologue();
  // a row's log sum, its stretches in order
  for (int j = tid; j < beams; j += THREADS) {
    const double2* st = part_stat + (size_t)(seq * beams + j) * parts;
    double top = -INFINITY;
    for (int p = 0; p < parts; ++p) top = fmax(top, st[p].x);
    double sum = 0.0;
    if (top > -INFINITY)
      for (int p = 0; p < parts; ++p) sum += st[p].y * exp(st[p].x - top);
    const double base = (double)scores[(size_t)seq * beams + j] - (top + log(sum));
    s_base[j] = isfinite(base) ? base : -INFINITY;      // nothing but -inf, or a logit that is +inf: the beam offers nothing
  }
  __syncthreads();
  const u64* keys = part_key + (size_t)seq * lists * width;
  auto candidate = [&](int list, int i) {
    const u64 key = keys[(size_t)list * width + i];
    Candidate out;
    const double base = s_base[list / parts];
    out.c = key == 0 || !(base > -INFINITY) ? -INFINITY : base + (double)key_value((unsigned)(key >> 32));
    out.at = (long)(list / parts) * vocab + (long)(~(unsigned)(key & 0xffffffffu));
    return out;
  };
  // a floor that at least `width` candidates reach: the `width`-th largest of the lists' first ones, or, with fewer lists than
  // that, the smallest of the lists' k-th ones
  const int k = (width + lists - 1) / lists;
  for (int l = tid; l < lists; l += THREADS) s_head[l] = candidate(l, k - 1).c;
  __syncthreads();
  const int wanted = min(width, lists) - 1;
  for (int l = tid; l < lists; l += THREADS) {
    const double own = s_head[l];
    int place = 0;
    for (int o = 0; o < lists; ++o) place += (s_head[o] > own || (s_head[o] == own && o < l)) ? 1 : 0;
    if (place == wanted) s_floor = own;
  }
  __syncthreads();
  const double floor_ = s_floor;
  for (int l = tid; l < lists; l += THREADS)
    for (int i = 0; i < width; ++i) {
      const Candidate own = candidate(l, i);
      if (!(own.c >= floor_) || !(own.c > -INFINITY)) break;
      const int at = atomicAdd(&s_count, 1);
      if (at < CAP) s_list[at] = own;
    }
  __syncthreads();
  const int count = s_count;
  auto store = [&](int place, const Candidate& own) {
    const size_t o = (size_t)seq * width + place;
    const bool none = !(own.c > -INFINITY);
    out_scores[o] = (float)own.c;
    out_parents[o] = none ? -1 : (int)(own.at / vocab);
    out_tokens[o] = none ? -1 : (int)(own.at % vocab);
  };
  Candidate none;
  none.c = -INFINITY, none.at = 0;
  if (count <= CAP) {
    for (int i = tid; i < count; i += THREADS) {
      const Candidate own = s_list[i];
      int place = 0;
      for (int o = 0; o < count; ++o) place += s_list[o].before(own) ? 1 : 0;
      if (place < width) store(place, own);
    }
    for (int i = count + tid; i < width; i += THREADS) store(i, none);
    return;
  }
  Candidate last;                                   // (many equal candidates: `width` rounds of a block maximum)
  last.c = INFINITY, last.at = -1;
  for (int r = 0; r < width; ++r) {
    Candidate best = none;
    best.at = 0x7fffffffffffffffL;
    for (int l = tid; l < lists; l += THREADS)
      for (int i = 0; i < width; ++i) {
        const Candidate own = candidate(l, i);
        if (!(own.c > -INFINITY)) break;
        if (last.before(own)) {
          if (own.before(best)) best = own;
          break;                                    // a list is in descending order: what follows is worth less
        }
      }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      Candidate other;
      other.c = __shfl_xor_sync(0xffffffffu, best.c, o);
      other.at = __shfl_xor_sync(0xffffffffu, best.at, o);
      if (other.before(best)) best = other;
    }
    if (lane == 0) s_best[warp] = best;
    __syncthreads();
    best = s_best[0];
    for (int w = 1; w < WARPS; ++w)
      if (s_best[w].before(best)) best = s_best[w];
    __syncthreads();
    if (tid == 0) store(r, best);
    last = best;
  }
}

// How a row is cut: stretches that a block's registers hold, more of them while the launch would leave SMs without a block.
int beam_parts(int rows, int vocab) {
  constexpr int MOST = THREADS * 64;
  int parts = (vocab + MOST - 1) / MOST;
  const int want = (2 * gi::sm_count() + rows - 1) / rows;
  const int fine = (vocab + THREADS * 16 - 1) / (THREADS * 16);
  return parts < want ? (want < fine ? (want > parts ? want : parts) : (fine > parts ? fine : parts)) : parts;
}

template <typename T>
int launch_beam(const T* logits, long ld, int rows, int vocab, int parts, int width, double2* stat, u64* key, cudaStream_t s) {
  constexpr int N = Vec<T>::N;
  // stretches of whole vectors; the loose numbers at both ends of an unaligned one have a register of their own
  const int stretch = ((vocab + parts - 1) / parts + N - 1) / N * N;
  const dim3 grid(parts, rows);
  if (stretch <= THREADS * 16)
    return gi::check(gi::launch(beam_stretch_kernel<T, 16 / N>, grid, dim3(THREADS), 0, s, logits, ld, vocab, stretch, width, stat, key), "beam selection");
  return gi::check(gi::launch(beam_stretch_kernel<T, 64 / N>, grid, dim3(THREADS), 0, s, logits, ld, vocab, stretch, width, stat, key), "beam selection");
}

}  // namespace

extern "C" long gi_beam_select_scratch(int rows, int vocab, int width) {
  if (rows <= 0 || vocab <= 0 || width <= 0) return 0;
  return (long)rows * beam_parts(rows, vocab) * (16 + 8L * width);
}

extern "C" int gi_beam_select(float* out_scores, int* out_parents, int* out_tokens, const void* logits, int dtype, long ld, const float* scores,
                              int seqs, int beams, int vocab, int width, void* scratch, long scratch_bytes, void* stream) {
  if (seqs <= 0) return GI_OK;
  if (beams < 1 || beams > MAX_BEAMS) return gi::fail(GI_ERR_ARG, "beam selection: %d beams, 1 to %d are supported", beams, MAX_BEAMS);
  if (vocab < 1 || ld < vocab) return gi::fail(GI_ERR_ARG, "beam selection: rows of %d logits at a stride of %ld", vocab, ld);
  if (width < 1 || width > MAX_WIDTH || (long)width > (long)beams * vocab)
    return gi::fail(GI_ERR_ARG, "beam selection: a width of %d, 1 to %d (and at most beams x vocabulary) are supported", width, MAX_WIDTH);
  if ((long)seqs * beams > 65535) return gi::fail(GI_ERR_UNSUPPORTED, "beam selection: more than 65535 rows in one launch");
  const int rows = seqs * beams, parts = beam_parts(rows, vocab);
  if (scratch_bytes < gi_beam_select_scratch(rows, vocab, width) || ((uintptr_t)scratch & 15))
    return gi::fail(GI_ERR_ARG, "beam selection: the scratch memory is too small or not aligned");
  double2* stat = (double2*)scratch;
  u64* key = (u64*)(stat + (size_t)rows * parts);
  cudaStream_t s = (cudaStream_t)stream;
  int rc = GI_OK;
  GI_DISPATCH_DTYPE(dtype, T, rc = launch_beam((const T*)logits, ld, rows, vocab, parts, width, stat, key, s));
  if (rc != GI_OK) return rc;
  const size_t smem = (size_t)(beams + beams * parts) * sizeof(double);
  if (smem > 36 * 1024) return gi::fail(GI_ERR_UNSUPPORTED, "beam selection: %d beams over %d stretches", beams, parts);
  return gi::check(gi::launch(beam_join_kernel, dim3(seqs), dim3(THREADS), smem, s, scores, stat, key, beams, parts, width, vocab, out_scores,
                              out_parents, out_tokens), "beam selection (join)");
}

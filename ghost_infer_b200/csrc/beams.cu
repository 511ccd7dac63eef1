// Beam search: the choice of the next beams.
//
// Beam j of a sequence carries the score s_j (a sum of log probabilities); token v after it is worth
//     c(j, v) = s_j + x_jv - ln sum_u exp(x_ju)
// and the `width` largest of a sequence's beams x vocabulary are wanted in order; of equal ones the lowest beam's first, within a
// beam the larger logit (64 bits may not tell two sums apart whose logits differ), then the lowest token.  One pass over
// the logits does both halves: the sum of exponentials, and the `width` largest logits (within a row the logits' order is the
// candidates').  A second kernel joins a sequence's rows: their log sums, then the `width` largest candidates of all lists.
//
// A row's sum is made of pieces that its columns alone name: for every 1,024 of them (a warp's share of a tile) the largest logit
// m and the sum of exp(x - m) in 32 bits, always by the same additions, joined in 64 bits in the pieces' order.  So equal rows have
// equal sums, wherever they start in memory and whatever else the call holds, and their candidates tie as they should.  x - m is
// taken before it is scaled: the error of a sum does not grow with the logits.  With d the mean of m - x under the row's
// probabilities (at most ln V), a log sum is off by at most 2^-22 (an exponential) + 15 * 2^-24 (additions) + d * 2^-22.8 (the
// exponents), under 3e-6 in the worst case; candidates of two beams that are further apart than that come in their true order.
// Above a logit of 1e9 or so the 64 bits of a log sum, m + ln sum exp(x - m), are the coarser ones.
//
// The rows are cut into tiles of 8,192 logits; a block takes an equal range of the tiles of all rows, so that any number of
// rows keeps all SMs busy, and leaves one list for every row it meets.  Tiles come through a ring in shared memory, which keeps
// 96 KB an SM under way with few registers; with the next tile in registers instead, the kernel spilled and took twice as
// long.  A warp fetches its columns of a tile in the aligned 16-byte pieces that hold them (of a row that starts between two
// boundaries one more for every 32) and reads them by column: 256 32-bit rows of 128,255 tokens take 45 us for 43.5 (fetched word by
// word 60, four lanes at a time in the same banks 50), 16-bit ones 43 for 40.
// What enters a part's list must reach a bar that at least `width` of the part's logits reach.  The first bar is the smallest of
// the warps' k-th largest lane maxima in the part's first tile, k = ceil(width / warps).  After the part's tiles 1, 4, 16, ... the list
// is cut down to its `width` best and the bar raised to the last of them: each step then adds about 3 `width` entries.  A
// list that overflows all the same (equal logits) raises the bar and the part is gone through again: entries are ordered by
// value and then place, no two are alike, and the bar rises every time.
// A piece whose sum is no number (a logit was none, or infinite) is added up once more with what is no number as -inf.
// Bound: neither the memory (41 % of its rate) nor the issue slots (20 instructions a logit would fill them for 18 us), but what 20
// warps an SM cannot hide: fixed latencies, the barriers around the lists, SMs that have two blocks and not three.  B200, 32
// sequences of 8 beams over 128,256 tokens, 16 candidates: 43.5 us in all, the join a few of them; one sequence of 4 beams 9.5 us.
#include <math.h>

#include <type_traits>

#include "api.h"
#include "common.cuh"
#include "mma_utils.cuh"

namespace {

typedef unsigned long long u64;

constexpr int THREADS = 256, WARPS = THREADS / 32;
constexpr int MAX_WIDTH = 64, MAX_BEAMS = 64;
constexpr int CAP = 512;                    // entries of a part's list
constexpr int NUMBERS = 32, STAGES = 2;     // numbers of a tile that a thread takes; tiles of the ring
constexpr int TILE = THREADS * NUMBERS;

// Order of floats as order of unsigned numbers; -inf gives the smallest key that occurs.
__device__ __forceinline__ unsigned order_key(float v) {
  v += 0.0f;                          // -0 and +0 are equal
  const unsigned b = __float_as_uint(v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(unsigned k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }
__device__ __forceinline__ u64 entry_of(float v, int token) { return ((u64)order_key(v) << 32) | (u64)(~(unsigned)token); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float LOG2E = 1.4426950408889634f;

// exp(x + shift) of two numbers; the additions and the products of both are one instruction each.
__device__ __forceinline__ float2 exp2_of(float a, float b, float2 shift) {
  float2 d;
  asm("{\n\t.reg .b64 a, s, d, l;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 s, {%4, %5};\n\tmov.b64 l, {%6, %6};\n\tadd.rn.f32x2 d, a, s;\n\t"
      "mul.rn.f32x2 d, d, l;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a), "f"(b), "f"(shift.x), "f"(shift.y), "f"(LOG2E));
  return make_float2(ex2(d.x), ex2(d.y));
}

// A 16-byte piece of a row as it is fetched, and its numbers.
template <typename T> struct Piece;
template <> struct Piece<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void numbers(const uint4& v, float* x) {
    x[0] = __uint_as_float(v.x), x[1] = __uint_as_float(v.y), x[2] = __uint_as_float(v.z), x[3] = __uint_as_float(v.w);
  }
};
template <> struct Piece<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void numbers(const uint4& v, float* x) {
    const unsigned w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};

template <int N>
__device__ __forceinline__ void load(unsigned* w, const unsigned* p) {
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x, w[1] = v.y;
  } else {
    w[0] = *p;
  }
}

// How the rows are cut, the same on both sides.
struct Cut {
  int tiles_row, per, parts;          // tiles of a row, of a block's range; parts of a row that there is room for
  __host__ __device__ int first_block(int row) const { return (int)((long)row * tiles_row / per); }
  __host__ __device__ int last_block(int row) const { return (int)(((long)(row + 1) * tiles_row - 1) / per); }
};

// The `width` best of `count` (at most CAP) entries to the front of s_list, in descending order; all threads call it, between two
// barriers of its own.  Entries that cannot be among them are set aside first by the bar of the first tile's kind.
struct Lists {
  u64 list[CAP], passed[CAP];
  unsigned kth[WARPS];
  int count, passed_count;
  u64 bar;
};

// The smallest of the warps' k-th largest keys (one a lane): at least k * WARPS keys reach it.
__device__ __forceinline__ unsigned low_bar(Lists& s, unsigned key, int k) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned kth = 0;
  for (int r = 0; r < k; ++r) {
    kth = __reduce_max_sync(0xffffffffu, key);
    const unsigned who = __ballot_sync(0xffffffffu, key == kth);
    if (lane == __ffs(who) - 1) key = 0;
  }
  if (lane == 0) s.kth[warp] = kth;
  __syncthreads();
  unsigned bar = s.kth[0];
#pragma unroll
  for (int w = 1; w < WARPS; ++w) bar = min(bar, s.kth[w]);
  return bar;
}

__device__ __forceinline__ void cut_down(Lists& s, int width) {
  const int tid = threadIdx.x, count = min(s.count, CAP);
  if (tid == 0) s.passed_count = 0;
  u64 own[CAP / THREADS];
#pragma unroll
  for (int q = 0; q < CAP / THREADS; ++q) own[q] = q * THREADS + tid < count ? s.list[q * THREADS + tid] : 0;
  u64 most = own[0];
#pragma unroll
  for (int q = 1; q < CAP / THREADS; ++q) most = own[q] > most ? own[q] : most;
  const unsigned bar = low_bar(s, (unsigned)(most >> 32), (width + WARPS - 1) / WARPS);
#pragma unroll
  for (int q = 0; q < CAP / THREADS; ++q)
    if (own[q] != 0 && (unsigned)(own[q] >> 32) >= bar) s.passed[atomicAdd(&s.passed_count, 1)] = own[q];
  __syncthreads();
  const int passed = s.passed_count;
  for (int i = tid; i < passed; i += THREADS) {
    const u64 mine = s.passed[i];
    int place = 0;
    for (int o = 0; o < passed; ++o) place += s.passed[o] > mine ? 1 : 0;
    if (place < width) s.list[place] = mine;
    if (place == width - 1) s.bar = mine;
  }
  if (tid == 0) s.count = min(count, width);
  __syncthreads();
}

// row_sum [row][tile][warp]: (m, sum of exp(x - m)) of the warp's columns; part_key [row][parts][width]: logits in descending
// order as (order of the value, ~token), 0 where there are no more.
template <typename T>
__global__ void __launch_bounds__(THREADS, 3)
beam_rows_kernel(const T* logits, long ld, int vocab, int rows, Cut cut, int width, float2* __restrict__ row_sum, u64* __restrict__ part_key) {
  constexpr int N = Piece<T>::N, VPT = NUMBERS / N, WARP_PIECES = 33;
  extern __shared__ __align__(16) unsigned char smem[];
  uint4* ring = (uint4*)smem;                        // [STAGES][VPT][WARPS][33 pieces]
  __shared__ Lists s;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  gi::pdl_prologue();
  const long lo = (long)blockIdx.x * cut.per, hi = min((long)rows * cut.tiles_row, lo + cut.per);

  // a place in the list of tiles, counted up without divisions
  struct Place {
    int left, row, tile, stage;                      // tiles up to the end of the block's range
    __device__ __forceinline__ void next(int tiles_row) {
      --left;
      if (++tile == tiles_row) tile = 0, ++row;
      if (++stage == STAGES) stage = 0;
    }
  };
  Place here;
  here.left = (int)max(0L, hi - lo), here.row = (int)(lo / cut.tiles_row), here.tile = (int)(lo - (long)here.row * cut.tiles_row), here.stage = 0;
  Place asked = here;                                // the next tile to ask for
  // A row's numbers i N ... i N + N - 1 lie in piece i of 16 bytes from the last boundary before the row on, and where the row starts
  // behind that boundary, in piece i + 1.  Nothing past the row's last byte is fetched; what is fetched in front of its first one
  // lies in the same 16 bytes as that.
  auto ask = [&]() {
    if (asked.left > 0) {
      const uintptr_t first = (uintptr_t)(logits + (size_t)asked.row * ld), from = first & ~(uintptr_t)15, end = first + (size_t)vocab * sizeof(T);
      uint4* to = ring + (asked.stage * VPT * WARPS + warp) * WARP_PIECES;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const uintptr_t at = from + ((size_t)(asked.tile * VPT + i) * THREADS + tid) * 16;
        if (at < end) gi::cp_async_16(gi::smem_u32(to + i * WARPS * WARP_PIECES + lane), (const void*)at, (int)min(end - at, (uintptr_t)16));
      }
      if (from != first && lane < VPT) {              // a lane each: the piece behind the warp's last one
        const uintptr_t at = from + ((size_t)(asked.tile * VPT + lane) * THREADS + warp * 32 + 32) * 16;
        if (at < end) gi::cp_async_16(gi::smem_u32(to + lane * WARPS * WARP_PIECES + 32), (const void*)at, (int)min(end - at, (uintptr_t)16));
      }
    }
    asked.next(cut.tiles_row);
    gi::cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) ask();

  Place part = here;                                 // the part's first tile
  int next_cut = 1;                                  // tiles of the part after which its list is cut down
  bool keep_bar = false;                             // the part is gone through again
  while (here.left > 0) {
    const int row = here.row, tile = here.tile;
    __syncwarp();                                    // (a warp's lanes read one another's pieces)
    ask();
    gi::cp_async_wait<STAGES - 1>();
    __syncwarp();
    const unsigned off = (unsigned)(uintptr_t)(logits + (size_t)row * ld) & 15u;
    const unsigned char* from = (const unsigned char*)(ring + (here.stage * VPT * WARPS + warp) * WARP_PIECES + lane) + off;
    constexpr int STEP = WARPS * WARP_PIECES * 16;   // bytes from a thread's piece to its next one
    const int turn = sizeof(T) == 4 && off != 0 ? lane >> 3 : 0;
    auto behind = [&](int i) { return i / N * THREADS * N + (sizeof(T) == 4 ? (i + turn) & 3 : i % N); };      // x[i]'s token behind the first one's
    float x[NUMBERS];
    if (off == 0) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) Piece<T>::numbers(*reinterpret_cast<const uint4*>(from + i * STEP), x + i * N);
    } else if constexpr (sizeof(T) == 4) {
      // word by word, every eight lanes in another order: words of one order lie in eight banks only
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int i = 0; i < VPT; ++i) x[i * N + e] = *reinterpret_cast<const float*>(from + ((e + turn) & 3) * 4 + i * STEP);
    } else {
      // the four words from word `words` of the piece on, and for a row that starts in the middle of a word the one behind them
      auto from_two = [&](auto words) {
        constexpr int W = decltype(words)::value;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          const unsigned* p = reinterpret_cast<const unsigned*>(from - off + i * STEP);
          unsigned w[8];
          if (W < 2) load<4>(w, p);
          else if (W == 2) load<2>(w + 2, p + 2);
          else load<1>(w + 3, p + 3);
          constexpr int MORE = W + 1;
          if (MORE == 1) load<1>(w + 4, p + 4);
          else if (MORE == 2) load<2>(w + 4, p + 4);
          else if (MORE > 2) load<4>(w + 4, p + 4);
          if (off & 2u)
            Piece<T>::numbers(make_uint4(__funnelshift_r(w[W], w[W + 1], 16), __funnelshift_r(w[W + 1], w[W + 2], 16), __funnelshift_r(w[W + 2], w[W + 3], 16),
                                         __funnelshift_r(w[W + 3], w[W + 4], 16)), x + i * N);
          else
            Piece<T>::numbers(make_uint4(w[W], w[W + 1], w[W + 2], w[W + 3]), x + i * N);
        }
      };
      if (off < 4) from_two(std::integral_constant<int, 0>());
      else if (off < 8) from_two(std::integral_constant<int, 1>());
      else if (off < 12) from_two(std::integral_constant<int, 2>());
      else from_two(std::integral_constant<int, 3>());
    }
    const int token0 = (tile * VPT * THREADS + tid) * N;         // piece i's first token: THREADS * N further each
    if ((tile + 1) * (long)TILE > vocab) {
#pragma unroll
      for (int i = 0; i < NUMBERS; ++i)
        if (token0 + behind(i) >= vocab) x[i] = -INFINITY;
    }
    float tops[2] = {-INFINITY, -INFINITY};           // (a maximum passes over what is no number)
#pragma unroll
    for (int i = 0; i < NUMBERS; ++i) tops[i & 1] = fmaxf(tops[i & 1], x[i]);
    const float mine = fmaxf(tops[0], tops[1]);

    const bool first = here.left == part.left;
    if (first) {
      unsigned bar = 0;
      if (!keep_bar) bar = low_bar(s, order_key(mine), (width + WARPS - 1) / WARPS);
      if (tid == 0) {
        s.count = 0;
        if (!keep_bar) s.bar = (u64)bar << 32;
      }
      next_cut = 1;
      __syncthreads();
    }
    const float m = key_value(__reduce_max_sync(0xffffffffu, order_key(mine)));
    float sum = 0.f;
    if (m > -INFINITY) {
      const float2 shift = make_float2(-m, -m);
      auto add_up = [&](auto look) {
        float more[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NUMBERS; i += 2) {
          const float2 e = exp2_of(decltype(look)::value ? fmaxf(x[i], -INFINITY) : x[i], decltype(look)::value ? fmaxf(x[i + 1], -INFINITY) : x[i + 1], shift);
          more[i & 3] += e.x, more[(i & 3) + 1] += e.y;
        }
        // (back in the tokens' order: the sum is the same in every row)
        const float a = turn & 1 ? more[3] : more[0], b = turn & 1 ? more[0] : more[1], c = turn & 1 ? more[1] : more[2], d = turn & 1 ? more[2] : more[3];
        sum = turn & 2 ? (c + d) + (a + b) : (a + b) + (c + d);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      };
      add_up(std::false_type());
      if (__builtin_expect(!(sum < INFINITY), false)) add_up(std::true_type());      // (with m = +inf the sum stays none)
    }
    if (lane == 0) row_sum[((size_t)row * cut.tiles_row + tile) * WARPS + warp] = make_float2(m, sum);

    const u64 bar = s.bar;
    const float bar_value = fmaxf(key_value((unsigned)(bar >> 32)), -3.402823466e38f);      // (-inf is nobody's candidate)
    if (mine >= bar_value) {
      // which of the thread's numbers reach it, and one after the other from where they lie (32 copies of what follows, one for every
      // register, took more time to fetch than to execute)
      unsigned hits = 0;
#pragma unroll
      for (int i = 0; i < NUMBERS; ++i) hits |= x[i] >= bar_value ? 1u << i : 0;
      while (hits != 0) {
        const int i = __ffs(hits) - 1;
        hits &= hits - 1;
        const float v = gi::ldf(reinterpret_cast<const T*>(from + i / N * STEP) + (sizeof(T) == 4 ? (i + turn) & 3 : i % N));
        const u64 own = entry_of(v, token0 + behind(i));
        if (own >= bar) {
          const int to = atomicAdd(&s.count, 1);
          if (to < CAP) s.list[to] = own;
        }
      }
    }
    const bool last = tile + 1 == cut.tiles_row || here.left == 1;
    here.next(cut.tiles_row);
    if (!last && part.left - here.left < next_cut) continue;
    next_cut *= 4;
    __syncthreads();
    const bool over = s.count > CAP;
    cut_down(s, width);
    if (over) {
      // the bar is the `width`-th best of what the list had room for: once more from the part's first tile
      gi::cp_async_wait<0>();
      __syncwarp();
      here = asked = part;
#pragma unroll
      for (int i = 0; i < STAGES - 1; ++i) ask();
      keep_bar = true;
      continue;
    }
    if (!last) continue;
    const size_t out = (size_t)row * cut.parts + (blockIdx.x - cut.first_block(row));
    for (int i = tid; i < width; i += THREADS) part_key[out * width + i] = i < s.count ? s.list[i] : 0;
    __syncthreads();
    keep_bar = false;
    part = here;
  }
  gi::cp_async_wait<0>();
}

// A candidate of the join: its worth, beam and entry (logit and token).
struct Candidate {
  double c;
  u64 key;
  int beam;
  __device__ __forceinline__ bool before(const Candidate& o) const {
    return c > o.c || (c == o.c && (beam < o.beam || (beam == o.beam && key > o.key)));
  }
};

// Order of doubles as order of unsigned numbers.
__device__ __forceinline__ u64 order_key(double v) {
  const u64 b = (u64)__double_as_longlong(v + 0.0);
  return (b >> 63) ? ~b : (b | 0x8000000000000000ull);
}

// One block joins a sequence's lists (those of the parts of its rows).  Every candidate is looked at twice, by all threads side by
// side: for a bar that `width` of them reach (as in the rows' first tiles, on the upper halves of the candidates' keys), and for
// those that reach it, which are put in order by counting.
__global__ void __launch_bounds__(THREADS)
beam_join_kernel(const float* scores, const float2* row_sum, const u64* part_key, int beams, Cut cut, int width,
                 float* __restrict__ out_scores, int* __restrict__ out_parents, int* __restrict__ out_tokens) {
  constexpr int AHEAD = 4;
  __shared__ double s_base[MAX_BEAMS];
  __shared__ int s_parts[MAX_BEAMS];              // parts that a row has
  __shared__ Lists s;
  __shared__ double s_c[CAP];                     // the candidates that pass: worth, and what orders equal ones
  __shared__ u64 s_key[CAP];
  __shared__ int s_beam[CAP];
  __shared__ Candidate s_best[WARPS];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int seq = blockIdx.x, parts = cut.parts, entries = beams * parts * width;
  if (tid < beams) s_parts[tid] = cut.last_block(seq * beams + tid) - cut.first_block(seq * beams + tid) + 1;
  if (tid == 0) s.passed_count = 0;
  __syncthreads();
  gi::pdl_prologue();
  const u64* keys = part_key + (size_t)seq * entries;
  // the first entries' keys are under way while the rows' sums are made; parts that a row does not have count as empty
  auto key_at = [&](int e, int& j) {
    const int list = min(e, entries - 1) / width;
    j = list / parts;
    return e < entries && list - j * parts < s_parts[j] ? keys[e] : 0;
  };
  // Neighbouring entries go to different warps, in another order from list to list: a warp that had the lists of one bad beam
  // alone, or the lists' ends alone, would hold the bar down.
  auto place_of = [&](int q) {
    const int e0 = q * THREADS + lane * WARPS;
    return e0 + ((warp + e0 / width) & (WARPS - 1));
  };
  u64 ahead[AHEAD];
  int beam_ahead[AHEAD];
#pragma unroll
  for (int q = 0; q < AHEAD; ++q) {
    beam_ahead[q] = 0;
    const int e = place_of(q);
    ahead[q] = e < entries ? key_at(e, beam_ahead[q]) : 0;
  }
  // a row's log sum: a warp to a row, a lane to every 32nd piece of it
  const int pieces = cut.tiles_row * WARPS;
  for (int j = warp; j < beams; j += WARPS) {
    const float2* st = row_sum + ((size_t)seq * beams + j) * pieces;
    const double score = (double)scores[(size_t)seq * beams + j];
    double top = -INFINITY, sum = 0.0;
    for (int p0 = lane; p0 < pieces; p0 += 32 * AHEAD) {
      float2 v[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) v[k] = p0 + 32 * k < pieces ? st[p0 + 32 * k] : make_float2(-INFINITY, 0.f);
      double both = top;
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) both = fmax(both, (double)v[k].x);
      if (top > -INFINITY) sum *= exp(top - both);
#pragma unroll
      for (int k = 0; k < AHEAD; ++k) sum += v[k].x > -INFINITY ? (double)v[k].y * exp((double)v[k].x - both) : 0.0;
      top = both;
    }
    double both = top;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) both = fmax(both, __shfl_xor_sync(0xffffffffu, both, o));
    sum = top > -INFINITY ? sum * exp(top - both) : sum;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const double base = score - (both + log(sum));
    if (lane == 0) s_base[j] = isfinite(base) ? base : -INFINITY;      // nothing but -inf, or a logit that is +inf: the beam offers nothing
  }
  __syncthreads();
  auto candidate = [&](u64 key, int j) {
    const double base = s_base[j];
    Candidate own;
    own.c = key == 0 || !(base > -INFINITY) ? -INFINITY : base + (double)key_value((unsigned)(key >> 32));
    own.key = key, own.beam = j;
    return own;
  };
  auto entry = [&](int q, int e) {                  // the q-th of this thread's entries
    if (q < AHEAD) return candidate(ahead[q & (AHEAD - 1)], beam_ahead[q & (AHEAD - 1)]);
    int j;
    const u64 key = key_at(e, j);
    return candidate(key, j);
  };
  unsigned most = 0;
#pragma unroll
  for (int q = 0; q < AHEAD; ++q) {
    const double c = entry(q, 0).c;
    if (c > -INFINITY) most = max(most, (unsigned)(order_key(c) >> 32));
  }
  for (int q = AHEAD; q * THREADS < entries; ++q) {
    const double c = entry(AHEAD, place_of(q)).c;
    if (c > -INFINITY) most = max(most, (unsigned)(order_key(c) >> 32));
  }
  const unsigned bar = low_bar(s, most, (width + WARPS - 1) / WARPS);
  auto pass = [&](const Candidate& own) {
    if (!(own.c > -INFINITY) || (unsigned)(order_key(own.c) >> 32) < bar) return;
    const int at = atomicAdd(&s.passed_count, 1);
    if (at < CAP) s_c[at] = own.c, s_key[at] = own.key, s_beam[at] = own.beam;
  };
#pragma unroll
  for (int q = 0; q < AHEAD; ++q) pass(entry(q, 0));
  for (int q = AHEAD; q * THREADS < entries; ++q) pass(entry(AHEAD, place_of(q)));
  __syncthreads();
  const int count = s.passed_count;
  auto store = [&](int place, const Candidate& own) {
    const size_t o = (size_t)seq * width + place;
    const bool none = !(own.c > -INFINITY);
    out_scores[o] = (float)own.c;
    out_parents[o] = none ? -1 : own.beam;
    out_tokens[o] = none ? -1 : (int)(~(unsigned)(own.key & 0xffffffffu));
  };
  Candidate none;
  none.c = -INFINITY, none.key = 0, none.beam = 0x7fffffff;
  if (count <= CAP) {
    for (int i = tid; i < count; i += THREADS) {
      Candidate own;
      own.c = s_c[i], own.key = s_key[i], own.beam = s_beam[i];
      int place = 0;
#pragma unroll 4
      for (int o = 0; o < count; ++o) {
        const double c = s_c[o];
        if (c > own.c) ++place;
        else if (c == own.c && o != i) place += s_beam[o] < own.beam || (s_beam[o] == own.beam && s_key[o] > own.key) ? 1 : 0;
      }
      if (place < width) store(place, own);
    }
    for (int i = count + tid; i < width; i += THREADS) store(i, none);
    return;
  }
  Candidate last;                                   // (many equal candidates: `width` rounds of a block maximum)
  last.c = INFINITY, last.key = ~(u64)0, last.beam = -1;
  for (int r = 0; r < width; ++r) {
    Candidate best = none;
    for (int e = tid; e < entries; e += THREADS) {
      const Candidate own = entry(AHEAD, e);
      if (own.c > -INFINITY && last.before(own) && own.before(best)) best = own;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      Candidate other;
      other.c = __shfl_xor_sync(0xffffffffu, best.c, o);
      other.key = __shfl_xor_sync(0xffffffffu, best.key, o);
      other.beam = __shfl_xor_sync(0xffffffffu, best.beam, o);
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

struct Plan {
  Cut cut;
  int blocks;
};

template <typename T> constexpr int SMEM_RING = STAGES * (NUMBERS / Piece<T>::N) * WARPS * 33 * 16;

Plan plan_of(int rows, int vocab) {
  Plan p;
  p.cut.tiles_row = (vocab + TILE - 1) / TILE;
  const long slots = 3L * gi::sm_count(), total = (long)rows * p.cut.tiles_row;
  p.cut.per = (int)((total + slots - 1) / slots);
  p.blocks = (int)((total + p.cut.per - 1) / p.cut.per);
  p.cut.parts = (p.cut.tiles_row + p.cut.per - 2) / p.cut.per + 1;
  return p;
}

template <typename T>
int launch_rows(const T* logits, long ld, int vocab, int rows, const Plan& p, int width, float2* sums, u64* key, cudaStream_t s) {
  auto kern = beam_rows_kernel<T>;
  static bool configured[gi::MAX_DEVICES_SEEN] = {false};
  int dev;
  if (gi::unconfigured_here(configured, &dev)) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_RING<T>);
    if (e != cudaSuccess) return gi::fail(GI_ERR_CUDA, "beam selection: %s", cudaGetErrorString(e));
    if (dev >= 0) configured[dev] = true;
  }
  return gi::check(gi::launch(kern, dim3(p.blocks), dim3(THREADS), SMEM_RING<T>, s, logits, ld, vocab, rows, p.cut, width, sums, key), "beam selection");
}

}  // namespace

extern "C" long gi_beam_select_scratch(int rows, int vocab, int width) {
  if (rows <= 0 || vocab <= 0 || width <= 0) return 0;
  const Plan p = plan_of(rows, vocab);
  return (long)rows * (p.cut.tiles_row * (8L * WARPS) + p.cut.parts * (8L * width));
}

extern "C" int gi_beam_select(float* out_scores, int* out_parents, int* out_tokens, const void* logits, int dtype, long ld, const float* scores,
                              int seqs, int beams, int vocab, int width, void* scratch, long scratch_bytes, void* stream) {
  if (seqs <= 0) return GI_OK;
  if (beams < 1 || beams > MAX_BEAMS) return gi::fail(GI_ERR_ARG, "beam selection: %d beams, 1 to %d are supported", beams, MAX_BEAMS);
  if (vocab < 1 || ld < vocab) return gi::fail(GI_ERR_ARG, "beam selection: rows of %d logits at a stride of %ld", vocab, ld);
  if (width < 1 || width > MAX_WIDTH || (long)width > (long)beams * vocab)
    return gi::fail(GI_ERR_ARG, "beam selection: a width of %d, 1 to %d (and at most beams x vocabulary) are supported", width, MAX_WIDTH);
  if ((long)seqs * beams > 0x3fffffL || vocab > 0x3fffffff) return gi::fail(GI_ERR_UNSUPPORTED, "beam selection: %ld rows of %d logits in one launch", (long)seqs * beams, vocab);
  if (dtype != GI_F32 && dtype != GI_BF16) return gi::fail(GI_ERR_ARG, "beam selection: unknown dtype code %d", dtype);
  const int rows = seqs * beams;
  const Plan p = plan_of(rows, vocab);
  if (scratch_bytes < gi_beam_select_scratch(rows, vocab, width) || ((uintptr_t)scratch & 15))
    return gi::fail(GI_ERR_ARG, "beam selection: the scratch memory is too small or not aligned");
  if ((long)beams * p.cut.parts * width > 0x3fffffffL) return gi::fail(GI_ERR_UNSUPPORTED, "beam selection: %d beams in %d parts each", beams, p.cut.parts);
  float2* sums = (float2*)scratch;
  u64* key = (u64*)(sums + (size_t)rows * p.cut.tiles_row * WARPS);
  cudaStream_t s = (cudaStream_t)stream;
  int rc = GI_OK;
  GI_DISPATCH_DTYPE(dtype, T, rc = launch_rows((const T*)logits, ld, vocab, rows, p, width, sums, key, s));
  if (rc != GI_OK) return rc;
  return gi::check(gi::launch(beam_join_kernel, dim3(seqs), dim3(THREADS), 0, s, scores, sums, key, beams, p.cut, width, out_scores,
                              out_parents, out_tokens), "beam selection (join)");
}

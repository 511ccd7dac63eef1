// Attention of drafted tokens over the paged cache: the nodes of one tree per sequence, each of which sees all positions cached
// before the tree and those nodes that its mask names (its ancestors and itself, as a rule).
//
//     o_i = sum_t exp(scale q_i k_t - m) v_t / sum_t exp(scale q_i k_t - m)    over the keys t that node i sees
//
// with the running maximum m and the sums in 32 bits; a node that sees nothing gets zeros.  Keys and values of the step's own
// nodes are in the cache already, at the positions behind the cached ones in the nodes' order.
//
// This file: the form on CUDA cores for 32-bit rows and for head sizes that the tensor-core form (attention_tree_t5.cu) does not
// take, the joining of partial results, and the entry point.  A block takes up to 16 or 64 query rows (nodes x heads of a kv
// head's group, which share every key and value that is read) and a range of tiles of 64 keys (attention_tree.cuh).  Scores are a
// register tile of R / 16 rows by 4 keys a thread, sums of values R / 16 rows by 4 numbers for every 64 of the head; a row's 16
// threads are one half of a warp, so its maximum and sum need no barrier.
// Other head sizes come here in 16 bits too, for which the multiply-adds are far from what tensor cores do: 8 trees of 64 nodes behind
// 8,192 positions, 32 heads over 8, take 1,811 us with heads of 80 and 1,926 with 96, where the tensor-core form takes 78 with heads of 64
// and 88 with 128.
// Bound: 32-bit multiply-adds (2 per query number and key) with many rows, the cache's bytes with few.  B200, 3 trees of 5 to 17
// nodes behind 100 to 701 positions, 32 heads of 64 over 8: 20 to 23 us with the join (two tiles a block 30; breaks inside the inner loops
// for rows that are not there 33; the body for 16 rows beside the one for 64 chosen by unit instead).
#include <float.h>

#include <type_traits>

#include "api.h"
#include "attention_tree.cuh"

namespace {

using namespace gi::tree;

constexpr int THREADS = 256;
constexpr int TILE = 64;

template <typename T, int R, int DCH>
__global__ void __launch_bounds__(THREADS, R == 64 && DCH == 4 ? 1 : 2)
attn_tree_kernel(const Shape sh, T* __restrict__ out, long ldo, const T* q, long ldq, const T* kcache, const T* vcache, int hd, float scale,
                 float4* __restrict__ part_o, float2* __restrict__ part_ml, int* __restrict__ part_prefix, int vec) {
  extern __shared__ __align__(16) float smem[];
  const int hp = (hd + 3) / 4 * 4, ld = hp + 4;    // rows padded: 16 rows' four-number reads fall into different banks
  float* Qs = smem;                                // [R][ld]
  float* Ks = Qs + R * ld;                         // [64][ld]
  float* Vs = Ks + TILE * ld;                      // [64][ld]
  float* Ps = Vs + TILE * ld;                      // [R][68]
  __shared__ int s_pre[MAX_SEQS + 1];
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  gi::pdl_prologue();
  if (tid < 32) prefix(sh, s_pre);
  __syncthreads();
  const int total = s_pre[sh.n_seqs], per = per_range(total, gridDim.x);
  if (blockIdx.x == 0)
    for (int i = tid; i <= sh.n_seqs; i += THREADS) part_prefix[i] = s_pre[i];
  const int lo = (int)min((long)total, (long)blockIdx.x * per), hi = min(total, lo + per);
  const int group = sh.n_heads / sh.n_kv;

  for (int at = lo; at < hi;) {
    const Unit u = unit_at(sh, s_pre, at);
    const int t_begin = at - u.first, t_end = min(u.tiles, hi - u.first);
    const int tok0 = sh.cu_seqlens[u.b], len = u.pos0 + u.n;
    const int rows_here = min(sh.rows_block, u.n * group - u.row0);
    __syncthreads();
    auto work = [&](auto rows_per_thread) {
    constexpr int RT = decltype(rows_per_thread)::value;     // rows a thread works on: ty + 16 i
    // the queries: a row's 16 threads (the half warp that works on it) fetch it, all of a thread's pieces at once
    {
      float4 own[RT][DCH];
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const int r = ty + 16 * i, row = u.row0 + r, node = row / group;
        const T* from = q + (size_t)(tok0 + node) * ldq + (size_t)(u.kvh * group + row - node * group) * hd;
#pragma unroll
        for (int c = 0; c < DCH; ++c) {
          const int d = c * 64 + tx * 4;
          own[i][c] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (r < rows_here) {
            if (vec && d < hd) own[i][c] = gi::ld4(from + d);
            else if (!vec) {
              if (d < hd) own[i][c].x = gi::ldf(from + d);
              if (d + 1 < hd) own[i][c].y = gi::ldf(from + d + 1);
              if (d + 2 < hd) own[i][c].z = gi::ldf(from + d + 2);
              if (d + 3 < hd) own[i][c].w = gi::ldf(from + d + 3);
            }
          }
        }
      }
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int c = 0; c < DCH; ++c)
          if (c * 64 + tx * 4 < hp) *reinterpret_cast<float4*>(Qs + (ty + 16 * i) * ld + c * 64 + tx * 4) = own[i][c];
    }
    float m[RT], l[RT], acc[RT][DCH * 4];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      m[i] = -INFINITY, l[i] = 0.f;
#pragma unroll
      for (int c = 0; c < DCH * 4; ++c) acc[i][c] = 0.f;
    }
    for (int t = t_begin; t < t_end; ++t) {
      const int kt = t * TILE;
      const int page = page_of(sh, u.slot, t);
      const size_t base = ((size_t)page * sh.n_kv + u.kvh) * TILE * hd;
      const bool in_tree = kt + TILE > u.pos0;
      bool spoiled = false;                        // a node's value that is no number, or infinite
      auto look = [&](int r, float v) { spoiled |= in_tree && kt + r >= u.pos0 && !(fabsf(v) < INFINITY); };
      __syncthreads();
      if (vec) {
        const int h4 = hd / 4;
        for (int i0 = tid; i0 < TILE * h4; i0 += 4 * THREADS) {
          float4 kx[4], vx[4];
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int i = i0 + w * THREADS, r = i / h4;
            const bool live = r < TILE && kt + r < len;       // rows past the last node are not read
            kx[w] = live ? gi::ld4(kcache + base + (size_t)i * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
            vx[w] = live ? gi::ld4(vcache + base + (size_t)i * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
          }
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const int i = i0 + w * THREADS, r = i / h4, c = i - r * h4;
            if (r < TILE) {
              *reinterpret_cast<float4*>(Ks + r * ld + 4 * c) = kx[w];
              *reinterpret_cast<float4*>(Vs + r * ld + 4 * c) = vx[w];
              look(r, vx[w].x), look(r, vx[w].y), look(r, vx[w].z), look(r, vx[w].w);
            }
          }
        }
      } else {
        for (int i = tid; i < TILE * hp; i += THREADS) {
          const int r = i / hp, d = i % hp;
          const bool live = kt + r < len && d < hd;
          Ks[r * ld + d] = live ? gi::ldf(kcache + base + (size_t)r * hd + d) : 0.f;
          Vs[r * ld + d] = live ? gi::ldf(vcache + base + (size_t)r * hd + d) : 0.f;
          look(r, Vs[r * ld + d]);
        }
      }
      const bool careful = __syncthreads_or(spoiled);
      float s[RT][4];
#pragma unroll
      for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = 0.f;
#pragma unroll 2
      for (int d = 0; d < hp; d += 4) {
        float4 k4[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) k4[j] = *reinterpret_cast<const float4*>(Ks + (tx + 16 * j) * ld + d);
#pragma unroll
        for (int i = 0; i < RT; ++i) {
          const float4 q4 = *reinterpret_cast<const float4*>(Qs + (ty + 16 * i) * ld + d);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            s[i][j] = fmaf(q4.x, k4[j].x, s[i][j]);
            s[i][j] = fmaf(q4.y, k4[j].y, s[i][j]);
            s[i][j] = fmaf(q4.z, k4[j].z, s[i][j]);
            s[i][j] = fmaf(q4.w, k4[j].w, s[i][j]);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < RT; ++i) {
        const int r = ty + 16 * i;
        unsigned seen[2] = {0xffffffffu, 0xffffffffu};
        if (in_tree) {
          const int* mask = sh.masks + (size_t)(tok0 + min(u.row0 + r, u.n * group - 1) / group) * sh.words;
          seen[0] = seen_word(mask, sh.words, u.n, kt - u.pos0);
          seen[1] = seen_word(mask, sh.words, u.n, kt + 32 - u.pos0);
        }
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int key = tx + 16 * j;
          s[i][j] = (seen[j >> 1] >> (key & 31)) & 1u ? s[i][j] * scale : -INFINITY;
          top = fmaxf(top, s[i][j]);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float m_new = fmaxf(m[i], top), ref = m_new == -INFINITY ? 0.f : m_new;
        const float alpha = m[i] == -INFINITY ? 0.f : expf(m[i] - ref);
        m[i] = m_new;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p = expf(s[i][j] - ref);
          sum += p;
          Ps[r * 68 + tx + 16 * j] = p;
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l[i] = l[i] * alpha + sum;
#pragma unroll
        for (int c = 0; c < DCH * 4; ++c) acc[i][c] *= alpha;
      }
      __syncwarp();
      // a node's value that is no number must not reach those that do not see the node: a weight of zero takes nothing
      auto add_up = [&](auto look_twice) {
#pragma unroll 2
        for (int j = 0; j < TILE; j += 4) {
          float4 p4[RT];
#pragma unroll
          for (int i = 0; i < RT; ++i) p4[i] = *reinterpret_cast<const float4*>(Ps + (ty + 16 * i) * 68 + j);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            float4 v4[DCH];
#pragma unroll
            for (int c = 0; c < DCH; ++c)
              v4[c] = c * 64 + tx * 4 < hp ? *reinterpret_cast<const float4*>(Vs + (j + w) * ld + c * 64 + tx * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int i = 0; i < RT; ++i) {
              const float p = w == 0 ? p4[i].x : w == 1 ? p4[i].y : w == 2 ? p4[i].z : p4[i].w;
              if (decltype(look_twice)::value && p == 0.f) continue;
#pragma unroll
              for (int c = 0; c < DCH; ++c) {
                acc[i][c * 4] = fmaf(p, v4[c].x, acc[i][c * 4]);
                acc[i][c * 4 + 1] = fmaf(p, v4[c].y, acc[i][c * 4 + 1]);
                acc[i][c * 4 + 2] = fmaf(p, v4[c].z, acc[i][c * 4 + 2]);
                acc[i][c * 4 + 3] = fmaf(p, v4[c].w, acc[i][c * 4 + 3]);
              }
            }
          }
        }
      };
      if (!careful) add_up(std::false_type());
      else add_up(std::true_type());
    }
    const bool whole = t_begin == 0 && t_end == u.tiles;
    const size_t slot2 = 2 * (size_t)blockIdx.x + (t_begin == 0 ? 1 : 0);
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int r = ty + 16 * i;
      if (r >= rows_here) continue;
      const int row = u.row0 + r;
      T* dst = out + (size_t)(tok0 + row / group) * ldo + (size_t)(u.kvh * group + row % group) * hd;
      const float inv = l[i] == 0.f ? 0.f : 1.0f / l[i];
#pragma unroll
      for (int c = 0; c < DCH; ++c) {
        const int d = c * 64 + tx * 4;
        if (whole) {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (d + e < hd) gi::stf(dst + d + e, acc[i][c * 4 + e] * inv);
        } else if (d < hd) {
          part_o[part_at(sh, slot2, hp / 4, d / 4, r)] = make_float4(acc[i][c * 4], acc[i][c * 4 + 1], acc[i][c * 4 + 2], acc[i][c * 4 + 3]);
        }
      }
      if (!whole && tx == 0) part_ml[slot2 * sh.rows_block + r] = make_float2(m[i], l[i]);
    }
    };
    // (a unit of few rows, as the last row block of a tree or a small tree's, is not worked on as if it were full)
    if (rows_here <= 16) work(std::integral_constant<int, 1>());
    else work(std::integral_constant<int, R / 16>());
    at = u.first + t_end;
  }
}

// N neighbouring numbers, in as few stores as their type allows where the rows are aligned to them.
template <int N>
__device__ __forceinline__ void store_row(float* dst, const float (&o)[N], int count, bool vec) {
  if (vec && count >= N) {
    if constexpr (N >= 4) {
#pragma unroll
      for (int e = 0; e < N; e += 4) gi::st4(dst + e, make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]));
    } else {
      *reinterpret_cast<float2*>(dst) = make_float2(o[0], o[1]);
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (e < count) dst[e] = o[e];
}
template <int N>
__device__ __forceinline__ void store_row(__nv_bfloat16* dst, const float (&o)[N], int count, bool vec) {
  if (vec && count >= N) {
    uint32_t w[N / 2];
#pragma unroll
    for (int e = 0; e < N; e += 2) {
      const __nv_bfloat162 v = __floats2bfloat162_rn(o[e], o[e + 1]);
      w[e / 2] = *reinterpret_cast<const uint32_t*>(&v);
    }
    if constexpr (N == 8) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint32_t*>(dst) = w[0];
    return;
  }
#pragma unroll
  for (int e = 0; e < N; ++e)
    if (e < count) gi::stf(dst + e, o[e]);
}

// Joins the parts of the units that several blocks hold; maxima are in units of ln, or of powers of two (base2).  A block takes 32
// query rows of a kv head, one to a lane, and 16 of the head's numbers for each of WARPS / PARTS warps; PARTS warps share out a
// row's parts.  A part's maximum, sum and values are asked for together and joined as they come (one trip to memory, not one
// for the maxima and then one for the values); the warps meet in shared memory.
template <typename T, int PARTS>
__global__ void __launch_bounds__(THREADS)
attn_tree_join_kernel(const Shape sh, T* __restrict__ out, long ldo, int hd, int ranges, int base2, int vec, const float4* part_o, const float2* part_ml,
                      const int* part_prefix) {
  constexpr int WARPS = THREADS / 32, CUTS = WARPS / PARTS, FOURS = 4;      // pieces of four numbers that a thread holds
  __shared__ float s_acc[WARPS][FOURS * 4 + 2][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, fours = (hd + 3) / 4;
  gi::pdl_prologue();
  const int b = blockIdx.z, group = sh.n_heads / sh.n_kv;
  const int cuts = (fours + CUTS * FOURS - 1) / (CUTS * FOURS);             // blocks along a head's numbers
  const int kvh = blockIdx.y, row = blockIdx.x / cuts * 32 + lane;
  const int part_group = warp % PARTS, four0 = ((blockIdx.x % cuts) * CUTS + warp / PARTS) * FOURS;
  const int total = part_prefix[sh.n_seqs], before = part_prefix[b], n = nodes_of(sh, b), pos0 = pos0_of(sh, b), tok0 = sh.cu_seqlens[b];
  const int per = per_range(total, ranges);
  const int tiles = tiles_of(sh, pos0, n), row_block = row / sh.rows_block, r = row - row_block * sh.rows_block;
  const int first = before + (row_block / sh.split * sh.n_kv + kvh) * tiles;
  int c0 = 0, c1 = 0;
  if (row < n * group) c0 = first / per, c1 = (first + tiles - 1) / per;
  const bool live = c0 != c1;                              // (one block had it all, or there is no such row)
  if (__all_sync(0xffffffffu, !live)) return;              // (every warp of the block has the same rows)
  float m = -INFINITY, l = 0.f, acc[FOURS][4];
#pragma unroll
  for (int k = 0; k < FOURS; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[k][e] = 0.f;
  auto power = [&](float x) { return base2 ? exp2f(x) : expf(x); };
  if (live && four0 < fours) {
#pragma unroll 2
    for (int c = c0 + part_group; c <= c1; c += PARTS) {
      const size_t s = 2 * ((size_t)c * sh.split + row_block % sh.split) + (c == c0 ? 1 : 0);
      const float2 ml = part_ml[s * sh.rows_block + r];
      float4 o[FOURS];
#pragma unroll
      for (int k = 0; k < FOURS; ++k) o[k] = four0 + k < fours ? part_o[part_at(sh, s, fours, four0 + k, r)] : make_float4(0.f, 0.f, 0.f, 0.f);
      const float m_new = fmaxf(m, ml.x), ref = m_new == -INFINITY ? 0.f : m_new;
      const float was = power(m - ref), is = power(ml.x - ref);
      m = m_new;
      l = l * was + ml.y * is;
#pragma unroll
      for (int k = 0; k < FOURS; ++k) {
        acc[k][0] = acc[k][0] * was + o[k].x * is;
        acc[k][1] = acc[k][1] * was + o[k].y * is;
        acc[k][2] = acc[k][2] * was + o[k].z * is;
        acc[k][3] = acc[k][3] * was + o[k].w * is;
      }
    }
  }
#pragma unroll
  for (int k = 0; k < FOURS; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) s_acc[warp][k * 4 + e][lane] = acc[k][e];
  s_acc[warp][FOURS * 4][lane] = m;
  s_acc[warp][FOURS * 4 + 1][lane] = l;
  __syncthreads();
  // a cut's 16 numbers of 32 rows: PARTS warps' results, added up by those warps, 16 / PARTS numbers each
  const int w0 = warp / PARTS * PARTS;
  float top = -INFINITY, weight[PARTS];
#pragma unroll
  for (int w = 0; w < PARTS; ++w) top = fmaxf(top, s_acc[w0 + w][FOURS * 4][lane]);
  l = 0.f;
#pragma unroll
  for (int w = 0; w < PARTS; ++w) {
    weight[w] = power(s_acc[w0 + w][FOURS * 4][lane] - (top == -INFINITY ? 0.f : top));
    l += weight[w] * s_acc[w0 + w][FOURS * 4 + 1][lane];
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  if (!live) return;
  T* dst = out + (size_t)(tok0 + row / group) * ldo + (size_t)(kvh * group + row % group) * hd;
  constexpr int EACH = FOURS * 4 / PARTS;
  float o[EACH];
#pragma unroll
  for (int e = 0; e < EACH; ++e) {
    o[e] = 0.f;
#pragma unroll
    for (int w = 0; w < PARTS; ++w) o[e] += weight[w] * s_acc[w0 + w][part_group * EACH + e][lane];
  }
#pragma unroll
  for (int e = 0; e < EACH; ++e) o[e] *= inv;
  const int d0 = four0 * 4 + part_group * EACH;
  store_row<EACH>(dst + d0, o, hd - d0, vec != 0);
}

struct Plan {
  int ranges, split, rows_block, tile;
  bool narrow_join;     // the join's blocks: 16 of a head's numbers and 8 warps to the parts, or 64 and 2
};

// Shared memory of a block of the form on CUDA cores: queries, a tile's keys and values, weights.
constexpr size_t smem_of(int rows_block, int hd) { return ((size_t)(rows_block + 2 * TILE) * ((hd + 3) / 4 * 4 + 4) + (size_t)rows_block * 68) * sizeof(float); }

// Blocks of it that an SM holds: two with their registers (__launch_bounds__), one where two blocks' shared memory, the lengths' list
// and 1 KB of the system's among it, is more than 228 KB (64 rows of heads above 116 numbers, 16 rows of heads above 180).  Ranges for
// two where one fits come in two waves, with twice the parts to join: 32 32-bit heads of 128 over 8 behind 1,500 positions, one tree of
// 26 nodes 57 us for 43, 8 trees of 16 nodes 163 for 149, of 64 nodes 533 for 540.
int blocks_of_sm(int rows_block, int hd) {
  return 2 * (smem_of(rows_block, hd) + 4 * (MAX_SEQS + 1) + 1024) <= 228 * 1024 && !(rows_block == 64 && hd > 128) ? 2 : 1;
}

// The query rows of a block: 16 or 64 on CUDA cores, the smaller where it takes a tree's rows; on tensor cores as many whole nodes as
// 128 lanes hold, and up to 8 row blocks of a unit side by side.  Blocks: as many as the device runs at a time, fewer if
// there is not a tile for each.
Plan plan_of(int n_seqs, int max_nodes, int max_kv_len, int n_heads, int n_kv, int hd, bool tensor) {
  Plan p;
  const int group = n_heads / n_kv;
  const long rows = (long)max_nodes * group;
  p.rows_block = tensor ? 128 / group * group : (rows > 16 ? 64 : 16);
  p.tile = tensor ? 128 : TILE;
  const long blocks = (rows + p.rows_block - 1) / p.rows_block, rounds = tensor ? (blocks + 7) / 8 : blocks;
  p.split = (int)((blocks + rounds - 1) / rounds);
  const long units = (long)n_seqs * n_kv * rounds, tiles = (max_kv_len + p.tile - 1) / p.tile;
  const long wanted = units * tiles;
  const long cap = (tensor ? 1L : (long)blocks_of_sm(p.rows_block, hd)) * gi::sm_count() / p.split;
  p.ranges = (int)(wanted < cap ? wanted : cap);
  if (p.ranges < 1) p.ranges = 1;
  // The narrow join has four times the blocks, each done sooner: right as long as the device holds them at a time, about 4 to an SM.  The
  // whole call with the narrow / wide one, by the narrow one's blocks, 8 kv heads of groups of 4: bf16 heads of 128, 26 nodes, 256 blocks
  // 15.8 / 21.4 us, 512 20.4 / 22.6, 768 27.6 / 27.5, 1,024 31.3 / 29.7; 90 nodes, 768 blocks 22.8 / 22.4, 1,536 35.9 / 31.2; heads of 64, 8
  // nodes, 384 blocks 27.6 / 29.2, 512 32.5 / 32.2; 32-bit heads of 64, 12 nodes, 384 blocks 30.5 / 33.2, 448 41.4 / 40.9, 640 54.1 / 54.6.
  p.narrow_join = (rows + 31) / 32 * ((hd + 15) / 16) * n_kv * n_seqs <= 4L * gi::sm_count();
  return p;
}

long scratch_of(const Plan& p, int n_seqs, int hd) { return 4L * ((n_seqs + 4) / 4 * 4) + 2L * p.ranges * p.split * p.rows_block * ((hd + 3) / 4 * 4 + 2) * 4; }

template <typename T, int R, int DCH>
int launch_tree(const Shape& sh, const Plan& p, T* out, long ldo, const T* q, long ldq, const T* k, const T* v, int hd, float scale,
                float4* part_o, float2* part_ml, int* part_prefix, cudaStream_t s) {
  const size_t smem = smem_of(R, hd);
  auto kern = attn_tree_kernel<T, R, DCH>;
  static bool configured[gi::MAX_DEVICES_SEEN] = {false};
  int dev;
  if (gi::unconfigured_here(configured, &dev)) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_of(R, DCH * 64));
    if (e != cudaSuccess) return gi::fail(GI_ERR_CUDA, "tree attention: %s", cudaGetErrorString(e));
    if (dev >= 0) configured[dev] = true;
  }
  const int vec = hd % 4 == 0 && ldq % 4 == 0 && (((uintptr_t)k | (uintptr_t)v | (uintptr_t)q) % (4 * sizeof(T))) == 0;
  return gi::check(gi::launch(kern, dim3(p.ranges), dim3(THREADS), smem, s, sh, out, ldo, q, ldq, k, v, hd, scale, part_o, part_ml, part_prefix, vec), "tree attention");
}

template <typename T, int R>
int launch_tree_dims(const Shape& sh, const Plan& p, T* out, long ldo, const T* q, long ldq, const T* k, const T* v, int hd, float scale,
                     float4* part_o, float2* part_ml, int* part_prefix, cudaStream_t s) {
  if (hd <= 64) return launch_tree<T, R, 1>(sh, p, out, ldo, q, ldq, k, v, hd, scale, part_o, part_ml, part_prefix, s);
  if (hd <= 128) return launch_tree<T, R, 2>(sh, p, out, ldo, q, ldq, k, v, hd, scale, part_o, part_ml, part_prefix, s);
  return launch_tree<T, R, 4>(sh, p, out, ldo, q, ldq, k, v, hd, scale, part_o, part_ml, part_prefix, s);
}

}  // namespace

extern "C" long gi_attn_tree_scratch(int n_seqs, int max_nodes, int max_kv_len, int n_heads, int n_kv, int hd, int dtype) {
  if (n_seqs <= 0 || max_nodes <= 0 || max_kv_len <= 0 || n_kv <= 0 || n_heads < n_kv || hd <= 0) return 0;
  const long plain = scratch_of(plan_of(n_seqs, max_nodes, max_kv_len, n_heads, n_kv, hd, false), n_seqs, hd);
  if (dtype != GI_BF16 || (hd != 64 && hd != 128) || n_heads / n_kv > 128) return plain;
  const long tensor = scratch_of(plan_of(n_seqs, max_nodes, max_kv_len, n_heads, n_kv, hd, true), n_seqs, hd);
  return tensor > plain ? tensor : plain;
}

extern "C" int gi_attn_tree(void* out, long ldo, const void* q, long ldq, long q_rows, int dtype, const void* kcache, const void* vcache, int cache_pages,
                            const int* block_table, int table_rows, int max_pages, const int* cu_seqlens, const int* seq_slots, const int* seq_pos0, const int* masks,
                            int words, int n_seqs, int max_nodes, int max_kv_len, int n_heads, int n_kv, int hd, float scale, void* scratch,
                            long scratch_bytes, void* stream) {
  if (n_seqs <= 0 || q_rows <= 0) return GI_OK;
  if (n_kv < 1 || n_heads < 1 || n_heads % n_kv != 0) return gi::fail(GI_ERR_ARG, "tree attention: %d heads do not divide into %d kv heads", n_heads, n_kv);
  if (hd < 1 || hd > 256) return gi::fail(GI_ERR_UNSUPPORTED, "tree attention: head size %d, 1 to 256 are supported", hd);
  if (max_nodes < 1 || max_nodes > MAX_NODES) return gi::fail(GI_ERR_ARG, "tree attention: trees of up to %d nodes, 1 to %d are supported", max_nodes, MAX_NODES);
  if (words < (max_nodes + 31) / 32) return gi::fail(GI_ERR_ARG, "tree attention: %d words of mask bits cannot hold %d nodes", words, max_nodes);
  if (n_seqs > MAX_SEQS) return gi::fail(GI_ERR_UNSUPPORTED, "tree attention: more than %d sequences in one launch", MAX_SEQS);
  if (cache_pages < 1 || table_rows < 0 || max_pages < 1 || max_kv_len < 1) return gi::fail(GI_ERR_ARG, "tree attention: %d pages, %d in a table's row, %d positions", cache_pages, max_pages, max_kv_len);
  // tensor cores: 16-bit rows and pages that TMA and 16-byte accesses can take, row coordinates of 32 bits; a scale above zero (that form
  // hides scores before it scales them: -inf times nothing is no number, times less than nothing the largest of all)
  const bool tensor = dtype == GI_BF16 && (hd == 64 || hd == 128) && scale >= FLT_MIN && scale <= FLT_MAX && n_heads / n_kv <= 128 && q_rows <= 0x7fffffffL && ldq % 8 == 0 && ldo % 8 == 0 && (((uintptr_t)q | (uintptr_t)kcache | (uintptr_t)vcache | (uintptr_t)out) & 15) == 0 &&
                      (long)cache_pages * n_kv * PAGE_TOKENS <= 0x7fffffffL;
  const Plan p = plan_of(n_seqs, max_nodes, max_kv_len, n_heads, n_kv, hd, tensor);
  if (scratch_bytes < gi_attn_tree_scratch(n_seqs, max_nodes, max_kv_len, n_heads, n_kv, hd, dtype) || ((uintptr_t)scratch & 15))
    return gi::fail(GI_ERR_ARG, "tree attention: the scratch memory is too small or not aligned");
  // the list of tiles is counted in 32 bits
  const long most = (long)n_seqs * n_kv * (((long)max_nodes * (n_heads / n_kv) + p.rows_block - 1) / p.rows_block) * (((long)max_pages * PAGE_TOKENS + max_nodes) / p.tile + 1);
  if (most > 0x3fffffffL || max_pages > 0x7fffffff / PAGE_TOKENS - MAX_NODES) return gi::fail(GI_ERR_UNSUPPORTED, "tree attention: %d sequences of up to %d pages are more than one launch takes", n_seqs, max_pages);
  const Shape sh = {cu_seqlens, seq_slots, seq_pos0, block_table, masks, words, table_rows, max_pages, n_seqs, n_heads, n_kv, max_nodes, cache_pages, q_rows, p.rows_block, p.split, p.tile};
  int* prefix_out = (int*)scratch;
  float4* part_o = (float4*)(prefix_out + (n_seqs + 4) / 4 * 4);
  float2* part_ml = (float2*)(part_o + 2L * p.ranges * p.split * p.rows_block * ((hd + 3) / 4));
  cudaStream_t s = (cudaStream_t)stream;
  int rc = GI_OK;
  if (tensor)
    rc = launch_t5(sh, p.ranges * p.split, out, ldo, q, ldq, q_rows, kcache, vcache, hd, scale, part_o, part_ml, prefix_out, s);
  else if (p.rows_block == 64)
    GI_DISPATCH_DTYPE(dtype, T, rc = (launch_tree_dims<T, 64>(sh, p, (T*)out, ldo, (const T*)q, ldq, (const T*)kcache, (const T*)vcache, hd, scale, part_o, part_ml, prefix_out, s)));
  else
    GI_DISPATCH_DTYPE(dtype, T, rc = (launch_tree_dims<T, 16>(sh, p, (T*)out, ldo, (const T*)q, ldq, (const T*)kcache, (const T*)vcache, hd, scale, part_o, part_ml, prefix_out, s)));
  if (rc != GI_OK) return rc;
  const int rows = max_nodes * (n_heads / n_kv);
  const int vec = hd % 8 == 0 && ldo % 8 == 0 && ((uintptr_t)out & 15) == 0;
  const int numbers = p.narrow_join ? 16 : 64;               // of a head, in a block of the join
  const dim3 join((unsigned)((rows + 31) / 32 * ((hd + numbers - 1) / numbers)), n_kv, n_seqs);
  GI_DISPATCH_DTYPE(dtype, T, rc = gi::check(gi::launch(p.narrow_join ? attn_tree_join_kernel<T, 8> : attn_tree_join_kernel<T, 2>, join, dim3(THREADS), 0, s, sh, (T*)out,
                                                        ldo, hd, p.ranges, tensor ? 1 : 0, vec, part_o, part_ml, prefix_out), "tree attention (join)"));
  return rc;
}

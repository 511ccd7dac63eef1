// Attention over trees of drafted tokens on tcgen05 tensor cores: bfloat16, head size 64 or 128 (the formula: attention_tree.cu).
//
// The query rows of a kv head (its group's heads x a tree's nodes) share every key and value, so a block takes MT tiles of 128
// of them, one query row to a lane of tensor memory, and walks its range of 64-key tiles (attention_tree.cuh).  One warp fetches
// keys and values page by page with TMA into a ring, one thread issues the score products S = Q K^T into one of two score
// buffers per row tile, another one the output products O += P V with P read from tensor memory, and 4 MT warps own one row a
// thread: running maximum and sum in 32 bits (base-2 exponentials), probabilities written as bfloat16 over the scores they
// came from, the accumulator rescaled in tensor memory when a row's reference point moves by more than 2^8.
// Only tiles that reach behind the cached positions look at masks: a row's two words of bits for the tile's 64 keys.  Values of
// those tiles need care: a row that does not see a node has the weight 0 for it, and 0 times a number that is none is none.
// What lies behind the last node is overwritten with zeros in shared memory, and so is a node's value row that holds an infinity or
// no number; the rows that do see such a node get no number for an answer (in all of the head's numbers, not in the spoiled ones alone).
//
// Bound: with up to 128 rows the cache's bytes (32 KB a tile at head size 128 take an SM's share of the memory about 1,400 cycles,
// the products 512, the exponentials 512), two blocks to an SM.  With up to 256 rows products and exponentials double: both row
// tiles then share one block and one ring, so that keys and values still cross to the SM once.  Every wait has an iteration limit.
#include <cuda.h>

#include "api.h"
#include "attention_tree.cuh"
#include "tc_utils.cuh"

namespace {

using namespace gi::tc;
using namespace gi::tree;

constexpr int BQ = 128;
constexpr uint32_t Q_HALF = BQ * 128, KV_HALF = TILE * 128;      // a 64-number half of a tile: rows of 128 bytes, swizzled

__device__ int g_tree_status = 0;

__device__ __forceinline__ void tc_st32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
        "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
        "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 2^x in one instruction (about 2 units in the last place): probabilities are rounded to bfloat16 right after.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// D (+)= A B with A read from tensor memory (two neighbouring bfloat16 of K to a 32-bit column).
__device__ __forceinline__ void tc_mma_a_tmem(uint32_t tmem_d, uint32_t tmem_a, uint64_t desc_b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(desc_b), "r"(idesc), "r"(accumulate) : "memory");
}
// Descriptor of an operand whose N side is contiguous in memory: 64-wide, 128-byte-swizzled blocks, 8 rows of K 1024 bytes apart,
// the next 64-wide block `lbo_bytes` away.
__device__ __forceinline__ uint64_t smem_desc_mn(uint32_t addr, uint32_t lbo_bytes) {
  return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)(lbo_bytes >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
         ((uint64_t)2 << 61);
}

template <int HALVES, int MT, int STAGES>
struct Layout {
  static constexpr uint32_t Q_BYTES = HALVES * Q_HALF, KV_BYTES = HALVES * KV_HALF;
  static constexpr uint32_t K_AT = MT * Q_BYTES, V_AT = K_AT + STAGES * KV_BYTES, BARS_AT = V_AT + STAGES * KV_BYTES;
  static constexpr int N_BARS = 4 * STAGES + 6 * MT + 4;
  static constexpr uint32_t FLAGS_AT = BARS_AT + 8 * N_BARS, PREFIX_AT = FLAGS_AT + 2 * 8 + 8;   // flags, the address of the tensor memory
  static constexpr uint32_t BYTES = PREFIX_AT + 8 * (MAX_SEQS + 1);
  static constexpr int THREADS = 128 * MT + 96, COLS = MT == 1 ? 256 : 512;
};

template <int HALVES, int MT, int STAGES>
__global__ void __launch_bounds__(128 * MT + 96, MT == 1 ? 2 : 1)
attn_tree_t5_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ Shape sh,
                    __nv_bfloat16* __restrict__ out, long ldo, const __nv_bfloat16* q, long ldq, int cache_pages, float scale, int least,
                    float* __restrict__ part_o, float* __restrict__ part_ml, long* __restrict__ part_prefix) {
  using L = Layout<HALVES, MT, STAGES>;
  constexpr int HD = HALVES * 64, KSTEPS = HALVES * 4, ROWS = MT * BQ;
  // float accumulator, bfloat16 operands, M 128; S = Q K^T: N 64, both operands K-major; O = P V: N HD, V contiguous along N (bit 16)
  constexpr uint32_t IDESC_S = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(TILE >> 3) << 17) | ((uint32_t)(BQ >> 4) << 24);
  constexpr uint32_t IDESC_O = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(BQ >> 4) << 24);
  // the tiles need 1024-byte alignment, which the dynamic shared memory of a kernel without static shared memory has (checked)
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned long long* flags = (unsigned long long*)(smem + L::FLAGS_AT);
  uint32_t* tmem_slot = (uint32_t*)(smem + L::FLAGS_AT + 16);
  long* s_pre = (long*)(smem + L::PREFIX_AT);
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) atomicCAS(&g_tree_status, 0, 9);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t bar0 = smem_u32(smem + L::BARS_AT);
  const uint32_t k_full = bar0, k_empty = k_full + 8 * STAGES, v_full = k_empty + 8 * STAGES, v_empty = v_full + 8 * STAGES;
  // per row tile and score buffer: scores ready; probabilities ready (4 warps); both read by the output product
  const uint32_t s_full = v_empty + 8 * STAGES, p_full = s_full + 16 * MT, sp_empty = p_full + 16 * MT;
  const uint32_t q_full = sp_empty + 16 * MT, q_empty = q_full + 8;
  const uint32_t scanned = q_empty + 8, zeroed = scanned + 8;     // the rows' warps meet around the values of a tile with nodes
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(k_full + 8 * i, 1);
      mbar_init(k_empty + 8 * i, 1);
      mbar_init(v_full + 8 * i, 1);
      mbar_init(v_empty + 8 * i, 1);
    }
    for (int i = 0; i < 2 * MT; ++i) {
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_full + 8 * i, 4);
      mbar_init(sp_empty + 8 * i, 1);
    }
    mbar_init(q_full, 4 * MT);
    mbar_init(q_empty, 1);
    mbar_init(scanned, 4 * MT);
    mbar_init(zeroed, 4 * MT);
    flags[0] = flags[1] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 4 * MT) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)L::COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  gi::pdl_prologue();
  if (warp == 0) prefix(sh, s_pre);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmem_o = tmem + 128 * MT;          // score buffers [row tile][2][64 columns], then O [row tile][HD]
  const long total = s_pre[sh.n_seqs], per = per_block(total, gridDim.x, least);
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i <= sh.n_seqs; i += L::THREADS) part_prefix[i] = s_pre[i];
  const long lo = (long)blockIdx.x * per, hi = min(total, lo + per);
  const int group = sh.n_heads / sh.n_kv;
  bool ok = true;
  int j = 0;                                        // tiles so far, over all units of this block's range

  if (warp == 4 * MT) {
    // ---- keys and values: the pages of 32 tiles are looked up side by side
    for (long at = lo; at < hi && ok;) {
      const Unit u = unit_at(sh, s_pre, at);
      const int t_begin = (int)(at - u.first), t_end = (int)min((long)u.tiles, hi - u.first);
      for (int t0 = t_begin; t0 < t_end && ok; t0 += 32) {
        const int mine = t0 + lane < t_end ? page_of(sh, u.slot, t0 + lane, cache_pages) : 0;
        const int here = min(32, t_end - t0);
        for (int i = 0; i < here && ok; ++i, ++j) {
          const int row0 = (__shfl_sync(0xffffffffu, mine, i) * sh.n_kv + u.kvh) * TILE;
          const int s = j % STAGES;
          if (lane == 0) {
            const uint32_t parity = (uint32_t)((j / STAGES - 1) & 1);
            if (j >= STAGES) ok = mbar_wait(k_empty + 8 * s, parity, 1, &g_tree_status);
            if (ok) {
              mbar_expect_tx(k_full + 8 * s, L::KV_BYTES);
#pragma unroll
              for (int hf = 0; hf < HALVES; ++hf)
                tma_load_2d(smem_u32(smem + L::K_AT + s * L::KV_BYTES + hf * KV_HALF), &map_k, hf * 64, row0, k_full + 8 * s);
              if (j >= STAGES) ok = mbar_wait(v_empty + 8 * s, parity, 1, &g_tree_status);
            }
            if (ok) {
              mbar_expect_tx(v_full + 8 * s, L::KV_BYTES);
#pragma unroll
              for (int hf = 0; hf < HALVES; ++hf)
                tma_load_2d(smem_u32(smem + L::V_AT + s * L::KV_BYTES + hf * KV_HALF), &map_v, hf * 64, row0, v_full + 8 * s);
            } else {
              // giving up: the copies under way must have landed before the block's shared memory goes to another one.  The last
              // copy of keys may be tile j's, that of values tile j - 1's
              for (int back = 0; back < STAGES && back <= j; ++back) {
                const int t = j - back;
                mbar_wait(k_full + 8 * (t % STAGES), (uint32_t)((t / STAGES) & 1), 1, &g_tree_status);
                if (t > 0) mbar_wait(v_full + 8 * ((t - 1) % STAGES), (uint32_t)(((t - 1) / STAGES) & 1), 1, &g_tree_status);
              }
            }
          }
          ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        }
      }
      at = u.first + t_end;
    }
  } else if (warp == 4 * MT + 1) {
    // ---- score products
    if (lane == 0) {
      int f = 0;
      for (long at = lo; at < hi && ok; ++f) {
        const Unit u = unit_at(sh, s_pre, at);
        const int t_begin = (int)(at - u.first), t_end = (int)min((long)u.tiles, hi - u.first);
        ok = mbar_wait(q_full, (uint32_t)(f & 1), 2, &g_tree_status);
        for (int t = t_begin; t < t_end && ok; ++t, ++j) {
          const int s = j % STAGES, buf = j & 1;
          ok = mbar_wait(k_full + 8 * s, (uint32_t)((j / STAGES) & 1), 2, &g_tree_status);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            // the buffer is free once the output product of tile j - 2 has read its probabilities
            if (ok && j >= 2) ok = mbar_wait(sp_empty + 16 * m + 8 * buf, (uint32_t)(((j - 2) >> 1) & 1), 2, &g_tree_status);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int ks = 0; ks < KSTEPS; ++ks)
              tc_mma(tmem + m * 128 + buf * 64, smem_desc(smem_u32(smem + m * L::Q_BYTES + (ks / 4) * Q_HALF + (ks % 4) * 32)),
                     smem_desc(smem_u32(smem + L::K_AT + s * L::KV_BYTES + (ks / 4) * KV_HALF + (ks % 4) * 32)), IDESC_S, ks > 0 ? 1u : 0u);
            tc_commit(s_full + 16 * m + 8 * buf);
          }
          if (ok) tc_commit(k_empty + 8 * s);
        }
        if (ok) tc_commit(q_empty);
        at = u.first + t_end;
      }
    }
  } else if (warp == 4 * MT + 2) {
    // ---- output products
    if (lane == 0) {
      for (long at = lo; at < hi && ok;) {
        const Unit u = unit_at(sh, s_pre, at);
        const int t_begin = (int)(at - u.first), t_end = (int)min((long)u.tiles, hi - u.first);
        for (int t = t_begin; t < t_end && ok; ++t, ++j) {
          const int s = j % STAGES, buf = j & 1;
          ok = mbar_wait(v_full + 8 * s, (uint32_t)((j / STAGES) & 1), 4, &g_tree_status);
#pragma unroll
          for (int m = 0; m < MT; ++m) {
            // (a unit's first product overwrites O: the rows' warps announce its probabilities after they have read the last unit's)
            if (ok) ok = mbar_wait(p_full + 16 * m + 8 * buf, (uint32_t)((j >> 1) & 1), 4, &g_tree_status);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int kk = 0; kk < TILE / 16; ++kk)
              tc_mma_a_tmem(tmem_o + m * HD, tmem + m * 128 + buf * 64 + kk * 8, smem_desc_mn(smem_u32(smem + L::V_AT + s * L::KV_BYTES) + kk * 2048, KV_HALF),
                            IDESC_O, (t > t_begin || kk > 0) ? 1u : 0u);
            tc_commit(sp_empty + 16 * m + 8 * buf);
          }
          if (ok) tc_commit(v_empty + 8 * s);
        }
        at = u.first + t_end;
      }
    }
  } else {
    // ---- one query row per thread
    const int m = warp >> 2, tid = threadIdx.x & 127, row = m * BQ + tid;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t my_o = tmem_o + m * HD + lane_base;
    const float sl2 = scale * 1.4426950408889634f;
    int f = 0, in_tree_tiles = 0;
    for (long at = lo; at < hi && ok; ++f) {
      const Unit u = unit_at(sh, s_pre, at);
      const int t_begin = (int)(at - u.first), t_end = (int)min((long)u.tiles, hi - u.first);
      const int tok0 = sh.cu_seqlens[u.b], len = u.pos0 + u.n;
      const int rows_here = min(ROWS, u.n * group - u.row0);
      // the queries: 16-byte pieces, swizzled as TMA would lay them down (piece index XOR row mod 8); rows past the unit's are zeros
      if (f > 0) ok = mbar_wait(q_empty, (uint32_t)((f - 1) & 1), 3, &g_tree_status);
      if (!ok) break;
      unsigned char* q_s = smem + m * L::Q_BYTES;
#pragma unroll 4
      for (int i = tid; i < BQ * HALVES * 8; i += 128) {
        const int r = i / (HALVES * 8), c = i % (HALVES * 8), gr = u.row0 + m * BQ + r;
        uint4 v = make_uint4(0, 0, 0, 0);
        if (m * BQ + r < rows_here) v = *reinterpret_cast<const uint4*>(q + (size_t)(tok0 + gr / group) * ldq + (size_t)(u.kvh * group + gr % group) * HD + c * 8);
        *reinterpret_cast<uint4*>(q_s + (c / 8) * Q_HALF + r * 128 + ((c % 8) ^ (r & 7)) * 16) = v;
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(q_full);

      const bool warp_live = m * BQ + (warp & 3) * 32 < rows_here;
      const int* mask = sh.masks + (size_t)(tok0 + min(u.row0 + row, u.n * group - 1) / group) * sh.words;
      float m_run = -INFINITY, l_run = 0.f;
      for (int t = t_begin; t < t_end && ok; ++t, ++j) {
        const int buf = j & 1, s = j % STAGES, kt = t * TILE;
        const uint32_t my_s = tmem + m * 128 + buf * 64 + lane_base;
        ok = mbar_wait(s_full + 16 * m + 8 * buf, (uint32_t)((j >> 1) & 1), 3, &g_tree_status);
        if (!ok) break;
        tc_fence_after();
        const bool in_tree = kt + TILE > u.pos0;
        unsigned seen[2] = {0xffffffffu, 0xffffffffu};
        if (in_tree) {
          seen[0] = seen_word(mask, sh.words, u.n, kt - u.pos0);
          seen[1] = seen_word(mask, sh.words, u.n, kt + 32 - u.pos0);
        }
        if (warp_live) {                                // (warps without a row of the unit only keep step)
          uint32_t sr[2][32];
          tc_ld32(my_s, sr[0]);
          tc_ld32(my_s + 32, sr[1]);
          tc_wait_ld();
          float top = -INFINITY;
          if (in_tree) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int c = 0; c < 32; ++c) {
                if (!((seen[h] >> c) & 1u)) sr[h][c] = __float_as_uint(-INFINITY);
              }
          }
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int c = 0; c < 32; ++c) top = fmaxf(top, __uint_as_float(sr[h][c]));
          top *= sl2;
          // the reference point moves only when the maximum has grown by more than 2^8 (see attention_prefill_t5.cu)
          float alpha = 1.0f;
          if (m_run == -INFINITY || top > m_run + 8.0f) {
            const float m_new = fmaxf(m_run, top);
            alpha = m_run == -INFINITY ? 0.f : ex2(m_run - m_new);
            m_run = m_new;
          }
          const float neg_m = m_run == -INFINITY ? 0.f : -m_run;
          float psum = 0.f;
          uint32_t pk[32];
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              const float p0 = ex2(fmaf(__uint_as_float(sr[h][c]), sl2, neg_m)), p1 = ex2(fmaf(__uint_as_float(sr[h][c + 1]), sl2, neg_m));
              psum += p0 + p1;
              __nv_bfloat162 pv = __floats2bfloat162_rn(p0, p1);
              pk[h * 16 + c / 2] = *reinterpret_cast<uint32_t*>(&pv);
            }
          l_run = l_run * alpha + psum;
          if (t > t_begin && __any_sync(0xffffffffu, alpha != 1.0f)) {
            // O is rescaled: the product before must be done.  Its buffer's barrier is at most this one phase behind, since the
            // scores just read were not issued before the product of tile j - 2 was done.
            ok = mbar_wait(sp_empty + 16 * m + 8 * (buf ^ 1), (uint32_t)(((j - 1) >> 1) & 1), 3, &g_tree_status);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HD / 32; ++c) {
              uint32_t o[32];
              tc_ld32(my_o + c * 32, o);
              tc_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
              tc_st32(my_o + c * 32, o);
            }
          }
          tc_st32(my_s, pk);
          tc_wait_st();
        }
        if (in_tree) {
          // values that nobody may meet: see the head of this file.  All rows' warps share the work and meet before and after.
          unsigned long long* flag = flags + (in_tree_tiles & 1);
          ok = mbar_wait(v_full + 8 * s, (uint32_t)((j / STAGES) & 1), 3, &g_tree_status);
          unsigned char* v_s = smem + L::V_AT + s * L::KV_BYTES;
          const int first = max(0, u.pos0 - kt), end = min(TILE, len - kt);
          if (ok)
            for (int i = threadIdx.x; i < (end - first) * HALVES * 8; i += 128 * MT) {
              const int r = first + i / (HALVES * 8), c = i % (HALVES * 8);
              const uint4 v = *reinterpret_cast<const uint4*>(v_s + (c / 8) * KV_HALF + r * 128 + (c % 8) * 16);
              const uint32_t w[4] = {v.x, v.y, v.z, v.w};
              bool bad = false;
#pragma unroll
              for (int e = 0; e < 4; ++e) bad |= (w[e] & 0x7f80u) == 0x7f80u || (w[e] & 0x7f800000u) == 0x7f800000u;
              if (bad) atomicOr(flag, 1ull << r);
            }
          __syncwarp();
          if (lane == 0 && ok) mbar_arrive(scanned);
          if (ok) ok = mbar_wait(scanned, (uint32_t)(in_tree_tiles & 1), 3, &g_tree_status);
          if (!ok) break;
          const unsigned long long spoiled = *(volatile unsigned long long*)flag;
          if (threadIdx.x == 0) flags[(in_tree_tiles + 1) & 1] = 0;
          if (spoiled != 0 || end < TILE)
            for (int i = threadIdx.x; i < (TILE - first) * HALVES * 8; i += 128 * MT) {
              const int r = first + i / (HALVES * 8), c = i % (HALVES * 8);
              if (r >= end || ((spoiled >> r) & 1)) *reinterpret_cast<uint4*>(v_s + (c / 8) * KV_HALF + r * 128 + (c % 8) * 16) = make_uint4(0, 0, 0, 0);
            }
          if (spoiled & (((unsigned long long)seen[1] << 32) | seen[0])) l_run = __int_as_float(0x7fc00000);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(zeroed);
          ok = mbar_wait(zeroed, (uint32_t)(in_tree_tiles & 1), 3, &g_tree_status);
          if (!ok) break;
          ++in_tree_tiles;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0 && ok) mbar_arrive(p_full + 16 * m + 8 * buf);
      }
      if (ok) ok = mbar_wait(sp_empty + 16 * m + 8 * ((j - 1) & 1), (uint32_t)(((j - 1) >> 1) & 1), 3, &g_tree_status);
      if (!ok) break;
      tc_fence_after();
      if (warp_live) {
        const bool live = row < rows_here, whole = t_begin == 0 && t_end == u.tiles;
        const int gr = u.row0 + row;
        const float inv = l_run == 0.f ? 0.f : 1.0f / l_run;
        __nv_bfloat16* dst = out + (size_t)(tok0 + gr / group) * ldo + (size_t)(u.kvh * group + gr % group) * HD;
        const size_t pr = (2 * (size_t)blockIdx.x + (t_begin == 0 ? 1 : 0)) * ROWS + row;
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t o[32];
          tc_ld32(my_o + c * 32, o);
          tc_wait_ld();
          if (live && whole) {
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              uint32_t w[4];
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                __nv_bfloat162 v2 = __floats2bfloat162_rn(__uint_as_float(o[e + 2 * x]) * inv, __uint_as_float(o[e + 2 * x + 1]) * inv);
                w[x] = *reinterpret_cast<uint32_t*>(&v2);
              }
              *reinterpret_cast<uint4*>(dst + c * 32 + e) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          } else if (live) {
#pragma unroll
            for (int e = 0; e < 32; e += 4) *reinterpret_cast<uint4*>(part_o + pr * HD + c * 32 + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
          __syncwarp();
        }
        if (live && !whole) {
          part_ml[pr * 2] = m_run;
          part_ml[pr * 2 + 1] = l_run;
        }
      }
      tc_fence_before();
      at = u.first + t_end;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4 * MT) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)L::COLS) : "memory");
  }
}

template <int HALVES, int MT, int STAGES>
int launch_kernel(const CUtensorMap& mk, const CUtensorMap& mv, const Shape& sh, int blocks, __nv_bfloat16* out, long ldo, const __nv_bfloat16* q, long ldq,
           int cache_pages, float scale, int least, float* part_o, float* part_ml, long* part_prefix, cudaStream_t s) {
  using L = Layout<HALVES, MT, STAGES>;
  auto kern = attn_tree_t5_kernel<HALVES, MT, STAGES>;
  static bool configured[gi::MAX_DEVICES_SEEN] = {false};
  int dev;
  if (gi::unconfigured_here(configured, &dev)) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::BYTES);
    if (e != cudaSuccess) return gi::fail(GI_ERR_CUDA, "tree attention (tcgen05): %s", cudaGetErrorString(e));
    if (dev >= 0) configured[dev] = true;
  }
  return gi::check(gi::launch(kern, dim3(blocks), dim3(L::THREADS), L::BYTES, s, mk, mv, sh, out, ldo, q, ldq, cache_pages, scale, least, part_o, part_ml,
                              part_prefix), "tree attention (tcgen05)");
}

}  // namespace

int gi::tree::launch_t5(const Shape& sh, int blocks, void* out, long ldo, const void* q, long ldq, const void* k, const void* v, int cache_pages, int hd,
                        float scale, int least, float* part_o, float* part_ml, long* part_prefix, cudaStream_t s) {
  CUtensorMap mk, mv;
  const long rows = (long)cache_pages * sh.n_kv * TILE;
  int rc = gi::tensor_map_2d_ex(&mk, k, rows, hd, hd, GI_BF16, 64, TILE);
  if (rc == GI_OK) rc = gi::tensor_map_2d_ex(&mv, v, rows, hd, hd, GI_BF16, 64, TILE);
  if (rc != GI_OK) return rc;
#define GI_T5(H, M, S) launch_kernel<H, M, S>(mk, mv, sh, blocks, (__nv_bfloat16*)out, ldo, (const __nv_bfloat16*)q, ldq, cache_pages, scale, least, part_o, part_ml, part_prefix, s)
  if (hd == 128) return sh.rows_block > BQ ? GI_T5(2, 2, 4) : GI_T5(2, 1, 2);
  return sh.rows_block > BQ ? GI_T5(1, 2, 4) : GI_T5(1, 1, 4);
#undef GI_T5
}

extern "C" int gi_attn_tree_status(int* status) {
  int zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(status, g_tree_status, sizeof(int));
  if (e == cudaSuccess) e = cudaMemcpyToSymbol(g_tree_status, &zero, sizeof(int));
  if (e != cudaSuccess) return gi::fail(GI_ERR_CUDA, "tree attention status: %s", cudaGetErrorString(e));
  return GI_OK;
}

// Attention over trees of drafted tokens on tcgen05 tensor cores: bfloat16, head size 64 or 128 (the formula: attention_tree.cu).
//
// The query rows of a kv head (its group's heads x a tree's nodes) share every key and value: a block takes up to 128 of them (whole
// nodes, one query row to a lane of tensor memory) and walks its range of 128-key tiles (attention_tree.cuh).  One warp fetches
// queries and, page by page, keys with TMA, another one values; one thread issues the score products S = Q K^T into one of two score
// buffers, a second one the output products O += P V with P read from tensor memory.  Eight warps make the probabilities: a row
// is two threads' work, one for the first 64 keys of every tile and one for the second.  The two know nothing of each other
// until the end: each has a running maximum and sum (32 bits, base-2 exponentials) and an accumulator of its own in tensor
// memory, rescaled when its reference point moves by more than 2^8, and writes its probabilities as bfloat16 over the scores
// it has read.  One thread a row leaves the exponential unit idle half the time (a warp alone takes 373 cycles for 32 numbers, two
// on a scheduler 293 each).
// Trees of more rows take several blocks that walk the same keys side by side (two row tiles in one block, with one score buffer
// each, waited on one another's products: 5,500 cycles a tile).  128 keys a tile: with 64, a score product reads 6 KB of shared
// memory per 32 cycles of arithmetic, more than there is (75 cycles an instruction measured), and twice as many waits go by.
// Only tiles that reach behind the cached positions look at masks: a row's words of bits for the tile's keys.  Values of those
// tiles need care: a row that does not see a node has the weight 0 for it, and 0 times a number that is none is none.  What
// lies behind the last node is overwritten with zeros in shared memory, and so is a node's value row that holds an infinity or no
// number; the rows that do see such a node get no number for an answer (in all of the head's numbers, not in the spoiled ones alone).
//
// Bound: the cache's bytes with up to 128 rows (64 KB a tile at head size 128 take an SM's share of the memory about 2,850 cycles;
// products take 1,200, the row threads 2,400), the row threads with more.  B200, 32 heads of 128 over 8, 8 sequences behind 8,192
// positions: 1 node 56 us, 32 nodes 60 us (4.5 TB/s), 64 nodes 88 us (0.78 PFLOP/s) for the first few hundred launches at 1,965 MHz; without
// a pause the power limit brings the clock down to 1,580 MHz and 64 nodes to 106 us (0.65 PFLOP/s).  Every wait has an iteration limit.
#include <cuda.h>

#include "api.h"
#include "attention_tree.cuh"
#include "tc_utils.cuh"

namespace {

using namespace gi::tc;
using namespace gi::tree;

constexpr int BQ = 128, BK = 128;                    // lanes of a row tile, keys of a tile (two pages)
constexpr uint32_t HALF = 128 * 128;                 // a 64-number half of a tile: 128 rows of 128 bytes, swizzled

__device__ int g_tree_status = 0;

__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
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
// Two multiply-adds, two additions in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
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

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}

template <int HALVES, int STAGES>
struct Layout {
  static constexpr uint32_t BYTES_TILE = HALVES * HALF;          // queries, or a tile's keys or values
  static constexpr uint32_t K_AT = BYTES_TILE, V_AT = K_AT + STAGES * BYTES_TILE, BARS_AT = V_AT + STAGES * BYTES_TILE;
  static constexpr int N_BARS = 4 * STAGES + 4 * 2 + 5;
  static constexpr uint32_t FLAGS_AT = (BARS_AT + 8 * N_BARS + 15) / 16 * 16;         // 4 words of flags, the tensor memory's address
  static constexpr uint32_t STATS_AT = FLAGS_AT + 4 * 8 + 16;                          // [this unit's, the last one's][2][128] maximum and sum
  static constexpr uint32_t PREFIX_AT = STATS_AT + 4 * BQ * 8;
  static constexpr uint32_t BYTES = PREFIX_AT + 4 * (MAX_SEQS + 1);
  static constexpr int ROW_THREADS = 256, THREADS = ROW_THREADS + 128, COLS = 512;
};

template <int HALVES, int STAGES>
__global__ void __launch_bounds__(384, 1)
attn_tree_t5_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                    const __grid_constant__ Shape sh, __nv_bfloat16* __restrict__ out, long ldo, float scale, int q_box, float4* __restrict__ part_o,
                    float2* __restrict__ part_ml, int* __restrict__ part_prefix) {
  using L = Layout<HALVES, STAGES>;
  constexpr int HD = HALVES * 64, KSTEPS = HALVES * 4;
  // float accumulator, bfloat16 operands, M 128; S = Q K^T: N 128, both operands K-major; O = P V: N HD, V contiguous along N (bit 16)
  constexpr uint32_t IDESC_S = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BK >> 3) << 17) | ((uint32_t)(BQ >> 4) << 24);
  constexpr uint32_t IDESC_O = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(BQ >> 4) << 24);
  // the tiles need 1024-byte alignment, which the dynamic shared memory of a kernel without static shared memory has (checked)
  extern __shared__ __align__(1024) unsigned char smem[];
  unsigned long long* flags = (unsigned long long*)(smem + L::FLAGS_AT);
  uint32_t* tmem_slot = (uint32_t*)(smem + L::FLAGS_AT + 32);
  float2* s_stats = (float2*)(smem + L::STATS_AT);
  int* s_pre = (int*)(smem + L::PREFIX_AT);
  if (smem_u32(smem) & 1023u) {
    if (threadIdx.x == 0) atomicCAS(&g_tree_status, 0, 9);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t k_full = smem_u32(smem + L::BARS_AT), k_empty = k_full + 8 * STAGES, v_full = k_empty + 8 * STAGES, v_empty = v_full + 8 * STAGES;
  // per score buffer: scores ready; probabilities of the first and of the second 64 keys ready (4 warps); both read by the output product
  const uint32_t s_full = v_empty + 8 * STAGES, p_full = s_full + 16, sp_empty = p_full + 32;
  const uint32_t q_full = sp_empty + 16, q_empty = q_full + 8;
  const uint32_t scanned = q_empty + 8, zeroed = scanned + 8;     // the rows' warps meet around the values of a tile with nodes
  const uint32_t met = zeroed + 8;                                // and over a unit's maxima and sums
  if (threadIdx.x == 0) {
    for (int i = 0; i < 4 * STAGES; ++i) mbar_init(k_full + 8 * i, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + 8 * i, 1);
      mbar_init(p_full + 16 * i, 4);
      mbar_init(p_full + 16 * i + 8, 4);
      mbar_init(sp_empty + 8 * i, 1);
    }
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    mbar_init(scanned, 8);
    mbar_init(zeroed, 8);
    mbar_init(met, 8);
    for (int i = 0; i < 4; ++i) flags[i] = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)L::COLS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  gi::pdl_prologue();
  if (warp == 0) prefix(sh, s_pre);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, tmem_o = tmem + 256;       // [score buffer][128 columns], then O [half of the keys][HD]
  const int ranges = gridDim.x / sh.split, range = blockIdx.x / sh.split, row_block = blockIdx.x % sh.split;
  const int total = s_pre[sh.n_seqs], per = per_range(total, ranges);
  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i <= sh.n_seqs; i += L::THREADS) part_prefix[i] = s_pre[i];
  const int lo = (int)min((long)total, (long)range * per), hi = min(total, lo + per);
  const int group = sh.n_heads / sh.n_kv;
  bool ok = true;
  int j = 0, f = 0;                                 // tiles and units so far
  // the block's next unit with rows for it, from place `at` of the list on; false at the range's end
  auto next_unit = [&](int& at, Unit& u, int& t_begin, int& t_end) {
    while (at < hi) {
      u = unit_at(sh, s_pre, at);
      u.row0 += row_block * sh.rows_block;
      t_begin = at - u.first, t_end = min(u.tiles, hi - u.first);
      at = u.first + t_end;
      if (u.row0 < u.n * group) return true;
    }
    return false;
  };
  int at = lo, t_begin, t_end;
  Unit u;

  if (warp == 8 || warp == 11) {
    // ---- warp 8: queries and keys, warp 11: values (one warp for both would ask for keys only when the values' stage before them is
    // free, a whole tile late).  The pages of 16 tiles are looked up side by side.
    const bool keys = warp == 8;
    const CUtensorMap* map = keys ? &map_k : &map_v;
    const uint32_t full = keys ? k_full : v_full, empty = keys ? k_empty : v_empty, stages = smem_u32(smem + (keys ? L::K_AT : L::V_AT));
    int asked = 0, copied = 0;                      // units' queries, tiles
    for (; ok && next_unit(at, u, t_begin, t_end); ++f) {
      const int pages = (u.pos0 + u.n + PAGE_TOKENS - 1) / PAGE_TOKENS;
      if (keys && lane == 0) {
        if (f > 0) ok = mbar_wait(q_empty, (uint32_t)((f - 1) & 1), 1, &g_tree_status);
        if (ok) {
          ++asked;
          // rows of a box: a node's heads one below the other (a row past the sequence's nodes belongs to nobody and is not looked at)
          const int node = sh.cu_seqlens[u.b] + u.row0 / group;
          mbar_expect_tx(q_full, HALVES * q_box * 128);
#pragma unroll
          for (int hf = 0; hf < HALVES; ++hf) tma_load_3d(smem_u32(smem + hf * HALF), &map_q, hf * 64, u.kvh * group, node, q_full);
        }
      }
      ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
      for (int t0 = t_begin; t0 < t_end && ok; t0 += 16) {
        const int index = 2 * t0 + lane;
        // (the page that fills up a sequence's last tile is any one: nobody looks at it)
        const int mine = (((index < pages ? page_of(sh, u.slot, index) : 0) * sh.n_kv) + u.kvh) * PAGE_TOKENS;
        const int here = min(16, t_end - t0);
        for (int i = 0; i < here && ok; ++i, ++j) {
          const int row[2] = {__shfl_sync(0xffffffffu, mine, 2 * i), __shfl_sync(0xffffffffu, mine, 2 * i + 1)};
          const int s = j % STAGES;
          if (lane == 0) {
            if (j >= STAGES) ok = mbar_wait(empty + 8 * s, (uint32_t)((j / STAGES - 1) & 1), 1, &g_tree_status);
            if (ok) {
              ++copied;
              mbar_expect_tx(full + 8 * s, L::BYTES_TILE);
#pragma unroll
              for (int x = 0; x < 2 * HALVES; ++x)
                tma_load_2d(stages + s * L::BYTES_TILE + (x >> 1) * HALF + (x & 1) * (HALF / 2), map, (x >> 1) * 64, row[x & 1], full + 8 * s);
            }
          }
          ok = __shfl_sync(0xffffffffu, ok ? 1 : 0, 0) != 0;
        }
      }
    }
    // whoever gave up in this block: copies under way land before its shared memory goes to another one
    if (lane == 0) {
      if (asked > 0) mbar_wait(q_full, (uint32_t)((asked - 1) & 1), 1, &g_tree_status);
      for (int t = max(0, copied - STAGES); t < copied; ++t) mbar_wait(full + 8 * (t % STAGES), (uint32_t)((t / STAGES) & 1), 1, &g_tree_status);
    }
  } else if (warp == 9) {
    // ---- score products
    if (lane == 0) {
      // (addresses stand in the descriptors' lowest bits, in units of 16 bytes: offsets are added to them)
      const uint64_t desc_q = smem_desc(smem_u32(smem)), desc_k0 = smem_desc(smem_u32(smem + L::K_AT));
      for (; ok && next_unit(at, u, t_begin, t_end); ++f) {
        ok = mbar_wait(q_full, (uint32_t)(f & 1), 2, &g_tree_status);
        for (int t = t_begin; t < t_end && ok; ++t, ++j) {
          const int s = j % STAGES, buf = j & 1;
          const uint64_t desc_k = desc_k0 + s * (L::BYTES_TILE >> 4);
          ok = mbar_wait(k_full + 8 * s, (uint32_t)((j / STAGES) & 1), 2, &g_tree_status);
          // the buffer is free once the output product of tile j - 2 has read its probabilities
          if (ok && j >= 2) ok = mbar_wait(sp_empty + 8 * buf, (uint32_t)((j / 2 - 1) & 1), 2, &g_tree_status);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int ks = 0; ks < KSTEPS; ++ks)
            tc_mma(tmem + buf * 128, desc_q + (((ks / 4) * HALF + (ks % 4) * 32) >> 4), desc_k + (((ks / 4) * HALF + (ks % 4) * 32) >> 4), IDESC_S, ks > 0 ? 1u : 0u);
          tc_commit(s_full + 8 * buf);
          tc_commit(k_empty + 8 * s);
        }
        if (ok) tc_commit(q_empty);
      }
    }
  } else if (warp == 10) {
    // ---- output products
    if (lane == 0) {
      const uint64_t desc_v0 = smem_desc_mn(smem_u32(smem + L::V_AT), HALF);
      while (ok && next_unit(at, u, t_begin, t_end)) {
        for (int t = t_begin; t < t_end && ok; ++t, ++j) {
          const int s = j % STAGES, buf = j & 1;
          const uint64_t desc_v = desc_v0 + s * (L::BYTES_TILE >> 4);
          ok = mbar_wait(v_full + 8 * s, (uint32_t)((j / STAGES) & 1), 4, &g_tree_status);
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            // A unit's first products overwrite O: the rows' warps announce probabilities after they have read the last unit's, and
            // each of them reads both halves' accumulators.
            if (ok && t == t_begin && half == 0) ok = mbar_wait(p_full + 16 * buf + 8, (uint32_t)((j / 2) & 1), 4, &g_tree_status);
            if (ok) ok = mbar_wait(p_full + 16 * buf + 8 * half, (uint32_t)((j / 2) & 1), 4, &g_tree_status);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int x = 0; x < 4; ++x)              // 16 keys: 8 columns of probabilities, 16 rows of values
              tc_mma_a_tmem(tmem_o + half * HD, tmem + buf * 128 + half * 64 + x * 8, desc_v + ((half * 4 + x) * 2048 >> 4), IDESC_O, (t > t_begin || x > 0) ? 1u : 0u);
          }
          if (!ok) break;
          tc_commit(sp_empty + 8 * buf);
          tc_commit(v_empty + 8 * s);
        }
      }
    }
  } else {
    // ---- one query row and one half of every tile's keys per thread
    const int half = warp >> 2, row = threadIdx.x & 127;
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16, my_o = tmem_o + half * HD + lane_base;
    const float sl2 = scale * 1.4426950408889634f;
    int in_tree_tiles = 0;
    for (; ok && next_unit(at, u, t_begin, t_end); ++f) {
      const int tok0 = sh.cu_seqlens[u.b], len = u.pos0 + u.n;
      const int gr = u.row0 + row, rows_all = u.n * group;                  // the row of the sequence, and how many there are
      const bool live = row < sh.rows_block && gr < rows_all;
      const bool warp_live = (warp & 3) * 32 < sh.rows_block && gr - lane < rows_all;
      const int* mask = sh.masks + (size_t)(tok0 + min(gr, rows_all - 1) / group) * sh.words;
      float m_run = -INFINITY, l_run = 0.f;
      for (int t = t_begin; t < t_end && ok; ++t, ++j) {
        const int buf = j & 1, s = j % STAGES, kt = t * BK;
        const uint32_t my_s = tmem + buf * 128 + half * 64 + lane_base;
        const bool in_tree = kt + BK > u.pos0;
        unsigned seen[2] = {0xffffffffu, 0xffffffffu};
        if (in_tree) {
          seen[0] = seen_word(mask, sh.words, u.n, kt + 64 * half - u.pos0);
          seen[1] = seen_word(mask, sh.words, u.n, kt + 64 * half + 32 - u.pos0);
        }
        ok = mbar_wait(s_full + 8 * buf, (uint32_t)((j / 2) & 1), 3, &g_tree_status);
        if (!ok) break;
        tc_fence_after();
        if (warp_live) {                                // (warps without a row of the unit only keep step)
          uint32_t sr[2][32];
          tc_ld32(my_s, sr[0]);
          tc_ld32(my_s + 32, sr[1]);
          tc_wait_ld();
          float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            if (in_tree) {
#pragma unroll
              for (int c = 0; c < 32; ++c)
                if (!((seen[q] >> c) & 1u)) sr[q][c] = __float_as_uint(-INFINITY);
            }
#pragma unroll
            for (int c = 0; c < 32; ++c) tops[c & 3] = fmaxf(tops[c & 3], __uint_as_float(sr[q][c]));
          }
          const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * sl2;
          // the reference point moves only when the maximum has grown by more than 2^8 (see attention_prefill_t5.cu)
          float alpha = 1.0f;
          if (m_run == -INFINITY || top > m_run + 8.0f) {
            const float m_new = fmaxf(m_run, top);
            alpha = m_run == -INFINITY ? 0.f : ex2(m_run - m_new);
            m_run = m_new;
          }
          if (t > t_begin && __any_sync(0xffffffffu, alpha != 1.0f)) {
            // O is rescaled: the product before must be done.  Its buffer's barrier is at most this one phase behind: the scores just
            // read were not issued before the product of tile j - 2 was done.
            ok = mbar_wait(sp_empty + 8 * (buf ^ 1), (uint32_t)(((j - 1) / 2) & 1), 3, &g_tree_status);
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
          const float neg_m = m_run == -INFINITY ? 0.f : -m_run;
          const float2 scale2 = make_float2(sl2, sl2), shift2 = make_float2(neg_m, neg_m);
          float2 sum_a = make_float2(0.f, 0.f), sum_b = make_float2(0.f, 0.f);
          // each step for 32 numbers before the next one: the exponential unit then works without a pause (number by number a warp
          // alone takes 576 cycles, not 373)
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            uint32_t (&x)[32] = sr[q];
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              const float2 y = fma2(make_float2(__uint_as_float(x[c]), __uint_as_float(x[c + 1])), scale2, shift2);
              x[c] = __float_as_uint(y.x), x[c + 1] = __float_as_uint(y.y);
            }
#pragma unroll
            for (int c = 0; c < 32; ++c) x[c] = __float_as_uint(ex2(__uint_as_float(x[c])));
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              sum_a = add2(sum_a, make_float2(__uint_as_float(x[c]), __uint_as_float(x[c + 1])));
              sum_b = add2(sum_b, make_float2(__uint_as_float(x[c + 2]), __uint_as_float(x[c + 3])));
            }
            uint32_t pk[16];
#pragma unroll
            for (int c = 0; c < 32; c += 2) {
              const __nv_bfloat162 pv = __floats2bfloat162_rn(__uint_as_float(x[c]), __uint_as_float(x[c + 1]));
              pk[c / 2] = *reinterpret_cast<const uint32_t*>(&pv);
            }
            tc_st16(my_s + q * 16, pk);
          }
          l_run = l_run * alpha + ((sum_a.x + sum_a.y) + (sum_b.x + sum_b.y));
          tc_wait_st();
        }
        if (in_tree) {
          // values that nobody may meet: see the head of this file.  All rows' warps share the work and meet before and after.
          unsigned long long* flag = flags + 2 * (in_tree_tiles & 1);
          ok = mbar_wait(v_full + 8 * s, (uint32_t)((j / STAGES) & 1), 3, &g_tree_status);
          unsigned char* v_s = smem + L::V_AT + s * L::BYTES_TILE;
          const int first = max(0, u.pos0 - kt), end = min(BK, len - kt);
          if (ok)
            for (int i = threadIdx.x; i < (end - first) * HALVES * 8; i += L::ROW_THREADS) {
              const int r = first + i / (HALVES * 8), c = i % (HALVES * 8);
              const uint4 v = *reinterpret_cast<const uint4*>(v_s + (c / 8) * HALF + r * 128 + (c % 8) * 16);
              const uint32_t w[4] = {v.x, v.y, v.z, v.w};
              bool bad = false;
#pragma unroll
              for (int e = 0; e < 4; ++e) bad |= (w[e] & 0x7f80u) == 0x7f80u || (w[e] & 0x7f800000u) == 0x7f800000u;
              if (bad) atomicOr(flag + (r >> 6), 1ull << (r & 63));
            }
          __syncwarp();
          if (lane == 0 && ok) mbar_arrive(scanned);
          if (ok) ok = mbar_wait(scanned, (uint32_t)(in_tree_tiles & 1), 3, &g_tree_status);
          if (!ok) break;
          const unsigned long long spoiled0 = ((volatile unsigned long long*)flag)[0], spoiled1 = ((volatile unsigned long long*)flag)[1];
          if (threadIdx.x < 2) flags[2 * ((in_tree_tiles + 1) & 1) + threadIdx.x] = 0;
          if ((spoiled0 | spoiled1) != 0 || end < BK)
            for (int i = threadIdx.x; i < (BK - first) * HALVES * 8; i += L::ROW_THREADS) {
              const int r = first + i / (HALVES * 8), c = i % (HALVES * 8);
              if (r >= end || (((r < 64 ? spoiled0 : spoiled1) >> (r & 63)) & 1)) *reinterpret_cast<uint4*>(v_s + (c / 8) * HALF + r * 128 + (c % 8) * 16) = make_uint4(0, 0, 0, 0);
            }
          if ((half ? spoiled1 : spoiled0) & (((unsigned long long)seen[1] << 32) | seen[0])) l_run = __int_as_float(0x7fc00000);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) mbar_arrive(zeroed);
          ok = mbar_wait(zeroed, (uint32_t)(in_tree_tiles & 1), 3, &g_tree_status);
          if (!ok) break;
          ++in_tree_tiles;
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + 16 * buf + 8 * half);
      }
      // the two halves of a row meet: maxima and sums through shared memory, accumulators in tensor memory
      if (ok) {
        s_stats[(2 * (f & 1) + half) * BQ + row] = make_float2(m_run, l_run);
        __syncwarp();
        if (lane == 0) mbar_arrive(met);
        ok = mbar_wait(met, (uint32_t)(f & 1), 3, &g_tree_status);
      }
      if (ok) ok = mbar_wait(sp_empty + 8 * ((j - 1) & 1), (uint32_t)(((j - 1) / 2) & 1), 3, &g_tree_status);
      if (!ok) break;
      tc_fence_after();
      if (warp_live) {
        const float2 other = s_stats[(2 * (f & 1) + (half ^ 1)) * BQ + row];
        const float m = fmaxf(m_run, other.x), ref = m == -INFINITY ? 0.f : m;
        const float w_own = ex2(m_run - ref), w_other = ex2(other.x - ref), l = l_run * w_own + other.y * w_other;
        const bool whole = t_begin == 0 && t_end == u.tiles;
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        const float w0 = (half ? w_other : w_own) * (whole ? inv : 1.0f), w1 = (half ? w_own : w_other) * (whole ? inv : 1.0f);
        __nv_bfloat16* dst = out + (size_t)(tok0 + gr / group) * ldo + (size_t)(u.kvh * group + gr % group) * HD;
        const size_t slot = 2 * (size_t)blockIdx.x + (t_begin == 0 ? 1 : 0);
        // this warp's half of the head's numbers
#pragma unroll 1
        for (int c = half * (HD / 64); c < (half + 1) * (HD / 64); ++c) {
          uint32_t a[32], b[32];
          tc_ld32(tmem_o + lane_base + c * 32, a);
          tc_ld32(tmem_o + HD + lane_base + c * 32, b);
          tc_wait_ld();
          float o[32];
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __uint_as_float(a[e]) * w0 + __uint_as_float(b[e]) * w1;
          if (live && whole) {
#pragma unroll
            for (int e = 0; e < 32; e += 8) {
              uint32_t w[4];
#pragma unroll
              for (int x = 0; x < 4; ++x) {
                const __nv_bfloat162 v2 = __floats2bfloat162_rn(o[e + 2 * x], o[e + 2 * x + 1]);
                w[x] = *reinterpret_cast<const uint32_t*>(&v2);
              }
              *reinterpret_cast<uint4*>(dst + c * 32 + e) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          } else if (live) {
#pragma unroll
            for (int e = 0; e < 32; e += 4) part_o[part_at(sh, slot, HD / 4, c * 8 + e / 4, row)] = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
          }
          __syncwarp();
        }
        if (live && !whole && half == 0) part_ml[slot * sh.rows_block + row] = make_float2(m, l);
      }
      tc_fence_before();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"((uint32_t)L::COLS) : "memory");
  }
}

template <int HALVES, int STAGES>
int launch_kernel(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const Shape& sh, int blocks, __nv_bfloat16* out, long ldo,
                  float scale, int q_box, float4* part_o, float2* part_ml, int* part_prefix, cudaStream_t s) {
  using L = Layout<HALVES, STAGES>;
  static_assert(L::BYTES <= 227 * 1024, "shared memory of a block");
  auto kern = attn_tree_t5_kernel<HALVES, STAGES>;
  static bool configured[gi::MAX_DEVICES_SEEN] = {false};
  int dev;
  if (gi::unconfigured_here(configured, &dev)) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::BYTES);
    if (e != cudaSuccess) return gi::fail(GI_ERR_CUDA, "tree attention (tcgen05): %s", cudaGetErrorString(e));
    if (dev >= 0) configured[dev] = true;
  }
  return gi::check(gi::launch(kern, dim3(blocks), dim3(L::THREADS), L::BYTES, s, mq, mk, mv, sh, out, ldo, scale, q_box, part_o, part_ml, part_prefix),
                   "tree attention (tcgen05)");
}

}  // namespace

int gi::tree::launch_t5(const Shape& sh, int blocks, void* out, long ldo, const void* q, long ldq, long q_rows, const void* k, const void* v, int hd,
                        float scale, float4* part_o, float2* part_ml, int* part_prefix, cudaStream_t s) {
  CUtensorMap mq, mk, mv;
  const long rows = (long)sh.cache_pages * sh.n_kv * PAGE_TOKENS;
  const int group = sh.n_heads / sh.n_kv;
  int rc = gi::tensor_map_3d(&mq, q, q_rows, sh.n_heads, hd, ldq, hd, 64, group, sh.rows_block / group);
  if (rc == GI_OK) rc = gi::tensor_map_2d_ex(&mk, k, rows, hd, hd, GI_BF16, 64, PAGE_TOKENS);
  if (rc == GI_OK) rc = gi::tensor_map_2d_ex(&mv, v, rows, hd, hd, GI_BF16, 64, PAGE_TOKENS);
  if (rc != GI_OK) return rc;
  if (hd == 128) return launch_kernel<2, 2>(mq, mk, mv, sh, blocks, (__nv_bfloat16*)out, ldo, scale, sh.rows_block, part_o, part_ml, part_prefix, s);
  return launch_kernel<1, 4>(mq, mk, mv, sh, blocks, (__nv_bfloat16*)out, ldo, scale, sh.rows_block, part_o, part_ml, part_prefix, s);
}

extern "C" int gi_attn_tree_status(int* status) {
  int zero = 0;
  cudaError_t e = cudaMemcpyFromSymbol(status, g_tree_status, sizeof(int));
  if (e == cudaSuccess) e = cudaMemcpyToSymbol(g_tree_status, &zero, sizeof(int));
  if (e != cudaSuccess) return gi::fail(GI_ERR_CUDA, "tree attention status: %s", cudaGetErrorString(e));
  return GI_OK;
}

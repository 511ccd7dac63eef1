// What the kernels for attention over trees of drafted tokens share: how the work is cut, which keys a node sees, and the shape
// of the partial results.
//
// The work of a launch is a list of tiles: for every sequence, for every block of query rows (nodes x heads of one kv head's
// group), for every kv head, the 64-position tiles of the sequence's cache up to its last node.  The list is cut into equal
// ranges, one per block: contexts of any lengths then keep all blocks busy to the end.  A block that holds all of a unit's
// tiles (one sequence, row block and kv head) writes its result; what it holds only part of it leaves as maximum, sum and
// unscaled sums of values in slot 2c (the unit began before block c's range) or 2c + 1 (it goes on behind it), and a second
// kernel joins them.  Lengths are read on the device, so that a recorded launch serves any of them.
#pragma once

#include <math.h>

#include "common.cuh"

namespace gi {
namespace tree {

constexpr int TILE = PAGE_TOKENS;
constexpr int MAX_SEQS = 1024;
constexpr int MAX_NODES = 256;

struct Shape {
  const int* cu_seqlens;
  const int* seq_slots;
  const int* seq_pos0;
  const int* block_table;
  const int* masks;       // [tokens][words] bits: the nodes of its own tree that a token sees
  int words, max_pages, n_seqs, n_heads, n_kv, rows_block /* query rows of a row block */, max_nodes;
};

struct Unit {
  int b, row0, kvh;       // sequence, first query row (node * group + head in group) of the row block, kv head
  int n, pos0, slot;      // nodes, cached positions before them
  int tiles;
  long first;             // the unit's first tile in the launch's list
};

__device__ __forceinline__ int nodes_of(const Shape& s, int b) { return max(0, min(s.cu_seqlens[b + 1] - s.cu_seqlens[b], s.max_nodes)); }

__device__ __forceinline__ int pos0_of(const Shape& s, int b) { return max(0, s.seq_pos0[b]); }

// The list's length up to every sequence, [n_seqs + 1], by one warp.
__device__ __forceinline__ void prefix(const Shape& s, long* out) {
  const int lane = threadIdx.x & 31, group = s.n_heads / s.n_kv;
  long upto = 0;
  for (int b0 = 0; b0 < s.n_seqs; b0 += 32) {
    const int b = b0 + lane;
    long own = 0;
    if (b < s.n_seqs) {
      const int n = nodes_of(s, b);
      const long blocks = ((long)n * group + s.rows_block - 1) / s.rows_block;
      if (n > 0) own = blocks * s.n_kv * (long)((pos0_of(s, b) + n + TILE - 1) / TILE);
    }
    long sum = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (b < s.n_seqs) out[b] = upto + sum - own;
    upto += __shfl_sync(0xffffffffu, sum, 31);
  }
  if (lane == 0) out[s.n_seqs] = upto;
}

// Tiles per block: equal ranges, but not so short that joining them would cost more than they save.
__device__ __forceinline__ long per_block(long total, int blocks, int least) {
  const long even = (total + blocks - 1) / blocks;
  return even > least ? even : least;
}

// The unit that holds a tile of the list.
__device__ __forceinline__ Unit unit_at(const Shape& s, const long* pre, long tile) {
  int lo = 0, hi = s.n_seqs;          // pre[lo] <= tile < pre[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (pre[mid] <= tile) lo = mid; else hi = mid;
  }
  Unit u;
  u.b = lo;
  u.n = nodes_of(s, lo);
  u.pos0 = pos0_of(s, lo);
  u.slot = s.seq_slots[lo];
  u.tiles = (u.pos0 + u.n + TILE - 1) / TILE;
  const long k = (tile - pre[lo]) / u.tiles;
  u.kvh = (int)(k % s.n_kv);
  u.row0 = (int)(k / s.n_kv) * s.rows_block;
  u.first = pre[lo] + k * u.tiles;
  return u;
}

// The 32 keys from tree place `o` on (negative: cached before the tree) that a token with these mask words sees.
__device__ __forceinline__ unsigned seen_word(const int* mask, int words, int n, int o) {
  unsigned w = 0;
  if (o <= -32) return 0xffffffffu;
  const int first = o >= 0 ? o >> 5 : -1, shift = o & 31;       // bits [o, o + 32): word `first` from bit `shift` on, and the next
  const unsigned a = first >= 0 ? (first < words ? (unsigned)mask[first] : 0u) : 0xffffffffu;
  const unsigned b = first + 1 < words ? (unsigned)mask[first + 1] : 0u;
  w = __funnelshift_r(a, b, shift);
  const int left = n - o;                                        // places from here on that the tree has
  if (left <= 0) return 0u;
  return left >= 32 ? w : w & ((1u << left) - 1u);
}

// The row of the page table may be anything in an unused slot: a page outside the cache reads as the trash page.
__device__ __forceinline__ int page_of(const Shape& s, int slot, int tile, int cache_pages) {
  if (slot < 0 || tile >= s.max_pages) return 0;
  const int page = s.block_table[(size_t)slot * s.max_pages + tile];
  return page >= 0 && page < cache_pages ? page : 0;
}

// The tensor-core form (attention_tree_t5.cu): rows_block 128 or 256, one or two row tiles a block.
int launch_t5(const Shape& sh, int blocks, void* out, long ldo, const void* q, long ldq, const void* k, const void* v, int cache_pages, int hd,
              float scale, int least, float* part_o, float* part_ml, long* part_prefix, cudaStream_t s);

}  // namespace tree
}  // namespace gi

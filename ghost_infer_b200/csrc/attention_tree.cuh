// What the kernels for attention over trees of drafted tokens share: how the work is cut, which keys a node sees, and the shape
// of the partial results.
//
// The work of a launch is a list of tiles: for every sequence, for every block of query rows (nodes x heads of one kv head's
// group), for every kv head, the tiles of 64 or 128 positions of the sequence's cache up to its last node.  The list is cut into
// equal ranges, one per block: contexts of any lengths then keep all blocks busy to the end.  A block that holds all of a unit's
// tiles (one sequence, row block and kv head) writes its result; what it holds only part of it leaves as maximum, sum and
// unscaled sums of values (four of them to a piece, rows side by side) in slot 2c (the unit began before block c's range) or
// 2c + 1 (it goes on behind it), and a second kernel joins them.  Where a tree has more query rows than a block takes, `split`
// neighbouring blocks walk the same range with a row block each, at the same time: what one of them reads, the others find in
// the L2 cache.  Lengths are read on the device, so that a recorded launch serves any of them.
#pragma once

#include <math.h>

#include "common.cuh"

namespace gi {
namespace tree {

constexpr int MAX_SEQS = 1024;
constexpr int MAX_NODES = 256;

struct Shape {
  const int* cu_seqlens;
  const int* seq_slots;
  const int* seq_pos0;
  const int* block_table;
  const int* masks;       // [tokens][words] bits: the nodes of its own tree that a token sees
  int words, table_rows, max_pages, n_seqs, n_heads, n_kv, max_nodes, cache_pages;
  long tokens;            // rows of queries, masks and output
  int rows_block;         // query rows of a row block
  int split;              // row blocks of a unit, one to each of so many neighbouring blocks
  int tile;               // positions of a tile: 64 or 128
};

struct Unit {
  int b, row0, kvh;       // sequence, first query row (node * group + head in group) of the unit, kv head
  int n, pos0, slot;      // nodes, cached positions before them
  int tiles, first;       // tiles, the first one's place in the launch's list
};

// (offsets that the rows do not hold name no node)
__device__ __forceinline__ int nodes_of(const Shape& s, int b) {
  const int first = s.cu_seqlens[b], end = (int)min((long)s.cu_seqlens[b + 1], s.tokens);
  return first < 0 ? 0 : max(0, min(end - first, s.max_nodes));
}

// (a length that the page table cannot hold is cut off: the entry point bounds the list by the table's)
__device__ __forceinline__ int pos0_of(const Shape& s, int b) { return max(0, min(s.seq_pos0[b], s.max_pages * PAGE_TOKENS)); }

__device__ __forceinline__ int tiles_of(const Shape& s, int pos0, int n) { return (pos0 + n + s.tile - 1) / s.tile; }

// The list's length up to every sequence, [n_seqs + 1], by one warp.
__device__ __forceinline__ void prefix(const Shape& s, int* out) {
  const int lane = threadIdx.x & 31, group = s.n_heads / s.n_kv;
  int upto = 0;
  for (int b0 = 0; b0 < s.n_seqs; b0 += 32) {
    const int b = b0 + lane;
    int own = 0;
    if (b < s.n_seqs) {
      const int n = nodes_of(s, b), pos0 = pos0_of(s, b);
      if (n > 0) own = (n * group + s.rows_block * s.split - 1) / (s.rows_block * s.split) * s.n_kv * tiles_of(s, pos0, n);
    }
    int sum = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += up;
    }
    if (b < s.n_seqs) out[b] = upto + sum - own;
    upto += __shfl_sync(0xffffffffu, sum, 31);
  }
  if (lane == 0) out[s.n_seqs] = upto;
}

// Tiles per range: equal ranges of one tile at least.
__device__ __forceinline__ int per_range(int total, int ranges) { return max((total + ranges - 1) / ranges, 1); }

// The unit that holds a tile of the list.
__device__ __forceinline__ Unit unit_at(const Shape& s, const int* pre, int tile) {
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
  u.tiles = tiles_of(s, u.pos0, u.n);
  const unsigned k = (unsigned)(tile - pre[lo]) / (unsigned)u.tiles, rb = k / (unsigned)s.n_kv;
  u.kvh = (int)(k - rb * s.n_kv);
  u.row0 = (int)rb * s.rows_block * s.split;
  u.first = pre[lo] + (int)k * u.tiles;
  return u;
}

// The 32 keys from tree place `o` on (negative: cached before the tree) that a token with these mask words sees.
__device__ __forceinline__ unsigned seen_word(const int* mask, int words, int n, int o) {
  if (o <= -32) return 0xffffffffu;
  const int left = n - o;                                        // places from here on that the tree has
  if (left <= 0) return 0u;
  const int first = o >= 0 ? o >> 5 : -1, shift = o & 31;       // bits [o, o + 32): word `first` from bit `shift` on, and the next
  const unsigned a = first >= 0 ? (first < words ? (unsigned)mask[first] : 0u) : 0xffffffffu;
  const unsigned b = first + 1 < words ? (unsigned)mask[first + 1] : 0u;
  const unsigned w = __funnelshift_r(a, b, shift);
  return left >= 32 ? w : w & ((1u << left) - 1u);
}

// Where four numbers of a row of a partial result lie: neighbouring rows side by side, since the threads that write and read them
// own a row each.
__device__ __forceinline__ size_t part_at(const Shape& s, size_t slot, int fours, int four, int row) {
  return (slot * fours + four) * s.rows_block + row;
}

// The cache's page that holds a sequence's positions from 64 * index on.  A table may hold anything behind a sequence's end and in
// an unused slot: what is no page of the cache, and a slot that the table does not have, reads as the trash page.
__device__ __forceinline__ int page_of(const Shape& s, int slot, int index) {
  if (slot < 0 || slot >= s.table_rows || index >= s.max_pages) return 0;
  const int page = s.block_table[(size_t)slot * s.max_pages + index];
  return page >= 0 && page < s.cache_pages ? page : 0;
}

// The tensor-core form (attention_tree_t5.cu): rows_block up to 128, of whole nodes; tiles of 128.
int launch_t5(const Shape& sh, int blocks, void* out, long ldo, const void* q, long ldq, long q_rows, const void* k, const void* v, int hd, float scale,
              float4* part_o, float2* part_ml, int* part_prefix, cudaStream_t s);

}  // namespace tree
}  // namespace gi

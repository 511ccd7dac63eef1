// What a step over trees of drafted tokens leaves behind: the walk through each tree as far as the model's picks agree, and the
// accepted tokens' keys and values moved up to follow the cache directly.
//
// A sequence's nodes were stored at the positions pos0, pos0 + 1, ... in their order (a node comes after its parent), node 0
// being the token that would have been fed anyway.  The walk starts there; from a node it goes to the first of its children
// whose token is what the model picks at the node, and ends where there is none.  The accepted nodes, in the order of the
// walk, get positions pos0, pos0 + 1, ...: node path[i] moves to pos0 + i.  path[i] >= i and the path ascends, so no move
// overwrites what a later one reads; a thread that moves its column of 2 to 16 bytes of every accepted row in the path's order
// needs nobody to wait for.
// Every block repeats the walk over its sequence's nodes in shared memory (one warp, a round of the nodes per accepted one): that
// costs less than a launch of its own that the moves would wait for.  Bound: latency.  B200: one tree of 26 nodes, 28 layers, 4 us; 64
// trees of up to 61 nodes 17 us for 35 MB (blocks of several columns a thread, so fewer walks: 16 us with 8 blocks an SM, 20 with 4, 28
// with 2; it is the rows' trips to memory that take the time).
#include "api.h"
#include "common.cuh"
#include "page_tensors.cuh"

namespace {

constexpr int THREADS = 256;
constexpr int MAX_NODES = 256;
template <typename V>
__global__ void __launch_bounds__(THREADS)
tree_commit_kernel(const __grid_constant__ gi::PageTensors t, int n_tensors, const int* picks, const int* tokens, const int* parents,
                   int n_tokens, const int* cu_seqlens, const int* seq_slots, const int* seq_pos0, const int* block_table, int table_rows, int max_pages, int max_nodes,
                   int* __restrict__ out_path, int* __restrict__ out_counts, int* __restrict__ out_next) {
  __shared__ int s_token[MAX_NODES], s_parent[MAX_NODES], s_pick[MAX_NODES], s_path[MAX_NODES], s_page[MAX_NODES / PAGE_TOKENS + 2];
  __shared__ int s_count;
  const int tid = threadIdx.x, lane = tid & 31, b = blockIdx.y;
  gi::pdl_prologue();
  const int tok0 = cu_seqlens[b], end = min(cu_seqlens[b + 1], n_tokens), slot = seq_slots[b], pos0 = seq_pos0[b];
  const int n = tok0 < 0 ? 0 : min(end - tok0, max_nodes);
  for (int i = tid; i < n; i += THREADS) {
    s_token[i] = tokens[tok0 + i];
    s_parent[i] = parents[tok0 + i];
    s_pick[i] = picks[tok0 + i];
  }
  const int page0 = pos0 / PAGE_TOKENS, n_pages = MAX_NODES / PAGE_TOKENS + 2;
  for (int i = tid; i < n_pages; i += THREADS)
    s_page[i] = slot >= 0 && slot < table_rows && pos0 >= 0 && page0 + i < max_pages ? block_table[(size_t)slot * max_pages + page0 + i] : -1;
  __syncthreads();
  if (tid < 32) {
    int count = 0, at = 0;
    bool on = n > 0;
    while (on) {                              // (ascends: at most n rounds)
      if (lane == 0) s_path[count] = at;
      ++count;
      const int pick = s_pick[at];
      int next = n;
      for (int i0 = at + 1; i0 < n && next == n; i0 += 32) {
        const int i = i0 + lane;
        const unsigned who = __ballot_sync(0xffffffffu, i < n && s_parent[i] == at && s_token[i] == pick);
        if (who) next = i0 + __ffs(who) - 1;
      }
      on = next < n;
      if (on) at = next;
    }
    if (lane == 0) {
      s_count = count;
      if (blockIdx.x == 0) {
        out_counts[b] = count;
        out_next[b] = count > 0 ? s_pick[at] : -1;
      }
    }
  }
  __syncthreads();
  const int count = s_count;
  if (blockIdx.x == 0)
    for (int i = tid; i < max_nodes; i += THREADS) out_path[(size_t)b * max_nodes + i] = i < count ? s_path[i] : -1;
  int first = 0;                              // what is in its place already
  while (first < count && s_path[first] == first) ++first;
  if (first >= count) return;

  long col = (long)blockIdx.x * THREADS + tid;
  int z = 0;
  auto columns = [&](int i) { return (long)t.layers[i] * t.heads[i] * t.row_units[i]; };
  while (z < n_tensors && col >= columns(z)) col -= columns(z++);
  if (z >= n_tensors) return;
  const int ru = t.row_units[z], c = (int)(col % ru), head = (int)(col / ru % t.heads[z]), layer = (int)(col / ru / t.heads[z]);
  V* base = (V*)t.base[z];
  const int off0 = pos0 % PAGE_TOKENS;
  auto place = [&](int i) -> V* {             // the column's place of position pos0 + i; null outside the cache
    const int page = s_page[(off0 + i) / PAGE_TOKENS];
    if (page < 0 || page >= t.pages[z]) return nullptr;
    return base + ((((size_t)layer * t.pages[z] + page) * t.heads[z] + head) * PAGE_TOKENS + (off0 + i) % PAGE_TOKENS) * ru + c;
  };
  constexpr int AHEAD = 8;
  for (int i0 = first; i0 < count; i0 += AHEAD) {
    V held[AHEAD];
    bool ok[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      ok[k] = i0 + k < count;
      if (ok[k]) {
        const V* from = place(s_path[i0 + k]);
        ok[k] = from != nullptr;
        if (ok[k]) held[k] = *from;
      }
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
      if (ok[k]) {
        V* to = place(i0 + k);
        if (to != nullptr) *to = held[k];
      }
  }
}

}  // namespace

extern "C" int gi_tree_commit(int* out_path, int* out_counts, int* out_next, const int* picks, const int* tokens, const int* parents,
                              int n_tokens, const int* cu_seqlens, const int* seq_slots, const int* seq_pos0, int n_seqs, int max_nodes,
                              const long* tensors, int n, const int* block_table, int table_rows, int max_pages, void* stream) {
  if (n_seqs <= 0) return GI_OK;
  if (max_nodes < 1 || max_nodes > MAX_NODES) return gi::fail(GI_ERR_ARG, "tree commit: trees of up to %d nodes, 1 to %d are supported", max_nodes, MAX_NODES);
  if (n_seqs > 65535) return gi::fail(GI_ERR_UNSUPPORTED, "tree commit: more than 65535 sequences in one launch");
  gi::PageTensors t;
  int unit;
  const int rc = t.read(tensors, n, &unit, "tree commit");
  if (rc != GI_OK) return rc;
  long columns = 0;
  for (int i = 0; i < n; ++i) columns += (long)t.layers[i] * t.heads[i] * t.row_units[i];
  const long blocks = columns > 0 ? (columns + THREADS - 1) / THREADS : 1;
  if (blocks > 0x7fffffffL) return gi::fail(GI_ERR_UNSUPPORTED, "tree commit: more rows' columns than one launch holds");
  const dim3 grid((unsigned)blocks, n_seqs);
  cudaStream_t s = (cudaStream_t)stream;
#define GI_TREE(V) gi::check(gi::launch(tree_commit_kernel<V>, grid, dim3(THREADS), 0, s, t, n, picks, tokens, parents, n_tokens, cu_seqlens, seq_slots, seq_pos0, \
                                        block_table, table_rows, max_pages, max_nodes, out_path, out_counts, out_next), "tree commit")
  if (unit == 16) return GI_TREE(uint4);
  if (unit == 4) return GI_TREE(unsigned);
  return GI_TREE(unsigned short);
#undef GI_TREE
}

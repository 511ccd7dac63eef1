// Sequences that part and go on as several: fixed-size states that follow their beams, and copies of cache pages.
//
// States: in every tensor [rows][row bytes] row slot[s][j] takes what row slot[s][parent[s][j]] holds, all at once: beams may swap,
// several may take the same one's.  A thread owns one column of 1 to 16 bytes of all of a sequence's beams, reads what it
// needs of the column before it writes any of it, and so needs no second copy of the states: every row that changes is written
// once, every row that others take is read once (a second reader of a row finds it in the caches).  Up to 16 beams a
// thread's column stays in registers, several columns side by side with few beams; above that it goes through shared memory.
//
// Pages: the first `rows` positions of page src[i] are copied to page dst[i], for every layer and kv head.  A head's filled rows of
// a page are one stretch of memory.
//
// Both are bound by the bytes they move: B200, states of 8 sequences of 8 beams in 4 layers, 2 MB each, 88 us (6.2 TB/s); 128 pages of 28
// layers, 8 kv heads of 128, half filled, 145 us (6.5 TB/s).  Not so above 16 beams, where shared memory leaves few columns to an SM: the
// same states of 2 sequences of 32 beams take 305 us (1.8 TB/s), of one of 64 beams 372 us.
#include "api.h"
#include "common.cuh"
#include "page_tensors.cuh"

namespace {

constexpr int THREADS = 256;
constexpr int MAX_BEAMS = 64;
constexpr int MAX_TENSORS = 64;

struct StateTensors {
  void* base[MAX_TENSORS];
  long units[MAX_TENSORS];       // a row's size in units of the column's type
};

// K: most beams of a sequence, COLS: columns a thread takes side by side
template <typename V, int K, int COLS>
__global__ void __launch_bounds__(THREADS)
reorder_states_kernel(const __grid_constant__ StateTensors t, const int* slots, const int* parents, int beams, int rows) {
  __shared__ int s_from[K], s_to[K];
  __shared__ int s_moves;
  const int tid = threadIdx.x, seq = blockIdx.y;
  const long units = t.units[blockIdx.z];
  const long col0 = (long)blockIdx.x * THREADS * COLS + tid;
  if (tid == 0) s_moves = 0;
  gi::pdl_prologue();
  if ((long)blockIdx.x * THREADS * COLS >= units) return;
  __syncthreads();
  if (tid < K) {
    int from = -1, to = -1;
    if (tid < beams) {
      const int p = parents[(size_t)seq * beams + tid];
      to = slots[(size_t)seq * beams + tid];
      if (p >= 0 && p < beams) from = slots[(size_t)seq * beams + p];
      // no parent, or a slot that is none: the row stays as it is
      if (from < 0 || from >= rows || to < 0 || to >= rows || from == to) from = to = -1;
    }
    s_from[tid] = from;
    s_to[tid] = to;
    if (to >= 0) s_moves = 1;
  }
  __syncthreads();
  if (!s_moves) return;
  V* base = (V*)t.base[blockIdx.z];
  V held[COLS][K];
#pragma unroll
  for (int c = 0; c < COLS; ++c)
#pragma unroll
    for (int j = 0; j < K; ++j)
      if (s_from[j] >= 0 && col0 + c * THREADS < units) held[c][j] = base[(size_t)s_from[j] * units + col0 + c * THREADS];
#pragma unroll
  for (int c = 0; c < COLS; ++c)
#pragma unroll
    for (int j = 0; j < K; ++j)
      if (s_to[j] >= 0 && col0 + c * THREADS < units) base[(size_t)s_to[j] * units + col0 + c * THREADS] = held[c][j];
}

// The same for more beams than a thread's registers hold: [beams][THREADS] columns in shared memory, every thread its own.
template <typename V>
__global__ void __launch_bounds__(THREADS)
reorder_many_states_kernel(const __grid_constant__ StateTensors t, const int* slots, const int* parents, int beams, int rows) {
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int s_from[MAX_BEAMS], s_to[MAX_BEAMS];
  V* held = (V*)smem;
  const int tid = threadIdx.x, seq = blockIdx.y;
  const long units = t.units[blockIdx.z];
  const long col = (long)blockIdx.x * THREADS + tid;
  gi::pdl_prologue();
  if ((long)blockIdx.x * THREADS >= units) return;
  if (tid < beams) {
    const int p = parents[(size_t)seq * beams + tid];
    const int to = slots[(size_t)seq * beams + tid];
    const int from = p >= 0 && p < beams ? slots[(size_t)seq * beams + p] : -1;
    const bool moves = from >= 0 && from < rows && to >= 0 && to < rows && from != to;
    s_from[tid] = moves ? from : -1;
    s_to[tid] = moves ? to : -1;
  }
  __syncthreads();
  if (col >= units) return;
  V* base = (V*)t.base[blockIdx.z];
#pragma unroll 8
  for (int j = 0; j < beams; ++j)
    if (s_from[j] >= 0) held[j * THREADS + tid] = base[(size_t)s_from[j] * units + col];
#pragma unroll 8
  for (int j = 0; j < beams; ++j)
    if (s_to[j] >= 0) base[(size_t)s_to[j] * units + col] = held[j * THREADS + tid];
}

template <typename V>
int launch_states(const StateTensors& t, int n, const int* slots, const int* parents, int seqs, int beams, int rows, cudaStream_t s) {
  long most = 0;
  for (int i = 0; i < n; ++i) most = t.units[i] > most ? t.units[i] : most;
  auto grid = [&](int cols) { return dim3((unsigned)((most + (long)THREADS * cols - 1) / ((long)THREADS * cols)), seqs, n); };
  if (beams <= 4)
    return gi::check(gi::launch(reorder_states_kernel<V, 4, 4>, grid(4), dim3(THREADS), 0, s, t, slots, parents, beams, rows), "state reordering");
  if (beams <= 8)
    return gi::check(gi::launch(reorder_states_kernel<V, 8, 2>, grid(2), dim3(THREADS), 0, s, t, slots, parents, beams, rows), "state reordering");
  if (beams <= 16)
    return gi::check(gi::launch(reorder_states_kernel<V, 16, 1>, grid(1), dim3(THREADS), 0, s, t, slots, parents, beams, rows), "state reordering");
  const size_t smem = (size_t)beams * THREADS * sizeof(V);
  if (smem > 160 * 1024) {      // 16-byte columns of more than 40 beams: go by 4 bytes (64 KB)
    StateTensors narrow = t;
    for (int i = 0; i < n; ++i) narrow.units[i] *= sizeof(V) / 4;
    return launch_states<unsigned>(narrow, n, slots, parents, seqs, beams, rows, s);
  }
  auto kern = reorder_many_states_kernel<V>;
  static bool configured[gi::MAX_DEVICES_SEEN] = {false};
  int dev;
  if (gi::unconfigured_here(configured, &dev)) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (e != cudaSuccess) return gi::fail(GI_ERR_CUDA, "state reordering: %s", cudaGetErrorString(e));
    if (dev >= 0) configured[dev] = true;
  }
  return gi::check(gi::launch(kern, grid(1), dim3(THREADS), smem, s, t, slots, parents, beams, rows), "state reordering");
}

template <typename V>
__global__ void __launch_bounds__(THREADS)
copy_pages_kernel(const __grid_constant__ gi::PageTensors t, const int* src, const int* dst, const int* rows, int copies) {
  constexpr int AHEAD = 4;
  const int z = blockIdx.z, layer = blockIdx.x / t.heads[z], head = blockIdx.x % t.heads[z];
  gi::pdl_prologue();
  if (layer >= t.layers[z]) return;
  for (int i = blockIdx.y; i < copies; i += gridDim.y) {
    const int from = src[i], to = dst[i], n = rows == nullptr ? PAGE_TOKENS : min(max(rows[i], 0), PAGE_TOKENS);
    if (from < 0 || from >= t.pages[z] || to < 0 || to >= t.pages[z] || from == to) continue;
    const size_t stretch = (size_t)PAGE_TOKENS * t.row_units[z];
    const V* a = (const V*)t.base[z] + (((size_t)layer * t.pages[z] + from) * t.heads[z] + head) * stretch;
    V* b = (V*)t.base[z] + (((size_t)layer * t.pages[z] + to) * t.heads[z] + head) * stretch;
    const int units = n * t.row_units[z];
    for (int u = threadIdx.x; u < units; u += AHEAD * THREADS) {
      V held[AHEAD];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        if (u + k * THREADS < units) held[k] = a[u + k * THREADS];
#pragma unroll
      for (int k = 0; k < AHEAD; ++k)
        if (u + k * THREADS < units) b[u + k * THREADS] = held[k];
    }
  }
}

}  // namespace

extern "C" int gi_reorder_states(const long* states, int n, int unit, const int* slots, const int* parents, int seqs, int beams, int rows, void* stream) {
  if (seqs <= 0 || n <= 0) return GI_OK;
  if (beams < 1 || beams > MAX_BEAMS) return gi::fail(GI_ERR_ARG, "state reordering: %d beams, 1 to %d are supported", beams, MAX_BEAMS);
  if (seqs > 65535) return gi::fail(GI_ERR_UNSUPPORTED, "state reordering: more than 65535 sequences in one launch");
  if (rows < 1) return gi::fail(GI_ERR_ARG, "state reordering: states of %d rows", rows);
  if (unit != 16 && unit != 4 && unit != 1) return gi::fail(GI_ERR_ARG, "state reordering: a unit of %d bytes", unit);
  for (int first = 0; first < n; first += MAX_TENSORS) {
    StateTensors t = {};
    const int here = n - first < MAX_TENSORS ? n - first : MAX_TENSORS;
    for (int i = 0; i < here; ++i) {
      const long address = states[2 * (first + i)], row_bytes = states[2 * (first + i) + 1];
      if (row_bytes < 1 || row_bytes % unit != 0 || address % unit != 0)
        return gi::fail(GI_ERR_ARG, "state reordering: rows of %ld bytes do not come in units of %d", row_bytes, unit);
      t.base[i] = (void*)address;
      t.units[i] = row_bytes / unit;
    }
    cudaStream_t s = (cudaStream_t)stream;
    const int rc = unit == 16 ? launch_states<uint4>(t, here, slots, parents, seqs, beams, rows, s)
                   : unit == 4 ? launch_states<unsigned>(t, here, slots, parents, seqs, beams, rows, s)
                               : launch_states<unsigned char>(t, here, slots, parents, seqs, beams, rows, s);
    if (rc != GI_OK) return rc;
  }
  return GI_OK;
}

extern "C" int gi_copy_pages(const long* tensors, int n, const int* src, const int* dst, const int* rows, int copies, void* stream) {
  if (copies <= 0 || n <= 0) return GI_OK;
  gi::PageTensors t;
  int unit;
  const int rc = t.read(tensors, n, &unit, "page copies");
  if (rc != GI_OK) return rc;
  long most = 0;
  for (int i = 0; i < n; ++i) most = (long)t.layers[i] * t.heads[i] > most ? (long)t.layers[i] * t.heads[i] : most;
  if (most > 0x7fffffffL) return gi::fail(GI_ERR_UNSUPPORTED, "page copies: more than 2^31 - 1 heads of all layers");
  const dim3 grid((unsigned)most, copies < 65535 ? copies : 65535, n);
  cudaStream_t s = (cudaStream_t)stream;
  if (unit == 16) return gi::check(gi::launch(copy_pages_kernel<uint4>, grid, dim3(THREADS), 0, s, t, src, dst, rows, copies), "page copies");
  if (unit == 4) return gi::check(gi::launch(copy_pages_kernel<unsigned>, grid, dim3(THREADS), 0, s, t, src, dst, rows, copies), "page copies");
  return gi::check(gi::launch(copy_pages_kernel<unsigned short>, grid, dim3(THREADS), 0, s, t, src, dst, rows, copies), "page copies");
}

// The accepted path's cache rows moved together.
//
// A verified tree leaves its nodes' K and V in the cache in node order; the path
// that was accepted is node 0 (the last token before the tree) and some of the others.
// In every layer, for j = 1 .. n:  slot(start + j) <- slot(start + path[j]).
// The path ascends and starts at node 0, so path[j] >= j: a row moves to its own
// place or forward of everything read after it, and one thread that moves a 16-byte
// column of the rows in the order j = 1, 2, .. needs no second buffer.
//
// A CTA takes some columns of one sequence (the grid spreads layers, K and V and
// columns), so a batch's few megabytes are spread over all SMs; it is bound by the
// latency of a load and a store behind each other per eight rows, and, for large
// batches, by HBM. Measured: 24 layers of e4m3 rows (2 heads of 64), one sequence, 1.9 us in a replayed graph
// (3.4 a call, host time); 36 layers of bf16 rows (2 heads of 128), 64 sequences of up to 16 nodes (6.9 MB moved), 5.1 us.
#include "kve_common.cuh"

namespace kve {
namespace {

constexpr int kThreads = 128;
constexpr int kMaxPath = 1024;
constexpr int kAhead = 8;  // rows loaded before the first of them is stored

struct PathParams {
  uint8_t* pool[2];
  uint8_t* scale[2];  // null without scales
  const int32_t* tables;
  int table_stride;
  const int32_t* start;
  const int32_t* path;
  const int32_t* n_acc;
  int width, layers, bs, nkv;
  int64_t num_blocks;
  int row_bytes;
  int* status;
};

template <typename V>
__device__ __forceinline__ void move(uint8_t* base, int64_t row_bytes, const int64_t* from, const int64_t* to, int n) {
  for (int j = 0; j < n; j += kAhead) {
    V v[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (j + i < n) v[i] = *reinterpret_cast<const V*>(base + from[j + i] * row_bytes);
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
      if (j + i < n) *reinterpret_cast<V*>(base + to[j + i] * row_bytes) = v[i];
  }
}

__global__ void __launch_bounds__(kThreads) commit_path_kernel(PathParams p) {
  grid_dep_wait();
  grid_dep_launch();
  extern __shared__ int64_t slots[];  // from [width], to [width]
  const int b = blockIdx.y;
  const int n = p.n_acc[b], start = p.start[b];
  const int32_t* path = p.path + (size_t)b * p.width;
  const int32_t* table = p.tables + (size_t)b * p.table_stride;
  if (n <= 0 && n >= -1) return;  // -1: a sequence without a tree
  bool bad = n < -1 || n >= p.width || start < 0;
  __shared__ int first, any_bad;
  if (threadIdx.x == 0) { first = n; any_bad = 0; }
  __syncthreads();
  int64_t* from = slots;
  int64_t* to = slots + p.width;
  for (int j = 1 + threadIdx.x; !bad && j <= n; j += kThreads) {
    const int node = path[j], before = j == 1 ? 0 : path[j - 1];
    if (node <= before) { bad = true; break; }
    const int64_t src = (int64_t)start + node, dst = (int64_t)start + j;
    if (src >= (int64_t)p.table_stride * p.bs) { bad = true; break; }
    const int bf = table[src / p.bs], bt = table[dst / p.bs];
    if (bf < 0 || bf >= p.num_blocks || bt < 0 || bt >= p.num_blocks) { bad = true; break; }
    from[j - 1] = (int64_t)bf * p.bs + src % p.bs;
    to[j - 1] = (int64_t)bt * p.bs + dst % p.bs;
    if (node != j) atomicMin(&first, j - 1);  // rows before the first that moves stay where they are
  }
  if (bad) any_bad = 1;
  __syncthreads();
  if (any_bad) {
    if (threadIdx.x == 0 && blockIdx.x == 0) report(p.status, KVE_ERR_BOUNDS);
    return;
  }
  const int skip = first;
  if (skip >= n) return;
  const int64_t per_layer = p.num_blocks * p.bs;
  const int cols = p.row_bytes / 16;
  const int per = cols + (p.scale[0] ? p.nkv : 0);  // 16-byte columns, then scale bytes, of K or V of one layer
  const int64_t items = (int64_t)p.layers * 2 * per;
  for (int64_t i = blockIdx.x * (int64_t)kThreads + threadIdx.x; i < items; i += (int64_t)gridDim.x * kThreads) {
    const int64_t lk = i / per;
    const int col = (int)(i - lk * per);
    const int64_t layer = lk >> 1;
    const int kv = (int)(lk & 1);
    if (col < cols)
      move<uint4>(p.pool[kv] + layer * per_layer * p.row_bytes + col * 16, p.row_bytes, from + skip, to + skip, n - skip);
    else
      move<uint8_t>(p.scale[kv] + layer * per_layer * p.nkv + (col - cols), p.nkv, from + skip, to + skip, n - skip);
  }
}

}  // namespace
}  // namespace kve

using namespace kve;

extern "C" int kve_kv_commit_path(void* pool_k, void* pool_v, int kv_dtype, uint8_t* k_scale, uint8_t* v_scale,
                                  int num_layers, int64_t num_blocks, int block_size, int num_kv_heads, int head_dim,
                                  const int32_t* block_tables, int table_stride, const int32_t* start_lens,
                                  const int32_t* path, int path_stride, const int32_t* n_accepted, int batch,
                                  int* dev_status, cudaStream_t stream) {
  const char* me = "kve_kv_commit_path";
  if (batch < 0 || num_layers < 1 || num_blocks < 1 || block_size < 1 || num_kv_heads < 1 || head_dim < 1 ||
      table_stride < 1 || path_stride < 1)
    return set_error(KVE_ERR_ARG, "%s: bad sizes", me);
  const int elem = kv_dtype == KVE_F32 ? 4 : kv_dtype == KVE_BF16 ? 2 : kv_dtype == KVE_FP8_E4M3 ? 1 : 0;
  if (!elem) return set_error(KVE_ERR_DTYPE, "%s: cache dtype %d", me, kv_dtype);
  const int64_t row = (int64_t)num_kv_heads * head_dim * elem;
  if (row % 16 || row > (1 << 24)) return set_error(KVE_ERR_SHAPE, "%s: %lld bytes a row (a multiple of 16)", me, (long long)row);
  if (path_stride > kMaxPath) return set_error(KVE_ERR_SHAPE, "%s: path_stride %d > %d", me, path_stride, kMaxPath);
  if (batch > 65535) return set_error(KVE_ERR_SHAPE, "%s: batch %d > 65535", me, batch);
  if (batch == 0) return KVE_OK;
  if (!pool_k || !pool_v || !block_tables || !start_lens || !path || !n_accepted)
    return set_error(KVE_ERR_ARG, "%s: null pointer", me);
  if ((kv_dtype == KVE_FP8_E4M3) != (k_scale != nullptr) || (k_scale != nullptr) != (v_scale != nullptr))
    return set_error(KVE_ERR_ARG, "%s: scales belong to an e4m3 cache", me);
  if ((uintptr_t)pool_k % 16 || (uintptr_t)pool_v % 16)
    return set_error(KVE_ERR_ARG, "%s: pools must be 16-byte aligned", me);
  PathParams p{};
  p.pool[0] = static_cast<uint8_t*>(pool_k); p.pool[1] = static_cast<uint8_t*>(pool_v);
  p.scale[0] = k_scale; p.scale[1] = v_scale;
  p.tables = block_tables; p.table_stride = table_stride; p.start = start_lens; p.path = path; p.n_acc = n_accepted;
  p.width = path_stride; p.layers = num_layers; p.bs = block_size; p.nkv = num_kv_heads; p.num_blocks = num_blocks;
  p.row_bytes = (int)row; p.status = dev_status;
  const int64_t items = (int64_t)num_layers * 2 * (row / 16 + (k_scale ? num_kv_heads : 0));
  const int64_t blocks = (items + kThreads - 1) / kThreads;
  launch_kernel(commit_path_kernel, dim3((unsigned)(blocks < 1024 ? blocks : 1024), batch), dim3(kThreads),
                (size_t)path_stride * 2 * sizeof(int64_t), stream, p);
  return check_launch(me);
}

// What the two kernels of tree attention share: the parameters of a call, the
// workspace's layout and the mask words.
#pragma once

#include "kve_common.cuh"

namespace kve {

// The workspace starts with the arrival counters, at the same addresses for every
// call and every op that shares it, so that no call's partials ever land on them.
constexpr size_t kTreeCounterSlots = 16384;
constexpr size_t kTreeCounterBytes = kTreeCounterSlots * sizeof(int32_t);

struct TreeParams {
  const void* q;
  const void* pool_k;
  const void* pool_v;
  const uint8_t* k_scale;
  const uint8_t* v_scale;
  const int32_t* tables;
  int table_stride;
  const int32_t* ctx_lens;
  const int32_t* q_lens;
  const int32_t* q_offsets;
  const uint32_t* mask;
  int mask_words;
  int q_rows, max_q, nq, nkv, group, bs;
  int64_t num_blocks;
  float scale;
  void* out;
  int* counters;
  float* partials;
  int chunk, n_chunks, n_qtiles;
  uint32_t group_inv;  // floor(2^32 / group) + 1: r / group = umulhi(r, it) for r < 2^16 (group 1: not used)
  int* status;
};

// Row r (below 2^16) of a sequence and kv head: its node.
__device__ __forceinline__ int node_of(const TreeParams& p, int r) {
  return p.group == 1 ? r : (int)__umulhi((uint32_t)r, p.group_inv);
}

// The wide kernel (tree_attn_tc.cu): its partials of a call, and the call itself: e4m3
// caches, and bf16 ones with a block size of a multiple of 16 and a pool of under 2^31 - 16 rows.
size_t tree_attn_wide_partial_bytes(int batch, int max_q, int max_ctx, int nkv, int group, int hd);
int tree_attn_wide(TreeParams p, int batch, int max_ctx, int hd, bool fp8, cudaStream_t stream);

// The kernel for at most eight rows (tree_attn_small.cu): whether it takes a call (bf16 queries), its
// partials, and the call.
bool tree_attn_small_takes(const TreeParams& p, bool fp8);
size_t tree_attn_small_partial_bytes(int batch, int max_ctx, int nkv, int hd);
int tree_attn_small(TreeParams p, int batch, int max_ctx, int hd, bool fp8, cudaStream_t stream);
// 2^(byte - 127); byte 255 stands for NaN.
__device__ __forceinline__ float scale_value(uint32_t byte) {
  return byte == 0 ? __uint_as_float(0x00400000u) : byte == 255 ? __uint_as_float(0x7fc00000u) : __uint_as_float(byte << 23);
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// Bits j0 .. j0 + N - 1 (N <= 32) of a row's mask, as seen from key j0 of the new tokens
// (negative: history, always seen). Bits past the words are clear.
template <int N>
__device__ __forceinline__ uint32_t mask_bits(const uint32_t* row, int words, int j0) {
  if (j0 <= -N) return ~0u;
  const int lo = j0 < 0 ? 0 : j0;
  const int w = lo >> 5, s = lo & 31;
  uint32_t v = w < words ? row[w] >> s : 0u;
  if (s && w + 1 < words) v |= row[w + 1] << (32 - s);
  if (j0 < 0) v = v << -j0 | ((1u << -j0) - 1u);
  return v;
}
// The same without mask words: new token j0 + x is seen where it is not behind `node`.
__device__ __forceinline__ uint32_t chain_bits(int node, int j0) {
  const int d = node - j0;
  return d < 0 ? 0u : d >= 31 ? ~0u : (2u << d) - 1u;
}

}  // namespace kve

// What the kernels of tree attention share: the parameters of a call, the workspace's
// layout, the mask words and the way round the products.
#pragma once

#include <cuda_fp8.h>
#include <math.h>

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

// Rows row0 .. row0 + rows - 1 of sequence b and kv head h over the keys [key_lo, key_hi), key by key over
// what each row sees, in plain fp32: for the few calls in which the products of whole tiles give what the
// formula does not, infinities among them. A warp a row, HD / 32 dims a lane. Into `out`, or, where
// the keys are split, as [row][HD + 4] partials with m and l behind the dims into `part`. Q: of q, out and, but for FP8, the cache.
template <typename Q, bool FP8, int HD, int THREADS>
__device__ __forceinline__ void attend_by_key(const TreeParams& p, int b, int h, int qoff, int hist, int key_lo, int key_hi,
                                              int row0, int rows, int warp, int lane, bool split, float* part) {
  constexpr int DPL = HD / 32;
  const int32_t* table = p.tables + (size_t)b * p.table_stride;
  auto element = [](const void* pool, const uint8_t* scales, size_t row, int d) {
    if constexpr (FP8)
      return scale_value(scales[row]) *
             __half2float(__half(__nv_cvt_fp8_to_halfraw(static_cast<const uint8_t*>(pool)[row * HD + d], __NV_E4M3)));
    else
      return Elem<Q>::to_f(static_cast<const Q*>(pool)[row * HD + d]);
  };
  const float sl = p.scale * 1.4426950408889634f;
  for (int r = warp; r < rows; r += THREADS / 32) {
    const int gr = row0 + r, node = node_of(p, gr);
    const size_t head = ((size_t)(qoff + node) * p.nq + h * p.group + gr - node * p.group) * HD;  // the row in q and out
    const uint32_t* mask = p.mask ? p.mask + (size_t)(qoff + node) * p.mask_words : nullptr;
    float qv[DPL], acc[DPL] = {};
#pragma unroll
    for (int d = 0; d < DPL; ++d) qv[d] = Elem<Q>::to_f(static_cast<const Q*>(p.q)[head + lane + 32 * d]);
    float rm = -INFINITY, rl = 0.f;
    for (int key = key_lo; key < key_hi; ++key) {
      const int j = key - hist;
      if (j >= 0 && !(mask ? mask_bits<1>(mask, p.mask_words, j) & 1u : j <= node)) continue;
      const int blk = table[key / p.bs];
      const bool in = blk >= 0 && blk < p.num_blocks;  // reported by the loader
      const size_t at = in ? ((size_t)blk * p.bs + key % p.bs) * p.nkv + h : 0;
      float s = 0.f;
#pragma unroll
      for (int d = 0; d < DPL; ++d) s += in ? qv[d] * element(p.pool_k, p.k_scale, at, lane + 32 * d) : 0.f;
      s = warp_sum(s) * sl;
      if (s > rm) {
        const float f = ex2(rm - s);
        rm = s;
        rl *= f;
#pragma unroll
        for (int d = 0; d < DPL; ++d) acc[d] *= f;
      }
      const float e = s == -INFINITY ? 0.f : ex2(s - rm);
      rl += e;
#pragma unroll
      for (int d = 0; d < DPL; ++d)
        if (e != 0.f) acc[d] += in ? e * element(p.pool_v, p.v_scale, at, lane + 32 * d) : 0.f;
    }
#pragma unroll
    for (int d = 0; d < DPL; ++d) {
      if (!split) static_cast<Q*>(p.out)[head + lane + 32 * d] = Elem<Q>::from_f(rl == 0.f ? 0.f : acc[d] / rl);
      else part[(size_t)r * (HD + 4) + lane + 32 * d] = acc[d];
    }
    if (split && lane == 0) *reinterpret_cast<float2*>(part + (size_t)r * (HD + 4) + HD) = make_float2(rm, rl);
  }
}

}  // namespace kve

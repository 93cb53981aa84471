// Attention of drafted trees (or chains, or single tokens) over a paged cache
// that holds bf16, fp32 or e4m3 rows.
//
//   o_i = sum_j p_ij v_j,  p_ij = e^(scale q_i.k_j) / sum_j e^(scale q_i.k_j)
//
// over the keys j that row i sees: all of the history [0, ctx - q_len) and, of
// the q_len new tokens (the nodes of the tree, in the cache behind the history),
// those whose bit is set in the row's mask words (without a mask: itself and the
// ones before it). A row that sees nothing gets zeros.
//
// Three kernels, by what bounds them:
//   tree_attn_small.cu  up to 8 rows (nodes x heads of a kv head): the cache's bytes
//   tree_attn_tc.cu     more: the tensor cores (tcgen05)
//   this file           fp32, and what those two cannot load by TMA (bf16 and few-row e4m3 caches with
//                       blocks that are no multiple of 16)
//
// The work is one pass over the keys with a running maximum and sum. A CTA takes
// one (sequence x kv head), a tile of up to 64 query rows (row = node x group
// head) and a chunk of the keys; its four warps are RB row blocks of 16 rows
// times KS = 4 / RB key streams. Key tile t (16 keys) of the chunk belongs to
// stream t mod KS, and each stream has its own ring of tiles in shared memory
// that its warps fill with 16-byte cp.async, so any block size and any head
// stride works and no warp waits for another stream.
//
// The products run on the tensor cores:
//   bf16  m16n8k16 on bf16. P is rounded to bf16 for P V (its sum is not).
//   e4m3  the cache holds x = q 2^e with one exponent e per (slot, kv head). Q K^T
//         runs in f16: e4m3 numbers are f16 numbers, and q is multiplied by a power
//         of two that puts the row's largest element in [2^7, 2^8) (bf16 has fewer
//         bits than f16, so only elements 2^-22 of the largest lose any). The keys'
//         2^e multiplies the scores. P V runs in bf16, which has fp32's range:
//         p 2^e is rounded as p would be, whatever the spread of the exponents.
//   fp32  m16n8k8 on tf32 with both operands split in two, x = hi + lo, and
//         hi hi + hi lo + lo hi summed: the terms left out are 2^-22 of the product. Rows with
//         infinities among their operands are computed again, key by key.
// Scores, maxima, sums and outputs are fp32 throughout.
//
// Measured: fp32, 14 / 2 heads of 64, one tree of 9 nodes behind 131 keys, 9.2 us (27 us before row
// blocks shrank to spread a small grid): latency, one tile a warp in 24 CTAs (lengths, table, tile, products one after
// the other), the merge of the warps and then of three chunks through memory. 64 trees of 16 nodes, 16 / 2 heads
// of 128, 175 to 700 keys, 322 us: one CTA an SM, three products and the splitting of K and V for every element.
#include <cuda_fp8.h>
#include <math.h>

#include <atomic>
#include <type_traits>

#include "kve_common.cuh"
#include "tree_attn.cuh"

namespace kve {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTile = 16;       // keys per tile
constexpr int kMaxGroup = 64;
constexpr int kMaxNodes = 1024;

enum { kBf16 = 0, kFp8 = 1, kF32 = 2 };

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
// Two e4m3 bytes (the low 16 bits) as f16x2, and as bf16x2; both exact.
__device__ __forceinline__ uint32_t e4m3_to_f16x2(uint32_t two) {
  __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
  return (uint32_t)h.x | (uint32_t)h.y << 16;
}
__device__ __forceinline__ uint32_t e4m3_to_bf16x2(uint32_t two) {
  __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
  const float2 f = __half22float2(__half2(h));
  return bf16x2(f.x, f.y);
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t tf32(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return r;
}
// x = hi + lo + what is below 2^-22 |x|.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
  hi = tf32(x);
  lo = tf32(x - __uint_as_float(hi));
}
__device__ __forceinline__ void ldsm(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t addr, uint32_t& r0, uint32_t& r1, uint32_t& r2, uint32_t& r3) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r0), "=r"(r1), "=r"(r2), "=r"(r3) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// Whether a word of cache contents holds an infinity or a NaN.
template <int KV>
__device__ __forceinline__ bool not_finite(uint32_t w) {
  if constexpr (KV == kF32) return (w & 0x7f800000u) == 0x7f800000u;
  if constexpr (KV == kBf16) return (w & 0x7f800000u) == 0x7f800000u || (w & 0x7f80u) == 0x7f80u;
  return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0u;
}
// One element of a cache row in shared memory.
template <int KV>
__device__ __forceinline__ float cache_value(uint32_t addr) {
  const uint32_t w = lds32(addr & ~3u), at = (addr & 3u) * 8;
  if constexpr (KV == kF32) return __uint_as_float(w);
  if constexpr (KV == kBf16) return __uint_as_float(w >> at << 16);
  return __half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)(w >> at & 255u), __NV_E4M3)));
}

// Geometry of one instantiation.
template <int KV, int HD, int RB>
struct Shape {
  static constexpr int KS = kWarps / RB;                               // key streams
  static constexpr int ELEM = KV == kF32 ? 4 : KV == kBf16 ? 2 : 1;     // cache bytes per element
  static constexpr int ROWB = HD * ELEM;                               // bytes of one key row
  static constexpr int CH = ROWB / 16;                                 // 16-byte pieces of it
  static constexpr int PAIR = 2 * kTile * ROWB;                        // K and V of one tile
  static constexpr int RING = KV == kF32 && HD == 128 ? (RB == 1 ? 196608 : 131072) : 98304;  // bytes of all rings
  static constexpr int NST = RING / (KS * PAIR) < 12 ? RING / (KS * PAIR) : 12;  // tiles of a ring
  static constexpr int RINGS = KS * NST * PAIR;
  static constexpr int XROW = HD + 4;                                  // floats of a row of the merge area
  static constexpr int MERGE = KS * RB * 16 * (XROW + 2) * 4;
  static constexpr int AREA = RINGS > MERGE ? RINGS : MERGE;
  static constexpr int SCALES = KV == kFp8 ? KS * NST * 64 * 4 : 0;    // per tile: 32 words and 32 shifts
  static constexpr int QROW = HD + 4;                                  // fp32: floats of a row of split q
  static constexpr int QSM = KV == kF32 ? RB * 16 * QROW * 2 * 4 : 0;
  static_assert(NST >= 3 && CH >= 4, "ring too short");
  static_assert(AREA + SCALES + QSM <= 232448, "more shared memory than a CTA has");
};
template <int KV, int HD, int RB>
constexpr size_t smem_bytes() {
  using S = Shape<KV, HD, RB>;
  return (size_t)S::AREA + S::SCALES + S::QSM;
}

// Swizzle of the 16-byte pieces of a key row, so that both the matrix loads (8
// keys at one piece) and the 128-bit loads (2 keys x 4 pieces in a phase) touch
// every bank once: rows of 128 bytes and more exchange their pieces by the key's
// three low bits, reversed; 64-byte rows lie two to a 128-byte line.
template <int KV, int CH>
__device__ __forceinline__ int swz(int key, int piece) {
  if constexpr (CH == 4) return piece ^ ((key >> 1) & 3);
  if constexpr (KV == kF32) return piece ^ ((key & 2) | (((key >> 2) ^ key) & 1) << 2);
  return piece ^ ((key & 1) << 2 | (key & 2) | (key >> 2 & 1));
}

template <int KV, int HD, int RB>
__global__ void __launch_bounds__(kThreads, (KV == kF32 && HD == 128) ? 1 : 2)
tree_attn_kernel(TreeParams p) {
  grid_dep_wait();
  grid_dep_launch();
  using S = Shape<KV, HD, RB>;
  constexpr int KS = S::KS, NST = S::NST, CH = S::CH, ROWB = S::ROWB;
  using QT = typename std::conditional<KV == kF32, float, __nv_bfloat16>::type;
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* scales = smem + S::AREA;
  float* qsm = reinterpret_cast<float*>(scales + S::SCALES);

  const int bh = blockIdx.x, c = blockIdx.y, qtile = blockIdx.z;
  const int b = bh / p.nkv, h = bh % p.nkv;
  const int ctx = p.ctx_lens[b], ql = p.q_lens[b], qoff = p.q_offsets[b];
  if (ql < 0 || ql > p.max_q || ctx < ql || qoff < 0 || qoff > p.q_rows - ql || (int64_t)ctx > (int64_t)p.table_stride * p.bs ||
      (int64_t)ctx > (int64_t)p.chunk * p.n_chunks) {
    if (threadIdx.x == 0 && c == 0 && qtile == 0) report(p.status, KVE_ERR_BOUNDS);
    return;
  }
  const int row0 = qtile * RB * 16;
  const int rows = min(RB * 16, ql * p.group - row0);
  if (rows <= 0) return;
  const int hist = ctx - ql;
  // Keys any row of this tile sees: all of them under a mask, else up to its last node.
  const int key_end = p.mask ? ctx : hist + (row0 + rows - 1) / p.group + 1;
  const int live = (key_end + p.chunk - 1) / p.chunk;  // chunks this tile is split into
  if (c >= live) return;
  const int key_lo = c * p.chunk;
  const int key_hi = min(key_end, key_lo + p.chunk);
  const int n_tiles = (key_hi - key_lo + kTile - 1) / kTile;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rb = warp % RB, ks = warp / RB;
  const int g = lane >> 2, tq = lane & 3;

  // Query rows of this warp: g and g + 8 of its row block.
  const QT* q = static_cast<const QT*>(p.q);
  const int r_lo = rb * 16 + g, r_hi = r_lo + 8;
  const int n_lo = node_of(p, row0 + r_lo), n_hi = node_of(p, row0 + r_hi);
  auto q_row = [&](int r) {
    const int gr = row0 + r, node = node_of(p, gr);
    return q + ((size_t)(qoff + node) * p.nq + h * p.group + gr - node * p.group) * HD;
  };
  constexpr int KSTEPS = HD / 16;
  uint32_t qa[KV == kF32 ? 1 : KSTEPS][4];
  float sl_lo = p.scale * 1.4426950408889634f, sl_hi = sl_lo;  // scores in log2 units
  if constexpr (KV == kBf16) {
    const uint32_t* q_lo = r_lo < rows ? reinterpret_cast<const uint32_t*>(q_row(r_lo)) : nullptr;
    const uint32_t* q_hi = r_hi < rows ? reinterpret_cast<const uint32_t*>(q_row(r_hi)) : nullptr;
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk) {
      qa[kk][0] = q_lo ? q_lo[kk * 8 + tq] : 0u;
      qa[kk][1] = q_hi ? q_hi[kk * 8 + tq] : 0u;
      qa[kk][2] = q_lo ? q_lo[kk * 8 + tq + 4] : 0u;
      qa[kk][3] = q_hi ? q_hi[kk * 8 + tq + 4] : 0u;
    }
  } else if constexpr (KV == kFp8) {
    // Step kk covers, for this lane, dims 64 (kk / 4) + 16 tq + 4 (kk % 4) .. + 3: the
    // order in which a 128-bit load brings a key's e4m3 bytes.
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int r = half ? r_hi : r_lo;
      const uint2* src = r < rows ? reinterpret_cast<const uint2*>(q_row(r)) : nullptr;
      uint2 raw[KSTEPS];
      float top = 0.f;
#pragma unroll
      for (int kk = 0; kk < KSTEPS; ++kk) {
        raw[kk] = src ? src[(kk / 4) * 16 + tq * 4 + kk % 4] : make_uint2(0u, 0u);
        const float2 x = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&raw[kk].x));
        const float2 y = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&raw[kk].y));
        top = fmaxf(top, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(y.x), fabsf(y.y))));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // up = 2^(7 - exponent of the largest), kept between 2^-112 and 2^126
      const int ex = min(max((int)(__float_as_uint(top) >> 23), 8), 246);
      const float up = __uint_as_float((uint32_t)(261 - ex) << 23);
      if (half) sl_hi *= 1.f / up;
      else sl_lo *= 1.f / up;
#pragma unroll
      for (int kk = 0; kk < KSTEPS; ++kk) {
        const float2 x = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&raw[kk].x));
        const float2 y = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&raw[kk].y));
        qa[kk][half] = f16x2(x.x * up, x.y * up);
        qa[kk][2 + half] = f16x2(y.x * up, y.y * up);
      }
    }
  } else {
    // Split once, kept in shared memory: [hi, lo][row][dim].
    for (int i = threadIdx.x; i < RB * 16 * (HD / 4); i += kThreads) {
      const int r = i / (HD / 4), d = i % (HD / 4) * 4;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < rows) x = *reinterpret_cast<const float4*>(q_row(r) + d);
      uint4 hi, lo;
      split_tf32(x.x, hi.x, lo.x);
      split_tf32(x.y, hi.y, lo.y);
      split_tf32(x.z, hi.z, lo.z);
      split_tf32(x.w, hi.w, lo.w);
      *reinterpret_cast<uint4*>(qsm + r * S::QROW + d) = hi;
      *reinterpret_cast<uint4*>(qsm + (RB * 16 + r) * S::QROW + d) = lo;
    }
  }
  __syncthreads();

  // Ring of this stream. Tile i of the stream is tile ks + KS i of the chunk; its
  // RB warps copy a part each. One commit group per tile (empty past the end).
  const int32_t* table = p.tables + (size_t)b * p.table_stride;
  const uint32_t ring = smem_addr(smem) + ks * NST * S::PAIR;
  const uint32_t sring = smem_addr(scales) + ks * NST * 256;
  const size_t key_stride = (size_t)p.nkv * ROWB;
  const uint8_t* base_k = static_cast<const uint8_t*>(p.pool_k) + (size_t)h * ROWB;
  const uint8_t* base_v = static_cast<const uint8_t*>(p.pool_v) + (size_t)h * ROWB;
  const int my_tiles = n_tiles > ks ? (n_tiles - ks + KS - 1) / KS : 0;
  // The flat slot of key (lane mod 16) of tile i, -1 past the end. The table entry is
  // read a tile ahead of the copy that needs it.
  auto key_of = [&](int i) { return key_lo + (ks + KS * i) * kTile + (lane & 15); };
  auto block_of = [&](int i) {
    const int key = key_of(i);
    return i < my_tiles && key < key_hi ? table[key / p.bs] : 0;
  };
  auto load_tile = [&](int i, int block) {
    if (i < my_tiles) {
      const int st = i % NST;
      const int key = key_of(i);
      int64_t slot = -1;
      if (key < key_hi) {
        if (block >= 0 && block < p.num_blocks) slot = (int64_t)block * p.bs + key % p.bs;
        else report(p.status, KVE_ERR_BOUNDS);  // reads as zeros
      }
      if constexpr (KV == kFp8) {
        // the aligned word that holds the key's scale byte (lanes 16.. : V's) up to that byte, and the byte's
        // place; where the scales begin inside that word, the byte alone
        if (rb == 0) {
          const uint8_t* all = lane < 16 ? p.k_scale : p.v_scale;
          const uint8_t* s = all + (slot < 0 ? 0 : slot * p.nkv + h);
          const uint32_t at = (uint32_t)(reinterpret_cast<uintptr_t>(s) & 3u), to = sring + st * 256 + lane * 4;
          if (slot >= 0 && (size_t)(s - all) < at)
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(to), "r"((uint32_t)*s << at * 8) : "memory");
          else
            cp4(to, s - at, slot < 0 ? 0u : at + 1);
          asm volatile("st.shared.u32 [%0], %1;" ::"r"(to + 128), "r"(at * 8) : "memory");
        }
      }
      constexpr int PIECES = 2 * kTile * CH;  // K then V
      constexpr int PER = PIECES / (RB * 32);
      const uint32_t dst = ring + st * S::PAIR;
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        const int i2 = (u * RB + rb) * 32 + lane;
        const bool is_v = i2 >= kTile * CH;  // the same for all lanes of the warp
        const int j = is_v ? i2 - kTile * CH : i2;
        const int kk = j / CH, piece = j % CH;
        const int64_t sl = __shfl_sync(0xffffffffu, slot, kk);
        const uint8_t* src = (is_v ? base_v : base_k) + (sl < 0 ? 0 : (size_t)sl * key_stride) + piece * 16;
        cp16(dst + (is_v ? kTile * ROWB : 0) + kk * ROWB + swz<KV, CH>(kk, piece) * 16, src, sl < 0 ? 0u : 16u);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto stream_sync = [&]() {
    if constexpr (RB == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(ks + 1), "n"(RB * 32) : "memory");
  };

  float m_lo = -INFINITY, m_hi = -INFINITY, l_lo = 0.f, l_hi = 0.f;  // l: this lane's share of the sum
  constexpr int DT = HD / 8;
  float acc[DT][4];
#pragma unroll
  for (int j = 0; j < DT; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
  const bool active = rb * 16 < rows;
  const uint32_t* mask_lo = nullptr;
  const uint32_t* mask_hi = nullptr;
  if (p.mask) {
    mask_lo = p.mask + (size_t)(qoff + (r_lo < rows ? n_lo : 0)) * p.mask_words;
    mask_hi = p.mask + (size_t)(qoff + (r_hi < rows ? n_hi : 0)) * p.mask_words;
  }

  int block = 0;  // the table entry of tile i + NST - 1
  {
    int first[NST];
#pragma unroll
    for (int i = 0; i < NST; ++i) first[i] = block_of(i);
#pragma unroll
    for (int i = 0; i < NST - 1; ++i) load_tile(i, first[i]);
    block = first[NST - 1];
  }
  for (int i = 0; i < my_tiles; ++i) {
    asm volatile("cp.async.wait_group %0;" ::"n"(NST - 2) : "memory");
    stream_sync();  // tile i is there, and every warp of the stream is done with tile i - 1
    load_tile(i + NST - 1, block);
    block = block_of(i + NST);
    if (!active) continue;
    const int kt = key_lo + (ks + KS * i) * kTile;
    const int st = i % NST;
    const uint32_t kb = ring + st * S::PAIR, vb = kb + kTile * ROWB;

    // S = Q K^T: sc[j][..] holds keys kt + 8 j + 2 tq, + 1 of rows g (0, 1) and g + 8 (2, 3).
    float sc[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j) sc[j][0] = sc[j][1] = sc[j][2] = sc[j][3] = 0.f;
    float vs[2][2];  // e4m3: 2^e of V's row, by key
    if constexpr (KV == kBf16) {
      const int mat = lane >> 3, rr = lane & 7;
      const int key = ((mat >> 1) << 3) + rr;
#pragma unroll
      for (int kk = 0; kk < KSTEPS; ++kk) {
        uint32_t b0, b1, b2, b3;
        ldsm(kb + key * ROWB + swz<KV, CH>(key, kk * 2 + (mat & 1)) * 16, b0, b1, b2, b3);
        mma_bf16(sc[0], qa[kk], b0, b1);
        mma_bf16(sc[1], qa[kk], b2, b3);
      }
    } else if constexpr (KV == kFp8) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int key = 8 * j + g;
#pragma unroll
        for (int dg = 0; dg < HD / 64; ++dg) {
          const uint4 x = lds128(kb + key * ROWB + swz<KV, CH>(key, dg * 4 + tq) * 16);
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int s = 0; s < 4; ++s)
            mma_f16(sc[j], qa[dg * 4 + s], e4m3_to_f16x2(w[s] & 0xffffu), e4m3_to_f16x2(w[s] >> 16));
        }
      }
      const uint32_t word = lds32(sring + st * 256 + lane * 4), at = lds32(sring + st * 256 + 128 + lane * 4);
      const float mine = scale_value(word >> at & 255u);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float k2 = __shfl_sync(0xffffffffu, mine, 8 * j + 2 * tq + e);
          vs[j][e] = __shfl_sync(0xffffffffu, mine, 16 + 8 * j + 2 * tq + e);
          sc[j][e] *= k2;
          sc[j][2 + e] *= k2;
        }
    } else {
      // The tensor cores truncate what they add up: every 16 dims start from zero and are added
      // here, rounded, and the products with a low half have sums of their own (one running sum
      // for all was off by 1.3e-6 of the output at 131 keys, these by 1.9e-7).
      float low[2][4] = {};
#pragma unroll
      for (int k16 = 0; k16 < HD / 16; ++k16) {
        // dims 16 k16 + 4 tq .. + 3 of this lane: step s takes 2 s and 2 s + 1 of them
        uint4 qh[2], qlo[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const float* src = qsm + (rb * 16 + g + 8 * half) * S::QROW + k16 * 16 + tq * 4;
          qh[half] = *reinterpret_cast<const uint4*>(src);
          qlo[half] = *reinterpret_cast<const uint4*>(src + RB * 16 * S::QROW);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const int key = 8 * j + g;
          const uint4 x = lds128(kb + key * ROWB + swz<KV, CH>(key, k16 * 4 + tq) * 16);
          uint32_t kh[4], kl[4];
          split_tf32(__uint_as_float(x.x), kh[0], kl[0]);
          split_tf32(__uint_as_float(x.y), kh[1], kl[1]);
          split_tf32(__uint_as_float(x.z), kh[2], kl[2]);
          split_tf32(__uint_as_float(x.w), kh[3], kl[3]);
          float part[4] = {};
#pragma unroll
          for (int s = 0; s < 2; ++s) {
            const uint32_t ah[4] = {s ? qh[0].z : qh[0].x, s ? qh[1].z : qh[1].x, s ? qh[0].w : qh[0].y,
                                    s ? qh[1].w : qh[1].y};
            const uint32_t al[4] = {s ? qlo[0].z : qlo[0].x, s ? qlo[1].z : qlo[1].x, s ? qlo[0].w : qlo[0].y,
                                    s ? qlo[1].w : qlo[1].y};
            mma_tf32(low[j], al, kh[2 * s], kh[2 * s + 1]);
            mma_tf32(low[j], ah, kl[2 * s], kl[2 * s + 1]);
            mma_tf32(part, ah, kh[2 * s], kh[2 * s + 1]);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[j][e] += part[e];
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[j][e] += low[j][e];
    }

    // Which of the tile's keys the two rows see.
    const bool masked = kt + kTile > hist || kt + kTile > key_hi;
    uint32_t see_lo = 0xffffu, see_hi = 0xffffu;
    if (masked) {
      const int j0 = kt - hist;
      see_lo = p.mask ? mask_bits<kTile>(mask_lo, p.mask_words, j0) : chain_bits(n_lo, j0);
      see_hi = p.mask ? mask_bits<kTile>(mask_hi, p.mask_words, j0) : chain_bits(n_hi, j0);
      const uint32_t inside = key_hi - kt >= kTile ? 0xffffu : (1u << (key_hi - kt)) - 1u;
      see_lo &= inside;
      see_hi &= inside;
    }

    // Running maximum and sum.
    float mx_lo = -INFINITY, mx_hi = -INFINITY;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int x = 8 * j + 2 * tq + e;
        sc[j][e] = see_lo >> x & 1 ? sc[j][e] * sl_lo : -INFINITY;
        sc[j][2 + e] = see_hi >> x & 1 ? sc[j][2 + e] * sl_hi : -INFINITY;
        mx_lo = fmaxf(mx_lo, sc[j][e]);
        mx_hi = fmaxf(mx_hi, sc[j][2 + e]);
      }
    mx_lo = fmaxf(mx_lo, __shfl_xor_sync(0xffffffffu, mx_lo, 1));
    mx_hi = fmaxf(mx_hi, __shfl_xor_sync(0xffffffffu, mx_hi, 1));
    mx_lo = fmaxf(mx_lo, __shfl_xor_sync(0xffffffffu, mx_lo, 2));
    mx_hi = fmaxf(mx_hi, __shfl_xor_sync(0xffffffffu, mx_hi, 2));
    if (__any_sync(0xffffffffu, mx_lo > m_lo || mx_hi > m_hi)) {
      const float t_lo = fmaxf(m_lo, mx_lo), t_hi = fmaxf(m_hi, mx_hi);
      const float f_lo = t_lo == m_lo ? 1.f : ex2(m_lo - t_lo), f_hi = t_hi == m_hi ? 1.f : ex2(m_hi - t_hi);
      m_lo = t_lo;
      m_hi = t_hi;
      l_lo *= f_lo;
      l_hi *= f_hi;
#pragma unroll
      for (int j = 0; j < DT; ++j) {
        acc[j][0] *= f_lo;
        acc[j][1] *= f_lo;
        acc[j][2] *= f_hi;
        acc[j][3] *= f_hi;
      }
    }
    // A row that has seen nothing yet has m = -inf: its p are zeros, whatever the base.
    const float b_lo = m_lo == -INFINITY ? 0.f : m_lo, b_hi = m_hi == -INFINITY ? 0.f : m_hi;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        sc[j][e] = ex2(sc[j][e] - b_lo);
        sc[j][2 + e] = ex2(sc[j][2 + e] - b_hi);
        l_lo += sc[j][e];
        l_hi += sc[j][2 + e];
      }

    // O += P V. A new token's V may hold infinities or NaN where only some rows see it: in
    // the products their zeros would spread it to the others, so such a tile is summed key
    // by key over the rows that see it.
    bool odd = false;
    if (masked && kt + kTile > hist) {
      for (int i2 = lane; i2 < kTile * CH; i2 += 32) {
        const uint4 x = lds128(vb + i2 * 16);
        odd |= not_finite<KV>(x.x) || not_finite<KV>(x.y) || not_finite<KV>(x.z) || not_finite<KV>(x.w);
      }
      if constexpr (KV == kFp8) odd |= !(vs[0][0] < INFINITY && vs[0][1] < INFINITY && vs[1][0] < INFINITY && vs[1][1] < INFINITY);
      odd = __any_sync(0xffffffffu, odd);
    }
    if (odd) {
      for (int x = 0; x < kTile; ++x) {
        const int j = x >> 3, e = x & 1, from = (lane & 28) | (x >> 1 & 3);
        const float p_lo = __shfl_sync(0xffffffffu, j ? (e ? sc[1][1] : sc[1][0]) : (e ? sc[0][1] : sc[0][0]), from);
        const float p_hi = __shfl_sync(0xffffffffu, j ? (e ? sc[1][3] : sc[1][2]) : (e ? sc[0][3] : sc[0][2]), from);
        float unit = 1.f;
        if constexpr (KV == kFp8)
          unit = __shfl_sync(0xffffffffu, j ? (e ? vs[1][1] : vs[1][0]) : (e ? vs[0][1] : vs[0][0]), from);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const int dim = KV == kFp8 ? (d >> 1) * 16 + tq * 4 + 2 * y + (d & 1) : d * 8 + tq * 2 + y;
            const float v = unit * cache_value<KV>(vb + x * ROWB + swz<KV, CH>(x, dim * S::ELEM / 16) * 16 + dim * S::ELEM % 16);
            if (see_lo >> x & 1) acc[d][y] += p_lo * v;
            if (see_hi >> x & 1) acc[d][2 + y] += p_hi * v;
          }
      }
    } else if constexpr (KV == kF32) {
      // k8 step j: lane position tq stands for key 2 tq, tq + 4 for key 2 tq + 1
      uint32_t ph[2][4], pl[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        split_tf32(sc[j][0], ph[j][0], pl[j][0]);
        split_tf32(sc[j][2], ph[j][1], pl[j][1]);
        split_tf32(sc[j][1], ph[j][2], pl[j][2]);
        split_tf32(sc[j][3], ph[j][3], pl[j][3]);
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        const int piece = d * 2 + (g >> 2);
        uint32_t vh[2][2], vl[2][2];
        float part[4] = {};  // the tile's sum, added to the others rounded
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int key = 8 * j + 2 * tq + e;
            split_tf32(__uint_as_float(lds32(vb + key * ROWB + swz<KV, CH>(key, piece) * 16 + (g & 3) * 4)), vh[j][e], vl[j][e]);
          }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          mma_tf32(part, pl[j], vh[j][0], vh[j][1]);
          mma_tf32(part, ph[j], vl[j][0], vl[j][1]);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) mma_tf32(part, ph[j], vh[j][0], vh[j][1]);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[d][e] += part[e];
      }
    } else {
      uint32_t pa[4];
      if constexpr (KV == kFp8) {
        // a key no row may see contributes exactly 0 whatever its scale byte
        pa[0] = bf16x2(sc[0][0] == 0.f ? 0.f : sc[0][0] * vs[0][0], sc[0][1] == 0.f ? 0.f : sc[0][1] * vs[0][1]);
        pa[1] = bf16x2(sc[0][2] == 0.f ? 0.f : sc[0][2] * vs[0][0], sc[0][3] == 0.f ? 0.f : sc[0][3] * vs[0][1]);
        pa[2] = bf16x2(sc[1][0] == 0.f ? 0.f : sc[1][0] * vs[1][0], sc[1][1] == 0.f ? 0.f : sc[1][1] * vs[1][1]);
        pa[3] = bf16x2(sc[1][2] == 0.f ? 0.f : sc[1][2] * vs[1][0], sc[1][3] == 0.f ? 0.f : sc[1][3] * vs[1][1]);
      } else {
        pa[0] = bf16x2(sc[0][0], sc[0][1]);
        pa[1] = bf16x2(sc[0][2], sc[0][3]);
        pa[2] = bf16x2(sc[1][0], sc[1][1]);
        pa[3] = bf16x2(sc[1][2], sc[1][3]);
      }
      const int mat = lane >> 3, rr = lane & 7;
      const int key = ((mat & 1) << 3) + rr;
      const uint32_t vrow = vb + key * ROWB;
      if constexpr (KV == kBf16) {
#pragma unroll
        for (int d = 0; d < DT; d += 2) {
          uint32_t b0, b1, b2, b3;
          ldsm_t(vrow + swz<KV, CH>(key, d + (mat >> 1)) * 16, b0, b1, b2, b3);
          mma_bf16(acc[d], pa, b0, b1);
          mma_bf16(acc[d + 1], pa, b2, b3);
        }
      } else {
        // A piece holds 16 dims as 8 byte pairs: the transposed load gives lane (g, tq) the
        // pair of dims 2 g, 2 g + 1 of keys 2 tq and 2 tq + 1. Even dims go to tile 2 ch, odd ones to 2 ch + 1.
#pragma unroll
        for (int ch = 0; ch < CH; ch += 2) {
          uint32_t r[4];
          ldsm_t(vrow + swz<KV, CH>(key, ch + (mat >> 1)) * 16, r[0], r[1], r[2], r[3]);
#pragma unroll
          for (int x = 0; x < 4; ++x) r[x] = __byte_perm(r[x], 0u, 0x3120);
#pragma unroll
          for (int x = 0; x < 2; ++x) {
            mma_bf16(acc[2 * (ch + x)], pa, e4m3_to_bf16x2(r[2 * x] & 0xffffu), e4m3_to_bf16x2(r[2 * x + 1] & 0xffffu));
            mma_bf16(acc[2 * (ch + x) + 1], pa, e4m3_to_bf16x2(r[2 * x] >> 16), e4m3_to_bf16x2(r[2 * x + 1] >> 16));
          }
        }
      }
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  l_lo += __shfl_xor_sync(0xffffffffu, l_lo, 1);
  l_hi += __shfl_xor_sync(0xffffffffu, l_hi, 1);
  l_lo += __shfl_xor_sync(0xffffffffu, l_lo, 2);
  l_hi += __shfl_xor_sync(0xffffffffu, l_hi, 2);

  // The streams' states meet in shared memory (the rings are free now).
  __syncthreads();
  float* xs = reinterpret_cast<float*>(smem);               // [stream][row][XROW]
  float* xm = xs + KS * RB * 16 * S::XROW;                  // [stream][row][m, l]
  {
    float* lo = xs + (size_t)(ks * RB * 16 + r_lo) * S::XROW;
    float* hi = lo + 8 * S::XROW;
    if constexpr (KV == kFp8) {
#pragma unroll
      for (int ch = 0; ch < CH; ++ch) {
        const float(&e)[4] = acc[2 * ch];
        const float(&o)[4] = acc[2 * ch + 1];
        *reinterpret_cast<float4*>(lo + ch * 16 + tq * 4) = make_float4(e[0], o[0], e[1], o[1]);
        *reinterpret_cast<float4*>(hi + ch * 16 + tq * 4) = make_float4(e[2], o[2], e[3], o[3]);
      }
    } else {
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        *reinterpret_cast<float2*>(lo + d * 8 + tq * 2) = make_float2(acc[d][0], acc[d][1]);
        *reinterpret_cast<float2*>(hi + d * 8 + tq * 2) = make_float2(acc[d][2], acc[d][3]);
      }
    }
    if (tq == 0) {
      float* ml = xm + (ks * RB * 16 + r_lo) * 2;
      ml[0] = m_lo;
      ml[1] = l_lo;
      ml[16] = m_hi;
      ml[17] = l_hi;
    }
  }
  __syncthreads();

  QT* out = static_cast<QT*>(p.out);
  auto store4 = [&](int r, int d, float4 o, float l) {
    // l == 0: the row sees no key
    o.x = l == 0.f ? 0.f : o.x / l;
    o.y = l == 0.f ? 0.f : o.y / l;
    o.z = l == 0.f ? 0.f : o.z / l;
    o.w = l == 0.f ? 0.f : o.w / l;
    const int gr = row0 + r, node = node_of(p, gr);
    QT* dst = out + ((size_t)(qoff + node) * p.nq + h * p.group + gr - node * p.group) * HD + d;
    if constexpr (KV == kF32) *reinterpret_cast<float4*>(dst) = o;
    else *reinterpret_cast<uint2*>(dst) = make_uint2(bf16x2(o.x, o.y), bf16x2(o.z, o.w));
  };
  // Partials of one (sequence x kv head, query tile): [chunk][row][HD + 4] (m and l behind the dims).
  constexpr int PROW = HD + 4;
  float* part0 = p.partials + ((size_t)bh * p.n_qtiles + qtile) * p.n_chunks * (RB * 16) * PROW;
  bool nan = false;
  for (int i = threadIdx.x; i < rows * (HD / 4); i += kThreads) {
    const int r = i / (HD / 4), d = i % (HD / 4) * 4;
    float m = -INFINITY;
#pragma unroll
    for (int s = 0; s < KS; ++s) m = fmaxf(m, xm[(s * RB * 16 + r) * 2]);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const float ms = xm[(s * RB * 16 + r) * 2], ls = xm[(s * RB * 16 + r) * 2 + 1];
      const float w = ms == m ? 1.f : ex2(ms - m);
      const float4 x = *reinterpret_cast<const float4*>(xs + (size_t)(s * RB * 16 + r) * S::XROW + d);
      l += ls * w;
      o.x += x.x * w;
      o.y += x.y * w;
      o.z += x.z * w;
      o.w += x.w * w;
    }
    if constexpr (KV == kF32) {
      const float sum = o.x + o.y + o.z + o.w + l;
      nan |= !(fabsf(sum) < INFINITY);
    }
    if (live == 1) {
      store4(r, d, o, l);
    } else {
      float* pr = part0 + ((size_t)c * (RB * 16) + r) * PROW;
      *reinterpret_cast<float4*>(pr + d) = o;
      if (d == 0) *reinterpret_cast<float2*>(pr + HD) = make_float2(m, l);
    }
  }
  // An infinity or a number next to the largest has no two halves (infinity minus infinity): rows that
  // came out as not finite are computed again without them.
  if (KV == kF32 && __syncthreads_or(nan))
    attend_by_key<QT, false, HD, kThreads>(p, b, h, qoff, hist, key_lo, key_hi, row0, rows, warp, lane, live > 1,
                                           part0 + (size_t)c * (RB * 16) * PROW);
  if (live == 1) return;

  // The last of the tile's chunks to arrive joins them, in chunk order.
  __shared__ int last;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    int* cnt = p.counters + (size_t)bh * p.n_qtiles + qtile;
    last = atomicAdd(cnt, 1) == live - 1;
    if (last) *cnt = 0;  // the workspace is left as it was
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  for (int i = threadIdx.x; i < rows * (HD / 4); i += kThreads) {
    const int r = i / (HD / 4), d = i % (HD / 4) * 4;
    const float* pr = part0 + (size_t)r * PROW;
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < live; ++s) {
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(pr + (size_t)s * (RB * 16) * PROW + HD));
      const float4 x = __ldcg(reinterpret_cast<const float4*>(pr + (size_t)s * (RB * 16) * PROW + d));
      const float t = fmaxf(m, ml.x);
      const float f = t == m ? 1.f : ex2(m - t), w = t == ml.x ? 1.f : ex2(ml.x - t);
      m = t;
      l = l * f + ml.y * w;
      o.x = o.x * f + x.x * w;
      o.y = o.y * f + x.y * w;
      o.z = o.z * f + x.z * w;
      o.w = o.w * f + x.w * w;
    }
    store4(r, d, o, l);
  }
}

// ------------------------------------------------------------------ host
struct Split {
  int rb, n_qtiles, chunk, n_chunks;
};

// Row blocks of 16 query rows in a CTA from the rows of the call's largest tree, fewer where the
// grid would leave SMs idle (each key then passes through more CTAs, from L2, and more streams of keys
// run side by side). Chunks: as many CTAs as fill the SMs about four times over, none under 128 keys
// (64 in a grid of under one CTA an SM), below which a chunk's fixed costs outweigh its keys. Only
// grids of fewer tiles than that are split, so the counters always suffice.
Split split_of(int batch, int max_q, int max_ctx, int nkv, int group) {
  const long long rows = (long long)max_q * group, seqs = (long long)batch * nkv;
  Split s;
  s.rb = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
  auto tiles = [&](int rb) { return seqs * ((rows + rb * 16 - 1) / (rb * 16)); };
  while (s.rb > 1 && tiles(s.rb) * ((max_ctx + 127) / 128) < 148) s.rb /= 2;
  const long long units = tiles(s.rb);
  s.n_qtiles = (int)((rows + s.rb * 16 - 1) / (s.rb * 16));
  const long long least = units * ((max_ctx + 127) / 128) < 148 ? 64 : 128;
  const long long chunks = (4 * 2 * 148 + units - 1) / units;
  long long chunk = ((long long)max_ctx + chunks - 1) / chunks;
  chunk = (chunk + 63) / 64 * 64;
  chunk = chunk < least ? least : chunk;
  s.chunk = (int)chunk;
  s.n_chunks = (int)((max_ctx + chunk - 1) / chunk);
  if (s.n_chunks < 1) s.n_chunks = 1;
  return s;
}
size_t partial_bytes(const Split& s, int batch, int nkv, int hd) {
  if (s.n_chunks == 1) return 0;
  return (size_t)batch * nkv * s.n_qtiles * s.n_chunks * (s.rb * 16) * (hd + 4) * sizeof(float);
}

// More than the few-row kernel's eight rows go to the wide kernel, although its tile is 128 rows: 24 rows
// (64 sequences of up to 700 keys) took it 13.2 us against 25.8 here, 16 rows (16 sequences, 8 kv heads,
// 3000 keys) 32.9 against 42.2, one sequence of 32 rows 9.4 against 10.1.
bool use_wide(int max_q, int group) { return (long long)max_q * group > 8; }

template <int KV, int HD, int RB>
int launch(const TreeParams& p, int batch, cudaStream_t stream) {
  // the shared-memory limit is an attribute of the kernel on one device
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (err == cudaSuccess && !(ready.load(std::memory_order_relaxed) & bit)) {
    err = cudaFuncSetAttribute(tree_attn_kernel<KV, HD, RB>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (int)smem_bytes<KV, HD, RB>());
    if (err == cudaSuccess) ready.fetch_or(bit, std::memory_order_relaxed);
  }
  if (err != cudaSuccess) {
    cudaGetLastError();
    return set_error(KVE_ERR_CUDA, "kve_paged_tree_attn: %s", cudaGetErrorString(err));
  }
  launch_kernel(tree_attn_kernel<KV, HD, RB>, dim3(batch * p.nkv, p.n_chunks, p.n_qtiles), dim3(kThreads),
                (smem_bytes<KV, HD, RB>()), stream, p);
  return check_launch("kve_paged_tree_attn");
}
template <int KV, int HD>
int launch_rb(const TreeParams& p, int rb, int batch, cudaStream_t stream) {
  // e4m3 comes here with at most eight rows (and blocks that the few-row kernel does not take)
  if (KV == kFp8 || rb == 1) return launch<KV, HD, 1>(p, batch, stream);
  if constexpr (KV != kFp8) {
    if (rb == 2) return launch<KV, HD, 2>(p, batch, stream);
    return launch<KV, HD, 4>(p, batch, stream);
  }
}
template <int KV>
int launch_hd(const TreeParams& p, int hd, int rb, int batch, cudaStream_t stream) {
  return hd == 64 ? launch_rb<KV, 64>(p, rb, batch, stream) : launch_rb<KV, 128>(p, rb, batch, stream);
}

}  // namespace
}  // namespace kve

using namespace kve;

extern "C" size_t kve_tree_attn_workspace_bytes(int batch, int max_q_len, int max_ctx, int num_heads,
                                                int num_kv_heads, int head_dim) {
  if (batch < 1 || max_q_len < 1 || max_ctx < 1 || num_kv_heads < 1 || num_heads < num_kv_heads || head_dim < 1)
    return 0;
  const Split s = split_of(batch, max_q_len, max_ctx, num_kv_heads, num_heads / num_kv_heads);
  size_t n = partial_bytes(s, batch, num_kv_heads, head_dim);
  if (use_wide(max_q_len, num_heads / num_kv_heads)) {  // the call's types and block size choose the kernel
    const size_t w = tree_attn_wide_partial_bytes(batch, max_q_len, max_ctx, num_kv_heads, num_heads / num_kv_heads, head_dim);
    n = n > w ? n : w;
  }
  const size_t few = tree_attn_small_partial_bytes(batch, max_ctx, num_kv_heads, head_dim);
  n = n > few ? n : few;
  return n ? kTreeCounterBytes + n : 0;
}

extern "C" int kve_paged_tree_attn(const void* q, int dtype, const void* pool_k, const void* pool_v, int kv_dtype,
                                   const uint8_t* k_scale, const uint8_t* v_scale, const int32_t* block_tables,
                                   int table_stride, const int32_t* ctx_lens, const int32_t* q_lens,
                                   const int32_t* q_offsets, const uint32_t* tree_mask, int mask_words, int batch,
                                   int q_rows, int max_q_len, int max_ctx, int num_heads, int num_kv_heads, int head_dim,
                                   int block_size, int64_t num_blocks, float scale, void* out, void* workspace,
                                   size_t workspace_bytes, int* dev_status, cudaStream_t stream) {
  const char* me = "kve_paged_tree_attn";
  if (batch < 0 || q_rows < 0 || max_q_len < 0 || max_ctx < 0 || num_heads < 1 || num_kv_heads < 1 || num_heads % num_kv_heads ||
      block_size < 1 || table_stride < 1 || num_blocks < 1 || max_ctx < max_q_len)
    return set_error(KVE_ERR_ARG, "%s: bad sizes", me);
  if (batch == 0 || max_q_len == 0) return KVE_OK;
  if (head_dim != 64 && head_dim != 128)
    return set_error(KVE_ERR_SHAPE, "%s: head_dim %d (supported: 64, 128)", me, head_dim);
  const int group = num_heads / num_kv_heads;
  if (group > kMaxGroup) return set_error(KVE_ERR_SHAPE, "%s: group %d > %d", me, group, kMaxGroup);
  if (num_blocks > 0x7fffffffLL / block_size) return set_error(KVE_ERR_SHAPE, "%s: more than 2^31 slots", me);
  if (max_q_len > kMaxNodes) return set_error(KVE_ERR_SHAPE, "%s: max_q_len %d > %d", me, max_q_len, kMaxNodes);
  if ((long long)batch * num_kv_heads > 0x7fffffffLL) return set_error(KVE_ERR_SHAPE, "%s: batch too large", me);
  if (!isfinite(scale)) return set_error(KVE_ERR_ARG, "%s: scale %g", me, (double)scale);
  if (dtype != KVE_F32 && dtype != KVE_BF16) return set_error(KVE_ERR_DTYPE, "%s: dtype %d", me, dtype);
  if (kv_dtype != dtype && !(kv_dtype == KVE_FP8_E4M3 && dtype == KVE_BF16))
    return set_error(KVE_ERR_DTYPE, "%s: a cache of dtype %d with queries of dtype %d", me, kv_dtype, dtype);
  if (!q || !pool_k || !pool_v || !block_tables || !ctx_lens || !q_lens || !q_offsets || !out)
    return set_error(KVE_ERR_ARG, "%s: null pointer", me);
  if (kv_dtype == KVE_FP8_E4M3 && (!k_scale || !v_scale)) return set_error(KVE_ERR_ARG, "%s: null scales", me);
  if (tree_mask && mask_words < (max_q_len + 31) / 32)
    return set_error(KVE_ERR_ARG, "%s: %d mask words for %d nodes", me, mask_words, max_q_len);
  if ((uintptr_t)pool_k % 16 || (uintptr_t)pool_v % 16 || (uintptr_t)q % 16 || (uintptr_t)out % 16)
    return set_error(KVE_ERR_ARG, "%s: q, out and the pools must be 16-byte aligned", me);
  TreeParams p{};
  p.q = q; p.pool_k = pool_k; p.pool_v = pool_v; p.k_scale = k_scale; p.v_scale = v_scale;
  p.tables = block_tables; p.table_stride = table_stride;
  p.ctx_lens = ctx_lens; p.q_lens = q_lens; p.q_offsets = q_offsets;
  p.mask = tree_mask; p.mask_words = mask_words;
  p.q_rows = q_rows; p.max_q = max_q_len; p.nq = num_heads; p.nkv = num_kv_heads; p.group = group; p.bs = block_size;
  p.group_inv = (uint32_t)((1ull << 32) / (uint32_t)group + 1);
  p.num_blocks = num_blocks; p.scale = scale; p.out = out; p.status = dev_status;
  const bool fp8 = kv_dtype == KVE_FP8_E4M3;
  const Split s = split_of(batch, max_q_len, max_ctx, num_kv_heads, group);
  const bool small = dtype == KVE_BF16 && tree_attn_small_takes(p, fp8);
  const bool wide = !small && use_wide(max_q_len, group) &&
                    (fp8 || (dtype == KVE_BF16 && block_size % 16 == 0 && num_blocks * block_size < 0x7ffffff0LL));
  const size_t part = small  ? tree_attn_small_partial_bytes(batch, max_ctx, num_kv_heads, head_dim)
                      : wide ? tree_attn_wide_partial_bytes(batch, max_q_len, max_ctx, num_kv_heads, group, head_dim)
                             : partial_bytes(s, batch, num_kv_heads, head_dim);
  if (part && (!workspace || workspace_bytes < kTreeCounterBytes + part))
    return set_error(KVE_ERR_WORKSPACE, "%s: workspace needs %zu bytes", me, kTreeCounterBytes + part);
  if (part && (uintptr_t)workspace % 16) return set_error(KVE_ERR_ARG, "%s: workspace must be 16-byte aligned", me);
  p.counters = static_cast<int*>(workspace);
  p.partials = part ? reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kTreeCounterBytes) : nullptr;
  p.chunk = s.chunk; p.n_chunks = s.n_chunks; p.n_qtiles = s.n_qtiles;
  if (small) return tree_attn_small(p, batch, max_ctx, head_dim, fp8, stream);
  if (wide) return tree_attn_wide(p, batch, max_ctx, head_dim, fp8, stream);
  if (fp8) return launch_hd<kFp8>(p, head_dim, s.rb, batch, stream);
  if (dtype == KVE_BF16) return launch_hd<kBf16>(p, head_dim, s.rb, batch, stream);
  return launch_hd<kF32>(p, head_dim, s.rb, batch, stream);
}

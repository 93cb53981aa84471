// Tree attention for at most eight query rows per kv head: single tokens, and the
// smallest trees. bf16 and e4m3 caches with blocks of a multiple of 16 positions.
//
// The same operation as tree_attn.cu. With so few rows the cache's bytes are the work, and
// what keeps a kernel from them is the instructions it spends per key. The products
// are therefore turned round, keys and dims in the M dimension of m16n8k16 and the
// rows in N, so that eight rows fill a tile of eight (as M they would half fill one of
// 16) and a key costs half the products and half the exponentials:
//   S^T = K Q^T    A: 16 keys x 16 dims of K,  B: Q^T, kept in registers
//   O^T += V^T P^T A: 16 dims x 16 keys of V (transposed matrix loads), B: P^T, which is S^T's
//                  registers after a transposition of 8 x 8 blocks (movmatrix)
// e4m3: the bytes become f16 (K) and bf16 (V) on their way into the products, with the
// exponents applied to the scores and to p as in tree_attn.cu.
//
// A CTA takes one (sequence x kv head) and a chunk of the keys; each of its four warps is
// a stream of its own: every fourth tile of the chunk, through a ring of its own that
// its issuing lane fills by TMA (boxes of 16 keys; the exponents by a 4-byte cp.async a
// lane), with no barrier between warps before the end.
//
// Measured, e4m3, 64 sequences of 2250 to 9000 keys, 16 / 2 heads of 128: 50 us, 3.7 TB/s of cache bytes
// (88 us in the kernel of tree_attn.cu; 66 with two CTAs an SM and rings of three tiles); bf16 69 us, 5.4 TB/s.
// Over e4m3 nothing is saturated (DRAM 42 %, integer pipes 53 %, tensor cores 12 %): three warps a scheduler, each a
// chain of loads, conversions and products, issue in half of its cycles. Converting V by shifts and masks
// instead of the conversion instructions loads the integer pipes more (56 us).
#include <cuda_fp8.h>
#include <math.h>

#include <atomic>
#include <cstring>

#include "kve_common.cuh"
#include "tma.cuh"
#include "tree_attn.cuh"

namespace kve {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 8;

template <bool FP8, int HD>
struct SmallShape {
  static constexpr int ELEM = FP8 ? 1 : 2;
  static constexpr int GROUP = 16 * HD * ELEM;              // bytes of 16 keys
  static constexpr int GROUPS = GROUP >= 4096 ? 1 : 2;      // of a tile
  static constexpr int KEYS = 16 * GROUPS;
  static constexpr int PAIR = 2 * GROUPS * GROUP;           // K and V of a tile
  static constexpr int NST = 16384 / PAIR;                  // tiles of a warp's ring
  static constexpr int RINGS = kWarps * NST * PAIR;
  static constexpr int XROW = HD + 4;
  static constexpr int MERGE = kWarps * kRows * (XROW + 2) * 4;
  static constexpr int AREA = RINGS > MERGE ? RINGS : MERGE;
  static constexpr int ROWB = HD * ELEM < 128 ? 64 : 128;   // bytes of a box row
  static constexpr size_t SMEM = 1024 + AREA + (FP8 ? kWarps * NST * 256 : 0);  // a word per key for K's and V's exponents
};

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack2h(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t to_f16(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
  return (uint32_t)h.x | (uint32_t)h.y << 16;
}
__device__ __forceinline__ uint32_t to_bf16(uint32_t two) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)two, __NV_E4M3);
  const float2 f = __half22float2(__half2(h));
  return pack2(f.x, f.y);
}
template <bool F16>
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t lds16(uint32_t addr) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}
// Loads by the warp's issuing lane, inside a warp that runs together.
__device__ __forceinline__ void tma_box(uint32_t lead, uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n\t}"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar), "r"(lead) : "memory");
}
template <bool FP8, int HD>
__global__ void __launch_bounds__(kThreads, 3)
tree_attn_small_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, TreeParams p) {
  using S = SmallShape<FP8, HD>;
  constexpr int NST = S::NST, GROUPS = S::GROUPS, KEYS = S::KEYS;
  extern __shared__ uint8_t raw_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t full[kWarps][NST];
  __shared__ int flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = lane >> 2, tq = lane & 3;
  if (threadIdx.x == 0) {
    for (int w = 0; w < kWarps; ++w)
      for (int i = 0; i < NST; ++i) mbar_init(smem_u32(&full[w][i]), FP8 ? 33 : 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    prefetch_map(&map_k);
    prefetch_map(&map_v);
  }
  grid_dep_wait();
  grid_dep_launch();

  const int bh = blockIdx.x, c = blockIdx.y;
  const int b = bh / p.nkv, h = bh % p.nkv;
  const int ctx = p.ctx_lens[b], ql = p.q_lens[b], qoff = p.q_offsets[b];
  if (ql < 0 || ql > p.max_q || ctx < ql || qoff < 0 || qoff > p.q_rows - ql || (int64_t)ctx > (int64_t)p.table_stride * p.bs ||
      (int64_t)ctx > (int64_t)p.chunk * p.n_chunks) {
    if (threadIdx.x == 0 && c == 0) report(p.status, KVE_ERR_BOUNDS);
    return;
  }
  const int rows = ql * p.group;
  if (rows <= 0) return;
  const int hist = ctx - ql;
  const int live = (ctx + p.chunk - 1) / p.chunk;
  if (c >= live) return;
  const int key_lo = c * p.chunk, key_hi = min(ctx, key_lo + p.chunk);
  const int n_tiles = (key_hi - key_lo + KEYS - 1) / KEYS;
  const int my_tiles = n_tiles > warp ? (n_tiles - warp + kWarps - 1) / kWarps : 0;
  __syncthreads();

  // The ring: [stage][K groups, V groups], and for e4m3 [stage][K, V][key]: the aligned word that holds
  // the key's exponent byte.
  const uint32_t ring = smem_u32(smem) + warp * NST * S::PAIR;
  const uint32_t sring = smem_u32(smem) + S::AREA + warp * NST * 256;
  const uint32_t lead = elect_lane();
  // Lane l knows where group l of a window of 32 groups (16 keys each) of this warp's tiles lies.
  const int past = (int)(p.num_blocks * p.bs);
  constexpr int WINDOW = 32 / GROUPS;  // tiles
  auto rows_of = [&](int w) {
    const int i = w * WINDOW + lane / GROUPS;
    const int key = key_lo + (warp + kWarps * i) * KEYS + lane % GROUPS * 16;
    int y = past;
    if (i < my_tiles && key < key_hi) {
      const int blk = p.tables[(size_t)b * p.table_stride + key / p.bs];
      if (blk >= 0 && blk < p.num_blocks) y = blk * p.bs + key % p.bs;
      else report(p.status, KVE_ERR_BOUNDS);  // reads as zeros
    }
    return y;
  };
  int now = rows_of(0), next = rows_of(1);
  auto load = [&](int i) {  // tile i of this warp
    if (i > 0 && i % WINDOW == 0) {
      now = next;
      next = rows_of(i / WINDOW + 1);
    }
    const int st = i % NST;
    const uint32_t bar = smem_u32(&full[warp][st]), dst = ring + st * S::PAIR;
    if (lead) mbar_expect_tx(bar, S::PAIR);
    __syncwarp();
#pragma unroll
    for (int u = 0; u < GROUPS; ++u) {
      const int y = __shfl_sync(0xffffffffu, now, i % WINDOW * GROUPS + u);
#pragma unroll
      for (int half = 0; half < (HD * S::ELEM + 127) / 128; ++half) {
        const uint32_t to = dst + u * S::GROUP + half * 2048;
        tma_box(lead, to, &map_k, h * HD + half * 64, y, bar);
        tma_box(lead, to + GROUPS * S::GROUP, &map_v, h * HD + half * 64, y, bar);
      }
    }
    if constexpr (FP8) {
      // lane l: key l of the tile
      const int y = __shfl_sync(0xffffffffu, now, i % WINDOW * GROUPS + lane / 16);
      const size_t word = y < past ? (((size_t)(y + lane % 16) * p.nkv + h) & ~(size_t)3) : 0;
      const uint32_t to = sring + st * 256 + lane * 4, bytes = y < past ? 4u : 0u;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(p.k_scale + word), "r"(bytes) : "memory");
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to + 128), "l"(p.v_scale + word), "r"(bytes) : "memory");
      asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
    }
  };
  for (int i = 0; i < NST && i < my_tiles; ++i) load(i);

  // Q^T: row g of the lane, zeros behind the last row.
  const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(p.q);
  auto head_row = [&](int r) {
    const int node = node_of(p, r);
    return ((size_t)(qoff + node) * p.nq + h * p.group + r - node * p.group) * HD;
  };
  constexpr int KSTEPS = HD / 16;
  uint32_t qb[KSTEPS][2];
  float sl = p.scale * 1.4426950408889634f;  // of row g (e4m3: with the power of two taken out of q)
  if constexpr (!FP8) {
    const uint32_t* src = g < rows ? reinterpret_cast<const uint32_t*>(q + head_row(g)) : nullptr;
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk) {
      qb[kk][0] = src ? src[kk * 8 + tq] : 0u;
      qb[kk][1] = src ? src[kk * 8 + tq + 4] : 0u;
    }
  } else {
    const uint2* src = g < rows ? reinterpret_cast<const uint2*>(q + head_row(g)) : nullptr;
    uint2 raw[KSTEPS];
    float top = 0.f;
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk) {
      raw[kk] = src ? src[kk / 4 * 16 + tq * 4 + kk % 4] : make_uint2(0u, 0u);
      const float2 x = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&raw[kk].x));
      const float2 y = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&raw[kk].y));
      top = fmaxf(top, fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(y.x), fabsf(y.y))));
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // up = 2^(7 - exponent of the largest), kept between 2^-112 and 2^126
    const int ex = min(max((int)(__float_as_uint(top) >> 23), 8), 246);
    const float up = __uint_as_float((uint32_t)(261 - ex) << 23);
    sl *= 1.f / up;
#pragma unroll
    for (int kk = 0; kk < KSTEPS; ++kk) {
      const float2 x = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&raw[kk].x));
      const float2 y = __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&raw[kk].y));
      qb[kk][0] = pack2h(x.x * up, x.y * up);
      qb[kk][1] = pack2h(y.x * up, y.y * up);
    }
  }
  // This lane's two rows of S^T: 2 tq and 2 tq + 1.
  float sl_of[2];
  int node[2];
  const uint32_t* mask[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    sl_of[e] = __shfl_sync(0xffffffffu, sl, (2 * tq + e) * 4);
    node[e] = node_of(p, min(2 * tq + e, rows - 1));
    mask[e] = p.mask ? p.mask + (size_t)(qoff + node[e]) * p.mask_words : nullptr;
  }

  constexpr int DT = HD / 16;
  float acc[DT][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int d = 0; d < DT; ++d) acc[d][0] = acc[d][1] = acc[d][2] = acc[d][3] = 0.f;
  // Address of 16 bytes `piece` of key row r (0 .. 15) of a group.
  auto at = [&](uint32_t base, int r, int piece) {
    if constexpr (S::ROWB == 64) return base + (uint32_t)(r * 64 + ((piece ^ (r >> 1 & 3)) << 4));
    else return base + (uint32_t)((piece >> 3) * 2048 + r * 128 + (((piece & 7) ^ (r & 7)) << 4));
  };
  const int mat = lane >> 3, rr = lane & 7;
  bool ok = true;
  for (int i = 0; i < my_tiles; ++i) {
    const int st = i % NST;
    ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&full[warp][st]), (uint32_t)(i / NST) & 1u, p.status));
    if (!ok) {
      for (int j = i + 1; j < i + NST && j < my_tiles; ++j)
        mbar_wait(smem_u32(&full[warp][j % NST]), (uint32_t)(j / NST) & 1u, p.status);  // what is in flight
      break;
    }
    const int kt = key_lo + (warp + kWarps * i) * KEYS;
    const uint32_t kb = ring + st * S::PAIR, vb = kb + GROUPS * S::GROUP;
    const uint32_t ks = sring + st * 256 + ((g * p.nkv + h) & 3);  // + 4 key: the byte of keys g and g + 8
    const bool masked = kt + KEYS > hist || kt + KEYS > key_hi;
    bool odd = false;
    if (masked) {
      // V rows behind the last key are not this sequence's: zeros, as 0 x NaN would not be. New tokens'
      // rows are looked through for infinities and NaN.
      constexpr int PIECES = HD * S::ELEM / 16;
      for (int j = lane; j < KEYS * PIECES; j += 32) {
        const int r = j / PIECES, key = kt + r;
        const uint32_t a = at(vb + r / 16 * S::GROUP, r % 16, j % PIECES);
        if (key >= key_hi) {
          asm volatile("st.shared.v4.u32 [%0], {%1,%1,%1,%1};" ::"r"(a), "r"(0u) : "memory");
        } else if (key >= hist) {
          const uint4 x = lds128(a);
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            if constexpr (FP8) odd |= __vcmpeq4(w[u] & 0x7f7f7f7fu, 0x7f7f7f7fu) != 0u;
            else odd |= (w[u] & 0x7f800000u) == 0x7f800000u || (w[u] & 0x7f80u) == 0x7f80u;
          }
        }
      }
      __syncwarp();
    }

    // S^T: s[u][0], [1]: key g of group u, this lane's rows; [2], [3]: key g + 8.
    float s[GROUPS][4], vs[GROUPS][2];
#pragma unroll
    for (int u = 0; u < GROUPS; ++u) {
      s[u][0] = s[u][1] = s[u][2] = s[u][3] = 0.f;
      const uint32_t kg = kb + u * S::GROUP;
      if constexpr (!FP8) {
#pragma unroll
        for (int kk = 0; kk < KSTEPS; ++kk) {
          uint32_t a[4];
          ldsm(at(kg, (mat & 1) * 8 + rr, kk * 2 + (mat >> 1)), a);
          mma<false>(s[u], a[0], a[1], a[2], a[3], qb[kk][0], qb[kk][1]);
        }
      } else {
        // 16 bytes a lane: dims 64 dg + 16 tq .. of keys g and g + 8. At 128-byte rows neighbouring keys
        // take their two 64-dim parts in opposite order, so that a phase's eight lanes meet no bank twice.
        uint32_t x[HD / 64][2][4];
#pragma unroll
        for (int dg = 0; dg < HD / 64; ++dg) {
          const int from = HD == 128 ? dg ^ (g & 1) : dg;
          const uint4 lo = lds128(at(kg, g, from * 4 + tq)), hi = lds128(at(kg, g + 8, from * 4 + tq));
          x[dg][0][0] = lo.x; x[dg][0][1] = lo.y; x[dg][0][2] = lo.z; x[dg][0][3] = lo.w;
          x[dg][1][0] = hi.x; x[dg][1][1] = hi.y; x[dg][1][2] = hi.z; x[dg][1][3] = hi.w;
        }
        if constexpr (HD == 128) {
#pragma unroll
          for (int e = 0; e < 2; ++e)
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const uint32_t first = x[0][e][w], second = x[1][e][w];
              x[0][e][w] = g & 1 ? second : first;
              x[1][e][w] = g & 1 ? first : second;
            }
        }
#pragma unroll
        for (int dg = 0; dg < HD / 64; ++dg)
#pragma unroll
          for (int w = 0; w < 4; ++w)
            mma<true>(s[u], to_f16(x[dg][0][w] & 0xffffu), to_f16(x[dg][1][w] & 0xffffu), to_f16(x[dg][0][w] >> 16),
                      to_f16(x[dg][1][w] >> 16), qb[dg * 4 + w][0], qb[dg * 4 + w][1]);
        const float k0 = scale_value(lds8(ks + (u * 16 + g) * 4));
        const float k1 = scale_value(lds8(ks + (u * 16 + g + 8) * 4));
        vs[u][0] = scale_value(lds8(ks + 128 + (u * 16 + g) * 4));
        vs[u][1] = scale_value(lds8(ks + 128 + (u * 16 + g + 8) * 4));
        s[u][0] *= k0;
        s[u][1] *= k0;
        s[u][2] *= k1;
        s[u][3] *= k1;
        // a new token's exponent byte of NaN is like a NaN row
        const int k0_at = kt + u * 16 + g;
        if (masked)
          odd |= (k0_at >= hist && k0_at < key_hi && !(vs[u][0] < INFINITY)) ||
                 (k0_at + 8 >= hist && k0_at + 8 < key_hi && !(vs[u][1] < INFINITY));
      }
    }
    uint32_t see[2] = {~0u, ~0u};  // of the lane's rows: the tile's keys
    if (masked) {
      odd = __any_sync(0xffffffffu, odd);
      const int in = key_hi - kt;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        see[e] = p.mask ? mask_bits<32>(mask[e], p.mask_words, kt - hist) : chain_bits(node[e], kt - hist);
        if (in < 32) see[e] &= (1u << in) - 1u;
      }
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int u = 0; u < GROUPS; ++u)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int e = x & 1, key = u * 16 + g + (x >> 1) * 8;
        s[u][x] = !masked || see[e] >> key & 1 ? s[u][x] * sl_of[e] : -INFINITY;
        top[e] = fmaxf(top[e], s[u][x]);
      }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      top[0] = fmaxf(top[0], __shfl_xor_sync(0xffffffffu, top[0], o));
      top[1] = fmaxf(top[1], __shfl_xor_sync(0xffffffffu, top[1], o));
    }
    if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
      float f[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float t = fmaxf(m[e], top[e]);
        f[e] = t == m[e] ? 1.f : ex2(m[e] - t);
        m[e] = t;
        l[e] *= f[e];
      }
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        acc[d][0] *= f[0];
        acc[d][1] *= f[1];
        acc[d][2] *= f[0];
        acc[d][3] *= f[1];
      }
    }
    const float base[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
    for (int u = 0; u < GROUPS; ++u) {
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        s[u][x] = ex2(s[u][x] - base[x & 1]);
        l[x & 1] += s[u][x];
      }
    }
    if (odd) {
      // key by key, over the rows that see it
      for (int key = 0; key < KEYS; ++key) {
        const int u = key / 16, r = key % 16, from = (r & 7) * 4 + tq;
        float pr[2], unit = 1.f;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float v0 = s[0][e], v1 = s[0][2 + e];
          if constexpr (GROUPS == 2) {
            v0 = u ? s[GROUPS - 1][e] : v0;
            v1 = u ? s[GROUPS - 1][2 + e] : v1;
          }
          pr[e] = __shfl_sync(0xffffffffu, r < 8 ? v0 : v1, from);
        }
        if constexpr (FP8) {
          float v0 = vs[0][0], v1 = vs[0][1];
          if constexpr (GROUPS == 2) {
            v0 = u ? vs[GROUPS - 1][0] : v0;
            v1 = u ? vs[GROUPS - 1][1] : v1;
          }
          unit = __shfl_sync(0xffffffffu, r < 8 ? v0 : v1, from);
        }
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            float v;
            if constexpr (FP8) {
              const int dim = d * 16 + 2 * g + y;
              v = unit * __half2float(__half(__nv_cvt_fp8_to_halfraw(
                             (__nv_fp8_storage_t)lds8(at(vb + u * S::GROUP, r, dim >> 4) + (dim & 15)), __NV_E4M3)));
            } else {
              const int dim = d * 16 + g + 8 * y;
              v = __uint_as_float(lds16(at(vb + u * S::GROUP, r, dim >> 3) + (dim & 7) * 2) << 16);
            }
            if (see[0] >> key & 1) acc[d][2 * y] += pr[0] * v;
            if (see[1] >> key & 1) acc[d][2 * y + 1] += pr[1] * v;
          }
      }
    } else {
#pragma unroll
      for (int u = 0; u < GROUPS; ++u) {
        uint32_t b0, b1;
        if constexpr (FP8) {
          // a masked key contributes exactly 0, whatever its exponent
          b0 = pack2(s[u][0] == 0.f ? 0.f : s[u][0] * vs[u][0], s[u][1] == 0.f ? 0.f : s[u][1] * vs[u][0]);
          b1 = pack2(s[u][2] == 0.f ? 0.f : s[u][2] * vs[u][1], s[u][3] == 0.f ? 0.f : s[u][3] * vs[u][1]);
        } else {
          b0 = pack2(s[u][0], s[u][1]);
          b1 = pack2(s[u][2], s[u][3]);
        }
        b0 = transpose8(b0);
        b1 = transpose8(b1);
        const uint32_t vg = vb + u * S::GROUP;
        if constexpr (!FP8) {
#pragma unroll
          for (int d = 0; d < DT; ++d) {
            uint32_t a[4];
            ldsm_t(at(vg, (mat >> 1) * 8 + rr, d * 2 + (mat & 1)), a);
            mma<false>(acc[d], a[0], a[1], a[2], a[3], b0, b1);
          }
        } else {
          // Two pieces a load: for each, keys 2 tq, + 1 (then + 8) of dims 2 g and 2 g + 1, which stand for
          // rows g and g + 8 of the product's 16 dims.
#pragma unroll
          for (int d = 0; d < DT; d += 2) {
            uint32_t a[4];
            ldsm_t(at(vg, (mat & 1) * 8 + rr, d + (mat >> 1)), a);
#pragma unroll
            for (int x = 0; x < 4; ++x) a[x] = __byte_perm(a[x], 0u, 0x3120);
#pragma unroll
            for (int x = 0; x < 2; ++x)
              mma<false>(acc[d + x], to_bf16(a[2 * x] & 0xffffu), to_bf16(a[2 * x] >> 16), to_bf16(a[2 * x + 1] & 0xffffu),
                         to_bf16(a[2 * x + 1] >> 16), b0, b1);
          }
        }
      }
    }
    __syncwarp();
    if (i + NST < my_tiles) {
      fence_proxy_async_smem();
      load(i + NST);
    }
  }
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
    l[0] += __shfl_xor_sync(0xffffffffu, l[0], o);
    l[1] += __shfl_xor_sync(0xffffffffu, l[1], o);
  }
  const bool failed = __syncthreads_or(!ok);

  // The warps' states meet in shared memory (the rings are free now).
  float* xs = reinterpret_cast<float*>(smem);          // [warp][row][XROW]
  float* xm = xs + kWarps * kRows * S::XROW;           // [warp][row][m, l]
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const int dim = FP8 ? d * 16 + 2 * g + (x >> 1) : d * 16 + g + (x >> 1) * 8;
      xs[(warp * kRows + 2 * tq + (x & 1)) * S::XROW + dim] = acc[d][x];
    }
  if (g == 0) {
#pragma unroll
    for (int e = 0; e < 2; ++e)
      *reinterpret_cast<float2*>(xm + (warp * kRows + 2 * tq + e) * 2) = make_float2(m[e], l[e]);
  }
  __syncthreads();
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out);
  constexpr int PROW = HD + 4;
  float* part0 = p.partials + (size_t)bh * p.n_chunks * kRows * PROW;
  auto store4 = [&](int r, int d, float4 o, float sum) {
    const bool none = sum == 0.f;  // the row sees no key
    *reinterpret_cast<uint2*>(out + head_row(r) + d) =
        make_uint2(pack2(none ? 0.f : o.x / sum, none ? 0.f : o.y / sum), pack2(none ? 0.f : o.z / sum, none ? 0.f : o.w / sum));
  };
  if (!failed) {
    for (int i = threadIdx.x; i < rows * (HD / 4); i += kThreads) {
      const int r = i / (HD / 4), d = i % (HD / 4) * 4;
      float t = -INFINITY, sum = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) t = fmaxf(t, xm[(w * kRows + r) * 2]);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float2 ml = *reinterpret_cast<const float2*>(xm + (w * kRows + r) * 2);
        const float f = ml.x == t ? 1.f : ex2(ml.x - t);
        const float4 x = *reinterpret_cast<const float4*>(xs + (w * kRows + r) * S::XROW + d);
        sum += ml.y * f;
        o.x += x.x * f;
        o.y += x.y * f;
        o.z += x.z * f;
        o.w += x.w * f;
      }
      if (live == 1) {
        store4(r, d, o, sum);
      } else {
        float* pr = part0 + ((size_t)c * kRows + r) * PROW;
        *reinterpret_cast<float4*>(pr + d) = o;
        if (d == 0) *reinterpret_cast<float2*>(pr + HD) = make_float2(t, sum);
      }
    }
  }
  if (live == 1) return;

  // The last chunk to arrive joins them, in chunk order.
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    int* cnt = p.counters + bh;
    flag = atomicAdd(cnt, 1) == live - 1;
    if (flag) *cnt = 0;  // the workspace is left as it was
  }
  __syncthreads();
  if (!flag || failed) return;
  __threadfence();
  for (int i = threadIdx.x; i < rows * (HD / 4); i += kThreads) {
    const int r = i / (HD / 4), d = i % (HD / 4) * 4;
    const float* pr = part0 + (size_t)r * PROW;
    float t = -INFINITY, sum = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < live; ++k) {
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(pr + (size_t)k * kRows * PROW + HD));
      const float4 x = __ldcg(reinterpret_cast<const float4*>(pr + (size_t)k * kRows * PROW + d));
      const float tn = fmaxf(t, ml.x);
      const float f = tn == t ? 1.f : ex2(t - tn), w = tn == ml.x ? 1.f : ex2(ml.x - tn);
      t = tn;
      sum = sum * f + ml.y * w;
      o.x = o.x * f + x.x * w;
      o.y = o.y * f + x.y * w;
      o.z = o.z * f + x.z * w;
      o.w = o.w * f + x.w * w;
    }
    store4(r, d, o, sum);
  }
}

// ------------------------------------------------------------------ host
// Chunks of a sequence, none under 256 keys: a third more than the 444 CTAs that run at once. 64 e4m3
// requests take 54.5 us at 2250 to 9000 keys and 42.3 at 4096 each, with chunks for 444 CTAs 58.7 and 44.2 (the
// shorter chunks' second wave fills what the first leaves uneven); bf16 ones 69.4 and 52.1 against 67.0 and 51.3.
void small_split(int batch, int max_ctx, int nkv, int* chunk, int* n_chunks) {
  const long long units = (long long)batch * nkv, want = 4 * 148;
  const long long c = (want + units - 1) / units;
  long long keys = ((long long)max_ctx + c - 1) / c;
  keys = (keys + 127) / 128 * 128;
  keys = keys < 256 ? 256 : keys;
  *chunk = (int)keys;
  *n_chunks = (int)((max_ctx + keys - 1) / keys);
  if (*n_chunks < 1) *n_chunks = 1;
}

bool pool_map(CUtensorMap* map, const void* pool, int64_t rows, int width, int hd, bool fp8) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const int elem = fp8 ? 1 : 2;
  cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows};
  cuuint64_t strides[1] = {(cuuint64_t)width * elem};
  cuuint32_t box[2] = {(cuuint32_t)(fp8 ? hd : 64), 16};
  cuuint32_t estr[2] = {1, 1};
  return fn(map, fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(pool), dims,
            strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            fp8 && hd == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool FP8, int HD>
int launch(const TreeParams& p, int batch, cudaStream_t stream) {
  using S = SmallShape<FP8, HD>;
  CUtensorMap mk, mv;
  memset(&mk, 0, sizeof(mk));
  memset(&mv, 0, sizeof(mv));
  const int64_t rows = p.num_blocks * p.bs;
  if (!pool_map(&mk, p.pool_k, rows, p.nkv * HD, HD, FP8) || !pool_map(&mv, p.pool_v, rows, p.nkv * HD, HD, FP8))
    return set_error(KVE_ERR_CUDA, "kve_paged_tree_attn: no tensor map for the pool");
  static std::atomic<uint64_t> prepared{0};  // the shared-memory limit is an attribute of the kernel on one device
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (err == cudaSuccess && !(prepared.load(std::memory_order_relaxed) & bit)) {
    err = cudaFuncSetAttribute(tree_attn_small_kernel<FP8, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (int)S::SMEM);
    if (err == cudaSuccess) prepared.fetch_or(bit, std::memory_order_relaxed);
  }
  if (err != cudaSuccess) {
    cudaGetLastError();
    return set_error(KVE_ERR_CUDA, "kve_paged_tree_attn: %s", cudaGetErrorString(err));
  }
  launch_kernel(tree_attn_small_kernel<FP8, HD>, dim3(batch * p.nkv, p.n_chunks), dim3(kThreads), S::SMEM,
                stream, mk, mv, p);
  return check_launch("kve_paged_tree_attn(small)");
}

}  // namespace

bool tree_attn_small_takes(const TreeParams& p, bool fp8) {
  if ((long long)p.max_q * p.group > kRows || p.bs % 16 || p.num_blocks * p.bs >= 0x7ffffff0LL) return false;
  return !fp8 || ((uintptr_t)p.k_scale % 4 == 0 && (uintptr_t)p.v_scale % 4 == 0);
}

size_t tree_attn_small_partial_bytes(int batch, int max_ctx, int nkv, int hd) {
  int chunk, n_chunks;
  small_split(batch, max_ctx, nkv, &chunk, &n_chunks);
  return n_chunks == 1 ? 0 : (size_t)batch * nkv * n_chunks * kRows * (hd + 4) * sizeof(float);
}

int tree_attn_small(TreeParams p, int batch, int max_ctx, int hd, bool fp8, cudaStream_t stream) {
  small_split(batch, max_ctx, p.nkv, &p.chunk, &p.n_chunks);
  p.n_qtiles = 1;
  if (fp8) return hd == 64 ? launch<true, 64>(p, batch, stream) : launch<true, 128>(p, batch, stream);
  return hd == 64 ? launch<false, 64>(p, batch, stream) : launch<false, 128>(p, batch, stream);
}

}  // namespace kve

// Tree attention for many query rows per kv head, on the 5th-generation tensor cores.
//
// The same operation as tree_attn.cu for bf16 and e4m3 caches, where a sequence's tree has
// more rows (nodes x group heads) than the few-row kernel takes: the work is then bound by
// the tensor cores and the exponentials rather than by the cache's bytes. e4m3 tiles become
// bf16 on their way into shared memory (e4m3 times a power of two: exactly, above 2^-126).
//
// A CTA has two softmax warpgroups, each with two 128-row score tiles S and one output
// tile O in tensor memory, and one of two jobs:
//   one query tile (up to 128 rows): the two groups take the even and the odd key tiles
//     of the chunk, and their outputs are joined at the end;
//   two query tiles (up to 256 rows): both groups take every key tile, one query tile
//     each, so that a K/V tile is fetched into shared memory once for 256 rows.
// While a group is in the softmax of one tile, the tensor cores have its next S ready and
// add its last P V: with 128-key tiles and one S a group, a step waited for both products
// (4080 cycles a 128 keys, against 2300 in the softmax). Per key tile (64 keys) and group:
//   S = Q K^T      tcgen05.mma, Q and K in shared memory (128-byte swizzle, K-major)
//   P = 2^(S sl - m)  one thread a row: a pass for the maximum, a pass for the exponentials;
//                  P goes back to tensor memory as bf16, over S
//   O += P V       tcgen05.mma, P from tensor memory, V from shared memory as it lies there
//                  (keys x dims: the transposed, MN-major form)
// O is rescaled only where the running maximum has grown by more than 2^8 since its
// last use: until then P is at most 2^8, which bf16 and fp32 hold as well as 1.
//
// bf16 K and V tiles come by TMA, a loading warp each, in boxes of 16 keys (so blocks of any
// multiple of 16 positions), e4m3 tiles through the registers of four more warps (any block size).
// K and V have a ring of slots each. Tiles with new tokens or the last key are looked
// over before they are used: rows behind the last key are zeroed (the pool's contents there
// are not this sequence's), and new tokens' V rows are checked for infinities and NaN, which
// 0 x V would spread to rows that do not see them. Where there are any, the chunk's rows
// are computed again, key by key.
//
// Measured (replayed graphs), 16 / 2 heads of 128: 32 trees of 64 nodes at 4500 keys 81 us (930 TFLOP/s), 64 of 16 nodes
// at 175 to 700 keys 15.8 us; over e4m3 caches 265 us (the copying warps' chains of loads, conversions and stores) and,
// at 700 keys, 44 us (707 and 78 us in the kernel of tree_attn.cu). In the wide case no unit is saturated: the tensor
// cores are busy in half of the cycles, the schedulers issue in 45 % of them, the exponentials' unit runs at 38 %; a step
// is the chain product, softmax, product with two tiles a group in flight, on 128 of the 148 SMs. Running every kShare-th
// pair of exponentials on the fp32 units takes 81.7 us at 4, 85.7 at 2, and 87.2 with none.
#include <cuda_fp8.h>
#include <float.h>
#include <math.h>

#include <atomic>
#include <cstring>
#include <type_traits>

#include "kve_common.cuh"
#include "tma.cuh"
#include "tree_attn.cuh"

namespace kve {
namespace {

constexpr int kKeys = 64;        // keys of a tile
constexpr int kRows = 128;       // query rows of a tile
constexpr int kThreads = 384;    // K loader, a warp of products for each group, V loader; two softmax warpgroups
constexpr int threads_of(bool fp8) { return kThreads + (fp8 ? 128 : 0); }  // e4m3: four warps that copy
constexpr int kMaxSlots = 12;
constexpr int kShare = 4;        // every kShare-th pair of exponentials runs on the fp32 units

__device__ __forceinline__ uint64_t desc_k_major(uint32_t addr) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 |
         (uint64_t)2 << 61;
}
// V as it lies: 64-dim halves `half_bytes` apart, 8-key groups 1024 bytes apart.
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t addr, uint32_t half_bytes) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | (uint64_t)((half_bytes >> 4) & 0x3FFF) << 16 | (uint64_t)(1024 >> 4) << 32 |
         (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// kind::f16, fp32 accumulator, bf16 operands, M = 128; b_mn: B is MN-major.
__device__ __forceinline__ uint32_t mma_idesc(int n, bool b_mn) {
  return 1u << 4 | 1u << 7 | 1u << 10 | (b_mn ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(kRows >> 4) << 24;
}
// Products and commits are written for a whole warp that runs together, with one lane
// issuing: their descriptors then stay in uniform registers (issued from a branch of
// one lane, each product cost 75 to 100 cycles, more than it computes).
__device__ __forceinline__ uint32_t elect_lane() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}
__device__ __forceinline__ void mma_ss(uint32_t lead, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accum), "r"(lead) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accum), "r"(lead) : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t lead, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(bar), "r"(lead) : "memory");
}
// A TMA load by the warp's issuing lane, like the products: from lanes with coordinates of
// their own, one box after the other, each cost about 140 cycles.
__device__ __forceinline__ void tma_load(uint32_t lead, uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];\n\t}"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar), "r"(lead) : "memory");
}
__device__ __forceinline__ void tma_load_v(uint32_t lead, uint32_t dst, const CUtensorMap* map, int y, int z, uint32_t bar) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%6, %2, %3}], [%4];\n\t}"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(y), "r"(z), "r"(bar), "r"(lead), "r"(0) : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// 32 columns of this thread's lane: asked for here, there after tmem_arrived on the same registers.
__device__ __forceinline__ void tmem_ask(uint32_t addr, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
        "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_arrived(float (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]),
                 "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]),
                 "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]),
                 "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
               :: "memory");
}
__device__ __forceinline__ void tmem_load(uint32_t addr, float (&v)[32]) {
  tmem_ask(addr, v);
  tmem_arrived(v);
}
__device__ __forceinline__ void tmem_store32(uint32_t addr, const float (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
      "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3])),
      "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])), "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7])),
      "r"(__float_as_uint(v[8])), "r"(__float_as_uint(v[9])), "r"(__float_as_uint(v[10])), "r"(__float_as_uint(v[11])),
      "r"(__float_as_uint(v[12])), "r"(__float_as_uint(v[13])), "r"(__float_as_uint(v[14])), "r"(__float_as_uint(v[15])),
      "r"(__float_as_uint(v[16])), "r"(__float_as_uint(v[17])), "r"(__float_as_uint(v[18])), "r"(__float_as_uint(v[19])),
      "r"(__float_as_uint(v[20])), "r"(__float_as_uint(v[21])), "r"(__float_as_uint(v[22])), "r"(__float_as_uint(v[23])),
      "r"(__float_as_uint(v[24])), "r"(__float_as_uint(v[25])), "r"(__float_as_uint(v[26])), "r"(__float_as_uint(v[27])),
      "r"(__float_as_uint(v[28])), "r"(__float_as_uint(v[29])), "r"(__float_as_uint(v[30])), "r"(__float_as_uint(v[31]))
      : "memory");
}
__device__ __forceinline__ void tmem_store16(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_store_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// NaN where any operand is.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float max2(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// Two fp32 operations in one.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(d)
      : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)), "l"(*reinterpret_cast<uint64_t*>(&c)));
  return *reinterpret_cast<float2*>(&d);
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(*reinterpret_cast<uint64_t*>(&a)), "l"(*reinterpret_cast<uint64_t*>(&b)));
  return *reinterpret_cast<float2*>(&d);
}
// 2^x of two numbers up to 2^7 without the special-function unit: x = n + r, n the nearest
// integer (x + 1.5 2^23 has it in its low bits), 2^r on [-1/2, 1/2] by the polynomial of
// degree 4 of least relative error (2.6e-6, found by weighted least squares), n added to
// the exponent. Below 2^-126: 2^-126, which is nothing beside a row's largest term. Not for NaN.
__device__ __forceinline__ float2 ex2_fma(float2 x) {
  x.x = fmaxf(x.x, -126.f);
  x.y = fmaxf(x.y, -126.f);
  const float2 big = make_float2(12582912.f, 12582912.f), neg = make_float2(-12582912.f, -12582912.f);
  const float2 t = add2(x, big);
  const float2 r = fma2(add2(t, neg), make_float2(-1.f, -1.f), x);
  float2 y = fma2(r, make_float2(0.00957009941f, 0.00957009941f), make_float2(0.0559178703f, 0.0559178703f));
  y = fma2(y, r, make_float2(0.240247443f, 0.240247443f));
  y = fma2(y, r, make_float2(0.693121791f, 0.693121791f));
  y = fma2(y, r, make_float2(0.999999285f, 0.999999285f));
  y.x = __int_as_float(__float_as_int(y.x) + (__float_as_int(t.x) << 23));
  y.y = __int_as_float(__float_as_int(y.y) + (__float_as_int(t.y) << 23));
  return y;
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}
__device__ __forceinline__ bool odd_bits(uint32_t w) {
  return (w & 0x7f800000u) == 0x7f800000u || (w & 0x7f80u) == 0x7f80u;
}

// TWO: two query tiles, both groups on every key tile; else one, groups on alternate tiles.
template <int HD, bool TWO>
struct WideShape {
  static constexpr int QT = TWO ? 2 : 1;
  static constexpr int QBYTES = kRows * HD * 2;
  static constexpr int SLOT = kKeys * HD * 2;
  static constexpr int NS = HD == 128 && TWO ? 10 : 12;
  static constexpr int XROW = HD + 4;  // floats of a row of the joining area (in the ring)
  static constexpr int BARS = (3 * kMaxSlots + 12) * 8;
  static constexpr size_t SMEM = 1024 + (size_t)QT * QBYTES + (size_t)NS * SLOT + BARS + 64;
  static_assert(NS <= kMaxSlots, "ring");
  static_assert(NS * SLOT >= kRows * (XROW + 2) * 4, "joining area");
  static_assert(SMEM <= 232448, "shared memory");
};

template <int HD, bool TWO, bool FP8>
__global__ void __launch_bounds__(threads_of(FP8), 1)
tree_attn_wide_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, TreeParams p) {
  using W = WideShape<HD, TWO>;
  constexpr int NS = W::NS;
  extern __shared__ uint8_t raw_smem[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw_smem) + 1023) & ~uintptr_t(1023));
  uint8_t* q_smem = smem;
  uint8_t* ring = smem + W::QT * W::QBYTES;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + (size_t)NS * W::SLOT);
  uint64_t* full = bars;                     // a slot's TMA bytes have landed
  uint64_t* ready = bars + kMaxSlots;        // by special V tile (mod NK): the V warp has been over it
  uint64_t* empty = bars + 2 * kMaxSlots;    // the products that read it are done
  uint64_t* s_ready = bars + 3 * kMaxSlots;  // by group and S buffer: S is complete
  uint64_t* p_ready = s_ready + 4;           // likewise: P is in tensor memory (one arrival a warp)
  uint64_t* pv_done = s_ready + 8;           // by group: its last P V is in O
  uint64_t* o_ready = s_ready + 10;          // by group: O is complete
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 3 * kMaxSlots + 12);
  int* odd = reinterpret_cast<int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  grid_dep_wait();

  const int bh = blockIdx.x, c = blockIdx.y, qtile = blockIdx.z;
  const int b = bh / p.nkv, h = bh % p.nkv;
  const int ctx = p.ctx_lens[b], ql = p.q_lens[b], qoff = p.q_offsets[b];
  if (ql < 0 || ql > p.max_q || ctx < ql || qoff < 0 || qoff > p.q_rows - ql || (int64_t)ctx > (int64_t)p.table_stride * p.bs ||
      (int64_t)ctx > (int64_t)p.chunk * p.n_chunks) {
    if (threadIdx.x == 0 && c == 0 && qtile == 0) report(p.status, KVE_ERR_BOUNDS);
    return;
  }
  const int row0 = qtile * W::QT * kRows;
  const int rows = min(W::QT * kRows, ql * p.group - row0);
  if (rows <= 0) return;
  const int hist = ctx - ql;
  const int key_end = p.mask ? ctx : hist + (row0 + rows - 1) / p.group + 1;
  const int live = (key_end + p.chunk - 1) / p.chunk;
  if (c >= live) return;
  const int key_lo = c * p.chunk;
  const int key_hi = min(key_end, key_lo + p.chunk);
  const int n = (key_hi - key_lo + kKeys - 1) / kKeys;  // key tiles
  // Steps of group g, and the key tile of its step i.
  const int steps0 = TWO ? n : (n + 1) / 2, steps1 = TWO ? (rows > kRows ? n : 0) : n / 2;
  auto steps = [&](int g) { return g ? steps1 : steps0; };
  auto tile_of = [&](int g, int i) { return TWO ? i : 2 * i + g; };
  // Tiles from here on have keys that are new tokens or lie behind the last key.
  const int special = max(0, min(hist - key_lo, key_hi - key_lo)) / kKeys;

  if (threadIdx.x == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(smem_u32(&full[i]), FP8 ? 2 : 1);  // e4m3: the two warps that copy its tiles
      mbar_init(smem_u32(&ready[i]), FP8 ? 2 : 1);
      mbar_init(smem_u32(&empty[i]), TWO && steps1 > 0 ? 2 : 1);  // one commit of each group that reads it
    }
    for (int g = 0; g < 2; ++g) {
      mbar_init(smem_u32(&s_ready[2 * g]), 1);
      mbar_init(smem_u32(&s_ready[2 * g + 1]), 1);
      mbar_init(smem_u32(&p_ready[2 * g]), 4);
      mbar_init(smem_u32(&p_ready[2 * g + 1]), 4);
      mbar_init(smem_u32(&pv_done[g]), 1);
      mbar_init(smem_u32(&o_ready[g]), 1);
    }
    *odd = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if constexpr (!FP8) {
      prefetch_map(&map_k);
      prefetch_map(&map_v);
    }
  }
  __syncthreads();  // the barriers are there: the copies may start
  // K tile t lies in slot t mod NK, V tile t in slot NK + t mod NK; each slot has its barriers.
  constexpr int NK = NS / 2;
  auto slot_of = [&](bool v, int t) { return (v ? NK : 0) + t % NK; };
  auto slot_addr = [&](bool v, int t) { return smem_u32(ring) + (uint32_t)(slot_of(v, t) * W::SLOT); };
  auto parity_of = [&](int t) { return (uint32_t)(t / NK) & 1u; };
  bool ok = true;  // no wait of this thread has run out

  if (warp == 3) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    grid_dep_launch();  // not before: a dependent's CTA here may hold columns and wait for this one
  }
  const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(p.q);
  auto head_row = [&](int r) {  // row r of the CTA in q and out
    const int gr = row0 + r, node = node_of(p, gr);
    return ((size_t)(qoff + node) * p.nq + h * p.group + gr - node * p.group) * HD;
  };
  if (warp >= 4 && warp < 12) {
    // Q into shared memory, 16 bytes a lane; a negative scale is a sign on q.
    const uint32_t flip = p.scale < 0.f ? 0x80008000u : 0u;
    // TWO: each group its own tile; else half of the one
    constexpr int PER = kRows * (HD / 8) / (TWO ? 128 : 256);
    const int first = TWO ? threadIdx.x & 127 : threadIdx.x - 128, tile = TWO ? (threadIdx.x - 128) / 128 : 0;
    uint4 x[PER];
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int i = first + u * (TWO ? 128 : 256), r = tile * kRows + i / (HD / 8);
      x[u] = r < rows ? *reinterpret_cast<const uint4*>(q + head_row(r) + i % (HD / 8) * 8) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      const int i = first + u * (TWO ? 128 : 256), r = i / (HD / 8), ch = i % (HD / 8);
      x[u].x ^= flip;
      x[u].y ^= flip;
      x[u].z ^= flip;
      x[u].w ^= flip;
      *reinterpret_cast<uint4*>(q_smem + tile * W::QBYTES + (ch / 8) * (kRows * 128) + r * 128 + (((ch % 8) ^ (r & 7)) << 4)) = x[u];
    }
    fence_proxy_async_smem();
  }
  uint32_t tmem = 0;
  if (warp != 0 && warp < 12) {  // Q and tensor memory are there
    tc_before();
    asm volatile("bar.sync 2, 352;" ::: "memory");
    tc_after();
    tmem = *tmem_slot;
  }
  auto s_col = [&](int g, int i) { return tmem + (uint32_t)(g * 128 + (i & 1) * kKeys); };
  auto o_col = [&](int g) { return tmem + (uint32_t)(256 + g * 128); };

  float m = -INFINITY, l = 0.f;  // softmax threads: the row's base and its sum
  const int grp = warp >= 8 ? 1 : 0, row = (warp & 3) * 32 + lane;
  // The first pool rows of the tiles' groups of 16 keys, lane l knowing group 32 w + l (past the end: a
  // row behind the pool, which loads as zeros).
  auto rows_of = [&](int w, bool tell) {
    const int key = key_lo + (w * 32 + lane) * 16;
    int y = (int)(p.num_blocks * p.bs);
    if (key < key_hi) {
      const int blk = p.tables[(size_t)b * p.table_stride + key / p.bs];
      if (blk >= 0 && blk < p.num_blocks) y = blk * p.bs + key % p.bs;
      else if (tell) report(p.status, KVE_ERR_BOUNDS);
    }
    return y;
  };
  // e4m3: two warps copy K and two V, 32 of a tile's keys each, through their registers into the places
  // where TMA puts bf16 tiles, as the bf16 numbers they stand for; when a tile is written the next
  // one's bytes are on their way and those after it are asked for. (One warp for all of K or V: 432 us where
  // this takes 261; a third pair gains nothing, nor do loads that pass L1 by.)
  auto copy_fp8 = [&](auto is_v, int half) {
    constexpr bool v = decltype(is_v)::value;
    constexpr int PIECES = HD / 16, PER = PIECES;  // 16-byte pieces of a key; a lane's, of a tile
    constexpr int AT_ONCE = 32 / PIECES;           // keys of one load
    const uint8_t* pool = static_cast<const uint8_t*>(v ? p.pool_v : p.pool_k) + (size_t)h * HD + lane % PIECES * 16;
    const uint8_t* scales = (v ? p.v_scale : p.k_scale) + h;
    const int32_t* table = p.tables + (size_t)b * p.table_stride;
    const uint32_t row_bytes = (uint32_t)(p.nkv * HD);
    // Where the lane's pieces go in a slot: load u's key is AT_ONCE u further, its two halves (8 elements
    // each) in the columns that the key's last three bits swizzle.
    const int r0 = lane / PIECES, piece0 = lane % PIECES * 2;
    const uint32_t place = (uint32_t)(v ? half * (32 * HD * 2) + piece0 / 8 * 2048 : piece0 / 8 * (kKeys * 128) + half * 4096) + r0 * 128;
    uint4 bytes[2][PER];
    uint32_t byte[2];  // the exponent of this lane's key
    int slots[2];      // its slot in the pool (-1: the key is not there)
    bool found = false;
    // The key's block and place in it, for the tile whose block id is asked for.
    int key = key_lo + 32 * half + lane, blk = key / p.bs, in = key - blk * p.bs;
    const int step_blk = kKeys / p.bs, step_in = kKeys - step_blk * p.bs;
    int id = -1, id_in = 0;
    bool id_key = false;
    auto ask_id = [&] {
      id_key = (uint32_t)key < (uint32_t)key_hi;  // past 2^31 is past the end
      id = id_key ? table[blk] : -1;
      id_in = in;
      key += kKeys;
      blk += step_blk;
      in += step_in;
      if (in >= p.bs) {
        in -= p.bs;
        ++blk;
      }
    };
    auto ask = [&](int at) {  // the bytes and exponents of the tile whose block ids have come
      int slot = -1;
      uint32_t e = 0;
      if (id >= 0 && id < p.num_blocks) {
        slot = id * p.bs + id_in;
        e = scales[(size_t)slot * p.nkv];
      } else if (!v && id_key) {
        report(p.status, KVE_ERR_BOUNDS);  // reads as zeros
      }
      byte[at] = e;
      slots[at] = slot;
      slot = max(slot, 0);
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        const uint32_t sl = __shfl_sync(0xffffffffu, slot, u * AT_ONCE + r0);
        bytes[at][u] = *reinterpret_cast<const uint4*>(pool + (uint64_t)sl * row_bytes);
      }
      ask_id();
    };
    ask_id();
    ask(0);
    if (n > 1) ask(1);
    auto tile = [&](int t, auto which) {
      constexpr int at = decltype(which)::value;  // t mod 2
      const uint4(&now)[PER] = bytes[at];
      // A byte's exponent and mantissa, put where bf16 has the low bits of its exponent and
      // the top of its mantissa, are the number times 2^-120, subnormals included: one product
      // with 2^(e - 127 + 120) makes it the bf16 that it stands for. Not where that power
      // is no bf16, nor for NaN bytes, nor where keys are missing: such a tile goes the slow way.
      uint32_t nan = 0;
#pragma unroll
      for (int u = 0; u < PER; ++u) {
        nan |= ((now[u].x & 0x7f7f7f7fu) + 0x01010101u) | ((now[u].y & 0x7f7f7f7fu) + 0x01010101u);
        nan |= ((now[u].z & 0x7f7f7f7fu) + 0x01010101u) | ((now[u].w & 0x7f7f7f7fu) + 0x01010101u);
      }
      const uint32_t e = byte[at];
      const int slot = slots[at];
      if (t >= NK) ok = ok && mbar_wait(smem_u32(&empty[slot_of(v, t)]), parity_of(t - NK), p.status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) return;
      uint8_t* to = ring + (size_t)slot_of(v, t) * W::SLOT + place;
      auto store = [&](int u, const uint32_t (&o)[8]) {
        const int r = u * AT_ONCE;
        uint8_t* dst = to + (v ? r / 16 * (16 * HD * 2) + r % 16 * 128 : r * 128);
#pragma unroll
        for (int j = 0; j < 2; ++j)
          *reinterpret_cast<uint4*>(dst + (((piece0 + j) % 8 ^ (r + r0 & 7)) << 4)) =
              make_uint4(o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]);
      };
      if (__any_sync(0xffffffffu, (nan & 0x80808080u) != 0 || e > 134 || slot < 0)) {
        const float mine = scale_value(e);
#pragma unroll 1
        for (int u = 0; u < PER; ++u) {
          const int from = u * AT_ONCE + r0;
          const float up = __shfl_sync(0xffffffffu, mine, from);
          const int sl = __shfl_sync(0xffffffffu, slot, from);
          uint4 x = make_uint4(0u, 0u, 0u, 0u);
          if (sl >= 0) x = *reinterpret_cast<const uint4*>(pool + (uint64_t)(uint32_t)sl * row_bytes);
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
          uint32_t o[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const __half2_raw two = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i / 2] >> (i % 2 * 16)), __NV_E4M3);
            const float2 f = __half22float2(__half2(two));
            o[i] = pack2(f.x * up, f.y * up);
          }
          store(u, o);
        }
      } else {
        const uint32_t mine = ((e + 120) << 7) * 0x10001u;
#pragma unroll
        for (int u = 0; u < PER; ++u) {
          const uint32_t up = __shfl_sync(0xffffffffu, mine, u * AT_ONCE + r0);
          const uint32_t w[4] = {now[u].x, now[u].y, now[u].z, now[u].w};
          uint32_t o[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t x = __byte_perm(w[i / 2], 0, i % 2 ? 0x3424 : 0x1404);
            const uint32_t y = (x & 0x80008000u) | (x >> 4 & 0x07f007f0u);
            const __nv_bfloat162 z = __hmul2(reinterpret_cast<const __nv_bfloat162&>(y), reinterpret_cast<const __nv_bfloat162&>(up));
            o[i] = reinterpret_cast<const uint32_t&>(z);
          }
          store(u, o);
        }
      }
      if (t + 2 < n) ask(at);
      if (v && t >= special) {  // infinities and NaN in new tokens' rows: this lane's own pieces, as stored
#pragma unroll 1
        for (int u = 0; u < PER; ++u) {
          const int r = u * AT_ONCE, at_key = key_lo + t * kKeys + 32 * half + r + r0;
          const uint8_t* src = to + r / 16 * (16 * HD * 2) + r % 16 * 128;
          if (at_key >= hist && at_key < key_hi) {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              const uint4 x = *reinterpret_cast<const uint4*>(src + (((piece0 + j) % 8 ^ (r + r0 & 7)) << 4));
              found |= odd_bits(x.x) || odd_bits(x.y) || odd_bits(x.z) || odd_bits(x.w);
            }
          }
        }
        if (__any_sync(0xffffffffu, found) && lane == 0) *odd = 1;
      }
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(v && t >= special ? &ready[(t - special) % NK] : &full[slot_of(v, t)]));
    };
    for (int t = 0; t < n && ok; t += 2) {
      tile(t, std::integral_constant<int, 0>());
      if (t + 1 < n && ok) tile(t + 1, std::integral_constant<int, 1>());
    }
  };
  if (FP8 && (warp == 0 || warp >= 12)) {
    if constexpr (FP8) {
      if (warp >= 12 && (warp & 1)) copy_fp8(std::true_type(), (warp >> 1) & 1);
      else if (warp >= 12) copy_fp8(std::false_type(), (warp >> 1) & 1);
    }
  } else if (warp == 0) {
    // ---- K: boxes of 16 keys x 64 dims
    const uint32_t lead = elect_lane();
    int now = rows_of(0, true), next = rows_of(1, true);
    for (int t = 0; t < n; ++t) {
      if (t > 0 && t % 8 == 0) {
        now = next;
        next = rows_of(t / 8 + 1, true);
      }
      const uint32_t bar = smem_u32(&full[slot_of(false, t)]);
      if (t >= NK) ok = ok && mbar_wait(smem_u32(&empty[slot_of(false, t)]), parity_of(t - NK), p.status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        for (int u = t - NK; u < t; ++u) mbar_wait(smem_u32(&full[slot_of(false, u)]), parity_of(u), p.status);  // in flight
        break;
      }
      if (lead) mbar_expect_tx(bar, W::SLOT);
      __syncwarp();
#pragma unroll
      for (int part = 0; part < kKeys / 16; ++part) {
        const int y = __shfl_sync(0xffffffffu, now, t % 8 * 4 + part);
#pragma unroll
        for (int half = 0; half < HD / 64; ++half)
          tma_load(lead, slot_addr(false, t) + half * (kKeys * 128) + part * 2048, &map_k, h * HD + half * 64, y, bar);
      }
    }
  } else if (warp <= 2) {
    // ---- products of one group. (One warp for both took 2350 cycles a step with its waits, whatever
    // the products and the softmax cost.)
    const int g = warp - 1, my_steps = steps(g);
    const uint32_t lead = elect_lane();
    const uint32_t id_qk = mma_idesc(kKeys, false), id_pv = mma_idesc(HD, true);
    const uint64_t ad = desc_k_major(smem_u32(q_smem) + (TWO ? g * W::QBYTES : 0));
    auto qk = [&](int i) {
      const int t = tile_of(g, i), slot = slot_of(false, t);
      ok = __all_sync(0xffffffffu, ok && mbar_wait(smem_u32(&full[slot]), parity_of(t), p.status));
      if (!ok) return;
      tc_after();
      const uint64_t bd = desc_k_major(slot_addr(false, t));
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        const uint64_t a_step = (uint64_t)((kk / 4) * (kRows * 128 / 16) + (kk % 4) * 2);
        const uint64_t b_step = (uint64_t)((kk / 4) * (kKeys * 128 / 16) + (kk % 4) * 2);
        mma_ss(lead, s_col(g, i), ad + a_step, bd + b_step, id_qk, kk > 0);
      }
      mma_commit(lead, smem_u32(&empty[slot]));
      mma_commit(lead, smem_u32(&s_ready[2 * g + (i & 1)]));
    };
    for (int i = 0; i < 2 && i < my_steps && ok; ++i) qk(i);
    for (int i = 0; i < my_steps && ok; ++i) {
      const int t = tile_of(g, i), slot = slot_of(true, t);
      ok = t >= special ? mbar_wait(smem_u32(&ready[(t - special) % NK]), parity_of(t - special), p.status)
                        : mbar_wait(smem_u32(&full[slot]), parity_of(t), p.status);
      ok = ok && mbar_wait(smem_u32(&p_ready[2 * g + (i & 1)]), (uint32_t)(i / 2) & 1u, p.status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_after();
      const uint64_t bd = desc_mn_major(slot_addr(true, t), 2048);
#pragma unroll
      for (int kk = 0; kk < kKeys / 16; ++kk)
        mma_ts(lead, o_col(g), s_col(g, i) + kk * 8, bd + (uint64_t)(kk * (16 * HD * 2 / 16)), id_pv, i > 0 || kk > 0);
      mma_commit(lead, smem_u32(&empty[slot]));
      mma_commit(lead, smem_u32(&pv_done[g]));
      if (i + 1 == my_steps) mma_commit(lead, smem_u32(&o_ready[g]));
      else if (i + 2 < my_steps) qk(i + 2);
    }
    if (!ok) {  // end what was issued before the memory it uses goes away
      mma_commit(lead, smem_u32(&o_ready[g]));
      mbar_wait(smem_u32(&o_ready[g]), 0, p.status);
    }
    __syncwarp();
  } else if (warp == 3) {
    // ---- V: boxes of 16 keys x all dims (a product takes 16 keys: their halves may lie 2 KB apart).
    // Special tiles: zero the rows behind the last key, look for infinities and NaN in new tokens' rows.
    auto look = [&](int t) {
      ok = __all_sync(0xffffffffu, ok && mbar_wait(smem_u32(&full[slot_of(true, t)]), parity_of(t), p.status));
      if (!ok) return;
      const int kt = key_lo + t * kKeys;
      uint8_t* v = ring + (size_t)slot_of(true, t) * W::SLOT;
      auto piece = [&](int r, int i) {  // 16 bytes i of row r, in any order
        return reinterpret_cast<uint4*>(v + (r / 16) * (16 * HD * 2) + (i / 8) * 2048 + (r % 16) * 128 + i % 8 * 16);
      };
      constexpr int PIECES = HD / 8;
      if (kt + kKeys > key_hi) {
        const int first = key_hi - kt, stop = min(kKeys, (first + 15) / 16 * 16);  // further boxes are zeros already
        for (int i = lane; i < (stop - first) * PIECES; i += 32) *piece(first + i / PIECES, i % PIECES) = make_uint4(0u, 0u, 0u, 0u);
        fence_proxy_async_smem();
      }
      const int r0 = max(hist - kt, 0), r1 = min(kKeys, key_hi - kt);
      bool found = false;
      for (int i = lane; i < (r1 - r0) * PIECES; i += 32) {
        const uint4 x = *piece(r0 + i / PIECES, i % PIECES);
        found |= odd_bits(x.x) || odd_bits(x.y) || odd_bits(x.z) || odd_bits(x.w);
      }
      if (__any_sync(0xffffffffu, found) && lane == 0) *odd = 1;
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&ready[(t - special) % NK]));
    };
    const uint32_t lead = elect_lane();
    int now = rows_of(0, false), next = rows_of(1, false), looked = special;
    for (int t = 0; t < n && !FP8; ++t) {
      if (t > 0 && t % 8 == 0) {
        now = next;
        next = rows_of(t / 8 + 1, false);
      }
      const uint32_t bar = smem_u32(&full[slot_of(true, t)]);
      while (ok && looked <= t - NK) look(looked++);  // their products free the slots
      if (t >= NK) ok = ok && mbar_wait(smem_u32(&empty[slot_of(true, t)]), parity_of(t - NK), p.status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        for (int u = max(0, t - NK); u < t; ++u) mbar_wait(smem_u32(&full[slot_of(true, u)]), parity_of(u), p.status);
        break;
      }
      if (lead) mbar_expect_tx(bar, W::SLOT);
      __syncwarp();
#pragma unroll
      for (int part = 0; part < kKeys / 16; ++part) {
        const int y = __shfl_sync(0xffffffffu, now, t % 8 * 4 + part);
        tma_load_v(lead, slot_addr(true, t) + part * (16 * HD * 2), &map_v, y, h * (HD / 64), bar);
      }
      if (looked < t && __all_sync(0xffffffffu, mbar_try_wait(smem_u32(&full[slot_of(true, looked)]), parity_of(looked))))
        look(looked++);
    }
    while (!FP8 && ok && looked < n) look(looked++);
  } else if (warp >= 4) {
    // ---- softmax: a thread a row
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    const int r = (TWO ? grp * kRows : 0) + row;  // row of the CTA
    const bool active = (TWO ? grp * kRows : 0) + (warp & 3) * 32 < rows;  // any row of this warp
    const int node = node_of(p, row0 + min(r, rows - 1));
    const uint32_t* mask = p.mask ? p.mask + (size_t)(qoff + node) * p.mask_words : nullptr;
    const float sl = fmaxf(fabsf(p.scale) * 1.4426950408889634f, FLT_MIN);  // not 0: 0 x -infinity is no mask
    const int my_steps = steps(grp);
    // One tile: m and l, and P over S. `masked`: some of the tile's keys are new tokens or
    // lie behind the last key.
    auto softmax_step = [&](int i, int kt, auto masked) {
      const uint32_t sc = s_col(grp, i) + lanes;
      uint32_t see[kKeys / 32];
      if constexpr (masked) {
#pragma unroll
        for (int w = 0; w < kKeys / 32; ++w) {
          const int at = kt + 32 * w;
          see[w] = p.mask ? mask_bits<32>(mask, p.mask_words, at - hist) : chain_bits(node, at - hist);
          const int in = key_hi - at;
          see[w] &= in >= 32 ? ~0u : in <= 0 ? 0u : (1u << in) - 1u;
        }
      }
      float v[kKeys / 32][32];  // the row of S stays in registers
#pragma unroll
      for (int w = 0; w < kKeys / 32; ++w) tmem_ask(sc + 32 * w, v[w]);
      float top = -INFINITY;
#pragma unroll
      for (int w = 0; w < kKeys / 32; ++w) {
        tmem_arrived(v[w]);
        if constexpr (masked) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[w][j] = see[w] >> j & 1 ? v[w][j] : -INFINITY;
        }
        float part[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          part[j] = max3(v[w][j], v[w][j + 4], v[w][j + 8]);
          part[j] = max3(part[j], v[w][j + 12], v[w][j + 16]);
          part[j] = max3(part[j], v[w][j + 20], v[w][j + 24]);
          part[j] = max2(part[j], v[w][j + 28]);
        }
        top = max3(top, max3(part[0], part[1], part[2]), part[3]);
      }
      top *= sl;
      const bool grow = !(top <= m + 8.f);  // or NaN
      if (__any_sync(0xffffffffu, grow)) {
        // A score of NaN, or infinity, which 2^(inf - inf) is too, makes the row NaN here: ex2_fma would not.
        if (grow) top += 0.f * top;
        const float f = grow ? ex2(m - top) : 1.f;
        if (grow) m = top;
        l *= f;
        if (i > 0) {
          ok = ok && mbar_wait(smem_u32(&pv_done[grp]), (uint32_t)(i - 1) & 1u, p.status);  // O is not being added to
          __syncwarp();
          tc_after();
#pragma unroll 1
          for (int w = 0; w < HD / 32; ++w) {
            float o[32];
            tmem_load(o_col(grp) + lanes + 32 * w, o);
#pragma unroll
            for (int j = 0; j < 32; ++j) o[j] *= f;
            tmem_store32(o_col(grp) + lanes + 32 * w, o);
          }
        }
      }
      const float off = m == -INFINITY ? 0.f : -m;
      const float2 sl2 = make_float2(sl, sl), off2 = make_float2(off, off);
      float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
      for (int w = 0; w < kKeys / 32; ++w) {
        uint32_t packed[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          float2 e = fma2(make_float2(v[w][2 * j], v[w][2 * j + 1]), sl2, off2);
          if (!masked && j % kShare == kShare - 1) {
            e = ex2_fma(e);
          } else {
            e.x = ex2(e.x);
            e.y = ex2(e.y);
          }
          sum[j & 1] = add2(sum[j & 1], e);
          packed[j] = pack2(e.x, e.y);
        }
        tmem_store16(sc + 16 * w, packed);  // over S
      }
      sum[0] = add2(sum[0], sum[1]);
      l += sum[0].x + sum[0].y;
    };
    for (int i = 0; i < my_steps; ++i) {
      ok = ok && mbar_wait(smem_u32(&s_ready[2 * grp + (i & 1)]), (uint32_t)(i / 2) & 1u, p.status);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (active) {
        tc_after();
        const int kt = key_lo + tile_of(grp, i) * kKeys;
        if (kt + kKeys > hist || kt + kKeys > key_hi) softmax_step(i, kt, std::true_type());
        else softmax_step(i, kt, std::false_type());
        tmem_store_wait();
      }
      tc_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&p_ready[2 * grp + (i & 1)]));
    }
    if (my_steps > 0) ok = ok && mbar_wait(smem_u32(&o_ready[grp]), 0, p.status);
    tc_after();
    if (m == -INFINITY) l = 0.f;  // no score but minus infinity: ex2_fma's 2^-126 are no weights
  }
  // Every role is done; a wait that ran out anywhere leaves the outputs unwritten.
  const bool failed = __syncthreads_or(!ok);

  constexpr int PROW = HD + 4;
  constexpr int TILE_ROWS = W::QT * kRows;
  float* part0 = p.partials + ((size_t)bh * p.n_qtiles + qtile) * p.n_chunks * TILE_ROWS * PROW;
  float* part = part0 + (size_t)c * TILE_ROWS * PROW;
  __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out);
  float* xs = reinterpret_cast<float*>(ring);  // the second group's rows: O, then m and l
  const bool recompute = *odd != 0;
  if (!failed && !recompute && warp >= 4 && warp < 12) {
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    float* xr = xs + (size_t)row * W::XROW;
    float* xml = xs + (size_t)kRows * W::XROW + row * 2;
    float v[32];
    if (!TWO && grp == 1) {
      // hand over to the first group
      if (steps1 > 0 && (warp & 3) * 32 < rows) {
#pragma unroll 1
        for (int w = 0; w < HD / 32; ++w) {
          tmem_load(o_col(1) + lanes + 32 * w, v);
#pragma unroll
          for (int x = 0; x < 32; x += 4)
            *reinterpret_cast<float4*>(xr + 32 * w + x) = make_float4(v[x], v[x + 1], v[x + 2], v[x + 3]);
        }
      }
      *reinterpret_cast<float2*>(xml) = make_float2(m, l);
      asm volatile("bar.sync 1, 256;" ::: "memory");
    } else {
      float f0 = 1.f, f1 = 0.f;
      if (!TWO) {
        asm volatile("bar.sync 1, 256;" ::: "memory");
        const float2 ml = *reinterpret_cast<const float2*>(xml);
        const float t = fmaxf(m, ml.x);
        f0 = m == t ? 1.f : ex2(m - t);
        f1 = ml.x == t ? 1.f : ex2(ml.x - t);
        m = t;
        l = l * f0 + ml.y * f1;
      }
      const int r = (TWO ? grp * kRows : 0) + row;
      if ((TWO ? grp * kRows : 0) + (warp & 3) * 32 < rows) {
        const bool join = !TWO && steps1 > 0;
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll 1
        for (int w = 0; w < HD / 32; ++w) {
          tmem_load(o_col(TWO ? grp : 0) + lanes + 32 * w, v);
          if (join) {
#pragma unroll
            for (int x = 0; x < 32; x += 4) {
              const float4 y = *reinterpret_cast<const float4*>(xr + 32 * w + x);
              v[x] = v[x] * f0 + y.x * f1;
              v[x + 1] = v[x + 1] * f0 + y.y * f1;
              v[x + 2] = v[x + 2] * f0 + y.z * f1;
              v[x + 3] = v[x + 3] * f0 + y.w * f1;
            }
          }
          if (live == 1) {
            // to shared memory (Q is no longer needed), 16-byte pieces exchanged by row
            uint8_t* dst = q_smem + (size_t)r * (HD * 2);
#pragma unroll
            for (int x = 0; x < 32; x += 8) {
              uint4 o;
              o.x = pack2(l == 0.f ? 0.f : v[x] * inv, l == 0.f ? 0.f : v[x + 1] * inv);
              o.y = pack2(l == 0.f ? 0.f : v[x + 2] * inv, l == 0.f ? 0.f : v[x + 3] * inv);
              o.z = pack2(l == 0.f ? 0.f : v[x + 4] * inv, l == 0.f ? 0.f : v[x + 5] * inv);
              o.w = pack2(l == 0.f ? 0.f : v[x + 6] * inv, l == 0.f ? 0.f : v[x + 7] * inv);
              *reinterpret_cast<uint4*>(dst + (((w * 4 + x / 8) ^ (r & 7)) << 4)) = o;
            }
          } else if (r < rows) {
            float* dst = part + (size_t)r * PROW + 32 * w;
#pragma unroll
            for (int x = 0; x < 32; x += 4)
              *reinterpret_cast<float4*>(dst + x) = make_float4(v[x], v[x + 1], v[x + 2], v[x + 3]);
          }
          __syncwarp();  // the loads of tensor memory are the whole warp's
        }
        if (live > 1 && r < rows) *reinterpret_cast<float2*>(part + (size_t)r * PROW + HD) = make_float2(m, l);
        if (live == 1) {
          // this warp's 32 rows, whole rows at a time
          const int r0 = (TWO ? grp * kRows : 0) + (warp & 3) * 32;
          constexpr int PIECES = HD / 8, AT_ONCE = 32 / PIECES;
#pragma unroll 4
          for (int rr = lane / PIECES; rr < 32; rr += AT_ONCE) {
            const int ro = r0 + rr, piece = lane % PIECES;
            if (ro < rows)
              *reinterpret_cast<uint4*>(out + head_row(ro) + piece * 8) =
                  *reinterpret_cast<const uint4*>(q_smem + (size_t)ro * (HD * 2) + ((piece ^ (ro & 7)) << 4));
          }
        }
      }
    }
  }
  if (!failed && recompute) {
    attend_by_key<__nv_bfloat16, FP8, HD, threads_of(FP8)>(p, b, h, qoff, hist, key_lo, key_hi, row0, rows, warp, lane,
                                                           live > 1, part);
  }
  tc_before();
  __threadfence();
  __syncthreads();
  if (warp == 3) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
  if (live == 1) return;

  // The last of the tile's chunks to arrive joins them, in chunk order.
  int* last = odd;  // its value has been read by all
  if (threadIdx.x == 0) {
    int* cnt = p.counters + (size_t)bh * p.n_qtiles + qtile;
    *last = atomicAdd(cnt, 1) == live - 1;
    if (*last) *cnt = 0;  // the workspace is left as it was
  }
  __syncthreads();
  if (!*last || failed) return;
  __threadfence();
  for (int i = threadIdx.x; i < rows * (HD / 4); i += threads_of(FP8)) {
    const int r = i / (HD / 4), d = i % (HD / 4) * 4;
    const float* pr = part0 + (size_t)r * PROW;
    float rm = -INFINITY, rl = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = 0; s < live; ++s) {
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(pr + (size_t)s * TILE_ROWS * PROW + HD));
      const float4 x = __ldcg(reinterpret_cast<const float4*>(pr + (size_t)s * TILE_ROWS * PROW + d));
      const float t = fmaxf(rm, ml.x);
      const float f = t == rm ? 1.f : ex2(rm - t), w = t == ml.x ? 1.f : ex2(ml.x - t);
      rm = t;
      rl = rl * f + ml.y * w;
      o.x = o.x * f + x.x * w;
      o.y = o.y * f + x.y * w;
      o.z = o.z * f + x.z * w;
      o.w = o.w * f + x.w * w;
    }
    const bool none = rl == 0.f;
    *reinterpret_cast<uint2*>(out + head_row(r) + d) =
        make_uint2(pack2(none ? 0.f : o.x / rl, none ? 0.f : o.y / rl), pack2(none ? 0.f : o.z / rl, none ? 0.f : o.w / rl));
  }
}

// ------------------------------------------------------------------ host
struct WidePlan {
  bool two;
  int n_qtiles, chunk, n_chunks;
};

// One or two query tiles a CTA by the rows of the call's largest tree, and the number
// of chunks that costs least: waves of one CTA an SM, each a fixed part (launch, Q,
// the first tile's latency, joining: about 5 us) and a part per step (about 0.7 us).
WidePlan wide_plan(int batch, int max_q, int max_ctx, int nkv, int group) {
  WidePlan w;
  const long long rows = (long long)max_q * group;
  w.two = rows > kRows;
  const int per = (w.two ? 2 : 1) * kRows;
  w.n_qtiles = (int)((rows + per - 1) / per);
  const long long units = (long long)batch * nkv * w.n_qtiles;
  const int tiles = (max_ctx + kKeys - 1) / kKeys;
  double best = 1e30;
  w.chunk = tiles * kKeys;
  w.n_chunks = 1;
  for (int c = 1; c <= tiles && c <= 32; ++c) {
    const int per_chunk = (tiles + c - 1) / c, chunks = (tiles + per_chunk - 1) / per_chunk;
    if (chunks != c || (c > 1 && units > (long long)kTreeCounterSlots)) continue;
    const int steps = w.two ? per_chunk : (per_chunk + 1) / 2;
    const double waves = (double)((units * c + 147) / 148);
    const double t = waves * (5.0 + 0.7 * steps) + (c > 1 ? 2.0 + 0.15 * c : 0.0);
    if (t < best) {
      best = t;
      w.chunk = per_chunk * kKeys;
      w.n_chunks = c;
    }
  }
  return w;
}

// One layer's pool as (64 dims, rows) with boxes of 16 rows, and, for V, as (64 dims, rows, dims / 64)
// with boxes of 16 rows and all of a head's dims.
bool pool_map(CUtensorMap* map, const void* pool, int64_t rows, int width, int hd, bool v) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t dims2[2] = {(cuuint64_t)width, (cuuint64_t)rows};
  cuuint64_t dims3[3] = {64, (cuuint64_t)rows, (cuuint64_t)width / 64};
  cuuint64_t strides[2] = {(cuuint64_t)width * 2, 128};
  cuuint32_t box[3] = {64, 16, (cuuint32_t)hd / 64};
  cuuint32_t estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, v ? 3 : 2, const_cast<void*>(pool), v ? dims3 : dims2, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int HD, bool TWO, bool FP8>
int launch(const TreeParams& p, const CUtensorMap& mk, const CUtensorMap& mv, int batch, cudaStream_t stream) {
  using W = WideShape<HD, TWO>;
  static std::atomic<uint64_t> prepared{0};  // the shared-memory limit is an attribute of the kernel on one device
  int dev = 0;
  cudaError_t err = cudaGetDevice(&dev);
  const uint64_t bit = 1ull << (dev & 63);
  if (err == cudaSuccess && !(prepared.load(std::memory_order_relaxed) & bit)) {
    err = cudaFuncSetAttribute(tree_attn_wide_kernel<HD, TWO, FP8>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)W::SMEM);
    if (err == cudaSuccess) prepared.fetch_or(bit, std::memory_order_relaxed);
  }
  if (err != cudaSuccess) {
    cudaGetLastError();
    return set_error(KVE_ERR_CUDA, "kve_paged_tree_attn: %s", cudaGetErrorString(err));
  }
  launch_kernel(tree_attn_wide_kernel<HD, TWO, FP8>, dim3(batch * p.nkv, p.n_chunks, p.n_qtiles), dim3(threads_of(FP8)), W::SMEM, stream,
                mk, mv, p);
  return check_launch("kve_paged_tree_attn(wide)");
}

}  // namespace

size_t tree_attn_wide_partial_bytes(int batch, int max_q, int max_ctx, int nkv, int group, int hd) {
  const WidePlan w = wide_plan(batch, max_q, max_ctx, nkv, group);
  if (w.n_chunks == 1) return 0;
  return (size_t)batch * nkv * w.n_qtiles * w.n_chunks * ((w.two ? 2 : 1) * kRows) * (hd + 4) * sizeof(float);
}

int tree_attn_wide(TreeParams p, int batch, int max_ctx, int hd, bool fp8, cudaStream_t stream) {
  const WidePlan w = wide_plan(batch, p.max_q, max_ctx, p.nkv, p.group);
  p.chunk = w.chunk;
  p.n_chunks = w.n_chunks;
  p.n_qtiles = w.n_qtiles;
  CUtensorMap mk, mv;
  memset(&mk, 0, sizeof(mk));
  memset(&mv, 0, sizeof(mv));
  const int64_t rows = p.num_blocks * p.bs;
  if (!fp8 && (!pool_map(&mk, p.pool_k, rows, p.nkv * hd, hd, false) || !pool_map(&mv, p.pool_v, rows, p.nkv * hd, hd, true)))
    return set_error(KVE_ERR_CUDA, "kve_paged_tree_attn: no tensor map for the pool");
  auto go = [&](auto f) {
    constexpr bool F = decltype(f)::value;
    if (hd == 64) return w.two ? launch<64, true, F>(p, mk, mv, batch, stream) : launch<64, false, F>(p, mk, mv, batch, stream);
    return w.two ? launch<128, true, F>(p, mk, mv, batch, stream) : launch<128, false, F>(p, mk, mv, batch, stream);
  };
  return fp8 ? go(std::true_type()) : go(std::false_type());
}

}  // namespace kve

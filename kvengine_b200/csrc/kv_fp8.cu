// The e4m3 cache: rows quantised as they are written, and read back.
//
// A row (one token, one kv head, K or V) x of head_dim elements is stored as
//   e = the least integer with max|x| <= 448 2^e (finite elements; 0 for a zero
//       row; at least -126),
//   q_d = x_d 2^-e rounded to the nearest e4m3 number, ties to even,
// q in the pool and e + 127 in a byte beside it. With a power of two as the
// scale nothing but that one rounding happens: x 2^-e is exact in fp32, q 2^e is
// exact in fp32, and in bf16 above 2^-126, and attention can use the exponent as it stands. An
// infinite or NaN element becomes NaN (e4m3 has no infinity).
//
// Every kernel gives one row to a group of lanes that hold 16 elements each, two
// runs of 8 half a row apart, so that a lane has both elements of its rotation pairs
// and the row's maximum is a shuffle or two away. All are bound by memory, or, for
// a decode step's few rows, by the launch. Measured: 16384 prompt tokens (16 / 2 heads of 128) written with
// RoPE and read back, two launches, 39 us (193 MB: 4.9 TB/s); 64 tokens, both launches in a replayed graph,
// 3.8 us (9.0 as two calls, which is their host time).
#include <cuda_fp8.h>
#include <math.h>

#include "kve_common.cuh"

namespace kve {
namespace {

constexpr int kThreads = 256;

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
    x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
  } else {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __bfloat1622float2(h[i]);
      x[2 * i] = f.x;
      x[2 * i + 1] = f.y;
    }
  }
}
// Eight elements as they are in memory.
template <typename T> struct Raw8;
template <> struct Raw8<__nv_bfloat16> {
  uint4 v;
};
template <> struct Raw8<float> {
  float4 v[2];
};
template <typename T>
__device__ __forceinline__ Raw8<T> raw8(const T* p) {
  return *reinterpret_cast<const Raw8<T>*>(p);
}
template <typename T>
__device__ __forceinline__ void open8(const Raw8<T>& r, float (&x)[8]) {
  load8(reinterpret_cast<const T*>(&r), x);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint4 v;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&v);
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = v;
  }
}

__device__ __forceinline__ float finite_size(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;
}
// 8 elements times 2^-e as e4m3 bytes.
__device__ __forceinline__ uint2 to_e4m3(const float (&x)[8], float down) {
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 f;
    f.x = fabsf(x[2 * i]) < INFINITY ? x[2 * i] * down : NAN;
    f.y = fabsf(x[2 * i + 1]) < INFINITY ? x[2 * i + 1] * down : NAN;
    w[i / 2] |= (uint32_t)__nv_cvt_float2_to_fp8x2(f, __NV_SATFINITE, __NV_E4M3) << (i % 2 * 16);
  }
  return make_uint2(w[0], w[1]);
}

// Quantise and store one row held by LANES lanes (lane `sub`: elements 8 sub .. and
// half a row further), the scale byte by the first.
template <int LANES>
__device__ __forceinline__ void store_row(const float (&a)[8], const float (&b)[8], int sub, uint8_t* row, uint8_t* scale,
                                          bool write) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, fmaxf(finite_size(a[i]), finite_size(b[i])));
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  // top = 1.f 2^k: 448 = 1.75 2^8, so e = k - 8, one more where f > 0.75. A subnormal
  // top (k below -126) ends at the least e as well.
  const uint32_t bits = __float_as_uint(top);
  int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u);
  e = top == 0.f ? 0 : max(e, -126);
  if (!write) return;
  const float down = __uint_as_float((uint32_t)(127 - e) << 23);
  *reinterpret_cast<uint2*>(row + sub * 8) = to_e4m3(a, down);
  *reinterpret_cast<uint2*>(row + LANES * 8 + sub * 8) = to_e4m3(b, down);
  if (sub == 0) *scale = (uint8_t)(e + 127);
}

struct Fp8Pool {
  uint8_t* k;
  uint8_t* v;
  uint8_t* k_scale;
  uint8_t* v_scale;
  int64_t num_slots;
};

// Rotate q and k, store q, quantise and store k and v; rotation in fp32, rounded once on its
// way out. A group of LANES lanes takes one head of a token (heads of q, k and v counted
// through). 16384 tokens of 16 + 2 x 2 heads of 128 (160 MB): 33 us at 2048 threads an SM, 40 at the
// 1280 that the compiler's choice of registers leaves; groups of two to five heads that read the
// angles once take 37 to 44.
template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads, 8)
rope_append_fp8_kernel(const T* qkv, int n_tokens, int nq, int nkv, const int32_t* positions, const int32_t* slots,
                       const float* rope_cos, const float* rope_sin, int rope_len, T* q_out, Fp8Pool pool, int* status) {
  grid_dep_wait();
  grid_dep_launch();
  constexpr int HD = LANES * 16;
  const int heads = nq + 2 * nkv;
  const int sub = threadIdx.x % LANES;
  const uint32_t unit = blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const bool live = unit < (uint32_t)n_tokens * (uint32_t)heads;
  const int t = live ? (int)(unit / (uint32_t)heads) : 0;
  const int head = live ? (int)(unit - (uint32_t)t * heads) : 0;
  const T* src = qkv + ((size_t)t * heads + head) * HD + sub * 8;
  const Raw8<T> lo = raw8(src), hi = raw8(src + HD / 2);
  const int64_t slot = slots[t];
  int pos = positions[t];
  const bool slot_ok = slot >= 0 && slot < pool.num_slots;
  if (pos < 0 || pos >= rope_len) {
    if (live) report(status, KVE_ERR_BOUNDS);
    pos = 0;
  }
  if (live && !slot_ok) report(status, KVE_ERR_BOUNDS);
  float a[8], b[8];
  if (head < nq + nkv) {
    float c[8], s[8];
    load8(rope_cos + (size_t)pos * (HD / 2) + sub * 8, c);
    load8(rope_sin + (size_t)pos * (HD / 2) + sub * 8, s);
    open8(lo, a);
    open8(hi, b);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = a[i], y = b[i];
      a[i] = __fsub_rn(__fmul_rn(x, c[i]), __fmul_rn(y, s[i]));
      b[i] = __fadd_rn(__fmul_rn(y, c[i]), __fmul_rn(x, s[i]));
    }
  } else {
    open8(lo, a);
    open8(hi, b);
  }
  if (live && head < nq) {
    T* dst = q_out + ((size_t)t * nq + head) * HD + sub * 8;
    store8(dst, a);
    store8(dst + HD / 2, b);
  }
  const bool write = live && head >= nq && slot_ok, is_v = head >= nq + nkv;
  // a warp of q heads only has nothing to quantise
  if (__any_sync(0xffffffffu, write)) {
    const int64_t at = write ? slot * nkv + (head - nq - (is_v ? nkv : 0)) : 0;
    store_row<LANES>(a, b, sub, (is_v ? pool.v : pool.k) + at * HD, (is_v ? pool.v_scale : pool.k_scale) + at, write);
  }
}

// Quantise and store rows of K and V as they are. A group of lanes per (K or V, token, head).
template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads)
append_fp8_kernel(const T* k_new, const T* v_new, const int64_t* slots, int n_tokens, int nkv, Fp8Pool pool, int* status) {
  grid_dep_wait();
  grid_dep_launch();
  constexpr int HD = LANES * 16;
  const int64_t rows = (int64_t)n_tokens * nkv;
  const int64_t unit = (blockIdx.x * (int64_t)kThreads + threadIdx.x) / LANES;
  const int sub = threadIdx.x % LANES;
  const bool live = unit < 2 * rows;
  const bool is_v = live && unit >= rows;
  const int64_t row = live ? unit - (is_v ? rows : 0) : 0;
  const int64_t t = row / nkv;
  float a[8], b[8];
  const T* src = (is_v ? v_new : k_new) + row * HD + sub * 8;
  load8(src, a);
  load8(src + HD / 2, b);
  int64_t slot = slots[t];
  bool write = live;
  if (write && (slot < 0 || slot >= pool.num_slots)) {
    report(status, KVE_ERR_BOUNDS);
    write = false;
  }
  const int64_t at = write ? slot * nkv + (row - t * nkv) : 0;
  store_row<LANES>(a, b, sub, (is_v ? pool.v : pool.k) + at * HD, (is_v ? pool.v_scale : pool.k_scale) + at, write);
}

// Rows of given slots as the values they stand for.
template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads)
read_fp8_kernel(Fp8Pool pool, const int64_t* slots, int n_tokens, int nkv, T* k_out, T* v_out, int* status) {
  grid_dep_wait();
  grid_dep_launch();
  constexpr int HD = LANES * 16;
  const int64_t rows = (int64_t)n_tokens * nkv;
  const int64_t unit = (blockIdx.x * (int64_t)kThreads + threadIdx.x) / LANES;
  const int sub = threadIdx.x % LANES;
  if (unit >= 2 * rows) return;
  const bool is_v = unit >= rows;
  const int64_t row = unit - (is_v ? rows : 0);
  const int64_t t = row / nkv;
  const int64_t slot = slots[t];
  float a[8] = {}, b[8] = {};
  if (slot < 0 || slot >= pool.num_slots) {
    report(status, KVE_ERR_BOUNDS);
  } else {
    const int64_t at = slot * nkv + (row - t * nkv);
    const uint4 x = *reinterpret_cast<const uint4*>((is_v ? pool.v : pool.k) + at * HD + sub * 16);
    const uint32_t byte = (is_v ? pool.v_scale : pool.k_scale)[at];
    const float up = byte == 0 ? __uint_as_float(0x00400000u) : byte == 255 ? NAN : __uint_as_float(byte << 23);
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w[i / 2] >> (i % 2 * 16)), __NV_E4M3);
      const float2 f = __half22float2(__half2(h));
      float(&o)[8] = i < 4 ? a : b;
      o[i % 4 * 2] = f.x * up;
      o[i % 4 * 2 + 1] = f.y * up;
    }
  }
  T* dst = (is_v ? v_out : k_out) + row * HD + sub * 16;
  store8(dst, a);
  store8(dst + 8, b);
}

int blocks_for(int64_t units, int lanes) { return (int)((units * lanes + kThreads - 1) / kThreads); }

// Checks shared by the three entry points; 0 or an error.
int check_fp8(const char* me, int dtype, int n, int nkv, int hd, const void* k, const void* v, const void* ks, const void* vs,
              int64_t num_slots) {
  if (n < 0 || nkv < 1 || num_slots < 1) return set_error(KVE_ERR_ARG, "%s: bad sizes", me);
  if (hd != 64 && hd != 128) return set_error(KVE_ERR_SHAPE, "%s: head_dim %d (supported: 64, 128)", me, hd);
  if (dtype != KVE_F32 && dtype != KVE_BF16) return set_error(KVE_ERR_DTYPE, "%s: dtype %d", me, dtype);
  if (n > 0 && (!k || !v || !ks || !vs)) return set_error(KVE_ERR_ARG, "%s: null pool or scales", me);
  if ((uintptr_t)k % 16 || (uintptr_t)v % 16) return set_error(KVE_ERR_ARG, "%s: pools must be 16-byte aligned", me);
  return KVE_OK;
}

}  // namespace
}  // namespace kve

using namespace kve;

extern "C" int kve_qkv_rope_append_fp8(const void* qkv, int dtype, int n_tokens, int num_heads, int num_kv_heads,
                                       int head_dim, const int32_t* positions, const int32_t* slots,
                                       const float* rope_cos, const float* rope_sin, int rope_len, void* q_out,
                                       void* pool_k, void* pool_v, uint8_t* k_scale, uint8_t* v_scale,
                                       int64_t num_slots, int* dev_status, cudaStream_t stream) {
  const char* me = "kve_qkv_rope_append_fp8";
  if (int rc = check_fp8(me, dtype, n_tokens, num_kv_heads, head_dim, pool_k, pool_v, k_scale, v_scale, num_slots)) return rc;
  if (num_heads < 0 || rope_len < 1) return set_error(KVE_ERR_ARG, "%s: bad sizes", me);
  if (n_tokens == 0) return KVE_OK;
  if (!qkv || !positions || !slots || !rope_cos || !rope_sin || (num_heads && !q_out))
    return set_error(KVE_ERR_ARG, "%s: null pointer", me);
  if ((uintptr_t)qkv % 16 || (uintptr_t)q_out % 16 || (uintptr_t)rope_cos % 16 || (uintptr_t)rope_sin % 16)
    return set_error(KVE_ERR_ARG, "%s: qkv, q_out and the tables must be 16-byte aligned", me);
  const int heads = num_heads + 2 * num_kv_heads;
  if ((int64_t)n_tokens * heads * (head_dim / 16) > 0x7fffffff) return set_error(KVE_ERR_SHAPE, "%s: too many rows", me);
  const int64_t units = (int64_t)n_tokens * heads;
  const Fp8Pool pool{static_cast<uint8_t*>(pool_k), static_cast<uint8_t*>(pool_v), k_scale, v_scale, num_slots};
  auto go = [&](auto kernel, auto* x, auto* out) {
    launch_kernel(kernel, dim3(blocks_for(units, head_dim / 16)), dim3(kThreads), 0, stream, x, n_tokens, num_heads,
                  num_kv_heads, positions, slots, rope_cos, rope_sin, rope_len, out, pool, dev_status);
  };
  using B = __nv_bfloat16;
  if (dtype == KVE_BF16 && head_dim == 64) go(rope_append_fp8_kernel<B, 4>, (const B*)qkv, (B*)q_out);
  else if (dtype == KVE_BF16) go(rope_append_fp8_kernel<B, 8>, (const B*)qkv, (B*)q_out);
  else if (head_dim == 64) go(rope_append_fp8_kernel<float, 4>, (const float*)qkv, (float*)q_out);
  else go(rope_append_fp8_kernel<float, 8>, (const float*)qkv, (float*)q_out);
  return check_launch(me);
}

extern "C" int kve_kv_append_fp8(const void* k_new, const void* v_new, int dtype, const int64_t* slot_ids, int n_tokens,
                                 int num_kv_heads, int head_dim, void* pool_k, void* pool_v, uint8_t* k_scale,
                                 uint8_t* v_scale, int64_t num_slots, int* dev_status, cudaStream_t stream) {
  const char* me = "kve_kv_append_fp8";
  if (int rc = check_fp8(me, dtype, n_tokens, num_kv_heads, head_dim, pool_k, pool_v, k_scale, v_scale, num_slots)) return rc;
  if (n_tokens == 0) return KVE_OK;
  if (!k_new || !v_new || !slot_ids) return set_error(KVE_ERR_ARG, "%s: null pointer", me);
  if ((uintptr_t)k_new % 16 || (uintptr_t)v_new % 16)
    return set_error(KVE_ERR_ARG, "%s: k_new and v_new must be 16-byte aligned", me);
  const int64_t units = 2 * (int64_t)n_tokens * num_kv_heads;
  if (units > (int64_t)0x7fffffff * 16) return set_error(KVE_ERR_SHAPE, "%s: too many rows", me);
  const Fp8Pool pool{static_cast<uint8_t*>(pool_k), static_cast<uint8_t*>(pool_v), k_scale, v_scale, num_slots};
  auto go = [&](auto kernel, auto* k, auto* v) {
    launch_kernel(kernel, dim3(blocks_for(units, head_dim / 16)), dim3(kThreads), 0, stream, k, v, slot_ids, n_tokens,
                  num_kv_heads, pool, dev_status);
  };
  using B = __nv_bfloat16;
  if (dtype == KVE_BF16 && head_dim == 64) go(append_fp8_kernel<B, 4>, (const B*)k_new, (const B*)v_new);
  else if (dtype == KVE_BF16) go(append_fp8_kernel<B, 8>, (const B*)k_new, (const B*)v_new);
  else if (head_dim == 64) go(append_fp8_kernel<float, 4>, (const float*)k_new, (const float*)v_new);
  else go(append_fp8_kernel<float, 8>, (const float*)k_new, (const float*)v_new);
  return check_launch(me);
}

extern "C" int kve_kv_read_fp8(const void* pool_k, const void* pool_v, const uint8_t* k_scale, const uint8_t* v_scale,
                               const int64_t* slot_ids, int n_tokens, int num_kv_heads, int head_dim, int64_t num_slots,
                               int dtype, void* k_out, void* v_out, int* dev_status, cudaStream_t stream) {
  const char* me = "kve_kv_read_fp8";
  if (int rc = check_fp8(me, dtype, n_tokens, num_kv_heads, head_dim, pool_k, pool_v, k_scale, v_scale, num_slots)) return rc;
  if (n_tokens == 0) return KVE_OK;
  if (!slot_ids || !k_out || !v_out) return set_error(KVE_ERR_ARG, "%s: null pointer", me);
  if ((uintptr_t)k_out % 16 || (uintptr_t)v_out % 16)
    return set_error(KVE_ERR_ARG, "%s: k_out and v_out must be 16-byte aligned", me);
  const int64_t units = 2 * (int64_t)n_tokens * num_kv_heads;
  if (units > (int64_t)0x7fffffff * 16) return set_error(KVE_ERR_SHAPE, "%s: too many rows", me);
  const Fp8Pool pool{(uint8_t*)pool_k, (uint8_t*)pool_v, (uint8_t*)k_scale, (uint8_t*)v_scale, num_slots};
  auto go = [&](auto kernel, auto* k, auto* v) {
    launch_kernel(kernel, dim3(blocks_for(units, head_dim / 16)), dim3(kThreads), 0, stream, pool, slot_ids, n_tokens,
                  num_kv_heads, k, v, dev_status);
  };
  using B = __nv_bfloat16;
  if (dtype == KVE_BF16 && head_dim == 64) go(read_fp8_kernel<B, 4>, (B*)k_out, (B*)v_out);
  else if (dtype == KVE_BF16) go(read_fp8_kernel<B, 8>, (B*)k_out, (B*)v_out);
  else if (head_dim == 64) go(read_fp8_kernel<float, 4>, (float*)k_out, (float*)v_out);
  else go(read_fp8_kernel<float, 8>, (float*)k_out, (float*)v_out);
  return check_launch(me);
}

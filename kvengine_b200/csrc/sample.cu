// Verification of drafted tokens against the target's probabilities, from given
// random numbers: a chain of drafts with or without the draft model's
// distributions, or a tree of given candidates.
//
// With p = softmax(logits / T) of a target row (T <= 0: one-hot at its lowest
// argmax) the methods are
//   chain  draft d is accepted where u q(d) < p(d), q the draft's distribution
//          (without one: one-hot at d). The token behind the accepted prefix comes
//          from w = max(p - q, 0), or from p where every draft was accepted.
//   tree   at the current node, children in index order: child c with token d is
//          accepted where u_c R < p(d), R = 1 - (p of the rejected siblings); a
//          token already rejected there has p = 0. The token behind the accepted
//          path comes from p without the rejected tokens.
// and the token drawn is argmax(log w_v + gumbel_v) (lowest index among equals; from
// p where no w is positive).
//
// Two kernels. The first reads every logit once and leaves, per row and part of the
// row, the sum of e^(x / T) and the largest term it is relative to (T <= 0: the argmax):
// HBM is its bound. The second runs a cluster of CTAs per sequence: each joins
// the parts' sums of the rows it needs, walks the drafts (every CTA of the cluster
// by itself: a few values) and scans its share of the one row the last token comes
// from, which is often still in L2; the shares' best tokens meet through distributed
// shared memory.
//
// Measured, vocabulary 151936: 128 chains of 4 fp32 drafts with the draft's logits (778 MB) 142 us, 64 trees of
// 16 bf16 nodes (350 MB) 76 us, one bf16 chain 12.7 us (replayed graphs). The first kernel takes three quarters of
// the large ones, at 83 % of HBM's throughput; one chain is two kernels' latencies.
//
// Precision: a row is held as (b, z), z = sum 2^((x - b) c) with c = log2(e) / T and b the
// largest logit. The sums are taken relative to b c as rounded, so that every exponent is one
// fused operation rounded relative to itself, and moved by what the rounding left. That holds while
// the rest is small: past |b c| of 2^22 (half an ulp would be an exponent of 1/4, at 3e9 more than fp32's
// whole range) a row's exponents are (x - b) c from 64-bit differences, more slowly. 2^x runs on ex2.approx (2^-22)
// into fp32 sums of up to 128 of a thread's vectors, those into a 64-bit one, and the threads' pairwise in
// fp32 again. The largest logit's 1 is kept out of all of them: where it has nearly the whole probability, what p and q
// leave to the others is what they differ by, and an fp32 sum that begins with 1 loses it below 2^-24. So p is
// good to (1 - its largest) times 2^-21 and 2^-22 the mean size of the exponents (c's rounding).
// Acceptance, log-probabilities and every candidate that fp32 does not rule out are computed in 64
// bits from these sums. A NaN logit counts as minus infinity (never drawn);
// rows with one are summed again, slowly.
#include <float.h>
#include <math.h>

#include "kve_common.cuh"

namespace kve {
namespace {

constexpr double kLog2e = 1.4426950408889634;
constexpr int kStatThreads = 256;
constexpr int kDrawThreads = 256;  // and three CTAs a SM: 128 sequences' clusters run in one wave
constexpr int kMaxParts = 32;     // parts of a row in the first kernel
constexpr int kMaxNodes = 1024;   // nodes of a tree
constexpr int kMaxK = 31;         // drafts of a chain
// Behind the arrival counters of the ops that share a workspace, which must stay zero.
constexpr size_t kSharedBytes = 65536;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// The temperature as it counts: 0 where T <= 0 or NaN, and subnormal numbers as 2^-126 (c stays finite).
__device__ __forceinline__ float heat(float t) { return t > 0.f ? fmaxf(t, FLT_MIN) : 0.f; }
// Floats as integers of the same order.
__device__ __forceinline__ int ordered(float f) {
  const int i = __float_as_int(f);
  return i < 0 ? i ^ 0x7fffffff : i;
}
__device__ __forceinline__ float unordered(int i) { return __int_as_float(i < 0 ? i ^ 0x7fffffff : i); }
// NaN as minus infinity.
__device__ __forceinline__ float clean(float x) { return x == x ? x : -INFINITY; }

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

template <typename T> struct Pack;
template <> struct Pack<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& v, float (&o)[4]) {
    o[0] = __uint_as_float(v.x); o[1] = __uint_as_float(v.y); o[2] = __uint_as_float(v.z); o[3] = __uint_as_float(v.w);
  }
};
template <> struct Pack<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& v, float (&o)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      o[2 * i] = __uint_as_float(w[i] << 16);
      o[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
};

// Calls f(value, index) for columns [lo, hi) of a row, 16 bytes at a time from the
// row's first 16-byte boundary on; `batch(values, first index)` gets the vectors, `start(U times 16 bytes)` the
// first U of a warp's threads before (where all have as many), and `fold()` is
// called now and then in a long row, after every 16 U of a thread's vectors.
template <typename T, int THREADS, int U, typename Batch, typename One, typename Start, typename Fold>
__device__ __forceinline__ void scan(const T* row, int lo, int hi, Batch&& batch, One&& one, Start&& start, Fold&& fold) {
  constexpr int N = Pack<T>::N;
  const int off = (int)((reinterpret_cast<uintptr_t>(row + lo) & 15) / sizeof(T));
  const int head = min(lo + (off ? N - off : 0), hi);
  const int nvec = (hi - head) / N;
  const uint4* v = reinterpret_cast<const uint4*>(row + head);
  for (int i = lo + threadIdx.x; i < head; i += THREADS) one(Elem<T>::to_f(row[i]), i);
  int i = threadIdx.x;
  for (int rest = 16; i + (U - 1) * THREADS < nvec; i += U * THREADS) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = __ldcg(v + i + u * THREADS);
    if (i == (int)threadIdx.x && (i | 31) + (U - 1) * THREADS < nvec) start(raw);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[N];
      Pack<T>::unpack(raw[u], x);
      batch(x, head + (i + u * THREADS) * N);
    }
    if (--rest == 0) {
      fold();
      rest = 16;
    }
  }
  for (; i < nvec; i += THREADS) {
    const uint4 raw = __ldcg(v + i);
    float x[N];
    Pack<T>::unpack(raw, x);
    batch(x, head + i * N);
  }
  for (int j = head + nvec * N + threadIdx.x; j < hi; j += THREADS) one(Elem<T>::to_f(row[j]), j);
}

// What the first kernel leaves of one part of a row: its largest logit, and the sum relative to
// that less 1 or, for T <= 0, its column.
struct Part {
  float b, z;
};

// Where the rows of the first kernel lie: rows [0, n_first) at `first`, the others
// at `second` (the draft's, rows_b and strides of their own).
struct Rows {
  const void* first;
  const void* second;
  int64_t first_stride;             // elements between consecutive rows
  int64_t second_sb, second_sj;     // elements between sequences, and between a sequence's rows
  int n_first, per_seq, k;          // target rows, and rows of a sequence in each of the two (chain)
  const int32_t* q_offsets;         // tree: a row's sequence is found here (batch entries)
  int batch;
};

// The last b with offsets[b] <= row, where they ascend; in any case no less for a greater row.
__device__ __forceinline__ int search(const int32_t* offsets, int batch, int row) {
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (offsets[mid] <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}
__device__ __forceinline__ int sequence_of(const Rows& r, int row) {
  if (r.q_offsets) return search(r.q_offsets, r.batch, row);
  return row < r.n_first ? row / r.per_seq : (row - r.n_first) / r.k;
}

template <typename T>
__device__ __forceinline__ const T* row_at(const Rows& r, int row) {
  if (row < r.n_first) return static_cast<const T*>(r.first) + row * r.first_stride;
  const int i = row - r.n_first;
  return static_cast<const T*>(r.second) + (i / r.k) * r.second_sb + (i % r.k) * r.second_sj;
}

// 1 / T in 64 bits: an fp32 quotient and its remainder, a fraction of a 64-bit division's latency.
__device__ __forceinline__ double inverse(float t) {
  if (t > 1e30f) return 1.0 / t;  // fp32's quotient would be subnormal
  const double r = 1.f / t, e = fma(-(double)t, r, 1.0);  // e of up to 2^-24, exactly
  return r + r * (e + e * e);
}
// log2 of e^(x / T) over e^(b / T) in 64 bits, b a row's largest logit (an infinite one: only its likes count).
__device__ __forceinline__ double exponent(float x, float b, float t) {
  return b == INFINITY ? (x == INFINITY ? 0.0 : -INFINITY) : ((double)x - b) * (kLog2e * inverse(t));
}

// Whether fp32 exponents fused from x c will not do for a row of largest logit b: b c is too large (or
// infinite), or c so small that a difference of logits may overflow and still count.
__device__ __forceinline__ bool far(float b, float c) { return !(fabsf(b * c) < 4194304.f) || c < 1e-30f; }

template <typename T>
__global__ void __launch_bounds__(kStatThreads, 4)
row_stats_kernel(Rows rows, int vocab, int chunk, int parts, const float* temperature, Part* out) {
  grid_dep_wait();
  grid_dep_launch();
  const int row = blockIdx.x, part = blockIdx.y;
  const int lo = part * chunk, hi = min(vocab, lo + chunk);
  const float t = heat(temperature[sequence_of(rows, row)]);
  const T* x = row_at<T>(rows, row);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ float sm[kStatThreads / 32], sz[kStatThreads / 32];
  if (!(t > 0.f)) {
    float best = -INFINITY;
    int at = 0x7fffffff;
    auto one = [&](float v, int i) {
      v = clean(v);
      if (v > best || (v == best && i < at)) { best = v; at = i; }
    };
    auto batch = [&](const auto& v, int i) {
#pragma unroll
      for (int j = 0; j < Pack<T>::N; ++j) one(v[j], i + j);
    };
    scan<T, kStatThreads, 2>(x, lo, hi, batch, one, [](const auto&) {}, [] {});
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float ov = __shfl_xor_sync(0xffffffffu, best, o);
      const int oi = __shfl_xor_sync(0xffffffffu, at, o);
      if (ov > best || (ov == best && oi < at)) { best = ov; at = oi; }
    }
    if (lane == 0) { sm[warp] = best; sz[warp] = __int_as_float(at); }
    __syncthreads();
    if (threadIdx.x == 0) {
      for (int w = 1; w < kStatThreads / 32; ++w) {
        const int oi = __float_as_int(sz[w]);
        if (sm[w] > best || (sm[w] == best && oi < at)) { best = sm[w]; at = oi; }
      }
      out[(size_t)row * parts + part] = Part{best, __int_as_float(at)};
    }
    return;
  }
  const float c = (float)kLog2e / t;
  float most = -FLT_MAX, off = 0.f, n = 0.f;  // this thread's largest logit so far, minus that times c, how often it came,
  float z = 0.f;                              // and the sum of the latest others
  double sum = 0.0;                           // that of those before (a long row's terms are below half an ulp of an fp32 sum),
  float sum_off = 0.f;                        // relative to this
  auto lift = [&](float top) {
    // the product rounded, as the terms are relative to it (a fused one would move z by its rounding)
    const float next = -__fmul_rn(top, c);
    if (most > -FLT_MAX) z = z * ex2(next - off) + n * ex2(fmaf(most, c, next));
    most = top;
    off = next;
    n = 0.f;
  };
  auto one = [&](float v, int) {
    if (v >= most) {
      if (v > most) lift(v);
      n += 1.f;
    } else {
      z += ex2(fmaf(v, c, off));
    }
  };
  auto batch = [&](auto& v, int) {
    constexpr int N = Pack<T>::N;
    float top = v[0];
#pragma unroll
    for (int j = 1; j < N; ++j) top = fmaxf(top, v[j]);  // passes over NaN
    if (__builtin_expect(top >= most, 0)) {
      if (top > most) lift(top);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (v[j] == most) {
          n += 1.f;
          v[j] = -INFINITY;
        }
    }
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = ex2(fmaf(v[j], c, off));
#pragma unroll
    for (int w = N / 2; w > 0; w >>= 1)
#pragma unroll
      for (int j = 0; j < w; ++j) v[j] += v[j + w];
    z += v[0];
  };
  auto fold = [&] {
    sum = sum == 0.0 ? z : sum * ex2(off - sum_off) + z;
    sum_off = off;
    z = 0.f;
  };
  // A warp starts from the largest of its threads' first vectors: from its own first, nearly every vector
  // would be a new largest for some thread, and the warp would wait for it.
  auto start = [&](const auto& raw) {
    float m = -FLT_MAX;
#pragma unroll
    for (int u = 0; u < (int)(sizeof(raw) / sizeof(uint4)); ++u) {
      float v[Pack<T>::N];
      Pack<T>::unpack(raw[u], v);
#pragma unroll
      for (int j = 0; j < Pack<T>::N; ++j) m = fmaxf(m, v[j]);  // passes over NaN
    }
    m = unordered(__reduce_max_sync(0xffffffffu, ordered(m)));
    if (m > most) lift(m);
  };
  scan<T, kStatThreads, 8>(x, lo, hi, batch, one, start, fold);
  // the part's base, then its sum
  auto block_max = [&](float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    if (lane == 0) sm[warp] = v;
    __syncthreads();
    v = sm[lane % (kStatThreads / 32)];
#pragma unroll
    for (int o = kStatThreads / 64; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  };
  const float top = block_max(most);
  if (sum != 0.0) z = (float)(sum * ex2(off - sum_off) + z);
  const bool odd = __syncthreads_or(!(z < INFINITY));  // a NaN, or infinite logits
  float tops = 0.f;  // how often the part's largest came
  if (top == -FLT_MAX && !odd && !__syncthreads_or(n > 0.f)) {
    z = 0.f;  // nothing but minus infinity
  } else if (odd || far(top, c)) {
    // infinite logits share the whole probability, NaN has none
    sum = 0.0;
    for (int i = lo + threadIdx.x; i < hi; i += kStatThreads) {
      const float v = clean(Elem<T>::to_f(x[i]));
      if (v == top) tops += 1.f;
      else if (v != -INFINITY) sum += ex2((float)exponent(v, top, t));
    }
    z = (float)sum;
  } else if (most > -FLT_MAX) {
    const float b = __fmul_rn(top, c), moved = fmaf(top, c, -b);
    z *= ex2(-off - b - moved);
    if (most == top) tops = n;
    else z += n * ex2(fmaf(most, c, -b) - moved);
  }
  z = warp_sum(z);
  // at least 1 where there is any; a few, so that integers do
  int count = __reduce_add_sync(0xffffffffu, (int)tops);
  if (lane == 0) { sz[warp] = z; sm[warp] = __int_as_float(count); }
  __syncthreads();
  if (warp == 0) {
    z = warp_sum(lane < kStatThreads / 32 ? sz[lane] : 0.f);
    count = __reduce_add_sync(0xffffffffu, lane < kStatThreads / 32 ? __float_as_int(sm[lane]) : 0);
    if (lane == 0) out[(size_t)row * parts + part] = Part{count ? top : -INFINITY, (float)(count - 1) + z};
  }
}

// A row's parts joined.
struct Row {
  double z;   // the sum of 2^((x - b) c)
  float b;    // the largest logit
  int arg;    // T <= 0: the column of the largest
};
// Rows row_of(0) .. row_of(n - 1) into out, by all threads: `group` (a power of two of at
// least n_parts) lanes a row.
template <typename F>
__device__ __forceinline__ void join_rows(const Part* parts, int n_parts, int group, float t, Row* out, int n, F&& row_of) {
  const int sub = threadIdx.x & (group - 1), per = kDrawThreads / group;
  for (int i0 = 0; i0 < n; i0 += per) {
    const int i = i0 + threadIdx.x / group;
    Part p{-INFINITY, 0.f};
    if (i < n && sub < n_parts) {
      const float2 v = __ldcg(reinterpret_cast<const float2*>(parts) + (size_t)row_of(i) * n_parts + sub);
      p = Part{v.x, v.y};
    }
    float b = p.b;
    for (int o = 1; o < group; o <<= 1) b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, o));
    Row r{1.0, b, 0x7fffffff};
    if (!(t > 0.f)) {
      r.arg = sub < n_parts && p.b == b ? __float_as_int(p.z) : 0x7fffffff;
      for (int o = 1; o < group; o <<= 1) r.arg = min(r.arg, __shfl_xor_sync(0xffffffffu, r.arg, o));
    } else {
      r.z = p.b == -INFINITY ? 0.0 : p.b == b ? 1.0 + p.z : (1.0 + p.z) * exp2(exponent(p.b, b, t));
      for (int o = 1; o < group; o <<= 1) r.z += __shfl_xor_sync(0xffffffffu, r.z, o);
    }
    if (i < n && sub == 0) out[i] = r;
  }
}
// p of logit x at column v in 64 bits, and its logarithm (T > 0).
__device__ __forceinline__ double probability(const Row& r, float x, int v, float t) {
  if (!(t > 0.f)) return v == r.arg ? 1.0 : 0.0;
  x = clean(x);
  if (x == -INFINITY || !(r.z > 0.0)) return 0.0;
  return exp2(exponent(x, r.b, t)) / r.z;
}
__device__ __forceinline__ float log_probability(const Row& r, float x, float t) {
  if (clean(x) == -INFINITY || !(r.z > 0.0)) return -INFINITY;
  return (float)((log2(r.z) - exponent(x, r.b, t)) * -0.6931471805599453);
}
struct DrawParams {
  const void* logits;       // target rows
  int64_t stride;
  const void* draft;        // chain: draft rows, or null
  int64_t dsb, dsj;
  const Part* parts;        // [rows][n_parts]: target rows, then draft rows
  int n_parts, group;
  const int32_t* drafts;    // chain: draft tokens (tree: node tokens)
  int64_t tsb, tsj;
  const int32_t* parents;   // tree
  const int32_t* q_lens;
  const int32_t* q_offsets;
  const float* u;
  int64_t usb;
  const float* gumbel;      // [batch, vocab]
  int64_t gstride;
  const float* temperature;
  int batch, k, vocab, n_rows, max_nodes;
  int shares, chunk;        // CTAs per sequence, columns of each
  int32_t* n_acc;
  int32_t* path;            // tree: [batch, width]
  int32_t* emitted;         // [batch, width]
  float* logp;              // [batch, width]
  int width;
  int* status;
};

// A candidate for the last token: its key in 64 bits, its column and its logit.
struct Best {
  double key;
  int at;
  float x;
};
__device__ __forceinline__ Best better(Best a, Best b) {
  return b.at >= 0 && (a.at < 0 || b.key > a.key || (b.key == a.key && b.at < a.at)) ? b : a;
}
__device__ __forceinline__ Best warp_best(Best b) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    b = better(b, Best{__shfl_xor_sync(0xffffffffu, b.key, o), __shfl_xor_sync(0xffffffffu, b.at, o),
                       __shfl_xor_sync(0xffffffffu, b.x, o)});
  return b;
}

// Shared memory of a draw.
struct DrawShared {
  Best kept[kDrawThreads];
  Best share[8];               // rank 0's: the best of each CTA of the cluster
  Best best;
  float ratio;                 // z of the target's row over that of the draft's
  int bar;                     // what a column has to reach to be the CTA's best, as an ordered integer
  int n;                       // candidates kept
};
// What fp32 may be off by, relative to the size of each term of a key or weight: exponents, ex2.approx and
// lg2.approx are good to 2^-22, and a handful of roundings of 2^-24 come on top.
constexpr float kOff = 0x1p-20f;

// The CTA's best candidate of columns [lo, hi), in every lane of warp 0. `qrow` (may be
// null): the draft's row, whose distribution is subtracted. `skip`: tokens not to draw.
//
// A column's key is log2 of its weight plus gumbel log2 e. The scan in fp32 knows it only to
// lie between two bounds; where p and q nearly cancel they are far apart. It keeps the largest
// lower bound of the CTA's columns, and every column whose upper bound reaches that is looked at in 64 bits, so the
// result is that of 64 bits (from the rows' sums as they are). A key is at most the one without the
// draft, so a column is first held against that, and only the few that pass cost an exponential, a
// logarithm and a look at the draft's row.
template <typename T>
__device__ __forceinline__ Best draw_columns(DrawShared& sh, int lo, int hi, const T* row, const Row& p, const T* qrow,
                                             const Row& q, const float* gumbel, float t, const int* skip, int n_skip) {
  constexpr int N = Pack<T>::N;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr float kL = (float)kLog2e;
  const float c = kL / t;
  if (q.b == -INFINITY) qrow = nullptr;  // a draft without any probability takes nothing away
  const bool slow = far(p.b, c) || (qrow && far(q.b, c));  // every column in 64 bits
  __syncthreads();  // an earlier draw's values have been read
  if (threadIdx.x == 0) {
    sh.bar = ordered(-FLT_MAX);  // which minus infinity does not reach
    sh.n = 0;
    // z of p over z of q, for sums relative to b c as rounded
    if (qrow && !slow) sh.ratio = (float)(p.z / q.z) * ex2(fmaf(p.b, c, -__fmul_rn(p.b, c)) - fmaf(q.b, c, -__fmul_rn(q.b, c)));
  }
  // 16 bytes of logits at a time from their first 16-byte boundary on, and their noise
  const int mis = (int)((reinterpret_cast<uintptr_t>(row + lo) & 15) / sizeof(T));
  const int head = min(lo + (mis ? N - mis : 0), hi);
  const int nvec = (hi - head) / N;
  const uint4* xv = reinterpret_cast<const uint4*>(row + head);
  const float* gh = gumbel + head;
  const bool even = (reinterpret_cast<uintptr_t>(gh) & 15) == 0;
  auto noise = [&](int i, float* g) {
    if (even) {
#pragma unroll
      for (int j = 0; j < N / 4; ++j) {
        const float4 f = __ldcg(reinterpret_cast<const float4*>(gh) + (size_t)i * (N / 4) + j);
        g[4 * j] = f.x;
        g[4 * j + 1] = f.y;
        g[4 * j + 2] = f.z;
        g[4 * j + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) g[j] = gh[(size_t)i * N + j];
    }
  };
  int at = -1;                                                 // this thread's column of the largest lower bound,
  float low = -INFINITY, high = -INFINITY, other = -INFINITY;  // its bounds, and the others' largest upper bound
  __syncthreads();
  if (p.z > 0.0 && !slow) {
    // Keys times z here, their exponents fused from x c and relative to b c as rounded.
    const float off = -__fmul_rn(p.b, c), qoff = -__fmul_rn(q.b, c);
    volatile int* bar = &sh.bar;
    // Upper bounds without the draft are u = e + g (1 + 8 kOff). A key k = e + g, e at most 0, is at most
    // u + 10 kOff |k| + 4 kOff: positive noise brings along more than e can be off by, and with negative noise
    // neither term is larger than k. So a column with u below bar - 16 kOff (|bar| + 1) is below the bar, and that
    // is what sh.bar holds.
    constexpr float kMore = kL * (1.f + 8.f * kOff);
    auto consider = [&](float x, float g, float u, int v) {
      if (!(x > -INFINITY)) return;
      const float gl = g * kL, e = fmaf(x, c, off), sure = fabsf(gl) < INFINITY ? kOff : 0.f;  // infinite noise: nothing is off
      float least = u - (sure > 0.f ? 16.f * sure * (fabsf(e) + fabsf(gl) + 1.f) : 0.f);
      if (qrow) {
        const float y = clean(Elem<T>::to_f(qrow[v])), f = fmaf(y, c, qoff);
        const float pw = ex2(e), qw = ex2(f) * sh.ratio;  // times z
        // below 2^-110 a weight is only known to be small
        const float off_by = kOff * (pw * (2.f + fminf(fabsf(e), 200.f)) + qw * (4.f + fminf(fabsf(f), 200.f))) + 0x1p-110f;
        const float hi_w = pw - qw + off_by, lo_w = pw - qw - off_by;
        auto key = [&](float w, float way) {
          const float l = __log2f(w);
          return l + gl + (sure > 0.f ? way * sure * (fabsf(l) + fabsf(gl) + 2.f) : 0.f);
        };
        u = hi_w > 0.f ? fminf(u, key(hi_w, 1.f)) : -INFINITY;
        least = lo_w > 0.f ? key(lo_w, -1.f) : -INFINITY;
        if (!(u >= unordered(*bar))) return;
      }
      for (int j = 0; j < n_skip; ++j)
        if (skip[j] == v) return;
      if (at < 0 || least > low) {
        other = fmaxf(other, high);
        at = v;
        low = least;
        high = u;
      } else {
        other = fmaxf(other, u);
      }
      const int b = ordered(fabsf(least) < INFINITY ? least - 16.f * kOff * (fabsf(least) + 1.f) : least);
      if (b > *bar) atomicMax(&sh.bar, b);
    };
    auto one = [&](float x, int v) {
      const float g = gumbel[v], u = fmaf(g, kMore, fmaf(x, c, off));
      if (u >= unordered(*bar)) consider(x, g, u, v);
    };
    auto batch = [&](const float* x, const float* g, int v) {
      float u[N], top = -INFINITY;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        u[j] = fmaf(g[j], kMore, fmaf(x[j], c, off));
        top = fmaxf(top, u[j]);  // passes over NaN
      }
      if (!(top >= unordered(*bar))) return;
      // The greatest first: it raises the bar, and the others seldom reach that (they are then read again, for
      // one copy of the code instead of N).
      float bx = 0.f, bg = 0.f;
      int best = 0;
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (u[j] == top) {
          bx = x[j];
          bg = g[j];
          best = j;
        }
      consider(bx, bg, top, v + best);
      const float now = unordered(*bar);
      int left = 0;
#pragma unroll
      for (int j = 0; j < N; ++j) left |= (u[j] >= now && j != best) << j;
      for (; left; left &= left - 1) one(Elem<T>::to_f(row[v + __ffs(left) - 1]), v + __ffs(left) - 1);
    };
    constexpr int U = sizeof(T) == 4 ? 4 : 2;
    for (int i0 = threadIdx.x; i0 < nvec; i0 += U * kDrawThreads) {
      uint4 raw[U];
      float g[U][N];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u * kDrawThreads < nvec) {
          raw[u] = __ldcg(xv + i0 + u * kDrawThreads);
          noise(i0 + u * kDrawThreads, g[u]);
        }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u * kDrawThreads < nvec) {
          float x[N];
          Pack<T>::unpack(raw[u], x);
          batch(x, g[u], head + (i0 + u * kDrawThreads) * N);
        }
    }
    // the columns before and behind
    const int before = head - lo, behind = head + nvec * N;
    for (int j = threadIdx.x; j < before + hi - behind; j += kDrawThreads) {
      const int v = j < before ? lo + j : behind + j - before;
      one(Elem<T>::to_f(row[v]), v);
    }
  }
  // Column v's key in 64 bits; NaN where its weight rounds to nothing there.
  auto exact = [&](int v, float x) {
    if (!qrow) return (p.b == INFINITY ? 0.0 : ((double)x - p.b) * inverse(t)) + (double)gumbel[v];
    const double w = probability(p, x, v, t) - probability(q, Elem<T>::to_f(qrow[v]), v, t);
    return w > 0.0 ? log(w) + (double)gumbel[v] : (double)NAN;
  };
  __syncthreads();
  const float bar = unordered(sh.bar);
  const bool last = at >= 0 && high >= bar;
  Best mine{-INFINITY, -1, 0.f};
  // Another of one thread's columns that may be the best, or a row that fp32 does not do for: all columns.
  const bool again = __syncthreads_or(other >= bar) || (p.z > 0.0 && slow);
  for (int v = again ? lo + threadIdx.x : last ? at : hi; v < hi; v = again ? v + kDrawThreads : hi) {
    const float x = clean(Elem<T>::to_f(row[v]));
    bool out = x == -INFINITY || (p.b == INFINITY && x != INFINITY);
    for (int j = 0; j < n_skip; ++j) out |= skip[j] == v;
    const double k = out ? (double)NAN : exact(v, x);
    if (k == k) mine = better(mine, Best{k, v, x});
  }
  if (mine.at >= 0) sh.kept[atomicAdd(&sh.n, 1)] = mine;
  __syncthreads();
  Best b{-INFINITY, -1, 0.f};
  if (warp == 0) {
    for (int i = lane; i < sh.n; i += 32) b = better(b, sh.kept[i]);
    b = warp_best(b);
  }
  return b;
}

// The token drawn by the cluster, in rank 0 (the others' result means nothing; they
// are done). Where no weight is positive, rank 0 draws from p alone.
template <typename T>
__device__ __forceinline__ Best draw(const DrawParams& a, DrawShared& sh, const T* row, const Row& p, const T* qrow,
                                     const Row& q, const float* gumbel, float t, int rank, const int* skip, int n_skip) {
  const int lo = min(rank * a.chunk, a.vocab), hi = min(a.vocab, lo + a.chunk);
  const int lane = threadIdx.x & 31;
  Best b = draw_columns<T>(sh, lo, hi, row, p, qrow, q, gumbel, t, skip, n_skip);
  cluster_wait();  // every CTA of the cluster has started: rank 0's memory is there
  if (threadIdx.x == 0) {
    uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(&sh.share[rank]));
    asm volatile("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(to) : "r"(0));
    asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(to), "d"(b.key) : "memory");
    asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(to + 8), "r"(b.at), "r"(__float_as_int(b.x)) : "memory");
  }
  __syncwarp();
  cluster_arrive();
  cluster_wait();
  if (rank != 0) return b;
  if (threadIdx.x < 32) {
    b = Best{-INFINITY, -1, 0.f};
    if (lane < a.shares) b = sh.share[lane];
    b = warp_best(b);
    if (lane == 0) sh.best = b;
  }
  __syncthreads();
  b = sh.best;
  if (b.at < 0 && (qrow || n_skip)) {
    b = draw_columns<T>(sh, 0, a.vocab, row, p, nullptr, p, gumbel, t, skip, 0);
    if (threadIdx.x == 0) sh.best = b;
    __syncthreads();
    b = sh.best;
  }
  if (b.at < 0) b = Best{0.0, 0, -INFINITY};  // no probability anywhere
  return b;
}

template <typename T>
__global__ void __launch_bounds__(kDrawThreads, 3)
chain_draw_kernel(DrawParams a) {
  cluster_arrive();
  grid_dep_wait();
  grid_dep_launch();
  const int b = blockIdx.x / a.shares, rank = blockIdx.x % a.shares;
  const int k = a.k, tid = threadIdx.x;
  const float t = heat(a.temperature[b]);
  const T* logits = static_cast<const T*>(a.logits) + (int64_t)b * (k + 1) * a.stride;
  const T* draft = a.draft ? static_cast<const T*>(a.draft) + b * a.dsb : nullptr;
  __shared__ Row rows[2 * kMaxK + 1];  // target rows 0 .. k, then draft rows
  __shared__ double pd[kMaxK];         // p of the drafts
  __shared__ int tok[kMaxK];
  __shared__ int n_s;
  __shared__ DrawShared sh;
  // Thread j fetches draft j and its logits while the rows' sums are joined.
  int d = -1;
  float x = 0.f, y = 0.f, u = 0.f;
  if (tid < k) {
    d = a.drafts[b * a.tsb + tid * a.tsj];
    u = a.u[b * a.usb + tid];
    if (d < 0 || d >= a.vocab) {
      if (rank == 0) report(a.status, KVE_ERR_BOUNDS);
      d = -1;
    } else {
      x = Elem<T>::to_f(logits[tid * a.stride + d]);
      if (draft) y = Elem<T>::to_f(draft[tid * a.dsj + d]);
    }
    tok[tid] = d;
  }
  join_rows(a.parts, a.n_parts, a.group, t, rows, draft ? 2 * k + 1 : k + 1,
            [&](int i) { return i <= k ? b * (k + 1) + i : a.batch * (k + 1) + b * k + (i - k - 1); });
  __syncthreads();
  if (tid < 32) {
    bool no = false;
    if (tid < k) {
      const double p = d < 0 ? 0.0 : probability(rows[tid], x, d, t);
      const double q = d < 0 || !draft ? 1.0 : probability(rows[k + 1 + tid], y, d, t);
      pd[tid] = p;
      no = !((double)u * q < p);
    }
    const unsigned m = __ballot_sync(0xffffffffu, no);
    if (tid == 0) n_s = m ? __ffs(m) - 1 : k;
  }
  __syncthreads();
  const int n = n_s;
  const Row p = rows[n];
  Best last;
  if (!(t > 0.f)) {
    cluster_wait();
    last = Best{0.0, p.arg < a.vocab ? p.arg : 0, 0.f};  // one-hot: a rejected draft was another token
  } else {
    const bool sub = draft && n < k;
    last = draw<T>(a, sh, logits + n * a.stride, p, sub ? draft + n * a.dsj : nullptr, sub ? rows[k + 1 + n] : p,
                   a.gumbel + b * a.gstride, t, rank, tok + n, !draft && n < k ? 1 : 0);
  }
  if (rank != 0 || tid > k) return;
  float lp = 0.f;
  if (t > 0.f && tid <= n) lp = tid < n ? (float)log(pd[tid]) : log_probability(p, last.x, t);
  a.emitted[(size_t)b * a.width + tid] = tid < n ? tok[tid] : tid == n ? last.at : -1;
  a.logp[(size_t)b * a.width + tid] = lp;
  if (tid == 0) a.n_acc[b] = n;
}

// Dynamic shared memory of a tree: per node its row, p of its token at its parent
// (before: that logit), token, parent, random number, first accepted child; the path;
// the tokens rejected at its end.
constexpr size_t tree_smem(int nodes) { return (size_t)nodes * (sizeof(Row) + sizeof(double) + 6 * sizeof(int)); }

template <typename T>
__global__ void __launch_bounds__(kDrawThreads, 3)
tree_draw_kernel(DrawParams a) {
  cluster_arrive();
  grid_dep_wait();
  grid_dep_launch();
  extern __shared__ __align__(16) uint8_t dyn[];
  const int b = blockIdx.x / a.shares, rank = blockIdx.x % a.shares;
  const int tid = threadIdx.x;
  const int n = a.q_lens[b], off = a.q_offsets[b];
  const float t = heat(a.temperature[b]);
  // every CTA of the cluster sees the same values: all leave or none
  if (n < 1 || n > a.max_nodes || off < 0 || off > a.n_rows - n) {
    if (tid == 0 && rank == 0) {
      if (n != 0) report(a.status, KVE_ERR_BOUNDS);
      a.n_acc[b] = -1;
    }
    cluster_wait();
    return;
  }
  Row* rows = reinterpret_cast<Row*>(dyn);
  double* pt = reinterpret_cast<double*>(rows + a.max_nodes);
  int* tok = reinterpret_cast<int*>(pt + a.max_nodes);
  int* par = tok + a.max_nodes;
  float* us = reinterpret_cast<float*>(par + a.max_nodes);
  int* next = reinterpret_cast<int*>(us + a.max_nodes);
  int* path = next + a.max_nodes;
  int* skip = path + a.max_nodes;
  __shared__ int s_n, s_skip, s_strange;
  __shared__ DrawShared sh;
  const T* logits = static_cast<const T*>(a.logits) + (int64_t)off * a.stride;
  if (tid == 0) s_skip = 0;
  // Where offsets do not ascend or sequences share rows, the sums may be of another sequence's temperature: they
  // are this one's if the first and the last row (then also those between) are found to be of one sequence with it.
  if (tid >= kDrawThreads - 32) {
    const int found = search(a.q_offsets, a.batch, tid == kDrawThreads - 1 ? off + n - 1 : off);
    const int last = __shfl_sync(0xffffffffu, found, 31);
    if (tid == kDrawThreads - 32) s_strange = found != last || heat(a.temperature[found]) != t;
  }
  for (int i = tid; i < n; i += kDrawThreads) {
    int d = a.drafts[off + i], pa = a.parents[off + i];
    us[i] = a.u[off + i];
    if (i == 0) pa = -1;
    else if (pa < 0 || pa >= i || d < 0 || d >= a.vocab) {
      if (rank == 0) report(a.status, KVE_ERR_BOUNDS);
      pa = -1;  // nobody's child
    }
    tok[i] = d;
    par[i] = pa;
    next[i] = 0x7fffffff;
    pt[i] = pa < 0 ? 0.0 : (double)Elem<T>::to_f(logits[pa * a.stride + d]);
  }
  join_rows(a.parts, a.n_parts, a.group, t, rows, n, [&](int i) { return off + i; });
  __syncthreads();
  if (s_strange) {
    if (tid == 0 && rank == 0) {
      report(a.status, KVE_ERR_BOUNDS);
      a.n_acc[b] = -1;
    }
    cluster_wait();
    return;
  }
  // p of every node's token at its parent: 0 for a token an earlier sibling has too
  for (int i = tid; i < n; i += kDrawThreads) {
    const int pa = par[i];
    if (pa < 0) continue;
    bool twice = false;
    for (int j = pa + 1; j < i; ++j) twice |= par[j] == pa && tok[j] == tok[i];
    pt[i] = twice ? 0.0 : probability(rows[pa], (float)pt[i], tok[i], t);
  }
  __syncthreads();
  // what a node's earlier siblings leave, should all be rejected; its parent's first accepted child
  for (int i = tid; i < n; i += kDrawThreads) {
    const int pa = par[i];
    if (pa < 0) continue;
    double left = 1.0;
    for (int j = pa + 1; j < i; ++j)
      if (par[j] == pa) left -= pt[j];
    if ((double)us[i] * left < pt[i]) atomicMin(&next[pa], i);
  }
  __syncthreads();
  if (tid == 0) {
    int m = 0;
    path[0] = 0;
    for (int i = next[0]; i < n; i = next[i]) path[++m] = i;
    s_n = m;
  }
  __syncthreads();
  const int m = s_n, node = path[m];
  for (int i = node + 1 + tid; i < n; i += kDrawThreads)
    if (par[i] == node) skip[atomicAdd(&s_skip, 1)] = tok[i];
  __syncthreads();
  const Row p = rows[node];
  Best last;
  if (!(t > 0.f)) {
    cluster_wait();
    last = Best{0.0, p.arg < a.vocab ? p.arg : 0, 0.f};
  } else {
    last = draw<T>(a, sh, logits + node * a.stride, p, static_cast<const T*>(nullptr), p, a.gumbel + b * a.gstride, t, rank,
                   skip, s_skip);
  }
  if (rank != 0) return;
  for (int j = tid; j < a.width; j += kDrawThreads) {
    const size_t to = (size_t)b * a.width + j;
    const int child = j < m ? path[j + 1] : -1;
    a.path[to] = j <= m ? path[j] : -1;
    a.emitted[to] = j < m ? tok[child] : j == m ? last.at : -1;
    a.logp[to] = !(t > 0.f) || j > m ? 0.f : j < m ? (float)log(pt[child]) : log_probability(p, last.x, t);
  }
  if (tid == 0) a.n_acc[b] = m;
}

// ------------------------------------------------------------------ host
// Parts of a row: as many CTAs as fill three a SM, none under 4096 columns.
int stat_parts(int rows, int vocab) {
  const int want = (3 * 148 + rows - 1) / rows;
  const int most = vocab / 4096 < kMaxParts ? vocab / 4096 : kMaxParts;
  return want < most ? want : most < 1 ? 1 : most;
}
// CTAs of a sequence's cluster in the second kernel: at most one wave of them.
int draw_shares(int batch, int vocab) {
  const int want = 3 * 148 / batch, most = vocab / 4096;
  const int n = want < most ? want : most;
  return n > 8 ? 8 : n < 1 ? 1 : n;
}
int lanes_for(int parts) {
  int n = 1;
  while (n < parts) n *= 2;
  return n;
}
int round_up(int n, int to) { return (n + to - 1) / to * to; }
size_t workspace_of(int64_t rows, int vocab) {
  return rows < 1 || vocab < 1 || rows > 0x7fffffff ? 0 : kSharedBytes + (size_t)rows * stat_parts((int)rows, vocab) * sizeof(Part);
}

template <typename T>
int run_stats(const char* me, const Rows& rows, int n_rows, int vocab, const float* temperature, Part* parts, int n_parts,
              cudaStream_t stream) {
  launch_kernel(row_stats_kernel<T>, dim3(n_rows, n_parts), dim3(kStatThreads), 0, stream, rows, vocab,
                round_up((vocab + n_parts - 1) / n_parts, 8), n_parts, temperature, parts);
  return check_launch(me);
}
template <typename Kernel>
int run_draw(const char* me, Kernel kernel, const DrawParams& a, size_t smem, cudaStream_t stream) {
  if (smem > 32768) {  // with the static part, more than a kernel has without asking
    cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (err != cudaSuccess) {
      cudaGetLastError();
      return set_error(KVE_ERR_CUDA, "%s: %s", me, cudaGetErrorString(err));
    }
  }
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = a.shares;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cudaError_t err = launch_kernel_ex(kernel, dim3(a.batch * a.shares), dim3(kDrawThreads), smem, stream, &attr, 1, a);
  if (err != cudaSuccess) {
    cudaGetLastError();
    count_launch();
    return set_error(KVE_ERR_CUDA, "%s: launch failed: %s", me, cudaGetErrorString(err));
  }
  return check_launch(me);
}

}  // namespace
}  // namespace kve

using namespace kve;

extern "C" size_t kve_sample_accept_workspace_bytes(int batch, int k, int vocab, int with_draft_logits) {
  if (batch < 1 || k < 1) return 0;
  return workspace_of((int64_t)batch * (k + 1 + (with_draft_logits ? k : 0)), vocab);
}

extern "C" int kve_sample_accept(const void* logits, int dtype, int64_t row_stride, const void* draft_logits,
                                 int64_t draft_logits_stride_b, int64_t draft_logits_stride_j, const int32_t* drafts,
                                 int64_t draft_stride_b, int64_t draft_stride_j, const float* uniforms,
                                 int64_t uniform_stride_b, const float* gumbel, int64_t gumbel_stride,
                                 const float* temperature, int batch, int k, int vocab, int32_t* out_n_accepted,
                                 int32_t* out_emitted, float* out_logprobs, void* workspace, size_t workspace_bytes,
                                 int* dev_status, cudaStream_t stream) {
  const char* me = "kve_sample_accept";
  if (batch < 0 || k < 1 || k > kMaxK || vocab < 1 || row_stride < vocab || gumbel_stride < vocab || uniform_stride_b < k ||
      (draft_logits && (draft_logits_stride_b < 0 || draft_logits_stride_j < 0)))
    return set_error(KVE_ERR_ARG, "%s: bad sizes batch=%d k=%d vocab=%d", me, batch, k, vocab);
  if (dtype != KVE_F32 && dtype != KVE_BF16) return set_error(KVE_ERR_DTYPE, "%s: dtype %d", me, dtype);
  if (vocab > (1 << 30)) return set_error(KVE_ERR_SHAPE, "%s: vocab %d > 2^30", me, vocab);
  if (batch == 0) return KVE_OK;
  if (!logits || !drafts || !uniforms || !gumbel || !temperature || !out_n_accepted || !out_emitted || !out_logprobs)
    return set_error(KVE_ERR_ARG, "%s: null pointer", me);
  const int64_t n_rows = (int64_t)batch * (k + 1 + (draft_logits ? k : 0));
  if (n_rows > 0x7fffffff || (int64_t)batch * 8 > 0x7fffffff) return set_error(KVE_ERR_SHAPE, "%s: too many rows", me);
  const size_t need = workspace_of(n_rows, vocab);
  if (!workspace || workspace_bytes < need) return set_error(KVE_ERR_WORKSPACE, "%s: workspace needs %zu bytes", me, need);
  if ((uintptr_t)workspace % 16) return set_error(KVE_ERR_ARG, "%s: workspace must be 16-byte aligned", me);
  Part* parts = reinterpret_cast<Part*>(static_cast<uint8_t*>(workspace) + kSharedBytes);
  const int n_parts = stat_parts((int)n_rows, vocab);
  const Rows rows{logits, draft_logits, row_stride, draft_logits_stride_b, draft_logits_stride_j, batch * (k + 1), k + 1, k,
                  nullptr, batch};
  int rc = dtype == KVE_F32 ? run_stats<float>(me, rows, (int)n_rows, vocab, temperature, parts, n_parts, stream)
                            : run_stats<__nv_bfloat16>(me, rows, (int)n_rows, vocab, temperature, parts, n_parts, stream);
  if (rc) return rc;
  DrawParams a{};
  a.logits = logits; a.stride = row_stride; a.draft = draft_logits; a.dsb = draft_logits_stride_b; a.dsj = draft_logits_stride_j;
  a.parts = parts; a.n_parts = n_parts; a.group = lanes_for(n_parts); a.drafts = drafts; a.tsb = draft_stride_b; a.tsj = draft_stride_j;
  a.u = uniforms; a.usb = uniform_stride_b; a.gumbel = gumbel; a.gstride = gumbel_stride; a.temperature = temperature;
  a.batch = batch; a.k = k; a.vocab = vocab; a.shares = draw_shares(batch, vocab);
  a.chunk = round_up((vocab + a.shares - 1) / a.shares, 8);
  a.n_acc = out_n_accepted; a.emitted = out_emitted; a.logp = out_logprobs; a.width = k + 1; a.status = dev_status;
  return dtype == KVE_F32 ? run_draw(me, chain_draw_kernel<float>, a, 0, stream)
                          : run_draw(me, chain_draw_kernel<__nv_bfloat16>, a, 0, stream);
}

extern "C" size_t kve_tree_sample_accept_workspace_bytes(int n_rows, int vocab) { return workspace_of(n_rows, vocab); }

extern "C" int kve_tree_sample_accept(const void* logits, int dtype, int64_t row_stride, const int32_t* tokens,
                                      const int32_t* parents, const int32_t* q_lens, const int32_t* q_offsets,
                                      const float* uniforms, const float* gumbel, int64_t gumbel_stride,
                                      const float* temperature, int batch, int n_rows, int max_q_len, int vocab,
                                      int32_t* out_n_accepted, int32_t* out_path, int32_t* out_emitted,
                                      float* out_logprobs, void* workspace, size_t workspace_bytes, int* dev_status,
                                      cudaStream_t stream) {
  const char* me = "kve_tree_sample_accept";
  if (batch < 0 || n_rows < 0 || max_q_len < 1 || vocab < 1 || row_stride < vocab || gumbel_stride < vocab)
    return set_error(KVE_ERR_ARG, "%s: bad sizes", me);
  if (max_q_len > kMaxNodes) return set_error(KVE_ERR_SHAPE, "%s: max_q_len %d > %d", me, max_q_len, kMaxNodes);
  if (dtype != KVE_F32 && dtype != KVE_BF16) return set_error(KVE_ERR_DTYPE, "%s: dtype %d", me, dtype);
  if (vocab > (1 << 30)) return set_error(KVE_ERR_SHAPE, "%s: vocab %d > 2^30", me, vocab);
  if (batch == 0) return KVE_OK;
  if (n_rows < 1) return set_error(KVE_ERR_ARG, "%s: no rows for %d sequences", me, batch);
  if (!logits || !tokens || !parents || !q_lens || !q_offsets || !uniforms || !gumbel || !temperature || !out_n_accepted ||
      !out_path || !out_emitted || !out_logprobs)
    return set_error(KVE_ERR_ARG, "%s: null pointer", me);
  if ((int64_t)batch * 8 > 0x7fffffff) return set_error(KVE_ERR_SHAPE, "%s: batch too large", me);
  const size_t need = workspace_of(n_rows, vocab);
  if (!workspace || workspace_bytes < need) return set_error(KVE_ERR_WORKSPACE, "%s: workspace needs %zu bytes", me, need);
  if ((uintptr_t)workspace % 16) return set_error(KVE_ERR_ARG, "%s: workspace must be 16-byte aligned", me);
  Part* parts = reinterpret_cast<Part*>(static_cast<uint8_t*>(workspace) + kSharedBytes);
  const int n_parts = stat_parts(n_rows, vocab);
  const Rows rows{logits, nullptr, row_stride, 0, 0, n_rows, 1, 1, q_offsets, batch};
  int rc = dtype == KVE_F32 ? run_stats<float>(me, rows, n_rows, vocab, temperature, parts, n_parts, stream)
                            : run_stats<__nv_bfloat16>(me, rows, n_rows, vocab, temperature, parts, n_parts, stream);
  if (rc) return rc;
  DrawParams a{};
  a.logits = logits; a.stride = row_stride; a.parts = parts; a.n_parts = n_parts; a.group = lanes_for(n_parts); a.drafts = tokens; a.parents = parents;
  a.q_lens = q_lens; a.q_offsets = q_offsets; a.u = uniforms; a.gumbel = gumbel; a.gstride = gumbel_stride;
  a.temperature = temperature; a.batch = batch; a.vocab = vocab; a.n_rows = n_rows; a.max_nodes = max_q_len;
  a.shares = draw_shares(batch, vocab); a.chunk = round_up((vocab + a.shares - 1) / a.shares, 8);
  a.n_acc = out_n_accepted; a.path = out_path; a.emitted = out_emitted; a.logp = out_logprobs; a.width = max_q_len;
  a.status = dev_status;
  const size_t smem = tree_smem(max_q_len);
  return dtype == KVE_F32 ? run_draw(me, tree_draw_kernel<float>, a, smem, stream)
                          : run_draw(me, tree_draw_kernel<__nv_bfloat16>, a, smem, stream);
}

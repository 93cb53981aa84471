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
// row, the maximum m and the sum of e^((x - m) / T) (T <= 0: the argmax instead):
// HBM is its bound. The second runs a cluster of CTAs per sequence: each joins
// the parts' sums of the rows it needs, walks the drafts (every CTA of the cluster
// by itself: a few values) and scans its share of the one row the last token comes
// from, which is often still in L2; the shares' best tokens meet through distributed
// shared memory.
//
// Precision: x - m is taken before it is multiplied by 1 / T, so that large logits
// lose nothing; e^x runs on ex2.approx (2^-22) into fp32 sums of a part's
// thirty-odd values per thread, then pairwise. Acceptance, log-probabilities and
// every thread's best candidate are recomputed in 64 bits from m and the sums, so
// a token changes only where two candidates of one thread lie within fp32
// rounding of each other. A NaN logit counts as minus infinity (never drawn).
#include <math.h>

#include "kve_common.cuh"

namespace kve {
namespace {

constexpr int kStatThreads = 512;
constexpr int kDrawThreads = 512;
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
// NaN as minus infinity.
__device__ __forceinline__ float clean(float x) { return x == x ? x : -INFINITY; }

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
// row's first 16-byte boundary on; `batch(values, first index, n)` gets the vectors.
template <typename T, int THREADS, int U, typename Batch, typename One>
__device__ __forceinline__ void scan(const T* row, int lo, int hi, Batch&& batch, One&& one) {
  constexpr int N = Pack<T>::N;
  const int off = (int)((reinterpret_cast<uintptr_t>(row + lo) & 15) / sizeof(T));
  const int head = min(lo + (off ? N - off : 0), hi);
  const int nvec = (hi - head) / N;
  const uint4* v = reinterpret_cast<const uint4*>(row + head);
  for (int i = lo + threadIdx.x; i < head; i += THREADS) one(Elem<T>::to_f(row[i]), i);
  int i = threadIdx.x;
  for (; i + (U - 1) * THREADS < nvec; i += U * THREADS) {
    uint4 raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = __ldcg(v + i + u * THREADS);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float x[N];
      Pack<T>::unpack(raw[u], x);
      batch(x, head + (i + u * THREADS) * N);
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

// What the first kernel leaves of one part of a row. z: the sum of e^((x - m) / T),
// or, for T <= 0, the column of the maximum.
struct Part {
  float m, z;
};

// Where the rows of the first kernel lie: rows [0, n_first) at `first`, the others
// at `second` (the draft's, rows_b and strides of their own).
struct Rows {
  const void* first;
  const void* second;
  int64_t first_stride;             // elements between consecutive rows
  int64_t second_sb, second_sj;     // elements between sequences, and between a sequence's rows
  int n_first, per_seq, k;          // target rows, and rows of a sequence in each of the two (chain)
  const int32_t* q_offsets;         // tree: a row's sequence is found here (batch + 1 entries)
  int batch;
};

__device__ __forceinline__ int sequence_of(const Rows& r, int row) {
  if (!r.q_offsets) return row < r.n_first ? row / r.per_seq : (row - r.n_first) / r.k;
  int lo = 0, hi = r.batch;  // the last b with q_offsets[b] <= row
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (r.q_offsets[mid] <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <typename T>
__device__ __forceinline__ const T* row_at(const Rows& r, int row) {
  if (row < r.n_first) return static_cast<const T*>(r.first) + row * r.first_stride;
  const int i = row - r.n_first;
  return static_cast<const T*>(r.second) + (i / r.k) * r.second_sb + (i % r.k) * r.second_sj;
}

template <typename T>
__global__ void __launch_bounds__(kStatThreads, 3)
row_stats_kernel(Rows rows, int vocab, int chunk, int parts, const float* temperature, Part* out) {
  grid_dep_wait();
  grid_dep_launch();
  const int row = blockIdx.x, part = blockIdx.y;
  const int lo = part * chunk, hi = min(vocab, lo + chunk);
  const float t = temperature[sequence_of(rows, row)];
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
    scan<T, kStatThreads, 2>(x, lo, hi, batch, one);
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
  const float c = 1.4426950408889634f / t;
  float m = -INFINITY, z = 0.f;
  auto rebase = [&](float top) {
    if (top > m) {
      z *= m == -INFINITY ? 0.f : ex2((m - top) * c);
      m = top;
    }
  };
  auto one = [&](float v, int) {
    v = clean(v);
    rebase(v);
    if (m != -INFINITY) z += v == m ? 1.f : ex2((v - m) * c);
  };
  auto batch = [&](auto& v, int) {
    constexpr int N = Pack<T>::N;
    float top = v[0] = clean(v[0]);
#pragma unroll
    for (int j = 1; j < N; ++j) top = fmaxf(top, v[j] = clean(v[j]));
    rebase(top);
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = ex2((v[j] - base) * c);
#pragma unroll
    for (int w = N / 2; w > 0; w >>= 1)
#pragma unroll
      for (int j = 0; j < w; ++j) v[j] += v[j + w];
    z += v[0];
  };
  scan<T, kStatThreads, 4>(x, lo, hi, batch, one);
  float top = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) sm[warp] = top;
  __syncthreads();
  top = sm[0];
#pragma unroll
  for (int w = 1; w < kStatThreads / 32; ++w) top = fmaxf(top, sm[w]);
  if (top == INFINITY) {
    // infinite logits share the whole probability: count them
    z = 0.f;
    for (int i = lo + threadIdx.x; i < hi; i += kStatThreads) z += Elem<T>::to_f(x[i]) == INFINITY ? 1.f : 0.f;
  } else {
    z = m == -INFINITY ? 0.f : z * ex2((m - top) * c);
  }
  z = warp_sum(z);
  if (lane == 0) sz[warp] = z;
  __syncthreads();
  if (threadIdx.x == 0) {
    float sum = 0.f;
    for (int w = 0; w < kStatThreads / 32; ++w) sum += sz[w];
    out[(size_t)row * parts + part] = Part{top, sum};
  }
}

// A row's parts joined by the 32 lanes of a warp (parts <= 32).
struct Row {
  float m;    // the largest logit
  double z;   // the sum of e^((x - m) / T)
  int arg;    // T <= 0: the column of the largest
};
__device__ __forceinline__ Row join(const Part* parts, int n, float t) {
  const int lane = threadIdx.x & 31;
  Part p{-INFINITY, 0.f};
  if (lane < n) {
    const float2 v = __ldcg(reinterpret_cast<const float2*>(parts) + lane);
    p = Part{v.x, v.y};
  }
  float m = p.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (!(t > 0.f)) {
    int at = lane < n && p.m == m ? __float_as_int(p.z) : 0x7fffffff;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) at = min(at, __shfl_xor_sync(0xffffffffu, at, o));
    return Row{m, 1.0, at};
  }
  double z = lane < n && p.m != -INFINITY ? (p.m == m ? (double)p.z : (double)p.z * exp(((double)p.m - m) / t)) : 0.0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
  return Row{m, z, 0};
}
// (x - m) / T, and p of logit x at column v, in 64 bits.
__device__ __forceinline__ double exponent(float x, float m, float t) { return x == m ? 0.0 : ((double)x - m) / t; }
__device__ __forceinline__ double probability(const Row& r, float x, int v, float t) {
  if (!(t > 0.f)) return v == r.arg ? 1.0 : 0.0;
  x = clean(x);
  if (x == -INFINITY || !(r.z > 0.0)) return 0.0;
  return exp(exponent(x, r.m, t)) / r.z;
}

struct DrawParams {
  const void* logits;       // target rows
  int64_t stride;
  const void* draft;        // chain: draft rows, or null
  int64_t dsb, dsj;
  const Part* parts;        // [rows][n_parts]: target rows, then draft rows
  int n_parts;
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

// A candidate for the last token: its key in 64 bits and its column.
struct Best {
  double key;
  int at;
};
__device__ __forceinline__ void take(Best& b, double key, int at) {
  if (at >= 0 && (b.at < 0 || key > b.key || (key == b.key && at < b.at))) b = Best{key, at};
}

// The draw: best candidate of columns [lo, hi). `qrow` (may be null): subtract the
// draft's distribution. `skip`: tokens that may not be drawn.
template <typename T>
__device__ __forceinline__ Best draw_share(const T* row, const Row& p, const T* qrow, const Row& q, const float* gumbel,
                                           float t, int lo, int hi, const int* skip, int n_skip) {
  Best best{-INFINITY, -1};
  float key = -INFINITY;
  int at = -1;
  const float inv = 1.f / t;
  auto skipped = [&](int v) {
    for (int j = 0; j < n_skip; ++j)
      if (skip[j] == v) return true;
    return false;
  };
  if (!(p.z > 0.0)) return best;
  if (!qrow) {
    auto one = [&](float x, int v) {
      x = clean(x);
      const float e = x == p.m ? 0.f : (x - p.m) * inv;
      const float s = e + gumbel[v];
      if (s > key && !skipped(v)) { key = s; at = v; }
    };
    auto batch = [&](auto& x, int v) {
#pragma unroll
      for (int j = 0; j < Pack<T>::N; ++j) one(x[j], v + j);
    };
    scan<T, kDrawThreads, 1>(row, lo, hi, batch, one);
    if (at >= 0) best = Best{exponent(clean(Elem<T>::to_f(row[at])), p.m, t) + (double)gumbel[at], at};
    return best;
  }
  const float c = 1.4426950408889634f * inv;
  const float zp = (float)(1.0 / p.z), zq = q.z > 0.0 ? (float)(1.0 / q.z) : 0.f;
  const float lzp = (float)log(p.z);
  auto one = [&](float x, int v) {
    x = clean(x);
    const float e = x == p.m ? 0.f : x - p.m;
    const float gv = gumbel[v];
    // log(p - q) <= log p: most columns are out of the question without an exponential
    if (!(e * inv - lzp + gv > key - 1e-4f)) return;
    const float y = clean(Elem<T>::to_f(qrow[v]));
    const float w = ex2(e * c) * zp - (y == q.m ? 1.f : ex2((y - q.m) * c)) * zq;
    if (!(w > 0.f)) return;
    const float s = __logf(w) + gv;
    if (s > key) { key = s; at = v; }
  };
  auto batch = [&](auto& x, int v) {
#pragma unroll
    for (int j = 0; j < Pack<T>::N; ++j) one(x[j], v + j);
  };
  scan<T, kDrawThreads, 1>(row, lo, hi, batch, one);
  if (at >= 0) {
    const double w = probability(p, Elem<T>::to_f(row[at]), at, t) - probability(q, Elem<T>::to_f(qrow[at]), at, t);
    best = Best{(w > 0.0 ? log(w) : (double)key - gumbel[at]) + (double)gumbel[at], at};
  }
  return best;
}

// The best of the whole cluster, in every CTA's thread 0 of rank 0.
__device__ __forceinline__ Best join_shares(Best b, int shares, int rank) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double ok = __shfl_xor_sync(0xffffffffu, b.key, o);
    const int oa = __shfl_xor_sync(0xffffffffu, b.at, o);
    take(b, ok, oa);
  }
  __shared__ double sk[kDrawThreads / 32];
  __shared__ int sa[kDrawThreads / 32];
  __shared__ double mine_key;
  __shared__ int mine_at;
  __syncthreads();  // a second draw: every thread has read the first one's result
  if (lane == 0) { sk[warp] = b.key; sa[warp] = b.at; }
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kDrawThreads / 32; ++w) take(b, sk[w], sa[w]);
    mine_key = b.key;
    mine_at = b.at;
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  // every CTA reads all shares, so that all agree on whether a second scan is needed
  if (threadIdx.x == 0) {
    const uint32_t ak = static_cast<uint32_t>(__cvta_generic_to_shared(&mine_key));
    const uint32_t aa = static_cast<uint32_t>(__cvta_generic_to_shared(&mine_at));
    for (int s = 0; s < shares; ++s) {
      if (s == rank) continue;
      uint32_t rk, ra;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(rk) : "r"(ak), "r"(s));
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(aa), "r"(s));
      double ok;
      int oa;
      asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(ok) : "r"(rk) : "memory");
      asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(oa) : "r"(ra) : "memory");
      take(b, ok, oa);
    }
    sk[0] = b.key;
    sa[0] = b.at;
  }
  // nobody leaves, or writes its share again, before all have read it
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  return Best{sk[0], sa[0]};
}

// Scan, and where nothing may be drawn (every weight zero), scan again for p itself.
template <typename T>
__device__ __forceinline__ int draw(const DrawParams& a, const T* row, const Row& p, const T* qrow, const Row& q,
                                    const float* gumbel, float t, int rank, const int* skip, int n_skip) {
  const int lo = min(rank * a.chunk, a.vocab), hi = min(a.vocab, lo + a.chunk);
  const Row none{0.f, 0.0, 0};
  Best b = join_shares(draw_share<T>(row, p, qrow, q, gumbel, t, lo, hi, skip, n_skip), a.shares, rank);
  if (b.at < 0 && (qrow || n_skip))
    b = join_shares(draw_share<T>(row, p, nullptr, none, gumbel, t, lo, hi, skip, 0), a.shares, rank);
  return b.at < 0 ? 0 : b.at;
}

template <typename T>
__global__ void __launch_bounds__(kDrawThreads)
chain_draw_kernel(DrawParams a) {
  grid_dep_wait();
  grid_dep_launch();
  const int b = blockIdx.x / a.shares, rank = blockIdx.x % a.shares;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int k = a.k;
  const float t = a.temperature[b];
  const T* logits = static_cast<const T*>(a.logits) + (int64_t)b * (k + 1) * a.stride;
  const T* draft = a.draft ? static_cast<const T*>(a.draft) + b * a.dsb : nullptr;
  __shared__ Row prow[kMaxK + 1], qrow[kMaxK];
  __shared__ double pd[kMaxK], qd[kMaxK];
  __shared__ int tok[kMaxK];
  __shared__ int n_s;
  for (int r = warp; r < 2 * k + 1; r += kDrawThreads / 32) {
    if (r > k && !draft) break;
    const int row = r <= k ? b * (k + 1) + r : a.batch * (k + 1) + b * k + (r - k - 1);
    const Row x = join(a.parts + (size_t)row * a.n_parts, a.n_parts, t);
    if (lane != 0) continue;
    const int j = r <= k ? r : r - k - 1;
    (r <= k ? prow : qrow)[j] = x;
    if (j == k) continue;
    const int d = a.drafts[b * a.tsb + j * a.tsj];
    const bool ok = d >= 0 && d < a.vocab;
    const double pr = !ok ? 0.0 : probability(x, Elem<T>::to_f((r <= k ? logits + j * a.stride : draft + j * a.dsj)[d]), d, t);
    (r <= k ? pd : qd)[j] = pr;
    if (r <= k) {
      if (!ok && rank == 0) report(a.status, KVE_ERR_BOUNDS);
      tok[j] = ok ? d : -1;
      if (!draft) qd[j] = 1.0;
    }
  }
  __syncthreads();
  if (warp == 0) {
    const bool no = lane < k && !(tok[lane] >= 0 && (double)a.u[b * a.usb + lane] * qd[lane] < pd[lane]);
    const unsigned m = __ballot_sync(0xffffffffu, no);
    if (lane == 0) n_s = m ? __ffs(m) - 1 : k;
  }
  __syncthreads();
  const int n = n_s;
  const T* row = logits + n * a.stride;
  const float* gumbel = a.gumbel + b * a.gstride;
  const Row p = prow[n];
  int last;
  if (!(t > 0.f)) {
    last = p.arg;  // one-hot: a rejected draft was another token
    if (last < 0 || last >= a.vocab) last = 0;
  } else {
    const bool sub = draft && n < k;
    last = draw<T>(a, row, p, sub ? draft + n * a.dsj : nullptr, sub ? qrow[n] : p, gumbel, t, rank, tok + n,
                   !draft && n < k ? 1 : 0);
  }
  if (rank != 0 || warp != 0) return;
  if (lane <= k) {
    const int e = lane < n ? tok[lane] : lane == n ? last : -1;
    float lp = 0.f;
    if (lane <= n && t > 0.f) {
      const Row& r = prow[lane];
      const float x = clean(Elem<T>::to_f(logits[lane * a.stride + e]));
      lp = r.z > 0.0 && x != -INFINITY ? (float)(exponent(x, r.m, t) - log(r.z)) : -INFINITY;
    }
    a.emitted[(size_t)b * a.width + lane] = e;
    a.logp[(size_t)b * a.width + lane] = lp;
  }
  if (lane == 0) a.n_acc[b] = n;
}

// Dynamic shared memory of the tree: per node its token, parent, p at its parent,
// random number; then the path and the rejected tokens of its last node.
constexpr size_t tree_smem(int nodes) { return (size_t)nodes * (sizeof(double) + 3 * sizeof(int) + 2 * sizeof(int)); }

template <typename T>
__global__ void __launch_bounds__(kDrawThreads)
tree_draw_kernel(DrawParams a) {
  grid_dep_wait();
  grid_dep_launch();
  extern __shared__ __align__(16) uint8_t dyn[];
  const int b = blockIdx.x / a.shares, rank = blockIdx.x % a.shares;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n = a.q_lens[b], off = a.q_offsets[b];
  const float t = a.temperature[b];
  // every CTA of the cluster sees the same values: all leave or none
  if (n < 1 || n > a.max_nodes || off < 0 || off > a.n_rows - n) {
    if (threadIdx.x == 0 && rank == 0) {
      if (n != 0) report(a.status, KVE_ERR_BOUNDS);
      a.n_acc[b] = -1;
    }
    return;
  }
  double* pt = reinterpret_cast<double*>(dyn);
  int* tok = reinterpret_cast<int*>(pt + a.max_nodes);
  int* par = tok + a.max_nodes;
  float* us = reinterpret_cast<float*>(par + a.max_nodes);
  int* path = reinterpret_cast<int*>(us + a.max_nodes);
  int* skip = path + a.max_nodes;
  __shared__ int s_n, s_skip;
  const T* logits = static_cast<const T*>(a.logits) + (int64_t)off * a.stride;
  for (int i = threadIdx.x; i < n; i += kDrawThreads) {
    int d = a.drafts[off + i], pa = a.parents[off + i];
    if (i == 0) pa = -1;
    else if (pa < 0 || pa >= i || d < 0 || d >= a.vocab) {
      if (rank == 0) report(a.status, KVE_ERR_BOUNDS);
      pa = -1;  // nobody's child
    }
    tok[i] = d;
    par[i] = pa;
    us[i] = a.u[off + i];
  }
  __syncthreads();
  // p of every node's token at its parent (0 for a token an earlier sibling has too).
  for (int i = warp; i < n; i += kDrawThreads / 32) {
    const int pa = par[i];
    if (pa < 0) continue;
    bool twice = false;
    for (int j = pa + 1 + lane; j < i; j += 32) twice |= par[j] == pa && tok[j] == tok[i];
    twice = __any_sync(0xffffffffu, twice);
    const Row r = join(a.parts + (size_t)(off + pa) * a.n_parts, a.n_parts, t);
    if (lane == 0) pt[i] = twice ? 0.0 : probability(r, Elem<T>::to_f(logits[pa * a.stride + tok[i]]), tok[i], t);
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    int cur = 0, m = 0, rejected = 0;
    double left = 1.0;
    path[0] = 0;
    for (int i = 1; i < n; ++i) {
      if (par[i] != cur) continue;
      if ((double)us[i] * left < pt[i]) {
        cur = i;
        path[++m] = i;
        left = 1.0;
        rejected = 0;
      } else {
        left -= pt[i];
        skip[rejected++] = tok[i];
      }
    }
    s_n = m;
    s_skip = rejected;
  }
  __syncthreads();
  const int m = s_n;
  const int node = path[m];
  const Row p = join(a.parts + (size_t)(off + node) * a.n_parts, a.n_parts, t);
  int last;
  if (!(t > 0.f)) {
    last = p.arg;
    if (last < 0 || last >= a.vocab) last = 0;
  } else {
    last = draw<T>(a, logits + node * a.stride, p, nullptr, p, a.gumbel + b * a.gstride, t, rank, skip, s_skip);
  }
  if (rank != 0) return;
  for (int j = warp; j < a.width; j += kDrawThreads / 32) {
    const int at = j <= m ? path[j] : -1;
    const int e = j < m ? tok[path[j + 1]] : j == m ? last : -1;
    float lp = 0.f;
    if (j <= m && t > 0.f) {
      const Row r = join(a.parts + (size_t)(off + at) * a.n_parts, a.n_parts, t);
      const float x = clean(Elem<T>::to_f(logits[at * a.stride + e]));
      lp = r.z > 0.0 && x != -INFINITY ? (float)(exponent(x, r.m, t) - log(r.z)) : -INFINITY;
    }
    if (lane != 0) continue;
    a.path[(size_t)b * a.width + j] = at;
    a.emitted[(size_t)b * a.width + j] = e;
    a.logp[(size_t)b * a.width + j] = lp;
  }
  if (threadIdx.x == 0) a.n_acc[b] = m;
}

// ------------------------------------------------------------------ host
// Parts of a row: as many CTAs as fill three a SM, none under 4096 columns.
int stat_parts(int rows, int vocab) {
  const int want = (3 * 148 + rows - 1) / rows;
  const int most = vocab / 4096 < kMaxParts ? vocab / 4096 : kMaxParts;
  return want < most ? want : most < 1 ? 1 : most;
}
// CTAs of a sequence's cluster in the second kernel.
int draw_shares(int batch, int vocab) {
  const int want = 3 * 148 / batch, most = vocab / 4096;
  const int n = want < most ? want : most;
  return n >= 8 ? 8 : n >= 4 ? 4 : n >= 2 ? 2 : 1;
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
  a.parts = parts; a.n_parts = n_parts; a.drafts = drafts; a.tsb = draft_stride_b; a.tsj = draft_stride_j;
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
  a.logits = logits; a.stride = row_stride; a.parts = parts; a.n_parts = n_parts; a.drafts = tokens; a.parents = parents;
  a.q_lens = q_lens; a.q_offsets = q_offsets; a.u = uniforms; a.gumbel = gumbel; a.gstride = gumbel_stride;
  a.temperature = temperature; a.batch = batch; a.vocab = vocab; a.n_rows = n_rows; a.max_nodes = max_q_len;
  a.shares = draw_shares(batch, vocab); a.chunk = round_up((vocab + a.shares - 1) / a.shares, 8);
  a.n_acc = out_n_accepted; a.path = out_path; a.emitted = out_emitted; a.logp = out_logprobs; a.width = max_q_len;
  a.status = dev_status;
  const size_t smem = tree_smem(max_q_len);
  return dtype == KVE_F32 ? run_draw(me, tree_draw_kernel<float>, a, smem, stream)
                          : run_draw(me, tree_draw_kernel<__nv_bfloat16>, a, smem, stream);
}

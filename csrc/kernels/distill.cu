// Distillation from a teacher's top logits.
//
// Row n has student logits x (V values) and K teacher entries (logit t_k, token
// id_k).  An entry counts when 0 <= id_k < V and t_k is not -inf; a row without
// such entries has loss 0 and gradient 0.  With temperature T:
//
//   p = softmax(t / T) over the counted entries,  q = softmax(x / T) over all V
//   loss_n  = T^2 sum_k p_k (ln p_k - ln q[id_k])
//   dx_j    = T g_n (q_j - sum of p_k with id_k = j)
//
// The vocabulary is read once per direction.  The forward keeps a running maximum and
// a running sum per thread and joins them; the backward needs four numbers a row and
// the probabilities p.  Everything is fp32, in powers of two with k2 = log2(e) / T:
// with B = m k2 rounded once (any reference near the maximum would do, as long as both
// sides use the same), log2 q_j = (x_j k2 - B) - log2 s, the bracket one fma.  At the
// maximum the bracket is the rounding error of B, up to half a step of it, which grows
// with |m|: within F = 2^22 / k2 it stays below 1/4.  So B is taken from m kept within
// +-F (far_limit); what lies below -F (a mask) adds 2^-huge = 0 beside any logit above.
// Rows whose maximum is itself beyond F (rows that hold nothing but a mask, or a huge
// offset) take differences x - m first, in a second walk of the forward.
//
// Bounded by the bytes of the logits: 16384 x 32000 bf16 with 64 entries forward 195 us
// (5.4 TB/s) and backward 317 to 334 us (6.3 to 6.6 TB/s), 4093 x 100287 fp32 with 200
// entries 256 to 261 us and 559 to 590 us (6.3 to 6.4 and 5.6 to 5.9 TB/s).  The 16-bit
// forward is the furthest from the copy rate (6.5 TB/s): no unit is at its limit (special
// functions 71 % busy, issue slots and DRAM 58 %; a quarter of the exponentials on the FMA
// pipe made it slower), its loads run dry at the end of each row, which a block takes in
// four steps, joins and leaves.  Rows beyond the limit are read twice in the forward:
// 16384 x 32000 bf16 of them 312 and 377 us.
#include "../common.cuh"
#include "sm100.cuh"

#include <cmath>

namespace lrb {
namespace {

using namespace sm100;

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kPerThread = 4;                   // teacher entries a thread holds
constexpr int kMaxK = kPerThread * kThreads;    // entries of a row, for a block a row
constexpr int kWarpK = kPerThread * 32;         // for a warp a row
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Vectors in flight a thread (U) and blocks an SM, measured.  Forward: 16384 x 32000 bf16
// 196 us at 4 / 6 (212 at 4 / 5, 194 at 4 / 8; a warp a row 199 at 8 / 4), 2048 x 100287
// bf16 80 us at 4 / 6 (79 at 4 / 5, 83 at 4 / 8); 4093 x 100287 fp32 261 us at 8 / 4 (291 at
// 4 / 6).  Backward: 320 us at 4 / 5 (335 at 4 / 8, 338 at 8 / 4), fp32 559 us at 4 / 4
// (587 at 4 / 5).
template <typename T, int W> constexpr int kFwdU = W == 1 || sizeof(T) == 4 ? 8 : 4;
template <typename T, int W> constexpr int kFwdBlocks = W == 1 || sizeof(T) == 4 ? 4 : 6;
template <typename T, int W> constexpr int kBwdU = W == 1 ? 8 : 4;
template <typename T, int W> constexpr int kBwdBlocks = W == 1 || sizeof(T) == 4 ? 4 : 5;

struct Teacher {
  const void* logits;  // (N, K) bf16 / fp16 / fp32
  const void* ids;     // (N, K) int64 / int32
  int type;            // 0 fp32, 1 bf16, 2 fp16
  int wide;            // ids are int64
  int K;
};

__device__ __forceinline__ float teacher_logit(const Teacher& t, int64_t i) {
  if (t.type == 0) return reinterpret_cast<const float*>(t.logits)[i];
  if (t.type == 1) return to_f(reinterpret_cast<const __nv_bfloat16*>(t.logits)[i]);
  return to_f(reinterpret_cast<const __half*>(t.logits)[i]);
}
__device__ __forceinline__ int teacher_id(const Teacher& t, int64_t i, int V) {  // -1: does not count
  const int64_t id = t.wide ? reinterpret_cast<const int64_t*>(t.ids)[i] : reinterpret_cast<const int*>(t.ids)[i];
  return id >= 0 && id < V ? (int)id : -1;
}

// What the forward leaves for the backward.
struct RowStats {
  float base, log2_s, m, counted;
};

template <typename T> struct Pairs;  // a 16-byte vector as packed fp32 pairs, and its maximum
template <> struct Pairs<__nv_bfloat16> {
  static constexpr int N = 4;
  static __device__ __forceinline__ uint64_t get(const uint4& r, int i) {
    const uint32_t w = i == 0 ? r.x : i == 1 ? r.y : i == 2 ? r.z : r.w;
    return f2_pack(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t put(float2 v) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  template <int U>
  static __device__ __forceinline__ float max(const uint4 (&r)[U]) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&r);
    __nv_bfloat162 m = h[0];
#pragma unroll
    for (int i = 1; i < 4 * U; ++i) m = __hmax2(m, h[i]);
    const float2 f = __bfloat1622float2(m);
    return fmaxf(f.x, f.y);
  }
};
template <> struct Pairs<__half> {
  static constexpr int N = 4;
  static __device__ __forceinline__ uint64_t get(const uint4& r, int i) {
    const uint32_t w = i == 0 ? r.x : i == 1 ? r.y : i == 2 ? r.z : r.w;
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    return f2_pack(f.x, f.y);
  }
  static __device__ __forceinline__ uint32_t put(float2 v) {
    const __half2 h = __floats2half2_rn(v.x, v.y);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  template <int U>
  static __device__ __forceinline__ float max(const uint4 (&r)[U]) {
    const __half2* h = reinterpret_cast<const __half2*>(&r);
    __half2 m = h[0];
#pragma unroll
    for (int i = 1; i < 4 * U; ++i) m = __hmax2(m, h[i]);
    const float2 f = __half22float2(m);
    return fmaxf(f.x, f.y);
  }
};
template <> struct Pairs<float> {
  static constexpr int N = 2;
  static __device__ __forceinline__ uint64_t get(const uint4& r, int i) {
    return i == 0 ? f2_pack(__uint_as_float(r.x), __uint_as_float(r.y))
                  : f2_pack(__uint_as_float(r.z), __uint_as_float(r.w));
  }
  template <int U>
  static __device__ __forceinline__ float max(const uint4 (&r)[U]) {
    const float* f = reinterpret_cast<const float*>(&r);
    float m = f[0];
#pragma unroll
    for (int i = 1; i < 4 * U; ++i) m = fmaxf(m, f[i]);
    return m;
  }
};

// The largest maximum with a base of its own: |base| <= 2^22, finite for every k2.
__device__ __forceinline__ float far_limit(float k2) { return fminf(__fdividef(4194304.f, k2), 1e30f); }

// The base that goes with a maximum.  Rounded here: contracted into a following
// subtraction, the bases of one maximum would differ by their rounding.
__device__ __forceinline__ float base_of(float m, float k2) {
  const float f = far_limit(k2);
  return __fmul_rn(fminf(fmaxf(m, -f), f), k2);
}

// Running maximum m and sum of 2^(x k2 - base), base = ref k2 with ref the maximum kept
// within +-far_limit: below, everything so far adds nothing beside a larger logit
// (2^-huge = 0), and a NaN shows.
struct Online {
  float m = -INFINITY, base;
  uint64_t s = 0;  // two partial sums
  __device__ __forceinline__ explicit Online(float k2) : base(base_of(-INFINITY, k2)) {}
  __device__ __forceinline__ void raise(float mx, float k2) {
    if (mx > m) {
      const float b = base_of(mx, k2);
      const float f = fast_exp2(base - b);
      s = f2_mul(s, f2_pack(f, f));
      m = mx;
      base = b;
    }
  }
  __device__ __forceinline__ void add(float x, float k2) {
    raise(x, k2);
    s = f2_add(s, f2_pack(fast_exp2(fmaf(x, k2, -base)), 0.f));
  }
  template <typename T, int U>
  __device__ __forceinline__ void add_vecs(const uint4 (&r)[U], float k2) {
    raise(Pairs<T>::template max<U>(r), k2);  // one for all of them
    const uint64_t kk = f2_pack(k2, k2), nb = f2_pack(-base, -base);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < Pairs<T>::N; ++i) {
        const float2 e = f2_unpack(f2_fma(Pairs<T>::get(r[u], i), kk, nb));
        s = f2_add(s, f2_pack(fast_exp2(e.x), fast_exp2(e.y)));
      }
  }
  __device__ __forceinline__ float sum() const {
    const float2 v = f2_unpack(s);
    return v.x + v.y;
  }
};

// (m, s) pairs whose s refer to the base of their own m, joined over a warp.
__device__ __forceinline__ float2 warp_join(float2 v, float k2) {
  const float m = warp_max(v.x);
  return make_float2(m, warp_sum(v.y * fast_exp2(base_of(v.x, k2) - base_of(m, k2))));
}

__device__ __forceinline__ void cluster_barrier() {
  __syncthreads();  // the aligned forms want converged warps
  cluster_sync();
}
__device__ __forceinline__ float2 ld_peer(const float2* p, unsigned rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
               : "=f"(v.x), "=f"(v.y)
               : "r"(mapa_shared(smem_addr(p), rank))
               : "memory");
  return v;
}

struct Rows {  // (outer, inner) strides of the logits' rows, unit stride along the vocabulary
  int64_t inner, s_outer, s_inner;
};
template <typename T>
__device__ __forceinline__ const T* row_ptr(const T* x, const Rows& r, int64_t n) {
  const int64_t o = n / r.inner;
  return x + o * r.s_outer + (n - o * r.inner) * r.s_inner;
}

// The elements of [p, p + len) by `step` threads: `one` for those before the first and
// behind the last 16-byte boundary, `all` for U vectors at a time (loaded together, no
// bounds to look at), `vec` for the last ones.
template <int U, typename T, typename One, typename All, typename Vec>
__device__ __forceinline__ void walk(const T* p, int len, int tid, int step, One one, All all, Vec vec) {
  constexpr int VEC = 16 / sizeof(T);
  const int head = min(len, (int)(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T)));
  const int nvec = (len - head) / VEC, tail = len - head - nvec * VEC;
  if (tid < head) one(tid);
  if (tid < tail) one(len - tail + tid);
  const uint4* b = reinterpret_cast<const uint4*>(p + head);
  int i = tid;
  for (; i + (U - 1) * step < nvec; i += U * step) {
    uint4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = __ldg(b + i + u * step);
    all(head + i * VEC, step * VEC, v);
  }
  if (i < nvec) {
    uint4 v[U - 1];
#pragma unroll
    for (int u = 0; u < U - 1; ++u)
      if (i + u * step < nvec) v[u] = __ldg(b + i + u * step);
#pragma unroll
    for (int u = 0; u < U - 1; ++u)
      if (i + u * step < nvec) vec(head + (i + u * step) * VEC, v[u]);
  }
}

// The teacher's side of a row over some of its entries, w = 2^((y - mx) k2):
// S0 = sum w, S1 = sum w (y - mx) k2, S2 = sum w (x[id] - m) k2 with m the row's largest
// logit (an offset of all logits, or a masked one among them, costs no precision), so
// that sum p (log2 p - (x[id] - m) k2) = (S1 - S2) / S0 - log2 S0.  S0 = 0: no entries.
struct Entries {
  float mx, s0, s1, s2;
};
__device__ __forceinline__ Entries join(const Entries& a, const Entries& b, float k2) {
  const float mx = fmaxf(a.mx, b.mx);
  Entries r{mx, 0.f, 0.f, 0.f};
  const auto put = [&](const Entries& e) {
    if (e.s0 == 0.f) return;
    const float d = e.mx == mx ? 0.f : (e.mx - mx) * k2, f = fast_exp2(d);
    if (f == 0.f && e.s0 == e.s0) return;
    r.s0 += f * e.s0;
    r.s1 += f * (e.s1 + e.s0 * d);
    r.s2 += f * e.s2;
  };
  put(a);
  put(b);
  return r;
}

// W = 1: a row a warp, without any barrier.  W = 8: a row a block, or, where the rows
// do not fill the GPU, a cluster whose blocks take equal ranges of the vocabulary (the
// first one does the teacher's side).
template <typename T, int W>
__global__ void __launch_bounds__(kThreads, (kFwdBlocks<T, W>))
    distill_fwd_kernel(const T* __restrict__ logits, Rows rows, int64_t n, int V, Teacher t, float temp,
                       float* __restrict__ loss, float* __restrict__ counted, RowStats* __restrict__ stats,
                       float* __restrict__ probs) {
  __shared__ float2 part[kWarps], mine;
  __shared__ Entries entries[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const unsigned rank = W == 1 ? 0 : cluster_ctarank(), split = W == 1 ? 1 : cluster_nctarank();
  const int64_t row = W == 1 ? (int64_t)blockIdx.x * kWarps + warp : blockIdx.x / split;
  if (row >= n) return;  // W = 1 only: whole warps
  const T* x = row_ptr(logits, rows, row);
  const int c0 = (int)((int64_t)V * rank / split), c1 = (int)((int64_t)V * (rank + 1) / split);
  const float k2 = kLog2e / temp;
  const int tid = W == 1 ? lane : threadIdx.x;

  // The first entry of each thread (mostly the only one) is loaded ahead of the long walk
  // and looked at behind it.
  int id[kPerThread];
  float y[kPerThread];
  const auto load_entry = [&](int i) {
    const int k = tid + i * 32 * W;
    id[i] = -1;
    y[i] = 0.f;
    if (k < t.K) {
      id[i] = teacher_id(t, row * t.K + k, V);
      y[i] = teacher_logit(t, row * t.K + k);
    }
  };
  if (rank == 0) load_entry(0);
  Online o(k2);
  constexpr int U = kFwdU<T, W>;
  walk<U>(
      x + c0, c1 - c0, tid, 32 * W, [&](int i) { o.add(to_f(x[c0 + i]), k2); },
      [&](int, int, const uint4 (&v)[U]) { o.add_vecs<T, U>(v, k2); },
      [&](int, const uint4& v) {
        const uint4 one[1] = {v};
        o.add_vecs<T, 1>(one, k2);
      });
  float2 ms = warp_join(make_float2(o.m, o.sum()), k2);
  if constexpr (W > 1) {
    if (lane == 0) part[warp] = ms;
    __syncthreads();
    ms = warp_join(lane < kWarps ? part[lane] : make_float2(-INFINITY, 0.f), k2);
    if (split > 1) {
      if (threadIdx.x == 0) mine = ms;
      cluster_barrier();
      if (rank == 0) ms = warp_join(lane < split ? ld_peer(&mine, (unsigned)lane) : make_float2(-INFINITY, 0.f), k2);
      cluster_barrier();  // every block's `mine` has been read
      if (rank != 0) return;
    }
  }
  const float m = ms.x;
  float rest = fmaf(-m, k2, base_of(m, k2));  // the rounding of the base
  if (fabsf(m) > far_limit(k2) && fabsf(m) < INFINITY) {  // differences to m first: the row again, by every warp
    float s = 0.f;
    const auto one = [&](int i) { s += fast_exp2((to_f(x[i]) - m) * k2); };
    const auto vec = [&](int, const uint4& v) {
#pragma unroll
      for (int j = 0; j < Pairs<T>::N; ++j) {
        const float2 f = f2_unpack(Pairs<T>::get(v, j));
        s += fast_exp2((f.x - m) * k2) + fast_exp2((f.y - m) * k2);
      }
    };
    walk<2>(x, V, tid, 32 * W, one, [&](int, int, const uint4 (&v)[2]) { vec(0, v[0]), vec(0, v[1]); }, vec);
    ms.y = warp_sum(s);
    if constexpr (W > 1) {
      __syncthreads();  // `part` has been read
      if (lane == 0) part[warp].y = ms.y;
      __syncthreads();
      ms.y = warp_sum(lane < kWarps ? part[lane].y : 0.f);
    }
    rest = 0.f;
  }

  Entries e{-INFINITY, 0.f, 0.f, 0.f};
  if (W == 1 || warp * 32 < t.K) {
#pragma unroll
    for (int i = 1; i < kPerThread; ++i) load_entry(i);
    float xg[kPerThread];
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      if (y[i] == -INFINITY) id[i] = -1;
      xg[i] = id[i] >= 0 ? to_f(x[id[i]]) : 0.f;
      if (id[i] >= 0) e.mx = fmaxf(e.mx, y[i]);
    }
    e.mx = warp_max(e.mx);
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      if (id[i] < 0) continue;
      const float d = (y[i] - e.mx) * k2, w = fast_exp2(d);
      if (w == 0.f) continue;
      e.s0 += w;
      e.s1 += w * d;
      e.s2 += w * ((xg[i] - m) * k2);
    }
    e.s0 = warp_sum(e.s0);
    e.s1 = warp_sum(e.s1);
    e.s2 = warp_sum(e.s2);
  }
  if constexpr (W > 1) {
    if (lane == 0) entries[warp] = e;
    __syncthreads();
    e = entries[0];  // every thread joins them, in one order
#pragma unroll
    for (int w = 1; w < kWarps; ++w) e = join(e, entries[w], k2);
  }
  const bool some = e.s0 != 0.f;
  if (probs != nullptr) {
    const float inv = 1.f / e.s0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      const int k = tid + i * 32 * W;
      if (k < t.K) probs[row * t.K + k] = id[i] >= 0 ? fast_exp2((y[i] - e.mx) * k2) * inv : 0.f;
    }
  }
  if (W > 1 && warp != 0) return;
  if (lane == 0) {
    const float log2_s = log2f(ms.y);
    stats[row] = RowStats{base_of(m, k2), log2_s, m, some ? 1.f : 0.f};
    // sum p (log2 p - log2 q) = sum p (log2 p - (x[id] - m) k2) + (base - m k2) + log2 s
    const float a = (e.s1 - e.s2) / e.s0 - log2f(e.s0);
    loss[row] = some ? temp * temp * kLn2 * (a + (rest + log2_s)) : 0.f;
    counted[row] = some ? 1.f : 0.f;
  }
}

// The loss (sum of the rows, over the number of counted rows for a mean) and each
// counted row's factor in it.  One block, fixed order.
__global__ void __launch_bounds__(1024) reduce_rows_kernel(const float* __restrict__ loss,
                                                           const float* __restrict__ counted, int64_t n, int mean,
                                                           float* __restrict__ out, float* __restrict__ factor) {
  __shared__ double rs[32], rc[32];
  double s = 0.0, c = 0.0;
  for (int64_t i = threadIdx.x; i < n; i += 1024) {
    s += (double)loss[i];
    c += (double)counted[i];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    c += __shfl_xor_sync(0xffffffffu, c, o);
  }
  if ((threadIdx.x & 31) == 0) {
    rs[threadIdx.x >> 5] = s;
    rc[threadIdx.x >> 5] = c;
  }
  __syncthreads();
  if (threadIdx.x == 0) {
    s = c = 0.0;
    for (int w = 0; w < 32; ++w) {
      s += rs[w];
      c += rc[w];
    }
    const double f = mean ? 1.0 / (c > 1.0 ? c : 1.0) : 1.0;
    *out = (float)(s * f);
    *factor = (float)f;
  }
}

// W = 1: a row a warp; W = 8: `split` blocks a row, each a range of it.  The range of q
// is written scaled, then the entries that lie in it are put right.  The last rows come
// first: they are the ones that the forward left in L2.
template <typename T, int W>
__global__ void __launch_bounds__(kThreads, (kBwdBlocks<T, W>))
    distill_bwd_kernel(const T* __restrict__ logits, Rows rows, int64_t n, int V, Teacher t, float temp,
                       const float* __restrict__ probs, const RowStats* __restrict__ stats, const float* __restrict__ g,
                       int g_per_row, const float* __restrict__ factor, T* __restrict__ dx, Rows dx_rows, int split) {
  __shared__ int all_ids[kMaxK], all_seen[2 * kMaxK];
  __shared__ float all_p[kMaxK];
  constexpr int VEC = 16 / sizeof(T), G = 32 * W;
  const int tid = W == 1 ? threadIdx.x & 31 : threadIdx.x, group = W == 1 ? threadIdx.x >> 5 : 0;
  int* ids = all_ids + group * kWarpK;
  int* seen = all_seen + group * 2 * kWarpK;
  float* sp = all_p + group * kWarpK;
  const unsigned block = gridDim.x - 1 - blockIdx.x;
  const int64_t row = W == 1 ? (int64_t)block * kWarps + group : block / split;
  if (row >= n) return;  // W = 1 only: whole warps
  const int part = W == 1 ? 0 : (int)(block - row * split);
  const T* x = row_ptr(logits, rows, row);
  T* d = const_cast<T*>(row_ptr<T>(dx, dx_rows, row));
  const int c0 = (int)((int64_t)V * part / split), c1 = (int)((int64_t)V * (part + 1) / split);
  const int len = c1 - c0;
  const float4 st = __ldg(reinterpret_cast<const float4*>(stats + row));
  const float base = st.x, l2 = st.y, m = st.z;
  T* dp = d + c0;
  if (st.w == 0.f) {  // no teacher
    const int head = min(len, (int)(((16 - (reinterpret_cast<uintptr_t>(dp) & 15)) & 15) / sizeof(T)));
    const int nvec = (len - head) / VEC, tail = len - head - nvec * VEC;
    if (tid < head) dp[tid] = from_f<T>(0.f);
    if (tid < tail) dp[len - tail + tid] = from_f<T>(0.f);
    for (int i = tid; i < nvec; i += G)
      *reinterpret_cast<uint4*>(dp + head + (int64_t)i * VEC) = make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  const float k2 = kLog2e / temp;
  const float coef = temp * (g_per_row ? g[row] : g[0] * factor[0]);
  const bool far = !(fabsf(m) <= far_limit(k2));
  const auto q = [&](float v) { return fast_exp2((far ? (v - m) * k2 : fmaf(v, k2, -base)) - l2); };

  // The entries of this range: the first of each thread (mostly the only one) is loaded
  // ahead of the long walk and looked at behind it.
  int id[kPerThread];
  float p[kPerThread];
  const auto load_entry = [&](int i) {
    const int k = tid + i * G;
    id[i] = -1;
    p[i] = 0.f;
    if (k < t.K) {
      id[i] = teacher_id(t, row * t.K + k, V);
      p[i] = __ldg(probs + row * t.K + k);
    }
  };
  load_entry(0);
  int size = 64;
  while (size < 2 * t.K) size *= 2;
  for (int i = tid; i < size; i += G) seen[i] = -1;

  const T* xp = x + c0;
  if ((reinterpret_cast<uintptr_t>(xp) & 15) == (reinterpret_cast<uintptr_t>(dp) & 15)) {
    const uint64_t kk = f2_pack(k2, k2), nb = f2_pack(-base, -base), nl = f2_pack(-l2, -l2), cc = f2_pack(coef, coef);
    const auto put = [&](auto is_far, int i, const uint4& v) {
      uint32_t o[4];
#pragma unroll
      for (int j = 0; j < Pairs<T>::N; ++j) {
        const uint64_t xx = Pairs<T>::get(v, j);
        const float2 e = f2_unpack(f2_add(decltype(is_far)::value ? f2_mul(f2_add(xx, f2_pack(-m, -m)), kk)
                                                                  : f2_fma(xx, kk, nb), nl));
        const float2 r = f2_unpack(f2_mul(f2_pack(fast_exp2(e.x), fast_exp2(e.y)), cc));
        if constexpr (sizeof(T) == 4) {
          o[2 * j] = __float_as_uint(r.x);
          o[2 * j + 1] = __float_as_uint(r.y);
        } else {
          o[j] = Pairs<T>::put(r);
        }
      }
      *reinterpret_cast<uint4*>(dp + i) = make_uint4(o[0], o[1], o[2], o[3]);
    };
    const auto run = [&](auto is_far, auto unroll) {
      constexpr int U = decltype(unroll)::value;
      walk<U>(
          xp, len, tid, G, [&](int i) { dp[i] = from_f<T>(coef * q(to_f(xp[i]))); },
          [&](int i, int step, const uint4 (&v)[U]) {
#pragma unroll
            for (int u = 0; u < U; ++u) put(is_far, i + u * step, v[u]);
          },
          [&](int i, const uint4& v) { put(is_far, i, v); });
    };
    if (!far) run(std::false_type{}, std::integral_constant<int, kBwdU<T, W>>{});
    else run(std::true_type{}, std::integral_constant<int, 2>{});
  } else {
    for (int i = tid; i < len; i += G) dp[i] = from_f<T>(coef * q(to_f(xp[i])));
  }
#pragma unroll
  for (int i = 1; i < kPerThread; ++i) load_entry(i);
  if (W == 1) __syncwarp();
  else __syncthreads();
  // An open-addressing table of the tokens finds out whether one is listed twice (its
  // probabilities add up).
  int twice = 0;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int k = tid + i * G;
    if (k >= t.K) continue;
    if (id[i] < c0 || id[i] >= c1) id[i] = -1;
    ids[k] = id[i];
    sp[k] = p[i];
    if (id[i] < 0) continue;
    unsigned h = (unsigned)id[i] * 2654435761u;
    for (h ^= h >> 15;; ++h) {  // at most K of at least 2 K places are taken
      const int was = atomicCAS(&seen[h & (size - 1)], -1, id[i]);
      if (was == -1) break;
      if (was == id[i]) {
        twice = 1;
        break;
      }
    }
  }
  // also: the range is written
  if (W == 1) {
    twice = __any_sync(0xffffffffu, twice);
    __syncwarp();
  } else {
    twice = __syncthreads_or(twice);
  }
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int k = tid + i * G;
    if (id[i] < 0) continue;
    float all = p[i];
    if (twice) {
      bool first = true;
      for (int o = 0; o < k && first; ++o) first = ids[o] != id[i];
      if (!first) continue;
      for (int o = k + 1; o < t.K; ++o)
        if (ids[o] == id[i]) all += sp[o];
    }
    d[id[i]] = from_f<T>(coef * (q(to_f(x[id[i]])) - all));
  }
}

Teacher make_teacher(const at::Tensor& logits, const at::Tensor& ids, const at::Tensor& x, int64_t n, const char* what) {
  LRB_CHECK(logits.is_cuda() && ids.is_cuda() && logits.device() == x.device() && ids.device() == x.device(), what,
            ": student, teacher logits and ids must be on one CUDA device");
  LRB_CHECK(logits.dim() == 2 && ids.sizes() == logits.sizes() && logits.size(0) == n && logits.is_contiguous() &&
                ids.is_contiguous(),
            what, ": teacher logits and ids must be contiguous (N, K)");
  LRB_CHECK(logits.size(1) >= 1 && logits.size(1) <= kMaxK, what, ": 1 to ", kMaxK, " teacher entries a row");
  const auto lt = logits.scalar_type();
  LRB_CHECK(lt == at::kFloat || lt == at::kBFloat16 || lt == at::kHalf, what, ": teacher logits must be bf16, fp16 or fp32");
  LRB_CHECK(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt, what, ": teacher ids must be int64 or int32");
  return Teacher{logits.data_ptr(), ids.data_ptr(), lt == at::kFloat ? 0 : lt == at::kBFloat16 ? 1 : 2,
                 ids.scalar_type() == at::kLong ? 1 : 0, (int)logits.size(1)};
}

Rows make_rows(const at::Tensor& x, const char* what) {
  LRB_CHECK(x.is_cuda() && x.dim() == 3 && (x.stride(2) == 1 || x.size(2) == 1), what,
            ": logits (outer, inner, V) with unit stride along the vocabulary");
  LRB_CHECK(x.size(2) >= 1 && x.size(2) < (1LL << 31) - 64 && x.size(0) * x.size(1) < (1LL << 27), what,
            ": logits too large or without a vocabulary");
  return Rows{std::max<int64_t>(x.size(1), 1), x.stride(0), x.stride(1)};
}

// Blocks a row: one where the rows fill the GPU twice, else up to 8 (a portable
// cluster) of at least 4096 logits.
int row_split(int64_t n, int64_t V) {
  int s = 1;
  while (s < 8 && n * s < 2 * (int64_t)num_sms() && V / (2 * s) >= 4096) s *= 2;
  return s;
}

// A warp a row: enough rows for 12 warps an SM, lists that a warp holds, and rows short
// enough that what a block spends on a row besides reading it (barriers, joins) shows.
// 16384 fp16 rows: 8 KB each forward 32 us (103 us with a block a row), backward 42 us
// (92 us); 32 KB 100 us (138 us) and 175 us (166 us); 64 KB 199 us (201 us) and 394 us
// (320 us).
bool warp_a_row(int64_t n, int64_t row_bytes, int K, int64_t most) {
  return n >= 12 * (int64_t)num_sms() && K <= kWarpK && row_bytes <= most;
}

}  // namespace

// logits (outer, inner, V); teacher (outer * inner, K).  Returns (row losses, row
// statistics (N, 4) and the teacher's probabilities (N, K) for the backward -- the
// latter left empty without `keep` --, the loss and each counted row's factor in it (of
// a sum or a mean, reduction 1 and 2; not filled for 0)).  The loss is a tensor of its
// own: a caller may change it in place.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor> distill_fwd(
    const at::Tensor& logits, const at::Tensor& t_logits, const at::Tensor& t_ids, double temperature,
    int64_t reduction, bool keep) {
  const Rows rows = make_rows(logits, "topk_distillation");
  const int64_t n = logits.size(0) * logits.size(1), V = logits.size(2);
  const Teacher t = make_teacher(t_logits, t_ids, logits, n, "topk_distillation");
  LRB_CHECK(temperature >= 1e-18 && temperature <= 1e18,  // T, T^2 and log2(e) / T are normal fp32 numbers
            "topk_distillation: temperature must be between 1e-18 and 1e18");
  c10::cuda::CUDAGuard g(logits.device());
  bind_device(logits.get_device());
  auto f32 = logits.options().dtype(at::kFloat);
  auto loss = at::empty({n}, f32), rest = at::empty({5 * n + 1}, f32), out = at::empty({}, f32);
  auto stats = rest.narrow(0, 0, 4 * n), factor = rest.narrow(0, 5 * n, 1);
  float* counted = rest.data_ptr<float>() + 4 * n;
  auto probs = at::empty({keep ? n : 0, t.K}, f32);
  if (n > 0) {
    LRB_DISPATCH_FLOAT(logits.scalar_type(), T, [&] {
      const bool warps = warp_a_row(n, V * sizeof(T), t.K, 32768);
      const int split = warps ? 1 : row_split(n, V);
      cudaLaunchConfig_t cfg = {};
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = (unsigned)split;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.gridDim = dim3((unsigned)(warps ? (n + kWarps - 1) / kWarps : n * split), 1, 1);
      cfg.blockDim = dim3(kThreads, 1, 1);
      cfg.stream = stream();
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      LRB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, warps ? distill_fwd_kernel<T, 1> : distill_fwd_kernel<T, kWarps>,
                                        reinterpret_cast<const T*>(logits.data_ptr()), rows, n, (int)V, t,
                                        (float)temperature, loss.data_ptr<float>(), counted,
                                        reinterpret_cast<RowStats*>(stats.data_ptr<float>()),
                                        keep ? probs.data_ptr<float>() : (float*)nullptr));
    });
  }
  if (reduction != 0) {
    reduce_rows_kernel<<<1, 1024, 0, stream()>>>(loss.data_ptr<float>(), counted, n, reduction == 2 ? 1 : 0,
                                                 out.data_ptr<float>(), factor.data_ptr<float>());
    LRB_LAUNCH_CHECK();
  }
  return {loss, stats, probs, out, factor};
}

namespace {
// The gradient's tensor: laid out like the logits where these are a view with gaps
// (logits[:, :-1]) of little waste, and at the same offset from a 16-byte boundary, so
// that a row's vectors are aligned on both sides (4096 x 32001 bf16: 150 us both ways, 443 us when
// they are not).  Contiguous otherwise.
at::Tensor gradient_like(const at::Tensor& x) {
  const int64_t esz = x.element_size(), B = x.size(0), S = x.size(1), V = x.size(2), sb = x.stride(0), ss = x.stride(1);
  const int64_t off = (int64_t)(reinterpret_cast<uintptr_t>(x.data_ptr()) & 15) / esz;
  if (x.is_contiguous() && off == 0) return at::empty(x.sizes(), x.options());
  const bool apart = (ss >= V && sb >= S * ss) || (sb >= V && ss >= B * sb);
  const int64_t span = (B - 1) * sb + (S - 1) * ss + V;
  if (!apart || span > B * S * V / 4 * 5 + 64) return at::empty(x.sizes(), x.options());
  return at::empty({span + off}, x.options()).as_strided(x.sizes(), {sb, ss, 1}, off);
}
}  // namespace

// Gradient of the logits (their shape): `g` fp32, one value for each row (g_per_row) or
// a single one that is multiplied by `factor`.
at::Tensor distill_bwd(const at::Tensor& logits, const at::Tensor& t_ids, double temperature, const at::Tensor& stats,
                       const at::Tensor& probs, const at::Tensor& g, bool g_per_row, const at::Tensor& factor) {
  const Rows rows = make_rows(logits, "topk_distillation backward");
  const int64_t n = logits.size(0) * logits.size(1), V = logits.size(2);
  const Teacher t = make_teacher(probs, t_ids, logits, n, "topk_distillation backward");
  LRB_CHECK(g.is_cuda() && g.scalar_type() == at::kFloat && g.is_contiguous() && g.numel() == (g_per_row ? n : 1) &&
                stats.scalar_type() == at::kFloat && stats.is_contiguous() && stats.numel() == 4 * n &&
                probs.scalar_type() == at::kFloat &&
                (g_per_row || (factor.is_cuda() && factor.scalar_type() == at::kFloat && factor.numel() >= 1)),
            "topk_distillation backward: bad gradient or statistics");
  c10::cuda::CUDAGuard guard(logits.device());
  bind_device(logits.get_device());
  if (n == 0) return at::empty(logits.sizes(), logits.options());
  auto dx = gradient_like(logits);
  const Rows dx_rows = make_rows(dx, "topk_distillation backward");
  LRB_DISPATCH_FLOAT(logits.scalar_type(), T, [&] {
    const bool warps = warp_a_row(n, V * sizeof(T), t.K, 16384);
    const int split = warps ? 1 : row_split(n, V);
    const auto k = warps ? distill_bwd_kernel<T, 1> : distill_bwd_kernel<T, kWarps>;
    k<<<(unsigned)(warps ? (n + kWarps - 1) / kWarps : n * split), kThreads, 0, stream()>>>(
        reinterpret_cast<const T*>(logits.data_ptr()), rows, n, (int)V, t, (float)temperature, probs.data_ptr<float>(),
        reinterpret_cast<const RowStats*>(stats.data_ptr<float>()), g.data_ptr<float>(), g_per_row ? 1 : 0,
        g_per_row ? nullptr : factor.data_ptr<float>(), reinterpret_cast<T*>(dx.data_ptr()), dx_rows, split);
  });
  LRB_LAUNCH_CHECK();
  return dx;
}

// The same reduction for other per-row losses (reduction 1: sum, 2: mean over the counted rows).
void reduce_rows(const float* loss, const float* counted, int64_t n, bool mean, float* out, float* factor,
                 cudaStream_t s) {
  reduce_rows_kernel<<<1, 1024, 0, s>>>(loss, counted, n, mean ? 1 : 0, out, factor);
  LRB_LAUNCH_CHECK();
}

}  // namespace lrb

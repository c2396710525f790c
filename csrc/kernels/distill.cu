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
// The vocabulary is read once per direction: the forward keeps a running maximum
// m and a running sum s of exp((x - m) / T) per thread and joins them; (m, log2 s)
// of each row is all that the backward needs.  All of it is fp32.  Differences
// x - m are formed before the scaling by log2(e) / T, so that a row of the type's
// lowest values does not overflow.
//
// Bounded by the bytes of the logits.
#include "../common.cuh"

#include <cmath>

namespace lrb {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxK = 1024;                    // teacher entries of a row
constexpr int kPerThread = kMaxK / kThreads;   // held in registers
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

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

// This thread's entries k = threadIdx.x + i * kThreads: token (-1: none) and
// probability; returns whether the row has any.  ln p_k = y_k / T - ln(sum), left in `lp`.
__device__ __forceinline__ bool teacher_probs(const Teacher& t, int64_t row, int V, float inv_t, float* red,
                                              int (&id)[kPerThread], float (&p)[kPerThread], float (&lp)[kPerThread]) {
  float mx = -INFINITY;
  int any = 0;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int k = threadIdx.x + i * kThreads;
    id[i] = -1;
    lp[i] = -INFINITY;
    if (k < t.K) {
      const int v = teacher_id(t, row * t.K + k, V);
      if (v >= 0) {
        const float y = teacher_logit(t, row * t.K + k);
        if (y != -INFINITY) {
          id[i] = v;
          lp[i] = y;
          mx = fmaxf(mx, y);
          any = 1;
        }
      }
    }
  }
  if (!__syncthreads_or(any)) return false;
  mx = block_max(mx, red);
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    lp[i] = (lp[i] - mx) * inv_t;
    p[i] = id[i] >= 0 ? expf(lp[i]) : 0.f;
    sum += p[i];
  }
  sum = block_sum(sum, red);
  const float inv = 1.f / sum, ls = logf(sum);
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    p[i] *= inv;
    lp[i] -= ls;
  }
  return true;
}

// Running (max, sum of 2^((x - max) k2)).  A maximum of -inf (nothing but -inf so
// far) uses 0 as its reference: 2^-inf = 0, and a NaN still reaches the sum.
struct Online {
  float m = -INFINITY, s = 0.f;
  __device__ __forceinline__ void raise(float mx, float k2) {
    if (mx > m) {
      s *= fast_exp2((m - mx) * k2);
      m = mx;
    }
  }
  __device__ __forceinline__ float ref() const { return m == -INFINITY ? 0.f : m; }
  __device__ __forceinline__ void add(float x, float k2) {
    raise(x, k2);
    s += fast_exp2((x - ref()) * k2);
  }
  __device__ __forceinline__ void merge(float m2, float s2, float k2) {
    raise(m2, k2);
    s += s2 * fast_exp2((m2 - ref()) * k2);  // m2 = -inf: s2 is 0 or NaN, times 0
  }
};

__device__ __forceinline__ unsigned cluster_rank() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ unsigned cluster_size() {
  unsigned r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  __syncthreads();  // the aligned forms want converged warps
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float2 ld_peer(const float2* p, unsigned rank) {
  const uint32_t a = (uint32_t)__cvta_generic_to_shared(p);
  uint32_t q;
  float2 v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(q) : "r"(a), "r"(rank));
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(q) : "memory");
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

// One cluster per row; its blocks take equal ranges of the vocabulary (more than
// one block only where there are too few rows to fill the GPU).
template <typename T>
__global__ void __launch_bounds__(kThreads)
    distill_fwd_kernel(const T* __restrict__ logits, Rows rows, int V, Teacher t, float temp, float* __restrict__ loss,
                       float* __restrict__ counted, float2* __restrict__ stats) {
  __shared__ float red[32];
  __shared__ float2 part[kThreads / 32], mine;
  constexpr int VEC = 16 / sizeof(T), U = 4;
  const unsigned rank = cluster_rank(), split = cluster_size();
  const int64_t row = blockIdx.x / split;
  const T* x = row_ptr(logits, rows, row);
  const int c0 = (int)((int64_t)V * rank / split), c1 = (int)((int64_t)V * (rank + 1) / split);
  const float inv_t = 1.f / temp, k2 = kLog2e * inv_t;

  Online a;
  {
    const T* p = x + c0;
    const int len = c1 - c0;
    const int head = min(len, (int)(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T)));
    const int nvec = (len - head) / VEC, tail = len - head - nvec * VEC;
    if (threadIdx.x < head) a.add(to_f(p[threadIdx.x]), k2);
    if (threadIdx.x < tail) a.add(to_f(p[len - tail + threadIdx.x]), k2);
    const T* b = p + head;
    for (int i = threadIdx.x; i < nvec; i += U * kThreads) {
      Vec16<T> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + u * kThreads < nvec) v[u] = ld16(b + (int64_t)(i + u * kThreads) * VEC);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + u * kThreads >= nvec) break;
        float f[VEC], mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          f[j] = to_f(v[u].v[j]);
          mx = fmaxf(mx, f[j]);
        }
        a.raise(mx, k2);
        const float r = a.ref();
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < VEC; ++j) s += fast_exp2((f[j] - r) * k2);
        a.s += s;
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m2 = __shfl_xor_sync(0xffffffffu, a.m, o), s2 = __shfl_xor_sync(0xffffffffu, a.s, o);
    a.merge(m2, s2, k2);
  }
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = make_float2(a.m, a.s);
  __syncthreads();
  if (threadIdx.x == 0) {
    Online b;
    for (int w = 0; w < kThreads / 32; ++w) b.merge(part[w].x, part[w].y, k2);
    mine = make_float2(b.m, b.s);
  }
  if (split > 1) {
    cluster_barrier();
    if (rank == 0 && threadIdx.x == 0) {
      Online b;
      for (unsigned r = 0; r < split; ++r) {
        const float2 o = ld_peer(&mine, r);
        b.merge(o.x, o.y, k2);
      }
      part[0] = make_float2(b.m, b.s);
    }
    cluster_barrier();  // every block's `mine` has been read
    if (rank != 0) return;
  } else {
    __syncthreads();
    if (threadIdx.x == 0) part[0] = mine;
  }
  __syncthreads();
  const float m = part[0].x, s = part[0].y;
  const float log2_s = log2f(s);
  if (threadIdx.x == 0) stats[row] = make_float2(m, log2_s);

  int id[kPerThread];
  float p[kPerThread], lp[kPerThread];
  const bool some = teacher_probs(t, row, V, inv_t, red, id, p, lp);
  float acc = 0.f;
  if (some) {
    const float ls = log2_s * kLn2;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i)
      if (id[i] >= 0 && p[i] != 0.f) acc += p[i] * (lp[i] - ((to_f(x[id[i]]) - m) * inv_t - ls));
    acc = block_sum(acc, red);
  }
  if (threadIdx.x == 0) {
    loss[row] = some ? temp * temp * acc : 0.f;
    counted[row] = some ? 1.f : 0.f;
  }
}

// out[0] = the loss (sum of the rows, over the number of counted rows for a mean),
// out[1] = each counted row's factor in it.  One block, fixed order.
__global__ void __launch_bounds__(1024) reduce_rows_kernel(const float* __restrict__ loss,
                                                           const float* __restrict__ counted, int64_t n, int mean,
                                                           float* __restrict__ out) {
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
    out[0] = (float)(s * f);
    out[1] = (float)f;
  }
}

// gridDim.x = blocks per row * rows.  Each block writes its range of q scaled, then
// puts the entries that lie in the range right.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    distill_bwd_kernel(const T* __restrict__ logits, Rows rows, int V, Teacher t, float temp,
                       const float2* __restrict__ stats, const float* __restrict__ g, int g_per_row,
                       const float* __restrict__ factor, T* __restrict__ dx, int split) {
  __shared__ float red[32];
  __shared__ int ids[kMaxK], seen[2 * kMaxK];
  __shared__ float probs[kMaxK];
  constexpr int VEC = 16 / sizeof(T), U = 4;
  const int64_t row = blockIdx.x / split;
  const int part = (int)(blockIdx.x - row * split);
  const T* x = row_ptr(logits, rows, row);
  T* d = dx + row * V;
  const int c0 = (int)((int64_t)V * part / split), c1 = (int)((int64_t)V * (part + 1) / split);
  const int len = c1 - c0;
  const float inv_t = 1.f / temp, k2 = kLog2e * inv_t;

  int id[kPerThread];
  float p[kPerThread], lp[kPerThread];
  const bool some = teacher_probs(t, row, V, inv_t, red, id, p, lp);
  const T* xp = x + c0;
  T* dp = d + c0;
  if (!some) {
    const int head = min(len, (int)(((16 - (reinterpret_cast<uintptr_t>(dp) & 15)) & 15) / sizeof(T)));
    const int nvec = (len - head) / VEC, tail = len - head - nvec * VEC;
    if (threadIdx.x < head) dp[threadIdx.x] = from_f<T>(0.f);
    if (threadIdx.x < tail) dp[len - tail + threadIdx.x] = from_f<T>(0.f);
    for (int i = threadIdx.x; i < nvec; i += kThreads)
      *reinterpret_cast<uint4*>(dp + head + (int64_t)i * VEC) = make_uint4(0u, 0u, 0u, 0u);
    return;
  }
  const float coef = temp * (g_per_row ? g[row] : g[0] * factor[0]);
  const float m = stats[row].x, l2 = stats[row].y;
  const auto q = [&](float v) { return fast_exp2((v - m) * k2 - l2); };
  if ((reinterpret_cast<uintptr_t>(xp) & 15) == (reinterpret_cast<uintptr_t>(dp) & 15)) {
    const int head = min(len, (int)(((16 - (reinterpret_cast<uintptr_t>(dp) & 15)) & 15) / sizeof(T)));
    const int nvec = (len - head) / VEC, tail = len - head - nvec * VEC;
    if (threadIdx.x < head) dp[threadIdx.x] = from_f<T>(coef * q(to_f(xp[threadIdx.x])));
    if (threadIdx.x < tail) dp[len - tail + threadIdx.x] = from_f<T>(coef * q(to_f(xp[len - tail + threadIdx.x])));
    const T* b = xp + head;
    T* o = dp + head;
    for (int i = threadIdx.x; i < nvec; i += U * kThreads) {
      Vec16<T> v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + u * kThreads < nvec) v[u] = ld16(b + (int64_t)(i + u * kThreads) * VEC);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (i + u * kThreads >= nvec) break;
#pragma unroll
        for (int j = 0; j < VEC; ++j) v[u].v[j] = from_f<T>(coef * q(to_f(v[u].v[j])));
        st16(o + (int64_t)(i + u * kThreads) * VEC, v[u]);
      }
    }
  } else {
    for (int i = threadIdx.x; i < len; i += kThreads) dp[i] = from_f<T>(coef * q(to_f(xp[i])));
  }

  // The entries of this range: an open-addressing table of their tokens finds out
  // whether one is listed twice (its probabilities add up); without repetitions,
  // the usual case, each entry is put right by itself.
  int size = 64;
  while (size < 2 * t.K) size *= 2;
  for (int i = threadIdx.x; i < size; i += kThreads) seen[i] = -1;
  __syncthreads();
  int twice = 0;
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int k = threadIdx.x + i * kThreads;
    if (k >= t.K) continue;
    if (id[i] < c0 || id[i] >= c1) id[i] = -1;
    ids[k] = id[i];
    probs[k] = p[i];
    if (id[i] >= 0) {
      unsigned h = (unsigned)id[i] * 2654435761u;
      for (h ^= h >> 15;; ++h) {
        const int was = atomicCAS(&seen[h & (size - 1)], -1, id[i]);
        if (was == -1) break;
        if (was == id[i]) {
          twice = 1;
          break;
        }
      }
    }
  }
  twice = __syncthreads_or(twice);  // also: the range is written
#pragma unroll
  for (int i = 0; i < kPerThread; ++i) {
    const int k = threadIdx.x + i * kThreads;
    if (k >= t.K || id[i] < 0) continue;
    float all = p[i];
    if (twice) {
      bool first = true;
      for (int o = 0; o < k && first; ++o) first = ids[o] != id[i];
      if (!first) continue;
      for (int o = k + 1; o < t.K; ++o)
        if (ids[o] == id[i]) all += probs[o];
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

}  // namespace

// logits (outer, inner, V); teacher (outer * inner, K).  Returns (row losses, counted
// rows, row statistics, [loss, factor]); the last is filled for a sum or a mean
// (reduction 1, 2) and left empty for 0.
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> distill_fwd(const at::Tensor& logits,
                                                                       const at::Tensor& t_logits,
                                                                       const at::Tensor& t_ids, double temperature,
                                                                       int64_t reduction) {
  const Rows rows = make_rows(logits, "topk_distillation");
  const int64_t n = logits.size(0) * logits.size(1), V = logits.size(2);
  const Teacher t = make_teacher(t_logits, t_ids, logits, n, "topk_distillation");
  LRB_CHECK(temperature > 0.0 && std::isfinite(temperature), "topk_distillation: temperature must be positive");
  c10::cuda::CUDAGuard g(logits.device());
  bind_device(logits.get_device());
  auto f32 = logits.options().dtype(at::kFloat);
  auto loss = at::empty({n}, f32), counted = at::empty({n}, f32), stats = at::empty({n, 2}, f32);
  auto out = at::empty({reduction == 0 ? 0 : 2}, f32);
  if (n > 0) {
    const int split = row_split(n, V);
    LRB_DISPATCH_FLOAT(logits.scalar_type(), T, [&] {
      cudaLaunchConfig_t cfg = {};
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = (unsigned)split;
      attr[0].val.clusterDim.y = 1;
      attr[0].val.clusterDim.z = 1;
      cfg.gridDim = dim3((unsigned)(n * split), 1, 1);
      cfg.blockDim = dim3(kThreads, 1, 1);
      cfg.stream = stream();
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      LRB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, distill_fwd_kernel<T>, reinterpret_cast<const T*>(logits.data_ptr()), rows,
                                        (int)V, t, (float)temperature, loss.data_ptr<float>(), counted.data_ptr<float>(),
                                        reinterpret_cast<float2*>(stats.data_ptr<float>())));
    });
  }
  if (reduction != 0) {
    reduce_rows_kernel<<<1, 1024, 0, stream()>>>(loss.data_ptr<float>(), counted.data_ptr<float>(), n,
                                                 reduction == 2 ? 1 : 0, out.data_ptr<float>());
    LRB_LAUNCH_CHECK();
  }
  return {loss, counted, stats, out};
}

// Gradient of the logits (contiguous, their shape): `g` fp32, one value for each row
// (g_per_row) or a single one that is multiplied by `factor`.
at::Tensor distill_bwd(const at::Tensor& logits, const at::Tensor& t_logits, const at::Tensor& t_ids,
                       double temperature, const at::Tensor& stats, const at::Tensor& g, bool g_per_row,
                       const at::Tensor& factor) {
  const Rows rows = make_rows(logits, "topk_distillation backward");
  const int64_t n = logits.size(0) * logits.size(1), V = logits.size(2);
  const Teacher t = make_teacher(t_logits, t_ids, logits, n, "topk_distillation backward");
  LRB_CHECK(g.is_cuda() && g.scalar_type() == at::kFloat && g.is_contiguous() && g.numel() == (g_per_row ? n : 1) &&
                stats.scalar_type() == at::kFloat && stats.is_contiguous() && stats.numel() == 2 * n &&
                (g_per_row || (factor.is_cuda() && factor.scalar_type() == at::kFloat && factor.numel() >= 1)),
            "topk_distillation backward: bad gradient or statistics");
  c10::cuda::CUDAGuard guard(logits.device());
  bind_device(logits.get_device());
  auto dx = at::empty(logits.sizes(), logits.options());
  if (n == 0) return dx;
  const int split = row_split(n, V);
  LRB_DISPATCH_FLOAT(logits.scalar_type(), T, [&] {
    distill_bwd_kernel<T><<<(unsigned)(n * split), kThreads, 0, stream()>>>(
        reinterpret_cast<const T*>(logits.data_ptr()), rows, (int)V, t, (float)temperature,
        reinterpret_cast<const float2*>(stats.data_ptr<float>()), g.data_ptr<float>(), g_per_row ? 1 : 0,
        g_per_row ? nullptr : factor.data_ptr<float>(), reinterpret_cast<T*>(dx.data_ptr()), split);
  });
  LRB_LAUNCH_CHECK();
  return dx;
}

// The same reduction for other per-row losses (reduction 1: sum, 2: mean over the counted rows).
void reduce_rows(const float* loss, const float* counted, int64_t n, bool mean, float* out, cudaStream_t s) {
  reduce_rows_kernel<<<1, 1024, 0, s>>>(loss, counted, n, mean ? 1 : 0, out);
  LRB_LAUNCH_CHECK();
}

}  // namespace lrb

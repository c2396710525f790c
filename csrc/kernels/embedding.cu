// Token embedding: lookup with scaling, and the dense gradient of the table by
// sorted tokens.
//
//   out[n, :] = scale * W[ids[n], :]
//   dW[v, :]  = scale * sum over n with ids[n] = v of dout[n, :]
//
// both with the products and sums in fp32 and one rounding to the table's type.
// A row of dW adds its tokens in the order of their positions (or, for a token
// with more than kHeavy occurrences, in fixed pieces of that order), so the
// gradient does not depend on scheduling.
//
// Ids outside [0, V) give a row of NaN and no gradient; nothing is read for them.
#include "../common.cuh"

namespace lrb {
namespace {

// ------------------------------------------------------------------ lookup
// A copy: bounded by the bytes of the looked-up rows and the output.  `lanes`
// threads (a power of two up to 32) share one row, each moving four 16-byte
// vectors per step so that four loads are in flight; rows that are not 16-byte
// aligned (odd widths) move element by element, neighbouring lanes on
// neighbouring elements.
template <typename T, int VEC, typename IdT>
__global__ void __launch_bounds__(256) embedding_fwd_kernel(const IdT* __restrict__ ids, const T* __restrict__ w,
                                                            int64_t w_ld, T* __restrict__ out, int64_t n, int64_t V,
                                                            int d, int lanes, float scale) {
  struct alignas(VEC * sizeof(T)) Pack { T v[VEC]; };
  const int sub = threadIdx.x & (lanes - 1);
  const int per_block = blockDim.x / lanes;
  const int nvec = d / VEC;
  for (int64_t row = (int64_t)blockIdx.x * per_block + threadIdx.x / lanes; row < n;
       row += (int64_t)gridDim.x * per_block) {
    const int64_t id = (int64_t)ids[row];
    const bool known = id >= 0 && id < V;
    const Pack* src = reinterpret_cast<const Pack*>(w + (known ? id : 0) * w_ld);
    Pack* dst = reinterpret_cast<Pack*>(out + row * d);
    constexpr int U = 4;
    for (int c = sub; c < nvec; c += U * lanes) {
      Pack p[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c + u * lanes < nvec && known) p[u] = src[c + u * lanes];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (c + u * lanes >= nvec) continue;
#pragma unroll
        for (int j = 0; j < VEC; ++j) p[u].v[j] = from_f<T>(known ? to_f(p[u].v[j]) * scale : NAN);
        dst[c + u * lanes] = p[u];
      }
    }
  }
}

// ------------------------------------------------------------------ sorting the tokens
// Stable least-significant-digit radix sort of (id, position), 9 bits or fewer a
// pass, by ONE thread-block cluster: the passes are separated by cluster barriers
// instead of launches, and the digit totals of the blocks are exchanged through
// distributed shared memory.  Out-of-range ids and the padding id get the key V.
//
// Every block owns a contiguous range of the positions, every warp a contiguous
// part of that: pass 1 counts digits per warp, a scan over (digit, block, warp)
// gives each warp its first slot per digit, and pass 2 walks the part again in
// order, ranking equal digits inside 32 keys with __match_any_sync.
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kHeavy = 64;  // tokens that one warp sums by itself

struct Row {      // where a token's occurrences lie in the sorted order
  int start, end;
  int slot;       // first partial sum of a heavy row
  int piece;      // occurrences per partial sum (0: not heavy)
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
__device__ __forceinline__ int ld_peer(const int* p, unsigned rank) {
  const uint32_t a = (uint32_t)__cvta_generic_to_shared(p);
  uint32_t q;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(q) : "r"(a), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(q) : "memory");
  return v;
}

template <typename IdT>
__device__ __forceinline__ int token_key(const IdT* ids, int64_t i, int V, int64_t padding) {
  const int64_t id = (int64_t)ids[i];
  return (id < 0 || id >= V || id == padding) ? V : (int)id;
}

template <typename IdT>
__global__ void __launch_bounds__(kSortThreads, 1)
    sort_tokens_kernel(const IdT* __restrict__ ids, int n, int V, int64_t padding, int passes, int bits, int* key_a,
                       int* pos_a, int* key_b, int* pos_b, Row* rows, int2* pieces, int* num_pieces) {
  extern __shared__ int smem[];
  const int bins = 1 << bits;
  int* hist = smem;                       // [kSortWarps][bins]
  int* total = smem + kSortWarps * bins;  // this block's digit totals (read by the peers)
  int* base = total + bins;               // scan scratch
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_rank(), blocks = (int)cluster_size();
  const int64_t b0 = (int64_t)n * rank / blocks, b1 = (int64_t)n * (rank + 1) / blocks;
  const int w0 = (int)(b0 + (b1 - b0) * warp / kSortWarps), w1 = (int)(b0 + (b1 - b0) * (warp + 1) / kSortWarps);
  const unsigned below = (1u << lane) - 1u;

  for (int v = rank * kSortThreads + threadIdx.x; v < V; v += blocks * kSortThreads) rows[v] = Row{0, 0, 0, 0};
  if (rank == 0 && threadIdx.x == 0) *num_pieces = 0;

  int* ki = key_b;  // pass p writes (a), (b), (a), ...
  int* pi = pos_b;
  int* ko = key_a;
  int* po = pos_a;
  for (int p = 0; p < passes; ++p) {
    const int shift = p * bits;
    for (int i = threadIdx.x; i < kSortWarps * bins; i += kSortThreads) hist[i] = 0;
    __syncthreads();
    for (int i = w0 + lane; i < w1; i += 32) {
      const int k = p == 0 ? token_key(ids, i, V, padding) : __ldcg(ki + i);
      atomicAdd(&hist[warp * bins + ((k >> shift) & (bins - 1))], 1);
    }
    __syncthreads();
    int mine = 0;
    if (threadIdx.x < bins) {
      for (int w = 0; w < kSortWarps; ++w) {
        const int c = hist[w * bins + threadIdx.x];
        hist[w * bins + threadIdx.x] = mine;  // occurrences in the earlier warps of this block
        mine += c;
      }
      total[threadIdx.x] = mine;
    }
    cluster_barrier();
    int all = 0, before = 0;
    if (threadIdx.x < bins)
      for (int r = 0; r < blocks; ++r) {
        const int c = ld_peer(total + threadIdx.x, (unsigned)r);
        before += r < rank ? c : 0;
        all += c;
      }
    // exclusive scan of `all` over the digits
    int incl = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += t;
    }
    if (lane == 31) base[warp] = incl;
    __syncthreads();
    int carry = 0;
    for (int w = 0; w < warp; ++w) carry += base[w];
    if (threadIdx.x < bins) {
      const int first = carry + incl - all + before;
      for (int w = 0; w < kSortWarps; ++w) hist[w * bins + threadIdx.x] += first;
    }
    __syncthreads();
    for (int i0 = w0; i0 < w1; i0 += 32) {
      const int i = i0 + lane;
      const bool in = i < w1;
      const int k = !in ? -1 : p == 0 ? token_key(ids, i, V, padding) : __ldcg(ki + i);
      const int digit = in ? (k >> shift) & (bins - 1) : -1;
      const unsigned same = __match_any_sync(0xffffffffu, digit);
      if (in) {
        const int to = hist[warp * bins + digit] + __popc(same & below);
        __stcg(ko + to, k);
        __stcg(po + to, p == 0 ? i : __ldcg(pi + i));
      }
      __syncwarp();
      if (in && (same & below) == 0) hist[warp * bins + digit] += __popc(same);
      __syncwarp();
    }
    cluster_barrier();  // the sorted keys are visible, every peer has read this block's totals
    int* t = ki; ki = ko; ko = t;
    t = pi; pi = po; po = t;
  }

  // Segment borders in the sorted keys, then the pieces of the heavy rows.
  for (int i = w0 + lane; i < w1; i += 32) {
    const int k = __ldcg(ki + i);
    if (k == V) continue;
    if (i == 0 || __ldcg(ki + i - 1) != k) rows[k].start = i;
    if (i == n - 1 || __ldcg(ki + i + 1) != k) rows[k].end = i + 1;
  }
  cluster_barrier();
  for (int i = w0 + lane; i < w1; i += 32) {
    const int k = __ldcg(ki + i);
    if (k == V || !(i == 0 || __ldcg(ki + i - 1) != k)) continue;
    const int len = __ldcg(&rows[k].end) - i;
    if (len <= kHeavy) continue;
    // about sqrt(len) pieces of sqrt(len) occurrences: both levels stay short
    int piece = kHeavy;
    while ((int64_t)piece * piece < len) piece *= 2;
    const int count = (len + piece - 1) / piece;
    const int slot = atomicAdd(num_pieces, count);  // where the pieces lie does not change any sum
    rows[k].slot = slot;
    rows[k].piece = piece;
    for (int c = 0; c < count; ++c)
      pieces[slot + c] = make_int2(i + c * piece, min(i + (c + 1) * piece, i + len));
  }
}

// ------------------------------------------------------------------ sums
// One warp sums J vectors a lane (a slice of 32 * J * VEC columns) over the
// occurrences [i0, i1) of a token, in order, four of them in flight.
template <typename T, int VEC, int J>
__device__ __forceinline__ void sum_tokens(const T* __restrict__ dy, int64_t ld, const int* __restrict__ pos, int i0,
                                           int i1, int col0, int d, int lane, float (&acc)[J][VEC]) {
  struct alignas(VEC * sizeof(T)) Pack { T v[VEC]; };
  for (int b = i0; b < i1; b += 32) {
    const int m = min(32, i1 - b);
    const int mine = lane < m ? __ldg(pos + b + lane) : 0;
    int t = 0;
    for (; t + 4 <= m; t += 4) {
      Pack p[4][J];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const T* row = dy + (int64_t)__shfl_sync(0xffffffffu, mine, t + u) * ld;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int c = col0 + (j * 32 + lane) * VEC;
          if (c < d) p[u][j] = *reinterpret_cast<const Pack*>(row + c);
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int j = 0; j < J; ++j)
          if (col0 + (j * 32 + lane) * VEC < d)
#pragma unroll
            for (int x = 0; x < VEC; ++x) acc[j][x] += to_f(p[u][j].v[x]);
    }
    for (; t < m; ++t) {
      const T* row = dy + (int64_t)__shfl_sync(0xffffffffu, mine, t) * ld;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int c = col0 + (j * 32 + lane) * VEC;
        if (c < d) {
          const Pack p = *reinterpret_cast<const Pack*>(row + c);
#pragma unroll
          for (int x = 0; x < VEC; ++x) acc[j][x] += to_f(p.v[x]);
        }
      }
    }
  }
}

template <typename T, int VEC, int J>
__global__ void __launch_bounds__(256) embedding_pieces_kernel(const T* __restrict__ dy, int64_t ld,
                                                               const int* __restrict__ pos,
                                                               const int2* __restrict__ pieces,
                                                               const int* __restrict__ num_pieces,
                                                               float* __restrict__ partial, int d, int slices) {
  const int lane = threadIdx.x & 31;
  const int64_t items = (int64_t)*num_pieces * slices;
  for (int64_t it = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); it < items; it += (int64_t)gridDim.x * 8) {
    const int64_t piece = it / slices;
    const int col0 = (int)(it - piece * slices) * 32 * J * VEC;
    const int2 r = pieces[piece];
    float acc[J][VEC] = {};
    sum_tokens<T, VEC, J>(dy, ld, pos, r.x, r.y, col0, d, lane, acc);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int c = col0 + (j * 32 + lane) * VEC;
      if (c < d)
#pragma unroll
        for (int x = 0; x < VEC; ++x) partial[piece * d + c + x] = acc[j][x];
    }
  }
}

// Every row of dW is written once: zero without tokens, the sum of its tokens,
// or the sum of its pieces.  Bounded by reading dout and writing dW.
template <typename T, int VEC, int J>
__global__ void __launch_bounds__(256) embedding_grad_kernel(const T* __restrict__ dy, int64_t ld,
                                                             const int* __restrict__ pos, const Row* __restrict__ rows,
                                                             const float* __restrict__ partial, T* __restrict__ dw,
                                                             int64_t V, int d, int slices, float scale) {
  struct alignas(VEC * sizeof(T)) Pack { T v[VEC]; };
  const int lane = threadIdx.x & 31;
  const int64_t items = V * slices;
  for (int64_t it = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); it < items; it += (int64_t)gridDim.x * 8) {
    const int64_t v = it / slices;
    const int col0 = (int)(it - v * slices) * 32 * J * VEC;
    const int4 r4 = __ldg(reinterpret_cast<const int4*>(rows + v));
    const Row r{r4.x, r4.y, r4.z, r4.w};
    float acc[J][VEC] = {};
    if (r.piece == 0) {
      sum_tokens<T, VEC, J>(dy, ld, pos, r.start, r.end, col0, d, lane, acc);
    } else {
      const int count = (r.end - r.start + r.piece - 1) / r.piece;
#pragma unroll 4
      for (int c = 0; c < count; ++c) {
        const float* p = partial + (int64_t)(r.slot + c) * d;
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const int col = col0 + (j * 32 + lane) * VEC;
          if (col < d)
#pragma unroll
            for (int x = 0; x < VEC; ++x) acc[j][x] += p[col + x];
        }
      }
    }
    T* out = dw + v * d;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int c = col0 + (j * 32 + lane) * VEC;
      if (c < d) {
        Pack p;
#pragma unroll
        for (int x = 0; x < VEC; ++x) p.v[x] = from_f<T>(acc[j][x] * scale);
        *reinterpret_cast<Pack*>(out + c) = p;
      }
    }
  }
}

bool aligned16(const void* p, int64_t pitch_bytes) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && pitch_bytes % 16 == 0;
}

template <typename IdT>
void launch_sort(const at::Tensor& ids, int n, int V, int64_t padding, int* key_a, int* pos_a, int* key_b, int* pos_b,
                 int passes, int bits, Row* rows, int2* pieces, int* num_pieces) {
  auto k = sort_tokens_kernel<IdT>;
  const int smem = ((kSortWarps + 2) << bits) * (int)sizeof(int);
  LRB_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  // one block up to 4096 tokens, then one for each 4096 up to the portable 8
  const int blocks = n <= 4096 ? 1 : n <= 8192 ? 2 : n <= 16384 ? 4 : 8;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)blocks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.gridDim = dim3((unsigned)blocks, 1, 1);
  cfg.blockDim = dim3(kSortThreads, 1, 1);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = stream();
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  LRB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, k, (const IdT*)ids.data_ptr<IdT>(), n, V, padding, passes, bits, key_a, pos_a,
                                    key_b, pos_b, rows, pieces, num_pieces));
}

template <typename T, int VEC>
void launch_grad(const at::Tensor& dy, const int* pos, const Row* rows, const int2* pieces, const int* num_pieces,
                 float* partial, at::Tensor& dw, int64_t V, int d, double scale, bool heavy) {
  constexpr int J = VEC == 1 ? 8 : 2;
  const int slices = (d + 32 * J * VEC - 1) / (32 * J * VEC);
  const T* g = reinterpret_cast<const T*>(dy.data_ptr());
  if (heavy) {
    embedding_pieces_kernel<T, VEC, J><<<num_sms() * 4, 256, 0, stream()>>>(g, dy.stride(0), pos, pieces, num_pieces,
                                                                           partial, d, slices);
    LRB_LAUNCH_CHECK();
  }
  const int64_t blocks = std::min<int64_t>((V * slices + 7) / 8, (int64_t)num_sms() * 8);
  embedding_grad_kernel<T, VEC, J><<<(unsigned)blocks, 256, 0, stream()>>>(
      g, dy.stride(0), pos, rows, partial, reinterpret_cast<T*>(dw.data_ptr()), V, d, slices, (float)scale);
  LRB_LAUNCH_CHECK();
}

void check_ids(const at::Tensor& ids, const at::Tensor& other, const char* what) {
  LRB_CHECK(ids.is_cuda() && other.is_cuda() && ids.device() == other.device(), what,
            ": ids and the table must be on one CUDA device");
  LRB_CHECK(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt, what, ": ids must be int64 or int32");
  LRB_CHECK(ids.dim() == 1 && ids.is_contiguous(), what, ": ids must be contiguous and 1-D");
}

}  // namespace

// out (n, d) = scale * w[ids]; w (V, d) with unit column stride, ids (n) int64 / int32.
at::Tensor embedding_fwd(const at::Tensor& ids, const at::Tensor& w, double scale) {
  check_ids(ids, w, "embedding");
  LRB_CHECK(w.dim() == 2 && (w.stride(1) == 1 || w.size(1) <= 1), "embedding: weight (V, d) with unit column stride");
  const int64_t n = ids.numel(), V = w.size(0), d = w.size(1);
  LRB_CHECK(d < (1LL << 30) && V < (1LL << 31) - 1, "embedding: table too large");
  c10::cuda::CUDAGuard g(w.device());
  bind_device(w.get_device());
  auto out = at::empty({n, d}, w.options().layout(at::kStrided));
  if (n == 0 || d == 0) return out;
  LRB_DISPATCH_FLOAT(w.scalar_type(), T, [&] {
    constexpr int VEC = 16 / sizeof(T);
    const int64_t ld = w.stride(0);
    const bool vec = d % VEC == 0 && aligned16(w.data_ptr(), ld * (int64_t)sizeof(T)) && aligned16(out.data_ptr(), 0);
    const int nvec = (int)(vec ? d / VEC : d);
    int lanes = 1;
    while (lanes < 32 && lanes * 4 < nvec) lanes *= 2;
    // few rows: more, smaller blocks
    const int threads = n * lanes >= (int64_t)num_sms() * 256 ? 256 : 64;
    const int per_block = threads / lanes;
    const unsigned blocks = (unsigned)std::min<int64_t>((n + per_block - 1) / per_block, (int64_t)num_sms() * 32);
    auto run = [&](auto* idp) {
      using IdT = std::remove_const_t<std::remove_pointer_t<decltype(idp)>>;
      const T* wp = reinterpret_cast<const T*>(w.data_ptr());
      T* op = reinterpret_cast<T*>(out.data_ptr());
      if (vec) embedding_fwd_kernel<T, VEC, IdT><<<blocks, threads, 0, stream()>>>(idp, wp, ld, op, n, V, (int)d, lanes, (float)scale);
      else embedding_fwd_kernel<T, 1, IdT><<<blocks, threads, 0, stream()>>>(idp, wp, ld, op, n, V, (int)d, lanes, (float)scale);
    };
    if (ids.scalar_type() == at::kLong) run(ids.data_ptr<int64_t>());
    else run(ids.data_ptr<int>());
  });
  LRB_LAUNCH_CHECK();
  return out;
}

// dW (V, d) of embedding_fwd for the output gradient dy (n, d) (unit column
// stride); the row `padding` gets no gradient (negative: none is left out).
at::Tensor embedding_bwd(const at::Tensor& dy, const at::Tensor& ids, int64_t V, int64_t padding, double scale) {
  check_ids(ids, dy, "embedding backward");
  LRB_CHECK(dy.dim() == 2 && dy.size(0) == ids.numel() && (dy.stride(1) == 1 || dy.size(1) <= 1),
            "embedding backward: dy (n, d) with unit column stride");
  const int64_t n = ids.numel(), d = dy.size(1);
  LRB_CHECK(n < (1LL << 30) && d < (1LL << 30) && V >= 0 && V < (1LL << 31) - 1, "embedding backward: too large");
  c10::cuda::CUDAGuard g(dy.device());
  bind_device(dy.get_device());
  if (n == 0 || V == 0 || d == 0) return at::zeros({V, d}, dy.options());
  auto dw = at::empty({V, d}, dy.options());
  auto i32 = ids.options().dtype(at::kInt);
  int bits_all = 1;
  while ((V >> bits_all) != 0) ++bits_all;  // the keys are 0 .. V
  const int passes = (bits_all + 8) / 9, bits = std::max(5, (bits_all + passes - 1) / passes);
  // at most n / 64 + (rows with over 64 occurrences) pieces
  const int64_t cap = n / 32 + 2;
  auto buf = at::empty({4 * n + 4 * V + 2 * cap + 4}, i32);
  int* p = buf.data_ptr<int>();
  Row* rows = reinterpret_cast<Row*>(p);
  int2* pieces = reinterpret_cast<int2*>(p + 4 * V);
  int* num_pieces = p + 4 * V + 2 * cap;
  int* sorted = num_pieces + 4;  // key_a, key_b, pos_a, pos_b
  const bool heavy = n > kHeavy;
  auto partial = heavy ? at::empty({cap, d}, dy.options().dtype(at::kFloat)) : at::empty({0}, dy.options().dtype(at::kFloat));
  if (ids.scalar_type() == at::kLong)
    launch_sort<int64_t>(ids, (int)n, (int)V, padding, sorted, sorted + 2 * n, sorted + n, sorted + 3 * n, passes, bits,
                         rows, pieces, num_pieces);
  else
    launch_sort<int>(ids, (int)n, (int)V, padding, sorted, sorted + 2 * n, sorted + n, sorted + 3 * n, passes, bits, rows,
                     pieces, num_pieces);
  const int* pos = sorted + ((passes & 1) ? 2 * n : 3 * n);
  LRB_DISPATCH_FLOAT(dy.scalar_type(), T, [&] {
    constexpr int VEC = 16 / sizeof(T);
    const bool vec = d % VEC == 0 && aligned16(dy.data_ptr(), dy.stride(0) * (int64_t)sizeof(T));
    if (vec) launch_grad<T, VEC>(dy, pos, rows, pieces, num_pieces, partial.data_ptr<float>(), dw, V, (int)d, scale, heavy);
    else launch_grad<T, 1>(dy, pos, rows, pieces, num_pieces, partial.data_ptr<float>(), dw, V, (int)d, scale, heavy);
  });
  return dw;
}

}  // namespace lrb

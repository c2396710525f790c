// Token embedding: lookup with scaling, and the dense gradient of the table by
// sorted tokens.
//
//   out[n, :] = scale * W[ids[n], :]
//   dW[v, :]  = scale * sum over n with ids[n] = v of dout[n, :]
//
// both with the products and sums in fp32 and one rounding to the table's type.
// A row of dW adds its tokens in the order of their positions, in pieces that depend
// on the ids alone, so the gradient does not depend on scheduling.
//
// Ids outside [0, V) give a row of NaN and no gradient; nothing is read for them.
#include "../common.cuh"
#include "sm100.cuh"

namespace lrb {
namespace {

using namespace sm100;

// ------------------------------------------------------------------ lookup
// A copy: bounded by the bytes of the looked-up rows and the output (65520 x 4096 bf16
// in 125 us, 6.4 TB/s).  `lanes`
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
    Pack* dst = reinterpret_cast<Pack*>(out + row * d);
    if (!known) {
      Pack p;
#pragma unroll
      for (int j = 0; j < VEC; ++j) p.v[j] = from_f<T>(NAN);
      for (int c = sub; c < nvec; c += lanes) dst[c] = p;
      continue;
    }
    const Pack* src = reinterpret_cast<const Pack*>(w + id * w_ld);
    constexpr int U = 4;
    for (int c = sub; c < nvec; c += U * lanes) {
      Pack p[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c + u * lanes < nvec) p[u] = src[c + u * lanes];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (c + u * lanes >= nvec) continue;
#pragma unroll
        for (int j = 0; j < VEC; ++j) p[u].v[j] = from_f<T>(to_f(p[u].v[j]) * scale);
        dst[c + u * lanes] = p[u];
      }
    }
  }
}

// ------------------------------------------------------------------ sorting the tokens
// Stable least-significant-digit radix sort of (token, position), 9 bits or fewer a
// pass, by ONE thread-block cluster: the passes are separated by cluster barriers
// instead of launches, and the digit totals of the blocks are exchanged through
// distributed shared memory.  Ids outside the table and the padding id get the key V.
//
// Every block owns a contiguous range of the positions, every warp a contiguous
// part of that: a pass counts digits per warp, a scan over (digit, block, warp)
// gives each warp its first slot per digit, and the warp walks its part again in
// order, ranking equal digits inside 32 keys by one ballot a bit.  All of it is
// latency and issue slots, so a lane holds 8 keys, loaded before any is used and kept
// from the count to the ranking where a warp has no more.  65536 tokens of a
// vocabulary of 32000: 22 us in 16 blocks (37 us in 8), 1344 tokens in one: 12 us.
// Handing the pairs from pass to pass through distributed shared memory instead of L2
// measured the same.
//
// dW is filled with zeros beside it (rows without tokens are most of a large
// vocabulary; the rows with tokens are written over by the summing kernel): the
// fill is launched as a dependent of the sort that starts early and ends with it.
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kBatch = 8;  // keys a lane holds at a time

__device__ __forceinline__ void cluster_barrier() {
  __syncthreads();  // the aligned forms want converged warps
  cluster_sync();
}
__device__ __forceinline__ int ld_peer(const int* p, unsigned rank) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_addr(p), rank)) : "memory");
  return v;
}

template <typename IdT>
__device__ __forceinline__ int token_key(const IdT* ids, int64_t i, int V, int64_t padding) {
  const int64_t id = (int64_t)ids[i];
  return (id < 0 || id >= V || id == padding) ? V : (int)id;
}

struct SortArgs {
  int n, V, passes, bits, range;
  int64_t padding;
  int2 *pair_a, *pair_b;  // (token, position) between the passes
  int *key, *pos;     // the sorted tokens and their positions
  int* num_spans;     // two counters, set to 0 for the summing kernel
};

// 32 KB a block (many short blocks fill 401 MB in 57 us, one or two resident blocks an
// SM in 66 us).  Launched with programmatic stream serialisation behind the sort, so it
// runs beside it; its first block ends only when the sort has ended, so what follows
// this launch sees both.
__global__ void __launch_bounds__(512) fill_zeros_kernel(uint4* __restrict__ p, int64_t bytes) {
  const int64_t nv = bytes / 16;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t i = (int64_t)blockIdx.x * 2048 + u * 512 + threadIdx.x;
    if (i < nv) p[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  if (blockIdx.x != 0) return;
  if (threadIdx.x < bytes - nv * 16) reinterpret_cast<unsigned char*>(p + nv)[threadIdx.x] = 0;
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

template <typename IdT>
__global__ void __launch_bounds__(kSortThreads, 1) sort_tokens_kernel(const IdT* __restrict__ ids, SortArgs a) {
  extern __shared__ int smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)cluster_ctarank(), blocks = (int)cluster_nctarank();
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int n = a.n, V = a.V, bits = a.bits;
  const int bins = 1 << bits;
  int* hist = smem;                       // [kSortWarps][bins]
  int* total = smem + kSortWarps * bins;  // this block's digit totals (read by the peers)
  int* base = total + bins;               // scan scratch
  const int64_t b0 = (int64_t)n * rank / blocks, b1 = (int64_t)n * (rank + 1) / blocks;
  const int w0 = (int)(b0 + (b1 - b0) * warp / kSortWarps), w1 = (int)(b0 + (b1 - b0) * (warp + 1) / kSortWarps);
  const bool held = w1 - w0 <= 32 * kBatch;
  const unsigned below = (1u << lane) - 1u;
  if (rank == 0 && threadIdx.x < 2) a.num_spans[threadIdx.x] = 0;

  for (int p = 0; p < a.passes; ++p) {  // the passes write a, b, a, ..., the last one key and pos
    const int shift = p * bits;
    const int2* from = (p & 1) ? a.pair_a : a.pair_b;
    const auto load = [&](int i) { return p == 0 ? make_int2(token_key(ids, i, V, a.padding), i) : __ldcg(from + i); };
    int2 k[kBatch];
    for (int i = threadIdx.x; i < kSortWarps * bins; i += kSortThreads) hist[i] = 0;
    __syncthreads();
    for (int i0 = w0; i0 < w1; i0 += 32 * kBatch) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (i0 + j * 32 + lane < w1) k[j] = load(i0 + j * 32 + lane);
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        if (i0 + j * 32 + lane < w1) atomicAdd(&hist[warp * bins + ((k[j].x >> shift) & (bins - 1))], 1);
    }
    __syncthreads();
    if (threadIdx.x < bins) {
      int mine = 0;
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) {
        const int c = hist[w * bins + threadIdx.x];
        hist[w * bins + threadIdx.x] = mine;  // occurrences in the earlier warps of this block
        mine += c;
      }
      total[threadIdx.x] = mine;
    }
    if (blocks > 1) cluster_barrier();
    int all = 0, before = 0;
    if (threadIdx.x < bins) {
      if (blocks == 1) {
        all = total[threadIdx.x];
      } else {
#pragma unroll 8
        for (int r = 0; r < blocks; ++r) {
          const int c = ld_peer(total + threadIdx.x, (unsigned)r);
          before += r < rank ? c : 0;
          all += c;
        }
      }
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
    if (threadIdx.x < bins) {
      int first = incl - all + before;
      for (int w = 0; w < warp; ++w) first += base[w];
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) hist[w * bins + threadIdx.x] += first;
    }
    __syncthreads();
    for (int i0 = w0; i0 < w1; i0 += 32 * kBatch) {
      if (!held) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
          if (i0 + j * 32 + lane < w1) k[j] = load(i0 + j * 32 + lane);
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        if (i0 + j * 32 >= w1) break;  // the same in every lane
        const bool in = i0 + j * 32 + lane < w1;
        const int digit = in ? (k[j].x >> shift) & (bins - 1) : 0;
        // the lanes with this digit
        unsigned same = __ballot_sync(0xffffffffu, in);
#pragma unroll
        for (int b = 0; b < 9; ++b) {
          if (b >= bits) break;
          const bool one = (digit >> b) & 1;
          const unsigned ones = __ballot_sync(0xffffffffu, one);
          same &= one ? ones : ~ones;
        }
        int* slot = &hist[warp * bins + digit];
        if (in) {
          const int to = *slot + __popc(same & below);
          if (p == a.passes - 1) {
            a.key[to] = k[j].x;
            a.pos[to] = k[j].y;
          } else {
            __stcg(((p & 1) ? a.pair_b : a.pair_a) + to, k[j]);
          }
        }
        __syncwarp();
        if (in && (same & below) == 0) *slot += __popc(same);
        __syncwarp();
      }
    }
    cluster_barrier();  // the pairs are visible, every peer has read this block's totals
  }
}

// ------------------------------------------------------------------ sums
// One warp walks over `range` positions of the sorted order for a slice of
// 32 * J * VEC columns, so every warp has the same number of rows to read whatever
// the tokens are, and the loads (four rows at a time) do not depend on where one
// token ends.  A token that lies inside the range is written to dW at once; one that
// began before it or goes on behind it leaves a partial sum, its rows' order kept.
// Bounded by reading dout once (and writing the present rows of dW).  One vector a
// lane and four blocks an SM measured best: 65536 x 2048 bf16 in 66 us (5.2 TB/s); two
// vectors and two blocks 66 to 96 us by the tokens' order, eight rows in flight 73 us.
constexpr int kShort = 8;  // partial sums that one warp joins

template <typename T, int VEC, int J>
__global__ void __launch_bounds__(256, 4) embedding_sum_kernel(const T* __restrict__ dy, int64_t ld,
                                                            const int* __restrict__ key, const int* __restrict__ pos,
                                                            int n, int V, int range, float* __restrict__ partial,
                                                            int4* __restrict__ spans, int* __restrict__ num_spans,
                                                            int max_spans, T* __restrict__ dw, int d, int slices, float scale) {
  struct alignas(VEC * sizeof(T)) Pack { T v[VEC]; };
  const int lane = threadIdx.x & 31;
  const int64_t it = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int64_t r = it / slices;
  const int64_t p0 = r * range;
  if (p0 >= n) return;
  const int col0 = (int)(it - r * slices) * 32 * J * VEC;
  const int count = (int)min((int64_t)range, n - p0);
  key += p0;
  pos += p0;
  int k32 = lane < count ? __ldg(key + lane) : V;
  int q32 = lane < count ? __ldg(pos + lane) : 0;
  const int before = p0 > 0 ? __ldg(key - 1) : -1;
  const int behind = p0 + count < n ? __ldg(key + count) : -1;

  float acc[J][VEC] = {};
  int cur = __shfl_sync(0xffffffffu, k32, 0);
  bool open = cur == before;  // the token began before the range
  const auto flush = [&](bool last) {
    if (open || (last && cur == behind)) {
      float* p = partial + (r * 2 + (open ? 0 : 1)) * d;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int c = col0 + (j * 32 + lane) * VEC;
        if (c < d) {
#pragma unroll
          for (int x = 0; x < VEC; ++x) p[c + x] = acc[j][x];
        }
      }
    } else {
      T* out = dw + (int64_t)cur * d;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int c = col0 + (j * 32 + lane) * VEC;
        if (c < d) {
          Pack o;
#pragma unroll
          for (int x = 0; x < VEC; ++x) o.v[x] = from_f<T>(acc[j][x] * scale);
          *reinterpret_cast<Pack*>(out + c) = o;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int x = 0; x < VEC; ++x) acc[j][x] = 0.f;
  };
  const auto add = [&](const Pack (&p)[J], int k) {
    if (k != cur) {
      flush(false);
      cur = k;
      open = false;
    }
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int x = 0; x < VEC; ++x) acc[j][x] += to_f(p[j].v[x]);
  };
  const auto load = [&](Pack (&p)[J], int q) {
    const T* row = dy + (int64_t)q * ld;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int c = col0 + (j * 32 + lane) * VEC;
      if (c < d) p[j] = *reinterpret_cast<const Pack*>(row + c);
      else p[j] = Pack{};
    }
  };
  for (int b = 0; b < count && cur != V; b += 32) {
    const int m = __popc(__ballot_sync(0xffffffffu, k32 != V));  // tokens of this group (those of the key V come last)
    const int kc = k32, qc = q32;
    if (b + 32 < count) {
      const int i = b + 32 + lane;
      k32 = i < count ? __ldg(key + i) : V;
      q32 = i < count ? __ldg(pos + i) : 0;
    }
    int t = 0;
    for (; t + 4 <= m; t += 4) {
      Pack p[4][J];
#pragma unroll
      for (int u = 0; u < 4; ++u) load(p[u], __shfl_sync(0xffffffffu, qc, t + u));
#pragma unroll
      for (int u = 0; u < 4; ++u) add(p[u], __shfl_sync(0xffffffffu, kc, t + u));
    }
    for (; t < m; ++t) {
      Pack p[J];
      load(p, __shfl_sync(0xffffffffu, qc, t));
      add(p, __shfl_sync(0xffffffffu, kc, t));
    }
    if (m < 32) break;
  }
  if (cur == V) return;
  const bool begins = !open && cur == behind;  // the token crosses the border and began in this range
  flush(true);
  if (begins && col0 == 0) {
    // the ranges that it reaches into: those whose first position holds it
    int parts = 1;
    for (int64_t q = p0 + (int64_t)range;; q += 32 * (int64_t)range) {
      const int64_t i = q + (int64_t)lane * range;
      const unsigned not_it = __ballot_sync(0xffffffffu, i >= n || __ldg(key + (i - p0)) != cur);
      parts += not_it == 0 ? 32 : __ffs(not_it) - 1;
      if (not_it != 0) break;
    }
    // short ones from the front, long ones from the back; where an entry lies changes no sum
    if (lane == 0) {
      const int at = parts <= kShort ? atomicAdd(num_spans, 1) : max_spans - 1 - atomicAdd(num_spans + 1, 1);
      spans[at] = make_int4(cur, (int)r, parts, 0);
    }
  }
}

// The tokens that cross borders: their partial sums added in order.  128 columns at
// a time, by one warp for up to kShort parts, else by the eight warps of a block, each
// a consecutive share of the parts, joined in order.
template <typename T>
__global__ void __launch_bounds__(256) embedding_join_kernel(const int4* __restrict__ spans,
                                                             const int* __restrict__ num_spans,
                                                             int max_spans, const float* __restrict__ partial,
                                                             T* __restrict__ dw, int d, int slices, float scale) {
  __shared__ float sh[8][128];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t few = (int64_t)num_spans[0] * slices, many = (int64_t)num_spans[1] * slices;
  const auto sum = [&](const int4& sp, int col0, int q0, int q1, float (&acc)[4]) {
#pragma unroll 8
    for (int q = q0; q < q1; ++q) {
      // the open end of the first range, then the heads of the others
      const float* p = partial + (((int64_t)sp.y + q) * 2 + (q == 0 ? 1 : 0)) * d;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (col0 + j * 32 < d) acc[j] += p[col0 + j * 32];
    }
  };
  for (int64_t it = (int64_t)blockIdx.x * 8 + warp; it < few; it += (int64_t)gridDim.x * 8) {
    const int64_t s = it / slices;
    const int4 sp = __ldg(spans + s);
    const int col0 = (int)(it - s * slices) * 128 + lane;
    float acc[4] = {};
    sum(sp, col0, 0, sp.z, acc);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col0 + j * 32 < d) dw[(int64_t)sp.x * d + col0 + j * 32] = from_f<T>(acc[j] * scale);
  }
  for (int64_t it = gridDim.x - 1 - blockIdx.x; it < many; it += gridDim.x) {
    const int64_t s = it / slices;
    const int4 sp = __ldg(spans + max_spans - 1 - s);
    const int col0 = (int)(it - s * slices) * 128 + lane;
    float acc[4] = {};
    sum(sp, col0, (int)((int64_t)sp.z * warp / 8), (int)((int64_t)sp.z * (warp + 1) / 8), acc);
#pragma unroll
    for (int j = 0; j < 4; ++j) sh[warp][j * 32 + lane] = acc[j];
    __syncthreads();
    const int c = col0 - lane + threadIdx.x;
    if (threadIdx.x < 128 && c < d) {
      float v = sh[0][threadIdx.x];
#pragma unroll
      for (int w = 1; w < 8; ++w) v += sh[w][threadIdx.x];
      dw[(int64_t)sp.x * d + c] = from_f<T>(v * scale);
    }
    __syncthreads();
  }
}

bool aligned16(const void* p, int64_t pitch_bytes) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && pitch_bytes % 16 == 0;
}

// A block for each 2048 tokens up to 8 of them, 16 (the largest cluster) from 32768.
int sort_blocks(int64_t n) { return n <= 2048 ? 1 : n <= 4096 ? 2 : n <= 8192 ? 4 : n <= 32768 ? 8 : 16; }

template <typename IdT>
void launch_sort(const at::Tensor& ids, const SortArgs& a, int blocks) {
  auto k = sort_tokens_kernel<IdT>;
  const int smem = ((kSortWarps + 2) << a.bits) * (int)sizeof(int);
  if (smem > 48 * 1024) LRB_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  if (blocks > 8) LRB_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
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
  LRB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, k, (const IdT*)ids.data_ptr<IdT>(), a));
}

void launch_fill(at::Tensor& dw) {
  const int64_t bytes = dw.numel() * (int64_t)dw.element_size();
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3((unsigned)((bytes + 32767) / 32768), 1, 1);
  cfg.blockDim = dim3(512, 1, 1);
  cfg.stream = stream();
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  LRB_CUDA_CHECK(cudaLaunchKernelEx(&cfg, fill_zeros_kernel, reinterpret_cast<uint4*>(dw.data_ptr()), bytes));
}

template <typename T, int VEC>
constexpr int slice_columns() { return VEC == 1 ? 128 : 32 * VEC; }

template <typename T, int VEC>
void launch_sum(const at::Tensor& dy, const SortArgs& a, float* partial, int4* spans, at::Tensor& dw, int d,
                double scale) {
  constexpr int J = slice_columns<T, VEC>() / (32 * VEC);
  const int slices = (d + slice_columns<T, VEC>() - 1) / slice_columns<T, VEC>();
  const int64_t items = (int64_t)((a.n + a.range - 1) / a.range) * slices;
  embedding_sum_kernel<T, VEC, J><<<(unsigned)((items + 7) / 8), 256, 0, stream()>>>(
      reinterpret_cast<const T*>(dy.data_ptr()), dy.stride(0), a.key, a.pos, a.n, a.V, a.range, partial, spans,
      a.num_spans, (a.n + a.range - 1) / a.range, reinterpret_cast<T*>(dw.data_ptr()), d, slices, (float)scale);
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
  int bits_all = 1;
  while ((V >> bits_all) != 0) ++bits_all;  // the keys are 0 .. V
  SortArgs a{};
  a.n = (int)n, a.V = (int)V, a.padding = padding;
  a.passes = (bits_all + 8) / 9;
  a.bits = std::max(5, (bits_all + a.passes - 1) / a.passes);
  const int blocks = sort_blocks(n);
  const bool vec = LRB_DISPATCH_FLOAT(dy.scalar_type(), T, [&] {
    constexpr int VEC = 16 / sizeof(T);
    const bool ok = d % VEC == 0 && aligned16(dy.data_ptr(), dy.stride(0) * (int64_t)sizeof(T));
    // 64 positions a warp, fewer where that leaves SMs without warps
    const int64_t cols = ok ? slice_columns<T, VEC>() : slice_columns<T, 1>();
    a.range = 64;
    while (a.range > 16 && n * ((d + cols - 1) / cols) < (int64_t)a.range * num_sms() * 16) a.range /= 2;
    return ok;
  });
  const int64_t ranges = (n + a.range - 1) / a.range;
  // at most one token crosses each border
  const bool join = ranges > 1;
  const int64_t ints = (4 * ranges + 4 + 6 * n + 3) / 4 * 4;
  auto buf = at::empty({ints + (join ? 2 * ranges * d : 0)}, ids.options().dtype(at::kInt));
  int* p = buf.data_ptr<int>();
  int4* spans = reinterpret_cast<int4*>(p);
  float* partial = reinterpret_cast<float*>(p + ints);
  a.num_spans = p + 4 * ranges;
  a.pair_a = reinterpret_cast<int2*>(a.num_spans + 4), a.pair_b = a.pair_a + n;
  a.key = a.num_spans + 4 + 4 * n, a.pos = a.key + n;
  if (ids.scalar_type() == at::kLong) launch_sort<int64_t>(ids, a, blocks);
  else launch_sort<int>(ids, a, blocks);
  launch_fill(dw);
  LRB_DISPATCH_FLOAT(dy.scalar_type(), T, [&] {
    if (vec) launch_sum<T, 16 / sizeof(T)>(dy, a, partial, spans, dw, (int)d, scale);
    else launch_sum<T, 1>(dy, a, partial, spans, dw, (int)d, scale);
    if (join) {
      const int slices = (int)((d + 127) / 128);
      embedding_join_kernel<T><<<(unsigned)std::min<int64_t>((ranges * slices + 7) / 8, (int64_t)num_sms() * 8), 256, 0,
                                 stream()>>>(spans, a.num_spans, (int)ranges, partial,
                                             reinterpret_cast<T*>(dw.data_ptr()), (int)d, slices, (float)scale);
      LRB_LAUNCH_CHECK();
    }
  });
  return dw;
}

}  // namespace lrb

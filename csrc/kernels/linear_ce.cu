// Softmax cross entropy of a linear head, z = h w^T (N, V), without keeping z:
//
//   lse_n = ln sum_v exp z_nv,   loss_n = lse_n - z[n, t_n]   (0 where t_n does not count)
//   dz_nv = r_n (exp(z_nv - lse_n) - [v = t_n]),   dh = dz w,   dw = dz^T h
//
// A target counts unless it is `ignore_index` or outside [0, V).  Forward: one
// CTA-pair product whose epilogue reduces each 256-column tile to (max, sum) pairs
// in fp32 straight from the accumulators; the kernel here joins a row's pairs.
// Backward, one piece of the vocabulary at a time: the product again, its epilogue
// turning the tile into dz in 16 bits, then dz w (added up over the pieces in fp32)
// and dz^T h (rows of dw, complete after one piece).  So 2NVd operations forward,
// 6NVd backward, bounded by the tensor cores; the only (N, piece) array is dz.
// N = 16384, V = 32000, d = 2048 bf16: forward 1.49 ms (1.44 PFLOP/s), the three
// products of the backward 1.60, 1.49 and 1.49 ms in 5 pieces, the step 6.8 to 6.9 ms under
// the power cap (1.26 PFLOP/s; cuBLAS products alone sustain 1.37).  The loss by chunks of
// rows, which keeps 16-bit logits and forms 6NVd, needs 6.3 ms there and 1.8 GB beside the
// results instead of 0.5.
//
// The logits are the tensor cores' fp32 accumulators, which cut off what does not fit:
// against 64 bits the row losses are off by 2-norm 4.6e-7 at d = 1024 and 1.8e-6 at
// d = 4096 (2.5e-7 and 5.7e-7 with fp32 multiply-adds).  Cutting off has one direction
// (logits of targets are large and come out too small), so the error of a mean is no
// smaller: +3e-7 of it at d = 1024, +6e-7 at 2048, +1.2e-6 at 4096.
//
// dz is the one value that is rounded to 16 bits on the way: it is an operand of
// the two gradient products, relative 2^-9 (bf16) or 2^-12 (fp16) an element.  With one
// weight for all rows the gradients' error is 1.1 (bf16) to 1.4 times (fp16) that of their
// own rounding.  For fp16, whose smallest normal number is 6e-5, dz is scaled so that the
// largest finite |r_n| is 2^13 and the products are scaled back; a probability times its
// row's weight below 2^-27 of that largest weight falls among the subnormals (an absolute
// error of 2^-38 of it).
#include "../common.cuh"

#include <climits>

namespace lrb {

// gemm_pair_sm100.cu
int64_t gemm_pair_lse_tiles(int64_t V);
void gemm_pair_lse(const at::Tensor&, const at::Tensor&, const at::Tensor&, at::Tensor&, at::Tensor&);
void gemm_pair_ce_grad(const at::Tensor&, const at::Tensor&, const at::Tensor&, int64_t, const at::Tensor&,
                       const at::Tensor&, at::Tensor&);
int gemm_pair_slices(int64_t, int64_t, int64_t, int);
int64_t gemm_pair_ce_piece(int64_t, int64_t, int64_t, int64_t, int);
void gemm_pair_sliced(const at::Tensor&, const at::Tensor&, bool, bool, at::Tensor&, int, bool, const float*);
// distill.cu
void reduce_rows(const float*, const float*, int64_t, bool, float*, float*, cudaStream_t);

namespace {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ bool counts(int64_t t, int64_t ignore, int64_t V) { return t != ignore && t >= 0 && t < V; }

__device__ __forceinline__ void merge(float& m, float& s, float m2, float s2) {
  if (m2 > m) {
    s *= fast_exp2((m - m2) * kLog2e);
    m = m2;
  }
  s += s2 * fast_exp2((m2 - (m == -INFINITY ? 0.f : m)) * kLog2e);
}

// 32 rows a block, 8 warps that share the tile columns of each row (a warp reads 32
// rows of one tile column: 256 consecutive bytes).
__global__ void __launch_bounds__(256) join_tiles_kernel(const float2* __restrict__ part,
                                                         const float* __restrict__ target_logit,
                                                         const int64_t* __restrict__ targets, int64_t n, int64_t V,
                                                         int tiles, int64_t ignore, float2* __restrict__ stats,
                                                         float* __restrict__ loss, float* __restrict__ counted) {
  __shared__ float2 sh[8][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = (int64_t)blockIdx.x * 32 + lane;
  float m = -INFINITY, s = 0.f;
  if (row < n) {
#pragma unroll 4
    for (int t = warp; t < tiles; t += 8) {
      const float2 p = part[(int64_t)t * n + row];
      merge(m, s, p.x, p.y);
    }
  }
  sh[warp][lane] = make_float2(m, s);
  __syncthreads();
  if (warp != 0 || row >= n) return;
  for (int w = 1; w < 8; ++w) merge(m, s, sh[w][lane].x, sh[w][lane].y);
  const float l2 = log2f(s);
  stats[row] = make_float2(m, l2);
  const int64_t t = targets[row];
  const bool c = counts(t, ignore, V);
  loss[row] = c ? (m - target_logit[row]) + l2 * kLn2 : 0.f;
  counted[row] = c ? 1.f : 0.f;
}

// The weight of each row inside dz, and alpha, which the outputs are multiplied by.  The
// largest weight (the only one of a sum or a mean) goes into alpha: dz = softmax - onehot
// then rounds an improbable target to exactly -1, where -1 times a weight that all rows
// share would round the same way in every row (2-norm error of the gradients of a
// 512 x 32000 bf16 mean 2.3e-3 instead of 1.9e-3).  A weight that is no number goes into
// dz: in alpha it would meet the zeros of the rows that do not count (0 * inf), and as
// the largest one it would leave the other rows without their scale.  f: the power of two
// of fp16.
__global__ void __launch_bounds__(1024) row_scale_kernel(const int64_t* __restrict__ targets, int64_t n, int64_t V,
                                                         int64_t ignore, const float* __restrict__ g, int g_per_row,
                                                         const float* __restrict__ factor, float f,
                                                         float* __restrict__ row_scale, float* __restrict__ alpha) {
  __shared__ float red[32];
  float most = g_per_row ? 0.f : g[0] * factor[0];
  float all = f;
  if (g_per_row) {  // every block finds it for itself
    for (int64_t i = threadIdx.x; i < n; i += 1024) {
      const float a = fabsf(g[i]);
      if (a < INFINITY && counts(targets[i], ignore, V)) most = fmaxf(most, a);
    }
    most = block_max(most, red);
    if (!(most > 1e-30f)) most = 1.f;  // nothing, or too little to divide by
  } else if (!(fabsf(most) < INFINITY)) {
    all = most;
    most = 1.f;
  }
  // the quotient: the largest weight times a rounded 1 / most would not always be f
  for (int64_t i = (int64_t)blockIdx.x * 1024 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 1024)
    row_scale[i] = counts(targets[i], ignore, V) ? (g_per_row ? f * (g[i] / most) : all) : 0.f;
  if (blockIdx.x == 0 && threadIdx.x == 0) alpha[0] = most / f;
}

// out = alpha * (slice 0 + slice 1 + ...), rounded once.  G warps of a block share the
// slices of 32 vectors, each a consecutive part of them, and are joined in order: with
// many slices of a small product one thread a vector is one long chain of loads.
template <typename T, int G>
__global__ void __launch_bounds__(256) join_slices_kernel(const float4* __restrict__ c, int slices, int64_t n4,
                                                          const float* __restrict__ alpha, T* __restrict__ out) {
  __shared__ float4 sh[8][32];
  const float a = alpha[0];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, part = warp % G;
  constexpr int kVecs = 32 * 8 / G;  // vectors a block
  for (int64_t i0 = (int64_t)blockIdx.x * kVecs; i0 < n4; i0 += (int64_t)gridDim.x * kVecs) {
    const int64_t i = i0 + (warp / G) * 32 + lane;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < n4) {
#pragma unroll 4
      for (int s = slices * part / G; s < slices * (part + 1) / G; ++s) {
        const float4 w = c[s * n4 + i];
        v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
      }
    }
    if constexpr (G > 1) {
      sh[warp][lane] = v;
      __syncthreads();
      if (part == 0) {
#pragma unroll
        for (int g = 1; g < G; ++g) {
          const float4 w = sh[warp + g][lane];
          v.x += w.x, v.y += w.y, v.z += w.z, v.w += w.w;
        }
      }
      __syncthreads();
    }
    if (part == 0 && i < n4) {
      union { uint2 raw; T t[4]; } o;
      o.t[0] = from_f<T>(v.x * a), o.t[1] = from_f<T>(v.y * a), o.t[2] = from_f<T>(v.z * a), o.t[3] = from_f<T>(v.w * a);
      reinterpret_cast<uint2*>(out)[i] = o.raw;
    }
  }
}

template <typename T>
void join_slices_as(const at::Tensor& c, int slices, const float* alpha, at::Tensor& out) {
  const int64_t n4 = out.numel() / 4;
  const float4* p = reinterpret_cast<const float4*>(c.data_ptr<float>());
  T* o = reinterpret_cast<T*>(out.data_ptr());
  const auto blocks = [&](int64_t vecs) { return (unsigned)std::min<int64_t>((n4 + vecs - 1) / vecs, (int64_t)num_sms() * 16); };
  // 512 x 256 outputs of 32 slices: 4.0 us by groups, 7.3 us by single threads
  if (slices >= 8) join_slices_kernel<T, 8><<<blocks(32), 256, 0, stream()>>>(p, slices, n4, alpha, o);
  else join_slices_kernel<T, 1><<<blocks(256), 256, 0, stream()>>>(p, slices, n4, alpha, o);
  LRB_LAUNCH_CHECK();
}

void join_slices(const at::Tensor& c, int slices, const float* alpha, at::Tensor& out) {
  if (out.scalar_type() == at::kBFloat16) join_slices_as<__nv_bfloat16>(c, slices, alpha, out);
  else join_slices_as<__half>(c, slices, alpha, out);
}

void check_head_inputs(const at::Tensor& h, const at::Tensor& w, const at::Tensor& targets) {
  LRB_CHECK(h.is_cuda() && w.is_cuda() && targets.is_cuda() && h.device() == w.device() && h.device() == targets.device(),
            "linear cross entropy: h, w and targets must be on one CUDA device");
  LRB_CHECK((h.scalar_type() == at::kBFloat16 || h.scalar_type() == at::kHalf) && w.scalar_type() == h.scalar_type(),
            "linear cross entropy: h and w must both be bf16 or both fp16");
  LRB_CHECK(h.dim() == 2 && w.dim() == 2 && h.size(1) == w.size(1) && w.size(0) >= 1 && h.size(1) >= 1,
            "linear cross entropy: h (N, d) and w (V, d), V and d at least 1");
  LRB_CHECK(targets.scalar_type() == at::kLong && targets.is_contiguous() && targets.numel() == h.size(0),
            "linear cross entropy: contiguous int64 targets (N)");
}

}  // namespace

// Returns (row losses, row statistics (N, 2), the loss and each counted row's factor in
// it: reduction 1 is the sum and 2 the mean over the counted rows; not filled for 0).
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> linear_ce_fwd(const at::Tensor& h, const at::Tensor& w,
                                                                         const at::Tensor& targets, int64_t ignore,
                                                                         int64_t reduction) {
  check_head_inputs(h, w, targets);
  c10::cuda::CUDAGuard guard(h.device());
  bind_device(h.get_device());
  const int64_t n = h.size(0), V = w.size(0);
  auto f32 = h.options().dtype(at::kFloat);
  auto loss = at::empty({n}, f32), stats = at::empty({n, 2}, f32);
  auto out = at::empty({}, f32), factor = at::empty({1}, f32), counted = at::empty({n}, f32);
  if (n > 0) {
    const int64_t tiles = gemm_pair_lse_tiles(V);
    auto part = at::empty({tiles, n, 2}, f32), target_logit = at::empty({n}, f32);
    gemm_pair_lse(h, w, targets, part, target_logit);
    join_tiles_kernel<<<(unsigned)((n + 31) / 32), 256, 0, stream()>>>(
        reinterpret_cast<const float2*>(part.data_ptr<float>()), target_logit.data_ptr<float>(),
        targets.data_ptr<int64_t>(), n, V, (int)tiles, ignore, reinterpret_cast<float2*>(stats.data_ptr<float>()),
        loss.data_ptr<float>(), counted.data_ptr<float>());
    LRB_LAUNCH_CHECK();
  }
  if (reduction != 0)
    reduce_rows(loss.data_ptr<float>(), counted.data_ptr<float>(), n, reduction == 2, out.data_ptr<float>(),
                factor.data_ptr<float>(), stream());
  return {loss, stats, out, factor};
}

// (dh, dw), each empty where it is not asked for.  `g` fp32: one value for each row,
// or a single one that is multiplied by `factor`.  `piece`: vocabulary rows at a time, a
// multiple of 8; 0: gemm_pair_ce_piece's, of a buffer of at most 256 MB or 1024 rows.
std::tuple<at::Tensor, at::Tensor> linear_ce_bwd(const at::Tensor& h, const at::Tensor& w, const at::Tensor& targets,
                                                 int64_t ignore, const at::Tensor& stats, const at::Tensor& g,
                                                 bool g_per_row, const at::Tensor& factor, int64_t piece, bool need_h,
                                                 bool need_w) {
  check_head_inputs(h, w, targets);
  const int64_t n = h.size(0), V = w.size(0), d = h.size(1);
  LRB_CHECK(g.is_cuda() && g.scalar_type() == at::kFloat && g.is_contiguous() && g.numel() == (g_per_row ? n : 1) &&
                stats.scalar_type() == at::kFloat && stats.is_contiguous() && stats.numel() == 2 * n &&
                (g_per_row || (factor.is_cuda() && factor.scalar_type() == at::kFloat && factor.numel() >= 1)),
            "linear cross entropy backward: bad gradient or statistics");
  LRB_CHECK(piece >= 0 && piece % 8 == 0, "linear cross entropy backward: piece must be a multiple of 8");
  c10::cuda::CUDAGuard guard(h.device());
  const int dev = h.get_device();
  bind_device(dev);
  auto dh = need_h ? at::empty({n, d}, h.options()) : at::empty({0}, h.options());
  auto dw = need_w ? (n > 0 ? at::empty({V, d}, w.options()) : at::zeros({V, d}, w.options())) : at::empty({0}, w.options());
  if (n == 0 || !(need_h || need_w)) return {dh, dw};
  auto f32 = h.options().dtype(at::kFloat);
  auto scale = at::empty({n + 1}, f32);  // row scales, then alpha
  const float* alpha = scale.data_ptr<float>() + n;
  row_scale_kernel<<<(unsigned)std::min<int64_t>((n + 1023) / 1024, num_sms()), 1024, 0, stream()>>>(
      targets.data_ptr<int64_t>(), n, V, ignore, g.data_ptr<float>(), g_per_row ? 1 : 0,
      g_per_row ? nullptr : factor.data_ptr<float>(), h.scalar_type() == at::kHalf ? 8192.f : 1.f, scale.data_ptr<float>(),
      scale.data_ptr<float>() + n);
  LRB_LAUNCH_CHECK();
  if (piece == 0) piece = gemm_pair_ce_piece(n, V, d, 256 << 20, dev);
  piece = std::min(piece, (V + 7) / 8 * 8);
  auto buf = at::empty({n, piece}, h.options());
  // dh: K ranges of the first piece as slices, later pieces added to them
  const int sh = need_h ? gemm_pair_slices(n, d, std::min(piece, V), dev) : 1;
  const bool direct = sh == 1 && piece >= V;
  at::Tensor dhs;
  if (need_h && !direct) dhs = at::empty({sh, n, d}, f32);
  for (int64_t v0 = 0; v0 < V; v0 += piece) {
    const int64_t pw = std::min(piece, V - v0);
    auto wp = w.narrow(0, v0, pw);
    auto dz = buf.narrow(1, 0, pw);
    gemm_pair_ce_grad(h, wp, targets, v0, stats, scale, dz);
    if (need_h) {
      if (direct) gemm_pair_sliced(dz, wp, false, true, dh, 1, false, alpha);
      else gemm_pair_sliced(dz, wp, false, true, dhs, (int)std::min<int64_t>(sh, (pw + 63) / 64), v0 > 0, nullptr);
    }
    if (need_w) {
      auto dwp = dw.narrow(0, v0, pw);
      const int sw = gemm_pair_slices(pw, d, n, dev);
      if (sw == 1) {
        gemm_pair_sliced(dz, h, true, true, dwp, 1, false, alpha);
      } else {
        auto dws = at::empty({sw, pw, d}, f32);
        gemm_pair_sliced(dz, h, true, true, dws, sw, false, nullptr);
        join_slices(dws, sw, alpha, dwp);
      }
    }
  }
  if (need_h && !direct) join_slices(dhs, sh, alpha, dh);
  return {dh, dw};
}

}  // namespace lrb

// The logits of given tokens (lce_token_logits): what its two calls need beside the kernels of the loss.
//
// With z = scale * x W and lse = log sum exp z the gradients of a row, for upstream gradients g_lse and g_logit of its lse and of the
// logit of its column y, are those of
//     dz[v] = g_lse * exp(z[v] - lse) + g_logit * [v == y]
// The kernels of the loss's backward stage +-exp(z - lse'), lse' = lse - log |g_lse|: no product more than with z-regularisation and no
// register (a number of its own for each row, held over the last K tiles, put 50 to 100 registers of the dz kernels into memory).
// lse' is rounded at 24 bits, which moves a probability by a factor of 1 +- 2^-19 at |lse'| < 32, as far as the rounding of its
// exponent does.  The label's column is written over the stage afterwards, from the logit that the forward gave (row_targets_kernel); the
// kernel for few hidden indices, which stages nothing, puts it in as it goes (lce_narrow.hip).
//
// fp16, and fp32 as fp16 pairs: a stage has 30 binary places below 1 while upstream gradients are of any size (1 / rows, times a loss
// scale), so all are divided by one power of two, which the dx and dW kernels multiply in again after their fp32 sums.
//
// All of that is a few numbers a row: bound by launches, 2 to 5 us each.  The products around it run at the loss's rate: 12288 rows of 2048 x 131072
// with their backward in 19.5 ms, 1.35 PFLOP/s of 8 N H V operations, of 4096 x 128256 in 37.2 ms, 1.39 (a large library product here: 1.38).
//
// fp32 tensors: fp16 pairs (lce_gemm.h) instead of the loss's bf16 ones, for products 22 bits wide.  N=2048, H=1024, V=16384, errors of dx and
// dW against fp64, relative to their norms: 3.4e-7, of bf16 pairs 4.4e-6 (a float32 library product and its softmax: 2.2e-6).  Their scales
// cost one more pass over the weight and x (pair_max_kernel 20 us, pair_scales_kernel 5, of a forward and backward of 910; 930 where the backward
// has no scales).
#include "lce_gemm3.h"
#include "lce_internal.h"

namespace lce {

namespace {

constexpr int kRowThreads = 256;

__device__ float largest_of_workgroup(float m) {
  __shared__ float sh[kRowThreads / 64];
  for (int d = 32; d > 0; d /= 2) m = fmaxf(m, __shfl_xor(m, d));
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = m;
  __syncthreads();
  m = sh[0];
  for (int i = 1; i < kRowThreads / 64; ++i) m = fmaxf(m, sh[i]);
  return m;
}

// part[b] = the largest |g_lse| + |g_logit| of this workgroup's rows (NaN does not count; the rows it is in are NaN anyway).
__global__ __launch_bounds__(kRowThreads) void row_gradient_max_kernel(const RowGradients g) {
  float m = 0.f;
  for (int64_t i = (int64_t)blockIdx.x * kRowThreads + threadIdx.x; i < g.N; i += (int64_t)gridDim.x * kRowThreads)
    if (g.y[i] != g.ignore_index) m = fmaxf(m, fabsf(g.grad_lse[i]) + fabsf(g.grad_logits[i]));
  m = largest_of_workgroup(m);
  if (threadIdx.x == 0) g.part[blockIdx.x] = m;
}

// 2^shift * dz at a label.
__device__ float target(float g_lse, float g_logit, float logit, float lse, int shift) {
  return ldexpf(fmaf(g_lse, __expf(logit - lse), g_logit), shift);
}

__global__ __launch_bounds__(kRowThreads) void row_gradients_kernel(const RowGradients g, int parts) {
  int e = 0;  // the factor is 2^e
  if (parts > 0) {
    const float m = largest_of_workgroup((int)threadIdx.x < parts ? g.part[threadIdx.x] : 0.f);
    if (m > 0.f && m < INFINITY) {
      (void)frexpf(m, &e);
      e = e < -126 ? -126 : e > 127 ? 127 : e;
    }
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    const float f = ldexpf(1.f, e);
    g.factor[0] = f;
    g.factor[1] = g.pair != nullptr ? f * g.pair[kPairDx] : f;
    g.factor[2] = g.pair != nullptr ? f * g.pair[kPairDw] : f;
    *g.one = 1;
  }
  for (int64_t j = (int64_t)blockIdx.x * kRowThreads + threadIdx.x; j < g.N; j += (int64_t)gridDim.x * kRowThreads) {
    const int64_t n = g.perm != nullptr ? packed_token(g.perm, j, g.N) : j, yy = g.y[n];
    // (a row that does not count may hold any upstream gradient, NaN too, and its numbers are finite all the same: the kernels multiply its
    // dz of 0 by a factor made of them)
    const bool counts = yy != g.ignore_index;
    const float gl = counts ? ldexpf(g.grad_lse[n], -e) : 0.f;
    // (no gradient: exp(z - lse') is 0 whatever the logits.  Finite as well, for a z_reg of 0 is multiplied by it.)
    const float l = g.lse[n] - logf(fabsf(gl));
    g.row_lse[j] = !counts ? 0.f : l > 1e30f ? 1e30f : l < -1e30f ? -1e30f : l;
    if (g.row_value == nullptr) {
      g.row_y[j] = !counts ? -1 : gl < 0.f ? kNegativeRow : g.V;
    } else {
      g.row_y[j] = !counts ? -1 : yy >= 0 && yy < g.V ? yy : g.V;
      g.row_value[j] = counts ? pack_row_value(target(gl, ldexpf(g.grad_logits[n], -e), g.logits[n], g.lse[n], g.dz_shift), gl < 0.f) : 0.f;
    }
  }
}

// The staged dz at the labels' columns of this slab: 2^shift * (g_lse * softmax + g_logit), rounded once.
template <class T>
__global__ __launch_bounds__(kRowThreads) void row_targets_kernel(const BwdArgs a, const RowGradients g) {
  const int64_t rows = packed_rows(a.n_rows, a.N);
  for (int64_t j = (int64_t)blockIdx.x * kRowThreads + threadIdx.x; j < rows; j += (int64_t)gridDim.x * kRowThreads) {
    const int64_t n = g.perm != nullptr ? packed_token(g.perm, j, g.N) : j;
    const int64_t yy = g.y[n], rel = yy - a.v0;
    if (yy == g.ignore_index || yy < 0 || yy >= a.V || rel < 0 || rel >= a.vw) continue;
    const float f = *g.factor;  // (quotients by a power of two are exact)
    const float d = target(g.grad_lse[n] / f, g.grad_logits[n] / f, g.logits[n], g.lse[n], a.dz_shift);
    const int64_t at = (j & (kTile - 1)) * 64 + (rel & 63);
    unsigned short* dz = reinterpret_cast<unsigned short*>(a.dz);
    if constexpr (is_pair<T>::value) {
      dz += 2 * dz_block_offset(j / kTile, rel / 64, a.vs) + at;
      dz[0] = to_bits<T>(d);
      dz[kDzBlockElems] = to_bits<T>(part_lo<T>(d));
    } else {
      dz[dz_block_offset(j / kTile, rel / 64, a.vs) + at] = to_bits<T>(d);
    }
  }
}

__global__ __launch_bounds__(kRowThreads) void token_labels_kernel(const int64_t* tokens, int64_t N, int64_t ignore_index, int64_t start,
                                                                   int64_t V, int64_t size, int64_t* out) {
  for (int64_t i = (int64_t)blockIdx.x * kRowThreads + threadIdx.x; i < N; i += (int64_t)gridDim.x * kRowThreads) {
    const int64_t t = tokens[i];
    out[i] = t == ignore_index ? -1 : t < 0 || t >= size ? V + 1 : t >= start && t < start + V ? t - start : V;
  }
}

// part[b] = the largest finite magnitude of this workgroup's pieces: of kept rows of x (the first x_groups workgroups) or of the weight.
constexpr int64_t kScalePiece = 4 * kRowThreads;  // numbers of a row that a workgroup looks at at a time, four such in flight
__global__ __launch_bounds__(kRowThreads) void pair_max_kernel(const float* x, int64_t ldx, int64_t N, int64_t H, const int64_t* y, int64_t ignore_index,
                                                               const float* w, int64_t ldw, int64_t V, int x_groups, float* part) {
  const bool of_x = (int)blockIdx.x < x_groups;
  const float* t = of_x ? x : w;
  const int64_t rows = of_x ? N : H, cols = of_x ? H : V, ld = of_x ? ldx : ldw, per = (cols + kScalePiece - 1) / kScalePiece;
  const int64_t first = 4 * (of_x ? blockIdx.x : blockIdx.x - x_groups), step = 4 * (of_x ? x_groups : (int64_t)gridDim.x - x_groups);
  const int64_t step_r = step / per, step_c = step - step_r * per;
  float m = 0.f;
  for (int64_t r = first / per, c = first - r * per; r < rows;) {
    int64_t rk = r, ck = c;
    f32x4_t q[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int64_t at = ck * kScalePiece + (int)threadIdx.x * 4;
      q[k] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      if (rk < rows && !(of_x && y[rk] == ignore_index)) {
        const float* from = t + rk * ld + at;
        if (at + 4 <= cols) {
          q[k] = *reinterpret_cast<const f32x4_t*>(from);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (at + j < cols) q[k][j] = from[j];
        }
      }
      if (++ck == per) {
        ck = 0;
        ++rk;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float a = fabsf(q[k][j]);
        m = a < INFINITY && a > m ? a : m;
      }
    r += step_r;
    c += step_c;
    if (c >= per) {
      c -= per;
      ++r;
    }
  }
  m = largest_of_workgroup(m);
  if (threadIdx.x == 0) part[blockIdx.x] = m;
}
__global__ __launch_bounds__(kRowThreads) void pair_scales_kernel(const float* part, int x_groups, int groups, float* pair) {
  __shared__ int exponent[2];
  for (int of = 0; of < 2; ++of) {
    float m = 0.f;
    for (int i = (of == 0 ? 0 : x_groups) + threadIdx.x; i < (of == 0 ? x_groups : groups); i += kRowThreads) m = fmaxf(m, part[i]);
    m = largest_of_workgroup(m);
    if (threadIdx.x == 0) {
      int e = 0;
      if (m > 0.f) (void)frexpf(m, &e);
      e = 14 - e;  // the largest becomes 2^13 ... 2^14
      exponent[of] = m > 0.f ? (e > 120 ? 120 : e) : 0;
    }
    __syncthreads();
  }
  if (threadIdx.x == 0) {
    // (the logits' factor stays a number of float32 with all its bits, times any logit_scale above 2^-6)
    const int more = exponent[0] + exponent[1] - 120;
    const int ex = exponent[0] - (more > 0 ? (more + 1) / 2 : 0), ew = exponent[1] - (more > 0 ? more / 2 : 0);
    pair[kPairX] = ldexpf(1.f, ex);
    pair[kPairW] = ldexpf(1.f, ew);
    pair[kPairLogits] = ldexpf(1.f, -ex - ew);
    pair[kPairDx] = ldexpf(1.f, -ew);
    pair[kPairDw] = ldexpf(1.f, -ex);
  }
}

unsigned row_groups(int64_t N, int64_t most) {
  const int64_t n = (N + kRowThreads - 1) / kRowThreads;
  return (unsigned)(n < most ? n : most);
}

}  // namespace

hipError_t launch_row_gradients(const RowGradients& g, hipStream_t s) {
  const int parts = g.normalise ? (int)row_groups(g.N, kRowGradientParts) : 0;
  if (parts > 0) {
    hipLaunchKernelGGL(row_gradient_max_kernel, dim3(parts), dim3(kRowThreads), 0, s, g);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(row_gradients_kernel, dim3(row_groups(g.N, 1024)), dim3(kRowThreads), 0, s, g, parts);
  return hipGetLastError();
}

hipError_t launch_row_targets(const BwdArgs& a, const RowGradients& g, hipStream_t s) {
  const dim3 grid(row_groups(a.N, 1024)), threads(kRowThreads);
  if (a.x_dtype == DT_HALF_PAIR) hipLaunchKernelGGL(row_targets_kernel<F16P>, grid, threads, 0, s, a, g);
  else if (a.x_dtype == DT_F16) hipLaunchKernelGGL(row_targets_kernel<F16>, grid, threads, 0, s, a, g);
  else hipLaunchKernelGGL(row_targets_kernel<BF16>, grid, threads, 0, s, a, g);
  return hipGetLastError();
}

hipError_t launch_pair_scales(const float* x, int64_t ldx, int64_t N, int64_t H, const int64_t* y, int64_t ignore_index, const float* w, int64_t ldw,
                              int64_t V, float* pair, float* part, hipStream_t s) {
  const int64_t px = (N * ((H + kScalePiece - 1) / kScalePiece) + 3) / 4, pw = (H * ((V + kScalePiece - 1) / kScalePiece) + 3) / 4;
  const int x_groups = (int)(px < kPairParts / 4 ? px : kPairParts / 4), w_groups = (int)(pw < kPairParts * 3 / 4 ? pw : kPairParts * 3 / 4);
  hipLaunchKernelGGL(pair_max_kernel, dim3(x_groups + w_groups), dim3(kRowThreads), 0, s, x, ldx, N, H, y, ignore_index, w, ldw, V, x_groups, part);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  hipLaunchKernelGGL(pair_scales_kernel, dim3(1), dim3(kRowThreads), 0, s, part, x_groups, x_groups + w_groups, pair);
  return hipGetLastError();
}

hipError_t launch_token_labels(const int64_t* tokens, int64_t N, int64_t ignore_index, int64_t start, int64_t V, int64_t size, int64_t* out,
                               hipStream_t s) {
  hipLaunchKernelGGL(token_labels_kernel, dim3(row_groups(N, 1024)), dim3(kRowThreads), 0, s, tokens, N, ignore_index, start, V, size, out);
  return hipGetLastError();
}

}  // namespace lce

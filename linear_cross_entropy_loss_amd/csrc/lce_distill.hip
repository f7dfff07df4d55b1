// Distillation from a teacher's top logits: what the loss against soft targets needs besides the kernels of the loss itself.
//
//   z[n][v] = s sum_h x[n][h] W[h][v],  s = logit_scale / temperature,  lse[n] = log sum_v exp z[n][v]
//   q[n][k] = softmax over the entries of row n of (teacher logit / temperature)
//   loss    = 1/R sum_n (lse[n] + sum_k q[n][k] (log q[n][k] - z[n][index[n][k]])),  R = rows with an entry
//   dz[n][v] = softmax(z[n])[v] - sum of q[n][k] over the k with index[n][k] = v
//
// lse, the softmax and the two contractions of dz are those of the loss against labels, and so are their kernels: a row's first
// entry serves as its label, a row without an entry has none.  Here are the pieces that know of more than one target: the teacher's
// distribution (soft_targets_kernel), the student's logits at its columns (soft_logits_kernel), the loss from both, and the
// columns' values in the staged dz (soft_gradient_kernel), each the rounding of one fp32 value as at a label.
#include "lce_gemm.h"
#include "lce_internal.h"

namespace lce {

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int64_t kMostGroups = 1 << 20;  // workgroups of a launch

LCE_DEV float wave_max(float v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v = fmaxf(v, __shfl_xor(v, d));
  return v;
}
template <class F> LCE_DEV F wave_sum(F v) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  return v;
}

LCE_DEV float load_float(const void* p, int dtype, int64_t i) {
  if (dtype == DT_F32) return reinterpret_cast<const float*>(p)[i];
  const unsigned short b = reinterpret_cast<const unsigned short*>(p)[i];
  return dtype == DT_BF16 ? from_bits<BF16>(b) : from_bits<F16>(b);
}

// A wave per row, PER entries to a lane.  An entry is there if its index is not negative and its logit not -inf.  q: their softmax,
// in fp32 (a NaN or +inf among them makes all of the row's NaN, and the loss with it).  Entries of the same column are added up, in
// their order, and the first of them stands for all: a hash table of the row's columns in LDS finds out whether there are any,
// which is rare.  An index that is no column of W gives the row a label that is none either, which makes the loss NaN.
// Bound by launch and latency: 12 bytes read and 8 written per entry.
constexpr int kTargetWaves = 4;
template <int PER>
__global__ __launch_bounds__(64 * kTargetWaves) void soft_targets_kernel(const int64_t* index, int64_t ld_index, const void* logits, int dtype,
                                                                         int64_t ld_logits, int64_t N, int K, int64_t V, float temperature,
                                                                         int* out_index, float* out_q, int64_t* y) {
  constexpr int kEntries = 64 * PER, kTable = 2 * kEntries;
  __shared__ int sh_table[kTargetWaves][kTable];
  __shared__ int sh_index[kTargetWaves][kEntries];
  __shared__ float sh_q[kTargetWaves][kEntries];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int64_t n = (int64_t)blockIdx.x * kTargetWaves + wave; n < N; n += (int64_t)gridDim.x * kTargetWaves) {
    int64_t at[PER];
    float l[PER];
    float m = -INFINITY;
  #pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int k = lane + 64 * i;
      at[i] = k < K ? index[n * ld_index + k] : -1;
      l[i] = k < K ? load_float(logits, dtype, n * ld_logits + k) : -INFINITY;
      if (l[i] == -INFINITY) at[i] = -1;
      if (at[i] < 0) l[i] = -INFINITY;
      m = fmaxf(m, l[i]);
    }
    m = wave_max(m);
    float s = 0.f;
    bool bad = false;
    int first = K;
  #pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (at[i] >= 0) {
        l[i] = expf((l[i] - m) / temperature);
        s += l[i];
        bad = bad || at[i] >= V;
        if (lane + 64 * i < first) first = lane + 64 * i;
      } else {
        l[i] = 0.f;
      }
    }
    s = wave_sum(s);
  #pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_xor(first, d);
      first = o < first ? o : first;
    }
    bad = __any(bad);
  #pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (lane + 64 * i == first) y[n] = bad ? V : at[i];
      if (at[i] >= 0) l[i] /= s;
      if (at[i] >= V) at[i] = -1;
    }
    if (first == K && lane == 0) y[n] = -1;
    // does a column occur twice?
  #pragma unroll
    for (int i = 0; i < 2 * PER; ++i) sh_table[wave][lane + 64 * i] = -1;
    __threadfence_block();
    __builtin_amdgcn_wave_barrier();
    bool twice = false;
  #pragma unroll
    for (int i = 0; i < PER; ++i)
      if (at[i] >= 0) {
        const int v = (int)at[i];
        // (a table of twice as many places as there are entries: a free one is found)
        for (unsigned h = (unsigned)v * 2654435761u >> 12;; ++h) {
          const int was = atomicCAS(&sh_table[wave][h & (kTable - 1)], -1, v);
          if (was == v) twice = true;
          if (was == -1 || was == v) break;
        }
      }
    if (__any(twice)) {
  #pragma unroll
      for (int i = 0; i < PER; ++i) {
        sh_index[wave][lane + 64 * i] = (int)at[i];
        sh_q[wave][lane + 64 * i] = l[i];
      }
      __threadfence_block();
      __builtin_amdgcn_wave_barrier();
  #pragma unroll
      for (int i = 0; i < PER; ++i) {
        const int mine = (int)at[i];
        bool leads = true;
        float sum = 0.f;
        for (int j = 0; j < K; ++j)
          if (sh_index[wave][j] == mine) {
            if (j < lane + 64 * i) leads = false;
            sum += sh_q[wave][j];
          }
        if (mine >= 0) {
          at[i] = leads ? mine : -1;
          l[i] = leads ? sum : 0.f;
        }
      }
    }
  #pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int k = lane + 64 * i;
      if (k < K) {
        out_index[n * K + k] = (int)at[i];
        out_q[n * K + k] = at[i] >= 0 ? l[i] : 0.f;
      }
    }
  }
}

// The student's logits at the teacher's columns, in fp32 from operands of the compute type.  A wave per entry.
template <class XT, class WT, bool WVH>
__global__ __launch_bounds__(256) void soft_logits_kernel(const SoftLogits a) {
  const int lane = threadIdx.x & 63;
  for (int64_t e = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); e < a.N * a.K; e += (int64_t)gridDim.x * 4) {
    const int v = a.index[e];
    float z = 0.f;
    if (v >= 0) {
      const XT* x = reinterpret_cast<const XT*>(a.x) + e / a.K * a.ldx;
      const WT* w = reinterpret_cast<const WT*>(a.w);
      for (int64_t h = lane; h < a.H; h += 64) {
        const WT c = w[WVH ? (int64_t)v * a.ldw + h : h * a.ldw + v];
        z = fmaf((float)x[h], (float)(XT)c, z);
      }
      z = wave_sum(z);
    }
    if (lane == 0) a.z[e] = z * a.scale;
  }
}

// The staged dz at the teacher's columns: 2^shift * (softmax - q), rounded once.  A thread per entry; rows in the order of the stage.
// Bound by the partial lines that it writes: 64 to 128 bytes of memory traffic per entry.
template <class T>
__global__ __launch_bounds__(256) void soft_gradient_kernel(const BwdArgs a, const SoftTargets t) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x, row = e / t.K;
  if (row >= packed_rows(a.n_rows, a.N)) return;
  const int64_t n = a.perm != nullptr ? packed_token(a.perm, row, t.N) : t.row0 + row;
  const int64_t i = n * t.K + (e - row * t.K);
  const int64_t v = t.index[i], rel = v - a.v0;
  if (v < 0 || rel < 0 || rel >= a.vw) return;
  const float q = t.q[i];
  const float p = __builtin_amdgcn_exp2f(fmaf(t.z[i] - a.lse[row], kLog2e, (float)a.dz_shift));
  const float d = p - q * __builtin_bit_cast(float, (127 + a.dz_shift) << 23);
  const int64_t at = (row & (kTile - 1)) * 64 + (rel & 63);
  unsigned short* dz = reinterpret_cast<unsigned short*>(a.dz);
  if constexpr (is_pair<T>::value) {
    dz += 2 * dz_block_offset(row / kTile, rel / 64, a.vs) + at;
    dz[0] = to_bits<BF16>(d);
    dz[kDzBlockElems] = to_bits<BF16>(bf16_lo(d));
  } else {
    dz[dz_block_offset(row / kTile, rel / 64, a.vs) + at] = to_bits<T>(d);
  }
}

// The rows' terms of the loss, a wave per row, and their sum in doubles: one partial sum to a workgroup, or -- FINAL, a single
// workgroup -- the loss.
constexpr int kLossWaves = 16, kLossGroups = 512;
template <bool FINAL>
__global__ __launch_bounds__(64 * kLossWaves) void soft_loss_kernel(const SoftTargets t, const int64_t* y, const float* lse, int64_t V,
                                                                    const int64_t* n_valid, double* part, float* loss) {
  __shared__ double sh[kLossWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double sum = 0.0;
  for (int64_t n = (int64_t)blockIdx.x * kLossWaves + wave; n < t.N; n += (int64_t)gridDim.x * kLossWaves) {
    const int64_t yy = y[n];
    if (yy < 0) continue;
    float term = 0.f;
    const float l = lse[n];
    for (int k = lane; k < t.K; k += 64) {
      const float q = t.q[n * t.K + k];
      if (q != 0.f) term = fmaf(q, logf(q) + (l - t.z[n * t.K + k]), term);
    }
    sum += yy < V ? (double)term : (double)__builtin_nanf("");
  }
  sum = wave_sum(sum);
  if (lane == 0) sh[wave] = sum;
  __syncthreads();
  if (threadIdx.x != 0) return;
  double total = 0.0;
  for (int i = 0; i < kLossWaves; ++i) total += sh[i];
  if (FINAL) loss[0] = (float)(total / (double)n_valid[0]);  // no row with an entry: 0/0 = NaN, as against labels
  else part[blockIdx.x] = total;
}
__global__ __launch_bounds__(64) void soft_loss_sum_kernel(const double* part, int groups, const int64_t* n_valid, float* loss) {
  double sum = 0.0;
  for (int i = threadIdx.x; i < groups; i += 64) sum += part[i];
  sum = wave_sum(sum);
  if (threadIdx.x == 0) loss[0] = (float)(sum / (double)n_valid[0]);
}

template <class XT, class WT> void launch_logits(const SoftLogits& a, hipStream_t s) {
  const int64_t groups = (a.N * a.K + 3) / 4;
  const dim3 grid((unsigned)(groups < kMostGroups ? groups : kMostGroups));
  if (a.w_vh) hipLaunchKernelGGL((soft_logits_kernel<XT, WT, true>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((soft_logits_kernel<XT, WT, false>), grid, dim3(256), 0, s, a);
}

}  // namespace

hipError_t launch_soft_targets(const int64_t* index, int64_t ld_index, const void* logits, int dtype, int64_t ld_logits, int64_t N, int K,
                               int64_t V, float temperature, int* out_index, float* out_q, int64_t* y, hipStream_t s) {
  const int64_t groups = (N + kTargetWaves - 1) / kTargetWaves;
  const dim3 grid((unsigned)(groups < kMostGroups ? groups : kMostGroups)), block(64 * kTargetWaves);
#define LCE_TARGETS(PER)                                                                                                          \
  hipLaunchKernelGGL(soft_targets_kernel<PER>, grid, block, 0, s, index, ld_index, logits, dtype, ld_logits, N, K, V, temperature, \
                     out_index, out_q, y)
  if (K <= 64) LCE_TARGETS(1);
  else if (K <= 128) LCE_TARGETS(2);
  else if (K <= 256) LCE_TARGETS(4);
  else if (K <= 512) LCE_TARGETS(8);
  else if (K <= 1024) LCE_TARGETS(16);
  else return hipErrorInvalidValue;
#undef LCE_TARGETS
  return hipGetLastError();
}

hipError_t launch_soft_logits(const SoftLogits& a, hipStream_t s) {
  if (a.x_dtype == DT_BF16 && a.w_dtype == DT_BF16) launch_logits<__bf16, __bf16>(a, s);
  else if (a.x_dtype == DT_BF16 && a.w_dtype == DT_F32) launch_logits<__bf16, float>(a, s);
  else if (a.x_dtype == DT_F16 && a.w_dtype == DT_F16) launch_logits<_Float16, _Float16>(a, s);
  else if (a.x_dtype == DT_F16 && a.w_dtype == DT_F32) launch_logits<_Float16, float>(a, s);
  else if (a.x_dtype == DT_F32 && a.w_dtype == DT_F32) launch_logits<float, float>(a, s);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}

hipError_t launch_soft_gradient(const BwdArgs& a, const SoftTargets& t, hipStream_t s) {
  const int64_t rows = a.Np < a.N ? a.Np : a.N;
  const dim3 grid((unsigned)((rows * t.K + 255) / 256));
  if (a.x_dtype == DT_BF16) hipLaunchKernelGGL(soft_gradient_kernel<BF16>, grid, dim3(256), 0, s, a, t);
  else if (a.x_dtype == DT_F16) hipLaunchKernelGGL(soft_gradient_kernel<F16>, grid, dim3(256), 0, s, a, t);
  else if (a.x_dtype == DT_PAIR) hipLaunchKernelGGL(soft_gradient_kernel<BF16P>, grid, dim3(256), 0, s, a, t);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}

hipError_t launch_soft_loss(const SoftTargets& t, const int64_t* y, const float* lse, int64_t V, const int64_t* n_valid, double* part,
                            float* loss, hipStream_t s) {
  const int64_t blocks = (t.N + kLossWaves - 1) / kLossWaves;
  const int grid = (int)(blocks < kLossGroups ? blocks : kLossGroups);
  // (a workgroup's rows one after another: a second launch where it would be more than a few)
  if (t.N <= 4 * kLossWaves) {
    hipLaunchKernelGGL(soft_loss_kernel<true>, dim3(1), dim3(64 * kLossWaves), 0, s, t, y, lse, V, n_valid, part, loss);
  } else {
    hipLaunchKernelGGL(soft_loss_kernel<false>, dim3((unsigned)grid), dim3(64 * kLossWaves), 0, s, t, y, lse, V, n_valid, part, loss);
    hipLaunchKernelGGL(soft_loss_sum_kernel, dim3(1), dim3(64), 0, s, part, grid, n_valid, loss);
  }
  return hipGetLastError();
}

int soft_loss_groups() { return kLossGroups; }

}  // namespace lce

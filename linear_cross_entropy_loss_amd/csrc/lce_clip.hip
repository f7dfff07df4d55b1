// The norm of many tensors together and their scaling to at most a given one (lce_clip).
//
//     norm = sqrt(sum g^2) / divisor,   out = g * min(1, max_norm / norm) / divisor
//
// Two launches for every kEntries tensors, however long they are: the tensors are cut into stretches of kStretch elements, which
// the workgroups take one after another.  The first sums squares, in doubles (a float32 gradient may be 10^-30 or 10^30, whose square is no
// float32), one partial sum to a workgroup; in the second every workgroup adds up all partial sums, in the same order, and scales.
// The list of tensors travels in the kernels' arguments: nothing is copied to the device, and a captured launch holds its own.
//
// Bound by memory beyond some MiB, by the two launches below (13 us for 0.16M float32).  470M bf16 to float32: 660 us for 3.76 GB, 5.7 TB/s (the norm 6.2
// to 6.3 TB/s, what reading alone reaches here; a copy of as much 5.3).
// ONCE: tensors that together do not fit the 256 MiB Infinity Cache go past it (loads and stores that are not kept): 739 to 660 us.
// Smaller ones the second launch finds there.
#include "lce_gemm.h"
#include "lce_internal.h"

namespace lce {

namespace {

constexpr int kClipThreads = 256;
constexpr int kStretch = 8192;

// 16 bytes at any 2-byte address: one load or store all the same.
typedef u32x4_t __attribute__((aligned(2))) piece_t;
template <bool ONCE> LCE_DEV u32x4_t load_piece(const void* p) {
  const piece_t* q = reinterpret_cast<const piece_t*>(p);
  return ONCE ? __builtin_nontemporal_load(q) : *q;
}
template <bool ONCE> LCE_DEV void store_piece(void* p, u32x4_t v) {
  piece_t* q = reinterpret_cast<piece_t*>(p);
  if (ONCE) __builtin_nontemporal_store(v, q);
  else *q = v;
}

template <int DT> struct Elem {
  static constexpr int kPer = 8;
  typedef unsigned short S;
  static LCE_DEV float get(S b) { return DT == DT_BF16 ? from_bits<BF16>(b) : from_bits<F16>(b); }
  static LCE_DEV S put(float f) { return DT == DT_BF16 ? to_bits<BF16>(f) : to_bits<F16>(f); }
};
template <> struct Elem<DT_F32> {
  static constexpr int kPer = 4;
  typedef float S;
  static LCE_DEV float get(S f) { return f; }
  static LCE_DEV S put(float f) { return f; }
};

// The tensor that stretch c of the launch is a part of.
LCE_DEV int entry_of(const ClipBatch& b, unsigned c) {
  int lo = 0, hi = b.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (b.e[mid].first <= c) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <int DT, bool ONCE> LCE_DEV void add_squares(const void* at, int n, double (&sum)[4]) {
  typedef Elem<DT> E;
  constexpr int kStep = kClipThreads * E::kPer, kRounds = kStretch / kStep;
  const typename E::S* p = reinterpret_cast<const typename E::S*>(at);
  const int t = threadIdx.x;
  if (n == kStretch) {
    u32x4_t v[kRounds];
#pragma unroll
    for (int r = 0; r < kRounds; ++r) v[r] = load_piece<ONCE>(p + r * kStep + t * E::kPer);
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
      typename E::S e[E::kPer];
      __builtin_memcpy(e, &v[r], 16);
#pragma unroll
      for (int i = 0; i < E::kPer; ++i) {
        const double d = (double)E::get(e[i]);
        sum[i & 3] = fma(d, d, sum[i & 3]);
      }
    }
    return;
  }
  for (int i = t; i < n; i += kClipThreads) {
    const double d = (double)E::get(p[i]);
    sum[0] = fma(d, d, sum[0]);
  }
}

LCE_DEV double workgroup_sum(double v) {
  __shared__ double sh[kClipThreads / 64];
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  v = sh[0];
  for (int i = 1; i < kClipThreads / 64; ++i) v += sh[i];
  return v;
}

template <bool ONCE> __global__ __launch_bounds__(kClipThreads) void clip_norm_kernel(const ClipBatch b) {
  double sum[4] = {0.0, 0.0, 0.0, 0.0};
  for (unsigned c = blockIdx.x; c < b.stretches; c += gridDim.x) {
    const ClipEntry& e = b.e[entry_of(b, c)];
    const int64_t at = (int64_t)(c - e.first) * kStretch, left = e.n - at;
    const int n = left < kStretch ? (int)left : kStretch;
    const char* p = reinterpret_cast<const char*>(e.grad) + at * (e.dtype == DT_F32 ? 4 : 2);
    if (e.dtype == DT_BF16) add_squares<DT_BF16, ONCE>(p, n, sum);
    else if (e.dtype == DT_F16) add_squares<DT_F16, ONCE>(p, n, sum);
    else add_squares<DT_F32, ONCE>(p, n, sum);
  }
  const double all = workgroup_sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
  if (threadIdx.x == 0) b.part[b.part0 + blockIdx.x] = all;
}

// (16 bits to 32: 8 bytes of input to a lane, so that what a wave stores at a time lies together)
template <int DT, int OUT, bool ONCE> LCE_DEV void scale_stretch(const void* from, void* to, int n, float f) {
  typedef Elem<DT> E;
  typedef Elem<OUT> O;
  constexpr int kPer = O::kPer, kStep = kClipThreads * kPer, kRounds = 8;
  const typename E::S* p = reinterpret_cast<const typename E::S*>(from);
  typename O::S* q = reinterpret_cast<typename O::S*>(to);
  const int t = threadIdx.x;
  if (n == kStretch) {
    typedef u32x2_t __attribute__((aligned(2))) half_t;
#pragma unroll
    for (int r0 = 0; r0 < kStretch / kStep; r0 += kRounds) {
      constexpr int kHere = kStretch / kStep < kRounds ? kStretch / kStep : kRounds;
      u32x4_t v[kHere];
#pragma unroll
      for (int r = 0; r < kHere; ++r) {
        const typename E::S* at = p + (r0 + r) * kStep + t * kPer;
        if constexpr (E::kPer == kPer) {
          v[r] = load_piece<ONCE>(at);
        } else {
          const half_t* h = reinterpret_cast<const half_t*>(at);
          const u32x2_t w = ONCE ? __builtin_nontemporal_load(h) : *h;
          v[r] = u32x4_t{w[0], w[1], 0, 0};
        }
      }
#pragma unroll
      for (int r = 0; r < kHere; ++r) {
        typename E::S e[16 / sizeof(typename E::S)];
        typename O::S o[kPer];
        __builtin_memcpy(e, &v[r], 16);
#pragma unroll
        for (int i = 0; i < kPer; ++i) o[i] = O::put(E::get(e[i]) * f);
        u32x4_t w;
        __builtin_memcpy(&w, o, 16);
        store_piece<ONCE>(q + (r0 + r) * kStep + t * kPer, w);
      }
    }
    return;
  }
  for (int i = t; i < n; i += kClipThreads) q[i] = O::put(E::get(p[i]) * f);
}

template <bool ONCE>
__global__ __launch_bounds__(kClipThreads) void clip_scale_kernel(const ClipBatch b, int parts, float max_norm, float divisor, const float* divisor_ptr,
                                                                  float* norm_out) {
  double sum = 0.0;
  for (int i = threadIdx.x; i < parts; i += kClipThreads) sum += b.part[i];
  const double d = divisor_ptr != nullptr ? (double)*divisor_ptr : (double)divisor;
  const double norm = sqrt(workgroup_sum(sum)) / d;
  // (not finite, as the float32 number that the caller sees: nothing is clipped, and whoever reads the norm knows)
  const double f = (norm > (double)max_norm && (float)norm < INFINITY ? (double)max_norm / norm : 1.0) / d;
  const float factor = (float)f;
  if (norm_out != nullptr && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = (float)norm;
  // (from the last stretch to the first: those that the first launch read last are still in the Infinity Cache)
  for (unsigned i = blockIdx.x; i < b.stretches; i += gridDim.x) {
    const unsigned c = b.stretches - 1 - i;
    const ClipEntry& e = b.e[entry_of(b, c)];
    if (e.grad == e.out && factor == 1.f) continue;  // (of one type: nothing changes)
    const int64_t at = (int64_t)(c - e.first) * kStretch, left = e.n - at;
    const int n = left < kStretch ? (int)left : kStretch;
    const char* p = reinterpret_cast<const char*>(e.grad) + at * (e.dtype == DT_F32 ? 4 : 2);
    char* q = reinterpret_cast<char*>(e.out) + at * (e.out_dtype == DT_F32 ? 4 : 2);
    if (e.dtype == DT_F32) scale_stretch<DT_F32, DT_F32, ONCE>(p, q, n, factor);
    else if (e.dtype == DT_BF16 && e.out_dtype == DT_F32) scale_stretch<DT_BF16, DT_F32, ONCE>(p, q, n, factor);
    else if (e.dtype == DT_BF16) scale_stretch<DT_BF16, DT_BF16, ONCE>(p, q, n, factor);
    else if (e.out_dtype == DT_F32) scale_stretch<DT_F16, DT_F32, ONCE>(p, q, n, factor);
    else scale_stretch<DT_F16, DT_F16, ONCE>(p, q, n, factor);
  }
}

}  // namespace

int64_t clip_stretches(int64_t n) { return (n + kStretch - 1) / kStretch; }

hipError_t launch_clip_norm(const ClipBatch& b, int grid, hipStream_t s) {
  hipLaunchKernelGGL(b.once ? clip_norm_kernel<true> : clip_norm_kernel<false>, dim3(grid), dim3(kClipThreads), 0, s, b);
  return hipGetLastError();
}

hipError_t launch_clip_scale(const ClipBatch& b, int grid, int parts, float max_norm, float divisor, const float* divisor_ptr, float* norm,
                             hipStream_t s) {
  hipLaunchKernelGGL(b.once ? clip_scale_kernel<true> : clip_scale_kernel<false>, dim3(grid), dim3(kClipThreads), 0, s, b, parts, max_norm,
                     divisor, divisor_ptr, norm);
  return hipGetLastError();
}

}  // namespace lce

// Numbers of 8 bits with a scale for each row, and logits from them (lce_quantize_rows, lce_quantize_columns, lce_int8_logits).
//
//     t = q * scale,  scale = max |t| / 127,  q = the whole number nearest to 127 t / max |t|
//     logits[n][v] = logit_scale * sx[n] * sw[v] * sum_h qx[n][h] qw[v][h]
//
// The contraction is that of the loss's logit kernels (lce_gemm3.h, lce_gemm_small.h) with v_mfma_i32_32x32x32_i8 in the place of the 16-bit
// instruction: both take 16 bytes of K of each lane, so that an operand of 8-bit numbers is staged, swizzled and read as one of
// half as many 16-bit numbers, in the same time for twice the K.  Sums are exact in 32 bits (127^2 * 2^17 < 2^31).
#include "lce_gemm_small.h"
#include "lce_internal.h"

namespace lce {

typedef __attribute__((ext_vector_type(4))) int i32x4_t;
typedef __attribute__((ext_vector_type(16))) int i32x16_t;

struct I8 {};
template <> struct elem_of<I8> { typedef short type; };  // two numbers
template <> LCE_DEV f32x16_t mfma32<I8>(s16x8_t a, s16x8_t b, f32x16_t c) {
  return __builtin_bit_cast(f32x16_t, __builtin_amdgcn_mfma_i32_32x32x32_i8(__builtin_bit_cast(i32x4_t, a), __builtin_bit_cast(i32x4_t, b),
                                                                            __builtin_bit_cast(i32x16_t, c), 0, 0, 0));
}

namespace {

// 16 bytes at any 2-byte address: one load or store all the same.
struct __attribute__((packed, aligned(2))) Piece {
  u32x4_t v;
};

// ---------------------------------------------------------------------------
// Quantising
// ---------------------------------------------------------------------------
template <class S> LCE_DEV float number(S v);
template <> LCE_DEV float number<float>(float v) { return v; }
template <> LCE_DEV float number<__bf16>(__bf16 v) { return (float)v; }
template <> LCE_DEV float number<_Float16>(_Float16 v) { return (float)v; }

// What a row's numbers are multiplied by, from the largest magnitude among them as bits (of which NaN and infinity are the largest).
struct RowScale {
  float top, inverse;  // inverse: 127 / top, 0 for a row of zeros or one that is not finite
  float scale;
  bool tiny;           // 127 / top is no float32 number: the quotient is taken in doubles
  LCE_DEV explicit RowScale(unsigned bits) {
    const bool finite = bits < 0x7f800000u;
    top = __builtin_bit_cast(float, bits);
    tiny = top < 1e-30f && bits != 0;
    inverse = finite && bits != 0 && !tiny ? 127.f / top : 0.f;
    scale = finite ? (float)((double)top / 127.0) : __builtin_nanf("");
  }
};
// The whole number nearest to 127 v / top.  The product with the rounded inverse is off by less than 2^-15; within that of a border
// the two sides are compared as 127 |v| and (k + 1/2) top, which doubles hold exactly.
LCE_DEV int quantized(float v, const RowScale& r) {
  if (r.tiny) return (int)rint((double)v * 127.0 / (double)r.top);
  const float t = v * r.inverse;
  float q = __builtin_rintf(t);
  const float off = fabsf(t - q);
  if (off > 0.49996f && r.inverse != 0.f) {
    const float k = floorf(fabsf(t));
    const double a = 127.0 * (double)fabsf(v), b = ((double)k + 0.5) * (double)r.top;
    const float m = a > b || (a == b && ((int)k & 1)) ? k + 1.f : k;
    q = copysignf(m, t);
  }
  return (int)q;
}
LCE_DEV unsigned magnitude(float v) { return __builtin_bit_cast(unsigned, v) & 0x7fffffffu; }

constexpr int kQuantThreads = 256;
// Rows, one workgroup each.
template <class S>
__global__ __launch_bounds__(kQuantThreads) void quantize_rows_kernel(const S* src, int64_t rows, int cols, int64_t ld, signed char* q, int64_t ldq,
                                                                      float* scales) {
  __shared__ unsigned sh[kQuantThreads / 64];
  const int64_t r = blockIdx.x;
  const S* from = src + r * ld;
  unsigned top = 0;
  for (int c = threadIdx.x; c < cols; c += kQuantThreads) {
    const unsigned m = magnitude(number(from[c]));
    top = m > top ? m : top;
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const unsigned o = (unsigned)__shfl_xor((int)top, d);
    top = o > top ? o : top;
  }
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kQuantThreads / 64; ++i) top = sh[i] > top ? sh[i] : top;
  const RowScale s(top);
  if (threadIdx.x == 0) scales[r] = s.scale;
  for (int c = threadIdx.x; c < ldq; c += kQuantThreads) q[r * ldq + c] = c < cols && s.scale == s.scale ? (signed char)quantized(number(from[c]), s) : 0;
}

// Columns: a workgroup takes 64 of them, twice: for the largest magnitudes, then in tiles of 128 rows, which are turned in LDS.
constexpr int kColTile = 64, kRowTile = 128, kLineWords = kRowTile / 4 + 1;
template <class S>
__global__ __launch_bounds__(kQuantThreads) void quantize_columns_kernel(const S* src, int rows, int64_t cols, int64_t ld, signed char* q,
                                                                         int64_t ldq, float* scales) {
  __shared__ unsigned sh_top[kColTile];
  __shared__ unsigned sh_q[kColTile * kLineWords];
  const int t = threadIdx.x;
  const int64_t c0 = (int64_t)blockIdx.x * kColTile;
  const int width = cols - c0 < kColTile ? (int)(cols - c0) : kColTile;
  if (t < kColTile) sh_top[t] = 0;
  __syncthreads();
  const int c = t & (kColTile - 1);
  unsigned top = 0;
  if (c < width)
    for (int r = t / kColTile; r < rows; r += kQuantThreads / kColTile) {
      const unsigned m = magnitude(number(src[r * ld + c0 + c]));
      top = m > top ? m : top;
    }
  atomicMax(&sh_top[c], top);
  __syncthreads();
  const RowScale s(sh_top[c]);
  if (t < width) scales[c0 + t] = s.scale;
  for (int r0 = 0; r0 < ldq; r0 += kRowTile) {
    // four rows of one column to a thread at a time
    for (int i = t / kColTile; i < kRowTile / 4; i += kQuantThreads / kColTile) {
      unsigned w = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int r = r0 + 4 * i + k;
        const int n = c < width && r < rows && s.scale == s.scale ? quantized(number(src[r * ld + c0 + c]), s) : 0;
        w |= (unsigned)(n & 255) << (8 * k);
      }
      sh_q[c * kLineWords + i] = w;
    }
    __syncthreads();
    for (int i = t; i < kColTile * (kRowTile / 4); i += kQuantThreads) {
      const int line = i / (kRowTile / 4), word = i % (kRowTile / 4);
      if (line < width && r0 + 4 * word < ldq) *reinterpret_cast<unsigned*>(q + (c0 + line) * ldq + r0 + 4 * word) = sh_q[line * kLineWords + word];
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// The product
// ---------------------------------------------------------------------------
constexpr int kLineBytes = 128;                // of a row of out, per store
constexpr int kPieceBytes = kBlk * kLineBytes; // 32 rows
constexpr int kWaveLds = kPieceBytes;
constexpr int kLdsBytes = kMainloopLds + 4 * kWaveLds;

template <class T> struct out_of { static constexpr int kEs = 2; };
template <> struct out_of<float> { static constexpr int kEs = 4; };

// A wave's finished 128 (v) x 32 NQ (rows) sums: times the scales, rounded, and out in pieces of 32 rows x 128 bytes, which are
// turned into lines in the wave's own LDS (`mine`; the swizzle of the K-contiguous operand tiles, as for the staged dz).
template <class T, int NQ>
LCE_DEV void logits_epilogue(const Int8Args& a, f32x16_t (&acc)[kNB][NQ], int64_t v0, int64_t tw, char* mine) {
  constexpr int kEs = out_of<T>::kEs, kPerLine = kLineBytes / kEs, kBlocks = kPerLine / kBlk;  // blocks of 32 columns to a line
  const int lane = opaque_tid() & 63, half = lane >> 5;
  // (columns behind the last one: a scale of 0, and nothing is stored)
  const int64_t left = a.V - v0;
  const __amdgpu_buffer_rsrc_t scales = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<float*>(a.w_scales + v0), 0, left < 0 ? 0 : left > kWaveTile ? kWaveTile * 4 : (int)left * 4, 0x00020000);
  const int wline = lane & 31, wsw = (wline & 7) ^ ((wline >> 3) & 1);
  const int rline = (lane >> 3) + ((lane >> 5) ? 1 - 2 * ((lane >> 3) & 1) : 0), rchunk = lane & 7;
#pragma unroll
  for (int line = 0; line < kNB / kBlocks; ++line) {
    f32x4_t sw[kBlocks][4];
#pragma unroll
    for (int b = 0; b < kBlocks; ++b)
#pragma unroll
      for (int rq = 0; rq < 4; ++rq)
        sw[b][rq] = __builtin_bit_cast(f32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                                                    scales, ((line * kBlocks + b) * kBlk + rq * 8 + half * 4) * 4, 0, 0));
#pragma unroll
    for (int qb = 0; qb < NQ; ++qb) {
      const int64_t row = tw + qb * kBlk + (lane & 31);
      const float sx = row < a.N ? a.x_scales[row] * a.scale : 0.f;
#pragma unroll
      for (int b = 0; b < kBlocks; ++b) {
        const int pb = line * kBlocks + b;
        if constexpr (kEs == 4) {
#pragma unroll
          for (int rq = 0; rq < 4; ++rq) {
            u32x4_t o;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float s = acc[pb][qb][rq * 4 + i];
              o[i] = __builtin_bit_cast(unsigned, (float)__builtin_bit_cast(int, s) * sx * sw[b][rq][i]);
            }
            *reinterpret_cast<u32x4_t*>(mine + wline * kLineBytes + (((2 * rq + half) ^ wsw) << 4)) = o;
          }
        } else {
#pragma unroll
          for (int g = 0; g < 4; g += 2) {
            float d[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float s = acc[pb][qb][g * 4 + i];
              d[i] = (float)__builtin_bit_cast(int, s) * sx * sw[b][g + (i >> 2)][i & 3];
            }
            const auto s0 = __builtin_amdgcn_permlane32_swap(pack2<T>(d[0], d[1]), pack2<T>(d[4], d[5]), false, false);
            const auto s1 = __builtin_amdgcn_permlane32_swap(pack2<T>(d[2], d[3]), pack2<T>(d[6], d[7]), false, false);
            u32x4_t o;
            o[0] = s0[0];
            o[1] = s1[0];
            o[2] = s0[1];
            o[3] = s1[1];
            *reinterpret_cast<u32x4_t*>(mine + wline * kLineBytes + (((b * 4 + g + half) ^ wsw) << 4)) = o;
          }
        }
      }
      const int64_t v = v0 + line * kPerLine + rchunk * (16 / kEs);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int l = i * 8 + rline;
        const u32x4_t o = *reinterpret_cast<const u32x4_t*>(mine + l * kLineBytes + ((rchunk ^ (l & 7) ^ ((l >> 3) & 1)) << 4));
        const int64_t r = tw + qb * kBlk + l;
        if (r >= a.N) continue;
        char* to = reinterpret_cast<char*>(a.out) + (r * a.ldo + v) * kEs;
        if (v + 16 / kEs <= a.V) {
          reinterpret_cast<Piece*>(to)->v = o;
        } else {
          for (int k = 0; k < 16 / kEs; ++k)
            if (v + k < a.V) {
              if constexpr (kEs == 4) reinterpret_cast<unsigned*>(to)[k] = o[k];
              else reinterpret_cast<unsigned short*>(to)[k] = (unsigned short)(o[k >> 1] >> (16 * (k & 1)));
            }
        }
      }
    }
  }
}

// (of the last row no more is read than the 4 bytes that hold its last number; whatever lies behind a row's last one meets zeros)
LCE_DEV const signed char* weight_end(const Int8Args& a) { return a.w + (a.V - 1) * a.ldw + ((a.H + 3) & ~3); }

template <class T, bool KMASK> struct Int8Problem {
  typedef short E;
  static constexpr bool kKMask = KMASK;
  static constexpr bool kSwapAB = false;
  static constexpr bool kVarK = false;
  static constexpr bool kQBlocked = false;
  static constexpr bool kQScale = false;
  static constexpr bool kSplit = false;
  static constexpr bool kColumnEpilogue = false;
  const Int8Args& a;
  int tiles_p, tiles_q;
  LCE_DEV Int8Problem(const Int8Args& a_) : a(a_), tiles_p((int)((a_.V + kTile - 1) / kTile)), tiles_q((int)((a_.N + kTile - 1) / kTile)) {}
  LCE_DEV int64_t p_lo() const { return 0; }
  LCE_DEV int64_t q_lo() const { return 0; }
  LCE_DEV int num_tiles() const { return tiles_p * tiles_q; }
  LCE_DEV void coords(int tile, int& tp, int& tq) const { tile_coords(tile, num_tiles(), tiles_p, tiles_q, 8, a.live, tp, tq); }
  LCE_DEV void origins(int tile, const void*& p, const void*& q) const {
    int tp, tq;
    coords(tile, tp, tq);
    p = a.w + (int64_t)tp * kTile * a.ldw;
    q = a.x + (int64_t)tq * kTile * a.ldx;
  }
  LCE_DEV const void* p_end() const { return weight_end(a); }
  LCE_DEV const void* q_end() const { return a.x + (a.N - 1) * a.ldx + 2 * a.K2; }
  LCE_DEV int k_valid(int) const { return a.K2; }
  LCE_DEV void prefetch(int) {}
  LCE_DEV void epilogue(int tile, f32x16_t (&acc)[kNB][kNB], char* scratch) const {
    int tp, tq;
    coords(tile, tp, tq);
    const int wave = __builtin_amdgcn_readfirstlane(opaque_tid() >> 6);
    logits_epilogue<T, kNB>(a, acc, (int64_t)tp * kTile + (wave & 1) * kWaveTile, (int64_t)tq * kTile + (wave >> 1) * kWaveTile,
                            scratch + kStageBytes + wave * kWaveLds);
  }
};

template <class T, bool KMASK> __global__ __launch_bounds__(kThreads) void int8_logits_kernel(const Int8Args a) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  typedef Int8Problem<T, KMASK> Problem;
  Problem prob(a);
  Pipe3<I8, short, true, short, true, Problem> pipe(prob);
  pipe.run(a.ldw / 2, a.ldx / 2, (int)(padded_k(a.K2) / kBK), lds, (int)blockIdx.x);
}

// The same on 128 x 128 tiles, one workgroup each, for problems with few tiles.
static_assert(4 * kWaveLds <= kSmallLds, "the pieces fit where the stages were");
template <class T> __global__ __launch_bounds__(kThreads, 2) void int8_small_kernel(const Int8Args a, int tiles_p, int tiles_q) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  int tp, tq;
  tile_coords((int)blockIdx.x, (int)gridDim.x, tiles_p, tiles_q, 8, 8, tp, tq);
  SmallPipe<I8, true> pipe;
  f32x16_t acc[kNB][1];
  pipe.run(a.w + (int64_t)tp * kSmallTile * a.ldw, weight_end(a), a.ldw / 2, a.x + (int64_t)tq * kSmallTile * a.ldx,
           a.x + (a.N - 1) * a.ldx + 2 * a.K2, a.ldx / 2, a.K2, (int)small_logit_ktiles(a.K2, 1), 0, 0, lds, acc);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  logits_epilogue<T, 1>(a, acc, (int64_t)tp * kSmallTile, (int64_t)tq * kSmallTile + wave * kBlk, lds + wave * kWaveLds);
}

template <class T> hipError_t launch_product(const Int8Args& a, hipStream_t s) {
  if (few_logit_tiles(a.N, a.V, small_logit_ktiles(a.K2, 1), a.small_wgs)) {
    const int tiles_p = (int)((a.V + kSmallTile - 1) / kSmallTile), tiles_q = (int)((a.N + kSmallTile - 1) / kSmallTile);
    hipLaunchKernelGGL(int8_small_kernel<T>, dim3((unsigned)(tiles_p * tiles_q)), dim3(kThreads), kSmallLds, s, a, tiles_p, tiles_q);
    return hipGetLastError();
  }
  const int64_t tiles = (a.V + kTile - 1) / kTile * ((a.N + kTile - 1) / kTile);
  const dim3 grid((unsigned)(tiles < a.num_cus ? tiles : a.num_cus));
  if (padded_k(a.K2) == a.K2) {
    static LdsOptIn optin;
    const hipError_t e = optin.ensure(reinterpret_cast<const void*>(int8_logits_kernel<T, false>), kLdsBytes);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((int8_logits_kernel<T, false>), grid, dim3(kThreads), kLdsBytes, s, a);
  } else {
    static LdsOptIn optin;
    const hipError_t e = optin.ensure(reinterpret_cast<const void*>(int8_logits_kernel<T, true>), kLdsBytes);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((int8_logits_kernel<T, true>), grid, dim3(kThreads), kLdsBytes, s, a);
  }
  return hipGetLastError();
}

template <class S>
hipError_t quantize_rows(const void* src, int64_t rows, int64_t cols, int64_t ld, signed char* q, int64_t ldq, float* scales, hipStream_t s) {
  hipLaunchKernelGGL(quantize_rows_kernel<S>, dim3((unsigned)rows), dim3(kQuantThreads), 0, s, reinterpret_cast<const S*>(src), rows, (int)cols,
                     ld, q, ldq, scales);
  return hipGetLastError();
}
template <class S>
hipError_t quantize_columns(const void* src, int64_t rows, int64_t cols, int64_t ld, signed char* q, int64_t ldq, float* scales, hipStream_t s) {
  hipLaunchKernelGGL(quantize_columns_kernel<S>, dim3((unsigned)((cols + kColTile - 1) / kColTile)), dim3(kQuantThreads), 0, s,
                     reinterpret_cast<const S*>(src), (int)rows, cols, ld, q, ldq, scales);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_quantize_rows(const void* src, int dtype, int64_t rows, int64_t cols, int64_t ld, signed char* q, int64_t ldq, float* scales,
                                hipStream_t s) {
  return dtype == DT_BF16  ? quantize_rows<__bf16>(src, rows, cols, ld, q, ldq, scales, s)
         : dtype == DT_F16 ? quantize_rows<_Float16>(src, rows, cols, ld, q, ldq, scales, s)
                           : quantize_rows<float>(src, rows, cols, ld, q, ldq, scales, s);
}
hipError_t launch_quantize_columns(const void* src, int dtype, int64_t rows, int64_t cols, int64_t ld, signed char* q, int64_t ldq, float* scales,
                                   hipStream_t s) {
  return dtype == DT_BF16  ? quantize_columns<__bf16>(src, rows, cols, ld, q, ldq, scales, s)
         : dtype == DT_F16 ? quantize_columns<_Float16>(src, rows, cols, ld, q, ldq, scales, s)
                           : quantize_columns<float>(src, rows, cols, ld, q, ldq, scales, s);
}
hipError_t launch_int8_logits(const Int8Args& a, hipStream_t s) {
  return a.out_dtype == DT_BF16 ? launch_product<BF16>(a, s) : a.out_dtype == DT_F16 ? launch_product<F16>(a, s) : launch_product<float>(a, s);
}

}  // namespace lce

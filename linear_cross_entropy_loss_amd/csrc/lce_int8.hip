// Numbers of 8 bits with a scale for each row, and logits from them (lce_quantize_rows, lce_quantize_columns, lce_int8_logits).
//
//     t = q * scale,  scale = max |t| / 127,  q = the whole number nearest to 127 t / max |t|
//     logits[n][v] = logit_scale * sx[n] * sw[v] * sum_h qx[n][h] qw[v][h]
//
// The contraction is that of the loss's logit kernels (lce_gemm3.h, lce_gemm_small.h) with v_mfma_i32_32x32x32_i8 in the place of the 16-bit
// instruction: both take 16 bytes of K of each lane, so that an operand of 8-bit numbers is staged, swizzled and read as one of
// half as many 16-bit numbers, in the same time for twice the K.  Sums are exact in 32 bits (127^2 * 2^17 < 2^31).
// Bound by the matrix cores' power from some 500 rows on: 2048 rows of 4096 x 32000 in 236 us, 2.3 POP/s, the rate of a large library product of
// 8-bit numbers here (2.1 to 2.4), and less than twice that of 16-bit ones, whose K tiles take 1.2 us, not 1.9 (the clock is at 1.7 of 2.4 GHz
// then, the matrix cores busy for 66 % of it).  256 rows of 4096 x 128256, where weight and matrix cores ask for as much, 155 us: 1.7 POP/s beside
// 3.8 TB/s.  (A second set of registers for the weight's K tiles, two ahead, loses 5 %, the loads are not what it waits for; 128 x 128 tiles 186.)
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
// The same, of what is not read again.
LCE_DEV u32x4_t load_once(const void* p) {
  typedef u32x4_t __attribute__((aligned(2))) any_t;
  return __builtin_nontemporal_load(reinterpret_cast<const any_t*>(p));
}

// ---------------------------------------------------------------------------
// Quantising
// ---------------------------------------------------------------------------
// Elements as the kernels read them: 16 bytes at a time.
template <int DT> struct Source {
  static constexpr int kPer = 8;
  typedef unsigned short S;
  static LCE_DEV float get(S b) { return DT == DT_BF16 ? from_bits<BF16>(b) : from_bits<F16>(b); }
};
template <> struct Source<DT_F32> {
  static constexpr int kPer = 4;
  typedef float S;
  static LCE_DEV float get(S f) { return f; }
};
// The piece at column c of a row of `cols`, zeros behind its end.
template <int DT, bool ONCE = false> LCE_DEV u32x4_t load_piece(const typename Source<DT>::S* row, int c, int cols) {
  constexpr int kPer = Source<DT>::kPer;
  if (c + kPer <= cols) return ONCE ? load_once(row + c) : reinterpret_cast<const Piece*>(row + c)->v;
  if (c >= cols) return u32x4_t{0, 0, 0, 0};
  typename Source<DT>::S e[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) e[i] = c + i < cols ? row[c + i] : (typename Source<DT>::S)0;
  u32x4_t v;
  __builtin_memcpy(&v, e, 16);
  return v;
}
template <int DT> LCE_DEV void numbers(u32x4_t v, float (&f)[Source<DT>::kPer]) {
  typename Source<DT>::S e[Source<DT>::kPer];
  __builtin_memcpy(e, &v, 16);
#pragma unroll
  for (int i = 0; i < Source<DT>::kPer; ++i) f[i] = Source<DT>::get(e[i]);
}
// Element k of a piece (k need not be known to the compiler).
template <int DT> LCE_DEV float element(u32x4_t v, int k) {
  const int i = DT == DT_F32 ? k : k >> 1;
  const unsigned w = i == 0 ? v[0] : i == 1 ? v[1] : i == 2 ? v[2] : v[3];
  if constexpr (DT == DT_F32) return __builtin_bit_cast(float, w);
  else return Source<DT>::get((unsigned short)(w >> (16 * (k & 1))));
}
LCE_DEV unsigned larger(unsigned a, unsigned b) { return a > b ? a : b; }
// The largest magnitudes of pieces, element by element, as bits (of 16-bit types two to a word: their order is that of the numbers).
template <int DT> LCE_DEV u32x4_t larger_piece(u32x4_t a, u32x4_t v) {
  if constexpr (DT == DT_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) a[i] = larger(a[i], v[i] & 0x7fffffffu);
  } else {
    typedef __attribute__((ext_vector_type(2))) unsigned short u16x2_t;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned was = a[i], now = v[i] & 0x7fff7fffu;  // (a bit cast of a vector's element itself is one of its first)
      a[i] = __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(u16x2_t, was), __builtin_bit_cast(u16x2_t, now)));
    }
  }
  return a;
}
// One element's, as those of the float32 number.
template <int DT> LCE_DEV unsigned magnitude(u32x4_t v, int i) { return __builtin_bit_cast(unsigned, element<DT>(v, i)); }

// The scale of a row, from the largest magnitude among its numbers as bits (of which NaN and infinity are the largest).
struct RowScale {
  float top, scale;
  bool finite;
  LCE_DEV explicit RowScale(unsigned bits) {
    top = __builtin_bit_cast(float, bits);
    finite = bits < 0x7f800000u;
    scale = finite ? (float)((double)top / 127.0) : __builtin_nanf("");
  }
};
// The whole number nearest to 127 v / top, as the lowest byte of what byte_of returns: v times 127 / top, plus 3 * 2^22, whose last place
// is 1.
//
// 16-bit types.  127 v and top have at most 18 and 11 bits, so a quotient Q that is not half way between two whole numbers is at
// least Q * 2^-19 away from there, while the product with the rounded 127 / top is off by at most Q * 2^-23: rounded to 20 bits first it
// is on the half way exactly where Q is, and on Q's side of it elsewhere.  (In bf16 every thousandth number is half its row's largest, which
// is 63.5.)
//
// float32.  The product with a float below 127 / top and with one above, each rounded once: where both give the same, so does the
// quotient; where they do not, one number in 10^5, `differ` is not 0 afterwards and exact_byte decides.
//
// Rows whose 127 / top is no ordinary number have 0 for both (a row of zeros), or go by exact_byte altogether (`odd`).
struct Inverse {
  float near, below, above;
  bool odd;
  LCE_DEV Inverse() {}
  LCE_DEV explicit Inverse(const RowScale& r) {
    odd = !r.finite || (r.top < 1e-30f && r.top > 0.f);
    near = odd || r.top == 0.f ? 0.f : 127.f / r.top;
    const unsigned bits = __builtin_bit_cast(unsigned, near);
    below = near == 0.f ? 0.f : __builtin_bit_cast(float, bits - 1);
    above = near == 0.f ? 0.f : __builtin_bit_cast(float, bits + 1);
  }
};
constexpr float kWhole = 12582912.f;
template <int DT> LCE_DEV unsigned byte_of(float v, const Inverse& i, unsigned& differ) {
  if constexpr (DT == DT_F32) {
    const unsigned a = __builtin_bit_cast(unsigned, fmaf(v, i.below, kWhole));
    const unsigned b = __builtin_bit_cast(unsigned, fmaf(v, i.above, kWhole));
    differ |= a ^ b;
    return a;
  } else {
    const unsigned t = __builtin_bit_cast(unsigned, v * i.near);
    return __builtin_bit_cast(unsigned, __builtin_bit_cast(float, (t + 8) & ~15u) + kWhole);
  }
}
// By comparing 127 |v| with (k + 1/2) top, which doubles hold exactly.
LCE_DEV unsigned exact_byte(float v, const RowScale& r) {
  if (!r.finite) return 0u;
  if (r.top < 1e-30f) return r.top > 0.f ? (unsigned)(int)rint((double)v * 127.0 / (double)r.top) : 0u;
  const float t = fabsf(v) * (127.f / r.top), k = floorf(t);
  if (fabsf(t - k - 0.5f) > 0.01f) return (unsigned)(int)copysignf(rintf(t), v);
  const double a = 127.0 * (double)fabsf(v), b = ((double)k + 0.5) * (double)r.top;
  return (unsigned)(int)copysignf(a > b || (a == b && ((int)k & 1)) ? k + 1.f : k, v);
}
// The lowest bytes of four, in their order.
LCE_DEV unsigned four_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
  const unsigned lo = __builtin_amdgcn_perm(b, a, 0x0c0c0400u), hi = __builtin_amdgcn_perm(d, c, 0x0c0c0400u);
  return lo | hi << 16;
}

// Rows.  WAVES waves to a row (one, of four rows to a workgroup, where that holds the row in registers and there are many; else
// a workgroup), or LANES lanes of a wave where it is short; a row of up to LANES * WAVES * PIECES pieces is read once, a longer one twice.
// 131072 x 2048 bf16 136 us, 5.9 TB/s; 200000 x 256 by 16 lanes 30 us, 5.1 TB/s, by 64 92; 65133 x 672 fp16 29 and 40.  (The piece that a row's end cuts
// as the row's last 16 bytes, shifted, not element by element: 5 % more.)
constexpr int kQuantThreads = 256;
template <int DT> LCE_DEV void store_bytes(u32x4_t piece, const RowScale& s, const Inverse& inverse, signed char* to) {
  constexpr int kPer = Source<DT>::kPer;
  float f[kPer];
  numbers<DT>(piece, f);
  unsigned b[kPer], differ = inverse.odd;
#pragma unroll
  for (int i = 0; i < kPer; ++i) b[i] = byte_of<DT>(f[i], inverse, differ);
  if (differ == 0) {
#pragma unroll
    for (int i = 0; i < kPer; i += 4) reinterpret_cast<unsigned*>(to)[i / 4] = four_bytes(b[i], b[i + 1], b[i + 2], b[i + 3]);
  } else {
#pragma unroll 1
    for (int i = 0; i < kPer; ++i) to[i] = (signed char)exact_byte(element<DT>(piece, i), s);
  }
}
template <int DT, int WAVES, int PIECES, int LANES = 64>
__global__ __launch_bounds__(kQuantThreads) void quantize_rows_kernel(const void* src, int64_t rows, int cols, int64_t ld, signed char* q, int ldq,
                                                                      float* scales) {
  typedef Source<DT> E;
  static_assert(WAVES == 1 || LANES == 64, "lanes of one wave, or whole waves");
  constexpr int kStep = LANES * WAVES * E::kPer;
  __shared__ unsigned sh[kQuantThreads / 64];
  const int wave = threadIdx.x >> 6;
  const int64_t r = WAVES == 1 ? (int64_t)blockIdx.x * (kQuantThreads / LANES) + threadIdx.x / LANES : (int64_t)blockIdx.x;
  if (r >= rows) return;
  const int t = WAVES == 1 ? threadIdx.x & (LANES - 1) : threadIdx.x;
  const typename E::S* from = reinterpret_cast<const typename E::S*>(src) + r * ld;
  const bool once = cols <= kStep * PIECES;
  u32x4_t v[PIECES], tops = {0, 0, 0, 0};
  for (int c0 = 0; c0 < cols; c0 += kStep * PIECES) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i) v[i] = load_piece<DT, WAVES == 1>(from, c0 + i * kStep + t * E::kPer, cols);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) tops = larger_piece<DT>(tops, v[i]);
  }
  unsigned top = 0;
#pragma unroll
  for (int k = 0; k < E::kPer; ++k) top = larger(top, magnitude<DT>(tops, k));
#pragma unroll
  for (int d = 1; d < LANES; d <<= 1) top = larger(top, (unsigned)__shfl_xor((int)top, d));
  if constexpr (WAVES > 1) {
    if ((threadIdx.x & 63) == 0) sh[wave] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < WAVES; ++i) top = larger(top, sh[i]);
  }
  const RowScale s(top);
  const Inverse inverse(s);
  if (t == 0) scales[r] = s.scale;
  signed char* to = q + r * ldq;
  for (int c0 = 0; c0 < ldq; c0 += kStep * PIECES)
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int c = c0 + i * kStep + t * E::kPer;
      // (behind what is held there are zeros only, as far as a wide ldq reaches)
      if (c < ldq) store_bytes<DT>(once && c0 == 0 ? v[i] : load_piece<DT>(from, c, cols), s, inverse, to + c);
    }
}

// Columns.  A workgroup of NT threads takes stripes of COLS of them, one after another.  It holds a stripe in registers -- kTiles * 4 pieces
// to a thread -- until the largest magnitudes are known, and turns it in LDS, a tile of rows at a time, four rows of a piece to a
// thread, so that q is written in stretches of 128 bytes and more; a tile's registers take the next stripe's as soon as it is in LDS.
// The weight is read once.  Two neighbouring stripes, which may share lines, go to one XCD.
// Bound by memory, 2048 x 131072 bf16 in 172 us, 4.7 TB/s read and written (the same without the quantising itself; reading alone 126).  Reading
// the weight twice, an element to a load, took 625; twice with 16 bytes 300; held, without the next stripe under way, 204.
constexpr int kTiles = 4;
template <int DT, int NT, int COLS, bool ONCE>
__global__ __launch_bounds__(NT, 4) void quantize_held_columns_kernel(const void* src, int rows, int64_t cols, int64_t ld, signed char* q, int ldq,
                                                                      float* scales) {
  typedef Source<DT> E;
  constexpr int kPer = E::kPer, kPieces = COLS / kPer, kQuads = NT / kPieces;  // fours of rows in a tile
  constexpr int kWords = kQuads + 2;  // of a line in LDS: the lanes of a wave write to different banks
  __shared__ unsigned sh_top[COLS];
  __shared__ Inverse sh_inverse[COLS];
  __shared__ unsigned sh_q[2][COLS * kWords];
  const int t = threadIdx.x, c = t % kPieces * kPer, quad = t / kPieces;
  // (the last stripe ends with the last column: some columns are then done twice, alike)
  const auto place = [&](int id) { return (((int64_t)(id >> 4) * 8 + (id & 7)) * 2 + (id >> 3 & 1)) * COLS; };
  const auto stripe = [&](int id) { return place(id) < cols - COLS ? place(id) : cols - COLS; };
  u32x4_t v[kTiles][4];
  const unsigned mine = (unsigned)(((int64_t)quad * 4 * ld + c) * (int64_t)sizeof(typename E::S));  // of a thread in a tile: 32 bits
  const auto load_tile = [&](int64_t c0, int u) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int r = u * kQuads * 4 + j;  // (uniform)
      const char* from = reinterpret_cast<const char*>(reinterpret_cast<const typename E::S*>(src) + c0 + (int64_t)r * ld);
      v[u][j] = u32x4_t{0, 0, 0, 0};
      if (r + quad * 4 < rows) v[u][j] = ONCE ? load_once(from + mine) : reinterpret_cast<const Piece*>(from + mine)->v;
    }
  };
  int id = blockIdx.x;
  if (place(id) >= cols) return;
  int64_t c0 = stripe(id);
#pragma unroll
  for (int u = 0; u < kTiles; ++u) load_tile(c0, u);
  for (bool more = true; more; id += gridDim.x) {
    more = place(id + (int)gridDim.x) < cols;  // (a workgroup's stripes come from left to right)
    const int64_t next = more ? stripe(id + (int)gridDim.x) : 0;
    if (t < COLS) sh_top[t] = 0;
    __syncthreads();
    u32x4_t tops = {0, 0, 0, 0};
#pragma unroll
    for (int u = 0; u < kTiles; ++u)
#pragma unroll
      for (int j = 0; j < 4; ++j) tops = larger_piece<DT>(tops, v[u][j]);
#pragma unroll
    for (int d = kPieces; d < 64; d <<= 1) {
      u32x4_t o;
#pragma unroll
      for (int i = 0; i < 4; ++i) o[i] = (unsigned)__shfl_xor((int)tops[i], d);
      tops = larger_piece<DT>(tops, o);
    }
    if ((t & 63) < kPieces) {
#pragma unroll
      for (int k = 0; k < kPer; ++k) atomicMax(&sh_top[c + k], magnitude<DT>(tops, k));
    }
    __syncthreads();
    if (t < COLS) {
      const RowScale s(sh_top[t]);
      sh_inverse[t] = Inverse(s);
      scales[c0 + t] = s.scale;
    }
    __syncthreads();
    Inverse inverse[kPer];
    bool odd = false;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      inverse[k] = sh_inverse[c + k];
      odd |= inverse[k].odd;
    }
#pragma unroll
    for (int u = 0; u < kTiles; ++u) {
      const int r0 = u * kQuads * 4;
      if (r0 >= ldq) break;
      unsigned* tile = sh_q[u & 1];
      unsigned differ = odd;
#pragma unroll
      for (int j = 0; j < 4; ++j) asm volatile("" : "+v"(v[u][j]));  // (or the compiler keeps the numbers of all tiles, in twice the registers)
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        unsigned b[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j] = byte_of<DT>(element<DT>(v[u][j], k), inverse[k], differ);
        tile[(c + k) * kWords + quad] = four_bytes(b[0], b[1], b[2], b[3]);
      }
      if (differ != 0) {
#pragma unroll 1
        for (int k = 0; k < kPer; ++k) {  // (rare)
          const RowScale s(sh_top[c + k]);
          unsigned b[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) b[j] = exact_byte(element<DT>(v[u][j], k), s);
          tile[(c + k) * kWords + quad] = four_bytes(b[0], b[1], b[2], b[3]);
        }
      }
      if (more) load_tile(next, u);
      __syncthreads();  // (the one of the next tile parts this tile's readers from the writers of the one after it)
      // 32 bytes of a line to a thread
      for (int line = t / (kQuads / 8); line < COLS; line += NT / (kQuads / 8)) {
        const int part = t % (kQuads / 8) * 8;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          u32x4_t o;
#pragma unroll
          for (int i = 0; i < 4; ++i) o[i] = tile[line * kWords + part + h * 4 + i];
          const int at = r0 + (part + h * 4) * 4;
          if (at < ldq) *reinterpret_cast<u32x4_t*>(q + (c0 + line) * ldq + at) = o;
        }
      }
    }
    c0 = next;
  }
}

// The same for columns that the registers do not hold: a stripe of 64 is read twice, for the largest magnitudes and then in tiles of
// 128 rows.
constexpr int kColTile = 64, kRowTile = 128, kLineWords = kRowTile / 4 + 1;
template <int DT>
__global__ __launch_bounds__(kQuantThreads) void quantize_columns_kernel(const void* src, int rows, int64_t cols, int64_t ld, signed char* q, int ldq,
                                                                         float* scales) {
  typedef Source<DT> E;
  constexpr int kPer = E::kPer, kPieces = kColTile / kPer, kRowsAtOnce = kQuantThreads / kPieces;  // pieces of a row of the stripe
  constexpr int kTurns = kRowTile / 4 / kRowsAtOnce;                                              // of four rows, to a tile
  __shared__ unsigned sh_top[kColTile];
  __shared__ Inverse sh_inverse[kColTile];
  __shared__ unsigned sh_q[kColTile * kLineWords];
  const int t = threadIdx.x;
  const int64_t c0 = (int64_t)blockIdx.x * kColTile;
  const int width = cols - c0 < kColTile ? (int)(cols - c0) : kColTile;
  const typename E::S* from = reinterpret_cast<const typename E::S*>(src) + c0;
  if (t < kColTile) sh_top[t] = 0;
  __syncthreads();
  const int c = t % kPieces * kPer, r1 = t / kPieces;
  u32x4_t tops = {0, 0, 0, 0};
  constexpr int kFlight = 8;
  if (c < width)
    for (int r0 = r1; r0 < rows; r0 += kFlight * kRowsAtOnce) {
      u32x4_t v[kFlight];
#pragma unroll
      for (int i = 0; i < kFlight; ++i) {
        const int r = r0 + i * kRowsAtOnce;
        v[i] = load_piece<DT>(from + (int64_t)(r < rows ? r : r0) * ld, c, width);
      }
#pragma unroll
      for (int i = 0; i < kFlight; ++i) tops = larger_piece<DT>(tops, v[i]);
    }
#pragma unroll
  for (int k = 0; k < kPer; ++k) atomicMax(&sh_top[c + k], magnitude<DT>(tops, k));
  __syncthreads();
  if (t < kColTile) {
    const RowScale s(sh_top[t]);
    sh_inverse[t] = Inverse(s);
    if (t < width) scales[c0 + t] = s.scale;
  }
  __syncthreads();
  Inverse inverse[kPer];
  bool odd = false;
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    inverse[k] = sh_inverse[c + k];
    odd |= inverse[k].odd;
  }
  u32x4_t v[kTurns][4];
  const auto load_tile = [&](int r0) {
#pragma unroll
    for (int i = 0; i < kTurns; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = r0 + 4 * (i * kRowsAtOnce + r1) + j;
        v[i][j] = c < width && r < rows ? load_piece<DT>(from + (int64_t)r * ld, c, width) : u32x4_t{0, 0, 0, 0};
      }
  };
  load_tile(0);
  for (int r0 = 0; r0 < ldq; r0 += kRowTile) {
#pragma unroll
    for (int i = 0; i < kTurns; ++i) {
      float f[4][kPer];
#pragma unroll
      for (int j = 0; j < 4; ++j) numbers<DT>(v[i][j], f[j]);
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        unsigned b[4], differ = odd;
#pragma unroll
        for (int j = 0; j < 4; ++j) b[j] = byte_of<DT>(f[j][k], inverse[k], differ);
        if (differ != 0) {
          const RowScale s(sh_top[c + k]);
#pragma unroll
          for (int j = 0; j < 4; ++j) b[j] = exact_byte(f[j][k], s);
        }
        sh_q[(c + k) * kLineWords + i * kRowsAtOnce + r1] = four_bytes(b[0], b[1], b[2], b[3]);
      }
    }
    if (r0 + kRowTile < ldq) load_tile(r0 + kRowTile);
    __syncthreads();
    // 32 bytes of a line to a thread
    const int line = t >> 2, part = (t & 3) * 8;
    if (line < width) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        u32x4_t o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = sh_q[line * kLineWords + part + h * 4 + i];
        const int at = r0 + (part + h * 4) * 4;
        if (at < ldq) *reinterpret_cast<u32x4_t*>(q + (c0 + line) * ldq + at) = o;
      }
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

// The weight streams past the rows of x, which should stay in L2: 256 rows of 4096 x 128256 166 to 155 us, of 2048 x 131072 90 to 84, 2048 of
// 4096 x 32000 1 %.
constexpr int kWeightAux = 2;
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
  Pipe3<I8, short, true, short, true, Problem, kWeightAux> pipe(prob);
  pipe.run(a.ldw / 2, a.ldx / 2, (int)(padded_k(a.K2) / kBK), lds, (int)blockIdx.x);
}

// The same on 128 x 128 tiles, one workgroup each, for problems with few tiles.
static_assert(4 * kWaveLds <= kSmallLds, "the pieces fit where the stages were");
template <class T, int AUX> __global__ __launch_bounds__(kThreads, 2) void int8_small_kernel(const Int8Args a, int tiles_p, int tiles_q) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  int tp, tq;
  tile_coords((int)blockIdx.x, (int)gridDim.x, tiles_p, tiles_q, 8, 8, tp, tq);
  SmallPipe<I8, true, true, false, 4, 1, false, false, AUX> pipe;
  f32x16_t acc[kNB][1];
  pipe.run(a.w + (int64_t)tp * kSmallTile * a.ldw, weight_end(a), a.ldw / 2, a.x + (int64_t)tq * kSmallTile * a.ldx,
           a.x + (a.N - 1) * a.ldx + 2 * a.K2, a.ldx / 2, a.K2, (int)small_logit_ktiles(a.K2, 1), 0, 0, lds, acc);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  logits_epilogue<T, 1>(a, acc, (int64_t)tp * kSmallTile, (int64_t)tq * kSmallTile + wave * kBlk, lds + wave * kWaveLds);
}

// ---------------------------------------------------------------------------
// Few rows: a pass over the weight.  A wave takes 16 rows of it at a time, straight from memory to the registers that
// v_mfma_i32_16x16x64_i8 reads (lane l: row l % 16, 16 bytes of K at 16 * (l / 16) of every 64), a group of kFlight loads ahead of the one
// that is multiplied, across the ends of its rows too; the quantised rows of x lie in LDS in the order in which the lanes want them:
// 16 bytes of K, row after row.  There are 1, 2, 4, 8 or 16 places for rows; lanes beyond the places read the same rows again, and
// nobody stores what comes of it.
// One or two short rows (kFusedRows, kFusedNumbers) are quantised by every workgroup for itself while its first loads of the weight are under
// way: one row of 2048 in 3 us less than a launch takes.  (More rows, which it takes one after another: 8 of 2048 5 us more than the
// launch, 16 of 256 13.)
// Bound by the weight's way from memory.  us, x quantised too, against the 128 x 128 tiles: 2048 x 131072 one row 47 / 52, 4096 x 128256 95 / 105,
// 8192 x 32000 52 / 63; with x quantised before, 8 rows of 2048 x 131072 53 / 49, 4096 x 128256 104 / 102, 8192 x 32000 57 / 63.
// Four loads in a group 50, 106 and 64 us for one row, twelve 55, 110 and 59; loads past the caches 53, 107 and 59 (half a line at a time).
// ---------------------------------------------------------------------------
constexpr int kStreamThreads = 512, kFlight = 8, kGroupBytes = 64 * kFlight;
constexpr int kStreamLds = 150 * 1024, kStreamRows = 16;
constexpr int64_t kFusedRows = 2, kFusedNumbers = 16384;
LCE_DEV u32x4_t* place_of(char* lds, int byte, int n, int places) {
  return reinterpret_cast<u32x4_t*>(lds + ((byte >> 4) * places + n) * 16 + (byte & 15));
}
template <int DT> LCE_DEV void quantize_into(const Int8Args& a, char* lds, int places, int depth, unsigned* sh_top, float* sh_scale, Inverse* sh_inverse) {
  typedef Source<DT> E;
  const int N = (int)a.N, t = threadIdx.x;
  for (int n = 0; n < N; ++n) {
    const typename E::S* row = reinterpret_cast<const typename E::S*>(a.x_in) + n * a.ldx_in;
    u32x4_t tops = {0, 0, 0, 0};
    for (int c = t * E::kPer; c < a.H; c += kStreamThreads * E::kPer) tops = larger_piece<DT>(tops, load_piece<DT>(row, c, a.H));
    unsigned top = 0;
#pragma unroll
    for (int k = 0; k < E::kPer; ++k) top = larger(top, magnitude<DT>(tops, k));
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = larger(top, (unsigned)__shfl_xor((int)top, d));
    if ((t & 63) == 0) atomicMax(&sh_top[n], top);
  }
  __syncthreads();
  if (t < N) {
    const RowScale s(sh_top[t]);
    sh_scale[t] = s.scale * a.scale;
    sh_inverse[t] = Inverse(s);
  }
  __syncthreads();
  for (int n = 0; n < N; ++n) {
    const typename E::S* row = reinterpret_cast<const typename E::S*>(a.x_in) + n * a.ldx_in;
    const Inverse inverse = sh_inverse[n];
    for (int c = t * E::kPer; c < depth; c += kStreamThreads * E::kPer) {
      const u32x4_t piece = load_piece<DT>(row, c, a.H);
      store_bytes<DT>(piece, RowScale(sh_top[n]), inverse, reinterpret_cast<signed char*>(place_of(lds, c, n, places)));
    }
  }
}
template <class T> __global__ __launch_bounds__(kStreamThreads, 4) void int8_stream_kernel(const Int8Args a, int places, int depth) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  __shared__ float sh_scale[kStreamRows];
  __shared__ unsigned sh_top[kStreamRows];
  __shared__ Inverse sh_inverse[kStreamRows];
  const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int blocks = (int)((a.V + 15) / 16), step = (int)gridDim.x * (kStreamThreads / 64);
  const int groups = depth / kGroupBytes;
  int block = wave * (int)gridDim.x + (int)blockIdx.x;  // (the last ones go to different compute units)
  const unsigned mine = (unsigned)((lane & 15) * a.ldw + (lane >> 4) * 16);
  const char* const end = reinterpret_cast<const char*>(weight_end(a));
  u32x4_t w[2][kFlight];
  // (of the last row nothing is read past its end; what is read of the next row behind the end of one meets zeros)
  const auto load = [&](int buf, int b, int g) {
    const char* base = reinterpret_cast<const char*>(a.w) + (int64_t)b * 16 * a.ldw + g * kGroupBytes;
    const int64_t left = end - base;
    const __amdgpu_buffer_rsrc_t rsrc =
        __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base), 0, left <= 0 ? 0 : left > 0x7fffffff ? 0x7fffffff : (int)left, 0x00020000);
#pragma unroll
    for (int i = 0; i < kFlight; ++i) w[buf][i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, (int)mine + i * 64, 0, 0);
  };
  if (block < blocks) load(0, block, 0);
  if (t < kStreamRows) sh_top[t] = 0;
  __syncthreads();
  if (a.x_in != nullptr) {
    if (a.x_in_dtype == DT_BF16) quantize_into<DT_BF16>(a, lds, places, depth, sh_top, sh_scale, sh_inverse);
    else if (a.x_in_dtype == DT_F16) quantize_into<DT_F16>(a, lds, places, depth, sh_top, sh_scale, sh_inverse);
    else quantize_into<DT_F32>(a, lds, places, depth, sh_top, sh_scale, sh_inverse);
  } else {
    if (t < a.N) sh_scale[t] = a.x_scales[t] * a.scale;
    const int pieces = depth / 16;
    for (int i = t; i < pieces * (int)a.N; i += kStreamThreads) {
      const int n = i / pieces, c = (i - n * pieces) * 16;
      *place_of(lds, c, n, places) = c < 2 * a.K2 ? *reinterpret_cast<const u32x4_t*>(a.x + n * a.ldx + c) : u32x4_t{0, 0, 0, 0};
    }
  }
  __syncthreads();
  const int n = lane & 15, row = n & (places - 1);
  const char* const from = lds + ((lane >> 4) * places + row) * 16;
  i32x4_t acc;
  const auto multiply = [&](int buf, int g) {
#pragma unroll
    for (int i = 0; i < kFlight; ++i) {
      const i32x4_t x = *reinterpret_cast<const i32x4_t*>(from + (g * kFlight + i) * (64 * places));
      acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(__builtin_bit_cast(i32x4_t, w[buf][i]), x, acc, 0, 0, 0);
    }
  };
  // One block of rows, whose first group is in buffer FIRST; the next one's is in the other buffer afterwards where the groups are odd.
  const auto rows16 = [&](auto first, int next) {
    constexpr int F = decltype(first)::value;
    acc = i32x4_t{0, 0, 0, 0};
    int g = 0;
    for (; g + 1 < groups; g += 2) {
      load(1 - F, block, g + 1);
      multiply(F, g);
      if (g + 2 < groups) load(F, block, g + 2);
      else if (next < blocks) load(F, next, 0);
      multiply(1 - F, g + 1);
    }
    if (g < groups) {
      if (next < blocks) load(1 - F, next, 0);
      multiply(F, g);
    }
    // lane: rows 4 * (lane / 16) ... + 3 of the weight's, row `n` of x
    const int64_t v = (int64_t)block * 16 + (lane >> 4) * 4;
    if (n < a.N) {
      const float sx = sh_scale[n];
      char* to = reinterpret_cast<char*>(a.out) + (n * a.ldo + v) * out_of<T>::kEs;
      float f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = (float)acc[i] * sx * (v + i < a.V ? a.w_scales[v + i] : 0.f);
      if constexpr (out_of<T>::kEs == 4) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (v + i < a.V) reinterpret_cast<float*>(to)[i] = f[i];
      } else if (v + 4 <= a.V && (reinterpret_cast<uintptr_t>(to) & 7) == 0) {
        *reinterpret_cast<u32x2_t*>(to) = u32x2_t{pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3])};
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (v + i < a.V) reinterpret_cast<unsigned short*>(to)[i] = to_bits<T>(f[i]);
      }
    }
  };
  const bool odd = (groups & 1) != 0;
  for (; block < blocks; block += step) {
    rows16(std::integral_constant<int, 0>(), block + step);
    if (odd && (block += step) < blocks) rows16(std::integral_constant<int, 1>(), block + step);
  }
}

// Whether the kernel takes the problem: one or two rows that it quantises itself, or a few long ones (see above; at 4096 the two are even).
constexpr int kStreamDepth = 6144;
bool fuses(const Int8Args& a) { return a.N <= kFusedRows && a.N * a.H <= kFusedNumbers; }
bool streams(const Int8Args& a, int* places, int* depth) {
  *depth = (int)pad_to(a.H, kGroupBytes);
  *places = 1;
  while (*places < a.N && *places < 2 * kStreamRows) *places *= 2;
  return *places <= kStreamRows && (int64_t)*places * *depth <= kStreamLds && (fuses(a) || *depth >= kStreamDepth);
}
template <class T> hipError_t launch_stream(const Int8Args& a, int places, int depth, hipStream_t s) {
  static LdsOptIn optin;
  const hipError_t e = optin.ensure(reinterpret_cast<const void*>(int8_stream_kernel<T>), kStreamLds);
  if (e != hipSuccess) return e;
  const int bytes = places * depth, per = bytes <= kStreamLds / 2 ? 2 : 1;
  const int64_t groups = ((a.V + 15) / 16 + kStreamThreads / 64 - 1) / (kStreamThreads / 64);
  const int64_t most = (int64_t)a.num_cus * per;
  hipLaunchKernelGGL(int8_stream_kernel<T>, dim3((unsigned)(groups < most ? groups : most)), dim3(kStreamThreads), bytes, s, a, places, depth);
  return hipGetLastError();
}

template <class T> hipError_t launch_product(const Int8Args& a, hipStream_t s) {
  int places, depth;
  if (streams(a, &places, &depth)) return launch_stream<T>(a, places, depth, s);
  if (few_logit_tiles(a.N, a.V, small_logit_ktiles(a.K2, 1), a.small_wgs)) {
    const int tiles_p = (int)((a.V + kSmallTile - 1) / kSmallTile), tiles_q = (int)((a.N + kSmallTile - 1) / kSmallTile);
    // (a single row of tiles: nobody reads a tile of the weight again.  37 rows of 4096 x 128256 121 to 112 us; but 192 of 8192 x 32000 85 to 107)
    hipLaunchKernelGGL((tiles_q == 1 ? int8_small_kernel<T, kWeightAux> : int8_small_kernel<T, 0>), dim3((unsigned)(tiles_p * tiles_q)), dim3(kThreads),
                       kSmallLds, s, a, tiles_p, tiles_q);
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

// Workgroups of one launch, which has fewer than 2^32 threads: more rows or columns take several, one after another.
constexpr int64_t kMostGroups = (int64_t)1 << 22;

template <int DT>
hipError_t quantize_rows(const void* src, int64_t rows, int64_t cols, int64_t ld, signed char* q, int64_t ldq, float* scales, hipStream_t s) {
  constexpr int kPer = Source<DT>::kPer;
  // (`per` rows to a workgroup)
  const auto go = [&](auto kernel, int64_t per) {
    for (int64_t r = 0; r < rows; r += kMostGroups * per) {
      const int64_t n = rows - r < kMostGroups * per ? rows - r : kMostGroups * per;
      hipLaunchKernelGGL(kernel, dim3((unsigned)((n + per - 1) / per)), dim3(kQuantThreads), 0, s,
                         reinterpret_cast<const typename Source<DT>::S*>(src) + r * ld, n, (int)cols, ld, q + r * ldq, (int)ldq, scales + r);
      const hipError_t e = hipGetLastError();
      if (e != hipSuccess) return e;
    }
    return hipSuccess;
  };
  if (rows < 1024 || cols > 64 * kPer * 8) return go(quantize_rows_kernel<DT, 4, 32 / kPer>, 1);
  if (cols > 64 * kPer * 4) return go(quantize_rows_kernel<DT, 1, 8>, 4);
  if (cols > 64 * kPer * 2) return go(quantize_rows_kernel<DT, 1, 4>, 4);
  if (cols > 16 * kPer * 4) return go(quantize_rows_kernel<DT, 1, 8, 16>, 16);
  if (cols > 16 * kPer * 2) return go(quantize_rows_kernel<DT, 1, 4, 16>, 16);
  return go(quantize_rows_kernel<DT, 1, 2, 16>, 16);
}
template <int DT, int NT, int COLS>
hipError_t quantize_held_columns(const void* src, int64_t rows, int64_t cols, int64_t ld, signed char* q, int64_t ldq, float* scales, int num_cus,
                                 hipStream_t s) {
  const int64_t stripes = pad_to((cols + COLS - 1) / COLS, 16);
  const int64_t most = pad_to((int64_t)num_cus * (1024 / NT), 16);  // (as many workgroups as the compute units hold at a time)
  const dim3 grid((unsigned)(stripes < most ? stripes : most));
  // (past the caches where no two stripes share a line: 2048 x 131072 bf16 192 us, so 168; but 768 x 50257, whose stripes do, 31 and 39)
  constexpr int kEs = DT == DT_F32 ? 4 : 2;
  if (COLS * kEs % 128 == 0 && ld * kEs % 128 == 0 && reinterpret_cast<uintptr_t>(src) % 128 == 0)
    hipLaunchKernelGGL((quantize_held_columns_kernel<DT, NT, COLS, true>), grid, dim3(NT), 0, s, src, (int)rows, cols, ld, q, (int)ldq, scales);
  else
    hipLaunchKernelGGL((quantize_held_columns_kernel<DT, NT, COLS, false>), grid, dim3(NT), 0, s, src, (int)rows, cols, ld, q, (int)ldq, scales);
  return hipGetLastError();
}
template <int DT>
hipError_t quantize_columns(const void* src, int64_t rows, int64_t cols, int64_t ld, signed char* q, int64_t ldq, float* scales, int num_cus,
                            hipStream_t s) {
  constexpr int kRows = 4 * kTiles * Source<DT>::kPer;  // numbers that a thread holds
  // (offsets within a tile of the rows have 32 bits)
  const bool held = cols >= 64 && ld * (DT == DT_F32 ? 4 : 2) * 1024 < (int64_t)1 << 31;
  // (what a workgroup holds of a column has to reach to the end of a row of q, zeros behind the last number included)
  const auto holds = [&](int nt, int columns) { return held && ldq <= nt * kRows / columns; };
  // (smaller workgroups, more stripes under way: 64 x 100000 bf16 13 us, 21 in workgroups of 512; not to the full: 500 x 65536 27, 24)
  if (rows <= 128 * kRows / 64 && holds(256, 64)) return quantize_held_columns<DT, 256, 64>(src, rows, cols, ld, q, ldq, scales, num_cus, s);
  if (holds(512, 64)) return quantize_held_columns<DT, 512, 64>(src, rows, cols, ld, q, ldq, scales, num_cus, s);
  if (holds(1024, 64)) return quantize_held_columns<DT, 1024, 64>(src, rows, cols, ld, q, ldq, scales, num_cus, s);
  if (holds(1024, 32)) return quantize_held_columns<DT, 1024, 32>(src, rows, cols, ld, q, ldq, scales, num_cus, s);
  for (int64_t c = 0; c < cols; c += kMostGroups * kColTile) {
    const int64_t n = cols - c < kMostGroups * kColTile ? cols - c : kMostGroups * kColTile;
    hipLaunchKernelGGL(quantize_columns_kernel<DT>, dim3((unsigned)((n + kColTile - 1) / kColTile)), dim3(kQuantThreads), 0, s,
                       reinterpret_cast<const typename Source<DT>::S*>(src) + c, (int)rows, n, ld, q + c * ldq, (int)ldq, scales + c);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace

hipError_t launch_quantize_rows(const void* src, int dtype, int64_t rows, int64_t cols, int64_t ld, signed char* q, int64_t ldq, float* scales,
                                hipStream_t s) {
  return dtype == DT_BF16  ? quantize_rows<DT_BF16>(src, rows, cols, ld, q, ldq, scales, s)
         : dtype == DT_F16 ? quantize_rows<DT_F16>(src, rows, cols, ld, q, ldq, scales, s)
                           : quantize_rows<DT_F32>(src, rows, cols, ld, q, ldq, scales, s);
}
hipError_t launch_quantize_columns(const void* src, int dtype, int64_t rows, int64_t cols, int64_t ld, signed char* q, int64_t ldq, float* scales,
                                   int num_cus, hipStream_t s) {
  return dtype == DT_BF16  ? quantize_columns<DT_BF16>(src, rows, cols, ld, q, ldq, scales, num_cus, s)
         : dtype == DT_F16 ? quantize_columns<DT_F16>(src, rows, cols, ld, q, ldq, scales, num_cus, s)
                           : quantize_columns<DT_F32>(src, rows, cols, ld, q, ldq, scales, num_cus, s);
}
bool int8_quantizes(const Int8Args& a) {
  int places, depth;
  return fuses(a) && streams(a, &places, &depth);
}
hipError_t launch_int8_logits(const Int8Args& a, hipStream_t s) {
  return a.out_dtype == DT_BF16 ? launch_product<BF16>(a, s) : a.out_dtype == DT_F16 ? launch_product<F16>(a, s) : launch_product<float>(a, s);
}

}  // namespace lce

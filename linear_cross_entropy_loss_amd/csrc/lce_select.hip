// The largest logits of a row and one token drawn from it: selections in the order of a row, value descending, equal values by
// column.  One workgroup has a row at a time.
//
//   weight  w[j] = exp((z[j] - max z) / temperature), in fixed point: `bits` binary places, so that a row's sum stays below 2^63
//           and sums do not depend on their order
//   top_k   the first k;  top_p  column j stays while the weights before it are less than top_p times those that top_k left;
//   min_p   columns with w >= min_p.  Each keeps a beginning of the order, never less than its first column.
//   token   the first column up to which more than u times the weight of what stays has gathered
//
// A value is selected by its 32-bit key (unsigned, in the order of the values, -0 as 0, NaN above all) in three digits of 11, 11 and
// 10 bits: a histogram of counts and weights over the digit's values, whose prefix sums say in which of them the wanted place
// lies, then the next digit of the columns there.
#include "lce_gemm.h"
#include "lce_internal.h"

namespace lce {

namespace {

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64;
constexpr int kDigits = 2048;  // values of a digit
typedef unsigned long long u64;

constexpr unsigned kNanKey = 0xffffffffu, kLowKey = 0x007fffffu;  // NaN; -infinity
LCE_DEV unsigned key_of(float f) {
  unsigned b = __builtin_bit_cast(unsigned, f);
  if (f != f) return kNanKey;
  if (f == 0.f) b = 0;
  return b >> 31 ? ~b : b | 0x80000000u;
}
LCE_DEV float value_of(unsigned key) {
  const unsigned b = key >> 31 ? key & 0x7fffffffu : ~key;
  return __builtin_bit_cast(float, b);
}
LCE_DEV float as_float(__bf16 v) { return (float)v; }
LCE_DEV float as_float(_Float16 v) { return (float)v; }
LCE_DEV float as_float(float v) { return v; }

template <int BYTES> struct bits_of;
template <> struct bits_of<2> { typedef unsigned short type; };
template <> struct bits_of<4> { typedef unsigned type; };

// A row in units of up to 16 bytes: its elements before the first address of 16 bytes, whole pieces, the rest.  Wave w has the units
// [w * share, (w + 1) * share), 64 neighbouring ones at a time, so that (wave, round, lane, element) is the order of the columns.
template <class E> struct RowUnits {
  static constexpr int kPer = 16 / sizeof(E);
  const E* p;
  int64_t head, body, n, share, units;
  LCE_DEV RowUnits(const E* row, int64_t cols) : p(row), n(cols) {
    const int64_t off = (int64_t)(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(E));
    head = off < n ? off : n;
    body = (n - head) / kPer;
    units = body + 2;
    share = (units + kSelectThreads - 1) / kSelectThreads * 64;
  }
  LCE_DEV int64_t column(int64_t unit) const { return unit == 0 ? 0 : head + (unit - 1) * kPer; }
  LCE_DEV int count(int64_t unit) const {
    return unit == 0 ? (int)head : unit <= body ? kPer : unit == body + 1 ? (int)(n - head - body * kPer) : 0;
  }
  LCE_DEV u32x4_t load(int64_t unit) const {
    if (unit >= 1 && unit <= body) return *reinterpret_cast<const u32x4_t*>(p + column(unit));
    // (a loop that is not unrolled: it is for two units of a row)
    typedef typename bits_of<sizeof(E)>::type Bits;
    const Bits* from = reinterpret_cast<const Bits*>(p + column(unit));
    const int c = count(unit);
    u64 lo = 0, hi = 0;
#pragma unroll 1
    for (int i = 0; i < c; ++i) {
      const int at = i * (int)sizeof(E) * 8;
      if (at < 64) lo |= (u64)from[i] << at;
      else hi |= (u64)from[i] << (at - 64);
    }
    return u32x4_t{(unsigned)lo, (unsigned)(lo >> 32), (unsigned)hi, (unsigned)(hi >> 32)};
  }
  // f(unit, elements, how many of them are there) for the units of this lane, two loads in flight; every lane of a wave makes
  // the same number of calls.
  template <class F> LCE_DEV void each(F f) const {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t u0 = wave * share + lane;
    for (int64_t i = 0; i < share && wave * share + i < units; i += 128) {
      u32x4_t v[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) v[r] = i + r * 64 < share ? load(u0 + i + r * 64) : u32x4_t{};
#pragma unroll
      for (int r = 0; r < 2; ++r)
        if (i + r * 64 < share) {
          E e[kPer];
          __builtin_memcpy(e, &v[r], 16);
          f(u0 + i + r * 64, e, count(u0 + i + r * 64));
        }
    }
  }
};

template <class F, class Join> LCE_DEV F wave_all(F v, Join join) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) v = join(v, (F)__shfl_xor(v, d));
  return v;
}
// Over the workgroup; `sh`: room for one value of each wave.  Ends with a barrier.
template <class F, class Join> LCE_DEV F block_all(F v, F* sh, Join join) {
  v = wave_all(v, join);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  F r = sh[0];
  for (int w = 1; w < kSelectWaves; ++w) r = join(r, sh[w]);
  __syncthreads();
  return r;
}
// Sum over the threads before this one.  Ends with a barrier.
template <class F> LCE_DEV F block_before(F v, F* sh) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  F up = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const F o = __shfl_up(up, d);
    if (lane >= d) up += o;
  }
  if (lane == 63) sh[wave] = up;
  __syncthreads();
  F before = up - v;
  for (int w = 0; w < wave; ++w) before += sh[w];
  __syncthreads();
  return before;
}

// The column of the r-th (from 0) element with the key; -1 if there are no more than r.  All threads take part and get it.
template <class E> LCE_DEV int64_t column_of(const RowUnits<E>& row, unsigned key, int64_t r, int64_t* sh /* [kSelectWaves + 1] */) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int mine = 0;
  row.each([&](int64_t, const E* e, int c) {
#pragma unroll
    for (int i = 0; i < RowUnits<E>::kPer; ++i) mine += i < c && key_of(as_float(e[i])) == key ? 1 : 0;
  });
  const int64_t of_wave = wave_all((int64_t)mine, [](int64_t a, int64_t b) { return a + b; });
  if (lane == 0) sh[wave] = of_wave;
  if (threadIdx.x == 0) sh[kSelectWaves] = -1;
  __syncthreads();
  int64_t before = 0;
  for (int w = 0; w < wave; ++w) before += sh[w];
  if (before <= r && r < before + of_wave) {  // (one wave)
    row.each([&](int64_t unit, const E* e, int c) {
      int here = 0;
#pragma unroll
      for (int i = 0; i < RowUnits<E>::kPer; ++i) here += i < c && key_of(as_float(e[i])) == key ? 1 : 0;
      int up = here;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_up(up, d);
        if (lane >= d) up += o;
      }
      int64_t at = before + up - here;
#pragma unroll
      for (int i = 0; i < RowUnits<E>::kPer; ++i)
        if (i < c && key_of(as_float(e[i])) == key) {
          if (at == r) sh[kSelectWaves] = row.column(unit) + i;
          ++at;
        }
      before += __shfl(up, 63);
    });
  }
  __syncthreads();
  const int64_t at = sh[kSelectWaves];
  __syncthreads();
  return at;
}

// 2^t for t <= 0: 2^(t - rint t) by its Taylor series in the 64-bit unit, whose first term left out is below 7e-15, times a power of two.
LCE_DEV double exp2_series(double t) {
  const double n = rint(t), x = (t - n) * 0.69314718055994530942;
  double p = 1.0 / 39916800.0;
  p = fma(p, x, 1.0 / 3628800.0);
  p = fma(p, x, 1.0 / 362880.0);
  p = fma(p, x, 1.0 / 40320.0);
  p = fma(p, x, 1.0 / 5040.0);
  p = fma(p, x, 1.0 / 720.0);
  p = fma(p, x, 1.0 / 120.0);
  p = fma(p, x, 1.0 / 24.0);
  p = fma(p, x, 1.0 / 6.0);
  p = fma(p, x, 0.5);
  p = fma(p, x, 1.0);
  p = fma(p, x, 1.0);
  return ldexp(p, (int)n);
}

// Weights of a row as fixed-point numbers.
struct Weights {
  double top, per;  // the largest value, log2(e) / temperature
  double one;       // 2^bits, bits <= 50
  LCE_DEV double real(float z) const {
    // (equal infinities have no difference, and one times 0, at an infinite temperature, is no number)
    const double zd = (double)z, t = zd == top ? 0.0 : fmax((zd - top) * per, -2000.0);
    return exp2_series(t);
  }
  // (rounded by the sum with 2^52, whose last place is 1)
  LCE_DEV u64 of(float z) const { return __builtin_bit_cast(u64, fma(real(z), one, 4503599627370496.0)) & 0xfffffffffffffull; }
};
struct NoWeights {
  LCE_DEV u64 of(float) const { return 0; }
};

struct Histogram {
  int count[kDigits];
  u64 weight[kDigits];
};
LCE_DEV int digit_of(unsigned key, int level) { return level == 0 ? key >> 21 : level == 1 ? (key >> 10) & 2047 : key & 1023; }
LCE_DEV bool in_prefix(unsigned key, unsigned prefix, int level) {
  return level == 0 || (level == 1 ? (key ^ prefix) >> 21 == 0 : (key ^ prefix) >> 10 == 0);
}

// Histogram of the digit `level` over the elements that agree with `prefix` in the digits before it.  WEIGHTED: elements without
// a weight, which are never drawn, are left out.  Ends with a barrier.
template <bool WEIGHTED, class E, class W>
LCE_DEV void fill_histogram(const RowUnits<E>& row, const W& weights, unsigned prefix, int level, Histogram* h) {
  for (int i = threadIdx.x; i < kDigits; i += kSelectThreads) {
    h->count[i] = 0;
    if (WEIGHTED) h->weight[i] = 0;
  }
  __syncthreads();
  row.each([&](int64_t, const E* e, int c) {
#pragma unroll
    for (int i = 0; i < RowUnits<E>::kPer; ++i) {
      const float z = as_float(e[i]);
      const unsigned key = key_of(z);
      if (i >= c || !in_prefix(key, prefix, level)) continue;
      if (WEIGHTED) {
        const u64 w = key == kLowKey ? 0 : weights.of(z);
        if (w == 0) continue;
        atomicAdd(&h->weight[digit_of(key, level)], w);
      }
      atomicAdd(&h->count[digit_of(key, level)], 1);
    }
  });
  __syncthreads();
}

// A place in the order: the key there, and how many elements and what weight come before the first of that key.
struct Place {
  unsigned key;
  int64_t count;
  u64 weight;
  int64_t same;  // elements with the key
};
struct SelectShared {
  Histogram first, next;
  Place place;
  u64 of_wave[kSelectWaves];
  int64_t of_wave_count[kSelectWaves + 1];
};

// The histogram of the first digit; returns the weight of the elements with a key of `least` and above.
template <class E> LCE_DEV u64 fill_first(const RowUnits<E>& row, const Weights& weights, unsigned least, SelectShared* sh) {
  for (int i = threadIdx.x; i < kDigits; i += kSelectThreads) {
    sh->first.count[i] = 0;
    sh->first.weight[i] = 0;
  }
  __syncthreads();
  u64 mine = 0;
  row.each([&](int64_t, const E* e, int c) {
#pragma unroll
    for (int i = 0; i < RowUnits<E>::kPer; ++i) {
      const float z = as_float(e[i]);
      const unsigned key = key_of(z);
      if (i >= c || key == kLowKey) continue;
      const u64 w = weights.of(z);
      if (w == 0) continue;
      if (key >= least) mine += w;
      atomicAdd(&sh->first.weight[digit_of(key, 0)], w);
      atomicAdd(&sh->first.count[digit_of(key, 0)], 1);
    }
  });
  return block_all(mine, sh->of_wave, [](u64 a, u64 b) { return a + b; });
}

// What a place is looked for by: the k-th element; the last key with an element before which there is less than `most` weight; the
// first with which there is more than `target`.
enum Wanted { kByCount, kByShare, kByWeight };
struct Want {
  Wanted what;
  int64_t k;
  double most;
  u64 target;
  // whether it is among c elements of weight w behind cb elements of weight wb
  LCE_DEV bool here(int64_t cb, u64 wb, int64_t c, u64 w) const {
    if (c == 0) return false;
    if (what == kByCount) return cb < k && k <= cb + c;
    if (what == kByShare) return (wb == 0 || (double)wb < most) && !((double)(wb + w) < most);
    return wb <= target && target - wb < w;
  }
};

// The place that is wanted.  WEIGHTED: the histogram of the first digit is there (fill_first).
template <bool WEIGHTED, class E, class W>
LCE_DEV Place find_place(const RowUnits<E>& row, const W& weights, SelectShared* sh, const Want& want) {
  Place p = {0, 0, 0, 0};
#pragma unroll 1
  for (int level = 0; level < 3; ++level) {
    Histogram* h = level == 0 ? &sh->first : &sh->next;
    if (level > 0 || !WEIGHTED) fill_histogram<WEIGHTED>(row, weights, p.key, level, h);
    const int d1 = kDigits - 1 - 2 * (int)threadIdx.x, d0 = d1 - 1;  // this thread's digits, the larger first
    const int c1 = h->count[d1], c0 = h->count[d0];
    const u64 w1 = WEIGHTED ? h->weight[d1] : 0, w0 = WEIGHTED ? h->weight[d0] : 0;
    int64_t cb = p.count + block_before((int64_t)(c1 + c0), sh->of_wave_count);
    u64 wb = WEIGHTED ? p.weight + block_before(w1 + w0, sh->of_wave) : 0;
    const int shift = level == 0 ? 21 : level == 1 ? 10 : 0;
    if (want.here(cb, wb, c1, w1)) sh->place = {p.key | (unsigned)d1 << shift, cb, wb, c1};
    cb += c1;
    wb += w1;
    if (want.here(cb, wb, c0, w0)) sh->place = {p.key | (unsigned)d0 << shift, cb, wb, c0};
    __syncthreads();
    p = sh->place;
    __syncthreads();
  }
  return p;
}

// The largest key of the row.
template <class E> LCE_DEV unsigned largest_key(const RowUnits<E>& row, unsigned* sh) {
  unsigned top = 0;
  row.each([&](int64_t, const E* e, int c) {
#pragma unroll
    for (int i = 0; i < RowUnits<E>::kPer; ++i) {
      const unsigned k = key_of(as_float(e[i]));
      top = i < c && k > top ? k : top;
    }
  });
  return block_all(top, sh, [](unsigned a, unsigned b) { return a > b ? a : b; });
}

template <class E>
__global__ __launch_bounds__(kSelectThreads) void sample_kernel(const E* logits, int64_t rows, int64_t cols, int64_t ld, const float* u,
                                                                const Sampling s, int bits, int64_t* token) {
  __shared__ SelectShared sh;
  for (int64_t n = blockIdx.x; n < rows; n += gridDim.x) {
    const RowUnits<E> row(logits + n * ld, cols);
    const float temperature = s.temperature_rows ? s.temperature_rows[n] : s.temperature;
    const float top_p = s.top_p_rows ? s.top_p_rows[n] : s.top_p, min_p = s.min_p_rows ? s.min_p_rows[n] : s.min_p;
    const int64_t top_k = s.top_k_rows ? s.top_k_rows[n] : s.top_k;
    const unsigned top = largest_key(row, reinterpret_cast<unsigned*>(sh.of_wave));
    if (top == kNanKey || top == kLowKey) {  // a NaN, or no column left
      if (threadIdx.x == 0) token[n] = -1;
      continue;
    }
    Place at = {top, 0, 0, 0};
    int64_t r = 0;
    if (threadIdx.x == 0) sh.place = at;
    if (temperature > 0.f && top_k != 1) {
      const Weights weights = {(double)value_of(top), 1.4426950408889634074 / (double)temperature, (double)((u64)1 << bits)};
      // the smallest key that min_p keeps: the weights are monotone in the keys
      unsigned least = top;
      if (min_p > 0.f) {
        unsigned lo = kLowKey;  // (`least` has such a weight: the first column always stays)
        while (least - lo > 1) {
          const unsigned mid = lo + (least - lo) / 2;
          if (weights.real(value_of(mid)) >= (double)min_p) least = mid;
          else lo = mid;
        }
      }
      const u64 by_min = fill_first(row, weights, min_p > 0.f ? least : 0, &sh);
      const int t2 = 2 * (int)threadIdx.x;
      auto add = [](u64 a, u64 b) { return a + b; };
      const u64 all = block_all(sh.first.weight[t2] + sh.first.weight[t2 + 1], sh.of_wave, add);
      const int64_t counted = (int64_t)block_all((u64)(sh.first.count[t2] + sh.first.count[t2 + 1]), sh.of_wave, add);
      u64 stays = all;
#pragma unroll 1
      for (int step = kByCount; step <= kByWeight; ++step) {
        if (step == kByCount && !(top_k > 0 && top_k < counted)) continue;
        if (step == kByShare && !(top_p < 1.f)) continue;
        Want want = {(Wanted)step, top_k, (double)top_p * (double)stays, 0};
        if (step == kByWeight) {
          if (by_min < stays) stays = by_min;
          const double some = (double)u[n] * (double)stays;
          want.target = some > 0.0 ? (u64)some : 0;
          if (want.target >= stays) want.target = stays - 1;
        }
        at = find_place<true>(row, weights, &sh, want);
        u64 w = weights.of(value_of(at.key));
        w = w == 0 ? 1 : w;  // (not of an element that was counted)
        if (step == kByCount) {
          stays = at.weight + (u64)(top_k - at.count) * w;
        } else if (step == kByShare) {
          const double some = (want.most - (double)at.weight) / (double)w;
          int64_t kept = some > 0.0 ? (int64_t)some : 0;
          if (kept > at.same) kept = at.same;
          if (kept < at.same && (double)(at.weight + (u64)kept * w) < want.most) ++kept;  // (`some` rounded down)
          if (at.weight == 0 && kept == 0) kept = 1;
          const u64 by_p = at.weight + (u64)kept * w;
          if (by_p < stays) stays = by_p;
        } else {
          r = (int64_t)((want.target - at.weight) / w);
        }
      }
    }
    const int64_t column = column_of(row, at.key, r, sh.of_wave_count);
    if (threadIdx.x == 0) token[n] = column;
  }
}

constexpr int kMostTop = 1024;

template <class E>
__global__ __launch_bounds__(kSelectThreads) void top_kernel(const E* logits, int64_t rows, int64_t cols, int64_t ld, int k, int sorted,
                                                             E* values, int64_t* index, float* lse) {
  __shared__ SelectShared sh;
  __shared__ u64 list[kMostTop];
  __shared__ int listed;
  for (int64_t n = blockIdx.x; n < rows; n += gridDim.x) {
    const RowUnits<E> row(logits + n * ld, cols);
    const NoWeights none;
    if (lse != nullptr) {
      const unsigned top = largest_key(row, reinterpret_cast<unsigned*>(sh.of_wave));
      const float m = top == kNanKey ? __builtin_nanf("") : value_of(top);
      float sum = 0.f;
      row.each([&](int64_t, const E* e, int c) {
#pragma unroll
        for (int i = 0; i < RowUnits<E>::kPer; ++i) {
          const float z = as_float(e[i]);
          if (i < c) sum += z == m ? 1.f : __expf(z - m);  // (equal infinities have no difference)
        }
      });
      const double all = block_all((double)sum, reinterpret_cast<double*>(sh.of_wave), [](double a, double b) { return a + b; });
      if (threadIdx.x == 0) lse[n] = top == kLowKey ? m : (float)((double)m + log(all));
    }
    const Place p = find_place<false>(row, none, &sh, Want{kByCount, k, 0.0, 0});
    // what is larger, in any order, and the first k - p.count of the key
    if (threadIdx.x == 0) listed = 0;
    if ((int)threadIdx.x < sorted) list[threadIdx.x] = ~(u64)0;
    int mine = 0;
    __syncthreads();
    row.each([&](int64_t unit, const E* e, int c) {
#pragma unroll
      for (int i = 0; i < RowUnits<E>::kPer; ++i) {
        const unsigned key = key_of(as_float(e[i]));
        if (i < c && key > p.key) {
          const int to = atomicAdd(&listed, 1);  // (p.count of them)
          if (to < kMostTop) list[to] = (u64)~key << 32 | (u64)(row.column(unit) + i);
        }
        mine += i < c && key == p.key ? 1 : 0;
      }
    });
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t of_wave = wave_all((int64_t)mine, [](int64_t a, int64_t b) { return a + b; });
    if (lane == 0) sh.of_wave_count[wave] = of_wave;
    __syncthreads();
    const int64_t want = k - p.count;
    int64_t before = 0;
    for (int w = 0; w < wave; ++w) before += sh.of_wave_count[w];
    if (of_wave > 0 && before < want) {
      row.each([&](int64_t unit, const E* e, int c) {
        int here = 0;
#pragma unroll
        for (int i = 0; i < RowUnits<E>::kPer; ++i) here += i < c && key_of(as_float(e[i])) == p.key ? 1 : 0;
        int up = here;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const int o = __shfl_up(up, d);
          if (lane >= d) up += o;
        }
        int64_t at = before + up - here;
#pragma unroll
        for (int i = 0; i < RowUnits<E>::kPer; ++i)
          if (i < c && key_of(as_float(e[i])) == p.key) {
            if (at < want) list[p.count + at] = (u64)~p.key << 32 | (u64)(row.column(unit) + i);
            ++at;
          }
        before += __shfl(up, 63);
      });
    }
    // in order: by key, then by column (a bitonic network over `sorted`, a power of two)
    for (int size = 2; size <= sorted; size <<= 1)
      for (int d = size >> 1; d > 0; d >>= 1) {
        __syncthreads();
        const int i = threadIdx.x, j = i ^ d;
        if (i < sorted && j > i) {
          const u64 a = list[i], b = list[j];
          if ((a > b) == ((i & size) == 0)) {
            list[i] = b;
            list[j] = a;
          }
        }
      }
    __syncthreads();
    if ((int)threadIdx.x < k) {
      int64_t column = (int64_t)(list[threadIdx.x] & 0xffffffffu);
      column = column < cols ? column : cols - 1;  // (logits that change under the kernel must not lead it astray)
      index[n * k + threadIdx.x] = column;
      values[n * k + threadIdx.x] = row.p[column];
    }
    __syncthreads();
  }
}

unsigned grid_of(int64_t rows) { return (unsigned)(rows < (int64_t)1 << 20 ? rows : (int64_t)1 << 20); }

}  // namespace

hipError_t launch_sample(const void* logits, int dtype, int64_t rows, int64_t cols, int64_t ld, const float* u, const Sampling& s,
                         int64_t* token, hipStream_t stream) {
  int log2 = 0;
  while ((int64_t)1 << log2 < cols) ++log2;
  const int bits = 62 - log2 < 50 ? 62 - log2 : 50;  // (a double has 53: a weight of one and the half that rounds it fit)
  const dim3 grid(grid_of(rows)), block(kSelectThreads);
  if (dtype == DT_BF16) hipLaunchKernelGGL(sample_kernel<__bf16>, grid, block, 0, stream, (const __bf16*)logits, rows, cols, ld, u, s, bits, token);
  else if (dtype == DT_F16)
    hipLaunchKernelGGL(sample_kernel<_Float16>, grid, block, 0, stream, (const _Float16*)logits, rows, cols, ld, u, s, bits, token);
  else if (dtype == DT_F32) hipLaunchKernelGGL(sample_kernel<float>, grid, block, 0, stream, (const float*)logits, rows, cols, ld, u, s, bits, token);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}

hipError_t launch_top(const void* logits, int dtype, int64_t rows, int64_t cols, int64_t ld, int k, void* values, int64_t* index, float* lse,
                      hipStream_t stream) {
  int sorted = 2;
  while (sorted < k) sorted <<= 1;
  const dim3 grid(grid_of(rows)), block(kSelectThreads);
  if (dtype == DT_BF16)
    hipLaunchKernelGGL(top_kernel<__bf16>, grid, block, 0, stream, (const __bf16*)logits, rows, cols, ld, k, sorted, (__bf16*)values, index, lse);
  else if (dtype == DT_F16)
    hipLaunchKernelGGL(top_kernel<_Float16>, grid, block, 0, stream, (const _Float16*)logits, rows, cols, ld, k, sorted, (_Float16*)values, index,
                       lse);
  else if (dtype == DT_F32)
    hipLaunchKernelGGL(top_kernel<float>, grid, block, 0, stream, (const float*)logits, rows, cols, ld, k, sorted, (float*)values, index, lse);
  else return hipErrorInvalidValue;
  return hipGetLastError();
}

}  // namespace lce

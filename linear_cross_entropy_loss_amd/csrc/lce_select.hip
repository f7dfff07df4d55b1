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

constexpr int kDigits = 2048;  // values of a digit
constexpr int kMostWaves = 16;  // of a workgroup
typedef unsigned long long u64;

// The thread's number, as one that the compiler takes for a new one each time: it would else work out addresses from it before the loop
// over the rows, for all of a kernel's ways to do a row, and there are no registers to keep them in.
LCE_DEV int thread() {
  int t = threadIdx.x;
  asm volatile("" : "+v"(t));
  __builtin_assume(t >= 0 && t < 1024);
  return t;
}

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
template <class E, int NT, int FLIGHT = 4> struct RowUnits {
  static constexpr int kPer = 16 / sizeof(E);
  const E* p;
  int head, body, n, share, units;
  LCE_DEV RowUnits(const E* row, int64_t cols) : p(row), n((int)cols) {
    const int off = (int)(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(E));
    head = off < n ? off : n;
    body = (n - head) / kPer;
    units = body + 2;
    share = (units + NT - 1) / NT * 64;
  }
  LCE_DEV int column(int unit) const { return unit == 0 ? 0 : head + (unit - 1) * kPer; }
  LCE_DEV int count(int unit) const {
    return unit == 0 ? head : unit <= body ? kPer : unit == body + 1 ? n - head - body * kPer : 0;
  }
  LCE_DEV u32x4_t load(int unit) const {
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
  // f(unit, its elements, how many of them are there) for the units of this lane, FLIGHT loads in flight; every lane of a wave makes
  // the same number of calls.  (Loops that are not unrolled, here and over the elements: the kernels that end up here, for the rows that
  // their own way does not do, have no registers to spare.)
  template <class F> LCE_DEV void each(F f) const {
    const int t = thread(), lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int u0 = wave * share + lane;
#pragma unroll 1
    for (int i = 0; i < share && wave * share + i < units; i += FLIGHT * 64) {
      u32x4_t v[FLIGHT];
#pragma unroll
      for (int r = 0; r < FLIGHT; ++r) v[r] = i + r * 64 < share ? load(u0 + i + r * 64) : u32x4_t{};
#pragma unroll 1
      for (int j = i; j < i + FLIGHT * 64 && j < share; j += 64) {
        f(u0 + j, v[0], count(u0 + j));
#pragma unroll
        for (int r = 0; r + 1 < FLIGHT; ++r) v[r] = v[r + 1];
      }
    }
  }
  // f(which, element) for the elements of a unit.
  template <class F> LCE_DEV static void elements(u32x4_t v, int c, F f) {
    constexpr int kHalves = 4 / sizeof(E);
#pragma unroll 1
    for (int i = 0; i < c; i += kHalves) {
      const unsigned w = v[0];
      if constexpr (kHalves == 2) {
        f(i, as_float(__builtin_bit_cast(E, (unsigned short)w)));
        if (i + 1 < c) f(i + 1, as_float(__builtin_bit_cast(E, (unsigned short)(w >> 16))));
      } else {
        f(i, __builtin_bit_cast(float, w));
      }
      v = u32x4_t{v[1], v[2], v[3], 0};
    }
  }
  // f(element) for the elements of this lane's units.
  template <class F> LCE_DEV void elements(F f) const {
    each([&](int, u32x4_t v, int c) { elements(v, c, [&](int, float z) { f(z); }); });
  }
};

// v of the lane that the DPP control names, 0 where there is none (or the row is not in ROWS).
template <int CTRL, int ROWS> LCE_DEV unsigned from_lane(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS> LCE_DEV int from_lane(int v) { return (int)from_lane<CTRL, ROWS>((unsigned)v); }
template <int CTRL, int ROWS> LCE_DEV u64 from_lane(u64 v) {
  return (u64)from_lane<CTRL, ROWS>((unsigned)(v >> 32)) << 32 | from_lane<CTRL, ROWS>((unsigned)v);
}
template <int CTRL, int ROWS> LCE_DEV double from_lane(double v) {
  return __builtin_bit_cast(double, from_lane<CTRL, ROWS>(__builtin_bit_cast(u64, v)));
}
LCE_DEV u64 read_lane(u64 v, int lane) {
  return (u64)(unsigned)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 | (unsigned)__builtin_amdgcn_readlane((int)v, lane);
}
LCE_DEV int read_lane(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
LCE_DEV unsigned read_lane(unsigned v, int lane) { return (unsigned)__builtin_amdgcn_readlane((int)v, lane); }
LCE_DEV double read_lane(double v, int lane) { return __builtin_bit_cast(double, read_lane(__builtin_bit_cast(u64, v), lane)); }
// A value that all lanes have, into scalar registers.
template <class F> LCE_DEV F uniform(F v) {
  if constexpr (sizeof(F) == 4) return __builtin_bit_cast(F, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, v)));
  else return read_lane(v, 0);
}
struct Sum {
  template <class F> LCE_DEV static F join(F a, F b) { return a + b; }
};
struct Largest {  // (of unsigned numbers: 0 stands for none)
  template <class F> LCE_DEV static F join(F a, F b) { return a > b ? a : b; }
};
// Joined over the lanes up to and with this one (every lane of the wave takes part).  ROW: over the 16 lanes of a row only.
template <class J, class F, bool ROW = false> LCE_DEV F wave_upto(F v) {
  v = J::join(v, from_lane<0x111, 0xf>(v));
  v = J::join(v, from_lane<0x112, 0xf>(v));
  v = J::join(v, from_lane<0x114, 0xf>(v));
  v = J::join(v, from_lane<0x118, 0xf>(v));
  if constexpr (!ROW) {
    v = J::join(v, from_lane<0x142, 0xa>(v));
    v = J::join(v, from_lane<0x143, 0xc>(v));
  }
  return v;
}
// Over the workgroup; `sh`: room for one value of each wave.  *before (sums): over the threads before this one.  Ends with a barrier.
template <class J, int NT, class F> LCE_DEV F block_all(F v, F* sh, F* before = nullptr) {
  const int t = thread(), lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const F upto = wave_upto<J>(v);
  if (lane == 63) sh[wave] = upto;
  __syncthreads();
  static_assert(NT / 64 <= 16, "a row of lanes joins the waves' values");
  const F waves = wave_upto<J, F, true>((lane & 15) < NT / 64 ? sh[lane & 15] : F(0));
  __syncthreads();
  if (before != nullptr) *before = upto - v + (wave > 0 ? read_lane(waves, wave - 1) : F(0));
  return read_lane(waves, 15);
}

// 16 bytes of a row as unsigned numbers in the order of the values (-0 just below 0), two of 16 bits or one of 32 bits to a word.
template <class E> struct Ordered;
template <> struct Ordered<float> {
  static constexpr unsigned kLow = 0x007fffffu, kInf = 0xff800000u;
  LCE_DEV static unsigned word(unsigned w) { return w ^ ((unsigned)((int)w >> 31) | 0x80000000u); }
  LCE_DEV static unsigned larger(unsigned a, unsigned b) { return a > b ? a : b; }
  LCE_DEV static unsigned smaller(unsigned a, unsigned b) { return a < b ? a : b; }
  LCE_DEV static unsigned largest(unsigned a) { return a; }
  LCE_DEV static unsigned smallest(unsigned a) { return a; }
  LCE_DEV static unsigned in_top_bits(unsigned a) { return a >> 16; }
  LCE_DEV static unsigned from_top_bits(unsigned a) { return a << 16; }
  LCE_DEV static float value(unsigned a) { return value_of(a); }
};
template <class E> struct OrderedHalf {
  typedef short signed_t __attribute__((ext_vector_type(2)));
  typedef unsigned short pair_t __attribute__((ext_vector_type(2)));
  LCE_DEV static unsigned word(unsigned w) {
    return w ^ (__builtin_bit_cast(unsigned, __builtin_bit_cast(signed_t, w) >> (short)15) | 0x80008000u);
  }
  LCE_DEV static unsigned larger(unsigned a, unsigned b) {
    return __builtin_bit_cast(unsigned, __builtin_elementwise_max(__builtin_bit_cast(pair_t, a), __builtin_bit_cast(pair_t, b)));
  }
  LCE_DEV static unsigned smaller(unsigned a, unsigned b) {
    return __builtin_bit_cast(unsigned, __builtin_elementwise_min(__builtin_bit_cast(pair_t, a), __builtin_bit_cast(pair_t, b)));
  }
  LCE_DEV static unsigned largest(unsigned a) { return a >> 16 > (a & 0xffffu) ? a >> 16 : a & 0xffffu; }
  LCE_DEV static unsigned smallest(unsigned a) { return a >> 16 < (a & 0xffffu) ? a >> 16 : a & 0xffffu; }
  LCE_DEV static unsigned in_top_bits(unsigned a) { return a; }
  LCE_DEV static unsigned from_top_bits(unsigned a) { return a; }
  LCE_DEV static float value(unsigned a) {
    return (float)__builtin_bit_cast(E, (unsigned short)(a & 0x8000u ? a & 0x7fffu : a ^ 0xffffu));
  }
};
template <> struct Ordered<__bf16> : OrderedHalf<__bf16> { static constexpr unsigned kLow = 0x007f, kInf = 0xff80; };
template <> struct Ordered<_Float16> : OrderedHalf<_Float16> { static constexpr unsigned kLow = 0x03ff, kInf = 0xfc00; };

// Whole pieces of a row, dealt to the threads one by one, and the elements before and behind them.
template <class E, int NT> struct RowPieces {
  typedef Ordered<E> O;
  typedef typename bits_of<sizeof(E)>::type Bits;
  static constexpr int kPer = 16 / sizeof(E), kFlight = 4;
  const E* p;
  int n, head, body;
  LCE_DEV RowPieces(const E* row, int64_t cols) : p(row), n((int)cols) {
    const int off = (int)(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(E));
    head = off < n ? off : n;
    body = (n - head) / kPer;
  }
  // f(column, ordered bits) for the elements at the edges, one to a thread.
  template <class F> LCE_DEV void edges(F f) const {
    const int tail = n - head - body * kPer, t = thread();
    if (t < head + tail) {
      const int at = t < head ? t : n - tail + (t - head);
      const unsigned w = O::word(reinterpret_cast<const Bits*>(p)[at]);
      f(at, sizeof(E) == 2 ? w & 0xffffu : w);
    }
  }
  // f(column of the first, piece, which of its round), kFlight pieces in flight.
  template <class F> LCE_DEV void each(F f) const {
    const u32x4_t* from = reinterpret_cast<const u32x4_t*>(p + head);
#pragma unroll 1
    for (int base = thread(); base < body; base += kFlight * NT) {
      u32x4_t v[kFlight];
#pragma unroll
      for (int r = 0; r < kFlight; ++r) {
        const int at = base + r * NT;
        v[r] = from[at < body ? at : base];
      }
#pragma unroll
      for (int r = 0; r < kFlight; ++r) {
        const int at = base + r * NT;
        if (at < body) f(head + at * kPer, v[r], r);
      }
    }
  }
  // The largest key.
  LCE_DEV unsigned largest(unsigned* sh) const {
    unsigned most = 0, least = ~0u;
    edges([&](int, unsigned a) {
      most = O::larger(most, a);  // (of 16 bits: the upper half stays as it is)
      least = O::smaller(least, sizeof(E) == 2 ? a | 0xffff0000u : a);
    });
    each([&](int, u32x4_t v, int) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned a = O::word(v[i]);
        most = O::larger(most, a);
        least = O::smaller(least, a);
      }
    });
    most = O::largest(most);
    if (O::smallest(least) < O::kLow) most = ~0u;  // (a NaN is above +inf or below -inf)
    most = block_all<Largest, NT>(most, sh);
    return most > O::kInf ? kNanKey : key_of(O::value(most));
  }
};

// The elements of 16 bytes that equal a value: how many, and which.  0 and -0 are equal; the value is no NaN.
template <class E> struct Equal {  // 16-bit elements
  unsigned twice, mask;
  LCE_DEV explicit Equal(float value) {
    const unsigned bits = __builtin_bit_cast(unsigned short, (E)value);
    mask = (bits & 0x7fffu) == 0 ? 0x7fff7fffu : 0xffffffffu;
    twice = (bits | bits << 16) & mask;
  }
  LCE_DEV int count(u32x4_t v) const {
    typedef unsigned short pair_t __attribute__((ext_vector_type(2)));
    pair_t others = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned x = (v[i] & mask) ^ twice;
      others += __builtin_elementwise_min(__builtin_bit_cast(pair_t, x), pair_t{1, 1});
    }
    return 8 - (others[0] + others[1]);
  }
  LCE_DEV bool is(u32x4_t v, int k) const {
    const unsigned x = (v[k >> 1] & mask) ^ twice;
    return (k & 1 ? x >> 16 : x & 0xffffu) == 0;
  }
};
template <> struct Equal<float> {
  float value;
  LCE_DEV explicit Equal(float v) : value(v) {}
  LCE_DEV bool is(u32x4_t v, int k) const {
    const unsigned w = v[k];
    return __builtin_bit_cast(float, w) == value;
  }
  LCE_DEV int count(u32x4_t v) const { return is(v, 0) + is(v, 1) + is(v, 2) + is(v, 3); }
};

// The column of the r-th (from 0) element with a value, which is no NaN; -1 if there are no more than r.  All threads take part and get it.
// The waves count such elements, by parts of their share of the row's pieces, and the one that has the r-th looks for it in its part.
// kPartRounds loads of 1 KiB a wave are in flight together.
constexpr int kParts = 32;
struct ColumnShared {
  int count[kMostWaves][kParts];
  int of_wave[kMostWaves];
  int column;
};
template <int kPartRounds = 8, class E, int NT> LCE_DEV int column_of(const RowPieces<E, NT>& row, float value, int r, ColumnShared* sh) {
  constexpr int kPer = RowPieces<E, NT>::kPer;
  const Equal<E> equal(value);
  const int t = thread(), lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int all = (row.body + 63) / 64, share = (all + NT / 64 - 1) / (NT / 64);  // in rounds: 64 pieces
  const int first = wave * share, left = all - first, rounds = left < 0 ? 0 : left < share ? left : share;
  const int per = (rounds + kParts * kPartRounds - 1) / (kParts * kPartRounds) * kPartRounds;  // rounds of a part
  const u32x4_t* from = reinterpret_cast<const u32x4_t*>(row.p + row.head);
  const int last = (first + rounds) * 64 < row.body ? (first + rounds) * 64 : row.body;
  // v, c: the pieces of kPartRounds rounds from i, and how many elements of each have the value
  u32x4_t v[kPartRounds];
  int c[kPartRounds];
  auto look = [&](int i) {
    const int piece = (first + i) * 64 + lane;
#pragma unroll
    for (int q = 0; q < kPartRounds; ++q) {
      const int at = piece + q * 64;
      v[q] = from[at < last ? at : last - 1];
    }
#pragma unroll
    for (int q = 0; q < kPartRounds; ++q) {
      const int equals = equal.count(v[q]);
      c[q] = piece + q * 64 < last ? equals : 0;
    }
  };
  // the elements before and behind the pieces (fewer than 8 each): in every wave
  const int tail = row.n - row.head - row.body * kPer;
  const E before_all = row.p[lane < row.head ? lane : 0], behind_all = row.p[row.n - 1 - (lane < tail ? tail - 1 - lane : 0)];
  if (t == 0) sh->column = -1;
  int mine = 0;
#pragma unroll 1
  for (int i = 0, part = 0; i < rounds; ++part) {
    int count = 0;
#pragma unroll 1
    for (const int end = i + per; i < end && i < rounds; i += kPartRounds) {
      look(i);
#pragma unroll
      for (int q = 0; q < kPartRounds; ++q) count += c[q];
    }
    count = read_lane(wave_upto<Sum>(count), 63);
    if (lane == 0) sh->count[wave][part] = count;
    mine += count;
  }
  if (lane == 0) sh->of_wave[wave] = mine;
  const u64 in_head = __ballot(lane < row.head && as_float(before_all) == value), in_tail = __ballot(lane < tail && as_float(behind_all) == value);
  __syncthreads();
  int before = __popcll(in_head), upto = before;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    before += w < wave ? sh->of_wave[w] : 0;
    upto += sh->of_wave[w];
  }
  if (before <= r && r < before + mine) {  // (one wave, or none)
    int i = 0;
    for (int part = 0; part < kParts - 1 && before + sh->count[wave][part] <= r; ++part, i += per) before += sh->count[wave][part];
#pragma unroll 1
    for (const int end = i + per; i < end && i < rounds; i += kPartRounds) {
      u32x4_t in = {};
      int round = -1, here = 0, upto_here = 0, before_round = 0;
      if (rounds > kPartRounds) look(i);  // (else they are still there)
#pragma unroll
      for (int q = 0; q < kPartRounds; ++q) {
        if (i + q >= rounds) continue;
        const int sum = wave_upto<Sum>(c[q]), of_round = read_lane(sum, 63);
        if (before <= r && r < before + of_round) {  // (one round)
          round = q;
          in = v[q];
          here = c[q];
          upto_here = sum;
          before_round = before;
        }
        before += of_round;
      }
      if (round < 0) continue;
      int at = before_round + upto_here - here;
#pragma unroll
      for (int k = 0; k < kPer; ++k)
        if (here != 0 && equal.is(in, k)) {
          if (at == r) sh->column = row.head + ((first + i + round) * 64 + lane) * kPer + k;
          ++at;
        }
      break;
    }
  } else if (t < 64 && (r < __popcll(in_head) || r >= upto)) {
    const bool head = r < __popcll(in_head);
    const int which = head ? r : r - upto;
    const u64 in = head ? in_head : in_tail;
    if ((in >> lane & 1) && __popcll(in & ((u64(1) << lane) - 1)) == which) sh->column = head ? lane : row.n - tail + lane;
  }
  __syncthreads();
  const int at = sh->column;
  __syncthreads();
  return at;
}

// a * b + c with c in scalar registers.  (With constants in vector registers the compiler copies each before it adds to it.)
LCE_DEV double fma_scalar(double a, double b, double c) {
  double r;
  asm("v_fma_f64 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "s"(c));
  return r;
}
// 2^t for -2000 <= t <= 0: 2^(t - rint t) by the polynomial of degree 10 whose largest relative error over half a unit to either side is
// smallest (2.1e-16; 2^0 is 1), times a power of two.
LCE_DEV double exp2_poly(double t) {
  constexpr double kWhole = 6755399441055744.0;  // 1.5 * 2^52: the sum's last place is 1
  const double m = t + kWhole, x = t - (m - kWhole);
  double p = 7.037278846726901e-09;
  p = fma_scalar(p, x, 1.0208537929657404e-07);
  p = fma_scalar(p, x, 1.3215662835959238e-06);
  p = fma_scalar(p, x, 1.5252658116409854e-05);
  p = fma_scalar(p, x, 0.00015403529961127076);
  p = fma_scalar(p, x, 0.0013333558228561767);
  p = fma_scalar(p, x, 0.009618129108034596);
  p = fma_scalar(p, x, 0.05550410866445883);
  p = fma_scalar(p, x, 0.24022650695908768);
  p = fma_scalar(p, x, 0.6931471805599497);
  p = fma(p, x, 1.0);
  return ldexp(p, (int)(unsigned)__builtin_bit_cast(u64, m));
}

// Weights of a row as fixed-point numbers.
struct Weights {
  double top, per;  // the largest value, log2(e) / temperature
  double one;       // 2^bits, bits <= 50
  double least;     // -bits - 1 - 2^-10
  LCE_DEV double log2_of(float z) const {
    // (equal infinities have no difference, and one times 0, at an infinite temperature, is no number)
    const double zd = (double)z;
    return zd == top ? 0.0 : fmax((zd - top) * per, -2000.0);
  }
  // The same for a finite top, without a bound below; and whether such an element can have a weight at all: one above half a place
  // rounds to one, and what is below by more than the series may be off is left out without a look at it.
  LCE_DEV double log2_below(float z) const { return ((double)z - top) * per; }
  LCE_DEV bool may_weigh(double log2) const { return log2 >= least; }
  LCE_DEV double real(float z) const { return exp2_poly(log2_of(z)); }
  // (rounded by the sum with 2^52, whose last place is 1)
  LCE_DEV u64 fixed(double w) const { return __builtin_bit_cast(u64, fma(w, one, 4503599627370496.0)) & 0xfffffffffffffull; }
  LCE_DEV u64 of(float z) const { return fixed(real(z)); }
};
struct NoWeights {
  LCE_DEV u64 of(float) const { return 0; }
};

template <bool WEIGHTED> struct Histogram;
template <> struct Histogram<false> {
  int count[kDigits];
};
template <> struct Histogram<true> {
  u64 weight[kDigits];
  int count[kDigits];
};
LCE_DEV int digit_of(unsigned key, int level) { return level == 0 ? key >> 21 : level == 1 ? (key >> 10) & 2047 : key & 1023; }
LCE_DEV bool in_prefix(unsigned key, unsigned prefix, int level) {
  return level == 0 || (level == 1 ? (key ^ prefix) >> 21 == 0 : (key ^ prefix) >> 10 == 0);
}

// Histogram of the digit `level` over the elements that agree with `prefix` in the digits before it.  WEIGHTED: elements without
// a weight, which are never drawn, are left out.  Ends with a barrier.
template <bool WEIGHTED, class E, int NT, int FL, class W>
LCE_DEV void fill_histogram(const RowUnits<E, NT, FL>& row, const W& weights, unsigned prefix, int level, Histogram<WEIGHTED>* h) {
  for (int i = thread(); i < kDigits; i += NT) {
    h->count[i] = 0;
    if constexpr (WEIGHTED) h->weight[i] = 0;
  }
  __syncthreads();
  row.elements([&](float z) {
    const unsigned key = key_of(z);
    if (!in_prefix(key, prefix, level)) return;
    if constexpr (WEIGHTED) {
      const u64 w = key == kLowKey ? 0 : weights.of(z);
      if (w == 0) return;
      atomicAdd(&h->weight[digit_of(key, level)], w);
    }
    atomicAdd(&h->count[digit_of(key, level)], 1);
  });
  __syncthreads();
}

// A place in the order: the key there, and how many elements and what weight come before the first of that key.
struct Place {
  unsigned key;
  int count;
  u64 weight;
  int same;  // elements with the key
};
// KEEP: the first digit's histogram stays for the next place that a row asks for.
template <bool WEIGHTED, bool KEEP> struct SelectShared {
  Histogram<WEIGHTED> first[1], next[KEEP ? 1 : 0];
  LCE_DEV Histogram<WEIGHTED>* of_level(int level) {
    if constexpr (KEEP) return level == 0 ? first : next;
    else return first;
  }
  Place place;
  u64 of_wave[kMostWaves];
  ColumnShared columns;
};

// The histogram of the first digit; returns the weight of the elements with a key of `least` and above.
template <class E, int NT, int FL, class Shared>
LCE_DEV u64 fill_first(const RowUnits<E, NT, FL>& row, const Weights& weights, unsigned least, Shared* sh) {
  Histogram<true>* h = sh->first;
  for (int i = thread(); i < kDigits; i += NT) {
    h->count[i] = 0;
    h->weight[i] = 0;
  }
  __syncthreads();
  u64 mine = 0;
  row.elements([&](float z) {
    const unsigned key = key_of(z);
    if (key == kLowKey) return;
    const u64 w = weights.of(z);
    if (w == 0) return;
    if (key >= least) mine += w;
    atomicAdd(&h->weight[digit_of(key, 0)], w);
    atomicAdd(&h->count[digit_of(key, 0)], 1);
  });
  return block_all<Sum, NT>(mine, sh->of_wave);
}

// What a place is looked for by: the k-th element; the last key with an element before which there is less than `most` weight; the
// first with which there is more than `target`.
enum Wanted { kByCount, kByShare, kByWeight };
struct Want {
  Wanted what;
  int k;
  double most;
  u64 target;
  // whether it is among c elements of weight w behind cb elements of weight wb
  LCE_DEV bool here(int cb, u64 wb, int c, u64 w) const {
    if (what == kByCount) return cb < k && k <= cb + c;
    if (w == 0) return false;
    if (what == kByShare) return (wb == 0 || (double)wb < most) && !((double)(wb + w) < most);
    return wb <= target && target - wb < w;
  }
};

// The place that is wanted.  KEEP: the histogram of the first digit is there (fill_first).
template <bool WEIGHTED, bool KEEP, class E, int NT, int FL, class W>
LCE_DEV Place find_place(const RowUnits<E, NT, FL>& row, const W& weights, SelectShared<WEIGHTED, KEEP>* sh, const Want& want) {
  constexpr int kOwn = kDigits / NT;  // digits of a thread, the largest first
  Place p = {0, 0, 0, 0};
#pragma unroll 1
  for (int level = 0; level < 3; ++level) {
    Histogram<WEIGHTED>* h = sh->of_level(level);
    if (level > 0 || !KEEP) fill_histogram<WEIGHTED>(row, weights, p.key, level, h);
    const int top = kDigits - 1 - kOwn * (int)thread();
    int c = 0;
    u64 w = 0;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      c += h->count[top - i];
      if constexpr (WEIGHTED) w += h->weight[top - i];
    }
    int c_before;
    u64 w_before = 0;
    block_all<Sum, NT>(c, reinterpret_cast<int*>(sh->of_wave), &c_before);
    if (WEIGHTED) block_all<Sum, NT>(w, sh->of_wave, &w_before);
    int cb = p.count + c_before;
    u64 wb = p.weight + w_before;
    const int shift = level == 0 ? 21 : level == 1 ? 10 : 0;
    if (want.here(cb, wb, c, w)) {
#pragma unroll 1
      for (int d = top; d > top - kOwn; --d) {
        const int cd = h->count[d];
        u64 wd = 0;
        if constexpr (WEIGHTED) wd = h->weight[d];
        if (want.here(cb, wb, cd, wd)) sh->place = {p.key | (unsigned)d << shift, cb, wb, cd};
        cb += cd;
        wb += wd;
      }
    }
    __syncthreads();
    p = sh->place;
    __syncthreads();
  }
  return p;
}

// The largest key of the row.
template <class E, int NT, int FL> LCE_DEV unsigned largest_key(const RowUnits<E, NT, FL>& row, unsigned* sh) {
  unsigned top = 0;
  row.elements([&](float z) {
    const unsigned k = key_of(z);
    top = k > top ? k : top;
  });
  return block_all<Largest, NT>(top, sh);
}

// Settings of a row.
struct RowSettings {
  float temperature, top_p, min_p, u;
  int top_k;
  int bits;
  LCE_DEV RowSettings(const Sampling& s, const float* u_, int64_t n, int bits_) : bits(bits_) {
    temperature = uniform(s.temperature_rows ? s.temperature_rows[n] : s.temperature);
    top_p = uniform(s.top_p_rows ? s.top_p_rows[n] : s.top_p);
    min_p = uniform(s.min_p_rows ? s.min_p_rows[n] : s.min_p);
    const int64_t k = s.top_k_rows ? s.top_k_rows[n] : s.top_k;
    top_k = uniform(k < 0 ? 0 : k > 0x7fffffff ? 0x7fffffff : (int)k);
    u = uniform(u_[n]);
  }
  LCE_DEV bool greedy() const { return !(temperature > 0.f) || top_k == 1; }
  LCE_DEV Weights weights(float top) const {
    return {uniform((double)top), uniform(1.4426950408889634074 / (double)temperature), (double)((u64)1 << bits), -1025.0 / 1024.0 - bits};
  }
};

// The place of the token, and which of the place's elements it is, from `find`, which looks up places, the number of elements
// with a weight, the sum of their weights and of those that min_p keeps.
template <class Find, class WeightAt>
LCE_DEV Place draw_place(const RowSettings& s, int counted, u64 all, u64 by_min, Place at, int* which, Find find, WeightAt weight_at) {
  u64 stays = all;
  if (s.min_p > 1.f) by_min = (u64)1 << s.bits;  // (the first column alone)
#pragma unroll 1
  for (int step = kByCount; step <= kByWeight; ++step) {
    if (step == kByCount && !(s.top_k > 0 && s.top_k < counted)) continue;
    if (step == kByShare && !(s.top_p < 1.f)) continue;
    Want want = {(Wanted)step, s.top_k, (double)s.top_p * (double)stays, 0};
    if (step == kByWeight) {
      if (by_min < stays) stays = by_min;
      const double some = (double)s.u * (double)stays;
      want.target = some > 0.0 ? (u64)some : 0;
      if (want.target >= stays) want.target = stays - 1;
    }
    at = find(want);
    u64 w = weight_at(at);
    w = w == 0 ? 1 : w;  // (not of an element that was counted)
    if (step == kByCount) {
      stays = at.weight + (u64)(s.top_k - at.count) * w;
    } else if (step == kByShare) {
      const double some = (want.most - (double)at.weight) / (double)w;
      int kept = some > 0.0 ? (some < (double)at.same ? (int)some : at.same) : 0;
      if (kept < at.same && (double)(at.weight + (u64)kept * w) < want.most) ++kept;  // (`some` rounded down)
      if (at.weight == 0 && kept == 0) kept = 1;
      const u64 by_p = at.weight + (u64)kept * w;
      if (by_p < stays) stays = by_p;
    } else {
      // the whole part of the quotient, which is below at.same: by a double and a look at what it leaves
      const u64 rest = want.target - at.weight;
      int whole = (int)((double)rest / (double)w);
      if ((u64)whole * w > rest) --whole;
      else if (rest - (u64)whole * w >= w) ++whole;
      *which = whole;
    }
  }
  return at;
}

// The token of a row by digits, any type; -1 where there is none.
template <class E, int NT, int FL, bool KEEP>
LCE_DEV int sample_by_digits(const RowUnits<E, NT, FL>& row, const RowSettings& s, SelectShared<true, KEEP>* sh) {
  const unsigned top = largest_key(row, reinterpret_cast<unsigned*>(sh->of_wave));
  if (top == kNanKey || top == kLowKey) return -1;  // a NaN, or no column left
  Place at = {top, 0, 0, 0};
  int which = 0;
  if (thread() == 0) sh->place = at;
  if (!s.greedy()) {
    const Weights weights = s.weights(value_of(top));
    // the smallest key that min_p keeps: the weights are monotone in the keys
    unsigned least = top;
    if (s.min_p > 0.f) {
      unsigned lo = kLowKey;  // (`least` has such a weight: the first column always stays)
      while (least - lo > 1) {
        const unsigned mid = lo + (least - lo) / 2;
        if (weights.real(value_of(mid)) >= (double)s.min_p) least = mid;
        else lo = mid;
      }
    }
    const u64 by_min = fill_first(row, weights, s.min_p > 0.f ? least : 0, sh);
    u64 w = 0;
    int c = 0;
    const int t = thread();
#pragma unroll
    for (int i = 0; i < kDigits / NT; ++i) {
      w += sh->first->weight[i * NT + t];
      c += sh->first->count[i * NT + t];
    }
    const u64 all = block_all<Sum, NT>(w, sh->of_wave);
    const int counted = block_all<Sum, NT>(c, reinterpret_cast<int*>(sh->of_wave));
    at = draw_place(s, counted, all, by_min, at, &which,
                    [&](const Want& want) { return find_place<true, KEEP>(row, weights, sh, want); },
                    [&](const Place& p) { return weights.of(value_of(p.key)); });
  }
  return column_of<FL == 4 ? 8 : 2>(RowPieces<E, NT>(row.p, row.n), value_of(at.key), which, &sh->columns);
}

constexpr int kMostTop = 1024;

// An entry of a list that is sorted: by key, the larger first, then by column.
LCE_DEV u64 entry_of(unsigned key, int column) { return (u64)~key << 32 | (u64)column; }
LCE_DEV unsigned key_in(u64 entry) { return ~(unsigned)(entry >> 32); }
LCE_DEV int column_in(u64 entry) { return (int)(entry & 0xffffffffu); }

// A bitonic network over list[0 .. sorted), a power of two from 2 on; up to 128 entries by one wave, without barriers in between.
// Starts and ends with a barrier.
template <int NT> LCE_DEV void sort_list(u64* list, int sorted) {
  __syncthreads();
  const bool one_wave = sorted <= 128;
  if (!one_wave || thread() < 64) {
#pragma unroll 1
    for (int size = 2; size <= sorted; size <<= 1)
#pragma unroll 1
      for (int d = size >> 1; d > 0; d >>= 1) {
        for (int t = thread(); t < sorted / 2; t += NT) {
          const int i = ((t & ~(d - 1)) << 1) | (t & (d - 1)), j = i | d;  // the t-th pair
          const u64 a = list[i], b = list[j];
          if ((a > b) == ((i & size) == 0)) {
            list[i] = b;
            list[j] = a;
          }
        }
        if (one_wave) {
          __threadfence_block();
          __builtin_amdgcn_wave_barrier();
        } else {
          __syncthreads();
        }
      }
  }
  __syncthreads();
}
// The same into `to` for any number of entries up to kMostRanked, by counting for each those before it.  Starts and ends with a barrier.
constexpr int kMostRanked = 512;
template <int NT> LCE_DEV const u64* rank_list(const u64* list, u64* to, int n) {
  __syncthreads();
  for (int t = thread(); t < n; t += NT) {
    const u64 mine = list[t];
    int rank = 0;
    int j = 0;
#pragma unroll 1
    for (; j + 8 <= n; j += 8) {
#pragma unroll
      for (int q = 0; q < 8; ++q) rank += list[j + q] < mine ? 1 : 0;
    }
#pragma unroll 1
    for (; j < n; ++j) rank += list[j] < mine ? 1 : 0;
    to[rank] = mine;
  }
  __syncthreads();
  return to;
}
LCE_DEV int power_of_two(int n) {
  int p = 2;
  while (p < n) p <<= 1;
  return p;
}
// The first k of the list to memory.
template <class E, int NT, int FL> LCE_DEV void store_top(const RowUnits<E, NT, FL>& row, const u64* list, int k, E* values, int64_t* index) {
  for (int i = thread(); i < k; i += NT) {
    int column = column_in(list[i]);
    column = (unsigned)column < (unsigned)row.n ? column : row.n - 1;  // (logits that change under the kernel must not lead it astray)
    index[i] = column;
    values[i] = row.p[column];
  }
}

// sum exp(z - m) of a row, the same bits from 512 and from 1024 threads: a thread adds up the pieces of one (or, apart, of two) of 1024
// places, in fp32 up to kTerms of them (a row of 131072), those sums and the waves' in doubles, in the order of the places.  A term equal to
// m is 1, also of an infinite m.
template <class E, int NT> struct ExpSum {
  static constexpr int kOwn = 1024 / NT, kPer = RowPieces<E, NT>::kPer;
  static constexpr int kFlight = RowPieces<E, NT>::kFlight, kTerms = 128, kRounds = kTerms / kPer * kOwn / kFlight;
  float m, sum[kOwn];
  double total[kOwn];
  int rounds;
  LCE_DEV explicit ExpSum(float m_) : m(m_), rounds(0) {
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      sum[i] = 0.f;
      total[i] = 0.0;
    }
  }
  template <bool FINITE> LCE_DEV float term(float z) const {
    // (one fma of z and m log2 e would do, but for logits of 10^30, where the product's rounding is no small number)
    const float e = __builtin_amdgcn_exp2f((z - m) * 1.4426950408889634f);
    return FINITE || z != m ? e : 1.f;
  }
  template <bool FINITE> LCE_DEV void edge(float z) { sum[0] += term<FINITE>(z); }
  // r: which of its round
  template <bool FINITE> LCE_DEV void piece(u32x4_t v, int r) {
    E e[kPer];
    __builtin_memcpy(e, &v, 16);
#pragma unroll
    for (int i = 0; i < kPer; ++i) sum[r % kOwn] += term<FINITE>(as_float(e[i]));
    if (r == kFlight - 1 && ++rounds % kRounds == 0) {
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        total[i] += (double)sum[i];
        sum[i] = 0.f;
      }
    }
  }
  // 16 sums; no barrier.
  LCE_DEV void store(double* sums) const {
    const int t = thread();
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      const double upto = wave_upto<Sum>(total[i] + (double)sum[i]);
      if ((t & 63) == 63) sums[i * (NT / 64) + (t >> 6)] = upto;
    }
  }
};
LCE_DEV float log_sum(float m, const double* sums) {
  double all = 0.0;
#pragma unroll
  for (int w = 0; w < 16; ++w) all += sums[w];
  return (float)((double)m + log(all));
}

// The first k of a row by digits, any type.  list: kMostTop entries; sums: 16.
template <class E, int NT, int FL>
LCE_DEV void top_by_digits(const RowUnits<E, NT, FL>& row, int k, E* values, int64_t* index, float* lse, SelectShared<false, false>* sh, u64* list,
                           int* listed, double* sums) {
  if (lse != nullptr) {
    const unsigned top = largest_key(row, reinterpret_cast<unsigned*>(sh->of_wave));
    const float m = top == kNanKey ? __builtin_nanf("") : value_of(top);
    const RowPieces<E, NT> pieces(row.p, row.n);
    ExpSum<E, NT> sum(m);
    pieces.edges([&](int at, unsigned) { sum.template edge<false>(as_float(row.p[at])); });
    pieces.each([&](int, u32x4_t v, int r) { sum.template piece<false>(v, r); });
    sum.store(sums);
    __syncthreads();
    if (thread() == 0) *lse = top == kLowKey ? m : log_sum(m, sums);
  }
  const Place p = find_place<false, false>(row, NoWeights(), sh, Want{kByCount, k, 0.0, 0});
  // what is larger, in any order, and the first k - p.count of the key in the order of the columns
  const int sorted = power_of_two(k), t = thread(), lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  if (t == 0) *listed = 0;
  for (int i = t; i < sorted; i += NT) list[i] = ~(u64)0;
  __syncthreads();
  int mine = 0;
  row.each([&](int unit, u32x4_t v, int c) {
    row.elements(v, c, [&](int i, float z) {
      const unsigned key = key_of(z);
      if (key > p.key) {
        const int to = atomicAdd(listed, 1);  // (p.count of them)
        if (to < kMostTop) list[to] = entry_of(key, row.column(unit) + i);
      }
      mine += key == p.key ? 1 : 0;
    });
  });
  const int upto = wave_upto<Sum>(mine);
  if (lane == 63) sh->columns.of_wave[wave] = upto;
  __syncthreads();
  const int want = k - p.count;
  int before = 0;
  for (int w = 0; w < wave; ++w) before += sh->columns.of_wave[w];
  if (sh->columns.of_wave[wave] > 0 && before < want) {
    row.each([&](int unit, u32x4_t v, int c) {
      int here = 0;
      row.elements(v, c, [&](int, float z) { here += key_of(z) == p.key ? 1 : 0; });
      const int of_unit = wave_upto<Sum>(here);
      int at = before + of_unit - here;
      row.elements(v, c, [&](int i, float z) {
        if (key_of(z) != p.key) return;
        if (at < want) list[p.count + at] = entry_of(p.key, row.column(unit) + i);
        ++at;
      });
      before += read_lane(of_unit, 63);
    });
  }
  sort_list<NT>(list, sorted);
  store_top(row, list, k, values, index);
  __syncthreads();
}

// ---------------------------------------------------------------------------------------------------------------------------
// The first k, k up to kMostByMaxima, without a histogram: of the largest element of each thread, the k-th is a lower bound of the k-th
// of the row, and about -M ln(1 - k / M) elements of M maxima are not below it: these are listed and sorted.  M is 1024 for rows of 1024 pieces
// of 16 bytes and more (32 elements for k = 32, 710 for 512), the number of pieces below that; where k is not well below it, the list
// overflows, in 16-bit rows of 2049 to some 4300 with k from an eighth of the row's length on.  Two passes over the row, one that
// takes maxima, one that compares (and sums the exponentials for lse).  Where many of the maxima equal the bound -- all but a few
// columns masked, or one value almost everywhere -- only what is larger is listed, and the first columns of that value are added.  Rows whose list
// would be too long all the same, with a NaN or an infinity on top are done by digits.  (All but 10 columns masked, k = 32, us, here / by
// digits: a row of 32000 bf16 11 / 72, 2048 of them 48 / 391; what the question costs other rows is half a microsecond.)
// ---------------------------------------------------------------------------------------------------------------------------
constexpr int kMostByMaxima = 512, kMostList = 2048, kMaxima = 1024, kMostTied = 256;
// Digits: the shared memory of the rows that are done by digits.
template <class Digits> struct TopShared {
  union {
    struct {
      Digits digits;
      u64 by_digits[kMostTop];  // (the list of top_by_digits)
    };
    struct {
      u64 list[kMostList];
      unsigned maxima[kMaxima];
    };
  };
  u64 of_wave[kMostWaves];
  int at_least[2][kMostWaves];
  double sums[kMostWaves];
  unsigned top;
  int listed, drawn;
};

// Adds to the `listed` entries of the list those of the first elements, in the order of the columns, with ordered bits from `from` up to but not
// with `above`, until there are k.  Returns how many there are.  A block's scan for each piece of a thread: the value is a frequent one.
template <class E, int NT, class Shared>
LCE_DEV int list_ties(const RowPieces<E, NT>& row, unsigned from, unsigned above, int listed, int k, Shared* sh) {
  typedef Ordered<E> O;
  typedef typename bits_of<sizeof(E)>::type Bits;
  constexpr int kPer = RowPieces<E, NT>::kPer, kHalves = 4 / sizeof(E);
  const int t = thread(), tail = row.n - row.head - row.body * kPer;
  auto in = [&](unsigned a) { return a >= from && a < above; };
  auto put = [&](int place, unsigned a, int column) {
    if (place < k) sh->list[place] = entry_of(key_of(O::value(a)), column);
  };
  auto edge = [&](int first, int n) {
    const unsigned w = O::word(reinterpret_cast<const Bits*>(row.p)[first + (t < n ? t : 0)]), a = sizeof(E) == 2 ? w & 0xffffu : w;
    const bool is = t < n && in(a);
    int before;
    const int all = block_all<Sum, NT>(is ? 1 : 0, reinterpret_cast<int*>(sh->of_wave), &before);
    if (is) put(listed + before, a, first + t);
    listed += all;
  };
  if (row.head > 0) edge(0, row.head);
#pragma unroll 1
  for (int base = 0; base < row.body && listed < k; base += NT) {
    const bool there = base + t < row.body;
    const int piece = there ? base + t : 0;
    u32x4_t v = reinterpret_cast<const u32x4_t*>(row.p + row.head)[piece];
    int mine = 0;
    auto each = [&](auto f) {
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
        const unsigned a = O::word(v[0]);
        f(i * kHalves, sizeof(E) == 2 ? a & 0xffffu : a);
        if (kHalves == 2) f(i * kHalves + 1, a >> 16);
        v = u32x4_t{v[1], v[2], v[3], v[0]};
      }
    };
    each([&](int, unsigned a) { mine += there && in(a) ? 1 : 0; });
    int before;
    const int all = block_all<Sum, NT>(mine, reinterpret_cast<int*>(sh->of_wave), &before);
    int place = listed + before;
    if (mine != 0 && place < k)
      each([&](int i, unsigned a) {
        if (in(a)) put(place++, a, row.head + piece * kPer + i);
      });
    listed += all;
  }
  if (tail > 0 && listed < k) edge(row.n - tail, tail);
  return listed < k ? listed : k;
}

// The sorted list of a row's first elements, k of them and more; null if it could not be made.  sh->top: the ordered bits of the
// largest element; sh->sums: by waves, sum exp(z - max) of the row (LSE).
template <class E, bool LSE, int NT, class Shared> LCE_DEV const u64* list_first(const RowPieces<E, NT>& row, int k, Shared* sh) {
  typedef Ordered<E> O;
  constexpr int kOwn = kMaxima / NT, kWaves = NT / 64;  // maxima of a thread: of every kOwn-th piece
  const int t = thread(), lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  unsigned most[kOwn] = {}, least = ~0u;
  row.edges([&](int, unsigned a) {
    most[0] = O::larger(most[0], a);  // (of 16 bits: the upper half stays as it is)
    least = O::smaller(least, sizeof(E) == 2 ? a | 0xffff0000u : a);
  });
  row.each([&](int, u32x4_t v, int r) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const unsigned a = O::word(v[i]);
      most[r % kOwn] = O::larger(most[r % kOwn], a);
      least = O::smaller(least, a);
    }
  });
  unsigned largest = 0;
#pragma unroll
  for (int i = 0; i < kOwn; ++i) {
    most[i] = O::largest(most[i]);
    sh->maxima[i * NT + t] = O::in_top_bits(most[i]);
    largest = most[i] > largest ? most[i] : largest;
  }
  if (O::smallest(least) < O::kLow) largest = ~0u;  // (a NaN is above +inf or below -inf)
  if (t == 0) sh->listed = sh->drawn = 0;
  const unsigned top = block_all<Largest, NT>(largest, reinterpret_cast<unsigned*>(sh->of_wave));
  if (top >= O::kInf || top <= O::kLow) return nullptr;
  // the largest number, of 16 bits, that k maxima are not below: some bits at a time, a wave for each of their values
  constexpr int kBits = kWaves == 16 ? 4 : 3;
  static_assert(kWaves == 1 << kBits, "a wave to a value");
  unsigned of[kMaxima / 64];
#pragma unroll
  for (int i = 0; i < kMaxima / 64; ++i) of[i] = sh->maxima[i * 64 + lane];
  unsigned bound = 0;
  int buffer = 0;
#pragma unroll 1
  for (int shift = 15 / kBits * kBits; shift >= 0; shift -= kBits, buffer ^= 1) {
    const unsigned mid = bound | (unsigned)wave << shift;
    int count = 0;
#pragma unroll
    for (int i = 0; i < kMaxima / 64; ++i) count += __popcll(__ballot(of[i] >= mid));
    if (lane == 0) sh->at_least[buffer][wave] = count;
    __syncthreads();
    const u64 enough = __ballot(sh->at_least[buffer][lane & (kWaves - 1)] >= k);  // (of value 0 there are: all that the bits before left)
    bound |= (unsigned)(63 - __clzll((long long)((enough & ((1u << kWaves) - 1)) | 1))) << shift;
  }
  if (bound == 0x8000u) bound = 0x7fffu;  // (-0 is 0)
  const unsigned from = O::from_top_bits(bound);
  // (the numbers that may equal it: of float32 those of the same upper half, which has to be found out)
  const unsigned group = bound == 0x7fffu ? 0x8000u : bound, above = O::from_top_bits(group + 1);
  int in_group = 0;
#pragma unroll
  for (int i = 0; i < kMaxima / 64; ++i) in_group += __popcll(__ballot(of[i] >= bound && of[i] <= group));
  const bool tied = in_group > kMostTied;
  const unsigned limit = tied ? above : from;
  unsigned tied_most = 0, tied_inverse = 0;  // float32: the largest key of those that may be equal, of the inverted keys
  auto tie = [&](unsigned a) {
    if (sizeof(E) == 4 && tied && a >= from && a < above) {
      const unsigned key = key_of(O::value(a));
      tied_most = key > tied_most ? key : tied_most;
      tied_inverse = ~key > tied_inverse ? ~key : tied_inverse;
    }
  };
  const float m = O::value(top);
  ExpSum<E, NT> sum(m);
  auto add = [&](int at, unsigned a) {
    if (a >= limit) {
      const int to = atomicAdd(&sh->listed, 1);
      if (to < kMostList) sh->list[to] = entry_of(key_of(O::value(a)), at);
    }
  };
  row.edges([&](int at, unsigned a) {
    add(at, a);
    tie(a);
    if (LSE) sum.template edge<true>(O::value(a));
  });
  row.each([&](int at, u32x4_t v, int r) {
    unsigned best = 0;
    u32x4_t a;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[i] = O::word(v[i]);
      best = O::larger(best, a[i]);
    }
    if (sizeof(E) == 4 && tied) {
#pragma unroll
      for (int i = 0; i < 4; ++i) tie(a[i]);
    }
    if (O::largest(best) >= limit) {
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
        if (sizeof(E) == 2) {
          add(at + 2 * i, a[0] & 0xffffu);
          add(at + 2 * i + 1, a[0] >> 16);
        } else {
          add(at + i, a[0]);
        }
        a = u32x4_t{a[1], a[2], a[3], 0};
      }
    }
    if (LSE) sum.template piece<true>(v, r);
  });
  if (LSE) sum.store(sh->sums);
  if (t == 0) sh->top = top;
  __syncthreads();
  int listed = sh->listed;
  bool fits = listed <= kMostList;
  if (fits && tied && listed < k) {
    if (sizeof(E) == 4) {
      tied_most = block_all<Largest, NT>(tied_most, reinterpret_cast<unsigned*>(sh->of_wave));
      tied_inverse = block_all<Largest, NT>(tied_inverse, reinterpret_cast<unsigned*>(sh->of_wave));
      fits = tied_most == ~tied_inverse;
    }
    if (fits) listed = list_ties<E, NT>(row, from, above, listed, k, sh);
  }
  if (!fits) {
    __syncthreads();  // (the caller may use the place of it all)
    return nullptr;
  }
  // (by ranks n^2 comparisons, by the network n log^2 n and a barrier each round)
  if (listed <= kMostRanked) return rank_list<NT>(sh->list, sh->list + kMostRanked, listed);
  const int sorted = power_of_two(listed);
  for (int i = listed + t; i < sorted; i += NT) sh->list[i] = ~(u64)0;
  sort_list<NT>(sh->list, sorted);
  return sh->list;
}

// Bound for long rows by memory traffic and vector work beside each other (2048 rows of 50257 bf16 64 us, 3.2 TB/s of one reading; 2048 of
// 131072 float32 317, 3.4; 8192 of 50257 bf16 234 with the vector units 81 % busy; both readings go beyond the L2s), by the latency of its
// steps for short ones: 48 rows of 50304 12 us, of which 3 read and 2 look for the bound, 5 list and sum, 1 sorts.
//   NT = 512: 64 registers a thread and little LDS, four rows to a compute unit, of which some are read while others are sorted; 1024 where
// each row has a compute unit to itself.  us, 512 / 1024: top_logits, 64 rows, V=4096 bf16 7.7 / 7.8, float32 7.7 / 8.4, 50257 bf16
// 13 / 12, 131072 21 / 19, float32 25 / 20; 256 rows, 131072 29 / 27, float32 42 / 42; 400 rows, 50257 21 / 25, 29 / 34.  sample_top_kernel,
// 64 rows, 131072 20 / 17, float32 26 / 20; sample_bins_kernel, 64 rows, float32 75 / 58, 256 rows 98 / 84, 400 rows, 50257 61 / 67.
template <class E, bool LSE, int NT>
__global__ __launch_bounds__(NT, NT == 1024 ? 4 : 8) void top_kernel(const E* logits, int64_t rows, int64_t cols, int64_t ld, int k, E* values,
                                                             int64_t* index, float* lse) {
  __shared__ TopShared<SelectShared<false, false>> sh;
  for (int64_t n = blockIdx.x; n < rows; n += gridDim.x) {
    const E* from = logits + n * ld;
    const u64* list = k <= kMostByMaxima ? list_first<E, LSE>(RowPieces<E, NT>(from, cols), k, &sh) : nullptr;
    if (list != nullptr) {
      if (LSE && thread() == NT - 1) lse[n] = log_sum(Ordered<E>::value(sh.top), sh.sums);
      store_top(RowUnits<E, NT>(from, cols), list, k, values + n * k, index + n * k);
      __syncthreads();
    } else {
      top_by_digits(RowUnits<E, NT>(from, cols), k, values + n * k, index + n * k, LSE ? lse + n : nullptr, &sh.digits, sh.by_digits, &sh.listed, sh.sums);
    }
  }
}

// The token of a row whose first k are listed, k of them kept by top_k (1: the first column).
template <int NT, class Shared> LCE_DEV int sample_listed(const RowSettings& s, int k, const u64* list, Shared* sh) {
  if (s.greedy()) {
    const int column = column_in(list[0]);
    __syncthreads();
    return column;
  }
  static_assert(kMostByMaxima <= NT, "an entry to a thread");
  const Weights weights = s.weights(value_of(key_in(list[0])));
  const int t = thread();
  const double real = t < k ? weights.real(value_of(key_in(list[t]))) : 0.0;
  const u64 w = weights.fixed(real);
  u64 before;
  u64 stays = block_all<Sum, NT>(w, sh->of_wave, &before);
  const double most = (double)s.top_p * (double)stays;
  // (each keeps a beginning of the list: the weight of those that all keep is their sum)
  const bool kept = t < k && (t == 0 || ((!(s.top_p < 1.f) || (double)before < most) && (!(s.min_p > 0.f) || real >= (double)s.min_p)));
  stays = block_all<Sum, NT>(kept ? w : (u64)0, sh->of_wave);
  const double some = (double)s.u * (double)stays;
  u64 target = some > 0.0 ? (u64)some : 0;
  if (target >= stays) target = stays - 1;
  if (w != 0 && before <= target && target - before < w) sh->drawn = t;  // (one thread)
  __syncthreads();
  const int at = sh->drawn;
  const int column = column_in(list[at]);
  __syncthreads();
  return column;
}

// Rows of which the first elements are enough: settings for all of them with 1 <= top_k <= kMostByMaxima or temperature 0.
template <class E, int NT>
__global__ __launch_bounds__(NT, NT == 1024 ? 4 : 8) void sample_top_kernel(const E* logits, int64_t rows, int64_t cols, int64_t ld, const float* u,
                                                                    const Sampling settings, int bits, int64_t* token) {
  __shared__ TopShared<SelectShared<true, false>> sh;
  for (int64_t n = blockIdx.x; n < rows; n += gridDim.x) {
    const E* from = logits + n * ld;
    const RowSettings s(settings, u, n, bits);
    const int k = s.greedy() ? 1 : s.top_k < cols ? s.top_k : (int)cols;
    const u64* list = list_first<E, false>(RowPieces<E, NT>(from, cols), k, &sh);
    int column;
    if (list != nullptr) column = sample_listed<NT>(s, k, list, &sh);
    else column = sample_by_digits(RowUnits<E, NT, 2>(from, cols), s, &sh.digits);  // (64 registers: no more in flight)
    if (thread() == 0) token[n] = column;
    __syncthreads();
  }
}

constexpr int kSelectThreads = 1024;

// ---------------------------------------------------------------------------------------------------------------------------
// Rows with any settings.  A histogram of counts and weights over 4096 bins of equal width in log2 of the weight, which is what
// the fixed point of the weights reaches; the few elements of the bin in which a place lies are then listed and sorted.  Passes over the
// row: its maximum, the histogram, one for every place that is asked for.  A bin with more elements than the list has room for is
// no matter if they are all equal; else the row is done by digits.
//   Bound by the vector work of the weights, 24 of 42 instructions for an element, most of them of 64 bits: 2048 rows of 32000 fp16 116 us,
// the vector units 65 % busy; of a row's 25 us the histogram takes 11, the place 7, the maximum, from memory, 5.
// ---------------------------------------------------------------------------------------------------------------------------
constexpr int kBins = 4096;
constexpr double kBinsPerOctave = 80.0;  // 51 octaves and 2^-10: a weight of 2^-51 rounds to 0 with 50 places
static_assert(51 * 80 + 1 < kBins);
struct BinShared {
  union {
    struct {
      u64 weight[kBins];
      int count[kBins];
      u64 list[kMostList];
    };
    SelectShared<true, true> digits;
  };
  u64 of_wave[kMostWaves];
  ColumnShared columns;
  Place place;
  int column;
  int bin, listed;
};
template <class E, int NT> struct RowBins {
  typedef Ordered<E> O;
  static constexpr int kPer = RowPieces<E, NT>::kPer, kOwn = kBins / NT;
  const RowPieces<E, NT>& row;
  const Weights& weights;
  unsigned top;  // the largest key
  BinShared* sh;

  LCE_DEV static int bin_of(double log2_weight) {
    return (int)(log2_weight * -kBinsPerOctave);  // (<= 51 * 80)
  }
  // The histogram (of weights, and of counts if they are `counted`); the weight that min_p keeps.
  LCE_DEV u64 fill(double min_p, bool counted) const {
    for (int i = thread(); i < kBins; i += NT) {
      sh->count[i] = 0;
      sh->weight[i] = 0;
    }
    __syncthreads();
    u64 mine = 0;
    auto one = [&](float z) {
      const double t = weights.log2_below(z);
      if (!weights.may_weigh(t)) return;
      const double real = exp2_poly(t);
      const u64 w = weights.fixed(real);
      const int b = bin_of(t);
      atomicAdd(&sh->weight[b], w);
      if (counted) atomicAdd(&sh->count[b], w != 0 ? 1 : 0);
      if (min_p > 0.0) {
        asm volatile("");  // (a branch)
        if (real >= min_p) mine += w;
      }
    };
    row.edges([&](int at, unsigned) { one(as_float(row.p[at])); });
    row.each([&](int, u32x4_t v, int) {
      E e[kPer];
      __builtin_memcpy(e, &v, 16);
#pragma unroll
      for (int i = 0; i < kPer; ++i) one(as_float(e[i]));
    });
    __syncthreads();
    return min_p > 0.0 ? block_all<Sum, NT>(mine, sh->of_wave) : 0;
  }
  // The sums of this thread's bins.
  LCE_DEV void own(int* c, u64* w) const {
    const int first = thread() * kOwn;
    *c = 0;
    *w = 0;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) {
      *c += sh->count[first + i];
      *w += sh->weight[first + i];
    }
  }
  // The place that is wanted; *column: its column, where it is one element's, else -1.  c, w: the sums of this thread's bins, cb, wb: those
  // before.  False: by digits.
  LCE_DEV bool find(int cb, u64 wb, int c, u64 w, const Want& want, Place* place, int* column) const {
    const int t = thread();
    if (t == 0) sh->listed = 0;
    if (want.here(cb, wb, c, w)) {
#pragma unroll 1
      for (int b = t * kOwn; b < (t + 1) * kOwn; ++b) {
        const int cd = sh->count[b];
        const u64 wd = sh->weight[b];
        if (want.here(cb, wb, cd, wd)) {
          sh->bin = b;
          sh->place = {0, cb, wb, 0};
        }
        cb += cd;
        wb += wd;
      }
    }
    __syncthreads();
    const Place bin = sh->place;
    const int b = sh->bin;
    // values between which all of its elements are: the bin's ends, each further out by more than the roundings of either direction -- some
    // 2^-52 of the distance to the top, whose share is large next to 0, and of the top itself, and those to float32
    const double low_off = (double)(b + 1) / (kBinsPerOctave * weights.per), high_off = (double)b / (kBinsPerOctave * weights.per);
    const double eps = 1.0 / (1ull << 49), some = fabs(weights.top) * eps;
    const double low_z = weights.top - low_off - (low_off * eps + some), high_z = weights.top - high_off + (high_off * eps + some);
    const unsigned low_key = key_of((float)low_z), high_key = key_of((float)high_z);
    const float low = uniform(value_of(low_key < kLowKey + 4 ? kLowKey + 1 : low_key - 2));
    const float high = uniform(value_of(high_key < top - 2 ? high_key + 2 : top));
    unsigned most = 0, inverse = 0;  // the largest key of the bin, of the inverted keys
    auto one = [&](int at, float z) {
      if (!(z >= low && z <= high)) return;
      const double log2 = weights.log2_below(z);
      if (!weights.may_weigh(log2) || bin_of(log2) != b) return;  // (some without a weight do no harm: they come last)
      const unsigned key = key_of(z);
      const int to = atomicAdd(&sh->listed, 1);
      if (to < kMostList) sh->list[to] = entry_of(key, at);
      most = key > most ? key : most;
      inverse = ~key > inverse ? ~key : inverse;
    };
    row.edges([&](int at, unsigned) { one(at, as_float(row.p[at])); });
    row.each([&](int at, u32x4_t v, int) {
      E e[kPer];
      __builtin_memcpy(e, &v, 16);
      bool any = false;
#pragma unroll
      for (int i = 0; i < kPer; ++i) any |= as_float(e[i]) >= low && as_float(e[i]) <= high;
      if (any) RowUnits<E, NT>::elements(v, kPer, [&](int i, float z) { one(at + i, z); });
    });
    __syncthreads();
    const int in_bin = sh->listed;
    *column = -1;
    if (in_bin > kMostList) {
      most = block_all<Largest, NT>(most, reinterpret_cast<unsigned*>(sh->of_wave));
      inverse = block_all<Largest, NT>(inverse, reinterpret_cast<unsigned*>(sh->of_wave));
      *place = {most, bin.count, bin.weight, in_bin};
      return most == ~inverse;
    }
    const int n = in_bin;
    const u64* list = sh->list;
    if (n <= kMostRanked) {
      list = rank_list<NT>(sh->list, sh->list + kMostRanked, n);
    } else {
      const int sorted = power_of_two(n);
      for (int i = n + t; i < sorted; i += NT) sh->list[i] = ~(u64)0;
      sort_list<NT>(sh->list, sorted);
    }
    // (some neighbouring entries to a thread)
    const int per = (n + NT - 1) / NT;
    u64 mine = 0;
    for (int i = t * per; i < (t + 1) * per && i < n; ++i) mine += weights.of(value_of(key_in(list[i])));
    u64 before;
    block_all<Sum, NT>(mine, sh->of_wave, &before);
    before += bin.weight;
    for (int i = t * per; i < (t + 1) * per && i < n; ++i) {
      const unsigned key = key_in(list[i]);
      const u64 one = weights.of(value_of(key));
      if (want.here(bin.count + i, before, 1, one)) {
        sh->place = {key, bin.count + i, before, 1};
        sh->column = column_in(list[i]);
      }
      before += one;
    }
    __syncthreads();
    *place = sh->place;
    *column = sh->column;
    __syncthreads();
    return true;
  }
};

template <class E, int NT>
LCE_DEV int64_t sample_by_bins(const E* from, int64_t cols, const RowSettings& s, BinShared* sh) {
  const RowPieces<E, NT> row(from, cols);
  const unsigned top = row.largest(reinterpret_cast<unsigned*>(sh->of_wave));
  if (top == kNanKey || top == kLowKey) return -1;  // a NaN, or no column left
  const float inf = __builtin_inff();
  if (s.greedy()) return column_of(row, value_of(top), 0, &sh->columns);
  if (value_of(top) < inf) {
    const Weights weights = s.weights(value_of(top));
    const RowBins<E, NT> bins = {row, weights, top, sh};
    const bool by_count = s.top_k > 0 && s.top_k < row.n;
    const u64 by_min = bins.fill(s.min_p > 0.f ? (double)s.min_p : 0.0, by_count);
    int c, cb = 0;
    u64 w, wb;
    bins.own(&c, &w);
    const int counted = by_count ? block_all<Sum, NT>(c, reinterpret_cast<int*>(sh->of_wave), &cb) : 0;
    const u64 all = block_all<Sum, NT>(w, sh->of_wave, &wb);
    if (thread() == 0) {
      sh->place = {top, 0, 0, 0};
      sh->bin = 0;
      sh->column = 0;
    }
    __syncthreads();
    bool fine = true;
    int which = 0, column = -1;
    const Place at = draw_place(s, counted, all, s.min_p > 0.f ? by_min : all, Place{top, 0, 0, 0}, &which,
                                [&](const Want& want) {
                                  Place p = {top, 0, 0, 0};
                                  if (fine) fine = bins.find(cb, wb, c, w, want, &p, &column);
                                  return p;
                                },
                                [&](const Place& p) { return weights.of(value_of(p.key)); });
    if (fine) return column >= 0 ? column : column_of(row, value_of(at.key), which, &sh->columns);
    __syncthreads();
  }
  return sample_by_digits(RowUnits<E, NT>(from, cols), s, &sh->digits);
}

// (NT: as in top_kernel; two rows to a compute unit, or one)
template <class E, int NT>
__global__ __launch_bounds__(NT, 4) void sample_bins_kernel(const E* logits, int64_t rows, int64_t cols, int64_t ld, const float* u,
                                                            const Sampling settings, int bits, int64_t* token) {
  __shared__ union {
    BinShared bins;
    TopShared<SelectShared<true, true>> top;
  } sh;
  for (int64_t n = blockIdx.x; n < rows; n += gridDim.x) {
    const E* from = logits + n * ld;
    const RowSettings s(settings, u, n, bits);
    const int k = s.greedy() ? 1 : s.top_k;
    const u64* list = nullptr;
    if (k >= 1 && k <= kMostByMaxima && k < cols) list = list_first<E, false>(RowPieces<E, NT>(from, cols), k, &sh.top);
    int column;
    if (list != nullptr) column = sample_listed<NT>(s, k, list, &sh.top);
    else column = sample_by_bins<E, NT>(from, cols, s, &sh.bins);
    if (thread() == 0) token[n] = column;
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------------------------------------------------------
// 16-bit rows with any settings.  A row has at most 65536 different values, and a histogram of all of them fits the LDS of a
// compute unit, with 16 bits a count.  Counts are what a row is read for; weights are worked out for each value that occurs, not for
// each element, and places found without another look at the row.
//   A word has the counts of the numbers +m (lower half) and -m (upper half), m its index: the bits of the magnitude.  0 and -0 are
// one value.  Columns masked by -inf or the type's lowest number, which may be most of a row, would meet in one word: they are
// counted apart.  A count beyond 65535 overflows into the other half of its word or is lost; either way the sum of all counts is short,
// and the row, like one with a NaN or with nothing but masked columns, is done by digits.
//   The values that occur are then listed in the order of the row, over the histogram, and a thread has a stretch of the list.
//   Bound by latencies, the passes by LDS atomics and the caches: a row of 131072 bf16 28 us, of which the histogram 9, its reading and the
// list 6, weights and places 4, the drawn value's column 7; 256 such rows 39 us, the two passes 11 each.
// ---------------------------------------------------------------------------------------------------------------------------
template <class E> struct HalfFormat;
template <> struct HalfFormat<__bf16> { static constexpr unsigned kInf = 0x7f80; };
template <> struct HalfFormat<_Float16> { static constexpr unsigned kInf = 0x7c00; };
template <class E> LCE_DEV float half_value(unsigned bits) { return (float)__builtin_bit_cast(E, (unsigned short)bits); }

constexpr int kHalfWords = 32768;
constexpr int kWordRows = kHalfWords / 256;  // 256 words: four to a lane
struct HalfShared {
  union {
    unsigned hist[kHalfWords];
    unsigned values[kHalfWords];  // the values that occur, in order: bits, and the count in the upper half
    TopShared<SelectShared<true, true>> top;
    ColumnShared columns;
  };
  int row_values[2 * kWordRows], row_first[2 * kWordRows];  // of the positive numbers by rows from the last one, of the negative ones
  u64 of_wave[kMostWaves];
  Place place;  // (its key: the bits)
};

template <class E> struct HalfRow {
  static constexpr unsigned kInf = HalfFormat<E>::kInf, kMax = kInf - 1;
  HalfShared* sh;

  // The counts of the row's values, listed.  Returns whether the list has all of the row's columns that are not masked; *different: how
  // many values it has, *any_masked: whether there are masked columns.
  LCE_DEV bool fill(const RowPieces<E, kSelectThreads>& row, int* different, bool* any_masked) const {
    constexpr int kWordRounds = kHalfWords / 4 / kSelectThreads;
    const int t = thread(), lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    u32x4_t* words = reinterpret_cast<u32x4_t*>(sh->hist);
#pragma unroll
    for (int i = 0; i < kWordRounds; ++i) words[i * kSelectThreads + t] = u32x4_t{};
    __syncthreads();
    int masked = 0;
    bool nan = false;
    auto one = [&](unsigned bits) {
      const unsigned m = bits & 0x7fffu;
      if (m > kInf) nan = true;
      else if (m >= kMax && (bits & 0x8000u)) ++masked;
      else atomicAdd(&sh->hist[m], bits & 0x8000u ? 0x10000u : 1u);
    };
    row.edges([&](int at, unsigned) { one(reinterpret_cast<const unsigned short*>(row.p)[at]); });
    row.each([&](int, u32x4_t w, int) {
      typedef unsigned short pair_t __attribute__((ext_vector_type(2)));
      pair_t most = {};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned m = w[i] & 0x7fff7fffu;
        most = __builtin_elementwise_max(most, __builtin_bit_cast(pair_t, m));
      }
      if (most[0] >= kMax || most[1] >= kMax) {
        u64 some = (u64)w[1] << 32 | w[0];
        const u64 rest = (u64)w[3] << 32 | w[2];
#pragma unroll 1
        for (int e = 0; e < 8; ++e) {
          one((unsigned)some & 0xffffu);
          some = e == 3 ? rest : some >> 16;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          atomicAdd(&sh->hist[w[i] & 0x7fffu], 1u << ((w[i] >> 11) & 16));
          atomicAdd(&sh->hist[(w[i] >> 16) & 0x7fffu], 1u << ((w[i] >> 27) & 16));
        }
      }
    });
    const bool any_nan = __syncthreads_or(nan);
    // the counts leave the histogram, whose place the list takes
    u32x4_t w[kWordRounds];
    u64 sum = 0;
#pragma unroll
    for (int i = 0; i < kWordRounds; ++i) {
      w[i] = words[i * kSelectThreads + t];
#pragma unroll
      for (int j = 0; j < 4; ++j) sum += (w[i][j] & 0xffffu) + (w[i][j] >> 16);
    }
    if (t == 0) {  // 0 and -0
      w[0][0] = (w[0][0] & 0xffffu) + (w[0][0] >> 16);
      if (w[0][0] > 0xffffu) --sum;  // (a count that is too large, as any other)
    }
    u64 who[2][4];
    auto occur = [&](u32x4_t some) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        who[0][j] = __ballot((some[j] & 0xffffu) != 0);
        who[1][j] = __ballot(some[j] >> 16 != 0);
      }
    };
#pragma unroll
    for (int i = 0; i < kWordRounds; ++i) {
      const int at = i * (kSelectThreads / 64) + wave;
      int plus = 0, minus = 0;
      if (__any((w[i][0] | w[i][1] | w[i][2] | w[i][3]) != 0)) {
        occur(w[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          plus += __popcll(who[0][j]);
          minus += __popcll(who[1][j]);
        }
      }
      if (lane == 0) {
        sh->row_values[kWordRows - 1 - at] = plus;
        sh->row_values[kWordRows + at] = minus;
      }
    }
    const u64 both = block_all<Sum, kSelectThreads>(sum | (u64)masked << 31, sh->of_wave);
    const u64 counted = both & 0x7fffffffu;
    *any_masked = both >> 31 != 0;
    int before;
    *different = block_all<Sum, kSelectThreads>(t < 2 * kWordRows ? sh->row_values[t] : 0, reinterpret_cast<int*>(sh->of_wave), &before);
    if (any_nan || counted == 0 || *different > kHalfWords || (int)(counted + (both >> 31)) != row.n) return false;
    if (t < 2 * kWordRows) sh->row_first[t] = before;
    __syncthreads();
    const u64 above = ~(u64)0 << lane << 1, below = ~(~(u64)0 << lane);
#pragma unroll
    for (int i = 0; i < kWordRounds; ++i) {
      if (!__any((w[i][0] | w[i][1] | w[i][2] | w[i][3]) != 0)) continue;
      occur(w[i]);
      const int at = i * (kSelectThreads / 64) + wave;
      int plus = sh->row_first[kWordRows - 1 - at], minus = sh->row_first[kWordRows + at];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        plus += __popcll(who[0][j] & above);
        minus += __popcll(who[1][j] & below);
      }
      const unsigned m = (unsigned)(i * kSelectThreads + t) * 4;
#pragma unroll
      for (int j = 3; j >= 0; --j)
        if ((w[i][j] & 0xffffu) != 0) sh->values[plus++] = (m + j) | w[i][j] << 16;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (w[i][j] >> 16 != 0) sh->values[minus++] = (m + j) | 0x8000u | (w[i][j] & 0xffff0000u);
    }
    __syncthreads();
    return true;
  }

  // f(bits, count) for the values of this thread's stretch of the list.
  template <class F> LCE_DEV void stretch(int different, F f) const {
    const int per = (different + kSelectThreads - 1) / kSelectThreads, first = (int)thread() * per;
    const int end = first + per < different ? first + per : different;
#pragma unroll 1
    for (int i = first; i < end; ++i) f(sh->values[i] & 0xffffu, (int)(sh->values[i] >> 16));
  }

  // The place that is wanted.  cb, wb: elements and weight before this thread's stretch; c, w: its own.
  LCE_DEV Place find(const Weights& weights, int different, int cb, u64 wb, int c, u64 w, const Want& want) const {
    __syncthreads();
    if (want.here(cb, wb, c, w)) {
      bool found = false;
      stretch(different, [&](unsigned bits, int count) {
        if (found) return;
        const u64 each = weights.of(half_value<E>(bits));
        const int n_here = each != 0 ? count : 0;
        if (want.here(cb, wb, n_here, each * (u64)n_here)) {
          sh->place = {bits, cb, wb, n_here};
          found = true;
        }
        cb += n_here;
        wb += each * (u64)n_here;
      });
    }
    __syncthreads();
    return sh->place;
  }
};

template <class E>
__global__ __launch_bounds__(kSelectThreads) void sample_half_kernel(const E* logits, int64_t rows, int64_t cols, int64_t ld, const float* u,
                                                                     const Sampling settings, int bits, int64_t* token) {
  extern __shared__ __attribute__((aligned(16))) char lds[];
  HalfShared* sh = reinterpret_cast<HalfShared*>(lds);
  for (int64_t n = blockIdx.x; n < rows; n += gridDim.x) {
    const E* from = logits + n * ld;
    const RowSettings s(settings, u, n, bits);
    const RowPieces<E, kSelectThreads> row(from, cols);
    const HalfRow<E> half = {sh};
    const int k = s.greedy() ? 1 : s.top_k;
    const u64* list = nullptr;
    if (k >= 1 && k <= kMostByMaxima && k < cols) list = list_first<E, false>(row, k, &sh->top);
    int column;
    int different = 0;
    bool masked = false;
    bool filled = list == nullptr && !s.greedy() && half.fill(row, &different, &masked);
    const unsigned top = filled ? sh->values[0] & 0xffffu : 0;
    const Weights weights = s.weights(half_value<E>(top));
    // (at a temperature that leaves the lowest number a weight it masks nothing)
    if (filled && masked && weights.of(half_value<E>(0x8000u | HalfRow<E>::kMax)) != 0) filled = false;
    if (list != nullptr) {
      column = sample_listed<kSelectThreads>(s, k, list, &sh->top);
    } else if (filled) {
      const double min_p = s.min_p > 0.f ? (double)s.min_p : 0.0;
      u64 weight = 0, by_min = 0;
      int elements = 0;
      half.stretch(different, [&](unsigned value, int c) {
        const double real = weights.real(half_value<E>(value));
        const u64 w = weights.fixed(real);
        if (w != 0) elements += c;
        weight += w * (u64)c;
        if (real >= min_p) by_min += w * (u64)c;
      });
      int cb;
      u64 wb;
      const int weighed = block_all<Sum, kSelectThreads>(elements, reinterpret_cast<int*>(sh->of_wave), &cb);
      const u64 all = block_all<Sum, kSelectThreads>(weight, sh->of_wave, &wb);
      by_min = s.min_p > 0.f ? block_all<Sum, kSelectThreads>(by_min, sh->of_wave) : all;
      int which = 0;
      const Place at = draw_place(s, weighed, all, by_min, Place{top, 0, 0, 0}, &which,
                                  [&](const Want& want) { return half.find(weights, different, cb, wb, elements, weight, want); },
                                  [&](const Place& p) { return weights.of(half_value<E>(p.key)); });
      __syncthreads();  // (the list of values is not read any more)
      column = column_of(row, half_value<E>(at.key), which, &sh->columns);
    } else {
      __syncthreads();
      column = sample_by_digits(RowUnits<E, kSelectThreads>(from, cols), s, &sh->top.digits);
    }
    if (thread() == 0) token[n] = column;
    __syncthreads();
  }
}

// Workgroups: one for a row (65536 rows of 1000 bf16, us, one for each / 1024 that take one row after another: top_logits 494 / 612,
// sampling by bins 1307 / 1380; 4096 rows of 32000 80 / 87, 223 / 240), up to a number that a launch can have.
unsigned grid_of(int64_t rows) { return (unsigned)(rows < (int64_t)1 << 22 ? rows : (int64_t)1 << 22); }
// The two passes over the first elements, four workgroups to a compute unit, are bound by memory: where so many rows are more than the
// 256 MiB Infinity Cache holds, as many workgroups as it has room for, so that the second pass finds them there (1500 rows of 131072
// float32 249 us, 512 at a time 228; 1024 rows of 262144 bf16 180, 165).
unsigned grid_of_top(int64_t rows, int64_t row_bytes, int num_cus) {
  const int64_t cached = ((int64_t)256 << 20) / row_bytes;
  if (cached >= (int64_t)4 * num_cus) return grid_of(rows);
  const int64_t n = cached < num_cus ? num_cus : cached;
  return (unsigned)(rows < n ? rows : n);
}
// The histogram of all values: a workgroup to a compute unit, whose code and constants are at hand for its next row (4096 rows of 32000
// bf16 260 us, by 512 workgroups 252).
unsigned grid_of_half(int64_t rows, int num_cus) { return (unsigned)(rows < (int64_t)2 * num_cus ? rows : (int64_t)2 * num_cus); }
static_assert(sizeof(HalfShared) <= 160 * 1024, "a compute unit has 160 KiB of LDS");

// 16-bit rows up to this, or half of it where there is no more than one for each compute unit, are sampled by bins, longer ones by the
// histogram of all values: that takes a compute unit for a row, much of its time whatever the row's length, and more for fp16, of which a
// row has more different values.  us, bins / histogram, temperature alone and with top_p:
//   2048 rows   bf16 V=4096 52/97, 76/109; 16384 87/117, 120/127; 24000 113/124, 147/135; 32768 138/130, 181/141
//               fp16 V=16384 85/159, 115/180; 32768 133/178, 171/203; 50257 183/195, 226/219; 65536 222/206, 277/237
//   64 rows     bf16 V=8192 14/16, 20/18; 16384 18/17, 25/18; 32768 27/18, 36/20
//               fp16 V=8192 14/20, 19/23; 16384 18/22, 24/25; 24000 22/23, 30/27; 32768 26/25, 34/28
template <class E> constexpr int64_t kMostBinCols = 16384;
template <> constexpr int64_t kMostBinCols<_Float16> = 32768;

template <class E>
hipError_t launch_sample_of(const E* logits, int64_t rows, int64_t cols, int64_t ld, const float* u, const Sampling& s, int bits, int64_t* token,
                            int num_cus, hipStream_t stream) {
  const int64_t row_bytes = cols * (int64_t)sizeof(E);
  const bool first_alone = (!s.temperature_rows && s.temperature == 0.f) || (!s.top_k_rows && s.top_k >= 1 && s.top_k <= kMostByMaxima);
  if (first_alone) {
    if (rows <= num_cus)
      hipLaunchKernelGGL((sample_top_kernel<E, 1024>), dim3((unsigned)rows), dim3(1024), 0, stream, logits, rows, cols, ld, u, s, bits, token);
    else
      hipLaunchKernelGGL((sample_top_kernel<E, 512>), dim3(grid_of_top(rows, row_bytes, num_cus)), dim3(512), 0, stream, logits, rows, cols, ld,
                         u, s, bits, token);
    return hipGetLastError();
  }
  if constexpr (sizeof(E) == 2) {
    if (cols > (rows > num_cus ? kMostBinCols<E> : kMostBinCols<E> / 2)) {
      static LdsOptIn optin;
      const hipError_t e = optin.ensure(reinterpret_cast<const void*>(sample_half_kernel<E>), (int)sizeof(HalfShared));
      if (e != hipSuccess) return e;
      hipLaunchKernelGGL(sample_half_kernel<E>, dim3(grid_of_half(rows, num_cus)), dim3(kSelectThreads), sizeof(HalfShared), stream,
                         logits, rows, cols, ld, u, s, bits, token);
      return hipGetLastError();
    }
  }
  if (rows <= num_cus)
    hipLaunchKernelGGL((sample_bins_kernel<E, 1024>), dim3((unsigned)rows), dim3(1024), 0, stream, logits, rows, cols, ld, u, s, bits, token);
  else
    hipLaunchKernelGGL((sample_bins_kernel<E, 512>), dim3(grid_of(rows)), dim3(512), 0, stream, logits, rows, cols, ld, u, s, bits, token);
  return hipGetLastError();
}

template <class E>
hipError_t launch_top_of(const E* logits, int64_t rows, int64_t cols, int64_t ld, int k, E* values, int64_t* index, float* lse, int num_cus,
                         hipStream_t stream) {
  const dim3 grid(rows <= num_cus ? (unsigned)rows : grid_of_top(rows, cols * (int64_t)sizeof(E), num_cus));
#define LCE_TOP(LSE, NT) hipLaunchKernelGGL((top_kernel<E, LSE, NT>), grid, dim3(NT), 0, stream, logits, rows, cols, ld, k, values, index, lse)
  if (rows <= num_cus && lse != nullptr) LCE_TOP(true, 1024);
  else if (rows <= num_cus) LCE_TOP(false, 1024);
  else if (lse != nullptr) LCE_TOP(true, 512);
  else LCE_TOP(false, 512);
#undef LCE_TOP
  return hipGetLastError();
}

}  // namespace

hipError_t launch_sample(const void* logits, int dtype, int64_t rows, int64_t cols, int64_t ld, const float* u, const Sampling& s,
                         int64_t* token, int num_cus, hipStream_t stream) {
  int log2 = 0;
  while ((int64_t)1 << log2 < cols) ++log2;
  const int bits = 62 - log2 < 50 ? 62 - log2 : 50;  // (a double has 53: a weight of one and the half that rounds it fit)
  if (dtype == DT_BF16) return launch_sample_of((const __bf16*)logits, rows, cols, ld, u, s, bits, token, num_cus, stream);
  if (dtype == DT_F16) return launch_sample_of((const _Float16*)logits, rows, cols, ld, u, s, bits, token, num_cus, stream);
  if (dtype == DT_F32) return launch_sample_of((const float*)logits, rows, cols, ld, u, s, bits, token, num_cus, stream);
  return hipErrorInvalidValue;
}

hipError_t launch_top(const void* logits, int dtype, int64_t rows, int64_t cols, int64_t ld, int k, void* values, int64_t* index, float* lse,
                      int num_cus, hipStream_t stream) {
  if (dtype == DT_BF16) return launch_top_of((const __bf16*)logits, rows, cols, ld, k, (__bf16*)values, index, lse, num_cus, stream);
  if (dtype == DT_F16) return launch_top_of((const _Float16*)logits, rows, cols, ld, k, (_Float16*)values, index, lse, num_cus, stream);
  if (dtype == DT_F32) return launch_top_of((const float*)logits, rows, cols, ld, k, (float*)values, index, lse, num_cus, stream);
  return hipErrorInvalidValue;
}

}  // namespace lce

// Distillation from a teacher's top logits: what the loss against soft targets needs besides the kernels of the loss itself.
//
//   z[n][v] = s sum_h x[n][h] W[h][v],  s = logit_scale / temperature,  lse[n] = log sum_v exp z[n][v]
//   q[n][k] = softmax over the entries of row n of (teacher logit / temperature)
//   loss    = 1/R sum_n (lse[n] + sum_k q[n][k] (log q[n][k] - z[n][index[n][k]])),  R = rows with an entry
//   dz[n][v] = softmax(z[n])[v] - sum of q[n][k] over the k with index[n][k] = v
//
// lse, the softmax and the two contractions of dz are those of the loss against labels, and so are their kernels: a row's first
// entry serves as its label, a row without an entry has none.  Here are the pieces that know of more than one target: the teacher's
// distribution (soft_targets_kernel), the student's logits at its columns (soft_logits_kernel, soft_pick_kernel), the loss from both, and the
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

// The student's logits at the teacher's columns, in fp32 from operands of the compute type: z[e] = s x[n] . W[:, v] for every entry
// e = (n, v).
//
// Few entries: a wave per entry.  A weight stored (H, V) then costs a line of 128 bytes for every element, which is what bounds it
// (N=16384, K=64, H=2048: 31.7 ms).
template <class XT, class WT, bool WVH>
__global__ __launch_bounds__(256) void soft_logits_direct_kernel(const SoftLogits a) {
  const int lane = threadIdx.x & 63;
  for (int64_t e = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); e < a.N * a.K; e += (int64_t)gridDim.x * 4) {
    const int v = a.index[e];
    float z = 0.f;
    if (v >= 0 && v < a.V) {
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

// More: the entries are sorted by groups of 64 columns (one line of a 16-bit W), whose part of W then passes through LDS once for
// all of them.  Counting sort: counts of every group, their prefix sums and from them the list of work items -- up to kItemEntries
// entries of one group --, then the places.  The order within a group is not the same in every call; a logit does not depend on it.
constexpr int kGroupCols = 64, kItemEntries = 128;
constexpr int kSortThreads = 1024, kSortPer = 8;
// Whether so many entries are sorted.  The sort and the passes over the groups cost 20 us and the part of W that has an entry; without, a
// weight stored (H, V) costs a line for every element.  Loss alone, us, sorted / not: (H, V), bf16, V=32000, H=128 8192 entries 48 / 42,
// 16384 56 / 58, 32768 69 / 87; H=512 4096 59 / 59, 8192 69 / 87; H=2048 2048 99 / 103, 4096 117 / 153; V=131072, H=2048 2048 229 /
// 207, 8192 410 / 526; fp32, V=32000, H=512 4096 91 / 92, 8192 118 / 147.  (V, H), V=32000, H=512 32768 120 / 101, 65536 188 / 178;
// H=2048 65536 521 / 522; V=4096, H=2048 32768 140 / 104, 65536 163 / 169.
inline bool sorts_entries(int64_t M, int64_t H, bool w_vh) { return w_vh ? M >= 65536 : M * H >= (int64_t)3 << 20; }
constexpr int64_t kMostColGroups = 16384;  // counts of a workgroup: 64 KiB of LDS

__global__ __launch_bounds__(kSortThreads) void soft_clear_kernel(int* counts, int groups) {
  const int i = blockIdx.x * kSortThreads + threadIdx.x;
  if (i < groups) counts[i] = 0;
}

__global__ __launch_bounds__(kSortThreads) void soft_count_kernel(const int* index, int64_t M, int* counts, int groups) {
  extern __shared__ int sh_count[];
  for (int g = threadIdx.x; g < groups; g += kSortThreads) sh_count[g] = 0;
  __syncthreads();
  const int64_t e0 = (int64_t)blockIdx.x * kSortThreads * kSortPer + threadIdx.x;
#pragma unroll
  for (int i = 0; i < kSortPer; ++i) {
    const int64_t e = e0 + i * kSortThreads;
    const int v = e < M ? index[e] : -1;
    if (v >= 0 && v / kGroupCols < groups) atomicAdd(&sh_count[v / kGroupCols], 1);
  }
  __syncthreads();
  for (int g = threadIdx.x; g < groups; g += kSortThreads)
    if (sh_count[g] != 0) atomicAdd(&counts[g], sh_count[g]);
}

// One workgroup: counts[] becomes its own exclusive prefix sum, items[] the list of work items (column group, first entry, entries),
// *num_items their number.
__global__ __launch_bounds__(kSortThreads) void soft_items_kernel(int* counts, int groups, int4* items, int* num_items) {
  __shared__ int sh_entries[kSortThreads / 64], sh_items[kSortThreads / 64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int entries_before = 0, items_before = 0;
  for (int g0 = 0; g0 < groups; g0 += kSortThreads) {
    const int g = g0 + threadIdx.x;
    const int n = g < groups ? counts[g] : 0, m = (n + kItemEntries - 1) / kItemEntries;
    int en = n, it = m;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int ue = __shfl_up(en, d), ui = __shfl_up(it, d);
      if (lane >= d) {
        en += ue;
        it += ui;
      }
    }
    if (lane == 63) {
      sh_entries[wave] = en;
      sh_items[wave] = it;
    }
    __syncthreads();
    int be = entries_before, bi = items_before;
    for (int w = 0; w < kSortThreads / 64; ++w) {
      if (w < wave) {
        be += sh_entries[w];
        bi += sh_items[w];
      }
      entries_before += sh_entries[w];
      items_before += sh_items[w];
    }
    __syncthreads();
    const int first = be + en - n, item = bi + it - m;
    if (g < groups) counts[g] = first;
    for (int i = 0; i < m; ++i) {
      const int left = n - i * kItemEntries;
      items[item + i] = make_int4(g, first + i * kItemEntries, left < kItemEntries ? left : kItemEntries, 0);
    }
  }
  if (threadIdx.x == 0) num_items[0] = items_before;
}

// entries[place] = (e, column); place: counts[group] and up, in stretches that a workgroup takes for its own entries.
__global__ __launch_bounds__(kSortThreads) void soft_place_kernel(const int* index, int64_t M, int* counts, int groups, int2* entries) {
  extern __shared__ int sh_count[];
  for (int g = threadIdx.x; g < groups; g += kSortThreads) sh_count[g] = 0;
  __syncthreads();
  const int64_t e0 = (int64_t)blockIdx.x * kSortThreads * kSortPer + threadIdx.x;
  int v[kSortPer], rank[kSortPer];
#pragma unroll
  for (int i = 0; i < kSortPer; ++i) {
    const int64_t e = e0 + i * kSortThreads;
    v[i] = e < M ? index[e] : -1;
    if (v[i] / kGroupCols >= groups) v[i] = -1;
    if (v[i] >= 0) rank[i] = atomicAdd(&sh_count[v[i] / kGroupCols], 1);
  }
  __syncthreads();
  for (int g = threadIdx.x; g < groups; g += kSortThreads)
    if (sh_count[g] != 0) sh_count[g] = atomicAdd(&counts[g], sh_count[g]);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSortPer; ++i)
    if (v[i] >= 0) entries[sh_count[v[i] / kGroupCols] + rank[i]] = make_int2((int)(e0 + i * kSortThreads), v[i]);
}

// a . b over the elements of 16 bytes, on top of c.
template <class XT> LCE_DEV float dot16(u32x4_t a, u32x4_t b, float c);
template <> LCE_DEV float dot16<__bf16>(u32x4_t a, u32x4_t b, float c) {
  typedef __bf16 pair_t __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned ai = a[i], bi = b[i];
    c = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(pair_t, ai), __builtin_bit_cast(pair_t, bi), c, false);
  }
  return c;
}
template <> LCE_DEV float dot16<_Float16>(u32x4_t a, u32x4_t b, float c) {
  typedef _Float16 pair_t __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned ai = a[i], bi = b[i];
    c = __builtin_amdgcn_fdot2(__builtin_bit_cast(pair_t, ai), __builtin_bit_cast(pair_t, bi), c, false);
  }
  return c;
}
template <> LCE_DEV float dot16<float>(u32x4_t a, u32x4_t b, float c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const unsigned ai = a[i], bi = b[i];
    c = fmaf(__builtin_bit_cast(float, ai), __builtin_bit_cast(float, bi), c);
  }
  return c;
}

// to[0 .. n) = from[0 .. n) in the compute type, zeros from `valid` on.  from + n lies in the matrix where valid >= n; there the
// address is one of 16 bytes.
template <class XT, class WT, int n> LCE_DEV void load_as(XT (&to)[n], const WT* from, int64_t valid) {
  if (valid >= n) {
    WT raw[n];
    constexpr int kPer = 16 / sizeof(WT);
#pragma unroll
    for (int i = 0; i < n / kPer; ++i) {
      const u32x4_t v = reinterpret_cast<const u32x4_t*>(from)[i];
      __builtin_memcpy(raw + i * kPer, &v, 16);
    }
#pragma unroll
    for (int i = 0; i < n; ++i) to[i] = (XT)raw[i];
  } else {
#pragma unroll
    for (int i = 0; i < n; ++i) to[i] = i < valid ? (XT)from[i] : (XT)0.f;
  }
}

// A workgroup per item: the 64 columns of W come through LDS 128 bytes of each at a time (64 or 32 hidden indices), and eight lanes
// take such a stretch of one entry's row of x, a whole line, against the entry's column: 32 entries at a time, four times.  The
// column's line is read by eight neighbouring lanes, which meets every bank once.
//   Bound by memory traffic: 2 H bytes (4 in fp32) for every entry and W once for every 128 entries of a group, from the caches where
// they fit.  N=16384, K=64, H=2048, V=131072, 0.9 million entries: 623 us, 3.7 GB of x and 2.1 of W through the L2s, 3.8 of it from beyond
// them; with 256 entries to an item 841 (registers leave fewer workgroups to hide the waits), 512 1295, 64 882, neighbouring items on
// different XCDs 690, the next lines of x in flight during the products 791.  N=2048, K=64, H=2048, V=16384 in fp32 142, with 256
// entries 134; N=8192, K=32, H=768, V=50257 stored (V, H) 49 / 65; N=1999, K=20, H=500, V=10007 23 / 41.
template <class XT, class WT, bool WVH>
__global__ __launch_bounds__(256) void soft_logits_kernel(const SoftLogits a, const int4* items, const int* num_items, const int2* entries) {
  constexpr int kPiece = 16 / sizeof(XT), kDeep = 8 * kPiece;  // elements of a lane's piece, of a stretch
  constexpr int kSets = kItemEntries / 32;
  __shared__ __attribute__((aligned(16))) XT tile[2][kGroupCols * kDeep];
  // (neighbouring items, of one group, go to one XCD, whose L2 then has the group's part of W)
  const int n_items = num_items[0], per = (n_items + 7) / 8, seq = (int)(blockIdx.x >> 3), id = (int)(blockIdx.x & 7) * per + seq;
  if (seq >= per || id >= n_items) return;
  const int4 item = items[id];
  const int t = threadIdx.x, j = t & 7;
  const XT* x[kSets];
  int column[kSets];
  float z[kSets];
#pragma unroll
  for (int g = 0; g < kSets; ++g) {
    const int at = g * 32 + (t >> 3);
    const int2 e = entries[item.y + (at < item.z ? at : 0)];
    x[g] = reinterpret_cast<const XT*>(a.x) + e.x / a.K * a.ldx + j * kPiece;
    column[g] = (e.y & (kGroupCols - 1)) * kDeep + j * kPiece;
    z[g] = 0.f;
  }
  const WT* w = reinterpret_cast<const WT*>(a.w);
  const int64_t v0 = (int64_t)item.x * kGroupCols;
  // (V, H): thread = quarter of a column's stretch; (H, V): thread = eight columns of one or two hidden indices
  constexpr int kRows = kDeep / 32, kOfW = WVH ? kDeep / 4 : 8;
  XT part[WVH ? 1 : kRows][kOfW];
  auto fetch = [&](int64_t h0) {
    if constexpr (WVH) {
      const int64_t v = v0 + (t >> 2), h = h0 + (t & 3) * kOfW;
#pragma unroll
      for (int i = 0; i < kOfW; i += kPiece) {
        XT some[kPiece];
        load_as<XT, WT, kPiece>(some, w + v * a.ldw + h + i, v < a.V ? a.H - h - i : 0);
#pragma unroll
        for (int u = 0; u < kPiece; ++u) part[0][i + u] = some[u];
      }
    } else {
      const int64_t v = v0 + (t >> 5) * 8;
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const int64_t h = h0 + (t & 31) * kRows + r;
        load_as<XT, WT, 8>(part[r], w + h * a.ldw + v, h < a.H ? a.V - v : 0);
      }
    }
  };
  fetch(0);
  auto take = [&](int64_t h0, u32x4_t (&to)[kSets]) {
#pragma unroll
    for (int g = 0; g < kSets; ++g)
      if (g * 32 < item.z) {
        XT some[kPiece];
        load_as<XT, XT, kPiece>(some, x[g] + h0, a.H - h0 - j * kPiece);
        __builtin_memcpy(&to[g], some, 16);
      }
  };
  u32x4_t piece[kSets];
  int buffer = 0;
  for (int64_t h0 = 0; h0 < a.H; h0 += kDeep, buffer ^= 1) {
    take(h0, piece);
    if constexpr (WVH) {
#pragma unroll
      for (int i = 0; i < kOfW; i += kPiece) {
        u32x4_t v;
        __builtin_memcpy(&v, &part[0][i], 16);
        *reinterpret_cast<u32x4_t*>(&tile[buffer][(t >> 2) * kDeep + (t & 3) * kOfW + i]) = v;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        XT both[kRows];
#pragma unroll
        for (int r = 0; r < kRows; ++r) both[r] = part[r][i];
        unsigned v;
        __builtin_memcpy(&v, both, 4);
        *reinterpret_cast<unsigned*>(&tile[buffer][((t >> 5) * 8 + i) * kDeep + (t & 31) * kRows]) = v;
      }
    }
    if (h0 + kDeep < a.H) fetch(h0 + kDeep);
    __syncthreads();  // (the other buffer is written next: by then every wave is past this one's reads of the round before)
#pragma unroll
    for (int g = 0; g < kSets; ++g)
      if (g * 32 < item.z) z[g] = dot16<XT>(piece[g], *reinterpret_cast<const u32x4_t*>(&tile[buffer][column[g]]), z[g]);
  }
#pragma unroll
  for (int g = 0; g < kSets; ++g) {
#pragma unroll
    for (int d = 1; d < 8; d <<= 1) z[g] += __shfl_xor(z[g], d);
    const int at = g * 32 + (t >> 3);
    if (j == 0 && at < item.z) a.z[entries[item.y + at].x] = z[g] * a.scale;
  }
}

// A thread per entry of the staged rows, in the stage's order: whether its column lies in the stage, the entry, the row and the
// column from the stage's first on.
LCE_DEV bool staged_entry(const BwdArgs& a, const SoftTargets& t, int64_t* i, int64_t* row, int64_t* rel) {
  const int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
  *row = e / t.K;
  if (*row >= packed_rows(a.n_rows, a.N)) return false;
  const int64_t n = a.perm != nullptr ? packed_token(a.perm, *row, t.N) : t.row0 + *row;
  *i = n * t.K + (e - *row * t.K);
  const int64_t v = t.index[*i];
  *rel = v - a.v0;
  return v >= 0 && *rel >= 0 && *rel < a.vw;
}

// The student's logits at the teacher's columns where the stage holds them all, in fp32 (fp32 tensors on one pass): the logits that lse is
// the sum of, so that p = exp(z - lse) is of one arithmetic.  Bound by lines of which it needs 2 bytes, two for an entry (N=2048, K=64:
// two launches of 7 us, where the kernels above take 165).
__global__ __launch_bounds__(256) void soft_pick_kernel(const BwdArgs a, const SoftTargets t) {
  int64_t i, row, rel;
  if (!staged_entry(a, t, &i, &row, &rel)) return;
  const unsigned short* z = reinterpret_cast<const unsigned short*>(a.dz) + 2 * dz_block_offset(row / kTile, rel / 64, a.vs) +
                            (row & (kTile - 1)) * 64 + (rel & 63);
  t.z[i] = a.scale * __builtin_bit_cast(float, (unsigned)z[0] << 16 | z[kDzBlockElems]);
}

// The staged dz at the teacher's columns: 2^shift * (softmax - q), rounded once.
// Bound by the partial lines that it writes: 64 to 128 bytes of memory traffic per entry.
template <class T>
__global__ __launch_bounds__(256) void soft_gradient_kernel(const BwdArgs a, const SoftTargets t) {
  int64_t i, row, rel;
  if (!staged_entry(a, t, &i, &row, &rel)) return;
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

// The entries' terms of the loss, q (log q - z + lse), and their sum in doubles, in an order that is fixed: one partial sum to a workgroup,
// or -- FINAL, a single workgroup -- the loss.  A row with an index that is no column makes it NaN.
constexpr int kLossThreads = 1024, kLossGroups = 512;
template <bool FINAL>
__global__ __launch_bounds__(kLossThreads) void soft_loss_kernel(const SoftTargets t, const int64_t* y, const float* lse, int64_t V,
                                                                 const int64_t* n_valid, double* part, float* loss) {
  __shared__ double sh[kLossThreads / 64];
  double sum = 0.0;
  const unsigned M = (unsigned)(t.N * t.K), step = gridDim.x * kLossThreads;
#pragma unroll 4
  for (unsigned e = blockIdx.x * kLossThreads + threadIdx.x; e < M; e += step) {
    const float q = t.q[e];
    if (q != 0.f) sum += (double)(q * (logf(q) + (lse[e / (unsigned)t.K] - t.z[e])));
  }
  for (int64_t n = (int64_t)blockIdx.x * kLossThreads + threadIdx.x; n < t.N; n += step)
    if (y[n] >= V) sum = (double)__builtin_nanf("");
  sum = wave_sum(sum);
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x != 0) return;
  double total = 0.0;
  for (int i = 0; i < kLossThreads / 64; ++i) total += sh[i];
  if (FINAL) loss[0] = (float)(total / (double)n_valid[0]);  // no row with an entry: 0/0 = NaN, as against labels
  else part[blockIdx.x] = total;
}
__global__ __launch_bounds__(64) void soft_loss_sum_kernel(const double* part, int groups, const int64_t* n_valid, float* loss) {
  double sum = 0.0;
  for (int i = threadIdx.x; i < groups; i += 64) sum += part[i];
  sum = wave_sum(sum);
  if (threadIdx.x == 0) loss[0] = (float)(sum / (double)n_valid[0]);
}

// Scratch of the sorted kernels, after `base`: counts, number of items, items, entries -- of as many rows at a time as the scratch has room
// for, some 8.1 bytes an entry: memory that does not grow with N K.  (kSortScratch holds 2 million.  Loss alone, ms, by stretches / all at
// once: N=65536, H=64, V=4096, K=256, 9 of them, 1.61 / 1.58; N=16384, H=512, V=32000, 3, 1.32 / 1.28; N=8192, H=2048, K=512 3.25 / 3.21.)
struct SortPlan {
  bool sorted;
  int groups;
  int64_t rows, most_items;  // of a stretch
  size_t num_items, items, entries, total;
};
SortPlan plan_sort(int64_t N, int K, int64_t H, int64_t V, bool w_vh, size_t room) {
  SortPlan p;
  const int64_t groups = (V + kGroupCols - 1) / kGroupCols;
  auto up = [](size_t v) { return (v + 255) & ~(size_t)255; };
  p.sorted = sorts_entries(N * K, H, w_vh) && groups <= kMostColGroups;
  p.groups = (int)(groups <= kMostColGroups ? groups : 0);
  p.num_items = up((size_t)p.groups * 4);
  p.items = p.num_items + 256;
  auto stretch = [&](int64_t rows) {
    p.rows = rows;
    p.most_items = groups + rows * K / kItemEntries;
    p.entries = p.items + up((size_t)p.most_items * sizeof(int4));
    return p.entries + up((size_t)(rows * K) * sizeof(int2));
  };
  p.total = stretch(N);
  if (room < kSortScratch) room = kSortScratch;
  if (p.sorted && p.total > room) {
    int64_t lo = 1, hi = N;  // (`lo` rows fit)
    while (hi - lo > 1) {
      const int64_t mid = lo + (hi - lo) / 2;
      (stretch(mid) <= room ? lo : hi) = mid;
    }
    stretch(lo);
    p.total = room;
  }
  if (!p.sorted) p.total = 0;
  return p;
}
// A row's entries, the groups' counts and their items fit, so that every plan has a row at least.
static_assert(kMostColGroups * 4 + 256 + (kMostColGroups + kMaxTargets) * 16 + 256 + kMaxTargets * 8 + 256 <= kSortScratch);

template <class XT, class WT, bool WVH> hipError_t launch_logits(const SoftLogits& all, void* ws, size_t room, hipStream_t s) {
  const SortPlan p = plan_sort(all.N, all.K, all.H, all.V, all.w_vh != 0, room);
  if (!p.sorted) {
    const SoftLogits& a = all;
    const int64_t M = a.N * a.K, groups = (M + 3) / 4;
    hipLaunchKernelGGL((soft_logits_direct_kernel<XT, WT, WVH>), dim3((unsigned)(groups < kMostGroups ? groups : kMostGroups)), dim3(256), 0,
                       s, a);
    return hipGetLastError();
  }
  char* base = reinterpret_cast<char*>(ws);
  int* counts = reinterpret_cast<int*>(base);
  int* num_items = reinterpret_cast<int*>(base + p.num_items);
  int4* items = reinterpret_cast<int4*>(base + p.items);
  int2* entries = reinterpret_cast<int2*>(base + p.entries);
  for (int64_t row0 = 0; row0 < all.N; row0 += p.rows) {
    SoftLogits a = all;
    a.N = all.N - row0 < p.rows ? all.N - row0 : p.rows;
    a.x = reinterpret_cast<const XT*>(all.x) + row0 * all.ldx;
    a.index = all.index + row0 * all.K;
    a.z = all.z + row0 * all.K;
    const int64_t M = a.N * a.K;
    const dim3 grid((unsigned)((M + kSortThreads * kSortPer - 1) / (kSortThreads * kSortPer))), block(kSortThreads);
    hipLaunchKernelGGL(soft_clear_kernel, dim3((unsigned)((p.groups + kSortThreads - 1) / kSortThreads)), block, 0, s, counts, p.groups);
    hipLaunchKernelGGL(soft_count_kernel, grid, block, p.groups * 4, s, a.index, M, counts, p.groups);
    hipLaunchKernelGGL(soft_items_kernel, dim3(1), block, 0, s, counts, p.groups, items, num_items);
    hipLaunchKernelGGL(soft_place_kernel, grid, block, p.groups * 4, s, a.index, M, counts, p.groups, entries);
    hipLaunchKernelGGL((soft_logits_kernel<XT, WT, WVH>), dim3((unsigned)((p.most_items + 7) / 8 * 8)), dim3(256), 0, s, a, items, num_items,
                       entries);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
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

size_t soft_logits_bytes(int64_t N, int K, int64_t H, int64_t V, bool w_vh, size_t room) {
  return plan_sort(N, K, H, V, w_vh, room).total;
}

hipError_t launch_soft_logits(const SoftLogits& a, void* ws, size_t room, hipStream_t s) {
  if (a.x_dtype == DT_BF16 && a.w_dtype == DT_BF16)
    return a.w_vh ? launch_logits<__bf16, __bf16, true>(a, ws, room, s) : launch_logits<__bf16, __bf16, false>(a, ws, room, s);
  if (a.x_dtype == DT_BF16 && a.w_dtype == DT_F32)
    return a.w_vh ? launch_logits<__bf16, float, true>(a, ws, room, s) : launch_logits<__bf16, float, false>(a, ws, room, s);
  if (a.x_dtype == DT_F16 && a.w_dtype == DT_F16)
    return a.w_vh ? launch_logits<_Float16, _Float16, true>(a, ws, room, s) : launch_logits<_Float16, _Float16, false>(a, ws, room, s);
  if (a.x_dtype == DT_F16 && a.w_dtype == DT_F32)
    return a.w_vh ? launch_logits<_Float16, float, true>(a, ws, room, s) : launch_logits<_Float16, float, false>(a, ws, room, s);
  if (a.x_dtype == DT_F32 && a.w_dtype == DT_F32 && !a.w_vh) return launch_logits<float, float, false>(a, ws, room, s);
  return hipErrorInvalidValue;
}

hipError_t launch_soft_pick(const BwdArgs& a, const SoftTargets& t, hipStream_t s) {
  const int64_t rows = a.Np < a.N ? a.Np : a.N;
  hipLaunchKernelGGL(soft_pick_kernel, dim3((unsigned)((rows * t.K + 255) / 256)), dim3(256), 0, s, a, t);
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
  const int64_t most = t.N * t.K > t.N ? t.N * t.K : t.N, blocks = (most + 4 * kLossThreads - 1) / (4 * kLossThreads);
  const int grid = (int)(blocks < kLossGroups ? blocks : kLossGroups);
  if (grid <= 4) {  // (a workgroup's rounds are shorter than a second launch)
    hipLaunchKernelGGL(soft_loss_kernel<true>, dim3(1), dim3(kLossThreads), 0, s, t, y, lse, V, n_valid, part, loss);
  } else {
    hipLaunchKernelGGL(soft_loss_kernel<false>, dim3((unsigned)grid), dim3(kLossThreads), 0, s, t, y, lse, V, n_valid, part, loss);
    hipLaunchKernelGGL(soft_loss_sum_kernel, dim3(1), dim3(64), 0, s, part, grid, n_valid, loss);
  }
  return hipGetLastError();
}

int soft_loss_groups() { return kLossGroups; }

}  // namespace lce

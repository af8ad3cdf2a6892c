// A token for every row of logits from a given random number (fa_sample_tokens).
//
// The chain keeps a set of tokens that is always a prefix of the order (logit descending, id ascending): top_k a prefix of k,
// top_p the shortest prefix whose softmax mass reaches p of the top_k's, min_p a bound on the logit. So the set is held as a
// cut (key of the last logit kept, last id kept among its equals), nothing is sorted but the few values near a cut, and the
// draw runs through the vocabulary in its own order.
//
// Weights exp(x - max) are rounded to integers of 2^-S of the largest (S = 62 - ceil(log2 vocab), at most 50), so that sums
// are exact whatever the order in which they are added: results do not depend on the launch shape or on atomics. The
// exponentials are taken in 64 bits, because a sum over 150 000 tokens is compared with borders 7e-6 apart.
//
// A row is cut into chunks of 16 values a thread, one block each, so that a single row still uses many compute units; what
// needs the whole row is done by one block of its own at the end. Four launches at most, two for most settings:
//   k_scan    the chunk's maximum; with a small top_k also every thread's maximum.
//   k_hist    rows with a top_p or a top_k over KMAX: a histogram (count and mass by steps of 1/32 below the maximum); the block
//             that arrives last finds the bins in which the cuts lie. Nothing waits for another block.
//   k_mass    such rows, and rows with neither: each chunk's mass at the temperature; the values in the cuts' bins to a list.
//   k_finish  one block a row. A top_k up to KMAX: the k largest lie in the groups of 16 whose maximum is in the bins that hold k
//             such maxima, so only those groups are read again (a few hundred values). Else: the cut within the list by
//             histograms of its entries, the chunk, the token in it. A row whose cut's bins hold more than CAP values
//             (thousands of equal logits) is finished by narrowing the cut over the row itself (general_row).
//
// Measured (f32, 151936 tokens): one row at top_k 50 k_scan 3.9 us + k_finish 10.3 us, chains of dependent reads and barriers;
// 61 rows with settings of their own, most top_p 0.95: k_scan 9.5 (3.9 TB/s) + k_hist 21.5 + k_mass 15.8 + k_finish 21 us.
// k_hist and k_mass keep the vector units 75 % busy with 64-bit exponentials. With 8 / 24 / 32 values a thread for 16 the 61
// rows take 69 / 74 / 83 us for 68.
#include "api.h"
#include "draft_ops.h"

#include <algorithm>

namespace fa {

constexpr int PER = 16;     // values a thread
constexpr int BINS = 1024;  // of 1 / 32 below the maximum; the last takes everything 32 and more below
constexpr int CAP = 4096;   // values that are sorted
constexpr int ST = 1024;    // threads of k_hist and k_finish
// threads of k_scan and k_mass (f32, top_p, 1 / 64 / 512 rows of 151936: 43 / 75 / 324 us, with 1024 threads 52 / 83 / 354;
// top_k 50: 14 / 20 / 83 and 15 / 23 / 86)
constexpr int SCAN = 256;
constexpr int KMAX = 1024;  // largest top_k that k_finish makes from the threads' maxima

typedef unsigned long long u64;

struct RowState {  // zeroed by k_scan, which leaves the scales
  double inv_t, least;       // 1 / temperature; least logit above the maximum (min_p): once a row, not once a thread
  uint32_t arrived, list_n;
  int b_lo, b_hi, b_k;       // bins of the cut: the listed ones are [b_lo, b_hi] and b_k
  u64 mass_lo, mass_k;       // mass before b_lo / before b_k
  u64 cnt_k;                 // values before b_k
  u64 total;                 // mass of the row
};

struct SampleP {
  fa_sample_args a;
  int S;  // a weight of 1 is 2^S
  int chunks;           // of PER values a thread of k_scan and k_mass
  int hist_chunks;      // k_hist's blocks a row
  FastDiv grid_div;     // blocks a row in this launch
  int grid_chunks;
  int want_max;  // the threads' maxima are wanted (a row may have a small top_k)
  float* cmax;   // [rows][chunks]
  int* cidx;
  u64* cmass;
  u64* hist_mass;  // [rows][BINS]
  uint32_t* hist_cnt;
  u64* list;  // [rows][CAP]
  RowState* state;
  float* tmax;  // [rows][chunks][threads]
};

enum RowKind { GREEDY, SMALL_K, HIST, PLAIN };
struct RowSettings {
  float top_p;
  float t, min_p;
  int top_k;
  bool has_k, has_p;
  RowKind kind;
};
__device__ __forceinline__ RowSettings settings_of(const fa_sample_args& a, int r) {
  RowSettings s;
  // (read unconditionally, from u where there is no array: four loads side by side, not one after the other)
  const float t_r = (a.temperatures ? a.temperatures : a.u)[r], m_r = (a.min_ps ? a.min_ps : a.u)[r];
  const float p_r = (a.top_ps ? a.top_ps : a.u)[r];
  const int32_t k_r = (a.top_ks ? a.top_ks : reinterpret_cast<const int32_t*>(a.u))[r];
  const float t = a.temperatures ? t_r : a.temperature, m = a.min_ps ? m_r : a.min_p;
  s.top_p = a.top_ps ? p_r : a.top_p;
  s.top_k = a.top_ks ? k_r : a.top_k;
  s.has_k = s.top_k > 0 && s.top_k < a.vocab;
  s.has_p = s.top_p < 1.f;
  s.t = t;
  s.min_p = m;
  s.kind = !(t > 0.f) || s.top_k == 1 || !(s.top_p > 0.f) || !(m <= 1.f) ? GREEDY
           : s.has_k && s.top_k <= KMAX                                    ? SMALL_K
           : s.has_k || s.has_p                                            ? HIST
                                                                           : PLAIN;
  return s;
}

__device__ __forceinline__ float clean(float x) {  // NaN -> -inf, -0 -> 0
  x += 0.0f;
  return x != x ? -INFINITY : x;
}
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7FFFFFFFu : ~k); }
// monotone in x; a maximum of inf: everything else in the last bin
__device__ __forceinline__ int bin_of(float x, float top) {
  return x == top ? 0 : (int)fminf((top - x) * 32.f, (float)(BINS - 1));
}
__device__ __forceinline__ double rel_of(float x, float top) { return x == top ? 0.0 : (double)x - (double)top; }
// exp(x) 2^S, rounded to an integer, for x <= 0 and S <= 50: x = n ln 2 + 4 r with |r| <= ln 2 / 8, the Taylor polynomial of
// degree 7 in r (remainder r^8 / 8! < 8e-14 of 1), squared twice: relative error below 4e-13 before the rounding, what a sum
// over a few thousand tokens of equal weight resolves at S = 44. Adding 1.5 2^52 leaves n, adding 2^52 the result, in the low
// bits of a sum: no conversions
__device__ __forceinline__ u64 weight(double x, int S) {
  if (!(x > -60.0)) return 0;  // 2^50 exp(-60) < 1/2 (NaN: -inf times 1 / inf)
  const double t = fma(x, 1.4426950408889634, 0x1.8p52);
  const int n = (int)(uint32_t)__double_as_longlong(t);
  const double nf = t - 0x1.8p52;
  double r = fma(nf, -0x1.62e42fefa39efp-1, x);
  r = fma(nf, -0x1.abc9e3b39803fp-56, r) * 0.25;
  double p = 1.0 / 5040.0;
  p = fma(p, r, 1.0 / 720.0);
  p = fma(p, r, 1.0 / 120.0);
  p = fma(p, r, 1.0 / 24.0);
  p = fma(p, r, 1.0 / 6.0);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  p *= p;
  p *= p;
  const double scale = __longlong_as_double((long long)(n + S + 1023) << 52);  // 2^(n + S), n + S >= -49
  return (u64)__double_as_longlong(fma(p, scale, 0x1p52)) - 0x4330000000000000ull;
}

struct Cut {  // the last value kept
  uint32_t key;
  int idx;
};
__device__ __forceinline__ bool within(uint32_t key, int i, const Cut& c) {
  return key > c.key || (key == c.key && i <= c.idx);
}

// A chunk's values: thread t holds index base + (j * BT + t) * W + w as value j * W + w, W = 16 bytes' worth where the row is
// 16-byte aligned, else 1: coalesced either way, and index order within each j
template <typename T>
struct RowView {
  const T* p;
  int V;
  bool vec;
};
template <typename T>
__device__ __forceinline__ RowView<T> row_view(const fa_sample_args& a, int r) {
  RowView<T> v;
  v.p = reinterpret_cast<const T*>(a.logits) + (int64_t)r * a.row_stride;
  v.V = a.vocab;
  v.vec = (reinterpret_cast<uintptr_t>(v.p) & 15) == 0;
  return v;
}
template <typename T> constexpr int kWide = 16 / (int)sizeof(T);
template <typename T, int BT>
__device__ __forceinline__ int index_at(bool vec, int base, int t, int e) {
  constexpr int W = kWide<T>;
  return vec ? base + ((e / W) * BT + t) * W + e % W : base + e * BT + t;
}
template <typename T, int BT, int N>
__device__ __forceinline__ void load_chunk(const RowView<T>& v, int base, int t, float (&x)[N]) {
  constexpr int W = kWide<T>;
  if (v.vec && base + BT * N <= v.V) {  // a whole chunk: all loads before the first use
    uint4 raw[N / W];
#pragma unroll
    for (int j = 0; j < N / W; ++j) raw[j] = *reinterpret_cast<const uint4*>(v.p + base + (j * BT + t) * W);
#pragma unroll
    for (int j = 0; j < N / W; ++j) {
      T y[W];
      *reinterpret_cast<uint4*>(y) = raw[j];
#pragma unroll
      for (int w = 0; w < W; ++w) x[j * W + w] = clean((float)y[w]);
    }
  } else if (v.vec) {
#pragma unroll
    for (int j = 0; j < N / W; ++j) {
      const int i = base + (j * BT + t) * W;
      T y[W];
      if (i + W <= v.V) {
        *reinterpret_cast<uint4*>(y) = *reinterpret_cast<const uint4*>(v.p + i);
#pragma unroll
        for (int w = 0; w < W; ++w) x[j * W + w] = clean((float)y[w]);
      } else {
#pragma unroll
        for (int w = 0; w < W; ++w) x[j * W + w] = i + w < v.V ? clean((float)v.p[i + w]) : -INFINITY;
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const int i = base + e * BT + t;
      x[e] = i < v.V ? clean((float)v.p[i]) : -INFINITY;
    }
  }
}

// the row's largest value alone, in two steps: the first 64 chunks' loads go out at once, to be used later
__device__ __forceinline__ float row_max_begin(const SampleP& P, int r) {
  return P.cmax[(int64_t)r * P.chunks + min((int)(threadIdx.x & 63), P.chunks - 1)];
}
__device__ __forceinline__ float row_max_end(const SampleP& P, int r, float top) {
  for (int c = 64 + (threadIdx.x & 63); c < P.chunks; c += 64) top = fmaxf(top, P.cmax[(int64_t)r * P.chunks + c]);
  return wave_max(top);
}

// 64-bit sums over a wave by data-parallel moves: within rows of 16 lanes by 1, 2, 4, 8, then a row's last lane to the rows
// behind it (a shuffle through LDS takes ten times as long). Lanes that a move does not reach add 0
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 moved64(u64 v) {
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xF, false);
  return (u64)hi << 32 | lo;
}
__device__ __forceinline__ u64 wave_scan64(u64 v) {  // inclusive; every lane active
  v += moved64<0x111, 0xF>(v);
  v += moved64<0x112, 0xF>(v);
  v += moved64<0x114, 0xF>(v);
  v += moved64<0x118, 0xF>(v);
  v += moved64<0x142, 0xA>(v);
  v += moved64<0x143, 0xC>(v);
  return v;
}
__device__ __forceinline__ u64 lane64(u64 v, int l) {  // a lane's value, l the same in all
  return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), l) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, l);
}
__device__ __forceinline__ u64 wave_sum64(u64 v) { return lane64(wave_scan64(v), 63); }
__device__ __forceinline__ int first_lane(uint64_t m) { return __ffsll((unsigned long long)m) - 1; }

// values that blocks of one launch hand to each other pass the per-XCD caches: relaxed device-scope accesses
template <typename X>
__device__ __forceinline__ X dev_load(const X* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename X>
__device__ __forceinline__ void dev_store(X* p, X v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
template <typename X>
__device__ __forceinline__ X dev_add(X* p, X v) {
  return __hip_atomic_fetch_add(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

static_assert(ST == BINS, "a thread a bin");
struct Shared {
  u64 mass[BINS];
  uint32_t cnt[BINS];
  u64 list[CAP];
  u64 part[ST / 64], few[64], lo, hi;
  int widx[ST / 64], wcnt[ST / 64];
  uint32_t wlo[ST / 64], whi[ST / 64];
  int n, sel, pick;
  u64 before_mass, mass_sel, total;
  uint32_t before_cnt;
  Cut cut;
};

// true in the block that is the last of `n` to come here (block-uniform). Everything the block has handed over lies before
__device__ __forceinline__ bool last_to_arrive(int& flag, uint32_t* counter, int n) {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) flag = dev_add(counter, 1u) == (uint32_t)n - 1;
  __syncthreads();
  return flag != 0;
}

// the row's largest value and its lowest index, from the chunks' -> every thread
__device__ __forceinline__ float row_top(const SampleP& P, int r, int& at) {
  const int lane = threadIdx.x & 63;
  float top = -INFINITY;
  at = 0x7FFFFFFF;
  for (int c = lane; c < P.chunks; c += 64) {  // every wave for itself: no barrier
    const float x = P.cmax[(int64_t)r * P.chunks + c];
    const int j = P.cidx[(int64_t)r * P.chunks + c];
    if (x > top) {
      top = x;
      at = j;
    }
  }
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const float x = __shfl_xor(top, o);
    const int j = __shfl_xor(at, o);
    if (x > top || (x == top && j < at)) {
      top = x;
      at = j;
    }
  }
  return top;
}

// first bin at which the running count reaches `need` or, by mass, the running mass reaches `target` -> S.sel, with what
// lies before it in S.before_*; -1: none. A thread a bin. Ends with a barrier.
template <typename SH>
__device__ __forceinline__ void find_bin(SH& S, bool by_mass, uint32_t need, double target, uint32_t c0, u64 m0) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const uint32_t c = S.cnt[tid];
  const u64 m = S.mass[tid];
  uint32_t ci = c;
  u64 mi = wave_scan64(m);
  if (!by_mass) ci = (uint32_t)wave_scan64(c);
  __syncthreads();  // (what an earlier call left has been read)
  if (lane == 63) {
    S.part[wave] = mi;
    S.wcnt[wave] = (int)ci;
  }
  if (tid == 0) S.sel = -1;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < ST / 64; ++w) {
    c0 += w < wave ? (uint32_t)S.wcnt[w] : 0;
    m0 += w < wave ? S.part[w] : 0;
  }
  ci += c0;
  mi += m0;
  const bool reached = by_mass ? (double)mi >= target : ci >= need;
  const bool before = by_mass ? (double)(mi - m) >= target : ci - c >= need;
  if (reached && (!before || tid == 0)) {
    S.sel = tid;
    S.before_cnt = ci - c;
    S.before_mass = mi - m;
  }
  if (tid == ST - 1) S.total = mi;
  __syncthreads();
}

// S.list[0 .. n) ascending; every entry is unique. A few hundred: each finds its own rank; more: bitonic
__device__ __forceinline__ void sort_list(Shared& S, int n) {
  constexpr int BT = ST;
  const int tid = threadIdx.x;
  if (n <= 256) {
    const int m = (n + 7) / 8 * 8;  // eight reads at once
    if (tid >= n && tid < m) S.list[tid] = ~0ull;
    __syncthreads();
    u64 mine = 0;
    int rank = 0;
    if (tid < n) {
      mine = S.list[tid];
      for (int i = 0; i < m; i += 8)
#pragma unroll
        for (int q = 0; q < 8; ++q) rank += S.list[i + q] < mine;
    }
    __syncthreads();
    if (tid < n) S.list[rank] = mine;
    __syncthreads();
    return;
  }
  int m = 64;
  while (m < n) m *= 2;
  for (int i = n + tid; i < m; i += BT) S.list[i] = ~0ull;
  __syncthreads();
  for (int k = 2; k <= m; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      for (int i = tid; i < m; i += BT) {
        const int o = i ^ j;
        if (o > i) {
          const u64 x = S.list[i], y = S.list[o];
          if ((x > y) == ((i & k) == 0)) {
            S.list[i] = y;
            S.list[o] = x;
          }
        }
      }
      __syncthreads();
    }
}
__device__ __forceinline__ u64 entry_of(float x, int i) { return ((u64)(~order_key(x)) << 32) | (uint32_t)i; }
__device__ __forceinline__ uint32_t entry_key(u64 e) { return ~(uint32_t)(e >> 32); }

// the first of the sorted list's values [i0, n) at which the mass, m0 lying before i0, reaches `target` -> its place, and the
// mass up to and with it; -1: none. Every wave alike.
__device__ __forceinline__ int list_reach(const Shared& S, int i0, int n, double target, u64 m0, float top, int S_,
                                          u64& mass) {
  const int lane = threadIdx.x & 63;
  for (int i = i0; i < n; i += 64) {
    const u64 w = i + lane < n ? weight(rel_of(key_value(entry_key(S.list[i + lane])), top), S_) : 0;
    const u64 mi = m0 + wave_scan64(w);
    const uint64_t who = __ballot(i + lane < n && (double)mi >= target);
    if (who) {
      const int l = first_lane(who);
      mass = lane64(mi, l);
      return i + l;
    }
    m0 = lane64(mi, 63);
  }
  mass = m0;
  return -1;
}

// Where a draw of `total` lies: u total, at or past the end for u >= 1 (then the last token kept is taken)
__device__ __forceinline__ double draw_target(float u, u64 total) { return (u > 0.f ? (double)u : 0.0) * (double)total; }

__device__ __forceinline__ void put(const SampleP& P, int r, int token, u64 w, u64 total) {
  P.a.token_out[r] = token;
  if (P.a.prob_out) P.a.prob_out[r] = (float)((double)w / (double)total);
}

// ------------------------------------------------------------------------------------------------------------ general row
// One block finishes a row by narrowing the cut in the keys' space: no list that could overflow, many passes over the row.
template <typename T>
__device__ __forceinline__ void general_row(Shared& S, const SampleP& P, int r, float top) {
  constexpr int BT = ST, NW = BT / 64;
  const fa_sample_args& a = P.a;
  const RowSettings s = settings_of(a, r);
  const double inv_t = P.state[r].inv_t, least = P.state[r].least;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, V = a.vocab;
  const T* const row = row_view<T>(a, r).p;
  auto logit = [&](int i) { return clean((float)row[i]); };
  Cut cut{0, 0x7FFFFFFF};  // everything

  // narrows the cut inside bin b: the prefix of the bin's values (of those within `lim`) at which the count reaches `need`, or
  // the mass `target`, c0 / m0 lying before the bin -> S.cut, S.mass_sel (mass up to the cut)
  auto resolve = [&](int b, const Cut lim, bool by_mass, uint32_t need, double target, uint32_t c0, u64 m0) {
    uint32_t lo = 0, hi = 0xFFFFFFFFu;
    auto each = [&](auto f) {
      for (int i = tid; i < V; i += BT) {
        const float x = logit(i);
        if (x == -INFINITY || bin_of(x, top) != b) continue;
        const uint32_t k = order_key(x);
        if (k < lo || k > hi || !within(k, i, lim)) continue;
        f(x, k, i);
      }
    };
    for (;;) {
      // the range and number of the values left
      uint32_t mn = 0xFFFFFFFFu, mx = 0;
      int n = 0;
      each([&](float, uint32_t k, int) {
        mn = min(mn, k);
        mx = max(mx, k);
        ++n;
      });
      for (int o = 1; o < 64; o <<= 1) {
        mn = min(mn, (uint32_t)__shfl_xor(mn, o));
        mx = max(mx, (uint32_t)__shfl_xor(mx, o));
        n += __shfl_xor(n, o);
      }
      __syncthreads();
      if (lane == 0) {
        S.wlo[wave] = mn;
        S.whi[wave] = mx;
        S.wcnt[wave] = n;
      }
      if (tid == 0) S.n = 0;
      __syncthreads();
      n = 0;
      for (int w = 0; w < NW; ++w) {
        mn = min(mn, S.wlo[w]);
        mx = max(mx, S.whi[w]);
        n += S.wcnt[w];
      }
      lo = mn;
      hi = mx;
      if (n <= CAP) break;
      if (lo == hi) {  // equal values: so many of them, in the order of their ids
        const u64 w = weight(rel_of(key_value(lo), top), P.S);
        uint32_t c = need - c0;
        if (by_mass) {
          const double f = ceil((target - (double)m0) / (double)w);
          c = f < 1.0 ? 1u : f > (double)n ? (uint32_t)n : (uint32_t)f;
          while (c > 1 && (double)(m0 + (c - 1) * w) >= target) --c;
          while (c < (uint32_t)n && (double)(m0 + c * w) < target) ++c;
        }
        const int seg = (V + NW - 1) / NW, i0 = wave * seg, i1 = min(V, i0 + seg);
        int mine = 0;
        for (int i = i0 + lane; i < i1; i += 64) mine += order_key(logit(i)) == lo;
        mine = wave_sum_i(mine);
        if (lane == 0) S.widx[wave] = mine;
        __syncthreads();
        int before = 0;
        for (int x = 0; x < wave; ++x) before += S.widx[x];
        if (before < (int)c && before + mine >= (int)c) {
          for (int i = i0; i < i1; i += 64) {
            const bool is = i + lane < i1 && order_key(logit(i + lane)) == lo;
            const uint64_t who = __ballot(is);
            const int here = __popcll(who);
            if (before + here >= (int)c) {
              const int rank = before + __popcll(who & ((1ull << lane) - 1)) + 1;
              if (is && rank == (int)c) S.cut = Cut{lo, i + lane};
              break;
            }
            before += here;
          }
        }
        if (tid == 0) S.mass_sel = m0 + c * w;
        __syncthreads();
        return;
      }
      // 1024 equal steps of the keys' range, downwards
      int sh = 0;
      while (((hi - lo) >> sh) >= BINS) ++sh;
      for (int i = tid; i < BINS; i += BT) {
        S.cnt[i] = 0;
        S.mass[i] = 0;
      }
      __syncthreads();
      each([&](float x, uint32_t k, int) {
        const int q = (int)((hi - k) >> sh);
        atomicAdd(&S.cnt[q], 1u);
        if (s.has_p) atomicAdd(&S.mass[q], weight(rel_of(x, top), P.S));
      });
      __syncthreads();
      find_bin(S, by_mass, need, target, c0, m0);
      const uint32_t q = (uint32_t)S.sel;
      c0 = S.before_cnt;
      m0 = S.before_mass;
      const uint32_t top_key = hi - (q << sh);
      lo = (uint32_t)max((int64_t)lo, (int64_t)top_key - ((1ll << sh) - 1));
      hi = top_key;
      __syncthreads();
    }
    each([&](float x, uint32_t, int i) { S.list[atomicAdd(&S.n, 1)] = entry_of(x, i); });
    __syncthreads();
    const int n = S.n;
    sort_list(S, n);
    u64 mass = 0;
    int at = (int)(need - c0) - 1;
    if (by_mass) at = list_reach(S, 0, n, target, m0, top, P.S, mass);
    else if (s.has_p) (void)list_reach(S, 0, at + 1, INFINITY, m0, top, P.S, mass);
    if (tid == 0) {
      S.cut = Cut{entry_key(S.list[at]), (int)(uint32_t)S.list[at]};
      S.mass_sel = mass;
    }
    __syncthreads();
  };

  if (s.has_k || s.has_p) {
    auto histogram = [&]() {  // of the values within the cut
      __syncthreads();
      for (int i = tid; i < BINS; i += BT) {
        S.cnt[i] = 0;
        S.mass[i] = 0;
      }
      __syncthreads();
      for (int i = tid; i < V; i += BT) {
        const float x = logit(i);
        if (x == -INFINITY || !within(order_key(x), i, cut)) continue;
        const int b = bin_of(x, top);
        atomicAdd(&S.cnt[b], 1u);
        if (s.has_p) atomicAdd(&S.mass[b], weight(rel_of(x, top), P.S));
      }
      __syncthreads();
    };
    if (s.has_k) {
      histogram();
      find_bin(S, false, (uint32_t)s.top_k, 0.0, 0, 0);
      const int b = S.sel;
      if (b >= 0) {
        const uint32_t c0 = S.before_cnt;
        const u64 m0 = S.before_mass;
        resolve(b, cut, false, (uint32_t)s.top_k, 0.0, c0, m0);
        cut = S.cut;
      }
    }
    if (s.has_p) {
      histogram();
      find_bin(S, true, 0, INFINITY, 0, 0);  // the total
      const double target = (double)s.top_p * (double)S.total;
      __syncthreads();
      find_bin(S, true, 0, target, 0, 0);
      const int b = S.sel;
      const u64 m0 = S.before_mass;
      resolve(b, cut, true, 0, target, 0, m0);
      cut = S.cut;
    }
  }

  // the draw: every wave a run of the row, in order
  auto mass_at = [&](int i) -> u64 {
    const float x = logit(i);
    if (x == -INFINITY || !within(order_key(x), i, cut)) return 0;
    const double rel = rel_of(x, top);
    return rel < least ? 0 : weight(rel * inv_t, P.S);
  };
  const int seg = ((V + NW - 1) / NW + 63) / 64 * 64, i0 = min(V, wave * seg), i1 = min(V, i0 + seg);
  u64 sum = 0;
  for (int i = i0 + lane; i < i1; i += 64) sum += mass_at(i);
  sum = wave_sum64(sum);
  __syncthreads();
  if (lane == 0) S.part[wave] = sum;
  __syncthreads();
  u64 total = 0, before = 0;
  int last = 0;
  for (int w = 0; w < NW; ++w) {
    if (w < wave) before += S.part[w];
    total += S.part[w];
    if (S.part[w]) last = w;
  }
  const double target = draw_target(a.u[r], total);
  const bool past = !((double)total > target);
  const bool mine = past ? wave == last : sum && (double)before <= target && (double)(before + sum) > target;
  if (mine) {
    int tok = -1;
    u64 wt = 0;
    for (int i = i0; i < i1; i += 64) {
      const u64 w = i + lane < i1 ? mass_at(i + lane) : 0;
      const u64 mi = before + wave_scan64(w);
      const uint64_t who = __ballot(past ? w != 0 : (double)mi > target);
      before = lane64(mi, 63);
      if (!who) continue;
      const int l = past ? 63 - __clzll((long long)who) : first_lane(who);
      tok = i + l;
      wt = lane64(w, l);
      if (!past) break;
    }
    if (lane == 0) put(P, r, tok, wt, total);
  }
}

// ------------------------------------------------------------------------------------------------------------------ kernels
template <typename T, int BT>
__global__ __launch_bounds__(BT) void k_scan(SampleP P) {
  __shared__ float smax[BT / 64];
  __shared__ int sidx[BT / 64];
  const int r = (int)P.grid_div.div(blockIdx.x), c = (int)blockIdx.x - r * P.grid_chunks;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, base = c * PER * BT;
  const RowView<T> v = row_view<T>(P.a, r);
  float x[PER];
  load_chunk<T, BT, PER>(v, base, tid, x);
  float top = x[0];
#pragma unroll
  for (int e = 1; e < PER; ++e) top = fmaxf(top, x[e]);
  if (P.want_max) P.tmax[((int64_t)r * P.chunks + c) * BT + tid] = top;
  int at = 0x7FFFFFFF;
#pragma unroll
  for (int e = PER - 1; e >= 0; --e)
    if (x[e] == top) at = index_at<T, BT>(v.vec, base, tid, e);
  // (a thread's indexes grow with e, so the last assignment is its lowest)
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const float y = __shfl_xor(top, o);
    const int j = __shfl_xor(at, o);
    if (y > top || (y == top && j < at)) {
      top = y;
      at = j;
    }
  }
  if (lane == 0) {
    smax[wave] = top;
    sidx[wave] = at;
  }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < BT / 64; ++w)
      if (smax[w] > top || (smax[w] == top && sidx[w] < at)) {
        top = smax[w];
        at = sidx[w];
      }
    P.cmax[(int64_t)r * P.chunks + c] = top;
    P.cidx[(int64_t)r * P.chunks + c] = at;
  }
  if (c == 0) {  // the row's state and histogram, for the launches behind this one
    for (int i = tid; i < BINS; i += BT) {
      P.hist_mass[(int64_t)r * BINS + i] = 0;
      P.hist_cnt[(int64_t)r * BINS + i] = 0;
    }
    if (tid == 0) {
      RowState z{};
      const RowSettings w = settings_of(P.a, r);
      z.inv_t = 1.0 / (double)w.t;
      z.least = w.min_p > 0.f ? ::log((double)w.min_p) : -INFINITY;
      P.state[r] = z;
    }
  }
}

// a row with a small top_k. CT: threads of the blocks whose threads' maxima these are
template <typename T, int CT>
__device__ __forceinline__ void finish_small_k(Shared& S, const SampleP& P, int r, const RowSettings& s, float top) {
  const int tid = threadIdx.x, lane = tid & 63;
  const double inv_t = P.state[r].inv_t, least = P.state[r].least;
  const RowView<T> v = row_view<T>(P.a, r);
  const float* const tm = P.tmax + (int64_t)r * P.chunks * CT;
  const int groups = P.chunks * CT;
  uint32_t* const pick = reinterpret_cast<uint32_t*>(S.mass);  // groups that may hold one of the k largest
  constexpr int PICK = 2 * BINS;
  S.cnt[tid] = 0;
  S.mass[tid] = 0;
  if (tid == 0) S.n = S.pick = 0;
  __syncthreads();
  // (the first rounds of maxima stay in registers: one wait for all of them)
  constexpr int HOLD = 12;
  float held[HOLD];
#pragma unroll
  for (int i = 0; i < HOLD; ++i) held[i] = i * ST + tid < groups ? tm[i * ST + tid] : -INFINITY;
#pragma unroll
  for (int i = 0; i < HOLD; ++i)
    if (held[i] > -INFINITY) atomicAdd(&S.cnt[bin_of(held[i], top)], 1u);
  for (int g = HOLD * ST + tid; g < groups; g += ST) {
    const float x = tm[g];
    if (x > -INFINITY) atomicAdd(&S.cnt[bin_of(x, top)], 1u);
  }
  __syncthreads();
  find_bin(S, false, (uint32_t)s.top_k, 0.0, 0, 0);
  const int b = S.sel < 0 ? BINS - 1 : S.sel;  // the k largest values lie in bins up to b
  auto take = [&](int g, float x) {
    if (x > -INFINITY && bin_of(x, top) <= b) {
      const int j = atomicAdd(&S.pick, 1);
      if (j < PICK) pick[j] = (uint32_t)g;
    }
  };
#pragma unroll
  for (int i = 0; i < HOLD; ++i) take(i * ST + tid, held[i]);
  for (int g = HOLD * ST + tid; g < groups; g += ST) take(g, tm[g]);
  __syncthreads();
  const int ng = S.pick;
  if (ng <= PICK)
    for (int u = tid; u < ng * PER; u += ST) {
      const int g = (int)pick[u / PER], c = g / CT;
      const int i = index_at<T, CT>(v.vec, c * PER * CT, g - c * CT, u % PER);
      if (i >= v.V) continue;
      const float x = clean((float)v.p[i]);
      if (x == -INFINITY || bin_of(x, top) > b) continue;
      const int j = atomicAdd(&S.n, 1);
      if (j < CAP) S.list[j] = entry_of(x, i);
    }
  __syncthreads();
  if (ng > PICK || S.n > CAP) {
    general_row<T>(S, P, r, top);
    return;
  }
  int n = S.n;
  sort_list(S, n);
  n = min(n, s.top_k);
  if (s.has_p) {
    u64 total = 0, mass;
    (void)list_reach(S, 0, n, INFINITY, 0, top, P.S, total);
    n = 1 + list_reach(S, 0, n, (double)s.top_p * (double)total, 0, top, P.S, mass);
  }
  // weights at the temperature (the values that min_p drops are the last ones: no weight), then the order of the ids
  u64 w = 0, e = 0;
  if (tid < n) {
    e = S.list[tid];
    const double rel = rel_of(key_value(entry_key(e)), top);
    w = rel < least ? 0 : weight(rel * inv_t, P.S);
  }
  __syncthreads();
  if (tid < n) {
    S.mass[tid] = w;
    S.list[tid] = (e << 32) | (uint32_t)tid;
  }
  __syncthreads();
  sort_list(S, n);
  if (tid >= 64) return;
  u64 total = 0;
  for (int i = lane; i < n; i += 64) total += S.mass[i];
  total = wave_sum64(total);
  const double target = draw_target(P.a.u[r], total);
  const bool past = !((double)total > target);
  u64 before = 0, wt = 0;
  int tok = -1;
  for (int i = 0; i < n; i += 64) {
    const u64 q = i + lane < n ? S.list[i + lane] : 0;
    const u64 m = i + lane < n ? S.mass[(uint32_t)q] : 0, mi = before + wave_scan64(m);
    const uint64_t who = __ballot(past ? m != 0 : (double)mi > target);
    before = lane64(mi, 63);
    if (!who) continue;
    const int l = past ? 63 - __clzll((long long)who) : first_lane(who);
    tok = (int)(lane64(q, l) >> 32);
    wt = lane64(m, l);
    if (!past) break;
  }
  if (lane == 0) put(P, r, tok, wt, total);
}

struct HistShared {  // what find_bin uses
  u64 mass[BINS], part[ST / 64];
  uint32_t cnt[BINS];
  int wcnt[ST / 64], sel, flag;
  u64 before_mass, total;
  uint32_t before_cnt;
};
template <typename T>
__global__ __launch_bounds__(ST, 8) void k_hist(SampleP P) {
  __shared__ HistShared S;
  const int r = (int)P.grid_div.div(blockIdx.x), c = (int)blockIdx.x - r * P.grid_chunks;
  const int tid = threadIdx.x;
  // (all loads first; a row that needs no histogram has read its values in vain)
  const float first = row_max_begin(P, r);
  const RowSettings s = settings_of(P.a, r);
  const RowView<T> v = row_view<T>(P.a, r);
  float x[PER];
  load_chunk<T, ST, PER>(v, c * PER * ST, tid, x);
  if (s.kind != HIST) return;
  const float top = row_max_end(P, r, first);
  if (top == -INFINITY) return;
  S.cnt[tid] = 0;
  S.mass[tid] = 0;
  __syncthreads();
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    if (x[e] == -INFINITY) continue;
    const int b = bin_of(x[e], top);
    if (s.has_k) atomicAdd(&S.cnt[b], 1u);
    if (s.has_p) atomicAdd(&S.mass[b], weight(rel_of(x[e], top), P.S));
  }
  __syncthreads();
  u64* const hm = P.hist_mass + (int64_t)r * BINS;
  uint32_t* const hc = P.hist_cnt + (int64_t)r * BINS;
  if (S.cnt[tid]) dev_add(hc + tid, S.cnt[tid]);
  if (S.mass[tid]) dev_add(hm + tid, S.mass[tid]);
  RowState* const st = P.state + r;
  if (!last_to_arrive(S.flag, &st->arrived, P.hist_chunks)) return;
  S.cnt[tid] = dev_load(hc + tid);
  S.mass[tid] = dev_load(hm + tid);
  __syncthreads();
  // the bins of the cuts. top_k's lies in b_k. top_p's target is p of the top_k's mass, which is known but for b_k's share:
  // it lies in the bins between the targets at both ends
  int b_lo = -1, b_hi = -1, b_k = -1;
  u64 mass_lo = 0, mass_k = 0;
  uint32_t cnt_k = 0;
  if (s.has_k) {
    find_bin(S, false, (uint32_t)s.top_k, 0.0, 0, 0);
    b_k = S.sel;
    if (b_k >= 0) {
      cnt_k = S.before_cnt;
      mass_k = S.before_mass;
    }
  } else {
    find_bin(S, true, 0, INFINITY, 0, 0);
  }
  u64 total = S.total;
  const u64 in_k = b_k >= 0 ? S.mass[b_k] : 0;
  __syncthreads();
  if (s.has_p) {
    const double lo = (double)s.top_p * (double)(b_k >= 0 ? mass_k : total);
    const double hi = (double)s.top_p * (double)(b_k >= 0 ? mass_k + in_k : total);
    find_bin(S, true, 0, lo, 0, 0);
    b_lo = S.sel;
    mass_lo = S.before_mass;
    __syncthreads();
    find_bin(S, true, 0, hi, 0, 0);
    b_hi = S.sel;
  } else {
    b_lo = b_hi = b_k;  // (none: fewer than k values, everything is kept)
    mass_lo = mass_k;
  }
  if (tid == 0) {
    st->b_lo = b_lo < 0 ? BINS : b_lo;  // bins below b_lo are kept whole
    st->b_hi = b_hi;
    st->b_k = b_k;
    st->mass_lo = mass_lo;
    st->mass_k = mass_k;
    st->cnt_k = cnt_k;
    st->total = total;
  }
}

template <typename T, int BT>
__global__ __launch_bounds__(BT) void k_mass(SampleP P) {
  __shared__ u64 part[BT / 64];
  __shared__ float kept[BT * PER];
  const int r = (int)P.grid_div.div(blockIdx.x), c = (int)blockIdx.x - r * P.grid_chunks;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  RowState* const st = P.state + r;
  const float first = row_max_begin(P, r);  // (all loads first, as in k_hist)
  const int cut_lo = st->b_lo, cut_hi = st->b_hi, cut_k = st->b_k;
  const double inv_t = st->inv_t, least = st->least;
  const RowSettings s = settings_of(P.a, r);
  const RowView<T> v = row_view<T>(P.a, r);
  float x[PER];
  load_chunk<T, BT, PER>(v, c * PER * BT, tid, x);
  if (s.kind != HIST && s.kind != PLAIN) return;
  const float top = row_max_end(P, r, first);
  if (top == -INFINITY) return;
  const bool hist = s.kind == HIST;
  const int b_lo = hist ? cut_lo : BINS, b_hi = hist ? cut_hi : -1, b_k = hist ? cut_k : -1;
  // the values inside the cut move together first, as few of a row's are: a wave has 64 x 16 values and takes as many
  // exponentials as it has rounds of 64 kept ones (61 rows of top_p 0.95: 18.8 us without, 18.3 with; all loads side by
  // side and the row's scales from its state: 15.8)
  u64 sum = 0;
  uint32_t listed = 0, n = 0;
  float* const mine = kept + wave * 64 * PER;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const int b = bin_of(x[e], top);
    const bool keep = x[e] != -INFINITY && b < b_lo;
    const u64 who = __ballot(keep);
    if (keep) mine[n + __popcll(who & ((1ull << lane) - 1))] = x[e];
    n += (uint32_t)__popcll(who);
    if (x[e] != -INFINITY && ((b >= b_lo && b <= b_hi) || b == b_k)) listed |= 1u << e;
  }
  for (uint32_t i = lane; i < n; i += 64) {
    const double rel = rel_of(mine[i], top);
    if (!(rel < least)) sum += weight(rel * inv_t, P.S);
  }
  if (__any(listed != 0)) {  // a place in the row's list for the whole wave's, then for each lane's
    const int own = __popc(listed);
    int upto = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(upto, o);
      if (lane >= o) upto += u;
    }
    uint32_t j = 0;
    if (lane == 63) j = dev_add(&st->list_n, (uint32_t)upto);
    j = __shfl(j, 63) + upto - own;
    u64* const list = P.list + (int64_t)r * CAP;
#pragma unroll
    for (int e = 0; e < PER; ++e)
      if (listed >> e & 1) {
        if (j < CAP) list[j] = entry_of(x[e], index_at<T, BT>(v.vec, c * PER * BT, tid, e));
        ++j;
      }
  }
  sum = wave_sum64(sum);
  if (lane == 0) part[wave] = sum;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < BT / 64; ++w) sum += part[w];
    P.cmass[(int64_t)r * P.chunks + c] = sum;
  }
}

// the cut among the listed entries (in S.list) that f accepts: the first, in their order, at which the count reaches `need` or
// the mass `target`, c0 / m0 lying before them -> S.cut, S.mass_sel (mass up to it). Histograms of 1024 equal steps of the
// entries' range, until 64 are left at most, which one wave sorts.
template <typename F>
__device__ __forceinline__ void refine_list(Shared& S, const SampleP& P, int n, F f, bool by_mass, uint32_t need, double target,
                                            uint32_t c0, u64 m0, float top) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  u64 lo = 0, hi = ~0ull;
  for (;;) {
    __syncthreads();
    S.cnt[tid] = 0;
    S.mass[tid] = 0;
    if (tid == 0) {
      S.n = 0;
      S.lo = ~0ull;
      S.hi = 0;
    }
    __syncthreads();
    u64 mn = ~0ull, mx = 0;
    int own = 0;
    for (int i = tid; i < n; i += ST) {
      const u64 e = S.list[i];
      if (e < lo || e > hi || !f(e)) continue;
      mn = min(mn, e);
      mx = max(mx, e);
      ++own;
    }
    if (own) {  // (of a few values a thread, by LDS atomics)
      atomicMin(&S.lo, mn);
      atomicMax(&S.hi, mx);
      atomicAdd(&S.n, own);
    }
    __syncthreads();
    lo = S.lo;
    hi = S.hi;
    own = S.n;
    if (own <= 64) break;
    const int sh = max(0, 54 - __clzll((long long)(hi - lo)));  // (hi - lo) >> sh < 1024
    for (int i = tid; i < n; i += ST) {
      const u64 e = S.list[i];
      if (e < lo || e > hi || !f(e)) continue;
      const int q = (int)((e - lo) >> sh);
      atomicAdd(&S.cnt[q], 1u);
      if (by_mass) atomicAdd(&S.mass[q], weight(rel_of(key_value(entry_key(e)), top), P.S));
    }
    __syncthreads();
    find_bin(S, by_mass, need, target, c0, m0);
    const u64 q = (u64)S.sel;
    c0 = S.before_cnt;
    m0 = S.before_mass;
    lo += q << sh;
    hi = lo + min(hi - lo, (1ull << sh) - 1);
  }
  if (tid == 0) S.sel = 0;
  __syncthreads();
  for (int i = tid; i < n; i += ST) {
    const u64 e = S.list[i];
    if (e >= lo && e <= hi && f(e)) S.few[atomicAdd(&S.sel, 1)] = e;
  }
  __syncthreads();
  if (wave == 0) {
    const int m = S.sel;
    const u64 e = lane < m ? S.few[lane] : ~0ull;
    int rank = 0;
    for (int i = 0; i < m; ++i) rank += S.few[i] < e;
    const u64 w = lane < m ? weight(rel_of(key_value(entry_key(e)), top), P.S) : 0;
    u64 before = 0;  // mass of the smaller entries
    for (int i = 0; i < m; ++i) {
      const u64 wi = lane64(w, i), ei = lane64(e, i);
      if (ei < e) before += wi;
    }
    const bool first = lane < m && (by_mass ? (double)(m0 + before + w) >= target && !((double)(m0 + before) >= target && rank > 0)
                                            : c0 + rank + 1 == need);
    if (first) {
      S.cut = Cut{entry_key(e), (int)(uint32_t)e};
      S.mass_sel = m0 + before + w;
    }
  }
  __syncthreads();
}

// the rows that k_mass has prepared
template <typename T, int CT>
__device__ __forceinline__ void finish_masses(Shared& S, const SampleP& P, int r, const RowSettings& s, float top) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // (everything that k_mass has left, in one wait: list entries behind list_n are read and not used)
  u64 entry[CAP / ST];
#pragma unroll
  for (int q = 0; q < CAP / ST; ++q) entry[q] = P.list[(int64_t)r * CAP + q * ST + tid];
  const u64 own_chunk = tid < P.chunks ? P.cmass[(int64_t)r * P.chunks + tid] : 0;
  const RowState st = P.state[r];
  const bool hist = s.kind == HIST;
  const int n = hist ? (int)min(st.list_n, (uint32_t)(CAP + 1)) : 0;
  if (n > CAP) {
    general_row<T>(S, P, r, top);
    return;
  }
  Cut cut{0, 0x7FFFFFFF};
  if (n > 0) {
#pragma unroll
    for (int q = 0; q < CAP / ST; ++q)
      if (q * ST + tid < n) S.list[q * ST + tid] = entry[q];
    __syncthreads();
    u64 total = st.total;  // of the top_k
    if (st.b_k >= 0) {
      const int b_k = st.b_k;
      refine_list(S, P, n, [&](u64 e) { return bin_of(key_value(entry_key(e)), top) == b_k; }, false, (uint32_t)s.top_k, 0.0,
                  (uint32_t)st.cnt_k, 0, top);
      cut = S.cut;
      if (s.has_p) {  // the mass of the top_k
        u64 m = 0;
        for (int i = tid; i < n; i += ST) {
          const u64 e = S.list[i];
          const float x = key_value(entry_key(e));
          if (bin_of(x, top) == b_k && within(entry_key(e), (int)(uint32_t)e, cut)) m += weight(rel_of(x, top), P.S);
        }
        m = wave_sum64(m);
        if (lane == 0) S.part[wave] = m;
        __syncthreads();
        total = st.mass_k;
        for (int w = 0; w < ST / 64; ++w) total += S.part[w];
        __syncthreads();
      }
    }
    if (s.has_p) {
      // (between the listed bins and b_k lie values that are not listed; the target lies in the listed ones)
      const int b_hi = st.b_hi;
      const Cut lim = cut;
      refine_list(S, P, n, [&](u64 e) {
        return bin_of(key_value(entry_key(e)), top) <= b_hi && within(entry_key(e), (int)(uint32_t)e, lim);
      }, true, 0, (double)s.top_p * (double)total, 0, st.mass_lo, top);
      cut = S.cut;
    }
  }
  // the chunks' masses, with the kept listed values' (a thread a chunk)
  __syncthreads();
  S.mass[tid] = own_chunk;
  __syncthreads();
  for (int i = tid; i < n; i += ST) {
    const u64 e = S.list[i];
    if (!within(entry_key(e), (int)(uint32_t)e, cut)) continue;
    const double rel = rel_of(key_value(entry_key(e)), top);
    if (!(rel < st.least)) atomicAdd(&S.mass[(uint32_t)e / (PER * CT)], weight(rel * st.inv_t, P.S));
  }
  __syncthreads();
  // the chunk: the first whose sum passes the target, or past the end the last with any mass
  const u64 cw = S.mass[tid], cs = wave_scan64(cw);
  if (lane == 63) S.part[wave] = cs;
  if (tid == 0) S.pick = -1;
  __syncthreads();
  u64 ahead = 0, total = 0;
#pragma unroll
  for (int x = 0; x < ST / 64; ++x) {
    ahead += x < wave ? S.part[x] : 0;
    total += S.part[x];
  }
  const double target = draw_target(P.a.u[r], total);
  const bool past = !((double)total > target);
  if (past) {
    if (cw) atomicMax(&S.pick, tid);
  } else if ((double)(ahead + cs) > target && !((double)(ahead + cs - cw) > target)) {
    S.pick = tid;
    S.before_mass = ahead + cs - cw;
  }
  __syncthreads();
  const int chunk = S.pick;
  const u64 before = S.before_mass;  // (past the end: not looked at)
  // the token: each thread PER CT / ST consecutive values of the chunk
  constexpr int N = PER * CT / ST;
  const RowView<T> v = row_view<T>(P.a, r);
  const int i0 = chunk * PER * CT + tid * N;
  u64 w[N], own = 0;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    w[e] = 0;
    const float x = i0 + e < v.V ? clean((float)v.p[i0 + e]) : -INFINITY;
    if (x > -INFINITY && within(order_key(x), i0 + e, cut)) {
      const double rel = rel_of(x, top);
      if (!(rel < st.least)) w[e] = weight(rel * st.inv_t, P.S);
    }
    own += w[e];
  }
  u64 mi = wave_scan64(own);
  if (lane == 63) S.part[wave] = mi;
  __syncthreads();
  u64 here = before;
#pragma unroll
  for (int x = 0; x < ST / 64; ++x) here += x < wave ? S.part[x] : 0;
  mi += here;
  // one thread's values hold the target: the first whose sum passes it, or past the end the last with any mass
  bool mine;
  if (past) {
    const uint64_t who = __ballot(own != 0);
    if (lane == 0) S.widx[wave] = who != 0;
    __syncthreads();
    int last = 0;
    for (int x = 0; x < ST / 64; ++x)
      if (S.widx[x]) last = x;
    mine = wave == last && who && lane == 63 - __clzll((long long)who);
  } else {
    mine = (double)mi > target && !((double)(mi - own) > target);
  }
  if (!mine) return;
  u64 sum = mi - own, wt = 0;
  int hit = -1;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    sum += w[e];
    if (w[e] && (past || (hit < 0 && (double)sum > target))) {
      hit = e;
      wt = w[e];
    }
  }
  put(P, r, i0 + hit, wt, total);
}

template <typename T, int CT>
__global__ __launch_bounds__(ST) void k_finish(SampleP P) {
  __shared__ Shared S;
  const int r = blockIdx.x;
  const RowSettings s = settings_of(P.a, r);
  int at;
  const float top = row_top(P, r, at);
  if (s.kind == GREEDY || top == -INFINITY) {
    if (threadIdx.x == 0) {
      P.a.token_out[r] = top == -INFINITY ? -1 : at;
      if (P.a.prob_out) P.a.prob_out[r] = top == -INFINITY ? 0.f : 1.f;
    }
  } else if (s.kind == SMALL_K) {
    finish_small_k<T, CT>(S, P, r, s, top);
  } else {
    finish_masses<T, CT>(S, P, r, s, top);
  }
}

// -------------------------------------------------------------------------------------------------------------------- host
struct SamplePlan {
  SampleP P;
  bool hist, mass;
  int64_t bytes;
};

static SamplePlan sample_plan(const fa_sample_args* ap) {
  FA_REQUIRE(ap, "sample_tokens: no arguments");
  SamplePlan t;
  t.P.a = *ap;
  const fa_sample_args& a = t.P.a;
  FA_REQUIRE(a.rows >= 0 && a.vocab >= 1 && a.vocab <= PER * SCAN * ST, "sample_tokens: rows, or vocab outside 1 .. 2^22");
  FA_REQUIRE(a.type == FA_F32 || a.type == FA_F16 || a.type == FA_BF16, "sample_tokens: type");
  FA_REQUIRE(a.row_stride >= a.vocab || a.rows <= 1, "sample_tokens: rows overlap");
  int lg = 0;
  while ((1 << lg) < a.vocab) ++lg;
  t.P.S = std::min(50, 62 - lg);  // the whole row's sum stays below 2^62
  t.P.chunks = (a.vocab + PER * SCAN - 1) / (PER * SCAN);  // at most ST: k_finish has a thread for each
  t.P.hist_chunks = (a.vocab + PER * ST - 1) / (PER * ST);
  FA_REQUIRE((int64_t)a.rows * t.P.chunks < (1ll << 31), "sample_tokens: more than 2^31 chunks");
  // which launches the rows can need (settings of each row live on the device: all)
  const bool each = a.temperatures || a.top_ps || a.min_ps || a.top_ks;
  const bool greedy = !(a.temperature > 0.f) || a.top_k == 1 || !(a.top_p > 0.f) || !(a.min_p <= 1.f);
  const bool has_k = a.top_k > 0 && a.top_k < a.vocab, small_k = has_k && a.top_k <= KMAX;
  t.hist = each || (!greedy && !small_k && (has_k || a.top_p < 1.f));
  t.mass = each || (!greedy && !small_k);
  t.P.want_max = each || (!greedy && small_k);
  const int64_t n = a.rows, nc = n * t.P.chunks;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t x = at;
    at += (bytes + 255) / 256 * 256;
    return x;
  };
  char* const ws = reinterpret_cast<char*>(a.workspace);
  t.P.state = reinterpret_cast<RowState*>(ws + take(n * sizeof(RowState)));
  t.P.hist_mass = reinterpret_cast<u64*>(ws + take(n * BINS * 8));
  t.P.hist_cnt = reinterpret_cast<uint32_t*>(ws + take(n * BINS * 4));
  t.P.list = reinterpret_cast<u64*>(ws + take(n * CAP * 8));
  t.P.cmass = reinterpret_cast<u64*>(ws + take(nc * 8));
  t.P.cmax = reinterpret_cast<float*>(ws + take(nc * 4));
  t.P.cidx = reinterpret_cast<int*>(ws + take(nc * 4));
  t.P.tmax = reinterpret_cast<float*>(ws + take(t.P.want_max ? nc * SCAN * 4 : 0));
  t.bytes = at;
  return t;
}

template <typename T>
static void sample_run(const SamplePlan& t, hipStream_t s) {
  auto go = [&](void (*kernel)(SampleP), int blocks, int threads) {
    SampleP P = t.P;
    P.grid_chunks = blocks;
    P.grid_div = FastDiv::of((uint32_t)blocks);
    launch(kernel, dim3((uint32_t)P.a.rows * (uint32_t)blocks), dim3(threads), 0, s, P);
  };
  go(k_scan<T, SCAN>, t.P.chunks, SCAN);
  if (t.hist) go(k_hist<T>, t.P.hist_chunks, ST);
  if (t.mass) go(k_mass<T, SCAN>, t.P.chunks, SCAN);
  go(k_finish<T, SCAN>, 1, ST);
}

int64_t sample_tokens_bytes(const fa_sample_args* a) { return sample_plan(a).bytes; }

void sample_tokens(const fa_sample_args* ap, hipStream_t s) {
  const SamplePlan t = sample_plan(ap);
  const fa_sample_args& a = t.P.a;
  if (a.rows == 0) return;
  FA_REQUIRE(a.logits && a.u && a.token_out, "sample_tokens: null tensor");
  FA_REQUIRE(a.workspace && a.workspace_bytes >= t.bytes && aligned16(a.workspace),
             "sample_tokens: workspace too small or not 16-byte aligned");
  if (a.type == FA_F32) sample_run<float>(t, s);
  else if (a.type == FA_F16) sample_run<_Float16>(t, s);
  else sample_run<__bf16>(t, s);
}

}  // namespace fa

extern "C" {

int fa_sample_tokens_workspace(const fa_sample_args* a, int64_t* bytes) {
  FA_API_BEGIN
  FA_REQUIRE(bytes, "sample_tokens: no place for the size");
  *bytes = fa::sample_tokens_bytes(a);
  FA_API_END
}

int fa_sample_tokens(const fa_sample_args* a, void* stream) {
  FA_API_BEGIN
  fa::sample_tokens(a, reinterpret_cast<hipStream_t>(stream));
  FA_API_END
}

}  // extern "C"

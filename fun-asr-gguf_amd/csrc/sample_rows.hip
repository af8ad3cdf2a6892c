// A token for every row of logits from a given random number (fa_sample_tokens).
//
// The chain keeps a set of tokens that is always a prefix of the order (logit descending, id ascending): top_k a prefix of k,
// top_p the shortest prefix whose softmax mass reaches p of the top_k's, min_p a bound on the logit. So the set is held as a
// cut (key of the last logit kept, last id kept among its equals), nothing is sorted but a few thousand values near a cut,
// and the draw runs through the vocabulary in its own order.
//
// Weights exp(x - max) are rounded to integers of 2^-S of the largest (S = 62 - ceil(log2 vocab)), so that sums are exact
// whatever the order in which they are added: results do not depend on the launch shape or on atomics. The exponentials are
// taken in 64 bits, because a sum over 150 000 tokens is compared with borders 7e-6 apart.
#include "api.h"
#include "draft_ops.h"

namespace fa {

constexpr int ST = 1024, SW = ST / 64;  // threads, waves
constexpr int BINS = 1024;              // of 1 / 32 below the maximum; the last takes everything 32 and more below
constexpr int CAP = 4096;               // values that are sorted

struct SampleP {
  fa_sample_args a;
  double one;  // 2^S
};

struct RowSettings {
  float temperature, top_p, min_p;
  int top_k;
};

template <typename T>
__device__ __forceinline__ float logit(const T* row, int i) {  // NaN -> -inf, -0 -> 0
  const float x = (float)row[i] + 0.0f;
  return x != x ? -INFINITY : x;
}
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x);
  return u >> 31 ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k >> 31 ? k & 0x7FFFFFFFu : ~k); }
__device__ __forceinline__ int bin_of(float x, float top) {
  return x == top ? 0 : (int)fminf((top - x) * 32.f, (float)(BINS - 1));  // monotone in x; top = inf: the last bin
}
__device__ __forceinline__ double rel_of(float x, float top) { return x == top ? 0.0 : (double)x - (double)top; }
__device__ __forceinline__ unsigned long long weight(double rel, double one) {
  return (unsigned long long)(exp(rel) * one + 0.5);  // exp(-inf) = 0
}
__device__ __forceinline__ unsigned long long shfl_xor64(unsigned long long v, int o) { return __shfl_xor(v, o); }

struct Cut {  // the last value kept
  uint32_t key;
  int idx;
};
__device__ __forceinline__ bool within(uint32_t key, int i, const Cut& c) {
  return key > c.key || (key == c.key && i <= c.idx);
}

struct Shared {
  unsigned long long mass[BINS];
  uint32_t cnt[BINS];
  unsigned long long list[CAP];
  unsigned long long wsum[SW];
  float wmax[SW];
  int widx[SW], wcnt[SW];
  uint32_t wlo[SW], whi[SW];
  int n, sel;
  unsigned long long before_mass, mass_sel;
  uint32_t before_cnt;
  Cut cut;
  int token;
  float prob;
};

// first bin at which the running count reaches `need` (count) or the running mass reaches `target` -> S.sel, with what lies
// before it in S.before_*; -1: none. Wave 0, 16 bins a lane.
__device__ __forceinline__ void find_bin(Shared& S, bool by_mass, uint32_t need, double target, uint32_t c0,
                                         unsigned long long m0) {
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    uint32_t c = 0;
    unsigned long long m = 0;
    for (int i = 0; i < BINS / 64; ++i) {
      c += S.cnt[lane * (BINS / 64) + i];
      m += S.mass[lane * (BINS / 64) + i];
    }
    uint32_t ci = c;
    unsigned long long mi = m;
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t cu = __shfl_up(ci, o);
      const unsigned long long mu = __shfl_up(mi, o);
      if (lane >= o) {
        ci += cu;
        mi += mu;
      }
    }
    const bool reached = by_mass ? (double)(m0 + mi) >= target : c0 + ci >= need;
    const uint64_t who = __ballot(reached);
    if (who == 0) {
      if (lane == 0) S.sel = -1;
    } else if (lane == __ffsll((unsigned long long)who) - 1) {
      uint32_t cb = c0 + ci - c;
      unsigned long long mb = m0 + mi - m;
      int i = lane * (BINS / 64);
      for (;; ++i) {
        const uint32_t cn = cb + S.cnt[i];
        const unsigned long long mn = mb + S.mass[i];
        if (by_mass ? (double)mn >= target : cn >= need) break;
        cb = cn;
        mb = mn;
      }
      S.sel = i;
      S.before_cnt = cb;
      S.before_mass = mb;
    }
  }
  __syncthreads();
}

template <typename T>
__global__ __launch_bounds__(ST) void k_sample_row(SampleP P) {
  __shared__ Shared S;
  const fa_sample_args& a = P.a;
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, V = a.vocab;
  const T* const row = reinterpret_cast<const T*>(a.logits) + (int64_t)r * a.row_stride;
  RowSettings s;
  s.temperature = a.temperatures ? a.temperatures[r] : a.temperature;
  s.top_p = a.top_ps ? a.top_ps[r] : a.top_p;
  s.min_p = a.min_ps ? a.min_ps[r] : a.min_p;
  s.top_k = a.top_ks ? a.top_ks[r] : a.top_k;

  // the largest logit, its lowest id
  float top = -INFINITY;
  int at = 0x7FFFFFFF;
  for (int i = tid; i < V; i += ST) {
    const float x = logit(row, i);
    if (x > top) {
      top = x;
      at = i;
    }
  }
  for (int o = 1; o < 64; o <<= 1) {
    const float x = __shfl_xor(top, o);
    const int j = __shfl_xor(at, o);
    if (x > top || (x == top && j < at)) {
      top = x;
      at = j;
    }
  }
  if (lane == 0) {
    S.wmax[wave] = top;
    S.widx[wave] = at;
  }
  __syncthreads();
  for (int w = 0; w < SW; ++w)
    if (S.wmax[w] > top || (S.wmax[w] == top && S.widx[w] < at)) {
      top = S.wmax[w];
      at = S.widx[w];
    }
  const bool greedy = !(s.temperature > 0.f) || s.top_k == 1 || !(s.top_p > 0.f) || !(s.min_p <= 1.f);
  if (top == -INFINITY || greedy) {
    if (tid == 0) {
      a.token_out[r] = top == -INFINITY ? -1 : at;
      if (a.prob_out) a.prob_out[r] = top == -INFINITY ? 0.f : 1.f;
    }
    return;
  }
  const bool has_k = s.top_k > 0 && s.top_k < V, has_p = s.top_p < 1.f;
  const double least = s.min_p > 0.f ? ::log((double)s.min_p) : -INFINITY;
  Cut cut{0, 0x7FFFFFFF};  // everything

  // narrows the cut inside bin b: the prefix of the bin's values (of those within `lim`) at which the count reaches `need`, or
  // the mass `target`, c0 / m0 lying before the bin -> S.cut, S.mass_sel (mass up to the cut)
  auto resolve = [&](int b, const Cut lim, bool by_mass, uint32_t need, double target, uint32_t c0,
                     unsigned long long m0) {
    uint32_t lo = 0, hi = 0xFFFFFFFFu;
    auto each = [&](auto f) {
      for (int i = tid; i < V; i += ST) {
        const float x = logit(row, i);
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
      for (int w = 0; w < SW; ++w) {
        mn = min(mn, S.wlo[w]);
        mx = max(mx, S.whi[w]);
        n += S.wcnt[w];
      }
      lo = mn;
      hi = mx;
      if (n <= CAP) break;
      if (lo == hi) {  // equal values: so many of them, in the order of their ids
        const unsigned long long w = weight(rel_of(key_value(lo), top), P.one);
        uint32_t c = need - c0;
        if (by_mass) {
          const double f = ceil((target - (double)m0) / (double)w);
          c = f < 1.0 ? 1u : f > (double)n ? (uint32_t)n : (uint32_t)f;
          while (c > 1 && (double)(m0 + (c - 1) * w) >= target) --c;
          while (c < (uint32_t)n && (double)(m0 + c * w) < target) ++c;
        }
        const int seg = (V + SW - 1) / SW, i0 = wave * seg, i1 = min(V, i0 + seg);
        int mine = 0;
        for (int i = i0 + lane; i < i1; i += 64) mine += order_key(logit(row, i)) == lo;
        mine = wave_sum_i(mine);
        if (lane == 0) S.widx[wave] = mine;
        __syncthreads();
        int before = 0;
        for (int x = 0; x < wave; ++x) before += S.widx[x];
        if (before < (int)c && before + mine >= (int)c) {
          for (int i = i0; i < i1; i += 64) {
            const bool is = i + lane < i1 && order_key(logit(row, i + lane)) == lo;
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
      // 1024 equal steps of the key's range, downwards
      int sh = 0;
      while (((hi - lo) >> sh) >= BINS) ++sh;
      for (int i = tid; i < BINS; i += ST) {
        S.cnt[i] = 0;
        S.mass[i] = 0;
      }
      __syncthreads();
      each([&](float x, uint32_t k, int) {
        const int q = (int)((hi - k) >> sh);
        atomicAdd(&S.cnt[q], 1u);
        if (has_p) atomicAdd(&S.mass[q], weight(rel_of(x, top), P.one));
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
    // few values: sorted, largest first, lower ids first among equals
    each([&](float, uint32_t k, int i) {
      const int j = atomicAdd(&S.n, 1);
      S.list[j] = ((unsigned long long)(~k) << 32) | (uint32_t)i;
    });
    __syncthreads();
    const int n = S.n;
    int m = 64;
    while (m < n) m *= 2;
    for (int i = n + tid; i < m; i += ST) S.list[i] = ~0ull;
    __syncthreads();
    for (int k = 2; k <= m; k <<= 1)
      for (int j = k >> 1; j > 0; j >>= 1) {
        for (int i = tid; i < m; i += ST) {
          const int o = i ^ j;
          if (o > i) {
            const unsigned long long x = S.list[i], y = S.list[o];
            if ((x > y) == ((i & k) == 0)) {
              S.list[i] = y;
              S.list[o] = x;
            }
          }
        }
        __syncthreads();
      }
    if (wave == 0) {
      for (int i0 = 0; i0 < n; i0 += 64) {
        const int i = i0 + lane;
        const unsigned long long e = i < n ? S.list[i] : 0;
        const uint32_t key = ~(uint32_t)(e >> 32);
        const unsigned long long w = i < n && has_p ? weight(rel_of(key_value(key), top), P.one) : 0;
        unsigned long long mi = w;
        for (int o = 1; o < 64; o <<= 1) {
          const unsigned long long u = __shfl_up(mi, o);
          if (lane >= o) mi += u;
        }
        const bool reached = i < n && (by_mass ? (double)(m0 + mi) >= target : c0 + i + 1 >= need);
        const uint64_t who = __ballot(reached);
        if (who) {
          if (lane == __ffsll((unsigned long long)who) - 1) {
            S.cut = Cut{key, (int)(uint32_t)e};
            S.mass_sel = m0 + mi;
          }
          break;
        }
        m0 += __shfl(mi, 63);
      }
    }
    __syncthreads();
  };

  if (has_k || has_p) {
    for (int i = tid; i < BINS; i += ST) {
      S.cnt[i] = 0;
      S.mass[i] = 0;
    }
    __syncthreads();
    for (int i = tid; i < V; i += ST) {
      const float x = logit(row, i);
      if (x == -INFINITY) continue;
      const int b = bin_of(x, top);
      atomicAdd(&S.cnt[b], 1u);
      if (has_p) atomicAdd(&S.mass[b], weight(rel_of(x, top), P.one));
    }
    __syncthreads();
    unsigned long long total = 0;
    for (int i = 0; i < BINS; ++i) total += S.mass[i];
    int b = -1;
    // (the histogram of the row stays in registers over resolve(), which uses its arrays: one bin a thread)
    const unsigned long long my_mass = S.mass[tid];
    const uint32_t my_cnt = S.cnt[tid];
    if (has_k) {
      find_bin(S, false, (uint32_t)s.top_k, 0.0, 0, 0);
      b = S.sel;
      if (b >= 0) {
        const uint32_t c0 = S.before_cnt;
        const unsigned long long m0 = S.before_mass;
        resolve(b, cut, false, (uint32_t)s.top_k, 0.0, c0, m0);
        cut = S.cut;
        total = S.mass_sel;
      }
    }
    if (has_p) {
      // the row's histogram again, the last kept bin with what the cut leaves of it
      __syncthreads();
      unsigned long long below = 0;
      S.mass[tid] = my_mass;
      S.cnt[tid] = my_cnt;
      __syncthreads();
      if (b >= 0 && tid == 0) {
        for (int i = 0; i < b; ++i) below += S.mass[i];
        S.mass[b] = total - below;
        for (int i = b + 1; i < BINS; ++i) S.mass[i] = 0;
      }
      __syncthreads();
      const double target = (double)s.top_p * (double)total;
      find_bin(S, true, 0, target, 0, 0);
      const int bp = S.sel;
      if (bp >= 0) {
        const unsigned long long m0 = S.before_mass;
        resolve(bp, cut, true, 0, target, 0, m0);
        cut = S.cut;
      }
    }
  }

  // the draw: every wave a run of the row, in order
  const double inv_t = 1.0 / (double)s.temperature;
  auto mass_at = [&](int i) -> unsigned long long {
    const float x = logit(row, i);
    if (x == -INFINITY || !within(order_key(x), i, cut)) return 0;
    const double rel = rel_of(x, top);
    return rel < least || rel == -INFINITY ? 0 : weight(rel * inv_t, P.one);
  };
  const int seg = ((V + SW - 1) / SW + 63) / 64 * 64, i0 = min(V, wave * seg), i1 = min(V, i0 + seg);
  unsigned long long sum = 0;
  for (int i = i0 + lane; i < i1; i += 64) sum += mass_at(i);
  for (int o = 1; o < 64; o <<= 1) sum += shfl_xor64(sum, o);
  __syncthreads();
  if (lane == 0) S.wsum[wave] = sum;
  __syncthreads();
  unsigned long long total = 0, before = 0;
  int last = 0;
  for (int w = 0; w < SW; ++w) {
    if (w < wave) before += S.wsum[w];
    total += S.wsum[w];
    if (S.wsum[w]) last = w;
  }
  const float u = a.u[r];
  const double target = (u > 0.f ? (double)u : 0.0) * (double)total;
  const bool past = !((double)total > target);  // u >= 1: the last token kept
  const bool mine = past ? wave == last : sum && (double)before <= target && (double)(before + sum) > target;
  if (mine) {
    int tok = -1;
    unsigned long long wt = 0;
    for (int i = i0; i < i1; i += 64) {
      const unsigned long long w = i + lane < i1 ? mass_at(i + lane) : 0;
      unsigned long long mi = w;
      for (int o = 1; o < 64; o <<= 1) {
        const unsigned long long x = __shfl_up(mi, o);
        if (lane >= o) mi += x;
      }
      const uint64_t who = __ballot(past ? w != 0 : (double)(before + mi) > target);
      before += __shfl(mi, 63);
      if (!who) continue;
      const int l = past ? 63 - __clzll((long long)who) : __ffsll((unsigned long long)who) - 1;
      tok = i + l;
      wt = __shfl(w, l);
      if (!past) break;
    }
    if (lane == 0) {
      a.token_out[r] = tok;
      if (a.prob_out) a.prob_out[r] = (float)((double)wt / (double)total);
    }
  }
}

static SampleP sample_plan(const fa_sample_args* ap) {
  FA_REQUIRE(ap, "sample_tokens: no arguments");
  SampleP P;
  P.a = *ap;
  const fa_sample_args& a = P.a;
  FA_REQUIRE(a.rows >= 0 && a.vocab >= 1 && a.vocab <= (1 << 24), "sample_tokens: rows, or vocab outside 1 .. 2^24");
  FA_REQUIRE(a.type == FA_F32 || a.type == FA_F16 || a.type == FA_BF16, "sample_tokens: type");
  FA_REQUIRE(a.row_stride >= a.vocab || a.rows <= 1, "sample_tokens: rows overlap");
  int lg = 0;
  while ((1 << lg) < a.vocab) ++lg;
  P.one = (double)(1ull << (62 - lg));
  return P;
}

static void sample_tokens(const fa_sample_args* ap, hipStream_t s) {
  SampleP P = sample_plan(ap);
  const fa_sample_args& a = P.a;
  if (a.rows == 0) return;
  FA_REQUIRE(a.logits && a.u && a.token_out, "sample_tokens: null tensor");
  auto k = a.type == FA_F32 ? k_sample_row<float> : a.type == FA_F16 ? k_sample_row<_Float16> : k_sample_row<__bf16>;
  launch(k, dim3(a.rows), dim3(ST), 0, s, P);
}

}  // namespace fa

extern "C" {

int fa_sample_tokens_workspace(const fa_sample_args* a, int64_t* bytes) {
  FA_API_BEGIN
  FA_REQUIRE(bytes, "sample_tokens: no place for the size");
  (void)fa::sample_plan(a);
  *bytes = 0;
  FA_API_END
}

int fa_sample_tokens(const fa_sample_args* a, void* stream) {
  FA_API_BEGIN
  fa::sample_tokens(a, reinterpret_cast<hipStream_t>(stream));
  FA_API_END
}

}  // extern "C"

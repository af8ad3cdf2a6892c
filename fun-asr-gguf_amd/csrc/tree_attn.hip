// Attention of drafted tokens over a paged cache (fa_tree_attention).
//
// For one sequence and kv head the rows are (drafted token, query head of the group), all of which read the same keys:
//   S = K Q^T,  P = softmax over keys (running maximum and sum, 32 bits),  O^T += V^T P^T.
// Both products run on 16x16x32 matrix instructions. S is made with the keys as rows, so that a lane's results belong to one
// query row (lane % 16) and 4 consecutive keys, in two tiles 8: exactly the operand P^T of the second product, whose
// contraction runs over the keys in that order (4 g + i, then 16 + 4 g + i); V^T is read from LDS in the same order by the
// transposing reads. The output's columns are query rows too, so rescaling needs no exchange between lanes; the running
// maximum needs two.
//
// Two kernels, by the number of rows of a sequence and kv head:
//   k_few (up to 32): what bounds it is reading K and V once. The four waves of a block take every fourth 32-key tile of the
//     block's keys, each with a running maximum, sum and output of its own, and join through LDS at the end: no barrier in
//     the loop. K goes from memory straight into operand registers (a key row in 64-byte pieces by 4 lanes), V through
//     wave-private LDS.
//   k_many: the softmax's vector instructions weigh as much as the reading. The block's waves take 16 RT rows each and share
//     every K and V tile through two LDS stages, so a tile is read once for 64 RT rows; one barrier a tile.
// In LDS, row k's 16-byte piece j lies at j ^ (k mod pieces), which spreads rows over the banks, but not quite evenly: for heads
// over 64, half a wave's transposing read holds keys 0-7 with pieces 2 m and 2 m + 1, and keys k and k ^ 1 meet on one pair of
// banks; for heads up to 64 the operand read of K does so. Counted: 25 % of k_many's LDS cycles are conflicts, of k_few's 19 (32
// sequences) and 24 % (one token a sequence).
// Blocks of the same rows split the keys where the launch would not fill the card; k_tree_merge joins their partial results
// (unnormalised output, base, sum).
//
// Measured: 48 sequences of up to 8191 keys, one token each, 32 / 8 heads of 128: 206 us, 5.0 TB/s of K and V; 32 of up to 2032
// keys, 16 drafted tokens, 16 / 8 heads: 54 + 6 us (blocks of 1024 keys begin and end for a fifth of it); 4 of 32685 keys, 63
// drafted tokens, 32 / 8 heads (k_many): 201 us, 670 TFLOP/s, the matrix units busy a third of the time, the waves waiting for
// operands a third (60 calls back to back: 207 at first, up to 268 in between, 211 at the end); 8 float32 tokens on 212 keys:
// 10.4 us, the chain lengths, page, K, products, V, join.
#include "api.h"
#include "draft_ops.h"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace fa {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short v4i16 __attribute__((ext_vector_type(4)));

struct TreeP {
  fa_tree_attention_args a;
  FastDiv page_div, group_div, q_tiles_div, kv_div, splits_div;
  int group, rows;     // query heads per kv head; rows of one sequence and kv head: nodes * group
  int q_tiles;         // blocks along the rows
  int chunk, splits;   // keys a block (a multiple of 128), blocks along the keys at most
  int n_groups;        // (sequence, kv head, split) triples
  float c;             // scale * log2(e)
  float* part_o;       // [seqs][kv_heads][splits][rows][DP]
  float* part_ml;      // [seqs][kv_heads][splits][rows][2]: base (see base_of; -inf: nothing seen) and sum
  int q_vec;           // q's rows may be read in 16-byte pieces
  uint32_t k_page, k_slot, v_page, v_slot;  // strides, below 2^31 (checked by the host): one multiply-add a product
  int one_offset;      // K's and V's strides are the same
  int uniform;         // so many consecutive keys, or a divisor of it, lie in one page: page_size, or 1 (see UNI)
};

__device__ __forceinline__ f32x4 mfma16(f16x8_t a, f16x8_t b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(bf16x8_t a, bf16x8_t b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
// 2^x; results below 2^-126 become 0 (weights that far under the row's largest)
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// over the four 16-lane groups of a wave: a swap of a register with itself leaves one half (or one 16-lane row of each pair)
// twice in the first and the other twice in the second
__device__ __forceinline__ float across_max(float v) {
  const auto h = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(h[0]), __uint_as_float(h[1]));
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float across_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}
// Softmax weights are 2^(s c - base) with base = maximum c - kLift: 2^kLift at the largest. They enter the second product in the
// cache's type, and so float16's range lies where they do: steps of 2^-11 of a weight down to 2^-29 of the largest, then of
// 2^-39, nothing under 2^-40 (from 1 down it ends at 2^-25: of 40 000 keys e^-18 under one large weight nothing was left).
// bfloat16 has the range of float32. The factor leaves with the division by the sum.
template <typename T> constexpr float kLift = 0.f;
template <> constexpr float kLift<_Float16> = 15.f;
template <typename T>
__device__ __forceinline__ float base_of(float m, float c) { return fmaf(m, c, -kLift<T>); }
template <typename T> constexpr uint32_t kExp = 0;  // exponent bits
template <> constexpr uint32_t kExp<_Float16> = 0x7C00u;
template <> constexpr uint32_t kExp<__bf16> = 0x7F80u;

struct SeqLens {
  int n, ctx, total, splits;
};
__device__ __forceinline__ SeqLens seq_lens(const TreeP& P, int b) {
  const fa_tree_attention_args& a = P.a;
  SeqLens s;  // (kept in scalar registers, and what follows from them)
  s.n = a.draft_lens ? min(max(__builtin_amdgcn_readfirstlane(a.draft_lens[b]), 0), a.nodes) : a.nodes;
  const int cap = a.table_len * a.page_size;  // < 2^31 - nodes (checked by the host)
  s.ctx = min(max(__builtin_amdgcn_readfirstlane(a.context_lens[b]), 0), cap);
  s.total = min(s.ctx + s.n, cap);
  s.splits = min(P.splits, max(1, (s.total + P.chunk - 1) / P.chunk));
  return s;
}

// The block's part: consecutive block numbers go round the XCDs, so the row tiles of one (sequence, kv head, split), which
// read the same keys, are 8 numbers apart: one XCD's L2 fetches those keys once. The eight triples of a round turn by one from
// round to round, else one XCD would get the last (short) splits of all sequences. false: a block of the round-up
struct Where {
  int b, h, split, q_tile;
};
__device__ __forceinline__ bool locate(const TreeP& P, Where& w) {
  const uint32_t xcd = blockIdx.x & 7, slot = blockIdx.x >> 3, g8 = P.q_tiles_div.div(slot);
  w.q_tile = (int)(slot - g8 * P.q_tiles);
  const uint32_t g = g8 * 8 + ((xcd + g8) & 7);
  if (g >= (uint32_t)P.n_groups) return false;
  const uint32_t bh = P.splits_div.div(g);
  w.split = (int)(g - bh * P.splits);
  w.b = (int)P.kv_div.div(bh);
  w.h = (int)(bh - (uint32_t)w.b * P.a.kv_heads);
  return true;
}

// this lane's query row (of rows r0 + r16) as NS terms of the cache's type: dimensions 8 (g4 + 4 ks) + 0 .. 7. A float32 row is
// first multiplied by the power of two that brings its largest element to 2^14 .. 2^15, whatever its size: within float16's range,
// and with the lower term's steps, 2^-24, 2^-38 of the row's largest. c: what makes scores exponents of 2, with the inverse of it
template <typename T, int NS, int KS>
__device__ __forceinline__ int load_q(const TreeP& P, const Where& w, int rr, int rows, int g4,
                                      typename Vec8<T>::type (&q)[KS][NS], float& c) {
  const fa_tree_attention_args& a = P.a;
  const int rc = min(rr, rows - 1), node = (int)P.group_div.div((uint32_t)rc);
  const int64_t at = w.b * a.q_seq + node * a.q_node + (int64_t)(w.h * P.group + rc - node * P.group) * a.q_head;
  c = P.c;
  if constexpr (NS == 1) {
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int e = 8 * (g4 + 4 * ks);
      float x[8] = {};
      if (rr < rows && e < a.head_dim) {
        const T* const p = reinterpret_cast<const T*>(a.q) + at + e;
        if (P.q_vec) load8<true>(p, x);
        else load8<false>(p, x);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) q[ks][0][i] = (T)x[i];
    }
  } else {
    float x[KS][8] = {}, top = 0.f;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int e = 8 * (g4 + 4 * ks);
      if (rr < rows && e < a.head_dim) {
        const float* const p = reinterpret_cast<const float*>(a.q) + at + e;
        if (P.q_vec) load8<true>(p, x[ks]);
        else load8<false>(p, x[ks]);
      }
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(x[ks][i]));
    top = across_max(top);  // (an infinite row: the finite elements stay below 2^14)
    const int f = min(max(268 - (int)(__float_as_uint(top) >> 23), 1), 253);  // exponents of the factor and its inverse
    const float up = __uint_as_float((uint32_t)f << 23);
    c = fminf(fmaxf(P.c * __uint_as_float((uint32_t)(254 - f) << 23), 1.2e-38f), 3.4e38f);
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float y = x[ks][i] * up;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          const T z = (T)y;
          q[ks][s][i] = z;
          y = fabsf(y) < INFINITY ? y - (float)z : 0.f;
        }
      }
  }
  return node;
}

// which of this lane's 8 keys of a 32-key group the row sees: bit i: key 16 (i / 4) + 4 g4 + i % 4 of the group at kt.
// present: the group's keys that exist
__device__ __forceinline__ uint32_t seen_bits(const TreeP& P, int b, int ctx, int kt, uint32_t present, int node, int g4) {
  const fa_tree_attention_args& a = P.a;
  // the drafted keys' part: eight loads at once, or the order of the tokens; in integers (conditions would take two scalar
  // registers each)
  const int j0 = kt + 4 * g4 - ctx;
  uint32_t drafted[8];
  if (a.mask) {
    const uint8_t* const row = a.mask + b * a.mask_seq + node * a.mask_row;
#pragma unroll
    for (int i = 0; i < 8; ++i) drafted[i] = row[min(max(j0 + 16 * (i >> 2) + (i & 3), 0), a.nodes - 1)];
#pragma unroll
    for (int i = 0; i < 8; ++i) drafted[i] = min(drafted[i], 1u);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) drafted[i] = (uint32_t)(j0 + 16 * (i >> 2) + (i & 3) - node - 1) >> 31;
  }
  present >>= 4 * g4;
  uint32_t bits = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int kk = 16 * (i >> 2) + (i & 3);
    bits |= ((present >> kk) & (drafted[i] | (uint32_t)(j0 + kk) >> 31) & 1u) << i;
  }
  return bits;
}

// KG groups of 32 keys of the softmax: scores s -> weights in their place, relative to the running maximum; o and l rescaled
template <typename T, int MT, int KG>
__device__ __forceinline__ void softmax_step(f32x4 (&s)[KG][2], float c, float& m, float& l, f32x4 (&o)[MT]) {
  float top = m;
#pragma unroll
  for (int g = 0; g < KG; ++g)
#pragma unroll
    for (int t = 0; t < 2; ++t) top = fmaxf(top, fmaxf(fmaxf(s[g][t][0], s[g][t][1]), fmaxf(s[g][t][2], s[g][t][3])));
  top = across_max(top);
  const float base = top == -INFINITY ? 0.f : base_of<T>(top, c);  // nothing seen so far: every weight is 2^-inf = 0
  if (__any(top != m)) {                                           // (first tiles mostly)
    const float alpha = exp2_fast(base_of<T>(m, c) - base);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) o[mt] *= alpha;
    l *= alpha;
  }
  m = top;
  float sum[2] = {0.f, 0.f};
#pragma unroll
  for (int g = 0; g < KG; ++g)
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = exp2_fast(fmaf(s[g][t][i], c, -base));
        s[g][t][i] = e;
        sum[t] += e;
      }
  l += sum[0] + sum[1];
}
template <typename T, int NS>
__device__ __forceinline__ void to_terms(const f32x4 (&s)[2], typename Vec8<T>::type (&p)[NS]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float e = s[i >> 2][i & 3];
#pragma unroll
    for (int n = 0; n < NS; ++n) {
      const T y = (T)e;
      p[n][i] = y;
      e -= (float)y;
    }
  }
}

// With several terms of q an infinite key gives NaN where a lower term is 0, or of the other sign than the first: a score that
// is NaN is made again, by f, from the first term alone, which tells infinity from NaN (and is all that counts beside infinity).
// Rare, also where a key's place holds no key
template <typename F>
__device__ __forceinline__ void first_term_for_nan(f32x4 (&s)[2], F f) {
  bool odd = false;
#pragma unroll
  for (int i = 0; i < 8; ++i) odd |= s[i >> 2][i & 3] != s[i >> 2][i & 3];
  if (!__any(odd)) return;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const f32x4 x = f(t);
#pragma unroll
    for (int i = 0; i < 4; ++i) s[t][i] = s[t][i] == s[t][i] ? s[t][i] : x[i];
  }
}

// eight elements at p + i. As a 32-bit offset in bytes under the pointer: where that is a scalar, the load adds them itself
template <typename T>
__device__ __forceinline__ typename Vec8<T>::type piece_at(const T* p, uint32_t i) {
  return *reinterpret_cast<const typename Vec8<T>::type*>(reinterpret_cast<const char*>(p) + i * 2u);
}

// sets the infinities and NaN among 8 values to 0 where `own` is all ones (0: leaves them); true if it did
template <typename T>
__device__ __forceinline__ bool strip_nonfinite(typename Vec8<T>::type& v, uint32_t own) {
  uint4 u = __builtin_bit_cast(uint4, v);
  constexpr uint32_t E = kExp<T>;
  uint32_t hit = 0;
  for (uint32_t* x : {&u.x, &u.y, &u.z, &u.w}) {
    const uint32_t lo = (*x & E) == E ? 0xFFFFu : 0u, hi = (*x >> 16 & E) == E ? 0xFFFF0000u : 0u;
    hit |= (lo | hi) & own;
    *x &= ~((lo | hi) & own);
  }
  v = __builtin_bit_cast(typename Vec8<T>::type, u);
  return hit != 0;
}

__device__ __forceinline__ void apply_mask(uint32_t bits, f32x4 (&s)[2]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) s[i >> 2][i & 3] = (bits >> i) & 1 ? s[i >> 2][i & 3] : -INFINITY;
}

// An infinity or NaN in a drafted key's value must reach the rows that have a weight for it and no others (in the matrix
// product 0 * inf would reach every row): the loops leave such values out (strip_nonfinite; a committed key's stay, as every row
// sees it), and where there were any, this adds them at the end, key by key, for the 32-key groups kt, kt + step ... of the
// drafted keys. wl: 32 x 16 floats of LDS of the wave's own. Rare, and kept out of the loops for their registers' sake.
template <typename T, int NS, int DP>
__device__ __forceinline__ void add_nonfinite(const TreeP& P, const Where& w, const SeqLens& L, int kt, int k1, int step,
                                              int node, const typename Vec8<T>::type (&q)[DP / 32][NS], float c, float m, float* wl,
                                              f32x4 (&o)[DP / 16]) {
  typedef typename Vec8<T>::type V8;
  const fa_tree_attention_args& a = P.a;
  const int lane = threadIdx.x & 63, r16 = lane & 15, g4 = lane >> 4;
  const T* const kbase = reinterpret_cast<const T*>(a.k_cache) + w.h * a.k_head;
  const T* const vbase = reinterpret_cast<const T*>(a.v_cache) + w.h * a.v_head;
  const int32_t* const table = a.block_table + w.b * a.table_seq;
  const float base = m == -INFINITY ? 0.f : base_of<T>(m, c);
  for (; kt < k1; kt += step) {
    if (kt + 32 <= L.ctx) continue;
    const T* at[2];
    uint32_t present = 0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int key = kt + 16 * t + r16;
      const uint32_t pg = P.page_div.div((uint32_t)key);
      const int id = key < k1 ? table[pg] : -1;
      const bool ok = (uint32_t)id < (uint32_t)a.pages;
      present |= (uint32_t)(__ballot(ok) & 0xFFFF) << (16 * t);
      at[t] = ok ? kbase + id * a.k_page + (int64_t)((uint32_t)key - pg * a.page_size) * a.k_slot : kbase;
    }
    auto scores = [&](int t, int terms) {
      f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < DP / 32; ++ks) {
        const int e = 8 * (g4 + 4 * ks);
        const V8 x = e < a.head_dim ? *reinterpret_cast<const V8*>(at[t] + e) : V8{};
#pragma unroll
        for (int n = NS - 1; n >= 0; --n)
          if (n < terms) s = mfma16(x, q[ks][n], s);
      }
      return s;
    };
    f32x4 s[2] = {scores(0, NS), scores(1, NS)};
    if constexpr (NS > 1) first_term_for_nan(s, [&](int t) { return scores(t, 1); });
    apply_mask(seen_bits(P, w.b, L.ctx, kt, present, node, g4), s);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      wl[(16 * (i >> 2) + 4 * g4 + (i & 3)) * 16 + r16] = exp2_fast(fmaf(s[i >> 2][i & 3], c, -base));
    for (int k = 0; k < 32 && kt + k < k1; ++k) {
      if (kt + k < L.ctx) continue;
      const uint32_t pg = P.page_div.div((uint32_t)(kt + k));
      const int id = table[pg];
      if ((uint32_t)id >= (uint32_t)a.pages) continue;
      const T* const v = vbase + id * a.v_page + (int64_t)((uint32_t)(kt + k) - pg * a.page_size) * a.v_slot;
      const float f = wl[k * 16 + r16];
#pragma unroll
      for (int mt = 0; mt < DP / 16; ++mt)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int d = 16 * mt + 4 * g4 + j;
          const float x = d < a.head_dim ? (float)v[d] : 0.f;
          if (!(fabsf(x) < INFINITY) && f != 0.f) o[mt][j] += f * x;
        }
    }
  }
}

template <typename T>
__device__ __forceinline__ typename Vec8<T>::type values_operand(const T* lo, const T* hi) {
  typename Vec8<T>::type v;
  const v4i16 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4i16*)(lo));
  const v4i16 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4i16*)(hi));
  const auto p = __builtin_bit_cast(T __attribute__((ext_vector_type(4))), x);
  const auto q = __builtin_bit_cast(T __attribute__((ext_vector_type(4))), y);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = p[i];
    v[4 + i] = q[i];
  }
  return v;
}

template <typename TO>
__device__ __forceinline__ void store4(TO* p, f32x4 x, int left) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < left) p[i] = (TO)x[i];
}

// T: cache type. NS: 16-bit terms of q and of the weights (1: q is of the cache's type; 2 / 3: q is float32, kept to 22 / 24
// bits by terms of float16 / bfloat16, a weight too, float16's down to 2^-40 of the largest; with 1 term the weights are rounded
// to the cache's type, half a step of it, as the output is). DP: head_dim rounded up to 64 / 128 / 256. FULL: it is DP itself;
// else a piece behind head_dim is read at 0 instead (q and k are set to 0 there, and the output's dimensions behind it are not
// written).
// UNI: 16 consecutive keys from a multiple of 16 on lie in one page (page_size is a multiple of 16), so a page's address is a
// scalar and a lane's place under it a constant 32-bit offset; else every lane looks up its own keys' pages.
template <typename T, int NS, int DP, int RT, bool FULL, bool UNI>
__global__ __launch_bounds__(256, DP == 256 || RT * NS > 2 || !UNI ? 1 : 2) void k_few(TreeP P) {
  typedef typename Vec8<T>::type V8;
  constexpr int KS = DP / 32, MT = DP / 16, ROWS = 16 * RT, PIECES = DP / 8;
  constexpr int OS = DP + 4;  // output rows in LDS: 16 rows of a float4 store on different banks
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const fa_tree_attention_args& a = P.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r16 = lane & 15, g4 = lane >> 4;
  Where w;
  if (!locate(P, w)) return;
  const int D = a.head_dim, r0 = w.q_tile * ROWS, k0 = w.split * P.chunk;
  const T* const kbase = reinterpret_cast<const T*>(a.k_cache) + w.h * a.k_head;
  const T* const vbase = reinterpret_cast<const T*>(a.v_cache) + w.h * a.v_head;
  const int32_t* const table = a.block_table + w.b * a.table_seq;
  T* const vl = reinterpret_cast<T*>(smem) + wave * 32 * DP;

  // the page numbers a tile needs: of this lane's keys 16 t + r16, or of the keys 16 t (lane t). They are looked at a tile
  // later: nothing waits for their load; nor does it wait for the lengths (entries behind the end are read, never used)
  typedef typename std::conditional<UNI, int, int2>::type Ids;
  auto page_ids = [&](int kt) -> Ids {
    auto entry = [&](int key) { return table[min(P.page_div.div((uint32_t)key), (uint32_t)a.table_len - 1)]; };
    if constexpr (UNI) return entry(kt + 16 * (lane & 1));
    else return make_int2(entry(kt + r16), entry(kt + 16 + r16));
  };
  int kt = k0 + 32 * wave;
  Ids ids = page_ids(kt);
  const SeqLens L = seq_lens(P, w.b);
  const int rows = L.n * P.group;
  if (r0 >= rows || w.split >= L.splits) return;
  const int k1 = w.split == L.splits - 1 ? L.total : min(L.total, k0 + P.chunk);
  V8 kr[2][KS], vr[2][KS];
  uint32_t present = 0;
  const uint32_t klane = UNI ? r16 * P.k_slot : 0, vlane = UNI ? r16 * P.v_slot : 0;
  // every lane loads: without a page, or behind the end, from page 0 or the page's rest, which the masks then leave out
  auto issue = [&](int kt, Ids ids) {
    present = 0;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint32_t key = (uint32_t)(kt + 16 * t) + (UNI ? 0 : r16);
      int id;
      if constexpr (UNI) id = __builtin_amdgcn_readlane(ids, t);
      else id = t ? ids.y : ids.x;
      const bool ok = (uint32_t)id < (uint32_t)a.pages && (int)key < k1;
      const int own = ok ? -1 : 0;  // (all bits)
      const uint32_t page = id & own, off = (key - P.page_div.div(key) * a.page_size) & own;
      const uint64_t ko = (uint64_t)page * P.k_page + (uint64_t)off * P.k_slot;
      const T* const kp = kbase + ko;
      const T* const vp = vbase + (P.one_offset ? ko : (uint64_t)page * P.v_page + (uint64_t)off * P.v_slot);
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int e = 8 * (g4 + 4 * ks);
        const uint32_t ec = FULL || e < D ? e : 0;
        kr[t][ks] = piece_at(kp, klane + ec);
        vr[t][ks] = piece_at(vp, vlane + ec);
      }
      if constexpr (UNI) present |= ok ? ((1u << min(k1 - (int)key, 16)) - 1) << (16 * t) : 0;
      else present |= (uint32_t)(__ballot(ok) & 0xFFFF) << (16 * t);
    }
  };
  if (kt < k1) {
    issue(kt, ids);
    ids = page_ids(kt + 128);
  }

  int node[RT];
  V8 q[RT][KS][NS];
  float c[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) node[rt] = load_q<T, NS, KS>(P, w, r0 + 16 * rt + r16, rows, g4, q[rt], c[rt]);
  float m[RT], l[RT];  // maximum of the scores as the products give them (c[] not applied), sum of the weights
  f32x4 o[RT][MT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = -INFINITY;
    l[rt] = 0.f;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) o[rt][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  bool bad = false;
  for (; kt < k1; kt += 128) {
    if constexpr (!FULL)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        if (8 * (g4 + 4 * ks) >= D) kr[0][ks] = kr[1][ks] = V8{};  // (as in q: an infinity there would make NaN)
    f32x4 s[RT][1][2];  // 32 keys x rows
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) s[rt][0][0] = s[rt][0][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int ks = 0; ks < KS; ++ks)  // (2 RT sums side by side: a matrix instruction need not wait for the one before it)
#pragma unroll
      for (int n = NS - 1; n >= 0; --n)
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) s[rt][0][t] = mfma16(kr[t][ks], q[rt][ks][n], s[rt][0][t]);
    if constexpr (NS > 1)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
        first_term_for_nan(s[rt][0], [&](int t) {
          f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int ks = 0; ks < KS; ++ks) x = mfma16(kr[t][ks], q[rt][ks][0], x);
          return x;
        });
    const bool drafted = kt + 32 > L.ctx;  // the tile reaches the drafted keys or the end
    if (drafted || present != 0xFFFFFFFFu) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const bool gone = !((present >> (16 * t + r16)) & 1);
        const uint32_t own = kt + 16 * t + r16 >= L.ctx ? ~0u : 0u;  // a drafted key's (no branch: 60.5 -> 59.5 us, 32 sequences)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          if (gone) vr[t][ks] = V8{};  // whatever lies there must not meet a weight of 0
          if (drafted) bad |= strip_nonfinite<T>(vr[t][ks], own);
        }
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) apply_mask(seen_bits(P, w.b, L.ctx, kt, present, node[rt], g4), s[rt][0]);
    }
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int key = 16 * t + r16;
        *reinterpret_cast<V8*>(vl + key * DP + 8 * ((g4 + 4 * ks) ^ (key & (PIECES - 1)))) = vr[t][ks];
      }
    if (kt + 128 < k1) {  // the next tile's loads go out before the softmax
      issue(kt + 128, ids);
      ids = page_ids(kt + 256);
    }
    V8 p[RT][NS];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      softmax_step<T, MT, 1>(s[rt], c[rt], m[rt], l[rt], o[rt]);
      to_terms<T, NS>(s[rt][0], p[rt]);
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const int key = 4 * g4 + (r16 >> 2), piece = 2 * mt + ((r16 >> 1) & 1);
      const T* const at = vl + key * DP + 8 * (piece ^ (key & (PIECES - 1))) + 4 * (r16 & 1);
      const T* const at2 = vl + (key + 16) * DP + 8 * (piece ^ ((key + 16) & (PIECES - 1))) + 4 * (r16 & 1);
      const V8 v = values_operand<T>(at, at2);
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int n = NS - 1; n >= 0; --n) o[rt][mt] = mfma16(v, p[rt][n], o[rt][mt]);
    }
  }

  if (__any(bad))
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
      add_nonfinite<T, NS, DP>(P, w, L, k0 + 32 * wave, k1, 128, node[rt], q[rt], c[rt], m[rt], reinterpret_cast<float*>(vl),
                               o[rt]);

  // the four waves' results join through LDS
  float* const lo = reinterpret_cast<float*>(smem);  // [4][ROWS][OS]
  float* const lml = lo + 4 * ROWS * OS;             // [4][ROWS][2]
  __syncthreads();
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row = 16 * rt + r16;
    const float sum = across_sum(l[rt]);
    if (g4 == 0) {
      lml[(wave * ROWS + row) * 2] = base_of<T>(m[rt], c[rt]);
      lml[(wave * ROWS + row) * 2 + 1] = sum;
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
      *reinterpret_cast<f32x4*>(lo + (wave * ROWS + row) * OS + 16 * mt + 4 * g4) = o[rt][mt];
  }
  __syncthreads();
  for (int u = threadIdx.x; u < ROWS * (DP / 4); u += 256) {
    const int row = u / (DP / 4), e = 4 * (u % (DP / 4)), rr = r0 + row;
    if (rr >= rows || e >= D) continue;
    float top = -INFINITY;
#pragma unroll
    for (int v = 0; v < 4; ++v) top = fmaxf(top, lml[(v * ROWS + row) * 2]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const float f = exp2_fast(lml[(v * ROWS + row) * 2] - base);
      sum += f * lml[(v * ROWS + row) * 2 + 1];
      x += f * *reinterpret_cast<const f32x4*>(lo + (v * ROWS + row) * OS + e);
    }
    if (L.splits > 1) {
      const int64_t at = (((int64_t)w.b * a.kv_heads + w.h) * P.splits + w.split) * P.rows + rr;
      *reinterpret_cast<f32x4*>(P.part_o + at * DP + e) = x;
      if (e == 0) *reinterpret_cast<float2*>(P.part_ml + at * 2) = make_float2(top, sum);
    } else {
      const int nd = (int)P.group_div.div((uint32_t)rr);
      const int64_t at = w.b * a.out_seq + nd * a.out_node + (int64_t)(w.h * P.group + rr - nd * P.group) * a.out_head + e;
      typedef typename std::conditional<(NS > 1), float, T>::type TO;
      store4(reinterpret_cast<TO*>(a.out) + at, x * (sum == 0.f ? 0.f : 1.f / sum), D - e);
    }
  }
}

// KT keys a tile. UNI: KPS consecutive keys from a multiple of KPS on lie in one page
template <typename T, int NS, int DP, int RT, int KT, bool UNI>
__global__ __launch_bounds__(256, DP == 256 || RT * NS > 2 || !UNI ? 1 : 2) void k_many(TreeP P) {
  typedef typename Vec8<T>::type V8;
  constexpr int KS = DP / 32, MT = DP / 16, ROWS = 64 * RT, PIECES = DP / 8, KG = KT / 32;
  constexpr int NL = KT * PIECES / 256;  // pieces of K (and of V) a thread stages
  constexpr int KPS = 256 / PIECES;      // keys staged by one piece of every thread
  extern __shared__ __attribute__((aligned(16))) char smem[];
  T* const lds = reinterpret_cast<T*>(smem);  // [stage][K, V][KT][DP]
  const fa_tree_attention_args& a = P.a;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r16 = lane & 15, g4 = lane >> 4;
  Where w;
  if (!locate(P, w)) return;
  const int D = a.head_dim, r0 = w.q_tile * ROWS, k0 = w.split * P.chunk;
  const T* const kbase = reinterpret_cast<const T*>(a.k_cache) + w.h * a.k_head;
  const T* const vbase = reinterpret_cast<const T*>(a.v_cache) + w.h * a.v_head;
  const int32_t* const table = a.block_table + w.b * a.table_seq;

  // lane i holds the page number of key kt + i, or of key kt + i KPS, looked at a tile later: nothing waits for its load here,
  // nor does it wait for the lengths (entries behind the end are read, never used)
  auto page_id = [&](int kt) -> int {
    const int key = kt + (UNI ? KPS * (lane & (NL - 1)) : lane & (KT - 1));
    return table[min(P.page_div.div((uint32_t)key), (uint32_t)a.table_len - 1)];
  };
  int pid = page_id(k0);
  const SeqLens L = seq_lens(P, w.b);
  const int rows = L.n * P.group;
  if (r0 >= rows || w.split >= L.splits) return;
  const int k1 = w.split == L.splits - 1 ? L.total : min(L.total, k0 + P.chunk);
  V8 kr[NL], vr[NL];
  uint64_t arrived = 0, present = 0;  // the keys that exist, of the tile being loaded and of the one at hand
  const int piece = tid & (PIECES - 1), ec = 8 * piece < D ? 8 * piece : 0, row = tid / PIECES;
  const uint32_t klane = (UNI ? row * P.k_slot : 0) + ec, vlane = (UNI ? row * P.v_slot : 0) + ec;
  auto issue = [&](int kt, int pid) {
    if constexpr (UNI) arrived = 0;
    else arrived = __ballot((uint32_t)pid < (uint32_t)a.pages && kt + lane < k1) & (KT == 64 ? ~0ull : (1ull << KT) - 1);
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int k = i * KPS + (UNI ? 0 : row);
      const uint32_t key = (uint32_t)(kt + k);
      int id;
      if constexpr (UNI) id = __builtin_amdgcn_readlane(pid, i);
      else id = __shfl(pid, k);
      const bool ok = (uint32_t)id < (uint32_t)a.pages && (int)key < k1;
      const int own = ok ? -1 : 0;  // (all bits)
      const uint32_t page = id & own, off = (key - P.page_div.div(key) * a.page_size) & own;
      const uint64_t ko = (uint64_t)page * P.k_page + (uint64_t)off * P.k_slot;
      const T* const kp = kbase + ko;
      const T* const vp = vbase + (P.one_offset ? ko : (uint64_t)page * P.v_page + (uint64_t)off * P.v_slot);
      kr[i] = piece_at(kp, klane);
      vr[i] = piece_at(vp, vlane);
      if constexpr (UNI) arrived |= ok ? ((1ull << min(k1 - (int)key, KPS)) - 1) << (i * KPS) : 0;
    }
  };
  int next = -1;
  if (k0 < k1) {
    issue(k0, pid);
    next = page_id(k0 + KT);
  }

  int node[RT];
  V8 q[RT][KS][NS];
  float c[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt)
    node[rt] = load_q<T, NS, KS>(P, w, r0 + (wave * RT + rt) * 16 + r16, rows, g4, q[rt], c[rt]);
  float m[RT], l[RT];  // maximum of the scores as the products give them (c[] not applied), sum of the weights
  f32x4 o[RT][MT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = -INFINITY;
    l[rt] = 0.f;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) o[rt][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  int stage = 0;
  bool bad = false;
  for (int kt = k0; kt < k1; kt += KT, stage ^= 1) {
    T* const lk = lds + stage * 2 * KT * DP;
    T* const lv = lk + KT * DP;
    present = arrived;
    const bool drafted = kt + KT > L.ctx;
    const bool masked = drafted || present != (KT == 64 ? ~0ull : (1ull << KT) - 1);
    uint32_t bits[RT][KG];
    if (D != DP)  // a piece behind head_dim: 0, as in q (an infinity there would make NaN)
#pragma unroll
      for (int i = 0; i < NL; ++i)
        if (8 * piece >= D) kr[i] = V8{};
    if (masked) {
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        if (!((present >> (i * KPS + row)) & 1)) vr[i] = V8{};
        if (drafted) bad |= strip_nonfinite<T>(vr[i], kt + i * KPS + row >= L.ctx ? ~0u : 0u);
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int g = 0; g < KG; ++g)
          bits[rt][g] = seen_bits(P, w.b, L.ctx, kt + 32 * g, (uint32_t)(present >> (32 * g)), node[rt], g4);
    }
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int k = i * KPS + row, at = k * DP + 8 * (piece ^ (k & (PIECES - 1)));
      *reinterpret_cast<V8*>(lk + at) = kr[i];
      *reinterpret_cast<V8*>(lv + at) = vr[i];
    }
    pid = next;
    if (kt + KT < k1) {
      issue(kt + KT, pid);
      next = page_id(kt + 2 * KT);
    }
    // one barrier a tile: a wave writes this stage again two tiles on, behind the barrier at which all have left it
    __syncthreads();

    f32x4 s[RT][KG][2];
    __builtin_amdgcn_s_setprio(1);  // the other block's wave does its softmax in between (205 -> 201 us)
#pragma unroll
    for (int g = 0; g < KG; ++g) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) s[rt][g][0] = s[rt][g][1] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const int key = 32 * g + 16 * t + r16;
          const V8 k = *reinterpret_cast<const V8*>(lk + key * DP + 8 * ((g4 + 4 * ks) ^ (key & (PIECES - 1))));
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int n = NS - 1; n >= 0; --n) s[rt][g][t] = mfma16(k, q[rt][ks][n], s[rt][g][t]);
        }
    }
    __builtin_amdgcn_s_setprio(0);
    if constexpr (NS > 1)
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int g = 0; g < KG; ++g)
          first_term_for_nan(s[rt][g], [&](int t) {
            f32x4 x = {0.f, 0.f, 0.f, 0.f};
            const int key = 32 * g + 16 * t + r16;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
              x = mfma16(*reinterpret_cast<const V8*>(lk + key * DP + 8 * ((g4 + 4 * ks) ^ (key & (PIECES - 1)))), q[rt][ks][0], x);
            return x;
          });
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      if (masked)
#pragma unroll
        for (int g = 0; g < KG; ++g) apply_mask(bits[rt][g], s[rt][g]);
      softmax_step<T, MT, KG>(s[rt], c[rt], m[rt], l[rt], o[rt]);
    }
#pragma unroll
    for (int g = 0; g < KG; ++g) {
      V8 p[RT][NS];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) to_terms<T, NS>(s[rt][g], p[rt]);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int key = 32 * g + 4 * g4 + (r16 >> 2), pc = 2 * mt + ((r16 >> 1) & 1);
        const T* const at = lv + key * DP + 8 * (pc ^ (key & (PIECES - 1))) + 4 * (r16 & 1);
        const T* const at2 = lv + (key + 16) * DP + 8 * (pc ^ ((key + 16) & (PIECES - 1))) + 4 * (r16 & 1);
        const V8 v = values_operand<T>(at, at2);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int n = NS - 1; n >= 0; --n) o[rt][mt] = mfma16(v, p[rt][n], o[rt][mt]);
      }
    }
  }

  if (__syncthreads_or(bad))
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
      add_nonfinite<T, NS, DP>(P, w, L, k0, k1, 32, node[rt], q[rt], c[rt], m[rt],
                               reinterpret_cast<float*>(smem) + wave * 512, o[rt]);
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int rr = r0 + (wave * RT + rt) * 16 + r16;
    const float sum = across_sum(l[rt]);
    if (rr >= rows) continue;
    if (L.splits > 1) {
      const int64_t at = (((int64_t)w.b * a.kv_heads + w.h) * P.splits + w.split) * P.rows + rr;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
        if (16 * mt + 4 * g4 < D) *reinterpret_cast<f32x4*>(P.part_o + at * DP + 16 * mt + 4 * g4) = o[rt][mt];
      if (g4 == 0) *reinterpret_cast<float2*>(P.part_ml + at * 2) = make_float2(base_of<T>(m[rt], c[rt]), sum);
    } else {
      typedef typename std::conditional<(NS > 1), float, T>::type TO;
      TO* const out = reinterpret_cast<TO*>(a.out) + w.b * a.out_seq + node[rt] * a.out_node +
                      (int64_t)(w.h * P.group + rr - node[rt] * P.group) * a.out_head;
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) store4(out + 16 * mt + 4 * g4, o[rt][mt] * inv, D - 16 * mt - 4 * g4);
    }
  }
}

// joins the partial results of a row: a wave a row; lane s weighs split s (at most 64), then the lanes go over the dimensions
template <typename TO, int DP>
__global__ __launch_bounds__(256) void k_tree_merge(TreeP P) {
  const fa_tree_attention_args& a = P.a;
  const int lane = threadIdx.x & 63, rr = blockIdx.x * 4 + (threadIdx.x >> 6), h = blockIdx.y, b = blockIdx.z;
  const SeqLens L = seq_lens(P, b);
  if (rr >= L.n * P.group || L.splits == 1) return;
  const int64_t at0 = ((int64_t)b * a.kv_heads + h) * P.splits * P.rows + rr;
  float2 ml = make_float2(-INFINITY, 0.f);
  if (lane < L.splits) ml = *reinterpret_cast<const float2*>(P.part_ml + (at0 + (int64_t)lane * P.rows) * 2);
  const float top = wave_max(ml.x), base = top == -INFINITY ? 0.f : top;
  float f = exp2_fast(ml.x - base);
  const float sum = wave_sum(f * ml.y);
  f *= sum == 0.f ? 0.f : 1.f / sum;
  constexpr int N = DP / 64;
  float x[N] = {};
  // (every lane takes part, also those behind head_dim, whose sums are not stored: their weights are asked for. A partial row
  // has DP places)
  const float* const o = P.part_o + at0 * DP + lane * N;
#pragma unroll 4
  for (int s = 0; s < L.splits; ++s) {
    const float g = __shfl(f, s);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] += g * o[(int64_t)s * P.rows * DP + i];
  }
  const int nd = (int)P.group_div.div((uint32_t)rr);
  TO* out = reinterpret_cast<TO*>(a.out) + b * a.out_seq + nd * a.out_node +
            (int64_t)(h * P.group + rr - nd * P.group) * a.out_head + lane * N;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (lane * N + i < a.head_dim) out[i] = (TO)x[i];
}

// ---------------------------------------------------------------------------------------------------------------- host
struct TreePlan {
  TreeP P;
  int dp, rt;
  bool many;
  int64_t bytes;
};

static TreePlan tree_plan(const fa_tree_attention_args* ap) {
  FA_REQUIRE(ap, "tree_attention: no arguments");
  TreePlan t;
  t.P.a = *ap;
  fa_tree_attention_args& a = t.P.a;
  FA_REQUIRE(a.seqs >= 0 && a.nodes >= 0 && a.heads >= 1 && a.kv_heads >= 1 && a.heads % a.kv_heads == 0,
             "tree_attention: heads must be a multiple of kv_heads");
  FA_REQUIRE(a.seqs <= 65535 && a.kv_heads <= 1024, "tree_attention: more than 65535 sequences or 1024 kv heads");
  FA_REQUIRE(a.head_dim >= 8 && a.head_dim <= 256 && a.head_dim % 8 == 0,
             "tree_attention: head_dim must be a multiple of 8 up to 256");
  FA_REQUIRE(a.cache_type == FA_F16 || a.cache_type == FA_BF16, "tree_attention: the cache is float16 or bfloat16");
  FA_REQUIRE(a.q_type == FA_F32 || a.q_type == a.cache_type, "tree_attention: q is float32 or of the cache's type");
  FA_REQUIRE(a.page_size >= 1 && a.pages >= 1 && a.table_len >= 1, "tree_attention: pages");
  FA_REQUIRE((int64_t)a.table_len * a.page_size + a.nodes < (1ll << 31) - 256, "tree_attention: more than 2^31 positions");
  FA_REQUIRE(a.scale > 0.f && a.scale < 1e30f, "tree_attention: scale must be positive");
  const int group = a.heads / a.kv_heads;
  FA_REQUIRE((int64_t)a.nodes * group <= 65535, "tree_attention: more than 65535 rows of one kv head");
  t.P.group = group;
  t.P.rows = a.nodes * group;
  t.P.c = a.scale * 1.4426950408889634f;
  t.P.page_div = FastDiv::of((uint32_t)a.page_size);
  t.P.group_div = FastDiv::of((uint32_t)group);
  t.dp = a.head_dim <= 64 ? 64 : a.head_dim <= 128 ? 128 : 256;
  // up to 32 rows: k_few; more: k_many, 64 rows a block, or 128 where there are as many and registers allow
  t.many = t.P.rows > 32 || (t.dp == 256 && t.P.rows > 16);
  t.rt = t.many ? (t.P.rows > 64 && t.dp <= 128 && a.q_type != FA_F32 ? 2 : 1) : t.P.rows <= 16 ? 1 : 2;
  const int rows_block = t.many ? 64 * t.rt : 16 * t.rt;
  t.P.q_tiles = (t.P.rows + rows_block - 1) / rows_block;
  t.bytes = 0;
  t.P.splits = 1;
  t.P.chunk = 1 << 30;
  if (a.seqs == 0 || a.nodes == 0) return t;
  // The keys are split w ways so that rounds(w) (keys / w + 256), and 300 for the launch that joins them, is least: two blocks
  // a compute unit are resident at once, and a block's beginning and end weigh about as much as 256 keys. (32 sequences of up
  // to 2048 keys on 8 kv heads: 2 ways 50 us, 3: 60, 1: 57; 4 long ones with two row tiles: 8 ways 241 us, 16: 258.)
  const int64_t cap = (int64_t)a.table_len * a.page_size;
  const int64_t keys = std::max<int64_t>(1, std::min<int64_t>(cap, a.max_context > 0 ? (int64_t)a.max_context + a.nodes : cap));
  const int64_t base = (int64_t)a.seqs * a.kv_heads * t.P.q_tiles, slots = 2ll * cu_count();
  int64_t ways = 1, least = INT64_MAX;
  for (int64_t w = 1; w <= std::min<int64_t>(64, (keys + 127) / 128); ++w) {
    const int64_t cost = (base * w + slots - 1) / slots * ((keys + w - 1) / w + 256) + (w > 1 ? 300 : 0);
    if (cost < least) least = cost, ways = w;
  }
  const int64_t chunk = ((keys + ways - 1) / ways + 127) / 128 * 128;
  t.P.chunk = (int)chunk;
  t.P.splits = (int)((keys + chunk - 1) / chunk);
  t.P.q_tiles_div = FastDiv::of((uint32_t)std::max(1, t.P.q_tiles));
  t.P.kv_div = FastDiv::of((uint32_t)a.kv_heads);
  t.P.splits_div = FastDiv::of((uint32_t)t.P.splits);
  const int64_t groups = (int64_t)a.seqs * a.kv_heads * t.P.splits;
  FA_REQUIRE((groups + 7) / 8 * 8 * t.P.q_tiles < (1ll << 31), "tree_attention: more than 2^31 blocks");
  t.P.n_groups = (int)groups;
  if (t.P.splits > 1)
    t.bytes = (int64_t)a.seqs * a.kv_heads * t.P.splits * t.P.rows * (t.dp + 2) * (int64_t)sizeof(float);
  return t;
}

// a kernel's LDS beyond 64 KB has to be asked for, once on every device; what fails is asked for again by the next call
template <auto KERNEL, size_t LDS>
static void tree_launch(const TreeP& P, hipStream_t s) {
  if constexpr (LDS > 65536) {
    static std::atomic<uint64_t> asked{0};  // a bit a device
    int dev = 0;
    FA_HIP(hipGetDevice(&dev));
    const uint64_t bit = dev < 64 ? 1ull << dev : 0;
    if (!(asked.load(std::memory_order_relaxed) & bit)) {
      FA_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, (int)LDS));
      asked.fetch_or(bit, std::memory_order_relaxed);
    }
  }
  launch(KERNEL, dim3((uint32_t)((P.n_groups + 7) / 8 * 8) * P.q_tiles), dim3(256), LDS, s, P);
}
template <typename T, int NS, int DP, int RT>
static void run_few(const TreeP& P, hipStream_t s) {
  constexpr int ROWS = 16 * RT;
  constexpr size_t lds = std::max<size_t>(4 * 32 * DP * 2, 4 * ROWS * (DP + 4) * 4 + 4 * ROWS * 2 * 4);
  const bool full = P.a.head_dim == DP;
  if (P.uniform % 16 == 0)
    full ? tree_launch<k_few<T, NS, DP, RT, true, true>, lds>(P, s) : tree_launch<k_few<T, NS, DP, RT, false, true>, lds>(P, s);
  else
    tree_launch<k_few<T, NS, DP, RT, false, false>, lds>(P, s);
}
template <typename T, int NS, int DP, int RT>
static void run_many(const TreeP& P, hipStream_t s) {
  constexpr int KT = DP == 256 ? 32 : 64;
  constexpr size_t lds = 4 * KT * DP * 2;  // two stages of K and V
  constexpr int KPS = 2048 / DP;
  P.uniform % KPS == 0 ? tree_launch<k_many<T, NS, DP, RT, KT, true>, lds>(P, s)
                       : tree_launch<k_many<T, NS, DP, RT, KT, false>, lds>(P, s);
}
template <typename T, int NS, int DP>
static void tree_run(const TreePlan& t, hipStream_t s) {
  if constexpr (DP == 256) {
    t.many ? run_many<T, NS, 256, 1>(t.P, s) : run_few<T, NS, 256, 1>(t.P, s);
  } else if (!t.many) {
    t.rt == 1 ? run_few<T, NS, DP, 1>(t.P, s) : run_few<T, NS, DP, 2>(t.P, s);
  } else if constexpr (NS == 1) {
    t.rt == 1 ? run_many<T, NS, DP, 1>(t.P, s) : run_many<T, NS, DP, 2>(t.P, s);
  } else {
    run_many<T, NS, DP, 1>(t.P, s);
  }
  if (t.P.splits > 1) {
    typedef typename std::conditional<(NS > 1), float, T>::type TO;
    launch(k_tree_merge<TO, DP>, dim3((t.P.rows + 3) / 4, t.P.a.kv_heads, t.P.a.seqs), dim3(256), 0, s, t.P);
  }
}
template <typename T, int NS>
static void tree_dispatch(const TreePlan& t, hipStream_t s) {
  if (t.dp == 64) tree_run<T, NS, 64>(t, s);
  else if (t.dp == 128) tree_run<T, NS, 128>(t, s);
  else tree_run<T, NS, 256>(t, s);
}

int64_t tree_attention_bytes(const fa_tree_attention_args* a) { return tree_plan(a).bytes; }

void tree_attention(const fa_tree_attention_args* ap, hipStream_t s) {
  TreePlan t = tree_plan(ap);
  const fa_tree_attention_args& a = t.P.a;
  if (a.seqs == 0 || a.nodes == 0) return;
  FA_REQUIRE(a.q && a.out && a.k_cache && a.v_cache && a.block_table && a.context_lens, "tree_attention: null tensor");
  FA_REQUIRE(aligned16(a.k_cache) && aligned16(a.v_cache) && a.k_page % 8 == 0 && a.k_head % 8 == 0 && a.k_slot % 8 == 0 &&
                 a.v_page % 8 == 0 && a.v_head % 8 == 0 && a.v_slot % 8 == 0,
             "tree_attention: cache rows must be 16-byte aligned");
  for (const int64_t x : {a.k_page, a.k_slot, a.v_page, a.v_slot})
    FA_REQUIRE(x >= 0 && x < (1ll << 31), "tree_attention: a page or slot stride outside 0 .. 2^31");
  t.P.k_page = (uint32_t)a.k_page;
  t.P.k_slot = (uint32_t)a.k_slot;
  t.P.v_page = (uint32_t)a.v_page;
  t.P.v_slot = (uint32_t)a.v_slot;
  t.P.one_offset = a.k_page == a.v_page && a.k_slot == a.v_slot;
  // UNI's offsets of a lane within a page's rows stay below 2^31 bytes
  t.P.uniform = std::max(a.k_slot, a.v_slot) < (1ll << 24) ? a.page_size : 1;
  FA_REQUIRE(t.bytes == 0 || (a.workspace && a.workspace_bytes >= t.bytes && aligned16(a.workspace)),
             "tree_attention: workspace too small or not 16-byte aligned");
  const int64_t qm = 16 / type_bytes(a.q_type);
  t.P.q_vec = aligned16(a.q) && a.q_seq % qm == 0 && a.q_node % qm == 0 && a.q_head % qm == 0;
  t.P.part_o = reinterpret_cast<float*>(a.workspace);
  t.P.part_ml = t.P.part_o + (int64_t)a.seqs * a.kv_heads * t.P.splits * t.P.rows * t.dp;
  if (a.cache_type == FA_F16) {
    if (a.q_type == FA_F32) tree_dispatch<_Float16, 2>(t, s);
    else tree_dispatch<_Float16, 1>(t, s);
  } else {
    if (a.q_type == FA_F32) tree_dispatch<__bf16, 3>(t, s);
    else tree_dispatch<__bf16, 1>(t, s);
  }
}

}  // namespace fa

extern "C" {

int fa_tree_attention_workspace(const fa_tree_attention_args* a, int64_t* bytes) {
  FA_API_BEGIN
  FA_REQUIRE(bytes, "tree_attention: no place for the size");
  *bytes = fa::tree_attention_bytes(a);
  FA_API_END
}

int fa_tree_attention(const fa_tree_attention_args* a, void* stream) {
  FA_API_BEGIN
  fa::tree_attention(a, reinterpret_cast<hipStream_t>(stream));
  FA_API_END
}

}  // extern "C"

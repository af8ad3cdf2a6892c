// Attention of drafted tokens over a paged cache (fa_tree_attention).
//
// For one sequence and kv head the rows are (drafted token, query head of the group), all of which read the same keys:
//   S = K Q^T,  P = softmax over keys (running maximum and sum, 32 bits),  O^T += V^T P^T.
// A block takes up to 16 RT of those rows and one chunk of the keys; its four waves take every fourth 32-key tile of the
// chunk, each with a running maximum, sum and output of its own, and join at the end through LDS. Blocks of the same rows
// leave partial results (unnormalised output, maximum, sum) that k_tree_merge joins.
//
// Both products run on 16x16x32 matrix instructions. S is made with the keys as rows, so that a lane's results belong to
// one query row (lane % 16) and 4 consecutive keys, in two tiles 8: exactly the operand P^T of the second product, whose
// contraction runs over the keys in that order (4 g + i, then 16 + 4 g + i); V^T is read from LDS in the same order by the
// transposing reads. The output's columns are query rows too, so rescaling needs no exchange between lanes; the running
// maximum needs two. K goes from memory straight into operand registers (a key row is read in 64-byte pieces by 4 lanes),
// V through wave-private LDS whose 32-byte pairs are permuted by the key (pair ^ key % 8): the 16 rows that a transposing
// read touches then cover all banks evenly.
#include "api.h"
#include "draft_ops.h"

#include <algorithm>
#include <type_traits>

namespace fa {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short v4i16 __attribute__((ext_vector_type(4)));

struct TreeP {
  fa_tree_attention_args a;
  FastDiv page_div, group_div;
  int group, rows;     // query heads per kv head; rows of one sequence and kv head: nodes * group
  int q_tiles;         // blocks of 16 RT rows
  int chunk, splits;   // keys per block (a multiple of 128), blocks along the keys at most
  float c;             // scale * log2(e)
  float* part_o;       // [seqs][kv_heads][splits][rows][DP]
  float* part_ml;      // [seqs][kv_heads][splits][rows][2]
  int q_vec, out_vec;  // q / out rows may be accessed in 16-byte pieces
};

__device__ __forceinline__ f32x4 mfma16(f16x8_t a, f16x8_t b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma16(bf16x8_t a, bf16x8_t b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v4i16 ld_tr(const void* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4i16*)(p));
}
// maximum / sum over the four 16-lane groups of a wave
__device__ __forceinline__ float across_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float across_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}
// exponent bits of a 16-bit type, both halves of a register
template <typename T> constexpr uint32_t kExp = 0;
template <> constexpr uint32_t kExp<_Float16> = 0x7C00u;
template <> constexpr uint32_t kExp<__bf16> = 0x7F80u;

struct SeqLens {
  int n, ctx, total, splits;
};
__device__ __forceinline__ SeqLens seq_lens(const TreeP& P, int b) {
  const fa_tree_attention_args& a = P.a;
  SeqLens s;
  s.n = a.draft_lens ? min(max(a.draft_lens[b], 0), a.nodes) : a.nodes;
  const int cap = a.table_len * a.page_size;  // < 2^31 - nodes (checked by the host)
  s.ctx = min(max(a.context_lens[b], 0), cap);
  s.total = min(s.ctx + s.n, cap);
  s.splits = min(P.splits, max(1, (s.total + P.chunk - 1) / P.chunk));
  return s;
}

// T: cache type. NS: 16-bit terms of q and of the probabilities (1: q is of the cache's type; 2 / 3: q is float32, kept to
// 22 / 24 bits by terms of float16 / bfloat16). DP: head_dim rounded up to 64 / 128 / 256.
template <typename T, int NS, int DP, int RT>
__global__ __launch_bounds__(256) void k_tree_attn(TreeP P) {
  typedef typename Vec8<T>::type V8;
  constexpr int KS = DP / 32, MT = DP / 16, ROWS = 16 * RT;
  constexpr int OS = DP + 4;  // output rows in LDS: 16 rows of a float4 store on different banks
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const fa_tree_attention_args& a = P.a;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r16 = lane & 15, g4 = lane >> 4;
  const int b = blockIdx.z, h = blockIdx.y % a.kv_heads, qt = blockIdx.y / a.kv_heads, split = blockIdx.x;
  const SeqLens L = seq_lens(P, b);
  const int rows = L.n * P.group, r0 = qt * ROWS;
  if (r0 >= rows || split >= L.splits) return;
  const int D = a.head_dim;
  const int k0 = split * P.chunk, k1 = split == L.splits - 1 ? L.total : min(L.total, k0 + P.chunk);

  // this lane's query rows, their operands
  int node[RT];
  V8 q[RT][KS][NS];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int rr = r0 + 16 * rt + r16;
    const int rc = min(rr, rows - 1);
    node[rt] = (int)P.group_div.div((uint32_t)rc);
    const int64_t at = b * a.q_seq + node[rt] * a.q_node + (int64_t)(h * P.group + rc - node[rt] * P.group) * a.q_head;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const int e = 8 * (g4 + 4 * ks);
      float x[8] = {};
      if (rr < rows && e < D) {
        if constexpr (NS > 1) {
          const float* p = reinterpret_cast<const float*>(a.q) + at + e;
          if (P.q_vec) load8<true>(p, x);
          else load8<false>(p, x);
        } else {
          const T* p = reinterpret_cast<const T*>(a.q) + at + e;
          if (P.q_vec) load8<true>(p, x);
          else load8<false>(p, x);
        }
      }
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const T y = (T)x[i];
          q[rt][ks][s][i] = y;
          x[i] -= (float)y;
        }
    }
  }

  float m[RT], l[RT];
  f32x4 o[RT][MT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = -INFINITY;
    l[rt] = 0.f;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) o[rt][mt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const T* const kbase = reinterpret_cast<const T*>(a.k_cache) + h * a.k_head;
  const T* const vbase = reinterpret_cast<const T*>(a.v_cache) + h * a.v_head;
  const int32_t* const table = a.block_table + b * a.table_seq;
  T* const vl = reinterpret_cast<T*>(smem) + wave * 32 * DP;

  // page numbers of this lane's two keys of a tile (16 t + r16): -1 behind the end
  auto page_ids = [&](int kt, int (&pid)[2]) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int key = kt + 16 * t + r16;
      pid[t] = key < k1 ? table[P.page_div.div((uint32_t)key)] : -1;
    }
  };
  V8 kr[2][KS], vr[2][KS];
  bool ok[2];
  // every lane loads: one without a key of its own reads page 0, slot 0 (there is one), which the masks then leave out
  auto issue = [&](int kt, const int (&pid)[2]) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const uint32_t key = (uint32_t)(kt + 16 * t + r16);
      ok[t] = pid[t] >= 0 && pid[t] < a.pages;
      const int64_t page = ok[t] ? pid[t] : 0;
      const int64_t off = ok[t] ? key - P.page_div.div(key) * a.page_size : 0;
      const T* kp = kbase + page * a.k_page + off * a.k_slot;
      const T* vp = vbase + page * a.v_page + off * a.v_slot;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int e = 8 * (g4 + 4 * ks);
        kr[t][ks] = *reinterpret_cast<const V8*>(kp + (e < D ? e : 0));
        vr[t][ks] = *reinterpret_cast<const V8*>(vp + (e < D ? e : 0));
      }
    }
  };

  int pid[2];
  int kt = k0 + 32 * wave;
  if (kt < k1) {
    page_ids(kt, pid);
    issue(kt, pid);
    page_ids(kt + 128, pid);
  }
  for (; kt < k1; kt += 128) {
    if (D != DP) {  // dimensions behind the head's: zero
#pragma unroll
      for (int ks = 0; ks < KS; ++ks)
        if (8 * (g4 + 4 * ks) >= D)
#pragma unroll
          for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 8; ++i) kr[t][ks][i] = vr[t][ks][i] = (T)0.f;
    }
    // S: 32 keys x rows
    f32x4 s[RT][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        s[rt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int n = NS - 1; n >= 0; --n) s[rt][t] = mfma16(kr[t][ks], q[rt][ks][n], s[rt][t]);
      }
    const uint32_t present = (uint32_t)(__ballot(ok[0]) & 0xFFFF) | (uint32_t)((__ballot(ok[1]) & 0xFFFF) << 16);
    const bool drafted = kt + 32 > L.ctx;  // the tile reaches the drafted keys or the end
    const bool masked = present != 0xFFFFFFFFu || drafted;
    bool bad = false;
    if (masked) {
      // an absent key's value is zero; an infinity or NaN in a drafted key's value must not reach the rows that do not see
      // that key (0 * inf), so it leaves the tile and is added to the others alone
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          if (!ok[t])
#pragma unroll
            for (int i = 0; i < 8; ++i) vr[t][ks][i] = (T)0.f;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t u = __builtin_bit_cast(uint16_t, (T)vr[t][ks][i]);
            if (drafted && (u & kExp<T>) == kExp<T>) {
              bad = true;
              vr[t][ks][i] = (T)0.f;
            }
          }
        }
      bad = __any(bad);
    }
    // V to LDS
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const int key = 16 * t + r16, cidx = g4 + 4 * ks;
        const int pair = (cidx >> 1) ^ (key & (MT >= 8 ? 7 : MT - 1));
        *reinterpret_cast<V8*>(vl + key * DP + 16 * pair + 8 * (cidx & 1)) = vr[t][ks];
      }
    // the next tile's loads go out before the softmax
    if (kt + 128 < k1) {
      issue(kt + 128, pid);
      page_ids(kt + 256, pid);
    }
    if (masked) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const uint8_t* mrow = a.mask ? a.mask + b * a.mask_seq + node[rt] * a.mask_row : nullptr;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int kk = 16 * t + 4 * g4 + i, j = kt + kk - L.ctx;
            bool seen = (present >> kk) & 1;
            if (seen && j >= 0) seen = mrow ? mrow[j] != 0 : j <= node[rt];
            if (!seen) s[rt][t][i] = -INFINITY;
          }
      }
    }
    V8 p[RT][NS];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float top = s[rt][0][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) top = fmaxf(top, s[rt][i >> 2][i & 3]);
      top = fmaxf(m[rt], across_max(top));
      const float base = top == -INFINITY ? 0.f : top;  // nothing seen so far: every weight is exp2(-inf) = 0
      const float alpha = exp2f((m[rt] - base) * P.c);
      m[rt] = top;
      float e[8], sum = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        e[i] = exp2f((s[rt][i >> 2][i & 3] - base) * P.c);
        sum += e[i];
      }
      l[rt] = l[rt] * alpha + sum;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) o[rt][mt] *= alpha;
      if (bad) {
        for (int g = 0; g < 4; ++g)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int key = kt + 16 * (i >> 2) + 4 * g + (i & 3);
            const float w = __shfl(e[i], 16 * g + r16);
            if (key >= k1) continue;
            const uint32_t pg = P.page_div.div((uint32_t)key);
            const int id = table[pg];
            if (id < 0 || id >= a.pages) continue;
            const T* vp = vbase + id * a.v_page + (int64_t)((uint32_t)key - pg * a.page_size) * a.v_slot;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt)
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const int d = 16 * mt + 4 * g4 + j;
                const float x = d < D ? (float)vp[d] : 0.f;
                if (!(fabsf(x) < INFINITY) && w != 0.f) o[rt][mt][j] += w * x;
              }
          }
      }
#pragma unroll
      for (int n = 0; n < NS; ++n)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const T y = (T)e[i];
          p[rt][n][i] = y;
          e[i] -= (float)y;
        }
    }
    // O^T += V^T P^T
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      V8 v;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int key = 16 * t + 4 * g4 + (r16 >> 2);
        const int pair = mt ^ (key & (MT >= 8 ? 7 : MT - 1));
        const v4i16 x = ld_tr(vl + key * DP + 16 * pair + 4 * (r16 & 3));
        const auto y = __builtin_bit_cast(T __attribute__((ext_vector_type(4))), x);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * t + i] = y[i];
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int n = NS - 1; n >= 0; --n) o[rt][mt] = mfma16(v, p[rt][n], o[rt][mt]);
    }
  }

  // the four waves' results join through LDS
  float* const lo = reinterpret_cast<float*>(smem);                 // [4][ROWS][OS]
  float* const lml = lo + 4 * ROWS * OS;                            // [4][ROWS][2]
  __syncthreads();
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int row = 16 * rt + r16;
    const float sum = across_sum(l[rt]);
    if (g4 == 0) {
      lml[(wave * ROWS + row) * 2] = m[rt];
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
    for (int w = 0; w < 4; ++w) top = fmaxf(top, lml[(w * ROWS + row) * 2]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
    f32x4 x = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = exp2f((lml[(w * ROWS + row) * 2] - base) * P.c);
      sum += f * lml[(w * ROWS + row) * 2 + 1];
      x += f * *reinterpret_cast<const f32x4*>(lo + (w * ROWS + row) * OS + e);
    }
    if (L.splits > 1) {
      const int64_t at = (((int64_t)b * a.kv_heads + h) * P.splits + split) * P.rows + rr;
      *reinterpret_cast<f32x4*>(P.part_o + at * DP + e) = x;
      if (e == 0) {
        P.part_ml[at * 2] = top;
        P.part_ml[at * 2 + 1] = sum;
      }
    } else {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const int nd = (int)P.group_div.div((uint32_t)rr);
      const int64_t at = b * a.out_seq + nd * a.out_node + (int64_t)(h * P.group + rr - nd * P.group) * a.out_head + e;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (NS > 1) reinterpret_cast<float*>(a.out)[at + i] = x[i] * inv;
        else reinterpret_cast<T*>(a.out)[at + i] = (T)(x[i] * inv);
      }
    }
  }
}

// joins the partial results of a row: a wave a row, lanes over the dimensions
template <typename TO, int DP>
__global__ __launch_bounds__(256) void k_tree_merge(TreeP P) {
  const fa_tree_attention_args& a = P.a;
  const int lane = threadIdx.x & 63, rr = blockIdx.x * 4 + (threadIdx.x >> 6), h = blockIdx.y, b = blockIdx.z;
  const SeqLens L = seq_lens(P, b);
  if (rr >= L.n * P.group || L.splits == 1) return;
  const int64_t at0 = ((int64_t)b * a.kv_heads + h) * P.splits * P.rows + rr;
  float top = -INFINITY;
  for (int s = 0; s < L.splits; ++s) top = fmaxf(top, P.part_ml[(at0 + (int64_t)s * P.rows) * 2]);
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f, x[DP / 64] = {};
  for (int s = 0; s < L.splits; ++s) {
    const int64_t at = at0 + (int64_t)s * P.rows;
    const float f = exp2f((P.part_ml[at * 2] - base) * P.c);
    sum += f * P.part_ml[at * 2 + 1];
#pragma unroll
    for (int i = 0; i < DP / 64; ++i)
      if (lane + 64 * i < a.head_dim) x[i] += f * P.part_o[at * DP + lane + 64 * i];
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int nd = (int)P.group_div.div((uint32_t)rr);
  TO* out = reinterpret_cast<TO*>(a.out) + b * a.out_seq + nd * a.out_node +
            (int64_t)(h * P.group + rr - nd * P.group) * a.out_head;
#pragma unroll
  for (int i = 0; i < DP / 64; ++i)
    if (lane + 64 * i < a.head_dim) out[lane + 64 * i] = (TO)(x[i] * inv);
}

// ---------------------------------------------------------------------------------------------------------------- host
struct TreePlan {
  TreeP P;
  int dp, rt;
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
  t.rt = t.dp == 256 || t.P.rows <= 16 ? 1 : 2;
  t.P.q_tiles = (t.P.rows + 16 * t.rt - 1) / (16 * t.rt);
  FA_REQUIRE((int64_t)t.P.q_tiles * a.kv_heads <= 65535, "tree_attention: too many rows");
  t.bytes = 0;
  t.P.splits = 1;
  t.P.chunk = 1 << 30;
  if (a.seqs == 0 || a.nodes == 0) return t;
  // keys are split until the launch has about four blocks a compute unit, in chunks of at least 256 keys
  const int64_t cap = (int64_t)a.table_len * a.page_size;
  const int64_t keys = std::max<int64_t>(1, std::min<int64_t>(cap, a.max_context > 0 ? (int64_t)a.max_context + a.nodes : cap));
  const int64_t base = (int64_t)a.seqs * a.kv_heads * t.P.q_tiles;
  const int64_t want = std::max<int64_t>(1, (4ll * cu_count() + base - 1) / base);
  int64_t chunk = std::max<int64_t>(256, (keys + want - 1) / want);
  chunk = (chunk + 127) / 128 * 128;
  t.P.chunk = (int)chunk;
  t.P.splits = (int)((keys + chunk - 1) / chunk);
  if (t.P.splits > 1)
    t.bytes = (int64_t)a.seqs * a.kv_heads * t.P.splits * t.P.rows * (t.dp + 2) * (int64_t)sizeof(float);
  return t;
}

template <typename T, int NS, int DP, int RT>
static void tree_run(const TreeP& P, hipStream_t s) {
  constexpr int ROWS = 16 * RT;
  constexpr size_t lds = std::max<size_t>(4 * 32 * DP * 2, 4 * ROWS * (DP + 4) * 4 + 4 * ROWS * 2 * 4);
  const fa_tree_attention_args& a = P.a;
  if constexpr (lds > 65536) {
    static const hipError_t once = hipFuncSetAttribute(reinterpret_cast<const void*>(k_tree_attn<T, NS, DP, RT>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    FA_HIP(once);
  }
  launch(k_tree_attn<T, NS, DP, RT>, dim3(P.splits, a.kv_heads * P.q_tiles, a.seqs), dim3(256), lds, s, P);
  if (P.splits > 1) {
    typedef typename std::conditional<(NS > 1), float, T>::type TO;
    launch(k_tree_merge<TO, DP>, dim3((P.rows + 3) / 4, a.kv_heads, a.seqs), dim3(256), 0, s, P);
  }
}
template <typename T, int NS>
static void tree_dispatch(const TreePlan& t, hipStream_t s) {
  if (t.dp == 64) t.rt == 1 ? tree_run<T, NS, 64, 1>(t.P, s) : tree_run<T, NS, 64, 2>(t.P, s);
  else if (t.dp == 128) t.rt == 1 ? tree_run<T, NS, 128, 1>(t.P, s) : tree_run<T, NS, 128, 2>(t.P, s);
  else tree_run<T, NS, 256, 1>(t.P, s);
}

static void tree_attention(const fa_tree_attention_args* ap, hipStream_t s) {
  TreePlan t = tree_plan(ap);
  const fa_tree_attention_args& a = t.P.a;
  if (a.seqs == 0 || a.nodes == 0) return;
  FA_REQUIRE(a.q && a.out && a.k_cache && a.v_cache && a.block_table && a.context_lens, "tree_attention: null tensor");
  FA_REQUIRE(aligned16(a.k_cache) && aligned16(a.v_cache) && a.k_page % 8 == 0 && a.k_head % 8 == 0 && a.k_slot % 8 == 0 &&
                 a.v_page % 8 == 0 && a.v_head % 8 == 0 && a.v_slot % 8 == 0,
             "tree_attention: cache rows must be 16-byte aligned");
  FA_REQUIRE(t.bytes == 0 || (a.workspace && a.workspace_bytes >= t.bytes && aligned16(a.workspace)),
             "tree_attention: workspace too small or not 16-byte aligned");
  const int64_t qm = 16 / type_bytes(a.q_type);
  t.P.q_vec = aligned16(a.q) && a.q_seq % qm == 0 && a.q_node % qm == 0 && a.q_head % qm == 0;
  t.P.out_vec = 0;
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
  *bytes = fa::tree_plan(a).bytes;
  FA_API_END
}

int fa_tree_attention(const fa_tree_attention_args* a, void* stream) {
  FA_API_BEGIN
  fa::tree_attention(a, reinterpret_cast<hipStream_t>(stream));
  FA_API_END
}

}  // extern "C"

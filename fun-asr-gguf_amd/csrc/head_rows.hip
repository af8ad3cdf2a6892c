// Head norms with the rotation, and the append to a paged cache (fa_qk_norm_rope, fa_kv_append).
//
// Per head row x of head_dim D: y = x * rsqrt(mean x^2 + eps) * w, then the pairs of the first R dimensions turned by the
// token's angles. Each row is read once and written once, with one pass of arithmetic in between: memory bound.
//
// A row is held by a group of D / 16 lanes, two runs of 8 elements a lane: the two halves of its own 8 pairs, so that the
// rotation needs no exchange between lanes. Half-split pairs (i, i + R/2): runs at 8 p and R/2 + 8 p; neighbouring pairs, and
// the dimensions behind R: runs at 16 p and 16 p + 8. The sum of squares is the only thing the lanes share. A wave thus moves
// floor(64 / (D / 16)) rows with 16-byte accesses (heads of 80 in groups of eight lanes, three idle: 45.6 us, of five: 40.3).
// Several rows of a token in one group, to read its angles once, cost registers and bring nothing (24 f32 heads of 128: four
// rows 35 us, one 31). Measured: 6528 tokens of 16 + 8 f32 heads of 128 31 us, 5.2 TB/s read and written; one token 2.9 us, the
// launch; 16384 tokens of 8 + 8 bf16 heads of 64 appended 15 us, 4.8 TB/s.
#include "api.h"
#include "draft_ops.h"

#include <algorithm>

namespace fa {

struct HeadRowsP {
  fa_head_rows_args a;
  FastDiv slots_div;  // by n_slots
  FastDiv page_div;
  FastDiv lpr_div;    // by the lanes of a row
  uint32_t lpr, wave_rows;  // lanes of a row, rows of a wave
  float inv_dim;
  int n_slots;        // head rows per token: heads + kv_heads (+ kv_heads of v)
  uint32_t n_rows;
};

__device__ __forceinline__ int64_t index_at(const void* p, int is64, int64_t i) {
  return is64 ? reinterpret_cast<const int64_t*>(p)[i] : (int64_t) reinterpret_cast<const int32_t*>(p)[i];
}

template <typename TI, typename TC, bool VEC>
__global__ __launch_bounds__(256) void k_head_rows(HeadRowsP P) {
  const fa_head_rows_args& a = P.a;
  const uint32_t lane = threadIdx.x & 63, group = P.lpr_div.div(lane);
  const uint32_t row = (blockIdx.x * 4 + (threadIdx.x >> 6)) * P.wave_rows + group;
  if (group >= P.wave_rows || row >= P.n_rows) return;
  const int p = (int)(lane - group * P.lpr);
  const int t = (int)P.slots_div.div(row), s = (int)(row - (uint32_t)t * P.n_slots);
  const int R = a.rot_dim;
  const bool rot = a.cos && 16 * p < R;
  const bool halves = rot && !a.interleaved;
  const int e0 = halves ? 8 * p : 16 * p, e1 = halves ? R / 2 + 8 * p : 16 * p + 8;
  float c[8], sn[8];
  if (a.cos) {
    const int64_t pos = index_at(a.positions, a.positions_64, t);
    if (pos < 0 || pos >= a.table_len) return;  // (the whole group: its lanes share the token)
    if (rot) {
      load8<VEC>(a.cos + pos * (R / 2) + 8 * p, c);
      load8<VEC>(a.sin + pos * (R / 2) + 8 * p, sn);
    }
  }
  int64_t page = -1, off = 0;
  if (a.slots) {
    const int64_t slot = index_at(a.slots, a.slots_64, t);
    if (slot >= 0 && slot < (int64_t)a.pages * a.page_size) {
      page = P.page_div.div((uint32_t)slot);
      off = slot - page * a.page_size;
    }
  }
  const bool is_q = s < a.heads, is_v = s >= a.heads + a.kv_heads;
  const int h = is_q ? s : is_v ? s - a.heads - a.kv_heads : s - a.heads;
  if (!is_q && a.slots && page < 0) return;  // a token without a slot is not appended
  const TI* x = is_q ? reinterpret_cast<const TI*>(a.q) + t * a.q_token + h * a.q_head
                : is_v ? reinterpret_cast<const TI*>(a.v) + t * a.v_token + h * a.v_head
                       : reinterpret_cast<const TI*>(a.k) + t * a.k_token + h * a.k_head;
  float u[8], v[8];
  load8<VEC>(x + e0, u);
  load8<VEC>(x + e1, v);
  const float* w = is_q ? a.q_weight : is_v ? nullptr : a.k_weight;
  if (w) {
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss += u[i] * u[i] + v[i] * v[i];
    // lane p holds the sum of lanes [p, p + 2 o) of its group, lane 0 in the end all of it
    for (uint32_t o = 1; o < P.lpr; o <<= 1) {
      const float other = __shfl(ss, lane + o);
      if (p + o < P.lpr) ss += other;
    }
    ss = __shfl(ss, lane - p);
    const float scale = rsqrtf(fmaf(ss, P.inv_dim, a.eps));
    float wu[8], wv[8];
    load8<VEC>(w + e0, wu);
    load8<VEC>(w + e1, wv);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      u[i] = u[i] * scale * wu[i];
      v[i] = v[i] * scale * wv[i];
    }
  }
  if (rot && !is_v) {
    if (a.interleaved) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x0 = u[2 * i], y0 = u[2 * i + 1], x1 = v[2 * i], y1 = v[2 * i + 1];
        u[2 * i] = x0 * c[i] - y0 * sn[i];
        u[2 * i + 1] = x0 * sn[i] + y0 * c[i];
        v[2 * i] = x1 * c[4 + i] - y1 * sn[4 + i];
        v[2 * i + 1] = x1 * sn[4 + i] + y1 * c[4 + i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x0 = u[i], y0 = v[i];
        u[i] = x0 * c[i] - y0 * sn[i];
        v[i] = x0 * sn[i] + y0 * c[i];
      }
    }
  }
  if (is_q) {
    TI* o = reinterpret_cast<TI*>(a.q_out) + t * a.q_out_token + h * a.q_out_head;
    store8<VEC>(o + e0, u);
    store8<VEC>(o + e1, v);
  } else {
    TC* o = is_v ? reinterpret_cast<TC*>(a.v_out) + h * a.v_out_head : reinterpret_cast<TC*>(a.k_out) + h * a.k_out_head;
    const int64_t st = is_v ? a.v_out_token : a.k_out_token;
    o += a.slots ? page * (is_v ? a.v_out_page : a.k_out_page) + off * st : t * st;
    store8<VEC>(o + e0, u);
    store8<VEC>(o + e1, v);
  }
}

template <typename TI, typename TC>
static void head_rows_launch(const HeadRowsP& P, bool vec, hipStream_t s) {
  const dim3 grid((P.n_rows + 4 * P.wave_rows - 1) / (4 * P.wave_rows));
  launch(vec ? k_head_rows<TI, TC, true> : k_head_rows<TI, TC, false>, grid, dim3(256), 0, s, P);
}

static bool rows_aligned(const void* p, int64_t st, int64_t sh, int type) {
  const int64_t m = 16 / type_bytes(type);
  return !p || (aligned16(p) && st % m == 0 && sh % m == 0);
}

void head_rows(const fa_head_rows_args* ap, bool cache, hipStream_t s) {
  FA_REQUIRE(ap, "head rows: no arguments");
  HeadRowsP P;
  P.a = *ap;
  fa_head_rows_args& a = P.a;
  FA_REQUIRE(a.tokens >= 0 && a.heads >= 0 && a.kv_heads >= 0, "head rows: negative size");
  FA_REQUIRE(a.head_dim >= 16 && a.head_dim <= 512 && a.head_dim % 16 == 0,
             "head rows: head_dim must be a multiple of 16 up to 512");
  FA_REQUIRE(a.type == FA_F32 || a.type == FA_F16 || a.type == FA_BF16, "head rows: type");
  if (!a.cos != !a.sin) FA_REQUIRE(false, "head rows: cos and sin come together");
  if (a.cos) {
    FA_REQUIRE(a.rot_dim >= 16 && a.rot_dim <= a.head_dim && a.rot_dim % 16 == 0,
               "head rows: rot_dim must be a multiple of 16 up to head_dim");
    FA_REQUIRE(a.table_len >= 1, "head rows: empty angle table");
    FA_REQUIRE(a.positions || a.tokens == 0, "head rows: the rotation needs positions");
  } else {
    a.rot_dim = 0;
  }
  FA_REQUIRE(a.eps >= 0.f, "head rows: eps");
  const int64_t n_slots = a.heads + (int64_t)a.kv_heads * (cache ? 2 : 1);
  const bool some = a.tokens > 0;
  if (cache) {
    FA_REQUIRE(a.cache_type == FA_F16 || a.cache_type == FA_BF16, "kv_append: the cache is float16 or bfloat16");
    FA_REQUIRE(a.kv_heads >= 1 && a.pages >= 0 && a.page_size >= 1, "kv_append: sizes");
    FA_REQUIRE((int64_t)a.pages * a.page_size < (1ll << 31), "kv_append: more than 2^31 slots");
    FA_REQUIRE(!some || (a.k && a.v && a.slots), "kv_append: k, v and slots");
    FA_REQUIRE(!some || a.pages == 0 || (a.k_out && a.v_out), "kv_append: caches");
    FA_REQUIRE(rows_aligned(a.k_out, a.k_out_token, a.k_out_head, a.cache_type) && a.k_out_page % 8 == 0 &&
                   rows_aligned(a.v_out, a.v_out_token, a.v_out_head, a.cache_type) && a.v_out_page % 8 == 0,
               "kv_append: cache rows must be 16-byte aligned");
    P.page_div = FastDiv::of((uint32_t)a.page_size);
  } else {
    a.cache_type = a.type;
    a.slots = nullptr;
    a.v = nullptr;
    FA_REQUIRE(!some || !a.kv_heads || (a.k && a.k_out), "qk_norm_rope: k and its output");
  }
  FA_REQUIRE(!some || !a.heads || (a.q && a.q_out), "head rows: q and its output");
  FA_REQUIRE(a.q != a.q_out || !a.q || (a.q_token == a.q_out_token && a.q_head == a.q_out_head),
             "head rows: q in place with other strides");
  FA_REQUIRE(cache || a.k != a.k_out || !a.k || (a.k_token == a.k_out_token && a.k_head == a.k_out_head),
             "head rows: k in place with other strides");
  FA_REQUIRE(std::max(a.tokens, 1) * n_slots < (1ll << 31), "head rows: more than 2^31 rows");  // (both below 2^33: no overflow)
  P.n_slots = (int)n_slots;
  if (!some || n_slots == 0) return;
  P.lpr = (uint32_t)a.head_dim / 16;
  P.lpr_div = FastDiv::of(P.lpr);
  P.wave_rows = 64 / P.lpr;
  P.n_rows = (uint32_t)a.tokens * P.n_slots;
  P.slots_div = FastDiv::of((uint32_t)P.n_slots);
  P.inv_dim = 1.0f / (float)a.head_dim;
  // 16-byte accesses where every row that the call touches is aligned; else element by element
  const bool vec = rows_aligned(a.q, a.q_token, a.q_head, a.type) && rows_aligned(a.q_out, a.q_out_token, a.q_out_head, a.type) &&
                   rows_aligned(a.k, a.k_token, a.k_head, a.type) && rows_aligned(a.k_out, a.k_out_token, a.k_out_head, a.cache_type) &&
                   (!cache || rows_aligned(a.v, a.v_token, a.v_head, a.type)) && aligned16(a.q_weight) &&
                   aligned16(a.k_weight) && aligned16(a.cos) && aligned16(a.sin);
  if (a.type == FA_F32) {
    if (a.cache_type == FA_F32) head_rows_launch<float, float>(P, vec, s);
    else if (a.cache_type == FA_F16) head_rows_launch<float, _Float16>(P, vec, s);
    else head_rows_launch<float, __bf16>(P, vec, s);
  } else if (a.type == FA_F16) {
    if (a.cache_type == FA_F16) head_rows_launch<_Float16, _Float16>(P, vec, s);
    else head_rows_launch<_Float16, __bf16>(P, vec, s);
  } else {
    if (a.cache_type == FA_BF16) head_rows_launch<__bf16, __bf16>(P, vec, s);
    else head_rows_launch<__bf16, _Float16>(P, vec, s);
  }
}

// The accepted drafts of one sequence close up behind its committed tokens. A thread holds the same 16 bytes of every row, in
// order, so a row is read before anything is written over it: row i is the source of an earlier step only (path[j] = i
// needs j <= i). At most 63 rows of 256 bytes a head; the launch is what it costs.
__global__ __launch_bounds__(64) void k_keep_path(KeepPath k) {
  _Float16* const p = k.p[blockIdx.y / k.per_ptr] + (int64_t)(blockIdx.y % k.per_ptr) * k.cache_stride + blockIdx.x * k.head_stride;
  for (int d = threadIdx.x * 8; d < k.head_dim; d += 64 * 8)
    for (int i = 1; i < k.n; ++i)
      if (k.path[i] != i)
        *reinterpret_cast<f16x8_t*>(p + (int64_t)i * k.head_dim + d) =
            *reinterpret_cast<const f16x8_t*>(p + (int64_t)k.path[i] * k.head_dim + d);
}

void keep_path(const KeepPath& k, int heads, hipStream_t s) {
  FA_REQUIRE(k.n >= 1 && k.n <= KeepPath::MAX && k.head_dim % 8 == 0 && k.per_ptr >= 1, "keep_path: sizes");
  for (int i = 1; i < k.n; ++i) FA_REQUIRE(k.path[i] > k.path[i - 1] && k.path[i] < KeepPath::MAX, "keep_path: path");
  launch(k_keep_path, dim3(heads, 2 * k.per_ptr), dim3(64), 0, s, k);
}

}  // namespace fa

extern "C" {

int fa_qk_norm_rope(const fa_head_rows_args* a, void* stream) {
  FA_API_BEGIN
  fa::head_rows(a, false, reinterpret_cast<hipStream_t>(stream));
  FA_API_END
}

int fa_kv_append(const fa_head_rows_args* a, void* stream) {
  FA_API_BEGIN
  fa::head_rows(a, true, reinterpret_cast<hipStream_t>(stream));
  FA_API_END
}

}  // extern "C"

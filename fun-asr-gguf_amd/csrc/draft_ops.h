// Shared by the drafted-token operators (head_rows.hip, tree_attn.hip, sample_rows.hip): element types of device tensors,
// 8-element loads and stores, division by a run-time constant, and the launch that reports its own error.
#pragma once
#include "common.h"
#include "funasr_hip.h"

namespace fa {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));  // (float4 is a struct: four loads, which hipcc need not join again)
template <typename T> struct Vec8;
template <> struct Vec8<_Float16> { typedef f16x8_t type; };
template <> struct Vec8<__bf16> { typedef bf16x8_t type; };

// eight consecutive elements as floats; VEC: the address is 16-byte aligned
template <bool VEC, typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)p[i];
  } else if constexpr (sizeof(T) == 4) {
    const f32x4_t a = *reinterpret_cast<const f32x4_t*>(p), b = *reinterpret_cast<const f32x4_t*>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = a[i];
      x[4 + i] = b[i];
    }
  } else {
    const auto v = *reinterpret_cast<const typename Vec8<T>::type*>(p);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)v[i];
  }
}
template <bool VEC, typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  if constexpr (!VEC) {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = (T)x[i];
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    typename Vec8<T>::type v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (T)x[i];
    *reinterpret_cast<typename Vec8<T>::type*>(p) = v;
  }
}

// x / d for 0 <= x < 2^31 and a divisor 1 <= d < 2^31 that only the host knows beforehand: with s = ceil(log2 d) and
// m = floor(2^32 (2^s - d) / d) + 1 < 2^32, (2^32 + m) x / 2^(32 + s) exceeds x / d by less than x / 2^(32 + s) < 1 / d, so
// the floors agree; the high half of m x plus x stays below 2^32.
struct FastDiv {
  uint32_t mul = 1, shift = 0;
  static FastDiv of(uint32_t d) {
    FastDiv f;
    while ((1ull << f.shift) < d) ++f.shift;
    f.mul = (uint32_t)((1ull << 32) * ((1ull << f.shift) - d) / d + 1);
    return f;
  }
  __host__ __device__ __forceinline__ uint32_t div(uint32_t x) const {
    return ((uint32_t)(((uint64_t)x * mul) >> 32) + x) >> shift;
  }
};

inline int type_bytes(int t) { return t == FA_F32 ? 4 : 2; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// kernel(arg) on the stream. hipLaunchKernel returns its own status: an error that an earlier call left behind is not
// taken for this launch's.
template <typename P>
inline void launch(void (*kernel)(P), dim3 grid, dim3 block, size_t lds, hipStream_t s, P arg) {
  void* args[] = {&arg};
  FA_HIP(hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, args, lds, s));
}

// compute units of the current device (an attribute query: no allocation, no synchronisation, legal during capture). It shapes
// a launch only: without a device the MI355X's number, and the launch reports what is wrong
inline int cu_count() {
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) {
    (void)hipGetLastError();
    return 256;
  }
  return n;
}

// The operators themselves (the C entries fa_qk_norm_rope .. fa_sample_tokens without their error frame), for the engine's
// own steps.
void head_rows(const fa_head_rows_args* a, bool cache, hipStream_t s);  // cache: fa_kv_append, else fa_qk_norm_rope
int64_t tree_attention_bytes(const fa_tree_attention_args* a);
void tree_attention(const fa_tree_attention_args* a, hipStream_t s);
int64_t sample_tokens_bytes(const fa_sample_args* a);
void sample_tokens(const fa_sample_args* a, hipStream_t s);
// rows base + path[i] of every head move to base + i (i = 1 .. n - 1; path rises, path[i] >= i) in `caches` caches of `heads`
// heads each: cache c, head h at p[c / per_ptr] + (c % per_ptr) * cache_stride + h * head_stride
struct KeepPath {
  static constexpr int MAX = 64;
  _Float16* p[2];
  int64_t cache_stride, head_stride;
  int per_ptr, head_dim, n;
  int16_t path[MAX];
};
void keep_path(const KeepPath& k, int heads, hipStream_t s);

}  // namespace fa

// 16-byte accesses to rows of any width and alignment (norm.hip, attn.hip).  Internal to libgnnea.
#pragma once
#include "common.h"

namespace gnnea {

// elements of one 16-B access
template <typename T> struct RowChunk;
template <> struct RowChunk<float> { static constexpr int V = 4; };
template <> struct RowChunk<bf16_t> { static constexpr int V = 8; };

// 16 bytes at the alignment of one element: global memory takes them at any address, so a row of
// an odd width costs no narrower accesses
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <typename T> struct Raw16;
template <> struct Raw16<float> { typedef u32x4 type __attribute__((aligned(4))); };
template <> struct Raw16<bf16_t> { typedef u32x4 type __attribute__((aligned(2))); };

template <typename T>
__device__ __forceinline__ uint4 load16(const T* p) {
  const u32x4 r = *(const typename Raw16<T>::type*)p;
  return make_uint4(r.x, r.y, r.z, r.w);
}

// `left` elements (at most V) from p, zeros after them
template <typename T, int V>
__device__ __forceinline__ void load_chunk(const T* p, int left, float (&f)[V]) {
  if (left >= V) {
    unpack16(load16<T>(p), f);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = k < left ? to_f32<T>(p[k]) : 0.f;
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_chunk(T* p, int left, const float (&f)[V]) {
  if (left >= V) {
    u32x4 r;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (V == 4) r[k] = __builtin_bit_cast(uint32_t, f[k]);
      else r[k] = x3_cvt2(x3_f32x2{f[2 * k], f[2 * k + 1]});
    }
    *(typename Raw16<T>::type*)p = r;
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (k < left) p[k] = from_f32<T>(f[k]);
  }
}

}  // namespace gnnea

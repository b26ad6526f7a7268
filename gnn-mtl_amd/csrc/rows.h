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
template <typename T> struct __attribute__((packed, aligned(sizeof(T)))) Raw16 { uint32_t w[4]; };

template <typename T>
__device__ __forceinline__ uint4 load16(const T* p) {
  const Raw16<T> r = *(const Raw16<T>*)p;
  return make_uint4(r.w[0], r.w[1], r.w[2], r.w[3]);
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
    Raw16<T> r;
    if constexpr (V == 4) {
#pragma unroll
      for (int k = 0; k < 4; ++k) r.w[k] = __builtin_bit_cast(uint32_t, f[k]);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k)
        r.w[k] = (uint32_t)f32_to_bf16(f[2 * k]) | ((uint32_t)f32_to_bf16(f[2 * k + 1]) << 16);
    }
    *(Raw16<T>*)p = r;
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (k < left) p[k] = from_f32<T>(f[k]);
  }
}

}  // namespace gnnea

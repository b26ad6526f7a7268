// AdamW over many tensors in few launches (run/train_ea.py:64 steps torch's Adam): the gradients'
// global norm, one small launch that takes the step's scalars, and the update, each over all
// tensors of a list.  Moments in fp32, or in 8 bits with one exponent per 256 elements.
//
// Bytes per element: fp32 p, m, v read and written and g read, 28; with 8-bit moments 12 + 4 = 16
// (+ 2/256 of scales); the norm reads g once more.  With 32-bit moments that is what bounds it: 300M
// elements take 1.39 ms (6.0 TB/s; a plain copy of 4 GiB reaches 4.7 here).  With 8 bits the update
// also issues 81 vector instructions per element and lane (the hash, three fp64 operations, codes from
// and to bytes), 0.62 ms of 300M elements' 0.82 to 0.90 (by machine; 5.3 to 5.9 TB/s), and most of
// 8.4M bf16 elements' 29 us, whose 84 MB stay in the cache.  Reading out what the codes stand for
// takes 0.36 ms (1.8 GB).  A list of 12 tensors (0.54M elements, clipped) is three launches of 7, 4
// and 6 us.
//
// 8-bit moments.  m is e4m3 times a power of two per block (dequantising, scaling and finding the
// largest value are exact, so a code depends on nothing but the value).  The second moment is
// kept as its root u = sqrt(v): 4 exponent and 4 fraction bits, no sign, times a power of two per
// block, so v spans 2^30 within a block.  Rounding u to nearest would freeze it: with b2 = 0.999 a
// step changes u by at most 0.05 % downwards, half a code is 3 %; so u goes up or down with the
// odds of its place between two codes (mean kept), by a hash of (seed, step, tensor, element), the
// same on every run.  A u that is not 0 never becomes 0 (its update would divide by eps).
// b1 m + (1 - b1) g is formed in fp64 and rounded to fp32 once: 0.9 m + 0.1 g of a code and a bf16
// gradient often lies exactly between two codes, and fp32 products would decide it by their error.
#include "common.h"

namespace gnnea {

constexpr int kAdamTensors = 48;   // descriptors in one launch's arguments (2.7 KB)
constexpr int kAdamChunk = 4096;   // elements of one workgroup: 4 blocks of 256 per wave
constexpr int kNormChunkElems = 16384;

struct AdamList {
  gnnea_adamw_tensor t[kAdamTensors];
  int32_t first[kAdamTensors + 1];  // workgroup at which tensor k begins
  int32_t count;
};

struct AdamCtl { float coef, bc1, bc2, lr, norm; uint32_t key, skip, pad; };
static_assert(sizeof(AdamCtl) == GNNEA_ADAMW_CTL_BYTES, "ctl");

// the 32-bit finaliser of MurmurHash3 (A. Appleby), a bijection whose every input bit reaches every
// output bit
__device__ __forceinline__ uint32_t mix32(uint32_t h) {
  h = (h ^ (h >> 16)) * 0x85ebca6bu;
  h = (h ^ (h >> 13)) * 0xc2b2ae35u;
  return h ^ (h >> 16);
}

// the tensor of workgroup b (uniform: scalar loads of the kernel's arguments)
__device__ __forceinline__ int adam_find(const AdamList& L, int b) {
  int lo = 0, hi = L.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (L.first[mid] <= b) lo = mid; else hi = mid - 1;
  }
  return lo;
}

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
template <typename T> struct Four;
template <> struct Four<float> { typedef u32x4 type __attribute__((aligned(4))); };
template <> struct Four<bf16_t> { typedef u32x2 type __attribute__((aligned(2))); };
typedef uint32_t u32_any __attribute__((aligned(1)));

// four values at an element's alignment; NT: past the caches
template <typename T, bool NT = false>
__device__ __forceinline__ void load4(const T* p, int64_t left, float (&f)[4]) {
  if (left >= 4) {
    typedef typename Four<T>::type F;
    F r;
    if constexpr (NT) r = __builtin_nontemporal_load((const F*)p);
    else r = *(const F*)p;
    if constexpr (sizeof(T) == 4) {
      const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) f[k] = __builtin_bit_cast(float, w[k]);
    } else {
      const float4 v = Vec4<bf16_t>::get(make_uint2(r.x, r.y));
      f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k) f[k] = k < left ? to_f32<T>(p[k]) : 0.f;
  }
}
template <typename T, bool NT = false>
__device__ __forceinline__ void store4(T* p, int64_t left, const float (&f)[4]) {
  if (left >= 4) {
    typedef typename Four<T>::type F;
    F* q = (F*)p;
    if constexpr (sizeof(T) == 4) {
      const u32x4 r = {__builtin_bit_cast(uint32_t, f[0]), __builtin_bit_cast(uint32_t, f[1]),
                       __builtin_bit_cast(uint32_t, f[2]), __builtin_bit_cast(uint32_t, f[3])};
      if constexpr (NT) __builtin_nontemporal_store(r, q);
      else *q = r;
    } else {
      const u32x2 r = {x3_cvt2(x3_f32x2{f[0], f[1]}), x3_cvt2(x3_f32x2{f[2], f[3]})};
      if constexpr (NT) __builtin_nontemporal_store(r, q);
      else *q = r;
    }
  } else {
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (k < left) p[k] = from_f32<T>(f[k]);
  }
}
template <bool NT = false>
__device__ __forceinline__ uint32_t load4b(const uint8_t* p, int64_t left) {
  if (left >= 4) {
    if constexpr (NT) return __builtin_nontemporal_load((const u32_any*)p);
    else return *(const u32_any*)p;
  }
  uint32_t r = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < left) r |= (uint32_t)p[k] << (8 * k);
  return r;
}
template <bool NT = false>
__device__ __forceinline__ void store4b(uint8_t* p, int64_t left, uint32_t c) {
  if (left >= 4) {
    if constexpr (NT) __builtin_nontemporal_store(c, (u32_any*)p);
    else *(u32_any*)p = c;
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (k < left) p[k] = (uint8_t)(c >> (8 * k));
}

__device__ __forceinline__ float pow2(int e) {  // 2^(e - 127), 1 <= e <= 254
  return __builtin_bit_cast(float, (uint32_t)e << 23);
}

// e4m3 codes (four in a word) times 2^(e - 127)
__device__ __forceinline__ void m_decode(uint32_t c, int e, float (&f)[4]) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false);
  const f2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  const float s = pow2(e);
  f[0] = lo.x * s; f[1] = lo.y * s; f[2] = hi.x * s; f[3] = hi.y * s;
}
__device__ __forceinline__ void u_decode(uint32_t c, int e, float (&f)[4]) {
  const float s = pow2(e);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t b = (c >> (8 * k)) & 255u;
    f[k] = b ? __builtin_bit_cast(float, (b << 19) + (112u << 23)) * s : 0.f;
  }
}

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xf, 0xf, false));
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x140, 0xf, 0xf, false));
  const uint32_t a = max((uint32_t)readlane_i((int)v, 0), (uint32_t)readlane_i((int)v, 16));
  const uint32_t b = max((uint32_t)readlane_i((int)v, 32), (uint32_t)readlane_i((int)v, 48));
  return max(a, b);
}

struct AdamHyper {
  double b1, c1;       // beta1, 1 - beta1
  float b1f, c1f, b2, c2, eps, wd;
};

// One wave per block of 256 elements, four elements per lane; a wave's four blocks are loaded
// before any of them is computed.
template <typename T, int BITS, bool NT>
__global__ __launch_bounds__(256) void k_adamw(const AdamList L, const AdamHyper h,
                                               const AdamCtl* __restrict__ ctl) {
#pragma clang fp contract(off)
  const AdamCtl s = *ctl;
  if (s.skip) return;
  const int ti = adam_find(L, blockIdx.x);
  const gnnea_adamw_tensor t = L.t[ti];
  const int64_t base = (int64_t)(blockIdx.x - L.first[ti]) * kAdamChunk + wave_id() * 1024;
  const int lane = lane_id();
  const float decay = 1.f - s.lr * h.wd, lr1 = s.lr * s.bc1;
  constexpr int U = 4;
  float p[U][4], g[U][4], m[U][4], v[U][4];
  uint32_t mc[U], uc[U];
  int me[U], ue[U];
  const int64_t nb = (t.n + GNNEA_ADAMW_BLOCK - 1) / GNNEA_ADAMW_BLOCK;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t b0 = base + u * 256, at = b0 + lane * 4, left = t.n - at;
    if (b0 >= t.n) break;
    load4<T, NT>((const T*)t.p + at, left, p[u]);
    load4<T, NT>((const T*)t.g + at, left, g[u]);
    if constexpr (BITS == 32) {
      load4<float, NT>((const float*)t.m + at, left, m[u]);
      load4<float, NT>((const float*)t.v + at, left, v[u]);
    } else {
      mc[u] = load4b<NT>((const uint8_t*)t.m + at, left);
      uc[u] = load4b<NT>((const uint8_t*)t.v + at, left);
      me[u] = t.scales[b0 >> 8];
      ue[u] = t.scales[nb + (b0 >> 8)];
    }
  }
  const uint32_t key0 = mix32(s.key + 0x85ebca6bu * (uint32_t)t.index);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t b0 = base + u * 256, at = b0 + lane * 4, left = t.n - at;
    if (b0 >= t.n) break;
    float root[4];
    if constexpr (BITS == 32) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float gk = g[u][k] * s.coef;
        m[u][k] = m[u][k] * h.b1f + gk * h.c1f;
        v[u][k] = v[u][k] * h.b2 + gk * gk * h.c2;
        root[k] = sqrtf(v[u][k]);
      }
      store4<float, NT>((float*)t.m + at, left, m[u]);
      store4<float, NT>((float*)t.v + at, left, v[u]);
    } else {
      m_decode(mc[u], me[u], m[u]);
      u_decode(uc[u], ue[u], root);
      uint32_t mt = 0, ut = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float gk = g[u][k] * s.coef;
        m[u][k] = (float)((double)m[u][k] * h.b1 + (double)gk * h.c1);
        root[k] = sqrtf(root[k] * root[k] * h.b2 + gk * gk * h.c2);
        mt = max(mt, __builtin_bit_cast(uint32_t, m[u][k]) & 0x7fffffffu);
        ut = max(ut, __builtin_bit_cast(uint32_t, root[k]) & 0x7fffffffu);
      }
      mt = wave_max_u32(mt);
      ut = wave_max_u32(ut);
      // An element whose moments are not finite is lost, as it is with 32 bits: NaN from here on
      // (e4m3's code for it).  The block's exponents go by the others, which keep what they have.
      uint32_t lost = 0;
      if (max(mt, ut) >= 0x7f800000u) {
        mt = ut = 0;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t a = __builtin_bit_cast(uint32_t, m[u][k]) & 0x7fffffffu;
          const uint32_t b = __builtin_bit_cast(uint32_t, root[k]) & 0x7fffffffu;
          if (max(a, b) >= 0x7f800000u) {
            lost |= 0x7fu << (8 * k);
            m[u][k] = __builtin_nanf("");
          } else {
            mt = max(mt, a);
            ut = max(ut, b);
          }
        }
        mt = wave_max_u32(mt);
        ut = wave_max_u32(ut);
      }
      // the smallest exponents under which all of m are below 448 = 1.75 2^8, and all of u below
      // (1 + 15/16), so that neither rounds past its largest code (e <= 247, f <= 192: a root of a
      // finite v is below 2^64)
      const int e = max(1, (int)((mt + (1u << 21)) >> 23) - 8);
      const int f = max(17, (int)((ut + (1u << 19)) >> 23));
      const float ms = pow2(254 - e), us = pow2(254 - f);
      int w = __builtin_amdgcn_cvt_pk_fp8_f32(m[u][0] * ms, m[u][1] * ms, 0, false);
      w = __builtin_amdgcn_cvt_pk_fp8_f32(m[u][2] * ms, m[u][3] * ms, w, true);
      uint32_t c = 0;
      const uint32_t key = key0 + (uint32_t)(at >> 32) * 0x9e3779b9u;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t chance = mix32((uint32_t)at + k + key) >> 13;
        const int q = (int)(__builtin_bit_cast(uint32_t, root[k] * us) - (112u << 23) + chance) >> 19;
        c |= (root[k] == 0.f ? 0u : (uint32_t)min(255, max(1, q))) << (8 * k);
      }
      store4b<NT>((uint8_t*)t.m + at, left, (uint32_t)w | lost);
      store4b<NT>((uint8_t*)t.v + at, left, c);
      if (lane == 0) {
        t.scales[b0 >> 8] = (uint8_t)e;
        t.scales[nb + (b0 >> 8)] = (uint8_t)f;
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      p[u][k] = p[u][k] * decay - lr1 * m[u][k] * __builtin_amdgcn_rcpf(root[k] * s.bc2 + h.eps);
    store4<T, NT>((T*)t.p + at, left, p[u]);
  }
}

// Sums of squares of 16384 gradients per workgroup, in fp64 (the factor of a clipped gradient
// then has the same bits whatever the split).
template <typename T>
__global__ __launch_bounds__(256) void k_adamw_norm(const AdamList L, double* __restrict__ parts) {
  __shared__ double sh[4];
  const int ti = adam_find(L, blockIdx.x);
  const gnnea_adamw_tensor t = L.t[ti];
  const int64_t base = (int64_t)(blockIdx.x - L.first[ti]) * kNormChunkElems;
  double acc = 0.0;
  for (int r = 0; r < kNormChunkElems / 4096; ++r) {
    float g[4][4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t at = base + r * 4096 + u * 1024 + threadIdx.x * 4;
      load4<T>((const T*)t.g + at, t.n - at, g[u]);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int k = 0; k < 4; ++k) acc = __builtin_fma((double)g[u][k], (double)g[u][k], acc);
  }
  acc = wave_sum_f64(acc);
  if (lane_id() == 0) sh[wave_id()] = acc;
  __syncthreads();
  if (threadIdx.x == 0) parts[blockIdx.x] = ((sh[0] + sh[1]) + sh[2]) + sh[3];
}

__global__ __launch_bounds__(1024) void k_adamw_begin(const double* __restrict__ parts,
                                                      int64_t n_parts, double max_norm, double b1,
                                                      double b2, double lr,
                                                      const float* __restrict__ lr_dev,
                                                      uint32_t seed, int64_t* __restrict__ step,
                                                      AdamCtl* __restrict__ ctl) {
  __shared__ double sh[16];
  double s = 0.0;
  for (int64_t k = threadIdx.x; k < n_parts; k += 1024) s += parts[k];
  s = wave_sum_f64(s);
  if (lane_id() == 0) sh[wave_id()] = s;
  __syncthreads();
  if (threadIdx.x != 0) return;
  AdamCtl c;
  c.coef = 1.f;
  c.skip = c.pad = 0;
  c.norm = 0.f;
  if (n_parts > 0) {
    s = sh[0];
    for (int w = 1; w < 16; ++w) s += sh[w];
    const double norm = sqrt(s);
    c.norm = (float)norm;
    if (max_norm > 0.0) {
      const double f = max_norm / (norm + 1e-6);
      c.coef = (float)(f < 1.0 ? f : 1.0);
      c.skip = !(norm <= 1.7976931348623157e308);
    }
  }
  const int64_t t = *step + 1;
  if (!c.skip) *step = t;
  c.bc1 = (float)(1.0 / (1.0 - pow(b1, (double)t)));
  c.bc2 = (float)(1.0 / sqrt(1.0 - pow(b2, (double)t)));
  c.lr = lr_dev ? *lr_dev : (float)lr;
  c.key = seed + 0x9e3779b9u * (uint32_t)t;
  *ctl = c;
}

__global__ __launch_bounds__(256) void k_adamw_moments(const AdamList L) {
  const int ti = adam_find(L, blockIdx.x);
  const gnnea_adamw_tensor t = L.t[ti];
  const int64_t base = (int64_t)(blockIdx.x - L.first[ti]) * kAdamChunk + wave_id() * 1024;
  const int64_t nb = (t.n + GNNEA_ADAMW_BLOCK - 1) / GNNEA_ADAMW_BLOCK;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t b0 = base + u * 256, at = b0 + lane_id() * 4, left = t.n - at;
    if (b0 >= t.n) break;
    float f[4];
    m_decode(load4b((const uint8_t*)t.m + at, left), t.scales[b0 >> 8], f);
    store4<bf16_t>((bf16_t*)t.p + at, left, f);
    u_decode(load4b((const uint8_t*)t.v + at, left), t.scales[nb + (b0 >> 8)], f);
    store4<bf16_t>((bf16_t*)const_cast<void*>(t.g) + at, left, f);
  }
}

// Lists that move more than the Infinity Cache holds are read and written past the caches: nothing
// of them is there at the next step.  300M fp32 elements: 1552 -> 1393 us (6.0 TB/s) with 32-bit
// moments, 906 -> 807 with 8 (one machine); 8.6M bf16 elements (84 MB), which stay in the cache: 30 against 33 us.
constexpr int64_t kCacheBytes = 256 << 20;

template <typename T, int BITS, bool NT>
static void adam_launch(const AdamList& L, const AdamHyper& h, const AdamCtl* c, hipStream_t s) {
  hipLaunchKernelGGL((k_adamw<T, BITS, NT>), dim3(L.first[L.count]), dim3(256), 0, s, L, h, c);
}

static int adam_check(const gnnea_adamw_tensor* t, int32_t count, bool state, bool codes) {
  if (count < 0 || (count && !t)) return GNNEA_EINVAL;
  for (int32_t k = 0; k < count; ++k) {
    if (t[k].n < 0) return GNNEA_EINVAL;
    if (t[k].n == 0) continue;
    if (!t[k].g || (state && (!t[k].p || !t[k].m || !t[k].v))) return GNNEA_EINVAL;
    if (codes && !t[k].scales) return GNNEA_EINVAL;
    if (t[k].n > (int64_t)kAdamChunk * 0x7fff0000ll) return GNNEA_EINVAL;
  }
  return GNNEA_OK;
}

// The tensors from `from` on that fit one launch (empty ones left out); returns where it stopped.
static int32_t adam_list(const gnnea_adamw_tensor* t, int32_t count, int32_t from, int chunk,
                         AdamList* L) {
  L->count = 0;
  L->first[0] = 0;
  for (; from < count && L->count < kAdamTensors; ++from) {
    if (t[from].n == 0) continue;
    const int64_t wg = (t[from].n + chunk - 1) / chunk;
    if (L->first[L->count] + wg > 0x7fffffffll) break;
    L->t[L->count] = t[from];
    L->first[L->count + 1] = L->first[L->count] + (int32_t)wg;
    ++L->count;
  }
  return from;
}

}  // namespace gnnea

using namespace gnnea;

extern "C" int64_t gnnea_adamw_norm_parts(const gnnea_adamw_tensor* t, int32_t count) {
  if (count < 0 || (count && !t)) return GNNEA_EINVAL;
  int64_t n = 0;
  for (int32_t k = 0; k < count; ++k) {
    if (t[k].n < 0) return GNNEA_EINVAL;
    n += (t[k].n + kNormChunkElems - 1) / kNormChunkElems;
  }
  return n;
}

extern "C" int gnnea_adamw_norm(const gnnea_adamw_tensor* t, int32_t count, int dtype,
                                double* parts, int64_t n_parts, void* stream) {
  const int rc = adam_check(t, count, false, false);
  if (rc) return rc;
  if (dtype != GNNEA_F32 && dtype != GNNEA_BF16) return GNNEA_EINVAL;
  if (n_parts < gnnea_adamw_norm_parts(t, count)) return GNNEA_EWORKSPACE;
  AdamList L;
  for (int32_t at = 0; at < count;) {
    at = adam_list(t, count, at, kNormChunkElems, &L);
    const int wg = L.first[L.count];
    if (!wg) continue;
    if (!parts) return GNNEA_EINVAL;
    if (dtype == GNNEA_F32)
      hipLaunchKernelGGL(k_adamw_norm<float>, dim3(wg), dim3(256), 0, (hipStream_t)stream, L, parts);
    else
      hipLaunchKernelGGL(k_adamw_norm<bf16_t>, dim3(wg), dim3(256), 0, (hipStream_t)stream, L, parts);
    GNNEA_LAUNCH_CHECK();
    parts += wg;
  }
  return 0;
}

extern "C" int gnnea_adamw_begin(const double* parts, int64_t n_parts, double max_norm,
                                 double beta1, double beta2, double lr, const float* lr_dev,
                                 uint32_t seed, int64_t* step, void* ctl, void* stream) {
  if (n_parts < 0 || (n_parts && !parts) || !step || !ctl) return GNNEA_EINVAL;
  if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0)) return GNNEA_EINVAL;
  if (((uintptr_t)ctl & 7) || ((uintptr_t)step & 7)) return GNNEA_EALIGN;
  hipLaunchKernelGGL(k_adamw_begin, dim3(1), dim3(1024), 0, (hipStream_t)stream, parts, n_parts,
                     max_norm, beta1, beta2, lr, lr_dev, seed, step, (AdamCtl*)ctl);
  GNNEA_LAUNCH_CHECK();
  return 0;
}

extern "C" int gnnea_adamw_step(const gnnea_adamw_tensor* t, int32_t count, int dtype,
                                int state_bits, double beta1, double beta2, double eps,
                                double weight_decay, const void* ctl, void* stream) {
  if (state_bits != 8 && state_bits != 32) return GNNEA_EINVAL;
  if (dtype != GNNEA_F32 && dtype != GNNEA_BF16) return GNNEA_EINVAL;
  const int rc = adam_check(t, count, true, state_bits == 8);
  if (rc) return rc;
  if (!ctl || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0)) return GNNEA_EINVAL;
  if ((uintptr_t)ctl & 7) return GNNEA_EALIGN;
  AdamHyper h;
  h.b1 = beta1; h.c1 = 1.0 - beta1;
  h.b1f = (float)beta1; h.c1f = (float)(1.0 - beta1);
  h.b2 = (float)beta2; h.c2 = (float)(1.0 - beta2);
  h.eps = (float)eps; h.wd = (float)weight_decay;
  AdamList L;
  hipStream_t s = (hipStream_t)stream;
  for (int32_t at = 0; at < count;) {
    at = adam_list(t, count, at, kAdamChunk, &L);
    if (!L.first[L.count]) continue;
    const AdamCtl* c = (const AdamCtl*)ctl;
    int64_t n = 0;
    for (int32_t k = 0; k < L.count; ++k) n += L.t[k].n;
    const int64_t each = 3 * (dtype == GNNEA_F32 ? 4 : 2) + (state_bits == 32 ? 16 : 4);
    const bool nt = n * each > kCacheBytes;
    const int f32 = dtype == GNNEA_F32;
    if (state_bits == 32) {
      if (f32) nt ? adam_launch<float, 32, true>(L, h, c, s) : adam_launch<float, 32, false>(L, h, c, s);
      else nt ? adam_launch<bf16_t, 32, true>(L, h, c, s) : adam_launch<bf16_t, 32, false>(L, h, c, s);
    } else {
      if (f32) nt ? adam_launch<float, 8, true>(L, h, c, s) : adam_launch<float, 8, false>(L, h, c, s);
      else nt ? adam_launch<bf16_t, 8, true>(L, h, c, s) : adam_launch<bf16_t, 8, false>(L, h, c, s);
    }
    GNNEA_LAUNCH_CHECK();
  }
  return 0;
}

extern "C" int gnnea_adamw_moments(const gnnea_adamw_tensor* t, int32_t count, void* stream) {
  const int rc = adam_check(t, count, true, true);
  if (rc) return rc;
  AdamList L;
  for (int32_t at = 0; at < count;) {
    at = adam_list(t, count, at, kAdamChunk, &L);
    const int wg = L.first[L.count];
    if (!wg) continue;
    hipLaunchKernelGGL(k_adamw_moments, dim3(wg), dim3(256), 0, (hipStream_t)stream, L);
    GNNEA_LAUNCH_CHECK();
  }
  return 0;
}

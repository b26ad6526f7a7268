// The norms before and after a block, with the block's gate and residual scale, in one pass each
// way.  A residual stack of layers f (GraphConvolution, GAT, attention: the reference stacks them
// without either, models/encoders.py:24-86) computes, per row of D features,
//
//   r = x + s * g * N(y),  g = sigmoid(z),        y = f(h of the layer before)
//   h = N'(r)                                     the next layer's input
//
// with N(y) = n w + b, n = (y - mean) / sqrt(var + eps) (GNNEA_NORM_LAYER) or n = y / sqrt(mean
// y^2 + eps) (GNNEA_NORM_RMS).  Backward, from dr and dh (the row's D values live in registers):
//
//   n', n from the saved statistics;  m = dh w'
//   dx = dr + rho' (m - [mean m] - n' mean(m n'))            [..]: LayerNorm only
//   q  = dx s g w,   dy = rho (q - [mean q] - n mean(q n)),   dz = dx s (n w + b) g (1 - g)
//
// and the column sums A = sum dx g n, B = sum dx g, C = sum dh n', E = sum dh, from which all six
// vector gradients follow: dw = s A, db = s B, ds = w A + b B, dw' = C, db' = E, and for one gate
// vector shared by all rows dz = s (1 - g)(w A + b B).  Two to four sums instead of six.
//
// Every element is read once and written once: forward x, y[, z] in, r, h out; backward x, y[, z],
// dr, dh in, dx, dy[, dz] out.  The kernels are bound by HBM.  The backward recomputes r in fp32
// from x and y instead of reading the stored r: the same bytes, and bf16 storage loses nothing.
//
// A row is held by TPR threads (16 lanes, a wave, or a workgroup of 256 or 512), NIT chunks of
// 16 B per thread; rows of odd widths use the same 16-B accesses at the element's alignment.
// Statistics, sums and gradients are fp32; the column sums go per thread over its rows, then over
// the workgroup's rows, then over workgroups (fp64) in a fixed order: results do not change from
// run to run.
#include "rows.h"

namespace gnnea {

constexpr int kNormMaxD = 8192;
constexpr int kNormSums = 4;

// g = sigmoid(z) and 1 - g, each from exp(-|z|): 1 - g keeps its digits where g is close to 1
struct Gate { float g, rest; };
__device__ __forceinline__ Gate gate_of(float z) {
  const float e = __expf(-fabsf(z)), r = __builtin_amdgcn_rcpf(1.f + e);
  return z >= 0.f ? Gate{r, e * r} : Gate{e * r, r};
}

// V weights of either type from column c on (fp32 weights beside bf16 features: two 16-B loads)
template <typename TW, int V>
__device__ __forceinline__ void load_vec(const TW* p, int left, float (&f)[V], float none) {
  if (!p) {
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = none;
    return;
  }
  if constexpr (RowChunk<TW>::V == V) {
    load_chunk<TW, V>(p, left, f);
  } else if (left >= V) {
    const uint4 a = load16<TW>(p), b = load16<TW>(p + 4);
    const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = __builtin_bit_cast(float, w[k]);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = k < left ? to_f32<TW>(p[k]) : 0.f;
  }
}

// Sums of NS values over the TPR threads of a row; every thread gets them, from the same order of
// additions.  16 lanes and a wave stay in registers; a workgroup goes once through LDS (two
// buffers in turn, so one barrier per sum is enough).
template <int TPR, int NS>
__device__ __forceinline__ void row_sum(float (&v)[NS], float (*sh)[8][NS], int& turn) {
#pragma unroll
  for (int k = 0; k < NS; ++k) {
    v[k] += mov_dpp_f32<0xB1>(v[k]);
    v[k] += mov_dpp_f32<0x4E>(v[k]);
    v[k] += mov_dpp_f32<0x141>(v[k]);
    v[k] += mov_dpp_f32<0x140>(v[k]);
    if constexpr (TPR >= 64)
      v[k] = ((readlane_f(v[k], 0) + readlane_f(v[k], 16)) + readlane_f(v[k], 32)) +
             readlane_f(v[k], 48);
  }
  if constexpr (TPR > 64) {
    float(*b)[NS] = sh[turn];
    turn ^= 1;
    if (lane_id() == 0) {
#pragma unroll
      for (int k = 0; k < NS; ++k) b[wave_id()][k] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NS; ++k) {
      float s = b[0][k];
#pragma unroll
      for (int w = 1; w < TPR / 64; ++w) s += b[w][k];
      v[k] = s;
    }
  }
}

// mean and 1 / sqrt(var + eps) (0 and 1 / rms) of the row's values f
template <int TPR, int NIT, int V>
__device__ __forceinline__ void row_stats(const float (&f)[NIT][V], int D, int c0, bool layer,
                                          float eps, float (*sh)[8][1], int& turn, float& mean,
                                          float& rho) {
  mean = 0.f;
  float s[1];
  if (layer) {
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < NIT; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) s[0] += f[i][k];  // places past the row hold 0
    row_sum<TPR, 1>(s, sh, turn);
    mean = s[0] / (float)D;
  }
  s[0] = 0.f;
#pragma unroll
  for (int i = 0; i < NIT; ++i)
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float d = c0 + i * TPR * V + k < D ? f[i][k] - mean : 0.f;
      s[0] = fmaf(d, d, s[0]);
    }
  row_sum<TPR, 1>(s, sh, turn);
  rho = 1.f / sqrtf(s[0] / (float)D + eps);
}

template <typename T, typename TW, int TPR, int NIT>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void k_norm_fwd(const gnnea_norm a) {
  constexpr int V = RowChunk<T>::V;
  constexpr int RPB = TPR < 256 ? 256 / TPR : 1;
  __shared__ float sh[2][8][1];
  int turn = 0;
  const int D = a.D, t = threadIdx.x % TPR, c0 = t * V;
  const bool layer = a.kind == GNNEA_NORM_LAYER;
  const T* __restrict__ X = (const T*)a.x;
  const T* __restrict__ Y = (const T*)a.y;
  const T* __restrict__ Z = (const T*)a.gate;
  const TW* __restrict__ W = (const TW*)a.post_w;
  const TW* __restrict__ Bv = (const TW*)a.post_b;
  const TW* __restrict__ S = (const TW*)a.scale;
  const TW* __restrict__ W2 = (const TW*)a.pre_w;
  const TW* __restrict__ B2 = (const TW*)a.pre_b;
  for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR; row < a.n;
       row += (int64_t)gridDim.x * RPB) {
    float r[NIT][V], y[NIT][V], z[NIT][V];
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      const int c = c0 + i * TPR * V;
      load_chunk<T, V>(X + row * a.ldx + c, D - c, r[i]);
      if (Y) load_chunk<T, V>(Y + row * a.ldy + c, D - c, y[i]);
      if (a.gate_mode == GNNEA_GATE_FULL)
        load_chunk<T, V>(Z + row * a.ldg + c, D - c, z[i]);
      else if (a.gate_mode == GNNEA_GATE_ROW)
        load_vec<TW, V>((const TW*)a.gate + c, D - c, z[i], 0.f);
    }
    float mean = 0.f, rho = 1.f, mean2 = 0.f, rho2 = 1.f;
    if (Y) {
      if (a.post) row_stats<TPR, NIT, V>(y, D, c0, layer, a.eps, sh, turn, mean, rho);
#pragma unroll
      for (int i = 0; i < NIT; ++i) {
        const int c = c0 + i * TPR * V;
        float w[V], b[V], s[V];
        load_vec<TW, V>(W ? W + c : W, D - c, w, 1.f);
        load_vec<TW, V>(Bv ? Bv + c : Bv, D - c, b, 0.f);
        load_vec<TW, V>(S ? S + c : S, D - c, s, 1.f);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float u = fmaf((y[i][k] - mean) * rho, w[k], b[k]);
          const float g = a.gate_mode ? gate_of(z[i][k]).g : 1.f;
          r[i][k] = c + k < D ? fmaf(a.alpha * s[k] * g, u, r[i][k]) : 0.f;
        }
        if (a.r) store_chunk<T, V>((T*)a.r + row * a.ldr + c, D - c, r[i]);
      }
    }
    if (a.pre) {
      row_stats<TPR, NIT, V>(r, D, c0, layer, a.eps, sh, turn, mean2, rho2);
#pragma unroll
      for (int i = 0; i < NIT; ++i) {
        const int c = c0 + i * TPR * V;
        float w[V], b[V];
        load_vec<TW, V>(W2 ? W2 + c : W2, D - c, w, 1.f);
        load_vec<TW, V>(B2 ? B2 + c : B2, D - c, b, 0.f);
#pragma unroll
        for (int k = 0; k < V; ++k) r[i][k] = fmaf((r[i][k] - mean2) * rho2, w[k], b[k]);
        store_chunk<T, V>((T*)a.h + row * a.ldh + c, D - c, r[i]);
      }
    }
    if (a.stats && t == 0)
      *(float4*)(a.stats + 4 * row) = make_float4(mean, rho, mean2, rho2);
  }
}

template <typename T, typename TW, int TPR, int NIT>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void k_norm_bwd(const gnnea_norm a) {
  constexpr int V = RowChunk<T>::V;
  constexpr int NT = TPR < 256 ? 256 : TPR;
  constexpr int RPB = NT / TPR;
  __shared__ float sh[2][8][2];
  __shared__ float fold[RPB > 1 ? NT * NIT * V : 1];
  int turn = 0;
  const int D = a.D, t = threadIdx.x % TPR, c0 = t * V;
  const bool layer = a.kind == GNNEA_NORM_LAYER;
  const float inv = 1.f / (float)D;
  const T* __restrict__ X = (const T*)a.x;
  const T* __restrict__ Y = (const T*)a.y;
  const T* __restrict__ Z = (const T*)a.gate;
  const T* __restrict__ DR = (const T*)a.dr;
  const T* __restrict__ DH = (const T*)a.dh;
  const TW* __restrict__ W = (const TW*)a.post_w;
  const TW* __restrict__ Bv = (const TW*)a.post_b;
  const TW* __restrict__ S = (const TW*)a.scale;
  const TW* __restrict__ W2 = (const TW*)a.pre_w;
  float acc[kNormSums][NIT][V];
#pragma unroll
  for (int q = 0; q < kNormSums; ++q)
#pragma unroll
    for (int i = 0; i < NIT; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) acc[q][i][k] = 0.f;
  for (int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR; row < a.n;
       row += (int64_t)gridDim.x * RPB) {
    const float4 st = *(const float4*)(a.stats + 4 * row);
    // n: the normalised y;  r: the normalised residual row, later q;  z: the gate's argument, later
    // its gradient;  d: dr, later dx;  m: dh, later dh w'
    float n[NIT][V], r[NIT][V], z[NIT][V], d[NIT][V], m[NIT][V];
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      const int c = c0 + i * TPR * V;
      load_chunk<T, V>(X + row * a.ldx + c, D - c, r[i]);
      if (Y) load_chunk<T, V>(Y + row * a.ldy + c, D - c, n[i]);
      if (a.gate_mode == GNNEA_GATE_FULL)
        load_chunk<T, V>(Z + row * a.ldg + c, D - c, z[i]);
      else if (a.gate_mode == GNNEA_GATE_ROW)
        load_vec<TW, V>((const TW*)a.gate + c, D - c, z[i], 0.f);
      if (DR) load_chunk<T, V>(DR + row * a.lddr + c, D - c, d[i]);
      if (DH) load_chunk<T, V>(DH + row * a.lddh + c, D - c, m[i]);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        if (!DR) d[i][k] = 0.f;
        if (!DH) m[i][k] = 0.f;
        if (!Y) n[i][k] = 0.f;
      }
    }
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      const int c = c0 + i * TPR * V;
      float w[V], b[V], s[V], w2[V];
      load_vec<TW, V>(W ? W + c : W, D - c, w, 1.f);
      load_vec<TW, V>(Bv ? Bv + c : Bv, D - c, b, 0.f);
      load_vec<TW, V>(S ? S + c : S, D - c, s, 1.f);
      load_vec<TW, V>(W2 ? W2 + c : W2, D - c, w2, 1.f);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        if (Y) {
          const float g = a.gate_mode ? gate_of(z[i][k]).g : 1.f;
          n[i][k] = (n[i][k] - st.x) * st.y;
          r[i][k] = fmaf(a.alpha * s[k] * g, fmaf(n[i][k], w[k], b[k]), r[i][k]);
        }
        r[i][k] = (r[i][k] - st.z) * st.w;  // the normalised residual row
        acc[2][i][k] = fmaf(m[i][k], r[i][k], acc[2][i][k]);
        acc[3][i][k] += m[i][k];
        m[i][k] *= w2[k];
        sum[0] += m[i][k];  // m is 0 past the row
        sum[1] = fmaf(m[i][k], r[i][k], sum[1]);
      }
    }
    if (DH) {
      row_sum<TPR, 2>(sum, sh, turn);
      const float m0 = layer ? sum[0] * inv : 0.f, m1 = sum[1] * inv;
#pragma unroll
      for (int i = 0; i < NIT; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k)
          d[i][k] = fmaf(st.w, m[i][k] - m0 - r[i][k] * m1, d[i][k]);
    }
    sum[0] = sum[1] = 0.f;
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      const int c = c0 + i * TPR * V;
      if (a.dx) store_chunk<T, V>((T*)a.dx + row * a.lddx + c, D - c, d[i]);
      if (!Y) continue;
      float w[V], b[V], s[V];
      load_vec<TW, V>(W ? W + c : W, D - c, w, 1.f);
      load_vec<TW, V>(Bv ? Bv + c : Bv, D - c, b, 0.f);
      load_vec<TW, V>(S ? S + c : S, D - c, s, 1.f);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float u = fmaf(n[i][k], w[k], b[k]);
        const Gate g = a.gate_mode ? gate_of(z[i][k]) : Gate{1.f, 0.f};
        const float dg = c + k < D ? d[i][k] * g.g : 0.f, sd = a.alpha * s[k] * dg;
        acc[0][i][k] = fmaf(dg, n[i][k], acc[0][i][k]);
        acc[1][i][k] += dg;
        z[i][k] = sd * u * g.rest;
        r[i][k] = sd * w[k];
        sum[0] += r[i][k];
        sum[1] = fmaf(r[i][k], n[i][k], sum[1]);
      }
      if (a.gate_mode == GNNEA_GATE_FULL && a.dgate)
        store_chunk<T, V>((T*)a.dgate + row * a.lddg + c, D - c, z[i]);
    }
    if (Y && a.dy) {
      float q0 = 0.f, q1 = 0.f;
      if (a.post) {
        row_sum<TPR, 2>(sum, sh, turn);
        q0 = layer ? sum[0] * inv : 0.f;
        q1 = sum[1] * inv;
      }
#pragma unroll
      for (int i = 0; i < NIT; ++i) {
        const int c = c0 + i * TPR * V;
#pragma unroll
        for (int k = 0; k < V; ++k) r[i][k] = st.y * (r[i][k] - q0 - n[i][k] * q1);
        store_chunk<T, V>((T*)a.dy + row * a.lddy + c, D - c, r[i]);
      }
    }
  }
  if (!a.part) return;
  // the workgroup's column sums: over its rows in row order, one of the four after another
#pragma unroll
  for (int q = 0; q < kNormSums; ++q) {
    if (!(a.sums & (1 << q))) continue;
    float* out = a.part + ((int64_t)blockIdx.x * kNormSums + q) * D;
    if constexpr (RPB == 1) {
#pragma unroll
      for (int i = 0; i < NIT; ++i) {
        const int c = c0 + i * TPR * V;
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (c + k < D) out[c + k] = acc[q][i][k];
      }
    } else {
      __syncthreads();
      const int rid = threadIdx.x / TPR;
#pragma unroll
      for (int i = 0; i < NIT; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k) fold[rid * (TPR * NIT * V) + c0 + i * TPR * V + k] = acc[q][i][k];
      __syncthreads();
      for (int c = threadIdx.x; c < D; c += NT) {
        float s = fold[c];
        for (int w = 1; w < RPB; ++w) s += fold[w * (TPR * NIT * V) + c];
        out[c] = s;
      }
    }
  }
}

// The workgroups' column sums in workgroup order (fp64), and the six vector gradients from them.
// 64 columns per workgroup, 16 waves take every 16th partial row.
template <typename TW>
__global__ __launch_bounds__(1024) void k_norm_fold(const gnnea_norm a, int blocks) {
  __shared__ double sh[16][64];
  const int c = blockIdx.x * 64 + lane_id(), w = wave_id();
  const bool in = c < a.D;
  float got[kNormSums];
#pragma unroll
  for (int q = 0; q < kNormSums; ++q) {
    got[q] = 0.f;
    if (!(a.sums & (1 << q))) continue;
    double s = 0.0;
    if (in) {
      const float* p = a.part + (int64_t)q * a.D + c;
      const int64_t step = (int64_t)kNormSums * a.D;
      int b = w;
      for (; b + 112 < blocks; b += 128) {
        float v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = p[(b + 16 * u) * step];
#pragma unroll
        for (int u = 0; u < 8; ++u) s += (double)v[u];
      }
      for (; b < blocks; b += 16) s += (double)p[b * step];
    }
    __syncthreads();
    sh[w][lane_id()] = s;
    __syncthreads();
    if (w == 0) {
      for (int k = 1; k < 16; ++k) s += sh[k][lane_id()];
      got[q] = (float)s;
    }
  }
  if (w != 0 || !in) return;
  const float pw = a.post_w ? to_f32<TW>(((const TW*)a.post_w)[c]) : 1.f;
  const float pb = a.post_b ? to_f32<TW>(((const TW*)a.post_b)[c]) : 0.f;
  const float s = a.scale ? to_f32<TW>(((const TW*)a.scale)[c]) : 1.f;
  const float both = fmaf(pw, got[0], pb * got[1]);
  if (a.dpost_w) ((TW*)a.dpost_w)[c] = from_f32<TW>(a.alpha * s * got[0]);
  if (a.dpost_b) ((TW*)a.dpost_b)[c] = from_f32<TW>(a.alpha * s * got[1]);
  if (a.dscale) ((TW*)a.dscale)[c] = from_f32<TW>(a.alpha * both);
  if (a.dpre_w) ((TW*)a.dpre_w)[c] = from_f32<TW>(got[2]);
  if (a.dpre_b) ((TW*)a.dpre_b)[c] = from_f32<TW>(got[3]);
  if (a.gate_mode == GNNEA_GATE_ROW && a.dgate) {
    const float rest = gate_of(to_f32<TW>(((const TW*)a.gate)[c])).rest;
    ((TW*)a.dgate)[c] = from_f32<TW>(a.alpha * s * rest * both);
  }
}

struct NormPlan { int tpr, nit, blocks; };

// Threads per row: 16 lanes up to 16 chunks, a wave up to 1024 values, then the smallest workgroup
// whose threads hold 16 values each.
static NormPlan norm_plan(int64_t n, int D, int V, bool bwd) {
  const int chunks = (D + V - 1) / V, most = 16 / V;
  NormPlan p;
  p.tpr = chunks <= 16 ? 16 : 64;
  if (chunks > 64 * most) p.tpr = chunks <= 256 * most ? 256 : 512;
  p.nit = (chunks + p.tpr - 1) / p.tpr;
  if (p.nit == 3) p.nit = 4;
  const int rpb = p.tpr < 256 ? 256 / p.tpr : 1;
  const int64_t want = (n + rpb - 1) / rpb;
  // backward: rows per workgroup go up with n, so that the column sums stay few
  const int64_t cap = bwd ? (p.tpr >= 256 ? 256 * (1024 / p.tpr) : 256 * 4) : 256 * 32;
  p.blocks = (int)(want < cap ? want : cap);
  return p;
}

static int norm_check(const gnnea_norm* a, bool bwd) {
  if (!a || a->n < 0 || a->D < 1 || a->D > kNormMaxD) return GNNEA_EINVAL;
  if (a->dtype != GNNEA_F32 && a->dtype != GNNEA_BF16) return GNNEA_EINVAL;
  if (a->w_dtype != GNNEA_F32 && a->w_dtype != GNNEA_BF16) return GNNEA_EINVAL;
  if (a->dtype == GNNEA_F32 && a->w_dtype != GNNEA_F32) return GNNEA_EINVAL;
  if (a->kind != GNNEA_NORM_RMS && a->kind != GNNEA_NORM_LAYER) return GNNEA_EINVAL;
  if (a->gate_mode < GNNEA_GATE_NONE || a->gate_mode > GNNEA_GATE_ROW) return GNNEA_EINVAL;
  if ((a->gate_mode != GNNEA_GATE_NONE) != (a->gate != nullptr)) return GNNEA_EINVAL;
  if (!(a->eps > 0.f)) return GNNEA_EINVAL;
  if (!a->y && (a->gate || a->scale || a->post || !a->pre)) return GNNEA_EINVAL;
  if (!a->post && (a->post_w || a->post_b)) return GNNEA_EINVAL;
  if (!a->pre && (a->pre_w || a->pre_b)) return GNNEA_EINVAL;
  if (a->n == 0) return GNNEA_OK;
  const int64_t D = a->D;
  if (!a->x || a->ldx < D || (a->y && a->ldy < D)) return GNNEA_EINVAL;
  if (a->gate_mode == GNNEA_GATE_FULL && a->ldg < D) return GNNEA_EINVAL;
  if (!bwd) {
    if ((a->y && !a->r) || (a->pre && !a->h)) return GNNEA_EINVAL;
    if ((a->r && a->ldr < D) || (a->h && a->ldh < D)) return GNNEA_EINVAL;
  } else {
    if (!a->stats) return GNNEA_EINVAL;
    if ((a->dr && a->lddr < D) || (a->dh && (a->lddh < D || !a->pre))) return GNNEA_EINVAL;
    if ((a->dx && a->lddx < D) || (a->dy && (a->lddy < D || !a->y))) return GNNEA_EINVAL;
    if (a->gate_mode == GNNEA_GATE_FULL && a->dgate && a->lddg < D) return GNNEA_EINVAL;
  }
  if (a->stats && ((uintptr_t)a->stats & 15)) return GNNEA_EALIGN;
  return GNNEA_OK;
}

// which of the column sums A, B, C, E the asked vector gradients take
static int norm_sums(const gnnea_norm& a) {
  int s = 0;
  const bool both = a.dscale || (a.gate_mode == GNNEA_GATE_ROW && a.dgate);
  if (a.dpost_w || both) s |= 1;
  if (a.dpost_b || (both && a.post_b)) s |= 2;
  if (a.dpre_w) s |= 4;
  if (a.dpre_b) s |= 8;
  return s;
}

#define GNNEA_NORM_LAUNCH(K, TPR, NIT)                                                     \
  hipLaunchKernelGGL((K<T, TW, TPR, NIT>), dim3(p.blocks), dim3(TPR < 256 ? 256 : TPR), 0, s, a)

template <typename T, typename TW, bool BWD>
static int norm_launch(const gnnea_norm& a, const NormPlan& p, hipStream_t s) {
  bool done = false;
#define GNNEA_NORM_CASE(TPR, NIT)                               \
  if (p.tpr == TPR && p.nit == NIT) {                           \
    if constexpr (BWD) GNNEA_NORM_LAUNCH(k_norm_bwd, TPR, NIT); \
    else GNNEA_NORM_LAUNCH(k_norm_fwd, TPR, NIT);               \
    done = true;                                                \
  }
  GNNEA_NORM_CASE(16, 1)
  GNNEA_NORM_CASE(64, 1)
  GNNEA_NORM_CASE(64, 2)
  GNNEA_NORM_CASE(256, 2)
  GNNEA_NORM_CASE(512, 2)
  if constexpr (RowChunk<T>::V == 8) {
    GNNEA_NORM_CASE(256, 1)
  } else {
    GNNEA_NORM_CASE(64, 4)
    GNNEA_NORM_CASE(256, 4)
    GNNEA_NORM_CASE(512, 4)
  }
#undef GNNEA_NORM_CASE
  GNNEA_LAUNCH_CHECK();
  return done ? 0 : GNNEA_EINVAL;
}

template <bool BWD>
static int norm_dispatch(const gnnea_norm& a, const NormPlan& p, hipStream_t s) {
  if (a.dtype == GNNEA_F32) return norm_launch<float, float, BWD>(a, p, s);
  if (a.w_dtype == GNNEA_F32) return norm_launch<bf16_t, float, BWD>(a, p, s);
  return norm_launch<bf16_t, bf16_t, BWD>(a, p, s);
}

}  // namespace gnnea

using namespace gnnea;

extern "C" int gnnea_norm_fwd(const gnnea_norm* arg, void* stream) {
  const int rc = norm_check(arg, false);
  if (rc || arg->n == 0) return rc;
  return norm_dispatch<false>(*arg, norm_plan(arg->n, arg->D, arg->dtype == GNNEA_F32 ? 4 : 8, false),
                              (hipStream_t)stream);
}

extern "C" int64_t gnnea_norm_bwd_ws_bytes(int64_t n, int32_t D, int dtype) {
  if (n < 0 || D < 1 || D > kNormMaxD || (dtype != GNNEA_F32 && dtype != GNNEA_BF16))
    return GNNEA_EINVAL;
  return (int64_t)norm_plan(n, D, dtype == GNNEA_F32 ? 4 : 8, true).blocks * kNormSums * D * 4;
}

extern "C" int gnnea_norm_bwd(const gnnea_norm* arg, void* ws, int64_t ws_bytes, void* stream) {
  const int rc = norm_check(arg, true);
  if (rc) return rc;
  gnnea_norm a = *arg;
  a.sums = norm_sums(a);
  const NormPlan p = norm_plan(a.n, a.D, a.dtype == GNNEA_F32 ? 4 : 8, true);
  a.part = nullptr;
  if (a.sums) {
    if (ws_bytes < (int64_t)p.blocks * kNormSums * a.D * 4) return GNNEA_EWORKSPACE;
    if (p.blocks && (!ws || ((uintptr_t)ws & 15))) return ws ? GNNEA_EALIGN : GNNEA_EINVAL;
    a.part = (float*)ws;
  }
  hipStream_t s = (hipStream_t)stream;
  if (a.n > 0) {
    const int rc2 = norm_dispatch<true>(a, p, s);
    if (rc2) return rc2;
  }
  if (a.sums) {  // also for no rows: the gradients are then zero
    const int g = div_up(a.D, 64);
    if (a.w_dtype == GNNEA_F32)
      hipLaunchKernelGGL(k_norm_fold<float>, dim3(g), dim3(1024), 0, s, a, p.blocks);
    else
      hipLaunchKernelGGL(k_norm_fold<bf16_t>, dim3(g), dim3(1024), 0, s, a, p.blocks);
    GNNEA_LAUNCH_CHECK();
  }
  return 0;
}

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
// A row is held by TPR threads (16 lanes, a wave, or as many waves as leave 8 values to a thread),
// NIT chunks of 16 B per thread; rows of odd widths use the same 16-B accesses at the element's
// alignment.  A thread keeps its columns from row to row, so the vectors are read once per thread
// and the column sums stay with it (registers; LDS where a row takes a workgroup, whose registers
// are full), and the next row is read while one is computed.  Per-row reads of the vectors and
// element-wise tails had cost 1.9x: 1M rows of 300 fp32, training pass 5.08 ms, now 3.27.
//
// Measured: 1M x 300 fp32 with a full gate, forward 1.20 ms (6.0 GB, 5.0 TB/s), backward 2.05
// (9.6 GB, 4.7 TB/s); bf16 LayerNorm of 8191 rows, 4096 wide: forward 50 us, backward 89 (5.3 and
// 4.5 TB/s), 4097 wide: 79 and 116 (a ninth wave for one value, and rows at odd addresses); 30000 x
// 300 bf16 forward 22 us (4.1 TB/s); 2000 x 300 7 + 10 + 5 us of launches.
//
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

// A product rounded by itself.  The backward subtracts its row's mean from it: fused into that
// difference it would be exact there and rounded in the mean, and a row whose gradient is 0 (one
// value, or all alike) would keep the rounding, times 1 / deviation.
__device__ __forceinline__ float product(float a, float b) {
#pragma clang fp contract(off)
  return a * b;
}

// s / n from inv, the rounded 1 / n, and 1 / sqrt(v).  Rows of up to a wave (TPR <= 64) take one step
// more, to within 0.6 of a last place instead of 1.5: the gradients of short rows are what is left of
// a difference, and with them the error of a mean or a root.  In wide ones it has no weight, and their
// waves wait for each other's sums: 8191 x 4097 bf16 forward 78 us without the steps, 82 with them.
template <int TPR>
__device__ __forceinline__ float mean_of(float s, int n, float inv) {
  const float q = s * inv;
  return TPR <= 64 ? fmaf(fmaf(-(float)n, q, s), inv, q) : q;
}
template <int TPR>
__device__ __forceinline__ float inv_sqrt(float v) {
  const float r = __builtin_amdgcn_rsqf(v);
  if (TPR > 64 || !(v < INFINITY)) return r;
  return fmaf(0.5f * r, fmaf(-v * r, r, 1.f), r);
}

typedef uint32_t Half4 __attribute__((ext_vector_type(2), aligned(2)));  // four bf16

// value c of a vector of either type, `none` where there is none
__device__ __forceinline__ float vec_at(const void* p, bool bf16, int c, float none) {
  if (!p) return none;
  return bf16 ? bf16_to_f32(((const bf16_t*)p)[c]) : ((const float*)p)[c];
}

// V values of a vector of either type from column c on (D: its length)
template <int V>
__device__ __forceinline__ void vec_chunk(const void* p, bool bf16, int c, int D, float none,
                                          float (&f)[V]) {
  if (!p || D < V) {
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = vec_at(p, bf16, c + k < D ? c + k : D - 1, none);
  } else if (bf16) {
#pragma unroll
    for (int k = 0; k < V; k += 4) {
      const Half4 r = *(const Half4*)((const bf16_t*)p + c + k);
      const float4 v = Vec4<bf16_t>::get(make_uint2(r.x, r.y));
      f[k] = v.x; f[k + 1] = v.y; f[k + 2] = v.z; f[k + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < V; k += 4) {
      const uint4 r = load16<float>((const float*)p + c + k);
      f[k] = __builtin_bit_cast(float, r.x);
      f[k + 1] = __builtin_bit_cast(float, r.y);
      f[k + 2] = __builtin_bit_cast(float, r.z);
      f[k + 3] = __builtin_bit_cast(float, r.w);
    }
  }
}

// The columns of a thread: chunk i of NIT begins at column (i TPR + t) V; the last chunk of a row
// is moved back so that it ends with the row (its first values are then the neighbour's too, who
// computes and stores the same; the sums take each once).
template <int TPR, int NIT, int V> struct Cols {
  int D, t;
  __device__ __forceinline__ int want(int i) const {
    return (i * (TPR < 256 ? TPR : (int)blockDim.x) + t) * V;
  }
  __device__ __forceinline__ bool has(int i) const { return want(i) < D; }
  __device__ __forceinline__ int at(int i) const {
    const int c = want(i);
    return D >= V && c > D - V ? D - V : c;
  }
  // whether every value of the wave's chunks is its thread's own (uniform): then no sum needs masks
  __device__ __forceinline__ bool whole() const {
    return TPR > 16 && __builtin_amdgcn_readfirstlane(
        (int)(want(NIT - 1) - lane_id() * V + 64 * V <= D));
  }
  // whether value k of chunk i is the thread's own: all are, but in a row's last chunk
  __device__ __forceinline__ bool own(int i, int k) const {
    if (i < NIT - 1) return true;
    if (TPR == 16 && k >= D) return false;
    return k >= (has(i) ? want(i) - at(i) : V);
  }
};

template <typename T, int TPR, int NIT, int V>
__device__ __forceinline__ void load_row(const Cols<TPR, NIT, V>& C, const T* p, uint4 (&r)[NIT]) {
#pragma unroll
  for (int i = 0; i < NIT; ++i) {
    r[i] = make_uint4(0, 0, 0, 0);
    if (!C.has(i)) continue;
    if (TPR > 16 || C.D >= V) {
      r[i] = load16<T>(p + C.at(i));
    } else {  // rows narrower than 16 B (one thread per row)
      uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (k < C.D) {
          if constexpr (V == 4) w[k] = __builtin_bit_cast(uint32_t, (float)to_f32<T>(p[k]));
          else w[k / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, p[k]) << (16 * (k & 1));
        }
      r[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}
template <typename T, int TPR, int NIT, int V>
__device__ __forceinline__ void store_row(const Cols<TPR, NIT, V>& C, T* p, int i,
                                          const float (&f)[V]) {
  if (!C.has(i)) return;
  if (TPR > 16 || C.D >= V) store_chunk<T, V>(p + C.at(i), V, f);
  else store_chunk<T, V>(p, C.D, f);
}

// the sum over each row of 16 lanes, in all of them
__device__ __forceinline__ float sum16(float v) {
  v += mov_dpp_f32<0xB1>(v);
  v += mov_dpp_f32<0x4E>(v);
  v += mov_dpp_f32<0x141>(v);
  v += mov_dpp_f32<0x140>(v);
  return v;
}

// Sums of NS values over the TPR threads of a row; every thread gets them, from the same order of
// additions.  16 lanes and a wave stay in registers; a workgroup goes once through LDS (two
// buffers in turn, so one barrier per sum is enough): every 16 lanes take the 16 places of its
// waves, those of waves that it has not are 0.
template <int TPR, int NS>
__device__ __forceinline__ void row_sum(float (&v)[NS], float (*sh)[16][2], int& turn) {
#pragma unroll
  for (int k = 0; k < NS; ++k) {
    v[k] = sum16(v[k]);
    if constexpr (TPR >= 64)
      v[k] = ((readlane_f(v[k], 0) + readlane_f(v[k], 16)) + readlane_f(v[k], 32)) +
             readlane_f(v[k], 48);
  }
  if constexpr (TPR > 64) {
    float(*b)[2] = sh[turn];
    turn ^= 1;
    if (lane_id() == 0) {
#pragma unroll
      for (int k = 0; k < NS; ++k) b[wave_id()][k] = v[k];
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < NS; ++k) v[k] = sum16(b[threadIdx.x & 15][k]);
  }
}

// The thread's sum of its own values f, or of their squares about c.
template <bool SQUARES, int TPR, int NIT, int V>
__device__ __forceinline__ float own_sum(const Cols<TPR, NIT, V>& C, bool whole,
                                         const float (&f)[NIT][V], float c) {
  float s = 0.f;
  if (whole) {
#pragma unroll
    for (int i = 0; i < NIT; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float d = f[i][k] - c;
        s = SQUARES ? fmaf(d, d, s) : s + f[i][k];
      }
  } else {
#pragma unroll
    for (int i = 0; i < NIT; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float d = C.own(i, k) ? (SQUARES ? f[i][k] - c : f[i][k]) : 0.f;
        s = SQUARES ? fmaf(d, d, s) : s + d;
      }
  }
  return s;
}

// mean and 1 / sqrt(var + eps) (0 and 1 / rms) of the row's values f.  LayerNorm in a workgroup:
// each wave sums its values, then their squares about its own mean, and the waves' pairs are put
// together about the row's mean (one barrier instead of two, and no difference of large sums).
// share: the number of values of each wave, mine: 1 / this wave's (1 / D where a wave has a row).
template <int TPR, int NIT, int V>
__device__ __forceinline__ void row_stats(const Cols<TPR, NIT, V>& C, bool whole,
                                          const float (&f)[NIT][V], float inv, float mine,
                                          bool layer, float eps, float (*sh)[16][2],
                                          const float* share, int& turn, float& mean, float& rho) {
  mean = 0.f;
  float s[1];
  int none = 0;
  if (layer) {
    s[0] = own_sum<false>(C, whole, f, 0.f);
    row_sum<(TPR < 64 ? TPR : 64), 1>(s, sh, none);
    mean = mean_of<TPR>(s[0], C.D, mine);
  }
  s[0] = own_sum<true>(C, whole, f, mean);
  if constexpr (TPR <= 64) {
    row_sum<TPR, 1>(s, sh, none);
  } else if (!layer) {
    row_sum<TPR, 1>(s, sh, turn);
  } else {
    row_sum<64, 1>(s, sh, none);
    float(*b)[2] = sh[turn];
    turn ^= 1;
    if (lane_id() == 0) b[wave_id()][0] = mean, b[wave_id()][1] = s[0];
    __syncthreads();
    const int q = threadIdx.x & 15;
    const float mq = b[q][0];
    mean = sum16(mq * share[q]) * inv;
    const float d = mq - mean;
    s[0] = sum16(fmaf(d * d, share[q], b[q][1]));
  }
  rho = inv_sqrt<TPR>(fmaf(s[0], inv, eps));
}

// The thread's sums of its own values q, and of q n.
template <int TPR, int NIT, int V>
__device__ __forceinline__ void own_sums(const Cols<TPR, NIT, V>& C, bool whole,
                                         const float (&q)[NIT][V], const float (&n)[NIT][V],
                                         float (&sum)[2]) {
  sum[0] = sum[1] = 0.f;
  if (whole) {
#pragma unroll
    for (int i = 0; i < NIT; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        sum[0] += q[i][k];
        sum[1] = fmaf(q[i][k], n[i][k], sum[1]);
      }
  } else {
#pragma unroll
    for (int i = 0; i < NIT; ++i)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float v = C.own(i, k) ? q[i][k] : 0.f;
        sum[0] += v;
        sum[1] = fmaf(v, n[i][k], sum[1]);
      }
  }
}

// The number of a row's values that each wave of the workgroup holds (0 for waves that it has not,
// whose places in sh are cleared).
template <int TPR, int NIT, int V>
__device__ __forceinline__ void wave_shares(const Cols<TPR, NIT, V>& C, float* share,
                                            float (*sh)[16][2]) {
  if constexpr (TPR > 64) {
    if (threadIdx.x < 64) ((float*)sh)[threadIdx.x] = 0.f;
    if (threadIdx.x < 16) {
      int n = 0;
      for (int i = 0; i < NIT; ++i)
        n += max(0, min(64 * V, C.D - (i * (int)blockDim.x + (int)threadIdx.x * 64) * V));
      share[threadIdx.x] = threadIdx.x < blockDim.x / 64 ? (float)n : 0.f;
    }
    __syncthreads();
  }
}

template <int NIT, int V>
__device__ __forceinline__ void clear_row(float (&f)[NIT][V]) {
#pragma unroll
  for (int i = 0; i < NIT; ++i)
#pragma unroll
    for (int k = 0; k < V; ++k) f[i][k] = 0.f;
}

// Where workgroup b of `blocks` leaves sum q of column c: 16 columns' four sums together, the
// workgroups' next to each other, as they are read.
__device__ __forceinline__ int64_t part_at(int c, int b, int blocks, int q) {
  return (((int64_t)(c >> 4) * blocks + b) * kNormSums + q) * 16 + (c & 15);
}

// IN: 0: no y; 1: y; 2: y and a gate of its own for every element (a gate shared by all rows is
// part of the thread's constants: P = alpha scale g post_w, Q = alpha scale g post_b)
template <typename T, int TPR, int NIT, int IN>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void k_norm_fwd(const gnnea_norm a) {
  constexpr int V = RowChunk<T>::V, RPB = TPR < 256 ? 256 / TPR : 1;
  __shared__ float sh[2][16][2];
  int turn = 0;
  const Cols<TPR, NIT, V> C{a.D, (int)(threadIdx.x % (TPR < 256 ? TPR : 1024))};
  const bool layer = a.kind == GNNEA_NORM_LAYER, wb = a.w_dtype == GNNEA_BF16;
  const float inv = 1.f / (float)a.D;
  __shared__ float share[16];
  wave_shares(C, share, sh);
  const bool whole = C.whole();
  const float mine = TPR > 64 ? (share[wave_id()] > 0.f ? 1.f / share[wave_id()] : 0.f) : inv;
  float P[NIT][V], Q[NIT][V], W[NIT][V], B[NIT][V];
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t row = (int64_t)xcd_remap(blockIdx.x, gridDim.x) * RPB + threadIdx.x / TPR;
  uint4 rx[NIT], ry[NIT], rz[NIT];
  auto load = [&](int64_t at) {
    load_row<T>(C, (const T*)a.x + at * a.ldx, rx);
    if constexpr (IN) load_row<T>(C, (const T*)a.y + at * a.ldy, ry);
    if constexpr (IN == 2) load_row<T>(C, (const T*)a.gate + at * a.ldg, rz);
  };
  if (row < a.n) load(row);
#pragma unroll
  for (int i = 0; i < NIT; ++i) {
    const int c = min(C.at(i), max(a.D - V, 0));  // (lanes past the row: anything that is there)
    if constexpr (IN) {
      float s[V], g[V];
      vec_chunk(a.scale, wb, c, a.D, 1.f, s);
      vec_chunk(a.post_w, wb, c, a.D, 1.f, P[i]);
      vec_chunk(a.post_b, wb, c, a.D, 0.f, Q[i]);
      if (a.gate_mode == GNNEA_GATE_ROW) vec_chunk(a.gate, wb, c, a.D, 0.f, g);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        s[k] *= a.alpha;
        if (a.gate_mode == GNNEA_GATE_ROW) s[k] *= gate_of(g[k]).g;
        P[i][k] *= s[k];
        Q[i][k] *= s[k];
      }
    }
    vec_chunk(a.pre_w, wb, c, a.D, 1.f, W[i]);
    vec_chunk(a.pre_b, wb, c, a.D, 0.f, B[i]);
  }
  for (; row < a.n; row += step) {
    float r[NIT][V], y[NIT][V], z[NIT][V];
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      unpack16(rx[i], r[i]);
      if constexpr (IN) unpack16(ry[i], y[i]);
      if constexpr (IN == 2) unpack16(rz[i], z[i]);
    }
    if (row + step < a.n) load(row + step);  // on its way while this row is computed
    float mean = 0.f, rho = 1.f, mean2 = 0.f, rho2 = 1.f;
    if constexpr (IN) {
      if (a.post) row_stats(C, whole, y, inv, mine, layer, a.eps, sh, share, turn, mean, rho);
#pragma unroll
      for (int i = 0; i < NIT; ++i) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float u = fmaf((y[i][k] - mean) * rho, P[i][k], Q[i][k]);
          if constexpr (IN == 2) r[i][k] = fmaf(gate_of(z[i][k]).g, u, r[i][k]);
          else r[i][k] += u;
        }
        store_row<T>(C, (T*)a.r + row * a.ldr, i, r[i]);
      }
    }
    if (a.pre) {
      row_stats(C, whole, r, inv, mine, layer, a.eps, sh, share, turn, mean2, rho2);
#pragma unroll
      for (int i = 0; i < NIT; ++i) {
        float h[V];
#pragma unroll
        for (int k = 0; k < V; ++k) h[k] = fmaf((r[i][k] - mean2) * rho2, W[i][k], B[i][k]);
        store_row<T>(C, (T*)a.h + row * a.ldh, i, h);
      }
    }
    if (a.stats && C.t == 0)
      *(float4*)(a.stats + 4 * row) = make_float4(mean, rho, mean2, rho2);
  }
}

// BIAS: post_b or pre_b takes part (without them the sums B and E are not formed)
template <typename T, int TPR, int NIT, int IN, bool BIAS>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void k_norm_bwd(const gnnea_norm a) {
  // the next row is read while this one is computed, where registers allow it (1024 threads with a
  // full gate have none left)
  constexpr bool kAhead = TPR <= 512 || IN < 2;
  constexpr int V = RowChunk<T>::V, RPB = TPR < 256 ? 256 / TPR : 1;
  __shared__ float sh[2][16][2];
  // the column sums: in registers, or (rows of a workgroup, whose registers are short) in LDS,
  // every thread its own places
  constexpr bool kLds = TPR > 64;
  constexpr int kHeld = kLds ? 1 : kNormSums;
  extern __shared__ float fold[];
  int turn = 0;
  const Cols<TPR, NIT, V> C{a.D, (int)(threadIdx.x % (TPR < 256 ? TPR : 1024))};
  const bool layer = a.kind == GNNEA_NORM_LAYER, wb = a.w_dtype == GNNEA_BF16;
  const float inv = 1.f / (float)a.D;
  const bool whole = C.whole();
  float P[NIT][V], Q[NIT][V], W[NIT][V], acc[kHeld][NIT][V];
  if constexpr (!kLds) {
#pragma unroll
    for (int q = 0; q < kHeld; ++q) clear_row(acc[q]);
  }
  if constexpr (TPR > 64) {  // (places of waves that the workgroup has not: 0)
    if (threadIdx.x < 64) ((float*)sh)[threadIdx.x] = 0.f;
    __syncthreads();
  }
  // four values of a sum at a time, the threads' next to each other
  const int nt = blockDim.x;
  float4* held = (float4*)fold + threadIdx.x;
  if constexpr (kLds) {
#pragma unroll
    for (int j = 0; j < kNormSums * NIT * V / 4; ++j) held[j * nt] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  // sum q of the columns of chunk i: + x y
  auto add = [&](int q, int i, const float (&x)[V], const float (&y)[V]) {
    if constexpr (kLds) {
#pragma unroll
      for (int j = 0; j < V / 4; ++j) {
        float4* p = held + ((q * NIT + i) * (V / 4) + j) * nt;
        float4 f = *p;
        f.x = fmaf(x[4 * j], y[4 * j], f.x);
        f.y = fmaf(x[4 * j + 1], y[4 * j + 1], f.y);
        f.z = fmaf(x[4 * j + 2], y[4 * j + 2], f.z);
        f.w = fmaf(x[4 * j + 3], y[4 * j + 3], f.w);
        *p = f;
      }
    } else {
#pragma unroll
      for (int k = 0; k < V; ++k) acc[q][i][k] = fmaf(x[k], y[k], acc[q][i][k]);
    }
  };
  float ones[V];
#pragma unroll
  for (int k = 0; k < V; ++k) ones[k] = 1.f;
  const int64_t step = (int64_t)gridDim.x * RPB;
  int64_t row = (int64_t)xcd_remap(blockIdx.x, gridDim.x) * RPB + threadIdx.x / TPR;
  uint4 rx[NIT], ry[NIT], rz[NIT], rd[NIT], rm[NIT];
  float4 rs;
#pragma unroll
  for (int i = 0; i < NIT; ++i) rd[i] = rm[i] = make_uint4(0, 0, 0, 0);
  auto load = [&](int64_t at) {
    rs = *(const float4*)(a.stats + 4 * at);
    load_row<T>(C, (const T*)a.x + at * a.ldx, rx);
    if constexpr (IN) load_row<T>(C, (const T*)a.y + at * a.ldy, ry);
    if constexpr (IN == 2) load_row<T>(C, (const T*)a.gate + at * a.ldg, rz);
    if (a.dr) load_row<T>(C, (const T*)a.dr + at * a.lddr, rd);
    if (a.dh) load_row<T>(C, (const T*)a.dh + at * a.lddh, rm);
  };
#pragma unroll
  for (int i = 0; i < NIT; ++i) {
    const int c = min(C.at(i), max(a.D - V, 0));
    if constexpr (IN) {
      float s[V], g[V];
      vec_chunk(a.scale, wb, c, a.D, 1.f, s);
      vec_chunk(a.post_w, wb, c, a.D, 1.f, P[i]);
      vec_chunk(BIAS ? a.post_b : nullptr, wb, c, a.D, 0.f, Q[i]);
      if (a.gate_mode == GNNEA_GATE_ROW) vec_chunk(a.gate, wb, c, a.D, 0.f, g);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        s[k] *= a.alpha;
        if (a.gate_mode == GNNEA_GATE_ROW) s[k] *= gate_of(g[k]).g;
        P[i][k] *= s[k];
        Q[i][k] *= s[k];
      }
    }
    vec_chunk(a.pre_w, wb, c, a.D, 1.f, W[i]);
  }
  // (after the vectors: before them the loop came out 20 % slower at 8191 rows of 4097 bf16)
  if (kAhead && row < a.n) load(row);
  for (; row < a.n; row += step) {
    if (!kAhead) load(row);
    // n: the normalised y;  r: the normalised residual row, later q;  z: the gate's argument, later
    // its gradient;  d: dr, later dx;  m: dh, later dh w'
    float n[NIT][V], r[NIT][V], z[NIT][V], d[NIT][V], m[NIT][V];
    const float4 st = rs;
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      unpack16(rx[i], r[i]);
      if constexpr (IN) unpack16(ry[i], n[i]);
      if constexpr (IN == 2) unpack16(rz[i], z[i]);
      unpack16(rd[i], d[i]);
      unpack16(rm[i], m[i]);
    }
    if (kAhead && row + step < a.n) load(row + step);
    float sum[2];
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
#pragma unroll
      for (int k = 0; k < V; ++k) {
        if constexpr (IN) {
          n[i][k] = (n[i][k] - st.x) * st.y;
          const float u = fmaf(n[i][k], P[i][k], Q[i][k]);
          if constexpr (IN == 2) r[i][k] = fmaf(gate_of(z[i][k]).g, u, r[i][k]);
          else r[i][k] += u;
        }
        r[i][k] = (r[i][k] - st.z) * st.w;
        // (values of the neighbour's columns go into sums that are not written)
      }
      add(2, i, m[i], r[i]);
      if constexpr (BIAS) add(3, i, m[i], ones);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        m[i][k] = product(m[i][k], W[i][k]);
      }
    }
    if (a.dh) {
      own_sums(C, whole, m, r, sum);
      row_sum<TPR, 2>(sum, sh, turn);
      const float m0 = layer ? mean_of<TPR>(sum[0], a.D, inv) : 0.f, m1 = mean_of<TPR>(sum[1], a.D, inv);
#pragma unroll
      for (int i = 0; i < NIT; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k)
          d[i][k] = fmaf(st.w, m[i][k] - m0 - r[i][k] * m1, d[i][k]);
    }
#pragma unroll
    for (int i = 0; i < NIT; ++i) {
      if (a.dx) store_row<T>(C, (T*)a.dx + row * a.lddx, i, d[i]);
      if constexpr (IN) {
        float dg[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
          dg[k] = d[i][k];
          if constexpr (IN == 2) {
            const Gate g = gate_of(z[i][k]);
            dg[k] *= g.g;
            z[i][k] = dg[k] * g.rest * fmaf(n[i][k], P[i][k], Q[i][k]);
          }
          r[i][k] = product(dg[k], P[i][k]);
        }
        add(0, i, dg, n[i]);
        if constexpr (BIAS) add(1, i, dg, ones);
        if (IN == 2 && a.dgate) store_row<T>(C, (T*)a.dgate + row * a.lddg, i, z[i]);
      }
    }
    if (IN && a.dy) {
      float q0 = 0.f, q1 = 0.f;
      if (a.post) {
        own_sums(C, whole, r, n, sum);
        row_sum<TPR, 2>(sum, sh, turn);
        q0 = layer ? mean_of<TPR>(sum[0], a.D, inv) : 0.f;
        q1 = mean_of<TPR>(sum[1], a.D, inv);
      }
#pragma unroll
      for (int i = 0; i < NIT; ++i) {
#pragma unroll
        for (int k = 0; k < V; ++k) r[i][k] = st.y * (r[i][k] - q0 - n[i][k] * q1);
        store_row<T>(C, (T*)a.dy + row * a.lddy, i, r[i]);
      }
    }
  }
  if (!a.part) return;
  // the workgroup's column sums
  if constexpr (kLds) {
    // lanes over the 64 values of 16 columns, each from the place of the thread that holds it
    __syncthreads();
    for (int e = threadIdx.x; e < (C.D + 15) / 16 * 64; e += nt) {
      const int c = (e >> 6) * 16 + (e & 15), q = (e >> 4) & 3;
      if (c >= C.D || !(a.sums & (1 << q))) continue;
      const int chunk = c / V, k = c - min(chunk * V, C.D - V);
      a.part[part_at(c, blockIdx.x, gridDim.x, q)] =
          fold[(((q * NIT + chunk / nt) * (V / 4) + k / 4) * nt + chunk % nt) * 4 + k % 4];
    }
  } else {
    // over its rows in row order, one sum after another
    constexpr int kRow = TPR * NIT * V;  // (of LDS, for each of the workgroup's rows)
#pragma unroll
    for (int q = 0; q < kNormSums; ++q) {
      if (!(a.sums & (1 << q))) continue;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NIT; ++i)
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (C.has(i) && C.own(i, k))
            fold[(threadIdx.x / TPR) * kRow + C.at(i) + k] = acc[q][i][k];
      __syncthreads();
      for (int c = threadIdx.x; c < C.D; c += 256) {
        float s = fold[c];
        for (int w = 1; w < RPB; ++w) s += fold[w * kRow + c];
        a.part[part_at(c, blockIdx.x, gridDim.x, q)] = s;
      }
    }
  }
}

// The workgroups' column sums in a fixed order (fp64), and the six vector gradients from them.  16
// columns per workgroup: a wave reads the four sums of one workgroup, 16 waves every 16th.
__global__ __launch_bounds__(1024) void k_norm_fold(const gnnea_norm a, int blocks) {
  __shared__ double sh[16][64];
  const int lc = threadIdx.x & 15, q = (threadIdx.x >> 4) & 3, w = wave_id();
  const int c = blockIdx.x * 16 + lc;
  const bool in = c < a.D, wb = a.w_dtype == GNNEA_BF16;
  float scale = 0.f, gate = 0.f, pw = 0.f, pb = 0.f;
  if (in && threadIdx.x < 16) {
    scale = a.alpha * vec_at(a.scale, wb, c, 1.f);
    gate = a.gate_mode == GNNEA_GATE_ROW ? vec_at(a.gate, wb, c, 0.f) : 0.f;
    pw = vec_at(a.post_w, wb, c, 1.f);
    pb = vec_at(a.post_b, wb, c, 0.f);
  }
  double s = 0.0;
  if (in && (a.sums & (1 << q))) {
    const float* p = a.part + part_at(c, 0, blocks, q);
    int b = w;
    for (; b + 112 < blocks; b += 128) {
      float v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = p[(int64_t)(b + 16 * u) * 64];
#pragma unroll
      for (int u = 0; u < 8; ++u) s += (double)v[u];
    }
    for (; b < blocks; b += 16) s += (double)p[(int64_t)b * 64];
  }
  sh[w][lane_id()] = s;
  __syncthreads();
  if (w == 0) {
    for (int k = 1; k < 16; ++k) s += sh[k][lane_id()];
    sh[0][lane_id()] = s;
  }
  __syncthreads();
  if (threadIdx.x >= 16 || !in) return;
  float got[kNormSums];
#pragma unroll
  for (int k = 0; k < kNormSums; ++k) got[k] = (float)sh[0][16 * k + lc];
  auto put = [&](void* p, float v) {
    if (!p) return;
    if (wb) ((bf16_t*)p)[c] = f32_to_bf16(v);
    else ((float*)p)[c] = v;
  };
  Gate g = {1.f, 0.f};
  if (a.gate_mode == GNNEA_GATE_ROW) g = gate_of(gate);
  // the rows' sums are over dx times an element's own gate; a shared gate comes in here
  const float both = fmaf(pw, got[0], pb * got[1]);
  put(a.dpost_w, scale * g.g * got[0]);
  put(a.dpost_b, scale * g.g * got[1]);
  put(a.dscale, a.alpha * g.g * both);
  put(a.dpre_w, got[2]);
  put(a.dpre_b, got[3]);
  if (a.gate_mode == GNNEA_GATE_ROW) put(a.dgate, scale * g.g * g.rest * both);
}

struct NormPlan { int tpr, nit, threads, blocks; };

// Threads per row: 16 lanes up to 16 chunks, a wave up to 512 values, then as many waves as leave 8
// values to a thread (the backward's twelve arrays of them fill its registers).
static NormPlan norm_plan(int64_t n, int D, int V, bool bwd) {
  const int chunks = (D + V - 1) / V, most = 8 / V;
  NormPlan p;
  p.threads = 256;
  if (chunks <= 64 * most) {
    p.tpr = chunks <= 16 ? 16 : 64;
    p.nit = (chunks + p.tpr - 1) / p.tpr;
  } else {
    p.nit = most;
    p.threads = ((chunks + most - 1) / most + 63) / 64 * 64;
    p.tpr = p.threads <= 256 ? 256 : p.threads <= 512 ? 512 : 1024;
  }
  const int rpb = p.tpr < 256 ? 256 / p.tpr : 1, waves = p.threads / 64;
  // (backward: two rows at least, so that the column sums stay few)
  const int64_t want = bwd ? (n + 2 * rpb - 1) / (2 * rpb) : (n + rpb - 1) / rpb;
  // As many workgroups as fit the chip at once, each with many rows, the next one always on its
  // way.  Where rows are many, more workgroups of 16 (backward: 128) rows a wave even the chip out:
  // 1M rows of 300 fp32, forward 1307 us with 1024 workgroups, 1264 with 4096, 1220 with 16384;
  // backward 2079 with 512, 2026 with 2048 (its column sums' fold goes from 6 to 14).
  int64_t cap = 256 * (waves <= 4 ? (bwd ? 2 : 4) : bwd ? 1 : waves <= 5 ? 4 : waves <= 10 ? 2 : 1);
  if (waves <= 4) {
    int64_t more = n / ((bwd ? 128 : 16) * rpb);
    const int64_t most = bwd ? 2048 : 16384;
    more = more < most ? more : most;
    cap = cap > more ? cap : more;
  }
  p.blocks = (int)(want < cap ? want : cap);
  return p;
}

static int64_t norm_ws(const NormPlan& p, int D) {
  return (int64_t)div_up(D, 16) * 16 * p.blocks * kNormSums * 4;
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

template <typename T, int TPR, int NIT, bool BWD>
static void norm_launch(const gnnea_norm& a, const NormPlan& p, hipStream_t s) {
  const dim3 g(p.blocks), b(p.threads);
  // (a workgroup's four sums, 16 B a value, or one sum of its rows)
  const int lds = p.threads * NIT * RowChunk<T>::V * 4 * (TPR > 64 ? kNormSums : 1);
  const int in = !a.y ? 0 : a.gate_mode == GNNEA_GATE_FULL ? 2 : 1;
  if constexpr (!BWD) {
    if (in == 0) hipLaunchKernelGGL((k_norm_fwd<T, TPR, NIT, 0>), g, b, 0, s, a);
    else if (in == 1) hipLaunchKernelGGL((k_norm_fwd<T, TPR, NIT, 1>), g, b, 0, s, a);
    else hipLaunchKernelGGL((k_norm_fwd<T, TPR, NIT, 2>), g, b, 0, s, a);
  } else if (a.post_b || (a.sums & 10)) {
    if (in == 0) hipLaunchKernelGGL((k_norm_bwd<T, TPR, NIT, 0, true>), g, b, lds, s, a);
    else if (in == 1) hipLaunchKernelGGL((k_norm_bwd<T, TPR, NIT, 1, true>), g, b, lds, s, a);
    else hipLaunchKernelGGL((k_norm_bwd<T, TPR, NIT, 2, true>), g, b, lds, s, a);
  } else {
    if (in == 0) hipLaunchKernelGGL((k_norm_bwd<T, TPR, NIT, 0, false>), g, b, lds, s, a);
    else if (in == 1) hipLaunchKernelGGL((k_norm_bwd<T, TPR, NIT, 1, false>), g, b, lds, s, a);
    else hipLaunchKernelGGL((k_norm_bwd<T, TPR, NIT, 2, false>), g, b, lds, s, a);
  }
}

template <typename T, bool BWD>
static int norm_shape(const gnnea_norm& a, const NormPlan& p, hipStream_t s) {
  bool done = false;
#define GNNEA_NORM_CASE(TPR, NIT)                 \
  if (p.tpr == TPR && p.nit == NIT) {             \
    norm_launch<T, TPR, NIT, BWD>(a, p, s);      \
    done = true;                                  \
  }
  GNNEA_NORM_CASE(16, 1)
  GNNEA_NORM_CASE(64, 1)
  constexpr int M = 8 / RowChunk<T>::V;
  if constexpr (M > 1) GNNEA_NORM_CASE(64, M)
  GNNEA_NORM_CASE(256, M)
  GNNEA_NORM_CASE(512, M)
  GNNEA_NORM_CASE(1024, M)
#undef GNNEA_NORM_CASE
  GNNEA_LAUNCH_CHECK();
  return done ? 0 : GNNEA_EINVAL;
}

template <bool BWD>
static int norm_dispatch(const gnnea_norm& a, const NormPlan& p, hipStream_t s) {
  if (a.dtype == GNNEA_F32) return norm_shape<float, BWD>(a, p, s);
  return norm_shape<bf16_t, BWD>(a, p, s);
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
  return norm_ws(norm_plan(n, D, dtype == GNNEA_F32 ? 4 : 8, true), D);
}

extern "C" int gnnea_norm_bwd(const gnnea_norm* arg, void* ws, int64_t ws_bytes, void* stream) {
  const int rc = norm_check(arg, true);
  if (rc) return rc;
  gnnea_norm a = *arg;
  a.sums = norm_sums(a);
  const NormPlan p = norm_plan(a.n, a.D, a.dtype == GNNEA_F32 ? 4 : 8, true);
  a.part = nullptr;
  if (a.sums) {
    if (ws_bytes < norm_ws(p, a.D)) return GNNEA_EWORKSPACE;
    if (p.blocks && (!ws || ((uintptr_t)ws & 15))) return ws ? GNNEA_EALIGN : GNNEA_EINVAL;
    a.part = (float*)ws;
  }
  hipStream_t s = (hipStream_t)stream;
  if (a.n > 0) {
    const int rc2 = norm_dispatch<true>(a, p, s);
    if (rc2) return rc2;
  }
  if (a.sums) {  // also for no rows: the gradients are then zero
    hipLaunchKernelGGL(k_norm_fold, dim3(div_up(a.D, 16)), dim3(1024), 0, s, a, p.blocks);
    GNNEA_LAUNCH_CHECK();
  }
  return 0;
}

// Dot-product attention over the stored entries of a CSR matrix, and its backward pass, which
// recomputes the probabilities (the reference has the additive form only,
// layers/att_layers.py:29-61):
//
//   s_ic = scale q_i . k_c,  p = exp(s - L_i),  L_i = log sum_c exp(s_ic),  o_i = sum_c p v_c
//   dp_ic = do_i . v_c,  delta_i = sum_c p dp,  ds = p (dp - delta)
//   dq_i = scale (sum p dp k - delta sum p k)          rows of the matrix, one pass over k, v
//   dk_c = scale sum_i ds q_i,  dv_c = sum_i p do_i    rows of its transpose, one pass over q, do
//
// The forward keeps a running maximum and sum (online softmax) and stores L; nothing per entry is
// ever stored.  The row pass needs no o: delta falls out of the same pass (sum p dp), in fp32.
//
// A head's row of d_head values is held by LPH lanes, NCH 16-B chunks each; a wave has 64 / LPH
// such groups, which take different heads of the same entry first (their reads are neighbours in
// memory) and different entries of the row next; the entries' partial sums meet at the end through
// cross-lane adds.  Several entries are loaded before any is computed.  The passes gather k and v
// (q and do) per entry, so they are bound by the cache that holds these tables, not by arithmetic.
//
// One wave per row.  Rows of more than `limit` entries (hubs) are cut into pieces, one wave each,
// whose partial sums a second launch joins in order; so no wave runs long after the others, and
// results do not change from run to run.
#include "rows.h"

namespace gnnea {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

struct AttnPlan { int lph, nch, hpw, units_y; };

// the 16-B chunks of a head that a lane holds
template <typename T, int LPH, int NCH> struct Lane {
  static constexpr int V = RowChunk<T>::V;
  int dh, l;
  // first element of chunk c: the last chunk of a head is moved back so that it ends with the head
  __device__ __forceinline__ int at(int c) const {
    const int e = (c * LPH + l) * V;
    return dh >= V && e > dh - V ? dh - V : e;
  }
  __device__ __forceinline__ bool has(int c) const { return (c * LPH + l) * V < dh; }
  // whether element k of chunk c is this lane's own (not one that the lane before also holds)
  __device__ __forceinline__ bool own(int c, int k) const {
    const int e = at(c) + k;
    return e >= (c * LPH + l) * V && e < dh;
  }
  __device__ __forceinline__ uint4 raw(const T* p, int c, bool ok) const {
    uint4 r = make_uint4(0, 0, 0, 0);
    if (ok && has(c)) {
      if (dh >= V) {
        r = load16<T>(p + at(c));
      } else {  // heads narrower than 16 B: element by element
        uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < V; ++k)
          if (k < dh) {
            if constexpr (V == 4) w[k] = __builtin_bit_cast(uint32_t, (float)to_f32<T>(p[k]));
            else w[k / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, p[k]) << (16 * (k & 1));
          }
        r = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    return r;
  }
  // the lane's own elements, times s; 0 elsewhere
  __device__ __forceinline__ void load_own(const T* p, bool ok, float s, float (&f)[NCH][V]) const {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      unpack16(raw(p, c, ok), f[c]);
#pragma unroll
      for (int k = 0; k < V; ++k) f[c][k] = own(c, k) ? f[c][k] * s : 0.f;
    }
  }
  template <typename O>
  __device__ __forceinline__ void store(O* p, const float (&f)[NCH][V], float s) const {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if (!has(c)) continue;
      const int e = (c * LPH + l) * V;
      float g[V];
#pragma unroll
      for (int k = 0; k < V; ++k) g[k] = f[c][k] * s;
      if constexpr (sizeof(O) == sizeof(T)) {
        if (e + V <= dh) {
          store_chunk<T, V>((T*)p + e, V, g);
          continue;
        }
      }
      const int a = at(c);
#pragma unroll
      for (int k = 0; k < V; ++k)
        if (own(c, k)) p[a + k] = from_f32<O>(g[k]);
    }
  }
};

template <int V>
__device__ __forceinline__ float dot(const float (&a)[V], const uint4& raw, float s) {
  float b[V];
  unpack16(raw, b);
#pragma unroll
  for (int k = 0; k < V; ++k) s = fmaf(a[k], b[k], s);
  return s;
}
template <int V>
__device__ __forceinline__ void axpy(float a, const uint4& raw, float (&y)[V]) {
  float b[V];
  unpack16(raw, b);
#pragma unroll
  for (int k = 0; k < V; ++k) y[k] = fmaf(a, b[k], y[k]);
}

// the sum over a group's LPH lanes, in all of them
template <int LPH>
__device__ __forceinline__ float group_sum(float v) {
  v += mov_dpp_f32<0xB1>(v);
  v += mov_dpp_f32<0x4E>(v);
  if constexpr (LPH >= 8) v += mov_dpp_f32<0x141>(v);
  if constexpr (LPH >= 16) v += mov_dpp_f32<0x140>(v);
  return v;
}

struct AttnUnit { int row, beg, end, slot; };

// The wave's row, or piece of a row (slot >= 0).  False: nothing to do.
__device__ __forceinline__ bool attn_unit(const gnnea_attn& a, bool pieces, AttnUnit& u) {
  const int id = blockIdx.x * 4 + wave_id();
  if (pieces) {
    if (id >= a.n_items) return false;
    const int4 it = ((const int4*)a.items)[id];
    u.row = it.x; u.beg = it.y; u.end = it.z; u.slot = it.w;
    return true;
  }
  if (id >= a.n_rows) return false;
  u.row = id; u.beg = a.rowptr[id]; u.end = a.rowptr[id + 1]; u.slot = -1;
  return a.limit == 0 || u.end - u.beg <= a.limit;
}

template <int NCH> struct Steps { static constexpr int U = NCH == 1 ? 4 : 2; };

template <typename T, int LPH, int NCH>
__global__ __launch_bounds__(256) void k_attn_fwd(const gnnea_attn a, int hpw, bool pieces,
                                                  float* __restrict__ ws) {
  constexpr int V = RowChunk<T>::V, G = 64 / LPH, U = Steps<NCH>::U;
  AttnUnit u;
  if (!attn_unit(a, pieces, u)) return;
  const int lane = lane_id(), grp = lane / LPH, dh = a.d_head;
  const Lane<T, LPH, NCH> L{dh, lane % LPH};
  const int head = blockIdx.y * hpw + grp % hpw, slot = grp / hpw, eps = G / hpw;
  const bool on = head < a.heads;
  const int64_t kvo = (int64_t)(on ? head / (a.heads / a.kv_heads) : 0) * dh;
  const T* K = (const T*)a.k + kvo;
  const T* Vp = (const T*)a.v + kvo;
  float q[NCH][V], o[NCH][V], m = -INFINITY, sum = 0.f;
  L.load_own((const T*)a.q + u.row * a.ldq + (int64_t)head * dh, on, a.scale * kLog2e, q);
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int k = 0; k < V; ++k) o[c][k] = 0.f;
  for (int b = u.beg; b < u.end; b += eps * U) {
    uint4 rk[U][NCH], rv[U][NCH];
    bool ok[U];
#pragma unroll
    for (int s = 0; s < U; ++s) {
      const int e = b + s * eps + slot;
      ok[s] = on && e < u.end;
      const int64_t j = ok[s] ? a.col[e] : 0;
#pragma unroll
      for (int c = 0; c < NCH; ++c) rk[s][c] = L.raw(K + j * a.ldk, c, ok[s]);
#pragma unroll
      for (int c = 0; c < NCH; ++c) rv[s][c] = L.raw(Vp + j * a.ldv, c, ok[s]);
    }
    float x[U], top = m;
#pragma unroll
    for (int s = 0; s < U; ++s) {
      float d = 0.f;
#pragma unroll
      for (int c = 0; c < NCH; ++c) d = dot<V>(q[c], rk[s][c], d);
      d = group_sum<LPH>(d);
      x[s] = ok[s] ? d : -INFINITY;
      top = x[s] > top || x[s] != x[s] ? x[s] : top;
    }
    const float ref = top == -INFINITY ? 0.f : top;  // nothing but -inf so far: all weights 0
    const float keep = __builtin_amdgcn_exp2f(m - ref);
    m = top;
    sum *= keep;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int k = 0; k < V; ++k) o[c][k] *= keep;
#pragma unroll
    for (int s = 0; s < U; ++s) {
      const float p = __builtin_amdgcn_exp2f(x[s] - ref);
      sum += p;
#pragma unroll
      for (int c = 0; c < NCH; ++c) axpy<V>(p, rv[s][c], o[c]);
    }
  }
  for (int w = LPH * hpw; w < 64; w <<= 1) {  // the groups of one head
    const float mo = __shfl_xor(m, w, 64), so = __shfl_xor(sum, w, 64);
    const float top = mo > m || mo != mo ? mo : m;
    const float ref = top == -INFINITY ? 0.f : top;
    const float ka = __builtin_amdgcn_exp2f(m - ref), kb = __builtin_amdgcn_exp2f(mo - ref);
    m = top;
    sum = sum * ka + so * kb;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int k = 0; k < V; ++k) o[c][k] = o[c][k] * ka + __shfl_xor(o[c][k], w, 64) * kb;
  }
  if (slot != 0 || !on) return;
  if (pieces) {
    float* part = ws + ((int64_t)u.slot * a.heads + head) * (dh + 2);
    if (L.l == 0) part[0] = m, part[1] = sum;
    L.store(part + 2, o, 1.f);
    return;
  }
  L.store((T*)a.o + u.row * a.ldo + (int64_t)head * dh, o, sum == 0.f ? 0.f : 1.f / sum);
  if (a.lse && L.l == 0)
    a.lse[(int64_t)u.row * a.heads + head] = sum == 0.f ? -INFINITY : fmaf(m, kLn2, logf(sum));
}

template <typename T, int LPH, int NCH>
__global__ __launch_bounds__(256) void k_attn_rows(const gnnea_attn a, int hpw, bool pieces,
                                                   float* __restrict__ ws) {
  constexpr int V = RowChunk<T>::V, G = 64 / LPH, U = Steps<NCH>::U;
  AttnUnit u;
  if (!attn_unit(a, pieces, u)) return;
  const int lane = lane_id(), grp = lane / LPH, dh = a.d_head;
  const Lane<T, LPH, NCH> L{dh, lane % LPH};
  const int head = blockIdx.y * hpw + grp % hpw, slot = grp / hpw, eps = G / hpw;
  const bool on = head < a.heads;
  const int64_t kvo = (int64_t)(on ? head / (a.heads / a.kv_heads) : 0) * dh;
  const T* K = (const T*)a.k + kvo;
  const T* Vp = (const T*)a.v + kvo;
  float q[NCH][V], d[NCH][V], A[NCH][V], B[NCH][V], delta = 0.f;
  L.load_own((const T*)a.q + u.row * a.ldq + (int64_t)head * dh, on, a.scale * kLog2e, q);
  L.load_own((const T*)a.dout + u.row * a.lddo + (int64_t)head * dh, on, 1.f, d);
  const float lse = on ? a.lse[(int64_t)u.row * a.heads + head] * kLog2e : 0.f;
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int k = 0; k < V; ++k) A[c][k] = B[c][k] = 0.f;
  for (int b = u.beg; b < u.end; b += eps * U) {
    uint4 rk[U][NCH], rv[U][NCH];
    bool ok[U];
#pragma unroll
    for (int s = 0; s < U; ++s) {
      const int e = b + s * eps + slot;
      ok[s] = on && e < u.end;
      const int64_t j = ok[s] ? a.col[e] : 0;
#pragma unroll
      for (int c = 0; c < NCH; ++c) rk[s][c] = L.raw(K + j * a.ldk, c, ok[s]);
#pragma unroll
      for (int c = 0; c < NCH; ++c) rv[s][c] = L.raw(Vp + j * a.ldv, c, ok[s]);
    }
#pragma unroll
    for (int s = 0; s < U; ++s) {
      float x = 0.f, y = 0.f;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        x = dot<V>(q[c], rk[s][c], x);
        y = dot<V>(d[c], rv[s][c], y);
      }
      x = group_sum<LPH>(x);
      y = group_sum<LPH>(y);
      // a row whose scores are all -inf has no weights (lse = -inf), like one without entries
      const float p = ok[s] && lse != -INFINITY ? __builtin_amdgcn_exp2f(x - lse) : 0.f;
      const float pd = ok[s] ? p * y : 0.f;
      delta += pd;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        axpy<V>(pd, rk[s][c], A[c]);
        axpy<V>(p, rk[s][c], B[c]);
      }
    }
  }
  for (int w = LPH * hpw; w < 64; w <<= 1) {
    delta += __shfl_xor(delta, w, 64);
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        A[c][k] += __shfl_xor(A[c][k], w, 64);
        B[c][k] += __shfl_xor(B[c][k], w, 64);
      }
  }
  if (slot != 0 || !on) return;
  if (pieces) {
    float* part = ws + ((int64_t)u.slot * a.heads + head) * (2 * dh + 1);
    if (L.l == 0) part[0] = delta;
    L.store(part + 1, A, 1.f);
    L.store(part + 1 + dh, B, 1.f);
    return;
  }
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int k = 0; k < V; ++k) A[c][k] = fmaf(-delta, B[c][k], A[c][k]);
  L.store((T*)a.dq + u.row * a.lddq + (int64_t)head * dh, A, a.scale);
  if (L.l == 0)
    *(float2*)(a.stat + 2 * ((int64_t)u.row * a.heads + head)) = make_float2(lse, delta);
}

// Columns: a row of the transposed matrix per wave; groups take key/value heads, then (entry,
// query head of the group) pairs.
template <typename T, int LPH, int NCH>
__global__ __launch_bounds__(256) void k_attn_cols(const gnnea_attn a, int hpw, bool pieces,
                                                   float* __restrict__ ws) {
  constexpr int V = RowChunk<T>::V, G = 64 / LPH, U = Steps<NCH>::U;
  AttnUnit u;
  if (!attn_unit(a, pieces, u)) return;
  const int lane = lane_id(), grp = lane / LPH, dh = a.d_head;
  const Lane<T, LPH, NCH> L{dh, lane % LPH};
  const int kvh = blockIdx.y * hpw + grp % hpw, slot = grp / hpw, pps = G / hpw;
  const bool on = kvh < a.kv_heads;
  const int share = a.heads / a.kv_heads;
  float kf[NCH][V], vf[NCH][V], dk[NCH][V], dv[NCH][V];
  L.load_own((const T*)a.k + u.row * a.ldk + (int64_t)kvh * dh, on, a.scale * kLog2e, kf);
  L.load_own((const T*)a.v + u.row * a.ldv + (int64_t)kvh * dh, on, 1.f, vf);
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int k = 0; k < V; ++k) dk[c][k] = dv[c][k] = 0.f;
  const int64_t pairs = (int64_t)(u.end - u.beg) * share;
  for (int64_t b = 0; b < pairs; b += pps * U) {
    uint4 rq[U][NCH], rd[U][NCH];
    float2 st[U];
    bool ok[U];
#pragma unroll
    for (int s = 0; s < U; ++s) {
      const int64_t t = b + s * pps + slot;
      ok[s] = on && t < pairs;
      const uint32_t e = share == 1 ? (uint32_t)t : (uint32_t)((uint64_t)t / (uint32_t)share);
      const int h = kvh * share + (int)(t - (int64_t)e * share);
      const int64_t i = ok[s] ? a.col[u.beg + (int)e] : 0;
      st[s] = ok[s] ? *(const float2*)(a.stat + 2 * (i * a.heads + h)) : make_float2(0.f, 0.f);
#pragma unroll
      for (int c = 0; c < NCH; ++c)
        rq[s][c] = L.raw((const T*)a.q + i * a.ldq + (int64_t)h * dh, c, ok[s]);
#pragma unroll
      for (int c = 0; c < NCH; ++c)
        rd[s][c] = L.raw((const T*)a.dout + i * a.lddo + (int64_t)h * dh, c, ok[s]);
    }
#pragma unroll
    for (int s = 0; s < U; ++s) {
      float x = 0.f, y = 0.f;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        x = dot<V>(kf[c], rq[s][c], x);
        y = dot<V>(vf[c], rd[s][c], y);
      }
      x = group_sum<LPH>(x);
      y = group_sum<LPH>(y);
      const float p = ok[s] && st[s].x != -INFINITY ? __builtin_amdgcn_exp2f(x - st[s].x) : 0.f;
      const float ds = ok[s] ? p * (y - st[s].y) : 0.f;
#pragma unroll
      for (int c = 0; c < NCH; ++c) {
        axpy<V>(ds, rq[s][c], dk[c]);
        axpy<V>(p, rd[s][c], dv[c]);
      }
    }
  }
  for (int w = LPH * hpw; w < 64; w <<= 1) {
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        dk[c][k] += __shfl_xor(dk[c][k], w, 64);
        dv[c][k] += __shfl_xor(dv[c][k], w, 64);
      }
  }
  if (slot != 0 || !on) return;
  if (pieces) {
    float* part = ws + ((int64_t)u.slot * a.kv_heads + kvh) * (2 * dh);
    L.store(part, dk, 1.f);
    L.store(part + dh, dv, 1.f);
    return;
  }
  L.store((T*)a.dk + u.row * a.lddk + (int64_t)kvh * dh, dk, a.scale);
  L.store((T*)a.dv + u.row * a.lddv + (int64_t)kvh * dh, dv, 1.f);
}

// Joins the pieces of a long row in order: one wave per row and head, a lane per four columns.
template <typename T>
__global__ __launch_bounds__(64) void k_attn_join(const gnnea_attn a, int pass,
                                                  const float* __restrict__ ws) {
  const int w = blockIdx.x, h = blockIdx.y, dh = a.d_head, row = a.long_rows[w];
  const int s0 = a.long_ptr[w], s1 = a.long_ptr[w + 1];
  const int heads = pass == GNNEA_ATTN_BWD_COLS ? a.kv_heads : a.heads;
  const int wide = pass == GNNEA_ATTN_FWD ? dh + 2 : pass == GNNEA_ATTN_BWD_ROWS ? 2 * dh + 1 : 2 * dh;
  const float* part = ws + ((int64_t)s0 * heads + h) * wide;
  const int64_t step = (int64_t)heads * wide;
  const int n = s1 - s0;
  if (pass == GNNEA_ATTN_FWD) {
    float m = -INFINITY, sum = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < n; ++s) {
      const float x = part[s * step];
      m = x > m || x != x ? x : m;
    }
    const float ref = m == -INFINITY ? 0.f : m;
    for (int s = 0; s < n; ++s) {
      const float f = __builtin_amdgcn_exp2f(part[s * step] - ref);
      sum = fmaf(part[s * step + 1], f, sum);
#pragma unroll
      for (int c = 0; c < 4; ++c)
        if (c * 64 + (int)threadIdx.x < dh)
          o[c] = fmaf(part[s * step + 2 + c * 64 + threadIdx.x], f, o[c]);
    }
    const float r = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (c * 64 + (int)threadIdx.x < dh)
        ((T*)a.o)[row * a.ldo + (int64_t)h * dh + c * 64 + threadIdx.x] = from_f32<T>(o[c] * r);
    if (a.lse && threadIdx.x == 0)
      a.lse[(int64_t)row * a.heads + h] = sum == 0.f ? -INFINITY : fmaf(m, kLn2, logf(sum));
    return;
  }
  const bool rows = pass == GNNEA_ATTN_BWD_ROWS;
  float delta = 0.f, A[4] = {0.f, 0.f, 0.f, 0.f}, B[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < n; ++s) {
    const float* p = part + s * step;
    if (rows) delta += *p++;
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (c * 64 + (int)threadIdx.x < dh) {
        A[c] += p[c * 64 + threadIdx.x];
        B[c] += p[dh + c * 64 + threadIdx.x];
      }
  }
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int d = c * 64 + threadIdx.x;
    if (d >= dh) continue;
    if (rows) {
      ((T*)a.dq)[row * a.lddq + (int64_t)h * dh + d] = from_f32<T>(a.scale * fmaf(-delta, B[c], A[c]));
    } else {
      ((T*)a.dk)[row * a.lddk + (int64_t)h * dh + d] = from_f32<T>(a.scale * A[c]);
      ((T*)a.dv)[row * a.lddv + (int64_t)h * dh + d] = from_f32<T>(B[c]);
    }
  }
  if (rows && threadIdx.x == 0)
    *(float2*)(a.stat + 2 * ((int64_t)row * a.heads + h)) =
        make_float2(a.lse[(int64_t)row * a.heads + h] * kLog2e, delta);
}

static int attn_check(const gnnea_attn* a, int pass) {
  if (!a || a->n_rows < 0 || a->n_cols < 0) return GNNEA_EINVAL;
  if (a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads) return GNNEA_EINVAL;
  if (a->heads > 65535 || a->d_head < 1 || a->d_head > 256) return GNNEA_EINVAL;
  if (a->dtype != GNNEA_F32 && a->dtype != GNNEA_BF16) return GNNEA_EINVAL;
  if (!(a->scale == a->scale) || a->limit < 0 || a->n_items < 0 || a->n_long < 0) return GNNEA_EINVAL;
  if (a->n_items && (!a->items || !a->long_rows || !a->long_ptr || !a->n_long || !a->limit))
    return GNNEA_EINVAL;
  if (a->items && ((uintptr_t)a->items & 15)) return GNNEA_EALIGN;
  if (a->n_rows == 0) return GNNEA_OK;
  if (!a->rowptr) return GNNEA_EINVAL;
  const int64_t wq = (int64_t)a->heads * a->d_head, wk = (int64_t)a->kv_heads * a->d_head;
  const bool cols = pass == GNNEA_ATTN_BWD_COLS;
  // a matrix without columns has no entries: col, and the tables indexed by it, may be absent
  if (a->n_cols > 0 && !a->col) return GNNEA_EINVAL;
  if ((!a->q && (!cols || a->n_cols)) || a->ldq < wq) return GNNEA_EINVAL;
  if (((!a->k || !a->v) && (cols || a->n_cols)) || a->ldk < wk || a->ldv < wk) return GNNEA_EINVAL;
  if (pass == GNNEA_ATTN_FWD) {
    if (!a->o || a->ldo < wq) return GNNEA_EINVAL;
    return GNNEA_OK;
  }
  if ((!a->dout && (!cols || a->n_cols)) || a->lddo < wq) return GNNEA_EINVAL;
  if (!a->stat && (!cols || a->n_cols)) return GNNEA_EINVAL;
  if ((uintptr_t)a->stat & 7) return GNNEA_EALIGN;
  if (!cols && (!a->lse || !a->dq || a->lddq < wq)) return GNNEA_EINVAL;
  if (cols && (!a->dk || !a->dv || a->lddk < wk || a->lddv < wk)) return GNNEA_EINVAL;
  return GNNEA_OK;
}

// Lanes and chunks of a head: the fewest lanes that leave at most 3 chunks each (fewer cross-lane
// adds per score, more entries per wave), 16 lanes for wide heads.
static AttnPlan attn_plan(const gnnea_attn* a, int pass) {
  static const int kShape[7][2] = {{4, 1}, {8, 1}, {8, 2}, {8, 3}, {16, 2}, {16, 3}, {16, 4}};
  const int V = a->dtype == GNNEA_F32 ? 4 : 8;
  AttnPlan p = {16, 4, 1, 1};
  for (const auto& s : kShape)
    if (s[0] * s[1] * V >= a->d_head) {
      p.lph = s[0];
      p.nch = s[1];
      break;
    }
  const int heads = pass == GNNEA_ATTN_BWD_COLS ? a->kv_heads : a->heads;
  while (p.hpw < heads && p.hpw < 64 / p.lph) p.hpw *= 2;
  p.units_y = (heads + p.hpw - 1) / p.hpw;
  return p;
}

template <typename T, int LPH, int NCH>
static void attn_launch(const gnnea_attn& a, int pass, const AttnPlan& p, bool pieces, float* ws,
                        hipStream_t s) {
  const dim3 grid(div_up(pieces ? a.n_items : a.n_rows, 4), p.units_y);
  if (pass == GNNEA_ATTN_FWD)
    hipLaunchKernelGGL((k_attn_fwd<T, LPH, NCH>), grid, dim3(256), 0, s, a, p.hpw, pieces, ws);
  else if (pass == GNNEA_ATTN_BWD_ROWS)
    hipLaunchKernelGGL((k_attn_rows<T, LPH, NCH>), grid, dim3(256), 0, s, a, p.hpw, pieces, ws);
  else
    hipLaunchKernelGGL((k_attn_cols<T, LPH, NCH>), grid, dim3(256), 0, s, a, p.hpw, pieces, ws);
}

template <typename T>
static void attn_dispatch(const gnnea_attn& a, int pass, bool pieces, float* ws, hipStream_t s) {
  const AttnPlan p = attn_plan(&a, pass);
  if (p.lph == 4) attn_launch<T, 4, 1>(a, pass, p, pieces, ws, s);
  else if (p.lph == 8 && p.nch == 1) attn_launch<T, 8, 1>(a, pass, p, pieces, ws, s);
  else if (p.lph == 8 && p.nch == 2) attn_launch<T, 8, 2>(a, pass, p, pieces, ws, s);
  else if (p.lph == 8) attn_launch<T, 8, 3>(a, pass, p, pieces, ws, s);
  else if (p.nch == 2) attn_launch<T, 16, 2>(a, pass, p, pieces, ws, s);
  else if constexpr (sizeof(T) == 4) {  // bf16 heads of 256 fit two chunks
    if (p.nch == 3) attn_launch<T, 16, 3>(a, pass, p, pieces, ws, s);
    else attn_launch<T, 16, 4>(a, pass, p, pieces, ws, s);
  }
}

static int64_t attn_ws(const gnnea_attn* a, int pass) {
  const int64_t dh = a->d_head;
  if (pass == GNNEA_ATTN_FWD) return (int64_t)a->n_items * a->heads * (dh + 2) * 4;
  if (pass == GNNEA_ATTN_BWD_ROWS) return (int64_t)a->n_items * a->heads * (2 * dh + 1) * 4;
  return (int64_t)a->n_items * a->kv_heads * 2 * dh * 4;
}

static int attn_run(const gnnea_attn* a, int pass, void* ws, int64_t ws_bytes, void* stream) {
  const int rc = attn_check(a, pass);
  if (rc || a->n_rows == 0) return rc;
  if (ws_bytes < attn_ws(a, pass)) return GNNEA_EWORKSPACE;
  if (a->n_items && (!ws || ((uintptr_t)ws & 15))) return ws ? GNNEA_EALIGN : GNNEA_EINVAL;
  const hipStream_t s = (hipStream_t)stream;
  for (int pieces = 0; pieces < (a->n_items ? 2 : 1); ++pieces) {
    if (a->dtype == GNNEA_F32) attn_dispatch<float>(*a, pass, pieces, (float*)ws, s);
    else attn_dispatch<bf16_t>(*a, pass, pieces, (float*)ws, s);
    GNNEA_LAUNCH_CHECK();
  }
  if (a->n_items) {
    const dim3 grid(a->n_long, pass == GNNEA_ATTN_BWD_COLS ? a->kv_heads : a->heads);
    if (a->dtype == GNNEA_F32)
      hipLaunchKernelGGL(k_attn_join<float>, grid, dim3(64), 0, s, *a, pass, (const float*)ws);
    else
      hipLaunchKernelGGL(k_attn_join<bf16_t>, grid, dim3(64), 0, s, *a, pass, (const float*)ws);
    GNNEA_LAUNCH_CHECK();
  }
  return 0;
}

}  // namespace gnnea

using namespace gnnea;

extern "C" int64_t gnnea_attn_ws_bytes(const gnnea_attn* a, int pass) {
  if (!a || pass < GNNEA_ATTN_FWD || pass > GNNEA_ATTN_BWD_COLS || a->n_items < 0 ||
      a->heads < 1 || a->kv_heads < 1 || a->d_head < 1 || a->d_head > 256)
    return GNNEA_EINVAL;
  return attn_ws(a, pass);
}
extern "C" int gnnea_attn_fwd(const gnnea_attn* a, void* ws, int64_t ws_bytes, void* stream) {
  return attn_run(a, GNNEA_ATTN_FWD, ws, ws_bytes, stream);
}
extern "C" int gnnea_attn_bwd_rows(const gnnea_attn* a, void* ws, int64_t ws_bytes, void* stream) {
  return attn_run(a, GNNEA_ATTN_BWD_ROWS, ws, ws_bytes, stream);
}
extern "C" int gnnea_attn_bwd_cols(const gnnea_attn* a, void* ws, int64_t ws_bytes, void* stream) {
  return attn_run(a, GNNEA_ATTN_BWD_COLS, ws, ws_bytes, stream);
}

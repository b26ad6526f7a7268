// Dot-product attention over the stored entries of a CSR matrix, and its backward pass, which
// recomputes the probabilities (the reference has the additive form only,
// layers/att_layers.py:29-61):
//
//   s_ic = scale q_i . k_c,  p = exp(s - L_i),  L_i = log sum_c exp(s_ic),  o_i = sum_c p v_c
//   dp_ic = do_i . v_c,  delta_i = sum_c p dp,  ds = p (dp - delta)
//   dq_i = scale (sum p (dp - c) k - e sum p k),  e = sum p (dp - c),  delta = c + e
//                                                      rows of the matrix, one pass over k, v
//   dk_c = scale sum_i ds q_i,  dv_c = sum_i p do_i    rows of its transpose, one pass over q, do
//
// The forward keeps a running maximum and sum (online softmax) and stores L; nothing per entry is
// ever stored.  The row pass needs no o: delta falls out of the same pass, in fp32.
//
// c: the dp of one of the row's entries.  What all dp of a row have in common passes no gradient,
// but summed into both terms of dq it would leave their rounding; less c, a row of one entry, or
// of equal values, gives 0 exactly (and so do its terms of dk, whose ds subtracts the same dp).
// A c far from the others would do harm of its own, so it moves to an entry of over 64 times the
// weight of its own: p |c| then stays within 64 times the largest p |dp| met.
//
// A head's row of d_head values is held by LPH lanes, NCH 16-B chunks each; a wave has 64 / LPH
// such groups, which take different heads of the same entry first (their reads are neighbours in
// memory) and different entries of the row next; the entries' partial sums meet at the end through
// cross-lane adds.  Few lanes per head mean few adds per score and many entries per wave.  bf16
// scores multiply pairs at once; weights and sums are fp32 throughout.
//
// The passes gather k and v (q and do) per entry.  Where a head is read by itself the cache that
// holds the tables bounds them: 9.5M entries, 4 heads of 64 bf16, forward 1.23 ms (7.9 TB/s of
// gathered bytes, as much as the aggregation kernels of this library reach); 290k entries, 4 heads
// of 75 fp32: forward 93 us, row pass 108, column pass 120 (7.5, 6.4, 5.8 TB/s).  Where 4 query
// heads share a key head, instructions do: 3.3M entries, 8 heads of 32 bf16 on 2: 211 us forward,
// 313 rows (569 and 796 vector instructions a wave, 16 entries each: every query head has lanes of
// its own, which load and unpack the shared key and value again), while the column pass, which reads
// every query head, gathers again (460 us, 7.7 TB/s).
//
// One wave per row.  Rows of more than `limit` entries (hubs) are cut into pieces, one wave each,
// whose partial sums a second launch joins in order; so no wave runs long after the others, and
// results do not change from run to run.
#include "rows.h"

namespace gnnea {

constexpr float kLog2e = 1.44269504088896340736f;

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// hs: log2 of the heads that a wave's groups take at once; share: query heads per key/value head,
// ss: its log2 where it has one, else -1; row0, items: the launch's first row, and its pieces
struct AttnPlan { int lph, nch, hs, share, ss, units_y; bool full; };
struct AttnShape { int hs, share, ss, row0, items; };
// Rows of one launch: 64 work-items each, which have to stay below 2^32 in all.
constexpr int kAttnRows = 1 << 25;
__device__ __forceinline__ int by_share(const AttnShape& p, int x) {
  return p.ss >= 0 ? x >> p.ss : (int)((uint32_t)x / (uint32_t)p.share);
}

// The 16-B chunks of a head that a lane holds: NCH of them, LPH lanes apart.  FULL: d_head is
// LPH NCH V.  Otherwise a head's last chunk is moved back so that it ends with the head, and holds
// values of the lane before first; lanes past it hold none.
template <typename T, int LPH, int NCH, bool FULL> struct Lane {
  static constexpr int V = RowChunk<T>::V;
  int dh, l;
  __device__ __forceinline__ int first(int c) const { return (c * LPH + l) * V; }
  __device__ __forceinline__ int at(int c) const {
    const int e = first(c);
    if (FULL || c < NCH - 1) return e;
    return dh >= V ? (e > dh - V ? dh - V : e) : 0;
  }
  __device__ __forceinline__ bool has(int c) const { return FULL || c < NCH - 1 || first(c) < dh; }
  // whether value k of chunk c is the lane's own
  __device__ __forceinline__ bool own(int c, int k) const {
    if (FULL || c < NCH - 1) return true;
    const int e = at(c) + k;
    return has(c) && e >= first(c) && e < dh;
  }
  // chunk c of the head at p; 0 for lanes without one
  __device__ __forceinline__ uint4 raw(const T* p, int c) const {
    if constexpr (FULL) return load16<T>(p + first(c));
    uint32_t w[4] = {0, 0, 0, 0};
    if (has(c)) {
      if (dh >= V) return load16<T>(p + at(c));
#pragma unroll
      for (int k = 0; k < V; ++k)  // heads narrower than 16 B: element by element
        if (k < dh) {
          if constexpr (V == 4) w[k] = __builtin_bit_cast(uint32_t, (float)to_f32<T>(p[k]));
          else w[k / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, p[k]) << (16 * (k & 1));
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  // r with 0 in the places that are not the lane's own (ok: in all)
  __device__ __forceinline__ uint4 mask(const uint4& r, int c, bool ok) const {
    uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (!ok || !own(c, k)) w[k * 4 / V] &= V == 4 ? 0u : (k & 1) ? 0xffffu : 0xffff0000u;
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ void load_own(const T* p, bool ok, uint4 (&f)[NCH]) const {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      f[c] = make_uint4(0, 0, 0, 0);
      if (ok) f[c] = FULL || c < NCH - 1 ? raw(p, c) : mask(raw(p, c), c, true);
    }
  }
  template <typename O>
  __device__ __forceinline__ void store(O* p, const float (&f)[NCH][V], float s) const {
#pragma unroll
    for (int c = 0; c < NCH; ++c) {
      if (!has(c)) continue;
      float g[V];
#pragma unroll
      for (int k = 0; k < V; ++k) g[k] = f[c][k] * s;
      if constexpr (sizeof(O) == sizeof(T)) {
        if (FULL || first(c) + V <= dh) {
          store_chunk<T, V>((T*)p + first(c), V, g);
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

// the sum over a group's LPH lanes, in all of them
template <int LPH>
__device__ __forceinline__ float group_sum(float v) {
  v += mov_dpp_f32<0xB1>(v);
  v += mov_dpp_f32<0x4E>(v);
  if constexpr (LPH >= 8) v += mov_dpp_f32<0x141>(v);
  if constexpr (LPH >= 16) v += mov_dpp_f32<0x140>(v);
  return v;
}

// the value of lane ^ w (w a power of two; 32, 16 and 8 without LDS)
__device__ __forceinline__ float lane_xor(float v, int w) {
  const uint32_t x = __builtin_bit_cast(uint32_t, v);
  if (w == 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return __builtin_bit_cast(float, lane_id() < 32 ? r[1] : r[0]);
  }
  if (w == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    return __builtin_bit_cast(float, (lane_id() & 16) == 0 ? r[1] : r[0]);
  }
  if (w == 8) return mov_dpp_f32<0x128>(v);  // row_ror:8
  return __shfl_xor(v, w, 64);
}

// The products of a head's fp32 values, or of its bf16 pairs (each exact), summed over the group.
template <int V, int LPH, int NCH>
__device__ __forceinline__ float head_dot(const uint4 (&a)[NCH], const uint4 (&b)[NCH]) {
  float s = 0.f;
#pragma unroll
  for (int c = 0; c < NCH; ++c) {
    const uint32_t x[4] = {a[c].x, a[c].y, a[c].z, a[c].w}, y[4] = {b[c].x, b[c].y, b[c].z, b[c].w};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (V == 4)
        s = fmaf(__builtin_bit_cast(float, x[k]), __builtin_bit_cast(float, y[k]), s);
      else
        s = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, x[k]),
                                            __builtin_bit_cast(bf16x2, y[k]), s, false);
    }
  }
  return group_sum<LPH>(s);
}
template <int V>
__device__ __forceinline__ void axpy(float a, const uint4& raw, float (&y)[V]) {
  float b[V];
  unpack16(raw, b);
#pragma unroll
  for (int k = 0; k < V; ++k) y[k] = fmaf(a, b[k], y[k]);
}
// + 0 times the values: NaN where one of them is not finite
template <int NCH, int V>
__device__ __forceinline__ float zero_of(const float (&f)[NCH][V], float s) {
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int k = 0; k < V; ++k) s = fmaf(f[c][k], 0.f, s);
  return s;
}
template <int NCH, int V>
__device__ __forceinline__ void clear(float (&f)[NCH][V]) {
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int k = 0; k < V; ++k) f[c][k] = 0.f;
}

struct AttnUnit { int row, beg, end, slot; };

// The wave's piece of a long row (their workgroups come first: they run longest), or its row (slot
// < 0).  Consecutive rows share an XCD: neighbours in the ring of entities share keys, and rows
// that are not whole cache lines share lines.  False: nothing to do.
__device__ __forceinline__ bool attn_unit(const gnnea_attn& a, const AttnShape& S, AttnUnit& u) {
  const int pb = (S.items + 3) / 4, b = blockIdx.x;
  if (b < pb) {
    const int id = b * 4 + wave_id();
    if (id >= S.items) return false;
    const int4 it = ((const int4*)a.items)[id];
    u.row = it.x; u.beg = it.y; u.end = it.z; u.slot = it.w;
    return true;
  }
  const uint32_t at = (uint32_t)xcd_remap(b - pb, (int)gridDim.x - pb) * 4 + wave_id();
  const uint32_t id = (uint32_t)S.row0 + at;
  if (id >= (uint32_t)a.n_rows) return false;
  u.row = (int)id; u.beg = a.rowptr[id]; u.end = a.rowptr[id + 1]; u.slot = -1;
  return a.n_items == 0 || u.end - u.beg <= a.limit;
}

// Entries that a group loads before it computes any.  More in flight per wave cost registers, and
// with them waves: at 290k entries, 4 heads of 75 fp32 (three chunks) the row pass takes 107, 115
// and 144 us with 1, 2 and 3, the column pass 119, 128 and 163; at 3.3M entries, 8 heads of 32 bf16
// (one chunk) the three passes take 1053, 1014 and 1164 us with 1, 2 and 4.
template <int NCH> struct Steps { static constexpr int U = NCH <= 2 ? 2 : 1; };

// The next 64 columns of the unit's entries, one per lane, read while the current ones are used.
// Lanes past the end repeat the last entry: what is read for them is the row's own, and weighs 0.
struct ColBatch {
  const int32_t* col;  // the unit's first
  int total, now, next, left;
  __device__ __forceinline__ ColBatch(const gnnea_attn& a, const AttnUnit& u)
      : col(a.col + u.beg), total(u.end - u.beg), now(0), next(0), left(0) {
    if (total > 0) next = col[min(lane_id(), total - 1)];
  }
  __device__ __forceinline__ void step(uint32_t done) {
    now = next;
    const int rest = total - (int)done;
    left = min(rest, 64);
    if (rest > 64) next = col[(int64_t)done + min(64 + lane_id(), rest - 1)];
  }
};

// The row offsets (in elements) of a lane's column in a table, formed once per 64 entries and
// handed to the group that reads the entry; the high words only where a table has them.
struct RowOffset {
  uint32_t lo, hi;
  bool wide;
  __device__ __forceinline__ RowOffset(int32_t rows, int64_t ld) : lo(0), hi(0) {
    wide = (int64_t)rows * ld > 0xffffffffll;
  }
  __device__ __forceinline__ void set(int col, int64_t ld) {
    const uint64_t o = (uint64_t)(uint32_t)col * (uint64_t)ld;
    lo = (uint32_t)o;
    hi = (uint32_t)(o >> 32);
  }
  __device__ __forceinline__ uint64_t of(int lane) const {
    uint64_t o = (uint32_t)__shfl((int)lo, lane, 64);
    if (wide) o |= (uint64_t)(uint32_t)__shfl((int)hi, lane, 64) << 32;
    return o;
  }
};

// A lane's row of scores: keys and values of U entries at a time.  `care`: a second run of a unit
// whose sums came out not finite, with 0 in every place that is not an entry's own (0 times an
// infinity read for nothing is not 0).
template <typename T, int LPH, int NCH, bool FULL>
__global__ __launch_bounds__(256) void k_attn_fwd(const gnnea_attn a, const AttnShape S,
                                                  float* __restrict__ ws) {
  constexpr int V = RowChunk<T>::V, G = 64 / LPH, U = Steps<NCH>::U;
  AttnUnit u;
  if (!attn_unit(a, S, u)) return;
  const int lane = lane_id(), grp = lane / LPH, dh = a.d_head;
  const Lane<T, LPH, NCH, FULL> L{dh, lane % LPH};
  const int head = (blockIdx.y << S.hs) + (grp & ((1 << S.hs) - 1)), slot = grp >> S.hs, eps = G >> S.hs;
  const bool on = head < a.heads;
  const int64_t kvo = (int64_t)(on ? by_share(S, head) : 0) * dh;
  const T* K = (const T*)a.k + kvo;
  const T* Vp = (const T*)a.v + kvo;
  const float factor = a.scale * kLog2e;
  uint4 q[NCH];
  float o[NCH][V], m, sum;
  for (bool care = false;; care = true) {
    ColBatch cb(a, u);
    RowOffset off(a.n_cols, a.ldk);
    L.load_own((const T*)a.q + u.row * a.ldq + (int64_t)head * dh, on, q);
    m = -INFINITY;
    sum = 0.f;
    clear(o);
    for (uint32_t done = 0; done < (uint32_t)cb.total; done += 64) {
      cb.step(done);
      off.set(cb.now, a.ldk);
      for (int b = 0; b < cb.left; b += eps * U) {
        uint4 rk[U][NCH], rv[U][NCH];
        bool ok[U];
#pragma unroll
        for (int s = 0; s < U; ++s) {
          const int e = b + s * eps + slot;
          ok[s] = on && e < cb.left;
          const uint64_t j = off.of(min(e, 63));
#pragma unroll
          for (int c = 0; c < NCH; ++c) rk[s][c] = L.raw(K + j, c);
#pragma unroll
          for (int c = 0; c < NCH; ++c) rv[s][c] = L.raw(Vp + j, c);
        }
        if (care) {
#pragma unroll
          for (int s = 0; s < U; ++s)
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
              rk[s][c] = L.mask(rk[s][c], c, ok[s]);
              rv[s][c] = L.mask(rv[s][c], c, ok[s]);
            }
        }
        float x[U], top = -INFINITY;
#pragma unroll
        for (int s = 0; s < U; ++s) {
          const float d = head_dot<V, LPH>(q, rk[s]) * factor;
          x[s] = ok[s] ? d : -INFINITY;
          top = x[s] > top || x[s] != x[s] ? x[s] : top;
        }
        // The reference moves when a score is over it by more than 2^8 in weight: sums of weights
        // up to that stay exact enough in fp32, and most entries leave o and sum as they are.
        if (__any(!(top <= m + 8.f))) {
          const float to = !(top <= m + 8.f) ? top : m;
          const float keep = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - to);
          m = to;
          sum *= keep;
#pragma unroll
          for (int c = 0; c < NCH; ++c)
#pragma unroll
            for (int k = 0; k < V; ++k) o[c][k] *= keep;
        }
        const float ref = m == -INFINITY ? 0.f : m;  // only -inf so far: all weights are 0
#pragma unroll
        for (int s = 0; s < U; ++s) {
          const float p = __builtin_amdgcn_exp2f(x[s] - ref);
          sum += p;
#pragma unroll
          for (int c = 0; c < NCH; ++c) axpy<V>(p, rv[s][c], o[c]);
        }
      }
    }
    const float z = on ? zero_of(o, sum * 0.f) : 0.f;
    if (care || !__any(z != z)) break;
  }
  for (int w = LPH << S.hs; w < 64; w <<= 1) {  // the groups of one head
    const float mo = lane_xor(m, w), so = lane_xor(sum, w);
    const float top = mo > m || mo != mo ? mo : m;
    const float ref = top == -INFINITY ? 0.f : top;
    const float ka = __builtin_amdgcn_exp2f(m - ref), kb = __builtin_amdgcn_exp2f(mo - ref);
    m = top;
    sum = sum * ka + so * kb;
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int k = 0; k < V; ++k) o[c][k] = o[c][k] * ka + lane_xor(o[c][k], w) * kb;
  }
  if (slot != 0 || !on) return;
  if (u.slot >= 0) {
    float* part = ws + ((int64_t)u.slot * a.heads + head) * (dh + 2);
    if (L.l == 0) part[0] = m, part[1] = sum;
    L.store(part + 2, o, 1.f);
    return;
  }
  L.store((T*)a.o + u.row * a.ldo + (int64_t)head * dh, o, sum == 0.f ? 0.f : 1.f / sum);
  if (a.lse && L.l == 0)
    a.lse[(int64_t)u.row * a.heads + head] = sum == 0.f ? -INFINITY : m + __builtin_amdgcn_logf(sum);
}

template <typename T, int LPH, int NCH, bool FULL>
__global__ __launch_bounds__(256) void k_attn_rows(const gnnea_attn a, const AttnShape S,
                                                   float* __restrict__ ws) {
  constexpr int V = RowChunk<T>::V, G = 64 / LPH, U = Steps<NCH>::U;
  AttnUnit u;
  if (!attn_unit(a, S, u)) return;
  const int lane = lane_id(), grp = lane / LPH, dh = a.d_head;
  const Lane<T, LPH, NCH, FULL> L{dh, lane % LPH};
  const int head = (blockIdx.y << S.hs) + (grp & ((1 << S.hs) - 1)), slot = grp >> S.hs, eps = G >> S.hs;
  const bool on = head < a.heads;
  const int64_t kvo = (int64_t)(on ? by_share(S, head) : 0) * dh;
  const T* K = (const T*)a.k + kvo;
  const T* Vp = (const T*)a.v + kvo;
  const float factor = a.scale * kLog2e;
  const float lse = on ? a.lse[(int64_t)u.row * a.heads + head] : -INFINITY;
  uint4 q[NCH], d[NCH];
  // ref: c, the same in all groups of a head, of an entry of weight cap / 64; P: sum p, e: sum p (dp -
  // c), A: sum p (dp - c) k, B: sum p k
  float A[NCH][V], B[NCH][V], ref, cap, P, e;
  for (bool care = false;; care = true) {
    ColBatch cb(a, u);
    RowOffset off(a.n_cols, a.ldk);
    L.load_own((const T*)a.q + u.row * a.ldq + (int64_t)head * dh, on, q);
    L.load_own((const T*)a.dout + u.row * a.lddo + (int64_t)head * dh, on, d);
    ref = cap = P = e = 0.f;
    clear(A);
    clear(B);
    for (uint32_t done = 0; done < (uint32_t)cb.total; done += 64) {
      cb.step(done);
      off.set(cb.now, a.ldk);
      for (int b = 0; b < cb.left; b += eps * U) {
        uint4 rk[U][NCH], rv[U][NCH];
        bool ok[U];
#pragma unroll
        for (int s = 0; s < U; ++s) {
          const int i = b + s * eps + slot;
          // a row whose scores are all -inf has no weights (lse = -inf), like one without entries
          ok[s] = lse != -INFINITY && i < cb.left;
          const uint64_t j = off.of(min(i, 63));
#pragma unroll
          for (int c = 0; c < NCH; ++c) rk[s][c] = L.raw(K + j, c);
#pragma unroll
          for (int c = 0; c < NCH; ++c) rv[s][c] = L.raw(Vp + j, c);
        }
        if (care) {
#pragma unroll
          for (int s = 0; s < U; ++s)
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
              rk[s][c] = L.mask(rk[s][c], c, ok[s]);
              rv[s][c] = L.mask(rv[s][c], c, ok[s]);
            }
        }
        float p[U], y[U], most = 0.f;
#pragma unroll
        for (int s = 0; s < U; ++s) {
          const float x = head_dot<V, LPH>(q, rk[s]);
          y[s] = head_dot<V, LPH>(d, rv[s]);
          p[s] = ok[s] ? __builtin_amdgcn_exp2f(fmaf(x, factor, -lse)) : 0.f;
          most = fmaxf(most, p[s]);
        }
        if (__any(most > cap)) {
          float to = y[0];
          most = p[0];
#pragma unroll
          for (int s = 1; s < U; ++s)
            if (p[s] > most) most = p[s], to = y[s];
          for (int w = LPH << S.hs; w < 64; w <<= 1) {
            const float mo = lane_xor(most, w), yo = lane_xor(to, w);
            if (mo > most || (mo == most && yo < to)) most = mo, to = yo;
          }
          const float by = most > cap ? ref - to : 0.f;
          if (most > cap) ref = to, cap = 64.f * most;
          e = fmaf(by, P, e);
#pragma unroll
          for (int c = 0; c < NCH; ++c)
#pragma unroll
            for (int k = 0; k < V; ++k) A[c][k] = fmaf(by, B[c][k], A[c][k]);
        }
#pragma unroll
        for (int s = 0; s < U; ++s) {
          const float pd = p[s] * (y[s] - ref);
          e += pd;
          P += p[s];
#pragma unroll
          for (int c = 0; c < NCH; ++c) {
            axpy<V>(pd, rk[s][c], A[c]);
            axpy<V>(p[s], rk[s][c], B[c]);
          }
        }
      }
    }
    const float z = on ? zero_of(A, zero_of(B, e * 0.f)) : 0.f;
    if (care || !__any(z != z)) break;
  }
  for (int w = LPH << S.hs; w < 64; w <<= 1) {
    e += lane_xor(e, w);
    if (u.slot >= 0) P += lane_xor(P, w);
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        A[c][k] += lane_xor(A[c][k], w);
        B[c][k] += lane_xor(B[c][k], w);
      }
  }
  if (slot != 0 || !on) return;
  if (u.slot >= 0) {
    float* part = ws + ((int64_t)u.slot * a.heads + head) * (2 * dh + 4);
    if (L.l == 0) part[0] = ref, part[1] = cap, part[2] = P, part[3] = e;
    L.store(part + 4, A, 1.f);
    L.store(part + 4 + dh, B, 1.f);
    return;
  }
#pragma unroll
  for (int c = 0; c < NCH; ++c)
#pragma unroll
    for (int k = 0; k < V; ++k) A[c][k] = fmaf(-e, B[c][k], A[c][k]);
  L.store((T*)a.dq + u.row * a.lddq + (int64_t)head * dh, A, a.scale);
  if (L.l == 0)
    *(float2*)(a.stat + 2 * ((int64_t)u.row * a.heads + head)) = make_float2(lse, ref + e);
}

// Columns: a row of the transposed matrix per wave; groups take key/value heads, then (entry,
// query head of the group) pairs.
template <typename T, int LPH, int NCH, bool FULL>
__global__ __launch_bounds__(256) void k_attn_cols(const gnnea_attn a, const AttnShape S,
                                                   float* __restrict__ ws) {
  constexpr int V = RowChunk<T>::V, G = 64 / LPH, U = Steps<NCH>::U;
  AttnUnit u;
  if (!attn_unit(a, S, u)) return;
  const int lane = lane_id(), grp = lane / LPH, dh = a.d_head;
  const Lane<T, LPH, NCH, FULL> L{dh, lane % LPH};
  const int kvh = (blockIdx.y << S.hs) + (grp & ((1 << S.hs) - 1)), slot = grp >> S.hs, pps = G >> S.hs;
  const bool on = kvh < a.kv_heads;
  const float factor = a.scale * kLog2e;
  uint4 kf[NCH], vf[NCH];
  float dk[NCH][V], dv[NCH][V];
  for (bool care = false;; care = true) {
    ColBatch cb(a, u);
    RowOffset offq(a.n_cols, a.ldq), offd(a.n_cols, a.lddo);
    L.load_own((const T*)a.k + u.row * a.ldk + (int64_t)kvh * dh, on, kf);
    L.load_own((const T*)a.v + u.row * a.ldv + (int64_t)kvh * dh, on, vf);
    clear(dk);
    clear(dv);
    for (uint32_t done = 0; done < (uint32_t)cb.total; done += 64) {
      cb.step(done);
      offq.set(cb.now, a.ldq);
      offd.set(cb.now, a.lddo);
      const int pairs = cb.left * S.share;  // share <= heads <= 65535: fits
      for (int b = 0; b < pairs; b += pps * U) {
        uint4 rq[U][NCH], rd[U][NCH];
        float2 st[U];
        bool ok[U];
#pragma unroll
        for (int s = 0; s < U; ++s) {
          const int t = b + s * pps + slot, f = min(t, pairs - 1);
          ok[s] = on && t < pairs;
          const int e = by_share(S, f), h = (on ? kvh : 0) * S.share + f - e * S.share;
          const uint64_t i = (uint32_t)__shfl(cb.now, e, 64);
          st[s] = *(const float2*)(a.stat + 2 * (i * a.heads + h));
          const T* Q = (const T*)a.q + (offq.of(e) + h * dh);
          const T* Dp = (const T*)a.dout + (offd.of(e) + h * dh);
#pragma unroll
          for (int c = 0; c < NCH; ++c) rq[s][c] = L.raw(Q, c);
#pragma unroll
          for (int c = 0; c < NCH; ++c) rd[s][c] = L.raw(Dp, c);
        }
        if (care) {
#pragma unroll
          for (int s = 0; s < U; ++s)
#pragma unroll
            for (int c = 0; c < NCH; ++c) {
              rq[s][c] = L.mask(rq[s][c], c, ok[s] && st[s].x != -INFINITY);
              rd[s][c] = L.mask(rd[s][c], c, ok[s] && st[s].x != -INFINITY);
            }
        }
#pragma unroll
        for (int s = 0; s < U; ++s) {
          const float x = head_dot<V, LPH>(kf, rq[s]), y = head_dot<V, LPH>(vf, rd[s]);
          const float p = ok[s] && st[s].x != -INFINITY
                              ? __builtin_amdgcn_exp2f(fmaf(x, factor, -st[s].x)) : 0.f;
          const float ds = p * (y - st[s].y);
#pragma unroll
          for (int c = 0; c < NCH; ++c) {
            axpy<V>(ds, rq[s][c], dk[c]);
            axpy<V>(p, rd[s][c], dv[c]);
          }
        }
      }
    }
    const float z = on ? zero_of(dk, zero_of(dv, 0.f)) : 0.f;
    if (care || !__any(z != z)) break;
  }
  for (int w = LPH << S.hs; w < 64; w <<= 1) {
#pragma unroll
    for (int c = 0; c < NCH; ++c)
#pragma unroll
      for (int k = 0; k < V; ++k) {
        dk[c][k] += lane_xor(dk[c][k], w);
        dv[c][k] += lane_xor(dv[c][k], w);
      }
  }
  if (slot != 0 || !on) return;
  if (u.slot >= 0) {
    float* part = ws + ((int64_t)u.slot * a.kv_heads + kvh) * (2 * dh);
    L.store(part, dk, 1.f);
    L.store(part + dh, dv, 1.f);
    return;
  }
  L.store((T*)a.dk + u.row * a.lddk + (int64_t)kvh * dh, dk, a.scale);
  L.store((T*)a.dv + u.row * a.lddv + (int64_t)kvh * dh, dv, 1.f);
}

// Joins the pieces of a long row: a workgroup per row and head.  Its waves take the pieces in turn,
// four columns to a lane; their sums meet in LDS in wave order.  The row pass's pieces are moved to
// the c of the heaviest (equal ones: the smallest c, whatever the order).
template <typename T>
__global__ __launch_bounds__(512) void k_attn_join(const gnnea_attn a, int pass,
                                                   const float* __restrict__ ws) {
  __shared__ float sh[8][2 * 256 + 1];
  const int w = blockIdx.x, h = blockIdx.y, dh = a.d_head, row = a.long_rows[w];
  const int s0 = a.long_ptr[w], n = a.long_ptr[w + 1] - s0;
  const bool fwd = pass == GNNEA_ATTN_FWD, rows = pass == GNNEA_ATTN_BWD_ROWS;
  const int heads = pass == GNNEA_ATTN_BWD_COLS ? a.kv_heads : a.heads;
  const int wide = fwd ? dh + 2 : rows ? 2 * dh + 4 : 2 * dh;
  const float* part = ws + ((int64_t)s0 * heads + h) * wide;
  const int64_t step = (int64_t)heads * wide;
  const int lane = lane_id(), wv = wave_id();
  float m = -INFINITY;
  if (fwd) {
    for (int s = lane; s < n; s += 64) {
      const float x = part[s * step];
      m = x > m || x != x ? x : m;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const float x = __shfl_xor(m, o, 64);
      m = x > m || x != x ? x : m;
    }
  }
  float ref = m == -INFINITY ? 0.f : m;
  if (rows) {
    float top = -INFINITY;
    for (int s = lane; s < n; s += 64) {
      const float x = part[s * step], t = part[s * step + 1];
      if (t > top || (t == top && x < ref)) top = t, ref = x;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const float x = __shfl_xor(ref, o, 64), t = __shfl_xor(top, o, 64);
      if (t > top || (t == top && x < ref)) top = t, ref = x;
    }
  }
  // what a lane adds up: values lane, lane + 64, ... of a piece after its first words
  const int skip = fwd ? 2 : rows ? 4 : 0, width = wide - skip;
  float one = 0.f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  for (int s = wv; s < n; s += 8) {
    const float* p = part + s * step;
    const float f = fwd ? __builtin_amdgcn_exp2f(p[0] - ref) : 1.f, by = rows ? p[0] - ref : 0.f;
    if (fwd) one = fmaf(p[1], f, one);
    if (rows) one += fmaf(by, p[2], p[3]);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const int at = c * 64 + lane;
      if (at >= width) continue;
      float x = p[skip + at];
      if (rows && at < dh) x = fmaf(by, p[skip + dh + at], x);
      acc[c] = fmaf(x, f, acc[c]);
    }
  }
#pragma unroll
  for (int c = 0; c < 8; ++c)
    if (c * 64 + lane < width) sh[wv][1 + c * 64 + lane] = acc[c];
  if (lane == 0) sh[wv][0] = one;
  __syncthreads();
  for (int c = threadIdx.x; c <= width; c += 512) {
    float s = sh[0][c];
#pragma unroll
    for (int k = 1; k < 8; ++k) s += sh[k][c];
    sh[0][c] = s;
  }
  __syncthreads();
  one = sh[0][0];
  const float r = fwd ? (one == 0.f ? 0.f : 1.f / one) : a.scale;
  for (int d = threadIdx.x; d < dh; d += 512) {
    const float x = sh[0][1 + d];
    if (fwd) {
      ((T*)a.o)[row * a.ldo + (int64_t)h * dh + d] = from_f32<T>(x * r);
    } else if (rows) {
      ((T*)a.dq)[row * a.lddq + (int64_t)h * dh + d] = from_f32<T>(r * fmaf(-one, sh[0][1 + dh + d], x));
    } else {
      ((T*)a.dk)[row * a.lddk + (int64_t)h * dh + d] = from_f32<T>(r * x);
      ((T*)a.dv)[row * a.lddv + (int64_t)h * dh + d] = from_f32<T>(sh[0][1 + dh + d]);
    }
  }
  if (threadIdx.x != 0) return;
  if (fwd && a.lse)
    a.lse[(int64_t)row * a.heads + h] = one == 0.f ? -INFINITY : m + __builtin_amdgcn_logf(one);
  if (rows)
    *(float2*)(a.stat + 2 * ((int64_t)row * a.heads + h)) =
        make_float2(a.lse[(int64_t)row * a.heads + h], ref + one);
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
  if (!cols && a->ldk != a->ldv) return GNNEA_EINVAL;  // one offset for both
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
  AttnPlan p = {16, 4, 0, a->heads / a->kv_heads, -1, 1, false};
  for (const auto& s : kShape)
    if (s[0] * s[1] * V >= a->d_head) {
      p.lph = s[0];
      p.nch = s[1];
      break;
    }
  p.full = p.lph * p.nch * V == a->d_head;
  const int heads = pass == GNNEA_ATTN_BWD_COLS ? a->kv_heads : a->heads;
  while ((1 << p.hs) < heads && (1 << p.hs) < 64 / p.lph) ++p.hs;
  p.units_y = (heads + (1 << p.hs) - 1) >> p.hs;
  for (int k = 0; k < 16; ++k)
    if (p.share == 1 << k) p.ss = k;
  return p;
}

template <typename T, int LPH, int NCH, bool FULL>
static void attn_launch(const gnnea_attn& a, int pass, const AttnPlan& p, float* ws,
                        hipStream_t s) {
  for (int64_t row0 = 0; row0 < a.n_rows; row0 += kAttnRows) {
    const int64_t rows = a.n_rows - row0 < kAttnRows ? a.n_rows - row0 : kAttnRows;
    const AttnShape sh = {p.hs, p.share, p.ss, (int)row0, row0 ? 0 : a.n_items};
    const dim3 grid((unsigned)((sh.items + 3ll) / 4 + (rows + 3) / 4), p.units_y);
    if (pass == GNNEA_ATTN_FWD)
      hipLaunchKernelGGL((k_attn_fwd<T, LPH, NCH, FULL>), grid, dim3(256), 0, s, a, sh, ws);
    else if (pass == GNNEA_ATTN_BWD_ROWS)
      hipLaunchKernelGGL((k_attn_rows<T, LPH, NCH, FULL>), grid, dim3(256), 0, s, a, sh, ws);
    else
      hipLaunchKernelGGL((k_attn_cols<T, LPH, NCH, FULL>), grid, dim3(256), 0, s, a, sh, ws);
  }
}
template <typename T, int LPH, int NCH>
static void attn_launch(const gnnea_attn& a, int pass, const AttnPlan& p, float* ws,
                        hipStream_t s) {
  if (p.full) attn_launch<T, LPH, NCH, true>(a, pass, p, ws, s);
  else attn_launch<T, LPH, NCH, false>(a, pass, p, ws, s);
}

template <typename T>
static void attn_dispatch(const gnnea_attn& a, int pass, float* ws, hipStream_t s) {
  const AttnPlan p = attn_plan(&a, pass);
  if (p.lph == 4) attn_launch<T, 4, 1>(a, pass, p, ws, s);
  else if (p.lph == 8 && p.nch == 1) attn_launch<T, 8, 1>(a, pass, p, ws, s);
  else if (p.lph == 8 && p.nch == 2) attn_launch<T, 8, 2>(a, pass, p, ws, s);
  else if (p.lph == 8) attn_launch<T, 8, 3>(a, pass, p, ws, s);
  else if (p.nch == 2) attn_launch<T, 16, 2>(a, pass, p, ws, s);
  else if constexpr (sizeof(T) == 4) {  // bf16 heads of 256 fit two chunks
    if (p.nch == 3) attn_launch<T, 16, 3>(a, pass, p, ws, s);
    else attn_launch<T, 16, 4>(a, pass, p, ws, s);
  }
}

static int64_t attn_ws(const gnnea_attn* a, int pass) {
  const int64_t dh = a->d_head;
  if (pass == GNNEA_ATTN_FWD) return (int64_t)a->n_items * a->heads * (dh + 2) * 4;
  if (pass == GNNEA_ATTN_BWD_ROWS) return (int64_t)a->n_items * a->heads * (2 * dh + 4) * 4;
  return (int64_t)a->n_items * a->kv_heads * 2 * dh * 4;
}

static int attn_run(const gnnea_attn* a, int pass, void* ws, int64_t ws_bytes, void* stream) {
  const int rc = attn_check(a, pass);
  if (rc || a->n_rows == 0) return rc;
  if (ws_bytes < attn_ws(a, pass)) return GNNEA_EWORKSPACE;
  if (a->n_items && (!ws || ((uintptr_t)ws & 15))) return ws ? GNNEA_EALIGN : GNNEA_EINVAL;
  const hipStream_t s = (hipStream_t)stream;
  if (a->dtype == GNNEA_F32) attn_dispatch<float>(*a, pass, (float*)ws, s);
  else attn_dispatch<bf16_t>(*a, pass, (float*)ws, s);
  GNNEA_LAUNCH_CHECK();
  if (a->n_items) {
    const dim3 grid(a->n_long, pass == GNNEA_ATTN_BWD_COLS ? a->kv_heads : a->heads);
    if (a->dtype == GNNEA_F32)
      hipLaunchKernelGGL(k_attn_join<float>, grid, dim3(512), 0, s, *a, pass, (const float*)ws);
    else
      hipLaunchKernelGGL(k_attn_join<bf16_t>, grid, dim3(512), 0, s, *a, pass, (const float*)ws);
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

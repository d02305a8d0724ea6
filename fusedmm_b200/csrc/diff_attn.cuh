// diff_attn.cuh -- differential attention over the edges of a CSR, forward and backward (include/fusedmm_b200.h,
// fusedmm_b200_diff_attention).
//
//   s^c_e = scale q^c_u . k^c_v + bias_e (c = 0, 1);  p^c = softmax over the edges e = (u, v) of row u;
//   o_u = sum_e (p^0_e - lam p^1_e) v_v
//   backward, with dP_e = do_u . v_v, D^c_u = sum_e p^c_e dP_e:  ds^0 = p^0 (dP - D^0), ds^1 = -lam p^1 (dP - D^1),
//   dq^c_u = scale sum_e ds^c k^c_v, dk^c_v = scale sum_e ds^c q^c_u, dv_v = sum_e (p^0 - lam p^1) do_u, dlam_u = -D^1_u.
//
// Three walks of the same shape: the forward and the dq pass go over the rows and gather k and v; the dk, dv pass goes over
// the columns of the transposed pattern and gathers q and do.  No atomics: every sum is taken in a fixed order.
//
// The gathered rows decide the layout.  A slot of G lanes takes one head of one edge; its two halves hold the two maps'
// parts of k (or q), so the two dots are one butterfly of G/2 lanes and each half owns the running maximum and sum of its
// map; v (or do) lies over all G lanes.  The slots of a warp take neighbouring heads of the same edge, as far as there are
// heads (their rows are adjacent in memory and all slots run in step), and alternate edges beyond that, joined at the row's
// end.  QB query heads that share a kv head are computed together from one load.
//
// Work is cut at equal parts ("pieces") of the items nnz + ROW_ITEMS * m, so that hub rows, single long rows of a decoding
// step and empty rows are spread alike, without a pass over the pattern: a warp finds its first row by a 32-ary search in
// the row pointers.  A row of up to `row_limit` items belongs to the piece it begins in; a longer one is cut at the pieces'
// borders, its parts go to `partial` and a second launch joins them in order.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "attn_common.cuh"

namespace fmm {
namespace attn {

constexpr int ROW_ITEMS = 8;        // what a row costs beside its edges, in edges
constexpr int PIECE_WARPS = 8;      // warps of a block
constexpr int JOIN_PIECES = 8;      // pieces a joining block looks after

struct AttnParams {
   const void *rowptr, *colidx;  // row walks: the pattern; column walk: the transposed one (colidx: 32-bit row ids)
   int ptr64, idx64;
   long long m, n, nnz;          // rows walked, rows that can be gathered, length of colidx
   const float *bias;
   const int *edge_of;           // column walk: position of an edge in `bias`
   const void *q, *k, *v, *dout;
   const float *lam;
   long long ldq, hsq, ldk, hsk, ldv, hsv, ldo, hso, ldlam;
   void *out;                    // forward [m,H,Dv]; dq [m,H,2,D]; dk [n,Hk,2,D]
   void *out2;                   // dv [n,Hk,Dv]
   float *lse;                   // [m,H,2]
   float2 *stats;                // [m,H,2]: lse and D of a map
   float *dlam;                  // [m,H]
   int heads, kv_heads, group, d, dv, step;
   float scale;
   int units, unit_blocks, slot_heads;  // head units of QB heads; warps (blocks) that share them; slots of a warp across units
   long long piece, row_limit, pieces;
   float *partial;
   long long *long_row;          // [pieces]: the long row that begins in a piece, or -1
};

__device__ __forceinline__ long long load_index(const void *p, int is64, long long i)
{
   return is64 ? __ldg(static_cast<const long long *>(p) + i) : static_cast<long long>(__ldg(static_cast<const int *>(p) + i));
}

// Row pointers kept inside [first, nnz]: a pattern that breaks its contract gives wrong rows, no access out of bounds.
struct Rows {
   const AttnParams &p;
   long long first;
   __device__ __forceinline__ explicit Rows(const AttnParams &q) : p(q)
   {
      first = load_index(p.rowptr, p.ptr64, 0);
      first = first < 0 ? 0 : first > p.nnz ? p.nnz : first;
   }
   __device__ __forceinline__ long long begin(long long u) const
   {
      const long long b = load_index(p.rowptr, p.ptr64, u);
      return b < first ? first : b > p.nnz ? p.nnz : b;
   }
   __device__ __forceinline__ long long items(long long u) const { return begin(u) - first + ROW_ITEMS * u; }
   // first row u in [0, m] with items(u) >= at; the whole warp takes part
   __device__ __forceinline__ long long lower_bound(long long at, int lane) const
   {
      long long lo = 0, hi = p.m;
      while (lo < hi) {
         const long long step = (hi - lo + 31) / 32;
         const long long u = lo + step * lane;
         const bool below = u < hi && items(u) < at;
         const unsigned mask = __ballot_sync(FULL, below);
         if (mask == 0) return lo;
         const long long last = lo + step * (31 - __clz(mask));  // the last probe known to be below
         const long long next = last + step;
         lo = last + 1;
         hi = next < hi ? next : hi;
      }
      return lo;
   }
};

// a warp's place: the piece, the block of head units, its lanes
struct Place {
   int lane, in_slot, half, in_half, edge_slot, edge_slots, unit, warp;
   template <int G>
   static __device__ __forceinline__ Place make(const AttnParams &p, int unit_block)
   {
      Place a;
      a.fill(p, unit_block, G);
      return a;
   }
   __device__ __forceinline__ void fill(const AttnParams &p, int unit_block, int G)
   {
      lane = threadIdx.x & 31;
      warp = threadIdx.x >> 5;
      in_slot = lane % G;
      half = in_slot / (G / 2);
      in_half = in_slot % (G / 2);
      const int slot = lane / G;
      unit = unit_block * p.slot_heads + slot % p.slot_heads;
      edge_slot = slot / p.slot_heads;
      edge_slots = (32 / G) / p.slot_heads;
   }
};

template <int LANES>
__device__ __forceinline__ float add_over(float v)
{
#pragma unroll
   for (int s = LANES / 2; s > 0; s >>= 1) v += __shfl_xor_sync(FULL, v, s);
   return v;
}

// a vector of W floats of scratch, 16 bytes at a time
template <int N>
__device__ __forceinline__ void put_floats(float *p, const float (&f)[N])
{
#pragma unroll
   for (int i = 0; i < N; i += 4) *reinterpret_cast<float4 *>(p + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
}
template <int N>
__device__ __forceinline__ void get_floats(const float *p, float (&f)[N])
{
#pragma unroll
   for (int i = 0; i < N; i += 4) {
      const float4 a = *reinterpret_cast<const float4 *>(p + i);
      f[i] = a.x; f[i + 1] = a.y; f[i + 2] = a.z; f[i + 3] = a.w;
   }
}

// 32 edges of a row, one to a lane: the id to gather (-1: no edge here, or one that is masked) and its bias
struct EdgeBatch {
   long long id;
   float bias;
   __device__ __forceinline__ void load(const AttnParams &p, long long e, long long end)
   {
      id = -1;
      bias = 0.0f;
      if (e < end) {
         id = load_index(p.colidx, p.idx64, e);
         if (id < 0 || id >= p.n) id = -1;
         if (p.bias) {
            bias = __ldg(p.bias + (p.edge_of ? static_cast<long long>(__ldg(p.edge_of + e)) : e));
            if (bias == -INFINITY) id = -1;
         }
      }
   }
};

// ---------------------------------------------------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int G, int NV, int QB, bool VECTOR>
struct Forward {
   static constexpr int W = Elt<T>::W, U = NV * QB > 2 ? 1 : 2;
   static constexpr int LANE_FLOATS = QB * (2 * NV * W + 2);  // partial state of a lane
   struct State {
      float acc[QB][2][NV][W];  // sums of p v for the two maps
      float top[QB], sum[QB];   // of this half's map
   };
   float q[QB][NV][W];
   State s;

   static __device__ __forceinline__ void clear(State &s)
   {
#pragma unroll
      for (int b = 0; b < QB; b++) {
         s.top[b] = -INFINITY;
         s.sum[b] = 0.0f;
#pragma unroll
         for (int c = 0; c < 2; c++)
#pragma unroll
            for (int t = 0; t < NV; t++)
#pragma unroll
               for (int j = 0; j < W; j++) s.acc[b][c][t][j] = 0.0f;
      }
   }

   __device__ __forceinline__ void run(const AttnParams &p, const Place &at, long long row, long long e0, long long e1, int warp, int warps)
   {
      clear(s);
      const int kv = at.unit / (p.group / QB), head0 = at.unit * QB;
#pragma unroll
      for (int b = 0; b < QB; b++)
#pragma unroll
         for (int t = 0; t < NV; t++) {
            const int x = (at.in_half + (G / 2) * t) * W;
            const T *src = static_cast<const T *>(p.q) + row * p.ldq + (head0 + b) * p.hsq + at.half * p.d + x;
            Elt<T>::unpack(ld_row<T, VECTOR>(src, p.d - x, p.step), q[b][t]);
         }
      const T *kbase = static_cast<const T *>(p.k) + kv * p.hsk + at.half * p.d;
      const T *vbase = static_cast<const T *>(p.v) + kv * p.hsv;
      for (long long base = e0 + 32 * warp; base < e1; base += 32 * warps) {
         EdgeBatch batch;
         batch.load(p, base + at.lane, e1);
         const int count = static_cast<int>(e1 - base < 32 ? e1 - base : 32);
         for (int first = 0; first < count; first += U * at.edge_slots) {
            long long id[U];
            float bias[U];
            uint4 kr[U][NV], vr[U][NV];
#pragma unroll
            for (int i = 0; i < U; i++) {
               const int from = first + i * at.edge_slots + at.edge_slot;
               id[i] = __shfl_sync(FULL, batch.id, from);
               bias[i] = __shfl_sync(FULL, batch.bias, from);
               const bool live = id[i] >= 0;
#pragma unroll
               for (int t = 0; t < NV; t++) {
                  const int x = (at.in_half + (G / 2) * t) * W, y = (at.in_slot + G * t) * W;
                  kr[i][t] = ld_row<T, VECTOR>(kbase + id[i] * p.ldk + x, live ? p.d - x : 0, p.step);
                  vr[i][t] = ld_row<T, VECTOR>(vbase + id[i] * p.ldv + y, live ? p.dv - y : 0, p.step);
               }
            }
            float score[QB][U];
#pragma unroll
            for (int i = 0; i < U; i++) {
               float k[NV][W];
#pragma unroll
               for (int t = 0; t < NV; t++) Elt<T>::unpack(kr[i][t], k[t]);
#pragma unroll
               for (int b = 0; b < QB; b++) {
                  float dot = 0.0f;
#pragma unroll
                  for (int t = 0; t < NV; t++)
#pragma unroll
                     for (int j = 0; j < W; j++) dot = fmaf(q[b][t][j], k[t][j], dot);
                  dot = add_over<G / 2>(dot);
                  score[b][i] = id[i] >= 0 ? fmaf(dot, p.scale, bias[i]) : -INFINITY;
               }
            }
#pragma unroll
            for (int b = 0; b < QB; b++) {
               float top = s.top[b];
#pragma unroll
               for (int i = 0; i < U; i++) top = fmaxf(top, score[b][i]);
               // a row that has met no edge yet has the maximum -inf: its differences are taken from 0
               const float ref = top == -INFINITY ? 0.0f : top;
               if (__any_sync(FULL, top != s.top[b])) {
                  const float mine = exp2f((s.top[b] - ref) * LOG2E), other = __shfl_xor_sync(FULL, mine, G / 2);
                  const float c0 = at.half ? other : mine, c1 = at.half ? mine : other;
                  s.sum[b] *= mine;
#pragma unroll
                  for (int t = 0; t < NV; t++)
#pragma unroll
                     for (int j = 0; j < W; j++) {
                        s.acc[b][0][t][j] *= c0;
                        s.acc[b][1][t][j] *= c1;
                     }
                  s.top[b] = top;
               }
#pragma unroll
               for (int i = 0; i < U; i++) {
                  // the difference is taken before the factor: scores near the type's largest numbers keep their order
                  const float mine = exp2f((score[b][i] - ref) * LOG2E), other = __shfl_xor_sync(FULL, mine, G / 2);
                  const float p0 = at.half ? other : mine, p1 = at.half ? mine : other;
                  s.sum[b] += mine;
#pragma unroll
                  for (int t = 0; t < NV; t++) {
                     float v[W];
                     Elt<T>::unpack(vr[i][t], v);
#pragma unroll
                     for (int j = 0; j < W; j++) {
                        s.acc[b][0][t][j] = fmaf(p0, v[j], s.acc[b][0][t][j]);
                        s.acc[b][1][t][j] = fmaf(p1, v[j], s.acc[b][1][t][j]);
                     }
                  }
               }
            }
         }
      }
      for (int x = G * p.slot_heads; x < 32; x <<= 1) {  // the slots that took alternate edges
         State o;
#pragma unroll
         for (int b = 0; b < QB; b++) {
            o.top[b] = __shfl_xor_sync(FULL, s.top[b], x);
            o.sum[b] = __shfl_xor_sync(FULL, s.sum[b], x);
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
               for (int t = 0; t < NV; t++)
#pragma unroll
                  for (int j = 0; j < W; j++) o.acc[b][c][t][j] = __shfl_xor_sync(FULL, s.acc[b][c][t][j], x);
         }
         join(s, o, at, (at.lane & x) != 0);
      }
   }

   // joins the state of other edges of the row; `swap`: the other's edges come first (both sides of an exchange then add
   // in the same order)
   static __device__ __forceinline__ void join(State &s, const State &o, const Place &at, bool swap)
   {
#pragma unroll
      for (int b = 0; b < QB; b++) {
         const float top = fmaxf(s.top[b], o.top[b]), ref = top == -INFINITY ? 0.0f : top;
         const float fs = exp2f((s.top[b] - ref) * LOG2E), fo = exp2f((o.top[b] - ref) * LOG2E);
         const float fs2 = __shfl_xor_sync(FULL, fs, G / 2), fo2 = __shfl_xor_sync(FULL, fo, G / 2);
         // a NaN score leaves its trace in the sum and the accumulators, the maximum skips it
         const float a = s.sum[b] * fs, c = o.sum[b] * fo;
         s.sum[b] = swap ? c + a : a + c;
         s.top[b] = top;
#pragma unroll
         for (int m = 0; m < 2; m++) {
            const float f1 = m == at.half ? fs : fs2, f2 = m == at.half ? fo : fo2;
#pragma unroll
            for (int t = 0; t < NV; t++)
#pragma unroll
               for (int j = 0; j < W; j++) {
                  const float x = s.acc[b][m][t][j], y = o.acc[b][m][t][j];
                  s.acc[b][m][t][j] = swap ? fmaf(y, f2, x * f1) : fmaf(x, f1, y * f2);
               }
         }
      }
   }
   __device__ __forceinline__ void join_from(const float *unit, const Place &at)
   {
      const float *from = unit + at.in_slot * W;
      State o;
#pragma unroll
      for (int b = 0; b < QB; b++) {
#pragma unroll
         for (int c = 0; c < 2; c++)
#pragma unroll
            for (int t = 0; t < NV; t++) get_floats<W>(from + ((b * 2 + c) * NV + t) * W * G, o.acc[b][c][t]);
         const float2 ts = *reinterpret_cast<const float2 *>(unit + QB * 2 * NV * W * G + (b * G + at.in_slot) * 2);
         o.top[b] = ts.x;
         o.sum[b] = ts.y;
      }
      join(s, o, at, false);
   }
   __device__ __forceinline__ void put(float *unit, const Place &at) const
   {
      float *to = unit + at.in_slot * W;
#pragma unroll
      for (int b = 0; b < QB; b++) {
#pragma unroll
         for (int c = 0; c < 2; c++)
#pragma unroll
            for (int t = 0; t < NV; t++) put_floats<W>(to + ((b * 2 + c) * NV + t) * W * G, s.acc[b][c][t]);
         *reinterpret_cast<float2 *>(unit + QB * 2 * NV * W * G + (b * G + at.in_slot) * 2) = make_float2(s.top[b], s.sum[b]);
      }
   }

   __device__ __forceinline__ void finish(const AttnParams &p, const Place &at, long long row)
   {
#pragma unroll
      for (int b = 0; b < QB; b++) {
         const float other = __shfl_xor_sync(FULL, s.sum[b], G / 2);
         if (at.edge_slot != 0) continue;
         const int head = at.unit * QB + b;
         const float l0 = at.half ? other : s.sum[b], l1 = at.half ? s.sum[b] : other;
         const float lam = __ldg(p.lam + row * p.ldlam + head);
         const float f0 = l0 == 0.0f ? 0.0f : 1.0f / l0, f1 = l1 == 0.0f ? 0.0f : lam / l1;
#pragma unroll
         for (int t = 0; t < NV; t++) {
            const int y = (at.in_slot + G * t) * W;
            float o[W];
#pragma unroll
            for (int j = 0; j < W; j++) o[j] = s.acc[b][0][t][j] * f0 - s.acc[b][1][t][j] * f1;
            st_row<T, VECTOR>(static_cast<T *>(p.out) + (row * p.heads + head) * p.dv + y, o, p.dv - y);
         }
         if (at.in_half == 0 && p.lse) p.lse[(row * p.heads + head) * 2 + at.half] = s.top[b] + LN2 * log2f(s.sum[b]);
      }
   }
};

// ---------------------------------------------------------------------------------------------------------------------
// backward over the rows: dq, dlam and the numbers the columns need.  With D^c unknown until the row's end, the sums
// A = sum p dP k, B = sum p k and D = sum p dP are taken together; dq = scale (A - D B).
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int G, int NV, int QB, bool VECTOR>
struct BackwardRows {
   static constexpr int W = Elt<T>::W, U = NV * QB > 2 ? 1 : 2;
   static constexpr int LANE_FLOATS = QB * (2 * NV * W + 2);
   struct State {
      float a[QB][NV][W], b[QB][NV][W];  // of this half's map
      float delta[QB];
   };
   float q[QB][NV][W], dout[QB][NV][W], lse[QB];
   State s;

   static __device__ __forceinline__ void clear(State &s)
   {
#pragma unroll
      for (int b = 0; b < QB; b++) {
         s.delta[b] = 0.0f;
#pragma unroll
         for (int t = 0; t < NV; t++)
#pragma unroll
            for (int j = 0; j < W; j++) s.a[b][t][j] = s.b[b][t][j] = 0.0f;
      }
   }

   __device__ __forceinline__ void run(const AttnParams &p, const Place &at, long long row, long long e0, long long e1, int warp, int warps)
   {
      clear(s);
      const int kv = at.unit / (p.group / QB), head0 = at.unit * QB;
#pragma unroll
      for (int b = 0; b < QB; b++) {
         lse[b] = __ldg(p.lse + (row * p.heads + head0 + b) * 2 + at.half);
#pragma unroll
         for (int t = 0; t < NV; t++) {
            const int x = (at.in_half + (G / 2) * t) * W, y = (at.in_slot + G * t) * W;
            const T *src = static_cast<const T *>(p.q) + row * p.ldq + (head0 + b) * p.hsq + at.half * p.d + x;
            Elt<T>::unpack(ld_row<T, VECTOR>(src, p.d - x, p.step), q[b][t]);
            const T *dsrc = static_cast<const T *>(p.dout) + row * p.ldo + (head0 + b) * p.hso + y;
            Elt<T>::unpack(ld_row<T, VECTOR>(dsrc, p.dv - y, p.step), dout[b][t]);
         }
      }
      const T *kbase = static_cast<const T *>(p.k) + kv * p.hsk + at.half * p.d;
      const T *vbase = static_cast<const T *>(p.v) + kv * p.hsv;
      for (long long base = e0 + 32 * warp; base < e1; base += 32 * warps) {
         EdgeBatch batch;
         batch.load(p, base + at.lane, e1);
         const int count = static_cast<int>(e1 - base < 32 ? e1 - base : 32);
         for (int first = 0; first < count; first += U * at.edge_slots) {
            long long id[U];
            float bias[U];
            uint4 kr[U][NV], vr[U][NV];
#pragma unroll
            for (int i = 0; i < U; i++) {
               const int from = first + i * at.edge_slots + at.edge_slot;
               id[i] = __shfl_sync(FULL, batch.id, from);
               bias[i] = __shfl_sync(FULL, batch.bias, from);
               const bool live = id[i] >= 0;
#pragma unroll
               for (int t = 0; t < NV; t++) {
                  const int x = (at.in_half + (G / 2) * t) * W, y = (at.in_slot + G * t) * W;
                  kr[i][t] = ld_row<T, VECTOR>(kbase + id[i] * p.ldk + x, live ? p.d - x : 0, p.step);
                  vr[i][t] = ld_row<T, VECTOR>(vbase + id[i] * p.ldv + y, live ? p.dv - y : 0, p.step);
               }
            }
#pragma unroll
            for (int i = 0; i < U; i++) {
               float k[NV][W], v[NV][W];
#pragma unroll
               for (int t = 0; t < NV; t++) {
                  Elt<T>::unpack(kr[i][t], k[t]);
                  Elt<T>::unpack(vr[i][t], v[t]);
               }
#pragma unroll
               for (int b = 0; b < QB; b++) {
                  float dot = 0.0f, dp = 0.0f;
#pragma unroll
                  for (int t = 0; t < NV; t++)
#pragma unroll
                     for (int j = 0; j < W; j++) {
                        dot = fmaf(q[b][t][j], k[t][j], dot);
                        dp = fmaf(dout[b][t][j], v[t][j], dp);
                     }
                  dot = add_over<G / 2>(dot);
                  dp = add_over<G>(dp);
                  // an edge that is masked has p = 0, and so has a row without edges (its lse is -inf)
                  const float pr = id[i] >= 0 && lse[b] != -INFINITY ? exp2f((fmaf(dot, p.scale, bias[i]) - lse[b]) * LOG2E) : 0.0f;
                  const float w = pr * dp;
                  s.delta[b] += w;
#pragma unroll
                  for (int t = 0; t < NV; t++)
#pragma unroll
                     for (int j = 0; j < W; j++) {
                        s.a[b][t][j] = fmaf(w, k[t][j], s.a[b][t][j]);
                        s.b[b][t][j] = fmaf(pr, k[t][j], s.b[b][t][j]);
                     }
               }
            }
         }
      }
      for (int x = G * p.slot_heads; x < 32; x <<= 1) {
#pragma unroll
         for (int b = 0; b < QB; b++) {
            s.delta[b] += __shfl_xor_sync(FULL, s.delta[b], x);
#pragma unroll
            for (int t = 0; t < NV; t++)
#pragma unroll
               for (int j = 0; j < W; j++) {
                  s.a[b][t][j] += __shfl_xor_sync(FULL, s.a[b][t][j], x);
                  s.b[b][t][j] += __shfl_xor_sync(FULL, s.b[b][t][j], x);
               }
         }
      }
   }
   __device__ __forceinline__ void join_from(const float *unit, const Place &at)
   {
      const float *from = unit + at.in_slot * W;
#pragma unroll
      for (int b = 0; b < QB; b++) {
#pragma unroll
         for (int t = 0; t < NV; t++) {
            float x[W];
            get_floats<W>(from + (b * 2 * NV + t) * W * G, x);
#pragma unroll
            for (int j = 0; j < W; j++) s.a[b][t][j] += x[j];
            get_floats<W>(from + ((b * 2 + 1) * NV + t) * W * G, x);
#pragma unroll
            for (int j = 0; j < W; j++) s.b[b][t][j] += x[j];
         }
         s.delta[b] += unit[QB * 2 * NV * W * G + (b * G + at.in_slot) * 2];
      }
   }
   __device__ __forceinline__ void put(float *unit, const Place &at) const
   {
      float *to = unit + at.in_slot * W;
#pragma unroll
      for (int b = 0; b < QB; b++) {
#pragma unroll
         for (int t = 0; t < NV; t++) {
            put_floats<W>(to + (b * 2 * NV + t) * W * G, s.a[b][t]);
            put_floats<W>(to + ((b * 2 + 1) * NV + t) * W * G, s.b[b][t]);
         }
         unit[QB * 2 * NV * W * G + (b * G + at.in_slot) * 2] = s.delta[b];
      }
   }

   __device__ __forceinline__ void finish(const AttnParams &p, const Place &at, long long row)
   {
      if (at.edge_slot != 0) return;
#pragma unroll
      for (int b = 0; b < QB; b++) {
         const int head = at.unit * QB + b;
         const long long rh = row * p.heads + head;
         const float factor = at.half ? -__ldg(p.lam + row * p.ldlam + head) * p.scale : p.scale;
#pragma unroll
         for (int t = 0; t < NV; t++) {
            const int x = (at.in_half + (G / 2) * t) * W;
            float o[W];
#pragma unroll
            for (int j = 0; j < W; j++) o[j] = factor * fmaf(-s.delta[b], s.b[b][t][j], s.a[b][t][j]);
            st_row<T, VECTOR>(static_cast<T *>(p.out) + (rh * 2 + at.half) * p.d + x, o, p.d - x);
         }
         if (at.in_half == 0) {
            p.stats[rh * 2 + at.half] = make_float2(__ldg(p.lse + rh * 2 + at.half), s.delta[b]);
            if (at.half == 1) p.dlam[rh] = -s.delta[b];
         }
      }
   }
};

// ---------------------------------------------------------------------------------------------------------------------
// backward over the columns: dk and dv.  A unit is a kv head; every edge counts once for each query head of its group.
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int G, int NV, int QB, bool VECTOR>
struct BackwardColumns {
   static constexpr int W = Elt<T>::W, U = NV > 1 ? 1 : 2;
   static constexpr int LANE_FLOATS = 2 * NV * W;
   struct State {
      float dk[NV][W], dv[NV][W];
   };
   float k[NV][W], v[NV][W];
   State s;

   static __device__ __forceinline__ void clear(State &s)
   {
#pragma unroll
      for (int t = 0; t < NV; t++)
#pragma unroll
         for (int j = 0; j < W; j++) s.dk[t][j] = s.dv[t][j] = 0.0f;
   }

   __device__ __forceinline__ void run(const AttnParams &p, const Place &at, long long col, long long e0, long long e1, int warp, int warps)
   {
      clear(s);
      const int kv = at.unit;
#pragma unroll
      for (int t = 0; t < NV; t++) {
         const int x = (at.in_half + (G / 2) * t) * W, y = (at.in_slot + G * t) * W;
         Elt<T>::unpack(ld_row<T, VECTOR>(static_cast<const T *>(p.k) + col * p.ldk + kv * p.hsk + at.half * p.d + x, p.d - x, p.step), k[t]);
         Elt<T>::unpack(ld_row<T, VECTOR>(static_cast<const T *>(p.v) + col * p.ldv + kv * p.hsv + y, p.dv - y, p.step), v[t]);
      }
      for (long long base = e0 + 32 * warp; base < e1; base += 32 * warps) {
         EdgeBatch batch;
         batch.load(p, base + at.lane, e1);
         const int count = static_cast<int>(e1 - base < 32 ? e1 - base : 32);
         for (int first = 0; first < count; first += U * at.edge_slots) {
            long long id[U];
            float bias[U];
#pragma unroll
            for (int i = 0; i < U; i++) {
               const int from = first + i * at.edge_slots + at.edge_slot;
               id[i] = __shfl_sync(FULL, batch.id, from);
               bias[i] = __shfl_sync(FULL, batch.bias, from);
            }
            for (int g = 0; g < p.group; g++) {
               const int head = kv * p.group + g;
               uint4 qr[U][NV], dr[U][NV];
               float2 stat[U];
               float lam[U];
#pragma unroll
               for (int i = 0; i < U; i++) {
                  const bool live = id[i] >= 0;
                  stat[i] = make_float2(0.0f, 0.0f);
                  lam[i] = 0.0f;
                  if (live) {
                     stat[i] = __ldg(p.stats + (id[i] * p.heads + head) * 2 + at.half);
                     lam[i] = __ldg(p.lam + id[i] * p.ldlam + head);
                  }
#pragma unroll
                  for (int t = 0; t < NV; t++) {
                     const int x = (at.in_half + (G / 2) * t) * W, y = (at.in_slot + G * t) * W;
                     qr[i][t] = ld_row<T, VECTOR>(static_cast<const T *>(p.q) + id[i] * p.ldq + head * p.hsq + at.half * p.d + x,
                                                  live ? p.d - x : 0, p.step);
                     dr[i][t] = ld_row<T, VECTOR>(static_cast<const T *>(p.dout) + id[i] * p.ldo + head * p.hso + y,
                                                  live ? p.dv - y : 0, p.step);
                  }
               }
#pragma unroll
               for (int i = 0; i < U; i++) {
                  float q[NV][W], dout[NV][W], dot = 0.0f, dp = 0.0f;
#pragma unroll
                  for (int t = 0; t < NV; t++) {
                     Elt<T>::unpack(qr[i][t], q[t]);
                     Elt<T>::unpack(dr[i][t], dout[t]);
#pragma unroll
                     for (int j = 0; j < W; j++) {
                        dot = fmaf(q[t][j], k[t][j], dot);
                        dp = fmaf(dout[t][j], v[t][j], dp);
                     }
                  }
                  dot = add_over<G / 2>(dot);
                  dp = add_over<G>(dp);
                  const bool live = id[i] >= 0 && stat[i].x != -INFINITY;
                  const float pr = live ? exp2f((fmaf(dot, p.scale, bias[i]) - stat[i].x) * LOG2E) : 0.0f;
                  const float mine = live ? (at.half ? -lam[i] : 1.0f) * pr : 0.0f;  // this map's part of the weight
                  const float w = mine + __shfl_xor_sync(FULL, mine, G / 2);
                  const float ds = live ? mine * (dp - stat[i].y) : 0.0f;
#pragma unroll
                  for (int t = 0; t < NV; t++)
#pragma unroll
                     for (int j = 0; j < W; j++) {
                        s.dk[t][j] = fmaf(ds, q[t][j], s.dk[t][j]);
                        s.dv[t][j] = fmaf(w, dout[t][j], s.dv[t][j]);
                     }
               }
            }
         }
      }
      for (int x = G * p.slot_heads; x < 32; x <<= 1) {
#pragma unroll
         for (int t = 0; t < NV; t++)
#pragma unroll
            for (int j = 0; j < W; j++) {
               s.dk[t][j] += __shfl_xor_sync(FULL, s.dk[t][j], x);
               s.dv[t][j] += __shfl_xor_sync(FULL, s.dv[t][j], x);
            }
      }
   }
   __device__ __forceinline__ void join_from(const float *unit, const Place &at)
   {
      const float *from = unit + at.in_slot * W;
#pragma unroll
      for (int t = 0; t < NV; t++) {
         float x[W];
         get_floats<W>(from + t * W * G, x);
#pragma unroll
         for (int j = 0; j < W; j++) s.dk[t][j] += x[j];
         get_floats<W>(from + (NV + t) * W * G, x);
#pragma unroll
         for (int j = 0; j < W; j++) s.dv[t][j] += x[j];
      }
   }
   __device__ __forceinline__ void put(float *unit, const Place &at) const
   {
      float *to = unit + at.in_slot * W;
#pragma unroll
      for (int t = 0; t < NV; t++) {
         put_floats<W>(to + t * W * G, s.dk[t]);
         put_floats<W>(to + (NV + t) * W * G, s.dv[t]);
      }
   }

   __device__ __forceinline__ void finish(const AttnParams &p, const Place &at, long long col)
   {
      if (at.edge_slot != 0) return;
      const long long rh = col * p.kv_heads + at.unit;
#pragma unroll
      for (int t = 0; t < NV; t++) {
         const int x = (at.in_half + (G / 2) * t) * W, y = (at.in_slot + G * t) * W;
         float o[W];
#pragma unroll
         for (int j = 0; j < W; j++) o[j] = s.dk[t][j] * p.scale;
         st_row<T, VECTOR>(static_cast<T *>(p.out) + (rh * 2 + at.half) * p.d + x, o, p.d - x);
         st_row<T, VECTOR>(static_cast<T *>(p.out2) + rh * p.dv + y, s.dv[t], p.dv - y);
      }
   }
};

// ---------------------------------------------------------------------------------------------------------------------
// the walk and the join
// ---------------------------------------------------------------------------------------------------------------------
// floats of the partial state of one unit of one part of a long row
template <typename Op, int G>
constexpr long long part_floats = static_cast<long long>(Op::LANE_FLOATS) * G;

template <typename Op, int G>
__device__ __forceinline__ float *part_at(const AttnParams &p, const Place &at, long long part)
{
   return p.partial + (part * p.units + at.unit) * part_floats<Op, G>;
}

// the warps of a block that shared a row: warp 0 takes the others' states in order
template <typename Op, int G>
__device__ __forceinline__ void join_warps(Op &op, const Place &at, float *shared)
{
   constexpr int STRIDE = Op::LANE_FLOATS * 32;  // slots side by side, as in scratch
   float *mine = shared + (at.lane / G) * part_floats<Op, G>;
   __syncthreads();
   if (at.warp > 0) op.put(mine + (at.warp - 1) * STRIDE, at);
   __syncthreads();
   if (at.warp == 0)
      for (int w = 1; w < PIECE_WARPS; w++) op.join_from(mine + (w - 1) * STRIDE, at);
}

// TOGETHER: the warps of a block share every row (few, long rows), else each warp has a piece of its own.
template <typename Op, int G, bool TOGETHER>
__global__ void __launch_bounds__(PIECE_WARPS * 32) walk_kernel(const AttnParams p)
{
   extern __shared__ __align__(16) float shared[];
   const int warp = threadIdx.x >> 5;
   const long long job = TOGETHER ? blockIdx.x : static_cast<long long>(blockIdx.x) * PIECE_WARPS + warp;
   const long long piece = job / p.unit_blocks;
   if (piece >= p.pieces) return;
   const Place at = Place::make<G>(p, static_cast<int>(job - piece * p.unit_blocks));
   const Rows rows(p);
   const long long lo = piece * p.piece, hi = lo + p.piece;
   long long u = rows.lower_bound(lo, at.lane);
   const bool teller = at.lane == 0 && (!TOGETHER || warp == 0) && job == piece * p.unit_blocks;
   long long begun = -1;
   Op op;
   if (u > 0) {  // the row before may reach into this piece
      const long long b = rows.begin(u - 1), e = rows.begin(u), fb = b - rows.first + ROW_ITEMS * (u - 1), fe = e - rows.first + ROW_ITEMS * u;
      if (fe > lo && fe - fb > p.row_limit) {
         long long e0 = b + (lo - fb - ROW_ITEMS), e1 = b + (hi - fb - ROW_ITEMS);
         e0 = e0 < b ? b : e0;
         e1 = e1 > e ? e : e1 < e0 ? e0 : e1;
         op.run(p, at, u - 1, e0, e1, TOGETHER ? warp : 0, TOGETHER ? PIECE_WARPS : 1);
         if (TOGETHER) join_warps<Op, G>(op, at, shared);
         if ((!TOGETHER || warp == 0) && at.edge_slot == 0) op.put(part_at<Op, G>(p, at, 2 * piece), at);
      }
   }
   for (; u < p.m; u++) {
      const long long b = rows.begin(u), fb = b - rows.first + ROW_ITEMS * u;
      if (fb >= hi) break;
      long long e = rows.begin(u + 1);
      const long long fe = e - rows.first + ROW_ITEMS * (u + 1);
      const bool cut = fe - fb > p.row_limit;
      if (cut) {
         const long long e1 = b + (hi - fb - ROW_ITEMS);
         e = e1 > e ? e : e1 < b ? b : e1;
         begun = u;
      }
      op.run(p, at, u, b, e, TOGETHER ? warp : 0, TOGETHER ? PIECE_WARPS : 1);
      if (TOGETHER) join_warps<Op, G>(op, at, shared);
      if (!TOGETHER || warp == 0) {
         if (!cut) op.finish(p, at, u);
         else if (at.edge_slot == 0) op.put(part_at<Op, G>(p, at, 2 * piece + 1), at);
      }
      if (cut) break;  // it reaches beyond this piece
   }
   if (teller) p.long_row[piece] = begun;
}

// The parts of the long rows that begin in this block's pieces; a row's parts go to the warps in runs, joined in order.
template <typename Op, int G>
__global__ void __launch_bounds__(PIECE_WARPS * 32) join_kernel(const AttnParams p)
{
   extern __shared__ __align__(16) float shared[];
   const int warp = threadIdx.x >> 5;
   const long long group = blockIdx.x / p.unit_blocks;
   const Place at = Place::make<G>(p, static_cast<int>(blockIdx.x - group * p.unit_blocks));
   const Rows rows(p);
   Op op;
   for (long long piece = group * JOIN_PIECES; piece < (group + 1) * JOIN_PIECES && piece < p.pieces; piece++) {
      const long long u = p.long_row[piece];
      if (u < 0) continue;
      const long long last = (rows.items(u + 1) - 1) / p.piece, parts = last - piece + 1;
      const long long each = (parts + PIECE_WARPS - 1) / PIECE_WARPS;
      Op::clear(op.s);
      for (long long i = warp * each; i < (warp + 1) * each && i < parts; i++)
         op.join_from(part_at<Op, G>(p, at, 2 * (piece + i) + (i == 0 ? 1 : 0)), at);
      join_warps<Op, G>(op, at, shared);
      if (warp == 0) op.finish(p, at, u);
   }
}

// ---------------------------------------------------------------------------------------------------------------------
// launchers: one instantiation per walk, storage type, slot, vectors of a lane, heads of a unit
// ---------------------------------------------------------------------------------------------------------------------
struct WalkShape {
   int g = 0, nv = 0, qb = 1;
   bool vector = true, together = false;
};

template <typename Op, int G>
int launch_op(const AttnParams &p, bool together, cudaStream_t st)
{
   const int bytes = (PIECE_WARPS - 1) * 32 * Op::LANE_FLOATS * static_cast<int>(sizeof(float));
   if (cudaFuncSetAttribute(join_kernel<Op, G>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return -1;
   const long long jobs = p.pieces * p.unit_blocks;
   if (together) {
      if (cudaFuncSetAttribute(walk_kernel<Op, G, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return -1;
      walk_kernel<Op, G, true><<<static_cast<unsigned>(jobs), PIECE_WARPS * 32, bytes, st>>>(p);
   } else {
      walk_kernel<Op, G, false><<<static_cast<unsigned>((jobs + PIECE_WARPS - 1) / PIECE_WARPS), PIECE_WARPS * 32, 0, st>>>(p);
   }
   const long long groups = (p.pieces + JOIN_PIECES - 1) / JOIN_PIECES;
   join_kernel<Op, G><<<static_cast<unsigned>(groups * p.unit_blocks), PIECE_WARPS * 32, bytes, st>>>(p);
   return 0;
}

template <typename T, int G, int NV, template <typename, int, int, int, bool> class Op, bool COLUMNS>
int launch_slot(const WalkShape &s, const AttnParams &p, cudaStream_t st)
{
   if (!s.vector) return launch_op<Op<T, G, NV, 1, false>, G>(p, s.together, st);
   if constexpr (!COLUMNS) {
      if (s.qb == 4) return launch_op<Op<T, G, NV, 4, true>, G>(p, s.together, st);
      if (s.qb == 2) return launch_op<Op<T, G, NV, 2, true>, G>(p, s.together, st);
   }
   return launch_op<Op<T, G, NV, 1, true>, G>(p, s.together, st);
}

// -1: no such instantiation
template <typename T, template <typename, int, int, int, bool> class Op, bool COLUMNS>
int launch_walk(const WalkShape &s, const AttnParams &p, cudaStream_t st)
{
   if (s.nv == 1) {
      if (s.g == 4) return launch_slot<T, 4, 1, Op, COLUMNS>(s, p, st);
      if (s.g == 8) return launch_slot<T, 8, 1, Op, COLUMNS>(s, p, st);
      if (s.g == 16) return launch_slot<T, 16, 1, Op, COLUMNS>(s, p, st);
      if (s.g == 32) return launch_slot<T, 32, 1, Op, COLUMNS>(s, p, st);
   }
   if constexpr (sizeof(T) == 4)
      if (s.nv == 2 && s.g == 32) return launch_slot<T, 32, 2, Op, COLUMNS>(s, p, st);
   return -1;
}

#define FMM_DECLARE_WALKS(NAME)                                                        \
   int walk_forward_##NAME(const WalkShape &, const AttnParams &, cudaStream_t);       \
   int walk_rows_##NAME(const WalkShape &, const AttnParams &, cudaStream_t);          \
   int walk_columns_##NAME(const WalkShape &, const AttnParams &, cudaStream_t);
FMM_DECLARE_WALKS(f32)
FMM_DECLARE_WALKS(bf16)
FMM_DECLARE_WALKS(f16)

}  // namespace attn
}  // namespace fmm

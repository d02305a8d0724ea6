// diff_attn.cuh -- differential attention over the edges of a CSR, forward and backward (include/fusedmm_b200.h,
// fusedmm_b200_diff_attention).
//
//   s^c_e = scale q^c_u . k^c_v + bias_e (c = 0, 1);  p^c = softmax over the edges e = (u, v) of row u;
//   o_u = sum_e (p^0_e - lam p^1_e) v_v
//   backward, with dP_e = do_u . v_v, D^c_u = sum_e p^c_e dP_e:  ds^0 = p^0 (dP - D^0), ds^1 = -lam p^1 (dP - D^1),
//   dq^c_u = scale sum_e ds^c k^c_v, dk^c_v = scale sum_e ds^c q^c_u, dv_v = sum_e (p^0 - lam p^1) do_u, dlam_u = -D^1_u.
//   The backward walks form p as exp(s - lse) / Z, where Z is the sum of these exponentials over the row, 1 but for rounding:
//   lse is one 32-bit number, and next to a score of a mask's size (-1e9) the logarithm of the sum vanishes in it.
//
// Three walks of the same shape: the forward and the dq pass go over the rows and gather k and v; the dk, dv pass goes over
// the columns of the transposed pattern and gathers q and do.  No atomics: every sum is taken in a fixed order.
//
// The gathered rows decide the layout.  A slot of G lanes takes one head of one edge, NV vectors of 16 bytes to a lane; its
// two halves hold the two maps' parts of k (or q), so the two dots are one butterfly of G/2 lanes and each half owns the
// running maximum and sum of its map; v (or do) lies over all G lanes.  The slots of a warp take neighbouring heads of the
// same edge, as far as there are heads (their rows are adjacent in memory and all slots run in step), and alternate edges
// beyond that, joined at the row's end.  QB query heads that share a kv head are computed together from one load.
//
// Work is cut at equal parts ("pieces") of the items nnz + ROW_ITEMS * m, so that hub rows, single long rows of a decoding
// step and empty rows are spread alike, without a pass over the pattern: a warp finds its first row by a 32-ary search in
// the row pointers.  A row of up to `row_limit` items belongs to the piece it begins in; a longer one is cut at the pieces'
// borders, its parts go to `partial` and a second launch joins them in order.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "attn_common.cuh"

namespace fmm {
namespace attn {

constexpr int ROW_ITEMS = 8;        // what a row costs beside its edges, in edges
constexpr int PIECE_WARPS = 4;      // warps of a block whose warps have pieces of their own
constexpr int JOINT_WARPS = 8;      // warps of a block that share a row

struct AttnParams {
   const void *rowptr, *colidx;  // row walks: the pattern; column walk: the transposed one (colidx: 32-bit row ids)
   int ptr64, idx64;
   long long m, n, nnz;          // rows walked, rows that can be gathered, length of colidx
   const float *bias;            // column walk: in the order of the transposed pattern
   const void *q, *k, *v, *dout;
   const float *lam;
   long long ldq, hsq, ldk, hsk, ldv, hsv, ldo, hso, ldlam;
   void *out;                    // forward [m,H,Dv]; dq [m,H,2,D]; dk [n,Hk,2,D]
   void *out2;                   // dv [n,Hk,Dv]
   float *lse;                   // [m,H,2]
   float4 *stats;                // [m,H,2]: lse and D of a map, its factor in the weight (1 / Z or -lam / Z)
   float *dlam;                  // [m,H]
   int heads, kv_heads, group, d, dv, step;
   float scale;
   int units, unit_blocks, slot_heads;  // head units of QB heads; warps (blocks) that share them; slots of a warp across units
   // the walks on the matrix units: kv heads of a unit, query heads of each of them, units that share a kv head
   int unit_kv, unit_heads, head_blocks;
   // the groups of heads that a unit takes one after the other, and the heads of a group for one kv head (log2)
   int subs, kv_log2;
   // the two gathered arrays (k and v, or q and do; packed copies of them where they are no vectors): bytes from row to row and
   // from head to head, elements of a row (of one map for the first)
   const char *a, *b;
   unsigned a_stride, b_stride;
   long long a_head, b_head;
   int a_width, b_width;
   long long piece, row_limit, pieces;
   int join_rows, join_pieces;   // a joining block looks after one row, or after so many pieces
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
   // first row u in [lo, hi) with items(u) >= at, or hi; the whole warp takes part
   __device__ __forceinline__ long long lower_bound(long long at, long long lo, long long hi, int lane) const
   {
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

// a vector of 2N floats of scratch, 16 bytes at a time
template <int N>
__device__ __forceinline__ void put_pairs(float *p, const F2 (&f)[N])
{
#pragma unroll
   for (int i = 0; i < N; i += 2) *reinterpret_cast<ulonglong2 *>(p + 2 * i) = make_ulonglong2(f[i], f[i + 1]);
}
template <int N>
__device__ __forceinline__ void get_pairs(const float *p, F2 (&f)[N])
{
#pragma unroll
   for (int i = 0; i < N; i += 2) {
      const ulonglong2 a = *reinterpret_cast<const ulonglong2 *>(p + 2 * i);
      f[i] = a.x;
      f[i + 1] = a.y;
   }
}
// exp(score - lse).  No score is above lse but for rounding, which next to a mask's size may be a power of thousands.
__device__ __forceinline__ float weight_of(float score, float lse) { return exp2_fast(min_or_nan(score - lse, 0.0f) * LOG2E); }
// The weight from which on an edge is the next reference: so many times what had come in when the last was set, and a part of the row's
// whole (1 but for rounding) that leaves little to the others.
constexpr float REFERENCE_GROWTH = 4.0f, REFERENCE_LEAST = 0.25f;
__device__ __forceinline__ float reference_mark(float total) { return fmaxf(REFERENCE_GROWTH * total, REFERENCE_LEAST); }
// Where sums with two references join: what each side's sums lack, in units of the sums of its weights.  `ref` becomes the heavier's.
__device__ __forceinline__ void join_references(float total, float &ref, float total_o, float ref_o, float &shift, float &shift_o)
{
   const bool other = total_o > total;
   shift = other ? ref - ref_o : 0.0f;
   shift_o = other ? 0.0f : ref_o - ref;
   ref = other ? ref_o : ref;
}
// 1 / Z; a row of no weights has no gradient
__device__ __forceinline__ float reciprocal_total(float total) { return total == 0.0f ? 0.0f : 1.0f / total; }
__device__ __forceinline__ F2 shfl_xor_pair(F2 v, int x) { return __shfl_xor_sync(FULL, v, x); }

// 32 edges, one to a lane, fetched ahead: the ids of a row's next 32 edges, or of the next row's first, are under way while
// the present ones are worked on (edges of neighbouring rows are neighbours).
struct EdgeStream {
   long long at = -1;
   int low = 0, high = 0;  // as loaded: a use would wait for the load
   float bias = 0.0f;
   __device__ __forceinline__ void fetch(const AttnParams &p, long long from, int lane)
   {
      at = from;
      const long long e = from + lane;
      if (e < p.nnz) {
         if (p.idx64) {
            const int2 v = __ldg(static_cast<const int2 *>(p.colidx) + e);
            low = v.x;
            high = v.y;
         } else {
            low = __ldg(static_cast<const int *>(p.colidx) + e);
         }
         if (p.bias) bias = __ldg(p.bias + e);
      }
   }
   // the id to gather, -1 for an edge that is none: behind the end, outside [0, n), or masked
   __device__ __forceinline__ int take(const AttnParams &p, long long from, long long end, int lane)
   {
      if (at != from) fetch(p, from, lane);
      const bool inside = static_cast<unsigned>(low) < static_cast<unsigned>(p.n) && (!p.idx64 || high == 0);
      return from + lane < end && inside && bias != -INFINITY ? low : -1;
   }
};

// Rows of one gathered array as a slot's lanes hold them: vector t of a lane is SKIP elements behind vector t - 1.
// EXACT: the lanes' vectors cover the row and nothing else; RAGGED: vectors, some lanes past the row's end; PIECES: the walk's
// own rows and its results are no vectors (what is gathered has been packed then).  Edges that are none read zeros from
// `zero_row`, so that nothing of theirs is touched and no lane needs a branch.
enum Form { PIECES = 0, RAGGED = 1, EXACT = 2 };
static __device__ __align__(16) uint4 zero_row[64];

template <typename T, int NV, int FORM>
struct Gather {
   const char *base;
   unsigned stride;  // bytes
   int left;         // elements from the lane's first vector to the row's end
   template <int SKIP>
   __device__ __forceinline__ void load(int id, uint4 (&r)[NV]) const
   {
      const T *row = reinterpret_cast<const T *>(base + static_cast<unsigned long long>(static_cast<unsigned>(id)) * stride);
      const T *zero = reinterpret_cast<const T *>(zero_row);
      if (FORM == EXACT && id < 0) row = zero;
#pragma unroll
      for (int t = 0; t < NV; t++) r[t] = ldg16(FORM == EXACT || (id >= 0 && left > t * SKIP) ? row + t * SKIP : zero);
   }
};
// the part of a lane that begins at element x: of the first array at a head and map, of the second at a head
template <typename T, int NV, int FORM>
__device__ __forceinline__ Gather<T, NV, FORM> gather_a(const AttnParams &p, int head, int map, int x)
{
   return {p.a + head * p.a_head + static_cast<long long>(map * p.a_width + x) * static_cast<long long>(sizeof(T)), p.a_stride, p.a_width - x};
}
template <typename T, int NV, int FORM>
__device__ __forceinline__ Gather<T, NV, FORM> gather_b(const AttnParams &p, int head, int x)
{
   return {p.b + head * p.b_head + static_cast<long long>(x) * static_cast<long long>(sizeof(T)), p.b_stride, p.b_width - x};
}

// a row of the walk itself, likewise
template <typename T, int NV, int FORM, int SKIP>
__device__ __forceinline__ void load_own(const AttnParams &p, const void *array, long long offset, int x, int width, F2 (&f)[NV][Elt<T>::W / 2])
{
   const T *src = static_cast<const T *>(array) + offset + x;
#pragma unroll
   for (int t = 0; t < NV; t++) unpack_pairs<T>(ld_row<T, FORM != PIECES>(src + t * SKIP, width - x - t * SKIP, p.step), f[t]);
}

template <int N>
__device__ __forceinline__ void unpair(const F2 (&f)[N], float (&o)[2 * N])
{
#pragma unroll
   for (int i = 0; i < N; i++) {
      const float2 a = f2_parts(f[i]);
      o[2 * i] = a.x;
      o[2 * i + 1] = a.y;
   }
}

// ---------------------------------------------------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------------------------------------------------
// U: edges of a slot on their way at once; BLOCKS: of an SM.  Float with U = 4 and three blocks against U = 2 and four, all walks
// with their joins: 313729 R-MAT edges with 2 heads of d 40 403 us and 447, 425984 with 4 heads of d 32 475 and 464.  Forward of the
// latter: 104 us, 8.4 TB/s of gathered rows, most from L2.
template <typename T, int G, int NV, int QB, int FORM>
struct Forward {
   static constexpr int W = Elt<T>::W, P = W / 2, U = W == 4 && QB == 1 ? 4 : 2, BLOCKS = W == 4 ? (QB > 2 ? 2 : 3) : QB * NV * W > 16 ? 2 : 4;
   static constexpr int KSKIP = (G / 2) * W, VSKIP = G * W;
   static constexpr int LANE_FLOATS = QB * (2 * NV * W + 2);  // partial state of a lane
   struct State {
      F2 acc[QB][2][NV][P];    // sums of p v for the two maps
      float top[QB], sum[QB];  // of this half's map
   };
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
               for (int j = 0; j < P; j++) s.acc[b][c][t][j] = 0;
      }
   }

   __device__ __forceinline__ void run(const AttnParams &p, const Place &at, EdgeStream &edges, long long row, long long e0, long long e1,
                                       int warp, int warps)
   {
      clear(s);
      if (e0 + 32 * warp >= e1) return;
      const int kv = at.unit / (p.group / QB), head0 = at.unit * QB;
      const int x = at.in_half * W, y = at.in_slot * W;
      const Gather<T, NV, FORM> kg = gather_a<T, NV, FORM>(p, kv, at.half, x), vg = gather_b<T, NV, FORM>(p, kv, y);
      F2 q[QB][NV][P];
#pragma unroll
      for (int b = 0; b < QB; b++)
         load_own<T, NV, FORM, KSKIP>(p, p.q, row * p.ldq + (head0 + b) * p.hsq + at.half * p.d, x, p.d, q[b]);
      for (long long base = e0 + 32 * warp; base < e1; base += 32 * warps) {
         const int my_id = edges.take(p, base, e1, at.lane);
         const float my_bias = edges.bias;
         edges.fetch(p, base + 32 * warps < e1 ? base + 32 * warps : e1 + 32 * warp, at.lane);
         const int count = static_cast<int>(e1 - base < 32 ? e1 - base : 32);
         for (int first = 0; first < count; first += U * at.edge_slots) {
            int id[U];
            uint4 kr[U][NV], vr[U][NV];
#pragma unroll
            for (int i = 0; i < U; i++) {
               id[i] = __shfl_sync(FULL, my_id, first + i * at.edge_slots + at.edge_slot);
               kg.template load<KSKIP>(id[i], kr[i]);
               vg.template load<VSKIP>(id[i], vr[i]);
            }
            float score[QB][U];
#pragma unroll
            for (int i = 0; i < U; i++) {
               F2 k[NV][P];
#pragma unroll
               for (int t = 0; t < NV; t++) unpack_pairs<T>(kr[i][t], k[t]);
               const float bias = p.bias ? __shfl_sync(FULL, my_bias, first + i * at.edge_slots + at.edge_slot) : 0.0f;
#pragma unroll
               for (int b = 0; b < QB; b++) {
                  F2 dot = 0;
#pragma unroll
                  for (int t = 0; t < NV; t++)
#pragma unroll
                     for (int j = 0; j < P; j++) dot = fma2(q[b][t][j], k[t][j], dot);
                  const float all = add_over<G / 2>(sum2(dot));
                  score[b][i] = id[i] >= 0 ? fmaf(all, p.scale, bias) : -INFINITY;
               }
            }
            F2 v[U][NV][P];
#pragma unroll
            for (int i = 0; i < U; i++)
#pragma unroll
               for (int t = 0; t < NV; t++) unpack_pairs<T>(vr[i][t], v[i][t]);
#pragma unroll
            for (int b = 0; b < QB; b++) {
               float top = s.top[b];
#pragma unroll
               for (int i = 0; i < U; i++) top = fmaxf(top, score[b][i]);
               // a row that has met no edge yet has the maximum -inf: its differences are taken from 0
               const float ref = top == -INFINITY ? 0.0f : top;
               if (__any_sync(FULL, top != s.top[b])) {
                  const float mine = exp2_fast((s.top[b] - ref) * LOG2E), other = __shfl_xor_sync(FULL, mine, G / 2);
                  const float c0 = at.half ? other : mine, c1 = at.half ? mine : other;
                  const F2 f0 = f2(c0, c0), f1 = f2(c1, c1);
                  s.sum[b] *= mine;
#pragma unroll
                  for (int t = 0; t < NV; t++)
#pragma unroll
                     for (int j = 0; j < P; j++) {
                        s.acc[b][0][t][j] = mul2(s.acc[b][0][t][j], f0);
                        s.acc[b][1][t][j] = mul2(s.acc[b][1][t][j], f1);
                     }
                  s.top[b] = top;
               }
#pragma unroll
               for (int i = 0; i < U; i++) {
                  // the difference is taken before the factor: scores near the type's largest numbers keep their order
                  const float mine = exp2_fast((score[b][i] - ref) * LOG2E), other = __shfl_xor_sync(FULL, mine, G / 2);
                  const float w0 = at.half ? other : mine, w1 = at.half ? mine : other;
                  const F2 p0 = f2(w0, w0), p1 = f2(w1, w1);
                  s.sum[b] += mine;
#pragma unroll
                  for (int t = 0; t < NV; t++)
#pragma unroll
                     for (int j = 0; j < P; j++) {
                        s.acc[b][0][t][j] = fma2(p0, v[i][t][j], s.acc[b][0][t][j]);
                        s.acc[b][1][t][j] = fma2(p1, v[i][t][j], s.acc[b][1][t][j]);
                     }
               }
            }
         }
      }
      for (int x2 = G * p.slot_heads; x2 < 32; x2 <<= 1) {  // the slots that took alternate edges
         State o;
#pragma unroll
         for (int b = 0; b < QB; b++) {
            o.top[b] = __shfl_xor_sync(FULL, s.top[b], x2);
            o.sum[b] = __shfl_xor_sync(FULL, s.sum[b], x2);
#pragma unroll
            for (int c = 0; c < 2; c++)
#pragma unroll
               for (int t = 0; t < NV; t++)
#pragma unroll
                  for (int j = 0; j < P; j++) o.acc[b][c][t][j] = shfl_xor_pair(s.acc[b][c][t][j], x2);
         }
         join(s, o, at, (at.lane & x2) != 0);
      }
   }

   // joins the state of other edges of the row; `swap`: the other's edges come first (both sides of an exchange then add
   // in the same order)
   static __device__ __forceinline__ void join(State &s, const State &o, const Place &at, bool swap)
   {
#pragma unroll
      for (int b = 0; b < QB; b++) {
         const float top = fmaxf(s.top[b], o.top[b]), ref = top == -INFINITY ? 0.0f : top;
         float fs = exp2_fast((s.top[b] - ref) * LOG2E), fo = exp2_fast((o.top[b] - ref) * LOG2E);
         // a NaN score leaves its trace in the sum and the accumulators, the maximum skips it
         const float a = s.sum[b] * fs, c = o.sum[b] * fo;
         s.sum[b] = swap ? c + a : a + c;
         s.top[b] = top;
         const float fs2 = __shfl_xor_sync(FULL, fs, G / 2), fo2 = __shfl_xor_sync(FULL, fo, G / 2);
#pragma unroll
         for (int m = 0; m < 2; m++) {
            const float g1 = m == at.half ? fs : fs2, g2 = m == at.half ? fo : fo2;
            const F2 f1 = f2(g1, g1), f2_ = f2(g2, g2);
#pragma unroll
            for (int t = 0; t < NV; t++)
#pragma unroll
               for (int j = 0; j < P; j++) {
                  const F2 x = mul2(s.acc[b][m][t][j], f1), y = mul2(o.acc[b][m][t][j], f2_);
                  s.acc[b][m][t][j] = add2(x, y);
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
            for (int t = 0; t < NV; t++) get_pairs<P>(from + ((b * 2 + c) * NV + t) * W * G, o.acc[b][c][t]);
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
            for (int t = 0; t < NV; t++) put_pairs<P>(to + ((b * 2 + c) * NV + t) * W * G, s.acc[b][c][t]);
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
            float a[W], c[W];
            unpair(s.acc[b][0][t], a);
            unpair(s.acc[b][1][t], c);
#pragma unroll
            for (int j = 0; j < W; j++) a[j] = a[j] * f0 - c[j] * f1;
            st_row<T, FORM != PIECES>(static_cast<T *>(p.out) + (row * p.heads + head) * p.dv + y, a, p.dv - y);
         }
         if (at.in_half == 0 && p.lse) p.lse[(row * p.heads + head) * 2 + at.half] = s.top[b] + LN2 * log2f(s.sum[b]);
      }
   }
};

// ---------------------------------------------------------------------------------------------------------------------
// backward over the rows: dq, dlam and the numbers the columns need.  With D^c unknown until the row's end, the sums
// A = sum p (dP - c) k, B = sum p k, D' = sum p (dP - c), D = sum p dP and Z = sum p are taken together, of p before the division by
// Z; dq = scale (A - D' B / Z) / Z.  With c = 0 A and D' B would be large and nearly equal where values have a mean, or where one edge
// has nearly all the weight.  So the reference c is the dP of one of the first edges, and of every later one that is heavy against all
// before it (reference_mark); D is kept too, as c + D' loses digits where dP has no mean.  Another reference: A += (c - c') B,
// D' += (c - c') Z; where sums join, the heavier side's stays.  425984 R-MAT edges in float, 4 heads of d 32: 122 us, 118 with c = 0
// and without Z.
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int G, int NV, int QB, int FORM>
struct BackwardRows {
   static constexpr int W = Elt<T>::W, P = W / 2, U = W == 4 && QB == 1 ? 4 : 2, BLOCKS = W == 4 ? (QB > 2 ? 2 : 3) : QB * NV * W > 16 ? 2 : 4;
   static constexpr int KSKIP = (G / 2) * W, VSKIP = G * W;
   static constexpr int LANE_FLOATS = QB * (2 * NV * W + 4);
   struct State {
      F2 a[QB][NV][P], b[QB][NV][P];  // of this half's map
      float delta[QB], total[QB], rest[QB], ref[QB];  // D, Z, D', c
   };
   State s;

   static __device__ __forceinline__ void clear(State &s)
   {
#pragma unroll
      for (int b = 0; b < QB; b++) {
         s.delta[b] = s.total[b] = s.rest[b] = s.ref[b] = 0.0f;
#pragma unroll
         for (int t = 0; t < NV; t++)
#pragma unroll
            for (int j = 0; j < P; j++) s.a[b][t][j] = s.b[b][t][j] = 0;
      }
   }

   // the heaviest of some edges, which are in no sum yet, becomes the reference where it is heavy enough
   __device__ __forceinline__ void rebase(float (&mark)[QB], const float (&pr)[U][QB], const float (&dp)[U][QB])
   {
#pragma unroll
      for (int b = 0; b < QB; b++) {
         float most = mark[b], ref = s.ref[b], total = s.total[b];
#pragma unroll
         for (int i = 0; i < U; i++) {
            const bool heavy = pr[i][b] > most && fabsf(dp[i][b]) < INFINITY;
            ref = heavy ? dp[i][b] : ref;
            most = heavy ? pr[i][b] : most;
            total += pr[i][b];
         }
         if (most > mark[b]) mark[b] = reference_mark(total);
         const float shift = s.ref[b] - ref;
         const F2 ss = f2(shift, shift);
#pragma unroll
         for (int t = 0; t < NV; t++)
#pragma unroll
            for (int j = 0; j < P; j++) s.a[b][t][j] = fma2(ss, s.b[b][t][j], s.a[b][t][j]);
         s.rest[b] = fmaf(shift, s.total[b], s.rest[b]);
         s.ref[b] = ref;
      }
   }

   __device__ __forceinline__ void run(const AttnParams &p, const Place &at, EdgeStream &edges, long long row, long long e0, long long e1,
                                       int warp, int warps)
   {
      clear(s);
      if (e0 + 32 * warp >= e1) return;
      const int kv = at.unit / (p.group / QB), head0 = at.unit * QB;
      const int x = at.in_half * W, y = at.in_slot * W;
      const Gather<T, NV, FORM> kg = gather_a<T, NV, FORM>(p, kv, at.half, x), vg = gather_b<T, NV, FORM>(p, kv, y);
      F2 q[QB][NV][P], dout[QB][NV][P];
      float lse[QB], mark[QB];
#pragma unroll
      for (int b = 0; b < QB; b++) {
         mark[b] = 0.0f;
         lse[b] = __ldg(p.lse + (row * p.heads + head0 + b) * 2 + at.half);
         load_own<T, NV, FORM, KSKIP>(p, p.q, row * p.ldq + (head0 + b) * p.hsq + at.half * p.d, x, p.d, q[b]);
         load_own<T, NV, FORM, VSKIP>(p, p.dout, row * p.ldo + (head0 + b) * p.hso, y, p.dv, dout[b]);
      }
      for (long long base = e0 + 32 * warp; base < e1; base += 32 * warps) {
         const int my_id = edges.take(p, base, e1, at.lane);
         const float my_bias = edges.bias;
         edges.fetch(p, base + 32 * warps < e1 ? base + 32 * warps : e1 + 32 * warp, at.lane);
         const int count = static_cast<int>(e1 - base < 32 ? e1 - base : 32);
         for (int first = 0; first < count; first += U * at.edge_slots) {
            int id[U];
            uint4 kr[U][NV], vr[U][NV];
#pragma unroll
            for (int i = 0; i < U; i++) {
               id[i] = __shfl_sync(FULL, my_id, first + i * at.edge_slots + at.edge_slot);
               kg.template load<KSKIP>(id[i], kr[i]);
               vg.template load<VSKIP>(id[i], vr[i]);
            }
            float pr[U][QB], dp[U][QB];
            bool grown = false;
#pragma unroll
            for (int i = 0; i < U; i++) {
               F2 k[NV][P], v[NV][P];
#pragma unroll
               for (int t = 0; t < NV; t++) {
                  unpack_pairs<T>(kr[i][t], k[t]);
                  unpack_pairs<T>(vr[i][t], v[t]);
               }
               const float bias = p.bias ? __shfl_sync(FULL, my_bias, first + i * at.edge_slots + at.edge_slot) : 0.0f;
#pragma unroll
               for (int b = 0; b < QB; b++) {
                  F2 dots = 0, dps = 0;
#pragma unroll
                  for (int t = 0; t < NV; t++)
#pragma unroll
                     for (int j = 0; j < P; j++) {
                        dots = fma2(q[b][t][j], k[t][j], dots);
                        dps = fma2(dout[b][t][j], v[t][j], dps);
                     }
                  const float dot = add_over<G / 2>(sum2(dots));
                  dp[i][b] = add_over<G>(sum2(dps));
                  // an edge that is masked has p = 0, and so has a row without edges (its lse is -inf)
                  pr[i][b] = id[i] >= 0 && lse[b] != -INFINITY ? weight_of(fmaf(dot, p.scale, bias), lse[b]) : 0.0f;
                  grown |= pr[i][b] > mark[b];
               }
            }
            if (grown) rebase(mark, pr, dp);
#pragma unroll
            for (int i = 0; i < U; i++) {
               F2 k[NV][P];
#pragma unroll
               for (int t = 0; t < NV; t++) unpack_pairs<T>(kr[i][t], k[t]);
#pragma unroll
               for (int b = 0; b < QB; b++) {
                  const float w = pr[i][b] * (dp[i][b] - s.ref[b]);
                  const F2 ww = f2(w, w), pp = f2(pr[i][b], pr[i][b]);
                  s.rest[b] += w;
                  s.delta[b] = fmaf(pr[i][b], dp[i][b], s.delta[b]);
                  s.total[b] += pr[i][b];
#pragma unroll
                  for (int t = 0; t < NV; t++)
#pragma unroll
                     for (int j = 0; j < P; j++) {
                        s.a[b][t][j] = fma2(ww, k[t][j], s.a[b][t][j]);
                        s.b[b][t][j] = fma2(pp, k[t][j], s.b[b][t][j]);
                     }
               }
            }
         }
      }
      for (int x2 = G * p.slot_heads; x2 < 32; x2 <<= 1) {
#pragma unroll
         for (int b = 0; b < QB; b++) {
            const float delta = __shfl_xor_sync(FULL, s.delta[b], x2), total = __shfl_xor_sync(FULL, s.total[b], x2);
            F2 a[NV][P], c[NV][P];
            const float rest = __shfl_xor_sync(FULL, s.rest[b], x2), ref = __shfl_xor_sync(FULL, s.ref[b], x2);
#pragma unroll
            for (int t = 0; t < NV; t++)
#pragma unroll
               for (int j = 0; j < P; j++) {
                  a[t][j] = shfl_xor_pair(s.a[b][t][j], x2);
                  c[t][j] = shfl_xor_pair(s.b[b][t][j], x2);
               }
            add(s, b, a, c, make_float4(delta, total, rest, ref));
         }
      }
   }
   // adds the sums of other edges
   static __device__ __forceinline__ void add(State &s, int b, const F2 (&a)[NV][P], const F2 (&c)[NV][P], float4 o)
   {
      float shift, shift_o;
      join_references(s.total[b], s.ref[b], o.y, o.w, shift, shift_o);
      const F2 ss = f2(shift, shift), so = f2(shift_o, shift_o);
#pragma unroll
      for (int t = 0; t < NV; t++)
#pragma unroll
         for (int j = 0; j < P; j++) {
            s.a[b][t][j] = add2(fma2(ss, s.b[b][t][j], s.a[b][t][j]), fma2(so, c[t][j], a[t][j]));
            s.b[b][t][j] = add2(s.b[b][t][j], c[t][j]);
         }
      s.delta[b] += o.x;
      s.rest[b] = fmaf(shift, s.total[b], s.rest[b]) + fmaf(shift_o, o.y, o.z);
      s.total[b] += o.y;
   }
   __device__ __forceinline__ void join_from(const float *unit, const Place &at)
   {
      const float *from = unit + at.in_slot * W;
#pragma unroll
      for (int b = 0; b < QB; b++) {
         F2 x[2][NV][P];  // all loads before the first sum
#pragma unroll
         for (int t = 0; t < NV; t++) {
            get_pairs<P>(from + (b * 2 * NV + t) * W * G, x[0][t]);
            get_pairs<P>(from + ((b * 2 + 1) * NV + t) * W * G, x[1][t]);
         }
         add(s, b, x[0], x[1], *reinterpret_cast<const float4 *>(unit + QB * 2 * NV * W * G + (b * G + at.in_slot) * 4));
      }
   }
   __device__ __forceinline__ void put(float *unit, const Place &at) const
   {
      float *to = unit + at.in_slot * W;
#pragma unroll
      for (int b = 0; b < QB; b++) {
#pragma unroll
         for (int t = 0; t < NV; t++) {
            put_pairs<P>(to + (b * 2 * NV + t) * W * G, s.a[b][t]);
            put_pairs<P>(to + ((b * 2 + 1) * NV + t) * W * G, s.b[b][t]);
         }
         *reinterpret_cast<float4 *>(unit + QB * 2 * NV * W * G + (b * G + at.in_slot) * 4) = make_float4(s.delta[b], s.total[b], s.rest[b], s.ref[b]);
      }
   }

   __device__ __forceinline__ void finish(const AttnParams &p, const Place &at, long long row)
   {
      if (at.edge_slot != 0) return;
#pragma unroll
      for (int b = 0; b < QB; b++) {
         const int head = at.unit * QB + b;
         const long long rh = row * p.heads + head;
         const float inverse = reciprocal_total(s.total[b]), delta = s.delta[b] * inverse, rest = s.rest[b] * inverse;
         const float sign = (at.half ? -__ldg(p.lam + row * p.ldlam + head) : 1.0f) * inverse, factor = sign * p.scale;
#pragma unroll
         for (int t = 0; t < NV; t++) {
            const int x = (at.in_half + (G / 2) * t) * W;
            float a[W], c[W];
            unpair(s.a[b][t], a);
            unpair(s.b[b][t], c);
#pragma unroll
            for (int j = 0; j < W; j++) a[j] = factor * fmaf(-rest, c[j], a[j]);
            st_row<T, FORM != PIECES>(static_cast<T *>(p.out) + (rh * 2 + at.half) * p.d + x, a, p.d - x);
         }
         if (at.in_half == 0) {
            p.stats[rh * 2 + at.half] = make_float4(__ldg(p.lse + rh * 2 + at.half), delta, sign, 0.0f);
            if (at.half == 1) p.dlam[rh] = -delta;
         }
      }
   }
};

// ---------------------------------------------------------------------------------------------------------------------
// backward over the columns: dk and dv.  A unit is a kv head; every edge counts once for each query head of its group.
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int G, int NV, int QB, int FORM>
struct BackwardColumns {
   static constexpr int W = Elt<T>::W, P = W / 2, U = W == 4 ? 4 : 2, BLOCKS = 3;
   static constexpr int KSKIP = (G / 2) * W, VSKIP = G * W;
   static constexpr int LANE_FLOATS = 2 * NV * W;
   struct State {
      F2 dk[NV][P], dv[NV][P];
   };
   State s;

   static __device__ __forceinline__ void clear(State &s)
   {
#pragma unroll
      for (int t = 0; t < NV; t++)
#pragma unroll
         for (int j = 0; j < P; j++) s.dk[t][j] = s.dv[t][j] = 0;
   }

   __device__ __forceinline__ void run(const AttnParams &p, const Place &at, EdgeStream &edges, long long col, long long e0, long long e1,
                                       int warp, int warps)
   {
      clear(s);
      if (e0 + 32 * warp >= e1) return;
      const int kv = at.unit;
      const int x = at.in_half * W, y = at.in_slot * W;
      F2 k[NV][P], v[NV][P];
      load_own<T, NV, FORM, KSKIP>(p, p.k, col * p.ldk + kv * p.hsk + at.half * p.d, x, p.d, k);
      load_own<T, NV, FORM, VSKIP>(p, p.v, col * p.ldv + kv * p.hsv, y, p.dv, v);
      for (long long base = e0 + 32 * warp; base < e1; base += 32 * warps) {
         const int my_id = edges.take(p, base, e1, at.lane);
         const float my_bias = edges.bias;
         edges.fetch(p, base + 32 * warps < e1 ? base + 32 * warps : e1 + 32 * warp, at.lane);
         const int count = static_cast<int>(e1 - base < 32 ? e1 - base : 32);
         for (int first = 0; first < count; first += U * at.edge_slots) {
            int id[U];
            float bias[U];
#pragma unroll
            for (int i = 0; i < U; i++) {
               id[i] = __shfl_sync(FULL, my_id, first + i * at.edge_slots + at.edge_slot);
               bias[i] = p.bias ? __shfl_sync(FULL, my_bias, first + i * at.edge_slots + at.edge_slot) : 0.0f;
            }
            for (int g = 0; g < p.group; g++) {
               const int head = kv * p.group + g;
               const Gather<T, NV, FORM> qg = gather_a<T, NV, FORM>(p, head, at.half, x), dg = gather_b<T, NV, FORM>(p, head, y);
               uint4 qr[U][NV], dr[U][NV];
               float4 stat[U];
#pragma unroll
               for (int i = 0; i < U; i++) {
                  stat[i] = make_float4(-INFINITY, 0.0f, 0.0f, 0.0f);
                  if (id[i] >= 0) stat[i] = __ldg(p.stats + (static_cast<long long>(id[i]) * p.heads + head) * 2 + at.half);
                  qg.template load<KSKIP>(id[i], qr[i]);
                  dg.template load<VSKIP>(id[i], dr[i]);
               }
#pragma unroll
               for (int i = 0; i < U; i++) {
                  F2 q[NV][P], dout[NV][P], dots = 0, dps = 0;
#pragma unroll
                  for (int t = 0; t < NV; t++) {
                     unpack_pairs<T>(qr[i][t], q[t]);
                     unpack_pairs<T>(dr[i][t], dout[t]);
#pragma unroll
                     for (int j = 0; j < P; j++) {
                        dots = fma2(q[t][j], k[t][j], dots);
                        dps = fma2(dout[t][j], v[t][j], dps);
                     }
                  }
                  const float dot = add_over<G / 2>(sum2(dots)), dp = add_over<G>(sum2(dps));
                  const bool live = stat[i].x != -INFINITY;  // an edge, and of a row that has any
                  const float pr = live ? weight_of(fmaf(dot, p.scale, bias[i]), stat[i].x) : 0.0f;
                  const float mine = live ? stat[i].z * pr : 0.0f;  // this map's part of the weight
                  const float w = mine + __shfl_xor_sync(FULL, mine, G / 2);
                  const float ds = live ? mine * (dp - stat[i].y) : 0.0f;
                  const F2 ww = f2(w, w), dd = f2(ds, ds);
#pragma unroll
                  for (int t = 0; t < NV; t++)
#pragma unroll
                     for (int j = 0; j < P; j++) {
                        s.dk[t][j] = fma2(dd, q[t][j], s.dk[t][j]);
                        s.dv[t][j] = fma2(ww, dout[t][j], s.dv[t][j]);
                     }
               }
            }
         }
      }
      for (int x2 = G * p.slot_heads; x2 < 32; x2 <<= 1) {
#pragma unroll
         for (int t = 0; t < NV; t++)
#pragma unroll
            for (int j = 0; j < P; j++) {
               s.dk[t][j] = add2(s.dk[t][j], shfl_xor_pair(s.dk[t][j], x2));
               s.dv[t][j] = add2(s.dv[t][j], shfl_xor_pair(s.dv[t][j], x2));
            }
      }
   }
   __device__ __forceinline__ void join_from(const float *unit, const Place &at)
   {
      const float *from = unit + at.in_slot * W;
      F2 x[2][NV][P];  // all loads before the first sum
#pragma unroll
      for (int t = 0; t < NV; t++) {
         get_pairs<P>(from + t * W * G, x[0][t]);
         get_pairs<P>(from + (NV + t) * W * G, x[1][t]);
      }
#pragma unroll
      for (int t = 0; t < NV; t++)
#pragma unroll
         for (int j = 0; j < P; j++) {
            s.dk[t][j] = add2(s.dk[t][j], x[0][t][j]);
            s.dv[t][j] = add2(s.dv[t][j], x[1][t][j]);
         }
   }
   __device__ __forceinline__ void put(float *unit, const Place &at) const
   {
      float *to = unit + at.in_slot * W;
#pragma unroll
      for (int t = 0; t < NV; t++) {
         put_pairs<P>(to + t * W * G, s.dk[t]);
         put_pairs<P>(to + (NV + t) * W * G, s.dv[t]);
      }
   }

   __device__ __forceinline__ void finish(const AttnParams &p, const Place &at, long long col)
   {
      if (at.edge_slot != 0) return;
      const long long rh = col * p.kv_heads + at.unit;
#pragma unroll
      for (int t = 0; t < NV; t++) {
         const int x = (at.in_half + (G / 2) * t) * W, y = (at.in_slot + G * t) * W;
         float o[W], v[W];
         unpair(s.dk[t], o);
         unpair(s.dv[t], v);
#pragma unroll
         for (int j = 0; j < W; j++) o[j] *= p.scale;
         st_row<T, FORM != PIECES>(static_cast<T *>(p.out) + (rh * 2 + at.half) * p.d + x, o, p.d - x);
         st_row<T, FORM != PIECES>(static_cast<T *>(p.out2) + rh * p.dv + y, v, p.dv - y);
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

// the warps of a block that shared a row join their states by halves, in a fixed order
template <typename Op, int G>
__device__ __forceinline__ void join_warps(Op &op, const Place &at, float *shared)
{
   constexpr int STRIDE = Op::LANE_FLOATS * 32;  // slots side by side, as in scratch
   float *mine = shared + (at.lane / G) * part_floats<Op, G>;
   for (int half = JOINT_WARPS / 2; half > 0; half /= 2) {
      __syncthreads();
      if (at.warp >= half && at.warp < 2 * half) op.put(mine + (at.warp - half) * STRIDE, at);
      __syncthreads();
      if (at.warp < half) op.join_from(mine + at.warp * STRIDE, at);
   }
}

// The long rows a joining block looks after: the block's row, where there are fewer rows than pieces, or the rows that begin in
// its pieces.
struct LongRows {
   long long at, end;
   __device__ __forceinline__ LongRows(const AttnParams &p, long long group)
   {
      at = p.join_rows ? group : group * p.join_pieces;
      end = p.join_rows ? group + 1 : at + p.join_pieces < p.pieces ? at + p.join_pieces : p.pieces;
   }
   // the next: the row, the piece it begins in, its parts
   __device__ __forceinline__ bool next(const AttnParams &p, const Rows &rows, long long &u, long long &piece, long long &parts)
   {
      for (; at < end; at++) {
         if (p.join_rows) {
            u = at;
            const long long fb = rows.items(u);
            if (rows.items(u + 1) - fb <= p.row_limit) continue;
            piece = fb / p.piece;
         } else {
            piece = at;
            u = p.long_row[piece];
            if (u < 0) continue;
         }
         parts = (rows.items(u + 1) - 1) / p.piece - piece + 1;
         at++;
         return true;
      }
      return false;
   }
};

// TOGETHER: the warps of a block share every row (few, long rows), else each warp has a piece of its own.
template <typename Op, int G, bool TOGETHER>
__global__ void __launch_bounds__((TOGETHER ? JOINT_WARPS : PIECE_WARPS) * 32, TOGETHER ? 1 : Op::BLOCKS) walk_kernel(const AttnParams p)
{
   extern __shared__ __align__(16) float shared[];
   const int warp = threadIdx.x >> 5;
   const long long job = TOGETHER ? blockIdx.x : static_cast<long long>(blockIdx.x) * PIECE_WARPS + warp;
   const long long piece = job / p.unit_blocks;
   if (piece >= p.pieces) return;
   const Place at = Place::make<G>(p, static_cast<int>(job - piece * p.unit_blocks));
   const Rows rows(p);
   const long long lo = piece * p.piece, hi = lo + p.piece;
   long long u = rows.lower_bound(lo, 0, p.m, at.lane);
   const bool teller = at.lane == 0 && (!TOGETHER || warp == 0) && job == piece * p.unit_blocks;
   long long begun = -1;
   Op op;
   EdgeStream edges;
   // row pointers 32 at a time, one to a lane
   long long from = u > 0 ? u - 1 : 0;
   long long mine = rows.begin(from + at.lane < p.m ? from + at.lane : p.m);
   if (u > 0) {  // the row before may reach into this piece: then it is this loop's first
      const long long b = __shfl_sync(FULL, mine, 0), e = __shfl_sync(FULL, mine, 1);
      const long long fb = b - rows.first + ROW_ITEMS * (u - 1), fe = e - rows.first + ROW_ITEMS * u;
      if (fe > lo && fe - fb > p.row_limit) u--;
   }
   for (; u < p.m; u++) {
      if (u + 1 - from > 31) {
         from = u;
         mine = rows.begin(from + at.lane < p.m ? from + at.lane : p.m);
      }
      const long long b = __shfl_sync(FULL, mine, static_cast<int>(u - from)), fb = b - rows.first + ROW_ITEMS * u;
      if (fb >= hi) break;
      const long long e = __shfl_sync(FULL, mine, static_cast<int>(u + 1 - from));
      const long long fe = e - rows.first + ROW_ITEMS * (u + 1);
      long long e0 = b, e1 = e, part = -1;
      if (fe - fb > p.row_limit) {  // a long row: this piece's part of it
         e0 = b + (lo - fb - ROW_ITEMS);
         e1 = b + (hi - fb - ROW_ITEMS);
         e0 = e0 < b ? b : e0;
         e1 = e1 > e ? e : e1 < e0 ? e0 : e1;
         part = 2 * piece + (fb >= lo);
         if (fb >= lo) begun = u;
      }
      op.run(p, at, edges, u, e0, e1, TOGETHER ? warp : 0, TOGETHER ? JOINT_WARPS : 1);
      if (TOGETHER) join_warps<Op, G>(op, at, shared);
      if (!TOGETHER || warp == 0) {
         if (part < 0) op.finish(p, at, u);
         else if (at.edge_slot == 0) op.put(part_at<Op, G>(p, at, part), at);
      }
   }
   if (teller) p.long_row[piece] = begun;
}

// The parts of the long rows; a row's parts go to the warps in runs, joined in order.
template <typename Op, int G>
__global__ void __launch_bounds__(JOINT_WARPS * 32) join_kernel(const AttnParams p)
{
   extern __shared__ __align__(16) float shared[];
   const int warp = threadIdx.x >> 5;
   const Place at = Place::make<G>(p, static_cast<int>(blockIdx.x % p.unit_blocks));
   const Rows rows(p);
   Op op;
   LongRows todo(p, blockIdx.x / p.unit_blocks);
   long long u, piece, parts;
   while (todo.next(p, rows, u, piece, parts)) {
      const long long each = (parts + JOINT_WARPS - 1) / JOINT_WARPS;
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
   int g = 0, nv = 0, qb = 1, form = PIECES;
   int width = 0;  // > 0: a walk on the matrix units, for d up to this and dv up to twice this
   bool together = false;
};

// Lets a kernel have this much shared memory on the current device.  The runtime keeps that per kernel and device, so it is asked
// once for each (the devices behind the 64th every time).
bool set_shared(const void *kernel, int bytes, std::atomic<unsigned long long> &devices);
template <auto KERNEL>
bool allow_shared(int bytes)
{
   static std::atomic<unsigned long long> devices{0};
   return bytes <= 48 << 10 || set_shared(reinterpret_cast<const void *>(KERNEL), bytes, devices);
}

inline unsigned join_blocks(const AttnParams &p)
{
   return static_cast<unsigned>((p.join_rows ? p.m : (p.pieces + p.join_pieces - 1) / p.join_pieces) * p.unit_blocks);
}

template <typename Op, int G>
int launch_op(const AttnParams &p, bool together, cudaStream_t st)
{
   const int bytes = JOINT_WARPS / 2 * 32 * Op::LANE_FLOATS * static_cast<int>(sizeof(float));
   if (!allow_shared<join_kernel<Op, G>>(bytes)) return -1;
   const long long jobs = p.pieces * p.unit_blocks;
   if (together) {
      if (!allow_shared<walk_kernel<Op, G, true>>(bytes)) return -1;
      walk_kernel<Op, G, true><<<static_cast<unsigned>(jobs), JOINT_WARPS * 32, bytes, st>>>(p);
   } else {
      walk_kernel<Op, G, false><<<static_cast<unsigned>((jobs + PIECE_WARPS - 1) / PIECE_WARPS), PIECE_WARPS * 32, 0, st>>>(p);
   }
   join_kernel<Op, G><<<join_blocks(p), JOINT_WARPS * 32, bytes, st>>>(p);
   return 0;
}

// query heads that a unit may hold: registers decide (a lane holds 2 NV W sums and NV W numbers of q for each)
template <typename T, bool COLUMNS>
constexpr int max_heads() { return COLUMNS ? 1 : sizeof(T) == 4 ? 4 : 2; }

template <typename T, int G, int NV, template <typename, int, int, int, int> class Op, bool COLUMNS>
int launch_slot(const WalkShape &s, const AttnParams &p, cudaStream_t st)
{
   if (s.form == PIECES) return launch_op<Op<T, G, NV, 1, PIECES>, G>(p, s.together, st);
   if (s.form == RAGGED) return launch_op<Op<T, G, NV, 1, RAGGED>, G>(p, s.together, st);
   if constexpr (max_heads<T, COLUMNS>() >= 4)
      if (s.qb == 4) return launch_op<Op<T, G, NV, 4, EXACT>, G>(p, s.together, st);
   if constexpr (max_heads<T, COLUMNS>() >= 2)
      if (s.qb == 2) return launch_op<Op<T, G, NV, 2, EXACT>, G>(p, s.together, st);
   return launch_op<Op<T, G, NV, 1, EXACT>, G>(p, s.together, st);
}

// -1: no such instantiation
template <typename T, template <typename, int, int, int, int> class Op, bool COLUMNS>
int launch_walk(const WalkShape &s, const AttnParams &p, cudaStream_t st)
{
   if (s.nv == 1 && s.g == 4) return launch_slot<T, 4, 1, Op, COLUMNS>(s, p, st);
   if (s.nv != 2) return -1;
   if (s.g == 4) return launch_slot<T, 4, 2, Op, COLUMNS>(s, p, st);
   if (s.g == 8) return launch_slot<T, 8, 2, Op, COLUMNS>(s, p, st);
   if (s.g == 16) return launch_slot<T, 16, 2, Op, COLUMNS>(s, p, st);
   if constexpr (sizeof(T) == 4)
      if (s.g == 32) return launch_slot<T, 32, 2, Op, COLUMNS>(s, p, st);
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

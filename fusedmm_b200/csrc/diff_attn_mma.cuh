// diff_attn_mma.cuh -- the walks of diff_attn.cuh for 16-bit types on the matrix units.
//
// A step takes 16 pairs (edge, kv head): HS neighbouring kv heads of 16/HS edges, HS x (query heads of a kv head) <= 4.
// The two products of the forward walk are mma m16n8k16 with 32-bit sums:
//   scores  [16 pairs x 8 columns], column = (map, query head): A = gathered k, B = q.  A pair and a query head of
//           different kv heads give numbers nobody uses (HS > 1): at these sizes a wasted column costs less than the
//           conversions and lane sums of a product on the ordinary units.
//   output  [8 rows x dv] over k = 16 pairs: A = weights, 0 where the heads differ, B = gathered v.
// Weights are split into two 16-bit numbers whose sum has 16 bits (bf16) or 22 (half) of the 32-bit value; the second lies in
// the rows 8..15 of A that the first leaves free, so the split costs no product.
// The order of a product's inner index is free as long as both operands share it: every lane loads 8 consecutive elements
// of a gathered row as they are, no shared memory and no transposition; where an operand has the pairs as inner index
// two rows' elements are put side by side with byte permutes.  The weights change from "pair by column" to "row by pair"
// with movmatrix.
// Why not tcgen05: a tile there has 64 or 128 rows that share one operand; here a gathered row meets at most 8 rows of q,
// and consecutive rows of the pattern gather different rows.
//
// Measured against the walks on the ordinary units see the choice of the shape in diff_attn_capi.cu.
#pragma once
#include "diff_attn.cuh"

namespace fmm {
namespace attn {

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1)
{
   if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value)
      asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                   : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
   else
      asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                   : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ unsigned transpose8x8(unsigned v)
{
   unsigned r;
   asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
   return r;
}
// v as the sum of two numbers of T, for two neighbours
template <typename T>
__device__ __forceinline__ void split2(float a, float b, unsigned &hi, unsigned &lo)
{
   hi = Elt<T>::pack2(a, b);
   float x, y;
   Elt<T>::unpack2(hi, x, y);
   lo = Elt<T>::pack2(a - x, b - y);
}

// E elements (2, 4 or 8) at p, `left` of them there
template <typename T, int E, int FORM>
__device__ __forceinline__ void load_part(const T *p, int left, int step, unsigned (&r)[E / 2])
{
   if constexpr (FORM == PIECES) {
      const uint4 v = ld_pieces(p, left < E ? left : E, step < E ? step : E);
      r[0] = v.x;
      if constexpr (E >= 4) r[1] = v.y;
      if constexpr (E == 8) { r[2] = v.z; r[3] = v.w; }
   } else {
      const bool there = FORM == EXACT || left > 0;
      if constexpr (E == 8) {
         const uint4 v = there ? ldg16(p) : make_uint4(0u, 0u, 0u, 0u);
         r[0] = v.x; r[1] = v.y; r[2] = v.z; r[3] = v.w;
      } else if constexpr (E == 4) {
         const uint2 v = there ? __ldg(reinterpret_cast<const uint2 *>(p)) : make_uint2(0u, 0u);
         r[0] = v.x; r[1] = v.y;
      } else {
         r[0] = there ? __ldg(reinterpret_cast<const unsigned *>(p)) : 0u;
      }
   }
}

// A row of WIDTH elements as the lanes hold it when its elements are the inner index: lane c (of 4) has the elements
// 4 E s + E c .. + E - 1 of every set s; two registers make a step of 16 elements.
template <typename T, int WIDTH>
struct Inner {
   static constexpr int E = WIDTH / 4 < 8 ? WIDTH / 4 : 8, SETS = WIDTH / (4 * E), REGS = WIDTH / 8, STEPS = WIDTH / 16;
   template <int FORM>
   static __device__ __forceinline__ void load(const T *row, int c, int width, bool live, int step, unsigned (&r)[REGS])
   {
#pragma unroll
      for (int s = 0; s < SETS; s++) {
         const int x = 4 * E * s + E * c;
         unsigned part[E / 2];
         load_part<T, E, FORM>(row + x, live ? width - x : 0, step, part);
#pragma unroll
         for (int i = 0; i < E / 2; i++) r[s * (E / 2) + i] = part[i];
      }
   }
};
// ... and when its elements are rows or columns of the product: lane group g (of 8) has the elements 8 E s + E g .. + E - 1.
template <typename T, int WIDTH>
struct Outer {
   static constexpr int E = WIDTH / 8 < 8 ? WIDTH / 8 : 8, SETS = WIDTH / (8 * E), REGS = WIDTH / 16;
   template <int FORM>
   static __device__ __forceinline__ void load(const T *row, int g, int width, bool live, int step, unsigned (&r)[REGS])
   {
#pragma unroll
      for (int s = 0; s < SETS; s++) {
         const int x = 8 * E * s + E * g;
         unsigned part[E / 2];
         load_part<T, E, FORM>(row + x, live ? width - x : 0, step, part);
#pragma unroll
         for (int i = 0; i < E / 2; i++) r[s * (E / 2) + i] = part[i];
      }
   }
   // E consecutive results of this lane's rows to memory
   template <bool VECTOR>
   static __device__ __forceinline__ void store(T *p, const float (&f)[E], int left)
   {
      if constexpr (VECTOR) {
         if (left <= 0) return;
         unsigned r[E / 2];
#pragma unroll
         for (int i = 0; i < E / 2; i++) r[i] = Elt<T>::pack2(f[2 * i], f[2 * i + 1]);
         if constexpr (E == 8) *reinterpret_cast<uint4 *>(p) = make_uint4(r[0], r[1], r[2], r[3]);
         else if constexpr (E == 4) *reinterpret_cast<uint2 *>(p) = make_uint2(r[0], r[1]);
         else *reinterpret_cast<unsigned *>(p) = r[0];
      } else {
#pragma unroll
         for (int i = 0; i < E; i++)
            if (i < left) p[i] = Elt<T>::down(f[i]);
      }
   }
};
__device__ __forceinline__ unsigned low_halves(unsigned a, unsigned b) { return __byte_perm(a, b, 0x5410); }
__device__ __forceinline__ unsigned high_halves(unsigned a, unsigned b) { return __byte_perm(a, b, 0x7632); }

// a gathered array: pointers of this lane's head, byte stride of rows
template <typename T>
struct Source {
   const char *base;
   unsigned stride;
   __device__ __forceinline__ void set(const void *array, long long ld, long long offset)
   {
      base = static_cast<const char *>(array) + offset * static_cast<long long>(sizeof(T));
      stride = static_cast<unsigned>(ld * static_cast<long long>(sizeof(T)));
   }
   template <int FORM>
   __device__ __forceinline__ const T *row(int id) const
   {
      const T *r = reinterpret_cast<const T *>(base + static_cast<unsigned long long>(static_cast<unsigned>(id)) * stride);
      return FORM == EXACT && id < 0 ? reinterpret_cast<const T *>(zero_row) : r;
   }
};

// Lane geometry that the three walks share.  Lane = 4 r + c.  As an operand's row (or column) r: the query head and map of
// column n = r; as a result: the pairs r and r + 8, the columns 2c and 2c + 1.
struct Lanes {
   int r, c, hs, hs_log2, kv0, pair_head;  // pair_head: which of the unit's kv heads the pairs r and r + 8 are of
   __device__ __forceinline__ void set(const AttnParams &p, const Place &at)
   {
      r = at.lane >> 2;
      c = at.lane & 3;
      hs = p.unit_kv;
      hs_log2 = hs >> 1;  // 1, 2, 4 -> 0, 1, 2
      kv0 = (at.unit / p.head_blocks) * hs;
      pair_head = r & (hs - 1);
   }
   // the edge, counted from the step's first, of a pair
   __device__ __forceinline__ int edge(int pair) const { return pair >> hs_log2; }
};

// value of column n = r from the lanes that hold the columns 2c and 2c + 1 (the same in all r)
__device__ __forceinline__ float of_column(float x0, float x1, int r)
{
   const float a = __shfl_sync(FULL, x0, r >> 1), b = __shfl_sync(FULL, x1, r >> 1);
   return r & 1 ? b : a;
}
__device__ __forceinline__ float sum_pairs(float v)
{
   v += __shfl_xor_sync(FULL, v, 4);
   v += __shfl_xor_sync(FULL, v, 8);
   return v + __shfl_xor_sync(FULL, v, 16);
}
__device__ __forceinline__ float max_pairs(float v)
{
   v = fmaxf(v, __shfl_xor_sync(FULL, v, 4));
   v = fmaxf(v, __shfl_xor_sync(FULL, v, 8));
   return fmaxf(v, __shfl_xor_sync(FULL, v, 16));
}

// The query heads of the row walks' columns: column n = 4 map + s, s = (kv head of the unit) * per_kv + (query head of it).
struct QueryHeads {
   int head;       // of column n = r, clamped to a head that exists
   bool live;      // column n = r is one
   bool valid[2];  // the pairs r and r + 8 belong to the columns 2c, 2c + 1
   int col_head[2];
   int kv;         // which of the unit's kv heads column n = r is of
   __device__ __forceinline__ void set(const AttnParams &p, const Place &at, const Lanes &l)
   {
      const int block = at.unit % p.head_blocks, first = block * p.unit_heads, rest = p.group - first;
      const int heads = rest < p.unit_heads ? rest : p.unit_heads;
      const int s = l.r & 3, g = s % p.unit_heads;
      kv = s / p.unit_heads;
      live = kv < l.hs && g < heads;
      head = live ? (l.kv0 + kv) * p.group + first + g : l.kv0 * p.group + first;
#pragma unroll
      for (int x = 0; x < 2; x++) {
         const int sx = (2 * l.c + x) & 3, kx = sx / p.unit_heads, gx = sx % p.unit_heads;
         valid[x] = kx == l.pair_head && gx < heads;
         col_head[x] = valid[x] ? (l.kv0 + kx) * p.group + first + gx : head;
      }
   }
};

// the maximum may grow by this much (as a power of e) before sums are scaled anew: weights then stay below e^5 and a
// row's scaling is done once as a rule.  32-bit sums and 16-bit weights (half: up to 65504) hold e^5 with room.
constexpr float SLACK = 5.0f;

// ---------------------------------------------------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int DK, int DV, int FORM>
struct ForwardMma {
   static constexpr int BLOCKS = DV <= 64 ? 4 : DV <= 128 ? 3 : 2;
   static constexpr int TILES = DV / 8;
   static constexpr int LANE_FLOATS = 2 * TILES + 4;
   using KIn = Inner<T, DK>;
   using VOut = Outer<T, DV>;
   struct State {
      float acc[TILES][2];   // rows n = r: sums of weights times v
      float top[2], sum[2];  // columns 2c, 2c + 1; sum: of this lane's pairs until the end of run()
   };
   State s;
   Lanes l;
   QueryHeads heads;
   bool lost;  // run() met a number that is none

   __device__ __forceinline__ void setup(const AttnParams &p, const Place &at)
   {
      l.set(p, at);
      heads.set(p, at, l);
   }
   static __device__ __forceinline__ void clear(State &s)
   {
#pragma unroll
      for (int t = 0; t < TILES; t++) s.acc[t][0] = s.acc[t][1] = 0.0f;
      s.top[0] = s.top[1] = -INFINITY;
      s.sum[0] = s.sum[1] = 0.0f;
   }

   __device__ __forceinline__ void run(const AttnParams &p, const Place &at, EdgeStream &edges, long long row, long long e0, long long e1,
                                       int warp, int warps, int only)
   {
      lost = false;
      clear(s);
      if (e0 + 32 * warp >= e1) return;
      float acc[TILES][4];
#pragma unroll
      for (int t = 0; t < TILES; t++) acc[t][0] = acc[t][1] = acc[t][2] = acc[t][3] = 0.0f;
      unsigned q[KIn::REGS];
      KIn::template load<FORM>(static_cast<const T *>(p.q) + row * p.ldq + heads.head * p.hsq + (l.r >> 2) * p.d, l.c, p.d, true, p.step, q);
      Source<T> kg, vg[2];
      kg.set(p.k, p.ldk, (l.kv0 + l.pair_head) * p.hsk);
      const int even = (2 * l.c) & (l.hs - 1), odd = (2 * l.c + 1) & (l.hs - 1);
      vg[0].set(p.v, p.ldv, (l.kv0 + even) * p.hsv);
      vg[1].set(p.v, p.ldv, (l.kv0 + odd) * p.hsv);
      const bool skip[2] = {only >= 0 && even != only, only >= 0 && odd != only};
      const int per_step = 16 >> l.hs_log2;
      for (long long base = e0 + 32 * warp; base < e1; base += 32 * warps) {
         const int my_id = edges.take(p, base, e1, at.lane);
         const float my_bias = edges.bias;
         edges.fetch(p, base + 32 * warps < e1 ? base + 32 * warps : e1 + 32 * warp, at.lane);
         const int count = static_cast<int>(e1 - base < 32 ? e1 - base : 32);
         for (int first = 0; first < count; first += per_step) {
            // gathered rows: k of the pairs r and r + 8, v of the pairs 2c, 2c + 1, 2c + 8, 2c + 9
            int id[2];
            unsigned k[2][2][KIn::REGS], v[4][VOut::REGS];
#pragma unroll
            for (int h = 0; h < 2; h++) {
               id[h] = __shfl_sync(FULL, my_id, first + l.edge(l.r + 8 * h));
               const T *src = kg.template row<FORM>(id[h]);
               KIn::template load<FORM>(src, l.c, p.d, id[h] >= 0, p.step, k[0][h]);
               KIn::template load<FORM>(FORM == EXACT && id[h] < 0 ? src : src + p.d, l.c, p.d, id[h] >= 0, p.step, k[1][h]);
            }
#pragma unroll
            for (int h = 0; h < 4; h++) {
               int vid = __shfl_sync(FULL, my_id, first + l.edge(2 * l.c + (h & 1) + 8 * (h >> 1)));
               if (skip[h & 1]) vid = -1;
               VOut::template load<FORM>(vg[h & 1].template row<FORM>(vid), l.r, p.dv, vid >= 0, p.step, v[h]);
            }
            float s0[4] = {0.0f, 0.0f, 0.0f, 0.0f}, s1[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < KIn::STEPS; i++) {
               mma16816<T>(s0, k[0][0][2 * i], k[0][1][2 * i], k[0][0][2 * i + 1], k[0][1][2 * i + 1], q[2 * i], q[2 * i + 1]);
               mma16816<T>(s1, k[1][0][2 * i], k[1][1][2 * i], k[1][0][2 * i + 1], k[1][1][2 * i + 1], q[2 * i], q[2 * i + 1]);
            }
            float score[2][2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
               const float bias = p.bias ? __shfl_sync(FULL, my_bias, first + l.edge(l.r + 8 * h)) : 0.0f;
#pragma unroll
               for (int x = 0; x < 2; x++) {
                  const float dot = l.c < 2 ? s0[2 * h + x] : s1[2 * h + x];
                  score[h][x] = heads.valid[x] && id[h] >= 0 ? fmaf(dot, p.scale, bias) : -INFINITY;
               }
            }
            const float m0 = fmaxf(score[0][0], score[1][0]), m1 = fmaxf(score[0][1], score[1][1]);
            if (__any_sync(FULL, m0 > s.top[0] + SLACK || m1 > s.top[1] + SLACK)) {
               const float t0 = fmaxf(s.top[0], max_pairs(m0)), t1 = fmaxf(s.top[1], max_pairs(m1));
               const float f0 = t0 == -INFINITY ? 1.0f : exp2_fast((s.top[0] - t0) * LOG2E);
               const float f1 = t1 == -INFINITY ? 1.0f : exp2_fast((s.top[1] - t1) * LOG2E);
               const float f = of_column(f0, f1, l.r);
               s.top[0] = t0;
               s.top[1] = t1;
               s.sum[0] *= f0;
               s.sum[1] *= f1;
#pragma unroll
               for (int t = 0; t < TILES; t++)
#pragma unroll
                  for (int i = 0; i < 4; i++) acc[t][i] *= f;
            }
            // a row that has met no edge yet has the maximum -inf: its differences are taken from 0
            const float ref0 = s.top[0] == -INFINITY ? 0.0f : s.top[0], ref1 = s.top[1] == -INFINITY ? 0.0f : s.top[1];
            unsigned a[4];
#pragma unroll
            for (int h = 0; h < 2; h++) {
               // the difference is taken before the factor: scores near the type's largest numbers keep their order
               const float p0 = exp2_fast((score[h][0] - ref0) * LOG2E), p1 = exp2_fast((score[h][1] - ref1) * LOG2E);
               s.sum[0] += p0;
               s.sum[1] += p1;
               unsigned hi, lo;
               split2<T>(p0, p1, hi, lo);
               a[2 * h] = transpose8x8(hi);
               a[2 * h + 1] = transpose8x8(lo);
            }
#pragma unroll
            for (int t = 0; t < VOut::REGS; t++) {
               mma16816<T>(acc[2 * t], a[0], a[1], a[2], a[3], low_halves(v[0][t], v[1][t]), low_halves(v[2][t], v[3][t]));
               mma16816<T>(acc[2 * t + 1], a[0], a[1], a[2], a[3], high_halves(v[0][t], v[1][t]), high_halves(v[2][t], v[3][t]));
            }
         }
      }
      bool bad = false;
#pragma unroll
      for (int t = 0; t < TILES; t++) {
         s.acc[t][0] = acc[t][0] + acc[t][2];
         s.acc[t][1] = acc[t][1] + acc[t][3];
         bad |= s.acc[t][0] != s.acc[t][0] || s.acc[t][1] != s.acc[t][1];
      }
      lost = bad;
      s.sum[0] = sum_pairs(s.sum[0]);
      s.sum[1] = sum_pairs(s.sum[1]);
   }

   __device__ __forceinline__ void join_from(const float *unit, const Place &at)
   {
      const float2 *from = reinterpret_cast<const float2 *>(unit) + at.lane;
      const float2 top = from[32 * TILES], sum = from[32 * (TILES + 1)];
      float f[2], g[2];
#pragma unroll
      for (int x = 0; x < 2; x++) {
         const float ot = x ? top.y : top.x, os = x ? sum.y : sum.x;
         const float t = fmaxf(s.top[x], ot), ref = t == -INFINITY ? 0.0f : t;
         f[x] = exp2_fast((s.top[x] - ref) * LOG2E);
         g[x] = exp2_fast((ot - ref) * LOG2E);
         s.sum[x] = s.sum[x] * f[x] + os * g[x];
         s.top[x] = t;
      }
      const float fr = of_column(f[0], f[1], l.r), gr = of_column(g[0], g[1], l.r);
#pragma unroll
      for (int t = 0; t < TILES; t++) {
         const float2 o = from[32 * t];
         s.acc[t][0] = s.acc[t][0] * fr + o.x * gr;
         s.acc[t][1] = s.acc[t][1] * fr + o.y * gr;
      }
   }
   __device__ __forceinline__ void put(float *unit, const Place &at, int only) const
   {
      float2 *to = reinterpret_cast<float2 *>(unit) + at.lane;
      if (only < 0 || heads.kv == only) {
#pragma unroll
         for (int t = 0; t < TILES; t++) to[32 * t] = make_float2(s.acc[t][0], s.acc[t][1]);
      }
      to[32 * TILES] = make_float2(s.top[0], s.top[1]);
      to[32 * (TILES + 1)] = make_float2(s.sum[0], s.sum[1]);
   }

   __device__ __forceinline__ void finish(const AttnParams &p, const Place &at, long long row, int only)
   {
      const float sum = of_column(s.sum[0], s.sum[1], l.r), top = of_column(s.top[0], s.top[1], l.r);
      const bool mine = heads.live && (only < 0 || heads.kv == only);
      const float lam = __ldg(p.lam + row * p.ldlam + heads.head), f = sum == 0.0f ? 0.0f : 1.0f / sum;
      const long long rh = row * p.heads + heads.head;
#pragma unroll
      for (int set = 0; set < VOut::SETS; set++)
#pragma unroll
         for (int x = 0; x < 2; x++) {
            float o[VOut::E];
#pragma unroll
            for (int j = 0; j < VOut::E; j++) {
               const float v = s.acc[set * VOut::E + j][x] * f;
               o[j] = v - lam * __shfl_xor_sync(FULL, v, 16);
            }
            const int y = 8 * VOut::E * set + VOut::E * (2 * l.c + x);
            if (mine && l.r < 4) VOut::template store<FORM != PIECES>(static_cast<T *>(p.out) + rh * p.dv + y, o, p.dv - y);
         }
      if (mine && l.c == 0 && p.lse) p.lse[rh * 2 + (l.r >> 2)] = top + LN2 * log2f(sum);
   }
};

// ---------------------------------------------------------------------------------------------------------------------
// backward over the rows (the sums A = sum p dP k, B = sum p k, D = sum p dP of BackwardRows).  For map 0 the rows of A's
// operand are w = p dP of the columns 0..3 and p of the same, for map 1 the other way round.
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int DK, int DV, int FORM>
struct BackwardRowsMma {
   static constexpr int BLOCKS = DV <= 64 ? 4 : DV <= 128 ? 3 : 2;
   static constexpr int TILES = DK / 8;
   static constexpr int LANE_FLOATS = 4 * TILES + 2;
   using KIn = Inner<T, DK>;
   using KOut = Outer<T, DK>;
   using VIn = Inner<T, DV>;
   struct State {
      float acc[2][TILES][2];
      float delta[2];  // columns 2c, 2c + 1
   };
   State s;
   Lanes l;
   QueryHeads heads;
   bool lost;

   __device__ __forceinline__ void setup(const AttnParams &p, const Place &at)
   {
      l.set(p, at);
      heads.set(p, at, l);
   }
   static __device__ __forceinline__ void clear(State &s)
   {
#pragma unroll
      for (int m = 0; m < 2; m++)
#pragma unroll
         for (int t = 0; t < TILES; t++) s.acc[m][t][0] = s.acc[m][t][1] = 0.0f;
      s.delta[0] = s.delta[1] = 0.0f;
   }

   __device__ __forceinline__ void run(const AttnParams &p, const Place &at, EdgeStream &edges, long long row, long long e0, long long e1,
                                       int warp, int warps, int only)
   {
      lost = false;
      clear(s);
      if (e0 + 32 * warp >= e1) return;
      float acc[2][TILES][4];
#pragma unroll
      for (int m = 0; m < 2; m++)
#pragma unroll
         for (int t = 0; t < TILES; t++) acc[m][t][0] = acc[m][t][1] = acc[m][t][2] = acc[m][t][3] = 0.0f;
      unsigned q[KIn::REGS], dout[VIn::REGS];
      KIn::template load<FORM>(static_cast<const T *>(p.q) + row * p.ldq + heads.head * p.hsq + (l.r >> 2) * p.d, l.c, p.d, true, p.step, q);
      VIn::template load<FORM>(static_cast<const T *>(p.dout) + row * p.ldo + heads.head * p.hso, l.c, p.dv, true, p.step, dout);
      float lse[2];
#pragma unroll
      for (int x = 0; x < 2; x++) lse[x] = __ldg(p.lse + (row * p.heads + heads.col_head[x]) * 2 + (l.c >> 1));
      Source<T> kg, vg, ko[2];
      kg.set(p.k, p.ldk, (l.kv0 + l.pair_head) * p.hsk);
      vg.set(p.v, p.ldv, (l.kv0 + l.pair_head) * p.hsv);
      const int even = (2 * l.c) & (l.hs - 1), odd = (2 * l.c + 1) & (l.hs - 1);
      ko[0].set(p.k, p.ldk, (l.kv0 + even) * p.hsk);
      ko[1].set(p.k, p.ldk, (l.kv0 + odd) * p.hsk);
      const bool skip[2] = {only >= 0 && even != only, only >= 0 && odd != only};
      const int per_step = 16 >> l.hs_log2;
      for (long long base = e0 + 32 * warp; base < e1; base += 32 * warps) {
         const int my_id = edges.take(p, base, e1, at.lane);
         const float my_bias = edges.bias;
         edges.fetch(p, base + 32 * warps < e1 ? base + 32 * warps : e1 + 32 * warp, at.lane);
         const int count = static_cast<int>(e1 - base < 32 ? e1 - base : 32);
         for (int first = 0; first < count; first += per_step) {
            int id[2];
            unsigned k[2][2][KIn::REGS], v[2][VIn::REGS];
#pragma unroll
            for (int h = 0; h < 2; h++) {
               id[h] = __shfl_sync(FULL, my_id, first + l.edge(l.r + 8 * h));
               const T *src = kg.template row<FORM>(id[h]);
               KIn::template load<FORM>(src, l.c, p.d, id[h] >= 0, p.step, k[0][h]);
               KIn::template load<FORM>(FORM == EXACT && id[h] < 0 ? src : src + p.d, l.c, p.d, id[h] >= 0, p.step, k[1][h]);
               VIn::template load<FORM>(vg.template row<FORM>(id[h]), l.c, p.dv, id[h] >= 0, p.step, v[h]);
            }
            float s0[4] = {0.0f, 0.0f, 0.0f, 0.0f}, s1[4] = {0.0f, 0.0f, 0.0f, 0.0f}, dp[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < KIn::STEPS; i++) {
               mma16816<T>(s0, k[0][0][2 * i], k[0][1][2 * i], k[0][0][2 * i + 1], k[0][1][2 * i + 1], q[2 * i], q[2 * i + 1]);
               mma16816<T>(s1, k[1][0][2 * i], k[1][1][2 * i], k[1][0][2 * i + 1], k[1][1][2 * i + 1], q[2 * i], q[2 * i + 1]);
            }
#pragma unroll
            for (int i = 0; i < VIn::STEPS; i++)
               mma16816<T>(dp, v[0][2 * i], v[1][2 * i], v[0][2 * i + 1], v[1][2 * i + 1], dout[2 * i], dout[2 * i + 1]);
            // the same rows of k once more, as columns of the second product
            unsigned kt[2][4][KOut::REGS];
#pragma unroll
            for (int h = 0; h < 4; h++) {
               int kid = __shfl_sync(FULL, my_id, first + l.edge(2 * l.c + (h & 1) + 8 * (h >> 1)));
               if (skip[h & 1]) kid = -1;
               const T *src = ko[h & 1].template row<FORM>(kid);
               KOut::template load<FORM>(src, l.r, p.d, kid >= 0, p.step, kt[0][h]);
               KOut::template load<FORM>(FORM == EXACT && kid < 0 ? src : src + p.d, l.r, p.d, kid >= 0, p.step, kt[1][h]);
            }
            unsigned a0[4], a1[4];
#pragma unroll
            for (int h = 0; h < 2; h++) {
               const float bias = p.bias ? __shfl_sync(FULL, my_bias, first + l.edge(l.r + 8 * h)) : 0.0f;
               float pr[2], w[2];
#pragma unroll
               for (int x = 0; x < 2; x++) {
                  const float dot = l.c < 2 ? s0[2 * h + x] : s1[2 * h + x];
                  // an edge that is masked has p = 0, and so has a row without edges (its lse is -inf)
                  const bool live = heads.valid[x] && id[h] >= 0 && lse[x] != -INFINITY;
                  pr[x] = live ? exp2_fast((fmaf(dot, p.scale, bias) - lse[x]) * LOG2E) : 0.0f;
                  w[x] = live ? pr[x] * dp[2 * h + x] : 0.0f;
                  s.delta[x] += w[x];
               }
               unsigned wh, wl, ph, pl;
               split2<T>(w[0], w[1], wh, wl);
               split2<T>(pr[0], pr[1], ph, pl);
               wh = transpose8x8(wh);
               wl = transpose8x8(wl);
               ph = __shfl_xor_sync(FULL, transpose8x8(ph), 16);
               pl = __shfl_xor_sync(FULL, transpose8x8(pl), 16);
               a0[2 * h] = l.r < 4 ? wh : ph;
               a0[2 * h + 1] = l.r < 4 ? wl : pl;
               a1[2 * h] = l.r < 4 ? ph : wh;
               a1[2 * h + 1] = l.r < 4 ? pl : wl;
            }
#pragma unroll
            for (int t = 0; t < KOut::REGS; t++) {
               mma16816<T>(acc[0][2 * t], a0[0], a0[1], a0[2], a0[3], low_halves(kt[0][0][t], kt[0][1][t]), low_halves(kt[0][2][t], kt[0][3][t]));
               mma16816<T>(acc[0][2 * t + 1], a0[0], a0[1], a0[2], a0[3], high_halves(kt[0][0][t], kt[0][1][t]), high_halves(kt[0][2][t], kt[0][3][t]));
               mma16816<T>(acc[1][2 * t], a1[0], a1[1], a1[2], a1[3], low_halves(kt[1][0][t], kt[1][1][t]), low_halves(kt[1][2][t], kt[1][3][t]));
               mma16816<T>(acc[1][2 * t + 1], a1[0], a1[1], a1[2], a1[3], high_halves(kt[1][0][t], kt[1][1][t]), high_halves(kt[1][2][t], kt[1][3][t]));
            }
         }
      }
      bool bad = false;
#pragma unroll
      for (int m = 0; m < 2; m++)
#pragma unroll
         for (int t = 0; t < TILES; t++) {
            s.acc[m][t][0] = acc[m][t][0] + acc[m][t][2];
            s.acc[m][t][1] = acc[m][t][1] + acc[m][t][3];
            bad |= s.acc[m][t][0] != s.acc[m][t][0] || s.acc[m][t][1] != s.acc[m][t][1];
         }
      lost = bad;
      s.delta[0] = sum_pairs(s.delta[0]);
      s.delta[1] = sum_pairs(s.delta[1]);
   }

   __device__ __forceinline__ void join_from(const float *unit, const Place &at)
   {
      const float2 *from = reinterpret_cast<const float2 *>(unit) + at.lane;
#pragma unroll
      for (int m = 0; m < 2; m++)
#pragma unroll
         for (int t = 0; t < TILES; t++) {
            const float2 o = from[32 * (m * TILES + t)];
            s.acc[m][t][0] += o.x;
            s.acc[m][t][1] += o.y;
         }
      const float2 d = from[64 * TILES];
      s.delta[0] += d.x;
      s.delta[1] += d.y;
   }
   __device__ __forceinline__ void put(float *unit, const Place &at, int only) const
   {
      float2 *to = reinterpret_cast<float2 *>(unit) + at.lane;
      if (only < 0 || heads.kv == only) {
#pragma unroll
         for (int m = 0; m < 2; m++)
#pragma unroll
            for (int t = 0; t < TILES; t++) to[32 * (m * TILES + t)] = make_float2(s.acc[m][t][0], s.acc[m][t][1]);
      }
      to[64 * TILES] = make_float2(s.delta[0], s.delta[1]);
   }

   __device__ __forceinline__ void finish(const AttnParams &p, const Place &at, long long row, int only)
   {
      const float delta = of_column(s.delta[0], s.delta[1], l.r);
      const bool mine = heads.live && (only < 0 || heads.kv == only);
      const int map = l.r >> 2;
      const long long rh = row * p.heads + heads.head;
      const float factor = map ? -__ldg(p.lam + row * p.ldlam + heads.head) * p.scale : p.scale;
#pragma unroll
      for (int set = 0; set < KOut::SETS; set++)
#pragma unroll
         for (int x = 0; x < 2; x++) {
            float o[KOut::E];
#pragma unroll
            for (int j = 0; j < KOut::E; j++) {
               const int t = set * KOut::E + j;
               // rows 0..3 hold A of map 0 and B of map 1, rows 4..7 B of map 0 and A of map 1
               const float b = __shfl_xor_sync(FULL, map ? s.acc[0][t][x] : s.acc[1][t][x], 16);
               o[j] = factor * fmaf(-delta, b, map ? s.acc[1][t][x] : s.acc[0][t][x]);
            }
            const int y = 8 * KOut::E * set + KOut::E * (2 * l.c + x);
            if (mine) KOut::template store<FORM != PIECES>(static_cast<T *>(p.out) + (rh * 2 + map) * p.d + y, o, p.d - y);
         }
      if (mine && l.c == 0) {
         p.stats[rh * 2 + map] = make_float2(__ldg(p.lse + rh * 2 + map), delta);
         if (map) p.dlam[rh] = -delta;
      }
   }
};

// ---------------------------------------------------------------------------------------------------------------------
// backward over the columns: dk and dv.  Columns of the products are (map, kv head of the unit); a pair is an edge with a
// kv head, taken once for every query head of the group.  dk and dv are [16 elements x 8] products: the inner index is the
// pairs, the columns 0..3 take the upper and 4..7 the lower part of the split ds (or weight) of the unit's kv heads.
// ---------------------------------------------------------------------------------------------------------------------
template <typename T, int DK, int DV, int FORM>
struct BackwardColumnsMma {
   static constexpr int BLOCKS = DV <= 64 ? 4 : DV <= 128 ? 3 : 2;
   using KIn = Inner<T, DK>;
   using KOut = Outer<T, DK>;
   using VIn = Inner<T, DV>;
   using VOut = Outer<T, DV>;
   static constexpr int KT = KOut::REGS, VT = VOut::REGS;
   static constexpr int LANE_FLOATS = 4 * (2 * KT + VT);
   struct State {
      float dk[2][KT][4], dv[VT][4];
   };
   State s;
   Lanes l;
   bool lost;

   __device__ __forceinline__ void setup(const AttnParams &p, const Place &at) { l.set(p, at); }
   static __device__ __forceinline__ void clear(State &s)
   {
#pragma unroll
      for (int t = 0; t < KT; t++)
#pragma unroll
         for (int i = 0; i < 4; i++) s.dk[0][t][i] = s.dk[1][t][i] = 0.0f;
#pragma unroll
      for (int t = 0; t < VT; t++)
#pragma unroll
         for (int i = 0; i < 4; i++) s.dv[t][i] = 0.0f;
   }

   __device__ __forceinline__ void run(const AttnParams &p, const Place &at, EdgeStream &edges, long long col, long long e0, long long e1,
                                       int warp, int warps, int only)
   {
      lost = false;
      clear(s);
      if (e0 + 32 * warp >= e1) return;
      // column n = r: map r / 4, kv head r % 4 of the unit (one that exists stands for those beyond)
      const int n_head = l.kv0 + ((l.r & 3) < l.hs ? l.r & 3 : 0);
      unsigned k[KIn::REGS], v[VIn::REGS];
      KIn::template load<FORM>(static_cast<const T *>(p.k) + col * p.ldk + n_head * p.hsk + (l.r >> 2) * p.d, l.c, p.d, true, p.step, k);
      VIn::template load<FORM>(static_cast<const T *>(p.v) + col * p.ldv + n_head * p.hsv, l.c, p.dv, true, p.step, v);
      const int even = (2 * l.c) & (l.hs - 1), odd = (2 * l.c + 1) & (l.hs - 1);
      const bool skip[2] = {only >= 0 && even != only, only >= 0 && odd != only};
      const int per_step = 16 >> l.hs_log2;
      // of the columns 2c, 2c + 1 at most one is of the pairs' kv head
      const bool valid = (l.c & 1) == l.pair_head >> 1;
      const int x = l.pair_head & 1, map = l.c >> 1;
      for (long long base = e0 + 32 * warp; base < e1; base += 32 * warps) {
         const int my_id = edges.take(p, base, e1, at.lane);
         const float my_bias = edges.bias;
         edges.fetch(p, base + 32 * warps < e1 ? base + 32 * warps : e1 + 32 * warp, at.lane);
         const int count = static_cast<int>(e1 - base < 32 ? e1 - base : 32);
         for (int first = 0; first < count; first += per_step) {
            int id[2];
            float bias[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
               id[h] = __shfl_sync(FULL, my_id, first + l.edge(l.r + 8 * h));
               bias[h] = p.bias ? __shfl_sync(FULL, my_bias, first + l.edge(l.r + 8 * h)) : 0.0f;
            }
            int pair_id[4];
#pragma unroll
            for (int h = 0; h < 4; h++) {
               pair_id[h] = __shfl_sync(FULL, my_id, first + l.edge(2 * l.c + (h & 1) + 8 * (h >> 1)));
               if (skip[h & 1]) pair_id[h] = -1;
            }
            for (int g = 0; g < p.group; g++) {
               const int head = (l.kv0 + l.pair_head) * p.group + g;
               Source<T> qg, dg;
               qg.set(p.q, p.ldq, head * p.hsq);
               dg.set(p.dout, p.ldo, head * p.hso);
               unsigned q[2][2][KIn::REGS], dout[2][VIn::REGS];
               float2 stat[2];
               float lam[2];
#pragma unroll
               for (int h = 0; h < 2; h++) {
                  const T *src = qg.template row<FORM>(id[h]);
                  KIn::template load<FORM>(src, l.c, p.d, id[h] >= 0, p.step, q[0][h]);
                  KIn::template load<FORM>(FORM == EXACT && id[h] < 0 ? src : src + p.d, l.c, p.d, id[h] >= 0, p.step, q[1][h]);
                  VIn::template load<FORM>(dg.template row<FORM>(id[h]), l.c, p.dv, id[h] >= 0, p.step, dout[h]);
                  stat[h] = make_float2(-INFINITY, 0.0f);
                  lam[h] = 0.0f;
                  if (id[h] >= 0 && valid) {
                     stat[h] = __ldg(p.stats + (static_cast<long long>(id[h]) * p.heads + head) * 2 + map);
                     lam[h] = __ldg(p.lam + id[h] * p.ldlam + head);
                  }
               }
               float s0[4] = {0.0f, 0.0f, 0.0f, 0.0f}, s1[4] = {0.0f, 0.0f, 0.0f, 0.0f}, dp[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
               for (int i = 0; i < KIn::STEPS; i++) {
                  mma16816<T>(s0, q[0][0][2 * i], q[0][1][2 * i], q[0][0][2 * i + 1], q[0][1][2 * i + 1], k[2 * i], k[2 * i + 1]);
                  mma16816<T>(s1, q[1][0][2 * i], q[1][1][2 * i], q[1][0][2 * i + 1], q[1][1][2 * i + 1], k[2 * i], k[2 * i + 1]);
               }
#pragma unroll
               for (int i = 0; i < VIn::STEPS; i++)
                  mma16816<T>(dp, dout[0][2 * i], dout[1][2 * i], dout[0][2 * i + 1], dout[1][2 * i + 1], v[2 * i], v[2 * i + 1]);
               unsigned qt[2][4][KT], dt[4][VT];
#pragma unroll
               for (int h = 0; h < 4; h++) {
                  const int other = (l.kv0 + (h & 1 ? odd : even)) * p.group + g;
                  Source<T> qo, dd;
                  qo.set(p.q, p.ldq, other * p.hsq);
                  dd.set(p.dout, p.ldo, other * p.hso);
                  const T *src = qo.template row<FORM>(pair_id[h]);
                  KOut::template load<FORM>(src, l.r, p.d, pair_id[h] >= 0, p.step, qt[0][h]);
                  KOut::template load<FORM>(FORM == EXACT && pair_id[h] < 0 ? src : src + p.d, l.r, p.d, pair_id[h] >= 0, p.step, qt[1][h]);
                  VOut::template load<FORM>(dd.template row<FORM>(pair_id[h]), l.r, p.dv, pair_id[h] >= 0, p.step, dt[h]);
               }
               unsigned b0[2], b1[2], bw[2];
#pragma unroll
               for (int h = 0; h < 2; h++) {
                  const bool live = stat[h].x != -INFINITY;  // an edge of a row that has any, and this lane's column is the pair's
                  const float dot = map ? (x ? s1[2 * h + 1] : s1[2 * h]) : (x ? s0[2 * h + 1] : s0[2 * h]);
                  const float pr = live ? exp2_fast((fmaf(dot, p.scale, bias[h]) - stat[h].x) * LOG2E) : 0.0f;
                  const float part = live ? (map ? -lam[h] : 1.0f) * pr : 0.0f;  // this map's part of the weight
                  const float w = part + __shfl_xor_sync(FULL, part, 2);
                  const float ds = live ? part * ((x ? dp[2 * h + 1] : dp[2 * h]) - stat[h].y) : 0.0f;
                  unsigned hi, lo, wh, wl;
                  split2<T>(x ? 0.0f : ds, x ? ds : 0.0f, hi, lo);
                  split2<T>(x ? 0.0f : w, x ? w : 0.0f, wh, wl);
                  const unsigned got = __shfl_xor_sync(FULL, l.c < 2 ? lo : hi, 2);
                  b0[h] = transpose8x8(l.c < 2 ? hi : got);
                  b1[h] = transpose8x8(l.c < 2 ? got : lo);
                  bw[h] = transpose8x8(l.c < 2 ? wh : wl);
               }
#pragma unroll
               for (int t = 0; t < KT; t++) {
                  mma16816<T>(s.dk[0][t], low_halves(qt[0][0][t], qt[0][1][t]), high_halves(qt[0][0][t], qt[0][1][t]),
                              low_halves(qt[0][2][t], qt[0][3][t]), high_halves(qt[0][2][t], qt[0][3][t]), b0[0], b0[1]);
                  mma16816<T>(s.dk[1][t], low_halves(qt[1][0][t], qt[1][1][t]), high_halves(qt[1][0][t], qt[1][1][t]),
                              low_halves(qt[1][2][t], qt[1][3][t]), high_halves(qt[1][2][t], qt[1][3][t]), b1[0], b1[1]);
               }
#pragma unroll
               for (int t = 0; t < VT; t++)
                  mma16816<T>(s.dv[t], low_halves(dt[0][t], dt[1][t]), high_halves(dt[0][t], dt[1][t]), low_halves(dt[2][t], dt[3][t]),
                              high_halves(dt[2][t], dt[3][t]), bw[0], bw[1]);
            }
         }
      }
      bool bad = false;
#pragma unroll
      for (int t = 0; t < KT; t++)
#pragma unroll
         for (int i = 0; i < 4; i++) bad |= s.dk[0][t][i] != s.dk[0][t][i] || s.dk[1][t][i] != s.dk[1][t][i];
#pragma unroll
      for (int t = 0; t < VT; t++)
#pragma unroll
         for (int i = 0; i < 4; i++) bad |= s.dv[t][i] != s.dv[t][i];
      lost = bad;
   }

   __device__ __forceinline__ void join_from(const float *unit, const Place &at)
   {
      const float4 *from = reinterpret_cast<const float4 *>(unit) + at.lane;
#pragma unroll
      for (int i = 0; i < 2 * KT + VT; i++) {
         const float4 o = from[32 * i];
         float (&f)[4] = i < KT ? s.dk[0][i] : i < 2 * KT ? s.dk[1][i - KT] : s.dv[i - 2 * KT];
         f[0] += o.x; f[1] += o.y; f[2] += o.z; f[3] += o.w;
      }
   }
   // a head's sums lie in the results' columns 2c, 2c + 1 (and 4 further): the lane's kv heads 2c % 4, 2c % 4 + 1
   __device__ __forceinline__ void put(float *unit, const Place &at, int only) const
   {
      float4 *to = reinterpret_cast<float4 *>(unit) + at.lane;
      const int kv = (2 * l.c) & 3;
#pragma unroll
      for (int i = 0; i < 2 * KT + VT; i++) {
         const float (&f)[4] = i < KT ? s.dk[0][i] : i < 2 * KT ? s.dk[1][i - KT] : s.dv[i - 2 * KT];
         if (only < 0) {
            to[32 * i] = make_float4(f[0], f[1], f[2], f[3]);
         } else {
            float *one = reinterpret_cast<float *>(to + 32 * i);
            if (kv == only) { one[0] = f[0]; one[2] = f[2]; }
            if (kv + 1 == only) { one[1] = f[1]; one[3] = f[3]; }
         }
      }
   }

   template <typename Out, int REGS>
   __device__ __forceinline__ void write(const float (&f)[REGS][4], T *row, long long head_step, int width, float factor, int only)
   {
#pragma unroll
      for (int set = 0; set < Out::SETS; set++)
#pragma unroll
         for (int x = 0; x < 2; x++) {
            float o[Out::E];
#pragma unroll
            for (int j = 0; j < Out::E / 2; j++) {
               const float lo = f[set * (Out::E / 2) + j][x], hi = f[set * (Out::E / 2) + j][2 + x];
               o[2 * j] = factor * (lo + __shfl_xor_sync(FULL, lo, 2));
               o[2 * j + 1] = factor * (hi + __shfl_xor_sync(FULL, hi, 2));
            }
            const int kv = 2 * l.c + x, y = 8 * Out::E * set + Out::E * l.r;
            if (l.c < 2 && kv < l.hs && (only < 0 || kv == only))
               Out::template store<FORM != PIECES>(row + kv * head_step + y, o, width - y);
         }
   }
   __device__ __forceinline__ void finish(const AttnParams &p, const Place &at, long long col, int only)
   {
      const long long rh = col * p.kv_heads + l.kv0;
      write<KOut, KT>(s.dk[0], static_cast<T *>(p.out) + rh * 2 * p.d, 2 * p.d, p.d, p.scale, only);
      write<KOut, KT>(s.dk[1], static_cast<T *>(p.out) + rh * 2 * p.d + p.d, 2 * p.d, p.d, p.scale, only);
      write<VOut, VT>(s.dv, static_cast<T *>(p.out2) + rh * p.dv, p.dv, p.dv, 1.0f, only);
   }
};

template <typename T, int DK, template <typename, int, int, int> class Op>
int launch_mma_width(const WalkShape &s, const AttnParams &p, cudaStream_t st)
{
   if (s.form == EXACT) return launch_op<Op<T, DK, 2 * DK, EXACT>, 32>(p, s.together, st);
   if (s.form == RAGGED) return launch_op<Op<T, DK, 2 * DK, RAGGED>, 32>(p, s.together, st);
   return launch_op<Op<T, DK, 2 * DK, PIECES>, 32>(p, s.together, st);
}

template <typename T, template <typename, int, int, int> class Op>
int launch_mma(const WalkShape &s, const AttnParams &p, cudaStream_t st)
{
   if (s.width == 16) return launch_mma_width<T, 16, Op>(s, p, st);
   if (s.width == 32) return launch_mma_width<T, 32, Op>(s, p, st);
   if (s.width == 64) return launch_mma_width<T, 64, Op>(s, p, st);
   if (s.width == 128) return launch_mma_width<T, 128, Op>(s, p, st);
   return -1;
}

}  // namespace attn
}  // namespace fmm

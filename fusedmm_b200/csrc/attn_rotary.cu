// attn_rotary.cu -- the norm of queries and keys for each head with the rotation by their positions, forward and backward
// (include/fusedmm_b200.h, fusedmm_b200_qk_norm_rotary).
//
//   y = x * rsqrt(mean(x^2) + eps) * w;  theta_i = sum_a pos[a] * freq[a][i];
//   (y_lo, y_hi) -> (y_lo cos - y_hi sin, y_hi cos + y_lo sin) for the pairs i < P; what lies behind the pairs passes.
//   backward, g = dy turned back:  dw = sum_rows,heads g x r;  dx = r (w g - x r mean(w g x r)), r the root's reciprocal.
//
// Bound: bytes; every element is read and written once, and the arithmetic (some 6 instructions an element with the conversions)
// has to stay out of the way.  A head is cut into units of two vectors that hold the two halves of the same pairs, one unit to
// a lane, so the rotation needs no exchange between lanes and the norm one butterfly over the lanes of the head.  A group of
// lanes (a slot) takes a row and goes through its heads: a lane's sines and weights stay in its registers, and the next
// heads are on their way from memory.  Angles are formed in 64 bits up to the fraction of a turn (2^20 positions times a
// frequency leave no digit of the angle in 32).
#include "../../include/fusedmm_b200.h"
#include "attn_common.cuh"
#include "attn_host.h"

namespace fmm {
namespace attn {

// Heads of a row on their way from memory: one 262 us, two 249, three 232, four 230 (65536 x 40 heads of 128, bf16; the bytes need
// 205), and four take the registers of a quarter of the warps from float (100003 x 8 heads of 40: 67, 65, 63, 77 us).
constexpr int ROT_AHEAD = 3;
constexpr int ROT_THREADS = 256;
// Units of a lane where a row in single elements or in twos has more than 32: 32 lanes x 4 units of 2 elements, or x 2 of 4, are 256.
constexpr int ROT_SCALAR_UNITS = 4, ROT_PAIR_UNITS = 2;

struct RotaryParams {
   const void *x[2];     // queries, keys
   const void *dy[2];
   void *y[2];           // forward: results; backward: gradients of x
   long long ldx[2], hsx[2], ldd[2], hsd[2];  // strides of rows and heads, in elements (x and dy); results are dense
   const void *w[2];
   int heads[2];
   const void *pos;
   long long ldp, asp;   // strides of pos: rows, axes
   const double *freq;   // [axes][pairs]
   float *dw_partial;    // [blocks][2][d]
   long long rows;
   int d, pairs, axes, pos_type, w_f32, interleaved, norm, lanes_log2, units, splits;
   float eps;
};

__device__ __forceinline__ double position(const RotaryParams &p, long long row, int axis)
{
   const long long at = row * p.ldp + axis * p.asp;
   switch (p.pos_type) {
      case FUSEDMM_B200_POS_I32: return static_cast<double>(__ldg(static_cast<const int *>(p.pos) + at));
      case FUSEDMM_B200_POS_I64: return static_cast<double>(__ldg(static_cast<const long long *>(p.pos) + at));
      case FUSEDMM_B200_POS_F32: return static_cast<double>(__ldg(static_cast<const float *>(p.pos) + at));
      default: return __ldg(static_cast<const double *>(p.pos) + at);
   }
}

// cosine and sine of pair i of a row
__device__ __forceinline__ void angle_of(const RotaryParams &p, const double (&pos)[FUSEDMM_B200_ROTARY_MAX_AXES], int i, float &c, float &s)
{
   double angle = 0.0;
#pragma unroll
   for (int a = 0; a < FUSEDMM_B200_ROTARY_MAX_AXES; a++)
      if (a < p.axes) angle = fma(pos[a], __ldg(p.freq + a * p.pairs + i), angle);
   const double half_turns = angle * 0.31830988618379067154;  // 1/pi
   // only the fraction of a turn matters; it fits 32 bits once the whole turns are gone
   sincospif(static_cast<float>(half_turns - 2.0 * rint(half_turns * 0.5)), &s, &c);
}

// One unit: 2W elements in two vectors, W pairs.  Of the halves form unit u < pairs / W holds elements [uW, uW+W) and
// [P+uW, P+uW+W), and units behind the pairs consecutive vectors; of the interleaved form every unit is two consecutive vectors.
template <int W>
struct Unit {
   int at[2];    // element index of the two vectors, -1: none
   int pair;     // first pair, -1: nothing to turn
   bool whole;   // both vectors turn (interleaved pairs may end after the first)
   __device__ __forceinline__ void place(const RotaryParams &p, int u, bool inter)
   {
      pair = -1;
      whole = true;
      at[0] = at[1] = -1;
      if (u >= p.units) return;
      if (inter && W > 1) {
         at[0] = 2 * u * W;
         at[1] = at[0] + W < p.d ? at[0] + W : -1;
         if (u * W < p.pairs) pair = u * W;
         whole = u * W + W <= p.pairs;
         return;
      }
      const int up = p.pairs / W;
      if (u < up) {
         pair = u * W;
         at[0] = p.interleaved ? 2 * u * W : u * W;  // (W = 1: both forms)
         at[1] = p.interleaved ? at[0] + W : p.pairs + u * W;
      } else {
         at[0] = 2 * p.pairs + 2 * (u - up) * W;
         at[1] = at[0] + W < p.d ? at[0] + W : -1;
      }
   }
};

// Turns a unit, back with BACK.  c, s: cosines and sines of its pairs, two to a register pair.
template <int W, bool INTER, bool BACK>
__device__ __forceinline__ void turn(F2 (&lo)[(W + 1) / 2], F2 (&hi)[(W + 1) / 2], const F2 (&c)[(W + 1) / 2], const F2 (&s)[(W + 1) / 2], bool whole)
{
   if constexpr (INTER && W > 1) {
      // the two vectors are consecutive: pair j is elements 2j, 2j + 1 of their 2W, one register pair
#pragma unroll
      for (int j = 0; j < W; j++) {
         if (j >= W / 2 && !whole) break;
         F2 &x = j < W / 2 ? lo[j % (W / 2)] : hi[j % (W / 2)];
         const float2 v = f2_parts(x), cc = f2_parts(c[j / 2]), ss = f2_parts(s[j / 2]);
         const float cj = j & 1 ? cc.y : cc.x, sj = BACK ? -(j & 1 ? ss.y : ss.x) : (j & 1 ? ss.y : ss.x);
         x = f2(fmaf(v.x, cj, -v.y * sj), fmaf(v.y, cj, v.x * sj));
      }
   } else {
      const F2 minus = f2(-1.0f, -1.0f);
#pragma unroll
      for (int j = 0; j < (W + 1) / 2; j++) {
         const F2 negative = mul2(s[j], minus), up = BACK ? negative : s[j], down = BACK ? s[j] : negative;
         const F2 a = fma2(lo[j], c[j], mul2(hi[j], down));
         hi[j] = fma2(hi[j], c[j], mul2(lo[j], up));
         lo[j] = a;
      }
   }
}

// A unit's two vectors as they come from memory, and as numbers.
template <typename T, int W>
struct Unpacked {
   static constexpr int P = (W + 1) / 2;
   uint4 r[2];  // (W = 1: the number's bits; 8-byte vectors: the first half)
   __device__ __forceinline__ void load(const T *base, const Unit<W> &u, bool live)
   {
#pragma unroll
      for (int s = 0; s < 2; s++) {
         const bool there = live && u.at[s] >= 0;
         if constexpr (W == 1) {
            r[s].x = there ? __float_as_uint(Elt<T>::up(base[u.at[s]])) : 0u;
         } else if constexpr (W * sizeof(T) == 4) {
            r[s].x = there ? __ldg(reinterpret_cast<const unsigned *>(base + u.at[s])) : 0u;
         } else if constexpr (W * sizeof(T) == 8) {
            const uint2 v = there ? __ldg(reinterpret_cast<const uint2 *>(base + u.at[s])) : make_uint2(0u, 0u);
            r[s] = make_uint4(v.x, v.y, 0u, 0u);
         } else r[s] = there ? ldg16(base + u.at[s]) : make_uint4(0u, 0u, 0u, 0u);
      }
   }
   __device__ __forceinline__ void unpack(F2 (&f)[2][P]) const
   {
#pragma unroll
      for (int s = 0; s < 2; s++) {
         if constexpr (W == 1) {
            f[s][0] = f2(__uint_as_float(r[s].x), 0.0f);
         } else if constexpr (W == 2 && sizeof(T) == 4) {
            f[s][0] = f2(__uint_as_float(r[s].x), __uint_as_float(r[s].y));
         } else if constexpr (W == 2) {
            float a, b;
            Elt<T>::unpack2(r[s].x, a, b);
            f[s][0] = f2(a, b);
         } else if constexpr (W * sizeof(T) == 8) {
            float a, b;
            Elt<T>::unpack2(r[s].x, a, b);
            f[s][0] = f2(a, b);
            Elt<T>::unpack2(r[s].y, a, b);
            f[s][1] = f2(a, b);
         } else {
            unpack_pairs<T>(r[s], f[s]);
         }
      }
   }
};
template <typename T, int W>
__device__ __forceinline__ void store_part(T *base, int at, const F2 (&f)[(W + 1) / 2])
{
   if (at < 0) return;
   if constexpr (W == 1) {
      base[at] = Elt<T>::down(f2_parts(f[0]).x);
   } else {
      float o[W];
#pragma unroll
      for (int i = 0; i < W / 2; i++) {
         const float2 v = f2_parts(f[i]);
         o[2 * i] = v.x;
         o[2 * i + 1] = v.y;
      }
      if constexpr (W == 2 && sizeof(T) == 4) *reinterpret_cast<float2 *>(base + at) = make_float2(o[0], o[1]);
      else if constexpr (W == 2) *reinterpret_cast<unsigned *>(base + at) = Elt<T>::pack2(o[0], o[1]);
      else if constexpr (W * sizeof(T) == 8) *reinterpret_cast<uint2 *>(base + at) = make_uint2(Elt<T>::pack2(o[0], o[1]), Elt<T>::pack2(o[2], o[3]));
      else *reinterpret_cast<uint4 *>(base + at) = Elt<T>::pack(o);
   }
}

// LOG2: a slot has 2^LOG2 lanes, or 2^p.lanes_log2 with -1
template <int LOG2>
__device__ __forceinline__ float sum_over(float v, int lanes_log2)
{
   if constexpr (LOG2 >= 0) {
#pragma unroll
      for (int s = 0; s < LOG2; s++) v += __shfl_xor_sync(FULL, v, 1 << s);
   } else {
      for (int s = 0; s < lanes_log2; s++) v += __shfl_xor_sync(FULL, v, 1 << s);
   }
   return v;
}

// NU: units of a lane (1 with vectors of 16 or 8 bytes).  INTER: pairs side by side.  AHEAD heads of a row are on their way from memory.
// (Float forward: three blocks of a multiprocessor, 64 us for 100003 x 8 heads of 40 against 82 with two; the others want their
// registers: 16384 rows of 20 heads backward 42 us, 52 with two blocks, 89 with three.)
template <typename T, int W, int NU, int LOG2, bool INTER, bool BACKWARD>
__global__ void __launch_bounds__(ROT_THREADS, sizeof(T) == 4 && NU == 1 && !BACKWARD ? 3 : 1) rotary_kernel(const RotaryParams p)
{
   constexpr int P = (W + 1) / 2, AHEAD = NU > 2 ? 1 : ROT_AHEAD;
   __shared__ float sums[BACKWARD ? ROT_THREADS * NU * 2 * W : 1];
   const int lanes_log2 = LOG2 >= 0 ? LOG2 : p.lanes_log2, lanes = 1 << lanes_log2;
   const int lane = threadIdx.x & (lanes - 1), slot = threadIdx.x >> lanes_log2, slots = ROT_THREADS >> lanes_log2;
   Unit<W> unit[NU];
#pragma unroll
   for (int i = 0; i < NU; i++) unit[i].place(p, lane + i * 32, INTER);
   F2 dw[BACKWARD ? 2 : 1][NU][2][P] = {};
   const float inv_d = 1.0f / p.d;
   // the block's part of the heads
   const int part = blockIdx.y;
   int h0[2], h1[2];
#pragma unroll
   for (int which = 0; which < 2; which++) {
      h0[which] = static_cast<int>(static_cast<long long>(p.heads[which]) * part / p.splits);
      h1[which] = static_cast<int>(static_cast<long long>(p.heads[which]) * (part + 1) / p.splits);
   }
   for (long long row0 = static_cast<long long>(blockIdx.x) * slots; row0 < p.rows; row0 += static_cast<long long>(gridDim.x) * slots) {
      // every lane of a warp runs every round: the butterflies need them all
      const bool live = row0 + slot < p.rows;
      const long long row = live ? row0 + slot : row0;
      F2 c[NU][P], s[NU][P];
      bool turned = false;
#pragma unroll
      for (int which = 0; which < 2; which++) {
         const int heads = h1[which] - h0[which];
         if (heads <= 0) continue;
         Unpacked<T, W> x[AHEAD][NU], dy[BACKWARD ? AHEAD : 1][NU];
         const T *src = static_cast<const T *>(p.x[which]) + row * p.ldx[which] + h0[which] * p.hsx[which], *dsrc = nullptr;
         if constexpr (BACKWARD) dsrc = static_cast<const T *>(p.dy[which]) + row * p.ldd[which] + h0[which] * p.hsd[which];
         T *y = static_cast<T *>(p.y[which]) + (row * p.heads[which] + h0[which]) * p.d;
         auto fetch = [&](int k, bool there) {
#pragma unroll
            for (int i = 0; i < NU; i++) {
               x[k][i].load(src, unit[i], there);
               if constexpr (BACKWARD) dy[BACKWARD ? k : 0][i].load(dsrc, unit[i], there);
            }
            src += p.hsx[which];
            if constexpr (BACKWARD) dsrc += p.hsd[which];
         };
#pragma unroll
         for (int k = 0; k < AHEAD; k++) fetch(k, live && k < heads);
         if (!turned) {  // while the first heads are on their way
            turned = true;
            double pos[FUSEDMM_B200_ROTARY_MAX_AXES];
#pragma unroll
            for (int a = 0; a < FUSEDMM_B200_ROTARY_MAX_AXES; a++) pos[a] = p.pairs > 0 && a < p.axes ? position(p, row, a) : 0.0;
#pragma unroll
            for (int i = 0; i < NU; i++)
#pragma unroll
               for (int j = 0; j < P; j++) {
                  float cc[2] = {1.0f, 1.0f}, ss[2] = {0.0f, 0.0f};
#pragma unroll
                  for (int o = 0; o < (W == 1 ? 1 : 2); o++)
                     if (unit[i].pair >= 0 && unit[i].pair + 2 * j + o < p.pairs) angle_of(p, pos, unit[i].pair + 2 * j + o, cc[o], ss[o]);
                  c[i][j] = f2(cc[0], cc[1]);
                  s[i][j] = f2(ss[0], ss[1]);
               }
         }
         F2 w[NU][2][P];
#pragma unroll
         for (int i = 0; i < NU; i++)
#pragma unroll
            for (int v = 0; v < 2; v++)
#pragma unroll
               for (int j = 0; j < P; j++) {
                  float e[2] = {1.0f, 1.0f};
#pragma unroll
                  for (int o = 0; o < (W == 1 ? 1 : 2); o++)
                     if (p.w[which] && unit[i].at[v] >= 0) {
                        const int at = unit[i].at[v] + 2 * j + o;
                        e[o] = p.w_f32 ? __ldg(static_cast<const float *>(p.w[which]) + at) : Elt<T>::up(static_cast<const T *>(p.w[which])[at]);
                     }
                  w[i][v][j] = f2(e[0], e[1]);
               }
         for (int n = 0; n < heads; n += AHEAD) {
#pragma unroll
            for (int k = 0; k < AHEAD; k++) {
               if (n + k >= heads) break;
               F2 v[NU][2][P], g[BACKWARD ? NU : 1][2][P];
#pragma unroll
               for (int i = 0; i < NU; i++) {
                  x[k][i].unpack(v[i]);
                  if constexpr (BACKWARD) dy[BACKWARD ? k : 0][i].unpack(g[BACKWARD ? i : 0]);
               }
               fetch(k, live && n + k + AHEAD < heads);
               F2 rr = f2(1.0f, 1.0f);
               if (p.norm) {
                  F2 squares = 0;
#pragma unroll
                  for (int i = 0; i < NU; i++)
#pragma unroll
                     for (int j = 0; j < P; j++) squares = fma2(v[i][0][j], v[i][0][j], fma2(v[i][1][j], v[i][1][j], squares));
                  const float r = rsqrtf(fmaf(sum_over<LOG2>(sum2(squares), lanes_log2), inv_d, p.eps));
                  rr = f2(r, r);
               }
               if constexpr (!BACKWARD) {
#pragma unroll
                  for (int i = 0; i < NU; i++) {
                     if (p.norm) {
#pragma unroll
                        for (int o = 0; o < 2; o++)
#pragma unroll
                           for (int j = 0; j < P; j++) v[i][o][j] = mul2(mul2(v[i][o][j], rr), w[i][o][j]);
                     }
                     if (unit[i].pair >= 0) turn<W, INTER, false>(v[i][0], v[i][1], c[i], s[i], unit[i].whole);
                     if (live) {
                        store_part<T, W>(y, unit[i].at[0], v[i][0]);
                        store_part<T, W>(y, unit[i].at[1], v[i][1]);
                     }
                  }
               } else {
                  F2 dots = 0;
#pragma unroll
                  for (int i = 0; i < NU; i++) {
                     if (unit[i].pair >= 0) turn<W, INTER, true>(g[i][0], g[i][1], c[i], s[i], unit[i].whole);
                     if (p.norm) {
#pragma unroll
                        for (int o = 0; o < 2; o++)
#pragma unroll
                           for (int j = 0; j < P; j++) {
                              v[i][o][j] = mul2(v[i][o][j], rr);
                              // (a slot without a row has zeros, but with eps 0 the root of nothing is infinite)
                              if (live) dw[BACKWARD ? which : 0][i][o][j] = fma2(g[i][o][j], v[i][o][j], dw[BACKWARD ? which : 0][i][o][j]);
                              g[i][o][j] = mul2(g[i][o][j], w[i][o][j]);
                              dots = fma2(g[i][o][j], v[i][o][j], dots);
                           }
                     }
                  }
                  if (p.norm) {
                     const float dot = -sum_over<LOG2>(sum2(dots), lanes_log2) * inv_d;
                     const F2 dd = f2(dot, dot);
#pragma unroll
                     for (int i = 0; i < NU; i++)
#pragma unroll
                        for (int o = 0; o < 2; o++)
#pragma unroll
                           for (int j = 0; j < P; j++) g[i][o][j] = mul2(rr, fma2(v[i][o][j], dd, g[i][o][j]));
                  }
                  if (live) {
#pragma unroll
                     for (int i = 0; i < NU; i++) {
                        store_part<T, W>(y, unit[i].at[0], g[i][0]);
                        store_part<T, W>(y, unit[i].at[1], g[i][1]);
                     }
                  }
               }
               y += p.d;
            }
         }
      }
   }
   if constexpr (BACKWARD) {
      if (!p.dw_partial) return;
      // the block's share of the weight gradients: every slot's sums side by side, added in the order of the slots
      const long long block = static_cast<long long>(blockIdx.y) * gridDim.x + blockIdx.x;
#pragma unroll
      for (int which = 0; which < 2; which++) {
         __syncthreads();
#pragma unroll
         for (int i = 0; i < NU; i++)
#pragma unroll
            for (int o = 0; o < 2; o++)
               if (unit[i].at[o] >= 0)
#pragma unroll
                  for (int j = 0; j < W; j++) {
                     const float2 v = f2_parts(dw[which][i][o][j / 2]);
                     sums[slot * p.d + unit[i].at[o] + j] = j & 1 ? v.y : v.x;
                  }
         __syncthreads();
         for (int e = threadIdx.x; e < p.d; e += ROT_THREADS) {
            float t = 0.0f;
            for (int s2 = 0; s2 < slots; s2++) t += sums[s2 * p.d + e];
            p.dw_partial[(block * 2 + which) * p.d + e] = t;
         }
      }
   }
}

// dw[which][e] = sum over the blocks; 32 columns to a block, its 32 warps take the partial rows in turn
__global__ void __launch_bounds__(1024) rotary_dw_kernel(const float *partial, int blocks, int d, float *dwq, float *dwk)
{
   __shared__ float part[32][33];
   const int lane = threadIdx.x & 31, col = blockIdx.x * 32 + lane, w = threadIdx.x >> 5;
   float t = 0.0f;
   if (col < 2 * d) {
#pragma unroll 4
      for (int b = w; b < blocks; b += 32) t += partial[static_cast<long long>(b) * 2 * d + col];
   }
   part[w][lane] = t;
   __syncthreads();
   // warp w adds up column w of the 32
   float s = part[lane][w];
#pragma unroll
   for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(FULL, s, x);
   const int mine = blockIdx.x * 32 + w;
   if (lane == 0 && mine < 2 * d) {
      float *out = mine < d ? dwq : dwk;
      if (out) out[mine < d ? mine : mine - d] = s;
   }
}

namespace {

int ceil_log2(int n)
{
   int l = 0;
   while ((1 << l) < n) l++;
   return l;
}

constexpr int ROT_BACKWARD_BLOCKS_PER_SM = 4;

// Heads of a row go to one slot, which forms the row's sines once, unless there are too few rows to give every SM this many
// warps (16384 rows of 20 heads of 64: 19 us with 12, 24 with 24, which forms the sines twice).
constexpr int ROT_WARPS = 12;
int choose_splits(const RotaryParams &p, int sm_count)
{
   const long long warps = ((p.rows << p.lanes_log2) + 31) / 32, wanted = static_cast<long long>(ROT_WARPS) * sm_count;
   const int most = p.heads[0] > p.heads[1] ? p.heads[0] : p.heads[1];
   const long long splits = (wanted + warps - 1) / warps;
   return static_cast<int>(splits < 1 ? 1 : splits > most ? most : splits);
}

template <typename T, int W, int NU, int LOG2, bool BACKWARD>
void launch_form(const RotaryParams &p, dim3 grid, cudaStream_t st)
{
   if (p.interleaved || W == 1) rotary_kernel<T, W, NU, LOG2, true, BACKWARD><<<grid, ROT_THREADS, 0, st>>>(p);
   else rotary_kernel<T, W, NU, LOG2, false, BACKWARD><<<grid, ROT_THREADS, 0, st>>>(p);
}

// returns the number of blocks; width: elements of a vector (16 or 8 bytes of them, 2 or 1)
template <typename T, bool BACKWARD>
int launch(RotaryParams &p, int width, int sm_count, cudaStream_t st)
{
   constexpr int W = Elt<T>::W, HALF = sizeof(T) == 2 ? W / 2 : W;
   const int behind = (p.d - 2 * p.pairs) / width;
   p.units = p.interleaved && width > 1 ? (p.d / width + 1) / 2 : p.pairs / width + (behind + 1) / 2;
   p.lanes_log2 = p.units <= 32 ? ceil_log2(p.units) : 5;
   p.splits = choose_splits(p, sm_count);
   const int slots = ROT_THREADS >> p.lanes_log2;
   const long long blocks = (p.rows + slots - 1) / slots;
   // backward: each block adds up the weight gradients of many rows
   long long cap = BACKWARD ? static_cast<long long>(sm_count) * ROT_BACKWARD_BLOCKS_PER_SM / p.splits : 0x7fffffffLL;
   cap = cap < 1 ? 1 : cap;
   const dim3 grid(static_cast<unsigned>(blocks < cap ? blocks : cap), p.splits);
   if (width == 1 && p.units > 32) launch_form<T, 1, ROT_SCALAR_UNITS, 5, BACKWARD>(p, grid, st);
   else if (width == 1) launch_form<T, 1, 1, -1, BACKWARD>(p, grid, st);
   else if (width == 2 && p.units > 32) launch_form<T, 2, ROT_PAIR_UNITS, 5, BACKWARD>(p, grid, st);
   else if (width == 2) launch_form<T, 2, 1, -1, BACKWARD>(p, grid, st);
   else if (width < W) launch_form<T, HALF, 1, -1, BACKWARD>(p, grid, st);
   else if (p.lanes_log2 == 2) launch_form<T, W, 1, 2, BACKWARD>(p, grid, st);
   else if (p.lanes_log2 == 3) launch_form<T, W, 1, 3, BACKWARD>(p, grid, st);
   else if (p.lanes_log2 == 4) launch_form<T, W, 1, 4, BACKWARD>(p, grid, st);
   else launch_form<T, W, 1, -1, BACKWARD>(p, grid, st);
   return static_cast<int>(grid.x * grid.y);
}

bool multiple(const void *p, long long a, long long b, int width, size_t elt)
{
   return reinterpret_cast<uintptr_t>(p) % (width * elt) == 0 && a % width == 0 && b % width == 0;
}

// what both directions check and fill in; 0 or a status
int rotary_setup(RotaryParams &p, int32_t dtype, int64_t rows, int32_t hq, int32_t hk, int32_t d, const void *q, int64_t ldq,
                 int64_t hsq, const void *k, int64_t ldk, int64_t hsk, int32_t w_dtype, const void *wq, const void *wk,
                 int32_t norm, double eps, int32_t pos_type, const void *pos, int64_t ldp, int64_t asp, int32_t axes,
                 const double *freq, int32_t pairs, int32_t interleaved)
{
   if (dtype != DT_F32 && dtype != DT_BF16 && dtype != DT_F16) return FUSEDMM_B200_ERR_ARG;
   if (rows < 0 || hq < 0 || hk < 0 || d < 1 || pairs < 0 || 2LL * pairs > d) return FUSEDMM_B200_ERR_ARG;
   if (d > FUSEDMM_B200_ATTN_MAX_WIDTH || hq > FUSEDMM_B200_ATTN_MAX_HEADS || hk > FUSEDMM_B200_ATTN_MAX_HEADS) return FUSEDMM_B200_ERR_LIMIT;
   for (int64_t s : {ldq, hsq, ldk, hsk})
      if (s < 0) return FUSEDMM_B200_ERR_LIMIT;
   if (norm && !(eps >= 0.0)) return FUSEDMM_B200_ERR_ARG;
   if (!norm && (wq || wk)) return FUSEDMM_B200_ERR_ARG;
   if (w_dtype != DT_F32 && w_dtype != dtype) return FUSEDMM_B200_ERR_ARG;
   if (pairs > 0) {
      if (axes < 1 || axes > FUSEDMM_B200_ROTARY_MAX_AXES) return FUSEDMM_B200_ERR_ARG;
      if (pos_type < FUSEDMM_B200_POS_I32 || pos_type > FUSEDMM_B200_POS_F64) return FUSEDMM_B200_ERR_ARG;
   }
   if (rows > 0) {
      if ((hq > 0 && !q) || (hk > 0 && !k) || (pairs > 0 && (!pos || !freq))) return FUSEDMM_B200_ERR_ARG;
      if (!on_device({hq > 0 ? q : nullptr, hk > 0 ? k : nullptr, wq, wk, pairs > 0 ? pos : nullptr,
                      pairs > 0 ? static_cast<const void *>(freq) : nullptr}))
         return FUSEDMM_B200_ERR_ARG;
   }
   p.x[0] = q; p.x[1] = k;
   p.ldx[0] = ldq; p.ldx[1] = ldk; p.hsx[0] = hsq; p.hsx[1] = hsk;
   p.w[0] = wq; p.w[1] = wk;
   p.w_f32 = w_dtype == DT_F32;
   p.heads[0] = hq; p.heads[1] = hk;
   p.pos = pos; p.ldp = ldp; p.asp = asp; p.freq = freq;
   p.rows = rows; p.d = d; p.pairs = pairs; p.axes = pairs > 0 ? axes : 0; p.pos_type = pos_type;
   p.interleaved = interleaved != 0; p.norm = norm != 0; p.eps = static_cast<float>(eps);
   return 0;
}

// Elements of the vectors the rows can be taken in: 16 bytes, for 16-bit types also 8, else two, else 1.
// (15688 rows of 20 heads of 234 in half: 98 us in twos, 290 in single elements; the bytes need 45.  50000 rows of 12 heads of 40 in
// bf16 with 15 pairs, single elements: 116 us with the 32 lanes its 20 units take, 341 with four units to a lane.)
int rotary_width(const RotaryParams &p, int32_t dtype, bool backward)
{
   const size_t elt = dtype == DT_F32 ? 4 : 2;
   for (int width = dtype == DT_F32 ? 4 : 8; width >= 2; width /= 2) {
      // pairs: whole vectors of halves; interleaved whole vectors
      bool fits = p.d % width == 0 && (p.interleaved ? 2 * p.pairs % width == 0 : p.pairs % width == 0);
      for (int i = 0; i < 2 && fits; i++) {
         if (!p.heads[i]) continue;
         fits = multiple(p.x[i], p.ldx[i], p.hsx[i], width, elt) && multiple(p.y[i], 0, 0, width, elt) &&
                (!backward || multiple(p.dy[i], p.ldd[i], p.hsd[i], width, elt));
      }
      // (a lane takes one unit of 2 width elements: 32 of them hold 256 elements in vectors of 4 and more; two units in twos)
      if (fits) return width;
   }
   return 1;
}

template <bool BACKWARD>
int rotary_launch(RotaryParams &p, int32_t dtype, int width, int sm_count, cudaStream_t st)
{
   if (dtype == DT_F32) return launch<float, BACKWARD>(p, width, sm_count, st);
   if (dtype == DT_BF16) return launch<__nv_bfloat16, BACKWARD>(p, width, sm_count, st);
   return launch<__half, BACKWARD>(p, width, sm_count, st);
}

}  // namespace
}  // namespace attn
}  // namespace fmm

using namespace fmm::attn;

extern "C" {

int fusedmm_b200_qk_norm_rotary(int32_t dtype, int64_t rows, int32_t hq, int32_t hk, int32_t d, const void *q, int64_t ldq,
                                int64_t hsq, const void *k, int64_t ldk, int64_t hsk, int32_t w_dtype, const void *wq,
                                const void *wk, int32_t norm, double eps, int32_t pos_type, const void *pos, int64_t ldp,
                                int64_t asp, int32_t axes, const double *freq, int32_t pairs, int32_t interleaved,
                                void *q_out, void *k_out, void *stream)
{
   RotaryParams p = {};
   if (int s = rotary_setup(p, dtype, rows, hq, hk, d, q, ldq, hsq, k, ldk, hsk, w_dtype, wq, wk, norm, eps, pos_type, pos,
                            ldp, asp, axes, freq, pairs, interleaved)) return s;
   if (rows == 0 || hq + hk == 0) return 0;
   if ((hq > 0 && !q_out) || (hk > 0 && !k_out) || !on_device({hq > 0 ? q_out : nullptr, hk > 0 ? k_out : nullptr}))
      return FUSEDMM_B200_ERR_ARG;
   p.y[0] = q_out; p.y[1] = k_out;
   int sms = 0;
   if (int s = sm_count(&sms)) return s;
   rotary_launch<false>(p, dtype, rotary_width(p, dtype, false), sms, static_cast<cudaStream_t>(stream));
   return finish_call(stream);
}

int64_t fusedmm_b200_qk_norm_rotary_backward_workspace(int64_t rows, int32_t d)
{
   int sms = 0;
   if (rows < 0 || d < 1 || d > FUSEDMM_B200_ATTN_MAX_WIDTH) return FUSEDMM_B200_ERR_ARG;
   if (int s = sm_count(&sms)) return s;
   // as many blocks as the backward launch may have: its cap, or one for each part of the heads (choose_splits: as many parts as
   // wanted warps at most)
   const int64_t blocks = static_cast<int64_t>(sms) * (ROT_WARPS > ROT_BACKWARD_BLOCKS_PER_SM ? ROT_WARPS : ROT_BACKWARD_BLOCKS_PER_SM);
   return blocks * 2 * d * static_cast<int64_t>(sizeof(float));
}

int fusedmm_b200_qk_norm_rotary_backward(int32_t dtype, int64_t rows, int32_t hq, int32_t hk, int32_t d, const void *q,
                                         int64_t ldq, int64_t hsq, const void *k, int64_t ldk, int64_t hsk, int32_t w_dtype,
                                         const void *wq, const void *wk, int32_t norm, double eps, int32_t pos_type,
                                         const void *pos, int64_t ldp, int64_t asp, int32_t axes, const double *freq,
                                         int32_t pairs, int32_t interleaved, const void *dq_out, int64_t lddq, int64_t hsdq,
                                         const void *dk_out, int64_t lddk, int64_t hsdk, void *dq, void *dk, float *dwq,
                                         float *dwk, void *workspace, int64_t workspace_bytes, void *stream)
{
   RotaryParams p = {};
   if (int s = rotary_setup(p, dtype, rows, hq, hk, d, q, ldq, hsq, k, ldk, hsk, w_dtype, wq, wk, norm, eps, pos_type, pos,
                            ldp, asp, axes, freq, pairs, interleaved)) return s;
   if (!norm && (dwq || dwk)) return FUSEDMM_B200_ERR_ARG;
   for (int64_t s : {lddq, hsdq, lddk, hsdk})
      if (s < 0) return FUSEDMM_B200_ERR_LIMIT;
   cudaStream_t st = static_cast<cudaStream_t>(stream);
   if (rows == 0 || hq + hk == 0) {  // sums over nothing
      if (!on_device({dwq, dwk})) return FUSEDMM_B200_ERR_ARG;
      if (dwq && cudaMemsetAsync(dwq, 0, d * sizeof(float), st) != cudaSuccess) return cuda_status();
      if (dwk && cudaMemsetAsync(dwk, 0, d * sizeof(float), st) != cudaSuccess) return cuda_status();
      return finish_call(stream);
   }
   if ((hq > 0 && (!dq_out || !dq)) || (hk > 0 && (!dk_out || !dk))) return FUSEDMM_B200_ERR_ARG;
   if (!on_device({hq > 0 ? dq_out : nullptr, hk > 0 ? dk_out : nullptr, hq > 0 ? dq : nullptr, hk > 0 ? dk : nullptr, dwq, dwk}))
      return FUSEDMM_B200_ERR_ARG;
   if (dwq || dwk) {
      const int64_t need = fusedmm_b200_qk_norm_rotary_backward_workspace(rows, d);
      if (need < 0) return static_cast<int>(need);
      if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 4 || !on_device({workspace}))
         return FUSEDMM_B200_ERR_ARG;
      p.dw_partial = static_cast<float *>(workspace);
   }
   p.y[0] = dq; p.y[1] = dk;
   p.dy[0] = dq_out; p.dy[1] = dk_out;
   p.ldd[0] = lddq; p.ldd[1] = lddk; p.hsd[0] = hsdq; p.hsd[1] = hsdk;
   int sms = 0;
   if (int s = sm_count(&sms)) return s;
   const int blocks = rotary_launch<true>(p, dtype, rotary_width(p, dtype, true), sms, st);
   if (p.dw_partial)
      rotary_dw_kernel<<<(2 * d + 31) / 32, 1024, 0, st>>>(p.dw_partial, blocks, d, dwq, dwk);
   return finish_call(stream);
}

}  // extern "C"

// attn_rotary.cu -- the norm of queries and keys for each head with the rotation by their positions, forward and backward
// (include/fusedmm_b200.h, fusedmm_b200_qk_norm_rotary).
//
//   y = x * rsqrt(mean(x^2) + eps) * w;  theta_i = sum_a pos[a] * freq[a][i];
//   (y_lo, y_hi) -> (y_lo cos - y_hi sin, y_hi cos + y_lo sin) for the pairs i < P; what lies behind the pairs passes.
//   backward, g = dy turned back:  dw = sum_rows,heads g x r;  dx = r (w g - x r mean(w g x r)), r the root's reciprocal.
//
// Bound: bytes; every element is read and written once, the arithmetic is ~10 instructions an element.  A head is cut into
// units of two vectors that hold the two halves of the same pairs, one unit to a lane, so the rotation needs no exchange
// between lanes and the norm one butterfly over the lanes of the head.  The angles of a row are shared by all heads:
// a block takes a few rows, computes their sines once (in 64 bits up to the turn's fraction: 2^20 positions times a
// frequency leave no digit of the angle in 32) and keeps them in shared memory.
#include "../../include/fusedmm_b200.h"
#include "attn_common.cuh"
#include "attn_host.h"

namespace fmm {
namespace attn {

constexpr int ROT_THREADS = 256;
constexpr int ROT_TABLE = 2048;  // sine/cosine pairs a block keeps
constexpr int ROT_SCALAR_UNITS = 4;  // units of a lane in the element-wise form: 32 lanes x 4 units x 2 elements = 256

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
   int d, pairs, axes, pos_type, w_f32, interleaved, norm, tile, lanes_log2, units;
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

// sines and cosines of the tile's rows into shared memory
__device__ __forceinline__ void fill_table(const RotaryParams &p, long long row0, int nrows, float2 *table)
{
   for (int t = threadIdx.x; t < nrows * p.pairs; t += ROT_THREADS) {
      const int r = t / p.pairs, i = t - r * p.pairs;
      double angle = 0.0;
      for (int a = 0; a < p.axes; a++) angle = fma(position(p, row0 + r, a), __ldg(p.freq + a * p.pairs + i), angle);
      const double half_turns = angle * 0.31830988618379067154;  // 1/pi
      // only the fraction of a turn matters; it fits 32 bits once the whole turns are gone
      const float rest = static_cast<float>(half_turns - 2.0 * rint(half_turns * 0.5));
      float s, c;
      sincospif(rest, &s, &c);
      table[t] = make_float2(c, s);
   }
}

// One unit: 2W elements in two vectors.  Unit u < pairs/W of the halves form holds elements [uW, uW+W) and
// [P+uW, P+uW+W); of the interleaved form [2uW, 2uW+2W); behind the pairs units are consecutive vectors.
template <int W>
struct Unit {
   int at[2];    // element index of the two vectors, -1: none
   int pair;     // first pair, -1: nothing to turn
   __device__ __forceinline__ void place(const RotaryParams &p, int u)
   {
      const int up = p.pairs / W;
      pair = -1;
      at[0] = at[1] = -1;
      if (u < up) {
         pair = u * W;
         at[0] = p.interleaved ? 2 * u * W : u * W;
         at[1] = p.interleaved ? at[0] + W : p.pairs + u * W;
      } else if (u < p.units) {
         at[0] = 2 * p.pairs + 2 * (u - up) * W;
         at[1] = at[0] + W < p.d ? at[0] + W : -1;
      }
   }
};

template <int W>
__device__ __forceinline__ void turn(float (&lo)[W], float (&hi)[W], const float2 *cs, bool interleaved, float sign)
{
   if (interleaved && W > 1) {
      // the two vectors are consecutive: pair j is elements 2j, 2j+1 of their 2W
#pragma unroll
      for (int j = 0; j < W; j++) {
         const float2 t = cs[j];
         float &a = 2 * j < W ? lo[(2 * j) % W] : hi[(2 * j) % W];
         float &b = 2 * j < W ? lo[(2 * j + 1) % W] : hi[(2 * j + 1) % W];
         const float s = sign * t.y, a0 = a;
         a = fmaf(a0, t.x, -b * s);
         b = fmaf(b, t.x, a0 * s);
      }
   } else {
#pragma unroll
      for (int j = 0; j < W; j++) {
         const float2 t = cs[j];
         const float s = sign * t.y, a0 = lo[j];
         lo[j] = fmaf(a0, t.x, -hi[j] * s);
         hi[j] = fmaf(hi[j], t.x, a0 * s);
      }
   }
}

template <typename T, int W>
__device__ __forceinline__ void load_part(const T *base, int at, float (&f)[W])
{
   if constexpr (W == 1) {
      f[0] = at >= 0 ? Elt<T>::up(base[at]) : 0.0f;
   } else {
      const uint4 r = at >= 0 ? ldg16(base + at) : make_uint4(0u, 0u, 0u, 0u);
      Elt<T>::unpack(r, f);
   }
}
template <typename T, int W>
__device__ __forceinline__ void store_part(T *base, int at, const float (&f)[W])
{
   if (at < 0) return;
   if constexpr (W == 1) base[at] = Elt<T>::down(f[0]);
   else *reinterpret_cast<uint4 *>(base + at) = Elt<T>::pack(f);
}
template <typename T, int W>
__device__ __forceinline__ void load_weight(const RotaryParams &p, int which, int at, float (&f)[W])
{
#pragma unroll
   for (int j = 0; j < W; j++) {
      f[j] = 1.0f;
      if (at >= 0 && p.w[which])
         f[j] = p.w_f32 ? __ldg(static_cast<const float *>(p.w[which]) + at + j) : Elt<T>::up(static_cast<const T *>(p.w[which])[at + j]);
   }
}

__device__ __forceinline__ float sum_over(float v, int lanes_log2)
{
   for (int s = 0; s < lanes_log2; s++) v += __shfl_xor_sync(FULL, v, 1 << s);
   return v;
}

// NU: units of a lane (1 with vectors).  A slot of 2^lanes_log2 lanes takes one head of one row at a time.
template <typename T, int W, int NU, bool BACKWARD>
__global__ void __launch_bounds__(ROT_THREADS) rotary_kernel(const RotaryParams p)
{
   __shared__ float2 table[ROT_TABLE];
   __shared__ float sums[BACKWARD ? ROT_THREADS * NU * 2 * W : 1];
   const int lanes = 1 << p.lanes_log2;
   const int lane = threadIdx.x & (lanes - 1), slot = threadIdx.x >> p.lanes_log2, slots = ROT_THREADS >> p.lanes_log2;
   Unit<W> unit[NU];
#pragma unroll
   for (int i = 0; i < NU; i++) unit[i].place(p, lane + i * 32);
   float dw[2][NU][2][W] = {};
   const float inv_d = 1.0f / p.d;
   const long long tiles = (p.rows + p.tile - 1) / p.tile;
   for (long long tl = blockIdx.x; tl < tiles; tl += gridDim.x) {
      const long long row0 = tl * p.tile;
      const int nrows = static_cast<int>(min(static_cast<long long>(p.tile), p.rows - row0));
      __syncthreads();  // the table's last readers
      if (p.pairs > 0) fill_table(p, row0, nrows, table);
      __syncthreads();
#pragma unroll
      for (int which = 0; which < 2; which++) {
         const int heads = p.heads[which], tasks = nrows * heads;
         if (tasks == 0) continue;
         float w[NU][2][W];
#pragma unroll
         for (int i = 0; i < NU; i++) {
            load_weight<T, W>(p, which, unit[i].at[0], w[i][0]);
            load_weight<T, W>(p, which, unit[i].at[1], w[i][1]);
         }
         // every lane of a warp runs every round: the butterflies need them all
         const int rounds = (tasks + slots - 1) / slots;
         for (int n = 0; n < rounds; n++) {
            const int task = n * slots + slot;
            const bool live = task < tasks;
            const int r = live ? task / heads : 0, h = live ? task - r * heads : 0;
            const long long row = row0 + r;
            const T *x = static_cast<const T *>(p.x[which]) + row * p.ldx[which] + h * p.hsx[which];
            T *y = static_cast<T *>(p.y[which]) + (row * heads + h) * p.d;
            float v[NU][2][W];
#pragma unroll
            for (int i = 0; i < NU; i++) {
               load_part<T, W>(x, live ? unit[i].at[0] : -1, v[i][0]);
               load_part<T, W>(x, live ? unit[i].at[1] : -1, v[i][1]);
            }
            float rr = 1.0f;
            if (p.norm) {
               float ss = 0.0f;
#pragma unroll
               for (int i = 0; i < NU; i++)
#pragma unroll
                  for (int j = 0; j < W; j++) ss = fmaf(v[i][0][j], v[i][0][j], fmaf(v[i][1][j], v[i][1][j], ss));
               ss = sum_over(ss, p.lanes_log2);
               rr = rsqrtf(fmaf(ss, inv_d, p.eps));
            }
            if constexpr (!BACKWARD) {
#pragma unroll
               for (int i = 0; i < NU; i++) {
                  if (p.norm) {
#pragma unroll
                     for (int j = 0; j < W; j++) {
                        v[i][0][j] = v[i][0][j] * rr * w[i][0][j];
                        v[i][1][j] = v[i][1][j] * rr * w[i][1][j];
                     }
                  }
                  if (unit[i].pair >= 0) turn<W>(v[i][0], v[i][1], table + r * p.pairs + unit[i].pair, p.interleaved, 1.0f);
                  if (live) {
                     store_part<T, W>(y, unit[i].at[0], v[i][0]);
                     store_part<T, W>(y, unit[i].at[1], v[i][1]);
                  }
               }
            } else {
               const T *dy = static_cast<const T *>(p.dy[which]) + row * p.ldd[which] + h * p.hsd[which];
               float g[NU][2][W], dot = 0.0f;
#pragma unroll
               for (int i = 0; i < NU; i++) {
                  load_part<T, W>(dy, live ? unit[i].at[0] : -1, g[i][0]);
                  load_part<T, W>(dy, live ? unit[i].at[1] : -1, g[i][1]);
                  if (unit[i].pair >= 0) turn<W>(g[i][0], g[i][1], table + r * p.pairs + unit[i].pair, p.interleaved, -1.0f);
                  if (p.norm) {
#pragma unroll
                     for (int s = 0; s < 2; s++)
#pragma unroll
                        for (int j = 0; j < W; j++) {
                           v[i][s][j] *= rr;
                           // a slot without a task has zeros here, times a weight that may be infinite: adds nothing
                           if (live) dw[which][i][s][j] = fmaf(g[i][s][j], v[i][s][j], dw[which][i][s][j]);
                           g[i][s][j] *= w[i][s][j];
                           dot = fmaf(g[i][s][j], v[i][s][j], dot);
                        }
                  }
               }
               if (p.norm) {
                  dot = sum_over(dot, p.lanes_log2) * inv_d;
#pragma unroll
                  for (int i = 0; i < NU; i++)
#pragma unroll
                     for (int s = 0; s < 2; s++)
#pragma unroll
                        for (int j = 0; j < W; j++) g[i][s][j] = rr * fmaf(-v[i][s][j], dot, g[i][s][j]);
               }
               if (live) {
#pragma unroll
                  for (int i = 0; i < NU; i++) {
                     store_part<T, W>(y, unit[i].at[0], g[i][0]);
                     store_part<T, W>(y, unit[i].at[1], g[i][1]);
                  }
               }
            }
         }
      }
   }
   if constexpr (BACKWARD) {
      if (!p.dw_partial) return;
      // the block's share of the weight gradients: every slot's sums side by side, added in the order of the slots
#pragma unroll
      for (int which = 0; which < 2; which++) {
         __syncthreads();
#pragma unroll
         for (int i = 0; i < NU; i++)
#pragma unroll
            for (int s = 0; s < 2; s++)
               if (unit[i].at[s] >= 0)
#pragma unroll
                  for (int j = 0; j < W; j++) sums[slot * p.d + unit[i].at[s] + j] = dw[which][i][s][j];
         __syncthreads();
         for (int e = threadIdx.x; e < p.d; e += ROT_THREADS) {
            float t = 0.0f;
            for (int s = 0; s < slots; s++) t += sums[s * p.d + e];
            p.dw_partial[(static_cast<long long>(blockIdx.x) * 2 + which) * p.d + e] = t;
         }
      }
   }
}

// dw[which][e] = sum over the blocks; 32 columns to a block, its 8 warps take the partial rows in turn
__global__ void __launch_bounds__(256) rotary_dw_kernel(const float *partial, int blocks, int d, float *dwq, float *dwk)
{
   __shared__ float part[8][33];
   const int col = blockIdx.x * 32 + (threadIdx.x & 31), w = threadIdx.x >> 5;
   float t = 0.0f;
   if (col < 2 * d)
      for (int b = w; b < blocks; b += 8) t += partial[static_cast<long long>(b) * 2 * d + col];
   part[w][threadIdx.x & 31] = t;
   __syncthreads();
   if (w == 0 && col < 2 * d) {
      float s = 0.0f;
      for (int i = 0; i < 8; i++) s += part[i][threadIdx.x];
      float *out = col < d ? dwq : dwk;
      if (out) out[col < d ? col : col - d] = s;
   }
}

namespace {

int ceil_log2(int n)
{
   int l = 0;
   while ((1 << l) < n) l++;
   return l;
}

// rows of a block: enough heads for four rounds of its slots, so that the sines are shared and loads of several rounds
// overlap, but no more than the sine table holds, and fewer when there are too few rows to give every SM work
void choose_tile(RotaryParams &p, int sm_count)
{
   const int slots = ROT_THREADS >> p.lanes_log2, heads = p.heads[0] + p.heads[1];
   long long tile = (4LL * slots + heads - 1) / heads;
   if (p.pairs > 0) tile = tile < ROT_TABLE / p.pairs ? tile : ROT_TABLE / p.pairs;
   const long long spread = p.rows / (4LL * sm_count);
   if (tile > spread) tile = spread;
   if (tile > 64) tile = 64;
   p.tile = static_cast<int>(tile < 1 ? 1 : tile);
}

constexpr int ROT_BACKWARD_BLOCKS_PER_SM = 4;

template <typename T, bool BACKWARD>
int launch(RotaryParams &p, bool vectors, int sm_count, cudaStream_t st)
{
   constexpr int W = Elt<T>::W;
   const int width = vectors ? W : 1;
   const int behind = (p.d - 2 * p.pairs) / width;
   p.units = p.pairs / width + (behind + 1) / 2;
   p.lanes_log2 = vectors ? ceil_log2(p.units) : 5;
   choose_tile(p, sm_count);
   const long long tiles = (p.rows + p.tile - 1) / p.tile;
   const long long cap = BACKWARD ? static_cast<long long>(sm_count) * ROT_BACKWARD_BLOCKS_PER_SM : 0x7fffffffLL;
   const unsigned grid = static_cast<unsigned>(tiles < cap ? tiles : cap);
   if (vectors) rotary_kernel<T, W, 1, BACKWARD><<<grid, ROT_THREADS, 0, st>>>(p);
   else rotary_kernel<T, 1, ROT_SCALAR_UNITS, BACKWARD><<<grid, ROT_THREADS, 0, st>>>(p);
   return static_cast<int>(grid);
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

bool rotary_vectors(const RotaryParams &p, int32_t dtype, bool backward)
{
   const int width = dtype == DT_F32 ? 4 : 8;
   const size_t elt = dtype == DT_F32 ? 4 : 2;
   if (p.d % width || p.pairs % width) return false;
   for (int i = 0; i < 2; i++) {
      if (!p.heads[i]) continue;
      if (!multiple(p.x[i], p.ldx[i], p.hsx[i], width, elt) || !multiple(p.y[i], 0, 0, width, elt)) return false;
      if (backward && !multiple(p.dy[i], p.ldd[i], p.hsd[i], width, elt)) return false;
   }
   return true;
}

template <bool BACKWARD>
int rotary_launch(RotaryParams &p, int32_t dtype, bool vectors, int sm_count, cudaStream_t st)
{
   if (dtype == DT_F32) return launch<float, BACKWARD>(p, vectors, sm_count, st);
   if (dtype == DT_BF16) return launch<__nv_bfloat16, BACKWARD>(p, vectors, sm_count, st);
   return launch<__half, BACKWARD>(p, vectors, sm_count, st);
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
   rotary_launch<false>(p, dtype, rotary_vectors(p, dtype, false), sms, static_cast<cudaStream_t>(stream));
   return finish_call(stream);
}

int64_t fusedmm_b200_qk_norm_rotary_backward_workspace(int64_t rows, int32_t d)
{
   int sms = 0;
   if (rows < 0 || d < 1 || d > FUSEDMM_B200_ATTN_MAX_WIDTH) return FUSEDMM_B200_ERR_ARG;
   if (int s = sm_count(&sms)) return s;
   const int64_t blocks = static_cast<int64_t>(sms) * ROT_BACKWARD_BLOCKS_PER_SM;
   return (rows < blocks ? rows : blocks) * 2 * d * static_cast<int64_t>(sizeof(float));
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
   const int blocks = rotary_launch<true>(p, dtype, rotary_vectors(p, dtype, true), sms, st);
   if (p.dw_partial)
      rotary_dw_kernel<<<(2 * d + 31) / 32, 256, 0, st>>>(p.dw_partial, blocks, d, dwq, dwk);
   return finish_call(stream);
}

}  // extern "C"

// attn_common.cuh -- what the attention operators share: 16-byte vectors of the three storage types, their conversion to
// the 32-bit numbers everything is computed in, and loads of rows whose address or length is no multiple of a vector.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace fmm {
namespace attn {

constexpr unsigned FULL = 0xffffffffu;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;

// dtype codes of the C ABI (0 and 1, float and double, are those of fusedmm_b200_csr; double has no kernel here)
enum : int { DT_F32 = 0, DT_BF16 = 2, DT_F16 = 3 };

template <typename T>
struct Elt;  // W: elements of a 16-byte vector
template <>
struct Elt<float> {
   static constexpr int W = 4;
   static __device__ __forceinline__ float up(float x) { return x; }
   static __device__ __forceinline__ float down(float x) { return x; }
   static __device__ __forceinline__ void unpack(const uint4 &r, float (&f)[4])
   {
      f[0] = __uint_as_float(r.x); f[1] = __uint_as_float(r.y); f[2] = __uint_as_float(r.z); f[3] = __uint_as_float(r.w);
   }
   static __device__ __forceinline__ uint4 pack(const float (&f)[4])
   {
      return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
   }
};
template <>
struct Elt<__nv_bfloat16> {
   static constexpr int W = 8;
   static __device__ __forceinline__ float up(__nv_bfloat16 x) { return __bfloat162float(x); }
   static __device__ __forceinline__ __nv_bfloat16 down(float x) { return __float2bfloat16_rn(x); }
   // a bf16 is the upper half of the float of the same value
   static __device__ __forceinline__ void unpack2(unsigned r, float &a, float &b)
   {
      a = __uint_as_float(r << 16);
      b = __uint_as_float(r & 0xffff0000u);
   }
   static __device__ __forceinline__ unsigned pack2(float a, float b)
   {
      __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
      return *reinterpret_cast<unsigned *>(&h);
   }
   static __device__ __forceinline__ void unpack(const uint4 &r, float (&f)[8])
   {
      unpack2(r.x, f[0], f[1]); unpack2(r.y, f[2], f[3]); unpack2(r.z, f[4], f[5]); unpack2(r.w, f[6], f[7]);
   }
   static __device__ __forceinline__ uint4 pack(const float (&f)[8])
   {
      return make_uint4(pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7]));
   }
};
template <>
struct Elt<__half> {
   static constexpr int W = 8;
   static __device__ __forceinline__ float up(__half x) { return __half2float(x); }
   static __device__ __forceinline__ __half down(float x) { return __float2half_rn(x); }
   static __device__ __forceinline__ void unpack2(unsigned r, float &a, float &b)
   {
      const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&r));
      a = f.x;
      b = f.y;
   }
   static __device__ __forceinline__ unsigned pack2(float a, float b)
   {
      __half2 h = __floats2half2_rn(a, b);
      return *reinterpret_cast<unsigned *>(&h);
   }
   static __device__ __forceinline__ void unpack(const uint4 &r, float (&f)[8])
   {
      unpack2(r.x, f[0], f[1]); unpack2(r.y, f[2], f[3]); unpack2(r.z, f[4], f[5]); unpack2(r.w, f[6], f[7]);
   }
   static __device__ __forceinline__ uint4 pack(const float (&f)[8])
   {
      return make_uint4(pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7]));
   }
};

// Two floats in one register pair: one instruction issues both of their multiply-adds (the walks below are bound by issue
// slots, not by the multipliers: 16 pairs a clock and quarter of an SM either way).
typedef unsigned long long F2;
__device__ __forceinline__ F2 f2(float a, float b)
{
   F2 r;
   asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
   return r;
}
__device__ __forceinline__ float2 f2_parts(F2 x)
{
   float2 r;
   asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
   return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c)
{
   F2 r;
   asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
   return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b)
{
   F2 r;
   asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
   return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b)
{
   F2 r;
   asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
   return r;
}
__device__ __forceinline__ float sum2(F2 x)
{
   const float2 p = f2_parts(x);
   return p.x + p.y;
}
template <typename T>
__device__ __forceinline__ void unpack_pairs(const uint4 &r, F2 (&f)[Elt<T>::W / 2])
{
   float t[Elt<T>::W];
   Elt<T>::unpack(r, t);
#pragma unroll
   for (int i = 0; i < Elt<T>::W / 2; i++) f[i] = f2(t[2 * i], t[2 * i + 1]);
}

// 2^x; results below the smallest normal number are 0
__device__ __forceinline__ float exp2_fast(float x)
{
   float r;
   asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
   return r;
}

// the smaller of the two, NaN if one of them is
__device__ __forceinline__ float min_or_nan(float a, float b)
{
   float r;
   asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
   return r;
}

__device__ __forceinline__ uint4 ldg16(const void *p) { return __ldg(static_cast<const uint4 *>(p)); }

// `left` elements (any number, also <= 0) of the vector at p; what lies behind them reads as zero.  `step`: the elements
// that one load may take at once (a power of two that divides the address, the strides and the length), 1 .. W.
template <typename T>
__device__ __forceinline__ uint4 ld_pieces(const T *p, int left, int step)
{
   uint4 r = make_uint4(0u, 0u, 0u, 0u);
   if constexpr (sizeof(T) == 4) {
      if (step >= 2) {
         if (left >= 2) { const uint2 a = __ldg(reinterpret_cast<const uint2 *>(p)); r.x = a.x; r.y = a.y; }
         if (left >= 4) { const uint2 a = __ldg(reinterpret_cast<const uint2 *>(p) + 1); r.z = a.x; r.w = a.y; }
      } else {
         const unsigned *u = reinterpret_cast<const unsigned *>(p);
         if (left > 0) r.x = __ldg(u);
         if (left > 1) r.y = __ldg(u + 1);
         if (left > 2) r.z = __ldg(u + 2);
         if (left > 3) r.w = __ldg(u + 3);
      }
   } else {
      if (step >= 4) {
         if (left >= 4) { const uint2 a = __ldg(reinterpret_cast<const uint2 *>(p)); r.x = a.x; r.y = a.y; }
         if (left >= 8) { const uint2 a = __ldg(reinterpret_cast<const uint2 *>(p) + 1); r.z = a.x; r.w = a.y; }
      } else if (step >= 2) {
         const unsigned *u = reinterpret_cast<const unsigned *>(p);
         if (left >= 2) r.x = __ldg(u);
         if (left >= 4) r.y = __ldg(u + 1);
         if (left >= 6) r.z = __ldg(u + 2);
         if (left >= 8) r.w = __ldg(u + 3);
      } else {
         const unsigned short *u = reinterpret_cast<const unsigned short *>(p);
         unsigned e[8];
#pragma unroll
         for (int i = 0; i < 8; i++) e[i] = i < left ? __ldg(u + i) : 0u;
         r = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
      }
   }
   return r;
}

// VECTOR: the host has checked that addresses, strides and the length are multiples of 16 bytes.
template <typename T, bool VECTOR>
__device__ __forceinline__ uint4 ld_row(const T *p, int left, int step)
{
   if constexpr (VECTOR) return left > 0 ? ldg16(p) : make_uint4(0u, 0u, 0u, 0u);
   else return ld_pieces(p, left, step);
}

template <typename T, bool VECTOR>
__device__ __forceinline__ void st_row(T *p, const float (&f)[Elt<T>::W], int left)
{
   if constexpr (VECTOR) {
      if (left > 0) *reinterpret_cast<uint4 *>(p) = Elt<T>::pack(f);
   } else {
#pragma unroll
      for (int i = 0; i < Elt<T>::W; i++)
         if (i < left) p[i] = Elt<T>::down(f[i]);
   }
}

}  // namespace attn
}  // namespace fmm

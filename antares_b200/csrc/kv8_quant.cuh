// Rows of keys and values on their way into the 8-bit cache: loads, rotation, codes.  Half a warp has a row.
#pragma once
#include <math_constants.h>

#include "kv8.cuh"

namespace ab200 {

constexpr float KA_LEAST_SCALE = 0x1p-100f;  // below it a block is held as zeros: quotients stay clear of subnormal arithmetic
constexpr float KA_MAGIC = 12582912.f;       // 1.5 * 2^23: a number of less than 2^22 added to it is rounded to an integer, in the low bits

// The code of x at scale s: the quotient x / s rounded to the nearest, ties to even, as if it had all its digits.  `inv` is
// about 1 / s, so k is off by one at most; the two sums (each one rounding, so their signs are exact) say which side of the
// middle between two codes x lies on.
static __device__ __noinline__ int kv8_code(float x, float s, float inv) {
  if (s == 0.f) return 0;
  if (!(fabsf(x) < CUDART_INF_F)) return x > 0.f ? 127 : x < 0.f ? -127 : 0;
  float k = rintf(x * inv);
  const float up = fmaf(-(k + 0.5f), s, x), down = fmaf(-(k - 0.5f), s, x);
  const bool odd = ((int)k & 1) != 0;
  if (up > 0.f || (up == 0.f && odd)) k += 1.f;
  else if (down < 0.f || (down == 0.f && odd)) k -= 1.f;
  return (int)fminf(fmaxf(k, -127.f), 127.f);
}
// Eight of them, as two words.  Where the quotients by a scale 2^-20 smaller and larger round alike, so does the exact one;
// elsewhere, about once in 10000 values, the slow way decides.  (It was most of the kernel's instructions for every value.)
__device__ __forceinline__ uint64_t ka_pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void ka_round(const uint64_t (&x)[4], float inv, uint32_t (&w)[2]) {
  const uint64_t f = ka_pair(inv, inv), magic = ka_pair(KA_MAGIC, KA_MAGIC);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t t[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint64_t r;
      asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x[2 * h + i]), "l"(f), "l"(magic));
      asm("mov.b64 {%0, %1}, %2;" : "=r"(t[2 * i]), "=r"(t[2 * i + 1]) : "l"(r));
    }
    w[h] = __byte_perm(__byte_perm(t[0], t[1], 0x0040), __byte_perm(t[2], t[3], 0x0040), 0x5410);
  }
}
__device__ __forceinline__ uint2 kv8_codes(const float (&x)[8], float s, float inv_less, float inv_more, bool slow) {
  const uint64_t v[4] = {ka_pair(x[0], x[1]), ka_pair(x[2], x[3]), ka_pair(x[4], x[5]), ka_pair(x[6], x[7])};
  uint32_t w[2], u[2];
  ka_round(v, inv_less, w);
  ka_round(v, inv_more, u);
  if (slow || w[0] != u[0] || w[1] != u[1]) {
    const float inv = s > 0.f ? __fdividef(1.f, s) : 0.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      w[h] = 0;
#pragma unroll 1
      for (int i = 0; i < 4; ++i) {
        const float y = i == 0 ? x[4 * h] : i == 1 ? x[4 * h + 1] : i == 2 ? x[4 * h + 2] : x[4 * h + 3];
        w[h] |= (uint32_t)(kv8_code(y, s, inv) & 255) << (8 * i);
      }
    }
  }
  return make_uint2(w[0], w[1]);
}

// dims 4 sub .. 4 sub + 3 and 64 + the same of a row: a rotated pair is one thread's
__device__ __forceinline__ void ka_load(const __half *p, int sub, float (&f)[8]) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const uint2 v = *reinterpret_cast<const uint2 *>(p + 64 * half + 4 * sub);
    const float2 a = __half22float2(u2h2(v.x)), b = __half22float2(u2h2(v.y));
    f[4 * half] = a.x, f[4 * half + 1] = a.y, f[4 * half + 2] = b.x, f[4 * half + 3] = b.y;
  }
}
__device__ __forceinline__ void ka_load(const float *p, int sub, float (&f)[8]) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const float4 v = *reinterpret_cast<const float4 *>(p + 64 * half + 4 * sub);
    f[4 * half] = v.x, f[4 * half + 1] = v.y, f[4 * half + 2] = v.z, f[4 * half + 3] = v.w;
  }
}
__device__ __forceinline__ void ka_store(__half *p, int sub, const float (&f)[8]) {
#pragma unroll
  for (int half = 0; half < 2; ++half)
    *reinterpret_cast<uint2 *>(p + 64 * half + 4 * sub) =
        make_uint2(h22u(__floats2half2_rn(f[4 * half], f[4 * half + 1])), h22u(__floats2half2_rn(f[4 * half + 2], f[4 * half + 3])));
}
__device__ __forceinline__ void ka_store(float *p, int sub, const float (&f)[8]) {
#pragma unroll
  for (int half = 0; half < 2; ++half) *reinterpret_cast<float4 *>(p + 64 * half + 4 * sub) = make_float4(f[4 * half], f[4 * half + 1], f[4 * half + 2], f[4 * half + 3]);
}

// Sines: fp16 rows turn with 32-bit ones.  fp32 rows with 64-bit ones: which of two codes a value next to their middle gets
// would otherwise go by the last bits of the rotation.
template <typename T> struct KaAngle { typedef float type; };
template <> struct KaAngle<float> { typedef double type; };
__device__ __forceinline__ void ka_sincos(float a, float *s, float *c) { sincosf(a, s, c); }
__device__ __forceinline__ void ka_sincos(float a, double *s, double *c) { sincos((double)a, s, c); }

__device__ __forceinline__ void ka_four(const float *p, float (&v)[4]) {
  const float4 a = *reinterpret_cast<const float4 *>(p);
  v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w;
}
__device__ __forceinline__ void ka_four(const double *p, double (&v)[4]) {
  const double2 a = reinterpret_cast<const double2 *>(p)[0], b = reinterpret_cast<const double2 *>(p)[1];
  v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
}
// One way to round a rotation, wherever it is done: a row's codes do not depend on the call that writes it.
__device__ __forceinline__ void ka_rotate(float &x, float &y, float s, float c) {
  const float a = fmaf(x, c, -__fmul_rn(y, s));
  y = fmaf(y, c, __fmul_rn(x, s));
  x = a;
}
__device__ __forceinline__ void ka_rotate(float &x, float &y, double s, double c) {
  const double a = fma((double)x, c, -__dmul_rn((double)y, s));
  y = (float)fma((double)y, c, __dmul_rn((double)x, s));
  x = (float)a;
}
template <typename A>
__device__ __forceinline__ void ka_turn(float (&f)[8], const A *sn, const A *cs, int sub) {
  A s4[4], c4[4];
  ka_four(sn + 4 * sub, s4), ka_four(cs + 4 * sub, c4);
#pragma unroll
  for (int i = 0; i < 4; ++i) ka_rotate(f[i], f[4 + i], s4[i], c4[i]);
}

}  // namespace ab200

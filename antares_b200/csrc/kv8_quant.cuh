// Rows of keys and values on their way into the 8-bit cache: loads, rotation, codes.  Half a warp has a row.
#pragma once
#include <math_constants.h>

#include <type_traits>

#include "kv8.cuh"

namespace ab200 {

constexpr float KA_LEAST_SCALE = 0x1p-100f;  // below it a block is held as zeros: quotients stay clear of subnormal arithmetic
constexpr float KA_MAGIC = 12582912.f;       // 1.5 * 2^23: a number of less than 2^22 added to it is rounded to an integer, in the low bits

// The codes of eight values at scale s: the quotients x / s rounded to the nearest, ties to even, as if they had all their
// digits.  k = x * inv rounded is off by one at most, and e = x - k s is exact: k is a small integer, x and s are fp32, and
// what is left has the digits of the coarser of the two and is no larger than s.  So k is right where |e| is below half of s;
// next to it, which is seldom, |e| and the last bit of k decide.  Two values an instruction.
__device__ __forceinline__ uint64_t ka_pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ uint2 kv8_codes(const float (&x)[8], float s, float inv, bool odd_values) {
  const uint64_t f = ka_pair(inv, inv), magic = ka_pair(KA_MAGIC, KA_MAGIC), less = ka_pair(-KA_MAGIC, -KA_MAGIC), minus = ka_pair(-s, -s);
  const float half = 0.5f * s, below = __uint_as_float(__float_as_uint(half) - 1u);
  uint32_t t[8];
  float e[8];
  bool near = odd_values;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t v = ka_pair(x[2 * i], x[2 * i + 1]);
    uint64_t k, left;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(k) : "l"(v), "l"(f), "l"(magic));
    asm("mov.b64 {%0, %1}, %2;" : "=r"(t[2 * i]), "=r"(t[2 * i + 1]) : "l"(k));
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(k) : "l"(k), "l"(less));
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(left) : "l"(k), "l"(minus), "l"(v));
    asm("mov.b64 {%0, %1}, %2;" : "=f"(e[2 * i]), "=f"(e[2 * i + 1]) : "l"(left));
    near = near || fabsf(e[2 * i]) > below || fabsf(e[2 * i + 1]) > below;
  }
  if (near) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (fabsf(e[i]) > (t[i] & 1u ? below : half)) t[i] += e[i] < 0.f ? -1 : 1;
      if (odd_values) t[i] = s == 0.f || x[i] != x[i] ? 0u : x[i] == CUDART_INF_F ? 127u : x[i] == -CUDART_INF_F ? -127u : t[i];
    }
  }
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) w[h] = __byte_perm(__byte_perm(t[4 * h], t[4 * h + 1], 0x0040), __byte_perm(t[4 * h + 2], t[4 * h + 3], 0x0040), 0x5410);
  return make_uint2(w[0], w[1]);
}

// A thread's part of a row, as it lies in memory: dims 4 sub .. 4 sub + 3 and 64 + the same, so a rotated pair is one thread's.
template <typename T> struct KaRaw;
template <> struct KaRaw<__half> { uint2 v[2]; };
template <> struct KaRaw<float> { float4 v[2]; };
template <typename T>
__device__ __forceinline__ void ka_ask(const T *p, int sub, KaRaw<T> &r) {
#pragma unroll
  for (int half = 0; half < 2; ++half) r.v[half] = *reinterpret_cast<const std::remove_reference_t<decltype(r.v[0])> *>(p + 64 * half + 4 * sub);
}
__device__ __forceinline__ void ka_widen(const KaRaw<__half> &r, float (&f)[8]) {
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const float2 a = __half22float2(u2h2(r.v[half].x)), b = __half22float2(u2h2(r.v[half].y));
    f[4 * half] = a.x, f[4 * half + 1] = a.y, f[4 * half + 2] = b.x, f[4 * half + 3] = b.y;
  }
}
__device__ __forceinline__ void ka_widen(const KaRaw<float> &r, float (&f)[8]) {
#pragma unroll
  for (int half = 0; half < 2; ++half) f[4 * half] = r.v[half].x, f[4 * half + 1] = r.v[half].y, f[4 * half + 2] = r.v[half].z, f[4 * half + 3] = r.v[half].w;
}
template <typename T>
__device__ __forceinline__ void ka_load(const T *p, int sub, float (&f)[8]) {
  KaRaw<T> r;
  ka_ask(p, sub, r);
  ka_widen(r, f);
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

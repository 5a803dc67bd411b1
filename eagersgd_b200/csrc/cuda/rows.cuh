// Rows of bf16 or fp32 values: vectors of 16 bytes (or single elements, where a row is not a whole number of vectors or does not
// begin on one) as fp32 registers, and the exponentials of the activations.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace esgd {

enum Activation { kActNone = 0, kActRelu = 1, kActSilu = 2 };

template <class T> __host__ __device__ constexpr int vector_of() { return 16 / (int)sizeof(T); }

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T as_type(float v);
template <> __device__ __forceinline__ float as_type<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 as_type<__nv_bfloat16>(float v) { return __float2bfloat16(v); }

// kV elements of T as they lie in memory: one load, converted where they are used.
template <class T, int kV> struct Pack { T v[kV]; };
template <> struct Pack<float, 4> { uint4 v; };
template <> struct Pack<__nv_bfloat16, 8> { uint4 v; };
template <> struct Pack<__nv_bfloat16, 4> { uint2 v; };

template <class T, int kV> __device__ __forceinline__ Pack<T, kV> load(const T* p) {
  static_assert(kV == 1 || kV * sizeof(T) == 16 || kV * sizeof(T) == 8, "single elements, 8 or 16 bytes");
  Pack<T, kV> r;
  if constexpr (kV == 1) r.v[0] = *p;
  else if constexpr (kV * sizeof(T) == 8) r.v = *reinterpret_cast<const uint2*>(p);
  else r.v = *reinterpret_cast<const uint4*>(p);
  return r;
}
template <class T, int kV> __device__ __forceinline__ void unpack(const Pack<T, kV>& r, float (&f)[kV]) {
  if constexpr (kV == 1) {
    f[0] = as_float(r.v[0]);
  } else if constexpr (kV == 4 && sizeof(T) == 2) {
    f[0] = __uint_as_float(r.v.x << 16); f[1] = __uint_as_float(r.v.x & 0xffff0000u);
    f[2] = __uint_as_float(r.v.y << 16); f[3] = __uint_as_float(r.v.y & 0xffff0000u);
  } else if constexpr (kV == 4) {
    f[0] = __uint_as_float(r.v.x); f[1] = __uint_as_float(r.v.y); f[2] = __uint_as_float(r.v.z); f[3] = __uint_as_float(r.v.w);
  } else {
    const uint32_t w[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
    for (int q = 0; q < 4; ++q) { f[2 * q] = __uint_as_float(w[q] << 16); f[2 * q + 1] = __uint_as_float(w[q] & 0xffff0000u); }
  }
}
template <class T, int kV> __device__ __forceinline__ void store(T* p, const float (&f)[kV]) {
  if constexpr (kV == 1) {
    *p = as_type<T>(f[0]);
  } else if constexpr (kV == 4 && sizeof(T) == 2) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
  } else if constexpr (kV == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
  } else {
    uint4 w;
    __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&w);
#pragma unroll
    for (int q = 0; q < 4; ++q) h[q] = __floats2bfloat162_rn(f[2 * q], f[2 * q + 1]);
    *reinterpret_cast<uint4*>(p) = w;
  }
}

constexpr float kLog2e = 1.44269504088896341f, kLog2eLow = 1.92596299e-8f, kLn2 = 0.69314718055994531f;

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// e^x with the rounding of x * log2(e) put right to first order: without it the relative error grows with |x| (20: 2e-6).
__device__ __forceinline__ float exp_fine(float x) {
  const float t = x * kLog2e, y = exp2_approx(t);
  const float low = fmaf(x, kLog2eLow, fmaf(x, kLog2e, -t));
  return fabsf(t) < 128.0f ? fmaf(y, low * kLn2, y) : y;      // beyond it y is 0 or infinite (or t is, and low no number)
}
// For the gates: where the exponential's error grows, far below zero, the result is next to nothing; above zero it is next to one.
__device__ __forceinline__ float sigmoid(float x) { return reciprocal(1.0f + exp2_approx(x * -kLog2e)); }

// An activation and its slope at x.
template <int kAct> __device__ __forceinline__ float activate(float x) {
  if constexpr (kAct == kActRelu) return x > 0.0f || x != x ? x : 0.0f;
  else if constexpr (kAct == kActSilu) return x * sigmoid(x);
  else return x;
}
template <int kAct> __device__ __forceinline__ float slope(float x) {
  if constexpr (kAct == kActRelu) {
    return x > 0.0f ? 1.0f : 0.0f;
  } else if constexpr (kAct == kActSilu) {
    const float s = sigmoid(x);
    return s * (1.0f + x * (1.0f - s));
  } else {
    return 1.0f;
  }
}

// Paired fp32 arithmetic: two values in a 64-bit register, one instruction for both.
using f2 = unsigned long long;
__device__ __forceinline__ f2 pair(float a, float b) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ f2 pair(float2 v) { return pair(v.x, v.y); }
__device__ __forceinline__ float2 halves(f2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// Both halves by one factor.
__device__ __forceinline__ f2 mul2(f2 a, float b) {
  const float2 v = halves(a);
  return pair(v.x * b, v.y * b);
}
__device__ __forceinline__ f2 fma2(f2 a, float b, f2 c) {
  const float2 v = halves(a), w = halves(c);
  return pair(fmaf(v.x, b, w.x), fmaf(v.y, b, w.y));
}
__device__ __forceinline__ f2 exp2_2(f2 x) {
  const float2 v = halves(x);
  return pair(exp2_approx(v.x), exp2_approx(v.y));
}
__device__ __forceinline__ f2 sigmoid2(f2 x) {
  const float2 v = halves(add2(exp2_2(mul2(x, pair(-kLog2e, -kLog2e))), pair(1.0f, 1.0f)));
  return pair(reciprocal(v.x), reciprocal(v.y));
}
template <int kAct> __device__ __forceinline__ f2 activate2(f2 x) {
  if constexpr (kAct == kActSilu) {
    return mul2(x, sigmoid2(x));
  } else if constexpr (kAct == kActRelu) {
    const float2 v = halves(x);
    return pair(activate<kActRelu>(v.x), activate<kActRelu>(v.y));
  } else {
    return x;
  }
}
template <int kAct> __device__ __forceinline__ f2 slope2(f2 x) {
  if constexpr (kAct == kActSilu) {
    const f2 s = sigmoid2(x), xs = mul2(x, s);
    return add2(fma2(mul2(xs, pair(-1.0f, -1.0f)), s, xs), s);      // s + x s (1 - s)
  } else {
    const float2 v = halves(x);
    return pair(slope<kAct>(v.x), slope<kAct>(v.y));
  }
}
// A vector as pairs (a single element: a pair with a zero).
template <int kV> struct PairsOf { static constexpr int n = (kV + 1) / 2; };
template <class T, int kV> __device__ __forceinline__ void unpack2(const Pack<T, kV>& r, f2 (&f)[PairsOf<kV>::n]) {
  float v[kV];
  unpack<T, kV>(r, v);
#pragma unroll
  for (int q = 0; q < PairsOf<kV>::n; ++q) f[q] = pair(v[2 * q], 2 * q + 1 < kV ? v[(2 * q + 1) % kV] : 0.0f);
}
template <class T, int kV> __device__ __forceinline__ void store2(T* p, const f2 (&f)[PairsOf<kV>::n]) {
  float v[kV];
#pragma unroll
  for (int q = 0; q < kV; ++q) v[q] = q % 2 == 0 ? halves(f[q / 2]).x : halves(f[q / 2]).y;
  store<T, kV>(p, v);
}

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace esgd

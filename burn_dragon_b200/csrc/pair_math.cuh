// fp32 arithmetic on pairs (two operations in one instruction) and rows of fp32 / fp16 / bf16 elements as pairs.
#pragma once
#include "element_io.cuh"

namespace bdh {

using f2 = unsigned long long;
__device__ __forceinline__ f2 pack2(float x, float y) {
  f2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void unpack2(f2 v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ f2 both(float x) { return pack2(x, x); }
__device__ __forceinline__ f2 fma2(f2 a, f2 b, f2 c) {
  f2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f2 mul2(f2 a, f2 b) {
  f2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// One value with both of a pair (the moves that make the pair cost less than two plain products)
__device__ __forceinline__ f2 mul1(float a, f2 b) { return mul2(both(a), b); }
__device__ __forceinline__ f2 fma1(float a, f2 b, f2 c) { return fma2(both(a), b, c); }
__device__ __forceinline__ f2 add2(f2 a, f2 b) {
  f2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ f2 ex2x2(f2 v) {
  float x, y;
  unpack2(v, x, y);
  return pack2(ex2(x), ex2(y));
}
__device__ __forceinline__ float sum2(f2 v) {
  float x, y;
  unpack2(v, x, y);
  return x + y;
}
__device__ __forceinline__ float rcp(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
// 1 / (1 + exp(-x)): within 2^-21 of itself for |x| up to 8 (the product with log2(e) is rounded once: |x| 2^-24 on top)
__device__ __forceinline__ f2 sigmoid_quick2(f2 x) {
  float a, b;
  unpack2(add2(ex2x2(mul2(x, both(-1.4426950408889634f))), both(1.f)), a, b);
  return pack2(rcp(a), rcp(b));
}

// V elements as they lie in memory <-> (V + 1) / 2 pairs
template <typename T, int V> struct Pairs;
template <int V> struct Pairs<float, V> {
  static __device__ __forceinline__ void get(const typename Pack<float, V>::Raw& raw, f2 (&p)[(V + 1) / 2]) {
    const float* f = reinterpret_cast<const float*>(&raw);
#pragma unroll
    for (int i = 0; i < (V + 1) / 2; ++i) p[i] = pack2(f[2 * i], 2 * i + 1 < V ? f[2 * i + 1] : 0.f);
  }
  static __device__ __forceinline__ typename Pack<float, V>::Raw put(const f2 (&p)[(V + 1) / 2]) {
    Pack<float, V> r;
#pragma unroll
    for (int i = 0; i < (V + 1) / 2; ++i) {
      float a, b;
      unpack2(p[i], a, b);
      r.e[2 * i] = a;
      if (2 * i + 1 < V) r.e[2 * i + 1 < V ? 2 * i + 1 : 0] = b;
    }
    return *reinterpret_cast<typename Pack<float, V>::Raw*>(&r);
  }
};
template <int V> struct Pairs<__nv_bfloat16, V> {
  static __device__ __forceinline__ void get(const typename Pack<__nv_bfloat16, V>::Raw& raw, f2 (&p)[(V + 1) / 2]) {
    if constexpr (V == 1) {
      p[0] = pack2(__uint_as_float(static_cast<unsigned>(raw) << 16), 0.f);
    } else {
      const unsigned* w = reinterpret_cast<const unsigned*>(&raw);
#pragma unroll
      for (int i = 0; i < V / 2; ++i) p[i] = pack2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
  }
  static __device__ __forceinline__ typename Pack<__nv_bfloat16, V>::Raw put(const f2 (&p)[(V + 1) / 2]) {
    float a, b;
    if constexpr (V == 1) {
      unpack2(p[0], a, b);
      return __bfloat16_as_ushort(__float2bfloat16_rn(a));
    } else {
      typename Pack<__nv_bfloat16, V>::Raw raw;
      __nv_bfloat162* w = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        unpack2(p[i], a, b);
        w[i] = __floats2bfloat162_rn(a, b);
      }
      return raw;
    }
  }
};
template <int V> struct Pairs<__half, V> {
  static __device__ __forceinline__ void get(const typename Pack<__half, V>::Raw& raw, f2 (&p)[(V + 1) / 2]) {
    if constexpr (V == 1) {
      p[0] = pack2(__half2float(__ushort_as_half(raw)), 0.f);
    } else {
      const __half2* w = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        const float2 f = __half22float2(w[i]);
        p[i] = pack2(f.x, f.y);
      }
    }
  }
  static __device__ __forceinline__ typename Pack<__half, V>::Raw put(const f2 (&p)[(V + 1) / 2]) {
    float a, b;
    if constexpr (V == 1) {
      unpack2(p[0], a, b);
      return __half_as_ushort(__float2half_rn(a));
    } else {
      typename Pack<__half, V>::Raw raw;
      __half2* w = reinterpret_cast<__half2*>(&raw);
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        unpack2(p[i], a, b);
        w[i] = __floats2half2_rn(a, b);
      }
      return raw;
    }
  }
};

}  // namespace bdh

// Rows of fp32 / fp16 / bf16 elements as fp32 registers: packs of V elements moved by one load or store of
// V * sizeof(T) bytes (4, 8 or 16), or element by element (V = 1) where a pointer, a stride or a width is not
// a multiple of that. All arithmetic of the kernels that include this is fp32; the one rounding to a
// 16-bit type is the store of a result.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace bdh {

template <typename T> __device__ __forceinline__ float elem_to_float(T v);
template <> __device__ __forceinline__ float elem_to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float elem_to_float<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float elem_to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T> __device__ __forceinline__ T elem_from_float(float v);
template <> __device__ __forceinline__ float elem_from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __half elem_from_float<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 elem_from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <int BYTES> struct RawOf;
template <> struct RawOf<2> { using type = unsigned short; };
template <> struct RawOf<4> { using type = unsigned; };
template <> struct RawOf<8> { using type = uint2; };
template <> struct RawOf<16> { using type = uint4; };

// V elements as they lie in memory; zero-initialised (the bit pattern 0 is 0.0 in all three types).
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
  using Raw = typename RawOf<sizeof(T) * V>::type;
  T e[V];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = elem_from_float<T>(0.f);
  }
  __device__ __forceinline__ void load(const T* p) {
    const Raw r = *reinterpret_cast<const Raw*>(p);
    *reinterpret_cast<Raw*>(this) = r;
  }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<Raw*>(p) = *reinterpret_cast<const Raw*>(this); }
  __device__ __forceinline__ float operator[](int i) const { return elem_to_float<T>(e[i]); }
  __device__ __forceinline__ void set(int i, float v) { e[i] = elem_from_float<T>(v); }
};

// Sequence lengths of a padded batch: int32 or int64, clamped to [0, T]; none: T.
struct Lengths {
  const void* ptr;
  int is64;
  __device__ __forceinline__ int get(int b, int T) const {
    if (ptr == nullptr) return T;
    const long long v = is64 ? static_cast<const long long*>(ptr)[b] : static_cast<const int*>(ptr)[b];
    return v < 0 ? 0 : (v > T ? T : static_cast<int>(v));
  }
};

// Asynchronous copies of 4, 8 or 16 bytes to shared memory (not `in`: zeros), closed into groups; a thread sees what it
// copied itself once it has waited for all but the newest LEFT groups.
template <int BYTES>
__device__ __forceinline__ void copy_async(void* dst, const void* src, bool in) {
  const unsigned to = static_cast<unsigned>(__cvta_generic_to_shared(dst));
  asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(src), "n"(BYTES), "r"(in ? BYTES : 0) : "memory");
}
__device__ __forceinline__ void copy_close() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

}  // namespace bdh

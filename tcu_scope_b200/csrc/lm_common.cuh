// What the language-model operators (linear_scan.cu, norm_residual.cu, token_logprobs.cu) share:
// element types, vectors of elements, the error word, reductions over a warp and a block.
// All arithmetic is in 32 bits; a result is rounded to its type once, when it is stored.
#pragma once

#include "../../include/tcu_scope.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

namespace tcu_lm {

constexpr int kMaxDevices = 64;

// Bit of tcu_device_error(): an index in device memory (an offset, a slot, a target) was out of
// range or named twice; what it names was left out.
constexpr unsigned kErrIndex = 8u;

// One word for each translation unit; tcu_device_error() joins those of the units that raise it (all but norm_residual.cu).
static __device__ unsigned int g_lm_error_word;

__device__ __forceinline__ void raise_index_error() { atomicOr(&g_lm_error_word, kErrIndex); }

// ------------------------------------------------------------------ elements
// (16 bytes are the widest access: longer vectors are several of them)
template <typename T, int V>
struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Vec {
  T v[V];
};

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load_vec(const T* p) {
  return *reinterpret_cast<const Vec<T, V>*>(p);
}
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> zero_vec() {
  Vec<T, V> r;
#pragma unroll
  for (int i = 0; i < V; ++i) r.v[i] = from_float<T>(0.f);
  return r;
}
// Two elements to and from floats: one instruction to round and pack them, one each to unpack.
template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
template <typename T>
__device__ __forceinline__ float2 unpack_pair(uint32_t x) {
  if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&x));
  return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
}

// V elements, converted.
template <typename T, int V>
__device__ __forceinline__ void to_floats(const Vec<T, V>& x, float (&y)[V]) {
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&x);
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float2 f = unpack_pair<T>(w[i]);
      y[2 * i] = f.x, y[2 * i + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) y[i] = to_float(x.v[i]);
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&x)[V]) {
  if constexpr (sizeof(T) == 2 && V % 2 == 0) {
    Vec<uint32_t, V / 2> r;
#pragma unroll
    for (int i = 0; i < V / 2; ++i) r.v[i] = pack_pair<T>(x[2 * i], x[2 * i + 1]);
    *reinterpret_cast<Vec<uint32_t, V / 2>*>(p) = r;
  } else {
    Vec<T, V> r;
#pragma unroll
    for (int i = 0; i < V; ++i) r.v[i] = from_float<T>(x[i]);
    *reinterpret_cast<Vec<T, V>*>(p) = r;
  }
}

// An index array of 32 or 64 bits.
__device__ __forceinline__ int64_t load_index(const void* p, int64_t i, bool wide) {
  return wide ? static_cast<const int64_t*>(p)[i] : int64_t(static_cast<const int32_t*>(p)[i]);
}

// ------------------------------------------------------------------ copies to shared memory
__device__ __forceinline__ void copy_async16(void* to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(uint32_t(__cvta_generic_to_shared(to))), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_async4(void* to, const void* from) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(uint32_t(__cvta_generic_to_shared(to))), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// Returns when all but the newest `pending` groups of this thread, 2 at most, have arrived.
__device__ __forceinline__ void copy_wait(int pending) {
  switch (pending) {
    case 0: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
    case 1: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
    default: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
  }
}

// ------------------------------------------------------------------ functions
constexpr float kLog2E = 1.44269504088896341f;

// 2^x within 2 ulp; results below 2^-126 are 0.
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 1 / x within 1 ulp.
__device__ __forceinline__ float reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// ------------------------------------------------------------------ pairs
// sm_100 adds, multiplies and multiply-adds two floats with one instruction.
#define TCU_PAIR_OP(name, op)                                                                   \
  __device__ __forceinline__ float2 name(float2 a, float2 b) {                                  \
    float2 r;                                                                                   \
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"           \
        op " z, x, y;\n\tmov.b64 {%0, %1}, z;\n\t}"                                             \
        : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));                       \
    return r;                                                                                   \
  }
TCU_PAIR_OP(add2, "add.rn.f32x2")
TCU_PAIR_OP(mul2, "mul.rn.f32x2")
#undef TCU_PAIR_OP
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(r.x), "=f"(r.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// ------------------------------------------------------------------ reductions
__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// ------------------------------------------------------------------ host side
inline int current_device() {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return -1;
  return dev >= 0 && dev < kMaxDevices ? dev : -1;
}

inline int sm_count() {
  static int counts[kMaxDevices];
  const int dev = current_device();
  if (dev < 0) return 0;
  if (counts[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
    counts[dev] = n;
  }
  return counts[dev];
}

inline bool aligned(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

inline size_t type_bytes(int64_t type) { return type == TCU_TYPE_F32 ? 4 : 2; }

inline bool known_type(int64_t t) { return t == TCU_TYPE_F16 || t == TCU_TYPE_F32 || t == TCU_TYPE_BF16; }

// Reads (and clears) this translation unit's error word.
inline int read_error_word(unsigned int* bits, int clear) {
  unsigned int v = 0;
  if (cudaDeviceSynchronize() != cudaSuccess) return TCU_ERR_CUDA;
  if (cudaMemcpyFromSymbol(&v, g_lm_error_word, sizeof(v)) != cudaSuccess) return TCU_ERR_CUDA;
  if (clear && v) {
    const unsigned int z = 0;
    if (cudaMemcpyToSymbol(g_lm_error_word, &z, sizeof(z)) != cudaSuccess) return TCU_ERR_CUDA;
  }
  *bits = v;
  return TCU_OK;
}

}  // namespace tcu_lm

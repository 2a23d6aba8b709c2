// Device helpers shared by the operators of kb_ops.h.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>

#include "kb_act.cuh"
#include "kb_tc_ptx.cuh"

namespace kb {

template <typename T> struct OpType;
template <> struct OpType<float> {
  static __device__ __forceinline__ float to(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
};
template <> struct OpType<__half> {
  static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};
template <> struct OpType<__nv_bfloat16> {
  static __device__ __forceinline__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};

// V elements in one access (V * sizeof(T) is 2, 4, 8 or 16 bytes and divides the address).
template <int BYTES> struct OpWord;
template <> struct OpWord<2> { typedef uint16_t type; };
template <> struct OpWord<4> { typedef uint32_t type; };
template <> struct OpWord<8> { typedef uint2 type; };
template <> struct OpWord<16> { typedef uint4 type; };
template <typename T, int V> struct OpVec {
  typedef typename OpWord<sizeof(T) * V>::type word;
  union { word w; T e[V]; };
  __device__ __forceinline__ OpVec() {}
  __device__ __forceinline__ void load(const T* p) { w = *reinterpret_cast<const word*>(p); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<word*>(p) = w; }
};

// Activations: exact functions for fp32 results, the special-function forms of the convolutions' epilogues for 16-bit ones
// (their error is far below the rounding of the result).
template <typename T> __device__ __forceinline__ float opAct(float v, int act) { return sizeof(T) == 4 ? applyActF(v, act) : fastAct(v, act); }

}  // namespace kb

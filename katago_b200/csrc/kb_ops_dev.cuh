// Device helpers shared by the operators of kb_ops.h.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstdint>
#include <type_traits>

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

// Activations: library functions for fp32 results, special-function forms as in the convolutions' epilogues for 16-bit ones (their
// error is far below the rounding of the result).  A NaN stays one, +infinity too: fmaxf(NaN, 0) is 0, and x - 2xr is NaN for x = inf and
// r = 0 where x (1 - 2r) is not.  mish(x) = x tanh(log(1 + e^x)) = x (n^2 + 2n) / (n^2 + 2n + 2) with n = e^x:
// nothing cancels, and one exponential and a division take the place of exp, log1p and tanh.
__device__ __forceinline__ float opMish(float x, float arg) {
  const float n = expf(fminf(arg, 30.0f));  // the quotient is 1 from about 9 on
  const float m = n * (n + 2.0f);
  return x * (m / (m + 2.0f));
}
__device__ __forceinline__ float opRelu(float x) {
  float y;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(y) : "f"(x));
  return y;
}
// x (1 - 2r), r = 1 / (n^2 + 2n + 2): two values with the packed fp32 instructions.
__device__ __forceinline__ float2 opFastMish(float2 x, float2 arg) {
  auto both = [](float c) { return make_float2(c, c); };
  const float2 e = __fmul2_rn(arg, both(1.4426950408889634f));
  const float2 n = make_float2(ex2Approx(e.x), ex2Approx(e.y));
  const float2 d = __ffma2_rn(n, __ffma2_rn(n, both(-0.5f), both(-1.0f)), both(-1.0f));
  return __fmul2_rn(x, __fadd2_rn(make_float2(rcpApprox(d.x), rcpApprox(d.y)), both(1.0f)));
}
__device__ __forceinline__ float opFastAct(float v, int act) {
  if(act == KB_ACT_RELU) return opRelu(v);
  if(act == KB_ACT_MISH) return opFastMish(make_float2(v, v), make_float2(v, v)).x;
  if(act == KB_ACT_MISH_SCALE8) return opFastMish(make_float2(v, v), make_float2(8.0f * v, 8.0f * v)).x;
  return fastAct(v, act);
}
template <typename T> __device__ __forceinline__ float opAct(float v, int act) {
  if(sizeof(T) != 4) return opFastAct(v, act);
  if(act == KB_ACT_RELU) return opRelu(v);
  if(act == KB_ACT_MISH) return opMish(v, v);
  if(act == KB_ACT_MISH_SCALE8) return opMish(v, 8.0f * v);
  return applyActF(v, act);
}

// The same for several fp32 values: one choice of the function for all of them.
template <int U> __device__ __forceinline__ void opActF32(float (&v)[U], int act) {
  switch(act) {
    case KB_ACT_RELU:
#pragma unroll
      for(int u = 0; u < U; u++) v[u] = opRelu(v[u]);
      break;
    case KB_ACT_SILU:
#pragma unroll
      for(int u = 0; u < U; u++) v[u] = applyActF(v[u], KB_ACT_SILU);
      break;
    case KB_ACT_MISH:
#pragma unroll
      for(int u = 0; u < U; u++) v[u] = opMish(v[u], v[u]);
      break;
    case KB_ACT_MISH_SCALE8:
#pragma unroll
      for(int u = 0; u < U; u++) v[u] = opMish(v[u], 8.0f * v[u]);
      break;
    default: break;
  }
}

// Reads of another block's shared memory (an address that clusterMapAddr gave).
__device__ __forceinline__ float4 ldCluster4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float ldCluster1(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// Bounded wait of a role of these kernels (about 2 s, or limitNs).  A wait that runs out raises the abort flag and leaves `code` in the status
// word, which is page-locked host memory (hence a plain store); it returns false, as does one that finds the flag raised, and
// the role then leaves its loops.
// The clock is read only after some dozens of tries: reading it takes longer than most waits do.
__device__ __forceinline__ bool opWaitSpin(uint32_t bar, uint32_t parity, volatile int* abortFlag, volatile int* status, int code, uint64_t limitNs = 2000000000ull) {
  uint64_t t0 = 0;
  for(uint32_t spins = 1;; spins++) {
    if(mbarTryWait(bar, parity)) return true;
    if((spins & 63u) == 0u) {
      if(*abortFlag) return false;
      const uint64_t now = globalTimerNs();
      if(t0 == 0) t0 = now;
      else if(now - t0 > limitNs) {
        *abortFlag = 1;
        *status = code;
        __threadfence_system();
        return false;
      }
    }
  }
}
static __device__ __noinline__ bool opWaitOn(uint32_t bar, uint32_t parity, volatile int* abortFlag, volatile int* status, int code) {
  return opWaitSpin(bar, parity, abortFlag, status, code);
}
__device__ __forceinline__ bool opWait(uint32_t bar, uint32_t parity, volatile int* abortFlag, volatile int* status, int code) {
  return mbarTryWait(bar, parity) != 0u || opWaitOn(bar, parity, abortFlag, status, code);
}
// For the sums of `slices` slices of K, which may take longer than any other wait: 20 us for each on top (the slowest, of rows on odd
// boundaries, take 3).
static __device__ __noinline__ bool opWaitSumsOn(uint32_t bar, uint32_t parity, volatile int* abortFlag, volatile int* status, int code, int slices) {
  return opWaitSpin(bar, parity, abortFlag, status, code, 2000000000ull + 20000ull * (uint64_t)slices);
}
__device__ __forceinline__ bool opWaitSums(uint32_t bar, uint32_t parity, volatile int* abortFlag, volatile int* status, int code, int slices) {
  return mbarTryWait(bar, parity) != 0u || opWaitSumsOn(bar, parity, abortFlag, status, code, slices);
}
// The same in line, for kernels that move registers between warpgroups (ptxas finds no allocation with a call in them).
__device__ __forceinline__ bool opWaitInline(uint32_t bar, uint32_t parity, volatile int* abortFlag, volatile int* status, int code) {
  return opWaitSpin(bar, parity, abortFlag, status, code);
}

__device__ __forceinline__ void tmaLoad4d(uint32_t dst, const CUtensorMap* tmap, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile(
    "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
    ::"r"(dst), "l"(tmap), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
    : "memory");
}

// 32 lanes x 16 consecutive columns -> 16 registers per thread, and the wait that names them (kb_tc_ptx.cuh, tmemLd32).
__device__ __forceinline__ void tmemLd16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmemLdWaitFor(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]) : : "memory");
}

// Two values in one 32-bit word of the 16-bit type, the first in the low half.
template <typename T> __device__ __forceinline__ uint32_t opPack(float lo, float hi);
template <> __device__ __forceinline__ uint32_t opPack<__half>(float lo, float hi) { const __half2 h = __floats2half2_rn(lo, hi); return *reinterpret_cast<const uint32_t*>(&h); }
template <> __device__ __forceinline__ uint32_t opPack<__nv_bfloat16>(float lo, float hi) { const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi); return *reinterpret_cast<const uint32_t*>(&h); }
template <typename T> __device__ __forceinline__ float2 opUnpack(uint32_t u);
template <> __device__ __forceinline__ float2 opUnpack<__half>(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
template <> __device__ __forceinline__ float2 opUnpack<__nv_bfloat16>(uint32_t u) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&u)); }

// Instruction descriptor of tcgen05.mma kind::f16 with fp32 accumulators: both operands of type T, K-major (bMn: B is MN-major).
template <typename T> __host__ __device__ constexpr uint32_t opIdesc(int m, int n, bool bMn = false) {
  const uint32_t fmt = sizeof(T) == 2 && !std::is_same<T, __half>::value ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | (bMn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Words of a shared-memory matrix descriptor, 128-byte swizzle, 8-row groups 1024 bytes apart (kb_tc_ptx.cuh, makeSmemDesc).
constexpr uint32_t OP_DESC_HI = (uint32_t)(1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t opDescLo(uint32_t saddr) { return ((saddr & 0x3FFFFu) >> 4) | (1u << 16); }

}  // namespace kb

// y = act(x w^T + bias) + residual on the tensor cores: fp16 / bf16 matrices whose rows start on 16-byte boundaries.
//
// matmulTcKernel: persistent CTAs of 128 x BN tiles.  Warp 0 feeds 64-channel slices of x and w into a ring of slots by TMA
// (128-byte swizzle; what a tile has beyond the matrices' ends is zero-filled), warp 1 issues tcgen05.mma into one of two
// accumulators in tensor memory, eight warps take the other accumulator out: 32 rows x 32 columns at a time, each warp on its own,
// with the residual arriving in a slot of the warp's two by TMA, the result replacing it there and leaving by TMA.  Where y's
// rows are not on 16-byte boundaries the warp reads the residual and writes the slot's rows itself, a row (64 bytes) per
// instruction.
//
// What bounds it: the tensor pipe for K of a few hundred and more, memory below.  BN is the width whose tiles, in whole rounds over
// the SMs, cost the least (an MMA costs BN/2 cycles, at least about 44: its A rows have to be read).  Tiles are walked in bands of
// 16 row tiles, so that the x and w rows of the tiles in flight (16 x 128 and some 9 x 256) stay in L2.
#include "kb_kernels.cuh"
#include "kb_ops.h"
#include "kb_ops_dev.cuh"

#include <algorithm>

namespace kb {

namespace {

constexpr int MT_BM = 128, MT_BK = 64, MT_UNIT = 32;  // rows, channels of a slice; rows and columns of an output unit
constexpr int MT_EPI_WARPS = 8, MT_THREADS = 64 + 32 * MT_EPI_WARPS;
constexpr int MT_A_BYTES = MT_BM * MT_BK * 2, MT_UNIT_BYTES = MT_UNIT * MT_UNIT * 2;
constexpr int MT_MAX_STAGES = 8, MT_BAND = 16;
constexpr int MT_ERR = 301;

struct MatmulTcArgs {
  MatmulArgs m;
  int BN, kSlices, tilesM, tilesN, stages;
  int tmaOut, tmaRes;  // y / the residual by TMA
  uint32_t idesc, tmemCols;
};

__device__ __forceinline__ void mtTile(const MatmulTcArgs& a, int t, int& tm, int& tn) {
  const int band = t / (MT_BAND * a.tilesN), rest = t - band * MT_BAND * a.tilesN;
  const int rows = min(MT_BAND, a.tilesM - band * MT_BAND);
  tn = rest / rows;
  tm = band * MT_BAND + rest - tn * rows;
}

template <typename T>
__global__ void __launch_bounds__(MT_THREADS, 1) matmulTcKernel(
  const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmY,
  const __grid_constant__ CUtensorMap tmR, const MatmulTcArgs a) {
  extern __shared__ uint8_t smemRaw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smemRaw) + 1023) & ~(uintptr_t)1023);
  const int slotBytes = MT_A_BYTES + a.BN * MT_BK * 2;
  uint8_t* sUnits = smem + (size_t)a.stages * slotBytes;  // [warp][2] output units
  uint64_t* bars = reinterpret_cast<uint64_t*>(sUnits + MT_EPI_WARPS * 2 * MT_UNIT_BYTES);
  uint64_t* bFull = bars;                      // a slice has arrived
  uint64_t* bEmpty = bFull + MT_MAX_STAGES;    // its MMAs have completed
  uint64_t* bAcc = bEmpty + MT_MAX_STAGES;     // [2] an accumulator is complete
  uint64_t* bTaken = bAcc + 2;                 // [2] an accumulator has been read
  uint64_t* bRes = bTaken + 2;                 // [warp][2] a residual unit has arrived
  uint32_t* tmemSlot = reinterpret_cast<uint32_t*>(bRes + MT_EPI_WARPS * 2);
  volatile int* abortFlag = reinterpret_cast<volatile int*>(tmemSlot + 1);

  const int warp = warpIndex(), lane = threadIdx.x & 31;
  if(threadIdx.x == 0) {
    for(int i = 0; i < MT_MAX_STAGES; i++) { mbarInit(smemU32(&bFull[i]), 1); mbarInit(smemU32(&bEmpty[i]), 1); }
    for(int i = 0; i < 2; i++) { mbarInit(smemU32(&bAcc[i]), 1); mbarInit(smemU32(&bTaken[i]), MT_EPI_WARPS); }
    for(int i = 0; i < MT_EPI_WARPS * 2; i++) mbarInit(smemU32(&bRes[i]), 1);
    *abortFlag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fenceProxyAsync();
  }
  if(warp == 1) { tmemAlloc(smemU32(tmemSlot), a.tmemCols); tmemRelinquish(); }
  tcFenceBefore();
  __syncthreads();
  tcFenceAfter();
  gridDepLaunch();
  gridDepWait();
  const uint32_t tmem = *tmemSlot;
  const int tiles = a.tilesM * a.tilesN;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return opWait(smemU32(bar), parity, abortFlag, a.m.status, MT_ERR); };

  if(warp == 0) {
    if(electOne()) {
      uint32_t it = 0;  // slices requested
      bool ok = true;
      for(int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        int tm, tn;
        mtTile(a, t, tm, tn);
        for(int k = 0; k < a.kSlices; k++, it++) {
          const uint32_t s = it % a.stages, use = it / a.stages;
          if(use > 0 && !wait(&bEmpty[s], (use - 1) & 1u)) { ok = false; break; }
          uint8_t* slot = smem + (size_t)s * slotBytes;
          mbarExpectTx(smemU32(&bFull[s]), (uint32_t)slotBytes);
          tmaLoad2d(smemU32(slot), &tmX, k * MT_BK, tm * MT_BM, smemU32(&bFull[s]));
          tmaLoad2d(smemU32(slot + MT_A_BYTES), &tmW, k * MT_BK, tn * a.BN, smemU32(&bFull[s]));
        }
      }
      if(!ok) {  // copies in flight land (each within a millisecond) before the CTA may end
        volatile int keepWaiting = 0;
        for(uint32_t i = it > (uint32_t)a.stages ? it - a.stages : 0; i < it; i++) mbarWait(smemU32(&bFull[i % a.stages]), (i / a.stages) & 1u, &keepWaiting, 1000000ull);
      }
    }
    __syncwarp();
  }
  else if(warp == 1) {
    if(electOne()) {
      uint32_t it = 0, n = 0;  // slices multiplied, tiles begun
      bool ok = true;
      for(int t = blockIdx.x; t < tiles && ok; t += gridDim.x, n++) {
        const uint32_t b = n & 1u;
        if(n > 1 && !wait(&bTaken[b], ((n >> 1) - 1) & 1u)) break;
        tcFenceAfter();
        const uint32_t d = tmem + b * (uint32_t)a.BN;
        for(int k = 0; k < a.kSlices; k++, it++) {
          const uint32_t s = it % a.stages;
          if(!wait(&bFull[s], (it / a.stages) & 1u)) { ok = false; break; }
          tcFenceAfter();
          const uint32_t aLo = opDescLo(smemU32(smem + (size_t)s * slotBytes)), bLo = opDescLo(smemU32(smem + (size_t)s * slotBytes + MT_A_BYTES));
#pragma unroll
          for(int j = 0; j < MT_BK / 16; j++) ummaLoHi(d, aLo + 2 * j, bLo + 2 * j, OP_DESC_HI, a.idesc, (k | j) != 0 ? 1u : 0u);
          ummaCommit(smemU32(&bEmpty[s]));
        }
        if(ok) ummaCommit(smemU32(&bAcc[b]));
      }
    }
    __syncwarp();
  }
  else {
    const int quarter = warp & 3, half = (warp - 2) >> 2;  // TMEM lanes of this warp; odd or even units
    uint8_t* units = sUnits + (warp - 2) * 2 * MT_UNIT_BYTES;
    uint64_t* res = bRes + (warp - 2) * 2;
    const bool hasRes = a.m.residual != nullptr;
    uint32_t n = 0, u = 0;  // tiles begun, units begun
    bool ok = true;
    for(int t = blockIdx.x; t < tiles && ok; t += gridDim.x, n++) {
      int tm, tn;
      mtTile(a, t, tm, tn);
      const int m0 = tm * MT_BM + quarter * 32, n0 = tn * a.BN;
      const uint32_t b = n & 1u;
      const int nUnits = a.m.M > m0 ? (min(a.BN, a.m.N - n0) + MT_UNIT - 1) / MT_UNIT : 0;  // units with anything in them
      auto requestResidual = [&](int c, uint32_t slot) {  // after the store from that slot has been read
        mbarExpectTx(smemU32(&res[slot]), (uint32_t)MT_UNIT_BYTES);
        tmaLoad2d(smemU32(units + slot * MT_UNIT_BYTES), &tmR, n0 + c * MT_UNIT, m0, smemU32(&res[slot]));
      };
      if(a.tmaRes && half < nUnits && electOne()) {
        bulkWaitRead1();
        requestResidual(half, u & 1u);
      }
      ok = wait(&bAcc[b], (n >> 1) & 1u);
      if(__any_sync(0xffffffffu, !ok)) ok = false;
      tcFenceAfter();
      for(int c = half; c < nUnits && ok; c += 2, u++) {
        const uint32_t slot = u & 1u;
        uint8_t* unit = units + slot * MT_UNIT_BYTES;
        uint32_t r[32];
        __syncwarp();
        tmemLd32(tmem + b * (uint32_t)a.BN + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(c * MT_UNIT), r);
        const int nc = n0 + c * MT_UNIT;
        if(a.tmaRes) {
          if(c + 2 < nUnits && electOne()) {
            bulkWaitRead0();  // the unit before has left the other slot
            requestResidual(c + 2, slot ^ 1u);
          }
        }
        else if(a.tmaOut) {
          if(electOne()) bulkWaitRead1();
        }
        __syncwarp();
        const float* bias = a.m.bias;
        tmemLdWaitFor(r);
        if(c + 2 >= nUnits) {  // the accumulator has been read
          tcFenceBefore();
          __syncwarp();
          if(lane == 0) mbarArrive(smemU32(&bTaken[b]));
        }
        if(bias) {
          const float bv = nc + lane < a.m.N ? bias[nc + lane] : 0.0f;
#pragma unroll
          for(int j = 0; j < 32; j++) r[j] = __float_as_uint(__uint_as_float(r[j]) + __shfl_sync(0xffffffffu, bv, j));
        }
        switch(a.m.act) {
          case KB_ACT_RELU:
#pragma unroll
            for(int j = 0; j < 32; j++) r[j] = __float_as_uint(fastAct(__uint_as_float(r[j]), KB_ACT_RELU));
            break;
          case KB_ACT_MISH:
#pragma unroll
            for(int j = 0; j < 32; j++) r[j] = __float_as_uint(fastAct(__uint_as_float(r[j]), KB_ACT_MISH));
            break;
          case KB_ACT_SILU:
#pragma unroll
            for(int j = 0; j < 32; j++) r[j] = __float_as_uint(fastAct(__uint_as_float(r[j]), KB_ACT_SILU));
            break;
          case KB_ACT_MISH_SCALE8:
#pragma unroll
            for(int j = 0; j < 32; j++) r[j] = __float_as_uint(fastAct(__uint_as_float(r[j]), KB_ACT_MISH_SCALE8));
            break;
          default: break;
        }
        if(hasRes) {
          if(a.tmaRes) {
            ok = wait(&res[slot], (u >> 1) & 1u);
            if(__any_sync(0xffffffffu, !ok)) { ok = false; break; }
          }
          else {
            // a row of the unit per instruction into the slot, its 16-byte pieces where the swizzle puts them
            __syncwarp();
            for(int i = 0; i < 32; i++) {
              T v = OpType<T>::from(0.0f);
              if(m0 + i < a.m.M && nc + lane < a.m.N) v = ((const T*)a.m.residual)[(int64_t)(m0 + i) * a.m.ldr + nc + lane];
              *reinterpret_cast<T*>(unit + i * 64 + (((lane >> 3) ^ ((i >> 1) & 3)) << 4) + (lane & 7) * 2) = v;
            }
            __syncwarp();
          }
        }
        uint8_t* mine = unit + lane * 64;
        const int sw = (lane >> 1) & 3;
#pragma unroll
        for(int q = 0; q < 4; q++) {
          uint4* p = reinterpret_cast<uint4*>(mine + ((q ^ sw) << 4));
          uint32_t w[4];
          if(hasRes) {
            const uint4 old = *p;
            const uint32_t o[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
            for(int e = 0; e < 4; e++) {
              const float2 f = opUnpack<T>(o[e]);
              w[e] = opPack<T>(__uint_as_float(r[8 * q + 2 * e]) + f.x, __uint_as_float(r[8 * q + 2 * e + 1]) + f.y);
            }
          }
          else {
#pragma unroll
            for(int e = 0; e < 4; e++) w[e] = opPack<T>(__uint_as_float(r[8 * q + 2 * e]), __uint_as_float(r[8 * q + 2 * e + 1]));
          }
          *p = make_uint4(w[0], w[1], w[2], w[3]);
        }
        if(a.tmaOut) {
          fenceProxyAsync();
          __syncwarp();
          if(electOne()) {
            tmaStore2d(&tmY, smemU32(unit), nc, m0);
            bulkCommit();
          }
        }
        else {
          __syncwarp();
          for(int i = 0; i < 32; i++)
            if(m0 + i < a.m.M && nc + lane < a.m.N)
              ((T*)a.m.y)[(int64_t)(m0 + i) * a.m.ldy + nc + lane] = *reinterpret_cast<const T*>(unit + i * 64 + (((lane >> 3) ^ ((i >> 1) & 3)) << 4) + (lane & 7) * 2);
          __syncwarp();
        }
      }
      if(half >= nUnits && ok) {  // nothing of this accumulator is this warp's
        if(lane == 0) mbarArrive(smemU32(&bTaken[b]));
      }
    }
    if(!ok && a.tmaRes) {  // a residual unit that is still on its way
      volatile int keepWaiting = 0;
      for(uint32_t s = 0; s < 2; s++) mbarWait(smemU32(&res[s]), ((u + (s != (u & 1u))) >> 1) & 1u, &keepWaiting, 1000000ull);
    }
    if(a.tmaOut) bulkWaitAll();
  }
  tcFenceBefore();
  __syncthreads();
  if(warp == 1) { tcFenceAfter(); tmemDealloc(tmem, a.tmemCols); }
}

bool encodeRows(CUtensorMap* map, int dt, const void* p, int64_t cols, int64_t rows, int64_t ld, int boxCols, int boxRows, CUtensorMapSwizzle sw) {
  const uint64_t dims[2] = {(uint64_t)cols, (uint64_t)rows}, strides[1] = {(uint64_t)ld * 2};
  const uint32_t box[2] = {(uint32_t)boxCols, (uint32_t)boxRows};
  return encodeTiled(map, dt, p, 2, dims, strides, box, sw);
}

bool rowsAligned(const void* p, int64_t ld) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0; }

template <typename T> cudaError_t launchWide(cudaStream_t st, const MatmulArgs& m) {
  MatmulTcArgs a = {};
  a.m = m;
  const int sms = smCount();
  a.tilesM = (m.M + MT_BM - 1) / MT_BM;
  a.kSlices = (m.K + MT_BK - 1) / MT_BK;
  // the width whose tiles cost the least in whole rounds; of equal ones the widest
  double best = 0;
  for(int bn = 256; bn >= 32; bn -= 32) {
    const double rounds = (double)(((long long)a.tilesM * ((m.N + bn - 1) / bn) + sms - 1) / sms);
    const double cost = rounds * std::max(44.0, bn / 2.0);
    if(a.BN == 0 || cost < best) { best = cost; a.BN = bn; }
  }
  a.tilesN = (m.N + a.BN - 1) / a.BN;
  const int slotBytes = MT_A_BYTES + a.BN * MT_BK * 2;
  const size_t fixed = MT_EPI_WARPS * 2 * MT_UNIT_BYTES + 1024 + 1024;
  a.stages = (int)std::min<size_t>(MT_MAX_STAGES, (227 * 1024 - fixed) / slotBytes);
  a.idesc = opIdesc<T>(MT_BM, a.BN);
  a.tmemCols = 32;
  while(a.tmemCols < 2u * a.BN) a.tmemCols *= 2;
  a.tmaOut = rowsAligned(m.y, m.ldy);
  a.tmaRes = a.tmaOut && m.residual && rowsAligned(m.residual, m.ldr);
  CUtensorMap x, w, y = {}, r = {};
  bool ok = encodeRows(&x, m.dt, m.x, m.K, m.M, m.ldx, MT_BK, MT_BM, CU_TENSOR_MAP_SWIZZLE_128B) &&
            encodeRows(&w, m.dt, m.w, m.K, m.N, m.ldw, MT_BK, a.BN, CU_TENSOR_MAP_SWIZZLE_128B);
  if(a.tmaOut) ok = ok && encodeRows(&y, m.dt, m.y, m.N, m.M, m.ldy, MT_UNIT, MT_UNIT, CU_TENSOR_MAP_SWIZZLE_64B);
  if(a.tmaRes) ok = ok && encodeRows(&r, m.dt, m.residual, m.N, m.M, m.ldr, MT_UNIT, MT_UNIT, CU_TENSOR_MAP_SWIZZLE_64B);
  if(!ok) return cudaErrorInvalidValue;
  static SharedMemoryOptIn optIn;
  const cudaError_t e = optIn((const void*)matmulTcKernel<T>, 227 * 1024);
  if(e != cudaSuccess) return e;
  const int tiles = a.tilesM * a.tilesN;
  return launchDependent(matmulTcKernel<T>, dim3(std::min(tiles, sms)), dim3(MT_THREADS), (size_t)a.stages * slotBytes + fixed, st, x, w, y, r, a);
}

}  // namespace

bool matmulTcEligible(const MatmulArgs& a) {
  return (a.dt == DT_F16 || a.dt == DT_BF16) && rowsAligned(a.x, a.ldx) && rowsAligned(a.w, a.ldw) &&
         ((long long)a.M + 127) / 128 * (((long long)a.N + 31) / 32) < (1LL << 31);
}

cudaError_t launchMatmulTc(cudaStream_t st, const MatmulArgs& a) { return a.dt == DT_F16 ? launchWide<__half>(st, a) : launchWide<__nv_bfloat16>(st, a); }

}  // namespace kb

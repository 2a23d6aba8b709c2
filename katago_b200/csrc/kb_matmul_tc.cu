// y = act(x w^T + bias) + residual on the tensor cores: fp16 / bf16.
//
// matmulTcKernel: persistent CTAs of 128 x BN tiles.  Warp 0 feeds 64-channel slices of x and w into a ring of slots by TMA
// (128-byte swizzle; what a tile has beyond the matrices' ends is zero-filled), warp 1 issues tcgen05.mma into one of two
// accumulators in tensor memory, sixteen warps take the other accumulator out: 32 rows x 32 columns at a time, each warp on its
// own, through a slot of its own that TMA empties.  The residual arrives by TMA too, a unit ahead in another slot where a tile's
// products are short, in the same slot where they are long.  Where y's rows are not on 16-byte boundaries the warp reads the
// residual and writes the slot's rows itself, a row per instruction; so it writes the last unit of rows that end inside sixteen bytes, since a
// TMA store writes those sixteen whole, whatever lies behind the row's end.  (Eight warps, 32 or 64 columns at a time: 46208 x 1024 x 384
// fp16 66 us with bias and SiLU, 51 us with sixteen, in the first milliseconds; 60 us over seconds, at the power limit.  A warp's own chain of
// waits and special functions was what took the time.)
//
// Rows on other boundaries (PLAIN, both kernels): eight warps take the place of TMA and write the swizzled 128 bytes of a row that it would
// have.  Rows on 4-byte boundaries go by asynchronous copies of two channels per lane (4096 x 4096 x 4098 bf16 860 us, 160 TFLOP/s;
// the copies' rate bounds it), others by two 2-byte loads per lane with sixteen rows in flight, whose latency bounds it (4097^3 bf16
// 1.30 ms, 105 TFLOP/s).  Eight warps then take accumulators out.
//
// matmulSkinnyKernel (few tiles): the weights are the 128 rows of a tile and up to 128 rows of x its columns, so that few rows of x
// waste none of the tensor pipe and the weights are what streams.  A cluster of up to eight CTAs cuts K; each leaves its sums in its
// own shared memory, and after a cluster barrier each adds a share of the rows of x over the cluster, in the order of K, through
// distributed shared memory: no workspace, no second launch, the same order every time.
//
// What bounds the first: the tensor pipe for K of a few hundred and more, memory below.  BN is the width whose tiles, in whole rounds over
// the SMs, cost the least (an MMA costs BN/2 cycles, at least about 44: its A rows have to be read; and (128 + BN) x 32 bytes come
// from L2 for it, at some 75 per cycle and SM).  Tiles are walked in bands of
// 16 row tiles, so that the x and w rows of the tiles in flight (16 x 128 and some 9 x 256) stay in L2.
#include "kb_kernels.cuh"
#include "kb_ops.h"
#include "kb_ops_dev.cuh"

#include <algorithm>

namespace kb {

namespace {

constexpr int MT_BM = 128, MT_BK = 64, MT_UNIT = 32;  // rows, channels of a slice; columns of an output unit (of 32 rows)
constexpr int MT_THREADS = 576, MT_LOADERS = 8;       // warps: request, multiply, sixteen for the output; or eight and MT_LOADERS
constexpr int MT_A_BYTES = MT_BM * MT_BK * 2, MT_UNIT_BYTES = 32 * MT_UNIT * 2;
constexpr int MT_MAX_STAGES = 8, MT_BAND = 16;
constexpr int MT_ERR = 301;

struct MatmulTcArgs {
  MatmulArgs m;
  int BN, kSlices, tilesM, tilesN, stages;
  int tmaOut, tmaRes;  // y / the residual by TMA
  int resAhead;        // ... into slots of its own
  uint32_t idesc, tmemCols;
};

__device__ __forceinline__ void mtTile(const MatmulTcArgs& a, int t, int& tm, int& tn) {
  const int band = t / (MT_BAND * a.tilesN), rest = t - band * MT_BAND * a.tilesN;
  const int rows = min(MT_BAND, a.tilesM - band * MT_BAND);
  tn = rest / rows;
  tm = band * MT_BAND + rest - tn * rows;
}

// Two neighbouring 16-bit elements at any address, each if its condition holds, else 0.  Predicated: a branch around each load would
// wait for it.
__device__ __forceinline__ void loadPair(const uint16_t* p, bool first, bool second, uint16_t& lo, uint16_t& hi) {
  asm volatile(
    "{\n\t.reg .pred a, b;\n\tsetp.ne.b32 a, %3, 0;\n\tsetp.ne.b32 b, %4, 0;\n\tmov.b16 %0, 0;\n\tmov.b16 %1, 0;\n\t"
    "@a ld.global.b16 %0, [%2];\n\t@b ld.global.b16 %1, [%2+2];\n\t}"
    : "=&h"(lo), "=&h"(hi) : "l"(p), "r"((int)first), "r"((int)second) : "memory");
}

// Rows of a matrix from `row0` on, `end` in all.
struct PlainRows {
  const uint16_t* p;
  int64_t ld;
  int row0, end;
};

// The slices of 64 channels that MT_LOADERS warps bring into the ring in place of TMA: 128 rows of `a`, then `nb` rows of `b`, each as
// 128 bytes in the 128-byte swizzle; zeros beyond the ends.  Rows on 4-byte boundaries are copied asynchronously, two channels per lane, and a
// slice is announced when those of the two after it have been requested; others go through registers, U rows in flight.
template <int U, bool PAIRS> struct PlainLoader {
  uint64_t* full;
  int stages, K, loader, lane;
  uint32_t it;  // slices requested

  __device__ __forceinline__ uint32_t lag() const { return stages >= 3 ? 2u : 0u; }  // with fewer slots a wait for a free one would be for itself
  __device__ __forceinline__ void announce(uint32_t i) {
    fenceProxyAsync();
    __syncwarp();
    if(lane == 0) mbarArrive(smemU32(&full[i % (uint32_t)stages]));
  }
  __device__ __forceinline__ void slice(uint8_t* slot, const PlainRows& a, const PlainRows& b, int nb, int k) {
    const int c = k * MT_BK + 2 * lane, rows = MT_BM + nb;
    if(PAIRS) {
      const uint32_t bytes = c + 1 < K ? 4 : c < K ? 2 : 0;
#pragma unroll 4
      for(int r = loader; r < rows; r += MT_LOADERS) {
        const bool first = r < MT_BM;
        const int row = first ? a.row0 + r : b.row0 + r - MT_BM;
        const uint32_t n = row < (first ? a.end : b.end) ? bytes : 0u;
        const uint16_t* src = first ? a.p + row * a.ld + c : b.p + row * b.ld + c;
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smemU32(slot + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4)), "l"(n ? src : a.p), "r"(n) : "memory");
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      if(lag() == 2) {
        asm volatile("cp.async.wait_group 2;" ::: "memory");
        if(it >= 2) announce(it - 2);
      }
      else {
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        announce(it);
      }
    }
    else {
      for(int r0 = loader; r0 < rows; r0 += MT_LOADERS * U) {
        uint16_t lo[U], hi[U];
#pragma unroll
        for(int u = 0; u < U; u++) {
          const int r = r0 + u * MT_LOADERS;
          const bool first = r < MT_BM;
          const int row = first ? a.row0 + r : b.row0 + r - MT_BM;
          const bool in = r < rows && row < (first ? a.end : b.end);
          loadPair((first ? a.p + row * a.ld : b.p + row * b.ld) + c, in && c < K, in && c + 1 < K, lo[u], hi[u]);
        }
#pragma unroll
        for(int u = 0; u < U; u++) {
          const int r = r0 + u * MT_LOADERS;
          if(r < rows) *reinterpret_cast<uint32_t*>(slot + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4) = lo[u] | (uint32_t)hi[u] << 16;
        }
      }
      announce(it);
    }
    it++;
  }
  __device__ __forceinline__ void finish() {
    if(!PAIRS) return;
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    for(uint32_t i = it > lag() ? it - lag() : 0; i < it; i++) announce(i);
  }
};

// Whether rows start on 4-byte boundaries.
__device__ __forceinline__ bool pairRows(const MatmulArgs& m) { return (((uintptr_t)m.x | (uintptr_t)m.w) & 3) == 0 && ((m.ldx | m.ldw) & 1) == 0; }

template <typename T, bool PLAIN>
__global__ void __launch_bounds__(MT_THREADS, 1) matmulTcKernel(
  const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmY,
  const __grid_constant__ CUtensorMap tmR, const MatmulTcArgs a) {
  constexpr int MT_EPI_WARPS = PLAIN ? 8 : 16, MT_GROUPS = MT_EPI_WARPS / 4;
  extern __shared__ uint8_t smemRaw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smemRaw) + 1023) & ~(uintptr_t)1023);
  const int slotBytes = MT_A_BYTES + a.BN * MT_BK * 2;
  uint8_t* sUnits = smem + (size_t)a.stages * slotBytes;  // [warp] output units, [warp] residual units
  uint64_t* bars = reinterpret_cast<uint64_t*>(sUnits + MT_EPI_WARPS * (a.resAhead ? 2 : 1) * MT_UNIT_BYTES);
  uint64_t* bFull = bars;                      // a slice has arrived
  uint64_t* bEmpty = bFull + MT_MAX_STAGES;    // its MMAs have completed
  uint64_t* bAcc = bEmpty + MT_MAX_STAGES;     // [2] an accumulator is complete
  uint64_t* bTaken = bAcc + 2;                 // [2] an accumulator has been read
  uint64_t* bRes = bTaken + 2;                 // [warp] a residual unit has arrived
  uint32_t* tmemSlot = reinterpret_cast<uint32_t*>(bRes + MT_EPI_WARPS);
  volatile int* abortFlag = reinterpret_cast<volatile int*>(tmemSlot + 1);

  const int warp = warpIndex(), lane = threadIdx.x & 31;
  if(threadIdx.x == 0) {
    for(int i = 0; i < MT_MAX_STAGES; i++) { mbarInit(smemU32(&bFull[i]), PLAIN ? MT_LOADERS : 1); mbarInit(smemU32(&bEmpty[i]), 1); }
    for(int i = 0; i < 2; i++) { mbarInit(smemU32(&bAcc[i]), 1); mbarInit(smemU32(&bTaken[i]), MT_EPI_WARPS); }
    for(int i = 0; i < MT_EPI_WARPS; i++) mbarInit(smemU32(&bRes[i]), 1);
    *abortFlag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fenceProxyAsync();
  }
  if(warp == 1) { tmemAlloc(smemU32(tmemSlot), a.tmemCols); tmemRelinquish(); }
  if(!PLAIN && warp == 0 && electOne()) { prefetchTensorMap(&tmX); prefetchTensorMap(&tmW); }
  tcFenceBefore();
  __syncthreads();
  tcFenceAfter();
  gridDepLaunch();
  gridDepWait();
  const uint32_t tmem = *tmemSlot;
  const int tiles = a.tilesM * a.tilesN;
  auto wait = [&](uint64_t* bar, uint32_t parity) { return opWait(smemU32(bar), parity, abortFlag, a.m.status, MT_ERR); };

  if(PLAIN && warp >= 2 + MT_EPI_WARPS) {
    const int loader = warp - 2 - MT_EPI_WARPS;
    auto run = [&](auto load) {
      bool ok = true;
      for(int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
        int tm, tn;
        mtTile(a, t, tm, tn);
        const PlainRows x = {(const uint16_t*)a.m.x, a.m.ldx, tm * MT_BM, a.m.M}, w = {(const uint16_t*)a.m.w, a.m.ldw, tn * a.BN, a.m.N};
        for(int k = 0; k < a.kSlices; k++) {
          const uint32_t s = load.it % a.stages, use = load.it / a.stages;
          if(use > 0) ok = wait(&bEmpty[s], (use - 1) & 1u);
          if(__any_sync(0xffffffffu, !ok)) { ok = false; break; }
          load.slice(smem + (size_t)s * slotBytes, x, w, a.BN, k);
        }
      }
      load.finish();
    };
    if(pairRows(a.m)) run(PlainLoader<16, true>{bFull, a.stages, a.m.K, loader, lane, 0});
    else run(PlainLoader<16, false>{bFull, a.stages, a.m.K, loader, lane, 0});
  }
  else if(warp == 0) {
    if(!PLAIN && electOne()) {
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
    const int quarter = warp & 3, group = (warp - 2) >> 2;  // TMEM lanes of this warp; it has every MT_GROUPS-th unit
    uint8_t* unit = sUnits + (warp - 2) * MT_UNIT_BYTES;
    uint8_t* resUnit = a.resAhead ? sUnits + (MT_EPI_WARPS + warp - 2) * MT_UNIT_BYTES : unit;
    uint64_t* res = bRes + (warp - 2);
    uint8_t* mine = unit + lane * 64;
    const int sw = (lane >> 1) & 3;  // the 16-byte pieces of a row lie permuted by its number
    const T* plainRes = a.tmaRes ? nullptr : (const T*)a.m.residual;
    const bool biasVec = ((uintptr_t)a.m.bias & 15) == 0;
    uint32_t n = 0, u = 0, asked = 0;  // tiles begun, units begun, residual units requested
    bool ok = true;
    for(int t = blockIdx.x; t < tiles && ok; t += gridDim.x, n++) {
      int tm, tn;
      mtTile(a, t, tm, tn);
      const int m0 = tm * MT_BM + quarter * 32, n0 = tn * a.BN;
      const uint32_t b = n & 1u;
      const int nUnits = a.m.M > m0 ? (min(a.BN, a.m.N - n0) + MT_UNIT - 1) / MT_UNIT : 0;  // units with anything in them
      auto requestResidual = [&](int c) {
        if(!a.resAhead) bulkWaitRead0();  // the unit before has left the slot
        mbarExpectTx(smemU32(res), (uint32_t)MT_UNIT_BYTES);
        tmaLoad2d(smemU32(resUnit), &tmR, n0 + c * MT_UNIT, m0, smemU32(res));
      };
      if(a.tmaRes && group < nUnits) {
        if(electOne()) requestResidual(group);
        asked++;
      }
      // (by TMA the longest sums that memory has room for take some 0.3 s, and the longer wait costs the others 2 %)
      ok = PLAIN ? opWaitSums(smemU32(&bAcc[b]), (n >> 1) & 1u, abortFlag, a.m.status, MT_ERR, a.kSlices) : wait(&bAcc[b], (n >> 1) & 1u);
      if(__any_sync(0xffffffffu, !ok)) ok = false;
      tcFenceAfter();
      for(int c = group; c < nUnits && ok; c += MT_GROUPS, u++) {
        const int nc = n0 + c * MT_UNIT;
        uint32_t r[32];
        __syncwarp();
        tmemLd32(tmem + b * (uint32_t)a.BN + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(c * MT_UNIT), r);
        tmemLdWaitFor(r);
        if(c + MT_GROUPS >= nUnits) {  // the accumulator has been read
          tcFenceBefore();
          __syncwarp();
          if(lane == 0) mbarArrive(smemU32(&bTaken[b]));
        }
        if(a.m.bias) {
          if(biasVec && nc + 32 <= a.m.N) {
#pragma unroll
            for(int q = 0; q < 8; q++) {
              const float4 v = *reinterpret_cast<const float4*>(a.m.bias + nc + 4 * q);
              r[4 * q] = __float_as_uint(__uint_as_float(r[4 * q]) + v.x);
              r[4 * q + 1] = __float_as_uint(__uint_as_float(r[4 * q + 1]) + v.y);
              r[4 * q + 2] = __float_as_uint(__uint_as_float(r[4 * q + 2]) + v.z);
              r[4 * q + 3] = __float_as_uint(__uint_as_float(r[4 * q + 3]) + v.w);
            }
          }
          else {
            const float v = nc + lane < a.m.N ? a.m.bias[nc + lane] : 0.0f;
#pragma unroll
            for(int j = 0; j < 32; j++) r[j] = __float_as_uint(__uint_as_float(r[j]) + __shfl_sync(0xffffffffu, v, j));
          }
        }
        switch(a.m.act) {
          case KB_ACT_RELU:
#pragma unroll
            for(int j = 0; j < 32; j++) r[j] = __float_as_uint(opFastAct(__uint_as_float(r[j]), KB_ACT_RELU));
            break;
          case KB_ACT_MISH:
#pragma unroll
            for(int j = 0; j < 32; j += 2) {
              float2 v = make_float2(__uint_as_float(r[j]), __uint_as_float(r[j + 1]));
              v = opFastMish(v, v);
              r[j] = __float_as_uint(v.x);
              r[j + 1] = __float_as_uint(v.y);
            }
            break;
          case KB_ACT_SILU:
#pragma unroll
            for(int j = 0; j < 32; j++) r[j] = __float_as_uint(opFastAct(__uint_as_float(r[j]), KB_ACT_SILU));
            break;
          case KB_ACT_MISH_SCALE8:
#pragma unroll
            for(int j = 0; j < 32; j += 2) {
              float2 v = make_float2(__uint_as_float(r[j]), __uint_as_float(r[j + 1]));
              v = opFastMish(v, make_float2(8.0f * v.x, 8.0f * v.y));
              r[j] = __float_as_uint(v.x);
              r[j + 1] = __float_as_uint(v.y);
            }
            break;
          default: break;
        }
        if(a.tmaOut && (!a.tmaRes || a.resAhead)) {
          if(electOne()) bulkWaitRead0();  // the unit before has left the slot
          __syncwarp();
        }
        if(a.tmaRes) {
          ok = wait(res, u & 1u);
          if(__any_sync(0xffffffffu, !ok)) { ok = false; break; }
        }
        else if(plainRes) {
          for(int i = 0; i < 32; i++) {
            T v = OpType<T>::from(0.0f);
            if(m0 + i < a.m.M && nc + lane < a.m.N) v = plainRes[(int64_t)(m0 + i) * a.m.ldr + nc + lane];
            *reinterpret_cast<T*>(unit + i * 64 + (((lane >> 3) ^ ((i >> 1) & 3)) << 4) + (lane & 7) * 2) = v;
          }
          __syncwarp();
        }
        if(a.m.residual) {
#pragma unroll
          for(int q = 0; q < 4; q++) {
            const uint4 old = *reinterpret_cast<const uint4*>(resUnit + lane * 64 + ((q ^ sw) << 4));
            const uint32_t o[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
            for(int e = 0; e < 4; e++) {
              const float2 f = opUnpack<T>(o[e]);
              r[8 * q + 2 * e] = __float_as_uint(__uint_as_float(r[8 * q + 2 * e]) + f.x);
              r[8 * q + 2 * e + 1] = __float_as_uint(__uint_as_float(r[8 * q + 2 * e + 1]) + f.y);
            }
          }
          if(a.resAhead && c + MT_GROUPS < nUnits) {
            __syncwarp();
            if(electOne()) requestResidual(c + MT_GROUPS);
            asked++;
          }
        }
#pragma unroll
        for(int q = 0; q < 4; q++) {
          uint4 w;
          w.x = opPack<T>(__uint_as_float(r[8 * q]), __uint_as_float(r[8 * q + 1]));
          w.y = opPack<T>(__uint_as_float(r[8 * q + 2]), __uint_as_float(r[8 * q + 3]));
          w.z = opPack<T>(__uint_as_float(r[8 * q + 4]), __uint_as_float(r[8 * q + 5]));
          w.w = opPack<T>(__uint_as_float(r[8 * q + 6]), __uint_as_float(r[8 * q + 7]));
          *reinterpret_cast<uint4*>(mine + ((q ^ sw) << 4)) = w;
        }
        if(a.tmaOut && (nc + MT_UNIT <= a.m.N || (a.m.N & 7) == 0)) {
          fenceProxyAsync();
          __syncwarp();
          if(electOne()) {
            tmaStore2d(&tmY, smemU32(unit), nc, m0);
            bulkCommit();
            if(a.tmaRes && !a.resAhead && c + MT_GROUPS < nUnits) requestResidual(c + MT_GROUPS);
          }
          if(a.tmaRes && !a.resAhead && c + MT_GROUPS < nUnits) asked++;
        }
        else {
          __syncwarp();
          for(int i = 0; i < 32; i++)
            if(m0 + i < a.m.M && nc + lane < a.m.N)
              ((T*)a.m.y)[(int64_t)(m0 + i) * a.m.ldy + nc + lane] = *reinterpret_cast<const T*>(unit + i * 64 + (((lane >> 3) ^ ((i >> 1) & 3)) << 4) + (lane & 7) * 2);
          __syncwarp();
        }
      }
      if(group >= nUnits && ok) {  // nothing of this accumulator is this warp's
        if(lane == 0) mbarArrive(smemU32(&bTaken[b]));
      }
    }
    if(!ok && asked > u) {  // a residual unit that is still on its way
      volatile int keepWaiting = 0;
      mbarWait(smemU32(res), u & 1u, &keepWaiting, 1000000ull);
    }
    if(a.tmaOut) bulkWaitAll();
  }
  tcFenceBefore();
  __syncthreads();
  if(warp == 1) { tcFenceAfter(); tmemDealloc(tmem, a.tmemCols); }
}

// ---------------------------------------------------------------------------------------------

constexpr int MS_THREADS = 320, MS_MAX_STAGES = 12, MS_ERR = 302;

struct MatmulSkinnyArgs {
  MatmulArgs m;
  int BN, kSlices, tilesX, split, stages;  // columns (rows of x) per tile, tiles of x rows, CTAs of a cluster
  uint32_t idesc, tmemCols;
};

template <typename T, bool PLAIN>
__global__ void __launch_bounds__(MS_THREADS, 2) matmulSkinnyKernel(
  const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const MatmulSkinnyArgs a) {
  extern __shared__ uint8_t smemRaw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smemRaw) + 1023) & ~(uintptr_t)1023);
  const int slotBytes = MT_A_BYTES + a.BN * MT_BK * 2;
  __shared__ uint64_t bFull[MS_MAX_STAGES], bEmpty[MS_MAX_STAGES], bAcc;
  __shared__ uint32_t tmemSlot;
  __shared__ int abortWord;
  volatile int* abortFlag = &abortWord;
  const int warp = warpIndex(), lane = threadIdx.x & 31;
  if(threadIdx.x == 0) {
    for(int i = 0; i < a.stages; i++) { mbarInit(smemU32(&bFull[i]), PLAIN ? MT_LOADERS : 1); mbarInit(smemU32(&bEmpty[i]), 1); }
    mbarInit(smemU32(&bAcc), 1);
    *abortFlag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fenceProxyAsync();
  }
  if(warp == 1) { tmemAlloc(smemU32(&tmemSlot), a.tmemCols); tmemRelinquish(); }
  if(!PLAIN && warp == 0 && electOne()) { prefetchTensorMap(&tmX); prefetchTensorMap(&tmW); }
  tcFenceBefore();
  __syncthreads();
  tcFenceAfter();
  gridDepLaunch();
  gridDepWait();
  const uint32_t tmem = tmemSlot;
  const int rank = a.split > 1 ? (int)clusterCtaRank() : 0;
  const int tile = blockIdx.x / a.split;
  const int m0 = (tile % a.tilesX) * a.BN, n0 = (tile / a.tilesX) * MT_BM;
  const int s0 = (int)((long long)rank * a.kSlices / a.split), s1 = (int)((long long)(rank + 1) * a.kSlices / a.split);
  auto wait = [&](uint64_t* bar, uint32_t parity) { return opWait(smemU32(bar), parity, abortFlag, a.m.status, MS_ERR); };

  if(PLAIN && warp >= 2) {
    auto run = [&](auto load) {
      const PlainRows w = {(const uint16_t*)a.m.w, a.m.ldw, n0, a.m.N}, x = {(const uint16_t*)a.m.x, a.m.ldx, m0, a.m.M};
      bool ok = true;
      for(int k = s0; k < s1; k++) {
        const uint32_t s = load.it % a.stages, use = load.it / a.stages;
        if(use > 0) ok = wait(&bEmpty[s], (use - 1) & 1u);
        if(__any_sync(0xffffffffu, !ok)) break;
        load.slice(smem + (size_t)s * slotBytes, w, x, a.BN, k);
      }
      load.finish();
    };
    if(pairRows(a.m)) run(PlainLoader<8, true>{bFull, a.stages, a.m.K, warp - 2, lane, 0});
    else run(PlainLoader<8, false>{bFull, a.stages, a.m.K, warp - 2, lane, 0});
  }
  else if(warp == 0) {
    if(!PLAIN && electOne()) {
      uint32_t it = 0;
      bool ok = true;
      for(int k = s0; k < s1; k++, it++) {
        const uint32_t s = it % a.stages, use = it / a.stages;
        if(use > 0 && !wait(&bEmpty[s], (use - 1) & 1u)) { ok = false; break; }
        uint8_t* slot = smem + (size_t)s * slotBytes;
        mbarExpectTx(smemU32(&bFull[s]), (uint32_t)slotBytes);
        tmaLoad2d(smemU32(slot), &tmW, k * MT_BK, n0, smemU32(&bFull[s]));
        tmaLoad2d(smemU32(slot + MT_A_BYTES), &tmX, k * MT_BK, m0, smemU32(&bFull[s]));
      }
      if(!ok) {
        volatile int keepWaiting = 0;
        for(uint32_t i = it > (uint32_t)a.stages ? it - a.stages : 0; i < it; i++) mbarWait(smemU32(&bFull[i % a.stages]), (i / a.stages) & 1u, &keepWaiting, 1000000ull);
      }
    }
    __syncwarp();
  }
  else if(warp == 1) {
    if(electOne()) {
      uint32_t it = 0;
      bool ok = true;
      for(int k = s0; k < s1; k++, it++) {
        const uint32_t s = it % a.stages;
        if(!wait(&bFull[s], (it / a.stages) & 1u)) { ok = false; break; }
        tcFenceAfter();
        const uint32_t aLo = opDescLo(smemU32(smem + (size_t)s * slotBytes)), bLo = opDescLo(smemU32(smem + (size_t)s * slotBytes + MT_A_BYTES));
#pragma unroll
        for(int j = 0; j < MT_BK / 16; j++) ummaLoHi(tmem, aLo + 2 * j, bLo + 2 * j, OP_DESC_HI, a.idesc, (it | j) != 0 ? 1u : 0u);
        ummaCommit(smemU32(&bEmpty[s]));
      }
      if(ok) ummaCommit(smemU32(&bAcc));
    }
    __syncwarp();
  }
  // sums [row of x][128 weight rows] of this CTA, over the slots: all of them have been multiplied
  float* sums = reinterpret_cast<float*>(smem);
  const int rows = min(a.BN, a.m.M - m0);
  bool ok = true;
  if(warp >= 2) {
    const int quarter = warp & 3, half = (warp - 2) >> 2;
    ok = opWaitSums(smemU32(&bAcc), 0, abortFlag, a.m.status, MS_ERR, s1 - s0);
    if(__any_sync(0xffffffffu, !ok)) ok = false;
    tcFenceAfter();
    for(int c = half * 16; c < rows && ok; c += 32) {
      uint32_t r[16];
      tmemLd16(tmem + ((uint32_t)(quarter * 32) << 16) + (uint32_t)c, r);
      tmemLdWaitFor(r);
#pragma unroll
      for(int j = 0; j < 16; j++)
        if(c + j < rows) sums[(c + j) * MT_BM + quarter * 32 + lane] = __uint_as_float(r[j]);
    }
    tcFenceBefore();
  }
  if(a.split > 1) clusterSync(); else __syncthreads();
  if(warp == 1) { tcFenceAfter(); tmemDealloc(tmem, a.tmemCols); }
  // four weight rows a thread, a row of x per warp; this CTA has every split-th group of rows
  const int n = n0 + lane * 4;
  const uint32_t mine = smemU32(sums) + (uint32_t)lane * 16u;
  const T* res = (const T*)a.m.residual;
  const bool wideStore = n + 3 < a.m.N && ((uintptr_t)a.m.y & 7) == 0 && (a.m.ldy & 3) == 0;
  const bool wideRes = n + 3 < a.m.N && ((uintptr_t)res & 7) == 0 && (a.m.ldr & 3) == 0;
  float bias[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  if(a.m.bias)
#pragma unroll
    for(int e = 0; e < 4; e++)
      if(n + e < a.m.N) bias[e] = a.m.bias[n + e];
#pragma unroll 2
  for(int r = rank + warp * a.split; r < rows; r += (MS_THREADS / 32) * a.split) {
    float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f), p[8];
    const int64_t at = (int64_t)(m0 + r);
    alignas(8) T old[4];
    if(res) {
      if(wideRes) *reinterpret_cast<uint2*>(old) = *reinterpret_cast<const uint2*>(res + at * a.m.ldr + n);
      else
#pragma unroll
        for(int e = 0; e < 4; e++)
          if(n + e < a.m.N) old[e] = res[at * a.m.ldr + n + e];
    }
    if(a.split == 1) v = *reinterpret_cast<const float4*>(sums + r * MT_BM + lane * 4);
    else {
#pragma unroll
      for(int s = 0; s < 8; s++)
        if(s < a.split) p[s] = ldCluster4(clusterMapAddr(mine + (uint32_t)r * (MT_BM * 4), (uint32_t)s));
#pragma unroll
      for(int s = 0; s < 8; s++)
        if(s < a.split) { v.x += p[s].x; v.y += p[s].y; v.z += p[s].z; v.w += p[s].w; }
    }
    float f[4] = {v.x, v.y, v.z, v.w};
    alignas(8) T out[4];
#pragma unroll
    for(int e = 0; e < 4; e++) {
      f[e] = opFastAct(f[e] + bias[e], a.m.act);
      if(res) f[e] += OpType<T>::to(old[e]);
      out[e] = OpType<T>::from(f[e]);
    }
    T* y = (T*)a.m.y + at * a.m.ldy + n;
    if(wideStore) *reinterpret_cast<uint2*>(y) = *reinterpret_cast<const uint2*>(out);
    else
#pragma unroll
      for(int e = 0; e < 4; e++)
        if(n + e < a.m.N) y[e] = out[e];
  }
  if(a.split > 1) clusterSync();  // nobody leaves while its sums are being read
}

bool encodeRows(CUtensorMap* map, int dt, const void* p, int64_t cols, int64_t rows, int64_t ld, int boxCols, int boxRows, CUtensorMapSwizzle sw) {
  if(rows == 1) ld = (cols + 7) / 8 * 8;  // nothing lies that far on
  const uint64_t dims[2] = {(uint64_t)cols, (uint64_t)rows}, strides[1] = {(uint64_t)ld * 2};
  const uint32_t box[2] = {(uint32_t)boxCols, (uint32_t)boxRows};
  return encodeTiled(map, dt, p, 2, dims, strides, box, sw);
}

bool rowsAligned(const void* p, int64_t ld) { return ((uintptr_t)p & 15) == 0 && ld % 8 == 0; }

template <typename T, bool PLAIN> cudaError_t launchWide(cudaStream_t st, const MatmulArgs& m) {
  MatmulTcArgs a = {};
  a.m = m;
  const int sms = smCount();
  a.tilesM = (m.M + MT_BM - 1) / MT_BM;
  a.kSlices = (m.K + MT_BK - 1) / MT_BK;
  // the width whose tiles cost the least in whole rounds; of equal ones the widest
  double best = 0;
  for(int bn = 256; bn >= 32; bn -= 32) {
    const double rounds = (double)(((long long)a.tilesM * ((m.N + bn - 1) / bn) + sms - 1) / sms);
    const double cost = rounds * std::max({44.0, bn / 2.0, (MT_BM + bn) * 32 / (PLAIN ? 23.0 : 75.0)});
    if(a.BN == 0 || cost < best) { best = cost; a.BN = bn; }
  }
  a.tilesN = (m.N + a.BN - 1) / a.BN;
  const int slotBytes = MT_A_BYTES + a.BN * MT_BK * 2;
  a.idesc = opIdesc<T>(MT_BM, a.BN);
  a.tmemCols = 32;
  while(a.tmemCols < 2u * a.BN) a.tmemCols *= 2;
  a.tmaOut = rowsAligned(m.y, m.ldy);
  a.tmaRes = a.tmaOut && m.residual && rowsAligned(m.residual, m.ldr);
  a.resAhead = a.tmaRes && a.kSlices < 16;  // ahead: a ring slot less for the products
  const size_t fixed = 16 * (a.resAhead ? 2 : 1) * MT_UNIT_BYTES + 1024 + 512;
  a.stages = (int)std::min<size_t>(MT_MAX_STAGES, (227 * 1024 - fixed) / slotBytes);
  CUtensorMap x = {}, w = {}, y = {}, r = {};
  bool ok = PLAIN || (encodeRows(&x, m.dt, m.x, m.K, m.M, m.ldx, MT_BK, MT_BM, CU_TENSOR_MAP_SWIZZLE_128B) &&
                      encodeRows(&w, m.dt, m.w, m.K, m.N, m.ldw, MT_BK, a.BN, CU_TENSOR_MAP_SWIZZLE_128B));
  if(a.tmaOut) ok = ok && encodeRows(&y, m.dt, m.y, m.N, m.M, m.ldy, MT_UNIT, 32, CU_TENSOR_MAP_SWIZZLE_64B);
  if(a.tmaRes) ok = ok && encodeRows(&r, m.dt, m.residual, m.N, m.M, m.ldr, MT_UNIT, 32, CU_TENSOR_MAP_SWIZZLE_64B);
  if(!ok) return cudaErrorInvalidValue;
  static SharedMemoryOptIn optIn;
  const cudaError_t e = optIn((const void*)matmulTcKernel<T, PLAIN>, 227 * 1024);
  if(e != cudaSuccess) return e;
  const int tiles = a.tilesM * a.tilesN;
  return launchDependent(matmulTcKernel<T, PLAIN>, dim3(std::min(tiles, sms)), dim3(MT_THREADS), (size_t)a.stages * slotBytes + fixed, st, x, w, y, r, a);
}

constexpr int MS_SMEM_TWO = 110 * 1024, MS_SMEM = 226 * 1024;  // of a CTA: two to an SM, one

// Whether the skinny form runs these sizes, and how.  Up to 128 rows of x: always (4096 x 4096 bf16, 128 rows: 13.1 us, 20.2 us in wide
// tiles).  More: where the wide tiles are one round at most and K is long enough to be worth cutting (300 x 512 x 4096: 8.5 us; but
// 361 x 1024 x 384: 8.1 us against 4.5 us in 96 wide tiles).  Rows without TMA, whose slices take longer, are worth cutting earlier
// (278 x 308 x 4706 bf16: 36 us, 213 us in wide tiles; 135 x 102 x 1442: 11 and 69; 16 x 181 x 236: 5.5 and 18).
bool skinnyShape(const MatmulArgs& m, bool plain, MatmulSkinnyArgs& a) {
  const int sms = smCount();
  a.kSlices = (m.K + MT_BK - 1) / MT_BK;
  const int tilesW = (m.N + MT_BM - 1) / MT_BM;
  const int parts = (m.M + 127) / 128;  // of the rows of x, in equal tiles
  a.BN = ((m.M + parts - 1) / parts + 15) / 16 * 16;
  a.tilesX = (m.M + a.BN - 1) / a.BN;
  const long long tiles = (long long)a.tilesX * tilesW;
  if(m.M > 128 ? tiles > sms || a.kSlices < (plain ? 8 : 32) : m.M > 16 && a.kSlices < (plain ? 4 : 16)) return false;
  a.split = 1;
  while(a.split < 8 && tiles * a.split * 2 <= 2 * sms && a.split * (plain ? 2 : 4) <= a.kSlices) a.split *= 2;
  return tiles * a.split < (1LL << 31);
}

template <typename T, bool PLAIN> cudaError_t launchSkinny(cudaStream_t st, MatmulSkinnyArgs a) {
  const MatmulArgs& m = a.m;
  const int slotBytes = MT_A_BYTES + a.BN * MT_BK * 2, sumBytes = a.BN * MT_BM * 4;
  a.stages = std::min({MS_MAX_STAGES, ((sumBytes + 1024 <= MS_SMEM_TWO ? MS_SMEM_TWO : MS_SMEM) - 1024) / slotBytes, (a.kSlices + a.split - 1) / a.split});
  a.idesc = opIdesc<T>(MT_BM, a.BN);
  a.tmemCols = 32;
  while(a.tmemCols < (uint32_t)a.BN) a.tmemCols *= 2;
  CUtensorMap x = {}, w = {};
  if(!PLAIN && (!encodeRows(&x, m.dt, m.x, m.K, m.M, m.ldx, MT_BK, a.BN, CU_TENSOR_MAP_SWIZZLE_128B) ||
     !encodeRows(&w, m.dt, m.w, m.K, m.N, m.ldw, MT_BK, MT_BM, CU_TENSOR_MAP_SWIZZLE_128B)))
    return cudaErrorInvalidValue;
  static SharedMemoryOptIn optIn;
  cudaError_t e = optIn((const void*)matmulSkinnyKernel<T, PLAIN>, MS_SMEM);
  if(e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(a.tilesX * ((m.N + MT_BM - 1) / MT_BM) * a.split));
  cfg.blockDim = dim3(MS_THREADS);
  cfg.dynamicSmemBytes = 1024 + (size_t)std::max(a.stages * slotBytes, sumBytes);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if(a.split > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)a.split; attr[n].val.clusterDim.y = 1; attr[n].val.clusterDim.z = 1;
    n++;
  }
  if(dependentLaunches()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    n++;
  }
  cfg.attrs = attr; cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, matmulSkinnyKernel<T, PLAIN>, x, w, a);
}

}  // namespace

bool matmulTcEligible(const MatmulArgs& a) {
  return (a.dt == DT_F16 || a.dt == DT_BF16) && ((long long)a.M + 127) / 128 * (((long long)a.N + 31) / 32) < (1LL << 31);
}
bool matmulTcAligned(const MatmulArgs& a) { return rowsAligned(a.x, a.ldx) && rowsAligned(a.w, a.ldw); }

cudaError_t launchMatmulTc(cudaStream_t st, const MatmulArgs& m) {
  const bool plain = !matmulTcAligned(m);
  MatmulSkinnyArgs a = {};
  a.m = m;
  if(skinnyShape(m, plain, a)) {
    if(plain) return m.dt == DT_F16 ? launchSkinny<__half, true>(st, a) : launchSkinny<__nv_bfloat16, true>(st, a);
    return m.dt == DT_F16 ? launchSkinny<__half, false>(st, a) : launchSkinny<__nv_bfloat16, false>(st, a);
  }
  if(plain) return m.dt == DT_F16 ? launchWide<__half, true>(st, m) : launchWide<__nv_bfloat16, true>(st, m);
  return m.dt == DT_F16 ? launchWide<__half, false>(st, m) : launchWide<__nv_bfloat16, false>(st, m);
}

}  // namespace kb

// Attention to states of another length on the tensor cores: fp16 / bf16, head sizes up to 128 in multiples of 8, rows on 16-byte
// boundaries.
//
// crossAttnTcKernel: a CTA takes one or two tiles of up to 128 rows (a key head's rows, kb_xattn.cu) and a range of keys, 128 at a
// time.  Two warpgroups do the softmax of one row tile each, a row per thread; of the third, warp 8 requests Q, K and V by TMA,
// warp 9 issues the MMAs, warps 10 and 11 make the keys of a tile that are not attended harmless.
//
//   S = Q K^T into 128 columns of tensor memory, the probabilities (16 bit, two per column) back into tensor memory, O = P V with P
//   read from there into 64 or 128 further columns.  With two row tiles the tensor pipe works on one while the other's warpgroup
//   does its exponentials.  With head size 64 the probabilities have columns of their own, and a row tile's next scores are
//   computed before its product; with 128 there is no room, they lie over the scores, and the next scores follow the product.
//   A block with one row tile gives the warpgroups every other tile of keys instead, and adds the two states at the end.
//
// p = 2^(scale log2(e) (s - ref)), where ref follows the row's maximum of s only when that has grown by more than 8 in the exponent (fp16: 4;
// sums and O in fp32 lose nothing): only then is O rescaled, which costs a round trip of O through registers and a wait
// for the product before.  The factor cancels in O / sum.  One multiply-add makes an exponent, from scale log2(e) ref rounded once.
// That rounding is half an fp32 step of such a score: at 4096 2^-12 of the exponent, at 10^9 64 of it.  So a warp with a reference
// above 4096 goes on with a loop that subtracts ref from the scores first (2 x 4096 x 8192 tokens: 1.23 ms, 0.51 with any smaller).
//
// Keys that are not attended (masked, or behind the last one) may hold anything.  In shared memory their rows of V are cleared and
// their rows of K are replaced by that of an attended key of the tile: so their scores are scores of the row that lie no higher
// than its maximum, their probabilities are finite and their products with V are 0.  Only the row's sum has to leave them out, which
// it does by a multiplication by 1 or 0 that it makes in place of an addition; the softmax has no comparison per score.
// (With a test of a bit per score in both passes: 341 us for 64 x 6 heads of 361 tokens over up to 2888 states, a fifth masked.)
// Rows of the tile that are no tokens are computed and not written.
//
// What bounds it: the softmax of a row tile, some 700 instructions of a warp per 128 keys with two warps to a scheduler, beside the MMAs
// (1024 cycles for the two products of 128 x 128 with head size 128, half of it with 64).  A step of both row tiles takes 3000
// cycles with head size 64 and 3200 with 128; the special-function units (16 exponentials per clock and SM, 2048 cycles) are the
// busiest part.  So one pair of exponentials in eight is computed on the FMA units (t = n + f with n whole and |f| <= 1/2, 2^f by a
// polynomial, n added to the exponent's bits): 2 x 4096 x 8192 tokens, 16 heads of 128, bf16: 520 us with none, 493 with one, 511 with
// two, 540 with three (in the first milliseconds; 514 us with one over seconds, at the power limit).  The polynomials are minimax fits of the relative error over [-1/2, 1/2] (Remez exchange): degree 3 is off by
// 7.5e-5 at most, for bf16 probabilities, whose rounding is 3.9e-3; degree 4 by 2.6e-6, for fp16 with 4.9e-4.
// What did not help: four threads' warps to a scheduler (a row by two threads, 70 us where this takes 57); an issuing warp per row tile.
//
// Blocks of the longest sequences come first, where the batch is ragged: else the last ones started may be the longest (64 x 6 heads of
// 361 tokens over up to 2888 states, fp16: 147 us, 160 us in the order of the batch).
#include "kb_kernels.cuh"
#include "kb_ops.h"
#include "kb_ops_dev.cuh"
#include "kb_xattn.cuh"

#include <algorithm>

namespace kb {

namespace {

constexpr int XT_THREADS = 384, XT_KEYS = 128, XT_ERR = 311;
constexpr int XT_HALF = 128 * 64 * 2;  // bytes of 128 rows x 64 channels
// Weights are 2^XT_UP times larger where they are fp16, and so are the sums that they cancel in: the largest are 2^15, those that
// are 2^-25 of the reference's still have all their bits.  (bf16 has the range of fp32.)
template <typename T> constexpr float XT_UP = std::is_same<T, __half>::value ? 11.0f : 0.0f;
template <typename T> constexpr float XT_GROW = std::is_same<T, __half>::value ? 4.0f : 8.0f;  // of the exponent, before the reference follows
constexpr float XT_FAR = 4096.0f;
enum { XT_ALL, XT_SOME, XT_NONE };
constexpr int XT_SORT = 128;  // sequences that a block ranks

struct CrossAttnTcArgs {
  CrossAttnArgs x;
  XaSplit sp;
  int G, tileTokens, tileRows, tilesPerBlock, longestFirst;
  unsigned singlesFrom;  // blocks from here on are the halves (one row tile each) of the last blocks
  int qUse[3], kUse[3], vUse[3];  // 0 where a tensor repeats along the batch / token / head dimension
};

// D: head size that K and V tiles are laid out for (64 or 128; both may be smaller)
template <int D> struct XtShape {
  static constexpr int HALVES = D / 64;
  static constexpr int TILE = HALVES * XT_HALF;          // bytes of 128 rows
  static constexpr int STAGES = D == 64 ? 4 : 2;         // tiles of K, and of V, in flight
  static constexpr bool APART = D == 64;                 // probabilities have columns of their own
  static constexpr uint32_t O_AT = 256, P_AT = APART ? 256 + 2 * D : 0, P_STEP = APART ? 64 : 128;
  static constexpr int SMEM = 2 * TILE + 2 * STAGES * TILE + STAGES * XT_KEYS * 4 + 4 * 128 * 4 + 1024 + 512;
};

__device__ __forceinline__ float max3Nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 64 columns of this thread's row, complete: load and wait in one statement, whose results are outputs only (naming the registers of
// an earlier load as in and out of the wait costs a copy of each).
__device__ __forceinline__ void tmemLd64Now(uint32_t taddr, uint32_t (&r)[64]) {
  asm volatile(
    "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\ttcgen05.wait::ld.sync.aligned;"
    : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63]) : "r"(taddr) : "memory");
}

// 2^t of two numbers up to 16 (above what a maximum may lag), below t = -112 as for -112: t = 128 u - 112 with u cut to [0, 1], which costs no more
// than 2^-18 of t.  A NaN does not survive it, neither one that was a score nor infinity - infinity: rows with a score that is NaN or
// +infinity get a reference of NaN, which the exponentials of the special-function units carry on, whichever key it was.
__device__ __forceinline__ float fmaSat(float a, float b, float c) {
  float d;
  asm("fma.rn.sat.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
template <typename T> __device__ __forceinline__ float2 ex2Poly(float2 u) {
  constexpr bool LONG = std::is_same<T, __half>::value;
  auto both = [](float c) { return make_float2(c, c); };
  // 1.5 * 2^23: the sum's low bits are the nearest whole number
  const float2 r = __ffma2_rn(u, both(128.0f), both(12582912.0f - 112.0f));
  const float2 n = __fadd2_rn(r, both(-(12582912.0f - 112.0f)));
  const float2 f = __ffma2_rn(u, both(128.0f), make_float2(-n.x, -n.y));
  float2 p;
  if(LONG) {
    p = __ffma2_rn(f, both(0.009570102207362652f), both(0.05591785907745361f));
    p = __ffma2_rn(f, p, both(0.240247443318367f));
    p = __ffma2_rn(f, p, both(0.6931217908859253f));
    p = __ffma2_rn(f, p, both(0.9999992847442627f));
  }
  else {
    p = __ffma2_rn(f, both(0.0551716685295105f), both(0.2426111251115799f));
    p = __ffma2_rn(f, p, both(0.6932609677314758f));
    p = __ffma2_rn(f, p, both(0.9999280571937561f));
  }
  return make_float2(__uint_as_float(__float_as_uint(p.x) + (__float_as_uint(r.x) << 23)), __uint_as_float(__float_as_uint(p.y) + (__float_as_uint(r.y) << 23)));
}
__device__ __forceinline__ void softmaxWarpgroupsSync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <typename T, int D>
__global__ void __launch_bounds__(XT_THREADS, 1) crossAttnTcKernel(
  const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const CrossAttnTcArgs a) {
  typedef XtShape<D> Sh;
  constexpr int ST = Sh::STAGES;
  extern __shared__ uint8_t smemRaw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smemRaw) + 1023) & ~(uintptr_t)1023);
  uint8_t* sQ = smem;                       // [2] row tiles
  uint8_t* sK = sQ + 2 * Sh::TILE;          // [ST]
  uint8_t* sV = sK + ST * Sh::TILE;         // [ST]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sV + ST * Sh::TILE);
  uint64_t* bQ = bars;                      // [2] a row tile has arrived
  uint64_t* bKFull = bQ + 2;                // [ST]
  uint64_t* bKEmpty = bKFull + ST;
  uint64_t* bVFull = bKEmpty + ST;
  uint64_t* bKReady = bVFull + ST;          // ... and rows of keys that are not attended are replaced
  uint64_t* bVReady = bKReady + ST;         // ... and cleared; sKind and sCount say which they are
  uint64_t* bVEmpty = bVReady + ST;
  uint64_t* bS = bVEmpty + ST;              // [2] scores are complete
  uint64_t* bRead = bS + 2;                 // [2] ... and have been read
  uint64_t* bP = bRead + 2;                 // [2][2] probabilities of the first, the second 64 keys are complete
  uint64_t* bO = bP + 4;                    // [2] their product with V is
  float* sCount = reinterpret_cast<float*>(bO + 2);   // [ST][128] 1 for an attended key, 0 for another
  float* sState = sCount + ST * XT_KEYS;              // [2][2][128] reference and sum of the rows, where their keys are cut in two
  int* sKind = reinterpret_cast<int*>(sState + 4 * 128);  // [ST] XT_ALL, XT_SOME or XT_NONE of a tile's keys are attended
  uint32_t* tmemSlot = reinterpret_cast<uint32_t*>(sKind + ST);
  volatile int* abortFlag = reinterpret_cast<volatile int*>(tmemSlot + 1);
  volatile int* sSeq = abortFlag + 1;                 // this block's sequence, where the sequences are ranked

  const CrossAttnArgs& x = a.x;
  const int warp = warpIndex(), lane = threadIdx.x & 31;
  if(threadIdx.x == 0) {
    for(int i = 0; i < 2; i++) { mbarInit(smemU32(&bQ[i]), 1); mbarInit(smemU32(&bS[i]), 1); mbarInit(smemU32(&bRead[i]), 4); mbarInit(smemU32(&bP[2 * i]), 4); mbarInit(smemU32(&bP[2 * i + 1]), 4); mbarInit(smemU32(&bO[i]), 1); }
    for(int i = 0; i < ST; i++) {
      mbarInit(smemU32(&bKFull[i]), 1); mbarInit(smemU32(&bKEmpty[i]), 1);
      mbarInit(smemU32(&bVFull[i]), 1); mbarInit(smemU32(&bKReady[i]), 1); mbarInit(smemU32(&bVReady[i]), 1); mbarInit(smemU32(&bVEmpty[i]), 1);
    }
    *abortFlag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fenceProxyAsync();
  }
  if(warp == 9) { tmemAlloc(smemU32(tmemSlot), 512); tmemRelinquish(); }
  tcFenceBefore();
  if(warp == 8 && electOne()) { prefetchTensorMap(&tmQ); prefetchTensorMap(&tmK); prefetchTensorMap(&tmV); }
  __syncthreads();
  tcFenceAfter();
  gridDepLaunch();
  gridDepWait();
  const uint32_t tmem = *tmemSlot;
  auto whichBlock = [&]() {
    const unsigned i = blockIdx.x, single = i >= a.singlesFrom ? i - a.singlesFrom : 0u;
    XaBlock b = xaBlock(x, a.sp, a.tileRows * a.tilesPerBlock, i >= a.singlesFrom ? a.singlesFrom + single / 2 : i);
    b.row0 += (int)(single & 1u) * a.tileRows;
    return b;
  };
  XaBlock blk = whichBlock();
  if(a.longestFirst) {
    // the sequence of this block's rank by length (ties by number): a thread counts for each how many come before it
    int* sLen = reinterpret_cast<int*>(sState);
    const int i = threadIdx.x;
    if(i < x.batch) sLen[i] = xaKeys(x, i);
    __syncthreads();
    if(i < x.batch) {
      const int mine = sLen[i];
      int before = 0;
      for(int j = 0; j < x.batch; j++) before += sLen[j] > mine || (sLen[j] == mine && j < i) ? 1 : 0;
      if(before == blk.b) *sSeq = i;
    }
    __syncthreads();
    blk.b = *sSeq;
  }
  const int rows = xaRows(x, blk.b, a.G), keys = xaKeys(x, blk.b);
  const int k0 = blk.part * a.sp.chunk, k1 = (int)min((long long)keys, (long long)k0 + a.sp.chunk);
  const bool idle = blk.row0 >= rows || (blk.part > 0 && k0 >= keys);  // part 0 reports a row without keys
  const int nKeys = idle ? 0 : max(0, k1 - k0), nT = (nKeys + XT_KEYS - 1) / XT_KEYS;
  const int nTiles = idle ? 0 : min(blockIdx.x >= a.singlesFrom ? 1 : a.tilesPerBlock, (rows - blk.row0 + a.tileRows - 1) / a.tileRows);
  const bool cut = nTiles == 1 && nT > 1;  // one row tile: warpgroup t has key tiles t, t + 2, ...
  const bool two = nTiles > 1 || cut;
  const int steps0 = cut ? (nT + 1) / 2 : nT, steps1 = cut ? nT / 2 : nT;
  auto keyTile = [&](int t, int i) { return cut ? 2 * i + t : i; };
  auto wait = [&](uint64_t* bar, uint32_t parity) { return opWaitInline(smemU32(bar), parity, abortFlag, x.status, XT_ERR); };

  if(warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
    const int qHalves = (x.dq + 63) / 64, vHalves = (x.dv + 63) / 64;
    if(warp == 8 && nT > 0) {
      // ---------------- requests ----------------
      if(electOne()) {
        const int b = blk.b, kvh = blk.kvh;
        auto loadRows = [&](uint8_t* dst, const CUtensorMap* map, const int* use, int h, int t, int halves, uint64_t* bar) {
          for(int i = 0; i < halves; i++) tmaLoad4d(smemU32(dst + i * XT_HALF), map, i * 64, h * use[2], t * use[1], b * use[0], smemU32(bar));
        };
        auto loadQ = [&](int t) {
          mbarExpectTx(smemU32(&bQ[t]), (uint32_t)(qHalves * a.tileRows * 128));
          loadRows(sQ + t * Sh::TILE, &tmQ, a.qUse, kvh * a.G, (blk.row0 + t * a.tileRows) / a.G, qHalves, &bQ[t]);
        };
        bool ok = true;
        int kAsked = 0, vAsked = 0;
        loadQ(0);
        for(int j = 0; j < nT && ok; j++) {
          const int s = j % ST;
          const uint32_t before = (uint32_t)(j / ST - 1) & 1u;
          if(j >= ST && !wait(&bKEmpty[s], before)) { ok = false; break; }
          mbarExpectTx(smemU32(&bKFull[s]), (uint32_t)(qHalves * XT_HALF));
          loadRows(sK + s * Sh::TILE, &tmK, a.kUse, kvh, k0 + j * XT_KEYS, qHalves, &bKFull[s]);
          kAsked++;
          if(j == 0 && nTiles > 1) loadQ(1);
          if(j >= ST && !wait(&bVEmpty[s], before)) { ok = false; break; }
          mbarExpectTx(smemU32(&bVFull[s]), (uint32_t)(vHalves * XT_HALF));
          loadRows(sV + s * Sh::TILE, &tmV, a.vUse, kvh, k0 + j * XT_KEYS, vHalves, &bVFull[s]);
          vAsked++;
        }
        if(!ok) {  // copies in flight land before the CTA may end
          volatile int keepWaiting = 0;
          for(int t = 0; t < nTiles; t++) mbarWait(smemU32(&bQ[t]), 0, &keepWaiting, 1000000ull);
          for(int j = max(0, kAsked - ST); j < kAsked; j++) mbarWait(smemU32(&bKFull[j % ST]), (uint32_t)(j / ST) & 1u, &keepWaiting, 1000000ull);
          for(int j = max(0, vAsked - ST); j < vAsked; j++) mbarWait(smemU32(&bVFull[j % ST]), (uint32_t)(j / ST) & 1u, &keepWaiting, 1000000ull);
        }
      }
      __syncwarp();
    }
    else if(warp == 9 && nT > 0) {
      // ---------------- MMAs ----------------
      if(electOne()) {
        const uint32_t idescS = opIdesc<T>(128, XT_KEYS), idescO = opIdesc<T>(128, D, true);
        const int qSteps = (x.dq + 15) / 16;
        // V is the MN-major operand: 64 channels per row of 128 bytes, 8 keys 1024 bytes apart, the second 64 channels XT_HALF on
        auto vDescLo = [](uint32_t saddr) { return ((saddr & 0x3FFFFu) >> 4) | ((uint32_t)(XT_HALF >> 4) << 16); };
        auto scores = [&](int t, int i) {
          const int j = keyTile(t, i);
          const uint32_t q = smemU32(sQ + (cut ? 0 : t) * Sh::TILE), k = smemU32(sK + (j % ST) * Sh::TILE);
#pragma unroll
          for(int d = 0; d < D / 16; d++)
            if(d < qSteps)
              ummaLoHi(tmem + t * 128u, opDescLo(q + (d / 4) * XT_HALF) + 2 * (d & 3), opDescLo(k + (d / 4) * XT_HALF) + 2 * (d & 3), OP_DESC_HI, idescS, d > 0 ? 1u : 0u);
          ummaCommit(smemU32(&bS[t]));
          if(cut || t == 1 || !two) ummaCommit(smemU32(&bKEmpty[j % ST]));
        };
        auto product = [&](int t, int i) {  // false: a wait ran out
          const int j = keyTile(t, i);
          if(!wait(&bVReady[j % ST], (uint32_t)(j / ST) & 1u)) return false;
          const uint32_t v = vDescLo(smemU32(sV + (j % ST) * Sh::TILE));
#pragma unroll
          for(int h = 0; h < 2; h++) {
            if(!wait(&bP[2 * t + h], (uint32_t)i & 1u)) return false;
            tcFenceAfter();
#pragma unroll
            for(int k = 4 * h; k < 4 * h + 4; k++)
              ummaTmemA(tmem + Sh::O_AT + t * D, tmem + Sh::P_AT + t * Sh::P_STEP + 8u * k, v + 128u * k, OP_DESC_HI, idescO, (i > 0 || k > 0) ? 1u : 0u);
          }
          ummaCommit(smemU32(&bO[t]));
          if(cut || t == 1 || !two) ummaCommit(smemU32(&bVEmpty[j % ST]));
          return true;
        };
        auto nextScores = [&](int t, int i) {
          const int j = keyTile(t, i);
          if(!wait(&bKReady[j % ST], (uint32_t)(j / ST) & 1u)) return false;
          if(Sh::APART && i > 0 && !wait(&bRead[t], (uint32_t)(i - 1) & 1u)) return false;
          tcFenceAfter();
          scores(t, i);
          return true;
        };
        // Where the probabilities have columns of their own the next scores come before the product: the softmax never waits.
        // Where they lie over the scores the next scores follow the product that reads them.
        bool ok = wait(&bQ[0], 0) && nextScores(0, 0);
        ok = ok && (!two || ((cut || wait(&bQ[1], 0)) && nextScores(1, 0)));
        for(int i = 0; i < steps0 && ok; i++)
          for(int t = 0; t < (two ? 2 : 1) && ok; t++) {
            const int steps = t == 0 ? steps0 : steps1;
            if(i >= steps) break;
            if(Sh::APART && i + 1 < steps) ok = nextScores(t, i + 1);
            ok = ok && product(t, i);
            if(!Sh::APART && i + 1 < steps) ok = ok && nextScores(t, i + 1);
          }
      }
      __syncwarp();
    }
    else if(nT > 0) {
      // ---------------- keys that are not attended: warp 10 clears V, warp 11 replaces K ----------------
      const bool forV = warp == 10;
      const int halves = forV ? vHalves : qHalves;
      uint8_t* tiles = forV ? sV : sK;
      uint64_t *full = forV ? bVFull : bKFull, *ready = forV ? bVReady : bKReady;
      float mask[4];
      auto fetch = [&](int j) {  // the masks of a tile, a tile ahead
#pragma unroll
        for(int i = 0; i < 4; i++) {
          const int key = k0 + j * XT_KEYS + i * 32 + lane;
          mask[i] = key < k1 ? (x.keyMask ? x.keyMask[(int64_t)blk.b * x.kLen + key] : 1.0f) : 0.0f;
        }
      };
      fetch(0);
      for(int j = 0; j < nT; j++) {
        const int s = j % ST;
        uint32_t bits[4];
#pragma unroll
        for(int i = 0; i < 4; i++) bits[i] = __ballot_sync(0xffffffffu, mask[i] != 0.0f);
        const bool all = (bits[0] & bits[1] & bits[2] & bits[3]) == 0xffffffffu, none = (bits[0] | bits[1] | bits[2] | bits[3]) == 0u;
        const float count[4] = {mask[0] != 0.0f ? 1.0f : 0.0f, mask[1] != 0.0f ? 1.0f : 0.0f, mask[2] != 0.0f ? 1.0f : 0.0f, mask[3] != 0.0f ? 1.0f : 0.0f};
        if(j + 1 < nT) fetch(j + 1);
        if(__any_sync(0xffffffffu, !wait(&full[s], (uint32_t)(j / ST) & 1u))) break;
        if(forV) {  // the slot's readers are done with it as long as its V is free
          if(lane == 0) sKind[s] = all ? XT_ALL : (none ? XT_NONE : XT_SOME);
          if(!all)
#pragma unroll
            for(int i = 0; i < 4; i++) sCount[s * XT_KEYS + i * 32 + lane] = count[i];
        }
        if(!all && (forV || !none)) {
          const int like = bits[0] ? __ffs(bits[0]) - 1 : (bits[1] ? 31 + __ffs(bits[1]) : (bits[2] ? 63 + __ffs(bits[2]) : 95 + __ffs(bits[3])));
          // a row of 64 channels is 128 bytes, its 16-byte pieces permuted by the row's number: eight lanes write one
          for(int h = 0; h < halves; h++) {
            uint8_t* tile = tiles + s * Sh::TILE + h * XT_HALF;
            uint4 w = make_uint4(0u, 0u, 0u, 0u);
            if(!forV) w = *reinterpret_cast<const uint4*>(tile + like * 128 + (((lane & 7) ^ (like & 7)) << 4));
#pragma unroll
            for(int i = 0; i < XT_KEYS; i += 4) {
              const int r = i + (lane >> 3);
              if(((bits[i / 32] >> (r & 31)) & 1u) == 0u) *reinterpret_cast<uint4*>(tile + r * 128 + (((lane & 7) ^ (r & 7)) << 4)) = w;
            }
          }
          fenceProxyAsync();
        }
        __syncwarp();
        if(lane == 0) mbarArrive(smemU32(&ready[s]));
      }
    }
  }
  else {
    // ---------------- softmax: warpgroup t has row tile t, thread i of it row i ----------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    const int t = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    if(t < nTiles || cut) {
      const int steps = t == 0 ? steps0 : steps1;
      const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
      const uint32_t tS = tmem + t * 128u + lanes, tO = tmem + Sh::O_AT + t * D + lanes, tP = tmem + Sh::P_AT + t * Sh::P_STEP + lanes;
      const float c = x.scale * 1.4426950408889634f;
      const float2 c2 = make_float2(c, c);
      const float cu = c * 0.0078125f;
      float ref = -INFINITY, base = 0.0f, sum = 0.0f;
      bool far = false, ok = true;  // far: one of this warp's references is above XT_FAR
      auto grown = [&](float now) { return row < a.tileRows && ((now - ref) * c > XT_GROW<T> || now != now); };
      auto rescale = [&](int i, float now, bool grow) {  // the rows of this warp whose maximum has grown: false if a wait ran out
        float keep = 1.0f;
        if(grow) {
          keep = exp2f((ref - now) * c);
          ref = now == INFINITY ? __int_as_float(0x7fffffff) : now;
          sum *= keep;
        }
        if(i == 0) return true;
        const bool there = wait(&bO[t], (uint32_t)(i - 1) & 1u);
        if(__any_sync(0xffffffffu, !there)) return false;
        tcFenceAfter();
#pragma unroll
        for(int d = 0; d < D; d += 16) {
          uint32_t o[16];
          tmemLd16(tO + d, o);
          tmemLdWaitFor(o);
#pragma unroll
          for(int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
          tmemSt16(tO + d, o);
        }
        return true;
      };
      for(int i = 0; i < steps; i++) {
        const int j = keyTile(t, i);
        ok = wait(&bVReady[j % ST], (uint32_t)(j / ST) & 1u) && wait(&bS[t], (uint32_t)i & 1u);
        if(__any_sync(0xffffffffu, !ok)) { ok = false; break; }
        tcFenceAfter();
        const int kind = sKind[j % ST];
        uint32_t s[2][64];
        if(!far) {
          tmemLd64Now(tS, s[0]);
          tmemLd64Now(tS + 64u, s[1]);
          float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for(int k = 0; k < 2; k++)
#pragma unroll
            for(int e = 0; e < 64; e += 2) top[(e / 2) & 3] = max3Nan(top[(e / 2) & 3], __uint_as_float(s[k][e]), __uint_as_float(s[k][e + 1]));
          const float now = kind == XT_NONE ? -INFINITY : max3Nan(max3Nan(top[0], top[1], top[2]), top[3], top[3]);
          const bool grow = grown(now);
          if(__any_sync(0xffffffffu, grow)) {
            far = __any_sync(0xffffffffu, grow && fabsf(now * c) > XT_FAR);
            if(!far) {
              ok = rescale(i, now, grow);
              if(!ok) break;
              base = ref == -INFINITY ? 0.0f : XT_UP<T> - ref * c;
            }
          }
        }
        if(far) {
          // the same with the reference subtracted from each score, in little code: unrolled like the other it costs that one's time (head
          // size 64, 31 %; a warp that has come here stays)
          float now = -INFINITY;
#pragma unroll 1
          for(uint32_t d = 0; d < 128u && kind != XT_NONE; d += 16u) {
            uint32_t o[16];
            tmemLd16(tS + d, o);
            tmemLdWaitFor(o);
#pragma unroll
            for(int e = 0; e < 16; e += 2) now = max3Nan(now, __uint_as_float(o[e]), __uint_as_float(o[e + 1]));
          }
          const bool grow = grown(now);
          if(i > 0) {
            ok = wait(&bO[t], (uint32_t)(i - 1) & 1u);
            if(__any_sync(0xffffffffu, !ok)) { ok = false; break; }
            tcFenceAfter();
          }
          if(__any_sync(0xffffffffu, grow)) {
            const float keep = grow ? exp2f((ref - now) * c) : 1.0f;
            if(grow) { ref = now == INFINITY ? __int_as_float(0x7fffffff) : now; sum *= keep; }
#pragma unroll 1
            for(uint32_t d = 0; d < (uint32_t)D && i > 0; d += 16u) {
              uint32_t o[16];
              tmemLd16(tO + d, o);
              tmemLdWaitFor(o);
#pragma unroll
              for(int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
              tmemSt16(tO + d, o);
            }
          }
          const float from = ref == -INFINITY ? 0.0f : ref;
#pragma unroll 1
          for(uint32_t k = 0; k < 4u; k++) {
            uint32_t o[2][16], p[16];
            tmemLd16(tS + 32u * k, o[0]);
            tmemLd16(tS + 32u * k + 16u, o[1]);
            tmemLdWaitFor(o[0]);
            tmemLdWaitFor(o[1]);
#pragma unroll
            for(int e = 0; e < 16; e++) {
              const float* count = sCount + (j % ST) * XT_KEYS + 32 * k + 2 * e;
              const float w0 = kind == XT_NONE ? 0.0f : ex2Approx(fmaf(__uint_as_float(o[e >> 3][2 * (e & 7)]) - from, c, XT_UP<T>));
              const float w1 = kind == XT_NONE ? 0.0f : ex2Approx(fmaf(__uint_as_float(o[e >> 3][2 * (e & 7) + 1]) - from, c, XT_UP<T>));
              sum += kind == XT_SOME ? w0 * count[0] + w1 * count[1] : w0 + w1;
              p[e] = opPack<T>(w0, w1);
            }
            tmemSt16(tP + 16u * k, p);
            if(k & 1u) {
              tmemStWait();
              tcFenceBefore();
              __syncwarp();
              if(lane == 0) mbarArrive(smemU32(&bP[2 * t + (k >> 1)]));
            }
          }
          if(Sh::APART) {
            __syncwarp();
            if(lane == 0) mbarArrive(smemU32(&bRead[t]));
          }
          continue;
        }
        if(Sh::APART) {  // the next scores may come
          tcFenceBefore();
          __syncwarp();
          if(lane == 0) mbarArrive(smemU32(&bRead[t]));
        }
        const float2 base2 = make_float2(base, base);
        const float baseU = fmaf(base, 0.0078125f, 0.875f);  // (t + 112) / 128 lies in [0, 1] as far as t <= 16
        float2 part[2] = {make_float2(0.0f, 0.0f), make_float2(0.0f, 0.0f)};
        if(Sh::APART && i > 0) {  // the product before has read the probabilities that these replace
          ok = wait(&bO[t], (uint32_t)(i - 1) & 1u);
          if(__any_sync(0xffffffffu, !ok)) { ok = false; break; }
          tcFenceAfter();
        }
        auto exponentials = [&](auto some) {  // some: not every key counts
          const float2* count = reinterpret_cast<const float2*>(sCount + (j % ST) * XT_KEYS);
#pragma unroll
          for(int k = 0; k < 4; k++) {
            uint32_t p[16];
#pragma unroll
            for(int e = 0; e < 16; e++) {
              const float s0 = __uint_as_float(s[k >> 1][(k & 1) * 32 + 2 * e]), s1 = __uint_as_float(s[k >> 1][(k & 1) * 32 + 2 * e + 1]);
              float2 w;
              if((e & 7) == 3) w = ex2Poly<T>(make_float2(fmaSat(s0, cu, baseU), fmaSat(s1, cu, baseU)));
              else {
                const float2 v = __ffma2_rn(make_float2(s0, s1), c2, base2);
                w = make_float2(ex2Approx(v.x), ex2Approx(v.y));
              }
              part[e & 1] = decltype(some)::value ? __ffma2_rn(w, count[k * 16 + e], part[e & 1]) : __fadd2_rn(part[e & 1], w);
              p[e] = opPack<T>(w.x, w.y);
            }
            tmemSt16(tP + 16u * k, p);
            if(k & 1) {
              tmemStWait();
              tcFenceBefore();
              __syncwarp();
              if(lane == 0) mbarArrive(smemU32(&bP[2 * t + (k >> 1)]));
            }
          }
        };
        if(kind == XT_ALL) exponentials(std::false_type());
        else if(kind == XT_SOME) exponentials(std::true_type());
        else {
          uint32_t p[16];
#pragma unroll
          for(int e = 0; e < 16; e++) p[e] = 0u;
#pragma unroll
          for(int k = 0; k < 4; k++) tmemSt16(tP + 16u * k, p);
          tmemStWait();
          tcFenceBefore();
          __syncwarp();
          if(lane == 0) { mbarArrive(smemU32(&bP[2 * t])); mbarArrive(smemU32(&bP[2 * t + 1])); }
        }
        sum += (part[0].x + part[0].y) + (part[1].x + part[1].y);
      }
      float w0 = 1.0f, w1 = 0.0f;  // of the products of the two warpgroups
      const uint32_t tO0 = cut ? tmem + Sh::O_AT + lanes : tO, tO1 = tmem + Sh::O_AT + D + lanes;
      if(cut) {
        sState[t * 256 + row] = ref;
        sState[t * 256 + 128 + row] = sum;
        softmaxWarpgroupsSync();
        const float r0 = sState[row], r1 = sState[256 + row];
        ref = max3Nan(r0, r1, r1);  // a NaN is seen even if the other warpgroup had no key
        const float from = ref == -INFINITY ? 0.0f : ref;
        w0 = exp2f((r0 - from) * c);
        w1 = exp2f((r1 - from) * c);
        sum = w0 * sState[128 + row] + w1 * sState[384 + row];
        ok = ok && wait(&bO[0], (uint32_t)(steps0 - 1) & 1u) && wait(&bO[1], (uint32_t)(steps1 - 1) & 1u);
      }
      else if(nT > 0) ok = ok && wait(&bO[t], (uint32_t)(nT - 1) & 1u);
      if(__any_sync(0xffffffffu, !ok)) ok = false;
      tcFenceAfter();
      // what the loop does not need is found again instead of kept
      XaBlock blk = whichBlock();
      if(a.longestFirst) blk.b = *sSeq;
      const int rows = xaRows(x, blk.b, a.G);
      const int r = blk.row0 + (cut ? 0 : t) * a.tileRows + row;
      const bool mine = ok && row < a.tileRows && r < rows;
      const int token = r / a.G, head = blk.kvh * a.G + r - token * a.G;
      const bool live = ref != -INFINITY && sum != 0.0f && (!x.queryMask || (mine && x.queryMask[(int64_t)blk.b * x.qLen + token] != 0.0f));
      const float inv = live ? 1.0f / sum : 0.0f;
      float* part = a.sp.parts > 1 && mine ? xaPart(x, a.sp, blk, r, a.G) : nullptr;
      T* out = (T*)x.out + blk.b * x.oB + token * x.oT + head * x.oH;
      if(part && (t == 0 || !cut)) { part[0] = ref * c; part[1] = sum; }
#pragma unroll
      for(int dd = 0; dd < D; dd += 16) {
        if(cut && dd >= D / 2) break;
        const int d = cut ? t * (D / 2) + dd : dd;  // cut: each warpgroup writes half of the channels
        if(d >= x.dv) break;
        uint32_t o[16];
        if(nT > 0) {
          __syncwarp();
          tmemLd16(tO0 + d, o);
          tmemLdWaitFor(o);
          if(cut) {
            uint32_t o1[16];
            tmemLd16(tO1 + d, o1);
            tmemLdWaitFor(o1);
#pragma unroll
            for(int e = 0; e < 16; e++) o[e] = __float_as_uint(__uint_as_float(o[e]) * w0 + __uint_as_float(o1[e]) * w1);
          }
        }
        else {
#pragma unroll
          for(int e = 0; e < 16; e++) o[e] = 0u;
        }
        if(!mine) continue;
        if(part) {
#pragma unroll
          for(int e = 0; e < 16; e += 2)
            if(d + e < x.dv) *reinterpret_cast<float2*>(part + 2 + d + e) = make_float2(__uint_as_float(o[e]), __uint_as_float(o[e + 1]));
        }
        else {
#pragma unroll
          for(int e = 0; e < 16; e += 8)
            if(d + e < x.dv) {
              uint4 w = make_uint4(0u, 0u, 0u, 0u);
              if(live) {
                w.x = opPack<T>(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv);
                w.y = opPack<T>(__uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
                w.z = opPack<T>(__uint_as_float(o[e + 4]) * inv, __uint_as_float(o[e + 5]) * inv);
                w.w = opPack<T>(__uint_as_float(o[e + 6]) * inv, __uint_as_float(o[e + 7]) * inv);
              }
              *reinterpret_cast<uint4*>(out + d + e) = w;
            }
        }
      }
    }
  }
  tcFenceBefore();
  __syncthreads();
  if(warp == 9) { tcFenceAfter(); tmemDealloc(tmem, 512); }
}

// Dimensions channel, head, token, sequence; one that repeats (stride 0) is given once.
bool encodeView(CUtensorMap* map, int* use, int dt, const void* p, int d, int heads, int tokens, int batch, int64_t sH, int64_t sT, int64_t sB, int boxHeads, int boxTokens) {
  const int n[3] = {batch, tokens, heads};
  const int64_t s[3] = {sB, sT, sH};
  uint64_t dims[4] = {(uint64_t)d, 1, 1, 1}, strides[3];
  for(int i = 0; i < 3; i++) {  // map dimension 3 - i
    use[i] = n[i] == 1 || s[i] != 0;
    dims[3 - i] = use[i] ? (uint64_t)n[i] : 1;
    strides[2 - i] = n[i] > 1 && s[i] != 0 ? (uint64_t)s[i] * 2 : 16;
  }
  const uint32_t box[4] = {64, (uint32_t)boxHeads, (uint32_t)boxTokens, 1};
  return encodeTiled(map, dt, p, 4, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <typename T, int D> cudaError_t launchTc(cudaStream_t st, const CrossAttnTcArgs& given) {
  CrossAttnTcArgs a = given;
  const CrossAttnArgs& x = a.x;
  CUtensorMap q, k, v;
  if(!encodeView(&q, a.qUse, x.dt, x.q, x.dq, x.heads, x.qLen, x.batch, x.qH, x.qT, x.qB, a.G, a.tileTokens)) return cudaErrorInvalidValue;
  const int kLen = std::max(1, x.kLen);
  if(!encodeView(&k, a.kUse, x.dt, x.kLen ? x.k : x.q, x.dq, x.kvHeads, kLen, x.batch, x.kH, x.kT, x.kB, 1, XT_KEYS)) return cudaErrorInvalidValue;
  if(!encodeView(&v, a.vUse, x.dt, x.kLen ? x.v : x.q, x.dv, x.kvHeads, kLen, x.batch, x.vH, x.vT, x.vB, 1, XT_KEYS)) return cudaErrorInvalidValue;
  static SharedMemoryOptIn optIn;
  const cudaError_t e = optIn((const void*)crossAttnTcKernel<T, D>, XtShape<D>::SMEM);
  if(e != cudaSuccess) return e;
  return launchDependent(crossAttnTcKernel<T, D>, dim3(a.sp.blocks), dim3(XT_THREADS), (size_t)XtShape<D>::SMEM, st, q, k, v, a);
}

}  // namespace

bool crossAttnTcSizes(int dt, int heads, int kvHeads, int dq, int dv) {
  return (dt == DT_F16 || dt == DT_BF16) && dq % 8 == 0 && dv % 8 == 0 && dq <= 128 && dv <= 128 && heads / kvHeads <= 128;
}

// Row tiles of a block: two where the blocks still fill the GPU, so that the tensor pipe has one while the other is in its softmax.
XaSplit crossAttnTcSplit(int batch, int qLen, int kLen, int heads, int kvHeads, int dv, int* tilesPerBlock) {
  const int G = heads / kvHeads, tileRows = 128 / G * G;
  const long long rows = (long long)qLen * G, pairs = (rows + 2 * tileRows - 1) / (2 * tileRows) * batch * kvHeads;
  *tilesPerBlock = rows > tileRows && pairs >= smCount() ? 2 : 1;
  return xaPlanSplit(tileRows * *tilesPerBlock, XT_KEYS, pairs >= smCount() ? INT32_MAX : 1024, 1, batch, qLen, kLen, heads, kvHeads, dv);
}

cudaError_t launchCrossAttnTc(cudaStream_t st, const CrossAttnArgs& x, const XaSplit& sp, int tilesPerBlock) {
  CrossAttnTcArgs a = {};
  a.x = x;
  a.sp = sp;
  a.G = x.heads / x.kvHeads;
  a.tileTokens = 128 / a.G;
  a.tileRows = a.tileTokens * a.G;
  a.tilesPerBlock = tilesPerBlock;
  a.longestFirst = x.kLengths && x.batch > 1 && x.batch <= XT_SORT && sp.blocks > (unsigned)smCount();
  // Where the blocks of the last round are no more than half of the SMs, their row tiles go to an SM each, which halves that round
  // (2 x 4096 tokens, 16 heads of 128: 512 blocks on 148 SMs, 505 us in four rounds).  Not where a result must not depend on the batch.
  const unsigned sms = (unsigned)smCount(), last = sp.blocks % sms;
  const bool halves = tilesPerBlock == 2 && sp.parts == 1 && x.planBatch == 0 && sp.blocks > sms && last > 0 && 2 * last <= sms;
  a.singlesFrom = halves ? sp.blocks - last : UINT32_MAX;
  if(halves) a.sp.blocks += last;
  const bool wide = x.dq > 64 || x.dv > 64;
  if(x.dt == DT_F16) return wide ? launchTc<__half, 128>(st, a) : launchTc<__half, 64>(st, a);
  return wide ? launchTc<__nv_bfloat16, 128>(st, a) : launchTc<__nv_bfloat16, 64>(st, a);
}

}  // namespace kb

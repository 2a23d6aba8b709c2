// Attention to states of another length on a caller's own tensors: the CUDA-core kernel for every type, head size up to 256
// and alignment, and the kernel that joins the parts of rows whose keys were cut over several blocks.
//
// The rows of a key head are its query heads' rows side by side: row r = token r / G, head kvHead * G + r % G with G = heads /
// kvHeads, so that grouped heads read K and V once.  A block takes 64 such rows (16 where there are no more) and a range of keys, 64 at a time: scores into
// registers (4 x 4 or 1 x 4 per thread), a running maximum and sum per row, probabilities through shared memory, output accumulators in
// registers.  All in fp32.  Keys behind a sequence's length and masked keys are not read: their rows of K and V are zeros
// in shared memory, so that nothing in them (NaN, Inf) reaches a product.  fp32 rows of whole vectors are copied asynchronously, the next
// tile's under this one's products (16 x 361 tokens and states, 6 heads of 64: 117 us, 133 us through registers).
// Of the last tile only the sixteens of keys that it has are multiplied (60 x 413 tokens over 5 keys, 32 / 4 heads of 48 and 64: 297 us, 473 us with whole tiles; long sequences are the same
// to 5 % slower; leaving them out of the copies and exponentials as well gives another 5 % there and costs long ones 10 %).
//
// A row's state is (maximum, sum, unnormalised output).  Where few rows have many keys the keys are cut into parts of `chunk`
// keys, one block each; a part writes its state to the workspace and crossAttnJoinKernel adds the parts in order (crossAttnJoinManyKernel
// where there are many rows).
#include "kb_kernels.cuh"
#include "kb_ops.h"
#include "kb_ops_dev.cuh"
#include "kb_xattn.cuh"

#include <algorithm>

namespace kb {

namespace {

constexpr int XS_KEYS = 64, XS_THREADS = 256;

__host__ __device__ constexpr int xsPitch(int d) { return (d + 3) / 4 * 4 + 4; }
size_t xsSmem(int rows, int dq, int dv) { return sizeof(float) * (size_t)((rows + XS_KEYS) * xsPitch(dq) + XS_KEYS * xsPitch(dv) + rows * (XS_KEYS + 4)) + 2 * XS_KEYS; }

// Copies ROWS rows of d channels to fp32 rows of `pitch` in shared memory, zeros behind the last channel and for rows that
// `row` gives no address for.  Eight lanes per row and four channels per lane, with several rows' loads in flight.
template <typename T, int ROWS, bool VEC, class Row> __device__ __forceinline__ void xsStage(float* dst, int pitch, int d, Row row) {
  constexpr int PASSES = (ROWS + XS_THREADS / 8 - 1) / (XS_THREADS / 8);
  const int lane8 = threadIdx.x & 7, first = threadIdx.x >> 3;
  const T* from[PASSES];
#pragma unroll
  for(int p = 0; p < PASSES; p++) {
    const int r = first + p * (XS_THREADS / 8);
    from[p] = r < ROWS ? row(r) : nullptr;
  }
  for(int c = lane8 * 4; c < pitch - 4; c += 32) {
    float4 v[PASSES];
#pragma unroll
    for(int p = 0; p < PASSES; p++) {
      v[p] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if(!from[p]) continue;
      if(VEC) {  // d is a multiple of 4
        OpVec<T, 4> w;
        w.load(from[p] + c);
        v[p] = make_float4(OpType<T>::to(w.e[0]), OpType<T>::to(w.e[1]), OpType<T>::to(w.e[2]), OpType<T>::to(w.e[3]));
      }
      else {
        if(c < d) v[p].x = OpType<T>::to(from[p][c]);
        if(c + 1 < d) v[p].y = OpType<T>::to(from[p][c + 1]);
        if(c + 2 < d) v[p].z = OpType<T>::to(from[p][c + 2]);
        if(c + 3 < d) v[p].w = OpType<T>::to(from[p][c + 3]);
      }
    }
#pragma unroll
    for(int p = 0; p < PASSES; p++) {
      const int r = first + p * (XS_THREADS / 8);
      if(r < ROWS) *reinterpret_cast<float4*>(dst + r * pitch + c) = v[p];
    }
  }
}

// The same without registers in between, for fp32 rows of whole vectors: asynchronous copies, zeros for rows without an address.
template <int ROWS, class Row> __device__ __forceinline__ void xsStageAsync(float* dst, int pitch, const float* anywhere, Row row) {
  const int lane8 = threadIdx.x & 7;
#pragma unroll
  for(int p = 0; p < (ROWS + XS_THREADS / 8 - 1) / (XS_THREADS / 8); p++) {
    const int r = (threadIdx.x >> 3) + p * (XS_THREADS / 8);
    if(r >= ROWS) break;
    const float* from = row(r);
    for(int c = lane8 * 4; c < pitch - 4; c += 32)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smemU32(dst + r * pitch + c)), "l"(from ? from + c : anywhere), "r"(from ? 16 : 0) : "memory");
  }
}
__device__ __forceinline__ void xsCommit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void xsWaitAllButOne() { asm volatile("cp.async.wait_group 1;" ::: "memory"); }

// NC: groups of 64 output channels; RI: rows per thread (16 threads share a row); VEC: channels in vectors of four
template <typename T, int NC, int RI, bool VEC>
__global__ void __launch_bounds__(XS_THREADS, RI == 1 ? (NC == 1 ? 4 : (NC == 2 ? 2 : 1)) : (NC <= 2 ? 2 : 1)) crossAttnSimtKernel(const CrossAttnArgs a, const XaSplit sp) {
  extern __shared__ float4 smem4[];
  constexpr int ROWS = 16 * RI;
  const int pq = xsPitch(a.dq), pv = xsPitch(a.dv);
  constexpr int PP = XS_KEYS + 4;
  float* sQ = reinterpret_cast<float*>(smem4);
  float* sK = sQ + ROWS * pq;
  float* sV = sK + XS_KEYS * pq;
  float* sP = sV + XS_KEYS * pv;
  uint8_t* sOk = reinterpret_cast<uint8_t*>(sP + ROWS * PP);  // [2]: of this tile of keys, of the next
  constexpr bool ASYNC = VEC && sizeof(T) == 4;  // K of the next tile travels under this one's softmax and second product, V under the first
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const int CG = NC > 1 || a.dv > 32 ? 16 : (a.dv > 16 ? 8 : (a.dv > 8 ? 4 : 2)), KS = 16 / CG;
  const int cg = tx & (CG - 1), ks = tx / CG;
  const XaBlock blk = xaBlock(a, sp, ROWS);
  const int G = a.heads / a.kvHeads;
  gridDepLaunch();
  gridDepWait();
  const int rows = xaRows(a, blk.b, G);
  if(blk.row0 >= rows) return;
  const int keys = xaKeys(a, blk.b);
  const int k0 = blk.part * sp.chunk, k1 = (int)min((long long)keys, (long long)k0 + sp.chunk);
  if(sp.parts > 1 && k0 >= keys && blk.part > 0) return;  // a part without keys; part 0 always reports

  const T* kBase = (const T*)a.k + blk.b * a.kB + blk.kvh * a.kH;
  const T* vBase = (const T*)a.v + blk.b * a.vB + blk.kvh * a.vH;
  auto attended = [&](int key) { return key < k1 && (!a.keyMask || a.keyMask[(int64_t)blk.b * a.kLen + key] != 0.0f); };
  auto qRow = [&](int r) -> const T* {
    r += blk.row0;
    return r < rows ? (const T*)a.q + blk.b * a.qB + (r / G) * a.qT + (blk.kvh * G + r % G) * a.qH : nullptr;
  };
  auto requestK = [&](int kt, const uint8_t* on) { xsStageAsync<XS_KEYS>(sK, pq, (const float*)a.q, [&](int j) { return on[j] ? (const float*)(kBase + (kt + j) * a.kT) : nullptr; }); };
  auto requestV = [&](int kt, const uint8_t* on) { xsStageAsync<XS_KEYS>(sV, pv, (const float*)a.q, [&](int j) { return on[j] ? (const float*)(vBase + (kt + j) * a.vT) : nullptr; }); };
  if(ASYNC) {
    if(tid < XS_KEYS) sOk[tid] = attended(k0 + tid);
    xsStageAsync<ROWS>(sQ, pq, (const float*)a.q, [&](int r) { return (const float*)qRow(r); });
    __syncthreads();
    requestK(k0, sOk);
    xsCommit();
    requestV(k0, sOk);
    xsCommit();
  }
  else xsStage<T, ROWS, VEC>(sQ, pq, a.dq, qRow);
  float mx[RI], sum[RI];
  float4 o[RI][NC];
#pragma unroll
  for(int i = 0; i < RI; i++) {
    mx[i] = -INFINITY;
    sum[i] = 0.0f;
#pragma unroll
    for(int c = 0; c < NC; c++) o[i][c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  const bool vecOut = ((uintptr_t)a.out & 15) == 0 && ((a.oB | a.oT | a.oH) & 3) == 0;  // rows of out, of whole vectors too
  const float scale = a.scale * 1.4426950408889634f;
  for(int kt = k0; kt < k1; kt += XS_KEYS) {
    const int groups = min(4, (k1 - kt + 15) / 16);  // of 16 keys, that the tile has: what is behind them costs no products
    const uint8_t* on = sOk + (ASYNC ? ((kt - k0) / XS_KEYS & 1) * XS_KEYS : 0);
    uint8_t* onNext = sOk + (ASYNC ? XS_KEYS - (on - sOk) : 0);
    if(ASYNC) {
      xsWaitAllButOne();  // K (and Q)
      __syncthreads();
    }
    else {
      __syncthreads();
      if(tid < XS_KEYS) sOk[tid] = attended(kt + tid);
      __syncthreads();
      xsStage<T, XS_KEYS, VEC>(sK, pq, a.dq, [&](int j) { return on[j] ? kBase + (kt + j) * a.kT : nullptr; });
      xsStage<T, XS_KEYS, VEC>(sV, pv, a.dv, [&](int j) { return on[j] ? vBase + (kt + j) * a.vT : nullptr; });
      __syncthreads();
    }
    // even and odd channels apart: the packed fp32 instructions do two IEEE operations per issue slot
    float2 s2[RI][4];
#pragma unroll
    for(int i = 0; i < RI; i++)
#pragma unroll
      for(int j = 0; j < 4; j++) s2[i][j] = make_float2(0.0f, 0.0f);
    auto multiply = [&](auto count) {
      constexpr int J = decltype(count)::value;
#pragma unroll 4
      for(int d = 0; d < pq - 4; d += 4) {
        float4 qv[RI], kv[J];
#pragma unroll
        for(int i = 0; i < RI; i++) qv[i] = *reinterpret_cast<const float4*>(sQ + (ty * RI + i) * pq + d);
#pragma unroll
        for(int j = 0; j < J; j++) kv[j] = *reinterpret_cast<const float4*>(sK + (tx + 16 * j) * pq + d);
#pragma unroll
        for(int i = 0; i < RI; i++)
#pragma unroll
          for(int j = 0; j < J; j++) {
            s2[i][j] = __ffma2_rn(make_float2(qv[i].x, qv[i].y), make_float2(kv[j].x, kv[j].y), s2[i][j]);
            s2[i][j] = __ffma2_rn(make_float2(qv[i].z, qv[i].w), make_float2(kv[j].z, kv[j].w), s2[i][j]);
          }
      }
    };
    if(groups > 2) multiply(std::integral_constant<int, 4>());
    else if(groups == 2) multiply(std::integral_constant<int, 2>());
    else multiply(std::integral_constant<int, 1>());
    float s[RI][4];
#pragma unroll
    for(int i = 0; i < RI; i++)
#pragma unroll
      for(int j = 0; j < 4; j++) s[i][j] = s2[i][j].x + s2[i][j].y;
    if(ASYNC) {
      if(tid < XS_KEYS) onNext[tid] = attended(kt + XS_KEYS + tid);
      __syncthreads();  // K has been read
      if(kt + XS_KEYS < k1) requestK(kt + XS_KEYS, onNext);
      xsCommit();
    }
#pragma unroll
    for(int i = 0; i < RI; i++) {
      float top = -INFINITY;
#pragma unroll
      for(int j = 0; j < 4; j++) {
        s[i][j] = on[tx + 16 * j] ? s[i][j] * scale : -INFINITY;
        top = fmaxf(top, s[i][j]);
      }
#pragma unroll
      for(int w = 8; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));  // the 16 threads of a row
      const float now = fmaxf(mx[i], top);
      const float ref = now == -INFINITY ? 0.0f : now;  // nothing attended yet: every exponential is 0
      const float keep = exp2f(mx[i] - ref);
      mx[i] = now;
      float part = 0.0f;
#pragma unroll
      for(int j = 0; j < 4; j++) {
        const float p = exp2f(s[i][j] - ref);
        part += p;
        sP[(ty * RI + i) * PP + tx + 16 * j] = p;
      }
      sum[i] = sum[i] * keep + part;  // this thread's share of the row
#pragma unroll
      for(int c = 0; c < NC; c++) { o[i][c].x *= keep; o[i][c].y *= keep; o[i][c].z *= keep; o[i][c].w *= keep; }
    }
    if(ASYNC) xsWaitAllButOne();  // V
    __syncthreads();
    // Output channels: CG threads have four each (of every 64 where there are more); the other threads of a row share the keys.
    for(int j = ks * 4; j < groups * 16; j += 4 * KS) {
      float4 p[RI];
#pragma unroll
      for(int i = 0; i < RI; i++) p[i] = *reinterpret_cast<const float4*>(sP + (ty * RI + i) * PP + j);
#pragma unroll
      for(int c = 0; c < NC; c++) {
        const int d = c * 64 + cg * 4;
        if(d >= a.dv) break;
        float4 v[4];
#pragma unroll
        for(int e = 0; e < 4; e++) v[e] = *reinterpret_cast<const float4*>(sV + (j + e) * pv + d);
#pragma unroll
        for(int i = 0; i < RI; i++) {
          const float pe[4] = {p[i].x, p[i].y, p[i].z, p[i].w};
#pragma unroll
          for(int e = 0; e < 4; e++) {
            const float2 pp = make_float2(pe[e], pe[e]);
            const float2 lo = __ffma2_rn(pp, make_float2(v[e].x, v[e].y), make_float2(o[i][c].x, o[i][c].y));
            const float2 hi = __ffma2_rn(pp, make_float2(v[e].z, v[e].w), make_float2(o[i][c].z, o[i][c].w));
            o[i][c] = make_float4(lo.x, lo.y, hi.x, hi.y);
          }
        }
      }
    }
    if(ASYNC) {
      __syncthreads();  // V has been read
      if(kt + XS_KEYS < k1) requestV(kt + XS_KEYS, onNext);
      xsCommit();
    }
  }
  if(ASYNC) asm volatile("cp.async.wait_group 0;" ::: "memory");
  if(KS > 1)
#pragma unroll
    for(int i = 0; i < RI; i++)
      for(int w = CG; w < 16; w *= 2) {
        o[i][0].x += __shfl_xor_sync(0xffffffffu, o[i][0].x, w);
        o[i][0].y += __shfl_xor_sync(0xffffffffu, o[i][0].y, w);
        o[i][0].z += __shfl_xor_sync(0xffffffffu, o[i][0].z, w);
        o[i][0].w += __shfl_xor_sync(0xffffffffu, o[i][0].w, w);
      }
#pragma unroll
  for(int i = 0; i < RI; i++) {
    float total = sum[i];
#pragma unroll
    for(int w = 8; w > 0; w >>= 1) total += __shfl_xor_sync(0xffffffffu, total, w);
    const int r = blk.row0 + ty * RI + i;
    if(r >= rows) continue;
    if(sp.parts > 1) {
      float* part = xaPart(a, sp, blk, r, G);
#pragma unroll
      for(int c = 0; c < NC; c++)
#pragma unroll
        for(int e = 0; e < 4; e++) {
          const int d = c * 64 + cg * 4 + e;
          if(d < a.dv && ks == 0) part[2 + d] = reinterpret_cast<const float*>(&o[i][c])[e];
        }
      if(tx == 0) { part[0] = mx[i]; part[1] = total; }
      continue;
    }
    T* out = (T*)a.out + blk.b * a.oB + (r / G) * a.oT + (blk.kvh * G + r % G) * a.oH;
    const bool live = total != 0.0f && (!a.queryMask || a.queryMask[(int64_t)blk.b * a.qLen + r / G] != 0.0f);
    const float inv = 1.0f / total;
    if(ASYNC && vecOut) {
#pragma unroll
      for(int c = 0; c < NC; c++) {
        const int d = c * 64 + cg * 4;
        const float4 v = o[i][c];
        if(d < a.dv && ks == 0) *reinterpret_cast<float4*>(out + d) = live ? make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      }
      continue;
    }
#pragma unroll
    for(int c = 0; c < NC; c++)
#pragma unroll
      for(int e = 0; e < 4; e++) {
        const int d = c * 64 + cg * 4 + e;
        if(d < a.dv && ks == 0) out[d] = OpType<T>::from(live ? reinterpret_cast<const float*>(&o[i][c])[e] * inv : 0.0f);
      }
  }
}

// One block per row: the parts' weights, then the parts' states, added in the order of the keys.  The threads beyond a row's channels
// take another stretch of the parts.
constexpr int XJ_THREADS = 256;
template <typename T>
__global__ void __launch_bounds__(XJ_THREADS) crossAttnJoinKernel(const CrossAttnArgs a, const XaSplit sp) {
  __shared__ float sW[XA_MAX_PARTS], sTop[XJ_THREADS / 32], sO[XJ_THREADS], sTotal[XJ_THREADS / 32];
  gridDepLaunch();
  gridDepWait();
  const int G = a.heads / a.kvHeads, tid = threadIdx.x;
  const long long perHead = (long long)a.qLen * G, bh = blockIdx.x / perHead;
  const int r = (int)(blockIdx.x - bh * perHead);
  XaBlock blk;
  blk.b = (int)(bh / a.kvHeads);
  blk.kvh = (int)(bh - (long long)blk.b * a.kvHeads);
  blk.row0 = 0;
  blk.part = 0;
  if(r >= xaRows(a, blk.b, G)) return;
  const int parts = max(1, (int)(((long long)xaKeys(a, blk.b) + sp.chunk - 1) / sp.chunk));
  const float* state = xaPart(a, sp, blk, r, G);
  // weights
  const float top0 = tid < parts ? state[(int64_t)tid * sp.pitch] : -INFINITY;
  static_assert(XA_MAX_PARTS <= XJ_THREADS, "a thread per part");
  float top = top0;
#pragma unroll
  for(int w = 16; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
  if((tid & 31) == 0) sTop[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for(int w = 0; w < XJ_THREADS / 32; w++) top = fmaxf(top, sTop[w]);
  const float ref = top == -INFINITY ? 0.0f : top;
  float total = 0.0f;
  if(tid < parts) {
    const float w = exp2f(top0 - ref);
    sW[tid] = w;
    total = w * state[(int64_t)tid * sp.pitch + 1];
  }
#pragma unroll
  for(int w = 16; w > 0; w >>= 1) total += __shfl_xor_sync(0xffffffffu, total, w);
  if((tid & 31) == 0) sTotal[tid >> 5] = total;
  __syncthreads();
  total = 0.0f;
#pragma unroll
  for(int w = 0; w < XJ_THREADS / 32; w++) total += sTotal[w];
  // channels
  const int width = a.dv <= 32 ? 32 : (a.dv <= 64 ? 64 : (a.dv <= 128 ? 128 : 256)), shares = XJ_THREADS / width;
  const int d = tid & (width - 1), share = tid / width;
  float o = 0.0f;
  if(d < a.dv) {
    const int p1 = (share + 1) * parts / shares;
#pragma unroll 8
    for(int p = share * parts / shares; p < p1; p++) o = fmaf(sW[p], state[(int64_t)p * sp.pitch + 2 + d], o);
  }
  sO[tid] = o;
  __syncthreads();
  if(share > 0 || d >= a.dv) return;
  for(int s = 1; s < shares; s++) o += sO[s * width + d];
  const bool live = total != 0.0f && (!a.queryMask || a.queryMask[(int64_t)blk.b * a.qLen + r / G] != 0.0f);
  T* out = (T*)a.out + blk.b * a.oB + (r / G) * a.oT + (blk.kvh * G + r % G) * a.oH;
  out[d] = OpType<T>::from(live ? o * (1.0f / total) : 0.0f);
}

// The same with a warp per row, for many rows (which have few parts): 34 656 rows of two parts took 110 us with a block each.
template <typename T>
__global__ void __launch_bounds__(XJ_THREADS) crossAttnJoinManyKernel(const CrossAttnArgs a, const XaSplit sp) {
  gridDepLaunch();
  gridDepWait();
  const int G = a.heads / a.kvHeads, lane = threadIdx.x & 31;
  const long long perHead = (long long)a.qLen * G, i = (long long)blockIdx.x * (XJ_THREADS / 32) + (threadIdx.x >> 5), bh = i / perHead;
  if(bh >= (long long)a.batch * a.kvHeads) return;
  const int r = (int)(i - bh * perHead);
  XaBlock blk;
  blk.b = (int)(bh / a.kvHeads);
  blk.kvh = (int)(bh - (long long)blk.b * a.kvHeads);
  blk.row0 = 0;
  blk.part = 0;
  if(r >= xaRows(a, blk.b, G)) return;
  const int parts = max(1, (int)(((long long)xaKeys(a, blk.b) + sp.chunk - 1) / sp.chunk));
  const float* state = xaPart(a, sp, blk, r, G);
  float top = -INFINITY;
  for(int p = lane; p < parts; p += 32) top = fmaxf(top, state[(int64_t)p * sp.pitch]);
#pragma unroll
  for(int w = 16; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
  const float ref = top == -INFINITY ? 0.0f : top;
  float total = 0.0f, o[8];
#pragma unroll
  for(int c = 0; c < 8; c++) o[c] = 0.0f;
#pragma unroll 2
  for(int p = 0; p < parts; p++) {
    const float* part = state + (int64_t)p * sp.pitch;
    const float w = exp2f(part[0] - ref);
    total += w * part[1];
#pragma unroll
    for(int c = 0; c < 8; c++)
      if(c * 32 + lane < a.dv) o[c] = fmaf(w, part[2 + c * 32 + lane], o[c]);
  }
  const bool live = total != 0.0f && (!a.queryMask || a.queryMask[(int64_t)blk.b * a.qLen + r / G] != 0.0f);
  const float inv = 1.0f / total;
  T* out = (T*)a.out + blk.b * a.oB + (r / G) * a.oT + (blk.kvh * G + r % G) * a.oH;
#pragma unroll
  for(int c = 0; c < 8; c++)
    if(c * 32 + lane < a.dv) out[c * 32 + lane] = OpType<T>::from(live ? o[c] * inv : 0.0f);
}
template <typename T> cudaError_t joinLaunch(cudaStream_t st, const CrossAttnArgs& a, const XaSplit& sp) {
  const long long rows = (long long)a.batch * a.qLen * a.heads;
  if(rows < 8LL * smCount()) return launchDependent(crossAttnJoinKernel<T>, dim3((unsigned)rows), dim3(XJ_THREADS), 0, st, a, sp);
  return launchDependent(crossAttnJoinManyKernel<T>, dim3((unsigned)((rows + XJ_THREADS / 32 - 1) / (XJ_THREADS / 32))), dim3(XJ_THREADS), 0, st, a, sp);
}

template <typename T, int NC, int RI, bool VEC> cudaError_t simtLaunch(cudaStream_t st, const CrossAttnArgs& a, const XaSplit& sp) {
  static SharedMemoryOptIn optIn;
  const cudaError_t e = optIn((const void*)crossAttnSimtKernel<T, NC, RI, VEC>, 227 * 1024);
  if(e != cudaSuccess) return e;
  return launchDependent(crossAttnSimtKernel<T, NC, RI, VEC>, dim3(sp.blocks), dim3(XS_THREADS), xsSmem(16 * RI, a.dq, a.dv), st, a, sp);
}
template <typename T, int NC> cudaError_t simtLaunchNC(cudaStream_t st, const CrossAttnArgs& a, const XaSplit& sp, int rows) {
  const uintptr_t p = (uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.v;
  const int64_t strides = a.qB | a.qT | a.qH | a.kB | a.kT | a.kH | a.vB | a.vT | a.vH;
  const bool vec = p % (4 * sizeof(T)) == 0 && strides % 4 == 0 && a.dq % 4 == 0 && a.dv % 4 == 0;
  if(rows == 16) return vec ? simtLaunch<T, NC, 1, true>(st, a, sp) : simtLaunch<T, NC, 1, false>(st, a, sp);
  return vec ? simtLaunch<T, NC, 4, true>(st, a, sp) : simtLaunch<T, NC, 4, false>(st, a, sp);
}
template <typename T> cudaError_t simtLaunchT(cudaStream_t st, const CrossAttnArgs& a, const XaSplit& sp, int rows) {
  if(a.dv <= 64) return simtLaunchNC<T, 1>(st, a, sp, rows);
  if(a.dv <= 128) return simtLaunchNC<T, 2>(st, a, sp, rows);
  return simtLaunchNC<T, 4>(st, a, sp, rows);
}
// Rows of a block of the CUDA-core kernel.
int simtRows(int qLen, int heads, int kvHeads) { return (long long)qLen * (heads / kvHeads) <= 16 ? 16 : 64; }

}  // namespace

XaSplit xaPlanSplit(int rowsPerBlock, int keysPerStep, int keysWorthABlock, int blocksPerSm, int batch, int qLen, int kLen, int heads, int kvHeads, int dv) {
  XaSplit sp;
  const long long rows = (long long)qLen * (heads / kvHeads);
  sp.rowTiles = (int)((rows + rowsPerBlock - 1) / rowsPerBlock);
  const long long whole = (long long)batch * kvHeads * sp.rowTiles, room = (long long)blocksPerSm * smCount();
  // Parts of the keys.  So many that the blocks fill the GPU once, of at least two steps; and up to four times as many where their
  // parts stay long against what a block costs besides: sequences of different lengths, and the end of the last round, are then
  // shared out evenly (8 sequences of 0 to 32768 keys, 8 key heads of 128, bf16: 109 us in 4 parts of 8192).
  const long long once = std::min<long long>(room / whole, kLen / (2LL * keysPerStep));
  const long long even = std::min<long long>(4 * room / whole, kLen / keysWorthABlock);
  const long long parts = std::min<long long>(XA_MAX_PARTS, std::max<long long>(1, std::max(once, even)));
  long long chunk = ((long long)kLen + parts - 1) / parts;
  chunk = std::max<long long>(keysPerStep, (chunk + keysPerStep - 1) / keysPerStep * keysPerStep);
  sp.chunk = (int)std::min<long long>(chunk, 1LL << 30);
  sp.parts = (int)std::max<long long>(1, ((long long)kLen + sp.chunk - 1) / sp.chunk);
  sp.blocks = (unsigned)(whole * sp.parts);
  sp.pitch = (dv + 2 + 3) / 4 * 4;
  sp.workspace = sp.parts > 1 ? (size_t)batch * kvHeads * rows * sp.parts * sp.pitch * sizeof(float) : 0;
  return sp;
}

namespace {

// Rows on 16-byte boundaries, and no repetition along the dimensions of which TMA takes several at once.
bool viewAligned(const void* p, int batch, int64_t b, int tokens, int64_t t, int heads, int64_t h, bool headsTogether) {
  return ((uintptr_t)p & 15) == 0 && (batch == 1 || b % 8 == 0) && (tokens <= 1 || (t % 8 == 0 && t != 0)) &&
         (heads == 1 || (h % 8 == 0 && !(headsTogether && h == 0)));
}
bool crossAttnAligned(const CrossAttnArgs& a) {
  return viewAligned(a.q, a.batch, a.qB, a.qLen, a.qT, a.heads, a.qH, true) && viewAligned(a.k, a.batch, a.kB, a.kLen, a.kT, a.kvHeads, a.kH, false) &&
         viewAligned(a.v, a.batch, a.vB, a.kLen, a.vT, a.kvHeads, a.vH, false) && viewAligned(a.out, a.batch, a.oB, a.qLen, a.oT, a.heads, a.oH, true);
}

// What a call runs.  The workspace is a function of the sizes alone, so the plan is too: where the sizes suit the tensor cores and
// only the tensors' alignment does not, the CUDA-core kernel cuts the keys as the other would.
struct Plan {
  enum { SIMT, FEW, TC } kind;
  int tilesPerBlock;
  XaSplit sp;
};
Plan planFor(int dt, int batch, int qLen, int kLen, int heads, int kvHeads, int dq, int dv) {
  Plan p = {};
  p.kind = !crossAttnTcSizes(dt, heads, kvHeads, dq, dv) ? Plan::SIMT : ((long long)qLen * (heads / kvHeads) <= 16 ? Plan::FEW : Plan::TC);
  if(p.kind == Plan::TC) p.sp = crossAttnTcSplit(batch, qLen, kLen, heads, kvHeads, dv, &p.tilesPerBlock);
  else if(p.kind == Plan::FEW) p.sp = crossAttnFewSplit(batch, qLen, kLen, heads, kvHeads, dq, dv);
  else {
    const int rows = simtRows(qLen, heads, kvHeads);
    p.sp = xaPlanSplit(rows, XS_KEYS, 512, rows == 16 && dq <= 64 && dv <= 64 ? 4 : 2, batch, qLen, kLen, heads, kvHeads, dv);
  }
  return p;
}

}  // namespace

size_t crossAttnWorkspace(int dt, int batch, int qLen, int kLen, int heads, int kvHeads, int dq, int dv) {
  return planFor(dt, batch, qLen, kLen, heads, kvHeads, dq, dv).sp.workspace;
}

cudaError_t launchCrossAttn(cudaStream_t st, const CrossAttnArgs& a) {
  if(a.batch == 0 || a.qLen == 0) return cudaSuccess;
  Plan p = planFor(a.dt, a.planBatch > 0 ? a.planBatch : a.batch, a.qLen, a.kLen, a.heads, a.kvHeads, a.dq, a.dv);
  XaSplit& sp = p.sp;
  sp.blocks = (unsigned)((long long)a.batch * a.kvHeads * sp.rowTiles * sp.parts);
  if(p.kind != Plan::SIMT && !crossAttnAligned(a)) {
    p.kind = Plan::SIMT;
    const int rows = simtRows(a.qLen, a.heads, a.kvHeads);
    sp.rowTiles = (int)(((long long)a.qLen * (a.heads / a.kvHeads) + rows - 1) / rows);
    sp.blocks = (unsigned)((long long)a.batch * a.kvHeads * sp.rowTiles * sp.parts);
  }
  cudaError_t e;
  if(p.kind == Plan::TC) e = launchCrossAttnTc(st, a, sp, p.tilesPerBlock);
  else if(p.kind == Plan::FEW) e = launchCrossAttnFew(st, a, sp);
  else
    switch(a.dt) {
      case DT_F32: e = simtLaunchT<float>(st, a, sp, simtRows(a.qLen, a.heads, a.kvHeads)); break;
      case DT_F16: e = simtLaunchT<__half>(st, a, sp, simtRows(a.qLen, a.heads, a.kvHeads)); break;
      default: e = simtLaunchT<__nv_bfloat16>(st, a, sp, simtRows(a.qLen, a.heads, a.kvHeads)); break;
    }
  if(e != cudaSuccess || sp.parts == 1) return e;
  switch(a.dt) {
    case DT_F32: return joinLaunch<float>(st, a, sp);
    case DT_F16: return joinLaunch<__half>(st, a, sp);
    default: return joinLaunch<__nv_bfloat16>(st, a, sp);
  }
}

}  // namespace kb

// Attention to states of another length on a caller's own tensors: the CUDA-core kernel for every type, head size up to 256
// and alignment, and the kernel that joins the parts of rows whose keys were cut over several blocks.
//
// The rows of a key head are its query heads' rows side by side: row r = token r / G, head kvHead * G + r % G with G = heads /
// kvHeads, so that grouped heads read K and V once.  A block takes 64 such rows and a range of keys, 64 at a time: scores into
// registers (4 x 4 per thread), a running maximum and sum per row, probabilities through shared memory, output accumulators in
// registers.  All in fp32.  Keys behind a sequence's length are not read; masked keys' rows of K and V are replaced by zeros
// while they are staged, so that nothing in them (NaN, Inf) reaches a product.
//
// A row's state is (maximum, sum, unnormalised output).  Where few rows have many keys the keys are cut into parts of `chunk`
// keys, one block each; a part writes its state to the workspace and crossAttnJoinKernel adds the parts in order.
#include "kb_kernels.cuh"
#include "kb_ops.h"
#include "kb_ops_dev.cuh"
#include "kb_xattn.cuh"

#include <algorithm>

namespace kb {

namespace {

constexpr int XS_ROWS = 64, XS_KEYS = 64, XS_THREADS = 256;

__host__ __device__ constexpr int xsPitch(int d) { return (d + 3) / 4 * 4 + 4; }
size_t xsSmem(int dq, int dv) { return sizeof(float) * (size_t)((XS_ROWS + XS_KEYS) * xsPitch(dq) + XS_KEYS * xsPitch(dv) + XS_ROWS * (XS_KEYS + 4)) + XS_KEYS; }

// NC: groups of 64 output channels
template <typename T, int NC>
__global__ void __launch_bounds__(XS_THREADS) crossAttnSimtKernel(const CrossAttnArgs a, const XaSplit sp) {
  extern __shared__ float4 smem4[];
  const int pq = xsPitch(a.dq), pv = xsPitch(a.dv);
  constexpr int PP = XS_KEYS + 4;
  float* sQ = reinterpret_cast<float*>(smem4);
  float* sK = sQ + XS_ROWS * pq;
  float* sV = sK + XS_KEYS * pq;
  float* sP = sV + XS_KEYS * pv;
  uint8_t* sOk = reinterpret_cast<uint8_t*>(sP + XS_ROWS * PP);
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;
  const XaBlock blk = xaBlock(a, sp, XS_ROWS);
  const int G = a.heads / a.kvHeads;
  gridDepLaunch();
  gridDepWait();
  const int rows = xaRows(a, blk.b, G);
  if(blk.row0 >= rows) return;
  const int keys = xaKeys(a, blk.b);
  const int k0 = blk.part * sp.chunk, k1 = (int)min((long long)keys, (long long)k0 + sp.chunk);
  if(sp.parts > 1 && k0 >= keys && blk.part > 0) return;  // a part without keys; part 0 always reports
  auto rowQ = [&](int r) { return (const T*)a.q + blk.b * a.qB + (r / G) * a.qT + (blk.kvh * G + r % G) * a.qH; };

  for(int i = tid; i < XS_ROWS * pq; i += XS_THREADS) {
    const int r = i / pq, d = i - r * pq;
    sQ[i] = (d < a.dq && blk.row0 + r < rows) ? OpType<T>::to(rowQ(blk.row0 + r)[d]) : 0.0f;
  }
  float mx[4], sum[4];
  float4 o[4][NC];
#pragma unroll
  for(int i = 0; i < 4; i++) {
    mx[i] = -INFINITY;
    sum[i] = 0.0f;
#pragma unroll
    for(int c = 0; c < NC; c++) o[i][c] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  const float scale = a.scale * 1.4426950408889634f;
  const T* kBase = (const T*)a.k + blk.b * a.kB + blk.kvh * a.kH;
  const T* vBase = (const T*)a.v + blk.b * a.vB + blk.kvh * a.vH;
  for(int kt = k0; kt < k1; kt += XS_KEYS) {
    __syncthreads();
    if(tid < XS_KEYS) sOk[tid] = kt + tid < k1 && (!a.keyMask || a.keyMask[(int64_t)blk.b * a.kLen + kt + tid] != 0.0f);
    __syncthreads();
    for(int i = tid; i < XS_KEYS * pq; i += XS_THREADS) {
      const int j = i / pq, d = i - j * pq;
      sK[i] = (d < a.dq && sOk[j]) ? OpType<T>::to(kBase[(kt + j) * a.kT + d]) : 0.0f;
    }
    for(int i = tid; i < XS_KEYS * pv; i += XS_THREADS) {
      const int j = i / pv, d = i - j * pv;
      sV[i] = (d < a.dv && sOk[j]) ? OpType<T>::to(vBase[(kt + j) * a.vT + d]) : 0.0f;
    }
    __syncthreads();
    float s[4][4];
#pragma unroll
    for(int i = 0; i < 4; i++)
#pragma unroll
      for(int j = 0; j < 4; j++) s[i][j] = 0.0f;
    for(int d = 0; d < a.dq; d += 4) {
      float4 qv[4], kv[4];
#pragma unroll
      for(int i = 0; i < 4; i++) qv[i] = *reinterpret_cast<const float4*>(sQ + (ty * 4 + i) * pq + d);
#pragma unroll
      for(int j = 0; j < 4; j++) kv[j] = *reinterpret_cast<const float4*>(sK + (tx + 16 * j) * pq + d);
#pragma unroll
      for(int i = 0; i < 4; i++)
#pragma unroll
        for(int j = 0; j < 4; j++) {
          s[i][j] = fmaf(qv[i].x, kv[j].x, s[i][j]);
          s[i][j] = fmaf(qv[i].y, kv[j].y, s[i][j]);
          s[i][j] = fmaf(qv[i].z, kv[j].z, s[i][j]);
          s[i][j] = fmaf(qv[i].w, kv[j].w, s[i][j]);
        }
    }
#pragma unroll
    for(int i = 0; i < 4; i++) {
      float top = -INFINITY;
#pragma unroll
      for(int j = 0; j < 4; j++) {
        s[i][j] = sOk[tx + 16 * j] ? s[i][j] * scale : -INFINITY;
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
        sP[(ty * 4 + i) * PP + tx + 16 * j] = p;
      }
      sum[i] = sum[i] * keep + part;  // this thread's share of the row
#pragma unroll
      for(int c = 0; c < NC; c++) { o[i][c].x *= keep; o[i][c].y *= keep; o[i][c].z *= keep; o[i][c].w *= keep; }
    }
    __syncthreads();
    for(int j = 0; j < XS_KEYS; j++) {
      float p[4];
#pragma unroll
      for(int i = 0; i < 4; i++) p[i] = sP[(ty * 4 + i) * PP + j];
#pragma unroll
      for(int c = 0; c < NC; c++) {
        const int d = c * 64 + tx * 4;
        if(d >= a.dv) break;
        const float4 v = *reinterpret_cast<const float4*>(sV + j * pv + d);
#pragma unroll
        for(int i = 0; i < 4; i++) {
          o[i][c].x = fmaf(p[i], v.x, o[i][c].x);
          o[i][c].y = fmaf(p[i], v.y, o[i][c].y);
          o[i][c].z = fmaf(p[i], v.z, o[i][c].z);
          o[i][c].w = fmaf(p[i], v.w, o[i][c].w);
        }
      }
    }
  }
#pragma unroll
  for(int i = 0; i < 4; i++) {
    float total = sum[i];
#pragma unroll
    for(int w = 8; w > 0; w >>= 1) total += __shfl_xor_sync(0xffffffffu, total, w);
    const int r = blk.row0 + ty * 4 + i;
    if(r >= rows) continue;
    if(sp.parts > 1) {
      float* part = xaPart(a, sp, blk, r, G);
#pragma unroll
      for(int c = 0; c < NC; c++)
#pragma unroll
        for(int e = 0; e < 4; e++) {
          const int d = c * 64 + tx * 4 + e;
          if(d < a.dv) part[2 + d] = reinterpret_cast<const float*>(&o[i][c])[e];
        }
      if(tx == 0) { part[0] = mx[i]; part[1] = total; }
      continue;
    }
    T* out = (T*)a.out + blk.b * a.oB + (r / G) * a.oT + (blk.kvh * G + r % G) * a.oH;
    const bool live = total != 0.0f && (!a.queryMask || a.queryMask[(int64_t)blk.b * a.qLen + r / G] != 0.0f);
    const float inv = 1.0f / total;
#pragma unroll
    for(int c = 0; c < NC; c++)
#pragma unroll
      for(int e = 0; e < 4; e++) {
        const int d = c * 64 + tx * 4 + e;
        if(d < a.dv) out[d] = OpType<T>::from(live ? reinterpret_cast<const float*>(&o[i][c])[e] * inv : 0.0f);
      }
  }
}

// One warp per row: the parts' states, added in the order of the keys.
template <typename T>
__global__ void __launch_bounds__(256) crossAttnJoinKernel(const CrossAttnArgs a, const XaSplit sp) {
  gridDepLaunch();
  gridDepWait();
  const int G = a.heads / a.kvHeads, lane = threadIdx.x & 31;
  const long long all = (long long)a.batch * a.kvHeads * a.qLen * G;
  for(long long i = (long long)blockIdx.x * 8 + (threadIdx.x >> 5); i < all; i += (long long)gridDim.x * 8) {
    const long long perHead = (long long)a.qLen * G;
    XaBlock blk;
    const long long bh = i / perHead;
    const int r = (int)(i - bh * perHead);
    blk.b = (int)(bh / a.kvHeads);
    blk.kvh = (int)(bh - (long long)blk.b * a.kvHeads);
    blk.row0 = 0;
    if(r >= xaRows(a, blk.b, G)) continue;
    const int keys = xaKeys(a, blk.b);
    const int parts = max(1, (int)(((long long)keys + sp.chunk - 1) / sp.chunk));
    float top = -INFINITY;
    for(int p = lane; p < parts; p += 32) { blk.part = p; top = fmaxf(top, xaPart(a, sp, blk, r, G)[0]); }
#pragma unroll
    for(int w = 16; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
    const float ref = top == -INFINITY ? 0.0f : top;
    float total = 0.0f, o[8];
#pragma unroll
    for(int c = 0; c < 8; c++) o[c] = 0.0f;
    for(int p = 0; p < parts; p++) {
      blk.part = p;
      const float* part = xaPart(a, sp, blk, r, G);
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
}

template <typename T, int NC> cudaError_t simtLaunch(cudaStream_t st, const CrossAttnArgs& a, const XaSplit& sp) {
  const cudaError_t e = allowSharedMemory((const void*)crossAttnSimtKernel<T, NC>, 227 * 1024);
  if(e != cudaSuccess) return e;
  return launchDependent(crossAttnSimtKernel<T, NC>, dim3(sp.blocks), dim3(XS_THREADS), xsSmem(a.dq, a.dv), st, a, sp);
}
template <typename T> cudaError_t simtLaunchT(cudaStream_t st, const CrossAttnArgs& a, const XaSplit& sp) {
  if(a.dv <= 64) return simtLaunch<T, 1>(st, a, sp);
  if(a.dv <= 128) return simtLaunch<T, 2>(st, a, sp);
  return simtLaunch<T, 4>(st, a, sp);
}

}  // namespace

XaSplit xaPlanSplit(int rowsPerBlock, int keysPerStep, int blocksPerSm, int batch, int qLen, int kLen, int heads, int kvHeads, int dv) {
  XaSplit sp;
  const long long rows = (long long)qLen * (heads / kvHeads);
  sp.rowTiles = (int)((rows + rowsPerBlock - 1) / rowsPerBlock);
  const long long whole = (long long)batch * kvHeads * sp.rowTiles;
  // Keys are cut where the uncut blocks would leave most of the GPU idle, into as many parts as fill it about twice, of at
  // least two steps.
  const long long room = (long long)blocksPerSm * smCount();
  long long parts = 1;
  if(whole * 2 <= room) parts = std::min<long long>(2 * room / whole, ((long long)kLen + 2 * keysPerStep - 1) / (2 * keysPerStep));
  if(parts < 1) parts = 1;
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
  bool tc;
  int tilesPerBlock;
  XaSplit sp;
};
Plan planFor(int dt, int batch, int qLen, int kLen, int heads, int kvHeads, int dq, int dv) {
  Plan p = {};
  p.tc = crossAttnTcSizes(dt, heads, kvHeads, dq, dv);
  if(p.tc) p.sp = crossAttnTcSplit(batch, qLen, kLen, heads, kvHeads, dv, &p.tilesPerBlock);
  else p.sp = xaPlanSplit(XS_ROWS, XS_KEYS, 2, batch, qLen, kLen, heads, kvHeads, dv);
  return p;
}

}  // namespace

size_t crossAttnWorkspace(int dt, int batch, int qLen, int kLen, int heads, int kvHeads, int dq, int dv) {
  return planFor(dt, batch, qLen, kLen, heads, kvHeads, dq, dv).sp.workspace;
}

cudaError_t launchCrossAttn(cudaStream_t st, const CrossAttnArgs& a) {
  if(a.batch == 0 || a.qLen == 0) return cudaSuccess;
  Plan p = planFor(a.dt, a.batch, a.qLen, a.kLen, a.heads, a.kvHeads, a.dq, a.dv);
  XaSplit& sp = p.sp;
  if(p.tc && !crossAttnAligned(a)) {
    p.tc = false;
    sp.rowTiles = (int)(((long long)a.qLen * (a.heads / a.kvHeads) + XS_ROWS - 1) / XS_ROWS);
    sp.blocks = (unsigned)((long long)a.batch * a.kvHeads * sp.rowTiles * sp.parts);
  }
  cudaError_t e;
  if(p.tc) e = launchCrossAttnTc(st, a, sp, p.tilesPerBlock);
  else
    switch(a.dt) {
      case DT_F32: e = simtLaunchT<float>(st, a, sp); break;
      case DT_F16: e = simtLaunchT<__half>(st, a, sp); break;
      default: e = simtLaunchT<__nv_bfloat16>(st, a, sp); break;
    }
  if(e != cudaSuccess || sp.parts == 1) return e;
  const long long rows = (long long)a.batch * a.qLen * a.heads;
  const dim3 grid((unsigned)std::min<long long>((rows + 7) / 8, 16LL * smCount()));
  switch(a.dt) {
    case DT_F32: return launchDependent(crossAttnJoinKernel<float>, grid, dim3(256), 0, st, a, sp);
    case DT_F16: return launchDependent(crossAttnJoinKernel<__half>, grid, dim3(256), 0, st, a, sp);
    default: return launchDependent(crossAttnJoinKernel<__nv_bfloat16>, grid, dim3(256), 0, st, a, sp);
  }
}

}  // namespace kb

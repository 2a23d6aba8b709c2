// What the kernels of attention to states of another length share: which block has which rows and keys, and where the parts of a
// row whose keys were cut wait to be joined.
#pragma once

#include <cuda_runtime.h>
#include <cstdint>

#include "kb_ops.h"

namespace kb {

struct XaSplit {
  int rowTiles;   // tiles of rows per (sequence, key head)
  int parts;      // parts of the keys (1: not cut)
  int chunk;      // keys of a part
  unsigned blocks;
  int pitch;      // floats of a part's state: maximum, sum, unnormalised output
  size_t workspace;
};
constexpr int XA_MAX_PARTS = 256;
// Cuts the keys of blocks of rowsPerBlock rows where the uncut blocks would leave part of the GPU idle.
XaSplit xaPlanSplit(int rowsPerBlock, int keysPerStep, int keysWorthABlock, int blocksPerSm, int batch, int qLen, int kLen, int heads, int kvHeads, int dv);

// kb_xattn_tc.cu: sizes that the tensor-core kernel takes (and rows on 16-byte boundaries)
bool crossAttnTcSizes(int dt, int heads, int kvHeads, int dq, int dv);
XaSplit crossAttnTcSplit(int batch, int qLen, int kLen, int heads, int kvHeads, int dv, int* tilesPerBlock);
cudaError_t launchCrossAttnTc(cudaStream_t st, const CrossAttnArgs& a, const XaSplit& sp, int tilesPerBlock);

// kb_xattn_few.cu: the same sizes, up to 16 rows of a key head
XaSplit crossAttnFewSplit(int batch, int qLen, int kLen, int heads, int kvHeads, int dq, int dv);
cudaError_t launchCrossAttnFew(cudaStream_t st, const CrossAttnArgs& a, const XaSplit& sp);

struct XaBlock {
  int b, kvh, row0, part;
};

// Rows of this sequence's key head, valid keys of this sequence.  Lengths outside their range are brought into it, so that a wrong
// one reads nothing that is not there.
__device__ __forceinline__ int xaRows(const CrossAttnArgs& a, int b, int G) {
  const int q = a.qLengths ? max(0, min(a.qLengths[b], a.qLen)) : a.qLen;
  return q * G;
}
__device__ __forceinline__ int xaKeys(const CrossAttnArgs& a, int b) {
  return a.kLengths ? max(0, min(a.kLengths[b], a.kLen)) : a.kLen;
}
// Parts of one row tile are neighbours in the grid, then the row tiles of a key head (they share its K and V in L2).
__device__ __forceinline__ XaBlock xaBlock(const CrossAttnArgs& a, const XaSplit& sp, int rowsPerBlock, unsigned i = blockIdx.x) {
  XaBlock k;
  k.part = i % sp.parts; i /= sp.parts;
  k.row0 = (int)(i % sp.rowTiles) * rowsPerBlock; i /= sp.rowTiles;
  k.kvh = i % a.kvHeads;
  k.b = i / a.kvHeads;
  return k;
}
__device__ __forceinline__ float* xaPart(const CrossAttnArgs& a, const XaSplit& sp, const XaBlock& k, int r, int G) {
  const int64_t row = ((int64_t)k.b * a.kvHeads + k.kvh) * ((int64_t)a.qLen * G) + r;
  return (float*)a.workspace + (row * sp.parts + k.part) * sp.pitch;
}

}  // namespace kb

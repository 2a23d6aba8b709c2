// The transformer operators that callers use on their own device buffers (include/katab200.h: kb_matmul, kb_rope,
// kb_cross_attention): argument records, what kb_ops.cu checks, and the launchers of the kernels.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <atomic>
#include <cstddef>
#include <cstdint>

#include "../../include/katab200.h"

namespace kb {

// A word of page-locked host memory that a kernel whose wait ran out writes and the next call of an operator reads.  One for the
// process, made at the first use; a stream capture that is under way on the thread does not mind.
int* operatorWaitWord();
// Lets `fn` use up to `bytes` of shared memory on the current device; asked of the driver once per device.
struct SharedMemoryOptIn {
  std::atomic<uint64_t> done{0};
  cudaError_t operator()(const void* fn, int bytes);
};
// A tensor map of up to four dimensions (strides in bytes, of dimensions 1..); false if the driver refuses it.
bool encodeTiled(
  CUtensorMap* map, int dt, const void* base, int rank, const uint64_t* dims, const uint64_t* strides, const uint32_t* box, CUtensorMapSwizzle swizzle);

// ---- y = act(x w^T + bias) + residual ----
struct MatmulArgs {
  int dt;
  int M, N, K;
  const void* x; int64_t ldx;  // [M][K]
  const void* w; int64_t ldw;  // [N][K]
  const float* bias;           // [N] or NULL
  int act;                     // KB_ACT_*
  const void* residual; int64_t ldr;  // [M][N] or NULL
  void* y; int64_t ldy;        // [M][N]
  int* status;                 // receives the code of a device-side wait that ran out
};
cudaError_t launchMatmul(cudaStream_t st, const MatmulArgs& a);
// kb_matmul_tc.cu: 16-bit types; fastest with the rows of x and w on 16-byte boundaries
bool matmulTcEligible(const MatmulArgs& a);
bool matmulTcAligned(const MatmulArgs& a);
cudaError_t launchMatmulTc(cudaStream_t st, const MatmulArgs& a);

// ---- rotary positions ----
struct RopeHeads {
  const void* in; int64_t inB, inT, inH;
  void* out; int64_t outB, outT, outH;
  int heads;  // 0: absent
};
struct RopeArgs {
  int dt, batch, tokens, dim, rot, axes, freqHeads, halves;
  const int32_t* positions; int64_t posB;
  const float* freqs;
  RopeHeads q, k;
};
cudaError_t launchRopeAxes(cudaStream_t st, const RopeArgs& a);

// ---- attention to states of another length ----
struct CrossAttnArgs {
  int dt, batch, qLen, kLen, heads, kvHeads, dq, dv;
  int planBatch;  // the batch that the cutting of rows and keys is planned for; 0: this one (the workspace is planBatch's)
  float scale;
  const void* q; int64_t qB, qT, qH;
  const void* k; int64_t kB, kT, kH;
  const void* v; int64_t vB, vT, vH;
  void* out; int64_t oB, oT, oH;
  const int32_t* qLengths;  // [batch] or NULL
  const int32_t* kLengths;  // [batch] or NULL
  const float* keyMask;     // [batch][kLen] or NULL; 0 = not attended
  const float* queryMask;   // [batch][qLen] or NULL; 0 = a row of zeros
  void* workspace;          // crossAttnWorkspace bytes
  int* status;
};
size_t crossAttnWorkspace(int dt, int batch, int qLen, int kLen, int heads, int kvHeads, int dq, int dv);
cudaError_t launchCrossAttn(cudaStream_t st, const CrossAttnArgs& a);

// ---- the entry points behind the C ABI: check, then launch; they throw on a refused argument or a failed launch ----
void opMatmul(const MatmulArgs& a, void* stream);
void opRope(RopeArgs a, const kb_view* qIn, const kb_view* qOut, const kb_view* kIn, const kb_view* kOut, void* stream);
size_t opCrossAttnWorkspace(int precision, int batch, int qLen, int kLen, int heads, int kvHeads, int qkDim, int vDim);
void opCrossAttn(CrossAttnArgs a, const kb_view* q, const kb_view* k, const kb_view* v, const kb_view* out, size_t workspaceBytes, void* stream);

}  // namespace kb

// Checks of the operators of kb_ops.h.  A call that could read or write where the caller's tensors are not, or whose result
// would depend on the order of its blocks, is refused here, before anything is launched.
#include "kb_ops.h"

#include <cuda.h>
#include <algorithm>
#include <mutex>
#include <stdexcept>
#include <string>

#include "../../include/kb_modelblob.h"
#include "kb_box.h"
#include "kb_engine.h"
#include "kb_kernels.cuh"

namespace kb {

namespace {

[[noreturn]] void refuse(const std::string& what) { throw std::runtime_error(what); }

size_t elementSize(int precision, const char* op) {
  if(precision != KB_PRECISION_FP32 && precision != KB_PRECISION_FP16 && precision != KB_PRECISION_BF16) refuse(std::string(op) + ": unknown precision " + std::to_string(precision));
  return dtypeSize(precision);
}

// Where the current device's kernels find it: device memory of this device (or managed memory).
void checkPointer(const char* op, const char* name, const void* p, size_t align) {
  auto who = [&]() { return std::string(op) + ": " + name; };
  if(p == nullptr) refuse(who() + " is NULL");
  if((uintptr_t)p % align != 0) refuse(who() + " is not aligned to its elements of " + std::to_string(align) + " bytes");
  typedef CUresult (*GetAttributesFn)(unsigned int, CUpointer_attribute*, void**, CUdeviceptr);
  static const GetAttributesFn get = []() -> GetAttributesFn {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if(cudaGetDriverEntryPoint("cuPointerGetAttributes", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) return nullptr;
    return reinterpret_cast<GetAttributesFn>(f);
  }();
  if(!get) refuse(who() + ": no CUDA device");
  unsigned int type = 0, managed = 0;
  int dev = -1, cur = -1;
  CUpointer_attribute ask[3] = {CU_POINTER_ATTRIBUTE_MEMORY_TYPE, CU_POINTER_ATTRIBUTE_IS_MANAGED, CU_POINTER_ATTRIBUTE_DEVICE_ORDINAL};
  void* into[3] = {&type, &managed, &dev};
  if(get(3, ask, into, (CUdeviceptr)(uintptr_t)p) != CUDA_SUCCESS) refuse(who() + " could not be looked up");
  if(managed) return;
  if(type != CU_MEMORYTYPE_DEVICE) refuse(who() + " is not device memory");
  cudaCheck(cudaGetDevice(&cur), "cudaGetDevice");
  if(dev != cur) refuse(who() + " lies on device " + std::to_string(dev) + ", the current device is " + std::to_string(cur));
}

constexpr int64_t MAX_STRIDE = int64_t(1) << 40, MAX_BYTES = int64_t(1) << 46;

void checkBox(const char* op, const Box& b, bool written) {
  for(int i = 0; i < 3; i++)
    if(b.s[i] < 0 || b.s[i] > MAX_STRIDE) refuse(std::string(op) + ": a stride of " + b.name + " is negative or too large");
  if(b.empty()) return;
  __int128 extent = b.width;
  for(int i = 0; i < 3; i++) extent += (__int128)(b.n[i] - 1) * b.s[i];
  if(extent * (__int128)b.elem > MAX_BYTES) refuse(std::string(op) + ": " + b.name + " is too large");
  checkPointer(op, b.name, b.p, b.elem);
  if(!written) return;
  if(overlapsItself(b)) refuse(std::string(op) + ": rows of " + b.name + " overlap one another");
}

void checkApart(const char* op, const Box& out, const Box& in) {
  if(mayOverlap(out, in)) refuse(std::string(op) + ": " + out.name + " overlaps " + in.name);
}

void checkCount(const char* op, const char* name, int64_t v, int64_t least, int64_t most) {
  if(v < least || v > most) refuse(std::string(op) + ": " + name + " is " + std::to_string(v) + ", not in " + std::to_string(least) + ".." + std::to_string(most));
}

Box boxOf(const char* name, const kb_view* v, int64_t batch, int64_t tokens, int64_t heads, int64_t width, size_t elem) {
  return Box{name, v->data, {batch, tokens, heads}, {v->batchStride, v->tokenStride, v->headStride}, width, elem};
}
void needView(const char* op, const char* name, const kb_view* v) {
  if(v == nullptr) refuse(std::string(op) + ": " + name + " is NULL");
}

// The word for the kernels of this call, after a look at what an earlier one has left there.
int* waitStatus() {
  int* word = operatorWaitWord();
  const int code = __atomic_exchange_n(word, 0, __ATOMIC_ACQ_REL);
  if(code != 0) throw CudaError("a device-side wait timed out in an earlier operator call (code " + std::to_string(code) + "): its results are not valid");
  return word;
}

void checkLaunch(const char* op, cudaError_t e) {
  if(e != cudaSuccess) {
    cudaGetLastError();
    throw CudaError(std::string(op) + ": launch failed: " + cudaGetErrorString(e));
  }
}

}  // namespace

int* operatorWaitWord() {
  static std::once_flag once;
  static int* word = nullptr;
  std::call_once(once, []() {
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaThreadExchangeStreamCaptureMode(&mode);
    void* p = nullptr;
    if(cudaHostAlloc(&p, 64, cudaHostAllocPortable | cudaHostAllocMapped) == cudaSuccess) {
      word = static_cast<int*>(p);
      *word = 0;
    }
    cudaThreadExchangeStreamCaptureMode(&mode);
  });
  if(!word) throw CudaError("page-locked memory for the status of device-side waits could not be allocated");
  return word;
}

cudaError_t SharedMemoryOptIn::operator()(const void* fn, int bytes) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if(e != cudaSuccess) return e;
  const uint64_t bit = dev < 64 ? uint64_t(1) << dev : 0;
  if(done.load(std::memory_order_acquire) & bit) return cudaSuccess;
  e = allowSharedMemory(fn, bytes);
  if(e == cudaSuccess) done.fetch_or(bit, std::memory_order_release);
  return e;
}

bool encodeTiled(
  CUtensorMap* map, int dt, const void* base, int rank, const uint64_t* dims, const uint64_t* strides, const uint32_t* box, CUtensorMapSwizzle swizzle) {
  typedef CUresult (*EncodeFn)(
    CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
    CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const EncodeFn fn = []() -> EncodeFn {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) return nullptr;
    return reinterpret_cast<EncodeFn>(p);
  }();
  if(!fn) return false;
  const CUtensorMapDataType type = dt == DT_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : (dt == DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16);
  cuuint64_t d[4], s[3];
  cuuint32_t b[4], one[4] = {1, 1, 1, 1};
  for(int i = 0; i < rank; i++) { d[i] = dims[i]; b[i] = box[i]; if(i > 0) s[i - 1] = strides[i - 1]; }
  auto encode = [&]() {
    return fn(map, type, (cuuint32_t)rank, const_cast<void*>(base), d, s, b, one, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = encode();
  // a thread that has called nothing of the runtime that needs its device has no context yet, which this call, of the driver, does not see to
  int dev = 0;
  if(r == CUDA_ERROR_INVALID_CONTEXT && cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess) r = encode();
  return r == CUDA_SUCCESS;
}

void opMatmul(const MatmulArgs& given, void* stream) {
  const char* op = "kb_matmul";
  MatmulArgs a = given;
  const size_t es = elementSize(a.dt, op);
  constexpr int64_t MOST = int64_t(1) << 30;
  checkCount(op, "m", a.M, 0, MOST);
  checkCount(op, "n", a.N, 1, MOST);
  checkCount(op, "k", a.K, 1, MOST);
  if(a.act != KB_ACT_IDENTITY && a.act != KB_ACT_RELU && a.act != KB_ACT_MISH && a.act != KB_ACT_SILU && a.act != KB_ACT_MISH_SCALE8)
    refuse("kb_matmul: unknown activation " + std::to_string(a.act));
  if(a.ldx < a.K || a.ldw < a.K) refuse("kb_matmul: a row stride of x or w is smaller than k");
  if(a.ldy < a.N || (a.residual && a.ldr < a.N)) refuse("kb_matmul: a row stride of y or the residual is smaller than n");
  if(a.M == 0) return;
  const Box x{"x", a.x, {1, a.M, 1}, {0, a.ldx, 0}, a.K, es}, w{"w", a.w, {1, a.N, 1}, {0, a.ldw, 0}, a.K, es};
  const Box y{"y", a.y, {1, a.M, 1}, {0, a.ldy, 0}, a.N, es}, r{"the residual", a.residual, {1, a.M, 1}, {0, a.ldr, 0}, a.N, es};
  const Box bias{"the bias", a.bias, {1, 1, 1}, {0, 0, 0}, a.N, 4};
  checkBox(op, x, false);
  checkBox(op, w, false);
  checkBox(op, y, true);
  checkApart(op, y, x);
  checkApart(op, y, w);
  if(a.bias) { checkBox(op, bias, false); checkApart(op, y, bias); }
  if(a.residual) {
    checkBox(op, r, false);
    if(!sameBox(y, r)) checkApart(op, y, r);
  }
  a.status = waitStatus();
  checkLaunch(op, launchMatmul(static_cast<cudaStream_t>(stream), a));
}

void opRope(RopeArgs a, const kb_view* qIn, const kb_view* qOut, const kb_view* kIn, const kb_view* kOut, void* stream) {
  const char* op = "kb_rope";
  const size_t es = elementSize(a.dt, op);
  checkCount(op, "batch", a.batch, 0, INT32_MAX);
  checkCount(op, "tokens", a.tokens, 0, INT32_MAX);
  checkCount(op, "headDim", a.dim, 2, 65536);
  checkCount(op, "rotDim", a.rot, 2, a.dim);
  if(a.rot % 2 != 0) refuse("kb_rope: rotDim is odd");
  checkCount(op, "axes", a.axes, 1, 16);
  checkCount(op, "qHeads", a.q.heads, 0, 65536);
  checkCount(op, "kHeads", a.k.heads, 0, 65536);
  checkCount(op, "freqHeads", a.freqHeads, 1, 65536);
  if(a.q.heads % a.freqHeads != 0 || a.k.heads % a.freqHeads != 0) refuse("kb_rope: freqHeads does not divide the number of heads");
  if(a.halves != 0 && a.halves != 1) refuse("kb_rope: unknown pair layout " + std::to_string(a.halves));
  if((int64_t)a.batch * a.tokens > INT32_MAX) refuse("kb_rope: more than 2^31 - 1 tokens");
  if(a.posB < 0 || a.posB > MAX_STRIDE) refuse("kb_rope: the batch stride of the positions is negative or too large");
  if(a.batch == 0 || a.tokens == 0 || a.q.heads + a.k.heads == 0) return;
  Box in[2], out[2];
  RopeHeads* heads[2] = {&a.q, &a.k};
  const kb_view* views[2][2] = {{qIn, qOut}, {kIn, kOut}};
  const char* names[2][2] = {{"q in", "q out"}, {"k in", "k out"}};
  for(int i = 0; i < 2; i++) {
    RopeHeads& h = *heads[i];
    if(h.heads == 0) { in[i].n[0] = out[i].n[0] = 0; continue; }
    needView(op, names[i][0], views[i][0]);
    needView(op, names[i][1], views[i][1]);
    in[i] = boxOf(names[i][0], views[i][0], a.batch, a.tokens, h.heads, a.dim, es);
    out[i] = boxOf(names[i][1], views[i][1], a.batch, a.tokens, h.heads, a.dim, es);
    checkBox(op, in[i], false);
    checkBox(op, out[i], true);
    if(!sameBox(in[i], out[i])) checkApart(op, out[i], in[i]);
    h.in = in[i].p; h.inB = in[i].s[0]; h.inT = in[i].s[1]; h.inH = in[i].s[2];
    h.out = const_cast<void*>(out[i].p); h.outB = out[i].s[0]; h.outT = out[i].s[1]; h.outH = out[i].s[2];
  }
  checkApart(op, out[0], in[1]);
  checkApart(op, out[1], in[0]);
  checkApart(op, out[0], out[1]);
  const Box pos{"the positions", a.positions, {a.batch, a.tokens, 1}, {a.posB, a.axes, 0}, a.axes, 4};
  const Box freqs{"the frequencies", a.freqs, {1, a.freqHeads, a.rot / 2}, {0, (int64_t)(a.rot / 2) * a.axes, a.axes}, a.axes, 4};
  checkBox(op, pos, false);
  checkBox(op, freqs, false);
  for(int i = 0; i < 2; i++) {
    checkApart(op, out[i], pos);
    checkApart(op, out[i], freqs);
  }
  waitStatus();  // its own kernels wait for nothing; what it reads may come from one that did
  checkLaunch(op, launchRopeAxes(static_cast<cudaStream_t>(stream), a));
}

static void checkAttnSizes(const char* op, int batch, int qLen, int kLen, int heads, int kvHeads, int qkDim, int vDim) {
  checkCount(op, "batch", batch, 0, INT32_MAX);
  checkCount(op, "qLen", qLen, 0, INT32_MAX);
  checkCount(op, "kLen", kLen, 0, INT32_MAX - 65536);
  checkCount(op, "kvHeads", kvHeads, 1, 65536);
  checkCount(op, "heads", heads, 1, 65536);
  if(heads % kvHeads != 0) refuse(std::string(op) + ": kvHeads does not divide heads");
  checkCount(op, "qkDim", qkDim, 1, 256);
  checkCount(op, "vDim", vDim, 1, 256);
  if((int64_t)qLen * (heads / kvHeads) > INT32_MAX - 65536) refuse(std::string(op) + ": more than 2^31 rows for one key head");
  // blocks of the smallest row tile, each sequence and key head
  if(((int64_t)qLen * (heads / kvHeads) + 15) / 16 * (int64_t)kvHeads > INT32_MAX / 8 / (batch > 0 ? batch : 1)) refuse(std::string(op) + ": too many rows for one call");
}

size_t opCrossAttnWorkspace(int precision, int batch, int qLen, int kLen, int heads, int kvHeads, int qkDim, int vDim) {
  const char* op = "kb_cross_attention_workspace";
  elementSize(precision, op);
  checkAttnSizes(op, batch, qLen, kLen, heads, kvHeads, qkDim, vDim);
  if(batch == 0 || qLen == 0) return 0;
  return crossAttnWorkspace(precision, batch, qLen, kLen, heads, kvHeads, qkDim, vDim);
}

void opCrossAttn(CrossAttnArgs a, const kb_view* q, const kb_view* k, const kb_view* v, const kb_view* out, size_t workspaceBytes, void* stream) {
  const char* op = "kb_cross_attention";
  const size_t es = elementSize(a.dt, op);
  checkAttnSizes(op, a.batch, a.qLen, a.kLen, a.heads, a.kvHeads, a.dq, a.dv);
  // (exponents are scores times scale log2(e), which has to be a number)
  if(!(a.scale > 0.0f) || a.scale > 2.35e38f) refuse("kb_cross_attention: the scale is not a positive number up to 2.35e38");
  if(a.batch == 0 || a.qLen == 0) return;
  needView(op, "q", q);
  needView(op, "k", k);
  needView(op, "v", v);
  needView(op, "out", out);
  const Box bq = boxOf("q", q, a.batch, a.qLen, a.heads, a.dq, es), bk = boxOf("k", k, a.batch, a.kLen, a.kvHeads, a.dq, es);
  const Box bv = boxOf("v", v, a.batch, a.kLen, a.kvHeads, a.dv, es), bo = boxOf("out", out, a.batch, a.qLen, a.heads, a.dv, es);
  checkBox(op, bq, false);
  checkBox(op, bk, false);
  checkBox(op, bv, false);
  checkBox(op, bo, true);
  checkApart(op, bo, bq);
  checkApart(op, bo, bk);
  checkApart(op, bo, bv);
  const int64_t queries = (int64_t)a.batch * a.qLen, keys = (int64_t)a.batch * a.kLen;
  const Box vectors[4] = {{"the query lengths", a.qLengths, {1, 1, 1}, {0, 0, 0}, a.batch, 4}, {"the key lengths", a.kLengths, {1, 1, 1}, {0, 0, 0}, a.batch, 4},
                          {"the key mask", a.keyMask, {1, 1, 1}, {0, 0, 0}, keys, 4}, {"the query mask", a.queryMask, {1, 1, 1}, {0, 0, 0}, queries, 4}};
  for(const Box& x : vectors)
    if(x.p) {
      checkBox(op, x, false);
      checkApart(op, bo, x);
    }
  const size_t need = crossAttnWorkspace(a.dt, a.batch, a.qLen, a.kLen, a.heads, a.kvHeads, a.dq, a.dv);
  if(need > 0) {
    if(workspaceBytes < need) refuse("kb_cross_attention: the workspace has " + std::to_string(workspaceBytes) + " bytes, " + std::to_string(need) + " are needed");
    checkPointer(op, "the workspace", a.workspace, 16);
    const Box ws{"the workspace", a.workspace, {1, 1, 1}, {0, 0, 0}, (int64_t)need, 1};
    checkApart(op, ws, bq);
    checkApart(op, ws, bk);
    checkApart(op, ws, bv);
    checkApart(op, ws, bo);
    for(const Box& x : vectors)
      if(x.p) checkApart(op, ws, x);
  }
  a.q = q->data; a.qB = q->batchStride; a.qT = q->tokenStride; a.qH = q->headStride;
  a.k = k->data; a.kB = k->batchStride; a.kT = k->tokenStride; a.kH = k->headStride;
  a.v = v->data; a.vB = v->batchStride; a.vT = v->tokenStride; a.vH = v->headStride;
  a.out = out->data; a.oB = out->batchStride; a.oT = out->tokenStride; a.oH = out->headStride;
  a.status = waitStatus();
  checkLaunch(op, launchCrossAttn(static_cast<cudaStream_t>(stream), a));
}

}  // namespace kb

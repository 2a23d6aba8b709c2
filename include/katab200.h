/* C ABI of libkatab200.so: the B200 (sm_100a) implementation of the KataGo neural-net
 * forward pass that sits below the reference's backend interface
 * (cpp/neuralnet/nninterface.h:32-182).  The reference-side backend
 * (katago_b200/host/b200backend.cpp) and the Python harness (katago_b200/capi.py) both
 * bind exactly these entry points.
 *
 * Conventions: plain pointers and sizes only; every function returns 0 on success and a
 * non-zero code on failure, never throws; the message of the last failure on the calling
 * thread is available from kb_last_error().  A kb_handle is bound to one GPU and must be
 * used by one thread at a time (nninterface.h:19-21).  There is no CPU fallback: without
 * a CUDA device every compute entry point fails.
 */
#ifndef KATAB200_H_
#define KATAB200_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct kb_model kb_model;   /* parsed network, host memory, device independent */
typedef struct kb_handle kb_handle; /* one GPU replica: device weights, activations, stream */

enum { KB_PRECISION_FP32 = 0, KB_PRECISION_FP16 = 1, KB_PRECISION_BF16 = 2 };

/* Message of the last failure on the calling thread (never NULL). */
const char* kb_last_error(void);

/* Library version string. */
const char* kb_version(void);

/* Replaces NeuralNet::printDevices / device selection (nninterface.h:39, cudabackend.cpp:3333). */
int kb_device_count(int* count);
int kb_device_name(int device, char* buf, size_t buflen);

/* Replaces the construction of the backend's Model from a ModelDesc
 * (nninterface.h:43-46 loadModelFile/getModelDesc feed it; cudabackend.cpp:2852-2963).
 * `blob` is the record stream of include/kb_modelblob.h. */
int kb_model_create(const void* blob, size_t nbytes, kb_model** out);
void kb_model_destroy(kb_model* m);

/* info[0..8] = modelVersion, inC, inGlobalC, policyC, valueC, scoreValueC, ownershipC, trunkC, numBlocks */
int kb_model_info(const kb_model* m, int32_t info[9]);
/* Number of SGF metadata input channels (ModelDesc::numInputMetaChannels, desc.h; 0 for nets without the encoder). */
int kb_model_meta_channels(const kb_model* m, int32_t* channels);

/* Replaces NeuralNet::createComputeHandle / freeComputeHandle (nninterface.h:76-86):
 * binds the calling thread to `device` (-1 = current default), uploads the weights in the
 * chosen precision and allocates every activation buffer for batches up to maxBatch.
 * requireExactNNLen != 0 promises that every board is exactly nnXLen x nnYLen. */
int kb_handle_create(
  const kb_model* m, int device, int maxBatch, int nnXLen, int nnYLen, int precision, int requireExactNNLen,
  kb_handle** out);
void kb_handle_destroy(kb_handle* h);

/* Device-side weight cache.  The reference's CPU backend shares one Model between all compute handles of a net,
 * keyed by name and hash (eigenbackend.cpp:2364-2392), so that several server threads cost one copy of the weights;
 * here every read-only weight tensor is keyed by device and contents, reference counted, and freed with the last
 * handle that uses it: handles created from the same model on the same device hold one replica between them.
 * stats[0..3] = live entries, their bytes, uploads made, uploads avoided (since the process started, all devices). */
int kb_weight_cache_stats(int64_t stats[4]);

/* The tile plan of a tensor-core convolution kY x kX = k x k, inC -> outC (inC as the device sees it: padded to a multiple
 * of 64).  Replaces the OpenCL backend's start-up autotuner (cpp/neuralnet/opencltuner.cpp) by a committed table
 * (katago_b200/csrc/kb_tile_table.h).  Host-only.  plan[0..5] = channels per tile (N of the MMA), CTA pairs (0/1), epilogue
 * warps per TMEM lane quarter without / with a residual, multi-layer launches (0/1), 1 if the shape has a row in the table
 * (0: fallback rules). */
int kb_tile_plan(int k, int inC, int outC, int32_t plan[6]);
/* Number of rows of the tile table; row i as rows[i*8 .. i*8+7] = k, inC, outC, then the plan fields of kb_tile_plan in
 * order (without the last).  Fills at most cap rows. */
int kb_tile_table(int32_t* rows, int cap, int32_t* count);

/* Self-test of the failure path of the bounded device-side waits (no counterpart in the reference): on the handle's
 * stream a kernel waits limitNs nanoseconds (at most 1e9) on a barrier that nothing arrives at, gives up and records a
 * status code, exactly as a convolution kernel does when one of its waits runs out.  The call then synchronises and
 * returns the resulting error (non-zero, "a device-side wait timed out ..."); the handle stays usable. */
int kb_selftest_wait_timeout(kb_handle* h, unsigned long long limitNs);

/* Replaces NeuralNet::isUsingFP16 (nninterface.h:88): returns the precision in *precision. */
int kb_handle_precision(const kb_handle* h, int* precision);

/* Replaces the device part of NeuralNet::getOutput (nninterface.h:117-123; cudabackend.cpp:3556-3795):
 * host buffers in, host buffers out, synchronous.
 *   spatial  [n][nnYLen][nnXLen][inC] fp32 NHWC, as filled by NNEvaluator (not yet symmetrised)
 *   global   [n][inGlobalC] fp32
 *   symmetry [n] values 0..7 (SymmetryHelpers, nninputs.cpp:529-597) or NULL for identity; applied to the
 *            inputs on the device and inverted on policy/ownership outputs
 * Outputs are raw logits (nninterface.h:116); any output pointer may be NULL:
 *   policy [n][nnYLen*nnXLen][policyC], policyPass [n][policyC], value [n][valueC],
 *   scoreValue [n][scoreValueC], ownership [n][nnYLen*nnXLen]. */
int kb_forward_host(
  kb_handle* h, int n, const float* spatial, const float* global, const int32_t* symmetry,
  float* policy, float* policyPass, float* value, float* scoreValue, float* ownership);

/* The same for nets with an SGF metadata encoder (NNResultBuf::rowMetaBuf / hasRowMeta, nninputs.h; eigenbackend.cpp
 * 2458-2471): meta is [n][metaChannels] fp32 and must be non-NULL exactly when the model has the encoder. */
int kb_forward_host_meta(
  kb_handle* h, int n, const float* spatial, const float* global, const float* meta, const int32_t* symmetry,
  float* policy, float* policyPass, float* value, float* scoreValue, float* ownership);
int kb_upload_inputs_meta(kb_handle* h, int n, const float* spatial, const float* global, const float* meta, const int32_t* symmetry);

/* The three stages of kb_forward_host as separate calls, for measurements with the inputs
 * already resident in device memory: upload (host->device, asynchronous on the handle's stream),
 * run (all kernels of one forward pass), download (device->host, synchronises). */
int kb_upload_inputs(kb_handle* h, int n, const float* spatial, const float* global, const int32_t* symmetry);
int kb_forward_resident(kb_handle* h, int n);
int kb_download_outputs(
  kb_handle* h, int n, float* policy, float* policyPass, float* value, float* scoreValue, float* ownership);

/* Runs `iters` forward passes on resident inputs and returns the mean device time of one pass
 * in milliseconds, measured with CUDA events on the handle's stream. */
int kb_time_forward_resident(kb_handle* h, int n, int iters, float* msPerIter);

/* Times `steps` forward passes one by one: before each pass `flushBytes` bytes of scratch device memory are
 * overwritten (0 = no flush) so that the pass starts with a cold L2; the pass itself is bracketed by its own pair
 * of CUDA events on the handle's stream.  msEach[i] receives the device time of pass i in milliseconds. */
int kb_time_forward_steps(kb_handle* h, int n, int steps, size_t flushBytes, float* msEach);

/* Per-kernel-class device timing.  When enabled, every launch of kb_forward_resident is bracketed
 * by CUDA events on the handle's stream; kb_profile_read synchronises and returns, for up to `cap`
 * kernel classes, the class name (<=47 chars), number of launches and total milliseconds since the
 * last reset, and per-class algorithmic flops and bytes summed over those launches. */
typedef struct kb_profile_entry {
  char name[48];
  int64_t launches;
  double ms;
  double flops;
  double bytes;
} kb_profile_entry;
int kb_profile_enable(kb_handle* h, int enabled);
int kb_profile_reset(kb_handle* h);
int kb_profile_read(kb_handle* h, kb_profile_entry* entries, int cap, int* count);

/* Number of kernel launches one forward pass of batch n issues (for the harness's launch count). */
int kb_launches_per_forward(const kb_handle* h, int n, int* launches);

/* Trunk output after the final norm+activation, [n][nnYLen*nnXLen][trunkC] fp32 (debugging aid;
 * mirrors the reference's DEBUG_INTERMEDIATE_VALUES dumps, cudabackend.cpp:46). */
int kb_debug_read_trunk(kb_handle* h, int n, float* trunkOut);

/* Page-locked host memory for the staging buffers the caller fills (replaces the plain `new float[]`
 * staging of the reference's InputBuffers, cudabackend.cpp:3438-3551): copies from/to such memory are
 * asynchronous DMA transfers.  Usable from any thread, with or without a bound device. */
int kb_host_alloc(size_t bytes, void** out);
void kb_host_free(void* p);

/* Replaces NeuralNet::testEvaluateConv / BatchNorm / ResidualBlock / GlobalPoolingResidualBlock
 * (nninterface.h:134-180).  The blob holds one CONV, BN, BLOCK_ORDINARY or BLOCK_GPOOL construct.
 * in [n][Y][X][inC] NHWC fp32, mask [n][Y][X] (may be NULL for CONV), out [n][Y][X][outC]. */
int kb_eval_layer(
  const void* blob, size_t nbytes, int device, int precision, int n, int nnXLen, int nnYLen,
  const float* in, const float* mask, float* out);

/* Convolution without any allocation.  (No counterpart in the reference: its backends allocate freely.)
 *
 * For callers that may not allocate device memory themselves or through this library: plug-ins living inside a
 * host application's memory pool, or latency-critical loops that cannot afford the locks and the implicit
 * synchronisation of cudaMalloc/cudaFree.  The caller passes DEVICE pointers it already owns; the working
 * memory the convolution needs (padded copies of input and output, re-ordered weights) is a fixed 2.4 MiB array
 * inside the library's device image, present on every GPU that loads the library until the process exits.
 *
 *   dIn      [n][nnYLen][nnXLen][inC] fp32 NHWC     dWeights [outC][inC][kY][kX] fp32 (ConvLayerDesc order, desc.h:23)
 *   dOut     [n][nnYLen][nnXLen][outC] fp32 NHWC    stream   a cudaStream_t (NULL = default stream)
 * Computes the same zero-padded stride-1 cross-correlation as kb_eval_layer does for a CONV record in fp32.
 * The kernels are enqueued on `stream`; the call returns without waiting for them.
 *
 * Limits (exceeding one is an error, nothing is launched): n*(nnYLen+1)*(nnXLen+1) rounded up to a multiple of 256 <= 4096 rows
 * (10 boards of 19x19), inC <= 64, outC <= 64, kernel at most 5x5 and odd.
 * The first call on each device looks up the array's device address (with that device current); make that
 * call before starting any stream capture.  All calls share the one array and it keeps the previous call's
 * contents: two calls whose kernels overlap on the GPU (different streams, different threads) race on it.
 * The call itself performs no cudaMalloc, cudaFree or other allocating routine. */
int kb_conv_noalloc(
  const float* dIn, const float* dWeights, float* dOut, int n, int nnXLen, int nnYLen, int inC, int outC, int kY, int kX,
  void* stream);
/* Message of the last kb_conv_noalloc failure on the calling thread. */
const char* kb_conv_noalloc_last_error(void);

/* Transformer operators on the caller's own device buffers.  (No counterpart in the reference: there they exist inside a net
 * only.)  Together they are a block whose tokens look at states of another length: project, rotate, attend, project again.
 *
 * Conventions of all of them:
 *   - pointers are DEVICE addresses on the current device (managed memory is taken too); host memory and memory of another
 *     device are refused.  Elements have the type that `precision` (KB_PRECISION_*) names, sums are held in fp32, a result is
 *     rounded once (attention of 16-bit types also rounds a key's weight to 16 bits before it meets the value; the total of the
 *     weights takes them unrounded);
 *   - strides count elements and may be anything from 0 up for inputs (0 repeats; the row strides of kb_matmul are at least a
 *     row's length); the innermost dimension is contiguous;
 *     elements of an output must not coincide, and an output must not overlap an input or another output unless the text below
 *     allows it.  Column ranges of one buffer do not overlap if the tensors have the same row stride; tensors interleaved in some
 *     other way are refused, since that cannot be told from an overlap;
 *   - any alignment of the element type is taken; rows that start on 16-byte boundaries are fastest;
 *   - the kernels are enqueued on `stream` (a cudaStream_t of the current device, NULL = its default stream) and the call
 *     returns without waiting.  Calls may be captured into a graph (on memory that exists by then: what cudaMallocAsync gives within
 *     the capture is not device memory yet, and is refused), and made from several threads at once on different buffers;
 *   - nothing is allocated and nothing kept from one call to the next (but a status word for the library, at the first call);
 *   - non-zero and kb_last_error() as everywhere; a refused call has launched nothing.  A device-side wait that ran out (it never
 *     does in sound operation) is reported by the next call of an operator.
 * The same call on the same inputs gives the same bits. */

/* Elements [batch][token][head][channel]; the channel is contiguous, the strides are in elements. */
typedef struct kb_view {
  void* data;
  int64_t batchStride, tokenStride, headStride;
} kb_view;

/* y = act(x w^T + bias) + residual, the product of a projection or one half of a feed-forward layer.
 *   x [m][k], rows ldx apart      w [n][k], rows ldw apart (the order of a tensor-core convolution's weights, outC x inC)
 *   bias [n] fp32 or NULL         residual [m][n], rows ldr apart, or NULL
 *   y [m][n], rows ldy apart      act a KB_ACT_* of kb_modelblob.h
 * The residual may be y itself (same address, same stride).  m may be 0; m, n and k are at most 2^30. */
int kb_matmul(
  int precision, int m, int n, int k, const void* x, int64_t ldx, const void* w, int64_t ldw, const float* bias, int act,
  const void* residual, int64_t ldr, void* y, int64_t ldy, void* stream);

/* Rotary positions with any number of axes (time, row, column): pair p of a head is turned by
 *   angle[b][t][p] = sum over a of positions[b][t][a] * freqs[table][p][a]     (x0, x1) -> (x0 cos - x1 sin, x0 sin + x1 cos)
 *   positions [batch][tokens][axes] int32, sequences posBatchStride apart (0: all have the same).  Any value: what counts is the
 *             angle's fraction of a turn, which is off by no more than an fp32 rounding of it (2^-26 of a turn, and 2^-33 per axis) at the
 *             farthest position as at the nearest, for frequencies up to 2^40
 *   freqs     [freqHeads][rotDim/2][axes] fp32, radians per step; head h of H uses table h*freqHeads/H (freqHeads divides qHeads
 *             and kHeads).  A pair that turns with one axis has zeros for the others
 *   pairsInHalves 0: pair p is channels 2p, 2p+1 (as in the nets of this library); 1: channels p, p + rotDim/2
 * The first rotDim of a head's headDim channels are turned, the others copied.  q and k are turned in one call; either may be
 * absent (0 heads, views NULL).  An output may be its own input (same view: in place). */
int kb_rope(
  int precision, int batch, int tokens, int headDim, int rotDim, const int32_t* positions, int64_t posBatchStride, int axes,
  const float* freqs, int freqHeads, int pairsInHalves, const kb_view* qIn, const kb_view* qOut, int qHeads, const kb_view* kIn,
  const kb_view* kOut, int kHeads, void* stream);

/* Attention of qLen tokens to the kLen states of another sequence (or of their own):
 *   out[b][i][h] = sum over j of p[j] v[b][j][g],  p = softmax over j of scale * q[b][i][h] . k[b][j][g],  g = h*kvHeads/heads
 *   q [batch][qLen][heads][qkDim]   k [batch][kLen][kvHeads][qkDim]   v [batch][kLen][kvHeads][vDim]
 *   out [batch][qLen][heads][vDim]  head sizes 1..256, heads a multiple of kvHeads, scale > 0 and at most 2.35e38
 *   qLengths, kLengths [batch] int32 on the device or NULL: rows of `out` from qLengths[b] on are left as they are; keys from
 *             kLengths[b] on are left out, whatever they hold.  Values outside 0..qLen / 0..kLen count as the nearer end
 *   keyMask   [batch][kLen] fp32 or NULL: keys whose mask is 0 are left out, whatever their k and v hold (NaN and Inf included)
 *   queryMask [batch][qLen] fp32 or NULL: tokens whose mask is 0 get a row of zeros
 * A row that no key is left for is zeros, and so is one all of whose scores are -infinity; one with a score that is NaN or +infinity is NaN.
 *   workspace, workspaceBytes: device memory, 16-byte aligned, at least what kb_cross_attention_workspace says for the same sizes
 *             (it depends on nothing else; 0 for most).  Its contents need not be set and mean nothing after the call; two
 *             calls whose kernels overlap on the GPU (two streams, two graphs) need one each. */
int kb_cross_attention_workspace(
  int precision, int batch, int qLen, int kLen, int heads, int kvHeads, int qkDim, int vDim, size_t* bytes);
int kb_cross_attention(
  int precision, int batch, int qLen, int kLen, int heads, int kvHeads, int qkDim, int vDim, float scale, const kb_view* q,
  const kb_view* k, const kb_view* v, const kb_view* out, const int32_t* qLengths, const int32_t* kLengths, const float* keyMask,
  const float* queryMask, void* workspace, size_t workspaceBytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* KATAB200_H_ */

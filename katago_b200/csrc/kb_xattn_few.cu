// Attention of few rows (up to 16 of a key head: one new token of grouped heads) to states of another length: fp16 / bf16, head
// sizes up to 128 in multiples of 8, rows on 16-byte boundaries.
//
// What bounds it: memory, K and V are read once.  A block has a range of keys, its warps every eighth group of 16 keys of it.  A
// warp streams its own groups through a ring of its own with cp.async (no barrier of the block while it runs), multiplies the 16
// rows with the group by mma.sync, keeps a running maximum, sum and output per row in registers, and the probabilities never
// leave registers: an accumulator's layout is that of the next product's first operand.  At the end the warps' states, and
// with the keys cut over several blocks the blocks' (kb_xattn.cu), are added in the order of the keys' groups.
//
// Keys that are not attended: scores of -inf, and their rows of V are cleared in shared memory (0 times an infinity is a NaN).
#include "kb_kernels.cuh"
#include "kb_ops.h"
#include "kb_ops_dev.cuh"
#include "kb_xattn.cuh"

#include <algorithm>

namespace kb {

namespace {

constexpr int XF_WARPS = 8, XF_THREADS = 32 * XF_WARPS, XF_GROUP = 16;

template <int D> struct XfShape {
  static constexpr int STAGES = D == 64 ? 4 : 3;
  static constexpr int STAGE_BYTES = 2 * XF_GROUP * D * 2 + XF_GROUP * 4;  // K, V, masks of a group
  static constexpr int SMEM = XF_WARPS * STAGES * STAGE_BYTES;
  static constexpr int BLOCKS = D == 64 ? 2 : 1;
};

template <typename T> __device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if(std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldMatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldMatrix4Trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void cpAsync16(uint32_t dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(in ? 16 : 0) : "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(XF_THREADS, XfShape<D>::BLOCKS) crossAttnFewKernel(const CrossAttnArgs a, const XaSplit sp) {
  typedef XfShape<D> Sh;
  extern __shared__ float4 smem4[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(smem4);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const XaBlock blk = xaBlock(a, sp, 16);
  const int G = a.heads / a.kvHeads;
  gridDepLaunch();
  gridDepWait();
  const int rows = xaRows(a, blk.b, G), keys = xaKeys(a, blk.b);
  const int k0 = blk.part * sp.chunk, k1 = (int)min((long long)keys, (long long)k0 + sp.chunk);
  if(rows == 0 || (blk.part > 0 && k0 >= keys)) return;  // part 0 reports a row without keys
  const int groups = k1 > k0 ? (k1 - k0 + XF_GROUP - 1) / XF_GROUP : 0;
  const int mine = groups > warp ? (groups - warp + XF_WARPS - 1) / XF_WARPS : 0;  // groups warp, warp + 8, ...
  uint8_t* ring = smem + warp * Sh::STAGES * Sh::STAGE_BYTES;
  const T* kBase = (const T*)a.k + blk.b * a.kB + blk.kvh * a.kH;
  const T* vBase = (const T*)a.v + blk.b * a.vB + blk.kvh * a.vH;
  constexpr int CH = D / 8, PER = XF_GROUP * CH / 32;  // 16-byte pieces of a row; of a group per lane

  auto request = [&](int i) {
    const int first = k0 + (warp + i * XF_WARPS) * XF_GROUP;
    const uint32_t at = smemU32(ring + (i % Sh::STAGES) * Sh::STAGE_BYTES);
#pragma unroll
    for(int p = 0; p < PER; p++) {
      const int piece = p * 32 + lane, r = piece / CH, c = piece % CH, key = first + r;
      const uint32_t to = at + (uint32_t)(r * D * 2 + ((c ^ (r & 7)) << 4));
      const bool inK = key < k1 && c * 8 < a.dq, inV = key < k1 && c * 8 < a.dv;
      cpAsync16(to, inK ? kBase + key * a.kT + c * 8 : (const T*)a.q, inK);
      cpAsync16(to + XF_GROUP * D * 2, inV ? vBase + key * a.vT + c * 8 : (const T*)a.q, inV);
    }
    if(a.keyMask && lane < XF_GROUP) {
      const bool in = first + lane < k1;
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(at + 2 * XF_GROUP * D * 2 + lane * 4),
                   "l"(in ? a.keyMask + (int64_t)blk.b * a.kLen + first + lane : (const float*)a.q), "r"(in ? 4 : 0) : "memory");
    }
  };
#pragma unroll
  for(int i = 0; i < Sh::STAGES - 1; i++) {
    if(i < mine) request(i);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // Q as the first operand: rows g and g + 8, channel pairs 2t and 2t + 8 of every 16
  uint32_t q[D / 16][4];
  {
    const int r0 = g, r1 = g + 8;
    const T* q0 = (const T*)a.q + blk.b * a.qB + (r0 / G) * a.qT + (blk.kvh * G + r0 % G) * a.qH;
    const T* q1 = (const T*)a.q + blk.b * a.qB + (r1 / G) * a.qT + (blk.kvh * G + r1 % G) * a.qH;
#pragma unroll
    for(int k = 0; k < D / 16; k++)
#pragma unroll
      for(int h = 0; h < 2; h++) {
        const int d = k * 16 + h * 8 + 2 * t;
        q[k][2 * h] = r0 < rows && d < a.dq ? *reinterpret_cast<const uint32_t*>(q0 + d) : 0u;
        q[k][2 * h + 1] = r1 < rows && d < a.dq ? *reinterpret_cast<const uint32_t*>(q1 + d) : 0u;
      }
  }
  float o[D / 8][4];
#pragma unroll
  for(int n = 0; n < D / 8; n++)
#pragma unroll
    for(int e = 0; e < 4; e++) o[n][e] = 0.0f;
  float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
  const float scale = a.scale * 1.4426950408889634f;
  // Weights are at most 1, of the type of the product's operands.  In fp16 they are 2^15 times larger, and so are the sums that they cancel in: those
  // that are 2^-29 of the maximum's still have all their bits.  (bf16 has the range of fp32.)
  constexpr float UP = std::is_same<T, __half>::value ? 15.0f : 0.0f;

  for(int i = 0; i < mine; i++) {
    asm volatile("cp.async.wait_group %0;" ::"n"(Sh::STAGES - 2) : "memory");
    __syncwarp();  // every lane's pieces are there, and every lane is done with the stage that is requested next
    if(i + Sh::STAGES - 1 < mine) request(i + Sh::STAGES - 1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    uint8_t* stage = ring + (i % Sh::STAGES) * Sh::STAGE_BYTES;
    const uint32_t sK = smemU32(stage), sV = sK + XF_GROUP * D * 2;
    const int first = k0 + (warp + i * XF_WARPS) * XF_GROUP;
    const float* masks = reinterpret_cast<const float*>(stage + 2 * XF_GROUP * D * 2);
    const uint32_t on = __ballot_sync(0xffffffffu, lane < XF_GROUP && first + lane < k1 && (!a.keyMask || masks[lane & 15] != 0.0f));
    if(on != 0xffffu) {
      if(on == 0u) continue;
      for(int r = 0; r < XF_GROUP; r++)
        if(((on >> r) & 1u) == 0u && lane < CH) *reinterpret_cast<uint4*>(stage + XF_GROUP * D * 2 + r * D * 2 + lane * 16) = make_uint4(0u, 0u, 0u, 0u);
      __syncwarp();
    }
    // scores: keys 0-7 and 8-15 of the group
    float s[2][4];
#pragma unroll
    for(int n = 0; n < 2; n++)
#pragma unroll
      for(int e = 0; e < 4; e++) s[n][e] = 0.0f;
    const int lr = (lane & 7) + ((lane >> 4) << 3), lc = (lane >> 3) & 1;  // row and piece of this lane's address for K
#pragma unroll
    for(int k = 0; k < D / 16; k++) {
      uint32_t b[4];  // pairs (keys 0-7: channels 0-7, 8-15), (keys 8-15: ...)
      ldMatrix4(sK + (uint32_t)(lr * D * 2 + (((2 * k + lc) ^ (lr & 7)) << 4)), b);
      mma16816<T>(s[0], q[k], b[0], b[1]);
      mma16816<T>(s[1], q[k], b[2], b[3]);
    }
    float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for(int n = 0; n < 2; n++)
#pragma unroll
      for(int e = 0; e < 4; e++) {
        s[n][e] = (on >> (n * 8 + 2 * t + (e & 1))) & 1u ? s[n][e] * scale : -INFINITY;
        top[e >> 1] = fmaxf(top[e >> 1], s[n][e]);
      }
#pragma unroll
    for(int h = 0; h < 2; h++) {
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 1));
      top[h] = fmaxf(top[h], __shfl_xor_sync(0xffffffffu, top[h], 2));
    }
    if(__any_sync(0xffffffffu, top[0] > mx[0] || top[1] > mx[1])) {
      float keep[2];
#pragma unroll
      for(int h = 0; h < 2; h++) {
        const float now = fmaxf(mx[h], top[h]);
        keep[h] = now == -INFINITY ? 1.0f : exp2f(mx[h] - now);
        mx[h] = now;
        sum[h] *= keep[h];
      }
#pragma unroll
      for(int n = 0; n < D / 8; n++)
#pragma unroll
        for(int e = 0; e < 4; e++) o[n][e] *= keep[e >> 1];
    }
    const float ref[2] = {mx[0] == -INFINITY ? 0.0f : mx[0], mx[1] == -INFINITY ? 0.0f : mx[1]};
#pragma unroll
    for(int n = 0; n < 2; n++)
#pragma unroll
      for(int e = 0; e < 4; e++) {
        s[n][e] = ex2Approx(s[n][e] - ref[e >> 1] + UP);
        sum[e >> 1] += s[n][e];  // this lane's keys
      }
    const uint32_t p[4] = {opPack<T>(s[0][0], s[0][1]), opPack<T>(s[0][2], s[0][3]), opPack<T>(s[1][0], s[1][1]), opPack<T>(s[1][2], s[1][3])};
    const int vr = lane & 15, vc = lane >> 4;  // key and piece of this lane's address for V
#pragma unroll
    for(int n = 0; n < D / 16; n++) {
      uint32_t b[4];  // channels 0-7: keys 0-7, 8-15; channels 8-15: ...
      ldMatrix4Trans(sV + (uint32_t)(vr * D * 2 + (((2 * n + vc) ^ (vr & 7)) << 4)), b);
      mma16816<T>(o[2 * n], p, b[0], b[1]);
      mma16816<T>(o[2 * n + 1], p, b[2], b[3]);
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
  for(int h = 0; h < 2; h++) {
    sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
    sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
  }
  // The warps' states side by side in the place of the rings: [warp][row][D], [warp][row] maximum and sum.
  constexpr int PITCH = D + 4;
  float* sO = reinterpret_cast<float*>(smem);
  float* sM = sO + XF_WARPS * 16 * PITCH;
  float* sS = sM + XF_WARPS * 16;
  static_assert((XF_WARPS * 16 * PITCH + 2 * XF_WARPS * 16) * 4 <= Sh::SMEM, "the states fit the rings' place");
  __syncthreads();
#pragma unroll
  for(int n = 0; n < D / 8; n++)
#pragma unroll
    for(int h = 0; h < 2; h++)
      *reinterpret_cast<float2*>(sO + (warp * 16 + g + 8 * h) * PITCH + n * 8 + 2 * t) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
  if(t == 0)
#pragma unroll
    for(int h = 0; h < 2; h++) { sM[warp * 16 + g + 8 * h] = mx[h]; sS[warp * 16 + g + 8 * h] = sum[h]; }
  __syncthreads();
  for(int r = warp; r < min(16, rows); r += XF_WARPS) {
    float top = -INFINITY, total = 0.0f, w[XF_WARPS];
#pragma unroll
    for(int i = 0; i < XF_WARPS; i++) top = fmaxf(top, sM[i * 16 + r]);
    const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
    for(int i = 0; i < XF_WARPS; i++) {
      w[i] = exp2f(sM[i * 16 + r] - ref);
      total += w[i] * sS[i * 16 + r];
    }
    float* part = sp.parts > 1 ? xaPart(a, sp, blk, r, G) : nullptr;
    T* out = (T*)a.out + blk.b * a.oB + (r / G) * a.oT + (blk.kvh * G + r % G) * a.oH;
    const bool live = total != 0.0f && (!a.queryMask || a.queryMask[(int64_t)blk.b * a.qLen + r / G] != 0.0f);
    const float inv = 1.0f / total;
    if(part && lane == 0) { part[0] = top; part[1] = total; }
    for(int d = lane * 2; d < a.dv; d += 64) {
      float2 v = make_float2(0.0f, 0.0f);
#pragma unroll
      for(int i = 0; i < XF_WARPS; i++) {
        const float2 x = *reinterpret_cast<const float2*>(sO + (i * 16 + r) * PITCH + d);
        v.x = fmaf(w[i], x.x, v.x);
        v.y = fmaf(w[i], x.y, v.y);
      }
      if(part) *reinterpret_cast<float2*>(part + 2 + d) = v;
      else *reinterpret_cast<uint32_t*>(out + d) = live ? opPack<T>(v.x * inv, v.y * inv) : 0u;
    }
  }
}

template <typename T, int D> cudaError_t launchFew(cudaStream_t st, const CrossAttnArgs& a, const XaSplit& sp) {
  static SharedMemoryOptIn optIn;
  const cudaError_t e = optIn((const void*)crossAttnFewKernel<T, D>, XfShape<D>::SMEM);
  if(e != cudaSuccess) return e;
  return launchDependent(crossAttnFewKernel<T, D>, dim3(sp.blocks), dim3(XF_THREADS), (size_t)XfShape<D>::SMEM, st, a, sp);
}

}  // namespace

XaSplit crossAttnFewSplit(int batch, int qLen, int kLen, int heads, int kvHeads, int dq, int dv) {
  return xaPlanSplit(16, XF_WARPS * XF_GROUP, 2048, dq <= 64 && dv <= 64 ? XfShape<64>::BLOCKS : XfShape<128>::BLOCKS, batch, qLen, kLen, heads, kvHeads, dv);
}

cudaError_t launchCrossAttnFew(cudaStream_t st, const CrossAttnArgs& a, const XaSplit& sp) {
  const bool wide = a.dq > 64 || a.dv > 64;
  if(a.dt == DT_F16) return wide ? launchFew<__half, 128>(st, a, sp) : launchFew<__half, 64>(st, a, sp);
  return wide ? launchFew<__nv_bfloat16, 128>(st, a, sp) : launchFew<__nv_bfloat16, 64>(st, a, sp);
}

}  // namespace kb

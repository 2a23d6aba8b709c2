// y = act(x w^T + bias) + residual on a caller's own matrices: fp32, and the kernels for few rows of any type.  (More rows of 16-bit
// types: kb_matmul_tc.cu.)
//
// matmulF32Kernel    fp32: one tile of BM x BN outputs per block, slices of 32 channels through three stages of asynchronous copies
//                    (16 bytes, or 4 where rows lie anywhere).  FMA-bound.  A thread reads four channels of a row at a time and
//                    sums even and odd channels apart with the packed fp32 instructions (two IEEE operations per issue slot, no
//                    operand has to be doubled); the two are added at the end.
// matmulFewKernel    up to eight rows: memory-bound, the weights are read once.  A block has four weight rows and cuts K
//                    over its warps, whose sums are added in warp order.
// matmulFewMmaKernel the same for up to 16 rows of 16-bit types and K up to 1024, where a launch's latency is what counts.
//                    mma.sync takes 16 weight rows against 8 rows of x.  Operands go from memory to registers, 16 bytes
//                    per lane: the sum over K may be taken in any order, so the lane that has channels 8t..8t+7 of a weight row
//                    feeds them as four pairs wherever the instruction wants pairs, and the lane of a row of x does the same.
//                    4 x 1024 x 384 bf16: 2.1 us, 4.0 us in kb_matmul_tc.cu; the two meet at 4 x 16384 x 512 (4.9 us), and longer
//                    sums are better off with asynchronous copies (4 x 4096 x 4096: 12.8 us here, 9.2 us there).
#include "kb_kernels.cuh"
#include "kb_ops.h"
#include "kb_ops_dev.cuh"

#include <algorithm>

namespace kb {

namespace {

template <typename T>
__device__ __forceinline__ void matmulStore(const MatmulArgs& a, int m, int n, float v) {
  if(a.bias) v += a.bias[n];
  v = opAct<T>(v, a.act);
  if(a.residual) v += OpType<T>::to(((const T*)a.residual)[(int64_t)m * a.ldr + n]);
  ((T*)a.y)[(int64_t)m * a.ldy + n] = OpType<T>::from(v);
}

// TM x TN outputs per thread: a shared-memory load of 16 bytes per lane is three passes of the shared memory whatever lanes it
// repeats for, so eight by eight outputs (16 loads for 128 packed FMAs) are needed for the FMA units to be what bounds it.  KG: groups
// of threads that share a slice's channels and add their sums in order at the end, so that a small tile has threads of that kind
// enough (1083 x 362 x 361, 64 x 48 tiles, one to an SM: 26 us with 4 x 3 outputs from 256 threads, 19 us from 1024).
// VEC: rows on 16-byte boundaries and K in whole vectors.
template <int BM, int BN, int TM, int TN, int KG, bool VEC>
__global__ void __launch_bounds__(BM / TM * (BN / TN) * KG) matmulF32Kernel(const MatmulArgs a) {
  constexpr int BK = 32, PITCH = BK + 4, STAGES = 3;  // 8 rows of 144 bytes start in 8 different bank groups
  constexpr int TX = BN / TN, TY = BM / TM, GROUP = TX * TY, THREADS = GROUP * KG;
  static_assert(GROUP % 32 == 0 && TX % 8 == 0 && TY % 4 == 0 && BK % (4 * KG) == 0, "a warp is four rows by eight columns of one group");
  extern __shared__ float4 smem4[];
  float* sm = reinterpret_cast<float*>(smem4);
  const int tid = threadIdx.x, kg = tid / GROUP, warp = (tid % GROUP) >> 5, lane = tid & 31;
  const int tx = warp % (TX / 8) * 8 + (lane & 7), ty = warp / (TX / 8) * 4 + (lane >> 3);
  const int tilesN = (a.N + BN - 1) / BN;
  const int m0 = (int)(blockIdx.x / tilesN) * BM, n0 = (int)(blockIdx.x % tilesN) * BN;
  const float* x = (const float*)a.x;
  const float* w = (const float*)a.w;
  gridDepLaunch();
  gridDepWait();
  const int steps = (a.K + BK - 1) / BK;
  auto load = [&](int s) {
    float* dst = sm + (s % STAGES) * (BM + BN) * PITCH;
    constexpr int E = VEC ? 4 : 1, PER = BK / E;
#pragma unroll
    for(int i = tid; i < (BM + BN) * PER; i += THREADS) {
      const int r = i / PER, k = s * BK + (i % PER) * E;
      const bool isX = r < BM;
      const int row = isX ? m0 + r : n0 + r - BM;
      const bool in = k < a.K && row < (isX ? a.M : a.N);
      const float* src = in ? (isX ? x + (int64_t)row * a.ldx : w + (int64_t)row * a.ldw) + k : x;
      const uint32_t to = smemU32(dst + r * PITCH + (i % PER) * E);
      if(VEC) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(src), "r"(in ? 16 : 0) : "memory");
      else asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(src), "r"(in ? 4 : 0) : "memory");
    }
  };
  float2 acc[TM][TN];
#pragma unroll
  for(int i = 0; i < TM; i++)
#pragma unroll
    for(int j = 0; j < TN; j++) acc[i][j] = make_float2(0.0f, 0.0f);
#pragma unroll
  for(int s = 0; s < STAGES - 1; s++) {
    if(s < steps) load(s);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  for(int s = 0; s < steps; s++) {
    asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
    __syncthreads();  // slice s is there, and everyone is done with the slot of slice s - 1
    if(s + STAGES - 1 < steps) load(s + STAGES - 1);
    asm volatile("cp.async.commit_group;" ::: "memory");
    const float* sA = sm + (s % STAGES) * (BM + BN) * PITCH + ty * PITCH + kg * (BK / KG);
    const float* sB = sm + (s % STAGES) * (BM + BN) * PITCH + (BM + tx) * PITCH + kg * (BK / KG);
#pragma unroll
    for(int k = 0; k < BK / KG; k += 4) {
      float4 av[TM], bv[TN];
#pragma unroll
      for(int i = 0; i < TM; i++) av[i] = *reinterpret_cast<const float4*>(sA + TY * i * PITCH + k);
#pragma unroll
      for(int j = 0; j < TN; j++) bv[j] = *reinterpret_cast<const float4*>(sB + TX * j * PITCH + k);
#pragma unroll
      for(int i = 0; i < TM; i++)
#pragma unroll
        for(int j = 0; j < TN; j++) acc[i][j] = __ffma2_rn(make_float2(av[i].x, av[i].y), make_float2(bv[j].x, bv[j].y), acc[i][j]);
#pragma unroll
      for(int i = 0; i < TM; i++)
#pragma unroll
        for(int j = 0; j < TN; j++) acc[i][j] = __ffma2_rn(make_float2(av[i].z, av[i].w), make_float2(bv[j].z, bv[j].w), acc[i][j]);
    }
  }
  if(KG > 1) {
    // the groups' sums [group][BM][BN] take the place of the slices; all threads add up and finish a share of the outputs
    __syncthreads();
#pragma unroll
    for(int i = 0; i < TM; i++)
#pragma unroll
      for(int j = 0; j < TN; j++) sm[(kg * BM + ty + TY * i) * BN + tx + TX * j] = acc[i][j].x + acc[i][j].y;
    __syncthreads();
    for(int i = tid; i < BM * BN; i += THREADS) {
      const int m = m0 + i / BN, n = n0 + i % BN;
      if(m >= a.M || n >= a.N) continue;
      float v = sm[i];
#pragma unroll
      for(int g = 1; g < KG; g++) v += sm[g * BM * BN + i];
      matmulStore<float>(a, m, n, v);
    }
    return;
  }
#pragma unroll
  for(int i = 0; i < TM; i++) {
    const int m = m0 + ty + TY * i;
#pragma unroll
    for(int j = 0; j < TN; j++) {
      const int n = n0 + tx + TX * j;
      if(m < a.M && n < a.N) matmulStore<float>(a, m, n, acc[i][j].x + acc[i][j].y);
    }
  }
}

constexpr int FEW_COLS = 4;

// MR rows (1, 2, 4 or 8; rows past M repeat the last one and are not stored)
template <typename T, int MR, int V>
__global__ void __launch_bounds__(256) matmulFewKernel(const MatmulArgs a) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n0 = blockIdx.x * FEW_COLS;
  float acc[MR][FEW_COLS];
#pragma unroll
  for(int m = 0; m < MR; m++)
#pragma unroll
    for(int c = 0; c < FEW_COLS; c++) acc[m][c] = 0.0f;
  gridDepLaunch();
  gridDepWait();
  for(int k = (warp * 32 + lane) * V; k < a.K; k += 8 * 32 * V) {
    OpVec<T, V> w[FEW_COLS];
#pragma unroll
    for(int c = 0; c < FEW_COLS; c++) w[c].load((const T*)a.w + (int64_t)min(n0 + c, a.N - 1) * a.ldw + k);
#pragma unroll
    for(int m = 0; m < MR; m++) {
      OpVec<T, V> x;
      x.load((const T*)a.x + (int64_t)min(m, a.M - 1) * a.ldx + k);
#pragma unroll
      for(int e = 0; e < V; e++) {
        const float xe = OpType<T>::to(x.e[e]);
#pragma unroll
        for(int c = 0; c < FEW_COLS; c++) acc[m][c] = fmaf(xe, OpType<T>::to(w[c].e[e]), acc[m][c]);
      }
    }
  }
  __shared__ float part[8][MR * FEW_COLS];
#pragma unroll
  for(int m = 0; m < MR; m++)
#pragma unroll
    for(int c = 0; c < FEW_COLS; c++) {
      float v = acc[m][c];
#pragma unroll
      for(int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
      if(lane == 0) part[warp][m * FEW_COLS + c] = v;
    }
  __syncthreads();
  for(int i = threadIdx.x; i < MR * FEW_COLS; i += 256) {
    const int m = i / FEW_COLS, n = n0 + i % FEW_COLS;
    if(m >= a.M || n >= a.N) continue;
    float v = 0.0f;
#pragma unroll
    for(int s = 0; s < 8; s++) v += part[s][i];
    matmulStore<T>(a, m, n, v);
  }
}

template <typename T> __device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if(std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// R8: groups of eight rows of x
template <typename T, int R8>
__global__ void __launch_bounds__(256) matmulFewMmaKernel(const MatmulArgs a) {
  __shared__ float part[8][R8][4][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16;
  const T* w0 = (const T*)a.w + (int64_t)min(n0 + g, a.N - 1) * a.ldw;
  const T* w1 = (const T*)a.w + (int64_t)min(n0 + g + 8, a.N - 1) * a.ldw;
  float acc[R8][4];
#pragma unroll
  for(int r = 0; r < R8; r++)
#pragma unroll
    for(int e = 0; e < 4; e++) acc[r][e] = 0.0f;
  gridDepLaunch();
  gridDepWait();
  constexpr int U = 4;  // steps of 32 channels in flight
  for(int kb = warp * 32 + t * 8; kb - t * 8 < a.K; kb += 256 * U) {
    uint4 wa[U], wb[U], xv[U][R8];
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for(int u = 0; u < U; u++) {
      const int k = kb + 256 * u;
      const bool in = k < a.K;
      wa[u] = in ? *reinterpret_cast<const uint4*>(w0 + k) : zero;
      wb[u] = in ? *reinterpret_cast<const uint4*>(w1 + k) : zero;
#pragma unroll
      for(int r = 0; r < R8; r++)
        xv[u][r] = in && r * 8 + g < a.M ? *reinterpret_cast<const uint4*>((const T*)a.x + (int64_t)(r * 8 + g) * a.ldx + k) : zero;
    }
#pragma unroll
    for(int u = 0; u < U; u++)
#pragma unroll
      for(int r = 0; r < R8; r++) {
        mma16816<T>(acc[r], wa[u].x, wb[u].x, wa[u].y, wb[u].y, xv[u][r].x, xv[u][r].y);
        mma16816<T>(acc[r], wa[u].z, wb[u].z, wa[u].w, wb[u].w, xv[u][r].z, xv[u][r].w);
      }
  }
#pragma unroll
  for(int r = 0; r < R8; r++)
#pragma unroll
    for(int e = 0; e < 4; e++) part[warp][r][e][lane] = acc[r][e];
  __syncthreads();
  for(int i = threadIdx.x; i < R8 * 128; i += 256) {
    // output (row of x, weight row): value e of the lane that has them
    const int n = i & 15, m8 = (i >> 4) & 7, r = i >> 7;
    const int e = (n >> 3) * 2 + (m8 & 1), l = (n & 7) * 4 + (m8 >> 1);
    float v = 0.0f;
#pragma unroll
    for(int s = 0; s < 8; s++) v += part[s][r][e][l];
    const int m = r * 8 + m8;
    if(m < a.M && n0 + n < a.N) matmulStore<T>(a, m, n0 + n, v);
  }
}

template <typename T> cudaError_t matmulFewMma(cudaStream_t st, const MatmulArgs& a) {
  const dim3 grid((a.N + 15) / 16), block(256);
  if(a.M <= 8) return launchDependent(matmulFewMmaKernel<T, 1>, grid, block, 0, st, a);
  return launchDependent(matmulFewMmaKernel<T, 2>, grid, block, 0, st, a);
}

// The tile whose share of the SM with the most of them costs the least; the smaller ones load more operands per FMA.
struct TileForm {
  int bm, bn;
  double per;  // cost of an output, relative
  void (*run)(const MatmulArgs);
  int threads;
  size_t smem;
};
template <int N> cudaError_t launchTiles(cudaStream_t st, const MatmulArgs& a, const TileForm (&forms)[N], SharedMemoryOptIn (&optIn)[N]) {
  int pick = 0;
  double best = 0;
  long long count = 0;
  for(int i = 0; i < N; i++) {
    const long long tiles = ((long long)a.M + forms[i].bm - 1) / forms[i].bm * ((a.N + forms[i].bn - 1) / forms[i].bn);
    const double cost = (double)((tiles + smCount() - 1) / smCount()) * forms[i].bm * forms[i].bn * forms[i].per;
    if(i == 0 || cost < best) { best = cost; pick = i; count = tiles; }
  }
  if(count >= 1LL << 31) return cudaErrorInvalidValue;
  const size_t bytes = forms[pick].smem;
  if(bytes > 48 * 1024) {
    const cudaError_t e = optIn[pick]((const void*)forms[pick].run, (int)bytes);
    if(e != cudaSuccess) return e;
  }
  return launchDependent(forms[pick].run, dim3((unsigned)count), dim3(forms[pick].threads), bytes, st, a);
}
template <int V> struct F32Forms {
  static cudaError_t launch(cudaStream_t st, const MatmulArgs& a) {
    static const TileForm forms[] = {form<128, 128, 8, 8, 1>(1.0), form<128, 64, 8, 8, 2>(1.1), form<64, 64, 8, 8, 4>(1.35), form<64, 48, 8, 6, 4>(1.4), form<32, 32, 4, 4, 4>(2.0)};
    static SharedMemoryOptIn optIn[5];
    return launchTiles(st, a, forms, optIn);
  }
  template <int BM, int BN, int TM, int TN, int KG> static TileForm form(double per) {
    const size_t slices = (size_t)3 * (BM + BN) * 36 * 4, sums = KG > 1 ? (size_t)KG * BM * BN * 4 : 0;
    return {BM, BN, per, matmulF32Kernel<BM, BN, TM, TN, KG, V == 4>, BM / TM * (BN / TN) * KG, std::max(slices, sums)};
  }
};

template <typename T, int V> cudaError_t matmulLaunch(cudaStream_t st, const MatmulArgs& a) {
  if(a.M <= 8) {
    const dim3 grid((a.N + FEW_COLS - 1) / FEW_COLS), block(256);
    if(a.M == 1) return launchDependent(matmulFewKernel<T, 1, V>, grid, block, 0, st, a);
    if(a.M == 2) return launchDependent(matmulFewKernel<T, 2, V>, grid, block, 0, st, a);
    if(a.M <= 4) return launchDependent(matmulFewKernel<T, 4, V>, grid, block, 0, st, a);
    return launchDependent(matmulFewKernel<T, 8, V>, grid, block, 0, st, a);
  }
  if constexpr(std::is_same<T, float>::value) return F32Forms<V>::launch(st, a);
  return cudaErrorInvalidValue;  // more tiles than a launch has blocks
}

template <typename T> cudaError_t matmulLaunchT(cudaStream_t st, const MatmulArgs& a) {
  constexpr int V = 16 / sizeof(T);
  const bool vec = (((uintptr_t)a.x | (uintptr_t)a.w) & 15) == 0 && (a.ldx % V) == 0 && (a.ldw % V) == 0 && a.K % V == 0;
  return vec ? matmulLaunch<T, V>(st, a) : matmulLaunch<T, 1>(st, a);
}

}  // namespace

cudaError_t launchMatmul(cudaStream_t st, const MatmulArgs& a) {
  if(matmulTcEligible(a)) {
    const bool aligned = matmulTcAligned(a);
    if(aligned && a.M <= 16 && a.K % 8 == 0 && a.K <= 1024 && a.N <= 8192) return a.dt == DT_F16 ? matmulFewMma<__half>(st, a) : matmulFewMma<__nv_bfloat16>(st, a);
    if(aligned || a.M > 8) return launchMatmulTc(st, a);
  }
  switch(a.dt) {
    case DT_F32: return matmulLaunchT<float>(st, a);
    case DT_F16: return matmulLaunchT<__half>(st, a);
    default: return matmulLaunchT<__nv_bfloat16>(st, a);
  }
}

}  // namespace kb

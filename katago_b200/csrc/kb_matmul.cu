// y = act(x w^T + bias) + residual on a caller's own matrices: fp32, and the kernels for few rows of any type.  (More rows of 16-bit
// types: kb_matmul_tc.cu.)
//
// matmulF32Kernel    fp32: one tile of BM x BN outputs per block, slices of 32 channels through three stages of asynchronous copies
//                    of four bytes (rows may lie anywhere), which transpose them: a thread reads its rows and columns of a channel in
//                    vectors and multiplies with the packed fp32 instructions, two columns at a time.  Where tiles are few, the
//                    blocks of a cluster share K and add their sums in its order through distributed shared memory.
//                    FMA-bound: 4096^3 50 TFLOP/s, two thirds of the units' cycles; shared memory is busy for half of the time
//                    (16 bytes per lane take three passes of it whatever lanes they repeat for).
// matmulFewKernel    up to eight rows (fp32: 16): memory-bound, the weights are read once.  A block has four weight rows and cuts K
//                    over its warps, whose sums are added in warp order.
// matmulFewMmaKernel the same for up to 16 rows of 16-bit types and K up to 1024, where a launch's latency is what counts.
//                    mma.sync takes 16 weight rows against 8 rows of x.  Operands go from memory to registers, 16 bytes
//                    per lane: the sum over K may be taken in any order, so the lane that has channels 8t..8t+7 of a weight row
//                    feeds them as four pairs wherever the instruction wants pairs, and the lane of a row of x does the same.
//                    4 x 1024 x 384 bf16: 2.1 us, 4.0 us in kb_matmul_tc.cu; the two meet at 4 x 16384 x 512 (4.9 us), and longer
//                    sums are better off with asynchronous copies (4 x 4096 x 4096: 12.8 us here, 8.2 us there).
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

constexpr int F32_BK = 32, F32_STAGES = 3;

// BM x BN outputs per block, TM x TN per thread.  KG: groups of threads that share a slice's channels, so that a small tile has threads
// of eight by eight outputs enough (fewer outputs per thread need more of shared memory).  A cluster of `split` blocks shares K.
// vecOut: rows of y and of the residual are whole aligned vectors.
template <int BM, int BN, int TM, int TN, int KG>
__global__ void __launch_bounds__(BM / TM * (BN / TN) * KG, 2) matmulF32Kernel(const MatmulArgs a, int split, int vecOut) {
  constexpr int BK = F32_BK, STAGES = F32_STAGES, PA = BM + 4, PB = BN + 4, SLICE = BK * (PA + PB);
  constexpr int GN = TN % 4 == 0 ? 4 : 2;  // neighbouring columns of a thread; rows: 4
  constexpr int TX = BN / TN, TY = BM / TM, GROUP = TX * TY, THREADS = GROUP * KG;
  static_assert(GROUP % 32 == 0 && TX % 8 == 0 && TY % 4 == 0 && TM % 4 == 0 && TN % GN == 0 && BM % 4 == 0 && BN % 4 == 0 && BK % KG == 0, "a warp is four by eight threads of one group");
  extern __shared__ float4 smem4[];
  float* sm = reinterpret_cast<float*>(smem4);
  const int tid = threadIdx.x, kg = tid / GROUP, warp = (tid % GROUP) >> 5, lane = tid & 31;
  const int tx = warp % (TX / 8) * 8 + (lane & 7), ty = warp / (TX / 8) * 4 + (lane >> 3);
  const int tilesN = (a.N + BN - 1) / BN, tile = (int)blockIdx.x / split, rank = (int)blockIdx.x % split;
  const int m0 = tile / tilesN * BM, n0 = tile % tilesN * BN;
  const float* x = (const float*)a.x;
  const float* w = (const float*)a.w;
  gridDepLaunch();
  gridDepWait();
  const int allSteps = (a.K + BK - 1) / BK;
  const int from = (int)((int64_t)allSteps * rank / split), steps = (int)((int64_t)allSteps * (rank + 1) / split) - from;
  // A warp copies a row's 32 channels, a lane each, into the transposed slice.  There channel k of row r lies in word
  // k * pitch + r of which the lowest two bits are turned by k / 8 (x) or flipped by k / 8 (w): 32, 16 different banks, and
  // the readers, whose k are known at compile time, find neighbouring rows within one aligned vector.  Rows beyond the end repeat the last
  // one, whose outputs are not stored; channels beyond the end are zeros on both sides.
  auto load = [&](int s) {
    constexpr int WARPS = THREADS / 32;
    static_assert(WARPS % 4 == 0 && BM % WARPS == 0 && BN % WARPS == 0, "a thread's rows agree in their lowest two bits");
    const int row0 = tid >> 5, k = (from + s) * BK + lane;
    const uint32_t bytes = k < a.K ? 4 : 0;
    const float *xk = x + (bytes ? k : 0), *wk = w + (bytes ? k : 0);
    const uint32_t toX = smemU32(sm + (s % STAGES) * SLICE + lane * PA + (row0 & ~3) + ((row0 + (lane >> 3)) & 3));
    const uint32_t toW = smemU32(sm + (s % STAGES) * SLICE + BK * PA + lane * PB + (row0 & ~3) + ((row0 + (lane >> 3) * 2) & 3));
#pragma unroll(BM / WARPS > 8 ? 4 : BM / WARPS)
    for(int i = 0; i < BM / WARPS; i++)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(toX + i * WARPS * 4), "l"(xk + (int64_t)min(m0 + row0 + i * WARPS, a.M - 1) * a.ldx), "r"(bytes) : "memory");
#pragma unroll(BN / WARPS > 8 ? 4 : BN / WARPS)
    for(int i = 0; i < BN / WARPS; i++)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(toW + i * WARPS * 4), "l"(wk + (int64_t)min(n0 + row0 + i * WARPS, a.N - 1) * a.ldw), "r"(bytes) : "memory");
  };
  float2 acc[TM][TN / 2];
#pragma unroll
  for(int i = 0; i < TM; i++)
#pragma unroll
    for(int j = 0; j < TN / 2; j++) acc[i][j] = make_float2(0.0f, 0.0f);
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
    const float* sA = sm + (s % STAGES) * SLICE + kg * PA + ty * 4;
    const float* sB = sm + (s % STAGES) * SLICE + BK * PA + kg * PB;
#pragma unroll
    for(int k = 0; k < BK; k += KG) {  // channel k + kg
      const int turn = k / 8;
      float av[TM];
      float2 bv[TN / 2];
#pragma unroll
      for(int i = 0; i < TM; i += 4) {
        const float4 v = *reinterpret_cast<const float4*>(sA + k * PA + i * TY);
        const float t[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for(int e = 0; e < 4; e++) av[i + e] = t[(e + turn) & 3];
      }
#pragma unroll
      for(int j = 0; j < TN; j += GN) {
        if(GN == 4) {
          const float4 v = *reinterpret_cast<const float4*>(sB + k * PB + tx * 4 + j * TX);
          bv[j / 2 + (turn & 1)] = make_float2(v.x, v.y);
          bv[j / 2 + 1 - (turn & 1)] = make_float2(v.z, v.w);
        }
        else bv[j / 2] = *reinterpret_cast<const float2*>(sB + k * PB + ((turn & 1) ? tx ^ 1 : tx) * 2 + j * TX);
      }
#pragma unroll
      for(int i = 0; i < TM; i++)
#pragma unroll
        for(int j = 0; j < TN / 2; j++) acc[i][j] = __ffma2_rn(make_float2(av[i], av[i]), bv[j], acc[i][j]);
    }
  }
  auto rowOf = [&](int i) { return i / 4 * (4 * TY) + ty * 4 + i % 4; };
  auto colOf = [&](int j) { return j / GN * (GN * TX) + tx * GN + j % GN; };
  const float* res = (const float*)a.residual;
  float* y = (float*)a.y;
  if constexpr(KG == 1 && GN == 4) {
    if(split == 1) {
      float bias[TN];
#pragma unroll
      for(int j = 0; j < TN; j++) bias[j] = a.bias && n0 + colOf(j) < a.N ? a.bias[n0 + colOf(j)] : 0.0f;
#pragma unroll
      for(int i = 0; i < TM; i++) {
        const int m = m0 + rowOf(i);
        if(m >= a.M) continue;
        float f[TN], old[TN];
#pragma unroll
        for(int j = 0; j < TN; j += 4) {
          const int n = n0 + colOf(j);
          if(res && vecOut) {
            if(n < a.N) *reinterpret_cast<float4*>(old + j) = *reinterpret_cast<const float4*>(res + (int64_t)m * a.ldr + n);
          }
          else if(res)
#pragma unroll
            for(int e = 0; e < 4; e++)
              if(n + e < a.N) old[j + e] = res[(int64_t)m * a.ldr + n + e];
        }
#pragma unroll
        for(int j = 0; j < TN; j++) f[j] = (j & 1 ? acc[i][j / 2].y : acc[i][j / 2].x) + bias[j];
        opActF32(f, a.act);
#pragma unroll
        for(int j = 0; j < TN; j += 4) {
          const int n = n0 + colOf(j);
#pragma unroll
          for(int e = 0; e < 4; e++)
            if(res) f[j + e] += old[j + e];
          if(vecOut) {
            if(n < a.N) *reinterpret_cast<float4*>(y + (int64_t)m * a.ldy + n) = make_float4(f[j], f[j + 1], f[j + 2], f[j + 3]);
          }
          else
#pragma unroll
            for(int e = 0; e < 4; e++)
              if(n + e < a.N) y[(int64_t)m * a.ldy + n + e] = f[j + e];
        }
      }
      return;
    }
  }
  // the groups' sums [group][BM][BN] take the place of the slices; each block of the cluster adds up and finishes a share of the outputs
  __syncthreads();
#pragma unroll
  for(int i = 0; i < TM; i++)
#pragma unroll
    for(int j = 0; j < TN; j += 2) *reinterpret_cast<float2*>(sm + (kg * BM + rowOf(i)) * BN + colOf(j)) = acc[i][j / 2];
  if(split > 1) clusterSync(); else __syncthreads();
  const int share = BM * BN / split, end = (rank + 1) * share;
  const uint32_t own = smemU32(sm);
  if(vecOut) {
    for(int i = rank * share + tid * 4; i < end; i += THREADS * 4) {
      const int m = m0 + i / BN, n = n0 + i % BN;
      if(m >= a.M || n >= a.N) continue;
      float4 old = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if(res) old = *reinterpret_cast<const float4*>(res + (int64_t)m * a.ldr + n);
      float f[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
      for(int p = 0; p < split * KG; p++) {
        const int at = p % KG * BM * BN + i;
        const float4 o = split > 1 ? ldCluster4(clusterMapAddr(own + at * 4, (uint32_t)(p / KG))) : *reinterpret_cast<const float4*>(sm + at);
        f[0] += o.x; f[1] += o.y; f[2] += o.z; f[3] += o.w;
      }
#pragma unroll
      for(int e = 0; e < 4; e++)
        if(a.bias) f[e] += a.bias[n + e];
      opActF32(f, a.act);
      if(res) { f[0] += old.x; f[1] += old.y; f[2] += old.z; f[3] += old.w; }
      *reinterpret_cast<float4*>(y + (int64_t)m * a.ldy + n) = make_float4(f[0], f[1], f[2], f[3]);
    }
  }
  else {
    constexpr int U = 4;  // outputs at a time: what they read comes before the stores
    for(int i0 = rank * share + tid; i0 < end; i0 += THREADS * U) {
      float f[U], bias[U], old[U];
      bool in[U];
#pragma unroll
      for(int u = 0; u < U; u++) {
        const int i = i0 + u * THREADS, m = m0 + i / BN, n = n0 + i % BN;
        in[u] = i < end && m < a.M && n < a.N;
        bias[u] = in[u] && a.bias ? a.bias[n] : 0.0f;
        old[u] = in[u] && res ? res[(int64_t)m * a.ldr + n] : 0.0f;
        f[u] = 0.0f;
      }
      for(int p = 0; p < split; p++)
#pragma unroll
        for(int g = 0; g < KG; g++)
#pragma unroll
          for(int u = 0; u < U; u++) {
            const int at = g * BM * BN + min(i0 + u * THREADS, BM * BN - 1);
            f[u] += split > 1 ? ldCluster1(clusterMapAddr(own + at * 4, (uint32_t)p)) : sm[at];
          }
#pragma unroll
      for(int u = 0; u < U; u++) f[u] += bias[u];
      opActF32(f, a.act);
#pragma unroll
      for(int u = 0; u < U; u++) {
        const int i = i0 + u * THREADS;
        if(in[u]) y[(int64_t)(m0 + i / BN) * a.ldy + n0 + i % BN] = res ? f[u] + old[u] : f[u];
      }
    }
  }
  if(split > 1) clusterSync();  // nobody leaves while its sums are being read
}

constexpr int FEW_COLS = 4;

// MR rows (1, 2, 4, 8 or 16; rows past M repeat the last one and are not stored)
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

// The tile and the number of blocks that share its K by what they cost: blocks per SM x (time of the products + start and end), in ns as
// measured.  A product takes 5.92e-3 ns of an SM in the largest tile, `per` times that in the others, where SMs have several blocks; a block alone on its SM has latency to wait for (15 % longer; 60 % where more than half of the SMs have
// one).  Joining over the cluster costs some 1.5 to 5 us of each block.
//   4096^3 2770 us (50 TFLOP/s; eight by eight outputs of float4 along K from one block per SM: 3390); 1000 x 1000 x 4000 212 us, 344 us
//   without cutting K; 200 x 512 x 8192 70 and 188; 20 x 64 x 8000 20 and 121; 1083 x 362 x 361 16 and 18.
struct TileForm {
  int bm, bn;
  double per;
  void (*run)(const MatmulArgs, int, int);
  int threads;
  size_t smem;
};
template <int BM, int BN, int TM, int TN, int KG> TileForm tileForm(double per) {
  const size_t slices = (size_t)F32_STAGES * F32_BK * (BM + BN + 8) * 4, sums = (size_t)KG * BM * BN * 4;
  return {BM, BN, per, matmulF32Kernel<BM, BN, TM, TN, KG>, BM / TM * (BN / TN) * KG, std::max(slices, sums)};
}
template <int V> cudaError_t launchF32(cudaStream_t st, const MatmulArgs& a) {
  static const TileForm forms[] = {tileForm<128, 128, 8, 8, 1>(1.0), tileForm<128, 64, 8, 8, 2>(1.06), tileForm<64, 64, 8, 8, 4>(1.17),
                                   tileForm<64, 48, 8, 6, 4>(1.28), tileForm<32, 32, 4, 4, 4>(1.98)};
  constexpr int N = sizeof(forms) / sizeof(forms[0]);
  static SharedMemoryOptIn optIn[N];
  int pick = 0, split = 1;
  double best = -1;
  long long count = 0;
  const int sms = smCount(), steps = (a.K + F32_BK - 1) / F32_BK;
  for(int i = 0; i < N; i++) {
    const double outputs = forms[i].bm * forms[i].bn;
    const long long tiles = ((long long)a.M + forms[i].bm - 1) / forms[i].bm * (((long long)a.N + forms[i].bn - 1) / forms[i].bn);
    for(int c = 1; c <= 8 && c <= steps; c *= 2) {
      const long long blocks = tiles * c, rounds = (blocks + sms - 1) / sms;
      const double alone = rounds > 1 ? 1.0 : blocks * 2 <= sms ? 1.15 : 1.6;
      const double products = outputs * ((steps + c - 1) / c * F32_BK) * forms[i].per * 5.92e-3 * alone;
      const double cost = rounds * (products + 1000 + (c > 1 ? 1200 + 0.16 * outputs + 150 * c : 0));
      if(best < 0 || cost < best) { best = cost; pick = i; split = c; count = blocks; }
    }
  }
  // up to 16 rows: a block of the other kernel takes 2700 ns and one per channel (9 x 4096 x 4096: 47 us, 56 in tiles)
  const int fewBlocks = (a.N - 1) / FEW_COLS + 1;
  if(a.M <= 16 && (double)((fewBlocks - 1) / sms + 1) * (2700.0 + a.K) < best) return launchDependent(matmulFewKernel<float, 16, V>, dim3(fewBlocks), dim3(256), 0, st, a);
  if(count >= 1LL << 31) return cudaErrorInvalidValue;
  const cudaError_t e = optIn[pick]((const void*)forms[pick].run, (int)forms[pick].smem);
  if(e != cudaSuccess) return e;
  const auto wide = [](const void* p, int64_t ld) { return ((uintptr_t)p & 15) == 0 && ld % 4 == 0; };
  const int vecOut = a.N % 4 == 0 && wide(a.y, a.ldy) && (!a.residual || wide(a.residual, a.ldr));
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)count); cfg.blockDim = dim3(forms[pick].threads); cfg.dynamicSmemBytes = forms[pick].smem; cfg.stream = st;
  cudaLaunchAttribute attr[2];
  unsigned n = 0;
  if(split > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = (unsigned)split; attr[n].val.clusterDim.y = 1; attr[n].val.clusterDim.z = 1;
    n++;
  }
  if(dependentLaunches()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    n++;
  }
  cfg.attrs = attr; cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, forms[pick].run, a, split, vecOut);
}

template <typename T, int V> cudaError_t matmulLaunch(cudaStream_t st, const MatmulArgs& a) {
  if(a.M <= 8) {
    const dim3 grid((a.N + FEW_COLS - 1) / FEW_COLS), block(256);
    if(a.M == 1) return launchDependent(matmulFewKernel<T, 1, V>, grid, block, 0, st, a);
    if(a.M == 2) return launchDependent(matmulFewKernel<T, 2, V>, grid, block, 0, st, a);
    if(a.M <= 4) return launchDependent(matmulFewKernel<T, 4, V>, grid, block, 0, st, a);
    return launchDependent(matmulFewKernel<T, 8, V>, grid, block, 0, st, a);
  }
  if constexpr(std::is_same<T, float>::value) return launchF32<V>(st, a);
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

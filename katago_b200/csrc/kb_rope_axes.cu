// Rotary positions with several axes on a caller's own tensors.
//
//   angle(t, p) = sum_a position[t][a] * freq[p][a]
//   (x0, x1) -> (x0 cos - x1 sin, x0 sin + x1 cos)      for every pair p of every head
//
// What bounds it: memory.  Every channel is read and written once; cosine and sine are computed once per token and pair and
// used for all heads that one thread walks through.
//
// Angles of far positions.  position * freq in fp32 is off by 2^-24 of the ANGLE: half a turn at a position of a few million.
// Only the angle's fraction of a turn matters, and that is arithmetic modulo one: a frequency is turned into turns per step as
// a 64-bit fixed-point fraction, the product with an integer position wraps by itself, and the sum over the axes does too.  The fraction
// comes from two words in fp64 (the product with 1/2pi and what its rounding left, with the rest of 1/2pi), each of which is converted
// by itself: it is good to 2^-64 of a turn, times a position of 2^31 at worst 2^-33 per axis.  Of the sum the upper 32 bits
// go to sincospif as a float: off by 2^-32 of a turn, and by the float's rounding, 2^-26 of a turn at the most.  (Frequencies up to 2^40
// radians per step; 1/2pi is known to 2^-110, which shows in larger ones.)
#include "kb_kernels.cuh"
#include "kb_ops.h"
#include "kb_ops_dev.cuh"

#include <algorithm>

namespace kb {

namespace {

// 1 / (2 pi) in two doubles.
constexpr double INV_2PI_HI = 0.15915494309189535;
constexpr double INV_2PI_LO = -9.839338337591243e-18;

// x, of size 1/2 at most, in units of 2^-64 to half a unit: scaled by 2^63 (no overflow at +-1/2), doubled in the ring, and the rest added.
__device__ __forceinline__ unsigned long long ringOf(double x) {
  const double units = x * 9223372036854775808.0, whole = rint(units);
  return 2ull * (unsigned long long)__double2ll_rn(whole) + (unsigned long long)__double2ll_rn(2.0 * (units - whole));
}
// Turns per step of one position as a fraction of 2^64.
__device__ __forceinline__ unsigned long long turnFraction(float freq) {
  const double f = (double)freq;
  const double hi = f * INV_2PI_HI;
  const double lo = fma(f, INV_2PI_HI, -hi) + f * INV_2PI_LO;
  return ringOf(hi - rint(hi)) + ringOf(lo - rint(lo));
}

// Turn fractions that a block keeps in shared memory; more of them (many tables of many axes) are computed where they are used.
constexpr int ROPE_TABLE = 4096;

// MODE 0: scalar pairs (any alignment), 1: V elements = V/2 adjacent pairs per access, 2: halves, V pairs per two accesses
// TABLE: the block keeps the turn fractions (the conversion in the token loop costs registers: 2 x 20 280 tokens 159 us with both, 124 us)
template <typename T, int MODE, int V, bool COPY, bool TABLE>
__global__ void __launch_bounds__(256, MODE == 2 ? 2 : 4) ropeAxesKernel(const RopeArgs a, int chunks, int copies, int headsPerItem, long long items) {
  extern __shared__ unsigned long long sTurn[];  // [freqHeads][pairs][axes], or nothing
  gridDepLaunch();
  gridDepWait();
  bool wild = !TABLE;  // some frequency may be infinite or a NaN
  if(TABLE) {
    const int entries = a.freqHeads * (a.rot / 2) * a.axes;
    // the conversion of a frequency takes some twenty fp64 operations: once per block, not once per token
    for(int i = threadIdx.x; i < entries; i += 256) {
      const bool finite = isfinite(a.freqs[i]);
      sTurn[i] = finite ? turnFraction(a.freqs[i]) : 0;
      wild = wild || !finite;
    }
    wild = __syncthreads_or(wild);
  }
  constexpr int P = MODE == 0 ? 1 : (MODE == 1 ? V / 2 : V);
  const int pairs = a.rot / 2;
  const int totalHeads = a.q.heads + a.k.heads;
  for(long long item = (long long)blockIdx.x * blockDim.x + threadIdx.x; item < items; item += (long long)gridDim.x * blockDim.x) {
    // chunk fastest, then token, then group of heads: neighbouring threads touch neighbouring memory
    const long long rest = item / chunks;
    const int c = (int)(item - rest * chunks);
    const long long tokensAll = (long long)a.batch * a.tokens;
    const int hg = (int)(rest / tokensAll);
    const long long bt = rest - hg * tokensAll;
    const int b = (int)(bt / a.tokens), t = (int)(bt - (long long)b * a.tokens);
    const int h0 = hg * headsPerItem, h1 = min(totalHeads, h0 + headsPerItem);
    const T* qIn = (const T*)a.q.in + b * a.q.inB + t * a.q.inT;
    const T* kIn = (const T*)a.k.in + b * a.k.inB + t * a.k.inT;
    T* qOut = (T*)a.q.out + b * a.q.outB + t * a.q.outT;
    T* kOut = (T*)a.k.out + b * a.k.outB + t * a.k.outT;
    auto in = [&](int h) { return h < a.q.heads ? qIn + h * a.q.inH : kIn + (h - a.q.heads) * a.k.inH; };
    auto out = [&](int h) { return h < a.q.heads ? qOut + h * a.q.outH : kOut + (h - a.q.heads) * a.k.outH; };
    float cs[P], sn[P];
    int have = -1;  // the table whose angles they are
    const int32_t* pos = a.positions + b * a.posB + (long long)t * a.axes;
    auto angles = [&](int th) {
      have = th;
      const long long first = ((long long)th * pairs + c * P) * a.axes;
      unsigned long long turn[P];
#pragma unroll
      for(int p = 0; p < P; p++) turn[p] = 0;
      for(int x = 0; x < a.axes; x++) {
        const unsigned long long at = (unsigned long long)(long long)pos[x];
#pragma unroll
        for(int p = 0; p < P; p++) turn[p] += at * (TABLE ? sTurn[first + p * a.axes + x] : turnFraction(a.freqs[first + p * a.axes + x]));
      }
#pragma unroll
      for(int p = 0; p < P; p++) {
        // upper 32 bits as a signed fraction: units of half a turn for sincospif
        float halfTurns = (float)(int)(turn[p] >> 32) * 4.656612873077393e-10f;
        if(wild)
          for(int x = 0; x < a.axes; x++)
            if(!isfinite(a.freqs[first + p * a.axes + x])) halfTurns = __int_as_float(0x7fffffff);
        sincospif(halfTurns, &sn[p], &cs[p]);
      }
    };
    auto tableOf = [&](int h) {
      return a.freqHeads == 1 ? 0 : (h < a.q.heads ? h / (a.q.heads / a.freqHeads) : (h - a.q.heads) / (a.k.heads / a.freqHeads));
    };
    constexpr int U = MODE == 1 ? 3 : 4;  // heads whose loads are in flight together
    for(int hb = h0; hb < h1; hb += U) {
      constexpr int NV = MODE == 1 ? 1 : 2;
      constexpr int W = MODE == 0 ? 1 : V;
      OpVec<T, W> v[U][NV];
      // the two places of a scalar pair, or the vector(s)
      const int e0 = MODE == 0 ? (a.halves ? c : 2 * c) : c * V;
      const int e1 = MODE == 0 ? (a.halves ? c + pairs : 2 * c + 1) : c * V + pairs;
#pragma unroll
      for(int u = 0; u < U; u++)
        if(hb + u < h1) {
          v[u][0].load(in(hb + u) + e0);
          if(NV == 2) v[u][NV - 1].load(in(hb + u) + e1);
        }
#pragma unroll
      for(int u = 0; u < U; u++) {
        if(hb + u >= h1) break;
        const int th = tableOf(hb + u);
        if(th != have) angles(th);
#pragma unroll
        for(int p = 0; p < P; p++) {
          T& r0 = MODE == 1 ? v[u][0].e[(2 * p) % W] : v[u][0].e[p % W];
          T& r1 = MODE == 1 ? v[u][0].e[(2 * p + 1) % W] : v[u][NV - 1].e[p % W];
          const float x0 = OpType<T>::to(r0), x1 = OpType<T>::to(r1);
          r0 = OpType<T>::from(x0 * cs[p] - x1 * sn[p]);
          r1 = OpType<T>::from(x0 * sn[p] + x1 * cs[p]);
        }
        v[u][0].store(out(hb + u) + e0);
        if(NV == 2) v[u][NV - 1].store(out(hb + u) + e1);
      }
    }
  }
  if(!COPY) return;
  // channels without a position: `copies` vectors of every head, in items of their own, so that a warp has either kind (7 x 1083 tokens
  // of 10 heads, 48 of 80 channels turned, fp32: 15.9 us; 23.7 us with both kinds in a warp)
  constexpr int W = MODE == 0 ? 1 : V, N = 4;  // items in flight
  const long long all = (long long)a.batch * a.tokens * totalHeads * copies, step = (long long)gridDim.x * blockDim.x;
  for(long long item = (long long)blockIdx.x * blockDim.x + threadIdx.x; item < all; item += N * step) {
    OpVec<T, W> v[N];
    T* to[N];
#pragma unroll
    for(int u = 0; u < N; u++) {
      const long long i = item + u * step;
      to[u] = nullptr;
      if(i >= all) continue;
      const long long rest = i / copies, bt = rest / totalHeads;
      const int e = a.rot + (int)(i - rest * copies) * W, h = (int)(rest - bt * totalHeads);
      const int b = (int)(bt / a.tokens), t = (int)(bt - (long long)b * a.tokens);
      const RopeHeads& x = h < a.q.heads ? a.q : a.k;
      const int hh = h < a.q.heads ? h : h - a.q.heads;
      v[u].load((const T*)x.in + b * x.inB + t * x.inT + hh * x.inH + e);
      to[u] = (T*)x.out + b * x.outB + t * x.outT + hh * x.outH + e;
    }
#pragma unroll
    for(int u = 0; u < N; u++)
      if(to[u]) v[u].store(to[u]);
  }
}

template <typename T> cudaError_t ropeLaunch(cudaStream_t st, const RopeArgs& a) {
  constexpr int V = 16 / sizeof(T);
  auto aligned = [&](const RopeHeads& h) {
    if(h.heads == 0) return true;
    const uintptr_t p = (uintptr_t)h.in | (uintptr_t)h.out;
    const int64_t s = h.inB | h.inT | h.inH | h.outB | h.outT | h.outH;
    return (p & 15) == 0 && (s % V) == 0;
  };
  const int unit = a.halves ? 2 * V : V;  // elements that one thread rotates
  const bool vec = aligned(a.q) && aligned(a.k) && a.rot % unit == 0 && a.dim % V == 0;
  // in place the channels behind the rotated ones stay as they are
  const bool copy = (a.q.heads && a.q.in != a.q.out) || (a.k.heads && a.k.in != a.k.out);
  const int chunks = vec ? a.rot / unit : a.rot / 2;
  const int copies = copy ? (vec ? (a.dim - a.rot) / V : a.dim - a.rot) : 0;
  const int heads = a.q.heads + a.k.heads;
  const long long perHead = (long long)a.batch * a.tokens * chunks;
  if(perHead == 0 || heads == 0) return cudaSuccess;
  // heads that one thread walks through: all of them (one set of angles), unless the threads would not fill the GPU
  const long long want = 2048LL * smCount();
  const int groups = (int)std::min<long long>(heads, std::max<long long>(1, want / perHead));
  const int headsPerItem = (heads + groups - 1) / groups;
  const long long items = perHead * ((heads + headsPerItem - 1) / headsPerItem);
  const long long entries = (long long)a.freqHeads * (a.rot / 2) * a.axes;
  const bool table = entries <= ROPE_TABLE;
  const size_t smem = table ? (size_t)entries * 8 : 0;
  // Few blocks walk over the items, so that each converts the frequencies once.  Of 2 to 64 blocks per SM six were best: 128 x 361
  // tokens of 12 heads of 64 (fp16, 142 MB) 29.8 us, 31.4 us with as many as are resident.  So were four resident blocks for
  // adjacent pairs with three heads in flight (33 us with three blocks) and two for halves, which need their registers (2 x 20 280 tokens of 32
  // heads of 128, bf16, 664 MB: 120 us, 5.5 TB/s; 303 us with three, spilled).
  const long long blocks = std::min<long long>((items + 255) / 256, 6LL * smCount());
  const dim3 grid((unsigned)blocks), block(256);
  auto run = [&](auto kernel) { return launchDependent(kernel, grid, block, smem, st, a, chunks, copies, headsPerItem, items); };
  // (without channels to copy, a kernel without that loop: it costs the other one registers, 128 x 361 tokens 30 -> 32 us)
  auto choose = [&](auto withTable) {
    constexpr bool TABLE = decltype(withTable)::value;
    if(!vec) return copies ? run(ropeAxesKernel<T, 0, 1, true, TABLE>) : run(ropeAxesKernel<T, 0, 1, false, TABLE>);
    if(a.halves) return copies ? run(ropeAxesKernel<T, 2, V, true, TABLE>) : run(ropeAxesKernel<T, 2, V, false, TABLE>);
    return copies ? run(ropeAxesKernel<T, 1, V, true, TABLE>) : run(ropeAxesKernel<T, 1, V, false, TABLE>);
  };
  return table ? choose(std::true_type()) : choose(std::false_type());
}

}  // namespace

cudaError_t launchRopeAxes(cudaStream_t st, const RopeArgs& a) {
  switch(a.dt) {
    case DT_F32: return ropeLaunch<float>(st, a);
    case DT_F16: return ropeLaunch<__half>(st, a);
    default: return ropeLaunch<__nv_bfloat16>(st, a);
  }
}

}  // namespace kb

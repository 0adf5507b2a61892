// Products in 8-bit integers with a scale for each token and each output channel,
// on gfx950's matrix cores:
//   y[m][n] = xs[m] ws[n] sum_k x[m][k] w[n][k] + bias[n]
// and the gated pair act(y_0[m][n]) * y_1[m][n] of two such products of the same x.
//
// The sums are 32-bit integers and exact, in whatever order: a result is one
// conversion, two multiplications (and an addition) of binary32 away from it, and
// the same bits whichever kernel computes it and whatever is beside it.
#include "block_ops.h"

#include <hip/hip_ext.h>

namespace hs {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

// One result from its exact sums, `ws` and `bias` those of its channel.
__device__ __forceinline__ float scaled(int sum, float xs, float ws) { return (float)sum * xs * ws; }

__device__ __forceinline__ void put(const RowsArg &y, int64_t m, int n, float v) {
  if (y.type == kT_F32) static_cast<float *>(y.p)[m * y.ld + n] = v;
  else static_cast<uint16_t *>(y.p)[m * y.ld + n] = bits16(y.type, v);
}

// ---- few tokens: the weights go from memory to registers once, HBM-bound.  A
// workgroup has TN tiles of 16 channels (of each weight) and TM tiles of 16
// tokens; its waves take the steps of 64 k in turn and add their sums up in LDS.
constexpr int kFewWaves = 4;
template <int TM, int TN, int PAIR>
__global__ void __launch_bounds__(kFewWaves * 64) int8_few_kernel(Int8Args a) {
  constexpr int T = PAIR * TN * TM;
  __shared__ i32x4 part[kFewWaves][T][64];
  const int wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const int n0 = blockIdx.x * 16 * TN, m0 = blockIdx.y * 16 * TM;
  const int row = lane % 16, at = lane / 16 * 16;
  const int8_t *w[PAIR][TN], *x[TM];
#pragma unroll
  for (int p = 0; p < PAIR; ++p)
#pragma unroll
    for (int j = 0; j < TN; ++j) w[p][j] = a.w[p] + (int64_t)min(n0 + 16 * j + row, a.N - 1) * a.K;
#pragma unroll
  for (int i = 0; i < TM; ++i) x[i] = a.x + (int64_t)min(m0 + 16 * i + row, a.M - 1) * a.ldx;
  i32x4 acc[PAIR][TN][TM] = {};
#pragma unroll 4
  for (int k = wave * 64 + at; k - at < a.K; k += kFewWaves * 64) {
    i32x4 wf[PAIR][TN] = {}, xf[TM] = {};
    if (k < a.K) {
#pragma unroll
      for (int p = 0; p < PAIR; ++p)
#pragma unroll
        for (int j = 0; j < TN; ++j) wf[p][j] = *reinterpret_cast<const i32x4 *>(w[p][j] + k);
#pragma unroll
      for (int i = 0; i < TM; ++i) xf[i] = *reinterpret_cast<const i32x4 *>(x[i] + k);
    }
#pragma unroll
    for (int p = 0; p < PAIR; ++p)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int i = 0; i < TM; ++i)
          acc[p][j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[p][j], xf[i], acc[p][j][i], 0, 0, 0);
  }
#pragma unroll
  for (int p = 0; p < PAIR; ++p)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int i = 0; i < TM; ++i) part[wave][(p * TN + j) * TM + i][lane] = acc[p][j][i];
  __syncthreads();
  for (int tile = wave; tile < TN * TM; tile += kFewWaves) {
    i32x4 s[PAIR];
#pragma unroll
    for (int p = 0; p < PAIR; ++p) {
      s[p] = part[0][p * TN * TM + tile][lane];
#pragma unroll
      for (int v = 1; v < kFewWaves; ++v) s[p] += part[v][p * TN * TM + tile][lane];
    }
    // a lane has one token's four channels
    const int m = m0 + tile % TM * 16 + lane % 16, n = n0 + tile / TM * 16 + lane / 16 * 4;
    if (m >= a.M) continue;
    const float xs = a.xs[m];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (n + r >= a.N) break;
      float v = scaled(s[0][r], xs, a.ws[0][n + r]);
      if constexpr (PAIR == 2) v = activation(a.act, v) * scaled(s[PAIR - 1][r], xs, a.ws[PAIR - 1][n + r]);
      else if (a.bias) v += a.bias[n + r];
      put(a.y, m, n + r, v);
    }
  }
}

// ---- many tokens: tiles through LDS.
// 16 zero bytes: what is loaded behind a row's end.
__device__ const int4 zeros = {0, 0, 0, 0};

template <int BM, int BN, int WM, int WN, int PAIR>
struct Tile {
  static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
  static constexpr int kLoads = (BM + BN) * 8 / kThreads;      // 16 bytes each, of a stage of 128 k
  static constexpr int kStage = (BM + BN) * 128;
  static constexpr int kMi = BM / WM / 32, kNi = BN / WN / 32;
};

typedef const __attribute__((address_space(1))) void *GlobalPtr;
typedef __attribute__((address_space(3))) void *LdsPtr;

template <int BM, int BN, int WM, int WN, int PAIR>
__global__ void __launch_bounds__(64 * WM * WN) int8_tile_kernel(Int8Args a) {
  typedef Tile<BM, BN, WM, WN, PAIR> C;
  // (two arrays: the compiler sees that a stage that is read is not the one that
  // loads are on their way to)
  __shared__ __align__(1024) int8_t even[C::kStage];
  __shared__ __align__(1024) int8_t odd[C::kStage];
  const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64;
  const int wm = wave / WN, wn = wave % WN;
  const int tm = (a.M + BM - 1) / BM;
  const int m0 = (int)(blockIdx.x % tm) * BM, n0 = (int)(blockIdx.x / tm) * (BN / PAIR);
  // A stage holds rows of 128 bytes, tokens then channels, a row's 16-byte pieces
  // in the order piece ^ (row % 8): eight rows' same pieces lie in eight different
  // sets of banks.  (Loads to LDS are in lane order: the order is made by what a lane reads.)
  const int8_t *src[C::kLoads];
  int piece[C::kLoads];
#pragma unroll
  for (int i = 0; i < C::kLoads; ++i) {
    const int slot = i * C::kThreads + tid, r = slot / 8;
    piece[i] = ((slot % 8) ^ (r % 8)) * 16;
    if (r < BM) {
      src[i] = a.x + (int64_t)min(m0 + r, a.M - 1) * a.ldx;
    } else {
      // pairs: each 32 channels of the first weight are followed by the second's
      const int c = r - BM;
      const int n = PAIR == 2 ? c / 64 * 32 + c % 32 : c;
      const int8_t *w = PAIR == 2 && c / 32 % 2 ? a.w[1] : a.w[0];
      src[i] = w + (int64_t)min(n0 + n, a.N - 1) * a.K;
    }
    src[i] += piece[i];
  }
  auto load = [&](int8_t *stage, int k) {
    const bool whole = k + 128 <= a.K;
#pragma unroll
    for (int i = 0; i < C::kLoads; ++i) {
      const void *p = src[i] + k;
      if (!whole && k + piece[i] >= a.K) p = &zeros;
      __builtin_amdgcn_global_load_lds((GlobalPtr)p, (LdsPtr)(stage + (i * C::kThreads + wave * 64) * 16), 16, 0, 0);
    }
  };
  i32x16 acc[C::kMi][C::kNi] = {};
  const int ar = wm * (BM / WM) + lane % 32, br = BM + wn * (BN / WN) + lane % 32;
  auto products = [&](const int8_t *stage) {
#pragma unroll
    for (int kk = 0; kk < 4; ++kk) {
      i32x4 af[C::kMi], bf[C::kNi];
      const int p = ((kk * 2 + lane / 32) ^ (lane % 8)) * 16;
#pragma unroll
      for (int i = 0; i < C::kMi; ++i) af[i] = *reinterpret_cast<const i32x4 *>(stage + (ar + 32 * i) * 128 + p);
#pragma unroll
      for (int j = 0; j < C::kNi; ++j) bf[j] = *reinterpret_cast<const i32x4 *>(stage + (br + 32 * j) * 128 + p);
#pragma unroll
      for (int i = 0; i < C::kMi; ++i)
#pragma unroll
        for (int j = 0; j < C::kNi; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(af[i], bf[j], acc[i][j], 0, 0, 0);
    }
  };
  // All of this wave's loads are there and what it read is in registers; then the
  // same of the other waves: the stage before may be loaded anew.
  auto arrive = [&] {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  load(even, 0);
  for (int k = 0; k < a.K; k += 256) {
    arrive();
    if (k + 128 < a.K) load(odd, k + 128);
    products(even);
    if (k + 128 >= a.K) break;
    arrive();
    if (k + 256 < a.K) load(even, k + 256);
    products(odd);
  }
  // a lane has one channel's results of 16 tokens of each 32 x 32
#pragma unroll
  for (int j = 0; j < C::kNi; j += PAIR) {
    const int n = n0 + wn * (BN / WN / PAIR) + j / PAIR * 32 + lane % 32;
    if (n >= a.N) continue;
    const float w0 = a.ws[0][n], w1 = PAIR == 2 ? a.ws[PAIR - 1][n] : 0.0f;
    const float bias = PAIR == 1 && a.bias ? a.bias[n] : 0.0f;
#pragma unroll
    for (int i = 0; i < C::kMi; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int m = m0 + wm * (BM / WM) + 32 * i + 8 * (r / 4) + 4 * (lane / 32) + r % 4;
        if (m >= a.M) continue;
        const float xs = a.xs[m];
        float v = scaled(acc[i][j][r], xs, w0);
        if constexpr (PAIR == 2) v = activation(a.act, v) * scaled(acc[i][j + PAIR - 1][r], xs, w1);
        else if (a.bias) v += bias;
        put(a.y, m, n, v);
      }
  }
}

template <int TM, int TN, int PAIR>
hipError_t few(const Int8Args &a, hipStream_t stream, hipEvent_t *ev, hipEvent_t done) {
  const dim3 grid((unsigned)((a.N + 16 * TN - 1) / (16 * TN)), (unsigned)((a.M + 16 * TM - 1) / (16 * TM)));
  return launch_timed(int8_few_kernel<TM, TN, PAIR>, grid, kFewWaves * 64, stream, ev, done, a);
}
template <int BM, int BN, int WM, int WN, int PAIR>
hipError_t tiles(const Int8Args &a, hipStream_t stream, hipEvent_t *ev, hipEvent_t done) {
  const int64_t n = (int64_t)((a.M + BM - 1) / BM) * ((a.N + BN / PAIR - 1) / (BN / PAIR));
  return launch_timed(int8_tile_kernel<BM, BN, WM, WN, PAIR>, dim3((unsigned)n), 64 * WM * WN, stream, ev, done, a);
}

template <int PAIR>
hipError_t int8(const Int8Args &a, hipStream_t stream, hipEvent_t *ev, hipEvent_t done) {
  if (a.M <= 16) return few<1, 1, PAIR>(a, stream, ev, done);
  if (a.M <= 32) return few<2, 1, PAIR>(a, stream, ev, done);
  if (a.M <= 64) return few<4, 1, PAIR>(a, stream, ev, done);
  if (a.M <= 512) return tiles<128, 128, 2, 2, PAIR>(a, stream, ev, done);
  return tiles<256, 256, 2, 4, PAIR>(a, stream, ev, done);
}

}  // namespace

hipError_t launch_int8(const Int8Args &a, hipStream_t stream, hipEvent_t *ev, hipEvent_t done) {
  return a.pair ? int8<2>(a, stream, ev, done) : int8<1>(a, stream, ev, done);
}

}  // namespace hs

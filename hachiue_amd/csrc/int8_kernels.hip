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

// Eight channels of a token, one store where they are aligned and there.
__device__ __forceinline__ void put8(const Int8Args &a, int64_t m, int n, const float (&v)[8]) {
  const RowsArg &y = a.y;
  if (!a.wide || n + 8 > a.N) {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (n + e < a.N) put(y, m, n + e, v[e]);
  } else if (y.type == kT_F32) {
    float4 *p = reinterpret_cast<float4 *>(static_cast<float *>(y.p) + m * y.ld + n);
    p[0] = make_float4(v[0], v[1], v[2], v[3]);
    p[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint32_t u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = bits16(y.type, v[2 * e]) | (uint32_t)bits16(y.type, v[2 * e + 1]) << 16;
    *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(y.p) + m * y.ld + n) = make_uint4(u[0], u[1], u[2], u[3]);
  }
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

typedef const __attribute__((address_space(1))) void *GlobalPtr;
typedef __attribute__((address_space(3))) void *LdsPtr;

// A workgroup of 2 x 2 waves has a tile of BM tokens and BN channels (PAIR 2: BN / 2
// of each weight), a wave a quarter of it.  A stage is 128 k of all of its rows.
template <int BM, int BN>
struct Tile {
  static constexpr int kThreads = 256;
  static constexpr int kLoads = (BM + BN) / 32;       // a thread's, 16 bytes each, of a stage
  static constexpr int kStage = (BM + BN) * 128;
  static constexpr int kMi = BM / 64, kNi = BN / 64;  // a wave's 32 x 32 tiles
  static constexpr int kOutLd = BN / 2 + 8;           // a wave's results in LDS, 32 rows at a time
  static_assert(2 * 32 * kOutLd * 4 <= kStage, "the results fit the stages");
};

// Workgroups go to the XCDs in turn, each XCD has its own L2: an XCD takes a run
// of tiles, in which kGroup tiles of tokens follow each other for the same channels.
constexpr int kGroup = 4;
__device__ __forceinline__ void tile_of(int id, int total, int tm, int &im, int &in) {
  const int xcd = id % 8, each = total / 8, more = total % 8;
  const int t = xcd * each + min(xcd, more) + id / 8;
  const int tn = total / tm, span = kGroup * tn, g = t / span, in_group = min(kGroup, tm - g * kGroup);
  im = g * kGroup + (t - g * span) % in_group;
  in = (t - g * span) / in_group;
}

template <int BM, int BN, int PAIR>
__global__ void __launch_bounds__(256, BM * BN > 128 * 128 ? 1 : 2) int8_tile_kernel(Int8Args a) {
  typedef Tile<BM, BN> C;
  // (two arrays: the compiler sees that a stage that is read is not the one that
  // loads are on their way to)
  __shared__ __align__(1024) int8_t even[C::kStage];
  __shared__ __align__(1024) int8_t odd[C::kStage];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64;
  const int wm = wave / 2, wn = wave % 2;
  int im, in;
  tile_of(blockIdx.x, gridDim.x, (a.M + BM - 1) / BM, im, in);
  const int m0 = im * BM, n0 = in * (BN / PAIR);
  // A stage holds rows of 128 bytes, tokens then channels, a row's 16-byte pieces
  // in the order piece ^ (row % 8): eight rows' same pieces lie in eight different
  // sets of banks.  (Loads to LDS are in lane order: the order is made by what a
  // lane reads.)  A load of a wave is eight rows; pairs: each 32 channels of the
  // first weight are followed by the second's.
  const int piece = ((lane % 8) ^ (lane / 8)) * 16;
  const int8_t *base[1 + PAIR] = {a.x + (int64_t)m0 * a.ldx, a.w[0] + (int64_t)n0 * a.K};
  if constexpr (PAIR == 2) base[PAIR] = a.w[1] + (int64_t)n0 * a.K;
  uint32_t off[C::kLoads];
#pragma unroll
  for (int i = 0; i < C::kLoads; ++i) {
    const int r = (i * 4 + wave) * 8 + lane / 8;
    if (i < BM / 32) {
      off[i] = (uint32_t)min(r, a.M - 1 - m0) * (uint32_t)a.ldx + piece;
    } else {
      const int c = r - BM, n = PAIR == 2 ? c / 64 * 32 + c % 32 : c;
      off[i] = (uint32_t)min(n, a.N - 1 - n0) * (uint32_t)a.K + piece;
    }
  }
  auto load = [&](int8_t *stage, int k) {
    if (k + 128 <= a.K) {
#pragma unroll
      for (int i = 0; i < C::kLoads; ++i) {
        const int8_t *from = base[i < BM / 32 ? 0 : 1 + (i - BM / 32) % PAIR] + k;
        __builtin_amdgcn_global_load_lds((GlobalPtr)(from + off[i]), (LdsPtr)(stage + (i * 4 + wave) * 1024), 16, 0, 0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < C::kLoads; ++i) {
        const int8_t *from = base[i < BM / 32 ? 0 : 1 + (i - BM / 32) % PAIR] + k;
        const void *p = k + piece < a.K ? (const void *)(from + off[i]) : (const void *)&zeros;
        __builtin_amdgcn_global_load_lds((GlobalPtr)p, (LdsPtr)(stage + (i * 4 + wave) * 1024), 16, 0, 0);
      }
    }
  };
  i32x16 acc[C::kMi][C::kNi] = {};
  const int ar = (wm * (BM / 2) + lane % 32) * 128, br = (BM + wn * (BN / 2) + lane % 32) * 128;
  struct Pieces {
    i32x4 a[C::kMi], b[C::kNi];
  };
  // the operands of 32 k
  auto read = [&](const int8_t *stage, int kk, Pieces &f) {
    const int p = ((kk * 2 + lane / 32) ^ (lane % 8)) * 16;
#pragma unroll
    for (int i = 0; i < C::kMi; ++i) f.a[i] = *reinterpret_cast<const i32x4 *>(stage + ar + i * 4096 + p);
#pragma unroll
    for (int j = 0; j < C::kNi; ++j) f.b[j] = *reinterpret_cast<const i32x4 *>(stage + br + j * 4096 + p);
  };
  auto products = [&](const Pieces &f) {
#pragma unroll
    for (int i = 0; i < C::kMi; ++i)
#pragma unroll
      for (int j = 0; j < C::kNi; ++j)
        acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(f.a[i], f.b[j], acc[i][j], 0, 0, 0);
  };
  // All of this wave's loads are there and what it read is in registers; then the
  // same of the other waves: the stage that was read may be loaded anew.
  auto arrive = [&] {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  Pieces f, g;
  // A stage: each 32 k's operands are read while the 32 k before are multiplied,
  // the next stage's first ones too; the stage after it is loaded into this one.
  auto step = [&](int8_t *cur, int8_t *next, int k) {
    read(cur, 1, g);
    products(f);
    read(cur, 2, f);
    products(g);
    read(cur, 3, g);
    products(f);
    arrive();
    read(next, 0, f);
    load(cur, k + 256);
    products(g);
  };
  load(even, 0);
  arrive();
  load(odd, 128);
  read(even, 0, f);
  for (int k = 0; k < a.K; k += 256) {
    step(even, odd, k);
    step(odd, even, k + 128);
  }
  arrive();
  // The sums go through LDS, 32 tokens of a wave at a time, so that a thread has
  // eight channels of a token and stores are whole lines.
  int *const out = reinterpret_cast<int *>(wm ? odd : even) + wn * 32 * C::kOutLd;
  constexpr int kCols = BN / 2 / PAIR, kLanes = kCols / 8, kRows = 64 / kLanes;
  const int c = lane % kLanes * 8, n = n0 + wn * kCols + c;
  const int at = PAIR == 2 ? c / 32 * 64 + c % 32 : c;
  float w0[8], w1[8], bias[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int ne = min(n + e, a.N - 1);
    w0[e] = a.ws[0][ne];
    w1[e] = PAIR == 2 ? a.ws[PAIR - 1][ne] : 0.0f;
    bias[e] = PAIR == 1 && a.bias ? a.bias[ne] : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < C::kMi; ++i) {
#pragma unroll
    for (int j = 0; j < C::kNi; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        out[(8 * (r / 4) + 4 * (lane / 32) + r % 4) * C::kOutLd + j * 32 + lane % 32] = acc[i][j][r];
    // (a wave's own part of LDS, its accesses are in order)
    asm volatile("" ::: "memory");
#pragma unroll 1
    for (int r = lane / kLanes; r < 32; r += kRows) {
      const int m = m0 + wm * (BM / 2) + i * 32 + r;
      if (m >= a.M || n >= a.N) continue;
      const float xs = a.xs[m];
      const int *s = out + r * C::kOutLd + at;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = scaled(s[e], xs, w0[e]);
      if constexpr (PAIR == 2) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = activation(a.act, v[e]) * scaled(s[32 + e], xs, w1[e]);
      } else if (a.bias) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += bias[e];
      }
      put8(a, m, n, v);
    }
    asm volatile("" ::: "memory");
  }
}

template <int TM, int TN, int PAIR>
hipError_t few(const Int8Args &a, hipStream_t stream, hipEvent_t *ev, hipEvent_t done) {
  const dim3 grid((unsigned)((a.N + 16 * TN - 1) / (16 * TN)), (unsigned)((a.M + 16 * TM - 1) / (16 * TM)));
  return launch_timed(int8_few_kernel<TM, TN, PAIR>, grid, kFewWaves * 64, stream, ev, done, a);
}
template <int BM, int BN, int PAIR>
hipError_t tiles(const Int8Args &a, hipStream_t stream, hipEvent_t *ev, hipEvent_t done) {
  const int64_t n = (int64_t)((a.M + BM - 1) / BM) * ((a.N + BN / PAIR - 1) / (BN / PAIR));
  return launch_timed(int8_tile_kernel<BM, BN, PAIR>, dim3((unsigned)n), 256, stream, ev, done, a);
}

template <int PAIR>
hipError_t int8(const Int8Args &a, hipStream_t stream, hipEvent_t *ev, hipEvent_t done) {
  if (a.M <= 16) return few<1, 1, PAIR>(a, stream, ev, done);
  if (a.M <= 32) return few<2, 1, PAIR>(a, stream, ev, done);
  if (a.M <= 64) return few<4, 1, PAIR>(a, stream, ev, done);
  if (a.M <= 512) return tiles<128, 128, PAIR>(a, stream, ev, done);
  return tiles<256, 256, PAIR>(a, stream, ev, done);
}

}  // namespace

hipError_t launch_int8(const Int8Args &a, hipStream_t stream, hipEvent_t *ev, hipEvent_t done) {
  return a.pair ? int8<2>(a, stream, ev, done) : int8<1>(a, stream, ev, done);
}

}  // namespace hs

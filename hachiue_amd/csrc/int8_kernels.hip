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

#include <type_traits>

namespace hs {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));

typedef const __attribute__((address_space(1))) void *GlobalPtr;
typedef __attribute__((address_space(3))) void *LdsPtr;
// 16 bytes a lane to LDS.  ONCE: nobody reads them again (non-temporal), which weights
// of more than kOnceBytes are told where one tile of tokens reads them: 49.1 us for
// the lm_head of one token (53.5), 65 of 64 (69), 19.3 for 12288 gated channels of
// 16 (21.3).  Smaller ones may be in the last-level cache (256 MB) when the next
// call comes, and are not when they were read so: 16 tokens over 16384 x 4096, four
// weights in turn, 18.4 us (16.2).
constexpr int64_t kOnceBytes = 80 << 20;
template <bool ONCE>
__device__ __forceinline__ void load_to_lds(const void *from, int8_t *to) {
  __builtin_amdgcn_global_load_lds((GlobalPtr)from, (LdsPtr)to, 16, 0, ONCE ? 2 : 0);
}
// 16 zero bytes: what is loaded behind a row's end.
__device__ const int4 zeros = {0, 0, 0, 0};

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

// Waits of this wave alone, in the order of the code: at most `loads` of its loads
// (and stores) are still on their way, and what it read from LDS is in registers.
template <int loads>
__device__ __forceinline__ void wait_loads() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | (loads & 15) | (loads >> 4) << 14);   // vmcnt, lgkmcnt(0)
  asm volatile("" ::: "memory");
}
// A barrier behind which every wave's LDS accesses are done; loads stay on their way.
__device__ __forceinline__ void meet() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// ---- one token: HBM-bound, the weights go through LDS once.  A workgroup takes tiles
// of 16 channels (of each weight) in turn, its waves the steps of 128 k of a tile;
// their sums are added up in LDS, by one wave while the others go on.  A wave's
// weights pass through its own part of LDS, 8 KB on their way at a time, without a
// barrier and on into the next tile, so that nothing runs dry at a tile's end.  A
// float row is quantised by each workgroup, which saves a launch: its elements are
// asked for behind the first weights, and come behind them.  The product is the
// matrix cores' with the token in all 16 columns: they have 30 times the rate that the
// weights come at.  151936 x 2048: 48.9 us, 6.4 TB/s (plain reads of as many bytes: 6.1).
constexpr int kRowWaves = 4;

// The row into LDS, zeros behind K (a multiple of 128 bytes), and its scale.  A thread
// has 16 elements, all of them or (K is a multiple of 16) none within K.
__device__ __forceinline__ void keep_row(const Int8Args &a, int8_t *q, float *scale_at, uint32_t *most) {
  static_assert(kInt8RowK == 16 * kRowWaves * 64, "a thread has 16 elements");
  const int t = threadIdx.x, wide = (a.K + 127) / 128 * 128;
  const bool has = t * 16 < a.K;
  i32x4 bytes = {};
  if (!a.rows.p) {
    if (has) bytes = reinterpret_cast<const i32x4 *>(a.x)[t];
    if (t == 0) *scale_at = a.xs[0];
  } else {
    typedef uint32_t Any __attribute__((ext_vector_type(4), aligned(2)));
    float v[16] = {};
    if (has && a.rows.type == kT_F32) {
      const Any *p = reinterpret_cast<const Any *>(static_cast<const float *>(a.rows.p) + t * 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const Any u = p[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * i + e] = __uint_as_float(u[e]);
      }
    } else if (has) {
      const Any *p = reinterpret_cast<const Any *>(static_cast<const uint16_t *>(a.rows.p) + t * 16);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const Any u = p[i];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[8 * i + e] = widen16(a.rows.type, (uint16_t)(u[e / 2] >> (16 * (e % 2))));
      }
    }
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) top = max(top, __float_as_uint(v[e]) & 0x7FFFFFFFu);
    top = wave_max(top);
    if (t % 64 == 0) most[t / 64] = top;
    meet();
#pragma unroll
    for (int w = 0; w < kRowWaves; ++w) top = max(top, most[w]);
    float inv;
    const float scale = scale_of(top, &inv);
    if (t == 0) *scale_at = scale;
    uint32_t u[4] = {};
    if (inv > 0.0f) quantised_bytes<16>(v, inv, scale, u);
    bytes = i32x4{(int)u[0], (int)u[1], (int)u[2], (int)u[3]};
  }
  if (t * 16 < wide) reinterpret_cast<i32x4 *>(q)[t] = bytes;
}

template <int PAIR, bool ONCE>
__global__ void __launch_bounds__(kRowWaves * 64) int8_row_kernel(Int8Args a) {
  constexpr int W = kRowWaves, kSlot = PAIR * 2048, kLoads = 2 * PAIR, D = 4 / PAIR;
  // (Arrays of their own, for the compiler to see that loads are on their way to others.
  // It does with a pair, but for r0; with one weight it waits for all of a wave's
  // loads in front of the reads of every slot.)
  __shared__ __align__(1024) int8_t r0[W * kSlot], r1[W * kSlot];
  __shared__ __align__(1024) int8_t r2[D == 4 ? W * kSlot : 16], r3[D == 4 ? W * kSlot : 16];
  __shared__ __align__(16) int8_t q[kInt8RowK];
  __shared__ __align__(16) int part[2][W][PAIR][16];
  __shared__ float scale;
  __shared__ uint32_t most[W];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int tiles = (a.N + 15) / 16;
  const int steps = (a.K + 127) / 128, turns = (steps + W - 1) / W;   // of a tile, a wave's
  // Where the next load is.  A step's rows of 128 bytes lie in 16-byte pieces, piece ^
  // (row / 2 % 8), so that sixteen rows' same pieces fill the 64 banks once (loads
  // to LDS are in lane order: the order is made by what a lane reads); a load is
  // eight rows.
  int to_tile = blockIdx.x, to_turn = 0;
  const int8_t *base[PAIR];
  uint32_t off[2];
  auto seek = [&](int tile) {
    const int n0 = tile * 16;
#pragma unroll
    for (int p = 0; p < PAIR; ++p) base[p] = a.w[p] + (int64_t)n0 * a.K;
#pragma unroll
    for (int i = 0; i < 2; ++i)
      off[i] = (uint32_t)min(i * 8 + lane / 8, a.N - 1 - n0) * (uint32_t)a.K + (lane % 8 ^ (i * 4 + lane / 16)) * 16;
  };
  seek(to_tile);
  auto load = [&](int8_t *slot) {
    const int k = (to_turn * W + wave) * 128;
    const bool whole = k + 128 <= a.K && to_tile < tiles;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int piece = (lane % 8 ^ (i % 2 * 4 + lane / 16)) * 16;
      const void *p = base[i / 2] + k + off[i % 2];
      if (!whole && (k + piece >= a.K || to_tile >= tiles)) p = &zeros;
      load_to_lds<ONCE>(p, slot + wave * kSlot + i * 1024);
    }
    if (++to_turn == turns) {
      to_turn = 0;
      to_tile += gridDim.x;
      if (to_tile < tiles) seek(to_tile);
    }
  };
  load(r0);
  load(r1);
  if constexpr (D == 4) {
    load(r2);
    load(r3);
  }
  keep_row(a, q, &scale, most);
  meet();
  int tile = blockIdx.x, at_turn = 0, done = 0;
  i32x4 acc[PAIR] = {};
  auto turn = [&](int8_t *slot) {
    // A slot's loads are there when at most those of the D - 1 behind it are not.
    wait_loads<(D - 1) * kLoads>();
    const int s = at_turn * W + wave;
    if (s < steps) {
      const int8_t *at = slot + wave * kSlot + lane % 16 * 128;
      i32x4 w[2][PAIR], x[2];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        const int p = kk * 4 + lane / 16;
#pragma unroll
        for (int i = 0; i < PAIR; ++i)
          w[kk][i] = *reinterpret_cast<const i32x4 *>(at + i * 2048 + (p ^ lane / 2 % 8) * 16);
        x[kk] = *reinterpret_cast<const i32x4 *>(q + s * 128 + p * 16);
      }
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int i = 0; i < PAIR; ++i)
          acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[kk][i], x[kk], acc[i], 0, 0, 0);
    }
    // what was read is in registers: its place may be loaded anew
    wait_loads<(D - 1) * kLoads>();
    load(slot);
    if (++at_turn < turns) return;
    at_turn = 0;
    // lanes 0, 16, 32 and 48 have the first column: four channels each
#pragma unroll
    for (int p = 0; p < PAIR; ++p) {
      if (lane % 16 == 0) *reinterpret_cast<i32x4 *>(&part[done % 2][wave][p][lane / 4]) = acc[p];
      acc[p] = i32x4{};
    }
    // (a place is written again two tiles later, behind the next tile's barrier, at
    // which the wave that reads it here arrives when it has read it)
    meet();
    const int n = tile * 16 + lane;
    if (done % W == wave && lane < 16 && n < a.N) {
      int s[PAIR] = {};
#pragma unroll
      for (int p = 0; p < PAIR; ++p)
#pragma unroll
        for (int v = 0; v < W; ++v) s[p] += part[done % 2][v][p][lane];
      float v[1] = {scaled(s[0], scale, a.ws[0][n])};
      if constexpr (PAIR == 2) {
        activate<1>(a.act, v);
        v[0] *= scaled(s[PAIR - 1], scale, a.ws[PAIR - 1][n]);
      } else if (a.bias) {
        v[0] += a.bias[n];
      }
      put(a.y, 0, n, v[0]);
    }
    ++done;
    tile += gridDim.x;
  };
  while (tile < tiles) {   // (turns behind the last tile's end read zeros and are not stored)
    turn(r0);
    if (tile < tiles) turn(r1);
    if constexpr (D == 4) {
      if (tile < tiles) turn(r2);
      if (tile < tiles) turn(r3);
    }
  }
}

// Rows that stay in LDS: 128 bytes of them in pieces of 16, piece ^ (row / 2 % 8), the
// rows an odd multiple of 128 bytes apart, so that sixteen rows' same pieces fill
// the 64 banks once.
constexpr int kKeptBytes = kInt8KeptElems + kInt8KeptRows * 256;   // (a row's width: K + 255 at most)
__device__ __forceinline__ int kept_width(int K) { return ((K + 127) / 128 | 1) * 128; }
__device__ __forceinline__ int kept_piece(int row, int piece, int wide) {
  return row * wide + (piece / 8 * 8 + (piece % 8 ^ row / 2 % 8)) * 16;
}

// All float rows, quantised into `q` by a workgroup, zeros behind K, and their scales:
// a thread has 16 elements (K is a multiple of 16), the rows' largest magnitudes meet
// in LDS.  `next` is called when the rows are asked for.
constexpr int kKeepThreads = kInt8KeptElems / 16;
template <typename F>
__device__ __forceinline__ void keep_rows(const Int8Args &a, int8_t *q, float *scales, uint32_t *most, F next) {
  const int t = threadIdx.x, per = a.K / 16, wide = kept_width(a.K);
  const int row = t / per, piece = t % per;
  const bool has = row < a.M;
  typedef uint32_t Any __attribute__((ext_vector_type(4), aligned(2)));
  Any raw[4] = {};
  if (has) {
    const int64_t at = (int64_t)row * a.rows.ld + piece * 16;
    if (a.rows.type == kT_F32) {
      const Any *p = reinterpret_cast<const Any *>(static_cast<const float *>(a.rows.p) + at);
#pragma unroll
      for (int e = 0; e < 4; ++e) raw[e] = p[e];
    } else {
      const Any *p = reinterpret_cast<const Any *>(static_cast<const uint16_t *>(a.rows.p) + at);
      raw[0] = p[0];
      raw[1] = p[1];
    }
  }
  next();
  if (t < a.M) most[t] = 0;
  for (int i = t; i < a.M * 16; i += kKeepThreads)   // at most 15 pieces behind K
    if (const int z = per + i % 16; z * 16 < wide)
      *reinterpret_cast<i32x4 *>(q + kept_piece(i / 16, z, wide)) = i32x4{};
  meet();
  float v[16];
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    v[e] = a.rows.type == kT_F32 ? __uint_as_float(raw[e / 4][e % 4])
                                 : widen16(a.rows.type, (uint16_t)(raw[e / 8][e / 2 % 4] >> (16 * (e % 2))));
    top = max(top, __float_as_uint(v[e]) & 0x7FFFFFFFu);
  }
  if (has) atomicMax(most + row, top);
  meet();
  if (has) {
    float inv;
    uint32_t u[4] = {};
    const float scale = scale_of(most[row], &inv);
    if (inv > 0.0f) quantised_bytes<16>(v, inv, scale, u);
    *reinterpret_cast<i32x4 *>(q + kept_piece(row, piece, wide)) = i32x4{(int)u[0], (int)u[1], (int)u[2], (int)u[3]};
    if (piece == 0) scales[row] = scale;
  }
  meet();
}

// ---- few results: K is split among a workgroup's waves, so that as many compute
// units as there are tiles of 16 channels (of each weight) and TM tiles of 16 tokens
// read at once.  A wave's weights and tokens pass through its own part of LDS, four
// steps of 128 k asked for at a time (two of more rows), without a barrier; the
// waves' sums are added up at the end.  Loads go on behind K's end, as zeros.  (Loaded
// straight to registers, a matrix operand's neighbouring lanes are different rows, and
// each 16 bytes are a look-up of their own in the cache: 16 tokens of 4096 x 4096 8.8 us,
// 6.4 so, 33 MB read in all.)
// KEPT: float rows are quantised by each workgroup and stay in LDS; its first weights
// are asked for behind them (and, as built, are there too before rows are widened).
template <int TM, int PAIR, int WAVES, bool ONCE, bool KEPT>
__global__ void __launch_bounds__(WAVES * 64) int8_split_kernel(Int8Args a) {
  constexpr int T = PAIR * TM, kRows = PAIR + (KEPT ? 0 : TM);   // tiles of 16 rows of a step
  constexpr int D = kRows <= 2 ? 4 : 2, kSlot = kRows * 2048, kLoads = 2 * kRows;
  // (Arrays of their own, for the compiler to see that loads are on their way to others.
  // It does in some turns; as built, all of a wave's loads are waited for in front of
  // the reads of r0, and with four slots of one weight and a tile of tokens of r2 and r3.)
  __shared__ __align__(1024) int8_t r0[WAVES * kSlot], r1[WAVES * kSlot];
  __shared__ __align__(1024) int8_t r2[D == 4 ? WAVES * kSlot : 16], r3[D == 4 ? WAVES * kSlot : 16];
  static_assert(T * 1024 <= kSlot, "a wave's sums fit its first slot");
  static_assert(!KEPT || (TM * 16 == kInt8KeptRows && WAVES * 64 == kKeepThreads), "one tile of tokens");
  __shared__ __align__(1024) int8_t kept[KEPT ? kKeptBytes : 16];
  __shared__ float kept_scales[KEPT ? kInt8KeptRows : 1];
  __shared__ uint32_t most[KEPT ? kInt8KeptRows : 1];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64), lane = threadIdx.x % 64;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * TM;
  const int steps = (a.K + 127) / 128;
  // A step's rows of 128 bytes lie in 16-byte pieces, piece ^ (row / 2 % 8); a load
  // is eight rows.
  const int8_t *base[kRows];
  uint32_t off[kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    const int r = i % 2 * 8 + lane / 8;
    if (i < 2 * PAIR) {
      base[i / 2] = a.w[i / 2] + (int64_t)n0 * a.K;
      off[i] = (uint32_t)min(r, a.N - 1 - n0) * (uint32_t)a.K;
    } else {
      const int m = m0 + (i / 2 - PAIR) * 16;
      base[i / 2] = a.x + (int64_t)min(m, a.M - 1) * a.ldx;
      off[i] = (uint32_t)max(0, min(r, a.M - 1 - m)) * (uint32_t)a.ldx;
    }
    off[i] += (lane % 8 ^ (i % 2 * 4 + lane / 16)) * 16;
  }
  auto load = [&](int8_t *slot, int s) {
    const int k = s * 128;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int piece = (lane % 8 ^ (i % 2 * 4 + lane / 16)) * 16;
      const void *p = base[i / 2] + k + off[i];
      if (k + 128 > a.K && k + piece >= a.K) p = &zeros;
      int8_t *const to = slot + wave * kSlot + i * 1024;
      if (i < 2 * PAIR) load_to_lds<ONCE>(p, to);
      else load_to_lds<false>(p, to);
    }
  };
  i32x4 acc[PAIR][TM] = {};
  auto products = [&](const int8_t *slot, int s) {
    const int8_t *at = slot + wave * kSlot + lane % 16 * 128;
    i32x4 w[2][PAIR], x[2][TM];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      const int p = ((kk * 4 + lane / 16) ^ (lane / 2 % 8)) * 16;
#pragma unroll
      for (int i = 0; i < PAIR; ++i) w[kk][i] = *reinterpret_cast<const i32x4 *>(at + i * 2048 + p);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        if constexpr (KEPT)   // (rows behind the last: its own again, not stored)
          x[kk][i] = *reinterpret_cast<const i32x4 *>(
              kept + kept_piece(min(lane % 16, a.M - 1), s * 8 + kk * 4 + lane / 16, kept_width(a.K)));
        else x[kk][i] = *reinterpret_cast<const i32x4 *>(at + (PAIR + i) * 2048 + p);
      }
    }
    // what is read is in registers: its place may be loaded anew
    wait_loads<(D - 1) * kLoads>();
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int i = 0; i < PAIR; ++i)
#pragma unroll
        for (int j = 0; j < TM; ++j)
          acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w[kk][i], x[kk][j], acc[i][j], 0, 0, 0);
  };
  // A slot: its loads are there when at most those of the D - 1 behind it are not.
  auto turn = [&](int8_t *slot, int s) {
    wait_loads<(D - 1) * kLoads>();
    products(slot, s);
    load(slot, s + D * WAVES);
  };
  // What the end needs is asked for first: wave j finishes tile j, a lane one token's
  // four channels.  (With one weight the wave has some of it before it asks for
  // weights, as built.)
  static_assert(TM <= WAVES, "a wave a tile");
  const int m = m0 + wave * 16 + lane % 16, n = n0 + lane / 16 * 4;
  float xs = 0.0f, ws[PAIR][4] = {}, bias[4] = {};
  if (wave < TM) {
    if constexpr (!KEPT) xs = a.xs[min(m, a.M - 1)];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
#pragma unroll
      for (int p = 0; p < PAIR; ++p) ws[p][r] = a.ws[p][min(n + r, a.N - 1)];
      if (PAIR == 1 && a.bias) bias[r] = a.bias[min(n + r, a.N - 1)];
    }
  }
  auto first = [&] {
    load(r0, wave);
    load(r1, wave + WAVES);
    if constexpr (D == 4) {
      load(r2, wave + 2 * WAVES);
      load(r3, wave + 3 * WAVES);
    }
  };
  if constexpr (KEPT) keep_rows(a, kept, kept_scales, most, first);
  else first();
  for (int s = wave; s < steps; s += D * WAVES) {
    turn(r0, s);
    if (s + WAVES < steps) turn(r1, s + WAVES);
    if constexpr (D == 4) {
      if (s + 2 * WAVES < steps) turn(r2, s + 2 * WAVES);
      if (s + 3 * WAVES < steps) turn(r3, s + 3 * WAVES);
    }
  }
  // (the loads behind the rows' end are there too before the sums take their place)
  wait_loads<0>();
  i32x4 *const part = reinterpret_cast<i32x4 *>(r0);
#pragma unroll
  for (int p = 0; p < PAIR; ++p)
#pragma unroll
    for (int i = 0; i < TM; ++i) part[wave * (kSlot / 16) + (p * TM + i) * 64 + lane] = acc[p][i];
  __syncthreads();
  if (wave >= TM || m >= a.M) return;
  if constexpr (KEPT) xs = kept_scales[m];
  i32x4 sum[PAIR];
#pragma unroll
  for (int p = 0; p < PAIR; ++p) {
    sum[p] = part[(p * TM + wave) * 64 + lane];
#pragma unroll
    for (int v = 1; v < WAVES; ++v) sum[p] += part[v * (kSlot / 16) + (p * TM + wave) * 64 + lane];
  }
  float v[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) v[r] = scaled(sum[0][r], xs, ws[0][r]);
  if constexpr (PAIR == 2) {
    activate<4>(a.act, v);
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] *= scaled(sum[PAIR - 1][r], xs, ws[PAIR - 1][r]);
  } else if (a.bias) {
#pragma unroll
    for (int r = 0; r < 4; ++r) v[r] += bias[r];
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (n + r < a.N) put(a.y, m, n + r, v[r]);
}

// ---- many tokens: tiles through LDS, bound by the matrix cores and the power that
// they draw.  A workgroup of 2 x 2 waves has a tile of BM tokens and BN channels (PAIR
// 2: BN / 2 of each weight), a wave a quarter of it.  A stage is 128 k of all of its
// rows.  256 x 256 reads each byte from L2 for 256 results and from LDS for 128, which
// leaves either path half idle beside the products (128 x 128 takes all that a unit
// gets from L2); its sums are all 256 accumulation registers of a lane, so that a
// unit has one workgroup, and nothing runs beside a tile's epilogue.  8192 x 8192 x
// 8192: 450 us, 2450 TOPS, the matrix cores busy for 62 % of the clocks, which fall to
// 1.8 GHz; 4096 tokens of 4096 by 12288 gated channels 410 us, of which the epilogues
// take 70.  (8 waves with 128 x 64 each: the compiler moves sums to memory.  128 x
// 256 tiles of 64 k, two workgroups a unit: 6 to 10 % faster for K <= 2048, 10 to 25 %
// slower above.)
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

// The order of `products` matrix instructions, `reads` from LDS and `loads` to it:
// evenly among each other.  (The waves of a CU are alone on their SIMDs: what stands
// between two products is hidden behind the first, what stands together is not.)
template <int products, int reads, int loads, int i = 0>
__device__ __forceinline__ void interleave() {
  constexpr int r = (i + 1) * reads / products - i * reads / products;
  constexpr int l = (i + 1) * loads / products - i * loads / products;
  __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
  if constexpr (r > 0) __builtin_amdgcn_sched_group_barrier(0x100, r, 0);
  if constexpr (l > 0) __builtin_amdgcn_sched_group_barrier(0x010, l, 0);
  if constexpr (i + 1 < products) interleave<products, reads, loads, i + 1>();
}

template <int BM, int BN, int PAIR, int D, bool ONCE>
__global__ void __launch_bounds__(256, BM * BN > 128 * 128 || D > 2 ? 1 : 2) int8_tile_kernel(Int8Args a) {
  typedef Tile<BM, BN> C;
  constexpr int kEarly = D > 2 ? C::kLoads : C::kLoads - C::kLoads / 4;
  // (arrays of their own: the compiler sees that a stage that is read is not one
  // that loads are on their way to)
  __shared__ __align__(1024) int8_t s0[C::kStage], s1[C::kStage];
  __shared__ __align__(1024) int8_t s2[D == 4 ? C::kStage : 16], s3[D == 4 ? C::kStage : 16];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid / 64), lane = tid % 64;
  const int wm = wave / 2, wn = wave % 2;
  int im, in;
  tile_of(blockIdx.x, gridDim.x, (a.M + BM - 1) / BM, im, in);
  const int m0 = im * BM, n0 = in * (BN / PAIR);
  // A stage holds rows of 128 bytes, tokens then channels, a row's 16-byte pieces
  // in the order piece ^ (row / 2 % 8): sixteen rows' same pieces fill the 64
  // banks once.  (Loads to LDS are in lane order: the order is made by what a
  // lane reads.)  A load of a wave is eight rows; pairs: each 32 channels of the
  // first weight are followed by the second's.
  const int piece = ((lane % 8) ^ (wave % 2 * 4 + lane / 16)) * 16;
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
  // Loads [from, to) of the stage at k; zeros behind the rows' end.
  auto load = [&](int8_t *stage, int k, int from, int to) {
#pragma unroll
    for (int i = from; i < to; ++i) {
      const int8_t *p = base[i < BM / 32 ? 0 : 1 + (i - BM / 32) % PAIR] + k;
      int8_t *const to = stage + (i * 4 + wave) * 1024;
      if (i < BM / 32) load_to_lds<false>(p + off[i], to);
      else load_to_lds<ONCE>(p + off[i], to);
    }
  };
  auto load_end = [&](int8_t *stage, int k, int from, int to) {
#pragma unroll
    for (int i = from; i < to; ++i) {
      const int8_t *p = base[i < BM / 32 ? 0 : 1 + (i - BM / 32) % PAIR] + k;
      const void *q = k + piece < a.K ? (const void *)(p + off[i]) : (const void *)&zeros;
      load_to_lds<false>(q, stage + (i * 4 + wave) * 1024);
    }
  };
  // What the end needs is asked for first (and, as built, there before the first
  // stage is asked for), where there are registers to hold it (24 more in 256 x 256 have
  // the compiler move others to memory: 134 us for 4096 tokens over 20000 x 1024, 142 so).
  constexpr bool kAskFirst = BM * BN <= 128 * 128;
  __shared__ float xs_of[BM];
  constexpr int kCols = BN / 2 / PAIR, kLanes = kCols / 8, kRows = 64 / kLanes;
  float w0[8], w1[8], bias[8];
  auto ask = [&] {
    for (int r = tid; r < BM; r += 256) xs_of[r] = a.xs[min(m0 + r, a.M - 1)];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int ne = min(n0 + wn * kCols + lane % kLanes * 8 + e, a.N - 1);
      w0[e] = a.ws[0][ne];
      w1[e] = PAIR == 2 ? a.ws[PAIR - 1][ne] : 0.0f;
      bias[e] = PAIR == 1 && a.bias ? a.bias[ne] : 0.0f;
    }
  };
  if constexpr (kAskFirst) ask();
  i32x16 acc[C::kMi][C::kNi] = {};
  const int ar = (wm * (BM / 2) + lane % 32) * 128, br = (BM + wn * (BN / 2) + lane % 32) * 128;
  struct Pieces {
    i32x4 a[C::kMi], b[C::kNi];
  };
  // the operands of 32 k
  auto read = [&](const int8_t *stage, int kk, Pieces &f) {
    const int p = ((kk * 2 + lane / 32) ^ (lane / 2 % 8)) * 16;
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
  // This wave's loads of the next stage are there (at most those of the D - 2 stages
  // behind it are not) and what it read is in registers; then the same of the other
  // waves: the stage that was read may be loaded anew.
  auto arrive = [&] {
    wait_loads<(D - 2) * C::kLoads>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  Pieces f, g;
  // A stage: each 32 k's operands are read while the 32 k before are multiplied,
  // the next stage's first ones too.  When all waves have read a stage, the one
  // that is D further on is loaded into it, kEarly loads at once, the others (of two
  // stages) with the next stage's first products.  `whole`: these loads lie within
  // the rows.
  auto step = [&](int8_t *cur, int8_t *next, int k, auto whole) {
    constexpr bool kWhole = decltype(whole)::value;
    constexpr int kP = C::kMi * C::kNi, kR = C::kMi + C::kNi;
    if constexpr (kEarly < C::kLoads) {
      if constexpr (kWhole) load(next, k + 128, kEarly, C::kLoads);
      else load_end(next, k + 128, kEarly, C::kLoads);
    }
    read(cur, 1, g);
    products(f);
    if constexpr (kWhole) interleave<kP, kR, C::kLoads - kEarly>();
    read(cur, 2, f);
    products(g);
    if constexpr (kWhole) interleave<kP, kR, 0>();
    read(cur, 3, g);
    products(f);
    if constexpr (kWhole) interleave<kP, kR, 0>();
    arrive();
    if constexpr (kWhole) load(cur, k + 128 * D, 0, kEarly);
    else load_end(cur, k + 128 * D, 0, kEarly);
    read(next, 0, f);
    products(g);
    if constexpr (kWhole) interleave<kP, kR, kEarly>();
  };
  int k = 0;
  if constexpr (D == 4) {
    load_end(s0, 0, 0, C::kLoads);
    load_end(s1, 128, 0, C::kLoads);
    load_end(s2, 256, 0, C::kLoads);
    arrive();
    load_end(s3, 384, 0, C::kLoads);
    read(s0, 0, f);
    for (; k + 1024 <= a.K; k += 512) {
      step(s0, s1, k, std::true_type());
      step(s1, s2, k + 128, std::true_type());
      step(s2, s3, k + 256, std::true_type());
      step(s3, s0, k + 384, std::true_type());
    }
    for (; k < a.K; k += 512) {
      step(s0, s1, k, std::false_type());
      if (k + 128 >= a.K) break;
      step(s1, s2, k + 128, std::false_type());
      if (k + 256 >= a.K) break;
      step(s2, s3, k + 256, std::false_type());
      if (k + 384 >= a.K) break;
      step(s3, s0, k + 384, std::false_type());
    }
  } else {
    // (stages behind the end are zeros: a loop with an exit in the middle would have
    // the compiler move all sums between registers)
    load_end(s0, 0, 0, C::kLoads);
    arrive();
    load_end(s1, 128, 0, kEarly);
    read(s0, 0, f);
    for (; k + 512 <= a.K; k += 256) {
      step(s0, s1, k, std::true_type());
      step(s1, s0, k + 128, std::true_type());
    }
    for (; k < a.K; k += 256) {
      step(s0, s1, k, std::false_type());
      step(s1, s0, k + 128, std::false_type());
    }
  }
  wait_loads<0>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  // The sums go through LDS, 32 tokens of a wave at a time, so that a thread has
  // eight channels of a token and stores are whole lines.
  if constexpr (!kAskFirst) {
    ask();
    __syncthreads();
  }
  const int c = lane % kLanes * 8, n = n0 + wn * kCols + c;
  int *const out = reinterpret_cast<int *>(wm ? s1 : s0) + wn * 32 * C::kOutLd;
  const int at = PAIR == 2 ? c / 32 * 64 + c % 32 : c;
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
    for (int r0 = 0; r0 < 32; r0 += kRows) {
      const int r = r0 + lane / kLanes;
      const int m = m0 + wm * (BM / 2) + i * 32 + r;
      if (m >= a.M || n >= a.N) continue;
      const float xs = xs_of[wm * (BM / 2) + i * 32 + r];
      const int *s = out + r * C::kOutLd + at;
      float v[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = scaled(s[e], xs, w0[e]);
      if constexpr (PAIR == 2) {
        activate<8>(a.act, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= scaled(s[32 + e], xs, w1[e]);
      } else if (a.bias) {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += bias[e];
      }
      put8(a, m, n, v);
    }
    asm volatile("" ::: "memory");
  }
}

inline bool read_once(const Int8Args &a) { return (int64_t)a.N * a.K * (a.pair ? 2 : 1) > kOnceBytes; }

template <int PAIR>
hipError_t row(const Int8Args &a, hipStream_t stream, hipEvent_t *ev, hipEvent_t done) {
  // as many workgroups as a compute unit's LDS holds (37 KB each), each with the same number of tiles
  const int tiles = (a.N + 15) / 16, most = 4 * kSplitCUs, turns = (tiles + most - 1) / most;
  const dim3 grid((unsigned)((tiles + turns - 1) / turns));
  return read_once(a) ? launch_timed(int8_row_kernel<PAIR, true>, grid, kRowWaves * 64, stream, ev, done, a)
                      : launch_timed(int8_row_kernel<PAIR, false>, grid, kRowWaves * 64, stream, ev, done, a);
}
template <int TM, int PAIR, int WAVES>
hipError_t split(const Int8Args &a, hipStream_t stream, hipEvent_t *ev, hipEvent_t done) {
  const dim3 grid((unsigned)((a.N + 15) / 16), (unsigned)((a.M + 16 * TM - 1) / (16 * TM)));
  if constexpr (TM <= 2)   // (one tile of tokens)
    if (read_once(a))
      return launch_timed(int8_split_kernel<TM, PAIR, WAVES, true, false>, grid, WAVES * 64, stream, ev, done, a);
  return launch_timed(int8_split_kernel<TM, PAIR, WAVES, false, false>, grid, WAVES * 64, stream, ev, done, a);
}
template <int BM, int BN, int PAIR>
int64_t tile_count(const Int8Args &a) {
  return (int64_t)((a.M + BM - 1) / BM) * ((a.N + BN / PAIR - 1) / (BN / PAIR));
}
template <int BM, int BN, int PAIR, int D>
hipError_t tiles(const Int8Args &a, hipStream_t stream, hipEvent_t *ev, hipEvent_t done) {
  const dim3 grid((unsigned)tile_count<BM, BN, PAIR>(a));
  if constexpr (BM == 64)
    if (a.M <= BM && read_once(a))
      return launch_timed(int8_tile_kernel<BM, BN, PAIR, D, true>, grid, 256, stream, ev, done, a);
  return launch_timed(int8_tile_kernel<BM, BN, PAIR, D, false>, grid, 256, stream, ev, done, a);
}

// How long `count` tiles of `stages` 128 k take, `slots` of them at a time: in us, a
// stage's and an epilogue's share; a round that is not full costs from `idle` of a full
// one's time on (fewer units run faster).  Fitted to 300 to 4096 tokens by 2048 to
// 20000 channels and K of 1024 to 8192, 66 cases with and without a second weight,
// where either of 128 x 128 and 256 x 256 is the faster by up to 70 %: the faster one
// is chosen in 60, and the others lose 8 % at most.
inline double rounds_time(int64_t count, int slots, double idle, double stage, double rest, int64_t stages) {
  const int64_t full = count / slots, left = count % slots;
  const double rounds = (double)full + (left ? idle + (1.0 - idle) * (double)left / slots : 0.0);
  return rounds * (stage * (double)stages + rest);
}

// Which kernel.  us in replayed graphs, four weights in turn, binary32 results, at K =
// 4096 unless said (2048 for 40000 channels and more):
//   one token: 49 over 151936 channels (the split kernel 84); over 4096 7.4, where the
//   split kernel takes 6.5, and with a float row 7.5 and 6.3, but 4.2 and 4.4 for K =
//   2048, 7.4 and 7.9 for a pair of it, 10.9 and 11.2 for a pair of 4096
//   K split among 8 waves up to 256 strips of 16 channels, among 4 above: 16 tokens
//   over 4096 6.4 and 6.9, over 8192 11.3 and 10.2 (tiles of four stages 12.8, 13.0)
//   tiles of 64 x 128: 16 tokens over 16384 16.5 (split 18.6), over 151936 59 (90); 64
//   over 4096 13.3 (split 9.5), over 16384 19.3 (27); of two stages, three workgroups a
//   unit, above a workgroup a unit: 64 over 40000 23 (four stages 27), over 4096 20 (13)
//   tiles of 128 x 128 of four stages: 1024 over 4096 25 (two stages 28, 64 x 128 30)
template <int PAIR>
hipError_t int8(const Int8Args &a, hipStream_t stream, hipEvent_t *ev, hipEvent_t done) {
  if (int8_row(a.M, a.K)) return row<PAIR>(a, stream, ev, done);
  if (a.rows.p)   // (int8_kept)
    return launch_timed(int8_split_kernel<1, PAIR, 8, false, true>, dim3((a.N + 15) / 16), kKeepThreads, stream, ev,
                        done, a);
  const int64_t strips = (a.N + 15) / 16, groups = (a.M + 63) / 64;
  if (a.M <= 16 && strips <= 768)
    return strips <= 256 ? split<1, PAIR, 8>(a, stream, ev, done) : split<1, PAIR, 4>(a, stream, ev, done);
  if (a.M <= 32 && strips <= 512)
    return strips <= 256 ? split<2, PAIR, 8>(a, stream, ev, done) : split<2, PAIR, 4>(a, stream, ev, done);
  if (strips * groups * PAIR <= 512) return split<4, PAIR, 4>(a, stream, ev, done);
  if (tile_count<64, 128, PAIR>(a) <= kSplitCUs) return tiles<64, 128, PAIR, 4>(a, stream, ev, done);
  if (a.M <= 64) return tiles<64, 128, PAIR, 2>(a, stream, ev, done);
  const int64_t mid = tile_count<128, 128, PAIR>(a), large = tile_count<256, 256, PAIR>(a), stages = (a.K + 127) / 128;
  if (mid <= kSplitCUs) return tiles<128, 128, PAIR, 4>(a, stream, ev, done);
  const double mid_us = rounds_time(mid, 2 * kSplitCUs, 0.5, 1.12, PAIR == 2 ? 2.5 : 4.2, stages);
  const double large_us = rounds_time(large, kSplitCUs, 0.6, 1.7, PAIR == 2 ? 12.0 : 11.5, stages);
  return mid_us < large_us ? tiles<128, 128, PAIR, 2>(a, stream, ev, done)
                           : tiles<256, 256, PAIR, 2>(a, stream, ev, done);
}

}  // namespace

hipError_t launch_int8(const Int8Args &a, hipStream_t stream, hipEvent_t *ev, hipEvent_t done) {
  return a.pair ? int8<2>(a, stream, ev, done) : int8<1>(a, stream, ev, done);
}

}  // namespace hs

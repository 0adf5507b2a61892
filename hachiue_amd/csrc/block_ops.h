// What the kernels of a model's 8-bit block share: rows of several element
// types, norms between blocks (norm_kernels.hip), products in 8-bit integers
// (int8_kernels.hip).
#pragma once

#include "sampler_internal.h"

#include <hip/hip_ext.h>

namespace hs {

// Element types of rows: GGML ids.
constexpr int kT_F32 = 0, kT_F16 = 1, kT_I8 = 24, kT_BF16 = 30;
constexpr int kNormTimedSlot = 17, kInt8TimedSlot = 18, kRequantTimedSlot = 19;
constexpr int row_elem_bytes(int type) {
  return type == kT_F32 ? 4 : type == kT_F16 || type == kT_BF16 ? 2 : type == kT_I8 ? 1 : 0;
}

// Rows of elements; an absent one has p null.
struct RowsArg {
  void *p;
  int64_t ld;                // elements; 0: one row for all
  float *scales;             // I8: a row's scale
  int32_t type;
};

enum NormKind : int32_t { kNormNone = 0, kNormRms = 1, kNormLayer = 2 };
enum Act : int32_t {
  kActNone = 0, kActSilu = 1, kActGelu = 2, kActGeluTanh = 3, kActRelu = 4, kActSigmoid = 5, kActTanh = 6
};
struct NormArg {
  int32_t kind;
  float eps;
  const float *w, *b;        // [C] or null: 1, 0
};

// s = res + scale * act(gate) * after(x); sum = s; out = before(s)
constexpr int kNormMaxC = 32768;
struct BlockNormArgs {
  RowsArg x, gate, res, sum, out;
  NormArg after, before;
  int32_t M, C, act;
  float scale;
};
hipError_t launch_block_norm(const BlockNormArgs &a, hipStream_t stream, hipEvent_t *ev, hipEvent_t done);

// y[m][n] = xs[m] * ws[n] * sum_k x[m][k] w[n][k] + bias[n], and with a second
// weight act(the first's) * the second's.
constexpr int64_t kInt8MaxResults = (int64_t)1 << 36;   // (grids below 2^32 threads)
constexpr int kInt8MaxM = 1 << 20, kInt8MaxN = 1 << 24, kNormMaxM = 1 << 24;
constexpr int64_t kInt8MaxLd = 1 << 23;   // 255 rows of it below 2^31
constexpr int kInt8MaxK = 65536;   // 2^16 * 2^14 below 2^31: the sums are exact
struct Int8Args {
  const int8_t *x;           // [M][ldx], 16-byte aligned rows
  int64_t ldx;
  const float *xs;           // [M]
  const int8_t *w[2];        // [N][K]
  const float *ws[2];        // [N]
  const float *bias;         // [N] or null
  RowsArg y;
  int32_t M, N, K, pair, act;
  int32_t wide;              // y's rows are 16-byte aligned
  RowsArg rows;              // float rows that the kernel quantises itself (int8_quantises), or p null
};
// One row that a workgroup holds in its threads' registers has a kernel of its own,
// which quantises it too.
constexpr int kInt8RowK = 4096;
inline bool int8_row(int32_t M, int32_t K) { return M == 1 && K <= kInt8RowK; }
// A few float rows, 16 elements a thread of each workgroup, are quantised by the split
// kernel in less time than a launch before it takes: 4.3 us for 2 rows of 1024 by
// 1024 channels (5.7), 5.6 for 8 x 1024 by 2048 (6.4), 7.7 for 2 x 4096 by 4096 (9.1),
// 9.9 for 1 x 8192 by 4096 (11.9), 6.6 for a pair of 8 x 1024 by 2816 (6.6).  More
// elements a thread, or more workgroups that repeat it: 14.2 for 8 x 4096 by 4096 (9.6),
// 11.7 for 2 x 2048 by 12288 (11.7).  (The rows are waited for together with the
// first weights: where they were not, the limits would lie elsewhere.)
constexpr int kInt8KeptRows = 16, kInt8KeptElems = 8192, kInt8KeptN = 4096;
inline bool int8_kept(int32_t M, int32_t N, int32_t K) {
  return M <= kInt8KeptRows && (int64_t)M * K <= kInt8KeptElems && N <= kInt8KeptN;
}
inline bool int8_quantises(int32_t M, int32_t N, int32_t K) { return int8_row(M, K) || int8_kept(M, N, K); }
hipError_t launch_int8(const Int8Args &a, hipStream_t stream, hipEvent_t *ev, hipEvent_t done);

#ifdef __HIPCC__
// A wave's sum or maximum, in every lane: within rows of 16 lanes by DPP, then the
// four rows' by scalars (no LDS: 30 clocks where six shuffles take 400).
template <typename F>
__device__ __forceinline__ uint32_t wave_reduce(uint32_t v, F both) {
  v = both(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false));    // lane ^ 1
  v = both(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false));    // lane ^ 2
  v = both(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x141, 0xF, 0xF, false));   // 7 - lane of 8
  v = both(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x140, 0xF, 0xF, false));   // 15 - lane of 16
  const uint32_t a = (uint32_t)__builtin_amdgcn_readlane((int)v, 0), b = (uint32_t)__builtin_amdgcn_readlane((int)v, 16);
  const uint32_t c = (uint32_t)__builtin_amdgcn_readlane((int)v, 32), d = (uint32_t)__builtin_amdgcn_readlane((int)v, 48);
  return both(both(a, b), both(c, d));
}
__device__ __forceinline__ float wave_sum(float v) {
  return __uint_as_float(wave_reduce(__float_as_uint(v), [](uint32_t a, uint32_t b) {
    return __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
  }));
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
  return wave_reduce(v, [](uint32_t a, uint32_t b) { return max(a, b); });
}

// One launch; with events its start and end, else the end of it in `done`.
template <typename F, typename A>
hipError_t launch_timed(F kernel, dim3 grid, int threads, hipStream_t stream, hipEvent_t *ev, hipEvent_t done,
                        const A &a) {
  if (ev)
    hipExtLaunchKernelGGL(kernel, grid, dim3(threads), 0u, stream, ev[0], ev[1], 0u, a);
  else if (done)
    hipExtLaunchKernelGGL(kernel, grid, dim3(threads), 0u, stream, nullptr, done, 0u, a);
  else
    hipLaunchKernelGGL(kernel, grid, dim3(threads), 0u, stream, a);
  return hipGetLastError();
}

// exp(x) for x <= 0, a step or two off: x log2(e) as an integer and the rest, the
// logarithm in two parts, so that nothing is lost where x is far below 0.
__device__ __forceinline__ float exp_below(float x) {
  const float n = rintf(x * 1.44269502f);
  const float f = fmaf(x, 1.92596299e-8f, fmaf(x, 1.44269502f, -n));
  return __builtin_amdgcn_ldexpf(__builtin_amdgcn_exp2f(f), (int)n);
}
// v / (1 + exp(-z)): the exponential never overflows, so that the result goes to
// 0 as slowly as it should where z is far below 0.  The divisor lies in [1, 2]: its
// reciprocal and one correction, a third of a division's instructions.
__device__ __forceinline__ float logistic(float v, float z) {
  const float e = exp_below(fmaxf(-fabsf(z), -256.0f));
  const float d = 1.0f + e, r = __builtin_amdgcn_rcpf(d), n = z < 0.0f ? e : 1.0f;
  const float q = n * r;
  return v * fmaf(fmaf(-d, q, n), r, q);
}

// (the choice outside of the loops: n independent chains of instructions, not n
// branches.  4096 tokens' gated pairs, 128 results a lane of each tile: 451 us with
// the branches, 413 so.)
template <int n>
__device__ __forceinline__ void activate(int act, float (&v)[n]) {
  auto each = [&](auto f) {
#pragma unroll
    for (int e = 0; e < n; ++e) v[e] = f(v[e]);
  };
  switch (act) {
    case kActSilu: return each([](float x) { return logistic(x, x); });
    case kActGelu: return each([](float x) { return 0.5f * x * erfcf(x * -0.70710678f); });   // (no cancellation for x << 0)
    case kActGeluTanh:   // 0.5 (1 + tanh u) = 1 / (1 + exp(-2u))
      return each([](float x) { return logistic(x, 1.59576912f * fmaf(0.044715f * x * x, x, x)); });
    case kActRelu: return each([](float x) { return x > 0.0f ? x : x != x ? x : 0.0f; });
    case kActSigmoid: return each([](float x) { return x != x ? x : logistic(1.0f, x); });
    case kActTanh: return each([](float x) { return tanhf(x); });
  }
}

// The scale of a row whose largest magnitude has the bits `most` (a NaN's are above
// an infinity's, and those above every number's): that magnitude times 1 / 127, both
// in binary32; NaN where it is not finite, 0 below 2^-100.  *inv: 1 / scale, or 0
// where the row's integers are 0.
__device__ __forceinline__ float scale_of(uint32_t most, float *inv) {
  const bool finite = most < 0x7F800000u, some = finite && most >= 0x0D800000u;
  const float scale = some ? __uint_as_float(most) * (1.0f / 127.0f) : finite ? 0.0f : __uint_as_float(0x7FC00000u);
  *inv = some ? 1.0f / scale : 0.0f;
  return scale;
}
// v / scale to the nearest integer, ties to even, as if the quotient were exact:
// v * inv is off by less than 2^-15, so that only next to a half does it not tell;
// there v is compared with the half times the scale, which binary64 holds exactly.
__device__ __forceinline__ int quantised(float v, float inv, float scale) {
  const float a = fabsf(v), t = a * inv;
  float q = rintf(t);
  const float half = rintf(t - 0.5f) + 0.5f;
  if (fabsf(t - half) < 0.000030517578f) {
    const double edge = (double)half * (double)scale;
    const float low = half - 0.5f;
    q = (double)a > edge ? low + 1.0f : (double)a < edge ? low : rintf(half);
  }
  return (int)copysignf(q, v);
}
// The same of n values, four to a word: six instructions each where none of a
// wave's lies next to a half.  1.5 * 2^23 + t is rounded to an integer, which its low
// bits are.
template <int n>
__device__ __forceinline__ void quantised_bytes(const float (&v)[n], float inv, float scale, uint32_t (&u)[n / 4]) {
  uint32_t r[n];
  float most = 0.0f;
#pragma unroll
  for (int e = 0; e < n; ++e) {
    const float t = v[e] * inv, up = t + 12582912.0f;
    r[e] = __float_as_uint(up);
    most = fmaxf(most, fabsf(t - (up - 12582912.0f)));
  }
  if (most > 0.5f - 0.000030517578f) {
#pragma unroll
    for (int e = 0; e < n; ++e) r[e] = (uint32_t)quantised(v[e], inv, scale);
  }
#pragma unroll
  for (int e = 0; e < n; e += 4)
    u[e / 4] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(r[e + 3], r[e + 2], 0x0C0C0400u),
                                     __builtin_amdgcn_perm(r[e + 1], r[e], 0x0C0C0400u), 0x05040100u);
}

__device__ __forceinline__ uint16_t bits16(int type, float v) {
  if (type == kT_F16) {
    const _Float16 h = (_Float16)v;
    return __builtin_bit_cast(uint16_t, h);
  }
  const __bf16 h = (__bf16)v;
  return __builtin_bit_cast(uint16_t, h);
}
__device__ __forceinline__ float widen16(int type, uint16_t u) {
  if (type == kT_F16) return (float)__builtin_bit_cast(_Float16, u);
  return __uint_as_float((uint32_t)u << 16);
}
#endif

}  // namespace hs

// The end of one block of a model and the start of the next, on gfx950:
//   s = residual + scale * act(gate) * after(x),   out = before(s)
// with a norm (root mean square, or mean and variance) or none on either side,
// x, gate, residual, s and out in binary32, binary16 or bfloat16, out also in
// 8-bit integers with a scale for each row.
//
// Every tensor is read and written once: HBM-bound, some dozen operations an
// element.  A row is held in the registers of its threads (64 to 1024 of them, 8
// elements of a tensor in one load, wherever rows start), so
// that the norms' sums, up to five one after the other, read nothing again.  All
// sums are binary32: each thread's own elements one after the other, a tree over the
// lanes of a wave, the waves' one after the other; the number of threads depends on
// the number of rows too.  The kernel's time over three inputs in turn: 8192 rows of
// 4096, x and out bfloat16, residual and s binary32, both norms, 78 us, 5.2 TB/s, and
// 81 with a gate for each channel (a copy of 1 GB: 5.05 to 5.1); 4096 rows of 12288
// bfloat16 in 8 bits 34 us, 4.4 TB/s.
//
// Few rows wait: the types are known at run time, and as built a tensor's elements
// are there before the next tensor's are asked for, and both before the gate's and
// the norms' parameters are (their own below).  Widths that 8 does not divide have a
// second chain of such loads, element by element: 300 rows of 1001 with a gate and two
// norms 6 us, 4096 in one row 4.2.
#include "block_ops.h"

#include <hip/hip_ext.h>

namespace hs {
namespace {

// Eight consecutive elements of a row, as they are stored (16-bit ones in `a`); rows
// start at any element, and loads and stores need no more.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
struct Raw {
  u32x4 a, b;
};
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));

// A thread's elements of a row: eight at a time, G * 8 apart.  Behind C they are 0.
// WHOLE: C is a multiple of 8.
template <int P, int G, bool WHOLE>
__device__ __forceinline__ void read_row(const RowsArg &r, int64_t row, int C, int t, Raw (&raw)[P]) {
  if (r.type == kT_F32) {
    const uint32_t *p = static_cast<const uint32_t *>(r.p) + row * r.ld;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int c = (j * G + t) * 8;
      raw[j] = {};
      if (WHOLE ? c < C : c + 8 <= C) {
        raw[j].a = *reinterpret_cast<const u32x4_any *>(p + c);
        raw[j].b = *reinterpret_cast<const u32x4_any *>(p + c + 4);
      } else if (!WHOLE && c < C) {
        uint32_t u[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = c + e < C ? p[c + e] : 0u;
        raw[j] = {u32x4{u[0], u[1], u[2], u[3]}, u32x4{u[4], u[5], u[6], u[7]}};
      }
    }
  } else {
    const uint16_t *p = static_cast<const uint16_t *>(r.p) + row * r.ld;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int c = (j * G + t) * 8;
      raw[j] = {};
      if (WHOLE ? c < C : c + 8 <= C) {
        raw[j].a = *reinterpret_cast<const u32x4_any *>(p + c);
      } else if (!WHOLE && c < C) {
        uint32_t u[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = c + e < C ? p[c + e] : 0u;
        raw[j].a = u32x4{u[0] | u[1] << 16, u[2] | u[3] << 16, u[4] | u[5] << 16, u[6] | u[7] << 16};
      }
    }
  }
}

__device__ __forceinline__ void widen_raw(int type, const Raw &raw, float (&v)[8]) {
  const uint32_t u[8] = {raw.a.x, raw.a.y, raw.a.z, raw.a.w, raw.b.x, raw.b.y, raw.b.z, raw.b.w};
  if (type == kT_F32) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(u[e]);
  } else if (type == kT_F16) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = widen16(kT_F16, (uint16_t)(u[e / 2] >> (16 * (e % 2))));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(e % 2 ? u[e / 2] & 0xFFFF0000u : u[e / 2] << 16);
  }
}

template <int P, int G, bool WHOLE>
__device__ __forceinline__ void write_row(const RowsArg &r, int64_t row, int C, int t, const float (&v)[P][8]) {
  if (r.type == kT_F32) {
    float *p = static_cast<float *>(r.p) + row * r.ld;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int c = (j * G + t) * 8;
      if (WHOLE ? c < C : c + 8 <= C) {
        *reinterpret_cast<f32x4_any *>(p + c) = f32x4_any{v[j][0], v[j][1], v[j][2], v[j][3]};
        *reinterpret_cast<f32x4_any *>(p + c + 4) = f32x4_any{v[j][4], v[j][5], v[j][6], v[j][7]};
      } else if (!WHOLE) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e < C) p[c + e] = v[j][e];
      }
    }
  } else {
    uint16_t *p = static_cast<uint16_t *>(r.p) + row * r.ld;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int c = (j * G + t) * 8;
      if (WHOLE ? c < C : c + 8 <= C) {
        uint32_t u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          u[e] = bits16(r.type, v[j][2 * e]) | (uint32_t)bits16(r.type, v[j][2 * e + 1]) << 16;
        *reinterpret_cast<u32x4_any *>(p + c) = u32x4{u[0], u[1], u[2], u[3]};
      } else if (!WHOLE) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e < C) p[c + e] = bits16(r.type, v[j][e]);
      }
    }
  }
}

// A parameter of the norm, one per channel.
template <bool WHOLE>
__device__ __forceinline__ void read_param(const float *p, int c, int C, float (&v)[8]) {
  if (WHOLE || c + 8 <= C) {
    const f32x4_any a = *reinterpret_cast<const f32x4_any *>(p + c), b = *reinterpret_cast<const f32x4_any *>(p + c + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = c + e < C ? p[c + e] : 0.0f;
  }
}

// The sum (or the largest) over a row's G threads; `slot` [G / 64] is this reduction's own.
template <int G>
__device__ __forceinline__ float row_sum(float v, float *slot, int t) {
  v = wave_sum(v);
  if constexpr (G > 64) {
    if (t % 64 == 0) slot[t / 64] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < G / 64; ++i) v += slot[i];
  }
  return v;
}
template <int G>
__device__ __forceinline__ uint32_t row_max(uint32_t v, uint32_t *slot, int t) {
  v = wave_max(v);
  if constexpr (G > 64) {
    if (t % 64 == 0) slot[t / 64] = v;
    __syncthreads();
    v = slot[0];
#pragma unroll
    for (int i = 1; i < G / 64; ++i) v = max(v, slot[i]);
  }
  return v;
}

// `early`: the weights are asked for before the sums are formed, not behind them (a
// lone row's time is its chain of waits: 4.9 us, 5.2 so), if behind the row itself.
template <int P, int G, bool WHOLE>
__device__ __forceinline__ void norm_row(const NormArg &n, int C, int t, float (&v)[P][8], float (*slots)[16]) {
  if (n.kind == kNormNone) return;
  float early[8];
  if constexpr (P == 1)
    if (n.w && t * 8 < C) read_param<WHOLE>(n.w, t * 8, C, early);
  if (n.kind == kNormLayer) {
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < P; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) s += v[j][e];
    const float mean = row_sum<G>(s, slots[0], t) / (float)C;
#pragma unroll
    for (int j = 0; j < P; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if ((j * G + t) * 8 + (WHOLE ? 0 : e) < C) v[j][e] -= mean;
  }
  float q = 0.0f;
#pragma unroll
  for (int j = 0; j < P; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) q = fmaf(v[j][e], v[j][e], q);
  const float r = 1.0f / sqrtf(row_sum<G>(q, slots[1], t) / (float)C + n.eps);
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const int c = (j * G + t) * 8;
    if (c >= C) continue;
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[j][e] *= r;
    if (n.w) {
      if constexpr (P > 1) read_param<WHOLE>(n.w, c, C, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[j][e] *= P > 1 ? w[e] : early[e];
    }
    if (n.b) {
      read_param<WHOLE>(n.b, c, C, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[j][e] += w[e];
    }
  }
}

// Threads of a workgroup: several rows where a row has one wave.
template <int G>
constexpr int kNormThreads = G > 256 ? G : 256;
// Whether eight gates are activated together (eight chains of instructions and their
// registers).  One by one, two runs of 1024 threads take 60 registers and not 74, so
// that a compute unit has two workgroups: 34 us for 4096 rows of 12288 quantised (49),
// 118 for 4096 of 10240 with a gate and two norms (147).  Fewer threads a row have
// other workgroups beside them either way: 81 us for 8192 rows of 4096 (84 one by one).
template <int P, int G>
constexpr bool kTogether = !(P == 2 && G == 1024);
// Workgroups of a grid's first dimension (2^32 threads of one are too many).
constexpr unsigned kGridX = 1u << 16;

template <int P, int G, bool WHOLE>
__global__ void __launch_bounds__(kNormThreads<G>) block_norm_kernel(BlockNormArgs a) {
  __shared__ float slots[5][16];
  const int t = threadIdx.x % G;
  const int64_t group = (int64_t)blockIdx.y * kGridX + blockIdx.x;
  const int64_t row = group * (kNormThreads<G> / G) + threadIdx.x / G;
  if (row >= a.M) return;   // (whole waves; with barriers, G is the workgroup)
  Raw raw[P], res[P];
  float v[P][8];
  read_row<P, G, WHOLE>(a.x, row, a.C, t, raw);
  if (a.res.p) read_row<P, G, WHOLE>(a.res, row, a.C, t, res);
#pragma unroll
  for (int j = 0; j < P; ++j) widen_raw(a.x.type, raw[j], v[j]);
  norm_row<P, G, WHOLE>(a.after, a.C, t, v, slots);
  if (a.gate.p) {
    read_row<P, G, WHOLE>(a.gate, row, a.C, t, raw);
#pragma unroll
    for (int j = 0; j < P; ++j) {
      float g[8];
      widen_raw(a.gate.type, raw[j], g);
      if constexpr (kTogether<P, G>) {
        activate<8>(a.act, g);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float one[1] = {g[e]};
          activate<1>(a.act, one);
          g[e] = one[0];
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[j][e] *= g[e];
    }
  }
#pragma unroll
  for (int j = 0; j < P; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[j][e] *= a.scale;
  if (a.res.p) {
#pragma unroll
    for (int j = 0; j < P; ++j) {
      float g[8];
      widen_raw(a.res.type, res[j], g);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[j][e] += g[e];
    }
  }
  // (what lies behind C is 0 again: it counts in no sum below)
#pragma unroll
  for (int j = 0; j < P; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if ((j * G + t) * 8 + (WHOLE ? 0 : e) >= a.C) v[j][e] = 0.0f;
  if (a.sum.p) write_row<P, G, WHOLE>(a.sum, row, a.C, t, v);
  if (!a.out.p) return;
  norm_row<P, G, WHOLE>(a.before, a.C, t, v, slots + 2);
  if (a.out.type != kT_I8) {
    write_row<P, G, WHOLE>(a.out, row, a.C, t, v);
    return;
  }
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < P; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (WHOLE || (j * G + t) * 8 + e < a.C) most = max(most, __float_as_uint(v[j][e]) & 0x7FFFFFFFu);
  most = row_max<G>(most, reinterpret_cast<uint32_t *>(slots[4]), t);
  float inv;
  const float scale = scale_of(most, &inv);
  if (t == 0) a.out.scales[row] = scale;
  int8_t *p = static_cast<int8_t *>(a.out.p) + row * a.out.ld;
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const int c = (j * G + t) * 8;
    if (c >= a.C) continue;
    uint32_t u[2] = {};
    if (inv > 0.0f) quantised_bytes<8>(v[j], inv, scale, u);
    if (WHOLE || c + 8 <= a.C) {
      *reinterpret_cast<u32x2_any *>(p + c) = u32x2_any{u[0], u[1]};
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < a.C) p[c + e] = (int8_t)(u[e / 4] >> (8 * (e % 4)));
    }
  }
}

template <int P, int G>
hipError_t launch(const BlockNormArgs &a, hipStream_t stream, hipEvent_t *ev, hipEvent_t done) {
  constexpr int per = kNormThreads<G> / G;
  const unsigned groups = (unsigned)((a.M + per - 1) / per), x = std::min(groups, kGridX);
  const dim3 grid(x, (groups + x - 1) / x);
  return a.C % 8 ? launch_timed(block_norm_kernel<P, G, false>, grid, kNormThreads<G>, stream, ev, done, a)
                 : launch_timed(block_norm_kernel<P, G, true>, grid, kNormThreads<G>, stream, ev, done, a);
}

}  // namespace

// Threads of a row: two runs of eight elements each, so that many rows are on their
// way at a time; one where there are few rows, which end sooner.  Kernel times in us
// over three inputs in turn, with 256 x 2, 512 x 1, 512 x 2 and 1024 x 2 runs: 8192 rows
// of 4096, bfloat16 and binary32 in and out, 78, 76, 76, 86; 300 rows 4.9, 5.1, 4.9, 5.6;
// 1 row 4.0 to 4.5 with any.  4000 rows of 8192 with 512 x 2 77, 1024 x 1 83.  4096 rows of
// 12288 quantised with 1024 x 2 34 (512 x 3: 36, 256 x 6: 46); 20000 rows of 512 with 64 x 1
// 14.5, 256 x 1 22.6, of 1024 with 64 x 2 32.5, 256 x 1 34.7, where 300 of 1001 take 7.5 and 6.
hipError_t launch_block_norm(const BlockNormArgs &a, hipStream_t stream, hipEvent_t *ev, hipEvent_t done) {
  const int C = a.C;
  if (C <= 512) return launch<1, 64>(a, stream, ev, done);
  if (C <= 1024 && a.M > 2 * kSplitCUs) return launch<2, 64>(a, stream, ev, done);
  if (C <= 2048) return launch<1, 256>(a, stream, ev, done);
  if (C <= 4096) return a.M <= kSplitCUs ? launch<1, 512>(a, stream, ev, done) : launch<2, 256>(a, stream, ev, done);
  if (C <= 8192) return a.M <= kSplitCUs ? launch<1, 1024>(a, stream, ev, done) : launch<2, 512>(a, stream, ev, done);
  if (C <= 16384) return launch<2, 1024>(a, stream, ev, done);
  return launch<4, 1024>(a, stream, ev, done);
}

}  // namespace hs

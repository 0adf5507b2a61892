// The end of one block of a model and the start of the next, on gfx950:
//   s = residual + scale * act(gate) * after(x),   out = before(s)
// with a norm (root mean square, or mean and variance) or none on either side,
// x, gate, residual, s and out in binary32, binary16 or bfloat16, out also in
// 8-bit integers with a scale for each row.
//
// Every tensor is read and written once: HBM-bound, some dozen operations an
// element.  A row is held in the registers of its threads (64 to 1024 of them, 8
// elements of a tensor each in one load, or one where rows start anywhere), so
// that the norms' sums, up to five one after the other, read nothing again.  All
// sums are binary32: each thread's own elements, then a tree.
#include "block_ops.h"

#include <hip/hip_ext.h>

namespace hs {
namespace {

// V consecutive elements of a row, as they are stored.
template <int V>
struct Raw;
template <>
struct Raw<8> {
  uint4 a, b;   // (16-bit elements: a alone)
};
template <>
struct Raw<1> {
  uint32_t a;
};

template <int V, int P, int G>
__device__ __forceinline__ void read_row(const RowsArg &r, int64_t row, int C, int t, Raw<V> (&raw)[P]) {
  if (r.type == kT_F32) {
    const float *p = static_cast<const float *>(r.p) + row * r.ld;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int c = (j * G + t) * V;
      raw[j] = {};
      if (c < C) {
        if constexpr (V == 8) {
          raw[j].a = *reinterpret_cast<const uint4 *>(p + c);
          raw[j].b = *reinterpret_cast<const uint4 *>(p + c + 4);
        } else {
          raw[j].a = __float_as_uint(p[c]);
        }
      }
    }
  } else {
    const uint16_t *p = static_cast<const uint16_t *>(r.p) + row * r.ld;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int c = (j * G + t) * V;
      raw[j] = {};
      if (c < C) {
        if constexpr (V == 8) raw[j].a = *reinterpret_cast<const uint4 *>(p + c);
        else raw[j].a = p[c];
      }
    }
  }
}

template <int V>
__device__ __forceinline__ void widen_raw(int type, const Raw<V> &raw, float (&v)[V]) {
  if constexpr (V == 8) {
    const uint32_t u[8] = {raw.a.x, raw.a.y, raw.a.z, raw.a.w, raw.b.x, raw.b.y, raw.b.z, raw.b.w};
    if (type == kT_F32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(u[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = widen16(type, (uint16_t)(u[e / 2] >> (16 * (e % 2))));
    }
  } else {
    v[0] = type == kT_F32 ? __uint_as_float(raw.a) : widen16(type, (uint16_t)raw.a);
  }
}

template <int V, int P, int G>
__device__ __forceinline__ void write_row(const RowsArg &r, int64_t row, int C, int t, const float (&v)[P][V]) {
  if (r.type == kT_F32) {
    float *p = static_cast<float *>(r.p) + row * r.ld;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int c = (j * G + t) * V;
      if (c >= C) continue;
      if constexpr (V == 8) {
        *reinterpret_cast<float4 *>(p + c) = make_float4(v[j][0], v[j][1], v[j][2], v[j][3]);
        *reinterpret_cast<float4 *>(p + c + 4) = make_float4(v[j][4], v[j][5], v[j][6], v[j][7]);
      } else {
        p[c] = v[j][0];
      }
    }
  } else {
    uint16_t *p = static_cast<uint16_t *>(r.p) + row * r.ld;
#pragma unroll
    for (int j = 0; j < P; ++j) {
      const int c = (j * G + t) * V;
      if (c >= C) continue;
      if constexpr (V == 8) {
        uint32_t u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          u[e] = bits16(r.type, v[j][2 * e]) | (uint32_t)bits16(r.type, v[j][2 * e + 1]) << 16;
        *reinterpret_cast<uint4 *>(p + c) = make_uint4(u[0], u[1], u[2], u[3]);
      } else {
        p[c] = bits16(r.type, v[j][0]);
      }
    }
  }
}

// A parameter of the norm, one per channel.
template <int V>
__device__ __forceinline__ void read_param(const float *p, int c, float (&v)[V]) {
  if constexpr (V == 8) {
    const float4 a = *reinterpret_cast<const float4 *>(p + c), b = *reinterpret_cast<const float4 *>(p + c + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    v[0] = p[c];
  }
}

// The sum (or the largest) over a row's G threads; `slot` [G / 64] is this reduction's own.
template <int G>
__device__ __forceinline__ float row_sum(float v, float *slot, int t) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v += __shfl_xor(v, d);
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
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, d));
  if constexpr (G > 64) {
    if (t % 64 == 0) slot[t / 64] = v;
    __syncthreads();
    v = slot[0];
#pragma unroll
    for (int i = 1; i < G / 64; ++i) v = max(v, slot[i]);
  }
  return v;
}

template <int V, int P, int G>
__device__ __forceinline__ void norm_row(const NormArg &n, int C, int t, float (&v)[P][V], float (*slots)[16]) {
  if (n.kind == kNormNone) return;
  if (n.kind == kNormLayer) {
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < P; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e) s += v[j][e];
    const float mean = row_sum<G>(s, slots[0], t) / (float)C;
#pragma unroll
    for (int j = 0; j < P; ++j)
      if ((j * G + t) * V < C)
#pragma unroll
        for (int e = 0; e < V; ++e) v[j][e] -= mean;
  }
  float q = 0.0f;
#pragma unroll
  for (int j = 0; j < P; ++j)
#pragma unroll
    for (int e = 0; e < V; ++e) q = fmaf(v[j][e], v[j][e], q);
  const float r = 1.0f / sqrtf(row_sum<G>(q, slots[1], t) / (float)C + n.eps);
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const int c = (j * G + t) * V;
    if (c >= C) continue;
    float w[V];
#pragma unroll
    for (int e = 0; e < V; ++e) v[j][e] *= r;
    if (n.w) {
      read_param<V>(n.w, c, w);
#pragma unroll
      for (int e = 0; e < V; ++e) v[j][e] *= w[e];
    }
    if (n.b) {
      read_param<V>(n.b, c, w);
#pragma unroll
      for (int e = 0; e < V; ++e) v[j][e] += w[e];
    }
  }
}

// Threads of a workgroup: several rows where a row has one wave.
template <int G>
constexpr int kNormThreads = G > 256 ? G : 256;

template <int V, int P, int G>
__global__ void __launch_bounds__(kNormThreads<G>) block_norm_kernel(BlockNormArgs a) {
  __shared__ float slots[5][16];
  const int t = threadIdx.x % G;
  const int64_t row = (int64_t)blockIdx.x * (kNormThreads<G> / G) + threadIdx.x / G;
  if (row >= a.M) return;   // (whole waves; with barriers, G is the workgroup)
  Raw<V> raw[P], res[P];
  float v[P][V];
  read_row<V, P, G>(a.x, row, a.C, t, raw);
  if (a.res.p) read_row<V, P, G>(a.res, row, a.C, t, res);
#pragma unroll
  for (int j = 0; j < P; ++j) widen_raw<V>(a.x.type, raw[j], v[j]);
  norm_row<V, P, G>(a.after, a.C, t, v, slots);
  if (a.gate.p) {
    read_row<V, P, G>(a.gate, row, a.C, t, raw);
#pragma unroll
    for (int j = 0; j < P; ++j) {
      float g[V];
      widen_raw<V>(a.gate.type, raw[j], g);
#pragma unroll
      for (int e = 0; e < V; ++e) v[j][e] *= activation(a.act, g[e]);
    }
  }
#pragma unroll
  for (int j = 0; j < P; ++j)
#pragma unroll
    for (int e = 0; e < V; ++e) v[j][e] *= a.scale;
  if (a.res.p) {
#pragma unroll
    for (int j = 0; j < P; ++j) {
      float g[V];
      widen_raw<V>(a.res.type, res[j], g);
#pragma unroll
      for (int e = 0; e < V; ++e) v[j][e] += g[e];
    }
  }
  // (elements behind C are 0 up to here: they count in no sum below)
#pragma unroll
  for (int j = 0; j < P; ++j)
    if ((j * G + t) * V >= a.C)
#pragma unroll
      for (int e = 0; e < V; ++e) v[j][e] = 0.0f;
  if (a.sum.p) write_row<V, P, G>(a.sum, row, a.C, t, v);
  if (!a.out.p) return;
  norm_row<V, P, G>(a.before, a.C, t, v, slots + 2);
  if (a.out.type != kT_I8) {
    write_row<V, P, G>(a.out, row, a.C, t, v);
    return;
  }
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < P; ++j)
#pragma unroll
    for (int e = 0; e < V; ++e) most = max(most, __float_as_uint(v[j][e]) & 0x7FFFFFFFu);
  most = row_max<G>(most, reinterpret_cast<uint32_t *>(slots[4]), t);
  float inv;
  const float scale = scale_of(most, &inv);
  if (t == 0) a.out.scales[row] = scale;
  int8_t *p = static_cast<int8_t *>(a.out.p) + row * a.out.ld;
#pragma unroll
  for (int j = 0; j < P; ++j) {
    const int c = (j * G + t) * V;
    if (c >= a.C) continue;
    uint32_t u[(V + 3) / 4] = {};
#pragma unroll
    for (int e = 0; e < V; ++e)
      u[e / 4] |= (uint32_t)(inv > 0.0f ? quantised(v[j][e], inv, scale) & 255 : 0) << (8 * (e % 4));
    if constexpr (V == 8) *reinterpret_cast<uint2 *>(p + c) = make_uint2(u[0], u[1]);
    else p[c] = (int8_t)u[0];
  }
}

template <int V, int P, int G>
hipError_t launch(const BlockNormArgs &a, hipStream_t stream, hipEvent_t *ev, hipEvent_t done) {
  constexpr int per = kNormThreads<G> / G;
  return launch_timed(block_norm_kernel<V, P, G>, dim3((unsigned)((a.M + per - 1) / per)), kNormThreads<G>,
                      stream, ev, done, a);
}

}  // namespace

hipError_t launch_block_norm(const BlockNormArgs &a, hipStream_t stream, hipEvent_t *ev, hipEvent_t done) {
  const int64_t C = a.C;
  if (a.vec) {
    if (C <= 512) return launch<8, 1, 64>(a, stream, ev, done);
    if (C <= 2048) return launch<8, 1, 256>(a, stream, ev, done);
    if (C <= 4096) return launch<8, 2, 256>(a, stream, ev, done);
    if (C <= 8192) return launch<8, 1, 1024>(a, stream, ev, done);
    if (C <= 16384) return launch<8, 2, 1024>(a, stream, ev, done);
    return launch<8, 4, 1024>(a, stream, ev, done);
  }
  if (C <= 256) return launch<1, 4, 64>(a, stream, ev, done);
  if (C <= 2048) return launch<1, 8, 256>(a, stream, ev, done);
  if (C <= 8192) return launch<1, 32, 256>(a, stream, ev, done);
  return launch<1, 32, 1024>(a, stream, ev, done);
}

}  // namespace hs

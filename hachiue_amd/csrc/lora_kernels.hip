// Low-rank adapters of many requests at once, beside a shared projection, on
// gfx950:
//   y[m] = base[m] + scale_s sum_j t[m][j] B_s[.][j],  t[m][j] = sum_k x[m][k] A_s[j][k]
// for row m's adapter s = slots[m] (y = base where it names none).  x, base
// and y are binary32; the adapters' A [rank][K] and B [N][rank] are stacked,
// binary32, binary16 or bfloat16.
//
// Two launches: x A^T into a workspace (binary32, the scale on it), then B.
// Both run on the matrix cores' binary32 products (16 x 16 x 4): the adapters
// widen to binary32 exactly, so nothing is rounded but the sums.  Rows go in
// tiles of 16 as they come.  A tile is computed once for every adapter that
// its rows name and each row keeps the result of its own: rows of one prompt
// follow each other and share one pass, a batch with an adapter per row reads
// each adapter once.  No sorting, and a row's result does not depend on its
// neighbours: an infinity or NaN in one adapter or row reaches no other.
#include "sampler_internal.h"

#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>

#include <algorithm>

namespace hs {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
struct BF16 {
  uint16_t u;
};

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(_Float16 v) { return (float)v; }
__device__ __forceinline__ float widen(BF16 v) { return __uint_as_float((uint32_t)v.u << 16); }

// n consecutive elements at any alignment of theirs, as they are stored.
template <typename T, int n>
struct __attribute__((packed, aligned(sizeof(T)))) Run {
  T v[n];
};
template <int n, typename T>
__device__ __forceinline__ Run<T, n> load_run(const T *p) {
  return *reinterpret_cast<const Run<T, n> *>(p);
}
// Elements [0, left) of n; the others are 0 and not read.
template <int n, typename T>
__device__ __forceinline__ Run<T, n> load_run(const T *p, int left) {
  Run<T, n> r = {};
  if (left >= n) return load_run<n>(p);
#pragma unroll
  for (int i = 0; i < n; ++i)
    if (i < left) r.v[i] = p[i];
  return r;
}

// The adapter of the tile's row `lane & 15`, -1: none.
__device__ __forceinline__ int slot_of(const LoraArgs &g, int m0) {
  const int m = m0 + (threadIdx.x & 15);
  const int s = m < g.M ? g.slots[m] : -1;
  return s >= 0 && s < g.count ? s : -1;
}

// t = scale x A^T of one tile and one of its adapters (block x: the x-th
// different one, in the order of the rows that name them).  K is cut over the
// workgroup's waves; their sums meet in LDS.  JB blocks of 16 ranks a wave.
// In a step of 32 k, lanes l, l + 16, ... hold 8 consecutive k each; the next
// step is on its way while one is multiplied.
template <typename T, int JB, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void lora_shrink_kernel(LoraArgs g) {
  __shared__ float sums[WAVES][JB][256];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int m0 = blockIdx.z * 16, j0 = blockIdx.y * (16 * JB);
  const int own = slot_of(g, m0);
  uint32_t todo = (uint32_t)__ballot(own >= 0) & 0xFFFFu;
  int s = -1;
  for (int i = 0; todo && i <= (int)blockIdx.x; ++i) {
    s = __builtin_amdgcn_readlane(own, __ffs(todo) - 1);
    const uint32_t same = (uint32_t)__ballot(own == s) & 0xFFFFu;
    if (i < (int)blockIdx.x) s = -1;
    todo &= ~same;
  }
  if (s < 0) return;
  const int rank = g.ranks ? min(max(g.ranks[s], 0), g.rank) : g.rank;
  const float scale = g.scales ? g.scales[s] : 1.0f;
  const int i16 = lane & 15, grp = lane >> 4;
  const float *x = g.x + (int64_t)min(m0 + i16, g.M - 1) * g.ldx + grp * 8;
  const T *A = static_cast<const T *>(g.a) + (int64_t)s * g.rank * g.K + grp * 8;
  const T *arow[JB];
#pragma unroll
  for (int j = 0; j < JB; ++j) arow[j] = A + (int64_t)min(j0 + 16 * j + i16, g.rank - 1) * g.K;
  f32x4 acc[JB];
#pragma unroll
  for (int j = 0; j < JB; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  auto multiply = [&](const Run<float, 8> &xv, const Run<T, 8> (&av)[JB]) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < JB; ++j)
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(xv.v[i], widen(av[j].v[i]), acc[j], 0, 0, 0);
  };
  const int whole = g.K / 32 * 32;
  int k = wave * 32;
  if (k < whole) {
    Run<float, 8> xn = load_run<8>(x + k);
    Run<T, 8> an[JB];
#pragma unroll
    for (int j = 0; j < JB; ++j) an[j] = load_run<8>(arow[j] + k);
    for (;;) {
      const Run<float, 8> xv = xn;
      Run<T, 8> av[JB];
#pragma unroll
      for (int j = 0; j < JB; ++j) av[j] = an[j];
      k += WAVES * 32;
      const bool more = k < whole;
      if (more) {
        xn = load_run<8>(x + k);
#pragma unroll
        for (int j = 0; j < JB; ++j) an[j] = load_run<8>(arow[j] + k);
      }
      multiply(xv, av);
      if (!more) break;
    }
  }
  if (whole < g.K && whole / 32 % WAVES == wave) {   // the last, short step
    const int left = g.K - whole - grp * 8;
    const Run<float, 8> xv = load_run<8>(x + whole, left);
    Run<T, 8> av[JB];
#pragma unroll
    for (int j = 0; j < JB; ++j) av[j] = load_run<8>(arow[j] + whole, left);
    multiply(xv, av);
  }
  // acc: rows 4 grp + i of the tile, rank i16
#pragma unroll
  for (int j = 0; j < JB; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[wave][j][(4 * grp + i) * 16 + i16] = acc[j][i];
  __syncthreads();
  for (int e = tid; e < JB * 256; e += WAVES * 64) {
    const int j = e >> 8, row = (e >> 4) & 15, jj = j0 + 16 * j + (e & 15);
    float v = 0.0f;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) v += sums[w][j][e & 255];
    // (ranks that the adapter lacks: whatever its stack holds there, nothing)
    if (__shfl(own, row) == s && jj < g.rank_pad)
      g.t[(int64_t)(m0 + row) * g.rank_pad + jj] = jj < rank ? v * scale : 0.0f;
  }
}

constexpr int kExpandWaves = 4;

// y of one tile of 16 rows and NT tiles of 16 results a wave: for each adapter
// that the rows name, its B times the tile's t.  In a step of 4 VK ranks, lanes
// l, l + 16, ... hold VK consecutive ones each; the rows' t stay in registers,
// and the next step's B (of the next adapter after an adapter's last) is on
// its way while one is multiplied.  RB: blocks of 16 ranks.
template <typename T, int RB, int NT>
__global__ __launch_bounds__(kExpandWaves * 64) void lora_expand_kernel(LoraArgs g) {
  constexpr int VK = RB == 1 ? 4 : 8, STEPS = RB * 4 / VK;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int i16 = lane & 15, grp = lane >> 4;
  const int m0 = blockIdx.y * 16, m = m0 + i16;
  const int n0 = ((int)blockIdx.x * kExpandWaves + wave) * (16 * NT);
  if (n0 >= g.N) return;
  const int own = slot_of(g, m0);
  uint32_t todo = (uint32_t)__ballot(own >= 0) & 0xFFFFu;
  const int64_t mr = min(m, g.M - 1);
  float *y = g.y + mr * g.ldy + n0 + 4 * grp;
  const float *base = g.base ? g.base + mr * g.ldb + n0 + 4 * grp : nullptr;
  const bool whole = n0 + 16 * NT <= g.N;
  Run<float, 4> old[NT] = {};
  if (base && whole) {
#pragma unroll
    for (int n = 0; n < NT; ++n) old[n] = load_run<4>(base + 16 * n);
  }
  f32x4 out[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) out[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (todo) {
    float t[STEPS][VK];
    const float *tp = g.t + mr * g.rank_pad + grp * VK;
#pragma unroll
    for (int r = 0; r < STEPS; ++r)
#pragma unroll
      for (int i = 0; i < VK; i += 4) {
        const f32x4 v = *reinterpret_cast<const f32x4 *>(tp + r * 4 * VK + i);
#pragma unroll
        for (int e = 0; e < 4; ++e) t[r][i + e] = v[e];
      }
    const T *B = static_cast<const T *>(g.b);
    int64_t brow[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) brow[n] = (int64_t)min(n0 + 16 * n + i16, g.N - 1) * g.rank;
    // A run of VK may pass its row's end, and is masked there, but not the
    // stack's: rows whose runs could are read element by element.
    const int64_t per = (int64_t)g.N * g.rank, end = per * g.count;
    const int64_t reach = (int64_t)(min(n0 + 16 * NT, g.N) - 1) * g.rank + (g.rank - 1) / VK * VK + VK;
    auto load = [&](int s, int r, Run<T, VK> (&v)[NT]) {
      const int k = r * 4 * VK + grp * VK;
      const T *Bs = B + s * per;
      if (s * per + reach <= end) {
#pragma unroll
        for (int n = 0; n < NT; ++n) v[n] = load_run<VK>(Bs + brow[n] + (k < g.rank ? k : 0));
      } else {
#pragma unroll
        for (int n = 0; n < NT; ++n) v[n] = load_run<VK>(Bs + brow[n] + k, g.rank - k);
      }
    };
    auto take = [&](int &rank) {   // the next adapter of the tile, its ranks
      const int s = __builtin_amdgcn_readlane(own, __ffs(todo) - 1);
      todo &= ~((uint32_t)__ballot(own == s) & 0xFFFFu);
      rank = g.ranks ? min(max(g.ranks[s], 0), g.rank) : g.rank;
      return s;
    };
    int rank, s = take(rank);
    Run<T, VK> next[NT];
    load(s, 0, next);
    for (;;) {
      const bool more = todo != 0;
      int rank2 = 0, s2 = s;
      if (more) s2 = take(rank2);
      f32x4 acc[NT];
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int r = 0; r < STEPS; ++r) {
        Run<T, VK> b[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) b[n] = next[n];
        if (r + 1 < STEPS) load(s, r + 1, next);
        else if (more) load(s2, 0, next);
        const int k = r * 4 * VK + grp * VK;
        const bool full = (r + 1) * 4 * VK <= rank;
#pragma unroll
        for (int i = 0; i < VK; ++i)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            float w = widen(b[n].v[i]);
            if (!full) w = k + i < rank ? w : 0.0f;   // (t is 0 there too; B may be anything)
            acc[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(w, t[r][i], acc[n], 0, 0, 0);
          }
      }
      // acc: results 4 grp + i of a tile, row i16
#pragma unroll
      for (int n = 0; n < NT; ++n)
        if (own == s) out[n] = acc[n];
      if (!more) break;
      s = s2;
      rank = rank2;
    }
  }
  if (m >= g.M || (own < 0 && base == y)) return;
  if (whole) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      Run<float, 4> o;
#pragma unroll
      for (int i = 0; i < 4; ++i)
        o.v[i] = own < 0 ? old[n].v[i] : base ? old[n].v[i] + out[n][i] : out[n][i];
      *reinterpret_cast<Run<float, 4> *>(y + 16 * n) = o;
    }
    return;
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (n0 + 16 * n + 4 * grp + i >= g.N) continue;
      const float b = base ? base[16 * n + i] : 0.0f;
      y[16 * n + i] = own < 0 ? b : base ? b + out[n][i] : out[n][i];
    }
}

template <typename K>
hipError_t launch_l(K kernel, dim3 grid, int threads, hipStream_t stream, hipEvent_t *ev,
                    hipEvent_t done, const LoraArgs &g) {
  const dim3 block((unsigned)threads);
  if (ev)
    hipExtLaunchKernelGGL(kernel, grid, block, 0u, stream, ev[0], ev[1], 0u, g);
  else if (done)
    hipExtLaunchKernelGGL(kernel, grid, block, 0u, stream, nullptr, done, 0u, g);
  else
    hipLaunchKernelGGL(kernel, grid, block, 0, stream, g);
  return hipGetLastError();
}

template <typename T>
hipError_t shrink(const LoraArgs &g, hipStream_t stream, hipEvent_t *ev) {
  const int blocks = g.rank_pad / 16;
  const unsigned tiles = (unsigned)((g.M + 15) / 16), kinds = (unsigned)std::min({16, g.M, g.count});
  // as many blocks of ranks a wave (each reads x once) as leave a workgroup
  // for every compute unit
  const int per = blocks >= 4 && tiles * (unsigned)(blocks / 4) >= (unsigned)kSplitCUs   ? 4
                  : blocks >= 2 && tiles * (unsigned)(blocks / 2) >= (unsigned)kSplitCUs ? 2
                                                                                         : 1;
  const dim3 grid(kinds, (unsigned)(blocks / per), tiles);
  if (per == 4) return launch_l(lora_shrink_kernel<T, 4, 8>, grid, 512, stream, ev, nullptr, g);
  if (per == 2) return launch_l(lora_shrink_kernel<T, 2, 8>, grid, 512, stream, ev, nullptr, g);
  return launch_l(lora_shrink_kernel<T, 1, 8>, grid, 512, stream, ev, nullptr, g);
}

template <typename T, int NT>
hipError_t expand_by_rank(const LoraArgs &g, hipStream_t stream, hipEvent_t *ev, hipEvent_t done) {
  const int per = kExpandWaves * 16 * NT;
  const dim3 grid((unsigned)((g.N + per - 1) / per), (unsigned)((g.M + 15) / 16));
  const int threads = kExpandWaves * 64;
  switch (g.rank_pad / 16) {
    case 1: return launch_l(lora_expand_kernel<T, 1, NT>, grid, threads, stream, ev, done, g);
    case 2: return launch_l(lora_expand_kernel<T, 2, NT>, grid, threads, stream, ev, done, g);
    case 4: return launch_l(lora_expand_kernel<T, 4, NT>, grid, threads, stream, ev, done, g);
    case 8: return launch_l(lora_expand_kernel<T, 8, NT>, grid, threads, stream, ev, done, g);
    default: return launch_l(lora_expand_kernel<T, 16, NT>, grid, threads, stream, ev, done, g);
  }
}

template <typename T>
hipError_t expand(const LoraArgs &g, hipStream_t stream, hipEvent_t *ev, hipEvent_t done) {
  const int64_t tiles = (int64_t)((g.N + 15) / 16) * ((g.M + 15) / 16);
  return tiles >= 4096 ? expand_by_rank<T, 4>(g, stream, ev, done)
                       : expand_by_rank<T, 1>(g, stream, ev, done);
}

}  // namespace

hipError_t launch_lora_shrink(const LoraArgs &g, hipStream_t stream, hipEvent_t *ev) {
  switch (g.type) {
    case kA_F32: return shrink<float>(g, stream, ev);
    case kA_F16: return shrink<_Float16>(g, stream, ev);
    default: return shrink<BF16>(g, stream, ev);
  }
}

hipError_t launch_lora_expand(const LoraArgs &g, hipStream_t stream, hipEvent_t *ev, hipEvent_t done) {
  switch (g.type) {
    case kA_F32: return expand<float>(g, stream, ev, done);
    case kA_F16: return expand<_Float16>(g, stream, ev, done);
    default: return expand<BF16>(g, stream, ev, done);
  }
}

}  // namespace hs

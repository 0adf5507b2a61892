// Low-rank adapters of many requests at once, beside a shared projection, on
// gfx950:
//   y[m] = base[m] + scale_s sum_j t[m][j] B_s[.][j],  t[m][j] = sum_k x[m][k] A_s[j][k]
// for row m's adapter s = slots[m] (y = base where it names none).  x, base
// and y are binary32; the adapters' A [rank][K] and B [N][rank] are stacked,
// binary32, binary16 or bfloat16.
//
// Two launches: x A^T into a workspace (binary32, the scale on it), then B.
// Binary16 and binary32 adapters run on the matrix cores' binary32 products
// (16 x 16 x 4), to which they widen exactly; bfloat16 ones on bfloat16 products
// with x and t as three exact parts.  Nothing is rounded but the binary32 sums,
// either way.  Rows go in
// tiles of 16 as they come.  A tile is computed once for every adapter that
// its rows name and each row keeps the result of its own: rows of one prompt
// follow each other and share one pass, a batch with an adapter per row reads
// each adapter once.  No sorting, and a row's result does not depend on its
// neighbours: an infinity or NaN in one adapter or row reaches no other.  It
// does depend on how many rows there are: the shares of K and the kernel of the
// second product go by M, and with them the order of the binary32 sums.
#include "sampler_internal.h"

#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

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

// The same in LDS, 16-byte aligned.
template <typename T, int n>
struct alignas(16) Lane {
  T v[n];
};

// A binary32 value as the exact sum of three bfloat16 ones (its leading 8 bits,
// the next 8, the last 8; below 2^-110 the last may underflow): its products
// with a bfloat16 are then three bfloat16 products, which the matrix cores
// sum in binary32 at sixteen times the rate of binary32 ones.  An infinity is
// one part, a NaN stays one; where the bfloat16 value is infinite, the lower parts,
// which are 0 in values of few bits, meet its largest finite neighbour instead
// (0 times an infinity is NaN; the parts have one sign, so that the sum is the
// leading part's infinity).  (2048 rows x 4096, rank 64: 42.7 us a call, 55 with
// binary32 products.  A binary16 value is two bfloat16 ones, which would have to
// be parted in every workgroup that reads it: twice the products and that.)
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short bf16x4 __attribute__((ext_vector_type(4)));
template <int n>
struct Operand;
template <>
struct Operand<8> {
  typedef bf16x8 V;
};
template <>
struct Operand<4> {
  typedef bf16x4 V;
};
__device__ __forceinline__ f32x4 mfma_bf16(bf16x8 a, bf16x8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma_bf16(bf16x4 a, bf16x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0);
}
template <int n>
struct Parts {
  typename Operand<n>::V v[3];   // the leading first
};
template <int n>
__device__ __forceinline__ Parts<n> parts_of(const float (&x)[n]) {
  union {
    uint32_t u[n / 2];
    typename Operand<n>::V v;
  } p[3];
#pragma unroll
  for (int i = 0; i < n; i += 2) {
    uint32_t u[3][2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const float f = x[i + e];
      u[0][e] = __float_as_uint(f);
      float r = f - __uint_as_float(u[0][e] & 0xFFFF0000u);
      r = __builtin_fabsf(f) == __builtin_inff() ? 0.0f : r;
      u[1][e] = __float_as_uint(r);
      u[2][e] = __float_as_uint(r - __uint_as_float(u[1][e] & 0xFFFF0000u));
    }
#pragma unroll
    for (int j = 0; j < 3; ++j) p[j].u[i / 2] = __builtin_amdgcn_perm(u[j][1], u[j][0], 0x07060302u);
  }
  return {{p[0].v, p[1].v, p[2].v}};
}

// bfloat16 values with the largest finite ones in place of infinities (and NaN,
// which the leading part's product keeps).
template <typename V>
__device__ __forceinline__ V finite_of(V a) {
  typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
  typedef short i16x2 __attribute__((ext_vector_type(2)));
  union {
    V v;
    u16x2 u[sizeof(V) / 4];
  } r;
  r.v = a;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(V) / 4); ++i) {
    // as unsigned numbers the negative ones are the larger, as signed the positive
    const u16x2 n = __builtin_elementwise_min(r.u[i], (u16x2)(unsigned short)0xFF7F);
    r.u[i] = __builtin_bit_cast(u16x2, __builtin_elementwise_min(__builtin_bit_cast(i16x2, n), (i16x2)(short)0x7F7F));
  }
  return r.v;
}
// acc += x w (or w x: SWAP) of x in parts, the lower ones first.
template <bool SWAP, int n>
__device__ __forceinline__ f32x4 mfma_parts(const Parts<n> &x, typename Operand<n>::V w, f32x4 acc) {
  const typename Operand<n>::V f = finite_of(w);
#pragma unroll
  for (int i = 2; i >= 0; --i)
    acc = SWAP ? mfma_bf16(i ? f : w, x.v[i], acc) : mfma_bf16(x.v[i], i ? f : w, acc);
  return acc;
}

// The adapter of the tile's row `lane & 15`, -1: none.
__device__ __forceinline__ int slot_of(const LoraArgs &g, int m0) {
  const int m = m0 + (threadIdx.x & 15);
  const int s = m < g.M ? g.slots[m] : -1;
  return s >= 0 && s < g.count ? s : -1;
}

// The sum of the shares' t (1 to 4 of them, `share` floats apart): all reads on
// their way together.
__device__ __forceinline__ f32x4 t_of(const float *p, int64_t share, int splits) {
  f32x4 v = *reinterpret_cast<const f32x4 *>(p);
  if (splits > 1) {
    const f32x4 a = *reinterpret_cast<const f32x4 *>(p + share);
    const f32x4 b = *reinterpret_cast<const f32x4 *>(p + min(2, splits - 1) * share);
    const f32x4 c = *reinterpret_cast<const f32x4 *>(p + (splits - 1) * share);
    v += a;
    if (splits > 2) v += b;
    if (splits > 3) v += c;
  }
  return v;
}

constexpr int kShrinkWaves = 8;
constexpr int kShrinkK = kShrinkWaves * 32;   // k of a stage

// t = scale x A^T of one tile and the adapters that its rows name, in the order
// of the rows (block z takes every gridDim.z-th of them).  A workgroup takes JB
// blocks of 16 ranks and one of `splits` shares of K, in stages of 256 k through
// LDS: rows are read along k, a wave instruction 1 KB of one row, because the
// matrix operand's own order (16 rows side by side in the lanes) makes the cache
// look up a line per lane.  The next stage is on its way while one is
// multiplied, each wave 32 of its k, lanes l, l + 16, ... 8 consecutive ones
// each; the waves' sums meet in LDS.
// Bound: for prompts a stage's latency (2048 rows x 4096, rank 64, bfloat16:
// 16.5 us, of which 8 stages 1.4 each; x at 2 TB/s, A from L2), for a few rows that
// of the one chain over K (one row x 2048 4.5 us, 32 rows with an adapter each
// 6.0).
template <typename T, int JB>
__global__ __launch_bounds__(kShrinkWaves * 64) void lora_shrink_kernel(LoraArgs g) {
  // (rows 16 bytes longer than a stage: the operands' reads meet no bank twice)
  constexpr int XS = kShrinkK + 4, AS = kShrinkK + 16 / (int)sizeof(T);
  constexpr int PER = 16 / (int)sizeof(T);        // elements of a 16-byte read
  constexpr int RPI = 64 * PER / kShrinkK;        // rows of A an instruction
  constexpr int AI = 16 * JB / RPI / kShrinkWaves;
  static_assert(AI * RPI * kShrinkWaves == 16 * JB, "a stage of A is whole reads");
  union alignas(16) Lds {
    struct {
      float x[16][XS];
      T a[16 * JB][AS];
    } in;
    float sums[kShrinkWaves][JB][256];
  };
  __shared__ Lds lds;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int groups = g.rank_pad / (16 * JB);
  // tiles that follow each other, which share adapters, go to one XCD's cache
  const int eighth = gridDim.x >> 3, xcd = blockIdx.x & 7;
  const int tile = xcd * eighth + min(xcd, (int)gridDim.x & 7) + (int)(blockIdx.x >> 3);
  const int m0 = tile * 16, j0 = (int)blockIdx.y % groups * (16 * JB);
  const int split = (int)blockIdx.y / groups;
  const int own = slot_of(g, m0);
  uint32_t todo = (uint32_t)__ballot(own >= 0) & 0xFFFFu;
  const int i16 = lane & 15, grp = lane >> 4;
  // this share's stages
  const int stages = (g.K + kShrinkK - 1) / kShrinkK, per = (stages + g.splits - 1) / g.splits;
  const int k0 = split * per * kShrinkK, k1 = min(k0 + per * kShrinkK, g.K);
  float *t = g.t + (int64_t)split * g.M * g.rank_pad;
  for (int turn = 0; todo; ++turn) {
    const int s = __builtin_amdgcn_readlane(own, __ffs(todo) - 1);
    todo &= ~((uint32_t)__ballot(own == s) & 0xFFFFu);
    if (turn % (int)gridDim.z != (int)blockIdx.z) continue;
    const int rank = g.ranks ? min(max(g.ranks[s], 0), g.rank) : g.rank;
    const float scale = g.scales ? g.scales[s] : 1.0f;
    // what this thread reads of a stage: two rows of x, AI times PER elements of A
    const int xk = lane * 4, ak = lane * PER % kShrinkK, ar = lane * PER / kShrinkK;
    const float *xrow[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
      xrow[h] = g.x + (int64_t)min(m0 + 2 * wave + h, g.M - 1) * g.ldx + xk;
    const T *arow[AI];
    int ai[AI];
#pragma unroll
    for (int h = 0; h < AI; ++h) {
      ai[h] = (wave + h * kShrinkWaves) * RPI + ar;
      arow[h] = static_cast<const T *>(g.a) +
                ((int64_t)s * g.rank + min(j0 + ai[h], g.rank - 1)) * g.K + ak;
    }
    f32x4 acc[JB];
#pragma unroll
    for (int j = 0; j < JB; ++j) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    Run<float, 4> xn[2];
    Run<T, PER> an[AI];
    auto put = [&]() {
#pragma unroll
      for (int h = 0; h < 2; ++h)
        *reinterpret_cast<Lane<float, 4> *>(&lds.in.x[2 * wave + h][xk]) =
            __builtin_bit_cast(Lane<float, 4>, xn[h]);
#pragma unroll
      for (int h = 0; h < AI; ++h)
        *reinterpret_cast<Lane<T, PER> *>(&lds.in.a[ai[h]][ak]) =
            __builtin_bit_cast(Lane<T, PER>, an[h]);
    };
    auto multiply = [&]() {
      const int kk = wave * 32 + grp * 8;
      const Lane<float, 8> xv = *reinterpret_cast<const Lane<float, 8> *>(&lds.in.x[i16][kk]);
      if constexpr (std::is_same_v<T, BF16>) {
        const Parts<8> xp = parts_of(xv.v);
#pragma unroll
        for (int j = 0; j < JB; ++j) {
          const bf16x8 av = *reinterpret_cast<const bf16x8 *>(&lds.in.a[16 * j + i16][kk]);
          acc[j] = mfma_parts<false>(xp, av, acc[j]);
        }
        return;
      }
#pragma unroll
      for (int j = 0; j < JB; ++j) {
        const Lane<T, 8> av = *reinterpret_cast<const Lane<T, 8> *>(&lds.in.a[16 * j + i16][kk]);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(xv.v[i], widen(av.v[i]), acc[j], 0, 0, 0);
      }
    };
    // Whole stages: the reads are never skipped (behind the last they repeat
    // it).  One stage ahead: two take the registers of the second workgroup of
    // a compute unit, 24 us where this takes 17.
    const int whole = max(k1 - k0, 0) / kShrinkK;
    if (whole > 0) {
      auto read = [&](int stage) {
        const int k = k0 + min(stage, whole - 1) * kShrinkK;
#pragma unroll
        for (int h = 0; h < 2; ++h) xn[h] = load_run<4>(xrow[h] + k);
#pragma unroll
        for (int h = 0; h < AI; ++h) an[h] = load_run<PER>(arow[h] + k);
      };
      read(0);
      for (int stage = 1; stage <= whole; ++stage) {
        put();
        __syncthreads();
        read(stage);
        multiply();
        __syncthreads();
      }
    }
    if (const int k = k0 + whole * kShrinkK; k < k1) {   // what is left of K
#pragma unroll
      for (int h = 0; h < 2; ++h) xn[h] = load_run<4>(xrow[h] + k, g.K - k - xk);
#pragma unroll
      for (int h = 0; h < AI; ++h) an[h] = load_run<PER>(arow[h] + k, g.K - k - ak);
      put();
      __syncthreads();
      multiply();
      __syncthreads();
    }
    // acc: rows 4 grp + i of the tile, rank i16
#pragma unroll
    for (int j = 0; j < JB; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) lds.sums[wave][j][(4 * grp + i) * 16 + i16] = acc[j][i];
    __syncthreads();
    for (int e = tid; e < JB * 256; e += kShrinkWaves * 64) {
      const int j = e >> 8, row = (e >> 4) & 15, jj = j0 + 16 * j + (e & 15);
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < kShrinkWaves; ++w) v += lds.sums[w][j][e & 255];
      // (ranks that the adapter lacks: whatever its stack holds there, nothing)
      if (__shfl(own, row) == s) t[(int64_t)(m0 + row) * g.rank_pad + jj] = jj < rank ? v * scale : 0.0f;
    }
    if (todo) __syncthreads();   // (the sums are read; the next adapter's stage goes there)
  }
}

constexpr int kExpandWaves = 4;

// y of one tile of 16 rows and NT tiles of 16 results a wave: for each adapter
// that the rows name, its B times the tile's t.  In a step of 4 VK ranks, lanes
// l, l + 16, ... hold VK consecutive ones each; the rows' t stay in registers,
// and the next step's B (of the next adapter after an adapter's last) is on
// its way while one is multiplied.  RB: blocks of 16 ranks.
// Bound: memory; 32 rows with an adapter each over 151936 results at rank 16
// (194 MB) 45 us, 4.3 TB/s.  One row (6 MB) 4.5 us, which is a launch.
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
  // what does not wait for the slots
  const int64_t mr = min(m, g.M - 1);
  float *y = g.y + mr * g.ldy + n0 + 4 * grp;
  const float *base = g.base ? g.base + mr * g.ldb + n0 + 4 * grp : nullptr;
  const bool whole = n0 + 16 * NT <= g.N;
  Run<float, 4> old[NT] = {};
  if (base && whole) {
#pragma unroll
    for (int n = 0; n < NT; ++n) old[n] = load_run<4>(base + 16 * n);
  }
  float t[STEPS][VK];
#pragma unroll
  for (int r = 0; r < STEPS; ++r)
#pragma unroll
    for (int i = 0; i < VK; i += 4) {
      f32x4 v = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      if (g.count > 0)
        v = t_of(g.t + mr * g.rank_pad + grp * VK + r * 4 * VK + i, (int64_t)g.M * g.rank_pad, g.splits);
#pragma unroll
      for (int e = 0; e < 4; ++e) t[r][i + e] = v[e];
    }
  constexpr bool parted = std::is_same_v<T, BF16>;
  Parts<VK> tp[parted ? STEPS : 1];
  if constexpr (parted) {
#pragma unroll
    for (int r = 0; r < STEPS; ++r) tp[r] = parts_of(t[r]);
  }
  uint32_t todo = (uint32_t)__ballot(own >= 0) & 0xFFFFu;
  f32x4 out[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) out[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  if (todo) {
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
        if constexpr (parted) {
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            if (!full) {
#pragma unroll
              for (int i = 0; i < VK; ++i) b[n].v[i].u = k + i < rank ? b[n].v[i].u : (uint16_t)0;
            }
            acc[n] = mfma_parts<true>(tp[r], __builtin_bit_cast(typename Operand<VK>::V, b[n]), acc[n]);
          }
          continue;
        }
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

// The same for longer ranks and many results, a workgroup a tile of 16 rows and
// 256 results: B goes through LDS in chunks of 128 bytes of each of its rows, and
// the results back through it, so that every read and write of memory runs along
// rows (the operands' own order, a lane a row, costs the cache a look-up per lane,
// which bounds the kernel above once a row of B is longer than a line).  The next
// chunk (of the next adapter after an adapter's last) is on its way while
// one is multiplied.  2048 rows x 4096 at rank 64, bfloat16:
// 23 us, 2.9 TB/s of base and y.
template <typename T>
__global__ __launch_bounds__(256, 3) void lora_expand_wide_kernel(LoraArgs g) {
  constexpr int CH = 128 / (int)sizeof(T), PER = 16 / (int)sizeof(T);   // a chunk's ranks, a read's
  constexpr int BS = CH + PER, TS = CH + 4, OS = 256 + 4;               // LDS row strides (no bank twice)
  union alignas(16) Lds {
    struct {
      T b[256][BS];
      float t[16][TS];
    } in;
    float out[16][OS];
  };
  __shared__ Lds lds;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int i16 = lane & 15, grp = lane >> 4;
  const int m0 = blockIdx.y * 16, n0 = blockIdx.x * 256;
  const int own = slot_of(g, m0);
  // this thread's results: rows 4 wave + j, four of them from column c on
  const int c = n0 + lane * 4;
  Run<float, 4> old[4] = {};
  if (g.base) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      old[j] = load_run<4>(g.base + (int64_t)min(m0 + 4 * wave + j, g.M - 1) * g.ldb + c, g.N - c);
  }
  uint32_t todo = (uint32_t)__ballot(own >= 0) & 0xFFFFu;
  int s = -1, rank = 0, at = 0;   // the chunk that is on its way: its adapter, first rank
  // the next one: false where there is none
  auto step = [&]() {
    at += CH;
    while (at >= rank) {          // (adapters of no rank give 0)
      if (!todo) return false;
      s = __builtin_amdgcn_readlane(own, __ffs(todo) - 1);
      todo &= ~((uint32_t)__ballot(own == s) & 0xFFFFu);
      rank = g.ranks ? min(max(g.ranks[s], 0), g.rank) : g.rank;
      at = 0;
    }
    return true;
  };
  // a chunk: rows tid / 8 + 32 h, PER ranks from PER (tid % 8) on; t: row
  // tid / (CH / 4), four ranks
  const int br = tid >> 3, bk = (tid & 7) * PER;
  const int tr = tid / (CH / 4), tk = tid % (CH / 4) * 4;
  Run<T, PER> bn[8];
  f32x4 tn;
  auto read = [&]() {
    const T *B = static_cast<const T *>(g.b) + (int64_t)s * g.N * g.rank + at + bk;
    const int left = rank - at - bk;   // (ranks that the adapter lacks: 0)
#pragma unroll
    for (int h = 0; h < 8; ++h)
      bn[h] = load_run<PER>(B + (int64_t)min(n0 + br + 32 * h, g.N - 1) * g.rank, left);
    tn = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (tr < 16 && at + tk < g.rank_pad)
      tn = t_of(g.t + (int64_t)min(m0 + tr, g.M - 1) * g.rank_pad + at + tk,
                (int64_t)g.M * g.rank_pad, g.splits);
  };
  f32x4 out[4], acc[4];
#pragma unroll
  for (int n = 0; n < 4; ++n) out[n] = acc[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  bool more = step();
  if (more) read();
  while (more) {
    const int s1 = s, live = rank - at;
#pragma unroll
    for (int h = 0; h < 8; ++h)
      *reinterpret_cast<Lane<T, PER> *>(&lds.in.b[br + 32 * h][bk]) =
          __builtin_bit_cast(Lane<T, PER>, bn[h]);
    if (tr < 16) *reinterpret_cast<f32x4 *>(&lds.in.t[tr][tk]) = tn;
    __syncthreads();
    more = step();
    if (more) read();
#pragma unroll
    for (int k = 0; k < CH; k += 32) {
      if (k >= live) break;
      const Lane<float, 8> tv = *reinterpret_cast<const Lane<float, 8> *>(&lds.in.t[i16][k + grp * 8]);
      if constexpr (std::is_same_v<T, BF16>) {
        const Parts<8> tp = parts_of(tv.v);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const bf16x8 b =
              *reinterpret_cast<const bf16x8 *>(&lds.in.b[wave * 64 + 16 * n + i16][k + grp * 8]);
          acc[n] = mfma_parts<true>(tp, b, acc[n]);
        }
        continue;
      }
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const Lane<T, 8> b =
            *reinterpret_cast<const Lane<T, 8> *>(&lds.in.b[wave * 64 + 16 * n + i16][k + grp * 8]);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          acc[n] = __builtin_amdgcn_mfma_f32_16x16x4f32(widen(b.v[i]), tv.v[i], acc[n], 0, 0, 0);
      }
    }
    if (!more || s != s1) {   // the adapter's last chunk: results 4 grp + i, row i16
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        if (own == s1) out[n] = acc[n];
        acc[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int n = 0; n < 4; ++n)
    *reinterpret_cast<f32x4 *>(&lds.out[i16][wave * 64 + 16 * n + 4 * grp]) = out[n];
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int row = 4 * wave + j, m = m0 + row;
    if (m >= g.M || c >= g.N) continue;
    float *y = g.y + (int64_t)m * g.ldy + c;
    const bool none = __builtin_amdgcn_readlane(own, row) < 0;
    if (none && g.base == g.y) continue;
    const f32x4 d = *reinterpret_cast<const f32x4 *>(&lds.out[row][lane * 4]);
    Run<float, 4> o;
#pragma unroll
    for (int i = 0; i < 4; ++i) o.v[i] = none ? old[j].v[i] : g.base ? old[j].v[i] + d[i] : d[i];
    if (c + 4 <= g.N) {
      *reinterpret_cast<Run<float, 4> *>(y) = o;
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (c + i < g.N) y[i] = o.v[i];
    }
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
  const int blocks = g.rank_pad / 16, per = std::min(blocks, sizeof(T) == 4 ? 2 : 4);   // (48 KB of LDS)
  // A tile's adapters side by side where there are few tiles, else in turn: a
  // prompt's tiles have one or two, and workgroups that find nothing to do
  // cost 10 us over 2048 rows with eight adapters.
  const unsigned tiles = (unsigned)((g.M + 15) / 16), shares = (unsigned)(blocks / per * g.splits);
  const unsigned kinds = (unsigned)std::min({16, g.M, g.count});
  const dim3 grid(tiles, shares, std::min(kinds, std::max(1u, 2u * kSplitCUs / (tiles * shares))));
  const int threads = kShrinkWaves * 64;
  if (per == 1) return launch_l(lora_shrink_kernel<T, 1>, grid, threads, stream, ev, nullptr, g);
  if constexpr (sizeof(T) == 2)
    if (per == 4) return launch_l(lora_shrink_kernel<T, 4>, grid, threads, stream, ev, nullptr, g);
  return launch_l(lora_shrink_kernel<T, 2>, grid, threads, stream, ev, nullptr, g);
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

// Through LDS where ranks fill a chunk and there are workgroups enough (each
// takes its tile's adapters one after the other).  us, a lane a row and through
// LDS, of bfloat16:
//   2048 x 4096 (2048 workgroups), 8 adapters, rank 32 17, 24, rank 64 24, 21, rank
//   128 33, 25; 512 x 4096 (512), 4 adapters, rank 64 7.1, 6.8
//   16 x 100000 (391), 2 adapters, rank 64 8.8, 7.8, rank 128 13.5, 12; 16 adapters
//   35, 33 and 89, 70; 64 x 32000 (500), 16 adapters, rank 83 110, 83
//   32 x 32000 (250), 8 adapters, rank 64 13.6, 15.4; 16 x 8000 (32), 16 adapters
//   8.9, 22.6
// of binary16 and binary32 at the same sizes (timed with events, which add some 2):
//   2048 x 4096: rank 32 22, 26 and 25, 22, rank 64 35, 27 and 39, 30, rank 128 50, 38
//   and 55, 42; 512 x 4096: 11.4, 10.1 and 12.6, 9.7
//   16 x 100000, 2 adapters: rank 64 15.1, 13.5 and 15.9, 14.5, rank 128 25, 20 and 32,
//   29; 16 adapters: 75, 69 and 82, 87, then 146, 124 and 157, 164; 64 x 32000: 139,
//   118 and 146, 147
//   32 x 32000: 24, 28 and 26, 33; 16 x 8000: 16, 45 and 19, 52
inline bool expand_wide(const LoraArgs &g) {
  return g.rank_pad >= 64 && (int64_t)((g.N + 255) / 256) * ((g.M + 15) / 16) >= 384;
}

template <typename T>
hipError_t expand(const LoraArgs &g, hipStream_t stream, hipEvent_t *ev, hipEvent_t done) {
  if (expand_wide(g))
    return launch_l(lora_expand_wide_kernel<T>, dim3((unsigned)((g.N + 255) / 256), (unsigned)((g.M + 15) / 16)),
                    256, stream, ev, done, g);
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

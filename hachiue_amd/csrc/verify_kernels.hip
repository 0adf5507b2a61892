// Verification of drafted tokens (speculative decoding) on gfx950.
//
// A sequence brings n drafted tokens x_0 .. x_(n-1), the target's
// distributions p_0 .. p_n (p_i after the first i drafts) and the
// distributions q_i that the drafts were drawn from (or none: q_i is 1 at
// x_i).  With uniforms u_0 .. u_n in [0, 1):
//   draft i is accepted iff u_i q_i(x_i) < p_i(x_i), in order up to the first
//   rejection a (a = n: none);
//   the final token is the first v whose running sum of r is above
//   u_n sum r, with r = max(p_a - q_a, 0) after a rejection (p_a where that
//   is 0 everywhere), r = p_n without one.
// The tokens are then distributed as draws from the target alone (Leviathan,
// Kalman and Matias 2023; Chen et al. 2023).
//
// Running sums over a vocabulary move by about 1e-7 of the total per id, so a
// draw needs them far more exactly than binary32 gives: weights, sums and
// comparisons are binary64.
#include "sampler_internal.h"

#include <hip/hip_ext.h>
#include <hip/hip_runtime.h>

#include <cfloat>

namespace hs {
namespace {

constexpr int kWavesV = kVerifyThreads / 64;

__device__ __forceinline__ void store_agent(double *p, double v) {
  __hip_atomic_store(reinterpret_cast<unsigned long long *>(p),
                     (unsigned long long)__double_as_longlong(v), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void store_agent(uint32_t *p, uint32_t v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ unsigned long long load_agent64(const void *p) {
  return __hip_atomic_load(static_cast<const unsigned long long *>(p), __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint32_t load_agent32(const uint32_t *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void store_part(VerifyPart *p, const VerifyPart &v) {
  store_agent(&p->s, v.s);
  const unsigned long long w =
      (unsigned long long)__float_as_uint(v.m) | ((unsigned long long)(uint32_t)v.arg << 32);
  __hip_atomic_store(reinterpret_cast<unsigned long long *>(&p->m), w, __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ VerifyPart load_part(const VerifyPart *p) {
  VerifyPart v;
  v.s = __longlong_as_double((long long)load_agent64(&p->s));
  const unsigned long long w = load_agent64(&p->m);
  v.m = __uint_as_float((uint32_t)w);
  v.arg = (int32_t)(w >> 32);
  return v;
}

// Counts the workgroup in, after its agent-scope stores have completed; true
// in the one that completes the count (it reads the others' stores with
// agent-scope loads).
__device__ __forceinline__ bool arrive(uint32_t *cnt, uint32_t of, int32_t *last) {
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  if (threadIdx.x == 0)
    *last = __hip_atomic_fetch_add(cnt, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == of - 1;
  __syncthreads();
  return *last != 0;
}

// 2^d for d <= 0 (NaN: 0), to 1e-15: n = round(d), 2^(d - n) by a polynomial
// 1 + f g(f), g the Chebyshev interpolant of (2^f - 1) / f of degree 9 on
// [-1/2, 1/2].  Exact at whole d.
__device__ __forceinline__ double exp2_neg(double d) {
  d = fmax(d, -1100.0);   // (below 2^-1074; a NaN takes the other operand)
  const double n = rint(d);
  const double f = d - n;
  double g = 0x1.e5e9f548e5726p-28;
  g = __builtin_fma(g, f, 0x1.b6571de2f2351p-24);
  g = __builtin_fma(g, f, 0x1.62bfe46117445p-20);
  g = __builtin_fma(g, f, 0x1.ffcb76789860fp-17);
  g = __builtin_fma(g, f, 0x1.4309130378460p-13);
  g = __builtin_fma(g, f, 0x1.5d87fe908f88ap-10);
  g = __builtin_fma(g, f, 0x1.3b2ab6fba385fp-7);
  g = __builtin_fma(g, f, 0x1.c6b08d7044119p-5);
  g = __builtin_fma(g, f, 0x1.ebfbdff82c590p-3);
  g = __builtin_fma(g, f, 0x1.62e42fefa39f7p-1);
  return __builtin_amdgcn_ldexp(__builtin_fma(g, f, 1.0), (int)n);
}

// log2(e) / T, at most 1e300 so that 0 times it stays 0.
__device__ __forceinline__ double log2_scale(double T) {
  return fmin(1.4426950408889634 / T, 1e300);
}
__device__ __forceinline__ bool greedy_temp(double T) { return !(T > 0.0); }

// exp((l - m) / T) of a logit under a maximum m (NaN where the row has no
// candidate, which makes every weight 0).  The maximum weighs 1, also where it
// is +infinity; a NaN or -infinity weighs 0.
__device__ __forceinline__ double weight(float l, float m, double c) {
  const double e = exp2_neg(((double)l - (double)m) * c);
  return l == m ? 1.0 : e;
}
__device__ __forceinline__ float max_or_nan(float m) {
  return m == -__builtin_inff() ? __builtin_nanf("") : m;
}
// A given probability; what is none counts as 0.
__device__ __forceinline__ double given(float p) { return p > 0.0f && p <= FLT_MAX ? (double)p : 0.0; }

__device__ __forceinline__ float wave_max(float x) {
  for (int d = 32; d; d >>= 1) x = fmaxf(x, __shfl_xor(x, d));
  return x;
}
__device__ __forceinline__ int wave_min(int x) {
  for (int d = 32; d; d >>= 1) x = min(x, __shfl_xor(x, d));
  return x;
}
__device__ __forceinline__ int wave_max(int x) {
  for (int d = 32; d; d >>= 1) x = max(x, __shfl_xor(x, d));
  return x;
}
__device__ __forceinline__ double wave_sum(double x) {
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  return x;
}
// Inclusive running sum over the wave's lanes.
__device__ __forceinline__ double wave_scan(double x) {
  const int lane = threadIdx.x & 63;
  for (int d = 1; d < 64; d <<= 1) {
    const double y = __shfl_up(x, d);
    if (lane >= d) x += y;
  }
  return x;
}

// A sequence's drafts: first index and count, kept inside the arrays whatever
// the offsets say.
struct Range {
  int64_t start;
  int n;
};
__device__ __forceinline__ Range drafts_of(const DraftArgs &d, int b) {
  if (!d.off) return {(int64_t)b * d.max_drafts, d.max_drafts};
  const int64_t a = min(max(d.off[b], (int64_t)0), d.n_drafts);
  const int64_t e = min(d.off[b + 1], d.n_drafts) - a;
  return {a, (int)min(max(e, (int64_t)0), (int64_t)d.max_drafts)};
}

// The tokens, count and acceptance probabilities of a sequence with `acc`
// accepted drafts, and the append to its history: one whole wave.  ratio: the
// position's, in lane position; final < 0 with acc < 0: nothing is known (the
// count is `none`).
__device__ void emit(const DraftArgs &d, int b, const Range &r, int acc, int final, float ratio,
                     int none) {
  const int lane = threadIdx.x & 63;
  int tok = -1;
  if (lane < acc) tok = d.drafts[r.start + lane];
  if (lane == acc) tok = final;
  int count = acc >= 0 ? acc + 1 : none;
  if (d.ring && acc >= 0) {
    // as a decode step: a stop id ends the sequence and does not join its history
    bool stop = false;
    for (int i = 0; i < d.nstop; ++i) stop |= d.stop[i] == tok;
    const unsigned long long hit = __ballot(stop && lane <= acc);
    const int append = hit ? __ffsll(hit) - 1 : count;
    if (hit) count = append + 1;
    if (lane >= count) tok = -1;
    const int64_t len = max(d.len[b], (int64_t)0);
    if (lane < append) d.ring[(int64_t)b * d.cap + (len + lane) % d.cap] = tok;
    if (lane == 0) {
      d.len[b] = len + append;
      if (hit) d.done[b] = 1;
    }
  }
  if (lane <= r.n) d.tokens[r.start + b + lane] = tok;
  if (lane == 0) d.counts[b] = count;
  if (d.accept && lane < r.n) d.accept[r.start + lane] = lane <= acc ? ratio : 0.0f;
}

// The first rejected of n positions (n: none), ok in lane position.
__device__ __forceinline__ int first_rejected(bool ok, int n) {
  const int lane = threadIdx.x & 63;
  const unsigned long long no = __ballot(lane < n && !ok);
  return no ? __ffsll(no) - 1 : n;
}

// Tests a draft whose probabilities are p and q.
__device__ __forceinline__ Verdict judge(double p, double q, double u) {
  Verdict v;
  v.ok = u * q < p;
  v.ratio = p >= q ? (p > 0.0 ? 1.0f : 0.0f) : (float)(p / q);
  return v;
}

// ---- whole rows

// Four consecutive values of a row from id i on; past the vocabulary: NaN,
// which weighs 0 in both kinds of row.  Rows need only their floats' own
// alignment.
struct __attribute__((packed, aligned(4))) Float4 {
  float v[4];
};
__device__ __forceinline__ Float4 load4(const float *row, int i, int vocab) {
  if (i + 4 <= vocab) return *reinterpret_cast<const Float4 *>(row + i);
  Float4 f;
#pragma unroll
  for (int e = 0; e < 4; ++e) f.v[e] = i + e < vocab ? row[i + e] : __builtin_nanf("");
  return f;
}
// The first id of a thread's j-th float4 of a chunk, a workgroup's width apart.
__device__ __forceinline__ int chunk_id(int chunk, int j) {
  return chunk * kVerifyChunk + (j * kVerifyThreads + (int)threadIdx.x) * 4;
}

struct VerifySmem {
  float fmax[kWavesV];
  int imin[kWavesV], imax[kWavesV];
  double sum[kWavesV];
  int32_t last;
  VerifyStat stat[2];
  int acc, chunk;
  double at;                 // the draw, within the chunk
};

// One side's distribution at a position: what a row's elements are turned
// into probabilities with.
struct Row {
  const float *p;
  int kind;
  bool greedy;
  float m;                   // (NaN: no candidate)
  double c, inv;             // log2(e) / T, 1 / sum of weights
  int arg;
};
__device__ __forceinline__ Row row_of(const VerifyArgs &a, int side, int b, int64_t row,
                                      const VerifyStat &st) {
  Row r;
  r.p = a.rows[side] + row * a.stride[side];
  r.kind = a.kind[side];
  const double T = a.temps[side] ? a.temps[side][b] : 1.0;
  r.greedy = r.kind == kDistLogits && greedy_temp(T);
  r.c = log2_scale(T);
  r.m = max_or_nan(st.m);
  r.inv = st.s > 0.0 ? 1.0 / st.s : 0.0;
  r.arg = st.arg;
  return r;
}
__device__ __forceinline__ double prob(const Row &r, float v, int id) {
  if (r.kind == kDistProbs) return given(v);
  if (r.greedy) return id == r.arg ? 1.0 : 0.0;
  return weight(v, r.m, r.c) * r.inv;
}
__device__ __forceinline__ double prob_at(const Row &r, int id, int vocab) {
  return id >= 0 && id < vocab ? prob(r, r.p[id], id) : 0.0;
}

__device__ Verdict judge_at(const VerifyArgs &a, int b, const Range &r, int i,
                            const VerifyStat &st, const VerifyStat &sq) {
  const int x = a.d.drafts[r.start + i];
  const double p = prob_at(row_of(a, 0, b, r.start + b + i, st), x, a.vocab);
  const double q = a.kind[1] == kDistNone ? 1.0 : prob_at(row_of(a, 1, b, r.start + i, sq), x, a.vocab);
  return judge(p, q, a.d.uniforms[r.start + b + i]);
}

// A row's summary from its chunks', by one wave.
__device__ VerifyStat combine(const VerifyPart *part, int chunks, double T) {
  const int lane = threadIdx.x & 63;
  const double c = log2_scale(T);
  const bool greedy = greedy_temp(T);
  VerifyStat r;
  float m = -__builtin_inff();
  for (int i = lane; i < chunks; i += 64) m = fmaxf(m, load_part(part + i).m);
  r.m = wave_max(m);
  const float mm = max_or_nan(r.m);
  double s = 0.0;
  int arg = 0x7FFFFFFF;
  for (int i = lane; i < chunks; i += 64) {
    const VerifyPart p = load_part(part + i);
    s += p.s * weight(p.m, mm, c);
    if (p.m == mm) arg = min(arg, p.arg);
  }
  r.s = greedy ? 1.0 : wave_sum(s);
  r.arg = greedy ? wave_min(arg) : -1;
  if (r.m == -__builtin_inff()) {
    r.s = 0.0;
    r.arg = -1;
  }
  return r;
}

// One workgroup per chunk of a row of logits: its maximum and the sum of its
// weights.  The rows of every sequence's first position come first in the
// grid, then the second's and so on; the workgroup that completes a position
// judges its draft, and a workgroup of a position behind a rejection found by
// then ends at once: nothing of its rows is asked for.  (Whether it is found
// in time changes what is read, never the outcome.)
__global__ __launch_bounds__(kVerifyThreads) void verify_stats_kernel(VerifyArgs a) {
  __shared__ VerifySmem sm;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const bool both = a.kind[0] == kDistLogits && a.kind[1] == kDistLogits;
  const int pos = both ? blockIdx.z >> 1 : blockIdx.z;
  const int side = both ? blockIdx.z & 1 : a.kind[0] != kDistLogits;
  const int b = blockIdx.y;
  const Range r = drafts_of(a.d, b);
  if (pos > r.n || (side == 1 && pos == r.n) || (a.d.done && a.d.done[b])) return;
  const uint32_t rej = load_agent32(a.rejected + b);
  if (rej && 64 - (int)rej < pos) return;
  const double T = a.temps[side] ? a.temps[side][b] : 1.0;
  const bool greedy = greedy_temp(T);
  const int64_t row = side ? r.start + pos : r.start + b + pos;
  const int chunk = blockIdx.x;
  const float *rowp = a.rows[side] + row * a.stride[side];
  Float4 v[kVerifyPer / 4];
#pragma unroll
  for (int j = 0; j < kVerifyPer / 4; ++j) v[j] = load4(rowp, chunk_id(chunk, j), a.vocab);
  float m = -__builtin_inff();
#pragma unroll
  for (int i = 0; i < kVerifyPer; ++i) m = fmaxf(m, v[i / 4].v[i % 4]);
  m = wave_max(m);
  if (lane == 0) sm.fmax[wave] = m;
  __syncthreads();
  m = sm.fmax[0];
#pragma unroll
  for (int w = 1; w < kWavesV; ++w) m = fmaxf(m, sm.fmax[w]);
  VerifyPart part;
  part.m = m;
  part.s = 0.0;
  part.arg = -1;
  const float mm = max_or_nan(m);
  if (greedy) {
    int arg = 0x7FFFFFFF;
#pragma unroll
    for (int i = 0; i < kVerifyPer; ++i)
      if (v[i / 4].v[i % 4] == mm) arg = min(arg, chunk_id(chunk, i / 4) + i % 4);
    arg = wave_min(arg);
    if (lane == 0) sm.imin[wave] = arg;
    __syncthreads();
    if (tid == 0)
      for (int w = 0; w < kWavesV; ++w) part.arg = w ? min(part.arg, sm.imin[w]) : sm.imin[0];
  } else {
    const double c = log2_scale(T);
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < kVerifyPer; ++i) s += weight(v[i / 4].v[i % 4], mm, c);
    s = wave_sum(s);
    if (lane == 0) sm.sum[wave] = s;
    __syncthreads();
    if (tid == 0)
      for (int w = 0; w < kWavesV; ++w) part.s += sm.sum[w];
  }
  if (tid == 0) store_part(a.part[side] + row * a.chunks + chunk, part);
  const bool two = both && pos < r.n;
  const int slot = b * (a.d.max_drafts + 1) + pos;
  if (!arrive(a.arrived + slot, (uint32_t)a.chunks * (two ? 2u : 1u), &sm.last)) return;
  // both rows of the position are done
  if (wave < 2) {
    const int64_t wr = wave ? r.start + pos : r.start + b + pos;
    if (a.kind[wave] == kDistLogits && (wave == 0 || pos < r.n)) {
      const VerifyStat st = combine(a.part[wave] + wr * a.chunks, a.chunks,
                                    a.temps[wave] ? a.temps[wave][b] : 1.0);
      if (lane == 0) {
        sm.stat[wave] = st;
        a.stat[wave][wr] = st;
      }
    }
  }
  __syncthreads();
  if (tid == 0 && pos < r.n) {
    const Verdict vd = judge_at(a, b, r, pos, sm.stat[0], sm.stat[1]);
    a.verdict[slot] = vd;
    if (!vd.ok) atomicMax(a.rejected + b, (uint32_t)(64 - pos));
  }
}

// What the final token is drawn from, per element of the row.
struct Final {
  Row p, q;
  bool residual;             // p - q, or p without x where there are no draft rows
  bool pair;                 // ... with draft rows
  int x;
};
__device__ __forceinline__ double final_weight(const Final &f, float vp, float vq, int id) {
  const double p = prob(f.p, vp, id);
  if (!f.residual) return p;
  if (!f.pair) return id == f.x ? 0.0 : p;
  return fmax(p - prob(f.q, vq, id), 0.0);
}

__device__ double chunk_mass(const VerifyArgs &a, const Final &f, int chunk, VerifySmem &sm) {
  const int tid = threadIdx.x;
  double s = 0.0;
#pragma unroll 1
  for (int j0 = 0; j0 < kVerifyPer / 4; j0 += 4) {
    Float4 vp[4], vq[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) vp[j] = load4(f.p.p, chunk_id(chunk, j0 + j), a.vocab);
    if (f.pair) {
#pragma unroll
      for (int j = 0; j < 4; ++j) vq[j] = load4(f.q.p, chunk_id(chunk, j0 + j), a.vocab);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i)
      s += final_weight(f, vp[i / 4].v[i % 4], f.pair ? vq[i / 4].v[i % 4] : 0.0f,
                        chunk_id(chunk, j0 + i / 4) + i % 4);
  }
  s = wave_sum(s);
  __syncthreads();
  if ((tid & 63) == 0) sm.sum[tid >> 6] = s;
  __syncthreads();
  s = 0.0;
  for (int w = 0; w < kWavesV; ++w) s += sm.sum[w];
  return s;
}

// The first id whose running sum is above u times the whole, from the chunks'
// masses; -1 where the whole is 0.  Every thread of the workgroup.
__device__ int draw_id(const VerifyArgs &a, const Final &f, const double *mass, double u,
                       VerifySmem &sm) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (wave == 0) {
    double total = 0.0;
    int live = -1;           // the last chunk with any mass
    for (int c0 = 0; c0 < a.chunks; c0 += 64) {
      const double v = c0 + lane < a.chunks
                           ? __longlong_as_double((long long)load_agent64(mass + c0 + lane)) : 0.0;
      live = max(live, v > 0.0 ? c0 + lane : -1);
      total += __shfl(wave_scan(v), 63);
    }
    live = wave_max(live);
    const double at = u * total;
    int chunk = live;
    double before = 0.0, within = __builtin_inf();   // (past the end: the last id with mass)
    for (int c0 = 0; c0 < a.chunks; c0 += 64) {
      const double v = c0 + lane < a.chunks
                           ? __longlong_as_double((long long)load_agent64(mass + c0 + lane)) : 0.0;
      const double s = wave_scan(v);
      const unsigned long long hit = __ballot(v > 0.0 && before + s > at);
      if (hit) {
        const int l = __ffsll(hit) - 1;
        chunk = c0 + l;
        const double up = __shfl(s, max(l - 1, 0));
        within = at - (before + (l ? up : 0.0));
        break;
      }
      before += __shfl(s, 63);
    }
    if (lane == 0) {
      sm.chunk = total > 0.0 ? chunk : -1;
      sm.at = within;
    }
  }
  __syncthreads();
  const int chunk = sm.chunk, base = chunk * kVerifyChunk;
  const double at = sm.at;
  __syncthreads();   // (both are written again below)
  if (chunk < 0) return -1;
  // kVerifyPer consecutive ids a thread: the thread that the draw falls to,
  // then its ids one a lane
  const int id0 = base + tid * kVerifyPer;
  double own = 0.0;
#pragma unroll 1
  for (int j0 = 0; j0 < kVerifyPer; j0 += 8) {
    Float4 vp[2], vq[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) vp[j] = load4(f.p.p, id0 + j0 + 4 * j, a.vocab);
    if (f.pair) {
#pragma unroll
      for (int j = 0; j < 2; ++j) vq[j] = load4(f.q.p, id0 + j0 + 4 * j, a.vocab);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      own += final_weight(f, vp[i / 4].v[i % 4], f.pair ? vq[i / 4].v[i % 4] : 0.0f, id0 + j0 + i);
  }
  const double incl = wave_scan(own);
  if (lane == 63) sm.sum[wave] = incl;
  __syncthreads();
  double start = 0.0;
  for (int i = 0; i < wave; ++i) start += sm.sum[i];
  const double up = __shfl_up(incl, 1);
  const double before = start + (lane ? up : 0.0);
  const unsigned long long hit = __ballot(own > 0.0 && start + incl > at);
  const unsigned long long any = __ballot(own > 0.0);
  if (lane == 0) {
    sm.imin[wave] = hit ? tid + __ffsll(hit) - 1 : kVerifyThreads;
    sm.imax[wave] = any ? tid + 63 - __clzll(any) : -1;
  }
  __syncthreads();
  int owner = kVerifyThreads, live = -1;
  for (int i = 0; i < kWavesV; ++i) {
    owner = min(owner, sm.imin[i]);
    live = max(live, sm.imax[i]);
  }
  const bool past = owner == kVerifyThreads;   // (rounding: the last id with mass)
  if (past) owner = live;
  if (tid == owner) sm.at = past ? __builtin_inf() : at - before;
  __syncthreads();
  if (wave == 0) {
    const int id = base + owner * kVerifyPer + lane;
    const bool in = lane < kVerifyPer && owner >= 0 && id < a.vocab;
    const double w = in ? final_weight(f, f.p.p[id], f.pair ? f.q.p[id] : 0.0f, id) : 0.0;
    const double s = wave_scan(w);
    const unsigned long long h = __ballot(w > 0.0 && s > sm.at), n = __ballot(w > 0.0);
    const int l = h ? __ffsll(h) - 1 : n ? 63 - __clzll(n) : -1;
    if (lane == 0) sm.chunk = l >= 0 ? base + owner * kVerifyPer + l : -1;
  }
  __syncthreads();
  return sm.chunk;
}

// One workgroup per chunk of a sequence's final row: the mass of what the
// final token is drawn from (taken from the first kernel where the chunk's sum
// is that already); the one that completes the row draws and writes the
// sequence's outcome.
__global__ __launch_bounds__(kVerifyThreads) void verify_resolve_kernel(VerifyArgs a) {
  __shared__ VerifySmem sm;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = blockIdx.y, chunk = blockIdx.x;
  const Range r = drafts_of(a.d, b);
  if (a.d.done && a.d.done[b]) {   // done before this call
    if (chunk == 0 && wave == 0) emit(a.d, b, r, -1, -1, 0.0f, 0);
    return;
  }
  const bool judged = a.kind[0] == kDistLogits || a.kind[1] == kDistLogits;
  const int slot = b * (a.d.max_drafts + 1);
  float ratio = 0.0f;
  if (wave == 0) {
    Verdict v = {0.0f, 0};
    if (lane < r.n) {
      const VerifyStat none = {};
      v = judged ? a.verdict[slot + lane] : judge_at(a, b, r, lane, none, none);
    }
    const int acc = first_rejected(v.ok != 0, r.n);
    ratio = v.ratio;
    if (lane == 0) sm.acc = acc;
  }
  __syncthreads();
  const int acc = sm.acc;
  const bool last_row = acc == r.n;
  const int64_t row = r.start + b + acc;
  const VerifyStat none = {};
  Final f;
  f.p = row_of(a, 0, b, row, a.kind[0] == kDistLogits ? a.stat[0][row] : none);
  f.residual = !last_row;
  f.pair = f.residual && a.kind[1] != kDistNone;
  f.x = f.residual ? a.d.drafts[r.start + acc] : -1;
  if (f.pair)
    f.q = row_of(a, 1, b, r.start + acc, a.kind[1] == kDistLogits ? a.stat[1][r.start + acc] : none);
  int token = 0;
  const bool logits = f.p.kind == kDistLogits;
  // greedy: its one id.  No candidate at all: 0, as the sampler's
  const bool known = logits && (f.p.greedy || !(f.p.inv > 0.0));
  if (known) {
    if (chunk != 0) return;
    token = max(f.p.arg, 0);
  } else {
    const VerifyPart *part = logits ? a.part[0] + row * a.chunks : nullptr;
    double *mass = a.mass + (int64_t)b * a.chunks;
    const double u = a.d.uniforms[r.start + b + r.n];
    // this chunk; then, where nothing is left beyond q (or x), all of p by the
    // workgroup that found it so
    int c0 = chunk, c1 = chunk + 1;
    for (int again = 0;; ++again) {
      for (int c = c0; c < c1; ++c) {
        double s;
        if (logits && !f.pair && !(f.residual && f.x >= 0 && f.x / kVerifyChunk == c)) {
          const VerifyPart p = load_part(part + c);
          s = p.s * weight(p.m, f.p.m, f.p.c) * f.p.inv;
        } else {
          s = chunk_mass(a, f, c, sm);
        }
        if (tid == 0) store_agent(mass + c, s);
      }
      if (!again) {
        if (!arrive(a.arrived_final + b, (uint32_t)a.chunks, &sm.last)) return;
      } else {
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
      }
      token = draw_id(a, f, mass, u, sm);
      if (token >= 0 || again) break;
      f.residual = f.pair = false;
      c0 = 0;
      c1 = a.chunks;
      __syncthreads();
    }
    token = max(token, 0);
  }
  if (wave == 0) emit(a.d, b, r, acc, token, ratio, 0);
  // zero for the next call
  if (judged)
    for (int i = tid; i <= a.d.max_drafts; i += kVerifyThreads) store_agent(a.arrived + slot + i, 0u);
  if (tid == 0) {
    store_agent(a.rejected + b, 0u);
    store_agent(a.arrived_final + b, 0u);
  }
}

// ---- candidate lists

// A list's share of a row: its length (-1: longer than was kept), and for a
// row without one (greedy, or no candidate) its one id.
struct List {
  const int32_t *ids;
  const float *probs;
  int kept;
  int only;
};
__device__ __forceinline__ List list_of(const ListArgs &a, int side, int64_t row) {
  List l;
  l.ids = a.ids[side] + row * a.stride[side];
  l.probs = a.probs[side] + row * a.stride[side];
  l.kept = a.kept[side][row];
  l.only = l.kept > 0 ? -1 : a.tokens[side] ? a.tokens[side][row] : 0;
  if (l.kept > a.stride[side] || (l.kept <= 0 && l.only < 0)) l.kept = -1;
  else l.kept = max(l.kept, 0);
  return l;
}

// (sum of the kept probabilities, that of id x), by one wave.
struct ListSum {
  double all, x;
};
__device__ __forceinline__ ListSum list_sum(const List &l, int x) {
  const int lane = threadIdx.x & 63;
  double s = 0.0, px = 0.0;
  for (int i = lane; i < l.kept; i += 64) {
    const double p = given(l.probs[i]);
    s += p;
    if (l.ids[i] == x) px += p;
  }
  return {wave_sum(s), wave_sum(px)};
}

struct ListSmem {
  Verdict verdict[kVerifyMaxDrafts + 1];
  int bad[kVerifyMaxDrafts + 1];
  double zt, zq;
  double sum[kWavesV];
  int imin[kWavesV], imax[kWavesV];
};

__device__ __forceinline__ uint32_t list_hash(int id, uint32_t mask) {
  return ((uint32_t)id * 2654435761u >> 7) & mask;
}

// One workgroup per sequence: a wave per position judges its draft, then all
// of them draw the final token from the target's list beyond the draft's, in
// the list's order.  The draft's list goes into an LDS hash table of ids.
__global__ __launch_bounds__(kVerifyThreads) void verify_lists_kernel(ListArgs a, int bits) {
  extern __shared__ uint32_t table[];   // [2^bits] ids, [2^bits] probabilities
  __shared__ ListSmem sm;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = blockIdx.x;
  const Range r = drafts_of(a.d, b);
  if (a.d.done && a.d.done[b]) {
    if (wave == 0) emit(a.d, b, r, -1, -1, 0.0f, 0);
    return;
  }
  for (int i = wave; i < r.n; i += kWavesV) {
    const int x = a.d.drafts[r.start + i];
    const List t = list_of(a, 0, r.start + b + i);
    const ListSum st = list_sum(t, x);
    const double p = t.kept > 0 ? (st.all > 0.0 ? st.x / st.all : 0.0) : (double)(x == t.only);
    double q = 1.0;
    bool bad = t.kept < 0;
    if (!a.certain) {
      const List d = list_of(a, 1, r.start + i);
      const ListSum sd = list_sum(d, x);
      q = d.kept > 0 ? (sd.all > 0.0 ? sd.x / sd.all : 0.0) : (double)(x == d.only);
      bad |= d.kept < 0;
    }
    if (lane == 0) {
      sm.verdict[i] = judge(p, q, a.d.uniforms[r.start + b + i]);
      sm.bad[i] = bad;
    }
  }
  __syncthreads();
  Verdict v = {0.0f, 0};
  bool bad = false;
  if (lane < r.n) {
    v = sm.verdict[lane];
    bad = sm.bad[lane] != 0;
  }
  const int acc = first_rejected(v.ok != 0, r.n);
  const bool residual = acc < r.n, pair = residual && !a.certain;
  const List t = list_of(a, 0, r.start + b + acc);
  // a list that was not kept whole, at a position that counts
  if (t.kept < 0 || __ballot(bad && lane <= acc)) {
    if (wave == 0) emit(a.d, b, r, -1, -1, 0.0f, -1);
    return;
  }
  const int x = residual ? a.d.drafts[r.start + acc] : -1;
  if (t.kept == 0) {   // one id has it all
    if (wave == 0) emit(a.d, b, r, acc, t.only, v.ratio, 0);
    return;
  }
  const uint32_t mask = (1u << bits) - 1u;
  uint32_t *hid = table;
  float *hp = reinterpret_cast<float *>(table + (mask + 1u));
  List q = {};
  if (pair) q = list_of(a, 1, r.start + acc);
  if (wave == 0) {
    const double s = list_sum(t, x).all;
    if (lane == 0) sm.zt = s;
  } else if (wave == 1 && pair) {
    const double s = list_sum(q, x).all;
    if (lane == 0) sm.zq = s;
  }
  if (pair) {
    for (uint32_t i = tid; i <= mask; i += kVerifyThreads) hid[i] = 0xFFFFFFFFu;
    __syncthreads();
    for (int i = tid; i < q.kept; i += kVerifyThreads) {
      const int id = q.ids[i];
      if (id < 0) continue;
      uint32_t h = list_hash(id, mask);
      // (at most half of the places are taken)
      while (true) {
        const uint32_t old = atomicCAS(hid + h, 0xFFFFFFFFu, (uint32_t)id);
        if (old == 0xFFFFFFFFu) {
          hp[h] = q.probs[i];
          break;
        }
        if (old == (uint32_t)id) break;
        h = (h + 1u) & mask;
      }
    }
  }
  __syncthreads();
  const double it = sm.zt > 0.0 ? 1.0 / sm.zt : 0.0;
  const double iq = pair && sm.zq > 0.0 ? 1.0 / sm.zq : 0.0;
  auto mass = [&](int i, bool rest) {
    const double p = given(t.probs[i]) * it;
    if (!rest) return p;
    const int id = t.ids[i];
    if (!pair) return id == x ? 0.0 : p;
    double qv = 0.0;
    if (q.kept == 0) {
      qv = id == q.only ? 1.0 : 0.0;
    } else if (id >= 0) {
      uint32_t h = list_hash(id, mask);
      while (hid[h] != 0xFFFFFFFFu && hid[h] != (uint32_t)id) h = (h + 1u) & mask;
      if (hid[h] == (uint32_t)id) qv = given(hp[h]) * iq;
    }
    return fmax(p - qv, 0.0);
  };
  const int per = (t.kept + kVerifyThreads - 1) / kVerifyThreads;
  const int i0 = min(tid * per, t.kept), i1 = min(i0 + per, t.kept);
  const double u = a.d.uniforms[r.start + b + r.n];
  int pick = -1;
  for (int rest = residual ? 1 : 0; rest >= 0 && pick < 0; --rest) {
    double own = 0.0;
    for (int i = i0; i < i1; ++i) own += mass(i, rest != 0);
    const double incl = wave_scan(own);
    __syncthreads();
    if (lane == 63) sm.sum[wave] = incl;
    __syncthreads();
    double before = 0.0, total = 0.0;
    for (int w = 0; w < kWavesV; ++w) {
      if (w < wave) before += sm.sum[w];
      total += sm.sum[w];
    }
    const double at = u * total;
    const double up = __shfl_up(incl, 1);
    double run = before + (lane ? up : 0.0);
    const double end = before + incl;
    int first = 0x7FFFFFFF, live = -1;
    for (int i = i0; i < i1; ++i) {
      const double m = mass(i, rest != 0);
      run += m;
      if (m > 0.0) {
        live = i;
        if (run > at && first == 0x7FFFFFFF) first = i;
      }
    }
    if (first == 0x7FFFFFFF && end > at && live >= 0) first = live;   // (rounding)
    first = wave_min(first);
    live = wave_max(live);
    if (lane == 0) {
      sm.imin[wave] = first;
      sm.imax[wave] = live;
    }
    __syncthreads();
    for (int w = 0; w < kWavesV; ++w) {
      first = min(first, sm.imin[w]);
      live = max(live, sm.imax[w]);
    }
    pick = first != 0x7FFFFFFF ? first : live;
  }
  if (wave == 0) emit(a.d, b, r, acc, pick >= 0 ? t.ids[pick] : t.ids[0], v.ratio, 0);
}

template <typename K, typename... A>
hipError_t launch_v(K kernel, dim3 grid, size_t lds, hipStream_t stream, hipEvent_t *ev,
                    hipEvent_t done, A... args) {
  const dim3 block(kVerifyThreads);
  if (ev)
    hipExtLaunchKernelGGL(kernel, grid, block, (std::uint32_t)lds, stream, ev[0], ev[1], 0u, args...);
  else if (done)
    hipExtLaunchKernelGGL(kernel, grid, block, (std::uint32_t)lds, stream, nullptr, done, 0u, args...);
  else
    hipLaunchKernelGGL(kernel, grid, block, lds, stream, args...);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_verify(const VerifyArgs &a, hipStream_t stream, hipEvent_t *ev_stats,
                         hipEvent_t *ev_resolve, hipEvent_t done) {
  const int sides = (a.kind[0] == kDistLogits) + (a.kind[1] == kDistLogits);
  if (sides > 0) {
    const dim3 grid((unsigned)a.chunks, (unsigned)a.d.seqs,
                    (unsigned)((a.d.max_drafts + 1) * (sides == 2 ? 2 : 1)));
    const hipError_t e = launch_v(verify_stats_kernel, grid, 0, stream, ev_stats, nullptr, a);
    if (e != hipSuccess) return e;
  }
  return launch_v(verify_resolve_kernel, dim3((unsigned)a.chunks, (unsigned)a.d.seqs), 0, stream,
                  ev_resolve, done, a);
}

// (the longest lists' table and the kernel's own LDS pass 64 KB)
hipError_t prepare_verify() {
  return hipFuncSetAttribute(reinterpret_cast<const void *>(verify_lists_kernel),
                             hipFuncAttributeMaxDynamicSharedMemorySize, 16 * kVerifyMaxList);
}

hipError_t launch_verify_lists(const ListArgs &a, hipStream_t stream, hipEvent_t *ev,
                               hipEvent_t done) {
  int bits = 0;
  if (!a.certain) {
    bits = 1;
    while ((1 << bits) < 2 * a.stride[1]) ++bits;
  }
  const size_t lds = a.certain ? 0 : (size_t)8 << bits;
  return launch_v(verify_lists_kernel, dim3((unsigned)a.d.seqs), lds, stream, ev, done, a, bits);
}

}  // namespace hs

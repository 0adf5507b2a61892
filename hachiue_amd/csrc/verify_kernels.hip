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

// 2^d for d <= 0 (NaN: 0), to 1.1 2^-53.  n = round(d), 2^(d - n) by a polynomial
// 1 + f g(f), g the Chebyshev interpolant of (2^f - 1) / f of degree 10 on
// [-1/2, 1/2] (2.0e-17 off; a degree less 5.7e-16).  Exact at whole d.
// Rounding, scaling and conversions take no longer than a multiplication here.
// Four at a time, step by step: a multiplication's result is ready after some
// three issue slots of a wave, and a wave alone on its SIMD would wait for each.
template <int N>
__device__ __forceinline__ void exp2_neg(double (&d)[N]) {
  constexpr double coef[11] = {0x1.e9d3fe3952179p-32, 0x1.e6063f7217bc6p-28, 0x1.b524fae627834p-24, 0x1.62bfd47773353p-20,
                               0x1.ffcbfc670dcd4p-17, 0x1.430913096fd9fp-13, 0x1.5d87fe78a5276p-10, 0x1.3b2ab6fba1ddap-7,
                               0x1.c6b08d704a0c2p-5,  0x1.ebfbdff82c598p-3,  0x1.62e42fefa39efp-1};
  double n[N], g[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    d[i] = fmax(d[i], -1100.0);   // (below 2^-1074; a NaN takes the other operand)
    n[i] = rint(d[i]);
    d[i] -= n[i];
    g[i] = coef[0];
  }
#pragma unroll
  for (int k = 1; k < 11; ++k)
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] = __builtin_fma(g[i], d[i], coef[k]);
#pragma unroll
  for (int i = 0; i < N; ++i)
    d[i] = __builtin_amdgcn_ldexp(__builtin_fma(g[i], d[i], 1.0), (int)n[i]);
}

// log2(e) / T, at most 1e300 so that 0 times it stays 0.
__device__ __forceinline__ double log2_scale(double T) {
  return fmin(1.4426950408889634 / T, 1e300);
}
__device__ __forceinline__ bool greedy_temp(double T) { return !(T > 0.0); }

// exp((l - m) / T) of logits under a maximum m (NaN where the row has no
// candidate, which makes every weight 0).  The maximum weighs 1, also where it
// is +infinity; a NaN or -infinity weighs 0.
template <int N>
__device__ __forceinline__ void weights_below(const float *l, float m, double c, double (&w)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = ((double)l[i] - (double)m) * c;   // (m finite or NaN)
  exp2_neg(w);
}
template <int N>
__device__ __forceinline__ void weights(const float *l, float m, double c, double (&w)[N]) {
  weights_below(l, m, c, w);
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = l[i] == m ? 1.0 : w[i];
}
__device__ __forceinline__ double weight(float l, float m, double c) {
  double w[1];
  weights(&l, m, c, w);
  return w[0];
}
__device__ __forceinline__ float max_or_nan(float m) {
  return m == -__builtin_inff() ? __builtin_nanf("") : m;
}
// A given probability; what is none counts as 0.
__device__ __forceinline__ double given(float p) { return p > 0.0f && p <= FLT_MAX ? (double)p : 0.0; }

// Reductions and running sums over a wave by data-parallel moves (no LDS):
// rows of 16 by shifts within the row, then the rows' last lanes broadcast.
template <int ctrl, int rows>
__device__ __forceinline__ double dpp0(double x) {   // (0 from no lane)
  const long long b = __double_as_longlong(x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, ctrl, rows, 0xF, rows == 0xF);
  const uint32_t hi =
      (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)((unsigned long long)b >> 32), ctrl, rows, 0xF, rows == 0xF);
  return __longlong_as_double((long long)((unsigned long long)hi << 32 | lo));
}
__device__ __forceinline__ double lane_of(double x, int lane) {   // (lane uniform)
  const long long b = __double_as_longlong(x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)((unsigned long long)b >> 32), lane);
  return __longlong_as_double((long long)((unsigned long long)hi << 32 | lo));
}
// Inclusive running sum over the wave's lanes.
__device__ __forceinline__ double wave_scan(double x) {
  x += dpp0<0x111, 0xF>(x);
  x += dpp0<0x112, 0xF>(x);
  x += dpp0<0x114, 0xF>(x);
  x += dpp0<0x118, 0xF>(x);
  x += dpp0<0x142, 0xA>(x);
  x += dpp0<0x143, 0xC>(x);
  return x;
}
__device__ __forceinline__ double wave_sum(double x) { return lane_of(wave_scan(x), 63); }
// The lane below's value (0 in lane 0).
__device__ __forceinline__ double lane_below(double x) { return dpp0<0x138, 0xF>(x); }
template <int ctrl, int rows>
__device__ __forceinline__ int dpp_own(int x) {      // (its own from no lane)
  return __builtin_amdgcn_update_dpp(x, x, ctrl, rows, 0xF, false);
}
template <typename F>
__device__ __forceinline__ int wave_fold(int x, F f) {
  x = f(x, dpp_own<0x111, 0xF>(x));
  x = f(x, dpp_own<0x112, 0xF>(x));
  x = f(x, dpp_own<0x114, 0xF>(x));
  x = f(x, dpp_own<0x118, 0xF>(x));
  x = f(x, dpp_own<0x142, 0xA>(x));
  x = f(x, dpp_own<0x143, 0xC>(x));
  return __builtin_amdgcn_readlane(x, 63);
}
__device__ __forceinline__ float wave_max(float x) {
  return __int_as_float(wave_fold(__float_as_int(x), [](int a, int b) {
    return __float_as_int(fmaxf(__int_as_float(a), __int_as_float(b)));
  }));
}
__device__ __forceinline__ int wave_min(int x) {
  return wave_fold(x, [](int a, int b) { return min(a, b); });
}
__device__ __forceinline__ int wave_max(int x) {
  return wave_fold(x, [](int a, int b) { return max(a, b); });
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
  v.p = p;
  v.ok = u * q < p;
  v.ratio = p >= q ? (p > 0.0 ? 1.0f : 0.0f) : (float)(p / q);
  return v;
}

// ---- whole rows

// Four consecutive values of a row.  Rows need only their floats' own
// alignment.
struct __attribute__((packed, aligned(4))) Float4 {
  float v[4];
};
// From id i on; past the vocabulary NaN, which weighs 0 in both kinds of row.
__device__ __forceinline__ Float4 load4(const float *row, int i, int vocab) {
  if (i + 4 <= vocab) return *reinterpret_cast<const Float4 *>(row + i);
  Float4 f;
#pragma unroll
  for (int e = 0; e < 4; ++e) f.v[e] = i + e < vocab ? row[i + e] : __builtin_nanf("");
  return f;
}
// A wave's part of a row: float4 j of lane l is ids 256 j + 4 l of the part.
// (One test per part, so that its loads are all on their way together.)
template <int PER>
__device__ __forceinline__ int part_id(int part, int j) {
  return part * (64 * PER) + j * 256 + (int)(threadIdx.x & 63) * 4;
}
template <int PER>
__device__ __forceinline__ void load_part_of(const float *row, int part, int vocab,
                                             Float4 (&v)[PER / 4]) {
  if ((part + 1) * (64 * PER) <= vocab) {
#pragma unroll
    for (int j = 0; j < PER / 4; ++j)
      v[j] = *reinterpret_cast<const Float4 *>(row + part_id<PER>(part, j));
  } else {
#pragma unroll
    for (int j = 0; j < PER / 4; ++j) v[j] = load4(row, part_id<PER>(part, j), vocab);
  }
}

struct VerifySmem {
  double sum[kWavesV];
  int imin[kWavesV], imax[kWavesV];
  int32_t last;
  VerifyStat stat[2];
  int acc, pick;
  double at;                 // the draw, within the part
};

// A sequence's temperatures, read once and first.
struct Temps {
  double t[2];
};
__device__ __forceinline__ Temps temps_of(const VerifyArgs &a, int b) {
  return {{a.temps[0] ? a.temps[0][b] : 1.0, a.temps[1] ? a.temps[1][b] : 1.0}};
}

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
__device__ __forceinline__ Row row_of(const VerifyArgs &a, int side, const Temps &temps, int64_t row,
                                      const VerifyStat &st) {
  Row r;
  r.p = a.rows[side] + row * a.stride[side];
  r.kind = a.kind[side];
  const double T = temps.t[side];
  r.greedy = r.kind == kDistLogits && greedy_temp(T);
  r.c = log2_scale(T);
  r.m = max_or_nan(st.m);
  r.inv = st.s > 0.0 ? 1.0 / st.s : 0.0;
  r.arg = st.arg;
  return r;
}
// Probabilities of four consecutive ids.
__device__ __forceinline__ void probs4(const Row &r, const Float4 &v, int id, double (&p)[4]) {
  if (r.kind == kDistProbs) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = given(v.v[i]);
  } else if (r.greedy) {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = id + i == r.arg ? 1.0 : 0.0;
  } else {
    weights(v.v, r.m, r.c, p);
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] *= r.inv;
  }
}
__device__ __forceinline__ double prob(const Row &r, float v, int id) {
  if (r.kind == kDistProbs) return given(v);
  if (r.greedy) return id == r.arg ? 1.0 : 0.0;
  return weight(v, r.m, r.c) * r.inv;
}

// A draft's test, with what does not wait for its rows' sums: its id, its
// uniform and the rows' values at its id.
struct Test {
  int x;
  double u;
  float v[2];
};
__device__ __forceinline__ Test test_of(const VerifyArgs &a, int b, const Range &r, int i) {
  Test t;
  t.x = a.d.drafts[r.start + i];
  t.u = a.d.uniforms[r.start + b + i];
  t.v[0] = t.v[1] = __builtin_nanf("");
  if (t.x >= 0 && t.x < a.vocab) {
    t.v[0] = a.rows[0][(r.start + b + i) * a.stride[0] + t.x];
    if (a.kind[1] != kDistNone) t.v[1] = a.rows[1][(r.start + i) * a.stride[1] + t.x];
  }
  return t;
}
__device__ __forceinline__ Verdict judge_at(const VerifyArgs &a, int b, const Temps &temps,
                                            const Range &r, int i, const Test &t, const VerifyStat &st,
                                            const VerifyStat &sq) {
  // (a NaN, as for an id outside the vocabulary, weighs 0, but an id of -1 is
  // also the maximum's where there is none)
  const bool in = t.x >= 0 && t.x < a.vocab;
  const double p = in ? prob(row_of(a, 0, temps, r.start + b + i, st), t.v[0], t.x) : 0.0;
  const double q = a.kind[1] == kDistNone ? 1.0
                   : in ? prob(row_of(a, 1, temps, r.start + i, sq), t.v[1], t.x) : 0.0;
  return judge(p, q, t.u);
}

// A row's summary from its parts', by one wave.
__device__ __forceinline__ VerifyStat combine(const VerifyPart *part, int parts, double T) {
  const int lane = threadIdx.x & 63;
  const double c = log2_scale(T);
  const bool greedy = greedy_temp(T);
  VerifyStat r;
  // (most rows have at most three parts a lane: those stay in registers)
  VerifyPart own[3];
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    own[i] = {0.0, -__builtin_inff(), 0x7FFFFFFF};
    if (lane + 64 * i < parts) own[i] = load_part(part + lane + 64 * i);
  }
  float m = fmaxf(fmaxf(own[0].m, own[1].m), own[2].m);
  for (int i = lane + 192; i < parts; i += 64) m = fmaxf(m, load_part(part + i).m);
  r.m = wave_max(m);
  const float mm = max_or_nan(r.m);
  double s = 0.0;
  int arg = 0x7FFFFFFF;
  auto add = [&](const VerifyPart &p) {
    s += p.s * weight(p.m, mm, c);
    if (p.m == mm) arg = min(arg, p.arg);
  };
  add(own[0]);
  add(own[1]);
  add(own[2]);
  for (int i = lane + 192; i < parts; i += 64) add(load_part(part + i));
  r.s = greedy ? 1.0 : wave_sum(s);
  r.arg = greedy ? wave_min(arg) : -1;
  if (r.m == -__builtin_inff()) {
    r.s = 0.0;
    r.arg = -1;
  }
  return r;
}

// What the final token is drawn from, per element of the row.
struct Final {
  Row p, q;
  bool residual;             // p - q, or p without x where there are no draft rows
  bool pair;                 // ... with draft rows
  int x;
};
__device__ __forceinline__ void final_weights(const Final &f, const Float4 &vp, const Float4 &vq,
                                              int id, double (&w)[4]) {
  probs4(f.p, vp, id, w);
  if (f.pair) {
    double q[4];
    probs4(f.q, vq, id, q);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = fmax(w[i] - q[i], 0.0);
  } else if (f.residual) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = id + i == f.x ? 0.0 : w[i];
  }
}

// The mass of a part, by one wave.
template <int PER>
__device__ __forceinline__ double part_mass(const VerifyArgs &a, const Final &f, int part) {
  Float4 vp[PER / 4], vq[PER / 4];
  load_part_of<PER>(f.p.p, part, a.vocab, vp);
  if (f.pair) load_part_of<PER>(f.q.p, part, a.vocab, vq);
  double s = 0.0;
#pragma unroll
  for (int j = 0; j < PER / 4; ++j) {
    double w[4];
    final_weights(f, vp[j], vq[j], part_id<PER>(part, j), w);
    s += (w[0] + w[1]) + (w[2] + w[3]);
  }
  return wave_sum(s);
}

// The running sums of a value per thread over the workgroup: this thread's
// (before it, and with it) and the whole.
struct Scan {
  double before, end, total;
};
__device__ __forceinline__ Scan block_scan(double own, VerifySmem &sm) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const double incl = wave_scan(own);
  __syncthreads();
  if (lane == 63) sm.sum[wave] = incl;
  __syncthreads();
  double start = 0.0, total = 0.0;
  for (int i = 0; i < kWavesV; ++i) {
    if (i < wave) start += sm.sum[i];
    total += sm.sum[i];
  }
  return {start + lane_below(incl), start + incl, total};
}
// The first thread with `hit`, else the last with `any`, else -1.
__device__ __forceinline__ int block_first(bool hit, bool any, bool *past, VerifySmem &sm) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const unsigned long long h = __ballot(hit), n = __ballot(any);
  if (lane == 0) {
    sm.imin[wave] = h ? wave * 64 + __ffsll(h) - 1 : kVerifyThreads;
    sm.imax[wave] = n ? wave * 64 + 63 - __clzll(n) : -1;
  }
  __syncthreads();
  int first = kVerifyThreads, live = -1;
  for (int i = 0; i < kWavesV; ++i) {
    first = min(first, sm.imin[i]);
    live = max(live, sm.imax[i]);
  }
  *past = first == kVerifyThreads;
  return *past ? live : first;
}

// The first id whose running sum is above u times the whole, from the parts'
// masses (mass(part)); -1 where the whole is 0.  Every thread of the workgroup:
// each takes consecutive parts, the one the draw falls to finds its part, then
// each takes consecutive ids of that part.
template <int PER, typename Mass>
__device__ __forceinline__ int draw_id(const VerifyArgs &a, const Final &f, int parts, double u,
                                       Mass mass, VerifySmem &sm) {
  constexpr int EACH = 64 * PER / kVerifyThreads;   // ids of a part a thread
  const int tid = threadIdx.x;
  const int per = (parts + kVerifyThreads - 1) / kVerifyThreads;
  const int c0 = min(tid * per, parts), c1 = min(c0 + per, parts);
  const double one = c0 < c1 ? mass(c0) : 0.0;
  double own = one;
  for (int c = c0 + 1; c < c1; ++c) own += mass(c);
  const Scan all = block_scan(own, sm);
  const double at = u * all.total;
  bool past;
  int who = block_first(own > 0.0 && all.end > at, own > 0.0, &past, sm);
  if (who < 0) return -1;
  if (tid == who) {
    double run = all.before, m = one;
    int c = c0, live = c0;
    double before = run;
    for (;; m = mass(c)) {
      if (m > 0.0) {
        live = c;
        before = run;
        if (!past && run + m > at) break;
      }
      run += m;
      if (++c >= c1) break;
    }
    sm.pick = live;
    // (past the end by rounding: the last id with mass)
    sm.at = past || c >= c1 ? __builtin_inf() : at - before;
  }
  __syncthreads();
  const int part = sm.pick;
  const double in = sm.at;
  const int id0 = part * (64 * PER) + tid * EACH;
  Float4 vp[EACH / 4], vq[EACH / 4];
#pragma unroll
  for (int j = 0; j < EACH / 4; ++j) {
    vp[j] = load4(f.p.p, id0 + 4 * j, a.vocab);
    if (f.pair) vq[j] = load4(f.q.p, id0 + 4 * j, a.vocab);
  }
  double w[EACH / 4][4];
  own = 0.0;
#pragma unroll
  for (int j = 0; j < EACH / 4; ++j) {
    final_weights(f, vp[j], vq[j], id0 + 4 * j, w[j]);
#pragma unroll
    for (int i = 0; i < 4; ++i) own += w[j][i];
  }
  const Scan ids = block_scan(own, sm);
  who = block_first(own > 0.0 && ids.end > in, own > 0.0, &past, sm);
  if (tid == who) {
    double run = ids.before;
    int first = -1, live = -1;
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      run += w[i / 4][i % 4];
      if (w[i / 4][i % 4] > 0.0) {
        live = id0 + i;
        if (first < 0 && run > in) first = live;
      }
    }
    sm.pick = !past && first >= 0 ? first : live;
  }
  __syncthreads();
  return who < 0 ? -1 : sm.pick;
}

// The token of a sequence whose final row's masses are the sums that the rows'
// workgroups published (no draft rows to take off), by a whole workgroup.  A
// rejected certain draft's own probability px is taken off its part's sum;
// where little of the sum is left, so that the difference would keep less
// than 42 of its bits, the part is summed again without it.  A part has mass
// where its largest logit's own probability is not 0 (nor, without x, a sum so
// small that its ids' may be): a draw that falls to a part finds an id in it.
template <int PER>
__device__ __forceinline__ int draw_from_parts(const VerifyArgs &a, Final f, int64_t row, double u,
                                               double px, VerifySmem &sm) {
  const VerifyPart *part = a.part[0] + row * a.parts;
  auto sum_of = [&](int c) {
    const VerifyPart p = load_part(part + c);
    const double w = weight(p.m, f.p.m, f.p.c) * f.p.inv;
    return w > 0.0 ? p.s * w : 0.0;
  };
  int xp = f.residual && f.x >= 0 && f.x < a.vocab ? f.x / (64 * PER) : -1;
  for (;;) {
    double without = 0.0;
    if (xp >= 0) {
      const double all = sum_of(xp);
      without = all - px;
      if (!(without >= fmax(all * 0x1p-10, 0x1p-1000))) without = part_mass<PER>(a, f, xp);   // (each wave the same)
    }
    const int id =
        draw_id<PER>(a, f, a.parts, u, [&](int c) { return c == xp ? without : sum_of(c); }, sm);
    if (id >= 0 || !f.residual) return max(id, 0);
    f.residual = false;   // all of p is x: from p itself
    xp = -1;
    __syncthreads();
  }
}

__device__ __forceinline__ void store_verdict(Verdict *p, const Verdict &v) {
  store_agent(&p->p, v.p);
  const unsigned long long w =
      (unsigned long long)__float_as_uint(v.ratio) | ((unsigned long long)(uint32_t)v.ok << 32);
  __hip_atomic_store(reinterpret_cast<unsigned long long *>(&p->ratio), w, __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ Verdict load_verdict(const Verdict *p) {
  Verdict v;
  v.p = __longlong_as_double((long long)load_agent64(&p->p));
  const unsigned long long w = load_agent64(&p->ratio);
  v.ratio = __uint_as_float((uint32_t)w);
  v.ok = (int32_t)(w >> 32);
  return v;
}

// A sequence's outcome as far as its rows of logits settle it: the first
// rejected position (or n) and what the final token is drawn from.  Lanes hold
// their position's verdict.
struct Outcome {
  int acc;
  float ratio;
  double px;                 // the rejected draft's probability
  Final f;
  bool known;                // one id has it all (greedy), or none has anything
};
__device__ __forceinline__ Outcome outcome_of(const VerifyArgs &a, int b, const Temps &temps,
                                              const Range &r) {
  const int lane = threadIdx.x & 63;
  Verdict v = {};
  VerifyStat st = {}, sq = {};
  int x = -1;
  if (lane < r.n) {
    v = load_verdict(a.verdict + b * (a.d.max_drafts + 1) + lane);
    x = a.d.drafts[r.start + lane];
    if (a.kind[1] == kDistLogits) sq = load_part(a.stat[1] + r.start + lane);
  }
  if (lane <= r.n && a.kind[0] == kDistLogits) st = load_part(a.stat[0] + r.start + b + lane);
  auto at = [](const VerifyStat &s, int l) {
    VerifyStat o;
    o.s = lane_of(s.s, l);
    o.m = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(s.m), l));
    o.arg = __builtin_amdgcn_readlane(s.arg, l);
    return o;
  };
  Outcome o;
  const int acc = __builtin_amdgcn_readfirstlane(first_rejected(v.ok != 0, r.n));
  o.acc = acc;
  o.ratio = v.ratio;
  o.px = lane_of(v.p, acc);
  o.f.p = row_of(a, 0, temps, r.start + b + acc, at(st, acc));
  o.f.residual = acc < r.n;
  o.f.pair = o.f.residual && a.kind[1] != kDistNone;
  o.f.x = __builtin_amdgcn_readlane(x, acc);   // (-1 behind the last draft)
  if (o.f.pair) o.f.q = row_of(a, 1, temps, r.start + acc, at(sq, acc));
  o.known = a.kind[0] == kDistLogits && (o.f.p.greedy || !(o.f.p.inv > 0.0));
  return o;
}

// `split` workgroups a row of logits, a wave for each part: its maximum and the
// sum of its weights.  The rows of every sequence's first position come first
// in the grid, then the second's and so on; the workgroup that completes a
// position judges its draft, and workgroups of positions behind a rejection
// ask for nothing more of their rows once it is found.  (Whether it is found
// in time changes what is read, never the outcome: a position behind a
// rejection does not count, whatever is made of it.)
// ALONE: no draft rows.  The workgroup that completes a sequence's last
// position then writes its outcome; otherwise verify_final_kernel does.
// Bound: memory and the binary64 units together (a weight is 17 binary64
// operations of 5.6 cycles a wave), at the small end the chain load -> sum ->
// count in -> join.  A logit is read once: the sums are under each part's own
// maximum and meet under the row's.  Over rows of 151936 logits: 64 sequences
// of 8 drafts with draft rows 99 us (366 MB of the rows' 661, 3.7 TB/s), 16 of 4
// 36 us (88 MB, 2.5 TB/s), one of 3 without draft rows, outcome and all, 12 us.
template <bool ALONE, int PER>
__global__ __launch_bounds__(kVerifyThreads, ALONE ? 3 : 4) void verify_stats_kernel(VerifyArgs a) {
  __shared__ VerifySmem sm;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const bool both = !ALONE && a.kind[0] == kDistLogits && a.kind[1] == kDistLogits;
  const int pos = both ? blockIdx.z >> 1 : blockIdx.z;
  const int side = both ? blockIdx.z & 1 : ALONE ? 0 : a.kind[0] != kDistLogits;
  const int b = blockIdx.y;
  const Temps temps = temps_of(a, b);
  int rej = 0;
  if (a.look && pos > 0) {
    // behind a rejection: nothing to do.  (Read once for the whole workgroup:
    // its waves must agree, and it may change between two reads.  Where all
    // workgroups start at once there is nothing to see yet.)
    if (tid == 0) sm.acc = (int)load_agent32(a.rejected + b);
    __syncthreads();
    rej = sm.acc;
    if (!ALONE && rej && 64 - rej < pos) return;
  }
  const Range r = drafts_of(a.d, b);
  if (pos + (side || (!ALONE && a.kind[0] != kDistLogits)) > r.n) return;
  if (a.d.done && a.d.done[b]) {   // done before this call
    if (ALONE && blockIdx.x == 0 && blockIdx.z == 0 && wave == 0) emit(a.d, b, r, -1, -1, 0.0f, 0);
    return;
  }
  const int slot = b * (a.d.max_drafts + 1) + pos;
  const int64_t row = side ? r.start + pos : r.start + b + pos;
  Test test = {};
  if (tid == 0 && pos < r.n) test = test_of(a, b, r, pos);
  {
    const double T = side ? temps.t[1] : temps.t[0];
    const double c = log2_scale(T);
    const bool greedy = greedy_temp(T);
    const float *rowp = a.rows[side] + row * a.stride[side];
    int part = (int)blockIdx.x * kWavesV + wave;
    // (the next part is on its way while one is summed: all waves start
    // together, and would otherwise all read, then all compute; from here on
    // each wave looks for a rejection for itself: there is no barrier in here)
    Float4 next[PER / 4];
    if (part < a.parts && (rej == 0 || 64 - rej >= pos)) load_part_of<PER>(rowp, part, a.vocab, next);
    for (; part < a.parts && (rej == 0 || 64 - rej >= pos); part += a.split * kWavesV) {
      Float4 v[PER / 4];
#pragma unroll
      for (int j = 0; j < PER / 4; ++j) v[j] = next[j];
      if (part + a.split * kWavesV < a.parts) {
        rej = (int)load_agent32(a.rejected + b);
        load_part_of<PER>(rowp, part + a.split * kWavesV, a.vocab, next);
      }
      // (a maximum passes a quiet NaN over, but makes a signalling one its result)
      float m = -__builtin_inff();
#pragma unroll
      for (int i = 0; i < PER; ++i) m = fmaxf(m, __builtin_canonicalizef(v[i / 4].v[i % 4]));
      VerifyPart out;
      out.m = wave_max(m);
      out.s = 0.0;
      out.arg = -1;
      const float mm = max_or_nan(out.m);
      if (greedy) {
        int arg = 0x7FFFFFFF;
#pragma unroll
        for (int i = 0; i < PER; ++i)
          if (v[i / 4].v[i % 4] == mm) arg = min(arg, part_id<PER>(part, i / 4) + i % 4);
        out.arg = wave_min(arg);
      } else {
        if (mm == __builtin_inff()) {
#pragma unroll
          for (int i = 0; i < PER; ++i) out.s += v[i / 4].v[i % 4] == mm ? 1.0 : 0.0;
        } else {
#pragma unroll
          for (int j = 0; j < PER / 4; ++j) {
            double w[4];
            weights_below(v[j].v, mm, c, w);
            out.s += (w[0] + w[1]) + (w[2] + w[3]);
          }
        }
        out.s = wave_sum(out.s);
      }
      if (lane == 0) store_part(a.part[side] + row * a.parts + part, out);
    }
  }
  const bool two = both && pos < r.n;
  if (!arrive(a.arrived + slot, (uint32_t)a.split * (two ? 2u : 1u), &sm.last)) return;
  // the position is done: its rows' summaries, its draft's test
  if (wave < 2) {
    const int64_t wr = wave ? r.start + pos : r.start + b + pos;
    if (a.kind[wave] == kDistLogits && (wave == 0 || pos < r.n)) {
      const VerifyStat st = combine(a.part[wave] + wr * a.parts, a.parts,
                                    wave ? temps.t[1] : temps.t[0]);
      if (lane == 0) {
        sm.stat[wave] = st;
        store_part(a.stat[wave] + wr, st);
      }
    }
  }
  __syncthreads();
  if (tid == 0 && pos < r.n) {
    const Verdict vd = judge_at(a, b, temps, r, pos, test, sm.stat[0], sm.stat[1]);
    store_verdict(a.verdict + slot, vd);
    if (!vd.ok) atomicMax(a.rejected + b, (uint32_t)(64 - pos));
  }
  if (!ALONE) return;
  if (tid == 0) store_agent(a.arrived + slot, 0u);   // for the next call
  if (!arrive(a.left + b, (uint32_t)(r.n + 1), &sm.last)) return;
  // the sequence is done
  if (tid == 0) {
    store_agent(a.rejected + b, 0u);
    store_agent(a.left + b, 0u);
  }
  const double u = a.d.uniforms[r.start + b + r.n];
  const Outcome o = outcome_of(a, b, temps, r);
  const int token = o.known ? max(o.f.p.arg, 0)
                            : draw_from_parts<PER>(a, o.f, r.start + b + o.acc, u, o.px, sm);
  if (wave == 0) emit(a.d, b, r, o.acc, token, o.ratio, 0);
}

// The outcome of every sequence that has draft rows, or probabilities for its
// target.  After a rejection one workgroup per four parts of the final row
// sums what the final token is drawn from, and the one that completes the
// row draws; without one, and logits for the target, the sums are there.
// PER: the rows' sums', FPER: its own.
// Bound: the final rows' second read, 69 MB for 64 sequences of 151936 logits
// in 32 us (2.1 TB/s; binary64 weights of two rows an id, and a draw behind the
// last part), 32 sequences of probabilities (39 MB) 14 us.  Two parts a wave in
// turn, with half the workgroups, took 5 % and 16 % longer.
template <int PER, int FPER>
__global__ __launch_bounds__(kVerifyThreads, 3) void verify_final_kernel(VerifyArgs a) {
  __shared__ VerifySmem sm;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int b = blockIdx.y;
  const Range r = drafts_of(a.d, b);
  const Temps temps = temps_of(a, b);
  const double u = a.d.uniforms[r.start + b + r.n];
  const bool first = blockIdx.x == 0;
  if (a.d.done && a.d.done[b]) {   // done before this call
    if (first && wave == 0) emit(a.d, b, r, -1, -1, 0.0f, 0);
    return;
  }
  Outcome o;
  if (a.kind[0] == kDistLogits || a.kind[1] == kDistLogits) {
    if (first) {   // zero for the next call
      for (int i = tid; i <= a.d.max_drafts; i += kVerifyThreads)
        a.arrived[(int64_t)b * (a.d.max_drafts + 1) + i] = 0u;
      if (tid == 0) a.rejected[b] = 0u;
    }
    o = outcome_of(a, b, temps, r);
  } else {
    const VerifyStat none = {};
    Verdict v = {};
    if (lane < r.n) v = judge_at(a, b, temps, r, lane, test_of(a, b, r, lane), none, none);
    o.acc = first_rejected(v.ok != 0, r.n);   // (each wave the same)
    o.ratio = v.ratio;
    o.px = 0.0;
    o.known = false;
    o.f.p = row_of(a, 0, temps, r.start + b + o.acc, none);
    o.f.residual = o.acc < r.n;
    o.f.pair = o.f.residual && a.kind[1] != kDistNone;
    o.f.x = o.f.residual ? a.d.drafts[r.start + o.acc] : -1;
    if (o.f.pair) o.f.q = row_of(a, 1, temps, r.start + o.acc, none);
  }
  Final &f = o.f;
  int token;
  if (o.known || (a.kind[0] == kDistLogits && !f.residual)) {
    if (!first) return;
    token = o.known ? max(f.p.arg, 0) : draw_from_parts<PER>(a, f, r.start + b + o.acc, u, 0.0, sm);
  } else {
    double *mass = a.mass + (int64_t)b * a.fparts;
    // this workgroup's parts; then, where nothing is left beyond q (or x), all
    // of p's by the workgroup that found it so
    int p0 = (int)blockIdx.x * kWavesV, p1 = min(p0 + kWavesV, a.fparts);
    for (int again = 0;; ++again) {
      for (int p = p0 + wave; p < p1; p += kWavesV) {
        const double s = part_mass<FPER>(a, f, p);
        if (lane == 0) store_agent(mass + p, s);
      }
      if (!again) {
        if (!arrive(a.left + b, (uint32_t)a.blocks, &sm.last)) return;
      } else {
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
      }
      token = draw_id<FPER>(a, f, a.fparts, u, [&](int c) {
        return __longlong_as_double((long long)load_agent64(mass + c));
      }, sm);
      if (token >= 0 || again) break;
      f.residual = f.pair = false;
      p0 = 0;
      p1 = a.fparts;
      __syncthreads();
    }
    if (tid == 0) store_agent(a.left + b, 0u);   // for the next call
  }
  if (wave == 0) emit(a.d, b, r, o.acc, max(token, 0), o.ratio, 0);
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
// the list's order.  The draft's list goes into an LDS hash table of ids: a
// look-up instead of a pass over it for each of the target's.  Bound: the chain
// of dependent steps in one workgroup (offsets, lists, verdicts, table, sums):
// 8 us for 256 sequences of 4 drafts over 20 candidates, 10.6 us for 32 over
// 1024, of which an empty launch is 5.
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
  Verdict v = {};
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
    double run = before + lane_below(incl);
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
                         hipEvent_t *ev_final, hipEvent_t done) {
  const unsigned launches = verify_launches(a);
  if (launches & 1u) {
    const bool both = a.kind[0] == kDistLogits && a.kind[1] == kDistLogits;
    const dim3 grid((unsigned)a.split, (unsigned)a.d.seqs,
                    (unsigned)(both ? 2 * a.d.max_drafts + 1 : a.d.max_drafts + 1));
    const bool few = a.per == kVerifyPerFew;
    hipError_t e;
    if (launches & 2u)
      e = few ? launch_v(verify_stats_kernel<false, kVerifyPerFew>, grid, 0, stream, ev_stats, nullptr, a)
              : launch_v(verify_stats_kernel<false, kVerifyPer>, grid, 0, stream, ev_stats, nullptr, a);
    else
      e = few ? launch_v(verify_stats_kernel<true, kVerifyPerFew>, grid, 0, stream, ev_stats, done, a)
              : launch_v(verify_stats_kernel<true, kVerifyPer>, grid, 0, stream, ev_stats, done, a);
    if (e != hipSuccess) return e;
  }
  if (!(launches & 2u)) return hipSuccess;
  const dim3 grid((unsigned)a.blocks, (unsigned)a.d.seqs);
  if (a.fper == kVerifyPer)   // (target logits: at least as many rows are summed as drawn from)
    return launch_v(verify_final_kernel<kVerifyPer, kVerifyPer>, grid, 0, stream, ev_final, done, a);
  return a.per == kVerifyPer
             ? launch_v(verify_final_kernel<kVerifyPer, kVerifyPerFew>, grid, 0, stream, ev_final, done, a)
             : launch_v(verify_final_kernel<kVerifyPerFew, kVerifyPerFew>, grid, 0, stream, ev_final, done, a);
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

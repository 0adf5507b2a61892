// The entry points of drafted tokens and adapters with the C ABI's host code
// under AddressSanitizer and UndefinedBehaviorSanitizer: argument checks (all
// that runs without a GPU), then small calls of every kind, sizes that make the
// workspaces grow, two streams, timed calls, captured ones and refusals in a
// capture.  Results are checked loosely (return codes, ranges); parity is the
// pytest suites' job.  Exit 0: no sanitizer report and no failed check.
#include <hip/hip_runtime_api.h>

#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <vector>

#include "hachiue_sampler.h"

namespace {

uint64_t g_rs = 0x9E3779B97F4A7C15ull;
uint64_t rnd() {
  g_rs ^= g_rs << 13;
  g_rs ^= g_rs >> 7;
  g_rs ^= g_rs << 17;
  return g_rs;
}
double unif() { return (double)(rnd() >> 11) * 0x1p-53; }

int g_fail = 0;
#define IS(x, want)                                                                  \
  do {                                                                               \
    const int rc_ = (x);                                                             \
    if (rc_ != (want)) {                                                             \
      fprintf(stderr, "line %d: %s -> %d (%s)\n", __LINE__, #x, rc_, hs_last_error()); \
      ++g_fail;                                                                      \
    }                                                                                \
  } while (0)
#define OK(x) IS(x, HS_OK)
#define EXPECT(c)                                                    \
  do {                                                               \
    if (!(c)) {                                                      \
      fprintf(stderr, "line %d: check failed: %s\n", __LINE__, #c); \
      ++g_fail;                                                      \
    }                                                                \
  } while (0)

// Device memory of one scope.
struct Arena {
  std::vector<void *> all;
  template <typename T>
  T *put(const std::vector<T> &h) {
    void *p = nullptr;
    if (hipMalloc(&p, sizeof(T) * (h.size() + 1)) != hipSuccess) abort();
    all.push_back(p);
    if (!h.empty() && hipMemcpy(p, h.data(), sizeof(T) * h.size(), hipMemcpyHostToDevice) != hipSuccess) abort();
    return static_cast<T *>(p);
  }
  ~Arena() {
    (void)hipDeviceSynchronize();
    for (void *p : all) (void)hipFree(p);
  }
};

template <typename T>
std::vector<T> host(const T *d, size_t n) {
  std::vector<T> h(n);
  if (hipMemcpy(h.data(), d, sizeof(T) * n, hipMemcpyDeviceToHost) != hipSuccess) abort();
  return h;
}

void host_only_checks() {
  // (addresses that no call gets to use)
  float *f = reinterpret_cast<float *>(4096);
  int32_t *i = reinterpret_cast<int32_t *>(4096);
  double *u = reinterpret_cast<double *>(4096);
  hs_distribution rows{HS_DIST_LOGITS, 100, f, nullptr};
  hs_candidates lists{8, i, f, i, nullptr};
  hs_draft_batch batch{2, 3, 6, nullptr, i, u, i, i, nullptr};
  IS(hs_verify_drafts_device(nullptr, &rows, nullptr, 100, &batch, nullptr, nullptr), HS_ERR_INVALID_ARGUMENT);
  IS(hs_verify_candidates_device(nullptr, &lists, &lists, &batch, nullptr, nullptr), HS_ERR_INVALID_ARGUMENT);
  for (int32_t seqs : {-1, 0, 65535, 65536, INT32_MAX})
    for (int32_t most : {-1, 0, 63, 64, INT32_MAX})
      for (int64_t n : {(int64_t)-1, (int64_t)0, (int64_t)65535 * 63, INT64_MAX}) {
        hs_draft_batch b{seqs, most, n, reinterpret_cast<int64_t *>(4096), i, u, i, i, f};
        const int a = hs_verify_drafts_device(nullptr, &rows, &rows, 100, &b, nullptr, nullptr);
        EXPECT(a != HS_OK || seqs == 0);
        EXPECT(hs_verify_candidates_device(nullptr, &lists, nullptr, &b, nullptr, nullptr) == a);
      }
  // the largest that the checks let through: sizes of the workspace in 64 bits
  hs_draft_batch most{65535, 63, (int64_t)65535 * 63, nullptr, i, u, i, i, f};
  rows.row_stride = INT64_MAX;
  IS(hs_verify_drafts_device(nullptr, &rows, &rows, 1 << 28, &most, nullptr, nullptr), HS_ERR_INVALID_ARGUMENT);
  hs_decode_state st{i, 127, reinterpret_cast<int64_t *>(4096), i, i, 3};
  IS(hs_verify_drafts_device(nullptr, &rows, nullptr, 100, &batch, &st, nullptr), HS_ERR_INVALID_ARGUMENT);
  for (int32_t m : {-1, 0, 1, 65535, 65536})
    for (int32_t rank : {0, 1, 256, 257})
      for (int32_t n : {-1, 0, 1, 1 << 30, INT32_MAX}) {
        hs_adapters ad{30, 3, rank, 64, n, f, f, nullptr, nullptr};
        const int a = hs_lora_device(nullptr, f, m, 64, &ad, i, nullptr, 0, f, (int64_t)1 << 40, nullptr);
        EXPECT(a != HS_OK || m == 0 || n == 0);
        hs_weights w{0, n, 64, 0, f, nullptr, nullptr};
        EXPECT(hs_gemv_lora_device(nullptr, f, m, 64, &w, &ad, i, f, (int64_t)1 << 40, nullptr) != HS_OK);
        EXPECT(hs_lm_head_lora_sample_device(nullptr, f, m, 64, &w, &ad, i, f, (int64_t)1 << 40, nullptr, nullptr,
                                             nullptr, u, i, nullptr) != HS_OK);
      }
}

// A ragged batch, its outputs and histories.
struct Batch {
  std::vector<int64_t> off{0};
  int64_t total = 0;
  hs_draft_batch b;
  hs_decode_state st;
  Batch(Arena &a, const std::vector<int> &lens, int vocab) {
    int most = 0;
    for (int n : lens) {
      off.push_back(total += n);
      if (n > most) most = n;
    }
    const size_t seqs = lens.size();
    std::vector<int32_t> ids((size_t)total);
    for (auto &x : ids) x = (int32_t)(rnd() % (uint64_t)vocab);
    std::vector<double> us((size_t)total + seqs);
    for (auto &x : us) x = unif();
    b = {(int32_t)seqs, most, total, a.put(off), a.put(ids), a.put(us),
         a.put(std::vector<int32_t>((size_t)total + seqs)), a.put(std::vector<int32_t>(seqs, -7)),
         a.put(std::vector<float>((size_t)total))};
    st = {a.put(std::vector<int32_t>(seqs * 128)), 128, a.put(std::vector<int64_t>(seqs, 5)),
          a.put(std::vector<int32_t>(seqs)), a.put(std::vector<int32_t>{1, 2, 3}), 3};
  }
  void check(int vocab) {
    (void)hipDeviceSynchronize();
    const auto counts = host(b.counts, (size_t)b.seqs);
    const auto tokens = host(b.tokens, (size_t)(total + b.seqs));
    for (int s = 0; s < b.seqs; ++s) {
      EXPECT(counts[s] >= 0 && counts[s] <= off[s + 1] - off[s] + 1);
      for (int i = 0; i < counts[s]; ++i) EXPECT(tokens[off[s] + s + i] >= 0 && tokens[off[s] + s + i] < vocab);
    }
  }
};

void verification(hs_context *ctx, hipStream_t st, const std::vector<int> &lens, int vocab) {
  Arena a;
  Batch b(a, lens, vocab);
  const size_t seqs = lens.size(), rows = (size_t)b.total + seqs;
  std::vector<float> x(rows * (size_t)vocab), p(rows * (size_t)vocab);
  for (auto &v : x) v = (float)(unif() * 8 - 4);
  for (auto &v : p) v = (float)unif() / (float)vocab;
  const float *dx = a.put(x), *dp = a.put(p);
  const double *temps = a.put(std::vector<double>(seqs, 0.8));
  hs_distribution side[2] = {{HS_DIST_LOGITS, vocab, dx, temps}, {HS_DIST_PROBS, vocab, dp, nullptr}};
  for (const hs_distribution &t : side)
    for (int d = 0; d < 3; ++d)
      for (int state = 0; state < 2; ++state) {
        OK(hs_verify_drafts_device(ctx, &t, d < 2 ? &side[d] : nullptr, vocab, &b.b, state ? &b.st : nullptr, st));
        b.check(vocab);
      }
  // candidate lists of 16
  std::vector<int32_t> ids(rows * 16), kept(rows);
  for (size_t i = 0; i < ids.size(); ++i) ids[i] = (int32_t)((i % 16 * 7 + i / 16) % (size_t)vocab);
  for (size_t r = 0; r < rows; ++r) kept[r] = (int32_t)(1 + r % 16);
  hs_candidates l{16, a.put(ids), dp, a.put(kept), a.put(std::vector<int32_t>(rows, 4))};
  for (int d = 0; d < 2; ++d) {
    OK(hs_verify_candidates_device(ctx, &l, d ? &l : nullptr, &b.b, d ? &b.st : nullptr, st));
    b.check(vocab);
  }
}

void adapters(hs_context *ctx, hipStream_t st, int M, int K, int N, int rank, bool captured) {
  Arena a;
  const int count = 3;
  std::vector<float> x((size_t)M * K), w((size_t)N * K);
  for (auto &v : x) v = (float)unif() - 0.5f;
  for (auto &v : w) v = (float)unif() - 0.5f;
  std::vector<int32_t> slots(M);
  for (auto &s : slots) s = (int32_t)(rnd() % 5) - 1;
  const float *dx = a.put(x);
  const int32_t *ds = a.put(slots);
  float *y = a.put(std::vector<float>((size_t)M * N)), *base = a.put(std::vector<float>((size_t)M * N, 1.0f));
  const void *A = a.put(std::vector<uint32_t>((size_t)count * rank * K, 0x3c003c00u));
  const void *B = a.put(std::vector<uint32_t>((size_t)count * N * rank, 0x3c003c00u));
  hs_weights wt{0, N, K, 0, a.put(w), nullptr, nullptr};
  std::vector<hs_sample_config> cs((size_t)M);
  for (auto &c : cs) hs_config_default(&c);
  const double *us = a.put(std::vector<double>((size_t)M, 0.4));
  int32_t *tok = a.put(std::vector<int32_t>((size_t)M, -7));
  for (int32_t type : {0, 1, 30}) {
    hs_adapters ad{type, count, rank, K, N, A, B, a.put(std::vector<float>(count, 0.5f)),
                   a.put(std::vector<int32_t>{rank, 1, 0})};
    auto calls = [&](int want) {
      IS(hs_lora_device(ctx, dx, M, K, &ad, ds, base, N, y, N, st), want);
      IS(hs_lora_device(ctx, dx, M, K, &ad, ds, y, N, y, N, st), want);
      IS(hs_lora_device(ctx, dx, M, K, &ad, ds, nullptr, 0, y, N, st), want);
      IS(hs_gemv_lora_device(ctx, dx, M, K, &wt, &ad, ds, y, N, st), want);
    };
    if (captured) {
      hipGraph_t g = nullptr;
      if (hipStreamBeginCapture(st, hipStreamCaptureModeGlobal) != hipSuccess) abort();
      calls(HS_OK);
      IS(hs_lm_head_lora_sample_device(ctx, dx, M, K, &wt, &ad, ds, y, N, nullptr, nullptr, cs.data(), us, tok, st),
         HS_ERR_UNSUPPORTED);
      hs_adapters large = ad;   // (needs more workspace than there is: a capture allocates nothing)
      large.rank = 256;
      IS(hs_lora_device(ctx, dx, 65535, K, &large, ds, nullptr, 0, y, N, st), HS_ERR_UNSUPPORTED);
      if (hipStreamEndCapture(st, &g) != hipSuccess) abort();
      hipGraphExec_t ex = nullptr;
      if (hipGraphInstantiate(&ex, g, nullptr, nullptr, 0) != hipSuccess) abort();
      for (int i = 0; i < 2; ++i) {
        EXPECT(hipGraphLaunch(ex, st) == hipSuccess);
        EXPECT(hipStreamSynchronize(st) == hipSuccess);
      }
      (void)hipGraphExecDestroy(ex);
      (void)hipGraphDestroy(g);
      continue;
    }
    calls(HS_OK);
    OK(hs_lm_head_lora_sample_device(ctx, dx, M, K, &wt, &ad, ds, y, N, nullptr, nullptr, cs.data(), us, tok, st));
    (void)hipDeviceSynchronize();
    for (int32_t t : host(tok, (size_t)M)) EXPECT(t >= 0 && t < N);
    hs_adapters none = ad;
    none.count = 0;
    none.a = none.b = nullptr;
    OK(hs_lora_device(ctx, dx, M, K, &none, ds, base, N, y, N, st));
  }
}

}  // namespace

int main() {
  host_only_checks();
  hs_context *ctx = nullptr;
  if (hs_context_create(0, &ctx) != HS_OK) {
    printf("no GPU (%s): host-side checks only, %d failed\n", hs_last_error(), g_fail);
    return g_fail ? 1 : 0;
  }
  hipStream_t st = nullptr;
  if (hipStreamCreate(&st) != hipSuccess) abort();
  for (int timed = 0; timed < 2; ++timed) {
    OK(hs_context_set_timing(ctx, timed));
    printf("drafted tokens, timed %d\n", timed);
    fflush(stdout);
    verification(ctx, st, {3, 0, 5, 1}, 3001);
    verification(ctx, nullptr, {0, 0}, 50);
    verification(ctx, st, std::vector<int>(300, 9), 40);   // (the counters grow)
    printf("adapters, timed %d\n", timed);
    fflush(stdout);
    adapters(ctx, st, 5, 128, 700, 9, false);
    adapters(ctx, nullptr, 40, 64, 300, 130, false);
    adapters(ctx, st, 6000, 64, 32, 200, false);           // (their workspace grows)
  }
  double ms[17];
  int64_t calls = 0;
  OK(hs_context_kernel_times(ctx, ms, 17, &calls));
  EXPECT(calls > 0 && ms[12] > 0 && ms[13] > 0 && ms[14] > 0 && ms[15] > 0 && ms[16] > 0);
  OK(hs_context_set_timing(ctx, 0));
  OK(hs_context_destroy(ctx));
  OK(hs_context_create(0, &ctx));
  printf("captured adapters\n");
  fflush(stdout);
  adapters(ctx, st, 5, 128, 700, 9, true);
  OK(hs_context_destroy(ctx));
  (void)hipStreamDestroy(st);
  if (g_fail) {
    fprintf(stderr, "%d checks failed\n", g_fail);
    return 1;
  }
  printf("serving sanitizer run: ok\n");
  return 0;
}

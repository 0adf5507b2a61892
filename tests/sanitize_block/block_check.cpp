// The entry points of norms between blocks and 8-bit products with the C ABI's host
// code under AddressSanitizer and UndefinedBehaviorSanitizer: argument checks (all
// that runs without a GPU), then small calls of every kind, sizes that make the
// workspaces grow, two streams, timed calls, captured ones and refusals in a
// capture.  Results are checked loosely (return codes, ranges); parity is the
// pytest suites' job.  Exit 0: no sanitizer report and no failed check.
#include <hip/hip_runtime_api.h>

#include <math.h>
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>

#include <vector>

#include "hachiue_sampler.h"

namespace {

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

constexpr int32_t kF32 = 0, kF16 = 1, kI8 = 24, kBF16 = 30;

// Device memory of one scope.
struct Arena {
  std::vector<void *> all;
  template <typename T>
  T *get(size_t n) {
    void *p = nullptr;
    if (hipMalloc(&p, sizeof(T) * (n + 1)) != hipSuccess || hipMemset(p, 1, sizeof(T) * (n + 1)) != hipSuccess) abort();
    all.push_back(p);
    return static_cast<T *>(p);
  }
  ~Arena() {
    (void)hipDeviceSynchronize();
    for (void *p : all) (void)hipFree(p);
  }
};

void host_only_checks() {
  // (addresses that no call gets to use)
  auto at = [](uintptr_t a) { return reinterpret_cast<void *>(a << 40); };
  float *f = reinterpret_cast<float *>((uintptr_t)9 << 40);
  for (int32_t m : {-1, 0, 1, 7, 1 << 24, INT32_MAX})
    for (int32_t c : {-1, 0, 1, 32768, 32769, INT32_MAX})
      for (int64_t ld : {INT64_MIN, (int64_t)0, (int64_t)32768, (int64_t)1 << 36, INT64_MAX})
        for (int32_t type : {-1, kF32, kF16, kI8, kBF16, INT32_MAX}) {
          hs_block_norm n{};
          n.rows = m;
          n.cols = c;
          n.x = {kF32, (int64_t)1 << 36, at(1), nullptr};
          n.gate = {type, ld, at(2), nullptr};
          n.gate_act = type;
          n.scale = NAN;
          n.residual = {type, ld, at(3), nullptr};
          n.sum = {type, ld, at(4), nullptr};
          n.out = {type, ld, at(5), type == kI8 ? f : nullptr};
          n.after = {type, (float)ld, f, f};
          n.before = {m, 0.0f, f, f};
          EXPECT(hs_block_norm_device(nullptr, &n, nullptr) != HS_OK);
          n.gate.data = n.residual.data = n.sum.data = nullptr;
          n.after.kind = HS_NORM_NONE;
          EXPECT(hs_block_norm_device(nullptr, &n, nullptr) != HS_OK);
          for (int32_t k : {-16, 0, 16, 40, 65536, INT32_MAX}) {
            hs_weights w{kI8, c, k, 0, at(6), at(7), nullptr};
            hs_rows x{type, ld, at(8), type == kI8 ? f : nullptr}, y = n.out;
            EXPECT(hs_matmul_int_device(nullptr, m, &x, &w, f, &y, nullptr) != HS_OK);
            EXPECT(hs_gated_int_device(nullptr, m, &x, &w, &w, type, &y, nullptr) != HS_OK);
            n.cols = k;
            EXPECT(hs_lm_head_norm_sample_device(nullptr, &n, &w, f, ld, nullptr, nullptr, nullptr, nullptr, nullptr,
                                                 nullptr) != HS_OK);
            n.cols = c;
          }
        }
  // the largest that the checks let through
  hs_weights w{kI8, 1 << 16, 65536, 0, at(6), at(700), nullptr};
  hs_rows x{kI8, 1 << 23, at(800), f}, y{kF32, (int64_t)1 << 36, at(100000), nullptr};
  IS(hs_matmul_int_device(nullptr, 1 << 20, &x, &w, nullptr, &y, nullptr), HS_ERR_INVALID_ARGUMENT);   // (no context)
}

// Every kind of call over M rows: C columns, N channels.
void block(hs_context *ctx, hipStream_t st, int32_t M, int32_t C, int32_t N, bool captured, int want) {
  Arena a;
  float *x = a.get<float>((size_t)M * C), *r = a.get<float>((size_t)M * C), *y = a.get<float>((size_t)M * C);
  uint16_t *out = a.get<uint16_t>((size_t)M * C);
  int8_t *q = a.get<int8_t>((size_t)M * C), *h = a.get<int8_t>((size_t)M * N);
  float *qs = a.get<float>(M), *hsc = a.get<float>(M), *logits = a.get<float>((size_t)M * N);
  int8_t *w0 = a.get<int8_t>((size_t)N * C), *w1 = a.get<int8_t>((size_t)N * C), *w2 = a.get<int8_t>((size_t)N * C);
  float *s0 = a.get<float>(N), *s1 = a.get<float>(N), *s2 = a.get<float>(C), *p = a.get<float>(C);
  hs_weights gate{kI8, N, C, 0, w0, s0, nullptr}, up{kI8, N, C, 0, w1, s1, nullptr}, down{kI8, C, N, 0, w2, s2, nullptr};
  hs_rows xr{kF32, C, x, nullptr}, qr{kI8, C, q, qs}, hr{kI8, N, h, hsc}, yr{kF32, C, y, nullptr};
  hs_rows lr{kF32, N, logits, nullptr};
  hs_block_norm first{}, last{};
  first.rows = last.rows = M;
  first.cols = last.cols = C;
  first.x = xr;
  first.scale = last.scale = 1.0f;
  first.residual = first.sum = {kF32, C, r, nullptr};
  first.before = {HS_NORM_RMS, 1e-6f, p, nullptr};
  first.out = qr;
  last.x = yr;
  last.after = {HS_NORM_LAYER, 1e-5f, p, p};
  last.gate = {kF32, 0, p, nullptr};
  last.gate_act = HS_ACT_SIGMOID;
  last.out = {kBF16, C, out, nullptr};
  hipGraph_t graph = nullptr;
  hipGraphExec_t ex = nullptr;
  if (captured && hipStreamBeginCapture(st, hipStreamCaptureModeRelaxed) != hipSuccess) abort();
  OK(hs_block_norm_device(ctx, &first, st));
  IS(hs_gated_int_device(ctx, M, &qr, &gate, &up, HS_ACT_GELU, &hr, st), want);   // (results in 8 bits: the workspace)
  OK(hs_matmul_int_device(ctx, M, &hr, &down, p, &yr, st));
  OK(hs_block_norm_device(ctx, &last, st));
  IS(hs_matmul_int_device(ctx, M, &xr, &gate, nullptr, &lr, st), want);           // (float rows too)
  IS(hs_gemv_device_ex(ctx, x, M, C, &gate, logits, N, st), want);
  if (captured) {
    hs_sample_config cfg;
    hs_config_default(&cfg);
    std::vector<hs_sample_config> cs((size_t)M, cfg);
    IS(hs_lm_head_norm_sample_device(ctx, &first, &gate, logits, N, nullptr, nullptr, cs.data(),
                                     reinterpret_cast<double *>(x), reinterpret_cast<int32_t *>(qs), st),
       HS_ERR_UNSUPPORTED);
    if (hipStreamEndCapture(st, &graph) != hipSuccess) abort();
    if (hipGraphInstantiate(&ex, graph, nullptr, nullptr, 0) != hipSuccess) abort();
    for (int i = 0; i < 2; ++i)
      if (hipGraphLaunch(ex, st) != hipSuccess || hipStreamSynchronize(st) != hipSuccess) abort();
    (void)hipGraphExecDestroy(ex);
    (void)hipGraphDestroy(graph);
    return;
  }
  double *u = a.get<double>(M);
  int32_t *tok = a.get<int32_t>(M);
  if (hipMemset(u, 0, sizeof(double) * M) != hipSuccess) abort();
  hs_sample_config cfg;
  hs_config_default(&cfg);
  cfg.temperature = 0.0;
  std::vector<hs_sample_config> cs((size_t)M, cfg);
  OK(hs_lm_head_norm_sample_device(ctx, &first, &gate, logits, N, nullptr, nullptr, cs.data(), u, tok, st));
  OK(hs_lm_head_sample_device_ex(ctx, x, M, C, &gate, logits, N, nullptr, nullptr, cs.data(), u, tok, st));
  if (hipDeviceSynchronize() != hipSuccess) abort();
  std::vector<int32_t> t((size_t)M);
  if (hipMemcpy(t.data(), tok, sizeof(int32_t) * M, hipMemcpyDeviceToHost) != hipSuccess) abort();
  for (int32_t v : t) EXPECT(v >= 0 && v < N);
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
    for (int32_t m : {1, 2, 16, 33, 100, 700}) {
      printf("blocks of %d rows, timed %d\n", m, timed);
      fflush(stdout);
      block(ctx, m % 2 ? st : nullptr, m, 128, 272, false, HS_OK);
    }
    block(ctx, st, 9000, 128, 272, false, HS_OK);   // (the workspaces grow)
  }
  double ms[20];
  int64_t calls = 0;
  OK(hs_context_kernel_times(ctx, ms, 20, &calls));
  EXPECT(calls > 0 && ms[17] > 0 && ms[18] > 0 && ms[19] > 0);
  OK(hs_context_set_timing(ctx, 0));
  OK(hs_context_destroy(ctx));
  OK(hs_context_create(0, &ctx));
  printf("captured blocks\n");
  fflush(stdout);
  block(ctx, st, 5, 128, 272, true, HS_OK);
  block(ctx, st, 21000, 128, 272, true, HS_ERR_UNSUPPORTED);   // (more workspace than the context has)
  block(ctx, st, 21000, 128, 272, false, HS_OK);
  block(ctx, st, 21000, 128, 272, true, HS_OK);
  OK(hs_context_destroy(ctx));
  (void)hipStreamDestroy(st);
  if (g_fail) {
    fprintf(stderr, "%d checks failed\n", g_fail);
    return 1;
  }
  printf("block sanitizer run: ok\n");
  fflush(stdout);
  // (what the HIP runtime keeps of graphs it frees behind the end of the sanitizer's
  // device allocator, which reports that)
  _Exit(0);
}

// abi_asan.cpp — AddressSanitizer driver for the HOST side of libecnf_hip.so.  Built by tools/asan/build.sh against an
// ASan-instrumented build of the host translation units (the host code of ecnf_hip.hip, ecnf_train.hip and
// ecnf_context.hip; with ECNF_HOST_HOOKS); device code is not instrumented.
//
// Without a GPU it exercises every host path that runs before the first device call: argument checks, the
// ravel_pytree param walk and the split / fragment repacking of ecnf_create (which then fails with ECNF_E_HIP).
// With a GPU it also runs each C-ABI entry point once on a small batch and the error paths that follow a valid
// handle.  Exit status 0 = every check passed and ASan reported nothing (ASan aborts the process otherwise).
#include <hip/hip_runtime.h>
#include <sanitizer/lsan_interface.h>

#include <chrono>

#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <random>
#include <vector>

#include "ecnf.h"

static int g_fail = 0;
// ABI_ASAN_TRACE=1: print each check's line (stderr) before it runs, so a stall names its call
static const bool g_trace = std::getenv("ABI_ASAN_TRACE") != nullptr;
#define CHECK(cond, ...)                                                   \
  do {                                                                     \
    if (g_trace) std::fprintf(stderr, "check line %d\n", __LINE__);       \
    if (!(cond)) {                                                         \
      std::fprintf(stderr, "FAIL %s:%d: %s: ", __FILE__, __LINE__, #cond); \
      std::fprintf(stderr, __VA_ARGS__);                                   \
      std::fprintf(stderr, " [last_error: %s]\n", ecnf_last_error());      \
      ++g_fail;                                                            \
    }                                                                      \
  } while (0)

// the four examples/config/*.yaml flow blocks (dw4, lj13, aldp, qm9)
static ecnf_cfg make_cfg(int n, int d, int nf, int h, int m, int l, int k, float scale) {
  ecnf_cfg c;
  c.n_nodes = n; c.dim = d; c.n_features = nf; c.hidden = h; c.time_embedding_dim = 16; c.mlp_width = m;
  c.mlp_depth = l; c.n_blocks = k; c.base_scale = scale; c.normalization_constant = 1.0f;
  return c;
}

static std::vector<float> random_params(const ecnf_cfg& c, unsigned seed) {
  size_t n = 0;
  ecnf_param_count(&c, &n);
  std::vector<float> p(n);
  std::mt19937 rng(seed);
  std::normal_distribution<float> nd(0.f, 0.08f);
  for (auto& v : p) v = nd(rng);
  return p;
}

template <typename T>
static T* dev_alloc(size_t n) {
  void* p = nullptr;
  if (hipMalloc(&p, n * sizeof(T) + 16) != hipSuccess) return nullptr;
  hipMemset(p, 0, n * sizeof(T) + 16);
  return static_cast<T*>(p);
}

static void host_checks() {
  CHECK(ecnf_abi_version() == ECNF_ABI_VERSION, "abi %d", ecnf_abi_version());
  size_t n = 0;
  CHECK(ecnf_param_count(nullptr, &n) == ECNF_E_INVALID, "NULL cfg");
  ecnf_cfg bad = make_cfg(13, 3, 1, 64, 128, 3, 3, 1.f);
  bad.hidden = 33;
  CHECK(ecnf_param_count(&bad, &n) == ECNF_E_UNSUPPORTED, "hidden 33");
  bad = make_cfg(13, 3, 1, 64, 128, 3, 3, 1.f);
  bad.dim = 4;
  CHECK(ecnf_param_count(&bad, &n) == ECNF_E_UNSUPPORTED, "dim 4");
  bad = make_cfg(13, 3, 1, 64, 128, 3, 11, 1.f);
  CHECK(ecnf_param_count(&bad, &n) == ECNF_E_UNSUPPORTED, "11 blocks");
  bad.n_blocks = 3;
  bad.base_scale = 0.f;
  CHECK(ecnf_param_count(&bad, &n) == ECNF_E_INVALID, "base_scale 0");
  const ecnf_cfg ok = make_cfg(13, 3, 1, 64, 128, 3, 3, 1.f);
  CHECK(ecnf_param_count(&ok, &n) == ECNF_OK && n > 0, "lj13 count");
  ecnf_handle* h = nullptr;
  std::vector<float> p = random_params(ok, 1);
  CHECK(ecnf_create(&ok, nullptr, p.size(), 0, &h) == ECNF_E_INVALID, "NULL params");
  CHECK(ecnf_create(&ok, p.data(), p.size() - 1, 0, &h) == ECNF_E_INVALID, "short blob");
  CHECK(ecnf_create(&ok, p.data(), p.size(), 0, nullptr) == ECNF_E_INVALID, "NULL out");
  ecnf_cfg odd = ok;
  odd.mlp_width = 96;
  CHECK(ecnf_create(&odd, p.data(), p.size(), 0, &h) != ECNF_OK, "mlp_width 96");
  // weights at / beyond the split range are refused on the host (|w| >= 2^15)
  std::vector<float> big = p;
  big[big.size() / 2] = 1e6f;
  int rc = ecnf_create(&ok, big.data(), big.size(), 0, &h);
  CHECK(rc != ECNF_OK || h != nullptr, "huge weight rc %d", rc);
  if (rc == ECNF_OK) ecnf_destroy(h);
  ecnf_target t;
  std::memset(&t, 0, sizeof t);
  t.kind = 7;
  CHECK(ecnf_target_log_prob(&t, nullptr, nullptr, 1, nullptr) == ECNF_E_INVALID, "bad target kind");
  CHECK(ecnf_lse_partials(nullptr, nullptr, -1, nullptr, nullptr) == ECNF_E_INVALID, "lse n < 0");
  ecnf_trainer* tr = nullptr;
  CHECK(ecnf_trainer_create(&bad, 8, 0, &tr) == ECNF_E_INVALID, "trainer bad cfg");
  CHECK(ecnf_trainer_create(&ok, 0, 0, &tr) == ECNF_E_INVALID, "trainer max_batch 0");
  CHECK(ecnf_destroy(nullptr) == ECNF_OK || true, "destroy NULL");
}

// one C-ABI round trip per entry point on `cfg` (GPU present); returns false when the create fails with ECNF_E_HIP
static bool device_checks(const ecnf_cfg& c, int B) {
  std::vector<float> p = random_params(c, 7);
  ecnf_handle* h = nullptr;
  const int rc = ecnf_create(&c, p.data(), p.size(), 0, &h);
  if (rc == ECNF_E_HIP) return false;   // no GPU: the host walk / repack above already ran under ASan
  CHECK(rc == ECNF_OK && h, "create rc %d", rc);
  if (rc != ECNF_OK) return true;
  const int ND = c.n_nodes * c.dim;
  float* z = dev_alloc<float>((size_t)B * ND);
  float* x = dev_alloc<float>((size_t)B * ND);
  float* v = dev_alloc<float>((size_t)B * ND);
  float* y = dev_alloc<float>((size_t)B * ND);
  float* tt = dev_alloc<float>(B);
  float* lp = dev_alloc<float>(B);
  float* dl = dev_alloc<float>(B);
  int32_t* feat = dev_alloc<int32_t>((size_t)B * c.n_nodes);
  int32_t* nfe = dev_alloc<int32_t>(B);
  int32_t* st = dev_alloc<int32_t>(B);
  std::vector<float> hz((size_t)B * ND);
  std::mt19937 rng(3);
  std::normal_distribution<float> nd(0.f, 1.f);
  for (auto& q : hz) q = nd(rng);
  hipMemcpy(z, hz.data(), hz.size() * sizeof(float), hipMemcpyHostToDevice);
  std::vector<float> ht(B, 0.5f);
  hipMemcpy(tt, ht.data(), B * sizeof(float), hipMemcpyHostToDevice);

  CHECK(ecnf_base_sample(h, z, x, B, nullptr) == ECNF_OK, "base_sample");
  CHECK(ecnf_base_log_prob(h, x, lp, B, nullptr) == ECNF_OK, "base_log_prob");
  CHECK(ecnf_vector_field(h, x, tt, feat, v, B, nullptr) == ECNF_OK, "vector_field");
  CHECK(ecnf_vector_field(h, nullptr, tt, feat, v, B, nullptr) == ECNF_E_INVALID, "vector_field NULL x");
  CHECK(ecnf_vector_field(h, x, tt, feat, v, -1, nullptr) == ECNF_E_INVALID, "vector_field batch -1");
  ecnf_solve_opts o;
  std::memset(&o, 0, sizeof o);
  o.solver = ECNF_SOLVER_EULER; o.divergence = ECNF_DIV_NONE; o.t0 = 0.f; o.t1 = 1.f; o.dt0 = 0.1f;
  o.rtol = 1e-5f; o.atol = 1e-5f; o.dtmin = 0.f; o.max_steps = 4096;
  CHECK(ecnf_integrate(h, &o, x, feat, nullptr, y, nullptr, nfe, st, B, nullptr) == ECNF_OK, "integrate euler");
  o.divergence = ECNF_DIV_HUTCHINSON;
  int rcd = ecnf_integrate(h, &o, x, feat, nullptr, y, dl, nfe, st, B, nullptr);
  CHECK(rcd == ECNF_E_INVALID, "hutchinson without eps: %d", rcd);
  rcd = ecnf_integrate(h, &o, x, feat, z, y, dl, nfe, st, B, nullptr);
  CHECK(rcd == ECNF_OK || rcd == ECNF_E_UNSUPPORTED, "hutchinson: %d", rcd);
  // the exact trace: caller workspace (ecnf_integrate_ws), the handle arena, the A/B forms
  o.divergence = ECNF_DIV_EXACT; o.t0 = 1.f; o.t1 = 0.f; o.dt0 = 0.5f;
  size_t wsb = 0;
  CHECK(ecnf_integrate_workspace_size(h, &o, B, &wsb) == ECNF_OK, "workspace size");
  float* ws = wsb ? dev_alloc<float>(wsb / sizeof(float) + 1) : nullptr;
  rcd = ecnf_integrate_ws(h, &o, x, feat, nullptr, y, dl, nfe, st, B, ws, wsb, nullptr);
  CHECK(rcd == ECNF_OK || rcd == ECNF_E_UNSUPPORTED, "exact with workspace: %d", rcd);
  if (wsb) {
    CHECK(ecnf_integrate_ws(h, &o, x, feat, nullptr, y, dl, nfe, st, B, ws, wsb / 2, nullptr) == ECNF_E_INVALID,
          "undersized workspace");
    CHECK(ecnf_reserve_workspace(h, wsb) == ECNF_OK, "reserve workspace");
  }
  CHECK(ecnf_set_exact_form(h, ECNF_EXACT_FORM_SPARSE) == ECNF_OK, "exact form");
  CHECK(ecnf_set_exact_form(h, 7) == ECNF_E_INVALID, "bad exact form");
  rcd = ecnf_integrate(h, &o, x, feat, nullptr, y, dl, nfe, st, B, nullptr);
  CHECK(rcd == ECNF_OK || rcd == ECNF_E_UNSUPPORTED, "exact (sparse form): %d", rcd);
  CHECK(ecnf_set_exact_form(h, ECNF_EXACT_FORM_DEFAULT) == ECNF_OK, "exact form default");
  rcd = ecnf_integrate(h, &o, x, feat, nullptr, y, dl, nfe, st, B, nullptr);
  CHECK(rcd == ECNF_OK || rcd == ECNF_E_UNSUPPORTED, "exact (arena): %d", rcd);
  o.t0 = 0.f; o.t1 = 1.f; o.dt0 = 0.1f; o.divergence = ECNF_DIV_HUTCHINSON;
  o.solver = 9;
  CHECK(ecnf_integrate(h, &o, x, feat, z, y, dl, nfe, st, B, nullptr) == ECNF_E_INVALID, "bad solver");
  CHECK(ecnf_set_precision(h, 5) == ECNF_E_INVALID, "bad precision");
  CHECK(ecnf_set_precision(h, ECNF_PREC_FP32) == ECNF_OK, "fp32");
  CHECK(ecnf_vector_field(h, x, tt, feat, v, B, nullptr) == ECNF_OK, "vector_field fp32");
  int32_t mpw = 0, mode = -1;
  CHECK(ecnf_molecules_per_workgroup(h, 0, &mpw) == ECNF_OK && mpw > 0, "mpw");
  CHECK(ecnf_chain_arithmetic(h, 0, &mode) == ECNF_OK, "chain arithmetic");
  CHECK(ecnf_update_params(h, p.data(), 0) == ECNF_OK, "update_params host");
  CHECK(hipDeviceSynchronize() == hipSuccess, "sync");
  std::vector<float> hy((size_t)B * ND);
  hipMemcpy(hy.data(), y, hy.size() * sizeof(float), hipMemcpyDeviceToHost);
  bool finite = true;
  for (float q : hy) finite = finite && std::isfinite(q);
  CHECK(finite, "non-finite integrate output");

  ecnf_trainer* tr = nullptr;
  if (ecnf_trainer_create(&c, B, 0, &tr) == ECNF_OK) {
    size_t np = p.size();
    float* dp = dev_alloc<float>(np);
    float* g = dev_alloc<float>(np);
    float* loss = dev_alloc<float>(1);
    hipMemcpy(dp, p.data(), np * sizeof(float), hipMemcpyHostToDevice);
    CHECK(ecnf_fm_loss_grad(tr, dp, x, z, tt, feat, 0.01f, B, loss, g, nullptr) == ECNF_OK, "loss_grad");
    CHECK(ecnf_fm_loss_grad(tr, dp, x, z, tt, feat, 0.01f, B + 1, loss, g, nullptr) == ECNF_E_INVALID,
          "loss_grad over max_batch");
    hipDeviceSynchronize();
    hipFree(dp); hipFree(g); hipFree(loss);
    ecnf_trainer_destroy(tr);
  }
  CHECK(ecnf_destroy(h) == ECNF_OK, "destroy");
  for (void* q : {(void*)z, (void*)x, (void*)v, (void*)y, (void*)tt, (void*)lp, (void*)dl, (void*)feat, (void*)nfe,
                  (void*)st, (void*)ws})
    if (q) hipFree(q);
  return true;
}

extern "C" int ecnf_debug_refuse_teams(int refuse);   // this build only (ECNF_HOST_HOOKS)

// a refused cooperative launch: auto team mode gives the batch path's bits, a forced mode reports the refusal
static void team_checks(const ecnf_cfg& c, int B) {
  const std::vector<float> p = random_params(c, 5);
  ecnf_handle* h = nullptr;
  CHECK(ecnf_create(&c, p.data(), p.size(), 0, &h) == ECNF_OK && h, "create");
  if (!h) return;
  const size_t n = (size_t)B * c.n_nodes * c.dim;
  float *x = dev_alloc<float>(n), *y = dev_alloc<float>(n);
  int32_t* feat = dev_alloc<int32_t>((size_t)B * c.n_nodes);
  std::vector<float> hx(n);
  std::mt19937 rng(4);
  std::normal_distribution<float> nd(0.f, 1.f);
  for (auto& q : hx) q = nd(rng);
  hipMemcpy(x, hx.data(), n * sizeof(float), hipMemcpyHostToDevice);
  ecnf_solve_opts o;
  std::memset(&o, 0, sizeof o);
  o.solver = ECNF_SOLVER_EULER; o.divergence = ECNF_DIV_NONE; o.t1 = 1.f; o.dt0 = 0.25f;
  o.rtol = o.atol = 1e-5f; o.max_steps = 4096;
  int32_t G = 0;
  CHECK(ecnf_team_workgroups(h, 0, B, &G) == ECNF_OK && G > 1, "auto teams: %d", G);
  auto solve = [&](int mode, bool refuse, std::vector<float>& out) {
    CHECK(ecnf_set_team(h, mode) == ECNF_OK, "mode %d", mode);
    hipMemset(y, 0, n * sizeof(float));
    ecnf_debug_refuse_teams(refuse);
    const int rc = ecnf_integrate(h, &o, x, feat, nullptr, y, nullptr, nullptr, nullptr, B, nullptr);
    ecnf_debug_refuse_teams(0);
    out.resize(n);
    CHECK(hipDeviceSynchronize() == hipSuccess, "sync");
    hipMemcpy(out.data(), y, n * sizeof(float), hipMemcpyDeviceToHost);
    return rc;
  };
  std::vector<float> batch, refused, again, none;
  CHECK(solve(1, false, batch) == ECNF_OK, "batch path");
  CHECK(solve(0, true, refused) == ECNF_OK, "auto, refused");
  CHECK(std::memcmp(batch.data(), refused.data(), n * sizeof(float)) == 0, "auto, refused: not the batch path's bits");
  CHECK(solve(7, true, none) == ECNF_E_HIP, "forced, refused");
  for (float q : none) CHECK(q == 0.f, "forced, refused: wrote %g", q);
  CHECK(solve(1, true, again) == ECNF_OK, "teams off need no cooperative launch");
  CHECK(std::memcmp(batch.data(), again.data(), n * sizeof(float)) == 0, "teams off, refused");
  CHECK(solve(0, false, again) == ECNF_OK, "auto");
  CHECK(std::memcmp(batch.data(), again.data(), n * sizeof(float)) == 0, "auto: not the batch path's bits");
  CHECK(ecnf_destroy(h) == ECNF_OK, "destroy");
  for (void* q : {(void*)x, (void*)y, (void*)feat}) hipFree(q);
}

// the context operators: refusals on the host; with a device also one small forward and backward pass of each
static void context_checks(bool gpu) {
  ecnf_qk_norm n;
  std::memset(&n, 0, sizeof n);
  size_t bytes = 0;
  CHECK(ecnf_qk_norm_workspace_size(nullptr, &bytes) == ECNF_E_INVALID, "norm NULL");
  CHECK(ecnf_qk_norm_rotary(&n, nullptr) == ECNF_E_UNSUPPORTED, "norm head_dim 0");
  CHECK(ecnf_qk_norm_rotary_grad(&n, nullptr, 0, nullptr) == ECNF_E_UNSUPPORTED, "norm grad head_dim 0");
  ecnf_attention a;
  std::memset(&a, 0, sizeof a);
  CHECK(ecnf_cross_attention_workspace_size(&a, 0, &bytes) == ECNF_E_INVALID, "attention empty");
  CHECK(ecnf_cross_attention(&a, nullptr, 0, nullptr) == ECNF_E_INVALID, "attention empty");
  CHECK(ecnf_cross_attention_grad(&a, nullptr, 0, nullptr) == ECNF_E_INVALID, "attention grad empty");
  CHECK(ecnf_vector_field_nodes(nullptr, nullptr, nullptr, nullptr, 1, nullptr, nullptr, 1, nullptr) == ECNF_E_INVALID, "nodes");
  CHECK(ecnf_integrate_nodes(nullptr, nullptr, nullptr, nullptr, 1, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 1,
                             nullptr, 0, nullptr) == ECNF_E_INVALID, "integrate nodes");
  CHECK(ecnf_fm_loss_grad_nodes(nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, 0.f, 1, nullptr, nullptr, nullptr,
                                nullptr) == ECNF_E_INVALID, "loss nodes");
  if (!gpu) return;
  const int B = 2, Lq = 5, Lk = 300, H = 2, D = 16;
  float *q = dev_alloc<float>(B * Lq * H * D), *k = dev_alloc<float>(B * Lk * H * D), *o = dev_alloc<float>(B * Lq * H * D);
  float *dq = dev_alloc<float>(B * Lq * H * D), *dk = dev_alloc<float>(B * Lk * H * D), *dv = dev_alloc<float>(B * Lk * H * D);
  float *lse = dev_alloc<float>(B * H * Lq), *w = dev_alloc<float>(D), *dw = dev_alloc<float>(D);
  int32_t* pos = dev_alloc<int32_t>(Lq);
  n.q.x = q; n.q.grad = o; n.q.out = dq; n.q.weight = w; n.q.weight_grad = dw; n.q.positions = pos;
  n.q.batch = B; n.q.length = Lq; n.q.heads = H; n.q.position_type = ECNF_POS_I32; n.q.position_stride[1] = 1;
  for (int64_t* st : {n.q.x_stride, n.q.grad_stride, a.q_stride, a.out_grad_stride}) st[0] = Lq * H * D, st[1] = H * D, st[2] = D;
  for (int64_t* st : {a.k_stride, a.v_stride}) st[0] = Lk * H * D, st[1] = H * D, st[2] = D;
  n.dtype = ECNF_DTYPE_F32; n.head_dim = D; n.n_axes = 1; n.axes[0] = D; n.eps = 1e-6f; n.theta = 1e4;
  CHECK(ecnf_qk_norm_rotary(&n, nullptr) == ECNF_OK, "norm");
  CHECK(ecnf_qk_norm_workspace_size(&n, &bytes) == ECNF_OK && bytes > 0, "norm workspace");
  float* ws = dev_alloc<float>(bytes / 4);
  CHECK(ecnf_qk_norm_rotary_grad(&n, ws, bytes, nullptr) == ECNF_OK, "norm grad");
  CHECK(ecnf_qk_norm_rotary_grad(&n, ws, bytes - 1, nullptr) == ECNF_E_INVALID, "norm grad, small workspace");
  hipFree(ws);
  a.q = q; a.k = k; a.v = k; a.out = o; a.out_grad = o; a.lse = lse; a.q_grad = dq; a.k_grad = dk; a.v_grad = dv;
  a.dtype = ECNF_DTYPE_F32; a.batch = a.context_batch = B; a.n_queries = Lq; a.context_length = Lk; a.heads = a.kv_heads = H;
  a.head_dim = D; a.scale = 0.25f;
  for (int grad = 0; grad < 2; ++grad) {
    CHECK(ecnf_cross_attention_workspace_size(&a, grad, &bytes) == ECNF_OK, "attention workspace");
    ws = dev_alloc<float>(bytes / 4 + 4);
    const int rc = grad ? ecnf_cross_attention_grad(&a, ws, bytes, nullptr) : ecnf_cross_attention(&a, ws, bytes, nullptr);
    CHECK(rc == ECNF_OK, "attention %d", grad);
    CHECK(hipDeviceSynchronize() == hipSuccess, "attention %d", grad);
    hipFree(ws);
  }
  for (void* p : {(void*)q, (void*)k, (void*)o, (void*)dq, (void*)dk, (void*)dv, (void*)lse, (void*)w, (void*)dw, (void*)pos})
    if (p) hipFree(p);
}

int main() {
  host_checks();
  const ecnf_cfg cfgs[] = {make_cfg(4, 2, 1, 64, 128, 3, 3, 1.f), make_cfg(13, 3, 1, 64, 128, 3, 3, 1.f),
                           make_cfg(22, 3, 22, 32, 64, 2, 3, 0.2f), make_cfg(29, 3, 1, 32, 256, 4, 5, 2.f)};
  int gpu = 0;
  for (const auto& c : cfgs) {
    if (g_trace) std::fprintf(stderr, "config N = %d, M = %d\n", c.n_nodes, c.mlp_width);
    gpu += device_checks(c, 5) ? 1 : 0;
  }
  context_checks(gpu > 0);
  if (gpu) team_checks(cfgs[3], 2);
  {
    size_t lay[32];
    for (int w = 0; w < 7; ++w) CHECK(ecnf_struct_layout(w, lay, 32) > 0, "struct layout %d", w);
    CHECK(ecnf_struct_layout(9, lay, 32) == -1, "bad struct");
  }
  // scoped leak check of every allocation made through the library above (the ROCm runtime's own allocations are
  // suppressed by lsan.supp); run here, while the process is live, instead of at exit (leak_check_at_exit=0)
  const auto t0 = std::chrono::steady_clock::now();
  const int leaked = __lsan_do_recoverable_leak_check();
  const double ms = std::chrono::duration<double, std::milli>(std::chrono::steady_clock::now() - t0).count();
  std::printf("abi_asan: leak check %s in %.0f ms\n", leaked ? "FOUND LEAKS" : "clean", ms);
  if (leaked) ++g_fail;
  std::printf("abi_asan: %s, %d failure(s)\n", gpu ? "host + device paths" : "host paths only (no GPU)", g_fail);
  return g_fail ? 1 : 0;
}

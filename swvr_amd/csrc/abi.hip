// C ABI entry points (include/swvr.h): argument checks, error reporting,
// launch timing, and dispatch to the forward / backward launchers.
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <cstddef>
#include <mutex>
#include <vector>

#include "../../include/swvr.h"
#include "launch.hpp"

namespace swvr {

namespace {

thread_local char g_err[512] = "";

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof(g_err), fmt, ap);
  va_end(ap);
  return code;
}

int hip_fail(hipError_t e, const char* what) {
  return fail(SWVR_EHIP, "%s: %s (%d)", what, hipGetErrorString(e), (int)e);
}

// ---- launch timing: event pairs per kernel kind, recorded on the launch stream
struct TimedLaunch {
  int kind;
  hipEvent_t start, stop;
};
std::mutex g_tmu;
bool g_timing = false;
std::vector<TimedLaunch> g_launches;
std::vector<hipEvent_t> g_pool;
// Start events of launches whose end is not yet recorded, keyed by (stream, kind):
// launches of one kind on different streams (or threads) pair their own events.
struct PendingLaunch {
  hipStream_t stream;
  int kind;
  hipEvent_t start;
};
std::vector<PendingLaunch> g_pending;

hipEvent_t take_event() {
  if (!g_pool.empty()) {
    hipEvent_t e = g_pool.back();
    g_pool.pop_back();
    return e;
  }
  hipEvent_t e = nullptr;
  if (hipEventCreate(&e) != hipSuccess) return nullptr;
  return e;
}

const char* kKindNames[kNumKinds] = {"fwd_tile_kernel",   "fwd_combine_kernel", "bwd_pack_kernel",
                                     "bwd_scores_kernel", "bwd_gemm_kernel",    "bwd_reduce_kernel",
                                     "fill_zero_kernel",  "operand_packing",    "bwd_expand_kernel",
                                     "mse_loss",          "quantize_e4m3",      "readout_f64",
                                     "probe_mfma",        "embedding",          "sort_ids",
                                     "distill",           "sample_tokens"};

bool is_dtype(int d) { return d == SWVR_BF16 || d == SWVR_F16 || d == SWVR_F32; }

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

int check_common(int dtype, int64_t N, int64_t K, int64_t V, int64_t D, const void* h, int64_t ldh, const void* W,
                 int64_t ldw, const void* E, int64_t lde) {
  if (!is_dtype(dtype)) return fail(SWVR_EDTYPE, "unsupported operand dtype tag %d", dtype);
  if (N < 0 || K < 0 || V < 0 || D < 0) return fail(SWVR_EINVAL, "negative size N=%lld K=%lld V=%lld D=%lld",
                                                    (long long)N, (long long)K, (long long)V, (long long)D);
  if (N > INT32_MAX || K > INT32_MAX || V > INT32_MAX || D > INT32_MAX)
    return fail(SWVR_EINVAL, "sizes must fit in 32 bits");
  if (D > swvr_max_d(dtype))
    return fail(SWVR_EDTYPE, "D=%lld exceeds the maximum %lld for this dtype", (long long)D,
                (long long)swvr_max_d(dtype));
  if (K % 8 != 0) return fail(SWVR_EINVAL, "K=%lld must be a multiple of 8 (pad h and W)", (long long)K);
  // tile-relative byte offsets of the kernels are 32-bit: 128 rows x K fp32 stay below 2^31
  if (K > (int64_t)1 << 21) return fail(SWVR_EINVAL, "K=%lld exceeds the maximum %lld", (long long)K, 1LL << 21);
  if (ldh < K || ldh % 8 != 0) return fail(SWVR_EINVAL, "ldh=%lld must be >= K and a multiple of 8", (long long)ldh);
  if (ldw < K || ldw % 8 != 0) return fail(SWVR_EINVAL, "ldw=%lld must be >= K and a multiple of 8", (long long)ldw);
  if (lde < D) return fail(SWVR_EINVAL, "lde=%lld must be >= D", (long long)lde);
  if (N > 0 && K > 0 && (!h || !aligned16(h))) return fail(SWVR_EINVAL, "h must be a non-null 16-byte aligned pointer");
  if (V > 0 && K > 0 && (!W || !aligned16(W))) return fail(SWVR_EINVAL, "W must be a non-null 16-byte aligned pointer");
  if (V > 0 && D > 0 && !E) return fail(SWVR_EINVAL, "E must be non-null");
  return SWVR_OK;
}

}  // namespace

void timing_begin(int kind, hipStream_t stream) {
  if (!g_timing) return;
  std::lock_guard<std::mutex> lk(g_tmu);
  hipEvent_t e = take_event();
  if (e && hipEventRecord(e, stream) == hipSuccess) g_pending.push_back({stream, kind, e});
}

void timing_end(int kind, hipStream_t stream) {
  if (!g_timing) return;
  std::lock_guard<std::mutex> lk(g_tmu);
  // the latest unmatched start of this kind on this stream
  for (size_t i = g_pending.size(); i-- > 0;) {
    if (g_pending[i].stream != stream || g_pending[i].kind != kind) continue;
    const hipEvent_t s = g_pending[i].start;
    g_pending.erase(g_pending.begin() + (std::ptrdiff_t)i);
    hipEvent_t e = take_event();
    if (e && hipEventRecord(e, stream) == hipSuccess)
      g_launches.push_back({kind, s, e});
    else
      g_pool.push_back(s);
    return;
  }
}

namespace {

// Storage dtype of h or W: the compute dtype, or fp32 under a 2-byte compute dtype.
int check_storage(int dtype, int h_dtype, int w_dtype) {
  const bool two = dtype == SWVR_BF16 || dtype == SWVR_F16;
  if (!(h_dtype == dtype || (two && h_dtype == SWVR_F32)))
    return fail(SWVR_EDTYPE, "h dtype tag %d with compute dtype %d", h_dtype, dtype);
  if (!(w_dtype == dtype || (two && w_dtype == SWVR_F32)))
    return fail(SWVR_EDTYPE, "W dtype tag %d with compute dtype %d", w_dtype, dtype);
  return SWVR_OK;
}

// A launch of 2^32 threads or more runs the remainder alone, without an error: such sizes are refused.
int check_threads(int64_t most) {
  return most + 1024 < ((int64_t)1 << 32) ? SWVR_OK : fail(SWVR_EINVAL, "sizes need a launch of 2^32 threads or more");
}

int fwd_common(int dtype, int h_dtype, int w_dtype, int64_t N, int64_t K, int64_t V, int64_t D, const void* h,
               int64_t ldh, const void* W, int64_t ldw, const void* E, int64_t lde, const float* bias,
               float logit_scale, float* O, float* lse, float* m_out, float* l_out, void* workspace,
               size_t workspace_bytes, void* stream, bool active = false, const float* weight = nullptr,
               float* scores = nullptr) {
  g_err[0] = 0;
  int rc = check_common(dtype, N, K, V, D, h, ldh, W, ldw, E, lde);
  if (rc != SWVR_OK) return rc;
  if ((rc = check_storage(dtype, h_dtype, w_dtype)) != SWVR_OK) return rc;
  if (N > 0 && ((D > 0 && !O) || (m_out ? !l_out : !lse)))
    return fail(SWVR_EINVAL, m_out ? "m, l and acc must be non-null" : "O and lse must be non-null");
  FwdPlan plan;
  if (!fwd_plan(dtype, N, K, V, D, &plan, active))
    return fail(SWVR_EDTYPE, "no forward kernel for dtype %d, D=%lld", dtype, (long long)D);
  if (N == 0) return SWVR_OK;
  // the merge's 4 columns of a token in a pass of DS, the flags' wave a token
  if ((rc = check_threads(std::max(N * ((std::min<int64_t>(D, plan.DS) + 3) / 4), active ? 64 * N : 0))) != SWVR_OK)
    return rc;
  if (!workspace || workspace_bytes < plan.ws_bytes)
    return fail(SWVR_EWORKSPACE, "forward workspace of %zu bytes needed, %zu given", plan.ws_bytes, workspace_bytes);
  FwdParams p{};
  p.h = h;
  p.ldh = ldh;
  p.W = W;
  p.ldw = ldw;
  p.E = E;
  p.lde = lde;
  p.bias = bias;
  p.scale = logit_scale;
  p.N = (int)N;
  p.K = (int)K;
  p.V = (int)V;
  p.D = (int)D;
  p.h_f32 = h_dtype != dtype;
  p.w_f32 = w_dtype != dtype;
  p.scores = scores;
  hipError_t e = active ? fwd_launch_active(dtype, plan, p, weight, static_cast<char*>(workspace), O, lse,
                                            static_cast<hipStream_t>(stream))
                        : fwd_launch(dtype, plan, p, static_cast<char*>(workspace), O, lse, m_out, l_out,
                                     static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "forward launch");
  return SWVR_OK;
}

int bwd_common(int dtype, int h_dtype, int w_dtype, int64_t N, int64_t K, int64_t V, int64_t D, const void* h,
                   int64_t ldh, const void* W, int64_t ldw, const void* E, int64_t lde, const float* bias,
                   float logit_scale, const float* O, const float* lse, const float* gO, const float* glse,
                   int64_t chunk, void* gh, int gh_dtype, void* gW, int gW_dtype, void* gE, int gE_dtype, float* gb,
                   void* workspace, size_t workspace_bytes, void* stream, const void* hq = nullptr,
                   int64_t K8 = 0, int64_t ldhq = 0, const float* h_scale = nullptr, const void* Wq = nullptr,
                   int64_t ldwq = 0, const float* w_scale = nullptr, const int* pt_id = nullptr,
                   const float* pt_val = nullptr, int64_t n_pt = 0, int pt_T = 1, const float* scores = nullptr,
                   int64_t lds = 0) {
  g_err[0] = 0;
  int rc = check_common(dtype, N, K, V, D, h, ldh, W, ldw, E, lde);
  if (rc != SWVR_OK) return rc;
  if ((rc = check_storage(dtype, h_dtype, w_dtype)) != SWVR_OK) return rc;
  if (chunk <= 0) return fail(SWVR_EINVAL, "chunk must be positive, got %lld", (long long)chunk);
  if (gh && !is_dtype(gh_dtype)) return fail(SWVR_EDTYPE, "unsupported gh dtype tag %d", gh_dtype);
  if (gW && !is_dtype(gW_dtype)) return fail(SWVR_EDTYPE, "unsupported gW dtype tag %d", gW_dtype);
  if (gE && !is_dtype(gE_dtype)) return fail(SWVR_EDTYPE, "unsupported gE dtype tag %d", gE_dtype);
  if (gb && !bias) return fail(SWVR_EINVAL, "gb requested without a bias");
  if (N > 0 && (!lse || (!glse && !pt_id) || (D > 0 && (!O || !gO))))
    return fail(SWVR_EINVAL, "O, lse, gO and glse must be non-null");
  BwdPlan plan;
  if (!bwd_plan(dtype, N, K, V, D, chunk, gh != nullptr, &plan, w_dtype != dtype, hq ? K8 : 0))
    return fail(SWVR_EDTYPE, "no backward kernel for dtype %d, D=%lld", dtype, (long long)D);
  // gO's packing, E's, delta's 16 lanes a token, gh's 4 columns
  if ((rc = check_threads(std::max({plan.N_pad * plan.DP, (int64_t)plan.V_pad * (plan.DP / 8), 16 * N,
                                    gh ? N * (K / 4) : 0}))) != SWVR_OK)
    return rc;
  if (N > 0 && (!workspace || workspace_bytes < plan.ws_bytes))
    return fail(SWVR_EWORKSPACE, "backward workspace of %zu bytes needed, %zu given", plan.ws_bytes, workspace_bytes);
  BwdParams p{};
  p.h = h;
  p.ldh = ldh;
  p.W = W;
  p.ldw = ldw;
  p.E = E;
  p.lde = lde;
  p.bias = bias;
  p.scale = logit_scale;
  p.N = (int)N;
  p.K = (int)K;
  p.V = (int)V;
  p.D = (int)D;
  p.O = O;
  p.lse = lse;
  p.gO = gO;
  p.glse = glse;
  p.gh = gh;
  p.gh_dtype = gh_dtype;
  p.gW = gW;
  p.gW_dtype = gW_dtype;
  p.gE = gE;
  p.gE_dtype = gE_dtype;
  p.gb = gb;
  p.ws = static_cast<char*>(workspace);
  p.h_f32 = h_dtype != dtype;
  p.w_f32 = w_dtype != dtype;
  p.hq = hq;
  p.ldhq = ldhq;
  p.Wq = Wq;
  p.ldwq = ldwq;
  p.h_scale = h_scale;
  p.w_scale = w_scale;
  p.K8 = (int)K8;
  p.pt_id = pt_id;
  p.pt_val = pt_val;
  p.n_pt = n_pt;
  p.pt_T = pt_T;
  p.scores = scores;
  p.lds = lds;
  hipError_t e = bwd_launch(dtype, plan, p, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "backward launch");
  return SWVR_OK;
}

}  // namespace

}  // namespace swvr

using namespace swvr;

extern "C" {

int swvr_abi_version(void) { return SWVR_ABI_VERSION; }

const char* swvr_last_error(void) { return g_err; }

int64_t swvr_max_d(int dtype) {
  if (dtype == SWVR_F32 || dtype == SWVR_BF16 || dtype == SWVR_F16) return SWVR_MAX_D;
  return 0;
}

size_t swvr_fwd_workspace_size(int dtype, int64_t N, int64_t K, int64_t V, int64_t D) {
  FwdPlan plan;
  if (N < 0 || V < 0 || D < 0 || !fwd_plan(dtype, N, K, V, D, &plan)) return 0;
  return plan.ws_bytes;
}

int swvr_fwd(int dtype, int64_t N, int64_t K, int64_t V, int64_t D, const void* h, int64_t ldh, const void* W,
             int64_t ldw, const void* E, int64_t lde, const float* bias, float logit_scale, float* O, float* lse,
             void* workspace, size_t workspace_bytes, void* stream) {
  return fwd_common(dtype, dtype, dtype, N, K, V, D, h, ldh, W, ldw, E, lde, bias, logit_scale, O, lse, nullptr,
                    nullptr, workspace, workspace_bytes, stream);
}

int swvr_fwd_mixed(int dtype, int h_dtype, int w_dtype, int64_t N, int64_t K, int64_t V, int64_t D, const void* h,
                   int64_t ldh, const void* W, int64_t ldw, const void* E, int64_t lde, const float* bias,
                   float logit_scale, float* O, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  return fwd_common(dtype, h_dtype, w_dtype, N, K, V, D, h, ldh, W, ldw, E, lde, bias, logit_scale, O, lse, nullptr,
                    nullptr, workspace, workspace_bytes, stream);
}

size_t swvr_fwd_active_workspace_size(int dtype, int64_t N, int64_t K, int64_t V, int64_t D) {
  FwdPlan plan;
  if (N < 0 || V < 0 || D < 0 || !fwd_plan(dtype, N, K, V, D, &plan, true)) return 0;
  return plan.ws_bytes;
}

int swvr_fwd_active(int dtype, int h_dtype, int w_dtype, int64_t N, int64_t K, int64_t V, int64_t D, const void* h,
                    int64_t ldh, const void* W, int64_t ldw, const void* E, int64_t lde, const float* bias,
                    float logit_scale, const float* weight, float* O, float* lse, void* workspace,
                    size_t workspace_bytes, void* stream) {
  if (N > 0 && !weight) {
    g_err[0] = 0;
    return fail(SWVR_EINVAL, "weight must be non-null");
  }
  return fwd_common(dtype, h_dtype, w_dtype, N, K, V, D, h, ldh, W, ldw, E, lde, bias, logit_scale, O, lse, nullptr,
                    nullptr, workspace, workspace_bytes, stream, true, weight);
}

int swvr_fwd_partial(int dtype, int64_t N, int64_t K, int64_t V, int64_t D, const void* h, int64_t ldh,
                     const void* W, int64_t ldw, const void* E, int64_t lde, const float* bias, float logit_scale,
                     float* m, float* l, float* acc, void* workspace, size_t workspace_bytes, void* stream) {
  if (!m && N > 0) {
    g_err[0] = 0;
    return fail(SWVR_EINVAL, "m, l and acc must be non-null");
  }
  return fwd_common(dtype, dtype, dtype, N, K, V, D, h, ldh, W, ldw, E, lde, bias, logit_scale, acc, nullptr, m, l,
                    workspace, workspace_bytes, stream);
}

int swvr_combine(int64_t S, int64_t N, int64_t D, const float* m, const float* l, const float* acc, float* O,
                 float* lse, void* stream) {
  g_err[0] = 0;
  if (S < 1 || N < 0 || D < 0) return fail(SWVR_EINVAL, "bad sizes S=%lld N=%lld D=%lld", (long long)S, (long long)N,
                                           (long long)D);
  if (S > INT32_MAX || N > INT32_MAX || D > INT32_MAX) return fail(SWVR_EINVAL, "sizes must fit in 32 bits");
  if (N == 0) return SWVR_OK;
  if (!m || !l || !lse || (D > 0 && (!acc || !O))) return fail(SWVR_EINVAL, "m, l, acc, O and lse must be non-null");
  hipError_t e = shard_combine((int)S, (int)N, (int)D, m, l, acc, O, lse, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "combine launch");
  return SWVR_OK;
}

size_t swvr_bwd_workspace_size_mixed(int dtype, int w_dtype, int64_t N, int64_t K, int64_t V, int64_t D,
                                     int64_t chunk, int need_gh) {
  BwdPlan plan;
  if (N < 0 || V < 0 || D < 0 || chunk <= 0 ||
      !bwd_plan(dtype, N, K, V, D, chunk, need_gh != 0, &plan, w_dtype != dtype))
    return 0;
  return plan.ws_bytes;
}

size_t swvr_bwd_workspace_size(int dtype, int64_t N, int64_t K, int64_t V, int64_t D, int64_t chunk, int need_gh) {
  return swvr_bwd_workspace_size_mixed(dtype, dtype, N, K, V, D, chunk, need_gh);
}

int64_t swvr_bwd_default_chunk(int dtype, int w_dtype, int64_t N, int64_t K, int64_t K8, int64_t V, int64_t D,
                               int need_gh) {
  if (!is_dtype(dtype) || N < 0 || K < 0 || K8 < 0 || V < 0 || D < 0) return 0;
  return bwd_default_chunk(dtype, N, K, V, D, need_gh != 0, w_dtype != dtype, K8);
}

int swvr_bwd_tiling(int dtype, int64_t N, int64_t K, int64_t V, int64_t D, int64_t chunk, int64_t* out, int n_out) {
  g_err[0] = 0;
  if (!out || n_out < 0) return fail(SWVR_EINVAL, "out must be non-null");
  BwdPlan plan;
  if (N < 0 || K < 0 || V < 0 || D < 0 || chunk <= 0)
    return fail(SWVR_EINVAL, "bad sizes N=%lld K=%lld V=%lld D=%lld chunk=%lld", (long long)N, (long long)K,
                (long long)V, (long long)D, (long long)chunk);
  if (!bwd_plan(dtype, N, K, V, D, chunk, true, &plan))
    return fail(SWVR_EDTYPE, "no backward kernel for dtype %d, D=%lld", dtype, (long long)D);
  const int64_t v[7] = {plan.BM, plan.BV, plan.G, plan.C, plan.n_chunks, plan.DP, plan.kind};
  const int n = n_out < 7 ? n_out : 7;
  for (int i = 0; i < n; ++i) out[i] = v[i];
  return 7;
}

int swvr_bwd_mixed(int dtype, int h_dtype, int w_dtype, int64_t N, int64_t K, int64_t V, int64_t D, const void* h,
                   int64_t ldh, const void* W, int64_t ldw, const void* E, int64_t lde, const float* bias,
                   float logit_scale, const float* O, const float* lse, const float* gO, const float* glse,
                   int64_t chunk, void* gh, int gh_dtype, void* gW, int gW_dtype, void* gE, int gE_dtype, float* gb,
                   void* workspace, size_t workspace_bytes, void* stream) {
  return bwd_common(dtype, h_dtype, w_dtype, N, K, V, D, h, ldh, W, ldw, E, lde, bias, logit_scale, O, lse, gO, glse,
                    chunk, gh, gh_dtype, gW, gW_dtype, gE, gE_dtype, gb, workspace, workspace_bytes, stream);
}

size_t swvr_bwd_fp8_workspace_size(int64_t N, int64_t K, int64_t K8, int64_t V, int64_t D, int64_t chunk,
                                   int need_gh) {
  BwdPlan plan;
  if (N < 0 || V < 0 || D < 0 || chunk <= 0 || K8 <= 0 ||
      !bwd_plan(SWVR_BF16, N, K, V, D, chunk, need_gh != 0, &plan, false, K8))
    return 0;
  return plan.ws_bytes;
}

int swvr_bwd_fp8(int64_t N, int64_t K, int64_t V, int64_t D, const void* h, int64_t ldh, const void* W, int64_t ldw,
                 const void* E, int64_t lde, const float* bias, float logit_scale, const void* hq, int64_t K8,
                 int64_t ldhq, const float* h_scale, const void* Wq, int64_t ldwq, const float* w_scale,
                 const float* O, const float* lse, const float* gO, const float* glse, int64_t chunk, void* gh,
                 int gh_dtype, void* gW, int gW_dtype, void* gE, int gE_dtype, float* gb, void* workspace,
                 size_t workspace_bytes, void* stream) {
  g_err[0] = 0;
  if (D > 128) return fail(SWVR_EDTYPE, "D=%lld exceeds the maximum 128 of the e4m3 scores", (long long)D);
  if (K8 < K || K8 % 16 != 0 || ldhq < K8 || ldhq % 16 != 0 || ldwq < K8 || ldwq % 16 != 0)
    return fail(SWVR_EINVAL, "K8=%lld (>= K), ldhq=%lld and ldwq=%lld (>= K8) must be multiples of 16",
                (long long)K8, (long long)ldhq, (long long)ldwq);
  if (K8 > ((int64_t)1 << 22)) return fail(SWVR_EINVAL, "K8=%lld too large", (long long)K8);
  if (N > 0 && V > 0 && (!hq || !Wq || !h_scale || !w_scale || !aligned16(hq) || !aligned16(Wq)))
    return fail(SWVR_EINVAL, "hq, Wq (16-byte aligned), h_scale and w_scale must be non-null");
  return bwd_common(SWVR_BF16, SWVR_BF16, SWVR_BF16, N, K, V, D, h, ldh, W, ldw, E, lde, bias, logit_scale, O, lse,
                    gO, glse, chunk, gh, gh_dtype, gW, gW_dtype, gE, gE_dtype, gb, workspace, workspace_bytes, stream,
                    hq, K8, ldhq, h_scale, Wq, ldwq, w_scale);
}

int swvr_bwd(int dtype, int64_t N, int64_t K, int64_t V, int64_t D, const void* h, int64_t ldh, const void* W,
             int64_t ldw, const void* E, int64_t lde, const float* bias, float logit_scale, const float* O,
             const float* lse, const float* gO, const float* glse, int64_t chunk, void* gh, int gh_dtype, void* gW,
             int gW_dtype, void* gE, int gE_dtype, float* gb, void* workspace, size_t workspace_bytes,
             void* stream) {
  return swvr_bwd_mixed(dtype, dtype, dtype, N, K, V, D, h, ldh, W, ldw, E, lde, bias, logit_scale, O, lse, gO, glse,
                        chunk, gh, gh_dtype, gW, gW_dtype, gE, gE_dtype, gb, workspace, workspace_bytes, stream);
}

// ---------------------------------------------------------------- embedding lookup
// The kernels step over columns and rows of the table in 32 bits, past the last by up to a workgroup's.
static bool embed_sizes(int64_t N, int64_t V, int64_t D) {
  return N >= 0 && V >= 0 && D >= 0 && N <= INT32_MAX && V <= SWVR_EMBED_MAX && D <= SWVR_EMBED_MAX;
}

static int check_embed(int dtype, int id64, int64_t N, int64_t V, int64_t D, const void* ids) {
  g_err[0] = 0;
  if (!is_dtype(dtype) && dtype != SWVR_F64) return fail(SWVR_EDTYPE, "unsupported dtype tag %d", dtype);
  if (id64 != 0 && id64 != 1) return fail(SWVR_EINVAL, "ids are int32 (0) or int64 (1), got %d", id64);
  if (!embed_sizes(N, V, D))
    return fail(SWVR_EINVAL, "bad sizes N=%lld V=%lld D=%lld (N below 2^31, V and D at most 2^30)", (long long)N,
                (long long)V, (long long)D);
  if (N > 0 && !ids) return fail(SWVR_EINVAL, "ids must be non-null");
  return SWVR_OK;
}

int swvr_embedding(int dtype, int id64, int64_t N, int64_t V, int64_t D, const void* ids, const void* E, int64_t lde,
                   double scale, void* out, int* sorted, void* stream) {
  const int rc = check_embed(dtype, id64, N, V, D, ids);
  if (rc != SWVR_OK) return rc;
  if (lde < D) return fail(SWVR_EINVAL, "lde=%lld must be >= D", (long long)lde);
  if (N > 0 && D > 0 && ((V > 0 && !E) || !out)) return fail(SWVR_EINVAL, "E and out must be non-null");
  swvr::EmbedParams p{};
  p.dtype = dtype;
  p.ids = ids;
  p.id64 = id64;
  p.N = N;
  p.V = (int)V;
  p.D = (int)D;
  p.E = E;
  p.lde = lde;
  p.scale = scale;
  p.out = out;
  hipError_t e = swvr::embed_lookup_launch(p, static_cast<hipStream_t>(stream));
  if (e == hipSuccess && sorted) e = swvr::embed_sort(p, sorted, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "embedding launch");
  return SWVR_OK;
}

size_t swvr_embedding_sorted_size(int64_t N, int64_t V) {
  if (!embed_sizes(N, V, 0)) return 0;
  return swvr::embed_sorted_ints(N, V) * sizeof(int);
}

size_t swvr_embedding_bwd_workspace_size(int dtype, int64_t N, int64_t V, int64_t D) {
  if ((!is_dtype(dtype) && dtype != SWVR_F64) || !embed_sizes(N, V, D)) return 0;
  return swvr::embed_grad_workspace_bytes(dtype, N, V, D);
}

int swvr_embedding_bwd(int dtype, int id64, int64_t N, int64_t V, int64_t D, const void* ids, const void* g,
                       int64_t ldg, double scale, const int* sorted, void* gE, void* workspace, size_t workspace_bytes,
                       void* stream) {
  const int rc = check_embed(dtype, id64, N, V, D, ids);
  if (rc != SWVR_OK) return rc;
  if (ldg < 0) return fail(SWVR_EINVAL, "ldg=%lld must not be negative", (long long)ldg);
  if (V > 0 && D > 0 && ((N > 0 && !g) || !gE)) return fail(SWVR_EINVAL, "g and gE must be non-null");
  const size_t need = swvr::embed_grad_workspace_bytes(dtype, N, V, D);
  if ((need > 0 && !workspace) || workspace_bytes < need)
    return fail(SWVR_EWORKSPACE, "embedding workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  swvr::EmbedParams p{};
  p.dtype = dtype;
  p.ids = ids;
  p.id64 = id64;
  p.N = N;
  p.V = (int)V;
  p.D = (int)D;
  p.scale = scale;
  p.g = g;
  p.ldg = ldg;
  p.gE = gE;
  hipError_t e = swvr::embed_grad_launch(p, sorted, static_cast<char*>(workspace), static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "embedding gradient launch");
  return SWVR_OK;
}

// ---------------------------------------------------------------- distillation
static size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

static int check_distill(int dtype, int64_t N, int64_t V, int64_t T, int id64, const void* ids, int64_t ldi,
                         float temperature, int reduction) {
  g_err[0] = 0;
  if (!is_dtype(dtype)) return fail(SWVR_EDTYPE, "unsupported operand dtype tag %d", dtype);
  // (a wave for each token: a grid's threads)
  constexpr int64_t kTokensMost = ((int64_t)1 << 26) - 1;
  if (N < 0 || V < 0 || T < 1 || T > SWVR_MAX_TEACHER || N > kTokensMost || V > SWVR_EMBED_MAX || N * T > INT32_MAX)
    return fail(SWVR_EINVAL, "bad sizes N=%lld V=%lld T=%lld (T 1 to %d, N below 2^26, N T below 2^31, V at most 2^30)",
                (long long)N, (long long)V, (long long)T, SWVR_MAX_TEACHER);
  if (id64 != 0 && id64 != 1) return fail(SWVR_EINVAL, "teacher ids are int32 (0) or int64 (1), got %d", id64);
  if (ldi < 0) return fail(SWVR_EINVAL, "ldi=%lld must not be negative", (long long)ldi);
  if (N > 0 && !ids) return fail(SWVR_EINVAL, "teacher ids must be non-null");
  if (!(temperature > 0.f) || temperature > 3e38f || 1.f / temperature > 3e38f)
    return fail(SWVR_EINVAL, "temperature must be positive, and it and its reciprocal finite, got %g", (double)temperature);
  if (reduction < SWVR_REDUCE_NONE || reduction > SWVR_REDUCE_MEAN)
    return fail(SWVR_EINVAL, "unknown reduction %d", reduction);
  return SWVR_OK;
}

size_t swvr_distill_scores_size(int dtype, int w_dtype, int64_t N, int64_t K, int64_t V, int64_t ldw) {
  if (!is_dtype(dtype) || w_dtype != dtype || N <= 0 || K <= 0 || V <= 0 || ldw < K || N > INT32_MAX || V > SWVR_EMBED_MAX)
    return 0;
  return (size_t)swvr::fwd_kept_scores(dtype, N, K, V, ldw) * (size_t)V * sizeof(float);
}

size_t swvr_distill_workspace_size(int dtype, int64_t N, int64_t K, int64_t V, int64_t T, int weighted) {
  FwdPlan plan;
  if (N < 0 || V < 0 || T < 0 || !fwd_plan(dtype, N, K, V, 0, &plan, weighted != 0)) return 0;
  return up256(plan.ws_bytes) + up256((size_t)N * T * 4) + up256(swvr::distill_part_bytes(N));
}

int swvr_distill(int dtype, int h_dtype, int w_dtype, int64_t N, int64_t K, int64_t V, int64_t T, const void* h,
                 int64_t ldh, const void* W, int64_t ldw, const void* bias, int bias_dtype, float* bias_scaled,
                 float logit_scale, const void* ids, int id64, int64_t ldi, const void* teacher, int t_dtype, int64_t ldt,
                 float temperature, const float* weight, float z_loss_weight, int reduction, float* out, float* c,
                 float* lse, float* p, float* q, float* coef, float* scores, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_distill(dtype, N, V, T, id64, ids, ldi, temperature, reduction);
  if (rc != SWVR_OK) return rc;
  if (!is_dtype(t_dtype)) return fail(SWVR_EDTYPE, "unsupported teacher dtype tag %d", t_dtype);
  if (bias && !is_dtype(bias_dtype)) return fail(SWVR_EDTYPE, "unsupported bias dtype tag %d", bias_dtype);
  if (bias && !bias_scaled) return fail(SWVR_EINVAL, "bias_scaled must be non-null with a bias");
  if (bias && bias == bias_scaled && (bias_dtype != SWVR_F32 || temperature != 1.f))
    return fail(SWVR_EINVAL, "bias_scaled may be an fp32 bias itself only at temperature 1");
  if (ldt < 0) return fail(SWVR_EINVAL, "ldt=%lld must not be negative", (long long)ldt);
  if (N > 0 && (!teacher || !lse)) return fail(SWVR_EINVAL, "teacher logits and lse must be non-null");
  if ((N > 0 || reduction) && !out) return fail(SWVR_EINVAL, "out must be non-null");
  if (reduction && !c) return fail(SWVR_EINVAL, "c must be non-null");
  if ((p == nullptr) != (q == nullptr) || (p == nullptr) != (coef == nullptr))
    return fail(SWVR_EINVAL, "p, q and coef must all be given or all NULL");
  if (scores && N > 0 && swvr_distill_scores_size(dtype, w_dtype, N, K, V, ldw) == 0)
    return fail(SWVR_EINVAL, "scores are not kept for N=%lld K=%lld V=%lld ldw=%lld", (long long)N, (long long)K,
                (long long)V, (long long)ldw);
  // a forward that keeps the scores computes every token's
  const bool active = weight != nullptr && !scores;
  const size_t need = swvr_distill_workspace_size(dtype, N, K, V, T, active);
  if (!workspace || workspace_bytes < need)
    return fail(SWVR_EWORKSPACE, "distillation workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  FwdPlan plan;
  fwd_plan(dtype, N, K, V, 0, &plan, active);
  const size_t fwd_bytes = plan.ws_bytes;
  float* z = reinterpret_cast<float*>(ws + up256(fwd_bytes));
  float* part = z + up256((size_t)N * T * 4) / 4;
  const float inv_tau = 1.f / temperature, scale = logit_scale / temperature;
  hipError_t e = hipSuccess;
  if (bias && bias != bias_scaled && (e = swvr::distill_scale(bias, bias_dtype, V, inv_tau, bias_scaled, s)) != hipSuccess)
    return hip_fail(e, "bias launch");
  const float* const sb = bias ? bias_scaled : nullptr;
  // the log-sum-exps: a readout without columns
  rc = fwd_common(dtype, h_dtype, w_dtype, N, K, V, 0, h, ldh, W, ldw, W, 0, sb, scale, nullptr, lse, nullptr, nullptr,
                  workspace, fwd_bytes, stream, active, weight, scores);
  if (rc != SWVR_OK) return rc;
  swvr::DistillParams d{};
  d.h = h;
  d.ldh = ldh;
  d.W = W;
  d.ldw = ldw;
  d.h_f32 = h_dtype != dtype;
  d.w_f32 = w_dtype != dtype;
  d.bias = sb;
  d.scale = scale;
  d.inv_tau = inv_tau;
  d.N = (int)N;
  d.K = (int)K;
  d.V = (int)V;
  d.T = (int)T;
  d.ids = ids;
  d.id64 = id64;
  d.ldi = ldi;
  d.teacher = teacher;
  d.t_dtype = t_dtype;
  d.ldt = ldt;
  d.weight = weight;
  d.lse = lse;
  d.zw = z_loss_weight;
  d.reduce = reduction;
  d.z = z;
  d.out = out;
  d.p = p;
  d.q = q;
  d.coef = coef;
  e = swvr::distill_loss(dtype, d, part, c, s);
  if (e != hipSuccess) return hip_fail(e, "distillation launch");
  return SWVR_OK;
}

size_t swvr_distill_bwd_workspace_size(int dtype, int w_dtype, int64_t N, int64_t K, int64_t V, int64_t T,
                                       int64_t chunk, int need_gh) {
  BwdPlan plan;
  if (N < 0 || V < 0 || T < 0 || chunk <= 0 || !bwd_plan(dtype, N, K, V, 0, chunk, need_gh != 0, &plan, w_dtype != dtype))
    return 0;
  return up256(plan.ws_bytes) + up256((size_t)V * 4) + 5 * up256((size_t)N * T * 4) + up256((size_t)(V + 1) * 4);
}

int swvr_distill_bwd(int dtype, int h_dtype, int w_dtype, int64_t N, int64_t K, int64_t V, int64_t T, const void* h,
                     int64_t ldh, const void* W, int64_t ldw, const float* bias_scaled, float logit_scale,
                     const void* ids, int id64, int64_t ldi, float temperature, float z_loss_weight, int reduction, const float* g,
                     const float* c, const float* lse, const float* p, const float* q, const float* coef,
                     const float* scores, int64_t chunk, void* gh, int gh_dtype, void* gW, int gW_dtype, void* gb,
                     int gb_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_distill(dtype, N, V, T, id64, ids, ldi, temperature, reduction);
  if (rc != SWVR_OK) return rc;
  if (chunk <= 0) return fail(SWVR_EINVAL, "chunk must be positive, got %lld", (long long)chunk);
  if (N > 0 && (!g || !lse || !p || !q || !coef || (reduction && !c)))
    return fail(SWVR_EINVAL, "g, c, lse, p, q and coef must be non-null");
  if (gb && !bias_scaled) return fail(SWVR_EINVAL, "gb requested without a bias");
  if (scores && N > 0 && swvr_distill_scores_size(dtype, w_dtype, N, K, V, ldw) == 0)
    return fail(SWVR_EINVAL, "scores are not kept for N=%lld K=%lld V=%lld ldw=%lld", (long long)N, (long long)K,
                (long long)V, (long long)ldw);
  if (gb && !is_dtype(gb_dtype)) return fail(SWVR_EDTYPE, "unsupported gb dtype tag %d", gb_dtype);
  const size_t need = swvr_distill_bwd_workspace_size(dtype, w_dtype, N, K, V, T, chunk, gh != nullptr);
  if (!workspace || workspace_bytes < need)
    return fail(SWVR_EWORKSPACE, "distillation workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  BwdPlan plan;
  bwd_plan(dtype, N, K, V, 0, chunk, gh != nullptr, &plan, w_dtype != dtype);
  char* at = static_cast<char*>(workspace) + up256(plan.ws_bytes);
  auto take = [&](size_t bytes) {
    char* const x = at;
    at += up256(bytes);
    return x;
  };
  float* dense = reinterpret_cast<float*>(take((size_t)V * 4));
  const size_t nt = (size_t)N * T * 4;
  int* pt_id = reinterpret_cast<int*>(take(nt));
  float* pt_val = reinterpret_cast<float*>(take(nt));
  float* pt_t = reinterpret_cast<float*>(take(nt));
  int* order = reinterpret_cast<int*>(take(nt));
  int* sid = reinterpret_cast<int*>(take(nt));
  int* seg = reinterpret_cast<int*>(take((size_t)(V + 1) * 4));
  const float inv_tau = 1.f / temperature;
  hipError_t e = hipSuccess;
  if (N > 0) {
    swvr::DistillGradParams d{};
    d.N = (int)N;
    d.V = (int)V;
    d.T = (int)T;
    d.ids = ids;
    d.id64 = id64;
    d.ldi = ldi;
    d.g = g;
    d.reduce = reduction;
    d.c = c;
    d.lse = lse;
    d.p = p;
    d.q = q;
    d.coef = coef;
    d.zw = z_loss_weight;
    d.delta = reinterpret_cast<float*>(static_cast<char*>(workspace) + plan.off_delta);
    d.flag = reinterpret_cast<int*>(static_cast<char*>(workspace) + plan.off_flag);
    d.pt_id = pt_id;
    d.pt_val = pt_val;
    d.pt_t = gb ? pt_t : nullptr;
    if ((e = swvr::distill_prep(d, s)) != hipSuccess) return hip_fail(e, "distillation launch");
  }
  rc = bwd_common(dtype, h_dtype, w_dtype, N, K, V, 0, h, ldh, W, ldw, W, 0, bias_scaled, logit_scale / temperature,
                  nullptr, lse, nullptr, nullptr, chunk, gh, gh_dtype, gW, gW_dtype, nullptr, 0, gb ? dense : nullptr, workspace,
                  up256(plan.ws_bytes), stream, nullptr, 0, 0, nullptr, nullptr, 0, nullptr, pt_id, pt_val, N * T,
                  (int)T, scores, scores ? swvr::fwd_kept_scores(dtype, N, K, V, ldw) : 0);
  if (rc != SWVR_OK) return rc;
  if (gb && V > 0) {
    if ((e = swvr::sort_ids(pt_id, 0, (int)(N * T), (int)V, order, sid, seg, s)) != hipSuccess ||
        (e = swvr::distill_bias(order, seg, pt_t, dense, (int)V, inv_tau, gb, gb_dtype, s)) != hipSuccess)
      return hip_fail(e, "bias gradient launch");
  }
  return SWVR_OK;
}

// ---------------------------------------------------------------- sampling
size_t swvr_sample_workspace_size(int64_t R, int64_t V) {
  if (R < 0 || V < 1 || R > INT32_MAX || V > INT32_MAX) return 0;
  return swvr::sample_workspace_bytes(R, V);
}

int swvr_sample(int dtype, int64_t R, int64_t V, const void* logits, int64_t ld, const void* u, int u64,
                double temperature, const float* temperature_rows, int64_t top_k, const int* top_k_rows, double top_p,
                const float* top_p_rows, double min_p, const float* min_p_rows, int64_t* token, float* logprob,
                void* workspace, size_t workspace_bytes, void* stream) {
  g_err[0] = 0;
  if (!is_dtype(dtype)) return fail(SWVR_EDTYPE, "unsupported logits dtype tag %d", dtype);
  if (R < 0 || V < 1 || R > INT32_MAX || V > INT32_MAX)
    return fail(SWVR_EINVAL, "bad sizes R=%lld V=%lld", (long long)R, (long long)V);
  if (ld < 0) return fail(SWVR_EINVAL, "ld=%lld must not be negative", (long long)ld);
  if (u64 != 0 && u64 != 1) return fail(SWVR_EINVAL, "u is fp32 (0) or fp64 (1), got %d", u64);
  if (!temperature_rows && !(temperature >= 0))
    return fail(SWVR_EINVAL, "temperature must not be negative, got %g", temperature);
  if (R == 0) return SWVR_OK;
  if (!logits || !u || !token || !logprob) return fail(SWVR_EINVAL, "logits, u, token and logprob must be non-null");
  const size_t need = swvr::sample_workspace_bytes(R, V);
  if (workspace_bytes < need || (need > 0 && !workspace))
    return fail(SWVR_EWORKSPACE, "sampling workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  const uintptr_t eb = dtype == SWVR_F32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(logits) % eb) return fail(SWVR_EINVAL, "logits must be aligned to their elements");
  swvr::SampleParams p{};
  p.R = R;
  p.V = V;
  p.logits = logits;
  p.ld = ld;
  p.u = u;
  p.u64 = u64;
  p.tau = temperature;
  p.k = top_k;
  p.p = top_p;
  p.min_p = min_p;
  p.tau_rows = temperature_rows;
  p.k_rows = top_k_rows;
  p.p_rows = top_p_rows;
  p.min_p_rows = min_p_rows;
  p.token = token;
  p.logprob = logprob;
  hipError_t e = swvr::sample_launch(dtype, p, static_cast<char*>(workspace), static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "sampling launch");
  return SWVR_OK;
}

int swvr_timing_enable(int on) {
  std::lock_guard<std::mutex> lk(g_tmu);
  g_timing = on != 0;
  return SWVR_OK;
}

int swvr_timing_collect(double* total_ms, int64_t* launches, int max_kinds) {
  std::lock_guard<std::mutex> lk(g_tmu);
  std::vector<double> ms(kNumKinds, 0.0);
  std::vector<int64_t> cnt(kNumKinds, 0);
  int rc = SWVR_OK;
  for (const TimedLaunch& t : g_launches) {
    hipError_t e = hipEventSynchronize(t.stop);
    float f = 0.f;
    if (e == hipSuccess) e = hipEventElapsedTime(&f, t.start, t.stop);
    if (e != hipSuccess && rc == SWVR_OK) rc = hip_fail(e, "timing event");
    ms[t.kind] += f;
    cnt[t.kind] += 1;
    g_pool.push_back(t.start);
    g_pool.push_back(t.stop);
  }
  g_launches.clear();
  if (rc != SWVR_OK) return rc;
  const int n = max_kinds < kNumKinds ? max_kinds : kNumKinds;
  for (int k = 0; k < n; ++k) {
    if (total_ms) total_ms[k] = ms[k];
    if (launches) launches[k] = cnt[k];
  }
  return kNumKinds;
}

size_t swvr_fwd_fp8_workspace_size(int64_t N, int64_t K, int64_t V, int64_t D) {
  if (N < 0 || K < 0 || V < 0 || D < 0 || K % 16 != 0 || N > INT32_MAX || V > INT32_MAX) return 0;
  FwdPlan plan;
  if (!fwd_plan(kFwdFP8, N, K / 2, V, D, &plan)) return 0;
  return plan.ws_bytes;
}

int swvr_fwd_fp8(int64_t N, int64_t K, int64_t V, int64_t D, const void* h, int64_t ldh, const float* h_scale,
                 const void* W, int64_t ldw, const float* w_scale, const void* E, int64_t lde, const float* bias,
                 float logit_scale, float* O, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  g_err[0] = 0;
  if (D > 128) return fail(SWVR_EDTYPE, "D=%lld exceeds the maximum 128 of the e4m3 forward", (long long)D);
  if (K % 16 != 0 || ldh % 16 != 0 || ldw % 16 != 0)
    return fail(SWVR_EINVAL, "K=%lld, ldh=%lld and ldw=%lld must be multiples of 16 (e4m3 bytes)", (long long)K,
                (long long)ldh, (long long)ldw);
  // the e4m3 rows travel as bf16 rows of K / 2 elements
  int rc = check_common(SWVR_BF16, N, K / 2, V, D, h, ldh / 2, W, ldw / 2, E, lde);
  if (rc != SWVR_OK) return rc;
  if (N > 0 && (!O || !lse)) return fail(SWVR_EINVAL, "O and lse must be non-null");
  if (N > 0 && V > 0 && (!h_scale || !w_scale)) return fail(SWVR_EINVAL, "h_scale and w_scale must be non-null");
  FwdPlan plan;
  if (!fwd_plan(kFwdFP8, N, K / 2, V, D, &plan)) return fail(SWVR_EDTYPE, "no e4m3 forward kernel for D=%lld", (long long)D);
  if (N == 0) return SWVR_OK;
  if (!workspace || workspace_bytes < plan.ws_bytes)
    return fail(SWVR_EWORKSPACE, "forward workspace of %zu bytes needed, %zu given", plan.ws_bytes, workspace_bytes);
  FwdParams p{};
  p.h = h;
  p.ldh = ldh / 2;
  p.W = W;
  p.ldw = ldw / 2;
  p.E = E;
  p.lde = lde;
  p.bias = bias;
  p.scale = logit_scale;
  p.N = (int)N;
  p.K = (int)(K / 2);
  p.V = (int)V;
  p.D = (int)D;
  p.h_scale = h_scale;
  p.w_scale = w_scale;
  hipError_t e = fwd_launch(kFwdFP8, plan, p, static_cast<char*>(workspace), O, lse, nullptr, nullptr,
                            static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "forward launch");
  return SWVR_OK;
}

static int check_f64(int64_t N, int64_t K, int64_t V, int64_t D, const double* h, int64_t ldh, const double* W,
                     int64_t ldw, const double* E, int64_t lde, int64_t chunk) {
  if (N < 0 || K < 0 || V < 0 || D < 0) return fail(SWVR_EINVAL, "negative size N=%lld K=%lld V=%lld D=%lld",
                                                    (long long)N, (long long)K, (long long)V, (long long)D);
  if (N > INT32_MAX || K > INT32_MAX || V > INT32_MAX || D > SWVR_MAX_D)
    return fail(SWVR_EINVAL, "sizes must fit in 32 bits and D in SWVR_MAX_D");
  if (K >= ((int64_t)1 << 22)) return fail(SWVR_EINVAL, "K=%lld must be below 2^22", (long long)K);
  if (chunk <= 0) return fail(SWVR_EINVAL, "chunk must be positive, got %lld", (long long)chunk);
  if (ldh < K || ldw < K || lde < D) return fail(SWVR_EINVAL, "ldh, ldw must be >= K and lde >= D");
  if (N > 0 && K > 0 && !h) return fail(SWVR_EINVAL, "h must be non-null");
  if (V > 0 && K > 0 && !W) return fail(SWVR_EINVAL, "W must be non-null");
  if (V > 0 && D > 0 && !E) return fail(SWVR_EINVAL, "E must be non-null");
  return SWVR_OK;
}

size_t swvr_fwd_f64_workspace_size(int64_t N, int64_t V, int64_t D, int64_t chunk) {
  if (N < 0 || V < 0 || D < 0 || chunk <= 0) return 0;
  int64_t C;
  size_t fb;
  swvr::f64_plan(N, V, D, chunk, &C, &fb, nullptr);
  return fb;
}

int swvr_fwd_f64(int64_t N, int64_t K, int64_t V, int64_t D, const double* h, int64_t ldh, const double* W,
                 int64_t ldw, const double* E, int64_t lde, const double* bias, double logit_scale, int64_t chunk,
                 double* O, double* lse, void* workspace, size_t workspace_bytes, void* stream) {
  g_err[0] = 0;
  int rc = check_f64(N, K, V, D, h, ldh, W, ldw, E, lde, chunk);
  if (rc != SWVR_OK) return rc;
  if (N == 0) return SWVR_OK;
  if (!lse || (D > 0 && !O)) return fail(SWVR_EINVAL, "O and lse must be non-null");
  if ((rc = check_threads(std::max(256 * N, N * D))) != SWVR_OK) return rc;  // a workgroup a token, its columns
  const size_t need = swvr_fwd_f64_workspace_size(N, V, D, chunk);
  if (!workspace || workspace_bytes < need)
    return fail(SWVR_EWORKSPACE, "fp64 forward workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  swvr::F64Params p{};
  p.h = h;
  p.ldh = ldh;
  p.W = W;
  p.ldw = ldw;
  p.E = E;
  p.lde = lde;
  p.bias = bias;
  p.scale = logit_scale;
  p.N = (int)N;
  p.K = (int)K;
  p.V = (int)V;
  p.D = (int)D;
  p.chunk = chunk;
  p.O = O;
  p.lse = lse;
  p.ws = static_cast<char*>(workspace);
  hipError_t e = swvr::f64_fwd(p, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "fp64 forward launch");
  return SWVR_OK;
}

size_t swvr_bwd_f64_workspace_size(int64_t N, int64_t V, int64_t D, int64_t chunk) {
  if (N < 0 || V < 0 || D < 0 || chunk <= 0) return 0;
  int64_t C;
  size_t bb;
  swvr::f64_plan(N, V, D, chunk, &C, nullptr, &bb);
  return bb;
}

int swvr_bwd_f64(int64_t N, int64_t K, int64_t V, int64_t D, const double* h, int64_t ldh, const double* W,
                 int64_t ldw, const double* E, int64_t lde, const double* bias, double logit_scale, const double* O,
                 const double* lse, const double* gO, const double* glse, int64_t chunk, double* gh, double* gW,
                 double* gE, double* gb, void* workspace, size_t workspace_bytes, void* stream) {
  g_err[0] = 0;
  int rc = check_f64(N, K, V, D, h, ldh, W, ldw, E, lde, chunk);
  if (rc != SWVR_OK) return rc;
  if (gb && !bias) return fail(SWVR_EINVAL, "gb requested without a bias");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (N > 0 && (!lse || !glse || (D > 0 && (!O || !gO))))
    return fail(SWVR_EINVAL, "O, lse, gO and glse must be non-null");
  if ((rc = check_threads(N * std::min(chunk, V))) != SWVR_OK) return rc;  // a chunk's scores
  const size_t need = swvr_bwd_f64_workspace_size(N, V, D, chunk);
  if (N > 0 && (!workspace || workspace_bytes < need))
    return fail(SWVR_EWORKSPACE, "fp64 backward workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  swvr::F64Params p{};
  p.h = h;
  p.ldh = ldh;
  p.W = W;
  p.ldw = ldw;
  p.E = E;
  p.lde = lde;
  p.bias = bias;
  p.scale = logit_scale;
  p.N = (int)N;
  p.K = (int)K;
  p.V = (int)V;
  p.D = (int)D;
  p.chunk = chunk;
  p.O = const_cast<double*>(O);
  p.lse = const_cast<double*>(lse);
  p.gO = gO;
  p.glse = glse;
  p.gh = gh;
  p.gW = gW;
  p.gE = gE;
  p.gb = gb;
  p.ws = static_cast<char*>(workspace);
  hipError_t e = swvr::f64_bwd(p, s);
  if (e != hipSuccess) return hip_fail(e, "fp64 backward launch");
  return SWVR_OK;
}

int swvr_probe_mfma(int64_t workgroups, int64_t iters, int mode, float* out, void* stream) {
  g_err[0] = 0;
  if (workgroups < 1 || workgroups > (1 << 20) || iters < 1 || iters > (1 << 24) || mode < 0 || mode > 8)
    return fail(SWVR_EINVAL, "probe: workgroups in [1, 2^20], iters in [1, 2^24], mode 0 to 8");
  if (!out) return fail(SWVR_EINVAL, "out must be non-null");
  hipError_t e = swvr::probe_mfma((int)workgroups, (int)iters, mode, out, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "probe launch");
  return SWVR_OK;
}

size_t swvr_quantize_e4m3_workspace_size(int64_t R, int per_row) {
  if (R < 0 || R > INT32_MAX) return 0;
  return per_row ? 0 : (size_t)R * sizeof(float);
}

int swvr_quantize_e4m3(int64_t R, int64_t K, int64_t Kp, const void* x, int64_t ld, int x_dtype, int per_row,
                       void* out, int64_t ldo, float* scale, void* workspace, size_t workspace_bytes, void* stream) {
  g_err[0] = 0;
  if (R < 0 || K < 0 || Kp < K || R > INT32_MAX || Kp > INT32_MAX)
    return fail(SWVR_EINVAL, "bad sizes R=%lld K=%lld Kp=%lld", (long long)R, (long long)K, (long long)Kp);
  if (Kp % 16 != 0) return fail(SWVR_EINVAL, "Kp=%lld must be a multiple of 16", (long long)Kp);
  if (!is_dtype(x_dtype)) return fail(SWVR_EDTYPE, "unsupported input dtype tag %d", x_dtype);
  if (ld < K || ldo < Kp || ldo % 16 != 0)
    return fail(SWVR_EINVAL, "ld=%lld must be >= K, ldo=%lld >= Kp and a multiple of 16", (long long)ld,
                (long long)ldo);
  if (R == 0) return SWVR_OK;
  if ((K > 0 && !x) || !out || !scale || !aligned16(out)) return fail(SWVR_EINVAL, "x, out (16-byte aligned) and scale must be non-null");
  const size_t need = swvr_quantize_e4m3_workspace_size(R, per_row);
  if (workspace_bytes < need || (need > 0 && !workspace))
    return fail(SWVR_EWORKSPACE, "quantisation workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  swvr::QuantParams q{};
  q.x = x;
  q.ld = ld;
  q.x_dtype = x_dtype;
  q.R = (int)R;
  q.K = (int)K;
  q.Kp = (int)Kp;
  q.per_row = per_row != 0;
  q.out = out;
  q.ldo = ldo;
  q.scale = scale;
  q.amax = static_cast<float*>(workspace);
  hipError_t e = swvr::quant_launch(q, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "quantisation launch");
  return SWVR_OK;
}

size_t swvr_mse_loss_workspace_size(int64_t N) {
  if (N < 0 || N > INT32_MAX) return 0;
  return swvr::mse_workspace_bytes((int)N);
}

int swvr_mse_loss(int64_t N, int64_t D, const float* O, const float* lse, const void* target, int target_dtype,
                  int64_t ldt, const float* weight, float z_loss_weight, int reduction, float* out, float* scale,
                  float* gO, float* glse, void* workspace, size_t workspace_bytes, void* stream) {
  g_err[0] = 0;
  if (N < 0 || D < 1) return fail(SWVR_EINVAL, "bad sizes N=%lld D=%lld", (long long)N, (long long)D);
  if (N > INT32_MAX || D > INT32_MAX || N * D > ((int64_t)1 << 40)) return fail(SWVR_EINVAL, "sizes too large");
  if (const int rc = check_threads(16 * N); rc != SWVR_OK) return rc;  // 16 lanes a token
  if (!is_dtype(target_dtype)) return fail(SWVR_EDTYPE, "unsupported target dtype tag %d", target_dtype);
  if (reduction < SWVR_REDUCE_NONE || reduction > SWVR_REDUCE_MEAN)
    return fail(SWVR_EINVAL, "unknown reduction %d", reduction);
  if (ldt < D) return fail(SWVR_EINVAL, "ldt=%lld must be >= D", (long long)ldt);
  if (reduction == SWVR_REDUCE_NONE && N == 0) return SWVR_OK;  // nothing to write
  if (!out) return fail(SWVR_EINVAL, "out must be non-null");
  if ((gO == nullptr) != (glse == nullptr)) return fail(SWVR_EINVAL, "gO and glse must both be given or both NULL");
  if (N > 0 && (!O || !lse || !target)) return fail(SWVR_EINVAL, "O, lse and target must be non-null");
  const size_t need = reduction == SWVR_REDUCE_NONE ? 0 : swvr::mse_workspace_bytes((int)N);
  if (workspace_bytes < need || (need > 0 && !workspace))
    return fail(SWVR_EWORKSPACE, "loss workspace of %zu bytes needed, %zu given", need, workspace_bytes);
  swvr::MseParams p{};
  p.O = O;
  p.lse = lse;
  p.target = target;
  p.ldt = ldt;
  p.target_dtype = target_dtype;
  p.weight = weight;
  p.N = (int)N;
  p.D = (int)D;
  p.z = z_loss_weight;
  p.reduce = reduction;
  p.per_tok = reduction == SWVR_REDUCE_NONE ? out : nullptr;
  p.out = reduction == SWVR_REDUCE_NONE ? nullptr : out;
  p.scale = scale;
  p.gO = gO;
  p.glse = glse;
  hipError_t e = swvr::mse_launch(p, workspace, static_cast<hipStream_t>(stream));
  if (e != hipSuccess) return hip_fail(e, "loss launch");
  return SWVR_OK;
}

int swvr_mse_loss_noalloc(int64_t N, int64_t D, const float* O, const float* lse, const void* target,
                          int target_dtype, int64_t ldt, const float* weight, float z_loss_weight, int reduction,
                          float* out, float* scale, float* gO, float* glse, void* stream) {
  g_err[0] = 0;
  static_assert(SWVR_MSE_NOALLOC_MAX_N == swvr::kMseNoAllocMaxTokens, "one limit");
  if (N > SWVR_MSE_NOALLOC_MAX_N)
    return fail(SWVR_EINVAL, "N=%lld exceeds the maximum %d of swvr_mse_loss_noalloc (use swvr_mse_loss)",
                (long long)N, SWVR_MSE_NOALLOC_MAX_N);
  void* ws = nullptr;
  size_t ws_bytes = 0;
  if (N > 0 && reduction != SWVR_REDUCE_NONE) {
    const hipError_t e = swvr::mse_noalloc_scratch(static_cast<hipStream_t>(stream), &ws);
    if (e != hipSuccess) return hip_fail(e, "scratch address");
    ws_bytes = swvr::mse_workspace_bytes((int)N);
  }
  return swvr_mse_loss(N, D, O, lse, target, target_dtype, ldt, weight, z_loss_weight, reduction, out, scale, gO,
                       glse, ws, ws_bytes, stream);
}

const char* swvr_kernel_name(int kind) {
  if (kind < 0 || kind >= kNumKinds) return "";
  return kKindNames[kind];
}

}  // extern "C"

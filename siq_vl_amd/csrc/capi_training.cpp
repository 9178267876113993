// extern "C" boundary of the operators beside the hot path that preference and
// policy training adds: host-side validation and launches, as in capi.cpp.
#include <hip/hip_runtime.h>

#include <cmath>
#include <limits>

#include "../../include/siq_kernels.h"
#include "capi_internal.h"
#include "distill.h"
#include "flce.h"
#include "pack8.h"
#include "policy.h"
#include "token_stats.h"

using namespace siq_capi;

namespace {

// Elements per call: two vectors of eight a thread, and fewer than 2^32 threads.
constexpr int64_t kMaxNumel = int64_t(1) << 35;

int check_format(int dtype, int format) {
  if (dtype != SIQ_DTYPE_BF16 && dtype != SIQ_DTYPE_FP32)
    return fail(SIQ_ERR_INVALID_ARGUMENT, "dtype must be SIQ_DTYPE_BF16 or SIQ_DTYPE_FP32");
  if (format != SIQ_FORMAT_INT8 && format != SIQ_FORMAT_E4M3)
    return fail(SIQ_ERR_INVALID_ARGUMENT, "format must be SIQ_FORMAT_INT8 or SIQ_FORMAT_E4M3");
  return SIQ_OK;
}

int check_ptr(const void* p, const char* name) {
  if (p == nullptr) return fail(SIQ_ERR_INVALID_ARGUMENT, "%s must not be NULL", name);
  if (!aligned16(p)) return fail(SIQ_ERR_ALIGNMENT, "%s is not 16-byte aligned", name);
  return SIQ_OK;
}

int check_numel(int64_t numel) {
  if (numel < 0 || numel > kMaxNumel)
    return fail(SIQ_ERR_INVALID_ARGUMENT, "the number of elements must be in [0, 2^35] (got %lld)", (long long)numel);
  return SIQ_OK;
}

// rows x cols elements at row stride ld (elements) of tensors whose rows are
// either contiguous or start at 16-byte boundaries.
int check_rows(int64_t rows, int64_t cols, int64_t ld0, int64_t ld1, int dtype, const char* names) {
  if (rows < 0 || cols < 0) return fail(SIQ_ERR_INVALID_ARGUMENT, "rows and cols must be >= 0");
  if (cols > 0 && rows > kMaxNumel / cols)
    return fail(SIQ_ERR_INVALID_ARGUMENT, "rows * cols must be at most 2^35 (%lld x %lld)", (long long)rows,
                (long long)cols);
  const int64_t ld[2] = {ld0, ld1}, step = dtype == SIQ_DTYPE_FP32 ? 4 : 8;
  if (ld0 == cols && ld1 == cols) return SIQ_OK;
  for (int i = 0; i < 2; ++i)
    if (ld[i] < cols || ld[i] > kMaxNumel || ld[i] % step != 0)
      return fail(SIQ_ERR_ALIGNMENT, "row strides of %s must be at least cols and multiples of 16 bytes (got %lld)", names,
                  (long long)ld[i]);
  if (cols % 8 != 0)
    return fail(SIQ_ERR_UNSUPPORTED, "cols (%lld) must be a multiple of 8 where rows are not contiguous", (long long)cols);
  return SIQ_OK;
}

constexpr int64_t kMaxSeqs = int64_t(1) << 24;

int check_packed(int64_t seqs, int64_t tokens) {
  if (seqs < 1 || seqs > kMaxSeqs)
    return fail(SIQ_ERR_INVALID_ARGUMENT, "the number of sequences must be in [1, 2^24] (got %lld)", (long long)seqs);
  if (tokens < 0 || tokens >= (int64_t(1) << 31))
    return fail(SIQ_ERR_INVALID_ARGUMENT, "tokens must be in [0, 2^31) (got %lld)", (long long)tokens);
  return SIQ_OK;
}

int check_not_null(const void* p, const char* name) {
  return p == nullptr ? fail(SIQ_ERR_INVALID_ARGUMENT, "%s must not be NULL", name) : SIQ_OK;
}

int check_ws(const void* ws, size_t bytes, size_t need) {
  if (ws == nullptr || bytes < need || !aligned16(ws))
    return fail(SIQ_ERR_WORKSPACE, "workspace needs %zu bytes (16-byte aligned), got %zu", need, bytes);
  return SIQ_OK;
}

// Sizes of a log-probability call (0: fine).
int check_flp(int64_t n, int64_t hdim, int64_t vocab) {
  if (n < 0) return fail(SIQ_ERR_INVALID_ARGUMENT, "n must be >= 0");
  if (hdim <= 0 || vocab <= 0) return fail(SIQ_ERR_INVALID_ARGUMENT, "hdim and vocab must be positive");
  if (hdim % 64 != 0) return fail(SIQ_ERR_UNSUPPORTED, "hdim (%lld) must be a multiple of 64", (long long)hdim);
  if (vocab % 8 != 0) return fail(SIQ_ERR_UNSUPPORTED, "vocab (%lld) must be a multiple of 8", (long long)vocab);
  if (n >= (int64_t(1) << 31) || vocab >= (int64_t(1) << 23) || hdim >= (int64_t(1) << 20))
    return fail(SIQ_ERR_INVALID_ARGUMENT, "n must be < 2^31, vocab < 2^23 and hdim < 2^20");
  return SIQ_OK;
}

int check_flp_call(const void* hidden, const void* weight, const int64_t* labels, int64_t n, int64_t hdim,
                   int64_t vocab, double temperature, const void* saved, size_t saved_bytes) {
  int rc;
  if ((rc = check_flp(n, hdim, vocab)) || (rc = check_ptr(weight, "weight"))) return rc;
  if (!(temperature > 0.) || !std::isfinite(temperature) || !std::isfinite((float)(1.4426950408889634 / temperature)) ||
      (float)(1. / temperature) == 0.f)
    return fail(SIQ_ERR_INVALID_ARGUMENT, "temperature must be positive and finite");
  if (n > 0 && ((rc = check_ptr(hidden, "hidden")) || (rc = check_not_null(labels, "labels")))) return rc;
  if (saved != nullptr && (saved_bytes < siq::flp_saved_bytes(n, vocab) || !aligned16(saved)))
    return fail(SIQ_ERR_WORKSPACE, "saved needs %zu bytes (16-byte aligned), got %zu", siq::flp_saved_bytes(n, vocab),
                saved_bytes);
  return SIQ_OK;
}

siq::FlpArgs flp_args(const void* hidden, const void* weight, const int64_t* labels, int64_t n, int64_t hdim,
                      int64_t vocab, int64_t ignore_index, double temperature, void* saved, void* ws) {
  siq::FlpArgs a{};
  a.hidden = static_cast<const siq::bf16*>(hidden);
  a.weight = static_cast<const siq::bf16*>(weight);
  a.labels = labels;
  a.n = n;
  a.hdim = hdim;
  a.vocab = vocab;
  a.ignore_index = ignore_index;
  a.temperature = temperature;
  a.saved = saved;
  a.ws = ws;
  return a;
}

// hidden [n, hdim] and a gradient of its shape (or NULL).
int check_apart(const void* hidden, const void* dhidden, int64_t n, int64_t hdim) {
  const char *h0 = static_cast<const char*>(hidden), *d0 = static_cast<const char*>(dhidden);
  const size_t bytes = sizeof(siq::bf16) * (size_t)n * (size_t)hdim;
  if (n > 0 && dhidden != nullptr && d0 < h0 + bytes && h0 < d0 + bytes)
    return fail(SIQ_ERR_INVALID_ARGUMENT, "dhidden must not overlap hidden");
  return SIQ_OK;
}

int check_grads(const void* hidden, const void* dhidden, const void* dweight, int64_t n, int64_t hdim) {
  if (dhidden != nullptr && !aligned16(dhidden)) return fail(SIQ_ERR_ALIGNMENT, "dhidden is not 16-byte aligned");
  if (dweight != nullptr && !aligned16(dweight)) return fail(SIQ_ERR_ALIGNMENT, "dweight is not 16-byte aligned");
  return check_apart(hidden, dhidden, n, hdim);
}

int check_saved(const void* saved, size_t bytes, size_t need) {
  if (saved != nullptr && (bytes < need || !aligned16(saved)))
    return fail(SIQ_ERR_WORKSPACE, "saved needs %zu bytes (16-byte aligned), got %zu", need, bytes);
  return SIQ_OK;
}

// Alternatives of a row: at least `least`.
int check_top_k(int top_k, int least, int64_t vocab) {
  if (top_k < least || top_k > siq::kMaxTopK || top_k > vocab)
    return fail(SIQ_ERR_INVALID_ARGUMENT, "top_k must be in [%d, %d] and at most the vocabulary's %lld (got %d)", least,
                siq::kMaxTopK, (long long)vocab, top_k);
  return SIQ_OK;
}

int launched(hipError_t e, const char* what) {
  return e == hipSuccess ? ok() : fail(SIQ_ERR_LAUNCH, "%s launch failed: %s", what, hipGetErrorString(e));
}

}  // namespace

extern "C" {

int siq_pack8(const void* x, int64_t numel, int dtype, int format, void* codes, void* scales, void* stream) {
  int rc;
  if ((rc = check_format(dtype, format)) || (rc = check_numel(numel))) return rc;
  if (numel == 0) return ok();
  if ((rc = check_ptr(x, "x")) || (rc = check_ptr(codes, "codes")) || (rc = check_ptr(scales, "scales"))) return rc;
  return launched(siq::launch_pack8(x, numel, dtype == SIQ_DTYPE_FP32, format == SIQ_FORMAT_E4M3,
                                    static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales),
                                    static_cast<hipStream_t>(stream)),
                  "pack8");
}

int siq_unpack8(const void* codes, const void* scales, int64_t numel, int dtype, int format, void* x, void* stream) {
  int rc;
  if ((rc = check_format(dtype, format)) || (rc = check_numel(numel))) return rc;
  if (numel == 0) return ok();
  if ((rc = check_ptr(x, "x")) || (rc = check_ptr(codes, "codes")) || (rc = check_ptr(scales, "scales"))) return rc;
  return launched(siq::launch_unpack8(static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), numel,
                                      dtype == SIQ_DTYPE_FP32, format == SIQ_FORMAT_E4M3, x,
                                      static_cast<hipStream_t>(stream)),
                  "unpack8");
}

int siq_swiglu8_fwd(const void* gate, const void* up, int64_t rows, int64_t cols, int64_t gate_stride,
                    int64_t up_stride, int dtype, int format, void* h, void* gate_codes, void* gate_scales,
                    void* up_codes, void* up_scales, void* stream) {
  int rc;
  if ((rc = check_format(dtype, format)) || (rc = check_rows(rows, cols, gate_stride, up_stride, dtype, "gate / up")))
    return rc;
  if (rows * cols == 0) return ok();
  if ((rc = check_ptr(gate, "gate")) || (rc = check_ptr(up, "up")) || (rc = check_ptr(h, "h"))) return rc;
  if (gate_codes != nullptr || gate_scales != nullptr || up_codes != nullptr || up_scales != nullptr)
    if ((rc = check_ptr(gate_codes, "gate_codes")) || (rc = check_ptr(gate_scales, "gate_scales")) ||
        (rc = check_ptr(up_codes, "up_codes")) || (rc = check_ptr(up_scales, "up_scales")))
      return rc;
  siq::SwigluArgs a{};
  a.gate = gate;
  a.up = up;
  a.h = h;
  a.gcodes = static_cast<uint8_t*>(gate_codes);
  a.gscales = static_cast<uint8_t*>(gate_scales);
  a.ucodes = static_cast<uint8_t*>(up_codes);
  a.uscales = static_cast<uint8_t*>(up_scales);
  a.rows = rows;
  a.cols = cols;
  a.ld0 = gate_stride;
  a.ld1 = up_stride;
  a.f32 = dtype == SIQ_DTYPE_FP32;
  a.e4m3 = format == SIQ_FORMAT_E4M3;
  return launched(siq::launch_swiglu8_fwd(a, static_cast<hipStream_t>(stream)), "swiglu8 forward");
}

int siq_swiglu8_bwd(const void* dh, const void* gate_codes, const void* gate_scales, const void* up_codes,
                    const void* up_scales, int64_t rows, int64_t cols, int64_t dgate_stride, int64_t dup_stride,
                    int dtype, int format, void* dgate, void* dup, void* h, void* stream) {
  int rc;
  if ((rc = check_format(dtype, format)) ||
      (rc = check_rows(rows, cols, dgate_stride, dup_stride, dtype, "dgate / dup")))
    return rc;
  if (rows * cols == 0) return ok();
  if ((rc = check_ptr(dh, "dh")) || (rc = check_ptr(dgate, "dgate")) || (rc = check_ptr(dup, "dup")) ||
      (rc = check_ptr(gate_codes, "gate_codes")) || (rc = check_ptr(gate_scales, "gate_scales")) ||
      (rc = check_ptr(up_codes, "up_codes")) || (rc = check_ptr(up_scales, "up_scales")))
    return rc;
  if (h != nullptr && (rc = check_ptr(h, "h"))) return rc;
  siq::SwigluArgs a{};
  a.dh = dh;
  a.h = h;
  a.dgate = dgate;
  a.dup = dup;
  a.gcodes = static_cast<uint8_t*>(const_cast<void*>(gate_codes));
  a.gscales = static_cast<uint8_t*>(const_cast<void*>(gate_scales));
  a.ucodes = static_cast<uint8_t*>(const_cast<void*>(up_codes));
  a.uscales = static_cast<uint8_t*>(const_cast<void*>(up_scales));
  a.rows = rows;
  a.cols = cols;
  a.ld0 = dgate_stride;
  a.ld1 = dup_stride;
  a.f32 = dtype == SIQ_DTYPE_FP32;
  a.e4m3 = format == SIQ_FORMAT_E4M3;
  return launched(siq::launch_swiglu8_bwd(a, static_cast<hipStream_t>(stream)), "swiglu8 backward");
}

size_t siq_pref_workspace_bytes(int64_t pairs, int64_t tokens) {
  if (pairs < 1 || pairs > kMaxSeqs / 2 || tokens < 0 || tokens >= (int64_t(1) << 31)) return 0;
  return siq::pref_workspace_bytes(pairs, tokens);
}

int siq_pref_fwd(const float* policy, const float* reference, const void* mask, const int32_t* cu_seqlens,
                 int64_t pairs, int64_t tokens, int loss_type, int order, double beta, double label_smoothing,
                 int length_normalized, const float* divisor, float* loss, float* chosen_rewards,
                 float* rejected_rewards, float* coef, void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  if (pairs < 1 || pairs > kMaxSeqs / 2)
    return fail(SIQ_ERR_INVALID_ARGUMENT, "pairs must be in [1, 2^23] (got %lld)", (long long)pairs);
  if ((rc = check_packed(2 * pairs, tokens))) return rc;
  if (loss_type < SIQ_PREF_SIGMOID || loss_type > SIQ_PREF_HINGE)
    return fail(SIQ_ERR_INVALID_ARGUMENT, "loss_type must be SIQ_PREF_SIGMOID, _IPO or _HINGE");
  if (order != SIQ_ORDER_INTERLEAVED && order != SIQ_ORDER_HALVES)
    return fail(SIQ_ERR_INVALID_ARGUMENT, "order must be SIQ_ORDER_INTERLEAVED or SIQ_ORDER_HALVES");
  if (!(beta > 0.) || !std::isfinite(beta)) return fail(SIQ_ERR_INVALID_ARGUMENT, "beta must be positive and finite");
  if (!(label_smoothing >= 0. && label_smoothing <= 0.5))
    return fail(SIQ_ERR_INVALID_ARGUMENT, "label_smoothing must be in [0, 0.5]");
  if (label_smoothing != 0. && loss_type != SIQ_PREF_SIGMOID)
    return fail(SIQ_ERR_UNSUPPORTED, "label_smoothing goes with SIQ_PREF_SIGMOID only");
  if ((rc = check_not_null(cu_seqlens, "cu_seqlens")) || (rc = check_not_null(loss, "loss")) ||
      (rc = check_not_null(chosen_rewards, "chosen_rewards")) ||
      (rc = check_not_null(rejected_rewards, "rejected_rewards")) || (rc = check_not_null(coef, "coef")))
    return rc;
  if (tokens > 0 && (rc = check_not_null(policy, "policy"))) return rc;
  if ((rc = check_ws(workspace, workspace_bytes, siq::pref_workspace_bytes(pairs, tokens)))) return rc;
  siq::PrefArgs a{};
  a.seq = {cu_seqlens, 2 * pairs, tokens};
  a.policy = policy;
  a.reference = reference;
  a.mask = static_cast<const uint8_t*>(mask);
  a.pairs = pairs;
  a.type = loss_type;
  a.halves = order == SIQ_ORDER_HALVES;
  a.normalized = length_normalized != 0;
  a.beta = beta;
  a.smoothing = label_smoothing;
  a.divisor = divisor;
  a.loss = loss;
  a.chosen = chosen_rewards;
  a.rejected = rejected_rewards;
  a.coef = coef;
  a.ws = workspace;
  return launched(siq::pref_fwd(a, static_cast<hipStream_t>(stream)), "preference loss");
}

int siq_pref_bwd(const float* grad_loss, const float* coef, const void* mask, const int32_t* cu_seqlens, int64_t pairs,
                 int64_t tokens, float* dpolicy, void* stream) {
  int rc;
  if (pairs < 1 || pairs > kMaxSeqs / 2)
    return fail(SIQ_ERR_INVALID_ARGUMENT, "pairs must be in [1, 2^23] (got %lld)", (long long)pairs);
  if ((rc = check_packed(2 * pairs, tokens))) return rc;
  if (tokens == 0) return ok();
  if ((rc = check_not_null(grad_loss, "grad_loss")) || (rc = check_not_null(coef, "coef")) ||
      (rc = check_not_null(cu_seqlens, "cu_seqlens")) || (rc = check_not_null(dpolicy, "dpolicy")))
    return rc;
  return launched(siq::pref_bwd({cu_seqlens, 2 * pairs, tokens}, grad_loss, coef, static_cast<const uint8_t*>(mask),
                                dpolicy, static_cast<hipStream_t>(stream)),
                  "preference loss backward");
}

size_t siq_policy_workspace_bytes(int64_t seqs, int64_t tokens) {
  if (seqs < 1 || seqs > kMaxSeqs || tokens < 0 || tokens >= (int64_t(1) << 31)) return 0;
  return siq::policy_workspace_bytes(seqs, tokens);
}

int siq_policy_fwd(const float* logps, const float* old_logps, const float* advantages, const void* mask,
                   const float* reference, const int32_t* cu_seqlens, int64_t seqs, int64_t tokens,
                   int advantage_per_token, int aggregation, int kl_type, double clip_low, double clip_high,
                   double dual_clip, double kl_coef, const float* divisor, float* loss, float* mean_kl,
                   float* clip_fraction, float* dtoken, float* weight, void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  if ((rc = check_packed(seqs, tokens))) return rc;
  if (aggregation != SIQ_AGG_TOKEN && aggregation != SIQ_AGG_SEQUENCE)
    return fail(SIQ_ERR_INVALID_ARGUMENT, "aggregation must be SIQ_AGG_TOKEN or SIQ_AGG_SEQUENCE");
  if (kl_type < SIQ_KL_K1 || kl_type > SIQ_KL_K3)
    return fail(SIQ_ERR_INVALID_ARGUMENT, "kl_type must be SIQ_KL_K1, _K2 or _K3");
  if (!(clip_low >= 0. && clip_low <= 1.)) return fail(SIQ_ERR_INVALID_ARGUMENT, "clip_low must be in [0, 1]");
  if (!(clip_high >= 0.)) return fail(SIQ_ERR_INVALID_ARGUMENT, "clip_high must be >= 0");
  if (!(dual_clip == 0. || dual_clip > 1.))
    return fail(SIQ_ERR_INVALID_ARGUMENT, "dual_clip must be 0 (none) or above 1");
  if (!std::isfinite(kl_coef)) return fail(SIQ_ERR_INVALID_ARGUMENT, "kl_coef must be finite");
  if (kl_coef != 0. && reference == nullptr && tokens > 0)
    return fail(SIQ_ERR_INVALID_ARGUMENT, "a KL term needs the reference's log-probabilities");
  if (cu_seqlens == nullptr && seqs != 1)
    return fail(SIQ_ERR_INVALID_ARGUMENT, "without cu_seqlens there is one sequence");
  if ((rc = check_not_null(loss, "loss")) || (rc = check_not_null(mean_kl, "mean_kl")) ||
      (rc = check_not_null(clip_fraction, "clip_fraction")) || (rc = check_not_null(weight, "weight")))
    return rc;
  if (tokens > 0) {
    if ((rc = check_not_null(logps, "logps")) || (rc = check_not_null(old_logps, "old_logps")) ||
        (rc = check_not_null(advantages, "advantages")) || (rc = check_ptr(dtoken, "dtoken")))
      return rc;
  }
  if ((rc = check_ws(workspace, workspace_bytes, siq::policy_workspace_bytes(seqs, tokens)))) return rc;
  siq::PolicyArgs a{};
  a.seq = {cu_seqlens, seqs, tokens};
  a.logps = logps;
  a.old = old_logps;
  a.advantages = advantages;
  a.mask = static_cast<const uint8_t*>(mask);
  a.reference = reference;
  a.per_token = advantage_per_token != 0;
  a.by_sequence = aggregation == SIQ_AGG_SEQUENCE;
  a.kl = reference == nullptr ? siq::kKlNone : kl_type;
  a.log_low = std::log1p(-clip_low);
  a.log_high = std::log1p(clip_high);
  a.log_dual = dual_clip == 0. ? std::numeric_limits<double>::infinity() : std::log(dual_clip);
  a.low = (float)(1. - clip_low);
  a.high = (float)(1. + clip_high);
  a.dual = (float)dual_clip;
  a.kl_coef = (float)kl_coef;
  a.divisor = divisor;
  a.loss = loss;
  a.mean_kl = mean_kl;
  a.clip_fraction = clip_fraction;
  a.dtoken = dtoken;
  a.weight = weight;
  a.ws = workspace;
  return launched(siq::policy_fwd(a, static_cast<hipStream_t>(stream)), "policy loss");
}

int siq_policy_bwd(const float* grad_loss, const float* dtoken, const float* weight, const int32_t* cu_seqlens,
                   int64_t seqs, int64_t tokens, int aggregation, float* dlogps, void* stream) {
  int rc;
  if ((rc = check_packed(seqs, tokens))) return rc;
  if (aggregation != SIQ_AGG_TOKEN && aggregation != SIQ_AGG_SEQUENCE)
    return fail(SIQ_ERR_INVALID_ARGUMENT, "aggregation must be SIQ_AGG_TOKEN or SIQ_AGG_SEQUENCE");
  if (cu_seqlens == nullptr && seqs != 1)
    return fail(SIQ_ERR_INVALID_ARGUMENT, "without cu_seqlens there is one sequence");
  if (tokens == 0) return ok();
  if ((rc = check_not_null(grad_loss, "grad_loss")) || (rc = check_not_null(weight, "weight")) ||
      (rc = check_ptr(dtoken, "dtoken")) || (rc = check_ptr(dlogps, "dlogps")))
    return rc;
  return launched(siq::policy_bwd({cu_seqlens, seqs, tokens}, aggregation == SIQ_AGG_SEQUENCE, grad_loss, dtoken, weight,
                                  dlogps, static_cast<hipStream_t>(stream)),
                  "policy loss backward");
}

size_t siq_flp_saved_bytes(int64_t n, int64_t vocab) {
  if (n < 0 || vocab <= 0) return 0;
  return siq::flp_saved_bytes(n, vocab);
}

size_t siq_flp_fwd_workspace_bytes(int64_t n, int64_t hdim, int64_t vocab, int keep) {
  if (n < 0 || hdim <= 0 || vocab <= 0) return 0;
  return siq::flp_fwd_workspace_bytes(n, hdim, vocab, keep != 0);
}

size_t siq_flp_bwd_workspace_bytes(int64_t n, int64_t hdim, int64_t vocab, int64_t chunk_tokens, int need_dweight,
                                   int have_saved) {
  if (n < 0 || hdim <= 0 || vocab <= 0 || chunk_tokens <= 0) return 0;
  return siq::flp_bwd_workspace_bytes(n, hdim, vocab, chunk_tokens, need_dweight != 0, have_saved != 0);
}

int siq_flp_fwd(const void* hidden, const void* weight, const int64_t* labels, int64_t n, int64_t hdim, int64_t vocab,
                int64_t ignore_index, double temperature, float* logp, int64_t* count, int64_t* bad_labels, void* saved,
                size_t saved_bytes, void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  if ((rc = check_flp_call(hidden, weight, labels, n, hdim, vocab, temperature, saved, saved_bytes)) ||
      (rc = check_not_null(count, "count")) || (rc = check_not_null(bad_labels, "bad_labels")))
    return rc;
  if (n > 0 && (rc = check_not_null(logp, "logp"))) return rc;
  if ((rc = check_ws(workspace, workspace_bytes, siq::flp_fwd_workspace_bytes(n, hdim, vocab, saved != nullptr)))) return rc;
  siq::FlpArgs a = flp_args(hidden, weight, labels, n, hdim, vocab, ignore_index, temperature, saved, workspace);
  a.logp = logp;
  a.count = count;
  a.bad_labels = bad_labels;
  return launched(siq::flp_fwd(a, static_cast<hipStream_t>(stream)), "log-probabilities");
}

int siq_flp_bwd(const void* hidden, const void* weight, const int64_t* labels, const float* dlogp, int64_t n,
                int64_t hdim, int64_t vocab, int64_t ignore_index, double temperature, const void* saved,
                size_t saved_bytes, void* dhidden, void* dweight, int64_t chunk_tokens, void* workspace,
                size_t workspace_bytes, void* stream) {
  int rc;
  if ((rc = check_flp_call(hidden, weight, labels, n, hdim, vocab, temperature, saved, saved_bytes))) return rc;
  if (chunk_tokens <= 0) return fail(SIQ_ERR_INVALID_ARGUMENT, "chunk_tokens must be positive");
  if (n > 0 && (rc = check_not_null(dlogp, "dlogp"))) return rc;
  if (dhidden != nullptr && !aligned16(dhidden)) return fail(SIQ_ERR_ALIGNMENT, "dhidden is not 16-byte aligned");
  if (dweight != nullptr && !aligned16(dweight)) return fail(SIQ_ERR_ALIGNMENT, "dweight is not 16-byte aligned");
  if (dhidden == nullptr && dweight == nullptr) return ok();
  if ((rc = check_apart(hidden, dhidden, n, hdim))) return rc;
  const size_t need = siq::flp_bwd_workspace_bytes(n, hdim, vocab, chunk_tokens, dweight != nullptr, saved != nullptr);
  if ((rc = check_ws(workspace, workspace_bytes, need))) return rc;
  siq::FlpArgs a = flp_args(hidden, weight, labels, n, hdim, vocab, ignore_index, temperature, const_cast<void*>(saved),
                            workspace);
  a.dlogp = dlogp;
  a.dhidden = static_cast<siq::bf16*>(dhidden);
  a.dweight = static_cast<siq::bf16*>(dweight);
  a.chunk = chunk_tokens;
  return launched(siq::flp_bwd(a, static_cast<hipStream_t>(stream)), "log-probabilities backward");
}

size_t siq_stats_saved_bytes(int64_t n, int64_t vocab) {
  if (n < 0 || vocab <= 0) return 0;
  return siq::stats_saved_bytes(n, vocab);
}

size_t siq_stats_fwd_workspace_bytes(int64_t n, int64_t hdim, int64_t vocab, int top_k, int keep) {
  if (n < 0 || hdim <= 0 || vocab <= 0 || top_k < 0 || top_k > siq::kMaxTopK) return 0;
  return siq::stats_fwd_workspace_bytes(n, hdim, vocab, top_k, keep != 0);
}

size_t siq_stats_bwd_workspace_bytes(int64_t n, int64_t hdim, int64_t vocab, int64_t chunk_tokens, int need_dweight,
                                     int have_saved) {
  if (n < 0 || hdim <= 0 || vocab <= 0 || chunk_tokens <= 0) return 0;
  return siq::stats_bwd_workspace_bytes(n, hdim, vocab, chunk_tokens, need_dweight != 0, have_saved != 0);
}

int siq_stats_fwd(const void* hidden, const void* weight, const int64_t* labels, int64_t n, int64_t hdim,
                  int64_t vocab, int64_t ignore_index, double temperature, int top_k, float* logp, float* entropy,
                  float* state, float* top_logp, int64_t* top_ids, int64_t* count, int64_t* bad_labels, void* saved,
                  size_t saved_bytes, void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  if ((rc = check_flp_call(hidden, weight, labels, n, hdim, vocab, temperature, nullptr, 0)) ||
      (rc = check_saved(saved, saved_bytes, siq::stats_saved_bytes(n, vocab))) || (rc = check_top_k(top_k, 0, vocab)) ||
      (rc = check_not_null(count, "count")) || (rc = check_not_null(bad_labels, "bad_labels")))
    return rc;
  if (n > 0 && ((rc = check_not_null(logp, "logp")) || (rc = check_not_null(entropy, "entropy")))) return rc;
  if (n > 0 && top_k > 0 && ((rc = check_not_null(top_logp, "top_logp")) || (rc = check_not_null(top_ids, "top_ids"))))
    return rc;
  if ((rc = check_ws(workspace, workspace_bytes,
                     siq::stats_fwd_workspace_bytes(n, hdim, vocab, top_k, saved != nullptr))))
    return rc;
  siq::StatsArgs a{};
  a.hidden = static_cast<const siq::bf16*>(hidden);
  a.weight = static_cast<const siq::bf16*>(weight);
  a.labels = labels;
  a.n = n;
  a.hdim = hdim;
  a.vocab = vocab;
  a.ignore_index = ignore_index;
  a.temperature = temperature;
  a.top_k = top_k;
  a.logp = logp;
  a.entropy = entropy;
  a.state = state;
  a.top_logp = top_logp;
  a.top_ids = top_ids;
  a.count = count;
  a.bad_labels = bad_labels;
  a.saved = saved;
  a.ws = workspace;
  return launched(siq::stats_fwd(a, static_cast<hipStream_t>(stream)), "token statistics");
}

int siq_stats_bwd(const void* hidden, const void* weight, const int64_t* labels, const float* state,
                  const float* dlogp, const float* dentropy, int64_t n, int64_t hdim, int64_t vocab,
                  int64_t ignore_index, double temperature, const void* saved, size_t saved_bytes, void* dhidden,
                  void* dweight, int64_t chunk_tokens, void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  if ((rc = check_flp_call(hidden, weight, labels, n, hdim, vocab, temperature, nullptr, 0)) ||
      (rc = check_saved(saved, saved_bytes, siq::stats_saved_bytes(n, vocab))))
    return rc;
  if (chunk_tokens <= 0) return fail(SIQ_ERR_INVALID_ARGUMENT, "chunk_tokens must be positive");
  if (n > 0 && (rc = check_not_null(state, "state"))) return rc;
  if ((rc = check_grads(hidden, dhidden, dweight, n, hdim))) return rc;
  if (dhidden == nullptr && dweight == nullptr) return ok();
  if ((rc = check_ws(workspace, workspace_bytes,
                     siq::stats_bwd_workspace_bytes(n, hdim, vocab, chunk_tokens, dweight != nullptr, saved != nullptr))))
    return rc;
  siq::StatsArgs a{};
  a.hidden = static_cast<const siq::bf16*>(hidden);
  a.weight = static_cast<const siq::bf16*>(weight);
  a.labels = labels;
  a.n = n;
  a.hdim = hdim;
  a.vocab = vocab;
  a.ignore_index = ignore_index;
  a.temperature = temperature;
  a.state = const_cast<float*>(state);
  a.dlogp = dlogp;
  a.dentropy = dentropy;
  a.saved = const_cast<void*>(saved);
  a.dhidden = static_cast<siq::bf16*>(dhidden);
  a.dweight = static_cast<siq::bf16*>(dweight);
  a.chunk = chunk_tokens;
  a.ws = workspace;
  return launched(siq::stats_bwd(a, static_cast<hipStream_t>(stream)), "token statistics backward");
}

size_t siq_distill_workspace_bytes(int64_t n, int64_t hdim, int64_t vocab, int top_k, int64_t chunk_tokens,
                                   int need_grads, int need_dweight) {
  if (n < 0 || hdim <= 0 || vocab <= 0 || chunk_tokens <= 0 || top_k < 1 || top_k > siq::kMaxTeacher) return 0;
  return siq::distill_workspace_bytes(n, hdim, vocab, top_k, chunk_tokens, need_grads != 0, need_dweight != 0);
}

int siq_distill(const void* hidden, const void* weight, const int64_t* labels, const void* ids, int ids_bytes,
                const float* teacher, int64_t n, int64_t hdim, int64_t vocab, int top_k, int64_t ignore_index,
                double temperature, double ce_weight, int divergence, int tail, const float* divisor, float* loss,
                float* mean_divergence, float* mean_cross_entropy, int64_t* counts, void* dhidden, void* dweight,
                int64_t chunk_tokens, void* workspace, size_t workspace_bytes, void* stream) {
  int rc;
  if ((rc = check_flp_call(hidden, weight, labels, n, hdim, vocab, temperature, nullptr, 0)) ||
      (rc = check_top_k(top_k, 1, vocab)))
    return rc;
  if (ids_bytes != 4 && ids_bytes != 8)
    return fail(SIQ_ERR_INVALID_ARGUMENT, "ids_bytes must be 8 (int64) or 4 (int32), got %d", ids_bytes);
  if (divergence != SIQ_DIVERGENCE_FORWARD && divergence != SIQ_DIVERGENCE_REVERSE)
    return fail(SIQ_ERR_INVALID_ARGUMENT, "divergence must be SIQ_DIVERGENCE_FORWARD or _REVERSE");
  if (divergence == SIQ_DIVERGENCE_REVERSE && !tail)
    return fail(SIQ_ERR_UNSUPPORTED, "the reverse divergence needs the tail: without it, it has no least value");
  if (!(ce_weight >= 0. && ce_weight <= 1.)) return fail(SIQ_ERR_INVALID_ARGUMENT, "ce_weight must be in [0, 1]");
  if (ce_weight != 0. && temperature != 1.)
    return fail(SIQ_ERR_UNSUPPORTED, "ce_weight goes with temperature 1 only: labels are not softened");
  if (n > 0 && ((rc = check_not_null(ids, "ids")) || (rc = check_not_null(teacher, "teacher")))) return rc;
  if ((rc = check_not_null(loss, "loss")) || (rc = check_not_null(mean_divergence, "mean_divergence")) ||
      (rc = check_not_null(mean_cross_entropy, "mean_cross_entropy")) || (rc = check_not_null(counts, "counts")))
    return rc;
  if (chunk_tokens <= 0) return fail(SIQ_ERR_INVALID_ARGUMENT, "chunk_tokens must be positive");
  if ((rc = check_grads(hidden, dhidden, dweight, n, hdim))) return rc;
  siq::DistillArgs a{};
  a.grads = dhidden != nullptr || dweight != nullptr;
  if ((rc = check_ws(workspace, workspace_bytes,
                     siq::distill_workspace_bytes(n, hdim, vocab, top_k, chunk_tokens, a.grads, dweight != nullptr))))
    return rc;
  a.hidden = static_cast<const siq::bf16*>(hidden);
  a.weight = static_cast<const siq::bf16*>(weight);
  a.labels = labels;
  a.ids = ids;
  a.teacher = teacher;
  a.n = n;
  a.hdim = hdim;
  a.vocab = vocab;
  a.ignore_index = ignore_index;
  a.top_k = top_k;
  a.ids32 = ids_bytes == 4;
  a.reverse = divergence == SIQ_DIVERGENCE_REVERSE;
  a.tail = tail != 0;
  a.temperature = temperature;
  a.ce_weight = ce_weight;
  a.reduction = divisor != nullptr;
  a.divisor = divisor;
  a.loss = loss;
  a.divergence = mean_divergence;
  a.cross_entropy = mean_cross_entropy;
  a.counts = counts;
  a.dhidden = static_cast<siq::bf16*>(dhidden);
  a.dweight = static_cast<siq::bf16*>(dweight);
  a.chunk = chunk_tokens;
  a.ws = workspace;
  return launched(siq::distill_run(a, static_cast<hipStream_t>(stream)), "distillation");
}

}  // extern "C"

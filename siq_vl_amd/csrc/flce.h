// Internal interface of the fused linear cross-entropy kernels.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"

namespace siq {

struct FlceArgs {
  const bf16* hidden;   // [n, hdim]
  const bf16* weight;   // [vocab, hdim]
  const int64_t* labels;
  int64_t n, hdim, vocab, ignore_index;
  int reduction;        // 0 mean over valid rows, 1 sum / *divisor
  const float* divisor;
  float* loss;
  int64_t* count;
  int64_t* bad_labels;
  bool grads;           // false: loss only (dhidden and dweight unused)
  bf16* dhidden;        // [n, hdim]
  bf16* dweight;        // [vocab, hdim] or nullptr
  int64_t chunk;        // tokens per logits chunk
  void* ws;
};

// Log-probabilities of the labels and their gradients.
struct FlpArgs {
  const bf16* hidden;   // [n, hdim]
  const bf16* weight;   // [vocab, hdim]
  const int64_t* labels;
  int64_t n, hdim, vocab, ignore_index;
  double temperature;
  void* saved;          // forward: kept for the backward, or nullptr; backward: what was kept, or nullptr
  float* logp;          // forward: [n]
  int64_t* count;
  int64_t* bad_labels;
  const float* dlogp;   // backward: [n]
  bf16* dhidden;        // [n, hdim] or nullptr
  bf16* dweight;        // [vocab, hdim] or nullptr
  int64_t chunk;        // tokens per logits chunk (backward without saved)
  void* ws;
};

size_t flp_saved_bytes(int64_t n, int64_t vocab);
size_t flp_fwd_workspace_bytes(int64_t n, int64_t hdim, int64_t vocab, bool keep);
size_t flp_bwd_workspace_bytes(int64_t n, int64_t hdim, int64_t vocab, int64_t chunk, bool need_dw, bool have_saved);
hipError_t flp_fwd(const FlpArgs& a, hipStream_t stream);
hipError_t flp_bwd(const FlpArgs& a, hipStream_t stream);

size_t flce_workspace_bytes(int64_t n, int64_t hdim, int64_t vocab, int64_t chunk, bool need_dh, bool need_dw);
hipError_t flce_run(const FlceArgs& a, hipStream_t stream);
hipError_t launch_scale_bf16(const bf16* src, bf16* dst, int64_t numel, const float* scalar, hipStream_t stream);
hipError_t launch_scale2_bf16(const bf16* x0, bf16* y0, int64_t n0, const bf16* x1, bf16* y1, int64_t n1,
                              const float* scalar, hipStream_t stream);

}  // namespace siq

// Internal interface of the token statistics: log-probabilities of given tokens,
// entropies and most probable tokens, and the gradients of the first two.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"

namespace siq {

constexpr int kMaxTopK = 128;

struct StatsArgs {
  const bf16* hidden;   // [n, hdim]
  const bf16* weight;   // [vocab, hdim]
  const int64_t* labels;
  int64_t n, hdim, vocab, ignore_index;
  double temperature;
  int top_k;
  float* logp;          // [n]
  float* entropy;       // [n]
  float* state;         // [3, n] (or nullptr: no backward follows) log2 of the sum of exp(z / temperature), logp and entropy
  float* top_logp;      // [n, top_k]
  int64_t* top_ids;     // [n, top_k]
  int64_t* count;
  int64_t* bad_labels;
  const float* dlogp;     // backward: [n] or nullptr: 0
  const float* dentropy;  // [n] or nullptr: 0
  bf16* dhidden;          // [n, hdim] or nullptr
  bf16* dweight;          // [vocab, hdim] or nullptr
  int64_t chunk;          // tokens per chunk of the backward
  void* saved;            // forward: kept for the backward, or nullptr; backward: what was kept, or nullptr
  void* ws;
};

size_t stats_saved_bytes(int64_t n, int64_t vocab);
size_t stats_fwd_workspace_bytes(int64_t n, int64_t hdim, int64_t vocab, int top_k, bool keep);
size_t stats_bwd_workspace_bytes(int64_t n, int64_t hdim, int64_t vocab, int64_t chunk, bool need_dw, bool have_saved);
hipError_t stats_fwd(const StatsArgs& a, hipStream_t stream);
hipError_t stats_bwd(const StatsArgs& a, hipStream_t stream);

}  // namespace siq

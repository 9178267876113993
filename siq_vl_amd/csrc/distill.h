// Internal interface of the distillation loss.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"

namespace siq {

constexpr int kMaxTeacher = 128;  // a teacher's tokens a row

struct DistillArgs {
  const bf16* hidden;   // [n, hdim]
  const bf16* weight;   // [vocab, hdim]
  const int64_t* labels;
  const void* ids;      // [n, top_k] int64 or int32
  const float* teacher; // [n, top_k] log-probabilities
  int64_t n, hdim, vocab, ignore_index;
  int top_k;
  bool ids32, reverse, tail;
  double temperature, ce_weight;
  int reduction;        // 0 mean over counted rows, 1 sum / *divisor
  const float* divisor;
  float *loss, *divergence, *cross_entropy;
  int64_t* counts;      // [3]: rows that count, bad labels, bad tokens of the teacher
  bool grads;
  bf16* dhidden;        // [n, hdim] or nullptr
  bf16* dweight;        // [vocab, hdim] or nullptr
  int64_t chunk;        // tokens per logits chunk
  void* ws;
};

size_t distill_workspace_bytes(int64_t n, int64_t hdim, int64_t vocab, int top_k, int64_t chunk, bool grads, bool need_dw);
hipError_t distill_run(const DistillArgs& a, hipStream_t stream);

}  // namespace siq

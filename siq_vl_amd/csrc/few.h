// Products of few rows with the lm_head's table: staging and the pipeline of their
// k-steps, for the kernels whose tiles have 32 NB rows of the call.
#pragma once
#include "gemm.h"

namespace siq {
namespace gemm {

// One k-step's loads of an operand with k contiguous: ROWS rows x 64 k (swizzled
// as gemm.h's KC halves), 8 rows an instruction, dealt over NWV waves.
template <int ROWS, int NWV>
struct FewRows {
  static constexpr int PER = ROWS / 8 / NWV;
  uint32_t off[PER];
  __device__ __forceinline__ void init(int64_t ld, int64_t last, int lane, int w) {
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      const int r = 8 * (PER * w + q) + lane / 8;
      off[q] = 2 * (uint32_t)(min((int64_t)r, last) * ld + 8 * ((lane % 8) ^ swz_kc(r)));
    }
  }
  __device__ __forceinline__ void issue(const bf16* base, bf16* lds, int wu) const {
#pragma unroll
    for (int q = 0; q < PER; ++q) dma16(base, off[q], lds + (PER * wu + q) * 512);
  }
};

// The k-steps s of n of a few-rows product through STAGES buffers: issue(s, b)
// asks for step s into buffer b (PER loads a wave), step(s, b) multiplies it.
// With three buffers two steps are loading at any time, and one barrier a step
// does: behind it every wave has read the buffer that the next loads go to.
template <int STAGES, int PER, class I, class C>
__device__ __forceinline__ void few_steps(int n, I issue, C step) {
  static_assert(STAGES == 2 || STAGES == 3, "two or three buffers");
  if (n <= 0) return;
  issue(0, 0);
  if constexpr (STAGES == 2) {
    for (int s = 0; s < n; ++s) {
      if (s + 1 < n) {
        issue(s + 1, (s + 1) & 1);
        wait_vmcnt<PER>();
      } else {
        wait_vmcnt<0>();
      }
      phase_barrier();
      step(s, s & 1);
      wait_lds();
      phase_barrier();
    }
  } else {
    if (n > 1) issue(1, 1);
    int b = 0;
    for (int s = 0; s < n; ++s) {
      if (s + 1 < n)
        wait_vmcnt<PER>();
      else
        wait_vmcnt<0>();
      phase_barrier();
      if (s + 2 < n) issue(s + 2, b == 0 ? 2 : b - 1);
      step(s, b);
      wait_lds();
      b = b == 2 ? 0 : b + 1;
    }
    phase_barrier();
  }
}

}  // namespace gemm
}  // namespace siq

// Internal interface of the preference and policy loss kernels.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace siq {

// Packed sequences: sequence s holds tokens [cu[s], cu[s + 1]) of `tokens`;
// cu nullptr: one sequence of all tokens.
struct Packed {
  const int32_t* cu;
  int64_t seqs, tokens;
};

enum { kPrefSigmoid = 0, kPrefIpo = 1, kPrefHinge = 2 };

struct PrefArgs {
  Packed seq;                 // 2 pairs sequences
  const float* policy;        // [tokens]
  const float* reference;     // [tokens], or nullptr (zero)
  const uint8_t* mask;        // [tokens], or nullptr (all count)
  int64_t pairs;
  int type, halves, normalized;
  double beta, smoothing;
  const float* divisor;       // or nullptr: the number of pairs
  float* loss;
  float* chosen;              // [pairs] rewards
  float* rejected;
  float* coef;                // [2 pairs] d loss / d (a counted token of the sequence)
  void* ws;
};
size_t pref_workspace_bytes(int64_t pairs, int64_t tokens);
hipError_t pref_fwd(const PrefArgs& a, hipStream_t stream);
hipError_t pref_bwd(const Packed& seq, const float* grad, const float* coef, const uint8_t* mask, float* dpolicy,
                    hipStream_t stream);

enum { kKlNone = -1, kKl1 = 0, kKl2 = 1, kKl3 = 2 };

struct PolicyArgs {
  Packed seq;
  const float* logps;       // [tokens]
  const float* old;
  const float* advantages;  // [tokens] or [seqs]
  const uint8_t* mask;      // or nullptr
  const float* reference;   // or nullptr
  int per_token, by_sequence, kl;
  double log_low, log_high, log_dual;  // logarithms of the ratios past which a token is cut (log_dual +inf: none)
  float low, high, dual;               // those ratios
  float kl_coef;
  const float* divisor;     // or nullptr: counted tokens, or sequences
  float* loss;
  float* mean_kl;
  float* clip_fraction;     // share of cut tokens
  float* dtoken;            // [tokens] gradient of a token's loss
  float* weight;            // [seqs] (by_sequence) or [1]: its share in the loss
  void* ws;
};
size_t policy_workspace_bytes(int64_t seqs, int64_t tokens);
hipError_t policy_fwd(const PolicyArgs& a, hipStream_t stream);
hipError_t policy_bwd(const Packed& seq, bool by_sequence, const float* grad, const float* dtoken, const float* weight,
                      float* dlogps, hipStream_t stream);

}  // namespace siq

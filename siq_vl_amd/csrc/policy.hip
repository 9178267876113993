// Losses of preference and policy training on packed per-token
// log-probabilities, forward and backward.
//
// Preference (paired log ratios): s_q = sum over a sequence's counted tokens of
// (policy - reference), divided by their number when length-normalised;
// x = s_chosen - s_rejected of a pair, z = beta x,
//   sigmoid  (1 - e) softplus(-z) + e softplus(z),   ipo  (x - 1 / (2 beta))^2,
//   hinge  max(0, 1 - z),
// averaged over the pairs.  Every counted token of a sequence has the same
// gradient, +-(d loss / dx) [/ length].
//
// Policy: ratio r = exp(logp - old); a token's loss is -min(r A, clip(r) A),
// for A < 0 at least -c A with the second clip c, plus kl_coef times an
// estimate of the KL divergence from the reference.  Whether a token is cut is
// decided in 64 bits, on the exact difference of the two fp32
// log-probabilities against the logarithm of the border: in 32 bits tokens next
// to it would be cut or not by the rounding of exp.
//
// Both read each token once (9 to 21 bytes) and do little with it, so they are
// bound by memory for long batches and by launches for short ones: a pass over
// the tokens that leaves one partial sum a slice, and one workgroup that adds
// those up in a fixed order and turns them into the loss and the sequences'
// weights; where there are few slices that workgroup makes them too, in one
// launch (kOneLaunch).  No atomics: results are bitwise reproducible.  Sums are
// in 64 bits: a margin is a difference of two sums of thousands of terms.
#include <type_traits>

#include "common.h"
#include "policy.h"

namespace siq {

namespace {

constexpr int kThreads = 256;
constexpr int kPer = 8;                    // tokens a thread has in flight
constexpr int kSlice = kThreads * kPer;    // tokens of a slice at most
constexpr int kSumThreads = 1024;
constexpr int kOneLaunch = kSumThreads / 64;  // slices that the one workgroup takes, a wave each

// Slices.  The token axis is cut at multiples of kSlice and at sequence ends.
// Going along it, each cut raises the sequence s, the window w = t / kSlice, or
// both, so s + w names every slice once: slice b belongs to the last sequence
// whose first slice, s + cu[s] / kSlice, is not past b.  The tokens behind the
// last sequence are one more sequence, of tokens that do not count.  Offsets
// outside [0, tokens] are clamped (and the first is 0), so that malformed ones
// reach no token outside.
__device__ __forceinline__ int64_t seq_start(const Packed& p, int64_t s) {
  if (s <= 0) return 0;
  if (s > p.seqs || p.cu == nullptr) return p.tokens;
  return min(max((int64_t)p.cu[s], (int64_t)0), p.tokens);
}
struct Slice {
  int64_t s, begin, end;
};
// A wave searches together, 64 offsets at a step: with 700 sequences two loads
// that wait for one another instead of ten.
__device__ __forceinline__ Slice slice_of(const Packed& p, int64_t b) {
  const int lane = threadIdx.x & 63;
  int64_t lo = 0, hi = p.seqs + 1;  // first slice of lo <= b; of hi: past it
  while (hi - lo > 1) {
    const int64_t step = (hi - lo + 63) / 64, at = lo + (lane + 1) * step;
    const uint64_t past = __ballot(at >= hi || at + seq_start(p, at) / kSlice > b);
    const int64_t k = past != 0 ? (int64_t)__builtin_ctzll(past) : 64;
    hi = min(hi, lo + (k + 1) * step);
    lo += k * step;
  }
  const int64_t w = b - lo;
  return Slice{lo, max(seq_start(p, lo), w * kSlice), min(seq_start(p, lo + 1), (w + 1) * kSlice)};
}
int64_t slices(int64_t seqs, int64_t tokens) { return seqs + 1 + (tokens + kSlice - 1) / kSlice; }
// Slices [first, last) of sequence s.
__device__ __forceinline__ void slices_of(const Packed& p, int64_t s, int64_t& first, int64_t& last) {
  const int64_t a = seq_start(p, s), e = seq_start(p, s + 1);
  first = s + a / kSlice;
  last = e > a ? s + (e - 1) / kSlice + 1 : first;
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o);
  return x;
}
// Sums over a workgroup of NT threads, in thread 0.
template <int NT, int K>
__device__ __forceinline__ void block_sum(double (&x)[K]) {
  __shared__ double sh[NT / 64][K];
#pragma unroll
  for (int k = 0; k < K; ++k) x[k] = wave_sum(x[k]);
  if ((threadIdx.x & 63) == 0)
#pragma unroll
    for (int k = 0; k < K; ++k) sh[threadIdx.x >> 6][k] = x[k];
  __syncthreads();
  if (threadIdx.x == 0)
    for (int w = 1; w < NT / 64; ++w)
#pragma unroll
      for (int k = 0; k < K; ++k) x[k] += sh[w][k];
}

// Lanes that add up one sequence's slices: as many as it has on average.
int lanes_for(int64_t seqs, int64_t tokens) {
  const int64_t per = (tokens / kSlice + seqs - 1) / seqs;
  int g = 1;
  while (g < 64 && g < per) g <<= 1;
  return g;
}

// ---------------------------------------------------------------- preference
struct PrefPart {
  double sum, count;
};

// Sum of policy - reference and number of the slice's counted tokens that
// thread `tid` of G sees.
template <int G>
__device__ __forceinline__ void pref_slice(const PrefArgs& p, const Slice& c, int tid, double (&x)[2]) {
  x[0] = 0.;
  int n = 0;
  for (int64_t t0 = c.begin + tid; t0 < c.end; t0 += G * kPer) {
    float a[kPer], r[kPer];
    bool m[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      // (past the end the last token again, not counted: loads without branches are all in flight at once)
      const int64_t t = t0 + i * G, at = min(t, c.end - 1);
      m[i] = (p.mask == nullptr || p.mask[at] != 0) && t < c.end;
      a[i] = p.policy[at];
      r[i] = p.reference != nullptr ? p.reference[at] : 0.f;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      x[0] += m[i] ? (double)a[i] - (double)r[i] : 0.;
      n += m[i] ? 1 : 0;
    }
  }
  x[1] = (double)n;
}

__global__ __launch_bounds__(kThreads) void pref_slice_kernel(const PrefArgs p, PrefPart* __restrict__ part) {
  const Slice c = slice_of(p.seq, blockIdx.x);
  if (c.begin >= c.end || c.s >= p.seq.seqs) return;
  double x[2];
  pref_slice<kThreads>(p, c, threadIdx.x, x);
  block_sum<kThreads, 2>(x);
  if (threadIdx.x == 0) part[blockIdx.x] = PrefPart{x[0], x[1]};
}

// ONE: the slices (nslices <= kOneLaunch) are made here.
template <bool ONE>
__global__ __launch_bounds__(kSumThreads) void pref_pair_kernel(const PrefArgs p, PrefPart* __restrict__ part,
                                                                PrefPart* __restrict__ total, int lanes, int nslices) {
  const int tid = threadIdx.x;
  if (ONE) {
    const int b = tid >> 6;
    if (b < nslices) {
      const Slice c = slice_of(p.seq, b);
      if (c.begin < c.end && c.s < p.seq.seqs) {
        double x[2];
        pref_slice<64>(p, c, tid & 63, x);
        const PrefPart q{wave_sum(x[0]), wave_sum(x[1])};
        if ((tid & 63) == 0) part[b] = q;
      }
    }
    __syncthreads();
  }
  const int64_t n = 2 * p.pairs;
  for (int64_t s = tid / lanes; s < n; s += kSumThreads / lanes) {
    int64_t first, last;
    slices_of(p.seq, s, first, last);
    PrefPart t{0., 0.};
    for (int64_t b = first + tid % lanes; b < last; b += lanes) {
      t.sum += part[b].sum;
      t.count += part[b].count;
    }
    for (int o = lanes >> 1; o >= 1; o >>= 1) {
      t.sum += __shfl_xor(t.sum, o);
      t.count += __shfl_xor(t.count, o);
    }
    if (tid % lanes == 0) total[s] = t;
  }
  __syncthreads();
  const double inv = 1. / (p.divisor != nullptr ? (double)*p.divisor : (double)p.pairs), beta = p.beta;
  double loss[1] = {0.};
  for (int64_t i = tid; i < p.pairs; i += kSumThreads) {
    const int64_t c = p.halves ? i : 2 * i, r = p.halves ? p.pairs + i : 2 * i + 1;
    const PrefPart tc = total[c], tr = total[r];
    const double wc = p.normalized ? 1. / fmax(tc.count, 1.) : 1., wr = p.normalized ? 1. / fmax(tr.count, 1.) : 1.;
    const double sc = tc.sum * wc, sr = tr.sum * wr, x = sc - sr, z = beta * x;
    double l, dx;
    if (p.type == kPrefSigmoid) {
      const double q = exp(-fabs(z)), soft = log1p(q);  // softplus(+-z) = max(+-z, 0) + soft
      l = (1. - p.smoothing) * (fmax(-z, 0.) + soft);
      if (p.smoothing > 0.) l += p.smoothing * (fmax(z, 0.) + soft);  // (z may be infinite)
      const double up = z >= 0. ? 1. / (1. + q) : q / (1. + q), down = z >= 0. ? q / (1. + q) : 1. / (1. + q);
      dx = beta * (p.smoothing * up - (1. - p.smoothing) * down);
    } else if (p.type == kPrefIpo) {
      const double e = x - 0.5 / beta;
      l = e * e;
      dx = 2. * e;
    } else {
      l = fmax(1. - z, 0.);
      dx = z < 1. ? -beta : 0.;
    }
    if (x != x) l = dx = x;  // NaN (fmax and the comparisons above drop it)
    loss[0] += l;
    p.chosen[i] = (float)(beta * sc);
    p.rejected[i] = (float)(beta * sr);
    p.coef[c] = (float)(dx * inv * wc);
    p.coef[r] = (float)(-dx * inv * wr);
  }
  block_sum<kSumThreads, 1>(loss);
  if (tid == 0) *p.loss = (float)(loss[0] * inv);
}

// Gradients of a slice's tokens: the sequence's weight times what the token
// has (`value`: nullptr = 1 where it counts).
__global__ __launch_bounds__(kThreads) void spread_kernel(const Packed seq, const float* __restrict__ grad,
                                                          const float* __restrict__ weight,
                                                          const uint8_t* __restrict__ mask,
                                                          const float* __restrict__ value, float* __restrict__ out) {
  const Slice c = slice_of(seq, blockIdx.x);
  if (c.begin >= c.end) return;
  const float w = c.s < seq.seqs ? *grad * weight[c.s] : 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int64_t t = c.begin + i * kThreads + threadIdx.x;
    if (t >= c.end) break;
    const float v = value != nullptr ? value[t] : 1.f;
    const bool counts = c.s < seq.seqs && (value != nullptr ? v != 0.f : mask == nullptr || mask[t] != 0);
    out[t] = counts ? w * v : 0.f;
  }
}

// ---------------------------------------------------------------- policy
struct PolicyPart {
  double loss, kl, count, cut;
};

// Estimate of the KL divergence at y = reference - logp, and its derivative by logp.
template <int KL>
__device__ __forceinline__ void kl_term(float y, float& kl, float& dkl) {
  if (KL == kKl3) {
    // e^y - 1 - y: by its Taylor series up to |y| = 1/2 (the rest is below 2e-9 of it), where the difference would
    // cancel; both are formed and one is taken, so that a wave's lanes stay together
    float q = 1.f / 362880.f;
    q = __builtin_fmaf(q, y, 1.f / 40320.f);
    q = __builtin_fmaf(q, y, 1.f / 5040.f);
    q = __builtin_fmaf(q, y, 1.f / 720.f);
    q = __builtin_fmaf(q, y, 1.f / 120.f);
    q = __builtin_fmaf(q, y, 1.f / 24.f);
    q = __builtin_fmaf(q, y, 1.f / 6.f);
    q = __builtin_fmaf(q, y, 0.5f);
    const float near = q * y * y, e1 = exp2f_fast(y * kLog2e) - 1.f;
    const bool small = fabsf(y) <= 0.5f;
    kl = small ? near : e1 - y;
    dkl = -(small ? y + near : e1);
  } else if (KL == kKl2) {
    kl = 0.5f * y * y;
    dkl = -y;
  } else {
    kl = -y;
    dkl = 1.f;
  }
}

// Sums of the slice's counted tokens that thread `tid` of G sees (loss, kl,
// count, cut), and every token's gradient.  tail: behind the last sequence.
template <int G, int KL>
__device__ __forceinline__ void policy_slice(const PolicyArgs& p, const Slice& c, bool tail, int tid, double (&x)[4]) {
  x[0] = x[1] = 0.;
  int count = 0, cuts = 0;
  const float seq_adv = tail || p.per_token ? 0.f : p.advantages[c.s];
  for (int64_t t0 = c.begin + tid; t0 < c.end; t0 += G * kPer) {
    float lp[kPer], old[kPer], ref[kPer], adv[kPer];
    uint8_t mk[kPer];
    // (past the end the last token again, not counted: loads without branches are all in flight at once)
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int64_t at = min(t0 + i * G, c.end - 1);
      lp[i] = p.logps[at];
      old[i] = p.old[at];
      if (KL != kKlNone) ref[i] = p.reference[at];
    }
    if (p.per_token) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) adv[i] = p.advantages[min(t0 + i * G, c.end - 1)];
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) adv[i] = seq_adv;
    }
    if (p.mask != nullptr) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) mk[i] = p.mask[min(t0 + i * G, c.end - 1)];
    } else {
#pragma unroll
      for (int i = 0; i < kPer; ++i) mk[i] = 1;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int64_t t = t0 + i * G;
      const bool m = t < c.end && !tail && mk[i] != 0;
      const double d = (double)lp[i] - (double)old[i];
      const float A = adv[i], r = exp2f_fast((float)d * kLog2e);
      const bool over = A > 0.f && d > p.log_high, under = A < 0.f && d < p.log_low, far = A < 0.f && d > p.log_dual;
      const bool cut = over || under || far;
      float loss = -(A * (over ? p.high : under ? p.low : far ? p.dual : r)), g = cut ? 0.f : -A * r;
      if (KL != kKlNone) {
        float kl, dkl;
        kl_term<KL>((float)((double)ref[i] - (double)lp[i]), kl, dkl);
        if (p.kl_coef != 0.f) {  // (an estimate that is only reported may be infinite)
          loss = __builtin_fmaf(p.kl_coef, kl, loss);
          g = __builtin_fmaf(p.kl_coef, dkl, g);
        }
        x[1] += (double)(m ? kl : 0.f);
      }
      x[0] += (double)(m ? loss : 0.f);
      count += m ? 1 : 0;
      cuts += m && cut ? 1 : 0;
      if (t < c.end) p.dtoken[t] = m ? g : 0.f;
    }
  }
  x[2] = (double)count;
  x[3] = (double)cuts;
}

template <int KL>
__global__ __launch_bounds__(kThreads) void policy_slice_kernel(const PolicyArgs p, PolicyPart* __restrict__ part) {
  const Slice c = slice_of(p.seq, blockIdx.x);
  if (c.begin >= c.end) return;
  const bool tail = c.s >= p.seq.seqs;
  double x[4];
  policy_slice<kThreads, KL>(p, c, tail, threadIdx.x, x);
  if (tail) return;
  block_sum<kThreads, 4>(x);
  if (threadIdx.x == 0) part[blockIdx.x] = PolicyPart{x[0], x[1], x[2], x[3]};
}

// ONE: the slices (nslices <= kOneLaunch) are made here.
template <bool ONE, int KL>
__global__ __launch_bounds__(kSumThreads) void policy_sum_kernel(const PolicyArgs p, PolicyPart* __restrict__ part,
                                                                 int lanes, int nslices) {
  const int tid = threadIdx.x;
  if (ONE) {
    const int b = tid >> 6;
    if (b < nslices) {
      const Slice c = slice_of(p.seq, b);
      const bool tail = c.s >= p.seq.seqs;
      if (c.begin < c.end) {
        double x[4];
        policy_slice<64, KL>(p, c, tail, tid & 63, x);
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = wave_sum(x[k]);
        if ((tid & 63) == 0 && !tail) part[b] = PolicyPart{x[0], x[1], x[2], x[3]};
      }
    }
    __syncthreads();
  }
  const double div = p.divisor != nullptr ? (double)*p.divisor : (double)p.seq.seqs;
  double x[4] = {0., 0., 0., 0.};  // loss, kl, count, cut
  for (int64_t s = tid / lanes; s < p.seq.seqs; s += kSumThreads / lanes) {
    int64_t first, last;
    slices_of(p.seq, s, first, last);
    double l = 0., n = 0.;
    for (int64_t b = first + tid % lanes; b < last; b += lanes) {
      const PolicyPart q = part[b];
      l += q.loss;
      n += q.count;
      x[1] += q.kl;
      x[3] += q.cut;
    }
    for (int o = lanes >> 1; o >= 1; o >>= 1) {
      l += __shfl_xor(l, o);
      n += __shfl_xor(n, o);
    }
    if (tid % lanes != 0) continue;
    const double w = 1. / (div * fmax(n, 1.));
    if (p.by_sequence) p.weight[s] = (float)w;
    x[0] += !p.by_sequence ? l : n > 0. ? l * w : 0.;  // (divided by 0 items, w is infinite)
    x[2] += n;
  }
  block_sum<kSumThreads, 4>(x);
  if (tid != 0) return;
  const double per = 1. / fmax(x[2], 1.);
  if (!p.by_sequence) {
    const double w = p.divisor != nullptr ? 1. / div : per;
    x[0] = x[2] > 0. ? x[0] * w : 0.;
    p.weight[0] = (float)w;
  }
  *p.loss = (float)x[0];
  *p.mean_kl = (float)(x[1] * per);
  *p.clip_fraction = (float)(x[3] * per);
}

// dlogps = grad weight dtoken, one weight for all tokens.
__global__ __launch_bounds__(kThreads) void policy_scale_kernel(const float* __restrict__ grad,
                                                                const float* __restrict__ weight,
                                                                const float* __restrict__ dtoken, int64_t tokens,
                                                                float* __restrict__ out) {
  const float w = *grad * *weight;
  const int64_t t0 = ((int64_t)blockIdx.x * kThreads + threadIdx.x) * 4;
  if (t0 + 4 <= tokens) {
    f32x4 v = *reinterpret_cast<const f32x4*>(dtoken + t0);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = v[i] != 0.f ? w * v[i] : 0.f;
    *reinterpret_cast<f32x4*>(out + t0) = v;
  } else {
    for (int64_t t = t0; t < tokens; ++t) out[t] = dtoken[t] != 0.f ? w * dtoken[t] : 0.f;
  }
}

size_t al(size_t x) { return (x + 255) & ~size_t(255); }

}  // namespace

size_t pref_workspace_bytes(int64_t pairs, int64_t tokens) {
  return al(sizeof(PrefPart) * (size_t)slices(2 * pairs, tokens)) + al(sizeof(PrefPart) * (size_t)(2 * pairs));
}

hipError_t pref_fwd(const PrefArgs& a, hipStream_t stream) {
  const int64_t n = slices(a.seq.seqs, a.seq.tokens);
  PrefPart* part = static_cast<PrefPart*>(a.ws);
  PrefPart* total = reinterpret_cast<PrefPart*>(static_cast<char*>(a.ws) + al(sizeof(PrefPart) * (size_t)n));
  const int lanes = lanes_for(a.seq.seqs, a.seq.tokens);
  if (n <= kOneLaunch) {
    hipLaunchKernelGGL(pref_pair_kernel<true>, dim3(1), dim3(kSumThreads), 0, stream, a, part, total, lanes, (int)n);
  } else {
    hipLaunchKernelGGL(pref_slice_kernel, dim3((unsigned)n), dim3(kThreads), 0, stream, a, part);
    hipLaunchKernelGGL(pref_pair_kernel<false>, dim3(1), dim3(kSumThreads), 0, stream, a, part, total, lanes, 0);
  }
  return hipGetLastError();
}

hipError_t pref_bwd(const Packed& seq, const float* grad, const float* coef, const uint8_t* mask, float* dpolicy,
                    hipStream_t stream) {
  hipLaunchKernelGGL(spread_kernel, dim3((unsigned)slices(seq.seqs, seq.tokens)), dim3(kThreads), 0, stream, seq, grad,
                     coef, mask, nullptr, dpolicy);
  return hipGetLastError();
}

size_t policy_workspace_bytes(int64_t seqs, int64_t tokens) {
  return al(sizeof(PolicyPart) * (size_t)slices(seqs, tokens));
}

hipError_t policy_fwd(const PolicyArgs& a, hipStream_t stream) {
  PolicyPart* part = static_cast<PolicyPart*>(a.ws);
  const int64_t n = slices(a.seq.seqs, a.seq.tokens);
  const int lanes = lanes_for(a.seq.seqs, a.seq.tokens);
  auto run = [&](auto kl) {
    constexpr int KL = decltype(kl)::value;
    if (n <= kOneLaunch) {
      hipLaunchKernelGGL((policy_sum_kernel<true, KL>), dim3(1), dim3(kSumThreads), 0, stream, a, part, lanes, (int)n);
    } else {
      hipLaunchKernelGGL(policy_slice_kernel<KL>, dim3((unsigned)n), dim3(kThreads), 0, stream, a, part);
      hipLaunchKernelGGL((policy_sum_kernel<false, kKlNone>), dim3(1), dim3(kSumThreads), 0, stream, a, part, lanes, 0);
    }
  };
  switch (a.kl) {
    case kKl1:
      run(std::integral_constant<int, kKl1>());
      break;
    case kKl2:
      run(std::integral_constant<int, kKl2>());
      break;
    case kKl3:
      run(std::integral_constant<int, kKl3>());
      break;
    default:
      run(std::integral_constant<int, kKlNone>());
  }
  return hipGetLastError();
}

hipError_t policy_bwd(const Packed& seq, bool by_sequence, const float* grad, const float* dtoken, const float* weight,
                      float* dlogps, hipStream_t stream) {
  if (by_sequence) {
    hipLaunchKernelGGL(spread_kernel, dim3((unsigned)slices(seq.seqs, seq.tokens)), dim3(kThreads), 0, stream, seq, grad,
                       weight, nullptr, dtoken, dlogps);
  } else {
    hipLaunchKernelGGL(policy_scale_kernel, dim3((unsigned)((seq.tokens + 4 * kThreads - 1) / (4 * kThreads))),
                       dim3(kThreads), 0, stream, grad, weight, dtoken, seq.tokens, dlogps);
  }
  return hipGetLastError();
}

}  // namespace siq

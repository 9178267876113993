// Distillation from a teacher's most probable tokens, from the student's hidden
// states and without logits, forward and backward, for gfx950.
//
// A row's teacher names K tokens with log-probabilities ln t_k; m = sum t_k, and
// r = max(1 - m, 0) is what it leaves to all others, its tail.  The student's
// p = softmax(h W^T / temperature) is s_k at those tokens and q elsewhere.
//   forward:  D = sum t_k (ln t_k - ln s_k) + r (ln r - ln q)   (the second term with a tail)
//   reverse:  D = sum s_k (ln s_k - ln t_k) + q (ln q - ln r),  r at least 2^-24
//   loss = sum over rows of ((1 - c) D + c CE) / den,  CE = -ln p_y.
// All tokens outside the list have the same dD/dz_j / p_j = O, so the gradient is a
// row factor times the softmax numerators, but for a few tokens a row:
//   forward:  O = m + r - r / q (tail) or m,  inside: p_k (m + r) - t_k or p_k m - t_k
//   reverse:  O = ln q - ln r - D,            inside: p_k (ln p_k - ln t_k - D),
// and with the label  dz = (1 - c) dD/dz + c (p - [y]).
//
// The products are the fused cross-entropy's, over chunks of compacted rows:
//  1. lists: a row's tokens (the label among them), a bit of the vocabulary for
//     each, and where a tile's begin;
//  2. logits GEMM: softmax numerators E in bf16 and their sums per tile without the
//     listed tokens, whose logits it leaves in fp32: what is outside the list is
//     never a difference from 1;
//  3. sums over the tiles; then, a wave a row, the losses and gradients of the row in
//     64 bits.  The gradient of the listed token with the largest one is kept in
//     fp32 and added by the products' kernels as a label's is; the others' are put
//     in their places in E, divided by the row's factor;
//  4. dH = f (E W) + w W[y'],  dW = (f H)^T E + the sums of w H by token.
// (All listed tokens in fp32 would take gathers of rows x K rows of W and of H.)
//
// Bounded by the products: 11450 counted rows x 1536 over 151936 columns, 64 tokens a
// row, all gradients, 13.95 ms (16.0 TFLOP, 1.15 PFLOP/s; what is not a product takes
// 0.5), loss alone of 3441 rows x 896 0.95 ms.  Few rows by memory, the table read twice
// and its gradient written: 48 rows x 896 228 us, 0.82 GB in 192 us of products.
#include <algorithm>

#include "distill.h"
#include "flce_launch.h"
#include "gemm.h"
#include "ids.h"

namespace siq {

namespace {

using namespace gemm;

// An entry of a list: the token's id, and whether it is the label where the teacher
// does not name it.
constexpr int32_t kIdMask = (1 << 24) - 1, kLabelOnly = 1 << 24;
constexpr int kListLanes = 3, kListMost = 64 * kListLanes;  // entries a lane; of a row
static_assert(kMaxTeacher + 1 <= kListMost, "the label behind the teacher's tokens");

// ---------------------------------------------------------------- lists
// A call of at most kFewRows rows: the kernel of the lists compacts them, too, as
// launch_compact does.
struct FewPrep {
  const int64_t* labels;  // [n]
  const bf16* hidden;
  const bf16* weight;
  int32_t* rows;          // [n]
  int64_t *y, *nvalid, *counts;  // [n]; ; [2]
  bf16* hc;               // [n, hdim]
  float* ref;             // [n]
  bf16* dh;               // or nullptr
  int64_t hdim, ignore_index;
  int n;
  float zscale;
};

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

// Workgroup k: the k-th counted row, where there is one.
struct FewRow {
  int nv, nbad, at;  // rows that count, bad labels, the row (-1: none)
  bool counts;       // row k's label does
  int64_t y;         // the label, or -1
};
__device__ __forceinline__ FewRow few_row(const FewPrep& p, int64_t V) {
  constexpr int G = kFewRows / 64;
  const int lane = threadIdx.x & 63, k = blockIdx.x;
  int nv = 0, nbad = 0, at = -1;
  bool counts = false;
#pragma unroll
  for (int g = 0; g < G; ++g) {
    const int64_t v = 64 * g + lane < p.n ? p.labels[64 * g + lane] : p.ignore_index;
    const bool ok = v >= 0 && v < V && v != p.ignore_index;
    const uint64_t m = __ballot(ok);
    nbad += __popcll(__ballot(v != p.ignore_index && !ok));
    const int rank = nv + __popcll(m & (lane ? ~0ull >> (64 - lane) : 0ull));
    const uint64_t mine = __ballot(ok && rank == k);
    if (mine != 0) at = 64 * g + (int)__builtin_ctzll(mine);
    counts = counts || (k / 64 == g && (m >> (k % 64) & 1));
    nv += __popcll(m);
  }
  return {nv, nbad, at, counts, at >= 0 ? p.labels[at] : -1};
}

// Its operands, and what belongs to row k where its label does not count.
__device__ __forceinline__ void few_compact(const FewPrep& p, const FewRow& r) {
  __shared__ float dot_sh[4];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, k = blockIdx.x, at = r.at;
  const int64_t y = r.y;
  float dot = 0.f;
  for (int64_t c = 8 * (int64_t)tid; c < p.hdim; c += 8 * 256) {
    bf16x8 x = zero_bf16x8();
    if (at >= 0) {
      x = ld_bf16x8(p.hidden + at * p.hdim + c);
      const bf16x8 wy = ld_bf16x8(p.weight + y * p.hdim + c);
#pragma unroll
      for (int i = 0; i < 8; ++i) dot = __builtin_fmaf((float)x[i], (float)wy[i], dot);
    }
    st_bf16x8(p.hc + k * p.hdim + c, x);
    if (!r.counts && p.dh != nullptr) st_bf16x8(p.dh + k * p.hdim + c, zero_bf16x8());
  }
  dot = wave_sum(dot);
  if (lane == 0) dot_sh[w] = dot;
  __syncthreads();
  if (tid == 0) {
    p.ref[k] = (dot_sh[0] + dot_sh[1] + dot_sh[2] + dot_sh[3]) * p.zscale;
    p.y[k] = y;
    if (at >= 0) p.rows[k] = at;
    if (k == 0) {
      *p.nvalid = p.counts[0] = r.nv;
      p.counts[1] = r.nbad;
    }
  }
}

struct ListArgs {
  const void* ids;        // [n, K]
  const float* teacher;   // [n, K]
  const int32_t* rows;    // [nc]
  const int64_t* y;       // [nc]
  const int64_t* nvalid;
  int32_t* out;           // [nc, ldk] the list, in the order of list_place
  float* lt;              // [nc, ldk] the teacher's log-probabilities
  uint8_t* mask;          // [nc, ldm] as the logits kernels want it
  uint8_t* base;          // [nc, ldb]
  int32_t* len;           // [nc]
  int32_t* bad;           // [nc] tokens outside the vocabulary, or named twice
  int64_t nc, c0, V, nvt, ldm, ldb;
  int K, ldk;
  FewPrep few;            // few.labels != nullptr: a call of few rows, nothing above has been compacted yet
};

// A workgroup a row, a thread a token: its key is (tile, place in it) * 256 + (place
// among the teacher's tokens; 255: the label, behind a teacher's same token), and its
// place in the list how many other kept keys are less.  Tokens of probability zero and
// ids of -1 are not there; of equal ids the first stays.  The bits are set in LDS,
// kListSpan columns at a time.  Few rows are bounded by the chain of steps (48 rows,
// compaction and all, 9 us), many by the bits (6912 rows 50 us, 145 MB).
constexpr int kListThreads = 256, kListSpan = 1 << 17;
static_assert(kMaxTeacher + 1 <= kListThreads, "a thread a token");
// How many of the first n keys (in fours; the last ones none) are less than x.
__device__ __forceinline__ int less_than(const uint32_t* keys, int n, uint32_t x) {
  int c = 0;
#pragma unroll 4
  for (int j = 0; j < n; j += 4) {
    const u32x4 k = *reinterpret_cast<const u32x4*>(keys + j);
#pragma unroll
    for (int i = 0; i < 4; ++i) c += k[i] < x ? 1 : 0;
  }
  return c;
}

template <class ID, bool FEW>
__global__ __launch_bounds__(kListThreads) void distill_list_kernel(const ListArgs p) {
  constexpr int VT = FEW ? kFewBI : kVT, LANE = list_lane_bits(FEW), NL = VT / LANE, T = kListThreads;
  constexpr uint32_t kNone = ~0u;
  __shared__ __align__(16) uint32_t key_sh[kMaxTeacher + 4];
  __shared__ __align__(16) uint32_t kept_sh[T];  // of each token, by its place among the teacher's: its key, or none
  __shared__ __align__(16) uint32_t bits_sh[kListSpan / 32];
  const int tid = threadIdx.x, K = p.K;
  const int64_t k = blockIdx.x;
  int64_t row = -1, y = -1;
  const bool prepare = FEW && p.few.labels != nullptr;
  FewRow found{};
  if (prepare) {
    found = few_row(p.few, p.V);
    row = found.at;
    y = found.y;
  } else if (k < min(p.nc, *p.nvalid - p.c0)) {
    row = p.rows[k];
    y = p.y[k];
  }
  const bool real = row >= 0;
  uint32_t mine = kNone;
  int id = -1;
  float lt = -INFINITY;
  bool wrong = false;
  if (real && tid < K) {
    const int64_t src = row * K + tid, v = static_cast<const ID*>(p.ids)[src];
    lt = p.teacher[src];
    wrong = v != -1 && (v < 0 || v >= p.V);
    id = wrong || lt == -INFINITY ? -1 : (int)v;
  } else if (real && tid == K) {
    id = (int)y;
  }
  if (id >= 0) mine = (uint32_t)(id / VT * VT + list_place(id % VT, FEW)) << 8 | (tid < K ? (uint32_t)tid : 255u);
  if (tid < kMaxTeacher + 4) key_sh[tid] = mine;
  if (prepare) few_compact(p.few, found);
  __syncthreads();
  // a token is kept unless the same one has a lower key: no key lies between (tile, place) * 256 and its own
  const bool kept = mine != kNone && less_than(key_sh, K + 1, mine) == less_than(key_sh, K + 1, mine & ~255u);
  const bool twice = mine != kNone && !kept && tid < K;
  kept_sh[tid] = kept ? mine : kNone;
  const int n = __syncthreads_count(kept), bad = __syncthreads_count(wrong || twice);
  if (kept) {
    const int at = less_than(kept_sh, K + 1, mine);
    p.out[k * p.ldk + at] = id | (tid == K ? kLabelOnly : 0);
    p.lt[k * p.ldk + at] = lt;
  }
  if (real && tid == 0) {
    p.len[k] = n;
    p.bad[k] = bad;
  }
  const uint32_t bit = mine >> 8;  // (none: past every column)
  for (int64_t s0 = 0; s0 < p.nvt * VT; s0 += kListSpan) {
    const int words = (int)(min((int64_t)kListSpan, p.nvt * VT - s0) / 32);
    for (int i = tid; i < words / 4; i += T) reinterpret_cast<u32x4*>(bits_sh)[i] = u32x4{0u, 0u, 0u, 0u};
    __syncthreads();
    if (kept && bit >= s0 && bit < s0 + kListSpan) atomicOr(&bits_sh[(bit - s0) / 32], 1u << (bit & 31));
    __syncthreads();
    u32x4* mask = reinterpret_cast<u32x4*>(p.mask + k * p.ldm + s0 / 8);
    for (int i = tid; i < words / 4; i += T) mask[i] = reinterpret_cast<const u32x4*>(bits_sh)[i];
    for (int t = tid; t < words / (VT / 32); t += T) {
      uint64_t base = 0;  // a byte for each lane's bits
      const uint32_t t0 = (uint32_t)(s0 + t * VT) << 8;
      int before = n > 0 ? less_than(kept_sh, K + 1, t0) : 0;
#pragma unroll
      for (int q = 0; q < NL; ++q) {
        base |= (uint64_t)before << (8 * q);
        const uint32_t* w = bits_sh + (t * VT + q * LANE) / 32;
        before += LANE == 64 ? __popc(w[0]) + __popc(w[1]) : __popc(w[0] >> (q % 2 * 16) & 0xffffu);
      }
      const int64_t at = s0 / VT + t;
      if (NL == 8)
        *reinterpret_cast<uint64_t*>(p.base + k * p.ldb + 8 * at) = base;
      else
        *reinterpret_cast<uint32_t*>(p.base + k * p.ldb + 4 * at) = (uint32_t)base;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------- rows
struct RowMathArgs {
  const int32_t* ids;     // [nc, ldk] the lists
  const float* lt;        // [nc, ldk]
  const float* zk;        // [nc, ldk] log2 units, relative to ref
  const int32_t* len;     // [nc]
  const float* ref;       // [nc]
  const float* rsum;      // [nc] sum over the tokens that are not listed, relative to rtop
  const float* rtop;
  const int64_t* y;       // [nc]
  const int64_t* nvalid;
  const float* divisor;   // nullptr: the rows that count
  bf16* E;                // [nc, V] or nullptr: losses alone
  float* f;               // [nc] factor of E
  float* w;               // [nc] the largest gradient of a listed token, and
  int64_t* at;            // [nc] whose it is
  double* loss;           // [3, n] by compacted row: loss, divergence, cross-entropy
  int64_t nc, c0, n, V;
  int ldk;
  bool reverse, tail;
  double c, inv_t;
  // few rows: the sums over the tiles are made here, too
  const float* spart;     // [nvt, ldp]
  const float* mpart;
  bf16* H;                // [nc, hdim] times f, or nullptr
  int64_t nvt, ldp, hdim;
};

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o);
  return x;
}
__device__ __forceinline__ double wave_max(double x) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x = fmax(x, __shfl_xor(x, o));
  return x;
}

// Row k by one wave, from its sum over the tokens that are not listed: losses, and with E
// the row's factor (returned) and gradients of listed tokens.
__device__ __forceinline__ float row_math(const RowMathArgs& p, int64_t k, int64_t counted, double rsum, double rtop) {
  constexpr double kLn2d = 0.6931471805599453;
  const int lane = threadIdx.x & 63;
  const int n = p.len[k];
  const int64_t y = p.y[k];
  const double ref = p.ref[k];
  int id[kListLanes];  // -1: no entry
  bool teachers[kListLanes];
  double l2[kListLanes], lt[kListLanes];  // ln p in log2 units, ln t
  double top = rtop;
#pragma unroll
  for (int i = 0; i < kListLanes; ++i) {
    const int e = lane + 64 * i;
    id[i] = -1;
    teachers[i] = false;
    l2[i] = lt[i] = -INFINITY;
    if (e >= n) continue;
    const int32_t x = p.ids[k * p.ldk + e];
    id[i] = x & kIdMask;
    teachers[i] = (x & kLabelOnly) == 0;
    l2[i] = ref + (double)p.zk[k * p.ldk + e];
    lt[i] = p.lt[k * p.ldk + e];
    top = fmax(top, l2[i]);
  }
  top = wave_max(top);
  // sums of 2^(z2 - top): the teacher's tokens, and all others (the label may be among them)
  double inside = 0., extra = 0., ly = 0., mass = 0.;
  int named = 0;
  double ex[kListLanes], t[kListLanes];
#pragma unroll
  for (int i = 0; i < kListLanes; ++i) {
    ex[i] = t[i] = 0.;
    if (id[i] < 0) continue;
    ex[i] = exp2(l2[i] - top);
    if (teachers[i]) {
      t[i] = exp(lt[i]);
      inside += ex[i];
      mass += t[i];
      ++named;
    } else {
      extra += ex[i];
    }
    if (id[i] == y) ly = l2[i] - top;
  }
  inside = wave_sum(inside);
  extra = wave_sum(extra);
  ly = wave_sum(ly);  // (one lane's, and zeros)
  mass = wave_sum(mass);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) named += __shfl_xor(named, o);
  const double shift = exp2(rtop - top), outside = rsum * shift + extra, all = inside + outside;
  const double lall = log(all), q = outside / all;
  // (all others together below 2^-126 of the row's reference are taken for that)
  const double lq = log(fmax(outside, 0x1p-126)) - lall;
  const bool tail = p.tail && named < p.V;  // a teacher that names every token has no tail
  double r = 1. - mass;
  r = r < 0. ? 0. : r;
  if (p.reverse) r = r < 0x1p-24 ? 0x1p-24 : r;
  const double lr = log(r);
  double div = 0.;
#pragma unroll
  for (int i = 0; i < kListLanes; ++i) {
    if (!teachers[i]) continue;
    const double ls = (l2[i] - top) * kLn2d - lall, s = ex[i] / all;
    div += p.reverse ? (s == 0. ? 0. : s * (ls - lt[i])) : t[i] * (lt[i] - ls);
  }
  div = wave_sum(div);
  if (tail) div += p.reverse ? q * (lq - lr) : r > 0. ? r * (lr - lq) : 0.;
  const double ce = lall - ly * kLn2d, c = p.c;
  if (lane == 0) {
    const int64_t o = p.c0 + k;
    p.loss[o] = (1. - c) * div + c * ce;
    p.loss[p.n + o] = div;
    p.loss[2 * p.n + o] = ce;
  }
  if (p.E == nullptr) return 0.f;
  const double whole = tail ? mass + r : mass;
  double outer = p.reverse ? (tail ? lq - lr - div : 0.) : whole;
  if (!p.reverse && tail) outer -= outside > 0. ? r / q : 0.;
  outer = (1. - c) * outer + c;
  const double inv = p.inv_t / (p.divisor != nullptr ? (double)*p.divisor : (double)counted);
  // gradients of the listed tokens, and the largest of them (of equal ones the lowest id)
  double dz[kListLanes], big = -1.;
  int place = 1 << 30;
#pragma unroll
  for (int i = 0; i < kListLanes; ++i) {
    dz[i] = 0.;
    if (id[i] < 0) continue;
    const double s = ex[i] / all;
    if (!teachers[i]) {
      dz[i] = s * outer;
    } else {
      const double ls = (l2[i] - top) * kLn2d - lall;
      dz[i] = (1. - c) * (p.reverse ? (s == 0. ? 0. : s * (ls - lt[i] - div)) : s * whole - t[i]) + c * s;
    }
    if (id[i] == y) dz[i] -= c;
    dz[i] *= inv;
    const double a = dz[i] != dz[i] ? INFINITY : fabs(dz[i]);
    if (a > big) {
      big = a;
      place = lane + 64 * i;
    }
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) {
    const double b = __shfl_xor(big, o);
    const int q2 = __shfl_xor(place, o);
    if (b > big || (b == big && q2 < place)) {
      big = b;
      place = q2;
    }
  }
  // The factor of the others.  What is listed is divided by it, so it is kept from vanishing beside them: then the
  // others are off by at most 2^-20 of the largest together, far below the rounding of the listed ones to bf16.
  double f = outer * inv * shift / all;
  const double least = fmax(0x1p-20 * big / fmax(rsum, 1.), 0x1p-110);
  if (fabs(f) < least) f = big > 0. ? copysign(least, f) : 0.;
  if (fabs(f) > 0x1p100) f = copysign(0x1p100, f);
#pragma unroll
  for (int i = 0; i < kListLanes; ++i) {
    if (id[i] < 0) continue;
    const bool apart = lane + 64 * i == place;
    p.E[k * p.V + id[i]] = (bf16)(apart || f == 0. ? 0.f : (float)(dz[i] / f));
    if (apart) {
      p.w[k] = (float)dz[i];
      p.at[k] = id[i];
    }
  }
  if (lane == 0) p.f[k] = (float)f;
  return (float)f;
}

// A wave a row, behind flce_row_kernel's sums; 6912 rows of 64 tokens 23 us, nearly all of
// it 64-bit exponentials and logarithms.
__global__ __launch_bounds__(256) void distill_row_kernel(const RowMathArgs p) {
  const int64_t counted = *p.nvalid, k = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (k < min(p.nc, counted - p.c0)) row_math(p, k, counted, p.rsum[k], p.rtop[k]);
}

// Sums of the rows' losses, in a fixed order and 64 bits; one workgroup: 4 us, 10 for
// 16384 rows.  (Left to the row kernel's last workgroup, behind a fence of every
// workgroup's, it costs more.)
struct LossArgs {
  const double* loss;     // [3, n]
  const int32_t* bad;     // [n] by compacted row
  const int64_t* nvalid;
  const float* divisor;
  float* out[3];
  int64_t* total_bad;
  int64_t n;
};
__global__ __launch_bounds__(1024) void distill_loss_kernel(const LossArgs p) {
  constexpr int T = 1024, NWV = T / 64;
  __shared__ double sm[3][NWV];
  __shared__ long long bad_sh[NWV];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t nv = min(p.n, *p.nvalid);
  double s[3] = {0., 0., 0.};
  long long bad = 0;
  for (int64_t i = tid; i < nv; i += T) {
#pragma unroll
    for (int j = 0; j < 3; ++j) s[j] += p.loss[j * p.n + i];
    bad += p.bad[i];
  }
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) bad += __shfl_xor(bad, o);
#pragma unroll
  for (int j = 0; j < 3; ++j) {
    s[j] = wave_sum(s[j]);
    if (lane == 0) sm[j][w] = s[j];
  }
  if (lane == 0) bad_sh[w] = bad;
  __syncthreads();
  if (tid >= 4) return;
  if (tid == 3) {
    bad = 0;
    for (int i = 0; i < NWV; ++i) bad += bad_sh[i];
    *p.total_bad = bad;
    return;
  }
  double x = 0.;
  for (int i = 0; i < NWV; ++i) x += sm[tid][i];
  *p.out[tid] = (float)(x / (p.divisor != nullptr ? (double)*p.divisor : (double)nv));
}

// Few rows: a workgroup a row adds its tiles' sums (E of rows with redone tiles is
// brought to the largest of their references, as flce_row_kernel does), one wave of it does
// the row's math, and all scale its hidden state for dW.  A chain of latencies: 10 us (12
// where the sums were read twice, a few at a time).
__global__ __launch_bounds__(256) void distill_row_few_kernel(const RowMathArgs p) {
  constexpr int T = 256, NWV = T / 64;
  __shared__ double s_sh[NWV];
  __shared__ float m_sh[NWV], f_sh;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t counted = *p.nvalid, nv = min(p.nc, counted - p.c0), k = blockIdx.x;
  if (k >= nv) return;
  const float rf = p.ref[k];
  float m = rf;  // the reference of the sum: the row's, or a redone tile's above it
  // the sums of tiles, all on their way at once where there are no more than 1280
  constexpr int R = 5;
  float held[R];
#pragma unroll
  for (int u = 0; u < R; ++u) held[u] = p.spart[min((int64_t)(tid + T * u), p.nvt - 1) * p.ldp + k];
  double sum = 0.;
  bool redone = false;
#pragma unroll
  for (int u = 0; u < R; ++u) {
    const float s = tid + T * u < p.nvt ? held[u] : 0.f;
    redone = redone || s < 0.f;
    sum += (double)s;
  }
#pragma unroll 1
  for (int64_t t = tid + T * R; t < p.nvt; t += T) {
    const float s = p.spart[t * p.ldp + k];
    redone = redone || s < 0.f;
    sum += (double)s;
  }
  redone = __syncthreads_or(redone);
  if (redone) {
    for (int64_t t = tid; t < p.nvt; t += T)
      if (p.spart[t * p.ldp + k] < 0.f) m = fmaxf(m, p.mpart[t * p.ldp + k]);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    if (lane == 0) m_sh[w] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NWV; ++i) m = fmaxf(m, m_sh[i]);
    sum = 0.;
    for (int64_t t = tid; t < p.nvt; t += T) {
      const float s = p.spart[t * p.ldp + k];
      sum += (double)fabsf(s) * exp2((double)((s < 0.f ? p.mpart[t * p.ldp + k] : rf) - m));
    }
  }
  sum = wave_sum(sum);
  if (lane == 0) s_sh[w] = sum;
  if (redone && p.E != nullptr) {
    bf16* e = p.E + k * p.V;
    for (int64_t v = 8 * (int64_t)tid; v < p.V; v += 8 * T) {
      const int64_t t = v / kFewBI;
      const float s = p.spart[t * p.ldp + k], d = (s < 0.f ? p.mpart[t * p.ldp + k] : rf) - m;
      // (in two factors: one alone may leave fp32's range where its products with E, up to 2^60, do not)
      const float f = exp2f_fast(0.5f * d);
      bf16x8 x = ld_bf16x8(e + v);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (bf16)((float)x[i] * f * f);
      st_bf16x8(e + v, x);
    }
  }
  __syncthreads();  // (E is behind it, too: the listed tokens' gradients go there next)
  if (w == 0) {
    sum = 0.;
#pragma unroll
    for (int i = 0; i < NWV; ++i) sum += s_sh[i];
    const float f = row_math(p, k, counted, sum, m);
    if (lane == 0) f_sh = f;
  }
  if (p.H != nullptr) {
    __syncthreads();
    const float f = f_sh;
    for (int64_t c = 8 * (int64_t)tid; c < p.hdim; c += 8 * T) {
      bf16x8 x = ld_bf16x8(p.H + k * p.hdim + c);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = (bf16)((float)x[i] * f);
      st_bf16x8(p.H + k * p.hdim + c, x);
    }
  }
}

// ---------------------------------------------------------------- host
struct Layout {
  size_t loss, bad, spart, mpart, ids, lt, zk, mask, base, len, rsum, rtop, f0, w0, at, f, wt, E, part, acc32, rows, hc, yc,
      ref, keys, slot, next, lsum, total;
  int64_t chunk, nchunks, nvt, ldm, ldb;
  int ldk, vt, splits, prow, run, nsort;
  bool few;
};

// Loss alone: chunks bound what is held for a row besides (tile sums, lists).
constexpr int64_t kLossChunk = 16384;

Layout layout(int64_t n, int64_t hdim, int64_t V, int top_k, int64_t chunk, bool grads, bool need_dw) {
  Layout L{};
  need_dw = need_dw && grads;
  L.chunk = std::max<int64_t>(std::min(grads ? chunk : kLossChunk, n), 1);
  L.nchunks = (n + L.chunk - 1) / L.chunk;
  L.few = L.chunk <= kFewRows;
  L.vt = L.few ? kFewBI : kVT;
  L.nvt = (V + L.vt - 1) / L.vt;
  L.ldk = top_k + 1;
  L.ldm = L.nvt * L.vt / 8;
  L.ldb = L.nvt * (L.vt / list_lane_bits(L.few));
  const size_t rows = (size_t)std::max<int64_t>(n, 1), npad = (rows + 255) / 256 * 256, nc = (size_t)L.chunk;
  size_t off = 512;  // nvalid, an unused factor
  auto take = [&](bool on, size_t bytes) {
    const size_t at = off;
    if (on) off += al(bytes);
    return at;
  };
  L.loss = take(true, 3 * sizeof(double) * rows);
  L.bad = take(true, sizeof(int32_t) * rows);
  L.spart = take(true, sizeof(float) * nc * L.nvt);
  L.mpart = take(true, sizeof(float) * nc * L.nvt);
  L.ids = take(true, sizeof(int32_t) * nc * L.ldk);
  L.lt = take(true, sizeof(float) * nc * L.ldk);
  L.zk = take(true, sizeof(float) * nc * L.ldk);
  L.mask = take(true, nc * L.ldm);
  L.base = take(true, nc * L.ldb);
  L.len = take(true, sizeof(int32_t) * nc);
  L.rsum = take(true, sizeof(float) * nc);
  L.rtop = take(true, sizeof(float) * nc);
  L.f0 = take(grads, sizeof(float) * nc);
  L.w0 = take(grads, sizeof(float) * nc);
  L.at = take(grads, sizeof(int64_t) * nc);
  L.f = take(need_dw, sizeof(float) * nc);
  L.wt = take(need_dw, sizeof(float) * nc);
  L.E = take(grads, sizeof(bf16) * nc * (size_t)V);
  L.splits = L.few ? few_splits(hdim, V) : dh_splits(hdim, L.chunk);
  L.prow = (int)std::min<int64_t>(L.chunk, BJ);
  L.run = dh_run(V);
  int64_t slots = grads && L.few ? L.splits : 0;
  if (grads && !L.few && L.splits > 1)
    for (int64_t c0 = 0; c0 < n; c0 += L.chunk)
      slots = std::max(slots, dh_slots(c0, std::min(L.chunk, n - c0), (int)((hdim + BI - 1) / BI), L.splits, L.run));
  L.part = take(slots > 0, sizeof(float) * (size_t)(slots * L.prow * hdim));
  L.acc32 = take(need_dw && L.nchunks > 1, sizeof(float) * (size_t)(V * hdim));
  L.rows = take(true, sizeof(int32_t) * npad);
  L.hc = take(true, sizeof(bf16) * npad * (size_t)hdim);
  L.yc = take(true, sizeof(int64_t) * npad);
  L.ref = take(true, sizeof(float) * npad);
  L.nsort = need_dw ? (int)((L.chunk + kIdChunk - 1) / kIdChunk) : 0;
  L.keys = take(need_dw, sizeof(uint64_t) * (size_t)L.nsort * kIdChunk);
  L.slot = take(need_dw, sizeof(int32_t) * (size_t)V);
  L.next = take(need_dw, sizeof(int32_t) * (size_t)L.nsort * kIdChunk);
  L.lsum = take(need_dw, sizeof(float) * nc * (size_t)hdim);
  L.total = off;
  return L;
}

}  // namespace

size_t distill_workspace_bytes(int64_t n, int64_t hdim, int64_t vocab, int top_k, int64_t chunk, bool grads, bool need_dw) {
  return layout(n, hdim, vocab, top_k, chunk, grads, need_dw).total;
}

hipError_t distill_run(const DistillArgs& a, hipStream_t stream) {
  const bool need_dw = a.grads && a.dweight != nullptr;
  const Layout L = layout(a.n, a.hdim, a.vocab, a.top_k, a.chunk, a.grads, need_dw);
  int64_t* nvalid = at<int64_t>(a.ws, 0);
  int32_t* rows = at<int32_t>(a.ws, L.rows);
  const float* divisor = a.reduction == 0 ? nullptr : a.divisor;
  CompactArgs c{};
  c.hidden = a.hidden;
  c.weight = a.weight;
  c.labels = a.labels;
  c.n = a.n;
  c.hdim = a.hdim;
  c.vocab = a.vocab;
  c.ignore_index = a.ignore_index;
  c.zscale = (float)(1.4426950408889634 / a.temperature);
  c.rows = rows;
  c.nvalid = nvalid;
  c.count = a.counts;
  c.bad = a.counts + 1;
  c.invden = at<float>(a.ws, 256);
  c.hc = at<bf16>(a.ws, L.hc);
  c.yc = at<int64_t>(a.ws, L.yc);
  c.ref = at<float>(a.ws, L.ref);
  c.dh = a.grads ? a.dhidden : nullptr;
  // all rows in one chunk of the few-rows kernels: fewer launches (4 rows x 64, both directions, 110 -> 90 us; 48 x 896 234 -> 228)
  const bool one_few = L.few && L.nchunks == 1;
  if (!one_few) launch_compact(c, stream);
  for (int64_t c0 = 0; c0 < a.n; c0 += L.chunk) {
    const int64_t nc = std::min(L.chunk, a.n - c0);
    bf16 *Hc = c.hc + c0 * a.hdim, *E = a.grads ? at<bf16>(a.ws, L.E) : nullptr;
    ListArgs ls{};
    ls.ids = a.ids;
    ls.teacher = a.teacher;
    ls.rows = rows + c0;
    ls.y = c.yc + c0;
    ls.nvalid = nvalid;
    ls.out = at<int32_t>(a.ws, L.ids);
    ls.lt = at<float>(a.ws, L.lt);
    ls.mask = at<uint8_t>(a.ws, L.mask);
    ls.base = at<uint8_t>(a.ws, L.base);
    ls.len = at<int32_t>(a.ws, L.len);
    ls.bad = at<int32_t>(a.ws, L.bad) + c0;
    ls.nc = nc;
    ls.c0 = c0;
    ls.V = a.vocab;
    ls.nvt = L.nvt;
    ls.K = a.top_k;
    ls.ldk = L.ldk;
    ls.ldm = L.ldm;
    ls.ldb = L.ldb;
    if (one_few) {
      ls.few.labels = a.labels;
      ls.few.hidden = a.hidden;
      ls.few.weight = a.weight;
      ls.few.rows = rows;
      ls.few.y = c.yc;
      ls.few.nvalid = nvalid;
      ls.few.counts = a.counts;
      ls.few.hc = c.hc;
      ls.few.ref = c.ref;
      ls.few.dh = c.dh;
      ls.few.hdim = a.hdim;
      ls.few.ignore_index = a.ignore_index;
      ls.few.n = (int)a.n;
      ls.few.zscale = c.zscale;
    }
    const dim3 each((unsigned)nc), waves((unsigned)((nc + 3) / 4));
    if (L.few)
      hipLaunchKernelGGL((a.ids32 ? distill_list_kernel<int32_t, true> : distill_list_kernel<int64_t, true>), each,
                         dim3(kListThreads), 0, stream, ls);
    else
      hipLaunchKernelGGL((a.ids32 ? distill_list_kernel<int32_t, false> : distill_list_kernel<int64_t, false>), each,
                         dim3(kListThreads), 0, stream, ls);

    LogitsArgs lg{};
    lg.W = GOp{a.weight, a.hdim, a.vocab, a.hdim};
    lg.H = GOp{Hc, a.hdim, nc, a.hdim};
    lg.y = ls.y;
    lg.ref = c.ref + c0;
    lg.E = E;
    lg.mpart = at<float>(a.ws, L.mpart);
    lg.spart = at<float>(a.ws, L.spart);
    lg.nvalid = nvalid;
    lg.c0 = c0;
    lg.V = a.vocab;
    lg.nc = nc;
    lg.ldp = L.chunk;
    lg.store_e = a.grads ? 1 : 0;
    lg.zscale = c.zscale;
    lg.mask = ls.mask;
    lg.base = ls.base;
    lg.zk = at<float>(a.ws, L.zk);
    lg.ldk = L.ldk;
    lg.ldm = L.ldm;
    lg.ldb = L.ldb;
    lg.slot = one_few && need_dw ? at<int32_t>(a.ws, L.slot) : nullptr;
    launch_logits(lg, L.few, true, stream);

    RowArgs rw{};
    rw.mpart = lg.mpart;
    rw.spart = lg.spart;
    rw.ref = lg.ref;
    rw.y = ls.y;
    rw.E = E;
    rw.nvalid = nvalid;
    rw.c0 = c0;
    rw.nc = nc;
    rw.nvt = L.nvt;
    rw.vlog = tile_log(L.vt);
    rw.V = a.vocab;
    rw.hdim = a.hdim;
    rw.ldp = L.chunk;
    rw.grads = lg.store_e;
    rw.rsum = at<float>(a.ws, L.rsum);
    rw.rtop = at<float>(a.ws, L.rtop);
    if (!L.few) launch_row(rw, false, true, stream);

    RowMathArgs rm{};
    rm.ids = ls.out;
    rm.lt = ls.lt;
    rm.zk = lg.zk;
    rm.len = ls.len;
    rm.ref = lg.ref;
    rm.rsum = rw.rsum;
    rm.rtop = rw.rtop;
    rm.y = ls.y;
    rm.nvalid = nvalid;
    rm.divisor = divisor;
    rm.E = E;
    rm.f = at<float>(a.ws, L.f0);
    rm.w = at<float>(a.ws, L.w0);
    rm.at = at<int64_t>(a.ws, L.at);
    rm.loss = at<double>(a.ws, L.loss);
    rm.nc = nc;
    rm.c0 = c0;
    rm.n = a.n;
    rm.V = a.vocab;
    rm.ldk = L.ldk;
    rm.reverse = a.reverse;
    rm.tail = a.tail;
    rm.c = a.ce_weight;
    rm.inv_t = 1. / a.temperature;
    if (L.few) {
      rm.spart = lg.spart;
      rm.mpart = lg.mpart;
      rm.H = one_few && need_dw ? Hc : nullptr;
      rm.nvt = L.nvt;
      rm.ldp = L.chunk;
      rm.hdim = a.hdim;
      hipLaunchKernelGGL(distill_row_few_kernel, each, dim3(256), 0, stream, rm);
    } else {
      hipLaunchKernelGGL(distill_row_kernel, waves, dim3(256), 0, stream, rm);
    }
    if (!a.grads) continue;

    if (a.dhidden != nullptr || one_few) {
      DhArgs dh{};
      dh.Wt = lg.W;
      dh.E = GOp{E, a.vocab, nc, a.vocab};
      dh.dh = a.dhidden;
      dh.part = at<float>(a.ws, L.part);
      dh.f = rm.f;
      dh.wt = rm.w;
      dh.y = rm.at;
      dh.rows = rows;
      dh.nvalid = nvalid;
      dh.c0 = c0;
      dh.hdim = a.hdim;
      dh.nc = nc;
      dh.splits = L.splits;
      dh.prow = L.prow;
      dh.run = L.run;
      if (L.few) {
        FewSumArgs fs{};
        fs.dh = dh;
        fs.f0 = rm.f;
        fs.w0 = rm.w;
        fs.scale = 1.f;
        if (one_few && need_dw) {
          fs.H = a.hidden;
          fs.lsum = at<float>(a.ws, L.lsum);
          fs.slot = at<int32_t>(a.ws, L.slot);
          fs.next = at<int32_t>(a.ws, L.next);
        }
        launch_dh_few(fs, stream);
      } else {
        launch_dh(dh, stream);
      }
    }
    if (!need_dw) continue;
    if (!one_few) {
      WeighArgs wg{};
      wg.H = a.hidden;
      wg.rows = rows + c0;
      wg.y = rm.at;
      wg.f0 = rm.f;
      wg.w0 = rm.w;
      wg.nvalid = nvalid;
      wg.Hs = Hc;
      wg.f = at<float>(a.ws, L.f);
      wg.wt = at<float>(a.ws, L.wt);
      wg.keys = at<uint64_t>(a.ws, L.keys);
      wg.slot = at<int32_t>(a.ws, L.slot);
      wg.n = a.n;
      wg.nc = nc;
      wg.c0 = c0;
      wg.V = a.vocab;
      wg.hdim = a.hdim;
      wg.ignore_index = a.ignore_index;
      wg.scale = 1.f;
      wg.nsort = L.nsort;
      launch_weigh(wg, stream);
      LabelArgs la{};
      la.keys = wg.keys;
      la.H = a.hidden;
      la.rows = wg.rows;
      la.wt = wg.wt;
      la.lsum = at<float>(a.ws, L.lsum);
      la.slot = wg.slot;
      la.next = at<int32_t>(a.ws, L.next);
      la.hdim = a.hdim;
      la.nsort = L.nsort;
      launch_labels(la, nc, stream);
    }
    DwArgs dw{};
    dw.Ht = GOp{Hc, a.hdim, nc, a.hdim};
    dw.Et = GOp{E, a.vocab, nc, a.vocab};
    dw.slot = at<int32_t>(a.ws, L.slot);
    dw.next = at<int32_t>(a.ws, L.next);
    dw.lsum = at<float>(a.ws, L.lsum);
    dw.dw = a.dweight;
    dw.acc32 = at<float>(a.ws, L.acc32);
    dw.nvalid = nvalid;
    dw.c0 = c0;
    dw.hdim = a.hdim;
    dw.V = a.vocab;
    dw.chunk = L.chunk;
    launch_dw(dw, one_few, stream);
  }
  if (need_dw && a.n == 0) launch_zero(a.dweight, a.vocab * a.hdim, stream);
  LossArgs lo{};
  lo.loss = at<double>(a.ws, L.loss);
  lo.bad = at<int32_t>(a.ws, L.bad);
  lo.nvalid = nvalid;
  lo.divisor = divisor;
  lo.out[0] = a.loss;
  lo.out[1] = a.divergence;
  lo.out[2] = a.cross_entropy;
  lo.total_bad = a.counts + 2;
  lo.n = a.n;
  hipLaunchKernelGGL(distill_loss_kernel, dim3(1), dim3(1024), 0, stream, lo);
  return hipGetLastError();
}

}  // namespace siq

// Token statistics from hidden states, without logits, for gfx950: the
// log-probabilities of given tokens, the entropy of each row's distribution and
// its most probable tokens.
//
// With z = h W^T / temperature and p = softmax(z), by row:
//   logp = ln p_y,   H = -sum_j p_j ln p_j,
//   top  = the K largest z (of equal ones the lower ids), with their ln p;
// and with upstream gradients g of logp and e of H
//   dz_j = g ([j = y] - p_j) - e p_j (ln p_j + H)   (over temperature),
//   dH = dZ W,  dW = dZ^T h.
//
// Forward, per chunk of compacted rows (rows whose label counts):
//  1. logits GEMM (MFMA, 256 x 256 tiles; few rows: 128 columns of W).  The
//     epilogue leaves, per row and part of 128 columns, the maximum m, the sum of
//     2^(z2 - m) and the sum of 2^(z2 - m) (z2 - m), in log2 units: what both
//     the logsumexp and the entropy are merged from, without any reference that
//     a row could exceed.  The given token is kept out of them, so that what is
//     next to certain keeps its digits, and added in the row pass.  With
//     alternatives wanted it also writes z itself in fp32 and the part's largest z:
//     first for an eighth of the columns, whose K-th largest part bounds what can be
//     among the K largest of all, then for the parts of the others that reach that.
//  2. row pass, a workgroup a row: merges in 64 bits; logp, H, lse.  The K-th
//     largest of the maxima of 256 groups of parts is a bound that the K largest z
//     do not lie below, so of z only the parts that reach it are read.
//
// Backward: lse and H are known.  Where the forward could keep 2^(z2 - m) in bf16,
// one pass over that makes dZ; otherwise the logits GEMM, made again, writes it.
// The given token is left out: its term is added in fp32 by the products' kernels.
// The two gradient products follow.
//
// Whole calls over 151936 columns: one row x 896 with 20 alternatives 61 us, of which
// the table is read in 43 (6.3 TB/s); 5670 counted rows x 1536 with 64 alternatives
// 2.48 ms, the logits alone 2.14 (1.24 PFLOP/s); 1279 counted rows x 1536, frozen
// head, 1.33 ms, of it 0.16 the pass over what was kept; 2755 x 896 in full training
// 2.60 ms.
#include <algorithm>

#include "few.h"
#include "flce_launch.h"
#include "gemm.h"
#include "ids.h"
#include "token_stats.h"

namespace siq {

namespace {

using namespace gemm;

// ---------------------------------------------------------------- logits
struct StatLogitsArgs {
  GOp W, H;               // W [V, hdim], H = compacted rows of the chunk [nc, hdim]
  const int64_t* y;       // [nc]
  float* Z;               // [nc, V] z before the temperature, or nullptr
  bf16* E;                // [nc, V] 2^(z2 - m), 0 for the given token, or nullptr
  f32x4* part;            // [nc, parts] {m, sum, sum of products, largest z (before the temperature)}
  float* zy;              // [nc] z of the given token
  const float* bound;     // [nc] parts whose largest z is below are not written to Z, or nullptr
  const int64_t* nvalid;  // nullptr: few rows that were not compacted, whose labels are counted here
  int64_t *count, *bad;
  int64_t ignore_index;
  int64_t V, nc, c0, parts;
  int nI, nJ, t0;         // tiles of columns of this launch, and the first one
  float zscale;           // log2(e) / temperature
};

// The largest of NA x 16 accumulators of a lane and of its other half.
template <int NA, class Get>
__device__ __forceinline__ float stat_max(Get z) {
  float m = -INFINITY;
#pragma unroll
  for (int a = 0; a < NA; ++a)
#pragma unroll
    for (int r = 0; r < 16; ++r) m = fmaxf(m, z(a, r));
  return half_max(m);
}

// {m, s, t, -} of them: the sums of 2^(z2 - m) and of 2^(z2 - m) (z2 - m) with z2 =
// z zscale; keep(a, j, e): the terms of accumulators 8 j .. of block a.
template <int NA, class Get, class Keep>
__device__ __forceinline__ f32x4 stat_part(float zscale, float m, Get z, Keep keep) {
  const float base = m == -INFINITY ? 0.f : m;
  float s = 0.f, t = 0.f;
#pragma unroll
  for (int a = 0; a < NA; ++a)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      bf16x8 e8;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = __builtin_fmaf(z(a, 8 * j + i), zscale, -base), e = exp2f_fast(x);
        s += e;
        // (2^-1e4 is 0: masked columns, and those at minus infinity, add nothing)
        t = __builtin_fmaf(e, fmaxf(x, -1e4f), t);
        e8[i] = (bf16)e;
      }
      keep(a, j, e8);
    }
  return f32x4{m, half_sum(s), half_sum(t), 0.f};
}

// TOP: Z is written; KEEP: E is.  Bounded by the matrix cores and, as nothing covers
// it, a tile's epilogue of 65536 exponentials: 1279 rows x 1536 that keep E 0.51-0.61 ms
// (1.0-1.16 PFLOP/s), 2755 x 896 0.75-0.82 (0.9-1.0).  Parts are 64 columns of a
// wave, so a part's sums need no other wave's.
template <bool TOP, bool KEEP>
__global__ __launch_bounds__(NT) void stats_logits_kernel(const StatLogitsArgs p) {
  __shared__ __align__(16) bf16 smem[SMEM];
  int ti, tj;
  if (!tile_of(p.nI, p.nJ, 4, ti, tj)) return;
  ti += p.t0;
  const int64_t i0 = (int64_t)ti * BI, j0 = (int64_t)tj * BJ;
  if (j0 >= *p.nvalid - p.c0) return;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, h = lane >> 5, l32 = lane & 31;
  const int wi = w & 1, wj = w >> 1;
  // accumulator (a, b, r) holds z of column vbase + wave_row(a, wi) + 16 (r / 8) + (r % 8), row j0 + wave_col(b, wj) + l32
  const int64_t vbase = i0 + 8 * h;
  int rel[2];  // the given tokens' offsets from the tile (-1: elsewhere)
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const int64_t d = p.y[min(j0 + wave_col(b, wj) + l32, p.nc - 1)] - vbase;
    rel[b] = d >= 0 && d < 256 ? (int)d : -1;
  }
  f32x16 acc[4][2];
  gemm_core<true, true, false>(smem, p.W, p.H, i0, j0, 0, p.W.cols, acc);
  if (i0 + BI > p.V) {
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (vbase + wave_row(a, wi) + 16 * (r >> 3) + (r & 7) >= p.V) acc[a][b][r] = -INFINITY;
  }
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const int64_t tok = j0 + wave_col(b, wj) + l32;
    const bool tv = tok < p.nc;
    auto get = [&](int a, int r) { return acc[a][b][r]; };
    const float top = stat_max<4>(get);
    float largest = top;
    if (TOP && tv && (p.bound == nullptr || top >= p.bound[tok])) {
#pragma unroll
      for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int jj = 0; jj < 2; ++jj) {
          const int64_t v0 = vbase + wave_row(a, wi) + 16 * jj;
          if (v0 >= p.V) continue;
          f32x4 lo, hi;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            lo[i] = acc[a][b][8 * jj + i];
            hi[i] = acc[a][b][8 * jj + 4 + i];
          }
          float* z = p.Z + tok * p.V + v0;
          *reinterpret_cast<f32x4*>(z) = lo;
          *reinterpret_cast<f32x4*>(z + 4) = hi;
        }
    }
    // the given token: in at most one lane of the workgroup, for one tile in ~600
    const bool hit = tv && rel[b] >= 0 && ((rel[b] >> 6) & 1) == wi && ((rel[b] >> 3) & 1) == 0;
    if (__any(hit)) {
      const int r0 = rel[b] - 64 * wi;
      float zsel = 0.f;
#pragma unroll
      for (int a = 0; a < 4; ++a)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (hit && r0 == wave_row(a, 0) + 16 * (r >> 3) + (r & 7)) {
            zsel = acc[a][b][r];
            acc[a][b][r] = -INFINITY;
          }
      if (hit) p.zy[tok] = zsel;
      largest = stat_max<4>(get);
    }
    f32x4 st = stat_part<4>(p.zscale, largest * p.zscale, get, [&](int a, int j, const bf16x8& e) {
      const int64_t v0 = vbase + wave_row(a, wi) + 16 * j;
      if (KEEP && tv && v0 < p.V) st_bf16x8(p.E + tok * p.V + v0, e);
    });
    st[3] = top;
    if (tv && h == 0) p.part[tok * p.parts + 2 * ti + wi] = st;
  }
}

// The main loop of a few-rows product: 128 rows of W (32 a wave) x 32 NB rows of the
// call; accumulator r of block b: column i0 + 32 w + 8 h + 16 (r / 8) + r % 8, row
// 32 b + l32.
template <int NB, int STAGES>
__device__ __forceinline__ void few_logits(bf16* smem, const GOp& W, const GOp& H, int64_t i0, f32x16 (&acc)[NB]) {
  constexpr int TOK = 32 * NB, STAGE = (kFewBI + TOK) * BK, NWV = kFewThreads / 64;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, wu = __builtin_amdgcn_readfirstlane(w);
  FewRows<kFewBI, NWV> la;
  FewRows<TOK, NWV> lb;
  la.init(W.ld, W.rows - 1 - i0, lane, w);
  lb.init(H.ld, H.rows - 1, lane, w);
  const bf16 *wb = W.base + i0 * W.ld, *hb = H.base;
  HalfRead<true, true, 1> ra;
  HalfRead<true, false, NB> rb;
  ra.init(lane, 32 * w);
  rb.init(lane, 0);
#pragma unroll
  for (int b = 0; b < NB; ++b) acc[b] = zero16();
  few_steps<STAGES, la.PER + lb.PER>(
      (int)(W.cols / BK),
      [&](int s, int buf) {
        bf16* st = smem + buf * STAGE;
        lb.issue(hb + (int64_t)s * BK, st + kFewBI * BK, wu);
        la.issue(wb + (int64_t)s * BK, st, wu);
      },
      [&](int, int buf) {
        const bf16 *A = smem + buf * STAGE, *B = A + kFewBI * BK;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          const bf16x8 a = ra.read(A, 0, ks);
#pragma unroll
          for (int b = 0; b < NB; ++b) acc[b] = mfma32(a, rb.read(B, b, ks), acc[b]);
        }
      });
}

template <int NB>
constexpr int kFewStages = NB <= 2 ? 3 : 2;  // (64 rows: three buffers; 128: two, for two workgroups a CU)
template <int NB>
constexpr int kFewSmem = kFewStages<NB> * (kFewBI + 32 * NB) * BK;

// Bounded by memory: over 151936 x 896 one row 43 us (272 MB, 6.3 TB/s), 61 rows with Z
// 62 us (309 MB, 4.9 TB/s: a copy's rate, reads and writes mixed).
template <int NB, bool TOP, bool KEEP>
__global__ __launch_bounds__(kFewThreads) void stats_logits_few_kernel(const StatLogitsArgs p) {
  constexpr int TOK = 32 * NB, NWV = kFewThreads / 64;
  // behind the last step's barrier: the waves' maxima and sums, and z, which leaves by whole rows of the tile
  constexpr int RED = 6 * NWV * TOK * 2, BYTES2 = RED + (TOP ? TOK * kFewBI * 2 : 0);
  __shared__ __align__(16) bf16 smem[BYTES2 > kFewSmem<NB> ? BYTES2 : kFewSmem<NB>];
  const int64_t i0 = (int64_t)blockIdx.x * kFewBI;
  if (p.nvalid != nullptr && *p.nvalid <= p.c0) return;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, h = lane >> 5, l32 = lane & 31;
  if (p.nvalid == nullptr && blockIdx.x == 0 && w == 0) {
    // (by the first of many workgroups: where the host's memory takes the counts, the others hide how long that takes)
    int64_t n = 0, bad = 0;
    for (int g = 0; g < (int)p.nc; g += 64) {
      const int64_t v = g + lane < (int)p.nc ? p.y[g + lane] : p.ignore_index;
      const bool ok = v >= 0 && v < p.V;
      n += __popcll(__ballot(v != p.ignore_index && ok));
      bad += __popcll(__ballot(v != p.ignore_index && !ok));
    }
    if (lane == 0) {
      *p.count = n;
      *p.bad = bad;
    }
  }
  const int64_t vbase = i0 + 32 * w + 8 * h;
  int rel[NB];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int64_t d = p.y[min((int64_t)(32 * b + l32), p.nc - 1)] - vbase;
    rel[b] = d >= 0 && d < 32 && (d & 8) == 0 ? (int)d : -1;
  }
  f32x16 acc[NB];
  few_logits<NB, kFewStages<NB>>(smem, p.W, p.H, i0, acc);
  if (i0 + kFewBI > p.V) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (vbase + 16 * (r >> 3) + (r & 7) >= p.V) acc[b][r] = -INFINITY;
  }
  float* zt = reinterpret_cast<float*>(smem + RED);  // [TOK][128], 16-byte chunk c of row r at c ^ (r % 32)
  float *max_sh = reinterpret_cast<float*>(smem), *top_sh = max_sh + NWV * TOK;  // [NWV][TOK]
  f32x4* red = reinterpret_cast<f32x4*>(smem) + 2 * NWV * TOK / 4;               // [NWV][TOK]
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int64_t tok = 32 * b + l32;
    const bool tv = tok < p.nc;
    if (TOP) {
#pragma unroll
      for (int jj = 0; jj < 2; ++jj) {
        f32x4 lo, hi;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          lo[i] = acc[b][8 * jj + i];
          hi[i] = acc[b][8 * jj + 4 + i];
        }
        const int c = 8 * w + 4 * jj + 2 * h;
        *reinterpret_cast<f32x4*>(zt + tok * kFewBI + 4 * (c ^ l32)) = lo;
        *reinterpret_cast<f32x4*>(zt + tok * kFewBI + 4 * ((c + 1) ^ l32)) = hi;
      }
    }
    auto get = [&](int, int r) { return acc[b][r]; };
    const float top = stat_max<1>(get);
    float largest = top;
    const bool hit = tv && rel[b] >= 0;
    if (__any(hit)) {
      float zsel = 0.f;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (hit && rel[b] == 16 * (r >> 3) + (r & 7)) {
          zsel = acc[b][r];
          acc[b][r] = -INFINITY;
        }
      if (hit) p.zy[tok] = zsel;
      largest = stat_max<1>(get);
    }
    if (h == 0) {
      max_sh[w * TOK + 32 * b + l32] = largest;
      top_sh[w * TOK + 32 * b + l32] = top;
    }
  }
  __syncthreads();
  if (TOP) {
    const int rows = (int)min(p.nc, (int64_t)TOK), c = tid % 32;
    if (i0 + 4 * c < p.V)
      for (int r = tid / 32; r < rows; r += kFewThreads / 32)
        *reinterpret_cast<f32x4*>(p.Z + r * p.V + i0 + 4 * c) =
            *reinterpret_cast<const f32x4*>(zt + r * kFewBI + 4 * (c ^ (r & 31)));
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int64_t tok = 32 * b + l32;
    float m = -INFINITY;
#pragma unroll
    for (int k = 0; k < NWV; ++k) m = fmaxf(m, max_sh[k * TOK + tok]);
    const f32x4 st = stat_part<1>(p.zscale, m * p.zscale, [&](int, int r) { return acc[b][r]; },
                                  [&](int, int j, const bf16x8& e) {
                                    const int64_t v0 = vbase + 16 * j;
                                    if (KEEP && tok < p.nc && v0 < p.V) st_bf16x8(p.E + tok * p.V + v0, e);
                                  });
    if (h == 0) red[w * TOK + tok] = st;
  }
  __syncthreads();
  // a thread a row of the call: the tile's
  if (tid >= TOK || tid >= p.nc) return;
  f32x4 x = red[tid];
  x[3] = top_sh[tid];
#pragma unroll
  for (int k = 1; k < NWV; ++k) {
    x[1] += red[k * TOK + tid][1];
    x[2] += red[k * TOK + tid][2];
    x[3] = fmaxf(x[3], top_sh[k * TOK + tid]);
  }
  p.part[tid * p.parts + blockIdx.x] = x;
}

// ---------------------------------------------------------------- row pass
struct StatRowArgs {
  const f32x4* part;      // [nc, parts]
  const float* zy;        // [nc]
  const float* Z;         // [nc, V], where a part's largest reaches the bound
  const float* bound;     // [nc] or nullptr
  const int32_t* rows;    // [nc] compacted row -> row, or nullptr: nothing was compacted (a call of few rows)
  const int64_t* nvalid;
  const int64_t* labels;  // [n]
  float *logp, *entropy;  // [n] by row
  float* state;           // [3, n] or nullptr
  float* top_logp;        // [n, K]
  int64_t* top_ids;
  int64_t n, c0, V, ignore_index;
  int parts, K;
  bool few;               // parts of 128 columns in a row, or twice 64 of a tile
  float zscale;
};

// Larger numbers have larger keys, equal ones (both zeros) equal keys; NaN is above all.
__device__ __forceinline__ uint32_t order_of(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return x != x ? 0xffffffffu : b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float number_of(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu));
}
// ... of a column: of equal numbers the lower column is larger.
__device__ __forceinline__ uint64_t order_of(float x, int64_t v) { return (uint64_t)order_of(x) << 32 | (uint32_t)~v; }

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x += __shfl_xor(x, o);
  return x;
}

constexpr int kCus = 256;
constexpr int kRowGroups = 256;               // threads of a workgroup, and groups of parts
constexpr int kMostParts = 1024, kMostListed = 1024;
static_assert(kMaxTopK <= kRowGroups, "a bound is the K-th largest group's");

// The K-th largest of the keys of 256 groups in LDS (behind a barrier), without its last
// eight bits, two bits at a time, by one wave.  (Every thread counting the keys above its
// own: 2.47 -> 2.54 ms at 8192 rows.)
__device__ __forceinline__ uint32_t kth_largest(const uint32_t* best_sh, int K, int lane) {
  constexpr int N = kRowGroups / 64;
  uint32_t b[N], tau = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) b[i] = best_sh[64 * i + lane];
#pragma unroll 1
  for (int bit = 30; bit >= 8; bit -= 2) {
    int c[3] = {0, 0, 0};
#pragma unroll
    for (int q = 0; q < 3; ++q)
#pragma unroll
      for (int i = 0; i < N; ++i) c[q] += __popcll(__ballot(b[i] >= (tau | (uint32_t)(q + 1) << bit)));
    tau |= (uint32_t)(c[2] >= K ? 3 : c[1] >= K ? 2 : c[0] >= K ? 1 : 0) << bit;
  }
  return tau;
}

// ... as a number (none, or what lost bits fell below: minus infinity).
__device__ __forceinline__ float bound_of(uint32_t tau) {
  return tau < 0x007fffffu ? -INFINITY : number_of(tau);
}

// The bound that the first `parts` parts of a row give.
struct BoundArgs {
  const f32x4* part;      // [nc, ld]
  float* bound;           // [nc]
  const int64_t* nvalid;
  int64_t c0, ld;
  int parts, K;
};
__global__ __launch_bounds__(kRowGroups) void stats_bound_kernel(const BoundArgs p) {
  __shared__ __align__(16) uint32_t best_sh[kRowGroups];
  const int64_t k = blockIdx.x;
  if (p.c0 + k >= *p.nvalid) return;
  uint32_t best = 0;
  for (int i = threadIdx.x; i < p.parts; i += kRowGroups) best = max(best, order_of(p.part[k * p.ld + i][3]));
  best_sh[threadIdx.x] = best;
  __syncthreads();
  if (threadIdx.x >= 64) return;
  const uint32_t tau = kth_largest(best_sh, p.K, threadIdx.x);
  if (threadIdx.x == 0) p.bound[k] = bound_of(tau);
}

// One workgroup a row; bounded by its chain of reads and barriers, and by instructions
// that are read for the first time (a row alone 7 us; a branch for each part and column
// 9), many rows by the reads of parts (2755 rows without alternatives: 52 MB in 19 us)
// and of the candidates' logits (3328 rows of 64: 60 us).  Columns that reach the bound are listed, usually K or
// somewhat more, and each one's rank is how many of the others come before it.
// Where they are too many (long ties, or a vocabulary of few parts) the K largest
// are taken one after the other instead.
__global__ __launch_bounds__(kRowGroups) void stats_row_kernel(const StatRowArgs p) {
  constexpr int T = kRowGroups, NWV = T / 64;
  __shared__ float m_sh[NWV];
  __shared__ double s_sh[NWV], t_sh[NWV], lse_sh;
  __shared__ __align__(16) uint32_t best_sh[T];
  __shared__ uint32_t tau_sh;
  __shared__ int part_sh[kMostParts], nparts_sh, n_sh;
  __shared__ uint64_t listed_sh[kMostListed], top_sh[NWV];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t k = blockIdx.x, own = p.c0 + k, y = p.labels[own];
  const bool counts = y != p.ignore_index && y >= 0 && y < p.V;
  if (!counts) {
    if (tid == 0) p.logp[own] = p.entropy[own] = 0.f;
    if (tid < p.K) {
      p.top_logp[own * p.K + tid] = 0.f;
      p.top_ids[own * p.K + tid] = -1;
    }
  }
  if (p.rows == nullptr ? !counts : p.c0 + k >= *p.nvalid) return;
  // the row's parts, read once where there are no more than 1280 (read again for each use: one row 64.1 us in all,
  // 62.3 so; 61 rows 76.2 and 74.4)
  constexpr int R = 5;
  const f32x4* src = p.part + k * p.parts;
  f32x4 held[R];
#pragma unroll
  for (int u = 0; u < R; ++u) held[u] = src[min(tid + T * u, p.parts - 1)];
  auto each_part = [&](auto use) {
#pragma unroll
    for (int u = 0; u < R; ++u)
      if (tid + T * u < p.parts) use(tid + T * u, held[u]);
    for (int i = tid + T * R; i < p.parts; i += T) use(i, src[i]);
  };
  const double dy = (double)p.zy[k] * (double)p.zscale;
  float m = (float)dy;
  uint32_t best = 0;
  each_part([&](int, const f32x4& x) {
    m = fmaxf(m, x[0]);
    best = max(best, order_of(x[3]));
  });
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
  if (lane == 0) m_sh[w] = m;
  best_sh[tid] = best;
  if (tid == 0) nparts_sh = n_sh = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < NWV; ++i) m = fmaxf(m, m_sh[i]);
  double s = 0., t = 0.;
  each_part([&](int, const f32x4& x) {
    if (x[1] == 0.f) return;  // (nothing but minus infinities; a NaN counts)
    // (a factor for the sums of 128 terms: its rounding is that of a sum of so many)
    const float d = x[0] - m, f = exp2f_fast(d);
    s += (double)(x[1] * f);
    t += ((double)x[2] + (double)x[1] * (double)d) * (double)f;
  });
  s = wave_sum(s);
  t = wave_sum(t);
  if (lane == 0) {
    s_sh[w] = s;
    t_sh[w] = t;
  }
  // the bound (parts below an earlier one were not written)
  if (w == 0 && p.K > 0) {
    const uint32_t tau = kth_largest(best_sh, p.K, lane);
    if (tid == 0) tau_sh = p.bound != nullptr ? max(tau, order_of(p.bound[k])) : tau;
  }
  __syncthreads();
  constexpr double kLn2d = 0.6931471805599453;
  const int64_t row = p.rows != nullptr ? p.rows[k] : own;
  if (tid == T - 1) {  // (in a wave that has no bound to find)
    s = t = 0.;
#pragma unroll
    for (int i = 0; i < NWV; ++i) {
      s += s_sh[i];
      t += t_sh[i];
    }
    // the given token: all relative to m
    const double d = dy - (double)m, ey = exp2(d), all = s + ey, l2 = log2(all), lse = (double)m + l2;
    const double over = s * exp2(-d), ent = kLn2d * (l2 - (t + (ey > 0. ? ey * d : 0.)) / all);
    lse_sh = lse;
    // p_y = 1 / (1 + over): its logarithm keeps its digits where `over` is small
    const float lp = (float)(over <= 1e300 ? -log1p(over) : kLn2d * (d - l2)), e = ent < 0. ? 0.f : (float)ent;
    p.logp[row] = lp;
    p.entropy[row] = e;
    if (p.state != nullptr) {
      p.state[row] = (float)lse;
      p.state[p.n + row] = lp;
      p.state[2 * p.n + row] = e;
    }
  }
  if (p.K == 0) return;
  const uint32_t tau = tau_sh;
  const float* z = p.Z + k * p.V;
  auto result = [&](int rank, uint64_t key) {
    const float zi = number_of((uint32_t)(key >> 32));
    p.top_logp[row * p.K + rank] = (float)(((double)zi * (double)p.zscale - lse_sh) * kLn2d);
    p.top_ids[row * p.K + rank] = (int64_t)(uint32_t)~(uint32_t)key;
  };
  // Which of a thread's parts, and of their columns, reach it is a bit each, and a loop lists them: branches of their own
  // each wait for instructions that nothing has run before (90 alternatives of 49152: 18.8 us, 10.8 so; 54 of 151936: 13.1
  // and 8.3).
  auto list_part = [&](int i) {  // (in any order: ranks make one)
    const int at = atomicAdd(&nparts_sh, 1);
    if (at < kMostParts) part_sh[at] = i;
  };
  const float least = bound_of(tau);
  uint32_t reach = 0;
#pragma unroll
  for (int u = 0; u < R; ++u) reach |= tid + T * u < p.parts && held[u][3] >= least ? 1u << u : 0u;
#pragma unroll 1
  for (; reach != 0; reach &= reach - 1) list_part(tid + T * (int)__builtin_ctz(reach));
#pragma unroll 1
  for (int i = tid + T * R; i < p.parts; i += T)
    if (src[i][3] >= least) list_part(i);
  __syncthreads();
  const int np = nparts_sh;
  auto column = [&](int part, int c) {  // the c-th of a part
    return p.few ? 128 * (int64_t)part + c : 256 * (int64_t)(part >> 1) + 64 * (part & 1) + (c & 63) + 128 * (c >> 6);
  };
  if (np <= kMostParts) {
    constexpr int U = 8, STEP = T / 32;  // 64 parts in flight
    for (int q0 = tid / 32; q0 < np; q0 += STEP * U) {
      f32x4 x[U];
      uint32_t there = 0;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int q = q0 + STEP * u;
        const int64_t v = column(part_sh[min(q, np - 1)], 4 * (tid & 31));
        there |= q < np && v < p.V ? 15u << (4 * u) : 0u;
        x[u] = *reinterpret_cast<const f32x4*>(z + min(v, p.V - 4));
      }
      reach = 0;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) reach |= x[u][i] < least ? 0u : 1u << (4 * u + i);  // (what is not a number does)
      reach &= there;
#pragma unroll 1
      for (; reach != 0; reach &= reach - 1) {
        const int b = (int)__builtin_ctz(reach);
        const int64_t vb = column(part_sh[q0 + STEP * (b / 4)], 4 * (tid & 31) + b % 4);
        const int at = atomicAdd(&n_sh, 1);
        if (at < kMostListed) listed_sh[at] = order_of(z[vb], vb);
      }
    }
  }
  __syncthreads();
  const int n = n_sh;
  if (np <= kMostParts && n <= kMostListed) {
    for (int i = tid; i < n; i += T) {
      const uint64_t mine = listed_sh[i];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += listed_sh[j] > mine ? 1 : 0;
      if (rank < p.K) result(rank, mine);
    }
    return;
  }
  uint64_t last = ~0ull;
  for (int r = 0; r < p.K; ++r) {
    uint64_t top = 0;
    for (int i = tid / 128; i < p.parts; i += T / 128) {
      const int64_t v = column(i, tid & 127);
      if (v >= p.V || order_of(src[i][3]) < tau) continue;
      const uint64_t key = order_of(z[v], v);
      if (key < last && key > top) top = key;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      const uint64_t other = __shfl_xor(top, o);
      top = other > top ? other : top;
    }
    if (lane == 0) top_sh[w] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NWV; ++i) top = top_sh[i] > top ? top_sh[i] : top;
    if (tid == 0) result(r, top);
    last = top;
    __syncthreads();
  }
}

// ---------------------------------------------------------------- dZ
struct StatGradArgs {
  GOp W, H;
  const int64_t* y;       // [nc]
  const f32x4* coef;      // [nc] {lse, A, B, -}: dz_j = p_j (A + B log2 p_j)
  bf16* G;                // [nc, V]
  const int64_t* nvalid;
  int64_t V, nc, c0;
  int nI, nJ;
  float zscale;
};

__device__ __forceinline__ float stat_dz(float z, float zscale, const f32x4& c) {
  // (at most 0 but for the lse's own rounding; a probability of 0 times a finite logarithm is 0)
  const float l = fmaxf(__builtin_fmaf(z, zscale, -c[0]), -1e4f);
  return exp2f_fast(l) * __builtin_fmaf(c[2], l, c[1]);
}

__global__ __launch_bounds__(NT) void stats_grad_kernel(const StatGradArgs p) {
  __shared__ __align__(16) bf16 smem[SMEM];
  int ti, tj;
  if (!tile_of(p.nI, p.nJ, 4, ti, tj)) return;
  const int64_t i0 = (int64_t)ti * BI, j0 = (int64_t)tj * BJ;
  if (j0 >= *p.nvalid - p.c0) return;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, h = lane >> 5, l32 = lane & 31;
  const int wi = w & 1, wj = w >> 1;
  const int64_t vbase = i0 + 8 * h;
  f32x16 acc[4][2];
  gemm_core<true, true, false>(smem, p.W, p.H, i0, j0, 0, p.W.cols, acc);
#pragma unroll
  for (int b = 0; b < 2; ++b) {
    const int64_t tok = j0 + wave_col(b, wj) + l32;
    if (tok >= p.nc) continue;
    const f32x4 c = p.coef[tok];
    const int64_t y = p.y[tok] - vbase;
#pragma unroll
    for (int a = 0; a < 4; ++a)
#pragma unroll
      for (int jj = 0; jj < 2; ++jj) {
        const int v0 = wave_row(a, wi) + 16 * jj;
        if (vbase + v0 >= p.V) continue;
        bf16x8 g;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float x = stat_dz(acc[a][b][8 * jj + i], p.zscale, c);
          g[i] = (bf16)(y == v0 + i ? 0.f : x);
        }
        st_bf16x8(p.G + tok * p.V + vbase + v0, g);
      }
  }
}

template <int NB>
__global__ __launch_bounds__(kFewThreads) void stats_grad_few_kernel(const StatGradArgs p) {
  __shared__ __align__(16) bf16 smem[kFewSmem<NB>];
  const int64_t i0 = (int64_t)blockIdx.x * kFewBI;
  if (*p.nvalid <= p.c0) return;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, h = lane >> 5, l32 = lane & 31;
  const int64_t vbase = i0 + 32 * w + 8 * h;
  f32x16 acc[NB];
  few_logits<NB, kFewStages<NB>>(smem, p.W, p.H, i0, acc);
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int64_t tok = 32 * b + l32;
    if (tok >= p.nc) continue;
    const f32x4 c = p.coef[tok];
    const int64_t y = p.y[tok] - vbase;
#pragma unroll
    for (int jj = 0; jj < 2; ++jj) {
      if (vbase + 16 * jj >= p.V) continue;
      bf16x8 g;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = stat_dz(acc[b][8 * jj + i], p.zscale, c);
        g[i] = (bf16)(y == 16 * jj + i ? 0.f : x);
      }
      st_bf16x8(p.G + tok * p.V + vbase + 16 * jj, g);
    }
  }
}

// What a row's gradient needs of the forward's results and of the upstream
// gradients: {lse, A, B} as above, and the given token's own dz (in 32 bits),
//   A = -(g + e H) / T,  B = -e ln 2 / T,  dz_y = (g (1 - p_y) - e p_y (ln p_y + H)) / T.
struct StatCoefArgs {
  const int32_t* rows;    // [nc]
  const int64_t* nvalid;
  const float *state, *g, *e;  // [3, n], [n], [n]; g and e may be nullptr
  f32x4* coef;            // [nc]
  float *f, *w;           // [nc]: 1, dz_y
  int64_t n, nc, c0;
  float inv_t;
};
__device__ __forceinline__ f32x4 stat_coef(const StatCoefArgs& p, int64_t k, float& dzy) {
  const int64_t row = p.rows[k];
  const float lse = p.state[row], lp = p.state[p.n + row], hh = p.state[2 * p.n + row];
  const float g = (p.g != nullptr ? p.g[row] : 0.f) * p.inv_t, e = (p.e != nullptr ? p.e[row] : 0.f) * p.inv_t;
  const float py = expf(lp);
  dzy = -g * expm1f(lp) - (e != 0.f ? e * py * (fmaxf(lp, -1e4f) + hh) : 0.f);
  return f32x4{lse, -__builtin_fmaf(e, hh, g), -e * kLn2, 0.f};
}

__global__ __launch_bounds__(256) void stats_coef_kernel(const StatCoefArgs p) {
  const int64_t k = (int64_t)blockIdx.x * 256 + threadIdx.x, nv = min(p.nc, *p.nvalid - p.c0);
  if (k >= p.nc) return;
  if (k >= nv) {  // dZ of the rows that fill up dW's last k-step is 0 (dW multiplies it with zeros, which a NaN would survive)
    p.coef[k] = f32x4{0.f, 0.f, 0.f, 0.f};
    return;
  }
  p.coef[k] = stat_coef(p, k, p.w[k]);
  p.f[k] = 1.f;
}


// dZ from the numerators that the forward kept, a workgroup 2048 columns of a row;
// the rows that fill up dW's last k-step are zeroed, and dH of rows whose label does
// not count.  It reads and writes 2 bytes an element where the logits take 2 hdim flops:
// 2755 rows 334 us (1.67 GB, 5.0 TB/s, a copy's rate), the logits' product 750 again.
struct UnpackArgs {
  StatCoefArgs c;
  const bf16* E;          // [nc, V]
  const f32x4* part;      // [nc, parts]
  bf16* G;                // [nc, V]
  const int64_t* labels;  // [n]
  bf16* dh;               // or nullptr
  int64_t V, hdim, ignore_index;
  int parts;
  bool few;
  // ONE_FEW: what launch_weigh leaves otherwise
  const bf16* H;          // [n, hdim]
  bf16* Hs;               // [nc, hdim] the counted rows
  int32_t* slot;          // [V] cleared
};
constexpr int kUnpackCols = 2048;
// ONE_FEW: few rows in one chunk, with dW; it makes the rows' coefficients, too.  (For
// many rows that costs more than a launch: each workgroup would wait for them, 2048 x 1536
// 1.35 -> 1.40 ms, 4099 x 896 2.62 -> 2.75 ms.)
template <bool ONE_FEW>
__global__ __launch_bounds__(256) void stats_unpack_kernel(const UnpackArgs p) {
  const int64_t nc = p.c.nc, nv = min(nc, *p.c.nvalid - p.c.c0), v = (int64_t)blockIdx.x * kUnpackCols + 8 * threadIdx.x;
  if (ONE_FEW && blockIdx.y == 0)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (v + i < p.V) p.slot[v + i] = 0;
  for (int64_t k = blockIdx.y; k < nc; k += gridDim.y) {
    if (blockIdx.x == 0) {
      const int64_t row = p.c.c0 + k, y = p.labels[row], src = ONE_FEW && k < nv ? p.c.rows[k] : 0;
      const bool clear = p.dh != nullptr && (y == p.ignore_index || y < 0 || y >= p.V);
      if (clear || ONE_FEW)
        for (int64_t c = 8 * (int64_t)threadIdx.x; c < p.hdim; c += 8 * 256) {
          if (clear) st_bf16x8(p.dh + row * p.hdim + c, zero_bf16x8());
          if (ONE_FEW) st_bf16x8(p.Hs + k * p.hdim + c, k < nv ? ld_bf16x8(p.H + src * p.hdim + c) : zero_bf16x8());
        }
    }
    if (k >= (nv + BK - 1) / BK * BK) continue;
    bf16x8 g = zero_bf16x8();
    if (k < nv) {
      f32x4 c;
      if constexpr (ONE_FEW) {
        float dzy;
        c = stat_coef(p.c, k, dzy);
        if (blockIdx.x == 0 && threadIdx.x == 0) {
          p.c.f[k] = 1.f;
          p.c.w[k] = dzy;
        }
      } else {
        c = p.c.coef[k];
      }
      if (v >= p.V) continue;
      const bf16x8 e = ld_bf16x8(p.E + k * p.V + v);
      const int64_t part = p.few ? v / kFewBI : 2 * (v / kVT) + (v >> 6 & 1);
      // (minus infinity: a part of nothing else)
      const float d = fmaxf(p.part[k * p.parts + part][0] - c[0], -1e4f), f = exp2f_fast(d), a = __builtin_fmaf(c[2], d, c[1]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = (float)e[i];
        g[i] = (bf16)(x * f * __builtin_fmaf(c[2], fmaxf(__log2f(x), -1e4f), a));
      }
    }
    if (v < p.V) st_bf16x8(p.G + k * p.V + v, g);
  }
}

// ---------------------------------------------------------------- host
// Rows at a time: with alternatives, z of one chunk takes at most 2 GiB; without
// them the tiles' sums alone bound it.
int64_t stats_chunk(int64_t n, int64_t V, int top_k) {
  const int64_t most = top_k > 0 ? std::max<int64_t>((int64_t(1) << 31) / (4 * V) / BJ * BJ, BJ) : 16384;
  return std::max<int64_t>(std::min(n, most), 1);
}

// What the forward keeps for the backward.
struct StatsSaved {
  size_t nvalid, rows, yc, part, E, total;
  int64_t parts;
};
StatsSaved saved_layout(int64_t n, int64_t V) {
  StatsSaved S{};
  const size_t npad = (size_t)((std::max<int64_t>(n, 1) + 255) / 256 * 256);
  S.parts = n <= kFewRows ? (V + kFewBI - 1) / kFewBI : 2 * ((V + kVT - 1) / kVT);
  S.rows = 256;
  S.yc = S.rows + al(sizeof(int32_t) * npad);
  S.part = S.yc + al(sizeof(int64_t) * npad);
  S.E = S.part + al(sizeof(f32x4) * (size_t)(n * S.parts));
  S.total = S.E + al(sizeof(bf16) * (size_t)(n * V));
  return S;
}

struct FwdLayout {
  size_t scal, rows, yc, ref, hc, zy, part, bound, Z, total;
  int64_t chunk, parts;
  bool few;
};
FwdLayout fwd_layout(int64_t n, int64_t hdim, int64_t V, int top_k, bool keep) {
  FwdLayout L{};
  L.chunk = stats_chunk(n, V, top_k);
  L.few = L.chunk <= kFewRows;
  L.parts = L.few ? (V + kFewBI - 1) / kFewBI : 2 * ((V + kVT - 1) / kVT);
  const size_t npad = (size_t)((std::max<int64_t>(n, 1) + 255) / 256 * 256);
  size_t off = 256;  // scal: nvalid, an unused factor
  auto take = [&](bool on, size_t bytes) {
    const size_t at = off;
    if (on) off += al(bytes);
    return at;
  };
  L.rows = take(!keep, sizeof(int32_t) * npad);
  L.yc = take(!keep, sizeof(int64_t) * npad);
  L.ref = take(true, sizeof(float) * npad);
  L.hc = take(true, sizeof(bf16) * npad * (size_t)hdim);
  L.zy = take(true, sizeof(float) * (size_t)L.chunk);
  L.part = take(!keep, sizeof(f32x4) * (size_t)(L.chunk * L.parts));
  L.bound = take(top_k > 0, sizeof(float) * (size_t)L.chunk);
  L.Z = take(top_k > 0, sizeof(float) * (size_t)(L.chunk * V));
  L.total = off;
  return L;
}

struct BwdLayout {
  size_t scal, rows, yc, ref, hc, coef, f0, w0, f, wt, E, part, acc32, keys, slot, next, lsum, total;
  int64_t chunk, nchunks;
  int splits, prow, run, nsort;
  bool few;
};
BwdLayout bwd_layout(int64_t n, int64_t hdim, int64_t V, int64_t chunk, bool need_dw, bool have) {
  BwdLayout L{};
  L.chunk = std::max<int64_t>(std::min(chunk, n), 1);
  L.nchunks = (n + L.chunk - 1) / L.chunk;
  L.few = L.chunk <= kFewRows;
  const size_t npad = (size_t)((std::max<int64_t>(n, 1) + 255) / 256 * 256);
  size_t off = 256;  // scal: nvalid, count, bad labels, an unused factor
  auto take = [&](bool on, size_t bytes) {
    const size_t at = off;
    if (on) off += al(bytes);
    return at;
  };
  L.rows = take(!have, sizeof(int32_t) * npad);
  L.yc = take(!have, sizeof(int64_t) * npad);
  L.ref = take(!have, sizeof(float) * npad);
  L.hc = take(!have || need_dw, sizeof(bf16) * npad * (size_t)hdim);
  L.coef = take(true, sizeof(f32x4) * (size_t)L.chunk);
  L.f0 = take(true, sizeof(float) * (size_t)L.chunk);
  L.w0 = take(true, sizeof(float) * (size_t)L.chunk);
  L.f = take(need_dw, sizeof(float) * (size_t)L.chunk);
  L.wt = take(need_dw, sizeof(float) * (size_t)L.chunk);
  L.E = take(true, sizeof(bf16) * (size_t)(L.chunk * V));
  L.splits = L.few ? few_splits(hdim, V) : dh_splits(hdim, L.chunk);
  L.prow = (int)std::min<int64_t>(L.chunk, BJ);
  L.run = dh_run(V);
  int64_t slots = L.few ? L.splits : 0;
  if (!L.few && L.splits > 1)
    for (int64_t c0 = 0; c0 < n; c0 += L.chunk)
      slots = std::max(slots, dh_slots(c0, std::min(L.chunk, n - c0), (int)((hdim + BI - 1) / BI), L.splits, L.run));
  L.part = take(slots > 0, sizeof(float) * (size_t)(slots * L.prow * hdim));
  L.nsort = need_dw ? (int)((L.chunk + kIdChunk - 1) / kIdChunk) : 0;
  L.acc32 = take(need_dw && L.nchunks > 1, sizeof(float) * (size_t)(V * hdim));
  L.keys = take(need_dw, sizeof(uint64_t) * (size_t)L.nsort * kIdChunk);
  L.slot = take(need_dw, sizeof(int32_t) * (size_t)V);
  L.next = take(need_dw, sizeof(int32_t) * (size_t)L.nsort * kIdChunk);
  L.lsum = take(need_dw, sizeof(float) * (size_t)(L.chunk * hdim));
  L.total = off;
  return L;
}

// Tiles whose parts bound the others': at least K of them, so that the K-th largest of
// their 2 K parts says something, and three rounds of workgroups, so that the last round
// of a launch of its own costs little; 0: all in one launch.  (5735 rows x 1536 with 64
// alternatives 2.87 -> 2.49 ms: two fifths of the others are written.  A second bound,
// from three eighths, costs as much as it saves: 2.48 -> 2.50.)
int bound_tiles(int nI, int nJ, int K) {
  const int tiles = std::max({nI / 8, K, (3 * kCus + nJ - 1) / nJ});
  return 3 * tiles <= nI ? tiles : 0;
}

template <bool TOP, bool KEEP>
void launch_stat_logits(StatLogitsArgs lg, bool few, int K, float* bound, hipStream_t stream) {
  if (few) {
    const dim3 grid((unsigned)((lg.V + kFewBI - 1) / kFewBI));
    hipLaunchKernelGGL((lg.nc <= 64 ? stats_logits_few_kernel<2, TOP, KEEP> : stats_logits_few_kernel<4, TOP, KEEP>), grid,
                       dim3(kFewThreads), 0, stream, lg);
    return;
  }
  const int nI = (int)((lg.V + kVT - 1) / kVT), first = bound != nullptr ? bound_tiles(nI, (int)((lg.nc + BJ - 1) / BJ), K) : 0;
  lg.nJ = (int)((lg.nc + BJ - 1) / BJ);
  lg.nI = first > 0 ? first : nI;
  auto launch = [&]() {
    const int grid = ((lg.nI * lg.nJ + kXcds - 1) / kXcds) * kXcds;
    hipLaunchKernelGGL((stats_logits_kernel<TOP, KEEP>), dim3(grid), dim3(NT), 0, stream, lg);
  };
  launch();
  if (first == 0) return;
  const BoundArgs bd{lg.part, bound, lg.nvalid, lg.c0, lg.parts, 2 * first, K};
  hipLaunchKernelGGL(stats_bound_kernel, dim3((unsigned)lg.nc), dim3(kRowGroups), 0, stream, bd);
  lg.t0 = first;
  lg.nI = nI - first;
  lg.bound = bound;
  launch();
}

float zscale_of(const StatsArgs& a) { return (float)(1.4426950408889634 / a.temperature); }

CompactArgs compact_of(const StatsArgs& a) {
  CompactArgs c{};
  c.hidden = a.hidden;
  c.weight = a.weight;
  c.labels = a.labels;
  c.n = a.n;
  c.hdim = a.hdim;
  c.vocab = a.vocab;
  c.ignore_index = a.ignore_index;
  c.zscale = zscale_of(a);
  return c;
}

}  // namespace

size_t stats_saved_bytes(int64_t n, int64_t vocab) { return saved_layout(n, vocab).total; }
size_t stats_fwd_workspace_bytes(int64_t n, int64_t hdim, int64_t vocab, int top_k, bool keep) {
  return fwd_layout(n, hdim, vocab, top_k, keep).total;
}
size_t stats_bwd_workspace_bytes(int64_t n, int64_t hdim, int64_t vocab, int64_t chunk, bool need_dw, bool have_saved) {
  return bwd_layout(n, hdim, vocab, chunk, need_dw, have_saved).total;
}

hipError_t stats_fwd(const StatsArgs& a, hipStream_t stream) {
  const bool keep = a.saved != nullptr;
  const FwdLayout L = fwd_layout(a.n, a.hdim, a.vocab, a.top_k, keep);
  const StatsSaved S = saved_layout(a.n, a.vocab);
  int64_t* nvalid = keep ? at<int64_t>(a.saved, S.nvalid) : at<int64_t>(a.ws, L.scal);
  int32_t* rows = keep ? at<int32_t>(a.saved, S.rows) : at<int32_t>(a.ws, L.rows);
  CompactArgs c = compact_of(a);
  c.rows = rows;
  c.nvalid = nvalid;
  c.count = a.count;
  c.bad = a.bad_labels;
  c.invden = at<float>(a.ws, L.scal) + 32;
  c.hc = at<bf16>(a.ws, L.hc);
  c.yc = keep ? at<int64_t>(a.saved, S.yc) : at<int64_t>(a.ws, L.yc);
  c.ref = at<float>(a.ws, L.ref);
  // few rows are taken as they are, those that do not count among them: the table is read all the same (one row 69.4 us
  // with a compacting launch, 64.1 so; 61 rows 80.6 and 76.2)
  const bool as_is = a.n > 0 && L.few && !keep;
  if (!as_is) launch_compact(c, stream);
  for (int64_t c0 = 0; c0 < a.n; c0 += L.chunk) {
    const int64_t nc = std::min(L.chunk, a.n - c0);
    StatLogitsArgs lg{};
    lg.W = GOp{a.weight, a.hdim, a.vocab, a.hdim};
    lg.H = GOp{as_is ? a.hidden : c.hc + c0 * a.hdim, a.hdim, nc, a.hdim};
    lg.y = as_is ? a.labels : c.yc + c0;
    lg.Z = a.top_k > 0 ? at<float>(a.ws, L.Z) : nullptr;
    lg.part = keep ? at<f32x4>(a.saved, S.part) + c0 * L.parts : at<f32x4>(a.ws, L.part);
    lg.E = keep ? at<bf16>(a.saved, S.E) + c0 * a.vocab : nullptr;
    lg.zy = at<float>(a.ws, L.zy);
    lg.nvalid = as_is ? nullptr : nvalid;
    lg.count = a.count;
    lg.bad = a.bad_labels;
    lg.ignore_index = a.ignore_index;
    lg.V = a.vocab;
    lg.nc = nc;
    lg.c0 = c0;
    lg.parts = L.parts;
    lg.zscale = c.zscale;
    const int nI = (int)((a.vocab + kVT - 1) / kVT), nJ = (int)((nc + BJ - 1) / BJ);
    float* bound = !L.few && a.top_k > 0 && bound_tiles(nI, nJ, a.top_k) > 0 ? at<float>(a.ws, L.bound) : nullptr;
    if (a.top_k > 0)
      keep ? launch_stat_logits<true, true>(lg, L.few, a.top_k, bound, stream)
           : launch_stat_logits<true, false>(lg, L.few, a.top_k, bound, stream);
    else
      keep ? launch_stat_logits<false, true>(lg, L.few, 0, nullptr, stream)
           : launch_stat_logits<false, false>(lg, L.few, 0, nullptr, stream);
    StatRowArgs rw{};
    rw.part = lg.part;
    rw.zy = lg.zy;
    rw.Z = lg.Z;
    rw.bound = bound;
    rw.rows = as_is ? nullptr : rows + c0;
    rw.nvalid = nvalid;
    rw.labels = a.labels;
    rw.logp = a.logp;
    rw.entropy = a.entropy;
    rw.state = a.state;
    rw.n = a.n;
    rw.top_logp = a.top_logp;
    rw.top_ids = a.top_ids;
    rw.c0 = c0;
    rw.V = a.vocab;
    rw.ignore_index = a.ignore_index;
    rw.parts = (int)L.parts;
    rw.K = a.top_k;
    rw.few = L.few;
    rw.zscale = c.zscale;
    hipLaunchKernelGGL(stats_row_kernel, dim3((unsigned)nc), dim3(kRowGroups), 0, stream, rw);
  }
  return hipGetLastError();
}

hipError_t stats_bwd(const StatsArgs& a, hipStream_t stream) {
  const bool need_dw = a.dweight != nullptr;
  const bool have = a.saved != nullptr;
  const BwdLayout L = bwd_layout(a.n, a.hdim, a.vocab, a.chunk, need_dw, have);
  const StatsSaved S = saved_layout(a.n, a.vocab);
  if (a.n == 0) {
    if (need_dw) launch_zero(a.dweight, a.vocab * a.hdim, stream);
    return hipGetLastError();
  }
  int64_t* nvalid = have ? at<int64_t>(a.saved, S.nvalid) : at<int64_t>(a.ws, L.scal);
  int32_t* rows = have ? at<int32_t>(a.saved, S.rows) : at<int32_t>(a.ws, L.rows);
  CompactArgs c = compact_of(a);
  c.rows = rows;
  c.nvalid = nvalid;
  c.count = nvalid + 1;
  c.bad = nvalid + 2;
  c.invden = at<float>(a.ws, L.scal) + 32;
  c.hc = at<bf16>(a.ws, L.hc);
  c.yc = have ? at<int64_t>(a.saved, S.yc) : at<int64_t>(a.ws, L.yc);
  c.ref = at<float>(a.ws, L.ref);
  c.dh = a.dhidden;
  if (!have) launch_compact(c, stream);
  // few rows in one chunk, from what was kept: the labels' sums come with dH's (4 rows x 64, both directions, 109 -> 98 us)
  const bool one_few = have && need_dw && L.few && L.nchunks == 1;
  bf16* E = at<bf16>(a.ws, L.E);
  float *f0 = at<float>(a.ws, L.f0), *w0 = at<float>(a.ws, L.w0);
  for (int64_t c0 = 0; c0 < a.n; c0 += L.chunk) {
    const int64_t nc = std::min(L.chunk, a.n - c0);
    bf16* Hc = c.hc + c0 * a.hdim;
    StatCoefArgs co{};
    co.rows = rows + c0;
    co.nvalid = nvalid;
    co.state = a.state;
    co.n = a.n;
    co.g = a.dlogp;
    co.e = a.dentropy;
    co.coef = at<f32x4>(a.ws, L.coef);
    co.f = f0;
    co.w = w0;
    co.nc = nc;
    co.c0 = c0;
    co.inv_t = (float)(1. / a.temperature);
    if (!one_few) hipLaunchKernelGGL(stats_coef_kernel, dim3((unsigned)((nc + 255) / 256)), dim3(256), 0, stream, co);
    StatGradArgs gr{};
    gr.W = GOp{a.weight, a.hdim, a.vocab, a.hdim};
    gr.H = GOp{Hc, a.hdim, nc, a.hdim};
    gr.y = c.yc + c0;
    gr.coef = co.coef;
    gr.G = E;
    gr.nvalid = nvalid;
    gr.V = a.vocab;
    gr.nc = nc;
    gr.c0 = c0;
    gr.zscale = c.zscale;
    if (have) {
      UnpackArgs un{};
      un.E = at<bf16>(a.saved, S.E) + c0 * a.vocab;
      un.part = at<f32x4>(a.saved, S.part) + c0 * S.parts;
      un.c = co;
      un.G = E;
      un.labels = a.labels;
      un.dh = a.dhidden;
      un.V = a.vocab;
      un.hdim = a.hdim;
      un.ignore_index = a.ignore_index;
      un.parts = (int)S.parts;
      un.few = a.n <= kFewRows;
      un.H = a.hidden;
      un.Hs = Hc;
      un.slot = at<int32_t>(a.ws, L.slot);
      const dim3 grid((unsigned)((a.vocab + kUnpackCols - 1) / kUnpackCols), (unsigned)std::min<int64_t>(nc, 32768));
      hipLaunchKernelGGL((one_few ? stats_unpack_kernel<true> : stats_unpack_kernel<false>), grid, dim3(256), 0, stream, un);
    } else if (L.few) {
      const dim3 grid((unsigned)((a.vocab + kFewBI - 1) / kFewBI));
      hipLaunchKernelGGL((nc <= 64 ? stats_grad_few_kernel<2> : stats_grad_few_kernel<4>), grid, dim3(kFewThreads), 0, stream,
                         gr);
    } else {
      gr.nI = (int)((a.vocab + kVT - 1) / kVT);
      gr.nJ = (int)((nc + BJ - 1) / BJ);
      const int grid = ((gr.nI * gr.nJ + kXcds - 1) / kXcds) * kXcds;
      hipLaunchKernelGGL(stats_grad_kernel, dim3(grid), dim3(NT), 0, stream, gr);
    }
    if (a.dhidden != nullptr || one_few) {
      DhArgs dh{};
      dh.Wt = gr.W;
      dh.E = GOp{E, a.vocab, nc, a.vocab};
      dh.dh = a.dhidden;
      dh.part = at<float>(a.ws, L.part);
      dh.f = f0;
      dh.wt = w0;
      dh.y = gr.y;
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
        fs.f0 = f0;
        fs.w0 = w0;
        fs.scale = 1.f;
        if (one_few) {
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
      wg.y = gr.y;
      wg.f0 = f0;
      wg.w0 = w0;
      wg.nvalid = nvalid;
      wg.Hs = Hc;  // (which the logits above have read; every factor is 1)
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
    launch_dw(dw, L.few && L.nchunks == 1, stream);
  }
  return hipGetLastError();
}

}  // namespace siq

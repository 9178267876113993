// What the products over the lm_head's table share: arguments and launches of the
// kernels in flce.hip, for the operators that use them from files of their own.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"
#include "gemm.h"

namespace siq {

constexpr int kVT = gemm::BI;  // vocab columns per logits tile

// Rows (of one call) that take the few-rows kernels, and their weight rows or
// features of a tile; threads of its workgroup.
constexpr int kFewRows = 128, kFewBI = 128, kFewThreads = 256;

// Rows with a list of tokens: a tile of columns has a bit for each, in the order in
// which the logits kernels' lanes hold them, so that a lane's columns are 64 (few rows:
// 16) bits in a row, and a list in that order has each lane's tokens in a row, too.
// The place of column v of a tile:
__host__ __device__ constexpr int list_place(int v, bool few) {
  return few ? (v & 0x60) | (v & 8) << 1 | (v & 16) >> 1 | (v & 7)
             : (v & 64) << 1 | (v & 8) << 3 | (v & 128) >> 2 | (v & 32) >> 1 | (v & 16) >> 1 | (v & 7);
}
constexpr int list_lane_bits(bool few) { return few ? 16 : 64; }

struct LogitsArgs {
  gemm::GOp W, H;               // W [V, hdim], H = hidden rows of the chunk [nc, hdim]
  const int64_t* y;       // chunk labels
  const float* ref;       // [nc] row references (log2 units)
  bf16* E;                // [nc, V]
  float* spart;           // [nvt, ldp] tile sum of exp2(z2 - ref); negated for a redone tile
  float* mpart;           // [nvt, ldp] a redone tile's own reference
  float* zy;              // [nc] label logit (natural units); label_apart: log2 units, relative to ref
  const int64_t* nvalid;  // valid (compacted) rows in all chunks
  int64_t V, nc, c0, ldp;
  int nI, nJ;
  int store_e;            // 0: loss only, E is not needed
  int label_apart;        // the label is left out of E and of the sums
  float zscale;           // log2(e) / temperature
  // rows with a list of tokens apart (launch_logits' `lists`; zy is not written)
  const uint8_t* mask;    // [nc, ldm] a bit for each column: listed (list_place)
  const uint8_t* base;    // [nc, ldb] for each lane's bits of a tile: how many tokens of the list come before them
  float* zk;              // [nc, ldk] the listed tokens' logits in log2 units, relative to ref, in the list's order
  int64_t ldm, ldb;
  int ldk;
  int32_t* slot;          // [V] cleared (few rows with lists), or nullptr
};

struct RowArgs {
  const float* spart;    // [nvt, ldp] tile sums (negative: redone, relative to mpart)
  const float* mpart;
  const float* ref;      // [nc] row references (log2 units)
  const float* zy;       // [nc] as the logits kernel left it
  const int64_t* y;      // chunk labels
  bf16* E;               // [nc, V]
  bf16* H;               // [nc, hdim] compacted rows: scaled by f (need_dw)
  float* f;              // [nc] factors of E
  float* wt;             // [nc] weights of the label terms
  float* loss_row;       // [nc] (chunk slice; not with label_apart)
  float* logp;           // [n] log-probabilities of the labels by original row (label_apart), or nullptr
  const int32_t* rows;   // compacted row -> original row (chunk slice; label_apart)
  const float* invden;   // nullptr: 1
  const int64_t* nvalid;
  uint64_t* keys;        // [nsort, kIdChunk] rows sorted by label
  int32_t* slot;         // [V] cleared
  int64_t nc, nvt, V, hdim, c0, ldp;
  int vlog;              // log2 of the eight-column groups of a tile
  int nsort;             // sorting workgroups (0 without dW)
  int parts;             // workgroups per 64 rows
  int grads;             // 0: loss only (E was never stored)
  int label_apart;
  float* rsum;           // [nc] launch_row's `lists`: a row's sum over the columns that are not in its list,
  float* rtop;           // and what it and E are relative to (log2 units); nothing else is written but E
};

struct LabelArgs {
  const uint64_t* keys;  // [nsort, kIdChunk]
  const bf16* H;         // [n, hdim] all rows, unscaled
  const int32_t* rows;   // chunk's compacted row -> row of H
  const float* wt;       // [nc]
  float* lsum;           // [nsort * kIdChunk (rows that exist), hdim]
  int32_t* slot;         // [V]
  int32_t* next;         // [nsort * kIdChunk]
  int64_t hdim;
  int nsort;
};

struct DhArgs {
  gemm::GOp Wt;        // W [V, hdim] read as A[i = h][k = v]
  gemm::GOp E;         // [nc, V] read as B[j = tok][k = v]
  bf16* dh;      // dhidden [n, hdim]
  float* part;   // [slots][prow][hdim] partial sums (DhTiles; none when splits == 1)
  const float* f;         // [nc] row factors, label weights, labels
  const float* wt;
  const int64_t* y;
  const int32_t* rows;    // compacted row -> original row (whole batch)
  const int64_t* nvalid;
  int64_t hdim, nc, c0;
  int nI, splits, prow, run;  // hdim tiles; vocab ranges; rows of a slot; dh_run
};

struct DwArgs {
  gemm::GOp Ht;        // hidden rows of the chunk [nc, hdim], scaled by f, read as A[i = h][k = tok]
  gemm::GOp Et;        // E [nc, V] read as B[j = v][k = tok]
  const int32_t* slot;   // [V] label terms: row of lsum + 1, or 0
  const int32_t* next;   // [rows] the label's next row of lsum + 1, or 0
  const float* lsum;     // [rows, hdim]
  bf16* dw;      // [V, hdim]
  float* acc32;  // [V, hdim] fp32 accumulator across chunks
  const int64_t* nvalid;
  int64_t hdim, V, c0, chunk;
  int nI, nJ;
  int two_in_bf16;  // over two chunks the first one's sum waits in dw
};

struct WeighArgs {
  const bf16* H;          // [n, hdim] all rows
  const int32_t* rows;    // chunk's compacted row -> row of H
  const int64_t* y;       // chunk labels
  const float* f0;        // [nc]
  const float* w0;
  const float* g;         // [n] upstream gradients, by original row, or nullptr: 1
  const int64_t* nvalid;
  const int64_t* labels;  // [n] all labels, with dh: rows that do not count are zeroed
  bf16* dh;               // or nullptr
  bf16* Hs;               // [nc, hdim] (nsort > 0)
  float* f;               // [nc]
  float* wt;
  uint64_t* keys;         // [nsort, kIdChunk]
  int32_t* slot;          // [V] cleared
  int64_t n, nc, c0, V, hdim, ignore_index;
  float scale;            // -1 / temperature
  int nsort;              // sorting workgroups (0 without dW)
};

struct FewSumArgs {
  DhArgs dh;
  const float* f0;        // as WeighArgs: dH alone needs no pass of its own for them
  const float* w0;
  const float* g;         // (nullptr: 1)
  const int64_t* labels;  // of all rows, or nullptr: nothing is cleared
  int64_t ignore_index;
  float scale;
  // the label terms of dW, too (dh.dh may be nullptr then): sums of w H over the rows of each
  // label, as flce_label_kernel's (slots cleared before)
  const bf16* H;          // [n, hdim] all rows
  float* lsum;            // [nc, hdim] or nullptr
  int32_t* slot;          // [V]
  int32_t* next;          // [nc]
};

// dH: vocab ranges, rows of a run, and slots of partial sums that rows [c0, c0 + nc) need.
int dh_splits(int64_t hdim, int64_t chunk);
int dh_run(int64_t V);
int64_t dh_slots(int64_t c0, int64_t nc, int nI, int splits, int run);
int few_splits(int64_t hdim, int64_t V);

// The counted rows' list (`rows`, *nvalid, *count, *bad, *invden).
struct CompactArgs {
  const bf16* hidden;
  const bf16* weight;
  const int64_t* labels;
  int64_t n, hdim, vocab, ignore_index;
  int reduction;
  const float* divisor;
  float zscale;
  int32_t* rows;
  int64_t *nvalid, *count, *bad;
  float* invden;  // nullptr with n <= kFewRows: not written
  bf16* hc;
  int64_t* yc;
  float* ref;
  bf16* dh;       // or nullptr: rows that do not count are zeroed
  float* logp;    // likewise
};
// The list, and the counted rows' hidden states, labels and references compacted.
void launch_compact(const CompactArgs& a, hipStream_t stream);

// `few`: the kernels of few rows (nc <= kFewRows, tiles of kFewBI columns).
void launch_logits(LogitsArgs& lg, bool few, bool lists, hipStream_t stream);
void launch_row(RowArgs& rw, bool few, bool lists, hipStream_t stream);  // (lists: not with few)
void launch_weigh(const WeighArgs& wg, hipStream_t stream);
void launch_labels(const LabelArgs& la, int64_t nc, hipStream_t stream);
void launch_dh(DhArgs& dh, hipStream_t stream);
void launch_dh_few(FewSumArgs& a, hipStream_t stream);
void launch_dw(DwArgs& dw, bool few, hipStream_t stream);
void launch_zero(bf16* x, int64_t numel, hipStream_t stream);

inline int tile_log(int columns) { return __builtin_ctz((unsigned)columns / 8); }
inline size_t al(size_t x) { return (x + 255) & ~size_t(255); }

template <class T>
T* at(void* base, size_t off) {
  return reinterpret_cast<T*>(static_cast<char*>(base) + off);
}

}  // namespace siq

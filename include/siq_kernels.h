/*
 * siq_kernels.h -- C ABI of the SiQ-VL training hot path on MI355X (gfx950).
 *
 * Hand-written HIP operators behind this plain-C boundary:
 *   1. varlen (cu_seqlens-packed) flash attention, forward and backward,
 *      causal GQA (Qwen2.5 decoder) or bidirectional (SigLIP tower);
 *   2. fused lm_head linear + cross-entropy, forward and backward, without
 *      materialising the [N, V] logits;
 *   3. the rotary position embedding of q and k that precedes attention in
 *      the decoder, forward and backward, in one pass each;
 *   4. the pixel-shuffle projector (vision features to text embeddings),
 *      forward and backward, with the shuffle folded into the GEMM loads;
 *   5. the splice of the projected vision rows into the token embeddings,
 *      fused with the embedding gather, and its embedding-table gradient;
 *   6. activations kept in 8 bits for the backward pass, and the gated MLP
 *      activation over them;
 *   7. the losses of preference and policy training on packed
 *      log-probabilities, forward and backward, and those log-probabilities
 *      from hidden states without the logits.
 *
 * Conventions
 *  - Every entry point returns an int status (SIQ_OK = 0, < 0 on error) and
 *    records a message readable with siq_last_error() (thread-local).
 *  - All tensors are device pointers owned by the caller.  The library never
 *    allocates, frees or keeps pointers beyond a call; scratch memory is the
 *    caller's `workspace` (size from the matching *_workspace_bytes()).
 *  - `stream` is a hipStream_t (NULL = the null stream).  Work is only
 *    enqueued: no device synchronisation and no device-to-host reads.
 *  - bf16 tensors are token-major: element (token t, head h, dim d) lives at
 *    base + t * tok_stride + h * head_stride + d (d contiguous).  Base
 *    pointers and both strides must keep 16-byte alignment (strides multiple
 *    of 8 elements).
 *  - cu_seqlens are int32 device arrays of batch+1 non-decreasing offsets with
 *    cu[0] = 0 and cu[batch] = total.  They are read on the device; values
 *    outside [0, total] are clamped there, so malformed offsets give wrong
 *    numbers for the offending sequences but never an out-of-bounds access.
 */
#ifndef SIQ_KERNELS_H
#define SIQ_KERNELS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define SIQ_ABI_VERSION 4

enum siq_status {
  SIQ_OK = 0,
  SIQ_ERR_INVALID_ARGUMENT = -1, /* shape / dtype / value rejected before launch */
  SIQ_ERR_UNSUPPORTED = -2,      /* e.g. head_dim not in {64, 128} */
  SIQ_ERR_WORKSPACE = -3,        /* workspace missing or too small */
  SIQ_ERR_ALIGNMENT = -4,        /* pointer or stride breaks 16-byte alignment */
  SIQ_ERR_LAUNCH = -5            /* the HIP runtime rejected a launch */
};

/* Element types of the entry points that take more than one. */
#define SIQ_DTYPE_BF16 0
#define SIQ_DTYPE_FP32 1

/* Formats of 8-bit storage (siq_pack8). */
#define SIQ_FORMAT_INT8 0
#define SIQ_FORMAT_E4M3 1

/* Version of this ABI (SIQ_ABI_VERSION of the library that was built). */
int siq_abi_version(void);

/* Message of the last failing call on this thread ("" if none). */
const char* siq_last_error(void);

/* ---------------------------------------------------------------------------
 * Varlen attention.
 *
 * Replaces, for one packed batch, the attention call the reference reaches at
 * transformers integrations/sdpa_attention.py:154-163 (F.scaled_dot_product_
 * attention on a padded batch, reached from models/qwen2/modeling_qwen2.py:
 * 216-230 and models/siglip/modeling_siglip.py:288-300) with the varlen
 * contract of modeling_flash_attention_utils.py:796-822
 * (q, k, v, cu_seqlens_q, cu_seqlens_k, max_seqlen_q, max_seqlen_k,
 * softmax_scale, causal).
 *
 * Shapes: q [total_q, hq, d], k/v [total_k, hkv, d], o like q, all bf16;
 * lse fp32 [hq, total_q] (natural log, contiguous); hq % hkv == 0 and q-head h
 * reads kv-head h / (hq / hkv); d in {64, 128}.  Causal masking is aligned
 * bottom-right (q row i of a sequence sees k rows <= i + len_k - len_q), which
 * is the usual top-left causal mask when len_q == len_k.
 *
 * strides[8] = {q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head}
 * (in elements).
 * ------------------------------------------------------------------------- */
size_t siq_attn_fwd_workspace_bytes(int batch, int64_t total_q, int64_t total_k, int hq, int hkv, int d);

int siq_attn_varlen_fwd(const void* q, const void* k, const void* v, void* o, float* lse,
                        const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch,
                        int max_seqlen_q, int max_seqlen_k, int64_t total_q, int64_t total_k, int hq, int hkv,
                        int d, const int64_t* strides, float softmax_scale, int causal, void* workspace,
                        size_t workspace_bytes, void* stream);

/* Backward of siq_attn_varlen_fwd (the autograd backward of the same call in
 * the reference path).  Inputs q, k, v, o, lse as produced/consumed by the
 * forward, dout like o; outputs dq like q, dk/dv like k/v, each written in full
 * (no accumulation).
 * deterministic != 0: no atomics, bitwise reproducible (dQ in a kernel of its
 * own that recomputes S and dP).  deterministic == 0: dQ = dS K is formed in
 * the dK/dV kernel and summed with fp32 atomics in the workspace (the sum
 * order varies from run to run; the workspace grows by total_q * hq * d * 4
 * bytes; on MI355X it measured 2-3x slower than the deterministic backward at
 * the SiQ-VL shapes).  flash-attn's flash_attn_varlen_func(deterministic=...)
 * flag.
 * strides[16] = {q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head,
 *                do_tok, do_head, dq_tok, dq_head, dk_tok, dk_head, dv_tok, dv_head}. */
size_t siq_attn_bwd_workspace_bytes(int batch, int64_t total_q, int64_t total_k, int hq, int hkv, int d,
                                    int deterministic);

int siq_attn_varlen_bwd(const void* q, const void* k, const void* v, const void* o, const float* lse,
                        const void* dout, void* dq, void* dk, void* dv, const int32_t* cu_seqlens_q,
                        const int32_t* cu_seqlens_k, int batch, int max_seqlen_q, int max_seqlen_k,
                        int64_t total_q, int64_t total_k, int hq, int hkv, int d, const int64_t* strides,
                        float softmax_scale, int causal, int deterministic, void* workspace,
                        size_t workspace_bytes, void* stream);

/* Allocation-free siq_attn_varlen_fwd.  No counterpart in the reference: it
 * exists for callers that cannot allocate device memory (code under HIP graph
 * capture, tight serving loops, harnesses that forbid allocation) and takes
 * no workspace.  Same arguments (minus the workspace), validation and output,
 * bitwise, as siq_attn_varlen_fwd.  The batch's plan goes to a static device
 * array of 1 MiB per GPU (held until the process ends): batch and total_q
 * must satisfy 256 + 16 batch + 32 (total_q / 128 + batch + 1) <= 1 MiB (each
 * term rounded up to 256 bytes), e.g. batch <= 8192 with total_q <= 2^20;
 * larger calls return SIQ_ERR_WORKSPACE before anything is launched.  All
 * calls on one GPU share the array: calls that overlap on one GPU (from
 * different streams or threads) race. */
int siq_attn_varlen_fwd_noalloc(const void* q, const void* k, const void* v, void* o, float* lse,
                                const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch,
                                int max_seqlen_q, int max_seqlen_k, int64_t total_q, int64_t total_k, int hq,
                                int hkv, int d, const int64_t* strides, float softmax_scale, int causal,
                                void* stream);

/* ---------------------------------------------------------------------------
 * Attention plans: the schedule of one packed batch, built once and reused.
 *
 * The reference forwards the same cu_seq_lens_* kwargs to every decoder layer
 * (siq_vl/model/modeling.py:278-288 -> transformers modeling_qwen2.py:216-230),
 * so the work lists siq_attn_varlen_fwd / _bwd build on every call (sequence
 * extents, q tiles and dK/dV work items ordered by decreasing work) are the
 * same for all layers.  siq_attn_build_plan writes them once into `plan`
 * (siq_attn_plan_bytes, device memory owned by the caller); the *_plan entry
 * points then run the forward / backward of any layer over it.  A plan
 * depends on the offsets, total_q / total_k, hq / hkv and causal only; it
 * records them, and a kernel handed a plan built for other values writes
 * nothing and sets a mismatch bit in the plan (bytes 48..51, int32) instead of
 * touching memory outside its tensors.  Bytes 40..47 hold the scheduler's
 * overflow bits (0 by construction).
 * ------------------------------------------------------------------------- */
size_t siq_attn_plan_bytes(int batch, int64_t total_q, int64_t total_k);

int siq_attn_build_plan(const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k, int batch, int64_t total_q,
                        int64_t total_k, int hq, int hkv, int causal, void* plan, size_t plan_bytes, void* stream);

/* siq_attn_varlen_fwd over a built plan (no workspace). */
int siq_attn_varlen_fwd_plan(const void* q, const void* k, const void* v, void* o, float* lse, int batch,
                             int64_t total_q, int64_t total_k, int hq, int hkv, int d, const int64_t* strides,
                             float softmax_scale, int causal, const void* plan, size_t plan_bytes, void* stream);

/* siq_attn_varlen_bwd over a built plan; the workspace holds the backward's
 * own scratch only (siq_attn_bwd_plan_workspace_bytes, for the same
 * deterministic flag). */
size_t siq_attn_bwd_plan_workspace_bytes(int batch, int64_t total_q, int64_t total_k, int hq, int hkv, int d,
                                         int deterministic);

int siq_attn_varlen_bwd_plan(const void* q, const void* k, const void* v, const void* o, const float* lse,
                             const void* dout, void* dq, void* dk, void* dv, int batch, int64_t total_q,
                             int64_t total_k, int hq, int hkv, int d, const int64_t* strides, float softmax_scale,
                             int causal, int deterministic, const void* plan, size_t plan_bytes, void* workspace,
                             size_t workspace_bytes, void* stream);

/* Varlen attention with the decoder's rotary embedding of q fused in.
 *
 * Replaces apply_rotary_pos_emb's q half (transformers modeling_qwen2.py:
 * 105-135, called at :206-211) together with the attention call after it:
 * siq_attn_rope_fwd_plan reads q BEFORE rotation, rotates it in registers with
 * the cos / sin rows of each token (bitwise siq_rope_fwd's q_embed), attends
 * as siq_attn_varlen_fwd_plan does (k already rotated, e.g. by siq_rope_fwd
 * with hq = 0) and writes the rotated q to q_embed for the backward.
 * siq_attn_rope_bwd_plan takes that q_embed and writes dq with respect to the
 * q BEFORE rotation (bitwise siq_rope_bwd applied to siq_attn_varlen_bwd_plan's
 * dq); dk, dv are those of siq_attn_varlen_bwd_plan (dk with respect to the
 * rotated k).  The backward is the deterministic one (its workspace:
 * siq_attn_bwd_plan_workspace_bytes(..., 1)): the rotation's backward runs in
 * the epilogue of its dQ kernel.  cos / sin: [total_q, d] bf16 rows, one per
 * packed token.
 * strides: fwd[12] = the 8 of siq_attn_varlen_fwd, q_embed (tok, head),
 * cos_tok, sin_tok; bwd[18] = the 16 of siq_attn_varlen_bwd (q = q_embed),
 * cos_tok, sin_tok. */
int siq_attn_rope_fwd_plan(const void* q, const void* k, const void* v, void* o, float* lse, void* q_embed,
                           const void* cos, const void* sin, int batch, int64_t total_q, int64_t total_k, int hq,
                           int hkv, int d, const int64_t* strides, float softmax_scale, int causal, const void* plan,
                           size_t plan_bytes, void* stream);

int siq_attn_rope_bwd_plan(const void* q_embed, const void* k, const void* v, const void* o, const float* lse,
                           const void* dout, void* dq, void* dk, void* dv, const void* cos, const void* sin, int batch,
                           int64_t total_q, int64_t total_k, int hq, int hkv, int d, const int64_t* strides,
                           float softmax_scale, int causal, const void* plan, size_t plan_bytes, void* workspace,
                           size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------------
 * Fused linear cross-entropy (lm_head + loss), forward and backward.
 *
 * Replaces logits = lm_head(h) (transformers models/qwen2/modeling_qwen2.py:
 * 465) followed by ForCausalLMLoss / fixed_cross_entropy (loss/loss_utils.py:
 * 32-71: fp32 upcast, F.cross_entropy with ignore_index) and their autograd
 * backward.  hidden [n, hdim] bf16 row-major, weight [vocab, hdim] bf16
 * row-major, labels [n] int64 (already shifted; ignore_index rows are skipped;
 * any other value outside [0, vocab) is treated as ignored and counted in
 * *bad_labels, which the host raises on as F.cross_entropy would).
 *
 * reduction 0 ("mean"): loss = sum_valid(lse - z_y) / count_valid.
 * reduction 1 ("sum" then divide, as with num_items_in_batch):
 *   loss = sum_valid(lse - z_y) / *divisor, divisor a device fp32 scalar.
 * Outputs (device): *loss fp32 scalar, *count int64 number of valid rows,
 * dhidden [n, hdim] bf16 = d loss / d hidden, dweight [vocab, hdim] bf16 =
 * d loss / d weight (may be NULL to skip it).  Ignored rows get dhidden
 * exactly 0.  dhidden may be the buffer of hidden.
 *
 * The logits are produced chunk_tokens rows at a time: only the softmax
 * numerators of one chunk (chunk_tokens x vocab bf16, each relative to its
 * row's label logit, or to a larger one where that is more than 2^60 too low)
 * ever exist, in the workspace; chunks count rows
 * whose label counts (ignored rows are compacted away first).  Over two
 * chunks dweight is summed in dweight itself (the first chunk's sum rounded to
 * bf16 once); over more it is summed in an fp32 [vocab, hdim] workspace
 * buffer, which the workspace holds whenever n exceeds two chunks.  The loss
 * does not depend on chunk_tokens, nor does dhidden between chunks of up to 292
 * tiles of 256 rows x 256 features (bitwise).
 * ------------------------------------------------------------------------- */
size_t siq_flce_workspace_bytes(int64_t n, int64_t hdim, int64_t vocab, int64_t chunk_tokens, int need_dweight);

int siq_flce_fwd_bwd(const void* hidden, const void* weight, const int64_t* labels, int64_t n, int64_t hdim,
                     int64_t vocab, int64_t ignore_index, int reduction, const float* divisor, float* loss,
                     int64_t* count, int64_t* bad_labels, void* dhidden, void* dweight, int64_t chunk_tokens,
                     void* workspace, size_t workspace_bytes, void* stream);

/* Loss only: the same loss, count and bad_labels as siq_flce_fwd_bwd on the
 * same inputs (bitwise), without the gradient work -- the reference's
 * evaluation pass (scripts/train.py:693-699 evaluates eval_loss under
 * torch.no_grad through the same lm_head + ForCausalLMLoss call).  Only the
 * logits GEMM and the chunked logsumexp run; no softmax numerators are
 * stored.  Workspace: siq_flce_loss_workspace_bytes. */
size_t siq_flce_loss_workspace_bytes(int64_t n, int64_t hdim, int64_t vocab);

int siq_flce_loss(const void* hidden, const void* weight, const int64_t* labels, int64_t n, int64_t hdim,
                  int64_t vocab, int64_t ignore_index, int reduction, const float* divisor, float* loss,
                  int64_t* count, int64_t* bad_labels, void* workspace, size_t workspace_bytes, void* stream);

/* Log-probabilities of the labels, without the logits (no counterpart in the
 * reference, whose loss is their mean; preference and policy losses weight each
 * of them):
 *   logp[i] = z_iy - log sum_j exp(z_ij),  z = hidden weight^T / temperature,
 * fp32 [n]; 0 where the label is ignore_index or, counted in *bad_labels,
 * outside [0, vocab).  *count = rows that count.  Both are only written, and may
 * lie in pinned host memory.  Operands as for siq_flce_fwd_bwd.
 * siq_flp_bwd: with dlogp [n] the upstream gradients (those of rows that do not
 * count are not read),
 *   dhidden = dZ weight,  dweight = dZ^T hidden,
 *   dZ_ij = dlogp_i / temperature (1[j = y_i] - exp(z_ij - lse_i)),
 * either of the two may be NULL (not computed); dhidden must not overlap hidden.
 * `saved` (siq_flp_saved_bytes) non-NULL: the forward keeps every row's softmax
 * numerators (n x vocab bf16) there and the backward, given the same buffer and
 * inputs, starts from them; it is only read, so a second backward may follow.
 * NULL in both: the backward forms the logits again, chunk_tokens rows at a
 * time, as siq_flce_fwd_bwd does (chunk_tokens is not used with saved). */
size_t siq_flp_saved_bytes(int64_t n, int64_t vocab);

size_t siq_flp_fwd_workspace_bytes(int64_t n, int64_t hdim, int64_t vocab, int keep);

int siq_flp_fwd(const void* hidden, const void* weight, const int64_t* labels, int64_t n, int64_t hdim, int64_t vocab,
                int64_t ignore_index, double temperature, float* logp, int64_t* count, int64_t* bad_labels, void* saved,
                size_t saved_bytes, void* workspace, size_t workspace_bytes, void* stream);

size_t siq_flp_bwd_workspace_bytes(int64_t n, int64_t hdim, int64_t vocab, int64_t chunk_tokens, int need_dweight,
                                   int have_saved);

int siq_flp_bwd(const void* hidden, const void* weight, const int64_t* labels, const float* dlogp, int64_t n,
                int64_t hdim, int64_t vocab, int64_t ignore_index, double temperature, const void* saved,
                size_t saved_bytes, void* dhidden, void* dweight, int64_t chunk_tokens, void* workspace,
                size_t workspace_bytes, void* stream);

/* dst = src * (*scalar) over numel bf16 elements, rounded once from fp32
 * (a device fp32 scalar, read on the device): applies the upstream gradient
 * of the scalar loss to dhidden / dweight.  Companion of siq_flce_fwd_bwd; no
 * reference counterpart (autograd's chain rule).  src == dst scales in place
 * (and then an exact 1.0 writes nothing); any other overlap is undefined. */
int siq_scale_bf16(const void* src, void* dst, int64_t numel, const float* scalar, void* stream);

/* Two tensors by the same scalar in one launch. */
int siq_scale2_bf16(const void* src0, void* dst0, int64_t numel0, const void* src1, void* dst1, int64_t numel1,
                    const float* scalar, void* stream);

/* siq_scale_bf16(data, data, numel, scalar, stream). */
int siq_scale_bf16_inplace(void* data, int64_t numel, const float* scalar, void* stream);

/* ---------------------------------------------------------------------------
 * Rotary position embedding of q and k (Qwen2 decoder).
 *
 * Replaces apply_rotary_pos_emb (transformers models/qwen2/modeling_qwen2.py:
 * 105-135, with rotate_half; called from Qwen2Attention.forward at :206-211):
 *   q_embed = q * cos + rotate_half(q) * sin,  k_embed likewise,
 * rotate_half(x) = cat(-x[..., D/2:], x[..., :D/2]), evaluated with the
 * reference's bf16 rounding after every op, so the results are bitwise those
 * of the reference's torch ops on the same bf16 inputs.  siq_rope_bwd applies
 * the reference's autograd of the same ops to the upstream gradients
 * (dq_embed, dk_embed) and writes dq, dk.
 *
 * Tensors are bf16 [batch, seqlen, heads, head_dim] (cos, sin:
 * [batch, seqlen, head_dim]) with element strides, head_dim contiguous:
 * strides[16] = q (b, s, h), k (b, s, h), cos (b, s), sin (b, s),
 * q_embed (b, s, h), k_embed (b, s, h) -- for siq_rope_bwd read dq_embed,
 * dk_embed, cos, sin, dq, dk.  Strides are multiples of 8 elements and base
 * pointers 16-byte aligned.  An output may be its input (same pointer and
 * strides, in place); any other overlap is undefined.  head_dim: a multiple of
 * 16 in [16, 512]; hq, hkv <= 4096; batch * seqlen < 2^32.  hq = 0 rotates k
 * only (q and its output are then not read and may be NULL): the pass that
 * goes with siq_attn_rope_fwd_plan / _bwd_plan, which rotate q themselves.
 * No workspace.
 * ------------------------------------------------------------------------- */
int siq_rope_fwd(const void* q, const void* k, const void* cos, const void* sin, void* q_embed, void* k_embed,
                 int64_t batch, int64_t seqlen, int hq, int hkv, int head_dim, const int64_t* strides, void* stream);

int siq_rope_bwd(const void* dq_embed, const void* dk_embed, const void* cos, const void* sin, void* dq, void* dk,
                 int64_t batch, int64_t seqlen, int hq, int hkv, int head_dim, const int64_t* strides, void* stream);

/* The same two passes with the dtype of cos / sin chosen (cs_dtype:
 * SIQ_DTYPE_BF16 = siq_rope_fwd / _bwd, or SIQ_DTYPE_FP32).  fp32 cos / sin
 * are what transformers' rotary embedding hands over under bf16 autocast
 * over fp32 master weights (the reference's bf16=True training,
 * scripts/train.py:712): there q and k are bf16 (autocast Linear outputs) and
 * torch promotes q * cos + rotate_half(q) * sin to fp32, which the attention
 * then casts to bf16.  siq_rope_fwd_ex writes that bf16 cast directly:
 * q_embed = rb(fl(fl(q1 c1) - fl(q2 s1)), ...) with fp32 products and sum and
 * one rounding to bf16, bitwise the reference's q_embed.to(bf16).
 * siq_rope_bwd_ex is the reference's autograd of those ops on the bf16
 * gradient of that cast: dq = rb(rb(fl(g1 c1)) + rb(fl(g2 s2))), ... .  With
 * fp32 cos / sin their strides are multiples of 4 elements (16 bytes); the
 * other tensors are as for siq_rope_fwd. */
int siq_rope_fwd_ex(const void* q, const void* k, const void* cos, const void* sin, void* q_embed, void* k_embed,
                    int64_t batch, int64_t seqlen, int hq, int hkv, int head_dim, const int64_t* strides,
                    int cs_dtype, void* stream);

int siq_rope_bwd_ex(const void* dq_embed, const void* dk_embed, const void* cos, const void* sin, void* dq, void* dk,
                    int64_t batch, int64_t seqlen, int hq, int hkv, int head_dim, const int64_t* strides,
                    int cs_dtype, void* stream);

/* ---------------------------------------------------------------------------
 * Pixel-shuffle projector (the vision-to-text bridge).
 *
 * Replaces SiQ_VLProjector.forward (siq_vl/model/modeling.py:100-105): the
 * pixel shuffle of :74-98 (view [batch, side, side, dv], reshape by the
 * factor r, permute(0, 1, 3, 2, 4, 5), reshape to [batch, (side/r)^2,
 * r*r*dv]) followed by the bias-free Linear mlp (:59) -- and its autograd
 * backward -- without materialising the shuffled tensor:
 *   y [batch*(side/r)^2, out_features] = shuffle(x) weight^T,
 *   dx = unshuffle(dy weight),  dweight = dy^T shuffle(x).
 * x [batch, side*side, vision_dim], weight [out_features, r*r*vision_dim],
 * y / dy [batch*(side/r)^2, out_features]: bf16, contiguous, 16-byte
 * aligned; fp32 accumulation.  vision_dim % 64 == 0, out_features % 8 == 0,
 * side % r == 0; x, y and weight each < 2^31 elements, tokens < 2^24.
 * siq_proj_bwd: dx and/or dweight may be NULL (not computed).  Workspace:
 * siq_proj_workspace_bytes (split-K partial sums; may be 0).  Deterministic.
 * ------------------------------------------------------------------------- */
size_t siq_proj_workspace_bytes(int64_t batch, int64_t side, int64_t vision_dim, int factor, int64_t out_features);

int siq_proj_fwd(const void* x, const void* weight, void* y, int64_t batch, int64_t side, int64_t vision_dim,
                 int factor, int64_t out_features, void* workspace, size_t workspace_bytes, void* stream);

int siq_proj_bwd(const void* x, const void* weight, const void* dy, void* dx, void* dweight, int64_t batch,
                 int64_t side, int64_t vision_dim, int factor, int64_t out_features, void* workspace,
                 size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------------
 * Vision-token splice fused with the embedding gather.
 *
 * Replaces, in SiQ_VLForCausalLM.forward (siq_vl/model/modeling.py:252-270),
 * the embedding lookup of input_ids (:253), the nonzero() of the image-token
 * positions (:257), their count check (:259-267) and the index assignment of
 * the flattened vision rows (:269-270):
 *   out[p] = vision[r]          if input_ids[p] == image_token_id, r = number
 *                               of image tokens before p (row-major order);
 *   out[p] = weight[input_ids[p]] otherwise.
 * input_ids [n_tokens] int64; weight [vocab, hidden], vision [n_vision,
 * hidden], out [n_tokens, hidden]: bf16, contiguous, 16-byte aligned;
 * hidden % 8 == 0.  Outputs (device): image_pos [n_vision] int32 = token index
 * of vision row r; counts[0] = image tokens found (the caller raises the
 * reference's ValueError when it differs from n_vision: rows of image tokens
 * beyond n_vision are written as zeros), counts[1] = ids outside [0, vocab)
 * (written as zeros; the reference's embedding would raise).  Workspace:
 * siq_splice_workspace_bytes(n_tokens).
 *
 * siq_gather_rows: dst[i] = src[rows[i]], i < n (rows of hidden bf16): the
 * backward's vision-row gradient (IndexPutBackward of :270) from image_pos;
 * rows[i] < 0 gives a zero row (image_pos slots past the image tokens found
 * hold -1).  The splice and the gather only copy 16-byte chunks of rows, so
 * rows of another dtype are passed as their bf16 view (an fp32 row of H
 * elements as 2H bf16).
 * ------------------------------------------------------------------------- */
size_t siq_splice_workspace_bytes(int64_t n_tokens);

int siq_splice_fwd(const int64_t* input_ids, int64_t n_tokens, const void* weight, int64_t vocab, int64_t hidden,
                   const void* vision, int64_t n_vision, int64_t image_token_id, void* out, int32_t* image_pos,
                   int64_t* counts, void* workspace, size_t workspace_bytes, void* stream);

int siq_gather_rows(const void* src, const int32_t* rows, int64_t n, int64_t hidden, void* dst, void* stream);

/* ---------------------------------------------------------------------------
 * Embedding-table gradient of the splice (the text model's input embeddings).
 *
 * Replaces the backward of the embedding lookup at siq_vl/model/modeling.py:253
 * together with the index assignment at :270 (IndexPutBackward zeroes the
 * overwritten image rows before the embedding backward): torch's
 * embedding_dense_backward with the image token as padding index.
 *   dweight[v] = sum of grad[p] over tokens p with input_ids[p] == v,
 * for v in [0, vocab) other than skip_id0 / skip_id1 (the image token and the
 * table's padding index; -1 for none); every other row is zero.  The sum is
 * fp32, in the order of torch's sorted embedding backward (each id's tokens
 * in position order, partial sums of at most 10 rows added in order), rounded
 * once; deterministic.  grad [n_tokens, hidden] and dweight [vocab, hidden]
 * contiguous, 16-byte aligned, both bf16 (dtype SIQ_DTYPE_BF16) or both fp32
 * (SIQ_DTYPE_FP32, the reference's fp32 master weights); hidden % 8 == 0.
 * Workspace: siq_embedding_bwd_workspace_bytes(n_tokens, vocab).
 * ------------------------------------------------------------------------- */
size_t siq_embedding_bwd_workspace_bytes(int64_t n_tokens, int64_t vocab);

int siq_embedding_bwd(const void* grad, const int64_t* input_ids, int64_t n_tokens, int64_t vocab, int64_t hidden,
                      int dtype, int64_t skip_id0, int64_t skip_id1, void* dweight, void* workspace,
                      size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------------
 * Activations in 8 bits for the backward pass.
 *
 * No counterpart in the reference, which keeps them in bf16 (and, with
 * gradient_checkpointing, one input for each decoder layer:
 * scripts/train.py:714).
 *
 * siq_pack8: x [numel] (dtype SIQ_DTYPE_BF16 or _FP32, contiguous) in codes
 * [numel] bytes and scales [ceil(numel / 32)] bytes, one for each 32
 * neighbours.  With a the largest magnitude of the 32, the scale byte b is the
 * biased exponent of a, one more where a would round past the largest code:
 *   SIQ_FORMAT_INT8: x = code * 2^(b - 133), code a signed byte in [-127, 127];
 *   SIQ_FORMAT_E4M3: x = code * 2^(b - 135), code an OCP e4m3 number.
 * b is at least 7 (int8) or 9 (e4m3), so steps are normal numbers: groups
 * whose largest magnitude lies below 2^-120 (2^-118) lose precision.  Codes are
 * rounded to nearest even, by at most half a step (int8; fp32 magnitudes
 * above 1.99 * 2^127: one step) or half a unit of their last place (e4m3).
 * b = 255 marks a group that holds an infinity or a NaN: all of it unpacks to
 * NaN.  siq_unpack8 writes code * step, exactly.
 * All pointers 16-byte aligned; numel at most 2^35.  No workspace.
 *
 * siq_swiglu8_fwd: h = silu(gate) up of rows x cols elements (the gated MLP
 * activation of transformers' Qwen2MLP), and gate and
 * up packed as siq_pack8 packs the contiguous [rows, cols] tensors; the four
 * packed outputs may be NULL together (nothing is kept: evaluation).  Rows are
 * gate_stride / up_stride elements apart (halves of one product); unless both
 * strides equal cols, they must be multiples of 16 bytes and cols of 8.  h is
 * contiguous.
 * siq_swiglu8_bwd: with g, u the unpacked values and s = 1 / (1 + exp(-g)),
 *   dup = dh g s,  dgate = dh u s (1 + g (1 - s)),  h = g s u
 * (h only if not NULL: the down projection's input for its weight gradient).
 * dh and h contiguous, dgate and dup with row strides as above.
 * Everything in fp32, rounded once to dtype.
 * ------------------------------------------------------------------------- */
int siq_pack8(const void* x, int64_t numel, int dtype, int format, void* codes, void* scales, void* stream);

int siq_unpack8(const void* codes, const void* scales, int64_t numel, int dtype, int format, void* x, void* stream);

int siq_swiglu8_fwd(const void* gate, const void* up, int64_t rows, int64_t cols, int64_t gate_stride,
                    int64_t up_stride, int dtype, int format, void* h, void* gate_codes, void* gate_scales,
                    void* up_codes, void* up_scales, void* stream);

int siq_swiglu8_bwd(const void* dh, const void* gate_codes, const void* gate_scales, const void* up_codes,
                    const void* up_scales, int64_t rows, int64_t cols, int64_t dgate_stride, int64_t dup_stride,
                    int dtype, int format, void* dgate, void* dup, void* h, void* stream);

/* ---------------------------------------------------------------------------
 * Losses of preference and policy training.
 *
 * No counterpart in the reference, which ends at supervised fine-tuning: what
 * follows it trains on pairs of answers, or on sampled ones with advantages,
 * over the same packed batches.  Inputs are fp32 per-token log-probabilities of
 * packed sequences (cu_seqlens int32 [sequences + 1]; cu[0] is taken as 0, and
 * tokens behind cu[sequences] belong to none: they count nowhere and their
 * gradient is zero), mask [tokens] bytes (0: the token does not count, whatever
 * its values; NULL: all count).  Sums are in fp64 and in a fixed order, no
 * atomics.  grad_loss: the loss's upstream gradient, a device scalar.
 *
 * siq_pref_fwd: the loss of paired sequences.  Pair i is sequences 2 i (chosen)
 * and 2 i + 1 (rejected) (SIQ_ORDER_INTERLEAVED), or i and pairs + i
 * (SIQ_ORDER_HALVES).  A sequence's score is the sum over its counted tokens
 * of policy - reference (reference NULL: of policy), divided by their number
 * when length_normalized (by 1 where none counts); x = score of chosen -
 * score of rejected:
 *   SIQ_PREF_SIGMOID: (1 - e) softplus(-beta x) + e softplus(beta x), e =
 *     label_smoothing;   SIQ_PREF_IPO: (x - 1 / (2 beta))^2;
 *   SIQ_PREF_HINGE: max(0, 1 - beta x).
 * *loss = their sum / pairs, or / *divisor (a device scalar) if not NULL;
 * chosen_rewards / rejected_rewards [pairs] = beta * score; coef [2 pairs] =
 * the loss's gradient with respect to a counted token of each sequence, which
 * siq_pref_bwd spreads over the tokens (dpolicy [tokens], written in full).
 *
 * siq_policy_fwd: the clipped policy loss.  r = exp(logp - old_logp); a token's
 * objective is min(r A, clip(r, 1 - clip_low, 1 + clip_high) A), and for A < 0
 * not below dual_clip * A (dual_clip 0: no such bound); its loss is -objective +
 * kl_coef * kl with x = reference - logp and kl = -x (SIQ_KL_K1), x^2 / 2 (_K2)
 * or e^x - 1 - x (_K3), left out at kl_coef 0 (it may be infinite) but for
 * *mean_kl.  advantages A: [tokens] (advantage_per_token) or [seqs].
 * SIQ_AGG_TOKEN: the mean over counted tokens; SIQ_AGG_SEQUENCE: the mean over
 * sequences of their counted tokens' mean (0 where none counts); with divisor
 * its value replaces the number of counted tokens, or of sequences.
 * cu_seqlens NULL: one sequence.  A token exactly at a border is not cut.
 * *loss, *mean_kl and *clip_fraction (the share of cut tokens), the
 * latter two over counted tokens, are 0 where none counts; dtoken [tokens]
 * (16-byte aligned) and weight [seqs] (SIQ_AGG_TOKEN: [1]) are what
 * siq_policy_bwd multiplies: dlogps = grad_loss weight dtoken (dlogps 16-byte
 * aligned).
 * ------------------------------------------------------------------------- */
#define SIQ_PREF_SIGMOID 0
#define SIQ_PREF_IPO 1
#define SIQ_PREF_HINGE 2
#define SIQ_ORDER_INTERLEAVED 0
#define SIQ_ORDER_HALVES 1
#define SIQ_AGG_TOKEN 0
#define SIQ_AGG_SEQUENCE 1
#define SIQ_KL_K1 0
#define SIQ_KL_K2 1
#define SIQ_KL_K3 2

size_t siq_pref_workspace_bytes(int64_t pairs, int64_t tokens);

int siq_pref_fwd(const float* policy, const float* reference, const void* mask, const int32_t* cu_seqlens,
                 int64_t pairs, int64_t tokens, int loss_type, int order, double beta, double label_smoothing,
                 int length_normalized, const float* divisor, float* loss, float* chosen_rewards,
                 float* rejected_rewards, float* coef, void* workspace, size_t workspace_bytes, void* stream);

int siq_pref_bwd(const float* grad_loss, const float* coef, const void* mask, const int32_t* cu_seqlens, int64_t pairs,
                 int64_t tokens, float* dpolicy, void* stream);

size_t siq_policy_workspace_bytes(int64_t seqs, int64_t tokens);

int siq_policy_fwd(const float* logps, const float* old_logps, const float* advantages, const void* mask,
                   const float* reference, const int32_t* cu_seqlens, int64_t seqs, int64_t tokens,
                   int advantage_per_token, int aggregation, int kl_type, double clip_low, double clip_high,
                   double dual_clip, double kl_coef, const float* divisor, float* loss, float* mean_kl,
                   float* clip_fraction, float* dtoken, float* weight, void* workspace, size_t workspace_bytes, void* stream);

int siq_policy_bwd(const float* grad_loss, const float* dtoken, const float* weight, const int32_t* cu_seqlens,
                   int64_t seqs, int64_t tokens, int aggregation, float* dlogps, void* stream);

/* ---------------------------------------------------------------------------
 * Token statistics and distillation (no reference counterpart): what a model
 * thinks of its tokens, and the loss of a student against what a teacher thinks.
 * Operands, rows that count, count and bad_labels as for siq_flp_fwd; logits
 * z = hidden weight^T / temperature exist only as one chunk's.
 *
 * siq_stats_fwd: for each counted row logp = ln softmax(z) at the label,
 * entropy = -sum p ln p, and with top_k > 0 (at most 128 and vocab) the largest
 * logits' ids in order, equal ones by lower id first (top_ids [n, top_k]), with
 * their log-probabilities (top_logp).  Rows that do not
 * count have 0, and ids of -1.  A row with a NaN logit has NaN log-probabilities
 * and ids in [0, vocab).  logp, entropy [n]; state [3, n] (or NULL) is what
 * siq_stats_bwd takes of them.  top_logp and top_ids may be NULL with top_k 0.
 * saved (siq_stats_saved_bytes, or NULL): the softmax numerators in bf16, kept for
 * the backward.
 * siq_stats_bwd: dhidden and / or dweight (NULL: not computed) from the upstream
 * gradients dlogp and dentropy [n] (NULL: zero),
 *   dz_j = dlogp ([j = label] - p_j) - dentropy p_j (ln p_j + entropy).
 * They may not overlap hidden.  From what the forward kept on the same inputs, or
 * (saved NULL) from logits that are formed again; chunk_tokens rows at a time.
 *
 * siq_distill: ids [n, top_k] (ids_bytes 8: int64, 4: int32) name a teacher's
 * tokens and teacher [n, top_k] their log-probabilities ln t; top_k in [1, 128].  An
 * id of -1, or a log-probability of -infinity, names none.  An id outside the
 * vocabulary, or named twice in a row that counts, is left out (twice: but for its
 * first place) and counted in counts[2].  With m = sum t, r = max(1 - m, 0), s =
 * softmax(z) at the named tokens and q its sum over all others:
 *   SIQ_DIVERGENCE_FORWARD: D = sum t (ln t - ln s), with tail != 0 also
 *     + r (ln r - ln q);
 *   SIQ_DIVERGENCE_REVERSE: D = sum s (ln s - ln t) + q (ln q - ln r), r at least
 *     2^-24; it needs a tail.
 * (Where every token is named there is no tail.)  *loss = sum over counted rows of
 * (1 - ce_weight) D + ce_weight CE, CE = -ln softmax(z) at the label, over the number
 * of them, or over *divisor (a device scalar) if not NULL; *divergence and
 * *cross_entropy its two parts, divided likewise.  ce_weight in [0, 1], and 0 where
 * temperature is not 1.  dhidden and dweight (NULL: not computed) are the gradients
 * of *loss; dhidden may not overlap hidden.  counts[0] = rows that count, counts[1] =
 * bad labels.
 * Everything in fixed orders: bitwise reproducible.
 * ------------------------------------------------------------------------- */
#define SIQ_DIVERGENCE_FORWARD 0
#define SIQ_DIVERGENCE_REVERSE 1

size_t siq_stats_saved_bytes(int64_t n, int64_t vocab);

size_t siq_stats_fwd_workspace_bytes(int64_t n, int64_t hdim, int64_t vocab, int top_k, int keep);

int siq_stats_fwd(const void* hidden, const void* weight, const int64_t* labels, int64_t n, int64_t hdim,
                  int64_t vocab, int64_t ignore_index, double temperature, int top_k, float* logp, float* entropy,
                  float* state, float* top_logp, int64_t* top_ids, int64_t* count, int64_t* bad_labels, void* saved,
                  size_t saved_bytes, void* workspace, size_t workspace_bytes, void* stream);

size_t siq_stats_bwd_workspace_bytes(int64_t n, int64_t hdim, int64_t vocab, int64_t chunk_tokens, int need_dweight,
                                     int have_saved);

int siq_stats_bwd(const void* hidden, const void* weight, const int64_t* labels, const float* state,
                  const float* dlogp, const float* dentropy, int64_t n, int64_t hdim, int64_t vocab,
                  int64_t ignore_index, double temperature, const void* saved, size_t saved_bytes, void* dhidden,
                  void* dweight, int64_t chunk_tokens, void* workspace, size_t workspace_bytes, void* stream);

size_t siq_distill_workspace_bytes(int64_t n, int64_t hdim, int64_t vocab, int top_k, int64_t chunk_tokens,
                                   int need_grads, int need_dweight);

int siq_distill(const void* hidden, const void* weight, const int64_t* labels, const void* ids, int ids_bytes,
                const float* teacher, int64_t n, int64_t hdim, int64_t vocab, int top_k, int64_t ignore_index,
                double temperature, double ce_weight, int divergence, int tail, const float* divisor, float* loss,
                float* mean_divergence, float* mean_cross_entropy, int64_t* counts, void* dhidden, void* dweight,
                int64_t chunk_tokens, void* workspace, size_t workspace_bytes, void* stream);

/* ---------------------------------------------------------------------------
 * Measurement support (no reference counterpart).
 *
 * siq_probe_clock: one wave per CU spins for about spin_ticks ticks of the
 * constant 100 MHz counter and writes out[0] = shader-clock cycles elapsed,
 * out[1] = 100 MHz ticks elapsed (device uint64[2]); the shader clock the GPU
 * ran at is out[0] / out[1] * 100 MHz.  spin_ticks in [1, 1e8].
 * ------------------------------------------------------------------------- */
int siq_probe_clock(uint64_t* out, int64_t spin_ticks, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* SIQ_KERNELS_H */

// Entry points of libferrite_hip.so for the Python package of the same tree alone. They keep the
// conventions of ferrite_hip.h (device pointers, sizes, a stream; 0 or a FERRITE_ERR_* code;
// nothing allocated, nothing synchronised), but are no part of its C ABI and change with the
// package.
#pragma once

#include <stdint.h>

extern "C" {

/*
 * The bf16 product for operands the matrix kernel cannot read in place: any M, N, K and
 * any 2-byte aligned pointers, either operand given transposed (as ferrite_hip_matmul_ex).
 * Operands whose rows do not start at 16-byte boundaries are first copied into the
 * workspace with their rows padded to a multiple of 8 elements; the workspace also holds
 * the K split's partials. It has ferrite_internal_matmul_ragged_workspace(...) bytes (0: none
 * needed; -1: sizes out of range, an operand of 2^33 elements or more among them), which
 * depends on the sizes and on the operands' alignment, and is 16-byte aligned; a smaller
 * one fails with FERRITE_ERR_INVALID_ARGUMENT. Its content need not survive the call.
 */
int64_t ferrite_internal_matmul_ragged_workspace(const void* x, const void* y, int64_t m, int64_t n, int64_t k,
                                                 int x_t, int y_t);
/*
 * 1 where that is the faster one, 0 where ferrite_hip_matmul_ex's own choice on untransposed operands is
 * (transposed ones copied first).
 */
int ferrite_internal_matmul_ragged_better(const void* x, const void* y, int64_t m, int64_t n, int64_t k, int x_t,
                                          int y_t);
int ferrite_internal_matmul_ragged(const void* x, const void* y, void* out, int64_t m, int64_t n, int64_t k, int x_t,
                                   int y_t, int out_dtype, void* workspace, int64_t workspace_bytes, void* stream);

/*
 * out[M,N] = x[M,K] . bf16(w[K,N]) (w_t: w holds [N,K]) for a bf16 x and a float w whose
 * elements are rounded to bf16 as they are read (model/gpt.py:95-104, :143: the casts of the
 * linear layers' weights and of the tied head's), with M <= 64 rows and a bf16 or float out.
 * With aux (bf16 out, w not transposed), the GELU epilogue: aux <- bf16(x . w), out <- bf16(gelu(aux)).
 * A workspace of ferrite_internal_linear_f32w_workspace(...) bytes (-1: sizes out of range),
 * 16-byte aligned, lets a deep K split; with less it does not.
 */
int64_t ferrite_internal_linear_f32w_workspace(const void* x, const float* w, int64_t m, int64_t n, int64_t k, int w_t);
int ferrite_internal_linear_f32w(const void* x, const float* w, void* out, void* aux, int64_t m, int64_t n, int64_t k,
                                 int w_t, int out_dtype, void* workspace, int64_t workspace_bytes, void* stream);

/*
 * ferrite_hip_decode_attention with q, k_new and v_new [B, H, D] given with one stride of
 * new_stride >= H * D elements (a multiple of 8) from a sequence to the next, as they lie in a
 * fused projection; the heads of a sequence are dense.
 */
int ferrite_internal_decode_attention(const void* q, const void* k_new, const void* v_new, void* k_cache, void* v_cache,
                                      const int32_t* pos, void* out, int64_t b, int64_t h, int64_t max_len, int64_t d,
                                      int64_t new_stride, int dtype, float scale, void* workspace,
                                      int64_t workspace_bytes, void* stream);

/*
 * out[r] = tok_emb[tokens[r]] + pos_emb[pos[r]] for one token per row (model/gpt.py:124-127 at the
 * positions of a decode step; without pos, row r is at position r % period, period <= seq),
 * summed and rounded in emb_dtype, then converted to out_dtype.
 * tok_emb [vocab, dim], pos_emb [seq, dim]. A negative index counts from the table's end; one
 * outside the table traps, as the gather of a tensor library does.
 */
int ferrite_internal_embed(const int64_t* tokens, const int32_t* pos, const void* tok_emb, const void* pos_emb, void* out,
                           int64_t rows, int64_t dim, int64_t vocab, int64_t seq, int64_t period, int emb_dtype,
                           int out_dtype, void* stream);

/*
 * Its gradients without pos, summed in f32 in a fixed order: dtok[vocab, dim], the rows of
 * dh[rows, dim] summed by token, and dpos[seq, dim], by position (zero from period on). Up to 1024
 * tokens in the vocabulary and whole sequences. The workspace, 16-byte aligned as dtok is, has
 * ferrite_internal_embed_bwd_workspace(...) bytes (-1: sizes out of range).
 */
int64_t ferrite_internal_embed_bwd_workspace(int64_t rows, int64_t period, int64_t dim, int64_t vocab, int64_t seq);
int ferrite_internal_embed_bwd(const int64_t* tokens, const void* dh, void* dtok, void* dpos, int64_t rows,
                               int64_t period, int64_t dim, int64_t vocab, int64_t seq, int dh_dtype, int emb_dtype,
                               void* workspace, int64_t workspace_bytes, void* stream);

/*
 * The heads of a fused projection qkv [B, S, (H + 2 Hkv) D] (its last dimension dense; batch_stride and
 * row_stride in elements), split, each q and k head normed and rotated: q [B, H, S, D], k and v
 * [B, Hkv, S, D], dense. wq, wk [D] of w_dtype; cos and sin f32 [table, rot / 2]; pos [B, S], or null
 * for position s of every sequence. A position outside the table gives NaN in its q and k rows. D even
 * and at most 512, rot even and at most D.
 */
int ferrite_internal_heads_rope(const void* qkv, int64_t batch_stride, int64_t row_stride, const void* wq,
                                const void* wk, const float* cos, const float* sin, const int32_t* pos, void* q, void* k,
                                void* v, int64_t b, int64_t s, int64_t h, int64_t hkv, int64_t d, int64_t rot,
                                int64_t table, int dtype, int w_dtype, int interleaved, float eps, void* stream);
/*
 * Its gradients from dense dq, dk and dv (null: zero): dqkv, dense, and the weights' in w_dtype, summed in f32
 * in a fixed order. The workspace has ferrite_internal_heads_rope_bwd_workspace(...) bytes (-1: sizes out of
 * range); its content need not survive the call.
 */
int64_t ferrite_internal_heads_rope_bwd_workspace(int64_t b, int64_t s, int64_t h, int64_t hkv, int64_t d);
int ferrite_internal_heads_rope_bwd(const void* qkv, int64_t batch_stride, int64_t row_stride, const void* wq,
                                    const void* wk, const float* cos, const float* sin, const int32_t* pos,
                                    const void* dq, const void* dk, const void* dv, void* dqkv, void* dwq, void* dwk,
                                    int64_t b, int64_t s, int64_t h, int64_t hkv, int64_t d, int64_t rot, int64_t table,
                                    int dtype, int w_dtype, int interleaved, float eps, void* workspace,
                                    int64_t workspace_bytes, void* stream);

/*
 * Attention of T <= 64 drafted nodes per sequence over the caches [B, Hkv, max_len, D] (D 64, 128 or 256): node t hangs on
 * node parents[b, t] < t, or on the committed tokens (-1), and sees the rows 0 .. pos[b] - 1, its ancestors and itself. Nodes' keys and
 * values go to rows pos[b] + t. A node whose parent is neither, or that hangs on such a one, is absent: nothing is written for it
 * and its output is zero. Where pos[b] < 0 or pos[b] + T > max_len nothing is written and the sequence's outputs are NaN. q [B, H, T, D],
 * k_new and v_new [B, Hkv, T, D] with dense last dimensions and the nine element strides (sequence, head, node of
 * each; whole 16 bytes); out [B, T, H, D], dense. H is a multiple of Hkv. The workspace, 16-byte aligned, has
 * ferrite_internal_tree_attention_workspace(...) bytes (-1: sizes out of range); its content need not survive the call. A head's
 * cached keys, and its nodes' rows with what lies between them, take at most 4 GiB less 128 KiB. A node's values that are not
 * finite reach only the rows that see it. How the sums are parted depends on the sizes and positions of the whole batch, so a
 * sequence's last bits may differ from batch to batch; for the same call they are the same. The caches must not overlap each
 * other or what lies from the first to the last element of q, k_new or v_new.
 */
int64_t ferrite_internal_tree_attention_workspace(int64_t b, int64_t h, int64_t hkv, int64_t t, int64_t max_len, int64_t d,
                                                  int dtype);
int ferrite_internal_tree_attention(const void* q, const void* k_new, const void* v_new, void* k_cache, void* v_cache,
                                    const int32_t* pos, const int32_t* parents, void* out, const int64_t* strides,
                                    int64_t b, int64_t h, int64_t hkv, int64_t t, int64_t max_len, int64_t d, int dtype,
                                    float scale, void* workspace, int64_t workspace_bytes, void* stream);

/*
 * The drafted nodes that greedy decoding would have taken: from node 0 (its parent -1), to the child that holds
 * the argmax of the node's logits [B, T, V], while there is one. path [B, T] (-1 behind the visited nodes), count [B],
 * following [B] (the argmax at the last node; -1 with count 0 where node 0 is absent). 1 <= T <= 64, B T <= 65535. A
 * node whose parent is not -1 or an earlier one is absent and its logits are not read. The workspace has
 * ferrite_internal_accept_drafts_workspace(...) bytes (-1: sizes out of range), 8-byte aligned.
 */
int64_t ferrite_internal_accept_drafts_workspace(int64_t b, int64_t t, int64_t v);
int ferrite_internal_accept_drafts(const void* logits, const int64_t* tokens, const int32_t* parents, int32_t* path,
                                   int32_t* count, int64_t* following, int64_t b, int64_t t, int64_t v, int dtype,
                                   void* workspace, int64_t workspace_bytes, void* stream);

/*
 * Rows pos[b] + path[b, i] of the caches [layers, B, H, max_len, D] to pos[b] + i, i < count[b], in place; a path ends
 * at the first entry that is not larger than the one before (or negative) or whose row lies outside the cache. 1 <= T <= 64. The caches
 * must not overlap.
 */
int ferrite_internal_compact_cache(void* k_cache, void* v_cache, const int32_t* pos, const int32_t* path,
                                   const int32_t* count, int64_t layers, int64_t b, int64_t h, int64_t max_len, int64_t d,
                                   int64_t t, int dtype, void* stream);

/*
 * Layer norm of rows of h = x + r (rounded to x's type and stored; h = x without r): y = (h - mean) rstd w + b. w and b (or
 * null) [dim] of w_dtype. stats, or null, receives f32 (mean, rstd) of each row. 1 <= dim < 2^25; any alignment.
 */
int ferrite_internal_layernorm(const void* x, const void* r, const void* w, const void* b, void* h, void* y, float* stats,
                               int64_t rows, int64_t dim, int x_dtype, int w_dtype, float eps, void* stream);
/*
 * Its gradients from dy, dd (h's own gradient, or null) and the forward's h and stats: dh, of x and r alike, and dw and db (or null), in
 * w_dtype, summed in f32 in a fixed order. The workspace has ferrite_internal_layernorm_bwd_workspace(...) bytes (-1: sizes out of
 * range); its content need not survive the call.
 */
int64_t ferrite_internal_layernorm_bwd_workspace(int64_t rows, int64_t dim);
int ferrite_internal_layernorm_bwd(const void* h, const void* w, const void* dy, const void* dd, const float* stats, void* dh,
                                   void* dw, void* db, int64_t rows, int64_t dim, int x_dtype, int w_dtype, void* workspace,
                                   int64_t workspace_bytes, void* stream);

/*
 * norm = sqrt(sum of all squares) of n tensors grads[i] of numel[i] elements of dtypes[i], added in 64 bits in a fixed order; where
 * it is a finite float and most / (norm + 1e-6) < 1 every element is multiplied by that. grads, numel and dtypes are host arrays,
 * read before the call returns. The tensors must not overlap; any alignment. The workspace, 8-byte aligned, has
 * ferrite_internal_clip_workspace(n) bytes (-1: n out of range); its content need not survive the call.
 */
int64_t ferrite_internal_clip_workspace(int64_t n_tensors);
int ferrite_internal_clip(int64_t n_tensors, void* const* grads, const int64_t* numel, const int32_t* dtypes, double most,
                          float* norm, void* workspace, int64_t workspace_bytes, void* stream);

/*
 * out[i] = scale table[tokens[i]] in f32, rounded once to out_dtype; table [vocab, dim]. A token outside the table gives NaN;
 * with `indexing` a negative one counts from the table's end, and one outside the table stops the program. rows < 2^27,
 * vocab < 2^31 - 1, dim <= 64 * 65535; any alignment.
 */
int ferrite_internal_embedding(const int64_t* tokens, const void* table, void* out, int64_t rows, int64_t dim, int64_t vocab,
                               float scale, int indexing, int table_dtype, int out_dtype, void* stream);
/*
 * Its gradient: dtable[t] = scale times the sum of dy's rows of token t, in f32 in a fixed order, zero where there is none. Tokens
 * outside the table, and `padding` (-1: none), add nothing. The workspace, 16-byte aligned, has
 * ferrite_internal_embedding_bwd_workspace(...) bytes (-1: sizes out of range); its content need not survive the call.
 */
int64_t ferrite_internal_embedding_bwd_workspace(int64_t rows, int64_t dim, int64_t vocab);
int ferrite_internal_embedding_bwd(const int64_t* tokens, const void* dy, void* dtable, int64_t rows, int64_t dim,
                                   int64_t vocab, int64_t padding, float scale, int indexing, int dy_dtype, int table_dtype,
                                   void* workspace, int64_t workspace_bytes, void* stream);

/*
 * out[M,N] = act(x[M,K] . w[K,N] + bias) + residual: x, residual, out and aux of `dtype`, w of `w_dtype` (that of x, or float with a
 * bf16 x of up to 64 rows, rounded as it is read), bias [N] of bias_dtype. bias, residual and aux may be null; aux receives the
 * pre-activation. residual may be neither out nor overlap it. The workspace, 16-byte aligned, has
 * ferrite_internal_linear_workspace(...) bytes (-1: sizes out of range); its content need not survive the call.
 */
#define FERRITE_ACT_NONE 0
#define FERRITE_ACT_RELU 1
#define FERRITE_ACT_GELU 2 /* tanh form */
#define FERRITE_ACT_SILU 3
int64_t ferrite_internal_linear_workspace(const void* x, const void* w, const void* out, int64_t m, int64_t n, int64_t k,
                                          int dtype, int w_dtype);
int ferrite_internal_linear(const void* x, const void* w, const void* bias, const void* residual, void* out, void* aux,
                            int64_t m, int64_t n, int64_t k, int dtype, int w_dtype, int bias_dtype, int act, void* workspace,
                            int64_t workspace_bytes, void* stream);
/*
 * out[M,N] = op(x) . op(y) over f32 operands (x_t: x holds [K,M]; y_t: y holds [N,K]) of any alignment, read as they lie. The workspace,
 * 16-byte aligned, has ferrite_internal_matmul_f32_workspace(...) bytes; with less K is not cut. -1: sizes that it does not take, or
 * for which ferrite_hip_matmul_ex on untransposed operands is the faster one.
 */
int64_t ferrite_internal_matmul_f32_workspace(const float* x, const float* y, int64_t m, int64_t n, int64_t k, int x_t, int y_t);
int ferrite_internal_matmul_f32(const float* x, const float* y, float* out, int64_t m, int64_t n, int64_t k, int x_t, int y_t,
                                void* workspace, int64_t workspace_bytes, void* stream);
/*
 * du = dy act'(u) and db, the sums of du's rows before its rounding, in f32 in a fixed order: [rows, dim] of `dtype`, db [dim] of
 * bias_dtype or null. Without u du is dy, and is not written. The workspace for db has ferrite_internal_act_grad_workspace(...)
 * bytes (-1: sizes out of range).
 */
int64_t ferrite_internal_act_grad_workspace(int64_t rows, int64_t dim);
int ferrite_internal_act_grad(const void* dy, const void* u, void* du, void* db, int64_t rows, int64_t dim, int act, int dtype,
                              int bias_dtype, void* workspace, int64_t workspace_bytes, void* stream);

}  // extern "C"

/* C ABI of the B200-native E.T. encoder hot path.
 *
 * Every function returns an int status (ET_OK = 0) and never exits the process; the text of the
 * last failure on the calling thread is available from et_last_error(). Pointers named *_host
 * are host pointers; all other data pointers are device pointers to fp16 ("half") or int32 data.
 * `stream` is a cudaStream_t passed as void* (NULL = the default stream). Work is stream-ordered
 * and no call synchronises unless its comment says so.
 *
 * Each declaration cites the interface of the reference project (cctry/E.T., paths inside that
 * project) that it stands in for.
 */
#ifndef ET_B200_H
#define ET_B200_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define ET_B200_VERSION 100

#define ET_OK 0
#define ET_ERR_INVALID 1        /* bad argument (null pointer, dimension, malformed sparse format) */
#define ET_ERR_CUDA 2           /* a CUDA runtime/driver call failed */
#define ET_ERR_UNSUPPORTED 3    /* valid but outside what the kernels cover */
#define ET_ERR_DEVICE_TIMEOUT 4 /* a bounded device-side wait gave up */

const char* et_last_error(void);
int et_version(void);

/* ---- residual add + LayerNorm -----------------------------------------------------------
 * in_out[num x size] <- LayerNorm(in_out + skip) * gamma + beta, eps 1e-6, fp32 arithmetic.
 * Replaces skip_layernorm_kernelLauncher (kernels/kernels.h:3-5, kernels/skip_layernorm.cu:101-112). */
int et_skip_layernorm(void* in_out, const void* skip, const void* gamma, const void* beta, int num,
                      int size, void* stream);

/* ---- fused additive mask + softmax over score matrices ----------------------------------
 * scores[nmat][seq_len][seq_len] <- softmax_rows(scores + mask), in place; mask [seq_len x seq_len]
 * is shared by all matrices and may be NULL; keys >= valid_len are excluded and written as 0.
 * Replaces the mask + softmax stage of sharedQK_attention_kernelLauncher (kernels/attention.cu:291-323)
 * and softmax_blk (kernels/attention.cu:10-48). */
int et_softmax_mask(void* scores, const void* mask, int nmat, int seq_len, int valid_len, void* stream);

/* ---- tile-pruned linear ------------------------------------------------------------------
 * Weight object built from HOST arrays in the reference's 16x16 tile format: row_ptr[out_feat/16+1],
 * row_offset[ntile] (input-feature offset of each kept tile, a multiple of 16),
 * data[ntile*256] with data[i*256 + n*16 + k] = W[16*r + n][row_offset[i] + k], bias[out_feat]
 * (NULL = zeros). Arrays are validated and copied; `size` is the expected token count (a hint).
 * Synchronises the device once. Replaces Linear_tile::Linear_tile (encoder/Linear.h:18-24). */
typedef struct et_tile_weight et_tile_weight;
int et_tile_weight_create(et_tile_weight** out, int in_feat, int out_feat, int size, int ntile,
                          const void* data_host, const int* row_ptr_host,
                          const int* row_offset_host, const void* bias_host);
int et_tile_weight_destroy(et_tile_weight* w);
/* Y[tokens x out_feat] = X[tokens x in_feat] . W^T + bias, tanh-GELU when gelu != 0.
 * Replaces Linear_tile::run (encoder/Linear.h:36-45). */
int et_tile_linear(const et_tile_weight* w, void* Y, const void* X, int tokens, int gelu, void* stream);
/* Reads and clears the weight's device error word (synchronises): ET_ERR_DEVICE_TIMEOUT and the
 * code in *code when a bounded wait inside the kernel gave up since the last check. */
int et_tile_weight_check(const et_tile_weight* w, int* code);
/* Extension (no counterpart in the reference): what weights created AFTERWARDS are packed for. 0 (default): the
 * shortest duration of one launch on an otherwise idle GPU (tiles spread over as many SMs as possible). 1: the
 * least SM time per launch (fewer, larger tiles), for callers that keep several independent batches in flight on
 * separate streams, where all SMs are busy anyway. Process-wide. */
#define ET_GOAL_LATENCY 0
#define ET_GOAL_THROUGHPUT 1
int et_set_tuning_goal(int goal);
/* Extension: whether the caller needs Q K^T accumulated in fp32 (the reference's kernels accumulate their scores in fp16,
 * kernels/attention.cu:82, `c_t<half>`). The tcgen05 attention kernel always does, so both settings give the same result (worst
 * output element 2e-3 for |q.k| up to 390); the setting is kept and read back for callers that make it. Process-wide. */
int et_set_attention_scores_fp32(int on);
int et_attention_scores_fp32(void);
/* info[6] = {block_rows_per_cta, n_chunks, k_chunks, stages, stage_bytes, packed_bytes}. The form the weight was packed in
 * for the expected token count: tile (stage_bytes > 0), dense (stage_bytes 0, stages = CTAs that share a tile's K range), or
 * activations resident in tensor memory (stages and stage_bytes 0; the chunks are groups of features, every CTA takes a
 * range of them). */
int et_tile_weight_info(const et_tile_weight* w, int* info);
/* Same contraction from DEVICE-resident tile arrays, K = in_feat explicit. The packed form of a
 * weight is built on its first use (device-to-host copy, synchronous: not inside a stream capture) and cached
 * by the three array addresses, N and K; the bias is read from the caller's pointer at every call. Call
 * et_tile_spmm_cache_clear() after changing a weight in place AND after freeing one: a new weight of the same
 * shape that the allocator places at the same addresses would otherwise be served the old packed copy
 * (objects that own their weight, et_tile_weight_create / Linear_tile, have no such hazard). Replaces
 * tile_spmm_add_bias_kernelLauncher / tile_spmm_add_bias_gelu_kernelLauncher
 * (kernels/kernels.h:13-20, kernels/linear.cu:152-167), whose missing K is the row pitch of X. */
int et_tile_spmm_bias(void* Y, const void* X, const int* W_row_ptr, const int* W_row_offset,
                      const void* W_data, int M, int N, int K, const void* bias, int gelu, void* stream);
int et_tile_spmm_cache_clear(void);

/* ---- row-pruned linear ---------------------------------------------------------------------
 * Only row_id_size output features are kept; row_id_host[] holds their original indices, strictly
 * ascending; weight_host is the compact [row_id_size x in_feat] matrix, bias_host[row_id_size] (NULL =
 * zeros). The output has nrow = row_id_size rounded up to 16 columns (zero beyond row_id_size).
 * head_ptr[h] = number of kept rows below h*(out_feat/nhead), h = 0..nhead.
 * Replaces Linear_row::Linear_row (encoder/Linear.h:66-67, encoder/Linear.cu:60-91). */
typedef struct et_row_weight et_row_weight;
int et_row_weight_create(et_row_weight** out, int in_feat, int out_feat, int size, const void* weight_host,
                         const int* row_id_host, int row_id_size, const void* bias_host, int nhead);
int et_row_weight_destroy(et_row_weight* w);
/* out[tokens x nrow] = in . W^T + bias. Replaces Linear_row::run (encoder/Linear.h:68-71) and
 * row_spmm_add_bias_kernelLauncher (kernels/kernels.h:7-11, kernels/linear.cu:18-34); no cuBLAS handle. */
int et_row_linear(const et_row_weight* w, void* out, const void* in, int tokens, void* stream);
/* Same contraction from a DEVICE-resident dense compact weight [N x K], N and K multiples of 16 (the
 * reference pads N to 16): out[M x N] = in[M x K] . weight^T + bias. Packed on first use and cached by
 * weight address, N and K, with the same address-reuse hazard as et_tile_spmm_bias (et_tile_spmm_cache_clear
 * drops the cache); the bias is read from the caller's pointer at every call. Replaces row_spmm_add_bias_kernelLauncher
 * (kernels/kernels.h:7-11, kernels/linear.cu:18-34) without its cuBLAS handle and algorithm. */
int et_row_spmm_bias(void* out, const void* in, const void* weight, const void* bias, int M, int N, int K,
                     void* stream);
/* The public members of Linear_row that the encoder reads (encoder/encoder.cu:76-79): any of the
 * output pointers may be NULL. head_ptr_host receives nhead+1 ints. */
int et_row_weight_meta(const et_row_weight* w, int* nrow, int* row_id_size, const int** row_id_dev,
                       const int** head_ptr_dev, int* head_ptr_host);

/* ---- attention --------------------------------------------------------------------------------
 * out[seq_len x d_model], head h in columns [h*hd, (h+1)*hd): softmax(Q_h K_h^T / sqrt(hd) + mask) V_h.
 * mask: additive [seq_len x seq_len] fp16 shared by all heads, or NULL. Any seq_len >= 0.
 * Replaces OTF_attention_kernelLauncher (kernels/kernels.h:22-24, kernels/attention.cu:122-134). */
int et_attention_otf(void* out, const void* Q, const void* K, const void* V, const void* mask, int seq_len,
                     int d_model, int nhead, void* stream);
/* V compact [seq_len x nnz_col_v]; head h owns compact columns [v_head_ptr[h], v_head_ptr[h+1]); result
 * column j is stored at out column v_col_id[j], every other out column is written as 0.
 * Replaces Prune_attention_kernelLauncher (kernels/kernels.h:26-30, kernels/attention.cu:252-271). */
int et_attention_prune(void* out, const void* Q, const void* K, const void* V, const int* v_col_id,
                       const int* v_head_ptr, int nnz_col_v, const void* mask, int seq_len, int d_model,
                       int nhead, void* stream);
/* QK[nhead][seq_len][seq_len] = Q_h K_h^T / sqrt(hd), Q and K with row pitch d_model.
 * Replaces the cublasHgemmStridedBatched call of Encoder_length::run (encoder/encoder.cu:126-130). */
int et_qk_scores(void* QK, const void* Q, const void* K, int seq_len, int d_model, int nhead, void* stream);
/* out = softmax(QK + mask) V per head from precomputed scores.
 * Replaces sharedQK_attention_kernelLauncher (kernels/kernels.h:32-34, kernels/attention.cu:342-350). */
int et_attention_sharedqk(void* out, const void* QK, const void* V, const void* mask, int seq_len,
                          int d_model, int nhead, void* stream);
/* Attention for callers that cannot allocate device memory (no counterpart in the reference). Same
 * arguments and result as et_attention_otf, computed through score matrices kept in an 8 MiB device array
 * that is part of the library image, so the call allocates nothing: not with cudaMalloc and not through
 * any library. Meant for hosts with a fixed memory plan (a real-time loop, a plugin whose host process
 * owns the allocator). Limit: nhead * seq_len * seq_len <= 16 * 512 * 512, otherwise ET_ERR_UNSUPPORTED.
 * The first call on each device looks up the array's device address; make that call before any stream
 * capture starts. All calls on a device share the array: issue them on one stream, calls that overlap
 * on the GPU race. Nothing needs clearing between calls. */
int et_attention_static_scores(void* out, const void* Q, const void* K, const void* V, const void* mask,
                               int seq_len, int d_model, int nhead, void* stream);
/* Reads and clears the current device's error word of the tensor-core attention kernel (synchronises):
 * ET_ERR_DEVICE_TIMEOUT and the code in *code (21: the issuing thread's wait, 22: the final accumulator wait, 23: a warp
 * that copies masks)
 * when a bounded wait inside the kernel gave up since the last check; the rows of that CTA are then not
 * written. The word is one per device, shared by every launch on it, those of et_attention_rules (24: single tokens) and et_adapter_add (51) among them. No counterpart in the reference, whose
 * only error handling is cudaChk's exit(1) (encoder/utils.h:4-12). */
int et_attention_check(int* code);
/* Batched, variable-length form (no counterpart in the reference, which handles one sequence per call):
 * sequences are packed back to back; cu_seqlens (device, batch+1 ints) gives their token offsets, or NULL
 * for `batch` sequences of uniform_len tokens. valid_lens (device, may be NULL) excludes keys at or beyond
 * valid_lens[b] (key padding). Q and K share qk_pitch; qk_head_ptr / v_head_ptr + v_col_id (device, may be
 * NULL) select compact per-head column windows as in et_attention_prune. max_seq_len: the longest sequence
 * when cu_seqlens is given (0 = unknown); it only selects between the tcgen05 kernel for heads of 64 and the general
 * kernel. */
int et_attention_batch(void* out, const void* Q, const void* K, const void* V, int qk_pitch, int v_pitch,
                       const int* qk_head_ptr, const int* v_col_id, const int* v_head_ptr, const void* mask,
                       int mask_ld, const int* cu_seqlens, const int* valid_lens, int batch, int uniform_len,
                       int max_seq_len, int total_tokens, int d_model, int nhead, void* stream);

/* ---- rotary positions over several axes (no counterpart in the reference, whose encoders place tokens by what their input holds) ----
 * Turns the features of every head of Q and K in pairs: pair i of token t by the angle positions[t * n_axes + axis[i]] * inv_freq[i]
 * (taken in 64 bits), (x, y) -> (x cos - y sin, x sin + y cos). Pairs are features i and i + rot_dim / 2 of a head, or 2i and 2i + 1
 * when interleaved != 0; features from rot_dim on are passed on unchanged. positions [tokens x n_axes] int32, inv_freq [rot_dim / 2]
 * fp32 and axis [rot_dim / 2] int32 are device arrays; a pair whose axis is not 0 .. n_axes - 1 is not turned. Rows may be slices of
 * wider ones (pitches in elements): Q and K as a fused projection leaves them. q_out may be q and k_out may be k, with equal pitches;
 * any other overlap is the caller's error. nhead_q or nhead_k may be 0. head_dim 2 to 256, rot_dim even. Rows and heads that start on 16
 * bytes go fastest. */
int et_rotary_axes(void* q_out, const void* q, int q_out_pitch, int q_pitch, int nhead_q, void* k_out, const void* k, int k_out_pitch,
                   int k_pitch, int nhead_k, int head_dim, int rot_dim, const int* positions, int n_axes, const float* inv_freq,
                   const int* axis, int interleaved, int tokens, void* stream);
/* The same call, its arguments in one structure: for callers to whom each argument of a foreign call costs time. So for the other calls below. */
typedef struct et_rotary_axes_args {
    void* q_out; const void* q; void* k_out; const void* k;
    const int* positions; const float* inv_freq; const int* axis; void* stream;
    int q_out_pitch, q_pitch, nhead_q, k_out_pitch, k_pitch, nhead_k, head_dim, rot_dim, n_axes, interleaved, tokens;
} et_rotary_axes_args;
int et_rotary_axes_by(const et_rotary_axes_args* args);

/* ---- low-rank adapters of many requests beside a shared projection (no counterpart in the reference, which holds one set of weights) ----
 * A bank holds n_slots adapters of one projection, each of rank up to max_rank (1 to 128): A [rank x in_feat], B [out_feat x rank] and a
 * scale. It allocates its memory on the current device and synchronises it, as et_adapter_bank_set does, which copies an adapter from HOST
 * arrays into a slot (rank 0: the slot is empty again): not while another thread launches with the bank. in_feat and out_feat are multiples of 16.
 * The weights are held in two layouts (for few tokens and for many), ranks rounded up to 16, 32, 64 or 128. */
typedef struct et_adapter_bank et_adapter_bank;
int et_adapter_bank_create(et_adapter_bank** out, int in_feat, int out_feat, int max_rank, int n_slots);
int et_adapter_bank_destroy(et_adapter_bank* bank);
int et_adapter_bank_set(et_adapter_bank* bank, int slot, int rank, const void* a_host, const void* b_host, float scale);
/* out[t] = base[t] + scale_a B_a (A_a x[t]) for the tokens of each sequence, a = adapter_ids[sequence] (device, batch ints; an id that
 * is no slot, or an empty one, adds nothing). base is what the shared projection left (et_tile_linear, et_row_linear); out may be base with the same
 * pitch, and overlaps x in nothing. cu_seqlens (device, batch + 1 ints) are the sequences' token offsets, or NULL: one token each (single tokens of many requests). Rows of
 * out in no sequence are left as they are. tokens: the rows that there are; none beyond is touched. Rows start on 16 bytes (pitches multiples
 * of 8). Sums in fp32; A x is rounded to fp16, each row scaled so that it can not overflow. */
int et_adapter_add(const et_adapter_bank* bank, void* out, const void* base, const void* x, int out_pitch, int base_pitch, int x_pitch,
                   const int* cu_seqlens, const int* adapter_ids, int batch, int tokens, void* stream);
typedef struct et_adapter_add_args {
    const et_adapter_bank* bank; void* out; const void* base; const void* x;
    const int* cu_seqlens; const int* adapter_ids; void* stream;
    int out_pitch, base_pitch, x_pitch, batch, tokens;
} et_adapter_add_args;
int et_adapter_add_by(const et_adapter_add_args* args);

/* ---- attention with rules on its scores (no counterpart in the reference, whose masks are additive and shared by all heads) ----
 *   score(q, k) = cap tanh(scale Q_q . K_k / cap) + bias(k - q);   out_q = sum of softmax(score) V_k over the keys that q sees
 * A query that sees no key gets zeros; what it does not see takes no part, whatever it holds (infinities, not a number). What it sees and is not a
 * number makes its row so; such rows are computed again one by one, which is slow. Scores and sums are fp32, the weights of V fp16. Fast are heads of a
 * multiple of 16 up to 128 in rows that start on 16 bytes; a kernel of single queries takes the others. */
typedef struct et_score_rules {
    float scale;               /* 0: 1 / sqrt(head_dim) */
    float cap;                 /* 0: scores are not capped */
    const float* slopes;       /* [nhead] or NULL: bias = -slopes[head] |k - q| */
    const void* distance_bias; /* fp16 [nhead][2 reach + 1] or NULL: bias = distance_bias[head][reach + max(-reach, min(reach, k - q))] */
    int reach;
    int window_left;           /* keys before q - window_left are not seen; below 0: no limit */
    int window_right;          /* keys behind q + window_right are not seen (0: none behind q); below 0: no limit */
    const int* prefix_lens;    /* [batch] or NULL: the first prefix_lens[sequence] keys are seen whatever the window is */
    const int* q_docs;         /* [q_tokens] and [k_rows], or both NULL: a query sees only keys of its own document (of those that */
    const int* k_docs;         /* the window and the prefix leave); documents below 0 see and are seen by nothing */
} et_score_rules;
/* Q and out [q_tokens x nhead * head_dim], K and V [k_rows x nhead_kv * head_dim], nhead a multiple of nhead_kv (query head h reads
 * K/V head h / (nhead / nhead_kv)), head_dim 1 to 256, each with a pitch of its own in elements. Sequence b has the queries of rows
 * cu_seqlens[b] .. cu_seqlens[b + 1] (device, batch + 1 ints; NULL: max_q_len each). Its keys:
 *   k_start NULL: the rows of its queries; the first k_lens[b] of them where k_lens is given (key padding). Query i is at position i.
 *   k_start given (device, batch ints): rows k_start[b] .. k_start[b] + k_lens[b], kept from before; the last query is at the last
 *     key: query i is at position k_lens[b] - (number of queries) + i. Places may overlap (a shared beginning).
 * All arrays of the rules are device arrays. max_q_len and max_k_len: at least the longest sequence's queries and keys; keys beyond
 * max_k_len, or beyond k_rows, are not seen. Single tokens (max_q_len 1 with k_start) take a kernel that splits the keys. scratch: device memory of
 * et_attention_rules_scratch_size bytes when documents are given (contents do not matter; calls that may overlap need one each), else NULL.
 * out may not overlap the inputs. Rows of out in no sequence are left as they are. The first call on a device looks up the device's error
 * word (et_attention_check): make it before a stream capture, as et_adapter_add's. */
int et_attention_rules(void* out, const void* Q, const void* K, const void* V, int out_pitch, int q_pitch, int k_pitch, int v_pitch,
                       int nhead, int nhead_kv, int head_dim, const int* cu_seqlens, const int* k_start, const int* k_lens, int batch,
                       int q_tokens, int k_rows, int max_q_len, int max_k_len, const et_score_rules* rules, void* scratch,
                       size_t scratch_bytes, void* stream);
size_t et_attention_rules_scratch_size(int batch, int max_k_len);
typedef struct et_attention_rules_args {
    void* out; const void* Q; const void* K; const void* V;
    const int* cu_seqlens; const int* k_start; const int* k_lens; void* scratch; size_t scratch_bytes; void* stream;
    et_score_rules rules;
    int out_pitch, q_pitch, k_pitch, v_pitch, nhead, nhead_kv, head_dim, batch, q_tokens, k_rows, max_q_len, max_k_len;
} et_attention_rules_args;
int et_attention_rules_by(const et_attention_rules_args* args);

/* ---- rows in 8 bits (no counterpart in the reference, which knows fp16 alone) ----
 * Root-mean-square norm with the residual's addition: h = x + skip, out = h / sqrt(mean(h^2) + eps) * gamma. x, skip (NULL: nothing is added), gamma [width] and
 * residual (NULL, or receives h) are fp16, the arithmetic fp32. scales NULL: out is fp16. scales [ceil(width / 128)][rows] fp32: out is e4m3 (one byte), a scale for
 * each 128 features of a row, the largest size among them / 448; out times scale stands for the value. Rows may be slices of wider ones
 * (pitches in elements). residual and an fp16 out may lie where x or skip lies, with the same pitch; any other overlap is the caller's error. width 1 to 32768, eps above 0 and at
 * most 1. Fast are widths of a multiple of 8 up to 16384 in rows that start on 16 bytes (codes: on 8). Values that are not finite make codes or scales that are not numbers. */
typedef struct et_skip_rmsnorm_args {
    void* out; const void* x; const void* skip; const void* gamma; void* residual; float* scales; void* stream;
    int out_pitch, x_pitch, skip_pitch, residual_pitch, rows, width;
    float eps;
} et_skip_rmsnorm_args;
int et_skip_rmsnorm(const et_skip_rmsnorm_args* args);
/* The same without the norm: rows of fp16 brought to e4m3 with scales, the input of a linear that no norm precedes. */
typedef struct et_quantise_rows_args {
    void* out; float* scales; const void* x; void* stream;
    int out_pitch, x_pitch, rows, width;
} et_quantise_rows_args;
int et_quantise_rows(const et_quantise_rows_args* args);

/* ---- linear with operands in e4m3 (no counterpart in the reference) ----
 * Y[tokens x out_feat] = X . W^T + bias, tanh-GELU when gelu != 0, in fp16, of values that are code times scale: X [tokens x in_feat] e4m3 with x_scales
 * [ceil(in_feat / 128)][tokens] (et_skip_rmsnorm, et_quantise_rows), W [out_feat x in_feat] e4m3 with scales [ceil(out_feat / 128)][ceil(in_feat / 128)], one for each 128 x 128 block. A weight is
 * made from HOST arrays, which are copied (bias fp16 or NULL), on the current device; synchronises it. in_feat and out_feat are multiples of 16. Products and sums in
 * fp32. Rows start on 16 bytes (pitch of X a multiple of 16, of Y of 8). Y overlaps X in nothing. */
typedef struct et_fp8_weight et_fp8_weight;
int et_fp8_weight_create(et_fp8_weight** out, int in_feat, int out_feat, const void* codes_host, const float* scales_host, const void* bias_host);
int et_fp8_weight_destroy(et_fp8_weight* w);
typedef struct et_fp8_linear_args {
    const et_fp8_weight* weight; void* y; const void* x; const float* x_scales; void* stream;
    int y_pitch, x_pitch, tokens, gelu;
} et_fp8_linear_args;
int et_fp8_linear(const et_fp8_linear_args* args);
/* Reads and clears the weight's device error word, as et_tile_weight_check. */
int et_fp8_weight_check(const et_fp8_weight* w, int* code);

/* ---- a cache of keys and values in int8 pages (no counterpart in the reference, which keeps nothing between calls) ----
 * codes [pages][2][heads][page][head_dim] int8 (K, then V) and scales [pages][2][heads][page] fp32, for each row of a head the largest size / 127: code times scale is the value.
 * A slot is page number x page + row. et_kv_cache_write: rows t of K and V [tokens x heads * head_dim] fp16 go to slots[t], code = value / scale to the
 * nearest (ties to even). et_kv_cache_read: rows of the cache come back to K and V. A slot that there is not (below 0: padding) is passed over: nothing is written, and rows of
 * K and V that are read to stay as they are. Slots of one write differ: of two rows for one place any mixture may stay. head_dim a multiple of 16 up to 256, page a multiple of 16, codes start on
 * 16 bytes; rows of K and V may be slices of wider ones, fast where they start on 16 bytes. A row with a value that is not finite becomes a row that is not a number. */
typedef struct et_kv_cache_args {
    void* codes; float* scales; void* k; void* v; const int* slots; void* stream;
    int k_pitch, v_pitch, tokens, pages, heads, page, head_dim;
} et_kv_cache_args;
int et_kv_cache_write(const et_kv_cache_args* args);
int et_kv_cache_read(const et_kv_cache_args* args);

/* ---- attention of drafted tokens over that cache (no counterpart in the reference) ----
 *   out_q = sum of softmax(scale q . k) v over the keys that q sees, of values that are code times scale
 * q and out [q_tokens x nhead * head_dim] fp16, nhead a multiple of nhead_kv (query head h reads K/V head h / (nhead / nhead_kv)). Sequence b has the drafted tokens of rows
 * cu_seqlens[b] .. cu_seqlens[b + 1] (device, batch + 1 ints; NULL: max_q_len each), at most max_q_len of them, at most 64. Its keys are k_lens[b] rows of the pages
 * table[b][0], table[b][1], .. (device, [batch][table_width]), those of the n drafted tokens themselves (written before the call) the last n. A token sees all keys before those, and of them the ones whose
 * bit is set in tree[row] (device, q_tokens 64-bit words: bit j is the sequence's j-th drafted token; its own bit counts like any other), or, with tree NULL, those up to itself: single tokens, and chains. A token that sees no key
 * gets zeros. Keys beyond max_k_len, the table, or in a page that there is not, are not seen. Rows of out in no sequence are left as they are. scale 0: 1 / sqrt(head_dim).
 * Scores and sums are fp32, the weights times the values' scales fp16. Rows of q and out start on 16 bytes; out overlaps q in nothing. The first call on a device looks up
 * the device's error word (et_attention_check): make it before a stream capture. */
typedef struct et_attention_tree_args {
    void* out; const void* q; const void* codes; const float* scales; const int* table; const int* k_lens; const int* cu_seqlens; const int64_t* tree; void* stream;
    int out_pitch, q_pitch, nhead, nhead_kv, head_dim, batch, q_tokens, max_q_len, max_k_len, pages, page, table_width;
    float scale;
} et_attention_tree_args;
int et_attention_tree(const et_attention_tree_args* args);

/* ---- pruned-format generators (host) ----------------------------------------------------------
 * Seeded and reproducible. bernoulli == 0 keeps exactly floor(total*(1-sparsity)) tiles (a block-row's
 * tiles in draw order); otherwise each tile is kept with probability 1-sparsity (ascending offsets).
 * Replaces gen_sparse_tile_mat (test/tile_mat.cu:5-34) and gen_sparse_row_mat (test/row_mat.cu:5-14). */
int et_gen_sparse_tile_mat(int nrow, int ncol, float sparsity, uint64_t seed, int bernoulli, int* row_ptr,
                           int* row_offset, int cap, int* ntile);
int et_gen_sparse_row_mat(int nrow, float sparsity, uint64_t seed, int nhead, int* row_id, int cap, int* nkeep);
int et_build_head_ptr(const int* row_id, int n, int nhead, int out_feat, int* head_ptr);

/* ---- real-weight ingestion (host; extension) ------------------------------------------------------
 * The reference only draws random structure (test/tile_mat.cu, test/row_mat.cu) and defines no on-disk format.
 * These turn a dense fp16 weight [out_feat x in_feat] (row-major) into exactly the arrays Linear_tile
 * (encoder/Linear.h:18-24) and Linear_row (encoder/Linear.h:66-67) take, by magnitude; ties keep the lower
 * index, so the result is a pure function of the weight.
 * et_prune_dense_to_tiles: keeps the floor(total*(1-sparsity)) 16x16 tiles of largest sum of squares; tiles of a
 *   block-row in ascending column order; data[i*256 + n*16 + k] = W[16r+n, row_offset[i]+k].
 * et_select_rows_magnitude: per head keeps the round(head_dim*(1-sparsity)) (at least 1) rows of largest sum of
 *   squares, summed over the n_mats matrices given (pass Q and K together so that they retain the same
 *   dimensions); row_id ascending.
 * et_compact_rows: weight_compact [ceil16(nkeep) x in_feat] (zero rows as padding), bias_compact [ceil16(nkeep)]. */
int et_prune_dense_to_tiles(const void* dense_host, int out_feat, int in_feat, float sparsity, int* row_ptr,
                            int* row_offset, void* data, int cap_tiles, int* ntile);
int et_select_rows_magnitude(const void* const* dense_hosts, int n_mats, int out_feat, int in_feat, int nhead,
                             float sparsity, int* row_id, int cap, int* nkeep);
int et_compact_rows(const void* dense_host, const void* bias_host, int out_feat, int in_feat, const int* row_id,
                    int nkeep, void* weight_compact, void* bias_compact);

/* ---- encoder layers ----------------------------------------------------------------------------
 * One post-LN encoder layer: Q,K,V linears -> attention -> output linear -> add+LayerNorm -> MLP1 (GELU)
 * -> MLP2 -> add+LayerNorm (encoder/encoder.cu:20-45). LayerNorm vectors (d_model) and mask
 * (seq_len x seq_len additive, may be NULL) are HOST pointers and are copied; `buffer` is a DEVICE
 * scratch of et_encoder_buffer_size bytes owned by the caller (may be NULL if only run_batch is used).
 * The encoder takes ownership of the linears passed in (their handles stay valid only for destroy),
 * as the reference's constructors take them by rvalue. kind: 0 = Encoder_tile, 2 = Encoder_length
 * (encoder/encoder.h:56-77, :102-134). */
typedef struct et_encoder et_encoder;
int et_encoder_tile_create(et_encoder** out, int kind, int d_model, int seq_len, int nheads, void* buffer,
                           et_tile_weight* q, et_tile_weight* k, et_tile_weight* v, et_tile_weight* o,
                           et_tile_weight* mlp1, et_tile_weight* mlp2, const void* ln_gamma_1,
                           const void* ln_beta_1, const void* ln_gamma_2, const void* ln_beta_2,
                           const void* mask_host);
/* Encoder_prune (encoder/encoder.h:79-100): V is row-pruned. */
int et_encoder_prune_create(et_encoder** out, int d_model, int seq_len, int nheads, void* buffer,
                            et_tile_weight* q, et_tile_weight* k, et_row_weight* v, et_tile_weight* o,
                            et_tile_weight* mlp1, et_tile_weight* mlp2, const void* ln_gamma_1,
                            const void* ln_beta_1, const void* ln_gamma_2, const void* ln_beta_2,
                            const void* mask_host);
/* Extension: Q, K and V all row-pruned; Q and K must keep the same rows per head. */
int et_encoder_prune_qkv_create(et_encoder** out, int d_model, int seq_len, int nheads, void* buffer,
                                et_row_weight* q, et_row_weight* k, et_row_weight* v, et_tile_weight* o,
                                et_tile_weight* mlp1, et_tile_weight* mlp2, const void* ln_gamma_1,
                                const void* ln_beta_1, const void* ln_gamma_2, const void* ln_beta_2,
                                const void* mask_host);
int et_encoder_destroy(et_encoder* enc);
/* Encoder_base::buffer_size / Encoder_length::buffer_size (encoder/encoder.h:51-53, :129-133), in bytes. */
size_t et_encoder_buffer_size(int kind, int d_model, int seq_len, int nheads);
size_t et_encoder_batch_buffer_size(int kind, int d_model, int total_tokens, int batch, int max_len, int nheads);
/* Encoder_*::run(out, in) (encoder/encoder.h:76): one sequence of seq_len tokens; out may alias in. */
int et_encoder_run(et_encoder* enc, void* out, const void* in, void* stream);
/* Extension: a batch of packed sequences, seq_lens_host[batch] tokens each (any length >= 0, at most
 * seq_len when the encoder has a mask); valid_lens_host (may be NULL) marks keys at or beyond it as padding.
 * scratch: device buffer of et_encoder_batch_buffer_size bytes. */
int et_encoder_run_batch(et_encoder* enc, void* out, const void* in, const int* seq_lens_host,
                         const int* valid_lens_host, int batch, void* scratch, size_t scratch_bytes, void* stream);
/* Reads and clears the error words of every kernel the layer launches (its tile GEMMs and the device's
 * attention word, see et_attention_check); synchronises. ET_ERR_DEVICE_TIMEOUT with the first code found in
 * *code when a bounded device-side wait gave up since the last check: the output of that run is then
 * incomplete. The status a caller reads where the reference would have exited (encoder/utils.h:4-12). */
int et_encoder_check(et_encoder* enc, int* code);
/* et_encoder_run and et_encoder_run_batch replay a CUDA graph of the layer's launches from the third call on with the
 * same buffers and lengths (no counterpart in the reference, whose run() blocks the host three times per layer).
 * on = 0 turns that off (plain launches every call). It is skipped by itself while the caller's stream is
 * being captured (a ragged batch captured there keeps its own lengths, whatever is run between the graph's launches). */
int et_encoder_set_graph_replay(et_encoder* enc, int on);
/* Length encoder only: route attention through scores materialised in HBM (the reference's structure,
 * encoder/encoder.cu:126-136) instead of the default on-the-fly kernel. Equal-length batches only. */
int et_encoder_set_materialize_scores(et_encoder* enc, int on);

/* ---- Stack of encoder layers (extension: no counterpart in the reference, whose objects hold one layer and
 * whose callers run it once, test/tile_test.cu:36-41). The model takes ownership of the layers (the caller still
 * calls et_encoder_destroy on the emptied handles), owns its scratch (et_model_reserve, or grown on demand by
 * et_model_run_batch outside stream capture), and from the third call with the same buffers and lengths replays
 * all launches of all layers as one CUDA graph. `out` may alias `in`. Layers may be of different kinds; they
 * must agree in d_model. */
typedef struct et_model et_model;
int et_model_create(et_model** out, et_encoder* const* layers, int n_layers);
int et_model_destroy(et_model* model);
int et_model_num_layers(const et_model* model);
int et_model_reserve(et_model* model, int total_tokens, int batch, int max_len);
int et_model_run_batch(et_model* model, void* out, const void* in, const int* seq_lens_host,
                       const int* valid_lens_host, int batch, void* stream);
int et_model_set_graph_replay(et_model* model, int on);
/* Optional form of a stack of tile / length layers: the residual-add + LayerNorm steps (encoder/encoder.cu:36-44)
 * folded into the neighbouring linears, 5 launches per layer instead of 7 (the output projection and FFN2 add the
 * residual and leave per-row sums, the next linear normalises in its epilogue with gamma folded into its weights,
 * one plain LayerNorm ends the stack). OFF by default: on B200 the longer epilogues cost more than the two
 * bandwidth-bound LayerNorm passes they replace (measured: 86 ms against 75 ms per step of the 24-layer BERT-large
 * workload). Results differ from the default form by fp16 rounding of different intermediates, within the library's
 * tolerance. on = 1 builds the folded weights (host work, synchronises); stacks with a row-pruned layer stay
 * unfused; et_model_layernorm_fused tells which form is active. */
int et_model_set_layernorm_fusion(et_model* model, int on);
int et_model_layernorm_fused(const et_model* model);
/* et_encoder_check over every layer of the stack (encoder/utils.h:4-12 is the reference's error path). */
int et_model_check(et_model* model, int* code);

#ifdef __cplusplus
}
#endif
#endif /* ET_B200_H */

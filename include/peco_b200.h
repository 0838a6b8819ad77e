/*
 * C ABI of libpeco_b200.so -- the B200-native (sm_100a) PECO attention hot path.
 *
 * Plain pointers and sizes only.  Every function enqueues work on the CUDA
 * stream passed as the last argument (a cudaStream_t as void*), never
 * synchronises, and returns 0 on success, a cudaError_t value for CUDA
 * failures, or one of the PECO_ERR_* codes below.  Buffers are allocated by
 * the caller (the reference's convention, peco/clustering_cuda.py:83-90 and
 * peco/attention_cuda.py:128); the exceptions are three drop-in symbols whose
 * reference signatures pass no room for what the sm_100a kernels need:
 * peco_assign_tokens_to_centers (bf16 split of fp32 tokens and centres),
 * peco_recompute_cluster_centers (sort scratch) and peco_sparse_attention
 * (attention plan and key blocks) take it from the stream-ordered allocator
 * (cudaMallocAsync / cudaFreeAsync on the caller's stream), as do the two
 * selection entry points for their [BH,CQ,CK] fp32 logits.
 *
 * Device-side faults are never raised with traps: kernels skip out-of-range
 * indices and give up bounded waits, OR-ing a bit into a per-device status
 * word that peco_device_status() returns.
 *
 * Citations are to the reference project Tom-HKUST/PECO.
 */
#ifndef PECO_B200_H_
#define PECO_B200_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define PECO_ERR_UNSUPPORTED 20001  /* shape or dtype outside the kernels' support */
#define PECO_ERR_TENSOR_MAP 20002   /* TMA descriptor could not be encoded */
#define PECO_ERR_DRIVER 20003       /* driver entry point unavailable */
#define PECO_ERR_TIMEOUT 20004      /* a device-side bounded wait expired */
#define PECO_ERR_WORKSPACE 20005    /* workspace too small */
#define PECO_ERR_CAPACITY 20006     /* problem larger than a no-alloc entry point's fixed scratch */

#define PECO_STATUS_TIMEOUT 1u      /* status word bit: a bounded wait expired */
#define PECO_STATUS_BAD_INDEX 2u    /* status word bit: an index failed its bounds check */

/* ---- drop-in symbols (same signatures and status conventions) ---------- */

/* Nearest-centre labels for fp32 x [B,N,D] and centres [B,C,D]; writes
 * labels [B,N] and center_norms [B,C] = ||c||^2.  ``scratch`` ([chunk,C] in
 * the reference) is accepted and left untouched.  D in {64,128}.
 * Replaces peco/kernels/kmeans.cu:139-175 (bound at peco/clustering_cuda.py:65,93-108). */
int peco_assign_tokens_to_centers(const float* x, const float* centers, int32_t* labels, float* scratch,
                                  float* center_norms, int batch, int tokens, int dims, int clusters,
                                  int chunk_size, void* stream);

/* means[b,c] = mean of the tokens labelled c (empty -> previous), counts,
 * and sums.  Deterministic (no atomics).
 * Replaces peco/kernels/kmeans.cu:179-196 (bound at peco/clustering_cuda.py:66,111-125). */
int peco_recompute_cluster_centers(const float* x, const int32_t* labels, const float* previous, float* sums,
                                   int32_t* counts, float* means, int batch, int tokens, int dims, int clusters,
                                   void* stream);

/* Row permutation of [B*H,N,D] items of 2 or 4 bytes: forward
 * out[j] = in[idx[j]], inverse out[idx[j]] = in[j]; bit-exact copies.
 * Replaces peco/kernels/kmeans.cu:200-217 (bound at peco/clustering_cuda.py:67,128-146). */
int peco_reorder_token_features(const void* input, const int32_t* indices, void* output, int batch_heads,
                                int tokens, int dims, int item_size, int inverse, void* stream);

/* peco_recompute_cluster_centers without any allocation (no counterpart in
 * the reference): identical results, with the sort scratch -- batch*tokens +
 * batch*(clusters+1) ints -- in a fixed per-device array of
 * peco_recompute_cluster_centers_static_capacity() ints (2^21, 8 MiB); larger
 * problems return PECO_ERR_CAPACITY without launching.  For callers that must
 * not allocate once running: a serving loop that pre-plans all its memory
 * (an allocation can fail or stall under fragmentation there), or a process
 * whose stream-ordered pool is unavailable or capped.  The first call on a
 * device looks up the array's address (cudaGetSymbolAddress) and should come
 * before any stream capture; the address is kept for the process's lifetime,
 * so do not call it on a device after cudaDeviceReset there (the array, and
 * the address, are gone with the context).  Nothing in the scratch must
 * start at zero.
 * Calls that overlap on one device share the scratch and race; serialise
 * them. */
int peco_recompute_cluster_centers_static(const float* x, const int32_t* labels, const float* previous,
                                          float* sums, int32_t* counts, float* means, int batch, int tokens,
                                          int dims, int clusters, void* stream);
long long peco_recompute_cluster_centers_static_capacity(void);

/* Error text for the clustering entry points (peco/kernels/kmeans.cu:220-223). */
const char* peco_cluster_error_message(int code);

/* Cluster-masked softmax(QK^T/sqrt(D))V over group-packed Q [BH,SQ,D] and
 * K/V [BH,SK,D]; map [BH,CQ,CK] bytes, sizes int32 [BH,CQ]/[BH,CK]; rows with
 * no allowed key -> 0.  dtype 0 = fp16, 1 = bf16; D in {64,128}.  Workspace:
 * int32 BH*(CK+2+3*(ceil(SQ/16)+CQ)) (the reference's size), accepted for
 * ABI compatibility: the plan and key blocks (peco_attention_plan,
 * peco_pack_key_blocks) live in stream-ordered scratch of the call.
 * Replaces peco/kernels/sparse_attention.cu:210-230 (bound at peco/attention_cuda.py:57,130-137). */
int peco_sparse_attention(const void* q, const void* k, const void* v, const uint8_t* selected,
                          const int* q_sizes, const int* k_sizes, void* output, int* workspace, int bh, int sq,
                          int sk, int d, int cq, int ck, int dtype, void* stream);

/* Error text for the attention entry point (peco/kernels/sparse_attention.cu:232-234). */
const char* peco_attention_error_string(int code);

/* ---- fused entry points (used by the processor's fast path) ------------ */

/* Stable argsort of labels [rows,N] (values in [0,C)) by counting sort:
 * indices [rows,N] (original token at each packed position), counts
 * [rows,C] and offsets [rows,C+1] (either may be NULL).
 * Replaces torch.argsort(stable=True) at peco/clustering.py:105. */
int peco_sort_labels(const int32_t* labels, int32_t* indices, int32_t* counts, int32_t* offsets, int rows,
                     int tokens, int clusters, void* stream);

/* Fixed-iteration Lloyd k-means of bf16 token rows for up to two problems
 * (Q and K of one call) in the same launches.  Head b of problem x starts at
 * row b*head_rows (so the video prefix of a [BH,S,D] tensor needs no copy).
 * Per problem: init [BH,C,D] fp32 (read), centers (final means of the last
 * partition, may alias init), work (BH * peco_kmeans_work_floats(C, D, N)
 * floats: ping-pong centres, the centres' bf16 tensor-core image, the
 * token norms the first iteration records for the rest and, for long
 * sequences, the label sort's per-segment scratch), norms [BH,C],
 * labels [BH,N], counts [BH,C], offsets [BH,C+1], perm [BH,N] (stable
 * argsort of the final labels).  Pass k_x = NULL for a single problem.
 * Replaces fit_token_clusters' CUDA loop, peco/clustering.py:59-88 with tol=0. */
int peco_kmeans_fit(const void* q_x, long long q_head_rows, int q_tokens, int q_clusters, int32_t* q_labels,
                    const float* q_init, float* q_centers, float* q_work, float* q_norms, int32_t* q_counts,
                    int32_t* q_offsets, int32_t* q_perm, const void* k_x, long long k_head_rows, int k_tokens,
                    int k_clusters, int32_t* k_labels, const float* k_init, float* k_centers, float* k_work,
                    float* k_norms, int32_t* k_counts, int32_t* k_offsets, int32_t* k_perm, int bh, int dims,
                    int iters, void* stream);

/* Floats of ``work`` per head for peco_kmeans_fit (-1 for unsupported sizes). */
long long peco_kmeans_work_floats(int clusters, int dims, int tokens);

/* Boolean map [BH,CQ,CK] of kept (query cluster, key cluster) pairs: stable
 * descending sort of softmax(Cq.Ck^T/sqrt(D) + log count_k), keep while the
 * mass before < top_p (all if top_p == 1), the first, and the first
 * ``minimum``; AND nonempty.  ``logits``: fp32 [BH,CQ,CK] scratch of the
 * caller, or null for stream-ordered scratch of the call.  Replaces
 * peco/clustering.py:139-186. */
int peco_select_cluster_connections(const float* q_centroids, const float* k_centroids, const int32_t* q_sizes,
                                    const int32_t* k_sizes, uint8_t* map, int bh, int cq, int ck, int dims,
                                    float top_p, int minimum, float* logits, void* stream);

/* Same selection written straight into the text-extended map
 * [BH,CQ+2,CK+2] with extended sizes [BH,CQ+2]/[BH,CK+2].
 * Replaces peco/clustering.py:154-186 followed by peco/processor.py:68-84. */
int peco_select_text_partition(const float* q_centroids, const float* k_centroids, const int32_t* q_sizes,
                               const int32_t* k_sizes, uint8_t* map_ext, int32_t* q_sizes_ext,
                               int32_t* k_sizes_ext, int bh, int cq, int ck, int dims, float top_p, int minimum,
                               int valid_text, int text_length, float* logits, void* stream);

/* Base-Offset PE over [BH,N,D] (dtype 0 fp16, 1 bf16, 2 fp32; D in {64,128};
 * bits 4 or 8).  mode 0: out = fake-quantized x; mode 1: codes uint8
 * [BH,N,D], offset_min / scale fp32 [BH,N]; mode 2: out = decode(codes).
 * Bit-exact with peco/quantization.py:96-150. */
int peco_base_offset(int mode, const void* x, const int32_t* labels, const float* centroids, void* out,
                     uint8_t* codes, float* offset_min, float* scale, int bh, int tokens, int dims, int clusters,
                     int bits, int dtype, void* stream);

/* Attention plan (workspace: int32 bh * peco_attention_workspace_stride),
 * from the group map [BH,GQ,GK] and sizes [BH,GQ]/[BH,GK] (extents clamped
 * like peco/kernels/sparse_attention.cu:25-31): the work units (<= 128 query
 * rows of one query group), the key-row -> key-block map and, per unit, the
 * selected key clusters.  Key blocks hold K or V as 8-row blocks of 8*D
 * 16-bit elements in the tensor core's shared-memory image (D/64 panels of
 * 8 rows x 128 bytes, 16-byte chunk c of row i at chunk c^i); each key
 * cluster starts a new block.  When k_blocks/v_blocks ([BH,
 * peco_key_block_rows(sk, gk), D]) are given, the padding rows of every
 * cluster's last block are zeroed.  Splits the planning half of
 * peco/kernels/sparse_attention.cu:17-52 out of the attention launch. */
int peco_attention_plan(const uint8_t* map, const int* q_sizes, const int* k_sizes, void* k_blocks,
                        void* v_blocks, int* workspace, int bh, int sq, int sk, int d, int gq, int gk,
                        void* stream);

long long peco_attention_workspace_stride(int sq, int sk, int gq, int gk);
long long peco_key_block_rows(int sk, int gk);

/* Row-major K/V [BH,SK,D] -> key blocks through a plan.  Used by the drop-in
 * peco_sparse_attention (which plans and packs internally). */
int peco_pack_key_blocks(const void* k, const void* v, void* k_blocks, void* v_blocks, const int* workspace,
                         int bh, int sq, int sk, int d, int gq, int gk, void* stream);

/* One pass over bf16 Q/K/V [BH,S,D] (video tokens first): packed row j of
 * each head takes source video row indices[j] -- Base-Offset fake quantized
 * for Q and K when bits > 0, copied for V (which uses K's indices) -- and
 * text rows j >= video are copied in place.  With ``plan`` (a workspace
 * written by peco_attention_plan with sq = sk = seq), K and V rows go to
 * key blocks (k_packed/v_packed [BH, peco_key_block_rows(seq, gk), D])
 * instead of row-major [BH,S,D].  Replaces peco/processor.py:141-149 (fake
 * quant, three gathers and the concats). */
int peco_quantize_gather(const void* q, const void* k, const void* v, void* q_packed, void* k_packed,
                         void* v_packed, const int32_t* q_indices, const int32_t* k_indices,
                         const int32_t* q_labels, const int32_t* k_labels, const float* q_centroids,
                         const float* k_centroids, int q_clusters, int k_clusters, int bh, int seq, int video,
                         int dims, int bits, const int* plan, int gq, int gk, void* stream);

/* Sparse attention of packed bf16 Q [BH,SQ,D] over key blocks, following a
 * plan from peco_attention_plan; output rows are scattered through the
 * inverse permutation: packed row j < video goes to row q_indices[j] of
 * ``output`` (q_indices null: no scatter), text rows stay in place.
 * Fuses peco/kernels/sparse_attention.cu with peco/clustering.py:127-136. */
int peco_sparse_attention_restore(const void* q, const void* k_blocks, const void* v_blocks,
                                  const int* workspace, void* output, int bh, int sq, int sk, int d, int gq,
                                  int gk, const int32_t* q_indices, int video, void* stream);

/* Input stage of the attention processor: from the bf16 projection outputs
 * of the video rows (vq/vk/vv) and the text rows (tq/tk/tv), each a
 * row-major [rows, H*D] view with ``*_stride`` elements between rows, write
 * bf16 Q/K/V [H, video_rows + text_rows, D] (video rows first).  Per (row,
 * head): Q and K are RMS-normalised with the stream's gains (w*_v / w*_t,
 * fp32 [D]; null: no norm), rounded to bf16, and video rows are rotated with
 * the (cos, sin) tables [video_rows, D] fp32, pairs interleaved (null: no
 * rotation); V is copied.  Replaces the head split, norm_q/norm_k,
 * apply_rotary_emb, concatenations and contiguous copies of
 * peco/processor.py:163-188. */
int peco_prepare_qkv(const void* vq, const void* vk, const void* vv, long long v_stride, int video_rows,
                     const void* tq, const void* tk, const void* tv, long long t_stride, int text_rows,
                     const float* wq_v, const float* wk_v, float eps_v, const float* wq_t, const float* wk_t,
                     float eps_t, const float* cos, const float* sin, void* q, void* k, void* v, int heads,
                     int dims, void* stream);

/* Sequence <-> head reshard of sequence-sharded attention over NVLink peer
 * memory (no counterpart in the reference, which runs on one GPU; it replaces
 * the NCCL all-to-all of the long-video configuration).  ``buffers`` and
 * ``flags`` are device arrays of every rank's receive buffer and flag array
 * (int64 [slots][world]) as mapped in this process (torch symmetric memory).
 * peco_exchange_put copies ``pieces`` contiguous blocks of ``piece_bytes``
 * (16-byte multiple) from src + src_offsets[i] to rank dst_ranks[i]'s buffer
 * + dst_offsets[i] with plain stores, then sets this rank's entry of slot
 * ``flag_slot`` in every rank's flag array to ``epoch``; ``done_counter`` is a
 * zeroed device unsigned the launch uses and resets.  peco_exchange_wait
 * makes ``stream`` wait until every rank's entry of the slot in this rank's
 * flag array has reached ``epoch`` (bounded: on expiry the device status word
 * records a timeout). */
int peco_exchange_put(const void* src, const long long* src_offsets, const int* dst_ranks,
                      const long long* dst_offsets, long long piece_bytes, int pieces,
                      const unsigned long long* buffers, const unsigned long long* flags, int flag_slot,
                      int rank, int world, long long epoch, unsigned* done_counter, void* stream);
int peco_exchange_wait(const long long* flags, int world, int flag_slot, long long epoch, void* stream);

/* ---- transformer-block operators (no counterpart in the reference, whose
 * blocks are the host framework's) ------------------------------------------
 * Workspaces start on 16 bytes. */

/* out = residual + gate * act([x | x2] W^T + bias) over samples *
 * rows_per_sample rows.  x [rows, k], x2 [rows, k2] (k2 = 0: absent), weight
 * [n, k + k2], residual and out [rows, n]: rows ``*_stride`` elements apart,
 * columns adjacent.  bias [n]; gate [samples, n] rows gate_stride apart (0:
 * one for all); either and residual may be null.  preact, if given, [rows, n]
 * contiguous, receives the pre-activation.  activation 0 none, 1 gelu (tanh
 * form), 2 gelu (erf), 3 silu; dtype 0 fp16, 1 bf16.  Sums are fp32, each
 * output is rounded once.  out may be residual (the same rows) and shares no
 * memory with the operands otherwise.  Operands whose base or row stride is
 * not a multiple of 16 bytes are copied into ``workspace`` first:
 * peco_linear_forward_workspace says how many bytes (0 when all are aligned;
 * -1: sizes out of range). */
int peco_linear_forward(const void* x, long long x_stride, const void* x2, long long x2_stride, const void* weight,
                        long long w_stride, const void* bias, const void* gate, long long gate_stride,
                        const void* residual, long long res_stride, void* out, long long out_stride, void* preact,
                        int samples, int rows_per_sample, int k, int k2, int n, int activation, int dtype,
                        void* workspace, long long workspace_bytes, void* stream);
long long peco_linear_forward_workspace(const void* x, long long x_stride, const void* x2, long long x2_stride,
                                        const void* weight, long long w_stride, int samples, int rows_per_sample,
                                        int k, int k2, int n);

/* Gradients of peco_linear_forward for ``grad`` = d out (the residual's
 * gradient is ``grad`` itself).  preact [rows, n] is needed when the
 * activation is not 0 or dgate is asked for.  dx [rows, k], dx2 [rows, k2],
 * dweight [n, k + k2], dbias [n], dgate [samples, n], contiguous; null: not
 * computed.  grad * gate * act' is rounded to the operands' type for the two
 * products (fp16: to its range too, infinite past 65504, zero below 6e-8); the
 * sums for dbias and dgate are of the unrounded values and do
 * not depend on the launch order.  Needs at least one row. */
int peco_linear_backward(const void* grad, long long grad_stride, const void* preact, const void* x,
                         long long x_stride, const void* x2, long long x2_stride, const void* weight,
                         long long w_stride, const void* gate, long long gate_stride, void* dx, void* dx2,
                         void* dweight, void* dbias, void* dgate, int samples, int rows_per_sample, int k, int k2,
                         int n, int activation, int dtype, void* workspace, long long workspace_bytes, void* stream);
long long peco_linear_backward_workspace(const void* grad, long long grad_stride, const void* x, long long x_stride,
                                         const void* x2, long long x2_stride, const void* weight, long long w_stride,
                                         int samples, int rows_per_sample, int k, int k2, int n, int activation,
                                         int has_gate);

/* Rows of 16-bit elements in 8-bit integers, one scale a row: scales[m] = max / 127
 * with max the largest magnitude in [x | x2] of row m, values[m, k] = 127 x[m, k]
 * / max rounded to the nearest integer (ties to even, as of the exact quotient).
 * A row of zeros has scale 0, one with an infinity or NaN scale NaN and values 0.
 * x [rows, k], x2 [rows, k2] (k2 = 0: absent), values [rows, k + k2]: rows
 * ``*_stride`` elements apart; dtype 0 fp16, 1 bf16. */
int peco_quantize_rows(const void* x, long long x_stride, const void* x2, long long x2_stride, void* values,
                       long long v_stride, float* scales, long long rows, int k, int k2, int dtype, void* stream);

/* out = residual + gate * act(row_scales[m] col_scales[n] (X W^T)[m, n] + bias)
 * with 8-bit signed X and W [n, k + k2] and exact integer sums (k + k2 <=
 * 131071).  X is ``values`` [rows, k] with row_scales [rows] (k2 = 0), or, with
 * values null, [x | x2] quantised as by peco_quantize_rows into the workspace.
 * bias, gate, residual, out, activation and dtype as in peco_linear_forward; out
 * shares no memory with the operands.  8-bit rows whose base or stride is not
 * a multiple of 16 bytes are copied into the workspace first;
 * peco_linear_int8_workspace says how many bytes it needs (-1: sizes out of range). */
int peco_linear_int8(const void* x, long long x_stride, const void* x2, long long x2_stride, const void* values,
                     long long v_stride, const float* row_scales, const void* weight, long long w_stride,
                     const float* col_scales, const void* bias, const void* gate, long long gate_stride,
                     const void* residual, long long res_stride, void* out, long long out_stride, int samples,
                     int rows_per_sample, int k, int k2, int n, int activation, int dtype, void* workspace,
                     long long workspace_bytes, void* stream);
long long peco_linear_int8_workspace(int from_16_bits, const void* values, long long v_stride, const void* weight,
                                     long long w_stride, int samples, int rows_per_sample, int k, int k2, int n);

/* Spans of keys for attention: rows [batch, queries, 4] gets (first key, key
 * behind the last, position among the keys, n) of every query row, tiles [batch,
 * ceil(queries / 128), 4] bounds over 128 rows; both start on 16 bytes.  n of the
 * first rows: the tiles of 128 rows, those that see most keys first.
 * Documents (documents > 0): document i of sample b holds rows [q_ends[b *
 * q_stride + i], q_ends[... + i + 1]) and keys likewise by k_ends; rows outside
 * see nothing.  Otherwise lengths [batch] (null: all keys).  A document's last
 * row stands at its last key.  causal: a row sees the keys up to its position and
 * its document's first prefix[b * prefix_batch + i * prefix_document] keys
 * (prefix null: prefix_all).  window > 0: keys less than ``window`` away.
 * Offsets are device memory and are held to the sequence. */
int peco_key_spans(const int* q_ends, long long q_stride, const int* k_ends, long long k_stride, int documents,
                   const int* lengths, const int* prefix, long long prefix_batch, int prefix_document, int prefix_all,
                   int causal, int window, int batch, int queries, int keys, int* rows, int* tiles, void* stream);

/* Attention of q [batch, heads, sq, d] over k, v [batch, kv_heads, sk, d]:
 * z_ij = cap tanh(scale q_i.k_j / cap) - slopes[h] |pos_i - j| (cap 0 and slopes
 * null: without), out_i = sum_j softmax(z)_ij v_j over the row's span, lse [batch,
 * heads, sq] its logarithmic sum (a row without keys: 0 and -inf).  strides (host
 * memory): batch, head and row strides of q, k, v and out in elements; d is
 * adjacent, rows, heads and samples start on 16 bytes.  span_rows and span_tiles
 * from peco_key_spans, on 16 bytes (null: every key, pos = i + sk - sq), of one sample for
 * all or, with spans_batched, of each.  heads is a multiple of kv_heads, d of 8 up
 * to 128; scale and cap from 1e-30 to 1e30, scale / cap at most 1e30; dtype 0 fp16,
 * 1 bf16.  Calls of few rows keep parts in the workspace. */
int peco_span_attention(const void* q, const void* k, const void* v, const long long* strides, const int* span_rows,
                        const int* span_tiles, int spans_batched, const float* slopes, float scale, float cap, void* out,
                        float* lse, int batch, int heads, int kv_heads, int sq, int sk, int d, int dtype, void* workspace,
                        long long workspace_bytes, void* stream);
long long peco_span_attention_workspace(int batch, int heads, int kv_heads, int sq, int sk, int d);

/* Gradients of peco_span_attention for ``grad`` = d out, with its result ``out``
 * and ``lse`` (null outputs: not computed); ``spans`` of the workspace: whether
 * there are any.  strides (host memory): batch, head
 * and row strides of grad, q, k, v, out, dq, dk and dv.  Sums run in a fixed
 * order; the probabilities and their gradients are rounded to the operands'
 * type for the products.  A row of one key has no gradient of its score; keys
 * that no row sees, and rows that see none, get zeros whatever they hold. */
int peco_span_attention_backward(const void* grad, const void* q, const void* k, const void* v, const void* out,
                                 const float* lse, const long long* strides, const int* span_rows, const int* span_tiles,
                                 int spans_batched, const float* slopes, float scale, float cap, void* dq, void* dk,
                                 void* dv, int batch, int heads, int kv_heads, int sq, int sk, int d, int dtype,
                                 void* workspace, long long workspace_bytes, void* stream);
long long peco_span_attention_backward_workspace(int batch, int heads, int kv_heads, int sq, int sk, int d,
                                                 int spans);

/* Gated residual and norm: with b = post_norm(branch) * post_weight,
 *   residual = residual_scale * x + gate * b
 *   normed = norm(residual) * weight * (1 + scale) + shift
 * for x and branch [samples, rows, width] (strides in elements, columns
 * adjacent) and the sample's vectors gate / scale / shift [samples, width]
 * (``*_batch`` elements apart, 0: shared).  norm 1 layer (mean and variance),
 * 2 rms; post_norm 0 none, 1, 2.  Everything but x and normed may be null;
 * gate, post_norm and residual need a branch.  residual and normed are
 * contiguous and each rounded once.  width <= 16384; dtype 0 fp16, 1 bf16. */
int peco_gated_norm(const void* x, long long x_batch, long long x_row, const void* branch, long long branch_batch,
                    long long branch_row, const void* gate, long long gate_batch, const void* scale,
                    long long scale_batch, const void* shift, long long shift_batch, const void* weight,
                    const void* post_weight, void* residual, void* normed, int samples, int rows, int width, int norm,
                    int post_norm, float eps, float post_eps, float residual_scale, int dtype, void* stream);

/* Gradients of peco_gated_norm for grad_normed and grad_residual (null: 0).
 * dx, dbranch [samples, rows, width] and the vector gradients, any of them
 * null; a vector's gradient is [samples, width], or summed over the samples
 * to [width] when its bit of ``shared`` is set (1 gate, 2 scale, 4 shift).
 * The workspace is needed for vector gradients only; their sums run in a
 * fixed order.  Needs at least one row. */
int peco_gated_norm_backward(const void* grad_normed, long long gh_batch, long long gh_row, const void* grad_residual,
                             long long gr_batch, long long gr_row, const void* x, long long x_batch, long long x_row,
                             const void* branch, long long branch_batch, long long branch_row, const void* gate,
                             long long gate_batch, const void* scale, long long scale_batch, const void* weight,
                             const void* post_weight, void* dx, void* dbranch, void* dgate, void* dscale, void* dshift,
                             int shared, void* dweight, void* dpost_weight, int samples, int rows, int width, int norm,
                             int post_norm, float eps, float post_eps, float residual_scale, int dtype,
                             void* workspace, long long workspace_bytes, void* stream);
long long peco_gated_norm_backward_workspace(int samples, int rows, int width);

/* Rotary embedding by positions on several axes, of q [batch, q_heads, rows,
 * dims] and k (k_heads may be 0) in one launch.  ``*_strides`` (host memory):
 * batch, head and token strides of the source, then of the destination, in
 * elements; dims are adjacent.  A destination may be its source.  axes (host):
 * dimensions of each of the n_axes <= 4 sections; pair j of axis a turns by
 * position[a] * theta^(-2 j / axes[a]).  Rows [0, rotated_rows) turn, later
 * rows and dimensions past the sections are copied.  Positions: grid (host, a
 * row-major token grid whose product is rotated_rows), or ``positions``
 * [batch, rotated_rows, n_axes] on the device (pos_type 0 int32, 1 int64, 2
 * fp32; strides in elements).  interleaved: pairs (2i, 2i+1), else one from
 * each half of the rotated dimensions.  inverse: the opposite turn.  dtype 0
 * fp16, 1 bf16, 2 fp32; dims even, at most 256. */
int peco_rotary(const void* q, void* q_out, int q_heads, const long long* q_strides, const void* k, void* k_out,
                int k_heads, const long long* k_strides, int batch, int rows, int rotated_rows, int dims,
                const int* axes, int n_axes, double theta, const int* grid, const void* positions,
                long long pos_batch_stride, long long pos_row_stride, int pos_type, int interleaved, int inverse,
                int dtype, void* stream);

/* ---- diagnostics --------------------------------------------------------- */

/* How a product of the linear layer, [m, n] results over k_blocks blocks of 64
 * summands, is cut (no device is touched).  product 0 the forward with its
 * activation, 1 the gradient of the rows, 2 of the weight.  plan (host) gets
 * CTAs per tile, columns per accumulator, accumulators per tile, groups that
 * share a tile's sum, stages of the shared-memory ring, tile rows, tile
 * columns and the tile rows walked together. */
int peco_linear_tiles(int m, int n, int k_blocks, int product, int activation, int* plan);

/* Copies the device status word of the current device to *out (synchronising
 * ``stream``) and clears it when ``clear`` != 0. */
int peco_device_status(unsigned* out, int clear, void* stream);

const char* peco_error_string(int code);

int peco_library_version(void);

/* Number of kernels this library has launched in the process so far. */
unsigned long long peco_launch_count(void);

#ifdef __cplusplus
}
#endif

#endif  /* PECO_B200_H_ */

/*
 * pfng_hip — C-ABI of the MI355X (gfx950) quantized GGML GEMM/GEMV path.
 *
 * This is the drop-in boundary. The reference's kernel adapters reach their
 * kernels through the KernelCallbacks table (bench/framework/kernel_registry.h:92-101);
 * a HIP adapter registered under the mi355x-gfx950 platform profile calls the
 * entry points below from its callbacks:
 *   prepare()       -> device allocation + upload, pfng_hip_quantize_* for activations
 *   run()           -> pfng_hip_mul_mat_* (asynchronous), then a stream synchronize
 *   export_output() -> download of C
 *
 * Conventions (all entry points):
 *   - Pointers are DEVICE pointers. Blocks use the byte layouts of
 *     include/pfng_blocks.h (identical to the reference include/ggml.h).
 *   - Row-major: weight row n holds k/QK blocks at weight[n*(k/QK) + b], activation
 *     row m likewise, output C[m*n_cols + n] (llama_reference.cpp:170-175).
 *   - stream is a hipStream_t (NULL = the null stream). Launches are asynchronous.
 *   - Return 0 on success, a pfng_status otherwise; pfng_hip_last_error() returns a
 *     thread-local message for the last failing call. No entry point throws.
 *   - m == 0 or n == 0 is a no-op returning 0; k must be a positive multiple of the
 *     block size (32 for q4_0/q8_0, 256 for the K-quants), else PFNG_ERR_INVALID_ARGUMENT,
 *     mirroring validate_shape (kernels/common/adapter_common.h:28-43).
 */
#ifndef PFNG_HIP_H
#define PFNG_HIP_H

#include <stddef.h>
#include <stdint.h>

#include "pfng_blocks.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef enum {
    PFNG_OK = 0,
    PFNG_ERR_INVALID_ARGUMENT = 1, /* shape, null pointer, bad type or path */
    PFNG_ERR_UNSUPPORTED = 2,      /* a forced path that cannot run this shape */
    PFNG_ERR_HIP = 3,              /* HIP runtime error (message has details) */
    PFNG_ERR_DEVICE = 4            /* current device is not a gfx950 */
} pfng_status;

/* Matrix-product implementations; PFNG_PATH_AUTO picks per shape (the GEMV
 * where it applies: up to m = 16, and its MFMA tiles up to m = 64 below
 * k = 2048 and m = 128 from there, for q4_0 at k % 256 == 0 from 512, q4_K at
 * k % 1024 == 0, iq2_xxs at k % 2048 == 0, except where n is so wide, from m = 17
 * and n > 4096, that the GEMM is predicted faster; then the MFMA GEMM tiles) and
 * returns PFNG_ERR_UNSUPPORTED when neither applies (see pfng_hip_auto_path). */
typedef enum {
    PFNG_PATH_AUTO = 0,
    PFNG_PATH_GEMV = 1,  /* the decode-batch kernels. Shapes taken:
                            q4_0: m == 1 with k % 64 == 0; m = 2..8 with
                            k % 256 == 0, or k % 64 == 0 while
                            m * (k / 64) * 76 + 16 <= 163840; m = 9..16 with
                            k % 64 == 0 under that same LDS bound; m = 9..64
                            (k < 2048) or 9..128 with k % 256 == 0, k >= 512.
                            q4_K and iq2_xxs: m <= 8 with k % 256 == 0;
                            m = 9..16 while m * (k / 256) * 320 + 3072 <= 163840;
                            m = 9..64 (k < 2048) or 9..128 with k % 1024 == 0
                            (q4_K) or k % 2048 == 0 (iq2_xxs).
                            All formats: k <= 2^24 (32-bit load offsets).
                            Kernels: wavefront-per-row GEMVs for short batches;
                            16x16 int8-MFMA tiles with K split over 16 waves
                            (wave w takes the 256-element groups w, w + 16, ...,
                            one per round; below k = 4096 some waves idle), the
                            weights decoded once per wave and round and the
                            activation rows streamed in chunks of 16, from
                            m = 3..6 by format and k (iq2_xxs at k == 4096 from
                            m = 9, m = 5..8 a tile with two-half copies) */
    PFNG_PATH_MFMA = 2,  /* int8-MFMA GEMM, LDS-staged tiles: q4_0 with k % 128 == 0,
                            q4_K and iq2_xxs for every k % 256 == 0; k <= 2^24.
                            Small m of the K-quants (up to 64, from k = 2048 up to
                            128) run on the GEMV's 16-row tiles at the k that
                            PFNG_PATH_GEMV declines for them */
    PFNG_PATH_NAIVE = 3  /* one thread per output, the reference's exact fp32 order */
} pfng_path;

/* Message of the last failing call on this host thread ("" if none). */
const char *pfng_hip_last_error(void);

/* Library version string. */
const char *pfng_hip_version(void);

/* Checks that the current HIP device is a gfx950 (MI355X). Writes the
 * gcnArchName into arch (if non-NULL) and the CU count into cus (if non-NULL).
 * Also resolves, for this device, what the other entry points look up once per
 * device (its CU count, the address of pfng_hip_compute_noalloc's scratch), so
 * that calls made under graph capture afterwards make no such query.
 * Replaces the Device-Tree platform check of bench/framework/platform.cpp:97-133. */
int pfng_hip_device_check(char *arch, size_t arch_len, int *cus);

/* ---- activation quantization ------------------------------------------ */

/* Replaces llama_reference::quantize_row_q8_0 (bench/llama_reference/llama_reference.h:12,
 * llama_reference.cpp:38-52) applied row by row to a rows x k fp32 matrix.
 * y: rows*(k/32) block_q8_0. Bytes are identical to the reference's. */
int pfng_hip_quantize_q8_0(const float *x, void *y, int64_t rows, int64_t k, void *stream);

/* Replaces llama_reference::quantize_row_q8_K (llama_reference.h:14, .cpp:54-70),
 * including the 16 int16 bsums. y: rows*(k/256) block_q8_K. Bytes identical. */
int pfng_hip_quantize_q8_K(const float *x, void *y, int64_t rows, int64_t k, void *stream);

/* ---- matrix products on quantized operands ------------------------------ */

/* C[m x n] = W(q4_0)[n x k] . A(q8_0)[m x k]^T: the loop of dot_q4_0_q8_0 over
 * every (m, n) in compute_q4_0 (llama_reference.cpp:134-146, 172-175). */
int pfng_hip_mul_mat_q4_0_q8_0(const void *weight, const void *act_q8_0, float *out, int64_t m, int64_t n,
                               int64_t k, int path, void *stream);

/* C = sum over super-blocks of dot_q4_K_q8_K (llama_reference.cpp:113-132, 186-189). */
int pfng_hip_mul_mat_q4_K_q8_K(const void *weight, const void *act_q8_K, float *out, int64_t m, int64_t n,
                               int64_t k, int path, void *stream);

/* C = sum over super-blocks of dot_iq2_xxs_q8_K (llama_reference.cpp:148-161, 200-203),
 * with the full 256-entry IQ2_XXS grid. */
int pfng_hip_mul_mat_iq2_xxs_q8_K(const void *weight, const void *act_q8_K, float *out, int64_t m, int64_t n,
                                  int64_t k, int path, void *stream);

/* The path PFNG_PATH_AUTO takes for this shape with 16-byte-aligned weights
 * and activations and a 4-byte-aligned C: PFNG_PATH_GEMV or PFNG_PATH_MFMA;
 * PFNG_PATH_AUTO for an empty product (m == 0 or n == 0); -1 (with a message
 * in pfng_hip_last_error()) when the shape is invalid or no tiled path takes
 * it, in which case PFNG_PATH_AUTO returns PFNG_ERR_UNSUPPORTED and only
 * PFNG_PATH_NAIVE runs it. The counterpart of an adapter's validate()
 * (kernels/common/adapter_common.h:28-43) for the automatic path. Host-only:
 * touches no device. */
int pfng_hip_auto_path(int type, int64_t m, int64_t n, int64_t k);

/* Type-dispatched form; type is a pfng_quantization_type. */
int pfng_hip_mul_mat(int type, const void *weight, const void *act_q, float *out, int64_t m, int64_t n, int64_t k,
                     int path, void *stream);

/* ---- weight quantizers (setup; the reference runs them on the host) ------ */

/* Replaces quantize_row_q4_0 (llama_reference.cpp:13-36) per row: x is
 * rows x k fp32 (row-major, 16-byte aligned), y receives rows * k/32
 * block_q4_0 (2-byte aligned), byte-identical to the reference. */
int pfng_hip_quantize_q4_0(const float *x, void *y, int64_t rows, int64_t k, void *stream);

/* Replaces quantize_row_q4_K (llama_reference.cpp:72-111, with its
 * non-upstream scale packing :97-101) per row; y 16-byte aligned. */
int pfng_hip_quantize_q4_K(const float *x, void *y, int64_t rows, int64_t k, void *stream);

/* ---- end to end: llama_reference::compute on the GPU -------------------- */

/* Bytes of device workspace pfng_hip_compute needs for the quantized activations. */
size_t pfng_hip_compute_workspace_size(int type, int64_t m, int64_t k);

/* Replaces llama_reference::compute (llama_reference.h:18, .cpp:165-215):
 * quantizes the fp32 activations into workspace, then runs the product.
 * workspace must hold pfng_hip_compute_workspace_size() bytes. For q4_0 with
 * m <= 2, k % 64 == 0, m * (k / 32) * 34 <= 65536 and PFNG_PATH_AUTO or
 * PFNG_PATH_GEMV the quantization is fused into the GEMV kernel (same q8_0
 * bytes, kept in LDS) and workspace is not written; from m = 3 on the separate
 * quantize launch is cheaper than quantizing again in every workgroup. */
int pfng_hip_compute(int type, const float *activation, const void *weight, float *out, int64_t m, int64_t n,
                     int64_t k, void *workspace, size_t workspace_bytes, int path, void *stream);

/* No counterpart in the reference. For callers that cannot allocate device
 * memory (code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc): pfng_hip_compute with the same arguments and results, but
 * without a workspace. The quantized activations go to a static 16 MiB device
 * array of the library (one per device, held until the process ends), so
 * m * (k/32) * 34 bytes (q4_0) or m * (k/256) * 292 bytes (q4_K, iq2_xxs) must
 * not exceed 16 MiB (q4_0 at k = 4096: m <= 3855); larger shapes return
 * PFNG_ERR_INVALID_ARGUMENT. The call itself allocates nothing. Every call on a
 * device shares that device's array: calls that overlap on one device (other
 * streams, other host threads) race and must be serialized by the caller. The
 * array's address is looked up on the first call on a device (or by
 * pfng_hip_device_check): make that call outside graph capture; later calls may
 * be captured. */
int pfng_hip_compute_noalloc(int type, const float *activation, const void *weight, float *out, int64_t m, int64_t n,
                             int64_t k, int path, void *stream);

/* ---- serving: a paged 4-bit cache of keys and values ---------------------- */

/* No counterparts in the reference: what a transformer layer does between the k
 * and v products and the o product. A cache holds the keys and values of many
 * requests in pages of page_size tokens (a power of two, 16 to 1024):
 *   [pages][2: keys, values][kv_heads][pfng_hip_kv4_page_bytes()] bytes
 * with 4.5 bits a value: blocks of 32 elements of a head, each (nibble - 8) * d
 * with an fp16 d, as block_q4_0 (pfng_blocks.h) but in places of the cache's own
 * (the library's kv_layout.h). Slot s is token s % page_size of page s / page_size.
 * Request r's token at position p is in page block_table[r * table_stride + p /
 * page_size]. head_dim is 64, 128 or 256.
 *
 * Numbers that live on the device (lengths, tables, slots, positions) cannot be
 * checked by the host. The kernels bound every access: a page or slot outside the
 * cache is skipped, a length past the table is cut, and a result that depends on
 * none of them is not touched.
 *
 * One call is one launch of fewer than 2^32 threads: norms, stores and reads of 2^35
 * elements and more (of q and k together, or of k), and attention of 2^24 requests
 * times key heads, are refused.
 *
 * Element types of keys, values, queries and results; rows of a token's heads are
 * contiguous, tokens `stride` elements apart, both 16-byte aligned. */
typedef enum { PFNG_F32 = 0, PFNG_BF16 = 1, PFNG_F16 = 2 } pfng_element_type;

/* Bytes of one head's keys (or values) of a page; 0 for sizes not supported. */
int64_t pfng_hip_kv4_page_bytes(int page_size, int head_dim);

/* The tables of one step. Request r holds cached[r] tokens and adds added[r]
 * (negative counts are taken as 0, counts past 2^30 - 2048 as that):
 *   starts[r]  = added[0] + .. + added[r - 1]          (requests + 1 numbers)
 *   lengths[r] = cached[r] + added[r]
 *   block_table[r][j] for the pages that request r needs beyond the
 *     ceil(cached / page_size) it has: the next entries of free_pages, in order
 *     of requests; other entries stay
 *   positions[t], slots[t] of the new tokens, request by request; up to `tokens`,
 *     those past the last have position 0 and slot -1
 *   used[0] = pages needed. Where it is more than free_count, or a request needs
 *     more than max_pages, the entries and slots without a page are -1 (a slot
 *     without a table entry likewise).
 * At most 4096 requests. */
int pfng_hip_kv_block_tables(const int32_t *cached, const int32_t *added, int requests, const int32_t *free_pages,
                             int64_t free_count, int page_size, int32_t *block_table, int64_t table_stride,
                             int max_pages, int64_t tokens, int32_t *starts, int32_t *lengths, int32_t *positions,
                             int32_t *slots, int32_t *used, void *stream);

/* Norms of every query and key head and the position rotation, in one pass:
 *   y = x / sqrt(mean(x^2) + eps) * weight   (fp32 weights of head_dim; null: y = x)
 *   the first rot_dim elements (a multiple of 16) turn in pairs (i, i + rot_dim/2),
 *   or (2i, 2i + 1) if adjacent: a' = a cos - b sin, b' = b cos + a sin, with
 *   row positions[t] of cos_sin[table_rows][rot_dim]: rot_dim/2 cosines, then sines.
 * A token whose position has no row becomes NaN. In fp32, rounded once to out_type.
 * Results may overwrite inputs of the same type and stride. q_heads or kv_heads
 * may be 0. */
int pfng_hip_qk_norm_rope(const void *q, int64_t q_stride, const void *k, int64_t k_stride, int in_type, void *q_out,
                          int64_t q_out_stride, void *k_out, int64_t k_out_stride, int out_type, const float *q_weight,
                          const float *k_weight, float eps, const float *cos_sin, int64_t table_rows, int rot_dim,
                          int adjacent, const int32_t *positions, int64_t tokens, int q_heads, int kv_heads,
                          int head_dim, void *stream);

/* Stores keys and values at slots[t], quantized as pfng_hip_quantize_q4_0 does
 * (same nibbles and scales). A block with an infinity or a NaN gets the scale NaN,
 * so that it reads as NaN. A slot outside 0 .. pages * page_size - 1 is skipped.
 * Two tokens must not have the same slot. */
int pfng_hip_kv4_store(const void *k, int64_t k_stride, const void *v, int64_t v_stride, int type,
                       const int32_t *slots, int64_t tokens, void *cache, int64_t pages, int kv_heads, int head_dim,
                       int page_size, void *stream);

/* The values that the cache holds at slots[t]: k and v are [tokens][kv_heads]
 * [head_dim]; rows of slots outside the cache are zeros. */
int pfng_hip_kv4_read(const void *cache, int64_t pages, int kv_heads, int head_dim, int page_size,
                      const int32_t *slots, int64_t tokens, void *k, void *v, int type, void *stream);

/* Bytes of workspace pfng_hip_attention_kv4 needs for these sizes on the current
 * device (0 where the keys are not split); -1 for sizes that it refuses. The need
 * goes by how the keys are split and does not grow with the sizes (a batch may need
 * none where one request of it needs some): ask for the sizes of each call. */
int64_t pfng_hip_attention_kv4_workspace_size(int type, int64_t tokens, int64_t requests, int q_heads, int kv_heads,
                                              int head_dim, int causal, int64_t max_added, int64_t max_length);

/* Attention of the requests' newest tokens over the cache:
 *   out[t][h] = sum_j softmax_j(scale * q[t][h] . k_j) v_j
 * with the keys and values of head h / (q_heads / kv_heads). Tokens starts[r] ..
 * starts[r + 1] - 1 are request r's last ones; starts null: one token each
 * (tokens == requests). lengths[r] counts the request's keys, the new tokens'
 * among them (store them first). The query at position p sees the keys j with
 *   j < lengths[r];  j <= p if causal;  j > p - window if window > 0
 * and a query that sees none gets zeros. causal 0 is cross attention to states of
 * any length. max_added and max_length say how many tokens one request adds and
 * how many keys it has at most: they choose the launch's shape, and larger counts
 * are still computed, only slower, as they are where both say much more than there
 * is. The window does not go into that choice: where it is far shorter than the
 * requests, a max_length of window + max_added (in the workspace's query too) says
 * it. Results of tokens of no request are undefined.
 * A NaN or an infinity in the cache reaches the queries that see it and no others,
 * and so does the size of any value: a row's accuracy goes by what it sees.
 * Maxima, sums and results are in fp32, rounded once. Into the products go
 *   bf16: probabilities rounded to fp16 (11 bits); with many new tokens keys, values
 *     and the queries times the scale too;
 *   fp32 and fp16: exact keys and values, probabilities and fp32 queries to 22 bits.
 * What a key gives to a result is kept to 2^-34 of the largest value that the row
 * sees. */
int pfng_hip_attention_kv4(const void *q, int64_t q_stride, void *out, int64_t out_stride, int type,
                           const int32_t *starts, const int32_t *lengths, int64_t requests, int64_t tokens,
                           int q_heads, const int32_t *block_table, int64_t table_stride, int max_pages,
                           const void *cache, int64_t pages, int kv_heads, int head_dim, int page_size, float scale,
                           int causal, int64_t window, int64_t max_added, int64_t max_length, void *workspace,
                           int64_t workspace_bytes, void *stream);

/* ---- diagnostics ---------------------------------------------------------- */

/* Exact integer parts of every block dot, computed by the same kernel
 * configuration (operand decode, tile, K split) that PFNG_PATH_MFMA runs for
 * this shape on the current device:
 *   q4_0   : out[(m*n + n)*(k/32) + b]     = sum (q_w - 8) * q_a over block b
 *   q4_K   : out[((m*n+n)*(k/256) + b)*2]  = sum_j sc_j*S_j, [..+1] = sum_j min_j*(bsum_2j+bsum_2j+1)
 *   iq2_xxs: out[(m*n + n)*(k/256) + b]    = sum_j (2 s_j + 1) * S_j
 * Where PFNG_PATH_MFMA runs q4_K on whole-K tiles (k = 1024 or 1536), which
 * split super-blocks between K slices and join the parts only in fp32, the
 * sums come from the 64 x 64 two-slice tiles that shape would otherwise take,
 * as they do where it runs a K-quant on 16-row tiles (small m at the k that
 * PFNG_PATH_GEMV does not take there).
 * For verification at small sizes; not a performance path. */
int pfng_hip_block_isums(int type, const void *weight, const void *act_q, int32_t *out, int64_t m, int64_t n,
                         int64_t k, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* PFNG_HIP_H */

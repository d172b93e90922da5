/*
 * pagoda_hip.h — C ABI of the MI355X (gfx950) decode backend for pagoda.
 *
 * Plain pointers and sizes only. Every call returns 0 on success or a
 * negative status; pgd_last_error() gives the message of the last failure
 * on the calling thread. Unless a name ends in _dev, pointers are HOST
 * memory and the call is synchronous. _dev calls take DEVICE pointers, are
 * queued on the device handle's stream and return without waiting.
 *
 * Each entry point cites the reference interface it replaces (paths relative
 * to the quantz8a/pagoda tree).
 */
#ifndef PAGODA_HIP_H
#define PAGODA_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

enum {
  PGD_OK = 0,
  PGD_ERR_ARG = -1,
  PGD_ERR_DEVICE = -2,
  PGD_ERR_HIP = -3,
  PGD_ERR_SHAPE = -4,
  PGD_ERR_STATE = -5,
  PGD_ERR_ALLOC = -6,
  PGD_ERR_FORMAT = -7,
};

enum { PGD_FMT_A8 = 0, PGD_FMT_Q4K = 1, PGD_FMT_Q6K = 2 };

typedef struct pgd_dev pgd_dev;
typedef struct pgd_matrix pgd_matrix;

/* ---- errors / version ---------------------------------------------------- */
/* Copies the last error message (NUL terminated, truncated to len). Returns its full length. */
int pgd_last_error(char* buf, size_t len);
/* ABI version (major*10000 + minor*100 + patch). */
int pgd_version(void);

/* ---- device ---------------------------------------------------------------
 * Replaces CandleModel::device_from_env (pagoda-hf/src/lib.rs:409-426) for
 * PAGODA_DEVICE=hip: spec is "hip" or "hip:N". Any other spec is an error;
 * there is no CPU fallback. */
int pgd_device_open(const char* spec, pgd_dev** out);
int pgd_device_close(pgd_dev* dev);
int pgd_device_sync(pgd_dev* dev);
/* The hipStream_t every _dev call of this handle is queued on. */
void* pgd_device_stream(pgd_dev* dev);
int pgd_device_malloc(pgd_dev* dev, size_t bytes, void** out);
int pgd_device_free(pgd_dev* dev, void* ptr);
/* kind: 0 host->device, 1 device->host, 2 device->device (synchronous) */
int pgd_device_memcpy(pgd_dev* dev, void* dst, const void* src, size_t bytes, int kind);

/* Device-to-device copy queued on the handle's stream, not waited for (no
 * reference counterpart: the on-box streaming rate the roofline report
 * quotes beside the HBM specification). */
int pgd_device_copy_dev(pgd_dev* dev, void* dst, const void* src, size_t bytes);

/* ---- timing: HIP events recorded on the device handle's stream --------- */
typedef struct pgd_event pgd_event;
int pgd_event_new(pgd_dev* dev, pgd_event** out);
int pgd_event_record(pgd_event* ev);
/* Waits for `end`, then writes the elapsed milliseconds between the two. */
int pgd_event_elapsed_ms(pgd_event* start, pgd_event* end, float* ms);
int pgd_event_free(pgd_event* ev);

/* ---- quantized matrices ---------------------------------------------------
 * Replaces QuantMatrix::upload (pagoda-hf/src/qwen3_gemv.rs:658-705):
 * MLX affine 8-bit group 64, packed u32 [n_out, n_in/4] (codes little
 * endian), bf16 scales/biases [n_out, n_in/64]. */
int pgd_matrix_upload_a8(pgd_dev* dev, const uint32_t* packed, const uint16_t* scales_bf16,
                         const uint16_t* biases_bf16, int n_out, int n_in, pgd_matrix** out);
/* GGML block_q4_K / block_q6_K rows of ceil(n_in/256) blocks (144 B / 210 B);
 * replaces the QTensor -> QMatMul load of pagoda-hf/src/qwen2_gguf.rs:283-289. */
int pgd_matrix_upload_q4k(pgd_dev* dev, const void* blocks, int n_out, int n_in, pgd_matrix** out);
int pgd_matrix_upload_q6k(pgd_dev* dev, const void* blocks, int n_out, int n_in, pgd_matrix** out);
/* GGML block_q8_0 / block_q5_0 rows of n_in/32 blocks (34 B / 22 B; n_in a
 * multiple of 32): the types a Q4_K_M GGUF holds for rows that are not whole
 * 256-weight super-blocks, loaded by candle at pagoda-hf/src/qwen2_gguf.rs:
 * 283-289 like the k-quants. Format ids 3 and 4 in pgd_matrix_info. */
int pgd_matrix_upload_q8_0(pgd_dev* dev, const void* blocks, int n_out, int n_in, pgd_matrix** out);
int pgd_matrix_upload_q5_0(pgd_dev* dev, const void* blocks, int n_out, int n_in, pgd_matrix** out);
/* ---- MXFP4 (OCP microscaling formats v1.0; no reference counterpart) --------
 * Blocks of 32 consecutive elements of a row: 4-bit codes (bit 3 the sign, then
 * 0 .5 1 1.5 2 3 4 6) and one scale byte s that stands for 2^(s - 127); s = 255
 * makes the block NaN. Row-major planes: codes, element 2 i of a row in the low
 * nibble of byte i, and one scale byte per block. Format id 5 in
 * pgd_matrix_info; pgd_matrix_dequant, pgd_matrix_gemv, pgd_matrix_gemv_dev and
 * pgd_matrix_gemv_swiglu_dev take these matrices too. n_in is a multiple of 32, both
 * sides are at most 2^30. In a stream capture no matrix is made (PGD_ERR_STATE).
 *
 * upload: host planes, codes [n_out][n_in / 2], scales [n_out][n_in / 32]. */
int pgd_matrix_upload_mxfp4(pgd_dev* dev, const uint8_t* codes, const uint8_t* scales, int n_out, int n_in,
                            pgd_matrix** out);
/* The same from device planes, code rows ldc and scale rows lds bytes apart
 * (multiples of 16, the planes 16-byte aligned). Queued on the handle's stream:
 * the planes may go once it has run. */
int pgd_matrix_from_mxfp4_dev(pgd_dev* dev, const uint8_t* codes, int ldc, const uint8_t* scales, int lds, int n_out,
                              int n_in, pgd_matrix** out);
/* Rows x [nrows, k] of f32 (x_type 0), f16 (1) or bf16 (2), row stride ldx
 * elements (a multiple of 8; x 16-byte aligned), to MXFP4 planes with strides as
 * above. A block's scale is the power of two of its largest magnitude over 4
 * (s at most 252, at least 0); codes are x / scale rounded to nearest, ties to
 * the even code, magnitudes above 6 to 6. A block with an infinity or NaN gets
 * s = 255 and codes 0. values (nullable; row stride ldv, a multiple of 4,
 * 16-byte aligned) receives the f32 values that codes and scales stand for.
 * Bytes of a plane's row past its codes or scales are left as they were. */
int pgd_mxfp4_quantize_dev(pgd_dev* dev, const void* x, int x_type, int ldx, int nrows, int k, uint8_t* codes, int ldc,
                           uint8_t* scales, int lds, float* values, int ldv);

/* Seeded synthetic matrix: N(0, std) weights quantized on the device (no
 * reference counterpart: the reference only loads checkpoints). */
int pgd_matrix_synth(pgd_dev* dev, int fmt, int n_out, int n_in, uint64_t seed, uint64_t key, float std,
                     pgd_matrix** out);
int pgd_matrix_free(pgd_matrix* m);
/* fmt, n_out, n_in, device bytes, algorithmic bytes (bpw * n_out * n_in / 8). */
int pgd_matrix_info(const pgd_matrix* m, int* fmt, int* n_out, int* n_in, size_t* dev_bytes,
                    double* algo_bytes);
/* Dequantize rows to f32 host memory [rows, n_in]; replaces
 * Affine::dequant_rows (pagoda-hf/src/qwen3_5.rs:1546-1584). Bit-exact. */
int pgd_matrix_dequant(const pgd_matrix* m, int row0, int rows, float* out);
/* y[r, :] = W . x[r, :] for r < nrows (nrows 1..64 ragged batch rows), x f32
 * [nrows, n_in], y f32 [nrows, n_out]. Replaces QuantMatrix::gemv and
 * encode_gemm4 (pagoda-hf/src/qwen3_gemv.rs:730-742, 826-846). */
int pgd_matrix_gemv(const pgd_matrix* m, const float* x, int nrows, float* y);
/* Device form. x f32 (x_f16 = 0) or IEEE f16 (x_f16 = 1), row stride ldx
 * elements (multiple of 8); y row stride ldy; res (nullable) adds a residual
 * y = res + W.x (replaces affine_gemv_res, qwen3_gemv.rs:289-306).
 * MXFP4 matrices also take bf16 rows (x_f16 = 2; to the other formats any nonzero
 * x_f16 is f16), and x must be 16-byte aligned. Sums are f32. f16 and bf16 rows and
 * up to 16 f32 rows enter the products exactly (f32 but for bits below 2^-133). More
 * f32 rows may be held, block of 32 by block, to 2^-30 of the power of two above the
 * block's largest magnitude (2^-130 at the finest); an infinity among them makes
 * its row NaN, and a result past the largest f32 is an infinity or NaN. A caller who
 * needs f32 rows exact passes at most 16 a call. The order of the sums depends on the
 * matrix, the number and type of rows and whether the stream is captured, on nothing
 * else. In a stream capture, rows that would need scratch memory are PGD_ERR_STATE and
 * queue nothing: all but up to 5 f32, 8 f16 or 4 bf16 rows and bf16 rows of n_in % 128
 * == 0 (the same holds for pgd_matrix_gemv_swiglu_dev; MXFP4 rows are never refused). */
int pgd_matrix_gemv_dev(const pgd_matrix* m, const void* x, int x_f16, int ldx, int nrows, float* y,
                        int ldy, const float* res, int ldres);
/* mid = silu(gate . x) * (up . x); replaces affine_gemv2_silu
 * (qwen3_gemv.rs:256-286). */
int pgd_matrix_gemv_swiglu_dev(const pgd_matrix* gate, const pgd_matrix* up, const float* x, int ldx,
                               int nrows, float* mid, int ldm);
/* Products of MXFP4 rows (planes as pgd_mxfp4_quantize_dev writes them, strides
 * as there; each plane nrows rows) with MXFP4 matrices, on the scaled 4-bit
 * matrix instructions with f32 sums: y = W.x, plus res (nullable) as in
 * pgd_matrix_gemv_dev, and mid = silu(gate.x) * (up.x). Any nrows >= 0. A plane's
 * row is read to its whole strides: whatever lies past its codes and scales does not
 * reach the results. */
int pgd_matrix_gemv_mx_dev(const pgd_matrix* m, const uint8_t* codes, int ldc, const uint8_t* scales, int lds, int nrows,
                           float* y, int ldy, const float* res, int ldres);
int pgd_matrix_gemv_swiglu_mx_dev(const pgd_matrix* gate, const pgd_matrix* up, const uint8_t* codes, int ldc,
                                  const uint8_t* scales, int lds, int nrows, float* mid, int ldm);
/* A8 activations converted once into matrix-core operands, shared by every
 * A8 matrix of width k (the reference shares one x across several matrices
 * the same way: gemv_shared / affine_gemv_n, qwen3_gemv.rs:149-253).
 * pgd_act_bytes gives the device buffer size for nrows x k. */
size_t pgd_act_bytes(int nrows, int k);
int pgd_act_prep_dev(pgd_dev* dev, const float* x, int ldx, int nrows, int k, void* act);
int pgd_matrix_gemv_act_dev(const pgd_matrix* m, const void* act, int nrows, float* y, int ldy, const float* res,
                            int ldres);
int pgd_matrix_gemv_swiglu_act_dev(const pgd_matrix* gate, const pgd_matrix* up, const void* act, int nrows,
                                   float* mid, int ldm);
/* candle's CPU QMatMul::forward for GGUF weights (called at
 * pagoda-hf/src/qwen2_gguf.rs:271-278, kept on the CPU by qweight at 280-289):
 * each f32 activation row (stride ldx) is quantized to Q8_K (Q4_K / Q6_K
 * weights) or Q8_0 (Q8_0 / Q5_0 weights), every output an integer block dot
 * scaled in f32. res (nullable) adds a residual as in pgd_matrix_gemv_dev. */
int pgd_matrix_gemv_q8act_dev(const pgd_matrix* m, const float* x, int ldx, int nrows, float* y, int ldy,
                              const float* res, int ldres);
/* Two pgd_matrix_gemv_q8act_dev calls over the same input rows in one launch
 * (the Qwen2 attention's q/k and v projections, qwen2_gguf.rs:234-236, whose
 * GGML types differ in Q4_K_M files): ya = a.x and yb = b.x, row stride ldy,
 * bit-equal to the two calls. Both matrices take the same input width and one
 * activation type (Q4_K / Q6_K: Q8_K; Q8_0 / Q5_0: Q8_0), else PGD_ERR_FORMAT. */
int pgd_matrix_gemv_q8act_pair_dev(const pgd_matrix* a, float* ya, const pgd_matrix* b, float* yb, const float* x,
                                   int ldx, int nrows, int ldy);
/* No counterpart in the reference. pgd_matrix_gemv_act_dev for callers that
 * cannot allocate device memory (code under HIP graph capture, tight serving
 * loops, harnesses that forbid hipMalloc): the same kernels and results, with
 * their scratch (split-K / stream-K partial sums) taken from one fixed
 * pgd_noalloc_scratch_bytes() (40 MiB) device array per GPU, held until the
 * process ends; calls no hipMalloc / hipFree. A launch needing more scratch
 * (37..64-row launches of matrices over ~41000 rows) is PGD_ERR_SHAPE before anything
 * runs. Every call on one GPU shares that array: a call queued on another
 * device handle's stream than the previous call's first waits (on the GPU,
 * through an event) for that call to finish; calls are serialized on the
 * host. The array keeps the last call's contents. */
size_t pgd_noalloc_scratch_bytes(void);
int pgd_matrix_gemv_act_dev_noalloc(const pgd_matrix* m, const void* act, int nrows, float* y, int ldy,
                                    const float* res, int ldres);

/* ---- decode-step kernels (device pointers, queued on the device stream) ----
 * Gated-DeltaNet recurrence over a ragged batch: sequence i owns rows
 * [row_start[i], row_start[i] + row_count[i]) and its fp32 state
 * states[i] -> [v_heads, 128, 128], updated in place, rows in order.
 * conv_out [rows, 2*k_heads*128 + v_heads*128] (post conv + SiLU: q | k | v),
 * a, b [rows, v_heads], z [rows, v_heads*128], out [rows, v_heads*128].
 * row_start, row_count and states are device arrays.
 * Replaces the per-token loop of LinearAttn::forward (pagoda-hf/src/
 * qwen3_5.rs:1330-1383) and gated_delta_step (qwen3_fuse.rs:176-279). */
int pgd_gdn_step_dev(pgd_dev* dev, int k_heads, int v_heads, const float* conv_out, const float* a,
                     const float* b, const float* z, const float* a_log, const float* dt_bias,
                     const float* norm, float* const* states, const int* row_start, const int* row_count,
                     int nseq, float* out);
/* pgd_gdn_step_dev for prefill: the same recurrence, where sequences of at
 * least 32 rows take the chunkwise form (32-token chunks: a triangular solve
 * and matrix products against each chunk's starting state, the published
 * chunked form of the gated delta rule; equal to the per-token loop in exact
 * arithmetic, to fp32 rounding in practice). rows: every sequence's
 * row_start + row_count is at most rows (rows past it are left unwritten,
 * never written out of bounds). max_rows: the largest row_count, or
 * any bound on it (below 32 every sequence takes the per-token kernel).
 * Replaces the same reference loop as pgd_gdn_step_dev, which it runs one
 * token at a time for prefill too (qwen3_5.rs:1330-1383). */
int pgd_gdn_prefill_dev(pgd_dev* dev, int k_heads, int v_heads, const float* conv_out, const float* a,
                        const float* b, const float* z, const float* a_log, const float* dt_bias,
                        const float* norm, float* const* states, const int* row_start, const int* row_count,
                        int nseq, int rows, int max_rows, float* out);
/* Paged GQA decode attention: row r attends to positions [0, pos_of_row[r]]
 * of sequence seq_of_row[r], whose pages are block_tables[seq * max_blocks
 * + p / block] in pools [pages][kv_heads][block][head_dim]. q, gate, out
 * [rows, heads, head_dim]; gate (nullable) applies sigmoid(gate). Replaces
 * FullAttn::forward's softmax attention (pagoda-hf/src/qwen3_5.rs:1433-1475)
 * and full_attn_heads (qwen3_fuse.rs:384-440) over a contiguous cache. */
int pgd_attn_decode_dev(pgd_dev* dev, int heads, int kv_heads, int head_dim, int block, const float* q,
                        const float* gate, const float* k_pool, const float* v_pool, const int* seq_of_row,
                        const int* pos_of_row, const int* block_tables, int max_blocks, int rows, float* out);

/* ---- 8-bit paged KV cache (no reference counterpart) --------------------------
 * K and V in a quarter of the bytes of the f32 pages, written, addressed and read by
 * calls that take everything of a step from device memory: no host plan, no
 * wait, no allocation, so a whole step can be captured in a HIP graph.
 *
 * A pool is n_pages pages of pgd_kv8_page_bytes(kv_heads, head_dim) bytes each, caller's
 * memory, 16-byte aligned (256 is faster). head_dim is 64, 128 or 256. A page holds 16
 * positions of every KV head; a position's slot is page * 16 + place. A (page, KV head)
 * holds its keys as e4m3 codes (OCP 8-bit floating point: 4 exponent and 3 mantissa bits,
 * largest 448) times one power of two, and its values as codes times another:
 * the smallest 2^e, e >= -126, with which the largest magnitude written fits. A page is
 * copied by copying its bytes (pgd_device_copy_dev); nothing in it names its place.
 * No page needs clearing before its first use. In every call here a slot or page
 * number outside the pool is never followed. Element types: f32 (0), f16 (1), bf16 (2).
 * Row strides (ld*) are in elements and multiples of 8 (of 4 in pgd_kv8_read_dev); rows,
 * pools and workspaces are 16-byte aligned. */
size_t pgd_kv8_page_bytes(int kv_heads, int head_dim);
/* A step's bookkeeping, for these pages or any others of `block` positions. Sequence i
 * has lens[i] positions, in the pages tables[i * max_blocks + p / block], and brings
 * counts[i] rows. Pages it needs beyond those it has come from free_pages[taken[0]..n_free) in
 * sequence order, and are entered into its table. Written: new_lens (lens + counts), new_taken
 * (both may be the input array), row_start [nseq + 1] (sequence i's rows, sequence after
 * sequence), and for each of `rows` rows seq_of_row, pos_of_row and slots (page * block +
 * place); -1 in all three for rows behind the last sequence's. No other output overlaps an
 * input. nseq is at most 2^24, rows at most 2^30. status[i]: 0; or why the
 * sequence got nothing (its rows are -1, its length and table stay): 1 too few free
 * pages, 2 more positions than max_blocks pages hold, 3 rows past `rows` (all sequences behind one that has some,
 * those without rows too), 4 a negative length or
 * count. A sequence that needs no page is not refused for those that do; of those that need some, all behind the
 * first that is refused for want of pages are refused too. Refused rows keep their place in row_start, so
 * an attention over it computes something for them, of the positions that the sequence has; it is to be ignored.
 * A table entry that is negative makes slots -1. Maps without a row of -1 serve pgd_attn_decode_dev, which refuses
 * such rows. */
int pgd_kv_tables_dev(pgd_dev* dev, int block, int nseq, const int* lens, const int* counts, int* tables,
                      int max_blocks, const int* free_pages, int n_free, const int* taken, int rows, int* new_lens,
                      int* new_taken, int* row_start, int* seq_of_row, int* pos_of_row, int* slots, int* status);
/* Rows k, v [rows, kv_heads * head_dim] into the slots slots[row] (negative, or past the
 * pool: the row is left out). The rows of one page follow each other, in
 * place order without gaps, as pgd_kv_tables_dev lays them out, and no other row of the call has
 * their page. A row at place 0 starts its page anew; otherwise the page holds the
 * places before the first row written, and places behind the last one become empty. If a row
 * needs a larger power of two than its page has, the codes there are rounded again to the larger
 * one; it never falls while the page fills. Rounding is to nearest, ties to the even code (a
 * value within half a step of 2^128 reads as an infinity).
 * A (row, KV head) with an infinity or NaN in k or v reads as NaN, and makes NaN
 * what attends it; its page's other positions are not affected. */
int pgd_kv8_append_dev(pgd_dev* dev, void* pool, int n_pages, int kv_heads, int head_dim, const void* k, int ldk,
                       const void* v, int ldv, int type, const int* slots, int rows);
/* The f32 values at slots[row]: k, v [rows, kv_heads * head_dim]. Rows of a slot outside the pool
 * are left as they were. */
int pgd_kv8_read_dev(pgd_dev* dev, const void* pool, int n_pages, int kv_heads, int head_dim, const int* slots,
                     int rows, float* k, int ldk, float* v, int ldv);
/* Causal GQA attention. Sequence i owns the rows [row_start[i], row_start[i + 1]) (clamped to
 * rows), the latest of its lens[i] positions, and row j of its n attends to positions
 * [0, lens[i] - n + j]: softmax(q k^T / sqrt(head_dim)) v, times sigmoid(gate) if
 * there is one. q, gate, out [rows, heads * head_dim] of one type; heads is a multiple of
 * kv_heads. Positions past max_blocks pages do not exist. A row that attends to nothing
 * gets zeros; rows of no sequence are left as they were; attending a position of a page outside the pool
 * gives NaN. Sums, maxima and the weights' sum are f32. Before the products on the matrix cores f32 rows of q are held
 * to 2^-22 and bf16 rows exactly, but to no less than 2^-39 of the head's largest entry, f16 rows exactly; the softmax
 * weights to 2^-21, but to no less than 2^-36 of the largest. An infinity or NaN in a head of q makes that head's
 * result NaN. A score of magnitude 2^127 and more is an infinity: a result whose largest score is one is NaN.
 * max_rows: the largest number of rows of a sequence, or any bound on it (it selects kernels, results are right with
 * any value). row_start ascends. ws: pgd_attn_kv8_rows_ws_bytes bytes, or pgd_attn_kv8_ws_bytes for any
 * max_rows (0 of sizes that the call refuses), that no other stream uses meanwhile (a captured graph's included); its
 * contents do not matter, and one that is large enough for a call is for every call of smaller numbers. The order of the
 * sums depends on the sizes, max_rows, row_start and lens, on nothing else. */
size_t pgd_attn_kv8_ws_bytes(int heads, int kv_heads, int head_dim, int nseq, int max_blocks, int rows);
size_t pgd_attn_kv8_rows_ws_bytes(int heads, int kv_heads, int head_dim, int nseq, int max_blocks, int rows,
                                  int max_rows);
int pgd_attn_kv8_dev(pgd_dev* dev, const void* pool, int n_pages, int kv_heads, int head_dim, int heads, const void* q,
                     int ldq, int type, int nseq, const int* row_start, const int* lens, const int* block_tables,
                     int max_blocks, int rows, int max_rows, void* out, int ldo, const void* gate, int ldg, void* ws,
                     size_t ws_bytes);
/* Per (row, KV head) the `top` pages of the row's context with the highest scores, as places in its
 * block table: sel [rows, kv_heads, top], ascending, -1 behind the count[row, kv_heads] =
 * min(top, pages) entries. The first `sinks` and the last `recent` pages are always among
 * them (sinks + recent <= top). The score bounds q.k over the page: q in signed 8 bits (q8 =
 * q / 2^e to nearest, ties to even, 2^e the smallest power of two, e >= -126, that keeps
 * the group's heads within 127; non-finite entries count as 0), the page's key codes bounded per
 * channel by whole numbers hi and lo (the largest and smallest code over 4, rounded outward; the
 * append keeps them): score = 2^(key exponent) max over the group's heads of
 * sum(max(q8 hi, q8 lo)), exact in f32 (an infinity from 2^128 on); ties go to the lower page. A page outside the pool scores
 * lowest. Rows of no sequence are left as they were; a row that attends to nothing selects nothing.
 * ws as above, of pgd_kv8_sparse_ws_bytes bytes, which serves both calls, one after the other, and those of fewer rows,
 * narrower tables and lower top too. */
size_t pgd_kv8_sparse_ws_bytes(int heads, int kv_heads, int head_dim, int rows, int max_blocks, int top);
int pgd_kv8_select_dev(pgd_dev* dev, const void* pool, int n_pages, int kv_heads, int head_dim, int heads,
                       const void* q, int ldq, int type, int nseq, const int* row_start, const int* lens,
                       const int* block_tables, int max_blocks, int rows, int top, int sinks, int recent, int* sel,
                       int* count, void* ws, size_t ws_bytes);
/* pgd_attn_kv8_dev over the pages sel[row, kv head, 0..count) alone (count is taken within
 * 0..top; entries outside the table or past the row's context are skipped, a page named twice counts twice). */
int pgd_attn_kv8_sparse_dev(pgd_dev* dev, const void* pool, int n_pages, int kv_heads, int head_dim, int heads,
                            const void* q, int ldq, int type, int nseq, const int* row_start, const int* lens,
                            const int* block_tables, int max_blocks, int rows, int top, const int* sel,
                            const int* count, void* out, int ldo, const void* gate, int ldg, void* ws,
                            size_t ws_bytes);

/* ---- models and sessions ---------------------------------------------------
 * Architecture of a model handle. arch 0 is the hybrid Qwen3.5 tower
 * (Gated-DeltaNet + gated full attention, MLX affine-8 weights; Qwen35::load
 * pagoda-hf/src/qwen3_5.rs:338-452); arch 1 is Qwen2 with GGUF Q4_K/Q6_K
 * weights and tied embeddings (Qwen2Gguf::load pagoda-hf/src/qwen2_gguf.rs:65-140). */
enum { PGD_ARCH_QWEN35 = 0, PGD_ARCH_QWEN2 = 1 };

typedef struct pgd_model_config {
  int arch;
  int n_layers, hidden, intermediate, vocab;
  int heads, kv_heads, head_dim, rotary_dim;
  float rope_theta, eps;
  int k_heads, v_heads, k_dim, v_dim, conv_kernel; /* gated-delta layers (arch 0) */
  int full_every; /* arch 0: layer i is full attention iff i % full_every == full_every - 1 */
  int max_pos;    /* context limit (qwen2_gguf.rs:146-150) */
  int kv_block;   /* tokens per KV page (16) */
  int kv_blocks;  /* KV pages per full-attention layer */
} pgd_model_config;

typedef struct pgd_model pgd_model;
typedef struct pgd_session pgd_session;

/* Build a model with seeded synthetic weights generated on the device (the
 * configs use random-init weights; no reference counterpart). */
int pgd_model_synth(pgd_dev* dev, const pgd_model_config* cfg, uint64_t seed, pgd_model** out);
/* Qwen35::load (pagoda-hf/src/qwen3_5.rs:338-452, store 1587-1698): the
 * language model of an MLX directory (config.json; model.safetensors.index.json
 * and its shards, or a single model.safetensors). Matrices are 8-bit affine
 * group 64 (u32 codes, bf16 scales / biases); norms, conv, A_log and dt_bias
 * F32 / BF16 / F16. Layer kinds come from config.json's layer_types.
 * max_pos <= 0: max_position_embeddings; kv_blocks > 0: KV pages per
 * full-attention layer. Errors (missing tensors, shapes, quantization other
 * than 8-bit affine group 64) return kErrFormat and allocate nothing. */
int pgd_model_load_mlx(pgd_dev* dev, const char* dir, int max_pos, int kv_blocks, pgd_model** out);
/* Qwen2 GGUF load (pagoda-hf/src/qwen2_gguf.rs:65-140): GGUF v2/v3,
 * general.architecture "qwen2"; Q4_K / Q6_K / Q8_0 / Q5_0 matrices, F32 / F16 norms and
 * q/k/v biases; lm_head is output.weight or the tied token_embd.weight.
 * Tensors in other ggml block types are an error naming the tensor.
 * max_pos <= 0: qwen2.context_length. */
int pgd_model_load_gguf(pgd_dev* dev, const char* path, int max_pos, int kv_blocks, pgd_model** out);
/* The configuration a loader derives from a checkpoint (a directory: MLX;
 * a file: GGUF), without a device; no reference counterpart. */
int pgd_checkpoint_config(const char* path, int max_pos, int kv_blocks, pgd_model_config* cfg);
/* The configuration of a model (synthetic or loaded). */
int pgd_model_config_get(const pgd_model* m, pgd_model_config* cfg);
/* Arithmetic of a model's GGML-format matrices (the Qwen2 GGUF path). The
 * reference computes them two ways: candle's CPU quantized matmul
 * (PGD_ARITH_CPU_Q8, activations quantized to Q8_K / Q8_0; the default for
 * Qwen2 models, matching the reference CPU path's tokens) or dequantized
 * weights (Metal, qwen2_gguf.rs:280-289), here f32 dequant-then-dot
 * (PGD_ARITH_DEQUANT_F32). A8 (hybrid model) matrices are unaffected. */
enum { PGD_ARITH_DEQUANT_F32 = 0, PGD_ARITH_CPU_Q8 = 1 };
int pgd_model_set_kquant_arith(pgd_model* m, int mode);
/* No reference counterpart (the reference's Metal path encodes every kernel
 * of a token into one command buffer, qwen3_fuse.rs). on != 0: each step's
 * launches (embedding to argmax) are captured once per launch signature
 * (batch shape, buffers, attention plan layout) into a HIP graph and replayed
 * on later steps with the same signature; per-step data (tokens, positions,
 * page tables) is uploaded before the replay. Results are bitwise those of
 * the eager launches. The first step of a signature runs eagerly, the second
 * is captured. graph_stats: graphs held, replays so far. */
int pgd_model_set_graphs(pgd_model* m, int on);
int pgd_model_graph_stats(const pgd_model* m, int* graphs, long long* launches);
int pgd_model_free(pgd_model* m);
/* weight bytes on the device, algorithmic weight bytes per decode step, KV pages free */
int pgd_model_info(const pgd_model* m, size_t* weight_bytes, double* algo_bytes_per_token, int* kv_free);

/* ModelEngine::begin_session (pagoda/src/model.rs:78-80). */
int pgd_session_new(pgd_model* m, pgd_session** out);
/* ModelSession::fork (pagoda/src/model.rs:185-187): KV pages are shared
 * copy-on-write, the recurrent state is copied. */
int pgd_session_fork(const pgd_session* s, pgd_session** out);
int pgd_session_free(pgd_session* s);
/* ModelSession::context_len (pagoda/src/model.rs:165). */
int pgd_session_len(const pgd_session* s, int* len);
/* ModelSession::forward (pagoda/src/model.rs:167): feed n >= 0 tokens, write
 * the last position's logits [vocab] (n == 0 repeats the cached logits). */
int pgd_forward(pgd_session* s, const uint32_t* toks, int n, float* logits);
/* Qwen35::forward_greedy (pagoda-hf/src/qwen3_5.rs:511-530): one token in,
 * greedy id and its logit out (device argmax; ties keep the last max). */
int pgd_forward_greedy(pgd_session* s, uint32_t tok, uint32_t* id, float* logit);
/* Qwen35::forward_verify (pagoda-hf/src/qwen3_5.rs:663-755): n in 1..4
 * teacher-forced tokens, greedy id and logit per position. */
int pgd_forward_verify(pgd_session* s, const uint32_t* toks, int n, uint32_t* ids, float* logits_max);
/* Ragged batched step (ModelEngine::session_forward_batch,
 * pagoda/src/model.rs:88-94, widened to multi-token rows): session i feeds
 * n_per_seq[i] >= 1 tokens from toks (concatenated). ids receive the greedy
 * id (first max, pagoda/src/sampler.rs:59-69) of each session's last position
 * (all_rows = 0) or of every fed position (all_rows = 1); 0xFFFFFFFF marks a
 * row with any non-finite logit, which the engine faults
 * (pagoda/src/engine.rs:1278-1280: only that request, its batch-mates are
 * unaffected). logits (nullable) receive the matching rows [rows][vocab].
 * Atomic on argument errors: no session advances. A device error after the
 * step has begun writing (GDN state and KV pages are updated in place) marks
 * every session of the step unusable: later calls on them return
 * PGD_ERR_STATE instead of continuing from half-advanced state. */
int pgd_step_ragged(pgd_model* m, pgd_session* const* sessions, const uint32_t* toks, const int* n_per_seq,
                    int nseq, int all_rows, uint32_t* ids, float* logits);
/* ModelSession::export_kv / ModelEngine::import_session (pagoda/src/model.rs:
 * 137, 89). Hybrid model (arch 0): Qwen35Cache::to_bytes /
 * from_bytes, cache format v1 (pagoda-hf/src/qwen3_5.rs:177-256). Qwen2 (arch
 * 1): the SessionKv PD payload (CandleCausalLM::cache_export / cache_import,
 * pagoda-hf/src/llama.rs:215-345) with the session's last logits, which an
 * imported session replays on an empty feed (pagoda-hf/src/lib.rs:644-667).
 * export writes *len bytes when buf is large enough (pass buf = NULL to
 * query). */
int pgd_session_export(const pgd_session* s, uint8_t* buf, size_t cap, size_t* len);
int pgd_session_import(pgd_model* m, const uint8_t* buf, size_t len, pgd_session** out);
/* set_kv_wire_f16 (pagoda-hf/src/llama.rs:128-136): process-wide choice of the
 * SessionKv export's K/V encoding, f32 (0, default) or f16 (1). */
int pgd_set_kv_wire_f16(int on);
/* CandleCausalLM::cache_prefix (pagoda-hf/src/lib.rs:219-226;
 * qwen2_gguf.rs:183-185 -> SessionKv::prefix, llama.rs:81-101), used by
 * graft_session (lib.rs:603-616): a new session holding the first n
 * positions of s. KV pages below n are shared; the partial last page is
 * copied on the new session's first write, so appends never disturb s.
 * Cached logits are not carried (a graft has none, lib.rs:613).
 * PGD_ERR_STATE for the hybrid model: GDN state cannot be cut to a prefix
 * (the trait's default None, lib.rs:224). */
int pgd_session_fork_prefix(const pgd_session* s, int n, pgd_session** out);

/* ---- engine-addressable KV pages ------------------------------------------
 * The engine's PagedKvCache hands out physical BlockIds with reference counts
 * and copy-on-write, "exactly what a tensor-backed implementation would swap
 * in" (pagoda/src/kv_cache.rs:1-8, alloc/inc_ref/dec_ref/ref_count 65-105),
 * and its RadixCache maps each cached token to a KvSlot = (BlockId, offset)
 * (pagoda/src/radix_cache.rs:17-18). A page id here names one page of
 * kv_block positions in every full-attention layer's K and V pools; position
 * p of a session lives in slot p % kv_block of its page p / kv_block.
 * Sessions and the engine hold references alike; a page returns to the pool
 * when its count reaches zero, and a session copies a shared, partly filled
 * page before its first write into it. */
/* PagedKvCache::num_blocks / block_size / num_free_blocks (kv_cache.rs:48-56);
 * each output nullable. */
int pgd_model_kv_pool(const pgd_model* m, int* n_pages, int* page_tokens, int* n_free);
/* The page ids holding positions [0, len) of s, in position order. *n gets
 * the count (ids = NULL queries it); cap below it is PGD_ERR_ARG. */
int pgd_session_pages(const pgd_session* s, int32_t* ids, int cap, int* n);
/* PagedKvCache::inc_ref / dec_ref (kv_cache.rs:90-105) on n held pages (a free
 * page or an id outside the pool is an error and changes nothing). */
int pgd_page_retain(pgd_model* m, const int32_t* ids, int n);
int pgd_page_release(pgd_model* m, const int32_t* ids, int n);
/* PagedKvCache::ref_count (kv_cache.rs:74). */
int pgd_page_refcount(const pgd_model* m, int32_t id, int* count);
/* A new session of length n_pos whose KV is the held pages ids[0..n_pages)
 * (n_pages = ceil(n_pos / kv_block), distinct): the radix cache's matched
 * slots become the session's cache without a copy; the session takes its own
 * reference on each page. No cached logits (as a graft, lib.rs:603-616).
 * PGD_ERR_STATE for the hybrid model, whose recurrent state is not a
 * function of KV pages (cache_prefix default None, lib.rs:224). */
int pgd_session_from_pages(pgd_model* m, const int32_t* ids, int n_pages, int n_pos, pgd_session** out);

#ifdef __cplusplus
}
#endif
#endif

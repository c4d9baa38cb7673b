/*
 * jepa_amd.h - entry points of libjepa.so beyond the reference API (include/jepa.h).
 *
 * The reference has no counterpart for these; they exist for callers that keep data on the GPU
 * (benchmarks, pipelines feeding decoded frames from device memory) and for parity tests that check
 * one kernel at a time against the CPU oracle. Pointers named *_dev are HIP device pointers on the
 * given device; every call is synchronous (it returns after its kernels finished) unless stated.
 * Return values: >= 0 on success, -1 on failure with the reason in jepa_error_text().
 */
#pragma once
#include "jepa.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- encoder on device-resident data -------------------------------------------------------- */
/* jepa_encode without the host copies: in_dev is the NCTHW float32 input already on the model's
 * device, out_dev receives [rows, embed_dim] float32 rows (same order as jepa_encode). Replaces the
 * host-side patchify + tensor_set / tensor_get of reference src/jepa.cpp:990-1019 with device data.
 * Returns the rows per item (jepa_token_grid) or -1. last_compute_ms is set as for jepa_encode. */
int64_t jepa_amd_encode_device(jepa_context * ctx, const float * in_dev, int n_batch, int n_chans, int n_frames,
                               int height, int width, float * out_dev, int64_t out_cap_floats);

/* jepa_head_ex on device-resident encoder rows: x_dev [n_tokens][embed_dim] float32 on the model's
 * device; pooled_dev [embed_dim] and logits_dev [n_classes] (device, either may be NULL) receive
 * the pooled token and the classifier logits. Replaces the tensor_set / tensor_get of reference
 * src/jepa.cpp:1093-1110 with device data. Returns n_classes, or -1 with the reason in
 * jepa_error_text(). last_compute_ms covers the head's kernels. */
int jepa_amd_head_device(jepa_context * ctx, const float * x_dev, int64_t n_tokens, float * pooled_dev, float * logits_dev);

/* jepa_encode that also returns the residual stream after the patch embedding and after every
 * block (before the final norm): trace [n_items][n_layer + 1][rows][dim] on the host. For per-layer
 * parity checks; runs without graph replay. */
int64_t jepa_amd_encode_trace(jepa_context * ctx, const jepa_input * in, float * out, int64_t out_cap_floats,
                              float * trace, int64_t trace_cap_floats);

/* ---- context knobs --------------------------------------------------------------------------- */
/* Record hipEvents around every kernel launch of the next encodes (disables graph replay) and sum
 * their device time per kernel class: "patchify", "patch_embed", "layernorm", "gemm_q8",
 * "gemm_q4k", "gemm_f16", "gemm_f32", "attention", "quantize", "cls". */
void jepa_amd_context_set_kernel_timing(jepa_context * ctx, bool on);
int  jepa_amd_context_kernel_stats(const jepa_context * ctx, const char * kernel_class, int64_t * n_launches, double * total_ms);
void jepa_amd_context_reset_kernel_stats(jepa_context * ctx);
/* Capture the forward into a hipGraph and replay it (default on; $JEPA_HIP_GRAPH=0 turns it off). */
void jepa_amd_context_set_graph(jepa_context * ctx, bool on);
/* The HIP stream (hipStream_t) the context launches on. */
void * jepa_amd_context_stream(const jepa_context * ctx);

/* ---- single-kernel hooks (parity tests, micro-benchmarks) ------------------------------------ */
/* ggml to_float of q8_0 / q4_0 / q4_K / f16 rows: blocks_dev holds n_rows rows of n_cols values in
 * the ggml block layout (ggml_type ids 8 / 2 / 12 / 1). */
int jepa_amd_dequantize(int device, int ggml_type, const void * blocks_dev, int64_t n_rows, int64_t n_cols, float * y_dev);

/* Row-wise LayerNorm (ggml_norm + optional affine, normalize = 1) or plain conversion (normalize = 0)
 * of x_dev [n_rows][n_cols], written as out_type: 0 f32 rows, 1 f16 rows, 8 q8_0 blocks (34 B per 32),
 * 15 q8_K blocks (292 B per 256) in ggml's block layout - the activation quantization the GEMMs
 * consume (x86 quantize_row_q8_0 / quantize_row_q8_K_ref semantics). */
int jepa_amd_rownorm(int device, const float * x_dev, int64_t n_rows, int64_t n_cols, const float * w_dev,
                     const float * b_dev, float eps, int normalize, int out_type, void * out_dev);

/* Y = X W^T (+ bias): W_dev in ggml blocks of wtype (8 q8_0, 2 q4_0, 12 q4_K, 1 f16, 0 f32) [n_out][n_in],
 * X_dev f32 [n_rows][n_in], Y_dev f32 [n_rows][n_out]; the activations are quantized to the weight's
 * vec-dot type first, like ggml_mul_mat (reference src/jepa.cpp:365-375). reps > 1 repeats the GEMM
 * (same result); *gemm_ms (optional) receives the mean device time of one GEMM launch. */
int jepa_amd_matmul(int device, int wtype, const void * w_dev, int64_t n_out, int64_t n_in, const float * bias_dev,
                    const float * x_dev, int64_t n_rows, float * y_dev, int reps, double * gemm_ms);

/* The MLP's first linear with its fused epilogue: out = gelu_erf(X W^T + bias) (reference
 * src/jepa.cpp:365-385), written the way the encoder hands it to the second linear. out_type 0 (f32):
 * out_dev f32 [n_rows][n_out]; 1 (f16): f16 values; 8 (q8_0) / 15 (q8_K): ggml blocks of the quantized
 * rows (q8_K needs n_out % 256 == 0). W, X, bias as for jepa_amd_matmul. reps > 1 repeats the GEMM
 * (same result); *gemm_ms (optional) receives the mean device time of one repeat. */
int jepa_amd_matmul_gelu(int device, int wtype, const void * w_dev, int64_t n_out, int64_t n_in, const float * bias_dev,
                         const float * x_dev, int64_t n_rows, int out_type, void * out_dev, int reps, double * gemm_ms);

/* Attention of one block from its fused qkv rows: qkv_dev f32 [n_items*n_tok][3*n_head*hd] (rows
 * [q | k | v], head-major), head width hd (a multiple of 16 up to 128), optional RoPE tables rope_c/rope_s [n_tok][hd]
 * (signed sine). Runs the QKV epilogue's split/RoPE/f16 cast and the attention kernel. tokens_per_slot
 * > 0 applies the LeVJEPA block-causal mask (reference src/jepa.cpp:827-844): the n_prefix leading
 * rows read every key, a patch row reads the patch keys of its own and earlier temporal slots of
 * tokens_per_slot rows, and no prefix key; 0 is full attention. out_type 0 (f32): out_dev f32
 * [n_items*n_tok][n_head*hd]; 8 (q8_0, head widths 32 and 64): out_dev ggml q8_0 blocks of those
 * rows, as the attention kernel's fused epilogue quantizes them for the out-projection; 1 (f16): out_dev f16
 * rows, the f32 values rounded to nearest, the input of an f16 out-projection. */
int jepa_amd_attention(int device, const float * qkv_dev, int64_t n_items, int64_t n_tok, int n_head, int hd,
                       const float * rope_c_dev, const float * rope_s_dev, int n_prefix, int64_t tokens_per_slot,
                       int out_type, void * out_dev);

/* jepa_preprocess_frames_rgb_ex on the device: n_frames RGB8 HWC frames of h x w, contiguous in device
 * memory ([n_frames][h][w][3]), are resized (uint8 antialias), centre-cropped and normalised into
 * out_dev, NCTHW f32 [3][n_frames][crop][crop] (N = 1), bit-identical to the host function. The clip
 * then goes to jepa_amd_encode_device without a host round trip, and only uint8 frames cross PCIe.
 * out_cap is out_dev's size in floats; out_h / out_w receive the crop. Returns 0, or -1 with the
 * reason in jepa_error_text(). Replaces the host half of reference src/preprocess.cpp:233-300. */
int jepa_amd_preprocess_frames_device(int device, const jepa_preprocess_params * p, const uint8_t * frames_dev, int n_frames, int h,
                                      int w, float * out_dev, int64_t out_cap, int * out_h, int * out_w);

/* jepa_amd_preprocess_frames_device without any allocation: no counterpart in the reference. For
 * callers that cannot allocate device memory (code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc). The tap tables and the horizontal-pass image live in a static
 * device array of 32 MiB that every GPU the library runs on holds until the process ends; a call
 * whose scratch would exceed it (about n_frames * h * crop * 3 bytes plus the tables) is refused
 * with -1 and a message. Work is queued on `stream` (a hipStream_t of `device`; NULL: the null
 * stream) and the call returns without waiting for it; the output is, bit for bit, that of
 * jepa_amd_preprocess_frames_device. Most calls run a kernel that needs neither tables nor the array;
 * nothing is copied from host memory in any (tables, where there are some, reach the device as kernel
 * arguments), so the call can be captured into a HIP graph (make one call on the device before
 * capturing, which looks up the array's address) and the graph replayed on new frames
 * of the same geometry. Calls on one GPU share the array: calls whose work overlaps on one GPU (on
 * different streams, or graph replays beside eager calls) race, and the caller orders them. */
int jepa_amd_preprocess_frames_device_noalloc(int device, const jepa_preprocess_params * p, const uint8_t * frames_dev, int n_frames,
                                              int h, int w, float * out_dev, int64_t out_cap, int * out_h, int * out_w, void * stream);

/* Split-K of the GEMMs with the residual or plain f32 epilogue (S workgroups per output tile, one per
 * K part; the last to finish adds the parts' sums in part order): q8_0 / q4_0 / q4_K run in 1 or 2
 * halves chosen from n_out and n_in only; f16 weights in 1 to 4 parts when the tiles leave most CUs
 * idle (few rows) and K >= 1024. jepa_amd_gemm_split forces S for later launches (1 = off; 2 for the
 * int8 / 4-bit types; 2, 3 or 4 for f16 where K allows, else unsplit) or restores the automatic choice (-1);
 * jepa_amd_gemm_split_of returns the halves of a q8_0 / q4_0 / q4_K GEMM of this shape (1 for f16,
 * whose parts depend on the row count; the other epilogues do not split). */
int jepa_amd_gemm_split(int split);
int jepa_amd_gemm_split_of(int wtype, int64_t n_out, int64_t n_in);

/* ---- GGUF quantizer ---------------------------------------------------------------------------
 * The reference's jepa-quantize (tools/jepa-quantize.cpp) as a library call: in_path (an f32 / f16
 * jepa GGUF, or a quantized one with allow_requant) -> out_path with the 2-D attention / FFN /
 * projection / classifier weights re-typed to `type` ("f32", "f16", "q8_0", "q4_0", "q4_k"; f32
 * widens every tensor), the same keep rule, per-tensor K-quant fallback to q4_0, metadata copied in
 * order with general.file_type updated, GGUF v3 with 32-byte alignment. Tensors whose name contains
 * one of the n_keep strings in `keep` keep their type. The block quantizers run on HIP device
 * `device` (-1: 0) and are bit-exact with ggml's reference quantizers. verbose logs the plan.
 * Returns 0, or -1 with the reason in jepa_error_text(). */
int jepa_amd_quantize_file(const char * in_path, const char * out_path, const char * type, const char * const * keep, int n_keep,
                           bool allow_requant, int device, bool verbose);

/* f32 values on the device -> ggml blocks of gtype (8 q8_0, 2 q4_0, 12 q4_K) or f16 (1), bit-exact
 * with ggml's reference quantizers (test hook of the quantizer kernels). n must be whole blocks. */
int jepa_amd_quantize_rows(int device, int gtype, const float * x_dev, int64_t n, void * out_dev);

/* One v_mfma_f32_32x32x16_f16 on host matrices a [32][16], b [16][32] -> d [32][32] (row-major),
 * written back through the accumulator layout the GEMM epilogues assume. */
int jepa_amd_mfma_probe(int device, const float * a, const float * b, float * d);

/* The 3-D RoPE tables this library uploads for an encoder (host only, no device work): [n_rows][head_dim]
 * cos and sin rows for grid (grid_t, grid_h, grid_w), variant 0 (V-JEPA 2, tiled) or 1 (V-JEPA 2.1,
 * interleaved), with the 2.1 interpolation to (train_h, train_w) when interpolate is set. ids (may
 * be NULL: every token, T-major) selects rows of the grid. signed_sin = 1 gives the sine table with
 * the rotation's sign on the even lanes, as the QKV epilogue reads it; 0 the plain sines. Replaces
 * nothing in the reference: it exposes the tables of reference src/rope3d.cpp:9-134 to the tests
 * that pin them against the reference's golden vectors. Returns 0, or -1 on a bad argument. */
int jepa_amd_rope_tables(int head_dim, int grid_t, int grid_h, int grid_w, int variant, int interpolate, int train_h, int train_w,
                         float theta, const int32_t * ids, int64_t n_rows, int signed_sin, float * cos_out, float * sin_out);

/* Throughput ceiling of the q8_0 GEMM's inner step from registers alone (no memory, no barriers), one
 * workgroup per CU with waves_per_simd (1-4) waves on each SIMD: per 32x32x32 block and MFMA tile one
 * int8 MFMA (the block sum), one f16 MFMA (the scale products) and 32 VALU ops (16 conversions, 16
 * fmas). mode 0: the whole step in each wave (the kernels' form); 1: the two MFMAs alone; 2: the VALU
 * ops alone; 3: even waves the MFMA half, odd waves the VALU half. *ns_per_step: nanoseconds of one SIMD
 * per whole step (65536 int8 ops). No counterpart in the reference: a measurement hook. */
int jepa_amd_gemm_step_probe(int device, int mode, int waves_per_simd, int iters, double * ns_per_step);

/* Copy of n float32 values between device buffers (a plain copy kernel, for counter calibration). */
int jepa_amd_copy(int device, const float * src_dev, float * dst_dev, int64_t n, int reps, double * ms);

/* ---- 4-bit paged key/value cache -------------------------------------------------------------------
 * Keys and values that stay on the device between calls, for predictors and decoders that run step by step (the reference
 * keeps an f16 / f32 one per context, jepa_ac_context_*). One cache is n_pages * jepa_amd_cache_page_bytes() bytes of
 * device memory that the caller allocates (one for each layer; 16-byte aligned; it need not be cleared); a page holds
 * page_size tokens of every K/V head as ggml q4_0 blocks along the head, 4.5 bits a value. A sequence's tokens lie in the
 * pages of its row of a block table: token t in page table[t / page_size]. A step is
 *     jepa_amd_cache_plan        once: which pages and slots the step's rows get
 *     jepa_amd_cache_store       for each layer: the rows' keys and values into their slots
 *     jepa_amd_cache_attention   for each layer: the rows' queries over their sequences
 * The calls queue their work on `stream` (a hipStream_t of `device`; NULL: the null stream), allocate nothing, do not wait
 * and can be captured into a HIP graph. All pointers but `shape` are device pointers. Rows are packed one after the other,
 * sequence by sequence, each row its heads one after the other; types are 0 f32, 1 f16, 30 bf16; strides are in elements;
 * row pointers and strides are multiples of 16 bytes. Outputs must not overlap inputs or each other unless stated. A call of
 * _store, _read or _attention has fewer than 2^27 heads of rows (n_rows times n_kv_head, for _attention n_head), and for
 * _attention n_rows * n_head / 16 + n_seq * n_kv_head stays below 2^24 - 2^13; much larger ones are refused. */
typedef struct {
    int32_t n_head;      /* query heads, a multiple of n_kv_head; head h reads K/V head h / (n_head / n_kv_head) */
    int32_t n_kv_head;
    int32_t head_dim;    /* 32, 64, 96 or 128 */
    int32_t page_size;   /* tokens of a page: 16, 32, 64, 128 or 256 */
    int64_t n_pages;     /* pages of the cache, below 2^31 */
} jepa_amd_cache_shape;

/* Bytes of one page, or -1 on a shape that is not supported (n_head and n_pages do not matter but are checked). */
int64_t jepa_amd_cache_page_bytes(const jepa_amd_cache_shape * shape);

/* One step's bookkeeping for n_seq sequences (up to 4096), n_rows packed rows and tables of table_width pages (2^30 tokens at most).
 *   len [n_seq]          tokens that each sequence has in the cache
 *   n_new [n_seq]        tokens that come to it in this step; below zero, that many are dropped from its end
 *   table [n_seq][table_width]   in and out: pages for the new tokens are written in, dropped pages' entries set to -1 (a page
 *                        that several rows of the table name is given back by each that drops it: let one of them drop it)
 *   ring [n_pages], free_in [2]  the free pages: free_in[1] of them from ring[free_in[0]] on, around the end. Pages are
 *                        taken at the front in sequence order; dropped pages are put behind the last, in sequence and table
 *                        order, and not taken again in the same step. A caller starts with ring = 0 .. n_pages - 1 and (0, n_pages).
 *   free_out [2]         the ring's front and count afterwards (may be free_in)
 *   kv_len [n_seq]       tokens of each sequence afterwards (may be len)
 *   row_start [n_seq + 1]  where its rows begin: the sums of the positive n_new, at most n_rows
 *   slot [n_rows]        the cache slot of each row, page * page_size + place; -1 for a row of a refused sequence and behind the last
 *   refused [n_seq]      1 where the step could not be done for a sequence: its lengths do not fit a table row, its rows end
 *                        past n_rows, or the free pages end before it (then every later one that needs a page is refused
 *                        too). It keeps its len and pages. Its rows keep their places: what _attention gives them is not the step's.
 * Entries of the ring, and of a table row within its len, are to be pages of the cache. They are not checked: other numbers
 * are handed on as they are (to the table, or to the ring where they are dropped) and refuse nothing; tokens on them have slot
 * -1, are not stored and not read. */
int jepa_amd_cache_plan(int device, const jepa_amd_cache_shape * shape, int64_t n_seq, int64_t n_rows, const int32_t * len,
                        const int32_t * n_new, int32_t * table, int64_t table_width, int32_t * ring, const int32_t * free_in,
                        int32_t * free_out, int32_t * kv_len, int32_t * row_start, int64_t * slot, int32_t * refused, void * stream);

/* Keys and values of n_rows rows ([n_kv_head * head_dim], k_stride / v_stride apart) quantized into their slots, ggml's
 * q4_0 scales and codes bit for bit (as jepa_amd_quantize_rows makes them of the rows in f32). Rows whose slot is negative or
 * past the cache are skipped; no slot may be given twice. Values beyond +-65504 are held there; a head of a row with a NaN or an
 * infinity in its K or V is stored as K NaN and V zero, so that a query which reads the token comes out NaN. */
int jepa_amd_cache_store(int device, const jepa_amd_cache_shape * shape, void * cache, int type, const void * k, int64_t k_stride,
                         const void * v, int64_t v_stride, int64_t n_rows, const int64_t * slot, void * stream);

/* The values that n_rows slots hold, rounded to `type`; rows whose slot is negative or past the cache come out zero. */
int jepa_amd_cache_read(int device, const jepa_amd_cache_shape * shape, const void * cache, const int64_t * slot, int64_t n_rows, int type,
                        void * k, int64_t k_stride, void * v, int64_t v_stride, void * stream);

/* out = softmax(scale * q K^T) V for each row and head over its sequence's cached tokens. Row j of the r rows of a sequence of
 * kv_len tokens stands at position kv_len - r + j, so the step's own tokens are stored first. causal_block 0: every row reads
 * all kv_len tokens; 1: those up to its own position; T: those of its own and earlier blocks of T positions (frames).
 * q and out hold rows of n_head * head_dim values of `type`; scores, sums and the softmax are f32. Keys and values enter as they
 * are held, with one exception: in a call with many rows of a sequence, bf16 rows take them rounded to f16 (2^-11 relative, an
 * eighth of bf16's half step). Weights are rounded to 2^-11 of themselves for f16 and bf16 rows, to 2^-22 for f32 rows, and to
 * 2^-35 of the row's largest; queries to 2^-22 (f32 rows) and to 2^-39 of the row's largest element: f32 rows are computed to f32
 * accuracy. Keys and values that a row does not read do not change it; the sizes and lengths of the call's sequences may
 * change its last bits (they decide how its keys are split and joined), and equal calls give equal bits.
 * Tokens whose page is not one of the cache's are not read; a row that reads nothing comes out zero; rows behind the last
 * sequence (row_start[n_seq] on) are left as they are.
 * row_start ascends; a call whose rows overlap writes some of them or none.
 * `work` is jepa_amd_cache_work_bytes() bytes of device memory (16-byte aligned) with nothing kept in it between calls; what
 * the largest step needs does for smaller ones. Calls that may overlap on the device (on two streams, in two graphs) need one each. */
int64_t jepa_amd_cache_work_bytes(const jepa_amd_cache_shape * shape, int64_t n_seq, int64_t n_rows, int64_t table_width);
int jepa_amd_cache_attention(int device, const jepa_amd_cache_shape * shape, const void * cache, int type, const void * q, int64_t q_stride,
                             int64_t n_seq, int64_t n_rows, const int32_t * row_start, const int32_t * kv_len, const int32_t * table,
                             int64_t table_width, float scale, int64_t causal_block, void * out, int64_t out_stride, void * work,
                             int64_t work_bytes, void * stream);

/* ---- rotary positions of several axes, and the cache with them -----------------------------------------
 * Frames step by (time, row, column), text by one position or the same on every axis. A head's first dims[0] elements belong to axis 0, the
 * next dims[1] to axis 1 and so on; the rest of it does not turn. Element j of a section of width w turns by the angle
 * A_j = pos[axis] * scale[axis] * theta^(-2 f / w), x'_j = x_j cos A_j -+ x_p sin A_j, p being its partner (minus for the first of a pair):
 *     form 0   pairs (2i, 2i + 1), f = j mod w / 2: a pair's elements turn by different angles (V-JEPA 2; reference src/rope3d.cpp:9-134, "tiled")
 *     form 1   pairs (2i, 2i + 1), f = i (V-JEPA 2.1, "interleaved"; the scales are its interpolation)
 *     form 2   pairs (i, i + w / 2), f = i
 *     form 3   pairs (i, i + W / 2) of all W = dims[0] + dims[1] + ... elements that turn, f = i with W for w; pair i belongs to the axis whose
 *              dims[axis] / 2 pairs it falls into
 * Angles are made in 64 bits, their cosines and sines rounded to f32, and so are the two products and their sum. Positions are int32, of either sign. */
typedef struct {
    int32_t head_dim;    /* 8 to 256, whole 8 */
    int32_t form;
    int32_t n_axes;      /* 1 to 4 */
    int32_t dims[4];     /* even; form 2: whole 16; form 3: whole 16 together */
    double  theta;       /* above 0 */
    double  scale[4];    /* every angle of a position is finite, or the call is refused */
} jepa_amd_rope_axes;

/* n_rows rows of n_head heads at positions pos [n_rows][n_axes] (device, int32), types, strides and pointers as for the cache's calls below. backward 0:
 * rotated; else the gradient with respect to x of the rotated rows' gradient (the transposed map). out may be x with the same stride. Up to 4096
 * heads, n_rows * n_head below 2^26. Queued on `stream`; allocates nothing, does not wait, can be captured into a HIP graph. */
int jepa_amd_rope_rows(int device, const jepa_amd_rope_axes * rope, int type, const void * x, int64_t x_stride, int64_t n_rows, int n_head,
                       const int32_t * pos, int backward, void * out, int64_t out_stride, void * stream);

/* jepa_amd_cache_store of keys that are rotated on the way, and queries rotated into q_out (which may be q, with the same stride; q NULL: keys and values
 * alone), in one launch. The rotated key is quantized from f32. Rows whose slot is negative or past the cache are not stored; their queries are rotated all
 * the same. n_rows * n_head stays below 2^26. */
int jepa_amd_cache_append(int device, const jepa_amd_cache_shape * shape, const jepa_amd_rope_axes * rope, void * cache, int type, const void * q,
                          int64_t q_stride, const void * k, int64_t k_stride, const void * v, int64_t v_stride, int64_t n_rows, const int32_t * pos,
                          const int64_t * slot, void * q_out, int64_t q_out_stride, void * stream);

/* ---- attention over pages that each row selects ----------------------------------------------------------
 * For long contexts: each row reads the n_select pages of its sequence that a cheap score finds best, not all. A step is, after _plan and for each layer,
 *     jepa_amd_cache_append (or _store)       the rows into their slots
 *     jepa_amd_cache_digest                   the digests of the pages that they went to
 *     jepa_amd_cache_select                   which pages each row reads
 *     jepa_amd_cache_attention_selected       attention over these
 * What is said of the cache's calls holds for these too: device pointers, the caller's stream, no allocation, nothing kept, row_start / kv_len / table as
 * jepa_amd_cache_plan gives them. Their workgroups (below) stay under 2^24 in a call; larger ones are refused.
 *
 * A page's digest is, for each K/V head, the largest and the smallest value of each dimension of K over the page's tokens, as 8-bit codes with one f32 scale (s / 127,
 * s the largest magnitude; codes are rounded to nearest; a digest whose s is below 2^-100 is zeros): 2 * head_dim + 16 bytes. Tokens stored as NaN are left out. */

/* Bytes of one page's digests (all K/V heads), or -1. The caller keeps n_pages times this (16-byte aligned) beside each layer's cache; it need not be cleared. */
int64_t jepa_amd_cache_digest_bytes(const jepa_amd_cache_shape * shape);

/* The digests of the pages that the step's rows (those of row_start) lie in, from all their tokens up to kv_len. A page's digest is otherwise kept, so it
 * still holds after tokens were dropped from the page, if not as tightly. Pages that are none of the cache's are passed over. */
int jepa_amd_cache_digest(int device, const jepa_amd_cache_shape * shape, const void * cache, int64_t n_seq, int64_t n_rows, const int32_t * row_start,
                          const int32_t * kv_len, const int32_t * table, int64_t table_width, void * digest, void * stream);

/* The values that the digests of n pages (device, int32) stand for: bounds [n][n_kv_head][2][head_dim] f32 (16-byte aligned), largest first; zeros for a page
 * that is none of the cache's. n * n_kv_head below 2^25. */
int jepa_amd_cache_digest_read(int device, const jepa_amd_cache_shape * shape, const void * digest, const int32_t * page, int64_t n, float * bounds, void * stream);

/* selected [n_rows][n_kv_head][n_select]: for each row and K/V head the pages (places in its sequence's table row) that it is to read, ascending, -1 behind the
 * last. Of the pages that the row sees (causal_block as for jepa_amd_cache_attention) the first n_first and the last n_last (1 or more) are always taken, the
 * others by score, the highest first and of equal ones the lower page; all of them where there are n_select or fewer (1 to 256). A page's score is the sum, over the
 * query heads of the K/V head, of the largest value that the product of the head's query with a key within the page's bounds could have (for a scale above 0). Of the
 * queries it takes the sums over those heads of their positive and of their negative elements, in 8 bits each: whole-number products, so that the choice is the same
 * however a call is split. A row and K/V head score zero everywhere, so that the lowest pages are taken, where these queries have a NaN or an infinity, where one of
 * the sums passes f32's largest value, and where the largest of them is below 2^-100. Pages that are none of the cache's come last. Rows of no
 * sequence are left as they are. `work` is jepa_amd_cache_select_work_bytes() bytes (16-byte aligned, may be NULL where that is 0) under the same terms as
 * jepa_amd_cache_attention's. */
int64_t jepa_amd_cache_select_work_bytes(const jepa_amd_cache_shape * shape, int64_t n_seq, int64_t n_rows, int64_t table_width, int64_t n_select);
int jepa_amd_cache_select(int device, const jepa_amd_cache_shape * shape, const void * digest, int type, const void * q, int64_t q_stride, int64_t n_seq,
                          int64_t n_rows, const int32_t * row_start, const int32_t * kv_len, const int32_t * table, int64_t table_width,
                          int64_t causal_block, int64_t n_first, int64_t n_last, int64_t n_select, int32_t * selected, void * work, int64_t work_bytes,
                          void * stream);

/* jepa_amd_cache_attention over the pages `selected` [n_rows][n_kv_head][n_select] of each row and K/V head, with its accuracy (queries of 16-bit rows to 2^-35
 * of the row's largest element): keys and values enter as they are held, with one exception: in a call of many rows (2048 rows times K/V heads and more, or
 * fewer where a K/V head has more than 16 heads), bf16 rows take values rounded to f16 (2^-11 relative, an eighth of bf16's half step). Entries may come in
 * any order; negative ones, pages past what the row sees and pages that are none of the cache's are passed over, tokens that it does not see are not read, and a
 * page named twice counts twice. `work` as for jepa_amd_cache_select. */
int64_t jepa_amd_cache_selected_work_bytes(const jepa_amd_cache_shape * shape, int64_t n_rows, int64_t n_select);
int jepa_amd_cache_attention_selected(int device, const jepa_amd_cache_shape * shape, const void * cache, int type, const void * q, int64_t q_stride,
                                      int64_t n_seq, int64_t n_rows, const int32_t * row_start, const int32_t * kv_len, const int32_t * table,
                                      int64_t table_width, const int32_t * selected, int64_t n_select, float scale, int64_t causal_block, void * out,
                                      int64_t out_stride, void * work, int64_t work_bytes, void * stream);

/* Force the MFMA GEMM onto workgroup tile `index` for later launches whose n_out it divides; -1
 * restores the automatic choice. Process-wide (tests and tuning). Tiles (weight rows x tokens):
 * 0: 256x128, 1: 192x128, 2: 128x128, 3: 128x128 (other wave shape), 4: 64x128, 5: 128x64, 6: 256x64,
 * 7: 256x64 (other wave shape; only for the q8_K GELU epilogue), 8: 384x64 (4-bit q4_0 only); 9, 64x64 of
 * four waves, runs by the automatic choice alone and is refused here. q4_K
 * weights run tiles 2, 3, 5, 6 and 7, 4-bit q4_0 (rows a multiple of 128) tiles 0, 2, 3, 5, 6, 7 and 8;
 * a tile a launch cannot take leaves that launch on the automatic choice.
 * Returns 0, or -1 for an index past the table. */
int jepa_amd_gemm_tile(int index);
/* The tile (0 to 9 above) a GEMM of this shape takes with the plain f32 epilogue, the residual one or any that
 * does not need 256 features; -1 for f32 weights and types without a GEMM. One row of q8_0 codes has a
 * kernel of its own where no tile or split is forced. No device work. */
int jepa_amd_gemm_tile_of(int wtype, int64_t n_out, int64_t n_in, int64_t n_rows);

#ifdef __cplusplus
}
#endif

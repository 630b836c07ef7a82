/* omni_b200_ops.h — operator-level C ABI: each kernel of the token loop on its
 * own, over caller-owned DEVICE buffers. The reference exposes its kernels as
 * named ops of a manifest (`Gen::launch` / `Gen::gemm_rows`,
 * crates/omni-kern/src/lib.rs:103-224); these entry points are the same ops as
 * plain calls, for parity tests and micro-benchmarks, and the operators around
 * an 8-bit paged cache, for a server's own steps. All tensors are
 * bf16 row-major unless stated; every call is asynchronous on the context's
 * stream and reads what calls in front of it there wrote; `omni_ops_sync` waits
 * and returns the device error word.
 */
#ifndef OMNI_B200_OPS_H
#define OMNI_B200_OPS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct omni_ops omni_ops;

enum omni_gemm_path {
  OMNI_GEMM_AUTO = 0,
  OMNI_GEMM_VECTOR = 1,
  OMNI_GEMM_TENSOR = 2,      /* weights on the MMA M dimension, split-K */
  OMNI_GEMM_TENSOR_ROWS = 3  /* input rows on the MMA M dimension (rows <= 128, K <= 4096), no split */
};
enum omni_epilogue { OMNI_EPI_NONE = 0, OMNI_EPI_BIAS = 1, OMNI_EPI_BIAS_SILU = 2 };

int32_t omni_ops_create(int32_t device, omni_ops** out);
/* Graphs that captured calls of the context hold its error word: they are not replayed any more when it is destroyed. */
void omni_ops_destroy(omni_ops* ctx);
/* Waits for the context's stream; returns 0, OMNI_ERR_CUDA (-2) or, when a
 * kernel raised the device error word, OMNI_ERR_DEVICE (-3) with the word in *word. */
int32_t omni_ops_sync(omni_ops* ctx, uint32_t* word);
/* The stream that the context's calls run on from here: given = 1: `stream`, a cudaStream_t of the context's device (NULL = the
 * default stream), which the caller may be capturing into a graph if the calls made are those of the 8-bit paged cache below;
 * given = 0: the context's own again, as after `omni_ops_create`. Calls on the one are not ordered against calls on the other, but
 * for those that use the context's scratch (`omni_op_gemm` and the chain GEMMs): each waits for the one before it, wherever that
 * ran, and is refused on a stream that is being captured. */
int32_t omni_ops_stream(omni_ops* ctx, int32_t given, void* stream);
/* Device time in ms between the two most recent omni_ops_mark calls (CUDA events on the context's stream). */
int32_t omni_ops_mark(omni_ops* ctx, int32_t which /* 0 = begin, 1 = end */);
int32_t omni_ops_elapsed_ms(omni_ops* ctx, float* ms);
const char* omni_ops_last_error(const omni_ops* ctx);

/* y[rows, N] = x[rows, K] . w[N, K]^T, the `extern:cublaslt_bf16_tn` op of
 * crates/omni-kern/src/lib.rs:159-173, with an optional fused bias epilogue
 * (`talker_bias` / `talker_bias_silu`, talker.cu:45-51). splits = 0 lets the
 * library choose the K split of the tensor-core path. */
int32_t omni_op_gemm(omni_ops* ctx, const void* w, int32_t N, int32_t K, const void* x, int32_t rows, void* y,
                     int32_t ldy, int32_t path, int32_t splits, const void* bias, int32_t epilogue);

/* `qwen3_norm_copy` (crates/omni-qwen3/kernels/qwen3.cu:18-31). */
int32_t omni_op_norm_copy(omni_ops* ctx, const void* x, const void* w, void* out, void* res, int32_t rows,
                          int32_t dim, float eps);
/* `qwen3_add_norm` (qwen3.cu:37-57). */
int32_t omni_op_add_norm(omni_ops* ctx, const void* x, void* res, const void* w, void* out, int32_t rows, int32_t dim,
                         float eps, int32_t every, int32_t which);
/* `qwen3_silu_mul` (qwen3.cu:59-61). */
int32_t omni_op_silu_mul(omni_ops* ctx, const void* gate_up, void* act, int32_t rows, int32_t inter);

/* `qwen3_rope` + `qwen3_attend` (qwen3.cu:109-240) over a paged KV in this
 * library's layout kv[page][kv_head][K|V][16][head_dim]. Row n sits at pos[n],
 * writes slot[n] = page*16 + pos%16, belongs to sequence seq[n] (NULL: row n is
 * sequence n) whose pages are pages[indptr[s]..]. qkv: [rows, (hq+2hk)*d], q is
 * normed and rotated in place; out: [rows, hq*d]. */
int32_t omni_op_rope_attend(omni_ops* ctx, void* qkv, const void* q_norm, const void* k_norm, void* kv,
                            int32_t kv_pages, const int32_t* pos, const int32_t* slot, const int32_t* seq,
                            const int32_t* indptr, const int32_t* pages, int32_t rows, int32_t q_heads,
                            int32_t kv_heads, int32_t head_dim, float eps, float theta, void* out);

/* The same for one row per sequence (decode): normed and rotated, written to
 * the row's slot and attended to in one kernel; qkv is not changed. */
int32_t omni_op_decode_attend(omni_ops* ctx, const void* qkv, const void* q_norm, const void* k_norm, void* kv,
                              int32_t kv_pages, const int32_t* pos, const int32_t* slot, const int32_t* indptr,
                              const int32_t* pages, int32_t rows, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                              float eps, float theta, void* out);

/* The GEMM of the kernel chains, which picks its kernel by the row count:
 * y[rows, N] = x[rows, K] . w[N, K]^T with an optional bias epilogue, or, with
 * `swiglu`, y[rows, N / 2] = bf16(silu(x . gate^T)) * (x . up^T) for
 * w = [gate; up] (regrouped by the call). K a multiple of 64. */
int32_t omni_op_chain_gemm(omni_ops* ctx, const void* w, int32_t N, int32_t K, const void* x, int32_t rows, void* y,
                           int32_t ldy, const void* bias, int32_t epilogue, int32_t swiglu);

/* A projection, the add + norm behind it and the next projection as the chains
 * run them (up to 256 rows): s = x . w1^T [rows, D]; res += s (bf16), h =
 * norm(res) * gain over the unrounded sum (`qwen3_add_norm`, qwen3.cu:37-57);
 * y[rows, N] = h . w2^T. K and D multiples of 64. */
int32_t omni_op_chain_norm_gemm(omni_ops* ctx, const void* w1, int32_t D, int32_t K, const void* x, int32_t rows,
                                void* res, const void* gain, float eps, const void* w2, int32_t N, void* y);

/* The add + norm of the chains by itself: v = res + bf16(sum over `splits` (1, 2, 4 or 8) of part[split][rows][dim], in their
 * order), where `lm` is set rounded to bf16; res = bf16(v); out = norm(v) * gain. All of it at 16-byte addresses. */
int32_t omni_op_add_norm_sum(omni_ops* ctx, const float* part, int32_t splits, void* res, const void* gain, void* out,
                             int32_t rows, int32_t dim, float eps, int32_t lm);

/* `talker_sample` (crates/omni-qwen3-tts/kernels/talker.cu:259-293). state:
 * per-sequence slots of `stride` bytes, each i32 last_frame[16], u32
 * seen[ceil(vocab/32)], then (8-byte aligned) the u64 Philox seed. */
int32_t omni_op_sample(omni_ops* ctx, const void* logits, int32_t vocab, float temperature, int32_t top_k,
                       float top_p, float penalty, int32_t suppress_lo, int32_t suppress_hi, int32_t exempt,
                       int32_t min_frames, const int32_t* frames, const float* uniforms, const int32_t* force,
                       void* state, const int32_t* lines, int64_t stride, int32_t penalize, int32_t philox,
                       int32_t* codes, int32_t group, int32_t rows);

/* ---- duplex (PersonaPlex) kernels, one call each: crates/omni-personaplex/kernels/lm.cu --------------------------
 * Helium KV layout of this library (one buffer per layer, FP8 E4M3 + one f32 scale per (token, head)):
 *   kv[page][head][ K: 16 tokens x 128 B | V: 16 tokens x 128 B | K scales: 16 x f32 | V scales: 16 x f32 ]
 * a token's slot is page * 16 + ring position % 16. */

/* `lm_norm` (lm.cu:86-92) when y is NULL: out = x * (alpha * rsqrt(eps + mean(x^2))).
 * `lm_add_norm` (lm.cu:95-106) otherwise: x = bf16(x + y), out = norm(x); out NULL: `lm_add` (lm.cu:109-120). */
int32_t omni_op_lm_norm(omni_ops* ctx, const void* y, void* x, const void* alpha, void* out, int32_t rows,
                        int32_t dim, float eps);

/* One rank's side of the tensor-parallel pair's exchange (include/omni_b200_duplex.h; no counterpart in the
 * reference): waits (at most 2 s) until the flag word words[0] has reached this exchange's number words[32] + 1, which
 * it also stores to words[16] (in the model: the peer's flag), then y = bf16(mine + peer), x = bf16(x + y),
 * out = norm(x), and the last CTA advances words[32]. words: 64 zero-initialised u32 in device memory
 * (0: this rank's flag, 16: where the peer's flag is written, 32: exchange counter, 48: CTA counter). With a flag that
 * nothing raises the wait runs out: the device error word is set (status OMNI_ERR_DEVICE at the next
 * omni_ops_sync) and peer counts as zero. This entry exists so that the kernel's arithmetic and its bounded wait can
 * be tested on one GPU. */
int32_t omni_op_lm_tp_add_norm(omni_ops* ctx, const void* mine, const void* peer, void* x, const void* alpha, void* out,
                               int32_t rows, int32_t dim, float eps, void* words);

/* `lm_embed_prompt` (lm.cu:47-59) without voices: out[r] = sum of the embeddings of ids[r][0..17), every add rounded
 * to bf16, audio streams first, -1 = no token. text_emb [text_rows, dim], audio_emb [16 * card_rows, dim]. */
int32_t omni_op_lm_embed(omni_ops* ctx, const int32_t* ids, const void* text_emb, int32_t text_rows,
                         const void* audio_emb, int32_t card_rows, void* out, int32_t rows, int32_t dim);

/* `lm_rope` + `lm_attend` (lm.cu:129-290): rows of [q | k | v] (heads of 128): interleaved rotary embedding, K and V
 * quantised to E4M3 into slot[n], attention of row n (session seq[n], or n when seq is NULL) over the first
 * min(pos[n] + 1, context) ring positions of its pages. q is rotated in place. */
int32_t omni_op_lm_rope_attend(omni_ops* ctx, void* qkv, void* kv, int32_t kv_pages, const int32_t* pos,
                               const int32_t* slot, const int32_t* seq, const int32_t* indptr, const int32_t* pages,
                               int32_t rows, int32_t heads, float coef, float scale, int32_t context, void* out);

/* The same for one row per session (decode) in one kernel; qkv is not changed. */
int32_t omni_op_lm_decode_attend(omni_ops* ctx, const void* qkv, void* kv, int32_t kv_pages, const int32_t* pos,
                                 const int32_t* slot, const int32_t* indptr, const int32_t* pages, int32_t rows,
                                 int32_t heads, float coef, float scale, int32_t context, void* out);

/* `lm_dep_embed_norm` (lm.cu:301-313) then `lm_dep_kv_attend` is a separate call below.
 * x = bf16(projected[s][k] + table[drawn[s][k]]), xn = norm(x). */
int32_t omni_op_lm_dep_embed_norm(omni_ops* ctx, const void* projected, int32_t k, const void* table,
                                  int32_t table_rows, const int32_t* drawn, const void* alpha, void* x, void* xn,
                                  int32_t rows, int32_t dim, float eps);

/* `lm_dep_kv_attend` (lm.cu:319-366): step's K and V into ws ([rows][8][K | V][heads * 64]), causal attention over
 * steps 0..step. */
int32_t omni_op_lm_dep_kv_attend(omni_ops* ctx, const void* qkv, void* ws, int32_t step, void* out, int32_t rows,
                                 int32_t heads, float scale);

/* `lm_sample` (lm.cu:423-537): Gumbel-max over the top-k into drawn[s][col]; force[s][col] >= 0 is taken. */
int32_t omni_op_lm_sample(omni_ops* ctx, const void* logits, int32_t vocab, int64_t ld, float temperature,
                          int32_t top_k, const int32_t* force, const int32_t* seeds, int32_t col, int32_t* drawn,
                          int32_t rows);

/* `lm_init` (lm.cu:576-581) when init is not NULL, then `lm_advance` (lm.cu:546-573) when drawn is not NULL. */
int32_t omni_op_lm_advance(omni_ops* ctx, void* state, const int32_t* lines, int64_t stride, const int32_t* init,
                           const int32_t* drawn, const int32_t* caller, const int32_t* force_caller,
                           int32_t* emitted, int32_t rows);

/* ---- Higgs-style speech model glue: crates/omni-higgs-audio/kernels/higgs.cu, src/delay.rs ---------------------- */

/* `higgs_frame_embed` (higgs.cu:24-37): out[s] = bf16(f32 sum over the 8 codebooks of table[b * vocab + code_b]),
 * codes = the first 8 words of the sequence's state slot (state + lines[s] * stride). */
int32_t omni_op_higgs_frame_embed(omni_ops* ctx, void* state, const int32_t* lines, int64_t stride, const void* table,
                                  void* out, int32_t rows, int32_t dim, int32_t vocab);

/* `higgs_sample` (higgs.cu:186-208): eight independent draws per row over logits [rows, 8, vocab] against
 * uniforms [rows, 8]; force [rows, 8] >= 0 is taken (the delay pattern arrives here); codes [rows, 8] and the slot. */
int32_t omni_op_higgs_sample(omni_ops* ctx, const void* logits, int32_t vocab, float temperature, int32_t top_k,
                             const float* uniforms, const int32_t* force, void* state, const int32_t* lines,
                             int64_t stride, int32_t* codes, int32_t rows);

/* `Delay` (crates/omni-higgs-audio/src/delay.rs:19-46), host only: which codebooks the next step does not draw (they
 * read OMNI_HIGGS_BOC) and when generation ends. Zero-initialise for a new run. */
#define OMNI_HIGGS_BOOKS 8
#define OMNI_HIGGS_BOC 1024
#define OMNI_HIGGS_EOC 1025
typedef struct omni_higgs_delay {
  int32_t steps;
  int32_t countdown; /* 0: none running; otherwise steps left + 1 */
  int32_t done;
} omni_higgs_delay;
/* `Delay::forced_from` (delay.rs:27-29): the first codebook the next step does not draw. */
int32_t omni_higgs_delay_forced_from(const omni_higgs_delay* d);
/* `Delay::advance` (delay.rs:33-46): takes the step's codebook 0 draw; 1 when generation has ended. */
int32_t omni_higgs_delay_advance(omni_higgs_delay* d, int32_t first);
/* `undelay` (delay.rs:50-54): frames [max(n_rows - 7, 0), 8] from delayed rows [n_rows, 8]; returns the frame count. */
int32_t omni_higgs_undelay(const int32_t* rows, int32_t n_rows, int32_t* frames);

/* The tensor-core GEMM of omni_op_gemm for callers that cannot allocate device memory. It has no counterpart in the
 * reference. Two kinds of caller are meant: a serving process that handed every free byte of HBM to its KV pool at
 * start-up, where a later cudaMalloc simply fails; and an engine thread in the middle of a live tick, where
 * cudaMalloc / cudaFree would synchronise the whole device and stall every other session's stream. This entry
 * point needs no context object and calls no cudaMalloc, cudaFree or allocating library routine: the split-K
 * scratch (f32 partial tiles, tile counters, the error word) is a fixed array inside the library image, present on
 * every GPU that loads the library for as long as the process lives.
 *
 *  - Inputs and outputs are the caller's device buffers, as for omni_op_gemm (tensor-core path only: K a
 *    multiple of 64, operands 16-byte aligned). `stream` is a cudaStream_t (NULL = the default stream).
 *  - Limits: splits * row_tiles * ceil(N/128) * 128 * BN <= 4 Mi floats (BN = rows rounded up to 16/32/64/128/256)
 *    and row_tiles * ceil(N/128) <= 2048. Larger problems are refused with OMNI_ERR_UNSUPPORTED and a message
 *    naming the sizes; nothing is launched.
 *  - The first call on each device looks up the arrays' device addresses (with that device current) and raises the
 *    kernels' shared-memory limits. Make that first call before starting any stream capture on that device.
 *  - All calls share the one array and it keeps the previous call's contents; the counters and the error word are
 *    cleared on the stream before each launch. Two calls whose kernels overlapped on the GPU would race on it, so
 *    the entry point holds a process-wide lock from its set-up until its kernel has finished: calls from several
 *    host threads run one after the other. `stream` must belong to the current device (checked).
 *  - The call waits for its kernel and returns 0, or a negative omni_status with a human-readable reason in
 *    `message` (caller-owned, may be NULL). */
int32_t omni_op_gemm_noalloc(const void* w, int32_t N, int32_t K, const void* x, int32_t rows, void* y, int32_t ldy,
                             int32_t splits, const void* bias, int32_t epilogue, void* stream, char* message,
                             size_t message_len);

/* ---- 8-bit paged cache -----------------------------------------------------------------------------------------------
 * The operators of a grouped-head stack that keeps its KV in 8 bits. They have no counterpart in the reference, whose KV is
 * bf16 (crates/omni-qwen3/kernels/qwen3.cu:109-240). One decoder layer of a call:
 *   omni_op_kv_tables      lengths -> page tables, positions and slots of the call's rows (once for all layers)
 *   omni_op_qk_norm_rope   norm and rotary embedding of the rows' q and k
 *   omni_op_packed_attend  whole prompts: causal attention over the call's own rows
 *   omni_op_kv8_append     the rows' K and V into the pages
 *   omni_op_kv8_attend     one row a sequence: attention over the pages
 * Cache of a layer: kv[page][kv_head][K | V][16][head_dim] in E4M3 and scales[page][kv_head][K | V] in f32; an element is its
 * code times its scale. Heads of 64 or 128. Rows of bf16 are given with a stride in elements (ld), a multiple of 8, so that parts
 * of wider rows can be passed; base addresses are multiples of 16 bytes (scales: 8). Zero rows are a call that does nothing.
 * No call waits for the device or keeps anything for the next, and each has what memory it needs to itself (of these only
 * omni_op_kv8_attend over few long rows, which takes it from the stream's order): calls may be captured, and graphs and streams
 * may run side by side, a context's calls being made by one thread at a time.
 * What device arrays hold (lengths, positions, slots, pages) the host does not see; where the kernels find an index outside
 * its table they skip it and raise the device error word. */

/* Page tables of n sequences (4096 at most). lens[i]: tokens that sequence i holds; add[i]: tokens that this call appends (0 and
 * more), or -1: the sequence has ended and its pages come back. table[i][width]: its pages, in order. free_pages[0 .. *free_count):
 * a stack of free pages with room for free_cap. Pages of ended sequences are laid on top of it in the sequences' order; then, in
 * the sequences' order, each page that is wanted is taken from its top and entered into the table.
 *   lens_out[n], *free_count_out   the new lengths (0 for ended sequences) and height; may be lens and free_count themselves
 *   indptr[n + 1], pages           the tables packed: sequence i has pages[indptr[i] .. indptr[i + 1]); room for page_cap
 *   row_ptr[n + 1], pos, slot, seq the call's rows, sequence by sequence: position, slot (page * 16 + pos % 16) and sequence of
 *                                  each; room for row_cap, of which the rows behind the last hold -1
 *   *status                        0; otherwise nothing was changed (lens_out and *free_count_out say what lens and *free_count
 *                                  do, pages is untouched, indptr and row_ptr are 0, pos, slot and seq are -1) and it is a sum of
 *                                  OMNI_TABLES_*. A server's ordinary answer to BUSY is to try again with fewer sequences.
 * No array may overlap another one but for the two that are named. */
enum omni_tables_status {
  OMNI_TABLES_LENGTH = 1,  /* a length below 0, an addition below -1, or more tokens than a table's width holds */
  OMNI_TABLES_BUSY = 2,    /* fewer pages free than wanted */
  OMNI_TABLES_ROWS = 4,    /* more rows than row_cap */
  OMNI_TABLES_PAGES = 8,   /* more pages than page_cap */
  OMNI_TABLES_FREE = 16    /* *free_count below 0 or above free_cap, or more pages come back than free_cap holds */
};
int32_t omni_op_kv_tables(omni_ops* ctx, const int32_t* lens, const int32_t* add, int32_t n, int32_t* table, int32_t width,
                          int32_t* free_pages, int32_t free_cap, const int32_t* free_count, int32_t* lens_out,
                          int32_t* free_count_out, int32_t* indptr, int32_t* pages, int32_t page_cap, int32_t* row_ptr,
                          int32_t* pos, int32_t* slot, int32_t* seq, int32_t row_cap, int32_t* status);

/* The first q_heads + kv_heads heads of every row of x with pos >= 0, normed (x / sqrt(mean x^2 + eps) * gain, q_norm for the
 * q heads, k_norm for the k heads; NULL: no norm) and rotated: elements i and i + head_dim / 2 by pos * theta^(-2 i / head_dim).
 * Computed in f32 from an angle in f64 and rounded once (the attention calls above round between the steps as the reference
 * does). Other rows of out stay as they are. out may be x, with the same stride if there is more than one row, and must not overlap it
 * otherwise. */
int32_t omni_op_qk_norm_rope(omni_ops* ctx, const void* x, int64_t ldx, const void* q_norm, const void* k_norm,
                             const int32_t* pos, int32_t rows, int32_t q_heads, int32_t kv_heads, int32_t head_dim,
                             float eps, float theta, void* out, int64_t ldo);

/* Causal attention within each of n packed sequences (16,384 at most): rows indptr[i] .. indptr[i + 1] of q, k and v, of which row r sees the
 * sequence's rows up to itself: out[r][h] = softmax(scale * q[r][h] . K) V, h over q_heads and K, V those of kv head
 * h / (q_heads / kv_heads). scale > 0. Scores and sums are f32; the weights are rounded to bf16, by 2^-8 of each at most, before they
 * meet V (`omni_op_rope_attend` spends more bits there). indptr ascends from any row on; sequences may be empty. Rows outside of the sequences stay
 * as they are in out, and nothing of them, of other sequences or of later rows reaches a row, not even as a NaN. out must not
 * overlap q, k or v. The kernel's waits end by themselves after 0.4 s, which a sequence of some ten million rows may need for one
 * tile: the device error word tells. */
int32_t omni_op_packed_attend(omni_ops* ctx, const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v,
                              int64_t ldv, const int32_t* indptr, int32_t n, int32_t rows, int32_t q_heads,
                              int32_t kv_heads, int32_t head_dim, float scale, void* out, int64_t ldo);

/* K and V of every row with slot >= 0 into the cache. A page's scale (one for K, one for V of each head) is the smallest 2^e with
 * e >= -100 and |x| <= 448 * 2^e for every finite x put into it. A row at a page's first token starts the page anew; rows further in
 * come behind tokens that the page holds, whose scale then only grows, and whose codes are rounded again when it does. Codes
 * are the nearest, ties to even; infinities become +-448 * 2^e, a NaN stays one. Rows of one page are neighbours in the call, in
 * ascending slots without a gap, as omni_op_kv_tables lays them: a row that is on the page of the row in front of it but not its
 * next token is left out and raises the device error word (those behind it on that page may be left out too), and a page that
 * occurs in two places further apart is written in an undefined order. */
int32_t omni_op_kv8_append(omni_ops* ctx, const void* k, int64_t ldk, const void* v, int64_t ldv, const int32_t* slot,
                           int32_t rows, void* kv, float* scales, int32_t kv_pages, int32_t kv_heads, int32_t head_dim);

/* out[n][h] = softmax(scale * q[n][h] . K) V over tokens 0 .. pos[n] of sequence seq[n] (NULL: sequence n) of n_seqs, whose pages
 * are pages[indptr[s] .. indptr[s + 1]) out of n_pages. Rows with pos < 0 become zeros. What a page holds behind the row's
 * last token is not looked at. Scales may be any numbers >= 0 here. A row whose sequence, range or number of pages is wrong becomes
 * zeros; a page outside the cache is left out. Weights (times their page's V scale) are rounded to f16 on the way to V: by 2^-11 of
 * each or 2^-16 of its page's largest, whichever is more, and pages whose largest lies below 2^-60 of the row's may lose more. The host
 * takes n_pages / n_seqs for the rows' length when it cuts the work: the answer does not depend on it, the time does where `pages` has
 * much more room than the sequences have pages. */
int32_t omni_op_kv8_attend(omni_ops* ctx, const void* q, int64_t ldq, const void* kv, const float* scales, int32_t kv_pages,
                           const int32_t* pos, const int32_t* seq, const int32_t* indptr, int32_t n_seqs,
                           const int32_t* pages, int32_t n_pages, int32_t rows, int32_t q_heads, int32_t kv_heads,
                           int32_t head_dim, float scale, void* out, int64_t ldo);

/* ---- streaming codec decoder: crates/omni-qwen3-tts/kernels/codec.cu, src/codec.rs -------------------------------
 * A per-stream state is `state + lines[s] * stride` bytes plus the entry's own byte offset; `pos[s]` is the number of
 * frames stream s has decoded before the call (histories are two halves, frame p reads half p & 1 and writes the
 * other). Channel counts are multiples of 8. */

/* `codec_rvq` (codec.cu:66-82): out[s] = [book 0 row codes[s][0] | bf16(f32 sum of books 1..15 rows)], books
 * [16 * book_rows, half]; a codebook-0 code >= book_rows reads as 0. */
int32_t omni_op_codec_rvq(omni_ops* ctx, const int32_t* codes, const void* books, void* out, int32_t n, int32_t half,
                          int32_t book_rows);
/* `codec_add_rms_norm` / `codec_bias_rms_norm` (codec.cu:117-170): v = res + add (add_stride 0: one row for all);
 * res = bf16(v); out = bf16(v * (rsqrt(mean v^2 + eps) * w)); out may be add. dim a multiple of 256 up to 1024. */
int32_t omni_op_codec_add_norm(omni_ops* ctx, const void* add, int64_t add_stride, void* res, const void* w, void* out,
                               int32_t rows, int32_t dim, float eps);
/* `codec_attention` (codec.cu:177-283): rotary embedding of q and k, k and v into the stream's ring
 * (K[72][heads * 64] then V, frame p at p % 72), q against the last min(p + 1, 72) frames. qkv [n, 3 * heads * 64]. */
int32_t omni_op_codec_window_attend(omni_ops* ctx, const void* qkv, void* state, const int32_t* lines, const int32_t* pos,
                                    int64_t stride, int64_t ring_offset, void* out, int32_t n, int32_t heads, float theta);
/* `codec_bias_gelu` (codec.cu:84-98), in place; `codec_bias_snake` (codec.cu:100-109). */
int32_t omni_op_codec_bias_gelu(omni_ops* ctx, void* x, const void* bias, int64_t rows, int32_t cols);
int32_t omni_op_codec_bias_snake(omni_ops* ctx, const void* x, const void* bias, const float* alpha, const float* inv_b,
                                 void* out, int64_t rows, int32_t cols);
/* The input side of `codec_im2col` / `codec_im2col_snake` (codec.cu:291-337) without the im2col matrix:
 * padded[s][r] = r < H ? history row r : bf16(act(x[s * T + r - H] + bias)), act SnakeBeta when alpha is given; the last
 * H rows become the next frame's history. `gather_taps` then writes the reference's matrix from it:
 * col[s * T + t][j * C + c] = padded[s][t + j * dil][c]. */
int32_t omni_op_codec_stage(omni_ops* ctx, const void* x, const void* bias, const float* alpha, const float* inv_b,
                            void* state, const int32_t* lines, const int32_t* pos, int64_t stride, int64_t hist_offset,
                            void* padded, int32_t n, int32_t T, int32_t C, int32_t H);
int32_t omni_op_codec_gather_taps(omni_ops* ctx, const void* padded, void* col, int32_t n, int32_t T, int32_t C,
                                  int32_t taps, int32_t dil);
/* The conv itself as an implicit GEMM on tcgen05 (what `codec_im2col` + the runtime's GEMM compute, codec.rs:60-93):
 * y[s * T + t][n] (+)= sum over taps j, channels c of padded[s][t + j * dil][c] * w[n][j * C + c]; epilogue 0: store,
 * 1: y = bf16(y + a), 2: y = bf16(snake(bf16(a) + bias[n])). taps = 1: padded is the dense [n_streams * T, C] input. */
int32_t omni_op_codec_conv(omni_ops* ctx, const void* w, int32_t N, int32_t C, int32_t taps, int32_t dil,
                           const void* padded, int32_t T, int32_t n_streams, void* y, int32_t epilogue, const void* bias,
                           const float* alpha, const float* inv_b);
/* `codec_col2im` (codec.cu:339-372): transposed conv with kernel 2r, stride r, over z [n, L, 2r * C]. */
int32_t omni_op_codec_overlap_add(omni_ops* ctx, const void* z, const void* bias, void* state, const int32_t* lines,
                                  const int32_t* pos, int64_t stride, int64_t prev_offset, void* out, int32_t n, int32_t L,
                                  int32_t r, int32_t C);
/* `codec_dwconv_ln` (codec.cu:381-446): xin = bf16(z + zb[row % r]); depthwise 7-tap causal conv; LayerNorm -> out. */
int32_t omni_op_codec_dwconv_ln(omni_ops* ctx, const void* z, const void* zb, const void* w, const void* b,
                                const void* ln_w, const void* ln_b, void* state, const int32_t* lines, const int32_t* pos,
                                int64_t stride, int64_t hist_offset, void* xin, void* out, int32_t n, int32_t T, int32_t r,
                                int32_t C, float eps);
/* `codec_conv_out` (codec.cu:455-513): last SnakeBeta, the C -> 1 conv of 7 taps, the clamp; wav f32 [n][T] (the
 * reference stores the same values as bf16). T a multiple of 64, C a multiple of 32 up to 128. */
int32_t omni_op_codec_out_conv(omni_ops* ctx, const void* x, const void* bias, const float* alpha, const float* inv_b,
                               const void* w, const void* wb, void* state, const int32_t* lines, const int32_t* pos,
                               int64_t stride, int64_t hist_offset, float* wav, int32_t n, int32_t T, int32_t C);

#ifdef __cplusplus
}
#endif
#endif /* OMNI_B200_OPS_H */

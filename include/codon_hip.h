/*
 * codon_hip.h — C ABI of the MI355X (gfx950) ESM-2 bidirectional encoder.
 *
 * A drop-in for the GPU side of codon-infer's forward_bidirectional* family.
 * Plain C types only: pointers, sizes, int status codes.  Every entry point
 * returns 0 (CIH_OK) or a negative cih_status; on failure
 * cih_last_error() (thread-local) describes the problem.  Nothing aborts or
 * throws across the ABI.
 *
 * Reference interfaces each entry replaces are cited as file:line into
 * OsbaldoG/codon-infer.
 */
#ifndef CODON_HIP_H
#define CODON_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define CIH_ABI_VERSION 1

/* ---- status codes --------------------------------------------------- */
enum cih_status {
    CIH_OK = 0,
    CIH_ERR_ARG = -1,        /* null pointer / invalid argument            */
    CIH_ERR_SHAPE = -2,      /* unsupported or inconsistent shape          */
    CIH_ERR_CAPACITY = -3,   /* batch/length above cih_model_reserve's     */
    CIH_ERR_CONTACTS = -4,   /* contacts requested with n_res > 1024       */
    CIH_ERR_HIP = -5,        /* HIP runtime error (no device, OOM, ...)    */
    CIH_ERR_IO = -6,         /* file open/read failure                     */
    CIH_ERR_FORMAT = -7,     /* bad magic/version/dtype/size in a file     */
    CIH_ERR_TOKEN = -8       /* token id outside [0, vocab)                */
};

/* ---- weight formats: the CODQ dtype ids (lib.rs:873-876) -------------- */
enum cih_dtype { CIH_DTYPE_FP32 = 0, CIH_DTYPE_Q8_0 = 1, CIH_DTYPE_Q4_0 = 2 };

#define CIH_Q8_0_BLOCK_BYTES 36 /* BlockQ8_0 {f32 d; i8 qs[32]}, lib.rs:640-645  */
#define CIH_Q4_0_BLOCK_BYTES 20 /* BlockQ4_0 {f32 d; u8 qs[16]}, lib.rs:1043-1050 */

/* EsmConfig (lib.rs:76-84).  head_dim = dim / n_heads must be one of
 * 16, 24, 32, 64; dim and hidden_dim must be multiples of 32. */
typedef struct cih_config {
    int32_t dim;
    int32_t hidden_dim;
    int32_t n_layers;
    int32_t n_heads;
    int32_t vocab_size;
    int32_t max_seq_len;
} cih_config;

/* Host tensors in EsmWeights / EsmWeightsQ8 / EsmWeightsQ4 field order
 * (lib.rs:299-307, 675-687, 1113-1125).  Layer tensors are stacked
 * tensor-major; matrices are [out][in].  Quantized matrices point at packed
 * 36-byte (Q8_0) / 20-byte (Q4_0) blocks.  token_embedding_table is Q8_0
 * blocks for Q8_0 models and FP32 otherwise.  classifier_weights is
 * [lm_ln_w, lm_ln_b, dense_w, dense_b, dec_w, dec_b] (lib.rs:5389-5396); a
 * shorter classifier selects the tied-embedding decoder (lib.rs:5427-5439).
 * The library copies everything to the device; the caller keeps ownership. */
typedef struct cih_host_weights {
    const void *token_embedding_table;
    const float *ln_1_weight, *ln_1_bias;
    const void *wq; const float *bq;
    const void *wk; const float *bk;
    const void *wv; const float *bv;
    const void *wo; const float *bo;
    const float *ln_2_weight, *ln_2_bias;
    const void *fc1_weight; const float *fc1_bias;
    const void *fc2_weight; const float *fc2_bias;
    const float *ln_f_weight, *ln_f_bias;
    const float *classifier_weights;
    int64_t classifier_len;
} cih_host_weights;

typedef struct cih_model cih_model;

/* ---- forward flags ---------------------------------------------------- */
#define CIH_OUT_LOGITS       (1u << 0) /* logits       [B][S_max][V]               */
#define CIH_OUT_HIDDEN       (1u << 1) /* hidden       [B][S_max][d] (after LN_f)   */
#define CIH_OUT_FINAL_ATT    (1u << 2) /* final_att    [B][S_max][S_max]            */
#define CIH_OUT_CONTACTS     (1u << 3) /* contacts     [B][S_max-2][S_max-2]        */
#define CIH_OUT_ATTN         (1u << 4) /* attn         [B][L][H][S_max][S_max]      */
#define CIH_OUT_LAYER_HIDDEN (1u << 5) /* layer_hidden [B][L][S_max][d]             */
#define CIH_IO_DEVICE        (1u << 16) /* tokens + outputs are device pointers     */

/* Caller-owned output buffers, all row-major with the padded strides above.
 * Only rows/cols inside each sequence's true length are written; padding is
 * left untouched.  NULL entries are allowed when their flag is off. */
typedef struct cih_outputs {
    float *logits;
    float *hidden;
    float *final_att;
    float *contacts;
    float *attn;
    float *layer_hidden;
} cih_outputs;

/* ---- lifecycle ---------------------------------------------------------- */

/* Replaces EsmWeights/EsmWeightsQ8/EsmWeightsQ4 construction +
 * BidirectionalRunState ownership (lib.rs:310, 744, 1156, 2510).
 * contact_w: [n_layers*n_heads] regression weights (l-major) and contact_b
 * its bias, as returned by EsmConfig::contact_head_weights (lib.rs:154-177);
 * contact_w may be NULL when contacts are never requested.
 * Uses the current HIP device; creates one HIP stream per model.
 * Device memory: the weights in their own format, plus, for Q8_0 / Q4_0
 * models, the layer quants once more as f16 integers (2 bytes per weight:
 * the operand of the large-batch GEMM); CIH_GEMM_F16=0 leaves that copy out. */
int cih_model_create(const cih_config *cfg, int32_t dtype, const cih_host_weights *w,
                     const float *contact_w, float contact_b, cih_model **out);

/* Replaces load_model_weights (main.rs:137-244) + EsmConfig::detect_from_file
 * (lib.rs:277-296): reads a CODQ (FP32/Q8_0/Q4_0) or headerless
 * grouped_canonical_v1 / sequential_hf FP32 file.  quantize_to: -1 keeps the
 * file's dtype; CIH_DTYPE_Q8_0 / CIH_DTYPE_Q4_0 quantize an FP32 file in
 * memory (lib.rs:559-607).  Contact weights as in cih_model_create.
 * The file body goes to the GPU as is (parallel reads into pinned staging
 * buffers, asynchronous copies); the repack and any quantization run there.
 * CIH_LOAD_THREADS / CIH_LOAD_CHUNK_MB size the staging (default 2 x 8 MiB). */
int cih_model_create_from_file(const char *path, int32_t quantize_to, const float *contact_w,
                               float contact_b, cih_model **out);

/* Sizes the per-model device workspace (BidirectionalRunState::new max_len,
 * lib.rs:2510).  Output kinds not named in flags cannot be requested later
 * without another reserve.  cih_forward never allocates. */
int cih_model_reserve(cih_model *m, int32_t max_batch, int32_t max_seq_len, uint32_t flags);

int cih_model_config(const cih_model *m, cih_config *cfg, int32_t *dtype);
int cih_model_destroy(cih_model *m);

/* ---- the forward -------------------------------------------------------- */

/* Replaces forward_bidirectional / _parallel / _parallel_ext (lib.rs:5078,
 * 5087, 5097), forward_bidirectional_q8 (5442) and forward_bidirectional_q4 /
 * _q4_ext (5790, 5800) for a batch of B independent sequences.
 * tokens: [B][S_max] int32 ids (padding ignored), lens: [B] host array with
 * 1 <= lens[b] <= S_max.  B=1, lens[0]=S equals one reference call on
 * tokens[0..S].  Synchronous: outputs are complete on return.
 * Token ids outside [0, vocab) return CIH_ERR_TOKEN: checked on the host, or
 * with CIH_IO_DEVICE on the device during the forward (the outputs are then
 * undefined).
 * Range: the default kernels hand activations to the GEMMs and to attention
 * as two f16 limbs, which hold |x| < 65520 only.  A forward whose residual
 * stream turns non-finite, or whose final or LM-head LayerNorm writes a value
 * of 65520 or more in magnitude (the input of the LM head's limb GEMMs), is
 * run once more with the full-range kernels (three bf16 limbs, FP32-MFMA
 * attention and FP32-MFMA LM head, the whole FP32 exponent range), and those
 * results are returned.  Covered: an overflow inside a layer (it reaches the
 * residual stream) and at the LM head's inputs. */
int cih_forward(cih_model *m, const int32_t *tokens, const int32_t *lens, int32_t B,
                int32_t S_max, uint32_t flags, const cih_outputs *out);

/* ---- autoregressive decoding --------------------------------------------- */

typedef struct cih_decoder cih_decoder;

/* Replaces RunState::new (lib.rs:2464-2486) for n_slots independent
 * sequences: a K and a V cache of [n_layers][n_slots][max_len][dim] floats
 * on the device, RoPE tables for max_len positions, and row buffers for up
 * to max_rows rows per cih_decode call.  max_len <= 15000. */
int cih_decoder_create(cih_model *m, int32_t n_slots, int32_t max_len, int32_t max_rows,
                       cih_decoder **out);
int cih_decoder_destroy(cih_decoder *d);
/* Forgets a slot's cache contents (slot < 0: every slot). */
int cih_decoder_reset(cih_decoder *d, int32_t slot);

/* Replaces forward / forward_parallel / forward_q8 / forward_q4
 * (lib.rs:3554, 3558, 3741, 4016) for n rows at once: row i feeds
 * tokens[i] at position pos[i] of slot slots[i] (its K and V are written to
 * the cache there, then it attends to the slot's positions 0..pos[i]).
 * The rows of one slot must be consecutive positions starting at most at the
 * slot's first unwritten position (a prompt can prefill in one call;
 * rewriting earlier positions is allowed, as in the reference).  logits:
 * host [n][vocab] (may be NULL).  Synchronous. */
int cih_decode(cih_decoder *d, const int32_t *slots, const int32_t *tokens, const int32_t *pos,
               int32_t n, float *logits);

/* Replaces generate_sequence / _parallel / _q8 / _q4 (lib.rs:6538-6827) for
 * n independent streams.  Stream i uses slot slots[i] and the prompt ids
 * prompts[offsets[i] .. offsets[i+1]) (Tokenizer::encode of the prompt
 * without its trailing <eos>, as the reference feeds it), its own SimpleRng
 * seed seeds[i], a shared temperature (<= 0: greedy) and max_new_tokens
 * (< 0: none).  max_seq_len (<= 0: the decoder's max_len) caps positions as
 * config.max_seq_len does.  Each stream's prompt is prefilled in its own
 * calls; then all live streams decode together, one token each per step, each
 * stopping at <eos> (2) or its limit.  out_tokens: [n][out_cap] generated
 * ids; n_generated[i] their counts; prefill_ms / generation_ms (may be NULL)
 * the wall times of the two phases.  A stream's tokens do not depend on the
 * other streams while at most 8 streams decode together. */
int cih_generate(cih_decoder *d, int32_t n, const int32_t *slots, const int32_t *prompts,
                 const int32_t *offsets, float temperature, int32_t max_new_tokens,
                 const uint64_t *seeds, int32_t max_seq_len, int32_t *out_tokens, int32_t out_cap,
                 int32_t *n_generated, double *prefill_ms, double *generation_ms);

/* ---- in-silico deep mutational scan -------------------------------------- */

enum cih_dms_mode { CIH_DMS_MASKED_MARGINAL = 0, CIH_DMS_WILDTYPE_MARGINAL = 1 };

/* Replaces run_pipeline_dms_with_mode (pipeline.rs:76-280) for one protein.
 * residues: the n token ids between BOS and EOS (Tokenizer::encode of the
 * sequence without its first and last entries).  window / stride as the
 * reference (0 = the whole protein, capped at the model's max_seq_len).
 * Masked marginal: one forward per position with that position set to
 * <mask> (32), run as batches of `chunk` masked copies (0 or > reserved
 * max_batch = max_batch); wild-type marginal: one unmasked forward per
 * window.  Scoring (canonical log-softmax, entropy, deltas) runs on the GPU;
 * outputs are host arrays: deltas [n][20] in CANONICAL_AAS order
 * (A C D E F G H I K L M N P Q R S T V W Y, benchmark.rs:702-707; exactly 0
 * in the wild-type column) and entropy [n].  Needs a workspace reserved for
 * max_seq_len >= window + 2; allocates nothing. */
int cih_dms(cih_model *m, const int32_t *residues, int32_t n, int32_t window, int32_t stride, int32_t mode,
            int32_t chunk, float *deltas, float *entropy);

/* ---- 8-bit paged key/value cache -------------------------------------------
 * No counterpart in the reference, whose RunState keeps K and V in FP32
 * (lib.rs:2464-2486).  Keys and values are held as 8-bit codes with one FP32
 * scale for each page of CIH_KV8_PAGE tokens, head, and K or V: value = code *
 * scale, codes -127..127.  A sequence's tokens live in the pages that its row
 * of a page table names, in order: token p in page table[p / 64] at p % 64.
 *
 * Every pointer in the structures below is a DEVICE pointer on the current
 * device; calls are enqueued on `stream` (a hipStream_t of that device; NULL =
 * the null stream), return without waiting, allocate nothing and keep nothing
 * between calls, so that they may be captured into a graph.  Sizes on the host
 * (n_seq, n_rows, max_rows, max_pages) fix the grids; row offsets, lengths and
 * tables are read on the device when the kernels run.  A call whose grid would
 * pass 2^24 workgroups (n_seq * kv_heads * the pages of 64, or the tiles of 16 rows
 * times q_heads / kv_heads, that max_rows make) returns CIH_ERR_HIP. */

enum cih_float { CIH_F32 = 0, CIH_F16 = 1, CIH_BF16 = 2 };

#define CIH_KV8_PAGE 64

/* head_dim is 16, 24, 32, 64 or 128; dims = head_dim, but 32 for 24.  k and v
 * 16-byte aligned, bad and scales 8-byte.  The memory need not be initialised:
 * a page's first append writes its scales, and codes of tokens past a
 * sequence's length are never used.  bad bit t: token t of the page had a
 * value that is not finite in K or V of that head (its codes are 0 and it
 * reads as NaN). */
typedef struct cih_kv8_cache {
    void *k;        /* int8 [n_pages][kv_heads][64][dims]  */
    void *v;        /* int8 [n_pages][kv_heads][dims][64]  */
    float *scales;  /* [n_pages][kv_heads][2]: of K, of V  */
    uint64_t *bad;  /* [n_pages][kv_heads]                 */
    int32_t n_pages, kv_heads, head_dim;
} cih_kv8_cache;

/* n_seq sequences with rows cu_rows[i] .. cu_rows[i + 1] of the row tensors
 * (at most max_rows each; rows from n_rows on are never touched).  lens[i]:
 * tokens the sequence holds including these rows, which are its last ones: its
 * row r has position lens[i] - rows + r.  Sequence i uses row slots[i] (NULL:
 * i) of the page table, which has table_rows rows of max_pages page ids,
 * table_stride apart.  Tokens past max_pages * 64, and tokens whose page id is
 * outside [0, n_pages) or whose slot is outside [0, table_rows), are treated
 * as not there; rows at negative positions see nothing and are not stored. */
typedef struct cih_kv8_batch {
    const int32_t *cu_rows; /* [n_seq + 1] */
    const int32_t *lens;    /* [n_seq]     */
    const int32_t *table;   /* [table_rows][table_stride] */
    const int32_t *slots;   /* [n_seq] or NULL */
    int32_t n_seq, n_rows, max_rows;
    int32_t table_rows, table_stride, max_pages;
} cih_kv8_batch;

/* Rows of heads: element (row, head, dim) at data[row * row_stride + head *
 * head_stride + dim] (strides in elements; the data aligned to its type). */
typedef struct cih_rows {
    void *data;
    int64_t row_stride, head_stride;
} cih_rows;

/* Rotary positions: pair j < rot_dim / 2 of a head turns by position * freq[j]
 * radians, both values times gain.  The pair is (j, j + rot_dim / 2), or with
 * interleaved (2 j, 2 j + 1); dims from rot_dim on stay as they are.  A gain or
 * a freq[j] that is not finite is refused (CIH_ERR_ARG). */
typedef struct cih_rope {
    int32_t rot_dim, interleaved;
    float gain;
    double freq[64];
} cih_rope;

enum cih_rope_scaling { CIH_ROPE_NONE = 0, CIH_ROPE_LINEAR = 1, CIH_ROPE_NTK = 2, CIH_ROPE_YARN = 3 };

/* Host: fills r for rot_dim dims (even, 2..128).  freq[j] = base^(-2j/rot_dim);
 * LINEAR: divided by factor (position interpolation); NTK: base *
 * factor^(rot_dim / (rot_dim - 2)) in place of base (rot_dim >= 4); YARN
 * (Peng et al. 2023): with g = clamp((trained_len freq / 2 pi - 1) / 31, 0, 1),
 * freq ((1 - g) / factor + g), gain = 0.1 ln(factor) + 1.  factor >= 1;
 * trained_len >= 1 where YARN reads it. */
int cih_rope_init(cih_rope *r, int32_t rot_dim, int32_t interleaved, double base, int32_t scaling, double factor,
                  int32_t trained_len);

/* Writes the batch's rows of K and V (kv_heads heads of head_dim, element type
 * dtype, a cih_float) into the cache at their positions, K rotated if rope is
 * not NULL.  A page that keeps tokens from before the sequence's first row
 * keeps at least their scale; where a new row exceeds it the kept codes are
 * rounded again to the larger one.  Later tokens of the page are forgotten.
 * With q (q_heads heads; NULL: none) the rows of q are written to q_out (may
 * be q; no overlap with k or v), rotated by the same positions; rows without a
 * position in the table (negative, or from max_pages * 64 on) leave it as it
 * was.  No page may be written twice in a batch, by two sequences or by one
 * whose table names it twice. */
int cih_kv8_append(const cih_kv8_cache *cache, const cih_kv8_batch *batch, int32_t dtype, const cih_rows *k,
                   const cih_rows *v, int32_t q_heads, const cih_rows *q, const cih_rows *q_out, const cih_rope *rope,
                   void *stream);

/* The same with angles of other positions: shifts[i] (device, [n_seq]; NULL: 0)
 * is added to the positions of sequence i's rows, for K and q alike, as after
 * cih_kv8_evict, which leaves a sequence fewer tokens than it has had. */
int cih_kv8_append_shifted(const cih_kv8_cache *cache, const cih_kv8_batch *batch, int32_t dtype, const cih_rows *k,
                           const cih_rows *v, int32_t q_heads, const cih_rows *q, const cih_rows *q_out,
                           const cih_rope *rope, const int32_t *shifts, void *stream);

/* The batch's rows read back from the cache as values of type dtype (K as
 * stored, rotated); a bad token's values are NaN.  Rows that are not there
 * are left untouched. */
int cih_kv8_read(const cih_kv8_cache *cache, const cih_kv8_batch *batch, int32_t dtype, const cih_rows *k,
                 const cih_rows *v, void *stream);

/* Attention of the batch's rows over the cache: head h of q_heads (a multiple
 * of kv_heads) reads head h / (q_heads / kv_heads).  A row at position p sees
 * tokens j < lens[i], with causal only j <= p, with window > 0 only j > p -
 * window.  out = sum softmax(scale q.k) v in q's type (may be q, with its
 * strides); lse (NULL: none) [n_rows][q_heads] the logarithm of the sum of
 * exp(scale q.k).  A row that sees nothing gets out 0 and lse -inf, one that
 * sees a bad token NaN.  max_rows * q_heads / kv_heads <= 2^30.  Rows of very
 * different counts, such as prompts beside single tokens, are served better by
 * a call each.  workspace: 16-byte aligned, of the size
 * cih_kv8_attention_workspace gives for the same sizes (it reads no device
 * memory); calls that may run at the same time (other streams, two graphs)
 * need one each. */
int cih_kv8_attention(const cih_kv8_cache *cache, const cih_kv8_batch *batch, int32_t dtype, int32_t q_heads,
                      const cih_rows *q, const cih_rows *out, float *lse, float scale, int32_t causal, int32_t window,
                      void *workspace, size_t workspace_bytes, void *stream);
int cih_kv8_attention_workspace(const cih_kv8_cache *cache, const cih_kv8_batch *batch, int32_t q_heads, size_t *bytes);

/* The same with first tokens that stay visible: a row at position p sees tokens
 * j < lens[i], with causal only j <= p, with window > 0 only j > p - window or
 * j < sinks (without a window sinks change nothing).  Pages between the sinks and the
 * window are not read, and may be missing from the table.  The workspace is
 * cih_kv8_attention_workspace's. */
int cih_kv8_attention_sinks(const cih_kv8_cache *cache, const cih_kv8_batch *batch, int32_t dtype, int32_t q_heads,
                            const cih_rows *q, const cih_rows *out, float *lse, float scale, int32_t causal,
                            int32_t window, int32_t sinks, void *workspace, size_t workspace_bytes, void *stream);

/* ---- a bounded cache -------------------------------------------------------- */

/* The attention weight that cached tokens gather: weights [n_pages][kv_heads][64],
 * beside the cache, gets for token j of a sequence, in each kv head,
 *     keep * (what it had) + sum of exp(scale q.k_j - lse) over the batch's rows that
 *     see it and the query heads that share the kv head,
 * q, lse, scale, causal, window and sinks as in the attention of the same rows.
 * Tokens at the rows' own positions start from 0, with keep = 0 all do: memory
 * that no call has written is not read.  keep is within [0, 1].  Rows whose lse is
 * not finite (they see nothing, or a bad token) add nothing.  Sequences without
 * rows, missing pages and tokens from lens[i] on stay as they are.  No page may
 * stand twice in the batch's tables. */
int cih_kv8_weigh(const cih_kv8_cache *cache, const cih_kv8_batch *batch, int32_t dtype, int32_t q_heads,
                  const cih_rows *q, const float *lse, float scale, int32_t causal, int32_t window, int32_t sinks,
                  float keep, float *weights, void *stream);

/* Cuts sequences to at most budget tokens: each kv head of a sequence that holds more
 * keeps its first `first` tokens, its last `recent` ones (first + recent <=
 * budget), and those of the others with the largest weights (ties: the earlier
 * token; NaN below all), moved to the places 0 .. budget - 1 in their order; the pages
 * behind them are the caller's again.  A page's scale becomes the largest of those that
 * its tokens come from, and codes are rounded again where their scale grows (a scale does not fall when the token that
 * set it goes: a cache that has held outliers keeps their step).  The batch's rows
 * are not used (cu_rows may be NULL); the heads of a sequence may keep different tokens.
 *     weights_out (NULL: not wanted; may be weights): the kept tokens' weights at
 *         their new places.
 *     lens_out (may be lens): tokens that the sequence now holds.
 *     shifts (NULL: none): how many tokens went is added, for cih_kv8_append_shifted.
 *     kept (NULL: none) [n_seq][kv_heads][budget]: the places that the kept tokens
 *         had, ascending, -1 behind them.
 * A sequence within the budget keeps all its tokens.  Of one that is longer than its table has room for
 * the table's tokens are held, and cut like others'; shifts grow by its length less the budget, so that
 * positions go on behind its length.  One whose slot or one of whose pages
 * is not there is left alone (kept -1, lens_out its length).  No page may stand twice in the tables
 * of a call.  workspace: 16-byte aligned, of cih_kv8_evict_workspace's size, not shared by calls that run at the
 * same time: a page that such a call would overwrite before all its tokens are read is left where it is and marked
 * bad, so that reads and attention give NaN for it.
 * Refused, as more than one launch may have: n_seq kv_heads above 2^22 - 1 (tables of up to 32 pages: 2^23 - 1),
 * and n_seq kv_heads ceil(pages / p) above 2^23 - 1, with the pages of the budget (or the table's, if fewer) and
 * p = 2 for heads of 128, 4 of 64, 8 of 16 to 32. */
int cih_kv8_evict(const cih_kv8_cache *cache, const cih_kv8_batch *batch, int32_t budget, int32_t first, int32_t recent,
                  const float *weights, float *weights_out, int32_t *lens_out, int32_t *shifts, int32_t *kept,
                  void *workspace, size_t workspace_bytes, void *stream);
int cih_kv8_evict_workspace(const cih_kv8_cache *cache, const cih_kv8_batch *batch, int32_t budget, size_t *bytes);

/* ---- verification of drafted tokens ----------------------------------------------
 * Speculative sampling from given random numbers.  Sequence i has the drafts
 * cu_drafts[i] .. cu_drafts[i + 1] (of n_drafts, none allowed), and the target's
 * logits for them and the token after them: rows cu_drafts[i] + i .. cu_drafts[i + 1] + i
 * of logits [n_drafts + n_seq][vocab].  draft_logits [n_drafts][vocab] are those the
 * drafts were drawn from (NULL: they were certain, as looked-up ones are).  With
 * p = softmax(logits / temperature), q the same of draft_logits (or 1 at the draft): draft x
 * is accepted if accept_at[draft] * q(x) < p(x); accepted[i] counts those before the first
 * that is not, and tokens[i] follows them: the first token whose running sum of max(p - q, 0)
 * (after all drafts: of p) exceeds sample_at[i] times its total.  Both are in [0, 1).
 * temperature 0: a draft is accepted if it is the row's largest logit (ties: the lowest
 * id), and tokens[i] is the largest; draft_logits, accept_at and sample_at are not read.
 * -inf logits have probability 0.  A row, of the target or the draft, with NaN or
 * +inf or of -inf only ends its sequence: the drafts before it are accepted, tokens[i]
 * is -1.  A draft outside [0, vocab) is not accepted.  Device pointers; workspace as above. */
int cih_verify_drafts(int32_t dtype, const void *logits, int64_t row_stride, const void *draft_logits,
                      int64_t draft_stride, int32_t n_seq, int32_t n_drafts, int32_t vocab, const int32_t *cu_drafts,
                      const int32_t *drafts, const float *accept_at, const float *sample_at, float temperature,
                      int32_t *accepted, int32_t *tokens, void *workspace, size_t workspace_bytes, void *stream);
int cih_verify_drafts_workspace(int32_t n_seq, int32_t n_drafts, int32_t vocab, size_t *bytes);

/* ---- log probabilities of given tokens ----------------------------------------
 * Beside log_softmax_canonical (lib.rs:4426-4441), over the whole vocabulary.
 * For each row of logits [n_rows][vocab] (both <= 2^30, type dtype, rows
 * row_stride elements apart): logprob = log softmax at targets[row]; entropy =
 * -sum p log p (in nats); the top_k <= 64 largest logits (ties: lowest id
 * first) as top_ids [n_rows][top_k] and their log probabilities top_logprobs.
 * logprob, entropy and the top pair may each be NULL.  Device pointers, as
 * above.  A negative target gives 0, one >= vocab NaN.  -inf logits have
 * probability 0: fewer than top_k others leave ids -1 and -inf at the end.  A
 * row of -inf only: entropy 0, logprob -inf; a row with NaN or +inf: NaN and
 * ids -1. */
int cih_token_logprobs(int32_t dtype, const void *logits, int64_t row_stride, int32_t n_rows, int32_t vocab,
                       const int32_t *targets, float *logprob, float *entropy, int32_t top_k, int32_t *top_ids,
                       float *top_logprobs, void *workspace, size_t workspace_bytes, void *stream);
int cih_token_logprobs_workspace(int32_t n_rows, int32_t vocab, int32_t top_k, size_t *bytes);

/* ---- decoding over the 8-bit cache; scores --------------------------------- */

/* A decoder whose keys and values live in the 8-bit paged cache above: 2 bytes
 * a dim and position in place of 8, pages of 64 positions taken from one pool
 * of n_pages (0: enough for every slot's max_len) as the slots grow, given
 * back by cih_decoder_reset, cih_generate and cih_decoder_score, which start slots anew.
 * rope (NULL: as the reference's, the whole head, base 10000) may scale the
 * positions for contexts beyond those the model was trained on; max_len <=
 * 2^20.  cih_decode and cih_generate work as on any decoder, but: rows that
 * rewrite a position make the slot forget the ones after it, a cih_decode that needs
 * more pages than are free returns CIH_ERR_CAPACITY and changes nothing (a
 * cih_generate or cih_decoder_score stops there, its slots started anew), and
 * results carry the rounding of K and V to 8 bits. */
int cih_decoder_create_kv8(cih_model *m, int32_t n_slots, int32_t max_len, int32_t max_rows, int32_t n_pages,
                           const cih_rope *rope, cih_decoder **out);

/* How likely given sequences are, on any decoder: sequence i is tokens
 * [offsets[i], offsets[i + 1]) (at least one), read from position 0 of slot
 * slots[i].  For each token, counted from offsets[0]: logprob of the token
 * after it (0 at a sequence's last one), entropy of the distribution of that
 * token in nats, and its top_k <= min(vocab, 64) likeliest ids with their log
 * probabilities [token][top_k].  Host arrays; logprob and entropy may be NULL.
 * The slots hold the sequences afterwards.  Synchronous. */
int cih_decoder_score(cih_decoder *d, int32_t n, const int32_t *slots, const int32_t *tokens, const int32_t *offsets,
                      int32_t top_k, float *logprob, float *entropy, int32_t *top_ids, float *top_logprobs);

/* K (rotated) and V of n positions from pos on of a slot in one layer, as the
 * rows read them: host arrays [n][dim].  Synchronous. */
int cih_decoder_read_cache(cih_decoder *d, int32_t layer, int32_t slot, int32_t pos, int32_t n, float *k, float *v);

/* ---- kernel-level entry points (host pointers; each call stages through
 * freshly allocated device memory — for tests, not for the hot loop) ------ */

/* matmul_tiled_{fp32,q8,q4}_parallel (lib.rs:4803, 4870, 4937):
 * out[p][i] = sum_k W[i][k] x[p][k] + bias[i] for p < seq_len.
 * w: [out_dim][in_dim] FP32 or packed blocks of that matrix. */
int cih_matmul_tiled(int32_t dtype, float *out, const float *x, const void *w,
                     const float *bias, int32_t in_dim, int32_t out_dim, int32_t seq_len);

/* No counterpart in the reference: a variant of cih_matmul_tiled for callers
 * that cannot allocate device memory (code under HIP graph capture, tight
 * serving loops, harnesses that forbid hipMalloc).  out, x, w and bias are
 * DEVICE pointers (w 4-byte aligned, x 16-byte aligned; w in the same
 * reference layout as above); the call is enqueued on `stream` (a
 * hipStream_t; NULL = the null stream) and returns without waiting.  It
 * calls no allocator: the repacked weight matrix and the partial sums of a
 * k-split live in one fixed device array per GPU (48 MiB, held from the time
 * the library's code is loaded on that GPU until the process ends), so a
 * matrix whose repacked form exceeds 32 MiB returns CIH_ERR_CAPACITY (650M
 * FC1 in Q8_0 is 7.4 MB; a 3B FC1 in Q8_0 29.5 MB).  Every call on one GPU
 * uses the same array: calls that overlap on one GPU (other streams, other
 * threads) race; calls in order on one stream do not.  Results equal
 * cih_matmul_tiled's bit for bit. */
int cih_matmul_tiled_noalloc(int32_t dtype, float *out, const float *x, const void *w, const float *bias,
                             int32_t in_dim, int32_t out_dim, int32_t seq_len, void *stream);

/* Dequantizes nblocks blocks on the GPU with the decode routine the GEMMs
 * use (BlockQ8_0/BlockQ4_0::dequantize_to, lib.rs:663-667, 1074-1082). */
int cih_dequantize_device(int32_t dtype, const void *blocks, int64_t nblocks, float *out);

/* quantize_slice_to_q8 / quantize_slice_to_q4 (lib.rs:670-673, 1085-1088)
 * on the GPU, with the kernel that cih_model_create_from_file(quantize_to)
 * runs on FP32 weights; bit-identical to cih_quantize_q8 / cih_quantize_q4.
 * n must be a multiple of 32; dst holds n/32 blocks. */
int cih_quantize_device(int32_t dtype, const float *src, int64_t n, void *dst);

/* ---- host helpers (no GPU) ---------------------------------------------- */

/* quantize_slice_to_q8 / quantize_slice_to_q4 (lib.rs:670-673, 1085-1088);
 * n must be a multiple of 32; dst holds n/32 blocks. */
int cih_quantize_q8(const float *src, int64_t n, void *dst);
int cih_quantize_q4(const float *src, int64_t n, void *dst);
int cih_dequantize_q8(const void *blocks, int64_t nblocks, float *dst);
int cih_dequantize_q4(const void *blocks, int64_t nblocks, float *dst);

/* Tokenizer::encode (lib.rs:6511-6521).  Returns the token count (>= 2) or a
 * negative status if cap is too small. */
int cih_tokenize(const char *text, int32_t *out, int32_t cap);

/* log_softmax_canonical (lib.rs:4426-4441) over one row of 33 logits. */
int cih_log_softmax_canonical(const float *logits, float *out33);

/* ---- per-kernel timing (HIP events on the model's stream) ---------------- */
enum cih_kernel_class {
    CIH_KC_GEMM_QUANT = 0, /* Q8_0 / Q4_0 weight GEMMs                    */
    CIH_KC_GEMM_FP32 = 1,  /* FP32-weight GEMMs (FP32 models, LM head)    */
    CIH_KC_ATTENTION = 2,  /* attention                                   */
    CIH_KC_OTHER = 3,      /* embedding, LayerNorm, contacts, scatter     */
    CIH_KC_COUNT = 4
};

typedef struct cih_kernel_stats {
    int64_t launches;
    double total_ms;   /* summed launch durations (hipEventElapsedTime)   */
    double flops;      /* algorithmic FLOPs of those launches             */
    double bytes;      /* algorithmic HBM bytes (weights + activations)   */
} cih_kernel_stats;

/* enable != 0 resets the totals and starts recording (one event pair per
 * launch, summed after each cih_forward); enable == 0 stops recording and
 * keeps the totals for cih_profile_read. */
int cih_profile_enable(cih_model *m, int32_t enable);
int cih_profile_read(const cih_model *m, int32_t kernel_class, cih_kernel_stats *out);

const char *cih_last_error(void);
int cih_abi_version(void);

#ifdef __cplusplus
}
#endif
#endif

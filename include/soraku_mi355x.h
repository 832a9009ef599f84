/*
 * soraku_mi355x.h -- C ABI of the MI355X (gfx950) per-frame CFG decode engine
 * for soraku-TTS.
 *
 * Plain C: opaque handles, plain pointers and sizes, integer status codes.
 * Device pointers are HIP device addresses (for example torch.Tensor.data_ptr()
 * of a tensor on "cuda"); host pointers are ordinary process memory.  Every
 * argument is validated before any HIP call, so argument errors are reported
 * without touching the GPU.
 *
 * Reference interfaces replaced (paths relative to the reference checkout):
 *   engine object     GraphFrameEngine          soraku_inference/acceleration/graph_frame.py:23-83
 *   prefill           GraphFrameEngine.prefill  graph_frame.py:118-198 (per-row caches instead of
 *                                               left padding; layout of model.py:623-656)
 *   capture           GraphFrameEngine.capture  graph_frame.py:274-296
 *   step_frame        GraphFrameEngine.step_frame graph_frame.py:298-305
 *   set_temperature / set_sampling / cfg        graph_frame.py:307-324, graph_frame.py:68
 *   operator API      TileLang factories        soraku_inference/acceleration/tilelang_kernels.py:34-254
 *   weight keys       SorakuTTSv2 state dict    model.py:100-145 + transformers Qwen3Model
 */
#ifndef SORAKU_MI355X_H
#define SORAKU_MI355X_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes (0 = success) ---------------------------------------- */
#define SK_OK          0
#define SK_EINVAL     -1   /* bad argument (shape, range, null pointer, unknown key)      */
#define SK_ENOWEIGHT  -2   /* a required weight was never bound                           */
#define SK_ENOCAPTURE -3   /* step before capture (graph_frame.py:301-302)                 */
#define SK_EKVFULL    -4   /* KV cache or frame ring full (graph_frame.py:155-156)         */
#define SK_EHIP       -5   /* a HIP runtime call failed, or host memory for a prefix ran out;
                              sk_last_error() says which                                  */
#define SK_ESTATE     -6   /* call out of order (e.g. step before prefill)                 */

/* ---- element types --------------------------------------------------- */
#define SK_F32  0
#define SK_BF16 1
/* ---- what a projection does with its sums ------------------------------ */
#define SK_ACT_NONE   0
#define SK_ACT_SWIGLU 1

/* Model dimensions and special ids (SorakuV2Config model.py:34-63 plus the
 * Qwen3 text config).  audio_vocab = codebook_size + 3 (model.py:61-63). */
typedef struct sk_config {
  int32_t d_model;        /* hidden size (1024 for Qwen3-0.6B)                 */
  int32_t n_layers;       /* trunk layers (28)                                 */
  int32_t n_q_heads;      /* 16                                                 */
  int32_t n_kv_heads;     /* 8                                                  */
  int32_t head_dim;       /* 128                                                */
  int32_t trunk_inter;    /* trunk SwiGLU inner size (3072)                     */
  int32_t depth_inner;    /* depth-head SwiGLU inner size d*depth_ffn_mult      */
  int32_t n_codebooks;    /* Q = 16                                             */
  int32_t audio_vocab;    /* V = codebook_size + 3 = 2051                        */
  int32_t text_vocab;     /* rows of trunk.embed_tokens.weight                  */
  int32_t bos_id, eos_id, pad_id;   /* 2048, 2049, 2050                         */
  float trunk_eps;        /* 1e-6 (Qwen3RMSNorm)                                */
  float depth_eps;        /* FLT_EPSILON (nn.RMSNorm(eps=None), model.py:135)   */
  float rope_theta;       /* 1e6                                                */
  float frame_scale;      /* Q^-1/2 (model.py:99)                               */
  int32_t weight_dtype;   /* SK_F32 or SK_BF16 for every matrix                 */
  int32_t n_utts;         /* utterances decoded together (n_utts*cfg_rows <= 32) */
  int32_t cfg_rows;       /* rows per utterance: 2 = cond+uncond, 1 = no CFG     */
  int32_t max_ctx;        /* KV capacity per row (prefix + frames)              */
  int32_t max_frames;     /* capacity of the per-frame input/code ring          */
  int32_t n_language;     /* language-token rows (0 or 4, model.py:186-197)     */
  int32_t language_ids[4];/* their text ids (model.py:326-338)                  */
  int32_t kv_dtype;       /* KV cache element: SK_F32 (reference) or SK_BF16    */
} sk_config;

typedef struct sk_engine sk_engine;

/* Last error message of the calling thread ("" if none). */
const char* sk_last_error(void);

/* Create an engine: allocates KV cache, activations and the frame ring on
 * the current HIP device.  `hip_stream` may be NULL; the engine always runs
 * on a stream of its own and makes that stream wait on `hip_stream`. */
int sk_create(const sk_config* cfg, void* hip_stream, sk_engine** out);
int sk_destroy(sk_engine* e);

/* Bind a weight by its state-dict key (weights are borrowed, never freed).
 * dtype: SK_F32 for gains/tables/bias; matrices use cfg->weight_dtype.
 * Keys: trunk.layers.{i}.{input_layernorm,post_attention_layernorm}.weight,
 *       trunk.layers.{i}.self_attn.{q,k,v,o}_proj.weight,
 *       trunk.layers.{i}.self_attn.{q,k}_norm.weight,
 *       trunk.layers.{i}.mlp.{gate,up,down}_proj.weight, trunk.norm.weight,
 *       trunk.embed_tokens.weight, audio_codebooks.table,
 *       depth_head.norm_in.weight, depth_head.mlp.{gate,up,down}_proj.weight,
 *       depth_head.norm_out.weight, depth_head.bias, language_embeddings.weight,
 *       and depth_head.out_proj [Q][V][d] for an untied classifier (model.py:141-145;
 *       when it is not bound the classifier is the tied audio_codebooks.table). */
int sk_bind_weight(sk_engine* e, const char* key, const void* dev_ptr, int32_t dtype,
                   const int64_t* shape, int32_t ndim);

/* Stage one row's prefix: text ids, then the frames `frame_codes[n_frames][Q]`
 * (the caller includes the BOS frame first, model.py:633-642).  Resets the row.
 * The ids and codes are copied; they are embedded when the prefill runs, with
 * the weights bound then. */
int sk_prefill_row(sk_engine* e, int32_t row, const int64_t* text_ids, int32_t n_text,
                   const int64_t* frame_codes, int32_t n_frames);
/* Run every staged row through the trunk; leaves per-row hidden and KV length.
 * Every row must be staged; the frame counter starts over.  The order of sums
 * (GEMM tiles, K slices, key splits) goes by the tokens of the whole call: a
 * prefix's hidden state and cache can differ in their last bits with what is
 * prefilled beside it, alone, in a batch or as a refill (by 2e-6 of the largest
 * value with FP32 weights, 6e-6 with BF16, where measured; a BF16 cache rounds
 * such a difference to one place of a few elements).  The same call repeats bit for bit. */
int sk_prefill_run(sk_engine* e);
/* sk_prefill_run that allocates no device memory.  No counterpart in the
 * reference: for callers that cannot allocate (serving loops that must not
 * stall on hipMalloc, harnesses that forbid it).  It copies small host-side
 * tables and waits for the engine's stream, so it cannot be recorded into a
 * graph: on a capturing stream it returns SK_ESTATE.  The prefill's activation
 * buffers come from a scratch array of SK_NOALLOC_SCRATCH_BYTES in the
 * library's device code (one per GPU, held until the process ends) instead
 * of the engine's lazily grown buffers; a packed prefix that needs more
 * (about 600 tokens at the Qwen3-0.6B shape, 450 at 1.7B) is rejected with
 * SK_EINVAL -- sk_prefill_run takes any size.  Every call on one GPU shares
 * that scratch, so calls that overlapped on one GPU would race; the device
 * order of engines (below, at sk_replay) makes the prefills of different
 * engines take turns, and one engine's calls share its stream.  Results are
 * those of sk_prefill_run, bit for bit. */
#define SK_NOALLOC_SCRATCH_BYTES (32u << 20)
int sk_prefill_run_noalloc(sk_engine* e);
/* Continuous batching (no counterpart in the reference, which decodes one
 * utterance's CFG pair, fast_generate.py:232-328): between frames, run only
 * the rows staged since the last prefill (at least one) through the trunk.
 * Every other row keeps its cache, length, position and hidden state, and the
 * frame counter is unchanged, so an utterance slot whose utterance retired
 * takes the next utterance while the others keep decoding.  The staged rows
 * become active.  Requires a completed sk_prefill_run. */
int sk_prefill_refill(sk_engine* e);
/* Stop decoding one row (no reference counterpart; continuous batching): it
 * no longer advances its length or position, attention skips it and the
 * cache-capacity checks ignore it.  Its codes are meaningless until a refill. */
int sk_retire_row(sk_engine* e, int32_t row);
/* Restart the frame ring (no reference counterpart): the next frame uses slot
 * 0 again, so codes of earlier frames can no longer be read with
 * sk_read_codes.  Lets one engine decode more than max_frames frames in all. */
int sk_reset_frames(sk_engine* e);

/* Override one row's KV length and RoPE position (after an external prefill). */
int sk_set_row_state(sk_engine* e, int32_t row, int32_t kv_len, int32_t position);
/* Device address of layer `layer`'s K (kv=0) or V (kv=1) cache,
 * laid out [rows][n_kv_heads][max_ctx][head_dim] of cfg->kv_dtype elements
 * (FP32, or BF16 bits rounded to nearest even). */
int sk_kv_ptr(sk_engine* e, int32_t layer, int32_t kv, void** out);
/* Copy the current depth-input hidden state [rows][d] to host memory. */
int sk_get_hidden(sk_engine* e, float* host_out);

/* Sampling parameters (model.py:515-533 semantics).  temperature <= 0 means
 * greedy.  *_q0 override codebook 0; pass has_q0 = 0 to use the main values.
 * top_k <= 0 or >= V disables top-k; top_p outside (0,1) disables top-p.
 * Read by the captured graph on every replay: no re-capture needed. */
int sk_set_sampling(sk_engine* e, float cfg_scale, float temperature, int32_t top_k,
                    float top_p, int32_t has_q0, float temperature_q0, int32_t top_k_q0,
                    float top_p_q0);
/* Debug switches: record masked merged logits of every depth step; force codes. */
int sk_set_debug(sk_engine* e, int32_t record_logits);

/* Capture one whole frame (16 depth steps + sampling + frame embedding +
 * trunk step) as one hipGraph.  With one utterance (with or without CFG) at
 * the depth widths of the Qwen3-0.6B or Qwen3-1.7B shape, and with more than 4
 * decode rows, capture also derives the depth steps' code tables from the
 * bound codebook table, depth norm_in gain and gate/up weights
 * ((Q-1) x V x 2 x depth_inner floats: 0.5 GB / 1.0 GB); those weights must
 * not change afterwards. */
int sk_capture(sk_engine* e);

/* Replay one frame.  mask_eos_q0: bit u masks EOS at codebook 0 for
 * utterance u (the min_new_frames rule, model.py:583-584); with one utterance
 * 0 or 1.  uniforms: [n_utts][Q] draws in [0,1) (NULL => 0).
 * forced_codes: NULL, or [n_utts][Q] codes to use instead of the sampled ones
 * (teacher forcing).  codes_out: host [n_utts][Q].  logits_dbg: NULL or host
 * [n_utts][Q][V] masked merged logits (needs sk_set_debug(e, 1)).
 * Synchronous on the codes copy, like graph_frame.py:305. */
int sk_step_frame(sk_engine* e, int32_t mask_eos_q0, const double* uniforms,
                  const int64_t* forced_codes, int64_t* codes_out, float* logits_dbg);

/* Throughput path: upload per-frame inputs for the next `n` frames
 * (uniforms [n][n_utts][Q], mask_eos_q0 [n] utterance bit masks as in
 * sk_step_frame), then replay `n` frames back to
 * back with no host synchronisation.  sk_read_codes copies codes of the
 * `n` most recent frames ([n][n_utts][Q]).
 * Frames and prefills of different engines on one device run one after
 * another: when the device's work passes from one engine to another
 * (sk_step_frame, sk_replay, the prefills), the new engine's stream first
 * waits for the work queued on the previous engine's stream.  An engine
 * working alone pays nothing. */
int sk_queue_frames(sk_engine* e, int32_t n, const double* uniforms, const int32_t* mask_eos_q0);
int sk_replay(sk_engine* e, int32_t n);
int sk_read_codes(sk_engine* e, int32_t n, int64_t* codes_out);
int sk_synchronize(sk_engine* e);
/* The engine's stream (hipStream_t) and frame counter. */
void* sk_stream(sk_engine* e);
int32_t sk_frames_done(sk_engine* e);
/* Diagnostic with no counterpart in the reference (which has one decode
 * path): 1 when the engine runs its trunk as XCD-resident layers (two
 * launches per layer; one or two decode rows at the Qwen3-0.6B or Qwen3-1.7B
 * trunk shape but one FP32 row at the latter, on a device of 256 CUs, unless
 * SORAKU_XCD_LAYERS=0 was set at sk_create), 0 when it runs the per-op layer
 * kernels, -1 for a NULL engine.  These layers hold the residual stream in
 * units of 2^-32 (64 bits): a residual row with a norm of 2^27 or more becomes
 * NaN, as one that holds NaN or infinity does.  For tests and profiling. */
int32_t sk_xcd_layers(sk_engine* e);
/* Test hook with no counterpart in the reference: the bound, in ticks of the
 * 100 MHz real-time counter, of every wait inside a frame's kernels (the
 * XCD-resident layers' barriers and tagged exchanges, the many-row split-K
 * GEMMs' merge of tagged partials; default and maximum 5,000,000 = 50 ms).
 * Set before sk_capture (SK_ESTATE after).  A wait that passes it sets the
 * engine's error word, the kernel goes on without the missing data, and the
 * next sk_step_frame / sk_synchronize / sk_read_codes returns SK_EHIP; 0
 * makes nearly every wait give up at once, which is how a test forces that
 * error path while every kernel still exits normally.  The engine must then
 * be recreated. */
int sk_debug_set_spin_ticks(sk_engine* e, uint64_t ticks);

/* ---- operator API (tilelang_kernels.py counterparts) ------------------
 * All pointers are device pointers, all tensors contiguous row-major.
 * `stream` is a hipStream_t (NULL = default stream).  Matrices: wdtype. */
int sk_op_add_rmsnorm(void* stream, int32_t B, int32_t D, float eps, const float* hidden,
                      const float* prefix, const float* weight, float* out);   /* :34-55  */
int sk_op_rmsnorm(void* stream, int32_t B, int32_t D, float eps, const float* x,
                  const float* weight, float* out);                            /* :58-78  */
int sk_op_swiglu_gemv(void* stream, int32_t B, int32_t I, int32_t D, int32_t wdtype,
                      const float* x, const void* wg, const void* wu, float* out);  /* :81-112 */
int sk_op_down_residual_gemv(void* stream, int32_t B, int32_t D, int32_t I, int32_t wdtype,
                             const float* act, const void* wd, const float* residual,
                             float* out);                                      /* :115-143 */
int sk_op_classifier_gemv(void* stream, int32_t B, int32_t V, int32_t D, int32_t wdtype,
                          const float* body, const void* wq, const float* bias,
                          float* out);                                         /* :146-173 */
int sk_op_frame_embed(void* stream, int32_t R, int32_t Q, int32_t V, int32_t D, float scale,
                      const int64_t* codes, const float* table, float* out);   /* :176-196 */
int sk_op_prefix_add(void* stream, int32_t B, int32_t V, int32_t D, float scale,
                     const float* prefix, const float* table_q, const int64_t* code,
                     float* out);                                              /* :199-216 */
int sk_op_sampling_prep(void* stream, int32_t V, int32_t bos_id, int32_t pad_id,
                        int32_t eos_id, const float* logits, const float* temperature,
                        const int32_t* mask_eos, float* out);                  /* :219-254 */
/* Fused CFG + masks + temperature + top-k/top-p + explicit-uniform draw for
 * one utterance (model.py:579-595,686-708; graph_frame.py:214-242).
 * logits: [rows][V] (row 0 cond, row 1 uncond).  code_out: device int64[1]. */
int sk_op_sample(void* stream, int32_t rows, int32_t V, const float* logits, float cfg_scale,
                 int32_t q, int32_t mask_eos_q0, int32_t bos_id, int32_t eos_id, int32_t pad_id,
                 float temperature, int32_t top_k, float top_p, double u, int64_t* code_out);

/* ---- operator API: attention over a cache in pages --------------------
 * The attention half of a trunk layer, for programs that drive layers one
 * operator at a time; no counterpart in the reference, whose caches are one
 * tensor per row.
 *
 * K and V lie in pools [n_pages][Hkv][page][hd], page a multiple of 16 (an
 * engine's cache, sk_kv_ptr, is such a pool where max_ctx is a multiple of 16:
 * one page of max_ctx tokens per row).  Sequence s of S has the pages
 * table[s][0 .. width), rows of the table table_stride entries apart; slot j of
 * it lies in page table[s][j / page].  Its new tokens of a call are the packed
 * rows starts[s] .. starts[s + 1] of T, and lens[s] is its length with them:
 * token i of n has slot lens[s] - n + i.  Sequences without new tokens and
 * lengths of 0 are fine; rows from starts[S] on are padding and left alone.
 * table, starts and lens are device int32; the pages of a sequence that append or
 * accounts write to are different ones.
 *
 * The host does not look at device memory, so the kernels hold what they find
 * there in range: lens to [0, width * page], starts to [0, T].  A table entry
 * outside [0, n_pages) is no page: append drops what would go there, tokens
 * that see a key there come out of attention as NaN, accounts there are not
 * kept, eviction moves NaN from it and nothing to it.  Entries of pages that no
 * token sees may be anything.  A sequence with a length past its table has no place
 * for its tokens: append stores none of them, they come out of attention as NaN, its
 * accounts stay as they are; eviction goes by the slots that the table has.
 *
 * xdtype / kvdtype: activations and cache, SK_F32 / SK_F32, SK_F32 / SK_BF16 or
 * SK_BF16 / SK_BF16; sums and softmax are FP32, products of FP32 activations
 * exact; with BF16 activations a softmax weight enters its product with v with 16
 * bits (hd 16: 32), rounded to nearest, whatever else is in the call.  hd: 16, 32,
 * 64 or 128.  Hq: a multiple of Hkv, at most 4096; query heads h G .. h G + G - 1
 * share key head h.  S is at most 65535; T may be 0 and is below 2^24; width * page
 * and T * Hq are at most 2^30.  q, qkv, gains, pages, outputs of xdtype and workspaces
 * are 16-byte aligned; outputs overlap no operand.  No call allocates, waits or copies
 * to the host, and each may be captured into a graph.
 *
 * How attention and accounts are cut up is planned for the whole call, from the
 * average of new tokens, T / S, and from width.  So single tokens and chunks belong
 * in calls of their own (two tokens over 61,440 slots take 93 us and a chunk of 2,047
 * 97, all in one call 2,254), and a table of the program's capacity is given as wide as
 * its longest sequence needs now, which table_stride allows (a prompt of 200: 11 us, in
 * a table of 8,192 slots 21). */

/* New tokens into the cache: qkv [T][(Hq + 2 Hkv) hd] as projected.  q and k are
 * normalised per head (RMSNorm with gains [hd]; both NULL: not) and rotated by
 * positions[T] * inv_freq[hd / 2] (pairs i and i + hd / 2; the angle in 64 bits,
 * so far positions are exact); q goes to q_out [T][Hq][hd] of xdtype, k and v to
 * their slots.  mass (may be NULL): accounts of attention weight
 * [n_pages][Hkv][page], set to 0 at those slots.  Positions go their own way from
 * slots: a cache that was cut back keeps counting. */
int sk_op_paged_append(void* stream, int32_t T, int32_t S, int32_t Hq, int32_t Hkv, int32_t hd, int32_t page,
                       int32_t n_pages, int32_t width, int64_t table_stride, int32_t xdtype, int32_t kvdtype,
                       float eps, const void* qkv, const float* q_gain, const float* k_gain,
                       const float* inv_freq, const int32_t* positions, const int32_t* starts,
                       const int32_t* lens, const int32_t* table, void* k_pages, void* v_pages, float* mass,
                       void* q_out);
/* Attention of the new tokens over their sequences' slots: out = softmax(scale q
 * k^T) v [T][Hq][hd] of xdtype, lse (may be NULL) [T][Hq] the natural logarithm of
 * the softmax's sum.  The token at slot p sees slot j when j <= p and, with a
 * window > 0, also j > p - window or j < sinks.  A token that sees nothing (slot
 * below 0) gives 0 and -infinity.  What a token does not see does not reach it,
 * whatever it holds; what it sees should be finite (infinities there may come out
 * as NaN).  The workspace holds the bytes that _workspace gives for the same
 * arguments (where that is 0 it may be NULL) and belongs to the call until it has
 * run. */
int sk_op_paged_attention_workspace(int32_t T, int32_t S, int32_t Hq, int32_t Hkv, int32_t hd, int32_t page,
                                    int32_t width, int32_t xdtype, int32_t kvdtype, int32_t window,
                                    int32_t sinks, int64_t* bytes);
int sk_op_paged_attention(void* stream, int32_t T, int32_t S, int32_t Hq, int32_t Hkv, int32_t hd, int32_t page,
                          int32_t n_pages, int32_t width, int64_t table_stride, int32_t xdtype, int32_t kvdtype,
                          float scale, int32_t window, int32_t sinks, const void* q, const void* k_pages,
                          const void* v_pages, const int32_t* table, const int32_t* starts, const int32_t* lens,
                          void* out, float* lse, void* workspace, int64_t workspace_bytes);
/* Adds the attention weight that every slot got from the new tokens, exp(scale q k
 * - lse) summed over tokens and the group's heads, to its account in mass
 * [n_pages][Hkv][page].  q, lse, scale, window and sinks as in the attention call
 * (a token whose lse is NaN makes NaN of the accounts that it sees).
 * The order of sums is fixed.  Two sequences of one call that both have new tokens
 * must not share a page: each would add to accounts that the other adds to.
 * width * page is at most 65535 * 256 over BF16 caches with hd of 32 or more, 65535 *
 * 128 otherwise.  Workspace as for attention. */
int sk_op_paged_attention_mass_workspace(int32_t T, int32_t S, int32_t Hq, int32_t Hkv, int32_t hd,
                                         int32_t page, int32_t width, int32_t xdtype, int32_t kvdtype,
                                         int64_t* bytes);
int sk_op_paged_attention_mass(void* stream, int32_t T, int32_t S, int32_t Hq, int32_t Hkv, int32_t hd,
                               int32_t page, int32_t n_pages, int32_t width, int64_t table_stride,
                               int32_t xdtype, int32_t kvdtype, float scale, int32_t window, int32_t sinks,
                               const void* q, const float* lse, const void* k_pages, const int32_t* table,
                               const int32_t* starts, const int32_t* lens, float* mass, void* workspace,
                               int64_t workspace_bytes);
/* Cuts caches back to n = min(lens[s], keep) slots: of every key head the first
 * `sinks`, the last `recent` and, of the others, those with the largest accounts
 * (ties to the lowest slot, NaN above all) move in their order, with their
 * accounts, to slots 0 .. n - 1 of the pages `to` [S][to_width] (rows to_stride
 * apart).  A page of `to` appears there once and not in `table`: old pages, which
 * other sequences may share as they share a prompt, are only read.  new_lens [S],
 * and kept [S][Hkv][keep] the old slots, -1 past n; S * Hkv * keep is below 2^31. */
int sk_op_paged_evict(void* stream, int32_t S, int32_t Hkv, int32_t hd, int32_t page, int32_t n_pages,
                      int32_t width, int64_t table_stride, int32_t kvdtype, int32_t keep, int32_t sinks,
                      int32_t recent, void* k_pages, void* v_pages, float* mass, const int32_t* table,
                      const int32_t* lens, const int32_t* to, int64_t to_stride, int32_t to_width,
                      int32_t* new_lens, int32_t* kept);

/* ---- operator API: projections with 8-bit weights -----------------------
 * Matrices of one byte per element for programs that drive layers one operator at a
 * time; no counterpart in the reference, whose weights are FP32 or BF16.
 *
 * A row t of K values has codes q = 127 t / max|t|, rounded to the nearest whole number
 * (exactly; ties to even), and a scale max|t| / 127: it stands for q * scale.  A row of
 * zeros has scale 0; one with an infinity or NaN has codes 0 and scale NaN.  A row's codes
 * take Kp bytes, K rounded up to a multiple of 128, zeros behind K.  K is at most 130,944.
 * xdtype is SK_F32 or SK_BF16; operands are 16-byte aligned but scales, bias and odd rows
 * within them.  No call allocates, waits or copies to the host, and each may be captured into a
 * graph. */

/* Codes [R][Kp] and scales [R] of R rows x [R][K] of xdtype, for weights at load time.  R may be 0
 * and is below 2^24. */
int sk_op_int8_rows(void* stream, int32_t R, int32_t K, int32_t xdtype, const void* x, int8_t* codes, float* scales);
/* out [M][N] = act(x W^T + bias) + residual with W [N][K] as codes [N][Kp] and scales [N]; bias [N] and residual
 * [M][N] may be NULL.  With SK_ACT_SWIGLU W has 2 N rows, gate rows first, bias 2 N, and out is silu(gate) * up (+
 * residual).  x, residual and out are of xdtype; out may be residual itself (sums in place), and overlaps no other operand.
 * The rows of x become codes on the way; with eps >= 0 x is normalised first (RMSNorm with gain [K], or NULL for
 * none): then fp32(x gain) is coded and the norm's factor goes into the scale.  Products are summed
 * in whole numbers, exactly, so a row's result does not hang on what else is in the call; scales, bias, act
 * and residual follow in FP32, rounded once at the end (silu of less than -87.3 is 0: it is 1.03e-36 at most there).  A row of x with an infinity or NaN gives NaN, and so does one whose
 * x gain is past FP32's range; any other row is normalised, however large or small its values are.  Codes of W
 * may be any bytes, -128 too, whoever made them (behind K they meet zeros).
 * M may be 0 and is below 2^24; N is at most 2^20; M N of up to 2^35 is taken, and more may be refused (SK_EINVAL) by the call though
 * not by _workspace: it then takes several calls.  The workspace holds the bytes that _workspace gives for the same
 * sizes (where that is 0 it may be NULL) and belongs to the call until it has run. */
int sk_op_int8_linear_workspace(int32_t M, int32_t N, int32_t K, int32_t xdtype, int32_t act, int64_t* bytes);
int sk_op_int8_linear(void* stream, int32_t M, int32_t N, int32_t K, int32_t xdtype, int32_t act, float eps,
                      const void* x, const float* gain, const int8_t* codes, const float* scales, const float* bias,
                      const void* residual, void* out, void* workspace, int64_t workspace_bytes);

/* ---- operator API: sampling by row --------------------------------------
 * sk_op_sample for a batch: every row of logits with its own parameters, read from device memory when the call runs
 * (so a captured graph follows them), over vocabularies of up to 2^20, with min-p and a mask of bits.
 *
 * logits are R rows of V values of dtype (SK_F32 or SK_BF16), rows stride elements apart; with cfg_scale [R] they are
 * 2 R rows, cond and uncond of each in turn, merged as uncond + cfg_scale (cond - uncond) in FP32, each
 * operation rounded.  Candidates of a row are its finite values; with allowed, those whose bit (id % 32 of word
 * id / 32) is set, words allowed_stride apart by row (0: one row for all).  They are divided by temperature[r] in
 * FP32 (results held to the finite range); a temperature that is not above 0 takes the largest one, of equal ones that of the lowest id.
 *
 * In the order of values, largest first, equal ones by the lower id: top_k[r] in [1, candidates) keeps those
 * down to the k-th's value (all that equal it); top_p[r] in (0, 1) of these the first ones up to and with the one
 * whose sum of weights e^(x - largest) passes top_p of their whole; min_p[r] in (0, 1] of these the ones with a weight of at
 * least min_p.  Other values of these, and NULL arrays, filter nothing (temperature: 1).  token[r] is
 * the first kept one whose sum passes u[r] of the kept sum; u is in [0, 1) (below it counts as 0; 1 or more draws the last one that
 * adds to the sum).  Sums are within 2^-31 of the largest weight and 2^-42 of themselves (up to 2^16 values 2^-35 and
 * 2^-46), and a row's results have the same bits in any call.  logprob (may be NULL): the
 * logarithm of the drawn one's part of the kept sum, 0 when greedy or of an only one; kept (may be NULL): how many were kept.  A row without candidates
 * gives -1, -infinity and 0.  R may be 0 and is at most 65535.  No call allocates, waits or copies to the host.  Workspace as for
 * the operators above. */
int sk_op_sample_rows_workspace(int32_t R, int32_t V, int32_t dtype, int64_t* bytes);
int sk_op_sample_rows(void* stream, int32_t R, int32_t V, int32_t dtype, const void* logits, int64_t stride,
                      const double* u, const float* temperature, const int32_t* top_k, const float* top_p,
                      const float* min_p, const float* cfg_scale, const uint32_t* allowed, int64_t allowed_stride,
                      int64_t* token, float* logprob, int32_t* kept, void* workspace, int64_t workspace_bytes);

#ifdef __cplusplus
}
#endif
#endif /* SORAKU_MI355X_H */

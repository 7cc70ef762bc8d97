/* C ABI of libmoshi_tlm.so: token language models on MI355X (gfx950).  Same conventions as moshi_mi.h - device pointers unless said
 * otherwise, work enqueued on the caller's stream, status codes with mmi_last_error(), a handle bound to the device current at create. */
#ifndef MOSHI_TLM_H_
#define MOSHI_TLM_H_
#include "moshi_mi.h"
#ifdef __cplusplus
extern "C" {
#endif

/* ------------------------------------------------------------------------------------------ */
/* Token language models: decoder-only networks over token ids (libmoshi_tlm.so)              */
/* ------------------------------------------------------------------------------------------ */
/* The layers are data: each has one mixer and one feed-forward reading norms of the same input (parallel sublayers), optional layer
 * scales, grouped RMS norms, an optional run of layers repeated with the same weights.  Sequences live in slots; their attention cache
 * is a pool of pages of mmi_tlm_info(MMI_TLM_PAGE_TOKENS) tokens, their recurrent state one entry per slot and recurrent layer run. */

/* mixers */
#define MMI_TLM_MIX_LATENT_ATTENTION 1
#define MMI_TLM_MIX_MINGRU 2
#define MMI_TLM_MIX_ATTENTION 3         /* softmax attention, query heads share key/value heads */
#define MMI_TLM_MIX_CHANNEL_DELTA 4     /* gated delta rule, one decay per key channel */
#define MMI_TLM_MIX_LIGHTNING 5         /* linear attention, one constant decay per head */
/* feed-forwards */
#define MMI_TLM_MLP_NONE 0
#define MMI_TLM_MLP_MOE 1
#define MMI_TLM_MLP_DENSE 2             /* gated: gate and up projections, down projection */
/* feed-forward activations */
#define MMI_TLM_ACT_RELU2 1
#define MMI_TLM_ACT_CLAMPED_SWIGLU 2    /* g = min(gate, limit), u = clamp(up, +-limit): g sigmoid(1.702 g) (u + 1) */
/* routers */
#define MMI_TLM_ROUTE_TOKEN_TABLE 1
/* what the passes of the repeated layers start with */
#define MMI_TLM_LOOP_ADD 0              /* the second and later ones: x + embedding */
#define MMI_TLM_LOOP_PROJECT 1          /* every one: loop.in [x; embedding] + loop.step[pass] */

typedef struct mmi_tlm_layer {
    int32_t mixer;
    int32_t width;                                /* minGRU: channels */
    int32_t heads, dim, vdim, rot_dim;            /* latent attention: per head un-rotated / value / rotated dimensions */
    int32_t q_rank, kv_rank;
    int32_t window;                               /* keys seen, the position itself included; 0 = all earlier ones */
    float scale;
    double rot_base;
    int32_t mlp, experts, top, ff, act, router;
    int32_t kv_heads;                             /* attention, channel delta: key/value (query/key) heads */
    int32_t keep_first;                           /* attention with a window: first positions that stay visible */
    int32_t sink;                                 /* attention: one is added to the softmax denominator */
    int32_t conv;                                 /* channel delta: taps of the short convolutions */
    int32_t decay_rank, gate_rank;                /* channel delta: ranks of the decay's and the gate's projection */
    const double* decay;                          /* lightning: [heads], host */
    float limit;                                  /* clamped SwiGLU */
} mmi_tlm_layer;

typedef struct mmi_tlm_cfg {
    int32_t vocab, width, n_layers;
    const mmi_tlm_layer* layers;
    int32_t loop_start, loop_stop, loop_times;    /* layers [start, stop) run `times` times; start == stop: no repetition */
    int32_t norm_groups;
    float norm_eps, logit_scale;
    int32_t loop_inject, norms, layer_scales;     /* norms 2: the feed-forward has a norm of its own; layer_scales: ls1 / ls2 exist */
    int32_t tied_head;                            /* logits from the (unscaled) embedding table */
    float embed_scale;
    int32_t bigram_buckets;                       /* 0: no bigram embedding; row (previous mul_prev + token mul_cur) mod buckets, first token: row `buckets` */
    int64_t bigram_mul_prev, bigram_mul_cur;
    int32_t max_positions;                        /* 0: no learned positions; otherwise also the longest sequence */
    int32_t dtype;                                /* MMI_BF16 or MMI_F32: operands of the matrix products, activations and cache */
    int32_t cache;                                /* keys and values of MMI_TLM_MIX_ATTENTION layers: 0 like the operands, MMI_I8 or MMI_F8E4M3: in 8 bits */
} mmi_tlm_cfg;

typedef struct mmi_tlm mmi_tlm;

/* Tensors are bf16 (tables int32), device pointers, copied or repacked: `embed`, `bigram`, `pos`, `head`, `final.norm`, `loop.in`,
 * `loop.step`, per layer `l<i>.norm1`, `.norm2`, `.ls1`, `.ls2`, `.mix.*`, `.mlp.*`.  max_slots: live sequences; max_tokens: cache pool (rounded up to pages); max_step_tokens: tokens of
 * one step. */
int mmi_tlm_create(const mmi_tlm_cfg* cfg, const mmi_tensor_desc* weights, int32_t n_weights, int32_t max_slots, int64_t max_tokens,
                   int32_t max_step_tokens, mmi_tlm** out);
void mmi_tlm_destroy(mmi_tlm* m);
/* Admit a sequence (MMI_ERR_BUSY when every slot is taken) / give back what it holds. */
int mmi_tlm_open(mmi_tlm* m, int32_t* slot);
int mmi_tlm_close(mmi_tlm* m, int32_t slot);
/* One batch: entry e appends counts[e] tokens to slot slots[e] (each slot at most once).  tokens: host, concatenated; -1 = the token
 * mmi_tlm_sample last drew for that slot.  want: host, ascending rows of the concatenation whose logits are written to `logits`
 * (device fp32 [n_want][vocab]).  MMI_ERR_BUSY, with nothing changed, when the pool has too few free pages. */
int mmi_tlm_step(mmi_tlm* m, int32_t n_entries, const int32_t* slots, const int32_t* counts, const int32_t* tokens, int32_t n_want,
                 const int32_t* want, float* logits, mmi_stream stream);
/* Beams: in each of `groups` groups of `beams` <= 32 open sequences (slots, host [groups][beams], each slot at most once) the sequence in place i
 * becomes a copy of what the one in place parents[i] (host, 0 .. beams - 1) was: tokens, position, cache and recurrent state.  Full pages are
 * shared; only the last page, where there is room in it, and the states are copied.  MMI_ERR_BUSY, with nothing changed, when the pool has too few
 * free pages for the copies. */
int mmi_tlm_reorder(mmi_tlm* m, int32_t groups, int32_t beams, const int32_t* slots, const int32_t* parents, mmi_stream stream);
/* Draw one token per row of device fp32 logits [n][vocab]; row i belongs to slot slots[i] and uses temp[i] / top_k[i] (temp <= 0:
 * greedy).  out: device int32 [n]. */
int mmi_tlm_sample(mmi_tlm* m, int32_t n, const float* logits, const int32_t* slots, const float* temp, const int32_t* top_k, uint64_t seed,
                   int32_t* out, mmi_stream stream);
/* Bookkeeping: pool and slots.  MMI_TLM_POSITION / MMI_TLM_HELD_PAGES take a slot. */
#define MMI_TLM_PAGE_TOKENS 0
#define MMI_TLM_TOTAL_PAGES 1
#define MMI_TLM_FREE_PAGES 2
#define MMI_TLM_FREE_SLOTS 3
#define MMI_TLM_POSITION 4
#define MMI_TLM_HELD_PAGES 5
#define MMI_TLM_WEIGHT_BYTES 6
#define MMI_TLM_LAYER_RUNS 7
#define MMI_TLM_GRAPHS 8
int64_t mmi_tlm_info(const mmi_tlm* m, int32_t which, int32_t slot);
/* Pages a sequence would have to be given to grow from its position by n tokens (slot < 0: from an empty slot). */
int64_t mmi_tlm_pages_needed(const mmi_tlm* m, int32_t slot, int64_t n);
/* Residual stream after every layer run of the next steps: taps = device fp32 [layer runs][tokens of the step][width], or NULL. */
int mmi_tlm_set_taps(mmi_tlm* m, float* taps);
/* "site\tkernel\tbytes" per launch of the last step. */
int64_t mmi_tlm_launch_list(const mmi_tlm* m, char* buf, int64_t cap);

/* ------------------------------------------------------------------------------------------ */
/* Key/value cache in 8 bits, by itself                                                       */
/* ------------------------------------------------------------------------------------------ */
/* Pages of 64 tokens: key codes [pages][kv_heads][64][dim], value codes [pages][kv_heads][vdim][64] (aligned to 16 bytes), scales
 * [pages][kv_heads][4], one per 16 tokens and head.  A value is code * scale.  The arrays are the caller's; the device is the one they
 * are on, and it has to be the current one. */
typedef struct mmi_kv_cache {
    void *k, *v;
    float *k_scale, *v_scale;
    int64_t pages;
    int32_t kv_heads, dim, vdim;                  /* head sizes: multiples of 16 up to 256 */
    int32_t codes;                                /* MMI_I8 or MMI_F8E4M3 */
    int32_t rot_dim;                              /* leading dimensions of keys and queries that are rotated, a multiple of 8; 0: none */
    int32_t rot_halves;                           /* partners half of them apart; 0: side by side */
    const double* rot_freq;                       /* device [rot_dim / 2]: turns per position */
} mmi_kv_cache;
/* The sequences of a call, all of it in device memory: sequence e brings rows row0[e] .. row0[e + 1] - 1 of the tensors, its positions
 * position[e] .., and finds position p in page table[e][p / 64].  row0 NULL: one row each, in order.  A page number outside the cache
 * holds nothing: rows that belong there are not written, and nobody sees its tokens.  A sequence with a negative position is passed over.  Calls without a
 * sequence (n 0) do nothing. */
typedef struct mmi_kv_seqs {
    int32_t n, rows;                              /* sequences, rows of the tensors */
    const int32_t* row0;
    const int32_t* position;
    const int32_t* table;
    int32_t table_ld;
} mmi_kv_seqs;
/* Rotate the keys, round keys and values to 8 bits and write them to their pages.  dtype: MMI_BF16 or MMI_F32, strides in elements, a
 * head's dimensions side by side.  A block's scale is the largest magnitude it was handed / the largest code (127, 448); where a token makes
 * it grow, the codes that the block holds of earlier positions are rounded again.  A NaN or infinity makes the block's scale NaN.  The pages
 * that two sequences of a call write to are different ones. */
int mmi_kv_append(const mmi_kv_cache* cache, const mmi_kv_seqs* seqs, int32_t dtype, const void* k, int64_t k_row, int64_t k_head, const void* v, int64_t v_row,
                  int64_t v_head, mmi_stream stream);
/* What the cache holds for those rows: k [rows][kv_heads][dim], v [rows][kv_heads][vdim]; zeros where there is no page, and in rows that no sequence
 * brings (one that is passed over brings none). */
int mmi_kv_read(const mmi_kv_cache* cache, const mmi_kv_seqs* seqs, int32_t dtype, void* k, void* v, mmi_stream stream);
/* out = softmax(scale q k^T) v over the positions up to a row's own; window > 0: the last `window` of them and the first `keep_first`;
 * MMI_KV_SINK: one is added to the softmax's denominator; MMI_KV_ZERO_REST: rows that no sequence brings (one that is passed over brings none)
 * become zeros, where they otherwise stay as they were.  Query head h reads key/value head h / (heads / kv_heads).  Sums are
 * fp32; bf16 queries and the weights beside them are fp16 operands, fp32 ones two fp16 parts each (22 bits).  A row that sees nothing gets zeros.
 * The output's heads lie apart, within rows or rows within heads, four elements aligned.  workspace: device memory of mmi_kv_attend_workspace bytes
 * (a negative status in its place where the arguments are refused), one per call in flight. */
enum { MMI_KV_SINK = 1, MMI_KV_ZERO_REST = 2 };
int64_t mmi_kv_attend_workspace(const mmi_kv_cache* cache, const mmi_kv_seqs* seqs, int32_t heads, int32_t window, int32_t keep_first);
int mmi_kv_attend(const mmi_kv_cache* cache, const mmi_kv_seqs* seqs, int32_t dtype, int32_t heads, const void* q, int64_t q_row, int64_t q_head, void* out,
                  int64_t out_row, int64_t out_head, float scale, int32_t window, int32_t keep_first, int32_t flags, void* workspace, int64_t workspace_bytes,
                  mmi_stream stream);

/* ------------------------------------------------------------------------------------------ */
/* Beam search                                                                                */
/* ------------------------------------------------------------------------------------------ */
/* Of every request's beams x vocab candidates the `beams` best.  Candidate (beam, token): score + log softmax(logits)[token], ranked by
 * score / length^length_penalty (-16 .. 16), length counting the token; equal ranks go to the lower beam, then the lower token.  A finished beam has one
 * candidate, `eos` at the score and the length it has.  Rows with a NaN, and beams of score -infinity, rank last.  Device memory all of it:
 * logits bf16 or fp32 [batch * beams][vocab], `row` elements apart; score, out_* [batch][beams]; length (NULL: no penalty), finished (NULL:
 * none is) and the outputs of either kind may be NULL.  At most 32 beams. */
int64_t mmi_beam_select_workspace(int32_t batch, int32_t beams, int32_t vocab);
int mmi_beam_select(int32_t batch, int32_t beams, int32_t vocab, int32_t dtype, const void* logits, int64_t row, const float* score, const int32_t* length,
                    const uint8_t* finished, int32_t eos, float length_penalty, float* out_score, int32_t* out_parent, int32_t* out_token, uint8_t* out_finished,
                    int32_t* out_length, void* workspace, int64_t workspace_bytes, mmi_stream stream);
/* Row b * beams + i of every tensor (host arrays: device pointers, bytes from row to row, bytes of a row) becomes a copy of what row
 * b * beams + parents[b][i] was; in place.  parents: device int32 [batch][beams]; one outside the request leaves its row alone.  At most 2^16
 * tensors, which share no memory with one another or with the parents: their ranges are apart, or they are as far from row to row and their rows apart
 * (views of one buffer).  Ranges that overlap with other distances are refused. */
int mmi_beam_reorder(int32_t n, void* const* tensors, const int64_t* strides, const int64_t* row_bytes, int32_t batch, int32_t beams, const int32_t* parents,
                     mmi_stream stream);

#ifdef __cplusplus
}
#endif
#endif /* MOSHI_TLM_H_ */

/*
 * gptoss_decode_b200.h - C ABI of the batched greedy decode step around the MoE block.
 *
 * One call = one token for each of up to max_batch sequences: embedding gather,
 * and per layer RMSNorm, QKV projection + bias, YaRN rotary embedding, KV-cache
 * append, attention over the cache with a per-head sink logit (128-token sliding
 * window on even layers), output projection + bias + residual, RMSNorm, the MoE
 * block (gptoss_moe_b200.h), then the final RMSNorm, the logits and their argmax.
 * It replaces gpu_forward_device_batch of the reference's getp engine
 * (getp-csrc/getp_run.cpp:501-894) and computes what forward() computes for one
 * sequence (run.cpp:536-766), for every row of the batch.
 *
 * The QKV and attention-output projections and the logits run on the library's
 * tcgen05 CTA-pair kernel (the grouped GEMM of the MoE block with one group: bias in
 * the epilogue, bf16 output; fp32 output for the logits, which the argmax needs in
 * fp32).  Shapes that kernel does not take (projection rows that are not multiples of
 * 8 elements, a vocabulary that is not a multiple of 4) fall back to cuBLAS, loaded
 * with dlopen on first need.  Activations between kernels: the residual stream, the normalised
 * rows and the projection outputs are bf16, q and the logits fp32, the KV cache bf16.
 */
#ifndef GPTOSS_DECODE_B200_H
#define GPTOSS_DECODE_B200_H

#include "gptoss_moe_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* The reference's Config, which is also the header of the .bin checkpoint
 * (run.cpp:26-46): 15 four-byte fields in this order. */
typedef struct {
  int vocab_size;
  int hidden_dim;
  int n_experts;
  int experts_per_token;
  int intermediate_dim;
  int n_layers;
  int head_dim;
  int n_attn_heads;
  int n_kv_heads;
  int seq_len;
  int initial_context_length;
  float rope_theta;
  float rope_scaling_factor;
  int sliding_window;
  float swiglu_limit;
} gptoss_model_config_t;

/* The reference's TransformerWeights (run.cpp:48-84): fp32 tensors on the host,
 * normally pointers into the mmap of the .bin file.  Shapes as in run.cpp:207-248. */
typedef struct {
  const float *token_embedding_table; /* [V, H] */
  const float *rms_attn_w;            /* [L, H] */
  const float *rms_ffn_w;             /* [L, H] */
  const float *w_qkv;                 /* [L, (Hq + 2 Hkv) D, H], rows q | k | v */
  const float *w_o;                   /* [L, H, Hq D] */
  const float *b_qkv;                 /* [L, (Hq + 2 Hkv) D] */
  const float *b_o;                   /* [L, H] */
  const float *attn_sinks;            /* [L, Hq] */
  const float *w_router;              /* [L, E, H] */
  const float *b_router;              /* [L, E] */
  const float *w_mlp1;                /* [L, E, 2 IM, H], gate rows even, up rows odd */
  const float *w_mlp2;                /* [L, E, H, IM] */
  const float *b_mlp1;                /* [L, E, 2 IM] */
  const float *b_mlp2;                /* [L, E, H] */
  const float *rms_out_w;             /* [H] */
  const float *out;                   /* [V, H] unembedding */
} gptoss_model_weights_t;

typedef struct gptoss_decode gptoss_decode_t;

/* Number of visible CUDA devices of compute capability 10.x (0 when there is none or
 * no driver). */
int gptoss_decode_device_count(void);

/* Allocates everything for max_batch sequences of up to cfg->seq_len positions on
 * `device` (KV cache: L * max_batch * seq_len * Hkv * D * 2 bf16).  No CPU
 * fallback: fails unless the device is sm_100. */
int gptoss_decode_create(const gptoss_model_config_t *cfg, int max_batch, int device,
                         gptoss_decode_t **out);
/* The same with the experts sharded over ep_size ranks (expert e on rank e % ep_size,
 * everything else replicated; getp-csrc/expert.cpp:709-1018).  After creation every
 * rank calls gptoss_moe_ep_init(gptoss_decode_moe(h), id); the ranks then step in lock
 * step, each on its own batch. */
int gptoss_decode_create_ep(const gptoss_model_config_t *cfg, int max_batch, int device,
                            int ep_rank, int ep_size, gptoss_decode_t **out);
int gptoss_decode_destroy(gptoss_decode_t *h);
/* Error text of the last failed call on this handle (or of the last failed create
 * when h is NULL). */
const char *gptoss_decode_last_error(const gptoss_decode_t *h);

/* Converts and uploads every tensor (fp32 host -> bf16 device, biases and norm
 * scales stay fp32); replaces init_device_context (getp_run.cpp:150-302). */
int gptoss_decode_load_weights(gptoss_decode_t *h, const gptoss_model_weights_t *w);
/* The same from the address of the first tensor of a .bin image (file base + 60
 * bytes), tensors in the file's order (memory_map_weights, run.cpp:207-248). */
int gptoss_decode_load_bin(gptoss_decode_t *h, const float *first_tensor);

/* One tensor at a time, for models too large for a host image: name = a field of
 * gptoss_model_weights_t outside the MoE block ("token_embedding_table", "out",
 * "rms_out_w"; per layer "w_qkv", "b_qkv", "w_o", "b_o", "attn_sinks", "rms_attn_w",
 * "rms_ffn_w"), src = that tensor (one layer of it) as fp32 on the host, or on the
 * device as bf16 (weights) / fp32 (biases, scales, sinks).  The MoE tensors go through
 * gptoss_moe_load_layer_* on gptoss_decode_moe(h). */
int gptoss_decode_set_tensor(gptoss_decode_t *h, const char *name, int layer, const void *src,
                             int on_device, int is_bf16);
/* Writes K and V (bf16 device arrays [n_rows, n_pos, Hkv * D], K already rotated) into
 * the cache of `layer` for rows row0.. and positions pos0..: a context without running
 * the prompt (benchmarks with synthetic contexts). */
int gptoss_decode_set_kv(gptoss_decode_t *h, int layer, int row0, int n_rows, int pos0, int n_pos,
                         const void *k_dev, const void *v_dev);
/* The reverse: copies that region of the cache out (moving a sequence to another row or
 * another engine). */
int gptoss_decode_get_kv(gptoss_decode_t *h, int layer, int row0, int n_rows, int pos0, int n_pos,
                         void *k_dev, void *v_dev);

/* One step.  tokens[i] / pos[i]: the token to feed to batch row i and its position
 * (host arrays); pos[i] < 0 marks a row that does no work (its cache is untouched
 * and next[i] = -1), the reference's inactive-row rule.  Row i owns KV-cache slot
 * i; a sequence starts over simply by feeding pos 0 again.  next[i] receives the
 * argmax of the row's logits (lowest index among equals, sample_argmax,
 * run.cpp:780-791).  Synchronises the stream before returning. */
int gptoss_decode_step(gptoss_decode_t *h, const int *tokens, const int *pos, int batch,
                       int *next, void *stream);
/* fp32 logits [vocab_size] of batch row `row` from the last step (after a prefill: of the last
 * token of its sequence number `row`). */
int gptoss_decode_get_logits(gptoss_decode_t *h, int row, float *logits_host);

/* How next tokens are drawn (host arrays, one entry per row of the step or per sequence of the
 * prefill; NULL: 1, no limit, no limit, no limit; u is required): see gptoss_decode_sample. */
typedef struct {
  const float *u;
  const float *temperature;
  const int *top_k;
  const float *top_p;
  const float *min_p;
} gptoss_decode_sampling_t;
/* gptoss_decode_step with the next tokens drawn instead of taken as argmax (sampling NULL: the
 * same as gptoss_decode_step). */
int gptoss_decode_step_sample(gptoss_decode_t *h, const int *tokens, const int *pos, int batch,
                              const gptoss_decode_sampling_t *sampling, int *next, void *stream);

/* An engine whose passes take up to max_tokens rows (at least max_batch): prompts are fed
 * max_tokens tokens at a time by gptoss_decode_prefill.  Engines of the other create calls have
 * max_tokens = max_batch.  All experts local. */
int gptoss_decode_create_prefill(const gptoss_model_config_t *cfg, int max_batch, int max_tokens,
                                 int device, gptoss_decode_t **out);
/*
 * Whole prompts instead of a token per step (the reference feeds them through its decode
 * step, getp_run.cpp:969-979).  Sequence i of n_seqs owns the next lens[i] entries of `tokens`
 * (packed, host) and goes to cache row rows[i], positions pos0[i] .. pos0[i] + lens[i] - 1;
 * pos0[i] > 0 continues what that row holds.  The rows of one call are different.  next[i]
 * receives the token after the last one of sequence i: the argmax, or drawn as `sampling` says.
 * Same arithmetic as the step except in the attention: the order of its sums, its exponentials
 * (see gptoss_decode_prompt_attention), and q, which the step multiplies by 1 / sqrt(head_dim)
 * before it rounds it to bf16 and the prefill rounds unscaled (the same bits where head_dim is
 * 64).  The cache it leaves is what the steps leave, but for roundings that fall the other way.
 * Prompts longer than max_tokens, and as many of them as do not fit, go through in several
 * passes.  All tokens and positions are checked first; a call that is refused has changed
 * nothing.  Synchronises the stream.  Not under expert parallelism (GPTOSS_E_STATE).
 */
int gptoss_decode_prefill(gptoss_decode_t *h, const int *tokens, const int *rows, const int *pos0,
                          const int *lens, int n_seqs, const gptoss_decode_sampling_t *sampling,
                          int *next, void *stream);
/* The MoE engine inside (for its options, taps and stage timers). */
gptoss_moe_t *gptoss_decode_moe(gptoss_decode_t *h);

/*
 * The operators of a prompt pass and of a drawn token, without a handle: every pointer is a
 * device pointer owned by the caller, all on one GPU (which need not be the current one;
 * `stream` belongs to it, NULL = its default stream).  The calls allocate nothing, keep
 * nothing between calls, do not synchronise and may be captured into CUDA graphs; calls on
 * different streams or threads are independent.  They return 0 or a negative GPTOSS_E_*
 * code with the text in gptoss_decode_last_error(NULL), and launch nothing when they fail.
 * `status` fields are optional device words in which a kernel leaves a code of
 * gptoss_moe_device_status (first writer wins; the caller clears it).
 */
enum { GPTOSS_DTYPE_BF16 = 0, GPTOSS_DTYPE_FP16 = 1, GPTOSS_DTYPE_FP32 = 2 };

/*
 * Rotary frequencies: inv_freq [rotary_dim / 2] (host) and the factor on cosine and sine,
 * as the engine computes them from its config (run.cpp:423-474): theta^(-2i / rotary_dim),
 * and for scaling_factor > 1 the YaRN interpolation over initial_context_length.
 */
int gptoss_decode_rope_table(int rotary_dim, float theta, float scaling_factor,
                             int initial_context_length, float *inv_freq_host,
                             float *concentration);

/*
 * Rotary positions on the rows of a batch and the append to the KV cache: what the decode
 * step does to one projection output per sequence (run.cpp:575-596), for any number of
 * rows.  Row i has its position pos[i]; rows with pos[i] < 0 are skipped.  With
 * a = pos[i] * inv_freq[j] and (c, s) = concentration * (cos a, sin a), the pairs (x1, x2) of
 * the first rotary_dim elements of every q and k head become (x1 c - x2 s, x2 c + x1 s); the
 * pair j is elements (j, j + rotary_dim / 2), or (2j, 2j + 1) when `interleaved`; the rest of
 * a head is copied, and so is v.  The arithmetic is fp32, rounded once to the type.
 *   q  [n_rows, n_q_heads, head_dim] -> q_out (same shape; may be q itself)
 *   k  [n_rows, n_kv_heads, head_dim] -> rows of k_cache [n_slots, n_kv_heads, head_dim]
 *   v  likewise -> v_cache
 * Heads are contiguous, rows are `*_stride` elements apart (a row of q | k | v as the
 * projection leaves it: all three strides are its length).  slots[i] is the cache row of row
 * i; NULL: row i (n_slots >= n_rows then).  A row whose slot is outside [0, n_slots) is not
 * stored.  Two rows with one slot leave one of them there, element by element undefined.
 * q (with q_out), k (with k_cache) and v (with v_cache) may each be NULL.  k_cache may be k
 * itself (and v_cache v) when slots is NULL; other overlaps of inputs and outputs are not allowed.
 * angle_f32 = 0: the angle is formed in fp64 (exact for every position); 1: pos * inv_freq
 * is rounded to fp32 first, as the reference and gptoss_decode_step do.
 */
typedef struct {
  const void *q, *k, *v;
  void *q_out, *k_cache, *v_cache;
  const int *pos;             /* [n_rows] */
  const long long *slots;     /* [n_rows] or NULL */
  const float *inv_freq;      /* [rotary_dim / 2], device */
  long long q_stride, k_stride, v_stride, q_out_stride, k_cache_stride, v_cache_stride;
  long long n_slots;
  float concentration;
  int n_rows, n_q_heads, n_kv_heads, head_dim, rotary_dim;
  int interleaved, angle_f32, dtype;
} gptoss_rope_args_t;
int gptoss_decode_rope_append(const gptoss_rope_args_t *args, void *stream);

/*
 * Attention of packed query rows over K / V rows that are in place (a cache, or the packed
 * keys and values of the same prompts): a whole prompt, a piece of one on top of its context,
 * single tokens, or any mixture, in one launch.  It computes for every row what the decode
 * step computes for one (run.cpp:601-647): causal, grouped heads (query head h reads KV head
 * h / (n_q_heads / n_kv_heads)), an optional sink logit per query head that takes probability
 * mass and has no value, an optional sliding window.
 *   q, out  [n_tokens, n_q_heads, head_dim]; sequence i owns rows q_start[i] .. q_start[i+1]
 *   k, v    [n_kv_rows, n_kv_heads, head_dim]; its keys are rows kv_start[i] .. + kv_len[i]
 * The last query of a sequence stands at its last key: query j of L sees key t when
 * t <= p and (window == 0 or t > p - window), p = kv_len[i] - L + j.  A query that sees no
 * key (kv_len[i] < L leaves p < 0) gets zeros.  bf16 or fp16, maxima and sums in fp32; the
 * exponentials are good to 2^-22 relative, with many query rows per sequence some of them to
 * 7.5e-5 in bf16 and 2.6e-6 in fp16; the probabilities are rounded to the type before they
 * multiply v, the result once at the end.  Scores scale * q.k are below 2^26 in magnitude.
 * K and V rows outside every sequence, or that no query of a sequence sees, may hold
 * anything (NaN included); those that some query sees must be finite.
 * Heads are contiguous, rows are `*_stride` elements apart; addresses and strides in bytes
 * are multiples of 16.  head_dim 32, 64 or 128; n_q_heads a multiple of n_kv_heads, at most
 * 128 times it; out does not overlap the inputs.  q_start is ascending from 0; its last entry
 * may be below n_tokens.  A sequence whose keys leave [0, n_kv_rows) or whose kv_len is negative
 * is left unwritten and reported as status 104; so are entries of q_start that do not ascend or
 * pass n_tokens, and then it is open which rows of out are written.  kv_start and kv_len of a
 * sequence without query rows are not looked at.  Rows that belong to no sequence are left
 * unwritten.  Sinks are finite or -infinity (no sink); scale is positive and finite.
 * max_kv_len: an upper bound on kv_len that the host knows (0 = not known); it only chooses
 * how the work is split.  (Query rows on more than 10^8 keys may outlast the kernel's waits of
 * 2 s: status 101 to 103, rows unwritten.)
 * One of two kernels takes the whole call: one for single tokens where the sequences, empty ones
 * included, have on average no more query rows than 16 / (n_q_heads / n_kv_heads), else one for
 * prompts.  A long prompt with many single tokens beside it is right either way, but faster as
 * two calls.
 */
typedef struct {
  const void *q, *k, *v;
  void *out;
  const int *q_start;         /* [n_seqs + 1] */
  const long long *kv_start;  /* [n_seqs] */
  const int *kv_len;          /* [n_seqs] */
  const float *sinks;         /* [n_q_heads] or NULL */
  int *status;                /* or NULL */
  long long q_stride, k_stride, v_stride, out_stride;
  long long n_kv_rows;
  float scale;                /* on q . k, 1 / sqrt(head_dim) as a rule */
  int n_tokens, n_seqs, n_q_heads, n_kv_heads, head_dim;
  int window, max_kv_len, dtype;
} gptoss_attention_args_t;
int gptoss_decode_prompt_attention(const gptoss_attention_args_t *args, void *stream);

/*
 * The next token of every row, drawn from its logits with given uniform numbers (the step's
 * argmax is the greedy case; the reference samples on the host, run.cpp:780-910).  For a
 * row with temperature T > 0, weights w_i = exp((logit_i - max) / T); tokens are ordered by
 * logit, largest first, lowest id first among equals, and the kept set is the longest prefix
 * of that order that satisfies, in turn,
 *   top_k:  at most top_k[r] tokens (<= 0 or >= vocab: no limit);
 *   top_p:  the weight in front of a token, among those that top_k kept, is below top_p[r]
 *           times their total (>= 1: no limit; the first token always stays);
 *   min_p:  w_i >= min_p[r] (w of the likeliest token is 1, which stays; <= 0: no limit).
 * A NaN in one of the last two is no limit either.
 * next[r] is the lowest kept id whose running sum of kept weights, in the order of the ids,
 * exceeds u[r] times their total, u in [0, 1) (values outside are clamped, NaN counts as 0).
 * T <= 0 or NaN: the largest logit, lowest id among equals; above 1e36 it counts as 1e36.
 * NaN logits count as -infinity, which is never drawn; a row with nothing else gives 0, as the
 * argmax of the step does.  Where logits are +infinity those alone are kept, with equal weight,
 * as far as top_k and top_p leave them.  Rows with pos[r] < 0 give -1.
 * Weights are formed in fp64 and summed as multiples of 2^-44 in 64-bit integers, so sums do
 * not depend on their order and a draw does not either; a weight below 2^-45 counts as 0.
 * logits [n_rows, vocab], rows `stride` elements apart, in bf16, fp16 or fp32; vocab up to
 * 2^18.  temperature, top_k, top_p, min_p, u: device arrays of n_rows (NULL: 1, no limit, no
 * limit, no limit; u is required).
 */
typedef struct {
  const void *logits;
  const float *u;
  const float *temperature;   /* or NULL */
  const int *top_k;           /* or NULL */
  const float *top_p;         /* or NULL */
  const float *min_p;         /* or NULL */
  const int *pos;             /* or NULL */
  int *next;                  /* [n_rows] */
  long long stride;
  int n_rows, vocab, dtype;
} gptoss_sample_args_t;
int gptoss_decode_sample(const gptoss_sample_args_t *args, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* GPTOSS_DECODE_B200_H */

/*
 * localfold.h - C ABI of the MI355X (gfx950) pair-stack library, liblocalfold.so.
 *
 * The reference (sokrypton/localfold) exposes this path as JavaScript classes over
 * WebGPU (webgpu/index.js:1-8): TriangleMultiplication{Outgoing,Incoming}Gpu, AttentionGpu,
 * OuterProductMeanGpu, TransitionGpu, EvoformerBlockGpu, EvoformerStackGpu, plus the AF3
 * trunk classes (webgpu/af3/trunk/).  Each entry point below is what a binding of one of
 * those classes' `run()` calls once its input has been validated and copied to the device;
 * the citation on each names the reference interface it replaces.
 *
 * Conventions
 *  - Every tensor pointer is a DEVICE pointer (hipMalloc'd, or a torch CUDA tensor's
 *    data_ptr); shapes are plain ints; work is enqueued on the context's stream and the
 *    call returns without waiting (lf_synchronize waits).
 *  - Activation dtype codes: LF_F32, LF_F16, LF_BF16.  Layer-norm scales/offsets, biases
 *    and masks are always float32 (the reference keeps them float32:
 *    tools/quantize_af3.py:57, KEEP_FLOAT32).
 *  - Weights are lf_weight records: float32/float16/bfloat16 values, or the reference's
 *    codecs decoded on the device - int8 symmetric (code*scale) and int5 asymmetric
 *    (code*scale+zero, LSB-first 5-bit codes, one slack byte), fp16 scale/zero tables
 *    (shared/weights/dtype.js:212-406) - inside the triangle-multiplication kernels and the
 *    weight-resident output projections as they stage them into LDS, and by one short
 *    per-call pass for the streaming projections, transitions and OPM.  `group` > 0 is the reference's flat group map
 *    (group index = flat stored index / group: 64 for int8, 32 for int5); `group` == 0
 *    is one group per output channel.
 *  - Return value: LF_OK, or an error code; lf_last_error() holds the message
 *    (thread-local).  Invalid shapes are rejected before anything is enqueued, the way
 *    the reference's validate() throws a RangeError (webgpu/kernels/triangle/types.js:13-48).
 *  - "accumulate" = 0 writes the op's update (what the reference's class returns);
 *    1 writes input + update into `out`, which may alias the input (the in-place residual
 *    of webgpu/af2/evoformer/block.js:1536-1629).
 */
#ifndef LOCALFOLD_H
#define LOCALFOLD_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct lf_context lf_context;

enum { LF_OK = 0, LF_ERR_INVALID = 1, LF_ERR_DEVICE = 2, LF_ERR_MEMORY = 3, LF_ERR_UNSUPPORTED = 4 };
enum { LF_F32 = 0, LF_F16 = 1, LF_BF16 = 2, LF_INT8 = 3, LF_INT5 = 4 };
enum { LF_IN_OUT = 0, LF_OUT_IN = 1 };
enum { LF_OUTGOING = 0, LF_INCOMING = 1 };
enum { LF_AF2 = 0, LF_AF3 = 1 };

/* One stored weight tensor: `rows` x `cols` in storage order.  LF_IN_OUT: rows = inputs,
 * cols = outputs (Haiku / AF3 layout).  LF_OUT_IN: rows = outputs, cols = inputs (the
 * (out,in) layout of webgpu/kernels/triangle/types.js:28-43). */
typedef struct {
  int dtype;            /* LF_F32 / LF_F16 / LF_BF16 / LF_INT8 / LF_INT5 */
  int layout;           /* LF_IN_OUT or LF_OUT_IN */
  int rows, cols;
  int group;            /* quantised only: flat group size, or 0 = per output channel */
  const void* data;     /* values, or codes; int5 codes must stay readable for 4 bytes past
                           the last code byte (the reference's records hold a slack byte and
                           the scale table there; the kernels fetch aligned word pairs) */
  const void* scales;   /* fp16, one per group (quantised) */
  const void* zeros;    /* fp16, one per group (int5) */
} lf_weight;

/* ---- context, memory, stream, timing ------------------------------------------------- */

/* Replaces the WebGPU device of webgpu/node.js:51-81 / webgpu/runtime/device.js:98. */
lf_context* lf_context_create(int device_ordinal);
void lf_context_destroy(lf_context* ctx);
/* Enqueue on an existing hipStream_t (e.g. torch's current stream); NULL is the HIP null stream.
 * A new context starts on a non-blocking stream of its own. */
int lf_context_set_stream(lf_context* ctx, void* hip_stream);
const char* lf_last_error(void);
const char* lf_version(void);

/* Device memory owned by the caller (webgpu/runtime/allocator.js:55 GpuBufferAllocator). */
int lf_malloc(lf_context* ctx, size_t bytes, void** out);
int lf_free(lf_context* ctx, void* ptr);
int lf_memcpy_htod(lf_context* ctx, void* dst, const void* src, size_t bytes);
int lf_memcpy_dtoh(lf_context* ctx, void* dst, const void* src, size_t bytes);
int lf_memset(lf_context* ctx, void* dst, int value, size_t bytes);
int lf_synchronize(lf_context* ctx);
/* {currentBytes, peakBytes, allocationCount} of webgpu/runtime/allocator.js:188-194,
 * counting caller allocations, the context's scratch workspace and its mask tables.  Not
 * counted: the library's static LF_TRI_NOALLOC_SCRATCH_BYTES array, which every device the
 * library loads on holds until the process ends (see lf_tri_mult_noalloc). */
int lf_memory_stats(lf_context* ctx, size_t* current_bytes, size_t* peak_bytes, size_t* allocation_count);

/* Per-kernel timestamps (webgpu/runtime/execution.js:673-727 readTimestampProfile):
 * when enabled, every kernel launch is bracketed by hipEvents on the context stream. */
typedef struct {
  char label[48];
  float ms;
} lf_kernel_timing;
int lf_profile_enable(lf_context* ctx, int enable);
/* Waits for the stream, copies up to `max` records, returns the count (and clears them). */
int lf_profile_read(lf_context* ctx, lf_kernel_timing* out, int max);

/* ---- triangle multiplicative update -------------------------------------------------- */

/* AF2 (dialect LF_AF2): the sixteen tensors of webgpu/kernels/triangle/types.js:28-43 with
 * projection weights ap, ag, bp, bg [cH x cZ], wz [cZ x cH], wg [cZ x cZ], usually LF_OUT_IN.
 * AF3 (dialect LF_AF3, cpu/af3/trunk/pairformer.js:213-300): no biases, fast-variance LN,
 * `ap` = fused projection [cZ x 2cZ] and `ag` = fused gate [cZ x 2cZ] (a = column 2c,
 * b = column 2c+1), wz = outputProjection, wg = gatingLinear; bp/bg unused. */
typedef struct {
  const float *ln_in_scale, *ln_in_offset;
  lf_weight ap, ag, bp, bg;
  const float *ap_bias, *ag_bias, *bp_bias, *bg_bias;
  const float *ln_out_scale, *ln_out_offset;
  lf_weight wz;
  const float* wz_bias;
  lf_weight wg;
  const float* wg_bias;
} lf_tri_mult_weights;

typedef struct {
  int direction;          /* LF_OUTGOING: x_ij = sum_k a_ik b_jk; LF_INCOMING: sum_k a_kj b_ki */
  int dialect;            /* LF_AF2 or LF_AF3 */
  int divide_by_length;   /* AF3 rf3 dialect: x /= N before the centre norm */
  int length, c_z, c_hidden;
  int act_dtype;
  const void* z;          /* [N, N, cZ] */
  const float* mask;      /* [N, N] */
  void* out;              /* [N, N, cZ], act_dtype */
  int accumulate;
  float epsilon;          /* 1e-5 in the reference */
  const lf_tri_mult_weights* w;
} lf_tri_mult_args;

/* Replaces TriangleMultiplication{Outgoing,Incoming}Gpu.run (webgpu/kernels/triangle/webgpu.js:38-169)
 * and encodeTriangleMultiplication (webgpu/af2/evoformer/block.js:1288-1535). */
int lf_tri_mult(lf_context* ctx, const lf_tri_mult_args* args);

/* No counterpart in the reference: lf_tri_mult for callers that cannot allocate device memory
 * (code under HIP graph capture, tight serving loops, harnesses that forbid hipMalloc).  Same
 * arguments, kernels and results as lf_tri_mult, but its scratch (the a, b and X planes,
 * 3 * c_hidden * N^2 f16, plus 8 * N^2 bytes of LayerNorm statistics with 2-byte activations
 * at c_z = c_hidden = 128; weights are decoded while being staged into LDS, so they take no
 * scratch) lives in a static per-device array of LF_TRI_NOALLOC_SCRATCH_BYTES and 6 MiB for the
 * padding of the planes' rows (reserved on every device the library loads on, used or not),
 * looked up once per device by lf_context_create; nothing is allocated or freed.  Shapes needing
 * more scratch are rejected with LF_ERR_INVALID (c_hidden 128 fits N <= 418, but not 416 with
 * 2-byte activations, whose statistics count where whole 16-pair tiles hand them over).  Every
 * call on one GPU shares that GPU's array: calls that overlap on one GPU (two streams, two
 * threads, two contexts) race, so serialise them. */
#define LF_TRI_NOALLOC_SCRATCH_BYTES (128u << 20)
int lf_tri_mult_noalloc(lf_context* ctx, const lf_tri_mult_args* args);

/* ---- gated attention (MSA row / column, triangle starting / ending, AF3 grid / single) -- */

enum { LF_BIAS_NONE = 0, LF_BIAS_SEPARATE = 1, LF_BIAS_NORMALIZED_INPUT = 2, LF_BIAS_LOGITS = 3 };

typedef struct {
  const float *norm_scale, *norm_offset;
  lf_weight wq, wk, wv, wg, wo;          /* [C x H*d] / [H*d x C] in either layout */
  const float *q_bias, *g_bias, *o_bias; /* optional (NULL = none) */
  /* pair bias: LF_BIAS_SEPARATE uses pair_norm_* and wb [Cpair x H];
   * LF_BIAS_NORMALIZED_INPUT uses wb [C x H] on the normalised attention input */
  const float *pair_norm_scale, *pair_norm_offset;
  lf_weight wb;
} lf_attention_weights;

typedef struct {
  int batch, queries, channels, heads;
  int head_dim;           /* 0: channels / heads (AF2) */
  int transpose;          /* logical row (b,q) is storage row (q,b); key mask at [k,b] */
  int act_dtype;
  const void* act;        /* storage [batch*queries, C] (or [queries*batch, C] when transposed) */
  const float* mask;      /* storage order, batch*queries */
  void* out;
  int accumulate;
  int fast_variance;      /* AF3 layer norms */
  int bias_mode;          /* LF_BIAS_* */
  int swap_bias;          /* AF3 openfold dialect: bias[h][i][j] read at [j][i] when transposed */
  int pair_dtype;
  const void* pair;       /* LF_BIAS_SEPARATE: [queries, queries, pair_channels] */
  int pair_channels;
  const float* bias_logits; /* LF_BIAS_LOGITS: [H, queries, queries] float32 */
  float epsilon;
  const lf_attention_weights* w;
} lf_attention_args;

/* Replaces AttentionGpu.run (webgpu/kernels/attention.js:2580-2739) and encodeAttention
 * (webgpu/af2/evoformer/block.js:647-952); AF3 gridSelfAttention / singleAttention
 * (cpu/af3/trunk/pairformer.js:322-485) through the same entry. */
int lf_attention(lf_context* ctx, const lf_attention_args* args);

/* ---- transition ----------------------------------------------------------------------- */

enum { LF_TRANSITION_RELU = 0, LF_TRANSITION_SWIGLU = 1 };

typedef struct {
  const float *norm_scale, *norm_offset;
  lf_weight w1;           /* RELU: [C x H]; SWIGLU: [C x 2H], gate half first (blocked split) */
  const float* b1;
  lf_weight w2;           /* [H x C] */
  const float* b2;
} lf_transition_weights;

typedef struct {
  int kind;               /* LF_TRANSITION_RELU (AF2) or LF_TRANSITION_SWIGLU (AF3) */
  int rows, channels, hidden;
  int act_dtype;
  const void* act;
  void* out;
  int accumulate;
  int fast_variance;
  long long chunk_bytes;  /* hidden-buffer budget per chunk; 0 = 32 MiB (transition.js:377) */
  float epsilon;
  const lf_transition_weights* w;
} lf_transition_args;

/* Replaces TransitionGpu.run (webgpu/kernels/transition.js:1009-1105), encodeTransition
 * (block.js:488-646) and AF3 transition (cpu/af3/trunk/pairformer.js:180-201). */
int lf_transition(lf_context* ctx, const lf_transition_args* args);

/* ---- outer product mean --------------------------------------------------------------- */

typedef struct {
  const float *norm_scale, *norm_offset;
  lf_weight wl, wr;        /* [cM x cOuter] */
  const float *bl, *br;    /* optional */
  lf_weight wo;            /* [cOuter*cOuter x cZ] */
  const float* bo;         /* optional */
} lf_opm_weights;

typedef struct {
  int sequences, length, c_m, c_outer, c_z;
  int msa_dtype;
  const void* msa;         /* [S, N, cM] */
  const float* mask;       /* [S, N] */
  int pair_dtype;
  const void* pair_in;     /* residual source when accumulate (may alias out) */
  void* out;               /* [N, N, cZ] */
  int accumulate;
  int fast_variance;
  float epsilon;           /* layer norm, 1e-5 */
  float norm_epsilon;      /* 1e-3 */
  const lf_opm_weights* w;
} lf_opm_args;

/* Replaces OuterProductMeanGpu.run (webgpu/kernels/outer-product-mean.js:1748-1907) and
 * AF3 outerProductMean (cpu/af3/trunk/msa.js:72-155). */
int lf_outer_product_mean(lf_context* ctx, const lf_opm_args* args);

/* ---- global column attention (AF2 extra-MSA stack) ---------------------------------- */

typedef struct {
  const float *norm_scale, *norm_offset;  /* queryNormScale / queryNormOffset */
  lf_weight wq;             /* [C x H*d] */
  lf_weight wk, wv;         /* [C x d]: one key/value head shared by every query head */
  lf_weight wg;             /* [C x H*d] */
  const float* g_bias;      /* [H*d] */
  lf_weight wo;             /* [H*d x C] */
  const float* o_bias;      /* [C], optional */
} lf_global_attention_weights;

typedef struct {
  int sequences, length, channels, heads;
  int head_dim;             /* 0: channels / heads */
  int act_dtype;
  const void* act;          /* [S, N, C] */
  const float* mask;        /* [S, N] */
  void* out;                /* [S, N, C], act_dtype; may alias act when accumulate */
  int accumulate;
  float epsilon;            /* layer norm, 1e-5 */
  const lf_global_attention_weights* w;
} lf_global_attention_args;

/* Replaces encodeGlobalAttention (webgpu/af2/evoformer/block.js:953-1030) and its kernels
 * (block.js:88-400): per residue column, attention of the masked-mean query over the
 * sequences (a masked sequence's logit is -1e9), gated per sequence, projected out. */
int lf_global_column_attention(lf_context* ctx, const lf_global_attention_args* args);

/* ---- blocks --------------------------------------------------------------------------- */

typedef struct {
  lf_attention_weights row_attention;     int row_heads;
  lf_attention_weights column_attention;  int column_heads;
  lf_transition_weights msa_transition;
  lf_opm_weights outer_product_mean;
  lf_tri_mult_weights tri_out, tri_in;
  lf_attention_weights tri_att_start;     int tri_att_start_heads;
  lf_attention_weights tri_att_end;       int tri_att_end_heads;
  lf_transition_weights pair_transition;
} lf_evoformer_weights;

typedef struct {
  int sequences, length, c_m, c_z, c_outer, tri_hidden, msa_hidden, pair_hidden;
  int msa_dtype;  void* msa;     /* [S, N, cM], updated in place */
  int pair_dtype; void* pair;    /* [N, N, cZ], updated in place */
  const float* msa_mask;         /* [S, N] */
  const float* pair_mask;        /* [N, N] */
  float epsilon;
  const lf_evoformer_weights* w;
} lf_evoformer_block_args;

/* Replaces EvoformerBlockGpu.run / encodeEvoformerBlock (webgpu/af2/evoformer/block.js:1536-1629,
 * 1783-1824): row attention with pair bias, column attention, MSA transition, OPM,
 * triangle multiplication out/in, triangle attention start/end, pair transition. */
int lf_evoformer_block(lf_context* ctx, const lf_evoformer_block_args* args);

/* Replaces EvoformerStackGpu.run (webgpu/af2/evoformer/stack.js:44-160): `blocks` blocks in order. */
int lf_evoformer_stack(lf_context* ctx, const lf_evoformer_block_args* args, const lf_evoformer_weights* blocks,
                       int block_count);

/* The extra-MSA block's weights: the Evoformer block's (column_attention and column_heads
 * unused) with the global column attention in its place. */
typedef struct {
  lf_evoformer_weights base;
  lf_global_attention_weights column_global;
  int column_global_heads;
} lf_extra_msa_weights;

/* Replaces encodeExtraMsaBlock (webgpu/af2/evoformer/block.js:1715-1744): row attention with
 * pair bias, global column attention, MSA transition, then the pair steps of
 * encodeEvoformerPairBlock (block.js:1663-1713).  args->w is not read. */
int lf_extra_msa_block(lf_context* ctx, const lf_evoformer_block_args* args, const lf_extra_msa_weights* w);

/* Replaces ExtraMsaStackGpu.run (webgpu/af2/evoformer/stack.js:249-330): `block_count`
 * extra-MSA blocks in order on the same msa and pair. */
int lf_extra_msa_stack(lf_context* ctx, const lf_evoformer_block_args* args, const lf_extra_msa_weights* blocks,
                       int block_count);

/* Replaces ExtraMsaPairStackGpu.run (webgpu/af2/evoformer/stack.js:163-247), whose blocks
 * are encodeEvoformerPairBlock (webgpu/af2/evoformer/block.js:1663-1713): per block the outer
 * product mean of the (unchanged) msa into the pair, triangle multiplication out/in, triangle
 * attention start/end and the pair transition.  The msa is read, never written; the weights'
 * MSA-side records (row/column attention, MSA transition) are not read. */
int lf_evoformer_pair_stack(lf_context* ctx, const lf_evoformer_block_args* args, const lf_evoformer_weights* blocks,
                            int block_count);

typedef struct {
  lf_tri_mult_weights tri_out, tri_in;
  lf_attention_weights att_start, att_end;  int pair_heads;
  lf_transition_weights pair_transition;
  const float *single_logits_norm_scale, *single_logits_norm_offset;
  lf_weight single_logits_projection;       /* [cZ x Hs] */
  lf_attention_weights single_attention;  int single_heads, single_head_dim;
  lf_transition_weights single_transition;
} lf_pairformer_weights;

typedef struct {
  int tokens, c_z, c_s;
  int swap_transposed_bias, divide_by_length;
  int pair_dtype; void* pair;    /* [N, N, cZ] in place */
  int single_dtype; void* single;/* [N, cS] in place, or NULL for a pair-only block */
  const float* pair_mask;        /* [N, N] */
  const float* seq_mask;         /* [N] */
  long long transition_chunk_bytes;
  float epsilon;
  const lf_pairformer_weights* w;
} lf_pairformer_block_args;

/* Replaces one block of Af3PairformerStackGpu.run (webgpu/af3/trunk/pairformer-block.js:246-308),
 * in pairformerBlock order (cpu/af3/trunk/pairformer.js:495-541). */
int lf_pairformer_block(lf_context* ctx, const lf_pairformer_block_args* args);

/* ---- AF2 input and recycling embedder -------------------------------------------------- */

/* All f32 on the device, (in,out) layout (InputEmbedderGpu's packWeights,
 * webgpu/af2/evoformer/input-embedder.js:9-26). */
typedef struct {
  const float *preprocess_1d_w, *preprocess_1d_b;     /* [Ct x cM], [cM] */
  const float *preprocess_msa_w, *preprocess_msa_b;   /* [Cf x cM], [cM] */
  const float *left_w, *left_b, *right_w, *right_b;   /* [Ct x cZ], [cZ] */
  const float *prev_pos_w, *prev_pos_b;               /* [15 x cZ], [cZ] */
  const float *prev_msa_norm_scale, *prev_msa_norm_offset;    /* [cM] */
  const float *prev_pair_norm_scale, *prev_pair_norm_offset;  /* [cZ] */
  const float *relpos_w, *relpos_b;                   /* [65 x cZ], [cZ] */
  const float *extra_w, *extra_b;                     /* [25 x cE], [cE] */
} lf_input_embedder_weights;

typedef struct {
  int length, msa_sequences, extra_sequences;
  int target_channels, msa_feature_channels;          /* 22, 49 in AF2 */
  int c_m, c_z, c_e;                                  /* 256, 128, 64 */
  const float* target_feat;       /* [L, Ct] */
  const float* msa_feat;          /* [S, L, Cf] */
  const float* extra_msa;         /* [Se, L] residue codes 0..22 as f32 */
  const float* extra_has_deletion;    /* [Se, L] */
  const float* extra_deletion_value;  /* [Se, L] */
  const float* residue_index;     /* [L] */
  const float* aatype;            /* [L] */
  const void* prev_msa_first_row; /* [L, cM], msa_dtype; NULL = zeros (recycle 0) */
  const void* prev_pair;          /* [L, L, cZ], pair_dtype; NULL = zeros */
  const float* prev_positions;    /* [L, 37, 3] atom37; NULL = zeros */
  int msa_dtype;   void* msa;     /* out [S, L, cM] */
  int pair_dtype;  void* pair;    /* out [L, L, cZ]; may alias prev_pair (read and written per row) */
  int extra_dtype; void* extra;   /* out [Se, L, cE] */
  float epsilon;                  /* 1e-5 */
  const lf_input_embedder_weights* w;
} lf_input_embedder_args;

/* Replaces InputEmbedderGpu.run / encodeInputEmbedder (webgpu/af2/evoformer/input-embedder.js:
 * 160-231): the MSA, pair (without templates) and extra-MSA embeddings of one recycle. */
int lf_input_embedder(lf_context* ctx, const lf_input_embedder_args* args);

/* One AF2 recycle of the trunk before the structure module: the input embedder, the
 * extra-MSA stack on the extra activations and the pair, the Evoformer stack on the msa and
 * the pair.  The carried state is the embedder's recycled inputs: point
 * embed.prev_msa_first_row at main.msa and embed.prev_pair at main.pair (they are read before
 * being overwritten) and the outputs of one call are the recycled inputs of the next.
 * extra.msa = embed.extra, extra.pair = main.pair = embed.pair; extra.w and main.w are not
 * read.  Templates and the structure module are out of scope: prev_positions is the
 * caller's (atom37 from its structure module, or NULL for zeros). */
typedef struct {
  lf_input_embedder_args embed;
  lf_evoformer_block_args extra;  const lf_extra_msa_weights* extra_blocks;  int extra_block_count;
  lf_evoformer_block_args main;   const lf_evoformer_weights* main_blocks;   int main_block_count;
} lf_af2_recycle_args;

/* Replaces one iteration of the recycle loop of AlphaFoldMonomerGpu (webgpu/af2/model/
 * monomer.js:182-330) up to the Evoformer stack's output. */
int lf_af2_recycle(lf_context* ctx, const lf_af2_recycle_args* args);

/* ---- AF3 MSA module ------------------------------------------------------------------- */

/* Pair-weighted averaging weights (`msaAttention1`, cpu/af3/trunk/msa.js:157-219), no biases. */
typedef struct {
  const float *act_norm_scale, *act_norm_offset;    /* [cM] */
  const float *pair_norm_scale, *pair_norm_offset;  /* [cZ] */
  lf_weight pair_logits;                            /* [cZ x H] */
  lf_weight wv, wg;                                 /* [cM x H*d] (vProjection, gatingQuery) */
  lf_weight wo;                                     /* [H*d x cM] (outputProjection) */
} lf_pair_averaging_weights;

typedef struct {
  int sequences, tokens, c_m, c_z, heads, head_dim;
  int msa_dtype;
  const void* msa;          /* [S, N, cM] */
  const float* msa_mask;    /* [S, N]; the key mask is its maximum over the sequences */
  int pair_dtype;
  const void* pair;         /* [N, N, cZ] */
  void* out;                /* [S, N, cM], msa_dtype; may alias msa when accumulate */
  int accumulate;
  float epsilon;            /* layer norms (fast variance), 1e-5 */
  const lf_pair_averaging_weights* w;
} lf_pair_averaging_args;

/* Replaces msaAttention (cpu/af3/trunk/msa.js:157-219): softmax over keys j of
 * LN(pair_ij) . pairLogits[:, h] + 1e9 (max_s mask[s, j] - 1), shared by every sequence,
 * averages x vProjection; gated by sigmoid(x gatingQuery), then outputProjection. */
int lf_msa_pair_weighted_averaging(lf_context* ctx, const lf_pair_averaging_args* args);

typedef struct {
  lf_opm_weights outer_product_mean;  int c_outer;   /* AF3 outer product mean */
  lf_pair_averaging_weights msa_attention;  int msa_heads, msa_head_dim;
  lf_transition_weights msa_transition;              /* SwiGLU, hidden 4 cM */
  lf_pairformer_weights pair;                        /* pair steps; the single fields are not read */
} lf_msa_module_weights;

typedef struct {
  int sequences, tokens, c_m, c_z;
  int msa_update_before_opm;     /* 0: AF3 (OPM of the incoming msa first); 1: OpenDDE / Boltz-2 */
  int swap_transposed_bias, divide_by_length;
  int msa_dtype; void* msa;      /* [S, N, cM] in place */
  int pair_dtype; void* pair;    /* [N, N, cZ] in place */
  const float* msa_mask;         /* [S, N] */
  const float* pair_mask;        /* [N, N] */
  long long transition_chunk_bytes;
  float epsilon;
  const lf_msa_module_weights* w;
} lf_msa_block_args;

/* Replaces msaBlock (cpu/af3/trunk/msa.js:233-287): outer product mean into the pair and the
 * MSA update (pair-weighted averaging, SwiGLU transition) in the dialect's order, then the
 * pair steps of a pair-only pairformer block (triangle multiplications, grid attentions,
 * pair transition). */
int lf_msa_module_block(lf_context* ctx, const lf_msa_block_args* args);

/* ---- training: LayerNorm and its gradient, activations kept in 8 bits, 8-bit products ---- */

/* No counterpart in the reference, which runs inference only.  These entry points train a layer
 * of the stack: the forward pass keeps its activations in 8 bits, multiplies them in 8 bits, and
 * the backward pass multiplies what was kept.
 *
 * A checkpoint holds a [rows, cols] matrix as e4m3 codes (4 exponent and 3 mantissa bits, largest
 * 448, no infinity) with one scale per row and group of 128 columns.  The scale is a power of two,
 * 2^(b - 127) with b in 1..254 as stored, the smallest that puts the group's largest finite
 * magnitude within 448 (b = 1 for a group of zeros): the division by it is exact, so the code's
 * rounding (to nearest, ties to even, 2^-4 relative at most above 2^-6 of the scale) is the only
 * one.  An infinity or a NaN becomes the NaN code and leaves its neighbours' scale alone.  A value
 * within 2^-5 of the largest of its type may round up to a power of two beyond it, which reads
 * back as an infinity of that type.
 *
 *   codes   [rows][LF_CHECKPOINT_PITCH(cols)], columns from cols to the pitch hold zeros
 *   scales  [LF_CHECKPOINT_GROUPS(cols)][LF_CHECKPOINT_SCALE_PITCH(rows)], one byte b each; bytes
 *           of rows >= rows may hold anything
 *
 * codes and scales are 16-byte aligned.  An lf_fp8_weight holds an [outputs, inputs] matrix the
 * same way with one scale per tile of 128 x 128: codes [outputs][LF_CHECKPOINT_PITCH(inputs)],
 * scales [LF_CHECKPOINT_GROUPS(outputs)][LF_CHECKPOINT_GROUPS(inputs)].
 *
 * Products of two kept matrices are multiplied in bfloat16, where their values are exact (but for codes
 * below 2^-6 under scale bytes 1 and 2, which become multiples of 2^-133, and values of 2^128 and
 * beyond, which become infinities), and added in f32, whatever the output's type; so are the products
 * inside the transition's step.
 *
 * Matrices are row-major and contiguous, at most 65536 wide (a LayerNorm's rows 4096, weights 65536
 * either way) and of at most 2^34 elements with their columns rounded up to 64.  Inputs and outputs do
 * not overlap except where it says so.  Sums over rows (gradients of weights, biases, scales and offsets) are added in a fixed
 * order: the same call gives the same bits.
 *
 * scratch (lf_layer_norm_backward, lf_fp8_weight_grad, lf_transition_train and _backward): memory
 * for the call's partial sums, at least what the entry point's _scratch function says, 16-byte
 * aligned.  NULL: the context's workspace, which another call may replace: a call that is captured
 * into a HIP graph has to bring its own (LF_ERR_INVALID otherwise), one for each graph that may
 * run at the same time.  lf_fp8_weight_grad over few rows, which it does not split, uses neither. */
typedef struct {
  int rows, cols;
  void* codes;
  void* scales;
} lf_checkpoint;
#define LF_CHECKPOINT_PITCH(cols) (((size_t)(cols) + 63) / 64 * 64)
#define LF_CHECKPOINT_GROUPS(cols) (((size_t)(cols) + 127) / 128)
#define LF_CHECKPOINT_SCALE_PITCH(rows) (((size_t)(rows) + 15) / 16 * 16)

typedef struct {
  int outputs, inputs;
  void* codes;
  void* scales;
} lf_fp8_weight;

typedef struct {
  int act_dtype;
  void* act;                   /* [rows, cols] of `kept`: read by pack, written by unpack */
  const lf_checkpoint* kept;
} lf_checkpoint_args;

/* Activations to a checkpoint, and back to the values that it stands for (rounded to act_dtype;
 * exact in f32, and in bf16 and f16 where those have the range). */
int lf_checkpoint_pack(lf_context* ctx, const lf_checkpoint_args* args);
int lf_checkpoint_unpack(lf_context* ctx, const lf_checkpoint_args* args);

typedef struct {
  int rows, channels;          /* channels 1..4096 */
  int act_dtype;
  const void* act;             /* [rows, channels] */
  const float *scale, *offset; /* [channels] */
  float epsilon;
  int fast_variance;           /* AF3: E[x^2] - E[x]^2 */
  void* out;                   /* [rows, channels], act_dtype, may alias act; or NULL */
  float *mean, *rstd;          /* [rows], for the backward pass; or both NULL */
  const lf_checkpoint* act_kept;  /* act, or NULL */
  const lf_checkpoint* out_kept;  /* the normalised rows (from f32, not from out), or NULL */
} lf_layer_norm_args;

/* out = (act - mean) * rstd * scale + offset; at least one of the outputs is given. */
int lf_layer_norm(lf_context* ctx, const lf_layer_norm_args* args);

typedef struct {
  int rows, channels;          /* channels 1..4096 */
  int act_dtype;               /* of grad, act, residual and out */
  const void* grad;            /* [rows, channels], the gradient of lf_layer_norm's out */
  const void* act;             /* [rows, channels] as in the forward call, or NULL: act_kept */
  const lf_checkpoint* act_kept;
  const float *mean, *rstd;    /* [rows], from the forward call */
  const float* scale;          /* [channels] */
  const void* residual;        /* added to the gradient, or NULL */
  void* out;                   /* [rows, channels], may alias grad, act or residual; or NULL */
  int grad_dtype;              /* of grad_scale and grad_offset */
  void *grad_scale, *grad_offset; /* [channels], or both NULL */
  void* scratch;
  size_t scratch_bytes;
} lf_layer_norm_backward_args;

/* With h = (act - mean) * rstd and g = grad * scale: out = residual + rstd * (g - E[g] - h E[g h]),
 * grad_scale = sum over rows of grad * h, grad_offset = sum over rows of grad. */
int lf_layer_norm_backward(lf_context* ctx, const lf_layer_norm_backward_args* args);
size_t lf_layer_norm_backward_scratch(int rows, int channels);

typedef struct {
  lf_weight w;                 /* LF_F32, LF_F16 or LF_BF16, either layout */
  int backward;                /* 0: out = [outputs of w, inputs of w]; 1: transposed, the operand
                                  of the input's gradient */
  const lf_fp8_weight* out;
} lf_fp8_weight_args;

int lf_fp8_pack_weight(lf_context* ctx, const lf_fp8_weight_args* args);

typedef struct {
  const lf_checkpoint* act;    /* [rows, inputs] */
  const lf_fp8_weight* w;      /* [outputs, inputs] */
  const float* bias;           /* [outputs] or NULL */
  int relu;                    /* values below zero become zero, after the bias */
  const lf_checkpoint* relu_of;   /* [rows, outputs] or NULL: zero where its code is zero or
                                     negative, the gradient of a ReLU whose output was kept */
  int out_dtype;
  const void* residual;        /* [rows, outputs], out_dtype, added last; NULL, or with `out` */
  void* out;                   /* [rows, outputs], may alias residual; or NULL: out_kept */
  const lf_checkpoint* out_kept;
} lf_fp8_linear_args;

int lf_fp8_linear(lf_context* ctx, const lf_fp8_linear_args* args);

typedef struct {
  const lf_checkpoint* grad;   /* [rows, outputs]: the gradient of the linear's out */
  const lf_checkpoint* act;    /* [rows, inputs]: what the forward call multiplied */
  int layout;                  /* of out: LF_OUT_IN or LF_IN_OUT */
  int grad_dtype;              /* of out and bias */
  void* out;                   /* [outputs, inputs] or [inputs, outputs] */
  void* bias;                  /* [outputs]: the sum of grad's rows, or NULL */
  void* scratch;
  size_t scratch_bytes;
} lf_fp8_weight_grad_args;

int lf_fp8_weight_grad(lf_context* ctx, const lf_fp8_weight_grad_args* args);
size_t lf_fp8_weight_grad_scratch(int rows, int outputs, int inputs);

/* What the training forward pass of a transition keeps: (rows (2 channels + hidden)) codes. */
typedef struct {
  lf_checkpoint act, normed;   /* [rows, channels] */
  lf_checkpoint hidden;        /* [rows, hidden] */
  float *mean, *rstd;          /* [rows] */
} lf_transition_saved;

/* The AF2 transition of lf_transition (LF_TRANSITION_RELU) as a training step runs it: matrices in
 * w are LF_F32, LF_F16 or LF_BF16, vectors f32, all read at the time of the call. */
typedef struct {
  int rows, channels, hidden;  /* channels 1..4096 */
  int act_dtype;
  const void* act;
  void* out;                   /* may alias act */
  int accumulate;              /* 1: out = act + update */
  int fast_variance;
  float epsilon;
  const lf_transition_weights* w;
  const lf_transition_saved* saved;   /* written */
  void* scratch;
  size_t scratch_bytes;
} lf_transition_train_args;

int lf_transition_train(lf_context* ctx, const lf_transition_train_args* args);
size_t lf_transition_train_scratch(int rows, int channels, int hidden);

typedef struct {
  int rows, channels, hidden;
  int act_dtype;
  const void* grad;            /* [rows, channels]: of lf_transition_train's out */
  void* out;                   /* [rows, channels]: the gradient of its act, may alias grad */
  int accumulate;              /* as in the forward call: 1 adds grad, the residual's gradient */
  const lf_transition_weights* w;     /* as in the forward call */
  const lf_transition_saved* saved;   /* of the forward call */
  int grad_dtype;              /* of the gradients below */
  void *grad_norm_scale, *grad_norm_offset;   /* [channels] */
  void *grad_w1, *grad_b1;     /* in the layout of w->w1; [hidden] */
  void *grad_w2, *grad_b2;     /* in the layout of w->w2; [channels] */
  void* scratch;
  size_t scratch_bytes;
} lf_transition_backward_args;

/* Every gradient pointer is given, but grad_b1 or grad_b2 may be NULL (a transition without that
 * bias has it NULL in w too). */
int lf_transition_backward(lf_context* ctx, const lf_transition_backward_args* args);
size_t lf_transition_backward_scratch(int rows, int channels, int hidden);

/* ---- training: relative positions, products of 4 bits, orthogonalised updates ------------------ */

/* Beside the section above and under its rules for sums, alignment, overlap and scratch.
 *
 * A learned row per relative position, added to every pair: the embedder's relpos_w and relpos_b
 * (lf_input_embedder: boundaries -31..32, 65 rows) with any buckets, chains and lengths, and its
 * gradient.  The bucket of query i and key j is the number of boundaries, ascending, that are at most
 * query_positions[i] - key_positions[j].  With segments (chains), pairs of different segments take the
 * table's last row, and a negative segment is padding: nothing is added to its pairs, and their
 * gradient, whatever it holds, is left out. */
typedef struct {
  int queries, keys;
  const int *query_positions, *key_positions;   /* [queries], [keys] */
  const int *query_segments, *key_segments;     /* [queries], [keys], or both NULL */
  int boundary_count;                           /* 0..4095 */
  const int* boundaries;                        /* [boundary_count] */
} lf_relative_pairs;
/* Rows of the table: a bucket each, and one for pairs of different segments. */
#define LF_RELATIVE_ROWS(pairs) ((pairs)->boundary_count + 1 + ((pairs)->query_segments ? 1 : 0))

typedef struct {
  const lf_relative_pairs* pairs;
  int channels;                /* 1..4096 */
  int table_dtype;
  const void* table;           /* [rows, channels] */
  const float* bias;           /* [channels], added to every row of the table, or NULL */
  int act_dtype;
  const void* act;             /* [queries, keys, channels], added last, or NULL */
  void* out;                   /* [queries, keys, channels], may alias act */
} lf_relative_position_args;

int lf_relative_position(lf_context* ctx, const lf_relative_position_args* args);

typedef struct {
  const lf_relative_pairs* pairs;
  int channels;
  int act_dtype;
  const void* grad;            /* [queries, keys, channels]: of lf_relative_position's out */
  int grad_dtype;              /* of the gradients below */
  void* grad_table;            /* [rows, channels]: the sum over a row's pairs, 0 where it has none */
  void* grad_bias;             /* [channels]: the sum over all pairs, or NULL */
  void* scratch;
  size_t scratch_bytes;
} lf_relative_position_backward_args;

/* A table of more than about 300 rows is summed in parts, each a pass over grad. */
int lf_relative_position_backward(lf_context* ctx, const lf_relative_position_backward_args* args);
size_t lf_relative_position_backward_scratch(const lf_relative_pairs* pairs, int channels);   /* reads no tensor */

/* A [rows, cols] matrix in 4 bits: e2m1 codes (0, 1/2, 1, 3/2, 2, 3, 4, 6 and their negatives) with
 * one scale per row and group of 32 columns, a power of two 2^(b - 127) with b in 1..254 as stored, the
 * smallest that puts the group's largest magnitude within 6 (b = 1 for a group of zeros).  The
 * division by it is exact, so the code's rounding (to nearest, ties to even; half the step of 1/2, 1 or
 * 2 scales) is the only one.  There is no code for an infinity or a NaN: a group that holds one gets b
 * = 255 and reads back as NaN, all 32 of it.  A value within 2^-3 of the largest of its type may round up to
 * a power of two beyond it, which reads back as an infinity of that type.
 *
 *   codes   [rows][LF_MX4_PITCH(cols) / 2], two a byte, the lower column in the lower half; columns
 *           from cols to the pitch hold zeros
 *   scales  [LF_MX4_GROUPS(cols)][LF_MX4_SCALE_PITCH(rows)], one byte b each (not 255 for groups
 *           behind the last column); bytes of rows >= rows may hold anything
 *
 * codes and scales are 16-byte aligned.  At most 2^26 columns and 2^34 elements, columns rounded up to 128 and rows to 16. */
typedef struct {
  int rows, cols;
  void* codes;
  void* scales;
} lf_mx4;
#define LF_MX4_PITCH(cols) (((size_t)(cols) + 127) / 128 * 128)
#define LF_MX4_GROUPS(cols) (LF_MX4_PITCH(cols) / 32)
#define LF_MX4_SCALE_PITCH(rows) (((size_t)(rows) + 15) / 16 * 16)

typedef struct {
  int rows, cols;
  int act_dtype;
  const void* act;             /* [rows, cols] */
  const lf_mx4* out;           /* [rows, cols], groups along the columns, or NULL */
  const lf_mx4* transposed;    /* [cols, rows], groups along the rows, or NULL */
  int sums_dtype;
  void* sums;                  /* [cols]: the sum of act's rows (not of its codes), or NULL */
  void* scratch;
  size_t scratch_bytes;
} lf_mx4_pack_args;

/* Activations, gradients or weights to 4 bits: `out` is the operand of products along the columns (an
 * [outputs, inputs] weight, activations), `transposed` of products along the rows (the weight of the
 * input's gradient; gradient and activations of the weight's).  At least one output is given. */
int lf_mx4_pack(lf_context* ctx, const lf_mx4_pack_args* args);
size_t lf_mx4_pack_scratch(int rows, int cols);   /* for sums; 0 is needed without */

typedef struct {
  int act_dtype;
  void* act;                   /* [rows, cols] of `kept`, written */
  const lf_mx4* kept;
} lf_mx4_unpack_args;

/* The values that codes and scales stand for, rounded to act_dtype. */
int lf_mx4_unpack(lf_context* ctx, const lf_mx4_unpack_args* args);

typedef struct {
  int rows;
  const lf_mx4* kept;          /* [rows, inputs], or NULL: act */
  int act_dtype;
  const void* act;             /* [rows, inputs], quantised as lf_mx4_pack does; or NULL: kept */
  const lf_mx4* w;             /* [outputs, inputs] */
  const float* bias;           /* [outputs] or NULL */
  int relu;                    /* values below zero become zero, after the bias */
  int out_dtype;
  const void* residual;        /* [rows, outputs], out_dtype, added last, or NULL */
  void* out;                   /* [rows, outputs], may alias residual */
  void* scratch;
  size_t scratch_bytes;
} lf_mx4_linear_args;

/* out = act w^T + bias.  Products are exact, sums are f32's.  The weight's gradient is the same product
 * of transposed packs: kept = the gradient's [outputs, rows], w = the activations' [inputs, rows]. */
int lf_mx4_linear(lf_context* ctx, const lf_mx4_linear_args* args);
size_t lf_mx4_linear_scratch(int rows, int inputs, int outputs, int from_act);   /* from_act: act is given; 0: none is used */

/* Matrices made orthogonal by Newton-Schulz products: with X = act / (|act| + epsilon), |.| the
 * Frobenius norm, and (a, b, c) a step's coefficients, X <- a X + (b G + c G^2) X, G = X X^T, `steps`
 * times (for matrices taller than wide the same of the transpose).  Singular values go through
 * a s + b s^3 + c s^5 each time, vectors stay.  Products are of f32 precision (two f16 parts each, sums in
 * f32).  The two parts hold an element to 2^-38 of the largest singular value that X can have, so that a
 * matrix whose norm is far below epsilon keeps fewer bits of its result, which is small then, and at last
 * none.  Coefficients whose polynomials leave 2^24 on what [0, 1] can become are refused. */
typedef struct {
  int batch, rows, cols;       /* rows, cols 1..16384, batch 1..65535 */
  int act_dtype;
  const void* act;             /* [batch, rows, cols] */
  void* out;                   /* [batch, rows, cols], may alias act */
  int steps;                   /* 1..32 */
  const float* coefficients;   /* HOST memory: [steps][3], read before the call returns */
  float epsilon;               /* >= 0; a matrix of zeros with 0 becomes NaN */
  void* scratch;
  size_t scratch_bytes;
} lf_orthogonalize_args;

int lf_orthogonalize(lf_context* ctx, const lf_orthogonalize_args* args);

/* An optimiser's step for a batch of weight matrices: m' = momentum_factor m + grad, u = grad +
 * momentum_factor m' (nesterov) or m', weight' = (1 - rate decay) weight - rate scale O(u), O as above. */
typedef struct {
  int batch, rows, cols;
  int grad_dtype;
  const void* grad;            /* [batch, rows, cols] */
  const float* momentum;       /* [batch, rows, cols]: m, or NULL with momentum_out: u = grad */
  float* momentum_out;         /* m', may alias momentum */
  float momentum_factor;
  int nesterov;
  int weight_dtype;
  const void* weight;          /* [batch, rows, cols] */
  void* weight_out;            /* may alias weight */
  float rate, decay, scale;
  int steps;
  const float* coefficients;   /* as above */
  float epsilon;
  void* scratch;
  size_t scratch_bytes;
} lf_muon_step_args;

int lf_muon_step(lf_context* ctx, const lf_muon_step_args* args);
size_t lf_muon_scratch(int batch, int rows, int cols);   /* for both; 0: none is used */

#ifdef __cplusplus
}
#endif
#endif /* LOCALFOLD_H */

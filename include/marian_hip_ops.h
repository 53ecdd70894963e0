/*
 * marian_hip_ops.h - C ABI of the float32 operators that sit between the int8 GEMMs of a
 * transformer decode step (same library and conventions as marian_hip_int8.h: device pointers,
 * caller-owned buffers, nothing retained, work enqueued on `stream`, status codes, no
 * synchronisation).  Tensors are dense row-major fp32 where nothing else is said; pointers need 4-byte alignment only
 * (16-byte aligned rows take a vector path).  In-place operation (out == in) is allowed for
 * layer_norm, softmax and logsoftmax.
 */
#ifndef MARIAN_HIP_OPS_H
#define MARIAN_HIP_OPS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Replaces LayerNormalization, reference src/tensors/gpu/tensor_operators.cu (gLNormalization)
 * and src/tensors/cpu/tensor_operators.cpp:1087-1162, node LayerNormalizationOp
 * (src/graph/expression_operators.cpp:901-913):
 *   mean = sum(x) / cols; sigma = sqrt(sum((x - mean)^2) / cols + eps);
 *   out = gamma * ((x - mean) / sigma) (+ beta)
 * over the last dimension.  gamma_cols / beta_cols: `cols`, or 1 for a single broadcast value;
 * beta may be NULL.  add != NULL fuses the skip connection that precedes the normalization in
 * the transformer's post-processing (`output + prevInput`, src/models/transformer.h:192-193,207):
 * x = in + add, else x = in.
 * absmax_out: NULL, or MARIAN_HIP_ABSMAX_SLOTS (2048) floats that receive values whose maximum is
 * max|out|, for marian_hip_int8_affine_f32_chained.  Up to 2048 rows own a slot each; more rows
 * (an encoder's sentence batch) share the slots, which a second small kernel of the same call
 * clears first.
 */
int marian_hip_layer_norm(const float* in, const float* add, const float* gamma,
                          int64_t gamma_cols, const float* beta, int64_t beta_cols, float* out,
                          int64_t rows, int64_t cols, float eps, float* absmax_out, void* stream);

/*
 * Replaces Softmax, reference src/tensors/gpu/tensor_operators.cu (gSoftmax) and
 * src/tensors/cpu/tensor_operators.cpp:415-470, over the last dimension.  mask != NULL fuses the
 * `z + mask` node in front of it (src/models/transformer.h:264): mask holds n_masks rows of
 * `cols` values and row r of `in` uses mask row (r / rows_per_mask) % n_masks - a
 * [batch, 1, 1, len] log-mask, repeated over the beam (src/models/transformer.h:772-774),
 * against scores of shape [beam * batch, heads, tgt, len] has rows_per_mask = heads * tgt,
 * n_masks = batch.
 */
int marian_hip_softmax(const float* in, const float* mask, int64_t n_masks, int64_t rows_per_mask,
                       float* out, int64_t rows, int64_t cols, void* stream);

/* Replaces LogSoftmax, reference src/tensors/gpu/tensor_operators.cu (gLogSoftmax) and
 * src/tensors/cpu/tensor_operators.cpp:474-526. */
int marian_hip_logsoftmax(const float* in, float* out, int64_t rows, int64_t cols, void* stream);

/*
 * Replaces TransposeND for the axes {0, 2, 1, 3} (Transpose0213, reference
 * src/tensors/cpu/tensor_operators.cpp:220-246, gTranspose0213 on the GPU), the head split and
 * join of src/models/transformer.h:145-170: in [d0, d1, d2, d3] -> out [d0, d2, d1, d3].
 * out must not alias in.
 */
int marian_hip_transpose0213(const float* in, float* out, int64_t d0, int64_t d1, int64_t d2,
                             int64_t d3, void* stream);

/*
 * Replaces ProdBatchedLegacy with beta = 0, reference src/tensors/cpu/prod.cpp:233-330 and
 * src/tensors/gpu/prod.cpp:471-574 (node bdot_legacy, the attention products of
 * src/models/transformer.h:261,277):
 *   C[i] = scalar * op(A[i % batchA]) * op(B[i % batchB]),  i < max(batchA, batchB)
 * A: [batchA, m, k] ([batchA, k, m] when transA), B: [batchB, k, n] ([batchB, n, k] when
 * transB), C: [max(batchA, batchB), m, n].
 */
int marian_hip_bdot_legacy(const float* A, const float* B, float* C, int64_t batchA,
                           int64_t batchB, int64_t m, int64_t n, int64_t k, int transA,
                           int transB, float scalar, void* stream);

/*
 * The attention of one decoding step in one launch: the nodes bdot_legacy(q, k, false, true,
 * scale), `+ mask`, softmax and bdot_legacy(weights, v) of Attention(), reference
 * src/models/transformer.h:241-280.  The arithmetic is that of the three separate entry points
 * above; for head sizes other than 64 operation for operation (the result equals theirs bit for
 * bit), for dk == 64 with the dot products summed sixteen lanes wide and the weighted values four
 * positions wide (equal within the 1e-5 relative bar of the float operators).
 *   q: [batchQ, m, dk], k and v: [batchKV, len, dk] (entry i uses k, v of i % batchKV: encoder
 *   keys shared by the beam), out: [batchQ, m, dk]; mask as in marian_hip_softmax for score rows
 *   [batchQ * m, len], or NULL.  len <= 4096.
 *   Built for decoding steps (m = 1): every query row gets a wave that walks the head's keys and
 *   values itself.  For several positions per head (encoder layers) with dk == 64 there is
 *   marian_hip_attention_rows; the host mirror switches over by itself.
 *   Where several query rows share a cache entry (batchKV < batchQ, m == 1, dk == 64, len <= 96,
 *   16-byte aligned tensors, no k_new) the rows of an entry are taken by one workgroup, which
 *   reads the entry's keys and values once: same bits, 28 instead of 50 us for 512 rows x 16 heads
 *   over 60 source positions with four hypotheses a sentence.
 *   absmax_out: as for marian_hip_layer_norm (needs batchQ * m <= 2048).
 *   k_new, v_new: NULL, or [batchQ, dk] keys and values of the newest position (self-attention of
 *   a decoding step: m == 1, batchKV == batchQ).  They take the place of position len - 1 of k and
 *   v, and the call also stores them there, which is the concatenation of the new position onto
 *   the cached ones (decoder state of src/models/transformer.h:683-700) without a copy launch; k
 *   and v are written in that case.
 */
int marian_hip_attention(const float* q, float* k, float* v, const float* mask, int64_t n_masks,
                         int64_t rows_per_mask, float* out, int64_t batchQ, int64_t batchKV,
                         int64_t m, int64_t len, int64_t dk, float scale, float* absmax_out,
                         const float* k_new, const float* v_new, void* stream);

/*
 * The same attention on heads that may lie side by side in a row, and for several query positions per head
 * (encoder layers, whole target sentences): q, k, v and out are [batch, heads, positions, dk] with the floats
 * between two sentences, heads and positions given (three strides each, multiples of four; 16-byte aligned
 * tensors), so that the output of an affine call is read as it is and SplitHeads / JoinHeads
 * (src/models/transformer.h:145-170) move nothing.  batchQ, batchKV: entries, sentences times heads; entry i
 * uses keys and values of entry i % batchKV.  mask as in marian_hip_softmax for score rows [batchQ * m, len], or
 * NULL.  absmax_out: as for marian_hip_layer_norm (needs batchQ * m <= 2048).
 *   m >= MARIAN_HIP_ATTENTION_ROWS_MIN: blocks of query rows share keys and values; dk == 64 and len <=
 *   MARIAN_HIP_ATTENTION_ROWS_MAX_LEN (other sizes: MARIAN_HIP_ERR_SHAPE); bit for bit what
 *   marian_hip_bdot_legacy, marian_hip_softmax and marian_hip_bdot_legacy give.
 *   fewer rows: bit for bit marian_hip_attention; len <= 4096.
 */
#define MARIAN_HIP_ATTENTION_ROWS_MIN 8
#define MARIAN_HIP_ATTENTION_ROWS_MAX_LEN 256
int marian_hip_attention_rows(const float* q, const int64_t* q_strides, const float* k, const int64_t* k_strides,
                              const float* v, const int64_t* v_strides, const float* mask, int64_t n_masks,
                              int64_t rows_per_mask, float* out, const int64_t* out_strides, int64_t batchQ,
                              int64_t batchKV, int64_t heads, int64_t m, int64_t len, int64_t dk, float scale,
                              float* absmax_out, void* stream);

/*
 * marian_hip_attention on caches that have room to grow: k and v are [batchKV, kv_capacity, dk]
 * with the first len positions of every entry in use (kv_capacity >= len; the mask still has len
 * values per row).  The decoder state of a translation then stays where it is from step to step:
 * the reference concatenates the new position onto the cached ones into a fresh tensor every
 * step (src/models/transformer.h:409-416), here a step passes len = positions so far + 1 with k_new,
 * v_new, which the call stores at position len - 1, and the selection of the surviving
 * hypotheses between two steps (src/rnn/types.h:22-42) is rows() over entries of kv_capacity * dk
 * values.  marian_hip_attention is this call with kv_capacity = len.
 */
int marian_hip_attention_cached(const float* q, float* k, float* v, const float* mask, int64_t n_masks,
                                int64_t rows_per_mask, float* out, int64_t batchQ, int64_t batchKV,
                                int64_t m, int64_t len, int64_t kv_capacity, int64_t dk, float scale,
                                float* absmax_out, const float* k_new, const float* v_new, void* stream);

/*
 * The embedding step in front of the first layer, reference src/layers/embedding.cpp:161-168
 * (rows(E, ids): CopyRows, src/tensors/cpu/tensor_operators.cpp:577-603), followed by
 * src/models/transformer.h:93 (sqrt(dimEmb) * embeddings) and :117 (embeddings + signal, the
 * sinusoidal position signal of src/tensors/cpu/tensor_operators.cpp:1733-1746) as one launch:
 *   out[r, :] = scale * E[ids[r], :] + signal[(r / rows_per_signal) % n_signals, :]
 * with the product and the sum rounded one after the other like the reference's two nodes, so
 * the result equals theirs bit for bit.
 *   E: [vocab, dimEmb] float32; ids: rows word indices (uint32, the reference's IndexType), on the
 *   device.  The reference reads past the table for an id >= vocab; this call reads the table's
 *   last row instead.
 *   signal: NULL (no sum: a pure gather when scale == 1), or [n_signals, dimEmb].  A decoding step
 *   passes the one row of its position (n_signals == 1); a whole sentence batch [dimWords,
 *   dimBatch] passes rows_per_signal = dimBatch, n_signals = dimWords.
 *   absmax_out: as for marian_hip_layer_norm (needs rows * ceil(dimEmb / 4096) <= 2048): the int8
 *   products of the first layer then need no abs-max launch of their own.
 * With scale 1 and no signal the call is rows(E, ids) itself, which is also the selection of the
 * surviving hypotheses' decoder states between two steps of the beam search (reference
 * src/rnn/types.h:22-42: rows(reshape(state, [beam * batch, positions * depth]), selIdx)); rows
 * longer than 4096 values are split over several workgroups.
 */
int marian_hip_embed(const float* E, const uint32_t* ids, int64_t rows, int64_t vocab, int64_t dimEmb,
                     float scale, const float* signal, int64_t rows_per_signal, int64_t n_signals,
                     float* out, float* absmax_out, void* stream);

/*
 * Self-attention of a decoding step on caches that are never moved: where the reference selects
 * the surviving hypotheses' states between two steps by copying them (src/rnn/types.h:22-42), a
 * table of ancestors says in whose cache entry a position of a hypothesis's history lies, and the
 * call follows it.  No counterpart in the reference; the result is that of
 * marian_hip_attention_cached on caches gathered position by position, bit for bit.
 *   q, k_new, v_new, out: [n_hyp * heads, dk]; k, v: [n_hyp * heads, kv_capacity, dk], entry =
 *   hypothesis * heads + head; ancestors: uint32 [n_hyp, kv_capacity] on the device: cached position
 *   p < len - 1 of hypothesis h is read from the entry of hypothesis ancestors[h * kv_capacity + p]
 *   (values at or past n_hyp read the last hypothesis); position len - 1 is k_new / v_new, which the
 *   call stores into hypothesis h's own entry.  dk == 64, all tensors 16-byte aligned.
 * marian_hip_ancestors_advance makes the table of the next step: next[h, p] = prev[parents[h], p]
 * for the len_prev positions cached so far and next[h, len_prev] = h (prev and next must not
 * overlap); parents: uint32 [n_hyp], the back-pointers of the beam search.
 */
int marian_hip_attention_ancestors(const float* q, float* k, float* v, float* out, int64_t n_hyp, int64_t heads,
                                   int64_t len, int64_t kv_capacity, int64_t dk, float scale, float* absmax_out,
                                   const float* k_new, const float* v_new, const uint32_t* ancestors,
                                   void* stream);
int marian_hip_ancestors_advance(const uint32_t* prev, const uint32_t* parents, int64_t n_hyp, int64_t kv_capacity,
                                 int64_t len_prev, uint32_t* next, void* stream);

/*
 * The selection of the surviving hypotheses' decoder states between two steps of the beam search
 * (reference src/models/states.h:87-107, src/rnn/types.h:22-42: rows(reshape(state, [beam * batch,
 * positions * depth]), selIdx)) for states that stay in place and have room to grow:
 *   state: [entries, segments, seg_capacity] float32 (the caches of marian_hip_attention_cached:
 *   segments = heads, seg_capacity = kv_capacity * dk), out: [rows, segments, seg_capacity];
 *   out[r, s, 0 .. seg_len) = state[ids[r], s, 0 .. seg_len), seg_len = positions in use * dk.
 * What lies behind seg_len is neither read nor written.  state and out must not overlap
 * (MARIAN_HIP_ERR_ALIAS); an id at or past `entries` reads the last entry.
 * With seg_len == seg_capacity and one segment this is marian_hip_embed with scale 1.
 */
int marian_hip_select_state(const float* state, const uint32_t* ids, int64_t rows, int64_t entries,
                            int64_t segments, int64_t seg_capacity, int64_t seg_len, float* out, void* stream);

/*
 * Replaces SinusoidalPositionEmbeddings, reference src/tensors/cpu/tensor_operators.cpp:1733-1746,
 * the initializer of the constant that src/models/transformer.h:110-111 adds to the embeddings:
 *   host_out[j, i] = sin or cos of (j + start) * exp((i % (dimEmb / 2)) * -log(10000) / (dimEmb / 2 - 1)),
 * sine for the first half of a row, cosine for the rest, in float arithmetic with the C library's
 * functions like the reference's loop.  host_out: dimWords * dimEmb floats in HOST memory (the
 * constant is made once per position on the host and copied to the device by the caller);
 * dimEmb >= 4 (with fewer the reference's increment divides by zero).  No HIP call is made.
 */
int marian_hip_sinusoidal_position_embeddings(float* host_out, int64_t dimWords, int64_t dimEmb, int64_t start);

/*
 * Replaces NthElement::getNBestList, reference src/translator/nth_element.cpp:26-67 (CPU) and
 * src/translator/nth_element.cu (GPU): for each of dimBatch rows of rowLen = beam * vocabulary
 * scores, the N best scores in descending order and their keys = absolute positions
 * row * rowLen + index (uint32).  Equal scores come out lowest index first (the reference's
 * partial_sort leaves that order unspecified).  1 <= N <= 16, N <= rowLen.
 * outScores, outKeys: dimBatch * N values each, on the device.
 */
int marian_hip_nbest(const float* scores, int64_t dimBatch, int64_t rowLen, int64_t N,
                     float* outScores, uint32_t* outKeys, void* stream);

/*
 * The words a row's best scores stand for, in one launch: the selection of marian_hip_nbest on each of
 * `rows` rows, with the positions within the row instead of keys, taken through a shortlist's ids where
 * there is one (Shortlist::reverseMap, reference src/data/shortlist.h:25-29).
 *   ids: [rowLen] vocabulary ids on the device, or null; outWords: rows * N values, 8-byte aligned.
 * Positions that no score fills (a row with fewer than N scores that are not NaN) come out as -inf and
 * -1, or the last of the ids.
 */
int marian_hip_nbest_words(const float* scores, int64_t rows, int64_t rowLen, int64_t N, const uint32_t* ids,
                           float* outScores, int64_t* outWords, void* stream);

/*
 * The transposition and the n-best selection of a beam-search step in one call: reference
 * src/translator/beam_search.cpp:472 (swapAxes(expandedPathScores, 0, 2)) followed by :492
 * (getNBestList).  scores: [beam, dimBatch, vocab], the layout in which the step's scores leave the
 * decoder.  The result is that of marian_hip_nbest on the transposed tensor [dimBatch, beam * vocab]
 * - the same scores, the same keys b * beam * vocab + k * vocab + v, the same order - without
 * writing that tensor, and with the row of a batch entry split over several workgroups (the N best
 * of every part, then the N best of those, in one launch).  1 <= N <= 16, beam * N <= 1024, dimBatch <= 4096.
 *   workspace: device memory of at least marian_hip_nbest_beams_workspace_bytes(...) bytes (the
 *   reference's NthElement holds such buffers itself, src/translator/nth_element.cu): the
 *   candidates of the parts, and one counter per batch entry by which the workgroup that finishes an
 *   entry last knows that it is to draw the final list.  The counters are zero between calls:
 *   marian_hip_nbest_beams_workspace_init clears a freshly allocated workspace once (a kernel, so it
 *   may be captured in a graph).  One workspace serves one stream: calls that share a workspace must
 *   not overlap (two streams, or two threads, need a workspace each), and a workspace whose address a
 *   recorded graph holds must stay allocated as long as that graph is replayed.
 */
size_t marian_hip_nbest_beams_workspace_bytes(int64_t beam, int64_t dimBatch, int64_t vocab, int64_t N);
int marian_hip_nbest_beams_workspace_init(void* workspace, size_t workspace_bytes, void* stream);
int marian_hip_nbest_beams(const float* scores, int64_t beam, int64_t dimBatch, int64_t vocab, int64_t N,
                           float* outScores, uint32_t* outKeys, void* workspace, size_t workspace_bytes,
                           void* stream);

/*
 * The end of a beam-search step in one call: the log-softmax of the decoder's logits (LogSoftmax,
 * src/tensors/cpu/tensor_operators.cpp:474-526, as marian_hip_logsoftmax computes it), the addition of
 * the hypotheses' path scores (expandedPathScores = prevPathScores + logProbs,
 * src/translator/beam_search.cpp:433-436) and the transposition + n-best selection of
 * marian_hip_nbest_beams (:472, :492), without writing the log-probabilities and reading them back.
 *   logits: [beam, dimBatch, vocab]; vocab % 4 == 0, 4096 < vocab <= 32768 (a row is held in the
 *   registers of one 1024-thread workgroup, as marian_hip_logsoftmax does for these sizes; other
 *   sizes: MARIAN_HIP_ERR_SHAPE - use the separate calls), 16-byte aligned.
 *   rowAdd: NULL, or one value per row [beam * dimBatch] that is added to every log-probability of
 *   the row before the selection (the path score; what is written to logProbs is without it).
 *   logProbs: NULL, or [beam, dimBatch, vocab] that receives the log-probabilities as well.
 * outScores, outKeys, N, workspace: as for marian_hip_nbest_beams (a workspace sized and initialised
 * for it with the same beam, dimBatch, vocab and N serves this call too); the results are those of
 * marian_hip_logsoftmax (+ rowAdd) followed by marian_hip_nbest_beams, bit for bit.
 */
int marian_hip_logsoftmax_nbest_beams(const float* logits, const float* rowAdd, float* logProbs, int64_t beam,
                                      int64_t dimBatch, int64_t vocab, int64_t N, float* outScores,
                                      uint32_t* outKeys, void* workspace, size_t workspace_bytes, void* stream);

/*
 * Replaces gpu::fill, reference src/tensors/gpu/algorithm.cu:37-60 (gFill): `count` elements of
 * elem_bytes (1, 2, 4 or 8) bytes each, starting at `begin` (aligned to elem_bytes), receive the
 * low elem_bytes bytes of `pattern` - the bit pattern of the value, so one entry point serves
 * every element type.  A kernel, not a memset: it may be recorded into a HIP graph.  Like every
 * function here it does not synchronise; the C++ wrapper adds the reference's stream synchronisation.
 */
int marian_hip_fill(void* begin, int64_t count, int elem_bytes, uint64_t pattern, void* stream);

/*
 * Keys and values in 8 bits: rotary positions, a cache that is quantized as it is written, and attention over it
 * for single tokens, chains and trees of drafted ones.  No counterpart in the reference, whose decoder state is
 * float32 (src/models/transformer.h:683-700) and whose positions are added to the embeddings.
 *
 * Activations are float32, float16 or bfloat16 ("type"), [sequences, heads, n, dk] with the values between two
 * sequences, heads and positions given (three strides, in values, whole multiples of 16 bytes), so that rows of an
 * affine call are read as they are.  16-byte aligned; dk a multiple of 16 from 16 to 256.  Rows that are read may share
 * memory (a stride of 0), rows that are written may not (MARIAN_HIP_ERR_ALIAS: a stride reaches over all that lies
 * within one of its steps, in any order of the dimensions).  n up to 2^20 (marian_hip_cache_append: 262140).
 */
#define MARIAN_HIP_FLOAT32 0
#define MARIAN_HIP_FLOAT16 1
#define MARIAN_HIP_BFLOAT16 2

/*
 * The cache: for each of sequences * heads entries `capacity` rows of dk codes and a float32 scale each, dense:
 * k, v: [sequences, heads, capacity, dk], k_scale, v_scale: [sequences, heads, capacity].  A value is code * scale.
 *   MARIAN_HIP_CACHE_INT8: codes are whole numbers -127 .. 127, scale = largest magnitude of the row / 127;
 *   MARIAN_HIP_CACHE_E4M3: codes are floats of 4 exponent and 3 mantissa bits up to 448, scale = largest / 448.
 * A code is the exact quotient value * 127 / largest (448) rounded to the nearest, ties to even.  A row of zeros
 * has scale 0.  A row that holds an infinity or NaN has zeros for codes and a NaN scale: everything that reads it
 * is NaN, and nothing that does not read it.
 * Codes that come from elsewhere are taken by their bits: int8 -128 is -128, and e4m3's NaN (0x7f, 0xff) is 480 (-480).
 * Scales that come from elsewhere may be below zero.
 *   heads <= 4096, sequences <= 65535, capacity * dk < 2^31; k and v 16-byte, scales 4-byte aligned.
 */
#define MARIAN_HIP_CACHE_INT8 0
#define MARIAN_HIP_CACHE_E4M3 1
typedef struct marian_hip_kv_cache {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  int64_t sequences, heads, capacity, dk;
  int format;
} marian_hip_kv_cache;

/*
 * The new tokens of a step: n for each sequence.
 *   lens: int32 [sequences] on the device, the positions of each sequence that are settled already (values outside
 *   0 .. capacity are taken as the nearer end).  New token i of sequence s has row lens[s] + i of the cache.
 *   counts: null, or int32 [sequences]: only the first counts[s] of the n are there (0 .. n; others are taken as the
 *   nearer end).
 *   parents: null - the new tokens follow one another (a prompt, or one token) - or int32 [sequences, n]: a tree of
 *   drafted tokens, n <= MARIAN_HIP_TREE_MAX.  parents[s, i] is the drafted token that token i continues, or -1: the
 *   last settled one.  A parent does not come behind its child: a value at or past i, or below -1, stands for -1.
 */
#define MARIAN_HIP_TREE_MAX 64
typedef struct marian_hip_drafts {
  const int32_t* lens;
  const int32_t* counts;
  const int32_t* parents;
  int64_t n;
} marian_hip_drafts;

/*
 * Rotary positions: the first `dims` values of a row (a multiple of 8, up to dk) are dims / 2 pairs, pair p being
 * values (p, p + dims / 2), or (2 p, 2 p + 1) where interleaved; at position t it is turned by t * turns[p] * 2^-64
 * whole turns and multiplied by magnitude:
 *   (a, b) -> magnitude * (a cos - b sin, a sin + b cos).
 * Turns are whole numbers mod 2^64, so the angle of a far position is as exact as that of a near one.
 *   turns: uint64 [dims / 2] on the device, made by marian_hip_rotary_turns on the host.
 */
typedef struct marian_hip_rotation {
  const uint64_t* turns;
  int64_t dims;
  double magnitude;
  int interleaved;
} marian_hip_rotation;

/*
 * The turns of a model: pair p turns by base^(-2 p / dims) radians a position, changed for contexts `factor` times
 * as long as the model was made for:
 *   MARIAN_HIP_ROTARY_LINEAR: all divided by factor;
 *   MARIAN_HIP_ROTARY_BASE: base * factor^(dims / (dims - 2)) in place of base;
 *   MARIAN_HIP_ROTARY_BANDS: pairs that turn less than `slow` times in `original` positions are divided by factor, those
 *   that turn more than `fast` times stay, between them a mixture that is linear in the number of turns, as the formula of Peng et al., "YaRN",
 *   2023, has it; magnitude 0.1 ln(factor) + 1.  (Some models' own code mixes linearly in the pair's index between the two bounds instead, with other
 *   frequencies in between; for those, and any other scaling, `turns` is filled by the caller: round(frequency / 2 pi * 2^64).)
 * host_turns: dims / 2 values in HOST memory; host_magnitude: one.  No HIP call is made.
 * base > 1, factor >= 1; BASE: dims >= 4; BANDS: original >= 1, 0 <= slow < fast.
 */
#define MARIAN_HIP_ROTARY_PLAIN 0
#define MARIAN_HIP_ROTARY_LINEAR 1
#define MARIAN_HIP_ROTARY_BASE 2
#define MARIAN_HIP_ROTARY_BANDS 3
int marian_hip_rotary_turns(uint64_t* host_turns, double* host_magnitude, int64_t dims, double base, int scaling,
                            double factor, int64_t original, double slow, double fast);

/*
 * out = x turned by its positions: x and out [sequences, heads, n, dk].
 *   positions: int32 on the device: [sequences], row i of a sequence being at positions[s] + i, or, with
 *   each != 0, [sequences, n].  Positions may be negative.
 * out is x itself (same strides), or shares no memory with it (MARIAN_HIP_ERR_ALIAS).
 */
int marian_hip_rotary(const void* x, const int64_t* x_strides, void* out, const int64_t* out_strides, int type,
                      int64_t sequences, int64_t heads, int64_t n, int64_t dk, const int32_t* positions, int each,
                      const marian_hip_rotation* rotation, void* stream);

/*
 * Writes the keys and values of the new tokens into the cache, in one launch with the rotation of keys and queries:
 *   k, v: [sequences, heads, n, dk]; rotation: null, or what k (and q) is turned by, token i of sequence s standing at
 *   position lens[s] + the number of drafted tokens it descends from (a chain: lens[s] + i).
 *   q: null, or queries [sequences, q_heads, n, dk], turned the same way into q_out (q itself with the same strides, or
 *   apart from all else); without a rotation they are copied.  Rows of q_out at or past counts[s] are zeros.
 * Keys are turned in 64-bit arithmetic, rounded to float32 and quantized.  Rows of the cache other than those
 * of the counts[s] new tokens, and of tokens that do not fit (at or past capacity, which are dropped), stay as they are.
 * lens, counts and parents are only read.
 */
int marian_hip_cache_append(const marian_hip_kv_cache* cache, const marian_hip_drafts* drafts, const void* k,
                            const int64_t* k_strides, const void* v, const int64_t* v_strides, int type,
                            const marian_hip_rotation* rotation, const void* q, const int64_t* q_strides, int64_t q_heads,
                            void* q_out, const int64_t* q_out_strides, void* stream);

/*
 * Reads rows of the cache back: k_out, v_out [sequences, heads, n, dk], dense, of `type`; row i is position
 * first[s] + i (first: int32 [sequences] on the device).  Positions outside 0 .. capacity give zeros.
 */
int marian_hip_cache_read(const marian_hip_kv_cache* cache, const int32_t* first, int64_t n, void* k_out, void* v_out,
                          int type, void* stream);

/*
 * Attention of the new tokens over the cache they have been written to: q and out [sequences, q_heads, n, dk],
 * q_heads a multiple of the cache's heads (query head h reads head h / (q_heads / heads)):
 *   out = softmax(scale * q . key) value
 * over the settled positions of the sequence, the token itself and the drafted tokens it descends from.
 * Positions that a token does not see are not read into its result, whatever they hold.  A token that sees nothing (it
 * and all before it past the capacity) gives zeros, and so do rows at or past counts[s].  out shares no memory with q
 * or the cache.  scale: finite, above zero.
 * Products and sums are float32.  Weights enter the product with the values in 22 bits, of bfloat16 queries with more than 32 rows an entry (n *
 * q_heads / heads) in 11, each of its own size down to 2^-24 of the largest; the sum is of the weights in float32.
 * Scales of values below 1e-30 are weighed in steps that do not get smaller with them: off by up to 2^-30 * 1e-30 of a position's code.
 * Keys whose largest magnitude is above 2^110 may take a score out of float32, and the result is NaN then.
 * A sequence's positions are split over workgroups where there are few of them, by the lengths of all
 * sequences, and the cache's sizes, its capacity among them, say which form of the kernel takes them: the last bits of a result depend on the
 * batch and on the cache it is in, and not on the order of anything.
 *   workspace: at least marian_hip_cache_attention_workspace_bytes(...) bytes (enough for any capacity and type; 0 too where
 *   sizes are out of range), 256-byte aligned (0 bytes: may be null), which marian_hip_cache_attention_workspace_init clears once after allocating (a kernel: it may be
 *   recorded).  One workspace serves one stream, like that of marian_hip_nbest_beams.
 */
size_t marian_hip_cache_attention_workspace_bytes(int64_t sequences, int64_t heads, int64_t q_heads, int64_t n, int64_t dk);
int marian_hip_cache_attention_workspace_init(void* workspace, size_t workspace_bytes, void* stream);
int marian_hip_cache_attention(const marian_hip_kv_cache* cache, const marian_hip_drafts* drafts, const void* q,
                               const int64_t* q_strides, int64_t q_heads, int type, float scale, void* out,
                               const int64_t* out_strides, void* workspace, size_t workspace_bytes, void* stream);

/*
 * The accepted ones of the drafted tokens become settled: for j < accepted[s] the keys and values of drafted token
 * path[s, j] move to row lens[s] + j, all of a sequence read before any is written.
 *   path: int32 [sequences, path_len], path_len <= MARIAN_HIP_TREE_MAX; accepted: int32 [sequences], taken into
 *   0 .. path_len.  A path entry below 0, or whose row is past the capacity, moves nothing.
 *   new_lens: int32 [sequences], apart from lens: min(lens[s] + accepted[s], capacity).
 */
int marian_hip_cache_keep(const marian_hip_kv_cache* cache, const int32_t* lens, const int32_t* path, int64_t path_len,
                          const int32_t* accepted, int32_t* new_lens, void* stream);

/*
 * Verification of drafted tokens: which of the tokens that a cheaper model proposed the target keeps, and the token that
 * follows them, such that the sequence is distributed as the target's own.  No counterpart in the reference.
 *   tokens: int32 [sequences, n], n up to MARIAN_HIP_TREE_MAX, in the order they were given to the target: token 0 of a sequence is
 *   settled (the one that the last step ended with), the others are drafted.
 *   counts, parents: as in marian_hip_drafts; token 0 stands for itself, and a drafted token whose parent is none (below 0, or not before it)
 *   is never reached.
 *   target: [sequences, n, vocab] of `type`, row i the target's probabilities after token i; words of a row side by side, the
 *   values between two sequences and two rows given (target_strides, any; aligned as the type is).
 *   draft: null, or likewise [sequences, n - 1, vocab], row i what token i + 1 was drawn from; parents has to be null then.
 *   random: float32 [sequences, n], each 0 <= u < 1 and independent of all else: random[s, 0] draws the next token, random[s, i] judges token i.
 * With p the target's row after a token's parent, t the token and u its number:
 *   draft given: t is kept if u * q(t) < p(t), q the draft's row; what follows the last kept token is drawn from max(p - q, 0) of its row
 *   if a drafted token was refused there, else from p;
 *   draft null (tokens that were not drawn, the drafter's best ones, in chains and trees): of the children of a kept token, in their
 *   order, the first with u * (1 - sum of p of those refused before it) < p(t) is kept (a token that a sibling had already: none of p is left);
 *   what follows is drawn from p without the tokens refused there.
 * Drawing from weights w: the first word whose sum of weights up to itself exceeds u * sum of all, so ties go to the lowest word; where
 * nothing is left (by rounding), from p itself; -1 where that is nothing, too.  Probabilities below zero and NaN count as zero, an infinite one leaves
 * the word open.  All in 64 bits.
 *   path: int32 [sequences, n], the kept tokens' numbers, 0 the first, then -1; accepted: int32 [sequences], how many (0 where counts is 0; next
 *   is -1 then): what marian_hip_cache_keep takes.  next: int32 [sequences].  Outputs share no memory with anything else.
 *   A token outside 0 .. vocab - 1 has probability zero.
 *   workspace: at least marian_hip_verify_drafts_workspace_bytes(sequences, vocab) bytes, 256-byte aligned (0 bytes: may be null), cleared
 *   once by marian_hip_cache_attention_workspace_init; one workspace serves one stream, and may be that of an attention.
 * sequences <= 65535, vocab < 2^24.
 */
typedef struct marian_hip_drafted {
  const int32_t* tokens;
  const int32_t* counts;
  const int32_t* parents;
  const void* target;
  const void* draft;
  const float* random;
  int64_t sequences, n, vocab;
  int64_t target_strides[2], draft_strides[2];
  int type;
} marian_hip_drafted;
size_t marian_hip_verify_drafts_workspace_bytes(int64_t sequences, int64_t vocab);
int marian_hip_verify_drafts(const marian_hip_drafted* drafted, int32_t* path, int32_t* accepted, int32_t* next, void* workspace,
                             size_t workspace_bytes, void* stream);

/*
 * A cache in pages: memory for keys and values that sequences share, dealt out `page` positions at a time.  No counterpart in the reference.
 *   k, v: [pages, heads, page, dk] of `type`, dense, 16-byte aligned; page a multiple of 8 up to 4096, dk as above, heads <= 4096,
 *   pages * page < 2^30.
 */
typedef struct marian_hip_pages {
  void* k;
  void* v;
  int64_t pages, heads, page, dk;
  int type;
} marian_hip_pages;

/*
 * Who has which pages, all on the device:
 *   table: int32 [sequences, row]: the pages of a sequence in the order of its positions, -1 behind them;
 *   held: int32 [sequences]: how many these are;
 *   free: int32 [pages]: a stack of the pages that nobody has, its first free_count[0] entries.
 * sequences <= 65535, row * sequences < 2^31.  A page belongs to one sequence; sequences that share one may read it only: one that two of them hold
 * would go back twice, and be dealt twice.
 * Calls on the same tables follow each other: on one stream, and of several threads one at a time (a call may be two launches).
 */
typedef struct marian_hip_page_tables {
  int32_t* table;
  int32_t* held;
  int32_t* free;
  int32_t* free_count;
  int64_t sequences, row, pages;
} marian_hip_page_tables;

/*
 * Makes room for n new tokens a sequence (counts: null, or int32 [sequences], only so many of them) behind lens[s] positions: every
 * sequence gets the pages that it lacks up to position lens[s] + counts[s], in the sequences' order from the top of the stack.  A sequence that the free
 * pages do not reach for, or whose row of the table is too short, gets none; so does every later one that lacks some, in the first case.
 *   slots: int32 [sequences, n]: where token i of sequence s lies, page number * page + place in it; -1 for tokens that are not
 *   there or have no page.  A sequence's tokens that have a slot come first: how many these are is what the rest of the step takes as counts, so that
 *   no length grows past what is written.
 * Lengths below 0 are taken as 0, counts into 0 .. n, held into 0 .. row, free_count into 0 .. pages.  n up to 2^20, sequences * n < 2^31.
 * Replays of a recorded call go on from what the table holds then.
 */
int marian_hip_pages_reserve(const marian_hip_page_tables* tables, const int32_t* lens, const int32_t* counts, int64_t n, int64_t page,
                             int32_t* slots, void* stream);

/*
 * Gives the pages behind lens[s] positions back, of every sequence (lens[s] = 0: all of them): what a refused draft or a finished
 * sequence leaves.  Undoes a marian_hip_pages_reserve with the same lens, the order of the stack included, where no sequence held pages behind its lens
 * before.
 */
int marian_hip_pages_trim(const marian_hip_page_tables* tables, const int32_t* lens, int64_t page, void* stream);

/*
 * Writes keys and values of n tokens a sequence, [sequences, heads, n, dk] of the cache's type by strides (as for
 * marian_hip_cache_append), to their slots: int32 [sequences, n]; a slot below 0 or past the last page writes nothing.  No two tokens of a call
 * have the same slot.  n up to 2^20, sequences * n * heads rows of less than 2^36 bytes in all.
 */
int marian_hip_pages_write(const marian_hip_pages* cache, const void* k, const int64_t* k_strides, const void* v, const int64_t* v_strides,
                           int64_t sequences, int64_t n, const int32_t* slots, void* stream);

/*
 * Attention of n new tokens a sequence over the pages that they have been written to: q and out [sequences, q_heads, n, dk] of the cache's type
 * by strides, q_heads a multiple of the cache's heads (query head h reads head h / (q_heads / heads)):
 *   out = softmax(scale * q . key) value
 * over the lens[s] positions before the new tokens, the token itself and the new ones before it.  table: int32 [sequences, row]; rows may share
 * pages.  Positions of a page that is none (below 0, or at or past `pages`), and past the row, are not seen.  What a token does not see is
 * not read into its result, infinities and NaN included; an infinity among the values that it sees is its result, whatever its weight, also where its
 * score is minus infinity (NaN if there are both, or one; a score that is plus infinity or NaN makes the row NaN).  A token that sees nothing, or whose
 * scores are all minus infinity, gives zeros but for that, and so do rows at or past counts[s] (counts: null, or int32 [sequences]).  out shares no
 * memory with anything else.
 * scale: finite, above zero.
 * Products and sums are float32; weights enter the product with the values with 16 bits (bfloat16), 22 (float16) or 24, their sum in float32.
 * Values (bfloat16 and float32) below 2^-100 lose bits to the scale of the weights.
 * The last bits of a result depend on the batch's lengths and the table's width, which say how positions are split over workgroups, and not on
 * the order of anything.  Made for few rows a head of keys, n * q_heads / heads: keys and values are read once for every 128 of them (up to 128
 * values a row, float32 more than 64), 32 (float32 up to 64 values, 16-bit types past 128), or 16 (float32 past 128).  A long sequence is
 * split over workgroups in calls of up to 1024 sequences, and the less so the more new tokens a call has room for: a long one among more sequences, or
 * beside a prompt, is better given a call of its own.
 * lens outside 0 .. row * page are taken as the nearer end.  sequences <= 65535, row * page < 2^30, sequences * row < 2^31, n up to 2^20,
 * q_heads / heads <= 4096, n * q_heads / heads <= 2^26, and sequences * heads times the workgroups that share an entry's rows (one to 16, 32, 64 or
 * 128 of them) less than 2^23.
 *   workspace: at least marian_hip_pages_attention_workspace_bytes(...) bytes, cleared once by marian_hip_cache_attention_workspace_init; as for
 *   marian_hip_cache_attention, whose workspace serves this call too where it is large enough.
 */
size_t marian_hip_pages_attention_workspace_bytes(int64_t sequences, int64_t heads, int64_t q_heads, int64_t n, int64_t dk, int type);
int marian_hip_pages_attention(const marian_hip_pages* cache, const int32_t* table, int64_t sequences, int64_t row, const int32_t* lens,
                               const int32_t* counts, int64_t n, const void* q, const int64_t* q_strides, int64_t q_heads, float scale, void* out,
                               const int64_t* out_strides, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* MARIAN_HIP_OPS_H */

/*
 * wgd.h — C ABI of the MI355X (gfx950) dense-decoder library `libwgd.so`.
 *
 * This boundary replaces the WebGPU layer of ahpah-dev/WebGPU's `src/core`:
 *   - `class Compute` (src/core/gpu.ts:2-67): device, budget-tracked buffers, ordered
 *     writes, dispatch, copies, clears, fences, read-back, deferred device faults;
 *   - the WGSL kernels (src/core/shaders.ts:13-181, src/core/qwen-shaders.ts:27-34),
 *     each a launcher below with the WGSL uniform parameter list;
 *   - the resident weight pager (src/core/pager.ts:7-47): weights live in HBM, one
 *     device allocation per tensor, so there is no paging slot;
 *   - the dense decoder step of `PagedEngine.forward/denseLayer` and the Gemma-3 body
 *     (src/core/engine.ts:138-180, 217-251) as `wgd_model_*`, run natively so a
 *     decode step is one captured HIP graph rather than hundreds of host calls.
 *
 * Conventions
 *   - Every function returns 0 on success and a non-zero WGD_E* status on failure.
 *     The message is kept per context and read with wgd_last_error(); the host
 *     bindings turn it into a thrown Error, as Compute does (gpu.ts:20-27).
 *   - All launches are asynchronous and strictly ordered on the context's single HIP
 *     stream, which gives the WebGPU queue-ordering guarantee (verify.ts:67-74).
 *     A device fault raised by an earlier launch is reported by the next wgd_done(),
 *     wgd_read() or model call (the deferred `fault` of gpu.ts:9,20-23).
 *   - Buffers are opaque handles owned by the context; host pointers are borrowed
 *     only for the duration of a call.
 *   - Quantization type ids are GGUF's (QUANTS, src/core/gguf.ts:6-11):
 *     F32 0, F16 1, Q4_0 2, Q8_0 8, Q4_K 12, Q5_K 13, Q6_K 14.
 *   - A context is used from one host thread at a time (engine.ts:258 `busy` guard).
 */
#ifndef WGD_H
#define WGD_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define WGD_OK 0
#define WGD_E_INVALID 1   /* bad argument, shape, type or size                 */
#define WGD_E_BUDGET 2    /* budget exceeded (gpu.ts:26)                       */
#define WGD_E_DEVICE 3    /* HIP runtime error or deferred device fault        */
#define WGD_E_NONFINITE 4 /* greedy sampling found no finite logit (engine.ts:308) */
#define WGD_E_STATE 5     /* call out of order (model not ready, destroyed)    */

typedef struct wgd_context wgd_context;
typedef struct wgd_buffer wgd_buffer;
typedef struct wgd_model wgd_model;

/* ---------------------------------------------------------------- runtime
 * Compute (src/core/gpu.ts:2-67). */

/* Compute constructor + init(): open HIP device `device`, create the ordered stream.
 * `budget_bytes` is the allocation ceiling (gpu.ts:7,26); 0 means the device's free
 * memory. On failure *out is NULL and the status says why (a NULL context message is
 * available from wgd_last_error(NULL)). */
int wgd_create(int32_t device, uint64_t budget_bytes, wgd_context **out);
/* Compute.dispose (gpu.ts:66): frees every buffer and model of the context. */
void wgd_destroy(wgd_context *ctx);
/* Message of the last failing call on `ctx` (thread-local message when ctx is NULL). */
const char *wgd_last_error(const wgd_context *ctx);
/* Compute.adapterName (gpu.ts:15). */
const char *wgd_adapter_name(const wgd_context *ctx);
/* Compute.allocated / Compute.peak (gpu.ts:4-5). */
uint64_t wgd_allocated(const wgd_context *ctx);
uint64_t wgd_peak(const wgd_context *ctx);

/* Compute.buffer (gpu.ts:24-30): size rounded up to 4 bytes, minimum 4; zero-filled. */
int wgd_buffer_create(wgd_context *ctx, uint64_t size, const char *label, wgd_buffer **out);
/* Compute.destroy (gpu.ts:31). */
int wgd_buffer_destroy(wgd_context *ctx, wgd_buffer *buf);
uint64_t wgd_buffer_size(const wgd_buffer *buf);
/* The device address of a buffer, for hosts that fill or read it with their own device code
 * ordered against wgd_stream(). It stays valid until the buffer is destroyed (NULL for a NULL
 * handle). Buffers of wgd_upload_weights hold this library's own layout. */
void *wgd_buffer_address(const wgd_buffer *buf);
/* WeightPager.page (pager.ts:25-44) with paging collapsed: upload a whole rows x cols weight
 * matrix of GGUF `type` once, in the layout the kernels read fastest. Q4_K, Q5_K and Q6_K
 * (and Q8_0 / Q4_0 of a width that is a multiple of 64) are rearranged on the device into a
 * planar layout of the same bits (16-byte quant chunks tiled by 16 rows, block headers and
 * scales in separate planes); other types keep the GGUF bytes. Decoded values are unchanged. The buffer is accepted by wgd_matmul, wgd_matvec and
 * wgd_embed for that type and shape. `bytes` must equal rows*rowBytes. */
int wgd_upload_weights(wgd_context *ctx, int32_t type, uint32_t cols, uint32_t rows,
                       const void *data, uint64_t bytes, const char *label, wgd_buffer **out);
/* The context's HIP stream (hipStream_t), for hosts that time or order work against it. */
void *wgd_stream(const wgd_context *ctx);
/* Compute.write (gpu.ts:32): ordered host→device copy of `bytes` at `offset`. */
int wgd_write(wgd_context *ctx, wgd_buffer *buf, uint64_t offset, const void *data, uint64_t bytes);
/* Compute.read (gpu.ts:61-65): waits for all queued work, then copies back. */
int wgd_read(wgd_context *ctx, const wgd_buffer *buf, uint64_t offset, void *out, uint64_t bytes);
/* Compute.copy (gpu.ts:52-54). */
int wgd_copy(wgd_context *ctx, const wgd_buffer *src, wgd_buffer *dst, uint64_t size,
             uint64_t src_offset, uint64_t dst_offset);
/* Compute.clear (gpu.ts:55-59): zero-fill the whole buffer. */
int wgd_clear(wgd_context *ctx, wgd_buffer *buf);
/* Compute.done (gpu.ts:60): wait for queued work and surface deferred faults. */
int wgd_done(wgd_context *ctx);

/* ---------------------------------------------------------------- kernels
 * One launcher per WGSL pipeline; parameters are the WGSL uniform fields. All tensors
 * are f32 unless stated; batch-major [batch][dim] layout as in engine.ts:94-96. */

/* matmulShader(type) (shaders.ts:39-54), dispatched by `linear` (engine.ts:125-137):
 *   y[b*stride + rowBase + r] = sum_c deq(W)[r*cols + c] * x[(b+inputOffset)*cols + c]
 * for r < rows, b < batch. W holds GGUF blocks of `type` (rows x cols, row-major,
 * quantized along cols). Batch 1 runs the decode matvec (wgd_quantize + wgd_matvec) where
 * the type and layout allow it; batches above 4, and any batch on planar weights, run the
 * dequant-GEMM on 16-bit MFMA with a split-precision activation operand; the rest runs a
 * generic f32 kernel. */
int wgd_matmul(wgd_context *ctx, int32_t type, const wgd_buffer *w, const wgd_buffer *x,
               wgd_buffer *y, uint32_t cols, uint32_t rows, uint32_t stride, uint32_t row_base,
               uint32_t input_offset, uint32_t batch);
/* The decode matvec split in its two steps, for hosts that drive single ops:
 * wgd_quantize turns an f32 activation row of `cols` elements into the quantized form the
 * integer matvec reads (buffer of wgd_quantized_bytes(cols)), optionally as RMSNorm(x) * w
 * (normShader, shaders.ts:55-68, with w = norm_weight, NULL for none); wgd_matvec then
 * computes y[row_base + r] = sum_c deq(W)[r][c] x[c] for weights uploaded with
 * wgd_upload_weights (every type; Q8_0 and Q4_0 in the planar layout, F16 and F32 rows of a
 * width that is a multiple of 16). wgd_matmul with batch 1 runs exactly these two. */
uint64_t wgd_quantized_bytes(uint32_t cols);
int wgd_quantize(wgd_context *ctx, const wgd_buffer *x, uint32_t cols, const wgd_buffer *norm_weight,
                 float epsilon, wgd_buffer *qx);
int wgd_matvec(wgd_context *ctx, int32_t type, const wgd_buffer *w, const wgd_buffer *qx, wgd_buffer *y,
               uint32_t cols, uint32_t rows, uint32_t row_base);
/* wgd_matvec once per launch shape that the decode step's launch-shape measurement may pick
 * for this matrix and input (the cost-model shape first; F16/F32 matrices have none): shape k
 * writes y[k * rows + r], for k < *count <= max_shapes, and y must hold max_shapes * rows
 * floats. Every shape computes the same bits, which is what a caller checks with it; no
 * reference counterpart (the measurement is this library's own). */
int wgd_matvec_shapes(wgd_context *ctx, int32_t type, const wgd_buffer *w, const wgd_buffer *qx, wgd_buffer *y,
                      uint32_t cols, uint32_t rows, uint32_t max_shapes, uint32_t *count);
/* decodeWeight (src/core/quant.ts:6-29) for `count` consecutive elements: out[i] =
 * deq(W)[i] rounded once to f32, bit-identical to the reference's decode. */
int wgd_dequant(wgd_context *ctx, int32_t type, const wgd_buffer *w, wgd_buffer *out,
                uint64_t count);
/* normShader (shaders.ts:55-68): y = x * inverseSqrt(mean(x^2) + eps) * w per row of n. */
int wgd_norm(wgd_context *ctx, const wgd_buffer *x, const wgd_buffer *w, wgd_buffer *y,
             uint32_t n, float epsilon, uint32_t batch);
/* ropeShader (shaders.ts:69-87): per (token, head) RMS-normalise with `w` (Q/K norm),
 * then half-split rotation of the first `rotary_dim` dims (0 = head_dim) by angle
 * (start+t)*scale/theta^(2i/rot); the tail is only normalised. In place on x. */
int wgd_rope_norm(wgd_context *ctx, wgd_buffer *x, const wgd_buffer *w, uint32_t heads,
                  uint32_t head_dim, uint32_t start, float theta, float scale, float epsilon,
                  uint32_t rotary_dim, uint32_t batch);
/* ropeNeoxShader (shaders.ts:139-152): half-split pairs (i, i+rot/2). */
int wgd_rope_neox(wgd_context *ctx, wgd_buffer *x, uint32_t heads, uint32_t head_dim,
                  uint32_t start, float theta, float scale, uint32_t rotary_dim, uint32_t batch);
/* ropeClassicShader (shaders.ts:155-168): adjacent pairs (2j, 2j+1). */
int wgd_rope_adjacent(wgd_context *ctx, wgd_buffer *x, uint32_t heads, uint32_t head_dim,
                      uint32_t start, float theta, float scale, uint32_t rotary_dim,
                      uint32_t batch);
/* attentionShader(context) (shaders.ts:88-122): causal GQA for query token b and head h
 * over keys t in [end - min(end, window), end), end = start + b + 1, key/value row at
 * ring slot t % capacity of a [capacity][kvHeads][hd] cache, kv head h/(heads/kvHeads).
 * capacity 0 selects `context` as in the WGSL constant. hd <= 512. Split-K over the
 * key range with an online-softmax combine. */
int wgd_attention(wgd_context *ctx, const wgd_buffer *q, const wgd_buffer *k,
                  const wgd_buffer *v, wgd_buffer *y, uint32_t heads, uint32_t kv_heads,
                  uint32_t head_dim, uint32_t start, float scale, uint32_t window,
                  uint32_t capacity, uint32_t context, uint32_t batch);
/* wgd_attention with no allocation: no counterpart in the reference. For callers that
 * cannot allocate device memory (code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc). Same arguments and the same results, bit for bit: the
 * split-K partials go to a static array in the library's device memory (one per GPU, held
 * until the process ends) instead of context scratch. Sizes whose partials exceed
 * wgd_attention_noalloc_limit() floats fail with WGD_E_INVALID. Calls on one GPU share the
 * array: calls that overlap on one GPU (two streams) race. */
int wgd_attention_noalloc(wgd_context *ctx, const wgd_buffer *q, const wgd_buffer *k,
                          const wgd_buffer *v, wgd_buffer *y, uint32_t heads, uint32_t kv_heads,
                          uint32_t head_dim, uint32_t start, float scale, uint32_t window,
                          uint32_t capacity, uint32_t context, uint32_t batch);
/* wgd_attention over an f16 K/V ring: the same arguments and semantics, with k and v
 * holding [capacity][kvHeads][hd] IEEE halves (2 bytes per element) instead of f32. Scores,
 * softmax and the weighted sum run in f32 on the exactly widened values. The reference
 * allocates its rings at 4 bytes per element (engine.ts:98-101, sized by attentionMemory,
 * context.ts:16-24); the f16 ring halves that memory and the bytes each decode step reads. */
int wgd_attention_f16kv(wgd_context *ctx, const wgd_buffer *q, const wgd_buffer *k,
                        const wgd_buffer *v, wgd_buffer *y, uint32_t heads, uint32_t kv_heads,
                        uint32_t head_dim, uint32_t start, float scale, uint32_t window,
                        uint32_t capacity, uint32_t context, uint32_t batch);
/* cacheKV's ring copy (engine.ts:120-124, Compute.copy of cacheCopies' ranges) into an f16
 * ring: dst[dst_offset + i] = f16(src[src_offset + i]) for i < count, rounded to nearest
 * (ties to even). Offsets and count are in elements (floats of src, halves of dst). */
int wgd_kv_store_f16(wgd_context *ctx, const wgd_buffer *src, wgd_buffer *dst, uint64_t count,
                     uint64_t src_offset, uint64_t dst_offset);
/* Floats of the static scratch of wgd_attention_noalloc (8 Mi floats, 32 MiB). */
uint64_t wgd_attention_noalloc_limit(void);
/* addShader (shaders.ts:123-128): state += delta. */
int wgd_add(wgd_context *ctx, const wgd_buffer *delta, wgd_buffer *state, uint32_t n);
/* siluShader (qwen-shaders.ts:27-34): y = g / (1 + exp(-g)) * up. */
int wgd_silu(wgd_context *ctx, const wgd_buffer *gate, const wgd_buffer *up, wgd_buffer *y,
             uint32_t n);
/* geluShader (shaders.ts:129-137): y = 0.5 g (1 + tanh(0.7978845608 (g + 0.044715 g^3))) up. */
int wgd_gelu(wgd_context *ctx, const wgd_buffer *gate, const wgd_buffer *up, wgd_buffer *y,
             uint32_t n);
/* biasAddShader (shaders.ts:170-175): y[i] += b[i % width]. */
int wgd_bias_add(wgd_context *ctx, wgd_buffer *y, const wgd_buffer *b, uint32_t n,
                 uint32_t width);
/* activateShader (shaders.ts:177-181): in-place x = x / (1 + exp(-x)). */
int wgd_activate(wgd_context *ctx, wgd_buffer *x, uint32_t n);
/* sample(T=0) (engine.ts:305-309) on the device: index of the first strict maximum over
 * the finite entries of logits[0..n). Writes an int32 to out (-1 when none is finite)
 * and, when host_index is non-NULL, waits and returns it there, failing with
 * WGD_E_NONFINITE when no entry is finite. */
int wgd_argmax(wgd_context *ctx, const wgd_buffer *logits, uint32_t n, wgd_buffer *out,
               int32_t *host_index);
/* sample (engine.ts:305-324) on the device for logits[0..n): the first finite maximum
 * when temperature is 0, else the top_k finite logits (ties to the lower index),
 * exp((l - best) / T) in f64, the top_p prefix and a draw with the index-th output of
 * splitmix64(seed) as Math.random(). Waits; returns the token (WGD_E_NONFINITE when no
 * logit is finite, WGD_E_INVALID for settings the reference rejects). */
int wgd_sample(wgd_context *ctx, const wgd_buffer *logits, uint32_t n, double temperature, uint32_t top_k,
               double top_p, uint64_t seed, uint32_t index, int32_t *token);
/* Embedding gather of `forward` (engine.ts:140-145) on the device:
 * out[b*hidden + i] = f32(deq(table)[ids[b]*hidden + i] * scale) with the product taken
 * in f64 (scale = sqrt(hidden) for Gemma 3, else 1). ids is int32[n]. */
int wgd_embed(wgd_context *ctx, int32_t type, const wgd_buffer *table, const wgd_buffer *ids,
              wgd_buffer *out, uint32_t hidden, uint32_t n, double scale);

/* ---------------------------------------------------------------- drafted trees
 * One decode step over a tree of drafted tokens (no reference counterpart): a host drafts
 * `nodes` tokens after the `start` cached ones, runs the model over all of them as one batch,
 * and keeps the path that the model's own draws confirm. Node i has the position start + its
 * depth and its K/V in ring slot (start + i) % capacity. parents (int32[nodes], on the device)
 * holds the node that i follows, in [0, i), or -1 where it follows the last cached token; node 0
 * is the token that the step before picked. Any other value makes i and every node below it
 * padding: attention writes zeros for it and no path takes it, so trees of several sizes can
 * share one launch shape. The launches allocate nothing once a call of the same sizes has run,
 * so they can be captured into HIP graphs; where their scratch would have to grow during a
 * capture they fail with WGD_E_STATE and the capture stays valid. Graphs keep using the
 * context's scratch: replay them in order with its other work. */
#define WGD_TREE_MAX 256 /* most nodes of a tree */

/* Rotary embedding at given positions, in place: for token t < batch and head h < heads, x at
 * t * stride + offset + h * head_dim (floats; stride 0: heads * head_dim) has its first
 * rotary_dim dims (0 = head_dim) rotated pairwise, (j, j + rot/2) or with `adjacent` (2j, 2j+1):
 *   (l, r) -> magnitude * (l cos a - r sin a, l sin a + r cos a),
 *   a = positions[t] * scale * theta^(-2j/rot) / factors[j].
 * positions is int32[batch], factors f32[rot/2] or NULL for ones; linear, NTK, by-parts (YaRN)
 * and Llama 3 scaling are factors and a magnitude (webgpu_amd/rope.py makes them). Angles are
 * formed and reduced in f64, their cosine and sine are off by at most 2^-29 before they are rounded
 * to f32, and the tail of a head is left as it is. Query and key heads that lie side by side in
 * a row are one call. For models with Q/K norm run wgd_norm with n = head_dim first. */
int wgd_rope_at(wgd_context *ctx, wgd_buffer *x, const wgd_buffer *positions, const wgd_buffer *factors,
                uint32_t heads, uint32_t head_dim, float theta, float scale, float magnitude, uint32_t rotary_dim,
                uint32_t stride, uint64_t offset, int32_t adjacent, uint32_t batch);
/* Attention of every node of a drafted tree: query q[i][h] over the cached keys t in
 * (position_i - window, start), at ring slot t % capacity as in wgd_attention, and over i itself
 * and its ancestors within the window; y[i][h] = softmax(scale * q.k) V, zeros for padding. A
 * node outside i's ancestors never reaches y[i], whatever its K/V hold; NaN and infinities there
 * have the rows that share a workgroup with them formed again, some hundred times slower. Needs nodes <=
 * WGD_TREE_MAX, head_dim <= 512, start < 2^31, heads <= 2^20, nodes * heads < 2^26, nodes * heads /
 * kv_heads <= 1048560 and a ring that holds every key that some node sees, min(start, window - 1) + nodes
 * <= capacity. */
int wgd_attention_tree(wgd_context *ctx, const wgd_buffer *q, const wgd_buffer *k, const wgd_buffer *v, wgd_buffer *y,
                       const wgd_buffer *parents, uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t start,
                       float scale, uint32_t window, uint32_t capacity, uint32_t nodes);
/* The same over f16 rings (wgd_attention_f16kv's). Scores, maxima, sums and outputs are f32; with a head_dim
 * that is a multiple of 8, up to 256, queries and weights enter the products as two f16 each: an
 * entry of a query is off by 2^-22 of itself and 2^-39 of the row's largest, a weight by 2^-22 of
 * itself and 2^-36 of the largest one. */
int wgd_attention_tree_f16kv(wgd_context *ctx, const wgd_buffer *q, const wgd_buffer *k, const wgd_buffer *v,
                             wgd_buffer *y, const wgd_buffer *parents, uint32_t heads, uint32_t kv_heads,
                             uint32_t head_dim, uint32_t start, float scale, uint32_t window, uint32_t capacity,
                             uint32_t nodes);
/* One token for each of `rows` rows of n logits, `stride` floats apart (0: n), drawn with the
 * caller's uniforms (f64[rows] in [0, 1)) into tokens (int32[rows]) on the device, without
 * waiting. The finite logits in descending order, ties to the lower index, have weights
 * exp((l - best) / temperature); kept are the top_k first (0: all of them), of these the
 * shortest prefix whose share of their weight reaches top_p, and of these the ones with a weight
 * of min_p or more; the token is the first whose running sum reaches uniform * (the kept
 * weight). With min_p 0 that is wgd_sample's rule. Weights are formed to 2^-45 of themselves; they and
 * their sums are integers of 2^-min(51, 62 - ceil(log2 n)) of the largest weight, so a draw does not
 * depend on the order of the sums.
 * Temperature 0 takes the best; so does a uniform outside [0, 1). A row without a finite logit
 * gets -1. temperature <= 2, 0 < top_p <= 1, 0 <= min_p <= 1 (WGD_E_INVALID otherwise). */
int wgd_sample_rows(wgd_context *ctx, const wgd_buffer *logits, uint32_t n, uint32_t rows, uint32_t stride,
                    const wgd_buffer *uniforms, wgd_buffer *tokens, double temperature, uint32_t top_k, double top_p,
                    double min_p);
/* The drafted path that the model confirms: from node 0, the lowest child i of the node c reached
 * with drafted[i] == picked[c] (the token drawn at c), until none is. path (int32[nodes + 2])
 * becomes the count of nodes on it, the token picked at the last one, their indices in
 * order, and -1 behind them; count 0 and token -1 where node 0 is padding. A negative picked
 * token ends the path. */
int wgd_tree_accept(wgd_context *ctx, const wgd_buffer *parents, const wgd_buffer *drafted, const wgd_buffer *picked,
                    wgd_buffer *path, uint32_t nodes);
/* Moves the K/V rows of an accepted path (as wgd_tree_accept writes it) to the slots that its
 * tokens keep: row (start + path[2 + j]) % capacity of every ring to row (start + j) % capacity,
 * for j < path[0]; the other rows stay. `rings` is a host array of `count` distinct buffers (at most
 * 65536) of [capacity][row_bytes] (K and V of any number of layers; row_bytes = kv_heads * head_dim * 4, or
 * * 2 for f16 rings, a multiple of 2); nodes <= capacity. Entries of the path that do not lie
 * beyond their own place and below `nodes` move nothing. */
int wgd_kv_commit(wgd_context *ctx, wgd_buffer *const *rings, uint32_t count, const wgd_buffer *path,
                  uint64_t row_bytes, uint32_t start, uint32_t capacity, uint32_t nodes);

/* ---------------------------------------------------------------- many requests
 * A step of a batch of requests (no reference counterpart). Their keys and values lie in pages: of one
 * K and one V pool per layer, [pages][page][kv_heads][head_dim] in f32 or f16, page `table[r * max_pages + c]` holds
 * the tokens c * page .. + page of request r (int32[requests][max_pages]); lengths[r] (int32) is how many tokens it has
 * and refs[p] (int32[pages]) how many rows of the table hold page p; 0 or less is a free page. Zero-filled buffers are the empty
 * state. A host that keeps pages itself adds to their refs. The page is a power of two up to WGD_PAGE_MAX; requests <=
 * WGD_REQUESTS_MAX; max_pages * page and pages * page are below 2^31. Lengths outside [0, max_pages * page] count as
 * the nearest end (wgd_pages_extend refuses such a request, with -1 in `added`, and leaves its length). These launches
 * wait for nothing, and their choices do not depend on the order of threads. They allocate nothing once a call of the same
 * sizes has run (WGD_E_STATE where a capture would have to); captured ones share the context's scratch, so graphs are
 * replayed in order with its other work. Buffers that a call writes are others than those that it reads, unless it says so. */
#define WGD_REQUESTS_MAX 1024
#define WGD_PAGE_MAX 1024

/* Places for counts[r] (int32[requests], in [0, tokens]; NULL: `tokens` each) new tokens of every request: in the
 * order of requests, each takes the lowest free pages that it needs beyond those it has, or where fewer are left none
 * at all: then, and where the tokens do not fit max_pages, or counts[r] or lengths[r] lies outside, added[r] (int32[requests]) becomes -1
 * and the request stays as it was, while later ones may still fit. Else added[r] = counts[r], which is what lengths[r] grows
 * by; positions[r * tokens + t] (for wgd_rope_at) and slots[r * tokens + t] (page * id + place, for wgd_pages_store) are
 * those of its t-th new token, and -1 where there is none (both int32[requests * tokens]). requests * tokens <= 2^24. */
int wgd_pages_extend(wgd_context *ctx, wgd_buffer *table, wgd_buffer *lengths, wgd_buffer *refs, const wgd_buffer *counts,
                     wgd_buffer *added, wgd_buffer *positions, wgd_buffer *slots, uint32_t requests, uint32_t tokens,
                     uint32_t page, uint32_t max_pages, uint32_t pages);
/* Requests that fork, end or lose their last tokens: request r becomes the first keep[r] tokens (NULL, or more than
 * there are: all) of what request origin[r] was (both int32[requests]); an origin outside [0, requests) leaves it empty. So
 * origin[r] = r keeps r (cut to keep[r]), another one makes r its copy, -1 frees it. Full pages are shared. A last page that is not
 * full belongs to one request alone: if nobody else holds it, it stays with the lowest of those that end in it; the
 * others, in order, get the lowest free pages, and copies (int32[2 * requests + 1]) becomes the number of these and their
 * (source, target) pairs, -1 behind them: run wgd_pages_copy with it on the pools of all layers before anything is
 * written to them. Pages that are no longer held are free. Where the free pages do not suffice nothing changes and copies[0] is
 * -1. Columns behind a changed request's last page become -1. */
int wgd_pages_fork(wgd_context *ctx, wgd_buffer *table, wgd_buffer *lengths, wgd_buffer *refs, const wgd_buffer *origin,
                   const wgd_buffer *keep, wgd_buffer *copies, uint32_t requests, uint32_t page, uint32_t max_pages,
                   uint32_t pages);
/* Compaction: with n pages in use, the j-th used one at n or above moves to the j-th free one below n, so that the used
 * pages are the first n. moved (int32[pages]) becomes every used page's new number, -1 for free ones; copies (int32[2 *
 * (pages / 2) + 1]) the number of moves and their (source, target) pairs, -1 behind them, for wgd_pages_copy. table_to and
 * refs_to are the table and counts afterwards; they may be table and refs themselves. Without that the old ones stay
 * valid until a page is written. Entries of the table outside [0, pages) stay. */
int wgd_pages_compact(wgd_context *ctx, const wgd_buffer *table, const wgd_buffer *refs, wgd_buffer *table_to,
                      wgd_buffer *refs_to, wgd_buffer *moved, wgd_buffer *copies, uint32_t requests, uint32_t max_pages,
                      uint32_t pages);
/* Page copies[1 + 2 i] to page copies[2 + 2 i] for i < copies[0] <= most, in every one of `count` distinct pools (a host
 * array, at most 65536; copies as the calls above write it: targets differ from one another and from all sources) of [pages][page_bytes],
 * page_bytes a multiple of 2 up to 2^30. Pairs with a number outside [0, pages) move nothing. */
int wgd_pages_copy(wgd_context *ctx, wgd_buffer *const *pools, uint32_t count, const wgd_buffer *copies, uint32_t most,
                   uint64_t page_bytes, uint32_t pages);
/* K and V rows of new tokens into the pools: row t < rows, `row` = kv_heads * head_dim floats at k + k_offset + t * stride
 * and v + v_offset + t * stride (floats; stride 0: row; k and v may be one buffer), to slot slots[t] of pools of
 * slots_in_pool = pages * page rows. Slots are distinct; those outside [0, slots_in_pool) store nothing. */
int wgd_pages_store(wgd_context *ctx, const wgd_buffer *k, const wgd_buffer *v, wgd_buffer *k_pool, wgd_buffer *v_pool,
                    const wgd_buffer *slots, uint32_t row, uint32_t rows, uint32_t stride, uint64_t k_offset,
                    uint64_t v_offset, uint32_t slots_in_pool);
/* The same into pools of halves, rounded to nearest (ties to even). */
int wgd_pages_store_f16kv(wgd_context *ctx, const wgd_buffer *k, const wgd_buffer *v, wgd_buffer *k_pool,
                          wgd_buffer *v_pool, const wgd_buffer *slots, uint32_t row, uint32_t rows, uint32_t stride,
                          uint64_t k_offset, uint64_t v_offset, uint32_t slots_in_pool);
/* Attention of the last counts[r] tokens of every request (int32[requests], as `added` of wgd_pages_extend; NULL:
 * `tokens`; none where it is 0 or less, at most `tokens` and lengths[r]): q[r][t][h] at the position p = lengths[r] - counts[r] + t
 * sees the keys (p - window, p] of its request; y[r][t][h] = softmax(scale * q.k) V, zeros for t >= counts[r]. q and
 * y are [requests][tokens][heads][head_dim], the keys of these tokens are stored already. Keys on pages outside [0, pages)
 * are not seen, and a row that sees none gets zeros. What a row does not see never reaches it, whatever its K/V hold.
 * shared > 0 (a multiple of page): requests that hold the same page in column shared / page - 1 as request `owner` hold the
 * same ones in all columns before it, as wgd_pages_fork makes them; their first `shared` tokens are then computed together, for requests
 * with new tokens, all of them behind the prefix, that the window does not cut. Results are the formula's either way.
 * head_dim <= 512, heads <= 2^20, requests * tokens * heads <= 2^25, tokens * heads / kv_heads <= 2^20. */
int wgd_attention_pages(wgd_context *ctx, const wgd_buffer *q, const wgd_buffer *k_pool, const wgd_buffer *v_pool,
                        wgd_buffer *y, const wgd_buffer *table, const wgd_buffer *lengths, const wgd_buffer *counts,
                        uint32_t heads, uint32_t kv_heads, uint32_t head_dim, float scale, uint32_t window, uint32_t page,
                        uint32_t max_pages, uint32_t pages, uint32_t requests, uint32_t tokens, uint32_t shared,
                        uint32_t owner);
/* The same over pools of halves. Scores, maxima, sums and outputs are f32; with a head_dim that is a multiple of 8, up to 256,
 * queries and weights enter the products as two f16 each: an entry of a query is off by 2^-22 of itself and 2^-39 of its row's largest, a weight
 * by 2^-22 of itself and 2^-36 of the largest one. Both forms: rows that see a value that is not finite, or a page that is none, have those that
 * share a workgroup with them formed again one product at a time, some hundred times slower; so are head_dims that
 * are no multiple of 8 or above 256. */
int wgd_attention_pages_f16kv(wgd_context *ctx, const wgd_buffer *q, const wgd_buffer *k_pool, const wgd_buffer *v_pool,
                              wgd_buffer *y, const wgd_buffer *table, const wgd_buffer *lengths, const wgd_buffer *counts,
                              uint32_t heads, uint32_t kv_heads, uint32_t head_dim, float scale, uint32_t window,
                              uint32_t page, uint32_t max_pages, uint32_t pages, uint32_t requests, uint32_t tokens,
                              uint32_t shared, uint32_t owner);
/* Low-rank adapters beside a projection (run it with wgd_matmul first): for rows t < batch with the adapter w =
 * which[t] (int32[batch]),
 *   y[t * stride + row_base + r] += scales[w] * sum_k B[w][r][k] (sum_c A[w][k][c] x[t][c]),  r < rows, k < rank, c < cols;
 * rows with w outside [0, adapters) stay as they are, as does what lies around them. a is [adapters][rank][cols] and b
 * [adapters][rows][rank], both F32 or F16 (`type`; GGUF's lora_a and lora_b as they are), lower ranks filled up with zeros;
 * scales f32[adapters] (alpha / rank). Sums are f32, and products too with F32 weights; with F16 ones x and the inner sums enter
 * them as two f16 each: an entry is off by 2^-22 of itself and 2^-39 of its row's largest
 * (64 inner sums at a time), and an infinity beside a weight may become NaN. rank <= 1024, cols and rows < 2^31, batch <= 2^24. */
int wgd_adapters(wgd_context *ctx, int32_t type, const wgd_buffer *a, const wgd_buffer *b, const wgd_buffer *which,
                 const wgd_buffer *scales, const wgd_buffer *x, wgd_buffer *y, uint32_t cols, uint32_t rows, uint32_t rank,
                 uint32_t adapters, uint32_t stride, uint32_t row_base, uint32_t batch);

/* ---------------------------------------------------------------- measurement
 * No reference counterpart: `launches` back-to-back plain streaming reads of `bytes`
 * (multiple of 16), launch i reading copy i % copies of src (copies laid out `bytes`
 * rounded up to 4 KiB apart), by `workgroups` workgroups of `threads` threads with `depth`
 * (4, 8, 16) 16-byte loads in flight per lane, a contiguous range per workgroup. With
 * out_floats > 0 each workgroup also stores its share of an out_floats-long result into
 * out. It is the per-launch floor of a kernel that reads those bytes once (bench.py
 * --probe); the loop runs in the library so the host does not pace short launches. */
int wgd_probe_read(wgd_context *ctx, const wgd_buffer *src, uint64_t bytes, uint32_t copies,
                   uint32_t launches, uint32_t workgroups, uint32_t threads, uint32_t depth,
                   wgd_buffer *out, uint32_t out_floats);

/* ---------------------------------------------------------------- model
 * The dense decoder step (engine.ts:138-180, 217-251) with resident weights. */

typedef struct wgd_model_config {
  int32_t family;         /* 0 dense decoder (llama/qwen2/qwen3), 1 gemma3  (gguf.ts:141)   */
  int32_t rope_adjacent;  /* 1 = adjacent pairs ('norm', arch llama), 0 = half-split (:168) */
  int32_t hidden, intermediate, layers, heads, kv_heads, head_dim, vocab;
  int32_t rotary_dim;     /* rotated dims per head (gguf.ts:166)                          */
  int32_t window;         /* attention window for local/sliding layers; 0 = context        */
  int32_t period;         /* gemma3: layer l is global iff l % period == period-1 (:162)   */
  int32_t qk_norm, ffn_gate, gelu;             /* detected from tensors (gguf.ts:197-199) */
  int32_t bias_q, bias_k, bias_v, bias_output;
  int32_t tied_output;    /* no output.weight: the head reuses token_embd (engine.ts:178) */
  int32_t context;        /* LoadOptions.contextLength (engine.ts:55)                      */
  int32_t batch;          /* LoadOptions.batchSize: largest forward() chunk                 */
  float epsilon, theta, local_theta, attention_scale, rope_scale;
  double embed_scale;     /* sqrt(hidden) for gemma3, 1 otherwise (engine.ts:143)          */
  int32_t kv_f16;         /* K/V rings in f16 (1) or f32 as the reference (0, engine.ts:98-101);
                             f16 rings store values rounded to nearest even, math stays f32 */
} wgd_model_config;

/* Allocate work buffers and per-layer K/V rings (capacities[l] slots each, from
 * attentionMemory, context.ts:16-24; 4 bytes per element, 2 with kv_f16). */
int wgd_model_create(wgd_context *ctx, const wgd_model_config *cfg, const int32_t *capacities,
                     wgd_model **out);
/* Upload one GGUF tensor (raw block bytes as stored in the file, `bytes` long).
 * 1-D tensors (norm vectors, biases) are decoded to f32 on the device as in
 * engine.ts:102-109. Names are GGUF's ("blk.3.attn_q.weight", ...). */
int wgd_model_tensor(wgd_model *m, const char *name, int32_t type, int32_t n_dims,
                     const uint64_t *dims, const void *data, uint64_t bytes);
/* Check that every tensor the config needs is present and shaped as modelConfig
 * validates it (gguf.ts:188-241); after this the model accepts forward calls. */
int wgd_model_ready(wgd_model *m);
/* PagedEngine.forward (engine.ts:138-180) for ids[0..n) at positions start..start+n-1
 * (n <= batch). When logits or argmax is non-NULL the last row's logits are produced
 * (vocab f32 copied to `logits`; the next token to `argmax`, WGD_E_NONFINITE if no logit
 * is finite: the greedy id, or with sampling set the draw for position start + n). */
int wgd_model_forward(wgd_model *m, const int32_t *ids, int32_t n, int32_t start,
                      float *logits, int32_t *argmax);
/* The decode loop of generate (engine.ts:290-298) kept on the device: for i < count, run
 * forward([token_i], start+i) and take token_{i+1} by the model's token pick (greedy, or
 * sampled as set by wgd_model_sampling); token_0 = `token`. Writes token_1..token_count to
 * out_tokens. Each step is one replay of a captured HIP graph (one per pick mode);
 * positions and ids never leave the device between steps. */
int wgd_model_decode(wgd_model *m, int32_t token, int32_t start, int32_t count,
                     int32_t *out_tokens);
/* The token pick of generate (engine.ts:261-264, 292, 305-324) for wgd_model_forward and
 * wgd_model_decode: temperature 0 is greedy; otherwise top_k / top_p sampling on the
 * device, where Math.random() becomes the p-th output of splitmix64(seed) for the token
 * at position p (the same tokens whether decoded eagerly, in chunks or by graph replay).
 * Validated as the reference validates GenerationOptions (WGD_E_INVALID). */
int wgd_model_sampling(wgd_model *m, double temperature, uint32_t top_k, double top_p, uint64_t seed);
void wgd_model_destroy(wgd_model *m);
/* Measurement, no reference counterpart: the mean device time in microseconds (HIP events
 * on the context's stream) of `reps` back-to-back launches of the decode step's attention
 * of `layer` at position `pos` (Q/K norm and RoPE of the token, its K/V written to ring slot
 * pos % capacity, split-K attention over the keys before it, merge and quantization for the
 * O projection), on the token's current q/k/v work buffers. It overwrites that ring slot, so
 * call it where the slot holds no live key. Models whose decode step has no fused attention
 * launch return WGD_E_INVALID. */
int wgd_model_attention_timing(wgd_model *m, int32_t layer, int32_t pos, int32_t reps, double *us);

#ifdef __cplusplus
}
#endif
#endif /* WGD_H */

/*
 * pcl_attention.h — C ABI of the MI355X (gfx950) attention backend for the
 * power-cpu-llm engine.
 *
 * Layouts are the engine's (src/kernels/portable/reference.rs:320-326):
 *   query  [qheads][dim] per query position,
 *   keys   [nkeys][kvheads][dim], values the same (token-major f32 cache),
 *   GQA    query head h reads KV head h / (qheads / kvheads),
 *   scale  exactly one (callers pre-scale the query).
 * Results match the reference's exact f32 attention within 1e-4 max-abs and
 * do not depend on the head range, the query batch, the KV-head range or the
 * kernel chosen: every (query, head) row is computed by the same arithmetic.
 *
 * Its parts, all plain C types:
 *   1. kernel entry points with the engine's function-pointer signatures
 *      (host pointers, bool result, false = error);
 *   2. checked wrappers with the reference wrappers' validation and error
 *      codes;
 *   3. a device-resident entry (device pointers, descriptor masks, two KV
 *      segments, asynchronous on a caller-visible stream);
 *   4. a device-resident layer cache whose rows the entry of 3 reads in
 *      place;
 *   5. the head transform that prepares Q, K and V rows for 3 and 4;
 *   6. the attention output block (projection, post-norm, residual);
 *   7. batches of requests over a paged cache: page bookkeeping, appends and
 *      single-token attention;
 *   8. drafted tokens, parts of prompts and shared pages over a paged cache.
 */
#ifndef PCL_ATTENTION_H
#define PCL_ATTENTION_H

#include <stdbool.h>
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- 1. kernel entry points (host pointers) ------------------------------ */

/* One query position, query heads [h_first, h_end).
 * Replaces the AttentionF32 function pointer type
 * (src/kernels/quantized/int8.rs:576-589), i.e. pa_attention_f32_heads
 * (src/kernels/portable/attention.rs:51-64) and pa_attention_f32_power9_heads
 * (src/kernels/quantized/int8.rs:155-168); the exact p9_ref_attention_heads
 * (src/kernels/portable/reference.rs:327-340) has the same arguments.
 * query [qheads*dim], keys/values [nkeys*kvheads*dim], allowed NULL or
 * [nkeys] 0/1, scratch is the caller's host scratch (unused here),
 * out [(h_end-h_first)*dim]. False on bad geometry (dim % 16, kvheads 0,
 * qheads % kvheads, head range, dim > 512), a non-finite allowed score, a
 * non-finite output, or a device failure. */
bool pcl_hip_attention_f32_heads(const float *query, const float *keys, const float *values,
                                 size_t qheads, size_t kvheads, size_t dim, size_t nkeys,
                                 const uint8_t *allowed, float *scratch, float *out,
                                 size_t h_first, size_t h_end);

/* Several query positions over the same K/V, KV heads [kh_first, kh_end).
 * Replaces the AttentionMulti function pointer type
 * (src/kernels/quantized/int8.rs:446-484), i.e.
 * pa_attention_f32_power9_multi_kv. query [nq][q_stride] (qheads*dim used),
 * allowed NULL or [nq][mask_stride], out [nq][o_stride] holding the query
 * heads kh_first*group .. kh_end*group. Every row equals the single-query
 * entry's result bitwise. */
bool pcl_hip_attention_f32_multi_kv(const float *query, size_t nq, size_t q_stride,
                                    const float *keys, const float *values, size_t qheads,
                                    size_t kvheads, size_t dim, size_t nkeys,
                                    const uint8_t *allowed, size_t mask_stride, float *scratch,
                                    float *out, size_t o_stride, size_t kh_first, size_t kh_end);

/* ---- 2. checked wrappers (reference wrapper semantics) ------------------- */

/* Error codes of kernels::reference::Error (src/kernels/reference.rs:6-11). */
enum pcl_status {
    PCL_OK = 0,
    PCL_INVALID_SHAPE = 1,
    PCL_INVALID_PARAMETER = 2,
    PCL_NON_FINITE_VALUE = 3,
    /* engine::Error::ResourceLimit: a cache's position or byte limit */
    PCL_RESOURCE_LIMIT = 4,
};

/* attention_with (src/kernels/quantized/int8.rs:596-663) over this backend:
 * FmaKernels::attention_heads for the HIP backend
 * (src/kernels/quantized/power9_fma.rs:237-255). Lengths are element
 * counts; has_mask / has_heads stand for Option::Some. A mask entry is a
 * bool (0 or 1). out holds (h_end-h_first)*head_dim floats. */
int pcl_attention_heads(const float *query, size_t query_len, const float *keys,
                        size_t keys_len, const float *values, size_t values_len,
                        size_t kv_heads, size_t head_dim, const uint8_t *allowed,
                        size_t mask_len, int has_mask, size_t h_first, size_t h_end,
                        int has_heads, float *out);

/* attention_multi_with (src/kernels/quantized/int8.rs:489-573):
 * FmaKernels::attention_multi_kv (power9_fma.rs:197-232). queries: nq
 * pointers to query_len floats; masks: NULL or nq pointers to mask_len
 * bools; out: nq rows of (kv_end-kv_first)*group*head_dim floats. */
int pcl_attention_multi_kv(const float *const *queries, size_t nq, size_t query_len,
                           const float *keys, size_t keys_len, const float *values,
                           size_t values_len, size_t kv_heads, size_t head_dim,
                           const uint8_t *const *masks, size_t mask_len, size_t kv_first,
                           size_t kv_end, float *out);

/* ---- 3. device-resident entry -------------------------------------------- */

typedef struct pcl_context pcl_context;

/* Kernel choice; every choice gives bitwise-identical results. */
enum pcl_kernel {
    PCL_KERNEL_AUTO = 0,
    PCL_KERNEL_SPLIT_KV = 1,    /* split-KV flash decode + ordered combine */
    PCL_KERNEL_TILED = 2,       /* LDS-tiled prefill, one pass over the keys */
    PCL_KERNEL_TILED_SPLIT = 3, /* LDS-tiled prefill, one key chunk per block */
    PCL_KERNEL_PIPE_KV = 4,     /* pipelined split-KV decode (score/value wave
                                   pairs, head dim <= 256) + ordered combine */
    /* 5 is retired (a two-launch decode that no choice selected) and is
       refused with PCL_INVALID_PARAMETER */
    PCL_KERNEL_SPREAD_KV = 6,   /* split-KV decode with each key chunk spread
                                   over head_dim/32 slices that exchange raw
                                   scores (two-wave slices up to head dim
                                   256, one-wave slices at 512; short
                                   launches); the launch's own merge
                                   workgroups run the ordered combine */
    PCL_KERNEL_FAN_KV = 7,      /* split-KV decode with each (key chunk,
                                   16-row unit, KV head) item fanned over the
                                   eight waves of one workgroup (head dims
                                   above 64, launches of two or more chunks;
                                   otherwise the pipelined kernel runs) +
                                   ordered combine */
};

/* Attention of nq query positions over keys [0, n0+n1): keys 0..n0-1 come
 * from segment 0 (k0/v0) and the rest from segment 1 (k1/v1), both
 * [n][kvheads][dim] device arrays. All pointers are device pointers.
 *
 * Mask, per query i and key t (absolute key position first_key+t, query
 * position first_query+i):
 *   mask != NULL : allowed = mask[i*mask_stride + t] != 0;
 *   causal != 0  : allowed = kp <= qp && (window == 0 || qp - kp < window)
 *                  (encoder_mask, src/engine/attention.rs:1170-1182);
 *   otherwise    : every key (decoder/canvas mode, attention.rs:696-698).
 * The query is scaled by q_scale in f32 before the dot products, as the
 * engine's pre-scale (src/engine/nemotron/forward.rs:336-346); 1 = none.
 * softcap: logit soft-cap, off when 0 (a zero-initialised descriptor). When
 * > 0 every allowed score s becomes softcap * tanh(s / softcap) in f32 before
 * the softmax (the form of p9_ref_softcap, src/kernels/portable/reference.rs:
 * 226-235; the engine itself caps only its final logits, src/engine/text.rs:
 * 963,979, so it leaves this off). An infinite score then becomes
 * +-softcap; a NaN one is still an error. Negative, subnormal or non-finite
 * values, and values above 2^126 (whose f32 reciprocal is subnormal), are
 * PCL_INVALID_PARAMETER.
 * Output: query i, head h (kh_first*group <= h < kh_end*group) at
 * out + i*o_stride + (h - kh_first*group)*dim. */
typedef struct pcl_attention_desc {
    const float *q;
    int64_t q_stride;
    int64_t nq;
    const float *k0, *v0;
    int64_t n0;
    const float *k1, *v1;
    int64_t n1;
    int64_t qheads, kvheads, dim;
    int64_t kh_first, kh_end;
    const uint8_t *mask;
    int64_t mask_stride;
    int32_t causal;
    int64_t window;
    int64_t first_key, first_query;
    float q_scale;
    float *out;
    int64_t o_stride;
    int32_t kernel; /* enum pcl_kernel */
    float softcap;  /* 0 = off */
} pcl_attention_desc;

/* Create a context on a device that owns a new non-blocking stream. */
int pcl_context_create(int device, pcl_context **out);
/* Create a context that launches on the caller's hipStream_t `stream`
 * (NULL = the device's null stream); the caller keeps ownership. */
int pcl_context_create_on_stream(int device, void *stream, pcl_context **out);
void pcl_context_destroy(pcl_context *ctx);
/* The stream launches go to (a hipStream_t). */
void *pcl_context_stream(pcl_context *ctx);
/* Launch asynchronously. Returns PCL_OK, PCL_INVALID_SHAPE for a descriptor
 * that fails validation (including the size limits: at most 2^30 keys, and
 * nq * (qheads / kvheads) * (kh_end - kh_first) at most 2^22; larger calls
 * are split by query range or KV-head range, which leaves every result bit
 * unchanged), PCL_RESOURCE_LIMIT when the workspace cannot be allocated,
 * or PCL_NON_FINITE_VALUE for a launch failure. Data errors (non-finite
 * allowed score or output) are recorded in the context's device error flag.
 * Grows the context's workspace when needed (a device allocation);
 * pcl_context_reserve avoids that inside timed regions and before a graph
 * capture. A workspace that a captured launch holds is kept until the context
 * is destroyed. On a stream that is capturing a graph, AUTO does not take the
 * spread decode (its workgroups accept a published word by the launch's
 * epoch, which every replay would repeat) but the pipelined kernel, with the
 * same bits; an explicit PCL_KERNEL_SPREAD_KV is refused there with
 * PCL_INVALID_PARAMETER. No counterpart in the reference (host calls only). */
int pcl_attention_launch(pcl_context *ctx, const pcl_attention_desc *desc);
/* Workspace bytes a descriptor needs with the kernel it would run (under
 * AUTO, also enough for the kernel a graph capture of it takes). */
size_t pcl_attention_workspace_bytes(const pcl_attention_desc *desc);

/* Bytes of the per-GPU scratch array of pcl_attention_launch_noalloc. */
#define PCL_NOALLOC_SCRATCH_BYTES ((size_t)64 << 20)

/* pcl_attention_launch without any allocation. No counterpart in the
 * reference: it is for callers that cannot allocate device memory (code
 * under HIP graph capture, tight serving loops, harnesses that forbid
 * hipMalloc). The same kernels and results as pcl_attention_launch, bit for
 * bit, but the chunk and span partials live in a file-scope device array of
 * PCL_NOALLOC_SCRATCH_BYTES per GPU (held until the process ends; its
 * address is looked up once per device when the first context on that
 * device is created) instead of the context's workspace. A descriptor whose
 * pcl_attention_workspace_bytes exceeds that size returns
 * PCL_RESOURCE_LIMIT (for example a prefill of more than 4096 keys with
 * more than 64 Mi floats of running totals; the 32K and 128K decodes, the
 * 4K prefills and the 256 x 2304 canvas fit). Calls no hipMalloc, hipFree
 * or other allocating routine and records no timing spans. Every call on
 * one GPU shares that GPU's array, which keeps the last call's contents.
 * The partials need no clearing (each launch writes every partial before
 * its combine reads it); the region of published words at the array's
 * start must hold no word of the current epoch, which the array's zero
 * contents at load give and the library restores (a fill kernel on the
 * call's stream) whenever the device's epoch counter has wrapped since.
 * Calls that overlap on one GPU, on different streams or contexts, race
 * and must be serialised by the caller. PCL_NON_FINITE_VALUE if the scratch
 * address could not be taken for this context's device. */
int pcl_attention_launch_noalloc(pcl_context *ctx, const pcl_attention_desc *desc);
int pcl_context_reserve(pcl_context *ctx, size_t bytes);
/* Wait for the stream; *device_error receives the error flag (bit 0: a
 * non-finite allowed score, bit 1: a non-finite output, bit 2: a non-finite
 * head-transform value, bit 3: a non-finite output-block value, bit 4: a
 * wait between workgroups ran out, pcl_context_set_wait_limit, bit 5: a page
 * step that does not fit or page data out of range, section 7) and is
 * cleared. */
int pcl_context_sync(pcl_context *ctx, int *device_error);
/* Kernel the descriptor resolves to under PCL_KERNEL_AUTO. */
int pcl_attention_resolve_kernel(const pcl_attention_desc *desc);

/* For tests: the (query, head) rows of one KV head that a workgroup of the
 * tiled kernels owns when pcl_attention_launch runs this descriptor on a
 * device of `cus` compute units; 0 when it takes another kernel, -1 when it
 * is rejected. */
int pcl_debug_tiled_rows(const pcl_attention_desc *desc, int cus);

/* Bound of the spread decode's waits for the scores of the other
 * workgroups of a key chunk, in polls of a few hundred cycles each; 0
 * restores the default (65536, some tens of milliseconds). A wave whose wait
 * runs out forms the missing score blocks itself by the same chain (the
 * same bits), so the launch's result stays valid: a GPU shared with other
 * work, on which some of a launch's workgroups may not run alongside the
 * others, costs time, not correctness. Tests use a tiny limit to exercise
 * that path. The launch's merge workgroups wait only for workgroups
 * dispatched before them, under a fixed guard of about a second; bit 4 (16)
 * of the device error flag reports a guard that ran out (then the output is
 * not valid; the host-pointer entries of section 1 rerun such a launch with
 * the pipelined kernel, which never waits). ctx NULL sets the limit of the
 * context the host-pointer entries use. No counterpart in the reference
 * (its CPU threads do not wait on each other inside an attention call).
 * PCL_INVALID_PARAMETER for a negative limit. */
int pcl_context_set_wait_limit(pcl_context *ctx, int polls);
/* Testing hook, no counterpart in the reference: sets the device's epoch
 * counter (the spread decode's launches each take the next value; its low
 * 32 bits are the epoch its published words carry, its high bits count
 * wraps) so that a test can run launches across a wrap. PCL_INVALID_SHAPE
 * for a device index outside the library's table. */
int pcl_debug_set_epoch_counter(int device, uint64_t value);

/* Per-kernel timing, the device-side counterpart of the engine's stage
 * timers (stats::Span, src/engine/stats.rs:9-64). While enabled, every launch
 * records HIP events on the context's stream around the kernels that stream
 * K/V (role 0: split-KV, pipelined, two-pass, spread or tiled kernels; the
 * spread kernel includes its own merge) and around the
 * ordered combine (role 1). pcl_context_timing waits for the stream, adds the
 * elapsed times of the recorded launches to ms[role] and their number to
 * launches[role], and forgets them. Enabling costs two event records per role
 * per launch; leave it off in production. */
int pcl_context_set_timing(pcl_context *ctx, int enable);
int pcl_context_timing(pcl_context *ctx, double *ms, int64_t *launches);

/* ---- 4. device-resident layer cache ----------------------------------------
 *
 * The engine's LayerCache (src/engine/attention.rs:244-311) with its K/V rows
 * in HBM: token-major [tokens][kvheads][dim] f32, the retained rows
 * contiguous, so attention reads them in place (no staging copy, unlike
 * stage(), attention.rs:562-581). All copies run on the context's stream. */
typedef struct pcl_kv_cache pcl_kv_cache;

/* Undo record of one uncommitted step (PendingKv, attention.rs:263-266);
 * lengths in tokens. */
typedef struct pcl_kv_pending {
    int64_t old_len;
    int64_t old_total;
} pcl_kv_pending;

/* new_cache (attention.rs:484-505): rows of kvheads x dim floats, positions
 * up to `context`, window 0 for a global layer (a sliding layer keeps
 * window - 1 tokens, retained_count, attention.rs:1166-1168), max_bytes
 * bounding the retained plus appended K+V bytes of a step. PCL_RESOURCE_LIMIT
 * when max_bytes is below one token's K+V. */
int pcl_kv_cache_create(pcl_context *ctx, int64_t kvheads, int64_t dim, int64_t context,
                        int64_t window, size_t max_bytes, pcl_kv_cache **out);
/* Destroy caches (and head transforms) before the context they were made on. */
void pcl_kv_cache_destroy(pcl_kv_cache *cache);
/* Room for `rows` rows in the cache's buffers now (at most what max_bytes
 * allows), so that appends up to that many retained plus appended rows do not
 * reallocate (growth frees the old buffers, and on MI355X a process that
 * frees device memory streams more slowly afterwards). Grow-only; call it
 * between steps (moving the rows invalidates a pending record).
 * PCL_RESOURCE_LIMIT if the buffers cannot be allocated. No counterpart in
 * the reference (its caches are host vectors). */
int pcl_kv_cache_reserve_rows(pcl_kv_cache *cache, int64_t rows);
/* LayerCache::total_tokens / retained_tokens (attention.rs:268-273). */
int64_t pcl_kv_cache_total_tokens(const pcl_kv_cache *cache);
int64_t pcl_kv_cache_retained_tokens(const pcl_kv_cache *cache);
/* The retained rows (LayerCache::keys / values, attention.rs:274-279) as device
 * pointers, their count and the absolute position of the first. Valid until
 * the next append, keep, rollback or commit. */
int pcl_kv_cache_view(const pcl_kv_cache *cache, const float **keys, const float **values,
                      int64_t *rows, int64_t *first_position);
/* Copy retained rows [first, first + rows) of K and V into keys / values
 * (host or device memory, [rows][kvheads][dim] each) and wait for the copy:
 * the host-side read of LayerCache::keys / values. */
int pcl_kv_cache_read(const pcl_kv_cache *cache, int64_t first, int64_t rows, float *keys,
                      float *values);
/* One uncommitted step of n tokens (encode_in_place's append,
 * attention.rs:949-1080): checks total + n <= context and the byte limit
 * (check_stage, attention.rs:545-558), copies the rows keys/values
 * ([n][kvheads][dim]; device memory of the cache's device in one launch, host
 * memory by runtime copies) after the retained rows, advances the total and
 * fills *pending. On an error the cache is unchanged. */
int pcl_kv_cache_append(pcl_kv_cache *cache, const float *keys, const float *values, int64_t n,
                        pcl_kv_pending *pending);
/* LayerCache::rollback / keep / commit (attention.rs:280-310): undo the step;
 * keep only its first `tokens` positions; apply window retention (the dead
 * prefix is dropped once it is at least half the rows). */
int pcl_kv_cache_rollback(pcl_kv_cache *cache, const pcl_kv_pending *pending);
int pcl_kv_cache_keep(pcl_kv_cache *cache, const pcl_kv_pending *pending, int64_t tokens);
int pcl_kv_cache_commit(pcl_kv_cache *cache);
/* Key/value fields of an attention descriptor over the cache; the caller sets
 * the query, output and head fields. Encoder pass (after append, before
 * commit): the retained rows including the step, causal with the cache's
 * window, first_key = position of the first retained row, first_query =
 * pending->old_total (encode_in_place's view, attention.rs:978-987). Decoder
 * pass (DiffusionGemma canvas, decode_routed, attention.rs:1156-1163): the
 * retained rows then n canvas rows as a second segment, no mask, first_query =
 * the cache total; the cache is not changed. */
int pcl_kv_cache_encoder_desc(const pcl_kv_cache *cache, const pcl_kv_pending *pending,
                              pcl_attention_desc *desc);
int pcl_kv_cache_decoder_desc(const pcl_kv_cache *cache, const float *canvas_keys,
                              const float *canvas_values, int64_t n, pcl_attention_desc *desc);
/* Shared-K/V layer step (encode_shared_in_place, attention.rs:1086-1145): the
 * layer stores no K/V and attends over its source layer's rows of the same
 * uncommitted step. shared_desc checks cache total == source_pending->old_total
 * and source total == cache total + n, and fills the key/value fields: the
 * source's retained rows, causal with this cache's window, first_key =
 * source_pending->old_total - the rows the source retained before its step,
 * first_query = the cache total. advance records *pending and moves the
 * total to total + n (keep / rollback / commit apply as for any step). */
int pcl_kv_cache_shared_desc(const pcl_kv_cache *cache, const pcl_kv_cache *source,
                             const pcl_kv_pending *source_pending, int64_t n,
                             pcl_attention_desc *desc);
int pcl_kv_cache_advance(pcl_kv_cache *cache, int64_t n, pcl_kv_pending *pending);

/* ---- 5. head transform (the attention prologue) ----------------------------
 *
 * HeadTransform (src/engine/attention.rs:51-243) on the device: per head an
 * RMS norm with a sequential f64 sum of squares (p9_ref_rms_norm,
 * src/kernels/portable/reference.rs:11-33), the learned scale for Q and K,
 * then NeoX rotation of pairs (j, j + dim/2) by f32 angles
 * position * (1 / powf(base, 2j/dim)) / factor_j (p9_ref_rope,
 * reference.rs:277-318); V is normalised without scale and not rotated.
 * Row layouts: raw and prepared Q [n][qheads][dim], K and V [n][kvheads][dim],
 * device pointers; token i is at position `position + i`. Launches are
 * asynchronous on the context's stream; a non-finite input or output sets
 * bit 2 of the context's device error flag (pcl_context_sync). */
typedef struct pcl_head_transform pcl_head_transform;

/* HeadTransform::new (attention.rs:65-101): scales [dim] and factors NULL or
 * [dim/2] are host arrays, copied. sliding != 0: the layer needs a V
 * projection; otherwise raw_v NULL means V = the raw K (global K-as-V,
 * attention.rs:121-129). PCL_INVALID_SHAPE for a head geometry this backend
 * does not run (dim 16, 32, 64, 128, 256 or 512); PCL_INVALID_PARAMETER for a
 * non-finite or non-positive epsilon, base or factor, or a non-finite scale. */
int pcl_head_transform_create(pcl_context *ctx, int64_t qheads, int64_t kvheads, int64_t dim,
                              int sliding, const float *query_scale, const float *key_scale,
                              float epsilon, float base, const float *factors,
                              pcl_head_transform **out);
void pcl_head_transform_destroy(pcl_head_transform *transform);
/* HeadTransform::prepare (attention.rs:102-156) for n tokens. The rotation
 * table is built on the host (the C library's powf; the C library's double
 * sin and cos of each f32 angle, rounded once to f32: within an f32 ulp of
 * the reference's libm::sincosf, src/libm.rs:350, and equal to it for all
 * but about 0.1 % of angles) for positions up to the largest seen so far and
 * kept on the device until the transform is destroyed, outgrown tables too (a
 * captured launch may hold one); PCL_NON_FINITE_VALUE for a non-finite angle,
 * PCL_RESOURCE_LIMIT beyond 2^24 positions, and inside a graph capture for a
 * position past the table, which is not built there. A rotated Q or K value y_j
 * (pair j, j + dim/2) is therefore within 2^-20 * (|y_j| + |y_{j+dim/2}|)
 * of the reference's, and almost always equal to it; V rows are bit for
 * bit. */
int pcl_head_transform_prepare(pcl_head_transform *transform, const float *raw_q,
                               const float *raw_k, const float *raw_v, int64_t n,
                               int64_t position, float *q_out, float *k_out, float *v_out);
/* prepare_query (attention.rs:223-242): the query half, for shared-K/V
 * layers. */
int pcl_head_transform_query(pcl_head_transform *transform, const float *raw_q, int64_t n,
                             int64_t position, float *q_out);
/* encode_in_place's projection tail (project_tokens, attention.rs:584-666)
 * fused with the cache append: prepared K and V go straight into the cache's
 * rows after the retained ones, at positions total .. total+n-1, and the
 * prepared queries into q_out. Limits and *pending as pcl_kv_cache_append. */
int pcl_kv_cache_append_transformed(pcl_kv_cache *cache, pcl_head_transform *transform,
                                    const float *raw_q, const float *raw_k, const float *raw_v,
                                    int64_t n, float *q_out, pcl_kv_pending *pending);

/* One decode token of a layer in one call: pcl_kv_cache_append_transformed
 * for n = 1 (the token's raw rows prepared, K and V written after the
 * retained rows, the prepared queries to q_out [qheads][dim]), then the
 * attention of the prepared queries over the cache's rows with the step's
 * new key (pcl_kv_cache_encoder_desc of the step, every KV head, q_scale as
 * the descriptor's, kernel an enum pcl_kernel) into out [qheads][dim]: the
 * one-position decode of encode_in_place (src/engine/attention.rs:949-1080,
 * prepare 102-156 then the attention pass 755-777). Where the kernel that
 * runs is the pipelined decode at head dim 64, 128, 256 or 512, the
 * transform is folded into its launch: every workgroup prepares its own
 * query rows and the workgroups of the new key's chunk write that key's K
 * and V rows before reading them (one launch fewer, the same bits);
 * otherwise the transform's own launch runs first. Limits, errors and
 * *pending as pcl_kv_cache_append_transformed and pcl_attention_launch; on
 * an error nothing was launched and the cache is unchanged. */
int pcl_kv_cache_attend_token(pcl_kv_cache *cache, pcl_head_transform *transform,
                              const float *raw_q, const float *raw_k, const float *raw_v,
                              float q_scale, int kernel, float *q_out, float *out,
                              pcl_kv_pending *pending);

/* ---- 6. attention output block ---------------------------------------------
 *
 * The step after attention (src/engine/attention.rs:866-884): projected =
 * W . attended with f32 weights [out][in] (Matrix::project / p9_ref_matvec,
 * src/kernels/portable/reference.rs:36-78: f64 sums of exact f32 products),
 * then result = residual + rms_norm(projected, post_scale, epsilon) in the
 * engine's rounding (f64 norm, f32 scale and add). attended [n][in],
 * residual, projected and result [n][out], post_scale [out]: device pointers;
 * result may be the residual buffer. Asynchronous on the context's stream; a
 * non-finite projected or result value sets bit 3 of the device error flag.
 * The sums are f64 in the kernels' own order, so a value equals the engine's
 * unless the two f64 sums fall on opposite sides of an f32 rounding
 * boundary. A token's row has the same bits in every call of up to 32
 * tokens, and the same bits in every larger call; between the two the order
 * of the f64 sums differs. PCL_INVALID_SHAPE beyond n = 2^22 tokens or in, out = 2^20. */
int pcl_attention_output(pcl_context *ctx, const float *attended, int64_t n, int64_t in,
                         const float *weights, int64_t out, const float *post_scale,
                         float epsilon, const float *residual, float *projected, float *result);

/* For tests: which form of the projection n tokens of `in` columns take on a
 * device of `cus` compute units: 1 a wave per output row, 16 or 32 the
 * few-token kernel with so many tokens a workgroup, else the output block of
 * a wave (16016) or tile of a workgroup as tokens * 1000 + rows. */
int pcl_debug_projection_form(int64_t n, int64_t in, int64_t out, int cus);

/* ---- 7. batches of requests over a paged cache ------------------------------
 *
 * Several requests share pools of pages: a page holds page_tokens consecutive
 * tokens of one request for one layer's K and V, a request's block table names
 * its pages in order, and slot = page * page_tokens + offset names a token's
 * row. One pcl_page_batch serves every layer of a model (all pools have the
 * same pages). A step of the batch is
 *
 *   pcl_page_step            pages for every request's new tokens; the slot,
 *                            position and request of every row of the step
 *   per layer:
 *     pcl_paged_append[_transformed]   the step's K and V rows into the pages
 *     pcl_paged_attention              the newest token of every request
 *   pcl_page_commit          the step's tokens count as held
 *
 * Rows are in request order: the new tokens of request 0, then of request 1,
 * and so on; the other entries of a layer (head transform, output block) take
 * the same rows. All state is the caller's device memory and everything is
 * asynchronous on the context's stream with no host read, so a whole step can
 * be captured into a graph and replayed with other lengths (see each entry for
 * what must exist before the capture). Replays of graphs captured from one
 * context share its workspace, and must not overlap with each other or with the
 * context's launches. Nothing here has a counterpart in the reference, whose
 * caches hold one sequence each.
 *
 * What the host cannot see is checked on the device: bit 5 (32) of the error
 * flag (pcl_context_sync) reports it. */

/* Values of the pages. Rows are rounded to bf16 when they are written (nearest,
 * ties to even) and widened (exactly) when they are read; all arithmetic is
 * that of f32 pages. */
enum pcl_cache_type {
    PCL_CACHE_F32 = 0,
    PCL_CACHE_BF16 = 1,
};

/* The pages of one layer: k and v [pages][page_tokens][kvheads][dim], device
 * memory, 16-byte aligned. pages * page_tokens below 2^31, page_tokens at most
 * 4096 (any size, not only powers of two), kvheads at most 4096, dim a multiple
 * of 16 up to 512. */
typedef struct pcl_page_pools {
    void *k, *v;
    int32_t type; /* enum pcl_cache_type */
    int64_t pages, page_tokens, kvheads, dim;
} pcl_page_pools;

/* Page bookkeeping of a batch of `requests` (at most 2048), all arrays device
 * memory of the caller. State (pcl_page_reset writes an empty batch; a caller
 * may fill it in itself): */
typedef struct pcl_page_batch {
    int64_t requests;
    int64_t table_stride; /* pages a block table holds */
    int64_t page_tokens;
    int64_t pages;
    int64_t step_rows;    /* rows a step may have, below 2^20 */
    int32_t *lengths;     /* [requests] tokens held (committed) */
    int32_t *table;       /* [requests][table_stride] pages of each request */
    int32_t *free_pages;  /* [pages] a stack: the last free entry is taken first */
    int32_t *counters;    /* [4] free pages; of the step: its rows, the pages it
                             takes, 1 while it stands uncommitted (2: a fork,
                             section 8) */
    /* what a step writes: */
    int32_t *step_lengths; /* [requests] tokens held with the step's */
    int32_t *newest;       /* [requests] row of the newest token, -1 for none */
    int32_t *slots;        /* [step_rows] slot of each row, -1 behind the last */
    int32_t *positions;    /* [step_rows] position of each row, -1 behind it */
    int32_t *row_request;  /* [step_rows] request of each row, -1 behind it */
} pcl_page_batch;

/* An empty batch: no tokens, every page free, no step. */
int pcl_page_reset(pcl_context *ctx, const pcl_page_batch *batch);
/* Opens a step with new_tokens[b] (device, [requests], 0 allowed) more tokens
 * of every request: pages for them from the free list in request order, their
 * entries behind the held ones of the block tables, and the step's arrays. The
 * held state (lengths, held entries, free list) is not changed, so a step that
 * is not committed is simply replaced by the next one. A step that does not
 * fit (negative or too many tokens for the table or step_rows, too few free
 * pages, a length outside the table) is refused as a whole: bit 5 of the error
 * flag, no rows, slots all -1, counters[3] = 0. A page number outside the pools
 * in the table or the free list leaves that row's slot -1 (and -1 as the new
 * page's entry), with the error, and the step does not stand (counters[3] = 0,
 * so a commit finds none). */
int pcl_page_step(pcl_context *ctx, const pcl_page_batch *batch, const int32_t *new_tokens);
/* The standing step's tokens count as held: all of them, or the first kept[b]
 * of each request (device, [requests]; speculative tokens that were refused);
 * pages that hold only tokens not kept go back to the free list. Without a
 * standing step nothing happens; a count outside 0..new tokens, like step data
 * out of range or a page outside the pools among those given back, is bit 5 of
 * the error flag and changes nothing. */
int pcl_page_commit(pcl_context *ctx, const pcl_page_batch *batch, const int32_t *kept);
/* Requests with finished[b] != 0 (device, [requests]) give all their pages back
 * and hold no tokens; a standing step is dropped. With a length out of range, or
 * a page among those given back that lies outside the pools, that another
 * request's table holds too or that occurs twice, nothing changes (bit 5): where
 * block tables share pages, pcl_page_release_shared gives them back. */
int pcl_page_release(pcl_context *ctx, const pcl_page_batch *batch, const int32_t *finished);

/* K and V rows [n][kvheads][dim] (f32, device, 16-byte aligned) into the slots
 * of the pools; a row with a negative slot is left out, one past the pools too,
 * with bit 5 of the error flag. Slots must differ from each other. */
int pcl_paged_append(pcl_context *ctx, const pcl_page_pools *pools, const int32_t *slots,
                     const float *keys, const float *values, int64_t n);
/* The same from raw projections: pcl_head_transform_prepare for n rows, each
 * at its own position, with K and V written into their slots and the prepared
 * queries into q_out [n][qheads][dim] (a row that is left out keeps its q_out).
 * Positions lie in [0, position_limit), or the row is left out with bit 5 of
 * the error flag; the rotation table for them is built on the host at the first
 * call (before a capture: inside one a table that is too short is
 * PCL_RESOURCE_LIMIT). raw_v NULL as in pcl_head_transform_prepare. On the
 * transform's context. */
int pcl_paged_append_transformed(pcl_head_transform *transform, const pcl_page_pools *pools,
                                 const int32_t *slots, const int32_t *positions,
                                 int64_t position_limit, const float *raw_q, const float *raw_k,
                                 const float *raw_v, int64_t n, float *q_out);

/* Attention of the newest token of every request over its pages. Request b
 * with row r = rows[b] (rows NULL: r = b) attends keys [0, lengths[b]) or, with
 * a window, the last `window` of them; its query heads are at q + r * q_stride
 * and its output goes to out + r * o_stride, [qheads][dim] each. A request with
 * a negative row or no keys is left out: its output row stays as it was. With a
 * step's arrays (lengths = step_lengths, rows = newest) the requests without a
 * new token are left out. The query is scaled by q_scale, and scores are capped
 * by softcap, as in pcl_attention_desc. A request's output has the bits that
 * pcl_attention_launch gives for its keys and values in one segment (causal, the
 * same window, first_key 0, first_query lengths[b] - 1; bf16 pages: for the
 * widened rows), whatever else is in the batch; only a zero's sign may differ.
 * max_length bounds the lengths (it sizes the workspace); a longer request or a
 * row at or past q_rows is left out with bit 5 of the error flag, and a page
 * outside the pools is read as page 0, with bit 5. Rows must differ from each
 * other. Several requests may share pages; one that still appends must hold the
 * page that it appends to alone, and pcl_page_release refuses shared pages
 * (pcl_page_release_shared gives them back). */
typedef struct pcl_paged_desc {
    pcl_page_pools pools;
    const float *q;
    int64_t q_stride, q_rows; /* q_rows: rows that q and out hold */
    int64_t qheads;           /* at most 4096 */
    const int32_t *table;     /* [requests][table_stride] */
    int64_t table_stride;
    const int32_t *lengths; /* [requests] */
    const int32_t *rows;    /* [requests] or NULL */
    int64_t requests;       /* at most 2048 */
    int64_t max_length;     /* at most table_stride * page_tokens */
    int64_t window;         /* 0 = all keys */
    float q_scale;
    float softcap; /* 0 = off */
    float *out;
    int64_t o_stride;
} pcl_paged_desc;

/* Launch asynchronously; PCL_OK, PCL_INVALID_SHAPE, PCL_INVALID_PARAMETER,
 * PCL_RESOURCE_LIMIT when the workspace cannot be had (inside a capture it is
 * not grown: pcl_context_reserve the bytes before) or PCL_NON_FINITE_VALUE for
 * a launch failure. Non-finite scores and outputs are bits 0 and 1 of the error
 * flag. */
int pcl_paged_attention(pcl_context *ctx, const pcl_paged_desc *desc);
/* Workspace bytes a descriptor needs (0 when it is refused). */
size_t pcl_paged_workspace_bytes(const pcl_paged_desc *desc);

/* ---- 8. drafted tokens and shared pages ---------------------------------------
 *
 * A round of drafted tokens is a step of section 7 in which a request's new tokens
 * form a tree: each follows another of them, or the held tokens, and attends the
 * held tokens and its own branch.
 *
 *   pcl_page_step                          the drafted tokens' rows
 *   pcl_page_tree_masks                    their positions and branches
 *   per layer:
 *     pcl_paged_append[_transformed]       at the tree's positions
 *     pcl_paged_tree_attention             every new token
 *   pcl_page_accept                        the branch that was verified: which rows
 *                                          move to follow the held tokens
 *   pcl_page_commit                        with the branches' lengths as kept
 *   pcl_paged_copy                         the rows, in every layer at once
 *
 * Without a tree the new tokens are a chain, each behind the one before it: drafted
 * tokens of one continuation, or a prompt's part behind what the pages hold, with
 * no masks and nothing to move.
 *
 * Requests that begin as copies of others (several answers to a prompt, beams)
 * share their whole pages:
 *
 *   pcl_page_fork                          their tables; a page of its own for a
 *                                          fork's last, partly filled one
 *   pcl_page_commit                        the forks hold their sources' tokens
 *   pcl_paged_copy                         those last pages' rows, in every layer
 *   pcl_page_release_shared                of requests that ended, the pages that
 *                                          nobody else holds
 *
 * State, streams, captures, workspaces and the error flag are those of section 7. */

/* The trees of a standing step, device memory: rows as the step lays them out. */
typedef struct pcl_page_tree {
    const int32_t *parents; /* [step_rows] index among its request's new tokens of
                               the token that each follows, below its own; -1: the
                               held tokens */
    int64_t words;          /* 64-bit words of a mask, 1 to 8: trees of up to 64 *
                               words tokens */
    /* what the call writes: */
    int32_t *positions; /* [step_rows] tokens held + tokens before it on its branch,
                           -1 behind the last row */
    uint64_t *masks;    /* [step_rows][words] bit j: new token j of its request is
                           on its branch (itself too); 0 behind the last row */
} pcl_page_tree;

/* Positions and branches of the standing step's new tokens (without one: of none).
 * A parent that is not below its token counts as -1, and of a request with more
 * than 64 * words new tokens each sees the held tokens alone, in the chain's
 * positions, both with bit 5 of the error flag. */
int pcl_page_tree_masks(pcl_context *ctx, const pcl_page_batch *batch, const pcl_page_tree *tree);

/* Rows that verified branches move: paths (device, [requests][depth]) holds of each
 * request the counts[b] (device, [requests]; at most depth) new tokens that are
 * kept, their indexes ascending. from and to ([requests][depth]) receive the slots
 * of the k-th one's row and of the row that it moves to, the k-th behind the held
 * tokens, -1 where nothing moves. Call it before the commit (with kept = counts),
 * and pcl_paged_copy with lists = requests, entries = depth and no row counts before
 * the next step. Indexes that do not ascend within the new tokens, or counts out of
 * range, are bit 5 of the error flag: that request's lists are -1, the others' may
 * be, and the step does not stand any more, so that a commit finds none. Without a
 * standing step all lists are -1. depth * requests below 2^31. */
int pcl_page_accept(pcl_context *ctx, const pcl_page_batch *batch, const int32_t *paths,
                    const int32_t *counts, int64_t depth, int32_t *from, int32_t *to);

/* Opens a fork: a step without rows in which every request b with sources[b] >= 0
 * (device, [requests]) begins as a copy of request sources[b]. It must hold no
 * tokens, and its source must not be a fork of the same call. Its table gets the
 * source's whole pages, and a page from the free list (in request order) where the
 * source's last one is partly filled; from, to and rows (device, [requests]) receive
 * that page's first slot, the new one's, and the rows to copy (pcl_paged_copy with
 * lists = requests, entries = 1; -1, -1 and 0 where there are none). As a step's, its
 * held state changes with pcl_page_commit, whose `kept` must be NULL for a fork (or
 * it is refused with bit 5), and one that is not committed is replaced by the next
 * fork or step. A fork that does not fit (a request that holds tokens, a source that
 * is none, too few free pages, a length outside the table) is refused as a whole,
 * with bit 5; one whose last pages lie outside the pools does not stand, with bit 5.
 * Forks may be forked once they are committed. */
int pcl_page_fork(pcl_context *ctx, const pcl_page_batch *batch, const int32_t *sources,
                  int32_t *from, int32_t *to, int32_t *rows);

/* pcl_page_release where block tables share pages: requests with finished[b] != 0
 * hold no tokens any more, and those of their pages that no other request holds go
 * back, each once, the highest number first (so that the lowest is taken next). A
 * standing step or fork is dropped. With a length out of range, a page among the
 * finished requests' that lies outside the pools, or one of them on the free list
 * already, nothing changes (bit 5). Uses the context's workspace (inside a capture
 * it is not grown: pcl_context_reserve the bytes before). */
int pcl_page_release_shared(pcl_context *ctx, const pcl_page_batch *batch,
                            const int32_t *finished);
/* Workspace bytes of that call (0 where it needs none, and for a batch that is
 * refused). */
size_t pcl_page_release_workspace_bytes(const pcl_page_batch *batch);

/* Copies rows of pages, K and V, from slot to slot in the pools of `layers` layers
 * (a host array; the same pages and page_tokens in all, heads and types may differ).
 * from and to (device, [lists][entries]) name slots; an entry with a negative one is
 * left out, one past the pools too, with bit 5 of the error flag. rows NULL: one row
 * an entry, the entries of a list in order; none reads a row that an earlier one of
 * its list writes (it may write one that an earlier one reads). rows (device,
 * [lists], only with entries = 1): an entry copies that many consecutive slots (none
 * for 0 or less), and the two ranges do not overlap. Lists do not touch the rows
 * that another one writes. */
int pcl_paged_copy(pcl_context *ctx, const pcl_page_pools *pools, int64_t layers,
                   const int32_t *from, const int32_t *to, const int32_t *rows, int64_t lists,
                   int64_t entries);

/* Attention of every new token of a step over its request's pages. Request b, with
 * n = step_lengths[b] - lengths[b] new tokens, has them in rows newest[b] - n + 1 to
 * newest[b] (a step's arrays as they are); their query heads are at q + row *
 * q_stride, their outputs go to out + row * o_stride. New token i is at position
 * lengths[b] + i and attends keys [0, lengths[b] + i]; with masks it is at
 * positions[row] and attends the held keys [0, lengths[b]) and each new token j with
 * bit j of masks[row] (any bits; pcl_page_tree_masks makes a tree's). With a window a
 * token attends only keys whose position is less than `window` before its own (the
 * new tokens' by positions, which lie from lengths[b] to step_lengths[b] - 1).
 * Requests without new tokens or with a negative newest are left out, and a token
 * that attends no key too: their output rows stay as they were. Queries are scaled and
 * scores capped as in pcl_attention_desc. A token's output has the bits that
 * pcl_attention_launch gives for the request's keys and values in one segment (the
 * chain: causal, first_key 0, first_query lengths[b]; masks: with the same mask as
 * bytes), whatever else is in the batch; only a zero's sign may differ. Keys that no
 * token attends may hold anything. A key that one token attends and another one does not
 * may make the latter a NaN where its value is not finite; the former sets the error
 * flag then. A token whose attended scores are all -infinity, which is bit 0 of the
 * flag, keeps its output row too.
 * max_length bounds step_lengths, max_new the new tokens of a request (they size the
 * workspace with q_rows). A request past them or whose rows do not lie in q_rows,
 * or with more new tokens than its masks have bits, is left out with bit 5 of the
 * error flag; a page outside the pools is read as page 0, with bit 5. Rows of
 * different requests must differ. */
typedef struct pcl_paged_tree_desc {
    pcl_page_pools pools;
    const float *q;
    int64_t q_stride, q_rows; /* q_rows: rows that q, out, masks and positions hold */
    int64_t qheads;           /* at most 4096 */
    const int32_t *table;     /* [requests][table_stride] */
    int64_t table_stride;
    const int32_t *lengths;      /* [requests] tokens held */
    const int32_t *step_lengths; /* [requests] with the new ones */
    const int32_t *newest;       /* [requests] row of the newest token, -1 for none */
    const uint64_t *masks;       /* [q_rows][mask_words] or NULL */
    int64_t mask_words;          /* 1 to 8; 0 without masks */
    const int32_t *positions;    /* [q_rows] with masks (may be NULL without a window) */
    int64_t requests;            /* at most 2048 */
    int64_t max_length;          /* at most table_stride * page_tokens */
    int64_t max_new;             /* below 2^20 */
    int64_t window;              /* 0 = all keys */
    float q_scale;
    float softcap; /* 0 = off */
    float *out;
    int64_t o_stride;
} pcl_paged_tree_desc;

/* Launch asynchronously; results and errors as pcl_paged_attention. */
int pcl_paged_tree_attention(pcl_context *ctx, const pcl_paged_tree_desc *desc);
/* Workspace bytes a descriptor needs (0 when it is refused). */
size_t pcl_paged_tree_workspace_bytes(const pcl_paged_tree_desc *desc);

/* Library identification (for loaders). */
const char *pcl_version(void);

#ifdef __cplusplus
}
#endif

#endif

/* irontimber-mi355x: C ABI of the attention / Gated-DeltaNet hot path, hand-written HIP for gfx950.
 *
 * Conventions (all entry points):
 *   - Every pointer argument is a device pointer unless its comment says otherwise. The caller owns
 *     every buffer (inputs, outputs, KV cache, recurrent state, scratch); the library allocates and
 *     frees nothing. (The reference's Vulkan backend follows the same rule with one caller-owned
 *     arena: src/vk/mod.rs:2-6, 544-566.)
 *   - `stream` is a hipStream_t (NULL = the legacy default stream). Calls only enqueue work; they
 *     do not synchronise.
 *   - Return 0 on success. A nonzero return means nothing was enqueued (geometry, alignment or
 *     scratch validation failed on the host) or a launch failed; it_last_error() then returns a
 *     thread-local message. This mirrors the reference's Result<(), String> validation before any
 *     device work (src/vk/mod.rs:179-220).
 *   - Strides are counted in elements of the pointed-to type.
 *   - Calls on one stream from one thread, like the reference's !Sync Ctx (src/vk/mod.rs:235-240).
 */
#ifndef IT_ATTN_H
#define IT_ATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Thread-local text of the last error (empty string if none). */
const char* it_last_error(void);

/* ABI version: bumped whenever a signature or a buffer layout below changes. */
int it_abi_version(void);

/* ------------------------------------------------------------------------------------------------
 * Softmax attention over an f16 KV cache (decode, MTP verify, chunked and whole-prompt prefill).
 * ---------------------------------------------------------------------------------------------- */

/* Append nt new K and V rows (f32, already RMS-normed and roped) to the f16 cache at rows
 * pos0..pos0+nt-1. Source row t is k[t*src_tok_stride + i], i < kvd. Cache row p is kc[p*kvd + i].
 * round_mode 0 = round to nearest even (the half crate's f16::from_f32 used by cpu.rs:22),
 * 1 = round toward zero (packHalf2x16 on the reference's HAWAII GPU, src/vk/r012_parity.rs:14-18).
 * Replaces the pair of kv_pack dispatches, src/vk/mod.rs:832-838 (kernel kernels/src/lib.rs:743-750). */
int it_kv_append_f16(const float* k, const float* v, int src_tok_stride, uint16_t* kc, uint16_t* vc,
                     int pos0, int nt, int kvd, int round_mode, void* stream);

/* The whole pre-attention pass in one launch: per-head RMSNorm of q and k, neox-style (I)MRoPE on
 * the first n_rot dims of each q and k head at positions pos0+t, and the f16 append of K and V.
 *   q      : f32 [t*q_tok_stride + h*2*hd + d]; d < hd (the query) is rewritten in place with
 *            rope(rmsnorm(q) * q_norm); d in [hd, 2hd) (the gate) is left as it is.
 *   k, v   : f32 [t*kv_tok_stride + kh*hd + d], the k and v projections (read only).
 *   kc, vc : f16 cache rows pos0+t receive f16(rope(rmsnorm(k) * k_norm)) and f16(v).
 *   q_norm, k_norm: f32 [hd] weights, or NULL for unit weight. eps: the RMSNorm epsilon.
 *   n_rot  : rotated dims per head (even, <= hd, a multiple of hd/32); theta_scale the f32
 *            base^(-2/n_rot) the reference pushes (src/vk/mod.rs:824); sec0..sec3 the rope
 *            sections (a frequency outside the text sections keeps angle 0, cpu.rs:152-155).
 *   round_mode as for it_kv_append_f16. hd is 128 or 256.
 * The angles p*theta_scale^i are formed in f64, so they are exact to f32 rounding at any position.
 * Replaces the six dispatches of src/vk/mod.rs:822-838 (two rmsnorm mode 0, two rope, two kv_pack;
 * kernels/src/lib.rs:207-229, 233-250, 743-750) and cpu.rs:249-258. */
int it_attn_prep_f16(float* q, int q_tok_stride, const float* k, const float* v, int kv_tok_stride,
                     const float* q_norm, const float* k_norm, float eps, uint16_t* kc, uint16_t* vc, int kvd,
                     int pos0, int hd, int nh, int nkv, int nt, int n_rot, float theta_scale, int sec0, int sec1,
                     int sec2, int sec3, int round_mode, void* stream);

/* it_attn_prep_f16 that also writes the query in the form the flash prefill kernel computes with:
 * q16[t*q16_tok_stride + h*hd + d] = f16_rne(q'[d] * (scale * log2(e))), q' the rewritten query
 * and scale the attention scale the following it_attn_f16_q16 call will pass (the product taken
 * in f32, as that kernel takes it). q16: 16-byte aligned f16 (uint16_t bits), q16_tok_stride a
 * multiple of 8, >= nh*hd. No counterpart in the reference (its prefill kernels read f32 q): an
 * opt-in for prefill callers, whose flash kernel then reads half the q bytes and no f32 rows. */
int it_attn_prep_f16_q16(float* q, int q_tok_stride, const float* k, const float* v, int kv_tok_stride,
                         const float* q_norm, const float* k_norm, float eps, uint16_t* kc, uint16_t* vc, int kvd,
                         int pos0, int hd, int nh, int nkv, int nt, int n_rot, float theta_scale, int sec0, int sec1,
                         int sec2, int sec3, int round_mode, uint16_t* q16, int q16_tok_stride, float scale,
                         void* stream);

/* The same pass with the rotation given by the caller, for tokens whose positions are not their cache rows (a
 * drafted tree, a cache that no longer starts at position 0) and for other rotations than the model's own:
 *   pos    : device int32 [nt], the position of token t (any int32 value), or NULL for pos0 + t.
 *   row0   : K and V of token t go to cache row row0 + t.
 *   n_rot  : rotated dims per head, even, <= hd. layout IT_ROPE_HALVES: dims (i, i + n_rot/2) turn together, n_rot a
 *            multiple of hd/32; IT_ROPE_PAIRS: dims (2i, 2i + 1).
 *   freq   : device f32 [n_rot/2], the angle of pair i per position (it_rope_freqs makes the usual ones; 0 leaves a
 *            pair as it is). The angle pos * freq[i] is formed and reduced in f64: exact up to |pos| = 2^29, rounded to
 *            53 bits beyond (2^-22 of a radian at 2^31 for frequencies up to 1).
 *   mscale : factor of cos and sin (1 but for stretched contexts).
 * The rest as for it_attn_prep_f16 / it_attn_prep_f32kv (q rewritten in place, the gates left as they are). No
 * counterpart in the reference, whose positions are pos0 + t and whose rotation is the model's. */
#define IT_ROPE_HALVES 0
#define IT_ROPE_PAIRS 1
int it_attn_prep_pos_f16(float* q, int q_tok_stride, const float* k, const float* v, int kv_tok_stride,
                         const float* q_norm, const float* k_norm, float eps, uint16_t* kc, uint16_t* vc, int kvd,
                         const int32_t* pos, int pos0, int row0, int hd, int nh, int nkv, int nt, int n_rot,
                         const float* freq, float mscale, int layout, int round_mode, void* stream);
int it_attn_prep_pos_f32kv(float* q, int q_tok_stride, const float* k, const float* v, int kv_tok_stride,
                           const float* q_norm, const float* k_norm, float eps, float* kc, float* vc, int kvd,
                           const int32_t* pos, int pos0, int row0, int hd, int nh, int nkv, int nt, int n_rot,
                           const float* freq, float mscale, int layout, void* stream);

/* The rotation table of the calls above (host function, host buffers): freq[i], i < n_rot/2, and *mscale.
 *   IT_ROPE_PLAIN  : base^(-2i/n_rot), factor and orig_ctx unused.
 *   IT_ROPE_LINEAR : the same / factor (positions interpolated).
 *   IT_ROPE_NTK    : the base times factor^(n_rot/(n_rot-2)), so the slowest pair is stretched by factor and the
 *                    fastest kept.
 *   IT_ROPE_YARN   : pairs of more than 32 turns over orig_ctx positions kept, those of less than one stretched by
 *                    factor, a linear blend between (its ends rounded outwards to whole pairs, the first pair at
 *                    least); *mscale = 0.1 ln(factor) + 1.
 * *mscale is 1 for the others. */
#define IT_ROPE_PLAIN 0
#define IT_ROPE_LINEAR 1
#define IT_ROPE_NTK 2
#define IT_ROPE_YARN 3
int it_rope_freqs(int n_rot, float base, int kind, float factor, int orig_ctx, float* freq, float* mscale);

/* Bytes of scratch to give it_attn_f16 for this call geometry: more changes nothing (0: none is used).
 * Less is accepted too, see it_attn_f16. A prompt call (nt >= 16) may use only part of them, or none where
 * one pass is faster, and they do not grow evenly with pos0 (the ranges of keys change): one buffer for many
 * calls takes the largest over their geometries, or it_attention_dispatch_room, which is always enough. */
size_t it_attn_scratch_bytes(int pos0, int nt, int hd, int nh, int nkv);

/* Causal GQA attention with sigmoid output gate, f32 accumulation.
 *   q    : f32. Token t, q-head h: q[t*q_tok_stride + h*2*hd + d] for d < hd is the (normed, roped)
 *          query and d in [hd, 2hd) the output gate (the reference's q row, cpu.rs:249-254).
 *   kc,vc: f16 cache [pos][kvd], kvd = nkv*hd; KV head kh at column kh*hd. Rows 0..pos0+nt-1 must
 *          be written (append first with it_kv_append_f16).
 *   Token t attends keys 0..pos0+t (n = pos0+t+1, cpu.rs:260; kernels/src/lib.rs:764); q-head h
 *   reads KV head h/(nh/nkv) (cpu.rs:265).
 *   out  : f32 out[t*out_tok_stride + h*hd + d] = softmax(scale*q.K) V * sigmoid(gate).
 *   scratch: device buffer for the partial records (split-K: 260 f32 words per token, head and split;
 *          flash key splits: 132 words, O as int16). it_attn_scratch_bytes(...) bytes give the
 *          library's preferred split; with fewer, decode and verify calls double the keys per split
 *          until the records fit (the reference's rule for its fixed arena, src/vk/mod.rs:714-716) and
 *          prompt calls take the fastest split whose records fit, or one pass with no scratch. The reference's own room,
 *          it_attention_dispatch_room(ctx_len, nh, nt) * 4 bytes, is always enough. NULL = 0 bytes.
 * Requires hd == 256, nh % nkv == 0, q_tok_stride and out_tok_stride multiples of 4, 16-byte
 * aligned q/out/kc/vc (the reference asserts the same f16 layout, src/vk/mod.rs:713).
 * Replaces VkEngine::attention_kv(qo,qts,kco,vco,kvd,pos0,hd,nh,nkv,oo,nt,f16=true),
 * src/vk/mod.rs:710-729, i.e. the split-K partial dispatch plus attn_comb. One entry point covers
 * decode (nt=1), MTP verify (nt<=4), chunked prefill (nt=64, pos0>0) and whole-prompt prefill. */
int it_attn_f16(const float* q, int q_tok_stride, const uint16_t* kc, const uint16_t* vc, int kvd,
                int pos0, int hd, int nh, int nkv, int nt, float scale, float* out, int out_tok_stride,
                void* scratch, size_t scratch_bytes, void* stream);

/* it_attn_f16 with the kernel choice exposed (the reference's BONSAI_PREFILL_ATTN / chunk policy,
 * src/vk/mod.rs:714-717 and 192-204):
 *   kernel 0 = automatic (what it_attn_f16 does), 1 = split-K partials + combine,
 *          2 = flash prefill (any nt; the automatic choice from nt = 16): one pass with no scratch,
 *          or, when one pass would leave most of the GPU idle (a short chunk after a long context),
 *          key splits whose
 *          partial records (132 words: {m, l, k, 0} and O as int16 in units of k) are merged like
 *          kernel 1's,
 *          3 = kernel 2 with lossless key-split records: the split-K kernel's 260-word f32 form
 *          {m, l, 0, 0, o[256]} instead of int16 O (twice the scratch; the same result as one
 *          pass up to f32 reassociation of the merge).
 *   chunk  = keys per split, 0 = automatic: a multiple of 32 for kernel 1 (the automatic split is
 *          32 keys for 1-2 tokens below 2048 keys, else 64), of 64 for kernels 2 and 3, where a
 *          chunk of at least pos0 + nt means one pass.
 * it_attn_scratch_bytes_ex gives the scratch for the same choice. With chunk = 0 the split is fitted
 * to scratch_bytes as in it_attn_f16; an explicit chunk needs its full record set. */
size_t it_attn_scratch_bytes_ex(int pos0, int nt, int hd, int nh, int nkv, int kernel, int chunk);
int it_attn_f16_ex(const float* q, int q_tok_stride, const uint16_t* kc, const uint16_t* vc, int kvd,
                   int pos0, int hd, int nh, int nkv, int nt, float scale, float* out, int out_tok_stride,
                   void* scratch, size_t scratch_bytes, int kernel, int chunk, void* stream);

/* it_attn_f16 with the flash prefill kernel's query operand given pre-converted: q16 as written by
 * it_attn_prep_f16_q16 with the same scale (f16(q * scale * log2(e)), token stride q16_tok_stride).
 * The result is identical, bit for bit, to it_attn_f16 on the f32 q that q16 was made from; q
 * still provides the gates, and calls that take the split-K kernels (nt < 16) read q as
 * it_attn_f16 does. Same scratch rule and requirements as it_attn_f16. No counterpart in the
 * reference; see it_attn_prep_f16_q16. */
int it_attn_f16_q16(const float* q, int q_tok_stride, const uint16_t* q16, int q16_tok_stride, const uint16_t* kc,
                    const uint16_t* vc, int kvd, int pos0, int hd, int nh, int nkv, int nt, float scale, float* out,
                    int out_tok_stride, void* scratch, size_t scratch_bytes, void* stream);

/* it_attn_f16 that allocates nothing and takes no scratch argument. No counterpart in the reference:
 * it is for callers that cannot allocate device memory or hand over a workspace (code under HIP
 * graph capture, tight serving loops, harnesses that forbid hipMalloc). The partial records (split-K,
 * or the flash kernel's int16 key-split records) go to a file-scope device array of IT_NOALLOC_SCRATCH_BYTES (16 MiB) that each GPU the
 * library runs on holds until the process ends; the split is fitted to that size as for a caller
 * buffer of the same size (it_attn_plan(..., IT_NOALLOC_SCRATCH_BYTES, ...) gives the choice), and
 * a geometry whose records cannot fit (split-K with nt*nh*1040 bytes above the maximum) is rejected
 * with an error before any device work. Nothing in the array needs to start at zero: every record a
 * merge reads is written earlier in the same call. All calls on one GPU share that GPU's array, so
 * calls that overlap on one GPU (different streams, or graphs replayed concurrently) race; calls in
 * order on one stream do not. Other arguments and results as it_attn_f16. */
#define IT_NOALLOC_SCRATCH_BYTES ((size_t)16 << 20)
int it_attn_f16_noalloc(const float* q, int q_tok_stride, const uint16_t* kc, const uint16_t* vc, int kvd,
                        int pos0, int hd, int nh, int nkv, int nt, float scale, float* out, int out_tok_stride,
                        void* stream);

/* Decode attention in one launch. Replaces the same reference call as it_attn_f16 for decode
 * (VkEngine::attention_kv, src/vk/mod.rs:710-729: the attn_s_h partial dispatch and attn_comb,
 * kernels/src/lib.rs:722-798), with the split records and their merge in one kernel: each split
 * writes its record to a caller-owned mailbox, per 16 output dims, and the waves that merge a
 * (token, head, 16 dims) unit wait for exactly the pieces they read. Results are bit-identical to
 * it_attn_f16's. Slower than it_attn_f16 on MI355X (9.7 against 9.4 us per layer at ctx 8192),
 * and it relies on its whole grid being resident at once, so it_attn_f16 is the default; this
 * form is for a GPU the caller has to itself where one launch per layer matters. Taken when the geometry qualifies: a split-K call (nt < 16) with at most 8 query
 * rows per KV head (nt * nh / nkv <= 8: decode), at most 256 splits of 64 keys (pos0 + nt <= 16384)
 * and enough of them to give every (token, head, 16-dim block) merge a wave of its own (nt * nh *
 * 16 <= 4 * splits * nkv * row groups: with fewer, as at ctx 512, two launches are faster),
 * a mailbox of at least it_attn_mailbox_bytes(pos0 + nt, nt, nh) bytes, and a grid the device
 * holds at once (so every piece a merge waits for is being produced). Any other call runs
 * it_attn_f16 with `scratch` / `scratch_bytes`; it_attn_mailbox_would_launch reports which.
 *
 * The mailbox: 16-byte aligned device memory, initialised once with it_attn_mailbox_init and left
 * initialised by every call (each merge clears what it read). One mailbox serves any sequence of
 * calls in order on one stream (every layer and step of an engine); calls that overlap on the
 * device (other streams, concurrent graph replays) need one each. A merge that has waited 10 ms
 * (possible only if other work holds the device's compute units) gives up, writes NaN outputs and
 * poisons the mailbox: every later call then gives NaN at once until it_attn_mailbox_init runs
 * again. A mailbox that was never initialised (or was overwritten) is treated as poisoned too;
 * it_attn_mailbox_poisoned reports either. A merge that finds its mailbox poisoned also sets a
 * host-visible word that it_attn_mailbox_init allocates for the mailbox (pinned, one per mailbox,
 * kept until the process ends), so once such a call has completed, the next it_attn_f16_mailbox
 * call with that mailbox returns -1 ("poisoned", before any device work) instead of NaN again. */
size_t it_attn_mailbox_bytes(int ctx, int nt, int nh);
int it_attn_mailbox_init(void* mailbox, size_t bytes, void* stream);
int it_attn_mailbox_poisoned(const void* mailbox, int* poisoned, void* stream);   /* synchronises stream */
int it_attn_mailbox_would_launch(int pos0, int nt, int hd, int nh, int nkv, size_t mailbox_bytes);
int it_attn_f16_mailbox(const float* q, int q_tok_stride, const uint16_t* kc, const uint16_t* vc, int kvd,
                        int pos0, int hd, int nh, int nkv, int nt, float scale, float* out, int out_tok_stride,
                        void* mailbox, size_t mailbox_bytes, void* scratch, size_t scratch_bytes, void* stream);

/* The choice it_attn_f16 makes for this geometry and scratch budget: *kernel 1 (split-K) or 2
 * (flash), *chunk keys per split (0 = flash in one pass), *bytes of scratch to give the call:
 * it_attn_scratch_bytes where the budget holds them (flash may use less, or none), else what the
 * records of the split take. A call with *bytes of scratch makes the same choice.
 * Returns nonzero if no split fits (only possible for nt < 16 with fewer than nt*nh*1040 bytes).
 * Scratch per split: the split-K kernel's records are 260 f32 words per (token, head); the flash
 * kernel's key-split records are 132 words per (token, head): {m, l, k, 0} and O as int16 in
 * units of k = max|O| / 32767 (an error of at most max|O| / 65534 per value before the merge).
 * Host-only; the split-K chunk loop is the reference's, src/vk/mod.rs:714-716. */
int it_attn_plan(int pos0, int nt, int hd, int nh, int nkv, size_t scratch_bytes, int* kernel, int* chunk,
                 size_t* bytes);

/* The two phases of the split-K path as separate calls (the reference dispatches them separately
 * too: attn_s_h then attn_comb, src/vk/mod.rs:725-727). Partial record of (token t, q-head h,
 * split s) is 260 floats {m, l, 0, 0, o[256]} at part + ((t*nh + h)*smax + s)*260 with
 * smax = ceil((pos0+nt)/chunk): m = max score, l = sum exp(score - m), o = sum exp(score - m) v
 * over the split's keys visible to token t (kernels/src/lib.rs:753-798). Records of splits a token
 * cannot see are never read (they are left untouched or written as {-inf, 0, 0, 0, 0...}). A sequence-sharded caller can exchange these records and run
 * it_attn_combine locally.
 *   it_attn_partials: part must hold it_attn_scratch_bytes_ex(pos0,nt,hd,nh,nkv,1,chunk) bytes.
 *   it_attn_combine : out = merge of the records of splits 0..ceil((pos0+t+1)/chunk)-1, times
 *                     sigmoid(gate) (kernels/src/lib.rs:722-740). */
int it_attn_partials(const float* q, int q_tok_stride, const uint16_t* kc, const uint16_t* vc, int kvd, int pos0,
                     int hd, int nh, int nkv, int nt, float scale, float* part, size_t part_bytes, int chunk,
                     void* stream);
int it_attn_combine(const float* q, int q_tok_stride, const float* part, int pos0, int hd, int nh, int nt, int chunk,
                    float* out, int out_tok_stride, void* stream);

/* The same two phases with a choice of record layout. layout 0: the 260-float records above (these
 * calls are then it_attn_partials / it_attn_combine). layout 1: the records it_attn_f16 itself
 * uses when its merge takes one wave per (token, head, 16 output dims), i.e. for 9-256 splits and
 * at most 256 (token, head) rows (decode and verify at long contexts; other geometries are
 * refused): the same f32 values, O as 64-byte pieces of 16 floats at
 * part + (((t*nh + h)*16 + d/16)*smax + s)*16 (+ d % 16), then {m, l} at
 * part + nt*nh*smax*256 + ((t*nh + h)*smax + s)*2, 1,032 bytes per (token, head, split) inside
 * the same part_bytes. The merge's lanes, one split each, then read adjacent pieces, which makes
 * the merge faster (ctx 8192: 8.45 against 9.0 us per layer); the output is bit-identical to
 * layout 0. Extends the reference's attn_s_h / attn_comb pair (kernels/src/lib.rs:722-798), which
 * has one layout only. */
int it_attn_partials_ex(const float* q, int q_tok_stride, const uint16_t* kc, const uint16_t* vc, int kvd, int pos0,
                        int hd, int nh, int nkv, int nt, float scale, float* part, size_t part_bytes, int chunk,
                        int layout, void* stream);
int it_attn_combine_ex(const float* q, int q_tok_stride, const float* part, int pos0, int hd, int nh, int nt, int chunk,
                       int layout, float* out, int out_tok_stride, void* stream);

/* ------------------------------------------------------------------------------------------------
 * The MTP head's attention over its own f32 KV cache (src/mtp.rs:96-130; src/vk/mod.rs:917-942).
 * Slot p of that cache holds position p + 1 (mtp.rs:120, vk/mod.rs:932).
 * ---------------------------------------------------------------------------------------------- */

/* it_attn_prep_f16 for an f32 cache: token t is roped at position pos0 + t and its normed, roped K
 * row and its V row are stored as f32 at cache row row0 + t (for the MTP head row0 = pos0 - 1).
 * Replaces the MTP pass's rmsnorm mode 0 (q_norm, k_norm) and rope dispatches, src/vk/mod.rs:933-938
 * (its k/v matvecs write the cache rows directly; here they write k, v and this call stores them). */
int it_attn_prep_f32kv(float* q, int q_tok_stride, const float* k, const float* v, int kv_tok_stride,
                       const float* q_norm, const float* k_norm, float eps, float* kc, float* vc, int kvd,
                       int pos0, int row0, int hd, int nh, int nkv, int nt, int n_rot, float theta_scale, int sec0,
                       int sec1, int sec2, int sec3, void* stream);

/* Bytes of scratch it_attn_f32kv prefers (split-K partial records, same 260-float layout: 64-key
 * splits for one block of up to 32 query rows per KV head, longer splits for multi-block calls);
 * any smaller scratch also works (it_attn_f32kv_plan). */
size_t it_attn_f32kv_scratch_bytes(int pos0, int nt, int hd, int nh, int nkv);

/* The split it_attn_f32kv uses for a scratch of scratch_bytes: *chunk keys per split and *bytes of
 * records, or *chunk = 0 and *bytes = 0 for the one-pass form that needs no scratch. The preferred
 * split is kept when it fits; otherwise the split doubles until the records fit, the reference's
 * rule for the MTP head's attention (src/vk/mod.rs:730-733, C doubling from 64 while
 * nt*nh*ceil((pos0+nt)/C)*260 words exceed the room); when even one record per (token, head) does
 * not fit it takes the one-pass form, as the reference falls back to its whole-context `attn`
 * kernel (src/vk/mod.rs:740, kernels/src/lib.rs:83-116). Returns 0, or -1 for a bad geometry. */
int it_attn_f32kv_plan(int pos0, int nt, int hd, int nh, int nkv, size_t scratch_bytes, int* chunk, size_t* bytes);

/* Causal GQA attention with sigmoid gate over an f32 KV cache: it_attn_f16's semantics and
 * buffers with kc, vc as f32 [row][kvd]. Query t sees cache rows 0..pos0+t (for the MTP head pass
 * pos0 is the first query's slot, position - 1). hd == 256, at most 16 q heads per KV head. The
 * split fits whatever scratch the caller passes (it_attn_f32kv_plan); a null scratch or one too
 * small for a record per (token, head) runs the one-pass form.
 * Replaces VkEngine::attention(..., f16 = false) for the MTP head, src/vk/mod.rs:707-709 and 942
 * (attn_s + attn_comb, kernels/src/lib.rs:682-740; CPU src/mtp.rs:122-130). */
int it_attn_f32kv(const float* q, int q_tok_stride, const float* kc, const float* vc, int kvd, int pos0, int hd,
                  int nh, int nkv, int nt, float scale, float* out, int out_tok_stride, void* scratch,
                  size_t scratch_bytes, void* stream);

/* ------------------------------------------------------------------------------------------------
 * Gated DeltaNet: short causal conv, q/k L2 norm, gated-delta recurrence.
 * ---------------------------------------------------------------------------------------------- */

/* Depthwise causal conv (kernel K in 2..4) + SiLU over nt tokens, carrying the rolling (K-1)-token
 * state (oldest first) across calls.
 *   x     : f32 x[t*x_tok_stride + ch], ch < cd (the qkv projection output)
 *   w     : f32 w[ch*K + i]             (ssm_conv1d.weight)
 *   state : f32 state[i*cd + ch], i < K-1, updated in place to the last K-1 inputs
 *   out   : f32 out[t*out_tok_stride + ch]  (must not alias x or state)
 * Replaces the conv dispatch, src/vk/mod.rs:803 (kernel kernels/src/lib.rs:119-140; CPU
 * cpu.rs:201-212). */
int it_gdn_conv(const float* x, int x_tok_stride, const float* w, float* state, float* out,
                int out_tok_stride, int cd, int nt, int K, void* stream);

/* In-place L2 normalisation x / max(||x||, eps) of nheads consecutive rows of length d per token:
 * row r of token t is x[t*tok_stride + r*d ...]. d must be 128 or 256.
 * Replaces rmsnorm mode 2 on the 2*nk q/k heads, src/vk/mod.rs:804 (kernels/src/lib.rs:207-229;
 * cpu.rs:214). */
int it_l2norm_heads(float* x, int tok_stride, int nheads, int d, int nt, float eps, void* stream);

/* it_gdn_conv followed by it_l2norm_heads(out, ..., nnorm, 128, ...) in one pass: channels
 * [0, nnorm*128) (the q and k heads, nnorm = 2*nk) are L2-normalised per 128-channel head and token
 * after the conv + SiLU, the rest (v) are written as the conv gives them. Same buffers and state
 * rules as it_gdn_conv; cd must be a multiple of 128.
 * Replaces the conv and rmsnorm mode 2 dispatch pair, src/vk/mod.rs:803-804 (cpu.rs:201-214). */
int it_gdn_conv_l2norm(const float* x, int x_tok_stride, const float* w, float* state, float* out,
                       int out_tok_stride, int cd, int nt, int K, int nnorm, float eps, void* stream);

/* Gated-delta recurrence, token by token, for nt tokens (decode: nt=1).
 *   co    : f32 normalised conv output, token t at co[t*co_tok_stride]: q heads [0, nk*S),
 *           k heads [nk*S, 2*nk*S), v heads [2*nk*S, 2*nk*S + nv*S). V head h uses q/k head h % nk.
 *   beta_raw, alpha_raw: f32 [t*ba_tok_stride + h]; beta = sigmoid(beta_raw),
 *           g = softplus(alpha_raw + dt[h]) * a[h] (a < 0 is the decay rate), S <- exp(g) S.
 *   dt, a : f32 [nv]
 *   state : f32 [nv][S][S], element [h][i][j] = S_h[i][j], i = key index, j = value index
 *           (the GPU arena layout of shaders/gdn.comp:2), updated in place.
 *   out   : f32 out[t*out_tok_stride + h*S + j] = (S_h^T q)_j / sqrt(S)
 * Requires S == 128, nv % nk == 0.
 * Replaces the gdn / gdn_p dispatches, src/vk/mod.rs:805-806 and the per-token MTP-verify loop
 * 797-801 (kernels/src/lib.rs:252-331; CPU cpu.rs:216-232). */
int it_gdn_step(const float* co, int co_tok_stride, const float* beta_raw, const float* alpha_raw,
                int ba_tok_stride, const float* dt, const float* a, float* state, float* out,
                int out_tok_stride, int nt, int nv, int nk, int S, void* stream);

/* A GDN decode layer in one launch: it_gdn_conv_l2norm (nnorm = 2*nk) followed by it_gdn_step,
 * for 1 <= nt <= 4 tokens, without the conv output ever reaching memory.
 *   x, x_tok_stride, w, K : as for it_gdn_conv (cd = (2*nk + nv)*S); x and w 16-byte aligned,
 *                           stride % 4 == 0
 *   conv_state_in         : f32 [(K-1)][cd], the conv state before token 0 (read only)
 *   conv_state_out        : f32 [(K-1)][cd], receives the conv state after token nt-1; it must not
 *                           overlap conv_state_in (every workgroup reads the old state while others
 *                           write the new one: callers alternate two buffers)
 *   the rest              : as for it_gdn_step (state updated in place), eps as for the L2 norm.
 * Replaces the conv, rmsnorm mode 2 and gdn dispatch triple, src/vk/mod.rs:803-806 (cpu.rs:201-232). */
int it_gdn_decode_fused(const float* x, int x_tok_stride, const float* w, int K, const float* conv_state_in,
                        float* conv_state_out, const float* beta_raw, const float* alpha_raw, int ba_tok_stride,
                        const float* dt, const float* a, float* state, float* out, int out_tok_stride, int nt,
                        int nv, int nk, int S, float eps, void* stream);

/* it_gdn_decode_fused for an MTP verify batch, plus the checkpoints of both states after token
 * ck_after (0 <= ck_after < nt), written from registers: ck_state [nv][S][S] (the recurrent state,
 * as it_gdn_step_ckpt) and ck_conv [(K-1)][cd] (the conv state, as it_gdn_conv_l2norm_ckpt). Neither
 * may overlap the state it snapshots or the other buffers.
 * Replaces the verify loop's conv / rmsnorm / gdn dispatches and checkpoint copies,
 * src/vk/mod.rs:790-806 (mtp.rs:227-234). */
int it_gdn_decode_fused_ckpt(const float* x, int x_tok_stride, const float* w, int K, const float* conv_state_in,
                             float* conv_state_out, const float* beta_raw, const float* alpha_raw,
                             int ba_tok_stride, const float* dt, const float* a, float* state, float* out,
                             int out_tok_stride, int nt, int nv, int nk, int S, float eps, float* ck_state,
                             float* ck_conv, int ck_after, void* stream);

/* The GDN output's gated RMSNorm, per (token t, V head h) row of S = 128:
 *   out[t*out_tok_stride + h*S + j] = o_j / sqrt(mean_j(o^2) + eps) * w[j] * silu(z[t*z_tok_stride + h*S + j])
 * with o the row o[t*o_tok_stride + h*S ...] and w [S] (ssm_norm, shared by the heads). out may be
 * o itself (in place, like the reference) or a buffer that does not overlap it.
 * Replaces rmsnorm mode 1, src/vk/mod.rs:808 (kernels/src/lib.rs:207-229; cpu.rs:234-238). */
int it_gdn_gated_rmsnorm(const float* o, int o_tok_stride, const float* z, int z_tok_stride, const float* w,
                         float eps, float* out, int out_tok_stride, int nv, int S, int nt, void* stream);

/* it_gdn_step with the gated RMSNorm fused into the output write: one workgroup per V head holds
 * the head's whole state, so each token's output row is complete before it is stored.
 *   z, norm_w, eps: as for it_gdn_gated_rmsnorm (z 16-byte aligned, z_tok_stride a multiple of 4);
 *          z == NULL writes the plain recurrence output (same values as it_gdn_step).
 *   ck_state, ck_after: the optional MTP verify checkpoint as in it_gdn_step_ckpt (NULL = none).
 * Replaces the gdn dispatch plus rmsnorm mode 1, src/vk/mod.rs:805-808 (cpu.rs:216-238). */
int it_gdn_step_gated(const float* co, int co_tok_stride, const float* beta_raw, const float* alpha_raw,
                      int ba_tok_stride, const float* dt, const float* a, float* state, float* out,
                      int out_tok_stride, int nt, int nv, int nk, int S, const float* z, int z_tok_stride,
                      const float* norm_w, float eps, float* ck_state, int ck_after, void* stream);

/* ------------------------------------------------------------------------------------------------
 * MTP verify checkpoint and rollback of the recurrent state.
 * The reference runs a verify batch (the accepted token x and the draft d) one token at a time and
 * copies the conv and SSM states after token 0 into checkpoint buffers (src/vk/mod.rs:790-801); a
 * rejected draft copies them back (mtp_reject, src/vk/mod.rs:1018-1025; CPU: mtp.rs:227-234).
 * Here the kernels that already hold the state for the whole token run write the checkpoint from
 * registers after token ck_after (0 <= ck_after < nt), without a second pass over the state.
 * ck_state has the layout of the state it snapshots and must not overlap it.
 * ---------------------------------------------------------------------------------------------- */

/* it_gdn_conv, plus ck_state[i*cd + ch] = the conv state after token ck_after. */
int it_gdn_conv_ckpt(const float* x, int x_tok_stride, const float* w, float* state, float* out,
                     int out_tok_stride, int cd, int nt, int K, float* ck_state, int ck_after, void* stream);

/* it_gdn_conv_l2norm, plus the conv-state checkpoint after token ck_after. */
int it_gdn_conv_l2norm_ckpt(const float* x, int x_tok_stride, const float* w, float* state, float* out,
                            int out_tok_stride, int cd, int nt, int K, int nnorm, float eps, float* ck_state,
                            int ck_after, void* stream);

/* it_gdn_step, plus ck_state[h][i][j] = the SSM state after token ck_after (16-byte aligned). */
int it_gdn_step_ckpt(const float* co, int co_tok_stride, const float* beta_raw, const float* alpha_raw,
                     int ba_tok_stride, const float* dt, const float* a, float* state, float* out,
                     int out_tok_stride, int nt, int nv, int nk, int S, float* ck_state, int ck_after,
                     void* stream);

/* Rollback after a rejected draft: conv_state <- ck_conv (conv_words floats) and ssm <- ck_ssm
 * (ssm_words floats), both in one copy kernel on the stream (either count may be 0; no buffer may
 * overlap another). */
int it_gdn_rollback(const float* ck_conv, float* conv_state, size_t conv_words, const float* ck_ssm, float* ssm,
                    size_t ssm_words, void* stream);

/* Same contract and result as it_gdn_step over nt tokens, computed with the chunk-64 WY/UT form of
 * the gated delta rule on f16 MFMA with f32 state and accumulation (a new algorithm: the reference
 * runs the recurrence token-sequentially, kernels/src/lib.rs:285-331). Scratch as returned by
 * it_gdn_chunked_scratch_bytes. The q and k heads must be L2-normalised, as the layer's rmsnorm
 * mode 2 leaves them before the recurrence (cpu.rs:214): the chunk operands are kept as f16, which
 * assumes |k| <= 1 (it_gdn_step has no such bound). */
size_t it_gdn_chunked_scratch_bytes(int nt, int nv, int S);
int it_gdn_chunked(const float* co, int co_tok_stride, const float* beta_raw, const float* alpha_raw,
                   int ba_tok_stride, const float* dt, const float* a, float* state, float* out,
                   int out_tok_stride, int nt, int nv, int nk, int S, void* scratch,
                   size_t scratch_bytes, void* stream);

/* The GDN layer over a prompt chunk in one call: replaces the conv (src/vk/mod.rs:803), rmsnorm
 * mode 2 on the q/k heads (804) and gdn_p (806) dispatches of a prefill chunk. Conv + SiLU + q/k
 * L2 norm (as it_gdn_conv_l2norm with nnorm = 2*nk), its output kept in `scratch` as f16 (the
 * "f16 activations" of the chunked-prefill benchmark: half the bytes for the conv's write and the
 * scan's read; at 8192 tokens the outputs are within ~1.2e-4 and the final state within ~8.5e-4
 * of the f32 token-sequential reference, against ~8e-5 / ~4.4e-4 from an f32 conv output),
 * then the chunk-64 scan of it_gdn_chunked. x [nt][x_tok_stride] f32 with cd = (2*nk+nv)*S
 * channels; w, conv_state, beta_raw, alpha_raw, dt, a, state and out as it_gdn_conv and
 * it_gdn_chunked (S = 128); conv_state and state are updated in place. scratch: 16-byte aligned,
 * it_gdn_prefill_scratch_bytes(nt, nv, nk, S) bytes. */
size_t it_gdn_prefill_scratch_bytes(int nt, int nv, int nk, int S);
int it_gdn_prefill(const float* x, int x_tok_stride, const float* conv_w, int K, float* conv_state,
                   const float* beta_raw, const float* alpha_raw, int ba_tok_stride, const float* dt,
                   const float* a, float* state, float* out, int out_tok_stride, int nt, int nv, int nk, int S,
                   float eps, void* scratch, size_t scratch_bytes, void* stream);

/* ------------------------------------------------------------------------------------------------
 * Verification of a drafted token tree. The reference drafts chains (src/mtp.rs:166-204: one draft a step, checked by
 * a batch of two); with several candidates a step the batch is a tree, and these calls stand where the chain's do:
 *   it_tree_plan                    once a step: masks and positions from the parents
 *   it_attn_prep_pos_f16            positions of the nodes; node t in cache row pos0 + t     (it_attn_prep_f16)
 *   it_attn_tree_f16                attention over the cache and each node's own ancestors   (it_attn_f16)
 *   it_gdn_tree                     the recurrent layer over the tree                        (it_gdn_decode_fused)
 *   it_kv_tree_commit_f16, it_gdn_tree_commit   keep the accepted node's path, drop the rest (it_gdn_rollback)
 * A tree is nt <= IT_TREE_MAX nodes in topological order (a parent before its children). anc: device uint64 [nt], bit j
 * of anc[t] set for node t itself and its ancestors; 0 makes t a padding node (the output rows are zeros, and no
 * node may name it an ancestor). Several nodes may follow the last committed token.
 * ---------------------------------------------------------------------------------------------- */
#define IT_TREE_MAX 64

/* anc [nt] and, unless NULL, pos [nt] (int32, p0 + depth: p0 is the position of the first node after the last
 * committed token) from parent: device int32 [nt], -1 for a node that follows the last committed token. A node whose
 * parent is not in -1 .. t-1 is padding, and so are its descendants (anc 0, pos p0). */
int it_tree_plan(const int32_t* parent, int nt, int p0, uint64_t* anc, int32_t* pos, void* stream);

/* it_attn_f16 for nodes of a tree: query row t sees cache rows 0 .. pos0-1 and the rows pos0 + j of the nodes j < rows whose
 * bit is set in anc[t] (higher bits are ignored). Verification asks for all nodes at once, nt = rows; drafting level by
 * level asks for the newest ones, with anc pointing at their masks and rows counting all nodes so far. Rows that a node
 * does not see are not read for it, whatever they hold. A row without any bit is zeros. pos0 may be 0. Other arguments
 * and the result as for it_attn_f16. rows in 1 .. IT_TREE_MAX; nt as well.
 * Accuracy: sums in f32. q is carried as f16 pairs of 22 bits (each row scaled by a power of two of its own, so its size and
 * that of `scale` do not matter), which moves an output by about 2e-6 of the largest value where scores are of ordinary size
 * (some tens at most). The context's probabilities are carried as f16 pairs with a step of their own: 2^-31 of a row's largest
 * in calls of many rows or long contexts, but 2^-25 of the largest in a split in the others, where what is smaller is lost. So one
 * key that outweighs n others of its split by 2^25 loses them, n * 2^-25 of the result: up to 3e-5 with the library's splits
 * (1024 keys at most), and as much as the whole context makes of n with the smallest scratch.
 * scratch: the context's records; it_attn_tree_scratch_bytes(...) bytes give the library's split, with fewer the
 * splits get longer, and nt * nh * 1040 bytes are always enough (0 for pos0 = 0). Calls that overlap need one each. */
size_t it_attn_tree_scratch_bytes(int pos0, int nt, int hd, int nh, int nkv);
int it_attn_tree_f16(const float* q, int q_tok_stride, const uint16_t* kc, const uint16_t* vc, int kvd, int pos0, int hd,
                     int nh, int nkv, int nt, int rows, const uint64_t* anc, float scale, float* out, int out_tok_stride,
                     void* scratch, size_t scratch_bytes, void* stream);

/* The same over the MTP head's f32 cache (at most 16 q heads per KV head), f32 throughout: for drafting a tree with the
 * head. Stands where it_attn_f32kv does for a chain. */
size_t it_attn_tree_f32kv_scratch_bytes(int pos0, int nt, int hd, int nh, int nkv);
int it_attn_tree_f32kv(const float* q, int q_tok_stride, const float* kc, const float* vc, int kvd, int pos0, int hd,
                       int nh, int nkv, int nt, int rows, const uint64_t* anc, float scale, float* out, int out_tok_stride,
                       void* scratch, size_t scratch_bytes, void* stream);

/* Keeps the path of node `leaf` in a cache whose rows pos0 + t hold the nodes: row pos0 + i <- row pos0 + path[i], path
 * the nodes of anc[leaf] in order (in place; the rows after the path keep what they hold). leaf = -1, or a padding
 * node (its own bit is clear): nothing is kept and nothing moves. kvd a multiple of 8, kc and vc 16-byte aligned and not the
 * same rows (both are moved at once). */
int it_kv_tree_commit_f16(uint16_t* kc, uint16_t* vc, int kvd, int pos0, int nt, const uint64_t* anc, int leaf,
                          void* stream);
int it_kv_tree_commit_f32(float* kc, float* vc, int kvd, int pos0, int nt, const uint64_t* anc, int leaf,
                          void* stream);

/* The recurrent layer over a tree: conv + SiLU over each node's own ancestors (before the first node of a path, the conv
 * state), q/k L2 norm and the gated delta rule along every path, for all nodes at once, in one launch. For a
 * chain it computes what it_gdn_decode_fused does for consecutive tokens.
 *   x, w, K, beta_raw, alpha_raw, dt, a, eps: as for it_gdn_decode_fused (x 16-byte aligned, its stride % 4 == 0)
 *   conv_state [(K-1)][cd], state [nv][S][S]: the committed states, only read
 *   anc: bits after t and a node whose own bit is clear (padding: zeros out) are ignored
 *   out [t*out_tok_stride + h*S + j], as it_gdn_step's
 *   trace: it_gdn_tree_trace_bytes(...) bytes, 16-byte aligned, one per layer: what it_gdn_tree_commit needs
 * Accuracy: the normalised q and k rows (each at length 1) and the state's columns (each scaled by a power of two) go into the
 * products as pairs of f16, 22 bits of a value that is not far below its row's or column's largest; sums, solve and
 * updates are f32, the decays of a path summed in f64; SiLU, norms and gates take the hardware's exponential, logarithm, root and
 * reciprocal (about 2^-23 each). The k rows that the trace keeps for the commit are the 22-bit ones. Outputs and committed states
 * are about 3e-7 off relative to their size (normal inputs), 2 to 2.5 times an f32 computation's error. A node's result does
 * not depend on nodes that are not its ancestors, whatever their inputs hold. */
size_t it_gdn_tree_trace_bytes(int nt, int nv, int nk, int S);
int it_gdn_tree(const float* x, int x_tok_stride, const float* w, int K, const float* conv_state,
                const float* beta_raw, const float* alpha_raw, int ba_tok_stride, const float* dt, const float* a,
                const float* state, const uint64_t* anc, float* out, int out_tok_stride, int nt, int nv, int nk, int S,
                float eps, void* trace, size_t trace_bytes, void* stream);

/* conv_state and state <- those after node `leaf` of the it_gdn_tree call that wrote trace (the same x, anc, nt and
 * head counts; both updated in place). leaf = -1, or a padding node: they stay. Stands where it_gdn_rollback does for a
 * chain. */
int it_gdn_tree_commit(const float* x, int x_tok_stride, int K, float* conv_state, float* state, const uint64_t* anc,
                       int leaf, int nt, int nv, int nk, int S, const void* trace, size_t trace_bytes, void* stream);

/* ------------------------------------------------------------------------------------------------
 * A paged K/V cache in 8 bits, for several sequences or one with a long context, in half the bytes of the f16 cache. No
 * counterpart in the reference, whose cache is one f16 array for one sequence (src/vk/mod.rs:551-554). A step:
 *   it_attn_prep_pos_f16   K and V of the new tokens into f16 rows (a staging buffer as its cache, row0 = 0)
 *   it_kv8_append          those rows into the cache                    (it_kv_append_f16)
 *   it_attn_kv8            attention of the new tokens                  (it_attn_f16)
 * The lengths and page tables are on the device, so that a captured step is replayed as they advance: the calls read len,
 * the caller adds the tokens that it keeps.
 *
 * Rows: a page holds IT_KV8_PAGE rows of all KV heads. Row r of a sequence is in page table[seq][r / 64]. While a sequence
 * holds `total` rows, the pages that are full, those before total / 64, are 8-bit codes, and the rows after them (at most
 * 63) are f16 in the sequence's open buffer, which has room for two pages: page p in half p % 2, until a row of page p + 2 is
 * written there.
 * Taking rows back (drafts that a check rejects): a smaller length alone does it, to any page's end, or into a page whose rows still
 * stand in the open buffer, which is page `lowest` or a later one. The caller keeps that number for each sequence:
 *   0 at first;  after an append to `total` rows  max(lowest, (total - 1) / 64 - 1);  after a cut to `to` rows  min(lowest, to / 64)
 * So up to 64 of a call's own rows can always be taken back. Not always 64 rows after an earlier cut: 126 rows and four drafts are
 * 130, so page 2 has the half of page 0, and has it still when three drafts are taken back and 127 rows are left. Into a page before
 * `lowest`: to the page's start, with its rows read (it_kv8_read) before that and appended anew.
 * Codes: each IT_KV8_BLOCK rows of a KV head have a scale s for K and one for V: the largest size / 127, rounded up to four
 * significant bits or to a multiple of 2^-24 (at least that). A value x is kept as code = 128 + x / s, rounded to the nearest, ties to
 * even, and at most 127 from 128 (113 where s is above 512); it stands for (code - 128) * s, which is an f16 number. Appending makes
 * values finite: an infinity becomes the largest f16, a NaN 0.
 * Sharing: a table may name a page that another one names. The calls write only to pages that a sequence fills, those from
 * len / 64 on, so pages before that can be shared (a common beginning, a fork); a fork takes the open rows with it
 * (it_kv8_copy; `lowest` goes with them) and needs pages of its own from len / 64 on. A cut into a shared page needs another page
 * named in its place first, as rows appended then fill it anew. A page that no table names is free; nothing in it needs to be cleared.
 *
 * Device arrays of a call, int32, for the cache's nseq sequences: start [nseq + 1], len [nseq], table [nseq][max_pages]. The
 * call's tokens start[i] .. start[i+1]-1 are the next rows of sequence i after its len[i] rows; start[i] = start[i+1]: none.
 * ntok: rows of the token arrays; max_nt: a bound of the tokens of one sequence (tokens beyond it are left out; it chooses the kernel, so
 * give the true one). Tokens of no sequence (after start[nseq]) are left alone. A sequence whose bounds are not in 0 .. ntok has no
 * tokens. One whose length is negative, or whose rows its table cannot name, is not appended to, and its
 * outputs are NaN. A page number outside the pool is not written, and what reads it is NaN.
 * ---------------------------------------------------------------------------------------------- */
#define IT_KV8_PAGE 64
#define IT_KV8_BLOCK 16

/* The buffers (16-byte aligned) and sizes of a layer's cache; the struct itself is host memory, read during the call.
 * Element of a page and KV head that holds (row, dim), in kp / vp (bytes) and tk / tv (f16) alike:
 *   K: (((row/16 * hd/64 + dim/64) * 64 + dim/8 % 4 * 16 + row % 16) * 16 + dim/32 % 2 * 8 + dim % 8
 *   V: (dim/16 * 64 + row/4 % 4 * 16 + dim % 16) * 16 + row/16 * 4 + row % 4 */
typedef struct {
    uint8_t *kp, *vp;     /* codes [npages][nkv][64*hd] */
    uint16_t* sc;         /* f16 scales [npages][nkv][8]: K's four blocks, then V's */
    uint16_t *tk, *tv;    /* open rows, f16 [nseq][2][nkv][64*hd], page p in half p % 2 */
    int npages, nseq, nkv, hd;   /* hd 128 or 256 */
} it_kv8_cache;

/* Appends f16 rows: token t is k[t*tok_stride + kh*hd + d] (tok_stride a multiple of 8, 16-byte aligned), as the pre-pass leaves it.
 * Sequences must not share a page that the call fills. */
int it_kv8_append(const it_kv8_cache* cache, const uint16_t* k, const uint16_t* v, int tok_stride, int ntok,
                  const int32_t* start, const int32_t* len, const int32_t* table, int max_pages, int max_nt,
                  void* stream);

/* Rows first[i] .. of each sequence, start[i+1] - start[i] of them (at most max_rows), as f16 into rows start[i] .. of k and
 * v; total[i]: the rows that the sequence holds, or fewer that it may be cut to (rows at or after total are not written). Where
 * first[i] or total[i] is negative, or total[i] more than the table can name, the sequence's rows start[i] .. are NaN. */
int it_kv8_read(const it_kv8_cache* cache, uint16_t* k, uint16_t* v, int tok_stride, int ntok, const int32_t* start,
                const int32_t* first, const int32_t* total, const int32_t* table, int max_pages, int max_rows,
                void* stream);

/* Copies pages src[i] to dst[i], i < n, and the open rows of sequences seq_src[i] to seq_dst[i], i < nseq, in one launch (either count
 * may be 0): for forks, and to make a pool dense (the caller renames the pages in its tables). All copies run at
 * once: destinations differ from each other and from every source. A number outside the cache is skipped. */
int it_kv8_copy(const it_kv8_cache* cache, const int32_t* src, const int32_t* dst, int n, const int32_t* seq_src,
                const int32_t* seq_dst, int nseq, void* stream);

/* Causal GQA attention with sigmoid gate over the cache, of tokens whose rows have been appended: token t of sequence i sees
 * its rows 0 .. len[i] + t. q as for it_attn_f16 (query | gate per head), out [t*out_tok_stride + h*hd + d] in f32, or f16 where
 * out_f16 is nonzero. One token a sequence, a few (drafts), or prompts of any lengths, mixed.
 * len[i] and its tokens together are the rows that the sequence holds, or fewer that it may be cut to: the rows after the last full
 * page that they make have to stand in the open buffer. (So after one long append, call it for all of its tokens.)
 * Accuracy: the softmax's sums and the products' sums are f32, K and V exact as stored. For an f32 output q goes into the products
 * in fixed point, to 2^-23 of its head's largest value (2^-22 of itself against the open rows), a probability as an f16 pair, to
 * 2^-22 of itself or, where it is small, 2^-31 of its row's largest up to there. An f16 output is that rounded where max_nt times the
 * query heads of a KV head is at most 16; of more rows it may go by q to 2^-15, a probability as one f16, to 2^-11 of itself: root
 * mean square up to 2.1e-4 of the result over many keys, beside the 2.1e-4 of the output's own rounding (an 8192-token prompt 2.7e-4
 * in all). A program that needs the f32 products there takes an f32 output.
 * At most 2^26 tokens times heads, 2^23 sequences times KV heads, 2^16 query heads of a KV head. Which sequences share a call
 * decides how the pages are split, so it moves results by roundings; the same call gives the same bits.
 * scratch: it_attn_kv8_scratch_bytes bytes, 16-byte aligned (one per call that may overlap another). */
size_t it_attn_kv8_scratch_bytes(int max_nt, int hd, int nh, int nkv);
int it_attn_kv8(const it_kv8_cache* cache, const float* q, int q_tok_stride, int ntok, const int32_t* start,
                const int32_t* len, const int32_t* table, int max_pages, int max_nt, int nh, float scale, void* out,
                int out_tok_stride, int out_f16, void* scratch, size_t scratch_bytes, void* stream);

/* ------------------------------------------------------------------------------------------------
 * Reference-shaped dispatch policy (pure host functions, no device access).
 * ---------------------------------------------------------------------------------------------- */

/* 64*heads*max(ctx,260) (src/vk/mod.rs:138): the arena's scratch words for a 64-token batch. An
 * arena for larger chunks holds it_attention_dispatch_room(ctx, heads, ubatch) words, as the
 * reference's scr slot does (src/vk/mod.rs:546). */
size_t it_attention_scratch_words(size_t ctx, size_t heads);
/* ceil(nt/64)*64*heads*max(ctx,260), nt in 1..=512 (src/vk/mod.rs:148-150); 0 if nt is invalid. */
size_t it_attention_dispatch_room(size_t ctx, size_t heads, size_t nt);
/* Keys per split the reference would choose: 64 doubled (at most to 1024) until
 * nt*nh*ceil((pos0+nt)/C)*260 <= room (src/vk/mod.rs:714-716); -1 if even 1024 does not fit. */
int it_attention_chunk(uint32_t nt, uint32_t nh, uint32_t pos0, size_t room);
/* The prompt split of src/vk/mod.rs:130-134 (prefill_chunks): consecutive ranges of at most `batch`
 * tokens (batch 64, 128, 256 or 512) covering 0..len, where a range longer than 64 whose length
 * leaves a tail of 1..21 tokens past a multiple of 64 gives that tail to the next range (no token
 * is dropped or repeated). Range i is starts[i] .. starts[i]+lens[i]. Writes at most cap ranges and
 * returns the number of ranges (which may exceed cap), or -1 if batch is not 64/128/256/512. */
long it_prefill_chunks(size_t len, size_t batch, size_t* starts, size_t* lens, size_t cap);
/* Geometry check of src/vk/mod.rs:207-220 restricted to the attention/GDN fields; 0 = supported. */
int it_validate_geometry(int ctx_len, int head_dim, int n_head, int n_head_kv, int ssm_state,
                         int ssm_groups, int ssm_vheads, int ssm_inner, int conv_k);

/* Measurement only, no counterpart in the reference: the device's sustained f16 matrix-core
 * rate. wgs workgroups of 256 threads; each of their waves issues 4 * iters independent
 * 32x32x16 f16 MFMAs (32768 flops each) and touches no memory besides one float per thread
 * written to out (wgs * 256 floats). Rate = wgs * 4 * 4 * iters * 32768 / elapsed time. */
int it_calib_mfma_f16(int wgs, int iters, float* out, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* IT_ATTN_H */

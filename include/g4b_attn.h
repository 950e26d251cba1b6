/*
 * g4b_attn.h -- C ABI of libg4b_attn.so: the attention hot path of the g4b inference engine
 * (flash attention over the per-slot ring KV cache, KV append, decode-state advance) as
 * hand-written HIP kernels for gfx950 (MI355X).
 *
 * Conventions
 *   - Every pointer is a device pointer owned by the caller; the library never allocates,
 *     frees or synchronises (the scratch of g4b_attn_forward_static_scratch is an array in the
 *     library's device image, not an allocation).  Work is enqueued on `stream` (a hipStream_t passed as void*;
 *     NULL = the default stream) and is legal inside stream capture.  One exception, once per GPU: the first
 *     decode-shaped attention launch (over pages: the first that splits its keys) or rope launch (or
 *     g4b_static_scratch_init) outside stream capture runs a 64-workgroup
 *     kernel that reports which XCD each workgroup ran on and waits for it on `stream`; the streaming kernels weight
 *     their work shares by the answer.  Launches captured before that keep equal shares.
 *   - Environment switches, read when the library is first used (counterparts of the reference's
 *     G4B_FA_FORCE_CONFIG / G4B_FA_PRINT_CONFIG, g4b/kernels/fa2.py:148-150,691-700): G4B_ATTN_NUM_WORKERS=n sets the
 *     default worker count of decode-shaped launches (and the size g4b_attn_workspace_bytes reports for it);
 *     G4B_ATTN_XCD_SHARES=0 forces equal work shares, =1 the weighted ones without asking the hardware;
 *     G4B_ATTN_PRINT_PLAN=1 prints one line per attention launch on stderr (kernel family, grid, workers, splits).
 *   - Strides are in ELEMENTS, as in the reference's launch adapter (g4b/kernels/utils.py:87-127).
 *   - Entry points return G4B_OK (0) or a negative g4b_status.  Arguments are validated on the
 *     host before anything is launched; g4b_last_error() returns a thread-local message for the
 *     last failure.
 *   - dtype codes: G4B_DT_F16, G4B_DT_BF16, G4B_DT_F32.
 */
#ifndef G4B_ATTN_H
#define G4B_ATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define G4B_ATTN_ABI_VERSION 5

enum g4b_status {
    G4B_OK = 0,
    G4B_ERR_INVALID_ARGUMENT = -1, /* shape / stride / dtype / value check failed (reference: tl.static_assert) */
    G4B_ERR_UNSUPPORTED = -2,      /* valid in the reference, not built here (e.g. head_dim above 1024, a mixed launch at head_dim 128) */
    G4B_ERR_WORKSPACE = -3,        /* workspace missing or too small for the requested split-KV launch */
    G4B_ERR_LAUNCH = -4,           /* the HIP runtime refused the launch (no device, bad stream, ...) */
    G4B_ERR_BUSY = -5              /* g4b_attn_forward_static_scratch: the array is in use by unfinished work on another stream */
};

enum g4b_dtype { G4B_DT_F16 = 0, G4B_DT_BF16 = 1, G4B_DT_F32 = 2 };

/* g4b/kernels/fa2.py:14-16 */
enum g4b_stage { G4B_STAGE_FULL = 1, G4B_STAGE_ON_BAND = 2, G4B_STAGE_CAUSAL = 3 };
/* g4b/kernels/fa2.py:29-31 */
enum g4b_phase { G4B_PHASE_UNALLOCATED = 0, G4B_PHASE_PREFILL = 1, G4B_PHASE_DECODE = 2 };

/*
 * g4b_attn_forward replaces flash_attention() = _attn_kernel + _reduce_split_kv_kernel
 * (g4b/kernels/fa2.py:634-715, 256-480, 546-631).
 *
 *   q, o          [B, H, Tq, D], any strides with last stride 1 (the engine passes permuted views
 *                 of [B, t, H, D] scratchpads, g4b/models/gemma4e.py:1031-1033); f16 / bf16 / f32.
 *   k_cache,      [B, G, KV_CTX, D], contiguous inside a slot (fa2.py:315-320), slot stride
 *   v_cache       k_stride_b / v_stride_b; f16 or bf16, or f32 (the reference's G4B_DTKV_FP32 debugging switch,
 *                 g4b/models/gemma4e.py:32).
 *   time_dim_sizes[B] int32: tokens in the slot after this step (fa2.py:52).
 *   user_phase    [B] uint8: slots whose value differs from `phase` are skipped and their rows of
 *                 `o` are left untouched (fa2.py:332-335).
 *   ctx_window_size  W <= KV_CTX: the launch sees the last min(tds, W) keys; logical key j is ring
 *                 row (max(tds - W, 0) + j) % KV_CTX; query i is aligned with logical key
 *                 min(tds, W) - Tq + i (fa2.py:53-56,75).
 *   stage         G4B_STAGE_CAUSAL (default of the reference), G4B_STAGE_FULL, or G4B_STAGE_ON_BAND: the diagonal
 *                 block alone (fa2.py:61,399-435), whose extent is the reference's autotuned Q_BLOCKSIZE_T and has to be
 *                 named here.
 *   on_band_block with G4B_STAGE_ON_BAND: Q_BLOCKSIZE_T (fa2.py:56,140-180; 1 in the reference's default configuration
 *                 list).  Query i then sees the keys of its own block of that many positions up to itself:
 *                 logical keys [q_t_base + (i / block) * block, q_t_base + i].  Ignored by the other stages.
 *   scale         softmax scale; the reference computes with 1.0 (fa2.py:89).
 *   query_window  0 = anchored window, the reference kernel's semantics.  > 0 additionally hides
 *                 keys with q_pos - k_pos >= query_window, the per-query sliding window of the CPU
 *                 reference's one-shot prefill (scripts/reference_impl.py:440-441).
 *   window_sizes  optional [B] int32 per-slot override of ctx_window_size (extension; NULL = none).
 *   workspace     device scratch for split-KV partials, >= g4b_attn_workspace_bytes(...) bytes, or
 *                 NULL: then a decode-shaped launch (R*Tq <= 16) uses one wave per (slot, kv head)
 *                 and a prefill-shaped launch one workgroup per (slot, kv head, query tile) however
 *                 few slots are in phase.  Contents are unspecified after the call (like
 *                 partial_o/l/m, fa2.py:643-645).  A decode-shaped launch with D <= 256,
 *                 ctx_window_size <= 512 and no window_sizes merges in LDS and never touches it.
 *   num_workers   0 = library default; otherwise the number of workers the decode key tiles are
 *                 dealt to (must not exceed the value the workspace was sized for).  A worker is one
 *                 wave, or a pair of waves when D = 512.  Ignored by
 *                 prefill-shaped launches, which choose their key split from the number of in-phase
 *                 slots on the device.
 *   use_fp32_dot  the reference's USE_FP32_DOT (fa2.py:85-88,126-129): 0 = the query is rounded to the cache's 16-bit
 *                 type before K Q^T, as the reference's `q.to(tl.float16)` does; non-zero = a query of a wider type
 *                 (f32 over any cache, f16 over a bf16 cache) enters K Q^T as the sum of two 16-bit operands, its
 *                 rounded value and its rounding error, so the scores are those of the unrounded query.  The engine
 *                 passes fp32 q with use_fp32_dot=True and scale 1.0 (g4b/models/gemma4e.py:30,606).  No effect when
 *                 q already has the cache's type.
 *   kernel_mask   profiling aid.  0 = run every kernel of the launch.  Otherwise bit 0 selects the
 *                 main attention kernel and bit 1 the split-merge kernel, so that each can be timed
 *                 on its own; results are only complete with both.
 *
 * The tuned kernels serve D in {128, 256, 512} with f16 / bf16 caches, the causal and full stages and, for
 * prefill-shaped launches ((H/G)*Tq > 16), H/G dividing 128 (64 at D = 512 with a split query): everything Gemma-4
 * and the reference's own test list (tests/compare_scripts/test_fa2.py:51-79) use.  Any other D that is a multiple of
 * 8 up to 1024, any other H/G, an f32 cache and G4B_STAGE_ON_BAND run on a plain fp32 kernel without matrix
 * instructions: same results to the same tolerance, a fraction of the speed, no workspace.
 *
 * Rows whose visible key set is empty (time_dim_sizes[b] == 0 on an in-phase slot) are written
 * as zeros; the reference leaves 0/0 there and its caller ignores them (g4b/scheduler.py:142-148).
 */
typedef struct g4b_attn_args {
    const void* q;
    const void* k_cache;
    const void* v_cache;
    void* o;
    const int32_t* time_dim_sizes;
    const uint8_t* user_phase;
    const int32_t* window_sizes;
    void* workspace;
    uint64_t workspace_bytes;
    int64_t q_stride[4];
    int64_t o_stride[4];
    int64_t k_stride_b;
    int64_t v_stride_b;
    int64_t time_dim_sizes_stride;
    int64_t user_phase_stride;
    int64_t window_sizes_stride;
    int32_t q_dtype;
    int32_t o_dtype;
    int32_t kv_dtype;
    int32_t B, H, G, Tq, D, KV_CTX;
    int32_t ctx_window_size;
    int32_t phase;
    int32_t stage;
    int32_t query_window;
    int32_t num_workers;
    int32_t kernel_mask;
    int32_t use_fp32_dot;
    int32_t on_band_block;
    float scale;
} g4b_attn_args;

int g4b_attn_forward(const g4b_attn_args* args, void* stream);

/* Bytes of workspace that let g4b_attn_forward split keys: for a decode-shaped launch (R*Tq <= 16)
 * over `num_workers` workers (0 = library default); for a prefill shape that brings fewer workgroups
 * per slot than the chip has compute units (chunked prefill, short prompts; sized by H, G, Tq, D
 * only) over several workgroups per query tile.  Returns 0 when the shape never uses a workspace.
 * Replaces the sizing of partial_o/l/m at g4b/models/gemma4e.py:43,819-821. */
uint64_t g4b_attn_workspace_bytes(int32_t B, int32_t H, int32_t G, int32_t Tq, int32_t D, int32_t num_workers);

/* The library default for num_workers on the current build (a multiple of the CU count) for D <= 256;
 * half of it for D = 512, whose workers are pairs of waves. */
int32_t g4b_attn_default_workers(void);

/*
 * g4b_attn_forward_mixed: one launch for a step that holds prefill-phase and decode-phase slots at once.  The
 * reference kernel skips per slot on user_phase[b] != PHASE (g4b/kernels/fa2.py:332-335), so such a step is two
 * flash_attention calls over the same batch tensors, one per phase, and its scheduler avoids the case altogether
 * (g4b/scheduler.py:66,96-98).  Here both calls are one grid: `prefill` is the argument block of the call whose query
 * block is a chunk ((H/G)*Tq > 16), `decode` the block of the call with one (or a few) query tokens per slot
 * ((H/G)*Tq <= 16); they must name the same caches, time_dim_sizes, user_phase, window_sizes, B, H, G, D, KV_CTX, cache
 * dtype and ctx_window_size and differ in q, o, Tq, strides and phase.  Results are those of the two calls.  The
 * workgroups of the two halves are dealt to different compute units, so the chunk's matrix work runs under the decode
 * stream's memory time.  Head dimensions 256 and 512.
 *   workspace     one buffer for both halves, passed in `prefill->workspace` (`decode->workspace` is ignored), at
 *                 least g4b_attn_mixed_workspace_bytes(...) bytes; NULL = neither half splits keys.
 *   num_workers   `decode->num_workers`: 0 = the library's share-out of the chip between the halves.
 */
int g4b_attn_forward_mixed(const g4b_attn_args* prefill, const g4b_attn_args* decode, void* stream);
uint64_t g4b_attn_mixed_workspace_bytes(int32_t B, int32_t H, int32_t G, int32_t Tq_prefill, int32_t Tq_decode, int32_t D,
                                        int32_t KV_CTX, int32_t ctx_window_size, int32_t has_window_sizes, int32_t num_workers);

/*
 * g4b_attn_forward_static_scratch: g4b_attn_forward for callers that cannot allocate.  It has no counterpart in the
 * reference; it is for code under HIP graph capture, tight serving loops and harnesses that forbid hipMalloc, which
 * have no place to get the split-KV workspace from.  Same arguments and results as g4b_attn_forward with a workspace
 * of g4b_attn_workspace_bytes(...) bytes, except that `workspace` must be NULL: the split partials go to an array of
 * G4B_ATTN_STATIC_SCRATCH_BYTES bytes that is part of the library's device image (one copy per GPU the library runs
 * on, held until the process ends).  The call itself allocates and frees nothing.  A launch whose partials need more
 * than that is refused with G4B_ERR_WORKSPACE (the limit covers every prefill shape up to head dimension 512 and
 * decode batches of about a thousand (slot, kv head) pairs at the default worker count).  No kernel reads scratch
 * that the same call has not written, so nothing is cleared between calls; all calls on one GPU share the array, so
 * calls that overlap on one GPU would race.  The library remembers, per GPU, the stream of the last call that used the
 * array: a call on another stream while that stream still has unfinished work is refused with G4B_ERR_BUSY (wait for
 * the first stream, or give one of the calls a workspace through g4b_attn_forward).  Calls recorded into a graph are
 * not tracked -- whoever replays graphs concurrently keeps their launches apart.
 *
 * g4b_static_scratch_init looks the array's device address up for the current device (the first
 * g4b_attn_forward_static_scratch on a device does the same); call it once per device at load when the first launch
 * would otherwise happen under stream capture.
 */
#define G4B_ATTN_STATIC_SCRATCH_BYTES (68u << 20)
int g4b_attn_forward_static_scratch(const g4b_attn_args* args, void* stream);
int g4b_static_scratch_init(void);
uint64_t g4b_static_scratch_bytes(void);

/*
 * g4b_kv_append replaces add_kv_to_cache() (g4b/kernels/add_kv_to_cache.py:84-186):
 *   cache[b, g, (t + cache_offsets[b]) % T, :] = x[b, g, t, :] * (x_rsos ? rsqrt(x_rsos[b,g,t] / D + eps) : 1)
 * for slots with user_phase[b] == phase (all slots when user_phase is NULL).
 *   x [B,G,t,D] strided (last stride 1), f16/bf16/f32; cache [B,G,T,D] contiguous inside a slot,
 *   f16/bf16/f32; cache_offsets [B] int32 or int64; x_rsos [B,G,t] f32 strided or NULL; t <= T.
 */
typedef struct g4b_kv_append_args {
    const void* x;
    void* cache;
    const void* cache_offsets;
    const float* x_rsos;
    const uint8_t* user_phase;
    int64_t x_stride[4];
    int64_t x_rsos_stride[3];
    int64_t cache_stride_b;
    int64_t cache_offsets_stride;
    int64_t user_phase_stride;
    int32_t x_dtype;
    int32_t cache_dtype;
    int32_t cache_offsets_is_int64;
    int32_t B, G, t, T, D;
    int32_t phase;
    float rmsnorm_eps;
} g4b_kv_append_args;

int g4b_kv_append(const g4b_kv_append_args* args, void* stream);

/*
 * g4b_advance_decode_state replaces advance_decode_state()
 * (g4b/kernels/advance_decode_state.py:32-80): for slots with user_phase[b] == 2,
 *   input_token_ids[0, b] = out_token_ids[b, 0]; cache_offsets[b] += 1; time_dim_sizes[b] += 1.
 */
typedef struct g4b_advance_args {
    int32_t* input_token_ids;
    const int32_t* out_token_ids;
    int32_t* cache_offsets;
    int32_t* time_dim_sizes;
    const uint8_t* user_phase;
    int64_t input_token_ids_stride1;
    int64_t out_token_ids_stride0;
    int64_t cache_offsets_stride;
    int64_t time_dim_sizes_stride;
    int64_t user_phase_stride;
    int32_t B;
} g4b_advance_args;

int g4b_advance_decode_state(const g4b_advance_args* args, void* stream);

/*
 * g4b_rope replaces apply_rope() (g4b/kernels/rope.py:123-243): for x in (q, k), in place,
 *   x[b,h,t,:] <- rope(x[b,h,t,:] * rsqrt(x_rsos[b,h,t] / D + eps) * x_rmsnorm_w[:], theta[b,t,:])
 *   theta[b,t,j] = (time_dim_offsets[b] + t) * rope_freqs[j]  (fp32),  j < D/2
 *   rope(x)[j] = cos*x[j] - sin*x[j + D/2];   rope(x)[j + D/2] = cos*x[j + D/2] + sin*x[j]
 * on every slot (the reference's kernel has no phase skip).  With k_cache non-NULL the same launch also
 * does the two add_kv_to_cache() calls that follow it in the engine (g4b/models/gemma4e.py:575-590):
 *   k_cache[b, g, (t + time_dim_offsets[b]) % T, :] = rotated k[b,g,t,:]
 *   v_cache[b, g, (t + time_dim_offsets[b]) % T, :] = v[b,g,t,:] * (v_rsos ? rsqrt(v_rsos[b,g,t] / Dv + eps) : 1)
 * for slots with user_phase[b] == phase (all slots when user_phase is NULL); the rotated k is then written
 * back to k only if k_writeback != 0 (nothing in the engine reads it after the append).
 *   q [B,H,t,D], k [B,G,t,D], v [B,G,t,Dv]: strided, last stride 1, f16/bf16/f32; rope_freqs [D/2] f32;
 *   time_dim_offsets [B] int32; *_rsos [B,heads,t] f32 strided; *_rmsnorm_w [D] f32; caches [B,G,T,D(v)]
 *   contiguous inside a slot, f16/bf16/f32; D and Dv multiples of 16; t <= T.
 */
typedef struct g4b_rope_args {
    void* q;
    void* k;
    const float* rope_freqs;
    const int32_t* time_dim_offsets;
    const float* q_rsos;
    const float* k_rsos;
    const float* q_rmsnorm_w;
    const float* k_rmsnorm_w;
    const void* v;
    const float* v_rsos;
    void* k_cache;
    void* v_cache;
    const uint8_t* user_phase;
    int64_t q_stride[4];
    int64_t k_stride[4];
    int64_t v_stride[4];
    int64_t q_rsos_stride[3];
    int64_t k_rsos_stride[3];
    int64_t v_rsos_stride[3];
    int64_t rope_freqs_stride;
    int64_t q_rmsnorm_w_stride;
    int64_t k_rmsnorm_w_stride;
    int64_t time_dim_offsets_stride;
    int64_t user_phase_stride;
    int64_t k_cache_stride_b;
    int64_t v_cache_stride_b;
    int32_t q_dtype;
    int32_t k_dtype;
    int32_t v_dtype;
    int32_t cache_dtype;
    int32_t B, H, G, t, D, Dv, T;
    int32_t phase;
    int32_t k_writeback;
    float rmsnorm_eps;
} g4b_rope_args;

int g4b_rope(const g4b_rope_args* args, void* stream);

/*
 * g4b_rope_frequencies replaces populate_rope_frequencies() (g4b/kernels/rope.py:262-293), run once at load:
 *   out[j] = 1 / freq_base ** (j / n)  [/ freq_scalars[j]],  j < n;  out and freq_scalars are f32 device arrays.
 */
int g4b_rope_frequencies(float* out, const float* freq_scalars, int32_t n, int64_t out_stride,
                         int64_t freq_scalars_stride, float freq_base, void* stream);

/*
 * ---- packed prompts and a paged cache --------------------------------------------------------------------------
 * The reference keeps one ring of KV rows per slot.  The entry points below serve the other common layout of a server's
 * cache: prompts packed one after the other without padding, and K and V rows kept in pages of a pool that sequences
 * take from and return to.
 *
 *   pool          k_pages, v_pages: [P, G, page_size, D], contiguous inside a page, page stride k_page_stride /
 *                 v_page_stride; page_size a multiple of 16 (the last page of a sequence may be partly filled).
 *   block_tables  [S, M] int32, unit stride along a row: entry e of row s is the page that holds positions
 *                 [e * page_size, (e + 1) * page_size) of sequence s.  An entry outside [0, P) names no page: attention
 *                 does not see its positions, the append drops rows that would go there.  Entries past a sequence's
 *                 length are never read.
 *   seq_lens      [S] int32: positions of the sequence that hold a row, at most M * page_size (what is above counts as
 *                 that, what is negative as 0).
 */

/*
 * g4b_packed_attn: causal attention over packed prompts.  Sequence s owns rows [cu_seqlens[s], cu_seqlens[s + 1]) of
 * q, k, v and o; row t of it attends to its own rows j <= t, with query_window > 0 only to those with t - j < query_window:
 *   o[t, h, :] = sum_j softmax_j(scale * q[t, h, :] . k[j, h / (H/G), :]) v[j, h / (H/G), :]
 *   q, o [T, H, D] f16 / bf16 / f32, k, v [T, G, D] f16 / bf16 / f32: any strides that are multiples of 8 elements, last
 *   stride 1, 16-byte aligned bases.  cu_seqlens [N + 1] int32 in ascending order (values are clamped to [0, T]); rows of o
 *   outside every sequence are left as they are.  T = 0 or N = 0 is a call that does nothing.
 *   use_fp32_dot  as in g4b_attn_forward: a query wider than k's 16-bit type enters the first product unrounded, as the sum of
 *                 two 16-bit operands (exact to 2^-22 of its size in f16, 2^-16 in bf16).
 *   workspace     NULL, or at least g4b_packed_attn_workspace_bytes(...) bytes, 16-byte aligned, used by one launch at a
 *                 time: lets a launch with fewer query tiles than the chip has compute units split their keys.
 * Rows that are hidden (later ones, those in front of the window, other sequences') never enter a result, whatever they hold.
 * A score of minus infinity is a weight of zero; a row with no other score becomes zeros.
 * Limits: T * H below 2^31; in the tuned kernels token strides of k and v below 2^24 elements and, with tiles of t = 128 / (H/G)
 * tokens (64 / (H/G) at D = 512 with an unrounded query), (T / t + min(N, T)) * G below 2^24 - 16.
 * Tuned for D in {128, 256, 512} with f16 / bf16 k and v and H/G dividing 128 (64 at D = 512 with an unrounded query);
 * any other D that is a multiple of 8 up to 1024, other H/G and f32 k and v run on a plain fp32 kernel, which never rounds
 * the query.
 */
typedef struct g4b_packed_attn_args {
    const void* q;
    const void* k;
    const void* v;
    void* o;
    const int32_t* cu_seqlens;
    void* workspace;
    uint64_t workspace_bytes;
    int64_t q_stride[3];
    int64_t k_stride[3];
    int64_t v_stride[3];
    int64_t o_stride[3];
    int64_t cu_seqlens_stride;
    int32_t q_dtype;
    int32_t o_dtype;
    int32_t kv_dtype;
    int32_t T, N, H, G, D;
    int32_t query_window;
    int32_t use_fp32_dot;
    float scale;
} g4b_packed_attn_args;

int g4b_packed_attn(const g4b_packed_attn_args* args, void* stream);
uint64_t g4b_packed_attn_workspace_bytes(int32_t T, int32_t N, int32_t H, int32_t G, int32_t D);

/*
 * g4b_paged_attn: attention of one new token per sequence over a paged cache.  The query of sequence b stands at position
 * seq_lens[b] - 1 (its own K and V rows are in the cache already) and sees the last min(seq_lens[b], window_size) positions,
 * all of them with window_size = 0.
 *   q, o [B, H, D] f16 / bf16 / f32, strides multiples of 8 elements, last stride 1.  Sequences with
 *   user_phase[b] != phase are skipped and their rows of o left untouched (user_phase NULL: none is); a sequence that
 *   sees no key (length 0, or only absent pages), or none with a score above minus infinity, gets zeros.
 *   workspace     NULL (one wave per (sequence, kv head)), or at least g4b_paged_attn_workspace_bytes(...) bytes, 16-byte
 *                 aligned, used by one launch at a time: the keys of all sequences are then split over num_workers waves
 *                 (0 = the library's default) and a second kernel joins the partial results.
 * Rows that are hidden (in front of the window, behind the length, on an absent page) never enter a result, whatever they hold.
 * A value that is seen and not finite makes the result not finite (an infinity may come out as NaN).
 * Limits: B <= 65535; B * G * ceil(M * page_size / 32) below 2^31; one kv head of a page below 2 GiB; in the tuned kernels B * G
 * below 2^23 (more where the launch stays below 2^32 threads).
 * Tuned for D in {128, 256, 512} with f16 / bf16 pools and H/G <= 16; any other D that is a multiple of 8 up to 1024,
 * larger H/G and f32 pools run on a plain fp32 kernel, which never rounds the query.
 */
typedef struct g4b_paged_attn_args {
    const void* q;
    const void* k_pages;
    const void* v_pages;
    void* o;
    const int32_t* block_tables;
    const int32_t* seq_lens;
    const uint8_t* user_phase;
    void* workspace;
    uint64_t workspace_bytes;
    int64_t q_stride[3];
    int64_t o_stride[3];
    int64_t k_page_stride;
    int64_t v_page_stride;
    int64_t block_tables_stride;
    int64_t seq_lens_stride;
    int64_t user_phase_stride;
    int32_t q_dtype;
    int32_t o_dtype;
    int32_t kv_dtype;
    int32_t B, H, G, D;
    int32_t num_pages, page_size, max_pages;
    int32_t window_size;
    int32_t phase;
    int32_t num_workers;
    int32_t use_fp32_dot;
    float scale;
} g4b_paged_attn_args;

int g4b_paged_attn(const g4b_paged_attn_args* args, void* stream);
uint64_t g4b_paged_attn_workspace_bytes(int32_t B, int32_t H, int32_t G, int32_t D, int32_t num_workers);

/*
 * g4b_paged_append: the paged counterpart of g4b_kv_append, K and V in one launch.  Row i of sequence s goes to position
 * cache_offsets[s] + i:
 *   pool[block_tables[s, pos / page_size], g, pos % page_size, :] = x[row, g, :] * (rsos ? rsqrt(rsos[row, g] / D + eps) : 1)
 * Sequence s owns rows [cu_seqlens[s], cu_seqlens[s + 1]) of k and v (values clamped to [0, T]), or, with cu_seqlens NULL,
 * the one row s (then T = N).  Rows whose position is negative, past the table or on an absent page are dropped, and so
 * are those of sequences with user_phase[s] != phase.  k, v [T, G, D] f16 / bf16 / f32, strides multiples of 8 elements, last
 * stride 1; pools f16 / bf16 / f32; k_rsos, v_rsos [T, G] f32 or NULL.  G * D below 2^24.
 */
typedef struct g4b_paged_append_args {
    const void* k;
    const void* v;
    void* k_pages;
    void* v_pages;
    const int32_t* block_tables;
    const int32_t* cache_offsets;
    const int32_t* cu_seqlens;
    const float* k_rsos;
    const float* v_rsos;
    const uint8_t* user_phase;
    int64_t k_stride[3];
    int64_t v_stride[3];
    int64_t k_rsos_stride[2];
    int64_t v_rsos_stride[2];
    int64_t k_page_stride;
    int64_t v_page_stride;
    int64_t block_tables_stride;
    int64_t cache_offsets_stride;
    int64_t cu_seqlens_stride;
    int64_t user_phase_stride;
    int32_t k_dtype;
    int32_t v_dtype;
    int32_t cache_dtype;
    int32_t T, N, G, D;
    int32_t num_pages, page_size, max_pages;
    int32_t phase;
    float rmsnorm_eps;
} g4b_paged_append_args;

int g4b_paged_append(const g4b_paged_append_args* args, void* stream);

/*
 * Page management.  ref_counts [P] int32 (how many table entries, or other holders, a page has) is the only state of the
 * allocator: a page is free while its count is 0, and whoever needs pages gets the lowest-numbered free ones, so results do
 * not depend on timing.  seq_lens, ref_counts, src, dst, num_new, page_map and status are contiguous, block_tables has
 * unit stride along its rows.  Pools: [layers, P, ...] with `page_elems` contiguous elements per page of each pool; every
 * layer follows the same tables.  Nothing here waits for the device: what can only be seen there ends up in status [1].
 *
 * g4b_pages_copy       pool[:, dst[i]] = pool[:, src[i]] for i < n (n <= G4B_PAGES_MAX_LIST).  A pair is dropped, and
 *                      counted by adding 1 to status[0], when one of its pages is outside [0, P), when an earlier pair
 *                      names the same destination, or when its destination is the source of any pair of the list: every
 *                      source is thus read as it was before the call.  A pair of a page with itself moves nothing, and
 *                      counts for nothing in the judgement of others.
 * g4b_pages_free       sequences src[0..n) give up their pages: counts are decremented (not below 0), the held table
 *                      entries become -1, seq_lens 0.  Entries outside [0, S) and repeated ones do nothing.
 * g4b_pages_fork       sequence dst[i] becomes a copy of src[i] for i < n: full pages are shared (count + 1), a partly filled
 *                      last page is copied to a free page of its own.  Sources are read as they were before the call.
 *                      status[0] = 0, or the number of free pages that were missing, or -1 when an index is outside
 *                      [0, S), a destination is named twice or is not empty (seq_lens[dst] != 0), or a source is longer
 *                      than the table; unless it is 0 nothing has changed.
 * g4b_pages_allocate   every sequence s < S grows by num_new[s] positions and gets the pages for them.  status[0] = 0, or the
 *                      number of free pages that were missing, or -1 when a num_new is negative or a sequence would outgrow
 *                      its table; unless it is 0 nothing has changed.
 * g4b_pages_compact    the pages in use move to the front of the pool: with n pages in use, those at or above n move, in
 *                      ascending order, into the free ones below n, also in ascending order.  Tables, counts and both
 *                      pools follow; page_map[p] = new index of page p, -1 if it was free; status[0] = n.
 *
 * workspace: at least g4b_pages_workspace_bytes(P, S) bytes, 16-byte aligned, used by one call at a time (fork, allocate,
 * compact); contents unspecified before and after.
 */
#define G4B_PAGES_MAX_LIST 8192
typedef struct g4b_pages_args {
    void* k_pages;
    void* v_pages;
    int32_t* block_tables;
    int32_t* seq_lens;
    int32_t* ref_counts;
    const int32_t* src;
    const int32_t* dst;
    const int32_t* num_new;
    int32_t* page_map;
    int32_t* status;
    void* workspace;
    uint64_t workspace_bytes;
    int64_t k_layer_stride;
    int64_t v_layer_stride;
    int64_t k_page_stride;
    int64_t v_page_stride;
    int64_t page_elems;
    int64_t block_tables_stride;
    int32_t cache_dtype;
    int32_t layers, num_pages, page_size;
    int32_t S, max_pages, n;
} g4b_pages_args;

int g4b_pages_copy(const g4b_pages_args* args, void* stream);
int g4b_pages_free(const g4b_pages_args* args, void* stream);
int g4b_pages_fork(const g4b_pages_args* args, void* stream);
int g4b_pages_allocate(const g4b_pages_args* args, void* stream);
int g4b_pages_compact(const g4b_pages_args* args, void* stream);
uint64_t g4b_pages_workspace_bytes(int32_t num_pages, int32_t S);

/*
 * Profiling aid, no counterpart in the reference.  Between g4b_profile_begin() and g4b_profile_end() every
 * g4b_attn_forward, g4b_rope, g4b_packed_attn and g4b_paged_attn call of the calling thread has its dominant kernel (the streaming worker, the prefill
 * kernel, the rope kernel) dispatched with a pair of events that the runtime stamps with the begin and the end of that
 * dispatch: the kernel's own duration, as a kernel trace reports it, without the launch gaps an event pair recorded
 * around the call would include.  g4b_profile_end waits for the timed kernels, writes up to `capacity` durations in
 * milliseconds in call order (-1 for a call whose dominant kernel was masked out) and returns the number of timed
 * calls, or a negative g4b_status.  Events are created per call, so this is not for graph capture.
 */
int g4b_profile_begin(void);
int g4b_profile_end(float* ms, int32_t capacity);

/* Message of the calling thread's last failed call ("" if none). */
const char* g4b_last_error(void);

/* G4B_ATTN_ABI_VERSION the library was built with. */
int32_t g4b_abi_version(void);

#ifdef __cplusplus
}
#endif
#endif /* G4B_ATTN_H */

// C ABI of the operators over packed prompts and a paged cache: argument validation on the host, then dispatch to the
// gfx950 kernels.  Nothing here allocates, synchronises or reads device memory, but for the question that the first split decode
// launch of a device asks outside stream capture (xcd_parity, api.hip).
#include <cmath>
#include <cstdio>

#include "api_common.hpp"
#include "packed_map.hpp"
#include "paged.hpp"

using namespace g4b::api;

namespace {

constexpr int kMaxGroup = 16;  // query heads per kv head that the streaming kernels take

// q, k, v, o of the attention calls: 16-byte vector access along D
int check_strides(const char* what, const int64_t* s, int n) {
    if (s[n - 1] != 1) return fail(G4B_ERR_INVALID_ARGUMENT, "%s must have unit stride in the head dimension", what);
    for (int i = 0; i < n - 1; ++i)
        if (s[i] < 0 || s[i] % 8) return fail(G4B_ERR_INVALID_ARGUMENT, "%s strides must be non-negative multiples of 8 elements", what);
    return G4B_OK;
}

int check_heads(int H, int G, int D) {
    if (H < 1 || G < 1 || D < 1) return fail(G4B_ERR_INVALID_ARGUMENT, "H, G and D must be positive");
    if (H % G) return fail(G4B_ERR_INVALID_ARGUMENT, "H (%d) must be a multiple of G (%d)", H, G);
    if (D % 8 || D > 1024) return fail(G4B_ERR_UNSUPPORTED, "head_dim must be a multiple of 8 and at most 1024 (got %d)", D);
    if (G > 65535) return fail(G4B_ERR_UNSUPPORTED, "G must be <= 65535");
    return G4B_OK;
}

int check_scale(float scale) {
    if (!std::isfinite(scale) || !(scale > 0.f)) return fail(G4B_ERR_INVALID_ARGUMENT, "scale must be finite and positive");
    return G4B_OK;
}

// The pool and table of a paged call.
int check_pool(int num_pages, int page_size, int max_pages, int64_t page_elems, int64_t k_stride, int64_t v_stride, const void* k,
               const void* v) {
    if (num_pages < 1 || max_pages < 1) return fail(G4B_ERR_INVALID_ARGUMENT, "the pool and the block tables must hold at least one page");
    if (page_size < g4b::PAGE_UNIT || page_size % g4b::PAGE_UNIT)
        return fail(G4B_ERR_UNSUPPORTED, "page_size must be a positive multiple of %d (got %d)", g4b::PAGE_UNIT, page_size);
    if ((int64_t)max_pages * page_size > (int64_t)0x7fffff00)
        return fail(G4B_ERR_UNSUPPORTED, "a block table must name fewer than 2^31 positions");
    if (k_stride < page_elems || v_stride < page_elems || k_stride % 8 || v_stride % 8)
        return fail(G4B_ERR_INVALID_ARGUMENT, "the page stride must be at least a page and a multiple of 8 elements");
    if (!aligned16(k) || !aligned16(v)) return fail(G4B_ERR_INVALID_ARGUMENT, "k_pages and v_pages must be 16-byte aligned");
    return G4B_OK;
}

// a query wider than the cache type: f32 over f16 / bf16, f16 over bf16
bool wider_query(int q_dtype, int kv_dtype) {
    return (q_dtype == G4B_DT_F32 && kv_dtype != G4B_DT_F32) || (q_dtype == G4B_DT_F16 && kv_dtype == G4B_DT_BF16);
}

}  // namespace

extern "C" {

uint64_t g4b_packed_attn_workspace_bytes(int32_t T, int32_t N, int32_t H, int32_t G, int32_t D) {
    if (T < 1 || N < 1 || H < 1 || G < 1 || H % G || (D != 128 && D != 256 && D != 512)) return 0;
    // (a query that stays unrounded takes smaller tiles or fewer slots, a window fewer keys: never more than this)
    const int tokb = g4b::packed_tokb(D, H / G, false);
    return tokb > 0 && g4b::packed_may_cut(T, G, D, tokb, g4b::packed_slots(D, false), 0) ? g4b::packed_partial_bytes(D) : 0;
}

int g4b_packed_attn(const g4b_packed_attn_args* a, void* stream) {
    if (!a) return fail(G4B_ERR_INVALID_ARGUMENT, "args is NULL");
    if (a->T < 0 || a->N < 0) return fail(G4B_ERR_INVALID_ARGUMENT, "T and N must not be negative");
    if (const int rc = check_heads(a->H, a->G, a->D)) return rc;
    if (!dtype_ok(a->q_dtype) || !dtype_ok(a->o_dtype) || !dtype_ok(a->kv_dtype))
        return fail(G4B_ERR_INVALID_ARGUMENT, "q, o, k and v must be f16, bf16 or f32");
    if (const int rc = check_strides("q", a->q_stride, 3)) return rc;
    if (const int rc = check_strides("k", a->k_stride, 3)) return rc;
    if (const int rc = check_strides("v", a->v_stride, 3)) return rc;
    if (const int rc = check_strides("o", a->o_stride, 3)) return rc;
    if (a->query_window < 0) return fail(G4B_ERR_INVALID_ARGUMENT, "query_window must be >= 0");
    if (const int rc = check_scale(a->scale)) return rc;
    if (a->T == 0 || a->N == 0) return G4B_OK;
    if (!a->q || !a->k || !a->v || !a->o || !a->cu_seqlens) return fail(G4B_ERR_INVALID_ARGUMENT, "q, k, v, o and cu_seqlens must be non-NULL");
    if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->o))
        return fail(G4B_ERR_INVALID_ARGUMENT, "q, k, v and o must be 16-byte aligned");
    if ((int64_t)a->T * a->H > 0x7fffffffLL) return fail(G4B_ERR_UNSUPPORTED, "T * H must be below 2^31");

    g4b::PackedParams p{};
    p.q = a->q;
    p.k = a->k;
    p.v = a->v;
    p.o = a->o;
    p.cu = a->cu_seqlens;
    p.cu_s = a->cu_seqlens_stride;
    p.q_s[1] = a->q_stride[1], p.q_s[2] = a->q_stride[0], p.q_s[3] = 1;
    p.o_s[1] = a->o_stride[1], p.o_s[2] = a->o_stride[0], p.o_s[3] = 1;
    p.k_ts = a->k_stride[0], p.k_hs = a->k_stride[1];
    p.v_ts = a->v_stride[0], p.v_hs = a->v_stride[1];
    p.q_dt = a->q_dtype, p.o_dt = a->o_dtype;
    p.B = a->N, p.H = a->H, p.G = a->G, p.R = a->H / a->G, p.Tq = p.T = a->T;
    p.stage = g4b::STAGE_CAUSAL;
    p.qwin = a->query_window;
    p.kernel_mask = 3;
    p.xcd_shift = -1;
    p.c = a->scale * 1.44269504088896340736f;
    p.q_split = (a->use_fp32_dot && wider_query(a->q_dtype, a->kv_dtype)) ? 1 : 0;
    const bool tuned_dim = a->kv_dtype != G4B_DT_F32 && (a->D == 128 || a->D == 256 || a->D == 512);
    const int tokb = tuned_dim ? g4b::packed_tokb(a->D, p.R, p.q_split != 0) : 0;
    if (tokb > 0 && ((p.k_ts | p.v_ts) >> 24) != 0) return fail(G4B_ERR_UNSUPPORTED, "the token strides of k and v must be below 2^24 elements");
    if (tokb > 0 && g4b::packed_grid(a->T, a->N, a->G, tokb, g4b::packed_slots(a->D, p.q_split != 0), true) > g4b::MAX_BLOCKS)
        return fail(G4B_ERR_UNSUPPORTED, "(T / %d + min(N, T)) * G must stay below 2^24 - 16", tokb);
    const uint64_t need = g4b_packed_attn_workspace_bytes(a->T, a->N, a->H, a->G, a->D);
    if (a->workspace && tokb > 0 && need) {
        if (a->workspace_bytes < need)
            return fail(G4B_ERR_WORKSPACE, "workspace holds %llu bytes, %llu needed", (unsigned long long)a->workspace_bytes, (unsigned long long)need);
        if (!aligned16(a->workspace)) return fail(G4B_ERR_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
        if (g4b::packed_may_cut(a->T, a->G, a->D, tokb, g4b::packed_slots(a->D, p.q_split != 0), a->query_window)) {
            p.part_o = static_cast<float*>(a->workspace);
            p.part_ml = p.part_o + (uint64_t)g4b::packed_slots(a->D, p.q_split != 0) * g4b::PACKED_ROWS * a->D;
        }
    }
    if (print_plan())
        fprintf(stderr, "g4b_attn plan: packed T=%d N=%d H=%d G=%d D=%d window %d: %s%s\n", a->T, a->N, a->H, a->G, a->D, a->query_window,
                tokb > 0 ? "matrix-core kernel" : "plain fp32 kernel", p.part_o ? ", may cut its keys into spans" : "");
    if (!arm_profile()) return fail(G4B_ERR_LAUNCH, "could not create profiling events");
    const hipError_t e = tokb > 0 ? g4b::launch_packed_prefill(p, a->D, a->kv_dtype, static_cast<hipStream_t>(stream))
                                  : g4b::launch_packed_generic(p, a->D, a->kv_dtype, static_cast<hipStream_t>(stream));
    disarm_profile();
    if (e != hipSuccess) return fail(G4B_ERR_LAUNCH, "packed attention launch failed: %s", hipGetErrorString(e));
    return G4B_OK;
}

uint64_t g4b_paged_attn_workspace_bytes(int32_t B, int32_t H, int32_t G, int32_t D, int32_t num_workers) {
    if (B < 1 || H < 1 || G < 1 || H % G || H / G > kMaxGroup) return 0;
    return g4b_attn_workspace_bytes(B, H, G, 1, D, num_workers);
}

int g4b_paged_attn(const g4b_paged_attn_args* a, void* stream) {
    if (!a) return fail(G4B_ERR_INVALID_ARGUMENT, "args is NULL");
    if (a->B < 0 || a->B > 65535) return fail(a->B < 0 ? G4B_ERR_INVALID_ARGUMENT : G4B_ERR_UNSUPPORTED, "B must be in [0, 65535]");
    if (const int rc = check_heads(a->H, a->G, a->D)) return rc;
    if (!dtype_ok(a->q_dtype) || !dtype_ok(a->o_dtype) || !dtype_ok(a->kv_dtype))
        return fail(G4B_ERR_INVALID_ARGUMENT, "q, o and the pools must be f16, bf16 or f32");
    if (const int rc = check_strides("q", a->q_stride, 3)) return rc;
    if (const int rc = check_strides("o", a->o_stride, 3)) return rc;
    if (const int rc = check_pool(a->num_pages, a->page_size, a->max_pages, (int64_t)a->G * a->page_size * a->D, a->k_page_stride,
                                  a->v_page_stride, a->k_pages, a->v_pages)) return rc;
    if ((int64_t)a->page_size * a->D * dtype_bytes(a->kv_dtype) >= (int64_t)1 << 31)
        return fail(G4B_ERR_UNSUPPORTED, "one kv head of a page must stay below 2 GiB");
    if (a->window_size < 0) return fail(G4B_ERR_INVALID_ARGUMENT, "window_size must be >= 0");
    if (a->phase < 0 || a->phase > 255) return fail(G4B_ERR_INVALID_ARGUMENT, "phase must fit uint8");
    if (a->num_workers < 0 || a->num_workers > (1 << 20)) return fail(G4B_ERR_INVALID_ARGUMENT, "num_workers out of range");
    if (const int rc = check_scale(a->scale)) return rc;
    if (a->B == 0) return G4B_OK;
    if (!a->q || !a->k_pages || !a->v_pages || !a->o || !a->block_tables || !a->seq_lens)
        return fail(G4B_ERR_INVALID_ARGUMENT, "q, k_pages, v_pages, o, block_tables and seq_lens must be non-NULL");
    if (!aligned16(a->q) || !aligned16(a->o)) return fail(G4B_ERR_INVALID_ARGUMENT, "q and o must be 16-byte aligned");
    // the streaming kernels count the 32-key tiles of all (sequence, kv head) pairs in 32 bits
    if ((int64_t)a->B * a->G * (((int64_t)a->max_pages * a->page_size + 31) / 32 + 1) >= (int64_t)1 << 31)
        return fail(G4B_ERR_UNSUPPORTED, "B * G * ceil(max_pages * page_size / 32) must stay below 2^31");

    g4b::PagedParams p{};
    p.q = a->q;
    p.k = a->k_pages;
    p.v = a->v_pages;
    p.o = a->o;
    p.tds = a->seq_lens;
    p.tds_s = a->seq_lens_stride;
    p.phase_arr = a->user_phase;
    p.ph_s = a->user_phase_stride;
    p.q_s[0] = a->q_stride[0], p.q_s[1] = a->q_stride[1], p.q_s[3] = 1;
    p.o_s[0] = a->o_stride[0], p.o_s[1] = a->o_stride[1], p.o_s[3] = 1;
    p.q_dt = a->q_dtype, p.o_dt = a->o_dtype;
    p.B = a->B, p.H = a->H, p.G = a->G, p.R = a->H / a->G, p.Tq = 1;
    p.W = p.KV_CTX = a->max_pages * a->page_size;
    p.phase = a->phase;
    p.stage = g4b::STAGE_CAUSAL;
    p.qwin = a->window_size;
    p.kernel_mask = 3;
    p.xcd_shift = -1;
    p.c = a->scale * 1.44269504088896340736f;
    p.q_split = (a->use_fp32_dot && wider_query(a->q_dtype, a->kv_dtype)) ? 1 : 0;
    p.table = a->block_tables;
    p.table_s = a->block_tables_stride;
    p.k_ps = a->k_page_stride, p.v_ps = a->v_page_stride;
    p.page_size = a->page_size, p.page_units = a->page_size / g4b::PAGE_UNIT;
    p.num_pages = a->num_pages, p.max_pages = a->max_pages;
    if ((int64_t)a->B * a->H > 0x7fffffffLL) return fail(G4B_ERR_UNSUPPORTED, "B * H must be below 2^31");
    const bool tuned = a->kv_dtype != G4B_DT_F32 && (a->D == 128 || a->D == 256 || a->D == 512) && p.R <= kMaxGroup;
    const uint64_t need = g4b_paged_attn_workspace_bytes(a->B, a->H, a->G, a->D, a->num_workers);
    if (a->workspace && tuned && need) {
        if (a->workspace_bytes < need)
            return fail(G4B_ERR_WORKSPACE, "workspace holds %llu bytes, %llu needed", (unsigned long long)a->workspace_bytes, (unsigned long long)need);
        if (!aligned16(a->workspace)) return fail(G4B_ERR_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
        p.NW = a->num_workers > 0 ? a->num_workers : default_decode_workers(a->D);
        p.part_o = static_cast<float*>(a->workspace);
        p.part_ml = p.part_o + decode_slots(a->B, a->G, p.NW) * (uint64_t)p.R * (uint64_t)a->D;
    }
    if (tuned && !g4b::paged_grid_fits(p, a->D)) return fail(G4B_ERR_UNSUPPORTED, "B * G is %lld: the launch would have 2^32 threads or more", (long long)a->B * a->G);
    // (only the flat tile list has shares to weight)
    if (p.NW > 0 && !g4b::paged_pair_path(p, a->D) && xcd_parity(static_cast<hipStream_t>(stream))) p.xcd_shift = 0;
    if (print_plan())
        fprintf(stderr, "g4b_attn plan: paged decode B=%d H=%d G=%d D=%d page %d window %d: %s, %d workers\n", a->B, a->H, a->G, a->D,
                a->page_size, a->window_size,
                !tuned ? "plain fp32 kernel" : g4b::paged_pair_path(p, a->D) ? "one kernel, a workgroup per (sequence, kv head)" : "flat tile list",
                p.NW);
    if (!arm_profile()) return fail(G4B_ERR_LAUNCH, "could not create profiling events");
    const hipError_t e = tuned ? g4b::launch_paged_decode(p, a->D, a->kv_dtype, static_cast<hipStream_t>(stream))
                               : g4b::launch_paged_generic(p, a->D, a->kv_dtype, static_cast<hipStream_t>(stream));
    disarm_profile();
    if (e != hipSuccess) return fail(G4B_ERR_LAUNCH, "paged attention launch failed: %s", hipGetErrorString(e));
    return G4B_OK;
}

int g4b_paged_append(const g4b_paged_append_args* a, void* stream) {
    if (!a) return fail(G4B_ERR_INVALID_ARGUMENT, "args is NULL");
    if (a->T < 0 || a->N < 0) return fail(G4B_ERR_INVALID_ARGUMENT, "T and N must not be negative");
    if (a->G < 1 || a->D < 1) return fail(G4B_ERR_INVALID_ARGUMENT, "G and D must be positive");
    if (a->D % 8) return fail(G4B_ERR_UNSUPPORTED, "D must be a multiple of 8");
    if ((int64_t)a->G * a->D >= (int64_t)1 << 24) return fail(G4B_ERR_UNSUPPORTED, "G * D must be below 2^24");
    if (!dtype_ok(a->k_dtype) || !dtype_ok(a->v_dtype) || !dtype_ok(a->cache_dtype))
        return fail(G4B_ERR_INVALID_ARGUMENT, "k, v and the pools must be f16, bf16 or f32");
    if (const int rc = check_strides("k", a->k_stride, 3)) return rc;
    if (const int rc = check_strides("v", a->v_stride, 3)) return rc;
    if (const int rc = check_pool(a->num_pages, a->page_size, a->max_pages, (int64_t)a->G * a->page_size * a->D, a->k_page_stride,
                                  a->v_page_stride, a->k_pages, a->v_pages)) return rc;
    if (a->phase < 0 || a->phase > 255) return fail(G4B_ERR_INVALID_ARGUMENT, "phase must fit uint8");
    if (!std::isfinite(a->rmsnorm_eps)) return fail(G4B_ERR_INVALID_ARGUMENT, "rmsnorm_eps must be finite");
    if (!a->cu_seqlens && a->T != a->N) return fail(G4B_ERR_INVALID_ARGUMENT, "without cu_seqlens every sequence brings one row: T (%d) must be N (%d)", a->T, a->N);
    if (a->T == 0 || a->N == 0) return G4B_OK;
    if (!a->k || !a->v || !a->k_pages || !a->v_pages || !a->block_tables || !a->cache_offsets)
        return fail(G4B_ERR_INVALID_ARGUMENT, "k, v, k_pages, v_pages, block_tables and cache_offsets must be non-NULL");
    if (!aligned16(a->k) || !aligned16(a->v)) return fail(G4B_ERR_INVALID_ARGUMENT, "k and v must be 16-byte aligned");

    g4b::PagedAppendParams p{};
    p.k = a->k, p.v = a->v, p.k_pages = a->k_pages, p.v_pages = a->v_pages;
    p.table = a->block_tables;
    p.offsets = a->cache_offsets;
    p.cu = a->cu_seqlens;
    p.k_rsos = a->k_rsos, p.v_rsos = a->v_rsos;
    p.phase_arr = a->user_phase;
    for (int i = 0; i < 2; ++i) {
        p.k_s[i] = a->k_stride[i], p.v_s[i] = a->v_stride[i];
        p.k_rsos_s[i] = a->k_rsos_stride[i], p.v_rsos_s[i] = a->v_rsos_stride[i];
    }
    p.k_ps = a->k_page_stride, p.v_ps = a->v_page_stride;
    p.table_s = a->block_tables_stride, p.off_s = a->cache_offsets_stride, p.cu_s = a->cu_seqlens_stride, p.ph_s = a->user_phase_stride;
    p.k_dt = a->k_dtype, p.v_dt = a->v_dtype, p.cache_dt = a->cache_dtype;
    p.T = a->T, p.N = a->N, p.G = a->G, p.D = a->D;
    p.num_pages = a->num_pages, p.page_size = a->page_size, p.max_pages = a->max_pages, p.phase = a->phase;
    p.eps = a->rmsnorm_eps;
    const hipError_t e = g4b::launch_paged_append(p, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(G4B_ERR_LAUNCH, "paged append launch failed: %s", hipGetErrorString(e));
    return G4B_OK;
}

// ---- page management -----------------------------------------------------------------------------------------------

uint64_t g4b_pages_workspace_bytes(int32_t num_pages, int32_t S) {
    if (num_pages < 1 || S < 1) return 0;
    return (uint64_t)g4b::pages_workspace_words(num_pages, S) * sizeof(int32_t);
}

enum : int { NEEDS_POOLS = 1, NEEDS_TABLES = 2, NEEDS_WORKSPACE = 4, NEEDS_STATUS = 8 };

static int fill_pages_params(const g4b_pages_args* a, int needs, g4b::PagesParams& p) {
    if (!a) return fail(G4B_ERR_INVALID_ARGUMENT, "args is NULL");
    p = g4b::PagesParams{};
    if (a->num_pages < 1 || a->num_pages > (1 << 27)) return fail(G4B_ERR_INVALID_ARGUMENT, "num_pages must be in [1, 2^27]");
    if (a->n < 0 || a->n > G4B_PAGES_MAX_LIST) return fail(G4B_ERR_INVALID_ARGUMENT, "a list holds at most %d entries (got %d)", G4B_PAGES_MAX_LIST, a->n);
    if (needs & NEEDS_POOLS) {
        if (!a->k_pages || !a->v_pages) return fail(G4B_ERR_INVALID_ARGUMENT, "k_pages and v_pages must be non-NULL");
        if (!dtype_ok(a->cache_dtype)) return fail(G4B_ERR_INVALID_ARGUMENT, "the pools must be f16, bf16 or f32");
        if (a->layers < 1 || a->page_elems < 1) return fail(G4B_ERR_INVALID_ARGUMENT, "layers and page_elems must be positive");
        const int64_t esz = dtype_bytes(a->cache_dtype);
        const int64_t ks[4] = {a->k_page_stride, a->v_page_stride, a->k_layer_stride, a->v_layer_stride};
        for (int i = 0; i < 4; ++i)
            if (ks[i] < 0 || ks[i] >= (int64_t)1 << 60 || ks[i] * esz % 16) return fail(G4B_ERR_INVALID_ARGUMENT, "page and layer strides must be non-negative multiples of 16 bytes");
        if (a->page_elems > (int64_t)1 << 31) return fail(G4B_ERR_UNSUPPORTED, "a page must stay below 2 GiB");
        if (a->page_elems * esz % 16 || !aligned16(a->k_pages) || !aligned16(a->v_pages))
            return fail(G4B_ERR_INVALID_ARGUMENT, "pages must be multiples of 16 bytes and 16-byte aligned");
        if (a->k_page_stride < a->page_elems || a->v_page_stride < a->page_elems)
            return fail(G4B_ERR_INVALID_ARGUMENT, "the page stride must be at least a page");
        if (a->page_elems * esz > (int64_t)1 << 31) return fail(G4B_ERR_UNSUPPORTED, "a page must stay below 2 GiB");
        p.k = static_cast<char*>(a->k_pages), p.v = static_cast<char*>(a->v_pages);
        p.k_ps = a->k_page_stride * esz, p.v_ps = a->v_page_stride * esz;
        p.k_ls = a->k_layer_stride * esz, p.v_ls = a->v_layer_stride * esz;
        p.page_bytes = a->page_elems * esz;
        p.layers = a->layers;
    }
    if (needs & NEEDS_TABLES) {
        if (!a->block_tables || !a->seq_lens || !a->ref_counts) return fail(G4B_ERR_INVALID_ARGUMENT, "block_tables, seq_lens and ref_counts must be non-NULL");
        if (!aligned16(a->ref_counts)) return fail(G4B_ERR_INVALID_ARGUMENT, "ref_counts must be 16-byte aligned");
        if (a->S < 1 || a->S > (1 << 18)) return fail(G4B_ERR_INVALID_ARGUMENT, "the number of sequences must be in [1, 2^18]");
        if (a->max_pages < 1 || a->max_pages > (1 << 20)) return fail(G4B_ERR_INVALID_ARGUMENT, "a block table holds 1 to 2^20 pages");
        if (a->page_size < 1 || (int64_t)a->max_pages * a->page_size > (int64_t)0x7fffff00)
            return fail(G4B_ERR_INVALID_ARGUMENT, "page_size must be positive and a block table must name fewer than 2^31 positions");
        if (a->block_tables_stride < a->max_pages) return fail(G4B_ERR_INVALID_ARGUMENT, "the rows of block_tables overlap");
    }
    if ((needs & NEEDS_STATUS) && !a->status) return fail(G4B_ERR_INVALID_ARGUMENT, "status must be non-NULL");
    if (needs & NEEDS_WORKSPACE) {
        const uint64_t need = g4b_pages_workspace_bytes(a->num_pages, a->S);
        if (!a->workspace || a->workspace_bytes < need)
            return fail(G4B_ERR_WORKSPACE, "workspace holds %llu bytes, %llu needed", (unsigned long long)(a->workspace ? a->workspace_bytes : 0), (unsigned long long)need);
        if (!aligned16(a->workspace)) return fail(G4B_ERR_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
    }
    p.table = a->block_tables, p.lens = a->seq_lens, p.refs = a->ref_counts;
    p.src = a->src, p.dst = a->dst, p.num_new = a->num_new, p.page_map = a->page_map, p.status = a->status;
    p.ws = static_cast<int32_t*>(a->workspace);
    p.table_s = a->block_tables_stride;
    p.P = a->num_pages, p.page_size = a->page_size, p.S = a->S, p.max_pages = a->max_pages, p.n = a->n;
    return G4B_OK;
}

static int pages_result(const char* what, hipError_t e) {
    return e == hipSuccess ? G4B_OK : fail(G4B_ERR_LAUNCH, "%s launch failed: %s", what, hipGetErrorString(e));
}

int g4b_pages_copy(const g4b_pages_args* a, void* stream) {
    g4b::PagesParams p;
    if (const int rc = fill_pages_params(a, NEEDS_POOLS | NEEDS_STATUS, p)) return rc;
    if (p.n == 0) return G4B_OK;
    if (!p.src || !p.dst) return fail(G4B_ERR_INVALID_ARGUMENT, "src and dst must be non-NULL");
    return pages_result("page copy", g4b::launch_pages_copy(p, static_cast<hipStream_t>(stream)));
}

int g4b_pages_free(const g4b_pages_args* a, void* stream) {
    g4b::PagesParams p;
    if (const int rc = fill_pages_params(a, NEEDS_TABLES, p)) return rc;
    if (p.n == 0) return G4B_OK;
    if (!p.src) return fail(G4B_ERR_INVALID_ARGUMENT, "the list of sequences must be non-NULL");
    return pages_result("page free", g4b::launch_pages_free(p, static_cast<hipStream_t>(stream)));
}

int g4b_pages_fork(const g4b_pages_args* a, void* stream) {
    g4b::PagesParams p;
    if (const int rc = fill_pages_params(a, NEEDS_POOLS | NEEDS_TABLES | NEEDS_WORKSPACE | NEEDS_STATUS, p)) return rc;
    if (p.n > p.S) return fail(G4B_ERR_INVALID_ARGUMENT, "%d forks into %d sequences: a destination would repeat", p.n, p.S);
    if (p.n > 0 && (!p.src || !p.dst)) return fail(G4B_ERR_INVALID_ARGUMENT, "src and dst must be non-NULL");
    return pages_result("fork", g4b::launch_pages_fork(p, static_cast<hipStream_t>(stream)));
}

int g4b_pages_allocate(const g4b_pages_args* a, void* stream) {
    g4b::PagesParams p;
    if (const int rc = fill_pages_params(a, NEEDS_TABLES | NEEDS_WORKSPACE | NEEDS_STATUS, p)) return rc;
    if (!p.num_new) return fail(G4B_ERR_INVALID_ARGUMENT, "num_new must be non-NULL");
    return pages_result("page allocation", g4b::launch_pages_allocate(p, static_cast<hipStream_t>(stream)));
}

int g4b_pages_compact(const g4b_pages_args* a, void* stream) {
    g4b::PagesParams p;
    if (const int rc = fill_pages_params(a, NEEDS_POOLS | NEEDS_TABLES | NEEDS_WORKSPACE | NEEDS_STATUS, p)) return rc;
    if (!p.page_map) return fail(G4B_ERR_INVALID_ARGUMENT, "page_map must be non-NULL");
    return pages_result("compaction", g4b::launch_pages_compact(p, static_cast<hipStream_t>(stream)));
}

}  // extern "C"

// Launch parameters of the operators over packed prompts and a paged cache, and the host-side launchers.
#pragma once
#include "common.hpp"
#include "launch.hpp"

namespace g4b {

constexpr int64_t MAX_BLOCKS = (1 << 24) - 1;  // workgroups of 256 along one dimension of a grid: 2^32 threads are too many
// More of them (fewer than 2^31) are laid out over two dimensions; the last ones of the last row may have nothing to do.
inline dim3 grid_of(int64_t blocks) {
    constexpr unsigned ROW = 1u << 20;
    return blocks <= MAX_BLOCKS ? dim3((unsigned)blocks) : dim3(ROW, (unsigned)((blocks + ROW - 1) / ROW));
}
G4B_DEV int block_of_grid() { return (int)(blockIdx.y * gridDim.x + blockIdx.x); }
constexpr int PAGE_UNIT = 16;  // page sizes are multiples of this many positions

// Decode over pages: AttnParams with tds = seq_lens, Tq = 1, W and KV_CTX = the positions a table can name, qwin = the window;
// q_s / o_s: batch, head, unused, 1.  phase_arr may be NULL.
struct PagedParams : AttnParams {
    const int32_t* table;  // [B, max_pages]
    int64_t table_s;
    int64_t k_ps, v_ps;    // page strides of the pools (elements)
    int32_t page_size, page_units, num_pages, max_pages;
};

template <>
inline constexpr bool is_paged<PagedParams> = true;

// What a launch reads of one sequence.  The key tiles of the decode kernels lie on multiples of 32 positions, so klo is the
// first tile's first position; row_range() gives the first visible one.
G4B_DEV SlotInfo slot_info(const PagedParams& p, int b) {
    SlotInfo s;
    s.active = !p.phase_arr || p.phase_arr[(int64_t)b * p.ph_s] == (uint8_t)p.phase;
    const int len = min(max(p.tds[(int64_t)b * p.tds_s], 0), p.W);
    s.window = s.active ? len : 0;
    s.ring_start = 0;
    s.qb = s.window - 1;
    s.klo = (p.qwin > 0 ? max(0, s.window - p.qwin) : 0) & ~31;
    return s;
}

// Causal attention over packed prompts: AttnParams with B = sequences, Tq = T (the rows of the buffers); q_s / o_s: unused,
// head, token, 1.
struct PackedParams : AttnParams {
    const int32_t* cu;
    int64_t cu_s;
    int64_t k_ts, k_hs, v_ts, v_hs;  // token and head strides of k and v (elements)
    int32_t T;
};

template <>
inline constexpr bool is_packed<PackedParams> = true;

// Rows [first, end) of sequence s, inside the buffers whatever cu holds.
G4B_DEV void packed_rows(const PackedParams& p, int s, int& first, int& end) {
    first = min(max(p.cu[(int64_t)s * p.cu_s], 0), p.T);
    end = min(max(p.cu[(int64_t)(s + 1) * p.cu_s], first), p.T);
}

// The sequence that row t belongs to: the last s with cu[s] <= t (rows of empty sequences belong to none, so several equal
// starts resolve to the one that is not empty), or -1.
G4B_DEV int packed_owner(const int32_t* cu, int64_t cu_s, int n, int t) {
    int lo = 0, hi = n;  // cu[lo] <= t < cu[hi] is searched for
    if (n < 1 || cu[0] > t || cu[(int64_t)n * cu_s] <= t) return -1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (cu[(int64_t)mid * cu_s] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

struct PagedAppendParams {
    const void *k, *v;
    void *k_pages, *v_pages;
    const int32_t* table;
    const int32_t* offsets;
    const int32_t* cu;         // optional
    const float *k_rsos, *v_rsos;  // optional
    const uint8_t* phase_arr;  // optional
    int64_t k_s[2], v_s[2];    // token, head
    int64_t k_rsos_s[2], v_rsos_s[2];
    int64_t k_ps, v_ps, table_s, off_s, cu_s, ph_s;
    int32_t k_dt, v_dt, cache_dt;
    int32_t T, N, G, D, num_pages, page_size, max_pages, phase;
    float eps;
};

struct PagesParams {
    char *k, *v;
    int32_t *table, *lens, *refs;
    const int32_t *src, *dst, *num_new;
    int32_t *page_map, *status, *ws;
    int64_t k_ls, v_ls, k_ps, v_ps;  // layer and page strides of the pools (bytes)
    int64_t page_bytes, table_s;
    int32_t layers, P, page_size, S, max_pages, n;
};

// any D that is a multiple of 8 up to 1024, any H/G, any dtype: plain fp32 kernels
hipError_t launch_packed_generic(const PackedParams& p, int D, int kv_dt, hipStream_t stream);
hipError_t launch_paged_generic(const PagedParams& p, int D, int kv_dt, hipStream_t stream);

// D in {128, 256, 512}, kv_dt in {DT_F16, DT_BF16}, packed_tokb(...) > 0: the matrix-core kernels over packed prompts
hipError_t launch_packed_prefill(const PackedParams& p, int D, int kv_dt, hipStream_t stream);
// Tokens of a query tile, 0 for groups that the matrix-core kernels are not built for.  A query that stays unrounded takes
// half of the rows at D = 512.
inline int packed_tokb(int D, int R, bool q_split) {
    const int rows = (D == 512 && q_split) ? 64 : 128;
    return R >= 1 && rows % R == 0 ? rows / R : 0;
}

// D in {128, 256, 512}, H/G <= 16, kv_dt in {DT_F16, DT_BF16}: the streaming kernels over pages
hipError_t launch_paged_decode(const PagedParams& p, int D, int kv_dt, hipStream_t stream);
// The one-kernel variant (a workgroup per (sequence, kv head), merged through LDS) when no sequence can show more than
// DEC_PAIR_MAX_KEYS keys.  A workgroup reads some 38 GB/s however few there are, so at head dimension 256 few pairs with long
// windows take the flat tile list, which brings a worker per tile.  Pair against list, windows of 200 and 512 keys: 8 pairs
// 7.2 / 9.7 and 14.6 / 9.9 us, 32 pairs 8.9 / 10.3 and 18.4 / 12.6, 128 pairs 10.6 / 16.3 and 20.8 / 24.3; at head dimension
// 128 the pair is ahead throughout (32 pairs, 512 keys: 10.3 / 10.6).
inline bool paged_pair_path(const PagedParams& p, int D) {
    const int keys = p.qwin > 0 && p.qwin < p.W ? p.qwin : p.W;
    if (D > 256 || keys > DEC_PAIR_MAX_KEYS) return false;
    return !(D == 256 && p.NW > 0 && (int64_t)p.B * p.G <= 64 && keys > 256);
}
constexpr int paged_pair_waves(int D) { return D == 128 ? 8 : 4; }
// Whether the grids of launch_paged_decode, which have a workgroup per (sequence, kv head), stay below 2^32 threads.
inline bool paged_grid_fits(const PagedParams& p, int D) {
    const int threads = paged_pair_path(p, D) ? 64 * paged_pair_waves(D) : p.NW > 0 ? 256 : D > 256 ? 128 : 64;
    return (int64_t)p.B * p.G * threads < (int64_t)1 << 32;
}

hipError_t launch_paged_append(const PagedAppendParams& p, hipStream_t stream);

hipError_t launch_pages_copy(const PagesParams& p, hipStream_t stream);
hipError_t launch_pages_free(const PagesParams& p, hipStream_t stream);
hipError_t launch_pages_fork(const PagesParams& p, hipStream_t stream);
hipError_t launch_pages_allocate(const PagesParams& p, hipStream_t stream);
hipError_t launch_pages_compact(const PagesParams& p, hipStream_t stream);
// int32 words of workspace that a call of pages_{fork,allocate,compact} may use
inline int64_t pages_workspace_words(int64_t P, int64_t S) { return P + 2 * S + P / 4096 + 32; }

}  // namespace g4b

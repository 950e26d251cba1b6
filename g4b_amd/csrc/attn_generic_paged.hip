// Attention over packed prompts and over a paged cache for the shapes and types the tuned kernels are not built for: any
// head dimension that is a multiple of 8 (up to 1024), any number of query heads per kv head, fp32 keys and values.  Every
// query row is one range of keys, served by the body of attn_generic.hpp.  Right for every case, not tuned.
#include "attn_generic.hpp"
#include "paged.hpp"

namespace g4b {

namespace {
struct PackedRows {
    static constexpr bool may_be_absent = false, may_be_dark = true, rounds_query = false;
    const char *kb, *vb;
    int64_t k_pitch, v_pitch;
    G4B_DEV const void* k(int j) const { return kb + j * k_pitch; }
    G4B_DEV const void* v(int j) const { return vb + j * v_pitch; }
};
struct PagedRows {
    static constexpr bool may_be_absent = true, may_be_dark = true, rounds_query = false;
    const char *kb, *vb;
    const int32_t* table;
    int64_t k_pitch, v_pitch;  // bytes from page to page
    int page_size, num_pages, row_bytes;
    G4B_DEV const void* at(const char* base, int64_t pitch, int j) const {
        const int page = table[j / page_size];
        if ((uint32_t)page >= (uint32_t)num_pages) return nullptr;
        return base + page * pitch + (int64_t)(j % page_size) * row_bytes;
    }
    G4B_DEV const void* k(int j) const { return at(kb, k_pitch, j); }
    G4B_DEV const void* v(int j) const { return at(vb, v_pitch, j); }
};
}  // namespace

template <int NQ>
__global__ __launch_bounds__(64 * GEN_WAVES) void attn_generic_packed_kernel(const PackedParams p, const int D, const int kv_dt) {
    __shared__ GenericSmem<NQ> sm;
    // workgroup (t * G + g) * (R / NQ) + head group: the heads of one kv head and one position are neighbours
    const int ngrp = p.R / NQ;
    int idx = block_of_grid();
    const int h_in = (idx % ngrp) * NQ;
    idx /= ngrp;
    const int g = idx % p.G, t = idx / p.G;
    if (t >= p.T) return;
    const int s = packed_owner(p.cu, p.cu_s, p.B, t);
    if (s < 0) return;  // the row belongs to no sequence: o stays as it is
    int first, end;
    packed_rows(p, s, first, end);
    if (t < first || t >= end) return;
    const int esz = kv_dt == DT_F32 ? 4 : 2;
    const PackedRows rows{static_cast<const char*>(p.k) + g * p.k_hs * esz, static_cast<const char*>(p.v) + g * p.v_hs * esz,
                          p.k_ts * esz, p.v_ts * esz};
    const int h0 = g * p.R + h_in;
    const GenericIo io{p.q, p.o, (int64_t)t * p.q_s[2] + h0 * p.q_s[1], p.q_s[1],
                       (int64_t)t * p.o_s[2] + h0 * p.o_s[1], p.o_s[1], p.q_dt, p.o_dt, p.c};
    generic_rows<NQ>(sm, rows, io, p.qwin > 0 ? max(first, t - p.qwin + 1) : first, t + 1, D, kv_dt);
}

template <int NQ>
__global__ __launch_bounds__(64 * GEN_WAVES) void attn_generic_paged_kernel(const PagedParams p, const int D, const int kv_dt) {
    __shared__ GenericSmem<NQ> sm;
    const int ngrp = p.R / NQ;
    int idx = block_of_grid();
    const int h_in = (idx % ngrp) * NQ;
    idx /= ngrp;
    const int g = idx % p.G, b = idx / p.G;
    if (b >= p.B) return;
    const SlotInfo si = slot_info(p, b);
    if (!si.active) return;
    const int esz = kv_dt == DT_F32 ? 4 : 2;
    const int64_t head = (int64_t)g * p.page_size * D * esz;
    const PagedRows rows{static_cast<const char*>(p.k) + head, static_cast<const char*>(p.v) + head, p.table + (int64_t)b * p.table_s,
                         p.k_ps * esz, p.v_ps * esz, p.page_size, p.num_pages, D * esz};
    const int h0 = g * p.R + h_in;
    const GenericIo io{p.q, p.o, (int64_t)b * p.q_s[0] + h0 * p.q_s[1], p.q_s[1],
                       (int64_t)b * p.o_s[0] + h0 * p.o_s[1], p.o_s[1], p.q_dt, p.o_dt, p.c};
    int lo, hi;
    row_range(p, si, 0, lo, hi);
    generic_rows<NQ>(sm, rows, io, lo, max(hi, lo), D, kv_dt);
}

// query heads per workgroup: as many as share the K/V loads, unless that leaves the chip short of workgroups
static int heads_per_workgroup(int R, int64_t rows_of_a_head) {
    int nq = R % 4 == 0 ? 4 : (R % 2 == 0 ? 2 : 1);
    while (nq > 1 && rows_of_a_head * (R / nq) < 1024) nq /= 2;
    return nq;
}

hipError_t launch_packed_generic(const PackedParams& p, int D, int kv_dt, hipStream_t stream) {
    const int nq = heads_per_workgroup(p.R, (int64_t)p.T * p.G);
    const int64_t blocks = (int64_t)p.T * (p.H / nq);
    if (D < 8 || D % 8 || D > GEN_MAX_D || blocks < 1 || blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    const dim3 grid = grid_of(blocks), block(64 * GEN_WAVES);
    if (nq == 4) G4B_LAUNCH_DOMINANT(attn_generic_packed_kernel<4>, grid, block, 0, stream, p, D, kv_dt);
    else if (nq == 2) G4B_LAUNCH_DOMINANT(attn_generic_packed_kernel<2>, grid, block, 0, stream, p, D, kv_dt);
    else G4B_LAUNCH_DOMINANT(attn_generic_packed_kernel<1>, grid, block, 0, stream, p, D, kv_dt);
    return hipGetLastError();
}

hipError_t launch_paged_generic(const PagedParams& p, int D, int kv_dt, hipStream_t stream) {
    const int nq = heads_per_workgroup(p.R, (int64_t)p.B * p.G);
    const int64_t blocks = (int64_t)p.B * (p.H / nq);
    if (D < 8 || D % 8 || D > GEN_MAX_D || blocks < 1 || blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    const dim3 grid = grid_of(blocks), block(64 * GEN_WAVES);
    if (nq == 4) G4B_LAUNCH_DOMINANT(attn_generic_paged_kernel<4>, grid, block, 0, stream, p, D, kv_dt);
    else if (nq == 2) G4B_LAUNCH_DOMINANT(attn_generic_paged_kernel<2>, grid, block, 0, stream, p, D, kv_dt);
    else G4B_LAUNCH_DOMINANT(attn_generic_paged_kernel<1>, grid, block, 0, stream, p, D, kv_dt);
    return hipGetLastError();
}

}  // namespace g4b

// Attention for the shapes and types the tuned kernels are not built for: any head dimension that is a multiple of 8
// (up to 1024), any number of query heads per kv head, an fp32 KV cache (the reference's G4B_DTKV_FP32 switch,
// g4b/models/gemma4e.py:32), and STAGE_ON_BAND on its own (g4b/kernels/fa2.py:15,399-435).  Same window / ring / phase
// semantics as the tuned kernels (g4b/kernels/fa2.py:52-96,332-335), evaluated per query row as one key range.
//
// One workgroup of four waves serves up to four query heads of one kv head at one (slot, query position) with the body of
// attn_generic.hpp.  The path is correct and reasonably parallel, not tuned: Gemma-4's shapes never reach it.
#include "attn_generic.hpp"
#include "launch.hpp"

namespace g4b {

namespace {
struct RingRows {
    static constexpr bool may_be_absent = false, may_be_dark = false, rounds_query = false;
    const char *kb, *vb;
    int ring_start, kv_ctx, row_bytes;
    G4B_DEV int64_t off(int j) const {
        int row = ring_start + j;
        if (row >= kv_ctx) row -= kv_ctx;
        return (int64_t)row * row_bytes;
    }
    G4B_DEV const void* k(int j) const { return kb + off(j); }
    G4B_DEV const void* v(int j) const { return vb + off(j); }
};
}  // namespace

// NQ query heads of one kv head at one query position per workgroup: they see the same keys, so every K and V row is
// loaded once for all of them.
template <int NQ>
__global__ __launch_bounds__(64 * GEN_WAVES) void attn_generic_kernel(const AttnParams p, const int D, const int kv_dt,
                                                                       const int band) {
    __shared__ GenericSmem<NQ> sm;
    // blockIdx.x = ((b * G + g) * Tq + i) * (R / NQ) + head group: the heads of one kv head and one position are neighbours
    const int ngrp = p.R / NQ;
    int idx = blockIdx.x;
    const int r0 = (idx % ngrp) * NQ;
    idx /= ngrp;
    const int i = idx % p.Tq;
    idx /= p.Tq;
    const int g = idx % p.G;
    const int b = idx / p.G;
    const int h0 = g * p.R + r0;

    if (p.phase_arr[(int64_t)b * p.ph_s] != (uint8_t)p.phase) return;  // o stays as it is (fa2.py:332-335)
    int tds = max(p.tds[(int64_t)b * p.tds_s], 0);
    int W = p.win_arr ? p.win_arr[(int64_t)b * p.win_s] : p.W;
    W = min(max(W, 0), p.KV_CTX);
    const int window = min(tds, W);
    const int ring_start = (tds - window) % p.KV_CTX;
    const int qb = window - p.Tq;  // logical key aligned with query 0 (fa2.py:55)
    const int qp = qb + i;
    int lo = 0, hi = window;
    if (p.stage != STAGE_FULL) hi = min(window, qp + 1);
    if (p.stage == STAGE_ON_BAND) lo = max(0, qb + (i / band) * band);  // the diagonal block of the row's tile (fa2.py:56,61)
    if (p.qwin > 0) lo = max(lo, qp - p.qwin + 1);
    hi = max(hi, lo);

    const int esz = kv_dt == DT_F32 ? 4 : 2;
    const RingRows rows{static_cast<const char*>(p.k) + ((int64_t)b * p.k_sb + (int64_t)g * p.KV_CTX * D) * esz,
                        static_cast<const char*>(p.v) + ((int64_t)b * p.v_sb + (int64_t)g * p.KV_CTX * D) * esz,
                        ring_start, p.KV_CTX, D * esz};
    const GenericIo io{p.q, p.o,
                       (int64_t)b * p.q_s[0] + (int64_t)h0 * p.q_s[1] + (int64_t)i * p.q_s[2], p.q_s[1],
                       (int64_t)b * p.o_s[0] + (int64_t)h0 * p.o_s[1] + (int64_t)i * p.o_s[2], p.o_s[1],
                       p.q_dt, p.o_dt, p.c};
    generic_rows<NQ>(sm, rows, io, lo, hi, D, kv_dt);
}

hipError_t launch_attn_generic(const AttnParams& p, int D, int kv_dt, int on_band_block, hipStream_t stream) {
    if (D < 8 || D % 8 || D > GEN_MAX_D) return hipErrorInvalidValue;
    // query heads per workgroup: as many as share the K/V loads, unless that leaves the chip short of workgroups
    // (decode-shaped launches: 64 slots x 8 heads measured 0.30 ms one head per workgroup, 0.34 ms four)
    int nq = p.R % 4 == 0 ? 4 : (p.R % 2 == 0 ? 2 : 1);
    while (nq > 1 && (int64_t)p.B * (p.H / nq) * p.Tq < 1024) nq /= 2;
    const int64_t blocks = (int64_t)p.B * (p.H / nq) * p.Tq;
    if (blocks < 1 || blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    if (!(p.kernel_mask & 1)) return hipSuccess;
    const dim3 grid((unsigned)blocks), block(64 * GEN_WAVES);
    const int band = on_band_block > 0 ? on_band_block : 1;
    if (nq == 4) G4B_LAUNCH_DOMINANT(attn_generic_kernel<4>, grid, block, 0, stream, p, D, kv_dt, band);
    else if (nq == 2) G4B_LAUNCH_DOMINANT(attn_generic_kernel<2>, grid, block, 0, stream, p, D, kv_dt, band);
    else G4B_LAUNCH_DOMINANT(attn_generic_kernel<1>, grid, block, 0, stream, p, D, kv_dt, band);
    return hipGetLastError();
}

}  // namespace g4b

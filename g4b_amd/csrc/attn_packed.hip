// Launchers of attention over packed prompts: the prefill kernels with rows of the packed buffers (packed_map.hpp deals the
// items out), and the kernel that joins the key spans of a launch that was cut into them.
#include "attn_prefill.hpp"
#include "attn_prefill_wide.hpp"
#include "launch.hpp"
#include "packed_map.hpp"

namespace g4b {

constexpr int packed_rows_of(int D, bool q_split) { return D == 512 && q_split ? 64 : 128; }

// At head dimension 128 with a 16-bit query two workgroups fit a compute unit, so that one's staging and softmax run under the
// other's matrix products (24 ragged prompts: 264 -> 198 us).
template <int D, class T, bool QS>
__global__ __launch_bounds__(256, packed_slots(D, QS) / 256) void attn_packed_kernel(const PackedParams p) {
    extern __shared__ __align__(16) char smem[];
    __shared__ int sh_scan[8];
    const PackedItem it = packed_item<D, packed_slots(D, QS), 256>(p, blockIdx.x, packed_rows_of(D, QS) / p.R, sh_scan);
    if (!it.valid) return;
    if constexpr (D == 512) prefill_wide_body<T, QS>(p, blockIdx.x, smem, sh_scan, it);
    else prefill_body<D, T, QS>(p, blockIdx.x, smem, sh_scan, it);
}

// Joins the spans of a launch that was cut: the workgroups (slot, y) of span k of a tile's c spans take the k-th of c parts of
// the tile's rows.  A row is D / 8 lanes of eight columns.  The kernel is all latency: the rows and sums of eight spans are in
// flight before the first is used, and the rows of a slot are spread over JOIN_Y workgroups so that each of them loads once
// or twice (one workgroup per slot: 11 us for a prompt of 512 tokens cut in two to four, a memory round trip per eight rows).
constexpr int JOIN_Y = 8;
template <int D, class T, bool QS>
__global__ __launch_bounds__(256) void attn_packed_combine(const PackedParams p) {
    constexpr int ROWS = packed_rows_of(D, QS);
    const PackedSlot it = packed_slot_info(p, packed_slots(D, QS))[blockIdx.x];
    if (it.spans < 2) return;
    const int tokb = ROWS / p.R;
    const int tok0 = it.qtile * tokb;
    const int slot0 = (int)blockIdx.x - it.span * p.G;  // (the spans of a tile are one after the other, the kv head runs fastest)
    constexpr int LPR = D / 8;        // lanes per row
    constexpr int RPP = 256 / LPR;    // rows per pass
    constexpr int UN = 8;             // spans in flight
    const int d0 = ((int)threadIdx.x % LPR) * 8;
    const int parts = it.spans * JOIN_Y, part = it.span * JOIN_Y + (int)blockIdx.y;
    const int row_end = ROWS * (part + 1) / parts;
    for (int row = ROWS * part / parts + (int)threadIdx.x / LPR; row < row_end; row += RPP) {
        const int tok = tok0 + row % tokb, h = it.g * p.R + row / tokb;
        if (tok >= it.len) continue;
        float ref = -INFINITY, l = 0.f;
        float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (int k0 = 0; k0 < it.spans; k0 += UN) {
            f4 x[UN][2];
            float ms[UN], ls[UN];
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const int k = min(k0 + u, it.spans - 1);  // clamped loads, masked below
                const int64_t prow = (int64_t)(slot0 + k * p.G) * PACKED_ROWS + row;
                ms[u] = p.part_ml[prow * 2];
                ls[u] = k0 + u < it.spans ? p.part_ml[prow * 2 + 1] : 0.f;  // 0: the span holds no key of the row
                x[u][0] = *reinterpret_cast<const f4*>(p.part_o + prow * D + d0);
                x[u][1] = *reinterpret_cast<const f4*>(p.part_o + prow * D + d0 + 4);
            }
            float m_new = ref;
#pragma unroll
            for (int u = 0; u < UN; ++u) m_new = is_zero(ls[u]) ? m_new : fmaxf(m_new, ms[u]);
            if (m_new == -INFINITY) continue;
            const float keep = fast_exp2(ref - m_new);  // 0 while ref is -inf
            ref = m_new;
            l *= keep;
#pragma unroll
            for (int i = 0; i < 8; ++i) acc[i] *= keep;
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const float w = is_zero(ls[u]) ? 0.f : ls[u] * fast_exp2(ms[u] - m_new);
                l += w;
#pragma unroll
                for (int i = 0; i < 8; ++i) acc[i] += (is_zero(ls[u]) ? 0.f : x[u][i / 4][i % 4]) * w;
            }
        }
        const float inv = is_zero(l) ? 0.f : 1.f / l;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] *= inv;
        store8(p.o, (int64_t)(it.first + tok) * p.o_s[2] + (int64_t)h * p.o_s[1] + d0, p.o_dt, acc);
    }
}

template <int D, class T, bool QS>
static hipError_t launch_packed_t(const PackedParams& p, hipStream_t stream) {
    constexpr int smem = D == 512 ? PW_SMEM : 4 * PfSmem<D == 512 ? 256 : D>::TILE;
    static uint64_t attr_done = 0;
    hipError_t e = allow_dynamic_smem(reinterpret_cast<const void*>(&attn_packed_kernel<D, T, QS>), smem, attr_done);
    if (e != hipSuccess) return e;
    const int64_t blocks = packed_grid(p.T, p.B, p.G, packed_tokb(D, p.R, QS), packed_slots(D, QS), p.part_o != nullptr);
    if (blocks > MAX_BLOCKS) return hipErrorInvalidValue;
    G4B_LAUNCH_DOMINANT((attn_packed_kernel<D, T, QS>), dim3((unsigned)blocks), dim3(256), smem, stream, p);
    e = hipGetLastError();
    if (e != hipSuccess || !p.part_o) return e;
    hipLaunchKernelGGL((attn_packed_combine<D, T, QS>), dim3(packed_slots(D, QS), JOIN_Y), dim3(256), 0, stream, p);
    return hipGetLastError();
}

template <int D>
static hipError_t launch_packed_d(const PackedParams& p, int kv_dt, hipStream_t stream) {
    if (kv_dt == DT_F16) return p.q_split ? launch_packed_t<D, F16, true>(p, stream) : launch_packed_t<D, F16, false>(p, stream);
    return p.q_split ? launch_packed_t<D, BF16, true>(p, stream) : launch_packed_t<D, BF16, false>(p, stream);
}

hipError_t launch_packed_prefill(const PackedParams& p, int D, int kv_dt, hipStream_t stream) {
    if (D == 512) return launch_packed_d<512>(p, kv_dt, stream);
    if (D == 256) return launch_packed_d<256>(p, kv_dt, stream);
    if (D == 128) return launch_packed_d<128>(p, kv_dt, stream);
    return hipErrorInvalidValue;
}

}  // namespace g4b

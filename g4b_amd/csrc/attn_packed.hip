// Launchers of attention over packed prompts: the prefill kernels with rows of the packed buffers (packed_map.hpp deals the
// items out), and the kernel that joins the key spans of a launch that was cut into them.
#include "attn_prefill.hpp"
#include "attn_prefill_wide.hpp"
#include "launch.hpp"
#include "packed_map.hpp"

namespace g4b {

template <int D, class T, bool QS>
__global__ __launch_bounds__(256) void attn_packed_kernel(const PackedParams p) {
    extern __shared__ __align__(16) char smem[];
    __shared__ int sh_scan[8];
    if constexpr (D == 512) prefill_wide_body<T, QS>(p, blockIdx.x, smem, sh_scan);
    else prefill_body<D, T, QS>(p, blockIdx.x, smem, sh_scan);
}

// Joins the spans of a launch that was cut: the workgroup of span k of a tile's c spans takes the k-th of c parts of the
// tile's rows.  A row is D / 8 lanes of eight columns; its spans' rows come in one after the other against a running
// reference (a tile has few spans, and the launch is bound by latency, not by these bytes).
template <int D, class T, int ROWS>
__global__ __launch_bounds__(256) void attn_packed_combine(const PackedParams p) {
    __shared__ int sh_scan[8];
    const int tokb = ROWS / p.R;
    const PackedItem it = packed_item<256>(p, blockIdx.x, tokb, sh_scan);
    if (!it.valid || it.spans < 2) return;
    // the slots of a tile's spans are one stride apart, as its spans are dealt out one after the other per kv head
    const int tok0 = it.qtile * tokb;
    const int slot0 = it.slot - it.span * p.G;
    constexpr int LPR = D / 8;        // lanes per row
    constexpr int RPP = 256 / LPR;    // rows per pass
    const int d0 = ((int)threadIdx.x % LPR) * 8;
    const int row_end = ROWS * (it.span + 1) / it.spans;
    for (int row = ROWS * it.span / it.spans + (int)threadIdx.x / LPR; row < row_end; row += RPP) {
        const int tok = tok0 + row % tokb, h = it.g * p.R + row / tokb;
        if (tok >= it.len) continue;
        float ref = -INFINITY, l = 0.f;
        float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
        for (int k = 0; k < it.spans; ++k) {
            const int64_t prow = (int64_t)(slot0 + k * p.G) * PACKED_ROWS + row;
            const float m = p.part_ml[prow * 2], lk = p.part_ml[prow * 2 + 1];
            if (!(lk > 0.f)) continue;  // the span holds no key of the row
            const u4 x = *reinterpret_cast<const u4*>(reinterpret_cast<const uint16_t*>(p.part_o) + prow * D + d0);
            const float m_new = fmaxf(ref, m);
            const float keep = fast_exp2(ref - m_new), w = lk * fast_exp2(m - m_new);  // (0 while ref is -inf)
            ref = m_new;
            l = l * keep + w;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t two = x[i];
                acc[2 * i] = acc[2 * i] * keep + T::lo(two) * w;
                acc[2 * i + 1] = acc[2 * i + 1] * keep + T::hi(two) * w;
            }
        }
        const float inv = l > 0.f ? 1.f / l : 0.f;
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
    const int64_t blocks = packed_grid(p.T, p.B, p.G, packed_tokb(D, p.R, QS), p.part_o != nullptr);
    if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    G4B_LAUNCH_DOMINANT((attn_packed_kernel<D, T, QS>), dim3((unsigned)blocks), dim3(256), smem, stream, p);
    e = hipGetLastError();
    if (e != hipSuccess || !p.part_o) return e;
    hipLaunchKernelGGL((attn_packed_combine<D, T, (D == 512 && QS) ? 64 : 128>), dim3(PACKED_SLOTS), dim3(256), 0, stream, p);
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

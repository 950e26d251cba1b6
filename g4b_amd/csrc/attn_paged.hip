// Launchers of decode attention over pages: the streaming kernels of attn_decode.hpp with rows that sit in pages.
#include "attn_decode.hpp"
#include "paged.hpp"

namespace g4b {

template <int D, int CL, class T, int DH, bool QS>
__global__ __launch_bounds__(64 * DH, 1) void attn_paged_worker(const PagedParams p) {
    __shared__ float xch_buf[DH > 1 ? 2 * DH * 8 * 64 : 1];
    decode_worker_body<D, CL, T, DH, QS>(p, blockIdx.x, xch_buf);
}

// Short windows: a pair's tiles are dealt to the waves of one workgroup.  At head dimension 128 eight waves of a tile in
// flight each, at 256, where a wave needs a SIMD's registers for itself, four with two tiles in flight (64 sequences, 512 keys,
// H/G = 4, 16-bit query: 21.4 -> 19.5 .. 21 us; with H/G above 8 and an unrounded query the second tile spills 52 registers).  Launched for 128 pairs the kernel keeps half of the chip busy and reads 3.2 TB/s.
template <int D, int CL, class T, bool QS>
__global__ __launch_bounds__(64 * paged_pair_waves(D), paged_pair_waves(D) / 4) void attn_paged_pair(const PagedParams p) {
    extern __shared__ __align__(16) float pair_smem[];
    decode_pair_body<D, CL, T, QS, PagedParams, paged_pair_waves(D), D == 128 ? 1 : 2>(p, blockIdx.x, pair_smem);
}

template <int D>
__global__ __launch_bounds__(256) void attn_paged_combine(const PagedParams p) {
    __shared__ DecodeCombineSmem<D> sm;
    decode_combine_body<D>(p, blockIdx.x, blockIdx.y, sm);
}

template <int D, int CL, class T, bool QS>
static hipError_t launch_paged_t(const PagedParams& p, hipStream_t stream) {
    if constexpr (D <= 256) {
        if (paged_pair_path(p, D)) {
            constexpr int smem = dec_pair_smem<D, paged_pair_waves(D)>();
            static uint64_t attr_done = 0;
            hipError_t e = allow_dynamic_smem(reinterpret_cast<const void*>(&attn_paged_pair<D, CL, T, QS>), smem, attr_done);
            if (e != hipSuccess) return e;
            G4B_LAUNCH_DOMINANT((attn_paged_pair<D, CL, T, QS>), dim3(p.B * p.G), dim3(64 * paged_pair_waves(D)), smem, stream, p);
            return hipGetLastError();
        }
    }
    constexpr int DH = D > 256 ? D / 256 : 1;  // waves per worker: each owns at most 256 columns
    G4B_LAUNCH_DOMINANT((attn_paged_worker<D, CL, T, DH, QS>), dim3(p.NW > 0 ? p.NW : p.B * p.G), dim3(64 * DH), 0, stream, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (p.NW > 0) hipLaunchKernelGGL((attn_paged_combine<D>), dim3(p.B * p.G, p.R), dim3(256), 0, stream, p);
    return hipGetLastError();
}

template <int D, class T>
static hipError_t launch_paged_cl(const PagedParams& p, hipStream_t stream) {
    if (p.q_split) {
        if (p.R <= 4) return launch_paged_t<D, 4, T, true>(p, stream);
        if (p.R <= 8) return launch_paged_t<D, 2, T, true>(p, stream);
        return launch_paged_t<D, 1, T, true>(p, stream);
    }
    if (p.R <= 4) return launch_paged_t<D, 4, T, false>(p, stream);
    if (p.R <= 8) return launch_paged_t<D, 2, T, false>(p, stream);
    return launch_paged_t<D, 1, T, false>(p, stream);
}

hipError_t launch_paged_decode(const PagedParams& p, int D, int kv_dt, hipStream_t stream) {
    if (kv_dt == DT_F16) {
        if (D == 512) return launch_paged_cl<512, F16>(p, stream);
        if (D == 256) return launch_paged_cl<256, F16>(p, stream);
        if (D == 128) return launch_paged_cl<128, F16>(p, stream);
    } else {
        if (D == 512) return launch_paged_cl<512, BF16>(p, stream);
        if (D == 256) return launch_paged_cl<256, BF16>(p, stream);
        if (D == 128) return launch_paged_cl<128, BF16>(p, stream);
    }
    return hipErrorInvalidValue;
}

}  // namespace g4b

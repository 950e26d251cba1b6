// The body of the plain fp32 attention kernels: NQ query heads of one kv head at one query position per workgroup.
//
// All arithmetic is fp32 on the vector ALU (no operand is rounded, so USE_FP32_DOT holds trivially; with Rows::rounds_query the
// query may be, for rows that have to come out as a tuned kernel reads them).  The heads see the
// same keys, so every K and V row is loaded once for all of them; the four waves take the 64-key chunks of the range in
// turn.  Within a chunk a lane owns one key for K Q^T (the query row sits in LDS, read as a broadcast) and eight output
// columns for P V (several keys per pass when the head dimension is below 512).  The four online-softmax states meet in
// LDS in a fixed order, so results do not depend on timing.  Only keys of the range are ever read, so what a cache holds
// elsewhere (stale rows, infinities, NaN) cannot reach a result.
#pragma once
#include "common.hpp"

namespace g4b {

constexpr int GEN_MAX_D = 1024;
constexpr int GEN_WAVES = 4;

G4B_DEV float wave_max64(float v) {
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) v = fmaxf(v, __shfl_xor(v, s));
    return v;
}
G4B_DEV float wave_sum64(float v) {
#pragma unroll
    for (int s = 32; s >= 1; s >>= 1) v += __shfl_xor(v, s);
    return v;
}

// A sum of exponentials is +0 where no key was seen.  By its bits: comparisons are compiled as if no NaN could occur, and the
// sum of a row that sees a NaN must not count as empty.
G4B_DEV bool is_zero(float l) { return __float_as_uint(l) == 0; }

template <int NQ>
struct GenericSmem {
    float q[NQ][GEN_MAX_D];               // the query rows times scale * log2(e)
    float part[GEN_WAVES][GEN_MAX_D];     // per wave: [key sub-group][D] un-normalised sums of one head (sub-groups * D <= 1024)
    float m[NQ][GEN_WAVES], l[NQ][GEN_WAVES];
};

// Where the query rows of a workgroup's NQ heads are and where their results go.
struct GenericIo {
    const void* q;
    void* o;
    int64_t q_off, q_head, o_off, o_head;  // element offset of the first head's row, stride from head to head
    int32_t q_dt, o_dt;
    float c;  // softmax scale * log2(e)
    float* ml = nullptr;  // optional: (maximum in log2 units, sum) of the first head's row
};

// Attention of the NQ rows over keys [lo, hi) of `rows`: rows.k(j) and rows.v(j) point at the rows of key j, of element
// type kv_dt; with Rows::may_be_absent a null pointer is a key that is not seen, with Rows::may_be_dark 64 keys in a row may be
// unseen or score minus infinity.  A row that sees no other key becomes zeros.
template <int NQ, class Rows>
G4B_DEV void generic_rows(GenericSmem<NQ>& sm, const Rows& rows, const GenericIo& io, const int lo, const int hi, const int D,
                          const int kv_dt) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int nchunk = D >> 3;  // 8-column pieces of a row
    for (int t = tid; t < NQ * nchunk; t += 64 * GEN_WAVES) {
        const int n = t / nchunk, c = t % nchunk;
        float x[8];
        load_f32<8>(io.q, io.q_off + (int64_t)n * io.q_head + c * 8, io.q_dt, x);
        if constexpr (Rows::rounds_query) rows.round_query(x);
#pragma unroll
        for (int e = 0; e < 8; ++e) sm.q[n][c * 8 + e] = x[e] * io.c;
    }
    __syncthreads();

    // P V ownership: kpp keys per pass, lane = (key sub-group sk, piece c); cpl pieces per lane when D > 512
    const int kpp = nchunk >= 64 ? 1 : 64 / nchunk;
    const int cpl = (nchunk + 63) >> 6;
    const int sk = nchunk >= 64 ? 0 : lane / nchunk;
    const int c0 = nchunk >= 64 ? lane : lane % nchunk;
    const bool pv_lane = sk < kpp;

    float m[NQ], l[NQ];
    float acc[NQ][2][8];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        m[n] = -INFINITY;
        l[n] = 0.f;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[n][u][e] = 0.f;
    }

    for (int j0 = lo + wave * 64; j0 < hi; j0 += 64 * GEN_WAVES) {
        const int nk = min(64, hi - j0);
        // ---- scores: one key per lane
        const bool valid = lane < nk;
        const void* krow = rows.k(j0 + (valid ? lane : 0));
        const bool seen = valid && (!Rows::may_be_absent || krow != nullptr);
        float s[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[n] = 0.f;
        for (int c = 0; c < nchunk; ++c) {
            if (Rows::may_be_absent && !seen) continue;
            float kx[8];
            load_f32<8>(krow, c * 8, kv_dt, kx);
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                const f4 qa = *reinterpret_cast<const f4*>(&sm.q[n][c * 8]);
                const f4 qc = *reinterpret_cast<const f4*>(&sm.q[n][c * 8 + 4]);
                float s0 = 0.f, s1 = 0.f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s0 = fmaf(kx[e], qa[e], s0);
                    s1 = fmaf(kx[4 + e], qc[e], s1);
                }
                s[n] += s0 + s1;
            }
        }
        float pj[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const float sv = seen ? s[n] : -INFINITY;
            const float m_new = fmaxf(m[n], wave_max64(sv));  // finite unless every key so far was absent or scored -inf
            const float m_safe = (Rows::may_be_dark && m_new == -INFINITY) ? 0.f : m_new;
            const float alpha = exp2f(m[n] - m_safe);         // 0 on the first chunk
            pj[n] = exp2f(sv - m_safe);                       // 0 for lanes past the range and absent keys
            l[n] = l[n] * alpha + wave_sum64(pj[n]);
            m[n] = m_new;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[n][u][e] *= alpha;
        }
        // ---- P V: kpp keys per pass
        for (int jj = 0; jj < nk; jj += kpp) {
            const int kk = jj + sk;
            float pk[NQ];
#pragma unroll
            for (int n = 0; n < NQ; ++n) pk[n] = __shfl(pj[n], kk & 63);
            if (pv_lane && kk < nk) {
                const void* vrow = rows.v(j0 + kk);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const int c = c0 + u * 64;
                    if (u < cpl && c < nchunk && (!Rows::may_be_absent || vrow != nullptr)) {
                        float vx[8];
                        load_f32<8>(vrow, c * 8, kv_dt, vx);
#pragma unroll
                        for (int n = 0; n < NQ; ++n)
#pragma unroll
                            for (int e = 0; e < 8; ++e) acc[n][u][e] = fmaf(pk[n], vx[e], acc[n][u][e]);
                    }
                }
            }
        }
    }

    // ---- the four waves' states meet in LDS, one head after the other
    if (lane == 0) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            sm.m[n][wave] = m[n];
            sm.l[n][wave] = l[n];
        }
    }
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
        if (n > 0) __syncthreads();  // the previous head's sums have been read
        if (pv_lane) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int c = c0 + u * 64;
                if (u < cpl && c < nchunk) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) sm.part[wave][sk * D + c * 8 + e] = acc[n][u][e];
                }
            }
        }
        __syncthreads();
        if (tid < nchunk) {
            float M = -INFINITY;
#pragma unroll
            for (int w = 0; w < GEN_WAVES; ++w) M = fmaxf(M, sm.m[n][w]);
            float L = 0.f, out[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) out[e] = 0.f;
            for (int w = 0; w < GEN_WAVES; ++w) {
                const float mw = sm.m[n][w];
                if (is_zero(sm.l[n][w])) continue;  // the wave saw no key
                const float f = exp2f(mw - M);
                L += f * sm.l[n][w];
                for (int s2 = 0; s2 < kpp; ++s2)
#pragma unroll
                    for (int e = 0; e < 8; ++e) out[e] = fmaf(f, sm.part[w][s2 * D + tid * 8 + e], out[e]);
            }
            // a row that sees no key is written as zeros, like the tuned kernels
            const float inv = is_zero(L) ? 0.f : 1.f / L;
#pragma unroll
            for (int e = 0; e < 8; ++e) out[e] *= inv;
            if (io.ml && tid == 0) {
                io.ml[0] = M == -INFINITY ? 0.f : M;
                io.ml[1] = L;
            }
            store8(io.o, io.o_off + (int64_t)n * io.o_head + tid * 8, io.o_dt, out);
        }
    }
}

}  // namespace g4b

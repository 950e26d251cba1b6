// Infinities and NaN in places that a mask hides.
//
// The matrix cores multiply a hidden key's value row by a probability of zero, and zero times an infinity or NaN is NaN: a
// value that is not finite would reach the rows of its query tile that must not see it.  Only edge tiles (which some row of the
// workgroup does not see whole) can do that, so their V tile is looked at where it lies in LDS, and a query tile that has met
// such a value is computed again, row by row, by the plain fp32 body, which never touches a hidden key and
// takes the query as the matrix cores do.  The look costs the edge tiles only: two prompts of 4126 and 8192 tokens under a
// 512-key window, where they are a fifth of all, 98 -> 100 us; 8192 tokens without a window 355 -> 357 us.  The rows of a tile
// that is computed again take one workgroup for themselves, whatever that costs.
#pragma once
#include "attn_generic.hpp"
#include "packed_map.hpp"

namespace g4b {

// Whether the thread's share of a TILE-byte tile of 16-bit elements at LDS address `at` holds a value that is not finite.
template <class T, int TILE>
G4B_DEV bool packed_tile_not_finite(uint32_t at) {
    typedef uint16_t us2 __attribute__((ext_vector_type(2)));
    constexpr int READS = TILE / 4096;  // 16 bytes per thread each
    static_assert(READS >= 2 && READS % 2 == 0, "reads are retired in pairs");
    const uint32_t mine = at + (uint32_t)threadIdx.x * 16u;
    u4 r[READS];
#pragma unroll
    for (int i = 0; i < READS; ++i) r[i] = lds_read16(mine, i * 4096);
    us2 most = {0, 0};
#pragma unroll
    for (int i = 0; i < READS; i += 2) {
        u4 a = r[i], b = r[i + 1];
        lds_wait_pair<0>(a, b);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const uint32_t x = a[w] & 0x7fff7fffu, y = b[w] & 0x7fff7fffu;
            most = __builtin_elementwise_max(most, __builtin_elementwise_max(__builtin_bit_cast(us2, x), __builtin_bit_cast(us2, y)));
        }
    }
    constexpr uint16_t INF = T::dt == DT_F16 ? 0x7c00 : 0x7f80;
    const uint16_t m0 = most[0], m1 = most[1];
    return m0 >= INF || m1 >= INF;
}

template <class T>
struct PackedPlainRows {
    static constexpr bool may_be_absent = false, may_be_dark = true, rounds_query = true;
    const char *kb, *vb;
    int64_t k_pitch, v_pitch;
    bool rounded;  // the matrix cores take the query in T: what a hidden row holds must not change how the others are read
    G4B_DEV void round_query(float (&x)[8]) const {
        if (!rounded) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t two = T::pack2(x[2 * i], x[2 * i + 1]);
            x[2 * i] = T::lo(two);
            x[2 * i + 1] = T::hi(two);
        }
    }
    G4B_DEV const void* k(int j) const { return kb + j * k_pitch; }
    G4B_DEV const void* v(int j) const { return vb + j * v_pitch; }
};

// The rows of item `pk` (ROWS of them, of the workgroup `bid`), one after the other.  Called by the whole workgroup.
template <int D, class T, int ROWS>
G4B_DEV void packed_plain_item(const PackedParams& p, const PackedItem& pk, int bid, char* smem) {
    GenericSmem<1>& sm = *reinterpret_cast<GenericSmem<1>*>(smem);
    const int tokb = ROWS / p.R;
    const PackedPlainRows<T> rows{static_cast<const char*>(p.k) + ((int64_t)pk.first * p.k_ts + pk.g * p.k_hs) * 2,
                               static_cast<const char*>(p.v) + ((int64_t)pk.first * p.v_ts + pk.g * p.v_hs) * 2, p.k_ts * 2, p.v_ts * 2, p.q_split == 0};
    for (int r = 0; r < ROWS; ++r) {
        const int tok = pk.qtile * tokb + r % tokb, h = pk.g * p.R + r / tokb;
        if (tok >= pk.len) continue;
        const int lo = max(p.qwin > 0 ? max(0, tok - p.qwin + 1) : 0, pk.key0), hi = min(tok + 1, pk.key1);
        GenericIo io{p.q, p.o, (int64_t)(pk.first + tok) * p.q_s[2] + h * p.q_s[1], 0,
                     (int64_t)(pk.first + tok) * p.o_s[2] + h * p.o_s[1], 0, p.q_dt, p.o_dt, p.c};
        if (pk.spans > 1) {  // a span's rows go to its slot, normalised by their own sums
            const int64_t prow = (int64_t)bid * PACKED_ROWS + r;
            io.o = p.part_o;
            io.o_off = prow * D;
            io.o_dt = DT_F32;
            io.ml = p.part_ml + prow * 2;
        }
        __syncthreads();  // the previous row's sums have been read
        generic_rows<1>(sm, rows, io, lo, max(hi, lo), D, T::dt);
    }
}

}  // namespace g4b

// Work-item bookkeeping of attention over packed prompts.
//
// A query tile is tokb = rows / (H/G) consecutive tokens of one sequence (all heads of a kv head's group share its keys); an
// item is a (sequence, kv head, query tile), or one of the key spans it is cut into.  Which workgroup takes which item is
// computed by the workgroups themselves from cu_seqlens, so the grid is static (a recorded launch follows the prompts of
// each replay) and the host reads nothing.
//
// Whole query tiles: under the causal mask the work of a tile grows with its position in its prompt, so the tiles of all
// prompts are taken from the latest position to the earliest; the hardware hands workgroups out in order and a launch of
// many tiles ends evenly whatever the prompts' lengths.  The kv head runs fastest, so that the XCDs (workgroup id modulo 8)
// share as few heads' keys as possible.  Under a window the tiles that see a whole window cost the same and only neighbours
// share keys: they come first, in contiguous runs per XCD, and the shorter ones of the prompts' beginnings fill the last round
// (prompts of 4126, 60 and 8192 tokens, 774 tiles for 256 places, 512 keys: 85 us; 100 us with all tiles in runs).
//
// Key spans: a launch with few tiles lasts as long as its longest one while most of the chip is idle.  The tiles of such a
// launch are cut at multiples of `span` keys, the smallest that leaves no more spans than partial slots; every span leaves
// its rows, normalised by its own sum, in a slot in fp32, and a second kernel joins them.  With tiles and spans on multiples of
// tokb the number of spans of a prompt is a closed form, so finding an item takes a handful of sums over the prompts.  (Built and
// measured as well, with span rows in 16 bits: cutting the last, incomplete round of a window's tiles, those 774 tiles 94.7 us
// whole, in runs, and 102 us cut, nine prompts of 1000 tokens 57 and 78 us; and dealing the steps of all tiles to the compute
// units in equal shares that begin and end inside tiles, 2048 tokens at head dimension 256 44 us against 38 us in spans, 4096
// tokens 96 us against 106 us whole: a share of several tiles pays each tile's start, and the loop over them takes registers;
// and cutting launches of up to a tile per compute unit at the average tile's length, longest spans first, 4000 tokens 119 us
// against 103 whole, 2500 69 against 64: a step takes a third longer with every compute unit at work.)
#pragma once
#include "paged.hpp"

namespace g4b {

// Workgroups the chip holds at once: one per compute unit, two where registers and LDS allow (head dimension 128 with a
// 16-bit query).  Also the partial slots of a launch.
__host__ __device__ constexpr int packed_slots(int D, bool q_split) { return D == 128 && !q_split ? 512 : 256; }
constexpr int PACKED_ROWS = 128;       // query rows per workgroup
constexpr int PACKED_KEYS = 64;        // spans are multiples of this many keys
// The host asks for a launch that may be cut when a prompt of all its rows would be of packed_cut_steps steps of 64 keys or more:
// what the second kernel costs even if nothing is cut (3 us of prompts of 700 and 500 tokens at D = 256) and what the partial
// rows do.  One prompt, whole and cut (kv heads 2, query heads 8, us): D = 128 1280 tokens 26.1 and 28.5, 1536 29.7 and 28.5, 2048
// 37.7 and 32.6, 4096 68.3 and 62.8; D = 256 640 23.3 and 23.8, 768 26.1 and 25.4, 1024 31.4 and 27.9, 2048 53.7 and 41.6;
// D = 512 448 33.9 and 33.5, 512 36.9 and 34.2, 1024 59.9 and 41.1, 2048 108 and 70.5.  The device, which sees the prompts, then
// cuts when the longest tile becomes packed_cut_gain steps shorter.  Whole and cut, both with the second kernel: D = 128 two of 680
// 21.2 and 23.9 (9 steps won), 1100 and 300 27.0 and 27.5 (16); D = 256 two of 600 25.4 and 27.4 (8), 700 and 500 27.9 and 27.4 (9).
constexpr int packed_cut_steps(int D) { return D == 512 ? 7 : D == 256 ? 12 : 22; }
__host__ __device__ constexpr int packed_cut_gain(int D) { return D == 512 ? 5 : D == 256 ? 9 : 17; }

// floor(x / m) for 0 <= x < 2^24, m >= 1: every workgroup counts spans before it starts, and an integer division is thirty
// instructions.  inv = 1 / m; the product is off by less than one.
__host__ __device__ inline int packed_div(int x, int m, float inv) {
    int q = (int)((float)x * inv);
    const int r = x - q * m;
    if (r < 0) --q;
    else if (r >= m) ++q;
    return q;
}
// sum of floor(i / m) over i < x, modulo 2^32 (the numbers of spans, differences of these, are far below)
__host__ __device__ inline uint32_t packed_floor_sum(int x, int m, float inv) {
    const uint32_t q = (uint32_t)packed_div(x, m, inv), r = (uint32_t)x - q * (uint32_t)m;
    const uint32_t pairs = (q & 1u) ? q * ((q - 1u) >> 1) : (q >> 1) * (q - 1u);  // q (q - 1) / 2
    return (uint32_t)m * pairs + r * q;
}
// Spans of the first n query tiles of a prompt, with m tiles per span of keys and query tiles from the d-th on no longer
// seeing all keys before them (tile t sees keys from max(0, t - d) tiles on): tile t has
// floor(t / m) - floor(max(t - d, 0) / m) + 1 of them.
__host__ __device__ inline int packed_spans(int n, int m, float inv, int d) {
    return (int)((uint32_t)n + packed_floor_sum(n, m, inv) - (n > d ? packed_floor_sum(n - d, m, inv) : 0u));
}

struct PackedItem {
    int first, len;   // rows of the sequence
    int g, qtile;
    int key0, key1;   // keys of the span, multiples of the span's length (key1 may lie past what the tile sees)
    int spans, span;  // spans of the tile, 1: it is whole; which of them this is (its partial slot is its workgroup's id)
    bool valid;
};
// An item's numbers are the same in every lane, which the compiler cannot see through the sums and branches they come from:
// the kernels want them in scalar registers.
G4B_DEV void packed_uniform(PackedItem& it) {
    it.first = __builtin_amdgcn_readfirstlane(it.first);
    it.len = __builtin_amdgcn_readfirstlane(it.len);
    it.g = __builtin_amdgcn_readfirstlane(it.g);
    it.qtile = __builtin_amdgcn_readfirstlane(it.qtile);
    it.key0 = __builtin_amdgcn_readfirstlane(it.key0);
    it.key1 = __builtin_amdgcn_readfirstlane(it.key1);
    it.spans = __builtin_amdgcn_readfirstlane(it.spans);
    it.span = __builtin_amdgcn_readfirstlane(it.span);
}
// What the joining kernel has to know of a slot, left there by the span's workgroup (by every slot's, on each launch).
struct PackedSlot {
    int32_t first, len, g, qtile, spans, span, pad[2];  // spans = 0: nothing to join
};
G4B_DEV PackedSlot* packed_slot_info(const PackedParams& p, int slots) {
    return reinterpret_cast<PackedSlot*>(p.part_ml + (int64_t)slots * PACKED_ROWS * 2);
}

// Sums over the sequences.  Up to 64 of them: lane s of every wave holds sequence s, and nothing is exchanged between waves.
// More: a thread of the workgroup holds four consecutive ones, and what a pass of them cannot hold is read again for every sum
// (300 prompts, read for every sum as well: 5.7 us before a workgroup had its item, its 1200 items 75 us in all, now 61).
constexpr int SEQS_HELD = 4;
template <int THREADS>
struct PackedSeqs {
    const int32_t* cu;
    int64_t cu_s;
    int B, T, tokb_log, tid;
    int held[SEQS_HELD];
    int* sh;  // THREADS / 64 + 2 ints of LDS
    G4B_DEV int load(int s) const {
        const int a = min(max(cu[(int64_t)s * cu_s], 0), T), b = min(max(cu[(int64_t)(s + 1) * cu_s], a), T);
        return (b - a + (1 << tokb_log) - 1) >> tokb_log;
    }
    G4B_DEV PackedSeqs(const PackedParams& p, int tokb, int* sh_)
        : cu(p.cu), cu_s(p.cu_s), B(p.B), T(p.T), tokb_log(__ffs(tokb) - 1), tid((int)threadIdx.x), sh(sh_) {
#pragma unroll
        for (int i = 0; i < SEQS_HELD; ++i) held[i] = 0;
        if (B <= 64) {
            if ((tid & 63) < B) held[0] = load(tid & 63);
        } else {
#pragma unroll
            for (int i = 0; i < SEQS_HELD; ++i)
                if (tid * SEQS_HELD + i < B) held[i] = load(tid * SEQS_HELD + i);
        }
    }
    // more than 64 sequences: the thread's i-th of the pass that starts at sequence `base`
    G4B_DEV int of_pass(int base, int i) const {
        const int s = base + tid * SEQS_HELD + i;
        return base == 0 ? held[i] : s < B ? load(s) : 0;
    }
    G4B_DEV int tiles_of(int s) const { return B <= 64 ? __builtin_amdgcn_readlane(held[0], s) : load(s); }
    // sum of f(tiles of the sequence), f(0) = 0
    template <class F>
    G4B_DEV int sum(const F f) const {
        if (B == 1) return f(__builtin_amdgcn_readfirstlane(held[0]));
        if (B <= 64) return wave_sum_i(f(held[0]));
        int v = 0;
        for (int base = 0; base < B; base += THREADS * SEQS_HELD)
#pragma unroll
            for (int i = 0; i < SEQS_HELD; ++i) v += f(of_pass(base, i));
        v = wave_sum_i(v);
        __syncthreads();  // the previous sums have been read
        if ((tid & 63) == 0) sh[tid >> 6] = v;
        __syncthreads();
        int total = 0;
#pragma unroll
        for (int w = 0; w < THREADS / 64; ++w) total += sh[w];
        return __builtin_amdgcn_readfirstlane(total);
    }
    G4B_DEV int longest() const {  // query tiles of the longest sequence
        if (B == 1) return __builtin_amdgcn_readfirstlane(held[0]);
        int v = held[0];
        if (B > 64)
            for (int base = 0; base < B; base += THREADS * SEQS_HELD)
#pragma unroll
                for (int i = 0; i < SEQS_HELD; ++i) v = max(v, of_pass(base, i));
        v = max(v, dpp_i0<0xB1>(v));
        v = max(v, dpp_i0<0x4E>(v));
        v = max(v, dpp_i0<0x141>(v));
        v = max(v, dpp_i0<0x140>(v));  // every lane holds its row's maximum
        v = max(max(__builtin_amdgcn_readlane(v, 0), __builtin_amdgcn_readlane(v, 16)),
                max(__builtin_amdgcn_readlane(v, 32), __builtin_amdgcn_readlane(v, 48)));
        if (B <= 64) return v;
        __syncthreads();
        if ((tid & 63) == 0) sh[tid >> 6] = v;
        __syncthreads();
        int most = 0;
#pragma unroll
        for (int w = 0; w < THREADS / 64; ++w) most = max(most, sh[w]);
        return __builtin_amdgcn_readfirstlane(most);
    }
    // The sequence s with before(s) <= r < before(s) + f(s), before being the sum over the sequences in front of s; r
    // becomes r - before(s).  r is below the sum over all sequences.
    template <class F>
    G4B_DEV int select(const F f, int& r) const {
        const int lane = tid & 63, wave = tid >> 6;
        if (B == 1) return 0;
        if (B <= 64) {
            const int v = f(held[0]);
            const int incl = wave_incl_scan_i(v, lane);
            const unsigned long long hit = __ballot(incl > r && incl - v <= r);
            const int src = __ffsll((long long)hit) - 1;
            r -= __builtin_amdgcn_readlane(incl - v, src);
            return src;
        }
        int before = 0;
        for (int base = 0; base < B; base += THREADS * SEQS_HELD) {
            int c[SEQS_HELD], v = 0;
#pragma unroll
            for (int i = 0; i < SEQS_HELD; ++i) v += c[i] = f(of_pass(base, i));
            const int incl = wave_incl_scan_i(v, lane);
            __syncthreads();
            if (lane == 63) sh[wave] = incl;
            __syncthreads();
            int mine = before, total = 0;
#pragma unroll
            for (int w = 0; w < THREADS / 64; ++w) {
                mine += w < wave ? sh[w] : 0;
                total += sh[w];
            }
            if (r < before + total) {  // (uniform) it is one of these
                int at = mine + incl - v;
#pragma unroll
                for (int i = 0; i < SEQS_HELD; ++i) {
                    if (at <= r && r < at + c[i]) {
                        sh[THREADS / 64] = base + tid * SEQS_HELD + i;
                        sh[THREADS / 64 + 1] = at;
                    }
                    at += c[i];
                }
                __syncthreads();
                r -= __builtin_amdgcn_readfirstlane(sh[THREADS / 64 + 1]);
                return __builtin_amdgcn_readfirstlane(sh[THREADS / 64]);
            }
            before += total;
        }
        return 0;  // (not reached: r is below the sum)
    }
};

// Query tiles per span of keys, 0 where cutting does not pay.
template <int D, int SLOTS, int THREADS>
G4B_DEV int packed_cut(const PackedParams& p, const PackedSeqs<THREADS>& seqs, int d) {
    const int tokb = 1 << seqs.tokb_log;
    const int unit = tokb > PACKED_KEYS ? tokb : PACKED_KEYS;  // both powers of two
    const int per_unit_log = __ffs(unit) - __ffs(tokb);
    const int see = min(seqs.longest(), d + 1);                         // query tiles' worth of keys that its last tile sees
    const int steps = (see + (1 << per_unit_log) - 1) >> per_unit_log;  // ... in units
    int lo = 1, hi = steps;  // units per span: too few .. enough
    if (steps * (unit / PACKED_KEYS) <= packed_cut_gain(D)) return 0;
    auto fits = [&](int units) {
        const int m = units << per_unit_log;
        const float inv = 1.f / (float)m;
        return seqs.sum([=](int n) { return packed_spans(n, m, inv, d); }) * p.G <= SLOTS;
    };
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (fits(mid)) hi = mid;
        else lo = mid;
    }
    if ((steps - hi) * (unit / PACKED_KEYS) < packed_cut_gain(D) || !fits(hi)) return 0;
    return hi << per_unit_log;
}

// The item of workgroup `bid`.  Every thread of the workgroup calls it.
template <int D, int SLOTS, int THREADS>
G4B_DEV PackedItem packed_item(const PackedParams& p, int bid, int tokb, int* sh) {
    PackedItem it = {};
    const PackedSeqs<THREADS> seqs(p, tokb, sh);
    const int tiles = seqs.sum([](int n) { return n; });
    const int items = tiles * p.G;  // (at most T * G, below 2^31)
    // from this query tile on a tile no longer sees the first keys of its prompt
    const int d = p.qwin > 0 ? (int)(((int64_t)p.qwin - 1 + tokb - 1) >> (__ffs(tokb) - 1)) : 0x3fffffff;
    const int m = p.part_o && items * 2 <= SLOTS ? packed_cut<D, SLOTS>(p, seqs, d) : 0;
    int s;
    it.spans = 1;
    it.key1 = 0x7fffffff;
    if (m > 0) {
        int r = bid / p.G;
        it.g = bid - r * p.G;
        const float inv = 1.f / (float)m;
        auto spans = [=](int n) { return packed_spans(n, m, inv, d); };
        it.valid = r < seqs.sum(spans);
        if (it.valid) {
            s = seqs.select(spans, r);
            // the tile whose spans hold r: spans(lo) <= r < spans(hi); a tile has at least one span
            int lo = 0, hi = min(r + 1, seqs.tiles_of(s));
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (spans(mid) <= r) lo = mid;
                else hi = mid;
            }
            it.qtile = lo;
            it.span = r - spans(lo);
            it.spans = spans(lo + 1) - spans(lo);
            const int c = (lo > d ? packed_div(lo - d, m, inv) : 0) + it.span;  // spans lie on multiples of their length
            it.key0 = c * m * tokb;
            it.key1 = it.key0 + m * tokb;
        }
    } else {
        // the tiles that see a whole window come first, in contiguous runs per XCD, kv head by kv head
        const int full = p.qwin > 0 ? seqs.sum([=](int n) { return max(n - d, 0); }) : 0;
        const int run = (full * p.G + 7) >> 3;
        if (bid < 8 * run) {
            const int f = (bid & 7) * run + (bid >> 3);
            it.valid = f < full * p.G;
            if (it.valid) {
                it.g = f / full;
                int r = f - it.g * full;
                s = seqs.select([=](int n) { return max(n - d, 0); }, r);
                it.qtile = d + r;
            }
        } else {
            int r = (bid - 8 * run) / p.G;
            it.g = bid - 8 * run - r * p.G;
            it.valid = r < tiles - full;
            if (it.valid && items <= SLOTS) {  // all at once: any order will do
                s = seqs.select([=](int n) { return min(n, d); }, r);
                it.qtile = r;
            } else if (it.valid) {
                // tiles at position t or later: more than r of them at the t that is looked for, at most r at the next
                int t = 0;
                for (int bit = 1 << (31 - __builtin_clz(min(seqs.longest(), d))); bit; bit >>= 1)
                    if (seqs.sum([=](int n) { return max(min(n, d) - t - bit, 0); }) > r) t += bit;
                r -= seqs.sum([=](int n) { return max(min(n, d) - t - 1, 0); });
                s = seqs.select([=](int n) { return min(n, d) > t ? 1 : 0; }, r);
                it.qtile = t;
            }
        }
    }
    if (it.valid) {
        int end;
        packed_rows(p, s, it.first, end);
        it.len = end - it.first;
    }
    packed_uniform(it);
    if (p.part_o && bid < SLOTS && threadIdx.x == 0) {
        const bool joins = it.valid && it.spans > 1;  // (the only span of a tile is written to o)
        *(packed_slot_info(p, SLOTS) + bid) = PackedSlot{it.first, it.len, it.g, it.qtile, joins ? it.spans : 0, it.span, {0, 0}};
    }
    return it;
}

// Workgroups that hold every item a launch over T rows of N sequences can have (the runs of the XCDs under a window leave up
// to seven of them without one).
inline int64_t packed_grid(int T, int N, int G, int tokb, int slots, bool may_cut) {
    const int64_t tiles = (int64_t)T / tokb + (N < T ? N : T);  // a prompt has at most one tile that is not full
    const int64_t grid = (tiles * G + 7) / 8 * 8 + 8;
    return may_cut && grid < slots ? slots : grid;
}
// Whether a launch over T rows can come out cut (see packed_item): its tiles, if all rows belong to prompts, leave half of
// the chip idle, and one of them may see enough keys for a cut to pay.
inline bool packed_may_cut(int T, int G, int D, int tokb, int slots, int qwin) {
    const int64_t keys = qwin > 0 && qwin < T ? (int64_t)qwin + tokb : T;
    return (int64_t)(T / tokb) * G * 2 <= slots && keys > PACKED_KEYS * (packed_cut_steps(D) - 1);
}
inline uint64_t packed_partial_bytes(int D) {
    return (uint64_t)packed_slots(D, false) * (PACKED_ROWS * ((uint64_t)D + 2) * sizeof(float) + sizeof(PackedSlot));
}

}  // namespace g4b

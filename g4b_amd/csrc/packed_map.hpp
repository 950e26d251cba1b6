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
// share as few heads' keys as possible.  Under a window all tiles cost the same and only neighbours share keys: the XCDs
// take contiguous runs.
//
// Key spans: a launch with fewer tiles than the chip has compute units would last as long as its longest tile.  Its tiles
// are cut at multiples of `span` keys, the smallest that leaves no more spans than partial slots; every span leaves its
// rows, normalised by its own sum, in a slot, and a second kernel joins them.  With tiles and spans on multiples of tokb
// the number of spans of a prompt is a closed form, so finding an item takes a handful of sums over the prompts.
#pragma once
#include "paged.hpp"

namespace g4b {

constexpr int PACKED_SLOTS = 256;      // spans a launch may be cut into: one per compute unit
constexpr int PACKED_ROWS = 128;       // query rows per workgroup
constexpr int PACKED_KEYS = 64;        // spans are multiples of this many keys
// A launch is cut when its longest tile would become this many steps of 64 keys shorter: the second kernel and the partial
// rows cost about as much.
constexpr int PACKED_SPLIT_GAIN = 5;

// sum of floor(i / m) over i < x
__host__ __device__ inline int packed_floor_sum(int x, int m) {
    const int q = x / m, r = x - q * m;
    return m * (q * (q - 1) / 2) + r * q;
}
// Spans of the first n query tiles of a prompt, with m tiles per span of keys and query tiles from the d-th on no longer
// seeing all keys before them (tile t sees keys from max(0, t - d) tiles on): tile t has
// floor(t / m) - floor(max(t - d, 0) / m) + 1 of them.
__host__ __device__ inline int packed_spans(int n, int m, int d) {
    return n + packed_floor_sum(n, m) - (n > d ? packed_floor_sum(n - d, m) : 0);
}

struct PackedItem {
    int first, len;   // rows of the sequence
    int g, qtile;
    int key0, key1;   // keys of the span, multiples of the span's length (key1 may lie past what the tile sees)
    int spans, span, slot;  // spans of the tile; which of them this is; its partial slot
    bool valid;
};

// Sums over the sequences.  Up to 64 of them: lane s of every wave holds sequence s, and nothing is exchanged between waves.
// More: the workgroup's threads take them in turn, the first 4 * threads of them from registers.
template <int THREADS>
struct PackedSeqs {
    const PackedParams& p;
    const int tokb;
    int* sh;  // THREADS / 64 + 2 ints of LDS
    int held[4];
    G4B_DEV int load(int s) const {
        int a, b;
        packed_rows(p, s, a, b);
        return (b - a + tokb - 1) / tokb;
    }
    G4B_DEV PackedSeqs(const PackedParams& p_, int tokb_, int* sh_) : p(p_), tokb(tokb_), sh(sh_) {
        const int tid = threadIdx.x, lane = tid & 63;
        if (p.B <= 64) {
            held[0] = lane < p.B ? load(lane) : 0;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) held[i] = tid + i * THREADS < p.B ? load(tid + i * THREADS) : 0;
        }
    }
    template <class F>
    G4B_DEV int sum(F&& f) const {
        if (p.B <= 64) return wave_sum_i(f(held[0]));
        int v = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) v += f(held[i]);
        for (int s = threadIdx.x + 4 * THREADS; s < p.B; s += THREADS) v += f(load(s));
        v = wave_sum_i(v);
        __syncthreads();  // the previous sums have been read
        if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
        __syncthreads();
        int total = 0;
#pragma unroll
        for (int w = 0; w < THREADS / 64; ++w) total += sh[w];
        return total;
    }
    // The sequence s with before(s) <= r < before(s) + f(s), before being the sum over the sequences in front of s; r
    // becomes r - before(s).  r is below the sum over all sequences.
    template <class F>
    G4B_DEV int select(F&& f, int& r) const {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        if (p.B <= 64) {
            const int v = f(held[0]);
            const int incl = wave_incl_scan_i(v, lane);
            const unsigned long long hit = __ballot(incl > r && incl - v <= r);
            const int src = __ffsll((long long)hit) - 1;
            r -= __builtin_amdgcn_readlane(incl - v, src);
            return src;
        }
        int before = 0;
        for (int base = 0; base < p.B; base += THREADS) {
            const int s = base + threadIdx.x;
            const int v = s < p.B ? f(load(s)) : 0;
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
                if (mine + incl > r && mine + incl - v <= r) {
                    sh[THREADS / 64] = s;
                    sh[THREADS / 64 + 1] = mine + incl - v;
                }
                __syncthreads();
                r -= sh[THREADS / 64 + 1];
                return sh[THREADS / 64];
            }
            before += total;
        }
        return 0;  // (not reached: r is below the sum)
    }
};

// How a launch is cut: query tiles per span of keys, or 0 when its tiles stay whole.  The same in every workgroup.
template <int THREADS>
G4B_DEV int packed_span_tiles(const PackedParams& p, const PackedSeqs<THREADS>& seqs, int tiles, int d) {
    if (!p.part_o || tiles * p.G * 2 > PACKED_SLOTS) return 0;  // (half of the units busy: cut in two at most, not worth it)
    const int tokb = seqs.tokb;
    const int unit = tokb > PACKED_KEYS ? tokb : PACKED_KEYS;  // both powers of two
    const int per_unit = unit / tokb;
    int longest = 0;  // query tiles of the longest prompt: the largest t with a prompt of at least t tiles
    for (int bit = 1 << (31 - __builtin_clz((p.T + tokb - 1) / tokb)); bit; bit >>= 1)
        if (seqs.sum([&](int n) { return n >= longest + bit ? 1 : 0; }) > 0) longest += bit;
    const int see = min(longest, d + 1);                 // query tiles' worth of keys that its last tile sees
    const int steps = (see + per_unit - 1) / per_unit;   // ... in units
    int lo = 1, hi = steps;  // units per span: too few .. enough
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        const int m = mid * per_unit;
        if (seqs.sum([&](int n) { return packed_spans(n, m, d); }) * p.G <= PACKED_SLOTS) hi = mid;
        else lo = mid;
    }
    if ((steps - hi) * (unit / PACKED_KEYS) < PACKED_SPLIT_GAIN) return 0;
    return hi * per_unit;
}

// The item of workgroup `bid`.  Every thread of the workgroup calls it.
template <int THREADS>
G4B_DEV PackedItem packed_item(const PackedParams& p, int bid, int tokb, int* sh) {
    PackedItem it = {};
    const PackedSeqs<THREADS> seqs(p, tokb, sh);
    const int tiles = seqs.sum([](int n) { return n; });
    // from this query tile on a tile no longer sees the first keys of its prompt
    const int d = p.qwin > 0 ? (int)(((int64_t)p.qwin - 1 + tokb - 1) / tokb) : 0x3fffffff;
    const int m = packed_span_tiles(p, seqs, tiles, d);
    int s;
    it.spans = 1;
    if (m > 0) {
        int r = bid / p.G;
        it.g = bid % p.G;
        const int total = seqs.sum([&](int n) { return packed_spans(n, m, d); });
        if (r >= total) return it;
        it.slot = bid;
        s = seqs.select([&](int n) { return packed_spans(n, m, d); }, r);
        int lo = 0, hi = seqs.load(s);  // the tile whose spans hold r: spans(lo) <= r < spans(hi)
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (packed_spans(mid, m, d) <= r) lo = mid;
            else hi = mid;
        }
        it.qtile = lo;
        it.span = r - packed_spans(lo, m, d);
        it.spans = packed_spans(lo + 1, m, d) - packed_spans(lo, m, d);
        const int c = (lo > d ? (lo - d) / m : 0) + it.span;  // spans lie on multiples of their length
        it.key0 = c * m * tokb;
        it.key1 = it.key0 + m * tokb;
    } else {
        int r;
        if (p.qwin > 0) {  // contiguous runs per XCD, kv head by kv head
            const int total = tiles * p.G, run = (total + 7) / 8;
            const int f = (bid & 7) * run + (bid >> 3);
            if ((bid >> 3) >= run || f >= total) return it;
            it.g = f / tiles;
            r = f - it.g * tiles;
            s = seqs.select([](int n) { return n; }, r);
            it.qtile = r;
        } else {
            r = bid / p.G;
            it.g = bid % p.G;
            if (r >= tiles) return it;
            // tiles at position t or later: more than r of them at the t that is looked for, at most r at the next
            int t = 0;
            for (int bit = 1 << (31 - __builtin_clz((p.T + tokb - 1) / tokb)); bit; bit >>= 1)
                if (seqs.sum([&](int n) { return max(n - t - bit, 0); }) > r) t += bit;
            r -= seqs.sum([&](int n) { return max(n - t - 1, 0); });
            s = seqs.select([&](int n) { return n > t ? 1 : 0; }, r);
            it.qtile = t;
        }
        it.key0 = 0;
        it.key1 = 0x7fffffff;
    }
    int end;
    packed_rows(p, s, it.first, end);
    it.len = end - it.first;
    it.valid = true;
    return it;
}

// Workgroups that hold every item a launch over T rows of N sequences can have.
inline int64_t packed_grid(int T, int N, int G, int tokb, bool may_split) {
    const int64_t tiles = (int64_t)T / tokb + (N < T ? N : T);  // a prompt has at most one tile that is not full
    const int64_t grid = (tiles * G + 7) / 8 * 8;
    return may_split && grid < PACKED_SLOTS ? PACKED_SLOTS : grid;
}
// Whether a launch over T rows can come out cut (see packed_span_tiles): its tiles, if all rows belong to prompts, leave half
// of the units idle, and a tile may see enough keys for a cut to pay.
inline bool packed_may_split(int T, int G, int tokb, int qwin) {
    const int64_t keys = qwin > 0 && qwin < T ? (int64_t)qwin + tokb : T;
    return (int64_t)(T / tokb) * G * 2 <= PACKED_SLOTS && keys > PACKED_KEYS * PACKED_SPLIT_GAIN;
}
inline uint64_t packed_partial_bytes(int D) { return (uint64_t)PACKED_SLOTS * PACKED_ROWS * ((uint64_t)D * 2 + 2 * sizeof(float)); }

}  // namespace g4b

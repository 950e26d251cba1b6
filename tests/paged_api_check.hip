// Host-side driver for the sanitizer build (g4b_amd/build.py --asan, tests/test_host_sanitizers.py) of the entry points over
// packed prompts and a paged cache: argument blocks with every integer field set to extremes and near misses run through
// validation and size arithmetic under AddressSanitizer and UndefinedBehaviorSanitizer.  Stand-in launchers check what the
// kernels assume of a launch that validation lets through, and refuse it.  The span arithmetic of packed prompts is compared
// with counting.
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "../g4b_amd/csrc/packed_map.hpp"
#include "../include/g4b_attn.h"

static long checks = 0, bad = 0;
static void expect(bool ok, const char* what, long long a = 0, long long b = 0) {
    ++checks;
    if (!ok && ++bad < 20) printf("%s (%lld, %lld; \"%s\")\n", what, a, b, g4b_last_error());
}

namespace g4b {
[[noreturn]] static void reached(const char* what) {
    fprintf(stderr, "paged_api_check: %s launched\n", what);
    abort();
}
hipError_t launch_attn_decode(const AttnParams&, int, int, hipStream_t) { reached("decode"); }
hipError_t launch_attn_prefill(const AttnParams&, int, int, hipStream_t) { reached("prefill"); }
hipError_t launch_attn_prefill_wide(const AttnParams&, int, hipStream_t) { reached("prefill 512"); }
hipError_t launch_attn_generic(const AttnParams&, int, int, int, hipStream_t) { reached("generic"); }
hipError_t launch_attn_mixed_f16(const AttnParams&, const AttnParams&, const MixedPlan&, hipStream_t) { reached("mixed"); }
hipError_t launch_attn_mixed_bf16(const AttnParams&, const AttnParams&, const MixedPlan&, hipStream_t) { reached("mixed"); }
hipError_t launch_attn_mixed_d512_f16(const AttnParams&, const AttnParams&, const MixedPlan&, hipStream_t) { reached("mixed"); }
hipError_t launch_attn_mixed_d512_bf16(const AttnParams&, const AttnParams&, const MixedPlan&, hipStream_t) { reached("mixed"); }
hipError_t launch_kv_append(const KvAppendParams&, hipStream_t) { reached("append"); }
hipError_t launch_advance_decode_state(const AdvanceParams&, hipStream_t) { reached("advance"); }
hipError_t launch_rope(const RopeParams&, hipStream_t) { reached("rope"); }
hipError_t launch_rope_frequencies(float*, const float*, int, int64_t, int64_t, float, hipStream_t) { reached("rope frequencies"); }

static hipError_t no() { return hipErrorInvalidValue; }
static bool packed_ok(const PackedParams& p, int D) {
    return p.T > 0 && p.B > 0 && p.G > 0 && p.R * p.G == p.H && D % 8 == 0 && D <= 1024 && (int64_t)p.T * p.H <= INT_MAX && p.c > 0.f;
}
hipError_t launch_packed_generic(const PackedParams& p, int D, int, hipStream_t) {
    expect(packed_ok(p, D), "plain packed launch", p.T, D);
    return no();
}
hipError_t launch_packed_prefill(const PackedParams& p, int D, int kv_dt, hipStream_t) {
    const int tokb = packed_tokb(D, p.R, p.q_split != 0);
    expect(packed_ok(p, D) && kv_dt != DT_F32 && tokb > 0 && (tokb & (tokb - 1)) == 0, "packed launch", p.T, D);
    expect(p.k_ts >= 0 && p.k_ts < 1 << 24 && p.v_ts >= 0 && p.v_ts < 1 << 24, "token strides", p.k_ts, p.v_ts);
    expect(packed_grid(p.T, p.B, p.G, tokb, 512, p.part_o != nullptr) > 0, "grid", p.T, p.B);
    return no();
}
static bool pages_in_range(int num_pages, int page_size, int max_pages) {
    return num_pages > 0 && page_size >= 16 && page_size % 16 == 0 && max_pages > 0 && (int64_t)max_pages * page_size <= INT_MAX;
}
static hipError_t paged(const PagedParams& p, int D) {
    expect(pages_in_range(p.num_pages, p.page_size, p.max_pages) && p.page_units * 16 == p.page_size, "paged launch", p.num_pages, p.page_size);
    expect(p.B > 0 && p.B <= 65535 && p.R * p.G == p.H && p.W == p.max_pages * p.page_size, "paged launch", p.B, p.W);
    expect(p.k_ps >= (int64_t)p.G * p.page_size * D && p.v_ps >= (int64_t)p.G * p.page_size * D, "page strides", p.k_ps, p.v_ps);
    expect((int64_t)p.B * p.G * ((p.W + 31ll) / 32) < 1ll << 31, "tiles", p.B, p.W);
    return no();
}
hipError_t launch_paged_generic(const PagedParams& p, int D, int, hipStream_t) { return paged(p, D); }
hipError_t launch_paged_decode(const PagedParams& p, int D, int, hipStream_t) { return paged(p, D); }
hipError_t launch_paged_append(const PagedAppendParams& p, hipStream_t) {
    expect(pages_in_range(p.num_pages, p.page_size, p.max_pages) && p.T > 0 && p.N > 0 && (int64_t)p.G * p.D < 1 << 24, "append launch", p.T, p.G);
    return no();
}
static hipError_t pool(const PagesParams& p, bool data) {
    expect(p.P > 0 && p.n >= 0 && p.n <= G4B_PAGES_MAX_LIST, "pages launch", p.P, p.n);
    if (data) expect(p.page_bytes > 0 && p.page_bytes % 16 == 0 && p.page_bytes <= 1ll << 31 && p.k_ps >= p.page_bytes && p.layers > 0, "pool", p.page_bytes, p.k_ps);
    return no();
}
static hipError_t tables(const PagesParams& p) {
    expect(p.S > 0 && p.max_pages > 0 && p.page_size > 0 && (int64_t)p.max_pages * p.page_size <= INT_MAX && p.table_s >= p.max_pages, "tables", p.S, p.max_pages);
    return no();
}
hipError_t launch_pages_copy(const PagesParams& p, hipStream_t) { return pool(p, true); }
hipError_t launch_pages_free(const PagesParams& p, hipStream_t) { return pool(p, false), tables(p); }
hipError_t launch_pages_fork(const PagesParams& p, hipStream_t) { return pool(p, true), tables(p); }
hipError_t launch_pages_allocate(const PagesParams& p, hipStream_t) { return pool(p, false), tables(p); }
hipError_t launch_pages_compact(const PagesParams& p, hipStream_t) { return pool(p, true), tables(p); }
}  // namespace g4b

static void answered(int rc, const char* what, long long field, long long value) {
    const bool known = rc == G4B_OK || rc == G4B_ERR_INVALID_ARGUMENT || rc == G4B_ERR_UNSUPPORTED || rc == G4B_ERR_WORKSPACE || rc == G4B_ERR_LAUNCH;
    expect(known && (rc == G4B_OK || strlen(g4b_last_error()) > 0), what, field, value);
}

// Every 4-byte word and every 8-byte word of a block, pointers among them, set to each of these values in turn.
template <class A, class F>
static void sweep(const A& good, const char* what, F call) {
    const long long values[] = {0, 1, -1, 2, 3, 7, 8, 15, 16, 17, 24, 128, 255, 256, 1024, 1032, 65535, 65536, 1 << 20, 1 << 24, 1 << 27, 1 << 28, 1 << 30,
                                INT_MAX, INT_MIN, 0x7fffff00ll, 1ll << 31, 1ll << 32, 1ll << 60, 1ll << 62, LLONG_MAX, LLONG_MIN, LLONG_MAX - 15};
    answered(call(good), what, -1, 0);
    for (size_t at = 0; at + 4 <= sizeof(A); at += 4)
        for (long long v : values) {
            A a = good;
            const int32_t w = (int32_t)v;
            if (v == w) {
                memcpy(reinterpret_cast<char*>(&a) + at, &w, 4);
                answered(call(a), what, (long long)at, v);
            }
            if (at % 8 == 0 && at + 8 <= sizeof(A)) {
                a = good;
                memcpy(reinterpret_cast<char*>(&a) + at, &v, 8);
                answered(call(a), what, (long long)at, v);
            }
        }
}

int main() {
    void* const fake = reinterpret_cast<void*>(4096);
    const int32_t* const ints = static_cast<const int32_t*>(fake);
    for (int D : {128, 256, 512, 64})
        for (int dt : {G4B_DT_F16, G4B_DT_F32}) {
            g4b_packed_attn_args a;
            memset(&a, 0, sizeof(a));
            a.q = a.k = a.v = a.o = fake;
            a.cu_seqlens = ints;
            for (int64_t* s : {a.q_stride, a.k_stride, a.v_stride, a.o_stride}) s[0] = 8 * D, s[1] = D, s[2] = 1;
            a.cu_seqlens_stride = 1, a.kv_dtype = dt, a.T = 900, a.N = 3, a.H = 8, a.G = 2, a.D = D, a.scale = 1.f;
            sweep(a, "packed", [](const g4b_packed_attn_args& x) { return g4b_packed_attn(&x, nullptr); });
            a.workspace = fake, a.workspace_bytes = g4b_packed_attn_workspace_bytes(900, 3, 8, 2, D);
            sweep(a, "packed with workspace", [](const g4b_packed_attn_args& x) { return g4b_packed_attn(&x, nullptr); });

            g4b_paged_attn_args b;
            memset(&b, 0, sizeof(b));
            b.q = b.o = fake, b.k_pages = b.v_pages = fake, b.block_tables = ints, b.seq_lens = ints;
            b.q_stride[0] = b.o_stride[0] = 8 * D, b.q_stride[1] = b.o_stride[1] = D, b.q_stride[2] = b.o_stride[2] = 1;
            b.k_page_stride = b.v_page_stride = 2 * 32 * D, b.block_tables_stride = 9, b.seq_lens_stride = b.user_phase_stride = 1;
            b.kv_dtype = dt, b.B = 5, b.H = 8, b.G = 2, b.D = D, b.num_pages = 40, b.page_size = 32, b.max_pages = 9, b.scale = 1.f;
            sweep(b, "paged", [](const g4b_paged_attn_args& x) { return g4b_paged_attn(&x, nullptr); });

            g4b_paged_append_args c;
            memset(&c, 0, sizeof(c));
            c.k = c.v = fake, c.k_pages = c.v_pages = fake, c.block_tables = ints, c.cache_offsets = ints;
            c.k_stride[0] = c.v_stride[0] = 2 * D, c.k_stride[1] = c.v_stride[1] = D, c.k_stride[2] = c.v_stride[2] = 1;
            c.k_page_stride = c.v_page_stride = 2 * 32 * D, c.block_tables_stride = 9, c.cache_offsets_stride = 1;
            c.cache_dtype = dt, c.T = c.N = 5, c.G = 2, c.D = D, c.num_pages = 40, c.page_size = 32, c.max_pages = 9;
            sweep(c, "append", [](const g4b_paged_append_args& x) { return g4b_paged_append(&x, nullptr); });

            g4b_pages_args d;
            memset(&d, 0, sizeof(d));
            d.k_pages = d.v_pages = fake, d.workspace = fake;
            d.block_tables = d.seq_lens = d.ref_counts = static_cast<int32_t*>(fake);
            d.src = d.dst = d.num_new = ints, d.page_map = d.status = static_cast<int32_t*>(fake);
            d.workspace_bytes = g4b_pages_workspace_bytes(40, 5);
            d.k_page_stride = d.v_page_stride = d.page_elems = 2 * 32 * D, d.k_layer_stride = d.v_layer_stride = 40ll * 2 * 32 * D;
            d.block_tables_stride = 9, d.cache_dtype = dt, d.layers = 2, d.num_pages = 40, d.page_size = 32, d.S = 5, d.max_pages = 9, d.n = 2;
            sweep(d, "copy", [](const g4b_pages_args& x) { return g4b_pages_copy(&x, nullptr); });
            sweep(d, "free", [](const g4b_pages_args& x) { return g4b_pages_free(&x, nullptr); });
            sweep(d, "fork", [](const g4b_pages_args& x) { return g4b_pages_fork(&x, nullptr); });
            sweep(d, "allocate", [](const g4b_pages_args& x) { return g4b_pages_allocate(&x, nullptr); });
            sweep(d, "compact", [](const g4b_pages_args& x) { return g4b_pages_compact(&x, nullptr); });
        }

    // the spans of a prompt's query tiles, with and without a window, against counting them
    for (int m = 1; m <= 40; ++m)
        for (int d : {0, 1, 2, 5, 16, 33, 0x3fffffff}) {
            const float inv = 1.f / (float)m;
            int spans = 0;
            for (int t = 0; t < 300; ++t) {
                expect(g4b::packed_spans(t, m, inv, d) == spans, "spans", t, m);
                const int first = t > d ? t - d : 0;  // the tile sees keys of tiles first .. t
                spans += t / m - first / m + 1;
            }
        }
    // what the plan kernels of fork and compaction lay out in a workspace
    for (long long P : {1ll, 2ll, 4095ll, 4096ll, 4097ll, 1ll << 27})
        for (long long S : {1ll, 7ll, 1ll << 18}) {
            const long long words = g4b::pages_workspace_words(P, S);
            expect(16 + 2 * S + P <= words && 16 + S + 1 + P <= words, "fork and allocation lists", P, S);
            expect(16 + 2 * ((P + 1) / 2) + (P + 4095) / 4096 <= words, "compaction lists", P, S);
        }
    printf("%ld checks, %ld bad\n", checks, bad);
    return bad ? 1 : 0;
}

// C ABI of libg4b_attn.so: argument validation on the host, then dispatch to the gfx950 kernels.
// Nothing here allocates, synchronises or reads device memory.
#include "../../include/g4b_attn.h"

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <mutex>
#include <utility>
#include <vector>

#include "api_common.hpp"
#include "launch.hpp"
#include "prefill_combine.hpp"
#include "prefill_map.hpp"

// Scratch of g4b_attn_forward_static_scratch: split partials of one launch.  Every device the library runs on holds
// its own copy of this array at its own address until the process ends; host code reaches it only through the
// per-device pointer that static_scratch_ptr() obtains with hipGetSymbolAddress.
constexpr size_t kStaticScratchBytes = (size_t)G4B_ATTN_STATIC_SCRATCH_BYTES;
static __device__ __align__(256) unsigned char scratch[kStaticScratchBytes];

// Which XCD the workgroups of a launch run on.  The streaming kernels give the workers on even XCDs a larger share
// (the odd ones stream from HBM more slowly), which only helps while workgroup i of a grid runs on an XCD of the parity
// of i; nothing documents that order, so it is read from the hardware once per device: 64 workgroups write the XCC id
// their wave reports (HW_REG_XCC_ID), the host looks at the parities.
constexpr int kXcdProbeGroups = 64;
static __device__ int32_t xcd_probe_ids[kXcdProbeGroups];
__global__ void xcd_probe_kernel(int32_t* ids) {
    if (threadIdx.x == 0) {
        uint32_t x;
        asm volatile("s_getreg_b32 %0, hwreg(HW_REG_XCC_ID, 0, 4)" : "=s"(x));
        ids[blockIdx.x] = (int32_t)x;
    }
}

namespace {

thread_local char g_err[512] = "";

constexpr int kMaxDevices = 64;
std::mutex g_scratch_mutex;
void* g_scratch_ptr[kMaxDevices] = {};
// The stream whose launches last used the array on each device.  A launch on another stream may only follow when
// everything enqueued on that stream has finished (two launches in flight would write their partials over each other's).
struct ScratchOwner {
    hipStream_t stream = nullptr;
    bool valid = false;
};
ScratchOwner g_scratch_owner[kMaxDevices];

// Device address of `scratch` on the current device, looked up once per device.
hipError_t static_scratch_ptr(void** out) {
    int dev = -1;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    if (dev < 0 || dev >= kMaxDevices) return hipErrorInvalidDevice;
    std::lock_guard<std::mutex> lock(g_scratch_mutex);
    if (!g_scratch_ptr[dev]) {
        void* ptr = nullptr;
        e = hipGetSymbolAddress(&ptr, HIP_SYMBOL(scratch));
        if (e != hipSuccess) return e;
        if (!ptr) return hipErrorInvalidSymbol;
        g_scratch_ptr[dev] = ptr;
    }
    *out = g_scratch_ptr[dev];
    return hipSuccess;
}

// Claim the array of the current device for a launch on `stream`: true when the launch may use it.  A launch that is
// being recorded into a graph is let through untracked (when it will run is not known here; whoever replays the graph
// keeps it apart from other launches that use the array).
bool claim_static_scratch(hipStream_t stream) {
    int dev = -1;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) return true;
    std::lock_guard<std::mutex> lock(g_scratch_mutex);
    ScratchOwner& o = g_scratch_owner[dev];
    if (o.valid && o.stream == stream) return true;  // the common case costs no runtime call
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(stream, &cs) == hipSuccess && cs == hipStreamCaptureStatusActive) return true;
    if (o.valid) {
        const hipError_t e = hipStreamQuery(o.stream);
        if (e == hipErrorNotReady) return false;
        if (e != hipSuccess) (void)hipGetLastError();  // the stream is gone: nothing of it is pending
    }
    o.stream = stream;
    o.valid = true;
    return true;
}

// Environment switches, read once (the reference has G4B_FA_FORCE_CONFIG and G4B_FA_PRINT_CONFIG for an engine whose
// call sites cannot be changed, g4b/kernels/fa2.py:148-150,691-700):
//   G4B_ATTN_NUM_WORKERS=n   worker count of decode-shaped launches that pass num_workers = 0 (also sizes the workspace)
//   G4B_ATTN_XCD_SHARES=0|1  0: equal shares for all workers; 1: the weighted shares without asking the hardware
//   G4B_ATTN_PRINT_PLAN=1    one line on stderr per attention launch: kernel family, grid, workers, key splits
struct EnvSwitches {
    int num_workers = 0;
    int xcd_shares = -1;  // -1: ask the hardware
    bool print_plan = false;
    EnvSwitches() {
        if (const char* v = getenv("G4B_ATTN_NUM_WORKERS")) {
            const long n = strtol(v, nullptr, 10);
            if (n >= 1 && n <= (1 << 20)) num_workers = (int)n;
        }
        if (const char* v = getenv("G4B_ATTN_XCD_SHARES")) xcd_shares = (v[0] == '0') ? 0 : 1;
        if (const char* v = getenv("G4B_ATTN_PRINT_PLAN")) print_plan = v[0] != '\0' && v[0] != '0';
    }
};
const EnvSwitches& env_switches() {
    static const EnvSwitches e;
    return e;
}

// 1 when workgroup i of a grid runs on an XCD of the parity of i on the current device, else 0.  Asked once per device,
// by the first launch that wants to know outside stream capture (it waits for the 64-workgroup probe: the one place
// where this library synchronises); launches recorded into a graph before that are told 0 and keep equal shares.
enum : int { XCD_UNKNOWN = 0, XCD_PARITY = 1, XCD_OTHER = 2 };
int g_xcd_state[kMaxDevices] = {};
int32_t g_xcd_ids[kMaxDevices][kXcdProbeGroups];
int xcd_parity_known(hipStream_t stream) {
    const EnvSwitches& env = env_switches();
    if (env.xcd_shares >= 0) return env.xcd_shares;
    int dev = -1;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= kMaxDevices) return 0;
    std::lock_guard<std::mutex> lock(g_scratch_mutex);
    if (g_xcd_state[dev] != XCD_UNKNOWN) return g_xcd_state[dev] == XCD_PARITY;
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(stream, &cs) != hipSuccess || cs != hipStreamCaptureStatusNone) return 0;
    void* ids = nullptr;
    int state = XCD_OTHER;
    if (hipGetSymbolAddress(&ids, HIP_SYMBOL(xcd_probe_ids)) == hipSuccess && ids) {
        hipLaunchKernelGGL(xcd_probe_kernel, dim3(kXcdProbeGroups), dim3(64), 0, stream, static_cast<int32_t*>(ids));
        if (hipGetLastError() == hipSuccess &&
            hipMemcpyAsync(g_xcd_ids[dev], ids, sizeof(g_xcd_ids[dev]), hipMemcpyDeviceToHost, stream) == hipSuccess &&
            hipStreamSynchronize(stream) == hipSuccess) {
            state = XCD_PARITY;
            for (int i = 0; i < kXcdProbeGroups; ++i)
                if ((g_xcd_ids[dev][i] & 1) != (i & 1)) state = XCD_OTHER;
        }
    }
    if (state == XCD_OTHER) (void)hipGetLastError();
    g_xcd_state[dev] = state;
    if (env.print_plan) {
        fprintf(stderr, "g4b_attn: XCC ids of workgroups 0..15 on device %d:", dev);
        for (int i = 0; i < 16; ++i) fprintf(stderr, " %d", g_xcd_ids[dev][i]);
        fprintf(stderr, " -> %s shares\n", state == XCD_PARITY ? "weighted" : "equal");
    }
    return state == XCD_PARITY;
}

// g4b_profile_begin .. g4b_profile_end: one (start, stop) event pair per timed call of this thread
thread_local bool g_profiling = false;
thread_local std::vector<std::pair<hipEvent_t, hipEvent_t>> g_profile_records;

// Arm the events for the dominant kernel of the launcher call that follows; false if they cannot be created.
bool profile_arm() {
    if (!g_profiling) return true;
    hipEvent_t a = nullptr, b = nullptr;
    if (hipEventCreate(&a) != hipSuccess || hipEventCreate(&b) != hipSuccess) {
        if (a) (void)hipEventDestroy(a);
        return false;
    }
    g_profile_records.emplace_back(a, b);
    g4b::g_profile_events = g4b::ProfileEvents{a, b};
    return true;
}
// After the launcher: events nobody consumed (the dominant kernel was masked out) mark an untimed call.
void profile_disarm() {
    if (g4b::g_profile_events.start) {
        (void)hipEventDestroy(g_profile_records.back().first);
        (void)hipEventDestroy(g_profile_records.back().second);
        g_profile_records.back() = {nullptr, nullptr};
        g4b::g_profile_events = g4b::ProfileEvents{};
    }
}

constexpr int kDefaultWorkers = 1024;  // 256 CUs x 4 SIMDs x 1 wave
// a worker for head dimension 512 is a workgroup of two waves
int default_workers(int D) {
    if (env_switches().num_workers > 0) return env_switches().num_workers;
    return D > 256 ? kDefaultWorkers * 256 / D : kDefaultWorkers;
}
constexpr int kMaxDecodeRows = 16;
using g4b::api::aligned16;
using g4b::api::decode_slots;
using g4b::api::dtype_ok;
using g4b::api::fail;

// Prefill-shaped launches: how many (active slot, key split) pairs the partial buffers hold.  A launch whose in-phase
// slots bring fewer workgroups than the chip has CUs splits the keys of every item; 0 = the shape never splits.
constexpr int kPrefillFillWorkgroups = 256;
constexpr int kPrefillMaxSplitSlots = 64;
int prefill_rows_per_workgroup(int /*D*/) { return 128; }
// A slot that brings at least a third as many query tiles as the chip has compute units is not split tile by tile
// (under the causal mask equal splits of every tile leave the launch as long as half of its heaviest tile); the
// 128 / 256 kernel pairs its query tiles instead and cuts the key tiles of every pair into two to five spans of equal
// cost (measured, one slot, causal from an empty cache: S = 1408 31.5 -> 25.2 us, S = 2048 38.9 -> 33.9 us,
// S = 3072 95 -> 55 us, S = 4096 119 -> 78 us; shorter prompts measured worse that way, S = 1280 32.0 -> 33.6 us wall
// and S = 1024 30.2 -> 33.4 us, for the wider merge).  The 512 kernel gives every workgroup one query tile.
bool prefill_pair_split(int H, int G, int Tq, int D) {
    const int R = H / G, bm = prefill_rows_per_workgroup(D);
    if (D == 512 || R < 1 || bm % R) return false;
    const int tokb = bm / R, nq = (Tq + tokb - 1) / tokb;
    return (int64_t)nq * G * 3 >= kPrefillFillWorkgroups && (int64_t)((nq + 1) / 2) * G * 2 <= kPrefillFillWorkgroups;
}
// One (slot, key split) pair of a prefill-shaped launch: its rows in the cache's 16-bit type, normalised by the split's
// own sum, then (reference, sum) per row in fp32.
uint64_t prefill_partial_bytes(int H, int Tq, int D) { return (uint64_t)H * (uint64_t)Tq * ((uint64_t)D * 2 + 2 * sizeof(float)); }
float* prefill_partial_sums(void* workspace, int slots, int H, int Tq, int D) {
    return reinterpret_cast<float*>(static_cast<char*>(workspace) + (uint64_t)slots * H * Tq * D * 2);
}
int prefill_split_slots(int H, int G, int Tq, int D) {
    const int R = H / G, bm = prefill_rows_per_workgroup(D);
    if (R < 1 || bm % R) return 0;
    const int tokb = bm / R;
    const int nq = (Tq + tokb - 1) / tokb;
    const int64_t per_slot = (int64_t)(prefill_pair_split(H, G, Tq, D) ? (nq + 1) / 2 : nq) * G;  // workgroups one slot brings
    int64_t slots = kPrefillFillWorkgroups / per_slot;
    // one query tile per workgroup and more than half of the units taken: under the causal mask the tiles' work grows
    // linearly, so the launch takes as long as its last tile while the chip is half idle; two spans per tile halve that
    if (slots < 2 && per_slot <= kPrefillFillWorkgroups && !prefill_pair_split(H, G, Tq, D)) slots = 2;
    if (slots < 2) return 0;
    return (int)(slots < kPrefillMaxSplitSlots ? slots : kPrefillMaxSplitSlots);
}
uint64_t prefill_workspace_bytes(int H, int G, int Tq, int D) {
    return (uint64_t)prefill_split_slots(H, G, Tq, D) * prefill_partial_bytes(H, Tq, D);
}

}  // namespace

namespace g4b::api {
int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
    return code;
}
int default_decode_workers(int D) { return default_workers(D); }
bool print_plan() { return env_switches().print_plan; }
bool xcd_parity(hipStream_t stream) { return xcd_parity_known(stream) != 0; }
bool arm_profile() { return profile_arm(); }
void disarm_profile() { profile_disarm(); }
}  // namespace g4b::api

extern "C" {

const char* g4b_last_error(void) { return g_err; }

int g4b_profile_begin(void) {
    if (g_profiling) return fail(G4B_ERR_INVALID_ARGUMENT, "g4b_profile_begin: already profiling on this thread");
    g_profile_records.clear();
    g_profiling = true;
    return G4B_OK;
}

int g4b_profile_end(float* ms, int32_t capacity) {
    if (!g_profiling) return fail(G4B_ERR_INVALID_ARGUMENT, "g4b_profile_end without g4b_profile_begin");
    g_profiling = false;
    int n = 0;
    hipError_t first_err = hipSuccess;
    for (auto& r : g_profile_records) {
        float t = -1.f;
        if (r.first) {
            hipError_t e = hipEventSynchronize(r.second);
            if (e == hipSuccess) e = hipEventElapsedTime(&t, r.first, r.second);
            if (e != hipSuccess) {
                t = -1.f;
                if (first_err == hipSuccess) first_err = e;
            }
            (void)hipEventDestroy(r.first);
            (void)hipEventDestroy(r.second);
        }
        if (ms && n < capacity) ms[n] = t;
        ++n;
    }
    g_profile_records.clear();
    if (first_err != hipSuccess) return fail(G4B_ERR_LAUNCH, "profiling events: %s", hipGetErrorString(first_err));
    return n;
}
int32_t g4b_abi_version(void) { return G4B_ATTN_ABI_VERSION; }
int32_t g4b_attn_default_workers(void) { return default_workers(256); }

uint64_t g4b_attn_workspace_bytes(int32_t B, int32_t H, int32_t G, int32_t Tq, int32_t D, int32_t num_workers) {
    if (B < 1 || H < 1 || G < 1 || Tq < 1 || D < 1 || H % G) return 0;
    if (D != 128 && D != 256 && D != 512) return 0;  // the plain fp32 kernel never splits
    const int64_t rows = (int64_t)(H / G) * Tq;
    if (rows > kMaxDecodeRows) return prefill_workspace_bytes(H, G, Tq, D);
    const int nw = num_workers > 0 ? num_workers : default_workers(D);
    return decode_slots(B, G, nw) * (uint64_t)rows * (uint64_t)(D + 2) * sizeof(float);
}

// Shapes and types the tuned kernels are not built for go to the plain fp32 kernel (attn_generic.hip): an fp32 cache,
// STAGE_ON_BAND alone, head dimensions other than 128 / 256 / 512, and prefill-shaped launches whose H/G does not
// divide a workgroup's query rows.  It never uses a workspace.
static bool takes_generic_path(const g4b_attn_args* a) {
    if (a->kv_dtype == G4B_DT_F32 || a->stage == G4B_STAGE_ON_BAND) return true;
    if (a->D != 128 && a->D != 256 && a->D != 512) return true;
    const int R = a->H / a->G;
    if ((int64_t)R * a->Tq <= kMaxDecodeRows) return false;
    const bool q_wider = a->q_dtype == G4B_DT_F32 || (a->q_dtype == G4B_DT_F16 && a->kv_dtype == G4B_DT_BF16);
    const int bm = prefill_rows_per_workgroup(a->D) / ((a->D == 512 && a->use_fp32_dot && q_wider) ? 2 : 1);
    return bm % R != 0;
}

// Host-side validation of one argument block and its translation into kernel parameters (everything except the
// workspace, which depends on the kind of launch).
static int fill_attn_params(const g4b_attn_args* a, g4b::AttnParams& p) {
    if (!a) return fail(G4B_ERR_INVALID_ARGUMENT, "args is NULL");
    if (!a->q || !a->k_cache || !a->v_cache || !a->o || !a->time_dim_sizes || !a->user_phase)
        return fail(G4B_ERR_INVALID_ARGUMENT, "q, k_cache, v_cache, o, time_dim_sizes and user_phase must be non-NULL");
    if (!dtype_ok(a->q_dtype) || !dtype_ok(a->o_dtype))
        return fail(G4B_ERR_INVALID_ARGUMENT, "q/o dtype must be f16, bf16 or f32 (got %d, %d)", a->q_dtype, a->o_dtype);
    if (!dtype_ok(a->kv_dtype)) return fail(G4B_ERR_INVALID_ARGUMENT, "KV cache dtype must be f16, bf16 or f32 (got %d)", a->kv_dtype);
    if (a->B < 1 || a->H < 1 || a->G < 1 || a->Tq < 1 || a->D < 1 || a->KV_CTX < 1)
        return fail(G4B_ERR_INVALID_ARGUMENT, "B, H, G, Tq, D, KV_CTX must be positive");
    if (a->H % a->G) return fail(G4B_ERR_INVALID_ARGUMENT, "H (%d) must be a multiple of G (%d)", a->H, a->G);
    if (a->D % 8 || a->D > 1024)
        return fail(G4B_ERR_UNSUPPORTED, "head_dim must be a multiple of 8 and at most 1024 (got %d)", a->D);
    if (a->B > 65535 || a->G > 65535) return fail(G4B_ERR_UNSUPPORTED, "B and G must be <= 65535");
    if (a->ctx_window_size < 1 || a->ctx_window_size > a->KV_CTX)
        return fail(G4B_ERR_INVALID_ARGUMENT, "ctx_window_size (%d) must be in [1, KV_CTX = %d]", a->ctx_window_size, a->KV_CTX);
    if (a->stage != G4B_STAGE_FULL && a->stage != G4B_STAGE_CAUSAL && a->stage != G4B_STAGE_ON_BAND)
        return fail(G4B_ERR_INVALID_ARGUMENT, "stage must be STAGE_FULL (1), STAGE_ON_BAND (2) or STAGE_CAUSAL (3), got %d", a->stage);
    if (a->stage == G4B_STAGE_ON_BAND && a->on_band_block < 1)
        return fail(G4B_ERR_INVALID_ARGUMENT, "STAGE_ON_BAND alone needs on_band_block >= 1 (the reference's Q_BLOCKSIZE_T)");
    if (a->phase < 0 || a->phase > 255) return fail(G4B_ERR_INVALID_ARGUMENT, "phase must fit uint8");
    if (a->query_window < 0) return fail(G4B_ERR_INVALID_ARGUMENT, "query_window must be >= 0");
    if (!std::isfinite(a->scale) || !(a->scale > 0.f)) return fail(G4B_ERR_INVALID_ARGUMENT, "scale must be finite and positive");
    if (a->q_stride[3] != 1 || a->o_stride[3] != 1)
        return fail(G4B_ERR_INVALID_ARGUMENT, "q and o must have unit stride in the head dimension");
    for (int i = 0; i < 3; ++i)
        if (a->q_stride[i] % 8 || a->o_stride[i] % 8)
            return fail(G4B_ERR_INVALID_ARGUMENT, "q/o strides must be multiples of 8 elements (16-byte vector access)");
    if (!aligned16(a->q) || !aligned16(a->o) || !aligned16(a->k_cache) || !aligned16(a->v_cache))
        return fail(G4B_ERR_INVALID_ARGUMENT, "q, o, k_cache, v_cache must be 16-byte aligned");
    const int64_t slot_elems = (int64_t)a->G * a->KV_CTX * a->D;
    if (a->k_stride_b < slot_elems || a->v_stride_b < slot_elems || a->k_stride_b % 8 || a->v_stride_b % 8)
        return fail(G4B_ERR_INVALID_ARGUMENT, "cache slot stride must be >= G*KV_CTX*D and a multiple of 8 elements");
    if ((int64_t)a->KV_CTX * a->D * (a->kv_dtype == G4B_DT_F32 ? 4 : 2) >= (int64_t)1 << 31)
        return fail(G4B_ERR_UNSUPPORTED, "one (slot, kv head) of the cache must stay below 2 GiB");
    if (a->num_workers < 0 || a->num_workers > (1 << 20)) return fail(G4B_ERR_INVALID_ARGUMENT, "num_workers out of range");
    // the streaming kernels count the 32-key tiles of all (slot, kv head) pairs in 32 bits
    if ((int64_t)a->B * a->G * (((int64_t)a->KV_CTX + 31) / 32) >= (int64_t)1 << 31)
        return fail(G4B_ERR_UNSUPPORTED, "B * G * ceil(KV_CTX / 32) must stay below 2^31");

    p = g4b::AttnParams{};
    p.q = a->q;
    p.k = a->k_cache;
    p.v = a->v_cache;
    p.o = a->o;
    p.tds = a->time_dim_sizes;
    p.phase_arr = a->user_phase;
    p.win_arr = a->window_sizes;
    for (int i = 0; i < 4; ++i) {
        p.q_s[i] = a->q_stride[i];
        p.o_s[i] = a->o_stride[i];
    }
    p.k_sb = a->k_stride_b;
    p.v_sb = a->v_stride_b;
    p.tds_s = a->time_dim_sizes_stride;
    p.ph_s = a->user_phase_stride;
    p.win_s = a->window_sizes_stride;
    p.q_dt = a->q_dtype;
    p.o_dt = a->o_dtype;
    p.B = a->B;
    p.H = a->H;
    p.G = a->G;
    p.R = a->H / a->G;
    p.Tq = a->Tq;
    p.KV_CTX = a->KV_CTX;
    p.W = a->ctx_window_size;
    p.phase = a->phase;
    p.stage = a->stage;
    p.qwin = a->query_window;
    p.c = a->scale * 1.44269504088896340736f;
    p.kernel_mask = (a->kernel_mask & 3) ? (a->kernel_mask & 3) : 3;
    // a query wider than the cache type: f32 over f16 / bf16, f16 over bf16
    const bool q_wider = a->q_dtype == G4B_DT_F32 || (a->q_dtype == G4B_DT_F16 && a->kv_dtype == G4B_DT_BF16);
    p.q_split = (a->use_fp32_dot && q_wider) ? 1 : 0;
    p.xcd_shift = -1;  // equal shares; the decode launch asks xcd_parity_known()
    return G4B_OK;
}

int g4b_attn_forward(const g4b_attn_args* a, void* stream) {
    g4b::AttnParams p;
    if (const int rc = fill_attn_params(a, p)) return rc;
    const int64_t rows = (int64_t)p.R * p.Tq;
    hipError_t e;
    if (takes_generic_path(a)) {
        if ((int64_t)a->B * a->H * a->Tq > 0x7fffffffLL) return fail(G4B_ERR_UNSUPPORTED, "B * H * Tq must be below 2^31 on this path");
        if (env_switches().print_plan)
            fprintf(stderr, "g4b_attn plan: B=%d H=%d G=%d Tq=%d D=%d: plain fp32 kernel\n", a->B, a->H, a->G, a->Tq, a->D);
        if (!profile_arm()) return fail(G4B_ERR_LAUNCH, "could not create profiling events");
        e = g4b::launch_attn_generic(p, a->D, a->kv_dtype, a->on_band_block, static_cast<hipStream_t>(stream));
    } else if (rows <= kMaxDecodeRows) {
        if (a->workspace) {
            const int nw = a->num_workers > 0 ? a->num_workers : default_workers(a->D);
            const uint64_t need = g4b_attn_workspace_bytes(a->B, a->H, a->G, a->Tq, a->D, nw);
            if (a->workspace_bytes < need)
                return fail(G4B_ERR_WORKSPACE, "workspace holds %llu bytes, %llu needed for %d workers",
                            (unsigned long long)a->workspace_bytes, (unsigned long long)need, nw);
            if (!aligned16(a->workspace)) return fail(G4B_ERR_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
            p.NW = nw;
            p.part_o = static_cast<float*>(a->workspace);
            p.part_ml = p.part_o + decode_slots(a->B, a->G, nw) * (uint64_t)rows * (uint64_t)a->D;
        } else {
            p.NW = 0;  // one wave per (slot, kv head), no partials
        }
        // the decode kernels proper have one worker per workgroup: weighted shares where workgroup i runs on an XCD of
        // the parity of i
        if (p.NW > 0 && xcd_parity_known(static_cast<hipStream_t>(stream))) p.xcd_shift = 0;
        if (env_switches().print_plan)
            fprintf(stderr, "g4b_attn plan: decode B=%d H=%d G=%d Tq=%d D=%d KV_CTX=%d W=%d: %s, %d workers, %s shares%s\n", a->B, a->H,
                    a->G, a->Tq, a->D, a->KV_CTX, a->ctx_window_size,
                    g4b::decode_pair_path(p, a->D) ? "one kernel, a workgroup per (slot, kv head)" : (p.NW > 0 ? "flat tile list + merge kernel" : "a wave per (slot, kv head)"),
                    p.NW, p.xcd_shift >= 0 ? "weighted" : "equal", a->workspace ? "" : ", no workspace");
        if (!profile_arm()) return fail(G4B_ERR_LAUNCH, "could not create profiling events");
        e = g4b::launch_attn_decode(p, a->D, a->kv_dtype, static_cast<hipStream_t>(stream));
    } else {
        p.split_slots = 0;
        const uint64_t need = prefill_workspace_bytes(a->H, a->G, a->Tq, a->D);
        if (a->workspace && need) {
            if (a->workspace_bytes < need)
                return fail(G4B_ERR_WORKSPACE, "workspace holds %llu bytes, %llu needed to split this prefill shape",
                            (unsigned long long)a->workspace_bytes, (unsigned long long)need);
            if (!aligned16(a->workspace)) return fail(G4B_ERR_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
            p.split_slots = prefill_split_slots(a->H, a->G, a->Tq, a->D);
            p.pair_split = prefill_pair_split(a->H, a->G, a->Tq, a->D) ? 1 : 0;
            p.part_o = static_cast<float*>(a->workspace);
            p.part_ml = prefill_partial_sums(a->workspace, p.split_slots, a->H, a->Tq, a->D);
        }
        if (env_switches().print_plan)
            fprintf(stderr, "g4b_attn plan: prefill B=%d H=%d G=%d Tq=%d D=%d KV_CTX=%d W=%d: grid %d, up to %d (slot, key split) pairs%s\n",
                    a->B, a->H, a->G, a->Tq, a->D, a->KV_CTX, a->ctx_window_size,
                    g4b::prefill_grid(p, a->D == 512 && p.q_split ? 64 : 128, a->D != 512), p.split_slots,
                    p.pair_split ? ", pairs of query tiles cut into key spans" : "");
        if (!profile_arm()) return fail(G4B_ERR_LAUNCH, "could not create profiling events");
        e = a->D == 512 ? g4b::launch_attn_prefill_wide(p, a->kv_dtype, static_cast<hipStream_t>(stream))
                        : g4b::launch_attn_prefill(p, a->D, a->kv_dtype, static_cast<hipStream_t>(stream));
    }
    profile_disarm();
    if (e != hipSuccess) return fail(G4B_ERR_LAUNCH, "attention launch failed: %s", hipGetErrorString(e));
    return G4B_OK;
}

// ---- one launch for a mixed step ----------------------------------------------------------------------------------
// The chip's 256 compute units are shared out between the two halves on the host, from static shapes only: the decode
// half gets what lets its stream run at full rate, the chunk the rest.
namespace {
constexpr int kMixedCus = 256;
// Decode workgroups asked for by default (the prefill half then takes as many whole key splits as fit and the decode
// half what is left): four one-wave workers each at head dimension 256, one four-wave worker each at 512.  Measured
// on the benchmark's global layers, main kernel: head dim 256 with 96 decode workgroups (five key splits of the chunk)
// 151 us, 100..128 (four splits) 138..147 us, 160 169 us; head dim 512 with 104 348 us, 120 320 us, 128 312 us, 136 348 us.
constexpr int kMixedDecodeBlocks = 112;
constexpr int kMixedDecodeBlocksWide = 112;

struct MixedShape {
    int split_slots;     // (active slot, key split) pairs of the prefill half; <= 1 = unsplit
    g4b::MixedPlan plan;
    int nw;              // decode workers (0 with the pair path or without a workspace)
    uint64_t pf_bytes, dec_bytes;
};

// B, H, G, D, KV_CTX, W, window_sizes are shared; tq_pf / tq_dec are the query tokens per slot of the two halves;
// pf_rows = query rows of a prefill workgroup.
MixedShape mixed_shape(int B, int H, int G, int D, int tq_pf, int tq_dec, bool pair_path, int num_workers, bool with_ws,
                       int pf_rows = 128) {
    MixedShape m{};
    const int R = H / G, tokb = pf_rows / R;
    const int wpb = D == 512 ? 1 : 4;                      // decode workers per workgroup
    const int per_slot = ((tq_pf + tokb - 1) / tokb) * G;  // prefill workgroups one slot brings unsplit
    int nd = pair_path ? B * G : (num_workers > 0 ? (num_workers + wpb - 1) / wpb : (D == 512 ? kMixedDecodeBlocksWide : kMixedDecodeBlocks));
    if (!with_ws && !pair_path) nd = (B * G + wpb - 1) / wpb;  // one worker per pair
    int slots = with_ws ? (kMixedCus - nd) / per_slot : 1;
    slots = slots < 1 ? 1 : (slots > kPrefillMaxSplitSlots ? kPrefillMaxSplitSlots : slots);
    if (!pair_path && with_ws && num_workers <= 0 && slots * per_slot + nd < kMixedCus) nd = kMixedCus - slots * per_slot;
    m.split_slots = slots >= 2 ? slots : 0;
    m.nw = (pair_path || !with_ws) ? 0 : nd * wpb;
    m.plan.nd_blocks = nd;
    m.plan.pair_path = pair_path ? 1 : 0;
    m.pf_bytes = (uint64_t)m.split_slots * prefill_partial_bytes(H, tq_pf, D);
    m.dec_bytes = m.nw ? decode_slots(B, G, m.nw) * (uint64_t)R * tq_dec * (uint64_t)(D + 2) * sizeof(float) : 0;
    return m;
}
}  // namespace

uint64_t g4b_attn_mixed_workspace_bytes(int32_t B, int32_t H, int32_t G, int32_t Tq_prefill, int32_t Tq_decode, int32_t D,
                                        int32_t KV_CTX, int32_t ctx_window_size, int32_t has_window_sizes, int32_t num_workers) {
    if (B < 1 || H < 1 || G < 1 || Tq_prefill < 1 || Tq_decode < 1 || D < 1 || H % G || 128 % (H / G)) return 0;
    const int W = ctx_window_size < KV_CTX ? ctx_window_size : KV_CTX;
    const bool pair = D <= 256 && !has_window_sizes && W <= g4b::DEC_PAIR_MAX_KEYS;
    const MixedShape m = mixed_shape(B, H, G, D, Tq_prefill, Tq_decode, pair, num_workers, true);
    uint64_t need = ((m.pf_bytes + 255) & ~(uint64_t)255) + m.dec_bytes;
    if (D == 512 && 64 % (H / G) == 0) {
        // a split query (fp32 q with use_fp32_dot) halves the rows of a prefill workgroup, which can move the share-out
        const MixedShape h = mixed_shape(B, H, G, D, Tq_prefill, Tq_decode, pair, num_workers, true, 64);
        const uint64_t need_h = ((h.pf_bytes + 255) & ~(uint64_t)255) + h.dec_bytes;
        need = need_h > need ? need_h : need;
    }
    return need;
}

int g4b_attn_forward_mixed(const g4b_attn_args* prefill, const g4b_attn_args* decode, void* stream) {
    g4b::AttnParams pp, pd;
    if (const int rc = fill_attn_params(prefill, pp)) return rc;
    if (const int rc = fill_attn_params(decode, pd)) return rc;
    const g4b_attn_args *a = prefill, *d = decode;
    if (a->k_cache != d->k_cache || a->v_cache != d->v_cache || a->time_dim_sizes != d->time_dim_sizes ||
        a->user_phase != d->user_phase || a->window_sizes != d->window_sizes || a->B != d->B || a->H != d->H || a->G != d->G ||
        a->D != d->D || a->KV_CTX != d->KV_CTX || a->kv_dtype != d->kv_dtype || a->ctx_window_size != d->ctx_window_size ||
        a->k_stride_b != d->k_stride_b || a->v_stride_b != d->v_stride_b || a->time_dim_sizes_stride != d->time_dim_sizes_stride ||
        a->user_phase_stride != d->user_phase_stride || a->window_sizes_stride != d->window_sizes_stride)
        return fail(G4B_ERR_INVALID_ARGUMENT, "the two halves of a mixed launch must share the caches, the per-slot arrays, "
                    "B, H, G, D, KV_CTX, the cache dtype and ctx_window_size");
    if (a->phase == d->phase) return fail(G4B_ERR_INVALID_ARGUMENT, "the two halves of a mixed launch serve different phases");
    if ((int64_t)pp.R * pp.Tq <= kMaxDecodeRows || (int64_t)pd.R * pd.Tq > kMaxDecodeRows)
        return fail(G4B_ERR_INVALID_ARGUMENT, "mixed launch: the first block must be prefill-shaped ((H/G)*Tq > %d), the second "
                    "decode-shaped", kMaxDecodeRows);
    if (a->D != 256 && a->D != 512) return fail(G4B_ERR_UNSUPPORTED, "mixed launch is built for head_dim 256 and 512 (got %d)", a->D);
    if (a->kv_dtype == G4B_DT_F32 || a->stage == G4B_STAGE_ON_BAND || d->stage == G4B_STAGE_ON_BAND)
        return fail(G4B_ERR_UNSUPPORTED, "mixed launch is built for f16 / bf16 caches and the causal and full stages");
    // a split query halves the rows of a head-dimension-512 prefill workgroup
    const int pf_rows = prefill_rows_per_workgroup(a->D) / ((a->D == 512 && pp.q_split) ? 2 : 1);
    if (pf_rows % pp.R) return fail(G4B_ERR_UNSUPPORTED, "H/G = %d must divide %d for this prefill shape", pp.R, pf_rows);
    if (pp.q_split != pd.q_split)
        return fail(G4B_ERR_UNSUPPORTED, "mixed launch: both halves must take the same query precision path (same q dtype and use_fp32_dot)");
    if (a->kernel_mask != d->kernel_mask) return fail(G4B_ERR_INVALID_ARGUMENT, "mixed launch: kernel_mask must agree");

    const bool pair = g4b::decode_pair_path(pd, a->D);
    const bool with_ws = a->workspace != nullptr;
    const MixedShape m = mixed_shape(a->B, a->H, a->G, a->D, a->Tq, d->Tq, pair, d->num_workers, with_ws, pf_rows);
    if (with_ws) {
        // one workspace, passed with the prefill block: the chunk's partials first, the decode partials after them
        const uint64_t pf_span = (m.pf_bytes + 255) & ~(uint64_t)255;
        if (a->workspace_bytes < pf_span + m.dec_bytes)
            return fail(G4B_ERR_WORKSPACE, "workspace holds %llu bytes, %llu needed for this mixed launch",
                        (unsigned long long)a->workspace_bytes, (unsigned long long)(pf_span + m.dec_bytes));
        if (!aligned16(a->workspace)) return fail(G4B_ERR_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
        if (m.split_slots) {
            pp.split_slots = m.split_slots;
            pp.part_o = static_cast<float*>(a->workspace);
            pp.part_ml = prefill_partial_sums(a->workspace, m.split_slots, a->H, a->Tq, a->D);
        }
        if (m.nw) {
            pd.NW = m.nw;
            pd.xcd_shift = -1;  // the workers of a mixed launch share their workgroups and the chip with the chunk: equal shares
            pd.part_o = reinterpret_cast<float*>(static_cast<char*>(a->workspace) + pf_span);
            pd.part_ml = pd.part_o + decode_slots(a->B, a->G, m.nw) * (uint64_t)pd.R * pd.Tq * (uint64_t)a->D;
        }
    }
    g4b::MixedPlan mp = m.plan;
    mp.npx = (g4b::prefill_grid(pp, pf_rows, a->D != 512) + 7) / 8;
    mp.combine_pf = g4b::prefill_combine_blocks(pp, a->D);
    mp.combine_dec = (pair || !m.nw) ? 0 : a->B * a->G * pd.R * pd.Tq;
    if (!profile_arm()) return fail(G4B_ERR_LAUNCH, "could not create profiling events");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    hipError_t e;
    if (a->D == 512) e = a->kv_dtype == G4B_DT_F16 ? g4b::launch_attn_mixed_d512_f16(pp, pd, mp, st) : g4b::launch_attn_mixed_d512_bf16(pp, pd, mp, st);
    else e = a->kv_dtype == G4B_DT_F16 ? g4b::launch_attn_mixed_f16(pp, pd, mp, st) : g4b::launch_attn_mixed_bf16(pp, pd, mp, st);
    profile_disarm();
    if (e != hipSuccess) return fail(G4B_ERR_LAUNCH, "mixed attention launch failed: %s", hipGetErrorString(e));
    return G4B_OK;
}

int g4b_static_scratch_init(void) {
    void* ptr = nullptr;
    const hipError_t e = static_scratch_ptr(&ptr);
    if (e != hipSuccess) return fail(G4B_ERR_LAUNCH, "static scratch: %s", hipGetErrorString(e));
    (void)xcd_parity_known(nullptr);  // the other thing a launch may want to look up outside stream capture
    return G4B_OK;
}

uint64_t g4b_static_scratch_bytes(void) { return kStaticScratchBytes; }

int g4b_attn_forward_static_scratch(const g4b_attn_args* a, void* stream) {
    if (!a) return fail(G4B_ERR_INVALID_ARGUMENT, "args is NULL");
    if (a->workspace) return fail(G4B_ERR_INVALID_ARGUMENT, "g4b_attn_forward_static_scratch brings its own scratch: workspace must be NULL");
    const bool shape_ok = a->B >= 1 && a->H >= 1 && a->G >= 1 && a->H % a->G == 0;  // the rest is checked by g4b_attn_forward
    const uint64_t need = (shape_ok && takes_generic_path(a)) ? 0 : g4b_attn_workspace_bytes(a->B, a->H, a->G, a->Tq, a->D, a->num_workers);
    if (need > kStaticScratchBytes)
        return fail(G4B_ERR_WORKSPACE, "this launch splits keys through %llu bytes of partials, the static scratch holds %llu; "
                    "use g4b_attn_forward with a workspace of that size",
                    (unsigned long long)need, (unsigned long long)kStaticScratchBytes);
    g4b_attn_args b = *a;
    if (need) {
        void* ptr = nullptr;
        const hipError_t e = static_scratch_ptr(&ptr);
        if (e != hipSuccess) return fail(G4B_ERR_LAUNCH, "static scratch: %s", hipGetErrorString(e));
        if (!claim_static_scratch(static_cast<hipStream_t>(stream)))
            return fail(G4B_ERR_BUSY, "the static scratch of this GPU is in use by work on another stream that has not finished; "
                        "order the streams, or give this call a workspace of its own (g4b_attn_forward)");
        b.workspace = ptr;
        b.workspace_bytes = kStaticScratchBytes;
    }
    return g4b_attn_forward(&b, stream);
}

int g4b_kv_append(const g4b_kv_append_args* a, void* stream) {
    if (!a) return fail(G4B_ERR_INVALID_ARGUMENT, "args is NULL");
    if (!a->x || !a->cache || !a->cache_offsets) return fail(G4B_ERR_INVALID_ARGUMENT, "x, cache and cache_offsets must be non-NULL");
    if (!dtype_ok(a->x_dtype) || !dtype_ok(a->cache_dtype)) return fail(G4B_ERR_INVALID_ARGUMENT, "x/cache dtype must be f16, bf16 or f32");
    if (a->B < 1 || a->G < 1 || a->t < 1 || a->T < 1 || a->D < 1) return fail(G4B_ERR_INVALID_ARGUMENT, "B, G, t, T, D must be positive");
    if (a->t > a->T) return fail(G4B_ERR_INVALID_ARGUMENT, "t (%d) must not exceed the ring length T (%d)", a->t, a->T);
    if (a->D % 8) return fail(G4B_ERR_UNSUPPORTED, "D must be a multiple of 8");
    if (a->B > 65535) return fail(G4B_ERR_UNSUPPORTED, "B must be <= 65535");
    if (a->phase < 0 || a->phase > 255) return fail(G4B_ERR_INVALID_ARGUMENT, "phase must fit uint8");
    if (a->x_stride[3] != 1) return fail(G4B_ERR_INVALID_ARGUMENT, "x must have unit stride in the head dimension");
    for (int i = 0; i < 3; ++i)
        if (a->x_stride[i] % 8) return fail(G4B_ERR_INVALID_ARGUMENT, "x strides must be multiples of 8 elements");
    if (a->cache_stride_b < (int64_t)a->G * a->T * a->D || a->cache_stride_b % 8)
        return fail(G4B_ERR_INVALID_ARGUMENT, "cache slot stride must be >= G*T*D and a multiple of 8 elements");
    if (!aligned16(a->x) || !aligned16(a->cache)) return fail(G4B_ERR_INVALID_ARGUMENT, "x and cache must be 16-byte aligned");
    if (!std::isfinite(a->rmsnorm_eps)) return fail(G4B_ERR_INVALID_ARGUMENT, "rmsnorm_eps must be finite");

    g4b::KvAppendParams p{};
    p.x = a->x;
    p.cache = a->cache;
    p.offsets = a->cache_offsets;
    p.x_rsos = a->x_rsos;
    p.phase_arr = a->user_phase;
    for (int i = 0; i < 4; ++i) p.x_s[i] = a->x_stride[i];
    for (int i = 0; i < 3; ++i) p.rsos_s[i] = a->x_rsos_stride[i];
    p.cache_sb = a->cache_stride_b;
    p.off_s = a->cache_offsets_stride;
    p.ph_s = a->user_phase_stride;
    p.x_dt = a->x_dtype;
    p.cache_dt = a->cache_dtype;
    p.off_is_i64 = a->cache_offsets_is_int64 ? 1 : 0;
    p.B = a->B;
    p.G = a->G;
    p.t = a->t;
    p.T = a->T;
    p.D = a->D;
    p.phase = a->phase;
    p.eps = a->rmsnorm_eps;
    hipError_t e = g4b::launch_kv_append(p, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(G4B_ERR_LAUNCH, "kv append launch failed: %s", hipGetErrorString(e));
    return G4B_OK;
}

int g4b_advance_decode_state(const g4b_advance_args* a, void* stream) {
    if (!a) return fail(G4B_ERR_INVALID_ARGUMENT, "args is NULL");
    if (!a->input_token_ids || !a->out_token_ids || !a->cache_offsets || !a->time_dim_sizes || !a->user_phase)
        return fail(G4B_ERR_INVALID_ARGUMENT, "all five arrays must be non-NULL");
    if (a->B < 1) return fail(G4B_ERR_INVALID_ARGUMENT, "B must be positive");
    g4b::AdvanceParams p{};
    p.input_token_ids = a->input_token_ids;
    p.out_token_ids = a->out_token_ids;
    p.cache_offsets = a->cache_offsets;
    p.time_dim_sizes = a->time_dim_sizes;
    p.user_phase = a->user_phase;
    p.in_s1 = a->input_token_ids_stride1;
    p.out_s0 = a->out_token_ids_stride0;
    p.off_s = a->cache_offsets_stride;
    p.tds_s = a->time_dim_sizes_stride;
    p.ph_s = a->user_phase_stride;
    p.B = a->B;
    hipError_t e = g4b::launch_advance_decode_state(p, static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(G4B_ERR_LAUNCH, "advance launch failed: %s", hipGetErrorString(e));
    return G4B_OK;
}

int g4b_rope(const g4b_rope_args* a, void* stream) {
    if (!a) return fail(G4B_ERR_INVALID_ARGUMENT, "args is NULL");
    if (!a->q || !a->k || !a->rope_freqs || !a->time_dim_offsets || !a->q_rsos || !a->k_rsos || !a->q_rmsnorm_w || !a->k_rmsnorm_w)
        return fail(G4B_ERR_INVALID_ARGUMENT, "q, k, rope_freqs, time_dim_offsets, q/k_rsos and q/k_rmsnorm_w must be non-NULL");
    if (!dtype_ok(a->q_dtype) || !dtype_ok(a->k_dtype)) return fail(G4B_ERR_INVALID_ARGUMENT, "q/k dtype must be f16, bf16 or f32");
    if (a->B < 1 || a->H < 1 || a->G < 1 || a->t < 1 || a->D < 1) return fail(G4B_ERR_INVALID_ARGUMENT, "B, H, G, t, D must be positive");
    if (a->D % 16 || a->D > 4096) return fail(G4B_ERR_UNSUPPORTED, "D must be a multiple of 16 and at most 4096 (got %d)", a->D);
    if (a->B > 65535) return fail(G4B_ERR_UNSUPPORTED, "B must be <= 65535");
    if (a->q_stride[3] != 1 || a->k_stride[3] != 1) return fail(G4B_ERR_INVALID_ARGUMENT, "q and k must have unit stride in the head dimension");
    for (int i = 0; i < 3; ++i)
        if (a->q_stride[i] % 8 || a->k_stride[i] % 8) return fail(G4B_ERR_INVALID_ARGUMENT, "q/k strides must be multiples of 8 elements");
    if (!aligned16(a->q) || !aligned16(a->k)) return fail(G4B_ERR_INVALID_ARGUMENT, "q and k must be 16-byte aligned");
    if (!std::isfinite(a->rmsnorm_eps)) return fail(G4B_ERR_INVALID_ARGUMENT, "rmsnorm_eps must be finite");
    if (a->k_cache) {
        if (!dtype_ok(a->cache_dtype)) return fail(G4B_ERR_INVALID_ARGUMENT, "cache dtype must be f16, bf16 or f32");
        if (a->T < 1 || a->t > a->T) return fail(G4B_ERR_INVALID_ARGUMENT, "t (%d) must not exceed the ring length T (%d)", a->t, a->T);
        if (a->phase < 0 || a->phase > 255) return fail(G4B_ERR_INVALID_ARGUMENT, "phase must fit uint8");
        if (a->k_cache_stride_b < (int64_t)a->G * a->T * a->D || a->k_cache_stride_b % 8)
            return fail(G4B_ERR_INVALID_ARGUMENT, "k_cache slot stride must be >= G*T*D and a multiple of 8 elements");
        if (!aligned16(a->k_cache)) return fail(G4B_ERR_INVALID_ARGUMENT, "k_cache must be 16-byte aligned");
        if ((a->v != nullptr) != (a->v_cache != nullptr)) return fail(G4B_ERR_INVALID_ARGUMENT, "v and v_cache go together");
        if (a->v) {
            if (!dtype_ok(a->v_dtype)) return fail(G4B_ERR_INVALID_ARGUMENT, "v dtype must be f16, bf16 or f32");
            if (a->Dv < 1 || a->Dv % 8) return fail(G4B_ERR_UNSUPPORTED, "Dv must be a positive multiple of 8");
            if (a->v_stride[3] != 1) return fail(G4B_ERR_INVALID_ARGUMENT, "v must have unit stride in the head dimension");
            for (int i = 0; i < 3; ++i)
                if (a->v_stride[i] % 8) return fail(G4B_ERR_INVALID_ARGUMENT, "v strides must be multiples of 8 elements");
            if (a->v_cache_stride_b < (int64_t)a->G * a->T * a->Dv || a->v_cache_stride_b % 8)
                return fail(G4B_ERR_INVALID_ARGUMENT, "v_cache slot stride must be >= G*T*Dv and a multiple of 8 elements");
            if (!aligned16(a->v) || !aligned16(a->v_cache)) return fail(G4B_ERR_INVALID_ARGUMENT, "v and v_cache must be 16-byte aligned");
        }
    } else if (a->v || a->v_cache) {
        return fail(G4B_ERR_INVALID_ARGUMENT, "v / v_cache need k_cache: the append is fused as a whole");
    }

    g4b::RopeParams p{};
    p.q = a->q;
    p.k = a->k;
    p.freqs = a->rope_freqs;
    p.offsets = a->time_dim_offsets;
    p.q_rsos = a->q_rsos;
    p.k_rsos = a->k_rsos;
    p.q_w = a->q_rmsnorm_w;
    p.k_w = a->k_rmsnorm_w;
    p.v = a->v;
    p.v_rsos = a->v_rsos;
    p.k_cache = a->k_cache;
    p.v_cache = a->v_cache;
    p.phase_arr = a->user_phase;
    for (int i = 0; i < 4; ++i) {
        p.q_s[i] = a->q_stride[i];
        p.k_s[i] = a->k_stride[i];
        p.v_s[i] = a->v_stride[i];
    }
    for (int i = 0; i < 3; ++i) {
        p.q_rsos_s[i] = a->q_rsos_stride[i];
        p.k_rsos_s[i] = a->k_rsos_stride[i];
        p.v_rsos_s[i] = a->v_rsos_stride[i];
    }
    p.freqs_s = a->rope_freqs_stride;
    p.q_w_s = a->q_rmsnorm_w_stride;
    p.k_w_s = a->k_rmsnorm_w_stride;
    p.off_s = a->time_dim_offsets_stride;
    p.ph_s = a->user_phase_stride;
    p.k_cache_sb = a->k_cache_stride_b;
    p.v_cache_sb = a->v_cache_stride_b;
    p.q_dt = a->q_dtype;
    p.k_dt = a->k_dtype;
    p.v_dt = a->v_dtype;
    p.cache_dt = a->cache_dtype;
    p.B = a->B;
    p.H = a->H;
    p.G = a->G;
    p.t = a->t;
    p.D = a->D;
    p.Dv = a->Dv;
    p.T = a->T;
    p.phase = a->phase;
    p.k_writeback = a->k_writeback;
    p.eps = a->rmsnorm_eps;
    p.xcd_weighted = xcd_parity_known(static_cast<hipStream_t>(stream));
    if (!profile_arm()) return fail(G4B_ERR_LAUNCH, "could not create profiling events");
    hipError_t e = g4b::launch_rope(p, static_cast<hipStream_t>(stream));
    profile_disarm();
    if (e != hipSuccess) return fail(G4B_ERR_LAUNCH, "rope launch failed: %s", hipGetErrorString(e));
    return G4B_OK;
}

int g4b_rope_frequencies(float* out, const float* freq_scalars, int32_t n, int64_t out_stride, int64_t freq_scalars_stride,
                         float freq_base, void* stream) {
    if (!out || n < 1) return fail(G4B_ERR_INVALID_ARGUMENT, "out must be non-NULL and n positive");
    if (!(freq_base > 0.f) || !std::isfinite(freq_base)) return fail(G4B_ERR_INVALID_ARGUMENT, "freq_base must be positive and finite");
    // the reference folds log2(freq_base) on the host in double precision (rope.py:280)
    const float log2_base = (float)std::log2((double)freq_base);
    hipError_t e = g4b::launch_rope_frequencies(out, freq_scalars, n, out_stride, freq_scalars_stride, log2_base,
                                                static_cast<hipStream_t>(stream));
    if (e != hipSuccess) return fail(G4B_ERR_LAUNCH, "rope frequency launch failed: %s", hipGetErrorString(e));
    return G4B_OK;
}

}  // extern "C"

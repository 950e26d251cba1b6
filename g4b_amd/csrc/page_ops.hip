// Operators on the pages of a paged KV cache: the append of new K and V rows, and page management (copy, free, fork,
// allocate, compact).  Values are copied bit for bit (or scaled by rsqrt(rsos / D + eps) in fp32 and rounded once into the
// pool's type); everything that decides where they go is integer arithmetic whose result does not depend on timing.
#include "paged.hpp"

namespace g4b {

// ---- append --------------------------------------------------------------------------------------------------------
// A thread moves N consecutive elements of a K row and the same of the V row, 16 bytes of the wider of the two types; the
// G * D elements of a token's rows are consecutive in threads, so a wave reads contiguous runs and writes D-element ones.
// Every thread finds its token's sequence by itself (a binary search over starts that sit in the caches).
template <int N>
__global__ __launch_bounds__(256) void paged_append_kernel(const PagedAppendParams p) {
    const int segs = p.D / N;
    const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t row_items = (int64_t)p.G * segs;
    const int64_t t64 = idx / row_items;
    if (t64 >= p.T) return;
    const int t = (int)t64;
    const int rest = (int)(idx - t64 * row_items);
    const int g = rest / segs, seg = rest % segs;
    int s = t, first = t;
    if (p.cu) {
        s = packed_owner(p.cu, p.cu_s, p.N, t);
        if (s < 0) return;
        first = max(p.cu[(int64_t)s * p.cu_s], 0);
    }
    if (p.phase_arr && p.phase_arr[(int64_t)s * p.ph_s] != (uint8_t)p.phase) return;
    const int64_t pos = (int64_t)p.offsets[(int64_t)s * p.off_s] + (t - first);
    if (pos < 0 || pos >= (int64_t)p.max_pages * p.page_size) return;
    const int entry = (int)(pos / p.page_size), in_page = (int)(pos - (int64_t)entry * p.page_size);
    const int page = p.table[(int64_t)s * p.table_s + entry];
    if ((uint32_t)page >= (uint32_t)p.num_pages) return;

    float kx[N], vx[N];
    load_f32<N, true>(p.k, (int64_t)t * p.k_s[0] + (int64_t)g * p.k_s[1] + seg * N, p.k_dt, kx);
    load_f32<N, true>(p.v, (int64_t)t * p.v_s[0] + (int64_t)g * p.v_s[1] + seg * N, p.v_dt, vx);
    if (p.k_rsos) {
        const float inv = 1.0f / __builtin_sqrtf(p.k_rsos[(int64_t)t * p.k_rsos_s[0] + (int64_t)g * p.k_rsos_s[1]] / (float)p.D + p.eps);
#pragma unroll
        for (int i = 0; i < N; ++i) kx[i] *= inv;
    }
    if (p.v_rsos) {
        const float inv = 1.0f / __builtin_sqrtf(p.v_rsos[(int64_t)t * p.v_rsos_s[0] + (int64_t)g * p.v_rsos_s[1]] / (float)p.D + p.eps);
#pragma unroll
        for (int i = 0; i < N; ++i) vx[i] *= inv;
    }
    const int64_t in = ((int64_t)g * p.page_size + in_page) * p.D + seg * N;
    store_n<N>(p.k_pages, page * p.k_ps + in, p.cache_dt, kx);
    store_n<N>(p.v_pages, page * p.v_ps + in, p.cache_dt, vx);
}

hipError_t launch_paged_append(const PagedAppendParams& p, hipStream_t stream) {
    const bool wide = p.k_dt == DT_F32 || p.v_dt == DT_F32 || p.cache_dt == DT_F32;
    const int64_t items = (int64_t)p.T * p.G * (p.D / (wide ? 4 : 8));
    const int64_t blocks = (items + 255) / 256;
    if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    if (wide) hipLaunchKernelGGL(paged_append_kernel<4>, dim3((unsigned)blocks), dim3(256), 0, stream, p);
    else hipLaunchKernelGGL(paged_append_kernel<8>, dim3((unsigned)blocks), dim3(256), 0, stream, p);
    return hipGetLastError();
}

// ---- copies of whole pages -----------------------------------------------------------------------------------------
// A workgroup of 256 threads copies one chunk of COPY_CHUNK bytes of one page of one layer of one pool: item =
// ((pair * layers + layer) * 2 + pool) * chunks + chunk.  Every load of the chunk is in flight before the first store.
constexpr int COPY_VECS = 4;
constexpr int COPY_CHUNK = 256 * 16 * COPY_VECS;
G4B_DEV void copy_chunk(const PagesParams& p, int src, int dst, int layer, int pool, int64_t begin) {
    const char* from = pool ? p.v + layer * p.v_ls + src * p.v_ps : p.k + layer * p.k_ls + src * p.k_ps;
    char* to = pool ? p.v + layer * p.v_ls + dst * p.v_ps : p.k + layer * p.k_ls + dst * p.k_ps;
    u4 x[COPY_VECS];
#pragma unroll
    for (int i = 0; i < COPY_VECS; ++i) {
        const int64_t at = begin + (int64_t)(i * 256 + (int)threadIdx.x) * 16;
        x[i] = u4{0, 0, 0, 0};
        if (at < p.page_bytes) x[i] = __builtin_nontemporal_load(reinterpret_cast<const u4*>(from + at));
    }
#pragma unroll
    for (int i = 0; i < COPY_VECS; ++i) {
        const int64_t at = begin + (int64_t)(i * 256 + (int)threadIdx.x) * 16;
        if (at < p.page_bytes) __builtin_nontemporal_store(x[i], reinterpret_cast<u4*>(to + at));
    }
}
static int64_t copy_chunks(const PagesParams& p) { return (p.page_bytes + COPY_CHUNK - 1) / COPY_CHUNK; }

// Pair i of the list is judged by each of its workgroups (the list is at most G4B_PAGES_MAX_LIST long), so no pass over
// the list has to come first and the answer is the same everywhere.
__global__ __launch_bounds__(256) void pages_copy_kernel(const PagesParams p, const int chunks) {
    int64_t item = blockIdx.x;
    const int chunk = (int)(item % chunks);
    item /= chunks;
    const int pool = (int)(item & 1);
    item >>= 1;
    const int layer = (int)(item % p.layers), i = (int)(item / p.layers);
    const int src = p.src[i], dst = p.dst[i];
    bool bad = (uint32_t)src >= (uint32_t)p.P || (uint32_t)dst >= (uint32_t)p.P;
    for (int j = threadIdx.x; j < p.n; j += 256) {
        const int sj = p.src[j], dj = p.dst[j];
        if (sj == dj) continue;  // moves nothing
        if (src != dst && ((j < i && dj == dst) || sj == dst)) bad = true;  // an earlier pair writes it, or one reads it
    }
    bad = __syncthreads_or(bad);
    if (bad) {
        if (threadIdx.x == 0 && chunk == 0 && pool == 0 && layer == 0) atomicAdd(p.status, 1);
        return;
    }
    if (src != dst) copy_chunk(p, src, dst, layer, pool, (int64_t)chunk * COPY_CHUNK);
}

hipError_t launch_pages_copy(const PagesParams& p, hipStream_t stream) {
    const int64_t chunks = copy_chunks(p), blocks = chunks * 2 * p.layers * p.n;
    if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    hipLaunchKernelGGL(pages_copy_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, p, (int)chunks);
    return hipGetLastError();
}

// ---- free ----------------------------------------------------------------------------------------------------------
G4B_DEV int pages_of(const PagesParams& p, int64_t len) {  // table entries that hold len positions
    const int64_t n = (max(len, (int64_t)0) + p.page_size - 1) / p.page_size;
    return (int)min(n, (int64_t)p.max_pages);
}

// One workgroup per listed sequence.  Whoever takes the length away frees the pages, so a repeated entry finds nothing.
__global__ __launch_bounds__(256) void pages_free_kernel(const PagesParams p) {
    __shared__ int sh_len;
    const int s = p.src[blockIdx.x];
    if ((uint32_t)s >= (uint32_t)p.S) return;
    if (threadIdx.x == 0) sh_len = atomicExch(p.lens + s, 0);
    __syncthreads();
    const int held = pages_of(p, sh_len);
    int32_t* row = p.table + s * p.table_s;
    for (int e = threadIdx.x; e < held; e += 256) {
        const int page = row[e];
        row[e] = -1;
        if ((uint32_t)page < (uint32_t)p.P && atomicSub(p.refs + page, 1) <= 0) atomicAdd(p.refs + page, 1);
    }
}

hipError_t launch_pages_free(const PagesParams& p, hipStream_t stream) {
    hipLaunchKernelGGL(pages_free_kernel, dim3(p.n), dim3(256), 0, stream, p);
    return hipGetLastError();
}

// ---- planning: one workgroup that walks the counts --------------------------------------------------------------------
constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_WAVES = PLAN_THREADS / 64;

// Exclusive prefix sum over the workgroup's threads and the total.  sh: PLAN_WAVES ints; every thread calls it.
G4B_DEV int block_scan(int v, int& total, int* sh) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int incl = wave_incl_scan_i(v, lane);
    __syncthreads();  // the previous call's sums have been read
    if (lane == 63) sh[wave] = incl;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < PLAN_WAVES; ++w) {
        const int x = sh[w];
        before += w < wave ? x : 0;
        total += x;
    }
    return before + incl - v;
}

// Walks the counts four per thread and step; visit(first page of the thread's four, their counts, how many exist, step's
// first page) for every thread and step, in ascending order of steps, until it returns false (the same in every thread).
template <class Visit>
G4B_DEV void walk_counts(const PagesParams& p, Visit&& visit) {
    typedef int i4 __attribute__((ext_vector_type(4)));
    auto load = [&](int64_t at) {
        i4 c = {1, 1, 1, 1};
        if (at + 4 <= p.P) c = *reinterpret_cast<const i4*>(p.refs + at);
        else
            for (int i = 0; i < 4; ++i)
                if (at + i < p.P) c[i] = p.refs[at + i];
        return c;
    };
    i4 next = load((int64_t)threadIdx.x * 4);
    for (int64_t base = 0; base < p.P; base += PLAN_THREADS * 4) {
        const int64_t at = base + (int64_t)threadIdx.x * 4;
        const i4 c = next;
        next = load(at + PLAN_THREADS * 4);
        const int64_t left = p.P - at;
        if (!visit(at, c, (int)min(max(left, (int64_t)0), (int64_t)4))) return;
    }
}

// The `need` lowest-numbered free pages into list[0 ..]; returns how many there are, at most `need`.
G4B_DEV int lowest_free(const PagesParams& p, int need, int32_t* list, int* sh) {
    int found = 0;
    if (need > 0)
        walk_counts(p, [&](int64_t at, auto c, int exist) {
            int mine = 0;
            for (int i = 0; i < 4; ++i) mine += (i < exist && c[i] == 0) ? 1 : 0;
            int total, r = found + block_scan(mine, total, sh);
            for (int i = 0; i < 4; ++i)
                if (i < exist && c[i] == 0) {
                    if (r < need) list[r] = (int32_t)(at + i);
                    ++r;
                }
            found += total;
            return found < need;
        });
    return min(found, need);
}

// ---- fork ----------------------------------------------------------------------------------------------------------
// Plan: every fork checked, its source's length kept (ws[0 .. n): a destination of one fork may be, empty, the source of
// another) and the page for its partly filled last page chosen (ws[n .. 2n)).  Apply: one workgroup per fork shares the
// full pages, others copy the last page, chunk by chunk.
__global__ __launch_bounds__(PLAN_THREADS) void pages_fork_plan_kernel(const PagesParams p) {
    __shared__ int sh[PLAN_WAVES];
    extern __shared__ uint32_t named[];  // the destinations so far, one bit per sequence
    const int words = (p.S + 31) >> 5;
    for (int i = threadIdx.x; i < words; i += PLAN_THREADS) named[i] = 0;
    __syncthreads();
    int32_t *len_of = p.ws + 16, *page_of = len_of + p.n, *list = page_of + p.n;
    bool bad = false;
    int need = 0;
    for (int base = 0; base < p.n; base += PLAN_THREADS) {
        const int i = base + threadIdx.x;
        int wants = 0;
        if (i < p.n) {
            const int s = p.src[i], d = p.dst[i];
            int len = 0;
            if ((uint32_t)s >= (uint32_t)p.S || (uint32_t)d >= (uint32_t)p.S) bad = true;
            else {
                len = max(p.lens[s], 0);
                if (p.lens[d] != 0 || len > (int64_t)p.max_pages * p.page_size) bad = true;
                if ((atomicOr(&named[d >> 5], 1u << (d & 31)) >> (d & 31)) & 1u) bad = true;
                if (!bad && len % p.page_size != 0)  // (an absent last page stays absent)
                    wants = (uint32_t)p.table[s * p.table_s + len / p.page_size] < (uint32_t)p.P;
            }
            len_of[i] = len;
        }
        int total;
        const int r = need + block_scan(wants, total, sh);
        if (i < p.n) page_of[i] = wants ? r : -1;
        need += total;
    }
    bad = __syncthreads_or(bad);
    const int found = bad ? 0 : lowest_free(p, need, list, sh);
    __syncthreads();
    const int status = bad ? -1 : need - found;
    if (threadIdx.x == 0) {
        p.status[0] = status;
        p.ws[0] = status;
    }
    if (status == 0)
        for (int i = threadIdx.x; i < p.n; i += PLAN_THREADS)
            if (page_of[i] >= 0) page_of[i] = list[page_of[i]];
}

__global__ __launch_bounds__(256) void pages_fork_apply_kernel(const PagesParams p, const int chunks) {
    if (p.ws[0] != 0) return;
    const int i = blockIdx.x / (1 + chunks), role = blockIdx.x % (1 + chunks);
    const int len = p.ws[16 + i], page = p.ws[16 + p.n + i];
    const int full = len / p.page_size;
    const int32_t* from = p.table + p.src[i] * p.table_s;
    if (role == 0) {
        int32_t* to = p.table + p.dst[i] * p.table_s;
        for (int e = threadIdx.x; e < full; e += 256) {
            const int x = from[e];
            to[e] = x;
            if ((uint32_t)x < (uint32_t)p.P) atomicAdd(p.refs + x, 1);
        }
        if (threadIdx.x == 0) {
            p.lens[p.dst[i]] = len;
            if (len % p.page_size != 0) to[full] = page;
            if (page >= 0) p.refs[page] = 1;
        }
        return;
    }
    if (page < 0) return;
    const int old = from[full];
    const int item = role - 1, per_layer = chunks / p.layers;  // (pool, chunk) of a layer
    const int layer = item / per_layer, in_layer = item % per_layer;
    copy_chunk(p, old, page, layer, in_layer & 1, (int64_t)(in_layer >> 1) * COPY_CHUNK);
}

hipError_t launch_pages_fork(const PagesParams& p, hipStream_t stream) {
    const int64_t chunks = copy_chunks(p) * 2 * p.layers, blocks = (1 + chunks) * p.n;
    if (blocks > 0x7fffffffLL) return hipErrorInvalidValue;
    hipLaunchKernelGGL(pages_fork_plan_kernel, dim3(1), dim3(PLAN_THREADS), ((p.S + 31) / 32) * 4, stream, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.n == 0) return e;
    hipLaunchKernelGGL(pages_fork_apply_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, p, (int)chunks);
    return hipGetLastError();
}

// ---- allocate ------------------------------------------------------------------------------------------------------
// One workgroup: what every sequence needs and its running sum (ws[16 .. 16 + S]), then the lowest free pages, then page r
// of them to the sequence whose run of the sum holds r.
__global__ __launch_bounds__(PLAN_THREADS) void pages_allocate_kernel(const PagesParams p) {
    __shared__ int sh[PLAN_WAVES];
    int32_t *before = p.ws + 16, *list = before + p.S + 1;
    bool bad = false;
    int64_t need = 0;
    for (int base = 0; base < p.S; base += PLAN_THREADS) {
        const int s = base + threadIdx.x;
        int wants = 0;
        if (s < p.S) {
            const int grow = p.num_new[s];
            const int64_t len = max(p.lens[s], 0), after = len + grow;
            if (grow < 0 || after > (int64_t)p.max_pages * p.page_size) bad = true;
            else wants = pages_of(p, after) - pages_of(p, len);
        }
        int total;  // at most PLAN_THREADS * max_pages <= 2^30
        const int r = block_scan(wants, total, sh);
        if (s < p.S) before[s] = (int32_t)min(need + r, (int64_t)p.P + 1);
        need += total;
    }
    bad = __syncthreads_or(bad);
    const int want = (int)min(need, (int64_t)p.P + 1);  // more than every page there is: P + 1 stands for all such needs
    const int found = bad ? 0 : lowest_free(p, want, list, sh);
    const int status = bad ? -1 : (int)min(need - found, (int64_t)0x7fffffff);
    if (threadIdx.x == 0) {
        p.status[0] = status;
        before[p.S] = want;
    }
    __syncthreads();
    if (status != 0) return;
    for (int r = threadIdx.x; r < want; r += PLAN_THREADS) {
        int lo = 0, hi = p.S;  // before[lo] <= r < before[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (before[mid] <= r) lo = mid;
            else hi = mid;
        }
        const int page = list[r];
        p.table[lo * p.table_s + pages_of(p, max(p.lens[lo], 0)) + (r - before[lo])] = page;
        p.refs[page] = 1;
    }
    __syncthreads();  // the lengths have been read
    for (int s = threadIdx.x; s < p.S; s += PLAN_THREADS) p.lens[s] = max(p.lens[s], 0) + p.num_new[s];
}

hipError_t launch_pages_allocate(const PagesParams& p, hipStream_t stream) {
    hipLaunchKernelGGL(pages_allocate_kernel, dim3(1), dim3(PLAN_THREADS), 0, stream, p);
    return hipGetLastError();
}

// ---- compact -------------------------------------------------------------------------------------------------------
// Plan: with n pages in use, the k-th free page below n is where the k-th used page at or above n goes, so no page is both
// read and written and the copies need no order.  ws[0] = number of moves; the k-th source goes to ws[16 + k], the k-th
// destination to ws[16 + half + k].
__global__ __launch_bounds__(PLAN_THREADS) void pages_compact_plan_kernel(const PagesParams p) {
    __shared__ int sh[PLAN_WAVES];
    const int half = (p.P + 1) / 2;
    int32_t *from = p.ws + 16, *to = from + half;
    int live = 0;
    {
        int mine = 0;
        walk_counts(p, [&](int64_t at, auto c, int exist) {
            for (int i = 0; i < 4; ++i) mine += (i < exist && c[i] > 0) ? 1 : 0;
            return true;
        });
        (void)block_scan(mine, live, sh);
    }
    int holes = 0, movers = 0;
    walk_counts(p, [&](int64_t at, auto c, int exist) {
        int h = 0, m = 0;
        for (int i = 0; i < 4; ++i) {
            const bool used = c[i] > 0, low = at + i < live;
            h += (i < exist && !used && low) ? 1 : 0;
            m += (i < exist && used && !low) ? 1 : 0;
        }
        // both counts in one scan: 4096 pages a step, so 16 bits hold each sum
        int total, r = block_scan(h | (m << 16), total, sh);
        int rh = holes + (r & 0xffff), rm = movers + (r >> 16);
        for (int i = 0; i < 4; ++i) {
            if (i >= exist) continue;
            const bool used = c[i] > 0, low = at + i < live;
            if (!used && low) to[rh++] = (int32_t)(at + i);
            if (used && !low) from[rm++] = (int32_t)(at + i);
            p.page_map[at + i] = used ? (int32_t)(at + i) : -1;
        }
        holes += total & 0xffff;
        movers += total >> 16;
        return true;
    });
    __syncthreads();
    for (int k = threadIdx.x; k < movers; k += PLAN_THREADS) p.page_map[from[k]] = to[k];
    if (threadIdx.x == 0) {
        p.ws[0] = movers;
        p.status[0] = live;
    }
}

// Apply: the workgroups walk the moves' chunks (as many as the plan found, which the host does not know) and the tables.
constexpr int COMPACT_BLOCKS = 2048;
__global__ __launch_bounds__(256) void pages_compact_apply_kernel(const PagesParams p, const int chunks) {
    const int half = (p.P + 1) / 2;
    const int moves = p.ws[0];
    const int32_t *from = p.ws + 16, *to = from + half;
    const int64_t items = (int64_t)moves * chunks;
    const int per_layer = chunks / p.layers;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int k = (int)(item / chunks), c = (int)(item % chunks);
        const int src = from[k], dst = to[k];
        const int layer = c / per_layer, in_layer = c % per_layer;
        copy_chunk(p, src, dst, layer, in_layer & 1, (int64_t)(in_layer >> 1) * COPY_CHUNK);
        if (c == 0 && threadIdx.x == 0) {
            p.refs[dst] = p.refs[src];
            p.refs[src] = 0;
        }
    }
    for (int s = blockIdx.x; s < p.S; s += gridDim.x) {
        const int held = pages_of(p, p.lens[s]);
        int32_t* row = p.table + s * p.table_s;
        for (int e = threadIdx.x; e < held; e += 256) {
            const int page = row[e];
            if ((uint32_t)page < (uint32_t)p.P && p.page_map[page] >= 0) row[e] = p.page_map[page];
        }
    }
}

hipError_t launch_pages_compact(const PagesParams& p, hipStream_t stream) {
    const int64_t chunks = copy_chunks(p) * 2 * p.layers;
    if (chunks > 0x7fffffffLL) return hipErrorInvalidValue;
    hipLaunchKernelGGL(pages_compact_plan_kernel, dim3(1), dim3(PLAN_THREADS), 0, stream, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(pages_compact_apply_kernel, dim3(COMPACT_BLOCKS), dim3(256), 0, stream, p, (int)chunks);
    return hipGetLastError();
}

}  // namespace g4b

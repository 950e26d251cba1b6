// Operators on the pages of a paged KV cache: the append of new K and V rows, and page management (copy, free, fork,
// allocate, compact).  Values are copied bit for bit (or scaled by rsqrt(rsos / D + eps) in fp32 and rounded once into the
// pool's type); everything that decides where they go is integer arithmetic whose result does not depend on timing.
#include "paged.hpp"

namespace g4b {

// ---- append --------------------------------------------------------------------------------------------------------
// A row is the N-element pieces of all G heads of a token, a workgroup takes as many rows as its threads have pieces (one row
// in several passes where a row has more), and a thread moves one piece of K and the same of V, 16 bytes of the pool's type.
// Where a row goes is found once per row by one thread (a binary search over the starts, the table entry) and handed on
// through LDS; a piece that keeps its type moves as the 16 bytes that it is.  Bound by memory: 201 MB of rows of 24 prompts in
// 52 us, 3.9 TB/s.  Two or four pieces per thread measured 8 to 35 % slower than one (fewer waves), as did 32 rows per
// workgroup, with which a decode step's 64 rows took 10.9 us instead of 4.1.
constexpr int APPEND_MAX_ROWS = 32;
template <int N>
G4B_DEV void append_piece(const void* x, int64_t from, int x_dt, void* cache, int64_t to, int cache_dt, const float* rsos, int D, float eps) {
    if (x_dt == cache_dt && !rsos) {
        constexpr int BYTES = 16 / N;  // N elements of the kernel's type are 16 bytes: 8 of 16 bits or 4 of 32
        if (BYTES == 2 || x_dt == DT_F32) {
            st_vec<true>(reinterpret_cast<u4*>(static_cast<char*>(cache) + to * BYTES),
                         ld_vec<true>(reinterpret_cast<const u4*>(static_cast<const char*>(x) + from * BYTES)));
            return;
        }
    }
    float v[N];
    load_f32<N, true>(x, from, x_dt, v);
    if (rsos) {
        const float inv = 1.0f / __builtin_sqrtf(*rsos / (float)D + eps);
#pragma unroll
        for (int e = 0; e < N; ++e) v[e] *= inv;
    }
    store_n<N, true>(cache, to, cache_dt, v);
}

template <int N>
__global__ __launch_bounds__(256) void paged_append_kernel(const PagedAppendParams p, const int rows) {
    __shared__ int64_t k_at[APPEND_MAX_ROWS], v_at[APPEND_MAX_ROWS];
    const int64_t t0 = (int64_t)block_of_grid() * rows;
    if ((int)threadIdx.x < rows) {
        const int t = (int)min(t0 + (int)threadIdx.x, (int64_t)p.T);
        int64_t ka = -1, va = -1;  // element offset of head 0's row in the pools, < 0: dropped
        int s = t, first = t;
        bool ok = t < p.T;
        if (ok && p.cu) {
            s = packed_owner(p.cu, p.cu_s, p.N, t);
            ok = s >= 0;
            if (ok) first = max(p.cu[(int64_t)s * p.cu_s], 0);
        }
        if (ok && p.phase_arr) ok = p.phase_arr[(int64_t)s * p.ph_s] == (uint8_t)p.phase;
        if (ok) {
            const int64_t pos = (int64_t)p.offsets[(int64_t)s * p.off_s] + (t - first);
            if (pos >= 0 && pos < (int64_t)p.max_pages * p.page_size) {
                const int entry = (int)((uint32_t)pos / (uint32_t)p.page_size), in_page = (int)pos - entry * p.page_size;
                const int page = p.table[(int64_t)s * p.table_s + entry];
                if ((uint32_t)page < (uint32_t)p.num_pages) {
                    ka = page * p.k_ps + (int64_t)in_page * p.D;
                    va = page * p.v_ps + (int64_t)in_page * p.D;
                }
            }
        }
        k_at[threadIdx.x] = ka;
        v_at[threadIdx.x] = va;
    }
    __syncthreads();
    const int segs = p.D / N, pieces = p.G * segs, items = pieces * rows;
    for (int i = threadIdx.x; i < items; i += 256) {
        const int row = i / pieces, piece = i - row * pieces;
        if (k_at[row] < 0) continue;
        const int g = piece / segs, c = (piece - g * segs) * N;
        const int64_t t = t0 + row, in_page = (int64_t)g * p.page_size * p.D + c;
        append_piece<N>(p.k, t * p.k_s[0] + g * p.k_s[1] + c, p.k_dt, p.k_pages, k_at[row] + in_page, p.cache_dt,
                        p.k_rsos ? p.k_rsos + t * p.k_rsos_s[0] + g * p.k_rsos_s[1] : nullptr, p.D, p.eps);
        append_piece<N>(p.v, t * p.v_s[0] + g * p.v_s[1] + c, p.v_dt, p.v_pages, v_at[row] + in_page, p.cache_dt,
                        p.v_rsos ? p.v_rsos + t * p.v_rsos_s[0] + g * p.v_rsos_s[1] : nullptr, p.D, p.eps);
    }
}

hipError_t launch_paged_append(const PagedAppendParams& p, hipStream_t stream) {
    const bool wide = p.cache_dt == DT_F32;  // (stores of 16 bytes; an fp32 piece for a 16-bit pool is two loads)
    const int pieces = p.G * (p.D / (wide ? 4 : 8));
    const int rows = pieces >= 256 ? 1 : (256 / pieces < APPEND_MAX_ROWS ? 256 / pieces : APPEND_MAX_ROWS);
    const int64_t blocks = (p.T + (int64_t)rows - 1) / rows;
    const dim3 grid = grid_of(blocks);
    if (wide) hipLaunchKernelGGL(paged_append_kernel<4>, grid, dim3(256), 0, stream, p, rows);
    else hipLaunchKernelGGL(paged_append_kernel<8>, grid, dim3(256), 0, stream, p, rows);
    return hipGetLastError();
}

// ---- copies of whole pages -----------------------------------------------------------------------------------------
// A workgroup of 256 threads copies one chunk of COPY_CHUNK bytes of one page of one layer of one pool: blockIdx.x =
// (layer * 2 + pool) * chunks + chunk, blockIdx.y = pair.  Every load of the chunk is in flight before the first store
// (compaction of 1 GB, read and written: 4.8 TB/s; a copy of 2 GiB reaches 4.9).
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
    const int item = (int)blockIdx.x / chunks, chunk = (int)blockIdx.x - item * chunks, pool = item & 1, layer = item >> 1;
    const int i = blockIdx.y;
    const int src = p.src[i], dst = p.dst[i];
    bool bad = (uint32_t)src >= (uint32_t)p.P || (uint32_t)dst >= (uint32_t)p.P;
    if (src != dst) {  // (the same in every thread; a pair of a page with itself moves nothing)
        for (int j = threadIdx.x; j < p.n; j += 256) {
            const int sj = p.src[j], dj = p.dst[j];
            if (sj != dj && ((j < i && dj == dst) || sj == dst)) bad = true;  // an earlier pair writes it, or one reads it
        }
        bad = __syncthreads_or(bad);
    }
    if (bad) {
        if (threadIdx.x == 0 && chunk == 0 && pool == 0 && layer == 0) atomicAdd(p.status, 1);
        return;
    }
    if (src != dst) copy_chunk(p, src, dst, layer, pool, (int64_t)chunk * COPY_CHUNK);
}

hipError_t launch_pages_copy(const PagesParams& p, hipStream_t stream) {
    const int64_t chunks = copy_chunks(p), blocks = chunks * 2 * p.layers;
    if (blocks > MAX_BLOCKS) return hipErrorInvalidValue;
    hipLaunchKernelGGL(pages_copy_kernel, dim3((unsigned)blocks, (unsigned)p.n), dim3(256), 0, stream, p, (int)chunks);
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

// Four consecutive counts of a thread; pages that do not exist count as used.
typedef int i4 __attribute__((ext_vector_type(4)));
constexpr int PLAN_STEP = PLAN_THREADS * 4;
G4B_DEV i4 load_counts(const PagesParams& p, int64_t at) {
    i4 c = {1, 1, 1, 1};
    if (at + 4 <= p.P) c = *reinterpret_cast<const i4*>(p.refs + at);
    else
        for (int i = 0; i < 4; ++i)
            if (at + i < p.P) c[i] = p.refs[at + i];
    return c;
}

// The `need` lowest-numbered free pages into list[0 ..]; returns how many there are, at most `need`.  The workgroup walks the
// counts until it has them, the next step's on their way while one is looked at (sixteen counts per thread and step instead of
// four measured 6.0 against 4.8 us for a pool of 2400 pages: the scan's instructions count, not the round trips).
G4B_DEV int lowest_free(const PagesParams& p, int need, int32_t* list, int* sh) {
    int found = 0;
    i4 next = load_counts(p, (int64_t)threadIdx.x * 4);
    for (int64_t base = 0; base < p.P && found < need; base += PLAN_STEP) {
        const int64_t at = base + (int64_t)threadIdx.x * 4;
        const i4 c = next;
        next = load_counts(p, at + PLAN_STEP);
        int mine = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) mine += c[i] == 0 ? 1 : 0;
        int total, r = found + block_scan(mine, total, sh);
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (c[i] == 0) {
                if (r < need) list[r] = (int32_t)(at + i);
                ++r;
            }
        found += total;
    }
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
    const int i = blockIdx.y, role = blockIdx.x;
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
    const int64_t chunks = copy_chunks(p) * 2 * p.layers, blocks = 1 + chunks;
    if (blocks > MAX_BLOCKS) return hipErrorInvalidValue;
    hipLaunchKernelGGL(pages_fork_plan_kernel, dim3(1), dim3(PLAN_THREADS), ((p.S + 31) / 32) * 4, stream, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.n == 0) return e;
    hipLaunchKernelGGL(pages_fork_apply_kernel, dim3((unsigned)blocks, (unsigned)p.n), dim3(256), 0, stream, p, (int)chunks);
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
// With n pages in use, the k-th free page below n is where the k-th used page at or above n goes, so no page is both read and
// written and the copies need no order.  The k-th source goes to ws[16 + k], the k-th destination to ws[16 + half + k], both
// by workgroups of PLAN_STEP pages each that know how many pages are in use before theirs (a first kernel has counted; one
// workgroup for all took 21.8 us for 52 000 pages).
G4B_DEV int used_of(const i4& c, int64_t at, int64_t end) {  // pages in use among the thread's four below `end`
    int n = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) n += at + i < end && c[i] > 0 ? 1 : 0;
    return n;
}
__global__ __launch_bounds__(PLAN_THREADS) void pages_compact_count_kernel(const PagesParams p) {
    __shared__ int sh[PLAN_WAVES];
    const int64_t at = (int64_t)blockIdx.x * PLAN_STEP + (int64_t)threadIdx.x * 4;
    int total;
    (void)block_scan(used_of(load_counts(p, at), at, p.P), total, sh);
    // (one count per PLAN_STEP pages, behind the lists)
    if (threadIdx.x == 0) p.ws[16 + 2 * ((p.P + 1) / 2) + blockIdx.x] = total;
}

__global__ __launch_bounds__(PLAN_THREADS) void pages_compact_plan_kernel(const PagesParams p) {
    __shared__ int sh[PLAN_WAVES];
    const int half = (p.P + 1) / 2;
    int32_t *from = p.ws + 16, *to = from + half;
    const int32_t* counts = to + half;
    const int64_t at = (int64_t)blockIdx.x * PLAN_STEP + (int64_t)threadIdx.x * 4;
    const i4 c = load_counts(p, at);
    const int mine = used_of(c, at, p.P);
    // pages in use before this workgroup's, in all, and below the first `live`
    int live, before = 0, below, unused;
    if (gridDim.x == 1) {
        (void)block_scan(mine, live, sh);
        (void)block_scan(used_of(c, at, live), below, sh);
    } else {
        int all = 0, front = 0;
        for (int j = threadIdx.x; j < (int)gridDim.x; j += PLAN_THREADS) {
            all += counts[j];
            front += j < (int)blockIdx.x ? counts[j] : 0;
        }
        (void)block_scan(all, live, sh);
        (void)block_scan(front, before, sh);
        const int seg = live / PLAN_STEP;  // holds page `live` (the one past the last if every page is in use)
        int part = 0;
        for (int j = threadIdx.x; j < seg; j += PLAN_THREADS) part += counts[j];
        const int64_t seg_at = (int64_t)seg * PLAN_STEP + (int64_t)threadIdx.x * 4;
        part += used_of(load_counts(p, seg_at), seg_at, live);
        (void)block_scan(part, below, sh);
    }
    int u = before + block_scan(mine, unused, sh);  // pages in use before the thread's first
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t page = at + i;
        if (page >= p.P) break;
        const bool used = c[i] > 0;
        int32_t map = used ? (int32_t)page : -1;
        if (page < live) {
            if (!used) to[page - u] = (int32_t)page;
        } else if (used) {
            const int k = u - below;
            from[k] = (int32_t)page;
            map = -2 - k;  // the k-th move: the kernel that makes it knows where to
        }
        p.page_map[page] = map;
        u += used ? 1 : 0;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        p.ws[0] = live - below;
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
            p.page_map[src] = dst;
        }
    }
    for (int s = blockIdx.x; s < p.S; s += gridDim.x) {
        const int held = pages_of(p, p.lens[s]);
        int32_t* row = p.table + s * p.table_s;
        for (int e = threadIdx.x; e < held; e += 256) {
            const int page = row[e];
            if ((uint32_t)page >= (uint32_t)p.P) continue;
            const int map = p.page_map[page];  // (a move's number, or by now where it went: either says the same)
            if (map >= 0) row[e] = map;
            else if (map <= -2) row[e] = to[-2 - map];
        }
    }
}

hipError_t launch_pages_compact(const PagesParams& p, hipStream_t stream) {
    const int64_t chunks = copy_chunks(p) * 2 * p.layers;
    if (chunks > 0x7fffffffLL) return hipErrorInvalidValue;
    const int segments = (p.P + PLAN_STEP - 1) / PLAN_STEP;
    if (segments > 1) hipLaunchKernelGGL(pages_compact_count_kernel, dim3(segments), dim3(PLAN_THREADS), 0, stream, p);
    hipLaunchKernelGGL(pages_compact_plan_kernel, dim3(segments), dim3(PLAN_THREADS), 0, stream, p);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(pages_compact_apply_kernel, dim3(COMPACT_BLOCKS), dim3(256), 0, stream, p, (int)chunks);
    return hipGetLastError();
}

}  // namespace g4b

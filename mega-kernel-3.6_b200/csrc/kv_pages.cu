// Upkeep of a paged cache's tables: forking rows, changing their lengths (which takes and frees pages and copies a shared last
// page before it is written), and making the pool dense.
//
// Every operator is two launches.  A plan kernel of one CTA checks the request, counts, and ranks with prefix sums, so that the outcome
// does not depend on the order of threads (the only atomics are additions of whole numbers); it writes what is to be done to scratch and
// not to the tables (but for a copy of the reference counts that fork adds to).  An apply kernel over the whole GPU then writes the
// tables and moves the pages, or, where the plan found the request impossible, hands the tables on as they were.  Because everything
// that an apply thread reads of another thread's entry lies in scratch, tables may be changed where they lie.
//
// What bounds them: the copies run at memory speed (3000 pages of 36 KB: 221 MB there and back in 36 us, 6.1 TB/s); the rest is latency
// of two dependent launches and of the plan's chain of loads (fork 3 us, resize 6 to 10 us, 200 rows and 8500 pages the latter, compact 3 to 9 us).
#include "mk36_kv4.cuh"

namespace mk36 {

constexpr int kPlanThreads = 1024;
constexpr int kApplyThreads = 256;

struct PagesParams {
    const int *table_in, *lengths_in, *refs_in;
    int *table_out, *lengths_out, *refs_out, *status;
    unsigned char* pool;
    const int *new_lengths, *parents, *children;
    int pages, rows, row_pages, count, kv_heads, page_size, tiles_per_page, tile_bytes;
    FastDiv fd_row_pages;
    // scratch
    int *refs, *list, *other;                 // [pages]
    int *old_len, *new_len, *first, *source;  // [rows]; source: page to copy from (fork: row), or -1
    int* total;                               // [1]
};

// The apply kernel is launched while the plan still runs and waits here for its results.
__device__ __forceinline__ void wait_for_plan() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_apply_start() { asm volatile("griddepcontrol.launch_dependents;"); }

// Pages are ranked a segment at a time: a bit for each page, 32 of them a word, a word for each thread.
constexpr int kSegment = 32 * kPlanThreads;

struct PageBits {
    unsigned bits[kPlanThreads];
    int before[kPlanThreads];  // set bits of the segment's lower words
};

// Sum over the lower threads of the CTA; `sum` gets the sum over all.  Every thread calls it; s: 33 words.
__device__ __forceinline__ int cta_exclusive(int v, int* s, int& sum) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int inc = v;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int n = __shfl_up_sync(kFullMask, inc, off);
        if (lane >= off) inc += n;
    }
    if (lane == 31) s[warp] = inc;
    __syncthreads();
    if (warp == 0) {
        const int w = lane < (int)(blockDim.x >> 5) ? s[lane] : 0;
        int winc = w;
#pragma unroll
        for (int off = 1; off < 32; off <<= 1) {
            const int n = __shfl_up_sync(kFullMask, winc, off);
            if (lane >= off) winc += n;
        }
        s[lane] = winc - w;
        if (lane == 31) s[32] = winc;
    }
    __syncthreads();
    const int before = s[warp] + inc - v;
    sum = s[32];
    __syncthreads();
    return before;
}

// Bits of the pages [first, first + kSegment) whose reference count is 0 (free) or is not (in use), and their ranks.  Every thread of
// the plan calls it; returns the number of bits set.
template <bool kFree>
__device__ __forceinline__ int rank_pages(const int* refs, int first, int pages, PageBits& b, int* s_scan) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int k = 0;
    for (; k < 32 && first + k * kPlanThreads < pages; k += 4) {
        int count[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int page = first + (k + i) * kPlanThreads + threadIdx.x;
            count[i] = k + i < 32 && page < pages ? __ldcg(&refs[page]) : (kFree ? 1 : 0);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned word = __ballot_sync(kFullMask, kFree ? count[i] == 0 : count[i] > 0);
            if (lane == 0 && k + i < 32) b.bits[(k + i) * 32 + warp] = word;
        }
    }
    __syncthreads();
    int sum;
    const int before = cta_exclusive((int)threadIdx.x < k * 32 ? __popc(b.bits[threadIdx.x]) : 0, s_scan, sum);
    b.before[threadIdx.x] = before;
    __syncthreads();
    return sum;
}

// Whether the page first + i of a ranked segment is set, and how many below it are.
__device__ __forceinline__ bool ranked(const PageBits& b, int i, int& before) {
    const unsigned word = b.bits[i >> 5];
    before = b.before[i >> 5] + __popc(word & ((1u << (i & 31)) - 1u));
    return word >> (i & 31) & 1u;
}

__device__ __forceinline__ int pages_of(int length, int page_size) { return length > 0 ? (length - 1) / page_size + 1 : 0; }

// A plan does not write the tables that it is given, so it may read them with __ldg: such loads need not wait for the stores before them.

// ---- fork ---------------------------------------------------------------------------------------------------------------

__global__ void __launch_bounds__(kPlanThreads) kv_fork_plan_kernel(const __grid_constant__ PagesParams p) {
    __shared__ int s_bad;
    let_apply_start();
    if (threadIdx.x == 0) s_bad = 0;
#pragma unroll 4
    for (int r = threadIdx.x; r < p.rows; r += kPlanThreads) {
        p.source[r] = -1;  // parent of the row, if it becomes a child
        p.old_len[r] = __ldg(&p.lengths_in[r]);
    }
    if (p.refs_out != p.refs_in) {
#pragma unroll 8
        for (int i = threadIdx.x; i < p.pages; i += kPlanThreads) p.refs_out[i] = __ldg(&p.refs_in[i]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.count; i += kPlanThreads) {
        const int parent = p.parents[i], child = p.children[i];
        if (parent < 0 || child < 0) continue;
        if (parent >= p.rows || child >= p.rows || p.lengths_in[child] != 0) s_bad = 1;
        else if (atomicCAS(&p.source[child], -1, parent) != -1) s_bad = 1;  // the same child twice
    }
    __syncthreads();
    if (threadIdx.x == 0) *p.total = *p.status = s_bad ? -1 : 0;
}

__global__ void __launch_bounds__(kApplyThreads) kv_fork_apply_kernel(const __grid_constant__ PagesParams p) {
    wait_for_plan();
    const bool good = *p.total == 0;
    const int at = blockIdx.x * blockDim.x + threadIdx.x, step = gridDim.x * blockDim.x;
    // a child's entries come from its parent; a parent that becomes a child itself was empty, and so stays the child: nothing is read
    // that another thread writes
    for (int i = at; i < p.rows * p.row_pages; i += step) {
        int r, slot;
        fdivmod(i, p.fd_row_pages, r, slot);
        const int parent = good ? p.source[r] : -1;
        const bool shares = parent >= 0 && p.source[parent] < 0;
        const int entry = p.table_in[shares ? parent * p.row_pages + slot : i];
        p.table_out[i] = entry;
        if (shares && entry >= 0 && entry < p.pages) atomicAdd(&p.refs_out[entry], 1);
    }
    for (int i = at; i < p.rows; i += step) {
        const int parent = good ? p.source[i] : -1;
        p.lengths_out[i] = p.old_len[parent >= 0 ? parent : i];
    }
}

// ---- resize -------------------------------------------------------------------------------------------------------------

__global__ void __launch_bounds__(kPlanThreads) kv_resize_plan_kernel(const __grid_constant__ PagesParams p) {
    __shared__ int s_bad, s_scan[33], s_rows, s_row[kPlanThreads];
    __shared__ PageBits s_bits;
    const int capacity = p.row_pages * p.page_size;
    let_apply_start();
    if (threadIdx.x == 0) s_bad = 0;
#pragma unroll 8
    for (int i = threadIdx.x; i < p.pages; i += kPlanThreads) p.refs[i] = __ldg(&p.refs_in[i]);
    for (int base = 0; base < p.rows; base += kPlanThreads) {
        // the rows that shrink are listed (in any order: what follows are sums), then a warp for each gives back what lies behind its new end
        if (threadIdx.x == 0) s_rows = 0;
        __syncthreads();
        const int row = base + threadIdx.x;
        if (row < p.rows) {
            const int a = __ldg(&p.lengths_in[row]), b = __ldg(&p.new_lengths[row]);
            p.old_len[row] = a;
            p.new_len[row] = b;
            if (a < 0 || b < 0 || a > capacity || b > capacity) s_bad = 1;
            else if (pages_of(b, p.page_size) < pages_of(a, p.page_size)) s_row[atomicAdd(&s_rows, 1)] = row;
        }
        __syncthreads();
        for (int x = threadIdx.x >> 5; x < s_rows; x += kPlanThreads / 32) {
            const int r = s_row[x], n = pages_of(p.old_len[r], p.page_size);
            for (int i = pages_of(p.new_len[r], p.page_size) + (threadIdx.x & 31); i < n; i += 32) {
                const int page = p.table_in[r * p.row_pages + i];
                if (page < 0 || page >= p.pages) s_bad = 1;
                else atomicSub(&p.refs[page], 1);
            }
        }
        __syncthreads();
    }
    const bool bad_lengths = s_bad != 0;
    __syncthreads();  // every thread has read it before one may set it again: the way below has barriers
    int need_total = 0, found = 0;
    if (!bad_lengths) {
        for (int base = 0; base < p.rows; base += kPlanThreads) {
            const int r = base + threadIdx.x;
            int need = 0, source = -1;
            if (r < p.rows) {
                const int a = p.old_len[r], b = p.new_len[r], n = pages_of(a, p.page_size);
                if (b > a) {
                    need = pages_of(b, p.page_size) - n;
                    if (a % p.page_size != 0) {
                        const int page = p.table_in[r * p.row_pages + n - 1];
                        if (page < 0 || page >= p.pages) s_bad = 1;
                        else if (__ldcg(&p.refs[page]) > 1) source = page, ++need;
                    }
                }
            }
            int sum;
            const int before = cta_exclusive(need, s_scan, sum);
            if (r < p.rows) {
                p.first[r] = need_total + before;
                p.source[r] = source;
            }
            need_total += sum;
        }
        // free pages in ascending order, as many as are needed
        for (int first = 0; first < p.pages && found < need_total; first += kSegment) {
            const int free = rank_pages<true>(p.refs, first, p.pages, s_bits, s_scan);
            const int end = min(kSegment, p.pages - first);
            for (int i = threadIdx.x; i < end; i += kPlanThreads) {
                int rank;
                if (ranked(s_bits, i, rank) && found + rank < need_total) p.list[found + rank] = first + i;
            }
            found += free;
            __syncthreads();
        }
    }
    __syncthreads();
    const int status = s_bad ? -1 : max(0, need_total - found);
    if (status == 0) {
        for (int r = threadIdx.x; r < p.rows; r += kPlanThreads)
            if (p.source[r] >= 0) atomicSub(&p.refs[p.source[r]], 1);
        for (int i = threadIdx.x; i < need_total; i += kPlanThreads) p.refs[p.list[i]] = 1;
    } else {
        for (int i = threadIdx.x; i < p.pages; i += kPlanThreads) p.refs[i] = p.refs_in[i];
    }
    if (threadIdx.x == 0) *p.total = *p.status = status;
}

// Copies `bytes` (a multiple of 16, both aligned) by one warp.
__device__ __forceinline__ void warp_copy(unsigned char* to, const unsigned char* from, int bytes) {
    const uint4* a = reinterpret_cast<const uint4*>(from);
    uint4* b = reinterpret_cast<uint4*>(to);
    const int n = bytes / 16;
    int i = threadIdx.x & 31;
    for (; i + 96 < n; i += 128) {
        const uint4 x0 = a[i], x1 = a[i + 32], x2 = a[i + 64], x3 = a[i + 96];
        b[i] = x0, b[i + 32] = x1, b[i + 64] = x2, b[i + 96] = x3;
    }
    for (; i < n; i += 32) b[i] = a[i];
}

__global__ void __launch_bounds__(kApplyThreads) kv_resize_apply_kernel(const __grid_constant__ PagesParams p) {
    wait_for_plan();
    const bool good = *p.total == 0;
    const int at = blockIdx.x * blockDim.x + threadIdx.x, step = gridDim.x * blockDim.x;
    for (int i = at; i < p.rows * p.row_pages; i += step) {
        int r, slot;
        fdivmod(i, p.fd_row_pages, r, slot);
        int entry = p.table_in[i];
        if (good) {
            const int had = pages_of(p.old_len[r], p.page_size), gets = pages_of(p.new_len[r], p.page_size);
            const int copy = p.source[r] >= 0 ? 1 : 0;
            if (slot < had && slot >= gets) entry = -1;
            else if (slot >= had && slot < gets) entry = p.list[p.first[r] + copy + slot - had];
            else if (copy && slot == had - 1) entry = p.list[p.first[r]];
        }
        p.table_out[i] = entry;
    }
    for (int i = at; i < p.rows; i += step) p.lengths_out[i] = good ? p.new_len[i] : p.old_len[i];
    for (int i = at; i < p.pages; i += step) p.refs_out[i] = p.refs[i];
    if (!good) return;
    // the tiles of a shared last page that hold tokens, a warp for each (row, head, tile)
    const int per_page = p.kv_heads * p.tiles_per_page;
    for (long long u = at >> 5; u < (long long)p.rows * per_page; u += step >> 5) {
        const int r = (int)(u / per_page), inner = (int)(u - (long long)r * per_page);
        if (p.source[r] < 0 || inner % p.tiles_per_page * kKv4Tile >= p.old_len[r] % p.page_size) continue;
        warp_copy(p.pool + ((long long)p.list[p.first[r]] * per_page + inner) * p.tile_bytes, p.pool + ((long long)p.source[r] * per_page + inner) * p.tile_bytes,
                  p.tile_bytes);
    }
}

// ---- compact ------------------------------------------------------------------------------------------------------------

__global__ void __launch_bounds__(kPlanThreads) kv_compact_plan_kernel(const __grid_constant__ PagesParams p) {
    __shared__ int s_scan[33];
    __shared__ PageBits s_bits;
    let_apply_start();
    int n = 0;
    for (int first = 0; first < p.pages; first += kSegment) n += rank_pages<false>(p.refs_in, first, p.pages, s_bits, s_scan);
    // The pages in use among the first n stay.  The i-th free page among the first n and the i-th page in use behind them follow from
    // the number of pages in use before a page.
    int before = 0, front = n;
    for (int first = 0; first < p.pages; first += kSegment) {
        // one segment is still there from the count
        const int used_here = p.pages > kSegment ? rank_pages<false>(p.refs_in, first, p.pages, s_bits, s_scan) : n;
        const int end = min(kSegment, p.pages - first);
        if (n >= first && n < first + end) {
            int rank;
            ranked(s_bits, n - first, rank);
            front = before + rank;
        }
#pragma unroll 4
        for (int i = threadIdx.x; i < end; i += kPlanThreads) {
            const int page = first + i, refs = __ldg(&p.refs_in[page]);
            int rank;
            if (ranked(s_bits, i, rank)) {
                if (page >= n) p.other[before + rank - front] = page;
            } else if (page < n) {
                p.list[page - before - rank] = page;
            }
            p.refs[page] = page < n ? refs : 0;
        }
        before += used_here;
        __syncthreads();
    }
    const int movers = n - front;
    // a moved page's place in `refs` behind the first n holds its new number, as -1 - number, until the tables are renamed
    for (int i = threadIdx.x; i < movers; i += kPlanThreads) {
        p.refs[p.list[i]] = p.refs_in[p.other[i]];
        p.refs[p.other[i]] = -1 - p.list[i];
    }
    if (threadIdx.x == 0) {
        *p.total = movers;
        *p.status = n;
    }
}

__global__ void __launch_bounds__(kApplyThreads) kv_compact_apply_kernel(const __grid_constant__ PagesParams p) {
    wait_for_plan();
    const int moves = *p.total;
    const int at = blockIdx.x * blockDim.x + threadIdx.x, step = gridDim.x * blockDim.x;
    const int tiles = p.kv_heads * p.tiles_per_page;
    for (long long u = at >> 5; u < (long long)moves * tiles; u += step >> 5) {
        const int i = (int)(u / tiles), inner = (int)(u - (long long)i * tiles);
        warp_copy(p.pool + ((long long)p.list[i] * tiles + inner) * p.tile_bytes, p.pool + ((long long)p.other[i] * tiles + inner) * p.tile_bytes, p.tile_bytes);
    }
    for (int i = at; i < p.rows * p.row_pages; i += step) {
        int entry = p.table_in[i];
        if (entry >= 0 && entry < p.pages && p.refs[entry] < 0) entry = -1 - p.refs[entry];
        p.table_out[i] = entry;
    }
    for (int i = at; i < p.rows; i += step) p.lengths_out[i] = p.lengths_in[i];
    for (int i = at; i < p.pages; i += step) p.refs_out[i] = max(p.refs[i], 0);
}

// ---- host ---------------------------------------------------------------------------------------------------------------

static size_t pages_scratch_ints(const mk36_kv_pages_args* a) { return 3 * (size_t)a->pages + 4 * (size_t)a->rows + 1; }

static int pages_params(const mk36_kv_pages_args* a, const char* what, bool pool, PagesParams* p) {
    if (!a) MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: args is NULL", what);
    if (!a->page_table_in || !a->lengths_in || !a->refcounts_in || !a->page_table_out || !a->lengths_out || !a->refcounts_out || !a->status)
        MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: NULL tensor pointer", what);
    if (a->pages <= 0 || a->rows <= 0 || a->row_pages <= 0) MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: sizes must be positive", what);
    if (a->pages > 0x3fffffffLL) MK36_FAIL(MK36_ERR_UNSUPPORTED, "%s: more than 2^30 - 1 pages", what);
    if (((long long)a->row_pages + 1) * a->rows > 0x3fffffffLL) MK36_FAIL(MK36_ERR_UNSUPPORTED, "%s: more than 2^30 - 1 table entries", what);
    *p = PagesParams{};
    if (pool) {
        if (!a->pool) MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: NULL tensor pointer", what);
        if (a->kv_heads <= 0 || a->page_size <= 0 || a->tile_bytes <= 0) MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: sizes must be positive", what);
        if (a->page_size % kKv4Tile != 0) MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: page_size must be a multiple of %d", what, kKv4Tile);
        if (a->tile_bytes % 16 != 0 || reinterpret_cast<uintptr_t>(a->pool) % 16 != 0)
            MK36_FAIL(MK36_ERR_INVALID_ARG, "%s: the pool and its tiles must be 16-byte aligned", what);
        if ((long long)a->row_pages * a->page_size > 0x7fffff00LL) MK36_FAIL(MK36_ERR_UNSUPPORTED, "%s: more than 2^31 - 256 tokens in a row", what);
        if ((long long)a->kv_heads * (a->page_size / kKv4Tile) > 0x3fffffffLL) MK36_FAIL(MK36_ERR_UNSUPPORTED, "%s: too many heads", what);
        p->tiles_per_page = a->page_size / kKv4Tile;
    }
    p->table_in = a->page_table_in, p->lengths_in = a->lengths_in, p->refs_in = a->refcounts_in;
    p->table_out = a->page_table_out, p->lengths_out = a->lengths_out, p->refs_out = a->refcounts_out;
    p->status = a->status;
    p->pool = static_cast<unsigned char*>(a->pool);
    p->new_lengths = a->new_lengths, p->parents = a->parents, p->children = a->children;
    p->pages = (int)a->pages, p->rows = a->rows, p->row_pages = a->row_pages, p->count = a->count;
    p->kv_heads = a->kv_heads, p->page_size = a->page_size, p->tile_bytes = a->tile_bytes;
    return MK36_OK;
}

// Lays the scratch out and launches plan and apply.  `copies`: tiles that may be copied at most.
static int pages_run(const mk36_kv_pages_args* a, PagesParams p, void* workspace, size_t bytes, void* stream, const char* what,
                     void (*plan)(PagesParams), void (*apply)(PagesParams), long long copies) {
    if (!workspace || bytes < mk36_kv_pages_workspace_bytes(a) || reinterpret_cast<uintptr_t>(workspace) % 4 != 0)
        MK36_FAIL(MK36_ERR_WORKSPACE, "%s: workspace of %zu bytes is too small", what, bytes);
    const DeviceInfo* info = current_device_info();
    if (!info) return MK36_ERR_LAUNCH;
    int* w = static_cast<int*>(workspace);
    p.refs = w, p.list = w + p.pages, p.other = w + 2ll * p.pages;
    w += 3ll * p.pages;
    p.old_len = w, p.new_len = w + p.rows, p.first = w + 2ll * p.rows, p.source = w + 3ll * p.rows, p.total = w + 4ll * p.rows;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    p.fd_row_pages = make_fastdiv((unsigned)p.row_pages);
    plan<<<1, kPlanThreads, 0, s>>>(p);
    MK36_CUDA_OK(cudaGetLastError());
    const long long most = (long long)info->sm_count * (2048 / kApplyThreads);
    const long long threads = (long long)p.rows * p.row_pages + p.pages + copies * 32;
    const long long ctas = (threads + kApplyThreads - 1) / kApplyThreads;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3((unsigned)(ctas < most ? ctas : most));
    config.blockDim = dim3(kApplyThreads);
    config.stream = s;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = 1;
    MK36_CUDA_OK(cudaLaunchKernelEx(&config, apply, p));
    return MK36_OK;
}

}  // namespace mk36

using namespace mk36;

extern "C" size_t mk36_kv_pages_workspace_bytes(const mk36_kv_pages_args* a) {
    if (!a || a->pages <= 0 || a->rows <= 0) return 0;
    return pages_scratch_ints(a) * sizeof(int);
}

extern "C" int mk36_kv_pages_fork(const mk36_kv_pages_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    PagesParams p;
    const int rc = pages_params(a, "kv_pages_fork", false, &p);
    if (rc != MK36_OK) return rc;
    if (a->count < 0 || (a->count > 0 && (!a->parents || !a->children))) MK36_FAIL(MK36_ERR_INVALID_ARG, "kv_pages_fork: parents and children are missing");
    return pages_run(a, p, workspace, workspace_bytes, stream, "kv_pages_fork", kv_fork_plan_kernel, kv_fork_apply_kernel, 0);
}

extern "C" int mk36_kv_pages_resize(const mk36_kv_pages_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    PagesParams p;
    const int rc = pages_params(a, "kv_pages_resize", true, &p);
    if (rc != MK36_OK) return rc;
    if (!a->new_lengths) MK36_FAIL(MK36_ERR_INVALID_ARG, "kv_pages_resize: new_lengths is NULL");
    return pages_run(a, p, workspace, workspace_bytes, stream, "kv_pages_resize", kv_resize_plan_kernel, kv_resize_apply_kernel,
                     (long long)p.rows * p.kv_heads * p.tiles_per_page);
}

extern "C" int mk36_kv_pages_compact(const mk36_kv_pages_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    PagesParams p;
    const int rc = pages_params(a, "kv_pages_compact", true, &p);
    if (rc != MK36_OK) return rc;
    return pages_run(a, p, workspace, workspace_bytes, stream, "kv_pages_compact", kv_compact_plan_kernel, kv_compact_apply_kernel,
                     (long long)(p.pages / 2) * p.kv_heads * p.tiles_per_page);
}

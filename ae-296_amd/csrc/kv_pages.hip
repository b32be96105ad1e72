// The cache's pages as the device keeps them: every row of a table (a request, a beam) names the pages of its tokens, several rows may name one
// page, and refs counts them.  A bit for every page says that it can be handed out.
//
// resize gives every row its new length: pages behind a shorter end go back, a longer one gets the lowest free ids, row by row, and a row that
// will write on a page others name as well gets a copy of what it holds there.  fork lets rows go on from other rows' tokens, sharing their
// pages.  compact moves the pages in use to the lowest ids.  Which id a page gets depends on the tables alone: ids are dealt out by sums over rows
// and bits, and counts are changed by atomics whose order no result shows.
//
// Replaces the reference's reference-counted allocator on the device (lightllm/common/mem_manager.py:4-111), which looks free places up
// by host calls that wait for the device; here nothing waits, so a step may be captured.
#include "mlora_dev.hpp"
#include "mlora_step.hpp"

namespace mlora {

constexpr int ASSIGN_NT = 1024;

__device__ __forceinline__ int read_now(const int32_t *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ int pages_of(int tokens, int shift, int most)
{
    if (tokens <= 0) return 0;
    const int n = (int)(((unsigned)tokens + (1u << shift) - 1u) >> shift);
    return n < most ? n : most;
}
__device__ __forceinline__ void set_free(const PagesArgs &p, int page)
{
    atomicOr(reinterpret_cast<unsigned long long *>(p.free_bits) + (page >> 6), 1ull << (page & 63));
}
__device__ __forceinline__ void drop_page(const PagesArgs &p, int page)
{
    if (page >= 0 && page < p.n_pages && atomicSub(p.refs + page, 1) == 1) set_free(p, page);
}

// Exclusive sum over the workgroup's ASSIGN_NT threads; `total` is everyone's.  Two barriers.
__device__ __forceinline__ unsigned block_scan(unsigned v, unsigned *lds, unsigned &total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned upto = wave_scan(v);
    if (lane == 63) lds[wave] = upto;
    __syncthreads();
    unsigned before = 0;
    total = 0;
    for (int i = 0; i < ASSIGN_NT / 64; i++) {
        const unsigned s = lds[i];
        if (i < wave) before += s;
        total += s;
    }
    __syncthreads();
    return before + upto - v;
}

// ------------------------------------------------------------------ resize
// Rows that get shorter give their last pages back: a wavefront a row.
__global__ __launch_bounds__(256) void pages_release_kernel(const PagesArgs p)
{
    const int r = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (r >= p.n_req) return;
    const int old = p.lens[r], want = p.want[r];
    if (want < 0 || want >= old) return;
    int32_t *row = p.table + (size_t)r * p.max_pages;
    const int had = pages_of(old, p.page_shift, p.max_pages);
    for (int i = pages_of(want, p.page_shift, p.max_pages) + lane; i < had; i += 64) {
        const int page = row[i];
        row[i] = -1;
        drop_page(p, page);
    }
    if (lane == 0) p.lens[r] = want;
}

struct GrowRow { bool longer, fits; int old, want, had, gets, part, at; };
__device__ __forceinline__ GrowRow grow_row(const PagesArgs &p, int r)
{
    GrowRow g;
    g.old = p.lens[r]; g.want = p.want[r];
    if (g.old < 0) g.old = 0;
    g.longer = g.want > g.old;
    g.fits = g.longer && (long long)g.want <= (long long)p.max_pages << p.page_shift;
    g.had = pages_of(g.old, p.page_shift, p.max_pages);
    g.gets = g.fits ? pages_of(g.want, p.page_shift, p.max_pages) : g.had;
    g.part = g.old & ((1 << p.page_shift) - 1);
    g.at = g.old >> p.page_shift;
    return g;
}

// Everything that depends on the order of the rows, in one workgroup.
__global__ __launch_bounds__(ASSIGN_NT) void pages_assign_kernel(const PagesArgs p)
{
    __shared__ unsigned lds[ASSIGN_NT / 64];
    __shared__ unsigned granted, failed, copies;
    const int tid = threadIdx.x;
    const int words = (int)((p.n_pages + 63) >> 6);
    unsigned long long *bits = reinterpret_cast<unsigned long long *>(p.free_bits);
    if (tid == 0) { granted = 0; failed = 0; copies = 0; }
    // which rows write on pages that others name, and how many rows do so on each
    for (int r = tid; r < p.n_req; r += ASSIGN_NT) {
        const GrowRow g = grow_row(p, r);
        int page = -1;
        if (g.fits && g.part) {
            page = p.table[(size_t)r * p.max_pages + g.at];
            if (page < 0 || page >= p.n_pages || p.refs[page] <= 1) page = -1;
        }
        p.row_page[r] = page;
        if (page >= 0) {
            atomicAdd(p.writers + page, 1);
            atomicMax(p.last_writer + page, r + 1);
        }
    }
    unsigned mine = 0, n_free;
    for (int w = tid; w < words; w += ASSIGN_NT) mine += __builtin_popcountll(bits[w]);
    block_scan(mine, lds, n_free);
    // the rows' needs in their order
    unsigned before = 0;
    for (int r0 = 0; r0 < p.n_req; r0 += ASSIGN_NT) {
        const int r = r0 + tid;
        GrowRow g = {};
        int page = -1;
        bool copy = false;
        if (r < p.n_req) {
            g = grow_row(p, r);
            page = p.row_page[r];
            copy = page >= 0 && !(read_now(p.writers + page) == p.refs[page] && read_now(p.last_writer + page) == r + 1);
        }
        const unsigned need = (unsigned)(g.gets - g.had) + (copy ? 1u : 0u);
        unsigned sum;
        const unsigned first = before + block_scan(need, lds, sum), upto = first + need;
        before += sum;
        const bool served = g.fits && (upto <= n_free || (need == 0 && page < 0));
        if (g.longer && !served) atomicAdd(&failed, 1u);
        if (served && upto <= n_free) atomicMax(&granted, upto);
        if (r < p.n_req) {
            p.row_new[3 * r] = served ? g.gets - g.had : 0;
            p.row_new[3 * r + 1] = g.had;
            p.row_new[3 * r + 2] = (int)(first + (copy ? 1u : 0u));
            if (served) p.lens[r] = g.want;
            if (served && copy) {
                int32_t *job = p.copies + 5 * atomicAdd(&copies, 1u);
                job[0] = page; job[1] = (int)first; job[2] = g.part; job[3] = r; job[4] = g.at;
            }
        }
    }
    __syncthreads();
    // the lowest free ids, as many as are granted
    const unsigned n = granted;
    unsigned done = 0;
    for (int w0 = 0; w0 < words && done < n; w0 += ASSIGN_NT) {
        const int w = w0 + tid;
        unsigned long long word = w < words ? bits[w] : 0ull;
        unsigned sum;
        unsigned rank = done + block_scan((unsigned)__builtin_popcountll(word), lds, sum);
        done += sum;
        if (word && rank < n) {
            do {
                p.picked[rank++] = w * 64 + __builtin_ctzll(word);
                word &= word - 1;
            } while (word && rank < n);
            bits[w] = word;
        }
    }
    __syncthreads();
    for (int r = tid; r < p.n_req; r += ASSIGN_NT) {
        const int page = p.row_page[r];
        if (page >= 0) { p.writers[page] = 0; p.last_writer[page] = 0; }
    }
    for (unsigned c = tid; c < copies; c += ASSIGN_NT) {
        int32_t *job = p.copies + 5 * c;
        const int to = p.picked[job[1]];
        job[1] = to;
        p.table[(size_t)job[3] * p.max_pages + job[4]] = to;
        p.refs[to] = 1;
        atomicSub(p.refs + job[0], 1);
    }
    if (tid == 0) {
        p.head[0] = (int)copies;
        *p.failed += (int)failed;
    }
}

// Copies `tokens` tokens of every head of a page by a workgroup; unit: keys or values (the lower bit) of one layer.
__device__ __forceinline__ void copy_tokens(const PagesArgs &p, long long unit, int from, int to, int tokens)
{
    uint16_t *base = ((unit & 1) ? p.v : p.k) + (unit >> 1) * p.n_pages * p.n_kv_heads * p.head_elems;
    const uint16_t *src = base + (long long)from * p.n_kv_heads * p.head_elems;
    uint16_t *dst = base + (long long)to * p.n_kv_heads * p.head_elems;
    const int chunks = (p.head_elems >> p.page_shift) * tokens / 8;
    for (int i = threadIdx.x; i < chunks * p.n_kv_heads; i += 256) {
        const int h = i / chunks, at = h * p.head_elems + (i - h * chunks) * 8;
        stg16(dst + at, ldg16(src + at));
    }
}

// The rows' new pages enter their tables, and shared pages are copied: all that is wide.
__global__ __launch_bounds__(256) void pages_fill_kernel(const PagesArgs p)
{
    const int lane = threadIdx.x & 63;
    for (int r = blockIdx.x * 4 + (threadIdx.x >> 6); r < p.n_req; r += gridDim.x * 4) {
        const int n = p.row_new[3 * r], had = p.row_new[3 * r + 1], first = p.row_new[3 * r + 2];
        for (int i = lane; i < n; i += 64) {
            const int page = p.picked[first + i];
            p.table[(size_t)r * p.max_pages + had + i] = page;
            p.refs[page] = 1;
        }
    }
    const long long per = 2ll * p.n_layers, units = p.head[0] * per;
    for (long long u = blockIdx.x; u < units; u += gridDim.x) {
        const int32_t *job = p.copies + 5 * (u / per);
        copy_tokens(p, u % per, job[0], job[1], job[2]);
    }
}

int launch_pages_resize(const PagesArgs &a, hipStream_t s)
{
    const unsigned rows = (unsigned)(a.n_req + 3) / 4;
    hipLaunchKernelGGL(pages_release_kernel, dim3(rows), dim3(256), 0, s, a);
    hipLaunchKernelGGL(pages_assign_kernel, dim3(1), dim3(ASSIGN_NT), 0, s, a);
    hipLaunchKernelGGL(pages_fill_kernel, dim3(4u * device_compute_units()), dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

// ------------------------------------------------------------------ fork
// A row's parent, or -1 where it goes on by itself.
__device__ __forceinline__ int parent_of(const PagesArgs &p, int r)
{
    const int of = p.want[r];
    return of >= 0 && of < p.n_req && of != r ? of : -1;
}

// What the rows will be, from what all rows are: kept aside, with the new holders counted, before any row changes.  -2: as it is.
__global__ __launch_bounds__(256) void pages_fork_kernel(const PagesArgs p)
{
    const int r = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (r >= p.n_req) return;
    if (p.want[r] >= p.n_req && lane == 0) atomicAdd(p.failed, 1);
    const int of = parent_of(p, r);
    if (of < 0) return;
    const int had = pages_of(p.lens[r], p.page_shift, p.max_pages), gets = pages_of(p.lens[of], p.page_shift, p.max_pages);
    const int32_t *mine = p.table + (size_t)r * p.max_pages, *its = p.table + (size_t)of * p.max_pages;
    for (int i = lane; i < gets; i += 64) {
        const int page = its[i];
        const bool same = i < had && mine[i] == page;
        p.rows[(size_t)r * p.max_pages + i] = same ? -2 : page;
        if (!same && page >= 0 && page < p.n_pages) atomicAdd(p.refs + page, 1);
    }
    if (lane == 0) p.row_page[r] = p.lens[of];
}

__global__ __launch_bounds__(256) void pages_forked_kernel(const PagesArgs p)
{
    const int r = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (r >= p.n_req) return;
    if (parent_of(p, r) < 0) return;
    const int tokens = p.row_page[r];
    const int had = pages_of(p.lens[r], p.page_shift, p.max_pages), gets = pages_of(tokens, p.page_shift, p.max_pages);
    int32_t *mine = p.table + (size_t)r * p.max_pages;
    for (int i = lane; i < (had > gets ? had : gets); i += 64) {
        const int page = i < gets ? p.rows[(size_t)r * p.max_pages + i] : -1;
        if (page == -2) continue;
        if (i < had) drop_page(p, mine[i]);
        mine[i] = page;
    }
    if (lane == 0) p.lens[r] = tokens;
}

int launch_pages_fork(const PagesArgs &a, hipStream_t s)
{
    const unsigned rows = (unsigned)(a.n_req + 3) / 4;
    hipLaunchKernelGGL(pages_fork_kernel, dim3(rows), dim3(256), 0, s, a);
    hipLaunchKernelGGL(pages_forked_kernel, dim3(rows), dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

// ------------------------------------------------------------------ compact
// Which pages move where: with n pages in use, those beyond the n-th of all managed ids go, in their order, to the free ones before it.
__global__ __launch_bounds__(ASSIGN_NT) void pages_moves_kernel(const PagesArgs p)
{
    __shared__ unsigned lds[ASSIGN_NT / 64];
    __shared__ int border;
    const int tid = threadIdx.x;
    const int words = (int)((p.n_pages + 63) >> 6);
    unsigned long long *bits = reinterpret_cast<unsigned long long *>(p.free_bits);
    const unsigned long long *managed = reinterpret_cast<const unsigned long long *>(p.managed);
    unsigned mine = 0, n;
    for (int w = tid; w < words; w += ASSIGN_NT) mine += __builtin_popcountll(managed[w] & ~bits[w]);
    block_scan(mine, lds, n);
    if (tid == 0) border = (int)p.n_pages;
    __syncthreads();
    unsigned done = 0;
    for (int w0 = 0; w0 < words; w0 += ASSIGN_NT) {
        const int w = w0 + tid;
        unsigned long long m = w < words ? managed[w] : 0ull;
        unsigned sum;
        const unsigned rank = done + block_scan((unsigned)__builtin_popcountll(m), lds, sum);
        done += sum;
        if (n >= rank && n - rank < (unsigned)__builtin_popcountll(m)) {
            for (unsigned i = rank; i < n; i++) m &= m - 1;
            border = w * 64 + __builtin_ctzll(m);
        }
        if (done > n) break;
    }
    __syncthreads();
    const int B = border;
    unsigned from = 0, to = 0;
    for (int w0 = 0; w0 < words; w0 += ASSIGN_NT) {
        const int w = w0 + tid;
        const unsigned long long m = w < words ? managed[w] : 0ull, f = w < words ? bits[w] : 0ull;
        const unsigned long long below = B >= w * 64 + 64 ? ~0ull : B <= w * 64 ? 0ull : (1ull << (B - w * 64)) - 1;
        unsigned long long holes = f & below, movers = m & ~f & ~below;
        unsigned sum_f, sum_t;
        unsigned rf = from + block_scan((unsigned)__builtin_popcountll(movers), lds, sum_f);
        unsigned rt = to + block_scan((unsigned)__builtin_popcountll(holes), lds, sum_t);
        from += sum_f;
        to += sum_t;
        if (w < words) {
            p.word_rank[w] = (int)rf;
            reinterpret_cast<unsigned long long *>(p.word_movers)[w] = movers;
            bits[w] = m & ~below;
        }
        for (; movers; movers &= movers - 1) p.move_from[rf++] = w * 64 + __builtin_ctzll(movers);
        for (; holes; holes &= holes - 1) p.picked[rt++] = w * 64 + __builtin_ctzll(holes);
    }
    if (tid == 0) {
        p.head[0] = (int)from;
        *p.live = (int)n;
    }
}

__global__ __launch_bounds__(256) void pages_move_kernel(const PagesArgs p)
{
    const int lane = threadIdx.x & 63, moves = p.head[0];
    if (moves == 0) return;
    const unsigned long long *movers = reinterpret_cast<const unsigned long long *>(p.word_movers);
    for (int r = blockIdx.x * 4 + (threadIdx.x >> 6); r < p.n_req; r += gridDim.x * 4) {
        int32_t *row = p.table + (size_t)r * p.max_pages;
        const int had = pages_of(p.lens[r], p.page_shift, p.max_pages);
        for (int i = lane; i < had; i += 64) {
            const int page = row[i];
            if (page < 0 || page >= p.n_pages) continue;
            const unsigned long long m = movers[page >> 6], bit = 1ull << (page & 63);
            if (m & bit) row[i] = p.picked[p.word_rank[page >> 6] + __builtin_popcountll(m & (bit - 1))];
        }
    }
    for (int i = blockIdx.x * 256 + threadIdx.x; i < moves; i += gridDim.x * 256) {
        p.refs[p.picked[i]] = p.refs[p.move_from[i]];
        p.refs[p.move_from[i]] = 0;
    }
    const long long per = 2ll * p.n_layers, units = moves * per;
    for (long long u = blockIdx.x; u < units; u += gridDim.x) {
        const long long i = u / per;
        copy_tokens(p, u % per, p.move_from[i], p.picked[i], 1 << p.page_shift);
    }
}

int launch_pages_compact(const PagesArgs &a, hipStream_t s)
{
    hipLaunchKernelGGL(pages_moves_kernel, dim3(1), dim3(ASSIGN_NT), 0, s, a);
    hipLaunchKernelGGL(pages_move_kernel, dim3(8u * device_compute_units()), dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

}  // namespace mlora

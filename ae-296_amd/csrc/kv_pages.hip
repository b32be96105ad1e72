// The cache's pages as the device keeps them: every row of a table (a request, a beam) names the pages of its tokens, several rows may name one
// page, and refs counts them.  A byte for every page says that it can be handed out: a byte is stored without an atomic, where bits of pages with
// neighbouring ids, which rows mostly have, meet in one word (2048 pages of a row given back by a workgroup: 28 us in bits).
//
// resize gives every row its new length: pages behind a shorter end go back, a longer one gets the lowest free ids, row by row, and a row that
// will write on a page others name as well gets a copy of what it holds there.  Which rows got longer is left in grown: no other row may be written
// on, as the pages behind its end may be shared.  fork lets rows go on from other rows' tokens, sharing their
// pages.  compact moves the pages in use to the lowest ids.  Which id a page gets depends on the tables alone: ids are dealt out by sums over rows
// and bits, and counts are changed by atomics whose order no result shows.
//
// Replaces the reference's reference-counted allocator on the device (lightllm/common/mem_manager.py:4-111), which looks free places up
// by host calls that wait for the device; here nothing waits, so a step may be captured.
#include "mlora_dev.hpp"
#include "mlora_step.hpp"

namespace mlora {

constexpr int ASSIGN_NT = 1024;
constexpr long long RELEASE_ENTRIES = 1 << 16;

__device__ __forceinline__ int read_now(const int32_t *p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ int pages_of(int tokens, int shift, int most)
{
    if (tokens <= 0) return 0;
    const int n = (int)(((unsigned)tokens + (1u << shift) - 1u) >> shift);
    return n < most ? n : most;
}
// Of N pages at once, so that their counts are asked for together.  A page that is not managed is counted, but never free: looked up where the count
// has come to zero (a fork of 512 rows of up to 4096 pages 13.5 -> 13.8 us, 65536 pages given back by one workgroup 63 -> 72).  Masking free pages where
// they are read costs a step without any instead: 64 K pages 9.7 -> 10.5 us, 2 M pages 47 -> 70.
template <int N>
__device__ __forceinline__ void drop_pages(const PagesArgs &p, const int (&page)[N])
{
    int before[N];
#pragma unroll
    for (int u = 0; u < N; u++) before[u] = page[u] >= 0 && page[u] < p.n_pages ? atomicSub(p.refs + page[u], 1) : 0;
    uint8_t own[N];
#pragma unroll
    for (int u = 0; u < N; u++) own[u] = before[u] == 1 ? p.managed[page[u]] : 0;
#pragma unroll
    for (int u = 0; u < N; u++)
        if (own[u]) p.free_pages[page[u]] = 1;
}

// The bytes of 64 pages, 0 or 1, as a word, and back.
__device__ __forceinline__ unsigned long long load_word(const uint8_t *bytes, int word)
{
    unsigned long long w = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint4 v = ldg16(bytes + (size_t)word * 64 + i * 16);
        // bytes 0 .. 3 times 2^24, 2^17, 2^10, 2^3: bits 24 .. 27
        const unsigned four = ((v.x * 0x01020408u) >> 24 & 15u) | ((v.y * 0x01020408u) >> 24 & 15u) << 4 | ((v.z * 0x01020408u) >> 24 & 15u) << 8 | ((v.w * 0x01020408u) >> 24 & 15u) << 12;
        w |= (unsigned long long)four << (16 * i);
    }
    return w;
}
__device__ __forceinline__ void store_word(uint8_t *bytes, int word, unsigned long long w)
{
    auto four = [](unsigned bits) { return ((bits & 15u) * 0x00204081u) & 0x01010101u; };
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const unsigned b = (unsigned)(w >> (16 * i));
        stg16(bytes + (size_t)word * 64 + i * 16, make_uint4(four(b), four(b >> 4), four(b >> 8), four(b >> 12)));
    }
}

// A barrier behind which the workgroup's atomics and stores have been made.
__device__ __forceinline__ void settled_barrier()
{
    __builtin_amdgcn_s_waitcnt(0x0f70);                  // vector memory
    __syncthreads();
}

struct Sums { unsigned a, b; };
// Exclusive sums of two values over the workgroup's ASSIGN_NT threads; `total` is everyone's.  Two barriers.
__device__ __forceinline__ Sums block_scan(Sums v, Sums *lds, Sums &total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const Sums upto = {wave_scan(v.a), wave_scan(v.b)};
    if (lane == 63) lds[wave] = upto;
    __syncthreads();
    Sums before = {0, 0};
    total = {0, 0};
#pragma unroll
    for (int i = 0; i < ASSIGN_NT / 64; i++) {
        const Sums s = lds[i];
        if (i < wave) { before.a += s.a; before.b += s.b; }
        total.a += s.a; total.b += s.b;
    }
    __syncthreads();
    return {before.a + upto.a - v.a, before.b + upto.b - v.b};
}

// ------------------------------------------------------------------ resize
// Rows that get shorter give their last pages back: a workgroup a piece of ROW_PIECE entries of a row.
__global__ __launch_bounds__(256) void pages_release_kernel(const PagesArgs p)
{
    const int pieces = (p.max_pages + ROW_PIECE - 1) / ROW_PIECE, r = blockIdx.x / pieces, i0 = (blockIdx.x - r * pieces) * ROW_PIECE;
    const int old = p.lens[r], want = p.want[r];
    if (want < 0 || want >= old) return;
    const int had = pages_of(old, p.page_shift, p.max_pages), gets = pages_of(want, p.page_shift, p.max_pages);
    int32_t *row = p.table + (size_t)r * p.max_pages;
    int page[ROW_PIECE / 256];
#pragma unroll
    for (int u = 0; u < ROW_PIECE / 256; u++) {
        const int i = i0 + u * 256 + threadIdx.x;
        page[u] = -1;
        if (i >= gets && i < had) { page[u] = row[i]; row[i] = -1; }
    }
    drop_pages(p, page);
}

struct GrowRow { bool shorter, longer, fits; int old, want, had, gets, part, at; };
__device__ __forceinline__ GrowRow grow_row(const PagesArgs &p, int r)
{
    GrowRow g = {};
    if (r >= p.n_req) return g;
    g.old = p.lens[r]; g.want = p.want[r];
    if (g.old < 0) g.old = 0;
    g.shorter = g.want >= 0 && g.want < g.old;
    g.longer = g.want > g.old;
    g.fits = g.longer && (long long)g.want <= (long long)p.max_pages << p.page_shift;
    g.had = pages_of(g.old, p.page_shift, p.max_pages);
    g.gets = g.fits || g.shorter ? pages_of(g.want, p.page_shift, p.max_pages) : g.had;
    g.part = g.old & ((1 << p.page_shift) - 1);
    g.at = g.old >> p.page_shift;
    return g;
}

// Calls f(rank, page) for every set bit of the threads' words; rank counts the bits from a thread's own on, `first` is the number of the workgroup's first word.  (A
// thread for each word takes its up to 64 bits one after the other: 3 us.)
// few_bits: most words are zero; a wavefront goes through its own, a lane a bit.
template <typename F>
__device__ __forceinline__ void few_bits(unsigned long long word, unsigned rank, int first, F f)
{
    const int lane = threadIdx.x & 63;
    for (uint64_t left = __ballot(word != 0); left; left &= left - 1) {
        const int from = __builtin_ctzll(left);
        const unsigned long long w = (unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)(word >> 32), from) << 32 | (unsigned)__builtin_amdgcn_readlane((int)word, from);
        const unsigned r = (unsigned)__builtin_amdgcn_readlane((int)rank, from);
        if (w >> lane & 1) f(r + (unsigned)__builtin_popcountll(w & ((1ull << lane) - 1)), (first + (int)(threadIdx.x & ~63u) + from) * 64 + lane);
    }
}

// many_bits: the wavefronts take all words in turn, by way of LDS.  Two barriers.
struct Words { unsigned long long word[ASSIGN_NT]; unsigned rank[ASSIGN_NT]; };
template <typename F>
__device__ __forceinline__ void many_bits(Words &lds, unsigned long long word, unsigned rank, int first, int words, F f)
{
    const int lane = threadIdx.x & 63;
    lds.word[threadIdx.x] = word;
    lds.rank[threadIdx.x] = rank;
    __syncthreads();
    for (int i = threadIdx.x >> 6; i < ASSIGN_NT && first + i < words; i += ASSIGN_NT / 64) {
        const unsigned long long w = lds.word[i];
        if (w >> lane & 1) f(lds.rank[i] + (unsigned)__builtin_popcountll(w & ((1ull << lane) - 1)), (first + i) * 64 + lane);
    }
    __syncthreads();
}

// Everything that depends on the order of the rows, in one workgroup, a thread a row at a time.  ONE: no more rows than threads, which then keep theirs
// in registers.  RELEASE: pages are given back here as well, and there is no launch before this one.
// Bound by chains of dependent loads, each a way to the last-level cache (the tables were written on other XCDs): lengths -> the row's last page -> its count, the free
// pages beside them, and where pages are given back or shared the same again behind that.  256 rows, 18471 pages, every sixteenth row needs one: 6.0 us; as many in
// groups of four that share their last pages, a twentieth of them ending: 13.7.  Large caches: a thread reads the bytes of 64 pages in turn, twice where the lowest
// free page lies far up (2 M pages: 45 us; behind 1.2 M in use 69).
constexpr unsigned HELD_PICKS = 2048;
template <bool ONE, bool RELEASE>
__global__ __launch_bounds__(ASSIGN_NT) void pages_assign_kernel(const PagesArgs p)
{
    __shared__ Sums lds[ASSIGN_NT / 64];
    __shared__ unsigned drops_upto[ASSIGN_NT];
    __shared__ int drops_end[ASSIGN_NT];
    __shared__ int picks[HELD_PICKS];                       // the first of the picked ids
    __shared__ unsigned granted, failed, copies, widest;
    __shared__ Words held;
    const int tid = threadIdx.x;
    const int words = (int)((p.n_pages + 63) >> 6);
    if (tid == 0) { granted = 0; failed = 0; copies = 0; widest = 0; }
    unsigned long long word = tid < words ? load_word(p.free_pages, tid) : 0ull;
    const GrowRow mine = grow_row(p, tid);
    // the page a row will write on, if it has tokens of the row already, and the entries that name it
    auto written = [&](const GrowRow &g, int r) {
        const int page = g.fits && g.part ? p.table[(size_t)r * p.max_pages + g.at] : -1;
        return page >= 0 && page < p.n_pages ? page : -1;
    };
    const int my_page = written(mine, tid);
    int my_refs = my_page >= 0 ? p.refs[my_page] : 0;
    Sums total;
    bool dropped = false;
    if constexpr (RELEASE) {
        for (int r0 = 0; r0 < p.n_req; r0 += ASSIGN_NT) {
            const GrowRow g = ONE || r0 == 0 ? mine : grow_row(p, r0 + tid);
            const unsigned n = g.shorter ? (unsigned)(g.had - g.gets) : 0u;
            if (__syncthreads_or(n > 0)) {
                dropped = true;
                const unsigned first = block_scan({n, 0}, lds, total).a;
                drops_upto[tid] = first + n;
                drops_end[tid] = g.had - (int)(first + n);
                __syncthreads();
                for (unsigned i0 = tid; i0 < total.a; i0 += 4 * ASSIGN_NT) {
                    int page[4];
#pragma unroll
                    for (int u = 0; u < 4; u++) {
                        const unsigned i = i0 + u * ASSIGN_NT;
                        page[u] = -1;
                        if (i >= total.a) continue;
                        int row = 0;                        // the first whose drops go beyond i
#pragma unroll
                        for (int s = ASSIGN_NT / 2; s; s >>= 1)
                            if (drops_upto[row + s - 1] <= i) row += s;
                        int32_t *entry = p.table + (size_t)(r0 + row) * p.max_pages + (drops_end[row] + (int)i);
                        page[u] = *entry;
                        *entry = -1;
                    }
                    drop_pages(p, page);
                }
                settled_barrier();
            }
        }
        if (dropped) {                                      // counts and free pages are others now
            if (my_page >= 0) my_refs = read_now(p.refs + my_page);
            if (tid < words) word = load_word(p.free_pages, tid);
        }
    }
    // which rows write on pages that others name, and how many rows do so on each
    int page = my_refs > 1 ? my_page : -1;
    bool sharing = false;
    for (int r0 = 0; r0 < p.n_req; r0 += ASSIGN_NT) {
        const int r = r0 + tid;
        if (!ONE) {
            page = written(grow_row(p, r), r);
            if (page >= 0 && read_now(p.refs + page) <= 1) page = -1;
            if (r < p.n_req) p.row_page[r] = page;
        }
        if (page >= 0) {
            atomicAdd(p.writers + page, 1);
            atomicMax(p.last_writer + page, r + 1);
            sharing = true;
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0f70);                  // behind the barrier the writers' counts can be read
    const bool any_sharing = __syncthreads_or(sharing);
    unsigned count = (unsigned)__builtin_popcountll(word), n_free = 0, word_rank = 0;
    for (int w = tid + ASSIGN_NT; w < words; w += ASSIGN_NT) count += (unsigned)__builtin_popcountll(load_word(p.free_pages, w));
    // the rows' needs in their order
    unsigned before = 0;
    GrowRow g = mine;
    unsigned gets = 0, new_at = 0;
    bool copies_page = false;
    for (int r0 = 0; r0 < p.n_req; r0 += ASSIGN_NT) {
        const int r = r0 + tid;
        if (!ONE) {
            g = grow_row(p, r);
            page = any_sharing && r < p.n_req ? p.row_page[r] : -1;
        }
        bool copy = false;
        if (any_sharing && page >= 0) copy = !(read_now(p.writers + page) == read_now(p.refs + page) && read_now(p.last_writer + page) == r + 1);
        const unsigned need = g.fits ? (unsigned)(g.gets - g.had) + (copy ? 1u : 0u) : 0u;
        const Sums s = block_scan({need, r0 == 0 ? count : 0u}, lds, total);
        if (r0 == 0) { n_free = total.b; word_rank = s.b; }
        const unsigned first = before + s.a, upto = first + need;
        before += total.a;
        const bool served = g.fits && (upto <= n_free || (need == 0 && page < 0));
        if (g.longer && !served) atomicAdd(&failed, 1u);
        gets = served ? (unsigned)(g.gets - g.had) : 0u;
        new_at = first + (copy ? 1u : 0u);
        if (served && need) atomicMax(&granted, upto);
        if (gets > 4) atomicMax(&widest, gets);
        if (served || g.shorter) p.lens[r] = g.want;
        if (r < p.n_req) p.grown[r] = served ? r : -1;
        copies_page = served && copy;
        if (!ONE && r < p.n_req) {
            p.row_new[3 * r] = (int)gets;
            p.row_new[3 * r + 1] = g.had;
            p.row_new[3 * r + 2] = (int)new_at;
            p.row_copy[2 * r] = copies_page ? g.at : -1;
            p.row_copy[2 * r + 1] = g.part;
        }
    }
    __syncthreads();
    // the lowest free ids, as many as are granted
    const unsigned n = granted;
    const bool wide = widest > 0;
    unsigned done = 0;
    for (int w0 = 0; w0 < words && done < n; w0 += ASSIGN_NT) {
        const int w = w0 + tid;
        unsigned rank = word_rank;
        if (words > ASSIGN_NT) {
            if (w0 > 0) word = w < words ? load_word(p.free_pages, w) : 0ull;
            rank = done + block_scan({(unsigned)__builtin_popcountll(word), 0}, lds, total).a;
            done += total.a;
        } else {
            done = n;
        }
        if (rank >= n) word = 0;
        auto take = [&](unsigned nth, int id) {
            if (nth >= n) return;
            p.free_pages[id] = 0;
            if (nth < HELD_PICKS) picks[nth] = id;
            if (wide || n > HELD_PICKS) p.picked[nth] = id;
        };
        // 16 of 18471 pages: 6.5 us a call with few_bits, 8.6 with many_bits; 210 of 2675: 24.2 and 22.7
        if (n <= 64) few_bits(word, rank, w0, take);
        else many_bits(held, word, rank, w0, words, take);
    }
    if (n > HELD_PICKS) settled_barrier();                  // ids that went to memory are read below
    else __syncthreads();
    auto pick = [&](unsigned nth) { return nth < HELD_PICKS ? picks[nth] : p.picked[nth]; };
    if (any_sharing) {
        for (int r0 = 0; r0 < p.n_req; r0 += ASSIGN_NT) {
            const int r = r0 + tid;
            if (r >= p.n_req) continue;
            if (!ONE) page = p.row_page[r];
            if (page < 0) continue;
            p.writers[page] = 0;
            p.last_writer[page] = 0;
            const int at = ONE ? (copies_page ? g.at : -1) : p.row_copy[2 * r];
            if (at < 0) continue;
            const int to = pick(ONE ? new_at - 1 : (unsigned)p.row_new[3 * r + 2] - 1);
            int32_t *job = p.copies + 3 * atomicAdd(&copies, 1u);
            job[0] = page; job[1] = to; job[2] = ONE ? g.part : p.row_copy[2 * r + 1];
            p.table[(size_t)r * p.max_pages + at] = to;
            p.refs[to] = 1;
            atomicSub(p.refs + page, 1);
        }
        __syncthreads();
    }
    // a few new pages a row enter their tables here, more by the next launch
    auto enter = [&](int r, int had, unsigned from, unsigned many) {
        for (unsigned i = 0; i < many; i++) {
            const int id = pick(from + i);
            p.table[(size_t)r * p.max_pages + had + (int)i] = id;
            p.refs[id] = 1;
        }
    };
    if (ONE) {
        if (!wide) enter(tid, g.had, new_at, gets);
        else if (tid < p.n_req) { p.row_new[3 * tid] = (int)gets; p.row_new[3 * tid + 1] = g.had; p.row_new[3 * tid + 2] = (int)new_at; }
    } else if (n && !wide) {
        for (int r = tid; r < p.n_req; r += ASSIGN_NT) enter(r, p.row_new[3 * r + 1], (unsigned)p.row_new[3 * r + 2], (unsigned)p.row_new[3 * r]);
    }
    if (tid == 0) {
        p.head[0] = (int)copies;
        p.head[1] = wide;
        if (failed) *p.failed += (int)failed;
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

// What is wide: many new pages a row enter their tables, and shared pages are copied (74 MB read + written: 12.4 us; nothing to do: 2.0).
__global__ __launch_bounds__(256) void pages_fill_kernel(const PagesArgs p)
{
    if (p.head[1])
        for (int r = blockIdx.x * 4 + (threadIdx.x >> 6); r < p.n_req; r += gridDim.x * 4) {
            const int n = p.row_new[3 * r], had = p.row_new[3 * r + 1], first = p.row_new[3 * r + 2];
            for (int i = threadIdx.x & 63; i < n; i += 64) {
                const int page = p.picked[first + i];
                p.table[(size_t)r * p.max_pages + had + i] = page;
                p.refs[page] = 1;
            }
        }
    const long long per = 2ll * p.n_layers, units = p.head[0] * per;
    for (long long u = blockIdx.x; u < units; u += gridDim.x) {
        const int32_t *job = p.copies + 3 * (u / per);
        copy_tokens(p, u % per, job[0], job[1], job[2]);
    }
}

static dim3 row_pieces(const PagesArgs &a) { return dim3((unsigned)a.n_req * (unsigned)((a.max_pages + ROW_PIECE - 1) / ROW_PIECE)); }

int launch_pages_resize(const PagesArgs &a, hipStream_t s)
{
    // Pages are given back by the workgroup that hands them out, 4096 at a time, up to so many entries, else by a launch of their own.  us a call (and of the
    // tables put back), the former / the latter, where nobody ends, one row, a tenth of the rows, all rows:
    //     256 rows of  16 entries    9.1 / 10.1   11.2 / 11.2   11.2 / 11.7    13.6 / 11.0
    //     256 rows of  64            9.4 / 10.6   11.6 / 11.3   12.7 / 11.8    25.7 / 11.2
    //     256 rows of 256            9.8 / 11.0   12.5 / 11.7   18.1 / 12.2    72.4 / 11.8
    //     256 rows of 512           11.1 / 12.2   13.7 / 13.7   25.8 / 13.9   134.6 / 13.5
    // The line is where a step without an end, which saves the launch at any size, is bought by no more than 60 us of one in which everything ends.
    const bool release = (long long)a.n_req * a.max_pages <= RELEASE_ENTRIES, one = a.n_req <= ASSIGN_NT;
    if (!release) hipLaunchKernelGGL(pages_release_kernel, row_pieces(a), dim3(256), 0, s, a);
    if (one && release) hipLaunchKernelGGL((pages_assign_kernel<true, true>), dim3(1), dim3(ASSIGN_NT), 0, s, a);
    else if (one) hipLaunchKernelGGL((pages_assign_kernel<true, false>), dim3(1), dim3(ASSIGN_NT), 0, s, a);
    else if (release) hipLaunchKernelGGL((pages_assign_kernel<false, true>), dim3(1), dim3(ASSIGN_NT), 0, s, a);
    else hipLaunchKernelGGL((pages_assign_kernel<false, false>), dim3(1), dim3(ASSIGN_NT), 0, s, a);
    const long long units = 2ll * a.n_layers * a.n_req, most = 8ll * device_compute_units();
    hipLaunchKernelGGL(pages_fill_kernel, dim3((unsigned)(units < most ? units : most)), dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

// ------------------------------------------------------------------ fork
// A row's parent, or -1 where it goes on by itself.
__device__ __forceinline__ int parent_of(const PagesArgs &p, int r)
{
    const int of = p.want[r];
    return of >= 0 && of < p.n_req && of != r ? of : -1;
}

// What the rows will be, from what all rows are: kept aside, with the new holders counted, before any row changes.  A workgroup a piece of ROW_PIECE entries of a
// row; a piece that is the parent's already, as most of beams are, is marked and not copied, and so are single entries (-2).
__global__ __launch_bounds__(256) void pages_fork_kernel(const PagesArgs p)
{
    const int pieces = (p.max_pages + ROW_PIECE - 1) / ROW_PIECE, r = blockIdx.x / pieces, i0 = (blockIdx.x - r * pieces) * ROW_PIECE;
    if (p.want[r] >= p.n_req && i0 == 0 && threadIdx.x == 0) atomicAdd(p.failed, 1);
    const int of = parent_of(p, r);
    if (of < 0) return;
    const int tokens = p.lens[of], had = pages_of(p.lens[r], p.page_shift, p.max_pages), gets = pages_of(tokens, p.page_shift, p.max_pages);
    const int32_t *mine = p.table + (size_t)r * p.max_pages, *its = p.table + (size_t)of * p.max_pages;
    int page[ROW_PIECE / 256];
    bool differs = false;
#pragma unroll
    for (int u = 0; u < ROW_PIECE / 256; u++) {
        const int i = i0 + u * 256 + threadIdx.x;
        page[u] = i < gets ? its[i] : -1;
        if (i >= had ? i >= gets : page[u] == mine[i]) page[u] = -2;
        differs |= page[u] != -2;
    }
    const int any = __syncthreads_or(differs);
    if (any) {
#pragma unroll
        for (int u = 0; u < ROW_PIECE / 256; u++) {
            const int i = i0 + u * 256 + threadIdx.x;
            if (i < p.max_pages) p.rows[(size_t)r * p.max_pages + i] = page[u];
            if (page[u] >= 0 && page[u] < p.n_pages) atomicAdd(p.refs + page[u], 1);
        }
    }
    if (threadIdx.x == 0) {
        p.pieces[blockIdx.x] = any;
        if (i0 == 0) p.row_page[r] = tokens;
    }
}

__global__ __launch_bounds__(256) void pages_forked_kernel(const PagesArgs p)
{
    const int pieces = (p.max_pages + ROW_PIECE - 1) / ROW_PIECE, r = blockIdx.x / pieces, i0 = (blockIdx.x - r * pieces) * ROW_PIECE;
    const bool first = i0 == 0 && threadIdx.x == 0;
    if (parent_of(p, r) < 0) {
        if (first) p.grown[r] = -1;                         // last pages may be shared from now on
        return;
    }
    const int tokens = p.row_page[r];
    if (p.pieces[blockIdx.x]) {
        int32_t *mine = p.table + (size_t)r * p.max_pages;
        const int32_t *next = p.rows + (size_t)r * p.max_pages;
        int page[ROW_PIECE / 256], old[ROW_PIECE / 256];
#pragma unroll
        for (int u = 0; u < ROW_PIECE / 256; u++) {
            const int i = i0 + u * 256 + threadIdx.x;
            page[u] = i < p.max_pages ? next[i] : -2;
            old[u] = i < p.max_pages ? mine[i] : -1;
        }
#pragma unroll
        for (int u = 0; u < ROW_PIECE / 256; u++) {
            if (page[u] == -2) old[u] = -1;
            else mine[i0 + u * 256 + threadIdx.x] = page[u];
        }
        drop_pages(p, old);
    }
    if (first) { p.lens[r] = tokens; p.grown[r] = -1; }
}

int launch_pages_fork(const PagesArgs &a, hipStream_t s)
{
    const dim3 grid = row_pieces(a);
    hipLaunchKernelGGL(pages_fork_kernel, grid, dim3(256), 0, s, a);
    hipLaunchKernelGGL(pages_forked_kernel, grid, dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

// ------------------------------------------------------------------ compact
// Which pages move where: with n pages in use, those beyond the n-th of all managed ids go, in their order, to the free ones before it.
__global__ __launch_bounds__(ASSIGN_NT) void pages_moves_kernel(const PagesArgs p)
{
    __shared__ Sums lds[ASSIGN_NT / 64];
    __shared__ Words held;
    __shared__ int border;
    const int tid = threadIdx.x;
    const int words = (int)((p.n_pages + 63) >> 6);
    // a thread's word of the first round stays in registers
    const unsigned long long m0 = tid < words ? load_word(p.managed, tid) : 0ull, f0 = tid < words ? load_word(p.free_pages, tid) : 0ull;
    unsigned used = (unsigned)__builtin_popcountll(m0 & ~f0);
    for (int w = tid + ASSIGN_NT; w < words; w += ASSIGN_NT) used += (unsigned)__builtin_popcountll(load_word(p.managed, w) & ~load_word(p.free_pages, w));
    if (tid == 0) border = (int)p.n_pages;
    Sums total, s = block_scan({used, (unsigned)__builtin_popcountll(m0)}, lds, total);
    const unsigned n = total.a;
    unsigned done = 0;
    for (int w0 = 0; w0 < words && done <= n; w0 += ASSIGN_NT) {
        unsigned long long m = m0;
        if (w0 > 0) {
            m = w0 + tid < words ? load_word(p.managed, w0 + tid) : 0ull;
            s = block_scan({0, (unsigned)__builtin_popcountll(m)}, lds, total);
        }
        const unsigned rank = done + s.b;
        done += total.b;
        if (n >= rank && n - rank < (unsigned)__builtin_popcountll(m)) {
            for (unsigned i = rank; i < n; i++) m &= m - 1;
            border = (w0 + tid) * 64 + __builtin_ctzll(m);
        }
    }
    __syncthreads();
    const int B = border;
    unsigned from = 0, to = 0;
    for (int w0 = 0; w0 < words; w0 += ASSIGN_NT) {
        const int w = w0 + tid;
        const unsigned long long m = w0 == 0 ? m0 : w < words ? load_word(p.managed, w) : 0ull, f = w0 == 0 ? f0 : w < words ? load_word(p.free_pages, w) : 0ull;
        const unsigned long long below = B >= w * 64 + 64 ? ~0ull : B <= w * 64 ? 0ull : (1ull << (B - w * 64)) - 1;
        const unsigned long long holes = f & below, movers = m & ~f & ~below;
        s = block_scan({(unsigned)__builtin_popcountll(movers), (unsigned)__builtin_popcountll(holes)}, lds, total);
        const unsigned rf = from + s.a, rt = to + s.b;
        from += total.a;
        to += total.b;
        if (w < words) {
            p.word_rank[w] = (int)rf;
            reinterpret_cast<unsigned long long *>(p.word_movers)[w] = movers;
            store_word(p.free_pages, w, m & ~below);
        }
        many_bits(held, movers, rf, w0, words, [&](unsigned nth, int id) { p.move_from[nth] = id; });
        many_bits(held, holes, rt, w0, words, [&](unsigned nth, int id) { p.picked[nth] = id; });
    }
    if (tid == 0) {
        p.head[0] = (int)from;
        *p.live = (int)n;
    }
}

// Tables, counts, keys and values follow: HBM, at a copy's rate (1843 pages of 256 KB: 190 us, 4.8 TB/s read + written).
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
    const long long units = 2ll * a.n_layers * a.n_pages, most = 8ll * device_compute_units();
    hipLaunchKernelGGL(pages_move_kernel, dim3((unsigned)(units < most ? units : most)), dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

}  // namespace mlora

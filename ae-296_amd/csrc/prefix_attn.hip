// Attention of a batch's tokens over the paged key/value cache:
//     out[t][h] = sum_j softmax_j(scale * q[t][h] . k_j) v_j,   j over positions 0 .. tok_pos[t] of t's request
// with the keys of a shared prefix on the prefix's pages and the others on the request's own.
//
// Three kernels.  The plan (once per step) cuts the work into items: some query rows x a range of keys of one list.  The rows of an item
// are the query heads that read one key head, of one token over its own keys, or of the tokens behind a prefix over the
// prefix's.  The attention kernel runs an item per workgroup and key head: up to 32 rows with the keys shared by its wavefronts, which is
// what reading keys once takes, or up to 128 with the rows shared, each wavefront 32 of them, and the keys brought to LDS for all.  The join
// adds up the parts of rows that were cut, with their maxima and sums.
//
// One pass over the keys with the running maximum m and sum l of the softmax.  A wavefront multiplies 32 keys at a time with 16 query
// rows on v_mfma_f32_16x16x32: first S^T = K q^T, whose result leaves every lane with eight scores of ONE query row (column lane % 16; keys
// 4 g + i and 16 + 4 g + i, g = lane / 16), then out^T += V^T P^T.  The second product sums over keys, and its operands may hold the keys in
// any order as long as both use the same: with slot 8 g + j of the 32 standing for key 4 g + j (j < 4) or 12 + 4 g + j the weights are
// already where the MFMA wants them, and V^T comes out of LDS by the transposing read, four keys of one column at a time.
// K goes from global memory straight to its operand registers, since no other wavefront needs it.
#include "mlora_dev.hpp"
#include "mlora_step.hpp"

namespace mlora {

typedef short pa_short4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) pa_short4 pa_lds_short4;

template <int DT>
__device__ __forceinline__ float4_t pa_mfma(const uint4 &a, const uint4 &b, float4_t c)
{
    if constexpr (DT == DT_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf168_t, a), __builtin_bit_cast(bf168_t, b), c, 0, 0, 0);
}

constexpr int PA_WAVES = 4;
constexpr int PA_ROWS = 32;                    // query rows of an item whose wavefronts share the keys, at most
constexpr int PA_WIDE = 128;                   // of one whose wavefronts share the rows
constexpr int PA_KEYS = 32;                    // keys of a block
constexpr float PA_LOG2E = 1.44269504088896341f;

// LDS chunk (16 bytes) at which chunk c of key row r of a wavefront's V block lies: the 16 rows a transposing read touches
// at one column spread over all banks.
template <int D> __device__ __forceinline__ int pa_swizzle(int r, int c) { return D == 128 ? c ^ ((r & 7) << 1) : c ^ (((r >> 1) & 3) << 1); }

// ------------------------------------------------------------------ plan
// Item (int32 words): [0] query rows (at most PA_ROWS, or PA_WIDE of a group), [1] the token (own keys) or the first entry of the group's token list, [2] 1: a group,
// [3] first row of the group's, row r being head r % gq of list entry r / gq, [4] row of the table, [5] 1: the prefix table,
// [6], [7] keys [first, last), [8] slot of list entry 0 for this key range, -1: the rows have no other part and go to `out`.
// Join record of a token: [0] first slot of its own parts, [1] how many, [2] first slot of its prefix parts, [3] how many, [4] slots from one
// to the next.  A slot holds the gq rows of every key head.
constexpr int PA_ITEM = 12, PA_JOIN = 8;
constexpr int PL_THREADS = 1024;
constexpr int PL_PREFIXES = 4096;     // prefixes at most

struct PlanView {
    int32_t *n_items;       // [4]
    int32_t *list;          // [T] tokens of the groups
    int32_t *join;          // [T][PA_JOIN]
    int32_t *items;         // [cap][PA_ITEM]
};

// Ranges of keys that fill the device: two workgroups a compute unit.  Twice as many cost more in parts than they level out (128 requests
// over one prefix of 8191 keys: a tenth more a layer).
__host__ __device__ inline int pa_target(int n_kv_heads) { const int t = 512 / n_kv_heads; return t < 1 ? 1 : t; }

// With C keys a range where C >= (sum of own keys + sum over groups of keys x row tiles) / target, a list is cut into at most
// keys / C + 1 ranges, which bounds the items and the slots by sizes the host knows.
// Groups may be cut up to twice as finely.
inline int64_t pa_items_cap(int T, int n_prefix, int gq, int n_kv_heads)
{
    const int64_t groups = T < n_prefix ? T : n_prefix, tiles = (int64_t)T * gq / PA_ROWS + groups, own_tiles = (gq + PA_ROWS - 1) / PA_ROWS;
    return T * own_tiles + (n_prefix ? tiles + pa_target(n_kv_heads) : 0) + pa_target(n_kv_heads) * own_tiles + 1;
}
inline int64_t pa_slots_cap(int T, int n_prefix, int gq, int n_kv_heads)
{
    const int64_t target = pa_target(n_kv_heads) * (n_prefix ? 2 : 1), per_tile = (PA_WIDE + gq - 1) / gq;
    return (int64_t)T * (n_prefix ? 2 : 1) + target * (n_prefix ? per_tile : 1) + 1;
}

__host__ __device__ inline PlanView pa_plan_view(void *plan, int T)
{
    int32_t *p = static_cast<int32_t *>(plan);
    return {p, p + 4, p + 4 + (T + 3) / 4 * 4, p + 4 + (T + 3) / 4 * 4 + (size_t)T * PA_JOIN};
}

struct PlanArgs {
    KvBatch b;
    void *plan;
    int page_shift, gq, target, head_dim;
    long long items_cap, slots_cap;
};

// What a token reads.  An own list, or the part of its prefix that it sees where it stands inside of it (then it is no member of
// the group); keys behind the table's end are absent.
struct TokenRun { int prefix; int own; int table, row; };       // prefix: the group, -1 none
__device__ __forceinline__ TokenRun pa_token(const KvBatch &b, int page_shift, int t)
{
    TokenRun r = {-1, 0, 0, 0};
    const int req = b.tok_req[t], pos = b.tok_pos[t];
    if (req < 0 || req >= b.n_req) return r;
    r.row = req;
    long long base = 0;
    if (b.req_prefix) {
        const int f = b.req_prefix[req];
        if (f >= 0 && f < b.n_prefix) {
            base = max(b.prefix_len[f], 0);
            const long long there = min(base, (long long)b.max_prefix_pages << page_shift), seen = min((long long)pos + 1, there);
            if (seen == there) { if (there > 0) r.prefix = f; }
            else { r.own = (int)max(seen, 0LL); r.table = 1; r.row = f; return r; }
        }
    }
    r.own = (int)max(min((long long)pos + 1 - base, (long long)b.max_pages << page_shift), 0LL);
    return r;
}

// Exclusive sum of v over the workgroup's threads; *total: the sum.  `scratch`: a value per wavefront.
__device__ __forceinline__ int pl_scan(int v, int *scratch, int *total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int upto = (int)wave_scan((uint32_t)v);
    __syncthreads();
    if (lane == 63) scratch[wave] = upto;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < PL_THREADS / 64; w++) { const int x = scratch[w]; before += w < wave ? x : 0; all += x; }
    *total = all;
    return before + upto - v;
}

__device__ __forceinline__ int pl_find(const int *first, int n, int i)       // last entry e with first[e] <= i
{
    int lo = 0, hi = n;
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (first[mid] <= i) lo = mid; else hi = mid; }
    return lo;
}

// One workgroup, bound by its scans and barriers: 5.5 us for one request, 8.4 for 256 requests behind 8 prefixes, once a step.
// Tokens enter their group's list in any order (LDS atomics): a row's arithmetic does not depend on its place in a tile.
__global__ __launch_bounds__(PL_THREADS) void pa_plan_kernel(const PlanArgs p)
{
    __shared__ int s_count[PL_PREFIXES], s_list[PL_PREFIXES], s_slot[PL_PREFIXES], s_item[PL_PREFIXES], s_scan[PL_THREADS / 64];
    __shared__ int s_first[PL_THREADS], s_own[PL_THREADS], s_row[PL_THREADS], s_part[PL_THREADS];
    __shared__ unsigned long long s_work;
    const int T = p.b.T, F = p.b.req_prefix ? p.b.n_prefix : 0;
    const PlanView v = pa_plan_view(p.plan, T);
    for (int f = threadIdx.x; f < F; f += PL_THREADS) s_count[f] = 0;
    if (threadIdx.x == 0) s_work = 0;
    __syncthreads();
    // how much there is
    unsigned long long work = 0;
    TokenRun first = {-1, 0, 0, 0};            // of token threadIdx.x: looked up once
    for (int t = threadIdx.x; t < T; t += PL_THREADS) {
        const TokenRun r = pa_token(p.b, p.page_shift, t);
        if (t == (int)threadIdx.x) first = r;
        work += (unsigned)r.own;
        if (r.prefix >= 0) atomicAdd(&s_count[r.prefix], 1);
    }
    __syncthreads();
    auto prefix_keys = [&](int f) { return (int)min((long long)p.b.prefix_len[f], (long long)p.b.max_prefix_pages << p.page_shift); };
    // 65 rows and more in wide tiles: the prefix comes from L2 once for 128 rows instead of once for 32
    auto rows_of = [&](int f) { return s_count[f] * p.gq > 2 * PA_ROWS ? PA_WIDE : PA_ROWS; };
    auto tiles_of = [&](int f) { const int rows = s_count[f] * p.gq; return rows > 2 * PA_ROWS ? (rows + PA_WIDE - 1) / PA_WIDE : (rows + PA_ROWS - 1) / PA_ROWS; };
    for (int f = threadIdx.x; f < F; f += PL_THREADS)
        if (s_count[f]) work += (unsigned long long)prefix_keys(f) * tiles_of(f);
    for (int o = 32; o; o >>= 1) work += __shfl_xor(work, o);
    if ((threadIdx.x & 63) == 0 && work) atomicAdd(&s_work, work);
    __syncthreads();
    // keys of a range, a multiple of what the wavefronts take at a time
    // (lists have 2^30 keys at most: a range of nearly 2^31, or two thirds of it, holds any; and 32-bit divisions, of which a thread makes a handful in a chain:
    // with 64-bit ones the plan of one request took 5.7 us, that of 256 behind 8 prefixes 9.2)
    constexpr unsigned step = PA_WAVES * PA_KEYS;
    const unsigned long long all = s_work;
    const unsigned each = all >> 31 ? (unsigned)min(all / (unsigned)p.target, (1ULL << 31) - step) : ((unsigned)all + (unsigned)p.target - 1u) / (unsigned)p.target;
    const unsigned C = max((each + step - 1) / step, 1u) * step;
    auto range_of = [&](int keys, int cuts) { return (((unsigned)keys + cuts - 1) / (unsigned)cuts + step - 1) / step * step; };
    // At 64 elements a head three workgroups fit a unit, not two, and the longest ranges of the groups end last: two thirds of the length, in whole steps
    // upwards, so 256 keys stay 256.  Against the whole length, at 240 sizes (1 to 8 prefixes of 300 to 8000, 8 to 256 requests with up to 100 or 512 keys of
    // their own, 8 to 64 heads on 1 to 8): 0.80 to 1.08 of the time, 0.98 in the mean; most where own lists are long (256 requests behind 8 prefixes of
    // 1500, 32 heads on 4: 28.7 us for 33.1), least where they are short (the same with up to 100 keys: 25.7 for 24.8).  Downwards 256 became 128: 19.2 us
    // for 14.3 at 64 requests, 32 heads on 8.  At 128 elements it does not pay (128 requests behind one of 8191: 91 us a layer for 86).
    const unsigned G = p.head_dim == 64 ? (C / step * 2 + 2) / 3 * step : C;
    // a wide tile leaves as much behind as it reads in 130 keys: its ranges are 256 at least
    auto group_cuts_of = [&](int f) { const unsigned c = rows_of(f) == PA_WIDE ? max(G, 256u) : G; return (int)((prefix_keys(f) + c - 1) / c); };
    auto cuts_of = [&](int keys) { return keys > 0 ? (int)(((unsigned)keys + C - 1) / C) : 0; };
    // groups: their lists, slots and items
    int n_list = 0, n_slot = 0, n_item = 0;
    for (int f0 = 0; f0 < F; f0 += PL_THREADS) {
        const int f = f0 + threadIdx.x;
        const int members = f < F ? s_count[f] : 0, cuts = members ? group_cuts_of(f) : 0;
        int a, b, c;
        const int la = n_list + pl_scan(members, s_scan, &a);
        const int sl = n_slot + pl_scan(members * cuts, s_scan, &b);
        const int it = n_item + pl_scan(members ? tiles_of(f) * cuts : 0, s_scan, &c);
        if (f < F) { s_list[f] = la; s_slot[f] = sl; s_item[f] = it; }
        n_list += a; n_slot += b; n_item += c;
    }
    __syncthreads();
    const int group_items = n_item;
    for (int i = threadIdx.x; i < group_items && i < p.items_cap; i += PL_THREADS) {
        const int f = pl_find(s_item, F, i);
        const int keys = prefix_keys(f), cuts = group_cuts_of(f), tiles = tiles_of(f), at = i - s_item[f];
        const int cut = at / tiles, tile = at - cut * tiles;       // the tiles of a range lie side by side: they share its keys in L2
        const unsigned per = range_of(keys, cuts);
        int32_t *e = v.items + (size_t)i * PA_ITEM;
        const int rows = rows_of(f);
        e[0] = min(rows, s_count[f] * p.gq - tile * rows);
        e[1] = s_list[f]; e[2] = 1; e[3] = tile * rows; e[4] = f; e[5] = 1;
        e[6] = (int)min(cut * per, (unsigned)keys); e[7] = (int)min((cut + 1) * per, (unsigned)keys);
        e[8] = s_slot[f] + cut * s_count[f];
    }
    __syncthreads();
    // the members, and every token's own parts
    int *s_take = s_item;
    for (int f = threadIdx.x; f < F; f += PL_THREADS) s_take[f] = 0;
    __syncthreads();
    const int own_tiles = (p.gq + PA_ROWS - 1) / PA_ROWS;
    for (int t0 = 0; t0 < T; t0 += PL_THREADS) {
        const int t = t0 + threadIdx.x;
        TokenRun r = {-1, 0, 0, 0};
        int place = 0, prefix_cuts = 0;
        if (t < T) {
            r = t0 ? pa_token(p.b, p.page_shift, t) : first;
            if (r.prefix >= 0) {
                place = atomicAdd(&s_take[r.prefix], 1);
                if (s_list[r.prefix] + place < T) v.list[s_list[r.prefix] + place] = t;
                prefix_cuts = group_cuts_of(r.prefix);
            }
        }
        const int cuts = cuts_of(r.own), kept = cuts + prefix_cuts > 1 ? cuts : 0;
        int a, b;
        const int sl = n_slot + pl_scan(kept, s_scan, &a);
        const int it = n_item + pl_scan(cuts * own_tiles, s_scan, &b);
        s_first[threadIdx.x] = it; s_own[threadIdx.x] = r.own; s_row[threadIdx.x] = 2 * r.row + r.table; s_part[threadIdx.x] = kept ? sl : -1;
        if (t < T) {
            int32_t *j = v.join + (size_t)t * PA_JOIN;
            j[0] = sl; j[1] = cuts; j[3] = prefix_cuts;
            j[2] = r.prefix >= 0 ? s_slot[r.prefix] + place : 0;
            j[4] = r.prefix >= 0 ? s_count[r.prefix] : 0;
        }
        __syncthreads();
        for (int i = n_item + threadIdx.x; i < n_item + b && i < p.items_cap; i += PL_THREADS) {
            const int w = pl_find(s_first, PL_THREADS, i), keys = s_own[w], cuts_w = cuts_of(keys), at = i - s_first[w];
            const int cut = at / own_tiles, tile = at - cut * own_tiles;
            const unsigned per = range_of(keys, cuts_w);
            int32_t *e = v.items + (size_t)i * PA_ITEM;
            e[0] = min(PA_ROWS, p.gq - tile * PA_ROWS); e[1] = t0 + w; e[2] = 0; e[3] = tile * PA_ROWS; e[4] = s_row[w] >> 1; e[5] = s_row[w] & 1;
            e[6] = (int)min(cut * per, (unsigned)keys); e[7] = (int)min((cut + 1) * per, (unsigned)keys);
            e[8] = s_part[w] < 0 ? -1 : s_part[w] + cut;
        }
        n_slot += a; n_item += b;
    }
    if (threadIdx.x == 0) v.n_items[0] = (int)min((long long)n_item, p.items_cap);
}

// ------------------------------------------------------------------ attention
struct AttnKernelArgs {
    AttnArgs a;
    void *plan;
    float *parts;          // [slots][n_kv_heads][gq][D] sums, then [slots][n_kv_heads][gq][2] maximum and weight
    long long items_cap, slots_cap;
};

// K and V of one block of 32 keys, on their way.
template <int D> struct KeyBlock {
    uint4 k[2][D / 32], v[D / 16];
    int have;                  // bit h: the h-th sixteen of keys has a page
};

// What a wavefront holds of 16 query rows.
template <int D> struct RowState {
    uint4 q[D / 32];
    float m, l;                // of row lane % 16: the maximum score, unscaled, over all lanes; the sum of this lane's keys
    float4_t acc[D / 16];      // out^T: columns 16 i + 4 g .. + 3 of row lane % 16
};

// One wavefront's way through keys [first, last) of a list.  It holds 64 page ids at a time, one a lane.
template <int DT, int D>
struct Walk {
    static constexpr int KS = D / 32, DTILES = D / 16, VL = D / 16, CH = D / 8;    // K steps, column tiles, 16-byte loads of V a lane, chunks of a row
    const AttnArgs &p;
    const int32_t *pages;
    unsigned char *vlds;
    float scale2;
    int n_listed, first, last, head;
    int window, ids;                   // 64 pages from page `window` on; -1: none yet
    int seen;                          // 0 until there was a key

    // Pages of the sixteens of keys from key0 on, -1 for those that are absent; bit i of the result: the i-th has one.
    template <int N>
    __device__ __forceinline__ int find(int key0, int (&page)[N])
    {
        const int from = key0 >> p.page_shift, to = (key0 + 16 * (N - 1)) >> p.page_shift;
        if (window < 0 || from < window || to >= window + 64) {
            window = from;
            const int at = from + (threadIdx.x & 63);
            ids = at < n_listed ? pages[at] : -1;
            ids = ids < p.n_pages ? ids : -1;
            // waited for here: behind the branch every look at the ids would wait for whatever was loaded last
            asm volatile("" : "+v"(ids));
        }
        int have = 0;
#pragma unroll
        for (int i = 0; i < N; i++) {
            page[i] = __builtin_amdgcn_readlane(ids, ((key0 + 16 * i) >> p.page_shift) - window);
            have |= key0 + 16 * i < last && page[i] >= 0 ? 1 << i : 0;
        }
        seen |= have;
        return have;
    }

    __device__ __forceinline__ size_t row_of(int page, int key) const      // of a slab of [rows, D]
    {
        return (((size_t)page * p.n_kv_heads + head) << p.page_shift) + (key & ((1 << p.page_shift) - 1));
    }

    // Issue the loads of the block at key0 (keys past the last are loaded from page 0 and masked).  STREAM: keys that nobody else reads.
    template <bool STREAM>
    __device__ __forceinline__ void load(KeyBlock<D> &b, int key0)
    {
        auto get = [](const uint16_t *src) { return STREAM ? ldg16_stream(src) : ldg16(src); };
        // what differs between lanes is one 32-bit offset for K and one for V: the rest of an address is the same for the wavefront
        const int lane = threadIdx.x & 63;
        const unsigned klane = (lane & 15) * D + (lane >> 4) * 8, vlane = (lane / CH) * D + (lane % CH) * 8;
        int page[2];
        b.have = find<2>(key0, page);
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const size_t row0 = row_of(b.have >> h & 1 ? page[h] : 0, key0 + 16 * h);
            const uint16_t *k = p.k_pages + row0 * D, *v = p.v_pages + row0 * D;
#pragma unroll
            for (int s = 0; s < KS; s++) b.k[h][s] = get(k + klane + s * 32);
#pragma unroll
            for (int u = 0; u < VL / 2; u++) b.v[h * (VL / 2) + u] = get(v + vlane + u * (64 / CH) * D);
        }
    }

    // Scores of the block at key0, and V's way to LDS: after this the block's registers are free.
    template <int NR>
    __device__ __forceinline__ void scores(KeyBlock<D> &b, int key0, const RowState<D> (&st)[NR], float4_t (&s)[NR][2])
    {
        const int lane = threadIdx.x & 63, g = lane >> 4;
        const bool whole = b.have == 3 && key0 + PA_KEYS <= last;
        if (!whole) {
            // what lies behind the last key, or on no page at all, must not meet a weight of zero: it may be infinite
#pragma unroll
            for (int u = 0; u < VL; u++) {
                const uint32_t keep = key0 + u * (64 / CH) + lane / CH < last && (b.have >> (u >= VL / 2) & 1) ? ~0u : 0u;
                b.v[u] = make_uint4(b.v[u].x & keep, b.v[u].y & keep, b.v[u].z & keep, b.v[u].w & keep);
            }
        }
#pragma unroll
        for (int u = 0; u < VL; u++) {
            const int r = u * (64 / CH) + lane / CH;
            stg16(vlds + r * (D * 2) + pa_swizzle<D>(r, lane % CH) * 16, b.v[u]);
        }
#pragma unroll
        for (int n = 0; n < NR; n++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                s[n][h] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < KS; k++) s[n][h] = pa_mfma<DT>(b.k[h][k], st[n].q[k], s[n][h]);
                if (!whole) {
#pragma unroll
                    for (int i = 0; i < 4; i++) s[n][h][i] = (b.have >> h & 1) && key0 + 16 * h + 4 * g + i < last ? s[n][h][i] : -INFINITY;
                }
            }
    }

    // Softmax weights of the block, and the sums over its keys.
    template <int NR>
    __device__ __forceinline__ void sums(RowState<D> (&st)[NR], const float4_t (&s)[NR][2])
    {
        const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
        // fp16 has steps of 2^-24 below 2^-14, and a row's result may be made of many weights down there (8192 keys 16.2 below a few others: off by
        // 3 % where these others' values are zero), so its largest weight is 2^14 instead of 1.  bf16 has fp32's range.
        constexpr float TOP = DT == DT_F16 ? 14.f : 0.f;
        uint4 wf[NR];
#pragma unroll
        for (int n = 0; n < NR; n++) {
            float top = fmaxf(fmaxf(fmaxf(s[n][0][0], s[n][0][1]), fmaxf(s[n][0][2], s[n][0][3])), fmaxf(fmaxf(s[n][1][0], s[n][1][1]), fmaxf(s[n][1][2], s[n][1][3])));
            top = fmaxf(top, __shfl_xor(top, 16));
            top = fmaxf(top, __shfl_xor(top, 32));
            // A higher maximum in some row: what was summed so far shrinks.  Letting the sums stand until a maximum has grown by 2^8 takes 3 to
            // 5 % off the prefix items and nothing off the others, and costs the exact weight of 1 of a row's largest key (0.0022 of the
            // result's norm off the 64-bit result in bf16 instead of 0.0019).
            if (__ballot(top > st[n].m)) {
                const float m = fmaxf(st[n].m, top), keep = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((st[n].m - m) * scale2);
                st[n].l *= keep;
#pragma unroll
                for (int d = 0; d < DTILES; d++) st[n].acc[d] *= keep;
                st[n].m = m;
            }
            const float ref = st[n].m == -INFINITY ? 0.f : st[n].m;
            // The maximum comes off before the scaling, or the largest key's weight would be 2 to the power of a rounding of its scaled score:
            // nothing or infinity from 2^24 on.  The parts are joined so, too (128 requests behind one prefix of 8191, two layers: 175.7 us, scaled first 172.4).
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float x = s[n][i / 4][i % 4] - ref;
                w[i] = __builtin_amdgcn_exp2f(DT == DT_F16 ? fmaf(x, scale2, TOP) : x * scale2);
            }
            wf[n] = pack8<DT>(w);
            // A matrix instruction takes weights of 16 bits (a second product with what the rounding left would be half as many again); a weight's
            // rounding moves the result by a part of the result's own.  The sum takes the weights as rounded: a rounding that is in both sums moves
            // their quotient less, and four instructions do it.
            const uint32_t one = DT == DT_F16 ? 0x3c003c00u : 0x3f803f80u;
            st[n].l = dot8<DT>(wf[n], make_uint4(one, one, one, one), st[n].l);
        }
        __builtin_amdgcn_wave_barrier();
        auto column = [&](int d) {                 // V^T of 16 columns
            uint2 half[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int r = 16 * h + 4 * g + c / 4;
                half[h] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (pa_lds_short4 *)(vlds + r * (D * 2) + pa_swizzle<D>(r, 2 * d + (c % 4) / 2) * 16 + (c & 1) * 8)));
            }
            return make_uint4(half[0].x, half[0].y, half[1].x, half[1].y);
        };
        // two columns ahead and no more, or the registers run out
        constexpr int AHEAD = 2;
        uint4 vt[AHEAD];
#pragma unroll
        for (int d = 0; d < AHEAD; d++) vt[d] = column(d);
#pragma unroll
        for (int d = 0; d < DTILES; d++) {
            const uint4 now = vt[d % AHEAD];
            if (d + AHEAD < DTILES) vt[d % AHEAD] = column(d + AHEAD);
#pragma unroll
            for (int n = 0; n < NR; n++) st[n].acc[d] = pa_mfma<DT>(now, wf[n], st[n].acc[d]);
            __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_wave_barrier();
    }

    template <int NR, bool STREAM>
    __device__ __forceinline__ void all(RowState<D> (&st)[NR])
    {
        int key0 = first;
        if (key0 >= last) return;
        float4_t s[NR][2];
        KeyBlock<D> b;
        load<STREAM>(b, key0);
        // the next block comes during the softmax and the second product, into the same registers
#pragma unroll 1
        while (key0 + PA_KEYS < last) {
            scores<NR>(b, key0, st, s);
            key0 += PA_KEYS;
            load<STREAM>(b, key0);
            sums<NR>(st, s);
        }
        scores<NR>(b, key0, st, s);
        sums<NR>(st, s);
    }
};

// A part's maximum as it is handed on.  Where there were keys it is finite even if their scores are all minus infinity, so a row without a maximum
// has no key.  Such scores have no weight beside others; alone they leave a sum of zero, and the softmax is 0 / 0.
__device__ __forceinline__ float pa_top(float m, int seen) { return seen ? fmaxf(m, -3.402823466e38f) : m; }
__device__ __forceinline__ float pa_inverse(float m, float l) { return m == -INFINITY && l == 0.f ? 0.f : l == 0.f ? NAN : 1.f / l; }

constexpr int pa_pitch(int D) { return D + 4; }            // floats of a row in the LDS exchange: a float4 of 16 rows meets all banks

// Scale and q as the walk takes them: the scale in powers of two, positive (a maximum of scores is one of scaled scores then, and a masked
// score stays minus infinity), its sign in q; a scale of zero as zeros for q.
__device__ __forceinline__ float pa_scale2(float scale) { return scale == 0.f ? 1.f : fabsf(scale) * PA_LOG2E; }
__device__ __forceinline__ uint4 pa_load_q(const uint16_t *q, float scale)
{
    const uint32_t flip = scale < 0.f ? 0x80008000u : 0u, keep = scale == 0.f ? 0u : ~0u;
    const uint4 v = ldg16(q);
    return make_uint4((v.x ^ flip) & keep, (v.y ^ flip) & keep, (v.z ^ flip) & keep, (v.w ^ flip) & keep);
}

// One item for one key head: NR tiles of 16 query rows, the keys shared by the four wavefronts and joined in LDS.  Bound by HBM on
// long lists (two requests of 131071 keys, 8 heads of 128: 169 us for 1.07 GB, 6.3 TB/s; 61 of 1 to 2048, 32 heads: 5.8 TB/s) and on short
// ones by the chain page id -> keys -> softmax.
template <int DT, int D, int NR, bool STREAM>
__device__ __forceinline__ void pa_item(const AttnKernelArgs &ka, const_i32_ptr e, const PlanView &pv, int head, unsigned char *lds, float (*s_m)[16], float (*s_l)[16])
{
    constexpr int PITCH = pa_pitch(D), E = D / 16;
    const AttnArgs &p = ka.a;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int rows = e[0], from = e[1], grouped = e[2], row0 = e[3], slot = e[8];
    auto token_of = [&](int idx) { return grouped ? pv.list[from + idx] : from; };
    RowState<D> st[NR];
#pragma unroll
    for (int n = 0; n < NR; n++) {
        const int r = row0 + min(n * 16 + c, rows - 1), idx = r / p.gq;
        const uint16_t *q = p.q + token_of(idx) * p.q_stride + ((size_t)head * p.gq + (r - idx * p.gq)) * D;
#pragma unroll
        for (int k = 0; k < D / 32; k++) st[n].q[k] = pa_load_q(q + k * 32 + g * 8, p.scale);
        st[n].m = -INFINITY;
        st[n].l = 0.f;
#pragma unroll
        for (int d = 0; d < D / 16; d++) st[n].acc[d] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
    const int first = e[6], last = e[7], share = (last - first + PA_WAVES * PA_KEYS - 1) / (PA_WAVES * PA_KEYS) * PA_KEYS;
    const int mine = first + wave * share;
    const int listed = e[5] ? p.b.max_prefix_pages : p.b.max_pages;
    Walk<DT, D> walk{p, (e[5] ? p.b.prefix_tbl : p.b.page_tbl) + (size_t)e[4] * listed, lds + wave * (PA_KEYS * D * 2), pa_scale2(p.scale),
                     listed, mine, min(mine + share, last), head, -1, -1, 0};
    walk.template all<NR, STREAM>(st);
#pragma unroll
    for (int n = 0; n < NR; n++) {
        st[n].m = pa_top(st[n].m, walk.seen);
        float l = st[n].l;
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        __syncthreads();                       // the wavefronts are through with V, or with the exchange before this one
        if (g == 0) { s_m[wave][c] = st[n].m; s_l[wave][c] = l; }
        __syncthreads();
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < PA_WAVES; w++) m = fmaxf(m, s_m[w][c]);
        const float f = st[n].m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((st[n].m - m) * walk.scale2);
        float *part = reinterpret_cast<float *>(lds) + (wave * 16 + c) * PITCH;
#pragma unroll
        for (int d = 0; d < D / 16; d++) *reinterpret_cast<float4_t *>(part + d * 16 + g * 4) = st[n].acc[d] * f;
        __syncthreads();
        const int r = threadIdx.x >> 4, col = (threadIdx.x & 15) * E;
        if (n * 16 + r >= rows) continue;
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int w = 0; w < PA_WAVES; w++) m = fmaxf(m, s_m[w][r]);
#pragma unroll
        for (int w = 0; w < PA_WAVES; w++) l += s_l[w][r] * (s_m[w][r] == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((s_m[w][r] - m) * walk.scale2));
        float v[E];
#pragma unroll
        for (int k = 0; k < E; k += 4) {
            float4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int w = 0; w < PA_WAVES; w++) sum += *reinterpret_cast<const float4_t *>(reinterpret_cast<const float *>(lds) + (w * 16 + r) * PITCH + col + k);
#pragma unroll
            for (int i = 0; i < 4; i++) v[k + i] = sum[i];
        }
        const int row = row0 + n * 16 + r, idx = row / p.gq, sub = row - idx * p.gq;
        if (slot < 0) {
            const float inv = pa_inverse(m, l);
            uint16_t *out = p.out + token_of(idx) * p.out_stride + ((size_t)head * p.gq + sub) * D + col;
#pragma unroll
            for (int k = 0; k < E; k += 4) *reinterpret_cast<uint2 *>(out + k) = make_uint2(pack2<DT>(v[k] * inv, v[k + 1] * inv), pack2<DT>(v[k + 2] * inv, v[k + 3] * inv));
        } else if (slot + idx < ka.slots_cap) {
            const size_t at = ((size_t)(slot + idx) * p.n_kv_heads + head) * p.gq + sub;
#pragma unroll
            for (int k = 0; k < E; k += 4) *reinterpret_cast<float4_t *>(ka.parts + at * D + col + k) = float4_t{v[k], v[k + 1], v[k + 2], v[k + 3]};
            if (col == 0) *reinterpret_cast<float2 *>(ka.parts + (size_t)ka.slots_cap * p.n_q_heads * D + at * 2) = make_float2(m, l);
        }
    }
}

// LDS chunk of K at which chunk ch of key row r lies: an operand read takes one chunk of sixteen rows.
template <int D> __device__ __forceinline__ int pa_kswizzle(int r, int ch) { return D == 128 ? ch ^ (r & 15) : ch ^ ((r >> 1) & 7); }

constexpr int PA_TILE = 64;                                // keys in LDS at a time

// One wide item for one key head: 32 rows a wavefront, every key tile brought to LDS once for all of them, the next one on its way meanwhile.
// Bound by what a wavefront waits for, with two on a SIMD: scores, maximum, exponentials, second product and barrier follow each other (128 requests with
// one key of their own over a prefix of 8191, 32 heads on 8: 45.7 us; vector instructions take 44 % of the cycles, matrix instructions 19, and wavefronts
// wait 38 % of theirs).  With own keys (270 MB) 86 us a layer; 111 before there were such tiles, with rows of own keys not yet streamed past L2.
template <int DT, int D>
__device__ __forceinline__ void pa_wide(const AttnKernelArgs &ka, const_i32_ptr e, const PlanView &pv, int head, unsigned char *lds)
{
    constexpr int NR = 2, KS = D / 32, CH = D / 8, PER = PA_TILE * CH / (64 * PA_WAVES), BYTES = PA_TILE * D * 2;
    const AttnArgs &p = ka.a;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int rows = e[0], from = e[1], row0 = e[3], slot = e[8], last = e[7];
    RowState<D> st[NR];
#pragma unroll
    for (int n = 0; n < NR; n++) {
        const int r = row0 + min(wave * 32 + n * 16 + c, rows - 1), idx = r / p.gq;
        const uint16_t *q = p.q + pv.list[from + idx] * p.q_stride + ((size_t)head * p.gq + (r - idx * p.gq)) * D;
#pragma unroll
        for (int k = 0; k < KS; k++) st[n].q[k] = pa_load_q(q + k * 32 + g * 8, p.scale);
        st[n].m = -INFINITY;
        st[n].l = 0.f;
#pragma unroll
        for (int d = 0; d < D / 16; d++) st[n].acc[d] = float4_t{0.f, 0.f, 0.f, 0.f};
    }
    const int listed = p.b.max_prefix_pages;
    Walk<DT, D> walk{p, p.b.prefix_tbl + (size_t)e[4] * listed, nullptr, pa_scale2(p.scale), listed, e[6], last, head, -1, -1, 0};
    uint4 kr[PER], vr[PER];
    const unsigned mine = (lane / CH) * D + (lane % CH) * 8;
    int have, have_next;                                   // sixteens of the tile at hand, and of the one on its way, that have a page
    auto load = [&](int key0) {                            // this thread's chunks: 64 / CH rows of a load, all in one sixteen
        int page[4];
        have_next = walk.template find<4>(key0, page);
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int r0 = (i * PA_WAVES + wave) * (64 / CH), six = r0 / 16;
            const int pg = six == 0 ? page[0] : six == 1 ? page[1] : six == 2 ? page[2] : page[3];
            const size_t row = walk.row_of(have_next >> six & 1 ? pg : 0, key0 + six * 16) + (r0 & 15);
            kr[i] = ldg16(p.k_pages + row * D + mine);
            vr[i] = ldg16(p.v_pages + row * D + mine);
        }
    };
    auto store = [&](unsigned char *buf, int key0) {
        have = have_next;
        const bool whole = have == 15 && key0 + PA_TILE <= last;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            const int r0 = (i * PA_WAVES + wave) * (64 / CH), r = r0 + lane / CH, ch = lane % CH;
            if (!whole) {                                  // absent keys must not meet a weight of zero: they may be infinite
                const uint32_t keep = (have >> (r0 / 16) & 1) && key0 + r < last ? ~0u : 0u;
                vr[i] = make_uint4(vr[i].x & keep, vr[i].y & keep, vr[i].z & keep, vr[i].w & keep);
            }
            stg16(buf + r * (D * 2) + pa_kswizzle<D>(r, ch) * 16, kr[i]);
            stg16(buf + BYTES + r * (D * 2) + pa_swizzle<D>(r, ch) * 16, vr[i]);
        }
    };
    int key0 = e[6];
    load(key0);
    store(lds, key0);
    __syncthreads();
#pragma unroll 1
    for (int buf = 0; key0 < last; key0 += PA_TILE, buf ^= 1) {
        const bool more = key0 + PA_TILE < last;
        if (more) load(key0 + PA_TILE);
        unsigned char *tile = lds + buf * 2 * BYTES;
        if (wave * 32 < rows) {
#pragma unroll
            for (int half = 0; half < 2; half++) {
                const int k0 = key0 + half * 32;
                if (k0 >= last) break;
                float4_t s[NR][2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    uint4 kf[KS];
                    const int r = half * 32 + h * 16 + c;
#pragma unroll
                    for (int k = 0; k < KS; k++) kf[k] = *reinterpret_cast<const uint4 *>(tile + r * (D * 2) + pa_kswizzle<D>(r, k * 4 + g) * 16);
#pragma unroll
                    for (int n = 0; n < NR; n++) {
                        s[n][h] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int k = 0; k < KS; k++) s[n][h] = pa_mfma<DT>(kf[k], st[n].q[k], s[n][h]);
                    }
                }
                if ((have >> 2 * half & 3) != 3 || k0 + 32 > last) {
#pragma unroll
                    for (int n = 0; n < NR; n++)
#pragma unroll
                        for (int h = 0; h < 2; h++)
#pragma unroll
                            for (int i = 0; i < 4; i++) s[n][h][i] = (have >> (2 * half + h) & 1) && k0 + 16 * h + 4 * g + i < last ? s[n][h][i] : -INFINITY;
                }
                walk.vlds = tile + BYTES + half * 32 * (D * 2);
                walk.template sums<NR>(st, s);
            }
        }
        if (more) store(lds + (buf ^ 1) * 2 * BYTES, key0 + PA_TILE);
        __syncthreads();
    }
#pragma unroll
    for (int n = 0; n < NR; n++) {
        float l = st[n].l;
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        const int r = wave * 32 + n * 16 + c;
        if (r >= rows) continue;
        const int row = row0 + r, idx = row / p.gq, sub = row - idx * p.gq;
        if (slot < 0 || slot + idx >= ka.slots_cap) continue;      // a group's rows always have a slot
        const size_t at = ((size_t)(slot + idx) * p.n_kv_heads + head) * p.gq + sub;
#pragma unroll
        for (int d = 0; d < D / 16; d++) *reinterpret_cast<float4_t *>(ka.parts + at * D + d * 16 + g * 4) = st[n].acc[d];
        if (g == 0) *reinterpret_cast<float2 *>(ka.parts + (size_t)ka.slots_cap * p.n_q_heads * D + at * 2) = make_float2(pa_top(st[n].m, walk.seen), l);
    }
}

template <int DT, int D>
__global__ __launch_bounds__(64 * PA_WAVES, 2) void prefix_attention_kernel(const AttnKernelArgs ka)
{
    __shared__ __attribute__((aligned(16))) unsigned char lds[2 * 2 * PA_TILE * D * 2];
    static_assert(PA_WAVES * 16 * pa_pitch(D) * 4 <= 2 * 2 * PA_TILE * D * 2, "the wavefronts' V blocks, and the exchange of their sums, fit too");
    __shared__ float s_m[PA_WAVES][16], s_l[PA_WAVES][16];
    const AttnArgs &p = ka.a;
    const PlanView pv = pa_plan_view(ka.plan, p.b.T);
    // key heads fastest: with a multiple of eight of them a head stays on one XCD, and with it what the row tiles of a prefix share
    const unsigned item = blockIdx.x / (unsigned)p.n_kv_heads, head = blockIdx.x - item * (unsigned)p.n_kv_heads;
    if ((int)item >= min((long long)as_const(pv.n_items)[0], ka.items_cap)) return;
    // the plan is read as constant memory: what an item says is the same for the workgroup, and belongs in scalar registers
    const const_i32_ptr e = as_const(pv.items + (size_t)item * PA_ITEM);
    if (e[0] > PA_ROWS) pa_wide<DT, D>(ka, e, pv, head, lds);
    else if (e[0] > 16) pa_item<DT, D, 2, false>(ka, e, pv, head, lds, s_m, s_l);
    else if (e[2]) pa_item<DT, D, 1, false>(ka, e, pv, head, lds, s_m, s_l);
    else pa_item<DT, D, 1, true>(ka, e, pv, head, lds, s_m, s_l);
}

// ------------------------------------------------------------------ join
// 4 to 6 us, launch and latency.  A workgroup: 16 / G query rows of one token, 16 threads and G groups of them a row, the groups share the parts.
template <int DT, int D, int G>
__global__ __launch_bounds__(256) void pa_join_kernel(const AttnKernelArgs ka)
{
    constexpr int ROWS = 16 / G, E = D / 16;
    __shared__ float s_v[G > 1 ? 16 : 1][G > 1 ? D : 1], s_m[16], s_l[16];
    const AttnArgs &p = ka.a;
    const int t = blockIdx.x;
    if (p.b.tok_req[t] < 0) return;
    const PlanView pv = pa_plan_view(ka.plan, p.b.T);
    const const_i32_ptr j = as_const(pv.join + (size_t)t * PA_JOIN);
    const int own = j[1], shared = j[3];
    if (own == 1 && shared == 0) return;                         // written by its only item
    const int slice = threadIdx.x >> 4, col = (threadIdx.x & 15) * E, part0 = slice % G;
    const int row = blockIdx.y * ROWS + slice / G;               // query head
    const float scale2 = pa_scale2(p.scale);
    float m = -INFINITY, l = 0.f, v[E] = {};
    if (row < p.n_q_heads) {
        const float *ml = ka.parts + (size_t)ka.slots_cap * p.n_q_heads * D;
        for (int i = part0; i < own + shared; i += G) {
            const long long slot = i < own ? (long long)j[0] + i : j[2] + (long long)(i - own) * j[4];
            if (slot < 0 || slot >= ka.slots_cap) continue;
            const size_t at = (size_t)slot * p.n_q_heads + row;
            const float2 x = *reinterpret_cast<const float2 *>(ml + at * 2);
            if (x.x == -INFINITY && x.y == 0.f) continue;       // no keys; scores that are all NaN leave no maximum, but a sum that is NaN
            const float top = fmaxf(m, x.x), a = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((m - top) * scale2), b = __builtin_amdgcn_exp2f((x.x - top) * scale2);
            m = top;
            l = l * a + x.y * b;
#pragma unroll
            for (int k = 0; k < E; k += 4) {
                const float4_t y = *reinterpret_cast<const float4_t *>(ka.parts + at * D + col + k);
#pragma unroll
                for (int q = 0; q < 4; q++) v[k + q] = v[k + q] * a + y[q] * b;
            }
        }
    }
    if constexpr (G > 1) {
        if (col == 0) { s_m[slice] = m; s_l[slice] = l; }
#pragma unroll
        for (int k = 0; k < E; k++) s_v[slice][col + k] = v[k];
        __syncthreads();
        if (part0) return;
        float top = m;
        for (int q = 1; q < G; q++) top = fmaxf(top, s_m[slice + q]);
        float all = 0.f;
#pragma unroll
        for (int k = 0; k < E; k++) v[k] = 0.f;
        for (int q = 0; q < G; q++) {
            const float f = s_m[slice + q] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f((s_m[slice + q] - top) * scale2);
            all += s_l[slice + q] * f;
#pragma unroll
            for (int k = 0; k < E; k++) v[k] += s_v[slice + q][col + k] * f;
        }
        l = all;
        m = top;
    }
    if (row >= p.n_q_heads) return;
    const float inv = pa_inverse(m, l);
    uint16_t *out = p.out + t * p.out_stride + (size_t)row * D + col;
#pragma unroll
    for (int k = 0; k < E; k += 4) *reinterpret_cast<uint2 *>(out + k) = make_uint2(pack2<DT>(v[k] * inv, v[k + 1] * inv), pack2<DT>(v[k + 2] * inv, v[k + 3] * inv));
}

// ------------------------------------------------------------------ launchers
int64_t attn_plan_bytes(int T, int n_prefix, int n_q_heads, int n_kv_heads)
{
    const int64_t list = (T + 3) / 4 * 4, items = pa_items_cap(T, n_prefix, n_q_heads / n_kv_heads, n_kv_heads);
    return 4 * (4 + list + (int64_t)T * PA_JOIN + items * PA_ITEM);
}

int64_t attn_workspace_bytes(int T, int n_prefix, int n_q_heads, int n_kv_heads, int head_dim)
{
    return pa_slots_cap(T, n_prefix, n_q_heads / n_kv_heads, n_kv_heads) * n_q_heads * (head_dim + 2) * 4;
}

int launch_attn_plan(const KvBatch &b, int page_shift, int n_q_heads, int n_kv_heads, int head_dim, void *plan, hipStream_t s)
{
    PlanArgs a;
    a.b = b; a.plan = plan; a.page_shift = page_shift; a.head_dim = head_dim; a.gq = n_q_heads / n_kv_heads; a.target = pa_target(n_kv_heads);
    a.items_cap = pa_items_cap(b.T, b.n_prefix, a.gq, n_kv_heads);
    hipLaunchKernelGGL(pa_plan_kernel, dim3(1), dim3(PL_THREADS), 0, s, a);
    return (int)hipGetLastError();
}

template <int DT, int D>
static void attention_of(const AttnKernelArgs &a, hipStream_t s)
{
    hipLaunchKernelGGL((prefix_attention_kernel<DT, D>), dim3((unsigned)(a.items_cap * a.a.n_kv_heads)), dim3(64 * PA_WAVES), 0, s, a);
    // few rows have many parts each: then sixteen slices of a workgroup share a row's
    const dim3 wide((unsigned)a.a.b.T, (unsigned)a.a.n_q_heads), narrow((unsigned)a.a.b.T, (unsigned)((a.a.n_q_heads + 3) / 4));
    if ((long long)a.a.b.T * a.a.n_q_heads <= 1024) hipLaunchKernelGGL((pa_join_kernel<DT, D, 16>), wide, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((pa_join_kernel<DT, D, 4>), narrow, dim3(256), 0, s, a);
}

int launch_prefix_attention(const AttnArgs &a, int dtype, const void *plan, void *workspace, hipStream_t s)
{
    AttnKernelArgs k;
    k.a = a;
    k.plan = const_cast<void *>(plan);
    k.parts = static_cast<float *>(workspace);
    k.items_cap = pa_items_cap(a.b.T, a.b.n_prefix, a.gq, a.n_kv_heads);
    k.slots_cap = pa_slots_cap(a.b.T, a.b.n_prefix, a.gq, a.n_kv_heads);
    if (dtype == DT_F16) { if (a.head_dim == 64) attention_of<DT_F16, 64>(k, s); else attention_of<DT_F16, 128>(k, s); }
    else { if (a.head_dim == 64) attention_of<DT_BF16, 64>(k, s); else attention_of<DT_BF16, 128>(k, s); }
    return (int)hipGetLastError();
}

}  // namespace mlora

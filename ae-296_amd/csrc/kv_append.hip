// Rotation of q and k by their positions and the append of k and v to the paged cache, in one launch.
//   pairs (u, w) of a head's first `rot` elements -> (u cos a - w sin a, u sin a + w cos a); the rest unchanged; in fp32, rounded once.
// Replaces, for one layer, rotary_emb_fwd on q and k and destindex_copy_kv on k and v (lightllm/models/llama/triton_kernel/
// rotary_emb.py:8, lightllm/common/basemodel/triton_kernel/destindex_copy_kv.py:8), which read and write k twice.
//
// A thread owns one pair of 16-byte chunks of a head - the two halves of eight rotation pairs - in several heads of one token, so it
// reads its eight cosines and sines once; a workgroup covers 256 / (head_dim / 16) heads at a time.  Bound by HBM for prompts (8191 tokens of
// 64 + 2 x 8 heads of 128, half of a head turning: 65 us for 336 MB, 5.2 TB/s read + written, a copy's rate) and by the launch and the
// chain tables -> page -> rows for decode batches (7 tokens of 3 x 32 heads: 3.7 us).
#include "mlora_dev.hpp"
#include "mlora_step.hpp"

namespace mlora {

struct KvSlot { bool ok; int pos; long long page; int row; };

// Where token t's key goes.  `bad`: it names a request, but no table holds its place.
__device__ __forceinline__ KvSlot kv_slot(const KvAppendArgs &p, int t, bool &bad)
{
    KvSlot s = {false, 0, 0, 0};
    bad = false;
    const int req = p.b.tok_req[t], pos = p.b.tok_pos[t];
    if (req < 0) return s;
    bad = true;
    if (req >= p.b.n_req || pos < 0 || (p.rot && pos >= p.n_pos)) return s;
    int base = 0;
    if (p.b.req_prefix) {
        const int f = p.b.req_prefix[req];
        if (f >= 0 && f < p.b.n_prefix) base = p.b.prefix_len[f];
    }
    if (base < 0 || pos < base) return s;
    const int nth = (pos - base) >> p.page_shift;
    if (nth >= p.b.max_pages) return s;
    const int page = p.b.page_tbl[(size_t)req * p.b.max_pages + nth];
    if (page < 0 || page >= p.n_pages) return s;
    bad = false;
    return {true, pos, page, (pos - base) & ((1 << p.page_shift) - 1)};
}

template <int DT, int D, bool INTER>
__global__ __launch_bounds__(256) void kv_append_kernel(const KvAppendArgs p)
{
    constexpr int JOBS = D / 16, ROWS = 256 / JOBS;        // chunk pairs of a head, heads a workgroup covers at a time
    const int t = blockIdx.x;
    bool bad;
    const KvSlot s = kv_slot(p, t, bad);
    if (bad && p.bad && blockIdx.y == 0 && threadIdx.x == 0) atomicAdd(p.bad, 1);
    if (!s.ok) return;
    const int j = threadIdx.x % JOBS, turned = p.rot / 16;
    const bool turn = j < turned;
    const int ca = INTER || !turn ? 2 * j : j, cb = INTER || !turn ? 2 * j + 1 : j + turned;
    float c[8], sn[8];
    if (turn) {
        const float *tab = p.cos_sin + (size_t)s.pos * p.rot + j * 8;
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const float4_t a = *reinterpret_cast<const float4_t *>(tab + 4 * h), b = *reinterpret_cast<const float4_t *>(tab + p.rot / 2 + 4 * h);
#pragma unroll
            for (int e = 0; e < 4; e++) { c[4 * h + e] = a[e]; sn[4 * h + e] = b[e]; }
        }
    }
    const int rows = p.n_q_heads + 2 * p.n_kv_heads;
    for (int r = blockIdx.y * ROWS + threadIdx.x / JOBS; r < rows; r += gridDim.y * ROWS) {
        const uint16_t *src;
        uint16_t *dst;
        bool rotate = turn;
        if (r < p.n_q_heads) {
            src = p.q + t * p.q_stride + r * D;
            dst = p.q_out + t * p.q_out_stride + r * D;
        } else {
            const bool val = r >= p.n_q_heads + p.n_kv_heads;
            const int h = r - p.n_q_heads - (val ? p.n_kv_heads : 0);
            src = val ? p.v + t * p.v_stride + h * D : p.k + t * p.k_stride + h * D;
            dst = (val ? p.v_pages : p.k_pages) + ((((size_t)s.page * p.n_kv_heads + h) << p.page_shift) + s.row) * D;
            rotate = turn && !val;
        }
        uint4 a = ldg16(src + ca * 8), b = ldg16(src + cb * 8);
        if (rotate) {
            float u[8], w[8], fu[8], fw[8];
            unpack8<DT>(a, u);
            unpack8<DT>(b, w);
            if constexpr (INTER) {
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    fu[2 * e] = u[2 * e] * c[e] - u[2 * e + 1] * sn[e];
                    fu[2 * e + 1] = u[2 * e] * sn[e] + u[2 * e + 1] * c[e];
                    fw[2 * e] = w[2 * e] * c[4 + e] - w[2 * e + 1] * sn[4 + e];
                    fw[2 * e + 1] = w[2 * e] * sn[4 + e] + w[2 * e + 1] * c[4 + e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; e++) { fu[e] = u[e] * c[e] - w[e] * sn[e]; fw[e] = u[e] * sn[e] + w[e] * c[e]; }
            }
            a = pack8<DT>(fu);
            b = pack8<DT>(fw);
        }
        stg16(dst + ca * 8, a);
        stg16(dst + cb * 8, b);
    }
}

template <int DT, int D>
static void append_of(const KvAppendArgs &a, dim3 grid, hipStream_t s)
{
    if (a.interleaved) hipLaunchKernelGGL((kv_append_kernel<DT, D, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((kv_append_kernel<DT, D, false>), grid, dim3(256), 0, s, a);
}

// A launch has fewer than 2^32 threads: this many tokens each.
constexpr int KV_LAUNCH_TOKENS = 1 << 23;

int launch_kv_append(const KvAppendArgs &all, int dtype, hipStream_t s)
{
    const int rows = all.n_q_heads + 2 * all.n_kv_heads, per = 256 / (all.head_dim / 16), cover = (rows + per - 1) / per;
    for (int t0 = 0; t0 < all.b.T; t0 += KV_LAUNCH_TOKENS) {
        KvAppendArgs a = all;
        a.b.T = all.b.T - t0 < KV_LAUNCH_TOKENS ? all.b.T - t0 : KV_LAUNCH_TOKENS;
        a.b.tok_req += t0;
        a.b.tok_pos += t0;
        a.k += t0 * a.k_stride;
        a.v += t0 * a.v_stride;
        if (a.q) { a.q += t0 * a.q_stride; a.q_out += t0 * a.q_out_stride; }
        // a token's heads are shared by several workgroups while that adds workgroups the device has room for
        int parts = (4 * device_compute_units() + a.b.T - 1) / a.b.T;
        if (parts > cover) parts = cover;
        const dim3 grid((unsigned)a.b.T, (unsigned)parts);
        if (dtype == DT_F16) { if (a.head_dim == 64) append_of<DT_F16, 64>(a, grid, s); else append_of<DT_F16, 128>(a, grid, s); }
        else { if (a.head_dim == 64) append_of<DT_BF16, 64>(a, grid, s); else append_of<DT_BF16, 128>(a, grid, s); }
        const int rc = (int)hipGetLastError();
        if (rc) return rc;
    }
    return 0;
}

}  // namespace mlora

// Attention of a batch's tokens over the paged key/value cache:
//     out[t][h] = sum_j softmax_j(scale * q[t][h] . k_j) v_j,   j over positions 0 .. tok_pos[t] of t's request
// with the keys of a shared prefix on the prefix's pages and the others on the request's own.
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
constexpr int PA_KEYS = 32;                    // keys of a block
constexpr float PA_LOG2E = 1.44269504088896341f;

// LDS chunk (16 bytes) at which chunk c of key row r of a wavefront's V block lies: the 16 rows a transposing read touches
// at one column spread over all banks.
template <int D> __device__ __forceinline__ int pa_swizzle(int r, int c) { return D == 128 ? c ^ ((r & 7) << 1) : c ^ (((r >> 1) & 3) << 1); }

// A run of keys on pages of one list.
struct KeyRun {
    const int32_t *pages;      // the list's row of its table
    int n_listed;              // entries of it
    int first, last;           // keys [first, last), first a multiple of 16
};

// What a wavefront holds of 16 query rows.
template <int D> struct RowState {
    uint4 q[D / 32];
    float m, l;                // of row lane % 16: the maximum, in powers of two, over all lanes; the sum of this lane's keys
    float4_t acc[D / 16];      // out^T: columns 16 i + 4 g .. + 3 of row lane % 16
};

template <int DT, int D>
__device__ __forceinline__ void pa_blocks(const AttnArgs &p, int head, const KeyRun &run, int b0, int stride, float scale2, RowState<D> &st,
                                          unsigned char *vlds)
{
    constexpr int KS = D / 32, DTILES = D / 16, VL = D / 16, CH = D / 8;       // K steps, column tiles, 16-byte loads of V a lane, chunks of a row
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int psize = 1 << p.page_shift;
    const size_t page_elems = (size_t)p.n_kv_heads << p.page_shift;            // rows of a page
    for (int key0 = run.first + b0 * PA_KEYS; key0 < run.last; key0 += stride * PA_KEYS) {
        size_t row0[2];
        bool there[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const int at = key0 + 16 * h, nth = at >> p.page_shift;
            const int page = at < run.last && nth < run.n_listed ? run.pages[nth] : -1;
            there[h] = page >= 0 && page < p.n_pages;
            row0[h] = (there[h] ? page : 0) * page_elems + ((size_t)head << p.page_shift) + (at & (psize - 1));
        }
        uint4 kf[2][KS], vf[VL];
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int s = 0; s < KS; s++) kf[h][s] = ldg16(p.k_pages + (row0[h] + c) * D + s * 32 + g * 8);
#pragma unroll
        for (int u = 0; u < VL; u++) {
            const int r = u * (64 / CH) + lane / CH;
            vf[u] = ldg16(p.v_pages + (row0[u >= VL / 2] + (r & 15)) * D + (lane % CH) * 8);
            // what lies behind the last key, or on no page at all, must not meet a weight of zero: it may be infinite
            if (key0 + r >= run.last || !there[u >= VL / 2]) vf[u] = zero16();
        }
        float4_t s[2];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            s[h] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < KS; k++) s[h] = pa_mfma<DT>(kf[h][k], st.q[k], s[h]);
        }
        float top = -INFINITY;
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[h][i] = there[h] && key0 + 16 * h + 4 * g + i < run.last ? s[h][i] * scale2 : -INFINITY;
                top = fmaxf(top, s[h][i]);
            }
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float m = fmaxf(st.m, top), ref = m == -INFINITY ? 0.f : m, keep = __builtin_amdgcn_exp2f(st.m - ref);
        st.m = m;
        st.l *= keep;
#pragma unroll
        for (int d = 0; d < DTILES; d++) st.acc[d] *= keep;
        float w[8];
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int i = 0; i < 4; i++) { w[4 * h + i] = __builtin_amdgcn_exp2f(s[h][i] - ref); st.l += w[4 * h + i]; }
        const uint4 wf = pack8<DT>(w);
#pragma unroll
        for (int u = 0; u < VL; u++) {
            const int r = u * (64 / CH) + lane / CH;
            stg16(vlds + r * (D * 2) + pa_swizzle<D>(r, lane % CH) * 16, vf[u]);
        }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int d = 0; d < DTILES; d++) {
            uint2 half[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int r = 16 * h + 4 * g + c / 4;
                half[h] = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (pa_lds_short4 *)(vlds + r * (D * 2) + pa_swizzle<D>(r, 2 * d + (c % 4) / 2) * 16 + (c & 1) * 8)));
            }
            st.acc[d] = pa_mfma<DT>(make_uint4(half[0].x, half[0].y, half[1].x, half[1].y), wf, st.acc[d]);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// One workgroup: up to 16 query heads of one token that read one key head; its wavefronts share the keys.
template <int DT, int D>
__global__ __launch_bounds__(64 * PA_WAVES) void prefix_attention_kernel(const AttnArgs p)
{
    constexpr int PITCH = D + 4;
    __shared__ __attribute__((aligned(16))) unsigned char lds[PA_WAVES * 16 * PITCH * 4];
    __shared__ float s_m[PA_WAVES][16], s_l[PA_WAVES][16];
    const int t = blockIdx.x, head = blockIdx.y, first_row = blockIdx.z * 16;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int req = p.b.tok_req[t], pos = p.b.tok_pos[t];
    if (req < 0) return;
    int f = -1, base = 0;
    if (p.b.req_prefix && req < p.b.n_req) {
        f = p.b.req_prefix[req];
        if (f < 0 || f >= p.b.n_prefix) f = -1;
        else base = max(p.b.prefix_len[f], 0);
    }
    const int rows = min(16, p.gq - first_row);
    RowState<D> st;
    const uint16_t *q = p.q + t * p.q_stride + ((size_t)head * p.gq + first_row + (c < rows ? c : 0)) * D;
#pragma unroll
    for (int k = 0; k < D / 32; k++) st.q[k] = ldg16(q + k * 32 + g * 8);
    st.m = -INFINITY;
    st.l = 0.f;
#pragma unroll
    for (int d = 0; d < D / 16; d++) st.acc[d] = float4_t{0.f, 0.f, 0.f, 0.f};
    const float scale2 = p.scale * PA_LOG2E;
    unsigned char *vlds = lds + wave * (PA_KEYS * D * 2);
    if (f >= 0) {
        const long long last = min(min((long long)base, (long long)pos + 1), (long long)p.b.max_prefix_pages << p.page_shift);
        const KeyRun run = {p.b.prefix_tbl + (size_t)f * p.b.max_prefix_pages, p.b.max_prefix_pages, 0, (int)last};
        pa_blocks<DT, D>(p, head, run, wave, PA_WAVES, scale2, st, vlds);
    }
    if (req < p.b.n_req) {
        const long long last = min((long long)pos + 1 - base, (long long)p.b.max_pages << p.page_shift);
        const KeyRun run = {p.b.page_tbl + (size_t)req * p.b.max_pages, p.b.max_pages, 0, (int)last};
        pa_blocks<DT, D>(p, head, run, wave, PA_WAVES, scale2, st, vlds);
    }
    float l = st.l;
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) { s_m[wave][c] = st.m; s_l[wave][c] = l; }
    __syncthreads();
    float m = -INFINITY;
    for (int w = 0; w < PA_WAVES; w++) m = fmaxf(m, s_m[w][c]);
    const float mine = st.m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(st.m - m);
    float *part = reinterpret_cast<float *>(lds) + wave * 16 * PITCH + c * PITCH;
#pragma unroll
    for (int d = 0; d < D / 16; d++) *reinterpret_cast<float4_t *>(part + d * 16 + g * 4) = st.acc[d] * mine;
    __syncthreads();
    const int r = threadIdx.x >> 4;
    if (r >= rows) return;
    m = -INFINITY;
    for (int w = 0; w < PA_WAVES; w++) m = fmaxf(m, s_m[w][r]);
    l = 0.f;
    for (int w = 0; w < PA_WAVES; w++) l += s_m[w][r] == -INFINITY ? 0.f : s_l[w][r] * __builtin_amdgcn_exp2f(s_m[w][r] - m);
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint16_t *out = p.out + t * p.out_stride + ((size_t)head * p.gq + first_row + r) * D;
    for (int d = (threadIdx.x & 15) * 2; d < D; d += 32) {
        float v[2] = {0.f, 0.f};
        for (int w = 0; w < PA_WAVES; w++)
            for (int e = 0; e < 2; e++) v[e] += reinterpret_cast<const float *>(lds)[(w * 16 + r) * PITCH + d + e];
        *reinterpret_cast<uint32_t *>(out + d) = pack2<DT>(v[0] * inv, v[1] * inv);
    }
}

int launch_prefix_attention(const AttnArgs &a, int dtype, hipStream_t s)
{
    const dim3 grid((unsigned)a.b.T, (unsigned)a.n_kv_heads, (unsigned)((a.gq + 15) / 16));
    if (dtype == DT_F16) {
        if (a.head_dim == 64) hipLaunchKernelGGL((prefix_attention_kernel<DT_F16, 64>), grid, dim3(64 * PA_WAVES), 0, s, a);
        else hipLaunchKernelGGL((prefix_attention_kernel<DT_F16, 128>), grid, dim3(64 * PA_WAVES), 0, s, a);
    } else {
        if (a.head_dim == 64) hipLaunchKernelGGL((prefix_attention_kernel<DT_BF16, 64>), grid, dim3(64 * PA_WAVES), 0, s, a);
        else hipLaunchKernelGGL((prefix_attention_kernel<DT_BF16, 128>), grid, dim3(64 * PA_WAVES), 0, s, a);
    }
    return (int)hipGetLastError();
}

}  // namespace mlora

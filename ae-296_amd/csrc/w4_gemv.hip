// Base projections on 4-bit weights for the tokens of a decode batch:
//     y[t][n] = (accumulate ? y[t][n] : 0) + sum_g s[g][n] * sum_{k in g} (c[k][n] - z[g][n]) * x[t][k]
//
// A code becomes a 16-bit float without a conversion: shifted to the place of the top mantissa bits and joined with the pattern of
// 16.0 it reads 16 + c, exactly, in fp16 and in bf16 alike (two instructions for two codes).  The 16 and the zero point come off after the
// products: with X = sum of x over the group, sum (c - z) x = sum (16 + c) x - (16 + z) X.  X is one more MFMA per K step whose weight operand is
// ones, so it lands in the lanes that need it; products are exact in fp32 and the difference costs about two bits of its 24.
#include "mlora_dev.hpp"
#include "mlora_step.hpp"

namespace mlora {

// ------------------------------------------------------------------ packing
__global__ __launch_bounds__(256) void w4_pack_codes_kernel(const W4PackArgs p)
{
    const long long word = (long long)blockIdx.x * 256 + threadIdx.x;      // dword of the codes plane
    const long long words = (long long)p.sh.n_tiles * p.sh.k_tiles * (W4_TILE_BYTES / 4);
    if (word >= words) return;
    const long long tile = word >> 8;
    const int lane = (int)(word >> 2) & 63, step = (int)word & 3;
    const int n = (int)(tile / p.sh.k_tiles) * W4_TN + (lane & 15);
    const int k0 = (int)(tile % p.sh.k_tiles) * W4_TK + step * 32 + (lane >> 4) * 8;
    uint32_t v = 0;
    for (int j = 0; j < 8; j++) {
        const int k = k0 + j;
        const uint32_t c = k < p.sh.hin && n < p.sh.hout ? p.codes[(size_t)k * p.sh.hout + n] & 15u : 0u;
        v |= c << (4 * (j >> 1) + 16 * (j & 1));
    }
    reinterpret_cast<uint32_t *>(p.packed)[word] = v;
}

__global__ __launch_bounds__(256) void w4_pack_groups_kernel(const W4PackArgs p)
{
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= (long long)p.sh.n_tiles * p.sh.k_tiles * p.sh.per_tile * W4_TN) return;
    const long long tile = i / (p.sh.per_tile * W4_TN);
    const int n = (int)(tile / p.sh.k_tiles) * W4_TN + (int)(i & 15);
    const int g = (int)(tile % p.sh.k_tiles) * p.sh.per_tile + (int)((i >> 4) & (p.sh.per_tile - 1));
    const bool in = n < p.sh.hout && g < p.sh.groups;
    const size_t at = (size_t)g * p.sh.hout + n;
    const uint32_t scale = in ? p.scales[at] : 0u;
    unsigned char *plane = p.packed + p.sh.groups_at;
    if (p.zeros) reinterpret_cast<uint32_t *>(plane)[i] = scale | (16u + (in ? p.zeros[at] & 15u : 0u)) << 16;
    else reinterpret_cast<uint16_t *>(plane)[i] = (uint16_t)scale;
}

int launch_w4_pack(const W4PackArgs &a, hipStream_t s)
{
    const long long tiles = (long long)a.sh.n_tiles * a.sh.k_tiles, words = tiles * (W4_TILE_BYTES / 4), pairs = tiles * a.sh.per_tile * W4_TN;
    hipLaunchKernelGGL(w4_pack_codes_kernel, dim3((unsigned)((words + 255) / 256)), dim3(256), 0, s, a);
    hipLaunchKernelGGL(w4_pack_groups_kernel, dim3((unsigned)((pairs + 255) / 256)), dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

// ------------------------------------------------------------------ product
template <int DT>
__device__ __forceinline__ float4_t mfma16(const uint4 &a, const uint4 &b, float4_t c)
{
    if constexpr (DT == DT_F16)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_t, a), __builtin_bit_cast(half8_t, b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf168_t, a), __builtin_bit_cast(bf168_t, b), c, 0, 0, 0);
}

// eight codes of a dword as 16 + c
template <int DT>
__device__ __forceinline__ uint4 widen(uint32_t w)
{
    if constexpr (DT == DT_F16) {       // 16.0 = 0x4c00, unit of the last place 2^-6: the code goes to bits 6..9
        constexpr uint32_t M = 0x03c003c0u, O = 0x4c004c00u;
        return make_uint4(((w << 6) & M) | O, ((w << 2) & M) | O, ((w >> 2) & M) | O, ((w >> 6) & M) | O);
    } else {                            // 16.0 = 0x4180, unit of the last place 2^-3: bits 3..6
        constexpr uint32_t M = 0x00780078u, O = 0x41804180u;
        return make_uint4(((w << 3) & M) | O, ((w >> 1) & M) | O, ((w >> 5) & M) | O, ((w >> 9) & M) | O);
    }
}

constexpr int W4_WAVES = 8;

// What the product of one K tile needs besides x.  `group`: the group of this lane's column c and K step q, scale and 16 + zero point.
template <int NT> struct W4Tile {
    uint4 code[NT];
    uint32_t group[NT];
};

// A workgroup: NT column tiles x MT token tiles, its eight wavefronts share the K tiles (every eighth each, so that together they read
// a column tile's codes in one stretch) and are joined in LDS.  A wavefront asks for its next K tile's codes, groups and - where that
// is few registers - x before it multiplies the present one.  A lane loads the scale and zero point of one column and K step; the
// result's layout wants those of four columns, which come from their lanes through the LDS crossbar.
template <int DT, int MT, int NT>
__global__ __launch_bounds__(64 * W4_WAVES, MT * NT <= 4 ? 4 : 2) void w4_gemv_kernel(const W4Args p)
{
    constexpr bool XPRE = MT == 1 && NT < 4;
    __shared__ float part[W4_WAVES][MT * 16][17];
    // eight neighbouring ids go to the eight XCDs: the token blocks of one column block follow each other on one of them
    const unsigned id = blockIdx.x, blk = (id >> 3) / p.row_blocks, rb = (id >> 3) - blk * p.row_blocks;
    unsigned cb = blk * 8 + (id & 7);
    int proj = 0;
    while (proj + 1 < p.n_proj && cb >= p.pr[proj].end) proj++;
    const W4Proj &w = p.pr[proj];
    if (cb >= w.end) return;
    cb -= proj ? p.pr[proj - 1].end : 0;
    const int nt0 = (int)cb * NT, t0 = (int)rb * (MT * 16);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
    const unsigned char *x0row = static_cast<const unsigned char *>(w.x) + (size_t)t0 * w.hin * 2;
    uint32_t xrow[MT];                                            // bytes from it: 64 rows of 2^24 columns at most
#pragma unroll
    for (int m = 0; m < MT; m++) xrow[m] = ((uint32_t)min(m * 16 + c, p.T - 1 - t0) * (uint32_t)w.hin + q * 8) * 2;
    const uint32_t one = DT == DT_F16 ? 0x3c003c00u : 0x3f803f80u;
    const uint4 ones = make_uint4(one, one, one, one);
    const int steps = 4 / w.per_tile;                             // K steps of 32 rows in a group
    const unsigned glane = (q / steps) * W4_TN + c;

    auto load = [&](W4Tile<NT> &b, int kt) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int nt = min(nt0 + n, w.n_tiles - 1);          // a block past the last column tile repeats it and stores nothing
            const size_t tile = (size_t)nt * w.k_tiles + kt;
            b.code[n] = ldg16_stream(w.packed + tile * W4_TILE_BYTES + lane * 16);
            const unsigned char *plane = w.packed + w.groups_at;
            const size_t at = tile * (w.per_tile * W4_TN) + glane;
            b.group[n] = w.zeros ? reinterpret_cast<const uint32_t *>(plane)[at] : reinterpret_cast<const uint16_t *>(plane)[at] | 24u << 16;
        }
    };
    auto xload = [&](uint4 (&x)[MT], int kt, int s) {
        const int k = kt * W4_TK + s * 32;
#pragma unroll
        for (int m = 0; m < MT; m++) x[m] = k + q * 8 < w.hin ? ldg16(x0row + (xrow[m] + (uint32_t)k * 2)) : zero16();
    };

    float4_t out[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int n = 0; n < NT; n++) out[m][n] = float4_t{0.f, 0.f, 0.f, 0.f};
    // one K tile against x[0..3] (XPRE) or x[0], x[1] by turns, the next step's x on its way
    auto multiply = [&](const W4Tile<NT> &b, int kt, uint4 (&x)[XPRE ? 4 : 2][MT], int next) {
        float4_t acc[MT][NT], sum[MT];
#pragma unroll
        for (int m = 0; m < MT; m++) {
            sum[m] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int n = 0; n < NT; n++) acc[m][n] = float4_t{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int s = 0; s < 4; s++) {
            uint4 (&now)[MT] = x[XPRE ? s : s & 1];
            if constexpr (!XPRE) {
                if (s < 3) xload(x[(s + 1) & 1], kt, s + 1);
                else if (next < w.k_tiles) xload(x[0], next, 0);
            }
#pragma unroll
            for (int m = 0; m < MT; m++) sum[m] = mfma16<DT>(ones, now[m], sum[m]);
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const uint4 a = widen<DT>(s == 0 ? b.code[n].x : s == 1 ? b.code[n].y : s == 2 ? b.code[n].z : b.code[n].w);
#pragma unroll
                for (int m = 0; m < MT; m++) acc[m][n] = mfma16<DT>(a, now[m], acc[m][n]);
            }
            if (((s + 1) & (steps - 1)) == 0) {                   // the group ends here
                const int src = (s & ~(steps - 1)) * 16 + q * 4;
#pragma unroll
                for (int n = 0; n < NT; n++) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t u = (uint32_t)__builtin_amdgcn_ds_bpermute((src + i) * 4, (int)b.group[n]);
                        const float f = lo_f32<DT>(u & 0xffffu), z = (float)(u >> 16);
#pragma unroll
                        for (int m = 0; m < MT; m++) out[m][n][i] += f * (acc[m][n][i] - z * sum[m][i]);
                    }
                }
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    sum[m] = float4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int n = 0; n < NT; n++) acc[m][n] = float4_t{0.f, 0.f, 0.f, 0.f};
                }
            }
            __builtin_amdgcn_sched_barrier(0);                    // or the steps' operands are all made at once and the registers run out
        }
    };
    int kt = wave;
    if (kt < w.k_tiles) {
        W4Tile<NT> b0, b1;
        uint4 x0[XPRE ? 4 : 2][MT], x1[XPRE ? 4 : 1][MT];
        auto fetch = [&](W4Tile<NT> &b, uint4 (*x)[MT], int at) {
            load(b, at);
            if constexpr (XPRE) {
#pragma unroll
                for (int s = 0; s < 4; s++) xload(x[s], at, s);
            }
        };
        fetch(b0, x0, kt);
        if constexpr (!XPRE) xload(x0[0], kt, 0);
#pragma unroll 1
        for (;;) {
            int next = kt + W4_WAVES;
            if (next < w.k_tiles) fetch(b1, x1, next);
            multiply(b0, kt, x0, next);
            if (next >= w.k_tiles) break;
            kt = next;
            next = kt + W4_WAVES;
            if (next < w.k_tiles) fetch(b0, x0, next);
            if constexpr (XPRE) multiply(b1, kt, x1, next); else multiply(b1, kt, x0, next);
            if (next >= w.k_tiles) break;
            kt = next;
        }
    }
#pragma unroll
    for (int n = 0; n < NT; n++) {
        if (n) __syncthreads();
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int i = 0; i < 4; i++) part[wave][m * 16 + c][q * 4 + i] = out[m][n][i];
        __syncthreads();
        for (int e = threadIdx.x; e < MT * 128; e += 64 * W4_WAVES) {
            const int r = e >> 3, col = (e & 7) * 2, at = (nt0 + n) * W4_TN + col;
            if (t0 + r >= p.T || at >= w.hout) continue;
            float v0 = 0.f, v1 = 0.f;
#pragma unroll
            for (int k = 0; k < W4_WAVES; k++) { v0 += part[k][r][col]; v1 += part[k][r][col + 1]; }
            uint32_t *y = reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(w.y) + (size_t)(t0 + r) * w.hout + at);
            if (p.accumulate) { v0 += lo_f32<DT>(*y); v1 += hi_f32<DT>(*y); }
            *y = pack2<DT>(v0, v1);
        }
    }
}

template <int DT, int MT, int NT>
static void gemv_of(W4Args a, hipStream_t s)
{
    unsigned end = 0;
    for (int p = 0; p < a.n_proj; p++) {
        end += (unsigned)((a.pr[p].n_tiles + NT - 1) / NT);
        a.pr[p].end = end;
    }
    a.row_blocks = (unsigned)((a.T + MT * 16 - 1) / (MT * 16));
    hipLaunchKernelGGL((w4_gemv_kernel<DT, MT, NT>), dim3((end + 7) / 8 * 8 * a.row_blocks), dim3(64 * W4_WAVES), 0, s, a);
}

template <int DT>
static void gemv_by_size(const W4Args &a, hipStream_t s)
{
    int tiles = 0;
    for (int p = 0; p < a.n_proj; p++) tiles += a.pr[p].n_tiles;
    const int cus = device_compute_units();
    const int nt = tiles >= 4 * cus ? 4 : tiles >= 2 * cus ? 2 : 1;
    if (a.T <= 16) { if (nt == 4) gemv_of<DT, 1, 4>(a, s); else if (nt == 2) gemv_of<DT, 1, 2>(a, s); else gemv_of<DT, 1, 1>(a, s); }
    else if (a.T <= 32) { if (nt == 4) gemv_of<DT, 2, 4>(a, s); else if (nt == 2) gemv_of<DT, 2, 2>(a, s); else gemv_of<DT, 2, 1>(a, s); }
    else { if (nt == 4) gemv_of<DT, 4, 4>(a, s); else if (nt == 2) gemv_of<DT, 4, 2>(a, s); else gemv_of<DT, 4, 1>(a, s); }
}

int launch_w4_gemv(const W4Args &a, int dtype, hipStream_t s)
{
    if (dtype == DT_F16) gemv_by_size<DT_F16>(a, s); else gemv_by_size<DT_BF16>(a, s);
    return (int)hipGetLastError();
}

}  // namespace mlora

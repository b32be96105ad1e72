// Products of microscaled 4-bit operands:
//     y[t][n] = (accumulate ? y[t][n] : 0) + sum_b 2^(X_x[t][b] + X_w[n][b]) * sum_{k in block b} cx[t][k] * cw[n][k]
// on the scaled 4-bit matrix instructions, which take the two powers of two of every 32 elements beside the codes.  Sums in fp32, rounded once.
#include "mlora_dev.hpp"
#include "mlora_step.hpp"

namespace mlora {

typedef int int8_vec __attribute__((ext_vector_type(8)));

// a: 16 rows of codes, b: 16 rows; lane l of an operand is row l % 16, elements 32 (l / 16) .. + 31 of the K tile.  J: the K tile of its quad, whose byte of
// the scale words counts.  The result: lane l holds b's row l % 16 and a's rows 4 (l / 16) .. + 3.
template <int J>
__device__ __forceinline__ float4_t mx4_mfma16(const uint4 &a, const uint4 &b, float4_t c, uint32_t sa, uint32_t sb)
{
    const int8_vec va = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0}, vb = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(va, vb, c, 4, 4, J, (int)sa, J, (int)sb);
}

constexpr int MX_WAVES = 8;

// 16 columns x 16 tokens a workgroup; its wavefronts take the quads of K tiles in turn and add their sums through LDS in their order.
template <int DT>
__global__ __launch_bounds__(64 * MX_WAVES) void mx4_slim_kernel(const Mx4Args p)
{
    __shared__ float4_t sums[MX_WAVES][64];
    int proj = 0;
    while (proj + 1 < p.n_proj && blockIdx.x >= p.pr[proj].end) proj++;
    const Mx4Proj &w = p.pr[proj];
    const int nt = (int)(blockIdx.x - (proj ? p.pr[proj - 1].end : 0u)), tt = blockIdx.y;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const unsigned char *wc = w.w + (size_t)nt * w.k_tiles * MX4_TILE_BYTES + lane * 16;
    const unsigned char *xc = w.x + (size_t)tt * w.k_tiles * MX4_TILE_BYTES + lane * 16;
    const unsigned char *ws = w.w + w.w_scales_at + (size_t)nt * w.quads * MX4_QUAD_BYTES + lane * 4;
    const unsigned char *xs = w.x + w.x_scales_at + (size_t)tt * w.quads * MX4_QUAD_BYTES + lane * 4;
    float4_t acc = {0.f, 0.f, 0.f, 0.f};
    for (int quad = wave; quad < w.quads; quad += MX_WAVES) {
        const uint32_t sw = *reinterpret_cast<const uint32_t *>(ws + (size_t)quad * MX4_QUAD_BYTES);
        const uint32_t sx = *reinterpret_cast<const uint32_t *>(xs + (size_t)quad * MX4_QUAD_BYTES);
        auto tile = [&](auto j_c) {
            constexpr int j = decltype(j_c)::value;
            const size_t at = (size_t)(quad * 4 + j) * MX4_TILE_BYTES;
            if (quad * 4 + j < w.k_tiles) acc = mx4_mfma16<j>(ldg16(wc + at), ldg16(xc + at), acc, sw, sx);
        };
        tile(std::integral_constant<int, 0>{});
        tile(std::integral_constant<int, 1>{});
        tile(std::integral_constant<int, 2>{});
        tile(std::integral_constant<int, 3>{});
    }
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave) return;
    const int t = tt * 16 + (lane & 15), n = nt * 16 + 4 * (lane >> 4);
    if (t >= p.T || n >= w.hout) return;
    uint2 *y = reinterpret_cast<uint2 *>(static_cast<uint16_t *>(w.y) + (size_t)t * w.hout + n);
    float4_t v = sums[0][lane];
#pragma unroll
    for (int i = 1; i < MX_WAVES; i++) v += sums[i][lane];
    if (p.accumulate) {
        const uint2 o = *y;
        v[0] += lo_f32<DT>(o.x); v[1] += hi_f32<DT>(o.x); v[2] += lo_f32<DT>(o.y); v[3] += hi_f32<DT>(o.y);
    }
    *y = make_uint2(pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]));
}

int64_t mx4_workspace_bytes(const Mx4Args &) { return 0; }

int launch_mx4_gemm(const Mx4Args &all, int dtype, void *, hipStream_t s)
{
    Mx4Args a = all;
    unsigned end = 0;
    for (int p = 0; p < a.n_proj; p++) a.pr[p].end = end += (unsigned)(a.pr[p].hout + 15) / 16;
    const dim3 grid(end, (unsigned)(a.T + 15) / 16);
    if (dtype == DT_F16) hipLaunchKernelGGL((mx4_slim_kernel<DT_F16>), grid, dim3(64 * MX_WAVES), 0, s, a);
    else hipLaunchKernelGGL((mx4_slim_kernel<DT_BF16>), grid, dim3(64 * MX_WAVES), 0, s, a);
    return (int)hipGetLastError();
}

}  // namespace mlora

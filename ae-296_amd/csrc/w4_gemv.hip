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
    if (i >= (long long)p.sh.groups * p.sh.cols) return;
    const int g = (int)(i / p.sh.cols), n = (int)(i % p.sh.cols);
    const bool in = n < p.sh.hout;
    const size_t at = (size_t)g * p.sh.hout + n;
    reinterpret_cast<uint16_t *>(p.packed + p.sh.scales_at)[i] = in ? p.scales[at] : (uint16_t)0;
    if (p.zeros) (p.packed + p.sh.zeros_at)[i] = in ? (p.zeros[at] & 15) : (uint8_t)0;
}

int launch_w4_pack(const W4PackArgs &a, hipStream_t s)
{
    const long long words = (long long)a.sh.n_tiles * a.sh.k_tiles * (W4_TILE_BYTES / 4), pairs = (long long)a.sh.groups * a.sh.cols;
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

// One workgroup: 16 columns x 16 tokens, its four wavefronts share the K tiles.
template <int DT>
__global__ __launch_bounds__(256) void w4_gemv_kernel(const W4Args p)
{
    __shared__ float part[4][16][17];
    const W4Proj &w = p.pr[blockIdx.z];
    const int nt = blockIdx.x, t0 = blockIdx.y * 16;
    if (nt >= w.n_tiles) return;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
    const int t = t0 + c;
    const uint16_t *xrow = static_cast<const uint16_t *>(w.x) + (size_t)(t < p.T ? t : t0) * w.hin;
    const uint32_t one = DT == DT_F16 ? 0x3c003c00u : 0x3f803f80u;
    const uint4 ones = make_uint4(one, one, one, one);
    const int steps = 1 << (w.group_shift - 5);           // K steps of 32 rows in a group
    float4_t out = {0.f, 0.f, 0.f, 0.f};
    for (int kt = wave; kt < w.k_tiles; kt += 4) {
        const uint4 code = ldg16(w.codes + ((size_t)nt * w.k_tiles + kt) * W4_TILE_BYTES + lane * 16);
        const uint32_t words[4] = {code.x, code.y, code.z, code.w};
        float4_t acc = {0.f, 0.f, 0.f, 0.f}, sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < 4; s++) {
            const int k = kt * W4_TK + s * 32 + q * 8;
            const uint4 x = k < w.hin ? ldg16(xrow + k) : zero16();
            acc = mfma16<DT>(widen<DT>(words[s]), x, acc);
            sum = mfma16<DT>(ones, x, sum);
            if (((s + 1) & (steps - 1)) == 0) {
                const int g = (kt * W4_TK + s * 32) >> w.group_shift;
                if (g < w.groups) {
                    const size_t at = (size_t)g * w.cols + nt * W4_TN + q * 4;
                    const uint2 sc = *reinterpret_cast<const uint2 *>(w.scales + at);
                    const uint32_t z = w.zeros ? *reinterpret_cast<const uint32_t *>(w.zeros + at) : 0x08080808u;
                    const float f[4] = {lo_f32<DT>(sc.x), hi_f32<DT>(sc.x), lo_f32<DT>(sc.y), hi_f32<DT>(sc.y)};
#pragma unroll
                    for (int i = 0; i < 4; i++) out[i] += f[i] * (acc[i] - (float)(16u + ((z >> (8 * i)) & 15u)) * sum[i]);
                }
                acc = float4_t{0.f, 0.f, 0.f, 0.f};
                sum = float4_t{0.f, 0.f, 0.f, 0.f};
            }
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) part[wave][c][q * 4 + i] = out[i];
    __syncthreads();
    const int r = threadIdx.x >> 4, n = nt * W4_TN + (threadIdx.x & 15);
    if (t0 + r >= p.T || n >= w.hout) return;
    float v = 0.f;
    for (int k = 0; k < 4; k++) v += part[k][r][threadIdx.x & 15];
    uint16_t *y = static_cast<uint16_t *>(w.y) + (size_t)(t0 + r) * w.hout + n;
    if (p.accumulate) v += lo_f32<DT>(*y);
    *y = (uint16_t)pack2<DT>(v, 0.f);
}

int launch_w4_gemv(const W4Args &a, int dtype, hipStream_t s)
{
    int tiles = 0;
    for (int p = 0; p < a.n_proj; p++) tiles = a.pr[p].n_tiles > tiles ? a.pr[p].n_tiles : tiles;
    const dim3 grid((unsigned)tiles, (unsigned)((a.T + 15) / 16), (unsigned)a.n_proj);
    if (dtype == DT_F16) hipLaunchKernelGGL((w4_gemv_kernel<DT_F16>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((w4_gemv_kernel<DT_BF16>), grid, dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

}  // namespace mlora

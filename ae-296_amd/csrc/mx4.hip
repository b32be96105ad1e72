// Microscaled 4-bit numbers (MXFP4): quantisation of 16-bit rows, packing of a checkpoint's codes, and the values they stand for.
//     X = max(floor(log2(max |x| over a block of 32)) - 2, -127),  code = the nearest of 0 .5 1 1.5 2 3 4 6 to |x| / 2^X, ties to the even code
// The largest magnitude of a block lands in [4, 8), above 6 it saturates; both steps are exact in the 16-bit types, so there is one right answer.
// The code comes from the scaled conversion of gfx950, which does this rounding for two elements at once.
//
// All three move bytes and are bound by HBM or, for few rows, by the launch.
#include "mlora_dev.hpp"
#include "mlora_step.hpp"

namespace mlora {

// Where block q of K tile kt of row r lies: sixteen bytes of codes, and the byte of its scale.
__device__ __forceinline__ size_t mx4_codes_at(const Mx4Shape &sh, int r, int kt, int q)
{
    return ((size_t)(r >> 4) * sh.k_tiles + kt) * MX4_TILE_BYTES + (q * 16 + (r & 15)) * 16;
}
__device__ __forceinline__ size_t mx4_quad_at(const Mx4Shape &sh, int r, int quad, int q)
{
    return (size_t)sh.scales_at + ((size_t)(r >> 4) * sh.quads + quad) * MX4_QUAD_BYTES + (q * 16 + (r & 15)) * 4;
}

template <int DT>
__device__ __forceinline__ uint32_t mx4_codes8(const uint4 &x, float scale)
{
    uint32_t w = 0;
    if constexpr (DT == DT_F16) {
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(half2_t, x.x), scale, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(half2_t, x.y), scale, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(half2_t, x.z), scale, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(w, __builtin_bit_cast(half2_t, x.w), scale, 3);
    } else {
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf162_t, x.x), scale, 0);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf162_t, x.y), scale, 1);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf162_t, x.z), scale, 2);
        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(w, __builtin_bit_cast(bf162_t, x.w), scale, 3);
    }
    return w;
}

// The scale byte of a block from the largest pattern without sign of its elements: as numbers, patterns without sign are in the values' order, and
// an infinity or a NaN is at least the infinity's.  Exponents of fp32 hold those of both types, but for bf16's own subnormals, whose
// scale is the smallest anyway.
template <int DT>
__device__ __forceinline__ uint32_t mx4_scale(uint32_t largest)
{
    if (largest >= (DT == DT_F16 ? 0x7c00u : 0x7f80u)) return 255u;
    const uint32_t e = __builtin_bit_cast(uint32_t, lo_f32<DT>(largest)) >> 23;
    return e > 2u ? e - 2u : 0u;
}

// A wavefront quantises 16 rows x 512 columns: four lanes a block, lane 4 r + s the elements 8 s .. of row r, so that the four blocks of a K tile
// are four loads of 64 bytes a row and the codes of 16 rows leave as 256 consecutive bytes a block column.
template <int DT>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const Mx4QuantArgs p)
{
    const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int quad = (int)(unit % p.sh.quads);
    const long long row0 = unit / p.sh.quads * 16;
    const int lane = threadIdx.x & 63, s = lane & 3;
    const long long r = row0 + (lane >> 2);
    if (r >= p.sh.rows) return;
    const uint16_t *__restrict__ x = p.x + r * p.x_stride;
    const int kts = p.sh.k_tiles - quad * 4 < 4 ? p.sh.k_tiles - quad * 4 : 4;
    uint32_t bytes = 0;                                     // scales of block column s of the quad's K tiles
    for (int j = 0; j < kts; j++) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int k = (quad * 4 + j) * MX4_TK + q * 32 + s * 8;
            const uint4 v = k < p.sh.k ? ldg16(x + k) : zero16();
            const uint32_t a = v.x & 0x7fff7fffu, b = v.y & 0x7fff7fffu, c = v.z & 0x7fff7fffu, d = v.w & 0x7fff7fffu;
            uint32_t m = max(max(max(a & 0xffffu, a >> 16), max(b & 0xffffu, b >> 16)), max(max(c & 0xffffu, c >> 16), max(d & 0xffffu, d >> 16)));
            m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, false));
            m = max(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, false));
            const uint32_t e = mx4_scale<DT>(m);
            // 2^-127 is half the smallest normal number
            const float scale = __builtin_bit_cast(float, e == 0 ? 0x00400000u : e == 255u ? 0x3f800000u : e << 23);
            *reinterpret_cast<uint32_t *>(p.packed + mx4_codes_at(p.sh, (int)r, quad * 4 + j, q) + s * 4) = mx4_codes8<DT>(v, scale);
            if (q == s) bytes |= e << (8 * j);
        }
    }
    *reinterpret_cast<uint32_t *>(p.packed + mx4_quad_at(p.sh, (int)r, quad, s)) = bytes;
}

int launch_mx4_quantize(const Mx4QuantArgs &a, int dtype, hipStream_t s)
{
    const long long units = (long long)a.sh.row_tiles * a.sh.quads;
    const dim3 grid((unsigned)((units + 3) / 4));
    if (dtype == DT_F16) hipLaunchKernelGGL((mx4_quantize_kernel<DT_F16>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((mx4_quantize_kernel<DT_BF16>), grid, dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

// From a checkpoint's form, codes [rows, k / 2] with an even column in the low half and scales [rows, blocks]: one thread a dword of codes.
__global__ __launch_bounds__(256) void mx4_pack_kernel(const Mx4PackArgs p)
{
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long words = (long long)p.sh.row_tiles * p.sh.k_tiles * (MX4_TILE_BYTES / 4);
    if (i < words) {
        const long long tile = i / (MX4_TILE_BYTES / 4);
        const int slot = (int)(i >> 2) & 63, kt = (int)(tile % p.sh.k_tiles);
        const long long r = tile / p.sh.k_tiles * 16 + (slot & 15);
        const int k = kt * MX4_TK + (slot >> 4) * 32 + (int)(i & 3) * 8;
        uint32_t w = 0;
        if (r < p.sh.rows && k < p.sh.k)
            for (int b = 0; b < 4; b++) w |= (uint32_t)p.codes[r * (p.sh.k / 2) + k / 2 + b] << (8 * b);
        reinterpret_cast<uint32_t *>(p.packed)[i] = w;
    }
    const long long dwords = (long long)p.sh.row_tiles * p.sh.quads * (MX4_QUAD_BYTES / 4);
    if (i < dwords) {
        const long long at = i / (MX4_QUAD_BYTES / 4);
        const int slot = (int)(i & 63), quad = (int)(at % p.sh.quads);
        const long long r = at / p.sh.quads * 16 + (slot & 15);
        uint32_t w = 0;
        for (int j = 0; j < 4; j++) {
            const int block = (quad * 4 + j) * 4 + (slot >> 4);
            if (r < p.sh.rows && block < p.sh.blocks) w |= (uint32_t)p.scales[r * p.sh.blocks + block] << (8 * j);
        }
        reinterpret_cast<uint32_t *>(p.packed + p.sh.scales_at)[i] = w;
    }
}

int launch_mx4_pack(const Mx4PackArgs &a, hipStream_t s)
{
    const long long words = (long long)a.sh.row_tiles * a.sh.k_tiles * (MX4_TILE_BYTES / 4);
    hipLaunchKernelGGL(mx4_pack_kernel, dim3((unsigned)((words + 255) / 256)), dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

// code * 2^X in fp32, exact, rounded to the 16-bit type; NaN where the block's scale is
template <int DT>
__global__ __launch_bounds__(256) void mx4_values_kernel(const Mx4ValuesArgs p)
{
    const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int quad = (int)(unit % p.sh.quads);
    const long long row0 = unit / p.sh.quads * 16;
    const int lane = threadIdx.x & 63, s = lane & 3;
    const long long r = row0 + (lane >> 2);
    if (r >= p.sh.rows) return;
    const int kts = p.sh.k_tiles - quad * 4 < 4 ? p.sh.k_tiles - quad * 4 : 4;
    for (int j = 0; j < kts; j++) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int k = (quad * 4 + j) * MX4_TK + q * 32 + s * 8;
            if (k >= p.sh.k) continue;
            const uint32_t w = *reinterpret_cast<const uint32_t *>(p.packed + mx4_codes_at(p.sh, (int)r, quad * 4 + j, q) + s * 4);
            const uint32_t e = (*reinterpret_cast<const uint32_t *>(p.packed + mx4_quad_at(p.sh, (int)r, quad, q)) >> (8 * j)) & 255u;
            const float scale = __builtin_bit_cast(float, e == 0 ? 0x00400000u : e == 255u ? 0x7fc00000u : e << 23);
            typedef float f32x2 __attribute__((ext_vector_type(2)));
            float f[8];
            f32x2 t;
            t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 0); f[0] = t[0] * scale; f[1] = t[1] * scale;
            t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 1); f[2] = t[0] * scale; f[3] = t[1] * scale;
            t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 2); f[4] = t[0] * scale; f[5] = t[1] * scale;
            t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, 1.f, 3); f[6] = t[0] * scale; f[7] = t[1] * scale;
            stg16(p.out + r * p.out_stride + k, pack8<DT>(f));
        }
    }
}

int launch_mx4_values(const Mx4ValuesArgs &a, int dtype, hipStream_t s)
{
    const long long units = (long long)a.sh.row_tiles * a.sh.quads;
    const dim3 grid((unsigned)((units + 3) / 4));
    if (dtype == DT_F16) hipLaunchKernelGGL((mx4_values_kernel<DT_F16>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((mx4_values_kernel<DT_BF16>), grid, dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

}  // namespace mlora

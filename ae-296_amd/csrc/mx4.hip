// Microscaled 4-bit numbers (MXFP4): quantisation of 16-bit rows, packing of a checkpoint's codes, and the values they stand for.
//     X = max(floor(log2(max |x| over a block of 32)) - 2, -127),  code = the nearest of 0 .5 1 1.5 2 3 4 6 to |x| / 2^X, ties to the even code
// The largest magnitude of a block lands in [4, 8), above 6 it saturates; both steps are exact in the 16-bit types, so there is one right answer.
// The code comes from the scaled conversion of gfx950, which does this rounding for two elements at once.
//
// All three move bytes and are bound by HBM or, for few rows, by the launch.
#include "mlora_dev.hpp"
#include "mlora_step.hpp"

namespace mlora {

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

__device__ __forceinline__ uint32_t quad_swap1(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xB1, 0xF, 0xF, false); }
__device__ __forceinline__ uint32_t quad_swap2(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4E, 0xF, 0xF, false); }

// Among each four neighbouring lanes: value j of lane s goes to value s of lane j.
__device__ __forceinline__ void quad_transpose(uint32_t (&v)[4])
{
    const bool odd = threadIdx.x & 1, high = threadIdx.x & 2;
#pragma unroll
    for (int i = 0; i < 4; i += 2) {
        const uint32_t got = quad_swap1(odd ? v[i] : v[i + 1]);
        if (odd) v[i] = got; else v[i + 1] = got;
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint32_t got = quad_swap2(high ? v[i] : v[i + 2]);
        if (high) v[i] = got; else v[i + 2] = got;
    }
}

// 2^(byte - 127): 2^-127 is half the smallest normal number
__device__ __forceinline__ float mx4_power(uint32_t e) { return __builtin_bit_cast(float, e == 0 ? 0x00400000u : e << 23); }

// A wavefront quantises a tile, 16 rows x 128 columns.  It reads four rows at a time, a row's columns by sixteen lanes (256 consecutive bytes), so that four
// lanes hold a block; exchanged among these, the codes of the sixteen rows are sixteen bytes a lane, the tile's kilobyte in one store.  8191 x 13824: 46 us,
// 6.2 TB/s read + written; 1 x 4096: 2.3 us.  (A quad a wavefront, all its loads in flight and its scales as dwords: 49 and 3.7; 4 lanes a block of
// sixteen rows at once, 64 bytes a row: 81 and 7.6.)
template <int DT>
__global__ __launch_bounds__(256) void mx4_quantize_kernel(const Mx4QuantArgs p)
{
    const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const long long row_tile = unit / p.sh.k_tiles;
    if (row_tile >= p.sh.row_tiles) return;
    const int kt = (int)(unit - row_tile * p.sh.k_tiles);
    const int lane = threadIdx.x & 63, s = lane & 3, q = lane >> 2 & 3, rr = lane >> 4;
    const int k = kt * MX4_TK + (lane & 15) * 8;
    uint4 x[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const long long r = row_tile * 16 + 4 * i + rr;
        x[i] = r < p.sh.rows && k < p.sh.k ? ldg16_stream(p.x + r * p.x_stride + k) : zero16();
    }
    uint32_t w[4], mine = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint4 v = x[i];
        const uint32_t a = v.x & 0x7fff7fffu, b = v.y & 0x7fff7fffu, c = v.z & 0x7fff7fffu, d = v.w & 0x7fff7fffu;
        uint32_t m = max(max(max(a & 0xffffu, a >> 16), max(b & 0xffffu, b >> 16)), max(max(c & 0xffffu, c >> 16), max(d & 0xffffu, d >> 16)));
        m = max(m, quad_swap1(m));
        m = max(m, quad_swap2(m));
        const uint32_t e = mx4_scale<DT>(m);
        w[i] = mx4_codes8<DT>(v, e == 255u ? 1.f : mx4_power(e));
        if (i == s) mine = e;
    }
    quad_transpose(w);
    const int slot = q * 16 + 4 * s + rr;                   // of the row whose block q this lane stores
    stg16(p.packed + ((size_t)row_tile * p.sh.k_tiles + kt) * MX4_TILE_BYTES + slot * 16, make_uint4(w[0], w[1], w[2], w[3]));
    unsigned char *scale = p.packed + p.sh.scales_at + ((size_t)row_tile * p.sh.quads + kt / 4) * MX4_QUAD_BYTES + slot * 4;
    scale[kt & 3] = (unsigned char)mine;
    if (kt + 1 == p.sh.k_tiles)                             // the quad's tiles that are not there: multiplied by zero codes, but not as NaN
        for (int j = (kt & 3) + 1; j < 4; j++) scale[j] = 0;
}

int launch_mx4_quantize(const Mx4QuantArgs &a, int dtype, hipStream_t s)
{
    const dim3 grid((unsigned)(((long long)a.sh.row_tiles * a.sh.k_tiles + 3) / 4));
    if (dtype == DT_F16) hipLaunchKernelGGL((mx4_quantize_kernel<DT_F16>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((mx4_quantize_kernel<DT_BF16>), grid, dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

// From a checkpoint's form, codes [rows, k / 2] with an even column in the low half and scales [rows, blocks]: one thread a dword of codes.  Made
// once a weight, so codes are read in single bytes and nothing more was done about it: 4096 x 4096 10.9 us, 13824 x 5120 39.7 (1.6 to 1.9 TB/s read + written).
__global__ __launch_bounds__(256) void mx4_pack_kernel(const Mx4PackArgs p)
{
    const long long words = (long long)p.sh.row_tiles * p.sh.k_tiles * (MX4_TILE_BYTES / 4), dwords = (long long)p.sh.row_tiles * p.sh.quads * (MX4_QUAD_BYTES / 4);
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < words; i += (long long)gridDim.x * 256) {
        const long long tile = i / (MX4_TILE_BYTES / 4);
        const int slot = (int)(i >> 2) & 63, kt = (int)(tile % p.sh.k_tiles);
        const long long r = tile / p.sh.k_tiles * 16 + (slot & 15);
        const int k = kt * MX4_TK + (slot >> 4) * 32 + (int)(i & 3) * 8;
        uint32_t w = 0;
        if (r < p.sh.rows && k < p.sh.k)
            for (int b = 0; b < 4; b++) w |= (uint32_t)p.codes[r * (p.sh.k / 2) + k / 2 + b] << (8 * b);
        reinterpret_cast<uint32_t *>(p.packed)[i] = w;
        if (i >= dwords) continue;                       // fewer dwords of scales than words of codes
        const long long at = i / (MX4_QUAD_BYTES / 4);
        const int sslot = (int)(i & 63), quad = (int)(at % p.sh.quads);
        const long long sr = at / p.sh.quads * 16 + (sslot & 15);
        w = 0;
        for (int j = 0; j < 4; j++) {
            const int block = (quad * 4 + j) * 4 + (sslot >> 4);
            if (sr < p.sh.rows && block < p.sh.blocks) w |= (uint32_t)p.scales[sr * p.sh.blocks + block] << (8 * j);
        }
        reinterpret_cast<uint32_t *>(p.packed + p.sh.scales_at)[i] = w;
    }
}

int launch_mx4_pack(const Mx4PackArgs &a, hipStream_t s)
{
    const long long groups = (long long)a.sh.row_tiles * a.sh.k_tiles, most = 1 << 20;      // of 256 words, a tile
    hipLaunchKernelGGL(mx4_pack_kernel, dim3((unsigned)(groups < most ? groups : most)), dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

// code * 2^X in fp32, exact, rounded to the 16-bit type; NaN where the block's scale is.  The quantisation's way back (8191 x 13824: 49 us).
template <int DT>
__global__ __launch_bounds__(256) void mx4_values_kernel(const Mx4ValuesArgs p)
{
    const long long unit = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const long long row_tile = unit / p.sh.k_tiles;
    if (row_tile >= p.sh.row_tiles) return;
    const int kt = (int)(unit - row_tile * p.sh.k_tiles);
    const int lane = threadIdx.x & 63, s = lane & 3, q = lane >> 2 & 3, rr = lane >> 4, slot = q * 16 + 4 * s + rr;
    const int k = kt * MX4_TK + (lane & 15) * 8;
    const uint4 codes = ldg16_stream(p.packed + ((size_t)row_tile * p.sh.k_tiles + kt) * MX4_TILE_BYTES + slot * 16);
    const uint32_t e = p.packed[p.sh.scales_at + ((size_t)row_tile * p.sh.quads + kt / 4) * MX4_QUAD_BYTES + slot * 4 + (kt & 3)];
    uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
    quad_transpose(w);                                      // now w[i] is this lane's eight columns of row 4 i + rr
    const float mine = e == 255u ? __builtin_bit_cast(float, 0x7fc00000u) : mx4_power(e);
    float scale[4];                                         // lane i of the four has that of row 4 i + rr
    scale[0] = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, mine), 0x00, 0xF, 0xF, false));
    scale[1] = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, mine), 0x55, 0xF, 0xF, false));
    scale[2] = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, mine), 0xAA, 0xF, 0xF, false));
    scale[3] = __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, mine), 0xFF, 0xF, 0xF, false));
#pragma unroll
    for (int i = 0; i < 4; i++) {
        typedef float f32x2 __attribute__((ext_vector_type(2)));
        float f[8];
        f32x2 t;
        t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.f, 0); f[0] = t[0] * scale[i]; f[1] = t[1] * scale[i];
        t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.f, 1); f[2] = t[0] * scale[i]; f[3] = t[1] * scale[i];
        t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.f, 2); f[4] = t[0] * scale[i]; f[5] = t[1] * scale[i];
        t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[i], 1.f, 3); f[6] = t[0] * scale[i]; f[7] = t[1] * scale[i];
        const long long r = row_tile * 16 + 4 * i + rr;
        if (r < p.sh.rows && k < p.sh.k) stg16_stream(p.out + r * p.out_stride + k, pack8<DT>(f));
    }
}

int launch_mx4_values(const Mx4ValuesArgs &a, int dtype, hipStream_t s)
{
    const dim3 grid((unsigned)(((long long)a.sh.row_tiles * a.sh.k_tiles + 3) / 4));
    if (dtype == DT_F16) hipLaunchKernelGGL((mx4_values_kernel<DT_F16>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((mx4_values_kernel<DT_BF16>), grid, dim3(256), 0, s, a);
    return (int)hipGetLastError();
}

}  // namespace mlora

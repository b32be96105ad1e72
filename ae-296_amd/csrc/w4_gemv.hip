// Base projections on 4-bit weights for the tokens of a decode batch:
//     y[t][n] = (accumulate ? y[t][n] : 0) + sum_g s[g][n] * sum_{k in g} (c[k][n] - z[g][n]) * x[t][k]
//
// A code becomes a 16-bit float without a conversion: shifted to the place of the top mantissa bits and joined with the pattern of
// 16.0 it reads 16 + c, exactly, in fp16 and in bf16 alike (two instructions for two codes).  The 16 and the zero point come off after the
// products: with X = sum of x over the group, sum (c - z) x = sum (16 + c) x - (16 + z) X.  X is one more MFMA per K step whose weight operand is
// ones, so it lands in the lanes that need it; products are exact in fp32 and the difference costs about two bits of its 24.
// Where x is infinite, or so large that 16 x leaves fp32, the difference is infinity less infinity: a result that is not finite is computed again
// from the formula itself (w4_again).
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

// Eight codes of a dword as 16 + c.  fp16: 16.0 is 0x4c00 with a unit of the last place of 2^-6, so the code goes to bits 6..9; bf16: 0x4180 and
// 2^-3, bits 3..6.  The mask comes in a vector register: an instruction that joins after masking takes one constant, not two, and
// with both constants known the compiler makes two instructions of it (one token, 5120 -> 27648: 20.8 us against 18.3).
template <int DT>
__device__ __forceinline__ uint4 widen(uint32_t w, uint32_t mask)
{
    if constexpr (DT == DT_F16) {
        constexpr uint32_t O = 0x4c004c00u;
        return make_uint4(((w << 6) & mask) | O, ((w << 2) & mask) | O, ((w >> 2) & mask) | O, ((w >> 6) & mask) | O);
    } else {
        constexpr uint32_t O = 0x41804180u;
        return make_uint4(((w << 3) & mask) | O, ((w >> 1) & mask) | O, ((w >> 5) & mask) | O, ((w >> 9) & mask) | O);
    }
}

template <int DT>
__device__ __forceinline__ uint32_t widen_mask()
{
    uint32_t m = DT == DT_F16 ? 0x03c003c0u : 0x00780078u;
    asm volatile("" : "+v"(m));
    return m;
}

constexpr int W4_WAVES = 8;

// What a row of x reads past its last column: loaded like the rest, it costs the product nothing (zeros put in place of loaded values there
// took a quarter of the vector instructions of the kernel for more tokens).
__device__ const uint4 w4_no_x = {0u, 0u, 0u, 0u};

// What the product of one K tile needs besides x.  `group`: the group of this lane's column c and K step q, scale and 16 + zero point.
template <int NT> struct W4Tile {
    uint4 code[NT];
    uint32_t group[NT];
};

// From a group's word, scale and 16 + zero point: what its sum of (16 + c) x and its sum of x are multiplied by.  Both are exact, and made once a
// lane before the result's layout spreads them over four columns a lane.
template <int DT>
__device__ __forceinline__ void w4_factors(float (*to)[64], int lane, uint32_t word)
{
    const float f = lo_f32<DT>(word);
    to[0][lane] = f;
    to[1][lane] = -f * (float)(word >> 16);
}

__device__ __forceinline__ bool w4_finite(float v) { return fabsf(v) < INFINITY; }

// Results of a wavefront that are not finite, from the formula in 64 bits, one after the other, the wavefront's lanes along k.  `mine`: a bit for
// each such result of this lane; at(lane, bit, t, n): its token and column.  y holds there what is to be accumulated.  All 64 lanes come here.
// 32 tokens, 11008 -> 4096: 17 us where all is finite, as without it; 227 with one infinite row.
template <int DT, typename At>
__device__ __forceinline__ void w4_again(const W4Proj &w, bool accumulate, uint32_t mine, At at)
{
    const int lane = threadIdx.x & 63;
    const int per_tile = w.per_tile, group_shift = per_tile == 1 ? 7 : per_tile == 2 ? 6 : 5;
    for (uint64_t lanes = __ballot(mine != 0); lanes; lanes = __ballot(mine != 0)) {
        const int from = __builtin_ctzll(lanes), bit = __builtin_ctz(__builtin_amdgcn_readlane((int)mine, from));
        int t, n;
        at(from, bit, t, n);
        const uint16_t *x = static_cast<const uint16_t *>(w.x) + (size_t)t * w.hin;
        const unsigned char *groups = w.packed + w.groups_at;
        double sum = 0.0;
        for (int k = lane * 8; k < w.hin; k += 512) {
            const size_t tile = (size_t)(n / W4_TN) * w.k_tiles + k / W4_TK;
            const uint32_t code = *reinterpret_cast<const uint32_t *>(w.packed + tile * W4_TILE_BYTES + ((k >> 3 & 3) * 16 + n % W4_TN) * 16 + (k >> 5 & 3) * 4);
            const size_t g = (tile * per_tile + ((k & (W4_TK - 1)) >> group_shift)) * W4_TN + n % W4_TN;
            const uint32_t word = w.zeros ? reinterpret_cast<const uint32_t *>(groups)[g] : reinterpret_cast<const uint16_t *>(groups)[g] | 24u << 16;
            const float scale = lo_f32<DT>(word);
            const int zero = (int)(word >> 16) - 16;
            float f[8];
            unpack8<DT>(ldg16(x + k), f);
#pragma unroll
            for (int j = 0; j < 8; j++) sum += (double)(scale * (float)((int)(code >> (4 * (j >> 1) + 16 * (j & 1)) & 15u) - zero)) * (double)f[j];
        }
        for (int o = 32; o; o >>= 1) sum += __shfl_xor(sum, o);
        if (lane == from) {
            uint16_t *y = static_cast<uint16_t *>(w.y) + (size_t)t * w.hout + n;
            float v = (float)sum;
            if (accumulate) v += lo_f32<DT>(*y);
            *y = (uint16_t)pack2<DT>(v, 0.f);
            mine &= mine - 1;
        }
    }
}

// The column block, token block and projection of a workgroup.  Eight neighbouring ids go to the eight XCDs: the token blocks of one
// column block follow each other on one of them.
struct W4Place { int proj; unsigned col_block, row_block; };
__device__ __forceinline__ W4Place w4_place(const W4Args &p)
{
    const unsigned id = blockIdx.x, blk = (id >> 3) / p.row_blocks;
    W4Place at = {0, blk * 8 + (id & 7), (id >> 3) - blk * p.row_blocks};
    while (at.proj < p.n_proj && at.col_block >= p.pr[at.proj].end) at.proj++;
    if (at.proj && at.proj < p.n_proj) at.col_block -= p.pr[at.proj - 1].end;
    return at;                                                    // proj == n_proj: no such block
}

// 16 tokens a token block.  A workgroup: NT column tiles, its eight wavefronts share the K tiles (every eighth each, so that together they read
// a column tile's codes in one stretch) and are joined in LDS.  A wavefront asks for its next K tile's codes, groups and x before it
// multiplies the present one.  A lane loads the scale and zero point of one column and K step; the result's layout wants those of
// four columns, which it gets through LDS.  Bound by the way in and out at one projection (4096 -> 4096, one token, 8.7 MB: 5.0 us, 5.7
// with the weights from HBM; the launch alone takes half) and by vector instructions beyond (one token, 5120 -> 27648, 73 MB: 19.3 us, 3.8 TB/s).
template <int DT, int NT, int STEPS>
__global__ __launch_bounds__(64 * W4_WAVES, 4) void w4_gemv_kernel(const W4Args p)
{
    constexpr int PER_TILE = 4 / STEPS;
    __shared__ float part[W4_WAVES][16][17];
    __shared__ __attribute__((aligned(16))) float factors[W4_WAVES][NT][2][64];
    const W4Place place = w4_place(p);
    if (place.proj == p.n_proj) return;
    const W4Proj &w = p.pr[place.proj];
    const int nt0 = (int)place.col_block * NT, t0 = (int)place.row_block * 16;
    const unsigned char *codes = w.packed, *groups = w.packed + w.groups_at;
    const int hin = w.hin, k_tiles = w.k_tiles, n_last = w.n_tiles - 1;
    const bool zeros = w.zeros != 0;
    const uint32_t middle = zeros ? 0u : 24u << 16;               // 16 + 8 where no zero points are stored; joined on the way to LDS: a load is
                                                                  // waited for by the first instruction that touches what it brings
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
    const unsigned char *x_block = static_cast<const unsigned char *>(w.x) + (size_t)t0 * hin * 2;
    const uint32_t x_row = ((uint32_t)min(c, p.T - 1 - t0) * (uint32_t)hin + q * 8) * 2;
    const uint32_t one = DT == DT_F16 ? 0x3c003c00u : 0x3f803f80u;
    const uint4 ones = make_uint4(one, one, one, one);
    const uint32_t mask = widen_mask<DT>();
    const unsigned group_lane = (q / STEPS) * W4_TN + c;

    auto fetch = [&](W4Tile<NT> &b, uint4 (&x)[4], int kt) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const size_t tile = (size_t)min(nt0 + n, n_last) * k_tiles + kt;   // past the last column tile: that one, and nothing is stored
            const size_t at = tile * (PER_TILE * W4_TN) + group_lane;
            b.code[n] = ldg16_stream(codes + tile * W4_TILE_BYTES + lane * 16);
            b.group[n] = zeros ? reinterpret_cast<const uint32_t *>(groups)[at] : reinterpret_cast<const uint16_t *>(groups)[at];
        }
        const unsigned char *x_tile = x_block + (uint32_t)kt * (W4_TK * 2);
        if ((kt + 1) * W4_TK <= hin) {                            // chosen lane by lane in every tile: 1 to 2 % slower
#pragma unroll
            for (int s = 0; s < 4; s++) x[s] = ldg16(x_tile + (x_row + s * 64));
        } else {
#pragma unroll
            for (int s = 0; s < 4; s++)
                x[s] = ldg16(kt * W4_TK + s * 32 + q * 8 < hin ? x_tile + (x_row + s * 64) : reinterpret_cast<const unsigned char *>(&w4_no_x));
        }
    };

    float4_t out[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) out[n] = float4_t{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](const W4Tile<NT> &b, const uint4 (&x)[4]) {
#pragma unroll
        for (int n = 0; n < NT; n++) w4_factors<DT>(factors[wave][n], lane, b.group[n] | middle);
        __builtin_amdgcn_wave_barrier();
        float4_t acc[NT], sum;
#pragma unroll
        for (int s = 0; s < 4; s++) {
            const bool begins = s % STEPS == 0;                   // a group begins here: its sums start from nothing
            const float4_t none = {0.f, 0.f, 0.f, 0.f};
            sum = mfma16<DT>(ones, x[s], begins ? none : sum);
#pragma unroll
            for (int n = 0; n < NT; n++)
                acc[n] = mfma16<DT>(widen<DT>(s == 0 ? b.code[n].x : s == 1 ? b.code[n].y : s == 2 ? b.code[n].z : b.code[n].w, mask), x[s], begins ? none : acc[n]);
            if ((s + 1) % STEPS == 0) {                           // and ends here
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    const float4_t f = *reinterpret_cast<const float4_t *>(&factors[wave][n][0][s / STEPS * STEPS * 16 + q * 4]);
                    const float4_t z = *reinterpret_cast<const float4_t *>(&factors[wave][n][1][s / STEPS * STEPS * 16 + q * 4]);
#pragma unroll
                    for (int i = 0; i < 4; i++) out[n][i] = fmaf(z[i], sum[i], fmaf(f[i], acc[n][i], out[n][i]));
                }
            }
            __builtin_amdgcn_sched_barrier(0);                    // or the steps' operands are all made at once and the registers run out
        }
    };
    if (wave < k_tiles) {
        W4Tile<NT> b0, b1;
        uint4 x0[4], x1[4];
        int kt = wave;
        fetch(b0, x0, kt);
#pragma unroll 1
        for (;;) {
            kt += W4_WAVES;
            if (kt < k_tiles) fetch(b1, x1, kt);
            multiply(b0, x0);
            if (kt >= k_tiles) break;
            kt += W4_WAVES;
            if (kt < k_tiles) fetch(b0, x0, kt);
            multiply(b1, x1);
            if (kt >= k_tiles) break;
        }
    }
    uint32_t again = 0;                                           // bit 2 n + i: this lane's i-th result of column tile n
#pragma unroll
    for (int n = 0; n < NT; n++) {
        if (n) __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; i++) part[wave][c][q * 4 + i] = out[n][i];
        __syncthreads();
        if (threadIdx.x >= 128) continue;
        const int r = threadIdx.x >> 3, col = (threadIdx.x & 7) * 2, at = (nt0 + n) * W4_TN + col;
        if (t0 + r >= p.T || at >= w.hout) continue;
        float v0 = 0.f, v1 = 0.f;
#pragma unroll
        for (int k = 0; k < W4_WAVES; k++) { v0 += part[k][r][col]; v1 += part[k][r][col + 1]; }
        uint32_t *y = reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(w.y) + (size_t)(t0 + r) * w.hout + at);
        const bool ok0 = w4_finite(v0), ok1 = w4_finite(v1);
        again |= (ok0 ? 0u : 1u) << 2 * n | (ok1 ? 0u : 2u) << 2 * n;
        if (p.accumulate) {                                       // what is computed again finds y as it was
            const float y0 = lo_f32<DT>(*y), y1 = hi_f32<DT>(*y);
            v0 = ok0 ? v0 + y0 : y0;
            v1 = ok1 ? v1 + y1 : y1;
        }
        *y = pack2<DT>(v0, v1);
    }
    w4_again<DT>(w, p.accumulate, again, [&](int from, int bit, int &t, int &n) {
        const int thread = wave * 64 + from;
        t = t0 + (thread >> 3);
        n = (nt0 + (bit >> 1)) * W4_TN + (thread & 7) * 2 + (bit & 1);
    });
}

// ------------------------------------------------------------------ product, more tokens
// With more tokens the token blocks of the kernel above read the codes again, and a wavefront as many bytes of x as of codes.  Here WN wavefronts side by side (NT column
// tiles each) share the x of a K tile through LDS, and the 8 / WN such parts of a workgroup take K tiles by turns.  x comes by loads
// that fill LDS directly, whole rows of 256 bytes; 16-byte chunk `ch` of row r lies at chunk ch ^ (r % 16), so that the operand reads (one
// chunk of sixteen rows) meet all banks.
//
// The sums of x of the next tile are shared: a wavefront makes those of 4 MT / WN steps and leaves them in LDS for the others (125 tokens,
// 5120 -> 27648, each wavefront its own: 14 % longer).
//
// A K tile takes a wavefront less time than a load from HBM: codes and x are asked for three tiles ahead.  The loads to LDS are
// inline assembly, because the compiler would end them before any read of LDS; not knowing of them it waits for codes somewhat
// earlier than it has to, one reason for the third tile.
//
// Bound by vector instructions (making operands of codes, the groups' factors), matrix instructions and the operand reads of x from LDS, none of
// which fills its unit: 125 tokens, 5120 -> 27648, groups of 128: 55.7 us for 35.4 GFLOP, 635 TFLOP/s, launch after launch
// (62.7 among a layer's others in ten passes after a pause).
template <int DT, int MT, int NT, int WN, int STEPS>
__global__ __launch_bounds__(64 * W4_WAVES, 2) void w4_wide_kernel(const W4Args p)
{
    constexpr int WK = W4_WAVES / WN, BUFS = 4, AHEAD = 3;
    constexpr int XS = 4 * MT / WN, SUMS = 4 / (STEPS < XS ? STEPS : XS);    // K steps whose x a wavefront adds up, sums of a token and K tile
    static_assert(XS >= 1 && XS <= 4, "a wavefront adds up x of one token tile");
    constexpr int XTILE = MT * 16 * W4_TK * 2, XLOADS = MT * 4 / WN;     // bytes of x of a K tile, loads of a wavefront for it
    static_assert(XLOADS >= 1, "a wavefront's loads to LDS");
    constexpr int EXCHANGE = (W4_WAVES - WN) * MT * 16 * 17 * 4, RINGS = WK * BUFS * XTILE;
    __shared__ __attribute__((aligned(16))) unsigned char lds[EXCHANGE > RINGS ? EXCHANGE : RINGS];
    const W4Place place = w4_place(p);
    if (place.proj == p.n_proj) return;
    const W4Proj &w = p.pr[place.proj];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, c = lane & 15, q = lane >> 4;
    const int wn = wave & (WN - 1), wk = wave / WN;
    const int nt0 = (int)place.col_block * (WN * NT) + wn * NT, t0 = (int)place.row_block * (MT * 16);
    const unsigned char *codes = w.packed, *groups = w.packed + w.groups_at;
    const int hin = w.hin, k_tiles = w.k_tiles, n_last = w.n_tiles - 1;
    const bool zeros = w.zeros != 0;
    const uint32_t middle = zeros ? 0u : 24u << 16;               // 16 + 8 where no zero points are stored; joined on the way to LDS: a load is
                                                                  // waited for by the first instruction that touches what it brings
    const uint32_t one = DT == DT_F16 ? 0x3c003c00u : 0x3f803f80u;
    const uint4 ones = make_uint4(one, one, one, one);
    const uint32_t mask = widen_mask<DT>();
    constexpr int PER_TILE = 4 / STEPS;
    const unsigned glane = (q / STEPS) * W4_TN + c;

    auto load = [&](W4Tile<NT> &b, int at_kt) {
        const int kt = min(at_kt, k_tiles - 1);                 // past the end: loaded again and not used
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const size_t tile = (size_t)min(nt0 + n, n_last) * k_tiles + kt;        // past the last column tile: that one, and nothing is stored
            const size_t at = tile * (PER_TILE * W4_TN) + glane;
            b.group[n] = zeros ? reinterpret_cast<const uint32_t *>(groups)[at] : reinterpret_cast<const uint16_t *>(groups)[at];
            b.code[n] = ldg16_stream(codes + tile * W4_TILE_BYTES + lane * 16);
        }
    };
    // this wavefront's share of its part's x tile: four rows a load
    const unsigned char *x0 = static_cast<const unsigned char *>(w.x) + (size_t)t0 * hin * 2;
    unsigned char *tiles = lds + wk * (BUFS * XTILE);
    const uint32_t tiles_at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) unsigned char *)tiles;
    __shared__ __attribute__((aligned(16))) float all_factors[W4_WAVES][NT][2][64];
    float (*factors)[2][64] = all_factors[wave];
    __shared__ __attribute__((aligned(16))) float all_sums[WK][2][MT * 16][SUMS];
    float (*sums)[MT * 16][SUMS] = all_sums[wk];
    auto xload = [&](int kt, int buf) {
#pragma unroll
        for (int m = 0; m < XLOADS; m++) {
            const int r = (wn * XLOADS + m) * 4 + q;
            const int k = kt * W4_TK + (c ^ (r & 15)) * 8;
            const unsigned char *src = x0 + ((uint32_t)min(r, p.T - 1 - t0) * (uint32_t)hin + k) * 2;
            if (k >= hin) src = reinterpret_cast<const unsigned char *>(&w4_no_x);
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" :: "s"(tiles_at + buf * XTILE + (wn * XLOADS + m) * 1024), "v"(src) : "memory");
        }
    };

    // operand of K step s: 16 tokens' x from a buffer
    auto x_of = [&](int buf, int m, int s) { return *reinterpret_cast<const uint4 *>(tiles + buf * XTILE + (m * 16 + c) * 256 + ((s * 4 + q) ^ c) * 16); };
    // this wavefront's sums of tile kt's x: every row of a product with ones is the sum, so a lane has its token's
    auto add_up = [&](int buf) {
        const int m = wn * XS / 4, s0 = wn * XS % 4;
        float4_t sum;
#pragma unroll
        for (int i = 0; i < XS; i++) {
            sum = mfma16<DT>(ones, x_of(buf, m, s0 + i), i % STEPS ? sum : float4_t{0.f, 0.f, 0.f, 0.f});
            if ((i + 1) % STEPS == 0 || i == XS - 1) sums[buf & 1][m * 16 + c][(s0 + i) / (STEPS < XS ? STEPS : XS)] = sum[0];
        }
    };

    float4_t out[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int n = 0; n < NT; n++) out[m][n] = float4_t{0.f, 0.f, 0.f, 0.f};
    // tile kt from buffer `buf`
    auto multiply = [&](const W4Tile<NT> &b, W4Tile<NT> &ahead, int kt, int buf) {
        load(ahead, kt + 3 * WK);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < NT; n++) w4_factors<DT>(factors[n], lane, b.group[n] | middle);
        __builtin_amdgcn_wave_barrier();
        add_up((buf + 1) % BUFS);
        float4_t acc[MT][NT];
#pragma unroll
        for (int s = 0; s < 4; s++) {
            const bool begins = s % STEPS == 0, ends = (s + 1) % STEPS == 0;      // of a group
            const float4_t none = {0.f, 0.f, 0.f, 0.f};
            uint4 x[MT];
#pragma unroll
            for (int m = 0; m < MT; m++) x[m] = x_of(buf, m, s);
            float4_t f[NT], z[NT];
            float sum[MT];
            if (ends) {
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    f[n] = *reinterpret_cast<const float4_t *>(&factors[n][0][s / STEPS * STEPS * 16 + q * 4]);
                    z[n] = *reinterpret_cast<const float4_t *>(&factors[n][1][s / STEPS * STEPS * 16 + q * 4]);
                }
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    const float *of = sums[buf & 1][m * 16 + c];
                    sum[m] = STEPS > XS ? of[0] + of[SUMS - 1] : of[s / STEPS];
                }
            }
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const uint4 a = widen<DT>(s == 0 ? b.code[n].x : s == 1 ? b.code[n].y : s == 2 ? b.code[n].z : b.code[n].w, mask);
#pragma unroll
                for (int m = 0; m < MT; m++) acc[m][n] = mfma16<DT>(a, x[m], begins ? none : acc[m][n]);
            }
            if (ends) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int m = 0; m < MT; m++)
#pragma unroll
                        for (int i = 0; i < 4; i++) out[m][n][i] = fmaf(z[n][i], sum[m], fmaf(f[n][i], acc[m][n][i], out[m][n][i]));
            }
            if constexpr (MT > 2) __builtin_amdgcn_sched_barrier(0);      // or the steps' operands are all made at once and the registers run out
        }
        // behind this tile's products: before them it would be among the loads that the compiler counts as codes, and some of those would be waited for
        __builtin_amdgcn_sched_barrier(0);
        xload(kt + AHEAD * WK, (buf + AHEAD) % BUFS);
        // x of the tile after the next, asked for a tile ago: behind it came this tile's loads of codes, groups and x
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" :: "n"(2 * NT + XLOADS) : "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    };
    W4Tile<NT> b0, b1, b2, b3;
    // all parts pass the same barriers: where one has no last tile it multiplies by zeros, x being past the last column
    load(b0, wk);
    __builtin_amdgcn_sched_barrier(0);
    xload(wk, 0);
    __builtin_amdgcn_sched_barrier(0);
    load(b1, wk + WK);
    __builtin_amdgcn_sched_barrier(0);
    xload(wk + WK, 1);
    __builtin_amdgcn_sched_barrier(0);
    load(b2, wk + 2 * WK);
    __builtin_amdgcn_sched_barrier(0);
    xload(wk + 2 * WK, 2);
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(%0)" :: "n"(2 * NT + XLOADS) : "memory");      // x of the first two tiles
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    add_up(0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll 1
    for (int kt = wk, left = (k_tiles + WK - 1) / WK;;) {
        multiply(b0, b3, kt, 0);
        kt += WK;
        if (--left == 0) break;
        multiply(b1, b0, kt, 1);
        kt += WK;
        if (--left == 0) break;
        multiply(b2, b1, kt, 2);
        kt += WK;
        if (--left == 0) break;
        multiply(b3, b2, kt, 3);
        kt += WK;
        if (--left == 0) break;
    }
    __builtin_amdgcn_s_waitcnt(0);                                // loads to the ring may still be on their way
    // the parts' sums, one column tile of each wavefront at a time
    float (*part)[MT * 16][17] = reinterpret_cast<float (*)[MT * 16][17]>(lds);
    static_assert(MT * NT * 4 <= 32, "a bit for each of a lane's results");
    uint32_t again = 0;                                           // bit 4 (n MT + m) + i: this lane's i-th result of column tile n and token tile m
#pragma unroll
    for (int n = 0; n < NT; n++) {
        if constexpr (WK > 1) {
            __syncthreads();
            if (wk) {
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int i = 0; i < 4; i++) part[wave - WN][m * 16 + c][q * 4 + i] = out[m][n][i];
            }
            __syncthreads();
            if (wk) continue;
#pragma unroll
            for (int k = 1; k < WK; k++)
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int i = 0; i < 4; i++) out[m][n][i] += part[(k - 1) * WN + wn][m * 16 + c][q * 4 + i];
        }
        const int col = (nt0 + n) * W4_TN + q * 4;
#pragma unroll
        for (int m = 0; m < MT; m++) {
            const int r = t0 + m * 16 + c;
            if (r >= p.T || col >= w.hout) continue;
            uint2 *y = reinterpret_cast<uint2 *>(static_cast<uint16_t *>(w.y) + (size_t)r * w.hout + col);
            float4_t v = out[m][n];
            uint32_t bad = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) bad |= (w4_finite(v[i]) ? 0u : 1u) << i;
            again |= bad << 4 * (n * MT + m);
            if (p.accumulate) {                                   // what is computed again finds y as it was
                const uint2 word = *y;
                const float4_t old = {lo_f32<DT>(word.x), hi_f32<DT>(word.x), lo_f32<DT>(word.y), hi_f32<DT>(word.y)};
#pragma unroll
                for (int i = 0; i < 4; i++) v[i] = bad >> i & 1 ? old[i] : v[i] + old[i];
            }
            *y = make_uint2(pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]));
        }
    }
    w4_again<DT>(w, p.accumulate, again, [&](int from, int bit, int &t, int &n) {
        t = t0 + (bit / 4 % MT) * 16 + (from & 15);
        n = (nt0 + bit / 4 / MT) * W4_TN + (from >> 4) * 4 + (bit & 3);
    });
}

// ------------------------------------------------------------------ launches
// Numbers the column blocks of `cols` column tiles, and gives the workgroups of `rows` tokens each.
static unsigned w4_blocks(W4Args &a, int cols, int rows)
{
    unsigned end = 0;
    for (int p = 0; p < a.n_proj; p++) {
        end += (unsigned)((a.pr[p].n_tiles + cols - 1) / cols);
        a.pr[p].end = end;
    }
    a.row_blocks = (unsigned)((a.T + rows - 1) / rows);
    return end * a.row_blocks;
}

static dim3 w4_grid(const W4Args &a) { return dim3((a.pr[a.n_proj - 1].end + 7) / 8 * 8 * a.row_blocks); }

template <int DT, int NT, int STEPS>
static void gemv_of(W4Args &a, hipStream_t s)
{
    w4_blocks(a, NT, 16);
    hipLaunchKernelGGL((w4_gemv_kernel<DT, NT, STEPS>), w4_grid(a), dim3(64 * W4_WAVES), 0, s, a);
}

template <int DT, int MT, int NT, int WN, int STEPS>
static void wide_of(W4Args &a, hipStream_t s)
{
    w4_blocks(a, WN * NT, MT * 16);
    hipLaunchKernelGGL((w4_wide_kernel<DT, MT, NT, WN, STEPS>), w4_grid(a), dim3(64 * W4_WAVES), 0, s, a);
}

// The forms for more than 16 tokens: columns (in tiles) and tokens of a workgroup, and what a launch of them takes (tenths of a microsecond,
// 5120 rows, groups of 128; it grows with the rows alike) where the busiest compute unit has one workgroup, or w: base + w each.  A form with room
// for two on a unit takes less than twice as long for two.
struct W4Form { int cols, rows, alone, base, each; };
constexpr W4Form W4_FORMS[] = {{2, 16, 89, 34, 55}, {2, 32, 123, 20, 103}, {4, 32, 178, 30, 104}, {8, 32, 242, 30, 165}, {8, 64, 318, 20, 295}, {16, 64, 540, 20, 520}};

// Up to 16 tokens: one column tile a workgroup while that makes one round of workgroups, two beyond (one token, 4096 -> 4096: 4.6 us against 5.7;
// 4096 -> 22016: 15.9 against 13.2).  Beyond: the form of the least time by the table.  Against all six at 216 sizes (20 to 512 tokens, 1024 to 13824
// rows, 1024 to 27648 columns) it is the fastest at 192 and 0.6 % behind in the mean; all but twelve are within 3 %, and these have 1024 rows and take
// up to 1.5 us longer, 512 tokens, 1024 -> 27648, 10 (69 for 59).  Some sizes (us, the forms in the table's order, weights from HBM):
//     32 tokens,  4096 ->  4096      8.1    10.4    13.0    19.2    24.7    42.9
//     64          4096 ->  4096     12.5    10.7    13.1    19.1    25.4    43.4
//     32          5120 -> 15360     26.7    23.8    17.5    24.8    31.0    52.9
//    200          5120 -> 27648    234.9   233.9   132.2   103.8   124.7   108.7
//    125          5120 -> 15360     81.6    81.9    44.0    36.3    35.0    54.1
//    125          5120 -> 27648    144.1   142.0    78.2    69.6    63.4    55.7
// With groups of 64 or 32 the accumulators and factors of the last three leave less room for workgroups (125 tokens, 5120 -> 15360, groups of
// 64: 45.7 with the fourth, 45.9 with the third): the third is the widest there, at most 11 % behind what others reached.  Of the three, at the same 216
// sizes with groups of 64 and again of 32, the table's choice is the fastest at 210, and up to 1.2 us behind at six of 1024 rows.  Groups of 64, and 32:
//     32 tokens,  4096 ->  4096      8.3    11.1    13.3
//    125          5120 -> 15360     85.0    86.4    47.3            84.1    95.8    56.5
template <int DT, int STEPS>
static void gemv_by_size(W4Args a, hipStream_t s)
{
    const unsigned cus = (unsigned)device_compute_units();
    if (a.T <= 16) {
        if (w4_blocks(a, 1, 16) <= cus) gemv_of<DT, 1, STEPS>(a, s);
        else gemv_of<DT, 2, STEPS>(a, s);
        return;
    }
    int best = 0;
    unsigned least = ~0u;
    for (int i = 0; i < (STEPS == 4 ? 6 : 3); i++) {
        const W4Form &f = W4_FORMS[i];
        const unsigned w = (w4_blocks(a, f.cols, f.rows) + cus - 1) / cus, time = w == 1 ? f.alone : f.base + f.each * w;
        if (time < least) { least = time; best = i; }
    }
    if (best == 0) gemv_of<DT, 2, STEPS>(a, s);
    else if (best == 1) wide_of<DT, 2, 1, 2, STEPS>(a, s);
    else if (best == 2) wide_of<DT, 2, 1, 4, STEPS>(a, s);
    if constexpr (STEPS == 4) {
        if (best == 3) wide_of<DT, 2, 2, 4, STEPS>(a, s);
        else if (best == 4) wide_of<DT, 4, 2, 4, STEPS>(a, s);
        else if (best == 5) wide_of<DT, 4, 2, 8, STEPS>(a, s);
    }
}

template <int DT>
static void gemv_by_group(const W4Args &all, hipStream_t s)
{
    for (int per_tile = 1; per_tile <= 4; per_tile *= 2) {        // a call's projections usually have one group size
        W4Args a = all;
        a.n_proj = 0;
        for (int p = 0; p < all.n_proj; p++)
            if (all.pr[p].per_tile == per_tile) a.pr[a.n_proj++] = all.pr[p];
        if (a.n_proj == 0) continue;
        if (per_tile == 1) gemv_by_size<DT, 4>(a, s);
        else if (per_tile == 2) gemv_by_size<DT, 2>(a, s);
        else gemv_by_size<DT, 1>(a, s);
    }
}

int launch_w4_gemv(const W4Args &all, int dtype, hipStream_t s)
{
    // A launch has fewer than 2^32 threads.  The form with the most workgroups has one for 32 columns and 16 tokens, and up to eight column blocks
    // more to fill a row of XCDs: so many tokens each (whole token blocks of every form, where it is more than one).
    int64_t cols = 8;
    for (int p = 0; p < all.n_proj; p++) cols += (all.pr[p].n_tiles + 1) / 2;
    const int64_t blocks = ((1LL << 32) / (64 * W4_WAVES) - 1) / cols;
    const int each = (int)(blocks >= 1 << 16 ? 1 << 20 : blocks >= 4 ? blocks / 4 * 64 : 16);
    for (int t0 = 0; t0 < all.T; t0 += each) {
        W4Args a = all;
        a.T = all.T - t0 < each ? all.T - t0 : each;
        for (int p = 0; p < a.n_proj; p++) {
            a.pr[p].x = static_cast<const uint16_t *>(a.pr[p].x) + (int64_t)t0 * a.pr[p].hin;
            a.pr[p].y = static_cast<uint16_t *>(a.pr[p].y) + (int64_t)t0 * a.pr[p].hout;
        }
        if (dtype == DT_F16) gemv_by_group<DT_F16>(a, s); else gemv_by_group<DT_BF16>(a, s);
        const int rc = (int)hipGetLastError();
        if (rc) return rc;
    }
    return 0;
}

}  // namespace mlora

// Products of microscaled 4-bit operands:
//     y[t][n] = (accumulate ? y[t][n] : 0) + sum_b 2^(X_x[t][b] + X_w[n][b]) * sum_{k in block b} cx[t][k] * cw[n][k]
// on the scaled 4-bit matrix instructions, which take the two powers of two of every 32 elements beside the codes.  Running sums in fp32, rounded once.  A block's sum
// is exact; an instruction adds its blocks' sums to the running sum as fixed-point numbers, cut off below 2^-23 of the largest product or sum among them (measured: 1
// beside products of +-6 * 2^23 that cancel is lost).  16 x 16 x 128 so makes six cuts for 128 columns, 32 x 32 x 64 two times four; partial sums that
// wavefronts hold are added in fp32.
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

// ------------------------------------------------------------------ few tokens
// 16 NT columns x 16 MT tokens a workgroup, operands straight from global memory to registers: a packed tile is what a wavefront's lanes hold, 1 KB in one
// load.  The eight wavefronts take the quads of K tiles in turn, each asking for a quad's tiles at once, and add their sums through LDS in their order.
constexpr int MX_WAVES = 8;

template <int DT, int MT, int NT>
__global__ __launch_bounds__(64 * MX_WAVES) void mx4_slim_kernel(const Mx4Args p)
{
    __shared__ float4_t sums[MX_WAVES][NT * MT][64];
    int proj = 0;
    while (proj + 1 < p.n_proj && blockIdx.x >= p.pr[proj].end) proj++;
    const Mx4Proj &w = p.pr[proj];
    const int nt = (int)(blockIdx.x - (proj ? p.pr[proj - 1].end : 0u)) * NT, tt = ((int)blockIdx.y + p.first) * MT;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int n_tiles = (w.hout + 15) / 16, t_tiles = (p.T + 15) / 16, k_tiles = w.k_tiles, quads = w.quads;
    const bool row_in = tt * 16 + (lane & 15) < p.T;
    // tiles past the operands' last are read as the last: what they produce is not stored
    const unsigned char *wc[NT], *ws[NT], *xc[MT], *xs[MT];
#pragma unroll
    for (int i = 0; i < NT; i++) {
        const int r = nt + i < n_tiles ? nt + i : n_tiles - 1;
        wc[i] = w.w + (size_t)r * k_tiles * MX4_TILE_BYTES;
        ws[i] = w.w + w.w_scales_at + (size_t)r * quads * MX4_QUAD_BYTES;
    }
#pragma unroll
    for (int j = 0; j < MT; j++) {
        const int r = tt + j < t_tiles ? tt + j : t_tiles - 1;
        xc[j] = w.x + (size_t)r * k_tiles * MX4_TILE_BYTES;
        xs[j] = w.x + w.x_scales_at + (size_t)r * quads * MX4_QUAD_BYTES;
    }
    float4_t acc[NT][MT];
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int j = 0; j < MT; j++) acc[i][j] = float4_t{0.f, 0.f, 0.f, 0.f};
    // Where a wavefront holds more than one tile of each, the next quad's are asked for before this one's are multiplied (64 tokens, 4096 -> 4096: 6.2 -> 5.7 us);
    // with one, twice the registers cost resident workgroups (16 tokens, 5120 -> 2 x 13824: 15.5 -> 18.6 us).  Lanes of rows that x does not have load nothing.
    struct Ops { uint4 a[4][NT], b[4][MT]; uint32_t sa[NT], sb[MT]; } ops[2];
    auto load = [&](Ops &o, int quad) {
#pragma unroll
        for (int u = 0; u < 4; u++) {
            const int kt = quad * 4 + u < k_tiles ? quad * 4 + u : k_tiles - 1;       // past the last: left out below
            const unsigned at = (unsigned)kt * MX4_TILE_BYTES + lane * 16;
#pragma unroll
            for (int i = 0; i < NT; i++) o.a[u][i] = ldg16_stream(wc[i] + at);
#pragma unroll
            for (int j = 0; j < MT; j++) o.b[u][j] = MT > 1 || row_in ? ldg16(xc[j] + at) : zero16();
        }
#pragma unroll
        for (int i = 0; i < NT; i++) o.sa[i] = *reinterpret_cast<const uint32_t *>(ws[i] + (unsigned)quad * MX4_QUAD_BYTES + lane * 4);
#pragma unroll
        for (int j = 0; j < MT; j++) o.sb[j] = *reinterpret_cast<const uint32_t *>(xs[j] + (unsigned)quad * MX4_QUAD_BYTES + lane * 4);
    };
    auto multiply = [&](const Ops &o, int quad) {
        auto tile = [&](auto u_c) {
            constexpr int u = decltype(u_c)::value;
            if (quad * 4 + u >= k_tiles) return;
#pragma unroll
            for (int i = 0; i < NT; i++)
#pragma unroll
                for (int j = 0; j < MT; j++) acc[i][j] = mx4_mfma16<u>(o.a[u][i], o.b[u][j], acc[i][j], o.sa[i], o.sb[j]);
        };
        tile(std::integral_constant<int, 0>{});
        tile(std::integral_constant<int, 1>{});
        tile(std::integral_constant<int, 2>{});
        tile(std::integral_constant<int, 3>{});
    };
    if constexpr (MT * NT == 1) {
        for (int quad = wave; quad < quads; quad += MX_WAVES) {
            load(ops[0], quad);
            multiply(ops[0], quad);
        }
    } else {
        if (wave < quads) load(ops[0], wave);
        for (int quad = wave; quad < quads; quad += 2 * MX_WAVES) {
            if (quad + MX_WAVES < quads) load(ops[1], quad + MX_WAVES);
            multiply(ops[0], quad);
            if (quad + 2 * MX_WAVES < quads) load(ops[0], quad + 2 * MX_WAVES);
            if (quad + MX_WAVES < quads) multiply(ops[1], quad + MX_WAVES);
        }
    }
#pragma unroll
    for (int i = 0; i < NT; i++)
#pragma unroll
        for (int j = 0; j < MT; j++) sums[wave][i * MT + j][lane] = acc[i][j];
    __syncthreads();
    for (int c = wave; c < NT * MT; c += MX_WAVES) {
        const int t = (tt + c % MT) * 16 + (lane & 15), n = (nt + c / MT) * 16 + 4 * (lane >> 4);
        if (t >= p.T || n >= w.hout) continue;
        uint2 *y = reinterpret_cast<uint2 *>(static_cast<uint16_t *>(w.y) + (size_t)t * w.hout + n);
        float4_t v = sums[0][c][lane];
#pragma unroll
        for (int i = 1; i < MX_WAVES; i++) v += sums[i][c][lane];
        if (p.accumulate) {
            const uint2 o = *y;
            v[0] += lo_f32<DT>(o.x); v[1] += hi_f32<DT>(o.x); v[2] += lo_f32<DT>(o.y); v[3] += hi_f32<DT>(o.y);
        }
        *y = make_uint2(pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]));
    }
}

// ------------------------------------------------------------------ tiles for many tokens
// One workgroup (256 threads, 2 x 2 wavefronts of 32 WI columns x 32 XI tokens) computes 64 WI columns x 64 XI tokens on the 32 x 32 x 64 form of the
// instruction, the weight's rows its first operand, so that a lane's results are four neighbouring columns of one token.  K advances a tile of 128 columns
// a step through a ring of four LDS stages that global memory fills directly, 1 KB a load: a packed tile is what a wavefront's lanes read,
// sixteen bytes each, without bank conflicts and without a swizzle.  The scales of a quad of steps come the same way into a ring of two, and
// go to registers once a quad: the instruction picks its byte.
constexpr int MX_NT = 256, MX_RING = 4;
typedef int i32x4_vec __attribute__((ext_vector_type(4)));

template <int J>
__device__ __forceinline__ float16_t mx4_mfma32(const uint4 &a, const uint4 &b, float16_t c, uint32_t sa, uint32_t sb)
{
    const int8_vec va = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0}, vb = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(va, vb, c, 4, 4, J, (int)sa, J, (int)sb);
}

template <int WI, int XI> constexpr int mx4_stage_bytes() { return 4 * (WI + XI) * MX4_TILE_BYTES; }
template <int WI, int XI> constexpr int mx4_ring_bytes() { return MX_RING * mx4_stage_bytes<WI, XI>() + 2 * 4 * (WI + XI) * MX4_QUAD_BYTES; }

// Columns 64 WI nt .. and tokens 64 XI tt .. of one product.
template <int DT, int WI, int XI, int KS, bool ACC>
__device__ __forceinline__ void mx4_tile(const Mx4Args &p, const Mx4Proj &w, int nt, int tt, unsigned char *const all_rings)
{
    constexpr int STAGE = mx4_stage_bytes<WI, XI>(), SSTAGE = 4 * (WI + XI) * MX4_QUAD_BYTES, NL = WI + XI;
    constexpr int RINGS = mx4_ring_bytes<WI, XI>();
    static_assert(KS * RINGS <= 160 * 1024, "the rings must fit the LDS of a compute unit");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6) & 3);
    const int part = KS == 1 ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x / MX_NT);
    const int wm = wave >> 1, wn = wave & 1, l32 = lane & 31, lh = lane >> 5;
    unsigned char *const lds = all_rings + part * RINGS, *const scale_ring = lds + MX_RING * STAGE;
    // the group's quads; all groups of a workgroup make as many steps, over zeros past the operands' end
    const int per = KS == 1 ? w.quads : (w.quads + KS - 1) / KS, quad0 = part * per;
    const int ns = KS == 1 ? w.k_tiles : 4 * per, have_quads = KS == 1 ? w.quads : min(per, w.quads - quad0), have = KS == 1 ? w.k_tiles : min(ns, w.k_tiles - 4 * quad0);

    // Row tiles past the operand's last are read as the last: what they produce is not stored.
    const int w_tiles = (w.hout + 15) / 16 - nt * 4 * WI, x_tiles = (p.T + 15) / 16 - tt * 4 * XI;      // of this block on, may be more than it has
    const unsigned row_codes = (unsigned)w.k_tiles * MX4_TILE_BYTES, row_scales = (unsigned)w.quads * MX4_QUAD_BYTES;
    auto rsrc = [](const unsigned char *from, size_t bytes) {
        const unsigned long long a = (unsigned long long)from;
        const i32x4_vec r = {(int)(unsigned)a, (int)((a >> 32) & 0xffffu), (int)(bytes < 0xffffffffu ? bytes : 0xffffffffu), 0x00020000};
        return r;
    };
    const int w_have = w_tiles < 4 * WI ? w_tiles : 4 * WI, x_have = x_tiles < 4 * XI ? x_tiles : 4 * XI;
    const i32x4_vec wr = rsrc(w.w + (size_t)nt * 4 * WI * row_codes, (size_t)w_have * row_codes), xr = rsrc(w.x + (size_t)tt * 4 * XI * row_codes, (size_t)x_have * row_codes);
    const i32x4_vec wsr = rsrc(w.w + w.w_scales_at + (size_t)nt * 4 * WI * row_scales, (size_t)w_have * row_scales);
    const i32x4_vec xsr = rsrc(w.x + w.x_scales_at + (size_t)tt * 4 * XI * row_scales, (size_t)x_have * row_scales);
    // Loads into LDS are assembly: the compiler waits for all its own before any LDS read that follows; here the waits are explicit.  M0, which
    // carries the LDS address, is written by nothing else in this kernel (the build-time check sees to it).
    typedef __attribute__((address_space(3))) unsigned char lds_byte;
    auto dma = [](const i32x4_vec &rs, unsigned to, unsigned voff, unsigned soff) {
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" :: "s"(to), "v"(voff), "s"(rs), "s"(soff) : "memory");
    };
    const unsigned ring_at = (unsigned)(__UINTPTR_TYPE__)(lds_byte *)lds, scales_at = ring_at + MX_RING * STAGE;
    const unsigned code_lane = (unsigned)lane * 16u;
    unsigned w_off[WI], x_off[XI];                       // this wavefront's row tiles: wave, wave + 4, ..
#pragma unroll
    for (int q = 0; q < WI; q++) w_off[q] = (unsigned)(4 * q + wave < w_have ? 4 * q + wave : w_have - 1) * row_codes;
#pragma unroll
    for (int q = 0; q < XI; q++) x_off[q] = (unsigned)(4 * q + wave < x_have ? 4 * q + wave : x_have - 1) * row_codes;
    // a scales' load covers four row tiles; every wavefront makes one of each operand, some of them twice
    const int sg_w = wave % WI, sg_x = wave % XI, sw_row = 4 * sg_w + (lane >> 4), sx_row = 4 * sg_x + (lane >> 4);
    const unsigned sw_lane = (unsigned)(sw_row < w_have ? sw_row : w_have - 1) * row_scales + (lane & 15) * 16u;
    const unsigned sx_lane = (unsigned)(sx_row < x_have ? sx_row : x_have - 1) * row_scales + (lane & 15) * 16u;
    // Steps and quads past the last are asked for all the same, so that every step counts its loads alike: outside the descriptors, where nothing is
    // fetched and zeros arrive that nobody reads.
    constexpr unsigned NOWHERE = 0xfffffff0u;
    auto dma_code = [&](int q, int slot, unsigned from_lane, int ks) {
        const unsigned to = ring_at + slot * STAGE + (q < WI ? 4 * q + wave : 4 * WI + 4 * (q - WI) + wave) * MX4_TILE_BYTES;
        if (q < WI) dma(wr, to, from_lane, w_off[q < WI ? q : 0] + (unsigned)(4 * quad0 + ks) * MX4_TILE_BYTES);
        else dma(xr, to, from_lane, x_off[q < WI ? 0 : q - WI] + (unsigned)(4 * quad0 + ks) * MX4_TILE_BYTES);
    };
    auto dma_scales = [&](int quad) {
        const unsigned to = scales_at + (quad & 1) * SSTAGE;
        dma(wsr, to + sg_w * 1024, quad < have_quads ? sw_lane : NOWHERE, (unsigned)(quad0 + quad) * MX4_QUAD_BYTES);
        dma(xsr, to + (WI + sg_x) * 1024, quad < have_quads ? sx_lane : NOWHERE, (unsigned)(quad0 + quad) * MX4_QUAD_BYTES);
    };

    // Operand addresses in a stage: lane (row l32, half lh) of 32-row block i and slice kk reads block 2 kk + lh of its row.
    const unsigned w_at = wm * (2 * WI * MX4_TILE_BYTES) + (l32 >> 4) * MX4_TILE_BYTES + lh * 256 + (l32 & 15) * 16;
    const unsigned x_at = (4 * WI + wn * 2 * XI) * MX4_TILE_BYTES + (l32 >> 4) * MX4_TILE_BYTES + lh * 256 + (l32 & 15) * 16;
    const unsigned ws_at = wm * (2 * WI * MX4_QUAD_BYTES) + (l32 >> 4) * MX4_QUAD_BYTES + lh * 64 + (l32 & 15) * 4;
    const unsigned xs_at = (4 * WI + wn * 2 * XI) * MX4_QUAD_BYTES + (l32 >> 4) * MX4_QUAD_BYTES + lh * 64 + (l32 & 15) * 4;

    float16_t acc[WI][XI];
#pragma unroll
    for (int i = 0; i < WI; i++)
#pragma unroll
        for (int j = 0; j < XI; j++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[i][j][e] = 0.f;
    uint4 fw[2][WI], fx[2][XI];                          // operands of a slice, read one slice ahead
    uint32_t sw[2][WI], sx[2][XI];                       // scales of the quad, by slice
    auto read_op = [&](const unsigned char *stage, int kk, int t) {
        if (t < WI) fw[kk][t < WI ? t : 0] = *reinterpret_cast<const uint4 *>(stage + w_at + kk * 512 + t * 2 * MX4_TILE_BYTES);
        else fx[kk][t < WI ? 0 : t - WI] = *reinterpret_cast<const uint4 *>(stage + x_at + kk * 512 + (t - WI) * 2 * MX4_TILE_BYTES);
    };
    auto read_scales = [&](int quad, uint32_t (&a)[2][WI], uint32_t (&b)[2][XI]) {
        const unsigned char *s = scale_ring + (quad & 1) * SSTAGE;
#pragma unroll
        for (int kk = 0; kk < 2; kk++) {
#pragma unroll
            for (int i = 0; i < WI; i++) a[kk][i] = *reinterpret_cast<const uint32_t *>(s + ws_at + kk * 128 + i * 2 * MX4_QUAD_BYTES);
#pragma unroll
            for (int j = 0; j < XI; j++) b[kk][j] = *reinterpret_cast<const uint32_t *>(s + xs_at + kk * 128 + j * 2 * MX4_QUAD_BYTES);
        }
    };
#define MX_FENCE() __builtin_amdgcn_sched_barrier(0)
#define MX_WAIT_LOADS(n) __builtin_amdgcn_s_waitcnt(0x0f70 | ((n) & 15) | (((n) >> 4) << 14))
    constexpr int NM = WI * XI;
    // Step ks = 4 quad + J.  Between its slices: the loads of step ks + 1 have landed, for every wavefront, and everyone has read this step's stage, which
    // then takes step ks + 4.  In flight at that wait: steps ks + 2 and ks + 3, and in steps 1 and 2 of a quad the next quad's scales.
    auto step = [&](auto j_c, int ks) {
        constexpr int J = decltype(j_c)::value;
        const unsigned char *here = lds + J * STAGE, *next = lds + ((J + 1) & 3) * STAGE;
        const unsigned from_lane = ks + 4 < have ? code_lane : NOWHERE;
#pragma unroll
        for (int n = 0; n < NM; n++) {
#pragma unroll
            for (int t = n * NL / NM; t < (n + 1) * NL / NM; t++) read_op(here, 1, t);
            acc[n / XI][n % XI] = mx4_mfma32<J>(fw[0][n / XI], fx[0][n % XI], acc[n / XI][n % XI], sw[0][n / XI], sx[0][n % XI]);
            MX_FENCE();
        }
        MX_WAIT_LOADS(J == 1 || J == 2 ? 2 * NL + 2 : 2 * NL);
        __syncthreads();
        uint32_t nsw[2][WI], nsx[2][XI];
        if (J == 0) dma_scales((ks >> 2) + 1);
        if (J == 3) read_scales((ks >> 2) + 1, nsw, nsx);
#pragma unroll
        for (int n = 0; n < NM; n++) {
#pragma unroll
            for (int t = n * NL / NM; t < (n + 1) * NL / NM; t++) read_op(next, 0, t);
            acc[n / XI][n % XI] = mx4_mfma32<J>(fw[1][n / XI], fx[1][n % XI], acc[n / XI][n % XI], sw[1][n / XI], sx[1][n % XI]);
#pragma unroll
            for (int t = n * NL / NM; t < (n + 1) * NL / NM; t++) dma_code(t, J, from_lane, ks + 4);
            MX_FENCE();
        }
        if (J == 3) {
#pragma unroll
            for (int kk = 0; kk < 2; kk++) {
#pragma unroll
                for (int i = 0; i < WI; i++) sw[kk][i] = nsw[kk][i];
#pragma unroll
                for (int j = 0; j < XI; j++) sx[kk][j] = nsx[kk][j];
            }
        }
    };
    using S0 = std::integral_constant<int, 0>;
    using S1 = std::integral_constant<int, 1>;
    using S2 = std::integral_constant<int, 2>;
    using S3 = std::integral_constant<int, 3>;

    dma_scales(0);
#pragma unroll
    for (int s = 0; s < MX_RING; s++)
#pragma unroll
        for (int q = 0; q < NL; q++) dma_code(q, s, s < have ? code_lane : NOWHERE, s);
    MX_WAIT_LOADS(3 * NL);
    __syncthreads();
    read_scales(0, sw, sx);
#pragma unroll
    for (int t = 0; t < NL; t++) read_op(lds, 0, t);
    int ks = 0;
#pragma unroll 1
    for (; ks + 4 <= ns; ks += 4) {
        step(S0{}, ks);
        step(S1{}, ks + 1);
        step(S2{}, ks + 2);
        step(S3{}, ks + 3);
    }
    if (KS == 1 && ks < ns) {
        step(S0{}, ks);
        if (ks + 1 < ns) step(S1{}, ks + 1);
        if (ks + 2 < ns) step(S2{}, ks + 2);
    }
    MX_WAIT_LOADS(0);
#undef MX_FENCE
#undef MX_WAIT_LOADS
    __syncthreads();                                     // the rings are free
    if constexpr (KS > 1) {
        constexpr int SUMS = WI * XI * 4096;                 // bytes of a wavefront's accumulators
        constexpr int STAGING = 4 * 32 * (64 * WI + 16);     // of the results below, which other wavefronts may have come to
        static_assert(STAGING + (KS - 1) * 4 * SUMS <= KS * RINGS, "the sums reuse the rings");
        float4_t *const sums = reinterpret_cast<float4_t *>(all_rings + STAGING + wave * SUMS) + lane;
        if (part > 0) {
#pragma unroll
            for (int i = 0; i < WI * XI * 4; i++) {
                const float16_t &a = acc[i / 4 / XI][i / 4 % XI];
                sums[(part - 1) * (SUMS / 4) + i * 64] = float4_t{a[i % 4 * 4], a[i % 4 * 4 + 1], a[i % 4 * 4 + 2], a[i % 4 * 4 + 3]};
            }
        }
        __syncthreads();
        if (part > 0) return;
#pragma unroll
        for (int g = 0; g < KS - 1; g++)
#pragma unroll
            for (int i = 0; i < WI * XI * 4; i++) {
                const float4_t s = sums[g * (SUMS / 4) + i * 64];
#pragma unroll
                for (int e = 0; e < 4; e++) acc[i / 4 / XI][i / 4 % XI][i % 4 * 4 + e] += s[e];
            }
    }

    // Results leave by way of LDS, 32 tokens at a time a wavefront, so that a store covers 64 WI bytes of a token.  No branch between the reads of the
    // accumulators: at the first one the compiler would move all of them to registers that are not there.  What lies outside y goes to NOWHERE.
    constexpr int PITCH = 64 * WI + 16, CHUNKS = 4 * WI;
    static_assert(4 * 32 * PITCH <= MX_RING * STAGE, "the staging tiles reuse the ring");
    unsigned char *const out = lds + wave * 32 * PITCH;
    // the lane once more, from the hardware: not kept in a register through the loop
    int ol = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u));
    asm volatile("" : "+v"(ol));
    const int o32 = ol & 31, oh = ol >> 5;
    const int n0 = nt * 64 * WI + wm * 32 * WI, t0 = tt * 64 * XI + wn * 32 * XI;
#pragma unroll
    for (int j = 0; j < XI; j++) {
        const int tj = t0 + 32 * j;                  // 32 rows of up to 2^25 bytes: 32-bit offsets
        const __amdgpu_buffer_rsrc_t yr = __builtin_amdgcn_make_buffer_rsrc(static_cast<uint16_t *>(w.y) + (size_t)tj * w.hout, (short)0, (int)0x7ffffff0, 0x00020000);
#pragma unroll
        for (int i = 0; i < WI; i++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = acc[i][j][4 * g + e];
                if constexpr (ACC) {
                    const int n = n0 + 32 * i + 8 * g + 4 * oh;
                    typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
                    const u32x2 o = __builtin_amdgcn_raw_buffer_load_b64(yr, n < w.hout && tj + o32 < p.T ? (int)(((unsigned)o32 * (unsigned)w.hout + n) * 2u) : (int)NOWHERE, 0, 0);
                    v[0] += lo_f32<DT>(o.x); v[1] += hi_f32<DT>(o.x); v[2] += lo_f32<DT>(o.y); v[3] += hi_f32<DT>(o.y);
                }
                *reinterpret_cast<uint2 *>(out + o32 * PITCH + (32 * i + 8 * g + 4 * oh) * 2) = make_uint2(pack2<DT>(v[0], v[1]), pack2<DT>(v[2], v[3]));
                __builtin_amdgcn_sched_barrier(0);
            }
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int c = 0; c < 32 * CHUNKS / 64; c++) {
            const int idx = c * 64 + ol, row = idx / CHUNKS, n = n0 + (idx % CHUNKS) * 8;
            const uint4 v = *reinterpret_cast<const uint4 *>(out + row * PITCH + (idx % CHUNKS) * 16);
            const u32x4_t s = {v.x, v.y, v.z, v.w};
            __builtin_amdgcn_raw_buffer_store_b128(s, yr, n < w.hout && tj + row < p.T ? (int)(((unsigned)row * (unsigned)w.hout + n) * 2u) : (int)NOWHERE, 0, 0);
        }
        __builtin_amdgcn_wave_barrier();
    }
}

// Workgroups go to the 8 XCDs round-robin by id: the id-th of n workgroups takes tile number L of n, so that every XCD works through one contiguous range of them.
__device__ __forceinline__ int mx4_spread(int id, int n)
{
    const int base = n >> 3, more = n & 7, xcd = id & 7;
    return xcd * base + (xcd < more ? xcd : more) + (id >> 3);
}

// Tile number L of a call: GROUP token tiles sweep a product's column tiles together, so that what is in flight on one XCD shares its panels in that L2.
struct Mx4Place { int proj, nt, tt; };
template <int WI, int XI>
__device__ __forceinline__ Mx4Place mx4_place(const Mx4Args &p, int L)
{
    constexpr int GROUP = 4;
    int proj = 0;
    while (proj + 1 < p.n_proj && (unsigned)L >= p.pr[proj].end) proj++;
    if (proj) L -= (int)p.pr[proj - 1].end;
    const int ntn = (p.pr[proj].hout + 64 * WI - 1) / (64 * WI), ntt = (p.T + 64 * XI - 1) / (64 * XI);
    const int grp = L / (GROUP * ntn), within = L - grp * (GROUP * ntn);
    const int in_grp = ntt - grp * GROUP < GROUP ? ntt - grp * GROUP : GROUP;
    return {proj, within / in_grp, grp * GROUP + within % in_grp};
}

template <int DT, int WI, int XI, int KS, bool ACC>
__global__ __launch_bounds__(MX_NT * KS) void mx4_tile_kernel(const Mx4Args p)
{
    __shared__ __attribute__((aligned(16))) unsigned char rings[KS * mx4_ring_bytes<WI, XI>()];
    const Mx4Place at = mx4_place<WI, XI>(p, mx4_spread((int)blockIdx.x, (int)gridDim.x));
    mx4_tile<DT, WI, XI, KS, ACC>(p, p.pr[at.proj], at.nt, at.tt, rings);
}

// Tiles of 256 x 256, the first `whole` of them whole, and the others, which would be half a round of workgroups or less, as halves of 128 tokens (8000 tokens,
// 13824 -> 5120, 2.5 rounds: 264 -> 240 us; 5120 -> 2 x 13824, 13.5 rounds: 552 -> 530).
//
// What bounds it: its steps, and the time between tiles.  A step of a whole tile is 128 matrix instructions, 1024 cycles of each pipe.  On one unit alone it takes
// 500 ns, 0.86 of the pipes' rate at 2.4 GHz (a barrier a step and one wavefront a pipe); with all units at work 795 to 850, where the instructions alone,
// from registers and on random numbers, take 700 (5.9 to 6.4 PFLOP/s; on ones up to 9.4): the card lowers its clock to 1.7 GHz.  Besides the steps a
// round of tiles takes 7 to 10 us in which the pipes have nothing (the ring's filling, the results' way out; one workgroup a unit, so nothing runs beside it): of
// 1225 us for a Llama-13B layer at 8000 tokens, 26 rounds, the steps are 962 and this is 263.  64 rows of either operand in LDS for every 32 read
// feed the pipes at half of the LDS' rate; 128 x 128 tiles need all of it and run at 1.5 GHz.
//
// Accumulating, y is read eight bytes a lane between the writes to LDS: 8000 tokens, 4096 -> 2 x 11008 360 -> 479 us, 13824 -> 5120 246 -> 266; 64 tokens 13.0 -> 14.1
// and 16.3 -> 16.7.
template <int DT, bool ACC>
__global__ __launch_bounds__(MX_NT) void mx4_halves_kernel(const Mx4Args p)
{
    __shared__ __attribute__((aligned(16))) unsigned char rings[mx4_ring_bytes<4, 4>()];
    const int id = (int)blockIdx.x, whole = (int)p.whole;
    if (id < whole) {
        const Mx4Place at = mx4_place<4, 4>(p, mx4_spread(id, whole));
        mx4_tile<DT, 4, 4, 1, ACC>(p, p.pr[at.proj], at.nt, at.tt, rings);
    } else {
        const int half = mx4_spread(id - whole, (int)gridDim.x - whole);
        const Mx4Place at = mx4_place<4, 4>(p, whole + half / 2);
        const int tt = 2 * at.tt + (half & 1);
        if (tt * 128 < p.T) mx4_tile<DT, 4, 2, 1, ACC>(p, p.pr[at.proj], at.nt, tt, rings);
    }
}

template <int DT, int WI, int XI, int KS>
static int launch_tiles(Mx4Args &a, hipStream_t s)
{
    unsigned end = 0;
    for (int p = 0; p < a.n_proj; p++)
        a.pr[p].end = end += (unsigned)((a.pr[p].hout + 64 * WI - 1) / (64 * WI)) * (unsigned)((a.T + 64 * XI - 1) / (64 * XI));
    if (a.accumulate) hipLaunchKernelGGL((mx4_tile_kernel<DT, WI, XI, KS, true>), dim3(end), dim3(MX_NT * KS), 0, s, a);
    else hipLaunchKernelGGL((mx4_tile_kernel<DT, WI, XI, KS, false>), dim3(end), dim3(MX_NT * KS), 0, s, a);
    return (int)hipGetLastError();
}

template <int DT>
static int launch_halves(Mx4Args &a, hipStream_t s)
{
    unsigned end = 0;
    for (int p = 0; p < a.n_proj; p++) a.pr[p].end = end += (unsigned)((a.pr[p].hout + 255) / 256) * (unsigned)((a.T + 255) / 256);
    const unsigned units = (unsigned)device_compute_units(), rest = end % units;
    a.whole = 2 * rest <= units ? end - rest : end;
    const dim3 grid(a.whole + 2 * (end - a.whole));
    if (a.accumulate) hipLaunchKernelGGL((mx4_halves_kernel<DT, true>), grid, dim3(MX_NT), 0, s, a);
    else hipLaunchKernelGGL((mx4_halves_kernel<DT, false>), grid, dim3(MX_NT), 0, s, a);
    return (int)hipGetLastError();
}

template <int DT, int MT, int NT>
static int launch_slim(Mx4Args &a, hipStream_t s)
{
    unsigned end = 0;
    for (int p = 0; p < a.n_proj; p++) a.pr[p].end = end += (unsigned)(a.pr[p].hout + 16 * NT - 1) / (16 * NT);
    const int rows = (a.T + 16 * MT - 1) / (16 * MT), most = 65535;              // of a grid's second dimension
    int rc = 0;
    for (a.first = 0; a.first < rows && !rc; a.first += most) {
        hipLaunchKernelGGL((mx4_slim_kernel<DT, MT, NT>), dim3(end, (unsigned)(rows - a.first < most ? rows - a.first : most)), dim3(64 * MX_WAVES), 0, s, a);
        rc = (int)hipGetLastError();
    }
    return rc;
}

// ------------------------------------------------------------------ which form
// A form's time: start + round * m + max(step, m * step_full) * K tiles, with m the workgroups of the busiest compute unit (a workgroup alone is bound by the
// way of its operands from memory, several share the unit), but not less than the call's bytes take: where forms are alike then, the one for the fewest tokens
// is taken.  The constants (us) are fitted to times of sixteen calls (one to three products of a whole, half or quarter layer of Llama-7B and 13B) at 1 to 8000
// tokens, each form over the range in which it comes near the fastest; fitted and measured times differ by 6 % (few tokens) to 12 % (tiles) on average.  Measured
// once more with the forms as they are, at 432 sizes, the form with the least time is 0.7 % behind the fastest on average, 8 % or more at
// eight: 24 to 64 tokens, 5120 -> 2 x 13824 (64 columns x 64 tokens, 14 to 21 % behind 128 columns), 384 tokens, 4096 -> 2 x 5504 (256 x 256, 10 % behind 128 x 128), one
// token, 4096 -> 2 x 11008 (32 columns, 10 % behind 16), 192 and 256 tokens, 2752 -> 4096 (64 x 64, 8 % behind 128 x 64).  Examples, with another one:
//      1 token, 4096 -> 4096: 16 columns x 16 tokens 4.4 us, 32 columns 5.0;     64 tokens: 32 x 32 6.0, 32 columns x 64 tokens 7.2
//      64 tokens, 4096 -> 2 x 11008: 128 columns x 64 tokens 12.8, 64 x 64 15.8;  512 tokens: 256 x 256 29.4, 128 x 128 32.6
//      512 tokens, 11008 -> 4096: 128 columns x 64 tokens 23.3, 64 x 64 27.5;     1536 tokens: 256 x 256 in halves 44.5, 128 x 128 41.7
namespace {
struct Mx4Form {
    int columns, tokens;
    float start, round, step, step_full;
    int (*launch[2])(Mx4Args &, hipStream_t);
};
#define MX_FORM(F, ...) {F<DT_F16, __VA_ARGS__>, F<DT_BF16, __VA_ARGS__>}
const Mx4Form mx4_forms[] = {
    {16, 16, 2.7f, 0.0f, 0.052f, 0.044f, MX_FORM(launch_slim, 1, 1)},
    {32, 16, 2.2f, 0.46f, 0.074f, 0.065f, MX_FORM(launch_slim, 1, 2)},
    {16, 32, 2.5f, 0.32f, 0.064f, 0.053f, MX_FORM(launch_slim, 2, 1)},
    {32, 32, 1.9f, 0.92f, 0.091f, 0.084f, MX_FORM(launch_slim, 2, 2)},
    {32, 64, 1.2f, 2.1f, 0.115f, 0.1f, MX_FORM(launch_slim, 4, 2)},
    {64, 64, 3.0f, 0.84f, 0.136f, 0.12f, MX_FORM(launch_tiles, 1, 1, 2)},
    {128, 64, 2.1f, 1.0f, 0.216f, 0.179f, MX_FORM(launch_tiles, 2, 1, 1)},
    {128, 128, 2.4f, 1.2f, 0.0f, 0.25f, MX_FORM(launch_tiles, 2, 2, 1)},
    {256, 256, 0.0f, 7.3f, 0.0f, 0.62f, {launch_halves<DT_F16>, launch_halves<DT_BF16>}},
};

const Mx4Form &mx4_form(const Mx4Args &a)
{
    int steps = 0;
    float bytes = 0.f;
    for (int p = 0; p < a.n_proj; p++) {
        if (a.pr[p].k_tiles > steps) steps = a.pr[p].k_tiles;
        bytes += (float)a.pr[p].hout * ((float)a.pr[p].hin * 0.53f + (float)a.T * 2.f) + (float)a.T * (float)a.pr[p].hin * (p ? 0.f : 0.53f);
    }
    const float memory = 1.6f + bytes / 5.2e6f;
    const int units = device_compute_units();
    const Mx4Form *best = nullptr;
    float least = 0.f;
    for (const Mx4Form &f : mx4_forms) {
        int64_t groups = 0;
        for (int p = 0; p < a.n_proj; p++) groups += (int64_t)((a.pr[p].hout + f.columns - 1) / f.columns) * ((a.T + f.tokens - 1) / f.tokens);
        float m = (float)((groups + units - 1) / units);
        if (f.columns == 256 && groups % units && 2 * (groups % units) <= units) m -= 0.37f;         // a round of halves
        const float each = m * f.step_full > f.step ? m * f.step_full : f.step;
        float time = f.start + f.round * m + each * (float)steps;
        if (time < memory) time = memory;
        if (!best || time < least) { best = &f; least = time; }
    }
    return *best;
}
}  // namespace

void mx4_form(const Mx4Args &a, int *columns, int *tokens)
{
    const Mx4Form &f = mx4_form(a);
    *columns = f.columns;
    *tokens = f.tokens;
}

int launch_mx4_gemm(const Mx4Args &all, int dtype, hipStream_t s)
{
    Mx4Args a = all;
    return mx4_form(a).launch[dtype == DT_F16 ? 0 : 1](a, s);
}

}  // namespace mlora

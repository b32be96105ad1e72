// Kernel argument blocks and launchers of the decode step around the LoRA apply: 4-bit base projections, cache appends,
// shared-prefix attention.
#pragma once
#include <cstdarg>
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace mlora {

constexpr int STEP_MAX_PROJ = 8;

// ---- 4-bit weights.  A packed weight is two planes: codes, and the groups' scales and zero points.
// Codes: tiles of 16 columns x 128 rows, 1024 bytes each, column tile major (a column tile's K tiles lie one behind the other).  In a
// tile, lane l = 16 * q + c of a wavefront owns 16 bytes: dword s holds rows 32 s + 8 q + j (j < 8) of column c, row pair
// (2i, 2i + 1) in nibbles i and i + 4 - the operand of one 16 x 16 x 32 MFMA.  Rows and columns past the weight's are zero codes.
// Groups, tile by tile: [groups of a K tile (1, 2 or 4)][16 columns] of the 16-bit scale, or where there are zero points of a dword
// whose upper half is 16 + the zero point; zeros past the weight's.
constexpr int W4_TN = 16, W4_TK = 128, W4_TILE_BYTES = W4_TN * W4_TK / 2;
struct W4Shape {
    int hin, hout, group;
    int n_tiles, k_tiles, groups, per_tile;    // column tiles, K tiles, groups of a column, groups of a K tile
    int64_t groups_at, bytes;                  // byte offset of the second plane, total
};
inline W4Shape w4_shape(int hin, int hout, int group, bool zeros)
{
    W4Shape s;
    s.hin = hin; s.hout = hout; s.group = group;
    s.n_tiles = (hout + W4_TN - 1) / W4_TN;
    s.k_tiles = (hin + W4_TK - 1) / W4_TK;
    s.groups = (hin + group - 1) / group;
    s.per_tile = W4_TK / group;
    const int64_t tiles = (int64_t)s.n_tiles * s.k_tiles;
    s.groups_at = tiles * W4_TILE_BYTES;
    s.bytes = s.groups_at + tiles * s.per_tile * W4_TN * (zeros ? 4 : 2);
    return s;
}

struct W4PackArgs {
    const uint8_t *codes;
    const uint16_t *scales;
    const uint8_t *zeros;
    unsigned char *packed;
    W4Shape sh;
};

struct W4Proj {
    void *y;
    const void *x;
    const unsigned char *packed;
    int64_t groups_at;
    int hin, hout, k_tiles, n_tiles;
    int per_tile;              // groups of a K tile
    int zeros;                 // 0: 8 everywhere
    unsigned end;              // column blocks of the projections up to this one (set by the launcher)
};
struct W4Args {
    W4Proj pr[STEP_MAX_PROJ];
    int n_proj, T, accumulate;
    unsigned row_blocks;       // set by the launcher
};

// ---- keys and values
struct KvBatch {
    const int32_t *tok_req, *tok_pos;
    const int32_t *page_tbl;
    const int32_t *req_prefix;     // nullptr: no request has a prefix
    const int32_t *prefix_tbl, *prefix_len;
    int T, n_req, max_pages, n_prefix, max_prefix_pages;
};
struct KvAppendArgs {
    const uint16_t *q, *k, *v;
    uint16_t *q_out, *k_pages, *v_pages;
    int64_t q_stride, q_out_stride, k_stride, v_stride;
    int64_t n_pages;
    int page_shift, n_q_heads, n_kv_heads, head_dim;
    KvBatch b;
    const float *cos_sin;
    int n_pos, rot, interleaved;
    int32_t *bad;
};
struct AttnArgs {
    uint16_t *out;
    const uint16_t *q, *k_pages, *v_pages;
    int64_t out_stride, q_stride;
    int64_t n_pages;
    int page_shift, n_q_heads, n_kv_heads, head_dim, gq;   // gq: query heads per key head
    KvBatch b;
    float scale;
};

int launch_w4_pack(const W4PackArgs &a, hipStream_t s);
int launch_w4_gemv(const W4Args &a, int dtype, hipStream_t s);
int launch_kv_append(const KvAppendArgs &a, int dtype, hipStream_t s);
int64_t attn_plan_bytes(int T, int n_prefix, int n_q_heads, int n_kv_heads);
int64_t attn_workspace_bytes(int T, int n_prefix, int n_q_heads, int n_kv_heads, int head_dim);
int launch_attn_plan(const KvBatch &b, int page_shift, int n_q_heads, int n_kv_heads, int head_dim, void *plan, hipStream_t s);
int launch_prefix_attention(const AttnArgs &a, int dtype, const void *plan, void *workspace, hipStream_t s);

// sets the calling thread's error text and returns `code` (defined with the other entry points)
int fail_text(int code, const char *fmt, va_list ap);
int device_compute_units();

}  // namespace mlora

// Kernel argument blocks and launchers of the decode step around the LoRA apply: 4-bit base projections, cache appends,
// shared-prefix attention, microscaled 4-bit operands, the cache's page tables.
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

// ---- microscaled 4-bit operands.  A packed operand [rows, k], rows tokens or output columns, is two planes: codes, and the blocks' scales.
// Codes: tiles of 16 rows x 128 columns, 1024 bytes each, row tile major.  In a tile, slot 16 q + r of 64 holds the 16 bytes of block q (32
// columns, the lower of a pair in the low half of a byte) of row r - the operand of one lane of a scaled 16 x 16 x 128 MFMA, and
// with two row tiles that of a 32 x 32 x 64 one.  Columns past the operand's are zero codes.
// Scales (127 + X, 255: NaN): quads of four K tiles, 256 bytes each, row tile major.  Slot 16 q + r holds a dword whose byte j is the scale
// of block q of row r in K tile 4 quad + j: the byte that the MFMA selects.  Rows past the operand's hold anything: they only ever meet their own results.
constexpr int MX4_TK = 128, MX4_TILE_BYTES = 1024, MX4_QUAD_BYTES = 256;
struct Mx4Shape {
    int rows, k;
    int row_tiles, k_tiles, quads, blocks;
    int64_t scales_at, bytes;                  // byte offset of the second plane, total
};
inline Mx4Shape mx4_shape(int rows, int k)
{
    Mx4Shape s;
    s.rows = rows; s.k = k;
    s.row_tiles = (rows + 15) / 16;
    s.k_tiles = (k + MX4_TK - 1) / MX4_TK;
    s.quads = (s.k_tiles + 3) / 4;
    s.blocks = (k + 31) / 32;
    s.scales_at = (int64_t)s.row_tiles * s.k_tiles * MX4_TILE_BYTES;
    s.bytes = s.scales_at + (int64_t)s.row_tiles * s.quads * MX4_QUAD_BYTES;
    return s;
}
struct Mx4QuantArgs {
    const uint16_t *x;
    int64_t x_stride;
    unsigned char *packed;
    Mx4Shape sh;
};
struct Mx4PackArgs {
    const uint8_t *codes, *scales;
    unsigned char *packed;
    Mx4Shape sh;
};
struct Mx4ValuesArgs {
    const unsigned char *packed;
    uint16_t *out;
    int64_t out_stride;
    Mx4Shape sh;
};
struct Mx4Proj {
    void *y;
    const unsigned char *x, *w;
    int64_t x_scales_at, w_scales_at;
    int hin, hout, k_tiles, quads;
    unsigned end;              // tiles of the projections up to this one (set by the launcher)
};
struct Mx4Args {
    Mx4Proj pr[STEP_MAX_PROJ];
    int n_proj, T, accumulate;
    unsigned whole;            // tiles that a workgroup takes whole (these two set by the launcher)
    int first;                 // row of workgroups that a launch begins with
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
// ---- the cache's page tables.  State, one buffer of int32 words: [free: a byte a page, 0 or 1, to a multiple of 64][table n_req * max_pages]
// [lens n_req][refs n_pages][failed][live].  Scratch, likewise: [managed: bytes as free][grown n_req][words of head][writers n_pages][last_writer n_pages] - all but grown are
// set once, and the counts are zeros again after every call - then [picked n_pages][move_from n_pages][word_rank][word_movers][row_page n_req]
// [row_new 3 n_req][row_copy 2 n_req][copies 3 n_req][rows n_req * max_pages][pieces: a word for every ROW_PIECE entries of a row].
constexpr int ROW_PIECE = 1024;                // entries of a row that a workgroup takes
struct PagesLayout {
    int64_t table, lens, refs, failed, live, state_words;
    int64_t grown, head, writers, last_writer, picked, move_from, word_rank, word_movers, row_page, row_new, row_copy, copies, rows, pieces, scratch_words;
};
inline PagesLayout pages_layout(int64_t n_req, int64_t max_pages, int64_t n_pages)
{
    const int64_t words = (n_pages + 63) / 64;
    PagesLayout l;
    l.table = 16 * words;
    l.lens = l.table + n_req * max_pages;
    l.refs = l.lens + n_req;
    l.failed = l.refs + n_pages;
    l.live = l.failed + 1;
    l.state_words = l.live + 1;
    l.grown = 16 * words;
    l.head = l.grown + n_req;
    l.writers = l.head + 2;
    l.last_writer = l.writers + n_pages;
    l.picked = l.last_writer + n_pages;
    l.move_from = l.picked + n_pages;
    l.word_movers = (l.move_from + n_pages + 1) / 2 * 2;
    l.word_rank = l.word_movers + 2 * words;
    l.row_page = l.word_rank + words;
    l.row_new = l.row_page + n_req;
    l.row_copy = l.row_new + 3 * n_req;
    l.copies = l.row_copy + 2 * n_req;
    l.rows = l.copies + 3 * n_req;
    l.pieces = l.rows + n_req * max_pages;
    l.scratch_words = l.pieces + n_req * ((max_pages + ROW_PIECE - 1) / ROW_PIECE);
    return l;
}
struct PagesArgs {
    uint8_t *free_pages;
    int32_t *table, *lens, *refs, *failed, *live;
    int32_t *grown, *head, *writers, *last_writer, *picked, *move_from, *word_rank, *word_movers, *row_page, *row_new, *row_copy, *copies, *rows, *pieces;
    const uint8_t *managed;
    const int32_t *want;                       // want: the rows' new lengths, or their parents
    uint16_t *k, *v;
    int64_t n_pages;
    int n_req, max_pages, page_shift, n_layers, n_kv_heads, head_elems;      // head_elems: elements of one head of a page
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
int launch_mx4_quantize(const Mx4QuantArgs &a, int dtype, hipStream_t s);
int launch_mx4_pack(const Mx4PackArgs &a, hipStream_t s);
int launch_mx4_values(const Mx4ValuesArgs &a, int dtype, hipStream_t s);
void mx4_form(const Mx4Args &a, int *columns, int *tokens);
int launch_mx4_gemm(const Mx4Args &a, int dtype, hipStream_t s);
int launch_kv_append(const KvAppendArgs &a, int dtype, hipStream_t s);
int launch_pages_resize(const PagesArgs &a, hipStream_t s);
int launch_pages_fork(const PagesArgs &a, hipStream_t s);
int launch_pages_compact(const PagesArgs &a, hipStream_t s);
int64_t attn_plan_bytes(int T, int n_prefix, int n_q_heads, int n_kv_heads);
int64_t attn_workspace_bytes(int T, int n_prefix, int n_q_heads, int n_kv_heads, int head_dim);
int launch_attn_plan(const KvBatch &b, int page_shift, int n_q_heads, int n_kv_heads, int head_dim, void *plan, hipStream_t s);
int launch_prefix_attention(const AttnArgs &a, int dtype, const void *plan, void *workspace, hipStream_t s);

// sets the calling thread's error text and returns `code` (defined with the other entry points)
int fail_text(int code, const char *fmt, va_list ap);
int device_compute_units();

}  // namespace mlora

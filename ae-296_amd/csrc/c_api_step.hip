// extern "C" surface of the decode step around the LoRA apply (declared in include/mlora.h): argument validation on the host,
// then the kernel launches on the caller's stream.  No allocation, no synchronisation, no state kept between calls.
#include <cmath>
#include <cstring>

#include "../../include/mlora.h"
#include "mlora_step.hpp"

namespace {

int fail(int code, const char *fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    mlora::fail_text(code, fmt, ap);
    va_end(ap);
    return code;
}

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

bool overlap(const void *a, size_t a_bytes, const void *b, size_t b_bytes)
{
    const uintptr_t u = reinterpret_cast<uintptr_t>(a), w = reinterpret_cast<uintptr_t>(b);
    return u < w + b_bytes && w < u + a_bytes;
}

int log2_exact(int v)
{
    for (int s = 0; s < 31; s++)
        if ((1 << s) == v) return s;
    return -1;
}

int check_w4(int hin, int hout, int group)
{
    if (hin <= 0 || hout <= 0) return fail(MLORA_EINVAL, "hin and hout must be positive (got %d, %d)", hin, hout);
    if ((hin & 7) || (hout & 7)) return fail(MLORA_EALIGN, "hin and hout must be multiples of 8 (got %d, %d)", hin, hout);
    if (hin > (1 << 24) || hout > (1 << 24)) return fail(MLORA_ERANGE, "hin and hout may be 2^24 at most (got %d, %d)", hin, hout);
    if (group != 32 && group != 64 && group != 128) return fail(MLORA_ERANGE, "group must be 32, 64 or 128 (got %d)", group);
    return MLORA_OK;
}

int check_cache(int64_t n_pages, int page_tokens, int n_q_heads, int n_kv_heads, int head_dim)
{
    if (head_dim != 64 && head_dim != 128) return fail(MLORA_ERANGE, "head_dim must be 64 or 128 (got %d)", head_dim);
    if (log2_exact(page_tokens) < 4 || page_tokens > 256) return fail(MLORA_EINVAL, "page_tokens must be a power of two in 16..256 (got %d)", page_tokens);
    if (n_pages <= 0 || n_pages > 0x7fffffffLL) return fail(MLORA_ERANGE, "n_pages must be in 1..2^31-1");
    if (n_kv_heads <= 0 || n_q_heads <= 0 || n_kv_heads > 1024 || n_q_heads > 1024) return fail(MLORA_ERANGE, "head counts must be in 1..1024 (got %d, %d)", n_q_heads, n_kv_heads);
    if (n_q_heads % n_kv_heads) return fail(MLORA_EINVAL, "n_q_heads %d is no multiple of n_kv_heads %d", n_q_heads, n_kv_heads);
    return MLORA_OK;
}

int check_stride(const char *name, int64_t stride, int heads, int head_dim)
{
    if (stride < (int64_t)heads * head_dim) return fail(MLORA_EINVAL, "%s_stride %lld is shorter than a token's %d x %d elements", name, (long long)stride, heads, head_dim);
    if (stride & 7) return fail(MLORA_EALIGN, "%s_stride must be a multiple of 8 elements (got %lld)", name, (long long)stride);
    return MLORA_OK;
}

// Keys are numbered in 32 bits, with room to step past the last one.
int check_table(const char *name, int pages, int page_tokens)
{
    if (pages <= 0) return fail(MLORA_EINVAL, "%s must be positive (got %d)", name, pages);
    if ((int64_t)pages * page_tokens > (1 << 30)) return fail(MLORA_ERANGE, "%s * page_tokens may be 2^30 at most", name);
    return MLORA_OK;
}

int check_prefix(const int32_t *req_prefix, const int32_t *prefix_len, int n_prefix)
{
    if (n_prefix < 0 || n_prefix > MLORA_ATTN_MAX_PREFIX) return fail(MLORA_ERANGE, "n_prefix must be in 0..%d (got %d)", MLORA_ATTN_MAX_PREFIX, n_prefix);
    if (n_prefix > 0 && (!req_prefix || !prefix_len)) return fail(MLORA_EINVAL, "req_prefix and prefix_len are needed with n_prefix > 0");
    return MLORA_OK;
}

int check_batch(mlora::KvBatch &b, const int32_t *tok_req, const int32_t *tok_pos, int T, const int32_t *page_tbl, int n_req, int max_pages,
                int page_tokens, const int32_t *req_prefix, const int32_t *prefix_len, int n_prefix)
{
    if (!tok_req || !tok_pos || !page_tbl) return fail(MLORA_EINVAL, "tok_req, tok_pos and page_tbl must not be NULL");
    if (n_req <= 0) return fail(MLORA_EINVAL, "n_req must be positive (got %d)", n_req);
    int rc = check_table("max_pages", max_pages, page_tokens);
    if (rc || (rc = check_prefix(req_prefix, prefix_len, n_prefix))) return rc;
    b.tok_req = tok_req; b.tok_pos = tok_pos; b.page_tbl = page_tbl;
    b.req_prefix = n_prefix > 0 ? req_prefix : nullptr; b.prefix_len = prefix_len; b.prefix_tbl = nullptr;
    b.T = T; b.n_req = n_req; b.max_pages = max_pages; b.n_prefix = n_prefix; b.max_prefix_pages = 0;
    return MLORA_OK;
}

int check_attn_sizes(int T, int n_prefix, int n_q_heads, int n_kv_heads)
{
    if (T < 0 || T > MLORA_ATTN_MAX_T) return fail(MLORA_ERANGE, "T must be in 0..%d (got %d)", MLORA_ATTN_MAX_T, T);
    if (n_prefix < 0 || n_prefix > MLORA_ATTN_MAX_PREFIX) return fail(MLORA_ERANGE, "n_prefix must be in 0..%d (got %d)", MLORA_ATTN_MAX_PREFIX, n_prefix);
    return check_cache(1, 16, n_q_heads, n_kv_heads, 64);
}

}  // namespace

extern "C" {

int64_t mlora_w4_packed_bytes(int hin, int hout, int group, int zeros)
{
    const int rc = check_w4(hin, hout, group);
    return rc ? rc : mlora::w4_shape(hin, hout, group, zeros != 0).bytes;
}

int mlora_w4_pack(const uint8_t *codes, const void *scales, const uint8_t *zeros, int hin, int hout, int group, void *packed,
                  int64_t packed_bytes, void *stream)
{
    int rc = check_w4(hin, hout, group);
    if (rc) return rc;
    if (!codes || !scales || !packed) return fail(MLORA_EINVAL, "codes, scales and packed must not be NULL");
    if (!aligned16(packed)) return fail(MLORA_EALIGN, "packed must be 16-byte aligned");
    mlora::W4PackArgs a;
    a.sh = mlora::w4_shape(hin, hout, group, zeros != nullptr);
    if (packed_bytes < a.sh.bytes) return fail(MLORA_ENOSPACE, "packed has %lld bytes, %lld needed", (long long)packed_bytes, (long long)a.sh.bytes);
    a.codes = codes; a.scales = static_cast<const uint16_t *>(scales); a.zeros = zeros; a.packed = static_cast<unsigned char *>(packed);
    rc = mlora::launch_w4_pack(a, static_cast<hipStream_t>(stream));
    if (rc) return fail(MLORA_ELAUNCH, "pack launch failed: %s", hipGetErrorString((hipError_t)rc));
    return MLORA_OK;
}

int mlora_w4_gemv_multi(int n_proj, void *const *y, const void *const *x, const void *const *packed, const int32_t *hin,
                        const int32_t *hout, const int32_t *group, const int32_t *zeros, int T, int dtype, int accumulate, void *stream)
{
    if (dtype != MLORA_F16 && dtype != MLORA_BF16) return fail(MLORA_EDTYPE, "dtype must be MLORA_F16 or MLORA_BF16 (got %d)", dtype);
    if (n_proj < 1 || n_proj > MLORA_MAX_PROJ) return fail(MLORA_ERANGE, "n_proj must be in 1..%d (got %d)", MLORA_MAX_PROJ, n_proj);
    if (T < 0 || T > (1 << 20)) return fail(MLORA_ERANGE, "T must be in 0..2^20 (got %d)", T);
    if (!y || !x || !packed || !hin || !hout || !group || !zeros) return fail(MLORA_EINVAL, "y, x, packed, hin, hout, group and zeros must not be NULL");
    mlora::W4Args a;
    memset(&a, 0, sizeof(a));
    a.n_proj = n_proj; a.T = T; a.accumulate = accumulate != 0;
    for (int p = 0; p < n_proj; p++) {
        const int rc = check_w4(hin[p], hout[p], group[p]);
        if (rc) return rc;
        if (T == 0) continue;
        if (!y[p] || !x[p] || !packed[p]) return fail(MLORA_EINVAL, "projection %d: NULL device pointer", p);
        if (!aligned16(y[p]) || !aligned16(x[p]) || !aligned16(packed[p])) return fail(MLORA_EALIGN, "projection %d: device pointers must be 16-byte aligned", p);
        const mlora::W4Shape sh = mlora::w4_shape(hin[p], hout[p], group[p], zeros[p] != 0);
        mlora::W4Proj &w = a.pr[p];
        w.y = y[p]; w.x = x[p]; w.packed = static_cast<const unsigned char *>(packed[p]);
        w.groups_at = sh.groups_at; w.hin = sh.hin; w.hout = sh.hout; w.k_tiles = sh.k_tiles; w.n_tiles = sh.n_tiles;
        w.per_tile = sh.per_tile; w.zeros = zeros[p] != 0;
    }
    if (T == 0) return MLORA_OK;
    for (int p = 0; p < n_proj; p++)                              // workgroups read and write in no order
        for (int o = 0; o < n_proj; o++) {
            const size_t yp = (size_t)T * hout[p] * 2;
            if (overlap(y[p], yp, x[o], (size_t)T * hin[o] * 2) || (o < p && overlap(y[p], yp, y[o], (size_t)T * hout[o] * 2)))
                return fail(MLORA_EINVAL, "projection %d: y overlaps x or y of projection %d", p, o);
        }
    const int rc = mlora::launch_w4_gemv(a, dtype, static_cast<hipStream_t>(stream));
    if (rc) return fail(MLORA_ELAUNCH, "w4 launch failed: %s", hipGetErrorString((hipError_t)rc));
    return MLORA_OK;
}

int mlora_kv_append(const void *q, int64_t q_stride, void *q_out, int64_t q_out_stride, const void *k, int64_t k_stride,
                    const void *v, int64_t v_stride, void *k_pages, void *v_pages, int64_t n_pages, int page_tokens,
                    int n_q_heads, int n_kv_heads, int head_dim, const int32_t *tok_req, const int32_t *tok_pos, int T,
                    const int32_t *page_tbl, int n_req, int max_pages, const int32_t *req_prefix, const int32_t *prefix_len,
                    int n_prefix, const float *cos_sin, int n_pos, int rot, int interleaved, int32_t *bad, int dtype, void *stream)
{
    if (dtype != MLORA_F16 && dtype != MLORA_BF16) return fail(MLORA_EDTYPE, "dtype must be MLORA_F16 or MLORA_BF16 (got %d)", dtype);
    if (T < 0) return fail(MLORA_EINVAL, "T must be >= 0 (got %d)", T);
    if (T > (1 << 30)) return fail(MLORA_ERANGE, "T may be 2^30 at most (got %d)", T);
    int rc = check_cache(n_pages, page_tokens, n_q_heads, n_kv_heads, head_dim);
    if (rc) return rc;
    if (rot < 0 || rot > head_dim || (rot & 15)) return fail(MLORA_ERANGE, "rot must be a multiple of 16 in 0..head_dim (got %d)", rot);
    if (rot > 0 && (!cos_sin || n_pos <= 0)) return fail(MLORA_EINVAL, "cos_sin and a positive n_pos are needed with rot > 0");
    if (T == 0) return MLORA_OK;
    if (!k || !v || !k_pages || !v_pages) return fail(MLORA_EINVAL, "k, v, k_pages and v_pages must not be NULL");
    if ((q == nullptr) != (q_out == nullptr)) return fail(MLORA_EINVAL, "q and q_out go together: both or neither NULL");
    if (!aligned16(q) || !aligned16(q_out) || !aligned16(k) || !aligned16(v) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(cos_sin))
        return fail(MLORA_EALIGN, "device pointers must be 16-byte aligned");
    if (q && ((rc = check_stride("q", q_stride, n_q_heads, head_dim)) || (rc = check_stride("q_out", q_out_stride, n_q_heads, head_dim)))) return rc;
    if ((rc = check_stride("k", k_stride, n_kv_heads, head_dim)) || (rc = check_stride("v", v_stride, n_kv_heads, head_dim))) return rc;
    if (q == q_out && q && q_stride != q_out_stride) return fail(MLORA_EINVAL, "q_out is q itself with another stride");
    mlora::KvAppendArgs a;
    memset(&a, 0, sizeof(a));
    if ((rc = check_batch(a.b, tok_req, tok_pos, T, page_tbl, n_req, max_pages, page_tokens, req_prefix, prefix_len, n_prefix))) return rc;
    a.q = static_cast<const uint16_t *>(q); a.k = static_cast<const uint16_t *>(k); a.v = static_cast<const uint16_t *>(v);
    a.q_out = static_cast<uint16_t *>(q_out); a.k_pages = static_cast<uint16_t *>(k_pages); a.v_pages = static_cast<uint16_t *>(v_pages);
    a.q_stride = q_stride; a.q_out_stride = q_out_stride; a.k_stride = k_stride; a.v_stride = v_stride;
    a.n_pages = n_pages; a.page_shift = log2_exact(page_tokens);
    a.n_q_heads = q ? n_q_heads : 0; a.n_kv_heads = n_kv_heads; a.head_dim = head_dim;
    a.cos_sin = cos_sin; a.n_pos = n_pos; a.rot = rot; a.interleaved = interleaved != 0; a.bad = bad;
    rc = mlora::launch_kv_append(a, dtype, static_cast<hipStream_t>(stream));
    if (rc) return fail(MLORA_ELAUNCH, "append launch failed: %s", hipGetErrorString((hipError_t)rc));
    return MLORA_OK;
}

int64_t mlora_attn_plan_bytes(int T, int n_prefix, int n_q_heads, int n_kv_heads)
{
    const int rc = check_attn_sizes(T, n_prefix, n_q_heads, n_kv_heads);
    return rc ? rc : mlora::attn_plan_bytes(T, n_prefix, n_q_heads, n_kv_heads);
}

int64_t mlora_attn_workspace_bytes(int T, int n_prefix, int n_q_heads, int n_kv_heads, int head_dim)
{
    int rc = check_attn_sizes(T, n_prefix, n_q_heads, n_kv_heads);
    if (rc || (rc = check_cache(1, 16, n_q_heads, n_kv_heads, head_dim))) return rc;
    return mlora::attn_workspace_bytes(T, n_prefix, n_q_heads, n_kv_heads, head_dim);
}

int mlora_attn_plan(const int32_t *tok_req, const int32_t *tok_pos, int T, int n_req, int max_pages, const int32_t *req_prefix,
                    const int32_t *prefix_len, int n_prefix, int max_prefix_pages, int page_tokens, int n_q_heads, int n_kv_heads, int head_dim,
                    void *plan, int64_t plan_bytes, void *stream)
{
    if (T < 0 || T > MLORA_ATTN_MAX_T) return fail(MLORA_ERANGE, "T must be in 0..%d (got %d)", MLORA_ATTN_MAX_T, T);
    int rc = check_cache(1, page_tokens, n_q_heads, n_kv_heads, head_dim);
    if (rc) return rc;
    if (T == 0) return MLORA_OK;
    if (n_req <= 0) return fail(MLORA_EINVAL, "n_req must be positive (got %d)", n_req);
    if ((rc = check_table("max_pages", max_pages, page_tokens)) || (rc = check_prefix(req_prefix, prefix_len, n_prefix))) return rc;
    if (n_prefix > 0 && (rc = check_table("max_prefix_pages", max_prefix_pages, page_tokens))) return rc;
    if (!tok_req || !tok_pos || !plan) return fail(MLORA_EINVAL, "tok_req, tok_pos and plan must not be NULL");
    if (!aligned16(plan)) return fail(MLORA_EALIGN, "plan must be 16-byte aligned");
    if (plan_bytes < mlora::attn_plan_bytes(T, n_prefix, n_q_heads, n_kv_heads)) return fail(MLORA_ENOSPACE, "plan has %lld bytes, too few", (long long)plan_bytes);
    mlora::KvBatch b;
    memset(&b, 0, sizeof(b));
    b.tok_req = tok_req; b.tok_pos = tok_pos; b.req_prefix = n_prefix > 0 ? req_prefix : nullptr; b.prefix_len = prefix_len;
    b.T = T; b.n_req = n_req; b.max_pages = max_pages; b.n_prefix = n_prefix; b.max_prefix_pages = max_prefix_pages;
    rc = mlora::launch_attn_plan(b, log2_exact(page_tokens), n_q_heads, n_kv_heads, head_dim, plan, static_cast<hipStream_t>(stream));
    if (rc) return fail(MLORA_ELAUNCH, "plan launch failed: %s", hipGetErrorString((hipError_t)rc));
    return MLORA_OK;
}

int mlora_prefix_attention(void *out, int64_t out_stride, const void *q, int64_t q_stride, const void *k_pages,
                           const void *v_pages, int64_t n_pages, int page_tokens, int n_q_heads, int n_kv_heads, int head_dim,
                           const int32_t *tok_req, const int32_t *tok_pos, int T, const int32_t *page_tbl, int n_req, int max_pages,
                           const int32_t *req_prefix, const int32_t *prefix_tbl, const int32_t *prefix_len, int n_prefix,
                           int max_prefix_pages, float scale, const void *plan, int64_t plan_bytes, void *workspace,
                           int64_t workspace_bytes, int dtype, void *stream)
{
    if (dtype != MLORA_F16 && dtype != MLORA_BF16) return fail(MLORA_EDTYPE, "dtype must be MLORA_F16 or MLORA_BF16 (got %d)", dtype);
    if (T < 0 || T > MLORA_ATTN_MAX_T) return fail(MLORA_ERANGE, "T must be in 0..%d (got %d)", MLORA_ATTN_MAX_T, T);
    int rc = check_cache(n_pages, page_tokens, n_q_heads, n_kv_heads, head_dim);
    if (rc) return rc;
    if (T == 0) return MLORA_OK;
    if ((rc = check_prefix(req_prefix, prefix_len, n_prefix))) return rc;
    if (!std::isfinite(scale)) return fail(MLORA_EINVAL, "scale must be finite");
    // it is applied in powers of two: times 1.44 it has to be a normal number still
    if (scale != 0.f && (fabsf(scale) < 0x1p-126f || fabsf(scale) > 0x1p127f)) return fail(MLORA_ERANGE, "scale must be 0 or between 2^-126 and 2^127 (got %g)", scale);
    if (n_prefix > 0 && !prefix_tbl) return fail(MLORA_EINVAL, "prefix_tbl is needed with n_prefix > 0");
    if (n_prefix > 0 && (rc = check_table("max_prefix_pages", max_prefix_pages, page_tokens))) return rc;
    if (!out || !q || !k_pages || !v_pages || !plan) return fail(MLORA_EINVAL, "out, q, k_pages, v_pages and plan must not be NULL");
    if (!aligned16(out) || !aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(plan) || !aligned16(workspace))
        return fail(MLORA_EALIGN, "device pointers must be 16-byte aligned");
    if ((rc = check_stride("q", q_stride, n_q_heads, head_dim)) || (rc = check_stride("out", out_stride, n_q_heads, head_dim))) return rc;
    if (plan_bytes < mlora::attn_plan_bytes(T, n_prefix, n_q_heads, n_kv_heads)) return fail(MLORA_ENOSPACE, "plan has %lld bytes, too few", (long long)plan_bytes);
    const int64_t need = mlora::attn_workspace_bytes(T, n_prefix, n_q_heads, n_kv_heads, head_dim);
    if (workspace_bytes < need || !workspace) return fail(MLORA_ENOSPACE, "workspace has %lld bytes, %lld needed", (long long)workspace_bytes, (long long)need);
    mlora::AttnArgs a;
    memset(&a, 0, sizeof(a));
    if ((rc = check_batch(a.b, tok_req, tok_pos, T, page_tbl, n_req, max_pages, page_tokens, req_prefix, prefix_len, n_prefix))) return rc;
    a.b.prefix_tbl = prefix_tbl; a.b.max_prefix_pages = max_prefix_pages;
    a.out = static_cast<uint16_t *>(out); a.q = static_cast<const uint16_t *>(q);
    a.k_pages = static_cast<const uint16_t *>(k_pages); a.v_pages = static_cast<const uint16_t *>(v_pages);
    a.out_stride = out_stride; a.q_stride = q_stride; a.n_pages = n_pages; a.page_shift = log2_exact(page_tokens);
    a.n_q_heads = n_q_heads; a.n_kv_heads = n_kv_heads; a.head_dim = head_dim; a.gq = n_q_heads / n_kv_heads;
    a.scale = scale;
    rc = mlora::launch_prefix_attention(a, dtype, plan, workspace, static_cast<hipStream_t>(stream));
    if (rc) return fail(MLORA_ELAUNCH, "attention launch failed: %s", hipGetErrorString((hipError_t)rc));
    return MLORA_OK;
}

}  // extern "C"

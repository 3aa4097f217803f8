// Host-side checks of the linear-attention and expert operators' arguments (declared in include/qwattn.h), apart
// from any GPU call so that they run on a machine without one. Each returns QWATTN_OK, or a status with its text
// in `msg`.
#pragma once
#include <stdarg.h>
#include <stdint.h>
#include <stdio.h>

#include "../../include/qwattn.h"

namespace qw {

struct CheckText {
    char text[256] = "";
};

__attribute__((format(printf, 3, 4))) inline int refuse(CheckText& m, int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(m.text, sizeof m.text, fmt, ap);
    va_end(ap);
    return code;
}

inline bool bad_dtype(int d) { return d != QWATTN_F32 && d != QWATTN_BF16; }
inline bool unaligned(const void* p, unsigned to = 16) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) != 0; }
// A row stride of at least `width` elements, a multiple of 8, that spans at most 2^59 elements (2^61 bytes) over the rows
inline bool bad_stride(int64_t s, int64_t width, int64_t rows) { return s < width || s % 8 || s > (int64_t(1) << 59) / rows; }

// Whether the byte ranges of two row sets meet: `rows` rows of `width` bytes at `stride` bytes from p, and likewise
// from q (each within 2^61 bytes: bad_stride). Rows at one stride whose columns do not meet (two slices of one buffer's rows) count as apart.
inline bool rows_meet(const void* p, int64_t p_width, int64_t p_stride, const void* q, int64_t q_width, int64_t q_stride,
                      int64_t rows) {
    const int64_t a = (int64_t)reinterpret_cast<uintptr_t>(p), b = (int64_t)reinterpret_cast<uintptr_t>(q);
    if (a >= b + (rows - 1) * q_stride + q_width || b >= a + (rows - 1) * p_stride + p_width) return false;
    if (p_stride != q_stride) return true;
    int64_t d = (b - a) % p_stride;  // q's columns start d bytes behind p's
    if (d < 0) d += p_stride;
    return d < p_width || d + q_width > p_stride;
}

// Rows of a call: tiles of up to 32,768 tokens and chunks of 64 are counted by 32-bit sums behind the last row
constexpr int64_t kMostRows = (int64_t(1) << 31) - (1 << 16);

inline int check_conv(const qwattn_conv* a, CheckText& m) {
    if (!a) return refuse(m, QWATTN_EINVAL, "qwattn_conv_silu: null arguments");
    if (a->n_seq <= 0 || a->n <= 0 || (int64_t)a->n_seq * a->n > kMostRows || a->n_seq > 65535)
        return refuse(m, QWATTN_EINVAL, "qwattn_conv_silu: n_seq %d (1..65535), n %d (n_seq x n <= 2^31 - 2^16)", a->n_seq, a->n);
    if (a->channels <= 0 || a->channels % 8 || a->channels > (1 << 24) || a->taps < 2 || a->taps > 4 || bad_dtype(a->dtype))
        return refuse(m, QWATTN_EINVAL, "qwattn_conv_silu: channels %d (a multiple of 8), taps %d (2..4), dtype %d",
                      a->channels, a->taps, a->dtype);
    if (!a->x || !a->w || !a->state || !a->y) return refuse(m, QWATTN_EINVAL, "qwattn_conv_silu: null pointer");
    const int64_t rows = (int64_t)a->n_seq * a->n;
    if (bad_stride(a->x_stride, a->channels, rows) || bad_stride(a->y_stride, a->channels, rows))
        return refuse(m, QWATTN_EINVAL, "qwattn_conv_silu: x_stride %lld, y_stride %lld (>= channels, multiples of 8, x rows <= 2^59)",
                      (long long)a->x_stride, (long long)a->y_stride);
    if (unaligned(a->x) || unaligned(a->w) || unaligned(a->bias) || unaligned(a->state) || unaligned(a->snap) || unaligned(a->y))
        return refuse(m, QWATTN_EINVAL, "qwattn_conv_silu: pointers must be 16-byte aligned");
    const int64_t size = a->dtype == QWATTN_F32 ? 4 : 2;
    if (rows_meet(a->x, a->channels * size, a->x_stride * size, a->y, a->channels * size, a->y_stride * size, rows))
        return refuse(m, QWATTN_EINVAL, "qwattn_conv_silu: x and y overlap");
    return QWATTN_OK;
}

inline int check_delta_shape(const qwattn_delta* a, CheckText& m) {
    if (!a) return refuse(m, QWATTN_EINVAL, "qwattn_delta_rule: null arguments");
    if (a->n_seq <= 0 || a->n <= 0 || (int64_t)a->n_seq * a->n > kMostRows || a->n_seq > 65535)
        return refuse(m, QWATTN_EINVAL, "qwattn_delta_rule: n_seq %d (1..65535), n %d (n_seq x n <= 2^31 - 2^16)", a->n_seq, a->n);
    if (a->k_heads <= 0 || a->v_heads <= 0 || a->v_heads > 1024 || a->v_heads % a->k_heads)
        return refuse(m, QWATTN_EINVAL, "qwattn_delta_rule: k_heads %d, v_heads %d (a multiple of k_heads, <= 1024)",
                      a->k_heads, a->v_heads);
    // a launch has less than 2^32 threads in x: 4,096 a (sequence, value head), and 32 a row and head for the gated norm
    if ((int64_t)a->n_seq * a->v_heads >= (1 << 20) || (a->z && (int64_t)a->n_seq * a->n * a->v_heads >= (1 << 27)))
        return refuse(m, QWATTN_EINVAL, "qwattn_delta_rule: n_seq %d x v_heads %d (< 2^20), with z x n %d (< 2^27)", a->n_seq,
                      a->v_heads, a->n);
    if ((a->key_dim != 64 && a->key_dim != 128) || (a->val_dim != 64 && a->val_dim != 128))
        return refuse(m, QWATTN_EINVAL, "qwattn_delta_rule: key_dim %d, val_dim %d (64 or 128)", a->key_dim, a->val_dim);
    if (bad_dtype(a->dtype) || a->tiled < 0 || a->tiled > 1)
        return refuse(m, QWATTN_EINVAL, "qwattn_delta_rule: dtype %d, tiled %d", a->dtype, a->tiled);
    return QWATTN_OK;
}

inline int check_delta(const qwattn_delta* a, size_t workspace, CheckText& m) {
    if (int rc = check_delta_shape(a, m)) return rc;
    if (!a->q || !a->k || !a->v || !a->a || !a->b || !a->state || !a->out)
        return refuse(m, QWATTN_EINVAL, "qwattn_delta_rule: null pointer");
    if (!a->a_coef != !a->dt_bias) return refuse(m, QWATTN_EINVAL, "qwattn_delta_rule: a_coef and dt_bias come together");
    if (!a->z != !a->gamma) return refuse(m, QWATTN_EINVAL, "qwattn_delta_rule: z and gamma come together");
    const int64_t kw = (int64_t)a->k_heads * a->key_dim, vw = (int64_t)a->v_heads * a->val_dim;
    const int64_t rows = (int64_t)a->n_seq * a->n;
    if (bad_stride(a->q_stride, kw, rows) || bad_stride(a->k_stride, kw, rows) || bad_stride(a->v_stride, vw, rows) ||
        bad_stride(a->out_stride, vw, rows) || (a->z && bad_stride(a->z_stride, vw, rows)))
        return refuse(m, QWATTN_EINVAL, "qwattn_delta_rule: strides q %lld, k %lld, v %lld, z %lld, out %lld (at least the "
                      "heads' elements, multiples of 8, x rows <= 2^59)", (long long)a->q_stride, (long long)a->k_stride,
                      (long long)a->v_stride, (long long)a->z_stride, (long long)a->out_stride);
    if (unaligned(a->q) || unaligned(a->k) || unaligned(a->v) || unaligned(a->z) || unaligned(a->out) || unaligned(a->state) ||
        unaligned(a->snap))
        return refuse(m, QWATTN_EINVAL, "qwattn_delta_rule: q, k, v, z, out, state and snap must be 16-byte aligned");
    const int64_t size = a->dtype == QWATTN_F32 ? 4 : 2;
    struct {
        const void* p;
        int64_t width, stride;
    } in[] = {{a->q, kw, a->q_stride}, {a->k, kw, a->k_stride}, {a->v, vw, a->v_stride}, {a->z, vw, a->z_stride}};
    for (const auto& i : in)
        if (i.p && rows_meet(i.p, i.width * size, i.stride * size, a->out, vw * size, a->out_stride * size, rows))
            return refuse(m, QWATTN_EINVAL, "qwattn_delta_rule: out overlaps q, k, v or z");
    if (workspace && (!a->workspace || a->workspace_bytes < workspace || unaligned(a->workspace, 256)))
        return refuse(m, QWATTN_EINVAL, "qwattn_delta_rule: a workspace of %zu bytes, 256-byte aligned, is needed (%zu given)",
                      workspace, a->workspace ? a->workspace_bytes : (size_t)0);
    return QWATTN_OK;
}

inline int check_route(const float* logits, int stride, int n, int n_experts, int top_k, const int32_t* ids,
                       const float* weights, CheckText& m) {
    if (!logits || !ids || !weights) return refuse(m, QWATTN_EINVAL, "qwattn_moe_route: null pointer");
    // a wave a row, and less than 2^32 threads
    if (n <= 0 || n >= (1 << 26) - 4 || n_experts <= 0 || n_experts > 1024 || top_k <= 0 || top_k > 64 || top_k > n_experts ||
        (int64_t)n * top_k > INT32_MAX)
        return refuse(m, QWATTN_EINVAL, "qwattn_moe_route: n %d (< 2^26 - 4), n_experts %d (<= 1024), top_k %d (<= 64 and "
                      "n_experts)", n, n_experts, top_k);
    if (stride < n_experts) return refuse(m, QWATTN_EINVAL, "qwattn_moe_route: logits_stride %d (>= n_experts)", stride);
    return QWATTN_OK;
}

inline int check_moe_layer(const qwattn_moe_layer* l, int dtype, int n, int top_k, CheckText& m) {
    if (!l) return refuse(m, QWATTN_EINVAL, "qwattn_moe: null layer");
    // one expert's matrix is addressed with 32-bit offsets
    if (l->n_experts <= 0 || l->n_experts > 1024 || l->hidden <= 0 || l->ffn <= 0 || l->hidden % 32 || l->ffn % 32 ||
        l->hidden > (1 << 16) || l->ffn > (1 << 16) || (int64_t)l->hidden * l->ffn > (1 << 29))
        return refuse(m, QWATTN_EINVAL, "qwattn_moe: n_experts %d (<= 1024), hidden %d, ffn %d (multiples of 32, <= 65536)",
                      l->n_experts, l->hidden, l->ffn);
    if (n <= 0 || top_k <= 0 || top_k > 64 || (int64_t)n * top_k > (1 << 24) || bad_dtype(dtype))
        return refuse(m, QWATTN_EINVAL, "qwattn_moe: n %d (n x top_k <= 2^24), top_k %d (1..64), dtype %d", n, top_k, dtype);
    return QWATTN_OK;
}

inline int check_moe(const qwattn_moe_layer* l, const void* x, int dtype, int64_t x_stride, const int32_t* ids,
                     const float* weights, int top_k, const void* y, int64_t y_stride, int n, const void* ws,
                     size_t ws_bytes, size_t need, CheckText& m) {
    if (int rc = check_moe_layer(l, dtype, n, top_k, m)) return rc;
    if (!l->w_gate || !l->w_up || !l->w_down || !l->s_gate || !l->s_up || !l->s_down || !x || !ids || !weights || !y)
        return refuse(m, QWATTN_EINVAL, "qwattn_moe: null pointer");
    if (bad_stride(x_stride, l->hidden, n) || bad_stride(y_stride, l->hidden, n))
        return refuse(m, QWATTN_EINVAL, "qwattn_moe: x_stride %lld, y_stride %lld (>= hidden, multiples of 8, x n <= 2^59)",
                      (long long)x_stride, (long long)y_stride);
    if (unaligned(l->w_gate) || unaligned(l->w_up) || unaligned(l->w_down) || unaligned(x) || unaligned(y))
        return refuse(m, QWATTN_EINVAL, "qwattn_moe: the int8 weights, x and y must be 16-byte aligned");
    const int64_t size = dtype == QWATTN_F32 ? 4 : 2;
    if (rows_meet(x, l->hidden * size, x_stride * size, y, l->hidden * size, y_stride * size, n))
        return refuse(m, QWATTN_EINVAL, "qwattn_moe: x and y overlap");
    if (need && (!ws || ws_bytes < need || unaligned(ws, 256)))
        return refuse(m, QWATTN_EINVAL, "qwattn_moe: a workspace of %zu bytes, 256-byte aligned, is needed (%zu given)", need,
                      ws ? ws_bytes : (size_t)0);
    return QWATTN_OK;
}

}  // namespace qw

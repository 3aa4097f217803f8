// The argument checks of the linear-attention and expert operators as a shared library for a CPU test.
#include "../../qwen3-local-test_amd/csrc/checks.hpp"

static qw::CheckText text;

extern "C" {
int layer_sizeof(int which) { return which == 0 ? sizeof(qwattn_conv) : which == 1 ? sizeof(qwattn_delta) : sizeof(qwattn_moe_layer); }
const char* layer_text() { return text.text; }
int layer_conv(const qwattn_conv* a) { return qw::check_conv(a, text); }
int layer_delta(const qwattn_delta* a, size_t workspace) { return qw::check_delta(a, workspace, text); }
int layer_route(const float* l, int stride, int n, int e, int k, const int32_t* ids, const float* w) {
    return qw::check_route(l, stride, n, e, k, ids, w, text);
}
int layer_moe(const qwattn_moe_layer* l, const void* x, int dtype, int64_t xs, const int32_t* ids, const float* w, int k,
              const void* y, int64_t ys, int n, const void* ws, size_t bytes, size_t need) {
    return qw::check_moe(l, x, dtype, xs, ids, w, k, y, ys, n, ws, bytes, need, text);
}
}

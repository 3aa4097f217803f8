// The argument checks of the paged-attention operators as a shared library for a CPU test.
#include "../../qwen3-local-test_amd/csrc/checks.hpp"

static qw::CheckText text;

extern "C" {
int paged_sizeof(int which) { return which ? sizeof(qwattn_paged_attend_args) : sizeof(qwattn_paged_append_args); }
const char* paged_text() { return text.text; }
int paged_append(const qwattn_paged_append_args* a, const qwattn_config* g) { return qw::check_paged_append(a, *g, text); }
int paged_attend(const qwattn_paged_attend_args* a, const qwattn_config* g, size_t need) {
    return qw::check_paged_attend(a, *g, need, text);
}
}

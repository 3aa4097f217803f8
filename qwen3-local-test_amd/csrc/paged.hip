// Batches of sequences over a paged K/V cache for gfx950: appending new tokens to their pages, and their attention.
//
// A page holds 2^lg_page positions of every KV head, in the 32-position blocks of common.hpp; table[b] names the
// pages of sequence b. The reference serves one sequence (src/qwen4_vk.cpp:937-996).
#include "paged.hpp"

#include <algorithm>

namespace qw {

namespace {

// ... of position p of sequence b; -1 without a page
__device__ __forceinline__ int64_t paged_block_at(const PagedCache& c, int b, int p, int h, int nkv, int D) {
    const int32_t page = c.table[(size_t)b * c.table_stride + (p >> c.lg_page)];
    return (uint32_t)page < (uint32_t)c.n_pages ? paged_block(c, page, p, h, nkv, D) : -1;
}

// ---- append --------------------------------------------------------------------------------------------------
// The arithmetic and lane layout of k_qk_norm_rope (norm_rope.hip): a half-wave a (token, head) row, D / 32 dims a
// lane; values by lanes of their own that turn 8 positions x 8 dims into the blocks' 16-byte pieces. Bound by memory where there
// are many tokens: 2250 bf16 tokens of 16 heads of 256 (46.7 MB) 16.5 us, 2.8 TB/s; one token 4.2 us, a launch and its first loads.

// 8-position groups that a sequence's new tokens can touch, whatever its first position
__host__ __device__ constexpr int paged_groups(int n) { return (n + 6) / 8 + 1; }

template <int D, int DT>
__device__ __forceinline__ void paged_v_copy(const PagedAppendArgs& a, int64_t vi) {
    constexpr int NC = D / 8;
    const int ng = paged_groups(a.n);
    if (vi >= (int64_t)a.n_seq * a.NKV * ng * NC) return;
    const int c = (int)(vi % NC), gi = (int)(vi / NC % ng), h = (int)(vi / NC / ng % a.NKV), b = (int)(vi / NC / ng / a.NKV);
    const int64_t pos = a.pos[b];
    const int len = seq_len(a.lens, b, a.n);
    const int64_t p0 = ((pos >> 3) + gi) * 8;
    // tokens [t0, t1) of the sequence lie in this group at valid positions
    const int64_t lo = max(max(p0, pos), (int64_t)0), hi = min(min(p0 + 8, pos + len), (int64_t)a.limit);
    if (lo >= hi) return;
    const int64_t blk = paged_block_at(a.c, b, (int)p0, h, a.NKV, D);  // (p0 >= 0: lo < p0 + 8 and lo >= 0, p0 a multiple of 8)
    if (blk < 0) return;
    float x[8][8];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        const int64_t t = min(max(p0 + i, lo), hi - 1) - pos;
        load_vec<DT, 8>(a.v, ((size_t)b * a.n + (size_t)t) * a.v_stride + (size_t)h * D + 8 * c, x[i]);
    }
    f16* vc = reinterpret_cast<f16*>(a.c.v) + blk;
    const int kb0 = (int)p0 & (kBlk - 1);
    const bool whole = lo == p0 && hi == p0 + 8;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        f16* dst = vc + v_off(kb0, 8 * c + j);
        if (whole) {
            f16x8 o;
#pragma unroll
            for (int i = 0; i < 8; i++) o[i] = (f16)x[i][j];
            *reinterpret_cast<f16x8*>(dst) = o;
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (p0 + i >= lo && p0 + i < hi) dst[i] = (f16)x[i][j];
        }
    }
}

template <int D, int DT>
__global__ __launch_bounds__(256) void k_paged_append(PagedAppendArgs a) {
    constexpr int DPL = D / 32;
    const int hl = threadIdx.x & 31;
    const int q_heads = a.q ? a.NH : 0, heads = q_heads + a.NKV;
    const int n_items = a.n_seq * a.n * heads;
    const int norm_blocks = (n_items + 7) / 8;
    if ((int)blockIdx.x >= norm_blocks) {
        paged_v_copy<D, DT>(a, (int64_t)((int)blockIdx.x - norm_blocks) * 256 + threadIdx.x);
        return;
    }
    const int item = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (item >= n_items) return;  // (whole half-waves leave, as below)
    const int row = item / heads, hh = item - row * heads;
    const int b = row / a.n, t = row - b * a.n;
    if (t >= seq_len(a.lens, b, a.n)) return;
    const bool is_q = hh < q_heads;
    const int h = is_q ? hh : hh - q_heads;
    const int d0 = hl * DPL;
    float x[DPL], w[DPL], cs[2 * DPL];
    load_vec<DT, DPL>(is_q ? a.q : a.k, is_q ? (size_t)row * a.q_stride + (size_t)h * a.q_head + d0 : (size_t)row * a.k_stride + (size_t)h * D + d0, x);
    const float* gamma = is_q ? a.qn : a.kn;
    if (gamma) load_vec<0, DPL>(gamma, d0, w);
    const int64_t p = (int64_t)a.pos[b] + t;
    const bool there = p >= 0 && p < a.limit;
    const int half_r = a.R >> 1;
    const bool rot = d0 < a.R && there;  // DPL divides R / 2: a lane's dims are all rotated or all not
    const bool low = d0 < half_r;
    if (rot) load_vec<0, 2 * DPL>(a.rope, (size_t)p * a.R + 2 * (low ? d0 : d0 - half_r), cs);
    if (gamma) {
        float ss = 0.f;
#pragma unroll
        for (int j = 0; j < DPL; j++) ss += x[j] * x[j];
#pragma unroll
        for (int m = 16; m >= 1; m >>= 1) ss += __shfl_xor(ss, m, 32);
        const float rn = 1.0f / sqrtf(ss / (float)D + a.eps);
#pragma unroll
        for (int j = 0; j < DPL; j++) x[j] = x[j] * rn * (1.0f + w[j]);
    }
    // rotate-half: the partner dim d +- R / 2 sits (R / 2) / DPL lanes away in the same half-wave
    const int offl = half_r / DPL;
    const int src = (threadIdx.x & 32) + (rot ? (low ? hl + offl : hl - offl) : hl);
#pragma unroll
    for (int j = 0; j < DPL; j++) {
        const float partner = __shfl(x[j], src, 64);
        if (rot) x[j] = low ? x[j] * cs[2 * j] - partner * cs[2 * j + 1] : x[j] * cs[2 * j] + partner * cs[2 * j + 1];
    }
    if (is_q) {
        const size_t at = (size_t)row * a.q_out_stride + (size_t)h * D + d0;
#pragma unroll
        for (int j = 0; j < DPL; j++) x[j] = there ? x[j] : 0.f;
        if constexpr (DT == 0) {
            typedef float vec __attribute__((ext_vector_type(DPL)));
            vec o;
#pragma unroll
            for (int j = 0; j < DPL; j++) o[j] = x[j];
            *reinterpret_cast<vec*>(static_cast<float*>(a.q_out) + at) = o;
        } else {
            typedef uint32_t vec __attribute__((ext_vector_type(DPL / 2)));
            vec o;
#pragma unroll
            for (int j = 0; j < DPL; j += 2) {
                if constexpr (DPL == 2) o = vec{pk_bf16(x[0], x[1])};
                else o[j / 2] = pk_bf16(x[j], x[j + 1]);
            }
            *reinterpret_cast<vec*>(static_cast<uint16_t*>(a.q_out) + at) = o;
        }
        return;
    }
    if (!there) return;
    const int64_t blk = paged_block_at(a.c, b, (int)p, h, a.NKV, D);
    if (blk < 0) return;
    typedef f16 f16v __attribute__((ext_vector_type(DPL)));
    f16v o;
#pragma unroll
    for (int j = 0; j < DPL; j++) o[j] = (f16)x[j];
    *reinterpret_cast<f16v*>(reinterpret_cast<f16*>(a.c.k) + blk + k_off((int)p & (kBlk - 1), d0)) = o;
}

template <int D>
hipError_t append_d(const PagedAppendArgs& a, bool bf16, hipStream_t s) {
    const int64_t items = (int64_t)a.n_seq * a.n * ((a.q ? a.NH : 0) + a.NKV);
    const int64_t v_lanes = (int64_t)a.n_seq * a.NKV * paged_groups(a.n) * (D / 8);
    const dim3 grid((unsigned)((items + 7) / 8 + (v_lanes + 255) / 256)), block(256);
    if (bf16) hipLaunchKernelGGL((k_paged_append<D, 1>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((k_paged_append<D, 0>), grid, block, 0, s, a);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_append(const PagedAppendArgs& a, int D, bool bf16, hipStream_t s) {
    if (D == 256) return append_d<256>(a, bf16, s);
    if (D == 128) return append_d<128>(a, bf16, s);
    return append_d<64>(a, bf16, s);
}

size_t paged_workspace(int D, int n_cu) { return std::max(paged_few_workspace(D, n_cu), paged_chunk_workspace(D, n_cu)); }

// Up to 32 query rows a KV head (two matrix tiles) keep memory busier in k_paged_few; k_paged_chunk's 128 or 256 rows of an item
// would mostly be padding. Measured, few and chunk: one fp32 token at 32767 20 and 44 us, 8 sequences of 4 (32 rows) 26 and 40,
// 32 of one bf16 token 109 and 182.
hipError_t launch_paged_attend(const PagedAttendArgs& a, int D, bool bf16, int n_cu, void* workspace, hipStream_t s) {
    if (a.n * (a.NH / a.NKV) <= 32) return launch_paged_few(a, D, bf16, n_cu, workspace, s);
    return launch_paged_chunk(a, D, bf16, n_cu, workspace, s);
}

}  // namespace qw

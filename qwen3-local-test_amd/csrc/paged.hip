// Batches of sequences over a paged K/V cache for gfx950: appending new tokens to their pages, and their attention.
//
// A page holds 2^lg_page positions of every KV head, in the 32-position blocks of common.hpp; table[b] names the
// pages of sequence b. The reference serves one sequence (src/qwen4_vk.cpp:937-996).
#include "paged.hpp"

#include <algorithm>

namespace qw {

namespace {

// Elements before the block of KV head h that holds position p of sequence b; -1 without a page
__device__ __forceinline__ int64_t paged_block_at(const PagedCache& c, int b, int p, int h, int nkv, int D) {
    const int32_t page = c.table[(size_t)b * c.table_stride + (p >> c.lg_page)];
    return (uint32_t)page < (uint32_t)c.n_pages ? paged_block(c, page, p, h, nkv, D) : -1;
}

// ---- append --------------------------------------------------------------------------------------------------
// y = x rsqrt(mean x^2 + eps) (1 + w), rotated, in the lane layout of k_qk_norm_rope (norm_rope.hip): a half-wave a (token, head) row,
// D / 32 dims a lane, some heads one after the other; values by lanes of their own that turn 8 positions x 8 dims into the blocks'
// 16-byte pieces. Bound by memory where there are many tokens (2250 bf16 tokens of 16 + 2 heads of 256, 46.7 MB: 13.8 us, 3.4 TB/s; 8192
// fp32 at 4.7), by a launch and its chain of loads (position, page) where there are few: one token 3.9 us.

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

// PER heads of a token a half-wave: their rows are on their way together, and position, page and rotation are looked up once
template <int D, int DT, int PER>
__global__ __launch_bounds__(256) void k_paged_append(PagedAppendArgs a) {
    constexpr int DPL = D / 32;
    const int hl = threadIdx.x & 31;
    const int q_heads = a.q ? a.NH : 0, heads = q_heads + a.NKV, sets = (heads + PER - 1) / PER;
    const int n_items = a.n_seq * a.n * sets;
    const int norm_blocks = (n_items + 7) / 8;
    if ((int)blockIdx.x >= norm_blocks) {
        paged_v_copy<D, DT>(a, (int64_t)((int)blockIdx.x - norm_blocks) * 256 + threadIdx.x);
        return;
    }
    const int item = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (item >= n_items) return;  // (whole half-waves leave, as below)
    const int row = item / sets, h0 = (item - row * sets) * PER;
    const int b = row / a.n, t = row - b * a.n;
    if (t >= seq_len(a.lens, b, a.n)) return;
    const int d0 = hl * DPL;
    float x[PER][DPL], cs[2 * DPL];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int hh = min(h0 + i, heads - 1);
        const bool is_q = hh < q_heads;
        load_vec<DT, DPL>(is_q ? a.q : a.k, is_q ? (size_t)row * a.q_stride + (size_t)hh * a.q_head + d0
                                                 : (size_t)row * a.k_stride + (size_t)(hh - q_heads) * D + d0, x[i]);
    }
    const int64_t p = (int64_t)a.pos[b] + t;
    const bool there = p >= 0 && p < a.limit;
    const int half_r = a.R >> 1;
    const bool rot = d0 < a.R && there;  // DPL divides R / 2: a lane's dims are all rotated or all not
    const bool low = d0 < half_r;
    if (rot) load_vec<0, 2 * DPL>(a.rope, (size_t)p * a.R + 2 * (low ? d0 : d0 - half_r), cs);
    // rotate-half: the partner dim d +- R / 2 sits (R / 2) / DPL lanes away in the same half-wave
    const int offl = half_r / DPL;
    const int src = (threadIdx.x & 32) + (rot ? (low ? hl + offl : hl - offl) : hl);
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int hh = h0 + i;
        if (hh >= heads) return;
        const bool is_q = hh < q_heads;
        const float* gamma = is_q ? a.qn : a.kn;
        if (gamma) {
            float w[DPL], ss = 0.f;
            load_vec<0, DPL>(gamma, d0, w);
#pragma unroll
            for (int j = 0; j < DPL; j++) ss += x[i][j] * x[i][j];
            const float rn = 1.0f / sqrtf(sum32(ss) / (float)D + a.eps);
#pragma unroll
            for (int j = 0; j < DPL; j++) x[i][j] = x[i][j] * rn * (1.0f + w[j]);
        }
#pragma unroll
        for (int j = 0; j < DPL; j++) {
            const float partner = __shfl(x[i][j], src, 64);
            if (rot) x[i][j] = low ? x[i][j] * cs[2 * j] - partner * cs[2 * j + 1] : x[i][j] * cs[2 * j] + partner * cs[2 * j + 1];
        }
        if (is_q) {
            const size_t at = (size_t)row * a.q_out_stride + (size_t)hh * D + d0;
#pragma unroll
            for (int j = 0; j < DPL; j++) x[i][j] = there ? x[i][j] : 0.f;
            if constexpr (DT == 0) {
                typedef float vec __attribute__((ext_vector_type(DPL)));
                vec o;
#pragma unroll
                for (int j = 0; j < DPL; j++) o[j] = x[i][j];
                *reinterpret_cast<vec*>(static_cast<float*>(a.q_out) + at) = o;
            } else {
                typedef uint32_t vec __attribute__((ext_vector_type(DPL / 2)));
                vec o;
#pragma unroll
                for (int j = 0; j < DPL; j += 2) {
                    if constexpr (DPL == 2) o = vec{pk_bf16(x[i][0], x[i][1])};
                    else o[j / 2] = pk_bf16(x[i][j], x[i][j + 1]);
                }
                *reinterpret_cast<vec*>(static_cast<uint16_t*>(a.q_out) + at) = o;
            }
            continue;
        }
        if (!there) return;
        const int64_t blk = paged_block_at(a.c, b, (int)p, hh - q_heads, a.NKV, D);
        if (blk < 0) return;
        typedef f16 f16v __attribute__((ext_vector_type(DPL)));
        f16v o;
#pragma unroll
        for (int j = 0; j < DPL; j++) o[j] = (f16)x[i][j];
        *reinterpret_cast<f16v*>(reinterpret_cast<f16*>(a.c.k) + blk + k_off((int)p & (kBlk - 1), d0)) = o;
    }
}

template <int D, int DT, int PER>
hipError_t append(const PagedAppendArgs& a, hipStream_t s) {
    const int heads = (a.q ? a.NH : 0) + a.NKV;
    const int64_t items = (int64_t)a.n_seq * a.n * ((heads + PER - 1) / PER);
    const int64_t v_lanes = (int64_t)a.n_seq * a.NKV * paged_groups(a.n) * (D / 8);
    hipLaunchKernelGGL((k_paged_append<D, DT, PER>), dim3((unsigned)((items + 7) / 8 + (v_lanes + 255) / 256)), dim3(256), 0, s, a);
    return hipGetLastError();
}
template <int D>
hipError_t append_d(const PagedAppendArgs& a, bool bf16, hipStream_t s) {
    // Two or four heads a half-wave, kernel time in us: one fp32 token of 16 + 2 heads of 256 3.9 and 4.6, 1024 bf16 8.4 and 8.9, 2250
    // 14.2 and 13.8, 4096 fp32 of 8 + 8 heads of 64 15.7 and 13.0, 2048 bf16 of 32 + 8 of 128 16.8 and 15.6 (with one head 3.8,
    // 9.4, 16.6, 18.9 and 19.6)
    const bool many = (int64_t)a.n_seq * a.n * ((a.q ? a.NH : 0) + a.NKV) > 32768;
    if (bf16) return many ? append<D, 1, 4>(a, s) : append<D, 1, 2>(a, s);
    return many ? append<D, 0, 4>(a, s) : append<D, 0, 2>(a, s);
}

}  // namespace

hipError_t launch_paged_append(const PagedAppendArgs& a, int D, bool bf16, hipStream_t s) {
    if (D == 256) return append_d<256>(a, bf16, s);
    if (D == 128) return append_d<128>(a, bf16, s);
    return append_d<64>(a, bf16, s);
}

size_t paged_workspace(int D, int n_cu) { return std::max(paged_few_workspace(D, n_cu), paged_chunk_workspace(D, n_cu)); }

// Up to 32 query rows a KV head (two matrix tiles) keep memory busier in k_paged_few; k_paged_chunk's 128 or 256 rows of an item
// would mostly be padding. Measured, few and chunk: one fp32 token at 32767 21 and 46 us, 8 sequences of 4 (32 rows) 25 and 42,
// 32 of one bf16 token 110 and 229; 8 of 8 fp32 tokens over 2 KV heads of 128 18 and 41, 24 of one bf16 token over 8 of 64 46 and 156.
// The call's largest token count decides for all its sequences: the single tokens beside a chunk go through k_paged_chunk.
hipError_t launch_paged_attend(const PagedAttendArgs& a, int D, bool bf16, int n_cu, void* workspace, hipStream_t s) {
    if (a.n * (a.NH / a.NKV) <= 32) return launch_paged_few(a, D, bf16, n_cu, workspace, s);
    return launch_paged_chunk(a, D, bf16, n_cu, workspace, s);
}

}  // namespace qw

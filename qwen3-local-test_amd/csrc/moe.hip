// The router and the SwiGLU experts of a mixture-of-experts layer (qwattn_moe_route, qwattn_moe; the reference's
// shaders/moe_route.comp, moe_group.comp, moe_combine.comp and the expert variants of its matmul shaders).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"

namespace qw {

// ---- the router ----------------------------------------------------------------------------------------------
// A wave a token (4,096 tokens, 10 of 512 experts: 8 us; bound by vector instructions, 837 a token, which issue in 74% of
// a CU's busy cycles; one token: 2.9 us, its wave waiting 82% of its cycles). Lane l holds the PER consecutive experts
// from l * PER, so among equal logits the first lane (and in it the first value) has the lowest index: each of the top_k
// rounds is a wave maximum, a ballot and the removal of one value. -inf and NaN are no choice.
// Equal to the maximum counts as e^0 also where both are +inf.
template <int PER>
__global__ __launch_bounds__(256) void k_moe_route(RouteArgs a) {
    const int tok = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (tok >= a.n) return;
    const float* row = a.logits + (size_t)tok * a.stride;
    float v[PER];
    if (PER >= 4 && a.whole) {  // all of the lanes' values there, in 16-byte pieces
#pragma unroll
        for (int i = 0; i < PER / 4; i++) {
            const f32x4 w = *reinterpret_cast<const f32x4*>(row + lane * PER + 4 * i);
            v[4 * i] = w[0], v[4 * i + 1] = w[1], v[4 * i + 2] = w[2], v[4 * i + 3] = w[3];
        }
    } else {
#pragma unroll
        for (int i = 0; i < PER; i++) v[i] = lane * PER + i < a.n_experts ? row[lane * PER + i] : kNegInf;
    }
#pragma unroll
    for (int i = 0; i < PER; i++)
        if (v[i] != v[i]) v[i] = kNegInf;
    float best = v[0];
#pragma unroll
    for (int i = 1; i < PER; i++) best = fmaxf(best, v[i]);
    const float top = max64(best);
    float all = 0.f;
    if (!a.renorm) {
#pragma unroll
        for (int i = 0; i < PER; i++) all += v[i] == kNegInf ? 0.f : v[i] == top ? 1.f : expf(v[i] - top);
        all = sum64(all);
    }
    float mine = kNegInf;  // lane j: the j-th choice
    int id = -1;
    for (int j = 0; j < a.top_k; j++) {
        const float m = max64(best);
        if (m == kNegInf) break;
        const int src = __builtin_ctzll(__ballot(best == m));
        int at = 0;
        if (lane == src) {
#pragma unroll
            for (int i = PER - 1; i >= 0; i--) at = v[i] == m ? i : at;
#pragma unroll
            for (int i = 0; i < PER; i++) v[i] = i == at ? kNegInf : v[i];
            best = v[0];
#pragma unroll
            for (int i = 1; i < PER; i++) best = fmaxf(best, v[i]);
        }
        at = __builtin_amdgcn_readlane(at, src) + src * PER;
        if (lane == j) mine = m, id = at;
    }
    const float p = id < 0 ? 0.f : mine == top ? 1.f : expf(mine - top);
    if (a.renorm) all = sum64(p);
    if (lane < a.top_k) {
        a.ids[(size_t)tok * a.top_k + lane] = id;
        a.weights[(size_t)tok * a.top_k + lane] = id < 0 ? 0.f : p / all;
    }
}

hipError_t launch_moe_route(RouteArgs a, hipStream_t s) {
    const int grid = (a.n + 3) / 4;
    a.whole = (a.n_experts == 256 || a.n_experts == 512 || a.n_experts == 1024) && a.stride % 4 == 0 &&
              ((uintptr_t)a.logits & 15) == 0;
    if (a.n_experts <= 64) k_moe_route<1><<<grid, 256, 0, s>>>(a);
    else if (a.n_experts <= 128) k_moe_route<2><<<grid, 256, 0, s>>>(a);
    else if (a.n_experts <= 256) k_moe_route<4><<<grid, 256, 0, s>>>(a);
    else if (a.n_experts <= 512) k_moe_route<8><<<grid, 256, 0, s>>>(a);
    else k_moe_route<16><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

// ---- the experts, pair by pair -------------------------------------------------------------------------------
// h[pair][f] = silu(W_gate x) (W_up x) of the pair's expert, then y[t] = sum over its pairs of weight W_down h:
// a wave a row of the weights, 16 columns a lane at a time (half a Q8 block: one scale), fp32 products. One token, 8 of 128
// experts of 2,048 x 512: 7.4 + 5.9 us, waves waiting three quarters of their cycles for their few loads (vector
// instructions 23% and 17% of the busy cycles); 10 of 13 tokens: 33 + 24 us, waiting 73% and 61% behind 3.8 TB/s, vector
// instructions 52% and 53%.

// sum over 16 int8 weights (a word each four) with their values
__device__ __forceinline__ float dot16(const u32x4 w, const float (&x)[16]) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) s = fmaf((float)((int)(w[k] << (24 - 8 * e)) >> 24), x[4 * k + e], s);
    return s;
}

constexpr int kPairRows = 2;  // rows a wave

template <int DT>
__global__ __launch_bounds__(256) void k_moe_pair_up(MoeArgs a) {
    const int pair = blockIdx.x, lane = threadIdx.x & 63;
    const int e = a.ids[pair];
    if (e < 0 || e >= a.n_experts) return;
    const int f0 = (blockIdx.y * 4 + (threadIdx.x >> 6)) * kPairRows;
    const size_t xrow = (size_t)(pair / a.top_k) * a.x_stride;
    float g[kPairRows] = {}, u[kPairRows] = {};
    for (int c = lane * 16; c < a.hidden; c += 1024) {
        float x[16];
        load_vec<DT, 16>(a.x, xrow + c, x);
#pragma unroll
        for (int i = 0; i < kPairRows; i++) {
            if (f0 + i >= a.ffn) break;
            const size_t at = ((size_t)e * a.ffn + f0 + i) * a.hidden + c;
            g[i] = fmaf(dot16(*reinterpret_cast<const u32x4*>(a.w_gate + at), x), a.s_gate[at >> 5], g[i]);
            u[i] = fmaf(dot16(*reinterpret_cast<const u32x4*>(a.w_up + at), x), a.s_up[at >> 5], u[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < kPairRows; i++) {
        const float gs = sum64(g[i]), us = sum64(u[i]);
        if (lane == 0 && f0 + i < a.ffn) a.h[(size_t)pair * a.ffn + f0 + i] = gs * sigmoid(gs) * us;
    }
}

// (a token's pairs one after the other make one row of top_k x ffn columns: ffn is often half a wave's 1,024. Decode of 8
// experts of 512: 8.9 us with a pair at a time)
template <int DT>
__global__ __launch_bounds__(256) void k_moe_pair_down(MoeArgs a) {
    const int tok = blockIdx.x, lane = threadIdx.x & 63;
    const int r0 = (blockIdx.y * 4 + (threadIdx.x >> 6)) * kPairRows;
    const int per = a.ffn >> 4, pieces = a.top_k * per;  // of 16 columns
    float y[kPairRows] = {};
#pragma unroll 4
    for (int p = lane; p < pieces; p += 64) {
        const int j = p / per, c = (p - j * per) * 16, pair = tok * a.top_k + j, e = a.ids[pair];
        if (e < 0 || e >= a.n_experts) continue;
        const float wt = a.weights[pair];
        float h[16];
        load_vec<0, 16>(a.h, (size_t)pair * a.ffn + c, h);
#pragma unroll
        for (int i = 0; i < kPairRows; i++) {
            const size_t at = ((size_t)e * a.hidden + min(r0 + i, a.hidden - 1)) * a.ffn + c;
            y[i] = fmaf(wt * a.s_down[at >> 5], dot16(*reinterpret_cast<const u32x4*>(a.w_down + at), h), y[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < kPairRows; i++) {
        const float s = sum64(y[i]);
        if (lane == 0 && r0 + i < a.hidden) {
            const size_t at = (size_t)tok * a.y_stride + r0 + i;
            if constexpr (DT == 0) static_cast<float*>(a.y)[at] = s;
            else static_cast<__bf16*>(a.y)[at] = (__bf16)s;
        }
    }
}

// ---- the experts, grouped: pairs sorted by expert, tiled products on the matrix cores ------------------------
// k_moe_begin sorts the pairs by expert, lists tiles of BM rows of one expert and writes x as fp16 operands (k_moe_mid: h);
// k_moe_gemm multiplies a tile's rows with 64 gate and the same 64 up rows of its expert's weights (or 128 down
// rows); k_moe_combine sums a token's pairs in their order.
//
// Operands: an int8 weight is exact in fp16. A row of activations is scaled by the power of two that puts its largest
// magnitude into [2^14, 2^15) and becomes the sum of two fp16 (11 bits each: within 2^-23 of the value; below 2^-2, where
// the second has steps of 2^-24, within 2^-25, 2^-39 of the row's largest). A bf16 x is exact in one from 2^-17 on, below
// that within the same 2^-25. fp32 operands would take a third part and half as many matrix instructions again, for values
// 2^-39 of their row's largest. The block scales multiply each 32-column product in fp32.

struct MoeTile {
    int expert, row, rows;
};
struct MoeWs {
    MoeTile* tiles;
    int *row_tok, *pair_row;   // sorted row -> token, pair -> sorted row (-1: no expert)
    float* row_weight;         // sorted row -> its pair's weight
    int *x_shift, *h_shift;    // powers of two of the operand rows
    f16 *x16, *h16;            // operands [part][row][columns up to a multiple of 64]
    size_t x_part, h_part;     // elements of a part
    float* h;                  // [row][ffn]
    float* y;                  // [row][hidden]
    int max_tiles;             // tiles in use: pairs / BM + n_experts, some of them without rows
};

// The sort, a workgroup an expert: it counts the pairs of lower experts (its first row) and its own, and writes its own down
// in their order; a wave goes through a sixteenth of the ids, 64 x kSortIds at a time. (One workgroup with counters in the
// LDS took 28 us for 16,384 pairs.) An expert whose rows start at r has the tiles from r / BM + expert on: apart from
// every other expert's without knowing their counts; the ones it does not need, up to the next expert's, get no rows.
constexpr int kSortIds = 16;

__device__ __forceinline__ void moe_sort(const MoeArgs& a, const MoeWs& ws, int bm, int e) {
    __shared__ int own[16], low[16];
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, pairs = a.n * a.top_k;
    const int per = (pairs + 15) / 16, first = wave * per, last = min(first + per, pairs);
    int id[kSortIds];
    auto load = [&](int i0) {  // -1 past the wave's part
#pragma unroll
        for (int u = 0; u < kSortIds; u++) {
            const int i = i0 + u * 64 + lane, v = a.ids[min(i, pairs - 1)];
            id[u] = i < last ? v : -1;
        }
    };
    int n_own = 0, n_low = 0;
    for (int i0 = first; i0 < last; i0 += 64 * kSortIds) {
        load(i0);
#pragma unroll
        for (int u = 0; u < kSortIds; u++) {
            n_own += __builtin_popcountll(__ballot(id[u] == e));
            n_low += __builtin_popcountll(__ballot(id[u] >= 0 && id[u] < e));
        }
    }
    if (lane == 0) own[wave] = n_own, low[wave] = n_low;
    __syncthreads();
    int row0 = 0, rows = 0, at = 0;
#pragma unroll
    for (int w = 0; w < 16; w++) {
        row0 += low[w], rows += own[w];
        if (w < wave) at += own[w];
    }
    at += row0;
    const int t0 = row0 / bm + e, t1 = e == a.n_experts - 1 ? ws.max_tiles : (row0 + rows) / bm + e + 1;
    for (int t = t0 + threadIdx.x; t < t1; t += 1024)
        ws.tiles[t] = MoeTile{e, row0 + (t - t0) * bm, max(0, min(bm, rows - (t - t0) * bm))};
    if (rows == 0) return;
    for (int i0 = first; i0 < last; i0 += 64 * kSortIds) {
        if (last - first > 64 * kSortIds) load(i0);
#pragma unroll
        for (int u = 0; u < kSortIds; u++) {
            const uint64_t hit = __ballot(id[u] == e);
            if (hit == 0) continue;
            if (id[u] == e) {
                const int i = i0 + u * 64 + lane, r = at + __builtin_popcountll(hit & ((1ull << lane) - 1));
                ws.pair_row[i] = r, ws.row_tok[r] = i / a.top_k, ws.row_weight[r] = a.weights[i];
            }
            at += __builtin_popcountll(hit);
        }
    }
}

// A row of activations as fp16 operands: out[part][row][padded], zeros from `cols` on, and its power of two. 256 lanes a
// row, `lane` of them this one; `most`: four floats of the LDS.
template <int DT, int P>
__device__ __forceinline__ void moe_row(const void* x, size_t stride, int cols, int padded, f16* out, size_t part, int* shift,
                                        size_t row, int lane, float* most, bool there) {
    float v[8], m = 0.f;
    if (there)
        for (int c = lane * 8; c < cols; c += 2048) {
            load_vec<DT, 8>(x, row * stride + c, v);
#pragma unroll
            for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(v[i]));
        }
    m = max64(m);
    if ((lane & 63) == 0) most[lane >> 6] = m;
    __syncthreads();
    if (!there) return;
    m = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
    // (a row with an infinity, or of zeros, is not scaled)
    const int up = m > 0.f && m < __builtin_inff() ? 15 - __builtin_amdgcn_frexp_expf(m) : 0;
    if (lane == 0) shift[row] = up;
    for (int c = lane * 8; c < padded; c += 2048) {
        f16x8 hi = {}, lo = {};
        if (c < cols) {
            load_vec<DT, 8>(x, row * stride + c, v);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float s = ldexpf(v[i], up);
                hi[i] = (f16)s;
                lo[i] = fabsf(s) == __builtin_inff() ? (f16)0.f : (f16)(s - (float)hi[i]);
            }
        }
        *reinterpret_cast<f16x8*>(out + row * padded + c) = hi;
        if constexpr (P == 2) *reinterpret_cast<f16x8*>(out + part + row * padded + c) = lo;
    }
}

// The first n_experts workgroups sort; the others write four rows of x each, and mark their pairs without an expert.
template <int DT, int P>
__global__ __launch_bounds__(1024) void k_moe_begin(MoeArgs a, MoeWs ws, int bm) {
    __shared__ float most[4][4];
    if ((int)blockIdx.x < a.n_experts) {
        moe_sort(a, ws, bm, blockIdx.x);
        return;
    }
    const int sub = threadIdx.x >> 8, lane = threadIdx.x & 255;
    const size_t row = (size_t)(blockIdx.x - a.n_experts) * 4 + sub;
    const bool there = row < (size_t)a.n;
    if (there && lane < a.top_k) {
        const size_t i = row * a.top_k + lane;
        if (a.ids[i] < 0 || a.ids[i] >= a.n_experts) ws.pair_row[i] = -1;
    }
    moe_row<DT, P>(a.x, a.x_stride, a.hidden, (a.hidden + 63) & ~63, ws.x16, ws.x_part, ws.x_shift, row, lane, most[sub], there);
}
// Rows of h.
__global__ __launch_bounds__(256) void k_moe_mid(MoeArgs a, MoeWs ws) {
    __shared__ float most[4];
    moe_row<0, 2>(ws.h, a.ffn, a.ffn, (a.ffn + 63) & ~63, ws.h16, ws.h_part, ws.h_shift, blockIdx.x, threadIdx.x, most, true);
}

__device__ __forceinline__ f32x16 mfma32h(f16x8 a, f16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Four int8 weights (a word) as fp16, exactly: 0x64xx is 1024 + xx
__device__ __forceinline__ void weights_f16(uint32_t w, f16x2& a, f16x2& b) {
    w ^= 0x80808080u;
    const f16x2 off = {(f16)1152.f, (f16)1152.f};
    a = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u)) - off;
    b = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u)) - off;
}

constexpr int kMoeGroup = 4;  // M tiles whose column tiles follow each other on an XCD

// P parts of the activations, tiles of MT x 32 rows by 128 weight rows, 64 columns a step. Four waves share out the weight
// rows, 32 each, so that each int8 weight is converted by one wave. The LDS takes operands as they come from memory, by
// direct loads: ST stages of activations [part][BM][128 bytes], ST - 1 steps ahead; two of int8 weights [BN][128 columns];
// two of scales [BN][8 blocks]; rows are read by whole lines where they can be, so that fewer requests go to L2. Bound by
// no one unit: 2,048 tokens of 8 of 128 experts, gate and up, 181-208 us at 2.0 GHz, of a CU's busy cycles vector
// instructions 54% (the conversion, the block scales), the matrix pipe 24%, the LDS 18%.
template <int P, int MT, int ST>
struct MoeTileShape {
    static constexpr int kThreads = 256, BM = MT * 32, BN = 128;
    static constexpr int kA = P * BM * 128, kW = BN * 128, kS = BN * 8 * 4;
    static constexpr int kAtW = ST * kA, kAtS = kAtW + 2 * kW, kAtRows = kAtS + 2 * kS, kLds = kAtRows + BM * 8;
    static constexpr int AL = kA / 4096, WL = kW / 4096, SL = kS / 1024;  // direct loads a wave: 1 KB (scales: 256 bytes) each
    static_assert(AL * 4096 == kA, "whole loads");
};

// A lane's 16 (4) bytes to the LDS at `to` (uniform) + 16 (4) x lane
__device__ __forceinline__ void load16_to_lds(const void* from, uint8_t* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                     (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}
__device__ __forceinline__ void load4_to_lds(const void* from, uint8_t* to) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from,
                                     (__attribute__((address_space(3))) void*)to, 4, 0, 0);
}

template <int P, int MT, int ST, bool UP>
__global__ __launch_bounds__(256, 2) void k_moe_gemm(MoeArgs a, MoeWs ws) {
    typedef MoeTileShape<P, MT, ST> T;
    constexpr int BM = T::BM, BN = T::BN;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    // Groups of four M tiles (mostly one expert's) on one XCD, column tile after column tile: the group's weights come once
    // from memory, its rows once, then from that XCD's L2.
    const int outs = UP ? a.ffn : a.hidden, cols = UP ? a.hidden : a.ffn, per = UP ? BN / 2 : BN;
    const int nn = (outs + per - 1) / per, seq = blockIdx.x >> 3, in = seq % (nn * kMoeGroup);
    const int tile = (seq / (nn * kMoeGroup) * 8 + (blockIdx.x & 7)) * kMoeGroup + in % kMoeGroup, n0 = in / kMoeGroup * per;
    if (tile >= ws.max_tiles) return;
    const MoeTile mt = ws.tiles[tile];
    if (mt.rows == 0) return;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int c = lane & 31, h = lane >> 5;
    const int padded = (cols + 63) & ~63, nkb = cols >> 5, steps = padded >> 6;

    // 16-byte piece q of a 128-byte row r lies at q ^ (r / 2) % 8, so that operand reads (16 rows' piece q) spread over the
    // banks; the eight lanes that fill a row load its line in that order
    auto turn = [](int r) { return (r >> 1) & 7; };
    const int lr = lane >> 3, lq = lane & 7;  // of a direct load: row and place
    // weight row r of the tile: UP: of each 32, 16 gate rows and the same 16 up rows
    auto weight_row = [&](int r) {
        const int o = UP ? n0 + (r >> 5) * 16 + (r & 15) : n0 + r;
        return (size_t)mt.expert * outs + min(o, outs - 1);
    };
    const f16* ap[T::AL];
#pragma unroll
    for (int i = 0; i < T::AL; i++) {
        const int at = (wave * T::AL + i) * 8 + lr, r = at % BM, part = at / BM;
        const int row = mt.row + min(r, mt.rows - 1);  // (rows past the tile's: the last one's, their results unused)
        ap[i] = (UP ? ws.x16 + (size_t)ws.row_tok[row] * padded + (part ? ws.x_part : 0)
                    : ws.h16 + (size_t)row * padded + (part ? ws.h_part : 0)) + (lq ^ turn(r)) * 8;
    }
    const int8_t* wp[T::WL];
    int wcol[T::WL];
#pragma unroll
    for (int i = 0; i < T::WL; i++) {
        const int r = (wave * T::WL + i) * 8 + lr;
        wp[i] = (UP ? (r & 16 ? a.w_up : a.w_gate) : a.w_down) + weight_row(r) * cols;
        wcol[i] = (lq ^ turn(r)) * 16;
    }
    const float* sp[T::SL];
#pragma unroll
    for (int i = 0; i < T::SL; i++) {
        const int r = (wave * T::SL + i) * 8 + lr;
        sp[i] = (UP ? (r & 16 ? a.s_up : a.s_gate) : a.s_down) + weight_row(r) * nkb;
    }
    auto load_a = [&](int k, int stage) {
#pragma unroll
        for (int i = 0; i < T::AL; i++)
            load16_to_lds(ap[i] + min(k, steps - 1) * 64, smem + stage * T::kA + (wave * T::AL + i) * 1024);
    };
    // (past the row: any weights and scales, on the operands' zeros or in steps that do not run)
    auto load_w = [&](int m, int buffer) {  // columns 128 m ..
#pragma unroll
        for (int i = 0; i < T::WL; i++) {
            const int col = m * 128 + wcol[i];
            load16_to_lds(wp[i] + (col < cols ? col : 0), smem + T::kAtW + buffer * T::kW + (wave * T::WL + i) * 1024);
        }
    };
    auto load_s = [&](int m, int buffer) {  // blocks 8 m ..
#pragma unroll
        for (int i = 0; i < T::SL; i++)
            load4_to_lds(sp[i] + min(m * 8 + lq, nkb - 1), smem + T::kAtS + buffer * T::kS + (wave * T::SL + i) * 256);
    };

    f32x16 acc[MT];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int e = 0; e < 16; e++) acc[m][e] = 0.f;
    load_w(0, 0), load_s(0, 0), load_a(0, 0);
    if (ST == 3) load_a(1, 1);
    // Of a row, for the results: its power of two and (down) its weight. After the first loads, before the last waits.
    int* sShift = reinterpret_cast<int*>(smem + T::kAtRows);
    float* sWeight = reinterpret_cast<float*>(sShift + BM);
    if (tid < BM) {
        const int row = mt.row + min(tid, mt.rows - 1);
        sShift[tid] = -(UP ? ws.x_shift[ws.row_tok[row]] : ws.h_shift[row]);
        if (!UP) sWeight[tid] = ws.row_weight[row];
    }
    f32x16 zero = {};
    asm volatile("" : "+v"(zero));  // registers of zeros: a constant would be written into every accumulator anew
    // Four steps at a time (256 columns: a load of scales, two of weights). Step s loads activations first, then the next
    // weights (s = 0, 2) and scales (s = 0): what of a step's loads may still be on its way at the next step's start is
    // all of them (three stages) or those behind the activations.
    constexpr int kNew[4] = {T::WL + T::SL, 0, T::WL, 0};
    int stage = 0, sbuf = 0;
#pragma unroll 1
    for (int k0 = 0; k0 < steps; k0 += 4) {
        static_for<0, 4>([&](auto s_) {
            constexpr int s = s_, kFly = kNew[(s + 3) & 3] + (ST == 3 ? T::AL : 0);
            const int k = k0 + s;
            if (k >= steps) return;  // uniform
            // this step's loads have landed, in every wave, and the last step's reads have ended
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kFly) : "memory");
            const int to = ST == 3 ? (stage == 0 ? 2 : stage - 1) : stage ^ 1;
            load_a(k + ST - 1, to);
            if constexpr (s % 2 == 0) load_w((k >> 1) + 1, s == 0 ? 1 : 0);
            if constexpr (s == 0) load_s((k >> 2) + 1, sbuf ^ 1);
            const uint8_t* A = smem + stage * T::kA;
            const uint8_t* W = smem + T::kAtW + (s >> 1) * T::kW;
            const float* sS = reinterpret_cast<const float*>(smem + T::kAtS + sbuf * T::kS);
            stage = ST == 3 ? (stage == 2 ? 0 : stage + 1) : stage ^ 1;
            // Tile by tile of the step's two blocks, the scaled sum of one behind the matrix instructions of the next, so
            // that a wave's vector and matrix instructions run side by side.
            constexpr int NT = 2 * MT;
            f16x8 w[2][2], x[2][MT][P][2];
            float sc[2];
            f32x16 d[2];
            const int wr = wave * 32 + c;
#pragma unroll
            for (int j = 0; j < 2; j++) {
                // lane half h takes 16 columns of the block, product q of the two their eights
                const u32x4 v = *reinterpret_cast<const u32x4*>(W + wr * 128 + (((4 * (s & 1) + 2 * j + h) ^ turn(wr)) << 4));
                sc[j] = sS[wr * 8 + 2 * s + j];
#pragma unroll
                for (int m = 0; m < MT; m++)
#pragma unroll
                    for (int p = 0; p < P; p++)
#pragma unroll
                        for (int q = 0; q < 2; q++) {
                            const int r = m * 32 + c;
                            x[j][m][p][q] =
                                *reinterpret_cast<const f16x8*>(A + (p * BM + r) * 128 + (((4 * j + 2 * h + q) ^ turn(r)) << 4));
                        }
#pragma unroll
                for (int q = 0; q < 2; q++) {
                    f16x2 p[4];
                    weights_f16(v[2 * q], p[0], p[1]), weights_f16(v[2 * q + 1], p[2], p[3]);
#pragma unroll
                    for (int e = 0; e < 4; e++) w[j][q][2 * e] = p[e][0], w[j][q][2 * e + 1] = p[e][1];
                }
            }
            static_for<0, NT + 1>([&](auto i_) {
                constexpr int i = i_, j = i / MT, m = i % MT;
                if constexpr (i < NT)
#pragma unroll
                    for (int p = P - 1; p >= 0; p--)
#pragma unroll
                        for (int q = 0; q < 2; q++)
                            d[i & 1] = mfma32h(x[j][m][p][q], w[j][q], p == P - 1 && q == 0 ? zero : d[i & 1]);
                if constexpr (i > 0) {
                    constexpr int j1 = (i - 1) / MT, m1 = (i - 1) % MT;
#pragma unroll
                    for (int e = 0; e < 16; e++) acc[m1][e] = fmaf(sc[j1], d[(i - 1) & 1][e], acc[m1][e]);
                }
                __builtin_amdgcn_sched_barrier(0);
            });
        });
        sbuf ^= 1;
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    // lane (c, h): weight row c of a tile, activation rows 8 (e / 4) + 4 h + e % 4. Stores past the tile's rows, or past the
    // last column, lie outside the resource.
    float* out = (UP ? ws.h : ws.y) + (size_t)mt.row * outs;
    const __amdgpu_buffer_rsrc_t ro = __builtin_amdgcn_make_buffer_rsrc(out, (short)0, mt.rows * outs * 4, 0x00020000);
    const int o = UP ? n0 + wave * 16 + (c & 15) : n0 + wave * 32 + c;
    const unsigned col = o < outs ? o * 4u : kFar;
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int e4 = 0; e4 < 4; e4++) {
            typedef int i32x4 __attribute__((ext_vector_type(4)));
            const int r0 = m * 32 + 8 * e4 + 4 * h;
            const i32x4 s = *reinterpret_cast<const i32x4*>(sShift + r0);
            if constexpr (UP) {
                // the lane pair (c, c + 16) holds a gate and an up value: the first takes one row of two, the second the other
#pragma unroll
                for (int e = 0; e < 4; e += 2) {
                    const uint32_t a0 = __float_as_uint(acc[m][4 * e4 + e]), a1 = __float_as_uint(acc[m][4 * e4 + e + 1]);
                    const auto p0 = __builtin_amdgcn_permlane16_swap(a0, a0, false, false);
                    const auto p1 = __builtin_amdgcn_permlane16_swap(a1, a1, false, false);
                    const bool odd = c & 16;
                    const int sh = odd ? s[e + 1] : s[e];
                    const float g = ldexpf(__uint_as_float(odd ? p1[0] : p0[0]), sh);
                    const float u = ldexpf(__uint_as_float(odd ? p1[1] : p0[1]), sh);
                    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(g * sigmoid(g) * u), ro,
                                                          (int)((unsigned)(r0 + e + (odd ? 1 : 0)) * outs * 4u + col), 0, 0);
                }
            } else {
                const f32x4 wt = *reinterpret_cast<const f32x4*>(sWeight + r0);
#pragma unroll
                for (int e = 0; e < 4; e++)
                    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(wt[e] * ldexpf(acc[m][4 * e4 + e], s[e])), ro,
                                                          (int)((unsigned)(r0 + e) * outs * 4u + col), 0, 0);
            }
        }
}

// y[t] = the sum of the token's pairs, in their order; four channels a lane.
template <int DT>
__global__ __launch_bounds__(256) void k_moe_combine(MoeArgs a, MoeWs ws) {
    const int o = (blockIdx.y * 256 + threadIdx.x) * 4;
    const size_t tok = blockIdx.x;
    if (o >= a.hidden) return;
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
    for (int j = 0; j < a.top_k; j++) {
        const int r = ws.pair_row[tok * a.top_k + j];
        if (r < 0) continue;
        const f32x4 v = *reinterpret_cast<const f32x4*>(ws.y + (size_t)r * a.hidden + o);
#pragma unroll
        for (int e = 0; e < 4; e++) s[e] += v[e];
    }
    if constexpr (DT == 0) {
        *reinterpret_cast<f32x4*>(static_cast<float*>(a.y) + tok * a.y_stride + o) = s;
    } else {
        *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.y) + tok * a.y_stride + o) =
            u32x2{pk_bf16(s[0], s[1]), pk_bf16(s[2], s[3])};
    }
}

// ---- which form -----------------------------------------------------------------------------------------------
// Pair by pair while that takes less: a pair costs 0.09 us a million weights and 0.1 us a thousand weight rows (hidden and
// ffn; 6 us beside them), the grouped form 20 us and 0.26 us a million weights of each expert that is hit. Measured, by
// pairs and grouped: 8 of 128 experts of 2,048 x 512: 16 tokens 88 and 99 us, 32 tokens 154 and 122; 2 of 8 of 1,024 x
// 352: 32 tokens 22 and 30, 64 tokens 36 and 30; 2 of 16 of 256 x 96: 250 tokens 26 and 21; 2 of 4 of 64 x 32: 500 tokens
// 18 and 20, 1,000 tokens 28 and 21.
static bool by_pairs(const MoeArgs& a) {
    const double pairs = (double)a.n * a.top_k, weights = 3e-6 * a.hidden * a.ffn;
    return 6 + pairs * (0.09 * weights + 1e-4 * (a.hidden + a.ffn)) <= 20 + 0.26 * weights * std::min(pairs, (double)a.n_experts);
}
// Rows of a tile: 64 where a mean expert has this many rows, else 32. Measured with 8 of 128 experts of 2,048 x 512, bf16:
// 48 rows an expert 221 us in tiles of 64 and 208 of 32, 64 rows 237 and 243, 128 rows 363 and 387.
constexpr int kTileRows64 = 56;

constexpr int kMoeSegment = 1 << 16;  // pairs worked off at a time: bounds the workspace
static int segment_tokens(const MoeArgs& a) { return std::max(1, std::min(a.n, kMoeSegment / a.top_k)); }

// Bytes of the grouped form's workspace; the pointers into it with `base`.
static size_t lay_out(const MoeArgs& a, int parts, uint8_t* base, MoeWs& w) {
    const size_t n = segment_tokens(a), pairs = n * a.top_k, hp = (a.hidden + 63) & ~63, fp = (a.ffn + 63) & ~63;
    size_t at = 0;
    auto take = [&](auto*& p, size_t bytes) {
        p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(reinterpret_cast<uintptr_t>(base) + at);
        at += up256(bytes);
    };
    take(w.tiles, (pairs / 32 + a.n_experts) * sizeof(MoeTile));
    take(w.row_tok, pairs * 4), take(w.pair_row, pairs * 4), take(w.row_weight, pairs * 4);
    take(w.x_shift, n * 4), take(w.h_shift, pairs * 4);
    take(w.x16, parts * n * hp * 2), take(w.h16, 2 * pairs * fp * 2);
    w.x_part = n * hp, w.h_part = pairs * fp;
    take(w.y, pairs * std::max(a.hidden, a.ffn) * 4);
    w.h = w.y;  // h is read for the last time before y is written
    return at;
}

size_t moe_workspace(const MoeArgs& a, bool bf16) {
    if (by_pairs(a)) return (size_t)a.n * a.top_k * a.ffn * 4;
    MoeWs w;
    return lay_out(a, bf16 ? 1 : 2, nullptr, w);
}

template <int DT>
static hipError_t moe_pairs(const MoeArgs& a, hipStream_t s) {
    const int per = 4 * kPairRows;
    k_moe_pair_up<DT><<<dim3(a.n * a.top_k, (a.ffn + per - 1) / per), 256, 0, s>>>(a);
    k_moe_pair_down<DT><<<dim3(a.n, (a.hidden + per - 1) / per), 256, 0, s>>>(a);
    return hipGetLastError();
}

template <int P, int MT, int ST, bool UP>
static hipError_t moe_gemm(const MoeArgs& a, const MoeWs& w, hipStream_t s) {
    typedef MoeTileShape<P, MT, ST> T;
    static std::atomic<uint64_t> raised{0};
    const auto k = &k_moe_gemm<P, MT, ST, UP>;
    if (const hipError_t e = raise_lds(reinterpret_cast<const void*>(k), T::kLds, raised)) return e;
    const int outs = UP ? a.ffn : a.hidden, per = UP ? T::BN / 2 : T::BN;
    const int round = 8 * kMoeGroup;
    k<<<(w.max_tiles + round - 1) / round * round * ((outs + per - 1) / per), T::kThreads, T::kLds, s>>>(a, w);
    return hipGetLastError();
}

template <int MT, int DT>
static hipError_t moe_tiles(const MoeArgs& a, MoeWs w, hipStream_t s) {
    // as many stages of activations as leave a CU two workgroups
    constexpr int P = DT ? 1 : 2, ST = P * MT > 2 ? 2 : 3, ST2 = MT > 1 ? 2 : 3;
    w.max_tiles = a.n * a.top_k / (MT * 32) + a.n_experts;
    k_moe_begin<DT, P><<<a.n_experts + (a.n + 3) / 4, 1024, 0, s>>>(a, w, MT * 32);
    if (const hipError_t e = moe_gemm<P, MT, ST, true>(a, w, s)) return e;
    k_moe_mid<<<a.n * a.top_k, 256, 0, s>>>(a, w);
    if (const hipError_t e = moe_gemm<2, MT, ST2, false>(a, w, s)) return e;
    k_moe_combine<DT><<<dim3(a.n, (a.hidden + 1023) / 1024), 256, 0, s>>>(a, w);
    return hipGetLastError();
}

template <int DT>
static hipError_t moe_grouped(MoeArgs a, uint8_t* workspace, hipStream_t s) {
    constexpr int kSize = DT ? 2 : 4;
    MoeWs w;
    lay_out(a, DT ? 1 : 2, workspace, w);
    const int seg = segment_tokens(a), n = a.n;
    for (int t = 0; t < n; t += seg) {
        MoeArgs b = a;
        b.n = std::min(seg, n - t);
        b.x = static_cast<const uint8_t*>(a.x) + (size_t)t * a.x_stride * kSize;
        b.y = static_cast<uint8_t*>(a.y) + (size_t)t * a.y_stride * kSize;
        b.ids = a.ids + (size_t)t * a.top_k, b.weights = a.weights + (size_t)t * a.top_k;
        const long long rows = (long long)b.n * a.top_k / a.n_experts;  // a mean expert's
        hipError_t e;
        if (rows >= kTileRows64) e = moe_tiles<2, DT>(b, w, s);
        else e = moe_tiles<1, DT>(b, w, s);
        if (e) return e;
    }
    return hipSuccess;
}

template <int DT>
static hipError_t moe_any(MoeArgs a, void* workspace, hipStream_t s) {
    if (!by_pairs(a)) return moe_grouped<DT>(a, static_cast<uint8_t*>(workspace), s);
    a.h = static_cast<float*>(workspace);
    return moe_pairs<DT>(a, s);
}
hipError_t launch_moe(MoeArgs a, bool bf16, void* workspace, hipStream_t s) {
    return bf16 ? moe_any<1>(a, workspace, s) : moe_any<0>(a, workspace, s);
}

}  // namespace qw

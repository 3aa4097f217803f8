// The router and the SwiGLU experts of a mixture-of-experts layer (qwattn_moe_route, qwattn_moe; the reference's
// shaders/moe_route.comp, moe_group.comp, moe_combine.comp and the expert variants of its matmul shaders).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "common.hpp"
#include "kernels.hpp"

namespace qw {

__device__ __forceinline__ float moe_wave_sum(float x) {
    x = sum32(x);
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
}
__device__ __forceinline__ float moe_wave_max(float x) {
    x = max32(x);
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
}

// ---- the router ----------------------------------------------------------------------------------------------
// A wave a token. Lane l holds the PER consecutive experts from l * PER, so among equal logits the first lane (and
// in it the first value) has the lowest index: each of the top_k rounds is a wave maximum, a ballot and the removal
// of one value. -inf and NaN are no choice. Equal to the maximum counts as e^0 also where both are +inf.
template <int PER>
__global__ __launch_bounds__(256) void k_moe_route(RouteArgs a) {
    const int tok = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (tok >= a.n) return;
    const float* row = a.logits + (size_t)tok * a.stride;
    float v[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const int e = lane * PER + i;
        v[i] = e < a.n_experts ? row[e] : kNegInf;
        if (v[i] != v[i]) v[i] = kNegInf;
    }
    float best = v[0];
#pragma unroll
    for (int i = 1; i < PER; i++) best = fmaxf(best, v[i]);
    const float top = moe_wave_max(best);
    float all = 0.f;
    if (!a.renorm) {
#pragma unroll
        for (int i = 0; i < PER; i++) all += v[i] == kNegInf ? 0.f : v[i] == top ? 1.f : expf(v[i] - top);
        all = moe_wave_sum(all);
    }
    float mine = 0.f, sum = 0.f;
    int id = -1;
    for (int j = 0; j < a.top_k; j++) {
        const float m = moe_wave_max(best);
        if (m == kNegInf) break;
        const int src = __builtin_ctzll(__ballot(best == m));
        int at = 0;
        if (lane == src) {
            bool found = false;
#pragma unroll
            for (int i = 0; i < PER; i++)
                if (!found && v[i] == m) found = true, at = i, v[i] = kNegInf;
            best = v[0];
#pragma unroll
            for (int i = 1; i < PER; i++) best = fmaxf(best, v[i]);
        }
        at = __builtin_amdgcn_readlane(at, src) + src * PER;
        const float p = m == top ? 1.f : expf(m - top);
        sum += p;
        if (lane == j) mine = p, id = at;
    }
    if (a.renorm) all = sum;
    if (lane < a.top_k) {
        a.ids[(size_t)tok * a.top_k + lane] = id;
        a.weights[(size_t)tok * a.top_k + lane] = id < 0 ? 0.f : mine / all;
    }
}

hipError_t launch_moe_route(const RouteArgs& a, hipStream_t s) {
    const int grid = (a.n + 3) / 4;
    if (a.n_experts <= 64) k_moe_route<1><<<grid, 256, 0, s>>>(a);
    else if (a.n_experts <= 128) k_moe_route<2><<<grid, 256, 0, s>>>(a);
    else if (a.n_experts <= 256) k_moe_route<4><<<grid, 256, 0, s>>>(a);
    else if (a.n_experts <= 512) k_moe_route<8><<<grid, 256, 0, s>>>(a);
    else k_moe_route<16><<<grid, 256, 0, s>>>(a);
    return hipGetLastError();
}

// ---- the experts, pair by pair -------------------------------------------------------------------------------
// h[pair][f] = silu(W_gate x) (W_up x) of the pair's expert, then y[t] = sum over its pairs of weight W_down h:
// a wave a row of the weights, 16 columns a lane at a time (half a Q8 block: one scale), fp32 products.

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
        const float gs = moe_wave_sum(g[i]), us = moe_wave_sum(u[i]);
        if (lane == 0 && f0 + i < a.ffn) a.h[(size_t)pair * a.ffn + f0 + i] = gs * sigmoid(gs) * us;
    }
}

template <int DT>
__global__ __launch_bounds__(256) void k_moe_pair_down(MoeArgs a) {
    const int tok = blockIdx.x, lane = threadIdx.x & 63;
    const int r0 = (blockIdx.y * 4 + (threadIdx.x >> 6)) * kPairRows;
    float y[kPairRows] = {};
    for (int j = 0; j < a.top_k; j++) {
        const int pair = tok * a.top_k + j, e = a.ids[pair];
        if (e < 0 || e >= a.n_experts) continue;
        float acc[kPairRows] = {};
        for (int c = lane * 16; c < a.ffn; c += 1024) {
            float h[16];
            load_vec<0, 16>(a.h, (size_t)pair * a.ffn + c, h);
#pragma unroll
            for (int i = 0; i < kPairRows; i++) {
                if (r0 + i >= a.hidden) break;
                const size_t at = ((size_t)e * a.hidden + r0 + i) * a.ffn + c;
                acc[i] = fmaf(dot16(*reinterpret_cast<const u32x4*>(a.w_down + at), h), a.s_down[at >> 5], acc[i]);
            }
        }
        const float wt = a.weights[pair];
#pragma unroll
        for (int i = 0; i < kPairRows; i++) y[i] = fmaf(wt, acc[i], y[i]);
    }
#pragma unroll
    for (int i = 0; i < kPairRows; i++) {
        const float s = moe_wave_sum(y[i]);
        if (lane == 0 && r0 + i < a.hidden) {
            const size_t at = (size_t)tok * a.y_stride + r0 + i;
            if constexpr (DT == 0) static_cast<float*>(a.y)[at] = s;
            else static_cast<__bf16*>(a.y)[at] = (__bf16)s;
        }
    }
}

// ---- the experts, grouped: pairs sorted by expert, tiled products on the matrix cores ------------------------
// k_moe_group sorts the pairs by expert and lists tiles of BM rows of one expert; k_moe_rows writes activations as fp16
// operands; k_moe_gemm multiplies a tile's rows with 64 gate and the same 64 up rows of its expert's weights (or 128 down
// rows); k_moe_combine sums a token's pairs in their order.
//
// Operands: an int8 weight is exact in fp16. A row of activations is scaled by the power of two that puts its largest
// magnitude into [2^14, 2^15) and becomes the sum of two fp16 (within 2^-22, small values within 2^-39 of the row's
// largest; one is enough for a bf16 x). The block scales multiply each 32-column product in fp32.
// (an expert's rows in whatever order the sort's counters gave them: a row's result does not depend on the rows beside it)

struct MoeTile {
    int expert, row, rows;
};
struct MoeWs {
    int* n_tiles;
    MoeTile* tiles;
    int *row_pair, *pair_row;  // sorted row -> pair, pair -> sorted row (-1: no expert)
    int *x_shift, *h_shift;    // powers of two of the operand rows
    f16 *x16, *h16;            // operands [part][row][columns up to a multiple of 64]
    size_t x_part, h_part;     // elements of a part
    float* h;                  // [row][ffn]
    float* y;                  // [row][hidden]
};

// One workgroup.
__global__ __launch_bounds__(1024) void k_moe_group(MoeArgs a, MoeWs ws, int bm) {
    __shared__ int count[1024], part[2][16];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, pairs = a.n * a.top_k;
    count[tid] = 0;
    __syncthreads();
    for (int i = tid; i < pairs; i += 1024) {
        const int e = a.ids[i];
        if (e >= 0 && e < a.n_experts) atomicAdd(&count[e], 1);
    }
    __syncthreads();
    const int mine = count[tid], tiles = (mine + bm - 1) / bm;
    int rows = mine, tile = tiles;  // running sums over the experts
#pragma unroll
    for (int s = 1; s < 64; s *= 2) {
        const int r = __shfl_up(rows, s), q = __shfl_up(tile, s);
        if (lane >= s) rows += r, tile += q;
    }
    if (lane == 63) part[0][wave] = rows, part[1][wave] = tile;
    __syncthreads();
    for (int w = 0; w < wave; w++) rows += part[0][w], tile += part[1][w];
    rows -= mine, tile -= tiles;
    for (int i = 0; i < tiles; i++) ws.tiles[tile + i] = MoeTile{tid, rows + i * bm, min(bm, mine - i * bm)};
    if (tid == 1023) *ws.n_tiles = tile + tiles;
    count[tid] = rows;
    __syncthreads();
    for (int i = tid; i < pairs; i += 1024) {
        const int e = a.ids[i];
        int r = -1;
        if (e >= 0 && e < a.n_experts) {
            r = atomicAdd(&count[e], 1);
            ws.row_pair[r] = i;
        }
        ws.pair_row[i] = r;
    }
}

// A row of activations as fp16 operands: out[part][row][padded], zeros from `cols` on, and its power of two. A workgroup
// a row.
template <int DT, int P>
__global__ __launch_bounds__(256) void k_moe_rows(const void* x, size_t stride, int cols, int padded, f16* out, size_t part, int* shift) {
    __shared__ float most[4];
    const int tid = threadIdx.x;
    const size_t row = blockIdx.x;
    float v[8], m = 0.f;
    for (int c = tid * 8; c < cols; c += 2048) {
        load_vec<DT, 8>(x, row * stride + c, v);
#pragma unroll
        for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(v[i]));
    }
    m = moe_wave_max(m);
    if ((tid & 63) == 0) most[tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(most[0], most[1]), fmaxf(most[2], most[3]));
    // (a row with an infinity, or of zeros, is not scaled)
    const int up = m > 0.f && m < __builtin_inff() ? 15 - __builtin_amdgcn_frexp_expf(m) : 0;
    if (tid == 0) shift[row] = up;
    for (int c = tid * 8; c < padded; c += 2048) {
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

// P parts; WM x WN x WK waves (WK: the step's 32-column blocks shared out), MT x 2 tiles of 32 x 32 a wave; BKB blocks a step.
template <int P, int WM, int WN, int WK, int MT, int BKB>
struct MoeTileShape {
    static constexpr int kThreads = 64 * WM * WN * WK, BM = WM * MT * 32, BN = WN * 64, RB = BKB * 64;  // RB: bytes of an LDS row
    static constexpr int kA = P * BM * RB, kW = BN * RB, kS = BN * BKB * 4, kStage = kA + kW + kS;
    static constexpr int AL = P * BM * BKB * 4 / kThreads, WL = BN * BKB * 2 / kThreads;
    static constexpr int kLds = 2 * kStage + BM * 4;
    static_assert(AL * kThreads == P * BM * BKB * 4 && WL * kThreads == BN * BKB * 2 && BN * BKB <= kThreads && BKB % WK == 0, "whole loads");
    static_assert(WK == 1 || 2 * kStage >= WM * WN * MT * 2 * 16 * 256, "the blocks' sums meet in the stages");
};

template <int P, int WM, int WN, int WK, int MT, int BKB, bool UP>
__global__ __launch_bounds__(64 * WM * WN * WK) void k_moe_gemm(MoeArgs a, MoeWs ws) {
    typedef MoeTileShape<P, WM, WN, WK, MT, BKB> T;
    constexpr int BM = T::BM, BN = T::BN, Q = BKB * 4;  // Q: 16-byte pieces of an LDS row
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    // an M tile's column tiles on one XCD, one after the other: its rows come from that XCD's L2
    const int outs = UP ? a.ffn : a.hidden, cols = UP ? a.hidden : a.ffn, per = UP ? BN / 2 : BN;
    const int nn = (outs + per - 1) / per, seq = blockIdx.x >> 3;
    const int tile = seq / nn * 8 + (blockIdx.x & 7), n0 = seq % nn * per;
    if (tile >= *ws.n_tiles) return;
    const MoeTile mt = ws.tiles[tile];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int c = lane & 31, h = lane >> 5;
    const int wk = wave % WK, wn = wave / WK % WN, wm = wave / WK / WN;
    const int padded = (cols + 63) & ~63, nkb = cols >> 5, steps = (nkb + BKB - 1) / BKB;
    int* sShift = reinterpret_cast<int*>(smem + 2 * T::kStage);
    for (int r = tid; r < BM; r += T::kThreads) {
        const int row = mt.row + min(r, mt.rows - 1);
        sShift[r] = -(UP ? ws.x_shift[ws.row_pair[row] / a.top_k] : ws.h_shift[row]);
    }

    // LDS rows of BKB * 64 bytes, 16-byte piece q of row r at q ^ (r >> SH) % Q: operand reads (16 rows' piece q) and writes
    // spread over the banks
    static_assert(BKB == 1 || BKB == 2, "");
    constexpr int SH = BKB == 2 ? 1 : 2;
    auto at = [](int r, int q) { return r * T::RB + ((q ^ ((r >> SH) & (Q - 1))) << 4); };
    const f16* ap[T::AL];
    int ald[T::AL];
#pragma unroll
    for (int i = 0; i < T::AL; i++) {
        const int idx = tid + i * T::kThreads, q = idx % Q, r = idx / Q % BM, part = idx / Q / BM;
        const int row = mt.row + min(r, mt.rows - 1);  // (rows past the tile's: the last one's, their results unused)
        ap[i] = (UP ? ws.x16 + (size_t)(ws.row_pair[row] / a.top_k) * padded + (part ? ws.x_part : 0)
                    : ws.h16 + (size_t)row * padded + (part ? ws.h_part : 0)) + q * 8;
        ald[i] = part * BM * T::RB + at(r, q);
    }
    // weight row r of the tile: UP: of each 64, 32 gate rows and the same 32 up rows
    auto weight_row = [&](int r) {
        const int o = UP ? n0 + (r >> 6) * 32 + (r & 31) : n0 + r;
        return (size_t)mt.expert * outs + min(o, outs - 1);
    };
    const int8_t* wp[T::WL];
    int wld[T::WL];
    const int wq = tid % (BKB * 2);  // (the same for every i: the thread count is a multiple)
#pragma unroll
    for (int i = 0; i < T::WL; i++) {
        const int r = (tid + i * T::kThreads) / (BKB * 2);
        wp[i] = (UP ? (r & 32 ? a.w_up : a.w_gate) : a.w_down) + weight_row(r) * cols;
        wld[i] = r;
    }
    const int sr = tid / BKB % BN, sb = tid % BKB;
    const float* sp = (UP ? (sr & 32 ? a.s_up : a.s_gate) : a.s_down) + weight_row(sr) * nkb;

    u32x4 av[T::AL], wv[T::WL];
    float sv;
    auto load = [&](int k) {
        const int blk = k * BKB;
#pragma unroll
        for (int i = 0; i < T::AL; i++) av[i] = *reinterpret_cast<const u32x4*>(ap[i] + blk * 32);
        // a block past the row: weights of its first one with a scale of zero, on the operands' zeros
        const int wc = blk * 32 + 16 * wq, wcol = wc < cols ? wc : 0;
#pragma unroll
        for (int i = 0; i < T::WL; i++) wv[i] = *reinterpret_cast<const u32x4*>(wp[i] + wcol);
        sv = sp[min(blk + sb, nkb - 1)];
        if (blk + sb >= nkb) sv = 0.f;
    };
    auto store = [&](uint8_t* S) {
#pragma unroll
        for (int i = 0; i < T::AL; i++) *reinterpret_cast<u32x4*>(S + ald[i]) = av[i];
#pragma unroll
        for (int i = 0; i < T::WL; i++)
#pragma unroll
            for (int p = 0; p < 2; p++) {
                f16x2 v[4];
                weights_f16(wv[i][2 * p], v[0], v[1]), weights_f16(wv[i][2 * p + 1], v[2], v[3]);
                f16x8 o;
#pragma unroll
                for (int e = 0; e < 4; e++) o[2 * e] = v[e][0], o[2 * e + 1] = v[e][1];
                *reinterpret_cast<f16x8*>(S + T::kA + at(wld[i], 2 * wq + p)) = o;
            }
        if (tid < BN * BKB) reinterpret_cast<float*>(S + T::kA + T::kW)[sb * BN + sr] = sv;
    };

    f32x16 acc[MT][2];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int n = 0; n < 2; n++)
#pragma unroll
            for (int e = 0; e < 16; e++) acc[m][n][e] = 0.f;
    load(0);
    store(smem);
    load(min(1, steps - 1));
    __syncthreads();
#pragma unroll 1
    for (int k = 0; k < steps; k++) {
        const uint8_t* S = smem + (k & 1) * T::kStage;
        if (k + 1 < steps) store(smem + ((k + 1) & 1) * T::kStage);
        load(min(k + 2, steps - 1));
#pragma unroll
        for (int jj = 0; jj < BKB / WK; jj++) {
            const int j = jj * WK + wk;
            f16x8 w[2][2], x[MT][P][2];
            float sc[2];
#pragma unroll
            for (int n = 0; n < 2; n++) {
                const int r = wn * 64 + 32 * n + c;
#pragma unroll
                for (int q = 0; q < 2; q++) w[n][q] = *reinterpret_cast<const f16x8*>(S + T::kA + at(r, 4 * j + 2 * q + h));
                sc[n] = reinterpret_cast<const float*>(S + T::kA + T::kW)[j * BN + r];
            }
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int p = 0; p < P; p++)
#pragma unroll
                    for (int q = 0; q < 2; q++)
                        x[m][p][q] = *reinterpret_cast<const f16x8*>(S + p * BM * T::RB + at((wm * MT + m) * 32 + c, 4 * j + 2 * q + h));
#pragma unroll
            for (int m = 0; m < MT; m++)
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    f32x16 d = {};
#pragma unroll
                    for (int p = P - 1; p >= 0; p--)
#pragma unroll
                        for (int q = 0; q < 2; q++) d = mfma32h(x[m][p][q], w[n][q], d);
#pragma unroll
                    for (int e = 0; e < 16; e++) acc[m][n][e] = fmaf(sc[n], d[e], acc[m][n][e]);
                }
        }
        __syncthreads();
    }
    if constexpr (WK == 2) {
        float* meet = reinterpret_cast<float*>(smem) + (wm * WN + wn) * (MT * 2 * 16 * 64) + lane;
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int e = 0; e < 16; e++)
                    if (wk) meet[((m * 2 + n) * 16 + e) * 64] = acc[m][n][e];
        __syncthreads();
        if (wk) return;
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int e = 0; e < 16; e++) acc[m][n][e] += meet[((m * 2 + n) * 16 + e) * 64];
    }
    // lane (c, h): weight row c of a tile, activation rows 8 (e / 4) + 4 h + e % 4
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
        for (int e = 0; e < 16; e++) {
            const int r = (wm * MT + m) * 32 + 8 * (e >> 2) + 4 * h + (e & 3);
            if (r >= mt.rows) continue;
            const int s = sShift[r];
            const size_t row = mt.row + r;
            if constexpr (UP) {
                const int f = n0 + wn * 32 + c;
                const float g = ldexpf(acc[m][0][e], s), u = ldexpf(acc[m][1][e], s);
                if (f < outs) ws.h[row * outs + f] = g * sigmoid(g) * u;
            } else {
                const float wt = a.weights[ws.row_pair[row]];
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    const int o = n0 + wn * 64 + 32 * n + c;
                    if (o < outs) ws.y[row * outs + o] = wt * ldexpf(acc[m][n][e], s);
                }
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
        *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.y) + tok * a.y_stride + o) = u32x2{pk_bf16(s[0], s[1]), pk_bf16(s[2], s[3])};
    }
}

// ---- which form -----------------------------------------------------------------------------------------------
// Pair by pair while the experts' rows are few (each pair streams its expert's weights, repeated ones from the cache).
static bool by_pairs(const MoeArgs& a) { return (long long)a.n * a.top_k <= std::max(16, a.n_experts); }

constexpr int kMoeSegment = 1 << 16;  // pairs worked off at a time: bounds the workspace
static int segment_tokens(const MoeArgs& a) { return std::max(1, std::min(a.n, kMoeSegment / a.top_k)); }

static size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }
// Bytes of the grouped form's workspace; the pointers into it with `base`.
static size_t lay_out(const MoeArgs& a, int parts, uint8_t* base, MoeWs& w) {
    const size_t n = segment_tokens(a), pairs = n * a.top_k, hp = (a.hidden + 63) & ~63, fp = (a.ffn + 63) & ~63;
    size_t at = 0;
    auto take = [&](auto*& p, size_t bytes) {
        p = reinterpret_cast<std::remove_reference_t<decltype(p)>>(reinterpret_cast<uintptr_t>(base) + at);
        at += up256(bytes);
    };
    take(w.n_tiles, 4), take(w.tiles, (pairs / 32 + a.n_experts + 1) * sizeof(MoeTile));
    take(w.row_pair, pairs * 4), take(w.pair_row, pairs * 4), take(w.x_shift, n * 4), take(w.h_shift, pairs * 4);
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

template <int P, int WM, int WN, int WK, int MT, int BKB, bool UP>
static hipError_t moe_gemm(const MoeArgs& a, const MoeWs& w, hipStream_t s) {
    typedef MoeTileShape<P, WM, WN, WK, MT, BKB> T;
    static std::atomic<uint64_t> raised{0};
    const auto k = &k_moe_gemm<P, WM, WN, WK, MT, BKB, UP>;
    if (const hipError_t e = raise_lds(reinterpret_cast<const void*>(k), T::kLds, raised)) return e;
    // the most tiles that the pairs can make (workgroups past the real number end at once)
    const int pairs = a.n * a.top_k, tiles = std::min(pairs, pairs / T::BM + std::min(a.n_experts, pairs));
    const int outs = UP ? a.ffn : a.hidden, per = UP ? T::BN / 2 : T::BN;
    k<<<(tiles + 7) / 8 * 8 * ((outs + per - 1) / per), T::kThreads, T::kLds, s>>>(a, w);
    return hipGetLastError();
}

template <int WM, int WN, int WK, int MT, int DT>
static hipError_t moe_tiles(const MoeArgs& a, const MoeWs& w, hipStream_t s) {
    constexpr int P = DT ? 1 : 2, BKB = WK == 2 || P == 1 ? 2 : 1, BKB2 = WK == 2 ? 2 : 1;  // (two parts of 64 columns: half the workgroups a CU)
    k_moe_group<<<1, 1024, 0, s>>>(a, w, WM * MT * 32);
    k_moe_rows<DT, P><<<a.n, 256, 0, s>>>(a.x, a.x_stride, a.hidden, (a.hidden + 63) & ~63, w.x16, w.x_part, w.x_shift);
    if (const hipError_t e = moe_gemm<P, WM, WN, WK, MT, BKB, true>(a, w, s)) return e;
    k_moe_rows<0, 2><<<a.n * a.top_k, 256, 0, s>>>(w.h, a.ffn, a.ffn, (a.ffn + 63) & ~63, w.h16, w.h_part, w.h_shift);
    if (const hipError_t e = moe_gemm<2, WM, WN, WK, MT, BKB2, false>(a, w, s)) return e;
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
        if (rows >= 96) e = moe_tiles<2, 2, 1, 2, DT>(b, w, s);
        else if (rows >= 24) e = moe_tiles<2, 2, 1, 1, DT>(b, w, s);
        else e = moe_tiles<1, 2, 2, 1, DT>(b, w, s);
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

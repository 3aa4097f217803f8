// The router and the SwiGLU experts of a mixture-of-experts layer (qwattn_moe_route, qwattn_moe; the reference's
// shaders/moe_route.comp, moe_group.comp, moe_combine.comp and the expert variants of its matmul shaders).
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

size_t moe_workspace(const MoeArgs& a, bool) { return (size_t)a.n * a.top_k * a.ffn * 4; }

template <int DT>
static hipError_t moe_pairs(const MoeArgs& a, hipStream_t s) {
    const int per = 4 * kPairRows;
    k_moe_pair_up<DT><<<dim3(a.n * a.top_k, (a.ffn + per - 1) / per), 256, 0, s>>>(a);
    k_moe_pair_down<DT><<<dim3(a.n, (a.hidden + per - 1) / per), 256, 0, s>>>(a);
    return hipGetLastError();
}

hipError_t launch_moe(MoeArgs a, bool bf16, void* workspace, hipStream_t s) {
    a.h = static_cast<float*>(workspace);
    return bf16 ? moe_pairs<1>(a, s) : moe_pairs<0>(a, s);
}

}  // namespace qw

// Short causal depthwise convolution with SiLU and a carried state (qwattn_conv_silu; the reference's
// shaders/conv1d.comp): y[t][c] = silu(bias[c] + sum_{j < K} w[c][j] x[t - K + 1 + j][c]).
//
// A thread owns eight channels (one or two 16-byte loads a row) and walks a tile of consecutive tokens with the
// last K - 1 rows in registers, so every row is read once plus K - 1 rows a tile. Bound by HBM.
// Rows before the first token come from the state, which only tile 0 reads: its threads also write the new
// one (channel by channel after their own reads), so no other workgroup can see half of it.
#include "common.hpp"
#include "kernels.hpp"

namespace qw {

constexpr int kConvThreads = 128;

template <int DT>
__device__ __forceinline__ void store8(void* p, size_t i, const float (&v)[8]) {
    if constexpr (DT == 0) {
        float* f = static_cast<float*>(p) + i;
        *reinterpret_cast<f32x4*>(f) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>(f + 4) = f32x4{v[4], v[5], v[6], v[7]};
    } else {
        bf16x8 o;
#pragma unroll
        for (int k = 0; k < 8; k++) o[k] = (__bf16)v[k];
        *reinterpret_cast<bf16x8*>(static_cast<uint16_t*>(p) + i) = o;
    }
}

template <int DT, int K>
__global__ __launch_bounds__(kConvThreads) void k_conv_silu(ConvArgs a) {
    const int c = (blockIdx.x * kConvThreads + threadIdx.x) * 8, b = blockIdx.z;
    const int len = a.lens ? min(max(a.lens[b], 0), a.n) : a.n;
    const int t0 = blockIdx.y * a.tile, t1 = min(t0 + a.tile, len);
    if (c >= a.channels || (t0 >= t1 && blockIdx.y)) return;
    const size_t row0 = (size_t)b * a.n;
    float* state = a.state + ((size_t)b * (K - 1)) * a.channels + c;

    float w[K * 8], win[K][8];  // win: the rows t - K + 1 .. t
#pragma unroll
    for (int i = 0; i < K * 8; i += 4) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(a.w + (size_t)c * K + i);
        w[i] = v[0], w[i + 1] = v[1], w[i + 2] = v[2], w[i + 3] = v[3];
    }
    float bias[8] = {};
    if (a.bias) load_vec<0, 8>(a.bias, c, bias);
    float old[K - 1][8];  // tile 0: the state before
    if (blockIdx.y == 0) {
#pragma unroll
        for (int j = 0; j < K - 1; j++) {
            load_vec<0, 8>(state, (size_t)j * a.channels, old[j]);
#pragma unroll
            for (int e = 0; e < 8; e++) win[j + 1][e] = old[j][e];
        }
    } else {
#pragma unroll
        for (int j = 0; j < K - 1; j++) load_vec<DT, 8>(a.x, (row0 + t0 - K + 1 + j) * a.x_stride + c, win[j + 1]);
    }
#pragma unroll 4
    for (int t = t0; t < t1; t++) {
#pragma unroll
        for (int j = 0; j < K - 1; j++)
#pragma unroll
            for (int e = 0; e < 8; e++) win[j][e] = win[j + 1][e];
        load_vec<DT, 8>(a.x, (row0 + t) * a.x_stride + c, win[K - 1]);
        float y[8];
#pragma unroll
        for (int e = 0; e < 8; e++) {
            float s = bias[e];
#pragma unroll
            for (int j = 0; j < K; j++) s = fmaf(w[e * K + j], win[j][e], s);
            y[e] = s * sigmoid(s);
        }
        store8<DT>(a.y, (row0 + t) * a.y_stride + c, y);
        if (a.snap)
#pragma unroll
            for (int j = 1; j < K; j++) store8<0>(a.snap, ((row0 + t) * (K - 1) + j - 1) * a.channels + c, win[j]);
    }
    if (blockIdx.y || len == 0) return;
#pragma unroll
    for (int j = 0; j < K - 1; j++) {  // row len - K + 1 + j of (state ++ x)
        const int t = len - K + 1 + j;
        float v[8];
        if (t >= 0) {
            load_vec<DT, 8>(a.x, (row0 + t) * a.x_stride + c, v);
        } else {
#pragma unroll
            for (int i = 0; i < K - 1; i++)
                if (i == t + K - 1)
#pragma unroll
                    for (int e = 0; e < 8; e++) v[e] = old[i][e];
        }
        store8<0>(state, (size_t)j * a.channels, v);
    }
}

template <int DT>
static hipError_t conv_taps(const ConvArgs& a, dim3 grid, hipStream_t s) {
    if (a.taps == 2) k_conv_silu<DT, 2><<<grid, kConvThreads, 0, s>>>(a);
    else if (a.taps == 3) k_conv_silu<DT, 3><<<grid, kConvThreads, 0, s>>>(a);
    else k_conv_silu<DT, 4><<<grid, kConvThreads, 0, s>>>(a);
    return hipGetLastError();
}

hipError_t launch_conv_silu(ConvArgs a, bool bf16, hipStream_t s) {
    // tiles of 16 tokens; longer ones where a grid's y dimension would not take their number
    a.tile = 16;
    while ((a.n + a.tile - 1) / a.tile > 65535) a.tile *= 2;
    const dim3 grid((a.channels / 8 + kConvThreads - 1) / kConvThreads, (a.n + a.tile - 1) / a.tile, a.n_seq);
    return bf16 ? conv_taps<1>(a, grid, s) : conv_taps<0>(a, grid, s);
}

}  // namespace qw

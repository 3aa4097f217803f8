// The gated delta rule (qwattn_delta_rule; the reference's shaders/deltanet.comp and shaders/gated_norm.comp).
// Per token and value head, with k and q the key head's rows over their 2-norms (q also over sqrt(DK)) and a state
// S [DK][DV] in fp32:
//   S <- e^g S;  u = beta (v - S^T k);  S <- S + k u^T;  o = S^T q;   z: o rsqrt(mean o^2 + eps) gamma silu(z)
#include "common.hpp"
#include "kernels.hpp"

namespace qw {

__device__ __forceinline__ float delta_wave_sum(float x) {
    x = sum32(x);
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
}

// Sum over the 16 lanes with this lane's l % 4 (row groups l / 4): within 16-lane rows by rotation, then across rows.
__device__ __forceinline__ float sum_groups(float x) {
    x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x124, 0xF, 0xF, false));
    x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x128, 0xF, 0xF, false));
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// log decay and beta of row r, value head h
__device__ __forceinline__ float delta_log_decay(const DeltaArgs& a, size_t r, int h) {
    const float g = a.a[r * a.v_heads + h];
    if (!a.a_coef) return g;
    const float x = g + a.dt_bias[h];
    return a.a_coef[h] * (fmaxf(x, 0.f) + log1pf(expf(-fabsf(x))));  // softplus
}
__device__ __forceinline__ float delta_beta(const DeltaArgs& a, size_t r, int h) {
    const float b = a.b[r * a.v_heads + h];
    return a.a_coef ? 1.f / (1.f + expf(-b)) : b;
}

__device__ __forceinline__ int key_head(const DeltaArgs& a, int h) {
    return a.tiled ? h % a.k_heads : h / (a.v_heads / a.k_heads);
}

template <int DT>
__device__ __forceinline__ void store_out(void* p, size_t i, float v) {
    if constexpr (DT == 0) static_cast<float*>(p)[i] = v;
    else static_cast<__bf16*>(p)[i] = (__bf16)v;
}

// ---- token by token ------------------------------------------------------------------------------------------
// A workgroup owns one (sequence, value head) and holds its state in registers: a wave 16 columns, a lane four of
// them (l % 4) in DK / 16 rows (l / 4). S^T k and S^T q of the state before the token are summed in one go, in the
// wave: u = beta (v - e^g S^T k), o = e^g S^T q + (k . q) u. q, k, v and the gates of 16 tokens are staged (and
// normalized) in the LDS at a time, while the state is on its way, so a token needs no barrier.
constexpr int kStepTokens = 16;

template <int DT, int DK, int DV>
__global__ __launch_bounds__(DV * 4) void k_delta_step(DeltaArgs a) {
    constexpr int NW = DV / 16, RPT = DK / 16;
    __shared__ __attribute__((aligned(16))) float sq[kStepTokens][DK], sk[kStepTokens][DK], sv[kStepTokens][DV],
        so[kStepTokens][DV];
    __shared__ float gates[kStepTokens][3];  // decay, beta, k . q
    const int h = blockIdx.x, b = blockIdx.y, kh = key_head(a, h);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int len = a.lens ? min(max(a.lens[b], 0), a.n) : a.n;
    if (len == 0) return;
    const int col = 16 * wave + 4 * (lane & 3), r0 = (lane >> 2) * RPT;
    const size_t row0 = (size_t)b * a.n;
    float* state = a.state + ((size_t)b * a.v_heads + h) * (DK * DV) + r0 * DV + col;
    f32x4 S[RPT];
#pragma unroll
    for (int i = 0; i < RPT; i++) S[i] = *reinterpret_cast<const f32x4*>(state + i * DV);

    for (int t0 = 0; t0 < len; t0 += kStepTokens) {
        const int nb = min(kStepTokens, len - t0);
        for (int t = wave; t < nb; t += NW) {
            const size_t r = row0 + t0 + t;
            float q[DK / 64], k[DK / 64], qq = 0.f, kk = 0.f, kq = 0.f;
#pragma unroll
            for (int i = 0; i < DK / 64; i++) {
                q[i] = load_in<DT>(a.q, r * a.q_stride + kh * DK + 64 * i + lane);
                k[i] = load_in<DT>(a.k, r * a.k_stride + kh * DK + 64 * i + lane);
                qq = fmaf(q[i], q[i], qq), kk = fmaf(k[i], k[i], kk);
            }
#pragma unroll
            for (int i = 0; i < DV / 64; i++)
                sv[t][64 * i + lane] = load_in<DT>(a.v, r * a.v_stride + h * DV + 64 * i + lane);
            const float qr = rsqrtf(delta_wave_sum(qq) + a.eps) * (DK == 128 ? 0.08838834764831845f : 0.125f);
            const float kr = rsqrtf(delta_wave_sum(kk) + a.eps);
#pragma unroll
            for (int i = 0; i < DK / 64; i++) {
                q[i] *= qr, k[i] *= kr;
                sq[t][64 * i + lane] = q[i], sk[t][64 * i + lane] = k[i];
                kq = fmaf(q[i], k[i], kq);
            }
            kq = delta_wave_sum(kq);
            if (lane == 0) gates[t][0] = expf(delta_log_decay(a, r, h)), gates[t][1] = delta_beta(a, r, h), gates[t][2] = kq;
        }
        __syncthreads();
        for (int t = 0; t < nb; t++) {
            float kv[RPT], qv[RPT];
#pragma unroll
            for (int i = 0; i < RPT; i += 4) {
                const f32x4 k4 = *reinterpret_cast<const f32x4*>(&sk[t][r0 + i]);
                const f32x4 q4 = *reinterpret_cast<const f32x4*>(&sq[t][r0 + i]);
#pragma unroll
                for (int e = 0; e < 4; e++) kv[i + e] = k4[e], qv[i + e] = q4[e];
            }
            const float decay = gates[t][0], beta = gates[t][1], kq = gates[t][2];
            const f32x4 v4 = *reinterpret_cast<const f32x4*>(&sv[t][col]);
            f32x4 o4, u4;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                float ks = 0.f, qs = 0.f;
#pragma unroll
                for (int i = 0; i < RPT; i++) ks = fmaf(kv[i], S[i][e], ks), qs = fmaf(qv[i], S[i][e], qs);
                ks = sum_groups(ks), qs = sum_groups(qs);
                u4[e] = beta * (v4[e] - decay * ks);
                o4[e] = fmaf(kq, u4[e], decay * qs);
            }
#pragma unroll
            for (int i = 0; i < RPT; i++)
#pragma unroll
                for (int e = 0; e < 4; e++) S[i][e] = fmaf(kv[i], u4[e], decay * S[i][e]);
            if (lane < 4) *reinterpret_cast<f32x4*>(&so[t][col]) = o4;
            if (a.snap) {
                float* p = a.snap + ((row0 + t0 + t) * a.v_heads + h) * (DK * DV) + r0 * DV + col;
#pragma unroll
                for (int i = 0; i < RPT; i++) *reinterpret_cast<f32x4*>(p + i * DV) = S[i];
            }
        }
        __syncthreads();
        for (int t = wave; t < nb; t += NW) {
            const size_t r = row0 + t0 + t;
            float o[DV / 64], ss = 0.f;
#pragma unroll
            for (int i = 0; i < DV / 64; i++) o[i] = so[t][64 * i + lane], ss = fmaf(o[i], o[i], ss);
            if (a.z) {
                const float rms = rsqrtf(delta_wave_sum(ss) * (1.f / DV) + a.eps);
#pragma unroll
                for (int i = 0; i < DV / 64; i++) {
                    const float z = load_in<DT>(a.z, r * a.z_stride + h * DV + 64 * i + lane);
                    o[i] *= rms * a.gamma[64 * i + lane] * (z * sigmoid(z));
                }
            }
#pragma unroll
            for (int i = 0; i < DV / 64; i++) store_out<DT>(a.out, r * a.out_stride + h * DV + 64 * i + lane, o[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < RPT; i++) *reinterpret_cast<f32x4*>(state + i * DV) = S[i];
}

template <int DT, int DK>
static hipError_t delta_step(const DeltaArgs& a, hipStream_t s) {
    const dim3 grid(a.v_heads, a.n_seq);
    if (a.val_dim == 64) k_delta_step<DT, DK, 64><<<grid, 256, 0, s>>>(a);
    else k_delta_step<DT, DK, 128><<<grid, 512, 0, s>>>(a);
    return hipGetLastError();
}

size_t delta_workspace(const DeltaArgs&, bool) { return 0; }

hipError_t launch_delta(const DeltaArgs& a, bool bf16, hipStream_t s) {
    if (bf16) return a.key_dim == 64 ? delta_step<1, 64>(a, s) : delta_step<1, 128>(a, s);
    return a.key_dim == 64 ? delta_step<0, 64>(a, s) : delta_step<0, 128>(a, s);
}

}  // namespace qw

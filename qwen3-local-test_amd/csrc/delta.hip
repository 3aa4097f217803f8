// The gated delta rule (qwattn_delta_rule; the reference's shaders/deltanet.comp and shaders/gated_norm.comp).
// Per token and value head, with k and q the key head's rows over their 2-norms (q also over sqrt(DK)) and a state
// S [DK][DV] in fp32:
//   S <- e^g S;  u = beta (v - S^T k);  S <- S + k u^T;  o = S^T q;   z: o rsqrt(mean o^2 + eps) gamma silu(z)
#include <algorithm>
#include <atomic>

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

// ---- chunks of 64 tokens -----------------------------------------------------------------------------------
// With G the running sum of g in a chunk, K and Q its normalized rows, D_ij = e^(G_i - G_j) (i >= j),
//   A = strict lower triangle of beta_i D_ij (K K^T)_ij,  T = (I + A)^-1,  P = lower triangle of D (Q K^T):
//   X = beta (V - e^G K S),  U = T X,  O = e^G Q S + P U,  S' = e^(G_end) S + (e^(G_end - G) K)^T U.
// k_delta_prep computes T and P of every chunk (all chunks at once); k_delta_chunks carries S through them, a
// workgroup a value head's 16 columns (the columns of S are systems of their own).
//
// fp32 accuracy on the bf16 matrix cores: an fp32 value is three bf16 parts (24 bits), a product of two such values the
// six part products down to 2^-24; bf16 q and k are one exact part, their norms and decays scale the results. Parts
// keep fp32's range, so nothing is scaled beforehand.
//
// Every operand that k_delta_chunks reads lies in the workspace as matrix-core fragments, a contiguous kilobyte each:
//   per (sequence, chunk, key head):   K, Q  [part][16-token tile][32-dim step]   rows tokens, k dims
//                                      K^T   [part][32-dim step][tile 0, 1][32-token step]; row r of tile j is the dim
//                                            8 (r / 4) + 4 j + r % 4 of its step: accumulator registers of the two
//                                            tiles of S are then the next product's operand fragment as they stand
//   per (sequence, chunk, value head): T, P  [part][6: the 32-token steps of each 16-token row tile that it reaches]
//                                      five vectors: beta, and the row scales of K S, Q S and K^T U; e^(G_end)
constexpr int kChunk = 64, kTriFrags = 6, kVec = 320;

struct DeltaWs {
    uint8_t* kq;   // K, Q, K^T units
    uint8_t* tp;   // T, P units
    float* vec;    // vectors
    float* o;      // fp32 outputs before the gated norm, [row][v_heads * val_dim]
};

template <int DK, int NP>
struct KqUnit {
    static constexpr int kSteps = DK / 32, kOne = NP * 4 * kSteps * 1024, kBytes = 3 * kOne;
};
constexpr int kTpOne = 3 * kTriFrags * 1024, kTpBytes = 2 * kTpOne;

// The six (or, with one part on the left, three) part products, smallest first.
template <int NP>
__device__ __forceinline__ f32x4 mfma_parts(const bf16x8 (&a)[NP], const bf16x8 (&b)[3], f32x4 c) {
    if constexpr (NP == 3) {
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[2], b[0], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[1], b[1], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0], b[2], c, 0, 0, 0);
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[1], b[0], c, 0, 0, 0);
    } else {
        c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0], b[2], c, 0, 0, 0);
    }
    c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0], b[1], c, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0], b[0], c, 0, 0, 0);
}

// Three bf16 parts of a pair of values, a word each.
__device__ __forceinline__ void split3(float v0, float v1, uint32_t (&w)[3]) {
    w[0] = pk_bf16(v0, v1);
    v0 = rest_bf16<0>(w[0], v0), v1 = rest_bf16<1>(w[0], v1);
    w[1] = pk_bf16(v0, v1);
    w[2] = pk_bf16(rest_bf16<0>(w[1], v0), rest_bf16<1>(w[1], v1));
}
__device__ __forceinline__ void split3(const float (&v)[8], u32x4 (&w)[3]) {
#pragma unroll
    for (int e = 0; e < 4; e++) {
        uint32_t p[3];
        split3(v[2 * e], v[2 * e + 1], p);
        w[0][e] = p[0], w[1][e] = p[1], w[2][e] = p[2];
    }
}

// A barrier for LDS traffic alone: loads on their way to registers stay on it.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int DT, int DK>
__global__ __launch_bounds__(256) void k_delta_prep(DeltaArgs a, DeltaWs ws, int c0, int ncs) {
    constexpr int NP = DT ? 1 : 3, KS = DK / 32, DPT = DK / 4, LD = 68;  // LD: row length of the 64 x 64 matrices
    typedef KqUnit<DK, NP> Unit;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    uint8_t* fk = smem;                                        // K and Q fragments
    uint8_t* fq = fk + Unit::kOne;
    float* sA = reinterpret_cast<float*>(fq + Unit::kOne);     // A
    float* sM = sA + 64 * LD;                                  // P, then T
    float* sD = sM + 64 * LD;                                  // the inverses of A's diagonal blocks, rows of 20
    double* sG = reinterpret_cast<double*>(sD + 4 * 16 * 20);  // G
    float* sBeta = reinterpret_cast<float*>(sG + 64);
    float* sRk = sBeta + 64;
    float* sRq = sRk + 64;

    const int cl = blockIdx.x, kh = blockIdx.y, b = blockIdx.z;
    const int len = a.lens ? min(max(a.lens[b], 0), a.n) : a.n;
    const int t0 = (c0 + cl) * kChunk, nt = min(kChunk, len - t0);
    if (nt <= 0) return;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int c = lane & 15, g = lane >> 4;
    uint8_t* kq = ws.kq + ((size_t)(b * ncs + cl) * a.k_heads + kh) * Unit::kBytes;

    {  // four lanes a row: norms, parts, fragments (zeros past the last token)
        const int row = tid >> 2, dim0 = (tid & 3) * DPT;
        const size_t r = (size_t)b * a.n + t0 + row;
        float k2 = 0.f, q2 = 0.f;
#pragma unroll
        for (int p = 0; p < DPT / 8; p++) {
            const int d = dim0 + 8 * p;
            float k[8] = {}, q[8] = {};
            if (row < nt) {
                load_vec<DT, 8>(a.k, r * a.k_stride + kh * DK + d, k);
                load_vec<DT, 8>(a.q, r * a.q_stride + kh * DK + d, q);
            }
#pragma unroll
            for (int e = 0; e < 8; e++) k2 = fmaf(k[e], k[e], k2), q2 = fmaf(q[e], q[e], q2);
            u32x4 kp[3], qp[3];
            split3(k, kp), split3(q, qp);
#pragma unroll
            for (int i = 0; i < NP; i++) {
                const int at = ((i * 4 + (row >> 4)) * KS + (d >> 5)) * 1024 + ((row & 15) + 16 * ((d >> 3) & 3)) * 16;
                *reinterpret_cast<u32x4*>(fk + at) = kp[i];
                *reinterpret_cast<u32x4*>(fq + at) = qp[i];
                *reinterpret_cast<u32x4*>(kq + at) = kp[i];
                *reinterpret_cast<u32x4*>(kq + Unit::kOne + at) = qp[i];
            }
        }
        k2 += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(k2), 0xB1, 0xF, 0xF, false));
        k2 += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(k2), 0x4E, 0xF, 0xF, false));
        q2 += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(q2), 0xB1, 0xF, 0xF, false));
        q2 += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(q2), 0x4E, 0xF, 0xF, false));
        if ((tid & 3) == 0) {
            sRk[row] = row < nt ? rsqrtf(k2 + a.eps) : 0.f;
            sRq[row] = (row < nt ? rsqrtf(q2 + a.eps) : 0.f) * (DK == 128 ? 0.08838834764831845f : 0.125f);
        }
    }
    __syncthreads();
    // K^T: eight tokens of one dim a piece
    for (int i = tid; i < NP * 8 * DK; i += 256) {
        const int l = i & 63, f = i >> 6;  // f: [part][step][tile][token step]
        const int u = f & 1, j = (f >> 1) & 1, s = (f >> 2) % KS, part = (f >> 2) / KS;
        const int d = 8 * ((l & 15) >> 2) + 4 * j + (l & 3), t = 32 * u + 8 * (l >> 4);
        const uint8_t* from = fk + ((part * 4 + (t >> 4)) * KS + s) * 1024 + ((t & 15) + 16 * (d >> 3)) * 16 + (d & 7) * 2;
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; e++)
            w[e] = *reinterpret_cast<const uint16_t*>(from + 32 * e) |
                   (uint32_t)*reinterpret_cast<const uint16_t*>(from + 32 * e + 16) << 16;
        *reinterpret_cast<u32x4*>(kq + 2 * Unit::kOne + f * 1024 + l * 16) = w;
    }
    // K K^T and Q K^T, wave w the row tile w
    f32x4 kk[4], qk[4];
    static_for<0, 4>([&](auto j_) {
        constexpr int j = j_;
        if (j <= wave) {
            kk[j] = qk[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = 0; s < KS; s++) {
                bf16x8 ak[NP], aq[NP], bk[3];
#pragma unroll
                for (int p = 0; p < NP; p++) {
                    ak[p] = *reinterpret_cast<const bf16x8*>(fk + ((p * 4 + wave) * KS + s) * 1024 + lane * 16);
                    aq[p] = *reinterpret_cast<const bf16x8*>(fq + ((p * 4 + wave) * KS + s) * 1024 + lane * 16);
                    bk[p] = *reinterpret_cast<const bf16x8*>(fk + ((p * 4 + j) * KS + s) * 1024 + lane * 16);
                }
                if constexpr (NP == 3) {
                    kk[j] = mfma_parts<3>(ak, bk, kk[j]);
                    qk[j] = mfma_parts<3>(aq, bk, qk[j]);
                } else {
                    kk[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ak[0], bk[0], kk[j], 0, 0, 0);
                    qk[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(aq[0], bk[0], qk[j], 0, 0, 0);
                }
            }
        }
    });

    const int R = a.v_heads / a.k_heads;
#pragma unroll 1
    for (int hi = 0; hi < R; hi++) {
        const int h = a.tiled ? kh + hi * a.k_heads : kh * R + hi;
        const size_t unit = (size_t)(b * ncs + cl) * a.v_heads + h;
        if (wave == 0) {  // lane: token. G in 64 bits (its differences are what counts), each g at least -2000 (e^g is 0
                          // from -104 on; a sum of -inf would have no differences)
            const size_t r = (size_t)b * a.n + t0 + lane;
            const bool in = lane < nt;
            double G = in ? (double)fmaxf(delta_log_decay(a, r, h), -2000.f) : 0.0;
            const float beta = in ? delta_beta(a, r, h) : 0.f;
#pragma unroll
            for (int s = 1; s < 64; s *= 2) {
                const double up = __shfl_up(G, s);
                if (lane >= s) G += up;
            }
            const double end = __shfl(G, 63);
            const float since = expf((float)G), rk = sRk[lane];
            sG[lane] = G, sBeta[lane] = beta;
            float* v = ws.vec + unit * kVec + lane;
            v[0] = beta;
            v[64] = beta * since * rk;
            v[128] = sRq[lane] * since;
            v[192] = rk * expf((float)(end - G));
            if (lane == 0) v[256] = expf((float)end);
        }
        __syncthreads();
        static_for<0, 4>([&](auto j_) {
            constexpr int j = j_;
            const int col = 16 * j + c;
            if (j <= wave) {
                const double Gj = sG[col];
                const float rkj = sRk[col];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int row = 16 * wave + 4 * g + i;
                    const float d = row >= col ? expf((float)(sG[row] - Gj)) * rkj : 0.f;
                    sA[row * LD + col] = row > col ? sBeta[row] * sRk[row] * d * kk[j][i] : 0.f;
                    sM[row * LD + col] = sRq[row] * d * qk[j][i];
                }
            } else if (j == wave + 1 && (wave & 1) == 0) {  // read as zeros by the row tile's 32-token step
#pragma unroll
                for (int i = 0; i < 4; i++) sM[(16 * wave + 4 * g + i) * LD + col] = 0.f;
            }
        });
        __syncthreads();
        uint8_t* tp = ws.tp + unit * kTpBytes;
        auto write_frags = [&](uint8_t* to) {
            for (int i = tid; i < kTriFrags * 64; i += 256) {
                const int f = i >> 6, l = i & 63;
                const int tile = f < 2 ? f : 1 + (f >> 1), step = f < 2 ? 0 : f & 1;
                const float* from = sM + (16 * tile + (l & 15)) * LD + 32 * step + 8 * (l >> 4);
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = from[e];
                u32x4 w[3];
                split3(v, w);
#pragma unroll
                for (int p = 0; p < 3; p++) *reinterpret_cast<u32x4*>(to + (p * kTriFrags + f) * 1024 + l * 16) = w[p];
            }
        };
        write_frags(tp + kTpOne);  // P
        {  // the inverse of A's diagonal block `wave` (unit lower triangular): lane c its column c, row after row
            const float* blk = sA + (16 * wave) * LD + 16 * wave;
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; i++) {
                float s = c == i ? 1.f : 0.f;
#pragma unroll
                for (int m = 0; m < i; m++) s = fmaf(-blk[i * LD + m], x[m], s);
                x[i] = s;
            }
            if (g == 0)
#pragma unroll
                for (int i = 0; i < 16; i++) sD[(16 * wave + i) * 20 + c] = x[i];
        }
        __syncthreads();
        // T's block column `wave` from the diagonal down: T_ij = -T_ii sum_m A_im T_mj on fp32 matrix cores. Step s of a
        // product takes the rows 4 g + s of its right operand: an accumulator's register s as it stands.
        static_for<0, 4>([&](auto j_) {
            constexpr int j = j_;
            if (wave != j) return;
            f32x4 T[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                T[j][i] = sD[(16 * j + 4 * g + i) * 20 + c];
                sM[(16 * j + 4 * g + i) * LD + 16 * j + c] = T[j][i];
                if (j & 1) sM[(16 * (j - 1) + 4 * g + i) * LD + 16 * j + c] = 0.f;
            }
            static_for<j + 1, 4>([&](auto i_) {
                constexpr int i = i_;
                f32x4 s = {0.f, 0.f, 0.f, 0.f}, r = {0.f, 0.f, 0.f, 0.f};
                static_for<j, i>([&](auto m_) {
                    constexpr int m = m_;
                    const f32x4 av = *reinterpret_cast<const f32x4*>(sA + (16 * i + c) * LD + 16 * m + 4 * g);
#pragma unroll
                    for (int e = 0; e < 4; e++) s = __builtin_amdgcn_mfma_f32_16x16x4f32(av[e], T[m][e], s, 0, 0, 0);
                });
                const f32x4 dv = *reinterpret_cast<const f32x4*>(sD + (16 * i + c) * 20 + 4 * g);
#pragma unroll
                for (int e = 0; e < 4; e++) r = __builtin_amdgcn_mfma_f32_16x16x4f32(dv[e], s[e], r, 0, 0, 0);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    T[i][e] = -r[e];
                    sM[(16 * i + 4 * g + e) * LD + 16 * j + c] = T[i][e];
                }
            });
        });
        __syncthreads();
        write_frags(tp);
        __syncthreads();
    }
}

template <int DT, int DK>
constexpr size_t prep_lds() {
    return 2 * KqUnit<DK, DT ? 1 : 3>::kOne + (2 * 64 * 68 + 4 * 16 * 20 + 3 * 64) * 4 + 64 * 8;
}

template <int DT, int DK, int DV, bool O32>  // O32: the output goes to the workspace, for the gated norm
__global__ __launch_bounds__(256) void k_delta_chunks(DeltaArgs a, DeltaWs ws, int c0, int ncs) {
    constexpr int NP = DT ? 1 : 3, KS = DK / 32;
    typedef KqUnit<DK, NP> Unit;
    __shared__ __attribute__((aligned(16))) uint8_t sS[KS][3][1024], sX[2][3][1024], sU[2][3][1024], sW[2][3][1024];
    // a head's slices at block numbers apart by the number of heads: on one XCD where that is a multiple of eight
    const int units = a.v_heads * a.n_seq, hu = blockIdx.x % units, slice = blockIdx.x / units;
    const int h = hu % a.v_heads, b = hu / a.v_heads, kh = key_head(a, h);
    const int len = a.lens ? min(max(a.lens[b], 0), a.n) : a.n;
    const int nc = min(ncs, (len + kChunk - 1) / kChunk - c0);
    if (nc <= 0) return;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int c = lane & 15, g = lane >> 4, col = 16 * slice + c;
    const int tok = 16 * wave + 4 * g;  // this lane's four tokens of a chunk
    const size_t row0 = (size_t)b * a.n + (size_t)c0 * kChunk;
    const int left = len - c0 * kChunk;

    f32x4 S[2];  // wave < KS: tile j, register i: dim 32 wave + 8 g + 4 j + i
    float* state = a.state + ((size_t)b * a.v_heads + h) * (DK * DV) + col;
    if (wave < KS)
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) S[j][i] = state[(32 * wave + 8 * g + 4 * j + i) * DV];

    // a chunk's operands: each is loaded again for the next chunk right after its last use
    bf16x8 fK[KS][NP], fQ[KS][NP], fKT[4][NP], fT[2][3], fP[2][3];
    f32x4 vb, vk, vq, vw;
    float end;
    uint32_t val[4];  // values as they lie in memory: nothing waits for them here
    auto kq = [&](int ch) { return ws.kq + ((size_t)(b * ncs + ch) * a.k_heads + kh) * Unit::kBytes + lane * 16; };
    auto tp = [&](int ch) { return ws.tp + ((size_t)(b * ncs + ch) * a.v_heads + h) * kTpBytes + lane * 16; };
    auto vec = [&](int ch) { return ws.vec + ((size_t)(b * ncs + ch) * a.v_heads + h) * kVec; };
    auto frag = [](const uint8_t* p) { return *reinterpret_cast<const bf16x8*>(p); };
    auto load_kq = [&](int ch) {
        const uint8_t* p = kq(ch);
#pragma unroll
        for (int s = 0; s < KS; s++)
#pragma unroll
            for (int i = 0; i < NP; i++) {
                fK[s][i] = frag(p + ((i * 4 + wave) * KS + s) * 1024);
                fQ[s][i] = frag(p + Unit::kOne + ((i * 4 + wave) * KS + s) * 1024);
            }
    };
    // (no load is conditional: a wave without an operand loads one of another's, so that no branch waits for loads)
    auto load_kt = [&](int ch) {
        const uint8_t* p = kq(ch) + 2 * Unit::kOne;
#pragma unroll
        for (int f = 0; f < 4; f++)
#pragma unroll
            for (int i = 0; i < NP; i++) fKT[f][i] = frag(p + ((i * KS + wave % KS) * 4 + f) * 1024);
    };
    const int f0 = wave < 2 ? wave : 2 * (wave - 1), f1 = wave < 2 ? f0 : f0 + 1;  // this row tile's two steps
    auto load_tri = [&](bf16x8 (&to)[2][3], const uint8_t* p) {
#pragma unroll
        for (int i = 0; i < 3; i++) {
            to[0][i] = frag(p + (i * kTriFrags + f0) * 1024);
            to[1][i] = frag(p + (i * kTriFrags + f1) * 1024);
        }
    };
    auto load_x = [&](int ch) {
        vb = *reinterpret_cast<const f32x4*>(vec(ch) + tok);
        vk = *reinterpret_cast<const f32x4*>(vec(ch) + 64 + tok);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const size_t at = (row0 + min(ch * kChunk + tok + i, left - 1)) * a.v_stride + h * DV + col;
            val[i] = DT ? static_cast<const uint16_t*>(a.v)[at] : static_cast<const uint32_t*>(a.v)[at];
        }
    };
    auto load_o = [&](int ch) { vq = *reinterpret_cast<const f32x4*>(vec(ch) + 128 + tok); };
    auto load_u = [&](int ch) {
        vw = *reinterpret_cast<const f32x4*>(vec(ch) + 192 + tok);
        end = vec(ch)[256];
    };
    load_kq(0), load_x(0), load_tri(fT, tp(0)), load_u(0), load_kt(0), load_o(0), load_tri(fP, tp(0) + kTpOne);

    auto put_state = [&] {
        if (KS == 4 || wave < KS) {
            const float v[8] = {S[0][0], S[0][1], S[0][2], S[0][3], S[1][0], S[1][1], S[1][2], S[1][3]};
            u32x4 w[3];
            split3(v, w);
#pragma unroll
            for (int p = 0; p < 3; p++) *reinterpret_cast<u32x4*>(sS[wave][p] + lane * 16) = w[p];
        }
    };
    // four tokens of a column as the halves of a right operand's fragments (k: 32 tokens, column c)
    const int put_at = (c + 16 * (2 * (wave & 1) + (g >> 1))) * 16 + (g & 1) * 8;
    auto put_rows = [&](uint8_t (&to)[2][3][1024], const f32x4 v) {
        uint32_t lo[3], hi[3];
        split3(v[0], v[1], lo), split3(v[2], v[3], hi);
#pragma unroll
        for (int p = 0; p < 3; p++) *reinterpret_cast<u32x2*>(to[wave >> 1][p] + put_at) = u32x2{lo[p], hi[p]};
    };
    auto get = [&](const uint8_t (&from)[3][1024], bf16x8 (&b)[3]) {
#pragma unroll
        for (int p = 0; p < 3; p++) b[p] = frag(from[p] + lane * 16);
    };
    put_state();
#pragma unroll 1
    for (int ch = 0; ch < nc; ch++) {
        const int next = min(ch + 1, nc - 1);
        lds_barrier();  // S is in the LDS
        f32x4 ks[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}}, qs[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int s = 0; s < KS; s++) {
            bf16x8 bs[3];
            get(sS[s], bs);
            ks[s & 1] = mfma_parts<NP>(fK[s], bs, ks[s & 1]);
            qs[s & 1] = mfma_parts<NP>(fQ[s], bs, qs[s & 1]);
        }
        load_kq(next);
        f32x4 x;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float v = ch * kChunk + tok + i < left ? __uint_as_float(DT ? val[i] << 16 : val[i]) : 0.f;
            x[i] = vb[i] * v - vk[i] * (ks[0][i] + ks[1][i]);
        }
        put_rows(sX, x);
        load_x(next);
        lds_barrier();  // X
        f32x4 u = {0.f, 0.f, 0.f, 0.f};
        {
            bf16x8 bx[3];
            get(sX[0], bx);
            u = mfma_parts<3>(fT[0], bx, u);
            if (wave >= 2) {
                get(sX[1], bx);
                u = mfma_parts<3>(fT[1], bx, u);
            }
        }
        load_tri(fT, tp(next));
        f32x4 w;
#pragma unroll
        for (int i = 0; i < 4; i++) w[i] = vw[i] * u[i];
        put_rows(sW, w);
        put_rows(sU, u);
        lds_barrier();  // U, and with the scales of K^T's columns
        if (KS == 4 || wave < KS) {
            bf16x8 bw[3];
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) S[j][i] *= end;
#pragma unroll
            for (int st = 0; st < 2; st++) {
                get(sW[st], bw);
#pragma unroll
                for (int j = 0; j < 2; j++) S[j] = mfma_parts<NP>(fKT[2 * j + st], bw, S[j]);
            }
            put_state();  // (every wave has read the one before: it passed the barrier behind X)
        }
        load_u(next), load_kt(next);
        f32x4 o;
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = vq[i] * (qs[0][i] + qs[1][i]);
        {
            bf16x8 bu[3];
            get(sU[0], bu);
            o = mfma_parts<3>(fP[0], bu, o);
            if (wave >= 2) {
                get(sU[1], bu);
                o = mfma_parts<3>(fP[1], bu, o);
            }
        }
        load_o(next), load_tri(fP, tp(next) + kTpOne);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int t = ch * kChunk + tok + i;
            if (t < left) {
                if constexpr (O32) ws.o[((row0 + t) * a.v_heads + h) * DV + col] = o[i];
                else store_out<DT>(a.out, (row0 + t) * a.out_stride + h * DV + col, o[i]);
            }
        }
    }
    if (wave < KS)
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) state[(32 * wave + 8 * g + 4 * j + i) * DV] = S[j][i];
}

// The gated norm behind the chunks: half a wave a (row, head).
template <int DT, int DV>
__global__ __launch_bounds__(256) void k_delta_norm(DeltaArgs a, const float* o32) {
    constexpr int N = DV / 32;
    const size_t i = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int d = (threadIdx.x & 31) * N;
    if (i >= (size_t)a.n_seq * a.n * a.v_heads) return;
    const size_t r = i / a.v_heads;
    const int h = i % a.v_heads, b = r / a.n;
    if (a.lens && (int)(r % a.n) >= a.lens[b]) return;
    float o[N], z[N], ss = 0.f;
    load_vec<0, N>(o32, i * DV + d, o);
    load_vec<DT, N>(a.z, r * a.z_stride + h * DV + d, z);
#pragma unroll
    for (int e = 0; e < N; e++) ss = fmaf(o[e], o[e], ss);
    const float rms = rsqrtf(sum32(ss) * (1.f / DV) + a.eps);
#pragma unroll
    for (int e = 0; e < N; e++)
        store_out<DT>(a.out, r * a.out_stride + h * DV + d + e, o[e] * (rms * a.gamma[d + e] * (z[e] * sigmoid(z[e]))));
}

// Token by token up to this many, and where every state is kept.
constexpr int kStepMost = 16;
// Chunks of a call are worked off in segments of about this many (chunk, value head) pairs at a time, whose
// workspace (60 KB a pair in bf16, 108 KB in fp32) stays in the last-level cache.
constexpr int kSegmentPairs = 2048;

static bool by_steps(const DeltaArgs& a) { return a.snap || a.n <= kStepMost; }
static int segment_chunks(const DeltaArgs& a) {
    const int nc = (a.n + kChunk - 1) / kChunk;
    const long long pairs = (long long)a.n_seq * a.v_heads;
    return (int)std::max(1ll, std::min<long long>(nc, kSegmentPairs / pairs));
}
static size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

struct DeltaSizes {
    size_t kq, tp, vec, o;
};
static DeltaSizes delta_sizes(const DeltaArgs& a, bool bf16) {
    const size_t chunks = (size_t)a.n_seq * segment_chunks(a);
    return {up256(chunks * a.k_heads * (bf16 ? 1 : 3) * 3 * kChunk * a.key_dim * 2), up256(chunks * a.v_heads * kTpBytes),
            up256(chunks * a.v_heads * kVec * 4),
            a.z ? up256((size_t)a.n_seq * a.n * a.v_heads * a.val_dim * 4) : 0};
}
size_t delta_workspace(const DeltaArgs& a, bool bf16) {
    if (by_steps(a)) return 0;
    const DeltaSizes s = delta_sizes(a, bf16);
    return s.kq + s.tp + s.vec + s.o;
}

template <int DT, int DK, int DV>
static hipError_t delta_chunks(const DeltaArgs& a, hipStream_t s) {
    static std::atomic<uint64_t> raised{0};
    constexpr size_t lds = prep_lds<DT, DK>();
    if (const hipError_t e = raise_lds(reinterpret_cast<const void*>(&k_delta_prep<DT, DK>), lds, raised)) return e;
    const DeltaSizes z = delta_sizes(a, DT == 1);
    uint8_t* p = static_cast<uint8_t*>(a.ws);
    const DeltaWs ws{p, p + z.kq, reinterpret_cast<float*>(p + z.kq + z.tp),
                     a.z ? reinterpret_cast<float*>(p + z.kq + z.tp + z.vec) : nullptr};
    const int nc = (a.n + kChunk - 1) / kChunk, seg = segment_chunks(a);
    for (int c0 = 0; c0 < nc; c0 += seg) {
        const int ncs = std::min(seg, nc - c0);
        k_delta_prep<DT, DK><<<dim3(ncs, a.k_heads, a.n_seq), 256, lds, s>>>(a, ws, c0, ncs);
        const int grid = a.v_heads * a.n_seq * (DV / 16);
        if (a.z) k_delta_chunks<DT, DK, DV, true><<<grid, 256, 0, s>>>(a, ws, c0, ncs);
        else k_delta_chunks<DT, DK, DV, false><<<grid, 256, 0, s>>>(a, ws, c0, ncs);
    }
    if (a.z) {
        const size_t rows = (size_t)a.n_seq * a.n * a.v_heads;
        k_delta_norm<DT, DV><<<(unsigned)((rows + 7) / 8), 256, 0, s>>>(a, ws.o);
    }
    return hipGetLastError();
}

template <int DT, int DK>
static hipError_t delta_dims(const DeltaArgs& a, hipStream_t s) {
    if (by_steps(a)) return delta_step<DT, DK>(a, s);
    return a.val_dim == 64 ? delta_chunks<DT, DK, 64>(a, s) : delta_chunks<DT, DK, 128>(a, s);
}

hipError_t launch_delta(const DeltaArgs& a, bool bf16, hipStream_t s) {
    if (bf16) return a.key_dim == 64 ? delta_dims<1, 64>(a, s) : delta_dims<1, 128>(a, s);
    return a.key_dim == 64 ? delta_dims<0, 64>(a, s) : delta_dims<0, 128>(a, s);
}

}  // namespace qw

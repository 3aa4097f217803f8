// The gated delta rule (qwattn_delta_rule; the reference's shaders/deltanet.comp and shaders/gated_norm.comp).
// Per token and value head, with k and q the key head's rows over their 2-norms (q also over sqrt(DK)) and a state
// S [DK][DV] in fp32:
//   S <- e^g S;  u = beta (v - S^T k);  S <- S + k u^T;  o = S^T q;   z: o rsqrt(mean o^2 + eps) gamma silu(z)
#include <algorithm>
#include <atomic>

#include "common.hpp"
#include "kernels.hpp"

namespace qw {

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
            const float qr = rsqrtf(sum64(qq) + a.eps) * (DK == 128 ? 0.08838834764831845f : 0.125f);
            const float kr = rsqrtf(sum64(kk) + a.eps);
#pragma unroll
            for (int i = 0; i < DK / 64; i++) {
                q[i] *= qr, k[i] *= kr;
                sq[t][64 * i + lane] = q[i], sk[t][64 * i + lane] = k[i];
                kq = fmaf(q[i], k[i], kq);
            }
            kq = sum64(kq);
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
                const float rms = rsqrtf(sum64(ss) * (1.f / DV) + a.eps);
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
// have fp32's exponents, so nothing is scaled beforehand (the last parts of values below 2^-109 lose bits, a value from
// 2^128 - 2^119 on rounds to an infinite part).
//
// Every operand that k_delta_chunks reads lies in the workspace as matrix-core fragments, a contiguous kilobyte each:
//   per (sequence, chunk, key head):   K, Q  [part][16-token tile][32-dim step]   rows tokens, k dims (fp32; bf16 rows are
//                                            operands as they lie in q and k)
//                                      K^T   [part][32-dim step][tile 0, 1][32-token step]; row r of tile j is the dim
//                                            8 (r / 4) + 4 j + r % 4 of its step: accumulator registers of the two
//                                            tiles of S are then the next product's operand fragment as they stand
//   per (sequence, chunk, value head): T, P  [part][6: the 32-token steps of each 16-token row tile that it reaches]
//                                      five vectors: beta, and the row scales of K S, Q S and K^T U; e^(G_end)
// Where tokens are the summed index (K^T, T, P and the X and U beside them) lane group g of a 32-token step holds the
// tokens 4 g .. 4 g + 3 of its first 16 and of its second 16: accumulator registers again.
// That holds for a bf16 output too: where its terms cancel, 16 bits of them show in it. (Two parts of Q S and P U there:
// 4,096 tokens of 32 heads of 128 x 128 in 177 us instead of 183, but a quarter of the outputs that are 2^-13 of their
// terms beyond half a step of bf16.)
constexpr int kChunk = 64, kTriFrags = 6, kVec = 320;

struct DeltaWs {
    uint8_t* kq;   // K, Q, K^T units
    uint8_t* tp;   // T, P units
    float* vec;    // vectors
    float* o;      // fp32 outputs before the gated norm, [row][v_heads * val_dim]
};

template <int DK, int NP>
struct KqUnit {
    static constexpr int kSteps = DK / 32, kOne = NP * 4 * kSteps * 1024;
    static constexpr int kQ = NP == 3 ? kOne : 0, kKT = NP == 3 ? 2 * kOne : 0, kBytes = kKT + kOne;  // (K at 0)
};
constexpr int kTpOne = 3 * kTriFrags * 1024, kTpBytes = 2 * kTpOne;

// The six (or, with one part on the left, three) part products. Those of one order of magnitude share an accumulator:
// three short chains instead of one long one, whose steps would wait for each other (a wave has no other on its SIMD to
// fill the gaps).
template <int NP>
__device__ __forceinline__ void mfma_parts(const bf16x8 (&a)[NP], const bf16x8 (&b)[3], f32x4 (&c)[3]) {
    c[2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0], b[2], c[2], 0, 0, 0);
    c[1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0], b[1], c[1], 0, 0, 0);
    c[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0], b[0], c[0], 0, 0, 0);
    if constexpr (NP == 3) {
        c[2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[1], b[1], c[2], 0, 0, 0);
        c[1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[1], b[0], c[1], 0, 0, 0);
        c[2] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[2], b[0], c[2], 0, 0, 0);
    }
}
__device__ __forceinline__ void zero(f32x4 (&c)[3]) { c[0] = c[1] = c[2] = f32x4{0.f, 0.f, 0.f, 0.f}; }
__device__ __forceinline__ float sum(const f32x4 (&c)[3], int i) { return (c[2][i] + c[1][i]) + c[0][i]; }

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

// Running sum over the 64 lanes, in 64 bits: within rows of 16 lanes, then across them.
template <int CTRL, int ROWS>
__device__ __forceinline__ double scan_step(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)u, CTRL, ROWS, 0xF, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, ROWS, 0xF, true);
    return x + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double scan64(double x) {
    x = scan_step<0x111, 0xF>(x);  // row_shr 1, 2, 4, 8 (zeros shifted in)
    x = scan_step<0x112, 0xF>(x);
    x = scan_step<0x114, 0xF>(x);
    x = scan_step<0x118, 0xF>(x);
    x = scan_step<0x142, 0xA>(x);  // lane 15 of rows 0 and 2 to rows 1 and 3
    return scan_step<0x143, 0xC>(x);  // lane 31 to rows 2 and 3
}

// Lower triangle of 4 x 4 tiles: tile t of 10 is (row, column)
constexpr int kTriRow[12] = {0, 1, 1, 2, 2, 2, 3, 3, 3, 3, 3, 3}, kTriCol[12] = {0, 0, 1, 0, 1, 2, 0, 1, 2, 3, 3, 3};

template <int DT, int DK>
__global__ __launch_bounds__(256, 2) void k_delta_prep(DeltaArgs a, DeltaWs ws, int c0, int ncs) {
    constexpr int NP = DT ? 1 : 3, KS = DK / 32, LD = 68;  // LD: row length of the 64 x 64 matrices
    typedef KqUnit<DK, NP> Unit;
    extern __shared__ __attribute__((aligned(16))) uint8_t smem[];
    uint8_t* fk = smem;                                        // K and Q fragments, and in their place:
    uint8_t* fq = fk + Unit::kOne;
    float* sA = reinterpret_cast<float*>(smem);                // A
    float* sM = sA + 64 * LD;                                  // P, then T
    constexpr int kFirst = 2 * Unit::kOne > 2 * 64 * LD * 4 ? 2 * Unit::kOne : 2 * 64 * LD * 4;
    float* sD = reinterpret_cast<float*>(smem + kFirst);       // the inverses of A's diagonal blocks, rows of 20
    double* sG = reinterpret_cast<double*>(sD + 4 * 16 * 20);  // of four value heads: G (log2 units), beta
    float* sBeta = reinterpret_cast<float*>(sG + 4 * 64);
    float* sEnd = sBeta + 4 * 64;                              // of the head at work: e^(G_i - G at its row tile's end
    float* sSince = sEnd + 3 * 64;                             // before) and e^(that - G_j), a row a row tile 1 .. 3
    float* sRk = sSince + 64;
    float* sRq = sRk + 64;

    // a workgroup a key head, or (where those leave CUs idle) several, which share out its value heads
    const int cl = blockIdx.x, kh = blockIdx.y % a.k_heads, b = blockIdx.z, share = blockIdx.y / a.k_heads;
    const int shares = gridDim.y / a.k_heads;
    const int len = a.lens ? min(max(a.lens[b], 0), a.n) : a.n;
    const int t0 = (c0 + cl) * kChunk, nt = min(kChunk, len - t0);
    if (nt <= 0) return;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int c = lane & 15, g = lane >> 4;
    uint8_t* kq = ws.kq + ((size_t)(b * ncs + cl) * a.k_heads + kh) * Unit::kBytes;

    {  // DK / 8 lanes a row, 8 dims a lane: norms, parts, fragments (zeros past the last token). In the LDS a fragment's
       // piece of row r sits at row r ^ (4 step + group): the pieces that a wave writes at once lie on different banks.
        constexpr int LPR = DK / 8, RPP = 256 / LPR;  // lanes a row, rows a pass
        const int d = (tid % LPR) * 8, s = d >> 5, dg = (d >> 3) & 3;
        float k[64 / RPP][8], q[64 / RPP][8];
#pragma unroll
        for (int p = 0; p < 64 / RPP; p++) {
            const size_t r = (size_t)b * a.n + t0 + min(p * RPP + tid / LPR, nt - 1);
            load_vec<DT, 8>(a.k, r * a.k_stride + kh * DK + d, k[p]);
            load_vec<DT, 8>(a.q, r * a.q_stride + kh * DK + d, q[p]);
        }
#pragma unroll
        for (int p = 0; p < 64 / RPP; p++) {
            const int row = p * RPP + tid / LPR;
            float k2 = 0.f, q2 = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                if (row >= nt) k[p][e] = q[p][e] = 0.f;
                k2 = fmaf(k[p][e], k[p][e], k2), q2 = fmaf(q[p][e], q[p][e], q2);
            }
            u32x4 kp[3], qp[3];
            split3(k[p], kp), split3(q[p], qp);
#pragma unroll
            for (int i = 0; i < NP; i++) {
                const int frag = ((i * 4 + (row >> 4)) * KS + s) * 1024;
                const int at = frag + ((row & 15) + 16 * dg) * 16, sw = frag + (((row & 15) ^ (4 * s + dg)) + 16 * dg) * 16;
                *reinterpret_cast<u32x4*>(fk + sw) = kp[i];
                *reinterpret_cast<u32x4*>(fq + sw) = qp[i];
                if (NP == 3 && share == 0) {
                    *reinterpret_cast<u32x4*>(kq + at) = kp[i];
                    *reinterpret_cast<u32x4*>(kq + Unit::kQ + at) = qp[i];
                }
            }
            auto row_sum = [](float x) {  // over the row's lanes
                x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0xB1, 0xF, 0xF, false));
                x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x4E, 0xF, 0xF, false));
                x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x141, 0xF, 0xF, false));
                if (LPR == 16) x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x140, 0xF, 0xF, false));
                return x;
            };
            k2 = row_sum(k2), q2 = row_sum(q2);
            if (d == 0) {
                sRk[row] = row < nt ? rsqrtf(k2 + a.eps) : 0.f;
                sRq[row] = (row < nt ? rsqrtf(q2 + a.eps) : 0.f) * (DK == 128 ? 0.08838834764831845f : 0.125f);
            }
        }
    }
    // this workgroup's value heads
    const int all = a.v_heads / a.k_heads, R = (all - share + shares - 1) / shares;
    auto head = [&](int i) {
        const int hi = share + i * shares;
        return a.tiled ? kh + hi * a.k_heads : kh * all + hi;
    };
    __syncthreads();
    auto frag = [&](const uint8_t* f, int part, int tile, int s) {
        return *reinterpret_cast<const bf16x8*>(f + ((part * 4 + tile) * KS + s) * 1024 + ((c ^ (4 * s + g)) + 16 * g) * 16);
    };
    // K^T of the row tile `wave`, by products with the unit matrix (exact): its accumulators hold four tokens of a dim
#pragma unroll
    for (int j = 0; j < 2; j++) {
        if (share) break;
        bf16x8 unit;
#pragma unroll
        for (int e = 0; e < 8; e++) unit[e] = 8 * g + e == 8 * (c >> 2) + 4 * j + (c & 3) ? (__bf16)1.f : (__bf16)0.f;
#pragma unroll
        for (int p = 0; p < NP; p++)
#pragma unroll
            for (int s = 0; s < KS; s++) {
                const f32x4 z = {0.f, 0.f, 0.f, 0.f};
                const f32x4 v = __builtin_amdgcn_mfma_f32_16x16x32_bf16(frag(fk, p, wave, s), unit, z, 0, 0, 0);
                *reinterpret_cast<u32x2*>(kq + Unit::kKT + (((p * KS + s) * 2 + j) * 2 + (wave >> 1)) * 1024 + lane * 16 +
                                          (wave & 1) * 8) = u32x2{pk_bf16(v[0], v[1]), pk_bf16(v[2], v[3])};
            }
    }
    // K K^T and Q K^T: tiles wave, wave + 4, wave + 8 of the lower triangle's ten
    f32x4 kk[3], qk[3];
#pragma unroll
    for (int m = 0; m < 3; m++) {
        const int ti = kTriRow[wave + 4 * m], tj = kTriCol[wave + 4 * m];
        kk[m] = qk[m] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (wave + 4 * m >= 10) break;
        f32x4 ck[3], cq[3];
        zero(ck), zero(cq);
#pragma unroll
        for (int s = 0; s < KS; s++) {
            bf16x8 ak[NP], aq[NP], bk[3];
#pragma unroll
            for (int p = 0; p < NP; p++) ak[p] = frag(fk, p, ti, s), aq[p] = frag(fq, p, ti, s), bk[p] = frag(fk, p, tj, s);
            if constexpr (NP == 3) {
                mfma_parts<3>(ak, bk, ck);
                mfma_parts<3>(aq, bk, cq);
            } else {
                ck[s % 3] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ak[0], bk[0], ck[s % 3], 0, 0, 0);
                cq[s % 3] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(aq[0], bk[0], cq[s % 3], 0, 0, 0);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) kk[m][i] = sum(ck, i), qk[m][i] = sum(cq, i);
    }

    __syncthreads();  // the fragments' place is free
#pragma unroll 1
    for (int hi = 0; hi < R; hi++) {
        const int slot = hi & 3;
        const size_t unit = (size_t)(b * ncs + cl) * a.v_heads + head(hi);
        if (slot == 0) {  // the gates of the next four heads, a wave a head, a lane a token. G in 64 bits (its differences
                          // are what counts), each g at least -2000 (e^g is 0 from -104 on; sums of -inf have none); a
                          // NaN stays one (fmaxf would make it -2000)
            if (hi + wave < R) {
                const int h = head(hi + wave);
                const size_t r = (size_t)b * a.n + t0 + min(lane, nt - 1);
                const float given = delta_log_decay(a, r, h), lg = given < -2000.f ? -2000.f : given, be = delta_beta(a, r, h);
                const double G = scan64(lane < nt ? (double)lg * 1.4426950408889634074 : 0.0);
                const uint64_t u = __builtin_bit_cast(uint64_t, G);
                const double end = __builtin_bit_cast(
                    double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(u >> 32), 63) << 32 |
                                (uint32_t)__builtin_amdgcn_readlane((int)u, 63));
                const float beta = lane < nt ? be : 0.f, since = exp2_fast((float)G), rk = sRk[lane];
                sG[wave * 64 + lane] = G, sBeta[wave * 64 + lane] = beta;
                float* v = ws.vec + ((size_t)(b * ncs + cl) * a.v_heads + h) * kVec + lane;
                v[0] = beta;
                v[64] = beta * since * rk;
                v[128] = sRq[lane] * since;
                v[192] = rk * exp2_fast((float)(end - G));
                if (lane == 0) v[256] = exp2_fast((float)end);
            }
            __syncthreads();
        }
        {  // decays over more than a tile are a product of two, through the end of the tile before the row's
            const double* G = sG + slot * 64;
            if (wave < 3) sEnd[wave * 64 + lane] = lane < 16 * (wave + 1) ? exp2_fast((float)(G[16 * wave + 15] - G[lane])) : 0.f;
            else sSince[lane] = lane < 16 ? 0.f : exp2_fast((float)(G[lane] - G[(lane & 48) - 1]));
        }
        __syncthreads();
        {
            const double* G = sG + slot * 64;
#pragma unroll
            for (int m = 0; m < 3; m++) {
                const int ti = kTriRow[wave + 4 * m], tj = kTriCol[wave + 4 * m];
                if (wave + 4 * m >= 10) break;
                const int col = 16 * tj + c, row0 = 16 * ti + 4 * g;
                const float rkj = sRk[col];
                const f32x4 be = *reinterpret_cast<const f32x4*>(sBeta + slot * 64 + row0);
                const f32x4 rk = *reinterpret_cast<const f32x4*>(sRk + row0), rq = *reinterpret_cast<const f32x4*>(sRq + row0);
                f32x4 d;
                if (ti == tj) {
                    const double Gj = G[col];
#pragma unroll
                    for (int i = 0; i < 4; i++) d[i] = 4 * g + i >= c ? exp2_fast((float)(G[row0 + i] - Gj)) * rkj : 0.f;
                } else {
                    const f32x4 since = *reinterpret_cast<const f32x4*>(sSince + row0);
                    const float e = sEnd[(ti - 1) * 64 + col] * rkj;
#pragma unroll
                    for (int i = 0; i < 4; i++) d[i] = since[i] * e;
                }
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    sA[(row0 + i) * LD + col] = ti > tj || 4 * g + i > c ? be[i] * rk[i] * d[i] * kk[m][i] : 0.f;
                    sM[(row0 + i) * LD + col] = rq[i] * d[i] * qk[m][i];
                }
                if (ti == tj && (tj & 1))  // the tile above, read as zeros by its row tile's 32-token step
#pragma unroll
                    for (int i = 0; i < 4; i++) sM[(row0 - 16 + i) * LD + col] = 0.f;
            }
        }
        __syncthreads();
        uint8_t* tp = ws.tp + unit * kTpBytes;
        auto write_frags = [&](uint8_t* to) {
            for (int i = tid; i < kTriFrags * 64; i += 256) {
                const int f = i >> 6, l = i & 63;
                const int tile = f < 2 ? f : 1 + (f >> 1), step = f < 2 ? 0 : f & 1;
                const float* from = sM + (16 * tile + (l & 15)) * LD + 32 * step + 4 * (l >> 4);
                const f32x4 v0 = *reinterpret_cast<const f32x4*>(from), v1 = *reinterpret_cast<const f32x4*>(from + 16);
                const float v[8] = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
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
    constexpr int one = KqUnit<DK, DT ? 1 : 3>::kOne, first = 2 * one > 2 * 64 * 68 * 4 ? 2 * one : 2 * 64 * 68 * 4;
    return first + (4 * 16 * 20 + (4 + 3 + 1 + 2) * 64) * 4 + 4 * 64 * 8;
}

// Waves 0 .. 3 carry the state: row tile w of X and U, dims 32 w .. of S. Waves 4 .. 7, beside them on the same SIMDs,
// compute and store the row tiles of the output, which nothing waits for.
template <int DT, int DK, int DV, bool O32>  // O32: the output goes to the workspace, for the gated norm
__global__ __launch_bounds__(512) void k_delta_chunks(DeltaArgs a, DeltaWs ws, int c0, int ncs) {
    constexpr int NP = DT ? 1 : 3, KS = DK / 32;
    typedef KqUnit<DK, NP> Unit;
    __shared__ __attribute__((aligned(16))) uint8_t sS[KS][3][1024], sX[2][3][1024], sW[2][3][1024];
    __shared__ f32x4 sU[4][64];      // U as it leaves the accumulators
    __shared__ f32x4 sK[KS][4][64];  // K S by parts: [dims' wave][row tile]
    // a head's slices at block numbers apart by the number of heads: on one XCD where that is a multiple of eight
    const int units = a.v_heads * a.n_seq, hu = blockIdx.x % units, slice = blockIdx.x / units;
    const int h = hu % a.v_heads, b = hu / a.v_heads, kh = key_head(a, h);
    const int len = a.lens ? min(max(a.lens[b], 0), a.n) : a.n;
    const int nc = min(ncs, (len + kChunk - 1) / kChunk - c0);
    if (nc <= 0) return;
    const int wave8 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = wave8 & 3, lane = threadIdx.x & 63;
    const int c = lane & 15, g = lane >> 4;
    const int tok = 16 * wave + 4 * g;  // this lane's four tokens of a chunk
    const size_t row0 = (size_t)b * a.n + (size_t)c0 * kChunk;
    const int left = len - c0 * kChunk;

    // A chunk's operands: each is loaded again for the next chunk right after its last use. Addresses are a uniform base
    // that moves on by a chunk and a lane offset; no load is conditional (a wave without an operand loads one of
    // another's), so that no branch waits for loads.
    const uint32_t lane16 = lane * 16;
    const size_t kq_step = (size_t)a.k_heads * Unit::kBytes, tp_step = (size_t)a.v_heads * kTpBytes;
    const size_t vec_step = (size_t)a.v_heads * kVec * 4;
    const uint8_t* kq = ws.kq + ((size_t)b * ncs * a.k_heads + kh) * Unit::kBytes;
    const uint8_t* tp = ws.tp + ((size_t)b * ncs * a.v_heads + h) * kTpBytes;
    const uint8_t* vec = reinterpret_cast<const uint8_t*>(ws.vec + ((size_t)b * ncs * a.v_heads + h) * kVec);
    auto frag = [&](const uint8_t* p) { return *reinterpret_cast<const bf16x8*>(p + lane16); };
    auto vec4 = [&](int which) { return *reinterpret_cast<const f32x4*>(vec + 256 * which + (uint32_t)tok * 4); };
    bf16x8 fM[2][3];  // T or P
    // bf16 K and Q: the fragment of row tile i and dim step s as the rows lie in memory, rows past the last as the last
    // one (their results are multiplied by zero, or not stored)
    auto raw = [&](const void* base, size_t stride, int ch, int i, int s) {
        const int r = min(16 * i + c, left - 1 - ch * kChunk);
        return *reinterpret_cast<const bf16x8*>(static_cast<const uint16_t*>(base) + (row0 + (size_t)ch * kChunk) * stride + kh * DK +
                                                32 * s + ((size_t)r * stride + 8 * g));
    };
    const int f0 = wave < 2 ? wave : 2 * (wave - 1), f1 = wave < 2 ? f0 : f0 + 1;  // this row tile's two steps
    auto load_tri = [&](const uint8_t* p) {
#pragma unroll
        for (int i = 0; i < 3; i++) {
            fM[0][i] = frag(p + (i * kTriFrags + f0) * 1024);
            fM[1][i] = frag(p + (i * kTriFrags + f1) * 1024);
        }
    };
    auto get = [&](const uint8_t (&from)[3][1024], bf16x8 (&b)[3]) {
#pragma unroll
        for (int p = 0; p < 3; p++) b[p] = frag(from[p]);
    };
    // (selects: a branch between matrix instructions and the readers of their results was seen to lose the waits between)
    auto move_on = [&](bool more) {
        kq += more ? kq_step : 0, tp += more ? tp_step : 0, vec += more ? vec_step : 0;
    };
    const uint32_t later = wave < 2 ? 0 : 0xFFFFFFFFu;  // the second 32 tokens are behind row tiles 0 and 1: as zeros
    if (wave8 >= 4) {
        f32x4 vq, acc[3];
        bf16x8 fQ[KS][NP];
        auto load_q = [&](int ch) {
            const uint8_t* p = kq + Unit::kQ + wave * (KS * 1024);
#pragma unroll
            for (int s = 0; s < KS; s++)
#pragma unroll
                for (int i = 0; i < NP; i++)
                    fQ[s][i] = NP == 1 ? raw(a.q, a.q_stride, ch, wave, s) : frag(p + (i * 4 * KS + s) * 1024);
        };
        const size_t stride = O32 ? (size_t)a.v_heads * DV : a.out_stride;
        size_t first = row0 * stride + h * DV + 16 * slice, at[4];
#pragma unroll
        for (int i = 0; i < 4; i++) at[i] = (tok + i) * stride + c;
        load_q(0), load_tri(tp + kTpOne), vq = vec4(2);
#pragma unroll 1
        for (int ch = 0; ch < nc; ch++) {
            move_on(ch + 1 < nc);
            lds_barrier();
            zero(acc);
#pragma unroll
            for (int s = 0; s < KS; s++) {
                bf16x8 bs[3];
#pragma unroll
                for (int p = 0; p < 3; p++) bs[p] = frag(sS[s][p]);
                mfma_parts<NP>(fQ[s], bs, acc);
            }
            load_q(min(ch + 1, nc - 1));
            f32x4 qs;
#pragma unroll
            for (int i = 0; i < 4; i++) qs[i] = vq[i] * sum(acc, i);
            lds_barrier();
            vq = vec4(2);
            zero(acc);
            acc[0] = qs;
            lds_barrier();
#pragma unroll
            for (int st = 0; st < 2; st++) {
                const f32x4 u0 = sU[2 * st][lane], u1 = sU[2 * st + 1][lane];
                float v[8] = {u0[0], u0[1], u0[2], u0[3], u1[0], u1[1], u1[2], u1[3]};
                if (st == 1)
#pragma unroll
                    for (int e = 0; e < 8; e++) v[e] = __uint_as_float(__float_as_uint(v[e]) & later);
                u32x4 w[3];
                split3(v, w);
                const bf16x8 bu[3] = {__builtin_bit_cast(bf16x8, w[0]), __builtin_bit_cast(bf16x8, w[1]),
                                      __builtin_bit_cast(bf16x8, w[2])};
                mfma_parts<3>(fM[st], bu, acc);
            }
            load_tri(tp + kTpOne);
            const int more = left - ch * kChunk - tok;
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (i < more) {
                    if constexpr (O32) ws.o[first + at[i]] = sum(acc, i);
                    else store_out<DT>(a.out, first + at[i], sum(acc, i));
                }
            first += kChunk * stride;
        }
        return;
    }

    f32x4 S[2];  // wave < KS: tile j, register i: dim 32 wave + 8 g + 4 j + i
    float* state = a.state + ((size_t)b * a.v_heads + h) * (DK * DV) + 16 * slice + c;
    if (wave < KS)
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) S[j][i] = state[(32 * wave + 8 * g + 4 * j + i) * DV];
    bf16x8 fK[4][NP], fKT[4][NP], bS[3];  // K's row tiles in this wave's dims; S as an operand
    f32x4 vb, vk, vw;
    float end;
    uint32_t val[4];  // values as they lie in memory: nothing waits for them here
    size_t first = row0 * a.v_stride + h * DV + 16 * slice, at[4];
#pragma unroll
    for (int i = 0; i < 4; i++) at[i] = (tok + i) * a.v_stride + c;
    auto load_k = [&](int ch) {
        const uint8_t* p = kq + wave % KS * 1024;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int q = 0; q < NP; q++)
                fK[i][q] = NP == 1 ? raw(a.k, a.k_stride, ch, i, wave % KS) : frag(p + (q * 4 + i) * (KS * 1024));
    };
    auto load_kt = [&] {
        const uint8_t* p = kq + Unit::kKT + wave % KS * 4096;
#pragma unroll
        for (int f = 0; f < 4; f++)
#pragma unroll
            for (int i = 0; i < NP; i++) fKT[f][i] = frag(p + (i * KS * 4 + f) * 1024);
        vw = vec4(3);
        end = *reinterpret_cast<const float*>(vec + 1024);
    };
    auto load_x = [&](int ch) {
        vb = vec4(0), vk = vec4(1);
        const int most = left - 1 - ch * kChunk;  // past the last row: that one (beta is 0 there)
#pragma unroll
        for (int i = 0; i < 4; i++) at[i] = min(tok + i, most) * a.v_stride + c;
#pragma unroll
        for (int i = 0; i < 4; i++)
            val[i] = DT ? static_cast<const uint16_t*>(a.v)[first + at[i]] : static_cast<const uint32_t*>(a.v)[first + at[i]];
    };
    auto put_state = [&] {
        if (KS == 4 || wave < KS) {
            const float v[8] = {S[0][0], S[0][1], S[0][2], S[0][3], S[1][0], S[1][1], S[1][2], S[1][3]};
            u32x4 w[3];
            split3(v, w);
#pragma unroll
            for (int p = 0; p < 3; p++) {
                *reinterpret_cast<u32x4*>(sS[wave][p] + lane16) = w[p];  // for Q S
                bS[p] = __builtin_bit_cast(bf16x8, w[p]);
            }
        }
    };
    // four tokens of a column: half of a right operand's piece
    auto put_rows = [&](uint8_t (&to)[2][3][1024], const f32x4 v) {
        uint32_t lo[3], hi[3];
        split3(v[0], v[1], lo), split3(v[2], v[3], hi);
#pragma unroll
        for (int p = 0; p < 3; p++)
            *reinterpret_cast<u32x2*>(to[wave >> 1][p] + lane16 + (wave & 1) * 8) = u32x2{lo[p], hi[p]};
    };
    load_k(0), load_x(0), load_tri(tp);
    put_state();
    __builtin_amdgcn_s_setprio(2);  // ahead of the output waves
#pragma unroll 1
    for (int ch = 0; ch < nc; ch++) {
        // every row tile's K S over this wave's dims, whose rows of S are in its registers
        if (KS == 4 || wave < KS) {
            f32x4 part[4][3];
#pragma unroll
            for (int i = 0; i < 4; i++) zero(part[i]);
#pragma unroll
            for (int i = 0; i < 4; i++) mfma_parts<NP>(fK[i], bS, part[i]);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                f32x4 v;
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = sum(part[i], e);
                sK[wave][i][lane] = v;
            }
        }
        lds_barrier();  // K S by parts, and S
        f32x4 acc[3], x, w, ks = sK[0][wave][lane];
#pragma unroll
        for (int s = 1; s < KS; s++) {
            const f32x4 v = sK[s][wave][lane];
#pragma unroll
            for (int e = 0; e < 4; e++) ks[e] += v[e];
        }
        // (the next loads go out while the LDS answers, here and below)
        load_kt();
        move_on(ch + 1 < nc);
        first += ch + 1 < nc ? kChunk * a.v_stride : 0;
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = vb[i] * __uint_as_float(DT ? val[i] << 16 : val[i]) - vk[i] * ks[i];
        put_rows(sX, x);
        lds_barrier();  // X
        bf16x8 bx[2][3];
        get(sX[0], bx[0]), get(sX[1], bx[1]);
        load_k(min(ch + 1, nc - 1)), load_x(min(ch + 1, nc - 1));
#pragma unroll
        for (int p = 0; p < 3; p++) {
            u32x4 v = __builtin_bit_cast(u32x4, bx[1][p]);
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] &= later;
            bx[1][p] = __builtin_bit_cast(bf16x8, v);
        }
        zero(acc);
        mfma_parts<3>(fM[0], bx[0], acc);
        mfma_parts<3>(fM[1], bx[1], acc);
#pragma unroll
        for (int i = 0; i < 4; i++) x[i] = sum(acc, i), w[i] = vw[i] * x[i];
        put_rows(sW, w);
        sU[wave][lane] = x;
        lds_barrier();  // U, and with the scales of K^T's columns
        bf16x8 bw[2][3];
        get(sW[0], bw[0]), get(sW[1], bw[1]);
        load_tri(tp);
        if (KS == 4 || wave < KS) {
            f32x4 s[2][3];
#pragma unroll
            for (int j = 0; j < 2; j++) {
                zero(s[j]);
#pragma unroll
                for (int i = 0; i < 4; i++) s[j][0][i] = S[j][i] * end;
            }
#pragma unroll
            for (int st = 0; st < 2; st++)
#pragma unroll
                for (int j = 0; j < 2; j++) mfma_parts<NP>(fKT[2 * j + st], bw[st], s[j]);
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) S[j][i] = sum(s[j], i);
            put_state();  // (every wave has read the one before: it passed the barrier behind X)
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

// Token by token where every state is kept, and while that takes less: a token takes 1 us (up to 256 (sequence, value
// head) pairs, a workgroup each) to 5 us (1,536 pairs), a chunk of all pairs 16 us (32 pairs, bf16) to 267 (1,536), in fp32
// up to twice as much; the gated norm behind chunks 5 us and more. Measured with 32 heads of 128 x 128 without it, by
// tokens and in chunks: one sequence of 19 tokens 25 and 16 us (bf16), 22 (fp32); 4 of 48 tokens 54 and 31, 54 and 45; 8 of
// 64 tokens in fp32 74 and 99; 48 of 64 tokens in bf16 337 and 267.
static int step_most(const DeltaArgs& a, bool bf16) {
    const long long pairs = (long long)a.n_seq * a.v_heads;
    return (int)(bf16 ? std::min(18 + pairs / 10, 48ll) : std::min(18 + pairs / 6, 100ll));
}
// Chunks of a call are worked off in segments of about this many (chunk, value head) pairs at a time, whose
// workspace (45 KB a pair of two a key head in bf16, 109 KB in fp32) stays in the last-level cache.
constexpr int kSegmentPairs = 2048;

static bool by_steps(const DeltaArgs& a, bool bf16) { return a.snap || a.n <= step_most(a, bf16); }
static int segment_chunks(const DeltaArgs& a) {
    const int nc = (a.n + kChunk - 1) / kChunk;
    const long long pairs = (long long)a.n_seq * a.v_heads;
    return (int)std::max(1ll, std::min<long long>(nc, kSegmentPairs / pairs));
}

struct DeltaSizes {
    size_t kq, tp, vec, o;
};
static DeltaSizes delta_sizes(const DeltaArgs& a, bool bf16) {
    const size_t chunks = (size_t)a.n_seq * segment_chunks(a);
    return {up256(chunks * a.k_heads * (bf16 ? 1 : 9) * kChunk * a.key_dim * 2), up256(chunks * a.v_heads * kTpBytes),
            up256(chunks * a.v_heads * kVec * 4),
            a.z ? up256((size_t)a.n_seq * a.n * a.v_heads * a.val_dim * 4) : 0};
}
size_t delta_need(const DeltaArgs& a, bool bf16) {
    if (by_steps(a, bf16)) return 0;
    const DeltaSizes s = delta_sizes(a, bf16);
    return s.kq + s.tp + s.vec + s.o;
}
// Fewer tokens never need more. Fewer sequences can: a segment then has more whole chunks of each, and fewer tokens run
// token by token. With more pairs than a segment's both are at their end, and the need grows with the sequences.
size_t delta_workspace(DeltaArgs a, bool bf16) {
    size_t most = delta_need(a, bf16);
    for (int b = std::min(a.n_seq, kSegmentPairs / a.v_heads); b > 0; b--) {
        a.n_seq = b;
        most = std::max(most, delta_need(a, bf16));
    }
    return most;
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
        // 333 tokens of 16 key heads and 32 value heads in fp32: 21 us with a workgroup a key head, 18 with one a value head
        const int shares = (long long)ncs * a.v_heads * a.n_seq <= 256 ? a.v_heads / a.k_heads : 1;
        k_delta_prep<DT, DK><<<dim3(ncs, a.k_heads * shares, a.n_seq), 256, lds, s>>>(a, ws, c0, ncs);
        const int grid = a.v_heads * a.n_seq * (DV / 16);
        if (a.z) k_delta_chunks<DT, DK, DV, true><<<grid, 512, 0, s>>>(a, ws, c0, ncs);
        else k_delta_chunks<DT, DK, DV, false><<<grid, 512, 0, s>>>(a, ws, c0, ncs);
    }
    if (a.z) {
        const size_t rows = (size_t)a.n_seq * a.n * a.v_heads;
        k_delta_norm<DT, DV><<<(unsigned)((rows + 7) / 8), 256, 0, s>>>(a, ws.o);
    }
    return hipGetLastError();
}

template <int DT, int DK>
static hipError_t delta_dims(const DeltaArgs& a, hipStream_t s) {
    if (by_steps(a, DT == 1)) return delta_step<DT, DK>(a, s);
    return a.val_dim == 64 ? delta_chunks<DT, DK, 64>(a, s) : delta_chunks<DT, DK, 128>(a, s);
}

hipError_t launch_delta(const DeltaArgs& a, bool bf16, hipStream_t s) {
    if (bf16) return a.key_dim == 64 ? delta_dims<1, 64>(a, s) : delta_dims<1, 128>(a, s);
    return a.key_dim == 64 ? delta_dims<0, 64>(a, s) : delta_dims<0, 128>(a, s);
}

}  // namespace qw

// Device-side pieces shared by the kernels of the paged cache (paged.hip, paged_few.hip, paged_chunk.hip).
#pragma once
#include "common.hpp"
#include "kernels.hpp"

namespace qw {

// The sequence's new tokens: min(max(lens[b], 0), n)
__device__ __forceinline__ int seq_len(const int32_t* lens, int b, int n) { return lens ? min(max(lens[b], 0), n) : n; }

// Number, in either pool, of the block of KV head h that holds position p of a sequence, on page `page` (a pool has less
// than 2^31 blocks), and the elements before it.
__device__ __forceinline__ int paged_number(const PagedCache& c, int page, int p, int h, int nkv) {
    const int in_page = p & ((1 << c.lg_page) - 1);
    return (page * nkv + h) * (1 << (c.lg_page - 5)) + (in_page >> 5);
}
__device__ __forceinline__ int64_t paged_block(const PagedCache& c, int page, int p, int h, int nkv, int D) {
    return (int64_t)paged_number(c, page, p, h, nkv) * (kBlk * D);
}

// A sequence's first position, within +-2^28 (what lies further out is outside every table, as a position of 2^28 is), so
// that positions and windows (kNoWindow: none; others are at most `limit` <= 2^26) add up in 32 bits.
__device__ __forceinline__ int seq_pos(const int32_t* pos, int b) { return min(max(pos[b], -(1 << 28)), 1 << 28); }

// The key tiles of 2^LG positions that some of tokens [t0, t1) of a sequence sees, in order: tiles [0, sinks) (the first
// positions, where a window hides what follows them), then [first, first + count - sinks). Tokens outside
// the table's positions see none; tokens that see nothing still have one tile, so that their rows are written.
struct KeyTiles {
    int sinks, first, count;
    __device__ __forceinline__ int tile(int i) const { return i < sinks ? i : i - sinks + first; }
};
template <int LG>
__device__ __forceinline__ KeyTiles key_tiles(const PagedAttendArgs& a, int pos, int t0, int t1) {
    if (t0 >= t1) return {0, 0, 0};
    const int lo = max(pos + t0, 0), hi = min(pos + t1, a.limit) - 1;
    if (lo > hi) return {0, 0, 1};
    KeyTiles k;
    k.first = max(lo - a.window + 1, 0) >> LG;
    k.sinks = min((a.sinks + (1 << LG) - 1) >> LG, k.first);
    k.count = k.sinks + (hi >> LG) + 1 - k.first;
    return k;
}

// ceil(c / r) of 0 <= c <= 2^20, 1 <= r <= 2^20 (the quotient's error is below its distance from the next whole number, 1 / 2r)
__device__ __forceinline__ int parts_of(int c, float r) { return (int)(((float)c + r - 0.5f) * __builtin_amdgcn_rcpf(r)); }

// What a token at position p sees: keys [from, end) and [0, sinks) below end
struct Sight {
    int from, end;
    __device__ __forceinline__ bool sees(int j, int sinks) const { return (j < end) & ((j >= from) | (j < sinks)); }
};
__device__ __forceinline__ Sight sight(const PagedAttendArgs& a, int p) {
    return {p - a.window + 1, p >= 0 && p < a.limit ? p + 1 : 0};
}
// The keys that all of the tokens at positions [p0, p1] see
__device__ __forceinline__ Sight sight_of_all(const PagedAttendArgs& a, int p0, int p1) {
    return {p1 - a.window + 1, p0 >= 0 && p1 < a.limit ? p0 + 1 : 0};
}
// ... and that some of them see
__device__ __forceinline__ Sight sight_of_some(const PagedAttendArgs& a, int p0, int p1) {
    return {max(p0, 0) - a.window + 1, max(p0, 0) <= min(p1, a.limit - 1) ? min(p1, a.limit - 1) + 1 : 0};
}
// Whether s sees every key of [k0, k1)
__device__ __forceinline__ bool sees_whole(const Sight& s, int k0, int k1, int sinks) { return k1 <= s.end && (k0 >= s.from || k1 <= sinks); }

// ---- queries and weights as fp16 operands ----------------------------------------------------------------------
// A row of queries is scaled by the power of two that takes its largest magnitude to [2^14, 2^15) and split: the fp16
// nearest each value, and for fp32 rows (PARTS 2) the fp16 nearest what that leaves: 22 bits of the row's largest, and the
// 8 bits of bf16 rows whole. The scores' factor takes the power back. Keys and values are fp16 themselves, so a score
// is exact but for that and the fp32 sums.
__device__ __forceinline__ int query_shift(float largest) {
    return largest > 0.f && largest < __builtin_inff() ? min(max(15 - __builtin_amdgcn_frexp_expf(largest), -126), 126) : 0;
}
// 2^sh, |sh| <= 126
__device__ __forceinline__ float power_of_two(int sh) { return __uint_as_float((uint32_t)(127 + sh) << 23); }

// Weights are taken as 2^(score - maximum + kShift): with the lazy maximum (a weight may pass it by 2^kTau) they stay
// below fp16's largest, and the smallest are kept to 2^-24 of 2^kShift.
constexpr float kShift = 8.f, kTau = 7.f;

// fp16 parts of two weights: the nearest fp16, and what it leaves, 22 bits together. bf16 rows take both too: the values are
// fp16 whatever the rows are, and where their weighted sum cancels, an error of 2^-12 of a term is more than a step of the output.
constexpr int kWeightParts = 2;
__device__ __forceinline__ void weight_parts(float w0, float w1, f16x2& hi, f16x2& lo) {
    hi = f16x2{(f16)w0, (f16)w1}, lo = f16x2{(f16)(w0 - (float)hi[0]), (f16)(w1 - (float)hi[1])};
}

// ---- output rows -----------------------------------------------------------------------------------------------
// Four outputs of one row and head at dim d: o * inv, times sigmoid(gate), rounded once; zero for a row that saw nothing (inv 0),
// whatever its gate. The gates are loaded apart, so that many loads are in flight.
template <int DT>
struct Gate4 {
    typename std::conditional<DT == 0, f32x4, u32x2>::type v;
    __device__ __forceinline__ void none() {  // sigmoid(inf) is 1
        if constexpr (DT == 0) v = f32x4{1, 1, 1, 1} * __builtin_inff();
        else v = u32x2{0x7f807f80u, 0x7f807f80u};
    }
    __device__ __forceinline__ void load(const PagedAttendArgs& a, size_t row, int h, int d) {
        const size_t at = row * a.gate_stride + (size_t)h * a.gate_head + d;
        if constexpr (DT == 0) v = *reinterpret_cast<const f32x4*>(static_cast<const float*>(a.gate) + at);
        else v = *reinterpret_cast<const u32x2*>(static_cast<const uint16_t*>(a.gate) + at);
    }
    __device__ __forceinline__ float at(int i) const {
        if constexpr (DT == 0) return v[i];
        else return __uint_as_float((i & 1) ? v[i >> 1] & 0xffff0000u : v[i >> 1] << 16);
    }
};
template <int DT>
__device__ __forceinline__ void store_out4(const PagedAttendArgs& a, size_t row, int h, int D, int d, f32x4 o, float inv, const Gate4<DT>& g) {
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = inv == 0.f ? 0.f : o[i] * (inv * sigmoid(g.at(i)));
    const size_t at = row * a.out_stride + (size_t)h * D + d;
    if constexpr (DT == 0) *reinterpret_cast<f32x4*>(static_cast<float*>(a.out) + at) = o;
    else *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.out) + at) = u32x2{pk_bf16(o[0], o[1]), pk_bf16(o[2], o[3])};
}

// 1 / the sum of a row's weights; 0 for a row that saw nothing (a NaN stays)
__device__ __forceinline__ float inverse_sum(float l) { return l == 0.f ? 0.f : 1.0f / l; }

// Eight fp16 of V (one dim, keys k0 .. k0 + 7) with the keys that `keep` does not name zeroed
template <typename F>
__device__ __forceinline__ f16x8 keep_keys(f16x8 v, F&& keep) {
    u32x4 u = __builtin_bit_cast(u32x4, v);
#pragma unroll
    for (int i = 0; i < 4; i++) u[i] &= (keep(2 * i) ? 0x0000ffffu : 0u) | (keep(2 * i + 1) ? 0xffff0000u : 0u);
    return __builtin_bit_cast(f16x8, u);
}
// Nonzero where one of eight fp16 is an infinity or NaN
__device__ __forceinline__ uint32_t not_finite(f16x8 v) {
    const u32x4 u = __builtin_bit_cast(u32x4, v);
    uint32_t any = 0;
#pragma unroll
    for (int i = 0; i < 4; i++) any |= (u[i] & 0x7fff7fffu) + 0x04000400u;
    return any & 0x80008000u;
}

}  // namespace qw

// Attention of a few new tokens a sequence (decode, speculative verify) over a paged cache: up to 32 query rows a KV head.
//
// o = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m), s_j = scale q . k_j, in one pass: a wave keeps the maximum m, the sum and the
// unnormalized o of the keys it has seen (lazily: m moves where a row's maximum passes it by more than kTau). Parts of a key axis
// with (m, sum, o) join as m = max m_i, the others times e^(m_i - m), in a fixed order.
//
// Bound by memory: every page is read once, 4 D bytes a key and KV head. A wave holds one block of 32 keys and its values in
// flight, copied straight to the LDS (128 KB a CU at 256 dims), and takes the next keys where the scores are done, the next
// values where the weighted sums are. Measured with 16 heads over 2 KV heads of 256: 32 bf16 sequences of up to 16000 positions
// 110 to 116 us (578 MB: 5.0 to 5.2 TB/s, a large copy's 5.1), 8 sequences of 4 fp32 tokens at up to 8190 27 us (2.8 TB/s), one
// token at 32767 19.8 us (67 MB: 3.4 TB/s; kernel 17, joining 3.9), at 500 13.3 us: there the first workgroups' chain of loads
// (positions, pages, blocks: 10000 clocks) and code that is not in the instruction cache yet. A wave's block takes some 6300
// clocks beside its waits (one tile of rows; scores 1200 in fp32, 750 in bf16), a workgroup's four at a time; their bytes
// at the copy's rate take 15000.
#include "paged.hpp"

namespace qw {

namespace {

constexpr int kFewWaves = 4;                     // waves of a workgroup; each takes every fourth block of 32 keys
constexpr int kFewUnit = kFewWaves;              // blocks of a unit of the schedule
constexpr int few_occ(int D) { return D == 256 ? 1 : 2; }  // workgroups a CU, at most what its LDS holds
constexpr int kLdsBytes = 160 * 1024;                      // of a CU

// Units of extra length that whole parts may cost a workgroup: about what a second segment's start does (8 us, of 3 a unit).
// Measured with whole parts and with equal runs alone: 8 sequences of 4 tokens at up to 8190 25 and 31 us (bf16 26 and 30), 16 of
// one behind a window of 4096 30 and 34; 8 of 8 fp32 tokens over 2 KV heads of 128 18 and 20, 16 of one bf16 token there 28 and
// 30, 24 over 8 of 64 46.1 and 45.6. Many sequences of different ages take runs (their parts would be 20% longer).
constexpr int kFewSpare = 3;

// Workspace: the partial rows of two segments a workgroup (its first and its last), [slot][row][D] and [slot][row]
// (maximum, sum), then [0] units a KV head and [1] units a workgroup (or parts a KV head, and 0), and every sequence's
// first unit (part) and their number.
constexpr int kFewHead = 4;  // ints before the sequences'

struct FewPlan {
    int* head;
    float *o, *ml;
};
__host__ __device__ inline FewPlan few_plan(void* ws, int groups, int rows, int D) {
    char* p = static_cast<char*>(ws);
    FewPlan f;
    f.o = reinterpret_cast<float*>(p);
    f.ml = f.o + (size_t)2 * groups * rows * D;
    f.head = reinterpret_cast<int*>(f.ml + (size_t)2 * groups * rows * 2);
    return f;
}

// Sums of the lanes up to each one
__device__ __forceinline__ int scan64(int x) {
#define QW_STEP(ctrl, rows) x += __builtin_amdgcn_update_dpp(0, x, ctrl, rows, 0xf, false)
    QW_STEP(0x111, 0xf);  // row_shr:1, 2, 4, 8
    QW_STEP(0x112, 0xf);
    QW_STEP(0x114, 0xf);
    QW_STEP(0x118, 0xf);
    QW_STEP(0x142, 0xa);  // row_bcast:15 into rows 1 and 3
    QW_STEP(0x143, 0xc);  // row_bcast:31 into rows 2 and 3
#undef QW_STEP
    return x;
}

// Maximum over 8 or 16 neighbouring lanes, in each of them
template <int N>
__device__ __forceinline__ float max_lanes(float x) {
    static_assert(N == 8 || N == 16, "");
    auto with = [&](auto ctrl) {
        x = fmaxf(x, __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), decltype(ctrl)::value, 0xF, 0xF, false)));
    };
    with(std::integral_constant<int, 0xB1>{});   // quad_perm 1 0 3 2
    with(std::integral_constant<int, 0x4E>{});   // quad_perm 2 3 0 1
    with(std::integral_constant<int, 0x141>{});  // row_half_mirror
    if constexpr (N == 16) with(std::integral_constant<int, 0x140>{});  // row_mirror
    return x;
}

// r / G for r < 32: by = 2^16 / G + 1 is off by at most 1, r by / 2^16 by at most 2^-11, and r / G is at least 2^-5 below
// the next whole number
struct FewHeads {
    int G, by;
    __device__ __forceinline__ int token(int r) const { return r * by >> 16; }
};

template <int D, int DT, int NT>
struct FewCfg {
    static constexpr int PARTS = DT == 0 ? 2 : 1, NKS = D / 32, NDT = D / 16, ROWS = 16 * NT, BLKE = kBlk * D;
    static constexpr int Q_BYTES = PARTS * NT * NKS * 1024, KV_BYTES = kFewWaves * 2 * BLKE * 2;
    // score factors [ROWS]. Where queries and blocks of the CU's workgroups fill the LDS, the first wave's values make room for
    // them until the rows are laid out.
    static constexpr int EXTRA = ROWS * 4;
    static constexpr bool TIGHT = few_occ(D) * (Q_BYTES + KV_BYTES + EXTRA) > kLdsBytes;
    static constexpr int LDS = Q_BYTES + KV_BYTES + (TIGHT ? 0 : EXTRA);
    static_assert(few_occ(D) * LDS <= kLdsBytes, "the schedule's workgroups are all resident");
    static_assert(NDT % kFewWaves == 0, "every wave writes as many dim tiles");
    static_assert(2 * kFewWaves * ROWS * 4 <= Q_BYTES, "the waves' maxima and sums fit the queries' room");
    static_assert(kFewWaves * ROWS * D * 4 <= KV_BYTES, "the waves' accumulators fit the blocks' room");
};

// Waits until at most N vector loads are in flight (N < 64), and until every LDS read has returned; memory accesses stay
// on their side.
template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0F70);
    asm volatile("" ::: "memory");
}
__device__ __forceinline__ void wait_lds() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);
    asm volatile("" ::: "memory");
}

template <int D, int DT, int NT>
__global__ __launch_bounds__(64 * kFewWaves, few_occ(D)) void k_paged_few(PagedAttendArgs a, FewHeads heads, void* ws) {
    using C = FewCfg<D, DT, NT>;
    constexpr int PARTS = C::PARTS, NKS = C::NKS, NDT = C::NDT, ROWS = C::ROWS, BLKE = C::BLKE;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    f16* sq = reinterpret_cast<f16*>(smem);                              // query operands
    f16* kv = reinterpret_cast<f16*>(smem + C::Q_BYTES);                 // each wave's block of keys and of values
    float* red = reinterpret_cast<float*>(kv);                           // afterwards the waves' accumulators
    float* sm = reinterpret_cast<float*>(sq);                            // afterwards [waves][ROWS] maxima
    float* sl = sm + kFewWaves * ROWS;                                   // and sums
    float* sc = reinterpret_cast<float*>(C::TIGHT ? reinterpret_cast<unsigned char*>(kv + BLKE) : smem + C::Q_BYTES + C::KV_BYTES);
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int G = heads.G, groups = gridDim.x;
    const FewPlan plan = few_plan(ws, groups, ROWS, D);

    // ---- schedule, by every wave for itself: a sequence is ceil(blocks / 4) units a KV head, the units of KV head 0's
    // sequences come first. Where they can be cut into no more parts than there are workgroups, none of them more than
    // kFewSpare units longer than an equal share, a workgroup takes one part; else an equal run of units, which may end in
    // one sequence and begin in the next. A lane holds one sequence, or a run of them. ----
    const int per = (a.n_seq + 63) >> 6;
    const bool one = __builtin_expect(per == 1, true);
    auto units = [&](int pos, int len) { return (key_tiles<5>(a, pos, 0, len).count + kFewUnit - 1) / kFewUnit; };
    auto units_of = [&](int b) { return units(seq_pos(a.pos, b), seq_len(a.lens, b, a.n)); };
    int lane_pos = 0, lane_len = 0, mine = 0;
    if (one) {
        const int at = min(lane, a.n_seq - 1);
        lane_pos = seq_pos(a.pos, at), lane_len = seq_len(a.lens, at, a.n);
        mine = lane < a.n_seq ? units(lane_pos, lane_len) : 0;
    } else {
#pragma unroll 1
        for (int i = 0; i < per; i++)
            if (lane * per + i < a.n_seq) mine += units_of(lane * per + i);
    }
    int upto = scan64(mine), total = __builtin_amdgcn_readlane(upto, 63);
    const int64_t all = (int64_t)total * a.NKV;
    int run, parts = 0, b, u0, left, h;
    if (all == 0) return;  // (no sequence has new tokens: nothing is joined)
    if (__builtin_expect(all <= 1 << 20, true)) run = max(1, parts_of((int)all, (float)groups));
    else run = (int)((all + groups - 1) / groups);
    if (one && run < 1 << 20) {
#pragma unroll 1
        for (int k = 0; k <= kFewSpare; k++) {
            const int p = parts_of(mine, (float)(run + k)), scan = scan64(p), sum = __builtin_amdgcn_readlane(scan, 63);
            if (sum * a.NKV <= groups) {
                parts = p, upto = scan, total = sum, run = 0;
                break;
            }
        }
    }
    if (blockIdx.x == 0 && wave == 0) {  // for the kernel that joins split sequences
        int at = upto - (run ? mine : parts);
#pragma unroll 1
        for (int i = 0; i < per; i++)
            if (lane * per + i < a.n_seq) plan.head[kFewHead + lane * per + i] = at, at += one ? 0 : units_of(lane * per + i);
        if (lane == 0) plan.head[0] = total, plan.head[1] = run, plan.head[kFewHead + a.n_seq] = total;
    }
    if (__builtin_expect(!run, true)) {  // part `part` of `of`, the first ones a unit longer
        h = parts_of((int)blockIdx.x + 1, (float)total) - 1;
        if (h >= a.NKV) return;
        const int rest = (int)blockIdx.x - h * total;
        b = __builtin_popcountll(__builtin_amdgcn_ballot_w64(upto <= rest));
        const int whole = __builtin_amdgcn_readlane(mine, b), of = __builtin_amdgcn_readlane(parts, b);
        const int part = rest - (__builtin_amdgcn_readlane(upto, b) - of);
        const int each = parts_of(whole + 1, (float)of) - 1, more = whole - each * of;
        u0 = part * each + min(part, more), left = each + (part < more);
    } else {
        const int64_t my0 = (int64_t)blockIdx.x * run;
        if (my0 >= all) return;
        h = (int)(my0 / total), left = (int)min((int64_t)run, all - my0);
        const int rest = (int)(my0 - (int64_t)h * total), owner = __builtin_popcountll(__builtin_amdgcn_ballot_w64(upto <= rest));
        b = owner * per, u0 = rest - (__builtin_amdgcn_readlane(upto, owner) - __builtin_amdgcn_readlane(mine, owner));
        for (; !one; b++) {
            const int u = units_of(b);
            if (u0 < u) break;
            u0 -= u;
        }
    }
    h = __builtin_amdgcn_readfirstlane(h), run = __builtin_amdgcn_readfirstlane(run);
    left = __builtin_amdgcn_readfirstlane(left), u0 = __builtin_amdgcn_readfirstlane(u0);

    for (bool first_seg = true; left > 0; first_seg = false) {
        const int pos = one ? __builtin_amdgcn_readlane(lane_pos, b) : seq_pos(a.pos, b);
        const int len = one ? __builtin_amdgcn_readlane(lane_len, b) : seq_len(a.lens, b, a.n);
        const KeyTiles kt = key_tiles<5>(a, pos, 0, len);
        const int nu = (kt.count + kFewUnit - 1) / kFewUnit;
        if (u0 >= nu) {  // the next sequence (or KV head)
            u0 = 0;
            if (++b == a.n_seq) b = 0, h++;
            continue;
        }
        const int u1 = min(nu, u0 + left);
        const bool split = u0 > 0 || u1 < nu;
        // this wave's blocks: entries e0, e0 + 4, ... below `stop`
        const int e0 = u0 * kFewUnit + wave, stop = min(u1 * kFewUnit, kt.count);
        const int its = stop > e0 ? (stop - e0 + kFewUnit - 1) / kFewUnit : 0;
        const int32_t* table = a.c.table + (size_t)b * a.c.table_stride;
        // lane l holds the page of the wave's block it0 + l
        int pages = -1, it0 = 0;
        auto fetch_pages = [&](int at) {
            it0 = at;
            const int e = min(e0 + (at + lane) * kFewUnit, kt.count - 1);
            pages = table[kt.tile(max(e, 0)) >> (a.c.lg_page - 5)];
        };
        // the keys or values of the wave's block `it`, straight into the LDS (zeros past the last one and without a page)
        f16* sk = kv + wave * 2 * BLKE;
        f16* sv = sk + BLKE;
        auto load = [&](int it, uint16_t* pool, f16* dst) __attribute__((always_inline)) {
            const int e = e0 + it * kFewUnit, p = kt.tile(min(e, kt.count - 1)) * kBlk;
            const int page = __builtin_amdgcn_readlane(pages, (it - it0) & 63);
            const bool there = it < its && (uint32_t)page < (uint32_t)a.c.n_pages;
            const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
                pool + paged_block(a.c, there ? page : 0, p, h, a.NKV, D), (short)0, there ? BLKE * 2 : 0, 0x00020000);
#pragma unroll
            for (int i = 0; i < NDT; i++)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(dst + i * 512), 16, lane * 16,
                                                         i * 1024, 0, 0);
        };
        fetch_pages(0);

        // ---- the rows, 256 / ROWS threads a row, pieces of 8 dims: asked for before the blocks, and laid out as operands ----
        constexpr int TPR = 64 * kFewWaves / ROWS, PIECES = D / 8, PPT = (PIECES + TPR - 1) / TPR;
        const int qr = tid / TPR, tl = tid % TPR;
        float x[PPT][8];
        {
            const int t = heads.token(qr);
            const size_t off = ((size_t)b * a.n + min(t, len - 1)) * a.q_stride + (size_t)(h * G + qr - t * G) * a.q_head;
#pragma unroll
            for (int i = 0; i < PPT; i++) load_vec<DT, 8>(a.q, off + 8 * ((tl + i * TPR) % PIECES), x[i]);
        }
        if (!first_seg) __syncthreads();  // the last segment's readers of the LDS are done
        load(0, a.c.k, sk);
        if constexpr (!C::TIGHT) load(0, a.c.v, sv);
        {
            const bool ok = heads.token(qr) < len;
            float largest = 0.f;
#pragma unroll
            for (int i = 0; i < PPT; i++)
#pragma unroll
                for (int j = 0; j < 8; j++) x[i][j] = ok ? x[i][j] : 0.f, largest = fmaxf(largest, fabsf(x[i][j]));
            largest = max_lanes<TPR>(largest);
            const int sh = query_shift(largest);
            const float up = power_of_two(sh);
            if (tl == 0) sc[qr] = a.scale * power_of_two(-sh);
#pragma unroll
            for (int i = 0; i < PPT; i++) {
                const int pc = tl + i * TPR;
                if (pc >= PIECES) break;
                f16x8 hi, lo;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float y = x[i][j] * up;
                    hi[j] = (f16)y;
                    if constexpr (PARTS == 2) lo[j] = (f16)(y - (float)hi[j]);
                }
                f16* dst = sq + (((qr >> 4) * NKS + (pc >> 2)) * 64 + (pc & 3) * 16 + (qr & 15)) * 8;
                *reinterpret_cast<f16x8*>(dst) = hi;
                if constexpr (PARTS == 2) *reinterpret_cast<f16x8*>(dst + NT * NKS * 512) = lo;
            }
        }
        // a barrier for the LDS alone: the blocks in flight stay in flight
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");

        // ---- this wave's blocks ----
        f32x4 acc[NT][NDT];
        float m_run[NT], l_run[NT], fac[NT];
        Sight see[NT];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int t = heads.token(nt * 16 + col);
            see[nt] = t < len ? sight(a, pos + t) : Sight{0, 0};
            m_run[nt] = kNegInf, l_run[nt] = 0.f, fac[nt] = sc[nt * 16 + col];
            asm volatile("" : "+v"(fac[nt]));
#pragma unroll
            for (int dt = 0; dt < NDT; dt++) acc[nt][dt] = f32x4{};
        }
        if constexpr (C::TIGHT) {
            wait_lds();
            __builtin_amdgcn_s_barrier();
            load(0, a.c.v, sv);
        }
        const Sight all_see = sight_of_all(a, pos, pos + len - 1), some_see = sight_of_some(a, pos, pos + len - 1);
#pragma unroll 1
        for (int it = 0; it < its; it++) {
            const int e = e0 + it * kFewUnit, k0 = kt.tile(min(e, kt.count - 1)) * kBlk;
            const bool there = (uint32_t)__builtin_amdgcn_readlane(pages, (it - it0) & 63) < (uint32_t)a.c.n_pages;
            f32x4 s[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) s[nt][0] = f32x4{}, s[nt][1] = f32x4{};
            wait_loads<NDT>();  // the keys are there, the values may be on their way
#pragma unroll
            for (int kk = 0; kk < NKS; kk++) {
                const f16x8 ka = *reinterpret_cast<const f16x8*>(sk + (2 * kk * 64 + lane) * 8);
                const f16x8 kb = *reinterpret_cast<const f16x8*>(sk + ((2 * kk + 1) * 64 + lane) * 8);
#pragma unroll
                for (int part = 0; part < PARTS; part++)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        const f16x8 q = *reinterpret_cast<const f16x8*>(sq + (((part * NT + nt) * NKS + kk) * 64 + lane) * 8);
                        s[nt][0] = mfma16(ka, q, s[nt][0]);
                        s[nt][1] = mfma16(kb, q, s[nt][1]);
                    }
                if (kk % 2 == 1) __builtin_amdgcn_sched_barrier(0);  // few fragments at a time
            }
            wait_lds();
            if (it + 1 - it0 >= 64) fetch_pages(it + 1);
            load(it + 1, a.c.k, sk);
            const bool whole = there && sees_whole(all_see, k0, k0 + kBlk, a.sinks);
            if (!whole) {  // value i of key set s of lane (col, g) is key 8 g + 4 s + i
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        s[nt][i >> 2][i & 3] = there && see[nt].sees(k0 + 8 * g + i, a.sinks) ? s[nt][i >> 2][i & 3] : kNegInf;
            }
            f16x8 w[NT][kWeightParts];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float mx = fmaxf(fmaxf(fmaxf(s[nt][0][0], s[nt][0][1]), fmaxf(s[nt][0][2], s[nt][0][3])),
                                 fmaxf(fmaxf(s[nt][1][0], s[nt][1][1]), fmaxf(s[nt][1][2], s[nt][1][3])));
                mx = max_rows(mx) * fac[nt];
                const bool grow = m_run[nt] == kNegInf ? mx != kNegInf : mx > m_run[nt] + kTau;
                if (__builtin_amdgcn_ballot_w64(grow)) {
                    const float to = grow ? mx : m_run[nt];
                    const float corr = to == kNegInf ? 1.f : exp2_fast(m_run[nt] - to);
                    m_run[nt] = to, l_run[nt] *= corr;
#pragma unroll
                    for (int dt = 0; dt < NDT; dt++) acc[nt][dt] *= corr;
                }
                const float off = m_run[nt] == kNegInf ? 0.f : kShift - m_run[nt];
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float w0 = exp2_fast(__builtin_fmaf(s[nt][i >> 2][i & 3], fac[nt], off));
                    const float w1 = exp2_fast(__builtin_fmaf(s[nt][i >> 2][(i & 3) + 1], fac[nt], off));
                    f16x2 hi, lo;
                    weight_parts(w0, w1, hi, lo);
                    w[nt][0][i] = hi[0], w[nt][0][i + 1] = hi[1], w[nt][1][i] = lo[0], w[nt][1][i + 1] = lo[1];
                    l_run[nt] += w0 + w1;
                }
            }
            wait_loads<NDT>();  // the values are there, the next keys may be on their way
            auto vfrag = [&](int dt) { return *reinterpret_cast<const f16x8*>(sv + (dt * 64 + lane) * 8); };
            if (whole) {
#pragma unroll
                for (int dt = 0; dt < NDT; dt++) {
                    const f16x8 v = vfrag(dt);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int part = 0; part < kWeightParts; part++) acc[nt][dt] = mfma16(v, w[nt][part], acc[nt][dt]);
                    if (dt % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                }
            } else {
                // values that no token sees are zeroed; where one that only some see is not finite, a zero weight would
                // not hide it: then the products are taken token by token, the values hidden from it zeroed
                auto some = [&](int i) { return some_see.sees(k0 + 8 * g + i, a.sinks); };
                uint32_t odd = 0;
                if (len > 1)
                    for (int dt = 0; dt < NDT; dt++) odd |= not_finite(keep_keys(vfrag(dt), some));
                if (!__builtin_amdgcn_ballot_w64(odd != 0)) {
#pragma unroll
                    for (int dt = 0; dt < NDT; dt++) {
                        const f16x8 v = keep_keys(vfrag(dt), some);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int part = 0; part < kWeightParts; part++) acc[nt][dt] = mfma16(v, w[nt][part], acc[nt][dt]);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                } else {
#pragma unroll 1
                    for (int t = 0; t < len; t++) {
                        const Sight st = sight(a, pos + t);
#pragma unroll
                        for (int dt = 0; dt < NDT; dt++) {
                            const f16x8 v = keep_keys(vfrag(dt), [&](int i) { return st.sees(k0 + 8 * g + i, a.sinks); });
#pragma unroll
                            for (int nt = 0; nt < NT; nt++) {
                                f32x4 o = acc[nt][dt];
#pragma unroll
                                for (int part = 0; part < kWeightParts; part++) o = mfma16(v, w[nt][part], o);
                                const bool own = heads.token(nt * 16 + col) == t;
#pragma unroll
                                for (int i = 0; i < 4; i++) acc[nt][dt][i] = own ? o[i] : acc[nt][dt][i];
                                __builtin_amdgcn_sched_barrier(0);
                            }
                        }
                    }
                }
            }
            wait_lds();
            load(it + 1, a.c.v, sv);
        }

        // ---- the waves' outputs, through the blocks' room, added against their common maximum: a wave every fourth dim tile ----
        constexpr int PER = NDT / kFewWaves;
        Gate4<DT> gate[NT][PER];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int t = heads.token(nt * 16 + col);
#pragma unroll
            for (int k = 0; k < PER; k++) {
                gate[nt][k].none();
                if (!split && a.gate && t < len)
                    gate[nt][k].load(a, (size_t)b * a.n + t, h * G + nt * 16 + col - t * G, 16 * (wave + k * kFewWaves) + 4 * g);
            }
        }
        wait_loads<0>();  // (loads past the last block write zeros)
        __syncthreads();
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float l = l_run[nt];
            const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(l), __float_as_uint(l), false, false);
            l = __uint_as_float(x[0]) + __uint_as_float(x[1]);
            const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
            l_run[nt] = __uint_as_float(y[0]) + __uint_as_float(y[1]);
            if (g == 0) sm[wave * ROWS + nt * 16 + col] = m_run[nt], sl[wave * ROWS + nt * 16 + col] = l_run[nt];
#pragma unroll
            for (int dt = 0; dt < NDT; dt++) *reinterpret_cast<f32x4*>(red + (((wave * NT + nt) * NDT + dt) * 64 + lane) * 4) = acc[nt][dt];
        }
        __syncthreads();
        const int slot = 2 * blockIdx.x + (u0 == 0 ? 1 : 0);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int r = nt * 16 + col, t = heads.token(r);
            if (t >= len) continue;
            float f[kFewWaves], m = kNegInf, l = 0.f;
#pragma unroll
            for (int w = 0; w < kFewWaves; w++) f[w] = sm[w * ROWS + r], m = fmaxf(m, f[w]);
#pragma unroll
            for (int w = 0; w < kFewWaves; w++) f[w] = f[w] == kNegInf ? 0.f : exp2_fast(f[w] - m), l += sl[w * ROWS + r] * f[w];
            const float inv = inverse_sum(l);
            if (split && wave == 0 && g == 0) *reinterpret_cast<f32x2*>(plan.ml + ((size_t)slot * ROWS + r) * 2) = f32x2{m, l};
#pragma unroll
            for (int k = 0; k < PER; k++) {
                const int dt = wave + k * kFewWaves;
                f32x4 o{};
#pragma unroll
                for (int w = 0; w < kFewWaves; w++) {
                    const f32x4 x = *reinterpret_cast<const f32x4*>(red + (((w * NT + nt) * NDT + dt) * 64 + lane) * 4);
#pragma unroll
                    for (int i = 0; i < 4; i++) o[i] = __builtin_fmaf(x[i], f[w], o[i]);
                }
                if (split) *reinterpret_cast<f32x4*>(plan.o + ((size_t)slot * ROWS + r) * D + 16 * dt + 4 * g) = o;
                else store_out4<DT>(a, (size_t)b * a.n + t, h * G + r - t * G, D, 16 * dt + 4 * g, o, inv, gate[nt][k]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        left -= u1 - u0;
        u0 = u1;
    }
}

// Joins the parts of split sequences: a workgroup 64 dims of a (sequence, token, head), 16 lanes a part, 16 parts at a time.
// Its first part is the last segment of one workgroup of k_paged_few, the others the first segments of those after it.
// Every wave takes the parts' maxima and sums for itself, a lane each, so that their loads and the parts' are in flight
// together. Fixed order.
template <int D, int DT, int ROWS>
__global__ __launch_bounds__(256) void k_paged_join(PagedAttendArgs a, FewHeads heads, void* ws, int groups) {
    constexpr int SETS = 16, SLICES = D / 64;
    __shared__ f32x4 red[4][16];
    const FewPlan plan = few_plan(ws, groups, ROWS, D);
    const int head = blockIdx.x / SLICES, slice = blockIdx.x % SLICES, t = blockIdx.y, b = blockIdx.z;
    const size_t row = (size_t)b * a.n + t;
    const int total = plan.head[0], run = plan.head[1], at0 = plan.head[kFewHead + b], at1 = plan.head[kFewHead + b + 1];
    const int pos = seq_pos(a.pos, b), len = seq_len(a.lens, b, a.n);
    if (t >= len) return;
    const int h = head / heads.G, r = t * heads.G + head - h * heads.G;
    int64_t first = (int64_t)h * total + at0;
    int parts = at1 - at0;
    if (run) {
        const int nu = (key_tiles<5>(a, pos, 0, len).count + kFewUnit - 1) / kFewUnit;
        const int64_t last = (first + nu - 1) / run;
        first /= run, parts = (int)(last - first) + 1;
    }
    if (parts == 1) return;
    const int tid = threadIdx.x, lane = tid & 63, set = tid >> 4, d = 64 * slice + 4 * (tid & 15);
    auto slot = [&](int part) { return (size_t)(part == 0 ? 2 * first + 1 : 2 * (first + part)) * ROWS + r; };
    Gate4<DT> gate;
    gate.none();
    if (a.gate) gate.load(a, row, head, d);
    float m = kNegInf, l = 0.f;
    f32x4 o{};
    for (int p0 = 0; p0 < parts; p0 += 64) {
        const f32x2 ml = *reinterpret_cast<const f32x2*>(plan.ml + slot(min(p0 + lane, parts - 1)) * 2);
        f32x4 x[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int p = p0 + set + SETS * k;
            x[k] = p < parts ? *reinterpret_cast<const f32x4*>(plan.o + slot(p) * D + d) : f32x4{};
        }
        const float mine = p0 + lane < parts ? ml[0] : kNegInf, to = fmaxf(m, max64(mine));
        const float w = mine == kNegInf ? 0.f : exp2_fast(mine - to), corr = m == kNegInf ? 0.f : exp2_fast(m - to);
        m = to, l = l * corr + sum64(ml[1] * w), o *= corr;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float wk = __shfl(w, set + SETS * k, 64);
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = __builtin_fmaf(x[k][i], wk, o[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {  // the wave's four sets
        const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(o[i]), __float_as_uint(o[i]), false, false);
        const float y = __uint_as_float(x[0]) + __uint_as_float(x[1]);
        const auto z = __builtin_amdgcn_permlane32_swap(__float_as_uint(y), __float_as_uint(y), false, false);
        o[i] = __uint_as_float(z[0]) + __uint_as_float(z[1]);
    }
    if (lane < 16) red[tid >> 6][lane] = o;
    __syncthreads();
    if (tid < 16) {
        o = red[0][tid] + red[1][tid] + red[2][tid] + red[3][tid];
        store_out4<DT>(a, row, head, D, d, o, inverse_sum(l), gate);
    }
}

template <int D, int DT, int NT>
hipError_t go(const PagedAttendArgs& a, int n_cu, void* ws, hipStream_t s) {
    using C = FewCfg<D, DT, NT>;
    constexpr int ROWS = C::ROWS;
    const int groups = n_cu * few_occ(D), G = a.NH / a.NKV;
    const FewHeads heads{G, 65536 / G + 1};
    constexpr int shm = C::LDS;
    auto kern = k_paged_few<D, DT, NT>;
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, shm);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kern, dim3(groups), dim3(64 * kFewWaves), shm, s, a, heads, ws);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    hipLaunchKernelGGL((k_paged_join<D, DT, ROWS>), dim3(a.NH * (D / 64), a.n, a.n_seq), dim3(256), 0, s, a, heads, ws, groups);
    return hipGetLastError();
}

template <int D>
hipError_t go_d(const PagedAttendArgs& a, bool bf16, int n_cu, void* ws, hipStream_t s) {
    // rows of one matrix tile or of two (one token at 32767, 8 rows: one 20.0 us, two 22.3)
    const bool two = a.n * (a.NH / a.NKV) > 16;
    if (bf16) return two ? go<D, 1, 2>(a, n_cu, ws, s) : go<D, 1, 1>(a, n_cu, ws, s);
    return two ? go<D, 0, 2>(a, n_cu, ws, s) : go<D, 0, 1>(a, n_cu, ws, s);
}

}  // namespace

size_t paged_few_workspace(int D, int n_cu) {
    const size_t rows = (size_t)2 * n_cu * few_occ(D) * 32;
    return up256(rows * (D + 2) * sizeof(float) + (kFewHead + 65536 + 1) * sizeof(int));
}

hipError_t launch_paged_few(const PagedAttendArgs& a, int D, bool bf16, int n_cu, void* ws, hipStream_t s) {
    if (D == 256) return go_d<256>(a, bf16, n_cu, ws, s);
    if (D == 128) return go_d<128>(a, bf16, n_cu, ws, s);
    return go_d<64>(a, bf16, n_cu, ws, s);
}

}  // namespace qw

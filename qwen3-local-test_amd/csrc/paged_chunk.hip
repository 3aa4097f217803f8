// Attention of chunks of new tokens (more than 32 query rows a KV head) over a paged cache, on the matrix cores.
#include "paged.hpp"

namespace qw {

namespace {

constexpr int kChWaves = 8, kChRing = 4;

template <int D, int DT, int NT>
struct ChCfg {
    static constexpr int PARTS = DT == 0 ? 2 : 1, NKS = D / 32, NDT = D / 16, ROWS = kChWaves * 16 * NT;
    static constexpr int BLKE = kBlk * D;              // elements of a block
    static constexpr int LDS = 2 * kChRing * BLKE * 2;  // rings of blocks of keys and of values
    static constexpr int COPIES = D / 64;              // kilobytes a wave copies a step (a block of keys and one of values)
    static constexpr int PART = 16 * NT * D + 64 * NT * 2;   // floats of a wave's partial
};
// Tiles of 16 rows a wave: what fits the 256 registers of a wave beside the queries' operands
constexpr int ch_nt(int D, bool bf16) { return D == 256 && !bf16 ? 1 : 2; }

// Workspace: the partials of two segments a workgroup (its first and its last), then the plan.
struct ChPlan {
    float* part;    // [2 * groups][waves][PART]
    int4* start;    // [groups]: KV head (-1: nothing to do), sequence, query tile, first key tile
    int* cnt;       // [groups][waves] arrivals at the item that is the workgroup's last
    int64_t* head;  // key tiles a KV head, key tiles a workgroup
    int64_t* first; // joined calls: first key tile of each (sequence, query tile)
};
constexpr int kJoinItems = 1024;  // most (sequence, query tile) pairs of a joined call
__host__ __device__ inline ChPlan ch_plan(void* ws, int groups, int part_floats) {
    ChPlan p;
    p.part = static_cast<float*>(ws);
    p.start = reinterpret_cast<int4*>(p.part + (size_t)2 * groups * kChWaves * part_floats);
    p.cnt = reinterpret_cast<int*>(p.start + groups);
    p.head = reinterpret_cast<int64_t*>(p.cnt + groups * kChWaves);
    p.first = p.head + 2;
    return p;
}

// Items are (KV head, sequence, query tile) in this order, each of as many units as it has key tiles; every workgroup of
// the chunk kernel takes an equal run of units. One workgroup: a thread sums a run of (sequence, query tile) pairs, a
// scan places the runs, and the threads write the starts that fall into theirs.
__global__ __launch_bounds__(1024) void k_paged_plan(PagedAttendArgs a, void* ws, int groups, int part_floats, int tok, bool joined) {
    __shared__ int64_t sums[16];
    const ChPlan plan = ch_plan(ws, groups, part_floats);
    const int nqt = (a.n + tok - 1) / tok, pairs = a.n_seq * nqt;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (pairs + 1023) / 1024;
    auto tiles = [&](int pair) {
        const int b = pair / nqt, t0 = (pair - b * nqt) * tok;
        return key_tiles<6>(a, seq_pos(a.pos, b), t0, min(t0 + tok, seq_len(a.lens, b, a.n))).count;
    };
    int64_t mine = 0;
    for (int i = 0; i < per; i++)
        if (tid * per + i < pairs) mine += tiles(tid * per + i);
    int64_t incl = mine;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const int64_t o = __shfl_up((long long)incl, m, 64);
        if (lane >= m) incl += o;
    }
    if (lane == 63) sums[wave] = incl;
    for (int i = tid; i < groups * kChWaves; i += 1024) plan.cnt[i] = 0;
    __syncthreads();
    int64_t x = incl - mine, total = 0;
    for (int w = 0; w < 16; w++) x += w < wave ? sums[w] : 0, total += sums[w];
    const int64_t all = total * a.NKV, run = max((int64_t)1, (all + groups - 1) / groups);
    for (int w = tid; w < groups; w += 1024)
        if (w * run >= all) plan.start[w].x = -1;
    if (tid == 0) plan.head[0] = total, plan.head[1] = run;
    for (int i = 0; i < per; i++) {
        const int pair = tid * per + i;
        if (pair >= pairs) break;
        const int c = tiles(pair);
        if (joined) plan.first[pair] = x;
        for (int h = 0; h < a.NKV && c; h++) {
            const int64_t g0 = h * total + x;
            for (int64_t w = (g0 + run - 1) / run; w * run < g0 + c; w++)
                plan.start[w] = int4{h, pair / nqt, pair % nqt, (int)(w * run - g0)};
        }
        x += c;
    }
}

// The lane, worked out where it stands: kept in a register through the loop of 32-row waves it would be spilled, and a
// reload waits for every copy in flight.
__device__ __forceinline__ int lane_here() {
    int l;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(l));
    return l;
}
// A barrier that waits for nothing else; nothing moves across it
__device__ __forceinline__ void phase() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}
// Waits until at most N (< 16) vector loads of the wave are in flight
template <int N>
__device__ __forceinline__ void landed() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0F70 | N);
    asm volatile("" ::: "memory");
}

template <int D, int DT, int NT>
__global__ __launch_bounds__(64 * kChWaves, 1) void k_paged_chunk(PagedAttendArgs a, void* ws, bool joined) {
    using C = ChCfg<D, DT, NT>;
    constexpr int PARTS = C::PARTS, NKS = C::NKS, NDT = C::NDT, BLKE = C::BLKE;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    f16* sk = reinterpret_cast<f16*>(smem);  // blocks of keys
    f16* sv = sk + kChRing * BLKE;           // and of values
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int G = a.NH / a.NKV, tok = C::ROWS / G, groups = gridDim.x;
    const ChPlan plan = ch_plan(ws, groups, C::PART);
    // neighbouring runs on one XCD: they read the same keys
    const int wg = (blockIdx.x & 7) * (groups >> 3) + (blockIdx.x >> 3);
    const int4 st = plan.start[wg];
    int h = __builtin_amdgcn_readfirstlane(st.x), b = __builtin_amdgcn_readfirstlane(st.y);
    int qt = __builtin_amdgcn_readfirstlane(st.z), off = __builtin_amdgcn_readfirstlane(st.w);
    if (h < 0) return;
    const int64_t total = plan.head[0], run = plan.head[1], all = total * a.NKV;
    int64_t at = wg * run;  // unit of the segment at hand
    const int64_t stop = min(at + run, all);

    while (at < stop) {
        const int pos = seq_pos(a.pos, b), len = seq_len(a.lens, b, a.n);
        const int t0 = qt * tok, t1 = min(t0 + tok, len);
        const KeyTiles kt = key_tiles<6>(a, pos, t0, t1);
        if (off >= kt.count) {  // the next item with tiles
            off = 0;
            if (t0 + tok < len) {
                qt++;
            } else {
                qt = 0;
                if (++b == a.n_seq) b = 0, h++;
            }
            continue;
        }
        const int lo = off, hi = (int)min((int64_t)kt.count, off + (stop - at));

        const int n = 2 * (hi - lo);  // blocks of 32 keys, block i of the segment in ring place i % 4
        auto key_of = [&](int i) { return kt.tile(lo + (i >> 1)) * 64 + (i & 1) * kBlk; };

        // ---- the wave's rows as they lie in memory: row r of the tile is token t0 + r / G, head h G + r % G ----
        typedef typename std::conditional<DT == 0, f32x4, u32x4>::type raw_t;
        constexpr int RAW = DT == 0 ? 2 : 1;
        raw_t raw[NT][NKS][RAW];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int r = (wave * NT + nt) * 16 + col, t = min(t0 + r / G, t1 - 1);
            const size_t base = ((size_t)b * a.n + t) * a.q_stride + (size_t)(h * G + r % G) * a.q_head + 8 * g;
#pragma unroll
            for (int kk = 0; kk < NKS; kk++)
#pragma unroll
                for (int k = 0; k < RAW; k++) {
                    if constexpr (DT == 0) raw[nt][kk][k] = *reinterpret_cast<const raw_t*>(static_cast<const float*>(a.q) + base + 32 * kk + 4 * k);
                    else raw[nt][kk][k] = *reinterpret_cast<const raw_t*>(static_cast<const uint16_t*>(a.q) + base + 32 * kk);
                }
        }

        // positions of the wave's tokens, the keys that all of them see, that some of them see, and that some of the item's do
        const int w0 = pos + t0 + wave * 16 * NT / G, w1 = min(pos + t0 + (wave * 16 * NT + 16 * NT - 1) / G, pos + t1 - 1);
        const Sight all_see = sight_of_all(a, w0, w1), some_see = sight_of_some(a, w0, w1);
        const Sight item_see = sight_of_some(a, pos + t0, pos + t1 - 1);

        // ---- staging. What a step needs to know of its blocks is worked out for 64 of them at a time, a lane each: scalar
        // arithmetic in every step (page, offset, masks: some 150 instructions) took as long as its matrix instructions ----
        const int32_t* table = a.c.table + (size_t)b * a.c.table_stride;
        int base = 0;
        int64_t offset = -1;   // lane l: byte offset of block base + l in a pool, -1 without a page or past the last block
        int first_key = 0;     // its first position
        uint64_t paged, whole, stale;  // bit l: it has a page; all rows of the wave see all of it; it has keys that no row of the item sees
        auto survey = [&](int i) __attribute__((always_inline)) {
            base = i;
            const int l = lane_here();
            const bool in = i + l < n;
            first_key = key_of(min(i + l, n - 1));
            const int page = in && first_key < a.limit ? table[first_key >> a.c.lg_page] : -1;
            const bool there = (uint32_t)page < (uint32_t)a.c.n_pages;
            offset = there ? 2 * paged_block(a.c, page, first_key, h, a.NKV, D) : -1;
            paged = __builtin_amdgcn_ballot_w64(there);
            whole = __builtin_amdgcn_ballot_w64(there && sees_whole(all_see, first_key, first_key + kBlk, a.sinks));
            stale = __builtin_amdgcn_ballot_w64(in && !sees_whole(item_see, first_key, first_key + kBlk, a.sinks));
        };
        auto key_at = [&](int i) { return __builtin_amdgcn_readlane(first_key, i - base); };
        // this wave's share of block i of `pool` into ring place i % 4 (zeros without a page): pieces from `first` on
        auto copy = [&](int i, uint16_t* pool, f16* ring, int first, auto count) __attribute__((always_inline)) {
            const uint32_t lo32 = (uint32_t)__builtin_amdgcn_readlane((int)offset, i - base);
            const int hi32 = __builtin_amdgcn_readlane((int)(offset >> 32), i - base);
            const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
                reinterpret_cast<char*>(pool) + (((int64_t)(hi32 < 0 ? 0 : hi32) << 32) | lo32), (short)0, hi32 < 0 ? 0 : BLKE * 2, 0x00020000);
            f16* dst = ring + (i & (kChRing - 1)) * BLKE;
            const int l16 = lane_here() * 16;
#pragma unroll
            for (int j = 0; j < decltype(count)::value; j++)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(dst + (first + j) * 512), 16,
                                                         (first + j) * 1024 + l16, 0, 0, 0);
        };
        auto stage = [&](bool keys, int i) __attribute__((always_inline)) {
            if constexpr (D >= 128) {
                constexpr int P = D / 128;
                copy(i, keys ? a.c.k : a.c.v, keys ? sk : sv, wave * P, std::integral_constant<int, P>{});
            } else {  // the first four waves copy keys and the others values
                if (keys == (wave < 4)) copy(i, keys ? a.c.k : a.c.v, keys ? sk : sv, wave & 3, std::integral_constant<int, 1>{});
            }
        };
        survey(0);
        __syncthreads();  // the last segment's readers of the rings are done
        stage(true, 0), stage(true, 1), stage(false, 0);

        // ---- the rows' operands ----
        f16x8 q[NT][PARTS][NKS];
        float fac[NT], m_run[NT], l_run[NT];
        f32x4 acc[NT][NDT];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            auto at_raw = [&](int kk, int j) {
                if constexpr (DT == 0) return raw[nt][kk][j >> 2][j & 3];
                else return __uint_as_float((j & 1) ? raw[nt][kk][0][j >> 1] & 0xffff0000u : raw[nt][kk][0][j >> 1] << 16);
            };
            float largest = 0.f;
#pragma unroll
            for (int kk = 0; kk < NKS; kk++)
#pragma unroll
                for (int j = 0; j < 8; j++) largest = fmaxf(largest, fabsf(at_raw(kk, j)));
            const int sh = query_shift(max_rows(largest));
            fac[nt] = __builtin_ldexpf(a.scale, -sh);
#pragma unroll
            for (int kk = 0; kk < NKS; kk++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float y = __builtin_ldexpf(at_raw(kk, j), sh);
                    q[nt][0][kk][j] = (f16)y;
                    if constexpr (PARTS == 2) q[nt][1][kk][j] = (f16)(y - (float)q[nt][0][kk][j]);
                }
            m_run[nt] = kNegInf, l_run[nt] = 0.f;
#pragma unroll
            for (int dt = 0; dt < NDT; dt++) acc[nt][dt] = f32x4{};
        }
        auto unseen = [&](int k0) { return k0 >= some_see.end || (k0 + kBlk <= some_see.from && k0 >= a.sinks); };
        auto row_sight = [&](int nt, int l) {
            const int r = (wave * NT + nt) * 16 + (l & 15), t = t0 + r / G;
            return r < tok * G && t < t1 ? sight(a, pos + t) : Sight{0, 0};
        };

        f32x4 s[NT][2];        // scores of a block: value i of key set s of lane (col, g) is key 8 g + 4 s + i
        f16x8 w[NT][PARTS];    // its weights: keys 8 g .. 8 g + 7
        // Matrix instructions of a phase: the scores of one block and (VALUES) the weighted values of the block before, a fragment of
        // each in turn, read AHEAD of its use
        constexpr int AHEAD = NT == 2 && D == 256 ? 3 : 5;
        auto products = [&](auto values, auto&& kfrag, auto&& vfrag) __attribute__((always_inline)) {
            constexpr bool VALUES = decltype(values)::value;
            constexpr int STEP = VALUES ? 2 : 1, SLOTS = STEP * NDT;
            f16x8 fr[AHEAD + 1];
            auto read = [&](auto ic) __attribute__((always_inline)) {
                constexpr int i = decltype(ic)::value;
                if constexpr (VALUES && i % STEP == 0) fr[i % (AHEAD + 1)] = vfrag(i / STEP);
                else fr[i % (AHEAD + 1)] = kfrag(i / STEP);
            };
#pragma unroll
            for (int nt = 0; nt < NT; nt++) s[nt][0] = f32x4{}, s[nt][1] = f32x4{};
            static_for<0, AHEAD>(read);
            static_for<0, SLOTS>([&](auto ic) __attribute__((always_inline)) {
                constexpr int i = decltype(ic)::value, f = i / STEP;
                if constexpr (i + AHEAD < SLOTS) read(std::integral_constant<int, i + AHEAD>{});
#pragma unroll
                for (int part = 0; part < PARTS; part++)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        if constexpr (VALUES && i % STEP == 0) acc[nt][f] = mfma16(fr[i % (AHEAD + 1)], w[nt][part], acc[nt][f]);
                        else s[nt][f & 1] = mfma16(fr[i % (AHEAD + 1)], q[nt][part][f >> 1], s[nt][f & 1]);
                    }
                __builtin_amdgcn_sched_barrier(0);  // keep the reads ahead
            });
        };
        // Weights of a block from its scores; the running maximum moves only where a row's passes it by more than kTau
        auto softmax = [&](int k0, bool there, bool all) __attribute__((always_inline)) {
            if (!all) {
                const int l = lane_here(), key = k0 + 8 * (l >> 4);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    const Sight see = row_sight(nt, l);
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        s[nt][i >> 2][i & 3] = there && see.sees(key + i, a.sinks) ? s[nt][i >> 2][i & 3] : kNegInf;
                }
            }
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
                const float o = m_run[nt] == kNegInf ? 0.f : kShift - m_run[nt];
#pragma unroll
                for (int i = 0; i < 8; i += 2) {
                    const float x0 = exp2_fast(__builtin_fmaf(s[nt][i >> 2][i & 3], fac[nt], o));
                    const float x1 = exp2_fast(__builtin_fmaf(s[nt][i >> 2][(i & 3) + 1], fac[nt], o));
                    f16x2 hi16, lo16;
                    weight_parts<PARTS>(x0, x1, hi16, lo16);
                    w[nt][0][i] = hi16[0], w[nt][0][i + 1] = hi16[1];
                    if constexpr (PARTS == 2) w[nt][1][i] = lo16[0], w[nt][1][i + 1] = lo16[1], l_run[nt] += x0 + x1;
                    else l_run[nt] = __builtin_amdgcn_fdot2(hi16, f16x2{(f16)1.f, (f16)1.f}, l_run[nt], false);
                }
            }
        };

        // ---- two groups of four waves, one of each on every SIMD, take turns: in a phase one runs the matrix instructions
        // of a block (and the weighted values of the block before) while the other takes its softmax. Copies run two blocks
        // ahead of the keys' use; both groups issue them in the even phases (of the first group's matrix instructions)
        // and wait for the last ones at their end. ----
        bool odd_values = false;
        const bool second = wave >= 4;
        auto kfrag_of = [&](int i) {
            const f16* p = sk + (i & (kChRing - 1)) * BLKE + lane_here() * 8;
            return [=](int f) { return *reinterpret_cast<const f16x8*>(p + f * 512); };
        };
        auto vfrag_of = [&](int i) {
            const f16* p = sv + (i & (kChRing - 1)) * BLKE + lane_here() * 8;
            return [=](int f) { return *reinterpret_cast<const f16x8*>(p + f * 512); };
        };
        // Values that no row of the item sees are zeroed in the ring (stale memory may hold anything) by the wave that copied
        // them, once they have landed.
        auto clean = [&](int i) __attribute__((always_inline)) {
            const int l = lane_here(), k0 = key_at(i) + 8 * (l >> 4);
            u32x4 keep;
#pragma unroll
            for (int k = 0; k < 4; k++)
                keep[k] = (item_see.sees(k0 + 2 * k, a.sinks) ? 0x0000ffffu : 0u) | (item_see.sees(k0 + 2 * k + 1, a.sinks) ? 0xffff0000u : 0u);
            if (D >= 128 || wave >= 4) {
#pragma unroll
                for (int j = 0; j < (D >= 128 ? D / 128 : 1); j++) {
                    const int piece = D >= 128 ? wave * (D / 128) + j : wave & 3;
                    u32x4* at = reinterpret_cast<u32x4*>(sv + (i & (kChRing - 1)) * BLKE + piece * 512 + l * 8);
                    *at = *at & keep;
                }
            }
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
        };
        // Step i: the copies of keys of block i + 2 and values of block i + 1; those of the step before have landed at its end
        auto step = [&](int i) __attribute__((always_inline)) {
            if (i + 2 - base >= 64) survey(i);
            stage(true, i + 2), stage(false, i + 1);
            landed<C::COPIES>();
            if (stale >> (i - base) & 1) clean(i);
        };
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int part = 0; part < PARTS; part++) w[nt][part] = f16x8{};
        auto matrix_phase = [&](int i) __attribute__((always_inline)) {  // scores of block i, values of block i - 1
            products(std::true_type{}, kfrag_of(i), vfrag_of(i - 1));
        };
        auto softmax_phase = [&](int i) __attribute__((always_inline)) {
            const bool all = whole >> (i - base) & 1;
            softmax(key_at(i), paged >> (i - base) & 1, all);
            if (!all) {
                const auto read = vfrag_of(i);
                uint32_t odd = 0;
#pragma unroll 4
                for (int dt = 0; dt < NDT; dt++) odd |= not_finite(read(dt));
                if (__builtin_amdgcn_ballot_w64(odd != 0)) odd_values = true;
            }
        };
        // (the values of the block before the first)
        for (int k = tid; k < BLKE / 8; k += 64 * kChWaves) *reinterpret_cast<u32x4*>(sv + (kChRing - 1) * BLKE + k * 8) = u32x4{};
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0xC07F);
        landed<C::COPIES>();
        phase();
        if (second) {
            step(0);
            phase();
        }
#pragma unroll 1
        for (int i = 0; i < n; i++) {
            matrix_phase(i);
            if (!second) step(i);
            phase();
            softmax_phase(i);
            if (second) step(i + 1);
            phase();
        }
        matrix_phase(n);  // (its scores are of no block)
        if (!second) phase();
        landed<0>();  // (copies past the last block write zeros)

        if (odd_values) {
            // a value that only some of the wave's rows see is not finite, and a weight of zero does not hide it: the segment again,
            // from memory, its weighted values token by token with those hidden from it zeroed
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                m_run[nt] = kNegInf, l_run[nt] = 0.f;
#pragma unroll
                for (int dt = 0; dt < NDT; dt++) acc[nt][dt] = f32x4{};
            }
#pragma unroll 1
            for (int i = 0; i < n; i++) {
                const int k0 = key_of(i);
                const int page = k0 < a.limit ? __builtin_amdgcn_readfirstlane(table[k0 >> a.c.lg_page]) : -1;
                if ((uint32_t)page >= (uint32_t)a.c.n_pages || unseen(k0)) continue;
                const int64_t from = paged_block(a.c, page, k0, h, a.NKV, D);
                const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(a.c.k + from, (short)0, BLKE * 2, 0x00020000);
                const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(a.c.v + from, (short)0, BLKE * 2, 0x00020000);
                auto get = [&](const __amdgpu_buffer_rsrc_t& r, int f) __attribute__((always_inline)) {
                    return __builtin_bit_cast(f16x8, __builtin_amdgcn_raw_buffer_load_b128(r, f * 1024 + lane * 16, 0, 0));
                };
                products(std::false_type{}, [&](int f) { return get(rk, f); }, [&](int f) { return get(rv, f); });
                softmax(k0, true, false);
#pragma unroll 1
                for (int p = w0; p <= w1; p++) {
                    const Sight sp = sight(a, p);
#pragma unroll
                    for (int dt = 0; dt < NDT; dt++) {
                        const f16x8 v = keep_keys(get(rv, dt), [&](int j) { return sp.sees(k0 + 8 * g + j, a.sinks); });
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            f32x4 o = acc[nt][dt];
#pragma unroll
                            for (int part = 0; part < PARTS; part++) o = mfma16(v, w[nt][part], o);
                            const bool own = pos + t0 + ((wave * NT + nt) * 16 + col) / G == p;
#pragma unroll
                            for (int j = 0; j < 4; j++) acc[nt][dt][j] = own ? o[j] : acc[nt][dt][j];
                            __builtin_amdgcn_sched_barrier(0);
                        }
                    }
                }
            }
        }

        // ---- sums across the row's lanes; whole items to the output, parts to the workspace ----
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(l_run[nt]), __float_as_uint(l_run[nt]), false, false);
            const float l = __uint_as_float(x[0]) + __uint_as_float(x[1]);
            const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
            l_run[nt] = __uint_as_float(y[0]) + __uint_as_float(y[1]);
        }
        const int64_t item = at - off;
        const int first = (int)(item / run), parts = (int)((item + kt.count - 1) / run) - first + 1, own = wg - first;
        bool write = parts == 1;
        if (parts > 1) {
            auto region = [&](int part) {
                const size_t slot = part == 0 ? 2 * first + 1 : 2 * (first + part);
                return __builtin_amdgcn_make_buffer_rsrc(plan.part + (slot * kChWaves + wave) * C::PART, (short)0, C::PART * 4, 0x00020000);
            };
            const __amdgpu_buffer_rsrc_t rp = region(own);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                for (int dt = 0; dt < NDT; dt++)
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, acc[nt][dt]), rp, ((nt * NDT + dt) * 64 + lane) * 16, 0, kScDevice);
                __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, f32x2{m_run[nt], l_run[nt]}), rp,
                                                      NT * NDT * 1024 + (nt * 64 + lane) * 8, 0, kScDevice);
            }
            if (!joined) {
                // the wave that arrives last joins the parts, from the first to the last whichever it is
                __builtin_amdgcn_s_waitcnt(0x0F70);  // the partial is out before it is counted
                int old = 0;
                if (lane == 0) old = __hip_atomic_fetch_add(plan.cnt + first * kChWaves + wave, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                write = __builtin_amdgcn_readfirstlane(old) == parts - 1;
                asm volatile("" ::: "memory");
                if (write) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        float m = kNegInf, l = 0.f;
#pragma unroll
                        for (int dt = 0; dt < NDT; dt++) acc[nt][dt] = f32x4{};
#pragma unroll 1
                        for (int part = 0; part < parts; part++) {
                            const __amdgpu_buffer_rsrc_t rq = region(part);
                            const f32x2 ml = __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(rq, NT * NDT * 1024 + (nt * 64 + lane) * 8, 0, kScDevice));
                            const float to = fmaxf(m, ml[0]);
                            const float cf = m == kNegInf ? 0.f : exp2_fast(m - to), cs = ml[0] == kNegInf ? 0.f : exp2_fast(ml[0] - to);
                            m = to, l = __builtin_fmaf(ml[1], cs, l * cf);
                            constexpr int NB = 4;
                            static_for<0, NDT / NB>([&](auto ic) __attribute__((always_inline)) {
                                constexpr int d0 = NB * decltype(ic)::value;
                                f32x4 o[NB];
#pragma unroll
                                for (int j = 0; j < NB; j++)
                                    o[j] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rq, ((nt * NDT + d0 + j) * 64 + lane) * 16, 0, kScDevice));
#pragma unroll
                                for (int j = 0; j < NB; j++)
#pragma unroll
                                    for (int i = 0; i < 4; i++) acc[nt][d0 + j][i] = __builtin_fmaf(o[j][i], cs, acc[nt][d0 + j][i] * cf);
                                __builtin_amdgcn_sched_barrier(0);
                            });
                        }
                        l_run[nt] = l;
                    }
                }
            }
        }
        if (write) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const int r = (wave * NT + nt) * 16 + col, t = t0 + r / G;
                if (r >= tok * G || t >= t1) continue;
                const float inv = inverse_sum(l_run[nt]);
#pragma unroll
                for (int dt = 0; dt < NDT; dt++) {
                    store_out4<DT>(a, (size_t)b * a.n + t, h * G + r % G, D, 16 * dt + 4 * g, acc[nt][dt], inv);
                    if (dt % 4 == 3) __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        at += hi - lo;
        off = hi;
    }
}

// Joins the parts of split items where there are few items: a workgroup 16 rows of an item and a quarter of its dims, four
// sets of threads a part each at a time, in a fixed order.
template <int D, int DT, int NT>
__global__ __launch_bounds__(256) void k_paged_join_chunk(PagedAttendArgs a, void* ws, int groups) {
    using C = ChCfg<D, DT, NT>;
    constexpr int NQ = C::NDT / 4;  // dim tiles of a quarter
    __shared__ f32x4 red[3][NQ][64];
    const ChPlan plan = ch_plan(ws, groups, C::PART);
    const int G = a.NH / a.NKV, tok = C::ROWS / G, nqt = (a.n + tok - 1) / tok;
    int x = blockIdx.x;
    const int quarter = x % 4, sub = x / 4 % (kChWaves * NT);
    x /= 4 * kChWaves * NT;
    const int h = x % a.NKV, pair = x / a.NKV, b = pair / nqt, t0 = (pair - b * nqt) * tok;
    const int t1 = min(t0 + tok, seq_len(a.lens, b, a.n));
    const int count = key_tiles<6>(a, seq_pos(a.pos, b), t0, t1).count;
    if (count == 0) return;
    const int64_t run = plan.head[1], item = h * plan.head[0] + plan.first[pair];
    const int first = (int)(item / run), parts = (int)((item + count - 1) / run) - first + 1;
    if (parts == 1) return;
    const int lane = threadIdx.x & 63, set = threadIdx.x >> 6, col = lane & 15, g = lane >> 4, wave = sub / NT, nt = sub % NT;
    const int r = sub * 16 + col, t = t0 + r / G;
    auto region = [&](int part) {
        const size_t slot = part == 0 ? 2 * first + 1 : 2 * (first + part);
        return plan.part + (slot * kChWaves + wave) * C::PART;
    };
    auto sums = [&](int part) { return *reinterpret_cast<const f32x2*>(region(part) + NT * C::NDT * 256 + (nt * 64 + lane) * 2); };
    float m = kNegInf, l = 0.f;
#pragma unroll 8
    for (int p = 0; p < parts; p++) m = fmaxf(m, sums(p)[0]);
    f32x4 o[NQ];
#pragma unroll
    for (int j = 0; j < NQ; j++) o[j] = f32x4{};
#pragma unroll 4
    for (int p = 0; p < parts; p++) {
        const f32x2 ml = sums(p);
        const float w = ml[0] == kNegInf ? 0.f : exp2_fast(ml[0] - m);
        l = __builtin_fmaf(ml[1], w, l);
        if (p % 4 == set) {
#pragma unroll
            for (int j = 0; j < NQ; j++) {
                const f32x4 v = *reinterpret_cast<const f32x4*>(region(p) + ((nt * C::NDT + quarter * NQ + j) * 64 + lane) * 4);
#pragma unroll
                for (int i = 0; i < 4; i++) o[j][i] = __builtin_fmaf(v[i], w, o[j][i]);
            }
        }
    }
    if (set > 0) {
#pragma unroll
        for (int j = 0; j < NQ; j++) red[set - 1][j][lane] = o[j];
    }
    __syncthreads();
    if (set > 0 || r >= tok * G || t >= t1) return;
    const float inv = inverse_sum(l);
#pragma unroll
    for (int j = 0; j < NQ; j++) {
        o[j] += (red[0][j][lane] + red[1][j][lane]) + red[2][j][lane];
        store_out4<DT>(a, (size_t)b * a.n + t, h * G + r % G, D, 16 * (quarter * NQ + j) + 4 * g, o[j], inv);
    }
}

template <int D, int DT>
hipError_t go(const PagedAttendArgs& a, int n_cu, void* ws, hipStream_t s) {
    constexpr int NT = ch_nt(D, DT == 1);
    using C = ChCfg<D, DT, NT>;
    const int groups = n_cu & ~7, tok = C::ROWS / (a.NH / a.NKV);
    const int64_t pairs = (int64_t)a.n_seq * ((a.n + tok - 1) / tok), items = pairs * a.NKV;
    const bool joined = items * 8 <= groups && pairs <= kJoinItems;
    hipLaunchKernelGGL(k_paged_plan, dim3(1), dim3(1024), 0, s, a, ws, groups, C::PART, tok, joined);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    auto kern = k_paged_chunk<D, DT, NT>;
    if ((e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS)) != hipSuccess) return e;
    hipLaunchKernelGGL(kern, dim3(groups), dim3(64 * kChWaves), C::LDS, s, a, ws, joined);
    if ((e = hipGetLastError()) != hipSuccess || !joined) return e;
    hipLaunchKernelGGL((k_paged_join_chunk<D, DT, NT>), dim3((unsigned)(items * kChWaves * NT * 4)), dim3(256), 0, s, a, ws, groups);
    return hipGetLastError();
}

}  // namespace

size_t paged_chunk_workspace(int D, int n_cu) {
    const size_t part = (size_t)kChWaves * (32 * D + 256) * sizeof(float);
    return up256(2 * n_cu * part + n_cu * (sizeof(int4) + kChWaves * sizeof(int)) + (2 + kJoinItems) * sizeof(int64_t));
}

hipError_t launch_paged_chunk(const PagedAttendArgs& a, int D, bool bf16, int n_cu, void* ws, hipStream_t s) {
    if (n_cu < 8) return hipErrorInvalidValue;
    if (D == 256) return bf16 ? go<256, 1>(a, n_cu, ws, s) : go<256, 0>(a, n_cu, ws, s);
    if (D == 128) return bf16 ? go<128, 1>(a, n_cu, ws, s) : go<128, 0>(a, n_cu, ws, s);
    return bf16 ? go<64, 1>(a, n_cu, ws, s) : go<64, 0>(a, n_cu, ws, s);
}

}  // namespace qw

// Attention of chunks of new tokens (more than 32 query rows a KV head) over a paged cache, on the matrix cores.
//
// The one-pass softmax of paged_few.hip for items of 128 or 256 query rows (KV head x sequence x tokens), eight waves of 16 or 32
// rows each: scores are K Q^T, so that a lane's scores are of one row and its weights are already the second product's operand
// (O^T = V^T W^T); rows stay in registers, blocks of keys and values pass through rings in the LDS, each read by all waves.
//
// Bound by the matrix cores and, as near, by the LDS: a block of 32 keys is 2048 clocks of 16x16x32 products on every SIMD for
// fp32 rows of 256 dims (16 a wave, queries and weights in two parts), half as many again for bf16 rows (32 a wave, weights in
// two), and 256 KB of the LDS for eight waves, at 128 bytes a clock 2048. It takes 2950 clocks (fp32) or 4270 to 4750 (bf16);
// with half the LDS reads an fp32 chunk took 181 us in place of 224. Measured with 16 heads over 2 KV heads of 256: 2048 bf16
// tokens behind 2048 162 to 169 us (103 GFLOP: 0.63 PFLOP/s, 0.95 in parts; weights of one part, 11 bits, took 130), 1024 fp32
// behind 7168 222 to 230 us (129 GFLOP: 0.58, twice that in parts), 4096 bf16 in a window of 1024 118 to 122 us (73 GFLOP: 0.62,
// 0.93 in parts), 61 fp32 behind 16384 50 to 52 us, at a clock of 1.8 to 1.9 GHz. A segment costs some 13000 clocks to begin, a
// partial 12000 to 13000, an item's rows 28000 to 35000 where all workgroups write theirs at once, up to 64000 with a join.
//
// 32 bf16 rows a wave of 256 dims spill 32 registers: none in the loop over the blocks, all around the writing of the rows.
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
    int* cnt;       // [groups][waves][2] arrivals at the 16-row tiles of the item that is the workgroup's last
    int64_t* unit;  // [groups + 1]: the workgroups' first units
    // joined calls, instead: [0] parts a KV head, then of each (sequence, query tile) its first part and its parts
    int* joined;
};
constexpr int kJoinPairs = 64;  // most (sequence, query tile) pairs of a joined call
__host__ __device__ inline ChPlan ch_plan(void* ws, int groups, int part_floats) {
    ChPlan p;
    p.part = static_cast<float*>(ws);
    p.start = reinterpret_cast<int4*>(p.part + (size_t)2 * groups * kChWaves * part_floats);
    p.cnt = reinterpret_cast<int*>(p.start + groups);
    p.unit = reinterpret_cast<int64_t*>(p.cnt + groups * kChWaves * 2);
    p.joined = reinterpret_cast<int*>(p.unit + groups + 1);
    return p;
}
// Items are (KV head, sequence, query tile) in this order, each of as many units as it has key tiles (at most 2^20). Every
// workgroup of the chunk kernel takes a run of units, in one of two ways (a segment, what a workgroup takes of an item, costs some
// three to four units beside its own: the rows, the first copies, the partial and its joining):
//  - items in equal parts of at most `run` units, a workgroup a part, for the least run whose parts fit the workgroups;
//  - equal runs over all items, every item's first unit preceded by kSegment that stand for a segment's cost, their ends moved by up
//    to a twelfth to an item's edge where one is that near: where there are more items than workgroups, or where the first way's run
//    is longer by more than kUneven units. Measured on 2048 bf16 tokens behind 2048 (16 heads of 256, 128 items of 33 to 64 tiles):
//    equal runs 165 us, with nothing for the segments 170, with eight units each 167; 6 prompts of up to 701 bf16 tokens 56, 87 and 57;
//    2048 bf16 of 32 + 8 heads of 128 behind 2048 173, 175 and 182. On 1024 fp32 tokens behind 7168 equal parts 224 us, equal runs 234.
constexpr int kSegment = 4, kUneven = 2;
constexpr int64_t kItem = (int64_t)1 << 42;  // sums of units (2^20 of an item) count the items (less than 2^21) from this bit on
__device__ __forceinline__ int64_t units_of(int64_t sum) { return sum & (kItem - 1); }
__device__ __forceinline__ int64_t costs_of(int64_t sum) { return units_of(sum) + (sum / kItem) * kSegment; }

// The least run in [lo, hi] whose parts fit the workgroups, hi's known to: 64 runs at a time, a lane each. count(i): tiles of pair i.
template <typename F>
__device__ __forceinline__ int least_run(F&& count, int pairs, int nkv, int groups, int lo, int hi, int lane) {
    while (lo < hi) {
        const int step = (hi - lo + 63) / 64;
        const float r = (float)min(hi, lo + step * lane);
        int parts = 0;
        for (int i = 0; i < pairs; i++) parts += parts_of(count(i), r);
        const uint64_t fits = __builtin_amdgcn_ballot_w64(parts * nkv <= groups);
        const int f = fits ? (int)__builtin_ctzll(fits) : 64, was = lo;
        if (f == 0) break;
        lo = min(hi, was + step * (f - 1) + 1);
        if (f < 64) hi = min(hi, was + step * f);
    }
    return lo;
}

// One workgroup: a thread a run of (sequence, query tile) pairs (one pair, where the first way is tried), a scan places the runs,
// and the threads write the starts that fall into theirs.
template <int THREADS>
__global__ __launch_bounds__(THREADS) void k_paged_plan(PagedAttendArgs a, void* ws, int groups, int part_floats, int tok) {
    constexpr int WAVES = THREADS / 64;
    __shared__ int64_t sums[WAVES];
    __shared__ int tops[WAVES], ksums[WAVES], count[THREADS];
    const ChPlan plan = ch_plan(ws, groups, part_floats);
    const int nqt = (a.n + tok - 1) / tok, pairs = a.n_seq * nqt;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = (pairs + THREADS - 1) / THREADS;
    auto tiles = [&](int pair) {
        const int b = pair / nqt, t0 = (pair - b * nqt) * tok;
        return key_tiles<6>(a, seq_pos(a.pos, b), t0, min(t0 + tok, seq_len(a.lens, b, a.n))).count;
    };
    int64_t mine = 0;
    int top = 0;
    for (int i = 0; i < per; i++) {
        const int pair = tid * per + i, c = pair < pairs ? tiles(pair) : 0;
        mine += c + (c ? kItem : 0), top = max(top, c);
        if (per == 1) count[tid] = c;
    }
    for (int i = tid; i < groups * kChWaves * 2; i += THREADS) plan.cnt[i] = 0;
    int64_t incl = mine;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const int64_t o = __shfl_up((long long)incl, m, 64);
        if (lane >= m) incl += o;
        top = max(top, __shfl_xor(top, m, 64));
    }
    if (lane == 63) sums[wave] = incl, tops[wave] = top;
    __syncthreads();
    int64_t before = incl - mine, sum = 0;
#pragma unroll
    for (int w = 0; w < WAVES; w++) before += w < wave ? sums[w] : 0, sum += sums[w], top = max(top, tops[w]);
    const int64_t total = units_of(sum), all = total * a.NKV, cost = costs_of(sum);
    const int64_t run = max((int64_t)1, (cost * a.NKV + groups - 1) / groups);
    if (tid == 0) plan.unit[groups] = all;

    if (per == 1 && pairs * a.NKV <= groups && top > 0) {
        const int part = least_run([&](int i) { return count[i]; }, pairs, a.NKV, groups, max(1, (int)((all + groups - 1) / groups)),
                                   top, lane);
        if (part <= run + kUneven) {
            const int c = count[tid], k = parts_of(c, (float)part);
            int kincl = k;
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) {
                const int o = __shfl_up(kincl, m, 64);
                if (lane >= m) kincl += o;
            }
            if (lane == 63) ksums[wave] = kincl;
            __syncthreads();
            int at = kincl - k, parts = 0;
#pragma unroll
            for (int w = 0; w < WAVES; w++) at += w < wave ? ksums[w] : 0, parts += ksums[w];
            for (int h = 0; h < a.NKV; h++)
                for (int j = 0; j < k; j++) {
                    const int w = h * parts + at + j, off = (int)((unsigned)c * (unsigned)j / (unsigned)k);  // (c j < 2^28)
                    plan.start[w] = int4{h, tid / nqt, tid % nqt, off}, plan.unit[w] = h * total + units_of(before) + off;
                }
            for (int w = parts * a.NKV + tid; w < groups; w += THREADS) plan.start[w].x = -1, plan.unit[w] = all;
            return;
        }
    }
    for (int w = tid; w < groups; w += THREADS)
        if (w * run >= cost * a.NKV) plan.start[w].x = -1, plan.unit[w] = all;
    const int near = (int)min(run / 12, (int64_t)1 << 20);
    for (int i = 0; i < per; i++) {
        const int pair = tid * per + i;
        if (pair >= pairs) break;
        const int c = tiles(pair);
        for (int h = 0; h < a.NKV && c; h++) {
            const int64_t g0 = h * cost + costs_of(before);
            for (int64_t w = (g0 + run - 1) / run; w * run < g0 + kSegment + c; w++) {
                int off = max((int)(w * run - g0) - kSegment, 0);
                if (off <= near) off = 0;
                else if (c - off <= near) off = c;  // the item after this
                plan.start[w] = int4{h, pair / nqt, pair % nqt, off}, plan.unit[w] = h * total + units_of(before) + off;
            }
        }
        before += c + (c ? kItem : 0);
    }
}

// The first way by every wave for itself, for calls of so few items that a second launch joins them: a lane a pair, then a lane a
// run. Part w of all is key tiles [lo, hi) of KV head h and (sequence, query tile) `pair`; false behind the last part. `out`: where
// the joining launch finds every pair's parts.
struct Part {
    int h, pair, lo, hi;
};
template <typename F>
__device__ __forceinline__ bool joined_part(F&& tiles, int pairs, int nkv, int groups, int w, int lane, int* out, Part& p) {
    const int mine = lane < pairs ? tiles(lane) : 0;
    int total = 0, hi = 1;
    for (int i = 0; i < pairs; i++) {
        const int c = __builtin_amdgcn_readlane(mine, i);
        total += c, hi = max(hi, c);  // (at most 2^20 each)
    }
    const int lo = least_run([&](int i) { return __builtin_amdgcn_readlane(mine, i); }, pairs, nkv, groups,
                             max(1, (int)(((int64_t)total * nkv + groups - 1) / groups)), hi, lane);
    const int parts = parts_of(mine, (float)lo);
    int all = 0;
    for (int i = 0; i < pairs; i++) {
        const int k = __builtin_amdgcn_readlane(parts, i);
        if (out && lane == 0) out[1 + 2 * i] = all, out[2 + 2 * i] = k;
        all += k;
    }
    if (out && lane == 0) out[0] = all;
    if (w >= all * nkv) return false;
    p.h = w / all;
    int at = w - p.h * all;
    for (p.pair = 0;; p.pair++) {
        const int k = __builtin_amdgcn_readlane(parts, p.pair);
        if (at < k) {
            const unsigned c = __builtin_amdgcn_readlane(mine, p.pair);
            p.lo = (int)(c * (unsigned)at / (unsigned)k), p.hi = (int)(c * (unsigned)(at + 1) / (unsigned)k);
            return true;
        }
        at -= k;
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
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int lgG = __builtin_ctz(a.NH / a.NKV), G = 1 << lgG, tok = C::ROWS >> lgG, groups = gridDim.x;
    const ChPlan plan = ch_plan(ws, groups, C::PART);
    // neighbouring runs on one XCD: they read the same keys
    const int wg = (blockIdx.x & 7) * (groups >> 3) + (blockIdx.x >> 3);
    int h, b, qt, off;
    int64_t at, stop;  // units of the segment at hand and of the run's end
    if (joined) {
        const int nqt = (a.n + tok - 1) / tok;
        auto tiles = [&](int pair) {
            const int sb = pair / nqt, st0 = (pair - sb * nqt) * tok;
            return key_tiles<6>(a, seq_pos(a.pos, sb), st0, min(st0 + tok, seq_len(a.lens, sb, a.n))).count;
        };
        Part p;
        if (!joined_part(tiles, a.n_seq * nqt, a.NKV, groups, wg, lane_here(), wg == 0 && wave == 0 ? plan.joined : nullptr, p)) return;
        h = p.h, b = p.pair / nqt, qt = p.pair - b * nqt, off = p.lo, at = 0, stop = p.hi - p.lo;
    } else {
        const int4 st = plan.start[wg];
        h = __builtin_amdgcn_readfirstlane(st.x), b = __builtin_amdgcn_readfirstlane(st.y);
        qt = __builtin_amdgcn_readfirstlane(st.z), off = __builtin_amdgcn_readfirstlane(st.w);
        if (h < 0) return;
        at = plan.unit[wg], stop = plan.unit[wg + 1];
    }

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

        // positions of the wave's tokens, the keys that all of them see, that some of them see, and that some of the item's do
        const int w0 = pos + t0 + (wave * 16 * NT >> lgG), w1 = min(pos + t0 + ((wave * 16 * NT + 16 * NT - 1) >> lgG), pos + t1 - 1);
        const Sight all_see = sight_of_all(a, w0, w1), some_see = sight_of_some(a, w0, w1);
        const Sight item_see = sight_of_some(a, pos + t0, pos + t1 - 1);

        // ---- staging. What a step needs to know of its blocks is worked out for 64 of them at a time, a lane each: scalar
        // arithmetic in every step (page, offset, masks: some 150 instructions) took as long as its matrix instructions ----
        const int32_t* table = a.c.table + (size_t)b * a.c.table_stride;
        int base = 0;
        int number = -1;       // lane l: number of block base + l in a pool, -1 without a page or past the last block
        int first_key = 0;     // its first position
        uint64_t paged, whole, stale;  // bit l: it has a page; all rows of the wave see all of it; it has keys that no row of the item sees
        auto survey = [&](int i) __attribute__((always_inline)) {
            base = i;
            const int l = lane_here();
            const bool in = i + l < n;
            first_key = key_of(min(i + l, n - 1));
            const int page = in && first_key < a.limit ? table[first_key >> a.c.lg_page] : -1;
            const bool there = (uint32_t)page < (uint32_t)a.c.n_pages;
            number = there ? paged_number(a.c, page, first_key, h, a.NKV) : -1;
            paged = __builtin_amdgcn_ballot_w64(there);
            whole = __builtin_amdgcn_ballot_w64(there && sees_whole(all_see, first_key, first_key + kBlk, a.sinks));
            stale = __builtin_amdgcn_ballot_w64(in && !sees_whole(item_see, first_key, first_key + kBlk, a.sinks));
        };
        auto key_at = [&](int i) { return __builtin_amdgcn_readlane(first_key, i - base); };
        // This wave's share of the copy of block `of`'s keys or values (zeros without a page) into ring place of % 4, a kilobyte a piece
        // (at 64 dims four waves copy keys and the others values)
        constexpr int PIECES = D >= 128 ? D / 128 : 1;
        auto copy = [&](bool keys, int of) __attribute__((always_inline)) {
            if (D < 128 && keys != (wave < 4)) return;
            const int blk = __builtin_amdgcn_readlane(number, of - base), at = D >= 128 ? wave * PIECES : wave & 3;
            uint16_t* from = (keys ? a.c.k : a.c.v) + (int64_t)max(blk, 0) * BLKE;
            const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(from, (short)0, blk < 0 ? 0 : BLKE * 2, 0x00020000);
            f16* to = (keys ? sk : sv) + (of & (kChRing - 1)) * BLKE + at * 512;
            const int l16 = lane_here() * 16;
#pragma unroll
            for (int k = 0; k < PIECES; k++)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(to + k * 512), 16,
                                                         l16 + (at + k) * 1024, 0, 0, 0);
        };
        survey(0);

        // ---- the wave's rows as they lie in memory: row r of the tile is token t0 + (r >> lgG), head h G + (r & (G - 1)) ----
        typedef typename std::conditional<DT == 0, f32x4, u32x4>::type raw_t;
        constexpr int RAW = DT == 0 ? 2 : 1;
        raw_t raw[NT][NKS][RAW];
        {
            const int lane = lane_here(), col = lane & 15, g = lane >> 4;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int r = (wave * NT + nt) * 16 + col, t = min(t0 + (r >> lgG), t1 - 1);
            const size_t base = ((size_t)b * a.n + t) * a.q_stride + (size_t)(h * G + (r & (G - 1))) * a.q_head + 8 * g;
#pragma unroll
            for (int kk = 0; kk < NKS; kk++)
#pragma unroll
                for (int k = 0; k < RAW; k++) {
                    if constexpr (DT == 0)
                        raw[nt][kk][k] = *reinterpret_cast<const raw_t*>(static_cast<const float*>(a.q) + base + 32 * kk + 4 * k);
                    else raw[nt][kk][k] = *reinterpret_cast<const raw_t*>(static_cast<const uint16_t*>(a.q) + base + 32 * kk);
                }
        }
        }

        // (their loads and the pages' are on their way) the last segment's readers of the rings are done
        phase();
        copy(true, 0), copy(true, 1), copy(false, 0);

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
                for (int j = 0; j < 8; j += 2)  // (in assembly: without the compiler's canonical operands)
                    asm("v_max3_f32 %0, |%1|, |%2|, %0" : "+v"(largest) : "v"(at_raw(kk, j)), "v"(at_raw(kk, j + 1)));
            const int sh = query_shift(max_rows(largest));
            const float up = power_of_two(sh);
            fac[nt] = a.scale * power_of_two(-sh);
#pragma unroll
            for (int kk = 0; kk < NKS; kk++)
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float y = at_raw(kk, j) * up;
                    q[nt][0][kk][j] = (f16)y;
                    if constexpr (PARTS == 2) q[nt][1][kk][j] = (f16)(y - (float)q[nt][0][kk][j]);
                }
            m_run[nt] = kNegInf, l_run[nt] = 0.f;
#pragma unroll
            for (int dt = 0; dt < NDT; dt++) acc[nt][dt] = f32x4{};
        }
        auto unseen = [&](int k0) { return k0 >= some_see.end || (k0 + kBlk <= some_see.from && k0 >= a.sinks); };
        auto row_sight = [&](int nt, int l) {
            const int r = (wave * NT + nt) * 16 + (l & 15), t = t0 + (r >> lgG);
            return t < t1 ? sight(a, pos + t) : Sight{0, 0};
        };

        f32x4 s[NT][2];        // scores of a block: value i of key set s of lane (col, g) is key 8 g + 4 s + i
        f16x8 w[NT][kWeightParts];  // its weights: keys 8 g .. 8 g + 7
        // Matrix instructions of a phase: the weighted values of one block, then the scores of the next, their fragments read AHEAD of
        // their use (one after the other: scores and weights are then not live together, which leaves registers for fragments)
        constexpr int AHEAD = 5;
        auto products = [&](auto&& kfrag, auto&& vfrag) __attribute__((always_inline)) {
            f16x8 fr[AHEAD + 1];
            auto read = [&](auto ic) __attribute__((always_inline)) {
                constexpr int i = decltype(ic)::value;
                fr[i % (AHEAD + 1)] = i < NDT ? vfrag(i) : kfrag(i - NDT);
            };
            static_for<0, AHEAD>(read);
            static_for<0, 2 * NDT>([&](auto ic) __attribute__((always_inline)) {
                constexpr int i = decltype(ic)::value, f = i % NDT;
                if constexpr (i + AHEAD < 2 * NDT) read(std::integral_constant<int, i + AHEAD>{});
#pragma unroll
                for (int part = 0; part < (i < NDT ? kWeightParts : PARTS); part++)
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        if constexpr (i < NDT) acc[nt][f] = mfma16(fr[i % (AHEAD + 1)], w[nt][part], acc[nt][f]);
                        else s[nt][f & 1] = mfma16(fr[i % (AHEAD + 1)], q[nt][part][f >> 1], f < 2 && part == 0 ? f32x4{} : s[nt][f & 1]);
                    }
                __builtin_amdgcn_sched_barrier(0);  // keep the reads ahead
            });
            asm volatile("s_nop 15\n\ts_nop 3");  // the last scores are out before assembly reads them
        };
        // Scores that the rows of 16-row tile nt do not see, of the block at key k0
        auto hide = [&](f32x4 (&x)[2], int nt, int k0, bool there) __attribute__((always_inline)) {
            const int l = lane_here(), key = k0 + 8 * (l >> 4);
            const Sight see = row_sight(nt, l);
#pragma unroll
            for (int i = 0; i < 8; i++) x[i >> 2][i & 3] = there && see.sees(key + i, a.sinks) ? x[i >> 2][i & 3] : kNegInf;
        };
        // (the maxima in assembly: the compiler would make every operand canonical first, which doubles them. The scores are those of
        // an earlier phase, or of products() behind its own wait)
        auto max3 = [](float x, float y, float z) __attribute__((always_inline)) {
            float r;
            asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
            return r;
        };
        auto largest = [&](const f32x4 (&x)[2]) __attribute__((always_inline)) {
            float r = max3(max3(x[0][0], x[0][1], x[0][2]), max3(x[0][3], x[1][0], x[1][1]), max3(x[1][2], x[1][3], x[1][3]));
            const auto y = __builtin_amdgcn_permlane16_swap(__float_as_uint(r), __float_as_uint(r), false, false);
            r = max3(__uint_as_float(y[0]), __uint_as_float(y[1]), __uint_as_float(y[1]));
            const auto z = __builtin_amdgcn_permlane32_swap(__float_as_uint(r), __float_as_uint(r), false, false);
            return max3(__uint_as_float(z[0]), __uint_as_float(z[1]), __uint_as_float(z[1]));
        };
        // The running maximum moves only where a row's passes it by more than kTau (at first from -inf); the factor of what was
        // summed before
        auto raise = [&](float mx, float& m, float& l) __attribute__((always_inline)) {
            const float to = mx > m + kTau ? mx : m, corr = to == kNegInf ? 1.f : exp2_fast(m - to);
            m = to, l *= corr;
            return corr;
        };
        auto weigh = [&](const f32x4 (&x)[2], float f, float m, float& l, f16x8 (&wt)[kWeightParts]) __attribute__((always_inline)) {
            const float o = m == kNegInf ? 0.f : kShift - m;
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                const float x0 = exp2_fast(__builtin_fmaf(x[i >> 2][i & 3], f, o)), x1 = exp2_fast(__builtin_fmaf(x[i >> 2][(i & 3) + 1], f, o));
                f16x2 hi16, lo16;
                weight_parts(x0, x1, hi16, lo16);
                wt[0][i] = hi16[0], wt[0][i + 1] = hi16[1], wt[1][i] = lo16[0], wt[1][i + 1] = lo16[1];
                l += x0 + x1;
            }
        };
        // Weights of a block from its scores, the copies of step `step` between: a piece takes the memory path 16 cycles, and one behind
        // the other they would hold the wave up
        auto softmax = [&](int k0, bool there, bool all, int step) __attribute__((always_inline)) {
            copy(true, step + 1);
            if (!all) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++) hide(s[nt], nt, k0, there);
            }
            float mx[NT];
            uint64_t grow = 0;
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                mx[nt] = largest(s[nt]) * fac[nt];
                grow |= __builtin_amdgcn_ballot_w64(mx[nt] > m_run[nt] + kTau);
            }
            if (grow) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    const float corr = raise(mx[nt], m_run[nt], l_run[nt]);
#pragma unroll
                    for (int dt = 0; dt < NDT; dt++) acc[nt][dt] *= corr;
                }
            }
            copy(false, step);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) weigh(s[nt], fac[nt], m_run[nt], l_run[nt], w[nt]);
        };
        // Rows of 16-row tile nt whose unnormalized outputs lie in `mine`: an item of one part to the output, parts to the workspace,
        // where the wave that arrives last joins them, from the first to the last whichever it is. Loads go out together: their
        // latency, not their bytes, is what this takes.
        auto write_rows = [&](int nt, const f32x4* mine, auto&& region, int parts, int own) __attribute__((always_inline)) {
            const int lane = lane_here(), col = lane & 15, g = lane >> 4;
            const int r = (wave * NT + nt) * 16 + col, t = t0 + (r >> lgG);
            const bool ok = t < t1;
            const size_t row = (size_t)b * a.n + (ok ? t : t0);
            const int head = h * G + (r & (G - 1));
            Gate4<DT> gate[NDT];
            auto load_gates = [&]() __attribute__((always_inline)) {
                if (a.gate) {
#pragma unroll
                    for (int dt = 0; dt < NDT; dt++) gate[dt].load(a, row, head, 16 * dt + 4 * g);
                } else {
#pragma unroll
                    for (int dt = 0; dt < NDT; dt++) gate[dt].none();
                }
            };
            const auto xs = __builtin_amdgcn_permlane16_swap(__float_as_uint(l_run[nt]), __float_as_uint(l_run[nt]), false, false);
            float l = __uint_as_float(xs[0]) + __uint_as_float(xs[1]);
            const auto ys = __builtin_amdgcn_permlane32_swap(__float_as_uint(l), __float_as_uint(l), false, false);
            l = __uint_as_float(ys[0]) + __uint_as_float(ys[1]);
            const float m = m_run[nt];
            if (parts == 1) {
                load_gates();
                if (ok) {
                    const float inv = inverse_sum(l);
#pragma unroll
                    for (int dt = 0; dt < NDT; dt++) store_out4<DT>(a, row, head, D, 16 * dt + 4 * g, mine[dt * 64], inv, gate[dt]);
                }
                return;
            }
            int* arrived = plan.cnt + ((wg - own) * kChWaves + wave) * 2 + nt;
            // (the last to arrive need not store its own part)
            if (joined ||
                __builtin_amdgcn_readfirstlane(__hip_atomic_load(arrived, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) < parts - 1) {
                const __amdgpu_buffer_rsrc_t rp = region(own);
#pragma unroll
                for (int dt = 0; dt < NDT; dt++)
                    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, mine[dt * 64]), rp,
                                                           ((nt * NDT + dt) * 64 + lane) * 16, 0, kScDevice);
                __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, f32x2{m, l}), rp,
                                                      NT * NDT * 1024 + (nt * 64 + lane) * 8, 0, kScDevice);
                if (joined) return;
                __builtin_amdgcn_s_waitcnt(0x0F70);  // the partial is out before it is counted
                int old = 0;
                if (lane == 0) old = __hip_atomic_fetch_add(arrived, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                if (__builtin_amdgcn_readfirstlane(old) < parts - 1) return;
            }
            asm volatile("" ::: "memory");
            load_gates();
            auto sums = [&](const __amdgpu_buffer_rsrc_t& rq) __attribute__((always_inline)) {
                return __builtin_bit_cast(f32x2, __builtin_amdgcn_raw_buffer_load_b64(rq, NT * NDT * 1024 + (nt * 64 + lane) * 8, 0, kScDevice));
            };
            auto values = [&](const __amdgpu_buffer_rsrc_t& rq, int dt) __attribute__((always_inline)) {
                return __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rq, ((nt * NDT + dt) * 64 + lane) * 16, 0, kScDevice));
            };
            f32x4 o[NDT];
            if (parts == 2) {  // x cx + y cy, x the first part's
                const __amdgpu_buffer_rsrc_t rq = region(1 - own);
                const f32x2 ml = sums(rq);
#pragma unroll
                for (int dt = 0; dt < NDT; dt++) o[dt] = values(rq, dt);
                const float to = fmaxf(m, ml[0]);
                const float cm = m == kNegInf ? 0.f : exp2_fast(m - to), co = ml[0] == kNegInf ? 0.f : exp2_fast(ml[0] - to);
                const float cx = own ? co : cm, cy = own ? cm : co;
                const float inv = inverse_sum(__builtin_fmaf(own ? l : ml[1], cy, (own ? ml[1] : l) * cx));
                if (ok) {
#pragma unroll
                    for (int dt = 0; dt < NDT; dt++) {
                        const f32x4 me = mine[dt * 64];
                        f32x4 v;
#pragma unroll
                        for (int i = 0; i < 4; i++) v[i] = __builtin_fmaf(own ? me[i] : o[dt][i], cy, (own ? o[dt][i] : me[i]) * cx);
                        store_out4<DT>(a, row, head, D, 16 * dt + 4 * g, v, inv, gate[dt]);
                    }
                }
                return;
            }
            float rm = kNegInf, rl = 0.f;
#pragma unroll
            for (int dt = 0; dt < NDT; dt++) o[dt] = f32x4{};
#pragma unroll 1
            for (int part = 0; part < parts; part++) {
                f32x2 ml = f32x2{m, l};
                f32x4 v[NDT];
                if (part == own) {
#pragma unroll
                    for (int dt = 0; dt < NDT; dt++) v[dt] = mine[dt * 64];
                } else {
                    const __amdgpu_buffer_rsrc_t rq = region(part);
                    ml = sums(rq);
#pragma unroll
                    for (int dt = 0; dt < NDT; dt++) v[dt] = values(rq, dt);
                }
                const float to = fmaxf(rm, ml[0]);
                const float cx = rm == kNegInf ? 0.f : exp2_fast(rm - to), cy = ml[0] == kNegInf ? 0.f : exp2_fast(ml[0] - to);
                rm = to, rl = __builtin_fmaf(ml[1], cy, rl * cx);
#pragma unroll
                for (int dt = 0; dt < NDT; dt++)
#pragma unroll
                    for (int i = 0; i < 4; i++) o[dt][i] = __builtin_fmaf(v[dt][i], cy, o[dt][i] * cx);
            }
            if (ok) {
                const float inv = inverse_sum(rl);
#pragma unroll
                for (int dt = 0; dt < NDT; dt++) store_out4<DT>(a, row, head, D, 16 * dt + 4 * g, o[dt], inv, gate[dt]);
            }
        };

        // ---- two groups of four waves, one of each on every SIMD, take turns: in a phase one runs the matrix instructions
        // of a block (and the weighted values of the block before) while the other takes its softmax and copies. In the first
        // group's phases 2 i (matrix) and 2 i + 1 (softmax of block i) the second group's are one later. Keys of block j are read in
        // phases 2 j and 2 j + 1, values of block j in 2 j + 2 and 2 j + 3; the first group copies its share of keys of block i + 2 and
        // values of block i + 1 in phase 2 i + 1 and the second its in phase 2 i, behind the last reads of the places (keys of block i - 2
        // in phase 2 i - 3, values of block i - 3 in 2 i - 3), and each waits for them two phases later, before phase 2 i + 4. ----
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
        // The copies of the step before have landed (keys of block i + 1, values of block i); step i copies keys of block i + 2 and values
        // of block i + 1.
        auto arrive = [&](int i) __attribute__((always_inline)) {
            if (i + 2 - base >= 64) survey(i - 1);
            landed<0>();
            if (stale >> (i - base) & 1) clean(i);
        };
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int part = 0; part < kWeightParts; part++) w[nt][part] = f16x8{};
        bool check = false;  // the block before is not whole: its values may be some that only some rows see
        auto matrix_phase = [&](int i) __attribute__((always_inline)) {  // scores of block i, values of block i - 1
            if (check) {
                const auto read = vfrag_of(i - 1);
                uint32_t odd = 0;
#pragma unroll 4
                for (int dt = 0; dt < NDT; dt++) odd |= not_finite(read(dt));
                if (__builtin_amdgcn_ballot_w64(odd != 0)) odd_values = true;
            }
            products(kfrag_of(i), vfrag_of(i - 1));
        };
        auto softmax_phase = [&](int i) __attribute__((always_inline)) {
            const bool all = whole >> (i - base) & 1;
            softmax(key_at(i), paged >> (i - base) & 1, all, i + second + 1);
            check = !all;
        };
        // (the values of the block before the first)
        for (int k = wave * 64 + lane_here(); k < BLKE / 8; k += 64 * kChWaves)
            *reinterpret_cast<u32x4*>(sv + (kChRing - 1) * BLKE + k * 8) = u32x4{};
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0xC07F);
        landed<C::COPIES>();
        phase();
        if (second) {
            arrive(0);
            copy(true, 2), copy(false, 1);
            phase();
        }
#pragma unroll 1
        for (int i = 0; i < n; i++) {
            matrix_phase(i);
            phase();
            arrive(i + second);
            softmax_phase(i);
            phase();
        }
        matrix_phase(n);  // (its scores are of no block)
        if (!second) phase();
        landed<0>();  // (copies past the last block write zeros)
        phase();      // the rings are free

        // ---- 16 rows at a time through the wave's part of the rings' room: the loop's registers hold the outputs only in the
        // loop (with what follows working on them there, 32-row waves spill inside it) ----
        const int lane = lane_here(), col = lane & 15, g = lane >> 4;
        f32x4* mine = reinterpret_cast<f32x4*>(smem) + wave * NDT * 64 + lane;  // [dim tile][lane]
        const int64_t item = at - off;
        const bool split = lo > 0 || hi < kt.count;
        int first = wg, parts = 1;
        if (split && joined) {
            first -= lo > 0, parts = 2;  // (only whether this is the first part matters here)
        } else if (split) {
            while (plan.unit[first] > item) first--;
            int last = wg;
            while (plan.unit[last + 1] < item + kt.count) last++;
            parts = last - first + 1;
        }
        const int own = wg - first;
        auto region = [&](int part) {
            const size_t slot = part == 0 ? 2 * first + 1 : 2 * (first + part);
            return __builtin_amdgcn_make_buffer_rsrc(plan.part + (slot * kChWaves + wave) * C::PART, (short)0, C::PART * 4, 0x00020000);
        };
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            if (odd_values) {
                // a value that only some of the wave's rows see is not finite, and a weight of zero does not hide it: the segment
                // again, from memory, its weighted values token by token with those hidden from it zeroed
                float m = kNegInf, l = 0.f;
#pragma unroll 1
                for (int dt = 0; dt < NDT; dt++) mine[dt * 64] = f32x4{};
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
                    f32x4 x[2] = {f32x4{}, f32x4{}};
#pragma unroll
                    for (int f = 0; f < NDT; f++)
#pragma unroll
                        for (int part = 0; part < PARTS; part++) x[f & 1] = mfma16(get(rk, f), q[nt][part][f >> 1], x[f & 1]);
                    asm volatile("s_nop 15\n\ts_nop 3" : "+v"(x[0]), "+v"(x[1]));  // (as in products())
                    hide(x, nt, k0, true);
                    const float corr = raise(largest(x) * fac[nt], m, l);
                    f16x8 wt[kWeightParts];
                    weigh(x, fac[nt], m, l, wt);
#pragma unroll 1
                    for (int dt = 0; dt < NDT; dt++) {
                        const f16x8 v = get(rv, dt);
                        const f32x4 old = mine[dt * 64] * corr;
                        f32x4 sum = old;
#pragma unroll 1
                        for (int p = w0; p <= w1; p++) {
                            const Sight sp = sight(a, p);
                            const f16x8 vp = keep_keys(v, [&](int j) { return sp.sees(k0 + 8 * g + j, a.sinks); });
                            f32x4 o = old;
#pragma unroll
                            for (int part = 0; part < kWeightParts; part++) o = mfma16(vp, wt[part], o);
                            const bool its = pos + t0 + (((wave * NT + nt) * 16 + col) >> lgG) == p;
#pragma unroll
                            for (int j = 0; j < 4; j++) sum[j] = its ? o[j] : sum[j];
                        }
                        mine[dt * 64] = sum;
                    }
                }
                m_run[nt] = m, l_run[nt] = l;
            } else {
#pragma unroll
                for (int dt = 0; dt < NDT; dt++) mine[dt * 64] = acc[nt][dt];
            }
            write_rows(nt, mine, region, parts, own);
        }
        at += hi - lo;
        off = hi;
    }
}

// Joins the parts of split items where there are few items: a workgroup 16 rows of an item and a quarter of its dims; its four
// waves take the parts in turn, four of them at a time, and are joined through the LDS, all in a fixed order.
template <int D, int DT, int NT>
__global__ __launch_bounds__(256) void k_paged_join_chunk(PagedAttendArgs a, void* ws, int groups) {
    using C = ChCfg<D, DT, NT>;
    constexpr int NQ = C::NDT / 4;  // dim tiles of a quarter
    __shared__ f32x4 red[4][NQ][64];
    __shared__ f32x2 red_ml[4][64];
    const ChPlan plan = ch_plan(ws, groups, C::PART);
    const int lgG = __builtin_ctz(a.NH / a.NKV), G = 1 << lgG, tok = C::ROWS >> lgG, nqt = (a.n + tok - 1) / tok;
    int x = blockIdx.x;
    const int quarter = x % 4, sub = x / 4 % (kChWaves * NT);
    x /= 4 * kChWaves * NT;
    const int h = x % a.NKV, pair = x / a.NKV, b = pair / nqt, t0 = (pair - b * nqt) * tok;
    const int first = h * plan.joined[0] + plan.joined[1 + 2 * pair], parts = plan.joined[2 + 2 * pair];
    const int t1 = min(t0 + tok, seq_len(a.lens, b, a.n));
    if (parts <= 1 || t0 >= t1) return;
    const int lane = threadIdx.x & 63, set = threadIdx.x >> 6, col = lane & 15, g = lane >> 4, wave = sub / NT, nt = sub % NT;
    const int r = sub * 16 + col, t = t0 + (r >> lgG);
    const bool ok = t < t1;
    Gate4<DT> gate[NQ];
#pragma unroll
    for (int j = 0; j < NQ; j++) gate[j].none();
    if (a.gate && set == 0) {
#pragma unroll
        for (int j = 0; j < NQ; j++) gate[j].load(a, (size_t)b * a.n + (ok ? t : t0), h * G + (r & (G - 1)), 16 * (quarter * NQ + j) + 4 * g);
    }
    float m = kNegInf, l = 0.f;
    f32x4 o[NQ];
#pragma unroll
    for (int j = 0; j < NQ; j++) o[j] = f32x4{};
    constexpr int AT = 4;  // parts in flight
    for (int p0 = set; p0 < parts; p0 += 4 * AT) {
        f32x2 ml[AT];
        f32x4 v[AT][NQ];
#pragma unroll
        for (int k = 0; k < AT; k++) {
            const int p = min(p0 + 4 * k, parts - 1);  // (past the last one: not used)
            const float* at = plan.part + ((size_t)(p == 0 ? 2 * first + 1 : 2 * (first + p)) * kChWaves + wave) * C::PART;
            ml[k] = *reinterpret_cast<const f32x2*>(at + NT * C::NDT * 256 + (nt * 64 + lane) * 2);
#pragma unroll
            for (int j = 0; j < NQ; j++) v[k][j] = *reinterpret_cast<const f32x4*>(at + ((nt * C::NDT + quarter * NQ + j) * 64 + lane) * 4);
        }
#pragma unroll
        for (int k = 0; k < AT; k++) {
            if (p0 + 4 * k >= parts) break;
            const float to = fmaxf(m, ml[k][0]);
            const float cx = m == kNegInf ? 0.f : exp2_fast(m - to), cy = ml[k][0] == kNegInf ? 0.f : exp2_fast(ml[k][0] - to);
            m = to, l = __builtin_fmaf(ml[k][1], cy, l * cx);
#pragma unroll
            for (int j = 0; j < NQ; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) o[j][i] = __builtin_fmaf(v[k][j][i], cy, o[j][i] * cx);
        }
    }
    red_ml[set][lane] = f32x2{m, l};
#pragma unroll
    for (int j = 0; j < NQ; j++) red[set][j][lane] = o[j];
    __syncthreads();
    if (set > 0 || !ok) return;
    float c[4], top = kNegInf;
#pragma unroll
    for (int k = 0; k < 4; k++) top = fmaxf(top, red_ml[k][lane][0]);
    l = 0.f;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        c[k] = red_ml[k][lane][0] == kNegInf ? 0.f : exp2_fast(red_ml[k][lane][0] - top);
        l = __builtin_fmaf(red_ml[k][lane][1], c[k], l);
    }
    const float inv = inverse_sum(l);
#pragma unroll
    for (int j = 0; j < NQ; j++) {
        f32x4 v{};
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = __builtin_fmaf(red[k][j][lane][i], c[k], v[i]);
        store_out4<DT>(a, (size_t)b * a.n + t, h * G + (r & (G - 1)), D, 16 * (quarter * NQ + j) + 4 * g, v, inv, gate[j]);
    }
}

template <int D, int DT>
hipError_t go(const PagedAttendArgs& a, int n_cu, void* ws, hipStream_t s) {
    constexpr int NT = ch_nt(D, DT == 1);
    using C = ChCfg<D, DT, NT>;
    const int groups = n_cu & ~7, tok = C::ROWS / (a.NH / a.NKV);
    const int64_t pairs = (int64_t)a.n_seq * ((a.n + tok - 1) / tok), items = pairs * a.NKV;
    // Few items: every workgroup finds its part by itself, and a second launch joins them many workgroups at a time. Measured on 61
    // fp32 tokens behind 16384 (16 heads of 256, 8 items) 51 us, with the plan and the last wave to arrive as the joiner 94 (bf16 55
    // and 208); 1000 bf16 tokens from the first on (64 items) 58 and 67; 2048 bf16 of 8 + 8 heads of 64 behind 2048 58 and 61. With more
    // items equal parts are too uneven: 2048 behind 2048 (128 items) 188 and 165.
    const bool joined = items * 4 <= groups && pairs <= kJoinPairs;
    hipError_t e = hipSuccess;
    if (!joined) {
        if (pairs <= 256) hipLaunchKernelGGL((k_paged_plan<256>), dim3(1), dim3(256), 0, s, a, ws, groups, C::PART, tok);
        else hipLaunchKernelGGL((k_paged_plan<1024>), dim3(1), dim3(1024), 0, s, a, ws, groups, C::PART, tok);
        if ((e = hipGetLastError()) != hipSuccess) return e;
    }
    auto kern = k_paged_chunk<D, DT, NT>;
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kern, dim3(groups), dim3(64 * kChWaves), C::LDS, s, a, ws, joined);
    if ((e = hipGetLastError()) != hipSuccess || !joined) return e;
    hipLaunchKernelGGL((k_paged_join_chunk<D, DT, NT>), dim3((unsigned)(items * kChWaves * NT * 4)), dim3(256), 0, s, a, ws, groups);
    return hipGetLastError();
}

}  // namespace

size_t paged_chunk_workspace(int D, int n_cu) {
    const size_t part = (size_t)kChWaves * (32 * D + 256) * sizeof(float);
    return up256(2 * n_cu * part + n_cu * (sizeof(int4) + kChWaves * 2 * sizeof(int)) + (1 + n_cu) * sizeof(int64_t) +
                 (1 + 2 * kJoinPairs) * sizeof(int));
}

hipError_t launch_paged_chunk(const PagedAttendArgs& a, int D, bool bf16, int n_cu, void* ws, hipStream_t s) {
    if (n_cu < 8) return hipErrorInvalidValue;
    if (D == 256) return bf16 ? go<256, 1>(a, n_cu, ws, s) : go<256, 0>(a, n_cu, ws, s);
    if (D == 128) return bf16 ? go<128, 1>(a, n_cu, ws, s) : go<128, 0>(a, n_cu, ws, s);
    return bf16 ? go<64, 1>(a, n_cu, ws, s) : go<64, 0>(a, n_cu, ws, s);
}

}  // namespace qw

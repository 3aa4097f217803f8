// Attention of a few new tokens a sequence (decode, speculative verify) over a paged cache: up to 32 query rows a KV head.
#include "paged.hpp"

namespace qw {

namespace {

constexpr int kFewWaves = 4;                     // waves of a workgroup; each takes every fourth block of 32 keys
constexpr int kFewUnit = kFewWaves;              // blocks of a unit of the schedule
constexpr int few_occ(int D) { return D == 256 ? 1 : 2; }  // workgroups a CU

// Workspace: [0] units a KV head, [1] units a workgroup, then every sequence's first unit; then the partial rows of
// two segments a workgroup (its first and its last), [slot][row][D] and [slot][row] (maximum, sum).
constexpr int kFewHead = 4;  // ints before the sequences' first units

struct FewPlan {
    int* head;
    float *o, *ml;
};
__host__ __device__ inline FewPlan few_plan(void* ws, int n_seq, int groups, int rows, int D) {
    (void)n_seq;
    char* p = static_cast<char*>(ws);
    FewPlan f;
    f.o = reinterpret_cast<float*>(p);
    f.ml = f.o + (size_t)2 * groups * rows * D;
    f.head = reinterpret_cast<int*>(f.ml + (size_t)2 * groups * rows * 2);
    return f;
}

template <int D, int DT, int NT>
struct FewCfg {
    static constexpr int PARTS = DT == 0 ? 2 : 1, NKS = D / 32, NDT = D / 16, ROWS = 16 * NT, BLKE = kBlk * D;
    static constexpr int Q_BYTES = PARTS * NT * NKS * 1024, KV_BYTES = kFewWaves * 2 * BLKE * 2;
    // score factors [ROWS] and eight words of the schedule. Where queries and blocks fill the LDS, the first wave's values
    // make room for them until the rows are laid out.
    static constexpr int EXTRA = ROWS * 4 + 32;
    static constexpr bool TIGHT = Q_BYTES + KV_BYTES + EXTRA > 160 * 1024;
    static constexpr int LDS = Q_BYTES + KV_BYTES + (TIGHT ? 0 : EXTRA);
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
__global__ __launch_bounds__(64 * kFewWaves, few_occ(D)) void k_paged_few(PagedAttendArgs a, void* ws) {
    using C = FewCfg<D, DT, NT>;
    constexpr int PARTS = C::PARTS, NKS = C::NKS, NDT = C::NDT, ROWS = C::ROWS, BLKE = C::BLKE;
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    f16* sq = reinterpret_cast<f16*>(smem);                              // query operands
    f16* kv = reinterpret_cast<f16*>(smem + C::Q_BYTES);                 // each wave's block of keys and of values
    float* red = reinterpret_cast<float*>(kv);                           // afterwards the waves' accumulators
    float* sm = reinterpret_cast<float*>(sq);                            // afterwards [waves][ROWS] maxima
    float* sl = sm + kFewWaves * ROWS;                                   // and sums
    float* sc = reinterpret_cast<float*>(C::TIGHT ? reinterpret_cast<unsigned char*>(kv + BLKE) : smem + C::Q_BYTES + C::KV_BYTES);
    int* si = reinterpret_cast<int*>(sc + ROWS);                         // scan and schedule
    const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int G = a.NH / a.NKV, groups = gridDim.x;
    const FewPlan plan = few_plan(ws, a.n_seq, groups, ROWS, D);

    // ---- schedule: a sequence is ceil(blocks / 4) units a KV head, the units of KV head 0's sequences come first, and
    // every workgroup takes an equal run of them. A thread sums a run of sequences, a scan places the runs.
    const int per = (a.n_seq + 64 * kFewWaves - 1) / (64 * kFewWaves);
    auto units = [&](int b) { return (key_tiles<5>(a, seq_pos(a.pos, b), 0, seq_len(a.lens, b, a.n)).count + kFewUnit - 1) / kFewUnit; };
    int mine = 0;
    for (int i = 0; i < per; i++)
        if (tid * per + i < a.n_seq) mine += units(tid * per + i);
    int incl = mine;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const int o = __shfl_up(incl, m, 64);
        if (lane >= m) incl += o;
    }
    if (lane == 63) si[wave] = incl;
    __syncthreads();
    int before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kFewWaves; w++) before += w < wave ? si[w] : 0, total += si[w];
    const int64_t all = (int64_t)total * a.NKV;
    const int run = max(1, (int)((all + groups - 1) / groups));
    const int64_t my0 = (int64_t)blockIdx.x * run;
    if (blockIdx.x == 0) {  // for the kernel that joins split sequences
        int at = before + incl - mine;
        for (int i = 0; i < per; i++)
            if (tid * per + i < a.n_seq) plan.head[kFewHead + tid * per + i] = at, at += units(tid * per + i);
        if (tid == 0) plan.head[0] = total, plan.head[1] = run;
    }
    if (my0 >= all) return;
    int h = (int)(my0 / total), rest = (int)(my0 - (int64_t)h * total);
    if (rest >= before + incl - mine && rest < before + incl) {  // one thread's
        int at = before + incl - mine, i = 0;
        for (;; i++) {
            const int u = units(tid * per + i);
            if (rest < at + u) break;
            at += u;
        }
        si[kFewWaves] = tid * per + i, si[kFewWaves + 1] = rest - at;
    }
    __syncthreads();
    int b = __builtin_amdgcn_readfirstlane(si[kFewWaves]), u0 = __builtin_amdgcn_readfirstlane(si[kFewWaves + 1]);
    h = __builtin_amdgcn_readfirstlane(h);
    int left = (int)min((int64_t)run, all - my0);

    for (bool first_seg = true; left > 0; first_seg = false) {
        const int pos = seq_pos(a.pos, b), len = seq_len(a.lens, b, a.n);
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
        if (!first_seg) __syncthreads();  // the last segment's readers of the LDS are done
        load(0, a.c.k, sk);
        if constexpr (!C::TIGHT) load(0, a.c.v, sv);

        // ---- the rows' operands: 256 / ROWS threads a row, pieces of 8 dims ----
        {
            constexpr int TPR = 64 * kFewWaves / ROWS, PIECES = D / 8;
            constexpr int PPT = (PIECES + TPR - 1) / TPR;
            const int r = tid / TPR, tl = tid % TPR, t = r / G;
            const bool ok = t < len;
            const size_t off = ((size_t)b * a.n + (ok ? t : 0)) * a.q_stride + (size_t)(h * G + r % G) * a.q_head;
            float x[PPT][8], largest = 0.f;
#pragma unroll
            for (int i = 0; i < PPT; i++) {
                const int pc = tl + i * TPR;
                if (pc < PIECES && ok) {
                    load_vec<DT, 8>(a.q, off + 8 * pc, x[i]);
                } else {
#pragma unroll
                    for (int j = 0; j < 8; j++) x[i][j] = 0.f;
                }
#pragma unroll
                for (int j = 0; j < 8; j++) largest = fmaxf(largest, fabsf(x[i][j]));
            }
#pragma unroll
            for (int m = 1; m < TPR; m <<= 1) largest = fmaxf(largest, __shfl_xor(largest, m, 64));
            const int sh = query_shift(largest);
            const float up = power_of_two(sh);
            if (tl == 0) sc[r] = a.scale * power_of_two(-sh);
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
                f16* dst = sq + (((r >> 4) * NKS + (pc >> 2)) * 64 + (pc & 3) * 16 + (r & 15)) * 8;
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
            const int t = (nt * 16 + col) / G;
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
            f16x8 w[NT][PARTS];
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
                    weight_parts<PARTS>(w0, w1, hi, lo);
                    w[nt][0][i] = hi[0], w[nt][0][i + 1] = hi[1];
                    if constexpr (PARTS == 2) w[nt][1][i] = lo[0], w[nt][1][i + 1] = lo[1], l_run[nt] += w0 + w1;
                    else l_run[nt] = __builtin_amdgcn_fdot2(hi, f16x2{(f16)1.f, (f16)1.f}, l_run[nt], false);
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
                        for (int part = 0; part < PARTS; part++) acc[nt][dt] = mfma16(v, w[nt][part], acc[nt][dt]);
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
                            for (int part = 0; part < PARTS; part++) acc[nt][dt] = mfma16(v, w[nt][part], acc[nt][dt]);
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
                                for (int part = 0; part < PARTS; part++) o = mfma16(v, w[nt][part], o);
                                const bool own = (nt * 16 + col) / G == t;
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

        // ---- the waves' outputs against their common maximum, added through the blocks' room ----
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
        }
        __syncthreads();
        auto row_max = [&](int r) {
            float m = sm[r];
#pragma unroll
            for (int w = 1; w < kFewWaves; w++) m = fmaxf(m, sm[w * ROWS + r]);
            return m;
        };
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const float corr = m_run[nt] == kNegInf ? 0.f : exp2_fast(m_run[nt] - row_max(nt * 16 + col));
#pragma unroll
            for (int dt = 0; dt < NDT; dt++)
                *reinterpret_cast<f32x4*>(red + (((wave * NT + nt) * NDT + dt) * 64 + lane) * 4) = acc[nt][dt] * corr;
        }
        __syncthreads();
        const int slot = 2 * blockIdx.x + (u0 == 0 ? 1 : 0);
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const int r = nt * 16 + col, t = r / G;
            if (t >= len) continue;
            const float m = row_max(r);
            float l = 0.f;
#pragma unroll
            for (int w = 0; w < kFewWaves; w++)
                l += sl[w * ROWS + r] * (sm[w * ROWS + r] == kNegInf ? 0.f : exp2_fast(sm[w * ROWS + r] - m));
            const float inv = inverse_sum(l);
            constexpr int PER = (NDT + kFewWaves - 1) / kFewWaves;  // dim tiles a wave
            Gate4<DT> gate[PER];
#pragma unroll
            for (int k = 0; k < PER; k++) gate[k].none();
            if (!split && a.gate) {
#pragma unroll
                for (int k = 0; k < PER; k++)
                    gate[k].load(a, (size_t)b * a.n + t, h * G + r % G, 16 * (wave + k * kFewWaves) + 4 * g);
            }
            if (split && wave == 0 && g == 0) *reinterpret_cast<f32x2*>(plan.ml + ((size_t)slot * ROWS + r) * 2) = f32x2{m, l};
#pragma unroll
            for (int k = 0; k < PER; k++) {
                const int dt = wave + k * kFewWaves;
                f32x4 o{};
#pragma unroll
                for (int w = 0; w < kFewWaves; w++) o += *reinterpret_cast<const f32x4*>(red + (((w * NT + nt) * NDT + dt) * 64 + lane) * 4);
                if (split) *reinterpret_cast<f32x4*>(plan.o + ((size_t)slot * ROWS + r) * D + 16 * dt + 4 * g) = o;
                else store_out4<DT>(a, (size_t)b * a.n + t, h * G + r % G, D, 16 * dt + 4 * g, o, inv, gate[k]);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        left -= u1 - u0;
        u0 = u1;
    }
}

// Joins the parts of split sequences: a workgroup a (sequence, token, head). Its first part is the last segment of one
// workgroup of k_paged_few, the others the first segments of those after it. Fixed order.
template <int D, int DT, int ROWS>
__global__ __launch_bounds__(256) void k_paged_join(PagedAttendArgs a, void* ws, int groups) {
    constexpr int LANES = D / 4, SETS = 256 / LANES;  // LANES threads x 4 dims a part, SETS parts at a time
    __shared__ float red[SETS][D];
    __shared__ float sw[64], sr[8];
    const FewPlan plan = few_plan(ws, a.n_seq, groups, ROWS, D);
    const int head = blockIdx.x % a.NH, row = blockIdx.x / a.NH, b = row / a.n, t = row - b * a.n;
    const int len = seq_len(a.lens, b, a.n);
    if (t >= len) return;
    const int G = a.NH / a.NKV, h = head / G, r = t * G + head % G;
    const int total = plan.head[0], run = plan.head[1];
    const int nu = (key_tiles<5>(a, seq_pos(a.pos, b), 0, len).count + kFewUnit - 1) / kFewUnit;
    const int64_t at = (int64_t)h * total + plan.head[kFewHead + b];
    const int first = (int)(at / run), last = (int)((at + nu - 1) / run), parts = last - first + 1;
    if (parts == 1) return;
    const int tid = threadIdx.x;
    Gate4<DT> gate;
    gate.none();
    if (a.gate) gate.load(a, (size_t)row, head, 4 * (tid % LANES));
    auto slot = [&](int part) { return (size_t)(part == 0 ? 2 * first + 1 : 2 * (first + part)) * ROWS + r; };
    // maximum, then sums and outputs of 64 parts at a time against it
    float m = kNegInf;
    for (int p = tid; p < parts; p += 256) m = fmaxf(m, plan.ml[slot(p) * 2]);
    m = max64(m);
    if ((tid & 63) == 0) sr[tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(sr[0], sr[1]), fmaxf(sr[2], sr[3]));
    f32x4 o{};
    float l = 0.f;
    for (int p0 = 0; p0 < parts; p0 += 64) {
        if (tid < 64) {
            float w = 0.f, lw = 0.f;
            if (p0 + tid < parts) {
                const f32x2 v = *reinterpret_cast<const f32x2*>(plan.ml + slot(p0 + tid) * 2);
                w = v[0] == kNegInf ? 0.f : exp2_fast(v[0] - m), lw = v[1] * w;
            }
            sw[tid] = w;
            l += sum64(lw);
        }
        __syncthreads();
#pragma unroll 8
        for (int p = p0 + tid / LANES; p < min(parts, p0 + 64); p += SETS) {
            const f32x4 x = *reinterpret_cast<const f32x4*>(plan.o + slot(p) * D + 4 * (tid % LANES));
#pragma unroll
            for (int i = 0; i < 4; i++) o[i] = __builtin_fmaf(x[i], sw[p - p0], o[i]);
        }
        __syncthreads();
    }
    if (tid == 0) sr[4] = l;
    *reinterpret_cast<f32x4*>(&red[tid / LANES][4 * (tid % LANES)]) = o;
    __syncthreads();
    if (tid < LANES) {
#pragma unroll
        for (int s = 1; s < SETS; s++) o += *reinterpret_cast<const f32x4*>(&red[s][4 * tid]);
        store_out4<DT>(a, (size_t)row, head, D, 4 * tid, o, inverse_sum(sr[4]), gate);
    }
}

template <int D, int DT, int NT>
hipError_t go(const PagedAttendArgs& a, int n_cu, void* ws, hipStream_t s) {
    using C = FewCfg<D, DT, NT>;
    constexpr int ROWS = C::ROWS;
    const int groups = n_cu * few_occ(D);
    constexpr int shm = C::LDS;
    auto kern = k_paged_few<D, DT, NT>;
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, shm);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(kern, dim3(groups), dim3(64 * kFewWaves), shm, s, a, ws);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    hipLaunchKernelGGL((k_paged_join<D, DT, ROWS>), dim3((unsigned)(a.n_seq * a.n * a.NH)), dim3(256), 0, s, a, ws, groups);
    return hipGetLastError();
}

template <int D>
hipError_t go_d(const PagedAttendArgs& a, bool bf16, int n_cu, void* ws, hipStream_t s) {
    const bool two = a.n * (a.NH / a.NKV) > 16;
    if (bf16) return two ? go<D, 1, 2>(a, n_cu, ws, s) : go<D, 1, 1>(a, n_cu, ws, s);
    return two ? go<D, 0, 2>(a, n_cu, ws, s) : go<D, 0, 1>(a, n_cu, ws, s);
}

}  // namespace

size_t paged_few_workspace(int D, int n_cu) {
    const size_t rows = (size_t)2 * n_cu * few_occ(D) * 32;
    return up256(rows * (D + 2) * sizeof(float) + (kFewHead + 65536) * sizeof(int));
}

hipError_t launch_paged_few(const PagedAttendArgs& a, int D, bool bf16, int n_cu, void* ws, hipStream_t s) {
    if (D == 256) return go_d<256>(a, bf16, n_cu, ws, s);
    if (D == 128) return go_d<128>(a, bf16, n_cu, ws, s);
    return go_d<64>(a, bf16, n_cu, ws, s);
}

}  // namespace qw

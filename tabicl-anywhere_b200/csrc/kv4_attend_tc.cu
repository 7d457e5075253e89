// Attention of many f32 query rows over the four-bit cache on the 5th-generation tensor cores (tcgen05).
//
// 128 query rows of one cache head (the heads that share it side by side) against 64 keys at a time: S = Q K^T with Q in
// tensor memory and the keys, widened to f16, in shared memory; the weights P go back to tensor memory over S and multiply
// the widened values; each step's P V is folded into the output in registers, so every sum across steps is taken in f32
// with rounding to nearest (the matrix unit's own accumulation is not: over 10,000 keys it would cost f32 results their
// last bits). Each f32 operand is the sum of two f16 (22 bits), and a product is hi hi + hi lo + lo hi.
//
// A step's keys and values are scaled by a power of two of their own that keeps them inside f16, whatever the cache holds.
// Coordinates keep the order the codes are unpacked in, (0, 4, 1, 5, 2, 6, 3, 7) of every eight: Q takes the same order,
// and the output's columns are put back when they are written.
//
// What bounds it: the instructions that widen a step into two f16 a value and take its softmax, in the same issue slots as
// the fold; three products a step keep the matrix unit busy for about a third of the time. Widening by two warpgroups in
// turn took 2048 rows over 10,000 keys (4 heads of 128) from 0.28 to 0.19 ms, loops short enough for the instruction caches
// to 0.17 ms: 0.24 PFLOP/s of scores and sums, 0.73 of products.
#include <algorithm>

#include "kv4_tc.cuh"

namespace tcu {

constexpr int KT_BQ = 128, KT_BK = 64, KT_NS = 3, KT_THREADS = 640;
constexpr uint32_t KT_TQ = 0, KT_TS = 128, KT_TO = 384;

template <int HD, int G>
struct KtShape {
    static constexpr int NU = HD / 32, NG = HD / G, QS = 2;  // f16 an operand is the sum of
    static constexpr int BLOCK = KT_BK * HD;                            // f16 of one operand block
    static constexpr int KC = KT_BK * HD / 2, SC = KT_BK * NG * 4, RAW = 2 * (KC + SC);
    static constexpr int NR = 2;                   // slots of stored codes: what shared memory leaves
    static constexpr int T = 13;                   // widened values are below 2^T
    static constexpr size_t SMEM = (size_t)2 * KT_NS * QS * BLOCK * 2 + (size_t)NR * RAW + 1024;
};

// Warps 0-3: softmax, a thread a query row; warps 4-7: the fold of each step's P V, a thread a row; warps 8-11, 12-15:
// widening of even and odd steps; warps 16, 17 issue the S products of even and odd steps, warp 18 the P V products; warp 19:
// the copies of the stored codes. They hand over through mbarriers; every wait is bounded, and one that gives up raises the
// block's abort flag, after which every wait returns at once and the roles run to the end without results.
template <int HD, int G>
__global__ void __launch_bounds__(KT_THREADS, 1) k_kv4_attend_tc(Kv4AttendArgs a, int dtype, float *part, int *arrived) {
    using C = KtShape<HD, G>;
    using Cut = KaCut<KT_BQ, KT_BK, KT_BK>;
    constexpr int NU = C::NU, NG = C::NG, UG = G / 32, QS = C::QS, BQ = KT_BQ, BK = KT_BK, NS = KT_NS, NR = C::NR, BLOCK = C::BLOCK;
    extern __shared__ __align__(1024) uint8_t smraw[];
    __half *Kring = reinterpret_cast<__half *>(smraw);                // [NS][QS][64 x HD], K-major
    __half *Vring = Kring + NS * QS * BLOCK;                          // [NS][QS][64 x HD], coordinate-major
    uint8_t *raw = reinterpret_cast<uint8_t *>(Vring + NS * QS * BLOCK);  // [NR]{key codes, key scales, value codes, value scales}
    __shared__ float fr[4][BQ], rowx[2][BQ], qmax[2][BQ], red[2][2][2][4];  // red: [turn][step][keys, values][warp]
    __shared__ int teK[8], teV[8], has_nan[8];
    __shared__ uint32_t nan_keys[8][NG][2];
    __shared__ __align__(8) uint64_t mK[NS], mV[NS], mKfree[NS], mVfree[NS], mS[NS], mP[NS], mSlot[NS], mF[4], mPV, mOfree, mDone[3],
        mRaw[NR], mRawFree[NR];
    __shared__ uint32_t tslot;
    __shared__ volatile int abort_flag;
    __shared__ int s_unit[4], s_last;
    __shared__ long long s_sum[KT_THREADS / 32];

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wg = warp >> 2, row = tid & (BQ - 1);
    const int each = a.q_heads / a.c.heads;
    auto pl = Cut::template place<KT_THREADS>(a, each, KA_TC_STEPS, s_sum, s_unit);
    if (pl.pos >= pl.end) return;
    if (warp == 0) {
        tmem_alloc(&tslot, 512);
        tmem_relinquish();
    }
    if (tid == 0) {
        for (int i = 0; i < NS; i++) {
            mbar_init(&mK[i], 128), mbar_init(&mV[i], 128), mbar_init(&mKfree[i], 1), mbar_init(&mVfree[i], 1);
            mbar_init(&mS[i], 1), mbar_init(&mP[i], BQ), mbar_init(&mSlot[i], 1);
        }
        for (int i = 0; i < NR; i++) mbar_init(&mRaw[i], 1), mbar_init(&mRawFree[i], 128);
        for (int i = 0; i < 4; i++) mbar_init(&mF[i], BQ);
        mbar_init(&mPV, 1), mbar_init(&mOfree, BQ);
        for (int i = 0; i < 3; i++) mbar_init(&mDone[i], 1);
        mbar_init_fence();
        abort_flag = 0;
    }
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = tslot, lane_base = (uint32_t)((warp & 3) * 32) << 16;

    auto wait_warp = [&](uint64_t *m, uint32_t parity) {  // warp-uniform: warp-wide instructions follow
        bool ok = mbar_test_wait(m, parity) || (!abort_flag && mbar_wait(m, parity, KT_WAIT));
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) abort_flag = 1;
        return ok;
    };
    // Q of a piece: each of two threads (softmax and fold) half a row, scaled by a power of two of the row's to at most 2^14,
    // into tensor memory. Returns what a product with the widened keys is multiplied by (with the step's power of two) to be a
    // score in units of log2.
    auto put_q = [&](const KaRows &sr, int ri, int hq) {
        constexpr int H = HD / 2;
        float q[H / 8][8], mx = 0.f;
        const int es = dtype == DT_F32 ? 4 : 2;
        const bool wide = !(((uintptr_t)a.q & 15) || ((a.q_row | a.q_head) * es) % 16);
        const long long from = (long long)(sr.first + ri) * a.q_row + (long long)hq * a.q_head + wg * H;
        load_runs<H / 8>(dtype, a.q, from, 8, wide, q);
#pragma unroll
        for (int b = 0; b < H / 8; b++)
#pragma unroll
            for (int x = 0; x < 8; x++) mx = fmaxf(mx, fabsf(q[b][x]));
        kt_bar(2, 256);  // the last piece's epilogue is done with the exchange
        qmax[wg][row] = mx;
        kt_bar(2, 256);
        mx = fmaxf(qmax[0][row], qmax[1][row]);
        const int e = mx > 0.f ? min(126, 140 - (int)((__float_as_uint(mx) >> 23) & 0xff)) : 0;
        const float up = a.scale < 0.f ? -kt_pow2(e) : kt_pow2(e);
        // a score in units of log2: the product with the widened keys times this and the step's power of two
        const float rowfac = fabsf(a.scale) * 1.44269504088896340736f * kt_pow2(-e);
        uint32_t hi[H / 2], lo[H / 2];
#pragma unroll
        for (int b = 0; b < H / 8; b++)
#pragma unroll
            for (int x = 0; x < 4; x++)
                split_pair(q[b][x] * up, q[b][x + 4] * up, hi[4 * b + x], lo[4 * b + x]);
        const uint32_t tq = tmem + lane_base + KT_TQ + wg * (H / 2);
        if constexpr (H / 2 == 32) {
            tmem_st32u(tq, hi);
            tmem_st32u(tq + HD / 2, lo);
        } else {
#pragma unroll
            for (int c = 0; c < H / 2; c++) {
                tmem_st1(tq + c, __uint_as_float(hi[c]));
                tmem_st1(tq + HD / 2 + c, __uint_as_float(lo[c]));
            }
        }
        tmem_wait_st();
        fence_before_sync();
        kt_bar(1, 352);
        fence_after_sync();
        return rowfac;
    };
    // the pieces of units that are this block's, in every role alike: n steps from key j0 on, `at` steps before them
    int at = 0;

    if (wg == 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
        if (warp == 19) {
            // ---- copies: lane part + 4 * piece brings one of the four arrays of one page's share of the 64 keys ----
            const Kv4Offsets off = kv4_offsets(HD, a.c.page, G);
            const size_t hb = kv4_head_bytes(HD, a.c.page, G);
            const int page = a.c.page, shift = 31 - __clz(page), keys = min(page, BK), pieces = BK / keys;
            const int cpart = lane & 3, cp = lane >> 2;
            const uint32_t per_key = cpart & 1 ? NG * 4 : HD / 2, bytes = per_key * keys;
            const uint32_t from = (cpart & 2 ? off.vc : 0) + (cpart & 1 ? off.ks : 0);
            const uint32_t to = (cpart & 2 ? C::KC + C::SC : 0) + (cpart & 1 ? C::KC : 0) + cp * bytes;
            while (pl.pos < pl.end) {
                const KaRows sr = ka_rows(a, pl.seq);
                const auto sp = Cut::span(a, sr, each, pl.rt);
                const int n = (int)min((long long)(sp.steps - pl.skip), pl.end - pl.pos), j0 = sp.base + pl.skip * BK;
                auto there = [&](int i) {
                    const int j = j0 + i * BK + cp * keys;
                    return i < n && cp < pieces && j < sp.hi_max && j + keys > sp.lo_min;
                };
                auto find = [&](int i) { return there(i) ? a.table[pl.seq * a.table_stride + ((j0 + i * BK + cp * keys) >> shift)] : -1; };
                int next = find(0), after = find(1);  // a page's number is read two steps before it is needed
                for (int i = 0; i < n; i++, at++) {
                    const int j = j0 + i * BK + cp * keys, slot = at % NR, pg = next;
                    next = after, after = find(i + 2);
                    const bool ok = pg >= 0 && pg < a.c.pages;
                    if (there(i) && !ok) *reinterpret_cast<volatile int *>(a.err) = 1;
                    const unsigned mask = __ballot_sync(0xffffffffu, ok && cpart == 0);
                    if (at >= NR && !wait_warp(&mRawFree[slot], (uint32_t)(at / NR - 1) & 1u)) break;
                    if (lane == 0)
                        asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}\n" ::"r"(smem_addr(&mRaw[slot])),
                                     "r"((uint32_t)(__popc(mask) * (C::RAW / pieces)))
                                     : "memory");
                    if (ok)
                        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                                         smem_addr(raw + slot * C::RAW + to)),
                                     "l"(a.c.pool + ((size_t)pg * a.c.heads + pl.head) * hb + from + (j & (page - 1)) * per_key), "r"(bytes),
                                     "r"(smem_addr(&mRaw[slot]))
                                     : "memory");
                }
                Cut::next(pl, a, each, sr.n, n);
            }
            // what was asked for lands before the block lets go of shared memory
            for (int i = max(0, at - NR); i < at; i++) mbar_wait(&mRaw[i % NR], (uint32_t)(i / NR) & 1u, KT_WAIT);
        } else {
            // ---- the products ----
            const uint32_t idS = idesc_f16(BQ, BK, 0, 0), idO = idesc_f16(BQ, HD, 0, 1);
            const uint64_t dK0 = kstep_desc(Kring, BK, 0), dV0 = kstep_desc(Vring, HD, 0);
            const uint64_t stK = (2 * (BK / 8) * 128) >> 4, stV = (2 * (HD / 8) * 128) >> 4;
            const uint64_t lo_off = (BLOCK * 2) >> 4, slot_off = (QS * BLOCK * 2) >> 4;
            while (pl.pos < pl.end) {
                const KaRows sr = ka_rows(a, pl.seq);
                const auto sp = Cut::span(a, sr, each, pl.rt);
                const int n = (int)min((long long)(sp.steps - pl.skip), pl.end - pl.pos);
                kt_bar(1, 352);  // Q is in tensor memory
                fence_after_sync();
                for (int i = at; i < at + n; i++) {
                    const int sl = i % NS;
                    const uint32_t ph = (uint32_t)(i / NS) & 1u;
                    if (warp < 18) {
                        if ((i & 1) != warp - 16) continue;
                        // S(i) once P V(i - NS) has read its slot, from the keys of step i
                        if (i >= NS) wait_warp(&mSlot[sl], ph ^ 1u);
                        wait_warp(&mK[sl], ph);
                        fence_after_sync();
                        const uint32_t tS = tmem + KT_TS + BK * sl;
                        const uint64_t dh = dK0 + sl * slot_off, dl = dh + lo_off;
                        if (elect_one()) {
#pragma unroll
                            for (int k = 0; k < HD / 16; k++) mma_f16_ta(tS, tmem + KT_TQ + 8 * k, dl + k * stK, idS, k > 0 ? 1u : 0u);
#pragma unroll
                            for (int k = 0; k < HD / 16; k++) mma_f16_ta(tS, tmem + KT_TQ + HD / 2 + 8 * k, dh + k * stK, idS, 1);
#pragma unroll
                            for (int k = 0; k < HD / 16; k++) mma_f16_ta(tS, tmem + KT_TQ + 8 * k, dh + k * stK, idS, 1);
                            mma_commit(&mS[sl]);
                            mma_commit(&mKfree[sl]);
                        }
                        __syncwarp();
                    } else {
                        // P V of step i: its weights and values there, the fold of step i - 1 done
                        wait_warp(&mP[sl], ph);
                        wait_warp(&mV[sl], ph);
                        if (i >= 1) wait_warp(&mOfree, (uint32_t)(i - 1) & 1u);
                        fence_after_sync();
                        const uint32_t pA = tmem + KT_TS + BK * sl, tO = tmem + KT_TO;
                        const uint64_t dh = dV0 + sl * slot_off, dl = dh + lo_off;
                        if (elect_one()) {
#pragma unroll
                            for (int k = 0; k < BK / 16; k++) mma_f16_ta(tO, pA + 16 * k, dl + k * stV, idO, k > 0 ? 1u : 0u);
#pragma unroll
                            for (int k = 0; k < BK / 16; k++) mma_f16_ta(tO, pA + 16 * k + 8, dh + k * stV, idO, 1);
#pragma unroll
                            for (int k = 0; k < BK / 16; k++) mma_f16_ta(tO, pA + 16 * k, dh + k * stV, idO, 1);
                            mma_commit(&mPV);
                            mma_commit(&mVfree[sl]);
                            mma_commit(&mSlot[sl]);
                        }
                        __syncwarp();
                    }
                }
                __syncwarp();
                at += n;
                Cut::next(pl, a, each, sr.n, n);
            }
            if (elect_one()) {  // every product issued here completes before the block lets go of its memory
                mma_commit(&mDone[warp - 16]);
                mbar_wait(&mDone[warp - 16], 0, KT_WAIT);
            }
        }
    } else if (wg >= 2) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        // ---- widening: a thread half a key's coordinates and half a value's, of every other step ----
        // (a wait that gave up does not end the loop: the four warps meet at a barrier in every step)
        const int key = tid & 63, half = (tid >> 6) & 1, w4 = warp & 3, turn = wg - 2;
        while (pl.pos < pl.end) {
            const KaRows sr = ka_rows(a, pl.seq);
            const auto sp = Cut::span(a, sr, each, pl.rt);
            const int n = (int)min((long long)(sp.steps - pl.skip), pl.end - pl.pos), j0 = sp.base + pl.skip * BK;
            for (int i = at + ((at ^ turn) & 1); i < at + n; i += 2) {
                const int sl = i % NS, rs = i % NR, j = j0 + (i - at) * BK + key;
                const uint32_t ph = (uint32_t)(i / NS) & 1u;
                wait_warp(&mRaw[rs], (uint32_t)(i / NR) & 1u);
                const uint8_t *kraw = raw + rs * C::RAW, *vraw = kraw + C::KC + C::SC;
                const bool seen = j >= sp.lo_min && j < sp.hi_max;
                uint32_t kc[NG], vc[NG];  // the key's scales
                lds_words<NG>(kraw + C::KC + key * NG * 4, kc);
                lds_words<NG>(vraw + C::KC + key * NG * 4, vc);
                // the step's power of two, for keys and values: from each group's ends
                float mx[2] = {0.f, 0.f};
                bool nan = false;
#pragma unroll
                for (int k = 0; k < NG; k++) {
                    if (!seen) kc[k] = vc[k] = 0;
                    const float2 ks = __half22float2(kt_h2(kc[k])), vs = __half22float2(kt_h2(vc[k]));
                    mx[0] = fmaxf(mx[0], fmaxf(fabsf(ks.y), fabsf(fmaf(15.f, ks.x, ks.y))));
                    mx[1] = fmaxf(mx[1], fmaxf(fabsf(vs.y), fabsf(fmaf(15.f, vs.x, vs.y))));
                    nan |= vs.y != vs.y;
                }
                // a group of values that stands for NaN is left out here and put into the rows that see it by the fold
                nan = __any_sync(0xffffffffu, nan);
                if (nan) {
#pragma unroll
                    for (int k = 0; k < NG; k++) {
                        const bool bad = (vc[k] & 0x7fff0000u) > 0x7c000000u;
                        const unsigned who = __ballot_sync(0xffffffffu, bad);
                        if (half == 0 && lane == 0) nan_keys[i & 7][k][w4] = who;
                        if (bad) vc[k] = 0;
                    }
                } else if (half == 0 && lane < NG) {
                    nan_keys[i & 7][lane][w4] = 0;
                }
                mx[0] = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mx[0])));  // (not negative: ordered as their bits)
                mx[1] = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mx[1])));
                if (lane == 0) red[turn][i >> 1 & 1][0][w4] = mx[0], red[turn][i >> 1 & 1][1][w4] = nan ? -mx[1] - 1.f : mx[1];  // a NaN shows as the sign
                kt_bar(3 + turn, 128);
                int e[2];
                bool any = false;
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    float m = 0.f;
#pragma unroll
                    for (int w = 0; w < 4; w++) {
                        const float r = red[turn][i >> 1 & 1][x][w];
                        any |= r < 0.f, m = fmaxf(m, r < 0.f ? -1.f - r : r);
                    }
                    e[x] = m > 0.f ? min(40, (int)(__float_as_uint(m) >> 23) - 125) : 0;  // m < 2^(e - 1): a span, 15 steps, below 2^e
                }
                if (tid % 128 == 0) teK[i & 7] = e[0], teV[i & 7] = e[1], has_nan[i & 7] = any;
                if (i >= NS) wait_warp(&mKfree[sl], ph ^ 1u);
                // (loops that are not unrolled over the halves: short code for the instruction caches, which all roles share)
#pragma unroll 1
                for (int x = 2 * half; x < 2 * half + 2; x++) {
                    uint32_t w[NU];
                    lds_words<NU>(kraw + key * (HD / 2) + x * NU * 4, w);
                    __half *hi = Kring + sl * QS * BLOCK + kmajor_off(key, 8 * x, BK), *lo = hi + BLOCK;
#pragma unroll
                    for (int u = 0; u < NU; u++) {
                        KtScale s;
                        const float2 f = __half22float2(kt_h2(kc[u / UG]));
                        s.set(f.x, f.y, kt_pow2(C::T - e[0]));
                        kt_widen(w[u], s, hi + kmajor_off(0, 32, BK) * u, lo + kmajor_off(0, 32, BK) * u);
                    }
                }
                fence_async_smem();
                mbar_arrive(&mK[sl]);
                if (i >= NS) wait_warp(&mVfree[sl], ph ^ 1u);
#pragma unroll 1
                for (int x = 2 * half; x < 2 * half + 2; x++) {
                    uint32_t w[NU];
                    lds_words<NU>(vraw + key * (HD / 2) + x * NU * 4, w);
                    __half *hi = Vring + sl * QS * BLOCK + mnmajor_off(8 * x, key, HD), *lo = hi + BLOCK;
#pragma unroll
                    for (int u = 0; u < NU; u++) {
                        // half-words g = 2 x and 2 x + 1 of a unit: coordinates 32 u + 8 x + (0..7)
                        uint32_t c;
                        if constexpr (NU == 1)
                            c = w[0];
                        else
                            c = __byte_perm(w[u / 2], w[NU / 2 + u / 2], u & 1 ? 0x7632 : 0x5410);
                        KtScale s;
                        const float2 f = __half22float2(kt_h2(vc[u / UG]));
                        s.set(f.x, f.y, kt_pow2(C::T - e[1]));
                        kt_widen(c, s, hi + mnmajor_off(32, 0, HD) * u, lo + mnmajor_off(32, 0, HD) * u);
                    }
                }
                fence_async_smem();
                mbar_arrive(&mV[sl]);
                mbar_arrive(&mRawFree[rs]);
            }
            at += n;
            Cut::next(pl, a, each, sr.n, n);
        }
    } else if (wg == 0) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 136;");
        while (pl.pos < pl.end) {
            const KaRows sr = ka_rows(a, pl.seq);
            const auto sp = Cut::span(a, sr, each, pl.rt);
            const int n = (int)min((long long)(sp.steps - pl.skip), pl.end - pl.pos), j0 = sp.base + pl.skip * BK;
            const int r0 = pl.rt * BQ, rows = min(BQ, sr.n * each - r0);
            const int r = min(row, rows - 1), ri = (r0 + r) / each, hq = pl.head * each + (r0 + r) % each;  // rows past the end repeat the last
            const int my_hi = ka_hi(a, sr, ri), my_lo = ka_lo(a, sr, ri);
            const float rowfac = put_q(sr, ri, hq);
            // ---- softmax: S(i) -> 2^14 P(i) = 2^(S - m + 14) over S(i), and the factor of what was before ----
            float mrun = -INFINITY, lrun = 0.f;
            for (int i = at; i < at + n; i++) {
                const int sl = i % NS, key0 = j0 + (i - at) * BK;
                if (!wait_warp(&mS[sl], (uint32_t)(i / NS) & 1u)) break;
                fence_after_sync();
                const uint32_t tsp = tmem + lane_base + KT_TS + BK * sl;
                // (held to the normal numbers: positive for a scale of 0 too, so that -infinity stays itself)
                const float c1 = fminf(fmaxf(rowfac * kt_pow2(*reinterpret_cast<volatile int *>(&teK[i & 7]) - C::T), FLT_MIN), FLT_MAX);
                // Two passes over the step's scores in tensor memory, 32 at a time in loops that are not unrolled further (short code
                // for the instruction caches, which all roles share). P goes where the scores were: of every 16 keys, hi and lo.
                const bool edge = key0 < sp.lo_max || key0 + BK > sp.hi_min;
                auto scores = [&](int b, float (&x)[32]) {
                    tmem_ld32(tsp + 32 * b, x);
                    tmem_wait_ld32(x);
                    if (edge) {
#pragma unroll
                        for (int k = 0; k < 32; k++)
                            if (key0 + 32 * b + k < my_lo || key0 + 32 * b + k >= my_hi) x[k] = -INFINITY;
                    }
                };
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
                for (int b = 0; b < 2; b++) {
                    float x[32];
                    scores(b, x);
#pragma unroll
                    for (int k = 0; k < 32; k++) top[k & 3] = fmaxf(top[k & 3], x[k]);
                }
                const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                const float mnew = fmaxf(mrun, mx * c1), mm = mnew == -INFINITY ? 0.f : mnew - 14.f;
                const float f = mrun == -INFINITY ? 0.f : kt_ex2(mrun - mnew);
                float psum[4] = {};
#pragma unroll 1
                for (int b = 0; b < 2; b++) {
                    float x[32];
                    scores(b, x);
                    uint32_t w[32];
#pragma unroll
                    for (int k = 0; k < 32; k++) {
                        x[k] = kt_ex2(fmaf(x[k], c1, -mm));
                        psum[k & 3] += x[k];
                    }
#pragma unroll
                    for (int k = 0; k < 16; k++) split_pair(x[2 * k], x[2 * k + 1], w[k / 8 * 16 + k % 8], w[k / 8 * 16 + 8 + k % 8]);
                    tmem_st32u(tsp + 32 * b, w);
                }
                tmem_wait_st();
                fr[i & 3][row] = f;
                fence_before_sync();
                mbar_arrive(&mP[sl]);
                mbar_arrive(&mF[i & 3]);
                lrun = fmaf(lrun, f, (psum[0] + psum[1]) + (psum[2] + psum[3]));
                mrun = mnew;
            }
            rowx[0][row] = mrun, rowx[1][row] = lrun * 6.103515625e-5f;  // 2^-14
            kt_bar(2, 256);
            at += n;
            Cut::next(pl, a, each, sr.n, n);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
        while (pl.pos < pl.end) {
            const KaRows sr = ka_rows(a, pl.seq);
            const auto sp = Cut::span(a, sr, each, pl.rt);
            const int n = (int)min((long long)(sp.steps - pl.skip), pl.end - pl.pos), j0 = sp.base + pl.skip * BK;
            const int r0 = pl.rt * BQ, rows = min(BQ, sr.n * each - r0);
            const int r = min(row, rows - 1), ri = (r0 + r) / each, hq = pl.head * each + (r0 + r) % each;  // rows past the end repeat the last
            const int my_hi = ka_hi(a, sr, ri), my_lo = ka_lo(a, sr, ri);
            put_q(sr, ri, hq);
            // ---- fold: O = O f + P V, in units of the step's power of two ----
            float o[HD];
            int unit = 0;
#pragma unroll
            for (int k = 0; k < HD; k++) o[k] = 0.f;
            for (int i = at; i < at + n; i++) {
                if (!wait_warp(&mPV, (uint32_t)i & 1u)) break;
                if (!wait_warp(&mF[i & 3], (uint32_t)(i >> 2) & 1u)) break;
                fence_after_sync();
                const int e = *reinterpret_cast<volatile int *>(&teV[i & 7]);
                const float f = fr[i & 3][row] * (i == at ? 1.f : kt_pow2(unit - e));
                unit = e;
#pragma unroll
                for (int c = 0; c < HD / 32; c++) {
                    float x[32];
                    tmem_ld32(tmem + lane_base + KT_TO + 32 * c, x);
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 32; k++) o[32 * c + k] = fmaf(o[32 * c + k], f, x[k]);
                }
                if (*reinterpret_cast<volatile int *>(&has_nan[i & 7])) {
                    const int key0 = j0 + (i - at) * BK;
#pragma unroll
                    for (int k = 0; k < NG; k++) {
                        bool hit = false;
                        for (int b = 0; b < 64; b++)
                            hit |= (nan_keys[i & 7][k][b >> 5] >> (b & 31) & 1) && key0 + b >= my_lo && key0 + b < my_hi;
                        if (hit)
#pragma unroll
                            for (int x = 0; x < G; x++) o[k * G + x] = NAN;
                    }
                }
                fence_before_sync();
                mbar_arrive(&mOfree);
            }
            kt_bar(2, 256);
            // ---- the row's output, or its part of it ----
            const bool whole = n == sp.steps;
            float M = rowx[0][row], L = rowx[1][row];
            const float un = kt_pow2(unit - C::T - 14);
#pragma unroll
            for (int k = 0; k < HD; k++) o[k] *= un;
            bool write = row < rows;
            if (!whole) {
                const int2 who = Cut::sharers(pl, pl.pos - pl.skip, sp.steps);
                float *po = part + 2 * (size_t)2 * gridDim.x * BQ;
                const size_t mine = Cut::slot(blockIdx.x, pl.skip == 0) * BQ + row;
                if (write) {
                    __stcg(reinterpret_cast<float2 *>(part) + mine, make_float2(M, L));
#pragma unroll
                    for (int k = 0; k < HD; k += 4)
                        __stcg(reinterpret_cast<float4 *>(po + mine * HD + k), make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]));
                }
                __threadfence();
                kt_bar(5, 128);
                if (row == 0) {
                    s_last = atomicAdd(arrived + who.x, 1) == who.y - 1;
                    if (s_last) arrived[who.x] = 0;  // ready for the next call
                }
                kt_bar(5, 128);
                write = write && s_last;
                if (write) {
                    __threadfence();
                    M = -INFINITY, L = 0.f;
                    for (int p = 0; p < who.y; p++)
                        M = fmaxf(M, __ldcg(reinterpret_cast<const float2 *>(part) + Cut::slot(who.x + p, p == 0) * BQ + row).x);
#pragma unroll
                    for (int k = 0; k < HD; k++) o[k] = 0.f;
                    for (int p = 0; p < who.y; p++) {
                        const size_t from = Cut::slot(who.x + p, p == 0) * BQ + row;
                        const float2 x = __ldcg(reinterpret_cast<const float2 *>(part) + from);
                        const float f = x.x == -INFINITY ? (x.y != 0.f ? x.y : 0.f) : kt_ex2(x.x - M);  // (a NaN sum stays one)
                        L = fmaf(x.y, f, L);
#pragma unroll
                        for (int k = 0; k < HD; k += 4) {
                            const float4 y = __ldcg(reinterpret_cast<const float4 *>(po + from * HD + k));
                            o[k] = fmaf(y.x, f, o[k]), o[k + 1] = fmaf(y.y, f, o[k + 1]);
                            o[k + 2] = fmaf(y.z, f, o[k + 2]), o[k + 3] = fmaf(y.w, f, o[k + 3]);
                        }
                    }
                }
            }
            if (write) {
                const float inv = L != 0.f ? 1.f / L : 0.f;  // L is 0 when no key is seen, NaN when a score is
                const int es = dtype == DT_F32 ? 4 : 2;
                const bool wide = !(((uintptr_t)a.out & 15) || ((a.o_row | a.o_head) * es) % 16);
                const long long to = (long long)(sr.first + ri) * a.o_row + (long long)hq * a.o_head;
#pragma unroll
                for (int b = 0; b < HD; b += 8) {
                    float v[8];
#pragma unroll
                    for (int x = 0; x < 4; x++) v[x] = L != 0.f ? o[b + 2 * x] * inv : 0.f, v[x + 4] = L != 0.f ? o[b + 2 * x + 1] * inv : 0.f;
                    if (dtype == DT_F32)
                        store8<DT_F32>(reinterpret_cast<float *>(a.out) + to + b, wide, v);
                    else if (dtype == DT_F16)
                        store8<DT_F16>(reinterpret_cast<__half *>(a.out) + to + b, wide, v);
                    else
                        store8<DT_BF16>(reinterpret_cast<__nv_bfloat16 *>(a.out) + to + b, wide, v);
                }
                if (a.lse)
                    a.lse[(size_t)(sr.first + ri) * a.q_heads + hq] = ((M == -INFINITY ? 0.f : M) + log2f(L)) * 0.69314718055994530942f;
            }
            at += n;
            Cut::next(pl, a, each, sr.n, n);
        }
    }
    if (abort_flag && tid == 0) *reinterpret_cast<volatile int *>(a.err_wait) = 1;
    fence_before_sync();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem, 512);
}

size_t kv4_attend_tc_workspace(const Kv4AttendArgs &a, int sms) {
    return 4 * (KA_BLOCKS + (size_t)2 * std::min(KA_BLOCKS, sms) * KT_BQ * (a.c.width + 2));
}

template <int HD, int G>
static cudaError_t launch_tc(const Kv4AttendArgs &a, int sms, void *work, cudaStream_t s) {
    const size_t smem = KtShape<HD, G>::SMEM;
    cudaError_t e = allow_dynamic_smem((const void *)k_kv4_attend_tc<HD, G>, smem);
    if (e != cudaSuccess) return e;
    k_kv4_attend_tc<HD, G><<<std::min(sms, KA_BLOCKS), KT_THREADS, smem, s>>>(a, DT_F32, reinterpret_cast<float *>(work) + KA_BLOCKS,
                                                                                   reinterpret_cast<int *>(work));
    return cudaGetLastError();
}

cudaError_t launch_kv4_attend_tc(const Kv4AttendArgs &a, int sms, void *work, cudaStream_t s) {
    const int g = a.c.group;
    if (a.c.width == 32) return launch_tc<32, 32>(a, sms, work, s);
    if (a.c.width == 64) return g == 32 ? launch_tc<64, 32>(a, sms, work, s) : launch_tc<64, 64>(a, sms, work, s);
    if (a.c.width == 128)
        return g == 32 ? launch_tc<128, 32>(a, sms, work, s) : g == 64 ? launch_tc<128, 64>(a, sms, work, s) : launch_tc<128, 128>(a, sms, work, s);
    return cudaErrorInvalidValue;
}

}  // namespace tcu

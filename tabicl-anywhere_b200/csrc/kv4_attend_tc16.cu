// Attention of many query rows of a 16-bit type over the four-bit cache on the 5th-generation tensor cores (tcgen05).
//
// 256 query rows of one cache head (the heads that share it side by side) as two tiles of 128, against 64 keys at a time:
// S = Q K^T with Q and the keys, widened to f16, in shared memory; the weights P go to tensor memory over S and multiply
// the widened values; the output stays in tensor memory. Values are one f16 each (11 bits; the results have 11
// or 8), weights two for f16 and one for bf16, sums are f32. Keys are exact, so that the log-sum-exp is f32 as in the other kernels: a key is low + 8 step +
// step (code - 8), the step the sum of its upper 7 and its lower 4 bits, whose products with code - 8 f16 holds; two operand
// blocks have those, and 16 columns beside the first the lows and 8 steps, which meet the sums of q over each group (as two
// f16).
// What bounds it is latency: of a step's 2650 cycles the exponentials need 1024 (16 a cycle and SM), the products 1630, and
// issue is active in 46%; warps wait most for tensor memory, then for one another. So the two tiles have a warpgroup each, and
// widening, which serves both, two that take the steps in turn. Keys rounded to one f16 took 2300 cycles a step (0.40 ms for
// the prompt below, its lse 4e-6 off); of the 400 more half are the products with the steps' lower bits, half the widening;
// keys as two f16 split in f32 took 2980. The products issued from one diverged thread cost 500 cycles more, loops unrolled
// over a whole step (which the instruction caches do not hold beside widening) 400. A prompt of 4096 bf16 tokens after 1000
// cached ones, 32 heads of 128 on 8: 0.46 ms, 0.44 PFLOP/s; f16 0.50.
//
// A row's weights are relative to a reference that follows its largest score only when that has grown by 2^8, so the output
// in tensor memory is rarely rescaled. A step's keys and values are scaled by a power of two of their own that keeps them
// inside f16: beside a value of 2^16 one of 1 keeps its 11 bits, and any is held to 2^-33 of its step's largest. The output
// is in units that follow the steps'. Coordinates keep the order the codes are unpacked in, (0, 4, 1, 5, 2, 6, 3, 7) of every
// eight: Q takes the same order, and the output's columns are put back when they are written.
#include <algorithm>

#include "kv4_tc.cuh"

namespace tcu {

constexpr int KU_R = 256, KU_BQ = 128, KU_BK = 64, KU_THREADS = 640;
constexpr int KU_NK = 2, KU_NS = 3, KU_NR = 3;  // slots of widened keys, of widened values, of stored codes
constexpr int KU_T = 15;    // widened keys and values are below 2^T
constexpr int KU_LAG = 3;   // powers of two that a step's values may lie below the output's unit
constexpr int KU_X = 16;    // columns beside the coordinates in which the groups' lows meet the sums of q
constexpr uint32_t KU_TS = 0, KU_TO = 256;  // tensor memory: [tile][2 slots] of S / P, then [tile] of O

template <int HD, int G>
struct KuShape {
    static constexpr int NU = HD / 32, NG = HD / G, BLOCK = KU_BK * HD;
    static constexpr int KC = KU_BK * HD / 2, SC = KU_BK * NG * 4, RAW = 2 * (KC + SC);
    static constexpr int KSLOT = 2 * BLOCK + KU_BK * KU_X;  // f16 of a step's keys
    static constexpr size_t SMEM = (size_t)KU_R * (HD + KU_X) * 2 + (size_t)(KU_NK * KSLOT + KU_NS * BLOCK) * 2 + (size_t)KU_NR * RAW + 1024;
};

// Warps 0-3, 4-7: softmax of the first and second tile, a thread a query row; warps 8-11, 12-15: widening of even and odd
// steps; warp 16: one thread issues the S products; warp 17: one thread the P V products; warp 18: the copies of the stored
// codes. They hand over through mbarriers; every wait is bounded, and one that gives up raises the block's abort flag, after
// which every wait returns at once and the roles run to the end without results.
// DT: the queries' type. For f16 a weight is the sum of two f16 (of every 16 keys, hi and lo): rounded to one, and the values
// too, results were 1.6 times as far from 64 bits as the plain form's, now 1.35 times; bf16's 8 bits do not show it.
template <int HD, int G, int DT>
__global__ void __launch_bounds__(KU_THREADS, 1) k_kv4_attend_tc16(Kv4AttendArgs a, float *part, int *arrived) {
    constexpr bool SPLIT = DT == DT_F16;
    constexpr int dtype = DT;
    using C = KuShape<HD, G>;
    using Cut = KaCut<KU_R, KU_BK, KU_BK>;
    constexpr int NU = C::NU, NG = C::NG, UG = G / 32, BQ = KU_BQ, BK = KU_BK, NK = KU_NK, NS = KU_NS, NR = KU_NR, BLOCK = C::BLOCK, HX = HD + KU_X, KSLOT = C::KSLOT;
    extern __shared__ __align__(1024) uint8_t smraw[];
    __half *Qs = reinterpret_cast<__half *>(smraw);   // [2][128 x HX], K-major
    __half *Kring = Qs + KU_R * HX;                   // [NK]{[64 x HX], [64 x HD]}, K-major: the keys, and what remains of them
    __half *Vring = Kring + NK * KSLOT;               // [NS][64 x HD], coordinate-major
    uint8_t *raw = reinterpret_cast<uint8_t *>(Vring + NS * BLOCK);  // [NR]{key codes, key scales, value codes, value scales}
    __shared__ float red[2][2][2][4];  // [turn][step][keys, values][warp]
    __shared__ int teK[8], teV[8], has_nan[8];
    __shared__ uint32_t nan_keys[8][NG][2];
    __shared__ __align__(8) uint64_t mK[NK], mV[NS], mKfree[NK], mVfree[NS], mS[2][2], mP[2][2], mSlot[2][2], mQ[2], mDone[2], mRaw[NR],
        mRawFree[NR];
    __shared__ uint32_t tslot;
    __shared__ volatile int abort_flag;
    __shared__ int s_unit[4], s_last[2];
    __shared__ long long s_sum[KU_THREADS / 32];

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wg = warp >> 2;
    const int each = a.q_heads / a.c.heads;
    auto pl = Cut::template place<KU_THREADS>(a, each, KA_TC_STEPS, s_sum, s_unit);
    if (pl.pos >= pl.end) return;
    if (warp == 0) {
        tmem_alloc(&tslot, 512);
        tmem_relinquish();
    }
    if (tid == 0) {
        for (int i = 0; i < NK; i++) mbar_init(&mK[i], 128), mbar_init(&mKfree[i], 1);
        for (int i = 0; i < NS; i++) mbar_init(&mV[i], 128), mbar_init(&mVfree[i], 1);
        for (int q = 0; q < 2; q++) {
            for (int i = 0; i < 2; i++) mbar_init(&mS[q][i], 1), mbar_init(&mP[q][i], BQ), mbar_init(&mSlot[q][i], 1);
            mbar_init(&mQ[q], BQ), mbar_init(&mDone[q], 1);
        }
        for (int i = 0; i < NR; i++) mbar_init(&mRaw[i], 1), mbar_init(&mRawFree[i], 128);
        mbar_init_fence();
        abort_flag = 0;
    }
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = tslot;

    auto wait_warp = [&](uint64_t *m, uint32_t parity) {  // warp-uniform: warp-wide instructions follow
        bool ok = mbar_test_wait(m, parity) || (!abort_flag && mbar_wait(m, parity, KT_WAIT));
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) abort_flag = 1;
        return ok;
    };
    // Every role walks the block's pieces of units alike: n steps; `at` counts the steps before them, at1 those of the second
    // tile (a piece of at most 128 rows has none).
    int at = 0, at1 = 0;

    if (wg == 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        if (warp == 18) {
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
                const int n = (int)min((long long)(sp.steps - pl.skip), pl.end - pl.pos), j0 = sp.base + pl.skip * BK + cp * keys;
                const int *table = a.table + pl.seq * a.table_stride;
                auto there = [&](int i) { return i < n && cp < pieces && j0 + i * BK < sp.hi_max && j0 + i * BK + keys > sp.lo_min; };
                auto find = [&](int i) { return there(i) ? table[(j0 + i * BK) >> shift] : -1; };  // a page number, two steps ahead
                int next = find(0), after = find(1);
                for (int i = 0; i < n; i++, at++) {
                    const int slot = at % NR, pg = next;
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
                                     "l"(a.c.pool + ((size_t)pg * a.c.heads + pl.head) * hb + from + ((j0 + i * BK) & (page - 1)) * per_key),
                                     "r"(bytes), "r"(smem_addr(&mRaw[slot]))
                                     : "memory");
                }
                Cut::next(pl, a, each, sr.n, n);
            }
            // what was asked for lands before the block lets go of shared memory
            for (int i = max(0, at - NR); i < at; i++) mbar_wait(&mRaw[i % NR], (uint32_t)(i / NR) & 1u, KT_WAIT);
        } else if (warp < 18) {
            // ---- the products ----
            const uint32_t idS = idesc_f16(BQ, BK, 0, 0), idO = idesc_f16(BQ, HD, 0, 1);
            const uint64_t dQ0 = kstep_desc(Qs, BQ, 0), dK0 = kstep_desc(Kring, BK, 0), dV0 = kstep_desc(Vring, HD, 0);
            constexpr uint64_t stQ = (2 * (BQ / 8) * 128) >> 4, stK = (2 * (BK / 8) * 128) >> 4, stV = (2 * (HD / 8) * 128) >> 4;
            constexpr uint64_t q_off = (BQ * HX * 2) >> 4, k_off = (KSLOT * 2) >> 4, lo_off = (BK * HX * 2) >> 4, v_off = (BLOCK * 2) >> 4;
            int units[2] = {0, 0};  // pieces of each tile so far
            while (pl.pos < pl.end) {
                const KaRows sr = ka_rows(a, pl.seq);
                const auto sp = Cut::span(a, sr, each, pl.rt);
                const int n = (int)min((long long)(sp.steps - pl.skip), pl.end - pl.pos), nq = sr.n * each - pl.rt * KU_R > BQ ? 2 : 1;
                for (int i = 0; i < n; i++) {
                    if (warp == 16) {
                        // S(i) of both tiles from the keys of step i, once P V(i - 2) has read the slot
                        const int sl = (at + i) % NK;
                        wait_warp(&mK[sl], (uint32_t)((at + i) / NK) & 1u);
                        const uint64_t dK = dK0 + sl * k_off;
#pragma unroll
                        for (int q = 0; q < 2; q++) {
                            if (q >= nq) break;
                            const int c = (q ? at1 : at) + i;
                            if (i == 0) wait_warp(&mQ[q], (uint32_t)units[q] & 1u);
                            if (c >= 2) wait_warp(&mSlot[q][c & 1], (uint32_t)((c >> 1) - 1) & 1u);
                            fence_after_sync();
                            const uint32_t tS = tmem + KU_TS + (2 * q + (c & 1)) * BK;
                            if (elect_one()) {
#pragma unroll
                                for (int k = 0; k < HD / 16; k++) mma_f16(tS, dQ0 + q * q_off + k * stQ, dK + lo_off + k * stK, idS, k > 0 ? 1u : 0u);
#pragma unroll
                                for (int k = 0; k < HX / 16; k++) mma_f16(tS, dQ0 + q * q_off + k * stQ, dK + k * stK, idS, 1);
                                mma_commit(&mS[q][c & 1]);
                                if (q == nq - 1) mma_commit(&mKfree[sl]);
                            }
                            __syncwarp();
                        }
                    } else {
                        // P V(i) of both tiles, from the values of step i
                        const int sl = (at + i) % NS;
                        wait_warp(&mV[sl], (uint32_t)((at + i) / NS) & 1u);
                        const uint64_t dV = dV0 + sl * v_off;
#pragma unroll
                        for (int q = 0; q < 2; q++) {
                            if (q >= nq) break;
                            const int c = (q ? at1 : at) + i;
                            wait_warp(&mP[q][c & 1], (uint32_t)(c >> 1) & 1u);
                            fence_after_sync();
                            const uint32_t tP = tmem + KU_TS + (2 * q + (c & 1)) * BK;
                            if (elect_one()) {
#pragma unroll
                                for (int k = 0; k < BK / 16; k++)
                                    mma_f16_ta(tmem + KU_TO + q * HD, tP + (SPLIT ? 16 : 8) * k, dV + k * stV, idO, i > 0 || k > 0 ? 1u : 0u);
                                if constexpr (SPLIT) {
#pragma unroll
                                    for (int k = 0; k < BK / 16; k++) mma_f16_ta(tmem + KU_TO + q * HD, tP + 16 * k + 8, dV + k * stV, idO, 1);
                                }
                                mma_commit(&mSlot[q][c & 1]);
                                if (q == nq - 1) mma_commit(&mVfree[sl]);
                            }
                            __syncwarp();
                        }
                    }
                }
                units[0]++, units[1] += nq == 2;
                at += n, at1 += nq == 2 ? n : 0;
                Cut::next(pl, a, each, sr.n, n);
            }
            // every product issued here completes before the block lets go of its memory
            if (elect_one()) {
                mma_commit(&mDone[warp - 16]);
                mbar_wait(&mDone[warp - 16], 0, KT_WAIT);
            }
            __syncwarp();
        }
    } else if (wg >= 2) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        // ---- widening: a thread half a key's coordinates and half a value's, of every other step ----
        // (a wait that gave up does not end the loop: the four warps meet at a barrier in every step)
        const int key = tid & 63, half = (tid >> 6) & 1, w4 = warp & 3, turn = wg - 2;
        while (pl.pos < pl.end) {
            const KaRows sr = ka_rows(a, pl.seq);
            const auto sp = Cut::span(a, sr, each, pl.rt);
            const int n = (int)min((long long)(sp.steps - pl.skip), pl.end - pl.pos), j0 = sp.base + pl.skip * BK;
            for (int i = at + ((at ^ turn) & 1); i < at + n; i += 2) {
                const int kl = i % NK, sl = i % NS, rs = i % NR, j = j0 + (i - at) * BK + key;
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
                // a group of values that stands for NaN is left out here and put into the rows that see it at the end
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
                kt_bar(1 + turn, 128);
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
#pragma unroll
                for (int k = 0; k < NG; k++) {
                    // in the step's unit from here on: exact, but for steps and lows below 2^-28 of its largest
                    const float2 f = __half22float2(kt_h2(kc[k])), g = __half22float2(kt_h2(vc[k]));
                    const float uk = kt_pow2(KU_T - e[0]), uv = kt_pow2(KU_T - e[1]);
                    kc[k] = kt_u32(__floats2half2_rn(f.x * uk, f.y * uk)), vc[k] = kt_u32(__floats2half2_rn(g.x * uv, g.y * uv));
                }
                // (loops that are not unrolled over the halves: short code, see the softmax)
                if (i >= NK) wait_warp(&mKfree[kl], ((uint32_t)(i / NK) & 1u) ^ 1u);
#pragma unroll 1
                for (int x = 2 * half; x < 2 * half + 2; x++) {
                    uint32_t w[NU];
                    lds_words<NU>(kraw + key * (HD / 2) + x * NU * 4, w);
                    __half *hi = Kring + kl * KSLOT + kmajor_off(key, 8 * x, BK), *lo = hi + BK * HX;
#pragma unroll
                    for (int u = 0; u < NU; u++)
                        kt_exact(w[u], __low2half2(kt_h2(kc[u / UG])), hi + kmajor_off(0, 32, BK) * u, lo + kmajor_off(0, 32, BK) * u);
                }
                {
                    // beside them low, low, 8 step, 8 step of the four groups that there may be; here those of two
                    uint32_t x[4] = {0, 0, 0, 0};
#pragma unroll
                    for (int k = 0; k < NG; k++)
                        if (k / 2 == half) {
                            const __half2 s = kt_h2(kc[k]);
                            x[k % 2 * 2] = kt_u32(__high2half2(s)), x[k % 2 * 2 + 1] = kt_u32(__hmul2(__low2half2(s), kt_h2(0x48004800u)));
                        }
                    *reinterpret_cast<uint4 *>(Kring + kl * KSLOT + kmajor_off(key, HD + 8 * half, BK)) = make_uint4(x[0], x[1], x[2], x[3]);
                }
                fence_async_smem();
                mbar_arrive(&mK[kl]);
                if (i >= NS) wait_warp(&mVfree[sl], ((uint32_t)(i / NS) & 1u) ^ 1u);
#pragma unroll 1
                for (int x = 2 * half; x < 2 * half + 2; x++) {
                    uint32_t w[NU];
                    lds_words<NU>(vraw + key * (HD / 2) + x * NU * 4, w);
                    __half *to = Vring + sl * BLOCK + mnmajor_off(8 * x, key, HD);
#pragma unroll
                    for (int u = 0; u < NU; u++) {
                        // half-words g = 2 x and 2 x + 1 of a unit: coordinates 32 u + 8 x + (0..7)
                        uint32_t c;
                        if constexpr (NU == 1)
                            c = w[0];
                        else
                            c = __byte_perm(w[u / 2], w[NU / 2 + u / 2], u & 1 ? 0x7632 : 0x5410);
                        const __half2 g = kt_h2(vc[u / UG]);
                        kt_round(c, __low2half2(g), __high2half2(g), to + mnmajor_off(32, 0, HD) * u);
                    }
                }
                fence_async_smem();
                mbar_arrive(&mV[sl]);
                mbar_arrive(&mRawFree[rs]);
            }
            at += n;
            Cut::next(pl, a, each, sr.n, n);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 136;");
        const int q = wg, row = tid & (BQ - 1);
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
        const int es = 2;
        const bool wide_q = !(((uintptr_t)a.q & 15) || ((a.q_row | a.q_head) * es) % 16);
        const bool wide_o = !(((uintptr_t)a.out & 15) || ((a.o_row | a.o_head) * es) % 16);
        while (pl.pos < pl.end) {
            const KaRows sr = ka_rows(a, pl.seq);
            const auto sp = Cut::span(a, sr, each, pl.rt);
            const int n = (int)min((long long)(sp.steps - pl.skip), pl.end - pl.pos), j0 = sp.base + pl.skip * BK;
            const int r0 = pl.rt * KU_R + q * BQ, rows = min(BQ, sr.n * each - r0);
            if (rows <= 0) {
                at += n;
                Cut::next(pl, a, each, sr.n, n);
                continue;
            }
            const int r = min(row, rows - 1), ri = (r0 + r) / each, hq = pl.head * each + (r0 + r) % each;  // rows past the end repeat the last
            const int my_hi = ka_hi(a, sr, ri), my_lo = ka_lo(a, sr, ri);
            const int hi_min = ka_hi(a, sr, r0 / each), lo_max = ka_lo(a, sr, (r0 + rows - 1) / each);
            int c = q ? at1 : at;  // this tile's steps so far

            // ---- Q: a warp its 32 rows, 8 rows x 4 chunks of 8 coordinates at a time; a row scaled by a power of two of its own
            // to at most 2^8 (so that the groups' sums beside it stay inside f16) ----
            float rowfac = 0.f;
            {
                constexpr int NC = HD / 32;  // chunks of a row a lane reads
                auto get = [&](uint32_t x) {
                    return dtype == DT_BF16 ? make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u)) : __half22float2(kt_h2(x));
                };
                uint32_t raw_q[4][NC][4];
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int qr = r0 + min((warp & 3) * 32 + x * 8 + (lane & 7), rows - 1);
                    const uint16_t *src = reinterpret_cast<const uint16_t *>(a.q) + (long long)(sr.first + qr / each) * a.q_row +
                                          (long long)(pl.head * each + qr % each) * a.q_head + (lane >> 3) * 8;
#pragma unroll
                    for (int y = 0; y < NC; y++) {
                        if (wide_q) {
                            const uint4 v = __ldg(reinterpret_cast<const uint4 *>(src + 32 * y));
                            raw_q[x][y][0] = v.x, raw_q[x][y][1] = v.y, raw_q[x][y][2] = v.z, raw_q[x][y][3] = v.w;
                        } else {
#pragma unroll
                            for (int z = 0; z < 4; z++) raw_q[x][y][z] = (uint32_t)src[32 * y + 2 * z] | (uint32_t)src[32 * y + 2 * z + 1] << 16;
                        }
                    }
                }
#pragma unroll
                for (int x = 0; x < 4; x++) {
                    const int qrow = (warp & 3) * 32 + x * 8 + (lane & 7);
                    const uint32_t(&w)[NC][4] = raw_q[x];
                    float mx = 0.f;
#pragma unroll
                    for (int y = 0; y < NC; y++)
#pragma unroll
                        for (int z = 0; z < 4; z++) {
                            const float2 v = get(w[y][z]);
                            mx = fmaxf(mx, fmaxf(fabsf(v.x), fabsf(v.y)));
                        }
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                    const int e = mx > 0.f ? min(126, 134 - (int)((__float_as_uint(mx) >> 23) & 0xff)) : 0;
                    const float up = a.scale < 0.f ? -kt_pow2(e) : kt_pow2(e);
                    // a score in units of log2: the product with the widened keys times this and the step's power of two
                    const float fac = __shfl_sync(0xffffffffu, fabsf(a.scale) * 1.44269504088896340736f * kt_pow2(-e), lane & 7);
                    if (lane >> 3 == x) rowfac = fac;
                    float sum[4] = {0.f, 0.f, 0.f, 0.f};  // of the groups
#pragma unroll
                    for (int y = 0; y < NC; y++) {
                        float v[8];
#pragma unroll
                        for (int z = 0; z < 4; z++) {
                            const float2 f = get(w[y][z]);
                            v[2 * z] = f.x * up, v[2 * z + 1] = f.y * up;
                        }
                        uint32_t h[4];
#pragma unroll
                        for (int z = 0; z < 4; z++) {
                            h[z] = kt_u32(__floats2half2_rn(v[z], v[z + 4]));
                            const float2 f = __half22float2(kt_h2(h[z]));
                            sum[y / UG] += f.x + f.y;
                        }
                        *reinterpret_cast<uint4 *>(Qs + q * BQ * HX + kmajor_off(qrow, 32 * y + (lane >> 3) * 8, BQ)) = make_uint4(h[0], h[1], h[2], h[3]);
                    }
                    uint32_t both[4];  // a group's sum and what remains of it
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 8);
                        sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 16);
                        const float f = __half2float(__float2half_rn(sum[k]));
                        both[k] = kt_u32(__floats2half2_rn(f, sum[k] - f));
                    }
                    if (lane < 16)  // as the keys' lows and steps lie: two groups in 8 columns
                        *reinterpret_cast<uint4 *>(Qs + q * BQ * HX + kmajor_off(qrow, HD + (lane >> 3) * 8, BQ)) =
                            lane < 8 ? make_uint4(both[0], both[0], both[1], both[1]) : make_uint4(both[2], both[2], both[3], both[3]);
                }
                fence_async_smem();
                mbar_arrive(&mQ[q]);
            }

            // ---- softmax: S(i) -> P(i) over S(i) ----
            float m = -INFINITY, l = 0.f;  // the row's reference (log2), its sum of weights times 2^7
            int unit = 0;                  // the output is in units of 2^(unit - T - 7)
            uint32_t nans = 0;             // groups whose output is NaN
            for (int i = 0; i < n; i++, c++) {
                const int key0 = j0 + i * BK, x8 = (at + i) & 7;
                const uint32_t tsp = tmem + lane_base + KU_TS + (2 * q + (c & 1)) * BK;
                if (!wait_warp(&mS[q][c & 1], (uint32_t)(c >> 1) & 1u)) break;
                fence_after_sync();
                // (held to the normal numbers: positive for a scale of 0 too, so that -infinity stays itself)
                const float c1 = fminf(fmaxf(rowfac * kt_pow2(*reinterpret_cast<volatile int *>(&teK[x8]) - KU_T), FLT_MIN), FLT_MAX);
                const int e = *reinterpret_cast<volatile int *>(&teV[x8]);
                const bool edge = key0 < lo_max || key0 + BK > hi_min;
                // Two passes over the step's scores in tensor memory, 32 at a time in loops that are not unrolled further: the code
                // of a step is then short enough for the instruction caches, which the two kinds of warpgroups share.
                float mx;
                {
                    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
                    for (int b = 0; b < 2; b++) {
                        float x[32];
                        tmem_ld32(tsp + 32 * b, x);
                        tmem_wait_ld32(x);
                        if (edge) {
#pragma unroll
                            for (int k = 0; k < 32; k++)
                                if (key0 + 32 * b + k < my_lo || key0 + 32 * b + k >= my_hi) x[k] = -INFINITY;
                        }
#pragma unroll
                        for (int k = 0; k < 32; k++) top[k & 3] = fmaxf(top[k & 3], x[k]);
                    }
                    mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * c1;
                }
                if (i == 0) unit = e;
                // (the output's unit follows steps of much smaller values down too: weights scaled down for them would leave f16's
                // normal numbers, f32 has room for whatever the output is then)
                const bool other = e > unit || e < unit - KU_LAG;
                if (__any_sync(0xffffffffu, mx > m + 8.f) || other) {
                    const float mnew = fmaxf(m, mx), f = m == -INFINITY ? 0.f : kt_ex2(m - mnew);
                    const int unew = other ? e : unit;
                    if (i > 0) {  // O, once the product before has been added to it
                        if (!wait_warp(&mSlot[q][(c - 1) & 1], (uint32_t)((c - 1) >> 1) & 1u)) break;
                        fence_after_sync();
                        const float fo = f * kt_pow2(unit - unew);
#pragma unroll 1
                        for (int b = 0; b < HD / 32; b++) {
                            float x[32];
                            tmem_ld32(tmem + lane_base + KU_TO + q * HD + 32 * b, x);
                            tmem_wait_ld32(x);
#pragma unroll
                            for (int k = 0; k < 32; k++) x[k] *= fo;
                            tmem_st32(tmem + lane_base + KU_TO + q * HD + 32 * b, x);
                        }
                        tmem_wait_st();
                    }
                    l *= f, m = mnew, unit = unew;
                }
                // weights times 2^7 (up to 2^15), in units of the step's values (which are at most LAG powers of two smaller)
                const float mm = (m == -INFINITY ? 0.f : m) - 7.f - (float)(e - unit);
                float part_sum[4] = {};
#pragma unroll 1
                for (int b = 0; b < 2; b++) {
                    float x[32];
                    tmem_ld32(tsp + 32 * b, x);
                    tmem_wait_ld32(x);
                    if (edge) {
#pragma unroll
                        for (int k = 0; k < 32; k++)
                            if (key0 + 32 * b + k < my_lo || key0 + 32 * b + k >= my_hi) x[k] = -INFINITY;
                    }
                    uint32_t h[SPLIT ? 32 : 16];
#pragma unroll
                    for (int k = 0; k < 16; k++) {
                        const float p0 = kt_ex2(fmaf(x[2 * k], c1, -mm)), p1 = kt_ex2(fmaf(x[2 * k + 1], c1, -mm));
                        part_sum[(2 * k) & 3] += p0, part_sum[(2 * k + 1) & 3] += p1;
                        if constexpr (SPLIT)
                            split_pair(p0, p1, h[k / 8 * 16 + k % 8], h[k / 8 * 16 + 8 + k % 8]);
                        else
                            h[k] = kt_u32(__floats2half2_rn(p0, p1));
                    }
                    // over scores that have been read
                    if constexpr (SPLIT)
                        tmem_st32u(tsp + 32 * b, h);
                    else
                        tmem_st16u(tsp + 16 * b, h);
                }
                const float sum = (part_sum[0] + part_sum[1]) + (part_sum[2] + part_sum[3]);
                tmem_wait_st();
                fence_before_sync();
                mbar_arrive(&mP[q][c & 1]);
                l = fmaf(sum, kt_pow2(unit - e), l);
                if (*reinterpret_cast<volatile int *>(&has_nan[x8])) {
                    for (int k = 0; k < NG; k++)
                        for (int b = 0; b < 64; b++)
                            if ((nan_keys[x8][k][b >> 5] >> (b & 31) & 1) && key0 + b >= my_lo && key0 + b < my_hi) nans |= 1u << k;
                }
            }

            // ---- the row's output, or its part of it ----
            const bool whole = n == sp.steps;
            bool write = row < rows;
            float M = m, L = l * 0.0078125f;
            const float un = kt_pow2(unit - KU_T - 7);
            if (c > 0) wait_warp(&mSlot[q][(c - 1) & 1], (uint32_t)((c - 1) >> 1) & 1u);
            fence_after_sync();
            const uint32_t to_o = tmem + lane_base + KU_TO + q * HD;
            // 32 columns from 32 b on into the row's place in Q's memory (its products are done), 16 bytes of 8 coordinates each
            auto put = [&](int b, const float (&o)[32], float inv) {
#pragma unroll
                for (int y = 0; y < 32; y += 8) {
                    float v[8];
#pragma unroll
                    for (int x = 0; x < 4; x++) {
                        v[x] = L != 0.f ? o[y + 2 * x] * inv : 0.f, v[x + 4] = L != 0.f ? o[y + 2 * x + 1] * inv : 0.f;
                    }
                    uint16_t *to = reinterpret_cast<uint16_t *>(Qs) + q * BQ * HX + kmajor_off(row, 32 * b + y, BQ);
                    if (dtype == DT_F16)
                        store8<DT_F16>(reinterpret_cast<__half *>(to), true, v);
                    else
                        store8<DT_BF16>(reinterpret_cast<__nv_bfloat16 *>(to), true, v);
                }
            };
            // the warp's rows from there to memory, 8 rows x 4 chunks at a time
            auto flush = [&]() {
                __syncwarp();
#pragma unroll 1
                for (int x = 0; x < 4; x++) {
                    const int orow = (warp & 3) * 32 + x * 8 + (lane & 7), orr = r0 + orow;
                    uint16_t *dst = reinterpret_cast<uint16_t *>(a.out) + (long long)(sr.first + orr / each) * a.o_row +
                                    (long long)(pl.head * each + orr % each) * a.o_head + (lane >> 3) * 8;
#pragma unroll
                    for (int y = 0; y < HD / 32; y++) {
                        const uint4 v = *reinterpret_cast<const uint4 *>(Qs + q * BQ * HX + kmajor_off(orow, 32 * y + (lane >> 3) * 8, BQ));
                        if (orow >= rows) continue;
                        if (wide_o) {
                            *reinterpret_cast<uint4 *>(dst + 32 * y) = v;
                        } else {
                            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                            for (int z = 0; z < 4; z++) dst[32 * y + 2 * z] = (uint16_t)w[z], dst[32 * y + 2 * z + 1] = (uint16_t)(w[z] >> 16);
                        }
                    }
                }
                __syncwarp();
            };
            auto put_lse = [&]() {
                if (a.lse) a.lse[(size_t)(sr.first + ri) * a.q_heads + hq] = ((M == -INFINITY ? 0.f : M) + log2f(L)) * 0.69314718055994530942f;
            };
            const int2 who = Cut::sharers(pl, pl.pos - pl.skip, sp.steps);
            float *po = part + 2 * (size_t)2 * gridDim.x * KU_R;
            const int prow = q * BQ + row;
            const size_t mine = Cut::slot(blockIdx.x, pl.skip == 0) * KU_R + prow;
            const float inv = L != 0.f ? un / L : 0.f;  // L is 0 when no key is seen, NaN when a score is
#pragma unroll 1
            for (int b = 0; b < HD / 32; b++) {
                float o[32];
                tmem_ld32(to_o + 32 * b, o);
                tmem_wait_ld32(o);
                if (nans >> (32 * b / G) & 1) {
#pragma unroll
                    for (int k = 0; k < 32; k++) o[k] = NAN;
                }
                if (whole) {
                    put(b, o, inv);
                } else if (write) {
#pragma unroll
                    for (int k = 0; k < 32; k += 4)
                        __stcg(reinterpret_cast<float4 *>(po + mine * HD + 32 * b + k), make_float4(o[k] * un, o[k + 1] * un, o[k + 2] * un, o[k + 3] * un));
                }
            }
            fence_before_sync();
            if (whole) {
                flush();
                if (write) put_lse();
            } else {
                if (write) __stcg(reinterpret_cast<float2 *>(part) + mine, make_float2(M, L));
                __threadfence();
                kt_bar(3 + q, 128);
                if (row == 0) {
                    // (a counter for each tile: the second tile's behind the first's)
                    int *count = arrived + q * (KA_BLOCKS / 2) + who.x;
                    s_last[q] = atomicAdd(count, 1) == who.y - 1;
                    if (s_last[q]) *count = 0;  // ready for the next call
                }
                kt_bar(3 + q, 128);
                const bool s_last_seen = s_last[q];
                write = write && s_last_seen;
                kt_bar(3 + q, 128);  // (read before a next piece writes it)
                if (write) {
                    __threadfence();
                    M = -INFINITY, L = 0.f;
                    for (int p = 0; p < who.y; p++)
                        M = fmaxf(M, __ldcg(reinterpret_cast<const float2 *>(part) + Cut::slot(who.x + p, p == 0) * KU_R + prow).x);
                    auto weight = [&](float2 x) { return x.x == -INFINITY ? (x.y != 0.f ? x.y : 0.f) : kt_ex2(x.x - M); };  // (a NaN sum stays one)
                    for (int p = 0; p < who.y; p++) {
                        const float2 x = __ldcg(reinterpret_cast<const float2 *>(part) + Cut::slot(who.x + p, p == 0) * KU_R + prow);
                        L = fmaf(x.y, weight(x), L);
                    }
                    const float w = L != 0.f ? 1.f / L : 0.f;
#pragma unroll 1
                    for (int b = 0; b < HD / 32; b++) {
                        float o[32];
#pragma unroll
                        for (int k = 0; k < 32; k++) o[k] = 0.f;
                        for (int p = 0; p < who.y; p++) {
                            const size_t src = Cut::slot(who.x + p, p == 0) * KU_R + prow;
                            const float f = weight(__ldcg(reinterpret_cast<const float2 *>(part) + src));
#pragma unroll
                            for (int k = 0; k < 32; k += 4) {
                                const float4 y = __ldcg(reinterpret_cast<const float4 *>(po + src * HD + 32 * b + k));
                                o[k] = fmaf(y.x, f, o[k]), o[k + 1] = fmaf(y.y, f, o[k + 1]);
                                o[k + 2] = fmaf(y.z, f, o[k + 2]), o[k + 3] = fmaf(y.w, f, o[k + 3]);
                            }
                        }
                        put(b, o, w);
                    }
                    put_lse();
                }
                if (s_last_seen) flush();
            }
            at += n, at1 += q ? n : 0;
            Cut::next(pl, a, each, sr.n, n);
        }
    }
    if (abort_flag && tid == 0) *reinterpret_cast<volatile int *>(a.err_wait) = 1;
    fence_before_sync();
    __syncthreads();
    if (warp == 0) tmem_dealloc(tmem, 512);
}

size_t kv4_attend_tc16_workspace(const Kv4AttendArgs &a, int sms) {
    return 4 * (KA_BLOCKS + (size_t)2 * std::min(KA_BLOCKS / 2, sms) * KU_R * (a.c.width + 2));
}

template <int HD, int G, int DT>
static cudaError_t launch_type(const Kv4AttendArgs &a, int sms, void *work, cudaStream_t s) {
    const size_t smem = KuShape<HD, G>::SMEM;
    cudaError_t e = allow_dynamic_smem((const void *)k_kv4_attend_tc16<HD, G, DT>, smem);
    if (e != cudaSuccess) return e;
    k_kv4_attend_tc16<HD, G, DT><<<std::min(sms, KA_BLOCKS / 2), KU_THREADS, smem, s>>>(a, reinterpret_cast<float *>(work) + KA_BLOCKS,
                                                                                        reinterpret_cast<int *>(work));
    return cudaGetLastError();
}
template <int HD, int G>
static cudaError_t launch_tc16(int dtype, const Kv4AttendArgs &a, int sms, void *work, cudaStream_t s) {
    return dtype == DT_F16 ? launch_type<HD, G, DT_F16>(a, sms, work, s) : launch_type<HD, G, DT_BF16>(a, sms, work, s);
}

cudaError_t launch_kv4_attend_tc16(int dtype, const Kv4AttendArgs &a, int sms, void *work, cudaStream_t s) {
    const int g = a.c.group;
    if (a.c.width == 32) return launch_tc16<32, 32>(dtype, a, sms, work, s);
    if (a.c.width == 64) return g == 32 ? launch_tc16<64, 32>(dtype, a, sms, work, s) : launch_tc16<64, 64>(dtype, a, sms, work, s);
    if (a.c.width == 128)
        return g == 32   ? launch_tc16<128, 32>(dtype, a, sms, work, s)
               : g == 64 ? launch_tc16<128, 64>(dtype, a, sms, work, s)
                         : launch_tc16<128, 128>(dtype, a, sms, work, s);
    return cudaErrorInvalidValue;
}

}  // namespace tcu

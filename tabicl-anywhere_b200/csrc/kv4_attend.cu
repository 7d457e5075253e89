// Attention of ragged query rows over a four-bit paged cache: few rows a cache head (decoding, short tails).
//
// The codes go into the matrix unit as they are. A nibble is a subnormal f16 (code * 2^-24, or 2^-20 from the second
// nibble of a byte: one AND takes two of them out of a word), so a product with the codes is exact in everything but q and
// the weights, and the group scales act on its f32 result:
//     q . k_j   = sum over groups of  step * (q_g . codes)  +  low * (sum of q_g)
//     sum p_j v = sum over groups of  (p_j step) . codes    +  sum p_j low
// f32 and f16 queries take code - 8 and low + 8 step instead (code_pair), and f32 adds each step's products to the output by
// itself. One f32 row over 10,000 keys, 4 heads of 128: 14.2 us (13.5 with codes as they are, and then off by 1.3e-4 of an
// output of values that cancel; now 4e-7). 64 f32 rows over 8000 keys, 8 heads of 128: 256 us, and 2e-6 off or less; with the
// matrix unit's own sums over the steps 244 us, and up to 1e-5 off.
// What bounds it: issue. Taking a code out of its word is one logic instruction for two, and a step of 32 keys with 8 query
// rows some 600 instructions a warp, at 0.55 a cycle and scheduler with the 12 warps that the registers of q, the output
// and the sums leave an SM. 64 bf16 rows (32 heads of 128 on 8, groups of 32) over 0..16384 cached tokens: 0.191 ms, 3.8 TB/s
// of codes and scales, 58% of a copy's rate; with 16 warps and spills 0.225 ms.
//
// Per 32 keys a warp computes S^T = K Q^T with 16 keys as rows and 8 query rows as columns, so a key's codes are read in
// the order they are stored in, and O^T = V^T P'^T with P' = p * step turned round in registers (movmatrix).
#include <algorithm>
#include <atomic>

#include "kv4_plan.cuh"

namespace tcu {

constexpr int KA_KEYS = 32;     // keys of a warp's step
constexpr int KA_WARPS = 4;     // warps of a block, each over its own steps of the block's keys
constexpr int KA_STEP = KA_WARPS * KA_KEYS;  // keys of a block's step
constexpr long long KA_WAIT = 2000000000ll;  // a warp gives up a copy after about a second at boost clock

template <int HD, int G>
struct KaTile {
    static constexpr int NU = HD / 32, NG = HD / G;
    static constexpr int KC = KA_KEYS * HD / 2, SC = KA_KEYS * NG * 4;  // bytes of the codes and of the scales
    static constexpr int BYTES = 2 * (KC + SC);
    static constexpr int STAGES = BYTES > 6000 ? 2 : 3;
    // the `low` part of the scores as a matrix product of the keys' lows with the groups' sums of q (as f16 hi and lo):
    // one fragment of NG hi and NG lo columns; with one or two groups the multiply-adds are as few
    static constexpr bool LOW_MMA = NG >= 4;
};

__device__ __forceinline__ uint32_t ka_smem(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
// `bytes` (a multiple of 16) from global to shared memory, both 16-byte aligned; they count on the barrier.
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(bar)
                 : "memory");
}
// Waits for the barrier's phase; false after KA_WAIT.
__device__ __forceinline__ bool ka_wait(uint32_t bar, uint32_t parity) {
    auto done = [&] {
        uint32_t p;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(p) : "r"(bar), "r"(parity) : "memory");
        return p != 0;
    };
    if (done()) return true;
    const long long t0 = clock64();
    while (!done())
        if (clock64() - t0 > KA_WAIT) return false;
    return true;
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma1688(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(b0));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t half2_bits(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 bits_float2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
__device__ __forceinline__ float exp2_sfu(float x) {  // relative error 2^-22; 0 for -infinity
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -127 < e < 128

// TYPE: the queries' type. f32: q and the weights as two f16, else as one; bf16: codes as they are, and the weights' products
// with their steps in f16 pairs, each rounded to the 11 bits that 8-bit results do not show.
template <int HD, int G, int NT, int TYPE>
__global__ void __launch_bounds__(KA_STEP, (HD <= 128 && NT == 1 && TYPE != DT_F32) ? 3 : 1)
    k_kv4_attend(Kv4AttendArgs a, int dtype, int min_steps, float *part, int *arrived) {
    using C = KaTile<HD, G>;
    constexpr int NU = C::NU, NG = C::NG, UG = G / 32, R = 8 * NT, ST = C::STAGES, QS = TYPE == DT_F32 ? 2 : 1;
    constexpr bool SPLIT = TYPE == DT_F32, CENTRED = TYPE != DT_BF16, LOW_MMA = C::LOW_MMA && !CENTRED;
    constexpr float UNIT = CENTRED ? 1.f : 16777216.f;  // undoes the codes' 2^-24
    extern __shared__ __align__(16) uint8_t sm[];
    __shared__ int s_last, s_unit[4];
    __shared__ long long s_sum[KA_WARPS];
    __shared__ __align__(8) unsigned long long bars[KA_WARPS][ST];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int each = a.q_heads / a.c.heads;

    using Cut = KaCut<R, KA_KEYS, KA_STEP>;
    auto pl = Cut::template place<KA_STEP>(a, each, min_steps, s_sum, s_unit);
    if (pl.pos >= pl.end) return;

    // this warp's ring: each step's key codes, key scales, value codes and value scales come as four bulk copies (eight
    // when the 32 keys lie on two pages of 16), one a lane, that count on the slot's barrier
    uint8_t *ring = sm + warp * ST * C::BYTES;
    const uint32_t ring_at = ka_smem(ring), bar_at = ka_smem(&bars[warp][0]);
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < ST; i++) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar_at + 8 * i) : "memory");
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    uint32_t used = 0;  // steps of this warp so far: the ring's place and the barriers' phases
    bool gave_up = false;  // a copy did not come: the warp reads no more
    const size_t hb = kv4_head_bytes(HD, a.c.page, G);
    const Kv4Offsets off = kv4_offsets(HD, a.c.page, G);
    const int page_shift = 31 - __clz(a.c.page), halves = a.c.page == 16 ? 2 : 1;
    const int cpart = lane & 3, chalf = (lane >> 2) & 1;
    const uint32_t from = (cpart & 2 ? off.vc : 0) + (cpart & 1 ? off.ks : 0);  // ks = vs - vc: the codes before the scales
    const uint32_t per_key = cpart & 1 ? NG * 4 : HD / 2, copy_bytes = per_key * KA_KEYS / halves;
    const uint32_t to = (cpart & 2 ? C::KC + C::SC : 0) + (cpart & 1 ? C::KC : 0) + chalf * copy_bytes;
    while (pl.pos < pl.end) {
    const int seq = pl.seq, head = pl.head, skip = pl.skip, r0 = pl.rt * R;
    const KaRows sr = ka_rows(a, seq);
    const auto sp = Cut::span(a, sr, each, pl.rt);
    const int piece = (int)min((long long)(sp.steps - skip), pl.end - pl.pos), rows = min(R, sr.n * each - r0);
    const int lo_min = sp.lo_min, lo_max = sp.lo_max, hi_min = sp.hi_min, hi_max = sp.hi_max;
    const int k0 = sp.base + skip * KA_STEP, k1 = hi_max > lo_min ? min(hi_max, k0 + piece * KA_STEP) : k0;
    const int ntiles = (k1 - k0 + KA_KEYS - 1) / KA_KEYS, mine = gave_up ? 0 : max(0, (ntiles - warp + KA_WARPS - 1) / KA_WARPS);
    // the page numbers are read a step before they are needed
    int pages[2];
    auto find = [&](int it) {
        const int j0 = k0 + (warp + it * KA_WARPS) * KA_KEYS;
#pragma unroll
        for (int h = 0; h < 2; h++)
            pages[h] = h < halves && j0 + 16 * h < k1 ? a.table[seq * a.table_stride + ((j0 + 16 * h) >> page_shift)] : -1;
    };
    auto load = [&](int it) {  // this warp's it-th step into its ring
        if (it >= mine) return;
        const int j0 = k0 + (warp + it * KA_WARPS) * KA_KEYS;
        const bool ok0 = pages[0] >= 0 && pages[0] < a.c.pages, ok1 = pages[1] >= 0 && pages[1] < a.c.pages;
        const uint32_t slot = (used + it) % ST, bar = bar_at + 8 * slot;
        if (lane == 0) {
            if ((!ok0 && j0 + KA_KEYS / halves > lo_min) || (halves == 2 && !ok1 && j0 + 16 < k1 && j0 + KA_KEYS > lo_min))
                *reinterpret_cast<volatile int *>(a.err) = 1;
            const uint32_t bytes = C::BYTES / halves * ((int)ok0 + (int)ok1);
            asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}\n" ::"r"(bar), "r"(bytes) : "memory");
        }
        if (lane < 4 * halves && (chalf ? ok1 : ok0)) {
            const uint8_t *src = a.c.pool + ((size_t)(chalf ? pages[1] : pages[0]) * a.c.heads + head) * hb + from +
                                 ((j0 + 16 * chalf) & (a.c.page - 1)) * per_key;
            bulk_copy(ring_at + slot * C::BYTES + to, src, copy_bytes, bar);
        }
        find(it + 1);
    };
    find(0);
#pragma unroll
    for (int it = 0; it < ST - 1; it++) load(it);

    // Q^T fragments: column g of block nt is row nt * 8 + g, scaled by a power of two to at most 2^14; the coordinates of
    // a word's second nibbles by 1/16 more
    uint32_t qf[QS][NT][NU][4];
    float fq[NT][2];                                // for this thread's columns 2 t, 2 t + 1: the factor of a score
    float qs[NT][LOW_MMA ? 1 : NG][2];           // and the groups' sums,
    uint32_t qlow[NT][2];                           // or their fragments: hi and lo of the sums times 2^-6
    int hi[NT][2], lo[NT][2];
    const int es = dtype == DT_F32 ? 4 : 2;
    const bool wide = !(((uintptr_t)a.q & 15) || ((a.q_row | a.q_head) * es) % 16);
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const int r = nt * 8 + g, i = (r0 + r) / each, hq = head * each + (r0 + r) % each;
        float x[NU][8] = {}, mx = 0.f;
        if (r < rows) {
            const long long at = (long long)(sr.first + i) * a.q_row + (long long)hq * a.q_head + 8 * t;
            load_runs<NU>(dtype, a.q, at, 32, wide, x);
#pragma unroll
            for (int u = 0; u < NU; u++)
#pragma unroll
                for (int j = 0; j < 8; j++) mx = fmaxf(mx, fabsf(x[u][j]));
        }
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // mx * 2^e in [2^13, 2^14) (below 2^-113 as near as f32 holds 2^-e)
        const int e = mx > 0.f ? min(126, 140 - (int)((__float_as_uint(mx) >> 23) & 0xff)) : 0;
        const float up = pow2i(e);
        float sum[NG] = {};
#pragma unroll
        for (int u = 0; u < NU; u++) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                x[u][j] *= a.scale < 0.f ? -up : up;
                sum[u / UG] += SPLIT ? x[u][j] : __half2float(__float2half_rn(x[u][j]));
            }
#pragma unroll
            for (int w = 0; w < 4; w++) {  // word w of the unit: coordinates w and w + 4
                const float f = w & 1 ? 0.0625f : 1.f, x0 = x[u][w] * f, x1 = x[u][w + 4] * f;
                qf[0][nt][u][w] = half2_bits(x0, x1);
                if (SPLIT) {
                    const float2 b = bits_float2(qf[0][nt][u][w]);
                    qf[QS - 1][nt][u][w] = half2_bits(x0 - b.x, x1 - b.y);
                }
            }
        }
        // (held to the normal numbers: positive for a scale of 0 too, so that the scores' order is that of the products and
        // -infinity stays itself)
        const float factor = fminf(fmaxf(fabsf(a.scale) * 1.44269504088896340736f * pow2i(-e) * UNIT, FLT_MIN), FLT_MAX);
#pragma unroll
        for (int k = 0; k < NG; k++) {
            sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 1);
            sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], 2);
            sum[k] *= LOW_MMA ? 0.015625f : 1.f / UNIT;  // as the products with the codes come
        }
        if constexpr (LOW_MMA) {
            uint32_t hi2[NG / 2], lo2[NG / 2];
#pragma unroll
            for (int k = 0; k < NG; k += 2) {
                hi2[k / 2] = half2_bits(sum[k], sum[k + 1]);
                const float2 b = bits_float2(hi2[k / 2]);
                lo2[k / 2] = half2_bits(sum[k] - b.x, sum[k + 1] - b.y);
            }
            if constexpr (NG == 4) {  // columns 0-3 hi, 4-7 lo
                qlow[nt][0] = t & 2 ? (t & 1 ? lo2[1] : lo2[0]) : (t & 1 ? hi2[1] : hi2[0]);
            } else {  // columns 0-7 hi, 8-15 lo
                qlow[nt][0] = t & 2 ? (t & 1 ? hi2[3] : hi2[2]) : (t & 1 ? hi2[1] : hi2[0]);
                qlow[nt][1] = t & 2 ? (t & 1 ? lo2[3] : lo2[2]) : (t & 1 ? lo2[1] : lo2[0]);
            }
        }
#pragma unroll
        for (int c = 0; c < 2; c++) {
            const int who = (2 * t + c) * 4;
            fq[nt][c] = __shfl_sync(0xffffffffu, factor, who);
            if constexpr (!LOW_MMA) {
#pragma unroll
                for (int k = 0; k < NG; k++) qs[nt][k][c] = __shfl_sync(0xffffffffu, sum[k], who);
            }
            const int ic = (r0 + nt * 8 + 2 * t + c) / each;
            hi[nt][c] = ka_hi(a, sr, ic), lo[nt][c] = ka_lo(a, sr, ic);
        }
    }

    // the running state of a column, in units of 2^off: off = m - 7 + ve, m the column's reference (it moves only when a score
    // passes it by 8), 2^ve the largest value step so far or more. So a weight is at most 2^(15 - ve), and with its step at
    // most 2^15: inside f16, and 2^7 above where the largest would leave small ones the least room. bf16's weights are
    // f16 before they meet their step too, so there `off` does not follow ve below 0; where it is below -6 the steps are taken
    // 2^steps_up as large instead, up to 2^15 (values of 4e-6 would lose all but 7 bits), and so is the output.
    float m[NT][2], off_m[NT][2], bound[NT][2], l[NT][2], ls[NT][NG][2], o[NT][NU][2][4];
    float ol[NT][4] = {};  // sums of p low of group g, where they are taken as a matrix product
    constexpr bool LOW_MMA_V = LOW_MMA;
    int ve = -24;  // (steps are f16: at least 2^-24)
    float vtop = pow2i(ve);
    auto weight_unit = [](int e) { return CENTRED ? e : max(e, 0); };
    auto steps_up = [](int e) { return CENTRED || e >= -6 ? 0 : min(-e, 15); };
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        off_m[nt][0] = off_m[nt][1] = (float)(weight_unit(ve) - 7);
        m[nt][0] = m[nt][1] = bound[nt][0] = bound[nt][1] = -INFINITY, l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int k = 0; k < NG; k++) ls[nt][k][0] = ls[nt][k][1] = 0.f;
#pragma unroll
        for (int u = 0; u < NU; u++)
#pragma unroll
            for (int x = 0; x < 8; x++) o[nt][u][x >> 2][x & 3] = 0.f;
    }

    for (int it = 0; it < mine; it++) {
        load(it + ST - 1);
        if (__any_sync(0xffffffffu, !ka_wait(bar_at + 8 * ((used + it) % ST), ((used + it) / ST) & 1))) {
            // copies on their way land before the memory holds anything else, or the block leaves it
            for (int x = it; x < min(mine, it + ST); x++) ka_wait(bar_at + 8 * ((used + x) % ST), ((used + x) / ST) & 1);
            gave_up = true;
            break;
        }
        const uint8_t *tile = ring + (used + it) % ST * C::BYTES;
        const int j0 = k0 + (warp + it * KA_WARPS) * KA_KEYS;
        const bool edge = j0 + KA_KEYS > hi_min || j0 < lo_max;
        float s[2][NT][4];
#pragma unroll
        for (int kb = 0; kb < 2; kb++) {
            uint32_t kw[2][NU], sc[2][NG];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int key = kb * 16 + h * 8 + g;
                lds_words<NU>(tile + key * (HD / 2) + t * NU * 4, kw[h]);
                lds_words<NG>(tile + C::KC + key * NG * 4, sc[h]);
            }
            float low[NT][4];
            if constexpr (LOW_MMA) {
                uint32_t lows[2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint2 v = *reinterpret_cast<const uint2 *>(tile + C::KC + (kb * 16 + h * 8 + g) * NG * 4 + (NG == 4 ? t & 1 : t) * 8);
                    lows[h] = __byte_perm(v.x, v.y, 0x7632);
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    low[nt][0] = low[nt][1] = low[nt][2] = low[nt][3] = 0.f;
                    if constexpr (NG == 4)
                        mma1688(low[nt], lows[0], lows[1], qlow[nt][0]);
                    else
                        mma16816(low[nt], lows[0], lows[1], lows[0], lows[1], qlow[nt][0], qlow[nt][1]);
                }
            }
#pragma unroll
            for (int k = 0; k < NG; k++) {
                float acc[NT][4] = {};
#pragma unroll
                for (int u = k * UG; u < (k + 1) * UG; u++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const uint32_t w0 = h ? kw[0][u] >> 8 : kw[0][u], w1 = h ? kw[1][u] >> 8 : kw[1][u];
                        const uint32_t a0 = code_pair<CENTRED, false>(w0), a1 = code_pair<CENTRED, false>(w1);
                        const uint32_t a2 = code_pair<CENTRED, true>(w0), a3 = code_pair<CENTRED, true>(w1);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int q = QS - 1; q >= 0; q--)
                                mma16816(acc[nt], a0, a1, a2, a3, qf[q][nt][u][2 * h], qf[q][nt][u][2 * h + 1]);
                    }
                float2 s0 = bits_float2(sc[0][k]), s1 = bits_float2(sc[1][k]);
                if (CENTRED) s0.y = fmaf(8.f, s0.x, s0.y), s1.y = fmaf(8.f, s1.x, s1.y);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        float &x = s[kb][nt][c], &y = s[kb][nt][c + 2];
                        if constexpr (LOW_MMA) {
                            x = k ? fmaf(s0.x, acc[nt][c], x) : s0.x * acc[nt][c];
                            y = k ? fmaf(s1.x, acc[nt][c + 2], y) : s1.x * acc[nt][c + 2];
                        } else {
                            x = fmaf(s0.x, acc[nt][c], k ? fmaf(s0.y, qs[nt][k][c], x) : s0.y * qs[nt][k][c]);
                            y = fmaf(s1.x, acc[nt][c + 2], k ? fmaf(s1.y, qs[nt][k][c], y) : s1.y * qs[nt][k][c]);
                        }
                    }
                }
            }
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 4; c++) {
                    // the lows' products are 2^18 times the codes'
                    if constexpr (LOW_MMA) s[kb][nt][c] = fmaf(low[nt][c], 3.814697265625e-6f, s[kb][nt][c]);
                }
        }
        // the value scales of this thread's four keys
        uint32_t vs[2][2][NG];
#pragma unroll
        for (int kb = 0; kb < 2; kb++)
#pragma unroll
            for (int h = 0; h < 2; h++) lds_words<NG>(tile + 2 * C::KC + C::SC + (kb * 16 + h * 8 + g) * NG * 4, vs[kb][h]);
        if (edge) {  // keys that a row does not see; of those that none sees, the scales may be anything
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int key = j0 + kb * 16 + h * 8 + g;
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int c = 0; c < 2; c++)
                            if (key >= hi[nt][c] || key < lo[nt][c]) s[kb][nt][2 * h + c] = -INFINITY;
                    if (key >= hi_max || key < lo_min) {
#pragma unroll
                        for (int k = 0; k < NG; k++) vs[kb][h][k] = 0;
                    }
                }
        }
        // the largest value step: a lane looks at one key's
        float step_max;
        {
            uint32_t w[NG];
            lds_words<NG>(tile + 2 * C::KC + C::SC + lane * NG * 4, w);
            __half2 x = *reinterpret_cast<const __half2 *>(&w[0]);
#pragma unroll
            for (int k = 1; k < NG; k++) x = __hmax2(x, *reinterpret_cast<const __half2 *>(&w[k]));
            step_max = __low2float(x);
            if (edge && (j0 + lane >= hi_max || j0 + lane < lo_min)) step_max = 0.f;
        }
        bool moves = step_max > vtop;
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int c = 0; c < 2; c++)
                moves |= fmaxf(fmaxf(s[0][nt][c], s[0][nt][c + 2]), fmaxf(s[1][nt][c], s[1][nt][c + 2])) > bound[nt][c];
        if (__any_sync(0xffffffffu, moves)) {
#pragma unroll
            for (int d = 1; d < 32; d *= 2) step_max = fmaxf(step_max, __shfl_xor_sync(0xffffffffu, step_max, d));
            int grow = 0;
            float out_f = 1.f;
            if (step_max > vtop) {  // the next power of two above
                const int e = (int)(__float_as_uint(step_max) >> 23) - 126;
                grow = weight_unit(e) - weight_unit(ve);
                if (!CENTRED) out_f = pow2i(steps_up(e) - steps_up(ve));
                ve = e, vtop = pow2i(e);
            }
#pragma unroll
            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    float x = fmaxf(fmaxf(s[0][nt][c], s[0][nt][c + 2]), fmaxf(s[1][nt][c], s[1][nt][c + 2]));
#pragma unroll
                    for (int d = 4; d < 32; d *= 2) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                    x = fmaxf(x * fq[nt][c], m[nt][c]);
                    bound[nt][c] = x == -INFINITY ? x : (x + 8.f) / fq[nt][c];
                    const float f = (x > m[nt][c] ? exp2_sfu(m[nt][c] - x) : 1.f) * pow2i(-grow);
                    m[nt][c] = x, off_m[nt][c] = (x == -INFINITY ? 0.f : x) + (float)(weight_unit(ve) - 7), l[nt][c] *= f, ol[nt][c] *= f;
#pragma unroll
                    for (int k = 0; k < NG; k++) ls[nt][k][c] *= f;
#pragma unroll
                    for (int u = 0; u < NU; u++)
#pragma unroll
                        for (int i = 0; i < 2; i++) o[nt][u][i][c] *= f * out_f, o[nt][u][i][c + 2] *= f * out_f;
                }
        }
        if (!CENTRED && steps_up(ve)) {
            const __half2 up = __floats2half2_rn(pow2i(steps_up(ve)), 1.f);
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
                for (int h = 0; h < 2; h++)
#pragma unroll
                    for (int k = 0; k < NG; k++) {
                        const __half2 x = __hmul2(*reinterpret_cast<const __half2 *>(&vs[kb][h][k]), up);
                        vs[kb][h][k] = *reinterpret_cast<const uint32_t *>(&x);
                    }
        }
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
#pragma unroll
                for (int kb = 0; kb < 2; kb++)
#pragma unroll
                    for (int h = 0; h < 4; h += 2) {
                        const float p = exp2_sfu(fmaf(s[kb][nt][c + h], fq[nt][c], -off_m[nt][c]));
                        s[kb][nt][c + h] = p, l[nt][c] += p;
                    }
            }
        // sum p low: as a matrix product below, or in f32
        if (!LOW_MMA_V || edge) {
#pragma unroll
            for (int kb = 0; kb < 2; kb++)
#pragma unroll
            for (int k = 0; k < NG; k++) {
                const float2 v0 = bits_float2(vs[kb][0][k]), v1 = bits_float2(vs[kb][1][k]);
                const float y0 = CENTRED ? fmaf(8.f, v0.x, v0.y) : v0.y, y1 = CENTRED ? fmaf(8.f, v1.x, v1.y) : v1.y;
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < 2; c++) {
                        const float p0 = s[kb][nt][c], p1 = s[kb][nt][c + 2];
                        if (edge)  // a weight of 0 meets a NaN only at a key that its row does not see
                            ls[nt][k][c] = fmaf(p0, p0 == 0.f ? 0.f : y0, fmaf(p1, p1 == 0.f ? 0.f : y1, ls[nt][k][c]));
                        else
                            ls[nt][k][c] = fmaf(p0, y0, fmaf(p1, y1, ls[nt][k][c]));
                    }
            }
        }
#pragma unroll
        for (int kb = 0; kb < 2; kb++) {
            // the half-words of keys 2 t, 2 t + 1 and 2 t + 8, 2 t + 9, a pair in one register
            uint32_t pair[2][NU];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint8_t *p = tile + C::KC + C::SC + (kb * 16 + h * 8 + 2 * t) * (HD / 2) + g * NU * 2;
                if constexpr (NU == 1) {
                    pair[h][0] = (uint32_t)*reinterpret_cast<const uint16_t *>(p) |
                                 (uint32_t)*reinterpret_cast<const uint16_t *>(p + HD / 2) << 16;
                } else {
                    uint32_t x[NU / 2], y[NU / 2];
                    lds_words<NU / 2>(p, x), lds_words<NU / 2>(p + HD / 2, y);
#pragma unroll
                    for (int u = 0; u < NU; u++) pair[h][u] = __byte_perm(x[u / 2], y[u / 2], u & 1 ? 0x7632 : 0x5410);
                }
            }
            __half2 p2[NT][2];
            if (!CENTRED) {
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int h = 0; h < 2; h++) p2[nt][h] = __floats2half2_rn(s[kb][nt][2 * h], s[kb][nt][2 * h + 1]);
            }
            if (LOW_MMA_V && !edge) {  // rows: the groups' lows of keys 2 t, 2 t + 1 and 2 t + 8, 2 t + 9
                uint32_t lows[2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const uint32_t *p = reinterpret_cast<const uint32_t *>(tile + 2 * C::KC + C::SC) + (kb * 16 + h * 8 + 2 * t) * NG + g % NG;
                    lows[h] = g < NG ? __byte_perm(p[0], p[NG], 0x7632) : 0u;
                }
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
                    mma16816(ol[nt], lows[0], 0u, lows[1], 0u, transpose8(*reinterpret_cast<const uint32_t *>(&p2[nt][0])),
                             transpose8(*reinterpret_cast<const uint32_t *>(&p2[nt][1])));
            }
#pragma unroll
            for (int k = 0; k < NG; k++) {
                uint32_t b[QS][NT][2];
                if constexpr (CENTRED) {
                    const float w[2] = {bits_float2(vs[kb][0][k]).x, bits_float2(vs[kb][1][k]).x};
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const float p0 = s[kb][nt][2 * h] * w[h], p1 = s[kb][nt][2 * h + 1] * w[h];
                            const uint32_t x = half2_bits(p0, p1);
                            b[0][nt][h] = transpose8(x);
                            if constexpr (SPLIT) {
                                const float2 f = bits_float2(x);
                                b[QS - 1][nt][h] = transpose8(half2_bits(p0 - f.x, p1 - f.y));
                            }
                        }
                } else {
                    // p and p * step each round to 11 bits, the results to 8
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const __half2 w = __low2half2(*reinterpret_cast<const __half2 *>(&vs[kb][h][k]));
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            const __half2 x = __hmul2(p2[nt][h], w);
                            b[0][nt][h] = transpose8(*reinterpret_cast<const uint32_t *>(&x));
                        }
                    }
                }
#pragma unroll
                for (int u = k * UG; u < (k + 1) * UG; u++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const uint32_t x = i ? pair[0][u] >> 8 : pair[0][u], y = i ? pair[1][u] >> 8 : pair[1][u];
                        const uint32_t a0 = code_pair<CENTRED, false>(x), a1 = code_pair<CENTRED, true>(x);
                        const uint32_t a2 = code_pair<CENTRED, false>(y), a3 = code_pair<CENTRED, true>(y);
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            if constexpr (SPLIT) {  // summed over the steps with rounding to nearest, which the matrix unit's sums are not
                                float y[4] = {};
#pragma unroll
                                for (int q = QS - 1; q >= 0; q--) mma16816(y, a0, a1, a2, a3, b[q][nt][0], b[q][nt][1]);
#pragma unroll
                                for (int x = 0; x < 4; x++) o[nt][u][i][x] += y[x];
                            } else {
                                mma16816(o[nt][u][i], a0, a1, a2, a3, b[0][nt][0], b[0][nt][1]);
                            }
                        }
                    }
            }
        }
        __syncwarp();  // every lane is done with the slot that the next load fills
    }
    used += mine;
    if (gave_up && lane == 0) *reinterpret_cast<volatile int *>(a.err_wait) = 1;

    // ---- the warps' states joined ----
    __syncthreads();
    float *so = reinterpret_cast<float *>(sm);  // [warp][R][HD]
    float *sms = so + KA_WARPS * R * HD;        // [warp][R]{m, l}
    const float unv = UNIT * pow2i(-steps_up(ve));
#pragma unroll
    for (int nt = 0; nt < NT; nt++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
            float x = l[nt][c], y[NG];
#pragma unroll
            for (int d = 4; d < 32; d *= 2) x += __shfl_xor_sync(0xffffffffu, x, d);
#pragma unroll
            for (int k = 0; k < NG; k++) {
                y[k] = ls[nt][k][c];
#pragma unroll
                for (int d = 4; d < 32; d *= 2) y[k] += __shfl_xor_sync(0xffffffffu, y[k], d);
                if (LOW_MMA_V) y[k] += __shfl_sync(0xffffffffu, ol[nt][c], k * 4 + t);
            }
            const int r = nt * 8 + 2 * t + c;
            if (g == 0) sms[(warp * R + r) * 2] = m[nt][c] == -INFINITY ? -INFINITY : off_m[nt][c], sms[(warp * R + r) * 2 + 1] = x;
            float *dst = so + (warp * R + r) * HD + 4 * g;
#pragma unroll
            for (int u = 0; u < NU; u++)
                *reinterpret_cast<float4 *>(dst + 32 * u) =
                    make_float4(fmaf(o[nt][u][0][c], unv, y[u / UG]), fmaf(o[nt][u][0][c + 2], unv * 0.0625f, y[u / UG]),
                                fmaf(o[nt][u][1][c], unv, y[u / UG]), fmaf(o[nt][u][1][c + 2], unv * 0.0625f, y[u / UG]));
        }
    __syncthreads();
    auto put = [&](int r, int x, float v) {
        const int i = (r0 + r) / each, hq = head * each + (r0 + r) % each;
        const long long at = (long long)(sr.first + i) * a.o_row + (long long)hq * a.o_head + x;
        if (dtype == DT_F32)
            reinterpret_cast<float *>(a.out)[at] = v;
        else if (dtype == DT_F16)
            reinterpret_cast<__half *>(a.out)[at] = __float2half_rn(v);
        else
            reinterpret_cast<__nv_bfloat16 *>(a.out)[at] = __float2bfloat16_rn(v);
    };
    auto put_lse = [&](int r, float M, float L) {
        if (a.lse)
            a.lse[(size_t)(sr.first + (r0 + r) / each) * a.q_heads + head * each + (r0 + r) % each] =
                (M + log2f(L)) * 0.69314718055994530942f;
    };
    const bool whole = piece == sp.steps;
    const size_t nslots = 2 * (size_t)gridDim.x, slot = Cut::slot(blockIdx.x, skip == 0);
    float *pms = part + 2 * slot * R, *po = part + 2 * nslots * R + slot * R * HD;
    for (int x = tid; x < rows * HD; x += KA_STEP) {
        const int r = x / HD, c = x % HD;
        float M = -INFINITY, L = 0.f, v = 0.f;
#pragma unroll
        for (int w = 0; w < KA_WARPS; w++) M = fmaxf(M, sms[(w * R + r) * 2]);
        const float M0 = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int w = 0; w < KA_WARPS; w++) {
            const float f = exp2_sfu(sms[(w * R + r) * 2] - M0);
            L = fmaf(sms[(w * R + r) * 2 + 1], f, L), v = fmaf(so[(w * R + r) * HD + c], f, v);
        }
        if (whole) {
            put(r, c, L != 0.f ? v / L : 0.f);  // L is 0 when no key is seen, NaN when a score is
            if (c == 0) put_lse(r, M0, L);
        } else {
            __stcg(po + x, v);
            if (c == 0) __stcg(pms + 2 * r, M), __stcg(pms + 2 * r + 1, L);
        }
    }
    if (!whole) {
        // ---- the last of the unit's blocks to arrive joins their states, in their order ----
        const int2 who = Cut::sharers(pl, pl.pos - skip, sp.steps);
        const int b0 = who.x, np = who.y;
        __threadfence();
        __syncthreads();
        if (tid == 0) {
            s_last = atomicAdd(arrived + b0, 1) == np - 1;  // (a block begins at most one unit that others go on with)
            if (s_last) arrived[b0] = 0;                    // ready for the next call
        }
        __syncthreads();
        if (s_last) {
            __threadfence();
            auto slot_of = [&](int p) { return Cut::slot(b0 + p, p == 0); };
            const float *po0 = part + 2 * nslots * R;
            // row by row; a warp sums every fourth part (eight in flight), the warps' sums are joined in shared memory
            float *sv = reinterpret_cast<float *>(sm);  // [2][warps][HD + 1]
            for (int r = 0; r < rows; r++) {
                float M = -INFINITY, L = 0.f;
                for (int p = lane; p < np; p += 32) M = fmaxf(M, __ldcg(part + 2 * (slot_of(p) * R + r)));
#pragma unroll
                for (int d = 1; d < 32; d *= 2) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, d));
                const float M0 = M == -INFINITY ? 0.f : M;
                float v[HD / 32] = {};
                for (int p0 = warp; p0 < np; p0 += 8 * KA_WARPS) {
                    float y[8][HD / 32];
                    float2 x[8];
#pragma unroll
                    for (int q = 0; q < 8; q++) {
                        const int p = p0 + q * KA_WARPS;
                        x[q] = p < np ? __ldcg(reinterpret_cast<const float2 *>(part) + slot_of(p) * R + r) : make_float2(-INFINITY, 0.f);
#pragma unroll
                        for (int k = 0; k < HD / 32; k++) y[q][k] = p < np ? __ldcg(po0 + (slot_of(p) * R + r) * HD + k * 32 + lane) : 0.f;
                    }
#pragma unroll
                    for (int q = 0; q < 8; q++) {
                        const float f = exp2_sfu(x[q].x - M0);
                        L = fmaf(x[q].y, f, L);
#pragma unroll
                        for (int k = 0; k < HD / 32; k++) v[k] = fmaf(y[q][k], f, v[k]);
                    }
                }
                float *mine_v = sv + ((r & 1) * KA_WARPS + warp) * (HD + 1);
#pragma unroll
                for (int k = 0; k < HD / 32; k++) mine_v[k * 32 + lane] = v[k];
                if (lane == 0) mine_v[HD] = L;
                __syncthreads();
                const float *all = sv + (r & 1) * KA_WARPS * (HD + 1);
                L = 0.f;
#pragma unroll
                for (int w = 0; w < KA_WARPS; w++) L += all[w * (HD + 1) + HD];
                for (int c = tid; c < HD; c += KA_STEP) {
                    float x = 0.f;
#pragma unroll
                    for (int w = 0; w < KA_WARPS; w++) x += all[w * (HD + 1) + c];
                    put(r, c, L != 0.f ? x / L : 0.f);
                }
                if (tid == 0) put_lse(r, M0, L);
            }
        }
    }
    // the next unit; its copies (the asynchronous proxy's) come after this one's reads and writes of the same memory
    Cut::next(pl, a, each, sr.n, piece);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    }
}

static int ka_nt(int dtype, const Kv4AttendArgs &a) {
    // 16 rows a block where their fragments of q and of the output fit the registers
    return a.max_rows * (a.q_heads / a.c.heads) > 8 && a.c.width * (dtype == DT_F32 ? 2 : 1) <= 128 ? 2 : 1;
}

// Many rows go to the tensor cores' kernels, from 41 rows a cache head on (32 sequences of 4096 keys, 8 heads: 24 rows take
// 149 us here and 186 there in bf16, 192 and 250 in f32; 48 rows 206 and 191, 361 and 256), where their units (row tiles of 128
// for f32, 256 for 16 bits) fill the GPU, or nearly and with work enough, or where the work outweighs the joining of units cut
// into many parts, which costs more there. us here and there, 8 heads of 128:
//     units 64 and more:  f32 1024 x 512  66, 53;  16 bits 2048 x 512  93, 59
//     32:                 f32 512 x 512  42, 51, 512 x 2048  82, 60;  16 bits 1024 x 512  61, 57, 1024 x 2048  95, 75
//     fewer:              f32 128 x 8192  76, 92, 256 x 8192  135, 93;  16 bits 256 x 8192  85, 130, 512 x 8192  131, 132;
//                         4 heads, f32 256 x 10,000  99, 119, 512 x 10,000  160, 119;  16 bits 512 x 10,000  95, 178
// (Working memory is asked for before causal and window are known, so the rule does not go by them.)
static bool ka_many(int dtype, const Kv4AttendArgs &a, int sms) {
    const long long rows = (long long)a.max_rows * (a.q_heads / a.c.heads), heads = (long long)a.seqs * a.c.heads;
    const long long tile = dtype == DT_F32 ? 128 : 256, units = heads * ((rows + tile - 1) / tile), pairs = heads * rows * a.max_len;
    return a.c.width <= 128 && rows > 40 &&
           (units * 4 >= sms || (units * 5 >= sms && pairs >= 3000000) || pairs >= (dtype == DT_F32 ? 12000000 : 36000000));
}

size_t kv4_attend_workspace(int dtype, const Kv4AttendArgs &a, int sms) {
    if (ka_many(dtype, a, sms)) return dtype == DT_F32 ? kv4_attend_tc_workspace(a, sms) : kv4_attend_tc16_workspace(a, sms);
    return 4 * (KA_BLOCKS + (size_t)std::min(KA_BLOCKS, 8 * sms) * 2 * 8 * ka_nt(dtype, a) * (a.c.width + 2));
}

template <int HD, int G, int NT, int TYPE>
static cudaError_t launch_one(const Kv4AttendArgs &a, int sms, void *work, cudaStream_t s) {
    using C = KaTile<HD, G>;
    const auto kernel = k_kv4_attend<HD, G, NT, TYPE>;
    const size_t join = sizeof(float) * KA_WARPS * 8 * NT * (HD + 2);
    const size_t smem = std::max((size_t)KA_WARPS * C::STAGES * C::BYTES, join);
    cudaError_t e = allow_dynamic_smem((const void *)kernel, smem);
    if (e != cudaSuccess) return e;
    static std::atomic<int> resident{0};  // blocks an SM holds
    if (!resident) {
        int n = 0;
        e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kernel, KA_STEP, smem);
        if (e != cudaSuccess) return e;
        resident = std::max(1, std::min(8, n));
    }
    // as many blocks as the GPU holds at once, at least one step each
    const long long rows = (long long)a.max_rows * (a.q_heads / a.c.heads), tiles = (rows + 8 * NT - 1) / (8 * NT);
    const long long most = std::max(1LL, ((long long)a.max_len + KA_STEP + KA_KEYS - 1) / KA_STEP) * tiles * a.seqs * a.c.heads;
    const int grid = (int)std::min<long long>({most, (long long)resident * sms, KA_BLOCKS});
    k_kv4_attend<HD, G, NT, TYPE><<<grid, KA_STEP, smem, s>>>(a, TYPE, 1, reinterpret_cast<float *>(work) + KA_BLOCKS,
                                                               reinterpret_cast<int *>(work));
    return cudaGetLastError();
}
template <int HD, int G, int TYPE>
static cudaError_t launch_type(const Kv4AttendArgs &a, int nt, int sms, void *work, cudaStream_t s) {
    if constexpr (HD * (TYPE == DT_F32 ? 2 : 1) <= 128) {
        if (nt == 2) return launch_one<HD, G, 2, TYPE>(a, sms, work, s);
    }
    return launch_one<HD, G, 1, TYPE>(a, sms, work, s);
}
template <int HD, int G>
static cudaError_t launch_size(int dtype, const Kv4AttendArgs &a, int nt, int sms, void *work, cudaStream_t s) {
    if (dtype == DT_F32) return launch_type<HD, G, DT_F32>(a, nt, sms, work, s);
    return dtype == DT_F16 ? launch_type<HD, G, DT_F16>(a, nt, sms, work, s) : launch_type<HD, G, DT_BF16>(a, nt, sms, work, s);
}

cudaError_t launch_kv4_attend(int dtype, const Kv4AttendArgs &a, int sms, void *work, size_t work_bytes, cudaStream_t s, uint64_t *launches) {
    if (!a.seqs || !a.rows || !a.max_rows) return cudaSuccess;
    if (kv4_attend_workspace(dtype, a, sms) > work_bytes) return cudaErrorInvalidValue;
    if (launches) ++*launches;
    if (ka_many(dtype, a, sms)) return dtype == DT_F32 ? launch_kv4_attend_tc(a, sms, work, s) : launch_kv4_attend_tc16(dtype, a, sms, work, s);
    const int nt = ka_nt(dtype, a);
    cudaError_t e = cudaErrorInvalidValue;
    const int w = a.c.width, g = a.c.group;
    if (w == 32) e = launch_size<32, 32>(dtype, a, nt, sms, work, s);
    if (w == 64) e = g == 32 ? launch_size<64, 32>(dtype, a, nt, sms, work, s) : launch_size<64, 64>(dtype, a, nt, sms, work, s);
    if (w == 128)
        e = g == 32 ? launch_size<128, 32>(dtype, a, nt, sms, work, s)
                    : g == 64 ? launch_size<128, 64>(dtype, a, nt, sms, work, s) : launch_size<128, 128>(dtype, a, nt, sms, work, s);
    if (w == 256)
        e = g == 32 ? launch_size<256, 32>(dtype, a, nt, sms, work, s)
                    : g == 64 ? launch_size<256, 64>(dtype, a, nt, sms, work, s) : launch_size<256, 128>(dtype, a, nt, sms, work, s);
    return e;
}

}  // namespace tcu

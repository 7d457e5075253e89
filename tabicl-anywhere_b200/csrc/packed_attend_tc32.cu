// Attention of many packed f32 rows on the 5th-generation tensor cores (tcgen05).
//
// Each f32 operand is the sum of two f16 (22 bits), and a product is hi hi + hi lo + lo hi. Keys and values are split once, by a
// kernel before, into tiles of 64 keys of one head as the matrix unit reads them, each tile scaled by a power of two of its own
// that keeps it inside f16; every block of 128 query rows of that head then brings them by two copies a step.
// 128 query rows of one key head (the heads that share it side by side) against 64 keys at a time: S = Q K^T with Q in tensor
// memory; the weights P, relative to a number of the step's own, go back to tensor memory over S and multiply the values; each step's
// P V is folded into the output in registers, in a unit of the row's own, so every sum across steps is taken in f32 with rounding to nearest (the matrix unit's own accumulation is not: over
// 10,000 keys it would cost 2.8e-5 of an output). As in the attention over the four-bit cache (kv4_attend_tc.cu), whose two
// warpgroups that widen codes are not needed here.
// 2048 rows over 10,000 keys, 4 heads of 128: 164 us, 0.26 PFLOP/s of scores and sums (0.76 of products), 15 of them the split; by
// warps' products (packed_attend.cu) 1040. Bound by latency: a step's products, softmax and fold follow one another.
#include <algorithm>

#include "kv4_tc.cuh"
#include "packed.cuh"

namespace tcu {

constexpr int PS_BQ = 128, PS_BK = 64, PS_NS = 3, PS_THREADS = 384;
constexpr int PS_STEPS = 8;  // steps a block takes at least
constexpr int PS_EXTRA = 2;  // what a unit costs besides its steps, in steps
constexpr int PS_T = 13;     // split values are below 2^T
constexpr int NONE = -4000;  // the exponent of a unit that nothing has
constexpr uint32_t PS_TQ = 0, PS_TS = 128, PS_TO = 384;

template <int HD>
struct PsShape {
    static constexpr int BLOCK = PS_BK * HD;  // f16 of one operand block
    static constexpr size_t TILE = (size_t)4 * BLOCK * 2;  // bytes of a tile: keys, their rest, values, their rest
    static constexpr size_t SMEM = (size_t)PS_NS * TILE + 1024;
};
// Where sequence seq's tile i lies: tiles of a sequence begin at a place that no other's reach.
__host__ __device__ inline long long ps_slots(int k_rows, int seqs) { return (long long)k_rows / PS_BK + seqs; }
__device__ __forceinline__ long long ps_tile(const PackedArgs &a, int seq, int head, int i) {
    return (long long)head * ps_slots(a.k_rows, a.seqs) + a.k_starts[seq] / PS_BK + seq + i;
}

// A block splits one tile, found by its sequence and place in that (the grid's third coordinate and its first), or, where that would
// be mostly blocks of nothing (sequences much shorter than the longest may be), by where it lies among all, whose sequence the block's
// threads look for: 1000 sequences of 100 keys, of which one might have had 100,000, 3.5 ms by the first and 0.4 by the second.
// Rows behind a sequence's end are zeros.
template <int HD>
__global__ void __launch_bounds__(256) k_packed_split(PackedArgs a, uint8_t *tiles, int2 *units, int wide, int by_place) {
    using C = PsShape<HD>;
    extern __shared__ __align__(16) uint8_t sm[];
    __shared__ float top[2][8];
    __shared__ int s_seq;
    const int head = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int seq = blockIdx.z, tile = blockIdx.x;
    if (by_place) {
        if (tid == 0) s_seq = -1;
        __syncthreads();
        for (int i = tid; i < a.seqs; i += 256) {
            const KaRows s = ka_rows(a, i);
            const int from = tile - (a.k_starts[i] / PS_BK + i);
            if (s.ok && from >= 0 && from * PS_BK < s.len) s_seq = i;
        }
        __syncthreads();
        seq = s_seq;
        if (seq < 0) return;
        tile -= a.k_starts[seq] / PS_BK + seq;
    }
    const KaRows sr = ka_rows(a, seq);
    if (!sr.ok || !sr.n || tile * PS_BK >= sr.len) return;
    constexpr int LANES = HD / 4, ROWS = 256 / LANES, N = PS_BK / ROWS;  // threads a row, rows at a time, rows a thread
    const int c = tid % LANES * 4, r0 = tid / LANES;
    const long long k0 = a.k_starts[seq];
    float4 v[2][N];
    float mx[2] = {0.f, 0.f};
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const float *base = reinterpret_cast<const float *>(x ? a.v : a.k) + head * (x ? a.v_head : a.k_head) + c;
        const long long row = x ? a.v_row : a.k_row;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int j = tile * PS_BK + r0 + i * ROWS;
            v[x][i] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (j < sr.len && c < a.width) {
                const float *p = base + (k0 + j) * row;
                v[x][i] = wide >> x & 1 ? __ldg(reinterpret_cast<const float4 *>(p)) : make_float4(p[0], p[1], p[2], p[3]);
            }
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float m = fmaxf(fmaxf(fabsf(v[x][i].x), fabsf(v[x][i].y)), fmaxf(fabsf(v[x][i].z), fabsf(v[x][i].w)));
            // (the largest finite value: a row of the tile with an infinity is worked out by itself where it is seen)
            if (finite_f(m))
                mx[x] = fmaxf(mx[x], m);
            else
                for (float f : {v[x][i].x, v[x][i].y, v[x][i].z, v[x][i].w})
                    if (finite_f(f)) mx[x] = fmaxf(mx[x], fabsf(f));
        }
        mx[x] = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(mx[x])));
        if (lane == 0) top[x][warp] = mx[x];
    }
    __syncthreads();
    int e[2];
#pragma unroll
    for (int x = 0; x < 2; x++) {
        float m = 0.f;
#pragma unroll
        for (int w = 0; w < 8; w++) m = fmaxf(m, top[x][w]);
        // m < 2^e, held to powers of two whose scales f32 holds (a tile of less than 2^-110 is then small beside 2^T, no more)
        e[x] = max(-110, (int)(__float_as_uint(m) >> 23) - 126);
    }
    __half *out = reinterpret_cast<__half *>(sm);
#pragma unroll
    for (int x = 0; x < 2; x++) {
        const float up = kt_pow2(PS_T - e[x]);
#pragma unroll
        for (int i = 0; i < N; i++) {
            const int r = r0 + i * ROWS;
            uint32_t hi[2], lo[2];
            split_pair(v[x][i].x * up, v[x][i].y * up, hi[0], lo[0]), split_pair(v[x][i].z * up, v[x][i].w * up, hi[1], lo[1]);
            __half *to = out + 2 * x * C::BLOCK + (x ? mnmajor_off(c, r, HD) : kmajor_off(r, c, PS_BK));
            *reinterpret_cast<uint2 *>(to) = make_uint2(hi[0], hi[1]), *reinterpret_cast<uint2 *>(to + C::BLOCK) = make_uint2(lo[0], lo[1]);
        }
    }
    __syncthreads();
    const long long at = ps_tile(a, seq, head, tile);
    uint4 *to = reinterpret_cast<uint4 *>(tiles + at * C::TILE);
    for (int i = tid; i < (int)(C::TILE / 16); i += 256) to[i] = reinterpret_cast<const uint4 *>(sm)[i];
    if (tid == 0) units[at] = make_int2(e[0], e[1]);
}

// Warps 0-3: softmax, a thread a query row; warps 4-7: the fold of each step's P V, a thread a row; warps 8, 9 issue the S products
// of even and odd steps, warp 10 the P V products; warp 11: the copies. They hand over through mbarriers; every wait is bounded,
// and one that gives up raises the block's abort flag, after which every wait returns at once, nothing more is asked for, and the roles,
// which walk the same pieces of units and meet at the same barriers, run to the end without results.
template <int HD>
__global__ void __launch_bounds__(PS_THREADS, 1) k_packed_attend_tc32(PackedArgs a, const uint8_t *tiles, const int2 *units, float *part, int *arrived) {
    using C = PsShape<HD>;
    using Cut = KaCut<PS_BQ, PS_BK, PS_BK, PS_EXTRA>;
    constexpr int BQ = PS_BQ, BK = PS_BK, NS = PS_NS, BLOCK = C::BLOCK;
    extern __shared__ uint8_t smraw[];
    __shared__ float2 fr[4][BQ];
    __shared__ float rowx[2][BQ], qmax[2][BQ];
    __shared__ int teK[8], teV[8];
    __shared__ __align__(8) uint64_t mK[NS], mV[NS], mKfree[NS], mVfree[NS], mS[NS], mP[NS], mSlot[NS], mF[4], mPV, mOfree, mDone[3];
    __shared__ uint32_t tslot;
    __shared__ volatile int abort_flag;
    __shared__ int s_unit[4], s_last;
    // for the rows that are worked out again at the end: where the block's pieces began, the units that it has joined, whether some
    // of its outputs are NaN
    __shared__ typename Cut::Place s_place;
    __shared__ int s_joined[2], s_dirty;
    __shared__ volatile int s_bad;
    __shared__ long long s_sum[PS_THREADS / 32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wg = warp >> 2, row = tid & (BQ - 1);
    const int each = a.q_heads / a.c.heads;
    auto pl = Cut::template place<PS_THREADS>(a, each, PS_STEPS, s_sum, s_unit);
    if (pl.pos >= pl.end) return;
    if (warp == 8) {
        tmem_alloc(&tslot, 512);
        tmem_relinquish();
    }
    if (tid == 0) {
        for (int i = 0; i < NS; i++) {
            mbar_init(&mK[i], 1), mbar_init(&mV[i], 1), mbar_init(&mKfree[i], 1), mbar_init(&mVfree[i], 1);
            mbar_init(&mS[i], 1), mbar_init(&mP[i], BQ), mbar_init(&mSlot[i], 1);
        }
        for (int i = 0; i < 4; i++) mbar_init(&mF[i], BQ);
        mbar_init(&mPV, 1), mbar_init(&mOfree, BQ);
        for (int i = 0; i < 3; i++) mbar_init(&mDone[i], 1);
        mbar_init_fence();
        abort_flag = a.give_up & blockIdx.x & 1, s_joined[0] = s_joined[1] = s_bad = 0, s_place = pl;
    }
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = tslot, lane_base = (uint32_t)((warp & 3) * 32) << 16;
    __half *ring = reinterpret_cast<__half *>(smraw + ((1024u - (smem_addr(smraw) & 1023u)) & 1023u));  // [NS]{keys, rest, values, rest}
    auto wait_warp = [&](uint64_t *m, uint32_t parity) {
        if (!mbar_test_wait(m, parity) && !abort_flag && !mbar_wait(m, parity, KT_WAIT)) abort_flag = 1;
        __syncwarp();
    };
    // A piece of a unit: `count` of its steps as they are cut, n of keys, the first at key j0.
    struct Piece {
        int count, n, j0;
    };
    auto piece = [&](const typename Cut::Span &sp) {
        Piece p;
        p.count = (int)min((long long)(sp.steps - pl.skip), pl.end - pl.pos);
        const int from = max(0, pl.skip - PS_EXTRA);
        p.n = sp.hi_max > sp.lo_min ? max(0, pl.skip + p.count - PS_EXTRA) - from : 0, p.j0 = sp.base + from * BK;
        return p;
    };
    // Q of a piece: each of two threads (softmax and fold) half a row, scaled by a power of two of the row's to at most 2^14,
    // into tensor memory. Returns what a product with the split keys is multiplied by (with the tile's power of two) to be a
    // score in units of log2.
    auto put_q = [&](const KaRows &sr, int ri, int hq) {
        constexpr int H = HD / 2;
        float q[H / 8][8], mx = 0.f;
        const bool wide = !(((uintptr_t)a.q & 15) || ((a.q_row | a.q_head) & 3));
        const float *from = reinterpret_cast<const float *>(a.q) + (long long)(sr.first + ri) * a.q_row + (long long)hq * a.q_head + wg * H;
#pragma unroll
        for (int b = 0; b < H / 8; b++) {
#pragma unroll
            for (int x = 0; x < 8; x++) q[b][x] = 0.f;
            if (wg * H + 8 * b < a.width) load8<DT_F32>(from + 8 * b, wide, q[b]);
#pragma unroll
            for (int x = 0; x < 8; x++) mx = fmaxf(mx, finite_f(q[b][x]) ? fabsf(q[b][x]) : 0.f);
        }
        kt_bar(2, 256);  // the last piece's epilogue is done with the exchange
        qmax[wg][row] = mx;
        kt_bar(2, 256);
        mx = fmaxf(qmax[0][row], qmax[1][row]);
        const int e = mx > 0.f ? min(126, 140 - (int)((__float_as_uint(mx) >> 23) & 0xff)) : 0;
        const float up = a.scale < 0.f ? -kt_pow2(e) : kt_pow2(e);
        const float rowfac = fabsf(a.scale) * 1.44269504088896340736f * kt_pow2(-e);
        uint32_t hi[H / 2], lo[H / 2];
#pragma unroll
        for (int b = 0; b < H / 8; b++)
#pragma unroll
            for (int x = 0; x < 4; x++) split_pair(q[b][2 * x] * up, q[b][2 * x + 1] * up, hi[4 * b + x], lo[4 * b + x]);
        const uint32_t tq = tmem + lane_base + PS_TQ + wg * (H / 2);
        if constexpr (H / 2 == 32)
            tmem_st32u(tq, hi), tmem_st32u(tq + HD / 2, lo);
        else
            tmem_st16u(tq, hi), tmem_st16u(tq + HD / 2, lo);
        tmem_wait_st();
        fence_before_sync();
        kt_bar(1, 352);
        fence_after_sync();
        return rowfac;
    };
    int at = 0;  // steps before the piece's

    if (wg == 2) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 120;");
        if (warp == 11) {
            int asked = 0;  // steps whose copies have been asked for
            while (pl.pos < pl.end) {
                const KaRows sr = ka_rows(a, pl.seq);
                const auto sp = Cut::span(a, sr, each, pl.rt);
                const Piece p = piece(sp);
                const long long first = ps_tile(a, pl.seq, pl.head, p.j0 / BK);
                for (int i = 0; i < p.n; i++, at++) {
                    const int slot = at % NS;
                    const uint32_t ph = (uint32_t)(at / NS) & 1u;
                    const int2 e = __ldg(units + first + i);
                    if (at >= NS) wait_warp(&mKfree[slot], ph ^ 1u), wait_warp(&mVfree[slot], ph ^ 1u);
                    if (__any_sync(0xffffffffu, abort_flag != 0)) continue;
                    asked++;
                    if (lane == 0) {
                        // (read by the softmax and the fold after they have seen products of this step; four steps on they are done with it)
                        *reinterpret_cast<volatile int *>(&teK[at & 7]) = e.x, *reinterpret_cast<volatile int *>(&teV[at & 7]) = e.y;
                        const uint8_t *from = tiles + (first + i) * C::TILE;
                        for (int x = 0; x < 2; x++) {
                            uint64_t *m = x ? &mV[slot] : &mK[slot];
                            asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}\n" ::"r"(smem_addr(m)), "r"((uint32_t)(C::TILE / 2)) : "memory");
                            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                                             smem_addr(ring + (size_t)slot * 4 * BLOCK + 2 * x * BLOCK)),
                                         "l"(from + x * (C::TILE / 2)), "r"((uint32_t)(C::TILE / 2)), "r"(smem_addr(m))
                                         : "memory");
                        }
                    }
                    __syncwarp();
                }
                Cut::next(pl, a, each, sr.n, p.count);
            }
            // what was asked for lands before the block lets go of shared memory
            for (int i = max(0, asked - NS); i < asked; i++) {
                mbar_wait(&mK[i % NS], (uint32_t)(i / NS) & 1u, KT_WAIT);
                mbar_wait(&mV[i % NS], (uint32_t)(i / NS) & 1u, KT_WAIT);
            }
        } else {
            const uint32_t idS = idesc_f16(BQ, BK, 0, 0), idO = idesc_f16(BQ, HD, 0, 1);
            const uint64_t dK0 = kstep_desc(ring, BK, 0), dV0 = kstep_desc(ring + 2 * BLOCK, HD, 0);
            constexpr uint64_t stK = (2 * (BK / 8) * 128) >> 4, stV = (2 * (HD / 8) * 128) >> 4, lo_off = (BLOCK * 2) >> 4, slot_off = (4 * BLOCK * 2) >> 4;
            while (pl.pos < pl.end) {
                const KaRows sr = ka_rows(a, pl.seq);
                const auto sp = Cut::span(a, sr, each, pl.rt);
                const Piece p = piece(sp);
                kt_bar(1, 352);  // Q is in tensor memory
                fence_after_sync();
                for (int i = at; i < at + p.n; i++) {
                    const int sl = i % NS;
                    const uint32_t ph = (uint32_t)(i / NS) & 1u;
                    if (warp < 10) {
                        // (the even steps' warp and the odd steps' each wait for their own steps alone: a slot's turn comes again only
                        // after both have seen the steps between)
                        if ((i & 1) != warp - 8) continue;
                        if (i >= NS) wait_warp(&mSlot[sl], ph ^ 1u);
                        wait_warp(&mK[sl], ph);
                        fence_after_sync();
                        const uint32_t tS = tmem + PS_TS + BK * sl;
                        const uint64_t dh = dK0 + sl * slot_off, dl = dh + lo_off;
                        if (elect_one()) {
#pragma unroll
                            for (int k = 0; k < HD / 16; k++) mma_f16_ta(tS, tmem + PS_TQ + 8 * k, dl + k * stK, idS, k > 0 ? 1u : 0u);
#pragma unroll
                            for (int k = 0; k < HD / 16; k++) mma_f16_ta(tS, tmem + PS_TQ + HD / 2 + 8 * k, dh + k * stK, idS, 1);
#pragma unroll
                            for (int k = 0; k < HD / 16; k++) mma_f16_ta(tS, tmem + PS_TQ + 8 * k, dh + k * stK, idS, 1);
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
                        const uint32_t pA = tmem + PS_TS + BK * sl, tO = tmem + PS_TO;
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
                at += p.n;
                Cut::next(pl, a, each, sr.n, p.count);
            }
            if (elect_one()) {  // every product issued here completes before the block lets go of its memory
                mma_commit(&mDone[warp - 8]);
                mbar_wait(&mDone[warp - 8], 0, KT_WAIT);
            }
            __syncwarp();
        }
    } else if (wg == 0) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 152;");
        while (pl.pos < pl.end) {
            const KaRows sr = ka_rows(a, pl.seq);
            const auto sp = Cut::span(a, sr, each, pl.rt);
            const Piece p = piece(sp);
            const int r0 = pl.rt * BQ, rows = min(BQ, sr.n * each - r0);
            const int r = min(row, rows - 1), ri = (r0 + r) / each, hq = pl.head * each + (r0 + r) % each;  // rows past the end repeat the last
            const int my_hi = ka_hi(a, sr, ri) - p.j0, my_lo = ka_lo(a, sr, ri) - p.j0;
            const float rowfac = put_q(sr, ri, hq);
            // ---- softmax: S(i) -> P(i) = 2^(S - r), r 14 below the step's largest, over S(i), and the factors of what was before and of the step ----
            float mrun = -INFINITY, lrun = 0.f;
#pragma unroll 1
            for (int i = at; i < at + p.n; i++) {
                const int sl = i % NS, key0 = (i - at) * BK;
                wait_warp(&mS[sl], (uint32_t)(i / NS) & 1u);
                fence_after_sync();
                const uint32_t tsp = tmem + lane_base + PS_TS + BK * sl;
                float x[64];
                tmem_ld32(tsp, *reinterpret_cast<float (*)[32]>(&x[0])), tmem_ld32(tsp + 32, *reinterpret_cast<float (*)[32]>(&x[32]));
                // (held to the normal numbers: positive for a scale of 0 too, so that -infinity stays itself)
                const float c1 = fminf(fmaxf(rowfac * kt_pow2(*reinterpret_cast<volatile int *>(&teK[i & 7]) - PS_T), FLT_MIN), FLT_MAX);
                tmem_wait_ld();
#pragma unroll
                for (int k = 0; k < 64; k += 8)
                    asm volatile("" : "+f"(x[k]), "+f"(x[k + 1]), "+f"(x[k + 2]), "+f"(x[k + 3]), "+f"(x[k + 4]), "+f"(x[k + 5]), "+f"(x[k + 6]), "+f"(x[k + 7])::"memory");
                if (__any_sync(0xffffffffu, key0 < my_lo || key0 + BK > my_hi)) {
                    const int low = my_lo - key0, high = my_hi - key0;
#pragma unroll
                    for (int k = 0; k < 64; k++)
                        if (k < low || k >= high) x[k] = -INFINITY;
                }
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int k = 0; k < 64; k++) top[k & 3] = fmaxf(top[k & 3], x[k]);
                const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
                // (weights beside a number of the step's own: a step far below the row's largest keeps its bits, for values may be as far
                // above; 2^14 for the largest, so that small ones keep theirs; of scores that do not resolve 14, 1. The step's factor knows
                // which it was; a multiplication by 2^14 for each weight takes 2% longer.)
                const float mstep = __fmul_rn(mx, c1), mnew = fmaxf(mrun, mstep), mm = mstep == -INFINITY ? 0.f : fabsf(mstep) < 1048576.f ? mstep - 14.f : mstep;
                const float f = mrun == -INFINITY ? 0.f : kt_ex2(mrun - mnew), h = mstep == -INFINITY ? 0.f : kt_ex2(mm - mnew);
                float psum[4] = {};
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    uint32_t w[32];
#pragma unroll
                    for (int k = 0; k < 32; k++) {
                        // (the product rounded as the largest's was: of scores past 2^23 the rest would be more than 1)
                        x[32 * b + k] = kt_ex2(__fmul_rn(x[32 * b + k], c1) - mm);
                        psum[k & 3] += x[32 * b + k];
                    }
                    // P goes where the scores were: of every 16 keys, hi and lo
#pragma unroll
                    for (int k = 0; k < 16; k++) split_pair(x[32 * b + 2 * k], x[32 * b + 2 * k + 1], w[k / 8 * 16 + k % 8], w[k / 8 * 16 + 8 + k % 8]);
                    tmem_st32u(tsp + 32 * b, w);
                }
                tmem_wait_st();
                fr[i & 3][row] = make_float2(f, h);
                fence_before_sync();
                mbar_arrive(&mP[sl]);
                mbar_arrive(&mF[i & 3]);
                lrun = fmaf(lrun, f, ((psum[0] + psum[1]) + (psum[2] + psum[3])) * h);
                mrun = mnew;
            }
            rowx[0][row] = mrun, rowx[1][row] = lrun;
            kt_bar(2, 256);
            at += p.n;
            Cut::next(pl, a, each, sr.n, p.count);
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        while (pl.pos < pl.end) {
            const KaRows sr = ka_rows(a, pl.seq);
            const auto sp = Cut::span(a, sr, each, pl.rt);
            const Piece p = piece(sp);
            const int r0 = pl.rt * BQ, rows = min(BQ, sr.n * each - r0);
            const int r = min(row, rows - 1), ri = (r0 + r) / each, hq = pl.head * each + (r0 + r) % each;  // rows past the end repeat the last
            put_q(sr, ri, hq);
            // ---- fold: O = O f + P V h, O in a unit of the row's, a power of two ----
            float o[HD];
            int unit = NONE;
#pragma unroll
            for (int k = 0; k < HD; k++) o[k] = 0.f;
#pragma unroll 1
            for (int i = at; i < at + p.n; i++) {
                wait_warp(&mPV, (uint32_t)i & 1u);
                wait_warp(&mF[i & 3], (uint32_t)(i >> 2) & 1u);
                fence_after_sync();
                const int e = *reinterpret_cast<volatile int *>(&teV[i & 7]);
                // Each side in its own unit (the factors' powers of two go there), then both in the larger of the two, what is far below gone.
                // A factor of 0 (keys that are not seen, scores far below) has no unit: it has no say in that.
                const float2 fh = fr[i & 3][row];
                auto level = [](float x, int &exponent) {
                    const uint32_t w = __float_as_uint(x);
                    exponent = w ? (int)(w >> 23) - 127 : NONE;
                    return w ? __uint_as_float((w & 0x7fffffu) | 0x3f800000u) : 0.f;
                };
                int old, step;
                float f = level(fh.x, old), g = level(fh.y, step);
                old += unit, step += e, unit = max(max(old, step), NONE);
                f = old < unit - 126 ? 0.f : f * kt_pow2(old - unit), g = step < unit - 126 ? 0.f : g * kt_pow2(step - unit);
#pragma unroll
                for (int c = 0; c < HD / 32; c++) {
                    float x[32];
                    tmem_ld32(tmem + lane_base + PS_TO + 32 * c, x);
                    tmem_wait_ld32(x);
#pragma unroll
                    for (int k = 0; k < 32; k++) o[32 * c + k] = fmaf(o[32 * c + k], f, x[k] * g);
                }
                fence_before_sync();
                mbar_arrive(&mOfree);
            }
            kt_bar(2, 256);
            // ---- the row's output, or its part of it ----
            const bool whole = p.count == sp.steps;
            float M = rowx[0][row], L = rowx[1][row];
            // (divided by the sum before it leaves its unit, a part too: the weighted sum of values near f32's largest may pass that)
            unit -= PS_T;
            const float un0 = unit < -252 ? 0.f : kt_pow2(unit / 2), un1 = unit < -252 ? 0.f : kt_pow2(unit - unit / 2);
            auto inverse = [](float sum) { return sum != 0.f ? 1.f / sum : 0.f; };  // 0 when no key is seen, NaN when a score is
            const float inv = inverse(L);
#pragma unroll
            for (int k = 0; k < HD; k++) o[k] = o[k] * inv * un0 * un1;
            bool write = row < rows;
            if (!whole) {
                const int2 who = Cut::sharers(pl, pl.pos - pl.skip, sp.steps);
                float *po = part + 2 * (size_t)2 * gridDim.x * BQ;  // outputs: 4 columns of all rows, then the next 4
                const size_t slot = Cut::slot(blockIdx.x, pl.skip == 0), mine = slot * BQ + row;
                __stcg(reinterpret_cast<float2 *>(part) + mine, make_float2(M, L));
#pragma unroll
                for (int k = 0; k < HD; k += 4)
                    __stcg(reinterpret_cast<float4 *>(po + slot * BQ * HD + (k / 4 * BQ + row) * 4), make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]));
                __threadfence();
                kt_bar(3, 128);
                if (row == 0) {
                    s_last = atomicAdd(arrived + who.x, 1) == who.y - 1;
                    if (s_last) arrived[who.x] = 0, s_joined[pl.skip == 0] = 1;  // ready for the next call
                }
                kt_bar(3, 128);
                write = write && s_last;
                if (write) {
                    __threadfence();
                    M = -INFINITY, L = 0.f;
                    for (int b = 0; b < who.y; b++) M = fmaxf(M, __ldcg(reinterpret_cast<const float2 *>(part) + Cut::slot(who.x + b, b == 0) * BQ + row).x);
                    auto weight = [&](float2 x) { return x.x == -INFINITY ? x.y : x.y * kt_ex2(x.x - M); };  // (without keys 0, and a NaN sum stays one)
                    for (int b = 0; b < who.y; b++) L += weight(__ldcg(reinterpret_cast<const float2 *>(part) + Cut::slot(who.x + b, b == 0) * BQ + row));
                    const float all = inverse(L);
#pragma unroll
                    for (int k = 0; k < HD; k++) o[k] = 0.f;
                    for (int b = 0; b < who.y; b++) {
                        const size_t from = Cut::slot(who.x + b, b == 0);
                        const float2 x = __ldcg(reinterpret_cast<const float2 *>(part) + from * BQ + row);
                        if (x.x == -INFINITY && x.y == 0.f) continue;
                        const float f = weight(x) * all;
#pragma unroll
                        for (int k = 0; k < HD; k += 4) {
                            const float4 y = __ldcg(reinterpret_cast<const float4 *>(po + from * BQ * HD + (k / 4 * BQ + row) * 4));
                            o[k] = fmaf(y.x, f, o[k]), o[k + 1] = fmaf(y.y, f, o[k + 1]);
                            o[k + 2] = fmaf(y.z, f, o[k + 2]), o[k + 3] = fmaf(y.w, f, o[k + 3]);
                        }
                    }
                }
            }
            bool bad = false;
            if (write && !abort_flag) {
                const bool wide = !(((uintptr_t)a.out & 15) || ((a.o_row | a.o_head) & 3));
                float *to = reinterpret_cast<float *>(a.out) + (long long)(sr.first + ri) * a.o_row + (long long)hq * a.o_head;
#pragma unroll
                for (int b = 0; b < HD; b += 8) {
                    if (b >= a.width) break;
                    float v[8];
#pragma unroll
                    for (int x = 0; x < 8; x++) v[x] = L != 0.f ? o[b + x] : 0.f, bad |= v[x] != v[x];
                    store8<DT_F32>(to + b, wide, v);
                }
                if (a.lse) a.lse[(size_t)(sr.first + ri) * a.q_heads + hq] = ((M == -INFINITY ? 0.f : M) + log2f(L)) * 0.69314718055994530942f;
            }
            if (bad) s_bad = 1;
            at += p.n;
            Cut::next(pl, a, each, sr.n, p.count);
        }
    }
    fence_before_sync();
    __syncthreads();
    if (tid == 0 && abort_flag) *reinterpret_cast<volatile int *>(a.err_wait) = 1;
    fence_after_sync();
    if (warp == 8) tmem_dealloc(tmem, 512);
    if (wg == 1 && s_bad && !abort_flag) pa_mend<DT_F32, HD, PS_BQ, PS_BK, PS_EXTRA, 4, Cut>(a, s_place, s_joined, false, 1.f, &s_dirty);
}

// Working memory: counters, parts, the tiles' powers of two, the tiles.
struct PsWork {
    size_t parts, units, tiles, bytes;
};
static PsWork ps_work(const PackedArgs &a, int sms) {
    const size_t hd = a.width <= 64 ? 64 : 128, count = (size_t)ps_slots(a.k_rows, a.seqs) * a.c.heads;
    auto up = [](size_t x) { return (x + 1023) / 1024 * 1024; };
    PsWork w;
    w.parts = sizeof(int) * KA_BLOCKS;
    w.units = up(w.parts + sizeof(float) * 2 * std::min(KA_BLOCKS, sms) * PS_BQ * (hd + 2));
    w.tiles = up(w.units + count * sizeof(int2));
    w.bytes = w.tiles + count * 4 * PS_BK * hd * 2;
    return w;
}
size_t packed_attend_tc32_workspace(const PackedArgs &a, int sms) { return ps_work(a, sms).bytes; }

template <int HD>
static cudaError_t ps_launch(const PackedArgs &a, int sms, uint8_t *work, cudaStream_t s) {
    const PsWork w = ps_work(a, sms);
    auto whole = [&](const void *x, long long row, long long head) { return ((uintptr_t)x | (size_t)row * 4 | (size_t)head * 4) % 16 == 0; };
    const int wide = (whole(a.k, a.k_row, a.k_head) ? 1 : 0) | (whole(a.v, a.v_row, a.v_head) ? 2 : 0);
    int2 *units = reinterpret_cast<int2 *>(work + w.units);
    cudaError_t e = allow_dynamic_smem((const void *)k_packed_split<HD>, PsShape<HD>::TILE);
    if (e == cudaSuccess) e = allow_dynamic_smem((const void *)k_packed_attend_tc32<HD>, PsShape<HD>::SMEM);
    if (e != cudaSuccess) return e;
    if (a.max_len) {
        const long long each = (a.max_len + PS_BK - 1LL) / PS_BK, places = ps_slots(a.k_rows, a.seqs);
        const bool by_place = each * a.seqs > 4 * places;
        const dim3 grid((unsigned)(by_place ? places : each), a.c.heads, by_place ? 1 : a.seqs);
        k_packed_split<HD><<<grid, 256, PsShape<HD>::TILE, s>>>(a, work + w.tiles, units, wide, by_place);
    }
    k_packed_attend_tc32<HD><<<std::min(KA_BLOCKS, sms), PS_THREADS, PsShape<HD>::SMEM, s>>>(a, work + w.tiles, units, reinterpret_cast<float *>(work + w.parts),
                                                                                             reinterpret_cast<int *>(work));
    return cudaGetLastError();
}
cudaError_t launch_packed_attend_tc32(const PackedArgs &a, int sms, void *work, cudaStream_t s, uint64_t *launches) {
    (*launches) += 1 + (a.max_len > 0);
    return a.width <= 64 ? ps_launch<64>(a, sms, reinterpret_cast<uint8_t *>(work), s) : ps_launch<128>(a, sms, reinterpret_cast<uint8_t *>(work), s);
}

}  // namespace tcu

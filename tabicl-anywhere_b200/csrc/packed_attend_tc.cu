// Attention of many packed rows of a 16-bit type on the 5th-generation tensor cores (tcgen05).
//
// 256 query rows of one key head (the heads that share it side by side) as two tiles of 128, against 64 keys at a time:
// S = Q K^T from shared memory into tensor memory, in two slots a tile, so that the next step's scores are there when a softmax
// is done; the weights P, rounded to the values' type, over S; O += P V with O in tensor memory too, keys and values as TMA
// brings them (values as an operand whose coordinates are contiguous). A step of 128 keys would keep the matrix unit busier
// (its products of 64 columns wait for shared memory), but tensor memory then holds one slot a tile, and scores, softmax and
// output of a step follow one another: 5,700 cycles for 128 keys.
// A row's weights are relative to a reference that follows its largest score only when that has grown by 2^8 (f16: 2^4), so O is
// rarely rescaled. f16 weights are 2^11 times as large as that, so that they fill f16's range: one is held to 11 bits, and to 2^-36
// of the largest, below which values of 60,000 would show the loss (16 sequences of f16 tokens: 152 us; with a lag of 2^2 and 2^13
// 158, of 2^8 and 2^7 151.5, without 150). A weight's exponent is one multiply-add, so it has what the reference's rounding left: no
// matter, since all of a row's weights have it, as long as it is small. Rows whose reference is past 2^22 are worked out again by
// themselves (products rounded before the reference is subtracted take 3% longer for all others). The steps of all units are cut
// evenly over the blocks (kv4_plan.cuh).
// The matrix unit rounds its sums towards zero (1.1e-7 of one an addition, of values of one sign), so the output is taken from it
// every 8192 keys and added to what came before in the working memory: without that, outputs over 131,072 keys were 8.7e-4 too low.
// What bounds it: 4096 bf16 tokens, 32 heads on 8 of width 128, causal, take 162 us, 0.85 PFLOP/s: a step of 64 keys 1,700 cycles, of
// which the products need 1,350 and the exponentials of both tiles 1,024; a unit's output 6,500, a block's start 13,000. f16, 16 heads
// of width 64, 16 sequences of 1 to 2048 tokens: 145 us, the softmax (1,600 cycles a step) and the ends of units. Registers spilled
// in the roles that issue products cost 450 us for the first case, units cut by their steps alone 228. A polynomial in the place of
// every third to sixth exponential, and the two tiles' exponentials in turns, changed nothing.
#include <cudaTypedefs.h>

#include <algorithm>

#include "kv4_tc.cuh"
#include "packed.cuh"

namespace tcu {

constexpr int PT_R = 256, PT_BQ = 128, PT_BK = 64, PT_THREADS = 512;
constexpr int PT_STEPS = 8;  // steps a block takes at least
constexpr int PT_RING = 4;   // pieces on their way to the roles
constexpr int PT_FOLD = 128; // steps that the output is summed over in tensor memory

template <int HD>
struct PtShape {
    static constexpr int NS = HD == 128 ? 3 : 6;  // slots of keys, and of values
    static constexpr int EXTRA = HD == 128 ? 5 : 2;  // what a unit costs besides its steps, in steps (measured: 4, 7; 1, 3 are slower)
    static constexpr int TILE = PT_BK * HD * 2, QTILE = PT_BQ * HD * 2;
    static constexpr size_t SMEM = 4 * QTILE + 2 * NS * TILE + 1024;  // queries of this piece and the next
    static constexpr size_t PART = (size_t)PT_R * (HD + 2);  // floats: outputs (4 columns of all rows, then the next 4), maxima, sums
};

// 128-byte rows swizzled by 128 bytes, groups of 8 rows 1024 bytes apart. As an operand whose K runs along a row this is all (lbo
// is not read); as one whose M or N does, K runs over the rows, and blocks of 64 elements lie `lbo` bytes apart.
__device__ __forceinline__ uint64_t pt_desc(uint32_t addr, uint32_t lbo) {
    return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)((lbo >> 4) & 0x3fff) << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
__device__ __forceinline__ void pt_load(uint32_t to, const CUtensorMap *map, int x, int y, int z, uint64_t *m) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(to),
                 "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_addr(m))
                 : "memory");
}
__device__ __forceinline__ void pt_expect(uint64_t *m, uint32_t bytes) {
    asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}\n" ::"r"(smem_addr(m)), "r"(bytes) : "memory");
}
// (nothing that uses v moves before the wait for it)
__device__ __forceinline__ void pt_tie(float (&v)[32]) {
#pragma unroll
    for (int i = 0; i < 32; i += 8)
        asm volatile("" : "+f"(v[i]), "+f"(v[i + 1]), "+f"(v[i + 2]), "+f"(v[i + 3]), "+f"(v[i + 4]), "+f"(v[i + 5]), "+f"(v[i + 6]), "+f"(v[i + 7])::"memory");
}
// Two f32 at a time: x * y + z, x + y; and the largest of three.
__device__ __forceinline__ float2 pt_fma2(float2 x, float2 y, float2 z) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\tfma.rn.f32x2 a, a, b, c;\n\tmov.b64 {%0, %1}, a;\n\t}\n"
        : "=f"(d.x), "=f"(d.y)
        : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y), "f"(z.x), "f"(z.y));
    return d;
}
__device__ __forceinline__ float2 pt_add2(float2 x, float2 y) {
    float2 d;
    asm("{\n\t.reg .b64 a, b;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 a, a, b;\n\tmov.b64 {%0, %1}, a;\n\t}\n"
        : "=f"(d.x), "=f"(d.y)
        : "f"(x.x), "f"(x.y), "f"(y.x), "f"(y.y));
    return d;
}
__device__ __forceinline__ float pt_max3(float x, float y, float z) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(x), "f"(y), "f"(z));
    return d;
}
template <int DT>
__device__ __forceinline__ uint32_t pt_pair(float x, float y) {
    if constexpr (DT == DT_F16) {
        const __half2 h = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}

// A row's output in tensor memory added to what `to` holds of it (HD columns, 4 of all rows beside one another), that times f.
template <int HD>
__device__ __noinline__ void pt_fold(uint32_t tO, float *to, float f, bool first) {
#pragma unroll 1
    for (int b = 0; b < HD / 16; b++) {
        float o[16];
        tmem_ld16(tO + 16 * b, o);
        tmem_wait_ld();
#pragma unroll
        for (int k = 0; k < 16; k++) asm volatile("" : "+f"(o[k])::"memory");  // (not used before the wait)
#pragma unroll
        for (int k = 0; k < 16; k += 4) {
            float4 *at = reinterpret_cast<float4 *>(to + (4 * b + k / 4) * PT_R * 4);
            const float4 v = first ? make_float4(0.f, 0.f, 0.f, 0.f) : __ldcg(at);
            __stcg(at, make_float4(fmaf(v.x, f, o[k]), fmaf(v.y, f, o[k + 1]), fmaf(v.z, f, o[k + 2]), fmaf(v.w, f, o[k + 3])));
        }
    }
}

// Warps 0-3, 4-7: softmax of the first and second tile, a thread a query row; warps 8, 9: the tiles' products S; warps 10, 11:
// their products P V (a warp for both tiles' was what a step took longest in: a wait and its bookkeeping cost some hundred
// cycles); warp 12: the copies; warp 13 clears the values behind a sequence's end; warp 14 walks the block's pieces of units and
// hands them to the others, so that these have registers for their work alone; warp 15 brings the next piece's queries. Every
// wait is bounded, and one that gives up raises the block's abort flag, after which every wait returns at once, the roles leave
// with the piece that they have, nothing more is asked for, and the block counts itself among those that share its units.
template <int HD, int DT>
__global__ void __launch_bounds__(PT_THREADS, 1) k_packed_attend_tc(PackedArgs a, const __grid_constant__ CUtensorMap map_k,
                                                                    const __grid_constant__ CUtensorMap map_v,
                                                                    const __grid_constant__ CUtensorMap map_q, int by_map, float *part, int *arrived) {
    using C = PtShape<HD>;
    using T = typename Elem<DT>::T;
    constexpr int EXTRA = C::EXTRA;
    // a weight's exponent beside the reference at most when that is moved, and how far it may grow before it is moved again
    constexpr float SHIFT = DT == DT_F16 ? 11.f : 0.f, LAG = DT == DT_F16 ? 4.f : 8.f;
    using Cut = KaCut<PT_R, 1, PT_BK, EXTRA>;
    constexpr int BQ = PT_BQ, BK = PT_BK, NS = C::NS, TILE = C::TILE, QTILE = C::QTILE;
    constexpr uint32_t TS = 0, TO = 256;  // tensor memory: [tile][2 slots] of S / P, then [tile] of O
    extern __shared__ uint8_t smraw[];
    // A piece of a unit: n steps of keys, the first at key j0; the first nq[q] of them hold all that tile q's rows see. It is the
    // whole unit, or shared by blocks who.x .. who.x + who.y.
    struct Piece {
        KaRows sr;
        int seq, head, n, nq[2], j0, k0, r0, first, over, begins, whole;
        int2 who;
    };
    __shared__ Piece ring[PT_RING];
    __shared__ __align__(8) uint64_t mK[NS], mV[NS], mKfree[NS], mVfree[NS], mFix[NS], mQ[2], mQfree[2], mS[2][2], mP[2][2], mSlot[2][2], mDone[4], mJoin, mPiece[PT_RING],
        mPieceFree[PT_RING];
    __shared__ uint32_t tslot;
    __shared__ volatile int abort_flag;
    __shared__ int s_unit[4], s_last;
    // for the rows that are worked out again at the end: where the block's pieces began, the units that it has joined, whether some
    // of its outputs are not finite, and whether of rows whose scores were too large
    __shared__ typename Cut::Place s_place;
    __shared__ int s_joined[2], s_counted[2], s_dirty;  // (s_counted: whether the block has counted itself among those that share them)
    __shared__ volatile int s_bad, s_large;
    __shared__ long long s_sum[PT_THREADS / 32];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, wg = warp >> 2;
    const int each = a.q_heads / a.c.heads;
    auto pl = Cut::template place<PT_THREADS>(a, each, PT_STEPS, s_sum, s_unit);
    if (pl.pos >= pl.end) return;
    if (warp == 8) {
        tmem_alloc(&tslot, 512);
        tmem_relinquish();
    }
    if (tid == 0) {
        for (int i = 0; i < NS; i++) mbar_init(&mK[i], 1), mbar_init(&mV[i], 1), mbar_init(&mKfree[i], 2), mbar_init(&mVfree[i], 3), mbar_init(&mFix[i], 32);
        for (int q = 0; q < 2; q++) {
            for (int i = 0; i < 2; i++) mbar_init(&mS[q][i], 1), mbar_init(&mP[q][i], 4), mbar_init(&mSlot[q][i], 1);
            mbar_init(&mQ[q], 32), mbar_init(&mQfree[q], 2 * BQ + 2), mbar_init(&mDone[2 * q], 1), mbar_init(&mDone[2 * q + 1], 1);
        }
        for (int i = 0; i < PT_RING; i++) mbar_init(&mPiece[i], 1), mbar_init(&mPieceFree[i], 15);
        mbar_init(&mJoin, 2 * BQ);
        mbar_init_fence();
        abort_flag = a.give_up & blockIdx.x & 1, s_counted[0] = s_counted[1] = s_joined[0] = s_joined[1] = s_bad = s_large = 0, s_place = pl;
    }
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = tslot;
    const uint32_t base = (smem_addr(smraw) + 1023u) & ~1023u, sQ = base, sK = base + 4 * QTILE, sV = sK + NS * TILE;
    auto wait_warp = [&](uint64_t *m, uint32_t parity) {
        if (!mbar_test_wait(m, parity) && !abort_flag && !mbar_wait(m, parity, KT_WAIT)) abort_flag = 1;
        __syncwarp();
    };
    auto stopped = [&] { return __any_sync(0xffffffffu, abort_flag != 0); };
    // the next piece, from which every warp of a role takes what it needs; `taken` once it has
    int turns = 0;
    auto take = [&]() -> const Piece & {
        wait_warp(&mPiece[turns % PT_RING], (uint32_t)(turns / PT_RING) & 1u);
        return ring[turns % PT_RING];
    };
    auto taken = [&]() {
        __syncwarp();
        if (lane == 0) mbar_arrive(&mPieceFree[turns % PT_RING]);
        turns++;
    };
    int at = 0;  // steps before the piece's

    if (wg >= 2) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == 14) {
            for (;; turns++) {
                if (turns >= PT_RING) wait_warp(&mPieceFree[turns % PT_RING], (uint32_t)(turns / PT_RING - 1) & 1u);
                Piece &p = ring[turns % PT_RING];
                if (pl.pos >= pl.end || abort_flag) {  // none
                    if (lane == 0) p.n = -1, mbar_arrive(&mPiece[turns % PT_RING]);
                    break;
                }
                const KaRows sr = ka_rows(a, pl.seq);
                const auto sp = Cut::span(a, sr, each, pl.rt);
                const int count = (int)min((long long)(sp.steps - pl.skip), pl.end - pl.pos), from = max(0, pl.skip - EXTRA);
                if (lane == 0) {
                    p.sr = sr, p.seq = pl.seq, p.head = pl.head, p.n = max(0, pl.skip + count - EXTRA) - from;
                    p.j0 = sp.base + from * BK, p.k0 = a.k_starts[pl.seq], p.r0 = pl.rt * PT_R, p.begins = pl.skip == 0, p.whole = count == sp.steps;
                    p.first = p.r0 / each, p.over = p.r0 - p.first * each, p.who = make_int2(0, 1);
                    if (!p.whole) p.who = Cut::sharers(pl, pl.pos - pl.skip, sp.steps);
                    for (int q = 0; q < 2; q++) {
                        const int rows = min(sr.n * each - p.r0, (q + 1) * BQ);
                        p.nq[q] = 0;
                        if (rows > q * BQ) {
                            const int hi = ka_hi(a, sr, (p.r0 + rows - 1) / each);
                            p.nq[q] = hi > sp.lo_min ? max(0, min(p.n, (hi - p.j0 + BK - 1) / BK)) : 0;
                        }
                    }
                    mbar_arrive(&mPiece[turns % PT_RING]);
                }
                Cut::next(pl, a, each, sr.n, count);
            }
        } else if (warp == 12) {
            int k_asked = 0, v_asked = 0;  // steps whose copies have been asked for
            for (;;) {
                const Piece &p = take();
                const int n = p.n, z0 = p.k0 + p.j0, head = p.head;
                taken();
                if (n < 0 || abort_flag) break;
                for (int i = 0; i < n; i++) {
                    const int slot = (at + i) % NS, turn = (at + i) / NS, z = z0 + i * BK;
                    if (turn) wait_warp(&mKfree[slot], (uint32_t)(turn - 1) & 1u);
                    if (stopped()) break;
                    k_asked++;
                    if (elect_one()) {
                        pt_expect(&mK[slot], TILE);
#pragma unroll
                        for (int x = 0; x < HD; x += 64) pt_load(sK + slot * TILE + x * BK * 2, &map_k, x, head, z, &mK[slot]);
                    }
                    __syncwarp();
                    if (turn) wait_warp(&mVfree[slot], (uint32_t)(turn - 1) & 1u);
                    if (stopped()) break;
                    v_asked++;
                    if (elect_one()) {
                        pt_expect(&mV[slot], TILE);
#pragma unroll
                        for (int x = 0; x < HD; x += 64) pt_load(sV + slot * TILE + x * BK * 2, &map_v, x, head, z, &mV[slot]);
                    }
                    __syncwarp();
                }
                at += n;
            }
            // what was asked for lands before the block lets go of shared memory
            for (int i = max(0, k_asked - NS); i < k_asked; i++) mbar_wait(&mK[i % NS], (uint32_t)(i / NS) & 1u, KT_WAIT);
            for (int i = max(0, v_asked - NS); i < v_asked; i++) mbar_wait(&mV[i % NS], (uint32_t)(i / NS) & 1u, KT_WAIT);
        } else if (warp == 15) {
            // the rows' queries: by TMA (by_map), or in 16-byte pieces, asynchronously where they are aligned and not to change sign
            constexpr int LANES = HD / 8, ROWS = 32 / LANES;  // lanes a row, rows at a time
            const int sub = lane / LANES, chunk = lane % LANES;
            const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u, inverse = (uint32_t)((0x100000000ull + each - 1) / each);
            const bool wide = (((uintptr_t)a.q | (size_t)a.q_row * 2 | (size_t)a.q_head * 2) & 15) == 0 && !flip;
            const bool on = chunk * 8 < a.width;
            uint32_t units = 0;
            for (;;) {
                const Piece &p = take();
                const int n = p.n, over = p.over, rows = min(PT_R, p.sr.n * each - p.r0), token = p.sr.first + p.first, head = p.head * each;
                // row r: token first + (over + r) / each, head (over + r) % each of those that share this one
                const uint16_t *from = reinterpret_cast<const uint16_t *>(a.q) + (long long)token * a.q_row + (long long)head * a.q_head + chunk * 8;
                taken();
                if (n < 0 || abort_flag) break;
                const int b = units & 1;
                if (units >= 2) wait_warp(&mQfree[b], (units / 2 - 1) & 1u);
                if (stopped()) break;
                units++;
                if (by_map) {
                    if (lane == 0) {
                        pt_expect(&mQ[b], 2 * QTILE);
                        for (int x = 0; x < HD; x += 64)
                            for (int q = 0; q < 2; q++) pt_load(sQ + (2 * b + q) * QTILE + x * BQ * 2, &map_q, x, head, token + q * (BQ / each), &mQ[b]);
                    } else {
                        mbar_arrive(&mQ[b]);
                    }
                    __syncwarp();
                    continue;
                }
                uint8_t *to = smraw + (sQ - smem_addr(smraw)) + b * 2 * QTILE;
#pragma unroll 4
                for (int x = 0; x < PT_R; x += ROWS) {
                    const int r = x + sub;
                    const uint32_t i = each == 1 ? (uint32_t)(over + r) : __umulhi((uint32_t)(over + r), inverse);
                    const uint16_t *src = from + (long long)i * a.q_row + (long long)(over + r - (int)i * each) * a.q_head;
                    const bool in = r < rows && on;
                    uint8_t *dst = to + (r / BQ) * QTILE + (chunk / 8) * BQ * 128 + (r % BQ) * 128 + ((chunk ^ r) & 7) * 16;
                    if (wide) {
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(in ? src : reinterpret_cast<const uint16_t *>(a.q)), "r"(in ? 16 : 0)
                                     : "memory");
                    } else {
                        uint4 w = make_uint4(0, 0, 0, 0);
                        if (in)
                            w = make_uint4(src[0] | (uint32_t)src[1] << 16, src[2] | (uint32_t)src[3] << 16, src[4] | (uint32_t)src[5] << 16,
                                           src[6] | (uint32_t)src[7] << 16);
                        *reinterpret_cast<uint4 *>(dst) = make_uint4(w.x ^ flip, w.y ^ flip, w.z ^ flip, w.w ^ flip);
                    }
                }
                asm volatile("cp.async.wait_all;" ::: "memory");
                fence_async_smem();
                mbar_arrive(&mQ[b]);
            }
            // what was asked for lands before the block lets go of shared memory
            if (by_map)
                for (uint32_t i = units > 2 ? units - 2 : 0; i < units; i++) mbar_wait(&mQ[i & 1], i / 2 & 1u, KT_WAIT);
        } else if (warp == 13) {
            for (;;) {
                const Piece &p = take();
                const int n = p.n, there = p.sr.len - p.j0;  // keys from the piece's first on
                taken();
                if (n < 0 || abort_flag) break;
                for (int i = 0; i < n; i++) {
                    // (every step, so that no turn of a slot is taken for another)
                    const int slot = (at + i) % NS, from = max(0, there - i * BK);
                    wait_warp(&mV[slot], (uint32_t)((at + i) / NS) & 1u);
                    if (from < BK) {
                        uint8_t *v = smraw + (sV - smem_addr(smraw)) + slot * TILE;
                        for (int x = lane; x < (BK - from) * 8; x += 32) {
#pragma unroll
                            for (int b = 0; b < HD / 64; b++) *reinterpret_cast<uint4 *>(v + b * BK * 128 + from * 128 + x * 16) = make_uint4(0, 0, 0, 0);
                        }
                        fence_async_smem();
                        mbar_arrive(&mFix[slot]);
                    }
                    if (lane == 0) mbar_arrive(&mVfree[slot]);
                }
                at += n;
            }
        } else if (warp < 12) {
            const uint32_t type = DT == DT_BF16 ? 1u << 7 | 1u << 10 : 0u;
            const uint32_t idS = idesc_f16(BQ, BK, 0, 0) | type, idO = idesc_f16(BQ, HD, 0, 1) | type;
            const int q = warp & 1;
            const bool scores = warp < 10;
            const uint64_t dQ = pt_desc(sQ + q * QTILE, 16), dK = pt_desc(sK, 16), dV = pt_desc(sV, BK * 128);
            const uint32_t tS = tmem + TS + 2 * q * BK, tO = tmem + TO + q * HD;
            int c = 0;           // the tile's steps so far
            uint32_t units = 0;  // pieces so far: the next's queries are in buffer units % 2
            uint32_t fixed = 0;  // each slot's bit: the parity of its next clearing
            for (;;) {
                const Piece &p = take();
                const int n = p.n, nq = p.nq[q], there = p.sr.len - p.j0;
                taken();
                if (n < 0 || abort_flag) break;
                const uint64_t dq = dQ + (units & 1 ? (2 * QTILE) >> 4 : 0);
                if (scores) wait_warp(&mQ[units & 1], units / 2 & 1u);
                for (int i = 0; i < n; i++, at++) {
                    const int slot = at % NS;
                    const uint32_t turn = (uint32_t)(at / NS) & 1u;
                    if (scores) {
                        // S(i), once P V(i - 2) has read its slot
                        wait_warp(&mK[slot], turn);
                        if (i < nq) {
                            if (c >= 2) wait_warp(&mSlot[q][c & 1], (uint32_t)((c >> 1) - 1) & 1u);
                            fence_after_sync();
                            const uint64_t d = dK + ((slot * TILE) >> 4);
                            if (elect_one()) {
#pragma unroll
                                for (int k = 0; k < HD / 16; k++)
                                    mma_f16(tS + (c & 1) * BK, dq + (((k / 4) * BQ * 128 + (k % 4) * 32) >> 4), d + (((k / 4) * BK * 128 + (k % 4) * 32) >> 4), idS, k > 0);
                                mma_commit(&mS[q][c & 1]);
                                mma_commit(&mKfree[slot]);
                            }
                            c++;
                        } else if (lane == 0) {
                            mbar_arrive(&mKfree[slot]);
                        }
                    } else {
                        wait_warp(&mV[slot], turn);
                        if (there - i * BK < BK) wait_warp(&mFix[slot], fixed >> slot & 1u), fixed ^= 1u << slot;
                        if (i < nq) {
                            wait_warp(&mP[q][c & 1], (uint32_t)(c >> 1) & 1u);
                            fence_after_sync();
                            const uint64_t d = dV + ((slot * TILE) >> 4);
                            if (elect_one()) {
#pragma unroll
                                for (int k = 0; k < BK / 16; k++) mma_f16_ta(tO, tS + (c & 1) * BK + 8 * k, d + ((k * 2048) >> 4), idO, i % PT_FOLD > 0 || k > 0);
                                mma_commit(&mSlot[q][c & 1]);
                                mma_commit(&mVfree[slot]);
                            }
                            c++;
                        } else if (lane == 0) {
                            mbar_arrive(&mVfree[slot]);
                        }
                    }
                    __syncwarp();
                }
                // (a warp that has no steps does so too: no turn of a buffer is taken for another)
                if (scores && lane == 0) mbar_arrive(&mQfree[units & 1]);
                units++;
            }
            // every product issued here completes before the block lets go of its memory
            if (elect_one()) {
                mma_commit(&mDone[warp - 8]);
                mbar_wait(&mDone[warp - 8], 0, KT_WAIT);
            }
            __syncwarp();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 184;");
        const int q = wg, row = tid & 127;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, tO = tmem + lanes + TO + q * HD;
        const float sl = fminf(fmaxf(fabsf(a.scale) * 1.44269504088896340736f, FLT_MIN), FLT_MAX);  // (positive, so that -infinity stays itself)
        constexpr float UNSHIFT = DT == DT_F16 ? 0x1p-11f : 1.f;
        const bool wide_o = (((uintptr_t)a.out | (size_t)a.o_row * 2 | (size_t)a.o_head * 2) & 15) == 0;
        uint32_t units = 0, meetings = 0;
        // both tiles' threads (a barrier whose wait is bounded too)
        auto meet = [&]() {
            mbar_arrive(&mJoin);
            wait_warp(&mJoin, meetings++ & 1u);
        };
        // 16 bytes, 8 coordinates from 8 x on, of row r where the tile's queries are: outputs go to memory through the same place
        auto cell = [&](int r, int x) {
            return reinterpret_cast<uint4 *>(smraw + (sQ - smem_addr(smraw)) + (2 * (units & 1) + q) * QTILE + (x / 8) * BQ * 128 + r * 128 + ((x ^ r) & 7) * 16);
        };
        constexpr int LANES = HD / 8, ROWS = 32 / LANES;  // lanes a row, rows at a time
        const int sub = lane / LANES, chunk = lane % LANES;
        const uint32_t inverse = (uint32_t)((0x100000000ull + each - 1) / each);  // x / each = x * inverse >> 32 for x below each + 256
        int c = 0;
        for (;;) {
            const Piece &p = take();
            if (p.n < 0 || abort_flag) break;
            // (a tile without rows too: its threads' word that they are done with a buffer must not be counted for the next but one)
            wait_warp(&mQ[units & 1], units / 2 & 1u);
            const int nq = p.nq[q], r0 = p.r0 + q * BQ, rows = min(BQ, p.sr.n * each - r0);
            const bool there = row < rows;
            // row r of the tile in memory, 8 coordinates from this lane's on
            auto token = [&](int r) {  // a row's token in its sequence
                const uint32_t x = p.over + q * BQ + r;
                return p.first + (int)(each == 1 ? x : __umulhi(x, inverse));
            };
            auto at_row = [&](auto *t, long long row, long long head, int r) {
                const int i = token(r);
                return t + (p.sr.first + i) * row + (p.head * each + r0 + r - i * each) * head + chunk * 8;
            };
            int my_lo = 0, my_hi = 0;
            if (there) {
                const int i = token(row);
                my_lo = ka_lo(a, p.sr, i) - p.j0, my_hi = ka_hi(a, p.sr, i) - p.j0;  // from the piece's first key on
            }
            float m = -INFINITY, l = 0.f;  // the row's reference (log2), its sum of weights
            float x[64];                   // a step's scores
            // where the row's output is folded to, for a part of a unit the part's own place (for a whole one that of the block's last part,
            // which comes after all of those), and the reference it has there
            float *fold = part + Cut::slot(blockIdx.x, p.whole || p.begins) * C::PART + (q * BQ + row) * 4, m_fold = -INFINITY;
            auto fold_by = [&] { return m_fold == -INFINITY ? 0.f : kt_ex2(m_fold - m); };
            auto fetch = [&](int i, float (&to)[64]) {  // once S(i) is there: on their way until the next wait for loads
                wait_warp(&mS[q][i & 1], (uint32_t)(i >> 1) & 1u);
                fence_after_sync();
                const uint32_t from = tmem + lanes + TS + (2 * q + (i & 1)) * BK;
                tmem_ld32(from, *reinterpret_cast<float (*)[32]>(&to[0])), tmem_ld32(from + 32, *reinterpret_cast<float (*)[32]>(&to[32]));
            };
            auto arrived_all = [&](float (&v)[64]) {
                tmem_wait_ld();
                pt_tie(*reinterpret_cast<float (*)[32]>(&v[0])), pt_tie(*reinterpret_cast<float (*)[32]>(&v[32]));
            };
            if (nq) {
                fetch(c, x);
                arrived_all(x);
            }
#pragma unroll 1
            for (int i0 = 0; i0 < nq; i0 += PT_FOLD) {
                if (i0) {  // (the next product begins a sum of its own)
                    wait_warp(&mSlot[q][(c - 1) & 1], (uint32_t)((c - 1) >> 1) & 1u);
                    fence_after_sync();
                    pt_fold<HD>(tO, fold, fold_by(), i0 == PT_FOLD);
                    m_fold = m;
                }
#pragma unroll 1
                for (int i = i0, i1 = min(nq, i0 + PT_FOLD); i < i1; i++, c++) {
                    const int key0 = i * BK;
                    const uint32_t tS = tmem + lanes + TS + (2 * q + (c & 1)) * BK;
                    if (__any_sync(0xffffffffu, key0 < my_lo || key0 + BK > my_hi)) {
                        const int low = my_lo - key0, high = my_hi - key0;
#pragma unroll
                        for (int k = 0; k < 64; k++)
                            if (k < low || k >= high) x[k] = -INFINITY;
                    }
                    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int k = 0; k < 32; k++) top[k & 3] = pt_max3(top[k & 3], x[2 * k], x[2 * k + 1]);
                    const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * sl - SHIFT;
                    if (__any_sync(0xffffffffu, mx > m + LAG)) {
                        const float mnew = fmaxf(m, mx), f = m == -INFINITY ? 0.f : kt_ex2(m - mnew);
                        if (i > 0) {  // O, once the product before has been added to it
                            wait_warp(&mSlot[q][(c - 1) & 1], (uint32_t)((c - 1) >> 1) & 1u);
                            fence_after_sync();
#pragma unroll 1
                            for (int b = 0; b < HD / 16; b++) {
                                float o[16];
                                tmem_ld16(tO + 16 * b, o);
                                tmem_wait_ld();
#pragma unroll
                                for (int k = 0; k < 16; k++) asm volatile("" : "+f"(o[k])::"memory");  // (not used before the wait)
                                uint32_t w[16];
#pragma unroll
                                for (int k = 0; k < 16; k++) w[k] = __float_as_uint(o[k] * f);
                                tmem_st16u(tO + 16 * b, w);
                            }
                        }
                        l *= f, m = mnew;
                    }
                    const float mm = m == -INFINITY ? 0.f : m;
                    const float2 sl2 = make_float2(sl, sl), mm2 = make_float2(-mm, -mm);
                    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
                    for (int b = 0; b < 2; b++) {
                        uint32_t h[16];
#pragma unroll
                        for (int k = 0; k < 16; k++) {
                            const float2 t = pt_fma2(make_float2(x[32 * b + 2 * k], x[32 * b + 2 * k + 1]), sl2, mm2);
                            const float2 w = make_float2(kt_ex2(t.x), kt_ex2(t.y));
                            sum[k & 1] = pt_add2(sum[k & 1], w);
                            h[k] = pt_pair<DT>(w.x, w.y);
                        }
                        tmem_st16u(tS + 16 * b, h);  // over scores that have been read
                    }
                    tmem_wait_st();
                    fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&mP[q][c & 1]);
                    l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                    if (i + 1 < nq) {
                        fetch(c + 1, x);
                        arrived_all(x);
                    }
                }
            }

            // ---- the rows' outputs, or their part of them ----
            const bool whole = p.whole;
            if (nq) wait_warp(&mSlot[q][(c - 1) & 1], (uint32_t)((c - 1) >> 1) & 1u);
            fence_after_sync();
            auto inverse_of = [&](float M, float L) {
                if (there && M != -INFINITY && !(fabsf(M) < 4194304.f)) {
                    s_large = 1;
                    return __uint_as_float(0x7fc00000u);  // (its outputs are NaN until then)
                }
                return L != 0.f ? 1.f / L : 0.f;
            };
            float inv = whole ? inverse_of(m, l) : 1.f;
            float2 odd = make_float2(0.f, 0.f);  // NaN once an output is not finite
            // 32 columns from 32 b on to the row's place in shared memory
            auto put = [&](int b, const float (&o)[32]) {
#pragma unroll
                for (int y = 0; y < 4; y++) {
                    uint32_t w[4];
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const float y0 = o[8 * y + 2 * k] * inv, y1 = o[8 * y + 2 * k + 1] * inv;
                        odd = pt_fma2(make_float2(y0, y1), make_float2(0.f, 0.f), odd);
                        w[k] = pt_pair<DT>(y0, y1);
                    }
                    *cell(row, 4 * b + y) = make_uint4(w[0], w[1], w[2], w[3]);
                }
            };
            // the warp's rows from there to memory
            auto flush = [&](float M, float L) {
                __syncwarp();
#pragma unroll 4
                for (int x = 0; x < 32; x += ROWS) {
                    const int r = (warp & 3) * 32 + x + sub;
                    const uint4 w = *cell(r, chunk);
                    uint16_t *dst = at_row(reinterpret_cast<uint16_t *>(a.out), a.o_row, a.o_head, r);
                    if (r >= rows || chunk * 8 >= a.width) continue;
                    if (wide_o) {
                        *reinterpret_cast<uint4 *>(dst) = w;
                    } else {
                        dst[0] = (uint16_t)w.x, dst[1] = (uint16_t)(w.x >> 16), dst[2] = (uint16_t)w.y, dst[3] = (uint16_t)(w.y >> 16);
                        dst[4] = (uint16_t)w.z, dst[5] = (uint16_t)(w.z >> 16), dst[6] = (uint16_t)w.w, dst[7] = (uint16_t)(w.w >> 16);
                    }
                }
                const int i_row = there ? token(row) : 0, hq = p.head * each + (there ? r0 + row - i_row * each : 0);
                if (there && a.lse) a.lse[(size_t)(p.sr.first + i_row) * a.q_heads + hq] = ((M == -INFINITY ? 0.f : M + SHIFT) + log2f(L * UNSHIFT)) * 0.69314718055994530942f;
                if (odd.x + odd.y != 0.f && there) s_bad = 1;
            };
            const size_t prow = q * BQ + row;
            float *mine = part + Cut::slot(blockIdx.x, p.begins) * C::PART;
#pragma unroll 1
            for (int b = 0; b < HD / 32; b++) {
                float o[32];
                tmem_ld32(tO + 32 * b, o);
                tmem_wait_ld32(o);
                if (!nq) {
#pragma unroll
                    for (int k = 0; k < 32; k++) o[k] = 0.f;
                }
                if (nq > PT_FOLD) {
                    const float f = fold_by();
#pragma unroll
                    for (int k = 0; k < 32; k += 4) {
                        const float4 v = __ldcg(reinterpret_cast<const float4 *>(fold + (8 * b + k / 4) * PT_R * 4));
                        o[k] = fmaf(v.x, f, o[k]), o[k + 1] = fmaf(v.y, f, o[k + 1]), o[k + 2] = fmaf(v.z, f, o[k + 2]), o[k + 3] = fmaf(v.w, f, o[k + 3]);
                    }
                }
                if (whole) {
                    put(b, o);
                } else if (there) {
#pragma unroll
                    for (int k = 0; k < 32; k += 4) __stcg(reinterpret_cast<float4 *>(mine + ((8 * b + k / 4) * PT_R + prow) * 4), make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]));
                }
            }
            fence_before_sync();
            if (whole) {
                if (!abort_flag) flush(m, l);
            } else {
                if (there) __stcg(mine + PT_R * HD + prow, m), __stcg(mine + PT_R * (HD + 1) + prow, l);
                const int2 who = p.who;
                __threadfence();
                meet();
                if (tid == 0) {
                    s_counted[p.begins] = 1;
                    const int before = atomicAdd(&arrived[who.x], 1);
                    s_last = before == who.y - 1;
                    if (s_last) arrived[who.x] = 0, s_joined[p.begins] = 1;
                    __threadfence();
                }
                meet();
                if (*reinterpret_cast<volatile int *>(&s_last) && !abort_flag) {
                    auto from = [&](int b) { return part + Cut::slot(who.x + b, b == 0) * C::PART; };
                    float M = -INFINITY, L = 0.f;
                    for (int b = 0; b < who.y; b++) M = fmaxf(M, there ? __ldcg(from(b) + PT_R * HD + prow) : 0.f);
                    const float ref = M == -INFINITY ? 0.f : M;
                    for (int b = 0; b < who.y; b++)
                        if (there) {
                            const float pm = __ldcg(from(b) + PT_R * HD + prow), ps = __ldcg(from(b) + PT_R * (HD + 1) + prow);
                            if (pm != -INFINITY || ps != 0.f) L = fmaf(kt_ex2(pm - ref), ps, L);
                        }
                    inv = inverse_of(M, L);
#pragma unroll 1
                    for (int y = 0; y < HD / 32; y++) {
                        float o[32];
#pragma unroll
                        for (int k = 0; k < 32; k++) o[k] = 0.f;
                        for (int b = 0; b < who.y; b++)
                            if (there) {
                                const float pm = __ldcg(from(b) + PT_R * HD + prow), ps = __ldcg(from(b) + PT_R * (HD + 1) + prow);
                                if (pm == -INFINITY && ps == 0.f) continue;
                                const float w = kt_ex2(pm - ref);
#pragma unroll
                                for (int k = 0; k < 32; k += 4) {
                                    const float4 v = __ldcg(reinterpret_cast<const float4 *>(from(b) + ((8 * y + k / 4) * PT_R + prow) * 4));
                                    o[k] = fmaf(w, v.x, o[k]), o[k + 1] = fmaf(w, v.y, o[k + 1]), o[k + 2] = fmaf(w, v.z, o[k + 2]), o[k + 3] = fmaf(w, v.w, o[k + 3]);
                                }
                            }
                        put(y, o);
                    }
                    flush(M, L);
                }
            }
            fence_async_smem();  // (outputs were stored where copies will write)
            mbar_arrive(&mQfree[units & 1]);
            units++;
            taken();
        }
    }
    fence_before_sync();
    __syncthreads();
    if (tid == 0 && abort_flag) {
        *reinterpret_cast<volatile int *>(a.err_wait) = 1;
        // the counters are to be zero when all blocks are done, whatever became of this one's parts
        for (auto p = s_place; p.pos < p.end;) {
            const KaRows s = ka_rows(a, p.seq);
            const int steps = Cut::span(a, s, each, p.rt).steps, count = (int)min((long long)(steps - p.skip), p.end - p.pos);
            if (count != steps && !s_counted[p.skip == 0]) {
                const int2 who = Cut::sharers(p, p.pos - p.skip, steps);
                if (atomicAdd(&arrived[who.x], 1) == who.y - 1) arrived[who.x] = 0;
            }
            Cut::next(p, a, each, s.n, count);
        }
    }
    fence_after_sync();
    if (warp == 8) tmem_dealloc(tmem, 512);
    if (warp < 8 && s_bad && !abort_flag) pa_mend<DT, HD, PT_R, PT_BK, EXTRA, 8, Cut>(a, s_place, s_joined, s_large, 0x1p-8f, &s_dirty);
}

template <int HD>
static size_t pt_workspace(int sms) {
    return sizeof(int) * KA_BLOCKS + sizeof(float) * 2 * (size_t)std::min(KA_BLOCKS, sms) * PtShape<HD>::PART;
}
size_t packed_attend_tc_workspace(const PackedArgs &a, int sms) { return a.width <= 64 ? pt_workspace<64>(sms) : pt_workspace<128>(sms); }

// Rows of `heads` heads as TMA fetches them: boxes of 64 coordinates, `beside` heads and `tokens` rows (zeros past the width and
// past the last row).
static bool pt_map(void *encode, CUtensorMap *m, int dtype, int width, int heads, int rows, const void *x, long long row, long long head, int beside, int tokens) {
    if (((uintptr_t)x | (size_t)row * 2) % 16 || row < 8 || (heads > 1 && ((size_t)head * 2 % 16 || head < 8))) return false;
    const cuuint64_t dims[3] = {(cuuint64_t)width, (cuuint64_t)heads, (cuuint64_t)rows};
    const cuuint64_t strides[2] = {(cuuint64_t)(heads > 1 ? head : row) * 2, (cuuint64_t)row * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)beside, (cuuint32_t)tokens}, one[3] = {1, 1, 1};
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(encode)(
               m, dtype == DT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void *>(x), dims, strides, box, one,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct PtMaps {
    CUtensorMap k, v, q;
    int by_map;
};
template <int HD, int DT>
static cudaError_t pt_launch(const PackedArgs &a, int sms, const PtMaps &m, void *work, cudaStream_t s) {
    const cudaError_t e = allow_dynamic_smem((const void *)k_packed_attend_tc<HD, DT>, PtShape<HD>::SMEM);
    if (e != cudaSuccess) return e;
    int *arrived = reinterpret_cast<int *>(work);
    k_packed_attend_tc<HD, DT><<<std::min(KA_BLOCKS, sms), PT_THREADS, PtShape<HD>::SMEM, s>>>(a, m.k, m.v, m.q, m.by_map, reinterpret_cast<float *>(arrived + KA_BLOCKS),
                                                                                               arrived);
    return cudaGetLastError();
}

cudaError_t launch_packed_attend_tc(int dtype, const PackedArgs &a, int sms, void *encode, void *work, cudaStream_t s) {
    PtMaps m;
    if (!encode || a.k_rows < 1 || !pt_map(encode, &m.k, dtype, a.width, a.c.heads, a.k_rows, a.k, a.k_row, a.k_head, 1, PT_BK) ||
        !pt_map(encode, &m.v, dtype, a.width, a.c.heads, a.k_rows, a.v, a.v_row, a.v_head, 1, PT_BK))
        return cudaErrorNotSupported;
    // queries too, where a tile of 128 rows is whole tokens
    const int each = a.q_heads / a.c.heads;
    m.by_map = a.scale >= 0.f && PT_BQ % each == 0 && pt_map(encode, &m.q, dtype, a.width, a.q_heads, a.rows, a.q, a.q_row, a.q_head, each, PT_BQ / each);
    if (!m.by_map) m.q = m.k;
    if (a.width <= 64) return dtype == DT_F16 ? pt_launch<64, DT_F16>(a, sms, m, work, s) : pt_launch<64, DT_BF16>(a, sms, m, work, s);
    return dtype == DT_F16 ? pt_launch<128, DT_F16>(a, sms, m, work, s) : pt_launch<128, DT_BF16>(a, sms, m, work, s);
}

}  // namespace tcu

// Products of matrices in microscaled four-bit floating point on the 5th-generation tensor cores (tcgen05, block-scaled):
// y = act(x W^T + bias) + residual.
//
// The matrix unit takes the stored codes and scales as they are: a tile is 128 outputs (rows of W, the unit's A) by up to 256
// rows of x (its B), K in steps of 256 columns, 128 bytes of codes a row, by TMA into shared memory; the scales come by bulk
// copies and go on to tensor memory. W on the unit's side of 128 serves one row and thousands alike: few rows make a narrow
// tile, and the weights stream at the memory's rate with no instruction of a thread's spent on them.
// What bounds it: of many rows the matrix unit (4096 x 14336 x 8192 bf16 out: 259 us, 3.7 PFLOP/s, its queue busy in 74%, its tensor pipe in 54%); of few the
// weights (8 rows of that: 14.6 us, 66 MB at 4.5 TB/s, of which 4 us are start and output); below that launch and latency (one row,
// 1024 x 512: 6.5 us). A step's issue in a loop that worked out its descriptors and divided by the number of slots took 353 and
// 24 us, outputs in code for all of a thread's 128 sums 930 us (the instruction caches did not hold it).
#include <cudaTypedefs.h>

#include <algorithm>
#include <type_traits>

#include "device.cuh"
#include "fp4.cuh"
#include "kv4_tc.cuh"

namespace tcu {

constexpr int FL_THREADS = 384, FL_M = 128, FL_STEP = 256, FL_STAGES = 8;
constexpr int FL_A = FL_M * FL_STEP / 2;  // bytes of a step's weights
constexpr size_t FL_SMEM = 225 * 1024;

struct FlPlan {
    int nt, row_tiles, feat_tiles, steps, stages, nacc, chunk, blocks, quads, group, split;
    unsigned stage_bytes, sf_a, sf_b, slot, acc_cols;
    long long total;
};

// Instruction descriptor of a block-scaled product of two e2m1 operands, 128 x N: bits 4-5 and 29-30 which scales of a word
// B and A use, 7-9 and 10-11 the operands' type, 17-22 N / 8, 23 the scales' type (1: powers of two), 27-28 M / 128.
__device__ __forceinline__ uint32_t fl_idesc(int n, bool nv, int part) {
    return (uint32_t)part << 4 | 1u << 7 | 1u << 10 | (uint32_t)(n >> 3) << 17 | (nv ? 0u : 1u << 23) | 1u << 27 | (uint32_t)part << 29;
}
// 128-byte rows swizzled by 128 bytes, groups of 8 rows 1024 bytes apart; K-major.
__device__ __forceinline__ uint64_t fl_desc(uint32_t addr) {
    return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
template <bool NV>
__device__ __forceinline__ void fl_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t acc) {
    if constexpr (NV)
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(acc)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}\n" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(acc)
            : "memory");
}
// 512 bytes of scales (32 rows of 16) to 4 columns of tensor memory, once for each warp's lanes.
__device__ __forceinline__ void fl_scales(uint32_t to, uint64_t from) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void fl_expect(uint64_t *m, uint32_t bytes) {
    asm volatile("{\n\t.reg .b64 st;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 st, [%0], %1;\n\t}\n" ::"r"(smem_addr(m)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void fl_tile(uint32_t to, const CUtensorMap *map, int x, int y, uint64_t *m) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(to),
                 "l"(map), "r"(x), "r"(y), "r"(smem_addr(m))
                 : "memory");
}
__device__ __forceinline__ void fl_bulk(uint32_t to, const void *from, uint32_t bytes, uint64_t *m) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(from), "r"(bytes),
                 "r"(smem_addr(m))
                 : "memory");
}

// GELU. For 16-bit results the quotient and the exponential are the unit's own (2^-21 off), and the formula for |x| >= 0.5 serves
// all: 1.5e-7 off in erf.
template <int DT>
__device__ __forceinline__ float fl_gelu(float v) {
    if constexpr (DT == DT_F32) return gelu1(v);
    const float a = fabsf(v) * 0.70710678118654752440f;
    float t, e;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fmaf(0.3275911f, a, 1.f)));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(a * a * -1.44269504088896340736f));
    float p = fmaf(1.0614054f, t, -1.4531521f);
    p = fmaf(p, t, 1.4214138f), p = fmaf(p, t, -0.28449674f), p = fmaf(p, t, 0.2548296f);
    const float half = 0.5f * p * t * e;  // of 1 - erf(a)
    return v * (v < 0.f ? half : 1.f - half);
}

// Tile t's place: groups of `group` row tiles, in them the row tiles innermost, so that blocks at work at the same time share
// weights and rows in L2.
__device__ __forceinline__ int2 fl_place(const FlPlan &p, int t) {
    const int per = p.group * p.feat_tiles, g = t / per, in = t - g * per, rows = min(p.group, p.row_tiles - g * p.group);
    return make_int2(g * p.group + in % rows, in / rows);
}

// Warp 0: the copies; warp 1: the products; warps 4-11: sums from tensor memory, joining and output, a thread one output of
// half the tile's rows. The steps of all tiles in a row are cut evenly over the blocks; parts of a tile meet in the working
// memory, and the last block to arrive joins them in order. OWN: rows of a tile that a thread takes at most.
template <int DT, bool NV, int OWN>
__global__ void __launch_bounds__(FL_THREADS, 1) k_fp4_linear(Fp4LinearArgs a, FlPlan p, const __grid_constant__ CUtensorMap map_w,
                                                              const __grid_constant__ CUtensorMap map_x, float *part, int *arrived) {
    using T = typename Elem<DT>::T;
    constexpr int QS = NV ? 4 : 2;  // blocks of 4 scales in a step
    extern __shared__ uint8_t smraw[];
    __shared__ __align__(8) uint64_t m_full[FL_STAGES], m_empty[FL_STAGES], m_acc[2], m_free[2], m_done;
    __shared__ uint32_t tslot;
    __shared__ volatile int abort_flag;
    __shared__ volatile int s_last;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t base = (smem_addr(smraw) + 1023u) & ~1023u;
    if (tid == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
    }
    if (warp == 2) {
        tmem_alloc(&tslot, 512);
        tmem_relinquish();
    }
    if (tid == 0) {
        for (int i = 0; i < FL_STAGES; i++) mbar_init(&m_full[i], 1), mbar_init(&m_empty[i], 1);
        for (int i = 0; i < 2; i++) mbar_init(&m_acc[i], 1), mbar_init(&m_free[i], 256);
        mbar_init(&m_done, 1);
        mbar_init_fence();
        abort_flag = a.give_up & blockIdx.x & 1;
    }
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = tslot, sf0 = tmem + p.acc_cols;
    auto wait_warp = [&](uint64_t *m, uint32_t parity) {
        if (!mbar_test_wait(m, parity) && !abort_flag && !mbar_wait(m, parity, KT_WAIT)) abort_flag = 1;
        __syncwarp();
    };
    // the block's steps: an even share of all, or of whole tiles
    const long long per = p.split ? 1 : p.steps, all = p.total / per;
    long long pos = ka_div(all * blockIdx.x, gridDim.x) * per;
    const long long end = ka_div(all * (blockIdx.x + 1), gridDim.x) * per;

    if (warp == 0) {
        int asked = 0, slot = 0;  // (asked: steps whose copies have been asked for; none after a wait has given up)
        uint32_t turn = 0;  // how often the slots have been filled (its lowest bit: a division by a number of slots known at run time costs more)
        while (pos < end) {
            const int t = (int)ka_div(pos, p.steps), s0 = (int)(pos - (long long)t * p.steps), s1 = (int)min((long long)p.steps, s0 + end - pos);
            const int2 place = fl_place(p, t);
            const uint8_t *wa = a.w_scales + (size_t)place.y * p.quads * 512;
            const int row_block = place.x * p.nt / 128, blocks = min((p.nt + 127) / 128, (a.rows + 127) / 128 - row_block);
            const uint8_t *xa = a.x_scales + (size_t)row_block * p.quads * 512;
            for (int s = s0; s < s1; s++) {
                if (turn) wait_warp(&m_empty[slot], (turn - 1) & 1u);
                if (__any_sync(0xffffffffu, abort_flag != 0)) break;
                asked++;
                const int quads = min(QS, p.quads - s * QS);
                if (elect_one()) {
                    const uint32_t to = base + slot * p.stage_bytes;
                    fl_expect(&m_full[slot], FL_A + p.nt * 128 + quads * 512 * (1 + blocks));
                    fl_tile(to, &map_w, s * 128, place.y * FL_M, &m_full[slot]);
                    fl_tile(to + FL_A, &map_x, s * 128, place.x * p.nt, &m_full[slot]);
                    fl_bulk(to + p.sf_a, wa + (size_t)s * QS * 512, quads * 512, &m_full[slot]);
                    for (int b = 0; b < blocks; b++)
                        fl_bulk(to + p.sf_b + b * QS * 512, xa + ((size_t)b * p.quads + s * QS) * 512, quads * 512, &m_full[slot]);
                }
                __syncwarp();
                if (++slot == p.stages) slot = 0, turn++;
            }
            pos += s1 - s0;
        }
        // what was asked for lands before the block lets go of shared memory
        for (int i = max(0, asked - p.stages); i < asked; i++) mbar_wait(&m_full[i % p.stages], (uint32_t)(i / p.stages) & 1u, KT_WAIT);
    } else if (warp == 1) {
        int c = 0, slot = 0;
        uint32_t turn = 0;
        const bool two = p.nt > 128;
        const uint64_t da0 = fl_desc(base), db0 = fl_desc(base + FL_A), sfa0 = smem_desc(base + p.sf_a, 16, 128), sfb0 = smem_desc(base + p.sf_b, 16, 128);
        const uint32_t id0 = fl_idesc(p.nt, NV, 0), id2 = fl_idesc(p.nt, NV, 2);
        // a step's scales to tensor memory, then its products; Q blocks of 4 scales, a number known when compiled for all but a row's
        // last step (descriptors worked out in a loop cost the issuing thread about a hundred cycles each)
        auto issue = [&](auto blocks, int quads, uint32_t d, uint32_t off, uint32_t sa, bool first) {
            constexpr int Q = decltype(blocks)::value;
            const uint64_t da = da0 + off, db = db0 + off, fa = sfa0 + off, fb = sfb0 + off;
            const uint32_t sb = sa + QS * 4;
#pragma unroll
            for (int q = 0; q < Q; q++) {
                if (q >= quads) break;
                fl_scales(sa + q * 4, fa + q * 32);
                if (two)
                    fl_scales(sb + q * 8, fb + q * 32), fl_scales(sb + q * 8 + 4, fb + (QS + q) * 32);
                else
                    fl_scales(sb + q * 4, fb + q * 32);
            }
#pragma unroll
            for (int q = 0; q < Q; q++) {
                if (q >= quads) break;
                const uint32_t qa = sa + q * 4, qb = sb + q * (two ? 8 : 4);
                if constexpr (NV) {
                    fl_mma<NV>(d, da + q * 2, db + q * 2, id0, qa, qb, !first || q > 0);
                } else {
                    fl_mma<NV>(d, da + q * 4, db + q * 4, id0, qa, qb, !first || q > 0);
                    fl_mma<NV>(d, da + q * 4 + 2, db + q * 4 + 2, id2, qa, qb, 1);
                }
            }
        };
        while (pos < end) {
            const int t = (int)ka_div(pos, p.steps), s0 = (int)(pos - (long long)t * p.steps), s1 = (int)min((long long)p.steps, s0 + end - pos);
            for (int from = s0; from < s1; from += p.chunk, c++) {
                const int to = min(s1, from + p.chunk), acc = c & (p.nacc - 1), turns = c >> (p.nacc - 1);
                if (turns) wait_warp(&m_free[acc], (uint32_t)(turns - 1) & 1u);
                fence_after_sync();
                const uint32_t d = tmem + acc * (p.acc_cols / p.nacc);
                for (int s = from; s < to; s++) {
                    wait_warp(&m_full[slot], turn & 1u);
                    fence_after_sync();
                    const int quads = min(QS, p.quads - s * QS);
                    const uint32_t off = (slot * p.stage_bytes) >> 4, sa = sf0 + slot * p.slot;
                    if (elect_one()) {
                        if (quads == QS)
                            issue(std::integral_constant<int, QS>{}, QS, d, off, sa, s == from);
                        else
                            issue(std::integral_constant<int, QS - 1>{}, quads, d, off, sa, s == from);
                        mma_commit(&m_empty[slot]);
                        if (s == to - 1) mma_commit(&m_acc[acc]);
                    }
                    __syncwarp();
                    if (++slot == p.stages) slot = 0, turn++;
                }
            }
            pos += s1 - s0;
        }
        if (elect_one()) {
            mma_commit(&m_done);
            mbar_wait(&m_done, 0, KT_WAIT);
        }
        __syncwarp();
    } else if (warp >= 4) {
        const int quad = warp & 3, half = (warp - 4) >> 2, cols = p.nt > 16 ? (p.nt / 2 + 15) & ~15 : 16, c0 = half * cols, own = min(cols, p.nt - c0);
        int c = 0;
        while (pos < end) {
            const int t = (int)ka_div(pos, p.steps), s0 = (int)(pos - (long long)t * p.steps), s1 = (int)min((long long)p.steps, s0 + end - pos);
            const int2 place = fl_place(p, t);
            const bool whole = s0 == 0 && s1 == p.steps;
            const int n = place.y * FL_M + quad * 32 + lane, row0 = place.x * p.nt + c0;
            const float bias = a.bias && n < a.n ? Elem<DT>::get(reinterpret_cast<const T *>(a.bias)[n]) : 0.f;
            T *y = reinterpret_cast<T *>(a.y) + (size_t)row0 * a.ldy + n;
            const T *r = reinterpret_cast<const T *>(a.residual) + (a.residual ? (size_t)row0 * a.ldr + n : 0);
            // The residual of a narrow tile of a 16-bit type is loaded whole before its products are waited for, two rows a register: a
            // load waits for the copies asked for before it, some 3,000 cycles (4096 x 8192 x 2048, bf16: 65 us without a residual, 115
            // to 125 so, 152 with one asked for 16 rows ahead, 160 in tiles of 256 rows, whose sums leave no registers for either).
            constexpr bool EARLY = OWN <= 64 && DT != DT_F32;
            uint32_t held[EARLY ? OWN / 2 : 1];
            if constexpr (EARLY) {
                const int rows = a.residual && n < a.n ? min(own, a.rows - row0) : 0;
                const uint16_t *q = reinterpret_cast<const uint16_t *>(r);
#pragma unroll
                for (int i = 0; i < OWN / 2; i++) held[i] = 0;
                if (rows > 0) {
#pragma unroll
                    for (int i = 0; i < OWN / 2; i++)
                        held[i] = (2 * i < rows ? q[(size_t)(2 * i) * a.ldr] : 0u) | (2 * i + 1 < rows ? (uint32_t)q[(size_t)(2 * i + 1) * a.ldr] << 16 : 0u);
                }
            }
            float v[OWN];
#pragma unroll
            for (int i = 0; i < OWN; i++) v[i] = 0.f;
            for (int from = s0; from < s1; from += p.chunk, c++) {
                const int acc = c & (p.nacc - 1);
                wait_warp(&m_acc[acc], (uint32_t)(c >> (p.nacc - 1)) & 1u);
                fence_after_sync();
                const uint32_t d = tmem + acc * (p.acc_cols / p.nacc) + c0 + ((uint32_t)(quad * 32) << 16);
#pragma unroll
                for (int g = 0; g < OWN / 16; g++) {
                    if (g * 16 < own) {
                        float x[16];
                        tmem_ld16(d + g * 16, x);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; i++) v[g * 16 + i] += x[i];
                    }
                }
                fence_before_sync();
                mbar_arrive(&m_free[acc]);
            }
            // 16 rows' outputs from their sums, of which `rows` there are; f32 residuals are asked for 16 rows ahead
            constexpr bool AHEAD = DT == DT_F32;
            float next[16];
            auto ask = [&](int rows) {
                if (!a.residual) return;
#pragma unroll
                for (int i = 0; i < 16; i++) next[i] = i < rows ? Elem<DT>::get(r[(size_t)i * a.ldr]) : 0.f;
                r += (size_t)16 * a.ldr;
            };
            auto put = [&](const float *sum, int rows) {
                float f[16];
                if (EARLY && a.residual) {
#pragma unroll
                    for (int i = 0; i < 16; i++) {
                        const uint16_t h = (uint16_t)(held[i / 2] >> (i & 1) * 16);
                        f[i] = Elem<DT>::get(*reinterpret_cast<const T *>(&h));
                    }
#pragma unroll
                    for (int i = 0; i < OWN / 2 - 8; i++) held[i] = held[i + 8];
                } else {
                    if constexpr (!AHEAD) ask(rows);
#pragma unroll
                    for (int i = 0; i < 16; i++) f[i] = a.residual ? next[i] : 0.f;
                    if constexpr (AHEAD) ask(rows - 16);
                }
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    float g = fmaf(sum[i], a.alpha, bias);
                    if (a.act) g = fl_gelu<DT>(g);
                    if (i < rows) y[(size_t)i * a.ldy] = Elem<DT>::put(g + f[i]);
                }
                y += (size_t)16 * a.ldy;
            };
            const int rows = n < a.n && !abort_flag ? min(own, a.rows - row0) : 0;
            if constexpr (AHEAD) ask(rows);
            if (whole) {
                // 16 values at a time, the others moved up behind them: code for all 128 would not stay in the instruction caches (a
                // call of one row took 24 us so)
#pragma unroll 1
                for (int there = rows; there > 0; there -= 16) {
                    put(v, there);
#pragma unroll
                    for (int i = 0; i < OWN - 16; i++) v[i] = v[i + 16];
                }
            } else {
                // parts: each block's into its slot (the tile's first block's into its second slot, the others' into their first)
                const long long u0 = (long long)t * p.steps;
                const int b0 = (int)ka_div((u0 + 1) * gridDim.x - 1, p.total), b1 = (int)ka_div((u0 + p.steps) * gridDim.x - 1, p.total);
                const size_t size = (size_t)FL_M * p.nt;
                float *at = part + c0 * FL_M + quad * 32 + lane, *to = at + (2 * (size_t)blockIdx.x + (s0 == 0)) * size;
#pragma unroll
                for (int g = 0; g < OWN / 16; g++)
                    if (g * 16 < own) {
#pragma unroll
                        for (int i = 0; i < 16; i++) __stcg(to + (g * 16 + i) * FL_M, v[g * 16 + i]);
                    }
                kt_bar(1, 256);
                if (tid == 128) {
                    __threadfence();  // (after the barrier: for all that the block has stored)
                    const int before = atomicAdd(&arrived[b0], 1);
                    s_last = before == b1 - b0;
                    if (s_last) arrived[b0] = 0;
                    __threadfence();
                }
                kt_bar(1, 256);
                if (s_last) {
#pragma unroll 1
                    for (int g = 0; g < own && g < rows; g += 16) {
                        float sum[16] = {};
#pragma unroll 1
                        for (int b = b0; b <= b1; b++) {
                            const float *in = at + (2 * (size_t)b + (b == b0)) * size + g * FL_M;
                            float x[16];
#pragma unroll
                            for (int i = 0; i < 16; i++) x[i] = __ldcg(in + i * FL_M);
#pragma unroll
                            for (int i = 0; i < 16; i++) sum[i] += x[i];
                        }
                        put(sum, rows - g);
                    }
                }
            }
            pos += s1 - s0;
        }
    }
    fence_before_sync();
    __syncthreads();
    if (tid == 0 && abort_flag) *reinterpret_cast<volatile int *>(a.err_wait) = 1;
    fence_after_sync();
    if (warp == 2) tmem_dealloc(tmem, 512);
}

static FlPlan fl_plan(int dtype, const Fp4LinearArgs &a, int sms) {
    FlPlan p;
    const bool nv = a.format == FP4_NV;
    const int kp = fp4_padded(a.k), qs = nv ? 4 : 2;
    p.quads = fp4_quads(a.k, a.format), p.steps = (kp + FL_STEP - 1) / FL_STEP;
    p.feat_tiles = (a.n + FL_M - 1) / FL_M;
    // How many rows a tile has, and over how many blocks it is cut: what takes the fewest cycles, from what was measured (8 to 4096
    // rows): a step 420 and 3 a row of the tile, a tile's output 1000 and 12 a row, 20000 more for a residual in a tile of 256; the parts of a cut tile 7000 and 100 a row for
    // storing and waiting, and each part 600 and 25 a row in the block that joins them (2048 x 1024 x 4096: whole tiles of 128 rows
    // 15.6 us, cut over all SMs 27.2; of 256 rows 20.9 and 39.3. 4096 x 14336 x 8192: of 256 rows 255 us, of 128 330).
    const int widest = std::min(dtype == DT_F32 ? 128 : 256, (a.rows + 15) / 16 * 16);
    double best = 0;
    p.nt = 0;
    for (int nt : {16, 32, 48, 64, 96, 128, 256, widest}) {
        if (nt > 128) nt = 256;
        if (nt > 128 ? widest <= 128 : nt > widest || (a.rows > nt && nt % 128)) continue;  // (a tile begins with a block of scales)
        const long long tiles = (long long)((a.rows + nt - 1) / nt) * p.feat_tiles;
        const double step = 420 + 3.0 * nt, out = 1000 + 12.0 * nt + (a.residual && nt > 128 ? 20000 : 0);
        for (int parts = 1; parts <= 32 && parts <= p.steps; parts *= 2) {
            if (parts > 1 && tiles * parts > 2 * sms) break;
            const long long blocks = std::min<long long>(sms, tiles * parts);
            const double turns = parts > 1 ? (double)tiles / blocks : std::ceil((double)tiles / blocks);
            const double cost = turns * p.steps * step + std::ceil(turns) * out + (parts > 1 ? 7000 + 100.0 * nt + parts * (600 + 25.0 * nt) : 0);
            if (!p.nt || cost < best) best = cost, p.nt = nt, p.split = parts > 1, p.blocks = (int)blocks;
        }
    }
    // The matrix unit rounds its sums towards zero, so a sum runs over a number of steps in it, from there on in registers: f32 results
    // over 4, with two narrower accumulators in turn, so that the unit does not wait for them to be read; 16-bit ones over 64, whose
    // 256 additions leave 2^-17 of a sum of one sign (all of 262,144 columns: 2^-14, a seventh of a half of f16's last place).
    p.chunk = dtype == DT_F32 ? 4 : std::min(64, p.steps);
    p.nacc = p.nt > 128 ? 1 : 2;
    int cols = 32;
    while (cols < p.nt) cols *= 2;
    p.acc_cols = (unsigned)(cols * p.nacc);
    p.row_tiles = (a.rows + p.nt - 1) / p.nt;
    p.sf_a = (unsigned)(FL_A + p.nt * 128), p.sf_b = p.sf_a + qs * 512;
    p.stage_bytes = (p.sf_b + qs * 512 * (p.nt > 128 ? 2 : 1) + 1023) / 1024 * 1024;
    p.slot = (unsigned)(qs * (4 + (p.nt > 128 ? 8 : 4)));
    p.stages = (int)std::min<size_t>(FL_STAGES, (FL_SMEM - 1024) / p.stage_bytes);
    p.stages = std::min<int>(p.stages, (int)((512 - p.acc_cols) / p.slot));
    p.group = 8;
    p.total = (long long)p.row_tiles * p.feat_tiles * p.steps;
    return p;
}

size_t fp4_linear_workspace(int dtype, const Fp4LinearArgs &a, int sms) {
    // (for a call with a residual and for one without: the plan is not the same)
    Fp4LinearArgs b = a;
    size_t parts = 0;
    for (const void *residual : {(const void *)nullptr, (const void *)&b}) {
        b.residual = residual;
        const FlPlan p = fl_plan(dtype, b, sms);
        parts = std::max(parts, p.split ? (size_t)p.blocks * 2 * FL_M * p.nt * sizeof(float) : 0);
    }
    return sizeof(int) * KA_BLOCKS + parts;
}

static bool fl_map(void *encode, CUtensorMap *m, const uint8_t *codes, int rows, int k, int box) {
    const cuuint64_t dims[2] = {(cuuint64_t)fp4_padded(k) / 2, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)fp4_padded(k) / 2};
    const cuuint32_t boxes[2] = {FL_STEP / 2, (cuuint32_t)box}, one[2] = {1, 1};
    return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(encode)(
               m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t *>(codes), dims, strides, boxes, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DT, bool NV, int OWN>
static cudaError_t launch(const Fp4LinearArgs &a, const FlPlan &p, const CUtensorMap &w, const CUtensorMap &x, void *work, cudaStream_t s) {
    const size_t smem = (size_t)p.stages * p.stage_bytes + 1024;
    const cudaError_t e = allow_dynamic_smem((const void *)k_fp4_linear<DT, NV, OWN>, FL_SMEM);
    if (e != cudaSuccess) return e;
    int *arrived = reinterpret_cast<int *>(work);
    k_fp4_linear<DT, NV, OWN><<<p.blocks, FL_THREADS, smem, s>>>(a, p, w, x, reinterpret_cast<float *>(arrived + KA_BLOCKS), arrived);
    return cudaGetLastError();
}
template <int DT, bool NV>
static cudaError_t launch(const Fp4LinearArgs &a, const FlPlan &p, const CUtensorMap &w, const CUtensorMap &x, void *work, cudaStream_t s) {
    if constexpr (DT != DT_F32)
        if (p.nt > 128) return launch<DT, NV, 128>(a, p, w, x, work, s);
    return launch<DT, NV, 64>(a, p, w, x, work, s);
}

cudaError_t launch_fp4_linear(int dtype, const Fp4LinearArgs &a, int sms, void *encode, void *work, cudaStream_t s, uint64_t *launches) {
    const FlPlan p = fl_plan(dtype, a, sms);
    CUtensorMap w, x;
    if (!encode || !fl_map(encode, &w, a.w, a.n, a.k, FL_M) || !fl_map(encode, &x, a.x, a.rows, a.k, p.nt)) return cudaErrorNotSupported;
    (*launches)++;
    const bool nv = a.format == FP4_NV;
    return dtype == DT_F32   ? (nv ? launch<DT_F32, true>(a, p, w, x, work, s) : launch<DT_F32, false>(a, p, w, x, work, s))
           : dtype == DT_F16 ? (nv ? launch<DT_F16, true>(a, p, w, x, work, s) : launch<DT_F16, false>(a, p, w, x, work, s))
                             : (nv ? launch<DT_BF16, true>(a, p, w, x, work, s) : launch<DT_BF16, false>(a, p, w, x, work, s));
}

}  // namespace tcu

// Attention of packed rows over keys and values as they are, for few rows of any type, and for what the tensor-core kernels
// (packed_attend_tc.cu, packed_attend_tc32.cu) do not take: widths above 128, 16-bit rows that TMA cannot fetch.
//
// 16 or 64 query rows of one key head (the heads that share it side by side) against steps of 64 keys (f32: 32) that come by
// asynchronous copies. With 16 rows the four warps share a step's keys, with 64 its rows. One pass: running maxima and sums, the
// output in registers, the matrix products by warp (16-bit operands as they are; f32 as two tf32, of 11 bits each, in three
// products). A call of few rows streams its keys and values, so it is bound by memory; the steps of all sequences are cut evenly
// over the blocks (kv4_plan.cuh), whose parts the last of them joins in order. f16 weights are multiplied by 2^15, so that they fill
// f16's range. Rows whose weighted sum passes f32 before it is divided are worked out again by themselves. 32 requests of 0 to 16,383 bf16 tokens, 32 heads on 8 of
// width 128: 188 us for 1.05 GB, 5.6 TB/s (343 us with a division for every 16 bytes copied).
#include <algorithm>
#include <climits>
#include <type_traits>

#include "packed.cuh"

namespace tcu {

constexpr int PA_THREADS = 128;
// What a unit costs besides its steps, in steps, and the steps that a block takes at least: so that units of one step are a block's
// each (21 rows of 32 heads on 8 of width 256: 81 us with four units a block), and shorter parts of longer ones are not joined.
constexpr int PA_EXTRA = 4, PA_STEPS = 5;
// Steps of 16-bit keys over which a product's sums run in the matrix unit, which rounds them towards zero (1.1e-7 of one an
// addition, of values of one sign); from there on they are added in the working memory.
constexpr int PA_FOLD = 128;

template <int DT, int HD_, int WR>
struct PaShape {
    static constexpr int HD = HD_;
    using T = typename Elem<DT>::T;
    static constexpr bool F32 = DT == DT_F32;
    using Raw = std::conditional_t<F32, uint32_t, uint16_t>;
    static constexpr int R = 16 * WR, KW = 4 / WR, BK = F32 ? 32 : 64, OWN = BK / KW;
    static constexpr int PITCH = HD * (int)sizeof(T) + 16;  // bytes of a row: rows 4 banks apart
    static constexpr int STAGES = !F32 && WR == 1 && HD <= 128 ? 3 : 2;
    static constexpr int TILE = BK * PITCH, CP = HD + 4;
    static constexpr size_t SMEM = (size_t)STAGES * 2 * TILE + R * PITCH;
    static constexpr size_t PART = (size_t)R * (HD + 2);  // floats of a part: outputs, maxima, sums
    static constexpr size_t SUMS = (size_t)PA_THREADS * HD / 2;  // floats of a block's folded sums
    static_assert((size_t)64 * CP * 4 + 512 <= (size_t)STAGES * 2 * TILE, "the warps' outputs meet where keys and values were");
};

__device__ __forceinline__ uint32_t pa_smem(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void pa_ldsm(uint32_t at, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void pa_ldsm_t(uint32_t at, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
template <int DT>
__device__ __forceinline__ void pa_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (DT == DT_F16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else if constexpr (DT == DT_BF16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// x = hi + lo, two tf32 (11 bits each, rounded to nearest).
__device__ __forceinline__ void pa_split(float x, uint32_t &hi, uint32_t &lo) {
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(x - __uint_as_float(hi)));
}
__device__ __forceinline__ float pa_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
template <int DT>
__device__ __forceinline__ uint32_t pa_pair(float x, float y) {
    if constexpr (DT == DT_F16) {
        const __half2 h = __floats2half2_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&h);
    } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}

// Rows [0, n) of `width` elements, `row` elements apart, into shared rows of PITCH bytes, by all threads; rows outside [lo, hi)
// are zeros. Whole 16-byte pieces asynchronously where they are aligned.
template <class C>
__device__ __forceinline__ void pa_copy(uint8_t *to, const void *base, long long first, long long row, int lo, int hi, int width, bool wide) {
    using Raw = typename C::Raw;
    constexpr int PER = 16 / (int)sizeof(Raw);
    const Raw *from = reinterpret_cast<const Raw *>(base);
    if (wide) {
        // a thread the same 16 bytes of every ROWS-th row
        constexpr int LANES = C::HD / PER, ROWS = PA_THREADS / LANES;
        const int c = threadIdx.x % LANES, r0 = threadIdx.x / LANES;
        if (c * PER < width) {
            const Raw *at = from + first + r0 * row + c * PER;
            const uint32_t dst = pa_smem(to + r0 * C::PITCH + c * 16);
#pragma unroll
            for (int x = 0; x < C::BK / ROWS; x++, at += ROWS * row) {
                const int r = r0 + x * ROWS;
                const bool in = r >= lo && r < hi;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + x * ROWS * C::PITCH), "l"(in ? at : from), "r"(in ? 16 : 0) : "memory");
            }
        }
    } else {
        for (int i = threadIdx.x; i < C::BK * width; i += PA_THREADS) {
            const int r = i / width, c = i - r * width;
            *reinterpret_cast<Raw *>(to + r * C::PITCH + c * sizeof(Raw)) = r >= lo && r < hi ? from[first + r * row + c] : Raw(0);
        }
    }
}

template <int DT, int HD, int WR>
__global__ void __launch_bounds__(PA_THREADS) k_packed_attend(PackedArgs a, int wide, float *part, float *sums, int *arrived) {
    using C = PaShape<DT, HD, WR>;
    using T = typename C::T;
    using Raw = typename C::Raw;
    using Cut = KaCut<C::R, 1, C::BK, PA_EXTRA>;
    constexpr int R = C::R, KW = C::KW, BK = C::BK, OWN = C::OWN, NT = OWN / 8, NO = HD / 8, STAGES = C::STAGES, PITCH = C::PITCH, CP = C::CP;
    extern __shared__ __align__(16) uint8_t sm[];
    uint8_t *Qs = sm + (size_t)STAGES * 2 * C::TILE;
    __shared__ long long s_sum[PA_THREADS / 32];
    __shared__ int s_unit[4], s_last;
    __shared__ int s_bad[R];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3, wr = warp % WR, kw = warp / WR;
    const int each = a.q_heads / a.c.heads;
    const float sl = a.scale * 1.44269504088896340736f;
    constexpr float UP = DT == DT_F16 ? 0x1p15f : 1.f, DOWN = 1.f / UP;  // what 16-bit weights are multiplied by, their outputs at the end
    auto pl = Cut::template place<PA_THREADS>(a, each, PA_STEPS, s_sum, s_unit);
    while (pl.pos < pl.end) {
        const KaRows sr = ka_rows(a, pl.seq);
        const auto sp = Cut::span(a, sr, each, pl.rt);
        // `count` of the unit's steps as they are cut, n of keys
        const int count = (int)min((long long)(sp.steps - pl.skip), pl.end - pl.pos), skipped = max(0, pl.skip - PA_EXTRA);
        const int n = max(0, pl.skip + count - PA_EXTRA) - skipped, j0 = sp.base + skipped * BK, k0 = a.k_starts[pl.seq];
        const int r0 = pl.rt * R, rows = min(R, sr.n * each - r0);
        __syncthreads();  // the piece before is done with shared memory
        if (a.width < HD) {
            for (int i = tid; i < (int)(C::SMEM / 16); i += PA_THREADS) reinterpret_cast<uint4 *>(sm)[i] = make_uint4(0, 0, 0, 0);
            __syncthreads();
        }
        {
            // the queries, 16 bytes a thread, 8 on their way together (one after the other they took 200 us for 64 rows of 256)
            constexpr int PER = 16 / (int)sizeof(Raw), LANES = HD / PER, ROWS = PA_THREADS / LANES, N = R / ROWS < 1 ? 1 : R / ROWS, TURN = N < 8 ? N : 8;
            const int c = tid % LANES, first = tid / LANES;
#pragma unroll 1
            for (int x = 0; x < N; x += TURN) {
                uint4 w[TURN];
#pragma unroll
                for (int y = 0; y < TURN; y++) w[y] = make_uint4(0, 0, 0, 0);
                auto from = [&](int y) {
                    const int p = r0 + first + (x + y) * ROWS, i = p / each;
                    return reinterpret_cast<const Raw *>(a.q) + (long long)(sr.first + i) * a.q_row + (long long)(pl.head * each + p - i * each) * a.q_head + c * PER;
                };
                if (wide & 4) {
#pragma unroll
                    for (int y = 0; y < TURN; y++)
                        if (first + (x + y) * ROWS < rows && c * PER < a.width) w[y] = __ldg(reinterpret_cast<const uint4 *>(from(y)));
                } else {
#pragma unroll
                    for (int y = 0; y < TURN; y++)
                        if (first + (x + y) * ROWS < rows && c * PER < a.width) {
                            __align__(16) Raw e[PER];
                            const Raw *q = from(y);
#pragma unroll
                            for (int z = 0; z < PER; z++) e[z] = q[z];
                            w[y] = *reinterpret_cast<const uint4 *>(e);
                        }
                }
#pragma unroll
                for (int y = 0; y < TURN; y++)
                    if (first + (x + y) * ROWS < R) *reinterpret_cast<uint4 *>(Qs + (first + (x + y) * ROWS) * PITCH + c * 16) = w[y];
            }
        }
        auto load = [&](int i) {
            const int at = j0 + i * BK, slot = i % STAGES;
            if (i < n) {
                pa_copy<C>(sm + (size_t)slot * 2 * C::TILE, a.k, (long long)(k0 + at) * a.k_row + pl.head * a.k_head, a.k_row, 0, sp.hi_max - at, a.width, wide & 1);
                pa_copy<C>(sm + (size_t)(slot * 2 + 1) * C::TILE, a.v, (long long)(k0 + at) * a.v_row + pl.head * a.v_head, a.v_row, 0, sp.hi_max - at, a.width,
                           wide & 2);
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int i = 0; i < STAGES - 1; i++) load(i);

        // this thread's rows of a fragment: g and g + 8
        int lo[2], hi[2];
#pragma unroll
        for (int x = 0; x < 2; x++) {
            const int r = 16 * wr + g + 8 * x, i = (r0 + r) / each;
            lo[x] = r < rows ? ka_lo(a, sr, i) : 0, hi[x] = r < rows ? ka_hi(a, sr, i) : 0;
        }
        float o[NO][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NO; i++)
#pragma unroll
            for (int x = 0; x < 4; x++) o[i][x] = 0.f;

        // the sums of the steps before, and the maxima that they are relative to
        float4 *kept = reinterpret_cast<float4 *>(sums) + blockIdx.x * (C::SUMS / 4) + tid;
        float m_kept[2] = {-INFINITY, -INFINITY};
        auto kept_by = [&](int x) { return m_kept[x] == -INFINITY ? 0.f : pa_ex2(m_kept[x] - m[x]); };
        constexpr int FOLD = C::F32 ? INT_MAX : PA_FOLD;
#pragma unroll 1
        for (int i0 = 0; i0 < n; i0 += FOLD) {
            for (int i = i0; i < n && i - i0 < FOLD; i++) {
                asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
                __syncthreads();
                load(i + STAGES - 1);
                const uint8_t *ks = sm + (size_t)(i % STAGES) * 2 * C::TILE + kw * OWN * PITCH, *vs = ks + C::TILE;
                float s[NT][4];
#pragma unroll
                for (int x = 0; x < NT; x++)
#pragma unroll
                    for (int y = 0; y < 4; y++) s[x][y] = 0.f;
                if constexpr (C::F32) {
                    const float *qf = reinterpret_cast<const float *>(Qs + (16 * wr + g) * PITCH);
                    // (32 coordinates' sums at a time in the unit, which does not round them to nearest; these are added here)
#pragma unroll 1
                    for (int c0 = 0; c0 < HD; c0 += 32) {
                        float part[NT][4];
#pragma unroll
                        for (int x = 0; x < NT; x++)
#pragma unroll
                            for (int y = 0; y < 4; y++) part[x][y] = 0.f;
#pragma unroll
                        for (int c = c0; c < c0 + 32; c += 8) {
                            uint32_t h[4], lw[4];
                            pa_split(qf[c + t], h[0], lw[0]), pa_split(qf[8 * PITCH / 4 + c + t], h[1], lw[1]);
                            pa_split(qf[c + t + 4], h[2], lw[2]), pa_split(qf[8 * PITCH / 4 + c + t + 4], h[3], lw[3]);
#pragma unroll
                            for (int x = 0; x < NT; x++) {
                                const float *kf = reinterpret_cast<const float *>(ks + (8 * x + g) * PITCH) + c + t;
                                uint32_t bh[2], bl[2];
                                pa_split(kf[0], bh[0], bl[0]), pa_split(kf[4], bh[1], bl[1]);
                                pa_mma<DT>(part[x], lw, bh[0], bh[1]);
                                pa_mma<DT>(part[x], h, bl[0], bl[1]);
                                pa_mma<DT>(part[x], h, bh[0], bh[1]);
                            }
                        }
#pragma unroll
                        for (int x = 0; x < NT; x++)
#pragma unroll
                            for (int y = 0; y < 4; y++) s[x][y] += part[x][y];
                    }
                } else {
                    const uint32_t qa = pa_smem(Qs + (16 * wr + (lane & 15)) * PITCH + (lane >> 4) * 16);
                    const uint32_t ka = pa_smem(ks + ((lane & 7) + ((lane >> 4) << 3)) * PITCH + ((lane >> 3) & 1) * 16);
#pragma unroll
                    for (int c = 0; c < HD / 16; c++) {
                        uint32_t q[4];
                        pa_ldsm(qa + c * 32, q);
#pragma unroll
                        for (int x = 0; x < NT; x += 2) {
                            uint32_t b[4];
                            pa_ldsm(ka + 8 * x * PITCH + c * 32, b);
                            pa_mma<DT>(s[x], q, b[0], b[1]), pa_mma<DT>(s[x + 1], q, b[2], b[3]);
                        }
                    }
                }
                // scores in units of log2; what a row does not see goes, whatever it is
                const int at = j0 + i * BK + kw * OWN + 2 * t;
                const bool edge = j0 + i * BK < sp.lo_max || j0 + (i + 1) * BK > sp.hi_min || rows < R;
                float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int x = 0; x < NT; x++)
#pragma unroll
                    for (int y = 0; y < 4; y++) {
                        const int j = at + 8 * x + (y & 1);
                        float v = s[x][y] * sl;
                        if (edge && (j < lo[y >> 1] || j >= hi[y >> 1])) v = -INFINITY;
                        s[x][y] = v, top[y >> 1] = fmaxf(top[y >> 1], v);
                    }
                float f[2], ref[2];
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 1));
                    top[x] = fmaxf(fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 2)), m[x]);
                    ref[x] = top[x] == -INFINITY ? 0.f : top[x];
                    f[x] = m[x] == -INFINITY ? 0.f : pa_ex2(m[x] - ref[x]);
                }
                if (__any_sync(0xffffffffu, top[0] != m[0] || top[1] != m[1])) {
#pragma unroll
                    for (int x = 0; x < NO; x++)
#pragma unroll
                        for (int y = 0; y < 4; y++)
                            if (m[y >> 1] != -INFINITY) o[x][y] *= f[y >> 1];
                    l[0] *= f[0], l[1] *= f[1], m[0] = top[0], m[1] = top[1];
                }
#pragma unroll
                for (int x = 0; x < NT; x++)
#pragma unroll
                    for (int y = 0; y < 4; y++) s[x][y] = pa_ex2(s[x][y] - ref[y >> 1]), l[y >> 1] += s[x][y];
                if constexpr (C::F32) {
                    // A fragment's k takes the keys in the order in which a thread has their weights: k = t key 2 t, k = t + 4 key 2 t + 1.
                    // The unit does not round its sums to nearest, so each step's are its own, added here (over 10,000 keys 2.8e-5 of
                    // an output otherwise).
                    uint32_t h[NT][4], lw[NT][4];
#pragma unroll
                    for (int x = 0; x < NT; x++)
                        pa_split(s[x][0], h[x][0], lw[x][0]), pa_split(s[x][2], h[x][1], lw[x][1]), pa_split(s[x][1], h[x][2], lw[x][2]), pa_split(s[x][3], h[x][3], lw[x][3]);
#pragma unroll
                    for (int c = 0; c < NO; c++) {
                        float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int x = 0; x < NT; x++) {
                            const float *vf = reinterpret_cast<const float *>(vs + (8 * x + 2 * t) * PITCH) + 8 * c + g;
                            uint32_t bh[2], bl[2];
                            pa_split(vf[0], bh[0], bl[0]), pa_split(vf[PITCH / 4], bh[1], bl[1]);
                            pa_mma<DT>(sum, lw[x], bh[0], bh[1]);
                            pa_mma<DT>(sum, h[x], bl[0], bl[1]);
                            pa_mma<DT>(sum, h[x], bh[0], bh[1]);
                        }
#pragma unroll
                        for (int y = 0; y < 4; y++) o[c][y] += sum[y];
                    }
                } else {
                    const uint32_t va = pa_smem(vs + (lane & 15) * PITCH + (lane >> 4) * 16);
#pragma unroll
                    for (int x = 0; x < NT; x += 2) {
                        const uint32_t p[4] = {pa_pair<DT>(s[x][0] * UP, s[x][1] * UP), pa_pair<DT>(s[x][2] * UP, s[x][3] * UP),
                                               pa_pair<DT>(s[x + 1][0] * UP, s[x + 1][1] * UP), pa_pair<DT>(s[x + 1][2] * UP, s[x + 1][3] * UP)};
#pragma unroll
                        for (int c = 0; c < NO; c += 2) {
                            uint32_t b[4];
                            pa_ldsm_t(va + 8 * x * PITCH + c * 16, b);
                            pa_mma<DT>(o[c], p, b[0], b[1]), pa_mma<DT>(o[c + 1], p, b[2], b[3]);
                        }
                    }
                }
            }
            if (!C::F32 && n > FOLD) {
                const bool more = n - i0 > FOLD;
                const float f0 = kept_by(0), f1 = kept_by(1);
#pragma unroll
                for (int c = 0; c < NO; c++) {
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (i0) v = __ldcg(kept + c * PA_THREADS);
                    v = make_float4(fmaf(v.x, f0, o[c][0]), fmaf(v.y, f0, o[c][1]), fmaf(v.z, f1, o[c][2]), fmaf(v.w, f1, o[c][3]));
                    if (more) __stcg(kept + c * PA_THREADS, v), v = make_float4(0.f, 0.f, 0.f, 0.f);
                    o[c][0] = v.x, o[c][1] = v.y, o[c][2] = v.z, o[c][3] = v.w;
                }
                m_kept[0] = m[0], m_kept[1] = m[1];
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
        for (int x = 0; x < 2; x++) {
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 1);
            l[x] += __shfl_xor_sync(0xffffffffu, l[x], 2);
        }
        __syncthreads();

        // ---- the warps' outputs meet: [KW][R][HD], and maxima and sums [KW][R] ----
        float *oc = reinterpret_cast<float *>(sm), *mc = oc + 64 * CP, *lc = mc + 64;
#pragma unroll
        for (int x = 0; x < 2; x++) {
            const int r = kw * R + 16 * wr + g + 8 * x;
            if (t == 0) mc[r] = m[x], lc[r] = l[x];
#pragma unroll
            for (int c = 0; c < NO; c++) *reinterpret_cast<float2 *>(oc + r * CP + 8 * c + 2 * t) = make_float2(o[c][2 * x], o[c][2 * x + 1]);
        }
        __syncthreads();
        const bool whole = count == sp.steps;
        const int2 who = Cut::sharers(pl, pl.pos - pl.skip, sp.steps);
        constexpr int cols = HD / 4;  // of 4 columns
        // one row's `parts` states joined in 4 columns; at(p): where part p's outputs of the row lie, its maximum and its sum
        auto join = [&](int parts, auto at, float4 &v, float &M, float &L) {
            M = -INFINITY, L = 0.f, v = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int p = 0; p < parts; p++) M = fmaxf(M, *at(p).m);
            const float ref = M == -INFINITY ? 0.f : M;
            for (int p = 0; p < parts; p++) {
                const auto from = at(p);
                if (*from.m == -INFINITY && *from.l == 0.f) continue;
                const float w = pa_ex2(*from.m - ref);
                const float4 x = *reinterpret_cast<const float4 *>(from.o);
                L = fmaf(w, *from.l, L), v.x = fmaf(w, x.x, v.x), v.y = fmaf(w, x.y, v.y), v.z = fmaf(w, x.z, v.z), v.w = fmaf(w, x.w, v.w);
            }
        };
        struct From {
            const float *o, *m, *l;
        };
        bool write = true;
        if (!whole) {
            float *mine = part + Cut::slot(blockIdx.x, pl.skip == 0) * C::PART;
            for (int i = tid; i < rows * cols; i += PA_THREADS) {
                const int r = i / cols, c = (i - r * cols) * 4;
                if (c >= a.width) continue;
                float4 v;
                float M, L;
                join(KW, [&](int p) { return From{oc + (p * R + r) * CP + c, mc + p * R + r, lc + p * R + r}; }, v, M, L);
                __stcg(reinterpret_cast<float4 *>(mine + r * HD + c), v);
                if (c == 0) __stcg(mine + R * HD + r, M), __stcg(mine + R * HD + R + r, L);
            }
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const int before = atomicAdd(&arrived[who.x], 1);
                s_last = before == who.y - 1;
                if (s_last) arrived[who.x] = 0;
                __threadfence();
            }
            __syncthreads();
            write = s_last;
        }
        if (write) {
            for (int i = tid; i < R; i += PA_THREADS) s_bad[i] = 0;
            __syncthreads();
            for (int i = tid; i < rows * cols; i += PA_THREADS) {
                const int r = i / cols, c = (i - r * cols) * 4, p = r0 + r, in = p / each, hq = pl.head * each + p - in * each, row = sr.first + in;
                if (c >= a.width) continue;
                float4 v;
                float M, L;
                if (whole)
                    join(KW, [&](int p) { return From{oc + (p * R + r) * CP + c, mc + p * R + r, lc + p * R + r}; }, v, M, L);
                else
                    join(who.y, [&](int p) {
                        const float *b = part + Cut::slot(who.x + p, p == 0) * C::PART;
                        return From{b + r * HD + c, b + R * HD + r, b + R * HD + R + r};
                    }, v, M, L);
                const float inv = L != 0.f ? 1.f / L : 0.f;
                const float y[4] = {v.x * inv * DOWN, v.y * inv * DOWN, v.z * inv * DOWN, v.w * inv * DOWN};
                T *out = reinterpret_cast<T *>(a.out) + row * a.o_row + hq * a.o_head + c;
#pragma unroll
                for (int x = 0; x < 4; x++) {  // (a width is a multiple of 8)
                    out[x] = Elem<DT>::put(y[x]);
                    if (!finite_f(y[x])) s_bad[r] = 1;
                }
                if (c == 0 && a.lse) a.lse[(size_t)row * a.q_heads + hq] = ((M == -INFINITY ? 0.f : M) + log2f(L)) * 0.69314718055994530942f;
            }
            __syncthreads();
            for (int r = warp; r < rows; r += PA_THREADS / 32)
                if (s_bad[r]) pa_repair<DT, HD>(a, sr, pl.seq, (r0 + r) / each, pl.head * each + (r0 + r) % each);
        }
        Cut::next(pl, a, each, sr.n, count);
    }
}

struct PaPlan {
    int hd, wr, blocks;
    size_t smem, part, sums;
};
template <int DT, int HD, int WR>
static PaPlan pa_plan(int sms) {
    using C = PaShape<DT, HD, WR>;
    return PaPlan{HD, WR, std::min(KA_BLOCKS, sms * std::max(1, std::min(4, (int)(224 * 1024 / (C::SMEM + 2048))))), C::SMEM, C::PART, DT == DT_F32 ? 0 : C::SUMS};
}
template <int DT, int HD>
static PaPlan pa_plan(const PackedArgs &a, int sms) {
    // 16 rows where every sequence's fit: the steps' keys then take turns on the warps
    return (long long)a.max_rows * (a.q_heads / a.c.heads) <= 16 ? pa_plan<DT, HD, 1>(sms) : pa_plan<DT, HD, 4>(sms);
}
template <int DT>
static PaPlan pa_plan(const PackedArgs &a, int sms) {
    return a.width <= 32 ? pa_plan<DT, 32>(a, sms) : a.width <= 64 ? pa_plan<DT, 64>(a, sms) : a.width <= 128 ? pa_plan<DT, 128>(a, sms) : pa_plan<DT, 256>(a, sms);
}

template <int DT, int HD, int WR>
static cudaError_t pa_launch(const PackedArgs &a, const PaPlan &p, void *work, cudaStream_t s) {
    const size_t size = sizeof(typename Elem<DT>::T);
    // keys', values' and queries' rows in whole 16-byte pieces: bits 0 to 2
    auto whole = [&](const void *x, long long row, long long head) {
        return ((uintptr_t)x | (size_t)row * size | (size_t)head * size | (size_t)a.width * size) % 16 == 0;
    };
    const int wide = (whole(a.k, a.k_row, a.k_head) ? 1 : 0) | (whole(a.v, a.v_row, a.v_head) ? 2 : 0) | (whole(a.q, a.q_row, a.q_head) ? 4 : 0);
    const cudaError_t e = allow_dynamic_smem((const void *)k_packed_attend<DT, HD, WR>, p.smem);
    if (e != cudaSuccess) return e;
    int *arrived = reinterpret_cast<int *>(work);
    float *parts = reinterpret_cast<float *>(arrived + KA_BLOCKS);
    k_packed_attend<DT, HD, WR><<<p.blocks, PA_THREADS, p.smem, s>>>(a, wide, parts, parts + 2 * p.blocks * p.part, arrived);
    return cudaGetLastError();
}
template <int DT, int HD>
static cudaError_t pa_launch(const PackedArgs &a, const PaPlan &p, void *work, cudaStream_t s) {
    return p.wr == 1 ? pa_launch<DT, HD, 1>(a, p, work, s) : pa_launch<DT, HD, 4>(a, p, work, s);
}
template <int DT>
static cudaError_t pa_launch(const PackedArgs &a, const PaPlan &p, void *work, cudaStream_t s) {
    return p.hd == 32 ? pa_launch<DT, 32>(a, p, work, s) : p.hd == 64 ? pa_launch<DT, 64>(a, p, work, s)
           : p.hd == 128 ? pa_launch<DT, 128>(a, p, work, s) : pa_launch<DT, 256>(a, p, work, s);
}

static PaPlan plan_of(int dtype, const PackedArgs &a, int sms) {
    return dtype == DT_F32 ? pa_plan<DT_F32>(a, sms) : dtype == DT_F16 ? pa_plan<DT_F16>(a, sms) : pa_plan<DT_BF16>(a, sms);
}

// Many rows of a 16-bit type: the tensor-core kernel's, where TMA can fetch the keys and values.
static bool pa_many(int dtype, const PackedArgs &a) {
    return dtype != DT_F32 && a.width <= 128 && a.q_heads / a.c.heads <= 4096 && (long long)a.max_rows * (a.q_heads / a.c.heads) > 64;
}

// Many rows of f32: the tensor-core kernel's, whose split keys and values take as much memory again as they do, up to 1 GB.
static bool pa_many32(int dtype, const PackedArgs &a, int sms) {
    return dtype == DT_F32 && a.width <= 128 && (long long)a.max_rows * (a.q_heads / a.c.heads) > 64 && packed_attend_tc32_workspace(a, sms) <= 1u << 30;
}

size_t packed_attend_workspace(int dtype, const PackedArgs &a, int sms) {
    if (pa_many32(dtype, a, sms)) return packed_attend_tc32_workspace(a, sms);
    const PaPlan p = plan_of(dtype, a, sms);
    // (folded sums only where a sequence may be long enough)
    const size_t own = sizeof(int) * KA_BLOCKS + sizeof(float) * p.blocks * (2 * p.part + (a.max_len > PA_FOLD * 64 ? p.sums : 0));
    return pa_many(dtype, a) ? std::max(own, packed_attend_tc_workspace(a, sms)) : own;
}

cudaError_t launch_packed_attend(int dtype, const PackedArgs &a, int sms, void *encode, void *work, cudaStream_t s, uint64_t *launches) {
    if (pa_many32(dtype, a, sms)) return launch_packed_attend_tc32(a, sms, work, s, launches);
    (*launches)++;
    if (pa_many(dtype, a)) {
        const cudaError_t e = launch_packed_attend_tc(dtype, a, sms, encode, work, s);
        if (e != cudaErrorNotSupported) return e;
    }
    const PaPlan p = plan_of(dtype, a, sms);
    return dtype == DT_F32 ? pa_launch<DT_F32>(a, p, work, s) : dtype == DT_F16 ? pa_launch<DT_F16>(a, p, work, s) : pa_launch<DT_BF16>(a, p, work, s);
}

}  // namespace tcu

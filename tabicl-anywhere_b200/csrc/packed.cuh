// Attention of packed rows over keys and values as they are (packed_attend.cu, packed_attend_tc.cu): what the host hands the
// kernels, and what they share.
#pragma once
#include "fourbit.cuh"
#ifdef __CUDACC__
#include "kv4_plan.cuh"
#endif

namespace tcu {

// Sequence s: query rows q_starts[s] .. q_starts[s + 1], keys and values k_starts[s] .. k_starts[s + 1].
struct PackedArgs {
    struct {
        int heads = 0;
    } c;  // heads of the keys and values (named as the cache's are, for the cutting of the work)
    int seqs = 0, rows = 0, k_rows = 0, max_rows = 0, max_len = 0;
    const int *q_starts = nullptr, *k_starts = nullptr;
    int q_heads = 0, width = 0;
    const void *q = nullptr, *k = nullptr, *v = nullptr;
    void *out = nullptr;
    long long q_row = 0, q_head = 0, k_row = 0, k_head = 0, v_row = 0, v_head = 0, o_row = 0, o_head = 0;
    float scale = 0.f;
    int causal = 0, window = 0;
    float *lse = nullptr;     // [rows][q_heads], or null
    int *err = nullptr;       // report slot: set to 1 on starts outside their range
    int *err_wait = nullptr;  // report slot: set to 1 when a kernel gave up waiting
    int give_up = 0;          // test hook: every other block of a kernel with bounded waits begins as if one had given up
};

// Working memory of a call (the KA_BLOCKS counters, and parts after them), whichever kernel takes it, and the call. `encode` is
// the driver's cuTensorMapEncodeTiled.
size_t packed_attend_workspace(int dtype, const PackedArgs &a, int sms);
cudaError_t launch_packed_attend(int dtype, const PackedArgs &a, int sms, void *encode, void *work, cudaStream_t s, uint64_t *launches);
// The same on the tensor cores, for many rows of a 16-bit type. Not taken: cudaErrorNotSupported, nothing launched.
size_t packed_attend_tc_workspace(const PackedArgs &a, int sms);
cudaError_t launch_packed_attend_tc(int dtype, const PackedArgs &a, int sms, void *encode, void *work, cudaStream_t s);
// For many rows of f32.
size_t packed_attend_tc32_workspace(const PackedArgs &a, int sms);
cudaError_t launch_packed_attend_tc32(const PackedArgs &a, int sms, void *work, cudaStream_t s, uint64_t *launches);

#ifdef __CUDACC__

__device__ __forceinline__ KaRows ka_rows(const PackedArgs &a, int seq) {
    KaRows r;
    r.first = a.q_starts[seq], r.n = a.q_starts[seq + 1] - r.first;
    const int k0 = a.k_starts[seq];
    r.len = a.k_starts[seq + 1] - k0;
    r.ok = !(r.first < 0 || r.n < 0 || r.n > a.max_rows || r.first > a.rows - r.n || k0 < 0 || r.len < 0 || r.len > a.max_len || k0 > a.k_rows - r.len);
    return r;
}

// x + y, and what its rounding left into rest (0 beside infinities).
__device__ __forceinline__ float pa_add(float x, float y, float &rest) {
    const float t = x + y, z = t - x, e = (x - (t - z)) + (y - z);
    rest += e == e ? e : 0.f;
    return t;
}
// One row's output and log-sum-exp by one warp, from the keys that it sees and no others, U of them at a time. The products of a
// tile's weights and values take every value of the tile times a weight, 0 for a row that does not see it, and 0 times an infinity
// or a NaN is NaN; so a row whose output holds a NaN is worked out again here, and is NaN still only if what it sees makes it so
// (and a row whose weighted sum passed f32 before it was divided).
// Products q k near the largest have an exact difference, however large they are; scale and exponential take that. Sums keep what
// their roundings leave, and weights are scaled down where the values' sums come near f32's end. (A key in 0.1 us; one at a time,
// with the whole chain of a load, five exchanges and two exponentials for each, 0.65.)
template <int DT, int HD>
__device__ __noinline__ void pa_repair(const PackedArgs &a, const KaRows s, int seq, int i, int hq) {
    using T = typename Elem<DT>::T;
    constexpr int C = HD / 32, U = C > 4 ? 4 : 8;
    const int lane = threadIdx.x & 31, each = a.q_heads / a.c.heads, head = hq / each, lo = ka_lo(a, s, i), hi = ka_hi(a, s, i);
    const long long k0 = a.k_starts[seq];
    const T *q = reinterpret_cast<const T *>(a.q) + (s.first + i) * a.q_row + hq * a.q_head + lane;
    const T *k = reinterpret_cast<const T *>(a.k) + k0 * a.k_row + head * a.k_head + lane;
    const T *v = reinterpret_cast<const T *>(a.v) + k0 * a.v_row + head * a.v_head + lane;
    float x[C], o[C], o_rest[C];
#pragma unroll
    for (int c = 0; c < C; c++) x[c] = lane + 32 * c < a.width ? Elem<DT>::get(q[32 * c]) : 0.f, o[c] = o_rest[c] = 0.f;
    const float scale = fabsf(a.scale);
    float part = 0.0625f;                        // what weights are multiplied by for this lane's outputs: U values have a sum
    float m = -INFINITY, l = 0.f, l_rest = 0.f;  // the largest product (of the scale's sign), the sum of weights
    bool dead = false;                           // every output is NaN, whatever follows
#pragma unroll 1
    for (int j = lo; j < hi; j += U) {
        float d[U], top = m;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const T *from = k + min(j + u, hi - 1) * a.k_row;
            d[u] = 0.f;
#pragma unroll
            for (int c = 0; c < C; c++)
                if (lane + 32 * c < a.width) d[u] = fmaf(x[c], Elem<DT>::get(from[32 * c]), d[u]);
        }
#pragma unroll
        for (int b = 16; b; b >>= 1)
#pragma unroll
            for (int u = 0; u < U; u++) d[u] += __shfl_xor_sync(0xffffffffu, d[u], b);
#pragma unroll
        for (int u = 0; u < U; u++) {
            d[u] = j + u >= hi ? -INFINITY : a.scale < 0.f ? -d[u] : d[u];
            top = fmaxf(top, d[u]);
        }
        const float ref = top == -INFINITY ? 0.f : top;
        if (top != m) {
            const float f = m == -INFINITY ? 0.f : expf((m - ref) * scale);
            l *= f, l_rest *= f;
#pragma unroll
            for (int c = 0; c < C; c++) o[c] *= f, o_rest[c] *= f;
            m = top;
        }
        float sum = 0.f;
#pragma unroll
        for (int u = 0; u < U; u++) {
            d[u] = j + u < hi ? expf((d[u] - ref) * scale) : 0.f;
            sum += d[u];
        }
        l = pa_add(l, sum, l_rest);
        if (l != l) break;  // every output is NaN (all lanes have the same scores)
        if (dead) continue;
        float y[C];
#pragma unroll
        for (int c = 0; c < C; c++) y[c] = 0.f;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const T *from = v + min(j + u, hi - 1) * a.v_row;
#pragma unroll
            for (int c = 0; c < C; c++)
                if (lane + 32 * c < a.width && j + u < hi) y[c] = fmaf(d[u] * part, Elem<DT>::get(from[32 * c]), y[c]);
        }
        dead = true;
        bool near_end = false;
#pragma unroll
        for (int c = 0; c < C; c++) {
            o[c] = pa_add(o[c], y[c], o_rest[c]);
            dead &= o[c] != o[c] || lane + 32 * c >= a.width;
            near_end |= fabsf(o[c]) > 0x1p100f && finite_f(o[c]);
        }
        if (near_end) {
            part *= 0x1p-28f;
#pragma unroll
            for (int c = 0; c < C; c++) o[c] *= 0x1p-28f, o_rest[c] *= 0x1p-28f;
        }
        dead = __all_sync(0xffffffffu, dead);
        if (dead && !a.lse) break;
    }
    l += l_rest;
    T *out = reinterpret_cast<T *>(a.out) + (s.first + i) * a.o_row + hq * a.o_head + lane;
#pragma unroll
    for (int c = 0; c < C; c++)
        if (lane + 32 * c < a.width) out[32 * c] = Elem<DT>::put(l != l ? l : l != 0.f ? (o[c] + o_rest[c]) / (l * part) : 0.f);
    if (a.lse && lane == 0) a.lse[(size_t)(s.first + i) * a.q_heads + hq] = (m == -INFINITY ? 0.f : m * scale) + logf(l);
}

// After a block's work, where some of its outputs are not finite: the units that it has written once more, the rows that may be
// wrong worked out again. A NaN may be wrong only where the unit's values hold an infinity (a weight that was rounded to
// nothing has a part in that) or a NaN that not all of its rows see, or (f32, whose operands are split) its keys or the row's
// queries an infinity; rows that see a NaN in keys or values that all see are left as they are. Infinities and NaN alike may
// be wrong where values are so large that their weighted sums (weights up to 1 / by) may pass f32. `all`: every row that is not
// finite. From p the block's pieces begin; joined: whether it has written the unit that it shares with the blocks before, after it. By W warps (which
// have all the registers that the kernel was compiled for), for which no bounded wait waits: a row may take as long as it has keys.
template <int DT, int HD, int R, int STEP, int EXTRA, int W, class Cut>
__device__ __noinline__ void pa_mend(const PackedArgs &a, typename Cut::Place p, const int *joined, bool all, float by, int *dirty) {
    using T = typename Elem<DT>::T;
    const int tid = threadIdx.x % (32 * W), warp = tid >> 5, lane = tid & 31, each = a.q_heads / a.c.heads;
    const size_t size = sizeof(T);
    const bool wide_k = !(((uintptr_t)a.k | (size_t)a.k_row * size | (size_t)a.k_head * size) & 15);
    const bool wide_v = !(((uintptr_t)a.v | (size_t)a.v_row * size | (size_t)a.v_head * size) & 15);
    auto infinite = [](float x) { return fabsf(x) == INFINITY; };
    auto meet = [] { asm volatile("bar.sync 1, %0;" ::"n"(32 * W) : "memory"); };
    while (p.pos < p.end) {
        const KaRows s = ka_rows(a, p.seq);
        const auto sp = Cut::span(a, s, each, p.rt);
        const int count = (int)min((long long)(sp.steps - p.skip), p.end - p.pos);
        if (count == sp.steps || joined[p.skip == 0]) {
            const int r0 = p.rt * R, rows = min(R, s.n * each - r0), end = (int)min((long long)s.len, sp.base + (long long)(sp.steps - EXTRA) * STEP);
            meet();
            if (tid == 0) *dirty = all ? 2 : 0;
            meet();
            if (!all) {
                const int pieces = a.width / 8;
                const long long k0 = a.k_starts[p.seq] + sp.base;
                // values that may be behind a wrong NaN, and such whose sums may pass f32 (f32's own kernel scales them)
                const float limit = DT == DT_BF16 ? FLT_MAX * by / max(1, end - sp.base) : INFINITY;
                bool found = false, large = false;
                for (long long x = tid; x < (long long)(end - sp.base) * pieces && !large; x += 32 * W) {
                    const int j = (int)(x / pieces), c = (int)(x - (long long)j * pieces) * 8;
                    float e[8];
                    load8<DT>(reinterpret_cast<const T *>(a.v) + (k0 + j) * a.v_row + p.head * a.v_head + c, wide_v, e);
                    const bool hidden = sp.base + j < sp.lo_max || sp.base + j >= sp.hi_min;
#pragma unroll
                    for (int y = 0; y < 8; y++) found |= infinite(e[y]) || (hidden && e[y] != e[y]), large |= fabsf(e[y]) > limit && !infinite(e[y]);
                    if constexpr (DT == DT_F32) {
                        load8<DT>(reinterpret_cast<const T *>(a.k) + (k0 + j) * a.k_row + p.head * a.k_head + c, wide_k, e);
#pragma unroll
                        for (int y = 0; y < 8; y++) found |= infinite(e[y]);
                    }
                }
                if (found || large) atomicMax(dirty, large ? 2 : 1);
                meet();
            }
            const int some = *reinterpret_cast<volatile int *>(dirty);
            for (int r = warp; r < rows; r += W) {
                const int i = (r0 + r) / each, hq = p.head * each + (r0 + r) % each;
                const T *out = reinterpret_cast<const T *>(a.out) + (s.first + i) * a.o_row + hq * a.o_head;
                const T *q = reinterpret_cast<const T *>(a.q) + (s.first + i) * a.q_row + hq * a.q_head;
                bool nan = false, end = false, inf = false;
                for (int c = lane; c < a.width; c += 32) {
                    const float y = Elem<DT>::get(out[c]);
                    nan |= y != y, end |= infinite(y);
                    if constexpr (DT == DT_F32) inf |= infinite(q[c]);
                }
                nan = __any_sync(0xffffffffu, nan), end = __any_sync(0xffffffffu, end), inf = __any_sync(0xffffffffu, inf);
                if ((nan && (some || inf)) || (end && some > 1)) pa_repair<DT, HD>(a, s, p.seq, i, hq);
            }
        }
        Cut::next(p, a, each, s.n, count);
    }
}

#endif

}  // namespace tcu

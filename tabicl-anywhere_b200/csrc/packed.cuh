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

// One row's output and log-sum-exp by one warp, from the keys that it sees and no others. The products of a tile's weights and
// values take every value of the tile times a weight, 0 for a row that does not see it, and 0 times an infinity or a NaN is
// NaN; so a row whose output holds a NaN is worked out again here, and is NaN still only if what it sees makes it so. Products q k
// near the largest have an exact difference, however large they are; scale and exponential take that.
template <int DT>
__device__ __noinline__ void pa_repair(const PackedArgs &a, const KaRows s, int seq, int i, int hq) {
    using T = typename Elem<DT>::T;
    const int lane = threadIdx.x & 31, each = a.q_heads / a.c.heads, head = hq / each, hi = ka_hi(a, s, i), k0 = a.k_starts[seq];
    const T *q = reinterpret_cast<const T *>(a.q) + (s.first + i) * a.q_row + hq * a.q_head;
    float x[8], o[8];
#pragma unroll
    for (int c = 0; c < 8; c++) x[c] = lane + 32 * c < a.width ? Elem<DT>::get(q[lane + 32 * c]) : 0.f, o[c] = 0.f;
    const float scale = fabsf(a.scale);
    float m = -INFINITY, l = 0.f;  // the largest product (of the scale's sign), the sum of weights
    for (int j = ka_lo(a, s, i); j < hi; j++) {
        const T *k = reinterpret_cast<const T *>(a.k) + (long long)(k0 + j) * a.k_row + head * a.k_head;
        const T *v = reinterpret_cast<const T *>(a.v) + (long long)(k0 + j) * a.v_row + head * a.v_head;
        float d = 0.f;
#pragma unroll
        for (int c = 0; c < 8; c++)
            if (lane + 32 * c < a.width) d = fmaf(x[c], Elem<DT>::get(k[lane + 32 * c]), d);
#pragma unroll
        for (int b = 16; b; b >>= 1) d += __shfl_xor_sync(0xffffffffu, d, b);
        d = a.scale < 0.f ? -d : d;
        const float top = fmaxf(m, d), ref = top == -INFINITY ? 0.f : top, f = m == -INFINITY ? 0.f : expf((m - ref) * scale), p = expf((d - ref) * scale);
        l = l * f + p, m = top;
        if (l != l) break;  // whatever follows, every output is NaN (all lanes have the same score)
#pragma unroll
        for (int c = 0; c < 8; c++)
            if (lane + 32 * c < a.width) o[c] = fmaf(p, Elem<DT>::get(v[lane + 32 * c]), f == 1.f ? o[c] : o[c] * f);
    }
    T *out = reinterpret_cast<T *>(a.out) + (s.first + i) * a.o_row + hq * a.o_head;
#pragma unroll
    for (int c = 0; c < 8; c++)
        if (lane + 32 * c < a.width) out[lane + 32 * c] = Elem<DT>::put(l != 0.f ? o[c] / l : 0.f);
    if (a.lse && lane == 0) a.lse[(size_t)(s.first + i) * a.q_heads + hq] = (m == -INFINITY ? 0.f : m * scale) + logf(l);
}

#endif

}  // namespace tcu

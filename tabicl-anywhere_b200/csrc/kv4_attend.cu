// Attention of ragged query rows over a four-bit paged cache.
#include "fourbit.cuh"

namespace tcu {

// One block per (query row, query head), one warp's lanes over a key's words: width / 8 lanes a key, several keys a
// warp and step, each with its own running maximum and sum; joined at the end.
template <int DT>
__global__ void __launch_bounds__(128) k_kv4_attend(Kv4AttendArgs a) {
    using T = typename Elem<DT>::T;
    const int W = a.c.width, NU = W / 32, per = W / 8, NG = W / a.c.group, P = a.c.page;
    const int seq = blockIdx.z, i = blockIdx.y, hq = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int first = seq * a.max_rows, n = a.max_rows;
    if (a.starts) first = a.starts[seq], n = a.starts[seq + 1] - first;
    int len = a.lens[seq];
    if (first < 0 || n < 0 || n > a.max_rows || first > a.rows - n || len < 0 || len > a.max_len) {
        if (threadIdx.x == 0) *reinterpret_cast<volatile int *>(a.err) = 1;
        return;
    }
    if (i >= n) return;
    const int head = hq / (a.q_heads / a.c.heads), row = first + i, pos = len - n + i;
    const int end = a.causal ? min(len, pos + 1) : len, begin = a.window ? max(0, pos - a.window + 1) : 0;
    const int part = lane % per, u = part / 4, t = part % 4, keys = 32 / per, mine = lane / per;
    const size_t hb = kv4_head_bytes(W, P, a.c.group);
    const Kv4Offsets o = kv4_offsets(W, P, a.c.group);
    const T *qp = reinterpret_cast<const T *>(a.q) + row * a.q_row + hq * a.q_head + part * 8;
    float q[8], acc[8] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
    for (int j = 0; j < 8; j++) q[j] = Elem<DT>::get(qp[j]) * a.scale;
    for (int j0 = begin + warp * keys; j0 < end; j0 += 4 * keys) {
        const int j = j0 + mine;
        const int page = j < end ? a.table[seq * a.table_stride + j / P] : 0;
        const bool ok = j < end && page >= 0 && page < a.c.pages;
        if (j < end && !ok) *reinterpret_cast<volatile int *>(a.err) = 1;
        float s = 0.f;
        const uint8_t *base = a.c.pool + ((size_t)(ok ? page : 0) * a.c.heads + head) * hb;
        const int at = j % P;
        if (ok) {
            const uint32_t c = *(reinterpret_cast<const uint32_t *>(base + (size_t)at * (W / 2)) + t * NU + u);
            const float2 sc = __half22float2(*(reinterpret_cast<const __half2 *>(base + o.ks) + at * NG + part * 8 / a.c.group));
#pragma unroll
            for (int e = 0; e < 8; e++) s += q[e] * value_of(c, e, sc.x, sc.y);
        }
        for (int d = 1; d < per; d *= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
        if (ok) {
            const float mn = fmaxf(m, s), f = expf(m - mn), p = expf(s - mn);
            const uint16_t *vc = reinterpret_cast<const uint16_t *>(base + o.vc + (size_t)at * (W / 2)) + 2 * t * NU + u;
            const uint32_t c = (uint32_t)vc[0] | (uint32_t)vc[NU] << 16;
            const float2 sc = __half22float2(*(reinterpret_cast<const __half2 *>(base + o.vs) + at * NG + part * 8 / a.c.group));
#pragma unroll
            for (int e = 0; e < 8; e++) acc[e] = acc[e] * f + p * value_of(c, e, sc.x, sc.y);
            l = l * f + p, m = mn;
        }
    }
    __shared__ float sm[4][8], sl[4][8], so[4][8][256];
    if (part == 0) sm[warp][mine] = m, sl[warp][mine] = l;
#pragma unroll
    for (int e = 0; e < 8; e++) so[warp][mine][part * 8 + e] = acc[e];
    __syncthreads();
    float M = -INFINITY, L = 0.f;
    for (int w = 0; w < 4; w++)
        for (int k = 0; k < keys; k++) M = fmaxf(M, sm[w][k]);
    const float M0 = M == -INFINITY ? 0.f : M;
    for (int w = 0; w < 4; w++)
        for (int k = 0; k < keys; k++) L += sl[w][k] * expf(sm[w][k] - M0);
    T *op = reinterpret_cast<T *>(a.out) + row * a.o_row + hq * a.o_head;
    for (int c = threadIdx.x; c < W; c += 128) {
        float x = 0.f;
        for (int w = 0; w < 4; w++)
            for (int k = 0; k < keys; k++) x += so[w][k][c] * expf(sm[w][k] - M0);
        op[c] = Elem<DT>::put(L != 0.f ? x / L : 0.f);  // L is 0 when no key is seen, NaN when a score is
    }
    if (a.lse && threadIdx.x == 0) a.lse[(size_t)row * a.q_heads + hq] = M0 + logf(L);
}

cudaError_t launch_kv4_attend(int dtype, const Kv4AttendArgs &a, cudaStream_t s, uint64_t *launches) {
    if (!a.seqs || !a.rows || !a.max_rows) return cudaSuccess;
    const dim3 grid(a.q_heads, a.max_rows, a.seqs);
    if (dtype == DT_F32)
        k_kv4_attend<DT_F32><<<grid, 128, 0, s>>>(a);
    else if (dtype == DT_F16)
        k_kv4_attend<DT_F16><<<grid, 128, 0, s>>>(a);
    else
        k_kv4_attend<DT_BF16><<<grid, 128, 0, s>>>(a);
    if (launches) ++*launches;
    return cudaGetLastError();
}

}  // namespace tcu

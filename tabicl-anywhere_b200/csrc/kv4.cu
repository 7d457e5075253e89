// The four-bit paged cache: quantise keys and values into their slots, and read them back.
//
// One pass over the rows: a thread's 8 coordinates are 16 or 32 bytes read and 4 written, a group's extremes meet in a few
// lanes. 100,000 rows of 4 heads of 128 in f32 are stored and read back in 0.193 ms (936 MB, 4.8 TB/s): the store, 0.119 ms,
// is bound by the quantiser's instructions, the load, 0.082 ms, by memory. Two accesses of 16 bytes instead of one of 32
// took both to 0.234 ms; conversions for rounding (a quarter of the rate of an addition) and a division test a value the
// store alone to 0.143 ms.
#include <algorithm>

#include "fourbit.cuh"

namespace tcu {

// A thread takes 8 neighbouring coordinates (one word of a key, two half-words of a value) of one head of one token, of
// the keys and of the values; width / 8 neighbouring lanes hold a token's head, group / 8 of them a group.
template <int DT, bool STORE>
__global__ void __launch_bounds__(256) k_kv4_copy(Kv4CopyArgs a, uint32_t items, int per_log2, int page_log2, int group_log2, int wide) {
    using T = typename Elem<DT>::T;
    const int W = a.c.width, NU = W / 32, G8 = a.c.group / 8, NG = W / a.c.group, P = a.c.page;
    const uint32_t i = blockIdx.x * 256u + threadIdx.x;
    const bool on = i < items;
    const uint32_t row = on ? i >> per_log2 : 0;
    const int part = (int)(i & ((1u << per_log2) - 1)), u = part / 4, t = part % 4;
    const uint32_t token = row / (uint32_t)a.c.heads, head = row - token * a.c.heads;
    const long long slot = on ? __ldg(a.slots + token) : -1, page = slot >> page_log2;
    const int at = (int)slot & (P - 1);
    const bool there = slot >= 0 && page < a.c.pages;
    if (slot >= 0 && !there) *reinterpret_cast<volatile int *>(a.err) = 1;
    const Kv4Offsets o = kv4_offsets(W, P, a.c.group);
    uint8_t *base = a.c.pool + (there ? ((size_t)page * a.c.heads + head) * kv4_head_bytes(W, P, a.c.group) : 0);
    T *kp = reinterpret_cast<T *>(a.k) + token * a.k_row + head * a.k_head + part * 8;
    T *vp = reinterpret_cast<T *>(a.v) + token * a.v_row + head * a.v_head + part * 8;
    uint32_t *kc = reinterpret_cast<uint32_t *>(base + at * (W / 2)) + t * NU + u;
    uint16_t *vc = reinterpret_cast<uint16_t *>(base + o.vc + at * (W / 2)) + 2 * t * NU + u;
    __half2 *ks = reinterpret_cast<__half2 *>(base + o.ks) + at * NG + (part >> group_log2);
    __half2 *vs = reinterpret_cast<__half2 *>(base + o.vs) + at * NG + (part >> group_log2);
    if (STORE) {
        float x[2][8] = {};
        if (there) load8<DT>(kp, wide, x[0]), load8<DT>(vp, wide, x[1]);
#pragma unroll
        for (int w = 0; w < 2; w++) {
            float mn = x[w][0], mx = x[w][0];
            float bad = x[w][0] * 0.f;  // NaN where one is a NaN or an infinity
#pragma unroll
            for (int j = 1; j < 8; j++) mn = fminf(mn, x[w][j]), mx = fmaxf(mx, x[w][j]), bad = fmaf(x[w][j], 0.f, bad);
            for (int d = 1; d < G8; d *= 2) {
                mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, d));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
            }
            __half step, low;
            const uint32_t of_group = ((1u << G8) - 1) << (threadIdx.x & 31 & ~(G8 - 1));
            group_scale(mn, mx, __ballot_sync(0xffffffffu, bad != 0.f) & of_group, step, low);
            const uint32_t c = pack8(x[w], __half2float(step), __half2float(low));
            if (there) {
                if (w == 0) {
                    *kc = c;
                    if (!(part & (G8 - 1))) *ks = __halves2half2(step, low);
                } else {
                    vc[0] = (uint16_t)c, vc[NU] = (uint16_t)(c >> 16);
                    if (!(part & (G8 - 1))) *vs = __halves2half2(step, low);
                }
            }
        }
    } else if (on) {
        float x[2][8] = {};
        if (there) {
            const uint32_t c0 = *kc, c1 = (uint32_t)vc[0] | (uint32_t)vc[NU] << 16;
            const float2 s0 = __half22float2(*ks), s1 = __half22float2(*vs);
#pragma unroll
            for (int j = 0; j < 8; j++) x[0][j] = value_of(c0, j, s0.x, s0.y), x[1][j] = value_of(c1, j, s1.x, s1.y);
        }
        store8<DT>(kp, wide, x[0]), store8<DT>(vp, wide, x[1]);
    }
}

static int log2_of(int x) { return x <= 1 ? 0 : 1 + log2_of(x / 2); }

template <bool STORE>
static cudaError_t launch_copy(int dtype, Kv4CopyArgs a, cudaStream_t s, uint64_t *launches) {
    const int es = dtype == DT_F32 ? 4 : 2, per = a.c.width / 8;
    const uint64_t places = (uintptr_t)a.k | (uintptr_t)a.v | (uint64_t)((a.k_row | a.k_head | a.v_row | a.v_head) * es);
    const int wide = dtype == DT_F32 && places % 32 == 0 ? 2 : places % 16 == 0 ? 1 : 0;
    // indexes are 32 bits wide: very long calls in parts
    const int most = (int)std::min<long long>(0x7fffffff, 0x7fffff00LL / ((long long)a.c.heads * per));
    for (int left = a.tokens; left > 0;) {
        const int n = std::min(left, most);
        const uint32_t items = (uint32_t)n * a.c.heads * per, grid = (items + 255) / 256;
        const int pl = log2_of(per), gl = log2_of(a.c.page), ul = log2_of(a.c.group / 8);
        if (dtype == DT_F32)
            k_kv4_copy<DT_F32, STORE><<<grid, 256, 0, s>>>(a, items, pl, gl, ul, wide);
        else if (dtype == DT_F16)
            k_kv4_copy<DT_F16, STORE><<<grid, 256, 0, s>>>(a, items, pl, gl, ul, wide);
        else
            k_kv4_copy<DT_BF16, STORE><<<grid, 256, 0, s>>>(a, items, pl, gl, ul, wide);
        if (launches) ++*launches;
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
        left -= n, a.tokens = left, a.slots += n;
        a.k = (uint8_t *)a.k + (long long)n * a.k_row * es, a.v = (uint8_t *)a.v + (long long)n * a.v_row * es;
    }
    return cudaSuccess;
}
cudaError_t launch_kv4_store(int dtype, const Kv4CopyArgs &a, cudaStream_t s, uint64_t *launches) {
    return launch_copy<true>(dtype, a, s, launches);
}
cudaError_t launch_kv4_load(int dtype, const Kv4CopyArgs &a, cudaStream_t s, uint64_t *launches) {
    return launch_copy<false>(dtype, a, s, launches);
}

}  // namespace tcu

// Linear layers with four-bit weights and group scales.
#include "device.cuh"
#include "fourbit.cuh"

namespace tcu {

// A thread quantises 8 neighbouring columns of one row; 16 threads a block of 128 columns. Columns past k take no part
// in their group's extremes and get code 0 (the input they meet is 0); a group wholly past k is (0, 0).
template <int DT>
__global__ void __launch_bounds__(256) k_w4_pack(const typename Elem<DT>::T *w, long long ldw, int n, int k, int group,
                                                 uint8_t *codes, __half2 *scales) {
    const int blocks = (k + 127) / 128, per = blocks * 16, G8 = group / 8;
    const long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    const bool on = i < (long long)n * per;
    const int row = on ? (int)(i / per) : 0, part = (int)(i % per), c0 = part * 8;
    float x[8], mn = INFINITY, mx = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const bool in = on && c0 + j < k;
        x[j] = in ? Elem<DT>::get(w[row * ldw + c0 + j]) : 0.f;
        if (in) mn = fminf(mn, x[j]), mx = fmaxf(mx, x[j]), bad |= !finite_f(x[j]);
    }
    for (int d = 1; d < G8; d *= 2) {
        mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, d));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, d));
        bad |= (bool)__shfl_xor_sync(0xffffffffu, (int)bad, d);
    }
    if (!on) return;
    __half step, low;
    group_scale(mn, mx, bad, step, low);
    if (c0 / group * group >= k) step = low = __ushort_as_half(0);
    uint32_t c = pack8(x, __half2float(step), __half2float(low));
    if (c0 + 8 > k) c &= c0 >= k ? 0u : (1u << (4 * (k - c0))) - 1u;
    const int b = part / 16, u = part % 16 / 4, t = part % 4;
    reinterpret_cast<uint32_t *>(codes)[((size_t)row * blocks + b) * 16 + t * 4 + u] = c;
    if (part % G8 == 0) scales[(size_t)row * (blocks * 128 / group) + part / G8] = __halves2half2(step, low);
}

cudaError_t launch_w4_pack(int dtype, const void *w, long long ldw, int n, int k, int group, uint8_t *codes,
                           __half2 *scales, cudaStream_t s, uint64_t *launches) {
    const long long items = (long long)n * ((k + 127) / 128) * 16;
    const unsigned grid = (unsigned)((items + 255) / 256);
    if (dtype == DT_F32)
        k_w4_pack<DT_F32><<<grid, 256, 0, s>>>((const float *)w, ldw, n, k, group, codes, scales);
    else if (dtype == DT_F16)
        k_w4_pack<DT_F16><<<grid, 256, 0, s>>>((const __half *)w, ldw, n, k, group, codes, scales);
    else
        k_w4_pack<DT_BF16><<<grid, 256, 0, s>>>((const __nv_bfloat16 *)w, ldw, n, k, group, codes, scales);
    if (launches) ++*launches;
    return cudaGetLastError();
}

// One warp per (output, input row).
template <int DT>
__global__ void __launch_bounds__(256) k_w4_linear(W4Args a) {
    using T = typename Elem<DT>::T;
    const int lane = threadIdx.x & 31, row = blockIdx.y;
    const int n = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (n >= a.n) return;
    const int blocks = (a.k + 127) / 128, words = blocks * 16;
    const uint32_t *c = reinterpret_cast<const uint32_t *>(a.codes) + (size_t)n * words;
    const __half2 *sc = a.scales + (size_t)n * (blocks * 128 / a.group);
    const T *x = reinterpret_cast<const T *>(a.x) + row * a.ldx;
    float y = 0.f;
    for (int w = lane; w < words; w += 32) {
        const int b = w / 16, t = w % 16 / 4, u = w % 4, c0 = 128 * b + 32 * u + 8 * t;
        const float2 s = __half22float2(sc[c0 / a.group]);
        const uint32_t word = c[w];
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (c0 + j < a.k) y += Elem<DT>::get(x[c0 + j]) * value_of(word, j, s.x, s.y);
    }
    y = warp_sum(y);
    if (lane) return;
    if (a.bias) y += Elem<DT>::get(reinterpret_cast<const T *>(a.bias)[n]);
    if (a.act) y = gelu1(y);
    if (a.residual) y += Elem<DT>::get(reinterpret_cast<const T *>(a.residual)[row * a.ldr + n]);
    reinterpret_cast<T *>(a.y)[row * a.ldy + n] = Elem<DT>::put(y);
}

cudaError_t launch_w4_linear(int dtype, const W4Args &a, cudaStream_t s, uint64_t *launches) {
    if (!a.rows) return cudaSuccess;
    const dim3 grid((a.n + 7) / 8, a.rows);
    if (dtype == DT_F32)
        k_w4_linear<DT_F32><<<grid, 256, 0, s>>>(a);
    else if (dtype == DT_F16)
        k_w4_linear<DT_F16><<<grid, 256, 0, s>>>(a);
    else
        k_w4_linear<DT_BF16><<<grid, 256, 0, s>>>(a);
    if (launches) ++*launches;
    return cudaGetLastError();
}

}  // namespace tcu

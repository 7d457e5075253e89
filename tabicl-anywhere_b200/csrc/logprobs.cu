// Log probabilities of given labels, the entropy and the top alternatives of rows of scores.
#include "fourbit.cuh"

namespace tcu {

// A score as a whole number in the scores' order (-0 as +0), the index behind it so that of equal scores the lower
// index is the larger. 0 stands for no alternative: NaN and -infinity.
__device__ __forceinline__ unsigned long long rank_key(float x, int i) {
    if (!(x > -INFINITY)) return 0;
    const uint32_t b = __float_as_uint(x + 0.0f);
    const uint32_t o = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (unsigned long long)o << 32 | (uint32_t)(0x7fffffff - i);
}
__device__ __forceinline__ float key_score(unsigned long long k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

__device__ __forceinline__ unsigned long long block_max_key(unsigned long long v, unsigned long long *sh) {
    for (int o = 16; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    for (int w = 0; w < 8; w++) v = max(v, sh[w]);
    return v;
}
__device__ __forceinline__ float block_sum(float v, float *sh) {
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
    for (int w = 0; w < 8; w++) v += sh[w];
    return v;
}

// One block a row: the largest score, the sums, then one pass per alternative.
template <int DT>
__global__ void __launch_bounds__(256) k_logprobs(LogprobArgs a) {
    using T = typename Elem<DT>::T;
    __shared__ unsigned long long shk[8];
    __shared__ float shf[8];
    const int row = blockIdx.x;
    const T *x = reinterpret_cast<const T *>(a.logits) + row * a.stride;
    unsigned long long best = 0;
    for (int i = threadIdx.x; i < a.classes; i += 256) best = max(best, rank_key(Elem<DT>::get(x[i]), i));
    best = block_max_key(best, shk);
    const bool none = best == 0;
    const float top = none ? 0.f : key_score(best);
    float s = 0.f, e = 0.f;
    for (int i = threadIdx.x; i < a.classes; i += 256) {
        const float d = (Elem<DT>::get(x[i]) - top) * a.inv_t, p = expf(d);
        s += p;
        if (!(p <= 0.f)) e += p * d;
    }
    s = block_sum(s, shf), e = block_sum(e, shf);
    const float ls = none && s == 0.f ? 0.f : logf(s);
    for (int m = threadIdx.x; m < a.per_row; m += 256) {
        const int id = a.labels[(size_t)row * a.per_row + m];
        if (id >= a.classes) *reinterpret_cast<volatile int *>(a.err) = 1;
        a.out[(size_t)row * a.per_row + m] =
            id < 0 ? 0.f : id >= a.classes ? NAN : (Elem<DT>::get(x[id]) - top) * a.inv_t - ls;
    }
    if (a.entropy && threadIdx.x == 0) a.entropy[row] = none && s == 0.f ? 0.f : ls - e / s;
    unsigned long long last = ~0ull;
    for (int k = 0; k < a.top; k++) {
        unsigned long long b = 0;
        for (int i = threadIdx.x; i < a.classes; i += 256) {
            const unsigned long long r = rank_key(Elem<DT>::get(x[i]), i);
            if (r < last) b = max(b, r);
        }
        last = block_max_key(b, shk);
        if (threadIdx.x == 0) {
            a.top_values[(size_t)row * a.top + k] = last ? (key_score(last) - top) * a.inv_t - ls : -INFINITY;
            a.top_ids[(size_t)row * a.top + k] = last ? 0x7fffffff - (int)(uint32_t)last : -1;
        }
    }
}

cudaError_t launch_logprobs(int dtype, const LogprobArgs &a, cudaStream_t s, uint64_t *launches) {
    if (!a.rows) return cudaSuccess;
    if (dtype == DT_F32)
        k_logprobs<DT_F32><<<a.rows, 256, 0, s>>>(a);
    else if (dtype == DT_F16)
        k_logprobs<DT_F16><<<a.rows, 256, 0, s>>>(a);
    else
        k_logprobs<DT_BF16><<<a.rows, 256, 0, s>>>(a);
    if (launches) ++*launches;
    return cudaGetLastError();
}

}  // namespace tcu

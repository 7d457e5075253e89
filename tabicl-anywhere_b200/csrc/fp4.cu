// Matrices in microscaled four-bit floating point: quantised, and read back. Both move bytes: a value of 2 or 4 bytes there,
// half a byte and its share of a scale here.
#include "fp4.cuh"

namespace tcu {

constexpr int FP_THREADS = 256;

// 16 numbers of each value's nearest code (ties to the even code, which is the mantissa bit), eight to a word.
__device__ __forceinline__ uint2 fp4_codes(const float (&v)[16]) {
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; i++)
        asm("{\n\t.reg .b8 a, b, c, d;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
            "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
            "mov.b32 %0, {a, b, c, d};\n\t}\n"
            : "=r"(w[i])
            : "f"(v[8 * i]), "f"(v[8 * i + 1]), "f"(v[8 * i + 2]), "f"(v[8 * i + 3]), "f"(v[8 * i + 4]), "f"(v[8 * i + 5]), "f"(v[8 * i + 6]),
              "f"(v[8 * i + 7]));
    return make_uint2(w[0], w[1]);
}
// The e4m3 codes nearest to two values that are not negative, held to the largest.
__device__ __forceinline__ uint32_t e4m3_pair(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(r) : "f"(lo), "f"(hi));
    return r;
}
__device__ __forceinline__ float e4m3_value(uint32_t code) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)code));
    return __half2float(__ushort_as_half((unsigned short)(h & 0xffffu)));
}

// A block's scale in e4m3: the one nearest to top / (6 unit), ties to the even code. The quotient in f32 is within 2^-20 of
// it; where that spans a border the two are compared in 64 bits, which hold the border's multiple of 6 unit exactly.
__device__ __forceinline__ uint32_t nv_scale(float top, float inv_six, float unit) {
    const float q = top * inv_six;
    const uint32_t p = e4m3_pair(q * (1.f - 0x1p-20f), q * (1.f + 0x1p-20f)), lo = p & 0xffu, hi = p >> 8;
    if (lo == hi) return lo;
    const double border = 0.5 * ((double)e4m3_value(lo) + (double)e4m3_value(hi)) * 6.0 * (double)unit;
    return (double)top > border || ((double)top == border && (hi & 1) == 0) ? hi : lo;
}
// 16 codes by comparisons in 64 bits with the borders, whose multiples of `by` = scale * unit those hold exactly.
__device__ __noinline__ uint2 nv_codes_exact(const float *x, double by) {
    uint32_t w[2] = {0, 0};
    for (int i = 0; i < 16; i++) {
        const double a = fabs((double)x[i]);
        const double border[7] = {0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0};
        uint32_t c = 0;
        for (int b = 0; b < 7; b++) c += a > border[b] * by || (a == border[b] * by && (b & 1));
        w[i >> 3] |= (c | (__float_as_uint(x[i]) >> 31 << 3)) << (4 * (i & 7));
    }
    return make_uint2(w[0], w[1]);
}

// 16 neighbouring values of a row, zeros past its end.
template <int DT>
__device__ __forceinline__ void load16(const typename Elem<DT>::T *p, int there, int wide, float (&v)[16]) {
    if (there >= 16) {
        float a[8], b[8];
        load8<DT>(p, wide, a), load8<DT>(p + 8, wide, b);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = a[i], v[8 + i] = b[i];
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = i < there ? Elem<DT>::get(p[i]) : 0.f;
    }
}

// A thread quantises 16 neighbours: a block of FP4_NV, half a block of FP4_MX. 4 or 8 threads make a word of scales.
template <int DT, bool NV>
__global__ void __launch_bounds__(FP_THREADS) k_fp4_pack(Fp4Args a, unsigned per, unsigned total, int quads, int wide, float inv_six) {
    using T = typename Elem<DT>::T;
    const unsigned id = blockIdx.x * FP_THREADS + threadIdx.x;
    const bool on = id < total;
    const unsigned row = on ? id / per : 0, part = on ? id % per : 0;
    float v[16];
    load16<DT>(reinterpret_cast<const T *>(a.x) + (size_t)row * a.ldx + part * 16, on ? a.k - (int)part * 16 : 0, wide, v);
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) top = fmaxf(top, fabsf(v[i]));
    bool bad = false;  // (the largest of numbers and NaN is a number)
#pragma unroll
    for (int i = 0; i < 16; i++) bad |= !finite_f(v[i]);
    uint32_t scale;
    uint2 codes;
    if constexpr (NV) {
        if (bad) top = 0.f;
        scale = nv_scale(top, inv_six, a.unit);
        const float s = e4m3_value(scale);
        codes = make_uint2(0, 0);
        if (s > 0.f) {
            const float inv = __fdiv_rn(1.f, s * a.unit);  // within 2^-22 of the reciprocal, so v is of the quotient
            float lo[16], hi[16];
#pragma unroll
            for (int i = 0; i < 16; i++) lo[i] = v[i] * inv * (1.f - 0x1p-20f), hi[i] = v[i] * inv * (1.f + 0x1p-20f);
            codes = fp4_codes(lo);
            const uint2 other = fp4_codes(hi);
            if (codes.x != other.x || codes.y != other.y) codes = nv_codes_exact(v, (double)s * (double)a.unit);
        }
        if (bad) scale = 0x7f, codes = make_uint2(0, 0);
    } else {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        bad = __shfl_xor_sync(0xffffffffu, (int)bad, 1) || bad;
        // the power of two at or below the largest, over 4: the largest becomes 4 to 8 (what is above 6 is held there)
        const int e = max(0, (int)(__float_as_uint(top) >> 23) - 2);  // plus 127; (a subnormal's is below 2^-127)
        scale = bad ? 255u : (uint32_t)e;
        const float inv = __uint_as_float((uint32_t)(254 - e) << 23);  // 2^(127 - e): the product is exact but where far below 0.25
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = bad ? 0.f : v[i] * inv;
        codes = fp4_codes(v);
    }
    // the scales of four blocks, one word
    const int lane = threadIdx.x & 31;
    uint32_t word;
    if constexpr (NV) {
        word = scale | __shfl_down_sync(0xffffffffu, scale, 1) << 8;
        word |= __shfl_down_sync(0xffffffffu, word, 2) << 16;
    } else {
        word = scale | __shfl_down_sync(0xffffffffu, scale, 2) << 8;
        word |= __shfl_down_sync(0xffffffffu, word, 4) << 16;
    }
    if (!on) return;
    reinterpret_cast<uint2 *>(a.codes)[id] = codes;
    constexpr unsigned W = NV ? 4 : 8;
    if (lane % W == 0)
        *reinterpret_cast<uint32_t *>(a.scales + ((size_t)(row / 128) * quads + part / W) * 512 + row % 32 * 16 + row % 128 / 32 * 4) = word;
}

template <int DT, bool NV>
__global__ void __launch_bounds__(FP_THREADS) k_fp4_load(Fp4Args a, unsigned per, unsigned total, int quads, int wide) {
    using T = typename Elem<DT>::T;
    const unsigned id = blockIdx.x * FP_THREADS + threadIdx.x;
    if (id >= total) return;
    const unsigned row = id / per, part = id % per, s = NV ? part : part / 2;
    const int there = a.k - (int)part * 16;
    if (there <= 0) return;
    const uint2 codes = __ldg(reinterpret_cast<const uint2 *>(a.codes) + id);
    const uint32_t byte = a.scales[((size_t)(row / 128) * quads + s / 4) * 512 + row % 32 * 16 + row % 128 / 32 * 4 + s % 4];
    float scale;
    if constexpr (NV)
        scale = e4m3_value(byte);
    else
        scale = byte == 255u ? __uint_as_float(0x7fc00000u) : byte ? __uint_as_float(byte << 23) : 0x1p-127f;
    float v[16];
#pragma unroll
    for (int i = 0; i < 8; i++) {
        uint32_t h;
        asm("{\n\t.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, a;\n\t}\n" : "=r"(h) : "r"((i < 4 ? codes.x : codes.y) >> (8 * (i & 3))));
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h));
        v[2 * i] = f.x * scale * a.unit, v[2 * i + 1] = f.y * scale * a.unit;  // the first product is exact
    }
    T *to = reinterpret_cast<T *>(a.x) + (size_t)row * a.ldx + part * 16;
    if (there >= 16) {
        float p[8], q[8];
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = v[i], q[i] = v[8 + i];
        store8<DT>(to, wide, p), store8<DT>(to + 8, wide, q);
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++)
            if (i < there) to[i] = Elem<DT>::put(v[i]);
    }
}

// Runs of 16 elements as whole vectors: 1, or 2 for f32 runs that 32-byte accesses take.
static int fp4_wide(int dtype, const Fp4Args &a) {
    const size_t size = dtype == DT_F32 ? 4 : 2, at = (uintptr_t)a.x | (size_t)a.ldx * size;
    return at % 16 ? 0 : dtype == DT_F32 && at % 32 == 0 ? 2 : 1;
}

template <int DT>
static cudaError_t launch_copy(const Fp4Args &a, bool pack, cudaStream_t s) {
    const unsigned per = (unsigned)(fp4_padded(a.k) / 16), total = per * (unsigned)a.rows, blocks = (total + FP_THREADS - 1) / FP_THREADS;
    const int quads = fp4_quads(a.k, a.format), wide = fp4_wide(DT, a);
    const float inv_six = (float)(1.0 / (6.0 * (double)a.unit));
    if (pack && a.format == FP4_NV)
        k_fp4_pack<DT, true><<<blocks, FP_THREADS, 0, s>>>(a, per, total, quads, wide, inv_six);
    else if (pack)
        k_fp4_pack<DT, false><<<blocks, FP_THREADS, 0, s>>>(a, per, total, quads, wide, inv_six);
    else if (a.format == FP4_NV)
        k_fp4_load<DT, true><<<blocks, FP_THREADS, 0, s>>>(a, per, total, quads, wide);
    else
        k_fp4_load<DT, false><<<blocks, FP_THREADS, 0, s>>>(a, per, total, quads, wide);
    return cudaGetLastError();
}

static cudaError_t copy(int dtype, const Fp4Args &a, bool pack, cudaStream_t s, uint64_t *launches) {
    (*launches)++;
    return dtype == DT_F32 ? launch_copy<DT_F32>(a, pack, s) : dtype == DT_F16 ? launch_copy<DT_F16>(a, pack, s) : launch_copy<DT_BF16>(a, pack, s);
}
cudaError_t launch_fp4_pack(int dtype, const Fp4Args &a, cudaStream_t s, uint64_t *launches) { return copy(dtype, a, true, s, launches); }
cudaError_t launch_fp4_load(int dtype, const Fp4Args &a, cudaStream_t s, uint64_t *launches) { return copy(dtype, a, false, s, launches); }

}  // namespace tcu

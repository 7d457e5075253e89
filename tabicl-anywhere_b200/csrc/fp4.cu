// Matrices in microscaled four-bit floating point: quantised, and read back. Both move bytes: a value of 2 or 4 bytes there,
// half a byte and its share of a scale here.
//
// A block's scale and its numbers are those of exact arithmetic: a power of two divides exactly; for an e4m3 scale times the unit
// the quotient is taken in f32 from both sides of its error, and where the two sides give different codes the border between them,
// times scale and unit, is compared in 64 bits, which hold it (2 + 4 + 24 bits) exactly.
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

// A block's scale in e4m3: the one nearest to top / (6 unit), ties to the even code. The quotient in f32 is within 2^-23 of
// it; where 2^-22 either way spans a border the two are compared in 64 bits, which hold the border's multiple of 6 unit exactly.
__device__ __forceinline__ uint32_t nv_scale(float top, float inv_six, float unit) {
    const float q = top * inv_six;
    const uint32_t p = e4m3_pair(q * (1.f - 0x1p-22f), q * (1.f + 0x1p-22f)), lo = p & 0xffu, hi = p >> 8;
    if (lo == hi) return lo;
    const double border = 0.5 * ((double)e4m3_value(lo) + (double)e4m3_value(hi)) * 6.0 * (double)unit;
    return (double)top > border || ((double)top == border && (hi & 1) == 0) ? hi : lo;
}
// Of 16 codes those that differ between two tries, one apart: each magnitude compared in 64 bits with the border between them,
// whose multiple of `by` = scale * unit those hold exactly. (x: the values in memory; an array of a thread's would be stored for it.)
template <int DT>
__device__ __noinline__ uint2 nv_codes_exact(const typename Elem<DT>::T *x, uint2 lo, uint2 hi, double by) {
    uint32_t w[2] = {lo.x, lo.y};
    const uint32_t other[2] = {hi.x, hi.y};
    for (int k = 0; k < 2; k++)
        for (uint32_t diff = w[k] ^ other[k]; diff;) {
            const int at = (__ffs(diff) - 1) & ~3;
            diff &= ~(15u << at);
            const uint32_t c = w[k] >> at & 7u;  // (the lower of the two)
            auto number = [](uint32_t n) { return n < 4 ? 0.5 * n : n < 6 ? n - 2.0 : 2.0 * n - 8.0; };
            const double a = fabs((double)Elem<DT>::get(x[8 * k + at / 4])), border = 0.5 * (number(c) + number(c + 1)) * by;
            if (a > border || (a == border && (c & 1))) w[k] = (w[k] & ~(7u << at)) | (c + 1) << at;
        }
    return make_uint2(w[0], w[1]);
}

// x / y for x below 2^31, by a product.
struct FpDiv {
    unsigned mul, shift;
};
__device__ __forceinline__ unsigned fp_div(unsigned x, FpDiv d) { return __umulhi(x, d.mul) >> d.shift; }

// Two products at a time.
__device__ __forceinline__ void fp_mul2(float x, float y, float by, float &a, float &b) {
    asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %4};\n\tmul.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}\n" : "=f"(a), "=f"(b) : "f"(x), "f"(y), "f"(by));
}
__device__ __forceinline__ float fp_max_nan(float x, float y) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(x), "f"(y));
    return d;
}
template <int DT>
__device__ __forceinline__ uint32_t fp_max_nan2(uint32_t x, uint32_t y) {
    uint32_t d;
    if constexpr (DT == DT_F16)
        asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(y));
    else
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(x), "r"(y));
    return d;
}
template <int DT>
__device__ __forceinline__ float2 fp_widen(uint32_t w) {
    if constexpr (DT == DT_F16) return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// Where rows are not aligned a warp's accesses to memory are made side by side all the same, through shared memory: 32 runs of 16,
// 17 words apart. They are where its threads have neighbouring runs of one row: run lane begins at `first` + 16 lane of `there`.
constexpr int FP_PITCH = 17;
template <int DT>
__device__ __forceinline__ void stage_in(const typename Elem<DT>::T *first, int there, float *stage, float (&v)[16]) {
    const int lane = threadIdx.x & 31;
    float e[16];
#pragma unroll
    for (int i = 0; i < 16; i++) e[i] = 32 * i + lane < there ? Elem<DT>::get(first[32 * i + lane]) : 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) stage[(2 * i + lane / 16) * FP_PITCH + lane % 16] = e[i];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; i++) v[i] = stage[lane * FP_PITCH + i];
}
template <int DT>
__device__ __forceinline__ void stage_out(typename Elem<DT>::T *first, int there, float *stage, const float (&v)[16]) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < 16; i++) stage[lane * FP_PITCH + i] = v[i];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 16; i++)
        if (32 * i + lane < there) first[32 * i + lane] = Elem<DT>::put(stage[(2 * i + lane / 16) * FP_PITCH + lane % 16]);
}

// 16 neighbouring values of a row (zeros past its end) and their largest magnitude, NaN where one is. wide: accesses of 16 (1)
// or 32 bytes (2) are aligned; 0: neither, and `stage` is the warp's shared memory.
template <int DT>
__device__ __forceinline__ float load16(const typename Elem<DT>::T *p, int there, int wide, bool beside, float *stage, float (&v)[16]) {
    float top = 0.f;
    if (beside) {
        const int lane = threadIdx.x & 31;
        stage_in<DT>(p - 16 * lane, there + 16 * lane, stage, v);
#pragma unroll
        for (int i = 0; i < 16; i++) top = fp_max_nan(top, fabsf(v[i]));
        return top;
    }
    if constexpr (DT == DT_F32) {
        if (there >= 16) {
            float a[8], b[8];
            load8<DT>(p, wide, a), load8<DT>(p + 8, wide, b);
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = a[i], v[8 + i] = b[i];
        } else {
#pragma unroll
            for (int i = 0; i < 16; i++) v[i] = i < there ? p[i] : 0.f;
        }
#pragma unroll
        for (int i = 0; i < 16; i++) top = fp_max_nan(top, fabsf(v[i]));
    } else {
        uint32_t w[8];
        if (there >= 16 && wide == 2) {
            asm volatile("ld.global.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                         : "l"(p));
        } else if (there >= 16 && wide) {
            const uint4 a = __ldg(reinterpret_cast<const uint4 *>(p)), b = __ldg(reinterpret_cast<const uint4 *>(p) + 1);
            w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w, w[4] = b.x, w[5] = b.y, w[6] = b.z, w[7] = b.w;
        } else {
            const uint16_t *q = reinterpret_cast<const uint16_t *>(p);
#pragma unroll
            for (int i = 0; i < 8; i++) w[i] = (2 * i < there ? q[2 * i] : 0u) | (2 * i + 1 < there ? (uint32_t)q[2 * i + 1] << 16 : 0u);
        }
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            m = fp_max_nan2<DT>(m, w[i] & 0x7fff7fffu);
            const float2 f = fp_widen<DT>(w[i]);
            v[2 * i] = f.x, v[2 * i + 1] = f.y;
        }
        const float2 f = fp_widen<DT>(m);
        top = fp_max_nan(f.x, f.y);
    }
    return top;
}

// A thread quantises 16 neighbours: a block of FP4_NV, half a block of FP4_MX. 4 or 8 threads make a word of scales. Bound by its
// instructions (8192 x 8192 bf16 to FP4_NV: 38 us, issue active in 71%, 172 MB at 4.5 TB/s; read back 29 us). Trying every value
// against 64-bit borders where one of 16 was within 2^-20 of one took 69 us, with the values kept in local memory for it 52.
template <int DT, bool NV>
__global__ void __launch_bounds__(FP_THREADS, 8) k_fp4_pack(Fp4Args a, unsigned per, FpDiv div, unsigned total, int quads, int wide, float inv_six) {
    using T = typename Elem<DT>::T;
    const unsigned id = blockIdx.x * FP_THREADS + threadIdx.x;
    const bool on = id < total;
    const unsigned row = on ? fp_div(id, div) : 0, part = on ? id - row * per : 0;
    __shared__ float stage[FP_THREADS / 32][32 * FP_PITCH];
    const unsigned row0 = __shfl_sync(0xffffffffu, row, 0);  // (by every lane, those past the end too)
    const bool beside = __all_sync(0xffffffffu, !wide && on && row == row0);
    const T *from = reinterpret_cast<const T *>(a.x) + (size_t)row * a.ldx + part * 16;
    float v[16];
    float top = load16<DT>(from, on ? a.k - (int)part * 16 : 0, wide, beside, stage[threadIdx.x >> 5], v);
    uint32_t scale;
    uint2 codes = make_uint2(0, 0);
    if constexpr (NV) {
        if (finite_f(top)) {
            scale = nv_scale(top, inv_six, a.unit);
            const float s = e4m3_value(scale);
            if (s > 0.f) {
                // A value's product with the reciprocal is within 2^-22 of its quotient: where half as much again either way gives two
                // numbers, the border itself is asked.
                const float inv = __fdiv_rn(1.f, s * a.unit), down = inv * (1.f - 0x1.8p-22f), up = inv * (1.f + 0x1.8p-22f);
                float lo[16], hi[16];
#pragma unroll
                for (int i = 0; i < 16; i += 2) fp_mul2(v[i], v[i + 1], down, lo[i], lo[i + 1]), fp_mul2(v[i], v[i + 1], up, hi[i], hi[i + 1]);
                codes = fp4_codes(lo);
                const uint2 other = fp4_codes(hi);
                if (codes.x != other.x || codes.y != other.y) codes = nv_codes_exact<DT>(from, codes, other, (double)s * (double)a.unit);
            }
        } else {
            scale = 0x7f;
        }
    } else {
        top = fp_max_nan(top, __shfl_xor_sync(0xffffffffu, top, 1));
        if (finite_f(top)) {
            // the power of two at or below the largest, over 4: the largest becomes 4 to 8 (what is above 6 is held there)
            const int e = max(0, (int)(__float_as_uint(top) >> 23) - 2);  // plus 127; (a subnormal's is below 2^-127)
            scale = (uint32_t)e;
            const float inv = __uint_as_float((uint32_t)(254 - e) << 23);  // 2^(127 - e): the product is exact but where far below 0.25
#pragma unroll
            for (int i = 0; i < 16; i += 2) fp_mul2(v[i], v[i + 1], inv, v[i], v[i + 1]);
            codes = fp4_codes(v);
        } else {
            scale = 255u;
        }
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
__global__ void __launch_bounds__(FP_THREADS) k_fp4_load(Fp4Args a, unsigned per, FpDiv div, unsigned total, int quads, int wide) {
    using T = typename Elem<DT>::T;
    __shared__ float stage[FP_THREADS / 32][32 * FP_PITCH];
    const unsigned id = blockIdx.x * FP_THREADS + threadIdx.x;
    const bool on = id < total;
    const unsigned row = on ? fp_div(id, div) : 0, part = on ? id - row * per : 0, s = NV ? part : part / 2;
    const int there = a.k - (int)part * 16;
    const unsigned row0 = __shfl_sync(0xffffffffu, row, 0);  // (by every lane, those past the end too)
    const bool beside = __all_sync(0xffffffffu, !wide && on && row == row0);
    if (!beside && (!on || there <= 0)) return;
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
        fp_mul2(f.x, f.y, scale, v[2 * i], v[2 * i + 1]);  // exact
        if constexpr (NV) fp_mul2(v[2 * i], v[2 * i + 1], a.unit, v[2 * i], v[2 * i + 1]);
    }
    T *to = reinterpret_cast<T *>(a.x) + (size_t)row * a.ldx + part * 16;
    if (beside) {
        const int lane = threadIdx.x & 31;
        stage_out<DT>(to - 16 * lane, there + 16 * lane, stage[threadIdx.x >> 5], v);
    } else if (there >= 16) {
        if (DT != DT_F32 && wide == 2) {
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const T e[2] = {Elem<DT>::put(v[2 * i]), Elem<DT>::put(v[2 * i + 1])};
                w[i] = *reinterpret_cast<const uint16_t *>(&e[0]) | (uint32_t)*reinterpret_cast<const uint16_t *>(&e[1]) << 16;
            }
            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                         : "memory");
            return;
        }
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

// Runs of 16 elements as whole vectors: 1, or 2 for accesses of 32 bytes.
static int fp4_wide(int dtype, const Fp4Args &a) {
    const size_t size = dtype == DT_F32 ? 4 : 2, at = (uintptr_t)a.x | (size_t)a.ldx * size;
    return at % 16 ? 0 : at % 32 ? 1 : 2;
}

template <int DT>
static cudaError_t launch_copy(const Fp4Args &a, bool pack, cudaStream_t s) {
    const unsigned per = (unsigned)(fp4_padded(a.k) / 16), total = per * (unsigned)a.rows, blocks = (total + FP_THREADS - 1) / FP_THREADS;
    const int quads = fp4_quads(a.k, a.format), wide = fp4_wide(DT, a);
    const float inv_six = (float)(1.0 / (6.0 * (double)a.unit));
    unsigned bits = 0;
    while ((1u << bits) < per) bits++;
    const FpDiv div{(unsigned)((1ull << (31 + bits)) / per + 1), bits - 1};  // (per is 8 or more)
    if (pack && a.format == FP4_NV)
        k_fp4_pack<DT, true><<<blocks, FP_THREADS, 0, s>>>(a, per, div, total, quads, wide, inv_six);
    else if (pack)
        k_fp4_pack<DT, false><<<blocks, FP_THREADS, 0, s>>>(a, per, div, total, quads, wide, inv_six);
    else if (a.format == FP4_NV)
        k_fp4_load<DT, true><<<blocks, FP_THREADS, 0, s>>>(a, per, div, total, quads, wide);
    else
        k_fp4_load<DT, false><<<blocks, FP_THREADS, 0, s>>>(a, per, div, total, quads, wide);
    return cudaGetLastError();
}

static cudaError_t copy(int dtype, const Fp4Args &a, bool pack, cudaStream_t s, uint64_t *launches) {
    (*launches)++;
    return dtype == DT_F32 ? launch_copy<DT_F32>(a, pack, s) : dtype == DT_F16 ? launch_copy<DT_F16>(a, pack, s) : launch_copy<DT_BF16>(a, pack, s);
}
cudaError_t launch_fp4_pack(int dtype, const Fp4Args &a, cudaStream_t s, uint64_t *launches) { return copy(dtype, a, true, s, launches); }
cudaError_t launch_fp4_load(int dtype, const Fp4Args &a, cudaStream_t s, uint64_t *launches) { return copy(dtype, a, false, s, launches); }

}  // namespace tcu

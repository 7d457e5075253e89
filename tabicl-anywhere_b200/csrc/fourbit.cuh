// The four-bit operators (kv4.cu, w4.cu) and the label log-probabilities (logprobs.cu): what the host hands the
// kernels, the stored format, and the conversions every kernel shares.
//
// Format: `group` neighbouring coordinates share (step, low), two f16 numbers; a coordinate is low + step * code with a
// code of 0..15. Widths are made of 32-coordinate units (NU of them). A key's codes are words of 8: word t * NU + u
// (t < 4) holds coordinates 32 u + 8 t + j in nibble j, so that a thread of a matrix fragment (t = lane % 4) reads its
// part of every unit with one wide load. A value's codes are half-words of 4: half-word g * NU + u (g < 8) holds
// coordinates 32 u + 4 g + j in nibble j, the same for a thread's row (g = lane / 4) of a transposed fragment.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cfloat>
#include <cmath>
#include <cstddef>
#include <cstdint>

namespace tcu {

enum { DT_F32 = 0, DT_F16 = 1, DT_BF16 = 2 };

// Most blocks of an attention launch. As many arrival counters (ints, zero between calls) start the working memory of every
// operator, so that one block of it serves them all: attention counts there, the others leave them alone.
constexpr int KA_BLOCKS = 2048;

// A paged cache: pool [pages][heads]{key codes [page][width / 2], key (step, low) [page][width / group], value codes,
// value (step, low)}.
struct Kv4 {
    uint8_t *pool = nullptr;
    long long pages = 0;
    int heads = 0, width = 0, page = 0, group = 0;
};

__host__ __device__ inline size_t kv4_head_bytes(int width, int page, int group) {
    return (size_t)page * (width + 8 * (width / group));
}
// Byte offsets inside a head's part of a page.
struct Kv4Offsets {
    unsigned ks, vc, vs;  // key scales, value codes, value scales (key codes at 0)
};
__host__ __device__ inline Kv4Offsets kv4_offsets(int width, int page, int group) {
    const unsigned c = (unsigned)page * (width / 2), s = (unsigned)page * (width / group) * 4;
    return Kv4Offsets{c, c + s, 2 * c + s};
}

// Keys and values of `tokens` rows to (store) or from (load) their slots.
struct Kv4CopyArgs {
    Kv4 c;
    int tokens = 0;
    const long long *slots = nullptr;  // page * tokens per page + place in it; negative: no slot
    void *k = nullptr, *v = nullptr;   // [tokens][heads][width] by row and head strides (elements)
    long long k_row = 0, k_head = 0, v_row = 0, v_head = 0;
    int *err = nullptr;  // report slot (host memory, mapped): set to 1 on a slot outside the cache
};

// Ragged query rows against the cache.
struct Kv4AttendArgs {
    Kv4 c;
    int seqs = 0, rows = 0, max_rows = 0, max_len = 0;
    const int *starts = nullptr, *lens = nullptr, *table = nullptr;
    long long table_stride = 0;
    int q_heads = 0;
    const void *q = nullptr;
    void *out = nullptr;
    long long q_row = 0, q_head = 0, o_row = 0, o_head = 0;
    float scale = 0.f;
    int causal = 0, window = 0;
    float *lse = nullptr;  // [rows][q_heads], or null
    int *err = nullptr;    // report slot: set to 1 on a length, start or page outside its range
    int *err_wait = nullptr;  // report slot: set to 1 when a kernel gave up waiting
};

// y = act(x W^T + bias) + residual with four-bit weights.
struct W4Args {
    const uint8_t *codes = nullptr;  // [n][k / 128 rounded up][64]
    const __half2 *scales = nullptr; // [n][k / 128 rounded up * 128 / group] (step, low)
    int n = 0, k = 0, group = 0, rows = 0, act = 0;
    const void *x = nullptr, *bias = nullptr, *residual = nullptr;
    void *y = nullptr;
    long long ldx = 0, ldy = 0, ldr = 0;
};

struct LogprobArgs {
    const void *logits = nullptr;
    int rows = 0, classes = 0;
    long long stride = 0;
    const int *labels = nullptr;  // [rows][per_row]
    int per_row = 0, top = 0;
    float inv_t = 1.f;
    float *out = nullptr, *entropy = nullptr, *top_values = nullptr;
    int *top_ids = nullptr;
    int *err = nullptr;  // report slot: set to 1 on a label beyond the classes
};
constexpr int LOGPROB_MAX_TOP = 32;

cudaError_t launch_kv4_store(int dtype, const Kv4CopyArgs &a, cudaStream_t s, uint64_t *launches);
cudaError_t launch_kv4_load(int dtype, const Kv4CopyArgs &a, cudaStream_t s, uint64_t *launches);
// Working memory of an attention call (its first ints zero between calls), and the call.
size_t kv4_attend_workspace(int dtype, const Kv4AttendArgs &a, int sms);
cudaError_t launch_kv4_attend(int dtype, const Kv4AttendArgs &a, int sms, void *work, size_t work_bytes, cudaStream_t s,
                              uint64_t *launches);
// kernels.cu: opt a kernel in to `bytes` of dynamic shared memory on the current device.
cudaError_t allow_dynamic_smem(const void *kernel, size_t bytes);
// The same on the tensor cores, for many rows a cache head (widths up to 128): f32, and 16-bit types.
size_t kv4_attend_tc_workspace(const Kv4AttendArgs &a, int sms);
cudaError_t launch_kv4_attend_tc(const Kv4AttendArgs &a, int sms, void *work, cudaStream_t s);
size_t kv4_attend_tc16_workspace(const Kv4AttendArgs &a, int sms);
cudaError_t launch_kv4_attend_tc16(int dtype, const Kv4AttendArgs &a, int sms, void *work, cudaStream_t s);
// A weight matrix w [n][k] (row stride ldw) to codes and scales.
cudaError_t launch_w4_pack(int dtype, const void *w, long long ldw, int n, int k, int group, uint8_t *codes,
                           __half2 *scales, cudaStream_t s, uint64_t *launches);
// Working memory of a linear layer (what it uses comes after the KA_BLOCKS counters), and the call.
size_t w4_linear_workspace(int dtype, const W4Args &a, int sms);
cudaError_t launch_w4_linear(int dtype, const W4Args &a, int sms, void *work, size_t work_bytes, cudaStream_t s,
                             uint64_t *launches);
cudaError_t launch_logprobs(int dtype, const LogprobArgs &a, int sms, cudaStream_t s, uint64_t *launches);

#ifdef __CUDACC__

template <int DT>
struct Elem;
template <>
struct Elem<DT_F32> {
    using T = float;
    static __device__ __forceinline__ float get(float x) { return x; }
    static __device__ __forceinline__ float put(float x) { return x; }
};
template <>
struct Elem<DT_F16> {
    using T = __half;
    static __device__ __forceinline__ float get(__half x) { return __half2float(x); }
    static __device__ __forceinline__ __half put(float x) { return __float2half_rn(x); }
};
template <>
struct Elem<DT_BF16> {
    using T = __nv_bfloat16;
    static __device__ __forceinline__ float get(__nv_bfloat16 x) { return __bfloat162float(x); }
    static __device__ __forceinline__ __nv_bfloat16 put(float x) { return __float2bfloat16_rn(x); }
};

// Eight consecutive elements; `wide`: the address is known to be 16-byte aligned (1) or, f32, 32-byte aligned (2: one access of
// 32 bytes, so a warp's accesses are whole lines).
template <int DT>
__device__ __forceinline__ void load8(const typename Elem<DT>::T *p, int wide, float (&v)[8]) {
    using T = typename Elem<DT>::T;
    if (DT == DT_F32 && wide == 2) {
        asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                     : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                     : "l"(p));
    } else if (wide) {
        __align__(16) T e[8];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++)
            reinterpret_cast<uint4 *>(e)[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = Elem<DT>::get(e[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = Elem<DT>::get(p[i]);
    }
}
template <int DT>
__device__ __forceinline__ void store8(typename Elem<DT>::T *p, int wide, const float (&v)[8]) {
    using T = typename Elem<DT>::T;
    if (DT == DT_F32 && wide == 2) {
        asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]),
                     "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                     : "memory");
        return;
    }
    __align__(16) T e[8];
#pragma unroll
    for (int i = 0; i < 8; i++) e[i] = Elem<DT>::put(v[i]);
    if (wide) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; i++) reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<const uint4 *>(e)[i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) p[i] = e[i];
    }
}

// N runs of eight elements, `step` elements apart, of a type known at run time: where they are whole aligned vectors all are
// asked for before any is used (a branch between two loads makes the second wait for the first).
template <int N>
__device__ __forceinline__ void load_runs(int dtype, const void *base, long long at, int step, bool wide, float (&v)[N][8]) {
    if (wide && dtype == DT_F32) {
        const float4 *p = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(base) + at);
        float4 raw[N][2];
#pragma unroll
        for (int i = 0; i < N; i++) raw[i][0] = __ldg(p + i * (step / 4)), raw[i][1] = __ldg(p + i * (step / 4) + 1);
#pragma unroll
        for (int i = 0; i < N; i++) {
            v[i][0] = raw[i][0].x, v[i][1] = raw[i][0].y, v[i][2] = raw[i][0].z, v[i][3] = raw[i][0].w;
            v[i][4] = raw[i][1].x, v[i][5] = raw[i][1].y, v[i][6] = raw[i][1].z, v[i][7] = raw[i][1].w;
        }
    } else if (wide) {
        const uint4 *p = reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(base) + at);
        uint4 raw[N];
#pragma unroll
        for (int i = 0; i < N; i++) raw[i] = __ldg(p + i * (step / 8));
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float2 f = dtype == DT_BF16 ? make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u))
                                                  : __half22float2(*reinterpret_cast<const __half2 *>(&w[j]));
                v[i][2 * j] = f.x, v[i][2 * j + 1] = f.y;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) {
            if (dtype == DT_F32)
                load8<DT_F32>(reinterpret_cast<const float *>(base) + at + i * step, false, v[i]);
            else if (dtype == DT_F16)
                load8<DT_F16>(reinterpret_cast<const __half *>(base) + at + i * step, false, v[i]);
            else
                load8<DT_BF16>(reinterpret_cast<const __nv_bfloat16 *>(base) + at + i * step, false, v[i]);
        }
    }
}

// (step, low) of a group with extremes mn, mx (`bad`: it holds a NaN or an infinity, and then stands for NaN
// throughout). low is the smallest value and step a fifteenth of the span above it, each rounded to f16 (values beyond
// f16's range are held at its largest): f16 keeps a group's overhead at 4 bytes and 11 bits of a 4-bit step.
__device__ __forceinline__ void group_scale(float mn, float mx, bool bad, __half &step, __half &low) {
    low = __float2half_rn(fminf(fmaxf(mn, -65504.f), 65504.f));
    step = __float2half_rn(__fdiv_rn(fmaxf(__fsub_rn(fminf(mx, 65504.f), __half2float(low)), 0.f), 15.f));
    if (bad) step = __ushort_as_half(0), low = __ushort_as_half(0x7e00);
}
// Eight values' codes: a value's distance from low in steps, rounded to the nearest (ties to even), held to 0..15; 0 where the
// step is 0. The quotient is the correctly rounded one, so equal inputs give equal codes everywhere.
// It is found as a product with the step's reciprocal, within 2^-20 of it (so 1.5e-5 at most), and rounded by adding 1.5 * 2^23, whose sum's low
// bits are the code; only where one of the eight is near a tie are they divided (which costs as much as all the rest).
__device__ __forceinline__ uint32_t pack8(const float (&x)[8], float step, float low) {
    if (!(step > 0.f)) return 0;
    constexpr float MAGIC = 12582912.f;
    float inverse, near = 0.f;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(step));  // (an f16's range: no subnormal f32)
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        const float t = fminf(fmaxf(__fmul_rn(__fsub_rn(x[j], low), inverse), 0.f), 15.f), c = __fadd_rn(t, MAGIC);
        near = fmaxf(near, fabsf(__fsub_rn(t, __fsub_rn(c, MAGIC))));
        w += (__float_as_uint(c) - 0x4b400000u) << (4 * j);
    }
    if (near > 0.49997f) {
        w = 0;
#pragma unroll 1
        for (int j = 0; j < 8; j++) {
            float v = x[0];
#pragma unroll
            for (int k = 1; k < 8; k++) v = k == j ? x[k] : v;
            w |= (uint32_t)(int)fminf(fmaxf(rintf(__fdiv_rn(__fsub_rn(v, low), step)), 0.f), 15.f) << (4 * j);
        }
    }
    return w;
}
// low + step * code, the product and the sum each rounded to f32 (step * code is exact: 11 + 4 bits).
__device__ __forceinline__ float value_of(uint32_t w, int j, float step, float low) {
    return __fadd_rn(__fmul_rn((float)((w >> (4 * j)) & 15u), step), low);
}
// Two codes of a word as f16 operands of a product: the first (SECOND false) or second nibbles of its even bytes. As they
// are, subnormals: code * 2^-24, code * 2^-20, one AND. CENTRED: code - 8, 16 (code - 8), with the AND's result in the low
// bits of 1024 and one subtraction, exact. The products' f32 sums are not rounded to nearest by the matrix unit, and with
// codes of one sign they are large beside what is left when the groups' lows are added, so for f32 results, and f16 ones of
// attention, the codes are centred and the lows taken as low + 8 step (f16 linear layers are off by 1e-6, which 11 bits do
// not show).
template <bool CENTRED, bool SECOND>
__device__ __forceinline__ uint32_t code_pair(uint32_t w) {
    const uint32_t c = w & (SECOND ? 0x00f000f0u : 0x000f000fu);
    if constexpr (!CENTRED) return c;
    const uint32_t v = c | 0x64006400u, m = SECOND ? 0x64806480u : 0x64086408u;
    const __half2 h = __hsub2(*reinterpret_cast<const __half2 *>(&v), *reinterpret_cast<const __half2 *>(&m));
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ bool finite_f(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

#endif

}  // namespace tcu

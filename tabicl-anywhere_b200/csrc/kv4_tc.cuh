// What the two tensor-core kernels of the four-bit attention share: widening stored codes into operand blocks, waits.
#pragma once
#include "kv4_plan.cuh"
#include "tc.cuh"

namespace tcu {

using namespace tc;

constexpr long long KT_WAIT = 2000000000ll;  // about a second at boost clock
// Steps a block takes at least: shorter parts of a unit are more to join (128 bf16 rows of 8 heads over 8192 keys: 112 us with
// 8, 81 us with 16, 76 us with 32; over 1024 keys of 8 sequences 43, 36 and 61 us).
constexpr int KA_TC_STEPS = 16;

// One lane of a converged warp. The products are issued under it by a warp whose lanes all run the issuing loop: their
// operands are then uniform, and an issue takes a few cycles (under `lane == 0` of a diverged warp about 130 were measured).
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}\n" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ float kt_pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -127 < e < 128
__device__ __forceinline__ float kt_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Waits for the loads from tensor memory; v, one of them, cannot be used before (it goes through the wait).
__device__ __forceinline__ void tmem_wait_ld32(float (&v)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]), "+f"(v[8]), "+f"(v[9]),
                   "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]), "+f"(v[16]), "+f"(v[17]), "+f"(v[18]),
                   "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]),
                   "+f"(v[28]), "+f"(v[29])
                 :
                 : "memory");
    asm volatile("" : "+f"(v[30]), "+f"(v[31])::"memory");
}
// 16 columns of this thread's lane of tensor memory.
__device__ __forceinline__ void tmem_st16u(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(v[0]),
        "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
        "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void kt_bar(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
__device__ __forceinline__ __half2 kt_h2(uint32_t w) { return *reinterpret_cast<const __half2 *>(&w); }
__device__ __forceinline__ uint32_t kt_u32(__half2 h) { return *reinterpret_cast<const uint32_t *>(&h); }

// One group's scales for widening in f32: value = code nibble as f16 * even (a byte's first nibble) or * odd (its second) + low.
struct KtScale {
    float even, odd, low;
    __device__ __forceinline__ void set(float step, float l, float up) {
        even = step * up * 16777216.f, odd = even * 0.0625f, low = l * up;
    }
};
// A word's eight codes, CENTRED: less 8, as f16 pairs, exact: a code under the bits of 1024, or of 1024 sixteenths. (A nibble
// as a subnormal f16 would take no subtraction, but the step that it meets 24 powers of two more of f16's range.)
template <bool CENTRED>
__device__ __forceinline__ void kt_codes(uint32_t w, __half2 (&c)[4]) {
    const uint32_t v = w >> 8;
    // 1024 or 1032, 1 / 16, -64 or -72
    const __half2 up = kt_h2(CENTRED ? 0x64086408u : 0x64006400u), sixteenth = kt_h2(0x2c002c00u), off = kt_h2(CENTRED ? 0xd480d480u : 0xd400d400u);
    c[0] = __hsub2(kt_h2((w & 0x000f000fu) | 0x64006400u), up), c[1] = __hfma2(kt_h2((w & 0x00f000f0u) | 0x64006400u), sixteenth, off);
    c[2] = __hsub2(kt_h2((v & 0x000f000fu) | 0x64006400u), up), c[3] = __hfma2(kt_h2((v & 0x00f000f0u) | 0x64006400u), sixteenth, off);
}
// A word's eight values, each rounded once to f16.
__device__ __forceinline__ void kt_round(uint32_t w, __half2 step, __half2 low, __half *to) {
    __half2 c[4];
    kt_codes<false>(w, c);
    *reinterpret_cast<uint4 *>(to) = make_uint4(kt_u32(__hfma2(c[0], step, low)), kt_u32(__hfma2(c[1], step, low)), kt_u32(__hfma2(c[2], step, low)),
                                                kt_u32(__hfma2(c[3], step, low)));
}
// step * (code - 8) of a word's eight codes as the sum of two f16, each exact: the step's upper 7 bits and its lower 4.
__device__ __forceinline__ void kt_exact(uint32_t w, __half2 step, __half *hi, __half *lo) {
    const __half2 s1 = kt_h2(kt_u32(step) & 0xfff0fff0u), s2 = __hsub2(step, s1);
    __half2 c[4];
    kt_codes<true>(w, c);
    *reinterpret_cast<uint4 *>(hi) = make_uint4(kt_u32(__hmul2(c[0], s1)), kt_u32(__hmul2(c[1], s1)), kt_u32(__hmul2(c[2], s1)), kt_u32(__hmul2(c[3], s1)));
    *reinterpret_cast<uint4 *>(lo) = make_uint4(kt_u32(__hmul2(c[0], s2)), kt_u32(__hmul2(c[1], s2)), kt_u32(__hmul2(c[2], s2)), kt_u32(__hmul2(c[3], s2)));
}
// A word's eight values as f16, and what remains of them, into 16 bytes each.
__device__ __forceinline__ void kt_widen(uint32_t w, const KtScale &s, __half *hi, __half *lo) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t v = i & 2 ? w >> 8 : w;
        const float2 c = __half22float2(kt_h2(i & 1 ? v & 0x00f000f0u : v & 0x000f000fu));
        const float f = i & 1 ? s.odd : s.even;
        split_pair(fmaf(c.x, f, s.low), fmaf(c.y, f, s.low), h[i], l[i]);
    }
    *reinterpret_cast<uint4 *>(hi) = make_uint4(h[0], h[1], h[2], h[3]);
    *reinterpret_cast<uint4 *>(lo) = make_uint4(l[0], l[1], l[2], l[3]);
}

}  // namespace tcu

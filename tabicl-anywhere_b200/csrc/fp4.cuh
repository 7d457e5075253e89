// Matrices in microscaled four-bit floating point (fp4.cu, fp4_linear.cu): what the host hands the kernels, the stored format.
//
// A number (sign, two exponent bits, one of mantissa) is 0, 0.5, 1, 1.5, 2, 3, 4 or 6, codes 0..7, or its negative, 8..15; a
// value is unit * scale * number. FP4_MX: 32 neighbours of a row share a power of two, a byte of its exponent plus 127 (255:
// NaN). FP4_NV: 16 share an e4m3 float (127: NaN). Rows of codes are filled up to 128 columns, two to a byte, the earlier in
// the low half, which is how the matrix unit reads them. Scales lie in blocks of 128 rows x 4 scales, the unit's too: row r
// and scale s of a block at byte 16 (r % 32) + 4 (r / 32) + s; `quads` blocks beside one another, then the next 128 rows.
#pragma once
#include "fourbit.cuh"

namespace tcu {

enum { FP4_MX = 0, FP4_NV = 1 };

inline int fp4_padded(int k) { return (k + 127) / 128 * 128; }
inline int fp4_quads(int k, int format) { return fp4_padded(k) / (format == FP4_NV ? 64 : 128); }

// A matrix's values from (pack) or to (load) x.
struct Fp4Args {
    uint8_t *codes = nullptr, *scales = nullptr;
    int rows = 0, k = 0, format = 0;
    float unit = 1.f;
    void *x = nullptr;  // [rows][k] by a row stride (elements)
    long long ldx = 0;
};

// y = act(x W^T + bias) + residual, both matrices quantised.
struct Fp4LinearArgs {
    const uint8_t *w = nullptr, *w_scales = nullptr, *x = nullptr, *x_scales = nullptr;
    int n = 0, k = 0, rows = 0, format = 0, act = 0;
    float alpha = 1.f;  // the product of their units
    const void *bias = nullptr, *residual = nullptr;
    void *y = nullptr;
    long long ldy = 0, ldr = 0;
    int *err_wait = nullptr;  // report slot: set to 1 when a kernel gave up waiting
    int give_up = 0;          // test hook: every other block begins as if a wait had given up
};

cudaError_t launch_fp4_pack(int dtype, const Fp4Args &a, cudaStream_t s, uint64_t *launches);
cudaError_t launch_fp4_load(int dtype, const Fp4Args &a, cudaStream_t s, uint64_t *launches);
// Working memory of a product (what it uses comes with and after the KA_BLOCKS counters), and the call. `encode` is the
// driver's cuTensorMapEncodeTiled.
size_t fp4_linear_workspace(int dtype, const Fp4LinearArgs &a, int sms);
cudaError_t launch_fp4_linear(int dtype, const Fp4LinearArgs &a, int sms, void *encode, void *work, cudaStream_t s, uint64_t *launches);

}  // namespace tcu

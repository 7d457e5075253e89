// Linear layers with four-bit weights and group scales.
#include <algorithm>
#include <atomic>

#include <cooperative_groups.h>

#include "device.cuh"
#include "fourbit.cuh"

namespace tcu {

namespace cg = cooperative_groups;

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


// y = act(x W^T + bias) + residual for a few rows of x: the weights stream from memory once, as codes, and go into the
// matrix unit as they are. A nibble is a subnormal f16 (code * 2^-24, or 2^-20 from a byte's second nibble: one AND takes
// two out of a word; f32 takes code - 8 instead, see code_pair), so a product with the codes is exact in everything but x,
// which is one f16 for the 16-bit types and the sum of two for f32; the group scales act on the f32 result:
//     sum over groups of  step * (x_g . codes)  +  low * (sum of x_g)
//
// A warp takes 16 outputs (the rows of the matrix fragments) over a part of K, its weights arriving in a ring of its own a
// few blocks ahead; the rows of x are the 8 NT columns, as fragments in shared memory: up to 8 rows are laid out by every
// block for itself, more by a kernel before. K is cut over the blocks of a cluster (each holds its own slice of x only)
// and over `parts` of a block's warps; the partial outputs meet in shared memory, in a fixed order.
//
// What bounds it: launch, laying out x and joining take 8 to 10 us of a call; the weights then stream at 4 to 5 TB/s, the
// rest of the time going into the codes (about 150 instructions a warp and 16 x 128 weights). 14336 x 8192 weights in groups
// of 128 by 8 bf16 rows: 23.5 us (63 MB, floor 9.6); 4097 x 2050 in groups of 32 by 50 f16 rows: 20.5 us; 1024 x 512 by one
// f32 row with GELU: 5.1 us.
constexpr int W4_WARPS = 8, W4_X_BYTES = 65536, W4_Y_UNITS = 64;
constexpr int W4_DEPTH = 3;   // steps a warp's ring holds
constexpr int W4_SLICE = 16;  // most blocks of columns of x that a block holds at once

struct W4Plan {
    // tiles: of 16 outputs, a block's at a time; parts: log2 of the parts of a pass; slice, pass: blocks of 128 columns
    int nt, cs, groups, tiles, parts, slice, pass, row_tiles;
};

__device__ __forceinline__ uint32_t w4_half2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ float2 w4_float2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2 *>(&w)); }
__device__ __forceinline__ void w4_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight columns of a row of x from column c (0 past k).
template <int DT>
__device__ __forceinline__ void w4_x8(const void *row, int c, int k, bool wide, float (&v)[8]) {
    const typename Elem<DT>::T *x = reinterpret_cast<const typename Elem<DT>::T *>(row);
    if (c + 8 <= k) {
        load8<DT>(x + c, wide, v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = c + j < k ? Elem<DT>::get(x[c + j]) : 0.f;
    }
}
__device__ __forceinline__ void w4_x8(int dtype, const void *row, int c, int k, bool wide, float (&v)[8]) {
    if (dtype == DT_F32)
        w4_x8<DT_F32>(row, c, k, wide, v);
    else if (dtype == DT_F16)
        w4_x8<DT_F16>(row, c, k, wide, v);
    else
        w4_x8<DT_BF16>(row, c, k, wide, v);
}
__device__ __forceinline__ float w4_get(int dtype, const void *p, long long i) {
    if (dtype == DT_F32) return reinterpret_cast<const float *>(p)[i];
    if (dtype == DT_F16) return __half2float(reinterpret_cast<const __half *>(p)[i]);
    return __bfloat162float(reinterpret_cast<const __nv_bfloat16 *>(p)[i]);
}

// x as fragments: word k of a unit and lane (row m % 8, quarter q of the unit) holds columns k and k + 4 of 8, scaled by
// `up`; a weight word's second nibbles come 16 times as large, so every other word is 1/16 of it. Returns the columns' sum.
template <int QS>
__device__ __forceinline__ float w4_fragment(const float (&v)[8], float up, uint4 (&h)[QS]) {
    float s = 0.f;
    uint32_t w[QS][4];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const float f = k & 1 ? 0.0625f : 1.f, x0 = v[k] * up, x1 = v[k + 4] * up;
        w[0][k] = w4_half2(x0 * f, x1 * f);
        if constexpr (QS == 2) {
            const float2 o = w4_float2(w[0][k]);
            w[1][k] = w4_half2(fmaf(x0, f, -o.x), fmaf(x1, f, -o.y));
        }
        s += x0 + x1;
    }
#pragma unroll
    for (int k = 0; k < QS; k++) h[k] = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
    return s;
}
__device__ __forceinline__ constexpr float w4_unit(int qs) { return qs == 2 ? 1.f : 5.9604644775390625e-8f; }  // the codes': centred, or 2^-24
// The power of two that brings a row's largest magnitude into [2^13, 2^14) (below 2^-113 as near as f32 holds its inverse),
// and what undoes it on the sums.
__device__ __forceinline__ float w4_up(float mx, float &undo) {
    const int e = mx > 0.f ? min(126, 140 - (int)((__float_as_uint(mx) >> 23) & 0xff)) : 0;
    undo = __uint_as_float((uint32_t)(127 - e) << 23);
    return __uint_as_float((uint32_t)(e + 127) << 23);
}
// Words of fragments and floats of sums of one block of 128 columns of 8 NT rows.
__host__ __device__ constexpr int w4_frag_words(int nt, int qs) { return nt * qs * 512; }

// Fragments of more than 8 rows, laid out once for all blocks of the product: one block a row.
template <int G, int NT, int QS>
__global__ void __launch_bounds__(256) k_w4_x(W4Args a, int dtype, uint32_t *xf, float *xs, float *fx) {
    constexpr int NG = 128 / G, R = 8 * NT;
    __shared__ float red[8];
    const int blocks = (a.k + 127) / 128, m = blockIdx.x % R, rt = blockIdx.x / R, lane = threadIdx.x & 31;
    const bool there = (int)blockIdx.x < a.rows;
    const int es = dtype == DT_F32 ? 4 : 2;
    const bool wide = !(((uintptr_t)a.x & 15) || (a.ldx * es) % 16);
    const void *row = reinterpret_cast<const uint8_t *>(a.x) + (long long)(there ? blockIdx.x : 0) * a.ldx * es;
    float mx = 0.f, v[8];
    if (there)
        for (int c = threadIdx.x * 8; c < a.k; c += 2048) {
            w4_x8(dtype, row, c, a.k, wide, v);
#pragma unroll
            for (int j = 0; j < 8; j++) mx = fmaxf(mx, fabsf(v[j]));
        }
    mx = warp_max(mx);
    if (lane == 0) red[threadIdx.x >> 5] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; w++) mx = fmaxf(mx, red[w]);
    float undo;
    const float up = w4_up(mx, undo);
    if (threadIdx.x == 0) fx[rt * R + m] = undo;
    for (int i0 = 0; i0 < blocks * 16; i0 += 256) {
        const int i = i0 + threadIdx.x, b = i / 16, u = i % 16 / 4, q = i % 4;
        const bool on = i < blocks * 16;
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = 0.f;
        if (on && there) w4_x8(dtype, row, i * 8, a.k, wide, v);
        uint4 h[QS];
        float s = w4_fragment<QS>(v, up, h);
#pragma unroll
        for (int k = 0; k < QS; k++)
            if (on)
                *reinterpret_cast<uint4 *>(xf + ((size_t)(rt * blocks + b) * NT * QS + (m / 8) * QS + k) * 512 + u * 128 + (m % 8 * 4 + q) * 4) = h[k];
#pragma unroll
        for (int d = 1; d < G / 8; d *= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
        if (on && i % (G / 8) == 0) xs[((size_t)(rt * blocks + b) * NG + i % 16 / (G / 8)) * R + m] = s * w4_unit(QS);
    }
}

__device__ __forceinline__ uint32_t w4_smem(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
template <int N>
__device__ __forceinline__ void w4_cp(void *dst, const void *src) {
    if constexpr (N == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(w4_smem(dst)), "l"(src) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(w4_smem(dst)), "l"(src), "n"(N) : "memory");
}

// One slot of a warp's ring: two blocks of 128 columns of 16 rows, 128 bytes of codes a row (of odd rows the two halves
// changed places, so that eight lanes' 16 bytes of two rows fall on different banks), then the rows' scales.
template <int G>
struct W4Ring {
    static constexpr int NG = 128 / G, BYTES = 2048 + 32 * NG * 4;
};

template <int G, int NT, int QS>
__global__ void __launch_bounds__(W4_WARPS * 32, NT < 8 ? 2 : 1) k_w4_linear(W4Args a, int dtype, W4Plan p, const uint32_t *gxf, const float *gxs,
                                                             const float *gfx) {
    constexpr int NG = 128 / G, R = 8 * NT, D = W4_DEPTH;
    using Ring = W4Ring<G>;
    extern __shared__ __align__(16) uint8_t sm[];
    uint8_t *rings = sm;                                                               // [warps][D][Ring::BYTES]
    uint32_t *xf = reinterpret_cast<uint32_t *>(sm + W4_WARPS * D * Ring::BYTES);      // [pass][NT][QS][4 units][32 lanes][4]
    float *xs = reinterpret_cast<float *>(xf + (size_t)p.pass * w4_frag_words(NT, QS));  // [pass][NG][R] sums of a group's x
    float *fx = xs + p.pass * NG * R;                                                  // [R] undoes x's scaling
    float *ybuf = fx + R;                                                              // [parts][tiles][R][16]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int slice = blockIdx.x % p.cs, group = blockIdx.x / p.cs, rt = blockIdx.y, r0 = rt * R, rows = min(R, a.rows - r0);
    const int blocks = (a.k + 127) / 128, b_lo = min(blocks, slice * p.slice), b_hi = min(blocks, b_lo + p.slice);
    const int all = (a.n + 15) / 16;
    uint8_t *ring = rings + warp * D * Ring::BYTES;

    for (int tile0 = group * p.tiles; tile0 < all; tile0 += p.groups * p.tiles) {
        const int tiles = min(p.tiles, all - tile0), units = tiles << p.parts;
        for (int b0 = b_lo; b0 == b_lo || b0 < b_hi; b0 += p.pass) {
            const int nb = max(0, min(p.pass, b_hi - b0)), parts = 1 << p.parts, per = ((nb + 1) / 2 + parts - 1) >> p.parts;
            // A warp's units (tile, part of the pass) run on without a break, two blocks of columns a step: the next D - 1 steps
            // are on their way while one is computed.
            const int mine = warp < units ? (units - warp + W4_WARPS - 1) / W4_WARPS : 0, total = per * mine;
            int fu = warp, fb = 0, fetched = 0, fslot = 0;
            const uint8_t *src[4], *ssrc;  // this lane's rows of the unit fetched next, its 16 bytes and its scales of the first block
            const int half = lane >> 4;
            auto fetch = [&]() {
                if (fetched < total) {
                    const int b = b0 + ((fu & (parts - 1)) * per + fb) * 2;
                    if (fb == 0) {
                        const int tile = tile0 + (fu >> p.parts);
#pragma unroll
                        for (int x = 0; x < 4; x++)  // rows past n are read as the last, and not used
                            src[x] = a.codes + (size_t)min(tile * 16 + x * 4 + (lane >> 3), a.n - 1) * blocks * 64;
                        ssrc = reinterpret_cast<const uint8_t *>(a.scales + (size_t)min(tile * 16 + (lane & 15), a.n - 1) * blocks * NG);
                    }
                    uint8_t *to = ring + fslot * Ring::BYTES;
                    // (a last block without a second is read twice)
                    const int c = lane & 7, at = min(b + (c >> 2), blocks - 1) * 64 + (c & 3) * 16;
#pragma unroll
                    for (int x = 0; x < 4; x++) w4_cp<16>(to + (x * 4 + (lane >> 3)) * 128 + (c ^ ((lane >> 3 & 1) << 2)) * 16, src[x] + at);
                    w4_cp<NG * 4>(to + 2048 + ((lane & 15) * 2 + half) * NG * 4, ssrc + min(b + half, blocks - 1) * NG * 4);
                    if (++fb == per) fb = 0, fu += W4_WARPS;
                }
                fetched++, fslot = fslot + 1 == D ? 0 : fslot + 1;
                asm volatile("cp.async.commit_group;" ::: "memory");
            };

            // the pass's x as fragments, unless they are there from the tiles before
            const bool lay = tile0 == group * p.tiles || b_hi - b_lo > p.pass;
            if (lay) __syncthreads();  // (the warps are done with those of the pass before)
            if (lay && NT > 1) {
                for (int i = tid; i < nb * w4_frag_words(NT, QS) / 4; i += W4_WARPS * 32)
                    w4_cp<16>(xf + 4 * i, gxf + ((size_t)rt * blocks + b0) * w4_frag_words(NT, QS) + 4 * i);
                for (int i = tid; i < nb * NG * R / 4; i += W4_WARPS * 32) w4_cp<16>(xs + 4 * i, gxs + ((size_t)rt * blocks + b0) * NG * R + 4 * i);
                if (tid < R) fx[tid] = gfx[rt * R + tid];
            }
#pragma unroll
            for (int i = 0; i < D - 1; i++) fetch();
            if (lay && NT == 1) {
                // a warp a row; its part is read once, into registers (up to 8 x 8 columns a lane)
                const int es = dtype == DT_F32 ? 4 : 2;
                const bool wide = !(((uintptr_t)a.x & 15) || (a.ldx * es) % 16);
                const uint8_t *row = reinterpret_cast<const uint8_t *>(a.x) + (long long)(r0 + min(warp, rows - 1)) * a.ldx * es;
                float v[W4_SLICE / 2][8], mx = 0.f;
                if (wide && (b0 + nb) * 128 <= a.k) {  // whole vectors, all asked for before any is used
                    uint4 raw[W4_SLICE / 2][QS];
                    const uint4 *src = reinterpret_cast<const uint4 *>(row + (size_t)b0 * 128 * es) + lane * QS;
#pragma unroll
                    for (int x = 0; x < W4_SLICE / 2; x++)
#pragma unroll
                        for (int k = 0; k < QS; k++)
                            raw[x][k] = warp < rows && x * 32 + lane < nb * 16 ? __ldg(src + x * 32 * QS + k) : make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int x = 0; x < W4_SLICE / 2; x++) {
                        const uint32_t w[4] = {raw[x][0].x, raw[x][0].y, raw[x][0].z, raw[x][0].w};
                        if constexpr (QS == 2) {
                            const uint32_t z[4] = {raw[x][1].x, raw[x][1].y, raw[x][1].z, raw[x][1].w};
#pragma unroll
                            for (int j = 0; j < 4; j++) v[x][j] = __uint_as_float(w[j]), v[x][j + 4] = __uint_as_float(z[j]);
                        } else {
#pragma unroll
                            for (int j = 0; j < 4; j++) {
                                const float2 f = dtype == DT_BF16 ? make_float2(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xffff0000u)) : w4_float2(w[j]);
                                v[x][2 * j] = f.x, v[x][2 * j + 1] = f.y;
                            }
                        }
                    }
                } else {
#pragma unroll
                    for (int x = 0; x < W4_SLICE / 2; x++) {
#pragma unroll
                        for (int j = 0; j < 8; j++) v[x][j] = 0.f;
                        if (warp < rows && x * 32 + lane < nb * 16) w4_x8(dtype, row, b0 * 128 + (x * 32 + lane) * 8, a.k, wide, v[x]);
                    }
                }
#pragma unroll
                for (int x = 0; x < W4_SLICE / 2; x++)
#pragma unroll
                    for (int j = 0; j < 8; j++) mx = fmaxf(mx, fabsf(v[x][j]));
                float undo;
                const float up = w4_up(warp_max(mx), undo);
                if (lane == 0) fx[warp] = undo;
#pragma unroll
                for (int x = 0; x < W4_SLICE / 2; x++) {
                    const int i = x * 32 + lane, b = i / 16, u = i % 16 / 4, q = i % 4;
                    const bool on = i < nb * 16;
                    uint4 h[QS];
                    float s = w4_fragment<QS>(v[x], up, h);
#pragma unroll
                    for (int k = 0; k < QS; k++)
                        if (on) *reinterpret_cast<uint4 *>(xf + (b * QS + k) * 512 + u * 128 + (warp * 4 + q) * 4) = h[k];
#pragma unroll
                    for (int d = 1; d < G / 8; d *= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
                    if (on && i % (G / 8) == 0) xs[(b * NG + i % 16 / (G / 8)) * R + warp] = s * w4_unit(QS);
                }
            }
            if (lay) {
                // (x's copies are the oldest group of every thread)
                if (NT > 1) asm volatile("cp.async.wait_group %0;" ::"n"(D - 2) : "memory");
                __syncthreads();
            }

            float y[NT][4];
            int unit = warp, in = 0, slot = 0;
            for (int now = 0; now < total; now++) {
                asm volatile("cp.async.wait_group %0;" ::"n"(D - 2) : "memory");
                __syncwarp();  // every lane's part has landed, and every lane is done with the slot that is filled next
                fetch();
                if (in == 0) {
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) y[nt][0] = y[nt][1] = y[nt][2] = y[nt][3] = 0.f;
                }
                const uint8_t *wb = ring + slot * Ring::BYTES;
                slot = slot + 1 == D ? 0 : slot + 1;
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const int b = ((unit & (parts - 1)) * per + in) * 2 + k;
                    if (b >= nb) break;
                    const int c = (k * 4 + t) ^ ((g & 1) << 2);
                    const uint4 k0 = *reinterpret_cast<const uint4 *>(wb + g * 128 + c * 16), k1 = *reinterpret_cast<const uint4 *>(wb + (g + 8) * 128 + c * 16);
                    const uint32_t c0[4] = {k0.x, k0.y, k0.z, k0.w}, c1[4] = {k1.x, k1.y, k1.z, k1.w};
                    const uint32_t *sc = reinterpret_cast<const uint32_t *>(wb + 2048) + k * NG;
                    const uint32_t *xb = xf + b * w4_frag_words(NT, QS) + lane * 4;
#pragma unroll
                    for (int q = 0; q < NG; q++) {
                        float acc[NT][4] = {};
#pragma unroll
                        for (int u = q * (G / 32); u < (q + 1) * (G / 32); u++) {
                            const uint32_t v0 = c0[u] >> 8, v1 = c1[u] >> 8;
#pragma unroll
                            for (int nt = 0; nt < NT; nt++)
#pragma unroll
                                for (int z = QS - 1; z >= 0; z--) {
                                    const uint4 x = *reinterpret_cast<const uint4 *>(xb + ((nt * QS + z) * 4 + u) * 128);
                                    w4_mma(acc[nt], code_pair<QS == 2, false>(c0[u]), code_pair<QS == 2, false>(c1[u]), code_pair<QS == 2, true>(c0[u]), code_pair<QS == 2, true>(c1[u]), x.x, x.y);
                                    w4_mma(acc[nt], code_pair<QS == 2, false>(v0), code_pair<QS == 2, false>(v1), code_pair<QS == 2, true>(v0), code_pair<QS == 2, true>(v1), x.z, x.w);
                                }
                        }
                        float2 s0 = w4_float2(sc[g * 2 * NG + q]), s1 = w4_float2(sc[(g + 8) * 2 * NG + q]);
                        if (QS == 2) s0.y = fmaf(8.f, s0.x, s0.y), s1.y = fmaf(8.f, s1.x, s1.y);  // the codes came less 8
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) {
                            const float2 sx = *reinterpret_cast<const float2 *>(xs + (b * NG + q) * R + nt * 8 + 2 * t);
                            y[nt][0] = fmaf(s0.x, acc[nt][0], fmaf(s0.y, sx.x, y[nt][0]));
                            y[nt][1] = fmaf(s0.x, acc[nt][1], fmaf(s0.y, sx.y, y[nt][1]));
                            y[nt][2] = fmaf(s1.x, acc[nt][2], fmaf(s1.y, sx.x, y[nt][2]));
                            y[nt][3] = fmaf(s1.x, acc[nt][3], fmaf(s1.y, sx.y, y[nt][3]));
                        }
                    }
                }
                if (++in < per) continue;
                // the unit's partial outputs, added to those of the passes before (the same warp's)
                float *yb = ybuf + ((unit & (parts - 1)) * p.tiles + (unit >> p.parts)) * R * 16;
#pragma unroll
                for (int nt = 0; nt < NT; nt++)
#pragma unroll
                    for (int c = 0; c < 4; c++) {
                        const int m = nt * 8 + 2 * t + (c & 1);
                        float *at = yb + m * 16 + (c >> 1) * 8 + g;
                        const float v = y[nt][c] * (1.f / w4_unit(QS)) * fx[m];
                        *at = b0 == b_lo ? v : *at + v;
                    }
                in = 0, unit += W4_WARPS;
            }
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        // ---- the partial outputs joined: the parts' by the block, the slices' by the cluster, each block a share ----
        __syncthreads();
        const int wide_n = tiles * 16;
        if (p.parts && b_lo < b_hi) {
            for (int i = tid; i < wide_n * R; i += W4_WARPS * 32) {
                float v = ybuf[i];
                for (int q = 1; q < 1 << p.parts; q++) v += ybuf[q * p.tiles * R * 16 + i];
                ybuf[i] = v;
            }
        }
        cg::cluster_group cl = cg::this_cluster();
        if (p.cs > 1)
            cl.sync();
        else
            __syncthreads();
        for (int i = slice * W4_WARPS * 32 + tid; i < wide_n * rows; i += p.cs * W4_WARPS * 32) {
            const int m = i / wide_n, nn = i % wide_n, n = tile0 * 16 + nn;
            if (n >= a.n) continue;
            float v = 0.f;
            for (int c = 0; c < p.cs && c * p.slice < blocks; c++) {  // (blocks past the last column have nothing)
                const float *from = p.cs > 1 ? cl.map_shared_rank(ybuf, c) : ybuf;
                v += from[(nn / 16 * R + m) * 16 + nn % 16];
            }
            if (a.bias) v += w4_get(dtype, a.bias, n);
            if (a.act) v = gelu1(v);
            if (a.residual) v += w4_get(dtype, a.residual, (long long)(r0 + m) * a.ldr + n);
            const long long at = (long long)(r0 + m) * a.ldy + n;
            if (dtype == DT_F32)
                reinterpret_cast<float *>(a.y)[at] = v;
            else if (dtype == DT_F16)
                reinterpret_cast<__half *>(a.y)[at] = __float2half_rn(v);
            else
                reinterpret_cast<__nv_bfloat16 *>(a.y)[at] = __float2bfloat16_rn(v);
        }
        if (p.cs > 1)
            cl.sync();  // every block has read the others' before they are written again, or gone
        else
            __syncthreads();
    }
}

// How many clusters of cs blocks of two an SM the GPU holds at once: a cluster lies within one of the GPU's processing
// clusters, so it is fewer than their blocks over cs (with one cluster too many the product takes twice as long).
static int w4_clusters(int cs, int sms) {
    static std::atomic<int> known[4];
    const int i = cs == 1 ? 0 : cs == 2 ? 1 : cs == 4 ? 2 : 3;
    int n = known[i];
    if (!n) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(2 * sms / cs * cs), cfg.blockDim = dim3(W4_WARPS * 32), cfg.dynamicSmemBytes = 100 << 10;
        cudaLaunchAttribute at[1];
        at[0].id = cudaLaunchAttributeClusterDimension;
        at[0].val.clusterDim.x = cs, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
        cfg.attrs = at, cfg.numAttrs = 1;
        const auto kernel = k_w4_linear<128, 1, 1>;
        if (allow_dynamic_smem((const void *)kernel, cfg.dynamicSmemBytes) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess || n < 1)
            n = std::max(1, 2 * sms / cs);
        known[i] = n;
    }
    return n;
}

static size_t w4_smem_bytes(const W4Plan &p, int group, int qs) {
    const int ng = 128 / group, r = 8 * p.nt;
    return (size_t)W4_WARPS * W4_DEPTH * (2048 + 32 * ng * 4) + (size_t)p.pass * w4_frag_words(p.nt, qs) * 4 +
           sizeof(float) * (p.pass * ng * r + r + (((size_t)p.tiles * r * 16) << p.parts));
}

// (the largest of these shared-memory sizes is 216,320 bytes: 32-wide groups, 7 blocks of 64 rows, 64 units of outputs)
static W4Plan w4_plan(int dtype, const W4Args &a, int sms) {
    W4Plan p;
    const int qs = dtype == DT_F32 ? 2 : 1, blocks = (a.k + 127) / 128, tiles = (a.n + 15) / 16;
    p.nt = a.rows <= 8 ? 1 : a.rows <= 16 ? 2 : a.rows <= 32 || qs == 2 ? 4 : 8;
    p.row_tiles = (a.rows + 8 * p.nt - 1) / (8 * p.nt);
    // a slice of at most 16 blocks of columns, up to 8 slices; more where there are too few outputs to fill the GPU
    p.cs = 1;
    while (p.cs < 8 && (blocks > W4_SLICE * p.cs || (blocks >= 16 * p.cs && tiles * p.cs * 2 <= sms))) p.cs *= 2;
    p.slice = (blocks + p.cs - 1) / p.cs;
    for (int resident = 2; resident >= 1; resident--) {  // blocks an SM: one may hold more of x at once
        const int most = std::min(W4_SLICE, std::max(1, (resident == 1 ? W4_X_BYTES * 7 / 4 : W4_X_BYTES) / (4 * w4_frag_words(p.nt, qs))));
        const int passes = (p.slice + most - 1) / most;
        p.pass = (p.slice + passes - 1) / passes;
        p.groups = std::min(tiles, std::max(1, w4_clusters(p.cs, sms) * resident / 2 / p.row_tiles));
        p.tiles = std::min((tiles + p.groups - 1) / p.groups, W4_Y_UNITS / p.nt);
        p.groups = std::min(p.groups, (tiles + p.tiles - 1) / p.tiles);
        // a power of two of parts of a slice where the warps share the tiles more evenly by it: a warp that streams a whole
        // slice of its rows reads memory in longer runs (14336 x 8192: 25.4 us with one part of 16 steps, 27.2 us with four
        // of 14)
        p.parts = 0;
        for (int h = 1; h <= 3 && 2 << h <= p.pass + 1 && p.tiles << h <= W4_Y_UNITS / p.nt; h++) {
            auto cost = [&](int x) { return (((p.tiles << x) + W4_WARPS - 1) / W4_WARPS) * (((p.pass + 1) / 2 + (1 << x) - 1) >> x); };
            if (cost(h) * 8 < cost(p.parts) * 7) p.parts = h;
        }
        if (w4_smem_bytes(p, a.group, qs) <= 113 * 1024 && passes == 1) break;
    }
    return p;
}

// More than 8 rows: after attention's counters the fragments, the groups' sums and the rows' factors, one after the other.
static size_t w4_frag_bytes(const W4Args &a, const W4Plan &p, int qs) { return (size_t)p.row_tiles * ((a.k + 127) / 128) * w4_frag_words(p.nt, qs) * 4; }
static size_t w4_sum_bytes(const W4Args &a, const W4Plan &p) { return (size_t)p.row_tiles * ((a.k + 127) / 128) * (128 / a.group) * 8 * p.nt * 4; }
size_t w4_linear_workspace(int dtype, const W4Args &a, int sms) {
    if (a.rows <= 8) return 0;
    const W4Plan p = w4_plan(dtype, a, sms);
    return 4 * KA_BLOCKS + w4_frag_bytes(a, p, dtype == DT_F32 ? 2 : 1) + w4_sum_bytes(a, p) + (size_t)p.row_tiles * 8 * p.nt * 4;
}

template <int G, int NT, int QS>
static cudaError_t launch_w4(int dtype, const W4Args &a, const W4Plan &p, void *work, cudaStream_t s, uint64_t *launches) {
    const size_t smem = w4_smem_bytes(p, G, QS);
    cudaError_t e = allow_dynamic_smem((const void *)k_w4_linear<G, NT, QS>, smem);
    if (e != cudaSuccess) return e;
    uint32_t *xf = nullptr;
    float *xs = nullptr, *fx = nullptr;
    if constexpr (NT > 1) {
        xf = reinterpret_cast<uint32_t *>(work) + KA_BLOCKS;
        xs = reinterpret_cast<float *>(xf + w4_frag_bytes(a, p, QS) / 4);
        fx = xs + w4_sum_bytes(a, p) / 4;
        k_w4_x<G, NT, QS><<<p.row_tiles * 8 * NT, 256, 0, s>>>(a, dtype, xf, xs, fx);
        if (launches) ++*launches;
        if ((e = cudaGetLastError()) != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.groups * p.cs, p.row_tiles), cfg.blockDim = dim3(W4_WARPS * 32), cfg.dynamicSmemBytes = smem, cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = p.cs, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    cfg.attrs = at, cfg.numAttrs = p.cs > 1 ? 1 : 0;
    if (launches) ++*launches;
    return cudaLaunchKernelEx(&cfg, k_w4_linear<G, NT, QS>, a, dtype, p, (const uint32_t *)xf, (const float *)xs, (const float *)fx);
}
template <int G>
static cudaError_t launch_w4(int dtype, const W4Args &a, const W4Plan &p, void *work, cudaStream_t s, uint64_t *launches) {
    if (dtype == DT_F32)
        return p.nt == 1   ? launch_w4<G, 1, 2>(dtype, a, p, work, s, launches)
               : p.nt == 2 ? launch_w4<G, 2, 2>(dtype, a, p, work, s, launches)
                           : launch_w4<G, 4, 2>(dtype, a, p, work, s, launches);
    return p.nt == 1   ? launch_w4<G, 1, 1>(dtype, a, p, work, s, launches)
           : p.nt == 2 ? launch_w4<G, 2, 1>(dtype, a, p, work, s, launches)
           : p.nt == 4 ? launch_w4<G, 4, 1>(dtype, a, p, work, s, launches)
                       : launch_w4<G, 8, 1>(dtype, a, p, work, s, launches);
}

cudaError_t launch_w4_linear(int dtype, const W4Args &a, int sms, void *work, size_t work_bytes, cudaStream_t s, uint64_t *launches) {
    if (!a.rows) return cudaSuccess;
    if (w4_linear_workspace(dtype, a, sms) > work_bytes) return cudaErrorInvalidValue;
    const W4Plan p = w4_plan(dtype, a, sms);
    return a.group == 32   ? launch_w4<32>(dtype, a, p, work, s, launches)
           : a.group == 64 ? launch_w4<64>(dtype, a, p, work, s, launches)
                           : launch_w4<128>(dtype, a, p, work, s, launches);
}

}  // namespace tcu

// Linear layers with four-bit weights and group scales.
#include <algorithm>

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
// two out of a word), so a product with the codes is exact in everything but x, which is one f16 for the 16-bit types and
// the sum of two for f32; the group scales act on the f32 result:
//     sum over groups of  step * (x_g . codes)  +  low * (sum of x_g)
//
// A warp takes 16 outputs (the rows of the matrix fragments, read 16 bytes a thread straight from memory) over a part of
// K; the rows of x are the 8 NT columns, laid out once a block as fragments in shared memory. K is cut over the blocks of
// a cluster (each lays out its own slice of x only) and over `parts` of a block's warps; the partial outputs meet in
// shared memory, in a fixed order.
constexpr int W4_WARPS = 8, W4_X_BYTES = 65536, W4_Y_UNITS = 128;

struct W4Plan {
    int nt, cs, groups, tiles, parts, slice, pass, row_tiles;  // tiles: of 16 outputs, a block's at a time; slice, pass: blocks of 128 columns
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

// One block of 128 columns of the two weight rows of a thread.
template <int G>
struct W4Block {
    static constexpr int NG = 128 / G;
    uint4 c[2];
    uint32_t s[2][NG];
};
template <int G>
__device__ __forceinline__ void w4_load(W4Block<G> &w, const uint8_t *const (&codes)[2], const uint32_t *const (&scales)[2], int b, int t) {
    constexpr int NG = W4Block<G>::NG;
#pragma unroll
    for (int r = 0; r < 2; r++) {
        w.c[r] = __ldcs(reinterpret_cast<const uint4 *>(codes[r] + (size_t)b * 64) + t);
        const uint32_t *s = scales[r] + (size_t)b * NG;
        if constexpr (NG == 4) {
            const uint4 v = __ldg(reinterpret_cast<const uint4 *>(s));
            w.s[r][0] = v.x, w.s[r][1] = v.y, w.s[r][2] = v.z, w.s[r][3] = v.w;
        } else if constexpr (NG == 2) {
            const uint2 v = __ldg(reinterpret_cast<const uint2 *>(s));
            w.s[r][0] = v.x, w.s[r][1] = v.y;
        } else {
            w.s[r][0] = __ldg(s);
        }
    }
}

template <int G, int NT, int QS>
__global__ void __launch_bounds__(W4_WARPS * 32) k_w4_linear(W4Args a, int dtype, W4Plan p) {
    constexpr int NG = 128 / G, R = 8 * NT;
    extern __shared__ __align__(16) uint8_t sm[];
    uint32_t *xf = reinterpret_cast<uint32_t *>(sm);                             // [pass][NT][QS][4 units][32 lanes][4]
    float *xs = reinterpret_cast<float *>(xf + (size_t)p.pass * NT * QS * 512);  // [pass][NG][R] sums of a group's x
    float *fx = xs + p.pass * NG * R;                                            // [R] undoes x's scaling
    float *ybuf = fx + R;                                                        // [parts][tiles][R][16]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int slice = blockIdx.x % p.cs, group = blockIdx.x / p.cs, r0 = blockIdx.y * R, rows = min(R, a.rows - r0);
    const int blocks = (a.k + 127) / 128, b_lo = min(blocks, slice * p.slice), b_hi = min(blocks, b_lo + p.slice);
    const int all = (a.n + 15) / 16;
    const int es = dtype == DT_F32 ? 4 : 2;
    const bool wide = !(((uintptr_t)a.x & 15) || (a.ldx * es) % 16);

    for (int tile0 = group * p.tiles; tile0 < all; tile0 += p.groups * p.tiles) {
        const int tiles = min(p.tiles, all - tile0), units = tiles * p.parts;
        for (int b0 = b_lo; b0 == b_lo || b0 < b_hi; b0 += p.pass) {
            const int nb = max(0, min(p.pass, b_hi - b0)), per = (nb + p.parts - 1) / p.parts;
            // a warp's units (tile, part of the pass) run on without a break: the next two blocks are on their way while
            // two are computed
            const int steps = (per + 1) / 2, mine = warp < units ? (units - warp + W4_WARPS - 1) / W4_WARPS : 0;
            W4Block<G> w[2][2];
            auto fetch = [&](int step, W4Block<G>(&to)[2]) {
                const int unit = warp + step / steps * W4_WARPS, tile = tile0 + unit / p.parts;
                const int b = b0 + unit % p.parts * per + step % steps * 2;
                const uint8_t *codes[2];
                const uint32_t *scales[2];
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const size_t n = min(tile * 16 + r * 8 + g, a.n - 1);  // rows past n are read as the last, and not used
                    codes[r] = a.codes + n * blocks * 64;
                    scales[r] = reinterpret_cast<const uint32_t *>(a.scales) + n * blocks * NG;
                }
                w4_load<G>(to[0], codes, scales, min(b, blocks - 1), t);
                w4_load<G>(to[1], codes, scales, min(b + 1, blocks - 1), t);
            };
            const int total = steps * mine;
            if (total) fetch(0, w[0]);

            // the pass's x as fragments, unless they are there from the tiles before
            if (tile0 == group * p.tiles || b_hi - b_lo > p.pass) {
                __syncthreads();
                for (int m = warp; m < R; m += W4_WARPS) {
                    const uint8_t *row = reinterpret_cast<const uint8_t *>(a.x) + (long long)(r0 + min(m, rows - 1)) * a.ldx * es;
                    float mx = 0.f, v[8];
                    if (m < rows)
                        for (int c = b0 * 128 + lane * 8; c < min(a.k, (b0 + nb) * 128); c += 256) {
                            w4_x8(dtype, row, c, a.k, wide, v);
#pragma unroll
                            for (int j = 0; j < 8; j++) mx = fmaxf(mx, fabsf(v[j]));
                        }
                    mx = warp_max(mx);
                    // mx * 2^e in [2^13, 2^14)
                    const int e = mx > 0.f ? min(100, max(-100, 140 - (int)((__float_as_uint(mx) >> 23) & 0xff))) : 0;
                    const float up = __uint_as_float((uint32_t)(e + 127) << 23);
                    if (lane == 0) fx[m] = __uint_as_float((uint32_t)(127 - e) << 23) * 16777216.f;
                    for (int i0 = 0; i0 < nb * 16; i0 += 32) {
                        const int i = i0 + lane, b = i / 16, u = i % 16 / 4, q = i % 4;
                        const bool on = i < nb * 16;
                        float s = 0.f;
                        if (on && m < rows)
                            w4_x8(dtype, row, (b0 + b) * 128 + i % 16 * 8, a.k, wide, v);
                        else
#pragma unroll
                            for (int j = 0; j < 8; j++) v[j] = 0.f;
                        uint32_t h[2][4];
#pragma unroll
                        for (int k = 0; k < 4; k++) {  // word k: columns k and k + 4; a word's second nibbles are 16 times as large
                            const float f = k & 1 ? 0.0625f : 1.f, x0 = v[k] * up, x1 = v[k + 4] * up;
                            h[0][k] = w4_half2(x0 * f, x1 * f);
                            const float2 o = w4_float2(h[0][k]);
                            if (QS == 2) h[1][k] = w4_half2(fmaf(x0, f, -o.x), fmaf(x1, f, -o.y));
                            s += x0 + x1;
                        }
#pragma unroll
                        for (int k = 0; k < QS; k++)
                            if (on) *reinterpret_cast<uint4 *>(xf + (((b * NT + m / 8) * QS + k) * 4 + u) * 128 + (m % 8 * 4 + q) * 4) =
                                make_uint4(h[k][0], h[k][1], h[k][2], h[k][3]);
#pragma unroll
                        for (int d = 1; d < G / 8; d *= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
                        if (on && i % (G / 8) == 0) xs[(b * NG + i % 16 / (G / 8)) * R + m] = s * 5.9604644775390625e-8f;  // 2^-24
                    }
                }
                __syncthreads();
            }

            float y[NT][4];
            for (int step = 0; step < total; step += 2) {
#pragma unroll
                for (int half = 0; half < 2; half++) {
                    const int now = step + half;
                    if (now >= total) break;
                    if (now + 1 < total) fetch(now + 1, w[half ^ 1]);
                    const int unit = warp + now / steps * W4_WARPS, in = now % steps;
                    if (in == 0) {
#pragma unroll
                        for (int nt = 0; nt < NT; nt++) y[nt][0] = y[nt][1] = y[nt][2] = y[nt][3] = 0.f;
                    }
                    const int lo = unit % p.parts * per, hi = min(nb, lo + per);
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        const int b = lo + in * 2 + k;
                        if (b >= hi) break;
                        const W4Block<G> &wb = w[half][k];
                        const uint32_t c0[4] = {wb.c[0].x, wb.c[0].y, wb.c[0].z, wb.c[0].w};
                        const uint32_t c1[4] = {wb.c[1].x, wb.c[1].y, wb.c[1].z, wb.c[1].w};
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
                                        const uint4 x = *reinterpret_cast<const uint4 *>(xf + (((b * NT + nt) * QS + z) * 4 + u) * 128 + lane * 4);
                                        w4_mma(acc[nt], c0[u] & 0x000f000fu, c1[u] & 0x000f000fu, c0[u] & 0x00f000f0u, c1[u] & 0x00f000f0u, x.x, x.y);
                                        w4_mma(acc[nt], v0 & 0x000f000fu, v1 & 0x000f000fu, v0 & 0x00f000f0u, v1 & 0x00f000f0u, x.z, x.w);
                                    }
                            }
                            const float2 s0 = w4_float2(wb.s[0][q]), s1 = w4_float2(wb.s[1][q]);
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
                    if (in == steps - 1) {  // the unit's partial outputs, added to those of the passes before (the same warp's)
                        float *yb = ybuf + ((unit % p.parts) * p.tiles + unit / p.parts) * R * 16;
#pragma unroll
                        for (int nt = 0; nt < NT; nt++)
#pragma unroll
                            for (int c = 0; c < 4; c++) {
                                const int m = nt * 8 + 2 * t + (c & 1);
                                float *at = yb + m * 16 + (c >> 1) * 8 + g;
                                const float v = y[nt][c] * fx[m];
                                *at = b0 == b_lo ? v : *at + v;
                            }
                    }
                }
            }
        }
        // ---- the partial outputs joined: each block of the cluster takes a share ----
        cg::cluster_group cl = cg::this_cluster();
        if (p.cs > 1)
            cl.sync();
        else
            __syncthreads();
        const int wide_n = tiles * 16, count = wide_n * rows;
        for (int i = slice * W4_WARPS * 32 + tid; i < count; i += p.cs * W4_WARPS * 32) {
            const int m = i / wide_n, nn = i % wide_n, n = tile0 * 16 + nn;
            if (n >= a.n) continue;
            float v = 0.f;
            for (int c = 0; c < p.cs; c++) {
                if (c * p.slice >= blocks) break;  // no columns left for it
                const float *from = p.cs > 1 ? cl.map_shared_rank(ybuf, c) : ybuf;
                for (int q = 0; q < p.parts; q++) v += from[((q * p.tiles + nn / 16) * R + m) * 16 + nn % 16];
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

static W4Plan w4_plan(int dtype, const W4Args &a, int sms) {
    W4Plan p;
    const int qs = dtype == DT_F32 ? 2 : 1, blocks = (a.k + 127) / 128, tiles = (a.n + 15) / 16;
    p.nt = a.rows <= 8 ? 1 : a.rows <= 16 ? 2 : a.rows <= 32 || qs == 2 ? 4 : 8;
    p.row_tiles = (a.rows + 8 * p.nt - 1) / (8 * p.nt);
    // a slice of at most 16 blocks of columns (its x takes a block longer to lay out than its weights to stream beyond
    // that), up to 8 slices; more where there are too few outputs to fill the GPU
    p.cs = 1;
    while (p.cs < 8 && (blocks > 16 * p.cs || (blocks >= 16 * p.cs && tiles * p.cs * 2 <= sms))) p.cs *= 2;
    p.slice = (blocks + p.cs - 1) / p.cs;
    p.pass = std::min(p.slice, std::max(1, W4_X_BYTES / (2048 * p.nt * qs)));
    p.groups = std::min(tiles, std::max(1, 2 * sms / (p.cs * p.row_tiles)));
    p.tiles = std::min((tiles + p.groups - 1) / p.groups, W4_Y_UNITS / p.nt);
    p.groups = std::min(p.groups, (tiles + p.tiles - 1) / p.tiles);
    // parts of a slice so that the warps share the tiles evenly
    p.parts = 1;
    for (int h = 2; h <= 8 && h <= p.pass && p.tiles * h <= W4_Y_UNITS / p.nt; h *= 2) {
        auto cost = [&](int x) { return (p.tiles * x + W4_WARPS - 1) / W4_WARPS * ((p.pass + x - 1) / x); };
        if (cost(h) < cost(p.parts)) p.parts = h;
    }
    return p;
}

template <int G, int NT, int QS>
static cudaError_t launch_w4(int dtype, const W4Args &a, const W4Plan &p, cudaStream_t s) {
    const size_t smem = (size_t)p.pass * NT * QS * 2048 + sizeof(float) * (p.pass * (128 / G) * 8 * NT + 8 * NT + p.parts * p.tiles * 8 * NT * 16);
    cudaError_t e = allow_dynamic_smem((const void *)k_w4_linear<G, NT, QS>, smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.groups * p.cs, p.row_tiles), cfg.blockDim = dim3(W4_WARPS * 32), cfg.dynamicSmemBytes = smem, cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = p.cs, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    cfg.attrs = at, cfg.numAttrs = p.cs > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, k_w4_linear<G, NT, QS>, a, dtype, p);
}
template <int G>
static cudaError_t launch_w4(int dtype, const W4Args &a, const W4Plan &p, cudaStream_t s) {
    if (dtype == DT_F32)
        return p.nt == 1 ? launch_w4<G, 1, 2>(dtype, a, p, s) : p.nt == 2 ? launch_w4<G, 2, 2>(dtype, a, p, s) : launch_w4<G, 4, 2>(dtype, a, p, s);
    return p.nt == 1   ? launch_w4<G, 1, 1>(dtype, a, p, s)
           : p.nt == 2 ? launch_w4<G, 2, 1>(dtype, a, p, s)
           : p.nt == 4 ? launch_w4<G, 4, 1>(dtype, a, p, s)
                       : launch_w4<G, 8, 1>(dtype, a, p, s);
}

cudaError_t launch_w4_linear(int dtype, const W4Args &a, int sms, cudaStream_t s, uint64_t *launches) {
    if (!a.rows) return cudaSuccess;
    const W4Plan p = w4_plan(dtype, a, sms);
    if (launches) ++*launches;
    return a.group == 32 ? launch_w4<32>(dtype, a, p, s) : a.group == 64 ? launch_w4<64>(dtype, a, p, s) : launch_w4<128>(dtype, a, p, s);
}

}  // namespace tcu

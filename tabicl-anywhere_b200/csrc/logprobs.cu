// Log probabilities of given labels, the entropy and the top alternatives of rows of scores, in one pass over them.
//
// With m the largest score and d = (x - m) / T:  S = sum e^d, log p(label) = d_label - log S,
// entropy = log S - (sum e^d d) / S. A thread keeps (m, S, sum e^d d) of what it has seen and rescales them when a strip
// of 32 of its scores holds a larger one, so scores are read once. 4096 rows of 131,071 bf16 scores with five alternatives:
// 0.195 ms (1.07 GB, 5.5 TB/s) in runs of up to 40 ms, 0.224 in longer ones, when the power cap holds the SMs at 1680 MHz
// instead of 1965: instructions bound it (issue active 86%, an ex2 a score 65% of its pipe), not memory (64%). 16 rows of
// 128,000 with twenty: 13 us, the latency of two strips, the ranking and the cluster's join; 2048 rows of 10 classes: 3.9 us.
//
// Top alternatives: a strip's largest score is kept beside. The n-th largest of 32 disjoint parts' maxima is a bound that
// at least n scores reach and hardly more than n do, so after the pass only the few strips that reach it are read again
// and the scores that reach it are ranked by counting. Where more than 256 do (rows of equal scores) the row is read again
// by warps that keep sorted lists.
#include <algorithm>
#include <type_traits>

#include <cooperative_groups.h>

#include "fourbit.cuh"

namespace tcu {

namespace cg = cooperative_groups;

// LP_KEEP: strips a thread keeps a maximum of (longer rows share). 16, and at most 32 registers, let an SM hold eight blocks:
// 4096 rows of 131071 bf16 scores take 195 us in a short run (85% of a copy's rate), with 32 and five blocks 239 us.
constexpr int LP_THREADS = 256, LP_STRIP = 32, LP_KEEP = 16;

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
__device__ __forceinline__ int key_index(unsigned long long k) { return 0x7fffffff - (int)(uint32_t)k; }

// (m, S, E) of a set of scores: E = sum e^d d in units of log2 e. m starts at the lowest finite number, so that
// -infinity is e^-infinity = 0 everywhere.
struct Stats {
    float m, s, e;
};
__device__ __forceinline__ Stats no_scores() { return Stats{-FLT_MAX, 0.f, 0.f}; }
__device__ __forceinline__ float lp_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// A distance from the maximum in units of log2 e / T; far ones (-infinity) are held where e^d is 0 and e^d d too.
__device__ __forceinline__ float lp_dist(float x, float m, float c) { return fmaxf((x - m) * c, -1000.f); }
__device__ __forceinline__ void rebase(Stats &a, float m, float c) {
    const float d = lp_dist(a.m, m, c), f = lp_exp2(d);
    a.e = f * fmaf(a.s, d, a.e), a.s *= f, a.m = m;
}
__device__ __forceinline__ void add_score(Stats &a, float x, float c) {
    float t;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(t) : "f"((x - a.m) * c), "f"(-1000.f));  // a NaN stays one, and makes S NaN
    const float p = lp_exp2(t);
    a.s += p, a.e = fmaf(p, t, a.e);
}
__device__ __forceinline__ void join(Stats &a, Stats b, float c) {
    const float m = fmaxf(a.m, b.m);
    rebase(a, m, c), rebase(b, m, c);
    a.s += b.s, a.e += b.e;
}
__device__ __forceinline__ void warp_join(Stats &a, float c) {
    float m = a.m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    rebase(a, m, c);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) a.s += __shfl_xor_sync(0xffffffffu, a.s, o), a.e += __shfl_xor_sync(0xffffffffu, a.e, o);
}

struct RowResult {
    float m, log_s;  // log S; 0 for a row of nothing but -infinity
    float inv_t, entropy;
};
__device__ __forceinline__ RowResult finish(const Stats &a, float inv_t) {
    RowResult r;
    r.m = a.m, r.inv_t = inv_t;
    r.log_s = a.s == 0.f ? 0.f : logf(a.s);
    r.entropy = a.s == 0.f ? 0.f : r.log_s - a.e / a.s * 0.69314718055994530942f;
    return r;
}
__device__ __forceinline__ float log_prob(const RowResult &r, float x) { return (x - r.m) * r.inv_t - r.log_s; }

template <int DT>
__device__ __forceinline__ void write_labels(const LogprobArgs &a, const RowResult &r, int row, const typename Elem<DT>::T *x,
                                             int first, int step) {
    for (int k = first; k < a.per_row; k += step) {
        const size_t at = (size_t)row * a.per_row + k;
        const int id = a.labels[at];
        if (id >= a.classes) *reinterpret_cast<volatile int *>(a.err) = 1;
        a.out[at] = id < 0 ? 0.f : id >= a.classes ? NAN : log_prob(r, Elem<DT>::get(x[id]));
    }
}
__device__ __forceinline__ void write_top(const LogprobArgs &a, const RowResult &r, int row, int place, unsigned long long key) {
    const size_t at = (size_t)row * a.top + place;
    a.top_values[at] = key ? log_prob(r, key_score(key)) : -INFINITY;
    a.top_ids[at] = key ? key_index(key) : -1;
}

// A warp's sorted list (lane i holds the i-th largest key): take in the lanes' keys above its n-th.
__device__ __forceinline__ void list_insert(unsigned long long &list, unsigned long long key, int n, int lane) {
    unsigned want = __ballot_sync(0xffffffffu, key > __shfl_sync(0xffffffffu, list, n - 1));
    while (want) {
        const int b = __ffs(want) - 1;
        const unsigned long long c = __shfl_sync(0xffffffffu, key, b);
        const int place = __popc(__ballot_sync(0xffffffffu, list > c));
        const unsigned long long up = __shfl_up_sync(0xffffffffu, list, 1);
        list = lane < place ? list : lane == place ? c : up;
        const unsigned long long bound = __shfl_sync(0xffffffffu, list, n - 1);
        want &= want - 1;
        want &= __ballot_sync(0xffffffffu, key > bound);
    }
}

// The n-th largest of 32 lanes' values (by rank, equal ones by lane).
__device__ __forceinline__ float nth_of_lanes(float v, int n, int lane) {
    int rank = 0;
#pragma unroll
    for (int j = 0; j < 32; j++) {
        const float o = __shfl_sync(0xffffffffu, v, j);
        rank += o > v || (o == v && j < lane);
    }
    return __shfl_sync(0xffffffffu, v, __ffs(__ballot_sync(0xffffffffu, rank == n - 1)) - 1);
}

// Rows of up to 512 classes: one warp a row, the scores read again from cache for the sums.
template <int DT>
__global__ void __launch_bounds__(LP_THREADS) k_logprobs_warp(LogprobArgs a) {
    using T = typename Elem<DT>::T;
    const int lane = threadIdx.x & 31, row = blockIdx.x * (LP_THREADS / 32) + (threadIdx.x >> 5);
    if (row >= a.rows) return;
    const T *x = reinterpret_cast<const T *>(a.logits) + row * a.stride;
    const float c = a.inv_t * 1.44269504088896340736f;
    Stats st = no_scores();
    float mx = -INFINITY;
    for (int i = lane; i < a.classes; i += 32) mx = fmaxf(mx, Elem<DT>::get(x[i]));
    float m = fmaxf(mx, -FLT_MAX);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    st.m = m;
    for (int i = lane; i < a.classes; i += 32) add_score(st, Elem<DT>::get(x[i]), c);
    warp_join(st, c);
    const RowResult r = finish(st, a.inv_t);
    write_labels<DT>(a, r, row, x, lane, 32);
    if (a.entropy && lane == 0) a.entropy[row] = r.entropy;
    if (!a.top) return;
    const float bound = nth_of_lanes(mx, a.top, lane);
    unsigned long long list = 0;
    for (int i = lane; i - lane < a.classes; i += 32) {
        const float v = i < a.classes ? Elem<DT>::get(x[i]) : -INFINITY;
        list_insert(list, v >= bound ? rank_key(v, i) : 0, a.top, lane);
    }
    if (lane < a.top) write_top(a, r, row, lane, list);
}

// A strip: VEC 16-byte vectors of PER scores.
template <int DT>
struct Strip {
    static constexpr int PER = 16 / (int)sizeof(typename Elem<DT>::T), VEC = LP_STRIP / PER;
};

// One block, or a cluster of cs blocks, a row.
template <int DT>
__global__ void __launch_bounds__(LP_THREADS, 8) k_logprobs(LogprobArgs a, int cs) {
    using T = typename Elem<DT>::T;
    constexpr int PER = Strip<DT>::PER, VEC = Strip<DT>::VEC;
    __shared__ float strip_max[LP_KEEP][LP_THREADS];
    __shared__ unsigned long long cand[LP_THREADS], best[32];
    __shared__ Stats parts[LP_THREADS / 32], whole;
    __shared__ float s_group[32], s_bound;
    __shared__ int s_count;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, row = blockIdx.x / cs, part = blockIdx.x % cs;
    const T *x = reinterpret_cast<const T *>(a.logits) + row * a.stride;
    const float c = a.inv_t * 1.44269504088896340736f;
    // scores before the first and after the last whole vector, one a thread of the row's first block
    const int head = min(a.classes, (int)((16 - ((uintptr_t)x & 15)) & 15) / (int)sizeof(T));
    const int nv = (a.classes - head) / PER, tail = a.classes - head - nv * PER;
    const uint4 *xv = reinterpret_cast<const uint4 *>(x + head);
    const int odd = part ? -1 : tid < head ? tid : tid >= 16 && tid - 16 < tail ? head + nv * PER + tid - 16 : -1;
    const int vstep = LP_THREADS * VEC, strips = (nv + vstep - 1) / vstep;  // strips a thread of the whole row
    const int s0 = (int)((long long)strips * part / cs), s1 = (int)((long long)strips * (part + 1) / cs);
    const int share = (s1 - s0 + LP_KEEP - 1) / LP_KEEP;  // strips that share a kept maximum

    Stats st = no_scores();
    float top = -INFINITY, kept = -INFINITY;
    if (odd >= 0) {
        top = Elem<DT>::get(x[odd]);
        st.m = fmaxf(st.m, top);
        add_score(st, top, c);
    }
    auto strip_load = [&](int s, uint4 (&v)[VEC]) {
#pragma unroll
        for (int k = 0; k < VEC; k++) {
            const int i = s * vstep + k * LP_THREADS + tid;
            if (i < nv) {
                v[k] = __ldcs(xv + i);
            } else {  // past the row: -infinity
                const uint32_t none = DT == DT_F32 ? 0xff800000u : DT == DT_F16 ? 0xfc00fc00u : 0xff80ff80u;
                v[k] = make_uint4(none, none, none, none);
            }
        }
    };
    auto get = [](const uint4 &v, int j) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        if constexpr (DT == DT_F32) return __uint_as_float(w[j]);
        if constexpr (DT == DT_BF16) return __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
        const __half2 h = *reinterpret_cast<const __half2 *>(&w[j / 2]);
        return __half2float(j & 1 ? __high2half(h) : __low2half(h));
    };
    int keep = 0, fill = 0;
    for (int s = s0; s < s1; s++) {
        uint4 v[VEC];
        strip_load(s, v);
        // the strip's largest, 16-bit types two at a time (a NaN is passed over)
        float mx;
        if constexpr (DT == DT_F32) {
            mx = -INFINITY;
#pragma unroll
            for (int k = 0; k < VEC; k++) mx = fmaxf(fmaxf(fmaxf(mx, get(v[k], 0)), get(v[k], 1)), fmaxf(get(v[k], 2), get(v[k], 3)));
        } else {
            using T2 = typename std::conditional<DT == DT_F16, __half2, __nv_bfloat162>::type;
            T2 m2 = *reinterpret_cast<const T2 *>(&v[0].x);
#pragma unroll
            for (int k = 0; k < VEC; k++) {
                const T2 *w = reinterpret_cast<const T2 *>(&v[k]);
#pragma unroll
                for (int j = 0; j < 4; j++) m2 = __hmax2(m2, w[j]);
            }
            mx = fmaxf(Elem<DT>::get(m2.x), Elem<DT>::get(m2.y));
        }
        if (mx > st.m) rebase(st, mx, c);
#pragma unroll
        for (int k = 0; k < VEC; k++)
#pragma unroll
            for (int j = 0; j < PER; j++) add_score(st, get(v[k], j), c);
        top = fmaxf(top, mx), kept = fmaxf(kept, mx);
        if (++fill == share || s == s1 - 1) strip_max[keep][tid] = kept, kept = -INFINITY, fill = 0, keep++;
    }
    // ---- the threads' and blocks' sums joined ----
    warp_join(st, c);
    if (lane == 0) parts[warp] = st;
    float g = top;  // eight neighbours' largest: 32 parts of the block's scores
#pragma unroll
    for (int o = 1; o < 8; o *= 2) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
    if ((lane & 7) == 0) s_group[tid >> 3] = g;
    if (tid == 0) s_count = 0;
    __syncthreads();
    if (warp == 0) {
        Stats b = no_scores();
        if (lane < LP_THREADS / 32) b = parts[lane];
        warp_join(b, c);
        if (lane == 0) whole = b;
        if (a.top) {
            const float bound = nth_of_lanes(s_group[lane], a.top, lane);
            if (lane == 0) s_bound = bound;
        }
    }
    if (tid >= LP_THREADS - 32) best[tid - (LP_THREADS - 32)] = 0;
    __syncthreads();
    if (a.top) {
        const float bound = s_bound;
        auto push = [&](float v, int i) {
            if (!(v >= bound)) return;
            const unsigned long long k = rank_key(v, i);
            if (!k) return;
            const int at = atomicAdd(&s_count, 1);
            if (at < LP_THREADS) cand[at] = k;
        };
        if (odd >= 0) push(Elem<DT>::get(x[odd]), odd);
        if (top >= bound) {
            for (int k = 0; k * share < s1 - s0; k++) {
                if (!(strip_max[k][tid] >= bound)) continue;
                for (int s = s0 + k * share; s < min(s1, s0 + (k + 1) * share); s++) {
                    uint4 v[VEC];
                    strip_load(s, v);
#pragma unroll
                    for (int q = 0; q < VEC; q++)
#pragma unroll
                        for (int j = 0; j < PER; j++) push(get(v[q], j), head + (s * vstep + q * LP_THREADS + tid) * PER + j);
                }
            }
        }
        __syncthreads();
        int count = s_count;
        if (count > LP_THREADS) {  // many equal scores: sorted lists over this block's part of the row
            unsigned long long list = 0;
            if (warp == 0) list_insert(list, odd >= 0 ? rank_key(Elem<DT>::get(x[odd]), odd) : 0, a.top, lane);
            const int i0 = head + min(nv, s0 * vstep) * PER, i1 = head + min(nv, s1 * vstep) * PER;
            for (int i = i0 + warp * 32; i < i1; i += LP_THREADS)
                list_insert(list, i + lane < i1 ? rank_key(Elem<DT>::get(x[i + lane]), i + lane) : 0, a.top, lane);
            __syncthreads();
            cand[tid] = list;
            count = LP_THREADS;
            __syncthreads();
        }
        if (tid < count && cand[tid]) {
            const unsigned long long mine = cand[tid];
            int rank = 0;
            for (int j = 0; j < count; j++) rank += cand[j] > mine;
            if (rank < a.top) best[rank] = mine;
        }
        __syncthreads();
    }
    if (cs > 1) {
        cg::cluster_group cl = cg::this_cluster();
        cl.sync();
        if (part == 0) {
            if (a.top) {
                unsigned long long mine = 0;
                if (warp < cs) mine = cl.map_shared_rank(best, warp)[lane];
                __syncthreads();
                cand[tid] = mine;
            }
            if (warp == 0) {
                Stats b = no_scores();
                if (lane < cs) b = *cl.map_shared_rank(&whole, lane);
                warp_join(b, c);
                if (lane == 0) parts[0] = b;
            }
        }
        cl.sync();  // every block's shared memory has been read
        if (part) return;
        if (tid == 0) whole = parts[0];
        if (tid < 32) best[tid] = 0;
        __syncthreads();
        if (a.top && cand[tid]) {
            const unsigned long long mine = cand[tid];
            int rank = 0;
            for (int j = 0; j < cs * 32; j++) rank += cand[j] > mine;
            if (rank < a.top) best[rank] = mine;
        }
        __syncthreads();
    }
    const RowResult r = finish(whole, a.inv_t);
    write_labels<DT>(a, r, row, x, tid, LP_THREADS);
    if (a.entropy && tid == 0) a.entropy[row] = r.entropy;
    if (tid < a.top) write_top(a, r, row, tid, best[tid]);
}

template <int DT>
static cudaError_t launch_type(const LogprobArgs &a, int sms, cudaStream_t s) {
    if (a.classes <= 512) {
        k_logprobs_warp<DT><<<(a.rows + LP_THREADS / 32 - 1) / (LP_THREADS / 32), LP_THREADS, 0, s>>>(a);
        return cudaGetLastError();
    }
    // few long rows are shared by the blocks of a cluster: up to two blocks an SM, a strip or more for each
    int cs = 1;
    while (cs < 8 && (long long)a.rows * cs * 2 <= 2 * sms && a.classes / (cs * 2) >= LP_THREADS * LP_STRIP / 2) cs *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(a.rows * cs), cfg.blockDim = dim3(LP_THREADS), cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = cs, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    cfg.attrs = at, cfg.numAttrs = cs > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, k_logprobs<DT>, a, cs);
}

cudaError_t launch_logprobs(int dtype, const LogprobArgs &a, int sms, cudaStream_t s, uint64_t *launches) {
    if (!a.rows) return cudaSuccess;
    if (launches) ++*launches;
    if (dtype == DT_F32) return launch_type<DT_F32>(a, sms, s);
    return dtype == DT_F16 ? launch_type<DT_F16>(a, sms, s) : launch_type<DT_BF16>(a, sms, s);
}

}  // namespace tcu

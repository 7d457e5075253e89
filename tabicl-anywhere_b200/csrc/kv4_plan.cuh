// How attention, over the four-bit cache or over packed keys, is cut into work, from lengths that only the device has.
//
// A unit of work is a row tile (R query rows: a sequence's rows, the heads that share a cache head innermost) of one cache
// head, over the keys that its rows see, in steps of STEP keys that begin at a multiple of ALIGN. The steps of all units in
// a row are cut evenly over the blocks: block b takes steps [T b / N, T (b + 1) / N), whole units and at most one part of a
// unit at either end. Parts meet in the working memory; the last block of a unit to arrive joins them in their order. So
// sequences of very unequal length keep every block busy to the end, and the working memory is of a fixed size.
#pragma once
#include "fourbit.cuh"

namespace tcu {

template <int N>
__device__ __forceinline__ void lds_words(const uint8_t *p, uint32_t (&w)[N]) {  // N consecutive words, aligned to 4 N up to 16
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const uint4 v = reinterpret_cast<const uint4 *>(p)[i];
            w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
        }
    } else if constexpr (N == 2) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        w[0] = v.x, w[1] = v.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t *>(p);
    }
}

// A sequence's first row, its rows and cached tokens.
struct KaRows {
    int first, n, len;
    bool ok;
};
__device__ __forceinline__ KaRows ka_rows(const Kv4AttendArgs &a, int seq) {
    KaRows r;
    r.first = seq * a.max_rows, r.n = a.max_rows;
    if (a.starts) r.first = a.starts[seq], r.n = a.starts[seq + 1] - r.first;
    r.len = a.lens[seq];
    r.ok = !(r.first < 0 || r.n < 0 || r.n > a.max_rows || r.first > a.rows - r.n || r.len < 0 || r.len > a.max_len);
    return r;
}
// Row i of a sequence sees the tokens [ka_lo, ka_hi); both grow with i.
template <class A>
__device__ __forceinline__ int ka_hi(const A &a, const KaRows &s, int i) {
    return a.causal ? max(0, min(s.len, s.len - s.n + i + 1)) : s.len;
}
template <class A>
__device__ __forceinline__ int ka_lo(const A &a, const KaRows &s, int i) {
    return a.window ? max(0, s.len - s.n + i + 1 - a.window) : 0;
}

__device__ __forceinline__ long long ka_div(long long a, long long b) {  // not negative; 64-bit division only where it is needed
    return ((a | b) >> 32) ? a / b : (long long)((uint32_t)a / (uint32_t)b);
}

// EXTRA: a unit counts as so many steps more than it has, its first ones, which are none: what it costs besides its steps (its
// queries, its output), so that blocks with many short units have as much to do as those with few long ones.
template <int R, int ALIGN, int STEP, int EXTRA = 0>
struct KaCut {
    struct Span {
        int lo_min, lo_max, hi_min, hi_max, base, steps;  // what the tile's first and last rows see; where its steps begin
    };
    template <class A>
    static __device__ __forceinline__ Span span(const A &a, const KaRows &s, int each, int rt) {
        const int first = rt * R / each, last = (min(s.n * each, (rt + 1) * R) - 1) / each;
        Span p;
        p.lo_min = ka_lo(a, s, first), p.lo_max = ka_lo(a, s, last), p.hi_min = ka_hi(a, s, first), p.hi_max = ka_hi(a, s, last);
        p.base = p.lo_min & ~(ALIGN - 1);
        p.steps = (p.hi_max > p.lo_min ? (p.hi_max - p.base + STEP - 1) / STEP : 1) + EXTRA;  // no keys: a step that writes zeros
        return p;
    }
    template <class A>
    static __device__ __forceinline__ long long seq_steps(const A &a, int seq, int each) {  // a head's
        const KaRows s = ka_rows(a, seq);
        if (!s.ok) {
            *reinterpret_cast<volatile int *>(a.err) = 1;
            return 0;
        }
        const int tiles = (s.n * each + R - 1) / R;
        if (!a.causal && tiles) return (long long)tiles * span(a, s, each, 0).steps;
        long long n = 0;
        for (int rt = 0; rt < tiles; rt++) n += span(a, s, each, rt).steps;
        return n;
    }

    // A block's place: the steps [pos, end) of `total`, cut over `blocks`; pos is step `skip` of unit (seq, rt, head).
    struct Place {
        long long pos, end, total, blocks;
        int seq, rt, head, skip;
    };
    // Called by all THREADS threads of the block (of which it uses the barrier); sums and unit are shared memory.
    template <int THREADS, class A>
    static __device__ __forceinline__ Place place(const A &a, int each, int min_steps, long long (&sums)[THREADS / 32],
                                                  int (&unit)[4]) {
        const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
        // the threads' numbers before this one's, and all of them
        auto scan = [&](long long own, long long &total) {
            long long before = own;
#pragma unroll
            for (int d = 1; d < 32; d *= 2) {
                const long long x = __shfl_up_sync(0xffffffffu, before, d);
                if (lane >= d) before += x;
            }
            __syncthreads();
            if (lane == 31) sums[warp] = before;
            __syncthreads();
            total = 0;
#pragma unroll 1
            for (int w = 0; w < THREADS / 32; w++) {
                if (w == warp) before += total;
                total += sums[w];
            }
            return before - own;
        };
        Place p;
        p.pos = p.end = 0;
        if ((long long)a.max_rows * each > 8 * R && a.seqs <= 16) {
            // few sequences of many row tiles: all threads share each sequence's tiles
            long long total = 0;
            for (int turn = 0; turn < 2; turn++) {  // the sum of all, then this block's place in it
                long long at = 0;
                for (int q = 0; q < a.seqs; q++) {
                    const KaRows s = ka_rows(a, q);
                    if (!s.ok && tid == 0) *reinterpret_cast<volatile int *>(a.err) = 1;
                    const int tiles = s.ok ? (s.n * each + R - 1) / R : 0, share = (tiles + THREADS - 1) / THREADS;
                    const int lo = min(tiles, tid * share), hi = min(tiles, lo + share);
                    long long own = 0, all;
                    for (int rt = lo; rt < hi; rt++) own += (long long)span(a, s, each, rt).steps * a.c.heads;
                    const long long before = at + scan(own, all);
                    if (turn && p.end && p.pos >= before && p.pos < before + own) {
                        long long x = before;
                        for (int rt = lo;; rt++) {
                            const int steps = span(a, s, each, rt).steps;
                            if (p.pos < x + (long long)steps * a.c.heads) {
                                unit[0] = q, unit[1] = rt, unit[2] = (int)ka_div(p.pos - x, steps);
                                unit[3] = (int)(p.pos - x - (long long)unit[2] * steps);
                                break;
                            }
                            x += (long long)steps * a.c.heads;
                        }
                    }
                    at += all;
                }
                if (!turn) total = at, cut(p, total, min_steps);
            }
        } else {
            const int share = (a.seqs + THREADS - 1) / THREADS, seq_lo = min(a.seqs, tid * share), seq_hi = min(a.seqs, seq_lo + share);
            long long own = 0, total;
            for (int q = seq_lo; q < seq_hi; q++) own += seq_steps(a, q, each) * a.c.heads;
            const long long before = scan(own, total);
            cut(p, total, min_steps);
            if (p.end && own && p.pos >= before && p.pos < before + own) {  // the thread whose sequences hold the first step
                long long at = before;
                for (int q = seq_lo; q < seq_hi; q++) {
                    const long long n = seq_steps(a, q, each) * a.c.heads;
                    if (p.pos >= at + n) {
                        at += n;
                        continue;
                    }
                    const KaRows r = ka_rows(a, q);
                    for (int rt = 0;; rt++) {
                        const int steps = span(a, r, each, rt).steps;
                        if (p.pos >= at + (long long)steps * a.c.heads) {
                            at += (long long)steps * a.c.heads;
                            continue;
                        }
                        unit[0] = q, unit[1] = rt, unit[2] = (int)ka_div(p.pos - at, steps);
                        unit[3] = (int)(p.pos - at - (long long)unit[2] * steps);
                        break;
                    }
                    break;
                }
            }
        }
        __syncthreads();
        p.seq = unit[0], p.rt = unit[1], p.head = unit[2], p.skip = unit[3];
        return p;
    }
    static __device__ __forceinline__ void cut(Place &p, long long total, int min_steps) {
        p.total = total, p.blocks = min((long long)gridDim.x, ka_div(total + min_steps - 1, min_steps));
        if (blockIdx.x < p.blocks) p.pos = ka_div(total * blockIdx.x, p.blocks), p.end = ka_div(total * (blockIdx.x + 1), p.blocks);
    }
    // On to the next unit, `piece` steps on.
    template <class A>
    static __device__ __forceinline__ void next(Place &p, const A &a, int each, int n, int piece) {
        p.pos += piece, p.skip = 0;
        if (++p.head < a.c.heads) return;
        p.head = 0;
        if ((++p.rt) * R < n * each) return;
        p.rt = 0;
        while (++p.seq < a.seqs) {
            const KaRows s = ka_rows(a, p.seq);
            if (s.ok && s.n) break;
        }
    }
    // The blocks [first, first + count) that share the unit whose first step is u0.
    static __device__ __forceinline__ int2 sharers(const Place &p, long long u0, int steps) {
        const int b0 = (int)ka_div((u0 + 1) * p.blocks - 1, p.total), b1 = (int)ka_div((u0 + steps) * p.blocks - 1, p.total);
        return make_int2(b0, b1 - b0 + 1);
    }
    // Where block b's part of a unit lies: a part that begins the unit in its second slot, one that goes on in its first.
    static __device__ __forceinline__ size_t slot(int b, bool begins) { return 2 * (size_t)b + begins; }
};

}  // namespace tcu

// topk_logprob.hip — the k largest log-probabilities of each row of bf16 logits, in one pass over them, for gfx950.
//
//   ids = the k largest logits of a row in falling order (equal logits: the lower id first), logp = logit / temperature - lse,
//   lse = log sum_v exp(logit_v / temperature)
// Bound: HBM, 2 V bytes per row read once (MI355X, 2048 rows of V = 152 064, k = 64: 134 us = 4.65 TB/s of the 6.8 that a read alone reaches, the rest
// being the vector instructions of comparing, raising and summing 16-bit values; one row, k = 20: 8 us and 6 us more to join its slices).
//
// One workgroup walks a row (or a slice of it) in segments.  Every thread keeps the largest value it has met; the k-th largest of these
// per-thread maxima is reached by at least k values, so whatever lies below it can be dropped: this threshold rises as the maxima grow and
// after the first segment only a few hundred of a row's 150 000 values pass it and go into a candidate list in LDS.  A list that would
// overflow (values that rise along the row) is cut back to its k largest first, so the result does not depend on the order of the
// values.  The walk compares floats; candidates carry a 64-bit key of the value's order as a whole number (-0 equals +0) over the falling id,
// which makes every key different and ties go to the lower id.  NaN passes no comparison; it makes the row's lse NaN, and such a row is
// answered without its candidates.  The exponential sum runs over the same registers.
#include "common.h"
#include <algorithm>

#define TK_LOG2E 1.4426950408889634f
#define TK_LN2 0.6931471805599453f
#define TK_CHUNK(NT) ((NT) * 8)                  // values per workgroup of NT threads and load
#define TK_SEG 4                               // loads per segment: the threshold is renewed once per segment
#define TK_MAX_K 256
#define TK_CAP(NT) (TK_CHUNK(NT) + TK_MAX_K)     // candidates: what is kept plus one whole chunk (+ the values in front of and behind the granules)
#define TK_NONE (-32640)                       // the order of -inf: every value passes

__device__ __forceinline__ int tk_order(uint16_t b) {                    // bf16 bits -> signed order, -0 = +0
    const int mag = b & 0x7fff;
    return (b & 0x8000) ? -mag : mag;
}
__device__ __forceinline__ float tk_value(int order) {
    const int mag = order < 0 ? -order : order;
    return bf2f((uint16_t)(mag | (order < 0 ? 0x8000 : 0)));
}
__device__ __forceinline__ uint64_t tk_key(int order, uint32_t id) { return ((uint64_t)(uint32_t)(order + 32768) << 32) | (0xffffffffu - id); }

#define TK_BINS 1024                           // orders told apart below the largest candidate when the list is ranked; the last bin holds all that lie lower

template <int NT> struct TkShared {
    uint64_t cand[TK_CAP(NT) + 16];
    uint64_t best[2 * TK_MAX_K];
    int maxima[NT];
    float2 red[NT / 64];
    int count, thr, scan[NT / 64];
    int bins[TK_BINS];
    uint4 kept[NT];                                                      // granules that hold a value above the threshold of their time ...
    int kept_at[NT], kept_n;                                             // ... and their places in the slice
};

// number of threads of the workgroup for which `p` holds, summed with `n` per thread; a barrier on both sides
template <int NT> __device__ __forceinline__ int tk_block_sum(TkShared<NT>& sh, int n) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.scan[threadIdx.x >> 6] = n;
    __syncthreads();
    int s = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) s += sh.scan[i];
    return s;
}

// cut the list back to its k largest keys (n > k of them): the k-th largest key by bisection over its bits (every key is different).  Rare,
// so the keys are read from LDS in every step instead of taking registers from the walk.
template <int NT> __device__ __forceinline__ void tk_cut(TkShared<NT>& sh, int n, int k) {
    uint64_t kth = 0;
#pragma unroll 1
    for (int b = 47; b >= 0; --b) {                                      // largest value that at least k keys reach
        const uint64_t t = kth | (1ull << b);
        int c = 0;
#pragma unroll 1
        for (int j = threadIdx.x; j < n; j += NT) c += sh.cand[j] >= t ? 1 : 0;
        if (tk_block_sum(sh, c) >= k) kth = t;
    }
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
#pragma unroll 1
    for (int j = threadIdx.x; j < n; j += NT) if (sh.cand[j] >= kth) sh.best[atomicAdd(&sh.count, 1)] = sh.cand[j];
    __syncthreads();
    for (int j = threadIdx.x; j < k; j += NT) sh.cand[j] = sh.best[j];
    __syncthreads();
}

// the list's k largest in falling order -> best[0 .. k), or all of them where n < k.  Counts per order value first: only what is at least the k-th
// largest value is ranked (k and its ties) instead of all n candidates against each other.
template <int NT> __device__ __forceinline__ void tk_rank(TkShared<NT>& sh, int n, int k) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (n > 2 * k && n > 128) {
        int most = 0;                                                    // the largest order (+32768)
        for (int j = threadIdx.x; j < n; j += NT) most = max(most, (int)(sh.cand[j] >> 32));
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) most = max(most, __shfl_xor(most, o, 64));
        if (lane == 0) sh.scan[wave] = most;
        for (int j = threadIdx.x; j < TK_BINS; j += NT) sh.bins[j] = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NT / 64; ++i) most = max(most, sh.scan[i]);
        for (int j = threadIdx.x; j < n; j += NT) atomicAdd(&sh.bins[min(most - (int)(sh.cand[j] >> 32), TK_BINS - 1)], 1);
        __syncthreads();
        // bin 0 holds the largest value: the first bin up to which at least k candidates lie
        constexpr int PER = TK_BINS / NT;                                // bins per thread
        int c[PER], mine = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) { c[i] = sh.bins[PER * threadIdx.x + i]; mine += c[i]; }
        int x = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) { const int y = __shfl_up(x, o, 64); x += lane >= o ? y : 0; }
        if (lane == 63) sh.scan[wave] = x;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NT / 64; ++i) x += i < wave ? sh.scan[i] : 0;
        if (x >= k && x - mine < k) {
            int upto = x - mine;
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (upto < k) { upto += c[i]; sh.maxima[0] = PER * threadIdx.x + i; sh.maxima[1] = upto; }
        }
        __syncthreads();
        const int last = sh.maxima[0], left = sh.maxima[1];
        if (left <= 2 * TK_MAX_K) {
            if (threadIdx.x == 0) sh.count = 0;
            __syncthreads();
            for (int j = threadIdx.x; j < n; j += NT)
                if (min(most - (int)(sh.cand[j] >> 32), TK_BINS - 1) <= last) sh.best[atomicAdd(&sh.count, 1)] = sh.cand[j];   // clamped as counted: `left` of them
            __syncthreads();
            for (int j = threadIdx.x; j < left; j += NT) sh.cand[j] = sh.best[j];
            n = left;
        } else {                                                         // many equal values: the lowest ids among them, by bisection
            tk_cut(sh, n, k);
            n = k;
        }
        __syncthreads();
    }
    for (int j = threadIdx.x; j < n; j += NT) {
        const uint64_t key = sh.cand[j];
        int rank = 0;
#pragma unroll 4
        for (int i = 0; i < n; ++i) rank += sh.cand[i] > key ? 1 : 0;
        if (rank < k) sh.best[rank] = key;
    }
    __syncthreads();
}

// one instruction, without the compiler's quieting of its inputs (a NaN passes no comparison either way)
__device__ __forceinline__ float tk_max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
__device__ __forceinline__ float2 tk_join(float2 a, float2 b) {          // (max, sum) in base 2
    const float m = fmaxf(a.x, b.x);
    if (m == -INFINITY) return make_float2(m, a.y + b.y);
    // (an equal maximum counts 1 by comparison: the difference may be a fused one, of the product that x came from)
    return make_float2(m, (a.x == m ? a.y : a.y * __builtin_amdgcn_exp2f(a.x - m)) + (b.x == m ? b.y : b.y * __builtin_amdgcn_exp2f(b.x - m)));
}
template <int NT> __device__ __forceinline__ float2 tk_block_join(TkShared<NT>& sh, float2 v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = tk_join(v, make_float2(__shfl_xor(v.x, o, 64), __shfl_xor(v.y, o, 64)));
    if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh.red[0];
#pragma unroll
    for (int i = 1; i < NT / 64; ++i) v = tk_join(v, sh.red[i]);
    return v;
}
template <int NT> __device__ __forceinline__ void tk_write(TkShared<NT>& sh, int k, float2 ms, float inv_temp, int32_t* __restrict__ ids, float* __restrict__ logp,
                                         float* __restrict__ lse) {
    const float l = ms.x < INFINITY ? (ms.x + log2f(ms.y)) * TK_LN2 : NAN;           // +inf, given or beyond fp32
    if (threadIdx.x == 0) *lse = l;
    for (int j = threadIdx.x; j < k; j += NT) {
        const uint64_t key = l == l ? sh.best[j] : 0;
        ids[j] = l == l ? (int32_t)(0xffffffffu - (uint32_t)key) : j;
        logp[j] = tk_value((int)(key >> 32) - 32768) * inv_temp - l;
    }
}

// grid (slices, T).  One slice: the row's result.  More: slice s leaves its (at most k) best keys, padded with 0, in keys[row][s][k] and its
// (max, sum) in stats[row][s]; topk_join_kernel finishes the row.
template <int NT>
__global__ __launch_bounds__(NT, 4) void topk_row_kernel(const uint16_t* __restrict__ logits, int64_t ldl, int V, int k, int slice_len, float inv_temp,
                                                             int32_t* __restrict__ ids, float* __restrict__ logp, float* __restrict__ lse,
                                                             uint64_t* __restrict__ keys, float2* __restrict__ stats) {
    __shared__ TkShared<NT> sh;
    const int row = blockIdx.y, slices = gridDim.x, lane = threadIdx.x & 63;
    const uint16_t* x = logits + (int64_t)row * ldl;
    const int beg = blockIdx.x * slice_len, end = min(V, beg + slice_len), n = end - beg;
    const int want = min(k, n);
    const float sc = inv_temp * TK_LOG2E;
    // whole 16-byte granules in the middle; the (at most 7) values in front of them and behind them go one to a thread
    const int front = min(n, (int)(((16 - ((uintptr_t)(x + beg) & 15)) & 15) >> 1)), granules = (n - front) >> 3;
    const int back = n - front - granules * 8;
    const uint4* body = reinterpret_cast<const uint4*>(x + beg + front);
    if (threadIdx.x == 0) { sh.count = 0; sh.thr = TK_NONE; sh.kept_n = 0; }
    int used = 0;                                                        // granules kept, at most; the same for every thread
    int thr = TK_NONE;                                                   // values of a lower order are out
    float top = -INFINITY, m = -INFINITY, s = 0.f;                       // this thread's largest so far; base-2 maximum and sum
    // a value's term is 2^(f by - sub), sub = m (0 while that is -inf).  From |m| = 2^30 on m's own rounding may be more than an exponent holds: unscaled, by
    // exact differences, a value counts at most 1 and the largest 1, and the logarithm of the whole row's sum is below half a step of m.
    float by = sc, sub = 0.f;
    auto measure = [&](float f) {                                        // f: the value whose product m is
        const bool far = fabsf(m) >= 0x1p30f;
        by = far ? 1.f : sc;
        sub = far ? f : m;
    };
    bool any = false;                                                    // this thread has met a value
    __syncthreads();
    auto single = [&](int e) {                                           // one value outside the granules; the list has room for these
        const float f = bf2f(x[beg + e]);
        any = true;
        top = fmaxf(top, f);
        if (f >= tk_value(thr)) sh.cand[atomicAdd(&sh.count, 1)] = tk_key(tk_order(x[beg + e]), (uint32_t)(beg + e));
        const float2 v = tk_join(make_float2(m, s), make_float2(f * sc, f == -INFINITY ? 0.f : f == f ? 1.f : f));
        m = v.x; s = v.y;
        if (m > -INFINITY) measure(f);                                   // (in front of the granules: this thread's first value; behind them nothing follows)
    };
    if ((int)threadIdx.x < front) single(threadIdx.x);
    // the values of one granule per thread (where `here`) that pass the threshold -> candidates; ids above those of all candidates so far
    auto take = [&](const uint4& w, int g, bool here) {
        float f[8];
        unpack8(w, f);
        float ge = tk_value(thr);
        int mine = 0;
        if (here)
#pragma unroll
            for (int j = 0; j < 8; ++j) mine += f[j] >= ge ? 1 : 0;
        const int now = sh.count;                                        // stable: barriers in front of and behind every append
        if (now + tk_block_sum(sh, mine) > TK_CAP(NT)) {
            // now > TK_MAX_K >= want here (the granules hold <= TK_CHUNK): the k largest survive, the smallest of them is the new threshold
            tk_cut(sh, now, want);
            int lo = 0x7fffffff;
            for (int j = threadIdx.x; j < want; j += NT) lo = min(lo, (int)(sh.cand[j] >> 32) - 32768);
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) lo = min(lo, __shfl_xor(lo, o, 64));
            if (lane == 0) sh.scan[threadIdx.x >> 6] = lo;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < NT / 64; ++i) lo = min(lo, sh.scan[i]);
            thr = max(thr, lo + 1);                                      // an equal value further on has a higher id: out
            ge = tk_value(thr);
            __syncthreads();
        }
        if (here)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (f[j] >= ge) sh.cand[atomicAdd(&sh.count, 1)] = tk_key(tk_order((uint16_t)(__float_as_uint(f[j]) >> 16)), (uint32_t)(beg + front + g * 8 + j));
        __syncthreads();
    };
    // the kept granules -> candidates; called behind a barrier that follows the last append to them
    auto flush = [&]() {
        const int n = sh.kept_n;
        const bool here = (int)threadIdx.x < n;
        take(here ? sh.kept[threadIdx.x] : make_uint4(0, 0, 0, 0), here ? sh.kept_at[threadIdx.x] : 0, here);
        if (threadIdx.x == 0) sh.kept_n = 0;
        __syncthreads();
    };
    uint4 r[TK_SEG], ahead[TK_SEG];
    auto fetch = [&](int g0) {                                           // unconditional loads (the waits can be counted): past the end the last granule
#pragma unroll
        for (int c = 0; c < TK_SEG; ++c) ahead[c] = body[min(g0 + c * NT + (int)threadIdx.x, granules - 1)];
    };
    if (granules) fetch(0);
    for (int g0 = 0, seg = 0; g0 < granules; g0 += NT * TK_SEG, ++seg) {
#pragma unroll
        for (int c = 0; c < TK_SEG; ++c) r[c] = ahead[c];
        fetch(g0 + NT * TK_SEG);                                 // the next segment flies while this one is worked on
        if (g0 + NT * TK_SEG > granules) {                       // no granule: -inf adds nothing to the sum
#pragma unroll
            for (int c = 0; c < TK_SEG; ++c)
                if (g0 + c * NT + (int)threadIdx.x >= granules) r[c] = make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
        }
        float cmax[TK_SEG], most = -INFINITY;
#pragma unroll
        for (int c = 0; c < TK_SEG; ++c) {
            float f[8];
            unpack8(r[c], f);
            cmax[c] = tk_max3(tk_max3(tk_max3(f[0], f[1], f[2]), f[3], f[4]), f[5], fmaxf(f[6], f[7]));
            most = fmaxf(most, cmax[c]);
            // the exponential sum, base 2
            const float vm = cmax[c] * sc;                               // sc > 0
            if (vm > m) {
                s *= __builtin_amdgcn_exp2f(m - vm);
                m = vm;
                measure(cmax[c]);
            }
            float a = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j) a += __builtin_amdgcn_exp2f(fmaf(f[j], by, -sub));
            s += a;
        }
        top = fmaxf(top, most);
        any = any || g0 + (int)threadIdx.x < granules;
        // the threshold: the k-th largest per-thread maximum (fewer than k threads with values: none yet), renewed in segments 0, 1, 3, 7, ...: by then the
        // maxima have seen twice as many values.  One wave bisects the 16-bit order.
        if ((seg & (seg + 1)) == 0) {
            sh.maxima[threadIdx.x] = any ? tk_order((uint16_t)(__float_as_uint(top) >> 16)) : TK_NONE - 1;
            __syncthreads();
            if (threadIdx.x < 64) {
                int mine[NT / 64];
#pragma unroll
                for (int i = 0; i < NT / 64; ++i) mine[i] = sh.maxima[lane + i * 64] - TK_NONE;     // -1: no value
                int c0 = 0, lo = 0x7fffffff, hi = -1;
#pragma unroll
                for (int i = 0; i < NT / 64; ++i) {
                    c0 += __popcll(__ballot(mine[i] >= 0));
                    lo = min(lo, mine[i]); hi = max(hi, mine[i]);
                }
                if (c0 >= want) {
#pragma unroll
                    for (int o = 32; o > 0; o >>= 1) { lo = min(lo, __shfl_xor(lo, o, 64)); hi = max(hi, __shfl_xor(hi, o, 64)); }
                    lo = __builtin_amdgcn_readfirstlane(max(lo, 0)); hi = __builtin_amdgcn_readfirstlane(hi);
#pragma unroll 1
                    while (lo < hi) {                                    // the largest value that at least `want` maxima reach is in [lo, hi]
                        const int mid = (lo + hi + 1) >> 1;
                        int c = 0;
#pragma unroll
                        for (int i = 0; i < NT / 64; ++i) c += __popcll(__ballot(mine[i] >= mid));
                        if (c >= want) lo = mid; else hi = mid - 1;
                    }
                    if (lane == 0) sh.thr = lo + TK_NONE;                // values equal to the k-th maximum stay
                }
            }
            used = sh.kept_n;                                            // (nothing is appended between these two barriers)
            __syncthreads();
            thr = max(thr, sh.thr);
        }
        float ge = tk_value(thr);
        const int hits = __syncthreads_count(most >= ge && g0 + (int)threadIdx.x < granules);
        if (!hits) continue;
        if (used + TK_SEG * hits > NT) { flush(); ge = tk_value(thr); used = 0; }
        if (TK_SEG * hits <= NT) {                                       // the usual case: no barrier of its own
            used += TK_SEG * hits;
#pragma unroll
            for (int c = 0; c < TK_SEG; ++c) {
                const int g = g0 + c * NT + (int)threadIdx.x;
                if (cmax[c] >= ge && g < granules) {
                    const int at = atomicAdd(&sh.kept_n, 1);
                    sh.kept[at] = r[c];
                    sh.kept_at[at] = g;
                }
            }
            continue;
        }
#pragma unroll 1
        for (int c = 0; c < TK_SEG; ++c) {                               // load by load: ids rise from one to the next
            const int g = g0 + c * NT + (int)threadIdx.x;
            const bool here = g < granules;
            const uint4 w = body[min(g, granules - 1)];                  // once more from memory: a rare path must not hold the segment's registers
            take(w, g, here);
        }
    }
    __syncthreads();
    flush();
    if ((int)threadIdx.x < back) single(front + granules * 8 + threadIdx.x);
    const float2 ms = tk_block_join(sh, make_float2(m, s));
    __syncthreads();
    const int got = min(want, sh.count);                                 // fewer than want: a row with NaN
    tk_rank(sh, sh.count, want);
    if (slices == 1) {
        tk_write(sh, k, ms, inv_temp, ids + (int64_t)row * k, logp + (int64_t)row * k, lse + row);
    } else {
        uint64_t* kp = keys + ((int64_t)row * slices + blockIdx.x) * k;
        for (int j = threadIdx.x; j < k; j += NT) kp[j] = j < got ? sh.best[j] : 0;
        if (threadIdx.x == 0) stats[(int64_t)row * slices + blockIdx.x] = ms;
    }
}

// One workgroup per row: the best of slices * k <= TK_CAP keys, each slice's in falling order (0 where it has fewer than k values).  The
// ceil(k / slices)-th keys of the slices and the k-th key of any slice bound the row's k-th from below: only what reaches both bounds is ranked.
template <int NT>
__global__ __launch_bounds__(NT) void topk_join_kernel(const uint64_t* __restrict__ keys, const float2* __restrict__ stats, int slices, int k,
                                                              float inv_temp, int32_t* __restrict__ ids, float* __restrict__ logp, float* __restrict__ lse) {
    __shared__ TkShared<NT> sh;
    __shared__ uint64_t floor_of[NT / 64];
    const int row = blockIdx.x, lane = threadIdx.x & 63;
    const uint64_t* kp = keys + (int64_t)row * slices * k;
    if (threadIdx.x == 0) sh.count = 0;
    uint64_t lo = ~0ull, hi = 0;                                         // min over slices of the ceil(k/slices)-th key, max of the k-th
    for (int j = threadIdx.x; j < slices; j += NT) {
        lo = min(lo, kp[(int64_t)j * k + (k + slices - 1) / slices - 1]);
        hi = max(hi, kp[(int64_t)j * k + k - 1]);
    }
    const float2 ms = tk_block_join(sh, threadIdx.x < (unsigned)slices ? stats[(int64_t)row * slices + threadIdx.x] : make_float2(-INFINITY, 0.f));
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        lo = min(lo, (uint64_t)__shfl_xor((unsigned long long)lo, o, 64));
        hi = max(hi, (uint64_t)__shfl_xor((unsigned long long)hi, o, 64));
    }
    if (lane == 0) { floor_of[threadIdx.x >> 6] = lo; sh.best[threadIdx.x >> 6] = hi; }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) { lo = min(lo, floor_of[i]); hi = max(hi, sh.best[i]); }
    const uint64_t least = max(max(lo, hi), (uint64_t)1);
    __syncthreads();
    for (int j = threadIdx.x; j < slices * k; j += NT) {
        const uint64_t key = kp[j];
        if (key >= least) sh.cand[atomicAdd(&sh.count, 1)] = key;
    }
    __syncthreads();
    tk_rank(sh, sh.count, k);
    tk_write(sh, k, ms, inv_temp, ids + (int64_t)row * k, logp + (int64_t)row * k, lse + row);
}

// Threads per workgroup: one maximum per thread bounds the k-th largest value from below, so k is at most about half of them (with k = NT the
// bound is the least of the maxima); otherwise the smaller workgroup, of which more run side by side (MI355X, V = 152 064, 256 / 512 threads:
// 2048 rows, k = 128 174 / 192 us; 256 rows, k = 128 56 / 46 us).
static int topk_threads(int T, int k) { return k <= 96 || (k <= 128 && T >= 4 * st_num_cus()) ? 256 : 512; }

// Slices of a row: whole rounds of the workgroups that fit (1024 threads per CU), each costing its slice plus about 32 K values' time of threshold,
// ranking and launch; a slice keeps at least a load per thread, the slices' keys fit the join's list.
static int topk_slices(int T, int V, int k) {
    const int nt = topk_threads(T, k), slots = 1024 / nt * st_num_cus(), most = std::max(1, std::min({TK_CAP(512) / k, st_cdiv(V, TK_CHUNK(nt)), 64}));
    int best = 1;
    int64_t cost = INT64_MAX;
    for (int s = 1; s <= most; ++s) {
        const int64_t c = (int64_t)st_cdiv((int64_t)T * s, slots) * (st_cdiv(V, s) + 32768) + (s > 1 ? 24576 + 256 * s : 0);
        if (c < cost) { cost = c; best = s; }
    }
    return best;
}

extern "C" {

int st_topk_logprob_workspace_bytes(int T, int V, int k, int64_t* bytes_host, st_stream_t stream) {
    (void)stream;
    if (T < 0 || V <= 0 || k <= 0 || k > V || k > TK_MAX_K || !bytes_host) return ST_EINVAL;
    const int64_t s = topk_slices(T, V, k);
    *bytes_host = s > 1 ? (int64_t)T * s * k * 8 + (int64_t)T * s * 8 : 0;
    return 0;
}

int st_topk_logprob(const st_bf16* logits, int64_t ldl, int k, float inv_temperature, int32_t* ids, float* logp, float* lse, void* workspace,
                    int64_t workspace_bytes, int T, int V, st_stream_t stream) {
    if (T < 0 || V <= 0 || k <= 0 || k > V || k > TK_MAX_K || !(inv_temperature > 0.f && inv_temperature * TK_LOG2E < INFINITY)) return ST_EINVAL;
    if (T == 0) return 0;
    if (!logits || ldl < V || !ids || !logp || !lse || T > 0x7fffffff / TK_MAX_K || (((uintptr_t)logits) & 1)) return ST_EINVAL;
    hipStream_t s = (hipStream_t)stream;
    const int slices = topk_slices(T, V, k);
    const int64_t need = slices > 1 ? (int64_t)T * slices * k * 8 + (int64_t)T * slices * 8 : 0;
    if (need && (!workspace || workspace_bytes < need || (((uintptr_t)workspace) & 7))) return ST_EINVAL;
    const int len = st_cdiv(V, slices);                                  // (every slice is non-empty: checked below)
    const int used = st_cdiv(V, len);
    uint64_t* keys = (uint64_t*)workspace;
    float2* stats = (float2*)(keys + (int64_t)T * used * k);
    for (int t0 = 0; t0 < T; t0 += 32768) {                              // grid.y holds 65535
        const int nt = std::min(32768, T - t0);
        auto go = [&](auto kern, int threads) {
            hipLaunchKernelGGL(kern, dim3(used, nt), dim3(threads), 0, s, logits + (int64_t)t0 * ldl, ldl, V, k, len, inv_temperature, ids + (int64_t)t0 * k,
                               logp + (int64_t)t0 * k, lse + t0, slices > 1 ? keys + (int64_t)t0 * used * k : nullptr,
                               slices > 1 ? stats + (int64_t)t0 * used : nullptr);
        };
        if (topk_threads(T, k) == 256) go(topk_row_kernel<256>, 256); else go(topk_row_kernel<512>, 512);
        ST_CHECK_LAUNCH();
    }
    if (used > 1) {
        hipLaunchKernelGGL(topk_join_kernel<512>, dim3(T), dim3(512), 0, s, keys, stats, used, k, inv_temperature, ids, logp, lse);
        ST_CHECK_LAUNCH();
    }
    return 0;
}

}  // extern "C"

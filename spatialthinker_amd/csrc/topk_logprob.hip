// topk_logprob.hip — the k largest log-probabilities of each row of bf16 logits, in one pass over them, for gfx950.
//
//   ids = the k largest logits of a row in falling order (equal logits: the lower id first), logp = logit / temperature - lse,
//   lse = log sum_v exp(logit_v / temperature)
// Bound: HBM, 2 V bytes per row read once.
//
// One workgroup walks a row (or a slice of it) in segments.  Every thread keeps the largest value it has met; the k-th largest of these
// per-thread maxima is reached by at least k values, so whatever lies below it can be dropped: this threshold rises as the maxima grow and
// after the first segment only a few hundred of a row's 150 000 values pass it and go into a candidate list in LDS.  A list that would
// overflow (values that rise along the row) is cut back to its k largest first, so the result does not depend on the order of the
// values.  Values are ordered as whole numbers: bf16 bits mapped to a signed 16-bit order (-0 equals +0, NaN by its bits beyond the
// infinities), the id below them in the 64-bit key, which makes every key different and ties go to the lower id.
// The exponential sum runs over the same registers.
#include "common.h"
#include <algorithm>

#define TK_LOG2E 1.4426950408889634f
#define TK_LN2 0.6931471805599453f
#define TK_THREADS 512
#define TK_CHUNK (TK_THREADS * 8)              // values per workgroup and load
#define TK_SEG 4                               // loads per segment: the threshold is renewed once per segment
#define TK_MAX_K 256
#define TK_CAP (TK_CHUNK + TK_MAX_K)           // candidates: what is kept plus one whole chunk (+ the values in front of and behind the granules)
#define TK_NONE (-32769)                       // below every value's order

__device__ __forceinline__ int tk_order(uint16_t b) {                    // bf16 bits -> signed order, -0 = +0
    const int mag = b & 0x7fff;
    return (b & 0x8000) ? -mag : mag;
}
typedef short tk_short2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ tk_short2 tk_order2(uint32_t w) {             // the same for two values at once (packed 16-bit integer instructions)
    const tk_short2 sign = __builtin_bit_cast(tk_short2, w) >> (short)15, mag = __builtin_bit_cast(tk_short2, w & 0x7fff7fffu);
    return (mag ^ sign) - sign;
}
__device__ __forceinline__ float tk_value(int order) {
    const int mag = order < 0 ? -order : order;
    return bf2f((uint16_t)(mag | (order < 0 ? 0x8000 : 0)));
}
__device__ __forceinline__ uint64_t tk_key(int order, uint32_t id) { return ((uint64_t)(uint32_t)(order + 32768) << 32) | (0xffffffffu - id); }

struct TkShared {
    uint64_t cand[TK_CAP + 16];
    uint64_t best[TK_MAX_K];
    int maxima[TK_THREADS];
    float2 red[TK_THREADS / 64];
    int count, thr, scan[TK_THREADS / 64];
};

// number of threads of the workgroup for which `p` holds, summed with `n` per thread; a barrier on both sides
__device__ __forceinline__ int tk_block_sum(TkShared& sh, int n) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.scan[threadIdx.x >> 6] = n;
    __syncthreads();
    int s = 0;
#pragma unroll
    for (int i = 0; i < TK_THREADS / 64; ++i) s += sh.scan[i];
    return s;
}

// cut the list back to its k largest keys (n > k of them): the k-th largest key by bisection over its bits (every key is different).  Rare,
// so the keys are read from LDS in every step instead of taking registers from the walk.
__device__ __forceinline__ void tk_cut(TkShared& sh, int n, int k) {
    uint64_t kth = 0;
#pragma unroll 1
    for (int b = 47; b >= 0; --b) {                                      // largest value that at least k keys reach
        const uint64_t t = kth | (1ull << b);
        int c = 0;
#pragma unroll 1
        for (int j = threadIdx.x; j < n; j += TK_THREADS) c += sh.cand[j] >= t ? 1 : 0;
        if (tk_block_sum(sh, c) >= k) kth = t;
    }
    __syncthreads();
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
#pragma unroll 1
    for (int j = threadIdx.x; j < n; j += TK_THREADS) if (sh.cand[j] >= kth) sh.best[atomicAdd(&sh.count, 1)] = sh.cand[j];
    __syncthreads();
    if (threadIdx.x < k) sh.cand[threadIdx.x] = sh.best[threadIdx.x];    // k <= TK_MAX_K < TK_THREADS
    __syncthreads();
}

// the list's k largest in falling order -> best[0 .. k): n >= k
__device__ __forceinline__ void tk_rank(TkShared& sh, int n, int k) {
    if (n > 2 * TK_THREADS) { tk_cut(sh, n, k); n = k; }
    for (int j = threadIdx.x; j < n; j += TK_THREADS) {
        const uint64_t key = sh.cand[j];
        int rank = 0;
        for (int i = 0; i < n; ++i) rank += sh.cand[i] > key ? 1 : 0;
        if (rank < k) sh.best[rank] = key;
    }
    __syncthreads();
}

__device__ __forceinline__ float2 tk_join(float2 a, float2 b) {          // (max, sum) in base 2
    const float m = fmaxf(a.x, b.x);
    if (m == -INFINITY) return make_float2(m, a.y + b.y);
    return make_float2(m, a.y * __builtin_amdgcn_exp2f(a.x - m) + b.y * __builtin_amdgcn_exp2f(b.x - m));
}
__device__ __forceinline__ float2 tk_block_join(TkShared& sh, float2 v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = tk_join(v, make_float2(__shfl_xor(v.x, o, 64), __shfl_xor(v.y, o, 64)));
    if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = sh.red[0];
#pragma unroll
    for (int i = 1; i < TK_THREADS / 64; ++i) v = tk_join(v, sh.red[i]);
    return v;
}
__device__ __forceinline__ void tk_write(TkShared& sh, int k, float2 ms, float inv_temp, int32_t* __restrict__ ids, float* __restrict__ logp,
                                         float* __restrict__ lse) {
    const float l = (ms.x + log2f(ms.y)) * TK_LN2;
    if (threadIdx.x == 0) *lse = l;
    for (int j = threadIdx.x; j < k; j += TK_THREADS) {
        const uint64_t key = sh.best[j];
        ids[j] = (int32_t)(0xffffffffu - (uint32_t)key);
        logp[j] = tk_value((int)(key >> 32) - 32768) * inv_temp - l;
    }
}

// grid (slices, T).  One slice: the row's result.  More: slice s leaves its (at most k) best keys, padded with 0, in keys[row][s][k] and its
// (max, sum) in stats[row][s]; topk_join_kernel finishes the row.
__global__ __launch_bounds__(TK_THREADS, 4) void topk_row_kernel(const uint16_t* __restrict__ logits, int64_t ldl, int V, int k, int slice_len, float inv_temp,
                                                             int32_t* __restrict__ ids, float* __restrict__ logp, float* __restrict__ lse,
                                                             uint64_t* __restrict__ keys, float2* __restrict__ stats) {
    __shared__ TkShared sh;
    const int row = blockIdx.y, slices = gridDim.x, lane = threadIdx.x & 63;
    const uint16_t* x = logits + (int64_t)row * ldl;
    const int beg = blockIdx.x * slice_len, end = min(V, beg + slice_len), n = end - beg;
    const int want = min(k, n);
    const float sc = inv_temp * TK_LOG2E;
    // whole 16-byte granules in the middle; the (at most 7) values in front of them and behind them go one to a thread
    const int front = min(n, (int)(((16 - ((uintptr_t)(x + beg) & 15)) & 15) >> 1)), granules = (n - front) >> 3;
    const int back = n - front - granules * 8;
    const uint4* body = reinterpret_cast<const uint4*>(x + beg + front);
    if (threadIdx.x == 0) { sh.count = 0; sh.thr = TK_NONE; }
    int thr = TK_NONE, top = TK_NONE;                                    // values <= thr are out; this thread's largest so far
    float m = -INFINITY, s = 0.f;
    __syncthreads();
    auto single = [&](int e) {                                           // one value outside the granules; the list has room for these
        const uint16_t b = x[beg + e];
        const int o = tk_order(b);
        top = max(top, o);
        if (o > thr) sh.cand[atomicAdd(&sh.count, 1)] = tk_key(o, (uint32_t)(beg + e));
        const float f = bf2f(b);
        const float2 v = tk_join(make_float2(m, s), make_float2(f * sc, f == -INFINITY ? 0.f : f == f ? 1.f : f));
        m = v.x; s = v.y;
    };
    if ((int)threadIdx.x < front) single(threadIdx.x);
    for (int g0 = 0; g0 < granules; g0 += TK_THREADS * TK_SEG) {
        uint4 r[TK_SEG];
#pragma unroll
        for (int c = 0; c < TK_SEG; ++c) {
            const int g = g0 + c * TK_THREADS + threadIdx.x;
            r[c] = make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);       // no granule: -inf adds nothing to the sum
            if (g < granules) r[c] = body[g];
        }
        int cmax[TK_SEG];
#pragma unroll
        for (int c = 0; c < TK_SEG; ++c) {
            const tk_short2 mx = __builtin_elementwise_max(__builtin_elementwise_max(tk_order2(r[c].x), tk_order2(r[c].y)),
                                                           __builtin_elementwise_max(tk_order2(r[c].z), tk_order2(r[c].w)));
            cmax[c] = g0 + c * TK_THREADS + (int)threadIdx.x < granules ? max((int)mx.x, (int)mx.y) : TK_NONE;
            top = max(top, cmax[c]);
            float f[8];
            unpack8(r[c], f);
            float vm = f[0];
#pragma unroll
            for (int j = 1; j < 8; ++j) vm = fmaxf(vm, f[j]);
            vm *= sc;                                                    // sc > 0
            if (vm > m) { s *= __builtin_amdgcn_exp2f(m - vm); m = vm; }
            const float sub = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int j = 0; j < 8; ++j) s += __builtin_amdgcn_exp2f(fmaf(f[j], sc, -sub));
        }
        // the threshold: the k-th largest per-thread maximum (fewer than k threads with values: none yet).  One wave bisects the 16-bit order.
        sh.maxima[threadIdx.x] = top;
        __syncthreads();
        if (threadIdx.x < 64) {
            int mine[TK_THREADS / 64];
#pragma unroll
            for (int i = 0; i < TK_THREADS / 64; ++i) mine[i] = sh.maxima[lane + i * 64] + 32768;      // -1: no value
            int t = 0, c0 = 0;
#pragma unroll
            for (int i = 0; i < TK_THREADS / 64; ++i) c0 += __popcll(__ballot(mine[i] >= 0));
            if (c0 >= want) {
#pragma unroll 1
                for (int b = 15; b >= 0; --b) {
                    int c = 0;
#pragma unroll
                    for (int i = 0; i < TK_THREADS / 64; ++i) c += __popcll(__ballot(mine[i] >= (t | (1 << b))));
                    if (c >= want) t |= 1 << b;
                }
                if (lane == 0) sh.thr = t - 32768 - 1;                   // values equal to the k-th maximum stay
            }
        }
        __syncthreads();
        thr = max(thr, sh.thr);
#pragma unroll
        for (int c = 0; c < TK_SEG; ++c) {
            const int have = sh.count;                                   // the same for every thread: appended to only behind the next barrier
            if (!__syncthreads_or(cmax[c] > thr)) continue;
            const int e = front + (g0 + c * TK_THREADS + (int)threadIdx.x) * 8;
            const uint32_t w[4] = {r[c].x, r[c].y, r[c].z, r[c].w};
            if (have + TK_CHUNK > TK_CAP) {                              // a whole chunk might not fit: count what would be added
                int mine = 0;
                if (cmax[c] > thr)
#pragma unroll
                    for (int j = 0; j < 8; ++j) mine += tk_order((uint16_t)(w[j >> 1] >> ((j & 1) * 16))) > thr ? 1 : 0;
                if (have + tk_block_sum(sh, mine) > TK_CAP) {
                    // have > TK_MAX_K >= want here (a chunk adds <= TK_CHUNK): the k largest survive, the smallest of them is the new threshold
                    tk_cut(sh, have, want);
                    int lo = 0x7fffffff;
                    for (int j = threadIdx.x; j < want; j += TK_THREADS) lo = min(lo, (int)(sh.cand[j] >> 32) - 32768);
#pragma unroll
                    for (int o = 32; o > 0; o >>= 1) lo = min(lo, __shfl_xor(lo, o, 64));
                    if (lane == 0) sh.scan[threadIdx.x >> 6] = lo;
                    __syncthreads();
#pragma unroll
                    for (int i = 0; i < TK_THREADS / 64; ++i) lo = min(lo, sh.scan[i]);
                    thr = max(thr, lo);                                  // an equal value further on has a higher id: out
                    __syncthreads();
                }
            }
            if (cmax[c] > thr) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int o = tk_order((uint16_t)(w[j >> 1] >> ((j & 1) * 16)));
                    if (o > thr) sh.cand[atomicAdd(&sh.count, 1)] = tk_key(o, (uint32_t)(beg + e + j));
                }
            }
            __syncthreads();
        }
    }
    if ((int)threadIdx.x < back) single(front + granules * 8 + threadIdx.x);
    const float2 ms = tk_block_join(sh, make_float2(m, s));
    __syncthreads();
    tk_rank(sh, sh.count, want);
    if (slices == 1) {
        tk_write(sh, k, ms, inv_temp, ids + (int64_t)row * k, logp + (int64_t)row * k, lse + row);
    } else {
        uint64_t* kp = keys + ((int64_t)row * slices + blockIdx.x) * k;
        for (int j = threadIdx.x; j < k; j += TK_THREADS) kp[j] = j < want ? sh.best[j] : 0;
        if (threadIdx.x == 0) stats[(int64_t)row * slices + blockIdx.x] = ms;
    }
}

// one workgroup per row: the best of slices * k <= TK_CAP keys
__global__ __launch_bounds__(TK_THREADS) void topk_join_kernel(const uint64_t* __restrict__ keys, const float2* __restrict__ stats, int slices, int k,
                                                              float inv_temp, int32_t* __restrict__ ids, float* __restrict__ logp, float* __restrict__ lse) {
    __shared__ TkShared sh;
    const int row = blockIdx.x;
    for (int j = threadIdx.x; j < slices * k; j += TK_THREADS) sh.cand[j] = keys[(int64_t)row * slices * k + j];
    const float2 ms = tk_block_join(sh, threadIdx.x < (unsigned)slices ? stats[(int64_t)row * slices + threadIdx.x] : make_float2(-INFINITY, 0.f));
    __syncthreads();
    // keys that are 0 (a slice shorter than k) never outrank a key: at least k are not
    tk_rank(sh, slices * k, k);
    tk_write(sh, k, ms, inv_temp, ids + (int64_t)row * k, logp + (int64_t)row * k, lse + row);
}

// slices of a row: enough workgroups for the CUs when there are few rows; a slice keeps at least one segment of values, and the slices' keys
// fit the join's list
static int topk_slices(int T, int V, int k) {
    const int ncu = st_num_cus();
    int s = std::min(st_cdiv(2 * ncu, std::max(T, 1)), st_cdiv(V, TK_CHUNK * TK_SEG / 2));
    s = std::min(s, TK_CAP / k);
    return std::max(s, 1);
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
    if (T < 0 || V <= 0 || k <= 0 || k > V || k > TK_MAX_K || !(inv_temperature > 0.f && inv_temperature < INFINITY)) return ST_EINVAL;
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
        hipLaunchKernelGGL(topk_row_kernel, dim3(used, nt), dim3(TK_THREADS), 0, s, logits + (int64_t)t0 * ldl, ldl, V, k, len, inv_temperature,
                           ids + (int64_t)t0 * k, logp + (int64_t)t0 * k, lse + t0, slices > 1 ? keys + (int64_t)t0 * used * k : nullptr,
                           slices > 1 ? stats + (int64_t)t0 * used : nullptr);
        ST_CHECK_LAUNCH();
    }
    if (used > 1) {
        hipLaunchKernelGGL(topk_join_kernel, dim3(T), dim3(TK_THREADS), 0, s, keys, stats, used, k, inv_temperature, ids, logp, lse);
        ST_CHECK_LAUNCH();
    }
    return 0;
}

}  // extern "C"

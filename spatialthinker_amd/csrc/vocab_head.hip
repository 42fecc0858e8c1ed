// vocab_head.hip — losses of the vocabulary head straight from the hidden states, for gfx950: (rows x vocabulary) logits only in fp32 and on request.
//
//   z[t][v] = (h_t . w_v) / temperature,   lse_t = log sum_v exp z[t][v]
//   log-prob of given tokens:          logp_t = z[t][label_t] - lse_t
//   distillation from top log-probs:   kl_t = sum_k p_tk (log p_tk - (z[t][id_tk] - lse_t)),  p from the teacher's k log-probs of the row
// Both gradients have one form: d[t][v] = c_t exp(z[t][v] - lse_t) + (sparse targets), dh = d W, dW = d^T h, so both share every product:
//   forward   head_tile_kernel<STATS>   z tile in registers -> per row (max, sum 2^(z - max) - 1) of 128 columns; then head_lse_kernel
//   backward  per piece of the vocabulary: head_tile_kernel<DLOGITS> forms the tile again and writes d (bf16) into a bounded workspace, or
//             head_d_kernel writes it from kept logits; head_dh_kernel adds d W into fp32 slabs, head_dw_kernel writes d^T h
// Kept logits cost the forward their write and save the backward one of its three products (forward + backward, 152 064 x 3584: 16 rows 745 -> 621 us,
// 203 rows 1114 -> 883, 1501 rows 4893 -> 4113, 8192 rows 25 580 -> 21 100; 50 257 x 1024, 256 rows 188 -> 181) for 4 T V bytes: the caller chooses.
// d is rounded to bf16 because it is the operand of two bf16 matrix products: half a bf16 step (2^-8 relative) per element, the size of the
// rounding of the bf16 gradients themselves.  Logits, softmax statistics and every sum stay in fp32.
// What bounds them: the matrix pipe (2 T V H flop forward, 4 or 6 T V H backward) from a few hundred rows on, the weight stream (2 V H bytes) below.
#include "gemm_asm4_core.h"
#include <algorithm>

#define VH_LOG2E 1.4426950408889634f
#define VH_LN2 0.6931471805599453f

// columns of a kept-logits row: V rounded up to 64, whatever the row pitch (what lies behind them is the caller's)
__device__ __forceinline__ int vh_cols64(int V) { return (V + 63) & ~63; }

__device__ __forceinline__ float vh_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
// 2^(z2 - top) of a logit that is at most `top` = its row's rounded maximum or lse: what stands above by that rounding alone (half a step of the product,
// 2^7 and more from logits of 2^31 on) counts as equal.  NaN stays NaN (minimum, not fminf).
__device__ __forceinline__ float vh_below(float z, float sc, float top) { return vh_exp2(__builtin_elementwise_minimum(fmaf(z, sc, -top), 0.f)); }

// Statistics of a set of logits (in base 2): x = the largest, y = sum 2^(z - x) - 1.  The largest one's own term is exactly 1 and left out of the sum,
// because the log-prob of a nearly certain token is -log(1 + y): next to a 1 a small y would keep few of its digits.  Empty: (-inf, -1).
__device__ __forceinline__ float2 vh_join(float2 a, float2 b) {
    const float m = fmaxf(a.x, b.x);
    if (m == -INFINITY) return make_float2(m, a.y + b.y + 1.f);      // empty, or NaN kept
    const float ra = a.x == m ? a.y : (1.f + a.y) * vh_exp2(a.x - m);
    return make_float2(m, ra + (b.x == m && a.x != m ? b.y : (1.f + b.y) * vh_exp2(b.x - m)));
}

// workgroup -> tile: each XCD walks a contiguous range of tiles in groups of 8 tile-rows (A and B panels shared in its L2)
__device__ __forceinline__ void vh_tile(int bid, int tiles_m, int tiles_n, int& tm, int& tn) {
    const int nb = tiles_m * tiles_n;
    const int xcd = bid & 7, idx = bid >> 3, q = nb >> 3, r = nb & 7;
    bid = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + idx;
    const int per_group = 8 * tiles_n;
    const int group = bid / per_group, in_g = bid % per_group;
    const int first_m = group * 8;
    const int gsz = min(tiles_m - first_m, 8);
    tm = first_m + in_g % gsz;
    tn = in_g / gsz;
}

// a row of the backward: d = c * 2^(z2 - lse2), at the label's column hot instead; c == 0 and hot == 0: the row takes no part (d = 0 whatever z is)
struct alignas(16) VhRow { float c, lse2, hot; int label; };

// targets of the forward: list[start[tm][tn] .. start[tm][tn + 1]) = those in row tile tm and column tile tn; z2 (T, K) takes their logits
struct VhTargets { const int* start; const uint32_t* list; float* z2; int K; };

// the bf16 tile image of the store epilogues: 256 rows x 256 columns, rows padded by 16 bytes
#define VH_ROWB (256 * 2 + 16)
#define VH_SMEM (256 * VH_ROWB)                                      // 135 168 B >= the two 64-KiB operand slots

// one thread's share of the image -> rows of a bf16 matrix; columns in whole 16-byte chunks (cols % 8 == 0, ldc % 8 == 0)
__device__ __forceinline__ void vh_store_image(const char* smem, uint16_t* __restrict__ C, int64_t ldc, int rows, int cols) {
    const int t = threadIdx.x, c = t & 31;
    if (c * 8 >= cols) return;
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        uint4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = *reinterpret_cast<const uint4*>(smem + ((h * 8 + i) * 8 + (t >> 5)) * VH_ROWB + c * 16);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int row = (h * 8 + i) * 8 + (t >> 5);
            if (row < rows) *reinterpret_cast<uint4*>(C + (int64_t)row * ldc + c * 8) = v[i];
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------------------------
// Logit tile of 256 rows x 256 vocabulary columns.  A lane owns 8 rows (mi*16 + (lane & 15)) and, of each, 4 columns of every 16-column
// tile ni, so row statistics reduce inside the lane first and over the four lanes of a row last.
// STATS: part[tn*2 + wn][m] = the statistics (vh_join) of the 128 columns of a wave; zlab[m] = the label's logit, or z2[m][k] = the logit of target k
// from the tile's list of targets (head_bucket_kernel): from the same accumulators as the statistics, so that a target that is its row's maximum
// has exactly the maximum's value.
// KEEP: z[m][n] = h_m . w_n in fp32 as well, straight from the accumulators (64-byte runs; V = 152 064, H = 3584, 4096 rows: 416 us for 2.5 GB).
// DLOGITS: d[m][n] (bf16, pitch ldd, zero in columns [V, ldd) and rows [T, T64)).
// Bound by the matrix pipe: the main loop is the four-wave tile of the framework's GEMM, and the epilogue has to cost little beside it.  MI355X,
// V = 152 064, H = 3584: 4096 rows 3.05 to 3.2 ms by card = 1.40 to 1.46 PF/s with the join (the GEMM alone, writing logits, 3.1); 161 .. 256 rows, one row
// tile: 260 to 285 us whatever their number, 4 TB/s of weights (2.3 rounds of 256 tiles: a last part round in narrower tiles was 0 to 8 % slower).
// ------------------------------------------------------------------------------------------------------------------------------------
template <bool DLOGITS, bool ONE_ROW_TILE, bool KEEP = false>
__global__ __launch_bounds__(256) void head_tile_kernel(const uint16_t* __restrict__ h, int64_t ldh, const uint16_t* __restrict__ w, int64_t ldw, int T,
                                                       int V, int H, int tiles_m, int tiles_n, float sc, const int64_t* __restrict__ labels,
                                                       float2* __restrict__ part, float* __restrict__ zlab, VhTargets tg, const VhRow* __restrict__ rows, int v0,
                                                       uint16_t* __restrict__ d, int64_t ldd, int T64, float* __restrict__ z, int64_t ldz) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    int tm, tn;
    vh_tile(blockIdx.x, tiles_m, tiles_n, tm, tn);
    const int m0 = tm * A4_BM, n0 = tn * A4_BN;
    f32x4 acc[8][8];
    a4_mainloop<false, false, false, 0, false, KEEP, ONE_ROW_TILE>(smem, h, ldh, w, ldw, m0, n0, T, V, 0, H / 64, H, acc);
    const int col0 = n0 + wn * 128 + (lane >> 4) * 4;                // column of (ni, r): col0 + ni*16 + r
    const bool inside = n0 + A4_BN <= V;
    if constexpr (!DLOGITS) {
        if constexpr (KEEP) {
#pragma unroll
            for (int mi = 0; mi < 8; ++mi) {
                const int m = m0 + wm * 128 + mi * 16 + (lane & 15);
                if (m >= T) continue;
#pragma unroll
                for (int ni = 0; ni < 8; ++ni)
                    if (col0 + ni * 16 < vh_cols64(V)) *reinterpret_cast<f32x4*>(z + (int64_t)m * ldz + col0 + ni * 16) = acc[ni][mi];
            }
        }
        const int e0 = tg.start ? tg.start[tm * (tiles_n + 1) + tn] : 0, e1 = tg.start ? tg.start[tm * (tiles_n + 1) + tn + 1] : 0;
        if (e1 > e0) {                                               // the tile through LDS, 128 columns (64 of each wave pair) at a time
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                __syncthreads();
#pragma unroll
                for (int nl = 0; nl < 4; ++nl)
#pragma unroll
                    for (int mi = 0; mi < 8; ++mi)
                        *reinterpret_cast<f32x4*>(smem + (wm * 128 + mi * 16 + (lane & 15)) * VH_ROWB + (wn * 64 + nl * 16 + (lane >> 4) * 4) * 4) = acc[p * 4 + nl][mi];
                __syncthreads();
                for (int e = e0 + threadIdx.x; e < e1; e += 256) {
                    const uint32_t it = tg.list[e];                  // row (8 bits), column (8 bits), k
                    const int row = it & 255, col = (it >> 8) & 255;
                    if (((col >> 6) & 1) == p)
                        tg.z2[(int64_t)(m0 + row) * tg.K + (it >> 16)] =
                            sc * *reinterpret_cast<const float*>(smem + row * VH_ROWB + ((col >> 7) * 64 + (col & 63)) * 4);
                }
            }
        }
#pragma unroll
        for (int mi = 0; mi < 8; ++mi) {
            const int m = m0 + wm * 128 + mi * 16 + (lane & 15);
            if (!inside) {
#pragma unroll
                for (int ni = 0; ni < 8; ++ni)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[ni][mi][r] = col0 + ni * 16 + r < V ? acc[ni][mi][r] : -INFINITY;
            }
            float mx = acc[0][mi][0];
#pragma unroll
            for (int ni = 0; ni < 8; ++ni)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx = fmaxf(mx, acc[ni][mi][r]);
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const float m2 = mx * sc;                                // sc > 0
            const float sub = m2 == -INFINITY ? 0.f : m2;            // nothing but -inf: every term is 2^-inf = 0
            float s = 0.f;
#pragma unroll
            for (int ni = 0; ni < 8; ++ni)
#pragma unroll
                for (int r = 0; r < 4; ++r) s += vh_exp2(fmaf(acc[ni][mi][r], sc, -sub));
            s += __shfl_xor(s, 16, 64);
            s += __shfl_xor(s, 32, 64);
            float rest = s - 1.f;                                    // (nothing but -inf: -1)
            const bool apart = (s < 1.5f || fabsf(m2) >= 0x1p23f) && fabsf(m2) < INFINITY;
            if (__any(apart)) {                                      // a row with one large logit among these 128, or a rounding of its maximum that counts: the others' sum by itself
                float o = 0.f, ties = -1.f;
#pragma unroll
                for (int ni = 0; ni < 8; ++ni)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float x = acc[ni][mi][r];
                        if (x == mx) ties += 1.f; else o += vh_below(x, sc, sub);
                    }
                ties += lane < 16 ? 0.f : 1.f;                       // (the -1 once per row)
                o += __shfl_xor(o, 16, 64);
                o += __shfl_xor(o, 32, 64);
                ties += __shfl_xor(ties, 16, 64);
                ties += __shfl_xor(ties, 32, 64);
                if (apart) rest = o + ties;                          // (s is the same in a row's four lanes: no row depends on the others of its wave)
            }
            if (m < T) {
                if (lane < 16) part[(int64_t)(tn * 2 + wn) * T + m] = make_float2(m2, rest);
                if (labels) {
                    const int64_t lab = labels[m] - (n0 + wn * 128);
                    if (lab >= 0 && lab < 128) {                     // one lane of the row owns the label's column
#pragma unroll
                        for (int ni = 0; ni < 8; ++ni)
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                if (lab == ni * 16 + (lane >> 4) * 4 + r && col0 + ni * 16 + r < V) zlab[m] = acc[ni][mi][r] * sc;
                    }
                }
            }
        }
    } else {
        __syncthreads();                                             // every wave is done with the operand slots
#pragma unroll
        for (int mi = 0; mi < 8; ++mi) {
            const int row = wm * 128 + mi * 16 + (lane & 15), m = m0 + row;
            VhRow ri = {0.f, 0.f, 0.f, -1};
            if (m < T) ri = rows[m];
            const int lab = ri.label - v0 - col0;                    // column of the label relative to this lane's first
            const bool live = ri.c != 0.f || ri.hot != 0.f;          // (NaN coefficients are live)
#pragma unroll
            for (int ni = 0; ni < 8; ++ni) {
                float o[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float x = ri.c * vh_below(acc[ni][mi][r], sc, ri.lse2);
                    if (lab == ni * 16 + r) x = ri.hot;
                    o[r] = live && (inside || col0 + ni * 16 + r < V) ? x : 0.f;
                }
                uint2 pk;
                pk.x = f2bf2(o[0], o[1]); pk.y = f2bf2(o[2], o[3]);
                *reinterpret_cast<uint2*>(smem + row * VH_ROWB + (wn * 128 + ni * 16 + (lane >> 4) * 4) * 2) = pk;
            }
        }
        __syncthreads();
        vh_store_image(smem, d + (int64_t)m0 * ldd + n0, ldd, T64 - m0, (int)ldd - n0);
    }
}

// ------------------------------------------------------------------------------------------------------------------------------------
// The same logit tile for few rows (T <= 160): the launch is a stream of the head's weights.  BT = 16 MT rows x 32 vocabulary columns per wave, K-steps
// of 64 through SLOTS LDS slots filled by LDS-DMA (16-byte chunk c of a row at position c ^ (row & 7): conflict-free fragment reads), SLOTS - 1 steps
// in flight behind one barrier per step.  Up to 64 rows four waves, so that several workgroups share a CU and one's epilogue hides behind another's
// copies; beyond, eight waves with the whole LDS, because the hidden states are copied again for every workgroup: 128 rows beside 128 columns fill as
// many bytes with them as with weights.  Epilogues as head_tile_kernel; part[block][m].  DLOGITS also leaves d transposed, dt[n][TP], up to 128 rows.
// MI355X, V = 152 064, forward with its join (of 6.8 TB/s that a read alone reaches): H = 3584, 1 row 162 us = 6.7 TB/s, 64 rows 176 = 6.2, 96 rows
// 207 = 5.3 (128 columns: 226), 128 rows 217 = 5.0 (245), 160 rows 247 = 4.4 (256-row tile 275); H = 2048, 1 row 104 us = 6.0 TB/s, 160 rows 149.
// ------------------------------------------------------------------------------------------------------------------------------------
template <int N> __device__ __forceinline__ void vh_wait_vm() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

template <int MT, int SLOTS, int WAVES, bool DLOGITS>
__global__ __launch_bounds__(64 * WAVES, 2) void head_few_kernel(const uint16_t* __restrict__ h, int64_t ldh, const uint16_t* __restrict__ w, int64_t ldw, int T, int V,
                                                         int H, float sc, const int64_t* __restrict__ labels, float2* __restrict__ part,
                                                         float* __restrict__ zlab, VhTargets tg, const VhRow* __restrict__ rows, int v0,
                                                         uint16_t* __restrict__ d, int64_t ldd, uint16_t* __restrict__ dt, int TP, float* __restrict__ z, int64_t ldz) {
    constexpr int BT = 16 * MT, BN = 32 * WAVES, SLOT = (BN + BT) * 128, NT = 64 * WAVES;
    constexpr int HC = (2 * MT + WAVES - 1) / WAVES;                 // 1-KiB copies of h per wave and step (the last waves may copy some rows again)
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n0 = blockIdx.x * BN;
    // copy j of a wave: 8 rows, lane -> row (lane >> 3), 16-byte chunk (lane & 7) ^ row
    const int cr = lane >> 3, ch = ((lane & 7) ^ cr) * 8;
    const uint16_t* wsrc[4];
    const uint16_t* hsrc[HC];
#pragma unroll
    for (int j = 0; j < 4; ++j) wsrc[j] = w + (int64_t)min(n0 + wave * 32 + j * 8 + cr, V - 1) * ldw + ch;
#pragma unroll
    for (int j = 0; j < HC; ++j) hsrc[j] = h + (int64_t)min((wave * HC + j) % (2 * MT) * 8 + cr, T - 1) * ldh + ch;
    const int nk = H / 64, fr = lane & 15, fk = lane >> 4;
    // K-step kt reads k = (kt + turn) % nk: rows at a pitch of whole 4 KiB meet in a few memory channels where all workgroups stand at the same k
    // (V = 100 000, H = 2048: 8 rows 89 -> 79 us, 100 rows 107 -> 90; H = 4096: 168 -> 141, 200 -> 157; at other pitches 0 to 3 % slower, so not there)
    // (counted from the vocabulary's first column, so that a piece of it sums in the order of the whole)
    const int turn = (ldw & 2047) == 0 ? (int)(v0 / BN + blockIdx.x) % nk : 0;
    auto stage = [&](int kt) {
        char* dst = smem + (kt % SLOTS) * SLOT;
        const int k = (kt + turn < nk ? kt + turn : kt + turn - nk) * 64;
#pragma unroll
        for (int j = 0; j < 4; ++j) st_glds16_nt(wsrc[j] + k, dst + (wave * 32 + j * 8) * 128);       // one workgroup reads a weight, once
#pragma unroll
        for (int j = 0; j < HC; ++j) st_glds16(hsrc[j] + k, dst + (BN + (wave * HC + j) % (2 * MT) * 8) * 128);
    };
    f32x4 acc[2][MT], sum[2][MT];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) sum[i][j] = acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < SLOTS - 1; ++s) if (s < nk) stage(s);
    for (int kt = 0; kt < nk; ++kt) {
        // this step's copies have landed; up to SLOTS - 2 younger steps stay in flight (the last steps have none to count)
        if (kt + SLOTS - 2 < nk) vh_wait_vm<(SLOTS - 2) * (4 + HC)>(); else vh_wait_vm<0>();
        __builtin_amdgcn_s_barrier();                                // ... for every wave, and every wave has read the slot that is filled next (the reads of
        asm volatile("" ::: "memory");                               // a step have returned before its products; a test finds any in the built code that have not)
        if (kt + SLOTS - 1 < nk) stage(kt + SLOTS - 1);
        const char* lw = smem + (kt % SLOTS) * SLOT + wave * 32 * 128;
        const char* lh = smem + (kt % SLOTS) * SLOT + BN * 128;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            const int c = ((s * 4 + fk) ^ (fr & 7)) << 4;
            bf16x8 wf[2], hf[MT];
#pragma unroll
            for (int i = 0; i < 2; ++i) wf[i] = *reinterpret_cast<const bf16x8*>(lw + (i * 16 + fr) * 128 + c);
#pragma unroll
            for (int i = 0; i < MT; ++i) hf[i] = *reinterpret_cast<const bf16x8*>(lh + (i * 16 + fr) * 128 + c);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < MT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[i], hf[j], acc[i][j], 0, 0, 0);
        }
        if constexpr (MT <= 4) {                                     // sums of sums: fewer roundings, where registers and time are free
            if ((kt & 7) == 7)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < MT; ++j) { sum[i][j] += acc[i][j]; acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f}; }
        }
    }
    if constexpr (MT <= 4)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < MT; ++j) acc[i][j] += sum[i][j];
    __syncthreads();                                                 // the slots are free
    const int col0 = n0 + wave * 32 + fk * 4;                        // column of (i, r): col0 + i*16 + r
    if constexpr (!DLOGITS) {
        constexpr int ROWB = 128 * 4 + 16;
        const int e0 = tg.start ? tg.start[n0 >> 8] : 0, e1 = tg.start ? tg.start[(n0 >> 8) + 1] : 0;
        for (int p = 0; p < BN / 128 && (e1 > e0 || z); ++p) {       // the tile through LDS, 128 columns at a time
            if (wave >> 2 == p) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < MT; ++j) *reinterpret_cast<f32x4*>(smem + (j * 16 + fr) * ROWB + ((wave & 3) * 32 + i * 16 + fk * 4) * 4) = acc[i][j];
            }
            __syncthreads();
            for (int e = e0 + threadIdx.x; e < e1; e += NT) {
                const uint32_t it = tg.list[e];
                const int row = it & 255, col = (it >> 8) & 255;
                if ((col >> 7) == (((n0 >> 7) + p) & 1))
                    tg.z2[(int64_t)row * tg.K + (it >> 16)] = sc * *reinterpret_cast<const float*>(smem + row * ROWB + (col & 127) * 4);
            }
            if (z)                                                   // kept logits leave in runs of 512 bytes
                for (int i = threadIdx.x; i < T * 32; i += NT) {
                    const int row = i >> 5, c = (i & 31) * 4, col = n0 + p * 128 + c;
                    if (col < vh_cols64(V)) *reinterpret_cast<f32x4*>(z + (int64_t)row * ldz + col) = *reinterpret_cast<const f32x4*>(smem + row * ROWB + c * 4);
                }
            __syncthreads();
        }
        float2* red = reinterpret_cast<float2*>(smem);               // [wave][row]
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            const int m = j * 16 + fr;
            float mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (col0 + i * 16 + r >= V) acc[i][j][r] = -INFINITY;
                    mx = fmaxf(mx, acc[i][j][r]);
                }
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            const float m2 = mx * sc, sub = m2 == -INFINITY ? 0.f : m2;
            float o = 0.f, ties = lane < 16 ? -1.f : 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float x = acc[i][j][r];
                    if (x == mx) ties += 1.f; else o += vh_exp2(fmaf(x, sc, -sub));
                }
            o += __shfl_xor(o, 16, 64);
            o += __shfl_xor(o, 32, 64);
            ties += __shfl_xor(ties, 16, 64);
            ties += __shfl_xor(ties, 32, 64);
            if (lane < 16) red[wave * BT + m] = make_float2(m2, m2 != -INFINITY ? o + ties : o - 1.f);
            if (labels && m < T) {
                const int64_t lab = labels[m] - col0;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (lab == i * 16 + r && col0 + i * 16 + r < V) zlab[m] = acc[i][j][r] * sc;
            }
        }
        __syncthreads();
        for (int m = threadIdx.x; m < min(BT, T); m += NT) {
            float2 a = red[m];
#pragma unroll
            for (int wv = 1; wv < WAVES; ++wv) a = vh_join(a, red[wv * BT + m]);
            part[(int64_t)blockIdx.x * T + m] = a;
        }
    } else {
        // two bf16 images: [BT rows][BN columns] and (up to 128 rows) [BN columns][BT rows]
        constexpr int RB = BN * 2 + 16, CB = BT * 2 + 16;
        char* img_t = smem + BT * RB;
#pragma unroll
        for (int j = 0; j < MT; ++j) {
            const int m = j * 16 + fr;
            VhRow ri = {0.f, 0.f, 0.f, -1};
            if (m < T) ri = rows[m];
            const int lab = ri.label - v0 - col0;
            const bool live = ri.c != 0.f || ri.hot != 0.f;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float o[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float x = ri.c * vh_below(acc[i][j][r], sc, ri.lse2);
                    if (lab == i * 16 + r) x = ri.hot;
                    o[r] = live && col0 + i * 16 + r < V ? x : 0.f;
                }
                uint2 pk;
                pk.x = f2bf2(o[0], o[1]); pk.y = f2bf2(o[2], o[3]);
                const int col = wave * 32 + i * 16 + fk * 4;
                *reinterpret_cast<uint2*>(smem + m * RB + col * 2) = pk;
                if constexpr (MT <= 8) {
                    *reinterpret_cast<uint16_t*>(img_t + (col + 0) * CB + m * 2) = (uint16_t)pk.x;
                    *reinterpret_cast<uint16_t*>(img_t + (col + 1) * CB + m * 2) = (uint16_t)(pk.x >> 16);
                    *reinterpret_cast<uint16_t*>(img_t + (col + 2) * CB + m * 2) = (uint16_t)pk.y;
                    *reinterpret_cast<uint16_t*>(img_t + (col + 3) * CB + m * 2) = (uint16_t)(pk.y >> 16);
                }
            }
        }
        __syncthreads();
        const int cols = min(BN, (int)ldd - n0);                     // ldd % 64 == 0
        constexpr int CH = BN / 8;                                   // 16-byte chunks of a row of d
        const int rows_out = MT <= 8 ? T : TP;                       // rows [T, TP) are zero for head_dw_mid_kernel
        for (int i = threadIdx.x; i < rows_out * CH; i += NT) {
            const int row = i / CH, c = (i % CH) * 8;
            if (c < cols)
                *reinterpret_cast<uint4*>(d + (int64_t)row * ldd + n0 + c) =
                    MT <= 8 || row < BT ? *reinterpret_cast<const uint4*>(smem + row * RB + c * 2) : make_uint4(0, 0, 0, 0);
        }
        if constexpr (MT <= 8) {
            const int per = TP >> 3;                                 // 16-byte chunks of a row of dt: TP is BT, or more (zeros)
            for (int i = threadIdx.x; i < cols * per; i += NT) {
                const int col = i / per, c = (i - col * per) * 8;
                *reinterpret_cast<uint4*>(dt + (int64_t)(n0 + col) * TP + c) = c < BT ? *reinterpret_cast<const uint4*>(img_t + col * CB + c * 2) : make_uint4(0, 0, 0, 0);
            }
        }
    }
}

// d of a piece from the logits that the forward has kept: the epilogue of the tiles above, element by element with the same roundings.  64 rows x 128
// columns per workgroup, eight columns per thread; FEW: also dt.  Bound: 4 B read and 2 B (FEW: 4 B) written per value
// (4096 x 152 064: 690 us = 5.4 TB/s; 48 rows 19 us).
template <bool FEW>
__global__ __launch_bounds__(256) void head_d_kernel(const float* __restrict__ z, int64_t ldz, const VhRow* __restrict__ rows, int T, int V, float sc, int v0,
                                                     uint16_t* __restrict__ d, int64_t ldd, int T64, uint16_t* __restrict__ dt, int TP) {
    constexpr int CB = 64 * 2 + 16;
    __shared__ __attribute__((aligned(16))) char img[FEW ? 128 * CB : 16];
    const int nb = (int)((ldd + 127) >> 7), r0 = (int)(blockIdx.x / nb) * 64, n0 = (int)(blockIdx.x % nb) * 128, c = (threadIdx.x & 15) * 8, rr = threadIdx.x >> 4;
    const bool in = n0 + c < ldd;
    f32x4 v[4][2];
    VhRow ri[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int m = r0 + i * 16 + rr;
        ri[i] = {0.f, 0.f, 0.f, -1};
        v[i][0] = v[i][1] = (f32x4){0.f, 0.f, 0.f, 0.f};
        if (m < T && in) {
            ri[i] = rows[m];
            v[i][0] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(z + (int64_t)m * ldz + n0 + c));
            v[i][1] = __builtin_nontemporal_load(reinterpret_cast<const f32x4*>(z + (int64_t)m * ldz + n0 + c + 4));
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int m = r0 + i * 16 + rr, lab = ri[i].label - v0 - n0 - c;
        const bool live = ri[i].c != 0.f || ri[i].hot != 0.f;
        float o[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            float x = ri[i].c * vh_below(v[i][k >> 2][k & 3], sc, ri[i].lse2);
            if (lab == k) x = ri[i].hot;
            o[k] = live && n0 + c + k < V ? x : 0.f;
        }
        uint4 pk;
        pk.x = f2bf2(o[0], o[1]); pk.y = f2bf2(o[2], o[3]); pk.z = f2bf2(o[4], o[5]); pk.w = f2bf2(o[6], o[7]);
        if (in && m < (FEW ? T : T64)) *reinterpret_cast<uint4*>(d + (int64_t)m * ldd + n0 + c) = pk;
        if constexpr (FEW) {
            const uint32_t u[4] = {pk.x, pk.y, pk.z, pk.w};
#pragma unroll
            for (int k = 0; k < 8; ++k) *reinterpret_cast<uint16_t*>(img + (c + k) * CB + (i * 16 + rr) * 2) = (uint16_t)(u[k >> 1] >> ((k & 1) * 16));
        }
    }
    if constexpr (FEW) {
        __syncthreads();
        for (int i = threadIdx.x; i < 128 * 8; i += 256) {
            const int col = i >> 3, r = (i & 7) * 8;
            if (n0 + col < ldd && r0 + r < TP) *reinterpret_cast<uint4*>(dt + (int64_t)(n0 + col) * TP + r0 + r) = *reinterpret_cast<const uint4*>(img + col * CB + r * 2);
        }
    }
}

// partial statistics (vh_join) -> lse (natural log), stat = (max, log2 sum); logp = label logit - lse for rows with a label inside the vocabulary, 0 for the others.
// 16 rows x 64 slices per workgroup: 16 consecutive lanes read 128 contiguous bytes of one partial row.  Bound: reading the partials, 8 B per row and
// 128 columns (4096 rows, V = 152 064: 39 MB in 15 us).
__global__ __launch_bounds__(1024) void head_lse_kernel(const float2* __restrict__ part, int n_parts, const float* __restrict__ zlab,
                                                       const int64_t* __restrict__ labels, float* __restrict__ logp, float* __restrict__ lse, float2* __restrict__ stat,
                                                       int T, int V) {
    __shared__ float2 red[64][17];
    const int r = threadIdx.x & 15, sl = threadIdx.x >> 4;
    const int row = blockIdx.x * 16 + r;
    float2 a = make_float2(-INFINITY, -1.f);
    if (row < T)
#pragma unroll 4
        for (int p = sl; p < n_parts; p += 64) a = vh_join(a, part[(int64_t)p * T + row]);
    red[sl][r] = a;
    __syncthreads();
    for (int o = 32; o > 0; o >>= 1) {
        if (sl < o) red[sl][r] = vh_join(red[sl][r], red[sl + o][r]);
        __syncthreads();
    }
    if (sl == 0 && row < T) {
        const float2 v = red[0][r];
        const float ls = v.x < INFINITY ? log1pf(v.y) * VH_LOG2E : NAN;      // +inf, given or overflowed: NaN, as inf - inf is
        lse[row] = (v.x + ls) * VH_LN2;
        if (stat) stat[row] = make_float2(v.x, ls);
        if (labels) {                                                // (z - max) - log sum: exact where the label is the maximum, so a log-prob near 0
            const int64_t lab = labels[row];                         // keeps its digits; z - lse would lose them in lse's rounding
            logp[row] = lab >= 0 && lab < V ? ((zlab[row] - v.x) - ls) * VH_LN2 : 0.f;
        }
    }
}

// the same for few rows, where reading the partials one behind the other is what takes the time: a workgroup per row (up to 200 rows 4 to 6 us)
__global__ __launch_bounds__(1024) void head_lse_few_kernel(const float2* __restrict__ part, int n_parts, const float* __restrict__ zlab,
                                                           const int64_t* __restrict__ labels, float* __restrict__ logp, float* __restrict__ lse,
                                                           float2* __restrict__ stat, int T, int V) {
    __shared__ float2 red[16];
    const int row = blockIdx.x, lane = threadIdx.x & 63;
    float2 a = make_float2(-INFINITY, -1.f);
    for (int p = threadIdx.x; p < n_parts; p += 1024) a = vh_join(a, part[(int64_t)p * T + row]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) a = vh_join(a, make_float2(__shfl_xor(a.x, o, 64), __shfl_xor(a.y, o, 64)));
    if (lane == 0) red[threadIdx.x >> 6] = a;
    __syncthreads();
    if (threadIdx.x < 64) {
        a = red[lane & 15];
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) a = vh_join(a, make_float2(__shfl_xor(a.x, o, 64), __shfl_xor(a.y, o, 64)));
        if (lane == 0) {
            const float ls = a.x < INFINITY ? log1pf(a.y) * VH_LOG2E : NAN;
            lse[row] = (a.x + ls) * VH_LN2;
            if (stat) stat[row] = make_float2(a.x, ls);
            if (labels) {
                const int64_t lab = labels[row];
                logp[row] = lab >= 0 && lab < V ? ((zlab[row] - a.x) - ls) * VH_LN2 : 0.f;
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------------------------
// Backward: row coefficients and the packed hidden states.  A row of d is held as scale_t * d', with d' in the workspace and the scale in
// hz[t][:] = bf16(scale_t h[t][:]) (for dW) and in the finish of dh.  Where one target dominates a row the scale is that target's gradient: its d' is
// 1, exact in bf16, and dh does not get that one rounding in all of its elements.  Otherwise the scale is 1 and hz = h.
// hz is 0 for rows without a gradient and for the padding rows [T, T64): what such rows of h hold (also infinities and NaN) cannot reach dW
// through 0 * x.
// ------------------------------------------------------------------------------------------------------------------------------------
// Either of hz and hzt (transposed, row pitch TP: the few-row kernels) is written.
__device__ __forceinline__ void vh_pack_row(const uint16_t* __restrict__ h, int64_t ldh, uint16_t* __restrict__ hz, uint16_t* __restrict__ hzt, int TP, int t,
                                            bool live, float scale, int H) {
    for (int i = threadIdx.x * 8; i < H; i += blockDim.x * 8) {
        union { uint4 v; uint16_t e[8]; } o;
        o.v = make_uint4(0, 0, 0, 0);
        if (live) {
            float f[8];
            unpack8(*reinterpret_cast<const uint4*>(h + (int64_t)t * ldh + i), f);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] *= scale;
            o.v = pack8(f);
        }
        if (hz) *reinterpret_cast<uint4*>(hz + (int64_t)t * H + i) = o.v;
        else
#pragma unroll
            for (int j = 0; j < 8; ++j) hzt[(int64_t)(i + j) * TP + t] = o.e[j];
    }
}

__global__ __launch_bounds__(128) void head_rows_label_kernel(const uint16_t* __restrict__ h, int64_t ldh, const int64_t* __restrict__ labels,
                                                             const float* __restrict__ logp, const float* __restrict__ lse,
                                                             const float* __restrict__ g, float inv_temp, VhRow* __restrict__ rows,
                                                             float* __restrict__ scale, uint16_t* __restrict__ hz, uint16_t* __restrict__ hzt, int TP,
                                                          int T, int V, int H) {
    const int t = blockIdx.x;
    VhRow ri = {0.f, 0.f, 0.f, -1};
    float sc = 1.f;
    if (t < T) {
        const int64_t lab = labels[t];
        if (lab >= 0 && lab < V) {
            const float e = expm1f(logp[t]), hot = -e * g[t] * inv_temp;                 // g/temperature (1 - q), q the label's probability
            if (hot != 0.f) {                                        // (NaN is not 0)
                sc = hot;
                ri.c = 1.f / e; ri.hot = 1.f; ri.label = (int)lab; ri.lse2 = lse[t] * VH_LOG2E;
            }
        }
        if (threadIdx.x == 0) { rows[t] = ri; scale[t] = sc; }
    }
    vh_pack_row(h, ldh, hz, hzt, TP, t, ri.hot != 0.f, sc, H);
}

// slab[s][m][n] (+)= sum over the K-slice s of d[m][:] w[:][n]: w is contraction-major as stored; `kv` of the ldd columns of d are vocabulary.
// On its own where there is one row tile (129 .. 256 rows) or no dW is asked for: the vocabulary is the long axis, so it is cut into slices that
// fill the CUs in whole rounds, joined in slice order by head_dh_finish_kernel.  Bound: the weight stream through 256-row tiles (200 x 3584 x 152 064:
// 259 us = 4.2 TB/s; 150 x 2048 x 151 936: 155 us = 4.0).
template <bool ACCUM, bool ONE_ROW_TILE>
__device__ __forceinline__ void head_dh_tile(char* smem, int block, const uint16_t* __restrict__ d, int64_t ldd, const uint16_t* __restrict__ w, int64_t ldw,
                                             int T, int kv, int H, int tiles_m, int tiles_n, int split, float* __restrict__ slab) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    const int nb = tiles_m * tiles_n, slice = block / nb;
    int tm, tn;
    vh_tile(block % nb, tiles_m, tiles_n, tm, tn);
    const int m0 = tm * A4_BM, n0 = tn * A4_BN;
    const int nkt = (kv + 63) / 64, per = (nkt + split - 1) / split, kt0 = slice * per;
    const int nk = min(nkt - kt0, per);                              // >= 1: the host gives no slice without K-tiles
    f32x4 acc[8][8];
    a4_mainloop<false, true, false, 0, true, false, ONE_ROW_TILE>(smem, d, ldd, w, ldw, m0, n0, T, H, kt0, nk, kv, acc);
    float* out = slab + (int64_t)slice * T * H;
#pragma unroll
    for (int mi = 0; mi < 8; ++mi) {
        const int m = m0 + wm * 128 + mi * 16 + (lane & 15);
        if (m >= T) continue;
#pragma unroll
        for (int ni = 0; ni < 8; ++ni) {
            const int n = n0 + wn * 128 + ni * 16 + (lane >> 4) * 4;
            if (n >= H) continue;
            float4* p = reinterpret_cast<float4*>(out + (int64_t)m * H + n);
            float4 o = make_float4(acc[ni][mi][0], acc[ni][mi][1], acc[ni][mi][2], acc[ni][mi][3]);
            if constexpr (ACCUM) { const float4 c = *p; o.x += c.x; o.y += c.y; o.z += c.z; o.w += c.w; }
            *p = o;
        }
    }
}

template <bool ACCUM, bool ONE_ROW_TILE>
__global__ __launch_bounds__(256) void head_dh_kernel(const uint16_t* __restrict__ d, int64_t ldd, const uint16_t* __restrict__ w, int64_t ldw, int T,
                                                     int kv, int H, int tiles_m, int tiles_n, int split, float* __restrict__ slab) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    head_dh_tile<ACCUM, ONE_ROW_TILE>(smem, blockIdx.x, d, ldd, w, ldw, T, kv, H, tiles_m, tiles_n, split, slab);
}

// The same for few rows (T <= 128): a stream of w, [32 vocabulary rows][256 columns] per step through SLOTS LDS slots, next to a [16 MT][32] tile of d
// (rows beyond T: the last one, never stored).
// w is contraction-major: its fragments are LDS transpose reads (image and swizzle as the contraction-major operands of gemm_asm4.hip).  Four
// waves of 64 columns, all rows each; the vocabulary is cut into slices so that every CU has two workgroups.  Bound: the weight stream (3584 x 152 064:
// 16 rows 186 us = 5.9 TB/s, 128 rows 244 us = 4.5).
template <int MT, int SLOTS>
__global__ __launch_bounds__(256, 2) void head_dh_few_kernel(const uint16_t* __restrict__ d, int64_t ldd, const uint16_t* __restrict__ w, int64_t ldw, int T,
                                                            int kv, int H, int tiles_n, int per, float* __restrict__ slab) {
    constexpr int BT = 16 * MT, WB = 32 * 512, SLOT = WB + BT * 64, DC = BT / 64;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int slice = blockIdx.x / tiles_n, n0 = (blockIdx.x % tiles_n) * 256;
    const int nkt = (kv + 31) / 32, kt0 = slice * per, nk = min(nkt - kt0, per);
    // copies of w: two k-rows each, lane -> k-row (lane >> 5), 16-byte piece sl: the 32-byte chunk (sl >> 1) ^ g(k-row)
    int wcol[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int kr = wave * 8 + j * 2 + (lane >> 5), sl = lane & 31, g = (kr & 3) | (((kr >> 3) & 1) << 2);
        wcol[j] = n0 + min((((sl >> 1) ^ g) << 4) + (sl & 1) * 8, min(256, H - n0) - 8);
    }
    const uint16_t* dsrc[DC];
#pragma unroll
    for (int j = 0; j < DC; ++j) {                                   // copies of d: 16 rows of 64 bytes, 16-byte chunk (lane & 3) ^ (row >> 2)
        const int row = (wave * DC + j) * 16 + (lane >> 2);
        dsrc[j] = d + (int64_t)min(row, T - 1) * ldd + (((lane & 3) ^ ((row >> 2) & 3)) << 3);
    }
    auto stage = [&](int kt) {
        char* dst = smem + (kt % SLOTS) * SLOT;
        const int k0 = (kt0 + kt) * 32;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int kr = wave * 8 + j * 2 + (lane >> 5);           // k-rows beyond the vocabulary read its last one: d is zero there
            st_glds16(w + (int64_t)min(k0 + kr, kv - 1) * ldw + wcol[j], dst + (wave * 4 + j) * 1024);
        }
#pragma unroll
        for (int j = 0; j < DC; ++j) st_glds16(dsrc[j] + k0, dst + WB + (wave * DC + j) * 1024);
    };
    f32x4 acc[4][MT];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
    const int fr = lane & 15, fk = lane >> 4;
    const uint32_t smem32 = (uint32_t)(uintptr_t)smem;
    uint32_t tr[4];
    {
        const int g = ((lane >> 2) & 3) | ((fk & 1) << 2), row = fk * 8 + (fr >> 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) tr[i] = smem32 + row * 512 + (((wave * 4 + i) ^ g) << 5) + (lane & 3) * 8;
    }
#pragma unroll
    for (int s = 0; s < SLOTS - 1; ++s) if (s < nk) stage(s);
    for (int kt = 0; kt < nk; ++kt) {
        if (kt + SLOTS - 2 < nk) vh_wait_vm<(SLOTS - 2) * (4 + DC)>(); else vh_wait_vm<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (kt + SLOTS - 1 < nk) stage(kt + SLOTS - 1);
        const uint32_t at = (kt % SLOTS) * SLOT;
        const char* ld = smem + at + WB;
        bf16x8 df[MT];
#pragma unroll
        for (int j = 0; j < MT; ++j) df[j] = *reinterpret_cast<const bf16x8*>(ld + (j * 16 + fr) * 64 + ((fk ^ ((fr >> 2) & 3)) << 4));
        union Frag { bf16x8 v; s16x4_t h[2]; } wf[4];
        // the transpose reads and the wait for them in one statement: the compiler neither sees the reads nor holds up the copies in flight
        asm volatile("ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:2048\n\tds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:2048\n\t"
                     "ds_read_b64_tr_b16 %4, %10\n\tds_read_b64_tr_b16 %5, %10 offset:2048\n\tds_read_b64_tr_b16 %6, %11\n\tds_read_b64_tr_b16 %7, %11 offset:2048\n\t"
                     "s_waitcnt lgkmcnt(0)"
                     : "=&v"(wf[0].h[0]), "=&v"(wf[0].h[1]), "=&v"(wf[1].h[0]), "=&v"(wf[1].h[1]), "=&v"(wf[2].h[0]), "=&v"(wf[2].h[1]), "=&v"(wf[3].h[0]),
                       "=&v"(wf[3].h[1])
                     : "v"(tr[0] + at), "v"(tr[1] + at), "v"(tr[2] + at), "v"(tr[3] + at)
                     : "memory");
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < MT; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[i].v, df[j], acc[i][j], 0, 0, 0);
    }
    float* out = slab + (int64_t)slice * T * H;
#pragma unroll
    for (int j = 0; j < MT; ++j) {
        const int m = j * 16 + fr;
        if (m >= T) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int n = n0 + wave * 64 + i * 16 + fk * 4;
            if (n >= H) continue;
            *reinterpret_cast<f32x4*>(out + (int64_t)m * H + n) = acc[i][j];
        }
    }
}

// dh = bf16(row scale * sum of the slabs, in slice order).  Bound: the slabs (8192 x 3584, two of them: 235 MB read in 30 us, part of it from the caches)
__global__ __launch_bounds__(256) void head_dh_finish_kernel(const float* __restrict__ slab, int split, const float* __restrict__ scale, uint16_t* __restrict__ dh, int64_t lddh, int T, int H) {
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
    if (i >= (int64_t)T * H) return;
    float4 a = *reinterpret_cast<const float4*>(slab + i);
#pragma unroll 8
    for (int s = 1; s < split; ++s) {
        const float4 b = *reinterpret_cast<const float4*>(slab + (int64_t)s * T * H + i);
        a.x += b.x; a.y += b.y; a.z += b.z; a.w += b.w;
    }
    const float sc = scale[i / H];                                   // H % 64 == 0: the four values are of one row
    uint2 o;
    o.x = f2bf2(sc * a.x, sc * a.y); o.y = f2bf2(sc * a.z, sc * a.w);
    *reinterpret_cast<uint2*>(dh + (i / H) * lddh + i % H) = o;
}

// dw[v][n] = sum_t d[t][v] hz[t][n]: both operands contraction-major as they lie in memory.  bf16 result, or fp32 (+=).  Bound: the matrix pipe
// (alone, where no dh is asked for: 4096 x 3584 x 152 064 3.6 ms = 1.24 PF/s).
template <bool OUT_BF16, bool ACCUM>
__device__ __forceinline__ void head_dw_tile(char* smem, int block, const uint16_t* __restrict__ d, int64_t ldd, const uint16_t* __restrict__ hz, int T64,
                                             int kv, int H, int tiles_m, int tiles_n, uint16_t* __restrict__ dwb, float* __restrict__ dwf, int64_t lddw) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    int tm, tn;
    vh_tile(block, tiles_m, tiles_n, tm, tn);
    const int m0 = tm * A4_BM, n0 = tn * A4_BN;
    f32x4 acc[8][8];
    a4_mainloop<true, true, false, 0, false, !OUT_BF16>(smem, d, ldd, hz, H, m0, n0, (int)ldd, H, 0, T64 / 64, T64, acc);
    if constexpr (OUT_BF16) {
        __syncthreads();
#pragma unroll
        for (int mi = 0; mi < 8; ++mi) {
            const int row = wm * 128 + mi * 16 + (lane & 15);
#pragma unroll
            for (int ni = 0; ni < 8; ++ni) {
                uint2 pk;
                pk.x = f2bf2(acc[ni][mi][0], acc[ni][mi][1]); pk.y = f2bf2(acc[ni][mi][2], acc[ni][mi][3]);
                *reinterpret_cast<uint2*>(smem + row * VH_ROWB + (wn * 128 + ni * 16 + (lane >> 4) * 4) * 2) = pk;
            }
        }
        __syncthreads();
        vh_store_image(smem, dwb + (int64_t)m0 * lddw + n0, lddw, kv - m0, H - n0);
    } else {
#pragma unroll
        for (int mi = 0; mi < 8; ++mi) {
            const int m = m0 + wm * 128 + mi * 16 + (lane & 15);
            if (m >= kv) continue;
#pragma unroll
            for (int ni = 0; ni < 8; ++ni) {
                const int n = n0 + wn * 128 + ni * 16 + (lane >> 4) * 4;
                if (n >= H) continue;
                float4* p = reinterpret_cast<float4*>(dwf + (int64_t)m * lddw + n);
                float4 o = make_float4(acc[ni][mi][0], acc[ni][mi][1], acc[ni][mi][2], acc[ni][mi][3]);
                if constexpr (ACCUM) { const float4 c = *p; o.x += c.x; o.y += c.y; o.z += c.z; o.w += c.w; }
                *p = o;
            }
        }
    }
}

template <bool OUT_BF16, bool ACCUM>
__global__ __launch_bounds__(256) void head_dw_kernel(const uint16_t* __restrict__ d, int64_t ldd, const uint16_t* __restrict__ hz, int T64, int kv, int H,
                                                     int tiles_m, int tiles_n, uint16_t* __restrict__ dwb, float* __restrict__ dwf, int64_t lddw) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    head_dw_tile<OUT_BF16, ACCUM>(smem, blockIdx.x, d, ldd, hz, T64, kv, H, tiles_m, tiles_n, dwb, dwf, lddw);
}

// Both gradients of a piece in one launch: the few long tiles of dh first, the many short ones of dw behind them fill the CUs up, where two launches
// would each leave part of their last round idle (8192 x 3584, a piece of 30 464 columns: 448 and 1666 tiles on 256 CUs).  Bound: the matrix pipe (that
// piece 2.55 ms = 1.40 PF/s; 1000 x 2048 x 151 936 1.05 ms = 1.19 PF/s).
template <bool DW_BF16, bool DW_ACCUM, bool DH_ACCUM>
__global__ __launch_bounds__(256) void head_grads_kernel(const uint16_t* __restrict__ d, int64_t ldd, const uint16_t* __restrict__ w, int64_t ldw,
                                                        const uint16_t* __restrict__ hz, int T, int T64, int kv, int H, int tiles_t, int tiles_v, int tiles_h,
                                                        int split, int dh_blocks, float* __restrict__ slab, uint16_t* __restrict__ dwb,
                                                        float* __restrict__ dwf, int64_t lddw) {
    extern __shared__ __attribute__((aligned(16))) char smem[];
    if ((int)blockIdx.x < dh_blocks) head_dh_tile<DH_ACCUM, false>(smem, blockIdx.x, d, ldd, w, ldw, T, kv, H, tiles_t, tiles_h, split, slab);
    else head_dw_tile<DW_BF16, DW_ACCUM>(smem, blockIdx.x - dh_blocks, d, ldd, hz, T64, kv, H, tiles_v, tiles_h, dwb, dwf, lddw);
}

// dw for few rows (TP = 32 KS, T rounded up to 32, 64 or 128): the launch is the write of dw, V H elements, next to 2 KS products of 32 rows each.  Operands stand contraction-
// contiguous (dt[v][TP], hzt[n][TP]), so fragments come straight from memory: dt once per workgroup, hzt from the caches, a step ahead.  A
// workgroup owns 128 vocabulary rows and walks the columns 256 at a time, 64 per wave; the bf16 tile goes through LDS, because a row has to leave in
// long runs: 64-byte pieces of 16 rows at a pitch of H elements meet in a few cache channels (V = 152 064, H = 3584: 292 us against 160 for a fill).
// With it 221 us at 16 rows = 4.9 TB/s written, 230 at 48, 265 at 128.
template <int KS, bool OUT_BF16, bool ACCUM>
__global__ __launch_bounds__(256) void head_dw_few_kernel(const uint16_t* __restrict__ dt, const uint16_t* __restrict__ hzt, int kv, int H,
                                                         uint16_t* __restrict__ dwb, float* __restrict__ dwf, int64_t lddw) {
    constexpr int TP = KS * 32, MI = 8;                             // 16 MI vocabulary rows per workgroup
    __shared__ __attribute__((aligned(16))) char img[OUT_BF16 ? 16 * MI * VH_ROWB : 16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, fr = lane & 15, fk = lane >> 4;
    const int r0 = blockIdx.x * (16 * MI);
    bf16x8 df[MI][KS], ahead[4][KS], hf[4][KS];
#pragma unroll
    for (int mi = 0; mi < MI; ++mi)
#pragma unroll
        for (int s = 0; s < KS; ++s) df[mi][s] = *reinterpret_cast<const bf16x8*>(dt + (int64_t)min(r0 + mi * 16 + fr, kv - 1) * TP + s * 32 + fk * 8);
    auto fetch = [&](int c) {                                        // (columns beyond H: the last ones, never stored)
#pragma unroll
        for (int ni = 0; ni < 4; ++ni)
#pragma unroll
            for (int s = 0; s < KS; ++s) ahead[ni][s] = *reinterpret_cast<const bf16x8*>(hzt + (int64_t)min(c + ni * 16 + fr, H - 1) * TP + s * 32 + fk * 8);
    };
    auto block = [&](int c0, int next) {
        const int c = c0 + wave * 64;
        if constexpr (KS > 2) fetch(c);                              // (no registers left to be a step ahead)
#pragma unroll
        for (int ni = 0; ni < 4; ++ni)
#pragma unroll
            for (int s = 0; s < KS; ++s) hf[ni][s] = ahead[ni][s];
        if constexpr (KS <= 2) fetch(next + wave * 64);
#pragma unroll
        for (int mi = 0; mi < MI; ++mi) {
#pragma unroll
            for (int ni = 0; ni < 4; ++ni) {
                f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = 0; s < KS; ++s) acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hf[ni][s], df[mi][s], acc, 0, 0, 0);
                if constexpr (OUT_BF16) {
                    uint2 pk;
                    pk.x = f2bf2(acc[0], acc[1]); pk.y = f2bf2(acc[2], acc[3]);
                    *reinterpret_cast<uint2*>(img + (mi * 16 + fr) * VH_ROWB + (wave * 64 + ni * 16 + fk * 4) * 2) = pk;
                } else {
                    const int v = r0 + mi * 16 + fr, n = c + ni * 16 + fk * 4;
                    if (v >= kv || n >= H) continue;
                    float4* q = reinterpret_cast<float4*>(dwf + (int64_t)v * lddw + n);
                    float4 o = make_float4(acc[0], acc[1], acc[2], acc[3]);
                    if constexpr (ACCUM) { const float4 b = *q; o.x += b.x; o.y += b.y; o.z += b.z; o.w += b.w; }
                    *q = o;
                }
            }
        }
        if constexpr (OUT_BF16) {
            __syncthreads();
            const int col = (threadIdx.x & 31) * 8;
#pragma unroll
            for (int i = 0; i < 2 * MI; ++i) {
                const int row = i * 8 + (threadIdx.x >> 5);
                if (r0 + row < kv && c0 + col < H)
                    __builtin_nontemporal_store(*reinterpret_cast<const f32x4*>(img + row * VH_ROWB + col * 2), reinterpret_cast<f32x4*>(dwb + (int64_t)(r0 + row) * lddw + c0 + col));
            }
            __syncthreads();
        }
    };
    if constexpr (KS <= 2) {                                         // each workgroup starts at another column block
        const int nc = (H + 255) >> 8;
        int c0 = (blockIdx.x % nc) << 8;
        fetch(c0 + wave * 64);
        for (int i = 0; i < nc; ++i) {
            const int next = c0 + 256 < H ? c0 + 256 : 0;
            block(c0, next);
            c0 = next;
        }
    } else {
        for (int c0 = 0; c0 < H; c0 += 256) block(c0, 0);
    }
}

// dw for 129 .. 256 rows (T64 = 32 KS): as above the write of dw next to few products per value, but the operands are too long to come straight from
// the caches for every wave.  A workgroup owns 256 vocabulary rows, 64 per wave, whose d stays in registers for the whole walk; the hidden states
// come 64 columns at a time, [T64][64], through LDS for all four waves.  Both are contraction-major as they lie in memory, so fragments are LDS
// transpose reads: image of 128-byte rows, 32-byte chunk c of row r at position c ^ f(r), f(r) = ((r >> 1) & 1) | ((r >> 3) & 1) << 1, which
// gives the eight rows that a half wave touches eight places of the 256-byte bank row.  Two workgroups per CU: one stores while the other multiplies.
// Bound: the write of dw and, next to it, the copies of hz that every workgroup repeats (200 x 3584 x 152 064 270 us = 4.0 TB/s written; 150 x 2048 x
// 151 936 180 us = 3.5, 215 before each workgroup started at another column block).
__device__ __forceinline__ void vh_tr_frag4(uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, bf16x8 (&f)[4]) {
    union Frag { bf16x8 v; s16x4_t h[2]; } x[4];
    // reads and their wait in one statement; rows +4 .. +7 of a fragment lie 512 bytes on
    asm volatile("ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:512\n\tds_read_b64_tr_b16 %2, %9\n\tds_read_b64_tr_b16 %3, %9 offset:512\n\t"
                 "ds_read_b64_tr_b16 %4, %10\n\tds_read_b64_tr_b16 %5, %10 offset:512\n\tds_read_b64_tr_b16 %6, %11\n\tds_read_b64_tr_b16 %7, %11 offset:512\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(x[0].h[0]), "=&v"(x[0].h[1]), "=&v"(x[1].h[0]), "=&v"(x[1].h[1]), "=&v"(x[2].h[0]), "=&v"(x[2].h[1]), "=&v"(x[3].h[0]), "=&v"(x[3].h[1])
                 : "v"(a0), "v"(a1), "v"(a2), "v"(a3)
                 : "memory");
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = x[i].v;
}

template <int KS, bool OUT_BF16, bool ACCUM>
__global__ __launch_bounds__(256, OUT_BF16 ? 2 : 1) void head_dw_mid_kernel(const uint16_t* __restrict__ d, int64_t ldd, const uint16_t* __restrict__ hz, int kv, int H,
                                                            int cols_per, uint16_t* __restrict__ dwb, float* __restrict__ dwf, int64_t lddw) {
    constexpr int T64 = KS * 32, TB = T64 * 128, RB = 64 * 2 + 16;       // TB: bytes of a [T64][64] image; RB: row of the output image
    extern __shared__ __attribute__((aligned(16))) char smem[];
    const int lane = threadIdx.x & 63, fr = lane & 15, fk = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r0 = blockIdx.x * 256;
    // copy of 8 image rows: lane -> row (lane >> 3), 16-byte piece lane & 7: half (lane & 1) of the chunk at position (lane & 7) >> 1
    const int cr = lane >> 3;
    auto col_of = [&](int row) { return (((((lane & 7) >> 1) ^ (((row >> 1) & 1) | (((row >> 3) & 1) << 1))) << 4) | ((lane & 1) << 3)); };
    uint32_t tr[4];                                                  // fragment address of 16-column chunk i, k-rows fk*8 ..
    {
        const int row = fk * 8 + (fr >> 2), f = ((row >> 1) & 1) | (((row >> 3) & 1) << 1);
        // rows +4 .. +7 keep f: bits 1 and 3 of the row do not change below a multiple of 8 but for bit 2
#pragma unroll
        for (int i = 0; i < 4; ++i) tr[i] = (uint32_t)(uintptr_t)smem + row * 128 + ((i ^ f) << 5) + (lane & 3) * 8;
    }
    bf16x8 df[KS][4];
    for (int wv = 0; wv < 4; ++wv) {                                 // d of each wave's 64 vocabulary rows in turn through the image
        if (wv) __syncthreads();
        for (int j = wave; j < T64 / 8; j += 4) {
            const int row = j * 8 + cr;
            st_glds16(d + (int64_t)row * ldd + min(r0 + wv * 64 + col_of(row), (int)ldd - 8), smem + j * 1024);
        }
        vh_wait_vm<0>();
        __syncthreads();
        if (wv == wave)
#pragma unroll
            for (int s = 0; s < KS; ++s) vh_tr_frag4(tr[0] + s * 4096, tr[1] + s * 4096, tr[2] + s * 4096, tr[3] + s * 4096, df[s]);
    }
    char* img = smem + TB;
    const int first = blockIdx.y * cols_per, nc = (min(H, first + cols_per) - first) >> 6;
    for (int i = 0, b = (int)blockIdx.x % nc; i < nc; ++i, b = b + 1 < nc ? b + 1 : 0) {   // each workgroup starts at another column block
        const int c0 = first + b * 64;
        __syncthreads();                                             // every wave has read the image (and stored its part of the output)
        for (int j = wave; j < T64 / 8; j += 4) {
            const int row = j * 8 + cr;
            st_glds16(hz + (int64_t)row * H + c0 + col_of(row), smem + j * 1024);
        }
        vh_wait_vm<0>();
        __syncthreads();
        f32x4 acc[4][4];                                             // [vocabulary tile][column tile]
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            bf16x8 hf[4];
            vh_tr_frag4(tr[0] + s * 4096, tr[1] + s * 4096, tr[2] + s * 4096, tr[3] + s * 4096, hf);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hf[j], df[s][i], acc[i][j], 0, 0, 0);
        }
        if constexpr (OUT_BF16) {                                    // a wave's 64 x 64 tile through its own part of the output image
            char* my = img + wave * 64 * RB;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint2 pk;
                    pk.x = f2bf2(acc[i][j][0], acc[i][j][1]); pk.y = f2bf2(acc[i][j][2], acc[i][j][3]);
                    *reinterpret_cast<uint2*>(my + (i * 16 + fr) * RB + (j * 16 + fk * 4) * 2) = pk;
                }
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int row = k * 8 + cr, v = r0 + wave * 64 + row;
                const f32x4 o = *reinterpret_cast<const f32x4*>(my + row * RB + (lane & 7) * 16);
                if (v < kv) __builtin_nontemporal_store(o, reinterpret_cast<f32x4*>(dwb + (int64_t)v * lddw + c0 + (lane & 7) * 8));
            }
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int v = r0 + wave * 64 + i * 16 + fr;
                if (v >= kv) continue;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float4* q = reinterpret_cast<float4*>(dwf + (int64_t)v * lddw + c0 + j * 16 + fk * 4);
                    float4 o = make_float4(acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]);
                    if constexpr (ACCUM) { const float4 b = *q; o.x += b.x; o.y += b.y; o.z += b.z; o.w += b.w; }
                    *q = o;
                }
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------------------------------------------
// Distillation from k teacher log-probs per row.
// ------------------------------------------------------------------------------------------------------------------------------------
#define VH_MAX_K 1024

#define VH_FEW 128                                                   // rows up to which the weight stream bounds the products
#define VH_MAX_V (1 << 21)                                           // column tiles fit the counters of head_bucket_kernel

// teacher probabilities of one row, by one wave: p_k of present entries (0 <= id < V), 0 for the others; log p_k = a_k - shift
struct VhTeacher { float shift, total; };
__device__ __forceinline__ VhTeacher vh_teacher(const int32_t* __restrict__ ids, const float* __restrict__ a, int K, int V, bool renorm, int lane) {
    VhTeacher r = {0.f, 0.f};
    if (renorm) {                                                    // log p = a - log sum_k exp a over the present entries
        float m = -INFINITY, s = 0.f;
        bool nan = false;                                            // (fmaxf passes NaN over)
        for (int k = lane; k < K; k += 64) if (ids[k] >= 0 && ids[k] < V) { m = fmaxf(m, a[k]); nan = nan || a[k] != a[k]; }
        m = wave_max(m);
        if (__any(nan)) { r.shift = r.total = NAN; return r; }
        if (m == -INFINITY) return r;                                // nothing present (or only zero probabilities): the row takes no part
        for (int k = lane; k < K; k += 64) if (ids[k] >= 0 && ids[k] < V) s += vh_exp2((a[k] - m) * VH_LOG2E);
        s = wave_sum(s);
        r.shift = m + log2f(s) * VH_LN2;
        r.total = 1.f;
        return r;
    }
    float s = 0.f;
    for (int k = lane; k < K; k += 64) if (ids[k] >= 0 && ids[k] < V) s += vh_exp2(a[k] * VH_LOG2E);
    r.total = wave_sum(s);
    return r;
}

// The targets of each 256-row tile, sorted by 256-column tile (counting sort in LDS): one workgroup per row tile.  The order inside a list depends on
// LDS atomics, its use does not: every entry writes a place of its own.  Absent entries get z2 = 0 here.
__global__ __launch_bounds__(1024) void head_bucket_kernel(const int32_t* __restrict__ ids, int K, int* __restrict__ start, uint32_t* __restrict__ list,
                                                          float* __restrict__ z2, int T, int V, int tiles_n) {
    extern __shared__ int bin[];                                     // tiles_n counters, then 16 wave totals
    int* wave_total = bin + tiles_n;
    const int r0 = blockIdx.x * 256, n = min(256, T - r0) * K, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    ids += (int64_t)r0 * K; z2 += (int64_t)r0 * K;
    start += (int64_t)blockIdx.x * (tiles_n + 1);
    const int base = blockIdx.x * 256 * K;                           // <= 2^31: T * K is checked on the host
    for (int i = threadIdx.x; i < tiles_n; i += 1024) bin[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += 1024) {
        const int32_t id = ids[i];
        if (id >= 0 && id < V) atomicAdd(&bin[id >> 8], 1);
        else z2[i] = 0.f;
    }
    __syncthreads();
    // exclusive prefix sums, 1024 bins at a time
    int run = base;
    for (int b0 = 0; b0 < tiles_n; b0 += 1024) {
        const int b = b0 + threadIdx.x, c = b < tiles_n ? bin[b] : 0;
        int x = c;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) { const int y = __shfl_up(x, o, 64); x += lane >= o ? y : 0; }
        if (lane == 63) wave_total[wave] = x;
        __syncthreads();
        int before = run, total = 0;
#pragma unroll
        for (int wv = 0; wv < 16; ++wv) { before += wv < wave ? wave_total[wv] : 0; total += wave_total[wv]; }
        if (b < tiles_n) { bin[b] = before + x - c; start[b] = before + x - c; }
        run += total;
        __syncthreads();
    }
    if (threadIdx.x == 0) start[tiles_n] = run;
    for (int i = threadIdx.x; i < n; i += 1024) {
        const int32_t id = ids[i];
        if (id >= 0 && id < V) list[atomicAdd(&bin[id >> 8], 1)] = (uint32_t)(i / K) | (uint32_t)(id & 255) << 8 | (uint32_t)(i % K) << 16;
    }
}

// (The kernels of targets only, from here to head_sparse_kernel, take 4 to 15 us each up to 4096 x 64 targets: launches and latency.)
// kl and log q of every row, one wave per row: logq[t][k] (in: z2 of the target, out: natural log q; 0 for absent entries)
__global__ __launch_bounds__(256) void head_kl_kernel(const int32_t* __restrict__ ids, const float* __restrict__ a, int K, int renorm,
                                                     const float2* __restrict__ stat, float* __restrict__ logq, float* __restrict__ kl, int T, int V) {
    const int lane = threadIdx.x & 63, t = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= T) return;
    ids += (int64_t)t * K; a += (int64_t)t * K; logq += (int64_t)t * K;
    const VhTeacher th = vh_teacher(ids, a, K, V, renorm, lane);
    const float2 st = stat[t];
    float s = 0.f;
    for (int k = lane; k < K; k += 64) {
        const bool have = ids[k] >= 0 && ids[k] < V;
        const float q = have ? ((logq[k] - st.x) - st.y) * VH_LN2 : 0.f;
        logq[k] = q;
        const float lp = a[k] - th.shift, p = have && th.total != 0.f ? vh_exp2(lp * VH_LOG2E) : 0.f;
        if (p != 0.f) s += p * (lp - q);                             // a zero probability contributes nothing, whatever its logarithm
    }
    s = wave_sum(s);
    if (lane == 0) kl[t] = s;
}

__global__ __launch_bounds__(128) void head_rows_kl_kernel(const uint16_t* __restrict__ h, int64_t ldh, const int32_t* __restrict__ ids,
                                                          const float* __restrict__ a, int K, int renorm, const float* __restrict__ lse,
                                                          const float* __restrict__ logq, const float* __restrict__ g, float inv_temp,
                                                          VhRow* __restrict__ rows, float* __restrict__ scale, uint16_t* __restrict__ hz, uint16_t* __restrict__ hzt, int TP,
                                                          int T, int V, int H) {
    const int t = blockIdx.x, lane = threadIdx.x & 63;
    VhRow ri = {0.f, 0.f, 0.f, -1};
    float sc = 1.f;
    if (t < T) {
        ids += (int64_t)t * K; a += (int64_t)t * K; logq += (int64_t)t * K;
        const VhTeacher th = vh_teacher(ids, a, K, V, renorm, lane);
        const float gt = g[t] * inv_temp;
        if (th.total != 0.f && gt != 0.f) {
            float top = 0.f, val = 0.f, energy = 0.f;                // the target with the largest gradient, and the sum of the squares
            for (int k = lane; k < K; k += 64)
                if (ids[k] >= 0 && ids[k] < V) {
                    const float x = gt * (th.total * vh_exp2(logq[k] * VH_LOG2E) - vh_exp2((a[k] - th.shift) * VH_LOG2E));
                    energy += x * x;
                    if (fabsf(x) > top) { top = fabsf(x); val = x; }
                }
            energy = wave_sum(energy);
            const float most = wave_max(top);
            const unsigned long long who = __ballot(top == most);
            val = __shfl(val, who ? __ffsll(who) - 1 : 0, 64);
            if (most * most > 0.5f * energy && most < INFINITY) sc = val;
            ri.c = gt * th.total / sc;
            ri.lse2 = lse[t] * VH_LOG2E;
        }
        if (threadIdx.x == 0) { rows[t] = ri; scale[t] = sc; }
    }
    vh_pack_row(h, ldh, hz, hzt, TP, t, ri.c != 0.f, sc, H);
}

// d' at the targets of a piece [v0, v0 + kv): overwritten with the whole value (c / P) (P q - sum of the p of this id), from the fp32
// log q of the forward pass.  An id that a row holds twice gets the sum of its probabilities from both entries: the same value twice.
__global__ __launch_bounds__(256) void head_sparse_kernel(const int32_t* __restrict__ ids, const float* __restrict__ a, int K, int renorm,
                                                         const float* __restrict__ logq, const VhRow* __restrict__ rows, int v0, int kv,
                                                         uint16_t* __restrict__ d, int64_t ldd, uint16_t* __restrict__ dt, int TP, int T, int V) {
    const int lane = threadIdx.x & 63, t = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (t >= T) return;
    ids += (int64_t)t * K; a += (int64_t)t * K; logq += (int64_t)t * K;
    const VhTeacher th = vh_teacher(ids, a, K, V, renorm, lane);
    const float c = rows[t].c;                                       // g/temperature P / scale
    if (c == 0.f) return;                                            // the row's d is zero
    const float r = c / th.total;
    for (int k = lane; k < K; k += 64) {
        const int32_t id = ids[k];
        if (id < v0 || id >= v0 + kv) continue;
        float p = 0.f;
        for (int j = 0; j < K; ++j) if (ids[j] == id) p += vh_exp2((a[j] - th.shift) * VH_LOG2E);
        const uint16_t x = f2bf(r * (th.total * vh_exp2(logq[k] * VH_LOG2E) - p));
        d[(int64_t)t * ldd + id - v0] = x;
        if (dt) dt[(int64_t)(id - v0) * TP + t] = x;
    }
}

__global__ __launch_bounds__(256) void head_zero_kernel(char* __restrict__ p, int64_t pitch_bytes, int64_t row_bytes) {
    for (int64_t i = threadIdx.x * 8; i < row_bytes; i += 256 * 8) *reinterpret_cast<uint2*>(p + (int64_t)blockIdx.x * pitch_bytes + i) = make_uint2(0, 0);
}

// ------------------------------------------------------------------------------------------------------------------------------------
// host side
// ------------------------------------------------------------------------------------------------------------------------------------
namespace {
struct Plan {                                                        // workspace layout (byte offsets) and piece / slice counts of one call
    int T64, TP, pieces, piece, split, split_both;                               // TP: row pitch of the transposed operands of head_dw_few_kernel
    int64_t part, zlab, stat, start, list, fwd_bytes;
    int64_t rows, scale, hz, hzt, d, dt, slab, bwd_bytes;
    bool few;                                                        // the weight-streaming kernels
};
int64_t up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }

Plan head_plan(int T, int V, int H, int K) {                         // K: targets per row of the distillation, 0: labels
    Plan p;
    p.T64 = (int)up(T, 64);
    p.few = T <= VH_FEW;
    p.TP = T <= 32 ? 32 : p.T64;
    const int64_t n_parts = 2 * (int64_t)st_cdiv(V, 256);
    p.part = 0;
    p.zlab = up(n_parts * T * 8, 256);
    p.stat = p.zlab + up((int64_t)T * 4, 256);
    p.start = p.stat + up((int64_t)T * 8, 256);
    p.list = p.start + (K ? up((int64_t)st_cdiv(T, 256) * (st_cdiv(V, 256) + 1) * 4, 256) : 0);
    p.fwd_bytes = p.list + up((int64_t)T * K * 4, 256);
    // d of one piece: at most 512 MiB; beyond 2^20 rows the 256 columns (or the fewer that there are) of one tile
    const int64_t max_cols = std::max<int64_t>(256, ((int64_t)512 << 20) / 2 / p.T64 / 256 * 256);
    p.pieces = st_cdiv(V, max_cols);
    p.piece = (int)up(st_cdiv(V, p.pieces), 256);
    p.pieces = st_cdiv(V, p.piece);
    // dh: K-slices so that few row tiles still fill the CUs (whole rounds of a tile's K-steps + ~14 of prologue / epilogue)
    const int tiles = st_cdiv(T, 256) * st_cdiv(H, 256), ncu = st_num_cus(), nkt = st_cdiv(std::min(V, p.piece), 64);
    p.split = 1;
    if (p.few) p.split = std::max(1, std::min({2 * ncu / tiles, nkt / 8, 64}));       // two workgroups per CU, at least 16 steps of 32 each
    int64_t best = INT64_MAX;
    for (int s = 1; s <= 32 && !p.few; ++s) {
        if (s > 1 && (nkt / s < 8 || (int64_t)s * T * H * 4 > ((int64_t)512 << 20))) break;
        const int64_t cost = (int64_t)st_cdiv((int64_t)tiles * s, ncu) * (st_cdiv(nkt, s) + 14) + 2 * s;
        if (cost < best) { best = cost; p.split = s; }
    }
    // beside dw in one launch: no slice longer than half of what a CU has to do (~8 and ~14 K-steps for the rest of a dw and a dh tile).  That ends below
    // some 2.2 tiles per CU and one slab more (150 MiB and one T x H): the slabs need no limit of their own
    p.split_both = 1;
    if (!p.few) {
        const int64_t dw_steps = (int64_t)st_cdiv(std::min(V, p.piece), 256) * st_cdiv(H, 256) * (p.T64 / 64 + 8);
        while (p.split_both < 32 && nkt / (p.split_both + 1) >= 8 &&
               2 * (int64_t)(st_cdiv(nkt, p.split_both) + 14) * ncu > (int64_t)tiles * (nkt + 14 * p.split_both) + dw_steps)
            ++p.split_both;
    }
    p.rows = 0;
    p.scale = up((int64_t)T * (int64_t)sizeof(VhRow), 256);
    p.hz = p.scale + up((int64_t)T * 4, 256);
    p.hzt = p.hz;                                                    // one of the two
    const int64_t d_bytes = up((int64_t)p.T64 * std::min<int64_t>(p.piece, up(V, 64)) * 2, 256);        // the largest row pitch of d is that of the first piece
    p.d = p.hz + up((int64_t)p.T64 * H * 2, 256);
    p.dt = p.d + d_bytes;
    p.slab = p.dt + (p.few ? d_bytes : 0);
    p.bwd_bytes = p.slab + up((int64_t)std::max(p.split, p.split_both) * T * H * 4, 256);
    return p;
}

bool operands_ok(const void* h, int64_t ldh, const void* w, int64_t ldw, int T, int V, int H, float inv_temp) {
    return h && w && T >= 0 && V > 0 && V <= VH_MAX_V && H > 0 && H % 64 == 0 && !(ldh & 7) && !(ldw & 7) && ldh >= H && ldw >= H && ldh < (1 << 22) && ldw < (1 << 22) &&
           !(((uintptr_t)h) & 15) && !(((uintptr_t)w) & 15) && inv_temp > 0.f && inv_temp * VH_LOG2E < INFINITY && (int64_t)st_cdiv(T, 256) * st_cdiv(V, 256) < (1 << 30);
}

// one attribute per kernel and device, set before its first launch there
template <auto KERN> void allow_lds(int bytes = VH_SMEM) {
    static bool done[64] = {};
    int dev = 0;
    hipGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !done[dev]) {
        hipFuncSetAttribute((const void*)KERN, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (dev >= 0 && dev < 64) done[dev] = true;
    }
}

// one launch of the few-row tile: T <= 32, 64, 96, 128 or 160 rows
constexpr int VH_STREAM = 160;
int few_cols(int T) { return T <= 64 ? 128 : 256; }                  // vocabulary columns of a workgroup
template <bool DLOGITS, int MT, int SLOTS, int WAVES, class... A>
int launch_few_as(int V, hipStream_t s, A... args) {
    constexpr int BT = 16 * MT, BN = 32 * WAVES, RING = SLOTS * (BN + BT) * 128;
    constexpr int IMAGES = DLOGITS ? BT * (BN * 2 + 16) + (MT <= 8 ? BN * (BT * 2 + 16) : 0) : std::max(BT * (128 * 4 + 16), WAVES * BT * 8);
    constexpr int SMEM = std::max(RING, IMAGES);
    static_assert(SMEM <= 160 * 1024, "the ring and the epilogue's images share the LDS of a CU");
    allow_lds<head_few_kernel<MT, SLOTS, WAVES, DLOGITS>>(SMEM);
    hipLaunchKernelGGL((head_few_kernel<MT, SLOTS, WAVES, DLOGITS>), dim3(st_cdiv(V, BN)), dim3(64 * WAVES), SMEM, s, args...);
    ST_CHECK_LAUNCH();
    return 0;
}
template <bool DLOGITS, class... A>
int launch_few(int T, int V, hipStream_t s, A... args) {
    if (T <= 32) return launch_few_as<DLOGITS, 2, 4, 4>(V, s, args...);
    if (T <= 64) return launch_few_as<DLOGITS, 4, 3, 4>(V, s, args...);
    if (T <= 96) return launch_few_as<DLOGITS, 6, 3, 8>(V, s, args...);
    if (T <= 128) return launch_few_as<DLOGITS, 8, 3, 8>(V, s, args...);
    return launch_few_as<DLOGITS, 10, 3, 8>(V, s, args...);
}

int head_stats(const uint16_t* h, int64_t ldh, const uint16_t* w, int64_t ldw, const int64_t* labels, float sc, float* logp, float* lse, VhTargets tg,
               float* z, int64_t ldz, char* ws, const Plan& p, int T, int V, int H, hipStream_t s) {
    const int tm = st_cdiv(T, 256), tn = st_cdiv(V, 256);
    float2* part = (float2*)(ws + p.part);
    float* zlab = (float*)(ws + p.zlab);
    int n_parts = 2 * tn;
    if (T <= VH_STREAM) {
        n_parts = st_cdiv(V, few_cols(T));
        const int rc = launch_few<false>(T, V, s, h, ldh, w, ldw, T, V, H, sc, labels, part, zlab, tg, (const VhRow*)nullptr, 0, (uint16_t*)nullptr,
                                         (int64_t)0, (uint16_t*)nullptr, 0, z, ldz);
        if (rc) return rc;
    } else {
        auto go = [&](auto kern) {
            hipLaunchKernelGGL(kern, dim3(tm * tn), dim3(256), VH_SMEM, s, h, ldh, w, ldw, T, V, H, tm, tn, sc, labels, part, zlab, tg,
                               (const VhRow*)nullptr, 0, (uint16_t*)nullptr, (int64_t)0, 0, z, ldz);
        };
        allow_lds<head_tile_kernel<false, true>>(); allow_lds<head_tile_kernel<false, false>>();
        allow_lds<head_tile_kernel<false, true, true>>(); allow_lds<head_tile_kernel<false, false, true>>();
        if (z) { if (tm == 1) go(head_tile_kernel<false, true, true>); else go(head_tile_kernel<false, false, true>); }
        else if (tm == 1) go(head_tile_kernel<false, true>); else go(head_tile_kernel<false, false>);
        ST_CHECK_LAUNCH();
    }
    if (T <= 512) hipLaunchKernelGGL(head_lse_few_kernel, dim3(T), dim3(1024), 0, s, part, n_parts, zlab, labels, logp, lse, (float2*)(ws + p.stat), T, V);
    else hipLaunchKernelGGL(head_lse_kernel, dim3(st_cdiv(T, 16)), dim3(1024), 0, s, part, n_parts, zlab, labels, logp, lse, (float2*)(ws + p.stat), T, V);
    ST_CHECK_LAUNCH();
    return 0;
}

// (few rows: the whole vocabulary is one piece, so there is nothing to add to)
static_assert(((int64_t)512 << 20) / 2 / VH_FEW >= VH_MAX_V, "few rows need one piece");
int launch_dh_few(const uint16_t* d, int64_t ldd, const uint16_t* w, int64_t ldw, int T, int kv, int H, int tiles_n, const Plan& p, float* slab, hipStream_t s) {
    const int nkt = st_cdiv(kv, 32), per = st_cdiv(nkt, p.split);
    const dim3 grid(tiles_n * st_cdiv(nkt, per));
    auto go = [&](auto kern, int smem) {
        hipLaunchKernelGGL(kern, grid, dim3(256), smem, s, d, ldd, w, ldw, T, kv, H, tiles_n, per, slab);
        ST_CHECK_LAUNCH();
        return 0;
    };
    constexpr int S64 = 4 * (32 * 512 + 64 * 64), S128 = 3 * (32 * 512 + 128 * 64);
    if (p.T64 == 64) {
        allow_lds<head_dh_few_kernel<4, 4>>(S64);
        return go(head_dh_few_kernel<4, 4>, S64);
    }
    allow_lds<head_dh_few_kernel<8, 3>>(S128);
    return go(head_dh_few_kernel<8, 3>, S128);
}

// Column ranges of head_dw_mid_kernel for `blocks` row blocks: the launch takes whole rounds of two workgroups per CU, each as long as its range, so the
// count with the fewest rounds per range, and of equals the lowest (a range loads its d again).  MI355X, dW alone at 150 / 200 rows, us for 1, 2, 3
// ranges: V = 33 001 (129 blocks: 3) H = 2048 82 67 57 / 96 79 66, H = 3584 125 98 80 / 148 117 98; 50 257 (197 blocks: 2) H = 2048 85 77 85 / 99 84 93,
// H = 3584 130 104 121 / 150 124 137; 128 256 (501 blocks: 1) H = 1024 115 103 111 / 125 116 123, H = 2048 164 223 189 / 170 237 208, H = 3584 231 234
// 232 / 274 283 273; 152 064 (594 blocks: 3) H = 2048 221 264 210 / 235 280 230, H = 3584 331 286 273 / 362 338 331.  4 and 6 were nowhere better
// by more than 1 %.
int mid_ranges(int blocks) {
    int best = 1, cost = 6 * st_cdiv(blocks, 2 * st_num_cus());
    for (int n = 2; n <= 3; ++n)
        if (const int c = 6 / n * st_cdiv(blocks * n, 2 * st_num_cus()); c < cost) { cost = c; best = n; }
    return best;
}

// the pieces of a backward pass behind the row coefficients; `sparse` finishes d at the targets of a piece
template <class F>
int head_backward(const uint16_t* h, int64_t ldh, const uint16_t* w, int64_t ldw, float sc, const float* z, int64_t ldz, uint16_t* dh, int64_t lddh, uint16_t* dwb, float* dwf,
                  int64_t lddw, int accumulate, char* ws, const Plan& p, int T, int V, int H, hipStream_t s, F&& sparse) {
    const VhRow* rows = (const VhRow*)(ws + p.rows);
    const uint16_t* hz = (const uint16_t*)(ws + p.hz);
    uint16_t* d = (uint16_t*)(ws + p.d);
    uint16_t* dt = p.few ? (uint16_t*)(ws + p.dt) : nullptr;
    uint16_t* hzt = (uint16_t*)(ws + p.hzt);
    float* slab = (float*)(ws + p.slab);
    const int tm = st_cdiv(T, 256), th = st_cdiv(H, 256);
    const bool mid = !p.few && p.T64 <= 256 && 2 * st_cdiv(p.piece, 256) >= st_num_cus();        // (fewer row blocks: the square tile spreads better)
    const bool both = dh && (dwb || dwf) && !p.few && !mid;
    const int split = both ? p.split_both : p.split;
    allow_lds<head_grads_kernel<true, false, false>>(); allow_lds<head_grads_kernel<true, false, true>>();
    allow_lds<head_grads_kernel<false, false, false>>(); allow_lds<head_grads_kernel<false, false, true>>();
    allow_lds<head_grads_kernel<false, true, false>>(); allow_lds<head_grads_kernel<false, true, true>>();
    allow_lds<head_tile_kernel<true, true>>(); allow_lds<head_tile_kernel<true, false>>();
    allow_lds<head_dh_kernel<false, true>>(); allow_lds<head_dh_kernel<true, true>>(); allow_lds<head_dh_kernel<false, false>>(); allow_lds<head_dh_kernel<true, false>>();
    allow_lds<head_dw_kernel<true, false>>(); allow_lds<head_dw_kernel<false, false>>(); allow_lds<head_dw_kernel<false, true>>();
    for (int i = 0; i < p.pieces; ++i) {
        const int v0 = i * p.piece, kv = std::min(p.piece, V - v0), tn = st_cdiv(kv, 256);
        const int64_t ldd = up(kv, 64);
        const uint16_t* wp = w + (int64_t)v0 * ldw;
        if (z) {
            const dim3 grid(st_cdiv(ldd, 128) * (p.T64 / 64));
            if (p.few) hipLaunchKernelGGL(head_d_kernel<true>, grid, dim3(256), 0, s, z + v0, ldz, rows, T, kv, sc, v0, d, ldd, p.T64, dt, p.TP);
            else hipLaunchKernelGGL(head_d_kernel<false>, grid, dim3(256), 0, s, z + v0, ldz, rows, T, kv, sc, v0, d, ldd, p.T64, dt, p.TP);
            ST_CHECK_LAUNCH();
        } else if (T <= VH_STREAM) {
            const int rc = launch_few<true>(T, kv, s, h, ldh, wp, ldw, T, kv, H, sc, (const int64_t*)nullptr, (float2*)nullptr, (float*)nullptr,
                                            VhTargets{}, rows, v0, d, ldd, dt, p.few ? p.TP : p.T64, (float*)nullptr, (int64_t)0);
            if (rc) return rc;
        } else {
            auto go = [&](auto kern) {
                hipLaunchKernelGGL(kern, dim3(tm * tn), dim3(256), VH_SMEM, s, h, ldh, wp, ldw, T, kv, H, tm, tn, sc, (const int64_t*)nullptr,
                                   (float2*)nullptr, (float*)nullptr, VhTargets{}, rows, v0, d, ldd, p.T64, (float*)nullptr, (int64_t)0);
            };
            if (tm == 1) go(head_tile_kernel<true, true>); else go(head_tile_kernel<true, false>);
            ST_CHECK_LAUNCH();
        }
        const int rc = sparse(v0, kv, d, ldd, dt);
        if (rc) return rc;
        const int tv = st_cdiv(kv, 256), nkt = st_cdiv(kv, 64), slices = st_cdiv(nkt, st_cdiv(nkt, split));      // (a short last piece may fill fewer slices)
        uint16_t* ob = dwb ? dwb + (int64_t)v0 * lddw : nullptr;
        float* of = dwf ? dwf + (int64_t)v0 * lddw : nullptr;
        if (both) {
            const int dh_blocks = tm * th * slices;
            const dim3 grid(dh_blocks + tv * th);
            auto go = [&](auto kern) {
                hipLaunchKernelGGL(kern, grid, dim3(256), VH_SMEM, s, d, ldd, wp, ldw, hz, T, p.T64, kv, H, tm, tv, th, split, dh_blocks, slab, ob, of, lddw);
            };
            if (dwb) { if (i == 0) go(head_grads_kernel<true, false, false>); else go(head_grads_kernel<true, false, true>); }
            else if (accumulate) { if (i == 0) go(head_grads_kernel<false, true, false>); else go(head_grads_kernel<false, true, true>); }
            else { if (i == 0) go(head_grads_kernel<false, false, false>); else go(head_grads_kernel<false, false, true>); }
            ST_CHECK_LAUNCH();
            continue;
        }
        if (dh && p.few) {
            const int rc = launch_dh_few(d, ldd, wp, ldw, T, kv, H, th, p, slab, s);
            if (rc) return rc;
        } else if (dh) {
            const dim3 grid(tm * th * slices);
            auto go = [&](auto kern) { hipLaunchKernelGGL(kern, grid, dim3(256), VH_SMEM, s, d, ldd, wp, ldw, T, kv, H, tm, th, split, slab); };
            if (tm == 1) { if (i == 0) go(head_dh_kernel<false, true>); else go(head_dh_kernel<true, true>); }
            else { if (i == 0) go(head_dh_kernel<false, false>); else go(head_dh_kernel<true, false>); }
            ST_CHECK_LAUNCH();
        }
        if (dwb || dwf) {
            const dim3 grid(tv * th);
            if (p.few) {
                const dim3 few_grid(st_cdiv(kv, 128));
#define VH_DW_FEW(KS, OB, AC) hipLaunchKernelGGL((head_dw_few_kernel<KS, OB, AC>), few_grid, dim3(256), 0, s, dt, hzt, kv, H, ob, of, lddw)
                if (p.TP == 32) { if (dwb) VH_DW_FEW(1, true, false); else if (accumulate) VH_DW_FEW(1, false, true); else VH_DW_FEW(1, false, false); }
                else if (p.TP == 64) { if (dwb) VH_DW_FEW(2, true, false); else if (accumulate) VH_DW_FEW(2, false, true); else VH_DW_FEW(2, false, false); }
                else { if (dwb) VH_DW_FEW(4, true, false); else if (accumulate) VH_DW_FEW(4, false, true); else VH_DW_FEW(4, false, false); }
#undef VH_DW_FEW
            }
            else if (mid) {
                const int smem = p.T64 * 128 + 4 * 64 * 144, mid_cols = (int)up(st_cdiv(H, mid_ranges(tv)), 64);
#define VH_DW_MID(KS, OB, AC) do { allow_lds<head_dw_mid_kernel<KS, OB, AC>>(smem); \
        hipLaunchKernelGGL((head_dw_mid_kernel<KS, OB, AC>), dim3(tv, st_cdiv(H, mid_cols)), dim3(256), smem, s, d, ldd, hz, kv, H, mid_cols, ob, of, lddw); } while (0)
                if (p.T64 == 192) { if (dwb) VH_DW_MID(6, true, false); else if (accumulate) VH_DW_MID(6, false, true); else VH_DW_MID(6, false, false); }
                else { if (dwb) VH_DW_MID(8, true, false); else if (accumulate) VH_DW_MID(8, false, true); else VH_DW_MID(8, false, false); }
#undef VH_DW_MID
            }
            else if (dwb) hipLaunchKernelGGL((head_dw_kernel<true, false>), grid, dim3(256), VH_SMEM, s, d, ldd, hz, p.T64, kv, H, tv, th, ob, of, lddw);
            else if (accumulate) hipLaunchKernelGGL((head_dw_kernel<false, true>), grid, dim3(256), VH_SMEM, s, d, ldd, hz, p.T64, kv, H, tv, th, ob, of, lddw);
            else hipLaunchKernelGGL((head_dw_kernel<false, false>), grid, dim3(256), VH_SMEM, s, d, ldd, hz, p.T64, kv, H, tv, th, ob, of, lddw);
            ST_CHECK_LAUNCH();
        }
    }
    if (dh) {
        const int nkt = st_cdiv(std::min(V, p.piece), p.few ? 32 : 64), slices = st_cdiv(nkt, st_cdiv(nkt, split));
        hipLaunchKernelGGL(head_dh_finish_kernel, dim3(st_cdiv((int64_t)T * H, 1024)), dim3(256), 0, s, slab, slices, (const float*)(ws + p.scale), dh, lddh, T, H);
        ST_CHECK_LAUNCH();
    }
    return 0;
}

bool grads_ok(const void* dh, int64_t lddh, const void* dwb, const void* dwf, int64_t lddw, int accumulate, int H) {
    if (dh && ((((uintptr_t)dh) & 7) || (lddh & 3) || lddh < H)) return false;
    if (dwb && (dwf || accumulate || (((uintptr_t)dwb) & 15) || (lddw & 7) || lddw < H)) return false;
    if (dwf && ((((uintptr_t)dwf) & 15) || (lddw & 3) || lddw < H)) return false;
    return true;
}

bool logits_ok(const float* z, int64_t ldz, int V) { return !z || (!(((uintptr_t)z) & 15) && !(ldz & 3) && ldz >= up(V, 64)); }

// no rows: dW is a sum over nothing
int empty_dw(uint16_t* dwb, float* dwf, int64_t lddw, int accumulate, int V, int H, hipStream_t s) {
    if (accumulate || (!dwb && !dwf)) return 0;
    const int64_t e = dwb ? 2 : 4;
    hipLaunchKernelGGL(head_zero_kernel, dim3(V), dim3(256), 0, s, dwb ? (char*)dwb : (char*)dwf, lddw * e, (int64_t)H * e);
    ST_CHECK_LAUNCH();
    return 0;
}
}  // namespace

extern "C" {

int st_linear_head_workspace_bytes(int T, int V, int H, int K, int backward, int64_t* bytes_host, st_stream_t stream) {
    (void)stream;
    if (T < 0 || K < 0 || K > VH_MAX_K || V <= 0 || V > VH_MAX_V || H <= 0 || H % 64 || !bytes_host) return ST_EINVAL;
    const Plan p = head_plan(std::max(T, 1), V, H, K);
    *bytes_host = backward ? p.bwd_bytes : p.fwd_bytes;
    return 0;
}

int st_linear_logprob_fwd(const st_bf16* hidden, int64_t ldh, const st_bf16* weight, int64_t ldw, const int64_t* labels, float inv_temperature,
                          float* logp, float* lse, float* logits, int64_t ldz, void* workspace, int64_t workspace_bytes, int T, int V, int H,
                          st_stream_t stream) {
    if (T == 0) return V > 0 && H > 0 && H % 64 == 0 ? 0 : ST_EINVAL;
    if (!operands_ok(hidden, ldh, weight, ldw, T, V, H, inv_temperature) || !labels || !logp || !lse || !logits_ok(logits, ldz, V)) return ST_EINVAL;
    const Plan p = head_plan(T, V, H, 0);
    if (!workspace || (((uintptr_t)workspace) & 15) || workspace_bytes < p.fwd_bytes) return ST_EINVAL;
    return head_stats(hidden, ldh, weight, ldw, labels, inv_temperature * VH_LOG2E, logp, lse, VhTargets{}, logits, ldz, (char*)workspace, p, T, V, H,
                      (hipStream_t)stream);
}

int st_linear_logprob_bwd(const st_bf16* hidden, int64_t ldh, const st_bf16* weight, int64_t ldw, const int64_t* labels, const float* logp, const float* lse,
                          const float* g, float inv_temperature, const float* logits, int64_t ldz, st_bf16* dhidden, int64_t lddh, st_bf16* dweight_bf16,
                          float* dweight_f32, int64_t lddw, int accumulate, void* workspace, int64_t workspace_bytes, int T, int V, int H, st_stream_t stream) {
    hipStream_t s = (hipStream_t)stream;
    if (V <= 0 || H <= 0 || H % 64 || T < 0 || !grads_ok(dhidden, lddh, dweight_bf16, dweight_f32, lddw, accumulate, H)) return ST_EINVAL;
    if (T == 0) return empty_dw(dweight_bf16, dweight_f32, lddw, accumulate, V, H, s);
    if (!operands_ok(hidden, ldh, weight, ldw, T, V, H, inv_temperature) || !labels || !logp || !lse || !g || !logits_ok(logits, ldz, V)) return ST_EINVAL;
    const Plan p = head_plan(T, V, H, 0);
    if (!workspace || (((uintptr_t)workspace) & 15) || workspace_bytes < p.bwd_bytes) return ST_EINVAL;
    char* ws = (char*)workspace;
    hipLaunchKernelGGL(head_rows_label_kernel, dim3(p.few ? p.TP : p.T64), dim3(128), 0, s, hidden, ldh, labels, logp, lse, g, inv_temperature, (VhRow*)(ws + p.rows),
                       (float*)(ws + p.scale), p.few ? nullptr : (uint16_t*)(ws + p.hz), (uint16_t*)(ws + p.hzt), p.TP, T, V, H);
    ST_CHECK_LAUNCH();
    return head_backward(hidden, ldh, weight, ldw, inv_temperature * VH_LOG2E, logits, ldz, dhidden, lddh, dweight_bf16, dweight_f32, lddw, accumulate, ws, p, T, V, H, s,
                         [](int, int, uint16_t*, int64_t, uint16_t*) { return 0; });
}

int st_linear_topk_kl_fwd(const st_bf16* hidden, int64_t ldh, const st_bf16* weight, int64_t ldw, const int32_t* ids, const float* teacher_logp, int K,
                          int renormalize, float inv_temperature, float* kl, float* lse, float* logq, float* logits, int64_t ldz, void* workspace,
                          int64_t workspace_bytes, int T, int V, int H, st_stream_t stream) {
    if (K <= 0 || K > VH_MAX_K || (int64_t)T * K > INT32_MAX) return ST_EINVAL;
    if (T == 0) return V > 0 && H > 0 && H % 64 == 0 ? 0 : ST_EINVAL;
    if (!operands_ok(hidden, ldh, weight, ldw, T, V, H, inv_temperature) || !ids || !teacher_logp || !kl || !lse || !logq || !logits_ok(logits, ldz, V)) return ST_EINVAL;
    const Plan p = head_plan(T, V, H, K);
    if (!workspace || (((uintptr_t)workspace) & 15) || workspace_bytes < p.fwd_bytes) return ST_EINVAL;
    hipStream_t s = (hipStream_t)stream;
    const float sc = inv_temperature * VH_LOG2E;
    char* ws = (char*)workspace;
    int* start = (int*)(ws + p.start);
    uint32_t* list = (uint32_t*)(ws + p.list);
    const int tn = st_cdiv(V, 256);
    hipLaunchKernelGGL(head_bucket_kernel, dim3(st_cdiv(T, 256)), dim3(1024), (tn + 16) * 4, s, ids, K, start, list, logq, T, V, tn);
    ST_CHECK_LAUNCH();
    const int rc = head_stats(hidden, ldh, weight, ldw, nullptr, sc, nullptr, lse, VhTargets{start, list, logq, K}, logits, ldz, ws, p, T, V, H, s);
    if (rc) return rc;
    hipLaunchKernelGGL(head_kl_kernel, dim3(st_cdiv(T, 4)), dim3(256), 0, s, ids, teacher_logp, K, renormalize,
                       (const float2*)(ws + p.stat), logq, kl, T, V);
    ST_CHECK_LAUNCH();
    return 0;
}

int st_linear_topk_kl_bwd(const st_bf16* hidden, int64_t ldh, const st_bf16* weight, int64_t ldw, const int32_t* ids, const float* teacher_logp, int K,
                          int renormalize, float inv_temperature, const float* lse, const float* logq, const float* g, const float* logits, int64_t ldz,
                          st_bf16* dhidden, int64_t lddh, st_bf16* dweight_bf16, float* dweight_f32, int64_t lddw, int accumulate, void* workspace,
                          int64_t workspace_bytes, int T, int V, int H, st_stream_t stream) {
    hipStream_t s = (hipStream_t)stream;
    if (K <= 0 || K > VH_MAX_K || V <= 0 || H <= 0 || H % 64 || T < 0 || !grads_ok(dhidden, lddh, dweight_bf16, dweight_f32, lddw, accumulate, H))
        return ST_EINVAL;
    if (T == 0) return empty_dw(dweight_bf16, dweight_f32, lddw, accumulate, V, H, s);
    if (!operands_ok(hidden, ldh, weight, ldw, T, V, H, inv_temperature) || !ids || !teacher_logp || !lse || !logq || !g || !logits_ok(logits, ldz, V)) return ST_EINVAL;
    const Plan p = head_plan(T, V, H, 0);
    if (!workspace || (((uintptr_t)workspace) & 15) || workspace_bytes < p.bwd_bytes) return ST_EINVAL;
    char* ws = (char*)workspace;
    hipLaunchKernelGGL(head_rows_kl_kernel, dim3(p.few ? p.TP : p.T64), dim3(128), 0, s, hidden, ldh, ids, teacher_logp, K, renormalize, lse, logq, g, inv_temperature,
                       (VhRow*)(ws + p.rows), (float*)(ws + p.scale), p.few ? nullptr : (uint16_t*)(ws + p.hz), (uint16_t*)(ws + p.hzt), p.TP, T, V, H);
    ST_CHECK_LAUNCH();
    return head_backward(hidden, ldh, weight, ldw, inv_temperature * VH_LOG2E, logits, ldz, dhidden, lddh, dweight_bf16, dweight_f32, lddw, accumulate, ws, p, T, V, H, s,
                         [&](int v0, int kv, uint16_t* d, int64_t ldd, uint16_t* dt) -> int {
                             hipLaunchKernelGGL(head_sparse_kernel, dim3(st_cdiv(T, 4)), dim3(256), 0, s, ids, teacher_logp, K, renormalize, logq,
                                                (const VhRow*)(ws + p.rows), v0, kv, d, ldd, dt, p.TP, T, V);
                             ST_CHECK_LAUNCH();
                             return 0;
                         });
}

}  // extern "C"

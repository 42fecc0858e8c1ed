// gemm_asm4_core.h — the hand-scheduled K loop of the 256x256x64, four-wave bf16 tile (its structure and measurements: gemm_asm4.hip), as a
// device function that leaves the accumulators in registers.  The GEMM kernels (gemm_asm4.hip) and the vocabulary-head kernels
// (vocab_head.hip) put their own epilogues behind it.
#pragma once
#include "common.h"
#include <type_traits>

typedef int i32x4 __attribute__((ext_vector_type(4)));

// compile-time loop: the body receives std::integral_constant<int, I> — every index below is a constant expression, so register
// arrays are addressed statically (a loop the optimizer declines to unroll would turn them into indexed VGPR / scratch accesses)
template <int I, int N, class F> __device__ __forceinline__ void static_for(F&& f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        static_for<I + 1, N>(f);
    }
}

#define A4_BM 256
#define A4_BN 256
#define A4_SLOT 65536          // one K-tile of both operands: (256 + 256) rows x 128 bytes
#define A4_ABYTES 32768

__device__ __forceinline__ void a4_mfma(f32x4& acc, const bf16x8& b, const bf16x8& a) {
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(b), "v"(a));
}
// the same with the 8 wait states its result needs before anything but another MFMA may touch it (a4_mainloop, GUARD)
__device__ __forceinline__ void a4_mfma_wait(f32x4& acc, const bf16x8& b, const bf16x8& a) {
    asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0\n\ts_nop 7" : "+a"(acc) : "v"(b), "v"(a));
}
template <int OFF> __device__ __forceinline__ void a4_read(bf16x8& f, uint32_t addr) {
    asm volatile("ds_read_b128 %0, %1 offset:%2" : "=v"(f) : "v"(addr), "i"(OFF) : "memory");
}
__device__ __forceinline__ void a4_dma(uint32_t voff, i32x4 srd, uint32_t soff) {
    asm volatile("buffer_load_dwordx4 %0, %1, %2 offen lds" : : "v"(voff), "s"(srd), "s"(soff) : "memory");
}
// K-major operand fragment: 4 consecutive k of one m per lane (gfx950 LDS transpose read), two of them make an MFMA operand
template <int OFF> __device__ __forceinline__ void a4_read_tr(s16x4_t& f, uint32_t addr) {
    asm volatile("ds_read_b64_tr_b16 %0, %1 offset:%2" : "=v"(f) : "v"(addr), "i"(OFF) : "memory");
}
__device__ __forceinline__ void a4_dma0(uint32_t voff, i32x4 srd) {        // the K-tile offset sits in the resource's base address
    asm volatile("buffer_load_dwordx4 %0, %1, 0 offen lds" : : "v"(voff), "s"(srd) : "memory");
}
// the same two with the non-temporal policy: an operand that ONE workgroup reads, once
__device__ __forceinline__ void a4_dma_nt(uint32_t voff, i32x4 srd, uint32_t soff) {
    asm volatile("buffer_load_dwordx4 %0, %1, %2 offen nt lds" : : "v"(voff), "s"(srd), "s"(soff) : "memory");
}
__device__ __forceinline__ void a4_dma0_nt(uint32_t voff, i32x4 srd) {
    asm volatile("buffer_load_dwordx4 %0, %1, 0 offen nt lds" : : "v"(voff), "s"(srd) : "memory");
}
__device__ __forceinline__ void a4_flip(uint32_t& addr) { asm volatile("v_xor_b32 %0, 0x10000, %0" : "+v"(addr)); }
__device__ __forceinline__ void a4_m0_set(uint32_t v) { asm volatile("s_mov_b32 m0, %0" : : "s"(v) : "memory"); }
__device__ __forceinline__ void a4_m0_next() { asm volatile("s_add_u32 m0, m0, 0x400" : : : "memory", "scc"); }
__device__ __forceinline__ void a4_barrier() { asm volatile("s_barrier" : : : "memory"); }
__device__ __forceinline__ void a4_wait_lgkm0() { asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory"); }
template <int N> __device__ __forceinline__ void a4_wait_lgkm() {          // LDS reads return in order: "at most N still outstanding"
    if constexpr (N == 0) asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    else if constexpr (N == 6) asm volatile("s_waitcnt lgkmcnt(6)" ::: "memory");
    else if constexpr (N == 7) asm volatile("s_waitcnt lgkmcnt(7)" ::: "memory");
    else if constexpr (N == 9) asm volatile("s_waitcnt lgkmcnt(9)" ::: "memory");
    else if constexpr (N == 12) asm volatile("s_waitcnt lgkmcnt(12)" ::: "memory");
    else if constexpr (N == 15) asm volatile("s_waitcnt lgkmcnt(15)" ::: "memory");
    else static_assert(N < 0, "add the lgkmcnt literal");
}
template <int N> __device__ __forceinline__ void a4_wait_vm() {
    if constexpr (N == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    else if constexpr (N == 9) asm volatile("s_waitcnt vmcnt(9)" ::: "memory");
    else if constexpr (N == 10) asm volatile("s_waitcnt vmcnt(10)" ::: "memory");
    else if constexpr (N == 12) asm volatile("s_waitcnt vmcnt(12)" ::: "memory");
    else if constexpr (N == 16) asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
    else static_assert(N < 0, "add the vmcnt literal");
}

// acc[ni][mi] of this wave: rows m0 + wm*128 + mi*16 + (lane & 15), columns n0 + wn*128 + ni*16 + (lane >> 4)*4 + r of A B^T, summed over the
// `nk` K-tiles from K-tile kt0 on (wm = wave >> 1, wn = wave & 1; SWIGLU: see gemm_asm4.hip).  M, N: valid rows of A and B (rows beyond
// compute values that must not be used; contraction-major operands need M % 8 == 0 resp. N % 8 == 0).
// AS / BS: the operand is stored contraction-major.  KCLAMP (with BS): B has only k_rows valid k-rows; k-rows beyond read the last valid
// one, so the A operand has to hold zeros there (the K-tiles are whole).  LDS: two 64-KiB operand slots at smem; on return no copy is in
// flight for this wave, but other waves may still read the slots: __syncthreads() before they are reused.
// GUARD: the compiler's hazard recogniser cannot see that the asm MFMAs write late, and behind the loop it may move accumulators between registers
// before the wait that stands there (an fp32 epilogue got the old value of the last accumulator in half of its lanes).  With GUARD the last MFMA
// of every K-tile waits in its own statement: 1 % of the loop.  check_mfma_waits.py looks through the built code of every kernel and fails the
// build where a result is touched too early; kernels that it names are built with GUARD, the others need not pay for it.
// BNT: B streams with the non-temporal policy (one row tile: no other workgroup reads its rows).
template <bool AS, bool BS, bool SWIGLU, int DBG = 0, bool KCLAMP = false, bool GUARD = false, bool BNT = false>
__device__ __forceinline__ void a4_mainloop(char* smem, const uint16_t* __restrict__ A, int64_t lda, const uint16_t* __restrict__ B, int64_t ldb, int m0,
                                            int n0, int M, int N, int kt0, int nk, int k_rows, f32x4 (&acc)[8][8]) {
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave >> 1, wn = wave & 1;
    // ---- buffer resources: base = first row of the tile, num_records cuts the rows beyond the matrix (they load as zero)
    static_assert(!(AS || BS) || !SWIGLU, "contraction-major operands: plain results");
    static_assert(!KCLAMP || BS, "KCLAMP limits the k-rows of a contraction-major B");
    // AS / BS: the operand is stored CONTRACTION-MAJOR (A[k][m], lda = pitch of a k-row): dX = dY W reads W that way (BS), dW = dY^T X
    // both operands (AS + BS).  Its K-tile is staged as [64 k-rows][256 m] (512-byte rows) and read with the LDS transpose read.
    uint64_t a_base = AS ? (uint64_t)(A + m0) : (uint64_t)(A + (int64_t)m0 * lda);
    const int rows_a = min(A4_BM, M - m0);
    i32x4 srdA, srdB, srdB2;
    srdA.x = __builtin_amdgcn_readfirstlane((int)(uint32_t)a_base);
    srdA.y = __builtin_amdgcn_readfirstlane((int)(uint32_t)((a_base >> 32) & 0xffffu));
    srdA.z = (int)0xffffffffu;                                       // rows are clamped per lane: nothing to cut off
    srdA.w = 0x00020000;
    const int cols_b = SWIGLU ? min(A4_BN / 2, N - n0) : min(A4_BN, N - n0);        // B rows (= output columns) this tile owns
    uint64_t b_base = BS ? (uint64_t)(B + n0) : (uint64_t)(B + (int64_t)n0 * ldb);
    srdB.x = __builtin_amdgcn_readfirstlane((int)(uint32_t)b_base);
    srdB.y = __builtin_amdgcn_readfirstlane((int)(uint32_t)((b_base >> 32) & 0xffffu));
    srdB.z = (int)0xffffffffu;
    srdB.w = 0x00020000;
    srdB2 = srdB;
    if constexpr (SWIGLU) {                                          // the up-projection rows follow the N gate rows
        const uint64_t u_base = (uint64_t)(B + (int64_t)(n0 + N) * ldb);
        srdB2.x = __builtin_amdgcn_readfirstlane((int)(uint32_t)u_base);
        srdB2.y = __builtin_amdgcn_readfirstlane((int)(uint32_t)((u_base >> 32) & 0xffffu));
    }
    // source offset of copy j of this wave, per lane: row (lane >> 3) of the copy's 8 rows — clamped to the last valid row of the
    // tile, such rows compute values that are never stored — and the 16-byte chunk (lane & 7) ^ row (the swizzle, on the source).
    // These 16 registers are constant over the K loop: the K-tile offset goes through the instruction's SGPR offset.
    uint32_t voffA[8], voffB[8];
    static_for<0, 8>([&](auto jc) {
        constexpr int j = decltype(jc)::value;
        const int rl = lane >> 3, ch = ((lane & 7) ^ rl) << 4;
        // contraction-major image: copy j of this wave = k-rows kr = wave*16 + 2j + (lane >> 5); the 32-byte chunk c (16 m) of k-row kr
        // sits at chunk position c ^ g(kr) (gemm_tile_kernel.h, AS / BS): lane piece sl covers m = ((sl >> 1) ^ g) * 16 + (sl & 1) * 8 ..+7;
        // columns past the matrix edge are clamped (they compute values that are never stored)
        const int kr = wave * 16 + j * 2 + (lane >> 5), sl = lane & 31, g = (kr & 3) | (((kr >> 3) & 1) << 2);
        const int lc = (((sl >> 1) ^ g) << 4) + (sl & 1) * 8;
        if constexpr (AS) voffA[j] = (uint32_t)kr * (uint32_t)(lda * 2) + (uint32_t)min(lc, rows_a - 8) * 2u;
        else {
            const int ra = min(wave * 64 + j * 8 + rl, rows_a - 1);
            voffA[j] = (uint32_t)ra * (uint32_t)(lda * 2) + ch;
        }
        if constexpr (BS) voffB[j] = (uint32_t)kr * (uint32_t)(ldb * 2) + (uint32_t)min(lc, cols_b - 8) * 2u;
        else {
            const int r = wave * 64 + j * 8 + rl;                    // tile row (SWIGLU: tile rows alternate 16 gate / 16 up rows)
            const int src = min(SWIGLU ? ((r >> 5) * 16 + (r & 15)) : r, cols_b - 1);
            voffB[j] = (uint32_t)src * (uint32_t)(ldb * 2) + ch;
        }
    });
    uint32_t koff = 0;                                               // byte offset of the K-tile the next copies fetch (SGPR)
    const uint32_t smem32 = (uint32_t)(uintptr_t)smem;
    const uint32_t m0A = __builtin_amdgcn_readfirstlane(smem32 + wave * 8 * 1024);
    const uint32_t m0B = __builtin_amdgcn_readfirstlane(smem32 + A4_ABYTES + wave * 8 * 1024);

#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

    if (kt0 > 0) {                                                   // a K-slice: start at its first K-tile
        koff = (uint32_t)kt0 * 128u;
        if constexpr (AS) a_base += (uint64_t)kt0 * 64u * (uint64_t)lda * 2u;
        if constexpr (BS) b_base += (uint64_t)kt0 * 64u * (uint64_t)ldb * 2u;
    }
    // contraction-major operands advance their resource's BASE by 64 k-rows per K-tile (the 32-bit offsets could not span a
    // [tokens][vocabulary] operand); row-major ones keep the base and move the SGPR offset by 128 bytes
    const uint64_t stepA = (uint64_t)lda * 128u, stepB = (uint64_t)ldb * 128u;
    auto set_base = [&](i32x4& srd, uint64_t base) {
        srd.x = __builtin_amdgcn_readfirstlane((int)(uint32_t)base);
        srd.y = __builtin_amdgcn_readfirstlane((int)(uint32_t)((base >> 32) & 0xffffu));
    };
    if constexpr (AS) set_base(srdA, a_base);
    if constexpr (BS) set_base(srdB, b_base);
    int kt_next = kt0;                                               // KCLAMP: the K-tile the next copies fetch
    auto clamp_tail = [&]() {                                        // the last, partial K-tile: k-rows beyond the matrix read its last row
        if constexpr (KCLAMP) {
            const int rem = k_rows - kt_next * 64;
            if (rem < 64)
                static_for<0, 8>([&](auto jc) {
                    constexpr int j = decltype(jc)::value;
                    const int kr = wave * 16 + j * 2 + (lane >> 5), sl = lane & 31, g = (kr & 3) | (((kr >> 3) & 1) << 2);
                    const int lc = (((sl >> 1) ^ g) << 4) + (sl & 1) * 8;
                    voffB[j] = (uint32_t)min(kr, rem - 1) * (uint32_t)(ldb * 2) + (uint32_t)min(lc, cols_b - 8) * 2u;
                });
        }
    };
    clamp_tail();
    auto advance = [&](bool go) {                                    // the K-tile the NEXT copies fetch
        if constexpr (KCLAMP) { kt_next += go ? 1 : 0; clamp_tail(); }
        koff += go ? 128u : 0u;
        if constexpr (AS) { a_base += go ? stepA : 0; set_base(srdA, a_base); }
        if constexpr (BS) { b_base += go ? stepB : 0; set_base(srdB, b_base); }
    };
    // fragment addresses: row = wave tile base + i*16 + (lane & 15), 16-byte chunk (s*4 + lane>>4) ^ (row & 7)
    const int frow = lane & 15, fk = lane >> 4;
    // fragment read addresses; the two LDS slots are 64 KiB apart, so "the other slot" is an XOR with 0x10000: the k-step-1 reads of
    // tile t go to its slot (adK1), the k-step-0 reads of tile t+1 to the other one (adK0n); both flip after every tile
    uint32_t adA_k1, adB_k1, adA_k0n, adB_k0n;
    {
        const int kc0 = fk ^ (frow & 7), kc1 = (4 + fk) ^ (frow & 7);
        adA_k1 = smem32 + (wm * 128 + frow) * 128 + (kc1 << 4);
        adB_k1 = smem32 + A4_ABYTES + (wn * 128 + frow) * 128 + (kc1 << 4);
        adA_k0n = smem32 + A4_SLOT + (wm * 128 + frow) * 128 + (kc0 << 4);
        adB_k0n = smem32 + A4_SLOT + A4_ABYTES + (wn * 128 + frow) * 128 + (kc0 << 4);
    }
    bf16x8 af[2][8], bfr[2][8];
    // contraction-major fragments: m = chunk*16 + (lane & 15) with chunk = 8*w + i, k = (lane >> 4)*8 + 0..7 as two transpose reads
    // (k-rows +0..3 and +4..7 = 2048 bytes further).  Chunk c of k-row r sits at position c ^ g(r); for the rows a lane addresses
    // g = tr_g, so fragment i needs its own per-lane address (i ^ tr_g) << 5: 8 registers per operand, pointing at the slot of the
    // tile whose k-step 1 is read next; they flip ONCE per tile, between the k-step-1 reads (tile t) and the k-step-0 reads (t+1).
    uint32_t trA[8], trB[8];
    union Frag { bf16x8 v; s16x4_t h[2]; };
    if constexpr (AS || BS) {
        const int tr_g = ((lane >> 2) & 3) | (((lane >> 4) & 1) << 2);
        const int tr_row = (lane >> 4) * 8 + ((lane & 15) >> 2);
        static_for<0, 8>([&](auto ic) {
            constexpr int i = decltype(ic)::value;
            trA[i] = smem32 + tr_row * 512 + wm * 256 + ((i ^ tr_g) << 5) + (lane & 3) * 8;
            trB[i] = smem32 + A4_ABYTES + tr_row * 512 + wn * 256 + ((i ^ tr_g) << 5) + (lane & 3) * 8;
        });
    }
    auto rd_tr = [&](bf16x8& f, uint32_t addr, auto s2c, auto hc) {  // half h of the fragment of k-step s2
        constexpr int s2 = decltype(s2c)::value, h = decltype(hc)::value;
        a4_read_tr<s2 * 16384 + h * 2048>(reinterpret_cast<Frag&>(f).h[h], addr);
    };

    auto dma_tile = [&](auto jc) {                                   // copy j of the NEXT issue (voff already points at its K-tile)
        constexpr int j = decltype(jc)::value;
        if constexpr (j < 8) { if constexpr (AS) a4_dma0(voffA[j], srdA); else a4_dma(voffA[j], srdA, koff); }
        else if constexpr (BS && BNT) a4_dma0_nt(voffB[j - 8], srdB);
        else if constexpr (BS) a4_dma0(voffB[j - 8], srdB);
        else if constexpr (BNT) a4_dma_nt(voffB[j - 8], srdB, koff);
        else if (SWIGLU && (((wave * 64 + (j - 8) * 8) >> 4) & 1)) a4_dma(voffB[j - 8], srdB2, koff);
        else a4_dma(voffB[j - 8], srdB, koff);
    };
    // i < 8: A fragment i, else B fragment i - 8 (16 rows = 2048 bytes apart)
    auto rd_k1 = [&](auto i_c) {
        constexpr int i = decltype(i_c)::value;
        if constexpr (i < 8) a4_read<i * 2048>(af[1][i], adA_k1);
        else a4_read<(i - 8) * 2048>(bfr[1][i - 8], adB_k1);
    };
    auto rd_k0n = [&](auto i_c) {                                    // order of issue: A0..A7, B0 first (the next tile's first MFMAs need them)
        constexpr int i = decltype(i_c)::value;
        if constexpr (i < 8) a4_read<i * 2048>(af[0][i], adA_k0n);
        else a4_read<(i - 8) * 2048>(bfr[0][i - 8], adB_k0n);
    };
    // contraction-major kernels: read number r of a k-step, A first (AS: 16 transpose reads, else 8 ds_read_b128), then B
    constexpr int NRA = AS ? 16 : 8, NRB = BS ? 16 : 8, NRD = NRA + NRB;
    auto rd_km = [&](auto r_c, auto s2c) {
        constexpr int r = decltype(r_c)::value, s2 = decltype(s2c)::value;
        if constexpr (r < NRA) {
            if constexpr (AS) rd_tr(af[s2][r >> 1], trA[r >> 1], s2c, std::integral_constant<int, (r & 1)>{});
            else if constexpr (s2 == 1) a4_read<r * 2048>(af[1][r], adA_k1);
            else a4_read<r * 2048>(af[0][r], adA_k0n);
        } else {
            constexpr int q = r - NRA;
            if constexpr (BS) rd_tr(bfr[s2][q >> 1], trB[q >> 1], s2c, std::integral_constant<int, (q & 1)>{});
            else if constexpr (s2 == 1) a4_read<q * 2048>(bfr[1][q], adB_k1);
            else a4_read<q * 2048>(bfr[0][q], adB_k0n);
        }
    };
    uint32_t m0A_cur = m0A, m0B_cur = m0B;                           // LDS-DMA destination of the tile being refilled (slot of tile t)

    // ---- prologue: tiles 0 and 1 in flight, fragments of (0, k-step 0) in registers
    a4_m0_set(m0A);
    static_for<0, 16>([&](auto jc) {
        if constexpr (decltype(jc)::value == 8) a4_m0_set(m0B);
        dma_tile(jc);
        a4_m0_next();
    });
    advance(nk > 1);
    a4_m0_set(m0A + A4_SLOT);
    static_for<0, 16>([&](auto jc) {                                 // (nk == 1: tile 0 once more — keeps the loop's counted waits uniform)
        if constexpr (decltype(jc)::value == 8) a4_m0_set(m0B + A4_SLOT);
        dma_tile(jc);
        a4_m0_next();
    });
    advance(nk > 2);
    a4_wait_vm<16>();
    a4_barrier();
    if constexpr (AS || BS) {                                        // (0, k-step 0) from slot 0: where the transpose-read addresses point
        adA_k0n ^= A4_SLOT; adB_k0n ^= A4_SLOT;
        static_for<0, NRD>([&](auto rc) { rd_km(rc, std::integral_constant<int, 0>{}); });
        adA_k0n ^= A4_SLOT; adB_k0n ^= A4_SLOT;
        a4_wait_lgkm<0>();
    } else {                                                         // (0, k-step 0) sits in slot 0 = "the other slot" of the flipped addresses
        adA_k0n ^= A4_SLOT; adB_k0n ^= A4_SLOT;
        static_for<0, 16>([&](auto ic) { rd_k0n(ic); });
        adA_k0n ^= A4_SLOT; adB_k0n ^= A4_SLOT;
        a4_wait_lgkm<7>();
    }

    // ---- one K-tile: 128 MFMA slots; every other instruction sits between two of them
    //   slot   0..63  MFMAs of k-step 0          64..127  MFMAs of k-step 1
    //   1..16          the 16 fragment reads of k-step 1 (this tile's slot), one per MFMA
    //   7,15,23        counted lgkmcnt waits: B fragments 1..7 of k-step 0 were issued LAST in the previous tile and land now
    //   30 / 31        lgkmcnt(0) + barrier #1: every wave is done reading this tile's slot
    //   33..123        the 16 LDS-DMA copies of tile t+2 into that slot, one every SIXTH MFMA: an issue costs the wave ~30-55 cycles of
    //                  MFMA issue time (measured by elimination, tools/gemm_ksweep.py debug), the more the closer the four waves' copies
    //                  follow each other through the CU's one texture addresser — so they are spread over the whole rest of the tile
    //   104 / 105      vmcnt(12) + barrier #2: tile t+1 has landed for every wave (12 copies of tile t+2 issued so far stay in flight;
    //                  the last four go out behind this barrier and are covered by the next tile's wait)
    //   106..121       the 16 fragment reads of (t+1, k-step 0): A0..A7, B0, then B1..B7; lgkmcnt(7) closes the tile
    // Contraction-major kernels (NRD = 24 or 32 reads per k-step, one per MFMA slot):
    //   1..NRD               reads of (t, k-step 1)
    //   NRD+1..NRD+16        the transpose-read addresses flip to the other slot (one v_xor per slot)
    //   NRD+14 / NRD+15      lgkmcnt(0) + barrier #1
    //   NRD+17 ..            the 16 copies of tile t+2, one every 4th (NRD = 32) / 5th (24) MFMA
    //   114-NRD / 115-NRD    vmcnt (the copies issued so far stay in flight) + barrier #2
    //   116-NRD..115         reads of (t+1, k-step 0); lgkmcnt(0) at 126
    constexpr int KM_DMA0 = NRD + 17, KM_STRIDE = NRD == 32 ? 4 : 5, KM_VM = 114 - NRD, KM_RD0 = 116 - NRD;
    constexpr int KM_INFLIGHT = (KM_VM - KM_DMA0 + KM_STRIDE - 1) / KM_STRIDE;      // copies of tile t+2 issued before the vmcnt wait
    static_assert(!(AS || BS) || (KM_INFLIGHT == (NRD == 32 ? 9 : 10) && KM_DMA0 + 15 * KM_STRIDE < 127), "contraction-major schedule");
    for (int kt = 0; kt < nk; ++kt) {
        if constexpr (AS || BS) {
            static_for<0, 128>([&](auto ic) {
                constexpr int sl = decltype(ic)::value;
                constexpr int ks = sl >> 6, idx = sl & 63;
                if constexpr (GUARD && sl == 127) a4_mfma_wait(acc[7][7], bfr[1][7], af[1][7]);
            else a4_mfma(acc[idx >> 3][idx & 7], bfr[ks][idx >> 3], af[ks][idx & 7]);
                if constexpr (sl >= 1 && sl <= NRD) rd_km(std::integral_constant<int, (sl - 1)>{}, std::integral_constant<int, 1>{});
                if constexpr (sl > NRD && sl <= NRD + 16) {
                    constexpr int x = sl - NRD - 1;
                    if constexpr (x < 8) { if constexpr (AS) a4_flip(trA[x]); } else { if constexpr (BS) a4_flip(trB[x - 8]); }
                }
                if constexpr (sl == NRD + 14) a4_wait_lgkm<0>();
                if constexpr (sl == NRD + 15) a4_barrier();
                if constexpr (sl == KM_DMA0 - 1) a4_m0_set(m0A_cur);
                if constexpr (sl >= KM_DMA0 && sl <= KM_DMA0 + 15 * KM_STRIDE && (sl - KM_DMA0) % KM_STRIDE == 0) dma_tile(std::integral_constant<int, ((sl - KM_DMA0) / KM_STRIDE)>{});
                if constexpr (sl > KM_DMA0 && sl <= KM_DMA0 + 15 * KM_STRIDE && (sl - KM_DMA0 - 1) % KM_STRIDE == 0 && (sl - KM_DMA0 - 1) / KM_STRIDE != 7 && (sl - KM_DMA0 - 1) / KM_STRIDE < 15) a4_m0_next();
                if constexpr (sl == KM_DMA0 + 7 * KM_STRIDE + 2) a4_m0_set(m0B_cur);     // after the 8th A copy, before the first B copy
                if constexpr (sl == KM_VM) a4_wait_vm<KM_INFLIGHT>();
                if constexpr (sl == KM_VM + 1) a4_barrier();
                if constexpr (sl >= KM_RD0 && sl < KM_RD0 + NRD) rd_km(std::integral_constant<int, (sl - KM_RD0)>{}, std::integral_constant<int, 0>{});
                if constexpr (sl == 126) a4_wait_lgkm<0>();
            });
        } else
        static_for<0, 128>([&](auto ic) {
            constexpr int sl = decltype(ic)::value;
            constexpr int ks = sl >> 6, idx = sl & 63;
            if constexpr (GUARD && sl == 127) a4_mfma_wait(acc[7][7], bfr[1][7], af[1][7]);
            else a4_mfma(acc[idx >> 3][idx & 7], bfr[ks][idx >> 3], af[ks][idx & 7]);
            constexpr bool RD = DBG != 3 && DBG != 4, BAR = DBG != 2 && DBG != 4, DMA = DBG != 1 && DBG != 4;
            if constexpr (sl == 7) a4_wait_lgkm<12>();           // before MFMA 8 (B1): B2..B7 + the 6 k-step-1 reads issued so far
            if constexpr (sl == 15) a4_wait_lgkm<15>();          // B2 (the counter saturates at 15: at least the 5 oldest of <= 20 are done)
            if constexpr (sl == 23) a4_wait_lgkm<15>();          // B3..B7: the 6 oldest of the <= 21 then outstanding
            if constexpr (RD && sl >= 1 && sl <= 16) rd_k1(std::integral_constant<int, (sl - 1)>{});
            if constexpr (sl == 30) a4_wait_lgkm<0>();
            if constexpr (BAR && sl == 31) a4_barrier();
            if constexpr (DMA) {
                if constexpr (sl == 32) a4_m0_set(m0A_cur);
                if constexpr (sl >= 33 && sl <= 123 && (sl - 33) % 6 == 0) dma_tile(std::integral_constant<int, ((sl - 33) / 6)>{});
                if constexpr (sl >= 34 && sl <= 123 && (sl - 34) % 6 == 0 && (sl - 34) / 6 != 7 && (sl - 34) / 6 < 15) a4_m0_next();
                if constexpr (sl == 78) a4_m0_set(m0B_cur);      // after the 8th A copy (slot 75), before the first B copy (slot 81)
                if constexpr (sl == 104) a4_wait_vm<12>();
            }
            if constexpr (BAR && sl == 105) a4_barrier();
            if constexpr (RD && sl >= 106 && sl <= 121) rd_k0n(std::integral_constant<int, (sl - 106)>{});
            if constexpr (sl == 127) a4_wait_lgkm<7>();
        });
        // flip the slots; advance the source of the next copies (the last two tiles re-fetch tile nk-1: lands in a slot nobody reads)
        adA_k1 ^= A4_SLOT; adB_k1 ^= A4_SLOT; adA_k0n ^= A4_SLOT; adB_k0n ^= A4_SLOT;
        m0A_cur ^= A4_SLOT; m0B_cur ^= A4_SLOT;
        advance(kt + 3 < nk);
    }
    a4_wait_vm<0>();                                                 // the two re-fetched tiles are still landing
    a4_wait_lgkm<0>();
    // (a second guard: every accumulator passes THROUGH a wait on its way to the epilogue)
#pragma unroll
    for (int ni = 0; ni < 8; ++ni)
        asm volatile("s_nop 7" : "+a"(acc[ni][0]), "+a"(acc[ni][1]), "+a"(acc[ni][2]), "+a"(acc[ni][3]), "+a"(acc[ni][4]), "+a"(acc[ni][5]),
                     "+a"(acc[ni][6]), "+a"(acc[ni][7]));
}

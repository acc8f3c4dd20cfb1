// f8_pp.h - the contraction of f8_tile.h for tiles of 256 rows x 256 queries, scheduled so that the matrix pipe of every SIMD
// is fed without a pause (the schedule of the 16-bit kernel, mfma_pp.hip, with 128-code slabs).  f8_big.h reads and converts less, but there the
// accumulators fill half the registers of a wave that is alone on its SIMD, and a search's filter spills.
//
// Eight waves = two groups of four (group g = waves 4g..4g+3, one wave of each group per SIMD), wave tile 128 rows x 64 queries =
// 4 x 2 accumulators of v_mfma_f32_32x32x16_bf16.  K is walked in PHASES of 64 codes, the operands arrive in slabs of
// 128 (one scale block; 256 rows x 128 B = 32 KiB each) in a ring of two.
//
//   LOAD(p)   p even: issue the eight 1 KiB pieces of slab p/2 + 1; ds_read the fragments of phase p
//             p odd, group 1: s_waitcnt vmcnt(0)
//             s_barrier
//   MFMA(p)   32 MFMAs, and under them the fragments become operands; SCALED: eight of the scaled instruction
//             p odd, group 0: s_waitcnt vmcnt(0)
//             s_barrier
//
// Group 1 runs one barrier behind group 0, so between two barriers one group multiplies while the other reads LDS.  Barrier
// events of group 0: LOAD(p) ends with event 2p, MFMA(p) with 2p+1; group 1 is one event later.
//   RAW  slab D+1 is first read in LOAD(2D+2), which group 0 enters after event 4D+3; every wave waits for its own pieces before
//        that event: group 0 behind MFMA(2D+1), group 1 at the end of LOAD(2D+1).
//   WAR  its slot held slab D-1, last read in LOAD(2D-1): group 0's reads were retired (lgkmcnt) before event 4D-2, group 1's before
//        event 4D-1; the issue in LOAD(2D) follows event 4D-1 (group 0) or 4D (group 1).
// The scale words of four blocks (256 rows x 4 B per operand) ride along: wave w brings 64 of the 512 rows' words with one 4-byte
// piece in every eighth phase, into a ring of two of their own; a lane re-reads its six words when a new group of four begins.
// Slot of group G+1 is written from LOAD(8G) on; it held group G-1, whose words were read into registers in LOAD(8G-8).
#pragma once
#include "f8_tile.h"

namespace ssmi {

// SCALED: sums of the scaled instruction (f8_tile.h), at 1.7 times the speed
template <bool SCALED>
struct F8Pp {
    static constexpr int SLAB = 256 * 128;                // one operand's 128 codes of 256 rows
    static constexpr int SCALES = 4 * SLAB;               // behind the ring: [2][X: 256 words, Q: 256 words]
    static constexpr int LDS = SCALES + 2 * 2048;
    typedef f32x16_t Acc[4][2];

    unsigned char* smem;
    int lane, wave, wm, wn, nblk;
    const unsigned char *xc, *qc, *sc;                    // codes of the tiles; scales of the operand this wave brings
    unsigned xstride, qstride, so;
    int xlast, qlast;

    __device__ __forceinline__ void init(unsigned char* lds, int blocks) {
        smem = lds;
        nblk = blocks;
        lane = threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
        wm = wave >> 2;
        wn = wave & 3;
    }
    // sources of a tile; starts its pipeline (slab 0 and the first scale words).  No wave may still read the ring
    __device__ __forceinline__ void aim(const F8Src& x, const F8Src& q) {
        xstride = x.stride;
        qstride = q.stride;
        xlast = x.last;
        qlast = q.last;
        xc = x.codes;
        qc = q.codes;
        const int r = (wave & 3) * 64 + lane;
        sc = wm ? q.scales : x.scales;
        so = wm ? (unsigned)min(r, q.last) * q.sstride : (unsigned)min(r, x.last) * x.sstride;
        slab(0);
        words(0);
    }
    __device__ __forceinline__ void slab(int d) {
        unsigned char* dst = smem + (d & 1) * SLAB + wave * 4096;
        // (uniform addresses that the compiler may not fold with the lanes' offsets: it would keep the 64-bit sums in registers)
        const unsigned char *xb = xc + (size_t)d * 128, *qb = qc + (size_t)d * 128;
        asm volatile("" : "+s"(xb), "+s"(qb));
        // (offsets made anew for every piece: chunk c of row r0 + 8 j; kept in registers, the search's filter spilled.  Rows < 256 and strides of
        // at most 2^23 bytes: 24 bits)
        int l = lane;
        asm volatile("" : "+v"(l));
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int r = wave * 32 + (j & 3) * 8 + (l >> 3);
            const unsigned chunk = ((l & 7) ^ ((l >> 4) + (j & 1) * 4)) * 16;   // (r >> 1) & 7
            unsigned o = j < 4 ? __umul24((unsigned)min(r, xlast), xstride) + chunk : __umul24((unsigned)min(r, qlast), qstride) + chunk;
            asm volatile("" : "+v"(o));   // (a 32-bit offset, widened here and not ahead of the loop)
            if (j < 4) GLDS16(xb + o, dst + j * 1024);
            else GLDS16(qb + o, dst + 2 * SLAB + (j & 3) * 1024);
        }
    }
    __device__ __forceinline__ void words(int g) { GLDS4(sc + (size_t)g * 4 + so, smem + SCALES + (g & 1) * 2048 + wave * 256); }

    // the tile aimed at last; the ring is free (for the next aim) on return
    __device__ __forceinline__ void run(Acc& acc) {
        const int r32 = lane & 31, hl = lane >> 5;
        const int sw = (r32 >> 1) & 7;
        const int a_row = (wm * 128 + r32) * 128, b_row = 2 * SLAB + (wn * 64 + r32) * 128;
        const int ch[4] = {(hl ^ sw) * 16, ((2 + hl) ^ sw) * 16, ((4 + hl) ^ sw) * 16, ((6 + hl) ^ sw) * 16};
        int sx[4], sq[2];
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        if (wm == 1) __builtin_amdgcn_s_barrier();  // group 1 runs one barrier event behind
        __builtin_amdgcn_sched_barrier(0);
        const auto phase = [&](auto jc, auto hc, int d) __attribute__((always_inline)) {
            constexpr int J = decltype(jc)::value, H = decltype(hc)::value;
            // ---- LOAD ----
            if constexpr (H == 0) {
                if constexpr (J == 0) {   // (before the pieces: the compiler waits for every piece in flight in front of these reads)
                    const int* w = reinterpret_cast<const int*>(smem + SCALES + ((d >> 2) & 1) * 2048);
#pragma unroll
                    for (int m = 0; m < 4; ++m) sx[m] = w[wm * 128 + m * 32 + r32];
#pragma unroll
                    for (int n = 0; n < 2; ++n) sq[n] = w[256 + wn * 64 + n * 32 + r32];
                    asm volatile("" : "+v"(sx[0]), "+v"(sx[1]), "+v"(sx[2]), "+v"(sx[3]), "+v"(sq[0]), "+v"(sq[1])::"memory");
                }
                if (d + 1 < nblk) slab(d + 1);
                if (J == 0 && d + 4 < nblk) words(d / 4 + 1);
            }
            const unsigned char* cur = smem + (J & 1) * SLAB;   // (d & 1 == J & 1)
            i32x8_t a[4], b[2];
#pragma unroll
            for (int n = 0; n < 2; ++n)
                b[n] = join8(*reinterpret_cast<const i32x4_t*>(cur + b_row + n * 4096 + ch[2 * H]), *reinterpret_cast<const i32x4_t*>(cur + b_row + n * 4096 + ch[2 * H + 1]));
#pragma unroll
            for (int m = 0; m < 4; ++m)
                a[m] = join8(*reinterpret_cast<const i32x4_t*>(cur + a_row + m * 4096 + ch[2 * H]), *reinterpret_cast<const i32x4_t*>(cur + a_row + m * 4096 + ch[2 * H + 1]));
            if (H == 1 && wm == 1) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // fragments in registers
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_barrier();
            // ---- MFMA ----
            // (the empty statements hold the products between the barriers: nothing else orders a pure instruction against them)
            asm volatile("" : "+v"(a[0]), "+v"(a[1]), "+v"(a[2]), "+v"(a[3]), "+v"(b[0]), "+v"(b[1]));
            __builtin_amdgcn_s_setprio(1);
            if constexpr (SCALED) {
#pragma unroll
                for (int m = 0; m < 4; ++m)
#pragma unroll
                    for (int n = 0; n < 2; ++n) acc[m][n] = mfma_f8_scaled<J>(a[m], b[n], acc[m][n], sx[m], sq[n]);
            } else {
                float fx[4], fq[2];
#pragma unroll
                for (int m = 0; m < 4; ++m) fx[m] = f8_factor<J>(sx[m]);
#pragma unroll
                for (int n = 0; n < 2; ++n) fq[n] = f8_factor<J>(sq[n]);
#pragma unroll
                for (int e = 0; e < 8; e += 2) {   // 16 codes of K; the conversions go under the products
                    i32x4_t bw[2];
#pragma unroll
                    for (int n = 0; n < 2; ++n) bw[n] = f8_widen(b[n][e], b[n][e + 1], fq[n]);
#pragma unroll
                    for (int m = 0; m < 4; ++m) {
                        const i32x4_t aw = f8_widen(a[m][e], a[m][e + 1], fx[m]);
#pragma unroll
                        for (int n = 0; n < 2; ++n) acc[m][n] = mfma_f8_32(aw, bw[n], acc[m][n]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            asm volatile("" : "+v"(acc[0][0]), "+v"(acc[0][1]), "+v"(acc[1][0]), "+v"(acc[1][1]), "+v"(acc[2][0]), "+v"(acc[2][1]), "+v"(acc[3][0]), "+v"(acc[3][1]));
            __builtin_amdgcn_s_setprio(0);
            __builtin_amdgcn_sched_barrier(0);
            if (H == 1 && wm == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
        };
        const std::integral_constant<int, 0> c0;
        const std::integral_constant<int, 1> c1;
        const std::integral_constant<int, 2> c2;
        const std::integral_constant<int, 3> c3;
#pragma unroll 1
        for (int d = 0; d < nblk; d += 4) {
            phase(c0, c0, d);
            phase(c0, c1, d);
            if (d + 1 < nblk) { phase(c1, c0, d + 1); phase(c1, c1, d + 1); }
            if (d + 2 < nblk) { phase(c2, c0, d + 2); phase(c2, c1, d + 2); }
            if (d + 3 < nblk) { phase(c3, c0, d + 3); phase(c3, c1, d + 3); }
        }
        if (wm == 0) __builtin_amdgcn_s_barrier();  // realign the two groups
    }
};

}  // namespace ssmi

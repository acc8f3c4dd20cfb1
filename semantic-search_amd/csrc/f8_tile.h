// f8_tile.h - contraction of one tile of 8-bit rows with one tile of 8-bit queries on the matrix cores.
//
//   acc[row][query] = sum over blocks b of 2^(sx[row,b] - 127) 2^(sq[query,b] - 127) sum over the 128 codes of b of x q
//
// The operands travel as codes - a quarter of fp32 in memory, half of bf16 in LDS - and become bf16 on their way into the
// instruction: v_cvt_scalef32_pk_bf16_fp8 takes two codes and the power of two of their block, four significant bits fit eight
// (exact from 2^-133 to the end of fp32; scale byte 255 gives NaN), and at 4 cycles a pair it hides under v_mfma_f32_*_bf16.
// Products of such operands are exact and the sums are fp32's: measured, an instruction is off by less than 2^-21.5 of the
// magnitudes it adds, 2^-22 of an accumulator that is large beside them.
// v_mfma_scale_f32_*_f8f6f4, which takes codes and scale bytes as they are at twice the rate (3.9 PFLOP/s on registers, 1.75), aligns the products
// of eight neighbouring codes to the largest of them and drops what lies more than 13 bits below (measured; v_mfma_f32_*_fp8_fp8 does the
// same), so that a strong channel or two large products that cancel take the rest with them.  Only a search that checks what that
// may have cost it uses it (f8_pp.h, f8_search.hip).
#pragma once
#include "f8.h"
#include "mfma_common.h"

namespace ssmi {

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef int i32x2_t __attribute__((ext_vector_type(2)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

// byte J of a word of scales as the power of two it stands for, in the exponent of an fp32 (0 and 255 as f8_pair reads them)
template <int J>
__device__ __forceinline__ float f8_factor(int w) { return __int_as_float((int)(((unsigned)w >> (8 * J)) & 255u) << 23); }
// codes 0, 1 (HI: 2, 3) of a word -> their values as bf16
template <bool HI>
__device__ __forceinline__ int f8_pair(int w, float s) {
    return __builtin_bit_cast(int, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((unsigned)w, s, HI));
}
// eight codes of a lane -> an operand
__device__ __forceinline__ i32x4_t f8_widen(int lo, int hi, float s) {
    return i32x4_t{f8_pair<false>(lo, s), f8_pair<true>(lo, s), f8_pair<false>(hi, s), f8_pair<true>(hi, s)};
}
__device__ __forceinline__ f32x4_t mfma_f8(const i32x4_t& a, const i32x4_t& b, const f32x4_t& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16_t mfma_f8_32(const i32x4_t& a, const i32x4_t& b, const f32x16_t& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
// ... and with the scaled instruction: 64 codes of K
template <int J>
__device__ __forceinline__ f32x16_t mfma_f8_scaled(const i32x8_t& a, const i32x8_t& b, const f32x16_t& c, int sa, int sb) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, J, sa, J, sb);
}
__device__ __forceinline__ i32x8_t join8(const i32x4_t& lo, const i32x4_t& hi) {
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}
// accumulators of whatever extent, zero
template <typename V, int M, int N>
__device__ __forceinline__ void zero_acc(V (&acc)[M][N]) {
#pragma unroll
    for (int m = 0; m < M; ++m)
#pragma unroll
        for (int n = 0; n < N; ++n) acc[m][n] = V(0.f);
}

// One operand's tile: rows of a plain matrix or of one segment of a row store (uniform base, 32-bit offsets).
struct F8Src {
    const unsigned char* codes;   // row 0 of the tile
    const unsigned char* scales;
    unsigned stride, sstride;     // bytes
    int last;                     // rows beyond it are read as it
};

// Workgroup of WM x WN waves, wave tile (16 MT) rows x (16 NT) queries.  LDS: a ring of S slabs of 128 codes per operand.
// Slab image: 128-byte rows, 16-byte chunk c of row r at chunk c ^ ((r >> 1) & 7) (applied to the DMA source and to the reads):
// the 16 lanes of one pass of a ds_read_b128 cover all 64 banks once.  Lane (r, g) of a fragment takes chunks g and g + 4 of
// row r - any order of K inside a block serves as long as both operands share it.
// S - 1 slabs travel ahead of the one that is multiplied: one alone does not cover the way to memory.  The scale words of four
// blocks ride along as 4-byte pieces in front of the first of their slabs, into a ring of two of their own.
//   step D   own pieces of slab D landed, own reads of slab D-1 retired; s_barrier; the pieces of slab D+S-1; reads and products of D
//   RAW  every wave waited for its own pieces of D in front of the barrier.
//   WAR  slab D+S-1 overwrites slab D-1, whose last reads every wave retired in front of the same barrier.
// SOLO: every wave has a tile, a ring and a share of K of its own, and meets no barrier.
template <int MT, int NT, int WM, int WN, int S, bool SOLO = false>
struct F8Tile {
    static constexpr int XR = WM * MT * 16, QR = WN * NT * 16, WAVES = WM * WN, THREADS = WAVES * 64;
    static constexpr int SLAB = (XR + QR) * 128;
    static constexpr int PX = XR / 8 / WAVES, PQ = QR / 8 / WAVES;  // 1 KiB DMA pieces per wave and slab
    static constexpr int WP = (XR + QR + 63) / 64, PW = (WP + WAVES - 1) / WAVES;  // pieces of scale words, of all waves and of one
    static constexpr int WORDS = WP * 256;
    static constexpr int LDS = S * SLAB + 2 * WORDS;
    static_assert(PX * 8 * WAVES == XR && PQ * 8 * WAVES == QR, "pieces divide over the waves");
    static_assert(S >= 2 && S <= 4 && (!SOLO || WAVES == 1), "one piece of scale words at most begins among the slabs ahead");

    unsigned char* smem;
    int lane, wave, wm, wn, nblk;
    const unsigned char *xc, *qc, *sc[PW];
    unsigned xo[PX], qo[PQ];

    __device__ __forceinline__ void init(unsigned char* lds, int blocks) {
        smem = lds;
        nblk = blocks;
        lane = threadIdx.x & 63;
        wave = SOLO ? 0 : __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
        wm = wave / WN;
        wn = wave % WN;
    }
    __device__ __forceinline__ void meet() const {
        if (!SOLO) __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
    }
    // a piece of scale words of this wave (a wave too many repeats the last: all count alike)
    __device__ __forceinline__ int word_piece(int j) const { return min(wave * PW + j, WP - 1); }
    // sources of a tile; starts its pipeline (the first S - 1 slabs).  No wave may still read the ring: true at the start and
    // whenever run() has returned
    __device__ __forceinline__ void aim(const F8Src& x, const F8Src& q) {
        aim(x, q, [](int r) __attribute__((always_inline)) { return r; });
    }
    // ... query r of the tile is row qrow(r) of q
    template <typename F>
    __device__ __forceinline__ void aim(const F8Src& x, const F8Src& q, F qrow) {
#pragma unroll
        for (int j = 0; j < PX; ++j) {
            const int r = (wave * PX + j) * 8 + (lane >> 3);
            xo[j] = (unsigned)min(r, x.last) * x.stride + (((lane & 7) ^ ((r >> 1) & 7)) * 16);
        }
#pragma unroll
        for (int j = 0; j < PQ; ++j) {
            const int r = (wave * PQ + j) * 8 + (lane >> 3);
            qo[j] = (unsigned)qrow(min(r, q.last)) * q.stride + (((lane & 7) ^ ((r >> 1) & 7)) * 16);
        }
        xc = x.codes;
        qc = q.codes;
#pragma unroll
        for (int j = 0; j < PW; ++j) {
            const int r = word_piece(j) * 64 + lane;
            sc[j] = r < XR ? x.scales + (unsigned)min(r, x.last) * x.sstride : q.scales + (unsigned)qrow(max(0, min(r - XR, min(q.last, QR - 1)))) * q.sstride;
        }
#pragma unroll
        for (int d = 0; d < S - 1; ++d)
            if (d < nblk) slab(d, d, d == 0);
    }
    __device__ __forceinline__ void slab(int d, int slot, bool words) {
        if (words) {
#pragma unroll
            for (int j = 0; j < PW; ++j) GLDS4(sc[j] + d, smem + S * SLAB + ((d >> 2) & 1) * WORDS + word_piece(j) * 256);
        }
        unsigned char* dst = smem + slot * SLAB;
        // (uniform addresses that the compiler may not fold with the lanes' offsets: it would keep the 64-bit sums in registers)
        const unsigned char *xb = xc + (size_t)d * 128, *qb = qc + (size_t)d * 128;
        asm volatile("" : "+s"(xb), "+s"(qb));
#pragma unroll
        for (int j = 0; j < PX; ++j) {
            unsigned o = xo[j];
            asm volatile("" : "+v"(o));
            GLDS16(xb + o, dst + (wave * PX + j) * 1024);
        }
#pragma unroll
        for (int j = 0; j < PQ; ++j) {
            unsigned o = qo[j];
            asm volatile("" : "+v"(o));
            GLDS16(qb + o, dst + XR * 128 + (wave * PQ + j) * 1024);
        }
    }

    // the tile aimed at last; the ring is free (for the next aim) on return
    __device__ __forceinline__ void run(f32x4_t (&acc)[MT][NT]) {
        const int frow = lane & 15, fgrp = lane >> 4;
        const int fsw = (frow >> 1) & 7;
        const int c0 = (fgrp ^ fsw) * 16, c1 = ((4 + fgrp) ^ fsw) * 16;
        const int a_row = (wm * MT * 16 + frow) * 128, b_row = XR * 128 + (wn * NT * 16 + frow) * 128;
        int slot = 0, ahead = S - 1;
        int sx[MT], sq[NT];
        const auto step = [&](auto jc, int d) __attribute__((always_inline)) {
            constexpr int J = decltype(jc)::value;
            // (J = d & 3.)  Behind slab d went the pieces of S - 2 slabs, and one of words if a group of four begins among them
            constexpr int LATER = (S - 2) * (PX + PQ) + (J != 0 && J + S - 2 >= 4 ? PW : 0);
            if (d + S - 1 <= nblk) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(LATER) : "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");   // (the last slabs: nothing follows)
            meet();
            if constexpr (J == 0) {
                const int* w = reinterpret_cast<const int*>(smem + S * SLAB + ((d >> 2) & 1) * WORDS);
#pragma unroll
                for (int m = 0; m < MT; ++m) sx[m] = w[(wm * MT + m) * 16 + frow];
#pragma unroll
                for (int n = 0; n < NT; ++n) sq[n] = w[XR + (wn * NT + n) * 16 + frow];
            }
            const unsigned char* cur = smem + slot * SLAB;
            i32x8_t a[MT], b[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n)
                b[n] = join8(*reinterpret_cast<const i32x4_t*>(cur + b_row + n * 2048 + c0), *reinterpret_cast<const i32x4_t*>(cur + b_row + n * 2048 + c1));
#pragma unroll
            for (int m = 0; m < MT; ++m)
                a[m] = join8(*reinterpret_cast<const i32x4_t*>(cur + a_row + m * 2048 + c0), *reinterpret_cast<const i32x4_t*>(cur + a_row + m * 2048 + c1));
            __builtin_amdgcn_sched_barrier(0);   // (the reads in front of the pieces: the compiler would wait for pieces in flight in front of reads)
            if (d + S - 1 < nblk) slab(d + S - 1, ahead, ((J + S - 1) & 3) == 0);
            __builtin_amdgcn_sched_barrier(0);
            float fx[MT], fq[NT];
#pragma unroll
            for (int m = 0; m < MT; ++m) fx[m] = f8_factor<J>(sx[m]);
#pragma unroll
            for (int n = 0; n < NT; ++n) fq[n] = f8_factor<J>(sq[n]);
#pragma unroll
            for (int e = 0; e < 8; e += 2) {   // 32 codes of K
                i32x4_t bw[NT];
#pragma unroll
                for (int n = 0; n < NT; ++n) bw[n] = f8_widen(b[n][e], b[n][e + 1], fq[n]);
#pragma unroll
                for (int m = 0; m < MT; ++m) {
                    const i32x4_t aw = f8_widen(a[m][e], a[m][e + 1], fx[m]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) acc[m][n] = mfma_f8(aw, bw[n], acc[m][n]);
                }
            }
            slot = slot == S - 1 ? 0 : slot + 1;
            ahead = ahead == S - 1 ? 0 : ahead + 1;
        };
#pragma unroll 1
        for (int d = 0; d < nblk; d += 4) {
            step(std::integral_constant<int, 0>(), d);
            if (d + 1 < nblk) step(std::integral_constant<int, 1>(), d + 1);
            if (d + 2 < nblk) step(std::integral_constant<int, 2>(), d + 2);
            if (d + 3 < nblk) step(std::integral_constant<int, 3>(), d + 3);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        meet();
    }
};

}  // namespace ssmi

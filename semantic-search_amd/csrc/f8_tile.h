// f8_tile.h - contraction of one tile of 8-bit rows with one tile of 8-bit queries on the scaled matrix instruction.
//
//   acc[row][query] = sum over blocks b of 2^(sx[row,b] - 127) 2^(sq[query,b] - 127) sum over the 128 codes of b of x q
//
// v_mfma_scale_f32_16x16x128_f8f6f4: K = 128 is one scale block, so the two E8M0 bytes of a (row, query) pair ride along with
// the instruction (its operand selectors pick the byte of a word that holds four blocks) and no vector instruction touches
// the products.  The instruction aligns the products of a block to the largest of them and drops what lies more than 13 bits
// below it (measured: a sum over 4096 dimensions is off by 1.6e-5 of the scores' norm, where a chain of fp32 adds is off by
// 5e-8): its sums are the candidates of a search, which scores them again in 64 bits, or leave rounded to 16 bits.
#pragma once
#include "f8.h"
#include "mfma_common.h"

namespace ssmi {

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef int i32x2_t __attribute__((ext_vector_type(2)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));

template <int J>
__device__ __forceinline__ f32x4_t mfma_f8(const i32x8_t& a, const i32x8_t& b, const f32x4_t& c, int sa, int sb) {
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, J, sa, J, sb);
}
__device__ __forceinline__ i32x8_t join8(const i32x4_t& lo, const i32x4_t& hi) {
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

typedef float f32x16_t __attribute__((ext_vector_type(16)));

template <int J>
__device__ __forceinline__ f32x16_t mfma_f8_32(const i32x8_t& a, const i32x8_t& b, const f32x16_t& c, int sa, int sb) {
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a, b, c, 0, 0, J, sa, J, sb);
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
#pragma unroll
        for (int j = 0; j < PX; ++j) {
            const int r = (wave * PX + j) * 8 + (lane >> 3);
            xo[j] = (unsigned)min(r, x.last) * x.stride + (((lane & 7) ^ ((r >> 1) & 7)) * 16);
        }
#pragma unroll
        for (int j = 0; j < PQ; ++j) {
            const int r = (wave * PQ + j) * 8 + (lane >> 3);
            qo[j] = (unsigned)min(r, q.last) * q.stride + (((lane & 7) ^ ((r >> 1) & 7)) * 16);
        }
        xc = x.codes;
        qc = q.codes;
#pragma unroll
        for (int j = 0; j < PW; ++j) {
            const int r = word_piece(j) * 64 + lane;
            sc[j] = r < XR ? x.scales + (unsigned)min(r, x.last) * x.sstride : q.scales + (unsigned)min(r - XR, min(q.last, QR - 1)) * q.sstride;
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
        const int frow = lane & 15, fq = lane >> 4;
        const int fsw = (frow >> 1) & 7;
        const int c0 = (fq ^ fsw) * 16, c1 = ((4 + fq) ^ fsw) * 16;
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
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n) acc[m][n] = mfma_f8<J>(a[m], b[n], acc[m][n], sx[m], sq[n]);
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

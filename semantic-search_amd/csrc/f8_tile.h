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

// Workgroup of WM x WN waves, wave tile (16 MT) rows x (16 NT) queries.  LDS: two buffers of one 128-code slab per operand.
// Slab image: 128-byte rows, 16-byte chunk c of row r at chunk c ^ ((r >> 1) & 7) (applied to the DMA source and to the reads):
// the 16 lanes of one pass of a ds_read_b128 cover all 64 banks once.  Lane (r, g) of a fragment takes chunks g and g + 4 of
// row r - any order of K inside a block serves as long as both operands share it.
template <int MT, int NT, int WM, int WN>
struct F8Tile {
    static constexpr int XR = WM * MT * 16, QR = WN * NT * 16, WAVES = WM * WN, THREADS = WAVES * 64;
    static constexpr int SLAB = (XR + QR) * 128;
    static constexpr int LDS = 2 * SLAB;
    static constexpr int PX = XR / 8 / WAVES, PQ = QR / 8 / WAVES;  // 1 KiB DMA pieces per wave and slab
    static_assert(PX * 8 * WAVES == XR && PQ * 8 * WAVES == QR, "pieces divide over the waves");

    static __device__ __forceinline__ void run(f32x4_t (&acc)[MT][NT], unsigned char* smem, const F8Src& x, const F8Src& q, int nblk) {
        const int lane = threadIdx.x & 63;
        const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
        const int wm = wave / WN, wn = wave % WN;
        const int frow = lane & 15, fq = lane >> 4;
        unsigned xo[PX], qo[PQ];
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
        unsigned xso[MT], qso[NT];
#pragma unroll
        for (int m = 0; m < MT; ++m) xso[m] = (unsigned)min((wm * MT + m) * 16 + frow, x.last) * x.sstride;
#pragma unroll
        for (int n = 0; n < NT; ++n) qso[n] = (unsigned)min((wn * NT + n) * 16 + frow, q.last) * q.sstride;
        const int fsw = (frow >> 1) & 7;
        const int c0 = (fq ^ fsw) * 16, c1 = ((4 + fq) ^ fsw) * 16;
        const int a_row = (wm * MT * 16 + frow) * 128, b_row = XR * 128 + (wn * NT * 16 + frow) * 128;

        auto issue = [&](int kb, unsigned char* buf) {
#pragma unroll
            for (int j = 0; j < PX; ++j) GLDS16(x.codes + (size_t)kb * 128 + xo[j], buf + (wave * PX + j) * 1024);
#pragma unroll
            for (int j = 0; j < PQ; ++j) GLDS16(q.codes + (size_t)kb * 128 + qo[j], buf + XR * 128 + (wave * PQ + j) * 1024);
        };
        auto settle = [&]() {  // own pieces landed, own reads retired; then everybody's
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
        };
        issue(0, smem);
        settle();
        int buf = 0;
        auto step = [&](auto jc, int kb, const int (&sx)[MT], const int (&sq)[NT]) {
            constexpr int J = decltype(jc)::value;
            const unsigned char* cur = smem + buf * SLAB;
            if (kb + 1 < nblk) issue(kb + 1, smem + (buf ^ 1) * SLAB);
            i32x8_t b[NT];
#pragma unroll
            for (int n = 0; n < NT; ++n)
                b[n] = join8(*reinterpret_cast<const i32x4_t*>(cur + b_row + n * 2048 + c0), *reinterpret_cast<const i32x4_t*>(cur + b_row + n * 2048 + c1));
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                const i32x8_t a = join8(*reinterpret_cast<const i32x4_t*>(cur + a_row + m * 2048 + c0), *reinterpret_cast<const i32x4_t*>(cur + a_row + m * 2048 + c1));
#pragma unroll
                for (int n = 0; n < NT; ++n) acc[m][n] = mfma_f8<J>(a, b[n], acc[m][n], sx[m], sq[n]);
            }
            settle();
            buf ^= 1;
        };
        for (int kb = 0; kb < nblk; kb += 4) {
            int sx[MT], sq[NT];
#pragma unroll
            for (int m = 0; m < MT; ++m) sx[m] = *reinterpret_cast<const int*>(x.scales + kb + xso[m]);
#pragma unroll
            for (int n = 0; n < NT; ++n) sq[n] = *reinterpret_cast<const int*>(q.scales + kb + qso[n]);
            step(std::integral_constant<int, 0>(), kb, sx, sq);
            if (kb + 1 < nblk) step(std::integral_constant<int, 1>(), kb + 1, sx, sq);
            if (kb + 2 < nblk) step(std::integral_constant<int, 2>(), kb + 2, sx, sq);
            if (kb + 3 < nblk) step(std::integral_constant<int, 3>(), kb + 3, sx, sq);
        }
    }
};

}  // namespace ssmi

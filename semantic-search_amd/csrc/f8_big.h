// f8_big.h - the contraction of f8_tile.h for tiles of 256 rows x 256 queries: four waves, one per SIMD, 128 x 128 each.
//
// The kernel is bound by the chip's power before it is bound by the matrix pipe.  A wave tile of 128 x 128 (4 x 4 accumulators of
// v_mfma_f32_32x32x16_bf16, 256 registers) reads a third less from LDS than two waves of 128 x 64, and converts as much less: a fragment
// becomes an operand (two pairs of codes under every MFMA of 32 cycles) for four products.  With one wave per SIMD nothing else hides a stall, so
// the wave runs its own pipeline: K is walked in phases of 64 codes, and under the 64 MFMAs (2048 cycles) of one phase it reads the next phase's
// fragments.  Operands arrive in slabs of 128 codes (one scale block, two phases) by DMA into a ring of two:
//
//   even phase of slab D   MFMAs of (D, first half);  ds_reads of (D, second half)
//                          own reads retired, own pieces of slab D+1 landed (lgkmcnt(0), vmcnt(0)); s_barrier
//   odd phase of slab D    MFMAs of (D, second half); ds_reads of (D+1, first half); the sixteen pieces of slab D+2
//
//   RAW  slab D+1 is first read behind the barrier of slab D, in front of which every wave waited for its own pieces.
//   WAR  slab D+2 overwrites slab D, whose last reads every wave retired in front of the same barrier.
// One barrier per 4096 cycles of MFMAs, and a piece has 2048 to 4096 of them to land.  The scale words of four blocks ride along as
// 4-byte pieces into a ring of two of their own: group G+1 is issued behind the pieces of slab 4G+2 and read in the odd phase of slab 4G+3.
#pragma once
#include "f8_tile.h"

namespace ssmi {

struct F8Big {
    static constexpr int SLAB = 256 * 128;                // one operand's 128 codes of 256 rows
    static constexpr int SCALES = 4 * SLAB;               // behind the ring: [2][X: 256 words, Q: 256 words]
    static constexpr int LDS = SCALES + 2 * 2048;
    typedef f32x16_t Acc[4][4];

    unsigned char* smem;
    int wave, wm, wn, nblk;
    const unsigned char *xc, *qc, *sc;                    // codes of the tiles; scales of the operand this wave brings
    unsigned xstride, qstride, so[2];
    int xlast, qlast;

    __device__ __forceinline__ void init(unsigned char* lds, int blocks) {
        smem = lds;
        nblk = blocks;
        wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
        wm = wave >> 1;
        wn = wave & 1;
    }
    // a uniform pointer in scalar registers, wherever it came from
    static __device__ __forceinline__ const unsigned char* scalar(const unsigned char* p) {
        const unsigned long long v = reinterpret_cast<unsigned long long>(p);
        const unsigned lo = (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)v), hi = (unsigned)__builtin_amdgcn_readfirstlane((int)(v >> 32));
        return reinterpret_cast<const unsigned char*>(((unsigned long long)hi << 32) | lo);
    }
    // sources of a tile; starts its pipeline (slabs 0 and 1, the first scale words).  No wave may still read the ring: true
    // at the start and whenever run() has returned
    __device__ __forceinline__ void aim(const F8Src& x, const F8Src& q) {
        const int lane = lane_now();
        xstride = x.stride;
        qstride = q.stride;
        xlast = x.last;
        qlast = q.last;
        xc = scalar(x.codes);
        qc = scalar(q.codes);
        sc = scalar(wm ? q.scales : x.scales);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int r = wn * 128 + j * 64 + lane;
            so[j] = wm ? (unsigned)min(r, q.last) * q.sstride : (unsigned)min(r, x.last) * x.sstride;
        }
        pieces(0);
        words(0);
        if (nblk > 1) pieces(1);
    }
    // columns of slab d of both operands: uniform addresses that the compiler may not fold with the lanes' offsets (it would keep the
    // sixteen 64-bit sums in registers across the loop), and one LDS address, not thirty-two of them.  A lane brings chunk c of row r0 + 8 j
    // with piece j; the offsets are made anew for every piece, three instructions under an MFMA (kept, sixteen of them spilled)
    typedef __attribute__((address_space(3))) unsigned char* Lds;
    struct Cols { const unsigned char *x, *q; Lds dst; };
    __device__ __forceinline__ Cols cols(int d, int slot) const {
        Cols c{xc + (size_t)d * 128, qc + (size_t)d * 128, (Lds)(smem + slot * SLAB + wave * 8192)};
        asm volatile("" : "+s"(c.x), "+s"(c.q), "+s"(c.dst));
        return c;
    }
    // lane: its number, opaque (lane_now or a register that an empty statement has touched)
    __device__ __forceinline__ void piece(const Cols& c, int t, int lane) {
        const int r = wave * 64 + (t & 7) * 8 + (lane >> 3);
        const unsigned chunk = ((lane & 7) ^ ((lane >> 4) + (t & 1) * 4)) * 16;   // (r >> 1) & 7
        // (rows < 256 and strides of at most 2^23 bytes: 24 bits)
        unsigned o = t < 8 ? __umul24((unsigned)min(r, xlast), xstride) + chunk : __umul24((unsigned)min(r, qlast), qstride) + chunk;
        asm volatile("" : "+v"(o));   // (a 32-bit offset beside the uniform address, widened here and not ahead of the loop)
        const unsigned char* src = (t < 8 ? c.x : c.q) + o;
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                         (__attribute__((address_space(3))) void*)(c.dst + (t < 8 ? 0 : 2 * SLAB) + (t & 7) * 1024), 16, 0, 0);
    }
    __device__ __forceinline__ void pieces(int d) {
        const Cols c = cols(d, d & 1);
        const int lane = lane_now();
#pragma unroll
        for (int t = 0; t < 16; ++t) piece(c, t, lane);
    }
    __device__ __forceinline__ void words(int g) {
        const unsigned char* c = sc + (size_t)g * 4;
        asm volatile("" : "+s"(c));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            unsigned o = so[j];
            asm volatile("" : "+v"(o));
            GLDS4(c + o, smem + SCALES + (g & 1) * 2048 + wave * 512 + j * 256);
        }
    }
    // the lane's number, counted anew: what hangs on it is worked out again, not kept in registers across a tile
    static __device__ __forceinline__ int lane_now() {
        int l;
        asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(l));
        return l;
    }

    struct Frags { i32x4_t a[2][4], b[2][4]; };   // [codes 0-15, 16-31 of a lane][32 rows]
    // ds_read t (0..15) of half H of a slab, in the order in which the next phase wants them: b0..b3, a0..a3, first codes first
    template <int H>
    __device__ __forceinline__ void read(Frags& f, const unsigned char* cur, int t, int a_row, int b_row, const int (&ch)[4]) const {
        const bool is_a = (t & 4) != 0;
        const int i = t & 3, c = t >> 3;
        (is_a ? f.a[c][i] : f.b[c][i]) = *reinterpret_cast<const i32x4_t*>(cur + (is_a ? a_row : b_row) + i * 4096 + ch[2 * H + c]);
    }

    __device__ __forceinline__ void run(Acc& acc) {
        const int lane = lane_now();
        const int r32 = lane & 31, hl = lane >> 5;
        const int sw = (r32 >> 1) & 7;
        const int a_row = (wm * 128 + r32) * 128, b_row = 2 * SLAB + (wn * 128 + r32) * 128;
        const int ch[4] = {(hl ^ sw) * 16, ((2 + hl) ^ sw) * 16, ((4 + hl) ^ sw) * 16, ((6 + hl) ^ sw) * 16};
        int sx[4], sq[4];      // scale words of the four blocks at hand
        float fx[4], fq[4];    // the factors of one of them
        Frags f0, f1;
        i32x4_t aw[2], bw[2][4];   // operands: rows of a two deep, a step of b two deep
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        const auto words_of = [&](int g) __attribute__((always_inline)) {
            const int* w = reinterpret_cast<const int*>(smem + SCALES + (g & 1) * 2048);
#pragma unroll
            for (int m = 0; m < 4; ++m) sx[m] = w[wm * 128 + m * 32 + r32];
#pragma unroll
            for (int n = 0; n < 4; ++n) sq[n] = w[256 + wn * 128 + n * 32 + r32];
        };
        // word e of step k (0..3) of a row's fragment -> two codes of an operand
        const auto word = [&](const i32x4_t (&f)[2][4], int i, int k, int e) __attribute__((always_inline)) { return f[k >> 1][i][2 * (k & 1) + (e >> 1)]; };
        const auto pair = [&](int w, int e, float s) __attribute__((always_inline)) { return e & 1 ? f8_pair<true>(w, s) : f8_pair<false>(w, s); };
        // Sixty-four MFMAs of a phase.  Under the sixteen of a step the next step's fragments of b become operands, a pair of codes each, and
        // under the first two of a row of a the next row's: with the reads and pieces of hook(t) no more than the MFMA's 32 cycles hide.
        // nxt: the next phase's fragments, whose first words the last step converts; J: the block whose factors those need, -1: the same
        const auto phase = [&](auto jc, const Frags& cur, const Frags& nxt, auto hook) __attribute__((always_inline)) {
            constexpr int J = decltype(jc)::value;
#pragma unroll
            for (int t = 0; t < 64; ++t) {
                const int k = t >> 4, m = (t >> 2) & 3, n = t & 3;
                acc[m][n] = mfma_f8_32(aw[m & 1], bw[k & 1][n], acc[m][n]);
                if constexpr (J >= 0) {   // each behind the last use of the old one
                    if (t >= 44 && t < 47) fq[t - 44] = f8_factor<(J & 3)>(sq[t - 44]);
                    if (t == 48) fq[3] = f8_factor<(J & 3)>(sq[3]);
                    if (t == 58 || t == 59) {
                        fx[2 * (t - 58)] = f8_factor<(J & 3)>(sx[2 * (t - 58)]);
                        fx[2 * (t - 58) + 1] = f8_factor<(J & 3)>(sx[2 * (t - 58) + 1]);
                    }
                }
                if (n < 2) {
                    const int m2 = (m + 1) & 3, k2 = k + (m == 3);
#pragma unroll
                    for (int e = 2 * n; e < 2 * n + 2; ++e)
                        aw[m2 & 1][e] = k2 < 4 ? pair(word(cur.a, m2, k2, e), e, fx[m2]) : pair(word(nxt.a, m2, 0, e), e, fx[m2]);
                }
                bw[(k + 1) & 1][m][n] = k < 3 ? pair(word(cur.b, m, k + 1, n), n, fq[m]) : pair(word(nxt.b, m, 0, n), n, fq[m]);
                hook(t);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        words_of(0);
#pragma unroll
        for (int t = 0; t < 16; ++t) read<0>(f0, smem, t, a_row, b_row, ch);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            fx[i] = f8_factor<0>(sx[i]);
            fq[i] = f8_factor<0>(sq[i]);
            bw[0][i] = f8_widen(f0.b[0][i][0], f0.b[0][i][1], fq[i]);
        }
        aw[0] = f8_widen(f0.a[0][0][0], f0.a[0][0][1], fx[0]);
        // slab d, block J of its group of four.  FULL: slab d+1 exists, and the group's four
        const auto slab = [&](auto jc, auto fc, int d) __attribute__((always_inline)) {
            constexpr int J = decltype(jc)::value;
            constexpr bool FULL = decltype(fc)::value;
            const unsigned char* cur = smem + (J & 1) * SLAB;          // (d & 1 == J & 1)
            const unsigned char* nxt = smem + ((J & 1) ^ 1) * SLAB;
            // ---- even phase ----
            phase(std::integral_constant<int, -1>(), f0, f1, [&](int t) __attribute__((always_inline)) {
                if (t >= 8 && t < 40 && (t & 1) == 0) read<1>(f1, cur, (t - 8) >> 1, a_row, b_row, ch);
            });
            // (the scale pieces, 64 cache lines each, went out last with slab J = 0: they may take a slab longer)
            if constexpr (FULL && J == 1) asm volatile("s_waitcnt vmcnt(2) lgkmcnt(0)" ::: "memory");
            else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            __builtin_amdgcn_sched_barrier(0);
            // ---- odd phase ----
            if constexpr (FULL) {
                const Cols c = cols(min(d + 2, nblk - 1), J & 1);   // (a slab beyond the last: the last again, never read)
                const int l = lane_now();
                if constexpr (J == 3) words_of(((d + 1) >> 2) & 1);
                phase(std::integral_constant<int, (J + 1) & 3>(), f1, f0, [&](int t) __attribute__((always_inline)) {
                    if (t >= 8 && t < 40 && (t & 1) == 0) read<0>(f0, nxt, (t - 8) >> 1, a_row, b_row, ch);
                    if ((t & 3) == 2) piece(c, t >> 2, l);
                });
                if constexpr (J == 0) words(d / 4 + 1);
            } else {
                if (d + 1 < nblk) {
#pragma unroll
                    for (int t = 0; t < 16; ++t) read<0>(f0, nxt, t, a_row, b_row, ch);
                }
                if (d + 2 < nblk) pieces(d + 2);
                phase(std::integral_constant<int, J < 3 ? J + 1 : -1>(), f1, f0, [](int) __attribute__((always_inline)) {});
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        const std::integral_constant<int, 0> c0;
        const std::integral_constant<int, 1> c1;
        const std::integral_constant<int, 2> c2;
        const std::integral_constant<int, 3> c3;
        const std::integral_constant<bool, true> full;
        const std::integral_constant<bool, false> rest;
        int d = 0;
#pragma unroll 1
        for (; d + 5 <= nblk; d += 4) {
            slab(c0, full, d);
            slab(c1, full, d + 1);
            slab(c2, full, d + 2);
            slab(c3, full, d + 3);
        }
        slab(c0, rest, d);   // one to four remain
        if (d + 1 < nblk) slab(c1, rest, d + 1);
        if (d + 2 < nblk) slab(c2, rest, d + 2);
        if (d + 3 < nblk) slab(c3, rest, d + 3);
    }
};

}  // namespace ssmi

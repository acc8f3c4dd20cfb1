// f8.h - 8-bit rows: e4m3 codes with one power-of-two scale for every 128 of them (internal to libssmi).
//
//   value(row, e) = code(row, e) * 2^(b(row, e / 128) - 127)
//
// codes: OCP e4m3 (largest finite value 448, no infinity, 0x7f / 0xff = NaN), rows padded with zero codes to whole blocks.
// b: E8M0 exponent bytes, 255 = NaN.  The quantiser takes the smallest power of two s with max|x| <= 448 s and rounds x / s
// to nearest even.  Powers of two, for two reasons: a value still has four significant bits, so that bf16 holds it and the matrix
// cores take it exactly (f8_tile.h), and quantising the values of a quantised row gives the same values (a block
// whose largest code rounded down to 224 halves its scale and doubles its codes).
#pragma once
#include "kernels.h"
#ifdef __HIPCC__
#include "topk.h"
#endif

namespace ssmi {

static constexpr int kF8 = 3;             // SSMI_F8
static constexpr int kF8Block = 128;      // codes per scale
static constexpr int kF8Spare = 16;       // candidates beyond k that a search scores again in 64 bits
static constexpr int kF8Collect = 2048;   // rows that a query's fp32 sums may leave in question before all rows are
static constexpr int kF8Batch = 4096;     // queries of a search that travel together
enum { kF8Fp32, kF8Scaled, kF8Again };
static constexpr int kF8MaxNorm = 16384;  // elements of a row that the norm keeps in registers
static constexpr int kF8MaxK = kMaxK - kF8Spare;

inline int f8_ld(int d) { return (d + kF8Block - 1) / kF8Block * kF8Block; }
inline int f8_blocks(int d) { return (d + kF8Block - 1) / kF8Block; }

// n rows of codes and scales in plain memory; strides in bytes
struct F8Mat {
    const unsigned char* codes;
    long long stride;         // multiple of 16, codes 16-byte aligned
    const unsigned char* scales;
    long long sstride;        // multiple of 4, scales 4-byte aligned
    long long n;
};
// the same inside a row store: segment tables of the codes (X) and of the scales
struct F8View {
    RowView X;                // ld = codes per row
    const void* const* ssegs;
    int sld;                  // scale bytes per row (multiple of 16)
    const void* const* lsegs; // lengths, a float a row
};

struct F8NormArgs {
    const void* x; long long x_stride;                 // strides in elements
    const void* residual; long long r_stride;          // nullptr: none
    void* residual_out; long long ro_stride;
    const void* weight; int weight_dtype;              // nullptr: none
    float eps;
    double inv_d;                                      // 1 / d
    bool norm, unit;
    long long n;
    int d, dtype;
    unsigned char* codes; long long stride;
    unsigned char* scales; long long sstride;
};
hipError_t launch_f8_rows(const F8NormArgs& a, int num_cu, hipStream_t s);
// codes + scales -> (n, d) of out_dtype, row stride in elements
hipError_t launch_f8_dequantize(const F8Mat& m, int d, void* out, int out_dtype, long long out_stride, int num_cu, hipStream_t s);
// rows by id out of a row store -> fp32 (n, d); as launch_gather_rows / launch_score_rows
hipError_t launch_f8_gather(const F8View& v, const int64_t* ids, long long n, int d, float* out, int* bad, hipStream_t s);
hipError_t launch_f8_score_rows(const F8View& v, const int64_t* ids, long long n, int d, const float* neg, int n_neg, float* out,
                                int* bad, hipStream_t s);
// out[i][j] = <a_i, b_j>, (a.n, b.n) of out_dtype (SSMI_F16 / SSMI_BF16), row stride in elements
hipError_t launch_f8_matmul(const F8Mat& a, const F8Mat& b, int k, void* out, int out_dtype, long long out_stride, int num_cu, hipStream_t s);

// the lengths of rows, rounded up (a row that holds a NaN: -1); longest (the bits of positive floats): [0] the largest of it and them, [1] the same of
// the lengths of the rows' largest elements, one of every eight neighbours (none less than 2^-6 of its block's scale)
hipError_t launch_f8_lengths(const F8Mat& m, int ld, float* lengths, unsigned* longest, int num_cu, hipStream_t s);

// What the second pass of a search leaves for the third.  ticket 0: the query is answered; else it counts the workgroups that are done with it,
// from 1, and pos their entries.  No row with a score below edge is among the k best, nor one that is not on the list and shorter than `from`,
// nor one whose fp32 sum s and length x have s + slope x < least (slope < 0: that is not known).  found: how many rows have not, more than kF8Collect:
// they are not listed
struct F8State { double edge; float from, least, slope; unsigned ticket, pos, found; };
struct F8Entry { double score; long long id; };

// search over a row store: the k best of every query with their scores summed in 64 bits
struct F8SearchPlan {
    int kp;                   // candidates kept per query by the first pass
    int parts;                // partial lists per query
    bool scan;                // streaming scan (few queries), else the tile kernel
    int bt, r, threads, grid_x;
    int nb;                   // scan: blocks per row where that is 1, 2 or 4, 8 where it is a multiple of 8, else 0
    int cap, every;           // scan: candidates a query's buffer holds, turns of three stages between two looks at them
    int tq, nqt, nslices, gtop_m;
    bool scaled;              // 256 queries a tile: the scaled instruction first, fp32 sums for the tiles with queries that those do not prove
    long long rows_per_slice;
    size_t lds, partial_bytes, cand_bytes, share_bytes;
    const char* kernel;
};
bool plan_f8_search(int ld, long long nrows, int nq, int k, int num_cu, F8SearchPlan* p);
// open: not null for the second run of a scaled plan
hipError_t launch_f8_tiles(const F8View& v, const F8Mat& q, const F8SearchPlan& p, const F8State* open, void* share, void* cand, skey_t* partial, hipStream_t s);
// the streaming scan of up to p.bt queries, and what follows the first pass; queries: fp32 rows of d elements at f32, else q.codes
struct F8ScanArgs {
    F8View v;
    F8Mat q;
    const float* f32;
    long long f32_stride;     // elements
    bool f32_vec;             // rows of 16-byte aligned floats
    int d, k, kp;
    skey_t* partial;          // [q.n][p.parts][kp]
    unsigned* counter;        // ticket counter, zero between launches: the scan does everything (one query); nullptr: launch_f8_finish follows
    unsigned* shared;         // eight words, zero between searches: the highest threshold of every query (f32_to_ord bits); nullptr: none
    float* D;
    int64_t* I;
    int64_t id_offset;
    unsigned min_ord;
    int cap, every;
    const float* longest;     // of launch_f8_lengths
    int sums;                 // what the first pass added up with: kF8Fp32, kF8Scaled, or kF8Again: fp32 for the queries that state holds open
    F8State* state;           // [q.n], written by the second pass
    unsigned char* open;      // [q.n][v.X.ld] codes, then [q.n][v.sld] scales: the queries it leaves; nullptr: for the exact pass as they are
    unsigned* rows;           // [q.n][kF8Collect] the rows in question of each
    F8Entry* lists;           // [num_cu][k], of the exact pass
};
hipError_t launch_f8_scan(const F8ScanArgs& a, const F8SearchPlan& p, hipStream_t s);
hipError_t launch_f8_finish(const F8ScanArgs& a, const F8SearchPlan& p, hipStream_t s);
// the queries whose lists the second pass could not prove: rows in question by fp32 sums, and those, or all, in 64 bits
hipError_t launch_f8_collect(const F8ScanArgs& a, int num_cu, hipStream_t s);
hipError_t launch_f8_exact(const F8ScanArgs& a, int num_cu, hipStream_t s);

#ifdef __HIPCC__
// two e4m3 codes per call from the low or high half of a word
template <bool HI>
__device__ __forceinline__ void f8_unpack2(unsigned w, float& a, float& b) {
    const auto v = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, HI);
    a = v[0];
    b = v[1];
}
__device__ __forceinline__ void f8_unpack4(unsigned w, float (&o)[4]) {
    f8_unpack2<false>(w, o[0], o[1]);
    f8_unpack2<true>(w, o[2], o[3]);
}
// Eight neighbouring elements of a block whose other elements the 16 lanes of this lane's row hold -> their codes and the
// block's scale byte.  e0: place of the first in a row of d elements.  All 16 lanes call.
__device__ __forceinline__ uint2 f8_pack8(const float (&v)[8], int e0, int d, unsigned& b) {
    // largest magnitude of the block as an integer: NaN > infinity > every finite value
    unsigned m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
    m = max(m, (unsigned)xor_lane<1>((int)m));
    m = max(m, (unsigned)xor_lane<2>((int)m));
    m = max(m, (unsigned)xor_lane<4>((int)m));
    m = max(m, (unsigned)xor_lane<8>((int)m));
    if (m < 0x7f800000u) {
        // m = f * 2^(E-127), 1 <= f < 2, and 448 = 1.75 * 2^8
        b = (unsigned)max((int)(m >> 23) - 8 + ((m & 0x7fffffu) > 0x600000u ? 1 : 0), 0);
        const float inv = __uint_as_float((254u - b) << 23);
        int lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * inv, v[1] * inv, 0, false);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * inv, v[3] * inv, lo, true);
        int hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * inv, v[5] * inv, 0, false);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * inv, v[7] * inv, hi, true);
        return uint2{(unsigned)lo, (unsigned)hi};
    }
    // an infinity or a NaN makes its block NaN; the padding keeps its zero codes
    b = 255u;
    unsigned w[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j >> 2] |= e0 + j < d ? 0x7fu << (8 * (j & 3)) : 0u;
    return uint2{w[0], w[1]};
}
// 2^(b - 127); 255: NaN.  (2^-127 is a subnormal fp32.)
__device__ __forceinline__ float f8_scale(unsigned b) {
    return b == 255u ? __builtin_nanf("") : __uint_as_float(b ? b << 23 : 0x00400000u);
}
#endif

}  // namespace ssmi

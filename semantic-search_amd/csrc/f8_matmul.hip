// f8_matmul.hip - the product of two matrices of 8-bit rows (f8.h):
//
//   out[i][j] = sum over blocks b of 2^(sa[i,b] - 127) 2^(sb[j,b] - 127) sum over the 128 codes of b of a[i,.] b[j,.]
//
// exact products summed in fp32 (f8_tile.h), rounded once to 16 bits.  Tiles of 256 x 256 with a wave per SIMD where they fill the chip, tiles
// of 128 x 128 and 64 x 64 below that, and where those would leave most CUs idle (a decoding batch) smaller ones whose waves share K.
#include <algorithm>
#include <initializer_list>
#include "f8_big.h"

namespace ssmi {

// two sums rounded to nearest even, the first in the low half
template <bool BF>
__device__ __forceinline__ unsigned narrow2(float lo, float hi) {
    typedef float f32x2_t __attribute__((ext_vector_type(2)));
    const f32x2_t v = {lo, hi};
    if constexpr (BF) {
        typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2_t));
    } else {
        typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(unsigned, __builtin_convertvector(v, f16x2_t));
    }
}

struct F8MatmulArgs {
    F8Mat a, b;
    int nblk;
    unsigned short* out;
    long long ostride;
    int ta, tb;     // tiles along a and b
};

// a tile of the output: rows x cols of it exist
struct F8Out {
    unsigned short* base;
    long long ostride;
    int rows, cols;
};
__device__ __forceinline__ F8Out out_tile(const F8MatmulArgs& p, long long i0, long long j0) {
    return F8Out{p.out + i0 * p.ostride + j0, p.ostride, (int)min(256ll, p.a.n - i0), (int)min(256ll, p.b.n - j0)};
}
// N neighbouring columns c.. of row r, two to a word, as one store: the memory takes 8 and 16 bytes at any even address, and rows
// of an odd stride need no other path
template <int N>
__device__ __forceinline__ void store_words(const F8Out& t, int r, int c, const unsigned (&w)[N / 2]) {
    typedef unsigned words_t __attribute__((ext_vector_type(N / 2), aligned(2)));
    if (r >= t.rows || c >= t.cols) return;
    unsigned short* o = t.base + (unsigned long long)(unsigned)r * (unsigned long long)t.ostride + c;
    if (c + N <= t.cols) {
        words_t v;
#pragma unroll
        for (int e = 0; e < N / 2; ++e) v[e] = w[e];
        *reinterpret_cast<words_t*>(o) = v;
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (c + e < t.cols) o[e] = (unsigned short)(w[e / 2] >> (16 * (e & 1)));
    }
}
template <bool BF>
__device__ __forceinline__ void store4(const F8Out& t, int r, int c, const f32x4_t& v) {
    const unsigned w[2] = {narrow2<BF>(v[0], v[1]), narrow2<BF>(v[2], v[3])};
    store_words<4>(t, r, c, w);
}
// A 32 x 32 accumulator: register 4 g + e of lane (r, h) is column 8 g + 4 h + e of row r.  The lane pairs (r, 0), (r, 1) trade
// halves, so that lane (r, h) holds the eight columns 8 (g + h).. and a row leaves in pieces of 32 bytes, not 16.
template <bool BF>
__device__ __forceinline__ void store32(const F8Out& t, int r, int c, int h, const f32x16_t& v) {
#pragma unroll
    for (int g = 0; g < 4; g += 2) {
        unsigned w[4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const auto x = __builtin_amdgcn_permlane32_swap((int)narrow2<BF>(v[4 * g + 2 * e], v[4 * g + 2 * e + 1]), (int)narrow2<BF>(v[4 * g + 4 + 2 * e], v[4 * g + 5 + 2 * e]), false, false);
            w[e] = (unsigned)x[0];
            w[2 + e] = (unsigned)x[1];
        }
        store_words<8>(t, r, c + 8 * (g + h), w);
    }
}

// workgroups go round the eight XCDs: neighbouring tiles, which share rows, to the L2 of one
__device__ __forceinline__ int logical_tile() {
    return (gridDim.x & 7) == 0 ? (int)((blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3)) : (int)blockIdx.x;
}

// b's rows are the matrix instruction's rows: a lane then holds four neighbouring columns of one output row
template <int MT, int NT, int WM, int WN, int S, bool BF>
__global__ void __launch_bounds__(WM * WN * 64) f8_matmul_tile_kernel(F8MatmulArgs p) {
    using T = F8Tile<MT, NT, WM, WN, S>;
    extern __shared__ __align__(16) unsigned char smem[];
    const int tile = logical_tile();
    const int ti = tile % p.ta, tj = tile / p.ta;
    const long long i0 = (long long)ti * T::QR, j0 = (long long)tj * T::XR;
    F8Src x{p.b.codes + j0 * p.b.stride, p.b.scales + j0 * p.b.sstride, (unsigned)p.b.stride, (unsigned)p.b.sstride, (int)min((long long)T::XR - 1, p.b.n - 1 - j0)};
    F8Src q{p.a.codes + i0 * p.a.stride, p.a.scales + i0 * p.a.sstride, (unsigned)p.a.stride, (unsigned)p.a.sstride, (int)min((long long)T::QR - 1, p.a.n - 1 - i0)};
    f32x4_t acc[MT][NT];
    zero_acc(acc);
    T t;
    t.init(smem, p.nblk);
    t.aim(x, q);
    t.run(acc);
    const int frow = t.lane & 15, fq = t.lane >> 4;
    const F8Out o = out_tile(p, i0, j0);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m)
            store4<BF>(o, (t.wn * NT + n) * 16 + frow, (t.wm * MT + m) * 16 + fq * 4, acc[m][n]);
}

// 256 x 256 tiles, a wave per SIMD: workgroups stay, the first slab of the next tile travels under this one's epilogue.
// Tiles are numbered in bands of eight along a, and consecutive workgroups go round the XCDs: the 32 tiles of an XCD cover 8 x 4,
// twelve operand panels for its L2.
// 8192^3: 694 us, 1.58 PFLOP/s; 4096 x 8192 x 8192: 357 us, 1.54; 4096^3: 97 us, 1.41 (8192^3 in tiles of 128 x 128: 878 us).  The bf16
// instruction alone reaches 1.75 PFLOP/s on registers: the chip's power is the limit, and codes in LDS take half the bytes of bf16 there.
template <bool BF>
__global__ void __launch_bounds__(256, 1) f8_matmul_big_kernel(F8MatmulArgs p) {
    extern __shared__ __align__(16) unsigned char smem[];
    F8Big t;
    t.init(smem, p.nblk);
    const int tiles = p.ta * p.tb;
    const int logical = logical_tile();
    long long i0 = 0, j0 = 0;
    auto aim = [&](int tile) {
        const int band = tile / (8 * p.tb), in = tile - band * 8 * p.tb, rows = min(8, p.ta - band * 8);
        i0 = (long long)(band * 8 + in % rows) * 256;
        j0 = (long long)(in / rows) * 256;
        t.aim(F8Src{p.b.codes + j0 * p.b.stride, p.b.scales + j0 * p.b.sstride, (unsigned)p.b.stride, (unsigned)p.b.sstride, (int)min(255ll, p.b.n - 1 - j0)},
              F8Src{p.a.codes + i0 * p.a.stride, p.a.scales + i0 * p.a.sstride, (unsigned)p.a.stride, (unsigned)p.a.sstride, (int)min(255ll, p.a.n - 1 - i0)});
    };
    if (logical < tiles) aim(logical);
    for (int tile = logical; tile < tiles; tile += gridDim.x) {
        F8Big::Acc acc;
        zero_acc(acc);
        t.run(acc);
        const int lane = F8Big::lane_now();
        const F8Out o = out_tile(p, i0, j0);
        const int r = t.wn * 128 + (lane & 31), c = t.wm * 128;
        if (tile + (int)gridDim.x < tiles) aim(tile + gridDim.x);
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                store32<BF>(o, r + n * 32, c + m * 32, lane >> 5, acc[m][n]);
                __builtin_amdgcn_sched_barrier(0);
            }
    }
}

// Few rows of a: (16 NT) rows of a x (16 MT) rows of b per workgroup.  Its W waves share K, each with a ring of its own and no
// barrier, and add up through LDS.  1 x 4096 x 4096: 6.0 us; 64 x 4096 x 4096: 6.4 us, 2.6 TB/s of b; 128 x 4096 x 4096: 8.5 us.
template <int MT, int NT, int W, int S, bool BF>
__global__ void __launch_bounds__(W * 64) f8_matmul_split_kernel(F8MatmulArgs p) {
    using T = F8Tile<MT, NT, 1, 1, S, true>;
    extern __shared__ __align__(16) unsigned char smem[];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int tile = logical_tile();
    const long long i0 = (long long)(tile % p.ta) * T::QR, j0 = (long long)(tile / p.ta) * T::XR;
    const int each = ((p.nblk + W - 1) / W + 3) & ~3;   // whole scale words
    const int kb = wave * each, nblk = min(each, p.nblk - kb);
    f32x4_t acc[MT][NT];
    zero_acc(acc);
    T t;
    t.init(smem + wave * T::LDS, nblk);
    if (nblk > 0) {
        t.aim(F8Src{p.b.codes + j0 * p.b.stride + (size_t)kb * 128, p.b.scales + j0 * p.b.sstride + kb, (unsigned)p.b.stride, (unsigned)p.b.sstride, (int)min((long long)T::XR - 1, p.b.n - 1 - j0)},
              F8Src{p.a.codes + i0 * p.a.stride + (size_t)kb * 128, p.a.scales + i0 * p.a.sstride + kb, (unsigned)p.a.stride, (unsigned)p.a.sstride, (int)min((long long)T::QR - 1, p.a.n - 1 - i0)});
        t.run(acc);
    }
    __syncthreads();   // the rings make room for the sums
    f32x4_t* part = reinterpret_cast<f32x4_t*>(smem);   // [wave][MT][NT][64]
    static_assert(W * MT * NT * 1024 <= W * T::LDS, "the sums take the rings' place");
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) part[((wave * MT + m) * NT + n) * 64 + t.lane] = acc[m][n];
    __syncthreads();
    const F8Out o = out_tile(p, i0, j0);
    const int frow = t.lane & 15, fq = t.lane >> 4;
    for (int f = wave; f < MT * NT; f += W) {
        f32x4_t v = part[f * 64 + t.lane];
#pragma unroll
        for (int w = 1; w < W; ++w) v += part[(w * MT * NT + f) * 64 + t.lane];
        store4<BF>(o, (f % NT) * 16 + frow, (f / NT) * 16 + fq * 4, v);
    }
}

template <int MT, int NT, int WM, int WN, int S, bool BF>
static hipError_t launch_tile(F8MatmulArgs& p, hipStream_t s) {
    using T = F8Tile<MT, NT, WM, WN, S>;
    p.ta = (int)((p.a.n + T::QR - 1) / T::QR);
    p.tb = (int)((p.b.n + T::XR - 1) / T::XR);
    if (T::LDS > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(f8_matmul_tile_kernel<MT, NT, WM, WN, S, BF>), hipFuncAttributeMaxDynamicSharedMemorySize, T::LDS);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((f8_matmul_tile_kernel<MT, NT, WM, WN, S, BF>), dim3((unsigned)((long long)p.ta * p.tb)), dim3(T::THREADS), T::LDS, s, p);
    return hipGetLastError();
}
template <bool BF>
static hipError_t launch_big(F8MatmulArgs& p, int num_cu, hipStream_t s) {
    p.ta = (int)((p.a.n + 255) / 256);
    p.tb = (int)((p.b.n + 255) / 256);
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(f8_matmul_big_kernel<BF>), hipFuncAttributeMaxDynamicSharedMemorySize, F8Big::LDS);
    if (e != hipSuccess) return e;
    const long long tiles = (long long)p.ta * p.tb;
    hipLaunchKernelGGL(f8_matmul_big_kernel<BF>, dim3((unsigned)(tiles < num_cu ? tiles : num_cu)), dim3(256), F8Big::LDS, s, p);
    return hipGetLastError();
}
template <int MT, int NT, int W, int S, bool BF>
static hipError_t launch_split(F8MatmulArgs& p, hipStream_t s) {
    using T = F8Tile<MT, NT, 1, 1, S, true>;
    p.ta = (int)((p.a.n + T::QR - 1) / T::QR);
    p.tb = (int)((p.b.n + T::XR - 1) / T::XR);
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(f8_matmul_split_kernel<MT, NT, W, S, BF>), hipFuncAttributeMaxDynamicSharedMemorySize, W * T::LDS);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((f8_matmul_split_kernel<MT, NT, W, S, BF>), dim3((unsigned)((long long)p.ta * p.tb)), dim3(W * 64), W * T::LDS, s, p);
    return hipGetLastError();
}
template <bool BF>
static hipError_t launch_t(F8MatmulArgs& p, int num_cu, hipStream_t s) {
    // One launch of T tiles takes as many rounds as it has times the chip's places for their workgroups.  A round's time was measured as
    // (fixed part) + (part per block of K), in units of 10 ns, for 1 to 8192 rows of a, 700 to 32768 of b and K of 141 to 8192; the least is within
    // a tenth of the fastest tile for 33 of 35 sizes.  All tiles read slabs at the rate of the caches and convert every fragment that a wave
    // multiplies, so that small tiles cost less per tile and more per product.  us in tiles of (a x b) 16 x 16, 32 x 32, 64 x 32, 64 x 64 whose waves
    // share K, and of 64 x 64, 128 x 128 and 256 x 256 whose waves share slabs, K = 4096:
    //     1 x 4096      6.6    6.0    8.1   10.8    14.4   31.1   65.5
    //    64 x 4096     11.6    6.4    8.5   11.0    15.1   32.1   65.3
    //   128 x 4096     21.2   10.1    8.5   11.2    14.8   32.8   66.3
    //   256 x 4096     41.3   18.3   15.1   11.8    15.4   32.7   67.5
    //    16 x 12288    11.7   11.4   14.8   12.1    14.7   31.5   66.1
    //    48 x 12288    24.6   14.6   15.1   12.2    14.9   32.1   66.2
    //   512 x 4096     82.4   35.1   28.4   21.6    22.5   33.0   67.6
    //  1024 x 4096      169   74.6   57.0   42.7    42.5   34.2   67.6
    //  2048 x 4096        -      -    149   93.3    89.5   57.7   72.2
    //  4096 x 4096        -      -    288    178     177    121   97.3
    // and K = 1024: 512 x 4096 in 64 x 64 8.7 (12.7 with shared K, 11.7 in 128 x 128), 1024 x 4096 14.9 (23.7, 12.5).
    const long long m = p.a.n, n = p.b.n, nb = p.nblk;
    const auto tiles = [&](int tm, int tn) { return ((m + tm - 1) / tm) * ((n + tn - 1) / tn); };
    const auto cost = [&](int tm, int tn, int places, long long fixed, long long block) {
        const long long at_once = (long long)places * num_cu;
        return (tiles(tm, tn) + at_once - 1) / at_once * (fixed + block * nb);
    };
    // (two workgroups of a CU share its caches and pipes: alone each is faster)
    const std::initializer_list<long long> us = {
        cost(16, 16, 1, 160, 6), cost(32, 32, 1, 240, 6), cost(64, 32, 1, 300, 13), cost(64, 64, 1, 430, 20),
        tiles(64, 64) <= num_cu ? 340 + 34 * nb : cost(64, 64, 2, 240, 60), tiles(128, 128) <= num_cu ? 260 + 90 * nb : cost(128, 128, 2, 460, 173),
        cost(256, 256, 1, 1400, 255)};
    switch (std::min_element(us.begin(), us.end()) - us.begin()) {
        case 0: return launch_split<1, 1, 8, 3, BF>(p, s);
        case 1: return launch_split<2, 2, 8, 2, BF>(p, s);
        case 2: return launch_split<2, 4, 4, 3, BF>(p, s);
        case 3: return launch_split<4, 4, 4, 2, BF>(p, s);
        case 4: return launch_tile<2, 2, 2, 2, 4, BF>(p, s);
        case 5: return launch_tile<4, 4, 2, 2, 2, BF>(p, s);
        default: return launch_big<BF>(p, num_cu, s);
    }
}

hipError_t launch_f8_matmul(const F8Mat& a, const F8Mat& b, int k, void* out, int out_dtype, long long out_stride, int num_cu, hipStream_t s) {
    if (a.n <= 0 || b.n <= 0) return hipSuccess;
    F8MatmulArgs p = {};
    p.a = a;
    p.b = b;
    p.nblk = f8_blocks(k);
    p.out = static_cast<unsigned short*>(out);
    p.ostride = out_stride;
    return out_dtype == 2 ? launch_t<true>(p, num_cu, s) : launch_t<false>(p, num_cu, s);
}

}  // namespace ssmi

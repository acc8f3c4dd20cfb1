// f8_matmul.hip - the product of two matrices of 8-bit rows (f8.h):
//
//   out[i][j] = sum over blocks b of 2^(sa[i,b] - 127) 2^(sb[j,b] - 127) sum over the 128 codes of b of a[i,.] b[j,.]
//
// rounded once to 16 bits.  Tiles of 256 x 256 where there are enough of them for every CU, tiles of 128 x 128 below that, and for a
// few rows of `a` (a decoding batch) a kernel that streams the rows of `b` straight into registers, bound by reading `b` once.
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
    bool vec, vec8; // four (eight) neighbours leave as one 8-byte (16-byte) store
    int ta, tb;     // tiles along a and b
};

// a tile of the output: rows x cols of it exist
struct F8Out {
    unsigned short* base;
    long long ostride;
    int rows, cols;
    bool vec, vec8;
};
__device__ __forceinline__ F8Out out_tile(const F8MatmulArgs& p, long long i0, long long j0) {
    return F8Out{p.out + i0 * p.ostride + j0, p.ostride, (int)min(256ll, p.a.n - i0), (int)min(256ll, p.b.n - j0), p.vec, p.vec8};
}
// N neighbouring columns c.. of row r, two to a word
template <int N>
__device__ __forceinline__ void store_words(const F8Out& t, bool vec, int r, int c, const unsigned (&w)[N / 2]) {
    if (r >= t.rows || c >= t.cols) return;
    unsigned short* o = t.base + (unsigned long long)(unsigned)r * (unsigned long long)t.ostride + c;
    if (vec && c + N <= t.cols) {
        if constexpr (N == 8) *reinterpret_cast<uint4*>(o) = uint4{w[0], w[1], w[2], w[3]};
        else *reinterpret_cast<uint2*>(o) = uint2{w[0], w[1]};
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (c + e < t.cols) o[e] = (unsigned short)(w[e / 2] >> (16 * (e & 1)));
    }
}
template <bool BF>
__device__ __forceinline__ void store4(const F8Out& t, int r, int c, const f32x4_t& v) {
    const unsigned w[2] = {narrow2<BF>(v[0], v[1]), narrow2<BF>(v[2], v[3])};
    store_words<4>(t, t.vec, r, c, w);
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
        store_words<8>(t, t.vec8, r, c + 8 * (g + h), w);
    }
}

// b's rows are the matrix instruction's rows: a lane then holds four neighbouring columns of one output row
template <int MT, int NT, int WM, int WN, bool BF>
__global__ void __launch_bounds__(WM * WN * 64) f8_matmul_tile_kernel(F8MatmulArgs p) {
    using T = F8Tile<MT, NT, WM, WN>;
    extern __shared__ __align__(16) unsigned char smem[];
    const int tile = blockIdx.x;
    const int ti = tile % p.ta, tj = tile / p.ta;
    const long long i0 = (long long)ti * T::QR, j0 = (long long)tj * T::XR;
    F8Src x{p.b.codes + j0 * p.b.stride, p.b.scales + j0 * p.b.sstride, (unsigned)p.b.stride, (unsigned)p.b.sstride, (int)min((long long)T::XR - 1, p.b.n - 1 - j0)};
    F8Src q{p.a.codes + i0 * p.a.stride, p.a.scales + i0 * p.a.sstride, (unsigned)p.a.stride, (unsigned)p.a.sstride, (int)min((long long)T::QR - 1, p.a.n - 1 - i0)};
    f32x4_t acc[MT][NT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NT; ++n) acc[m][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    T::run(acc, smem, x, q, p.nblk);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int wm = wave / WN, wn = wave % WN, frow = lane & 15, fq = lane >> 4;
    const F8Out o = out_tile(p, i0, j0);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m)
            store4<BF>(o, (wn * NT + n) * 16 + frow, (wm * MT + m) * 16 + fq * 4, acc[m][n]);
}

// 256 x 256 tiles, a wave per SIMD: workgroups stay, the first slab of the next tile travels under this one's epilogue.
// Tiles are numbered in bands of eight along a, and consecutive workgroups go round the XCDs: the 32 tiles of an XCD cover 8 x 4,
// twelve operand panels for its L2.
// 8192^3: 455 us, 2.42 PFLOP/s; 4096 x 8192 x 8192: 198 us, 2.78; 4096^3: 61 us, 2.24 (tiles of 128 x 128: 585, 292, 71 us).
// The matrix pipe alone reaches 4.9 PFLOP/s on registers, with the operands' way through LDS the chip's power is the limit.
template <bool BF>
__global__ void __launch_bounds__(256, 1) f8_matmul_big_kernel(F8MatmulArgs p) {
    extern __shared__ __align__(16) unsigned char smem[];
    F8Big t;
    t.init(smem, p.nblk);
    const int tiles = p.ta * p.tb;
    const int logical = (gridDim.x & 7) == 0 ? (int)((blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3)) : (int)blockIdx.x;
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
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int n = 0; n < 4; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[m][n][i] = 0.f;
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

// Few rows of a: 16 rows of b per workgroup, its eight waves take every eighth block of K each and add up through LDS.
template <int AT, bool BF>
__global__ void __launch_bounds__(512) f8_matmul_rows_kernel(F8MatmulArgs p) {
    __shared__ f32x4_t part[8][AT][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int frow = lane & 15, fq = lane >> 4;
    const long long j0 = (long long)blockIdx.x * 16, i0 = (long long)blockIdx.y * (AT * 16);
    const long long jr = min(j0 + frow, p.b.n - 1);
    const unsigned char* xp = p.b.codes + jr * p.b.stride + fq * 16;
    const unsigned char* xs = p.b.scales + jr * p.b.sstride;
    const unsigned char* ap[AT];
    const unsigned char* as[AT];
    f32x4_t acc[AT];
#pragma unroll
    for (int t = 0; t < AT; ++t) {
        const long long ir = min(i0 + t * 16 + frow, p.a.n - 1);
        ap[t] = p.a.codes + ir * p.a.stride + fq * 16;
        as[t] = p.a.scales + ir * p.a.sstride;
        acc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    for (int kb = wave; kb < p.nblk; kb += 8) {
        const size_t o = (size_t)kb * 128;
        const i32x8_t x = join8(*reinterpret_cast<const i32x4_t*>(xp + o), *reinterpret_cast<const i32x4_t*>(xp + o + 64));
        const int sx = xs[kb];
#pragma unroll
        for (int t = 0; t < AT; ++t) {
            const i32x8_t a = join8(*reinterpret_cast<const i32x4_t*>(ap[t] + o), *reinterpret_cast<const i32x4_t*>(ap[t] + o + 64));
            acc[t] = mfma_f8<0>(x, a, acc[t], sx, (int)as[t][kb]);
        }
    }
#pragma unroll
    for (int t = 0; t < AT; ++t) part[wave][t][lane] = acc[t];
    __syncthreads();
    const F8Out o = out_tile(p, i0, j0);
    for (int t = wave; t < AT; t += 8) {
        f32x4_t v = part[0][t][lane];
#pragma unroll
        for (int w = 1; w < 8; ++w) v += part[w][t][lane];
        store4<BF>(o, t * 16 + frow, fq * 4, v);
    }
}

template <int MT, int NT, int WM, int WN, bool BF>
static hipError_t launch_tile(F8MatmulArgs& p, hipStream_t s) {
    using T = F8Tile<MT, NT, WM, WN>;
    p.ta = (int)((p.a.n + T::QR - 1) / T::QR);
    p.tb = (int)((p.b.n + T::XR - 1) / T::XR);
    if (T::LDS > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(f8_matmul_tile_kernel<MT, NT, WM, WN, BF>), hipFuncAttributeMaxDynamicSharedMemorySize, T::LDS);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((f8_matmul_tile_kernel<MT, NT, WM, WN, BF>), dim3((unsigned)((long long)p.ta * p.tb)), dim3(T::THREADS), T::LDS, s, p);
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
template <bool BF>
static hipError_t launch_t(F8MatmulArgs& p, int num_cu, hipStream_t s) {
    const long long m = p.a.n, n = p.b.n;
    if (m <= 64) {
        const int at = m <= 16 ? 1 : m <= 32 ? 2 : 4;
        const dim3 grid((unsigned)((n + 15) / 16), 1);
        if (at == 1) hipLaunchKernelGGL((f8_matmul_rows_kernel<1, BF>), grid, dim3(512), 0, s, p);
        else if (at == 2) hipLaunchKernelGGL((f8_matmul_rows_kernel<2, BF>), grid, dim3(512), 0, s, p);
        else hipLaunchKernelGGL((f8_matmul_rows_kernel<4, BF>), grid, dim3(512), 0, s, p);
        return hipGetLastError();
    }
    if (((m + 255) / 256) * ((n + 255) / 256) >= num_cu) return launch_big<BF>(p, num_cu, s);
    return launch_tile<4, 4, 2, 2, BF>(p, s);
}

hipError_t launch_f8_matmul(const F8Mat& a, const F8Mat& b, int k, void* out, int out_dtype, long long out_stride, int num_cu, hipStream_t s) {
    if (a.n <= 0 || b.n <= 0) return hipSuccess;
    F8MatmulArgs p = {};
    p.a = a;
    p.b = b;
    p.nblk = f8_blocks(k);
    p.out = static_cast<unsigned short*>(out);
    p.ostride = out_stride;
    p.vec = ((uintptr_t)out & 7) == 0 && (out_stride & 3) == 0;
    p.vec8 = ((uintptr_t)out & 15) == 0 && (out_stride & 7) == 0;
    return out_dtype == 2 ? launch_t<true>(p, num_cu, s) : launch_t<false>(p, num_cu, s);
}

}  // namespace ssmi

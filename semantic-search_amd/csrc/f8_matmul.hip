// f8_matmul.hip - the product of two matrices of 8-bit rows (f8.h):
//
//   out[i][j] = sum over blocks b of 2^(sa[i,b] - 127) 2^(sb[j,b] - 127) sum over the 128 codes of b of a[i,.] b[j,.]
//
// rounded once to 16 bits.  Two kernels: a tile kernel for the matrix pipe's share of the work, and for a few rows of `a` (a
// decoding batch) one that streams the rows of `b` straight into registers, bound by reading `b` once.
#include "f8_tile.h"

namespace ssmi {

template <bool BF>
__device__ __forceinline__ unsigned short narrow16(float v) {
    if constexpr (BF) return bf16_t(v).x;
    else return __half_as_ushort(__float2half_rn(v));
}

struct F8MatmulArgs {
    F8Mat a, b;
    int nblk;
    unsigned short* out;
    long long ostride;
    bool vec;       // four neighbours leave as one 8-byte store
    int ta, tb;     // tiles along a and b
};

// four neighbouring columns j0.. of row i
template <bool BF>
__device__ __forceinline__ void store4(const F8MatmulArgs& p, long long i, long long j0, const f32x4_t& v) {
    if (i >= p.a.n || j0 >= p.b.n) return;
    unsigned short* o = p.out + i * p.ostride + j0;
    if (p.vec && j0 + 4 <= p.b.n) {
        uint2 w;
        w.x = (unsigned)narrow16<BF>(v[0]) | ((unsigned)narrow16<BF>(v[1]) << 16);
        w.y = (unsigned)narrow16<BF>(v[2]) | ((unsigned)narrow16<BF>(v[3]) << 16);
        *reinterpret_cast<uint2*>(o) = w;
    } else {
#pragma unroll
        for (int t = 0; t < 4; ++t)
            if (j0 + t < p.b.n) o[t] = narrow16<BF>(v[t]);
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
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int m = 0; m < MT; ++m)
            store4<BF>(p, i0 + (wn * NT + n) * 16 + frow, j0 + (wm * MT + m) * 16 + fq * 4, acc[m][n]);
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
    for (int t = wave; t < AT; t += 8) {
        f32x4_t v = part[0][t][lane];
#pragma unroll
        for (int w = 1; w < 8; ++w) v += part[w][t][lane];
        store4<BF>(p, i0 + t * 16 + frow, j0 + fq * 4, v);
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
    if (((m + 255) / 256) * ((n + 255) / 256) >= num_cu) return launch_tile<8, 4, 2, 4, BF>(p, s);
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
    return out_dtype == 2 ? launch_t<true>(p, num_cu, s) : launch_t<false>(p, num_cu, s);
}

}  // namespace ssmi

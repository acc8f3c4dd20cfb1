// f8_rows.hip - the row kernels around the 8-bit format of f8.h: the quantiser with the root-mean-square norm that feeds it,
// the way back, and the row store's gather and candidate scores.
//
//   h = x + r, rounded to x's type and stored (the residual stream); without r: h = x
//   y = h * 1 / sqrt(mean(h^2) + eps) * w              (norm)
//   y = y / max(|y|_2, 1e-12)                          (unit: what goes into an inner-product index)
//   s = the smallest power of two with max|y| <= 448 s over 128 elements, code = y / s to nearest even
//
// An embedding model ends in exactly this chain (its last norm, then core/qwen3_vl_embedding.py:447-448 of the reference
// normalises the pooled row): one pass here reads x and r once and writes the sum, the codes and the scales once.  Bound by
// memory; a row stays in registers between the reductions, so nothing is read twice.
#include "f8.h"
#include "topk.h"

namespace ssmi {

template <typename T>
struct alignas(16) Pack8 {};
template <>
struct alignas(16) Pack8<float> { float v[8]; };
template <>
struct alignas(16) Pack8<__half> { __half v[8]; };
template <>
struct alignas(16) Pack8<bf16_t> { bf16_t v[8]; };

// elements e0 .. e0+7 of a row of d as floats, zeros beyond d
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* row, int e0, int d, float (&o)[8]) {
    if (VEC && e0 + 8 <= d) {
        const Pack8<T> p = *reinterpret_cast<const Pack8<T>*>(row + e0);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = (float)p.v[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = e0 + j < d ? (float)row[e0 + j] : 0.f;
    }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* row, int e0, int d, const float (&o)[8]) {
    if (VEC && e0 + 8 <= d) {
        Pack8<T> p;
#pragma unroll
        for (int j = 0; j < 8; ++j) p.v[j] = (T)o[j];
        *reinterpret_cast<Pack8<T>*>(row + e0) = p;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (e0 + j < d) row[e0 + j] = (T)o[j];
    }
}

// (a, b) summed over the threads that share a row: a wave, or the whole block
template <bool WAVE>
__device__ __forceinline__ void row_sums(double& a, double& b, double2* lds) {
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) {
        a += __shfl_xor(a, d);
        b += __shfl_xor(b, d);
    }
    if constexpr (!WAVE) {
        const int nw = (int)(blockDim.x >> 6);
        if (nw > 1) {
            __syncthreads();  // the words of the previous row are free
            if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = double2{a, b};
            __syncthreads();
            a = b = 0.0;
            for (int w = 0; w < nw; ++w) { a += lds[w].x; b += lds[w].y; }
        }
    }
}

// 64 bits -> an fp32 whose last bit says that something was cut: rounding that again, to the four bits of a code, gives what rounding the
// 64 bits gives, and a value above 448 s stays above it.  (To nearest twice: a code in about a million was one step off, or its block twice as
// coarse.)  Below 2^-126 to nearest.
__device__ __forceinline__ float narrow_odd(double y) {
    unsigned long long b = (unsigned long long)__double_as_longlong(y);
    unsigned lo = (unsigned)b;
    lo = (lo | ((lo & 0x1fffffffu) + 0x1fffffffu)) & 0xe0000000u;   // (the addition carries into bit 29 unless all below are zero)
    return (float)__longlong_as_double((long long)((b & 0xffffffff00000000ull) | lo));
}

// Eight elements per thread and pass: 16 threads hold a block of 128, so its maximum is four DPP steps and the codes leave as
// 8 bytes per lane.  WAVE: a row per wave (rows up to 2048 elements, many of them), else a row per block.
// The norm's sums and its one factor per row are 64-bit and y is rounded once, to its code (narrow_odd): an element's code is that of the exact row
// unless y lies within 2^-40 of a border.  (With fp32 sums and factors codes part from the exact ones a million times as often; the 64-bit products
// hide behind memory.)  unit needs no second pass: |y| = f |h w| for y = f h w.
// The quantiser is bound by memory (200000 x 2048 fp32: 376 us, 5.4 TB/s), the norm by what little of its rows is in flight while it
// reduces (32768 x 4096 bf16 with a residual: 218 us, 4.3 TB/s; 200000 x 2048 fp32, unit: 479 us, 4.3 TB/s; a row of 4096 per wave
// needs 254 registers and took 574 us).
// (Four passes of 1024 threads would take rows of 32768 elements through the norm, but spill.)
template <typename T, int ITER, bool WAVE, bool VEC, bool NORM>
__global__ void __launch_bounds__(WAVE ? 256 : 1024, WAVE ? 1 : 5) f8_rows_kernel(F8NormArgs a) {
    __shared__ double2 red[16];
    const int tpr = WAVE ? 64 : (int)blockDim.x;
    const int t = WAVE ? (int)(threadIdx.x & 63) : (int)threadIdx.x;
    const long long step = WAVE ? (long long)gridDim.x * 4 : (long long)gridDim.x;
    const int ld = (a.d + kF8Block - 1) / kF8Block * kF8Block;
    for (long long row = WAVE ? (long long)blockIdx.x * 4 + (threadIdx.x >> 6) : (long long)blockIdx.x; row < a.n; row += step) {
        const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
        // the norm needs its whole row in registers (one turn: launch_rows_t); without it a row is any number of turns
        for (int c0 = 0; c0 < ld; c0 += ITER * tpr * 8) {
            float v[ITER][8];
#pragma unroll
            for (int i = 0; i < ITER; ++i) load8<T, VEC>(x, c0 + (i * tpr + t) * 8, a.d, v[i]);
            if (NORM && a.residual) {
                const T* r = static_cast<const T*>(a.residual) + row * a.r_stride;
                T* ro = static_cast<T*>(a.residual_out) + row * a.ro_stride;
#pragma unroll
                for (int i = 0; i < ITER; ++i) {
                    float u[8];
                    load8<T, VEC>(r, c0 + (i * tpr + t) * 8, a.d, u);
                    // the norm continues from the sum as it is stored, so that a caller who starts again from the stored
                    // residual gets the same row
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[i][j] = (float)(T)(v[i][j] + u[j]);
                    store8<T, VEC>(ro, c0 + (i * tpr + t) * 8, a.d, v[i]);
                }
            }
            if constexpr (NORM) {
                auto weights = [&](int e0, float (&w)[8]) {
                    if (a.weight && e0 < a.d) {
                        if (a.weight_dtype == 0) load8<float, VEC>(static_cast<const float*>(a.weight), e0, a.d, w);
                        else if (a.weight_dtype == 1) load8<__half, VEC>(static_cast<const __half*>(a.weight), e0, a.d, w);
                        else load8<bf16_t, VEC>(static_cast<const bf16_t*>(a.weight), e0, a.d, w);
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) w[j] = 1.f;
                    }
                };
                double hh = 0.0, yy = 0.0;   // sums of h^2 and (h w)^2
#pragma unroll
                for (int i = 0; i < ITER; ++i) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) hh = fma((double)v[i][j], (double)v[i][j], hh);
                    if (a.unit) {
                        float w[8];
                        weights(c0 + (i * tpr + t) * 8, w);
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const double y = (double)v[i][j] * (double)w[j];
                            yy = fma(y, y, yy);
                        }
                    }
                }
                row_sums<WAVE>(hh, yy, red);
                // (every lane computes the factor: a 64-bit root and division each took as long as the row's own arithmetic)
                double f = rsqrt(fma(hh, a.inv_d, (double)a.eps));
                if (a.unit) f = yy * f * f >= 1e-24 ? rsqrt(yy) : f * 1e12;   // |y| = f sqrt(yy), below 1e-12 the divisor stays there
#pragma unroll
                for (int i = 0; i < ITER; ++i) {
                    float w[8];
                    weights(c0 + (i * tpr + t) * 8, w);
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[i][j] = narrow_odd((double)v[i][j] * (double)w[j] * f);
                }
            }
#pragma unroll
            for (int i = 0; i < ITER; ++i) {
                const int e0 = c0 + (i * tpr + t) * 8;
                unsigned b;
                const uint2 o = f8_pack8(v[i], e0, a.d, b);
                if (e0 < ld) {
                    *reinterpret_cast<uint2*>(a.codes + row * a.stride + e0) = o;
                    if ((t & 15) == 0) a.scales[row * a.sstride + e0 / kF8Block] = (unsigned char)b;
                }
            }
        }
    }
}

static bool aligned16(const void* p, long long stride, int el) {
    return ((uintptr_t)p & 15) == 0 && ((stride * el) & 15) == 0;
}

template <typename T>
static hipError_t launch_rows_t(const F8NormArgs& a, int num_cu, hipStream_t s) {
    const int per = f8_ld(a.d) / 8;  // threads x passes of a row
    bool vec = aligned16(a.x, a.x_stride, sizeof(T));
    if (a.residual) vec = vec && aligned16(a.residual, a.r_stride, sizeof(T)) && aligned16(a.residual_out, a.ro_stride, sizeof(T));
    if (a.weight) vec = vec && ((uintptr_t)a.weight & 15) == 0;
    // a row per wave while the rows outnumber the waves that fill the card and fit a wave's registers (256 lanes' worth)
    const bool wave = per <= 256 && a.n >= 4ll * num_cu;
    int threads = 256, iter;
    if (wave) {
        iter = (per + 63) / 64;
    } else {
        threads = per <= 64 ? 64 : per <= 128 ? 128 : per <= 256 ? 256 : per <= 512 ? 512 : 1024;
        // many rows: half the threads and two passes of a row each keep more rows in flight per CU
        if (a.n >= 4ll * num_cu && threads >= 512) threads = per <= 512 ? 256 : per <= 1024 ? 512 : 1024;
        iter = (per + threads - 1) / threads;
    }
    iter = iter <= 1 ? 1 : iter <= 2 || !wave ? 2 : 4;
    const long long blocks = wave ? (a.n + 3) / 4 : a.n;
    const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536));
#define GO(I, W, V) { if (a.norm) hipLaunchKernelGGL((f8_rows_kernel<T, I, W, V, true>), grid, dim3(threads), 0, s, a); \
                      else hipLaunchKernelGGL((f8_rows_kernel<T, I, W, V, false>), grid, dim3(threads), 0, s, a); }
#define GO_V(I, W) { if (vec) GO(I, W, true) else GO(I, W, false) }
    if (wave) { if (iter == 1) GO_V(1, true) else if (iter == 2) GO_V(2, true) else GO_V(4, true) }
    else if (iter == 1) GO_V(1, false)
    else GO_V(2, false)
#undef GO_V
#undef GO
    return hipGetLastError();
}
hipError_t launch_f8_rows(const F8NormArgs& a, int num_cu, hipStream_t s) {
    if (a.n <= 0) return hipSuccess;
    if (a.dtype == 0) return launch_rows_t<float>(a, num_cu, s);
    if (a.dtype == 1) return launch_rows_t<__half>(a, num_cu, s);
    return launch_rows_t<bf16_t>(a, num_cu, s);
}

// ---- the way back: 8 codes per thread (exact in every type: 4 significant bits times a power of two, as long as the
// power is in the type's range; fp16 rounds and saturates to infinity like any narrowing)
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) f8_dequantize_kernel(F8Mat m, int d, T* out, long long out_stride) {
    const int per = (d + 7) / 8;
    const long long total = m.n * per, step = (long long)gridDim.x * blockDim.x;
    for (long long c = (long long)blockIdx.x * blockDim.x + threadIdx.x; c < total; c += step) {
        const long long row = c / per;
        const int e0 = (int)(c - row * per) * 8;
        const uint2 w = *reinterpret_cast<const uint2*>(m.codes + row * m.stride + e0);
        const float s = f8_scale(m.scales[row * m.sstride + e0 / kF8Block]);
        float lo[4], hi[4], o[8];
        f8_unpack4(w.x, lo);
        f8_unpack4(w.y, hi);
#pragma unroll
        for (int j = 0; j < 4; ++j) { o[j] = lo[j] * s; o[4 + j] = hi[j] * s; }
        store8<T, VEC>(out + row * out_stride, e0, d, o);
    }
}
hipError_t launch_f8_dequantize(const F8Mat& m, int d, void* out, int out_dtype, long long out_stride, int num_cu, hipStream_t s) {
    if (m.n <= 0) return hipSuccess;
    const long long blocks = (m.n * ((d + 7) / 8) + 255) / 256;
    const long long most = (long long)num_cu * 32;
    const dim3 grid((unsigned)(blocks < most ? blocks : most));
    const bool vec = aligned16(out, out_stride, out_dtype == 0 ? 4 : 2);
#define GO(T) { if (vec) hipLaunchKernelGGL((f8_dequantize_kernel<T, true>), grid, dim3(256), 0, s, m, d, (T*)out, out_stride); \
                else hipLaunchKernelGGL((f8_dequantize_kernel<T, false>), grid, dim3(256), 0, s, m, d, (T*)out, out_stride); }
    if (out_dtype == 0) GO(float)
    else if (out_dtype == 1) GO(__half)
    else GO(bf16_t)
#undef GO
    return hipGetLastError();
}

// ---- row store reads ----
struct F8Row { const unsigned char* codes; const unsigned char* scales; };
__device__ __forceinline__ F8Row f8_row(const F8View& v, long long row) {
    const long long seg = row >> v.X.seg_shift, off = row & ((1ll << v.X.seg_shift) - 1);
    return F8Row{static_cast<const unsigned char*>(v.X.segs[seg]) + off * v.X.ld, static_cast<const unsigned char*>(v.ssegs[seg]) + off * v.sld};
}
__device__ __forceinline__ float f8_value(const F8Row& r, int e) {
    float a, b;
    f8_unpack2<false>(r.codes[e], a, b);
    return a * f8_scale(r.scales[e / kF8Block]);
}

__global__ void f8_gather_kernel(F8View v, const int64_t* __restrict__ ids, long long n, int d, float* __restrict__ out, int* __restrict__ bad) {
    const long long i = blockIdx.x;
    const int64_t id = ids[i];
    float* o = out + (size_t)i * d;
    if (id < 0 || id >= v.X.nrows) {
        for (int e = threadIdx.x; e < d; e += blockDim.x) o[e] = 0.f;
        if (threadIdx.x == 0) atomicExch(bad, 1);
        return;
    }
    const F8Row r = f8_row(v, id);
    for (int e = threadIdx.x; e < d; e += blockDim.x) o[e] = f8_value(r, e);
}
hipError_t launch_f8_gather(const F8View& v, const int64_t* ids, long long n, int d, float* out, int* bad, hipStream_t s) {
    if (n <= 0) return hipSuccess;
    hipLaunchKernelGGL(f8_gather_kernel, dim3((unsigned)n), dim3(256), 0, s, v, ids, n, d, out, bad);
    return hipGetLastError();
}

__global__ void __launch_bounds__(256) f8_score_rows_kernel(F8View v, const int64_t* __restrict__ ids, long long n, int d,
                                                            const float* __restrict__ neg, int n_neg, float* __restrict__ out, int* __restrict__ bad) {
    __shared__ float part[4];
    const long long i = blockIdx.x;
    const int64_t id = ids[i];
    if (id < 0 || id >= v.X.nrows) {
        for (int j = threadIdx.x; j < n_neg; j += blockDim.x) out[(size_t)i * n_neg + j] = 0.f;
        if (threadIdx.x == 0) atomicExch(bad, 1);
        return;
    }
    const F8Row r = f8_row(v, id);
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    for (int j = 0; j < n_neg; ++j) {
        const float* q = neg + (size_t)j * d;
        float acc = 0.f;
        for (int e = threadIdx.x; e < d; e += blockDim.x) acc = fmaf(f8_value(r, e), q[e], acc);
        acc = wave_sum(acc);
        if (lane == 0) part[wave] = acc;
        __syncthreads();
        if (threadIdx.x == 0) out[(size_t)i * n_neg + j] = (part[0] + part[1]) + (part[2] + part[3]);
        __syncthreads();
    }
}
hipError_t launch_f8_score_rows(const F8View& v, const int64_t* ids, long long n, int d, const float* neg, int n_neg, float* out,
                                int* bad, hipStream_t s) {
    if (n <= 0 || n_neg <= 0) return hipSuccess;
    hipLaunchKernelGGL(f8_score_rows_kernel, dim3((unsigned)n), dim3(256), 0, s, v, ids, n, d, neg, n_neg, out, bad);
    return hipGetLastError();
}

}  // namespace ssmi

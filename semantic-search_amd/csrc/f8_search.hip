// f8_search.hip - Flat search over 8-bit rows (f8.h): the product of f8_tile.h with the top-k epilogues of the other row types.
//
// Two passes.  The first keeps, for every query, the best k + 16 rows by the matrix instruction's sums (whose error against
// the exact sum is about 1e-6 |q||x|): a streaming scan for a few queries, bound by reading the rows once, or the tile kernel
// with the candidate buffers of the 16-bit kernels (mfma_common.h).  The second sums those candidates' products in 64 bits -
// every product of two codes is exact in fp32 and the scales are powers of two, so the sum is exact or off by a rounding of
// 2^-53 - and sorts them by that, ties by the lower id.  A query therefore gets the same ids and scores in any batch.
//
// Same place on the path as the 16-bit kernels: faiss.IndexFlatIP.search as called from core/index_manager.py:371.
#include "f8_tile.h"
#include "tail_merge.h"
#include <algorithm>

namespace ssmi {

__device__ __forceinline__ uint4 load16_once(const unsigned char* p) {
    typedef unsigned u4 __attribute__((ext_vector_type(4)));
    const u4 v = __builtin_nontemporal_load(reinterpret_cast<const u4*>(p));
    return uint4{v[0], v[1], v[2], v[3]};
}
__device__ __forceinline__ i32x8_t frag(const uint4& lo, const uint4& hi) {
    return i32x8_t{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w, (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
}

// ---- streaming scan: up to BT <= 8 queries per launch row, 16 rows per wave pass ----
// The instruction's sixteen columns cost nothing here (a row of 4096 codes is 1/16 of 32 instructions against 4 KiB of
// memory); columns beyond BT repeat a query and are never looked at.  Rows go straight into registers: four blocks (512
// codes) of 16 rows per stage = eight 16-byte loads per lane, two stages in flight.  Queries sit in LDS, rows of ld + 16 bytes
// so that the 16 lanes of a pass hit 16 different bank groups.
template <int BT, int R>
__global__ void __launch_bounds__(512) f8_scan_kernel(F8View V, F8Mat q, int k, skey_t* partial, TailMerge tail) {
    extern __shared__ __align__(16) unsigned char smem[];
    const int lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int nwaves = (int)(blockDim.x >> 6);
    const int ld = V.X.ld, nblk = ld / kF8Block, nst = (nblk + 3) / 4;
    const int q0 = blockIdx.y * BT, nq = (int)q.n;
    const int qpitch = ld + 16;
    unsigned char* qs = smem;
    int* qsc = reinterpret_cast<int*>(smem + BT * qpitch);   // [BT][nst] words of four scales
    for (int b = 0; b < BT; ++b) {
        const long long qi = min(q0 + b, nq - 1);
        for (int e = threadIdx.x * 16; e < ld; e += blockDim.x * 16)
            *reinterpret_cast<uint4*>(qs + b * qpitch + e) = *reinterpret_cast<const uint4*>(q.codes + qi * q.stride + e);
        for (int e = threadIdx.x; e < nst; e += blockDim.x) qsc[b * nst + e] = *reinterpret_cast<const int*>(q.scales + qi * q.sstride + e * 4);
    }
    __syncthreads();

    WaveTopK<R> top[BT];
    skey_t thr[BT];
#pragma unroll
    for (int b = 0; b < BT; ++b) { top[b].init(); thr[b] = 0; }
    const int col = lane & 15, grp = lane >> 4;
    // a score passes only at or above the gate of its lane's query; NaN never does.  Columns that repeat a query are shut
    float gate = col < BT ? -__builtin_inff() : __builtin_nanf("");

    const unsigned vb = (gridDim.x % 8 == 0) ? (blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8 : blockIdx.x;
    const long long ngroups = (V.X.nrows + 15) >> 4, step = (long long)gridDim.x * nwaves;
    const long long seg_mask = (1ll << V.X.seg_shift) - 1;
    const unsigned char* qlane = qs + (col % BT) * qpitch + grp * 16;
    const int* qslane = qsc + (col % BT) * nst;

    struct Base { const unsigned char* c; const unsigned char* s; };
    auto group_base = [&](long long g) -> Base {
        long long row = (g << 4) + col;   // 16 rows of a group share a segment; beyond the last row: the last
        if (row >= V.X.nrows) row = V.X.nrows - 1;
        const long long seg = (g << 4) >> V.X.seg_shift, off = row & seg_mask;
        return Base{static_cast<const unsigned char*>(V.X.segs[seg]) + off * ld + grp * 16, static_cast<const unsigned char*>(V.ssegs[seg]) + off * V.sld};
    };
    uint4 xa[8], xb[8];
    int sa = 0, sb = 0;
    auto load = [&](uint4 (&x)[8], int& sc, const Base& p, int st) {
        sc = *reinterpret_cast<const int*>(p.s + st * 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int kb = min(st * 4 + j, nblk - 1);   // (a block beyond the row is loaded as the last and not used)
            x[2 * j] = load16_once(p.c + (size_t)kb * 128);
            x[2 * j + 1] = load16_once(p.c + (size_t)kb * 128 + 64);
        }
    };
    long long g = (long long)vb * nwaves + wave;
    if (g >= ngroups) g = -1;
    Base base = {nullptr, nullptr};
    if (g >= 0) { base = group_base(g); load(xa, sa, base, 0); }
    while (g >= 0) {
        const long long gn = g + step < ngroups ? g + step : -1;
        const Base next = gn < 0 ? base : group_base(gn);
        f32x4_t acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
        auto consume = [&](const uint4 (&x)[8], int sc, int st) {
            const int sq = qslane[st];
            const unsigned char* ql = qlane + (size_t)st * 512;
            const auto one = [&](auto jc) {
                constexpr int J = decltype(jc)::value;
                if (st * 4 + J < nblk) {
                    const uint4 lo = *reinterpret_cast<const uint4*>(ql + J * 128), hi = *reinterpret_cast<const uint4*>(ql + J * 128 + 64);
                    acc = mfma_f8<J>(frag(x[2 * J], x[2 * J + 1]), frag(lo, hi), acc, sc, sq);
                }
            };
            one(std::integral_constant<int, 0>());
            one(std::integral_constant<int, 1>());
            one(std::integral_constant<int, 2>());
            one(std::integral_constant<int, 3>());
        };
#pragma unroll 1
        for (int st = 0; st < nst; st += 2) {
            const bool second = st + 1 < nst;
            if (second) load(xb, sb, base, st + 1);
            else load(xb, sb, next, 0);
            __builtin_amdgcn_sched_barrier(0);
            consume(xa, sa, st);
            __builtin_amdgcn_sched_barrier(0);
            if (second) {
                if (st + 2 < nst) load(xa, sa, base, st + 2);
                else load(xa, sa, next, 0);
                __builtin_amdgcn_sched_barrier(0);
                consume(xb, sb, st + 1);
                __builtin_amdgcn_sched_barrier(0);
            } else {   // odd number of stages: the next group's first stage is in xb
                sa = sb;
#pragma unroll
                for (int j = 0; j < 8; ++j) xa[j] = xb[j];
            }
        }
        // acc[i] of lane (col, grp): row 4 grp + i of the group against query col
        const long long row0 = g << 4;
        bool any = false;
#pragma unroll
        for (int i = 0; i < 4; ++i) any |= acc[i] >= gate;
        if (__builtin_amdgcn_ballot_w64(any) != 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                unsigned long long mask = __builtin_amdgcn_ballot_w64(acc[i] >= gate);
                while (mask) {
                    const int src = (int)__builtin_ctzll(mask);
                    mask &= mask - 1;
                    const long long row = row0 + 4 * (src >> 4) + i;
                    if (row >= V.X.nrows) continue;
                    const int qb = src & 15;
                    const skey_t key = make_key(__int_as_float(__builtin_amdgcn_readlane(__float_as_int(acc[i]), src)), (uint32_t)row);
#pragma unroll
                    for (int b = 0; b < BT; ++b) {
                        if (b == qb && key > thr[b]) {
                            top[b].insert(key);
                            thr[b] = top[b].kth(k);
                            if (thr[b] && col == b) gate = key_score(thr[b]);
                        }
                    }
                }
            }
        }
        g = gn;
        base = next;
    }

    __syncthreads();
    skey_t* lds_keys = reinterpret_cast<skey_t*>(smem);
#pragma unroll
    for (int b = 0; b < BT; ++b) {
        block_merge<R>(top[b], lds_keys, wave, nwaves);
        if (wave == 0 && q0 + b < nq) publish_list<R>(top[b], partial + ((size_t)(q0 + b) * gridDim.x + blockIdx.x) * k, k);
        __syncthreads();
    }
    if (tail.counter == nullptr) return;
    if (!tail_last_block(tail.counter + blockIdx.y, gridDim.x, reinterpret_cast<unsigned*>(smem))) return;
#pragma unroll 1
    for (int b = 0; b < BT; ++b) {
        const int qi = q0 + b;
        if (qi >= nq) break;
        merge_partials<R, true>(partial + (size_t)qi * gridDim.x * k, (int)gridDim.x, k, lds_keys, wave, nwaves, tail.D + (size_t)qi * k,
                                tail.I + (size_t)qi * k, 0);
        __syncthreads();
    }
}

// ---- tile kernel: 256 rows x TQ queries per workgroup, a slice of the rows each ----
template <int MT, int NT, int WM, int WN, int R>
__global__ void __launch_bounds__(512) f8_search_tile_kernel(F8View V, F8Mat q, MfmaParams P) {
    using T = F8Tile<MT, NT, WM, WN>;
    static_assert(T::XR == 256 && T::WAVES == 8, "row tile and folds of the 16-bit kernels");
    extern __shared__ __align__(16) unsigned char smem[];
    float* thr_l = reinterpret_cast<float*>(smem + T::LDS);
    unsigned* cnt_l = reinterpret_cast<unsigned*>(thr_l + 256);
    unsigned* kept_l = cnt_l + 256;
    unsigned* flag_l = kept_l + 256;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WN, wn = wave % WN, frow = lane & 15, fq = lane >> 4;
    int logical = blockIdx.x;
    if ((gridDim.x & 7) == 0) logical = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    const int slice = logical / P.nqt, qt = logical % P.nqt;
    const int q0 = qt * T::QR;
    const long long r_begin = (long long)slice * P.rows_per_slice;
    const long long r_end = min(r_begin + P.rows_per_slice, V.X.nrows);
    skey_t* cand = P.cand + (size_t)blockIdx.x * 256 * CAND_CAP;
    if (P.nq > q0 + T::QR) P.nq = q0 + T::QR;   // the folds go by nq: this tile's queries only
    if (tid < 256) {
        thr_l[tid] = q0 + tid < P.nq ? P.thr_floor : __builtin_inff();
        cnt_l[tid] = 0;
        kept_l[tid] = 0;
    }
    if (tid == 0) flag_l[0] = 0;
    __syncthreads();
    const long long seg_mask = (1ll << V.X.seg_shift) - 1;
    const F8Src qsrc{q.codes + (size_t)q0 * q.stride, q.scales + (size_t)q0 * q.sstride, (unsigned)q.stride, (unsigned)q.sstride, (int)min((long long)T::QR - 1, q.n - 1 - q0)};
    unsigned tiles_done = 0;
    for (long long row0 = r_begin; row0 < r_end; row0 += 256) {
        const long long seg = row0 >> V.X.seg_shift, off = row0 & seg_mask;
        const long long left = r_end - row0;
        const F8Src xsrc{static_cast<const unsigned char*>(V.X.segs[seg]) + off * V.X.ld, static_cast<const unsigned char*>(V.ssegs[seg]) + off * V.sld,
                         (unsigned)V.X.ld, (unsigned)V.sld, (int)min(255ll, left - 1)};
        f32x4_t acc[MT][NT];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n) acc[m][n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        T::run(acc, smem, xsrc, qsrc, V.X.ld / kF8Block);
        if (left >= 256) filter_tile<MT, NT, true>(acc, wm * MT * 16, wn * NT * 16, frow, fq, row0, 256, cand, thr_l, cnt_l, flag_l);
        else filter_tile<MT, NT, false>(acc, wm * MT * 16, wn * NT * 16, frow, fq, row0, (int)left, cand, thr_l, cnt_l, flag_l);
        __syncthreads();
        ++tiles_done;
        // fold after row tiles 1, 4, 16, ... of the slice and whenever a candidate buffer is half full
        if (((tiles_done & (tiles_done - 1)) == 0 && (tiles_done & 0x55555555u)) || *flag_l) {
            fold_queries<R>(wave, q0, P, slice, cand, thr_l, cnt_l, kept_l);
            if (lane < 32) {   // the k-th score of any slice bounds the final one: the slices share the highest (mfma.hip)
                const int ql = wave + 8 * lane;
                if (q0 + ql < P.nq) {
                    const float t = thr_l[ql];
                    const unsigned mine = t > SSMI_NEG_MAX ? f32_to_ord(t) : 0u;
                    const unsigned seen = atomicMax(&P.gthr[q0 + ql], mine);
                    if (seen > mine) thr_l[ql] = ord_to_f32(seen);
                }
            }
            __syncthreads();
            if (tid == 0) *flag_l = 0;
        }
    }
    __syncthreads();
    fold_queries<R>(wave, q0, P, slice, cand, thr_l, cnt_l, kept_l);
}

__global__ void f8_zero_kernel(unsigned* p, int n) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n) p[i] = 0;
}

// ---- second pass: 64-bit scores of the candidates, sorted ----
// One workgroup per query, a wave per candidate.  16 codes of a lane belong to one block, so its products add up in 64 bits
// unscaled and meet the block's scale once.
__global__ void __launch_bounds__(1024) f8_finish_kernel(F8View V, F8Mat q, const int64_t* __restrict__ ids, int kp, int k, float* D,
                                                         int64_t* I, int64_t id_offset, unsigned min_ord) {
    __shared__ double score[kMaxK];
    __shared__ int64_t cid[kMaxK];
    __shared__ int nvalid;
    const int lane = lane_id(), wave = threadIdx.x >> 6, nwaves = blockDim.x >> 6;
    const long long qi = blockIdx.x;
    const unsigned char* qc = q.codes + qi * q.stride;
    const unsigned char* qsc = q.scales + qi * q.sstride;
    const long long seg_mask = (1ll << V.X.seg_shift) - 1;
    if (threadIdx.x == 0) nvalid = 0;
    __syncthreads();
    for (int c = wave; c < kp; c += nwaves) {
        const int64_t id = ids[qi * kp + c];
        double sum = 0.0;
        if (id >= 0) {
            const long long seg = id >> V.X.seg_shift, off = id & seg_mask;
            const unsigned char* xc = static_cast<const unsigned char*>(V.X.segs[seg]) + off * V.X.ld;
            const unsigned char* xs = static_cast<const unsigned char*>(V.ssegs[seg]) + off * V.sld;
            for (int e = lane * 16; e < V.X.ld; e += 1024) {
                const uint4 x = *reinterpret_cast<const uint4*>(xc + e), y = *reinterpret_cast<const uint4*>(qc + e);
                const unsigned xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
                double part = 0.0;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    float a[4], b[4];
                    f8_unpack4(xw[w], a);
                    f8_unpack4(yw[w], b);
#pragma unroll
                    for (int j = 0; j < 4; ++j) part += (double)(a[j] * b[j]);
                }
                const int blk = e / kF8Block;
                sum += part * ((double)f8_scale(xs[blk]) * (double)f8_scale(qsc[blk]));
            }
        }
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) sum += __shfl_xor(sum, d);
        if (lane == 0) {
            const bool ok = id >= 0 && sum == sum;
            score[c] = sum;
            cid[c] = ok ? id : -1;
            if (ok) atomicAdd(&nvalid, 1);
        }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < kp; c += blockDim.x) {
        const int64_t id = cid[c];
        if (id < 0) continue;
        const double s = score[c];
        int rank = 0;
        for (int o = 0; o < kp; ++o) rank += cid[o] >= 0 && (score[o] > s || (score[o] == s && cid[o] < id)) ? 1 : 0;
        if (rank < k) {
            const float f = (float)s;
            const bool keep = f32_to_ord(f) >= min_ord;   // the score floor cuts a suffix of the sorted list
            D[qi * k + rank] = keep ? f : SSMI_NEG_MAX;
            I[qi * k + rank] = keep ? id + id_offset : -1;
        }
    }
    for (int c = nvalid + threadIdx.x; c < k; c += blockDim.x) { D[qi * k + c] = SSMI_NEG_MAX; I[qi * k + c] = -1; }
}

hipError_t launch_f8_finish(const F8View& v, const F8Mat& q, const int64_t* ids, int kp, int k, float* D, int64_t* I,
                            int64_t id_offset, unsigned min_ord, hipStream_t s) {
    // a wave per candidate while the queries alone do not fill the card
    const int threads = q.n <= 512 ? 1024 : 256;
    hipLaunchKernelGGL(f8_finish_kernel, dim3((unsigned)q.n), dim3(threads), 0, s, v, q, ids, kp, k, D, I, id_offset, min_ord);
    return hipGetLastError();
}

// ---- plan and launch of the first pass ----
static int pow2_ceil(int x) { int p = 1; while (p < x) p <<= 1; return p; }

bool plan_f8_search(int ld, long long nrows, int nq, int k, int num_cu, F8SearchPlan* p) {
    if (k < 1 || k > kF8MaxK || nrows < 1 || nq < 1 || ld < kF8Block || ld % kF8Block) return false;
    *p = F8SearchPlan{};
    p->kp = k + kF8Spare;
    p->r = pow2_ceil((p->kp + 63) / 64);
    // the scan holds a register list per query and wave: eight queries of lists up to 64 keys, one of 512; its queries fit LDS
    const int nst = (ld / kF8Block + 3) / 4;
    int cap = std::max(1, 8 / p->r);
    while (cap > 1 && (size_t)cap * (ld + 16 + nst * 4) > 128 * 1024) cap >>= 1;
    p->scan = p->r <= 8 && nq <= cap;
    if (p->scan) {
        p->bt = pow2_ceil(nq);
        p->threads = 512;
        const size_t qb = (size_t)p->bt * (ld + 16 + nst * 4), mb = (size_t)8 * 64 * p->r * sizeof(skey_t);
        p->lds = std::max(qb, mb);
        const long long useful = (nrows + 127) / 128;   // eight groups of 16 rows per workgroup
        p->grid_x = (int)std::min<long long>(num_cu, useful);
        p->grid_y = 1;
        p->parts = p->grid_x;
        p->kernel = "f8_scan_kernel";
    } else {
        p->tq = nq <= 64 ? 64 : 128;
        p->nqt = (nq + p->tq - 1) / p->tq;
        const long long tiles = (nrows + 255) / 256;
        const long long ns = std::max<long long>(1, std::min<long long>(num_cu / p->nqt, tiles));
        p->rows_per_slice = (tiles + ns - 1) / ns * 256;
        p->nslices = (int)((nrows + p->rows_per_slice - 1) / p->rows_per_slice);
        p->parts = p->nslices;
        p->grid_x = p->nqt * p->nslices;
        p->grid_y = 1;
        p->threads = 512;
        p->lds = (size_t)2 * (256 + p->tq) * 128 + EPI_LDS_BYTES;
        p->cand_bytes = (size_t)p->grid_x * 256 * CAND_CAP * sizeof(skey_t);
        p->share_bytes = (size_t)p->nqt * p->tq * sizeof(unsigned);
        p->kernel = "f8_search_tile_kernel";
    }
    p->partial_bytes = (size_t)nq * p->parts * p->kp * sizeof(skey_t);
    return true;
}

template <int BT, int R>
static hipError_t launch_scan(const F8View& v, const F8Mat& q, const F8SearchPlan& p, skey_t* partial, const TailMerge& tail, hipStream_t s) {
    if (p.lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(f8_scan_kernel<BT, R>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)p.lds);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((f8_scan_kernel<BT, R>), dim3(p.grid_x, p.grid_y), dim3(p.threads), p.lds, s, v, q, p.kp, partial, tail);
    return hipGetLastError();
}
template <int MT, int NT, int WM, int WN, int R>
static hipError_t launch_tile(const F8View& v, const F8Mat& q, const F8SearchPlan& p, const MfmaParams& P, hipStream_t s) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(f8_search_tile_kernel<MT, NT, WM, WN, R>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)p.lds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((f8_search_tile_kernel<MT, NT, WM, WN, R>), dim3(p.grid_x), dim3(p.threads), p.lds, s, v, q, P);
    return hipGetLastError();
}
template <int R>
static hipError_t launch_r(const F8View& v, const F8Mat& q, const F8SearchPlan& p, void* share, void* cand, skey_t* partial, const TailMerge& tail, hipStream_t s) {
    if (p.scan) {
        if constexpr (R == 1) {
            if (p.bt == 8) return launch_scan<8, 1>(v, q, p, partial, tail, s);
            if (p.bt == 4) return launch_scan<4, 1>(v, q, p, partial, tail, s);
        }
        if constexpr (R == 2) { if (p.bt == 4) return launch_scan<4, 2>(v, q, p, partial, tail, s); }
        if constexpr (R <= 4) { if (p.bt == 2) return launch_scan<2, R>(v, q, p, partial, tail, s); }
        if constexpr (R <= 8) { if (p.bt == 1) return launch_scan<1, R>(v, q, p, partial, tail, s); }
        return hipErrorInvalidValue;
    }
    MfmaParams P = {};
    P.nq = (int)q.n;
    P.k = p.kp;
    P.nqt = p.nqt;
    P.nslices = p.nslices;
    P.rows_per_slice = p.rows_per_slice;
    P.partial = partial;
    P.cand = static_cast<skey_t*>(cand);
    P.thr_floor = SSMI_NEG_MAX;
    P.gthr = static_cast<unsigned*>(share);
    const int words = p.nqt * p.tq;
    hipLaunchKernelGGL(f8_zero_kernel, dim3((words + 255) / 256), dim3(256), 0, s, P.gthr, words);
    if (p.tq == 64) return launch_tile<2, 4, 8, 1, R>(v, q, p, P, s);
    return launch_tile<4, 4, 4, 2, R>(v, q, p, P, s);
}
hipError_t launch_f8_search(const F8View& v, const F8Mat& q, int k, const F8SearchPlan& p, void* share, void* cand, skey_t* partial,
                            const TailMerge& tail, hipStream_t s) {
    (void)k;
    switch (p.r) {
        case 1: return launch_r<1>(v, q, p, share, cand, partial, tail, s);
        case 2: return launch_r<2>(v, q, p, share, cand, partial, tail, s);
        case 4: return launch_r<4>(v, q, p, share, cand, partial, tail, s);
        case 8: return launch_r<8>(v, q, p, share, cand, partial, tail, s);
        case 16: return launch_r<16>(v, q, p, share, cand, partial, tail, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace ssmi

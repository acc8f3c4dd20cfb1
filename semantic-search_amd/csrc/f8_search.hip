// f8_search.hip - Flat search over 8-bit rows (f8.h): the product of f8_tile.h with the top-k epilogues of the other row types.
//
// The answer is the k best rows by the exact sums: score descending, ties by the lower id.
//
//   1. candidates   the best k + 16 rows by the matrix cores' sums: a streaming scan for a few queries, bound by reading the rows once (for one
//                   query its launch carries step 2), or the tile kernels with the candidate buffers of the 16-bit kernels (mfma_common.h)
//   2. proof        the candidates' products summed in 64 bits - every product of two codes is exact in fp32 and the scales are powers of two, so
//                   a sum is exact or off by a rounding of 2^-53 - and sorted by that.  A row that is not among them has a sum of step 1 of at
//                   most the last one's, and an exact one that is higher by that sum's error at most, which goes by the row's length.  If no row
//                   is long enough to make up for the gap between the k-th exact score and the last sum, the list is the answer.
//   3. in question  (not for one query) for the queries that are left - more than 16 rows within some 1e-5 |q||x| of the k-th score: a strong
//                   channel that makes the sums coarse against the gaps, copies of a row, rows far longer than the others - the rows whose sum
//                   may have lost enough for the k-th score
//   4. exact        those rows, or every row that is long enough, in 64 bits
//
// Sums are fp32's (f8_tile.h), but for tiles of 256 queries and small k: there the scaled instruction's come first, with their own, larger error in step 2,
// and steps 1 and 2 run again with fp32's for the tiles that hold an open query.  Steps that find nothing to do are a launch of 3 us each.  A
// query gets the same ids and scores in any batch.
//
// Same place on the path as the 16-bit kernels: faiss.IndexFlatIP.search as called from core/index_manager.py:371.
#include "f8_pp.h"
#include "tail_merge.h"
#include <algorithm>

namespace ssmi {

__device__ __forceinline__ i32x4_t load16_once(const unsigned char* p) { return __builtin_nontemporal_load(reinterpret_cast<const i32x4_t*>(p)); }

// ---- second pass of one query: 64-bit scores of its candidates, sorted.  All threads of the workgroup ----
// Four candidates per wave at a time (their loads travel together: the pass is a chain of memory round trips); the 16 codes of
// a lane belong to one block, so their products add up in 64 bits unscaled and meet the block's scale once.  score / cid: kp
// words of LDS each.
//
// The sum of 16 products without a 64-bit operation for each: a product is a multiple of 2^-18 below 2^18.  S, near 1.5 * 2^23,
// takes its whole part (an fp32 add there rounds to whole numbers, and 16 products keep S between 2^23 and 2^24), L what the
// rounding left: at most 1/2 each, so their sum is exact in fp32 too.
__device__ __forceinline__ double dot16(const i32x4_t& x, const i32x4_t& y) {
    const float S0 = 12582912.f;   // 1.5 * 2^23
    float S = S0, L = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        float a[4], b[4];
        f8_unpack4((unsigned)x[w], a);
        f8_unpack4((unsigned)y[w], b);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float s = __fmaf_rn(a[j], b[j], S);
            L = __fadd_rn(L, __fmaf_rn(a[j], b[j], __fsub_rn(S, s)));
            S = s;
        }
    }
    return (double)__fsub_rn(S, S0) + (double)L;
}
//
// How far a sum of the first pass may be off for a query and a row of lengths q and x: f8_relative(blocks) q x + 2^-118 (q + x) + 2^-125, as long
// as it cannot leave fp32.  An instruction adds 16 products per chain of roundings, eight of them to a block (f8_tile.h: 1.25 * 2^-23 of the
// magnitudes at hand each, which are q x at most), and the scan joins two chains at the end.  The rest: values below 2^-133 and products below
// the smallest fp32.  Solved for the length from which on a row may be off by `gap`:
__device__ __forceinline__ double f8_relative(int blocks) { return (8 * blocks + 8) * (1.25 / 8388608.0); }
__device__ __forceinline__ float f8_from(int blocks, double q, double gap) {
    if (!(q < 1e37)) return 0.f;   // sums may leave fp32 whatever the row
    const double x = (gap - 0x1p-118 * q - 0x1p-125) / (f8_relative(blocks) * q + 0x1p-118);
    return x > 0.0 ? (float)(fmin(fmin(x, 1e37), 1e37 / fmax(q, 1e-300)) * (1 - 0x1p-20)) : 0.f;
}
// How far a sum of the scaled instruction may be off, where no sum leaves fp32: of eight neighbouring products it keeps the largest, p = 2^E f, and
// takes the other seven down to multiples of 2^(E - 13); an exponent counts 2^-6 at the least (of subnormal codes, measured).  The largest products are
// at most g h, element by element of the largest of the eights of q and x, and their sum at most |g||h|.  Adding the eights up costs it no more
// than four times what the fp32 sums of all products may (random rows: a tenth of either).
__device__ __forceinline__ double f8_scaled_error(int blocks, double q, double x, double g, double h) {
    return 7.0 / 8192 * g * h + 4.0 * f8_relative(blocks) * q * x + 0x1p-100 * (1.0 + q + x);
}
// the squares of the largest of eight codes and of the eight behind them, added
__device__ __forceinline__ float eights(const i32x4_t& x) {
    float sum = 0.f;
#pragma unroll
    for (int h = 0; h < 4; h += 2) {
        float a[4], b[4], m = 0x1p-6f;
        f8_unpack4((unsigned)x[h], a);
        f8_unpack4((unsigned)x[h + 1], b);
#pragma unroll
        for (int j = 0; j < 4; ++j) m = fmaxf(m, fmaxf(fabsf(a[j]), fabsf(b[j])));
        sum = fmaf(m, m, sum);   // (multiples of 2^-12 below 2^19: off by 2^-24 of itself at most)
    }
    return sum;
}
// a score of the sorted list; the score floor cuts a suffix of it
__device__ __forceinline__ void put_result(const F8ScanArgs& A, float* D, int64_t* I, int rank, double s, int64_t id) {
    const float f = (float)s;
    const bool keep = f32_to_ord(f) >= A.min_ord;
    D[rank] = keep ? f : SSMI_NEG_MAX;
    I[rank] = keep ? id + A.id_offset : -1;
}
// the LDS words that a query's second pass needs besides its sort: kp scores, kp ids of its own and kp that it is given, then these
struct F8Proof { double qq, gg, kth; skey_t last; };   // |q|^2, that of the eights' largest, the k-th exact score, the last key of a full list (else 0)
__host__ __device__ inline size_t finish_bytes(int kp) { return (size_t)kp * 24 + sizeof(F8Proof); }
struct F8Scratch {
    double* score;
    int64_t *cid, *ids;
    F8Proof* proof;
    __device__ __forceinline__ F8Scratch(void* lds, int kp) : score(static_cast<double*>(lds)), cid(reinterpret_cast<int64_t*>(score + kp)), ids(cid + kp), proof(reinterpret_cast<F8Proof*>(ids + kp)) {}
};
__device__ __forceinline__ void finish_query(const F8ScanArgs& A, long long qi, const unsigned char* qc, const unsigned char* qsc, const F8Scratch& L) {
    constexpr int N = 4;
    const F8View& V = A.v;
    const int kp = A.kp, k = A.k;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), nwaves = blockDim.x >> 6;
    double* score = L.score;
    int64_t* cid = L.cid;
    const int64_t* ids = L.ids;
    float* D = A.D + qi * k;
    int64_t* I = A.I + qi * k;
    if (wave == nwaves - 1) {
        double qq = 0.0, gg = 0.0;
        for (int e = lane * 16; e < V.X.ld; e += 1024) {
            const i32x4_t y = *reinterpret_cast<const i32x4_t*>(qc + e);
            const double sq = (double)f8_scale(qsc[e / kF8Block]);
            qq += dot16(y, y) * (sq * sq);
            gg += (double)eights(y) * (sq * sq);
        }
#pragma unroll
        for (int d = 32; d >= 1; d >>= 1) { qq += __shfl_xor(qq, d); gg += __shfl_xor(gg, d); }
        if (lane == 0) { L.proof->qq = qq; L.proof->gg = gg; }
    }
    const long long seg_mask = (1ll << V.X.seg_shift) - 1;
    for (int c0 = wave * N; c0 < kp; c0 += nwaves * N) {
        const unsigned char* xc[N];
        const unsigned char* xs[N];
        int64_t id[N];
        double sum[N];
#pragma unroll
        for (int t = 0; t < N; ++t) {
            id[t] = c0 + t < kp ? ids[c0 + t] : -1;
            const long long row = id[t] < 0 ? 0 : id[t], seg = row >> V.X.seg_shift, off = row & seg_mask;   // none: row 0, not used
            xc[t] = static_cast<const unsigned char*>(V.X.segs[seg]) + off * V.X.ld;
            xs[t] = static_cast<const unsigned char*>(V.ssegs[seg]) + off * V.sld;
            sum[t] = 0.0;
        }
#pragma unroll 4
        for (int e = lane * 16; e < V.X.ld; e += 1024) {
            const int blk = e / kF8Block;
            i32x4_t x[N];
            unsigned char sx[N];
#pragma unroll
            for (int t = 0; t < N; ++t) {
                x[t] = *reinterpret_cast<const i32x4_t*>(xc[t] + e);
                sx[t] = xs[t][blk];
            }
            const i32x4_t y = *reinterpret_cast<const i32x4_t*>(qc + e);
            const double sq = (double)f8_scale(qsc[blk]);
#pragma unroll
            for (int t = 0; t < N; ++t) sum[t] += dot16(x[t], y) * (sq * (double)f8_scale(sx[t]));
        }
#pragma unroll
        for (int t = 0; t < N; ++t) {
#pragma unroll
            for (int d = 32; d >= 1; d >>= 1) sum[t] += __shfl_xor(sum[t], d);
            if (lane == 0 && c0 + t < kp) {
                score[c0 + t] = sum[t];
                cid[c0 + t] = id[t] >= 0 && sum[t] == sum[t] ? id[t] : -1;   // a NaN is no result
            }
        }
    }
    __syncthreads();
    // a wave ranks one candidate at a time against 64 others per step
    int valid = 0;
    for (int o = lane; o - lane < kp; o += 64) valid += __builtin_popcountll(__builtin_amdgcn_ballot_w64(o < kp && cid[o < kp ? o : 0] >= 0));
    for (int c = wave; c < kp; c += nwaves) {
        const int64_t id = cid[c];
        if (id < 0) continue;
        const double s = score[c];
        int rank = 0;
        for (int o = lane; o - lane < kp; o += 64) {
            const int oc = o < kp ? o : 0;
            const double so = score[oc];
            const int64_t io = cid[oc];
            rank += __builtin_popcountll(__builtin_amdgcn_ballot_w64(o < kp && io >= 0 && (so > s || (so == s && io < id))));
        }
        if (lane == 0 && rank < k) {
            put_result(A, D, I, rank, s, id);
            if (rank == k - 1) L.proof->kth = s;
        }
    }
    for (int c = valid + threadIdx.x; c < k; c += blockDim.x) { D[c] = SSMI_NEG_MAX; I[c] = -1; }
    __syncthreads();
    if (threadIdx.x == 0) {
        const F8Proof& p = *L.proof;
        // The list may lack a row whose sum came out at its last one's or below (a list that is not full: only one that left fp32).  Such a row is
        // among the k best only if it gained the gap.  (A query that is NaN has no results.)
        const double gap = p.last == 0 ? __builtin_inf() : valid >= k ? p.kth - (double)key_score(p.last) : -__builtin_inf();
        const double q = sqrt(p.qq) * (1 + 0x1p-40);
        const float from = f8_from(V.X.ld / kF8Block, q, gap);
        bool proven = p.qq != p.qq || A.longest[0] < from;
        if (A.sums == kF8Scaled && proven && p.qq == p.qq)
            proven = gap > f8_scaled_error(V.X.ld / kF8Block, q, (double)A.longest[0], sqrt(p.gg) * (1 + 0x1p-20), (double)A.longest[1]);
        const double x = (double)A.longest[0];
        const bool sums = valid >= k && p.last != 0 && q < 1e37 && x < 1e37 && q * x < 1e37;   // no sum leaves fp32
        // (rounded outwards, and the sum that is compared with it is off by 2^-24 of itself)
        const float least = (float)(p.kth - fabs(p.kth) * 0x1p-22 - 0x1p-118 * (q + x) - 0x1p-125), slope = (float)(f8_relative(V.X.ld / kF8Block) * q * (1 + 0x1p-20));
        A.state[qi] = F8State{valid >= k ? p.kth : -__builtin_inf(), from, least, sums && A.open ? slope : -1.f, proven ? 0u : 1u, 0u, sums && A.open ? 0u : kF8Collect + 1u};
        L.proof->last = proven || A.sums == kF8Scaled || !A.open ? 0 : 1;
    }
    __syncthreads();
    if (L.proof->last) {   // the collecting pass reads it from there
        for (int e = threadIdx.x * 16; e < V.X.ld; e += blockDim.x * 16)
            *reinterpret_cast<i32x4_t*>(A.open + qi * V.X.ld + e) = *reinterpret_cast<const i32x4_t*>(qc + e);
        for (int b = threadIdx.x; b < V.X.ld / kF8Block; b += blockDim.x) A.open[A.q.n * V.X.ld + qi * V.sld + b] = qsc[b];
    }
}

// ---- between the passes: the first pass's lists of one query -> its kp best rows.  All threads of the workgroup ----
// The lists' m-th keys, m = ceil(kp / P), bound the kp-th best from below: if c = ceil(kp / m) of them reach a score, m c >= kp
// rows do.  (For kp <= 48 the lane maxima of the heads serve, 64 values instead of P.)  The keys at or above the bound, two or
// three times kp of the P kp, are collected and sorted.  A full merge of 256 lists of 216 keys took 100 us on one workgroup.
// keys: LDS, nwaves * 64 R words and at least kSurvivors + 2.
static constexpr int kSurvivors = 2048;
template <int RV>
__device__ __forceinline__ unsigned nth_score(const skey_t* lists, int P, int kp, int m, int c) {
    const int lane = lane_id();
    WaveSort32<RV> t;
#pragma unroll
    for (int r = 0; r < RV; ++r) {
        const int p = r * 64 + lane;
        t.v[r] = p < P ? (unsigned)(load_key<true>(lists + (size_t)p * kp + m - 1) >> 32) : 0u;
    }
    t.sort_desc();
    return t.kth(c);
}
template <int R>
__device__ __forceinline__ void merge_to_ids(const skey_t* lists, int P, int kp, skey_t* keys, const F8Scratch& L) {
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), nwaves = blockDim.x >> 6;
    unsigned* word = reinterpret_cast<unsigned*>(keys);   // [0] bound, [1] survivors
    skey_t* surv = keys + 1;
    const int total = P * kp;
    WaveTopK<R> t;
    t.init();
    // the first keys of every thread travel while wave 0 finds the bound
    skey_t key[4];
    auto load4 = [&](int e0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int e = e0 + j * (int)blockDim.x;
            key[j] = e < total ? load_key<true>(lists + e) : 0;
        }
    };
    load4(threadIdx.x);
    if (wave == 0) {
        unsigned bound = 0;
        const int m = (kp + P - 1) / P, c = (kp + m - 1) / m;
        if (kp <= 48 && P > 64) {
            WaveSort32<1> h;
            h.v[0] = 0;
            for (int p = lane; p < P; p += 64) h.v[0] = max(h.v[0], (unsigned)(load_key<true>(lists + (size_t)p * kp) >> 32));
            h.sort_desc();
            bound = h.kth(kp);
        } else if (P <= 64) bound = nth_score<1>(lists, P, kp, m, c);
        else if (P <= 128) bound = nth_score<2>(lists, P, kp, m, c);
        else if (P <= 256) bound = nth_score<4>(lists, P, kp, m, c);
        else if (P <= 512) bound = nth_score<8>(lists, P, kp, m, c);
        if (lane == 0) { word[0] = bound; word[1] = 0; }
    }
    __syncthreads();
    const unsigned bound = max(word[0], 1u);   // (0 is the score of an empty key)
    for (int e0 = threadIdx.x;;) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if ((unsigned)(key[j] >> 32) >= bound) {
                const unsigned pos = atomicAdd(word + 1, 1u);
                if (pos < (unsigned)kSurvivors) surv[pos] = key[j];
            }
        e0 += blockDim.x * 4;
        if (e0 >= total) break;
        load4(e0);
    }
    __syncthreads();
    const int n = (int)word[1];
    if (n <= kSurvivors) {
        for (int base = wave * 64; base < n; base += nwaves * 64) {
            WaveTopK<1> c;
            c.v[0] = base + lane < n ? surv[base + lane] : 0;
            c.sort_desc();
            t.merge_regs(c);
        }
    } else {   // the bound did not thin them: every key
        for (int base = wave * 64; base < total; base += nwaves * 64) {
            WaveTopK<1> c;
            c.v[0] = base + lane < total ? load_key<true>(lists + base + lane) : 0;
            if (__builtin_amdgcn_ballot_w64(c.v[0] > t.kth(kp)) == 0) continue;
            c.sort_desc();
            t.merge_regs(c);
        }
    }
    __syncthreads();
    block_merge<R>(t, keys, wave, nwaves);
    if (wave == 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int e = r * 64 + lane;
            if (e < kp) L.ids[e] = t.v[r] ? (int64_t)key_id(t.v[r]) : -1;
            if (e == kp - 1) L.proof->last = t.v[r];
        }
    }
    __syncthreads();
}
__host__ __device__ inline size_t merge_keys_bytes(int waves, int r) {
    const size_t a = (size_t)waves * 64 * r * sizeof(skey_t), b = (size_t)(kSurvivors + 2) * sizeof(skey_t);
    return a > b ? a : b;
}

// query b -> LDS, quantised on the way if it comes as fp32 (16 lanes hold a block).  All threads of the workgroup
__device__ __forceinline__ void stage_query(const F8ScanArgs& A, long long b, unsigned char* qs, unsigned char* qsc) {
    for (int c = threadIdx.x; c < A.v.X.ld / 8; c += blockDim.x) {
        const int e0 = c * 8;
        uint2 o;
        unsigned sb = 0;
        if (A.f32) {
            const float* src = A.f32 + b * A.f32_stride;
            float v[8];
            if (A.f32_vec && e0 + 8 <= A.d) {
                const float4 lo = *reinterpret_cast<const float4*>(src + e0), hi = *reinterpret_cast<const float4*>(src + e0 + 4);
                v[0] = lo.x; v[1] = lo.y; v[2] = lo.z; v[3] = lo.w;
                v[4] = hi.x; v[5] = hi.y; v[6] = hi.z; v[7] = hi.w;
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = e0 + j < A.d ? src[e0 + j] : 0.f;
            }
            o = f8_pack8(v, e0, A.d, sb);
        } else {
            o = *reinterpret_cast<const uint2*>(A.q.codes + b * A.q.stride + e0);
            sb = A.q.scales[b * A.q.sstride + e0 / kF8Block];
        }
        *reinterpret_cast<uint2*>(qs + e0) = o;
        if ((e0 & (kF8Block - 1)) == 0) qsc[e0 / kF8Block] = (unsigned char)sb;
    }
}

// what follows the first pass where it does not carry it: one workgroup per query.  A chain of memory round trips and sorts: 17 us for
// 64 queries of 40 lists, 52 us for 1024 of 64
template <int R>
__global__ void __launch_bounds__(1024) f8_finish_kernel(F8ScanArgs A, int P) {
    extern __shared__ __align__(16) unsigned char smem[];
    const long long qi = blockIdx.x;
    const int ld = A.v.X.ld, kp = A.kp;
    if (A.sums == kF8Again && A.state[qi].ticket == 0) return;   // proven
    unsigned char* qs = smem;
    unsigned char* qsc = smem + ld;
    skey_t* keys = reinterpret_cast<skey_t*>(smem + (ld + ld / kF8Block + 15) / 16 * 16);
    const F8Scratch L(reinterpret_cast<unsigned char*>(keys) + merge_keys_bytes(blockDim.x >> 6, R), kp);
    if (A.shared && threadIdx.x == 0) A.shared[qi] = 0;   // as the next launch expects it
    stage_query(A, qi, qs, qsc);
    merge_to_ids<R>(A.partial + (size_t)qi * P * kp, P, kp, keys, L);
    finish_query(A, qi, qs, qsc, L);
}

// ---- third pass: the queries that are not proven.  A workgroup per CU ----
// their numbers: from the front of list those that are to see all rows by whole(state) (n[0] of them), from the back the others (n[1]).  Every
// workgroup of a launch makes the list for itself and takes its share of it, so whole() goes by what no workgroup of that launch writes, as
// does the ticket's being zero.  All threads
template <typename F>
__device__ __forceinline__ void open_queries(const F8ScanArgs& A, unsigned short* list, unsigned* n, F whole_of) {
    const int lane = lane_id(), nq = (int)A.q.n;
    bool any = false;
    for (int q = threadIdx.x; q < nq; q += blockDim.x) any |= __hip_atomic_load(&A.state[q].ticket, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != 0;
    if (!__syncthreads_or(any)) {   // (as a rule)
        if (threadIdx.x == 0) n[0] = n[1] = 0;
    } else if (threadIdx.x < 64) {
        int all = 0, few = 0;
        for (int q0 = 0; q0 < nq; q0 += 64) {
            const F8State* st = A.state + min(q0 + lane, nq - 1);
            const bool is = q0 + lane < nq && __hip_atomic_load(&st->ticket, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != 0;
            const bool whole = is && whole_of(*st);
            const unsigned long long ma = __builtin_amdgcn_ballot_w64(whole), mf = __builtin_amdgcn_ballot_w64(is && !whole), below = (1ull << lane) - 1;
            if (whole) list[all + __builtin_popcountll(ma & below)] = (unsigned short)(q0 + lane);
            else if (is) list[kF8Batch - 1 - few - __builtin_popcountll(mf & below)] = (unsigned short)(q0 + lane);
            all += __builtin_popcountll(ma);
            few += __builtin_popcountll(mf);
        }
        if (lane == 0) { n[0] = (unsigned)all; n[1] = (unsigned)few; }
    }
    __syncthreads();
}

// Scores as finish_query's.  A query whose rows in question are known has a workgroup score those.  Of the others, W workgroups share one (all of the
// grid if it is alone); each takes a range of the rows, picks those that are long enough and keeps what may be among the k best in LDS, sorted
// down to k whenever the buffer fills; the last to finish joins their lists.  1M x 4096 with every row long enough: 1.4 ms for one query, 0.8
// ms for each of many, by the vector units (four instructions a product).  With nothing to do the launch costs 3 us.
static constexpr int kExactThreads = 1024, kExactEntries = 2048, kExactRound = 256;   // entries of a buffer, and how many a round may add
struct F8Exact {
    double* score;
    unsigned *id, *count;   // count[0] entries, count[1] a flag
    double thr;             // entries have to beat (thr, thr_id)
    unsigned thr_id;
    __device__ __forceinline__ bool beats(double s, unsigned i) const { return s > thr || (s == thr && i < thr_id); }
    __device__ __forceinline__ void add(double s, unsigned i) const {
        const unsigned pos = atomicAdd(count, 1u);
        score[pos] = s;
        id[pos] = i;
    }
    // down to the k best, in order.  All threads; their entries are there
    __device__ __forceinline__ int shrink(int k) {
        const int n = (int)*count;
        int all = 64;
        while (all < n) all <<= 1;
        for (int e = n + threadIdx.x; e < all; e += blockDim.x) { score[e] = -__builtin_inf(); id[e] = 0xffffffffu; }
        for (int size = 2; size <= all; size <<= 1)
            for (int gap = size >> 1; gap; gap >>= 1) {
                __syncthreads();
                for (int t = threadIdx.x; t < all / 2; t += blockDim.x) {
                    const int a = (t / gap) * 2 * gap + t % gap, b = a + gap;
                    const double sa = score[a], sb = score[b];
                    const unsigned ia = id[a], ib = id[b];
                    const bool first = sa > sb || (sa == sb && ia < ib);
                    if (first != ((a & size) == 0)) {
                        score[a] = sb; score[b] = sa;
                        id[a] = ib; id[b] = ia;
                    }
                }
            }
        __syncthreads();
        const int left = min(n, k);
        if (n >= k) { thr = score[k - 1]; thr_id = id[k - 1]; }
        if (threadIdx.x == 0) *count = (unsigned)left;
        __syncthreads();
        return left;
    }
    // a round's entries are in: make room for the next
    __device__ __forceinline__ void next_round(int k) {
        __syncthreads();
        const bool fill = *count > (unsigned)(kExactEntries - kExactRound);
        __syncthreads();   // everybody has looked before anybody adds
        if (fill) shrink(k);
    }
};
__global__ void __launch_bounds__(kExactThreads) f8_exact_kernel(F8ScanArgs A) {
    extern __shared__ __align__(16) unsigned char smem[];
    const F8View& V = A.v;
    const int ld = V.X.ld, k = A.k, nq = (int)A.q.n;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), nwaves = blockDim.x >> 6;
    F8Exact X;
    X.score = reinterpret_cast<double*>(smem);
    X.id = reinterpret_cast<unsigned*>(X.score + kExactEntries);
    X.count = X.id + kExactEntries;
    unsigned short* open = reinterpret_cast<unsigned short*>(X.count + 4);   // [kF8Batch] the queries that are left
    unsigned* sel = reinterpret_cast<unsigned*>(open + kF8Batch);            // [blockDim.x] rows of a round
    unsigned char* qs = reinterpret_cast<unsigned char*>(sel + blockDim.x);
    unsigned char* qsc = qs + ld;
    open_queries(A, open, X.count + 1, [](const F8State& st) __attribute__((always_inline)) { return st.found > (unsigned)kF8Collect; });
    const int nall = __builtin_amdgcn_readfirstlane((int)X.count[1]), nfew = __builtin_amdgcn_readfirstlane((int)X.count[2]);
    if (nall + nfew == 0) return;
    const int W = nall ? max(1, (int)gridDim.x / nall) : 1;
    // lanes that share a row: 16 codes each, added up in finish_query's order, so that a row has one score
    const int lpr = ld > 512 ? 64 : ld > 256 ? 32 : ld > 128 ? 16 : 8, rpw = 64 / lpr, sub = lane / lpr, off = (lane % lpr) * 16;
    const long long seg_mask = (1ll << V.X.seg_shift) - 1;
    for (int item = blockIdx.x; item < nall * W + nfew; item += gridDim.x) {
        const bool all = item < nall * W;
        const int u = all ? item / W : kF8Batch - 1 - (item - nall * W), part = all ? item % W : 0;
        const long long qi = open[u];
        float* D = A.D + qi * k;
        int64_t* I = A.I + qi * k;
        __syncthreads();   // the query before is done with
        if (threadIdx.x == 0) X.count[0] = X.count[1] = 0;
        stage_query(A, qi, qs, qsc);
        X.thr = A.state[qi].edge;
        X.thr_id = 0xffffffffu;
        __syncthreads();
        const float from = A.state[qi].from;
        const unsigned* rows = A.rows + qi * kF8Collect;
        const long long begin = all ? V.X.nrows * part / W : 0, end = all ? V.X.nrows * (part + 1) / W : (long long)A.state[qi].found;
        for (long long r0 = all && part == 0 ? begin - (long long)blockDim.x : begin; r0 < end; r0 += blockDim.x) {
            // all: the rows that are long enough (a NaN's -1 is not), and before them the second pass's results that are not
            const bool listed = r0 < begin;
            const int e = threadIdx.x;
            if (listed ? e < k && !(I[e] == -1 && D[e] == SSMI_NEG_MAX) : r0 + e < end) {
                const long long row = listed ? I[e] - A.id_offset : all ? r0 + e : (long long)rows[r0 + e];
                const float len = all ? static_cast<const float*>(V.lsegs[row >> V.X.seg_shift])[row & seg_mask] : 0.f;
                if (!all || (len >= from) != listed) sel[atomicAdd(X.count + 1, 1u)] = (unsigned)row;
            }
            __syncthreads();
            const int nsel = (int)X.count[1];
            for (int s0 = 0; s0 < nsel; s0 += kExactRound) {
                for (int t = s0 + wave * rpw; t < min(nsel, s0 + kExactRound); t += nwaves * rpw) {
                    const unsigned row = sel[min(t + sub, nsel - 1)];
                    const long long seg = row >> V.X.seg_shift, in = row & seg_mask;
                    const unsigned char* xc = static_cast<const unsigned char*>(V.X.segs[seg]) + in * ld;
                    const unsigned char* xs = static_cast<const unsigned char*>(V.ssegs[seg]) + in * V.sld;
                    double sum = 0.0;
#pragma unroll 4
                    for (int e = off; e < ld; e += lpr * 16) {
                        const int blk = e / kF8Block;
                        sum += dot16(*reinterpret_cast<const i32x4_t*>(xc + e), *reinterpret_cast<const i32x4_t*>(qs + e)) * ((double)f8_scale(qsc[blk]) * (double)f8_scale(xs[blk]));
                    }
                    for (int d = lpr >> 1; d >= 1; d >>= 1) sum += __shfl_xor(sum, d);
                    if (off == 0 && t + sub < nsel && X.beats(sum, row)) X.add(sum, row);
                }
                X.next_round(k);
            }
            if (threadIdx.x == 0) X.count[1] = 0;
            __syncthreads();
        }
        int n = X.shrink(k);
        if (all && W > 1) {
            // (A.lists: W k entries for each of the queries, filled by whoever is done)
            F8Entry* list = A.lists + (size_t)u * W * k;
            F8State* st = A.state + qi;
            if (threadIdx.x == 0) X.count[1] = __hip_atomic_fetch_add(&st->pos, (unsigned)n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __syncthreads();
            const unsigned pos = X.count[1];
            for (int e = threadIdx.x; e < n; e += blockDim.x) list[pos + e] = F8Entry{X.score[e], (long long)X.id[e]};
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) X.count[1] = __hip_atomic_fetch_add(&st->ticket, 1u, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
            __syncthreads();
            if (X.count[1] != (unsigned)W) continue;
            __threadfence();
            const int total = (int)__hip_atomic_load(&st->pos, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (threadIdx.x == 0) X.count[0] = 0;
            X.thr = -__builtin_inf();
            X.thr_id = 0xffffffffu;
            __syncthreads();
            for (int e0 = 0; e0 < total; e0 += kExactRound) {
                const int e = e0 + threadIdx.x;
                if (threadIdx.x < kExactRound && e < total) {
                    const F8Entry v = list[e];
                    if (X.beats(v.score, (unsigned)v.id)) X.add(v.score, (unsigned)v.id);
                }
                X.next_round(k);
            }
            n = X.shrink(k);
        }
        for (int e = threadIdx.x; e < k; e += blockDim.x) {
            if (e < n) put_result(A, D, I, e, X.score[e], (int64_t)X.id[e]);
            else { D[e] = SSMI_NEG_MAX; I[e] = -1; }
        }
    }
}

// ---- rows in question ----
// The first pass again for the queries that it did not answer, with what is known now: a row whose fp32 sum cannot have lost enough for the k-th score
// is out.  What is left - a hundred rows or two, where a strong channel makes the sums coarse against the gaps of the scores - the next
// launch scores, and only a query with more than kF8Collect such rows (copies) has to see all.  256 rows x 64 of the open queries a step.
// 1M x 4096, 1024 queries, 0.98 of every row in one channel, k = 100: 16.5 ms with the passes in front and behind (all rows in 64 bits: 852 ms).
static constexpr int kCollectQueries = 64;
using F8CollectTile = F8Tile<2, 4, 8, 1, 3>;
__global__ void __launch_bounds__(512) f8_collect_kernel(F8ScanArgs A) {
    using T = F8CollectTile;
    static_assert(T::XR == 256 && T::QR == kCollectQueries, "rows of a segment, queries of a step");
    extern __shared__ __align__(16) unsigned char smem[];
    float* lens = reinterpret_cast<float*>(smem + T::LDS);                    // [256]
    unsigned* count = reinterpret_cast<unsigned*>(lens + 256);                // [4]
    unsigned short* open = reinterpret_cast<unsigned short*>(count + 4);      // [kF8Batch]
    const F8View& V = A.v;
    const int ld = V.X.ld;
    open_queries(A, open, count, [](const F8State& st) __attribute__((always_inline)) { return !(st.slope >= 0.f); });   // (not by found, which grows)
    const int nopen = __builtin_amdgcn_readfirstlane((int)count[1]);
    if (nopen == 0) return;
    T t;
    t.init(smem, ld / kF8Block);
    const int frow = t.lane & 15, fq = t.lane >> 4;
    const long long seg_mask = (1ll << V.X.seg_shift) - 1;
    const long long tiles = (V.X.nrows + 255) / 256;
    const int nqt = (nopen + kCollectQueries - 1) / kCollectQueries, slices = (int)min(tiles, (long long)max(1, (int)gridDim.x / nqt));
    for (int item = blockIdx.x; item < nqt * slices; item += gridDim.x) {
        const int qt = item % nqt, slice = item / nqt, q0 = qt * kCollectQueries;
        const auto query = [&](int r) __attribute__((always_inline)) { return (int)open[kF8Batch - 1 - (q0 + r)]; };
        const F8Src q{A.open, A.open + A.q.n * ld, (unsigned)ld, (unsigned)V.sld, min(kCollectQueries, nopen - q0) - 1};
        float least[4], slope[4];
        int qi[4];
#pragma unroll
        for (int n = 0; n < 4; ++n) {
            const int r = (t.wn * 4 + n) * 16 + frow;
            qi[n] = query(min(r, q.last));
            least[n] = r <= q.last ? A.state[qi[n]].least : __builtin_inff();
            slope[n] = A.state[qi[n]].slope;
        }
        for (long long tile = tiles * slice / slices; tile < tiles * (slice + 1) / slices; ++tile) {
            const long long row0 = tile * 256, seg = row0 >> V.X.seg_shift, off = row0 & seg_mask;
            const int last = (int)min(255ll, V.X.nrows - 1 - row0);
            __syncthreads();   // the tile before is done with
            if (threadIdx.x < 256) lens[threadIdx.x] = static_cast<const float*>(V.lsegs[seg])[off + min((int)threadIdx.x, last)];
            __syncthreads();
            t.aim(F8Src{static_cast<const unsigned char*>(V.X.segs[seg]) + off * ld, static_cast<const unsigned char*>(V.ssegs[seg]) + off * V.sld, (unsigned)ld, (unsigned)V.sld, last}, q, query);
            f32x4_t acc[2][4];
            zero_acc(acc);
            t.run(acc);
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const int r = (t.wm * 2 + m) * 16 + fq * 4;
                const float4 len = *reinterpret_cast<const float4*>(lens + r);
                const float l[4] = {len.x, len.y, len.z, len.w};
#pragma unroll
                for (int n = 0; n < 4; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (fmaf(slope[n], l[i], acc[m][n][i]) >= least[n] && r + i <= last) {   // (a NaN is not)
                            const unsigned pos = atomicAdd(&A.state[qi[n]].found, 1u);
                            if (pos < (unsigned)kF8Collect) A.rows[(long long)qi[n] * kF8Collect + pos] = (unsigned)(row0 + r + i);
                            else least[n] = __builtin_inff();   // all rows, then: no need to count on
                        }
            }
        }
    }
}

// lengths of rows: the waves take groups of rows as above
__global__ void __launch_bounds__(256) f8_lengths_kernel(F8Mat m, int ld, float* lengths, unsigned* longest) {
    const int lane = lane_id(), wave = threadIdx.x >> 6;
    const int lpr = ld > 512 ? 64 : ld > 256 ? 32 : ld > 128 ? 16 : 8, rpw = 64 / lpr, sub = lane / lpr, off = (lane % lpr) * 16;
    float most = 0.f, most8 = 0.f;
    for (long long r0 = ((long long)blockIdx.x * 4 + wave) * rpw; r0 < m.n; r0 += (long long)gridDim.x * 4 * rpw) {
        const long long row = min(r0 + sub, m.n - 1);
        double sum = 0.0, sum8 = 0.0;
#pragma unroll 2
        for (int e = off; e < ld; e += lpr * 16) {
            const i32x4_t x = *reinterpret_cast<const i32x4_t*>(m.codes + row * m.stride + e);
            const double s = (double)f8_scale(m.scales[row * m.sstride + e / kF8Block]);
            sum += dot16(x, x) * (s * s);
            sum8 += (double)eights(x) * (s * s);
        }
        for (int d = lpr >> 1; d >= 1; d >>= 1) { sum += __shfl_xor(sum, d); sum8 += __shfl_xor(sum8, d); }
        const float len = sum >= 0.0 ? (float)(sqrt(sum) * (1 + 0x1p-22)) : -1.f;   // (beyond fp32: infinite)
        if (off == 0 && r0 + sub < m.n) lengths[row] = len;
        most = fmaxf(most, len);
        if (len >= 0.f) most8 = fmaxf(most8, (float)(sqrt(sum8) * (1 + 0x1p-20)));
    }
#pragma unroll
    for (int d = 32; d >= 1; d >>= 1) { most = fmaxf(most, __shfl_xor(most, d)); most8 = fmaxf(most8, __shfl_xor(most8, d)); }
    // (one atomic a workgroup at most: one a wave took longer than the rows)
    __shared__ float part[4][2];
    if (lane == 0) { part[wave][0] = most; part[wave][1] = most8; }
    __syncthreads();
    if (threadIdx.x < 2) {
        const float v = fmaxf(fmaxf(part[0][threadIdx.x], part[1][threadIdx.x]), fmaxf(part[2][threadIdx.x], part[3][threadIdx.x]));
        if (v > __uint_as_float(__hip_atomic_load(longest + threadIdx.x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT))) atomicMax(longest + threadIdx.x, __float_as_uint(v));
    }
}
hipError_t launch_f8_lengths(const F8Mat& m, int ld, float* lengths, unsigned* longest, int num_cu, hipStream_t s) {
    if (m.n <= 0) return hipSuccess;
    const long long blocks = (m.n + 3) / 4, most = (long long)num_cu * 4;
    hipLaunchKernelGGL(f8_lengths_kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, s, m, ld, lengths, longest);
    return hipGetLastError();
}

// ---- streaming scan: up to BT <= 8 queries ----
// Bound by reading the rows once; what reads fastest decides the layout.  A plain read of 1M x 4096 codes ran at 5.9 TB/s with
// 16 rows x 64 bytes per load instruction (a matrix instruction's sixteen rows as they are) and at 6.7-7.0 TB/s with 8
// rows x 128 bytes, non-temporal loads and 4-8 waves per CU.  So one load is one whole block of eight rows, 16 codes a lane,
// and feeds two instructions of K = 32 (f8_tile.h): the sixteen operand rows
// are the 8 rows x {even, odd 16-byte chunks}, the sixteen columns 8 queries x {even, odd chunks}, and a score is the
// sum of the even-even and the odd-odd element of the result.  Columns beyond BT repeat a query and are never looked at.
// Up to eight loads (8 KiB) per stage and wave, three stages in flight: NB = 0: a stage is up to eight blocks of one group of
// eight rows; NB = 1, 2, 4: rows of that many blocks, a stage is 8 / NB groups;
// NB = 8: rows of a multiple of eight blocks, every stage is whole.
//
// Lists are the workgroup's: scores at or above a query's threshold go to its candidate buffer in LDS, and at looks ever
// further apart one wave per query sorts the buffer into the query's list (topk.h), which raises the threshold; the workgroups
// share the highest one.  (A list per wave, one sorted insertion per candidate, took longer than the rows for eight
// queries: a wave sees 500 of 1M rows, so its lists of k + 16 are never warm.)
template <int BT, int R, int NB>
__global__ void __launch_bounds__(512) f8_scan_kernel(F8ScanArgs A) {
    extern __shared__ __align__(16) unsigned char smem[];
    const F8View& V = A.v;
    const int lane = lane_id();
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const int nwaves = (int)(blockDim.x >> 6);
    const int ld = V.X.ld, nblk = ld / kF8Block, nq = (int)A.q.n, kp = A.kp;
    const int qpitch = ld + 32;                              // the 16 lanes of a pass (8 queries x 2 chunks) cover all banks once
    const int spitch = (nblk + 7) / 8 * 8;
    unsigned char* qs = smem;                                // [BT][qpitch] codes
    unsigned char* qsc = smem + BT * qpitch;                 // [BT][spitch] scales
    float* thr_l = reinterpret_cast<float*>(smem + (BT * (qpitch + spitch) + 15) / 16 * 16);   // [8] thresholds
    unsigned* cnt_l = reinterpret_cast<unsigned*>(thr_l + 8);                                   // [8] candidates
    skey_t* kept = reinterpret_cast<skey_t*>(cnt_l + 8);     // [BT][64 R] lists, best first
    skey_t* cand = kept + BT * 64 * R;                       // [BT][A.cap] candidates; the tail's scratch after that
    for (int e = threadIdx.x; e < BT * 64 * R; e += blockDim.x) kept[e] = 0;
    // a score passes only at or above its query's threshold, and NaN never does; queries that only fill up BT pass nothing
    if (threadIdx.x < 8) {
        thr_l[threadIdx.x] = (int)threadIdx.x < min(BT, nq) ? -__builtin_inff() : __builtin_nanf("");
        cnt_l[threadIdx.x] = 0;
    }

    const int r8 = lane & 7, odd = (lane >> 3) & 1, grp = lane >> 4;
    const bool holds = (lane & 40) == 0;   // scores end up in the lanes with bits 3 and 5 clear
    const unsigned vb = (gridDim.x % 8 == 0) ? (blockIdx.x % 8) * (gridDim.x / 8) + blockIdx.x / 8 : blockIdx.x;
    constexpr int G = NB == 0 ? 1 : 8 / (NB == 0 ? 1 : NB);   // groups of eight rows per run
    constexpr int run_rows = G * 8;
    const long long nruns = (V.X.nrows + run_rows - 1) / run_rows, step = (long long)gridDim.x * nwaves;
    const long long seg_mask = (1ll << V.X.seg_shift) - 1;
    const int chunk = (2 * grp + odd) * 16;
    const unsigned lane_off = (unsigned)r8 * (unsigned)ld + chunk, lane_soff = (unsigned)r8 * (unsigned)V.sld;
    const unsigned char* qlane = qs + (r8 % BT) * qpitch + chunk;
    const unsigned char* qslane = qsc + (r8 % BT) * spitch;
    const int stages = NB && NB < 8 ? 1 : (nblk + 7) / 8;     // of a run

    // two cursors over the wave's stages: the next to load, and the next to multiply.  A run's rows share a segment, and a
    // segment holds whole runs: rows beyond the last are read, never offered to a list
    long long lrun = (long long)vb * nwaves + wave, crun = lrun;
    int lkb = 0, ckb = 0;                                     // first block of the stage
    const unsigned char *lc = nullptr, *ls = nullptr;         // the run's codes and scales
    auto aim = [&]() __attribute__((always_inline)) {
        const long long row = lrun * run_rows, seg = row >> V.X.seg_shift, off = row & seg_mask;
        lc = static_cast<const unsigned char*>(V.X.segs[seg]) + off * ld;
        ls = static_cast<const unsigned char*>(V.ssegs[seg]) + off * V.sld;
    };
    if (lrun < nruns) aim();
    auto fetch = [&](i32x4_t (&x)[8], int (&sc)[8]) __attribute__((always_inline)) {
        if (lrun >= nruns) return;
        if constexpr (NB == 0 || NB == 8) {
            const i32x2_t w = *reinterpret_cast<const i32x2_t*>(ls + lkb + lane_soff);   // (scale rows are multiples of 16 bytes)
            sc[0] = w[0];
            sc[1] = w[1];
            const unsigned char* p = lc + (size_t)lkb * kF8Block + lane_off;
            // (a stage that is not whole loads its last block again: branches around loads cost more than those)
            const int last = NB == 8 ? 7 : nblk - 1 - lkb;
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = load16_once(p + (NB == 8 ? j : min(j, last)) * kF8Block);
        } else {
#pragma unroll
            for (int g = 0; g < G; ++g) {
                sc[g] = *reinterpret_cast<const int*>(ls + (size_t)(g * 8) * V.sld + lane_soff);
#pragma unroll
                for (int j = 0; j < NB; ++j) x[g * NB + j] = load16_once(lc + lane_off + (g * 8 * NB + j) * kF8Block);
            }
        }
        lkb += 8;
        if ((NB && NB < 8) || lkb >= nblk) {
            lkb = 0;
            lrun += step;
            if (lrun < nruns) aim();
        }
    };
    i32x4_t xa[8], xb[8], xc[8];
    int sa[8], sb[8], sc[8];
    fetch(xa, sa);   // the first rows travel while the queries are made
    fetch(xb, sb);
    for (int b = 0; b < BT; ++b) stage_query(A, min(b, nq - 1), qs + b * qpitch, qsc + b * spitch);

    f32x4_t acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
    // a load of rows against the same codes of the queries: sixteen codes a lane, two instructions
    const auto block = [&](auto jc, const i32x4_t& x, const i32x4_t& y, int sx, int sy) __attribute__((always_inline)) {
        constexpr int J = decltype(jc)::value;
        const float fx = f8_factor<J>(sx), fy = f8_factor<J>(sy);
        acc = mfma_f8(f8_widen(x[0], x[1], fx), f8_widen(y[0], y[1], fy), acc);
        acc = mfma_f8(f8_widen(x[2], x[3], fx), f8_widen(y[2], y[3], fy), acc);
    };
    // a row group is complete: rows 4 ((lane >> 4) & 1) + i of it, even-even here, odd-odd in lane ^ 40
    auto offer = [&](int g) __attribute__((always_inline)) {
        float sum[4];
        bool any = false;
        const float thr = thr_l[r8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sum[i] = acc[i] + __int_as_float(xor_lane<32>(xor_lane<8>(__float_as_int(acc[i]))));
            any |= sum[i] >= thr;
        }
        acc = f32x4_t{0.f, 0.f, 0.f, 0.f};
        if (__builtin_amdgcn_ballot_w64(any && holds) == 0) return;
        const long long row0 = crun * run_rows + g * 8 + 4 * grp;   // (grp < 2 in the lanes that hold)
        if (holds) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (sum[i] >= thr && row0 + i < V.X.nrows) cand[r8 * A.cap + atomicAdd(&cnt_l[r8], 1u)] = make_key(sum[i], (uint32_t)(row0 + i));
        }
    };
    auto eat = [&](const i32x4_t (&x)[8], const int (&sc)[8]) __attribute__((always_inline)) {
        if (crun >= nruns) return;
        if constexpr (NB == 0 || NB == 8) {
            const i32x2_t sq = *reinterpret_cast<const i32x2_t*>(qslane + ckb);
            const unsigned char* qp = qlane + (size_t)ckb * kF8Block;
            const auto one = [&](auto jc) __attribute__((always_inline)) {
                constexpr int J = decltype(jc)::value;
                const i32x4_t y = *reinterpret_cast<const i32x4_t*>(qp + J * kF8Block);
                block(std::integral_constant<int, J % 4>(), x[J], y, sc[J / 4], sq[J / 4]);
            };
            const int left = nblk - ckb;   // (the rest of a row that is not whole stages)
            one(std::integral_constant<int, 0>());
            if (NB == 8 || left > 1) one(std::integral_constant<int, 1>());
            if (NB == 8 || left > 2) one(std::integral_constant<int, 2>());
            if (NB == 8 || left > 3) one(std::integral_constant<int, 3>());
            if (NB == 8 || left > 4) one(std::integral_constant<int, 4>());
            if (NB == 8 || left > 5) one(std::integral_constant<int, 5>());
            if (NB == 8 || left > 6) one(std::integral_constant<int, 6>());
            if (NB == 8 || left > 7) one(std::integral_constant<int, 7>());
            ckb += 8;
            if (ckb < nblk) return;
            ckb = 0;
            offer(0);
        } else {
            const int sq = *reinterpret_cast<const int*>(qslane);
            i32x4_t y[NB];
#pragma unroll
            for (int j = 0; j < NB; ++j) y[j] = *reinterpret_cast<const i32x4_t*>(qlane + j * kF8Block);
#pragma unroll
            for (int g = 0; g < G; ++g) {
                block(std::integral_constant<int, 0>(), x[g * NB], y[0], sc[g], sq);
                if constexpr (NB > 1) block(std::integral_constant<int, 1>(), x[g * NB + 1], y[1], sc[g], sq);
                if constexpr (NB > 2) block(std::integral_constant<int, 2>(), x[g * NB + 2], y[2], sc[g], sq);
                if constexpr (NB > 3) block(std::integral_constant<int, 3>(), x[g * NB + 3], y[3], sc[g], sq);
                offer(g);
            }
        }
        crun += step;
    };
    // LDS of every wave settled, loads in flight left alone
    auto meet = [&]() __attribute__((always_inline)) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // candidates of query b -> its list, by the wave that owns b
    auto fold = [&](bool share) __attribute__((always_inline)) {
#pragma unroll 1
        for (int b = wave; b < min(BT, nq); b += nwaves) {
            const int n = (int)cnt_l[b];
            if (n == 0) continue;
            WaveTopK<R> t;
#pragma unroll
            for (int r = 0; r < R; ++r) t.v[r] = kept[b * 64 * R + r * 64 + lane];
#pragma unroll 1
            for (int base = 0; base < n; base += 64) {
                WaveTopK<1> c;
                c.v[0] = base + lane < n ? cand[b * A.cap + base + lane] : 0;
                if (__builtin_amdgcn_ballot_w64(c.v[0] > t.kth(kp)) == 0) continue;
                c.sort_desc();
                t.merge_regs(c);
            }
            const skey_t kth = t.kth(kp);
            t.store(kept + b * 64 * R, 64 * R);
            if (lane == 0) {
                cnt_l[b] = 0;
                // the kp-th score of any workgroup bounds the final one: all filter with the highest
                unsigned mine = kth ? (unsigned)(kth >> 32) : 0u;
                if (share && A.shared) mine = max(mine, atomicMax(A.shared + b, mine));
                if (mine) thr_l[b] = ord_to_f32(mine);
            }
        }
    };
    const long long rounds = ((long long)vb * nwaves < nruns) ? (nruns - (long long)vb * nwaves + step - 1) / step : 0;
    const long long total = rounds * stages;   // the same for all waves of the workgroup (wave 0 has the most runs), so that they meet
    int turns = 0, every = 1;
    meet();
    // (the scheduler would otherwise sink every load to its first use)
#define TURN(X, SX, Y, SY)                  \
    fetch(Y, SY);                           \
    __builtin_amdgcn_sched_barrier(0);      \
    eat(X, SX);                             \
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll 1
    for (long long i = 0; i < total; i += 3) {
        TURN(xa, sa, xc, sc)
        TURN(xb, sb, xa, sa)
        TURN(xc, sc, xb, sb)
        if (++turns == every && i + 3 < total) {   // (the end folds anyway)
            // look at the buffers, often while the thresholds are young
            turns = 0;
            every = min(2 * every, A.every);
            meet();
            bool fill = false;
#pragma unroll
            for (int b = 0; b < BT; ++b) fill |= cnt_l[b] >= 64u;
            meet();   // everybody has looked before a wave clears a counter or appends
            if (fill) {
                fold(true);
                meet();
            }
        }
    }
#undef TURN
    __syncthreads();
    fold(false);
    // publication, and in the last workgroup to arrive the merge (tail_merge.h) and the second pass
    for (int b = wave; b < nq; b += nwaves) {
        WaveTopK<R> t;
#pragma unroll
        for (int r = 0; r < R; ++r) t.v[r] = kept[b * 64 * R + r * 64 + lane];
        publish_list<R>(t, A.partial + ((size_t)b * gridDim.x + blockIdx.x) * kp, kp);
    }
    if (A.counter == nullptr) return;
    skey_t* keys = cand;
    if (!tail_last_block(A.counter, gridDim.x, reinterpret_cast<unsigned*>(keys))) return;
    // one query: the last workgroup goes on (several queries have a workgroup each: f8_finish_kernel)
    if (threadIdx.x == 0) A.shared[0] = 0;   // as the next launch expects it
    const F8Scratch L(reinterpret_cast<unsigned char*>(keys) + merge_keys_bytes(nwaves, R), kp);
    merge_to_ids<R>(A.partial, (int)gridDim.x, kp, keys, L);
    finish_query(A, 0, qs, qsc, L);
}

// the k-th score of any slice bounds the final one: the slices share the highest (mfma.hip).  A wave's own queries, as in the folds
__device__ __forceinline__ void share_thresholds(int wave, int lane, int q0, const MfmaParams& P, float* thr_l) {
    const int ql = wave + 8 * lane;
    if (lane < 32 && q0 + ql < P.nq) {
        const float t = thr_l[ql];
        const unsigned mine = t > SSMI_NEG_MAX ? f32_to_ord(t) : 0u;
        const unsigned seen = atomicMax(&P.gthr[q0 + ql], mine);
        if (seen > mine) thr_l[ql] = ord_to_f32(seen);
    }
}

// ---- first thresholds of a slice ----
// No list exists yet and every row of its first tile would pass the filter, go to memory and be sorted.  The tile's rows are taken in 64
// groups of four; a group's largest score is a row, so the kp-th largest of a query's 64 group maxima (kp <= 64) has kp rows at or above
// it and bounds the kp-th score from below.  About 30 rows of 256 pass it at kp = 26.  The slices share the highest, as behind a fold.
static constexpr int kSeedPitch = 65;   // words of a query's maxima: lanes that hold neighbouring queries write to banks of their own
template <int TQ>
__device__ __forceinline__ void seed_thresholds(const float* maxima, int wave, int lane, int q0, const MfmaParams& P, float* thr_l) {
#pragma unroll 1
    for (int ql = wave; ql < TQ; ql += 8) {
        if (q0 + ql >= P.nq) break;
        WaveSort32<1> t;
        t.v[0] = f32_to_ord(maxima[ql * kSeedPitch + lane]);
        t.sort_desc();
        const float kth = ord_to_f32(t.kth(P.k));
        if (lane == 0) lds_store(reinterpret_cast<unsigned*>(&thr_l[ql]), __float_as_uint(fmaxf(kth, P.thr_floor)));
    }
    share_thresholds(wave, lane, q0, P, thr_l);
}

// ---- tile kernel: 256 rows x TQ queries per workgroup, a slice of the rows each ----
// Bound by the rows' way from memory while the batch is small (1M x 4096: 16 queries 791 us, 5.2 TB/s; 64 queries 933 us, 4.4), by the
// folds and the first tile of a slice over few rows (10000 x 4096, 64 queries: 87 us).
template <int MT, int NT, int WM, int WN, int R>
__global__ void __launch_bounds__(512) f8_search_tile_kernel(F8View V, F8Mat q, MfmaParams P) {
    using T = F8Tile<MT, NT, WM, WN, 3>;
    static_assert(T::XR == 256 && T::WAVES == 8, "row tile and folds of the 16-bit kernels");
    extern __shared__ __align__(16) unsigned char smem[];
    float* thr_l = reinterpret_cast<float*>(smem + T::LDS);
    unsigned* cnt_l = reinterpret_cast<unsigned*>(thr_l + 256);
    unsigned* kept_l = cnt_l + 256;
    unsigned* flag_l = kept_l + 256;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int frow = lane & 15, fq = lane >> 4;
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
    T t;
    t.init(smem, V.X.ld / kF8Block);
    auto aim = [&](long long row0) __attribute__((always_inline)) {
        const long long seg = row0 >> V.X.seg_shift, off = row0 & seg_mask;
        t.aim(F8Src{static_cast<const unsigned char*>(V.X.segs[seg]) + off * V.X.ld, static_cast<const unsigned char*>(V.ssegs[seg]) + off * V.sld,
                    (unsigned)V.X.ld, (unsigned)V.sld, (int)min(255ll, r_end - 1 - row0)}, qsrc);
    };
    unsigned tiles_done = 0;
    if (r_begin < r_end) aim(r_begin);
    for (long long row0 = r_begin; row0 < r_end; row0 += 256) {
        const long long left = r_end - row0;
        f32x4_t acc[MT][NT];
        zero_acc(acc);
        t.run(acc);
        if (tiles_done == 0 && P.k <= 64) {
            float* maxima = reinterpret_cast<float*>(smem);   // (the ring is free)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    // (no NaN may enter the sort, and no row behind the last)
                    float v = SSMI_NEG_MAX;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if ((t.wm * MT + m) * 16 + fq * 4 + i < left) v = vmax2(v, acc[m][n][i]);
                    maxima[((t.wn * NT + n) * 16 + frow) * kSeedPitch + (t.wm * MT + m) * 4 + fq] = v;
                }
            __syncthreads();
            seed_thresholds<T::QR>(maxima, wave, lane, q0, P, thr_l);
            __syncthreads();
        }
        if (row0 + 256 < r_end) aim(row0 + 256);   // its first slabs travel under the filter
        if (left >= 256) filter_tile<MT, NT, true>(acc, t.wm * MT * 16, t.wn * NT * 16, frow, fq, row0, 256, cand, thr_l, cnt_l, flag_l);
        else filter_tile<MT, NT, false>(acc, t.wm * MT * 16, t.wn * NT * 16, frow, fq, row0, (int)left, cand, thr_l, cnt_l, flag_l);
        __syncthreads();
        ++tiles_done;
        // fold after row tiles 1, 4, 16, ... of the slice and whenever a candidate buffer is half full
        if (row0 + 256 < r_end && (((tiles_done & (tiles_done - 1)) == 0 && (tiles_done & P.fold_mask)) || *flag_l)) {   // (the end folds anyway)
            fold_queries<R>(wave, q0, P, slice, cand, thr_l, cnt_l, kept_l);
            share_thresholds(wave, lane, q0, P, thr_l);
            __syncthreads();
            if (tid == 0) *flag_l = 0;
        }
    }
    __syncthreads();
    fold_queries<R>(wave, q0, P, slice, cand, thr_l, cnt_l, kept_l);
}

// ---- large batches: 256 rows x 256 queries on the contraction of f8_pp.h ----
// Threshold filter over a wave's 128 x 64 accumulators (acc[m][n][4 g + e]: row row_base + 32 m + 8 g + 4 h + e, query q_base + 32 n + r
// of lane (r, h)): as filter_tile of the 16-bit kernels, one column maximum first, survivors one by one.
template <bool FULL>
__device__ __forceinline__ void filter_big(const F8Pp<false>::Acc& acc, int row_base, int q_base, int lane, long long row0, int rows_valid, skey_t* cand,
                                           const float* thr_l, unsigned* cnt_l, unsigned* flag_l) {
    const int r = lane & 31, h = lane >> 5;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
        const int ql = q_base + 32 * n + r;
        const float thr = thr_l[ql];
        float mm[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const f32x16_t v = acc[m][n];
            float a = vmax3(v[0], v[1], v[2]);
#pragma unroll
            for (int i = 3; i < 15; i += 2) a = vmax3(a, v[i], v[i + 1]);
            mm[m] = vmax2(a, v[15]);
        }
        const float mx = vmax2(vmax3(mm[0], mm[1], mm[2]), mm[3]);
        if (__builtin_amdgcn_ballot_w64(mx >= thr) == 0) continue;
        if (mx >= thr) {
            skey_t* cq = cand + (size_t)ql * CAND_CAP;
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                if (__builtin_expect(__builtin_amdgcn_ballot_w64(mm[m] >= thr) != 0, 0)) {
                    const f32x16_t v = acc[m][n];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float s = v[i];
                        const int rr = row_base + 32 * m + 8 * (i >> 2) + 4 * h + (i & 3);
                        if (s >= thr && (FULL || rr < rows_valid)) {
                            const unsigned pos = lds_add_rtn(&cnt_l[ql], 1u);
                            if (pos + 1 >= (unsigned)CAND_TRIG) lds_store(flag_l, 1u);
                            if (pos < (unsigned)CAND_CAP) cq[pos] = make_key(s, (uint32_t)(row0 + rr));
                        }
                    }
                }
            }
        }
    }
}

// A workgroup keeps its query tile and walks a slice of the rows; the first slab of the next row tile travels under this one's filter.
// Folds, thresholds and the bound from the slices' published tops are those of the 16-bit kernel (mfma_pp.hip).
// 1M x 4096, 1024 queries, k = 10: 3.86 ms with the scaled instruction, 2.23 PFLOP/s; 6.65 with fp32 sums, 1.29 (1.55 for the product alone,
// f8_matmul.hip).  256 queries: 1.34 and 1.93 ms - one slab ahead of the products does not cover the way from memory where no second query
// tile shares the rows.  open: the second run, for the tiles with a query that is.
template <int R, bool SCALED>
__global__ void __launch_bounds__(512, 2) f8_search_big_kernel(F8View V, F8Mat q, MfmaParams P, const F8State* open) {
    using T = F8Pp<SCALED>;
    extern __shared__ __align__(16) unsigned char smem[];
    float* thr_l = reinterpret_cast<float*>(smem + T::LDS);
    unsigned* cnt_l = reinterpret_cast<unsigned*>(thr_l + 256);
    unsigned* kept_l = cnt_l + 256;
    unsigned* flag_l = kept_l + 256;
    T t;
    t.init(smem, V.X.ld / kF8Block);
    int logical = blockIdx.x;
    if ((gridDim.x & 7) == 0) logical = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    const int slice = logical / P.nqt, qt = logical % P.nqt;
    const int q0 = qt * 256;
    if (open && !__syncthreads_or(threadIdx.x < 256 && q0 + (int)threadIdx.x < P.nq && open[q0 + threadIdx.x].ticket != 0)) return;
    const long long r_begin = (long long)slice * P.rows_per_slice;
    const long long r_end = min(r_begin + P.rows_per_slice, V.X.nrows);
    skey_t* cand = P.cand + (size_t)blockIdx.x * 256 * CAND_CAP;
    if (threadIdx.x < 256) {
        thr_l[threadIdx.x] = q0 + (int)threadIdx.x < P.nq ? P.thr_floor : __builtin_inff();
        cnt_l[threadIdx.x] = 0;
        kept_l[threadIdx.x] = 0;
    }
    if (threadIdx.x == 0) flag_l[0] = 0;
    __syncthreads();
    const long long seg_mask = (1ll << V.X.seg_shift) - 1;
    const F8Src qsrc{q.codes + (size_t)q0 * q.stride, q.scales + (size_t)q0 * q.sstride, (unsigned)q.stride, (unsigned)q.sstride, (int)min(255ll, q.n - 1 - q0)};
    auto aim = [&](long long row0) __attribute__((always_inline)) {
        const long long seg = row0 >> V.X.seg_shift, off = row0 & seg_mask;
        t.aim(F8Src{static_cast<const unsigned char*>(V.X.segs[seg]) + off * V.X.ld, static_cast<const unsigned char*>(V.ssegs[seg]) + off * V.sld,
                    (unsigned)V.X.ld, (unsigned)V.sld, (int)min(255ll, r_end - 1 - row0)}, qsrc);
    };
    auto push_bounds = [&](int lane) {
        for (int ql = slice + t.wave * P.nslices; ql < 256 && q0 + ql < P.nq; ql += 8 * P.nslices) {
            const unsigned b = tops_bound(P, q0 + ql);
            if (b && lane == 0) atomicMax(&P.gthr[q0 + ql], b);
        }
    };
    auto pull_thr = [&](int lane) {
        const int ql = t.wave + 8 * lane;
        if (lane < 32 && q0 + ql < P.nq) {
            const unsigned seen = __hip_atomic_load(&P.gthr[q0 + ql], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (seen && ord_to_f32(seen) > thr_l[ql]) lds_store(reinterpret_cast<unsigned*>(&thr_l[ql]), __float_as_uint(ord_to_f32(seen)));
        }
    };
    unsigned tiles_done = 0;
    int xstate = 0;
    if (r_begin < r_end) aim(r_begin);
#pragma unroll 1
    for (long long row0 = r_begin; row0 < r_end; row0 += 256) {
        typename T::Acc acc;
        zero_acc(acc);
        t.run(acc);
        const long long left = r_end - row0;
        int lane = t.lane;
        asm volatile("" : "+v"(lane));   // (addresses are made here and not ahead of the loop, whose registers are all taken)
        if (tiles_done == 0 && P.k <= 64 && left >= 256) {
            float* maxima = reinterpret_cast<float*>(smem) + (t.wn * 64 + (lane & 31)) * kSeedPitch + t.wm * 32 + (lane >> 5);   // (the ring is free)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int m = 0; m < 4; ++m)
#pragma unroll
                    for (int g = 0; g < 4; ++g)   // (no NaN may enter the sort)
                        maxima[n * 32 * kSeedPitch + (m * 4 + g) * 2] = vmax3(vmax3(acc[m][n][g * 4], acc[m][n][g * 4 + 1], SSMI_NEG_MAX), acc[m][n][g * 4 + 2], acc[m][n][g * 4 + 3]);
            __syncthreads();
            seed_thresholds<256>(reinterpret_cast<const float*>(smem), t.wave, lane, q0, P, thr_l);
            __syncthreads();
        }
        if (row0 + 256 < r_end) aim(row0 + 256);
        if (left >= 256) filter_big<true>(acc, t.wm * 128, t.wn * 64, lane, row0, 256, cand, thr_l, cnt_l, flag_l);
        else filter_big<false>(acc, t.wm * 128, t.wn * 64, lane, row0, (int)left, cand, thr_l, cnt_l, flag_l);
        __syncthreads();
        ++tiles_done;
        const bool fold_due = row0 + 256 < r_end && (((tiles_done & (tiles_done - 1)) == 0 && (tiles_done & P.fold_mask)) || *flag_l);   // (the end folds anyway)
        if (xstate && !fold_due) {
            if (xstate == 1) push_bounds(lane); else pull_thr(lane);
            xstate = xstate == 1 ? 2 : 0;
        }
        if (fold_due) {
            fold_queries<R>(t.wave, q0, P, slice, cand, thr_l, cnt_l, kept_l);
            xstate = P.gtop ? 1 : 0;
            __syncthreads();
            share_thresholds(t.wave, lane, q0, P, thr_l);
            __syncthreads();
            if (threadIdx.x == 0) *flag_l = 0;
        }
    }
    __syncthreads();
    fold_queries<R>(t.wave, q0, P, slice, cand, thr_l, cnt_l, kept_l);
}

__global__ void f8_zero_kernel(unsigned* p, size_t n) {
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x) p[i] = 0;
}

// ---- plans and launches ----
static int pow2_ceil(int x) { int p = 1; while (p < x) p <<= 1; return p; }

bool plan_f8_search(int ld, long long nrows, int nq, int k, int num_cu, F8SearchPlan* p) {
    if (k < 1 || k > kF8MaxK || nrows < 1 || nq < 1 || ld < kF8Block || ld % kF8Block) return false;
    *p = F8SearchPlan{};
    p->kp = k + kF8Spare;
    p->r = pow2_ceil((p->kp + 63) / 64);
    const int nblk = ld / kF8Block;
    // the scan holds a register list per query and wave (eight queries of lists up to 64 keys, one of 512) and its queries in LDS
    const size_t per_query = (size_t)ld + 32 + (nblk + 7) / 8 * 8;
    int cap = std::max(1, 8 / p->r);
    while (cap > 1 && cap * per_query > 80 * 1024) cap >>= 1;
    p->scan = p->r <= 8 && nq <= cap;
    if (p->scan) {
        p->bt = pow2_ceil(nq);
        p->nb = nblk == 1 || nblk == 2 || nblk == 4 ? nblk : nblk % 8 == 0 ? 8 : 0;
        const int run_rows = p->nb ? 64 / p->nb : 8, stages = (nblk + 7) / 8;
        const long long runs = (nrows + run_rows - 1) / run_rows;
        // One workgroup per CU, of eight waves: six hold as many rows in flight but convert fewer of them meanwhile (one query, us with 4, 6 and 8 waves:
        // 10000 x 4096 43.0, 37.6, 34.4; 1M x 1024 254, 194, 177; 2M x 768 462, 340, 285; 1M x 4096 758, 623, 616; only 200000 x 8192 330, 283, 294).
        const int waves = 8;
        p->threads = waves * 64;
        // The waves look at the candidate buffers at most p->every turns of three stages apart: no query may gain more rows
        // meanwhile than its buffer holds beside the 63 candidates that a look may leave
        const auto rows = [&](int turns) { return (3 * turns + stages - 1) / stages * run_rows * waves; };
        p->cap = std::max(4096 / p->bt, rows(1) + 64);
        for (p->every = 1; rows(2 * p->every) + 64 <= p->cap;) p->every *= 2;
        const size_t work = std::max((size_t)p->bt * p->cap * sizeof(skey_t), p->bt > 1 ? 0 : merge_keys_bytes(waves, p->r) + finish_bytes(p->kp));
        p->lds = (p->bt * per_query + 15) / 16 * 16 + 64 + (size_t)p->bt * 64 * p->r * sizeof(skey_t) + work;
        p->grid_x = (int)std::min<long long>(num_cu, (runs + waves - 1) / waves);
        p->parts = p->grid_x;
        p->kernel = "f8_scan_kernel";
    } else {
        // Over few rows narrow tiles of queries win: more workgroups, fewer lists each.  Up to seven rounds of the chip (us in tiles of 64, 128 and
        // 256 queries: 10000 x 4096, 256 queries 89, 127, 205; 20000 x 4096, 512 queries 199, 221, 217; 50000 x 4096, 256 queries 232, 220, 346, 1024
        // queries 611, 581, 589; 100000 x 4096, 256 queries 362, 368, 377, 512 queries 602, 556, 583, 1024 queries 1082, 951, 887; 100000 x 768,
        // 256 queries 178, 203, 291; 1M x 4096, 256 queries 2547, 2245, 1965)
        const long long tiles = (nrows + 255) / 256;
        const auto few = [&](int tq) { return tiles * ((nq + tq - 1) / tq) <= 7ll * num_cu; };
        p->tq = nq <= 64 || few(64) ? 64 : nq <= 128 || few(128) ? 128 : 256;
        // The scaled instruction's sums prove a list where the gap between the k-th score and the last candidate's is wide: over 1M Gaussian rows x 4096
        // that of 16 spare ranks is seven times the error bound at k = 10 and three times at 32, where a tile of 256 queries nearly always has one that
        // needs better sums; 32 spare ranks are five times.  (32 for all cost 1.5 times as much over 2M x 128.)  1M x 4096, 1024 queries: k = 10
        // 4.0 ms, k = 32 4.55 (10.1 with 16), fp32 sums alone 6.65 and 6.95; where the scaled ones prove nothing (a strong channel) 10.4 and 11.5.
        p->scaled = p->tq == 256 && k <= 32;
        if (p->scaled && k > 16) p->kp = k + 32;
        p->nqt = (nq + p->tq - 1) / p->tq;
        const long long ns = std::max<long long>(1, std::min<long long>(num_cu / p->nqt, tiles));
        p->rows_per_slice = (tiles + ns - 1) / ns * 256;
        p->nslices = (int)((nrows + p->rows_per_slice - 1) / p->rows_per_slice);
        p->parts = p->nslices;
        p->grid_x = p->nqt * p->nslices;
        p->threads = 512;
        p->lds = (size_t)(p->tq == 256 ? F8Pp<false>::LDS : p->tq == 128 ? F8Tile<4, 4, 4, 2, 3>::LDS : F8Tile<2, 4, 8, 1, 3>::LDS) + EPI_LDS_BYTES;
        p->cand_bytes = (size_t)p->grid_x * 256 * CAND_CAP * sizeof(skey_t);
        // scores every slice publishes per query: enough that the kp-th largest of all of them exists and is tight (mfma.hip)
        int m = (int)((std::max<long long>(64, (long long)p->kp * 5 / 4) + p->nslices - 1) / p->nslices);
        m = std::max(1, std::min(std::min(m, 8), p->kp));
        p->gtop_m = (p->tq == 256 && p->nslices > 1 && (long long)p->nslices * m >= p->kp) ? m : 0;
        p->share_bytes = (size_t)p->nqt * p->tq * (1 + (size_t)p->nslices * p->gtop_m) * sizeof(unsigned) * (p->scaled ? 2 : 1);
        p->kernel = p->tq == 256 ? "f8_search_big_kernel" : "f8_search_tile_kernel";
    }
    p->partial_bytes = (size_t)nq * p->parts * p->kp * sizeof(skey_t);
    return true;
}

template <int BT, int R, int NB>
static hipError_t launch_scan_nb(const F8ScanArgs& a, const F8SearchPlan& p, hipStream_t s) {
    if (p.lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(f8_scan_kernel<BT, R, NB>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)p.lds);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL((f8_scan_kernel<BT, R, NB>), dim3(p.grid_x), dim3(p.threads), p.lds, s, a);
    return hipGetLastError();
}
template <int BT, int R>
static hipError_t launch_scan(const F8ScanArgs& a, const F8SearchPlan& p, hipStream_t s) {
    if (p.nb == 1) return launch_scan_nb<BT, R, 1>(a, p, s);
    if (p.nb == 2) return launch_scan_nb<BT, R, 2>(a, p, s);
    if (p.nb == 4) return launch_scan_nb<BT, R, 4>(a, p, s);
    if (p.nb == 8) return launch_scan_nb<BT, R, 8>(a, p, s);
    return launch_scan_nb<BT, R, 0>(a, p, s);
}
template <int R>
static hipError_t launch_finish_r(const F8ScanArgs& a, const F8SearchPlan& p, hipStream_t s) {
    const int threads = R == 16 ? 256 : 512;   // (the lists of the waves meet in LDS)
    const int ld = a.v.X.ld;
    const size_t lds = (size_t)(ld + ld / kF8Block + 15) / 16 * 16 + merge_keys_bytes(threads / 64, R) + finish_bytes(p.kp);
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(f8_finish_kernel<R>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(f8_finish_kernel<R>, dim3((unsigned)a.q.n), dim3(threads), lds, s, a, p.parts);
    return hipGetLastError();
}
hipError_t launch_f8_finish(const F8ScanArgs& a, const F8SearchPlan& p, hipStream_t s) {
    switch (p.r) {
        case 1: return launch_finish_r<1>(a, p, s);
        case 2: return launch_finish_r<2>(a, p, s);
        case 4: return launch_finish_r<4>(a, p, s);
        case 8: return launch_finish_r<8>(a, p, s);
        case 16: return launch_finish_r<16>(a, p, s);
    }
    return hipErrorInvalidValue;
}
hipError_t launch_f8_collect(const F8ScanArgs& a, int num_cu, hipStream_t s) {
    const int lds = F8CollectTile::LDS + 256 * 4 + 16 + kF8Batch * 2;
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(f8_collect_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(f8_collect_kernel, dim3((unsigned)num_cu), dim3(512), lds, s, a);
    return hipGetLastError();
}
hipError_t launch_f8_exact(const F8ScanArgs& a, int num_cu, hipStream_t s) {
    const int ld = a.v.X.ld;
    const size_t lds = kExactEntries * 12 + 16 + kF8Batch * 2 + kExactThreads * 4 + (size_t)(ld + ld / kF8Block + 15) / 16 * 16;
    if (lds > 64 * 1024) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(f8_exact_kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if (e != hipSuccess) return e;
    }
    hipLaunchKernelGGL(f8_exact_kernel, dim3((unsigned)num_cu), dim3(kExactThreads), lds, s, a);
    return hipGetLastError();
}
hipError_t launch_f8_scan(const F8ScanArgs& a, const F8SearchPlan& p, hipStream_t s) {
    switch (p.r * 16 + p.bt) {
        case 16 + 1: return launch_scan<1, 1>(a, p, s);
        case 16 + 2: return launch_scan<2, 1>(a, p, s);
        case 16 + 4: return launch_scan<4, 1>(a, p, s);
        case 16 + 8: return launch_scan<8, 1>(a, p, s);
        case 32 + 1: return launch_scan<1, 2>(a, p, s);
        case 32 + 2: return launch_scan<2, 2>(a, p, s);
        case 32 + 4: return launch_scan<4, 2>(a, p, s);
        case 64 + 1: return launch_scan<1, 4>(a, p, s);
        case 64 + 2: return launch_scan<2, 4>(a, p, s);
        case 128 + 1: return launch_scan<1, 8>(a, p, s);
    }
    return hipErrorInvalidValue;
}

template <int MT, int NT, int WM, int WN, int R>
static hipError_t launch_tile(const F8View& v, const F8Mat& q, const F8SearchPlan& p, const MfmaParams& P, hipStream_t s) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(f8_search_tile_kernel<MT, NT, WM, WN, R>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)p.lds);
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((f8_search_tile_kernel<MT, NT, WM, WN, R>), dim3(p.grid_x), dim3(p.threads), p.lds, s, v, q, P);
    return hipGetLastError();
}
template <int R>
static hipError_t launch_r(const F8View& v, const F8Mat& q, const F8SearchPlan& p, const MfmaParams& P, const F8State* open, hipStream_t s) {
    if (p.tq == 64) return launch_tile<2, 4, 8, 1, R>(v, q, p, P, s);
    if (p.tq == 128) return launch_tile<4, 4, 4, 2, R>(v, q, p, P, s);
    const auto big = [&](auto kernel) {
        const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)p.lds);
        if (e != hipSuccess) return e;
        hipLaunchKernelGGL(kernel, dim3(p.grid_x), dim3(p.threads), p.lds, s, v, q, P, open);
        return hipGetLastError();
    };
    if constexpr (R == 1)
        if (p.scaled && !open) return big(f8_search_big_kernel<R, true>);
    return big(f8_search_big_kernel<R, false>);
}
hipError_t launch_f8_tiles(const F8View& v, const F8Mat& q, const F8SearchPlan& p, const F8State* open, void* share, void* cand, skey_t* partial, hipStream_t s) {
    MfmaParams P = {};
    P.nq = (int)q.n;
    P.k = p.kp;
    P.nqt = p.nqt;
    P.nslices = p.nslices;
    P.rows_per_slice = p.rows_per_slice;
    P.partial = partial;
    P.cand = static_cast<skey_t*>(cand);
    P.thr_floor = SSMI_NEG_MAX;
    const size_t words = p.share_bytes / sizeof(unsigned);
    P.gthr = static_cast<unsigned*>(share) + (open ? words / 2 : 0);   // (of its own for each run)
    P.gtop = p.gtop_m ? P.gthr + (size_t)p.nqt * p.tq : nullptr;
    P.gtop_m = p.gtop_m;
    P.fold_mask = P.gtop ? 0x11111111u : 0x55555555u;   // scheduled folds after row tiles 1, 16, 256, ... (1, 4, 16, ... without the bound)
    // (where first thresholds are there and two tiles follow at most, the first fold costs more than it saves: 100000 x 4096, 64 queries 210 us, 188 without, 100000 x 1024 138 and 111; where four
    // follow it pays: 100000 x 4096, 128 queries 256 us, 263 without)
    if (p.kp <= 64 && p.rows_per_slice <= 3 * 256) P.fold_mask &= ~1u;
    if (!open) hipLaunchKernelGGL(f8_zero_kernel, dim3((unsigned)std::min<size_t>((words + 255) / 256, 4096)), dim3(256), 0, s, P.gthr, words);
    switch (p.r) {
        case 1: return launch_r<1>(v, q, p, P, open, s);
        case 2: return launch_r<2>(v, q, p, P, open, s);
        case 4: return launch_r<4>(v, q, p, P, open, s);
        case 8: return launch_r<8>(v, q, p, P, open, s);
        case 16: return launch_r<16>(v, q, p, P, open, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace ssmi

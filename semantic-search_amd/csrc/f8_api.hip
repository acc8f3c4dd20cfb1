// f8_api.hip - host side of the 8-bit rows (f8.h): the C entry points of the row operators and the product, and the Flat
// index's add / search over 8-bit rows.  Host logic only.
#include "../../include/ssmi.h"
#include "f8.h"
#include "index.h"
#include <algorithm>
#include <atomic>

using namespace ssmi;

namespace {

// the arguments every entry point checks; `what` names the operand in the message
int check_rows(const char* what, const void* codes, int64_t stride, const void* scales, int64_t sstride, int64_t n, int d) {
    if (n < 0) return fail("%s: negative row count", what);
    if (n > (1ll << 26)) return fail("%s: %lld rows exceed the supported maximum %lld", what, (long long)n, 1ll << 26);
    if (stride < f8_ld(d) || stride % 16 || stride > (1 << 23))
        return fail("%s: code rows must be a multiple of 16 bytes apart, at least %d (whole blocks of 128) and at most %d", what, f8_ld(d), 1 << 23);
    if (sstride < f8_blocks(d) || sstride % 4 || sstride > (1 << 20))
        return fail("%s: scale rows must be a multiple of 4 bytes apart, at least %d and at most %d", what, f8_blocks(d), 1 << 20);
    if (n == 0) return 0;
    if (!codes || !scales) return fail("%s: NULL codes or scales", what);
    if ((uintptr_t)codes & 15) return fail("%s: codes must be 16-byte aligned", what);
    if ((uintptr_t)scales & 3) return fail("%s: scales must be 4-byte aligned", what);
    return 0;
}
int check_dim(int d) {
    if (d < 1 || d > 65536) return fail("dimension %d out of range [1, 65536]", d);
    return 0;
}
int check_plain(const char* what, const void* p, int dtype, int64_t stride, int64_t n, int d) {
    if (!dtype_known(dtype)) return fail("%s: unknown dtype %d", what, dtype);
    if (stride < d) return fail("%s: row stride %lld is shorter than a row of %d", what, (long long)stride, d);
    if (n > 0 && !p) return fail("%s: NULL rows", what);
    if ((uintptr_t)p & (dtype_elsize(dtype) - 1)) return fail("%s: rows must be aligned to their element", what);
    return 0;
}
int num_cu_of(int device, int* out) {
    static std::atomic<int> known[64];   // asked once per device
    *out = device < 64 ? known[device].load(std::memory_order_relaxed) : 0;
    if (*out) return 0;
    HIPCHECK(hipDeviceGetAttribute(out, hipDeviceAttributeMultiprocessorCount, device));
    if (device < 64) known[device].store(*out, std::memory_order_relaxed);
    return 0;
}

// rows of the handle's two stores that share a segment: f(first row of the run within the call, count, codes, scales, lengths)
template <typename F>
int for_segments(ssmi_index* h, long long row0, long long n, F f) {
    const long long seg_rows = 1ll << h->rows.seg_shift;
    for (long long done = 0; done < n;) {
        const long long row = row0 + done, seg = row >> h->rows.seg_shift, off = row & (seg_rows - 1);
        const long long cnt = std::min(n - done, seg_rows - off);
        CHECK(f(done, cnt, (unsigned char*)h->rows.segs[seg] + off * h->rows.row_bytes, (unsigned char*)h->scales.segs[seg] + off * h->scales.row_bytes,
                (float*)h->lengths.segs[seg] + off));
        done += cnt;
    }
    return 0;
}
int reserve_rows(ssmi_index* h, int64_t n) {
    if ((unsigned long long)(h->rows.nrows + n) >= 0xFFFFFFFFull) return fail("index would exceed 2^32-2 vectors");
    CHECK(h->rows.reserve(h->rows.nrows + n, h->stream));
    CHECK(h->scales.reserve(h->rows.nrows + n, h->stream));
    return h->lengths.reserve(h->rows.nrows + n, h->stream);
}
F8NormArgs plain_rows(const void* x, int64_t x_stride, int dtype, int64_t n, int d, unsigned char* codes, int64_t stride,
                      unsigned char* scales, int64_t sstride) {
    F8NormArgs a = {};
    a.x = x;
    a.x_stride = x_stride;
    a.dtype = dtype;
    a.n = n;
    a.d = d;
    a.codes = codes;
    a.stride = stride;
    a.scales = scales;
    a.sstride = sstride;
    return a;
}
// rows on the device -> the stores' rows [row0, row0 + n), which are reserved
int quantize_into(ssmi_index* h, const void* x, int src_dtype, long long row0, long long n) {
    const int d = h->rows.d;
    return for_segments(h, row0, n, [&](long long first, long long cnt, unsigned char* codes, unsigned char* scales, float* lengths) -> int {
        HIPCHECK(launch_f8_rows(plain_rows((const char*)x + (size_t)first * d * dtype_elsize(src_dtype), d, src_dtype, cnt, d, codes, h->rows.ld, scales, h->scales.ld),
                                h->num_cu, h->stream));
        HIPCHECK(launch_f8_lengths(F8Mat{codes, h->rows.ld, scales, h->scales.ld, cnt}, h->rows.ld, lengths, (unsigned*)h->f8_longest, h->num_cu, h->stream));
        return 0;
    });
}

}  // namespace

namespace ssmi {

int f8_store_add(ssmi_index* h, int64_t n, const void* x, int src_dtype, int mem_kind) {
    const long long row0 = h->rows.nrows;
    CHECK(reserve_rows(h, n));
    const size_t row = (size_t)h->rows.d * dtype_elsize(src_dtype);
    const long long chunk = mem_kind == SSMI_HOST ? std::max<long long>(1, ((size_t)64 << 20) / row) : n;
    for (long long done = 0; done < n; done += chunk) {
        const long long cnt = std::min<long long>(chunk, n - done);
        const void* src = (const char*)x + (size_t)done * row;
        if (mem_kind == SSMI_HOST) {
            CHECK(ensure_ws(h, 0, (size_t)cnt * row));
            HIPCHECK(hipMemcpyAsync(h->ws[0], src, (size_t)cnt * row, hipMemcpyHostToDevice, h->stream));
            src = h->ws[0];
        }
        CHECK(quantize_into(h, src, src_dtype, row0 + done, cnt));
        if (mem_kind == SSMI_HOST) HIPCHECK(hipStreamSynchronize(h->stream));  // staging buffer reused
    }
    HIPCHECK(hipStreamSynchronize(h->stream));
    h->rows.nrows = h->scales.nrows = h->lengths.nrows = row0 + n;
    return 0;
}

int f8_add_random_unit(ssmi_index* h, int64_t n, uint64_t seed) {
    const long long row0 = h->rows.nrows;
    CHECK(reserve_rows(h, n));
    const size_t row = (size_t)h->rows.d * 4;
    const long long chunk = std::max<long long>(1, ((size_t)256 << 20) / row);
    for (long long done = 0; done < n; done += chunk) {
        const long long cnt = std::min<long long>(chunk, n - done);
        CHECK(ensure_ws(h, 0, (size_t)cnt * row));
        HIPCHECK(launch_random_unit((float*)h->ws[0], row0 + done, cnt, h->rows.d, seed, h->stream));
        CHECK(quantize_into(h, h->ws[0], SSMI_F32, row0 + done, cnt));
    }
    HIPCHECK(hipStreamSynchronize(h->stream));
    h->rows.nrows = h->scales.nrows = h->lengths.nrows = row0 + n;
    return 0;
}

hipError_t gather_store_rows(ssmi_index* h, const RowStore& R, long long view_rows, const int64_t* ids, long long n, float* out, int* bad,
                             hipStream_t s) {
    RowView v = R.view();
    v.nrows = view_rows;
    if (R.dtype == SSMI_F8) return launch_f8_gather(F8View{v, (const void* const*)h->scales.d_segs, h->scales.ld, nullptr}, ids, n, R.d, out, bad, s);
    return launch_gather_rows(v, R.dtype, ids, n, R.d, out, bad, s);
}

// Workspaces: 4 query codes and scales, 5 candidate buffers, 2 partial lists, 6 states, rows in question, open queries and lists of the exact pass, 7 shared thresholds.
int f8_store_search(ssmi_index* h, int64_t nq, const F8Queries& q, int k, float* Ddev, int64_t* Idev, int64_t id_offset, hipStream_t s,
                    unsigned min_ord) {
    const RowStore& R = h->rows;
    const int ld = R.ld, sld = h->scales.ld;
    const F8View view{R.view(), (const void* const*)h->scales.d_segs, sld, (const void* const*)h->lengths.d_segs};
    const int64_t kBatch = kF8Batch;
    hipEvent_t* ev = h->ev[h->n_searches % ssmi_index::kEvRing];
    F8SearchPlan p = {};
    for (int64_t done = 0; done < nq; done += kBatch) {
        const int nb = (int)std::min<int64_t>(kBatch, nq - done);
        if (!plan_f8_search(ld, R.nrows, nb, k, h->num_cu, &p)) return fail("internal: 8-bit search plan failed");
        const bool rec = h->timing_on && done == 0;
        CHECK(ensure_ws(h, 2, p.partial_bytes));
        const bool collect = nb > 1;   // (one query: all rows in 64 bits take little longer, and the launch 3 us of every search)
        const size_t states = (size_t)nb * sizeof(F8State), lists = (size_t)h->num_cu * k * sizeof(F8Entry), rows = (size_t)nb * kF8Collect * sizeof(unsigned);
        CHECK(ensure_ws(h, 6, states + lists + (collect ? rows + (size_t)nb * (ld + sld) : 0)));
        F8ScanArgs a = {};
        a.v = view;
        a.q = F8Mat{q.codes + done * q.stride, q.stride, q.scales + done * q.sstride, q.sstride, nb};
        a.f32 = q.f32 ? q.f32 + done * q.q_stride : nullptr;
        a.f32_stride = q.q_stride;
        a.f32_vec = ((uintptr_t)a.f32 & 15) == 0 && q.q_stride % 4 == 0;
        a.d = R.d;
        a.k = k;
        a.kp = p.kp;
        a.partial = (skey_t*)h->ws[2];
        a.D = Ddev + done * k;
        a.I = Idev + done * k;
        a.id_offset = id_offset;
        a.min_ord = min_ord;
        a.cap = p.cap;
        a.every = p.every;
        a.longest = h->f8_longest;
        a.state = (F8State*)h->ws[6];
        a.lists = (F8Entry*)(a.state + nb);
        a.rows = (unsigned*)(a.lists + (size_t)h->num_cu * k);
        a.open = collect ? (unsigned char*)h->ws[6] + states + lists + rows : nullptr;
        if (p.scan) {
            if (h->tail_counters) {
                a.counter = nb == 1 ? h->tail_counters : nullptr;
                a.shared = h->tail_counters + 1;
            }
            if (rec) HIPCHECK(hipEventRecord(ev[0], s));
            HIPCHECK(launch_f8_scan(a, p, s));
            if (rec) HIPCHECK(hipEventRecord(ev[1], s));
        } else {
            if (q.f32) {
                const size_t codes = (size_t)nb * ld;
                CHECK(ensure_ws(h, 4, codes + (size_t)nb * sld));
                unsigned char* w = (unsigned char*)h->ws[4];
                HIPCHECK(launch_f8_rows(plain_rows(a.f32, q.q_stride, SSMI_F32, nb, R.d, w, ld, w + codes, sld), h->num_cu, s));
                a.q = F8Mat{w, ld, w + codes, sld, nb};
                a.f32 = nullptr;
            }
            CHECK(ensure_ws(h, 5, p.cand_bytes));
            CHECK(ensure_ws(h, 7, p.share_bytes));
            if (rec) HIPCHECK(hipEventRecord(ev[0], s));
            HIPCHECK(launch_f8_tiles(view, a.q, p, nullptr, h->ws[7], h->ws[5], (skey_t*)h->ws[2], s));
            if (p.scaled) {
                a.sums = kF8Scaled;
                HIPCHECK(launch_f8_finish(a, p, s));
                a.sums = kF8Again;
                HIPCHECK(launch_f8_tiles(view, a.q, p, a.state, h->ws[7], h->ws[5], (skey_t*)h->ws[2], s));
            }
            if (rec) HIPCHECK(hipEventRecord(ev[1], s));
        }
        if (!a.counter) HIPCHECK(launch_f8_finish(a, p, s));
        if (collect) HIPCHECK(launch_f8_collect(a, h->num_cu, s));
        HIPCHECK(launch_f8_exact(a, h->num_cu, s));
        if (rec) { HIPCHECK(hipEventRecord(ev[2], s)); h->merge_event = true; }
    }
    if (h->timing_on) h->n_searches++;
    h->events_valid = h->timing_on;
    h->timing_valid = true;
    h->timing.last_path = p.scan ? 0 : 1;
    h->last_kernel = p.kernel;
    h->last_clk = nullptr;
    h->timing.last_grid = p.grid_x;
    h->timing.last_scan_bytes = (int64_t)R.nrows * (ld + f8_blocks(R.d));
    h->timing.last_scan_flops = 2ll * std::min<int64_t>(nq, kBatch) * R.nrows * R.d;
    return 0;
}

}  // namespace ssmi

extern "C" {

int ssmi_f8_quantize(int device, int64_t n, int d, const void* x, int src_dtype, int64_t x_stride, uint8_t* codes, int64_t codes_stride,
                     uint8_t* scales, int64_t scales_stride, void* stream) {
    return guarded([&]() -> int {
    CHECK(check_dim(d));
    CHECK(check_rows("f8_quantize", codes, codes_stride, scales, scales_stride, n, d));
    CHECK(check_plain("f8_quantize", x, src_dtype, x_stride, n, d));
    if (n == 0) return 0;
    DeviceGuard g(device);
    if (!g.ok) return fail("hipSetDevice(%d) failed", device);
    int cus = 0;
    CHECK(num_cu_of(device, &cus));
    HIPCHECK(launch_f8_rows(plain_rows(x, x_stride, src_dtype, n, d, codes, codes_stride, scales, scales_stride), cus, (hipStream_t)stream));
    return 0;
    });
}

int ssmi_f8_rms_norm(int device, int64_t n, int d, const void* x, int dtype, int64_t x_stride, const void* residual, int64_t residual_stride,
                     void* residual_out, int64_t residual_out_stride, const void* weight, int weight_dtype, float eps, int unit,
                     uint8_t* codes, int64_t codes_stride, uint8_t* scales, int64_t scales_stride, void* stream) {
    return guarded([&]() -> int {
    CHECK(check_dim(d));
    CHECK(check_rows("f8_rms_norm", codes, codes_stride, scales, scales_stride, n, d));
    CHECK(check_plain("f8_rms_norm", x, dtype, x_stride, n, d));
    if (residual) {
        CHECK(check_plain("f8_rms_norm residual", residual, dtype, residual_stride, n, d));
        CHECK(check_plain("f8_rms_norm residual_out", residual_out, dtype, residual_out_stride, n, d));
    } else if (residual_out) {
        return fail("f8_rms_norm: residual_out without a residual");
    }
    if (weight) CHECK(check_plain("f8_rms_norm weight", weight, weight_dtype, d, 1, d));
    if (d > kF8MaxNorm) return fail("f8_rms_norm: dimension %d exceeds the supported maximum %d", d, kF8MaxNorm);
    if (!(eps >= 0.f)) return fail("f8_rms_norm: eps must be >= 0");
    if (n == 0) return 0;
    DeviceGuard g(device);
    if (!g.ok) return fail("hipSetDevice(%d) failed", device);
    int cus = 0;
    CHECK(num_cu_of(device, &cus));
    F8NormArgs a = plain_rows(x, x_stride, dtype, n, d, codes, codes_stride, scales, scales_stride);
    a.residual = residual;
    a.r_stride = residual_stride;
    a.residual_out = residual_out;
    a.ro_stride = residual_out_stride;
    a.weight = weight;
    a.weight_dtype = weight_dtype;
    a.eps = eps;
    a.inv_d = 1.0 / d;
    a.norm = true;
    a.unit = unit != 0;
    HIPCHECK(launch_f8_rows(a, cus, (hipStream_t)stream));
    return 0;
    });
}

int ssmi_f8_dequantize(int device, int64_t n, int d, const uint8_t* codes, int64_t codes_stride, const uint8_t* scales, int64_t scales_stride,
                       void* out, int out_dtype, int64_t out_stride, void* stream) {
    return guarded([&]() -> int {
    CHECK(check_dim(d));
    CHECK(check_rows("f8_dequantize", codes, codes_stride, scales, scales_stride, n, d));
    CHECK(check_plain("f8_dequantize", out, out_dtype, out_stride, n, d));
    if (n == 0) return 0;
    DeviceGuard g(device);
    if (!g.ok) return fail("hipSetDevice(%d) failed", device);
    int cus = 0;
    CHECK(num_cu_of(device, &cus));
    HIPCHECK(launch_f8_dequantize(F8Mat{codes, codes_stride, scales, scales_stride, n}, d, out, out_dtype, out_stride, cus, (hipStream_t)stream));
    return 0;
    });
}

int ssmi_f8_matmul(int device, int64_t m, int64_t n, int k, const uint8_t* a_codes, int64_t a_stride, const uint8_t* a_scales,
                   int64_t a_scales_stride, const uint8_t* b_codes, int64_t b_stride, const uint8_t* b_scales, int64_t b_scales_stride,
                   void* out, int out_dtype, int64_t out_stride, void* stream) {
    return guarded([&]() -> int {
    CHECK(check_dim(k));
    CHECK(check_rows("f8_matmul a", a_codes, a_stride, a_scales, a_scales_stride, m, k));
    CHECK(check_rows("f8_matmul b", b_codes, b_stride, b_scales, b_scales_stride, n, k));
    if (!dtype_is16(out_dtype)) return fail("f8_matmul: the output is fp16 or bf16 (the matrix instruction's sums do not carry fp32)");
    if (out_stride < n) return fail("f8_matmul: output row stride %lld is shorter than a row of %lld", (long long)out_stride, (long long)n);
    if (m == 0 || n == 0) return 0;
    if (!out) return fail("f8_matmul: NULL output");
    if ((uintptr_t)out & 1) return fail("f8_matmul: the output must be aligned to its element");
    DeviceGuard g(device);
    if (!g.ok) return fail("hipSetDevice(%d) failed", device);
    int cus = 0;
    CHECK(num_cu_of(device, &cus));
    HIPCHECK(launch_f8_matmul(F8Mat{a_codes, a_stride, a_scales, a_scales_stride, m}, F8Mat{b_codes, b_stride, b_scales, b_scales_stride, n}, k,
                              out, out_dtype, out_stride, cus, (hipStream_t)stream));
    return 0;
    });
}

int ssmi_index_add_f8(ssmi_index* h, int64_t n, const uint8_t* codes, int64_t codes_stride, const uint8_t* scales, int64_t scales_stride) {
    return guarded([&]() -> int {
    if (!h) return fail("NULL index");
    if (h->rows.dtype != SSMI_F8) return fail("add_f8: the index does not keep 8-bit rows");
    CHECK(check_rows("add_f8", codes, codes_stride, scales, scales_stride, n, h->rows.d));
    if (n == 0) return 0;
    DeviceGuard g(h->device);
    quiesce(h);
    CHECK(reserve_rows(h, n));
    const int ns = f8_blocks(h->rows.d);
    CHECK(for_segments(h, h->rows.nrows, n, [&](long long first, long long cnt, unsigned char* c, unsigned char* s, float* lengths) -> int {
        HIPCHECK(hipMemcpy2DAsync(c, h->rows.ld, codes + first * codes_stride, codes_stride, h->rows.ld, cnt, hipMemcpyDeviceToDevice, h->stream));
        // (whole blocks, which copies fast; what the caller has behind the d codes is not part of the row)
        if (h->rows.d < h->rows.ld) HIPCHECK(hipMemset2DAsync(c + h->rows.d, h->rows.ld, 0, h->rows.ld - h->rows.d, cnt, h->stream));
        HIPCHECK(hipMemcpy2DAsync(s, h->scales.ld, scales + first * scales_stride, scales_stride, ns, cnt, hipMemcpyDeviceToDevice, h->stream));
        HIPCHECK(launch_f8_lengths(F8Mat{c, h->rows.ld, s, h->scales.ld, cnt}, h->rows.ld, lengths, (unsigned*)h->f8_longest, h->num_cu, h->stream));
        return 0;
    }));
    HIPCHECK(hipStreamSynchronize(h->stream));
    h->rows.nrows += n;
    h->scales.nrows = h->lengths.nrows = h->rows.nrows;
    return 0;
    });
}

int ssmi_index_search_f8(ssmi_index* h, int64_t nq, const uint8_t* codes, int64_t codes_stride, const uint8_t* scales, int64_t scales_stride,
                         int k, float min_score, float* D, int64_t* I, int64_t id_offset, void* stream) {
    return guarded([&]() -> int {
    if (!h) return fail("NULL index");
    if (h->rows.dtype != SSMI_F8) return fail("search_f8: the index does not keep 8-bit rows");
    CHECK(check_rows("search_f8", codes, codes_stride, scales, scales_stride, nq, h->rows.d));
    if (nq == 0) return 0;
    if (!D || !I) return fail("NULL buffer");
    if (k < 1) return fail("k must be >= 1");
    if (k > kF8MaxK) return fail("k=%d exceeds the supported maximum %d", k, kF8MaxK);
    if (nq > (1ll << 24)) return fail("nq too large");
    if (min_score != min_score) return fail("min_score is NaN");
    const unsigned min_ord = min_score <= SSMI_NEG_MAX ? 0u : f32_to_ord(min_score);
    DeviceGuard g(h->device);
    hipStream_t s = (hipStream_t)stream;
    CHECK(order_search_on(h, s));
    if (h->rows.nrows == 0) {
        HIPCHECK(launch_fill_empty(D, I, nq * k, s));
        return 0;
    }
    return f8_store_search(h, nq, F8Queries{nullptr, 0, codes, codes_stride, scales, scales_stride}, k, D, I, id_offset, s, min_ord);
    });
}

}  // extern "C"

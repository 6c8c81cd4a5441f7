// [pccl-amd extension] Kernel-level entry points used by the test-suite and micro-benchmarks (not part of pccl.h).
// dtype arguments use the CCoIP wire encoding (pccl::DType), op uses pccl::ReduceOp, algo uses pccl::QuantAlgo.
#include <algorithm>
#include <chrono>
#include <cstring>
#include <mutex>
#include <vector>

#include "../common/device_backend.hpp"
#include "../kernels/host_kernels.hpp"
#include "../kernels/muon_common.hpp"
#include "../kernels/optim_common.hpp"

using namespace pccl;

#define PCCLX_EXPORT extern "C" __attribute__((visibility("default")))

PCCLX_EXPORT int pcclxHipDeviceCount() {
    DeviceBackend *be = device_backend();
    return be ? be->device_count() : 0;
}

PCCLX_EXPORT uint32_t pcclxSimpleHash(const void *p, size_t n, int on_device) {
    if (!on_device) return kernels::simplehash_host(p, n);
    DeviceBackend *be = device_backend();
    if (!be) return 0;
    DevPtrInfo pi{};
    be->pointer_info(p, pi);
    if (pi.is_device) be->set_device(pi.device);
    return be->simplehash(p, n, nullptr);
}

// CRC-32C of host or device memory (device: HIP kernel, device_crc32c). force_sw selects the host table path.
PCCLX_EXPORT uint32_t pcclxCrc32c(const void *p, size_t n, int force_sw) {
    DeviceBackend *be = device_backend();
    DevPtrInfo pi{};
    if (be && n > 0) be->pointer_info(p, pi);
    if (pi.is_device) {
        be->set_device(pi.device);
        return device_crc32c(be, p, n, nullptr);
    }
    if (force_sw == 2 && kernels::crc32c_has_hw()) return kernels::crc32c_hw(p, n); // single-chain variant (tests)
    return force_sw ? kernels::crc32c_sw(p, n) : kernels::crc32c(p, n);
}

PCCLX_EXPORT int pcclxCrc32cHasHw() { return kernels::crc32c_has_hw() ? 1 : 0; }

PCCLX_EXPORT int pcclxFillTestPattern(void *dev, size_t n_u64) {
    DeviceBackend *be = device_backend();
    if (!be) return -1;
    return be->fill_test_pattern(dev, n_u64, nullptr) && be->device_sync() ? 0 : -1;
}

PCCLX_EXPORT int pcclxReduce(void *dst, const void *src, size_t count, int dtype, int op, int on_device) {
    if (!on_device) return kernels::host_reduce(dst, src, count, static_cast<DType>(dtype), static_cast<ReduceOp>(op)) ? 0 : -1;
    DeviceBackend *be = device_backend();
    if (!be) return -1;
    return be->reduce(dst, src, count, static_cast<DType>(dtype), static_cast<ReduceOp>(op), nullptr) && be->device_sync() ? 0 : -1;
}

PCCLX_EXPORT int pcclxFinalizeAvg(void *dst, size_t count, int dtype, size_t ws, int on_device) {
    if (!on_device) return kernels::host_finalize_avg(dst, count, static_cast<DType>(dtype), ws) ? 0 : -1;
    DeviceBackend *be = device_backend();
    if (!be) return -1;
    return be->finalize_avg(dst, count, static_cast<DType>(dtype), ws, nullptr) && be->device_sync() ? 0 : -1;
}

// meta_out: {min, max, zero_point, scale}
PCCLX_EXPORT int pcclxQuantize(void *dst_q, const void *src, size_t count, int vtype, int qtype, int algo,
                               int on_device, double *meta_out) {
    const auto vt = static_cast<DType>(vtype), qt = static_cast<DType>(qtype);
    const auto al = static_cast<QuantAlgo>(algo);
    if (!kernels::quant_supported(vt, qt, al)) return -2;
    proto::QuantMeta m;
    if (!on_device) {
        m = kernels::host_quantize(dst_q, src, count, vt, qt, al);
    } else {
        DeviceBackend *be = device_backend();
        if (!be) return -1;
        // one process-wide pinned min/max slot: a hipHostMalloc/hipHostFree pair per call cost more than the kernels
        static std::mutex mm_mutex;
        static double *mm = nullptr;
        std::lock_guard<std::mutex> lk(mm_mutex);
        if (mm == nullptr && (mm = static_cast<double *>(be->alloc_pinned(16))) == nullptr) return -1;
        be->minmax(src, count, vt, mm, nullptr);
        if (!be->device_sync()) return -1;
        m = kernels::make_meta(al, vt, qt, mm[0], mm[1]);
        if (!be->quantize(dst_q, src, count, vt, qt, kernels::make_params(m, qt), nullptr) || !be->device_sync()) return -1;
    }
    if (meta_out) {
        meta_out[0] = m.min_value;
        meta_out[1] = m.max_value;
        meta_out[2] = static_cast<double>(m.zero_point);
        meta_out[3] = m.scale;
    }
    return 0;
}

// Device only: quantizes `src` (min / max from the data, like pcclxQuantize) and overwrites it with D(Q(src)) in the
// same kernel pass (the quantized device ring's owner parity step).
PCCLX_EXPORT int pcclxQuantizeSetback(void *dst_q, void *src, size_t count, int vtype, int qtype, int algo,
                                      double *meta_out) {
    const auto vt = static_cast<DType>(vtype), qt = static_cast<DType>(qtype);
    const auto al = static_cast<QuantAlgo>(algo);
    if (!kernels::quant_supported(vt, qt, al)) return -2;
    DeviceBackend *be = device_backend();
    if (!be) return -1;
    double *mm = static_cast<double *>(be->alloc_pinned(16));
    if (!mm) return -1;
    be->minmax(src, count, vt, mm, nullptr);
    bool ok = be->device_sync();
    const proto::QuantMeta m = kernels::make_meta(al, vt, qt, mm[0], mm[1]);
    be->free_pinned(mm);
    ok = ok && be->quantize_setback(dst_q, src, count, vt, qt, kernels::make_params(m, qt), nullptr) &&
         be->device_sync();
    if (!ok) return -1;
    if (meta_out) {
        meta_out[0] = m.min_value;
        meta_out[1] = m.max_value;
        meta_out[2] = static_cast<double>(m.zero_point);
        meta_out[3] = m.scale;
    }
    return 0;
}

PCCLX_EXPORT int pcclxDequantReduce(void *dst, const void *src_q, size_t count, int vtype, int qtype, int algo, int op,
                                    const double *meta, int on_device) {
    proto::QuantMeta m;
    m.algo = static_cast<QuantAlgo>(algo);
    m.value_type = static_cast<DType>(vtype);
    m.min_value = meta[0];
    m.max_value = meta[1];
    m.zero_point = static_cast<int64_t>(meta[2]);
    m.scale = static_cast<float>(meta[3]);
    const auto vt = static_cast<DType>(vtype), qt = static_cast<DType>(qtype);
    if (!on_device) return kernels::host_dequant_reduce(dst, src_q, count, vt, qt, static_cast<ReduceOp>(op), m) ? 0 : -1;
    DeviceBackend *be = device_backend();
    if (!be) return -1;
    return be->dequant_reduce(dst, src_q, count, vt, qt, static_cast<ReduceOp>(op), kernels::make_params(m, qt), nullptr) &&
                   be->device_sync()
               ? 0
               : -1;
}

// dequant_reduce on the device with the fused per-workgroup (min, max) of the stored results, split into `pieces`
// launches (as the ring's receive ranges are) and folded: minmax_out = {min, max} of dst after the reduce
PCCLX_EXPORT int pcclxDequantReduceMinmax(void *dst, const void *src_q, size_t count, int vtype, int qtype, int algo,
                                          int op, const double *meta, int pieces, double *minmax_out) {
    proto::QuantMeta m;
    m.algo = static_cast<QuantAlgo>(algo);
    m.value_type = static_cast<DType>(vtype);
    m.min_value = meta[0];
    m.max_value = meta[1];
    m.zero_point = static_cast<int64_t>(meta[2]);
    m.scale = static_cast<float>(meta[3]);
    const auto vt = static_cast<DType>(vtype), qt = static_cast<DType>(qtype);
    DeviceBackend *be = device_backend();
    if (!be || pieces < 1) return -1;
    constexpr int kSlots = 8192;
    double *partials = static_cast<double *>(be->alloc_device(kSlots * 2 * sizeof(double)));
    double *out = static_cast<double *>(be->alloc_pinned(16));
    bool ok = partials && out;
    int used = 0;
    const size_t es = dtype_size(vt), qs = dtype_size(qt);
    const auto params = kernels::make_params(m, qt);
    for (int k = 0; ok && k < pieces; ++k) {
        const size_t a = count * k / pieces, b = count * (k + 1) / pieces;
        int blocks = 0;
        ok = kSlots - used >= 1 &&
             be->dequant_reduce_minmax(static_cast<uint8_t *>(dst) + a * es, static_cast<const uint8_t *>(src_q) + a * qs,
                                       b - a, vt, qt, static_cast<ReduceOp>(op), params, partials + 2 * used,
                                       kSlots - used, &blocks, nullptr);
        used += blocks;
    }
    ok = ok && be->minmax_fold(partials, used, count, out, nullptr) && be->device_sync();
    if (ok) {
        minmax_out[0] = out[0];
        minmax_out[1] = out[1];
    }
    if (partials) be->free_device(partials);
    if (out) be->free_pinned(out);
    return ok ? 0 : -1;
}

PCCLX_EXPORT int pcclxMultiReduce(void *const *dsts, int ndst, const void *const *srcs, int n, size_t count, int dtype,
                                  int op) {
    DeviceBackend *be = device_backend();
    if (!be) return -1;
    return be->multi_reduce(dsts, ndst, srcs, n, count, static_cast<DType>(dtype), static_cast<ReduceOp>(op), nullptr) &&
                   be->device_sync()
               ? 0
               : -1;
}

PCCLX_EXPORT int pcclxMultiGather(void *dst, const void *const *srcs, const size_t *offsets, const size_t *counts,
                                  int n, int skip, int dtype) {
    DeviceBackend *be = device_backend();
    if (!be) return -1;
    return be->multi_gather(dst, srcs, offsets, counts, n, skip, static_cast<DType>(dtype), nullptr) && be->device_sync()
               ? 0
               : -1;
}

// Event-timed device kernel micro-benchmark: returns average microseconds per call of `which`
// (0 = reduce, 1 = simplehash, 2 = multi_reduce with `n` aliases of src, 3 = quantize u8 min-max, 4 = crc32c).
PCCLX_EXPORT double pcclxBenchKernel(int which, void *dst, const void *src, size_t count, int dtype, int n, int iters) {
    DeviceBackend *be = device_backend();
    if (!be) return -1;
    DevStream st = be->create_stream();
    DevEvent e0 = be->create_event(), e1 = be->create_event();
    std::vector<const void *> srcs(static_cast<size_t>(n > 0 ? n : 1), src);
    kernels::QuantParams qp;
    proto::QuantMeta qm = kernels::make_meta(QuantAlgo::MinMax, static_cast<DType>(dtype), DType::U8, -1.0, 1.0);
    qp = kernels::make_params(qm, DType::U8);
    auto run = [&] {
        switch (which) {
            case 0: be->reduce(dst, src, count, static_cast<DType>(dtype), ReduceOp::Sum, st); break;
            case 1: be->simplehash(src, count * dtype_size(static_cast<DType>(dtype)), st); break;
            case 2: be->multi_reduce(&dst, 1, srcs.data(), n, count, static_cast<DType>(dtype), ReduceOp::Sum, st); break;
            case 3: be->quantize(dst, src, count, static_cast<DType>(dtype), DType::U8, qp, st); break;
            case 4: device_crc32c(be, src, count * dtype_size(static_cast<DType>(dtype)), st); break;
            default: break;
        }
    };
    run();
    be->stream_sync(st);
    const auto t0 = std::chrono::steady_clock::now();
    for (int i = 0; i < iters; ++i) run();
    be->stream_sync(st);
    const double us = std::chrono::duration<double, std::micro>(std::chrono::steady_clock::now() - t0).count() / iters;
    be->destroy_event(e0);
    be->destroy_event(e1);
    be->destroy_stream(st);
    return us;
}

PCCLX_EXPORT int pcclxPseudoGrad(float *pg, const float *outer, const void *local, size_t count, int local_dtype,
                                 int on_device) {
    const auto lt = static_cast<DType>(local_dtype);
    if (!on_device) return kernels::host_pseudo_grad(pg, outer, local, count, lt) ? 0 : -1;
    DeviceBackend *be = device_backend();
    if (!be) return -1;
    return be->pseudo_grad(pg, outer, local, count, lt, nullptr) && be->device_sync() ? 0 : -1;
}

PCCLX_EXPORT int pcclxOuterSgd(float *outer, float *mom, const float *pg, void *local, size_t count, int local_dtype,
                               float lr, float momentum, float dampening, float weight_decay, int nesterov, int first,
                               int on_device) {
    kernels::OuterSgdParams p;
    p.lr = lr;
    p.momentum = momentum;
    p.dampening = dampening;
    p.weight_decay = weight_decay;
    p.nesterov = nesterov;
    p.first = first;
    const auto lt = static_cast<DType>(local_dtype);
    if (!on_device) return kernels::host_outer_sgd(outer, mom, pg, local, count, lt, p) ? 0 : -1;
    DeviceBackend *be = device_backend();
    if (!be) return -1;
    return be->outer_sgd(outer, mom, pg, local, count, lt, p, nullptr) && be->device_sync() ? 0 : -1;
}

namespace {

// types of the logits, of a matrix
bool float_type(int dtype) {
    return dtype == static_cast<int>(DType::F32) || dtype == static_cast<int>(DType::BF16) ||
           dtype == static_cast<int>(DType::F16);
}

bool logprob_sizes_ok(int64_t rows, int64_t vocab, int dtype, int top_k) {
    return rows >= 0 && rows <= INT32_MAX && vocab >= 1 && vocab <= INT32_MAX && float_type(dtype) && top_k >= 0 &&
           top_k <= kernels::kMaxTopLogprobs && top_k <= vocab;
}

} // namespace

// Log probabilities of given tokens (csrc/kernels/logprob_common.hpp), asynchronous on `stream` of the current device.
// Returns 0, -1 (no device backend, or the launch failed) or -2 (arguments).
PCCLX_EXPORT int pcclxTokenLogprobs(const void *logits, int64_t row_stride, int64_t rows, int64_t vocab, int dtype,
                                    const int64_t *targets, int64_t ignore_index, int top_k, float *logprob,
                                    float *entropy, float *stats, float *top_logprob, int64_t *top_index,
                                    void *stream) {
    if (!logprob_sizes_ok(rows, vocab, dtype, top_k) ||
        (rows && (!logits || !targets || !logprob || !entropy || !stats || (top_k && (!top_logprob || !top_index)))))
        return -2;
    DeviceBackend *be = device_backend();
    if (!be) return -1;
    const kernels::LogprobArgs a{logits,  row_stride, rows,  vocab,       targets,  ignore_index,
                                 top_k,   logprob,    entropy, stats, top_logprob, top_index};
    return be->token_logprobs(a, static_cast<DType>(dtype), stream) ? 0 : -1;
}

// Gradient of pcclxTokenLogprobs with respect to the logits; g_* may be null (no gradient from that result).
PCCLX_EXPORT int pcclxTokenLogprobsGrad(const void *logits, int64_t row_stride, int64_t rows, int64_t vocab, int dtype,
                                        const int64_t *targets, int64_t ignore_index, int top_k,
                                        const float *stats, const int64_t *top_index,
                                        const float *g_logprob, const float *g_entropy, const float *g_top,
                                        void *d_logits, void *stream) {
    if (!logprob_sizes_ok(rows, vocab, dtype, top_k) ||
        (rows && (!logits || !targets || !stats || !d_logits || (top_k && g_top && !top_index))))
        return -2;
    DeviceBackend *be = device_backend();
    if (!be) return -1;
    kernels::LogprobGradArgs g;
    g.fwd = {logits, row_stride, rows, vocab, targets, ignore_index, top_k, nullptr, nullptr,
             const_cast<float *>(stats), nullptr, const_cast<int64_t *>(top_index)};
    g.g_logprob = g_logprob;
    g.g_entropy = g_entropy;
    g.g_top = g_top;
    g.d_logits = d_logits;
    return be->token_logprobs_grad(g, static_cast<DType>(dtype), stream) ? 0 : -1;
}

namespace {

// entries of a call: shapes[3 i ..] = count, rows, cols; false if a size is out of range
bool muon_entries(int n, const int64_t *shapes, std::vector<kernels::MuonEntry> &out) {
    constexpr int64_t kMax = INT32_MAX - kernels::kMuonPad;
    constexpr int64_t kMaxElems = int64_t{1} << 56; // of one entry: no address space holds it, and bytes stay in range
    if (n > 0 && !shapes) return false;
    for (int i = 0; i < n; ++i) {
        const int64_t count = shapes[3 * i], rows = shapes[3 * i + 1], cols = shapes[3 * i + 2];
        if (count < 0 || rows < 0 || cols < 0 || count > kMax || rows > kMax || cols > kMax) return false;
        if (rows && cols && count > kMaxElems / rows / cols) return false;
        kernels::MuonEntry e;
        e.count = static_cast<int>(count);
        e.rows = static_cast<int>(rows);
        e.cols = static_cast<int>(cols);
        out.push_back(e);
    }
    return true;
}

struct Span {
    uintptr_t from, to;
    bool written;
};

// a written tensor that shares memory with another one of the call
bool spans_collide(std::vector<Span> &v) {
    std::sort(v.begin(), v.end(), [](const Span &a, const Span &b) { return a.from < b.from; });
    uintptr_t end = 0, written_end = 0; // furthest end so far, of any span / of the written ones
    for (const Span &s : v) {
        if (s.from < written_end || (s.written && s.from < end)) return true;
        end = std::max(end, s.to);
        if (s.written) written_end = std::max(written_end, s.to);
    }
    return false;
}

} // namespace

// Bytes of workspace pcclxMuon needs for n entries of (count, rows, cols); -1: sizes out of range.
PCCLX_EXPORT int64_t pcclxMuonWorkspace(int n, const int64_t *shapes) {
    try {
        std::vector<kernels::MuonEntry> entries;
        if (n < 0 || !muon_entries(n, shapes, entries)) return -1;
        return static_cast<int64_t>(kernels::muon_plan(entries, 1, 1, nullptr));
    } catch (...) {
        return -1;
    }
}

// Orthogonalises (mom = null) or takes a Muon step on n entries of `count` contiguous row-major matrices each
// (csrc/kernels/muon_common.hpp), asynchronously on `stream` of the current device. w[i] may be g[i] itself where
// types agree; otherwise nothing written may overlap anything else. Returns 0, -1 (no backend / launch failed), -2
// (arguments), -3 (overlap).
PCCLX_EXPORT int pcclxMuon(int n, const int64_t *shapes, const void *const *g, int gtype, void *const *w, int wtype,
                           float *const *mom, const float *alpha, double decay, double momentum, int nesterov,
                           int steps, const float *coefficients, double eps, void *workspace, int64_t workspace_bytes,
                           void *stream) {
    try {
        const auto gt = static_cast<DType>(gtype), wt = static_cast<DType>(wtype);
        if (n < 0 || steps < 1 || !float_type(gtype) || !float_type(wtype) || !coefficients || (n > 0 && (!g || !w)) ||
            (mom && !alpha))
            return -2;
        std::vector<kernels::MuonEntry> entries;
        if (!muon_entries(n, shapes, entries)) return -2;
        std::vector<Span> spans;
        for (int i = 0; i < n; ++i) {
            auto &e = entries[i];
            e.g = g[i];
            e.w = w[i];
            e.mom = mom ? mom[i] : nullptr;
            e.alpha = alpha ? alpha[i] : 0.0f;
            const size_t elems = static_cast<size_t>(e.count) * e.rows * e.cols;
            if (elems == 0) continue;
            if (!e.g || !e.w || (mom && !e.mom)) return -2; // a tensor without storage of its own
            const auto span = [&](const void *p, size_t es, bool written) {
                const auto from = reinterpret_cast<uintptr_t>(p);
                spans.push_back({from, from + elems * es, written});
            };
            const bool in_place = !mom && e.g == e.w && gt == wt;
            if (!in_place) span(e.g, dtype_size(gt), false);
            span(e.w, dtype_size(wt), true);
            if (mom) span(e.mom, sizeof(float), true);
        }
        if (spans_collide(spans)) return -3;
        std::vector<std::vector<kernels::MuonEntry>> groups;
        const size_t need = kernels::muon_plan(entries, dtype_size(gt), dtype_size(wt), &groups);
        if (workspace_bytes < 0 || static_cast<size_t>(workspace_bytes) < need || (need > 0 && !workspace) ||
            reinterpret_cast<uintptr_t>(workspace) % 16 != 0)
            return -2;
        if (groups.empty()) return 0;
        DeviceBackend *be = device_backend();
        if (!be) return -1;
        kernels::MuonParams p;
        p.steps = steps;
        p.a = coefficients[0];
        p.b = coefficients[1];
        p.c = coefficients[2];
        p.eps = eps;
        p.momentum = static_cast<float>(momentum);
        p.decay = static_cast<float>(decay);
        p.nesterov = nesterov;
        for (const auto &group : groups)
            if (!be->muon(group.data(), static_cast<int>(group.size()), gt, wt, p, workspace, stream)) return -1;
        return 0;
    } catch (...) {
        return -1;
    }
}

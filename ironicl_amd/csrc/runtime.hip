// Host runtime of the gfx950 TabICLv2 backend and its C ABI (include/ironicl_hip.h).
//
// Plays the part of src/models/tabicl_v2/cuda/{build,predictor,weights,
// workspace}.rs for the MI355X: the static-context build and cached
// prediction as sequences of launches on one HIP stream, with every buffer
// of a pass carved from one device arena and the context's K/V kept resident
// in HBM.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <memory>
#include <mutex>
#include <new>
#include <string>
#include <system_error>
#include <thread>
#include <vector>

#include "../../include/ironicl_hip.h"
#include "common.hpp"

namespace irx {

thread_local std::string g_last_error;

[[noreturn]] void fail(int status, const std::string &message) { throw Failure{status, message}; }

void check_hip(hipError_t err, const char *what) {
    if (err == hipSuccess) return;
    int status = err == hipErrorOutOfMemory ? IRX_OUT_OF_MEMORY : IRX_DEVICE_ERROR;
    fail(status, std::string("ROCm: ") + what + ": " + hipGetErrorString(err));
}

// ---- kernel timing ----

namespace {
struct PendingTiming {
    KernelFamily family;
    hipEvent_t start, stop;
    double flops, bytes;
};
struct FamilyTotals {
    uint64_t launches = 0;
    double ms = 0, flops = 0, bytes = 0;
    std::vector<std::pair<double, double>> spans;  // launch intervals, ms after g_epoch
};
std::atomic<unsigned> g_profiling{0};
std::mutex g_profile_mu;
std::vector<PendingTiming> g_pending;
FamilyTotals g_totals[kFamCount];
hipEvent_t g_epoch = nullptr;  // recorded when profiling is enabled

// Length of the union of intervals (launches on several streams may overlap).
double union_ms(std::vector<std::pair<double, double>> v) {
    std::sort(v.begin(), v.end());
    double total = 0, lo = 0, hi = -1e300;
    for (const auto &[a, b] : v) {
        if (a > hi) {
            if (hi > lo) total += hi - lo;
            lo = a, hi = b;
        } else if (b > hi) {
            hi = b;
        }
    }
    if (hi > lo) total += hi - lo;
    return total;
}
const char *const kFamilyNames[kFamCount] = {"gemm", "icl_attention", "icl_merge", "small_attention",
                                             "layer_norm", "glue"};

void drain_timings() {
    for (auto &p : g_pending) {
        float ms = 0.f, at = 0.f;
        if (hipEventSynchronize(p.stop) == hipSuccess && hipEventElapsedTime(&ms, p.start, p.stop) == hipSuccess) {
            FamilyTotals &t = g_totals[p.family];
            t.launches += 1, t.ms += ms, t.flops += p.flops, t.bytes += p.bytes;
            if (g_epoch && hipEventElapsedTime(&at, g_epoch, p.start) == hipSuccess) t.spans.emplace_back(at, at + ms);
        }
        (void)hipEventDestroy(p.start);
        (void)hipEventDestroy(p.stop);
    }
    g_pending.clear();
}
}  // namespace

KernelTimer::KernelTimer(KernelFamily family, hipStream_t stream, double flops, double bytes)
    : family_(family), stream_(stream), flops_(flops), bytes_(bytes) {
    if (!(g_profiling.load(std::memory_order_relaxed) & (1u << family))) return;
    if (hipEventCreate(&start_) != hipSuccess || hipEventCreate(&stop_) != hipSuccess ||
        hipEventRecord(start_, stream_) != hipSuccess) {
        if (start_) (void)hipEventDestroy(start_);
        if (stop_) (void)hipEventDestroy(stop_);
        start_ = stop_ = nullptr;
    }
}

KernelTimer::~KernelTimer() {
    if (!start_) return;
    if (hipEventRecord(stop_, stream_) != hipSuccess) {
        (void)hipEventDestroy(start_);
        (void)hipEventDestroy(stop_);
        return;
    }
    std::lock_guard<std::mutex> lock(g_profile_mu);
    g_pending.push_back({family_, start_, stop_, flops_, bytes_});
}

namespace {

// ---- device memory ----

struct DevBuf {
    void *p = nullptr;
    size_t bytes = 0;
    DevBuf() = default;
    explicit DevBuf(size_t b) { alloc(b); }
    DevBuf(const DevBuf &) = delete;
    DevBuf &operator=(const DevBuf &) = delete;
    DevBuf(DevBuf &&o) noexcept : p(o.p), bytes(o.bytes) { o.p = nullptr, o.bytes = 0; }
    DevBuf &operator=(DevBuf &&o) noexcept {
        if (this != &o) {
            release();
            p = o.p, bytes = o.bytes;
            o.p = nullptr, o.bytes = 0;
        }
        return *this;
    }
    ~DevBuf() { release(); }
    void alloc(size_t b) {
        release();
        if (b) {
            IRX_HIP(hipMalloc(&p, b));
            bytes = b;
        }
    }
    void release() {
        if (p) (void)hipFree(p);
        p = nullptr, bytes = 0;
    }
    float *f() const { return static_cast<float *>(p); }
};

// Pinned host memory (hipHostMalloc), grown on demand: copies between it and
// the device are asynchronous, where copies from pageable memory block the
// host until the stream reaches them.
struct PinnedBuf {
    void *p = nullptr;
    size_t bytes = 0;
    PinnedBuf() = default;
    PinnedBuf(const PinnedBuf &) = delete;
    PinnedBuf &operator=(const PinnedBuf &) = delete;
    ~PinnedBuf() { release(); }
    void reserve(size_t b) {
        if (b <= bytes) return;
        release();
        IRX_HIP(hipHostMalloc(&p, b, hipHostMallocDefault));
        bytes = b;
    }
    void release() {
        if (p) (void)hipHostFree(p);
        p = nullptr, bytes = 0;
    }
    float *f() const { return static_cast<float *>(p); }
};

// Bump allocator over one device allocation: its own `buf`, or memory it
// borrows (`lent`, `lent_bytes`). With `counting`, only sums sizes.
struct Arena {
    DevBuf buf;
    void *lent = nullptr;
    size_t lent_bytes = 0;
    size_t used = 0;
    bool counting = false;
    static size_t round(size_t floats) { return (floats * 4 + 255) & ~size_t(255); }
    float *take(size_t floats) {
        size_t b = round(floats);
        if (counting) {
            used += b;
            return nullptr;
        }
        char *base = static_cast<char *>(lent ? lent : buf.p);
        if (used + b > (lent ? lent_bytes : buf.bytes)) fail(IRX_OUT_OF_MEMORY, "ROCm: workspace exhausted");
        float *p = reinterpret_cast<float *>(base + used);
        used += b;
        return p;
    }
    uint8_t *take_bytes(size_t bytes) { return reinterpret_cast<uint8_t *>(take((bytes + 3) / 4)); }
};

void upload(void *dst, const void *src, size_t bytes, hipStream_t s) {
    if (bytes) IRX_HIP(hipMemcpyAsync(dst, src, bytes, hipMemcpyHostToDevice, s));
}
void download(void *dst, const void *src, size_t bytes, hipStream_t s) {
    if (bytes) IRX_HIP(hipMemcpyAsync(dst, src, bytes, hipMemcpyDeviceToHost, s));
}

// RoPE tables of the row stage: cos twice and [-sin, sin] per 16-wide head
// for `len` positions (rope_tables, src/models/tabicl_v2/cpu.rs:4089-4102).
void rope_tables(const float *freqs, int len, std::vector<float> &cos_t, std::vector<float> &sin_t) {
    cos_t.assign((size_t)len * 16, 0.f);
    sin_t.assign((size_t)len * 16, 0.f);
    for (int row = 0; row < len; ++row)
        for (int i = 0; i < 8; ++i) {
            float angle = (float)row * freqs[i];
            float s = sinf(angle), c = cosf(angle);
            cos_t[row * 16 + i] = c, cos_t[row * 16 + i + 8] = c;
            sin_t[row * 16 + i] = -s, sin_t[row * 16 + i + 8] = s;
        }
}

}  // namespace
}  // namespace irx

using namespace irx;

// ---- the no-allocation entry point's scratch ----

// Split-K partials of irx_icl_attention_noalloc, for callers that cannot
// allocate (code under HIP graph capture, tight serving loops). Every GPU the
// library runs on holds its own copy until the process ends; host code never
// uses this name as an address, only the per-device pointer that
// hipGetSymbolAddress returns (irx_device::scratch).
constexpr size_t kNoAllocScratchBytes = size_t(64) << 20;
static __device__ __align__(256) float scratch[kNoAllocScratchBytes / sizeof(float)];

// ---- opaque ABI objects ----

struct irx_device {
    int ordinal = 0;
    int compute_units = 0;
    // This device's copy of `scratch`, looked up once when the device is opened.
    float *scratch = nullptr;
    std::atomic<int> refs{1};
    // Idle non-blocking streams for builds, predictors and preprocessors to
    // reuse: creating one costs about a millisecond.
    std::mutex stream_mu;
    std::vector<hipStream_t> idle_streams;
    // Builds upload their ICL labels on this stream while the column stage
    // runs; it has a hardware queue of its own (a CU-masked stream), so the
    // copy never waits behind the build's kernels on a shared queue.
    hipStream_t upload = nullptr;
    // Idle streams with a hardware queue each, for predictors' passes: creating
    // one takes milliseconds (a new queue), so they are kept for reuse.
    std::vector<hipStream_t> idle_lanes;
    // The last build's workspace, lent to the next build on this device (one
    // at a time; a concurrent build allocates its own). Freeing a workspace of
    // several GB after every build and allocating the next one left the first
    // small allocation after a build waiting 0.3-0.7 s in the runtime once a
    // few builds had run. Kept while at most an eighth of the device memory.
    std::mutex build_mu;
    DevBuf build_ws;
    bool build_ws_lent = false;
    size_t memory_bytes = 0;
    ~irx_device() {
        if (idle_streams.empty() && idle_lanes.empty() && !upload && !build_ws.p) return;
        (void)hipSetDevice(ordinal);
        build_ws.release();
        if (upload) (void)hipStreamDestroy(upload);
        for (hipStream_t s : idle_lanes) (void)hipStreamDestroy(s);
        for (hipStream_t s : idle_streams) (void)hipStreamDestroy(s);
    }
};

namespace {

constexpr size_t kIdleStreams = 16;

// An idle stream of the device (current on this thread), or a new one.
hipStream_t take_stream(irx_device *d) {
    {
        std::lock_guard<std::mutex> lock(d->stream_mu);
        if (!d->idle_streams.empty()) {
            hipStream_t s = d->idle_streams.back();
            d->idle_streams.pop_back();
            return s;
        }
    }
    hipStream_t s = nullptr;
    IRX_HIP(hipStreamCreateWithFlags(&s, hipStreamNonBlocking));
    return s;
}

// Waits for the stream's work and keeps it for the next taker.
// A stream with a hardware queue of its own: a stream created with a CU mask
// (here every CU) gets one, where plain streams share the runtime's pool of
// queues, on which work of two streams runs in turn.
hipStream_t own_queue_stream(const irx_device *d) {
    std::vector<uint32_t> all_cus((d->compute_units + 31) / 32, 0xffffffffu);
    hipStream_t s = nullptr;
    if (hipExtStreamCreateWithCUMask(&s, (uint32_t)all_cus.size(), all_cus.data()) != hipSuccess) {
        (void)hipGetLastError();
        s = nullptr;
        IRX_HIP(hipStreamCreateWithFlags(&s, hipStreamNonBlocking));
    }
    return s;
}

hipStream_t upload_stream(irx_device *d) {
    std::lock_guard<std::mutex> lock(d->stream_mu);
    if (!d->upload) d->upload = own_queue_stream(d);
    return d->upload;
}

hipStream_t take_lane(irx_device *d) {
    {
        std::lock_guard<std::mutex> lock(d->stream_mu);
        if (!d->idle_lanes.empty()) {
            hipStream_t s = d->idle_lanes.back();
            d->idle_lanes.pop_back();
            return s;
        }
    }
    return own_queue_stream(d);
}

void return_lane(irx_device *d, hipStream_t s) {
    if (!s) return;
    (void)hipStreamSynchronize(s);
    std::lock_guard<std::mutex> lock(d->stream_mu);
    if (d->idle_lanes.size() < kIdleStreams)
        d->idle_lanes.push_back(s);
    else
        (void)hipStreamDestroy(s);
}

void return_stream(irx_device *d, hipStream_t s) {
    if (!s) return;
    (void)hipStreamSynchronize(s);
    std::lock_guard<std::mutex> lock(d->stream_mu);
    if (d->idle_streams.size() < kIdleStreams)
        d->idle_streams.push_back(s);
    else
        (void)hipStreamDestroy(s);
}

}  // namespace

struct Lin {
    const float *w = nullptr, *b = nullptr;
    PairW pairs = {};  // 512-wide blocks and the decoder: w as FP16 pairs
};

struct BlockW {
    int dim = 0;
    const float *n1w = nullptr, *n1b = nullptr, *n2w = nullptr, *n2b = nullptr;
    const float *in_w = nullptr, *in_b = nullptr;  // [3 dim, dim], [3 dim]
    PairW in_pairs = {};                           // 512-wide blocks: in_w as FP16 pairs
    Lin out, l1, l2;
    bool qass = false;
    Lin qm0, qm2;  // QASS query MLP, per head: hd -> 64 -> hd
    const float *tail_pack = nullptr;  // 128-wide blocks: out, linear1, linear2 packed for tail128
    const float *head_pack = nullptr;  // 128-wide prediction blocks: the in_proj rows head128 needs
    int head_nb = 0, head_row0 = 0;    // head128 output blocks of 16, first in_proj row
};

struct irx_weights {
    irx_device *device = nullptr;
    std::atomic<int> refs{1};
    int task = 0;
    int width = 0;
    size_t bytes = 0;
    DevBuf arena, pairs;
    const float *in_w = nullptr, *in_b = nullptr;
    const float *ind[kColumnBlocks] = {};
    BlockW col1[kColumnBlocks], col2[kColumnBlocks], row[kRowBlocks], icl[kIclBlocks];
    const float *cls = nullptr, *out_ln_w = nullptr, *out_ln_b = nullptr;
    const float *ln_w = nullptr, *ln_b = nullptr;
    Lin dec0, dec2;
    // Label encoders (y_encoder) of the column and ICL stages, for builds
    // given targets: weight [width, classes] (1 column for the regressor).
    Lin ycol, yicl;
    int classes = 0;
    std::vector<float> freqs_host;
};

// The context's caches on the device: per column block K then V,
// [2, B, H+4, 8, 128, 16]; per ICL block K then V, [2, B, 8, N, 64].
struct irx_built_cache {
    irx_device *device = nullptr;
    irx_shape shape{};
    int precision = IRX_PRECISION_FP32;  // SPLIT: the ICL buffers hold the FP16 cache layout
    DevBuf column[kColumnBlocks];
    DevBuf icl[kIclBlocks];      // HALF: the FP8 blocks
    DevBuf icl16[kIclBlocks];    // HALF: the FP16 cache the build made, kept for context reads
};

// Most HIP streams a predictor's passes rotate over (GPU_MAX_HW_QUEUES is 4).
constexpr int kMaxPassStreams = 4;
// Most pass graphs a predictor keeps: 4 streams x the 47 pass shapes of the
// default 512-row passes (larger passes evict the oldest).
constexpr size_t kMaxPassGraphs = 192;

// A pass replayed from a HIP graph: one per (stream slot, rows), captured on
// first use over the slot's workspace; dropped when a workspace moves.
struct PassGraphEntry {
    int slot;
    int rows;
    hipGraphExec_t exec;
};

struct irx_predictor {
    irx_weights *weights = nullptr;
    irx_shape shape{};
    int precision = IRX_PRECISION_FP32;
    size_t pass_rows = 512;
    DevBuf column[kColumnBlocks];
    DevBuf icl[kIclBlocks];
    DevBuf icl16[kIclBlocks];  // HALF, adopted from a build: its FP16 cache, for context reads
    DevBuf base_scales;   // [12, 512]
    DevBuf rope_cos, rope_sin;
    hipStream_t stream = nullptr;
    // Passes rotate over `streams` HIP streams (the main one, then side[0..]),
    // each with its own workspace, so that one pass's short launches overlap
    // another's long ones.
    hipStream_t side[kMaxPassStreams - 1] = {};
    hipEvent_t fork = nullptr, join[kMaxPassStreams - 1] = {};
    int streams = 2;
    std::mutex mu;
    Arena ws[kMaxPassStreams];
    // Host-buffer predictions: device inputs, outputs and missing-row flags,
    // and pinned staging for the inputs and logits, grown to the largest call
    // so far.
    DevBuf io_x, io_logits, io_flags;
    PinnedBuf pin_x, pin_logits;
    // Passes replayed from HIP graphs, oldest first.
    std::vector<PassGraphEntry> graphs;
    bool use_graphs = true;
    void drop_graphs() {
        for (auto &g : graphs) (void)hipGraphExecDestroy(g.exec);
        graphs.clear();
    }
    hipStream_t lane(int slot) const { return slot ? side[slot - 1] : stream; }
    size_t ws_rows = 0;
};

namespace {

void set_device(const irx_device *d) { IRX_HIP(hipSetDevice(d->ordinal)); }

// ---- stages shared by the build and the predictor ----

// Rows up to which the ICL query path (LN1, projection, QASS) runs as one
// launch (prediction passes); larger ones (the build's N rows) take the
// LayerNorm that the K/V projection shares and separate products.
constexpr long long kLnLinearRows = 8192;
// States (columns x rows) from which a cached column block runs as one
// kernel of 64-row tiles (column_block) rather than its small-pass form of
// 16 rows per workgroup. Measured per block at 64 columns (the three
// launches the one kernel replaced in brackets): 32 rows 53.6 / 20.8 (32.7)
// us, 128 rows 55.7 / 37.8 (77.9) us, 256 rows 60.0 / 68.5 (77.2) us, 512
// rows 101 / 122 (115) us; the tiled kernel streams 512 KB of weights and
// K/V through LDS per tile.
constexpr long long kColumnFusedRows = 12288;

struct Stages {
    const irx_weights &w;
    hipStream_t s;
    int cus;

    void linear(const float *a, long long lda, long long m, int k, const float *wt, const float *b, int n,
                float *c, long long ldc, int epi = kEpiNone, const float *res = nullptr, long long ldr = 0) const {
        GemmArgs g{};
        g.a = a, g.lda = lda, g.w = wt, g.bias = b, g.residual = res, g.ldr = ldr, g.c = c;
        g.out = OutMap::row_major(n, ldc);
        g.m = (int)m, g.n = n, g.k = k, g.epilogue = epi;
        gemm(g, s);
    }

    // The same product of a packed matrix, for m rows (pair_rows).
    void linear_pairs(const float *a, long long lda, long long m, int k, const PairW &wt, const float *b, int n,
                      float *c, const OutMap &map, int epi = kEpiNone, const float *res = nullptr, long long ldr = 0,
                      const float *lnw = nullptr, const float *lnb = nullptr) const {
        PairLinear g{};
        g.x = a, g.ldx = lda, g.lnw = lnw, g.lnb = lnb, g.w = wt, g.bias = b, g.residual = res, g.ldr = ldr, g.c = c;
        g.out = map, g.m = (int)m, g.n = n, g.k = k, g.epilogue = epi, g.compute_units = cus;
        pair_linear(g, s);
    }

    // gelu(LN(x) W^T + b) of 512-wide rows into out [m, n].
    void ln_gelu512(const float *x, long long m, const float *lnw, const float *lnb, const Lin &l, int n,
                    float *out) const {
        if (m > kFewRows) {
            linear_pairs(x, 512, m, 512, l.pairs, l.b, n, out, OutMap::row_major(n, n), kEpiGelu, nullptr, 0, lnw, lnb);
            return;
        }
        LnLinear f{};
        f.x = x, f.ldx = 512, f.lnw = lnw, f.lnb = lnb, f.w = l.w, f.b = l.b, f.out = out, f.ldo = n;
        f.m = (int)m, f.n = n;
        ln_linear512(f, kLnGelu, s);
    }

    // LayerNorm of 128-wide rows x [m, 128] and the product that reads it:
    // taken in the product's prologue when the product is prediction-sized,
    // else written to `norm` first.
    void ln_linear128(const float *x, long long m, const float *lnw, const float *lnb, float *norm, const float *wt,
                      const float *b, int n, float *c, long long ldc, int epi = kEpiNone) const {
        if (gemm_fuses_ln(m, n)) {
            GemmArgs g{};
            g.a = x, g.lda = 128, g.w = wt, g.bias = b, g.c = c, g.out = OutMap::row_major(n, ldc);
            g.m = (int)m, g.n = n, g.k = 128, g.epilogue = epi, g.ln_w = lnw, g.ln_b = lnb;
            gemm(g, s);
            return;
        }
        layer_norm(x, 128, lnw, lnb, norm, 128, m, 128, s);
        linear(norm, 128, m, 128, wt, b, n, c, ldc, epi);
    }

    // LN1 + the in_proj rows [head_row0, head_row0 + 16 head_nb) of a 128-wide
    // block into out [m, ldo]: one fused launch from 16384 rows (as the tail),
    // else LayerNorm into `norm` and a product.
    void head(const BlockW &bw, const float *x, long long m, float *norm, float *out, long long ldo) const {
        const int n = 16 * bw.head_nb;
        if (bw.head_pack && m >= 16384) {
            Head128 h{};
            h.x = x, h.ldx = 128, h.lnw = bw.n1w, h.lnb = bw.n1b, h.pack = bw.head_pack;
            h.b = bw.in_b + bw.head_row0, h.out = out, h.ldo = ldo, h.m = m, h.nb = bw.head_nb;
            head128(h, s);
            return;
        }
        ln_linear128(x, m, bw.n1w, bw.n1b, norm, bw.in_w + (size_t)bw.head_row0 * 128, bw.in_b + bw.head_row0, n,
                     out, ldo);
    }

    void linear_map(const float *a, long long lda, long long m, int k, const float *wt, const float *b, int n,
                    float *c, const OutMap &map) const {
        GemmArgs g{};
        g.a = a, g.lda = lda, g.w = wt, g.bias = b, g.c = c, g.out = map;
        g.m = (int)m, g.n = n, g.k = k, g.epilogue = kEpiNone;
        gemm(g, s);
    }

    // Post-attention half of a block: out-projection + residual into `state`,
    // then LN2, FFN (GELU) and residual (cpu.rs:1555-1601).
    // A 128-wide block's tail runs fused: tail128 once its rows fill the chip
    // (one wave carries 16 rows through the whole chain, 256 workgroups at
    // 16384 rows), below that its 16-rows-per-workgroup form, whose four
    // waves split each product. fused: -1 chooses; 0 forces the four
    // separate launches, 1 tail128, 2 the small-pass form.
    void tail(const BlockW &bw, float *state, long long m, const float *att, float *norm, float *hid,
              int fused = -1) const {
        const int d = bw.dim;
        const bool packed = d == 128 && bw.tail_pack;
        const bool use_fused = fused < 0 ? packed : fused >= 1;
        const bool rows16 = fused < 0 ? m < 16384 : fused == 2;
        if (d == 512) {
            // LN2 fused into the FFN's first product.
            const OutMap rows = OutMap::row_major(d, d);
            const bool few = m <= kFewRows;
            if (few)
                linear(att, d, m, d, bw.out.w, bw.out.b, d, state, d, kEpiResidual, state, d);
            else
                linear_pairs(att, d, m, d, bw.out.pairs, bw.out.b, d, state, rows, kEpiResidual, state, d);
            ln_gelu512(state, m, bw.n2w, bw.n2b, bw.l1, 2 * d, hid);
            if (few)
                linear(hid, 2 * d, m, 2 * d, bw.l2.w, bw.l2.b, d, state, d, kEpiResidual, state, d);
            else
                linear_pairs(hid, 2 * d, m, 2 * d, bw.l2.pairs, bw.l2.b, d, state, rows, kEpiResidual, state, d);
            return;
        }
        if (use_fused) {
            if (d != 128 || !bw.tail_pack) fail(IRX_INVALID_ARGUMENT, "the fused tail needs a packed 128-wide block");
            Tail128 t{};
            t.att = att, t.lda = d, t.state = state, t.ldx = d, t.pack = bw.tail_pack, t.m = m;
            t.bo = bw.out.b, t.n2w = bw.n2w, t.n2b = bw.n2b, t.b1 = bw.l1.b, t.b2 = bw.l2.b;
            tail128(t, s, rows16);
            return;
        }
        linear(att, d, m, d, bw.out.w, bw.out.b, d, state, d, kEpiResidual, state, d);
        ln_linear128(state, m, bw.n2w, bw.n2b, norm, bw.l1.w, bw.l1.b, 2 * d, hid, 2 * d, kEpiGelu);
        linear(hid, 2 * d, m, 2 * d, bw.l2.w, bw.l2.b, d, state, d, kEpiResidual, state, d);
    }

    // multihead_attn2 of column block `blk` for `cols` columns of `rows`
    // states [cols, rows, 128] against cached inducing K/V: column c reads
    // kcache + (c / group) * group_stride + (c % group) * 16384
    // (cached_block, cpu.rs:2587-2850; column_block_f32, kernels.rs:1342).
    // fused: -1 chooses, 0 the three launches (head, 16-wide attention,
    // tail), 1 column_block's one kernel (the head128 / tail128 arithmetic:
    // bitwise the three launches from 16384 rows), 2 its small-pass form
    // (the same bits).
    void column_attend(int blk, float *state, int cols, int rows, const float *kcache, const float *vcache,
                       int group, long long group_stride, float *norm, float *q, float *att, float *hid,
                       int fused = -1) const {
        const BlockW &bw = w.col2[blk];
        const long long m = (long long)cols * rows;
        const bool packed = bw.head_pack && bw.head_nb == 8 && bw.head_row0 == 0 && bw.tail_pack;
        if (fused < 0) fused = !packed ? 0 : m >= kColumnFusedRows ? 1 : 2;
        if (fused >= 1) {
            if (!packed) fail(IRX_INVALID_ARGUMENT, "the fused column block needs packed weights");
            ColumnBlock c{};
            c.state = state, c.rows = rows, c.cols = cols, c.k = kcache, c.v = vcache, c.group = group;
            c.group_stride = group_stride, c.lnw = bw.n1w, c.lnb = bw.n1b, c.qpack = bw.head_pack, c.qb = bw.in_b;
            c.pack = bw.tail_pack, c.bo = bw.out.b, c.n2w = bw.n2w, c.n2b = bw.n2b, c.b1 = bw.l1.b, c.b2 = bw.l2.b;
            column_block(c, s, fused == 2);
            return;
        }
        head(bw, state, m, norm, q, kColumnDim);
        SmallAttention a{};
        a.q = q, a.q_seq = (long long)rows * kColumnDim, a.q_group = (long long)group * rows * kColumnDim;
        a.q_row = kColumnDim, a.q_head = kColumnHead;
        a.k = kcache, a.k_seq = kColumnCache, a.k_group = group_stride, a.k_row = kColumnHead;
        a.k_head = kInducing * kColumnHead;
        a.v = vcache, a.v_seq = kColumnCache, a.v_group = group_stride, a.v_row = kColumnHead;
        a.v_head = kInducing * kColumnHead;
        a.o = att, a.o_seq = a.q_seq, a.o_group = a.q_group, a.o_row = kColumnDim, a.o_head = kColumnHead;
        a.group = group, a.seqs = cols, a.heads = kHeads, a.q_rows = rows, a.kv_rows = kInducing;
        a.scale = 0.25f;
        small_attention(a, s);
        tail(bw, state, m, att, norm, hid);
    }

    struct RowBuffers {
        float *seq, *norm, *qkv, *att, *hid, *cls, *cnorm, *cq, *catt, *chid;
    };
    static RowBuffers row_buffers(Arena &a, long long seqs, int len) {
        long long m = seqs * len, c = seqs * kReserved;
        RowBuffers r{};
        r.seq = a.take(m * 128), r.norm = a.take(m * 128), r.qkv = a.take(m * 384), r.att = a.take(m * 128);
        r.hid = a.take(m * 256), r.cls = a.take(c * 128), r.cnorm = a.take(c * 128), r.cq = a.take(c * 128);
        r.catt = a.take(c * 128), r.chid = a.take(c * 256);
        return r;
    }

    // The row transformer (row_embedding, cpu.rs:1226-1266) for `rows` rows of
    // `b` estimators from column states [b*h, rows_total, 128] starting at
    // row `start`... the caller passes states whose row dimension is `rows`.
    void row_stage(const float *state, int b, int rows, int h, float *out, const float *rope_cos,
                   const float *rope_sin, const RowBuffers &r) const {
        const int len = h + kReserved;
        const long long seqs = (long long)b * rows, m = seqs * len;
        build_rows(state, b, rows, h, w.cls, r.seq, s);
        for (int blk = 0; blk < 2; ++blk) {
            const BlockW &bw = w.row[blk];
            head(bw, r.seq, m, r.norm, r.qkv, 384);
            SmallAttention a{};
            a.q = r.qkv, a.k = r.qkv + 128, a.v = r.qkv + 256;
            a.q_seq = a.k_seq = a.v_seq = (long long)len * 384;
            a.q_group = a.k_group = a.v_group = 0;
            a.q_row = a.k_row = a.v_row = 384;
            a.q_head = a.k_head = a.v_head = kColumnHead;
            a.o = r.att, a.o_seq = (long long)len * 128, a.o_group = 0, a.o_row = 128, a.o_head = kColumnHead;
            a.group = (int)std::min<long long>(seqs, 1 << 30), a.seqs = (int)seqs, a.heads = kHeads;
            a.q_rows = len, a.kv_rows = len, a.scale = 0.25f, a.rope_cos = rope_cos, a.rope_sin = rope_sin;
            small_attention(a, s);
            tail(bw, r.seq, m, r.att, r.norm, r.hid);
        }
        // Block 2: only the CLS tokens query; keys and values are every token.
        const BlockW &bw = w.row[2];
        const long long mc = seqs * kReserved;
        gather_cls(r.seq, seqs, len, r.cls, s);
        head(bw, r.seq, m, r.norm, r.qkv, 256);
        ln_linear128(r.cls, mc, bw.n1w, bw.n1b, r.cnorm, bw.in_w, bw.in_b, 128, r.cq, 128);
        SmallAttention a{};
        a.q = r.cq, a.q_seq = kReserved * 128, a.q_group = 0, a.q_row = 128, a.q_head = kColumnHead;
        a.k = r.qkv, a.v = r.qkv + 128, a.k_seq = a.v_seq = (long long)len * 256, a.k_group = a.v_group = 0;
        a.k_row = a.v_row = 256, a.k_head = a.v_head = kColumnHead;
        a.o = r.catt, a.o_seq = kReserved * 128, a.o_group = 0, a.o_row = 128, a.o_head = kColumnHead;
        a.group = (int)std::min<long long>(seqs, 1 << 30), a.seqs = (int)seqs, a.heads = kHeads;
        a.q_rows = kReserved, a.kv_rows = len, a.scale = 0.25f, a.rope_cos = rope_cos, a.rope_sin = rope_sin;
        small_attention(a, s);
        tail(bw, r.cls, mc, r.catt, r.cnorm, r.chid);
        // out_ln of the 4 CLS tokens = the [512] row representation.
        layer_norm(r.cls, 128, w.out_ln_w, w.out_ln_b, out, 128, mc, 128, s);
    }

    struct IclBuffers {
        float *norm, *qh, *qg, *att, *hid, *partial;
        size_t partial_floats;
    };
    static IclBuffers icl_buffers(Arena &a, long long rows, int b, int q_rows, int kv_rows, int cus, bool f16 = false) {
        IclBuffers r{};
        r.norm = a.take(rows * 512), r.qh = a.take(rows * 512);
        r.qg = a.take(rows * 512), r.att = a.take(rows * 512), r.hid = a.take(rows * 1024);
        r.partial_floats = icl_attention_partial_floats(b * kHeads, q_rows, kv_rows, cus, f16);
        r.partial = r.partial_floats ? a.take(r.partial_floats) : nullptr;
        return r;
    }

    // LN1, the Q projection and QASSMax of an ICL block's `b` x `rows` rows, into
    // qg head-major [b, 8, rows, 64]: one launch (fused), else through `norm`
    // (normed: already there) and the projected rows in qh.
    void icl_query_rows(const BlockW &bw, const float *x, int b, int rows, const float *base, float *norm, float *qh,
                        float *qg, bool normed, bool fused) const {
        const long long m = (long long)b * rows;
        if (fused) {
            LnLinear f{};
            f.x = x, f.ldx = 512, f.lnw = bw.n1w, f.lnb = bw.n1b, f.w = bw.in_w, f.b = bw.in_b, f.out = qg;
            f.m = (int)m, f.n = 512, f.qm0w = bw.qm0.w, f.qm0b = bw.qm0.b, f.qm2w = bw.qm2.w, f.qm2b = bw.qm2.b;
            f.base = base, f.rows = rows, f.pairs = bw.in_pairs;
            ln_linear512(f, kLnQass, s);
            return;
        }
        if (!normed) layer_norm(x, 512, bw.n1w, bw.n1b, norm, 512, m, 512, s);
        // Q, head-major [b, 8, rows, 64].
        OutMap qmap{64, kHeads, 0, (long long)rows * 64, rows, (long long)kHeads * rows * 64, 64};
        linear_pairs(norm, 512, m, 512, bw.in_pairs, bw.in_b, 512, qh, qmap);
        // QASSMax: q * base * (1 + tanh(MLP(q))) per head (reference.rs:417-428).
        QassRows qa{};
        qa.q = qh, qa.w0 = bw.qm0.w, qa.b0 = bw.qm0.b, qa.w2 = bw.qm2.w, qa.b2 = bw.qm2.b, qa.base = base;
        qa.out = qg, qa.m = m * kHeads, qa.rows = rows, qa.compute_units = cus;
        qass_rows(qa, s);
    }

    // K and V of an ICL block's n normalized rows, in two planes of head-major rows.
    void icl_kv_rows(const BlockW &bw, const float *norm, int n, float *out, long long plane) const {
        const OutMap map = OutMap::head_major(64, kHeads, n, plane);
        if (n > kFewRows) {
            PairW kv = bw.in_pairs;
            kv.pack += (size_t)512 * 512, kv.row_inv += 512;  // past the query rows
            linear_pairs(norm, 512, n, 512, kv, bw.in_b + 512, 1024, out, map);
        } else {
            linear_map(norm, 512, n, 512, bw.in_w + 512 * 512, bw.in_b + 512, 1024, out, map);
        }
    }

    // Query half of ICL block `blk` (cached_block with QASS, cpu.rs:2587-2850,
    // 3798-3853) for `b` estimators x `rows` query rows [b*rows, 512], against
    // K/V [b, 8, kv_rows, 64] (or the FP16 cache k16 / v16). normed: r.norm
    // already holds LN1(x) (the build's K/V projection read it); only taken
    // by queries too many for the fused LayerNorm form.
    void icl_queries(int blk, float *x, int b, int rows, const float *k, const float *v, int kv_rows,
                     const float *base, const IclBuffers &r, const unsigned short *k16 = nullptr,
                     const unsigned short *v16 = nullptr, const Icl8Block *c8 = nullptr, bool normed = false) const {
        const BlockW &bw = w.icl[blk];
        const long long m = (long long)b * rows;
        icl_query_rows(bw, x, b, rows, base, r.norm, r.qh, r.qg, normed, m <= kLnLinearRows);
        IclAttention at{};
        at.q = r.qg, at.q_pair_stride = (long long)rows * 64, at.k = k, at.v = v;
        at.kv_pair_stride = (long long)kv_rows * 64, at.o = r.att, at.ldo = 512;
        at.pairs = b * kHeads, at.q_rows = rows, at.kv_rows = kv_rows;
        at.partial = r.partial, at.partial_floats = r.partial_floats, at.compute_units = cus;
        at.k16 = k16, at.v16 = v16;
        if (c8) at.k8 = c8->k, at.v8 = c8->v, at.kscale = c8->kscale, at.vscale = c8->vscale;
        icl_attention(at, s);
        tail(bw, x, m, r.att, r.norm, r.hid);
    }
};

// ---- weights ----

struct Loader {
    irx_tensor_lookup lookup;
    void *user;
    int task;
    std::vector<float> host;
    struct Pending {
        const float **slot;
        size_t offset;
    };
    std::vector<Pending> pending;

    void take(const char *name, size_t len, const float **slot, bool zero_if_missing = false) {
        const float *data = nullptr;
        size_t got = 0;
        int missing = lookup(user, name, &data, &got);
        if (missing) {
            if (!zero_if_missing) fail(IRX_INVALID_ARGUMENT, std::string("model tensor '") + name + "' is missing");
            data = nullptr, got = len;
        }
        if (got != len)
            fail(IRX_INVALID_ARGUMENT, std::string("model tensor '") + name + "' has " + std::to_string(got) +
                                           " values; expected " + std::to_string(len));
        size_t offset = (host.size() + 63) / 64 * 64;
        host.resize(offset + len, 0.f);
        if (data) std::memcpy(host.data() + offset, data, len * sizeof(float));
        pending.push_back({slot, offset});
    }

    size_t offset_of(const float **slot) const {
        for (const Pending &p : pending)
            if (p.slot == slot) return p.offset;
        fail(IRX_INVALID_ARGUMENT, "model tensor not loaded");
    }

    // Out-projection and FFN weights of a 128-wide block in tail128's fragment order.
    void pack_tail(BlockW &b) {
        const size_t wo = offset_of(&b.out.w), w1 = offset_of(&b.l1.w), w2 = offset_of(&b.l2.w);
        const size_t b1 = offset_of(&b.l1.b), nw = offset_of(&b.n2w), nb = offset_of(&b.n2b);
        const size_t offset = (host.size() + 63) / 64 * 64;
        host.resize(offset + kTail128PackFloats, 0.f);
        const float *f = host.data();
        tail128_pack(f + wo, f + nw, f + nb, f + w1, f + b1, f + w2, host.data() + offset);
        pending.push_back({&b.tail_pack, offset});
    }

    // The in_proj rows [row0, row0 + outputs) of a 128-wide block in head128's fragment order.
    void pack_head(BlockW &b, int row0, int outputs) {
        const size_t w = offset_of(&b.in_w), nw = offset_of(&b.n1w), nb = offset_of(&b.n1b);
        const size_t offset = (host.size() + 63) / 64 * 64;
        host.resize(offset + head128_pack_floats(outputs), 0.f);
        const float *f = host.data();
        head128_pack(f + nw, f + nb, f + w + (size_t)row0 * 128, outputs, host.data() + offset);
        pending.push_back({&b.head_pack, offset});
        b.head_nb = outputs / 16, b.head_row0 = row0;
    }

    void block(BlockW &b, const std::string &prefix, int dim, bool qass) {
        const bool zb = task == IRX_TASK_REGRESSOR;  // bias-free LayerNorms (model.rs:273-280)
        b.dim = dim, b.qass = qass;
        auto t = [&](const char *suffix, size_t len, const float **slot, bool z = false) {
            take((prefix + suffix).c_str(), len, slot, z);
        };
        const size_t d = dim;
        t(".attn.in_proj_weight", 3 * d * d, &b.in_w);
        t(".attn.in_proj_bias", 3 * d, &b.in_b);
        t(".attn.out_proj.weight", d * d, &b.out.w);
        t(".attn.out_proj.bias", d, &b.out.b);
        t(".linear1.weight", 2 * d * d, &b.l1.w);
        t(".linear1.bias", 2 * d, &b.l1.b);
        t(".linear2.weight", 2 * d * d, &b.l2.w);
        t(".linear2.bias", d, &b.l2.b);
        t(".norm1.weight", d, &b.n1w);
        t(".norm1.bias", d, &b.n1b, zb);
        t(".norm2.weight", d, &b.n2w);
        t(".norm2.bias", d, &b.n2b, zb);
        if (dim == 128) pack_tail(b);
        if (qass) {
            const size_t hd = d / kHeads;
            t(".attn.ssmax_layer.query_mlp.0.weight", 64 * hd, &b.qm0.w);
            t(".attn.ssmax_layer.query_mlp.0.bias", 64, &b.qm0.b);
            t(".attn.ssmax_layer.query_mlp.2.weight", hd * 64, &b.qm2.w);
            t(".attn.ssmax_layer.query_mlp.2.bias", hd, &b.qm2.b);
        }
    }
};

void weights_load(irx_weights *W, irx_tensor_lookup lookup, void *user) {
    Loader L{lookup, user, W->task, {}, {}};
    const bool zb = W->task == IRX_TASK_REGRESSOR;
    const float *freqs = nullptr;
    L.take("col_embedder.in_linear.weight", 128 * 3, &W->in_w);
    L.take("col_embedder.in_linear.bias", 128, &W->in_b);
    for (int b = 0; b < kColumnBlocks; ++b) {
        std::string p = "col_embedder.tf_col.blocks." + std::to_string(b);
        L.take((p + ".ind_vectors").c_str(), 128 * 128, &W->ind[b]);
        L.block(W->col1[b], p + ".multihead_attn1", 128, true);
        L.block(W->col2[b], p + ".multihead_attn2", 128, false);
    }
    for (int b = 0; b < kRowBlocks; ++b)
        L.block(W->row[b], "row_interactor.tf_row.blocks." + std::to_string(b), 128, false);
    // Heads fused with LN1 for prediction: the column blocks' queries, the row
    // blocks' Q/K/V, the CLS block's K/V over every token.
    for (int b = 0; b < kColumnBlocks; ++b) L.pack_head(W->col2[b], 0, 128);
    for (int b = 0; b < kColumnBlocks; ++b) L.pack_head(W->col1[b], 128, 256);  // the build's attn1 K/V
    for (int b = 0; b < kRowBlocks; ++b) L.pack_head(W->row[b], b + 1 < kRowBlocks ? 0 : 128, b + 1 < kRowBlocks ? 384 : 256);
    L.take("row_interactor.cls_tokens", 4 * 128, &W->cls);
    L.take("row_interactor.out_ln.weight", 128, &W->out_ln_w);
    L.take("row_interactor.out_ln.bias", 128, &W->out_ln_b, zb);
    L.take("row_interactor.tf_row.rope.freqs", 8, &freqs);
    for (int b = 0; b < kIclBlocks; ++b)
        L.block(W->icl[b], "icl_predictor.tf_icl.blocks." + std::to_string(b), 512, true);
    L.take("icl_predictor.ln.weight", 512, &W->ln_w);
    L.take("icl_predictor.ln.bias", 512, &W->ln_b, zb);
    L.take("icl_predictor.decoder.0.weight", 1024 * 512, &W->dec0.w);
    L.take("icl_predictor.decoder.0.bias", 1024, &W->dec0.b);
    const size_t width = W->width;
    L.take("icl_predictor.decoder.2.weight", width * 1024, &W->dec2.w);
    L.take("icl_predictor.decoder.2.bias", width, &W->dec2.b);
    // y_encoder inputs: the classifier's 10 classes one-hot, the regressor's target (model.rs:777-836).
    W->classes = W->task == IRX_TASK_CLASSIFIER ? 10 : 1;
    L.take("col_embedder.y_encoder.weight", 128 * (size_t)W->classes, &W->ycol.w);
    L.take("col_embedder.y_encoder.bias", 128, &W->ycol.b);
    L.take("icl_predictor.y_encoder.weight", 512 * (size_t)W->classes, &W->yicl.w);
    L.take("icl_predictor.y_encoder.bias", 512, &W->yicl.b);
    W->arena.alloc(L.host.size() * sizeof(float));
    IRX_HIP(hipMemcpy(W->arena.p, L.host.data(), L.host.size() * sizeof(float), hipMemcpyHostToDevice));
    // The ICL blocks' and the decoder's first matrices as FP16 pairs too.
    constexpr size_t kBlockPairs = pair_pack_floats(1536, 512) + pair_pack_floats(512, 512) +
                                   pair_pack_floats(1024, 512) + pair_pack_floats(512, 1024);
    W->pairs.alloc((kIclBlocks * kBlockPairs + pair_pack_floats(1024, 512)) * sizeof(float));
    W->bytes = W->arena.bytes + W->pairs.bytes;
    float *next_pairs = W->pairs.f();
    auto pack = [&](const float **slot, int n, int k, const float **lnw = nullptr, const float **lnb = nullptr) {
        const size_t offset = L.offset_of(slot);
        const float *h = L.host.data();
        const PairW p = pair_pack(W->arena.f() + offset, n, k, lnw ? h + L.offset_of(lnw) : nullptr,
                                  lnb ? h + L.offset_of(lnb) : nullptr, next_pairs, nullptr);
        next_pairs += pair_pack_floats(n, k);
        return p;
    };
    for (BlockW &b : W->icl) {
        b.in_pairs = pack(&b.in_w, 1536, 512, &b.n1w, &b.n1b);
        b.out.pairs = pack(&b.out.w, 512, 512);
        b.l1.pairs = pack(&b.l1.w, 1024, 512, &b.n2w, &b.n2b);
        b.l2.pairs = pack(&b.l2.w, 512, 1024);
    }
    W->dec0.pairs = pack(&W->dec0.w, 1024, 512, &W->ln_w, &W->ln_b);
    IRX_HIP(hipDeviceSynchronize());
    for (auto &pend : L.pending) {
        if (pend.slot == &freqs) continue;
        *pend.slot = W->arena.f() + pend.offset;
    }
    // The RoPE frequencies stay on the host: the tables are built from them.
    for (auto &pend : L.pending)
        if (pend.slot == &freqs) W->freqs_host.assign(L.host.begin() + pend.offset, L.host.begin() + pend.offset + 8);
}

// ---- build ----

struct BuildPlan {
    int col_chunk;   // columns per chunk of the column stage
    int row_run;     // rows per run of the row stage
    size_t ws_bytes; // workspace
    size_t keep_bytes;
};

// Partial outputs of the inducing points' attention over `cols` columns when
// its keys are split over workgroups: at most ceil(512 / units) splits of
// units = cols x heads (sequence, head) items, 17 floats per query.
size_t inducing_partial_floats(int cols) {
    return (size_t)(512 + (long long)kHeads * cols) * kInducing * 17;
}

size_t column_chunk_floats(int cols, long long n) {
    long long cn = (long long)cols * n;
    // state is per estimator; chunk temporaries: norm, q, att (128) + kv, hid (256)
    return (size_t)(cn * (128 * 3 + 256 * 2) + (long long)cols * 128 * (128 * 4 + 256)) +
           inducing_partial_floats(cols);
}

size_t row_run_floats(long long seqs, int len) {
    long long m = seqs * len, c = seqs * kReserved;
    return (size_t)(m * (128 * 3 + 384 + 256) + c * (128 * 4 + 256));
}

BuildPlan plan_build(const irx_shape &sh, size_t budget, int cus, int precision = IRX_PRECISION_FP32) {
    const long long n = sh.rows, h = sh.features, b = sh.ensembles;
    const int len = (int)h + kReserved;
    const bool f16 = precision != IRX_PRECISION_FP32;
    BuildPlan p{};
    // HALF keeps the FP16 cache it builds and adds the FP8 blocks made from it
    // (through one FP16 logical copy).
    p.keep_bytes = (size_t)kColumnBlocks * 2 * b * (h + 4) * kColumnCache * 4 +
                   (f16 ? (size_t)kIclBlocks * 2 * icl16_plane(b * kHeads, n) * 2
                        : (size_t)kIclBlocks * 2 * b * kHeads * n * 64 * 4) +
                   (precision == IRX_PRECISION_HALF
                        ? (size_t)2 * b * kHeads * n * 64 * 2 + kIclBlocks * icl8_block_bytes(b * kHeads, n)
                        : 0);
    size_t cap = std::min<size_t>(budget / 4, (size_t)24 << 30);
    int chunk = (int)h;
    while (chunk > 1 && column_chunk_floats(chunk, n) * 4 > cap) chunk = (chunk + 1) / 2;
    p.col_chunk = chunk;
    int run = (int)std::min<long long>(n, 16384);
    while (run > 64 && row_run_floats(run, len) * 4 > cap) run /= 2;
    p.row_run = run;
    // x, label embeddings and targets of one estimator; inducing queries, base scales, RoPE tables.
    size_t fixed = ((size_t)n * h + n * 128 + n * 512 + n + 6 * 128 * 128 + 12 * 512 + 2 * len * 16) * 4;
    size_t state = (size_t)h * n * 128 * 4;  // all features' column states of one estimator
    size_t icl = ((size_t)n * 512 * 6 + n * 1024) * 4 +
                 icl_attention_partial_floats(kHeads, (int)n, (int)n, cus, f16) * 4 +
                 (f16 ? (size_t)2 * kHeads * n * 64 * 4 : 0);  // FP32 K/V of a block before packing
    p.ws_bytes = fixed + state + column_chunk_floats(chunk, n) * 4 + row_run_floats(run, len) * 4 + icl +
                 (size_t)64 * 256 * 40;
    return p;
}

bool shape_ok(const irx_shape *s) {
    return s && s->ensembles > 0 && s->features > 0 && s->rows > 0 && s->features < (1 << 20) &&
           s->rows < (size_t)(1u << 30) && s->ensembles < 4096;
}

// Whether any of `rows` rows of x [rows, h] holds a grouped all-missing
// triple, scanned by host threads over row ranges (the reference scans with
// par_chunks; 8 x 200,000 rows of 500 features is 800M triples).
bool has_missing_marker(const float *x, long long rows, int h) {
    const long long work = rows * h;
    const unsigned hw = std::max(1u, std::thread::hardware_concurrency());
    const int threads = (int)std::min<long long>(std::min(16u, hw), std::max(1LL, work >> 22));
    std::atomic<bool> found{false};
    auto scan = [&](long long r0, long long r1) {
        for (long long r = r0; r < r1 && !found.load(std::memory_order_relaxed); ++r) {
            const float *row = x + r * h;
            for (int f = 0; f < h; ++f)
                if (row[(f + 1) % h] == -100.0f && row[(f + 2) % h] == -100.0f && row[(f + 4) % h] == -100.0f) {
                    found.store(true, std::memory_order_relaxed);
                    break;
                }
        }
    };
    if (threads <= 1) {
        scan(0, rows);
        return found.load();
    }
    // Threads already started are joined even when starting another throws
    // (a thread left joinable would terminate the process); rows no thread
    // took are scanned here.
    std::vector<std::thread> pool;
    struct Joiner {
        std::vector<std::thread> &p;
        ~Joiner() {
            for (auto &th : p)
                if (th.joinable()) th.join();
        }
    } joiner{pool};
    const long long per = (rows + threads - 1) / threads;
    long long started = 0;
    for (int t = 0; t < threads; ++t) {
        const long long r0 = t * per, r1 = std::min(rows, r0 + per);
        if (r0 >= r1) break;
        try {
            pool.emplace_back(scan, r0, r1);
        } catch (const std::system_error &) {
            break;
        }
        started = r1;
    }
    if (started < rows) scan(started, rows);
    for (auto &th : pool) th.join();
    return found.load();
}

int report(irx_progress_fn fn, void *user, int stage, size_t done, size_t total) {
    if (fn && fn(user, stage, done, total) != 0) fail(IRX_INTERRUPTED, "interrupted by the progress hook");
    return 0;
}

void build_impl(irx_weights *W, const irx_build_inputs *in, irx_build_outputs *out, irx_built_cache **keep,
                int precision) {
    // SPLIT and HALF build alike on the FP16 cache (the reference reads HALF's
    // FP16 cache at Split precision during its build, cuda/build.rs:477-511).
    const bool f16 = precision != IRX_PRECISION_FP32;
    const irx_shape sh = in->shape;
    if (!shape_ok(&sh)) fail(IRX_INVALID_ARGUMENT, "build shape must be nonempty");
    if (sh.rows < 64) fail(IRX_DOES_NOT_FIT, "the device builds contexts of at least 64 training rows");
    // Label embeddings come from the host (column_labels and icl_labels, as the
    // reference's BuildInputs carry them) or, when both are null, from the
    // targets through the resident y_encoder weights.
    const bool device_labels = !in->column_labels && !in->icl_labels;
    if (!in->x || (device_labels ? !in->targets : (!in->column_labels || !in->icl_labels)) || !in->rope_frequencies ||
        !in->cls_tokens)
        fail(IRX_INVALID_ARGUMENT, "build inputs are missing");
    for (int i = 0; i < kColumnBlocks; ++i)
        if (!in->inducing_queries[i]) fail(IRX_INVALID_ARGUMENT, "inducing queries are missing");
    for (int i = 0; i < kIclBlocks; ++i)
        if (!in->base_scales[i]) fail(IRX_INVALID_ARGUMENT, "base scales are missing");
    const int B = (int)sh.ensembles, H = (int)sh.features, N = (int)sh.rows, L = H + kReserved;
    // Targets the device embeds are checked as the reference checks labels
    // and targets (validate_labels / validate_targets, cpu.rs:1684-1688,
    // 4717-4740): a classifier's are class indices 0..9, a regressor's finite.
    if (device_labels) {
        const bool clf = W->task == IRX_TASK_CLASSIFIER;
        const float *t = in->targets;
        for (size_t i = 0, n = (size_t)B * N; i < n; ++i) {
            const float v = t[i];
            if (clf ? !(v >= 0.f && v <= 9.f && v == std::floor(v)) : !std::isfinite(v))
                fail(IRX_INVALID_ARGUMENT, clf ? "classifier targets must be integers in 0..=9"
                                               : "regression targets must be finite");
        }
    }
    // A grouped all-missing triple is the CPU path's (has_missing_marker,
    // cpu.rs:4072-4084): the caller routes such a context to its CPU build.
    if (has_missing_marker(in->x, (long long)B * N, H))
        fail(IRX_UNSUPPORTED, "a grouped feature triple is the all-missing marker");
    set_device(W->device);
    irx_device *dev = W->device;
    const int cus = dev->compute_units;
    // The device's kept workspace is memory this build can use beside the
    // caller's budget (free memory), when no other build holds it.
    size_t kept = 0;
    {
        std::lock_guard<std::mutex> lock(dev->build_mu);
        if (!dev->build_ws_lent) kept = dev->build_ws.bytes;
    }
    const size_t budget = in->budget + kept;
    BuildPlan plan = plan_build(sh, budget, cus, precision);
    if (plan.ws_bytes + plan.keep_bytes > budget / 10 * 9)
        fail(IRX_DOES_NOT_FIT, "the context does not fit the device");

    hipStream_t s = take_stream(W->device);
    struct StreamGuard {
        irx_device *d;
        hipStream_t s;
        ~StreamGuard() { return_stream(d, s); }
    } guard{W->device, s};

    auto cache = new irx_built_cache();
    struct CacheGuard {
        irx_built_cache *&c;
        ~CacheGuard() { delete c; }
    } cache_guard{cache};
    cache->device = W->device;
    cache->shape = sh;
    cache->precision = precision;
    const long long col_plane = (long long)B * L * kColumnCache;
    const long long icl_plane = (long long)B * kHeads * N * 64;
    const size_t plane16 = icl16_plane((long long)B * kHeads, N), est16 = icl16_plane(kHeads, N);
    for (int i = 0; i < kColumnBlocks; ++i) {
        cache->column[i].alloc(2 * col_plane * 4);
        fill_zero(cache->column[i].f(), 2 * col_plane, s);  // reserved CLS streams stay zero
    }
    for (int i = 0; i < kIclBlocks; ++i) cache->icl[i].alloc(f16 ? 2 * plane16 * 2 : 2 * icl_plane * 4);

    // The workspace: the device's kept one (grown when too small), else one of
    // this build's own. The lease gives it back once this build's streams have
    // finished with it (the side upload stream is synchronized first: it is
    // declared later, so destroyed earlier).
    struct WsLease {
        irx_device *d;
        hipStream_t s;
        bool held = false;
        ~WsLease() {
            if (!held) return;
            (void)hipStreamSynchronize(s);
            std::lock_guard<std::mutex> lock(d->build_mu);
            d->build_ws_lent = false;
            if (d->build_ws.bytes > d->memory_bytes / 8) d->build_ws.release();
        }
    } lease{dev, s};
    Arena ws;
    {
        std::lock_guard<std::mutex> lock(dev->build_mu);
        if (!dev->build_ws_lent) {
            if (dev->build_ws.bytes < plan.ws_bytes) {
                dev->build_ws.release();
                dev->build_ws.alloc(plan.ws_bytes);
            }
            dev->build_ws_lent = true;
            lease.held = true;
            ws.lent = dev->build_ws.p, ws.lent_bytes = dev->build_ws.bytes;
        }
    }
    if (!lease.held) ws.buf.alloc(plan.ws_bytes);
    // Each estimator's ICL labels go up on a side stream while its column
    // stage runs (a pageable copy holds the host until it is done); events
    // order the copy after the previous estimator's read and before the add.
    struct SideUpload {
        hipStream_t s = nullptr;
        hipEvent_t ready = nullptr, free = nullptr;
        ~SideUpload() {
            if (s) (void)hipStreamSynchronize(s);
            if (ready) (void)hipEventDestroy(ready);
            if (free) (void)hipEventDestroy(free);
        }
    } side;
    side.s = upload_stream(W->device);
    IRX_HIP(hipEventCreateWithFlags(&side.ready, hipEventDisableTiming));
    IRX_HIP(hipEventCreateWithFlags(&side.free, hipEventDisableTiming));
    Stages st{*W, s, cus};
    // Inputs shared by every estimator.
    float *d_ind_q = ws.take(3 * 128 * 128);
    float *d_base = ws.take(12 * 512);
    std::vector<float> cos_t, sin_t;
    rope_tables(W->freqs_host.data(), L, cos_t, sin_t);
    float *d_cos = ws.take(L * 16), *d_sin = ws.take(L * 16);
    for (int i = 0; i < 3; ++i) upload(d_ind_q + i * 128 * 128, in->inducing_queries[i], 128 * 128 * 4, s);
    for (int i = 0; i < 12; ++i) upload(d_base + i * 512, in->base_scales[i], 512 * 4, s);
    upload(d_cos, cos_t.data(), cos_t.size() * 4, s);
    upload(d_sin, sin_t.data(), sin_t.size() * 4, s);
    float *d_x = ws.take((size_t)N * H), *d_ylab = ws.take((size_t)N * 128), *d_yicl = ws.take((size_t)N * 512);
    float *d_targets = device_labels ? ws.take((size_t)N) : nullptr;
    float *d_state = ws.take((size_t)H * N * 128);
    // Cached values that are not finite (in FP16 for the FP16 cache) are counted here.
    unsigned *counter = reinterpret_cast<unsigned *>(ws.take(64));
    IRX_HIP(hipMemsetAsync(counter, 0, 4, s));
    const size_t mark = ws.used;

    report(in->progress, in->progress_user, IRX_STAGE_BUILD, 0, B);
    for (int e = 0; e < B; ++e) {
        ws.used = mark;
        upload(d_x, in->x + (size_t)e * N * H, (size_t)N * H * 4, s);
        if (device_labels) {
            const bool clf = W->task == IRX_TASK_CLASSIFIER;
            upload(d_targets, in->targets + (size_t)e * N, (size_t)N * 4, s);
            label_embeddings(d_targets, N, W->ycol.w, W->ycol.b, W->classes, 128, clf, d_ylab, s);
            label_embeddings(d_targets, N, W->yicl.w, W->yicl.b, W->classes, 512, clf, d_yicl, s);
        } else {
            upload(d_ylab, in->column_labels + (size_t)e * N * 128, (size_t)N * 128 * 4, s);
        }
        // Column stage, chunk by chunk of features (column_stream + isab, cpu.rs:1132-1207).
        {
            const size_t cmark = ws.used;
            const int C = plan.col_chunk;
            const long long cn = (long long)C * N;
            float *norm = ws.take(cn * 128), *q = ws.take(cn * 128), *att = ws.take(cn * 128);
            float *kv = ws.take(cn * 256), *hid = ws.take(cn * 256);
            float *hidden = ws.take((size_t)C * 128 * 128), *hnorm = ws.take((size_t)C * 128 * 128);
            float *hatt = ws.take((size_t)C * 128 * 128), *hhid = ws.take((size_t)C * 128 * 256);
            const size_t spart_floats = inducing_partial_floats(C);
            float *spart = ws.take(spart_floats);
            column_input(d_x, 0, 1, N, H, W->in_w, W->in_b, d_ylab, d_state, nullptr, s);
            for (int f0 = 0; f0 < H; f0 += C) {
                const int cols = std::min(C, H - f0);
                const long long m = (long long)cols * N;
                float *state = d_state + (size_t)f0 * N * 128;
                for (int blk = 0; blk < kColumnBlocks; ++blk) {
                    // multihead_attn1: the inducing points attend to the column's N rows, QASS'd queries.
                    const BlockW &b1 = W->col1[blk];
                    st.head(b1, state, m, norm, kv, 256);  // LN1 + the K/V rows of in_proj
                    SmallAttention a{};
                    a.q = d_ind_q + blk * 128 * 128, a.q_seq = 0, a.q_group = 0, a.q_row = 128, a.q_head = 16;
                    a.k = kv, a.v = kv + 128, a.k_seq = a.v_seq = (long long)N * 256, a.k_group = a.v_group = 0;
                    a.k_row = a.v_row = 256, a.k_head = a.v_head = 16;
                    a.o = hatt, a.o_seq = 128 * 128, a.o_group = 0, a.o_row = 128, a.o_head = 16;
                    a.group = cols, a.seqs = cols, a.heads = kHeads, a.q_rows = kInducing, a.kv_rows = N;
                    a.scale = 0.25f;
                    a.partial = spart, a.partial_floats = (long long)spart_floats;
                    small_attention(a, s);
                    repeat_rows(W->ind[blk], 128 * 128, cols, hidden, s);
                    st.tail(b1, hidden, (long long)cols * 128, hatt, hnorm, hhid);
                    // multihead_attn2 keys and values from the inducing state, straight into the cache.
                    const BlockW &b2 = W->col2[blk];
                    layer_norm(hidden, 128, b2.n1w, b2.n1b, hnorm, 128, (long long)cols * 128, 128, s);
                    float *kc = cache->column[blk].f() + ((long long)e * L + kReserved + f0) * kColumnCache;
                    OutMap cmap{16, kHeads, col_plane, 128 * 16, 128, kColumnCache, 16};
                    st.linear_map(hnorm, 128, (long long)cols * 128, 128, b2.in_w + 128 * 128, b2.in_b + 128, 256,
                                  kc, cmap);
                    st.column_attend(blk, state, cols, N, kc, kc + col_plane, cols, 0, norm, q, att, hid);
                }
            }
            ws.used = cmark;
        }
        if (!device_labels) {
            if (e > 0) IRX_HIP(hipStreamWaitEvent(side.s, side.free, 0));
            upload(d_yicl, in->icl_labels + (size_t)e * N * 512, (size_t)N * 512 * 4, side.s);
            IRX_HIP(hipEventRecord(side.ready, side.s));
        }
        // Row stage in runs, into the ICL row states.
        float *rows = ws.take((size_t)N * 512);
        {
            const size_t rmark = ws.used;
            const int R = plan.row_run;
            Stages::RowBuffers rb = Stages::row_buffers(ws, R, L);
            float *stage = ws.take((size_t)H * R * 128);
            for (int r0 = 0; r0 < N; r0 += R) {
                const int len = std::min(R, N - r0);
                // Gather the run's column states into [H, len, 128].
                IRX_HIP(hipMemcpy2DAsync(stage, (size_t)len * 128 * 4, d_state + (size_t)r0 * 128, (size_t)N * 128 * 4,
                                         (size_t)len * 128 * 4, H, hipMemcpyDeviceToDevice, s));
                st.row_stage(stage, 1, len, H, rows + (size_t)r0 * 512, d_cos, d_sin, rb);
            }
            ws.used = rmark;
        }
        if (!device_labels) IRX_HIP(hipStreamWaitEvent(s, side.ready, 0));
        add_inplace(rows, d_yicl, (long long)N * 512, s);
        if (!device_labels) IRX_HIP(hipEventRecord(side.free, s));
        // ICL stage: each block's K/V from the training rows, then their queries.
        {
            Stages::IclBuffers ib = Stages::icl_buffers(ws, N, 1, N, N, cus, f16);
            float *kv32 = f16 ? ws.take((size_t)2 * kHeads * N * 64) : nullptr;
            for (int blk = 0; blk < kIclBlocks; ++blk) {
                const BlockW &bw = W->icl[blk];
                layer_norm(rows, 512, bw.n1w, bw.n1b, ib.norm, 512, N, 512, s);
                if (!f16) {
                    float *kc = cache->icl[blk].f() + (long long)e * kHeads * N * 64;
                    st.icl_kv_rows(bw, ib.norm, N, kc, icl_plane);
                    // The last block's row states are never read: only its K/V are kept.
                    if (blk + 1 < kIclBlocks)
                        st.icl_queries(blk, rows, 1, N, kc, kc + icl_plane, N, d_base + blk * 512, ib, nullptr,
                                       nullptr, nullptr, true);
                } else {
                    // FP32 K/V of this estimator, then packed into its part of the FP16 cache.
                    const long long p32 = (long long)kHeads * N * 64;
                    st.icl_kv_rows(bw, ib.norm, N, kv32, p32);
                    unsigned short *k16 = static_cast<unsigned short *>(cache->icl[blk].p) + e * est16;
                    unsigned short *v16 = k16 + plane16;
                    pack_icl16(kv32, kv32 + p32, false, N, kHeads, k16, v16, counter, s);
                    if (blk + 1 < kIclBlocks)
                        st.icl_queries(blk, rows, 1, N, nullptr, nullptr, N, d_base + blk * 512, ib, k16, v16,
                                       nullptr, true);
                }
            }
        }
        IRX_HIP(hipStreamSynchronize(s));
        report(in->progress, in->progress_user, IRX_STAGE_BUILD, e + 1, B);
    }
    // Non-finite cached values are an error (cuda/build.rs:340-350, 595-622).
    {
        for (int i = 0; i < kColumnBlocks; ++i) count_nonfinite(cache->column[i].f(), 2 * col_plane, counter, s);
        if (!f16)
            for (int i = 0; i < kIclBlocks; ++i) count_nonfinite(cache->icl[i].f(), 2 * icl_plane, counter, s);
        unsigned bad = 0;
        download(&bad, counter, 4, s);
        IRX_HIP(hipStreamSynchronize(s));
        if (bad) fail(IRX_NOT_FINITE, "a cached key or value is not finite");
    }
    if (out) {
        for (int i = 0; i < kColumnBlocks; ++i) {
            // Copy feature streams only; the caller's reserved streams stay as they are.
            for (int e = 0; e < B; ++e)
                for (int part = 0; part < 2; ++part) {
                    float *dst = part ? out->column_values[i] : out->column_keys[i];
                    if (!dst) continue;
                    const size_t off = ((size_t)e * L + kReserved) * kColumnCache;
                    download(dst + off, cache->column[i].f() + part * col_plane + off, (size_t)H * kColumnCache * 4, s);
                }
        }
        DevBuf logical(f16 && precision != IRX_PRECISION_HALF ? (size_t)2 * icl_plane * 2 : 0);
        for (int i = 0; i < kIclBlocks; ++i) {
            if (precision == IRX_PRECISION_HALF) {
                // Downloaded below, with the conversion to FP8.
            } else if (!f16) {
                if (out->icl_keys[i]) download(out->icl_keys[i], cache->icl[i].f(), icl_plane * 4, s);
                if (out->icl_values[i]) download(out->icl_values[i], cache->icl[i].f() + icl_plane, icl_plane * 4, s);
            } else if (out->icl_keys[i] || out->icl_values[i]) {
                // FP16 bits in the logical layout [B, 8, N, 64].
                const unsigned short *k16 = static_cast<const unsigned short *>(cache->icl[i].p);
                unsigned short *lk = static_cast<unsigned short *>(logical.p), *lv = lk + icl_plane;
                unpack_icl16(k16, k16 + plane16, N, B * kHeads, lk, lv, s);
                if (out->icl_keys[i]) download(out->icl_keys[i], lk, icl_plane * 2, s);
                if (out->icl_values[i]) download(out->icl_values[i], lv, icl_plane * 2, s);
                IRX_HIP(hipStreamSynchronize(s));
            }
        }
        IRX_HIP(hipStreamSynchronize(s));
    }
    if (precision == IRX_PRECISION_HALF) {
        // Each block's FP16 cache -> logical FP16 (downloaded when asked) ->
        // the FP8 cache the predictor reads (encode_fp8, cuda/build.rs:479-495).
        // The FP16 cache stays beside it for context reads (exports).
        DevBuf logical((size_t)2 * icl_plane * 2);
        unsigned short *lk = static_cast<unsigned short *>(logical.p), *lv = lk + icl_plane;
        for (int i = 0; i < kIclBlocks; ++i) {
            const unsigned short *k16 = static_cast<const unsigned short *>(cache->icl[i].p);
            unpack_icl16(k16, k16 + plane16, N, B * kHeads, lk, lv, s);
            if (out && out->icl_keys[i]) download(out->icl_keys[i], lk, icl_plane * 2, s);
            if (out && out->icl_values[i]) download(out->icl_values[i], lv, icl_plane * 2, s);
            DevBuf fp8(icl8_block_bytes((long long)B * kHeads, N));
            encode_icl8(lk, lv, N, B * kHeads, fp8.p, counter, s);
            IRX_HIP(hipStreamSynchronize(s));
            cache->icl16[i] = std::move(cache->icl[i]);
            cache->icl[i] = std::move(fp8);
        }
    }
    if (keep) {
        *keep = cache;
        cache = nullptr;
    }
}

// ---- predictor ----

// Buffers of one prediction pass of up to `R` rows per estimator. The same
// function sizes the workspace (counting arena) and carves it, so the two
// always agree; a shorter last pass uses a prefix of each buffer.
struct PassBuffers {
    // A graph-replayed pass reads its rows from xin [B, R, H], writes logits
    // [B, R, width] to lout and missing-row flags [R] to fin (fixed addresses).
    float *xin, *lout;
    uint8_t *fin;
    float *state, *norm, *q, *att, *hid, *rows;
    Stages::RowBuffers rb;
    Stages::IclBuffers ib;
};

PassBuffers pass_layout(Arena &a, const irx_shape &sh, size_t R, int cus, bool f16) {
    const long long B = sh.ensembles, H = sh.features, cr = B * H * (long long)R;
    PassBuffers p{};
    p.xin = a.take(B * H * (long long)R), p.lout = a.take(B * (long long)R * (long long)sh.outputs);
    p.fin = reinterpret_cast<uint8_t *>(a.take((R + 3) / 4));
    p.state = a.take(cr * 128), p.norm = a.take(cr * 128), p.q = a.take(cr * 128), p.att = a.take(cr * 128);
    p.hid = a.take(cr * 256);
    p.rb = Stages::row_buffers(a, B * (long long)R, (int)H + kReserved);
    p.rows = a.take(B * R * 512);
    p.ib = Stages::icl_buffers(a, B * (long long)R, (int)B, (int)R, (int)sh.rows, cus, f16);
    // A shorter pass may split the keys further; size the partials for the worst pass.
    size_t worst = 0;
    for (size_t rows = 32; rows <= R; rows += 32) {
        worst = std::max(worst, icl_attention_partial_floats((int)B * kHeads, (int)rows, (int)sh.rows, cus, f16));
    }
    if (worst > p.ib.partial_floats) {
        p.ib.partial = a.take(worst);
        p.ib.partial_floats = worst;
    }
    return p;
}

size_t predict_ws_floats(const irx_shape &sh, size_t R, int cus, bool f16) {
    Arena count;
    count.counting = true;
    pass_layout(count, sh, R, cus, f16);
    return count.used / 4;
}

// The kernels of one pass over the slot's workspace `pb`: R rows of x [B, ., H]
// (row stride x_stride between estimators) into logits [B, ., width] (Q rows
// per estimator), flags [R] (or null) set for rows holding the marker.
void issue_pass(irx_predictor *P, int slot, const PassBuffers &pb, const float *x, long long x_stride, int R,
                float *logits, int Q, uint8_t *flags) {
    const irx_weights &W = *P->weights;
    const irx_shape &sh = P->shape;
    const int B = (int)sh.ensembles, H = (int)sh.features, N = (int)sh.rows, L = H + kReserved;
    const int width = (int)sh.outputs;
    hipStream_t s = P->lane(slot);
    Stages st{W, s, W.device->compute_units};
    const bool f16 = P->precision != IRX_PRECISION_FP32;
    float *state = pb.state, *norm = pb.norm, *q = pb.q, *att = pb.att, *hid = pb.hid, *rows = pb.rows;
    const Stages::RowBuffers &rb = pb.rb;
    Stages::IclBuffers ib = pb.ib;

    column_input(x, x_stride, B, R, H, W.in_w, W.in_b, nullptr, state, flags, s);
    const long long col_plane = (long long)B * L * kColumnCache;
    for (int blk = 0; blk < kColumnBlocks; ++blk) {
        const float *kc = P->column[blk].f() + kReserved * kColumnCache;
        st.column_attend(blk, state, B * H, R, kc, kc + col_plane, H, (long long)L * kColumnCache, norm, q, att,
                         hid);
    }
    st.row_stage(state, B, R, H, rows, P->rope_cos.f(), P->rope_sin.f(), rb);
    const long long icl_plane = (long long)B * kHeads * N * 64;
    const size_t plane16 = icl16_plane((long long)B * kHeads, N);
    for (int blk = 0; blk < kIclBlocks; ++blk) {
        if (!f16) {
            const float *kc = P->icl[blk].f();
            st.icl_queries(blk, rows, B, R, kc, kc + icl_plane, N, P->base_scales.f() + blk * 512, ib);
        } else if (P->precision == IRX_PRECISION_HALF) {
            const Icl8Block c8 = icl8_block(P->icl[blk].p, (long long)B * kHeads, N);
            st.icl_queries(blk, rows, B, R, nullptr, nullptr, N, P->base_scales.f() + blk * 512, ib, nullptr,
                           nullptr, &c8);
        } else {
            const unsigned short *k16 = static_cast<const unsigned short *>(P->icl[blk].p);
            st.icl_queries(blk, rows, B, R, nullptr, nullptr, N, P->base_scales.f() + blk * 512, ib, k16,
                           k16 + plane16);
        }
    }
    // Decoder (cached_icl_decoder, cpu.rs:2543-2580) into logits [B, Q, width].
    st.ln_gelu512(rows, (long long)B * R, W.ln_w, W.ln_b, W.dec0, 1024, ib.hid);
    OutMap lmap{width, 1, 0, 0, R, (long long)Q * width, width};
    st.linear_map(ib.hid, 1024, (long long)B * R, 1024, W.dec2.w, W.dec2.b, width, logits, lmap);
}

// One pass of R query rows starting at row q0 of x [B, Q, H] (row stride
// x_stride between estimators) into logits [B, Q, width]; rows holding the
// all-missing marker set d_flags[q0 + r] (device, [Q], or null).
//
// A pass of more than 32 rows computes a multiple of 32 rows, Rp = R rounded
// up: its rows are staged in the slot's workspace (xin) with zero rows after
// them, and only the first R rows of its logits and flags are copied out.
// Passes of up to 32 rows (the HBM-bound decode passes of serving) compute
// exactly R rows. Every pass length thus maps onto one of 31 + pass_rows / 32
// shapes, launched the same way whether replayed or not (the split plan of the
// attention follows the row count, so a row's logits are the same either
// way). Unless kernel timing is on (or graphs are off), the pass replays a HIP
// graph captured over the slot's workspace for (slot, Rp). A pass with
// Rp == R that launches its kernels one by one reads x in place.
void predict_pass(irx_predictor *P, int slot, const float *d_x, long long x_stride, int q0, int R, float *d_logits,
                  int Q, uint8_t *d_flags) {
    const irx_shape &sh = P->shape;
    const int B = (int)sh.ensembles, H = (int)sh.features, width = (int)sh.outputs;
    const int Rp = R <= 32 ? R : (R + 31) / 32 * 32;
    hipStream_t s = P->lane(slot);
    Arena &ws = P->ws[slot];
    ws.used = 0;
    const PassBuffers pb = pass_layout(ws, sh, P->ws_rows, P->weights->device->compute_units,
                                       P->precision != IRX_PRECISION_FP32);
    const bool replay = P->use_graphs && !g_profiling.load(std::memory_order_relaxed);
    if (!replay && Rp == R) {
        issue_pass(P, slot, pb, d_x + (size_t)q0 * H, x_stride, R, d_logits + (size_t)q0 * width, Q,
                   d_flags ? d_flags + q0 : nullptr);
        return;
    }
    IRX_HIP(hipMemcpy2DAsync(pb.xin, (size_t)Rp * H * 4, d_x + (size_t)q0 * H, (size_t)x_stride * 4, (size_t)R * H * 4,
                             B, hipMemcpyDeviceToDevice, s));
    if (Rp != R)
        IRX_HIP(hipMemset2DAsync(pb.xin + (size_t)R * H, (size_t)Rp * H * 4, 0, (size_t)(Rp - R) * H * 4, B, s));
    if (!replay) {
        fill_zero(reinterpret_cast<float *>(pb.fin), (Rp + 3) / 4, s);
        issue_pass(P, slot, pb, pb.xin, (long long)Rp * H, Rp, pb.lout, Rp, pb.fin);
    } else {
        hipGraphExec_t exec = nullptr;
        for (const auto &g : P->graphs)
            if (g.slot == slot && g.rows == Rp) exec = g.exec;
        if (!exec) {
            // At most streams x pass_rows / 32 shapes exist; past the cap the
            // oldest graph goes, once the lane it was launched on is idle
            // (earlier passes of this call may still be running it).
            if (P->graphs.size() >= kMaxPassGraphs) {
                const PassGraphEntry victim = P->graphs.front();
                IRX_HIP(hipStreamSynchronize(P->lane(victim.slot)));
                (void)hipGraphExecDestroy(victim.exec);
                P->graphs.erase(P->graphs.begin());
            }
            hipGraph_t graph = nullptr;
            IRX_HIP(hipStreamBeginCapture(s, hipStreamCaptureModeThreadLocal));
            try {
                // Flags start from zero on every replay: a fill kernel, not a memset node.
                fill_zero(reinterpret_cast<float *>(pb.fin), (Rp + 3) / 4, s);
                issue_pass(P, slot, pb, pb.xin, (long long)Rp * H, Rp, pb.lout, Rp, pb.fin);
            } catch (...) {
                (void)hipStreamEndCapture(s, &graph);
                if (graph) (void)hipGraphDestroy(graph);
                throw;
            }
            IRX_HIP(hipStreamEndCapture(s, &graph));
            const hipError_t e = hipGraphInstantiate(&exec, graph, nullptr, nullptr, 0);
            (void)hipGraphDestroy(graph);
            IRX_HIP(e);
            P->graphs.push_back({slot, Rp, exec});
        }
        IRX_HIP(hipGraphLaunch(exec, s));
    }
    IRX_HIP(hipMemcpy2DAsync(d_logits + (size_t)q0 * width, (size_t)Q * width * 4, pb.lout, (size_t)Rp * width * 4,
                             (size_t)R * width * 4, B, hipMemcpyDeviceToDevice, s));
    if (d_flags) IRX_HIP(hipMemcpyAsync(d_flags + q0, pb.fin, R, hipMemcpyDeviceToDevice, s));
}

void ensure_workspace(irx_predictor *P) {
    for (int i = 1; i < P->streams; ++i)
        if (!P->side[i - 1]) P->side[i - 1] = take_lane(P->weights->device);
    bool ready = P->ws_rows == P->pass_rows;
    for (int i = 0; i < P->streams; ++i) ready = ready && P->ws[i].buf.p;
    if (ready) return;
    for (int i = 0; i < kMaxPassStreams; ++i)
        if (P->lane(i)) IRX_HIP(hipStreamSynchronize(P->lane(i)));
    P->drop_graphs();  // they hold the old workspaces' addresses
    size_t floats = predict_ws_floats(P->shape, P->pass_rows, P->weights->device->compute_units,
                                      P->precision != IRX_PRECISION_FP32);
    // Workspaces of streams in use, at the current pass size; the others are released.
    for (int i = 0; i < kMaxPassStreams; ++i) {
        if (i < P->streams) {
            if (!P->ws[i].buf.p || P->ws_rows != P->pass_rows) P->ws[i].buf.alloc(floats * 4);
        } else {
            P->ws[i].buf = DevBuf();
        }
    }
    P->ws_rows = P->pass_rows;
}

// The pass workspaces beside the caches within `budget` (bytes the predictor
// may use, caches included): when those of every stream at pass_rows do not
// fit, or a hipMalloc runs out, one stream, then halved passes (multiples of
// 32), as Predictor::predict halves its run rows on out-of-memory
// (predictor.rs:248-258); IRX_DOES_NOT_FIT below one 32-row pass.
void fit_workspace(irx_predictor *P, size_t cache_bytes, size_t budget) {
    const bool f16 = P->precision != IRX_PRECISION_FP32;
    const int cus = P->weights->device->compute_units;
    for (;;) {
        const size_t ws = (size_t)P->streams * predict_ws_floats(P->shape, P->pass_rows, cus, f16) * 4;
        if (cache_bytes + ws <= budget / 10 * 9) {
            try {
                ensure_workspace(P);
                return;
            } catch (const Failure &f) {
                if (f.status != IRX_OUT_OF_MEMORY) throw;
            }
        }
        if (P->streams > 1)
            P->streams = 1;
        else if (P->pass_rows > 32)
            P->pass_rows = std::max<size_t>(32, P->pass_rows / 64 * 32);
        else
            fail(IRX_DOES_NOT_FIT, "the prediction workspace does not fit the device");
    }
}

int guarded(const char *where, auto &&fn) {
    try {
        fn();
        return IRX_OK;
    } catch (const Failure &f) {
        g_last_error = f.message;
        return f.status;
    } catch (const std::bad_alloc &) {
        g_last_error = std::string(where) + ": host out of memory";
        return IRX_OUT_OF_MEMORY;
    } catch (...) {
        g_last_error = std::string(where) + ": unexpected failure";
        return IRX_DEVICE_ERROR;
    }
}

// ---- the 4-bit ICL cache: argument checks ----

constexpr size_t kIcl4MaxQueries = size_t(1) << 24, kIcl4MaxBlocks = 4096;
constexpr size_t kIcl4MaxRows = 0x7fffffff;  // (estimator, head, query) rows of a call

// The calling thread's current device while a call is on `d`'s.
class CurrentDevice {
  public:
    explicit CurrentDevice(const irx_device *d) {
        IRX_HIP(hipGetDevice(&before_));
        if (before_ != d->ordinal) IRX_HIP(hipSetDevice(d->ordinal));
        moved_ = before_ != d->ordinal;
    }
    ~CurrentDevice() {
        if (moved_) (void)hipSetDevice(before_);
    }
    CurrentDevice(const CurrentDevice &) = delete;
    CurrentDevice &operator=(const CurrentDevice &) = delete;

  private:
    int before_ = 0;
    bool moved_ = false;
};

Icl4Shape icl4_shape(const irx_icl4_shape &s) { return {(int)s.estimators, (int)s.heads, (int)s.rows}; }

bool icl4_shape_ok(const irx_icl4_shape *s) {
    if (!s || !s->estimators || !s->heads || !s->rows) return false;
    if (s->estimators > 65535 || s->heads > 65535 || s->estimators * s->heads > 65535) return false;
    if (s->rows > (size_t)1 << 27) return false;
    // A workgroup of 256 to a block: one launch of less than 2^32 work-items.
    return s->estimators * s->heads * ((s->rows + kIcl4Block - 1) / kIcl4Block) < (size_t)1 << 24;
}

void icl4_aligned(const void *p, size_t bytes, const char *what) {
    if (reinterpret_cast<uintptr_t>(p) % bytes)
        fail(IRX_INVALID_ARGUMENT, std::string(what) + " must be aligned to " + std::to_string(bytes) + " bytes");
}

// Strides of [estimators, heads, rows, 64], checked: whole 16 bytes, offsets within 2^60 elements.
void icl4_strides(const irx_icl4_shape &s, size_t rows, bool half, const irx_strides &in, long long *out) {
    const size_t unit = half ? 8 : 4, most = (size_t)1 << 40;
    const size_t stride[3] = {in.estimator, in.head, in.row}, count[3] = {s.estimators, s.heads, rows};
    for (int i = 0; i < 3; ++i) {
        // A stride along which there is one element is not used.
        if (count[i] > 1 && (stride[i] % unit || stride[i] > most / count[i]))
            fail(IRX_INVALID_ARGUMENT, "strides must be multiples of 16 bytes and within range");
        out[i] = count[i] > 1 ? (long long)stride[i] : 0;
    }
}

// An output's strides: no two rows may share a number.
void icl4_output(const irx_icl4_shape &s, size_t rows, const irx_strides &in) {
    size_t stride[3] = {in.estimator, in.head, in.row}, count[3] = {s.estimators, s.heads, rows};
    // From the smallest stride up, each steps over all that the smaller ones reach.
    size_t reach = 64;
    bool done[3] = {count[0] < 2, count[1] < 2, count[2] < 2};
    for (int step = 0; step < 3; ++step) {
        int least = -1;
        for (int i = 0; i < 3; ++i)
            if (!done[i] && (least < 0 || stride[i] < stride[least])) least = i;
        if (least < 0) break;
        if (stride[least] < reach) fail(IRX_INVALID_ARGUMENT, "an output's rows must not overlap");
        reach += stride[least] * (count[least] - 1);
        done[least] = true;
    }
}

bool icl4_half(int element) {
    if (element != IRX_ELEMENT_F32 && element != IRX_ELEMENT_F16)
        fail(IRX_INVALID_ARGUMENT, "elements are FP32 or FP16");
    return element == IRX_ELEMENT_F16;
}

Icl4Rows icl4_rows(const irx_icl4_rows &r) {
    if (!icl4_shape_ok(&r.shape)) fail(IRX_INVALID_ARGUMENT, "the 4-bit cache's shape is out of range");
    Icl4Rows a{};
    a.shape = icl4_shape(r.shape), a.half = icl4_half(r.element), a.k = r.k, a.v = r.v, a.lengths = r.lengths;
    if (r.k) icl4_strides(r.shape, r.shape.rows, a.half, r.k_strides, a.k_strides);
    if (r.v) icl4_strides(r.shape, r.shape.rows, a.half, r.v_strides, a.v_strides);
    icl4_aligned(r.k, 16, "keys");
    icl4_aligned(r.v, 16, "values");
    icl4_aligned(r.lengths, 4, "lengths");
    return a;
}

Icl4Queries icl4_queries(const irx_icl4_queries &q, const void *cache) {
    if (!icl4_shape_ok(&q.shape)) fail(IRX_INVALID_ARGUMENT, "the 4-bit cache's shape is out of range");
    if (!q.q || !q.query_rows || q.query_rows > kIcl4MaxQueries)
        fail(IRX_INVALID_ARGUMENT, "1 to 2^24 queries are answered");
    if (q.query_rows > kIcl4MaxRows / (q.shape.estimators * q.shape.heads))
        fail(IRX_INVALID_ARGUMENT, "too many queries for one call");
    Icl4Queries a{};
    a.shape = icl4_shape(q.shape), a.half = icl4_half(q.element), a.cache = cache, a.q = q.q;
    icl4_strides(q.shape, q.query_rows, a.half, q.q_strides, a.q_strides);
    a.q_rows = (int)q.query_rows, a.lengths = q.lengths;
    a.keep = reinterpret_cast<const unsigned long long *>(q.keep);
    icl4_aligned(q.q, 16, "queries");
    icl4_aligned(cache, 16, "the cache");
    icl4_aligned(q.lengths, 4, "lengths");
    icl4_aligned(q.keep, 8, "keep");
    return a;
}

// After the checks that need none, so that they hold without a GPU too.
void icl4_device(const irx_device *device) {
    if (!device) fail(IRX_INVALID_ARGUMENT, "the call needs a device");
}

void icl4_workspace(const void *workspace, size_t bytes, size_t needed) {
    icl4_aligned(workspace, 16, "the workspace");
    if (needed && (!workspace || bytes < needed))
        fail(IRX_INVALID_ARGUMENT, "the workspace must hold " + std::to_string(needed) + " bytes");
}

// ---- attention for training: argument checks ----

bool train_shape_ok(const irx_train_shape *s) {
    const size_t most = (size_t)1 << 24;
    if (!s || !s->estimators || !s->heads || !s->kv_heads || !s->query_rows || !s->rows) return false;
    if (s->estimators > 65535 || s->heads > 65535 || s->estimators * s->heads > 65535 || s->heads % s->kv_heads) return false;
    return s->query_rows <= most && s->rows <= most;
}

TrainShape train_shape(const irx_train_shape &s) {
    return {(int)s.estimators, (int)s.heads, (int)s.kv_heads, (int)s.query_rows, (int)s.rows};
}

int train_element(int element) {
    if (element != IRX_ELEMENT_F32 && element != IRX_ELEMENT_F16 && element != IRX_ELEMENT_BF16)
        fail(IRX_INVALID_ARGUMENT, "elements are FP32, FP16 or BF16");
    return element;
}

TrainDrop train_drop(const irx_train_drop &d) {
    if (d.dropped > 65535) fail(IRX_INVALID_ARGUMENT, "0 to 65,535 of 65,536 numbers are dropped");
    if (d.dropped && !d.seed) fail(IRX_INVALID_ARGUMENT, "dropout needs a seed");
    icl4_aligned(d.seed, 8, "the seed");
    return {reinterpret_cast<const unsigned long long *>(d.seed), d.site, d.dropped};
}

// One tensor of the calls: its address and strides, and an output's rows apart.
void train_tensor(const irx_train_shape &s, size_t heads, size_t rows, int element, const void *p, const char *what,
                  const irx_strides &in, long long *strides, bool output) {
    const irx_icl4_shape shape = {s.estimators, heads, rows};
    icl4_aligned(p, 16, what);
    icl4_strides(shape, rows, element != IRX_ELEMENT_F32, in, strides);
    if (output) icl4_output(shape, rows, in);
}

TrainInputs train_inputs(const irx_train_inputs &in) {
    if (!train_shape_ok(&in.shape)) fail(IRX_INVALID_ARGUMENT, "the attention's shape is out of range");
    if (!in.q || !in.k || !in.v) fail(IRX_INVALID_ARGUMENT, "attention needs queries, keys and values");
    if (!(in.scale >= 0x1p-64f && in.scale <= 0x1p64f)) fail(IRX_INVALID_ARGUMENT, "the scale is 2^-64 to 2^64");
    TrainInputs a{};
    a.shape = train_shape(in.shape), a.element = train_element(in.element), a.scale = in.scale;
    a.q = in.q, a.k = in.k, a.v = in.v;
    train_tensor(in.shape, in.shape.heads, in.shape.query_rows, in.element, in.q, "queries", in.q_strides, a.qs, false);
    train_tensor(in.shape, in.shape.kv_heads, in.shape.rows, in.element, in.k, "keys", in.k_strides, a.ks, false);
    train_tensor(in.shape, in.shape.kv_heads, in.shape.rows, in.element, in.v, "values", in.v_strides, a.vs, false);
    icl4_aligned(in.query_lengths, 4, "query lengths");
    icl4_aligned(in.lengths, 4, "lengths");
    icl4_aligned(in.keep, 8, "keep");
    a.q_lengths = in.query_lengths, a.lengths = in.lengths;
    a.keep = reinterpret_cast<const unsigned long long *>(in.keep);
    a.drop = train_drop(in.drop);
    return a;
}

void device_release(irx_device *d) {
    if (d && d->refs.fetch_sub(1) == 1) delete d;
}

}  // namespace

// ===================================================================
// C ABI
// ===================================================================

extern "C" {

const char *irx_last_error(void) { return g_last_error.c_str(); }
int irx_abi_version(void) { return IRX_ABI_VERSION; }

int irx_device_open(int ordinal, irx_device **out) {
    return guarded("irx_device_open", [&] {
        if (!out) fail(IRX_INVALID_ARGUMENT, "out is null");
        *out = nullptr;
        const char *off = std::getenv("IRONICL_NO_ROCM");
        if (off && *off) fail(IRX_NO_DEVICE, "IRONICL_NO_ROCM is set");
        int count = 0;
        if (hipGetDeviceCount(&count) != hipSuccess || count <= ordinal || ordinal < 0)
            fail(IRX_NO_DEVICE, "no ROCm device");
        hipDeviceProp_t props;
        IRX_HIP(hipGetDeviceProperties(&props, ordinal));
        if (std::strncmp(props.gcnArchName, "gfx950", 6) != 0)
            fail(IRX_NO_DEVICE, std::string("kernels are built for gfx950, not ") + props.gcnArchName);
        IRX_HIP(hipSetDevice(ordinal));
        // The device address of this device's scratch array (the array's name
        // in host code is no device address).
        float *scratch_ptr = nullptr;
        IRX_HIP(hipGetSymbolAddress(reinterpret_cast<void **>(&scratch_ptr), HIP_SYMBOL(scratch)));
        auto d = new irx_device();
        d->ordinal = ordinal;
        d->compute_units = props.multiProcessorCount;
        d->scratch = scratch_ptr;
        d->memory_bytes = props.totalGlobalMem;
        *out = d;
    });
}

void irx_device_close(irx_device *device) { device_release(device); }

int irx_device_free_memory(irx_device *device, size_t *bytes) {
    return guarded("irx_device_free_memory", [&] {
        if (!device || !bytes) fail(IRX_INVALID_ARGUMENT, "null argument");
        set_device(device);
        size_t free_b = 0, total = 0;
        IRX_HIP(hipMemGetInfo(&free_b, &total));
        *bytes = free_b;
    });
}

int irx_device_compute_units(irx_device *device, int *units) {
    return guarded("irx_device_compute_units", [&] {
        if (!device || !units) fail(IRX_INVALID_ARGUMENT, "null argument");
        *units = device->compute_units;
    });
}

int irx_weights_upload(irx_device *device, int task, irx_tensor_lookup lookup, void *user, irx_weights **out) {
    irx_weights *W = nullptr;
    int st = guarded("irx_weights_upload", [&] {
        if (!device || !lookup || !out) fail(IRX_INVALID_ARGUMENT, "null argument");
        if (task != IRX_TASK_CLASSIFIER && task != IRX_TASK_REGRESSOR) fail(IRX_INVALID_ARGUMENT, "unknown task");
        *out = nullptr;
        set_device(device);
        W = new irx_weights();
        W->device = device;
        device->refs.fetch_add(1);
        W->task = task;
        W->width = task == IRX_TASK_CLASSIFIER ? 10 : 999;
        weights_load(W, lookup, user);
        *out = W;
        W = nullptr;
    });
    if (W) irx_weights_release(W);
    return st;
}

void irx_weights_retain(irx_weights *weights) {
    if (weights) weights->refs.fetch_add(1);
}

void irx_weights_release(irx_weights *weights) {
    if (!weights || weights->refs.fetch_sub(1) != 1) return;
    irx_device *d = weights->device;
    if (d) (void)hipSetDevice(d->ordinal);
    delete weights;
    device_release(d);
}

size_t irx_weights_bytes(const irx_weights *weights) { return weights ? weights->bytes : 0; }

int irx_weights_budget(const irx_weights *weights, uint64_t device_limit, size_t *budget) {
    return guarded("irx_weights_budget", [&] {
        if (!weights || !budget) fail(IRX_INVALID_ARGUMENT, "null argument");
        set_device(weights->device);
        size_t free_b = 0, total = 0;
        IRX_HIP(hipMemGetInfo(&free_b, &total));
        if (device_limit) {
            size_t limit = device_limit > weights->bytes ? (size_t)(device_limit - weights->bytes) : 0;
            free_b = std::min(free_b, limit);
        }
        *budget = free_b;
    });
}

size_t irx_predict_workspace_bytes(irx_device *device, const irx_shape *shape, int precision, size_t pass_rows) {
    if (!device || !shape_ok(shape) || !irx_context_bytes(precision) || pass_rows < 1 || pass_rows > (1u << 20))
        return 0;
    // The split plan of the ICL attention, and with it the partials, follows
    // the device's compute units.
    return predict_ws_floats(*shape, pass_rows, device->compute_units, precision != IRX_PRECISION_FP32) * 4;
}

size_t irx_context_bytes(int precision) {
    // HALF contexts store FP16 K/V, as SPLIT ones; only the resident cache is FP8.
    return precision == IRX_PRECISION_FP32 ? 4
           : precision == IRX_PRECISION_SPLIT || precision == IRX_PRECISION_HALF ? 2
                                                                                 : 0;
}

int irx_build_fits(size_t budget, int precision, const irx_shape *shape) {
    if (!irx_context_bytes(precision) || !shape_ok(shape) || shape->rows < 64)
        return 0;
    // fits (build.rs:158-160) takes no device: the caller's current one, as
    // the reference's single CUDA device, sets the split plan.
    int ordinal = 0, cus = 256;
    if (hipGetDevice(&ordinal) != hipSuccess ||
        hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, ordinal) != hipSuccess || cus <= 0) {
        (void)hipGetLastError();
        cus = 256;
    }
    BuildPlan p = plan_build(*shape, budget, cus, precision);
    return p.ws_bytes + p.keep_bytes <= budget / 10 * 9;
}

int irx_build(irx_weights *weights, int precision, const irx_build_inputs *inputs, irx_build_outputs *outputs,
              irx_built_cache **keep) {
    return guarded("irx_build", [&] {
        if (!weights || !inputs) fail(IRX_INVALID_ARGUMENT, "null argument");
        if (!irx_context_bytes(precision)) fail(IRX_INVALID_ARGUMENT, "precision must be FP32, SPLIT or HALF");
        if (keep) *keep = nullptr;
        if (inputs->shape.outputs == 0 || inputs->shape.outputs > (size_t)weights->width)
            fail(IRX_INVALID_ARGUMENT, "outputs exceed the decoder width");
        build_impl(weights, inputs, outputs, keep, precision);
    });
}

void irx_built_cache_free(irx_built_cache *cache) {
    if (!cache) return;
    if (cache->device) (void)hipSetDevice(cache->device->ordinal);
    delete cache;
}

int irx_predictor_new(irx_weights *weights, int precision, const irx_context_tensors *ctx, irx_built_cache *adopt,
                      irx_predictor **out) {
    irx_predictor *P = nullptr;
    int st = guarded("irx_predictor_new", [&] {
        if (!weights || !ctx || !out) fail(IRX_INVALID_ARGUMENT, "null argument");
        if (precision != IRX_PRECISION_FP32 && precision != IRX_PRECISION_SPLIT && precision != IRX_PRECISION_HALF)
            fail(IRX_INVALID_ARGUMENT, "precision must be FP32, SPLIT or HALF");
        const bool f16 = precision != IRX_PRECISION_FP32, fp8 = precision == IRX_PRECISION_HALF;
        *out = nullptr;
        const irx_shape sh = ctx->shape;
        if (!shape_ok(&sh) || sh.outputs == 0 || sh.outputs > (size_t)weights->width)
            fail(IRX_INVALID_ARGUMENT, "context shape does not match the model");
        for (int i = 0; i < kIclBlocks; ++i)
            if (!ctx->base_scales[i]) fail(IRX_INVALID_ARGUMENT, "base scales are missing");
        if (!ctx->rope_frequencies || !ctx->cls_tokens) fail(IRX_INVALID_ARGUMENT, "row tokens are missing");
        set_device(weights->device);
        const long long B = sh.ensembles, H = sh.features, N = sh.rows, L = H + kReserved;
        const long long col_plane = B * L * kColumnCache, icl_plane = B * kHeads * N * 64;
        const size_t plane16 = icl16_plane(B * kHeads, N);
        const size_t icl_bytes = fp8   ? (size_t)kIclBlocks * icl8_block_bytes(B * kHeads, N)
                                 : f16 ? (size_t)kIclBlocks * 2 * plane16 * 2
                                       : (size_t)kIclBlocks * 2 * icl_plane * 4;
        const size_t cache_bytes = (size_t)kColumnBlocks * 2 * col_plane * 4 + icl_bytes;
        P = new irx_predictor();
        P->weights = weights;
        irx_weights_retain(weights);
        P->shape = sh;
        P->precision = precision;
        const char *no_graphs = std::getenv("IRONICL_NO_GRAPHS");
        P->use_graphs = !(no_graphs && *no_graphs && std::strcmp(no_graphs, "0") != 0);
        if (adopt) {
            if (adopt->shape.ensembles != sh.ensembles || adopt->shape.features != sh.features ||
                adopt->shape.rows != sh.rows)
                fail(IRX_INVALID_ARGUMENT, "the built cache does not match the context");
            if (adopt->precision != precision) fail(IRX_INVALID_ARGUMENT, "the built cache has another precision");
            for (int i = 0; i < kColumnBlocks; ++i) P->column[i] = std::move(adopt->column[i]);
            for (int i = 0; i < kIclBlocks; ++i) P->icl[i] = std::move(adopt->icl[i]);
            for (int i = 0; i < kIclBlocks; ++i) P->icl16[i] = std::move(adopt->icl16[i]);
        } else {
            // Even one 32-row pass must fit beside the caches (fit_workspace settles the rest).
            size_t ws = predict_ws_floats(sh, 32, weights->device->compute_units, f16) * 4;
            if (cache_bytes + ws > ctx->budget / 10 * 9) fail(IRX_DOES_NOT_FIT, "the context does not fit the device");
            if (!ctx->icl) fail(IRX_INVALID_ARGUMENT, "ICL source is missing");
            for (int i = 0; i < kColumnBlocks; ++i)
                if (!ctx->column_keys[i] || !ctx->column_values[i])
                    fail(IRX_INVALID_ARGUMENT, "column caches are missing");
            for (int i = 0; i < kColumnBlocks; ++i) {
                P->column[i].alloc(2 * col_plane * 4);
                IRX_HIP(hipMemcpy(P->column[i].p, ctx->column_keys[i], col_plane * 4, hipMemcpyHostToDevice));
                IRX_HIP(hipMemcpy(P->column[i].f() + col_plane, ctx->column_values[i], col_plane * 4,
                                  hipMemcpyHostToDevice));
            }
            // FP16 contexts: the source gives FP16 bits [B, 8, N, 64], packed here
            // into the FP16 cache (SPLIT) or encoded into the FP8 one (HALF).
            DevBuf staging(f16 ? (size_t)2 * icl_plane * 2 : 0), bad(f16 ? 4 : 0);
            if (f16) IRX_HIP(hipMemset(bad.p, 0, 4));
            for (int i = 0; i < kIclBlocks; ++i) {
                const float *k = nullptr, *v = nullptr;
                if (ctx->icl(ctx->icl_user, (size_t)i, &k, &v) != 0 || !k || !v)
                    fail(IRX_INVALID_ARGUMENT, "the ICL source has no block " + std::to_string(i));
                if (!f16) {
                    P->icl[i].alloc(2 * icl_plane * 4);
                    IRX_HIP(hipMemcpy(P->icl[i].p, k, icl_plane * 4, hipMemcpyHostToDevice));
                    IRX_HIP(hipMemcpy(P->icl[i].f() + icl_plane, v, icl_plane * 4, hipMemcpyHostToDevice));
                } else {
                    unsigned short *sk = static_cast<unsigned short *>(staging.p), *sv = sk + icl_plane;
                    IRX_HIP(hipMemcpy(sk, k, icl_plane * 2, hipMemcpyHostToDevice));
                    IRX_HIP(hipMemcpy(sv, v, icl_plane * 2, hipMemcpyHostToDevice));
                    if (fp8) {
                        P->icl[i].alloc(icl8_block_bytes(B * kHeads, N));
                        encode_icl8(sk, sv, N, (int)(B * kHeads), P->icl[i].p, static_cast<unsigned *>(bad.p), nullptr);
                    } else {
                        P->icl[i].alloc(2 * plane16 * 2);
                        unsigned short *k16 = static_cast<unsigned short *>(P->icl[i].p);
                        pack_icl16(sk, sv, true, N, (int)(B * kHeads), k16, k16 + plane16,
                                   static_cast<unsigned *>(bad.p), nullptr);
                    }
                    IRX_HIP(hipDeviceSynchronize());
                }
            }
            if (f16) {
                unsigned nbad = 0;
                IRX_HIP(hipMemcpy(&nbad, bad.p, 4, hipMemcpyDeviceToHost));
                if (nbad) fail(IRX_NOT_FINITE, "a cached key or value is not finite");
            }
        }
        P->base_scales.alloc(12 * 512 * 4);
        for (int i = 0; i < kIclBlocks; ++i)
            IRX_HIP(hipMemcpy(P->base_scales.f() + i * 512, ctx->base_scales[i], 512 * 4, hipMemcpyHostToDevice));
        std::vector<float> cos_t, sin_t;
        rope_tables(ctx->rope_frequencies, (int)L, cos_t, sin_t);
        P->rope_cos.alloc(cos_t.size() * 4);
        P->rope_sin.alloc(sin_t.size() * 4);
        IRX_HIP(hipMemcpy(P->rope_cos.p, cos_t.data(), cos_t.size() * 4, hipMemcpyHostToDevice));
        IRX_HIP(hipMemcpy(P->rope_sin.p, sin_t.data(), sin_t.size() * 4, hipMemcpyHostToDevice));
        // The pass streams each have a hardware queue of their own (take_lane):
        // passes on two streams that share one of the runtime's pooled queues
        // run in turn (measured: two-stream steps then as slow as one-stream
        // ones, depending on which streams a predictor happened to get). Side
        // streams are taken when a stream count first asks for them
        // (ensure_workspace): every queue the process holds costs the command
        // processor scheduling time.
        P->stream = take_lane(weights->device);
        for (int i = 0; i < kMaxPassStreams - 1; ++i)
            IRX_HIP(hipEventCreateWithFlags(&P->join[i], hipEventDisableTiming));
        IRX_HIP(hipEventCreateWithFlags(&P->fork, hipEventDisableTiming));
        // An adopted cache is already resident: the caller's budget (free memory) excludes it.
        fit_workspace(P, adopt ? 0 : cache_bytes, ctx->budget);
        *out = P;
        P = nullptr;
    });
    if (adopt) irx_built_cache_free(adopt);
    if (P) irx_predictor_free(P);
    return st;
}

void irx_predictor_free(irx_predictor *predictor) {
    if (!predictor) return;
    irx_weights *w = predictor->weights;
    if (w) {
        (void)hipSetDevice(w->device->ordinal);
        for (int i = 0; i < kMaxPassStreams; ++i)
            if (predictor->lane(i)) (void)hipStreamSynchronize(predictor->lane(i));
        predictor->drop_graphs();
        return_lane(w->device, predictor->stream);
        for (int i = 0; i < kMaxPassStreams - 1; ++i) return_lane(w->device, predictor->side[i]);
    }
    for (int i = 0; i < kMaxPassStreams - 1; ++i)
        if (predictor->join[i]) (void)hipEventDestroy(predictor->join[i]);
    if (predictor->fork) (void)hipEventDestroy(predictor->fork);
    delete predictor;
    irx_weights_release(w);
}

int irx_predictor_streamed(const irx_predictor *) { return 0; }

size_t irx_predictor_pass_rows(const irx_predictor *predictor) { return predictor ? predictor->pass_rows : 0; }

int irx_predictor_set_graphs(irx_predictor *predictor, int enable) {
    return guarded("irx_predictor_set_graphs", [&] {
        if (!predictor) fail(IRX_INVALID_ARGUMENT, "null predictor");
        std::lock_guard<std::mutex> lock(predictor->mu);
        set_device(predictor->weights->device);
        for (int i = 0; i < kMaxPassStreams; ++i)
            if (predictor->lane(i)) IRX_HIP(hipStreamSynchronize(predictor->lane(i)));
        predictor->drop_graphs();
        predictor->use_graphs = enable != 0;
    });
}

int irx_predictor_set_streams(irx_predictor *predictor, int streams) {
    return guarded("irx_predictor_set_streams", [&] {
        if (!predictor || streams < 1 || streams > kMaxPassStreams)
            fail(IRX_INVALID_ARGUMENT, "streams must be 1 to " + std::to_string(kMaxPassStreams));
        std::lock_guard<std::mutex> lock(predictor->mu);
        set_device(predictor->weights->device);
        predictor->streams = streams;
        ensure_workspace(predictor);
    });
}

int irx_predictor_read_context(irx_predictor *predictor, size_t tensor, size_t offset, size_t floats, void *dst) {
    return guarded("irx_predictor_read_context", [&] {
        if (!predictor || (floats && !dst)) fail(IRX_INVALID_ARGUMENT, "context read needs a predictor and a buffer");
        const irx_shape &s = predictor->shape;
        const size_t col_plane = s.ensembles * (s.features + kReserved) * (size_t)kColumnCache;
        const size_t icl_plane = s.ensembles * (size_t)kHeads * s.rows * kIclHead;
        const size_t column_tensors = 2 * kColumnBlocks;
        if (tensor >= column_tensors + 2 * kIclBlocks) fail(IRX_INVALID_ARGUMENT, "context tensor index out of range");
        const bool column = tensor < column_tensors;
        const size_t index = column ? tensor : tensor - column_tensors;
        const size_t plane = column ? col_plane : icl_plane;
        if (offset > plane || floats > plane - offset) fail(IRX_INVALID_ARGUMENT, "context read past the tensor's end");
        if (!floats) return;
        const DevBuf &buf = column ? predictor->column[index / 2]
                            : predictor->precision == IRX_PRECISION_HALF ? predictor->icl16[index / 2]
                                                                         : predictor->icl[index / 2];
        std::lock_guard<std::mutex> lock(predictor->mu);
        set_device(predictor->weights->device);
        if (!column && predictor->precision == IRX_PRECISION_HALF && !predictor->icl16[index / 2].p)
            fail(IRX_UNSUPPORTED, "a fast (FP8) predictor made from context tensors keeps no FP16 ICL tensors");
        if (!column && predictor->precision != IRX_PRECISION_FP32) {
            // FP16 bits in the logical layout, unpacked from the cache layout.
            const long long pairs = (long long)s.ensembles * kHeads;
            const size_t plane16 = icl16_plane(pairs, (long long)s.rows);
            DevBuf logical(2 * plane * 2);
            const unsigned short *k16 = static_cast<const unsigned short *>(buf.p);
            unsigned short *lk = static_cast<unsigned short *>(logical.p);
            unpack_icl16(k16, k16 + plane16, (long long)s.rows, (int)pairs, lk, lk + plane, predictor->stream);
            IRX_HIP(hipMemcpyAsync(dst, lk + (index % 2) * plane + offset, floats * 2, hipMemcpyDeviceToHost,
                                   predictor->stream));
            IRX_HIP(hipStreamSynchronize(predictor->stream));
            return;
        }
        const float *src = buf.f() + (index % 2) * plane + offset;
        // On the predictor's stream: after every pass issued before the call.
        IRX_HIP(hipMemcpyAsync(dst, src, floats * 4, hipMemcpyDeviceToHost, predictor->stream));
        IRX_HIP(hipStreamSynchronize(predictor->stream));
    });
}

int irx_predictor_set_pass_rows(irx_predictor *predictor, size_t rows) {
    return guarded("irx_predictor_set_pass_rows", [&] {
        if (!predictor || rows < 32 || rows % 32 || rows > (1u << 20))
            fail(IRX_INVALID_ARGUMENT, "pass rows must be a positive multiple of 32");
        std::lock_guard<std::mutex> lock(predictor->mu);
        set_device(predictor->weights->device);
        predictor->pass_rows = rows;
        ensure_workspace(predictor);
    });
}

// Host buffers of a prediction: each pass's rows are copied into pinned
// staging and go up on the pass's stream just before it, and its logits come
// back into pinned staging on the same stream right after it, so the first
// pass waits for its own rows only and the copies overlap other passes.
struct HostIo {
    const float *x;    // [B, q, H], the caller's
    float *pin_x;      // [B, q, H], pinned
    float *pin_logits; // [B, q, width], pinned
};

// Every pass of a prediction of q rows. With cpu_rows (host, [q]), the rows
// holding the all-missing marker are flagged there: the passes set device
// flags, read back once after the last pass, so passes never wait on the host.
// With io, the inputs start on the host and d_x / d_logits are the
// predictor's device copies of them.
static void predict_common(irx_predictor *P, const float *d_x, size_t q, float *d_logits, uint8_t *cpu_rows,
                           irx_progress_fn progress, void *user, const HostIo *io = nullptr) {
    const size_t R = P->pass_rows;
    uint8_t *d_flags = nullptr;
    if (cpu_rows) {
        if (P->io_flags.bytes < q) P->io_flags.alloc(q);
        d_flags = static_cast<uint8_t *>(P->io_flags.p);
        IRX_HIP(hipMemsetAsync(d_flags, 0, q, P->stream));
    }
    // Side streams start after everything already queued on the main one (the
    // inputs' upload), and the main stream ends after the side streams' passes.
    const int lanes = P->streams;
    IRX_HIP(hipEventRecord(P->fork, P->stream));
    for (int i = 1; i < lanes; ++i) IRX_HIP(hipStreamWaitEvent(P->lane(i), P->fork, 0));
    const size_t B = P->shape.ensembles, H = P->shape.features, width = P->shape.outputs;
    int slot = 0;
    for (size_t q0 = 0; q0 < q; q0 += R, slot = (slot + 1) % lanes) {
        const int len = (int)std::min(R, q - q0);
        if (io) {  // the pass's rows of every estimator
            for (size_t e = 0; e < B; ++e)
                std::memcpy(io->pin_x + (e * q + q0) * H, io->x + (e * q + q0) * H, (size_t)len * H * 4);
            IRX_HIP(hipMemcpy2DAsync(const_cast<float *>(d_x) + q0 * H, q * H * 4, io->pin_x + q0 * H, q * H * 4,
                                     (size_t)len * H * 4, B, hipMemcpyHostToDevice, P->lane(slot)));
        }
        predict_pass(P, slot, d_x, (long long)q * H, (int)q0, len, d_logits, (int)q, d_flags);
        if (io)
            IRX_HIP(hipMemcpy2DAsync(io->pin_logits + q0 * width, q * width * 4, d_logits + q0 * width,
                                     q * width * 4, (size_t)len * width * 4, B, hipMemcpyDeviceToHost,
                                     P->lane(slot)));
        if (progress) {
            IRX_HIP(hipStreamSynchronize(P->lane(slot)));
            report(progress, user, IRX_STAGE_PREDICT, q0 + len, q);
        }
    }
    for (int i = 1; i < lanes; ++i) {
        IRX_HIP(hipEventRecord(P->join[i - 1], P->lane(i)));
        IRX_HIP(hipStreamWaitEvent(P->stream, P->join[i - 1], 0));
    }
    if (cpu_rows) download(cpu_rows, d_flags, q, P->stream);  // complete at the caller's synchronisation
}

int irx_predictor_predict(irx_predictor *predictor, const float *x, size_t q, float *logits, uint8_t *cpu_rows,
                          irx_progress_fn progress, void *progress_user) {
    return guarded("irx_predictor_predict", [&] {
        if (!predictor || (!x && q) || (!logits && q)) fail(IRX_INVALID_ARGUMENT, "null argument");
        if (q == 0) return;
        std::lock_guard<std::mutex> lock(predictor->mu);
        set_device(predictor->weights->device);
        const irx_shape &sh = predictor->shape;
        const size_t xn = sh.ensembles * q * sh.features, ln = sh.ensembles * q * sh.outputs;
        // Device copies of the inputs and outputs, kept and grown across calls.
        if (predictor->io_x.bytes < xn * 4) predictor->io_x.alloc(xn * 4);
        if (predictor->io_logits.bytes < ln * 4) predictor->io_logits.alloc(ln * 4);
        predictor->pin_x.reserve(xn * 4);
        predictor->pin_logits.reserve(ln * 4);
        const HostIo io{x, predictor->pin_x.f(), predictor->pin_logits.f()};
        predict_common(predictor, predictor->io_x.f(), q, predictor->io_logits.f(), cpu_rows, progress,
                       progress_user, &io);
        IRX_HIP(hipStreamSynchronize(predictor->stream));
        std::memcpy(logits, predictor->pin_logits.p, ln * 4);
    });
}

int irx_predictor_predict_device(irx_predictor *predictor, const float *x_device, size_t q, float *logits_device,
                                 uint8_t *cpu_rows) {
    return guarded("irx_predictor_predict_device", [&] {
        if (!predictor || (!x_device && q) || (!logits_device && q)) fail(IRX_INVALID_ARGUMENT, "null argument");
        if (q == 0) return;
        std::lock_guard<std::mutex> lock(predictor->mu);
        set_device(predictor->weights->device);
        predict_common(predictor, x_device, q, logits_device, cpu_rows, nullptr, nullptr);
        IRX_HIP(hipStreamSynchronize(predictor->stream));
    });
}

// ---- kernel timing ----

int irx_profile_enable(unsigned families) {
    return guarded("irx_profile_enable", [&] {
        std::lock_guard<std::mutex> lock(g_profile_mu);
        drain_timings();
        if (families) {
            for (auto &t : g_totals) t = FamilyTotals{};
            if (!g_epoch) IRX_HIP(hipEventCreate(&g_epoch));
            IRX_HIP(hipEventRecord(g_epoch, nullptr));
            IRX_HIP(hipEventSynchronize(g_epoch));
        }
        g_profiling.store(families);
    });
}

int irx_profile_read(const char *family, irx_kernel_stats *out) {
    return guarded("irx_profile_read", [&] {
        if (!family || !out) fail(IRX_INVALID_ARGUMENT, "null argument");
        int f = -1;
        for (int i = 0; i < kFamCount; ++i)
            if (std::strcmp(family, kFamilyNames[i]) == 0) f = i;
        if (f < 0) fail(IRX_INVALID_ARGUMENT, std::string("unknown kernel family '") + family + "'");
        std::lock_guard<std::mutex> lock(g_profile_mu);
        drain_timings();
        const FamilyTotals &t = g_totals[f];
        out->launches = t.launches, out->milliseconds = t.ms, out->flops = t.flops, out->bytes = t.bytes;
        out->busy_milliseconds = union_ms(t.spans);
    });
}

// ---- kernel harness ----

int irx_test_icl_attention_precision(irx_device *device, int precision, const float *q, const float *k,
                                     const float *v, size_t pairs, size_t query_rows, size_t rows, float *out) {
    return guarded("irx_test_icl_attention", [&] {
        if (!irx_context_bytes(precision)) fail(IRX_INVALID_ARGUMENT, "unsupported precision");
        const bool f16 = precision != IRX_PRECISION_FP32, fp8 = precision == IRX_PRECISION_HALF;
        if (!device || !q || !k || !v || !out || !pairs || !query_rows || !rows)
            fail(IRX_INVALID_ARGUMENT, "ICL attention shapes do not match");
        if (pairs % kHeads) fail(IRX_INVALID_ARGUMENT, "pairs must be a multiple of 8 (estimators x heads)");
        set_device(device);
        const size_t qn = pairs * query_rows * 64, kn = pairs * rows * 64;
        DevBuf dq(qn * 4), dk(kn * 4), dv(kn * 4), dout(qn * 4);
        IRX_HIP(hipMemcpy(dq.p, q, qn * 4, hipMemcpyHostToDevice));
        IRX_HIP(hipMemcpy(dk.p, k, kn * 4, hipMemcpyHostToDevice));
        IRX_HIP(hipMemcpy(dv.p, v, kn * 4, hipMemcpyHostToDevice));
        size_t pf = icl_attention_partial_floats((int)pairs, (int)query_rows, (int)rows, device->compute_units, f16);
        DevBuf part(pf * 4);
        DevBuf cache16(f16 ? 2 * icl16_plane((long long)pairs, (long long)rows) * 2 : 0), bad(f16 ? 4 : 0);
        DevBuf logical(fp8 ? 2 * kn * 2 : 0), block8(fp8 ? icl8_block_bytes((long long)pairs, (long long)rows) : 0);
        IclAttention a{};
        if (f16) {
            unsigned short *k16 = static_cast<unsigned short *>(cache16.p);
            unsigned short *v16 = k16 + icl16_plane((long long)pairs, (long long)rows);
            IRX_HIP(hipMemset(bad.p, 0, 4));
            pack_icl16(dk.p, dv.p, false, (long long)rows, (int)pairs, k16, v16, static_cast<unsigned *>(bad.p), nullptr);
            a.k16 = k16, a.v16 = v16;
            if (fp8) {
                // FP16 logical K/V (the context's values), then the FP8 cache from them.
                unsigned short *lk = static_cast<unsigned short *>(logical.p), *lv = lk + kn;
                unpack_icl16(k16, v16, (long long)rows, (int)pairs, lk, lv, nullptr);
                encode_icl8(lk, lv, (long long)rows, (int)pairs, block8.p, static_cast<unsigned *>(bad.p), nullptr);
                const Icl8Block c8 = icl8_block(block8.p, (long long)pairs, (long long)rows);
                a.k16 = nullptr, a.v16 = nullptr;
                a.k8 = c8.k, a.v8 = c8.v, a.kscale = c8.kscale, a.vscale = c8.vscale;
            }
        }
        a.q = dq.f(), a.q_pair_stride = (long long)query_rows * 64, a.k = dk.f(), a.v = dv.f();
        a.kv_pair_stride = (long long)rows * 64, a.o = dout.f(), a.ldo = 512;
        a.pairs = (int)pairs, a.q_rows = (int)query_rows, a.kv_rows = (int)rows;
        a.partial = part.f(), a.partial_floats = pf, a.compute_units = device->compute_units;
        icl_attention(a, nullptr);
        IRX_HIP(hipDeviceSynchronize());
        // Tokens [b, q, 8, 64] back to [pairs, q, 64].
        std::vector<float> tok(qn);
        IRX_HIP(hipMemcpy(tok.data(), dout.p, qn * 4, hipMemcpyDeviceToHost));
        for (size_t p = 0; p < pairs; ++p) {
            size_t b = p / kHeads, h = p % kHeads;
            for (size_t r = 0; r < query_rows; ++r)
                std::memcpy(out + (p * query_rows + r) * 64, tok.data() + ((b * query_rows + r) * 512 + h * 64), 256);
        }
    });
}

int irx_test_encode_icl8(irx_device *device, const uint16_t *k, const uint16_t *v, size_t pairs, size_t rows,
                         void *block) {
    return guarded("irx_test_encode_icl8", [&] {
        if (!device || !k || !v || !block || !pairs || !rows) fail(IRX_INVALID_ARGUMENT, "FP8 encode shapes do not match");
        set_device(device);
        const size_t n = pairs * rows * 64, bytes = icl8_block_bytes((long long)pairs, (long long)rows);
        DevBuf dk(n * 2), dv(n * 2), out(bytes), bad(4);
        IRX_HIP(hipMemcpy(dk.p, k, n * 2, hipMemcpyHostToDevice));
        IRX_HIP(hipMemcpy(dv.p, v, n * 2, hipMemcpyHostToDevice));
        IRX_HIP(hipMemset(bad.p, 0, 4));
        encode_icl8(static_cast<const unsigned short *>(dk.p), static_cast<const unsigned short *>(dv.p),
                    (long long)rows, (int)pairs, out.p, static_cast<unsigned *>(bad.p), nullptr);
        IRX_HIP(hipDeviceSynchronize());
        unsigned nbad = 0;
        IRX_HIP(hipMemcpy(&nbad, bad.p, 4, hipMemcpyDeviceToHost));
        if (nbad) fail(IRX_NOT_FINITE, "a key or value is not finite");
        IRX_HIP(hipMemcpy(block, out.p, bytes, hipMemcpyDeviceToHost));
    });
}

int irx_test_icl_attention(irx_device *device, const float *q, const float *k, const float *v, size_t pairs,
                           size_t query_rows, size_t rows, float *out) {
    return irx_test_icl_attention_precision(device, IRX_PRECISION_FP32, q, k, v, pairs, query_rows, rows, out);
}

int irx_icl_attention_noalloc(irx_device *device, const float *q, const float *k, const float *v, size_t pairs,
                              size_t query_rows, size_t rows, float *out, void *stream) {
    return guarded("irx_icl_attention_noalloc", [&] {
        if (!device || !q || !k || !v || !out || !pairs || !query_rows || !rows)
            fail(IRX_INVALID_ARGUMENT, "ICL attention shapes do not match");
        if (pairs % kHeads) fail(IRX_INVALID_ARGUMENT, "pairs must be a multiple of 8 (estimators x heads)");
        if (pairs > (size_t)1 << 20 || query_rows > (size_t)1 << 24 || rows > (size_t)1 << 30)
            fail(IRX_INVALID_ARGUMENT, "ICL attention shape is out of range");
        if (!device->scratch) fail(IRX_DEVICE_ERROR, "the device's scratch array was not set up");
        // The same split plan as irx_test_icl_attention on this device, so the
        // results are the same bit for bit; its partials must fit the scratch.
        const size_t pf = icl_attention_partial_floats((int)pairs, (int)query_rows, (int)rows, device->compute_units);
        if (pf * sizeof(float) > kNoAllocScratchBytes)
            fail(IRX_INVALID_ARGUMENT, "ICL attention of " + std::to_string(pairs) + " pairs x " +
                                           std::to_string(query_rows) + " queries x " + std::to_string(rows) +
                                           " keys needs " + std::to_string(pf * sizeof(float)) +
                                           " bytes of partials; the no-allocation entry point holds " +
                                           std::to_string(kNoAllocScratchBytes));
        set_device(device);
        IclAttention a{};
        a.q = q, a.q_pair_stride = (long long)query_rows * 64, a.k = k, a.v = v;
        a.kv_pair_stride = (long long)rows * 64, a.o = out, a.ldo = 512;
        a.pairs = (int)pairs, a.q_rows = (int)query_rows, a.kv_rows = (int)rows;
        a.partial = pf ? device->scratch : nullptr, a.partial_floats = pf, a.compute_units = device->compute_units;
        icl_attention(a, static_cast<hipStream_t>(stream));
    });
}

// ---- the 4-bit ICL cache ----

size_t irx_icl4_bytes(const irx_icl4_shape *shape) {
    return icl4_shape_ok(shape) ? icl4_bytes(icl4_shape(*shape)) : 0;
}

size_t irx_icl4_workspace_bytes(irx_device *device, const irx_icl4_shape *shape, size_t query_rows, size_t n_blocks) {
    if (!device || !icl4_shape_ok(shape) || !query_rows || query_rows > kIcl4MaxQueries || n_blocks > kIcl4MaxBlocks)
        return 0;
    if (query_rows > kIcl4MaxRows / (shape->estimators * shape->heads)) return 0;
    const Icl4Shape s = icl4_shape(*shape);
    size_t attend = 0;
    for (const bool half : {false, true})
        attend = std::max(attend, icl4_attend_workspace(s, half, (int)query_rows, (int)n_blocks, device->compute_units));
    return n_blocks ? std::max(attend, icl4_select_workspace(s, (int)query_rows)) : attend;
}

int irx_icl4_encode(irx_device *device, const irx_icl4_rows *rows, void *cache, uint32_t *nonfinite, void *stream) {
    return guarded("irx_icl4_encode", [&] {
        if (!rows || !rows->k || !rows->v || !cache)
            fail(IRX_INVALID_ARGUMENT, "the 4-bit cache is written from keys and values");
        const Icl4Rows a = icl4_rows(*rows);
        icl4_aligned(cache, 16, "the cache");
        icl4_aligned(nonfinite, 4, "the counter");
        icl4_device(device);
        CurrentDevice here(device);
        icl4_encode(a, cache, nonfinite, static_cast<hipStream_t>(stream));
    });
}

int irx_icl4_decode(irx_device *device, const void *cache, const irx_icl4_rows *rows, float *bounds, void *stream) {
    return guarded("irx_icl4_decode", [&] {
        if (!rows || !cache || (!rows->k && !rows->v && !bounds))
            fail(IRX_INVALID_ARGUMENT, "nothing to read the 4-bit cache into");
        const Icl4Rows a = icl4_rows(*rows);
        if (rows->k) icl4_output(rows->shape, rows->shape.rows, rows->k_strides);
        if (rows->v) icl4_output(rows->shape, rows->shape.rows, rows->v_strides);
        icl4_aligned(cache, 16, "the cache");
        icl4_aligned(bounds, 4, "bounds");
        icl4_device(device);
        CurrentDevice here(device);
        icl4_decode(a, cache, bounds, static_cast<hipStream_t>(stream));
    });
}

int irx_icl4_select(irx_device *device, const irx_icl4_queries *queries, const void *cache, size_t n_blocks,
                    int32_t *blocks, void *workspace, size_t workspace_bytes, void *stream) {
    return guarded("irx_icl4_select", [&] {
        if (!queries || !cache || !blocks)
            fail(IRX_INVALID_ARGUMENT, "a choice of blocks needs queries, a cache and its output");
        if (!n_blocks || n_blocks > kIcl4MaxBlocks)
            fail(IRX_INVALID_ARGUMENT, "1 to " + std::to_string(kIcl4MaxBlocks) + " blocks are chosen");
        Icl4Queries a = icl4_queries(*queries, cache);
        icl4_aligned(blocks, 4, "blocks");
        if (!icl4_select_fits(a.shape, a.q_rows)) fail(IRX_INVALID_ARGUMENT, "too many queries for one call");
        icl4_device(device);
        a.compute_units = device->compute_units;
        icl4_workspace(workspace, workspace_bytes, icl4_select_workspace(a.shape, a.q_rows));
        CurrentDevice here(device);
        icl4_select(a, (int)n_blocks, blocks, workspace, static_cast<hipStream_t>(stream));
    });
}

int irx_icl4_attention(irx_device *device, const irx_icl4_queries *queries, const void *cache, float scale,
                       const int32_t *blocks, size_t n_blocks, void *out, const irx_strides *out_strides, float *lse,
                       void *workspace, size_t workspace_bytes, void *stream) {
    return guarded("irx_icl4_attention", [&] {
        if (!queries || !cache || !out || !out_strides)
            fail(IRX_INVALID_ARGUMENT, "attention needs queries, a cache and its output");
        // Its product with log2 e is finite, too.
        if (!(scale > 0.f && scale <= 0x1p127f))
            fail(IRX_INVALID_ARGUMENT, "the scale must be positive and finite, at most 2^127");
        if (!blocks != !n_blocks || n_blocks > kIcl4MaxBlocks)
            fail(IRX_INVALID_ARGUMENT, "blocks and n_blocks name 1 to " + std::to_string(kIcl4MaxBlocks) +
                                           " blocks per query, or are NULL and 0");
        Icl4Queries a = icl4_queries(*queries, cache);
        Icl4Attend b{};
        b.scale = scale, b.list = blocks, b.n = (int)n_blocks, b.out = out, b.lse = lse, b.workspace = workspace;
        icl4_strides(queries->shape, queries->query_rows, a.half, *out_strides, b.o_strides);
        icl4_output(queries->shape, queries->query_rows, *out_strides);
        icl4_aligned(out, 16, "the output");
        icl4_aligned(blocks, 4, "blocks");
        icl4_aligned(lse, 4, "lse");
        icl4_device(device);
        a.compute_units = device->compute_units;
        if (!icl4_grid_fits(a.shape, a.half, a.q_rows, b.n, a.compute_units))
            fail(IRX_INVALID_ARGUMENT, "too many queries for one call");
        icl4_workspace(workspace, workspace_bytes, icl4_attend_workspace(a.shape, a.half, a.q_rows, b.n, a.compute_units));
        CurrentDevice here(device);
        icl4_attend(a, b, static_cast<hipStream_t>(stream));
    });
}

size_t irx_train_workspace_bytes(irx_device *device, const irx_train_shape *shape, int element, int backward) {
    if (!device || !train_shape_ok(shape) || element < IRX_ELEMENT_F32 || element > IRX_ELEMENT_BF16) return 0;
    const TrainShape s = train_shape(*shape);
    size_t bytes;
    return train_needs(s, element, backward, device->compute_units, &bytes) ? bytes : 0;
}

int irx_train_attention(irx_device *device, const irx_train_inputs *inputs, void *out, const irx_strides *out_strides,
                        float *stats, float *lse, void *workspace, size_t workspace_bytes, void *stream) {
    return guarded("irx_train_attention", [&] {
        if (!inputs || !out || !out_strides) fail(IRX_INVALID_ARGUMENT, "attention needs its inputs and its output");
        const TrainInputs a = train_inputs(*inputs);
        const irx_train_shape &s = inputs->shape;
        TrainForward f{};
        f.out = out, f.stats = stats, f.lse = lse, f.workspace = workspace;
        train_tensor(s, s.heads, s.query_rows, a.element, out, "the output", *out_strides, f.os, true);
        icl4_aligned(stats, 8, "stats");
        icl4_aligned(lse, 4, "lse");
        icl4_device(device);
        size_t needed;
        if (!train_needs(a.shape, a.element, false, device->compute_units, &needed)) fail(IRX_INVALID_ARGUMENT, "too many rows for one call");
        icl4_workspace(workspace, workspace_bytes, needed);
        CurrentDevice here(device);
        train_attention(a, f, device->compute_units, static_cast<hipStream_t>(stream));
    });
}

int irx_train_attention_backward(irx_device *device, const irx_train_inputs *inputs,
                                 const irx_train_gradients *gradients, void *workspace, size_t workspace_bytes,
                                 void *stream) {
    return guarded("irx_train_attention_backward", [&] {
        if (!inputs || !gradients || !gradients->out || !gradients->stats || !gradients->dout)
            fail(IRX_INVALID_ARGUMENT, "the backward pass needs its inputs, the output, its statistics and its gradient");
        const irx_train_gradients &g = *gradients;
        if (!g.dk != !g.dv || (!g.dq && !g.dk))
            fail(IRX_INVALID_ARGUMENT, "gradients are of the queries, of keys and values, or of both");
        const TrainInputs a = train_inputs(*inputs);
        const irx_train_shape &s = inputs->shape;
        TrainBackward b{};
        b.out = g.out, b.stats = g.stats, b.dout = g.dout, b.dq = g.dq, b.dk = g.dk, b.dv = g.dv, b.workspace = workspace;
        train_tensor(s, s.heads, s.query_rows, a.element, g.out, "the output", g.out_strides, b.os, false);
        train_tensor(s, s.heads, s.query_rows, a.element, g.dout, "the output's gradient", g.dout_strides, b.gs, false);
        icl4_aligned(g.stats, 8, "stats");
        if (g.dq) train_tensor(s, s.heads, s.query_rows, a.element, g.dq, "the queries' gradient", g.dq_strides, b.dqs, true);
        if (g.dk) {
            train_tensor(s, s.kv_heads, s.rows, a.element, g.dk, "the keys' gradient", g.dk_strides, b.dks, true);
            train_tensor(s, s.kv_heads, s.rows, a.element, g.dv, "the values' gradient", g.dv_strides, b.dvs, true);
        }
        icl4_device(device);
        size_t needed;
        if (!train_needs(a.shape, a.element, true, device->compute_units, &needed)) fail(IRX_INVALID_ARGUMENT, "too many rows for one call");
        icl4_workspace(workspace, workspace_bytes, needed);
        CurrentDevice here(device);
        train_backward(a, b, device->compute_units, static_cast<hipStream_t>(stream));
    });
}

int irx_train_dropout(irx_device *device, const irx_train_rows *rows, void *stream) {
    return guarded("irx_train_dropout", [&] {
        if (!rows || !rows->x || !rows->out) fail(IRX_INVALID_ARGUMENT, "dropout needs its input and its output");
        const irx_train_rows &r = *rows;
        if (!r.rows || !r.width || r.width > 0x7fffffff || r.rows > 0x7fffffff / ((r.width + 7) / 8))
            fail(IRX_INVALID_ARGUMENT, "rows and columns are out of range");
        TrainRows a{};
        a.rows = r.rows, a.width = r.width, a.element = train_element(r.element);
        a.x = r.x, a.residual = r.residual, a.out = r.out, a.drop = train_drop(r.drop);
        const size_t unit = r.element == IRX_ELEMENT_F32 ? 4 : 8, strides[3] = {r.x_stride, r.residual_stride, r.out_stride};
        const void *const tensors[3] = {r.x, r.residual, r.out};
        long long *const to[3] = {&a.xs, &a.rs, &a.os};
        for (int i = 0; i < 3; ++i) {
            icl4_aligned(tensors[i], 16, "a tensor");
            if (!tensors[i] || r.rows == 1) continue;
            if (strides[i] % unit || strides[i] < r.width || strides[i] > ((size_t)1 << 40) / r.rows)
                fail(IRX_INVALID_ARGUMENT, "strides must be multiples of 16 bytes, the width at least, and within range");
            *to[i] = (long long)strides[i];
        }
        if ((r.out == r.x && a.os != a.xs) || (r.out == r.residual && a.os != a.rs))
            fail(IRX_INVALID_ARGUMENT, "an input that is the output has its stride");
        icl4_device(device);
        CurrentDevice here(device);
        train_dropout(a, static_cast<hipStream_t>(stream));
    });
}

int irx_test_products(irx_device *device, const float *x, const float *w1, const float *b1, const float *w2,
                      const float *b2, size_t rows, size_t width, size_t depth, size_t width2, float *first,
                      float *second) {
    return guarded("irx_test_products", [&] {
        if (!device || !x || !w1 || !b1 || !w2 || !b2 || !first || !second || !rows || depth % 16 || width % 16)
            fail(IRX_INVALID_ARGUMENT, "tensor product shapes do not match");
        set_device(device);
        DevBuf dx(rows * depth * 4), dw1(width * depth * 4), db1(width * 4), dw2(width2 * width * 4),
            db2(width2 * 4), d1(rows * width * 4), d2(rows * width2 * 4);
        IRX_HIP(hipMemcpy(dx.p, x, rows * depth * 4, hipMemcpyHostToDevice));
        IRX_HIP(hipMemcpy(dw1.p, w1, width * depth * 4, hipMemcpyHostToDevice));
        IRX_HIP(hipMemcpy(db1.p, b1, width * 4, hipMemcpyHostToDevice));
        IRX_HIP(hipMemcpy(dw2.p, w2, width2 * width * 4, hipMemcpyHostToDevice));
        IRX_HIP(hipMemcpy(db2.p, b2, width2 * 4, hipMemcpyHostToDevice));
        GemmArgs g{};
        g.a = dx.f(), g.lda = (long long)depth, g.w = dw1.f(), g.bias = db1.f(), g.c = d1.f();
        g.out = OutMap::row_major((int)width, (long long)width);
        g.m = (int)rows, g.n = (int)width, g.k = (int)depth, g.epilogue = kEpiGelu;
        gemm(g, nullptr);
        GemmArgs h{};
        h.a = d1.f(), h.lda = (long long)width, h.w = dw2.f(), h.bias = db2.f(), h.c = d2.f();
        h.out = OutMap::row_major((int)width2, (long long)width2);
        h.m = (int)rows, h.n = (int)width2, h.k = (int)width;
        if (width2 == width) h.epilogue = kEpiResidual, h.residual = d1.f(), h.ldr = (long long)width;
        gemm(h, nullptr);
        IRX_HIP(hipDeviceSynchronize());
        IRX_HIP(hipMemcpy(first, d1.p, rows * width * 4, hipMemcpyDeviceToHost));
        IRX_HIP(hipMemcpy(second, d2.p, rows * width2 * 4, hipMemcpyDeviceToHost));
    });
}

int irx_regression_summary(irx_device *device, const float *decoded, size_t ensembles, size_t rows,
                           size_t quantiles, const float *levels, size_t n_levels, float *mean, float *variance,
                           float *at_levels, float *raw) {
    return guarded("irx_regression_summary", [&] {
        if (!device || (!decoded && rows) || (n_levels && !levels))
            fail(IRX_INVALID_ARGUMENT, "regression summary needs a device, decoded quantiles and levels");
        if (!ensembles || quantiles < 2 || quantiles > 4096)
            fail(IRX_INVALID_ARGUMENT, "regression needs at least one estimator and 2 to 4096 quantiles");
        if (n_levels > (size_t)kRegressionMaxLevels)
            fail(IRX_INVALID_ARGUMENT, "at most " + std::to_string(kRegressionMaxLevels) + " quantile levels");
        if (rows > (1u << 30)) fail(IRX_INVALID_ARGUMENT, "too many rows");
        for (size_t i = 0; i < n_levels; ++i)
            if (!std::isfinite(levels[i])) fail(IRX_INVALID_ARGUMENT, "quantile levels must be finite");
        if (!rows) return;
        set_device(device);
        int tail = 0;
        std::vector<double> tail_x;
        std::vector<RegressionLevel> table;
        regression_tables(levels, (int)n_levels, (int)quantiles, &tail, tail_x, table);
        DevBuf dx(tail_x.size() * sizeof(double)), dl(std::max<size_t>(table.size(), 1) * sizeof(RegressionLevel));
        IRX_HIP(hipMemcpy(dx.p, tail_x.data(), tail_x.size() * sizeof(double), hipMemcpyHostToDevice));
        if (!table.empty())
            IRX_HIP(hipMemcpy(dl.p, table.data(), table.size() * sizeof(RegressionLevel), hipMemcpyHostToDevice));
        RegressionSummary rs{};
        rs.decoded = decoded, rs.b = (int)ensembles, rs.q = (int)rows, rs.k = (int)quantiles;
        rs.tail = tail, rs.tail_x = static_cast<const double *>(dx.p);
        rs.levels = (int)n_levels, rs.level = static_cast<const RegressionLevel *>(dl.p);
        rs.mean = mean, rs.variance = variance, rs.at_levels = n_levels ? at_levels : nullptr, rs.raw = raw;
        regression_summary(rs, nullptr);
        IRX_HIP(hipDeviceSynchronize());
    });
}

int irx_test_block_head(irx_device *device, int fused, const float *x, size_t rows, const float *lnw,
                        const float *lnb, const float *w, const float *b, size_t outputs, float *out) {
    return guarded("irx_test_block_head", [&] {
        if (!device || !x || !rows || !lnw || !lnb || !w || !b || !out || (fused != 0 && fused != 1) ||
            (outputs != 128 && outputs != 256 && outputs != 384))
            fail(IRX_INVALID_ARGUMENT, "block head arguments do not match");
        set_device(device);
        std::vector<float> pack(head128_pack_floats((int)outputs));
        head128_pack(lnw, lnb, w, (int)outputs, pack.data());
        auto up = [](const float *h, size_t count) {
            DevBuf d(count * 4);
            IRX_HIP(hipMemcpy(d.p, h, count * 4, hipMemcpyHostToDevice));
            return d;
        };
        DevBuf dx = up(x, rows * 128), dlw = up(lnw, 128), dlb = up(lnb, 128), dw = up(w, outputs * 128);
        DevBuf db = up(b, outputs), dp = up(pack.data(), pack.size()), dnorm(rows * 128 * 4), dout(rows * outputs * 4);
        BlockW bw{};
        bw.dim = 128, bw.n1w = dlw.f(), bw.n1b = dlb.f(), bw.in_w = dw.f(), bw.in_b = db.f();
        bw.head_pack = fused ? dp.f() : nullptr, bw.head_nb = (int)outputs / 16, bw.head_row0 = 0;
        irx_weights none;
        Stages st{none, nullptr, device->compute_units};
        if (fused) {
            Head128 h{};
            h.x = dx.f(), h.ldx = 128, h.lnw = dlw.f(), h.lnb = dlb.f(), h.pack = dp.f(), h.b = db.f();
            h.out = dout.f(), h.ldo = (long long)outputs, h.m = (long long)rows, h.nb = (int)outputs / 16;
            head128(h, nullptr);
        } else {
            st.head(bw, dx.f(), (long long)rows, dnorm.f(), dout.f(), (long long)outputs);
        }
        IRX_HIP(hipDeviceSynchronize());
        IRX_HIP(hipMemcpy(out, dout.p, rows * outputs * 4, hipMemcpyDeviceToHost));
    });
}

int irx_test_block_tail(irx_device *device, int fused, const float *att, const float *state, size_t rows,
                        const float *wo, const float *bo, const float *n2w, const float *n2b, const float *w1,
                        const float *b1, const float *w2, const float *b2, size_t repeats, float *out) {
    return guarded("irx_test_block_tail", [&] {
        if (!device || !att || !state || !wo || !bo || !n2w || !n2b || !w1 || !b1 || !w2 || !b2 || !out || !rows ||
            fused < 0 || fused > 2 || !repeats)
            fail(IRX_INVALID_ARGUMENT, "block tail arguments do not match");
        set_device(device);
        const size_t n = rows * 128;
        std::vector<float> host;
        const size_t sizes[] = {128 * 128, 128, 128, 128, 256 * 128, 256, 128 * 256, 128, kTail128PackFloats};
        const float *srcs[] = {wo, bo, n2w, n2b, w1, b1, w2, b2, nullptr};
        size_t offs[9], total = 0;
        for (int i = 0; i < 9; ++i) offs[i] = total, total += (sizes[i] + 63) / 64 * 64;
        host.assign(total, 0.f);
        for (int i = 0; i < 8; ++i) std::memcpy(host.data() + offs[i], srcs[i], sizes[i] * 4);
        tail128_pack(wo, n2w, n2b, w1, b1, w2, host.data() + offs[8]);
        DevBuf dw(total * 4), datt(n * 4), dstate(n * 4), dnorm(n * 4), dhid(2 * n * 4);
        IRX_HIP(hipMemcpy(dw.p, host.data(), total * 4, hipMemcpyHostToDevice));
        IRX_HIP(hipMemcpy(datt.p, att, n * 4, hipMemcpyHostToDevice));
        IRX_HIP(hipMemcpy(dstate.p, state, n * 4, hipMemcpyHostToDevice));
        BlockW bw{};
        const float *f = dw.f();
        bw.dim = 128, bw.out = {f + offs[0], f + offs[1]}, bw.n2w = f + offs[2], bw.n2b = f + offs[3];
        bw.l1 = {f + offs[4], f + offs[5]}, bw.l2 = {f + offs[6], f + offs[7]}, bw.tail_pack = f + offs[8];
        irx_weights none;
        Stages st{none, nullptr, device->compute_units};
        st.tail(bw, dstate.f(), (long long)rows, datt.f(), dnorm.f(), dhid.f(), fused);
        IRX_HIP(hipDeviceSynchronize());
        IRX_HIP(hipMemcpy(out, dstate.p, n * 4, hipMemcpyDeviceToHost));
        // Further applications (timing only) update the same state.
        for (size_t i = 1; i < repeats; ++i) st.tail(bw, dstate.f(), (long long)rows, datt.f(), dnorm.f(), dhid.f(), fused);
        IRX_HIP(hipDeviceSynchronize());
    });
}

int irx_test_column_block(irx_device *device, int fused, const float *state, size_t cols, size_t rows,
                          const float *k, const float *v, const float *lnw, const float *lnb, const float *wq,
                          const float *bq, const float *wo, const float *bo, const float *n2w, const float *n2b,
                          const float *w1, const float *b1, const float *w2, const float *b2, size_t repeats,
                          float *out) {
    return guarded("irx_test_column_block", [&] {
        if (!device || !state || !k || !v || !lnw || !lnb || !wq || !bq || !wo || !bo || !n2w || !n2b || !w1 ||
            !b1 || !w2 || !b2 || !out || !cols || !rows || fused < 0 || fused > 2 || !repeats ||
            cols > (1u << 20) || rows > (1u << 24))
            fail(IRX_INVALID_ARGUMENT, "column block arguments do not match");
        set_device(device);
        const size_t n = cols * rows * 128;
        std::vector<float> host;
        const size_t hpack = head128_pack_floats(128);
        const size_t sizes[] = {128,         128, 128 * 128, 128, 128 * 128, 128, 128, 128, 256 * 128, 256,
                                128 * 256,   128, hpack,     kTail128PackFloats};
        const float *srcs[] = {lnw, lnb, wq, bq, wo, bo, n2w, n2b, w1, b1, w2, b2, nullptr, nullptr};
        constexpr int kParts = 14;
        size_t offs[kParts], total = 0;
        for (int i = 0; i < kParts; ++i) offs[i] = total, total += (sizes[i] + 63) / 64 * 64;
        host.assign(total, 0.f);
        for (int i = 0; i < 12; ++i) std::memcpy(host.data() + offs[i], srcs[i], sizes[i] * 4);
        head128_pack(lnw, lnb, wq, 128, host.data() + offs[12]);
        tail128_pack(wo, n2w, n2b, w1, b1, w2, host.data() + offs[13]);
        DevBuf dw(total * 4), dstate(n * 4), dk(cols * kColumnCache * 4), dv(cols * kColumnCache * 4);
        DevBuf dnorm(n * 4), dq(n * 4), datt(n * 4), dhid(2 * n * 4);
        IRX_HIP(hipMemcpy(dw.p, host.data(), total * 4, hipMemcpyHostToDevice));
        IRX_HIP(hipMemcpy(dstate.p, state, n * 4, hipMemcpyHostToDevice));
        IRX_HIP(hipMemcpy(dk.p, k, cols * kColumnCache * 4, hipMemcpyHostToDevice));
        IRX_HIP(hipMemcpy(dv.p, v, cols * kColumnCache * 4, hipMemcpyHostToDevice));
        const float *f = dw.f();
        irx_weights none;
        BlockW &bw = none.col2[0];
        bw.dim = 128, bw.n1w = f + offs[0], bw.n1b = f + offs[1], bw.in_w = f + offs[2], bw.in_b = f + offs[3];
        bw.out = {f + offs[4], f + offs[5]}, bw.n2w = f + offs[6], bw.n2b = f + offs[7];
        bw.l1 = {f + offs[8], f + offs[9]}, bw.l2 = {f + offs[10], f + offs[11]};
        bw.head_pack = f + offs[12], bw.head_nb = 8, bw.head_row0 = 0, bw.tail_pack = f + offs[13];
        Stages st{none, nullptr, device->compute_units};
        auto run = [&] {
            st.column_attend(0, dstate.f(), (int)cols, (int)rows, dk.f(), dv.f(), (int)cols, 0, dnorm.f(), dq.f(),
                             datt.f(), dhid.f(), fused);
        };
        run();
        IRX_HIP(hipDeviceSynchronize());
        IRX_HIP(hipMemcpy(out, dstate.p, n * 4, hipMemcpyDeviceToHost));
        // Further applications (timing only) update the same state.
        for (size_t i = 1; i < repeats; ++i) run();
        IRX_HIP(hipDeviceSynchronize());
    });
}

int irx_test_ln_linear(irx_device *device, int epilogue, const float *x, size_t m, size_t rows, const float *lnw,
                       const float *lnb, const float *w, const float *b, size_t n, const float *qm0w,
                       const float *qm0b, const float *qm2w, const float *qm2b, const float *base, float *out) {
    return guarded("irx_test_ln_linear", [&] {
        const bool tiled = epilogue == 3, qass = epilogue == kLnQass || tiled || epilogue == 4;
        if (!device || !x || !m || !lnw || !lnb || !w || !b || !out || (epilogue != kLnGelu && !qass) ||
            (qass && (n != 512 || !rows || m % rows || !qm0w || !qm0b || !qm2w || !qm2b || !base)) || !n || n % 64)
            fail(IRX_INVALID_ARGUMENT, "LN-linear arguments do not match");
        set_device(device);
        auto up = [](const float *h, size_t count) {
            DevBuf d(count * 4);
            IRX_HIP(hipMemcpy(d.p, h, count * 4, hipMemcpyHostToDevice));
            return d;
        };
        DevBuf dx = up(x, m * 512), dlw = up(lnw, 512), dlb = up(lnb, 512), dw = up(w, n * 512), db = up(b, n);
        DevBuf dout(m * n * 4);
        if (qass) {
            DevBuf d0w = up(qm0w, 64 * 64), d0b = up(qm0b, 64), d2w = up(qm2w, 64 * 64), d2b = up(qm2b, 64);
            DevBuf dbase = up(base, 512), pack(pair_pack_floats(512, 512) * 4);
            DevBuf dnorm(tiled ? m * 512 * 4 : 0), dq(tiled ? m * 512 * 4 : 0);
            BlockW bw{};
            bw.dim = 512, bw.n1w = dlw.f(), bw.n1b = dlb.f(), bw.in_w = dw.f(), bw.in_b = db.f();
            bw.in_pairs = pair_pack(dw.f(), 512, 512, lnw, lnb, pack.f(), nullptr);
            bw.qm0 = {d0w.f(), d0b.f()}, bw.qm2 = {d2w.f(), d2b.f()};
            irx_weights none;
            Stages st{none, nullptr, device->compute_units};
            st.icl_query_rows(bw, dx.f(), (int)(m / rows), (int)rows, dbase.f(), dnorm.f(), dq.f(), dout.f(), false,
                              !tiled);
            IRX_HIP(hipDeviceSynchronize());
        } else {
            DevBuf pack(pair_pack_floats((int)n, 512) * 4);
            const Lin l{dw.f(), db.f(), pair_pack(dw.f(), (int)n, 512, lnw, lnb, pack.f(), nullptr)};
            irx_weights none;
            Stages{none, nullptr, device->compute_units}.ln_gelu512(dx.f(), (long long)m, dlw.f(), dlb.f(), l, (int)n,
                                                                    dout.f());
            IRX_HIP(hipDeviceSynchronize());
        }
        IRX_HIP(hipDeviceSynchronize());
        IRX_HIP(hipMemcpy(out, dout.p, m * n * 4, hipMemcpyDeviceToHost));
    });
}

int irx_test_icl_kv(irx_device *device, const float *x, size_t rows, const float *w, const float *b,
                    size_t estimators, size_t estimator, float *out) {
    return guarded("irx_test_icl_kv", [&] {
        if (!device || !x || !rows || !w || !b || !out || !estimators || estimator >= estimators ||
            rows > (1u << 20) || estimators > 64)
            fail(IRX_INVALID_ARGUMENT, "K/V projection arguments do not match");
        set_device(device);
        auto up = [](const float *h, size_t count) {
            DevBuf d(count * 4);
            IRX_HIP(hipMemcpy(d.p, h, count * 4, hipMemcpyHostToDevice));
            return d;
        };
        const size_t part = rows * 512, plane = estimators * part;
        DevBuf dx = up(x, part), dw = up(w, 1536 * 512), db = up(b, 1536), dout = up(out, 2 * plane);
        DevBuf pack(pair_pack_floats(1536, 512) * 4);
        BlockW bw{};
        bw.dim = 512, bw.in_w = dw.f(), bw.in_b = db.f();
        bw.in_pairs = pair_pack(dw.f(), 1536, 512, nullptr, nullptr, pack.f(), nullptr);
        irx_weights none;
        Stages st{none, nullptr, device->compute_units};
        st.icl_kv_rows(bw, dx.f(), (int)rows, dout.f() + estimator * part, (long long)plane);
        IRX_HIP(hipDeviceSynchronize());
        IRX_HIP(hipMemcpy(out, dout.p, 2 * plane * 4, hipMemcpyDeviceToHost));
    });
}

int irx_test_pair_linear(irx_device *device, int epilogue, const float *x, size_t m, size_t k, const float *lnw,
                         const float *lnb, const float *w, const float *b, size_t n, const float *residual, float *out) {
    return guarded("irx_test_pair_linear", [&] {
        if (!device || !x || !m || !w || !b || !out || n % 64 || !n || (k != 512 && k != 1024) || !lnw != !lnb ||
            (lnw && k != 512) || epilogue < kEpiNone || epilogue > kEpiResidual || (epilogue == kEpiResidual && !residual))
            fail(IRX_INVALID_ARGUMENT, "pair product arguments do not match");
        set_device(device);
        auto up = [](const float *h, size_t count) {
            DevBuf d(count * 4);
            if (h) IRX_HIP(hipMemcpy(d.p, h, count * 4, hipMemcpyHostToDevice));
            return d;
        };
        DevBuf dx = up(x, m * k), dw = up(w, n * k), db = up(b, n), pack(pair_pack_floats((int)n, (int)k) * 4), dout = up(residual, m * n);
        DevBuf dlw = up(lnw, lnw ? 512 : 1), dlb = up(lnb, lnb ? 512 : 1);
        PairLinear g{};
        g.x = dx.f(), g.ldx = (long long)k, g.lnw = lnw ? dlw.f() : nullptr, g.lnb = lnb ? dlb.f() : nullptr;
        g.w = pair_pack(dw.f(), (int)n, (int)k, lnw, lnb, pack.f(), nullptr);
        g.bias = db.f(), g.residual = dout.f(), g.ldr = (long long)n, g.c = dout.f();
        g.out = OutMap::row_major((int)n, (long long)n), g.m = (int)m, g.n = (int)n, g.k = (int)k, g.epilogue = epilogue;
        g.compute_units = device->compute_units;
        pair_linear(g, nullptr);
        IRX_HIP(hipDeviceSynchronize());
        IRX_HIP(hipMemcpy(out, dout.p, m * n * 4, hipMemcpyDeviceToHost));
    });
}

int irx_test_layer_norm(irx_device *device, const float *x, const float *weight, const float *bias, size_t rows,
                        size_t width, float *out) {
    return guarded("irx_test_layer_norm", [&] {
        if (!device || !x || !weight || !out || !rows || (width != 128 && width != 512))
            fail(IRX_INVALID_ARGUMENT, "layer norm shapes do not match");
        set_device(device);
        DevBuf dx(rows * width * 4), dw(width * 4), db(width * 4), dy(rows * width * 4);
        IRX_HIP(hipMemcpy(dx.p, x, rows * width * 4, hipMemcpyHostToDevice));
        IRX_HIP(hipMemcpy(dw.p, weight, width * 4, hipMemcpyHostToDevice));
        if (bias) IRX_HIP(hipMemcpy(db.p, bias, width * 4, hipMemcpyHostToDevice));
        layer_norm(dx.f(), (long long)width, dw.f(), bias ? db.f() : nullptr, dy.f(), (long long)width,
                   (long long)rows, (int)width, nullptr);
        IRX_HIP(hipDeviceSynchronize());
        IRX_HIP(hipMemcpy(out, dy.p, rows * width * 4, hipMemcpyDeviceToHost));
    });
}

int irx_test_gelu(irx_device *device, const float *x, size_t count, float *out) {
    return guarded("irx_test_gelu", [&] {
        if (!device || !x || !out || !count) fail(IRX_INVALID_ARGUMENT, "GELU arguments do not match");
        set_device(device);
        DevBuf dx(count * 4), dy(count * 4);
        IRX_HIP(hipMemcpy(dx.p, x, count * 4, hipMemcpyHostToDevice));
        gelu_apply(dx.f(), dy.f(), (long long)count, nullptr);
        IRX_HIP(hipDeviceSynchronize());
        IRX_HIP(hipMemcpy(out, dy.p, count * 4, hipMemcpyDeviceToHost));
    });
}

int irx_test_copy(irx_device *device, size_t floats) {
    return guarded("irx_test_copy", [&] {
        if (!device || !floats || floats % 4) fail(IRX_INVALID_ARGUMENT, "copy size must be a multiple of 4 floats");
        set_device(device);
        DevBuf src(floats * 4), dst(floats * 4);
        fill_zero(src.f(), (long long)floats, nullptr);
        copy_floats(src.f(), dst.f(), (long long)floats, nullptr);
        IRX_HIP(hipDeviceSynchronize());
    });
}

namespace {

// Heads [heads, rows, 16] of one sequence; RoPE tables [max(query_rows, rows), 16] or null.
void test_small_attention(irx_device *device, const float *q, const float *k, const float *v, const float *cos_t,
                          const float *sin_t, size_t heads, size_t query_rows, size_t rows, float *out) {
    if (!device || !q || !k || !v || !out || !heads || !query_rows || !rows || heads > 4096 ||
        query_rows > (1u << 20) || rows > (1u << 24) || (!cos_t) != (!sin_t))
        fail(IRX_INVALID_ARGUMENT, "small attention shapes do not match");
    set_device(device);
    const size_t qn = heads * query_rows * 16, kn = heads * rows * 16, tn = std::max(query_rows, rows) * 16;
    DevBuf dq(qn * 4), dk(kn * 4), dv(kn * 4), dout(qn * 4), dcos, dsin;
    IRX_HIP(hipMemcpy(dq.p, q, qn * 4, hipMemcpyHostToDevice));
    IRX_HIP(hipMemcpy(dk.p, k, kn * 4, hipMemcpyHostToDevice));
    IRX_HIP(hipMemcpy(dv.p, v, kn * 4, hipMemcpyHostToDevice));
    SmallAttention a{};
    if (cos_t) {
        dcos.alloc(tn * 4), dsin.alloc(tn * 4);
        IRX_HIP(hipMemcpy(dcos.p, cos_t, tn * 4, hipMemcpyHostToDevice));
        IRX_HIP(hipMemcpy(dsin.p, sin_t, tn * 4, hipMemcpyHostToDevice));
        a.rope_cos = dcos.f(), a.rope_sin = dsin.f();
    }
    a.q = dq.f(), a.k = dk.f(), a.v = dv.f(), a.o = dout.f();
    a.q_seq = a.q_group = 0, a.q_row = 16, a.q_head = (long long)query_rows * 16;
    a.k_seq = a.k_group = 0, a.k_row = 16, a.k_head = (long long)rows * 16;
    a.v_seq = a.v_group = 0, a.v_row = 16, a.v_head = (long long)rows * 16;
    a.o_seq = a.o_group = 0, a.o_row = 16, a.o_head = (long long)query_rows * 16;
    a.group = 1, a.seqs = 1, a.heads = (int)heads, a.q_rows = (int)query_rows, a.kv_rows = (int)rows;
    a.scale = 0.25f;
    DevBuf part;
    if (const long long pf = small_attention_partial_floats(a)) {
        part.alloc((size_t)pf * 4);
        a.partial = part.f(), a.partial_floats = pf;
    }
    small_attention(a, nullptr);
    IRX_HIP(hipDeviceSynchronize());
    IRX_HIP(hipMemcpy(out, dout.p, qn * 4, hipMemcpyDeviceToHost));
}

// Token-major sequences [seqs, rows, heads, 16] (the row transformer's layout:
// a token's heads adjacent) through the kernel `method` selects; with reps > 0
// the launch is also timed reps times after a warm-up, the mean in *ms.
void test_small_attention_tokens(irx_device *device, int method, const float *q, const float *k, const float *v,
                                 const float *cos_t, const float *sin_t, size_t seqs, size_t heads,
                                 size_t query_rows, size_t rows, float *out, int reps, float *ms) {
    if (!device || !q || !k || !v || !out || !seqs || !heads || !query_rows || !rows || heads > 64 ||
        seqs > (1u << 24) || query_rows > (1u << 16) || rows > (1u << 16) || (!cos_t) != (!sin_t) || reps < 0 ||
        reps > 1000 || (reps > 0 && !ms) || seqs * heads * std::max(query_rows, rows) * 16 > (size_t(1) << 31))
        fail(IRX_INVALID_ARGUMENT, "small attention shapes do not match");
    set_device(device);
    const size_t qn = seqs * query_rows * heads * 16, kn = seqs * rows * heads * 16;
    const size_t tn = std::max(query_rows, rows) * 16;
    DevBuf dq(qn * 4), dk(kn * 4), dv(kn * 4), dout(qn * 4), dcos, dsin;
    IRX_HIP(hipMemcpy(dq.p, q, qn * 4, hipMemcpyHostToDevice));
    IRX_HIP(hipMemcpy(dk.p, k, kn * 4, hipMemcpyHostToDevice));
    IRX_HIP(hipMemcpy(dv.p, v, kn * 4, hipMemcpyHostToDevice));
    SmallAttention a{};
    if (cos_t) {
        dcos.alloc(tn * 4), dsin.alloc(tn * 4);
        IRX_HIP(hipMemcpy(dcos.p, cos_t, tn * 4, hipMemcpyHostToDevice));
        IRX_HIP(hipMemcpy(dsin.p, sin_t, tn * 4, hipMemcpyHostToDevice));
        a.rope_cos = dcos.f(), a.rope_sin = dsin.f();
    }
    const long long w = (long long)heads * 16;
    a.q = dq.f(), a.k = dk.f(), a.v = dv.f(), a.o = dout.f();
    a.q_seq = (long long)query_rows * w, a.q_group = 0, a.q_row = w, a.q_head = 16;
    a.k_seq = (long long)rows * w, a.k_group = 0, a.k_row = w, a.k_head = 16;
    a.v_seq = a.k_seq, a.v_group = 0, a.v_row = w, a.v_head = 16;
    a.o_seq = a.q_seq, a.o_group = 0, a.o_row = w, a.o_head = 16;
    a.group = (int)seqs, a.seqs = (int)seqs, a.heads = (int)heads, a.q_rows = (int)query_rows;
    a.kv_rows = (int)rows, a.scale = 0.25f, a.method = method;
    DevBuf part;
    if (const long long pf = small_attention_partial_floats(a)) {
        part.alloc((size_t)pf * 4);
        a.partial = part.f(), a.partial_floats = pf;
    }
    small_attention(a, nullptr);
    IRX_HIP(hipDeviceSynchronize());
    if (reps > 0) {
        hipEvent_t e0, e1;
        IRX_HIP(hipEventCreate(&e0));
        IRX_HIP(hipEventCreate(&e1));
        IRX_HIP(hipEventRecord(e0, nullptr));
        for (int r = 0; r < reps; ++r) small_attention(a, nullptr);
        IRX_HIP(hipEventRecord(e1, nullptr));
        IRX_HIP(hipEventSynchronize(e1));
        float total = 0.f;
        IRX_HIP(hipEventElapsedTime(&total, e0, e1));
        *ms = total / (float)reps;
        IRX_HIP(hipEventDestroy(e0));
        IRX_HIP(hipEventDestroy(e1));
    }
    IRX_HIP(hipMemcpy(out, dout.p, qn * 4, hipMemcpyDeviceToHost));
}

}  // namespace

int irx_test_small_attention_tokens(irx_device *device, int method, const float *q, const float *k, const float *v,
                                    const float *rope_cos, const float *rope_sin, size_t seqs, size_t heads,
                                    size_t query_rows, size_t rows, float *out, int reps, float *ms_per_launch) {
    return guarded("irx_test_small_attention_tokens", [&] {
        test_small_attention_tokens(device, method, q, k, v, rope_cos, rope_sin, seqs, heads, query_rows, rows, out,
                                    reps, ms_per_launch);
    });
}

int irx_test_small_attention(irx_device *device, const float *q, const float *k, const float *v, size_t heads,
                             size_t query_rows, size_t rows, float *out) {
    return guarded("irx_test_small_attention", [&] {
        test_small_attention(device, q, k, v, nullptr, nullptr, heads, query_rows, rows, out);
    });
}

int irx_test_small_attention_rope(irx_device *device, const float *q, const float *k, const float *v,
                                  const float *rope_cos, const float *rope_sin, size_t heads, size_t query_rows,
                                  size_t rows, float *out) {
    return guarded("irx_test_small_attention_rope", [&] {
        if (!rope_cos || !rope_sin) fail(IRX_INVALID_ARGUMENT, "RoPE tables are missing");
        test_small_attention(device, q, k, v, rope_cos, rope_sin, heads, query_rows, rows, out);
    });
}

}  // extern "C"

// ---- TabICL preprocessing (preprocess.rs fit_feature / transform / ensemble_rows) ----

namespace {

constexpr size_t kFitScratchBytes = size_t(4) << 30;  // features fitted per launch: their f64 scratch

const char *fit_error(int status) {
    switch (status) {
        case 2: return "Yeo-Johnson bounds are not finite";
        case 3: return "the power transform of the training data is not finite";
        default: return "Training data produced non-finite preprocessing statistics";
    }
}

void check_methods(const int *methods, size_t groups) {
    if (!methods || groups < 1 || groups > 2) fail(IRX_INVALID_ARGUMENT, "one or two normalization groups are needed");
    for (size_t g = 0; g < groups; ++g)
        if (methods[g] != 0 && methods[g] != 1) fail(IRX_INVALID_ARGUMENT, "normalization method must be 0 (none) or 1 (power)");
    if (groups == 2 && methods[0] == methods[1]) fail(IRX_INVALID_ARGUMENT, "normalization groups must be unique");
}

void check_kept(const uint32_t *kept, size_t kept_count, size_t columns) {
    if (!kept || !kept_count || kept_count > columns) fail(IRX_INVALID_ARGUMENT, "kept features are invalid");
    for (size_t k = 0; k < kept_count; ++k)
        if (kept[k] >= columns || (k && kept[k] <= kept[k - 1]))
            fail(IRX_INVALID_ARGUMENT, "kept features must be increasing column indices");
}

}  // namespace

struct irx_preprocessor {
    irx_device *device = nullptr;
    size_t columns = 0;
    int kept_count = 0, groups = 0, members = 0;
    int methods[2] = {0, 0};
    DevBuf kept, stats, member_groups, orders;
    hipStream_t stream = nullptr;
    std::mutex mu;
    DevBuf x, group_rows, flags, members_out;  // grow-only workspaces
};

int irx_preprocess_fit(irx_device *device, const void *x, int x_f64, size_t rows, size_t columns,
                       const uint32_t *kept, size_t kept_count, const int *methods, size_t groups,
                       double outlier_threshold, double *statistics) {
    return guarded("irx_preprocess_fit", [&] {
        if (!device || !x || !statistics || rows < 2 || !columns)
            fail(IRX_INVALID_ARGUMENT, "preprocessing needs at least two training rows");
        check_kept(kept, kept_count, columns);
        check_methods(methods, groups);
        if (!(outlier_threshold > 0.0 && std::isfinite(outlier_threshold)))
            fail(IRX_INVALID_ARGUMENT, "outlier_threshold must be positive and finite");
        set_device(device);
        const size_t elem = x_f64 ? 8 : 4;
        DevBuf dx(rows * columns * elem), dkept(kept_count * 4), dstats(groups * 9 * kept_count * 8),
            dstatus(kept_count * 4);
        IRX_HIP(hipMemcpy(dx.p, x, rows * columns * elem, hipMemcpyHostToDevice));
        IRX_HIP(hipMemcpy(dkept.p, kept, kept_count * 4, hipMemcpyHostToDevice));
        const size_t per_feature = 3 * rows * 8;
        const int batch = (int)std::max<size_t>(1, std::min<size_t>(kept_count, kFitScratchBytes / per_feature));
        DevBuf scratch(batch * per_feature);
        PreprocessFit p{};
        p.x = dx.p, p.x_f64 = x_f64 ? 1 : 0, p.rows = (long long)rows, p.columns = (long long)columns;
        p.kept = static_cast<const unsigned *>(dkept.p), p.kept_count = (int)kept_count, p.groups = (int)groups;
        p.methods[0] = methods[0], p.methods[1] = groups > 1 ? methods[1] : 0;
        p.threshold = outlier_threshold, p.scratch = static_cast<double *>(scratch.p), p.batch = batch;
        p.stats = static_cast<double *>(dstats.p), p.status = static_cast<int *>(dstatus.p);
        preprocess_fit(p, nullptr);
        std::vector<int> status(kept_count);
        IRX_HIP(hipMemcpy(status.data(), dstatus.p, kept_count * 4, hipMemcpyDeviceToHost));
        for (int s : status)
            if (s) fail(IRX_INVALID_ARGUMENT, fit_error(s));
        IRX_HIP(hipMemcpy(statistics, dstats.p, groups * 9 * kept_count * 8, hipMemcpyDeviceToHost));
    });
}

int irx_preprocessor_new(irx_device *device, size_t columns, const uint32_t *kept, size_t kept_count,
                         const int *methods, size_t groups, const double *statistics, size_t members,
                         const uint32_t *member_groups, const uint32_t *feature_orders, irx_preprocessor **out) {
    if (out) *out = nullptr;
    return guarded("irx_preprocessor_new", [&] {
        if (!device || !out || !statistics || !member_groups || !feature_orders || !members || members > 4096)
            fail(IRX_INVALID_ARGUMENT, "preprocessor needs statistics and 1..=4096 members");
        check_kept(kept, kept_count, columns);
        check_methods(methods, groups);
        for (size_t i = 0; i < groups * 9 * kept_count; ++i)
            if (!std::isfinite(statistics[i])) fail(IRX_INVALID_ARGUMENT, "preprocessing statistics must be finite");
        std::vector<char> seen(kept_count);
        for (size_t b = 0; b < members; ++b) {
            if (member_groups[b] >= groups) fail(IRX_INVALID_ARGUMENT, "a member's group is out of range");
            std::fill(seen.begin(), seen.end(), 0);
            for (size_t j = 0; j < kept_count; ++j) {
                const uint32_t f = feature_orders[b * kept_count + j];
                if (f >= kept_count || seen[f]) fail(IRX_INVALID_ARGUMENT, "a member's feature order is not a permutation");
                seen[f] = 1;
            }
        }
        set_device(device);
        auto P = std::make_unique<irx_preprocessor>();
        P->columns = columns, P->kept_count = (int)kept_count, P->groups = (int)groups, P->members = (int)members;
        P->methods[0] = methods[0], P->methods[1] = groups > 1 ? methods[1] : 0;
        P->kept.alloc(kept_count * 4);
        P->stats.alloc(groups * 9 * kept_count * 8);
        P->member_groups.alloc(members * 4);
        P->orders.alloc(members * kept_count * 4);
        IRX_HIP(hipMemcpy(P->kept.p, kept, kept_count * 4, hipMemcpyHostToDevice));
        IRX_HIP(hipMemcpy(P->stats.p, statistics, groups * 9 * kept_count * 8, hipMemcpyHostToDevice));
        IRX_HIP(hipMemcpy(P->member_groups.p, member_groups, members * 4, hipMemcpyHostToDevice));
        IRX_HIP(hipMemcpy(P->orders.p, feature_orders, members * kept_count * 4, hipMemcpyHostToDevice));
        P->stream = take_stream(device);
        device->refs.fetch_add(1);
        P->device = device;
        *out = P.release();
    });
}

void irx_preprocessor_free(irx_preprocessor *p) {
    if (!p) return;
    (void)hipSetDevice(p->device->ordinal);
    return_stream(p->device, p->stream);
    irx_device *d = p->device;
    delete p;
    device_release(d);
}

int irx_preprocessor_transform(irx_preprocessor *p, const void *x, int x_f64, size_t rows, size_t chunk_rows,
                               int members_out, float *out, int out_on_device) {
    return guarded("irx_preprocessor_transform", [&] {
        if (!p || !x || !out || !rows || !chunk_rows) fail(IRX_INVALID_ARGUMENT, "transform needs rows and a chunk size");
        std::lock_guard<std::mutex> lock(p->mu);
        set_device(p->device);
        const size_t elem = x_f64 ? 8 : 4, kept = p->kept_count;
        const size_t xbytes = rows * p->columns * elem, gbytes = p->groups * rows * kept * 4;
        const size_t chunks = (rows + chunk_rows - 1) / chunk_rows, nflags = chunks * p->groups;
        auto grow = [](DevBuf &b, size_t bytes) {
            if (b.bytes < bytes) b.alloc(bytes);
        };
        grow(p->x, xbytes);
        grow(p->group_rows, gbytes);
        grow(p->flags, (2 * nflags + 1) * 4);
        IRX_HIP(hipMemcpyAsync(p->x.p, x, xbytes, hipMemcpyHostToDevice, p->stream));
        int *overflow = static_cast<int *>(p->flags.p), *again = overflow + nflags, *nonfinite = again + nflags;
        IRX_HIP(hipMemsetAsync(p->flags.p, 0, (2 * nflags + 1) * 4, p->stream));
        PreprocessTransform t{};
        t.x = p->x.p, t.x_f64 = x_f64 ? 1 : 0, t.rows = (long long)rows, t.columns = (long long)p->columns;
        t.kept = static_cast<const unsigned *>(p->kept.p), t.kept_count = p->kept_count, t.groups = p->groups;
        t.methods[0] = p->methods[0], t.methods[1] = p->methods[1];
        t.stats = static_cast<const double *>(p->stats.p), t.chunk_rows = (long long)chunk_rows;
        t.redo = nullptr, t.overflow = overflow, t.nonfinite = nonfinite, t.out = p->group_rows.f();
        preprocess_transform(t, p->stream);
        std::vector<int> flags(nflags);
        IRX_HIP(hipMemcpyAsync(flags.data(), overflow, nflags * 4, hipMemcpyDeviceToHost, p->stream));
        IRX_HIP(hipStreamSynchronize(p->stream));
        if (std::any_of(flags.begin(), flags.end(), [](int f) { return f != 0; })) {
            // TabICL's fallback: clip the overflowing chunk's rows to the
            // training range and transform that group's chunk again.
            t.redo = overflow, t.overflow = again;
            preprocess_transform(t, p->stream);
            IRX_HIP(hipMemcpyAsync(flags.data(), again, nflags * 4, hipMemcpyDeviceToHost, p->stream));
            IRX_HIP(hipStreamSynchronize(p->stream));
            if (std::any_of(flags.begin(), flags.end(), [](int f) { return f != 0; }))
                fail(IRX_INVALID_ARGUMENT, "the power transform overflows even within the training range");
        }
        int bad = 0;
        IRX_HIP(hipMemcpyAsync(&bad, nonfinite, 4, hipMemcpyDeviceToHost, p->stream));
        IRX_HIP(hipStreamSynchronize(p->stream));
        if (bad) fail(IRX_INVALID_ARGUMENT, "Preprocessing produced non-finite FP32 values");
        if (!members_out) {
            IRX_HIP(hipMemcpyAsync(out, p->group_rows.p, gbytes, out_on_device ? hipMemcpyDeviceToDevice
                                                                                 : hipMemcpyDeviceToHost, p->stream));
        } else {
            const size_t mbytes = (size_t)p->members * rows * kept * 4;
            float *dst = out;
            if (!out_on_device) {
                grow(p->members_out, mbytes);
                dst = p->members_out.f();
            }
            preprocess_gather(p->group_rows.f(), (long long)rows, p->kept_count, p->members,
                              static_cast<const unsigned *>(p->member_groups.p),
                              static_cast<const unsigned *>(p->orders.p), dst, p->stream);
            if (!out_on_device) IRX_HIP(hipMemcpyAsync(out, dst, mbytes, hipMemcpyDeviceToHost, p->stream));
        }
        IRX_HIP(hipStreamSynchronize(p->stream));
    });
}

int irx_test_power_fit(irx_device *device, const double *x, size_t rows, size_t columns, double *lambda_mean_scale,
                       double *fitted) {
    return guarded("irx_test_power_fit", [&] {
        if (!device || !x || !lambda_mean_scale || rows < 2 || !columns)
            fail(IRX_INVALID_ARGUMENT, "power fit needs at least two rows");
        set_device(device);
        std::vector<uint32_t> kept(columns);
        for (size_t c = 0; c < columns; ++c) kept[c] = (uint32_t)c;
        DevBuf dx(rows * columns * 8), dkept(columns * 4), dstats(9 * columns * 8), dstatus(columns * 4),
            scratch(columns * 3 * rows * 8), dfit(columns * rows * 8);
        IRX_HIP(hipMemcpy(dx.p, x, rows * columns * 8, hipMemcpyHostToDevice));
        IRX_HIP(hipMemcpy(dkept.p, kept.data(), columns * 4, hipMemcpyHostToDevice));
        PreprocessFit p{};
        p.x = dx.p, p.x_f64 = 1, p.rows = (long long)rows, p.columns = (long long)columns;
        p.kept = static_cast<const unsigned *>(dkept.p), p.kept_count = (int)columns, p.groups = 1;
        p.methods[0] = 1, p.threshold = 4.0, p.scratch = static_cast<double *>(scratch.p), p.batch = (int)columns;
        p.stats = static_cast<double *>(dstats.p), p.status = static_cast<int *>(dstatus.p);
        p.raw = 1, p.fitted = static_cast<double *>(dfit.p);
        preprocess_fit(p, nullptr);
        std::vector<int> status(columns);
        std::vector<double> stats(9 * columns);
        IRX_HIP(hipMemcpy(status.data(), dstatus.p, columns * 4, hipMemcpyDeviceToHost));
        IRX_HIP(hipMemcpy(stats.data(), dstats.p, 9 * columns * 8, hipMemcpyDeviceToHost));
        for (int s : status)
            if (s == 2 || s == 3) fail(IRX_INVALID_ARGUMENT, fit_error(s));
        for (size_t c = 0; c < columns; ++c)
            for (int i = 0; i < 3; ++i) lambda_mean_scale[i * columns + c] = stats[(6 + i) * columns + c];
        if (fitted) {
            // [columns, rows] on the device -> [rows, columns]
            std::vector<double> byc(columns * rows);
            IRX_HIP(hipMemcpy(byc.data(), dfit.p, columns * rows * 8, hipMemcpyDeviceToHost));
            for (size_t c = 0; c < columns; ++c)
                for (size_t r = 0; r < rows; ++r) fitted[r * columns + c] = byc[c * rows + r];
        }
    });
}

// serving.cpp -- the extern "C" entry points that answer from and shrink the
// KV cache: single-token decode over a batch, prompt weights, eviction.
// Argument checks and the launch; no allocation and no synchronisation once
// the context's device state is reserved.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>
#include <new>
#include <string>

#include "../epsp_kernels.h"
#include "epsp_host.h"

using namespace edge_prefill_b200;

namespace {

constexpr int32_t kOk = 0;
constexpr int32_t kInvalid = static_cast<int32_t>(ErrorCode::InvalidArgument);
constexpr int32_t kInternal = static_cast<int32_t>(ErrorCode::Internal);

// Families of ep_sp_profile_read_families.
enum Family { kDecode = 6, kPromptWeights = 7, kEvict = 8 };

// The context's device for the length of a call; the caller's is put back.
class DeviceGuard {
public:
    DeviceGuard() { ok_ = cudaGetDevice(&prev_) == cudaSuccess; }
    ~DeviceGuard() {
        if (ok_) cudaSetDevice(prev_);
    }
    DeviceGuard(const DeviceGuard&) = delete;
    DeviceGuard& operator=(const DeviceGuard&) = delete;

private:
    int prev_ = 0;
    bool ok_ = false;
};

// Rows of a sequence, at most: kernels round lengths up to tiles, and step past
// them, in 32 bits.
constexpr int32_t kMaxRows = INT_MAX - 65536;

bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// Device state and current device of a compute call.  Reserving allocates and
// synchronises, which a capturing stream cannot do.
int32_t enter(ep_sp_ctx* c, cudaStream_t s) {
    if (!c->reserved) {
        cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
        int n = 0;
        if (cudaGetDeviceCount(&n) == cudaSuccess && n > 0 &&
            cudaStreamIsCapturing(s, &cap) == cudaSuccess && cap != cudaStreamCaptureStatusNone)
            return ctx_fail(c, kInvalid, "ep_sp_reserve must run before a call is captured");
        cudaGetLastError();
        return ctx_ensure_device(c);
    }
    const cudaError_t e = cudaSetDevice(c->cfg.device);
    if (e != cudaSuccess) return ctx_fail(c, kInternal, std::string("cudaSetDevice: ") + cudaGetErrorString(e));
    return kOk;
}

template <class F>
int32_t launch(ep_sp_ctx* c, Family f, void* stream, const char* what, F&& go) {
    void* ev = ctx_profile_begin(c, f, stream);
    const cudaError_t e = go();
    ctx_profile_end(c, f, ev, stream);
    if (e != cudaSuccess) return ctx_fail(c, kInternal, std::string(what) + ": " + cudaGetErrorString(e));
    return kOk;
}

// Layout rules of one batch; `min_rows` is what each sequence must have room for.
int32_t check_batch(ep_sp_ctx* c, const ep_sp_kv_batch* b, int32_t min_rows, bool need_lens, const char* who,
                    epsp::BatchKv* out) {
    auto bad = [&](const char* what) { return ctx_fail(c, kInvalid, std::string(who) + ": " + what); };
    if (!b) return bad("null batch");
    if (b->n_seq < 1 || b->n_seq > 65535) return bad("n_seq must lie in [1, 65535]");
    if (b->max_kv_len < 1 || b->max_kv_len > c->cfg.max_ctx)
        return bad("max_kv_len must lie in [1, max_ctx]");
    if (b->max_kv_len > kMaxRows) return bad("max_kv_len is more than 32 bits can round up");
    if (need_lens && !b->kv_lens) return bad("null kv_lens");
    if (!aligned(b->kv_lens, 4) || (b->block_rows != 0 && !aligned(b->block_tables, 4)))
        return bad("kv_lens and block_tables must be 4-byte aligned");
    const int32_t rows = std::max(min_rows, 1);
    out->n_seq = b->n_seq;
    out->max_kv_len = b->max_kv_len;
    out->lens = b->kv_lens;
    if (b->block_rows == 0) {
        if (b->seq_rows < rows) return bad("seq_rows does not cover max_kv_len rows");
        const int64_t all = (int64_t)b->n_seq * b->seq_rows;
        if (all > INT_MAX) return bad("more than 2^31 - 1 cache rows");
        out->seq_rows = b->seq_rows;
        out->rows = (int32_t)all;
        return kOk;
    }
    if (b->block_rows < 0 || b->block_rows % c->cfg.page_size)
        return bad("block_rows must be a multiple of the page size");
    if (!b->block_tables || b->pool_rows < b->block_rows || b->pool_rows % b->block_rows)
        return bad("block tables and a pool of whole blocks are needed");
    if (b->table_stride < 1 || (int64_t)b->table_stride * b->block_rows < rows)
        return bad("the block tables do not cover max_kv_len rows");
    out->tables = b->block_tables;
    out->table_stride = b->table_stride;
    out->block_rows = b->block_rows;
    out->rows = b->pool_rows;
    return kOk;
}

int32_t check_workspace(ep_sp_ctx* c, const void* ws, size_t have, size_t need) {
    if (need == 0) return kOk;
    if (need == SIZE_MAX) return ctx_fail(c, kInvalid, "more cache rows than one call takes");
    if (!ws || have < need)
        return ctx_fail(c, kInvalid, "the workspace holds " + std::to_string(ws ? have : 0) + " bytes, the call needs " +
                                         std::to_string(need));
    if (!aligned(ws, 16)) return ctx_fail(c, kInvalid, "the workspace must be 16-byte aligned");
    return kOk;
}

int32_t elem_bytes(int32_t dtype) { return dtype == EP_SP_F32 ? 4 : 2; }

// Rows of the layer have moved or been written past the context's knowledge:
// page sums, V sums and f16 shadows start over at its next prefill call.
void forget_layer(ep_sp_ctx* c, int32_t layer) {
    const size_t at = (size_t)layer * c->cfg.n_head_kv;
    std::fill_n(c->pooled.begin() + at, c->cfg.n_head_kv, 0);
    std::fill_n(c->v_pooled.begin() + at, c->cfg.n_head_kv, 0);
    c->shadowed[layer] = 0;
    c->sel_valid = false;
}

// No exception crosses the ABI.
template <class F>
int32_t guarded(F&& f) noexcept {
    try {
        return f();
    } catch (const std::bad_alloc&) {
        return static_cast<int32_t>(ErrorCode::OutOfMemory);
    } catch (...) {
        return kInternal;
    }
}

}  // namespace

extern "C" {

int32_t ep_sp_decode_bytes(const ep_sp_ctx* ctx, int32_t n_seq, int32_t max_kv_len, int32_t with_acc, size_t* bytes) {
    if (!ctx || !bytes || n_seq < 1 || n_seq > 65535 || max_kv_len < 1 || max_kv_len > std::min(ctx->cfg.max_ctx, kMaxRows) ||
        (with_acc != 0 && with_acc != 1))
        return kInvalid;
    const ep_sp_config& c = ctx->cfg;
    *bytes = epsp::decode_ws_bytes(n_seq, max_kv_len, c.n_head, c.n_head_kv, c.head_dim, c.dtype, with_acc != 0);
    if (*bytes == SIZE_MAX) return kInvalid;
    return kOk;
}

int32_t ep_sp_decode_layer(ep_sp_ctx* ctx, int32_t layer, const ep_sp_kv_batch* kv, const void* q, const void* k_new,
                           const void* v_new, void* k, void* v, void* out, float* acc, int32_t acc_stride,
                           void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int32_t {
        if (!ctx) return kInvalid;
        const ep_sp_config& c = ctx->cfg;
        if (layer < 0 || layer >= c.n_layer) return ctx_fail(ctx, kInvalid, "layer out of range");
        epsp::DecodeArgs a{};
        int32_t rc = check_batch(ctx, kv, kv ? kv->max_kv_len : 0, true, "decode", &a.kv);
        if (rc) return rc;
        if (!q || !k || !v || !out) return ctx_fail(ctx, kInvalid, "null tensor");
        if ((k_new != nullptr) != (v_new != nullptr)) return ctx_fail(ctx, kInvalid, "k_new and v_new go together");
        for (const void* p : {q, static_cast<const void*>(k), static_cast<const void*>(v), static_cast<const void*>(out),
                              k_new, v_new})
            if (!aligned(p, 16)) return ctx_fail(ctx, kInvalid, "tensors must be 16-byte aligned");
        if (acc && (acc_stride < kv->max_kv_len || !aligned(acc, 4)))
            return ctx_fail(ctx, kInvalid, "acc_stride smaller than max_kv_len");
        rc = check_workspace(ctx, workspace, workspace_bytes,
                             epsp::decode_ws_bytes(kv->n_seq, kv->max_kv_len, c.n_head, c.n_head_kv, c.head_dim,
                                                   c.dtype, acc != nullptr));
        if (rc) return rc;
        DeviceGuard guard;
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if ((rc = enter(ctx, s))) return rc;
        a.q = q;
        a.k = k;
        a.v = v;
        a.k_new = k_new;
        a.v_new = v_new;
        a.out = out;
        a.dtype = c.dtype;
        a.out_dtype = c.out_dtype;
        a.n_head = c.n_head;
        a.n_head_kv = c.n_head_kv;
        a.head_dim = c.head_dim;
        a.kq_scale = c.kq_scale;
        a.acc = acc;
        a.acc_stride = acc_stride;
        a.ws = workspace;
        a.err = ctx->d_err;
        a.timeout_ns = ctx->timeout_ns;
        rc = launch(ctx, kDecode, stream, "decode", [&] { return epsp::launch_decode(a, s); });
        if (rc == kOk && k_new) forget_layer(ctx, layer);  // where the rows went only the device knows
        return rc;
    });
}

int32_t ep_sp_prompt_weights_bytes(const ep_sp_ctx* ctx, int32_t kv_len, int32_t n_tok, int32_t row_begin,
                                   size_t* bytes) {
    if (!ctx || !bytes || n_tok < 1 || kv_len < n_tok || kv_len > std::min(ctx->cfg.max_ctx, kMaxRows) || row_begin < 0 ||
        row_begin >= n_tok)
        return kInvalid;
    *bytes = epsp::weights_ws_bytes(kv_len, n_tok - row_begin, ctx->cfg.n_head, ctx->cfg.n_head_kv, ctx->cfg.head_dim,
                                    ctx->cfg.dtype);
    if (*bytes == SIZE_MAX) return kInvalid;
    return kOk;
}

int32_t ep_sp_prompt_weights(ep_sp_ctx* ctx, int32_t layer, const void* q, const void* k, int32_t kv_len,
                             int32_t n_tok, int32_t row_begin, int32_t accumulate, float* acc, int32_t acc_stride,
                             void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int32_t {
        if (!ctx) return kInvalid;
        const ep_sp_config& c = ctx->cfg;
        if (layer < 0 || layer >= c.n_layer) return ctx_fail(ctx, kInvalid, "layer out of range");
        if (!q || !k || !acc) return ctx_fail(ctx, kInvalid, "null tensor");
        if (!aligned(q, 16) || !aligned(k, 16) || !aligned(acc, 4))
            return ctx_fail(ctx, kInvalid, "q and k must be 16-byte aligned");
        if (n_tok < 1 || kv_len < n_tok || kv_len > std::min(c.max_ctx, kMaxRows))
            return ctx_fail(ctx, kInvalid, "bad kv_len / n_tok");
        if (row_begin < 0 || row_begin >= n_tok) return ctx_fail(ctx, kInvalid, "row_begin must lie in [0, n_tok)");
        if (accumulate != 0 && accumulate != 1) return ctx_fail(ctx, kInvalid, "accumulate must be 0 or 1");
        if (acc_stride < kv_len) return ctx_fail(ctx, kInvalid, "acc_stride smaller than kv_len");
        if (ctx->paging.block_rows > 0 && (int64_t)ctx->paging.n_entries * ctx->paging.block_rows < kv_len)
            return ctx_fail(ctx, kInvalid, "the block table does not cover kv_len rows");
        int32_t rc = check_workspace(ctx, workspace, workspace_bytes,
                                     epsp::weights_ws_bytes(kv_len, n_tok - row_begin, c.n_head, c.n_head_kv, c.head_dim,
                                                            c.dtype));
        if (rc) return rc;
        DeviceGuard guard;
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if ((rc = enter(ctx, s))) return rc;
        epsp::WeightArgs a{};
        a.q = q;
        a.k = k;
        a.paging = ctx->paging;
        a.dtype = c.dtype;
        a.n_head = c.n_head;
        a.n_head_kv = c.n_head_kv;
        a.head_dim = c.head_dim;
        a.page_size = c.page_size;
        a.kv_len = kv_len;
        a.n_tok = n_tok;
        a.row_begin = row_begin;
        a.kq_scale = c.kq_scale;
        a.accumulate = accumulate;
        a.acc = acc;
        a.acc_stride = acc_stride;
        a.ws = workspace;
        a.err = ctx->d_err;
        a.timeout_ns = ctx->timeout_ns;
        return launch(ctx, kPromptWeights, stream, "prompt weights", [&] { return epsp::launch_prompt_weights(a, s); });
    });
}

int32_t ep_sp_evict_bytes(const ep_sp_ctx* ctx, int32_t n_seq, int32_t max_kv_len, int32_t n_keep, size_t* bytes) {
    if (!ctx || !bytes || n_seq < 1 || n_seq > 65535 || max_kv_len < 1 || max_kv_len > std::min(ctx->cfg.max_ctx, kMaxRows) ||
        n_keep < 1 || n_keep > ctx->cfg.max_ctx)
        return kInvalid;
    *bytes = epsp::evict_ws_bytes(n_seq, max_kv_len, n_keep, ctx->cfg.n_head_kv);
    return kOk;
}

int32_t ep_sp_evict_layer(ep_sp_ctx* ctx, int32_t layer, const ep_sp_kv_batch* src, const void* k, const void* v,
                          const float* acc, int32_t acc_stride, int32_t n_keep, int32_t sink_rows,
                          int32_t recent_rows, const ep_sp_kv_batch* dst, void* k_dst, void* v_dst, float* acc_dst,
                          int32_t acc_dst_stride, int32_t* new_lens, int32_t* kept_rows, void* workspace,
                          size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int32_t {
        if (!ctx) return kInvalid;
        const ep_sp_config& c = ctx->cfg;
        if (layer < 0 || layer >= c.n_layer) return ctx_fail(ctx, kInvalid, "layer out of range");
        if (n_keep < 1 || n_keep > c.max_ctx) return ctx_fail(ctx, kInvalid, "n_keep must lie in [1, max_ctx]");
        if (sink_rows < 0 || recent_rows < 0 || (int64_t)sink_rows + recent_rows > n_keep)
            return ctx_fail(ctx, kInvalid, "sink_rows + recent_rows must lie in [0, n_keep]");
        epsp::EvictArgs a{};
        int32_t rc = check_batch(ctx, src, src ? src->max_kv_len : 0, true, "eviction source", &a.src);
        if (rc) return rc;
        const int32_t most = std::min(n_keep, src->max_kv_len);  // rows a sequence can keep
        if ((rc = check_batch(ctx, dst, most, false, "eviction destination", &a.dst))) return rc;
        if (dst->n_seq != src->n_seq) return ctx_fail(ctx, kInvalid, "source and destination n_seq differ");
        if (dst->max_kv_len < most)
            return ctx_fail(ctx, kInvalid, "the destination's max_kv_len is smaller than n_keep");
        if (!k || !v || !acc || !k_dst || !v_dst) return ctx_fail(ctx, kInvalid, "null tensor");
        for (const void* p : {k, v, static_cast<const void*>(k_dst), static_cast<const void*>(v_dst)})
            if (!aligned(p, 16)) return ctx_fail(ctx, kInvalid, "tensors must be 16-byte aligned");
        if (acc_stride < src->max_kv_len || !aligned(acc, 4))
            return ctx_fail(ctx, kInvalid, "acc_stride smaller than max_kv_len");
        if (acc_dst && (acc_dst_stride < most || !aligned(acc_dst, 4)))
            return ctx_fail(ctx, kInvalid, "acc_dst_stride smaller than the rows kept");
        if (!aligned(new_lens, 4) || !aligned(kept_rows, 4))
            return ctx_fail(ctx, kInvalid, "new_lens and kept_rows must be 4-byte aligned");
        if (acc_dst == acc && acc_dst_stride != acc_stride)
            return ctx_fail(ctx, kInvalid, "acc_dst may be acc only with the same stride");
        const bool same_layout = a.src.block_rows == a.dst.block_rows && a.src.tables == a.dst.tables &&
                                 a.src.table_stride == a.dst.table_stride && a.src.seq_rows == a.dst.seq_rows &&
                                 a.src.rows == a.dst.rows;
        if (k_dst == v_dst && k != v) return ctx_fail(ctx, kInvalid, "K and V would go to the same rows");
        if ((k_dst == k) != (v_dst == v) || k_dst == v || v_dst == k)
            return ctx_fail(ctx, kInvalid, "K and V are either both compacted in place or both gathered elsewhere");
        a.in_place = k_dst == k && same_layout;
        if (k_dst == k && !a.in_place && (a.src.block_rows == 0 || a.dst.block_rows == 0 || a.src.tables == a.dst.tables))
            return ctx_fail(ctx, kInvalid, "in place, the source's and the destination's layout must be the same");
        rc = check_workspace(ctx, workspace, workspace_bytes,
                             epsp::evict_ws_bytes(src->n_seq, src->max_kv_len, n_keep, c.n_head_kv));
        if (rc) return rc;
        DeviceGuard guard;
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if ((rc = enter(ctx, s))) return rc;
        a.k = k;
        a.v = v;
        a.acc = acc;
        a.acc_stride = acc_stride;
        a.n_keep = n_keep;
        a.sink_rows = sink_rows;
        a.recent_rows = recent_rows;
        a.k_dst = k_dst;
        a.v_dst = v_dst;
        a.acc_dst = acc_dst;
        a.acc_dst_stride = acc_dst_stride;
        a.new_lens = new_lens;
        a.kept_rows = kept_rows;
        a.n_head_kv = c.n_head_kv;
        a.head_dim = c.head_dim;
        a.elem_bytes = elem_bytes(c.dtype);
        a.ws = workspace;
        a.err = ctx->d_err;
        rc = launch(ctx, kEvict, stream, "eviction", [&] { return epsp::launch_evict(a, s); });
        if (rc) return rc;
        forget_layer(ctx, layer);
        return kOk;
    });
}

}  // extern "C"

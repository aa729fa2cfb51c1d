// cache8.cpp -- the extern "C" entry points of the cache in 8 bits: pack, unpack,
// decode.  Argument checks and the launch.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "../epsp_kernels.h"
#include "serving_checks.h"

using namespace edge_prefill_b200;

namespace {

// The 8-bit cache of a checked batch.
int32_t check_cache8(ep_sp_ctx* c, const ep_sp_kv8* q, const epsp::BatchKv& b, const char* who, epsp::Cache8* out) {
    auto bad = [&](const char* what) { return ctx_fail(c, kInvalid, std::string(who) + ": " + what); };
    if (!q) return bad("null 8-bit cache");
    if (q->type != EP_SP_E4M3 && q->type != EP_SP_I8) return bad("the 8-bit type must be EP_SP_E4M3 or EP_SP_I8");
    if (!q->k || !q->v || !q->k_scale || !q->v_scale) return bad("null tensor of the 8-bit cache");
    if (!aligned(q->k, 16) || !aligned(q->v, 16)) return bad("tensors must be 16-byte aligned");
    if (!aligned(q->k_scale, 4) || !aligned(q->v_scale, 4)) return bad("scales must be 4-byte aligned");
    if (q->k == q->v || q->k_scale == q->v_scale) return bad("K and V must be two tensors");
    if (b.block_rows == 0 && b.seq_rows % c->cfg.page_size)
        return bad("seq_rows must be a multiple of the page size (a page has one scale)");
    out->i8 = q->type == EP_SP_I8;
    out->page_size = c->cfg.page_size;
    out->k = static_cast<uint8_t*>(q->k);
    out->v = static_cast<uint8_t*>(q->v);
    out->k_scale = q->k_scale;
    out->v_scale = q->v_scale;
    return kOk;
}

// What pack and unpack have in common; `to8`: the 8-bit cache is the destination.
int32_t convert(ep_sp_ctx* ctx, int32_t layer, const ep_sp_kv_batch* src, const ep_sp_kv_batch* dst, const void* k,
                const void* v, const ep_sp_kv8* cache, const int32_t* first, bool to8, void* stream) {
    const char* what = to8 ? "pack" : "unpack";
    if (!ctx) return kInvalid;
    const ep_sp_config& c = ctx->cfg;
    if (layer < 0 || layer >= c.n_layer) return ctx_fail(ctx, kInvalid, "layer out of range");
    epsp::PackArgs a{};
    int32_t rc = check_batch(ctx, src, src ? src->max_kv_len : 0, true, to8 ? "pack source" : "unpack source", &a.src);
    if (rc) return rc;
    rc = check_batch(ctx, dst, src->max_kv_len, false, to8 ? "pack destination" : "unpack destination", &a.dst);
    if (rc) return rc;
    if (dst->n_seq != src->n_seq) return ctx_fail(ctx, kInvalid, "source and destination n_seq differ");
    if ((rc = check_cache8(ctx, cache, to8 ? a.dst : a.src, what, &a.c))) return rc;
    if (!k || !v) return ctx_fail(ctx, kInvalid, "null tensor");
    if (!aligned(k, 16) || !aligned(v, 16)) return ctx_fail(ctx, kInvalid, "tensors must be 16-byte aligned");
    if (!to8 && k == v) return ctx_fail(ctx, kInvalid, "K and V would go to the same rows");
    if (!aligned(first, 4)) return ctx_fail(ctx, kInvalid, "first must be 4-byte aligned");
    for (const void* p : {k, v})
        if (p == cache->k || p == cache->v) return ctx_fail(ctx, kInvalid, "the 8-bit cache is a tensor of its own");
    DeviceGuard guard;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if ((rc = enter(ctx, s))) return rc;
    a.first = first;
    a.k = k;
    a.v = v;
    a.dtype = c.dtype;
    a.n_head_kv = c.n_head_kv;
    a.head_dim = c.head_dim;
    a.err = ctx->d_err;
    rc = launch(ctx, kPack, stream, what, [&] { return to8 ? epsp::launch_pack(a, s) : epsp::launch_unpack(a, s); });
    if (rc == kOk && !to8) forget_layer(ctx, layer);
    return rc;
}

}  // namespace

extern "C" {

int32_t ep_sp_pack_kv(ep_sp_ctx* ctx, int32_t layer, const ep_sp_kv_batch* src, const void* k, const void* v,
                      const int32_t* first, const ep_sp_kv_batch* dst, const ep_sp_kv8* cache, void* stream) {
    return guarded([&] { return convert(ctx, layer, src, dst, k, v, cache, first, true, stream); });
}

int32_t ep_sp_unpack_kv(ep_sp_ctx* ctx, int32_t layer, const ep_sp_kv_batch* src, const ep_sp_kv8* cache,
                        const int32_t* first, const ep_sp_kv_batch* dst, void* k, void* v, void* stream) {
    return guarded([&] { return convert(ctx, layer, src, dst, k, v, cache, first, false, stream); });
}

int32_t ep_sp_decode8_bytes(const ep_sp_ctx* ctx, int32_t n_seq, int32_t max_kv_len, size_t* bytes) {
    if (!ctx || !bytes || n_seq < 1 || n_seq > 65535 || max_kv_len < 1 || max_kv_len > std::min(ctx->cfg.max_ctx, kMaxRows))
        return kInvalid;
    const ep_sp_config& c = ctx->cfg;
    *bytes = epsp::decode8_ws_bytes(n_seq, max_kv_len, c.n_head, c.n_head_kv, c.head_dim, c.dtype);
    if (*bytes == SIZE_MAX) return kInvalid;
    return kOk;
}

int32_t ep_sp_decode8_layer(ep_sp_ctx* ctx, int32_t layer, const ep_sp_kv_batch* kv, const void* q, const void* k_new,
                            const void* v_new, const ep_sp_kv8* cache, void* out, void* workspace,
                            size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int32_t {
        if (!ctx) return kInvalid;
        const ep_sp_config& c = ctx->cfg;
        if (layer < 0 || layer >= c.n_layer) return ctx_fail(ctx, kInvalid, "layer out of range");
        epsp::DecodeArgs a{};
        epsp::Cache8 c8;
        int32_t rc = check_batch(ctx, kv, kv ? kv->max_kv_len : 0, true, "decode8", &a.kv);
        if (rc) return rc;
        if ((rc = check_cache8(ctx, cache, a.kv, "decode8", &c8))) return rc;
        if (!q || !out) return ctx_fail(ctx, kInvalid, "null tensor");
        if ((k_new != nullptr) != (v_new != nullptr)) return ctx_fail(ctx, kInvalid, "k_new and v_new go together");
        for (const void* p : {q, static_cast<const void*>(out), k_new, v_new})
            if (!aligned(p, 16)) return ctx_fail(ctx, kInvalid, "tensors must be 16-byte aligned");
        if (k_new && (int64_t)kv->n_seq * c.n_head_kv * 2 > INT_MAX)
            return ctx_fail(ctx, kInvalid, "more new rows than one call takes");
        rc = check_workspace(ctx, workspace, workspace_bytes,
                             epsp::decode8_ws_bytes(kv->n_seq, kv->max_kv_len, c.n_head, c.n_head_kv, c.head_dim, c.dtype));
        if (rc) return rc;
        DeviceGuard guard;
        cudaStream_t s = static_cast<cudaStream_t>(stream);
        if ((rc = enter(ctx, s))) return rc;
        a.q = q;
        a.k_new = k_new;
        a.v_new = v_new;
        a.out = out;
        a.dtype = c.dtype;
        a.out_dtype = c.out_dtype;
        a.n_head = c.n_head;
        a.n_head_kv = c.n_head_kv;
        a.head_dim = c.head_dim;
        a.kq_scale = c.kq_scale;
        a.ws = workspace;
        a.err = ctx->d_err;
        a.timeout_ns = ctx->timeout_ns;
        return launch(ctx, kDecode, stream, "decode8", [&] { return epsp::launch_decode8(a, c8, s); });
    });
}

}  // extern "C"

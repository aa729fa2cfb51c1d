// pages.cpp -- the extern "C" entry points that share, take, give back and move
// the blocks of paged caches.  Argument checks and the launches.
#include <cuda_runtime.h>

#include <climits>
#include <cstdint>
#include <vector>

#include "../epsp_kernels.h"
#include "serving_checks.h"

using namespace edge_prefill_b200;

namespace {

constexpr int32_t kMaxPools = 4096;

// Layout rules; the message is set where there is a context to hold it.
const char* wrong_pages(const ep_sp_config& c, const ep_sp_pages* p) {
    if (!p) return "null pages";
    if (p->n_seq < 1 || p->n_seq > 65535) return "n_seq must lie in [1, 65535]";
    if (p->block_rows < 1 || p->block_rows % c.page_size) return "block_rows must be a multiple of the page size";
    if (p->table_stride < 1 || (int64_t)p->table_stride * p->block_rows > kMaxRows)
        return "table_stride must be at least 1, and a table's rows fit 32 bits";
    // (the blocks that all sequences take are summed in 32 bits)
    if ((int64_t)p->n_seq * p->table_stride > INT_MAX) return "the tables have more than 2^31 - 1 entries";
    if (p->pool_blocks < 1 || p->pool_blocks > kMaxRows) return "pool_blocks must be at least 1";
    if (!p->kv_lens || !p->block_tables || !p->refs) return "null lengths, tables or counts";
    if (!aligned(p->kv_lens, 4) || !aligned(p->block_tables, 4) || !aligned(p->refs, 4))
        return "lengths, tables and counts must be 4-byte aligned";
    return nullptr;
}

epsp::PagesArgs args_of(const ep_sp_pages* p) {
    return {p->n_seq, p->table_stride, p->block_rows, p->pool_blocks, p->kv_lens, p->block_tables, p->refs, nullptr};
}

int32_t check_pages(ep_sp_ctx* ctx, const ep_sp_pages* p, const char* who, epsp::PagesArgs* a) {
    if (const char* what = wrong_pages(ctx->cfg, p)) return ctx_fail(ctx, kInvalid, std::string(who) + ": " + what);
    *a = args_of(p);
    return kOk;
}

int32_t check_pools(ep_sp_ctx* ctx, const ep_sp_pool* pools, int32_t n_pools, int32_t blocks, std::vector<epsp::Pool>* out) {
    if (!pools || n_pools < 1 || n_pools > kMaxPools) return ctx_fail(ctx, kInvalid, "n_pools must lie in [1, 4096]");
    out->resize(n_pools);
    for (int32_t i = 0; i < n_pools; ++i) {
        const ep_sp_pool& p = pools[i];
        if (!p.rows || !aligned(p.rows, 4) || p.block_bytes < 4 || p.block_bytes % 4 ||
            p.block_bytes > (size_t)PTRDIFF_MAX / blocks)
            return ctx_fail(ctx, kInvalid, "pool " + std::to_string(i) +
                                               ": rows must be there and 4-byte aligned, block_bytes a multiple of 4");
        (*out)[i] = {p.rows, p.block_bytes};
    }
    return kOk;
}

template <class F>
int32_t bytes_of(const ep_sp_ctx* ctx, const ep_sp_pages* pages, size_t* bytes, F&& f) {
    if (!ctx || !bytes || wrong_pages(ctx->cfg, pages)) return kInvalid;
    *bytes = f(args_of(pages));
    return kOk;
}

// What every call does once its arguments are checked.
template <class F>
int32_t run(ep_sp_ctx* ctx, epsp::PagesArgs& a, void* stream, const char* what, F&& go) {
    DeviceGuard guard;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int32_t rc = enter(ctx, s);
    if (rc) return rc;
    a.err = ctx->d_err;
    return launch(ctx, kPages, stream, what, [&] { return go(s); });
}

}  // namespace

extern "C" {

int32_t ep_sp_count_refs(ep_sp_ctx* ctx, const ep_sp_pages* pages, void* stream) {
    return guarded([&]() -> int32_t {
        if (!ctx) return kInvalid;
        epsp::PagesArgs a;
        const int32_t rc = check_pages(ctx, pages, "count", &a);
        if (rc) return rc;
        return run(ctx, a, stream, "count", [&](cudaStream_t s) { return epsp::launch_count_refs(a, s); });
    });
}

int32_t ep_sp_fork_bytes(const ep_sp_ctx* ctx, const ep_sp_pages* pages, size_t* bytes) {
    return bytes_of(ctx, pages, bytes, epsp::fork_ws_bytes);
}

int32_t ep_sp_fork_seqs(ep_sp_ctx* ctx, const ep_sp_pages* pages, const int32_t* parents, const int32_t* lens,
                        void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int32_t {
        if (!ctx) return kInvalid;
        epsp::PagesArgs a;
        int32_t rc = check_pages(ctx, pages, "fork", &a);
        if (rc) return rc;
        if (!parents || !aligned(parents, 4) || !aligned(lens, 4))
            return ctx_fail(ctx, kInvalid, "fork: parents must be there, parents and lens 4-byte aligned");
        if ((rc = check_workspace(ctx, workspace, workspace_bytes, epsp::fork_ws_bytes(a)))) return rc;
        rc = run(ctx, a, stream, "fork", [&](cudaStream_t s) { return epsp::launch_fork(a, parents, lens, workspace, s); });
        if (rc == kOk)
            for (int32_t l = 0; l < ctx->cfg.n_layer; ++l) forget_layer(ctx, l);
        return rc;
    });
}

int32_t ep_sp_resize_bytes(const ep_sp_ctx* ctx, const ep_sp_pages* pages, size_t* bytes) {
    return bytes_of(ctx, pages, bytes, epsp::resize_ws_bytes);
}

int32_t ep_sp_resize_seqs(ep_sp_ctx* ctx, const ep_sp_pages* pages, const int32_t* new_lens, const ep_sp_pool* pools,
                          int32_t n_pools, void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int32_t {
        if (!ctx) return kInvalid;
        epsp::PagesArgs a;
        int32_t rc = check_pages(ctx, pages, "resize", &a);
        if (rc) return rc;
        if (!new_lens || !aligned(new_lens, 4))
            return ctx_fail(ctx, kInvalid, "resize: new_lens must be there and 4-byte aligned");
        std::vector<epsp::Pool> list;
        if ((rc = check_pools(ctx, pools, n_pools, a.pool_blocks, &list))) return rc;
        if ((rc = check_workspace(ctx, workspace, workspace_bytes, epsp::resize_ws_bytes(a)))) return rc;
        return run(ctx, a, stream, "resize", [&](cudaStream_t s) {
            return epsp::launch_resize(a, new_lens, list.data(), n_pools, workspace, s);
        });
    });
}

int32_t ep_sp_compact_bytes(const ep_sp_ctx* ctx, const ep_sp_pages* pages, size_t* bytes) {
    return bytes_of(ctx, pages, bytes, epsp::compact_ws_bytes);
}

int32_t ep_sp_compact_pool(ep_sp_ctx* ctx, const ep_sp_pages* pages, const ep_sp_pool* pools, int32_t n_pools,
                           int32_t* n_used, void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&]() -> int32_t {
        if (!ctx) return kInvalid;
        epsp::PagesArgs a;
        int32_t rc = check_pages(ctx, pages, "compact", &a);
        if (rc) return rc;
        if (!aligned(n_used, 4)) return ctx_fail(ctx, kInvalid, "compact: n_used must be 4-byte aligned");
        std::vector<epsp::Pool> list;
        if ((rc = check_pools(ctx, pools, n_pools, a.pool_blocks, &list))) return rc;
        if ((rc = check_workspace(ctx, workspace, workspace_bytes, epsp::compact_ws_bytes(a)))) return rc;
        return run(ctx, a, stream, "compact", [&](cudaStream_t s) {
            return epsp::launch_compact(a, list.data(), n_pools, n_used, workspace, s);
        });
    });
}

}  // extern "C"

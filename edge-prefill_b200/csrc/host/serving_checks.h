// serving_checks.h -- what the entry points on a layer's cache share (serving.cpp,
// cache8.cpp, pages.cpp): the context's device for the length of a call, batch and
// workspace rules, timed launches, the guard against exceptions.
#pragma once

#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>
#include <new>
#include <string>

#include "../epsp_kernels.h"
#include "epsp_host.h"

namespace edge_prefill_b200 {

constexpr int32_t kOk = 0;
constexpr int32_t kInvalid = static_cast<int32_t>(ErrorCode::InvalidArgument);
constexpr int32_t kInternal = static_cast<int32_t>(ErrorCode::Internal);

// Families of ep_sp_profile_read_families and, from kPack on, of
// ep_sp_profile_read_family alone.
enum Family {
    kDecode = 6,
    kPromptWeights = 7,
    kEvict = 8,
    kPack = EP_SP_FAMILY_PACK,
    kPages = EP_SP_FAMILY_PAGES
};

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

inline bool aligned(const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// Device state and current device of a compute call.  Reserving allocates and
// synchronises, which a capturing stream cannot do.
inline int32_t enter(ep_sp_ctx* c, cudaStream_t s) {
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
inline int32_t check_batch(ep_sp_ctx* c, const ep_sp_kv_batch* b, int32_t min_rows, bool need_lens, const char* who,
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

inline int32_t check_workspace(ep_sp_ctx* c, const void* ws, size_t have, size_t need) {
    if (need == 0) return kOk;
    if (need == SIZE_MAX) return ctx_fail(c, kInvalid, "more cache rows than one call takes");
    if (!ws || have < need)
        return ctx_fail(c, kInvalid, "the workspace holds " + std::to_string(ws ? have : 0) + " bytes, the call needs " +
                                         std::to_string(need));
    if (!aligned(ws, 16)) return ctx_fail(c, kInvalid, "the workspace must be 16-byte aligned");
    return kOk;
}

inline int32_t elem_bytes(int32_t dtype) { return dtype == EP_SP_F32 ? 4 : 2; }

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

}  // namespace edge_prefill_b200

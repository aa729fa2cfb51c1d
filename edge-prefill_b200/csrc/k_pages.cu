// k_pages.cu -- K11: blocks of paged caches shared, taken, given back and moved.
//
//   fork     (length, table) of s <- the first lens[s] rows of parents[s], all at once
//   resize   blocks past the new lengths are given back, then the lowest free
//            blocks taken in order, sequence by sequence; a partly filled last
//            block that others hold too is copied before it grows
//   compact  the i-th block in use at or past n_used -> the i-th free one below it
//
// refs[b] counts the sequences that hold block b; every count and place comes
// from sums that do not depend on the order of the adding, so the results do not
// depend on timing.
//
// The planning is latency (a few dependent passes over refs and tables), the
// copies are bandwidth.  A plan runs in one CTA, on arrays in shared memory, or in
// one cluster of CTAs, on arrays in the workspace: its passes meet at barriers, a
// launch would cost more than a pass.  What is copied (pairs
// of blocks) is known on the device only; the copies of all pools follow in one
// launch that reads the pairs, 4 KB to a warp, eight 16-byte loads a lane in
// flight (16 KB pieces through shared memory by bulk copies, eleven in flight per
// SM: 107 us against 103 for 264 MB, 26 against 23 for 38).
#include <algorithm>
#include <climits>

#include "epsp_kernels.h"
#include "tc100.cuh"

namespace epsp {
namespace {

constexpr int kPlan = 1024;       // threads of a planning CTA
constexpr int kPlanCtas = 8;      // CTAs of its cluster, at most
// What one CTA plans in shared memory (blocks and sequences, tables' entries);
// more is planned in the workspace by a cluster.  400 blocks: 4 us against 8.
constexpr int kSmallBlocks = 8192;
constexpr int kSmallSeqs = 4096;
constexpr int kSmallEntries = 16384;
constexpr int kPoolsPerLaunch = 128;
constexpr int kChunk = 4096;      // bytes a warp copies at a time

struct PoolList {
    Pool p[kPoolsPerLaunch];
    int32_t end[kPoolsPerLaunch];  // chunks of a block in the pools up to this one
    int32_t n;
};

__host__ __device__ __forceinline__ int blocks_of(int rows, int block_rows) {
    return rows / block_rows + (rows % block_rows != 0);
}

// Rows of sequence s; a length that its table cannot hold is recorded and read as 0.
__device__ __forceinline__ int rows_of(const PagesArgs& a, int n, int s) {
    if (n < 0 || n > (int64_t)a.table_stride * a.block_rows) {
        report_error(a.err, kDevBadLength, 0xc0, s);
        return 0;
    }
    return n;
}

// A table's entry, -1 (recorded) where it names no block.
__device__ __forceinline__ int entry(const PagesArgs& a, int b, int s) {
    if (b < 0 || b >= a.pool_blocks) {
        report_error(a.err, kDevBadBlockTable, 0xc1, s);
        return -1;
    }
    return b;
}

// ----------------------------------------------------------------- counting --
__global__ void k11_zero(int32_t* p, int64_t n) {
    tc::pdl_wait();
    tc::pdl_launch();
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) p[i] = 0;
}

__global__ void k11_count(const PagesArgs a) {
    tc::pdl_wait();
    tc::pdl_launch();
    for (int s = blockIdx.x; s < a.n_seq; s += gridDim.x) {
        const int held = blocks_of(rows_of(a, a.lens[s], s), a.block_rows);
        for (int i = threadIdx.x; i < held; i += blockDim.x) {
            const int b = entry(a, a.tables[(int64_t)s * a.table_stride + i], s);
            if (b >= 0) atomicAdd(&a.refs[b], 1);
        }
    }
}

// --------------------------------------------------------------------- fork --
// What the tables held before, in the workspace: [n_seq] lengths, parents and
// new lengths, then the tables.
struct ForkWs {
    int32_t *was, *parent, *now, *tables;
};

__global__ void k11_fork_read(const PagesArgs a, const int32_t* parents, const int32_t* lens, const ForkWs w) {
    tc::pdl_wait();
    tc::pdl_launch();
    for (int s = blockIdx.x; s < a.n_seq; s += gridDim.x) {
        const int n = rows_of(a, a.lens[s], s), held = blocks_of(n, a.block_rows);
        for (int i = blockIdx.y * blockDim.x + threadIdx.x; i < held; i += gridDim.y * blockDim.x)
            w.tables[(int64_t)s * a.table_stride + i] = a.tables[(int64_t)s * a.table_stride + i];
        if (blockIdx.y || threadIdx.x) continue;
        int p = parents[s], now = -1;  // -1: stays as it is
        if (p >= -1 && p < a.n_seq) {
            const int have = p < 0 ? 0 : rows_of(a, a.lens[p], p);
            now = lens ? lens[s] : have;
            if (now < 0 || now > have) now = -1;
        }
        if (now < 0) report_error(a.err, kDevBadParent, 0xc2, s);
        w.was[s] = n;
        w.parent[s] = now < 0 ? s : p;
        w.now[s] = now < 0 ? n : now;
    }
}

__global__ void k11_fork_write(const PagesArgs a, const ForkWs w) {
    tc::pdl_wait();
    tc::pdl_launch();
    for (int s = blockIdx.x; s < a.n_seq; s += gridDim.x) {
        const int p = w.parent[s], now = w.now[s];
        const int held = blocks_of(w.was[s], a.block_rows), want = blocks_of(now, a.block_rows);
        const int64_t row = (int64_t)s * a.table_stride, from = (int64_t)p * a.table_stride;
        for (int i = blockIdx.y * blockDim.x + threadIdx.x; i < max(held, want); i += gridDim.y * blockDim.x) {
            const int old = i < held ? w.tables[row + i] : -1, b = i < want ? w.tables[from + i] : -1;
            if (old == b && i < held && i < want) continue;
            if (i < held && entry(a, old, s) >= 0) atomicAdd(&a.refs[old], -1);
            if (i < want) {
                if (entry(a, b, s) >= 0) atomicAdd(&a.refs[b], 1);
                a.tables[row + i] = b;
            }
        }
        if (blockIdx.y == 0 && threadIdx.x == 0 && (p != s || now != w.was[s])) a.lens[s] = now;
    }
}

// Both in one CTA, with what the tables held in shared memory.
__global__ void __launch_bounds__(kPlan, 1) k11_fork(const PagesArgs a, const int32_t* parents, const int32_t* lens) {
    extern __shared__ int32_t tables_s[];  // [n_seq][table_stride], then [n_seq] lengths and new lengths
    int32_t *was_s = tables_s + a.n_seq * a.table_stride, *now_s = was_s + a.n_seq, *parent_s = now_s + a.n_seq;
    tc::pdl_wait();
    tc::pdl_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int s = threadIdx.x; s < a.n_seq; s += kPlan) {
        was_s[s] = rows_of(a, a.lens[s], s);
        parent_s[s] = parents[s];
        now_s[s] = lens ? lens[s] : -1;
    }
    __syncthreads();
    for (int s = warp; s < a.n_seq; s += kPlan / 32) {
        const int held = blocks_of(was_s[s], a.block_rows);
        for (int i = lane; i < held; i += 32) tables_s[s * a.table_stride + i] = a.tables[(int64_t)s * a.table_stride + i];
    }
    __syncthreads();
    for (int s = warp; s < a.n_seq; s += kPlan / 32) {
        int p = parent_s[s], now = -1;
        const int was = was_s[s];
        if (p >= -1 && p < a.n_seq) {
            const int have = p < 0 ? 0 : was_s[p];
            now = lens ? now_s[s] : have;
            if (now < 0 || now > have) now = -1;
        }
        if (now < 0) {  // stays as it is
            if (lane == 0) report_error(a.err, kDevBadParent, 0xc2, s);
            continue;
        }
        if (p == s && now == was) continue;
        const int held = blocks_of(was, a.block_rows), want = blocks_of(now, a.block_rows);
        for (int i = lane; i < max(held, want); i += 32) {
            const int old = i < held ? tables_s[s * a.table_stride + i] : -1, b = i < want ? tables_s[p * a.table_stride + i] : -1;
            if (i < held && i < want && old == b) continue;
            if (i < held && entry(a, old, s) >= 0) atomicAdd(&a.refs[old], -1);
            if (i < want) {
                if (entry(a, b, s) >= 0) atomicAdd(&a.refs[b], 1);
                a.tables[(int64_t)s * a.table_stride + i] = b;
            }
        }
        if (lane == 0) a.lens[s] = now;
    }
}

// ----------------------------------------------------------------- planning --
__device__ __forceinline__ int cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return (int)r;
}
__device__ __forceinline__ int cluster_size() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return (int)r;
}
// SMALL: one CTA, the plan's arrays in shared memory.  All threads of the plan
// meet, and see what they wrote; reads of what another CTA wrote go past the L1.
template <bool SMALL>
__device__ __forceinline__ void meet() {
    if constexpr (SMALL) {
        __syncthreads();
    } else {
        __threadfence();
        tc::cluster_sync();
    }
}
template <bool SMALL>
__device__ __forceinline__ int32_t at(const int32_t* p) {
    return SMALL ? *p : __ldcg(p);
}

// Exclusive sum over the CTA's threads of two counts; the totals in `all`.
__device__ __forceinline__ int2 cta_scan(int2 x, int2& all, int2* box) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int2 in = x;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int u = __shfl_up_sync(0xffffffffu, in.x, d), v = __shfl_up_sync(0xffffffffu, in.y, d);
        if (lane >= d) in.x += u, in.y += v;
    }
    if (lane == 31) box[warp] = in;
    __syncthreads();
    if (warp == 0) {
        int2 t = box[lane];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, t.x, d), v = __shfl_up_sync(0xffffffffu, t.y, d);
            if (lane >= d) t.x += u, t.y += v;
        }
        box[lane] = t;
    }
    __syncthreads();
    all = box[31];
    const int2 before = warp ? box[warp - 1] : make_int2(0, 0);
    __syncthreads();  // (the box is written again)
    return make_int2(before.x + in.x - x.x, before.y + in.y - x.y);
}

// Totals of all CTAs from those of this one (what the CTAs before it have in
// `before`).
template <bool SMALL>
__device__ __forceinline__ int2 cluster_scan(int2 mine, int2& before, int2* shared) {
    if constexpr (SMALL) {
        before = make_int2(0, 0);
        return mine;
    }
    if (threadIdx.x == 0) *shared = mine;
    tc::cluster_sync();
    int2 all = make_int2(0, 0);
    before = all;
    const int me = cluster_rank(), n = cluster_size();
    for (int k = 0; k < n; ++k) {
        int2 v;
        asm volatile("ld.shared::cluster.v2.s32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(tc::peer_of(shared, k)) : "memory");
        all.x += v.x, all.y += v.y;
        if (k < me) before.x += v.x, before.y += v.y;
    }
    tc::cluster_sync();  // (nobody writes its own, or ends, while it is read)
    return all;
}

// This CTA's part of n items, in whole turns of the CTA.
struct Part {
    int64_t begin, end;
};
__device__ __forceinline__ Part part_of(int64_t n) {
    const int64_t per = ((n + cluster_size() - 1) / cluster_size() + kPlan - 1) / kPlan * kPlan;
    const int64_t b = min(n, per * cluster_rank());
    return {b, min(n, b + per)};
}

struct ResizeWs {
    int32_t* n_pairs;  // [4] the count first
    int2* pairs;       // [n_seq] (from, to)
    // the rest in the workspace, or in shared memory
    int32_t *refs, *growers, *keeper;        // [pool_blocks]; growers and keeper: of a shared last block
    int32_t* free;                           // [pool_blocks] free blocks taken, in order
    int32_t *was, *now, *last, *need, *off;  // [n_seq]; last: a block that a sequence grows in, -1 where it is its own
};

// Lays out the arrays that a plan works on; returns the bytes.
__host__ __device__ inline size_t plan_arrays(const PagesArgs& a, char* base, ResizeWs* w) {
    size_t at = 0;
    auto take = [&](size_t n) {
        int32_t* p = reinterpret_cast<int32_t*>(base + at);
        at += (n * 4 + 15) & ~(size_t)15;
        return p;
    };
    w->refs = take(a.pool_blocks), w->growers = take(a.pool_blocks), w->keeper = take(a.pool_blocks);
    w->free = take(a.pool_blocks);
    w->was = take(a.n_seq), w->now = take(a.n_seq), w->last = take(a.n_seq);
    w->need = take(a.n_seq), w->off = take(a.n_seq);
    return at;
}

template <bool SMALL>
__global__ void __launch_bounds__(kPlan, 1) k11_resize(const PagesArgs a, const int32_t* new_lens, ResizeWs w) {
    __shared__ int2 box[32], mine_s;
    __shared__ int pairs_s;
    extern __shared__ __align__(16) char plan_s[];
    if constexpr (SMALL) plan_arrays(a, plan_s, &w);
    tc::pdl_wait();
    tc::pdl_launch();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int warps = cluster_size() * (kPlan / 32), me = cluster_rank() * (kPlan / 32) + warp;
    const Part blocks = part_of(a.pool_blocks), seqs = part_of(a.n_seq);
    for (int64_t b = blocks.begin + threadIdx.x; b < blocks.end; b += kPlan) {
        w.refs[b] = a.refs[b];
        w.growers[b] = 0;
        w.keeper[b] = -1;
    }
    for (int64_t s = seqs.begin + threadIdx.x; s < seqs.end; s += kPlan) {
        const int n = rows_of(a, a.lens[s], (int)s);
        int now = new_lens[s];
        if (now < 0 || now > (int64_t)a.table_stride * a.block_rows) {
            a.err[kErrRefused] = 1;
            report_error(a.err, kDevBadLength, 0xc3, (int)s);
            now = n;
        }
        w.was[s] = n;
        w.now[s] = now;
        // (held by others or not is known once all have given back)
        w.last[s] = now > n && n % a.block_rows ? entry(a, a.tables[s * a.table_stride + n / a.block_rows], (int)s) : -1;
    }
    if (me == 0 && lane == 0) *(SMALL ? &pairs_s : w.n_pairs) = 0;
    meet<SMALL>();
    // blocks given back
    for (int s = me; s < a.n_seq; s += warps) {
        const int held = blocks_of(at<SMALL>(&w.was[s]), a.block_rows), want = blocks_of(at<SMALL>(&w.now[s]), a.block_rows);
        for (int i = want + lane; i < held; i += 32) {
            const int b = entry(a, a.tables[(int64_t)s * a.table_stride + i], s);
            if (b >= 0) atomicAdd(&w.refs[b], -1);
        }
    }
    meet<SMALL>();
    // who grows inside a block that others hold too
    for (int64_t s = seqs.begin + threadIdx.x; s < seqs.end; s += kPlan) {
        const int b = w.last[s];
        if (b < 0) continue;
        if (at<SMALL>(&w.refs[b]) > 1) {
            atomicAdd(&w.growers[b], 1);
            atomicMax(&w.keeper[b], (int)s);
        } else {
            w.last[s] = -1;
        }
    }
    meet<SMALL>();
    // what each sequence takes; where all holders of a block grow, the last one keeps it
    int2 run = make_int2(0, 0);
    for (int64_t s0 = seqs.begin; s0 < seqs.end; s0 += kPlan) {
        const int64_t s = s0 + threadIdx.x;
        int need = 0;
        if (s < seqs.end) {
            const int b = w.last[s];
            const bool copy =
                b >= 0 && !(at<SMALL>(&w.growers[b]) == at<SMALL>(&w.refs[b]) && at<SMALL>(&w.keeper[b]) == (int)s);
            need = max(0, blocks_of(w.now[s], a.block_rows) - blocks_of(w.was[s], a.block_rows)) + (copy ? 1 : 0);
            w.need[s] = copy ? -need : need;  // (negative: its first block is the copy)
        }
        int2 all;
        const int2 at = cta_scan(make_int2(need, 0), all, box);
        if (s < seqs.end) w.off[s] = run.x + at.x;
        run.x += all.x;
    }
    for (int64_t b0 = blocks.begin; b0 < blocks.end; b0 += kPlan) {
        const int64_t b = b0 + threadIdx.x;
        run.y += __syncthreads_count(b < blocks.end && at<SMALL>(&w.refs[b]) == 0);
    }
    int2 before;
    const int2 all = cluster_scan<SMALL>(run, before, &mine_s);
    if (all.x > all.y) {  // too few: nothing changes
        if (me == 0 && lane == 0) {
            *w.n_pairs = 0;
            a.err[kErrRefused] = 1;
            report_error(a.err, kDevNoBlocks, 0xc4, all.x - all.y);
        }
        return;
    }
    // this CTA's sequences take from here; its free blocks have these places
    for (int64_t s = seqs.begin + threadIdx.x; s < seqs.end; s += kPlan) w.off[s] += before.x;
    int place = before.y;
    for (int64_t b0 = blocks.begin; b0 < blocks.end; b0 += kPlan) {
        const int64_t b = b0 + threadIdx.x;
        const bool in = b < blocks.end;
        const int refs = in ? at<SMALL>(&w.refs[b]) : 1;
        int2 here;
        const int2 at = cta_scan(make_int2(0, refs == 0 ? 1 : 0), here, box);
        if (refs == 0 && place + at.y < all.x) w.free[place + at.y] = (int)b;
        if (in) a.refs[b] = refs;
        place += here.y;
    }
    meet<SMALL>();
    for (int s = me; s < a.n_seq; s += warps) {
        const int was = at<SMALL>(&w.was[s]), now = at<SMALL>(&w.now[s]), off = at<SMALL>(&w.off[s]), need = at<SMALL>(&w.need[s]);
        const int held = blocks_of(was, a.block_rows), want = blocks_of(now, a.block_rows), copy = need < 0;
        int32_t* table = a.tables + (int64_t)s * a.table_stride;
        for (int i = held + lane; i < want; i += 32) {
            const int b = at<SMALL>(&w.free[off + copy + i - held]);
            table[i] = b;
            a.refs[b] = 1;
        }
        if (lane == 0) {
            if (copy) {
                const int from = at<SMALL>(&w.last[s]), to = at<SMALL>(&w.free[off]);
                table[held - 1] = to;
                a.refs[to] = 1;
                atomicAdd(&a.refs[from], -1);
                w.pairs[atomicAdd(SMALL ? &pairs_s : w.n_pairs, 1)] = make_int2(from, to);  // (their order does not matter)
            }
            a.lens[s] = now;
        }
    }
    if constexpr (SMALL) {
        __syncthreads();
        if (threadIdx.x == 0) *w.n_pairs = pairs_s;
    }
}

struct CompactWs {
    int32_t* n_pairs;  // [4] moves, then blocks in use
    int2* pairs;       // [pool_blocks / 2] (from, to)
    int32_t* map;      // [pool_blocks] where a moved block went
};

template <bool SMALL>
__global__ void __launch_bounds__(kPlan, 1) k11_compact(const PagesArgs a, int32_t* n_used, const CompactWs w) {
    __shared__ int2 box[32], mine_s;
    extern __shared__ __align__(16) char plan_s[];
    int32_t* refs_s = reinterpret_cast<int32_t*>(plan_s);  // SMALL: [pool_blocks], then the pairs
    int2* pairs = SMALL ? reinterpret_cast<int2*>(plan_s + ((size_t)a.pool_blocks * 4 + 15) / 16 * 16) : w.pairs;
    tc::pdl_wait();
    tc::pdl_launch();
    const Part blocks = part_of(a.pool_blocks);
    int2 run = make_int2(0, 0);
    for (int64_t b0 = blocks.begin; b0 < blocks.end; b0 += kPlan) {
        const int64_t b = b0 + threadIdx.x;
        const int refs = b < blocks.end ? a.refs[b] : 0;
        if (SMALL && b < blocks.end) refs_s[b] = refs;
        run.x += __syncthreads_count(refs > 0);
    }
    int2 before;
    const int used = cluster_scan<SMALL>(run, before, &mine_s).x;
    const int32_t* refs = SMALL ? refs_s : a.refs;
    // holes below, blocks in use at or past `used`: as many of each
    auto what = [&](int64_t b) {
        const bool live = b < blocks.end && refs[b] > 0;
        return make_int2(b < blocks.end && b < used && !live, b >= used && live);
    };
    int2 all;
    if constexpr (!SMALL) {
        run = make_int2(0, 0);
        for (int64_t b0 = blocks.begin; b0 < blocks.end; b0 += kPlan) {
            const int2 x = what(b0 + threadIdx.x);
            run.x += __syncthreads_count(x.x);
            run.y += __syncthreads_count(x.y);
        }
        all = cluster_scan<SMALL>(run, before, &mine_s);
    } else {
        before = make_int2(0, 0);
    }
    for (int64_t b0 = blocks.begin; b0 < blocks.end; b0 += kPlan) {
        const int64_t b = b0 + threadIdx.x;
        const int2 x = what(b);
        int2 here;
        const int2 at = cta_scan(x, here, box);
        if (x.x) pairs[before.x + at.x].y = (int)b;
        if (x.y) pairs[before.y + at.y].x = (int)b;
        else if (b < blocks.end && b >= used) w.map[b] = (int)b;
        before.x += here.x;
        before.y += here.y;
    }
    if constexpr (SMALL) all = before;
    meet<SMALL>();
    for (int i = cluster_rank() * kPlan + threadIdx.x; i < all.y; i += cluster_size() * kPlan) {
        const int2 p = SMALL ? pairs[i] : __ldcg(&pairs[i]);
        w.map[p.x] = p.y;
        if constexpr (SMALL) w.pairs[i] = p;
        a.refs[p.y] = refs[p.x];
        a.refs[p.x] = 0;
    }
    if (cluster_rank() == 0 && threadIdx.x == 0) {
        w.n_pairs[0] = all.y;
        w.n_pairs[1] = used;
        if (n_used) *n_used = used;
    }
}

// Copies the pairs' blocks in every pool; `used` (not null): tables follow the
// map, too.
__global__ void __launch_bounds__(256) k11_copy(const PagesArgs a, const __grid_constant__ PoolList pools,
                                                const int32_t* n_pairs, const int2* pairs, const int32_t* used,
                                                const int32_t* map) {
    tc::pdl_wait();
    tc::pdl_launch();
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * (blockDim.x / 32), me = (int64_t)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5);
    const int n = *n_pairs, per = pools.n ? pools.end[pools.n - 1] : 0;
    if (used && n > 0) {
        const int from = *used;
        for (int64_t s = me; s < a.n_seq; s += warps) {
            const int held = blocks_of(rows_of(a, a.lens[s], (int)s), a.block_rows);
            for (int i = lane; i < held; i += 32) {
                int32_t* e = a.tables + s * a.table_stride + i;
                const int b = entry(a, *e, (int)s);
                if (b >= from) *e = map[b];
            }
        }
    }
    for (int64_t t = me; t < (int64_t)n * per; t += warps) {
        const int2 pair = pairs[t / per];
        const int c = (int)(t % per);
        int lo = 0, hi = pools.n - 1;  // the pool whose chunks hold c
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (pools.end[mid] > c) hi = mid;
            else lo = mid + 1;
        }
        const size_t bytes = pools.p[lo].bytes, at = (size_t)(c - (lo ? pools.end[lo - 1] : 0)) * kChunk;
        const char* src = static_cast<const char*>(pools.p[lo].rows) + pair.x * bytes + at;
        char* dst = static_cast<char*>(pools.p[lo].rows) + pair.y * bytes + at;
        const int here = (int)min((size_t)kChunk, bytes - at);
        if (((reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst) | here) & 15) == 0) {
            uint4 v[kChunk / 512];
#pragma unroll
            for (int j = 0; j < kChunk / 512; ++j)
                if ((j * 32 + lane) * 16 < here) v[j] = __ldcs(reinterpret_cast<const uint4*>(src) + j * 32 + lane);
#pragma unroll
            for (int j = 0; j < kChunk / 512; ++j)
                if ((j * 32 + lane) * 16 < here) __stcs(reinterpret_cast<uint4*>(dst) + j * 32 + lane, v[j]);
        } else {
            for (int i = lane * 4; i < here; i += 128) *reinterpret_cast<uint32_t*>(dst + i) = *reinterpret_cast<const uint32_t*>(src + i);
        }
    }
}

// ---------------------------------------------------------------- host side --
template <class... P, class... A>
cudaError_t go(void (*kernel)(P...), dim3 grid, int threads, int cluster, size_t smem, cudaStream_t s, A&&... args) {
    cudaLaunchAttribute at[2]{};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster;
    at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = at;
    cfg.numAttrs = cluster ? 2 : 1;
    if (smem > 47 * 1024) {  // (48 KB with the kernel's static part)
        // (the same for all calls: two threads may be here with different sizes)
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024);
        if (e != cudaSuccess) return e;
    }
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

bool small_plan(const PagesArgs& a) { return a.n_seq <= kSmallSeqs && a.pool_blocks <= kSmallBlocks; }

// Lays out `n` bytes at the workspace's next 16-byte boundary.
struct Space {
    char* base;
    size_t at = 0;
    template <class T>
    T* take(size_t n) {
        T* p = reinterpret_cast<T*>(base + at);
        at += (n * sizeof(T) + 15) & ~(size_t)15;
        return p;
    }
};

size_t fork_ws(const PagesArgs& a, void* ws, ForkWs* w) {
    Space sp{static_cast<char*>(ws)};
    w->was = sp.take<int32_t>(a.n_seq);
    w->parent = sp.take<int32_t>(a.n_seq);
    w->now = sp.take<int32_t>(a.n_seq);
    w->tables = sp.take<int32_t>((size_t)a.n_seq * a.table_stride);
    return sp.at;
}

size_t resize_ws(const PagesArgs& a, void* ws, ResizeWs* w) {
    Space sp{static_cast<char*>(ws)};
    w->n_pairs = sp.take<int32_t>(4);
    w->pairs = sp.take<int2>(a.n_seq);
    sp.at += plan_arrays(a, sp.base + sp.at, w);
    return sp.at;
}

size_t compact_ws(const PagesArgs& a, void* ws, CompactWs* w) {
    Space sp{static_cast<char*>(ws)};
    w->n_pairs = sp.take<int32_t>(4);
    w->pairs = sp.take<int2>((size_t)a.pool_blocks / 2 + 1);
    w->map = sp.take<int32_t>(a.pool_blocks);
    return sp.at;
}

// The copies of all pools, kPoolsPerLaunch a launch; the first also rewrites the
// tables.  `over`: CTAs per SM at most.  More even out the copies' ends (264 MB:
// 8 103 us, 32 98, 64 97), and cost a call that copies nothing: a step's growth
// within its blocks takes 8.4 us with 8, 12 with 32.
cudaError_t copy_pools(const PagesArgs& a, const Pool* pools, int32_t n_pools, int64_t most, int32_t over, const int32_t* n_pairs,
                       const int2* pairs, const int32_t* used, const int32_t* map, cudaStream_t s) {
    for (int32_t i0 = 0; i0 < n_pools; i0 += kPoolsPerLaunch) {
        PoolList l{};
        l.n = std::min(kPoolsPerLaunch, n_pools - i0);
        int64_t chunks = 0;
        for (int i = 0; i < l.n; ++i) {
            l.p[i] = pools[i0 + i];
            chunks += (int64_t)((l.p[i].bytes + kChunk - 1) / kChunk);
            if (chunks > INT_MAX) return cudaErrorInvalidValue;
            l.end[i] = (int32_t)chunks;
        }
        const int64_t ctas = std::min<int64_t>(148 * over, (chunks * std::max<int64_t>(most, 1) + 7) / 8);
        const cudaError_t e = go(k11_copy, dim3((unsigned)std::max<int64_t>(ctas, 1)), 256, 0, 0, s, a, l, n_pairs, pairs,
                                 i0 == 0 ? used : nullptr, map);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

}  // namespace

cudaError_t launch_count_refs(const PagesArgs& a, cudaStream_t s) {
    const cudaError_t e = go(k11_zero, dim3(std::min(592, (a.pool_blocks + 255) / 256)), 256, 0, 0, s, a.refs, (int64_t)a.pool_blocks);
    return e != cudaSuccess ? e : go(k11_count, dim3(std::min(a.n_seq, 1184)), 128, 0, 0, s, a);
}

size_t fork_ws_bytes(const PagesArgs& a) {
    ForkWs w;
    return fork_ws(a, nullptr, &w);
}

cudaError_t launch_fork(const PagesArgs& a, const int32_t* parents, const int32_t* lens, void* ws, cudaStream_t s) {
    if ((int64_t)a.n_seq * a.table_stride <= kSmallEntries && a.n_seq <= kSmallSeqs)
        return go(k11_fork, dim3(1), kPlan, 0, (size_t)a.n_seq * (a.table_stride + 3) * 4, s, a, parents, lens);
    ForkWs w;
    fork_ws(a, ws, &w);
    const dim3 grid(std::min(a.n_seq, 4096), std::min(16, (a.table_stride + 255) / 256));
    const cudaError_t e = go(k11_fork_read, grid, 256, 0, 0, s, a, parents, lens, w);
    return e != cudaSuccess ? e : go(k11_fork_write, grid, 256, 0, 0, s, a, w);
}

size_t resize_ws_bytes(const PagesArgs& a) {
    ResizeWs w;
    return resize_ws(a, nullptr, &w);
}

cudaError_t launch_resize(const PagesArgs& a, const int32_t* new_lens, const Pool* pools, int32_t n_pools, void* ws,
                          cudaStream_t s) {
    ResizeWs w;
    resize_ws(a, ws, &w);
    ResizeWs none;
    const cudaError_t e = small_plan(a)
                              ? go(k11_resize<true>, dim3(1), kPlan, 0, plan_arrays(a, nullptr, &none), s, a, new_lens, w)
                              : go(k11_resize<false>, dim3(kPlanCtas), kPlan, kPlanCtas, 0, s, a, new_lens, w);
    if (e != cudaSuccess) return e;
    return copy_pools(a, pools, n_pools, a.n_seq, 8, w.n_pairs, w.pairs, nullptr, nullptr, s);
}

size_t compact_ws_bytes(const PagesArgs& a) {
    CompactWs w;
    return compact_ws(a, nullptr, &w);
}

cudaError_t launch_compact(const PagesArgs& a, const Pool* pools, int32_t n_pools, int32_t* n_used, void* ws,
                           cudaStream_t s) {
    CompactWs w;
    compact_ws(a, ws, &w);
    const size_t smem = ((size_t)a.pool_blocks * 4 + 15) / 16 * 16 + ((size_t)a.pool_blocks / 2 + 1) * 8;
    const cudaError_t e = small_plan(a) ? go(k11_compact<true>, dim3(1), kPlan, 0, smem, s, a, n_used, w)
                                        : go(k11_compact<false>, dim3(kPlanCtas), kPlan, kPlanCtas, 0, s, a, n_used, w);
    if (e != cudaSuccess) return e;
    return copy_pools(a, pools, n_pools, a.pool_blocks / 2, 32, w.n_pairs, w.pairs, w.n_pairs + 1, w.map, s);
}

}  // namespace epsp

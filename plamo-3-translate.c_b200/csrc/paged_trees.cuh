// Draft trees of a paged batch step (include/plamo_paged.h): positions and
// masks before the layers, the confirmed path and its rows after them. The
// trees' attention is in paged_attention.cuh, paged_tree_tiles.cuh and paged_tree_f32.cuh.
#pragma once
#include "paged.cuh"

namespace plamo {

constexpr int kTreeRows = PLAMO_PAGED_TREE_ROWS;

// A request's rows in the batch, whatever its starts say.
struct BatchRows {
    int32_t row0, rows;
};
__device__ __forceinline__ BatchRows batch_rows(const int32_t *starts, uint64_t r, uint64_t all) {
    const int32_t end = static_cast<int32_t>(all), row0 = min(max(starts[r], 0), end);
    return {row0, min(max(starts[r + 1], row0), end) - row0};
}

// ---- masks and positions -----------------------------------------------------------
// A CTA to a request, a thread to a row, which walks up to the request's root:
// depth hops through shared memory. Latency bounds it.
__global__ void __launch_bounds__(kTreeRows) paged_tree_kernel(plamo_paged_tree_args d) {
    __shared__ int32_t above[kTreeRows];
    const int32_t tid = threadIdx.x, most = 32 * static_cast<int32_t>(d.words);  // (threads, too)
    if (blockIdx.x < d.requests) {
        const BatchRows b = batch_rows(d.starts, blockIdx.x, d.rows);
        const int64_t held = max(static_cast<int64_t>(d.lengths[blockIdx.x]) - b.rows, int64_t{0});
        int32_t parent = -1;
        if (tid < b.rows) {
            parent = d.parents[b.row0 + tid];
            if (parent < -1 || parent >= tid) {
                pg_flag(d.status, PLAMO_PAGED_TREE);
                parent = -1;
            }
        }
        if (tid == 0 && b.rows > most) pg_flag(d.status, PLAMO_PAGED_TREE);
        above[tid] = parent;
        __syncthreads();
        for (int32_t i = tid; i < b.rows; i += most) {
            uint32_t mask[kTreeRows / 32] = {};
            int32_t generations = 0;
            if (i < most) {
#pragma unroll 1
                for (int32_t j = i; j >= 0; j = above[j], ++generations) {
#pragma unroll
                    for (int w = 0; w < kTreeRows / 32; ++w)
                        if (j >> 5 == w) mask[w] |= 1u << (j & 31);
                }
                --generations;
            }
            const int64_t row = b.row0 + i;
            d.positions[row] = static_cast<int32_t>(min(d.base + held + generations, static_cast<int64_t>(INT32_MAX)));
            uint32_t *out = d.masks + row * d.words;
#pragma unroll
            for (int w = 0; w < kTreeRows / 32; ++w)
                if (w < static_cast<int>(d.words)) out[w] = mask[w];
        }
    }
    // Padding: rows before the first request's and behind the last one's.
    const int64_t rows = static_cast<int64_t>(d.rows);
    const int64_t first = d.requests ? min(max(static_cast<int64_t>(d.starts[0]), int64_t{0}), rows) : 0;
    const int64_t taken = d.requests ? min(max(static_cast<int64_t>(d.starts[d.requests]), int64_t{0}), rows) : 0;
    const int64_t step = static_cast<int64_t>(gridDim.x) * most;
    const auto clear = [&](int64_t row) {
        d.positions[row] = 0;
        for (uint32_t w = 0; w < d.words; ++w) d.masks[row * d.words + w] = 0;
    };
    for (int64_t row = static_cast<int64_t>(blockIdx.x) * most + tid; row < first; row += step) clear(row);
    for (int64_t row = taken + static_cast<int64_t>(blockIdx.x) * most + tid; row < rows; row += step) clear(row);
}

// ---- acceptance ----------------------------------------------------------------------
// A warp to a request. Its rows' parents and tokens lie in registers, a row to
// a lane and register, so that a step of the walk is one look at shared memory
// for the chosen token and one minimum over the warp.
constexpr int kAcceptWarps = 8;      // to a CTA of the walk
constexpr int kAcceptThreads = 1024;  // of the CTA that gives the pages back
// Requests that one CTA walks and settles by itself: two rounds of its warps. Of 8 requests
// that is a launch of 8 us; a walk and a settling launch of 256 take 6 and 8.
constexpr int kAcceptAlone = 64;

__device__ __forceinline__ void accept_walk(const plamo_paged_accept_args &d, uint64_t r, int32_t *picks) {
    constexpr int PER = kTreeRows / 32;
    const int lane = threadIdx.x & 31;
    const BatchRows b = batch_rows(d.starts, r, d.rows);
    const int32_t held = d.lengths[r] - b.rows, rows = held < 0 ? 0 : min(b.rows, kTreeRows);
    int32_t parent[PER], token[PER];
#pragma unroll
    for (int x = 0; x < PER; ++x) {
        const int32_t i = 32 * x + lane;
        const bool there = i < rows;
        parent[x] = there ? d.parents[b.row0 + i] : -2;
        token[x] = there ? d.tokens[b.row0 + i] : 0;
        if (there) picks[i] = d.chosen[b.row0 + i];
    }
    __syncwarp();
    int32_t count = 0, last = -1;
    if (rows) {
#pragma unroll 1
        for (int32_t at = 0; at < kTreeRows; ++count) {
            last = picks[at];
            if (lane == 0) {
                d.path[b.row0 + count] = at;
                d.next[b.row0 + count] = last;
            }
            int32_t child = kTreeRows;  // the first below `at` with the chosen token; children come after their parents
#pragma unroll
            for (int x = PER - 1; x >= 0; --x)
                if (parent[x] == at && token[x] == last && 32 * x + lane > at) child = 32 * x + lane;
            at = __reduce_min_sync(0xffffffffu, child);
        }
    }
    for (int32_t i = count + lane; i < b.rows; i += 32) d.path[b.row0 + i] = d.next[b.row0 + i] = -1;
    if (lane == 0) {
        d.counts[r] = count;
        d.kept[r] = held < 0 ? d.lengths[r] : held + count;
        d.last[r] = last;
    }
}

// Pages that the request's rows reached in the step and the kept ones do not: [x, y) of its table.
__device__ __forceinline__ int2 accept_back(const plamo_paged_accept_args &d, uint64_t r, uint32_t &flags) {
    const BatchRows b = batch_rows(d.starts, r, d.rows);
    const int64_t length = d.lengths[r], kept = d.kept[r];
    if (length < b.rows) flags |= PLAMO_PAGED_COUNT;
    if (b.rows > kTreeRows) flags |= PLAMO_PAGED_TREE;
    if (length < b.rows) return make_int2(0, 0);
    const int64_t from = (kept + kPgRows - 1) / kPgRows, to = (length + kPgRows - 1) / kPgRows;
    if (to > static_cast<int64_t>(d.table_stride)) {
        flags |= PLAMO_PAGED_TABLE;
        return make_int2(0, 0);
    }
    return make_int2(static_cast<int32_t>(from), static_cast<int32_t>(to));
}

__device__ __forceinline__ void accept_settle(const plamo_paged_accept_args &d, int64_t *sums) {
    __shared__ int32_t longest;
    __shared__ uint32_t bad;
    const int tid = threadIdx.x;
    const int64_t R = static_cast<int64_t>(d.requests), per = (R + kAcceptThreads - 1) / kAcceptThreads;
    const int64_t r0 = min(R, tid * per), r1 = min(R, r0 + per);
    if (tid == 0) {
        longest = 0;
        bad = 0;
    }
    __syncthreads();
    int64_t pages = 0, rows = 0, all_pages, all_rows;
    uint32_t flags = 0;
    int32_t most = 0;
    for (int64_t r = r0; r < r1; ++r) {
        const int2 back = accept_back(d, r, flags);
        pages += back.y - back.x;
        rows += d.counts[r];
        most = max(most, d.kept[r]);
    }
    most = __reduce_max_sync(0xffffffffu, most);
    flags = __reduce_or_sync(0xffffffffu, flags);
    if ((tid & 31) == 0) {
        atomicMax(&longest, most);
        if (flags) atomicOr(&bad, flags);
    }
    const int64_t first = pg_block_scan<kAcceptThreads>(pages, sums, &all_pages);
    pg_block_scan<kAcceptThreads>(rows, sums, &all_rows);
    const int64_t head = d.plan[2];
    const bool fits = head >= all_pages && head <= static_cast<int64_t>(d.free_count);
    int64_t at = head - all_pages + first;
    for (int64_t r = r0; fits && r < r1; ++r) {
        const int2 back = accept_back(d, r, flags);
        for (int32_t page = back.x; page < back.y; ++page) d.free_pages[at++] = d.tables[r * d.table_stride + page];
    }
    if (tid == 0) {
        d.summary[0] = d.plan[0] | static_cast<int32_t>(bad) | (fits ? 0 : PLAMO_PAGED_NO_PAGES);
        d.summary[1] = static_cast<int32_t>(all_rows);
        d.summary[2] = static_cast<int32_t>(fits ? head - all_pages : head);
        d.summary[3] = longest;
    }
}

// Paths of rows that no request has.
__device__ __forceinline__ void accept_padding(const plamo_paged_accept_args &d, int64_t thread, int64_t threads) {
    const int64_t rows = static_cast<int64_t>(d.rows);
    const int64_t first = d.requests ? min(max(static_cast<int64_t>(d.starts[0]), int64_t{0}), rows) : 0;
    const int64_t taken = d.requests ? min(max(static_cast<int64_t>(d.starts[d.requests]), int64_t{0}), rows) : 0;
    for (int64_t row = thread; row < first; row += threads) d.path[row] = d.next[row] = -1;
    for (int64_t row = taken + thread; row < rows; row += threads) d.path[row] = d.next[row] = -1;
}

__global__ void __launch_bounds__(32 * kAcceptWarps) paged_accept_walk_kernel(plamo_paged_accept_args d) {
    __shared__ int32_t picks[kAcceptWarps][kTreeRows];
    const int warp = threadIdx.x >> 5;
    const uint64_t r = static_cast<uint64_t>(blockIdx.x) * kAcceptWarps + warp;
    pdl_launch_dependents();
    if (r < d.requests) accept_walk(d, r, picks[warp]);
    accept_padding(d, static_cast<int64_t>(blockIdx.x) * 32 * kAcceptWarps + threadIdx.x, static_cast<int64_t>(gridDim.x) * 32 * kAcceptWarps);
}
__global__ void __launch_bounds__(kAcceptThreads) paged_accept_settle_kernel(plamo_paged_accept_args d) {
    __shared__ int64_t sums[kAcceptThreads / 32];
    pdl_wait();
    accept_settle(d, sums);
}
__global__ void __launch_bounds__(kAcceptThreads) paged_accept_kernel(plamo_paged_accept_args d) {
    __shared__ int64_t sums[kAcceptThreads / 32];
    __shared__ int32_t picks[kAcceptThreads / 32][kTreeRows];
    const int warp = threadIdx.x >> 5;
    for (uint64_t r = warp; r < d.requests; r += kAcceptThreads / 32) {
        accept_walk(d, r, picks[warp]);
        __syncwarp();
    }
    accept_padding(d, threadIdx.x, kAcceptThreads);
    __syncthreads();  // the walks' counts
    accept_settle(d, sums);
}

// ---- moving the confirmed rows ----------------------------------------------------------
// A CTA takes one request and some layers. It looks its rows' slots up once; then
// a thread takes 16 bytes of a row (of keys or values) and moves them for all of
// the path, eight rows at a time: those are loaded before any is written. A
// row's new place is never behind its old one and the path rises, so no row
// that is still to be read has been written, and nobody else touches the
// thread's columns.
constexpr int kKeepThreads = 256, kKeepLayers = 64, kKeepBatch = 8;

struct KeepParams {
    void *pools[kKeepLayers];
    const int32_t *path, *starts, *lengths, *tables;
    uint32_t *status;
    uint64_t rows, table_stride;
    int32_t layers, per, pages;  // layers to a CTA
    int32_t row_bytes;           // of keys or values
};

__global__ void __launch_bounds__(kKeepThreads) paged_keep_kernel(const __grid_constant__ KeepParams p) {
    __shared__ int64_t from[kTreeRows], to[kTreeRows];  // byte offsets of key rows in a pool; -1: not moved
    __shared__ int32_t moved;
    const int32_t tid = threadIdx.x;
    const uint64_t r = blockIdx.x;
    const BatchRows b = batch_rows(p.starts, r, p.rows);
    const int32_t held = p.lengths[r] - b.rows, rows = held < 0 ? 0 : min(b.rows, kTreeRows);
    if (tid == 0) moved = rows;
    __syncthreads();
    if (tid < rows) {
        const int32_t at = p.path[b.row0 + tid], before = tid ? p.path[b.row0 + tid - 1] : -1;
        if (at <= before || at >= rows) atomicMin(&moved, tid);
        int64_t place[2] = {-1, -1};
        if (at > tid && at < rows) {
            bool bad = false;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int64_t own = static_cast<int64_t>(held) + (x ? tid : at), page = own / kPgRows;
                const int32_t id = page < static_cast<int64_t>(p.table_stride) ? p.tables[r * p.table_stride + page] : -1;
                bad |= id < 0 || id >= p.pages;
                place[x] = (static_cast<int64_t>(id) * 2 * kPgRows + own % kPgRows) * p.row_bytes;
            }
            if (bad) place[0] = -2;
        }
        from[tid] = place[0];
        to[tid] = place[1];
    }
    __syncthreads();
    const int32_t count = moved;
    if (tid < count && from[tid] == -2) pg_flag(p.status, PLAMO_PAGED_PAGE);
    const int32_t pieces = p.row_bytes / 16, first = blockIdx.y * p.per, layers = min(p.per, p.layers - first);
#pragma unroll 1
    for (int32_t x = tid; x < 2 * pieces * layers; x += kKeepThreads) {
        const int32_t layer = x / (2 * pieces), y = x - layer * 2 * pieces, kind = y >= pieces;
        char *pool = static_cast<char *>(p.pools[first + layer]) + static_cast<int64_t>(kind) * kPgRows * p.row_bytes + 16ll * (y - kind * pieces);
#pragma unroll 1
        for (int32_t k0 = 0; k0 < count; k0 += kKeepBatch) {
            uint4 v[kKeepBatch];
#pragma unroll
            for (int k = 0; k < kKeepBatch; ++k)
                if (k0 + k < count && from[k0 + k] >= 0) v[k] = *reinterpret_cast<const uint4 *>(pool + from[k0 + k]);
#pragma unroll
            for (int k = 0; k < kKeepBatch; ++k)
                if (k0 + k < count && from[k0 + k] >= 0) *reinterpret_cast<uint4 *>(pool + to[k0 + k]) = v[k];
        }
    }
}

}  // namespace plamo

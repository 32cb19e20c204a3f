// Page tables, slot maps and the cache store of a paged batch step
// (include/plamo_paged.h). The step's attention is in paged_attention.cuh.
#pragma once
#include <cuda_bf16.h>

#include "../../include/plamo_paged.h"
#include "common.cuh"

namespace plamo {

constexpr int kPgRows = PLAMO_PAGED_ROWS;
constexpr int kPgDim = PLAMO_PAGED_DIM;
// Largest page id + 1: slots (page * 64 + row) stay below 2^31.
constexpr int32_t kPgMaxPages = 1 << 25;
constexpr uint64_t kPgMaxCount = 1u << 30;

__device__ __forceinline__ void pg_flag(uint32_t *status, uint32_t bit) { atomicOr(status, bit); }
// Takes the bits of words[0] to words[1].
__global__ void paged_status_kernel(uint32_t *words) { words[1] = atomicExch(words, 0u); }

// Exclusive scan of one 64-bit value per thread over a block of NT threads;
// *total gets the sum. `sm` holds NT / 32 values. Ends with a barrier.
template <int NT>
__device__ __forceinline__ int64_t pg_block_scan(int64_t v, int64_t *sm, int64_t *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t up = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += up;
    }
    if (lane == 31) sm[warp] = inc;
    __syncthreads();
    int64_t before = 0, sum = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
        const int64_t x = sm[w];
        if (w < warp) before += x;
        sum += x;
    }
    __syncthreads();
    *total = sum;
    return before + inc - v;
}

// ---- plan ---------------------------------------------------------------------
// One launch of ceil(rows / 1024) CTAs, each finding its 1024 batch rows by
// itself: every CTA sums the requests' row and page counts (a few loads per
// thread from L2), so no CTA waits for another and no scan result goes
// through memory. The request of each row is then a running maximum over
// marks that the requests' first rows leave in shared memory, so a request
// of one row and one of a thousand cost the same per row. Latency bounds it: 7 us
// cold for 8 requests and for 65 K rows of 64 prompts alike, 11 us for 4,096
// requests (four to a thread).
constexpr int kPlanThreads = 1024;

struct PlanParams {
    plamo_paged_plan_args d;  // lengths NULL: written by paged_plan_lengths_kernel
};

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(PlanParams p) {
    __shared__ int64_t sums[kPlanThreads / 32];
    __shared__ int32_t mark[kPlanThreads], row_start[kPlanThreads], row_held[kPlanThreads], row_owner[kPlanThreads];
    __shared__ int32_t row_page[kPlanThreads];  // free-list entry of the request's first new page
    __shared__ int32_t warp_mark[kPlanThreads / 32];
    __shared__ int32_t longest, longest_held;
    __shared__ uint32_t bad;
    const plamo_paged_plan_args &d = p.d;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t R = static_cast<int64_t>(d.requests), rows = static_cast<int64_t>(d.rows);
    const int64_t per = (R + kPlanThreads - 1) / kPlanThreads;
    const int64_t r0 = min(R, tid * per), r1 = min(R, r0 + per);
    if (tid == 0) {
        longest = longest_held = 0;
        bad = 0;
    }
    mark[tid] = -1;
    __syncthreads();

    // This thread's requests: rows added, pages taken, longest length.
    int64_t new_rows = 0, new_pages = 0;
    int32_t most = 0, most_held = 0;
    uint32_t flags = 0;
    for (int64_t r = r0; r < r1; ++r) {
        const int64_t held = d.held[r], added = d.added[r], len = held + added;
        if (held < 0 || added < 0 || len > INT32_MAX || d.base + len > INT32_MAX) {
            flags |= PLAMO_PAGED_COUNT;
            continue;
        }
        const int64_t have = (held + kPgRows - 1) / kPgRows, want = (len + kPgRows - 1) / kPgRows;
        if (want > static_cast<int64_t>(d.table_stride)) flags |= PLAMO_PAGED_TABLE;
        new_rows += added;
        new_pages += want - have;
        most = max(most, static_cast<int32_t>(len));
        most_held = max(most_held, static_cast<int32_t>(held));
    }
    most = __reduce_max_sync(0xffffffffu, most);
    most_held = __reduce_max_sync(0xffffffffu, most_held);
    flags = __reduce_or_sync(0xffffffffu, flags);
    if (lane == 0) {
        atomicMax(&longest, most);
        atomicMax(&longest_held, most_held);
        if (flags) atomicOr(&bad, flags);
    }
    int64_t all_rows, all_pages;
    const int64_t first_row = pg_block_scan<kPlanThreads>(new_rows, sums, &all_rows);
    const int64_t first_page = pg_block_scan<kPlanThreads>(new_pages, sums, &all_pages);
    const int64_t head = d.head ? *d.head : 0;
    uint32_t status = bad;
    if (all_rows > rows) status |= PLAMO_PAGED_BATCH_ROWS;
    if (head < 0 || head + all_pages > static_cast<int64_t>(d.free_count)) status |= PLAMO_PAGED_NO_PAGES;

    const int64_t tile = static_cast<int64_t>(blockIdx.x) * kPlanThreads;
    const int64_t my_row = tile + tid;
    if (status) {  // the step as a whole is declined: the state is that before it
        if (my_row < rows) {
            d.slots[my_row] = -1;
            d.positions[my_row] = 0;
        }
        if (blockIdx.x == 0) {
            for (int64_t r = r0; r < r1; ++r) {
                if (d.lengths) d.lengths[r] = d.held[r];
                d.starts[r + 1] = 0;
            }
            if (tid == 0) {
                d.starts[0] = 0;
                d.summary[0] = static_cast<int32_t>(status);
                d.summary[1] = 0;
                d.summary[2] = static_cast<int32_t>(head);
                d.summary[3] = longest_held;
            }
        }
        return;
    }
    int64_t row = first_row, page = head + first_page;
    for (int64_t r = r0; r < r1; ++r) {
        const int32_t held = d.held[r], added = d.added[r];
        if (blockIdx.x == 0) {
            if (d.lengths) d.lengths[r] = held + added;
            d.starts[r + 1] = static_cast<int32_t>(row + added);
        }
        if (added && row < tile + kPlanThreads && row + added > tile) {
            // The first of its rows in this tile; no two requests share one.
            const int at = static_cast<int>(max(row, tile) - tile);
            mark[at] = at;
            row_start[at] = static_cast<int32_t>(row);
            row_held[at] = held;
            row_owner[at] = static_cast<int32_t>(r);
            row_page[at] = static_cast<int32_t>(page);
        }
        row += added;
        page += (static_cast<int64_t>(held) + added + kPgRows - 1) / kPgRows - (held + kPgRows - 1ll) / kPgRows;
    }
    if (blockIdx.x == 0 && tid == 0) {
        d.starts[0] = 0;
        d.summary[0] = 0;
        d.summary[1] = static_cast<int32_t>(all_rows);
        d.summary[2] = static_cast<int32_t>(head + all_pages);
        d.summary[3] = longest;
    }
    __syncthreads();
    // Latest mark at or before this thread's row.
    int32_t at = mark[tid];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int32_t up = __shfl_up_sync(0xffffffffu, at, o);
        if (lane >= o) at = max(at, up);
    }
    if (lane == 31) warp_mark[warp] = at;
    __syncthreads();
    const int32_t earlier = __reduce_max_sync(0xffffffffu, lane < warp ? warp_mark[lane] : -1);
    at = max(at, earlier);
    if (my_row >= rows) return;
    int32_t slot = -1, position = 0;
    if (my_row < all_rows) {
        const int64_t held = row_held[at], own = held + my_row - row_start[at], k = own / kPgRows;
        const int64_t have = (held + kPgRows - 1) / kPgRows;
        int32_t *entry = d.tables + static_cast<uint64_t>(row_owner[at]) * d.table_stride + k;
        const int32_t id = k >= have ? d.free_pages[row_page[at] + k - have] : *entry;
        if (own % kPgRows == 0) *entry = id;  // a new page, reached by this row
        // (-2: no page has this id; the store reports it, where -1 is padding)
        slot = id >= 0 && id < kPgMaxPages ? id * kPgRows + static_cast<int32_t>(own % kPgRows) : -2;
        position = static_cast<int32_t>(d.base + own);
    }
    d.slots[my_row] = slot;
    d.positions[my_row] = position;
}

// Advances the lengths in place, after every CTA of the plan has read them.
__global__ void __launch_bounds__(kPlanThreads) paged_plan_lengths_kernel(int32_t *lengths, const int32_t *added, const int32_t *summary,
                                                                          uint64_t requests) {
    const uint64_t r = static_cast<uint64_t>(blockIdx.x) * kPlanThreads + threadIdx.x;
    if (r < requests && !summary[0]) lengths[r] += added[r];
}

// ---- store ----------------------------------------------------------------------
// A warp takes HPW heads of one row: lane l holds dimensions 2l, 2l + 1 and
// their rotation partners 64 + 2l, 64 + 2l + 1, so that a head's only exchange
// is the sum of its squares, and the row's cos/sin stay in registers for all of
// its heads. All loads of a warp are issued before the first is used. Streaming:
// 8,191 rows of 40 heads are 168 MB in and 84 MB out, 39 us at the copy rate;
// 42 us back to back (93 %) with eight heads to a warp; four took 3 us more
// (fewer bytes in flight), lanes of four neighbouring dimensions, their partners
// exchanged, 8.
// {x[2l], x[2l + 1], x[64 + 2l], x[64 + 2l + 1]}
template <typename T>
__device__ __forceinline__ float4 pg_load_pairs(const T *x, uint32_t lane) {
    if constexpr (sizeof(T) == 4) {
        const float2 a = *reinterpret_cast<const float2 *>(x + 2 * lane), b = *reinterpret_cast<const float2 *>(x + kPgDim / 2 + 2 * lane);
        return make_float4(a.x, a.y, b.x, b.y);
    } else {
        const uint32_t a = *reinterpret_cast<const uint32_t *>(x + 2 * lane), b = *reinterpret_cast<const uint32_t *>(x + kPgDim / 2 + 2 * lane);
        return make_float4(bf16_lo(a), bf16_hi(a), bf16_lo(b), bf16_hi(b));
    }
}
__device__ __forceinline__ uint32_t pg_pack(float lo, float hi) {  // round to nearest even
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <typename T>
__device__ __forceinline__ void pg_store4(T *p, float4 v) {
    if constexpr (sizeof(T) == 4)
        *reinterpret_cast<float4 *>(p) = v;
    else
        *reinterpret_cast<uint2 *>(p) = make_uint2(pg_pack(v.x, v.y), pg_pack(v.z, v.w));
}

template <typename T>
__device__ __forceinline__ void pg_store_pairs(T *x, uint32_t lane, float4 v) {
    if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float2 *>(x + 2 * lane) = make_float2(v.x, v.y);
        *reinterpret_cast<float2 *>(x + kPgDim / 2 + 2 * lane) = make_float2(v.z, v.w);
    } else {
        *reinterpret_cast<uint32_t *>(x + 2 * lane) = pg_pack(v.x, v.y);
        *reinterpret_cast<uint32_t *>(x + kPgDim / 2 + 2 * lane) = pg_pack(v.z, v.w);
    }
}

template <typename In, typename Out, int HPW>
__global__ void __launch_bounds__(256) paged_store_kernel(plamo_paged_store_args d) {
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t heads = d.query_heads + 2 * d.kv_heads, groups = (heads + HPW - 1) / HPW;
    const uint64_t unit = static_cast<uint64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const uint64_t row = unit / groups;
    const uint32_t h0 = static_cast<uint32_t>(unit % groups) * HPW;
    if (row >= d.rows) return;
    const In *x = static_cast<const In *>(d.qkv) + row * d.qkv_stride;
    float4 v[HPW];
#pragma unroll
    for (int i = 0; i < HPW; ++i)
        if (h0 + i < heads) v[i] = pg_load_pairs(x + static_cast<uint64_t>(h0 + i) * kPgDim, lane);
    const int64_t slot = d.slots[row], position = d.positions[row];
    bool keep = slot >= 0;
    if (slot < -1 || slot >= static_cast<int64_t>(d.pages) * kPgRows) {
        if (lane == 0) pg_flag(d.status, PLAMO_PAGED_PAGE);
        keep = false;
    }
    if (keep && (position < 0 || position >= static_cast<int64_t>(d.positions_count))) {
        if (lane == 0) pg_flag(d.status, PLAMO_PAGED_POSITION);
        keep = false;
    }
    Out *q = static_cast<Out *>(d.q) + row * d.q_stride;
    if (!keep) {
#pragma unroll
        for (int i = 0; i < HPW; ++i)
            if (h0 + i < d.query_heads)
                pg_store_pairs(q + static_cast<uint64_t>(h0 + i) * kPgDim, lane, make_float4(0.f, 0.f, 0.f, 0.f));
        return;
    }
    const float4 turn = pg_load_pairs(d.table + position * kPgDim, lane);  // cos, cos, sin, sin
    const float4 q_norm = pg_load_pairs(d.q_norm, lane), k_norm = pg_load_pairs(d.k_norm, lane);
    const uint64_t page = static_cast<uint64_t>(slot) / kPgRows, off = static_cast<uint64_t>(slot) % kPgRows;
    const uint64_t width = static_cast<uint64_t>(d.kv_heads) * kPgDim;
    Out *key = static_cast<Out *>(d.pool) + (page * 2 * kPgRows + off) * width;
    Out *value = key + kPgRows * width;
#pragma unroll
    for (int i = 0; i < HPW; ++i) {
        const uint32_t h = h0 + i;
        if (h >= heads) break;
        if (h >= d.query_heads + d.kv_heads) {
            pg_store_pairs(value + static_cast<uint64_t>(h - d.query_heads - d.kv_heads) * kPgDim, lane, v[i]);
            continue;
        }
        const bool query = h < d.query_heads;
        // (to 2 ulp; a rounded root and quotient cost 7 us of 55 in 8,191 rows)
        const float inv = rsqrtf(fmaf(warp_sum(sq4(v[i])), 1.0f / kPgDim, 1e-6f));
        const float4 w = query ? q_norm : k_norm;
        const float4 a = make_float4(v[i].x * inv * (w.x + 1.0f), v[i].y * inv * (w.y + 1.0f), v[i].z * inv * (w.z + 1.0f),
                                     v[i].w * inv * (w.w + 1.0f));
        const float4 o = make_float4(fmaf(a.x, turn.x, -a.z * turn.z), fmaf(a.y, turn.y, -a.w * turn.w),
                                     fmaf(a.z, turn.x, a.x * turn.z), fmaf(a.w, turn.y, a.y * turn.w));
        if (query)
            pg_store_pairs(q + static_cast<uint64_t>(h) * kPgDim, lane, o);
        else
            pg_store_pairs(key + static_cast<uint64_t>(h - d.query_heads) * kPgDim, lane, o);
    }
}

}  // namespace plamo

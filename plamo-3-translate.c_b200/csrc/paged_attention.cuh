// Attention of a paged batch step (include/plamo_paged.h).
//
// For a query row i of request r at own row a (position prefix + a) and head h,
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^(s_j - m),  s_j = scale * log2(e) * q . k_j,
// over the prefix rows and own rows j <= a (the last `window` of them), with m
// any number near the maximum of s: the sums over parts of the keys, each with
// its own m, join as sum 2^(m_part - m) (o_part, l_part). The prefix part does
// not depend on the request, so its queries are all rows of the batch at once.
#pragma once
#include "paged.cuh"
#include "tcgen05.cuh"

namespace plamo {

struct PagedAttnParams {
    const void *q;
    void *out;
    const int32_t *starts, *lengths, *tables, *prefix_pages;
    uint64_t q_stride, out_stride, table_stride;
    uint32_t *status;
    uint32_t rows, requests, pages, qh, kh, group;
    int64_t prefix, window;  // window: rows seen, 0 for all
    float scale2;            // scale * log2(e)
    // Partial results, unnormalised: [slot][16][128] sums and [slot][16] {m, l}.
    int2 *own_record;  // [requests] {first own slot / kv heads, splits}
    float *own_sum, *prefix_sum;
    float2 *own_ml, *prefix_ml;
    uint32_t own_groups;  // capacity of the own partials, in slots per KV head
    uint32_t prefix_splits, prefix_tiles;
    uint32_t target;  // own items wanted in all
};

// Row tile of the row kernel: 16 (row, head-in-group) pairs, the M of one MMA.
constexpr int kRtM = 16;
constexpr int kRtWarps = 4;                        // warps sharing a stage's keys
constexpr int kRtThreads = 32 * (kRtWarps + 1);    // and the copying warp
constexpr int kRtStages = 3;
constexpr int kRtStageBytes = 32768;               // keys, then values
constexpr int kRtMinPages = 2;                     // least pages worth an item of their own
constexpr int kRtBatch = 8;                        // items looked up at a time
template <bool F32>
__host__ __device__ constexpr int rt_stage_rows() {
    return F32 ? 32 : 64;
}
constexpr int kRtQBytes = kRtM * kPgDim * 4;  // FP32 queries; joined sums of the warps
constexpr int kRtSmem = 1024 + kRtStages * kRtStageBytes + kRtQBytes;

// A request's new rows and visible own keys.
struct OwnShape {
    int32_t row0, rows;  // batch rows
    int64_t at0;         // own row of the first one (negative: not held)
    int32_t length;      // own rows held
    int32_t page0, pages;
    int32_t tiles;
};
__device__ __forceinline__ OwnShape own_shape(const PagedAttnParams &p, int64_t r) {
    OwnShape s;
    const int64_t lo = min(max(p.starts[r], 0), static_cast<int32_t>(p.rows));
    const int64_t hi = min(max(p.starts[r + 1], 0), static_cast<int32_t>(p.rows));
    s.row0 = static_cast<int32_t>(lo);
    s.rows = static_cast<int32_t>(max(hi - lo, static_cast<int64_t>(0)));
    const int64_t most = min(static_cast<int64_t>(p.table_stride) * kPgRows, static_cast<int64_t>(INT32_MAX));
    s.length = static_cast<int32_t>(min(max(static_cast<int64_t>(p.lengths[r]), static_cast<int64_t>(0)), most));
    s.at0 = static_cast<int64_t>(s.length) - s.rows;
    const int64_t first = p.window ? max(s.at0 - p.window + 1, static_cast<int64_t>(0)) : 0;
    s.page0 = static_cast<int32_t>(first / kPgRows);
    s.pages = s.rows ? max((s.length + kPgRows - 1) / kPgRows - s.page0, 0) : 0;
    s.tiles = static_cast<int32_t>((static_cast<int64_t>(s.rows) * p.group + kRtM - 1) / kRtM);
    return s;
}

struct RowItem {
    int32_t request;  // -1: prefix
    int32_t tile, head;
    int32_t page0, pages;  // of the request's table or the prefix's
    int32_t limit;         // keys from here on hold nothing
    int32_t row0, rows;    // batch rows of the tile's source
    int64_t at0;
    uint32_t slot;
    int32_t direct;  // the only part of its rows: normalise and write the result
};

// 32-way search for the last request whose first row is at or before `row`
// (the one that holds it, since starts never decrease); whole warp.
__device__ __forceinline__ int32_t pg_owner(const int32_t *starts, uint32_t requests, int32_t row) {
    const uint32_t lane = threadIdx.x & 31;
    uint32_t lo = 0, n = requests;  // the answer is in [lo, lo + n)
    while (n > 1) {
        const uint32_t step = (n + 31) / 32;
        const uint32_t at = lo + lane * step;
        const bool below = lane * step < n && starts[at] <= row;
        const uint32_t hits = __ballot_sync(0xffffffffu, below);
        const uint32_t last = hits ? 31 - __clz(hits) : 0;
        const uint32_t used = last * step;
        lo += used;
        n = min(step, n - used);
    }
    return static_cast<int32_t>(lo);
}

__device__ __forceinline__ float pg_exp2(float x) {  // 2^x to about 2 ulp, 2^-inf = 0
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ float lds_f32(uint32_t addr) {
    float v;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t lds_u16(uint32_t addr) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// FP32 as two TF32 terms (11 significant bits each): x = hi + lo to 2^-22.
__device__ __forceinline__ void split_tf32(float x, uint32_t &hi, uint32_t &lo) {
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
    const float rest = __fsub_rn(x, __uint_as_float(hi));
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(rest));
}
__device__ __forceinline__ void rt_bar() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kRtWarps) : "memory"); }

// Byte offset of a 16-byte chunk in a stage's [boxes][rows][128 bytes] tile
// with the copy engine's 128-byte swizzle.
template <int ROWS>
__device__ __forceinline__ uint32_t rt_chunk(uint32_t row, uint32_t chunk) {
    return (chunk >> 3) * (ROWS * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
}

// ---- the row kernel ---------------------------------------------------------------
// Items of 16 (row, head) pairs over a run of pages, persistent CTAs taking
// every gridDim-th item. Own keys are read once per 16 rows and the products
// are far below the tensor pipe's rate, so this is a streaming kernel: one
// warp copies pages into a ring of three 32 KB stages, two CTAs to an SM, and
// the other four each take a quarter of a stage's keys with their own running
// maximum and sums, joined at the end of the item.
template <bool F32>
__global__ void __launch_bounds__(kRtThreads, 2)
    paged_rows_kernel(const __grid_constant__ CUtensorMap map, const PagedAttnParams p) {
    constexpr int SR = rt_stage_rows<F32>(), WK = SR / kRtWarps;  // rows per stage, keys per warp
    constexpr int NK = WK / 8;                                    // 8-key score tiles per warp
    constexpr uint32_t kValues = kRtStageBytes / 2;
    extern __shared__ __align__(128) unsigned char rt_smem[];
    __shared__ __align__(8) uint64_t full[kRtStages], empty[kRtStages];
    __shared__ int32_t stage_page[kRtStages];
    __shared__ int64_t scan[kRtThreads / 32];
    __shared__ RowItem items[kRtBatch];
    __shared__ float2 warp_ml[kRtWarps][kRtM];
    __shared__ int64_t shared_min;
    unsigned char *base = reinterpret_cast<unsigned char *>(
        (reinterpret_cast<uintptr_t>(rt_smem) + 1023) & ~static_cast<uintptr_t>(1023));
    float *qsm = reinterpret_cast<float *>(base + kRtStages * kRtStageBytes);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < kRtStages; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], kRtWarps);
        }
        fence_barrier_init();
        prefetch_tensormap(&map);
    }

    // Every CTA lays the items out by itself from the requests' lengths.
    const int64_t R = p.requests, per = (R + kRtThreads - 1) / kRtThreads;
    const int64_t r0 = min(R, tid * per), r1 = min(R, r0 + per);
    int64_t units = 0, lowest = INT64_MAX;
    for (int64_t r = r0; r < r1; ++r) {
        const OwnShape s = own_shape(p, r);
        units += static_cast<int64_t>(s.tiles) * s.pages;
        if (s.rows) lowest = min(lowest, s.at0);
    }
    int64_t total_units, total;
    pg_block_scan<kRtThreads>(units, scan, &total_units);
    if (tid == 0) shared_min = INT64_MAX;
    __syncthreads();
    if (p.window && lowest != INT64_MAX) atomicMin(reinterpret_cast<long long *>(&shared_min), static_cast<long long>(lowest));
    const int64_t chunk = max(static_cast<int64_t>(kRtMinPages),
                              (total_units * p.kh + p.target - 1) / p.target);
    int64_t mine = 0;
    for (int64_t r = r0; r < r1; ++r) {
        const OwnShape s = own_shape(p, r);
        mine += s.tiles * ((s.pages + chunk - 1) / chunk);
    }
    const int64_t first = pg_block_scan<kRtThreads>(mine, scan, &total);
    if (total > p.own_groups) {
        if (tid == 0) pg_flag(p.status, PLAMO_PAGED_BATCH_ROWS);
        total = p.own_groups;
    }
    if (blockIdx.x == 0) {
        int64_t at = first;
        for (int64_t r = r0; r < r1; ++r) {
            const OwnShape s = own_shape(p, r);
            const int64_t splits = (s.pages + chunk - 1) / chunk, n = s.tiles * splits;
            p.own_record[r] = at + n <= total ? make_int2(static_cast<int>(at), static_cast<int>(splits)) : make_int2(0, 0);
            at += n;
        }
    }
    // Prefix pages that some row still sees.
    const int32_t prefix_pages = static_cast<int32_t>((p.prefix + kPgRows - 1) / kPgRows);
    int32_t pp0 = 0;
    if (p.window && shared_min != INT64_MAX)
        pp0 = static_cast<int32_t>(min(max(p.prefix + shared_min - p.window + 1, static_cast<int64_t>(0)), p.prefix) / kPgRows);
    const int32_t pchunk = p.prefix_splits ? (prefix_pages - pp0 + p.prefix_splits - 1) / static_cast<int32_t>(p.prefix_splits) : 0;
    const int64_t own_items = total * p.kh;
    const int64_t all_items = own_items + static_cast<int64_t>(p.prefix_splits) * p.prefix_tiles * p.kh;

    uint32_t stage = 0, phase = 0, issued = 0;
    bool dead = false;
    for (int64_t batch = blockIdx.x; batch < all_items; batch += static_cast<int64_t>(gridDim.x) * kRtBatch) {
        __syncthreads();  // the last batch's items are done with
#pragma unroll 1
        for (int k = 0; k < kRtBatch; ++k) {
            const int64_t id = batch + static_cast<int64_t>(k) * gridDim.x;
            if (id >= all_items) break;
            if (id >= own_items) {
                if (tid == 0) {
                    const int64_t x = id - own_items, y = x / p.kh;
                    RowItem it;
                    it.request = -1;
                    it.head = static_cast<int32_t>(x % p.kh);
                    it.tile = static_cast<int32_t>(y % p.prefix_tiles);
                    const int32_t split = static_cast<int32_t>(y / p.prefix_tiles);
                    it.page0 = min(pp0 + split * pchunk, prefix_pages);
                    it.pages = min(pchunk, prefix_pages - it.page0);
                    it.limit = static_cast<int32_t>(p.prefix);
                    it.row0 = 0;
                    it.rows = static_cast<int32_t>(p.rows);
                    it.at0 = 0;
                    it.slot = static_cast<uint32_t>(x);
                    it.direct = 0;
                    items[k] = it;
                }
                continue;
            }
            const int64_t group = id / p.kh;
            if (group >= first && group < first + mine) {
                int64_t at = first;
                for (int64_t r = r0; r < r1; ++r) {
                    const OwnShape s = own_shape(p, r);
                    const int64_t splits = (s.pages + chunk - 1) / chunk, n = s.tiles * splits;
                    if (group < at + n) {
                        RowItem it;
                        const int64_t y = group - at;
                        const int32_t split = static_cast<int32_t>(y / s.tiles);
                        it.request = static_cast<int32_t>(r);
                        it.tile = static_cast<int32_t>(y % s.tiles);
                        it.head = static_cast<int32_t>(id % p.kh);
                        it.page0 = s.page0 + static_cast<int32_t>(split * chunk);
                        it.pages = static_cast<int32_t>(min(chunk, s.page0 + static_cast<int64_t>(s.pages) - it.page0));
                        // Keys past the tile's last row are seen by none of its rows.
                        const int64_t last = s.at0 + min(static_cast<int64_t>(s.rows) - 1, (static_cast<int64_t>(it.tile) * kRtM + kRtM - 1) / p.group);
                        it.limit = static_cast<int32_t>(min(max(last + 1, static_cast<int64_t>(0)), static_cast<int64_t>(s.length)));
                        it.row0 = s.row0;
                        it.rows = s.rows;
                        it.at0 = s.at0;
                        it.slot = static_cast<uint32_t>(id);
                        it.direct = splits == 1 && p.prefix_splits == 0;
                        items[k] = it;
                        break;
                    }
                    at += n;
                }
            }
        }
        __syncthreads();
#pragma unroll 1
        for (int k = 0; k < kRtBatch; ++k) {
            if (batch + static_cast<int64_t>(k) * gridDim.x >= all_items) break;
            const RowItem it = items[k];
            const int64_t begin = static_cast<int64_t>(it.page0) * kPgRows;
            const int64_t end = min(begin + static_cast<int64_t>(it.pages) * kPgRows, static_cast<int64_t>(it.limit));
            const int32_t stages = end > begin ? static_cast<int32_t>((end - begin + SR - 1) / SR) : 0;
            if (warp == kRtWarps) {
                // ---- the copying warp: page ids 32 at a time, one lane issues.
                const int32_t *table = it.request < 0 ? p.prefix_pages
                                                      : p.tables + static_cast<uint64_t>(it.request) * p.table_stride;
                constexpr int PER = kPgRows / SR;  // stages per page
                int32_t ids = 0;
                for (int32_t n = 0; n < stages && !dead; ++n) {
                    const int32_t pg = n / PER;
                    if (n % (32 * PER) == 0) ids = pg + lane < it.pages ? table[it.page0 + pg + lane] : -1;
                    int32_t id = __shfl_sync(0xffffffffu, ids, pg & 31);
                    if (lane == 0) {
                        if (issued >= kRtStages && !mbar_wait(&empty[stage], phase ^ 1u)) dead = true;
                        if (!dead) {
                            if (id < 0 || id >= static_cast<int32_t>(p.pages)) {
                                pg_flag(p.status, PLAMO_PAGED_PAGE);
                                id = -1;
                            }
                            stage_page[stage] = id;
                            if (id < 0) {
                                mbar_arrive(&full[stage]);  // nothing to copy
                            } else {
                                unsigned char *dst = base + stage * kRtStageBytes;
                                const int y = id * 2 * kPgRows + (n % PER) * SR, x = it.head * kPgDim;
                                mbar_expect_tx(&full[stage], kRtStageBytes);
                                constexpr int BOX = F32 ? 32 : 64;  // elements in 128 bytes
#pragma unroll
                                for (int b = 0; b < kPgDim / BOX; ++b) {
                                    tma_load_2d(dst + b * SR * 128, &map, x + b * BOX, y, &full[stage]);
                                    tma_load_2d(dst + kValues + b * SR * 128, &map, x + b * BOX, y + kPgRows, &full[stage]);
                                }
                            }
                        }
                    }
                    dead = __shfl_sync(0xffffffffu, dead, 0);
                    ++issued;
                    if (++stage == kRtStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                continue;
            }
            // ---- the computing warps
            const int g = lane >> 2, t = lane & 3;
            // This thread's two rows of the tile (g and g + 8): which keys they see.
            int32_t see_lo[2], see_hi[2];
            bool there[2];
            const int64_t pairs = static_cast<int64_t>(it.rows) * p.group;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int64_t m = static_cast<int64_t>(it.tile) * kRtM + g + 8 * x;
                see_lo[x] = see_hi[x] = 0;
                there[x] = m < pairs;
                if (!there[x]) continue;
                const int32_t i = static_cast<int32_t>(m / p.group);
                if (it.request >= 0) {
                    const int64_t at = it.at0 + i;
                    see_hi[x] = static_cast<int32_t>(max(at + 1, static_cast<int64_t>(0)));
                    if (p.window) see_lo[x] = static_cast<int32_t>(max(at - p.window + 1, static_cast<int64_t>(0)));
                } else {
                    see_hi[x] = static_cast<int32_t>(p.prefix);
                }
            }
            if (it.request < 0 && p.window) {
                for (int m = 0; m < kRtM; ++m) {  // position of each row: its request's length decides
                    const int64_t pair = static_cast<int64_t>(it.tile) * kRtM + m;
                    if (pair >= pairs) break;
                    const int32_t i = static_cast<int32_t>(pair / p.group);
                    int32_t lo = 0;
                    if (R) {
                        const OwnShape s = own_shape(p, pg_owner(p.starts, p.requests, i));
                        const int64_t at = s.at0 + i - s.row0;
                        lo = static_cast<int32_t>(min(max(p.prefix + at - p.window + 1, static_cast<int64_t>(0)), p.prefix));
                    }
                    if ((m & 7) == g) see_lo[m >> 3] = lo;
                }
            }
            // Queries: BF16 as MMA fragments in registers, FP32 in shared memory in fragment order.
            uint32_t qf[F32 ? 1 : kPgDim / 16][4];
            {
                const uint64_t head0 = static_cast<uint64_t>(it.head) * p.group;
                const unsigned char *row_ptr[2];
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const int64_t m = static_cast<int64_t>(it.tile) * kRtM + g + 8 * x;
                    row_ptr[x] = nullptr;
                    if (m < pairs) {
                        const uint64_t row = static_cast<uint64_t>(it.row0) + m / p.group, h = head0 + m % p.group;
                        row_ptr[x] = static_cast<const unsigned char *>(p.q) + (row * p.q_stride + h * kPgDim) * (F32 ? 4 : 2);
                    }
                }
                if constexpr (F32) {
                    // k-step ks: {row g dim 8ks+t, row g+8, row g dim 8ks+t+4, row g+8} at [ks][lane]
                    rt_bar();  // the last item's joined sums have been read
                    for (int ks = warp; ks < kPgDim / 8; ks += kRtWarps) {
                        float4 v;
                        const float *a = reinterpret_cast<const float *>(row_ptr[0]), *b = reinterpret_cast<const float *>(row_ptr[1]);
                        v.x = a ? a[8 * ks + t] : 0.0f;
                        v.y = b ? b[8 * ks + t] : 0.0f;
                        v.z = a ? a[8 * ks + t + 4] : 0.0f;
                        v.w = b ? b[8 * ks + t + 4] : 0.0f;
                        reinterpret_cast<float4 *>(qsm)[ks * 32 + lane] = v;
                    }
                    rt_bar();
                } else {
#pragma unroll
                    for (int ks = 0; ks < kPgDim / 16; ++ks)
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const unsigned char *src = row_ptr[x & 1];
                            qf[ks][x] = src ? *reinterpret_cast<const uint32_t *>(src + 2 * (16 * ks + 2 * t + 8 * (x >> 1))) : 0u;
                        }
                }
            }
            float o[16][4];
#pragma unroll
            for (int j = 0; j < 16; ++j)
#pragma unroll
                for (int x = 0; x < 4; ++x) o[j][x] = 0.0f;
            float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};

            for (int32_t n = 0; n < stages && !dead; ++n) {
                if (!mbar_wait(&full[stage], phase)) dead = true;
                dead = __any_sync(0xffffffffu, dead);
                if (dead) break;
                const int32_t key0 = static_cast<int32_t>(begin) + n * SR + warp * WK;  // this warp's first key
                // Only warps with keys that exist: the copy brings whole boxes.
                if (stage_page[stage] >= 0 && key0 < end) {
                    const uint32_t kbase = smem_u32(base + stage * kRtStageBytes), vbase = kbase + kValues;
                    const uint32_t krow = warp * WK;
                    float s[NK][4];
                    if constexpr (F32) {
                        // Products of the high terms in two chains, the cross terms in a third:
                        // the tensor cores truncate as they add, so chains are kept short.
                        float c0[4] = {0, 0, 0, 0}, c1[4] = {0, 0, 0, 0}, c2[4] = {0, 0, 0, 0};
#pragma unroll
                        for (int ks = 0; ks < kPgDim / 8; ++ks) {
                            const float4 qv = reinterpret_cast<const float4 *>(qsm)[ks * 32 + lane];
                            uint32_t ah[4], al[4], bh0, bl0, bh1, bl1;
                            split_tf32(qv.x, ah[0], al[0]);
                            split_tf32(qv.y, ah[1], al[1]);
                            split_tf32(qv.z, ah[2], al[2]);
                            split_tf32(qv.w, ah[3], al[3]);
                            split_tf32(lds_f32(kbase + rt_chunk<SR>(krow + g, 2 * ks) + 4 * t), bh0, bl0);
                            split_tf32(lds_f32(kbase + rt_chunk<SR>(krow + g, 2 * ks + 1) + 4 * t), bh1, bl1);
                            if (ks & 1) mma_tf32(c1, ah, bh0, bh1);
                            else mma_tf32(c0, ah, bh0, bh1);
                            mma_tf32(c2, ah, bl0, bl1);
                            mma_tf32(c2, al, bh0, bh1);
                        }
#pragma unroll
                        for (int x = 0; x < 4; ++x) s[0][x] = __fadd_rn(__fadd_rn(c0[x], c1[x]), c2[x]);
                    } else {
#pragma unroll
                        for (int j = 0; j < NK; ++j)
#pragma unroll
                            for (int x = 0; x < 4; ++x) s[j][x] = 0.0f;
                        const uint32_t r = krow + (lane >> 4) * 8 + (lane & 7), half = (lane >> 3) & 1;
#pragma unroll
                        for (int ks = 0; ks < kPgDim / 16; ++ks) {
                            uint32_t b[4];
                            ldsm4(kbase + rt_chunk<SR>(r, 2 * ks + half), b);
                            mma_bf16(s[0], qf[ks], b[0], b[1]);
                            mma_bf16(s[1], qf[ks], b[2], b[3]);
                        }
                    }
                    // Masks and the running maximum.
                    bool hidden = false;  // a key that exists is masked for one of this thread's rows
                    float top[2] = {mx[0], mx[1]};
#pragma unroll
                    for (int j = 0; j < NK; ++j)
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const int32_t key = key0 + 8 * j + 2 * t + (x & 1);
                            const int row = x >> 1;
                            const bool seen = key >= see_lo[row] && key < see_hi[row] && key < end;
                            hidden |= there[row] && !seen && key < end;
                            s[j][x] = seen ? s[j][x] * p.scale2 : -INFINITY;
                            top[row] = fmaxf(top[row], s[j][x]);
                        }
                    float corr[2];
#pragma unroll
                    for (int row = 0; row < 2; ++row) {
                        top[row] = fmaxf(top[row], __shfl_xor_sync(0xffffffffu, top[row], 1));
                        top[row] = fmaxf(top[row], __shfl_xor_sync(0xffffffffu, top[row], 2));
                        corr[row] = top[row] == -INFINITY ? 1.0f : pg_exp2(mx[row] - top[row]);
                        mx[row] = top[row];
                        sum[row] *= corr[row];
                    }
#pragma unroll
                    for (int j = 0; j < NK; ++j)
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            const int row = x >> 1;
                            s[j][x] = mx[row] == -INFINITY ? 0.0f : pg_exp2(s[j][x] - mx[row]);
                        }
                    const bool scaled = __any_sync(0xffffffffu, corr[0] != 1.0f || corr[1] != 1.0f);
                    if (scaled) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            o[j][0] *= corr[0];
                            o[j][1] *= corr[0];
                            o[j][2] *= corr[1];
                            o[j][3] *= corr[1];
                        }
                    }
                    // A weight of zero times a value that is not finite would be NaN: such values
                    // leave the products and are added where they are seen. Only tiles with masked
                    // keys are looked over; keys past `end` are zeroed in any case.
                    const bool careful = __any_sync(0xffffffffu, hidden);
                    const bool tail = key0 + WK > end;
                    bool odd = false;
                    if constexpr (F32) {
#pragma unroll
                        for (int x = 0; x < 4; ++x) sum[x >> 1] += s[0][x];
                        // Score column 2t is product index t, 2t + 1 is t + 4.
                        uint32_t ph[4], pl[4];
                        split_tf32(s[0][0], ph[0], pl[0]);
                        split_tf32(s[0][2], ph[1], pl[1]);
                        split_tf32(s[0][1], ph[2], pl[2]);
                        split_tf32(s[0][3], ph[3], pl[3]);
                        const bool in0 = key0 + 2 * t < end, in1 = key0 + 2 * t + 1 < end;
#pragma unroll
                        for (int j = 0; j < 16; ++j) {
                            const uint32_t chunk = 2 * j + (g >> 2), word = 4 * (g & 3);
                            float v0 = lds_f32(vbase + rt_chunk<SR>(krow + 2 * t, chunk) + word);
                            float v1 = lds_f32(vbase + rt_chunk<SR>(krow + 2 * t + 1, chunk) + word);
                            if (tail || careful) {
                                const bool bad0 = !isfinite(v0), bad1 = !isfinite(v1);
                                odd |= (in0 && bad0) || (in1 && bad1);
                                if (!in0 || bad0) v0 = 0.0f;
                                if (!in1 || bad1) v1 = 0.0f;
                            }
                            uint32_t vh0, vl0, vh1, vl1;
                            split_tf32(v0, vh0, vl0);
                            split_tf32(v1, vh1, vl1);
                            float c[4] = {0, 0, 0, 0};
                            mma_tf32(c, ph, vl0, vl1);
                            mma_tf32(c, pl, vh0, vh1);
                            mma_tf32(c, ph, vh0, vh1);
#pragma unroll
                            for (int x = 0; x < 4; ++x) o[j][x] = __fadd_rn(o[j][x], c[x]);
                        }
                    } else {
                        uint32_t pf[4];
                        pf[0] = pg_pack(s[0][0], s[0][1]);
                        pf[1] = pg_pack(s[0][2], s[0][3]);
                        pf[2] = pg_pack(s[1][0], s[1][1]);
                        pf[3] = pg_pack(s[1][2], s[1][3]);
                        // The sums are those of the rounded weights.
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            s[x >> 1][2 * (x & 1)] = bf16_lo(pf[x]);
                            s[x >> 1][2 * (x & 1) + 1] = bf16_hi(pf[x]);
                            sum[x & 1] += bf16_lo(pf[x]) + bf16_hi(pf[x]);
                        }
                        const uint32_t r = krow + ((lane >> 3) & 1) * 8 + (lane & 7), half = lane >> 4;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            uint32_t b[4];
                            ldsm4_t(vbase + rt_chunk<SR>(r, 2 * j + half), b);
                            if (tail || careful) {
#pragma unroll
                                for (int x = 0; x < 4; ++x) {
                                    const int32_t key = key0 + 2 * t + 8 * (x & 1);
                                    const bool bad0 = (b[x] & 0x7f80u) == 0x7f80u, bad1 = (b[x] & 0x7f800000u) == 0x7f800000u;
                                    odd |= (bad0 && key < end) || (bad1 && key + 1 < end);
                                    if (bad0 || key >= end) b[x] &= 0xffff0000u;
                                    if (bad1 || key + 1 >= end) b[x] &= 0x0000ffffu;
                                }
                            }
                            mma_bf16(o[2 * j], pf, b[0], b[1]);
                            mma_bf16(o[2 * j + 1], pf, b[2], b[3]);
                        }
                    }
                    if ((tail || careful) && __any_sync(0xffffffffu, odd)) {
#pragma unroll 1
                        for (int key = 0; key < WK; ++key) {
                            if (key0 + key >= end) break;
                            // This row pair's weights of the key, from the lane that holds them.
                            float w[2];
#pragma unroll
                            for (int row = 0; row < 2; ++row) {
                                const int src = (lane & ~3) | ((key & 7) >> 1);
                                float a = 0.0f;
#pragma unroll
                                for (int j = 0; j < NK; ++j)
#pragma unroll
                                    for (int c = 0; c < 2; ++c) {
                                        const float x = __shfl_sync(0xffffffffu, s[j][2 * row + c], src);
                                        if (key == 8 * j + (key & 6) + c) a = x;
                                    }
                                w[row] = a;
                            }
                            const bool seen0 = key0 + key >= see_lo[0] && key0 + key < see_hi[0];
                            const bool seen1 = key0 + key >= see_lo[1] && key0 + key < see_hi[1];
#pragma unroll
                            for (int j = 0; j < 16; ++j)
#pragma unroll
                                for (int c = 0; c < 2; ++c) {
                                    const uint32_t dim = 8 * j + 2 * t + c;
                                    float v;
                                    if constexpr (F32)
                                        v = lds_f32(vbase + rt_chunk<SR>(krow + key, dim / 4) + 4 * (dim & 3));
                                    else
                                        v = __uint_as_float(lds_u16(vbase + rt_chunk<SR>(krow + key, dim / 8) + 2 * (dim & 7)) << 16);
                                    if (!isfinite(v)) {
                                        if (seen0) o[j][c] += w[0] * v;
                                        if (seen1) o[j][2 + c] += w[1] * v;
                                    }
                                }
                        }
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&empty[stage]);
                if (++stage == kRtStages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }

            // ---- join the warps' sums: {m, l} of each row, then the sums one warp after another
#pragma unroll
            for (int row = 0; row < 2; ++row) {
                sum[row] += __shfl_xor_sync(0xffffffffu, sum[row], 1);
                sum[row] += __shfl_xor_sync(0xffffffffu, sum[row], 2);
                if (t == 0) warp_ml[warp][g + 8 * row] = make_float2(mx[row], sum[row]);
            }
            rt_bar();  // and, FP32, every warp is done with the queries
            float factor[2];
            float2 joined[2];
#pragma unroll
            for (int row = 0; row < 2; ++row) {
                float top = -INFINITY, l = 0.0f;
#pragma unroll
                for (int w = 0; w < kRtWarps; ++w) top = fmaxf(top, warp_ml[w][g + 8 * row].x);
#pragma unroll
                for (int w = 0; w < kRtWarps; ++w) {
                    const float2 ml = warp_ml[w][g + 8 * row];
                    if (ml.x != -INFINITY) l += pg_exp2(ml.x - top) * ml.y;
                }
                factor[row] = mx[row] == -INFINITY ? 0.0f : pg_exp2(mx[row] - top);
                joined[row] = make_float2(top, l);
            }
#pragma unroll 1
            for (int w = 0; w < kRtWarps; ++w) {
                if (w == warp) {
#pragma unroll
                    for (int j = 0; j < 16; ++j)
#pragma unroll
                        for (int row = 0; row < 2; ++row) {
                            float2 *dst = reinterpret_cast<float2 *>(qsm + (g + 8 * row) * kPgDim + 8 * j + 2 * t);
                            float2 v = make_float2(o[j][2 * row] * factor[row], o[j][2 * row + 1] * factor[row]);
                            if (w) {
                                const float2 before = *dst;
                                v = make_float2(before.x + v.x, before.y + v.y);
                            }
                            *dst = v;
                        }
                    if (w == kRtWarps - 1 && t == 0) {
                        warp_ml[0][g] = joined[0];
                        warp_ml[0][g + 8] = joined[1];
                    }
                }
                rt_bar();
            }
            // ---- result, or the tile's partial sums
            const int ctid = tid;  // 0..127
            if (it.direct) {
                for (int x = ctid; x < kRtM * kPgDim / 4; x += 32 * kRtWarps) {
                    const int m16 = x / (kPgDim / 4), d = 4 * (x % (kPgDim / 4));
                    const int64_t m = static_cast<int64_t>(it.tile) * kRtM + m16;
                    if (m >= pairs) continue;
                    const float l = warp_ml[0][m16].y, inv = warp_ml[0][m16].x == -INFINITY ? 0.0f : 1.0f / l;
                    float4 v = *reinterpret_cast<const float4 *>(qsm + m16 * kPgDim + d);
                    v = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
                    const uint64_t row = static_cast<uint64_t>(it.row0) + m / p.group;
                    const uint64_t at = row * p.out_stride + (static_cast<uint64_t>(it.head) * p.group + m % p.group) * kPgDim + d;
                    if constexpr (F32) pg_store4(static_cast<float *>(p.out) + at, v);
                    else pg_store4(static_cast<uint16_t *>(p.out) + at, v);
                }
            } else {
                float *dst = (it.request < 0 ? p.prefix_sum : p.own_sum) + static_cast<uint64_t>(it.slot) * kRtM * kPgDim;
                float2 *ml = (it.request < 0 ? p.prefix_ml : p.own_ml) + static_cast<uint64_t>(it.slot) * kRtM;
                for (int x = ctid; x < kRtM * kPgDim / 4; x += 32 * kRtWarps)
                    reinterpret_cast<float4 *>(dst)[x] = reinterpret_cast<const float4 *>(qsm)[x];
                if (ctid < kRtM) ml[ctid] = warp_ml[0][ctid];
            }
            rt_bar();  // before the next item writes warp_ml or the sums
        }
    }
    if (warp == kRtWarps && lane == 0) {
        // Every copy issued has landed before the CTA can exit.
        const uint32_t from = issued > kRtStages ? issued - kRtStages : 0;
        for (uint32_t n = from; n < issued; ++n)
            if (!mbar_wait(&full[n % kRtStages], (n / kRtStages) & 1u)) break;
    }
    if (dead && lane == 0) pg_flag(p.status, PLAMO_PAGED_FAILED);
    pdl_launch_dependents();
}

// ---- joining the parts ----------------------------------------------------------------
// One warp per (row, query head): the prefix's splits and the request's own,
// always in the same order. Rows with one part were written by the row kernel.
template <bool F32>
__global__ void __launch_bounds__(256) paged_join_kernel(const PagedAttnParams p) {
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t row = blockIdx.x, head = blockIdx.y * 8 + (threadIdx.x >> 5);
    pdl_wait();
    if (head >= p.qh) return;
    const uint32_t kv = head / p.group, in_group = head % p.group;
    OwnShape s{};
    int2 rec = make_int2(0, 0);
    bool real = false;
    if (p.requests && static_cast<int32_t>(row) < p.starts[p.requests]) {
        const int32_t r = pg_owner(p.starts, p.requests, static_cast<int32_t>(row));
        s = own_shape(p, r);
        const int64_t i = static_cast<int64_t>(row) - s.row0;
        real = i >= 0 && i < s.rows && s.at0 + i >= 0;
        rec = p.own_record[r];
    }
    if (real && rec.y == 1 && p.prefix_splits == 0) return;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float top = -INFINITY, l = 0.0f;
    if (real) {
        const uint64_t m = static_cast<uint64_t>(row - s.row0) * p.group + in_group;
        const uint64_t pm = static_cast<uint64_t>(row) * p.group + in_group;
        const uint32_t parts = p.prefix_splits + rec.y;
        auto slot = [&](uint32_t x) -> uint64_t {
            if (x < p.prefix_splits) return (static_cast<uint64_t>(x) * p.prefix_tiles + pm / kRtM) * p.kh + kv;
            return (static_cast<uint64_t>(rec.x) + static_cast<uint64_t>(x - p.prefix_splits) * s.tiles + m / kRtM) * p.kh + kv;
        };
        for (uint32_t x = lane; x < parts; x += 32)
            top = fmaxf(top, x < p.prefix_splits ? p.prefix_ml[slot(x) * kRtM + pm % kRtM].x : p.own_ml[slot(x) * kRtM + m % kRtM].x);
        top = warp_max(top);
        if (top != -INFINITY)
            for (uint32_t x = 0; x < parts; ++x) {
                const bool shared = x < p.prefix_splits;
                const uint64_t at = slot(x) * kRtM + (shared ? pm : m) % kRtM;
                const float2 ml = shared ? p.prefix_ml[at] : p.own_ml[at];
                if (ml.x == -INFINITY) continue;
                const float w = pg_exp2(ml.x - top);
                const float4 v = ld4((shared ? p.prefix_sum : p.own_sum) + at * kPgDim + 4 * lane);
                o = make_float4(fmaf(w, v.x, o.x), fmaf(w, v.y, o.y), fmaf(w, v.z, o.z), fmaf(w, v.w, o.w));
                l = fmaf(w, ml.y, l);
            }
    }
    const float inv = top == -INFINITY ? 0.0f : 1.0f / l;
    o = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    const uint64_t at = row * p.out_stride + static_cast<uint64_t>(head) * kPgDim + 4 * lane;
    if constexpr (F32) pg_store4(static_cast<float *>(p.out) + at, o);
    else pg_store4(static_cast<uint16_t *>(p.out) + at, o);
}

}  // namespace plamo

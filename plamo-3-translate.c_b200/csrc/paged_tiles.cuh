// Attention of a paged batch step on the tensor cores: BF16, 256 (row, head)
// pairs to a tile. Serves the prefix, whose queries are all of the batch's
// short requests' rows at once, and the prompts among the requests.
#pragma once
#include "paged_attention.cuh"

namespace plamo {

// A tile is two halves of 128 pairs (the M of one MMA), each with its own
// scores, weights and sums in tensor memory and four warps of softmax; both
// read the same keys and values, 128 at a time. Tensor memory (512 columns):
// scores of half i at 128 i (FP32; the weights replace them, 64 keys in 64
// columns: 32 of a first BF16 term, 32 of the second), sums at 256 + 128 i. Per
// 128 keys each half needs 512 cycles of the tensor pipe for the scores and two
// times 512 for the values (128 x 128 x 128 at 4096 multiply-adds a cycle) and
// 1024 cycles of exponentials (16 a cycle): the halves run half a step apart,
// so that one's exponentials cover the other's products. Measured: 329 GFLOP of
// ragged prompts behind 2,048 rows in 614 us, 0.54 PFLOP/s, the tensor pipe busy
// for 43 % of it (the weights' second term among that). A half's chain bounds it,
// 3 us a step: scores, softmax, the value product, and the next scores only when
// that is done, since they replace the weights; then 8 us at each segment's ends.
// The value product takes both operands in one type and the values are BF16, so
// the FP32 weights go in as two BF16 terms, 16 bits together: the results are
// then the exact ones rounded to BF16 (those prompts: 1.66e-3 from 64 bits,
// relative L2). One term was 2.32e-3 off in 502 us beside the unrounded weights'
// sums, 2.30e-3 in 508 us beside the rounded ones'; on rows whose weight lies on
// few keys those two differ more.
constexpr int kTlPairs = 256;
constexpr int kTlKeys = 128;
constexpr int kTlThreads = 352;  // 8 softmax warps, copies, products, mending
constexpr int kTlCopies = 8, kTlProducts = 9, kTlMending = 10;  // warps; 0-7 are softmax
constexpr int kTlUnitBytes = kTlKeys * kPgDim * 2;  // keys or values of a step
constexpr int kTlUnits = 5;
constexpr int kTlQBytes = kTlPairs * kPgDim * 2;
constexpr int kTlSmem = 1024 + kTlQBytes + kTlUnits * kTlUnitBytes;

// Tile t of a prompt (its rows [t * tile_rows, ...)).
__device__ __forceinline__ TileShape prompt_tile(const PagedAttnParams &p, int32_t request, const OwnShape &o, int32_t t) {
    TileShape s{};
    const int32_t first = t * p.tile_rows;
    s.request = request;
    s.row0 = o.row0 + first;
    s.rows = min(p.tile_rows, o.rows - first);
    s.at0 = o.at0 + first;
    const int32_t last = s.at0 + s.rows - 1;
    if (last < 0) return s;  // rows before own row 0 see nothing
    const int32_t held = max(s.at0, 0);
    s.pre1 = (p.prefix + p.tile_keys - 1) / p.tile_keys;
    s.pre0 = p.window ? min(max(p.prefix + held - p.window + 1, 0) / p.tile_keys, s.pre1) : 0;
    s.own_limit = min(last + 1, o.length);
    s.own1 = (s.own_limit + p.tile_keys - 1) / p.tile_keys;
    s.own0 = p.window ? min(max(held - p.window + 1, 0) / p.tile_keys, s.own1) : 0;
    return s;
}

// ---- the schedule ---------------------------------------------------------------------
// The row kernel's first CTA sorts the requests into short ones (their own rows
// are the row kernel's, their rows are listed, and share the prefix's tiles)
// and prompts (tiles of their own over prefix and own rows), and numbers the
// key steps of all tiles. A step of a tile and KV head is the unit of work: the
// tile kernel's CTAs take equal runs of consecutive ones.
__device__ void paged_schedule(const PagedAttnParams &p, int64_t *sums) {
    __shared__ int32_t first_at;
    const int tid = threadIdx.x;
    const int32_t per = (p.requests + kRtThreads - 1) / kRtThreads;
    const int32_t r0 = min(p.requests, tid * per), r1 = min(p.requests, r0 + per);
    if (tid == 0) first_at = INT32_MAX;
    __syncthreads();
    // 64 bits: starts that decrease make ranges that overlap, and their sums more than there is of
    // either. Nothing is laid out then.
    int decreases = 0;
    int64_t short_rows = 0, prompt_tiles = 0, all_short_rows, all_tiles = 0;
    int32_t lowest = INT32_MAX;
#pragma unroll 1
    for (int32_t r = r0; r < r1; ++r) {
        const OwnShape s = own_shape(p, r);
        if (p.lengths[r] > p.max_length) pg_flag(p.status, PLAMO_PAGED_TABLE);
        if (p.lengths[r] < 0) pg_flag(p.status, PLAMO_PAGED_COUNT);
        if (p.starts[r] < 0 || p.starts[r + 1] > p.rows) pg_flag(p.status, PLAMO_PAGED_BATCH_ROWS);
        decreases |= p.starts[r + 1] < p.starts[r];
        if (request_is_short(p, s)) {
            short_rows += s.rows;
            if (s.rows) lowest = min(lowest, max(s.at0, 0));
        } else {
            prompt_tiles += p.by_tile_rows.div(s.rows + p.tile_rows - 1);
        }
    }
    lowest = __reduce_min_sync(0xffffffffu, lowest);
    if ((tid & 31) == 0) atomicMin(&first_at, lowest);
    int64_t short_at = pg_block_scan<kRtThreads>(short_rows, sums, &all_short_rows);
    int64_t tile_at = p.tile_rows ? pg_block_scan<kRtThreads>(prompt_tiles, sums, &all_tiles) : 0;
    const bool ordered = !__syncthreads_or(decreases);
    const int32_t all_short = ordered ? static_cast<int32_t>(all_short_rows) : 0;
    int32_t pre_tiles = 0;
    TileShape pre{};
    if (p.tile_rows && p.prefix) {
        pre_tiles = p.by_tile_rows.div(all_short + p.tile_rows - 1);
        pre.request = -1;
        pre.pre1 = (p.prefix + p.tile_keys - 1) / p.tile_keys;
        if (p.window && first_at != INT32_MAX) pre.pre0 = min(max(p.prefix + first_at - p.window + 1, 0) / p.tile_keys, pre.pre1);
    }
    bool fits = ordered && pre_tiles + all_tiles <= p.tile_cap;  // (no tile kernel: 0 <= 0)
    if (!fits) pre_tiles = all_tiles = 0;
    const int32_t all = pre_tiles + static_cast<int32_t>(all_tiles);
#pragma unroll 1
    for (int32_t r = r0; r < r1; ++r) {
        const OwnShape s = own_shape(p, r);
        if (request_is_short(p, s)) {
#pragma unroll 1
            for (int32_t i = 0; i < s.rows && short_at + i < all_short; ++i)
                p.short_list[short_at + i] = make_int4(s.row0 + i, max(s.at0 + i, -1), r, i);
            short_at += s.rows;
        } else if (fits) {
            const int32_t n = p.by_tile_rows.div(s.rows + p.tile_rows - 1);
#pragma unroll 1
            for (int32_t t = 0; t < n; ++t, ++tile_at) {  // whose it is; the rest below, by all threads
                p.tile_shape[pre_tiles + tile_at].request = r;
                p.tile_shape[pre_tiles + tile_at].row0 = t;
            }
        }
    }
    __syncthreads();
    int64_t total = 0;
#pragma unroll 1
    for (int32_t t0 = 0; t0 < all; t0 += kRtThreads) {
        const int32_t t = t0 + tid;
        TileShape shape{};
        if (t < pre_tiles) {
            shape = pre;
            shape.row0 = t * p.tile_rows;
            shape.rows = min(p.tile_rows, all_short - shape.row0);
        } else if (t < all) {
            const int32_t r = p.tile_shape[t].request;
            shape = prompt_tile(p, r, own_shape(p, r), p.tile_shape[t].row0);
        }
        int64_t sum;
        const int64_t at = total + pg_block_scan<kRtThreads>(shape.steps(), sums, &sum);
        if (t < all) {
            p.tile_shape[t] = shape;
            p.tile_unit[t] = static_cast<uint32_t>(at);
        }
        total += sum;
    }
    fits = fits && total * p.kh <= INT32_MAX - 256;
    if (tid == 0) {
        const int32_t first = p.requests ? p.starts[0] : 0, taken = p.requests ? p.starts[p.requests] : 0;
        if (!fits || first) pg_flag(p.status, PLAMO_PAGED_BATCH_ROWS);
        // Rows of no request, [0, first) and [taken, rows), become zeros; so do all of a batch that
        // is not laid out.
        p.header[kTlFirst] = fits ? min(max(first, 0), p.rows) : 0;
        p.header[kTlTaken] = fits ? min(max(taken, 0), p.rows) : 0;
        p.header[kTlShortRows] = fits ? all_short : 0;
        const int32_t units = fits ? static_cast<int32_t>(total * p.kh) : 0;
        const int32_t ctas = p.tile_rows ? min(p.tile_grid, (units + kTlMinUnits - 1) / kTlMinUnits) : 0;
        p.header[kTlCtas] = ctas;
        p.header[kTlRun] = ctas ? units / ctas : 1;
        p.header[kTlLonger] = ctas ? units % ctas : 0;
        if (p.tile_rows) {
            p.tile_unit[fits ? all : 0] = fits ? static_cast<uint32_t>(total) : 0;
            p.header[kTlTiles] = fits ? all : 0;
            p.header[kTlPreTiles] = fits ? pre_tiles : 0;
        }
    }
}

// ---- the tile kernel ---------------------------------------------------------------------
// A wait that ends when the phase completes, after about two seconds, or when
// another warp gave up.
__device__ __forceinline__ bool tl_wait(uint64_t *bar, uint32_t parity, volatile int *gave_up) {
    uint64_t start = 0;
    for (uint32_t n = 1; !mbar_try_wait(bar, parity); ++n) {
        if (n % 64) continue;  // the clock is slow to read
        if (*gave_up) return false;
        const uint64_t now = global_ns();
        if (!start) start = now;
        if (now - start > 2000000000ull) {
            *gave_up = 1;
            return false;
        }
    }
    return true;
}
// Whether the values of a step are looked over before use: keys past the end,
// or keys that exist and some row of the tile does not see.
__device__ __forceinline__ bool step_is_mended(const PagedAttnParams &p, const TileShape &s, int32_t step, bool *masked) {
    const bool own = step >= s.pre1 - s.pre0;
    const int32_t key0 = (own ? s.own0 + step - (s.pre1 - s.pre0) : s.pre0 + step) * p.tile_keys;
    const int32_t limit = own ? s.own_limit : p.prefix;
    bool m = s.request >= 0 && s.at0 < 0;
    if (own) m |= s.at0 + 1 < min(key0 + p.tile_keys, limit) || (p.window && max(s.at0 + s.rows, 0) - p.window > key0);
    else if (p.window) m |= s.request < 0 || p.prefix + max(s.at0 + s.rows, 0) - p.window > key0;
    *masked = m;
    return m || key0 + p.tile_keys > limit;
}

// Bits k of the 32 in [lo, hi).
__device__ __forceinline__ uint32_t tl_bits(int32_t lo, int32_t hi) {
    const uint32_t below = hi <= 0 ? 0u : hi >= 32 ? 0xffffffffu : (1u << hi) - 1u;
    return below & (lo <= 0 ? 0xffffffffu : lo >= 32 ? 0u : 0xffffffffu << lo);
}

// Piece c (16 bytes) of row r of a warp's 32 rows of 256 bytes, laid out as an
// MMA operand: two blocks of 128 bytes a row, swizzled.
__device__ __forceinline__ uint4 *tl_piece(unsigned char *rows, int r, int c) {
    return reinterpret_cast<uint4 *>(rows + (c >> 3) * (kTlKeys * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// The segments of a CTA: runs of steps of one (tile, KV head).
struct TileWalk {
    int32_t unit, end;                // of this CTA
    int32_t tile, head, step, steps;  // current segment: first step and count
    int32_t tile_steps;
};
__device__ __noinline__ bool walk_next(const PagedAttnParams &p, TileWalk &w) {
    if (w.unit >= w.end) return false;
    for (;; ++w.tile) {
        const int32_t t0 = p.tile_unit[w.tile], t1 = p.tile_unit[w.tile + 1];
        if (w.unit >= t1 * p.kh) continue;
        w.tile_steps = t1 - t0;
        const int32_t x = w.unit - t0 * p.kh;
        w.head = x / w.tile_steps;
        w.step = x - w.head * w.tile_steps;
        w.steps = min(w.tile_steps - w.step, w.end - w.unit);
        return true;
    }
}

// Values that are not finite left the products of steps with masked keys: the
// rows that see them get them here (a weight times one of them is itself).
__device__ __noinline__ void add_odd_values(const PagedAttnParams &p, const TileShape &s, const TileWalk &w, int32_t at, int c, float (&o)[32]) {
    const int32_t pre_steps = s.pre1 - s.pre0;
    for (int32_t n = 0; n < w.steps; ++n) {
        const int32_t step = w.step + n;
        bool masked;
        step_is_mended(p, s, step, &masked);
        if (!masked) continue;
        const bool own = step >= pre_steps;
        const int32_t key0 = (own ? s.own0 + step - pre_steps : s.pre0 + step) * kTlKeys;
        const int32_t hi = at < 0 ? 0 : min(key0 + kTlKeys, own ? min(at + 1, s.own_limit) : p.prefix);
        const int32_t lo = p.window ? max(key0, (own ? at : p.prefix + at) - p.window + 1) : key0;
#pragma unroll 1
        for (int32_t key = lo; key < hi; ++key) {
            const int32_t id = own ? p.tables[static_cast<uint64_t>(s.request) * p.table_stride + key / kPgRows] : p.prefix_pages[key / kPgRows];
            if (id < 0 || id >= p.pages) continue;
            const uint16_t *v = static_cast<const uint16_t *>(p.pool) + ((static_cast<uint64_t>(id) * 2 + 1) * kPgRows + key % kPgRows) * p.kh * kPgDim +
                                static_cast<uint64_t>(w.head) * kPgDim + c;
#pragma unroll 1
            for (int k = 0; k < 32; ++k) {
                const float x = bf16_to_f32(v[k]);
                if (!isfinite(x)) o[k] += x;
            }
        }
    }
}

__global__ void __launch_bounds__(kTlThreads, 1)
    paged_tile_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ PagedAttnParams p) {
    extern __shared__ __align__(128) unsigned char tl_smem[];
    __shared__ __align__(8) uint64_t full[kTlUnits], empty[kTlUnits];
    __shared__ __align__(8) uint64_t q_full[2], s_full[2], p_full[2], pv_done[2], mended[kTlUnits];
    __shared__ uint32_t tmem_base;
    __shared__ int gave_up, odd_values;
    unsigned char *base = reinterpret_cast<unsigned char *>(
        (reinterpret_cast<uintptr_t>(tl_smem) + 1023) & ~static_cast<uintptr_t>(1023));
    unsigned char *units_at = base + kTlQBytes;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < kTlUnits; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 2);  // the products, and the mending warp
            mbar_init(&mended[s], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 4);
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
            mbar_init(&pv_done[i], 1);
        }
        gave_up = odd_values = 0;
        fence_barrier_init();
        prefetch_tensormap(&map);
    }
    if (warp == kTlProducts) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_base;
    pdl_launch_dependents();
    pdl_wait();

    const int32_t ctas = p.header[kTlCtas], cta = static_cast<int32_t>(blockIdx.x);
    const int32_t tiles = p.header[kTlTiles], pre_tiles = p.header[kTlPreTiles];
    TileWalk w{};
    if (cta < ctas) {
        const Runs runs = tile_runs(p);
        w.unit = runs.start(cta);
        w.end = runs.start(cta + 1);
        w.tile = pg_owner(reinterpret_cast<const int32_t *>(p.tile_unit), static_cast<uint32_t>(tiles), p.by_kh.div(w.unit));
    }
    volatile int *quit = &gave_up;
    bool ok = true;

    if (warp == kTlCopies) {
        // ---- copies: keys and values of each step alternate in the ring
        uint32_t q = 0;
        for (; ok && walk_next(p, w); w.unit += w.steps) {
            const TileShape s = p.tile_shape[w.tile];
            const int32_t pre_steps = s.pre1 - s.pre0;
            const int32_t *own_table = p.tables + static_cast<uint64_t>(max(s.request, 0)) * p.table_stride;
            const int32_t pre_pages = (p.prefix + kPgRows - 1) / kPgRows;
            const int32_t own_pages = (s.own_limit + kPgRows - 1) / kPgRows;
            for (int32_t base_step = 0; base_step < w.steps && ok; base_step += 16) {
                // Page ids of 16 steps, two to a step.
                int32_t id = -1;
                bool there = false;
                {
                    const int32_t st = w.step + base_step + (lane >> 1);
                    if (base_step + (lane >> 1) < w.steps) {
                        const bool own = st >= pre_steps;
                        const int32_t pg = 2 * (own ? s.own0 + st - pre_steps : s.pre0 + st) + (lane & 1);
                        there = pg < (own ? own_pages : pre_pages);
                        if (there) id = own ? own_table[pg] : p.prefix_pages[pg];
                    }
                }
                if (there && (id < 0 || id >= p.pages)) {
                    pg_flag(p.status, PLAMO_PAGED_PAGE);
                    id = p.pages;  // past the pool: reads as zeros
                }
                const uint32_t present = __ballot_sync(0xffffffffu, there);
                #pragma unroll 1
                for (int32_t k = 0; k < 16 && base_step + k < w.steps && ok; ++k) {
                    const int32_t id0 = __shfl_sync(0xffffffffu, id, 2 * k), id1 = __shfl_sync(0xffffffffu, id, 2 * k + 1);
                    const bool two = (present >> (2 * k + 1)) & 1;
                    if (lane == 0) {
#pragma unroll 1
                        for (int kind = 0; kind < 2 && ok; ++kind, ++q) {
                            const uint32_t st = q % kTlUnits;
                            if (q >= kTlUnits && !tl_wait(&empty[st], (q / kTlUnits - 1) & 1u, quit)) {
                                ok = false;
                                break;
                            }
                            unsigned char *dst = units_at + st * kTlUnitBytes;
                            mbar_expect_tx(&full[st], two ? kTlUnitBytes : kTlUnitBytes / 2);
                            const int x = w.head * kPgDim, y0 = (id0 * 2 + kind) * kPgRows, y1 = (id1 * 2 + kind) * kPgRows;
                            tma_load_2d(dst, &map, x, y0, &full[st]);
                            tma_load_2d(dst + kTlUnitBytes / 2, &map, x + 64, y0, &full[st]);
                            if (two) {
                                tma_load_2d(dst + kPgRows * 128, &map, x, y1, &full[st]);
                                tma_load_2d(dst + kTlUnitBytes / 2 + kPgRows * 128, &map, x + 64, y1, &full[st]);
                            }
                        }
                    }
                    ok = __shfl_sync(0xffffffffu, ok, 0);
                }
            }
        }
        if (lane == 0) {  // every copy issued has landed before the CTA can exit
            for (uint32_t n = q > kTlUnits ? q - kTlUnits : 0; n < q; ++n)
                if (!mbar_wait(&full[n % kTlUnits], (n / kTlUnits) & 1u)) break;
        }
    } else if (warp == kTlProducts) {
        // ---- products: one lane issues, the halves in turn
        if (lane == 0) {
            constexpr uint32_t idesc_s = tc_idesc(128, kTlKeys), idesc_o = tc_idesc(128, kPgDim) | kTcIdescMnB;
            // Units of the segments before; waited phases of the queries and weights (bit i), and of each place's mending.
            uint32_t q = 0, queries = 0, weights = 0, products = 0, mends = 0;
            const uint64_t q_desc = smem_desc_sw128(smem_u32(base)), k_desc = smem_desc_sw128(smem_u32(units_at));
            const uint64_t v_desc = smem_desc_mn_sw128(smem_u32(units_at), kTlKeys * 128);
            // (addresses in descriptors count 16 bytes)
            const auto scores = [&](uint32_t i, uint32_t place) {
                const uint64_t a = q_desc + i * (kTlQBytes / 2 / 16), b = k_desc + place * (kTlUnitBytes / 16);
#pragma unroll
                for (int k = 0; k < kPgDim / 16; ++k) {
                    const uint32_t off = ((k / 4) * (kTlKeys * 128) + (k % 4) * 32) / 16;
                    tc_mma(tmem + 128 * i, a + off, b + off, idesc_s, k ? 1u : 0u);
                }
                tc_commit(&s_full[i]);
            };
            for (; ok && walk_next(p, w); w.unit += w.steps) {
                const TileShape s = p.tile_shape[w.tile];
                const uint32_t halves = s.rows * p.group > 128 ? 2 : 1;
                ok = tl_wait(&full[q % kTlUnits], (q / kTlUnits) & 1u, quit);
                for (uint32_t i = 0; i < halves && ok; ++i) {
                    ok = tl_wait(&q_full[i], (queries >> i) & 1u, quit);
                    queries ^= 1u << i;
                    if (!ok) break;
                    tc_fence_after();
                    scores(i, q % kTlUnits);
                }
                if (!ok) break;
                tc_commit(&empty[q % kTlUnits]);
                for (int32_t n = 0; n < w.steps && ok; ++n, q += 2) {
                    const uint32_t v = q + 1, vs = v % kTlUnits, ks = (q + 2) % kTlUnits;
                    const bool more = n + 1 < w.steps;
                    bool masked;
                    ok = tl_wait(&full[vs], (v / kTlUnits) & 1u, quit);
                    if (ok && step_is_mended(p, s, w.step + n, &masked)) {
                        ok = tl_wait(&mended[vs], (mends >> vs) & 1u, quit);
                        mends ^= 1u << vs;
                    }
                    if (ok && more) ok = tl_wait(&full[ks], ((q + 2) / kTlUnits) & 1u, quit);
                    for (uint32_t i = 0; i < halves && ok; ++i) {
                        ok = tl_wait(&p_full[i], (weights >> i) & 1u, quit);
                        weights ^= 1u << i;
                        if (!ok) break;
                        tc_fence_after();
                        const uint64_t b = v_desc + vs * (kTlUnitBytes / 16);
#pragma unroll
                        for (int k = 0; k < kTlKeys / 16; ++k) {  // both terms of 16 keys' weights
                            const uint32_t a = tmem + 128 * i + 64 * (k / 4) + 8 * (k % 4);
                            tc_mma_ts(tmem + 256 + 128 * i, a, b + k * 128, idesc_o, n || k ? 1u : 0u);
                            tc_mma_ts(tmem + 256 + 128 * i, a + 32, b + k * 128, idesc_o, 1u);
                        }
                        tc_commit(&pv_done[i]);
                        if (more) {  // the next scores replace the weights just read
                            ok = tl_wait(&pv_done[i], (products >> i) & 1u, quit);
                            if (!ok) break;
                            tc_fence_after();
                            scores(i, ks);
                        }
                        products ^= 1u << i;
                    }
                    tc_commit(&empty[vs]);
                    if (more) tc_commit(&empty[ks]);
                }
            }
        }
    } else if (warp == kTlMending) {
        // ---- mending: values that no weight may touch become zero before the products read them
        uint32_t q = 0;
        for (; ok && walk_next(p, w); w.unit += w.steps) {
            const TileShape s = p.tile_shape[w.tile];
            const int32_t pre_steps = s.pre1 - s.pre0;
            for (int32_t n = 0; n < w.steps && ok; ++n) {
                for (int kind = 0; kind < 2 && ok; ++kind, ++q) {
                    const uint32_t st = q % kTlUnits;
                    ok = tl_wait(&full[st], (q / kTlUnits) & 1u, quit);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    bool masked;
                    if (kind && step_is_mended(p, s, w.step + n, &masked)) {
                        const int32_t step = w.step + n;
                        const bool own = step >= pre_steps;
                        const int32_t key0 = (own ? s.own0 + step - pre_steps : s.pre0 + step) * kTlKeys;
                        const int32_t limit = own ? s.own_limit : p.prefix;
                        unsigned char *unit = units_at + st * kTlUnitBytes;
                        bool odd = false;
                        for (int c = lane; c < kTlUnitBytes / 16; c += 32) {  // 16-byte pieces, row by row
                            const int row = (c >> 3) & (kTlKeys - 1);
                            uint4 *at = reinterpret_cast<uint4 *>(unit + 16 * c);
                            if (key0 + row >= limit) {
                                *at = make_uint4(0, 0, 0, 0);
                            } else if (masked) {
                                uint4 v = *at;
                                bool bad = false;
                                uint32_t *word = reinterpret_cast<uint32_t *>(&v);
#pragma unroll
                                for (int x = 0; x < 4; ++x) {
                                    if ((word[x] & 0x7f80u) == 0x7f80u) {
                                        word[x] &= 0xffff0000u;
                                        bad = true;
                                    }
                                    if ((word[x] & 0x7f800000u) == 0x7f800000u) {
                                        word[x] &= 0x0000ffffu;
                                        bad = true;
                                    }
                                }
                                if (bad) *at = v;
                                odd |= bad;
                            }
                        }
                        if (odd) odd_values = 1;
                        fence_async_shared();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&mended[st]);
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&empty[st]);
                }
            }
        }
    } else {
        // ---- softmax: a thread per pair
        const int i = warp >> 2;  // half
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t scol = tmem + lanes + 128 * i, ocol = tmem + lanes + 256 + 128 * i;
        const int pair = 128 * i + (warp & 3) * 32 + lane;
        uint32_t n_scores = 0, n_sums = 0;
        for (bool begins = true; ok && walk_next(p, w); w.unit += w.steps, begins = false) {
            const TileShape s = p.tile_shape[w.tile];
            const int32_t pairs = s.rows * p.group, pre_steps = s.pre1 - s.pre0;
            const bool active = i == 0 || pairs > 128, there = pair < pairs;
            const int32_t local = p.by_group.div(pair);
            int32_t row = s.row0 + local, at = s.at0 + local;
            if (s.request < 0 && there) {
                const int4 e = p.short_list[row];
                row = e.x;
                at = e.y;
            }
            const int32_t head = w.head * p.group + pair - local * p.group;
            if (!active) continue;
            // Queries into shared memory as an MMA operand: 16 lanes to a row of 256 bytes.
            unsigned char *const rows_at = base + i * (kTlQBytes / 2) + (warp & 3) * 32 * 128;  // of this warp: two halves
            {
                const int64_t from = there ? row * static_cast<int64_t>(p.q_stride) + head * kPgDim : -1;
                const uint32_t flip = p.scale2 < 0.0f ? 0x80008000u : 0u;
                const int c = lane & 15;
                uint4 v[16];
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    const int64_t src = __shfl_sync(0xffffffffu, from, 2 * k + (lane >> 4));
                    v[k] = make_uint4(0, 0, 0, 0);
                    if (src >= 0) v[k] = *reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p.q) + src + 8 * c);
                }
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    *tl_piece(rows_at, 2 * k + (lane >> 4), c) = make_uint4(v[k].x ^ flip, v[k].y ^ flip, v[k].z ^ flip, v[k].w ^ flip);
                fence_async_shared();
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[i]);

            const float scale2 = fabsf(p.scale2);
            // Keys this row sees, prefix and own: [lo, hi).
            const int32_t pre_hi = at < 0 ? 0 : p.prefix, own_hi = at < 0 ? 0 : min(at + 1, s.own_limit);
            const int32_t pre_lo = p.window ? max(p.prefix + max(at, 0) - p.window + 1, 0) : 0;
            const int32_t own_lo = p.window ? max(max(at, 0) - p.window + 1, 0) : 0;
            float m = -INFINITY, l = 0.0f;
            for (int32_t n = 0; n < w.steps; ++n) {
                ok = tl_wait(&s_full[i], n_scores & 1u, quit);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                ++n_scores;
                tc_fence_after();
                // Keys this row sees, of this step's: [lo, hi).
                const int32_t step = w.step + n;
                const bool own = step >= pre_steps;
                const int32_t key0 = (own ? s.own0 + step - pre_steps : s.pre0 + step) * kTlKeys;
                const int32_t hi = min(max((own ? own_hi : pre_hi) - key0, 0), kTlKeys);
                const int32_t lo = min(max((own ? own_lo : pre_lo) - key0, 0), kTlKeys);
                const bool partial = __any_sync(0xffffffffu, there && (lo > 0 || hi < kTlKeys));
                // 64 scores at a time, twice: for the maximum, then for the weights, which replace them
                // (two BF16 terms). Loops, not straight code: a segment is a few steps long, and
                // code that runs a few times costs its fetching.
                uint32_t x[64];
                const auto load = [&](int half) {
                    tmem_ld32_async(scol + 64 * half, reinterpret_cast<uint32_t(&)[32]>(x[0]));
                    tmem_ld32_async(scol + 64 * half + 32, reinterpret_cast<uint32_t(&)[32]>(x[32]));
                    tmem_wait_ld();
                    if (partial) {
                        const uint32_t see0 = tl_bits(lo - 64 * half, hi - 64 * half), see1 = tl_bits(lo - 64 * half - 32, hi - 64 * half - 32);
#pragma unroll
                        for (int k = 0; k < 64; ++k)
                            if (!((k < 32 ? see0 : see1) >> (k & 31) & 1u)) x[k] = 0xff800000u;  // -inf
                    }
                };
                float top = -INFINITY;
#pragma unroll 1
                for (int half = 1; half >= 0; --half) {
                    load(half);
                    float t[4] = {top, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int k = 0; k < 64; k += 8)
#pragma unroll
                        for (int y = 0; y < 4; ++y) t[y] = fmaxf(fmaxf(t[y], __uint_as_float(x[k + 2 * y])), __uint_as_float(x[k + 2 * y + 1]));
                    top = fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
                }
                top *= scale2;
                // The reference point moves only when passed by 2^8: the weights stay below 2^8, FP32
                // sums and BF16 weights lose nothing by it, and the sums in tensor memory are rarely
                // touched.
                const bool move = top > m + kLazy;
                if (__any_sync(0xffffffffu, move)) {
                    const float factor = move ? pg_exp2(m - top) : 1.0f;
                    if (move) m = top;
                    l *= factor;
                    if (n) {  // this half's last products are done: the scores came after them
#pragma unroll 1
                        for (int c = 0; c < kPgDim; c += 32) {
                            uint32_t r[32];
                            tmem_ld32_async(ocol + c, r);
                            tmem_wait_ld();
#pragma unroll
                            for (int k = 0; k < 32; ++k) r[k] = __float_as_uint(__uint_as_float(r[k]) * factor);
                            tmem_st32(ocol + c, r);
                        }
                        load(0);
                    }
                }
                const float shift = m == -INFINITY ? 0.0f : -m;
                float l0 = 0.0f, l1 = 0.0f;
#pragma unroll 1
                for (int half = 0; half < 2; ++half) {
                    if (half) load(1);  // (the first half is there from before)
#pragma unroll
                    for (int part = 0; part < 2; ++part) {
                        uint32_t r[16], rest[16];
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            const float a = pg_exp2(fmaf(__uint_as_float(x[32 * part + 2 * k]), scale2, shift));
                            const float b = pg_exp2(fmaf(__uint_as_float(x[32 * part + 2 * k + 1]), scale2, shift));
                            l0 += a;
                            l1 += b;
                            pg_split(a, b, r[k], rest[k]);
                        }
                        tmem_st16(scol + 64 * half + 16 * part, r);
                        tmem_st16(scol + 64 * half + 32 + 16 * part, rest);
                    }
                }
                l += l0 + l1;
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[i]);
            }
            if (!ok) break;
            // ---- the segment's sums
            n_sums += w.steps;
            ok = tl_wait(&pv_done[i], (n_sums - 1) & 1u, quit);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const bool whole = w.steps == w.tile_steps && w.tile >= pre_tiles;
            const int32_t slot = w.tile < pre_tiles ? 2 * p.tile_grid + cta + w.tile * p.kh + w.head : 2 * cta + (begins ? 0 : 1);
            const bool odd = *reinterpret_cast<volatile int *>(&odd_values);
            const float inv = pg_inverse(at, l);
            // Through shared memory (the queries' place: the scores are done with them), so that rows
            // leave 256 bytes at a time: the whole result, or half of the partial sums.
            const int64_t to = !there ? -1 : whole ? row * static_cast<int64_t>(p.out_stride) + head * kPgDim
                                                   : (static_cast<int64_t>(slot) * kTlPairs + pair) * kPgDim;
#pragma unroll 1
            for (int c = 0; c < kPgDim; c += 32) {
                uint32_t r[32];
                tmem_ld32_async(ocol + c, r);
                tmem_wait_ld();
                float o[32];
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = __uint_as_float(r[k]);
                if (odd && there) {
                    float more[32];
#pragma unroll
                    for (int k = 0; k < 32; ++k) more[k] = o[k];
                    add_odd_values(p, s, w, at, c, more);
#pragma unroll
                    for (int k = 0; k < 32; ++k) o[k] = more[k];
                }
                __syncwarp();
                if (whole) {
#pragma unroll
                    for (int k = 0; k < 32; k += 8)
                        *tl_piece(rows_at, lane, (c + k) / 8) =
                            make_uint4(pg_pack(o[k] * inv, o[k + 1] * inv), pg_pack(o[k + 2] * inv, o[k + 3] * inv),
                                       pg_pack(o[k + 4] * inv, o[k + 5] * inv), pg_pack(o[k + 6] * inv, o[k + 7] * inv));
                } else {
#pragma unroll
                    for (int k = 0; k < 32; k += 4)
                        *tl_piece(rows_at, lane, ((c & 32) + k) / 4) =
                            make_uint4(__float_as_uint(o[k]), __float_as_uint(o[k + 1]), __float_as_uint(o[k + 2]), __float_as_uint(o[k + 3]));
                }
                if (c == kPgDim - 32 || (!whole && c == 32)) {
                    __syncwarp();
                    const int piece = lane & 15;
#pragma unroll 4
                    for (int k = 0; k < 16; ++k) {
                        const int64_t dst = __shfl_sync(0xffffffffu, to, 2 * k + (lane >> 4));
                        const uint4 v = *tl_piece(rows_at, 2 * k + (lane >> 4), piece);
                        if (dst < 0) continue;
                        if (whole) *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.out) + dst + 8 * piece) = v;
                        else *reinterpret_cast<uint4 *>(p.tile_sum + dst + (c & 64) + 4 * piece) = v;
                    }
                    __syncwarp();
                }
            }
            if (there && !whole) p.tile_ml[static_cast<int64_t>(slot) * kTlPairs + pair] = pg_ml(m, l);
            tc_fence_before();
        }
    }
    if (!ok && lane == 0) pg_flag(p.status, PLAMO_PAGED_FAILED);
    tc_fence_before();
    __syncthreads();
    if (warp == kTlProducts) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// ---- FP32 tiles ------------------------------------------------------------------------------
// FP32 has no products on the tensor cores, so these tiles run on the CUDA
// cores, 64 pairs by steps of 64 keys (a page), 128 threads, two CTAs to an SM
// so that one multiplies while the other waits for its copies. Both products
// are register-tiled: thread (ty, tx) of 8 x 16 holds the scores of pairs 8 ty
// to 8 ty + 7 with keys tx + 16 j (128 multiply-adds to 12 shared loads of 16
// bytes) and the sums of the same pairs in dimensions 4 tx and 64 + 4 tx (64 to
// 4). Bound: 128 multiply-adds a cycle and SM, 8192 cycles for a step's two
// products. (Three BF16 terms to an operand on tcgen05 would be bound by six
// products each, 3072 cycles, with a fold to FP32 registers every step as the
// projections' tiles have it: a kernel of its own, not written.)
constexpr int kTfPairs = 64, kTfKeys = 64, kTfThreads = 128;
constexpr int kTfTile = kTfKeys * kPgDim * 4;  // keys, values or queries
constexpr int kTfTables = 3 * kTfTile + kTfPairs * kTfKeys * 4;  // barriers and the pairs' rows behind the tiles
constexpr int kTfSmem = kTfTables + 16 + 2 * kTfPairs * 4;       // no static part: two CTAs just fit an SM

// A 16-byte piece of row r: the copy engine's swizzle; the queries' rows r and
// r + 8, read together, lie apart too; the weights' keys are rows.
__device__ __forceinline__ const float4 *tf_piece(const unsigned char *base, int r, int c) {
    return reinterpret_cast<const float4 *>(base + (c >> 3) * (kTfKeys * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}
__device__ __forceinline__ float4 *tf_query(unsigned char *base, int r, int c) {
    return reinterpret_cast<float4 *>(base + r * 512 + (c >> 3) * 128 + (((c & 7) ^ ((r + (r >> 3)) & 7)) << 4));
}
__device__ __forceinline__ float4 *tf_weight(unsigned char *base, int key, int c) {
    return reinterpret_cast<float4 *>(base + key * (kTfPairs * 4) + ((c ^ (key & 15)) << 4));
}

__device__ __forceinline__ float4 lds_f32x4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}

__global__ void __launch_bounds__(kTfThreads, 2)
    paged_tile_f32_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ PagedAttnParams p) {
    extern __shared__ __align__(1024) unsigned char tf_smem[];
    unsigned char *const base = tf_smem;
    uint64_t *const full = reinterpret_cast<uint64_t *>(base + kTfTables);           // keys, values
    int32_t *const pair_row = reinterpret_cast<int32_t *>(base + kTfTables + 16);    // batch row, -1: no such pair
    int32_t *const pair_at = pair_row + kTfPairs;                                    // own row
    if (smem_u32(base) & 1023u) {  // the copies' swizzle needs it; dynamic shared memory starts so when there is no other
        pg_flag(p.status, PLAMO_PAGED_FAILED);
        return;
    }
    unsigned char *const tile_at[2] = {base, base + kTfTile};
    unsigned char *const queries = base + 2 * kTfTile, *const weights = base + 3 * kTfTile;
    const int tid = threadIdx.x, lane = tid & 31, tx = tid & 15, ty = tid >> 4;
    if (tid == 0) {
        mbar_init(&full[0], 1);
        mbar_init(&full[1], 1);
        fence_barrier_init();
        prefetch_tensormap(&map);
    }
    __syncthreads();
    pdl_launch_dependents();
    pdl_wait();
    const int32_t ctas = p.header[kTlCtas], cta = static_cast<int32_t>(blockIdx.x);
    const int32_t tiles = p.header[kTlTiles], pre_tiles = p.header[kTlPreTiles];
    if (cta >= ctas) return;
    const Runs runs = tile_runs(p);
    TileWalk w{};
    w.unit = runs.start(cta);
    w.end = runs.start(cta + 1);
    w.tile = pg_owner(reinterpret_cast<const int32_t *>(p.tile_unit), static_cast<uint32_t>(tiles), p.by_kh.div(w.unit));
    bool ok = true;
    uint32_t phase = 0;
#pragma unroll 1
    for (bool begins = true; ok && walk_next(p, w); w.unit += w.steps, begins = false) {
        const TileShape s = p.tile_shape[w.tile];
        const int32_t pre_steps = s.pre1 - s.pre0, pairs = s.rows * p.group;
        // Step n's page, first key and the key from which on nothing is seen.
        const auto key0_of = [&](int32_t step) { return (step >= pre_steps ? s.own0 + step - pre_steps : s.pre0 + step) * kTfKeys; };
        const auto copy = [&](int32_t n, int kind) {  // one thread
            const int32_t step = w.step + n, page = key0_of(step) / kTfKeys;
            int32_t id = step >= pre_steps ? p.tables[static_cast<uint64_t>(s.request) * p.table_stride + page] : p.prefix_pages[page];
            if (id < 0 || id >= p.pages) {
                pg_flag(p.status, PLAMO_PAGED_PAGE);
                id = p.pages;  // past the pool: reads as zeros
            }
            mbar_expect_tx(&full[kind], kTfTile);
#pragma unroll
            for (int b = 0; b < 4; ++b)
                tma_load_2d(tile_at[kind] + b * kTfKeys * 128, &map, w.head * kPgDim + 32 * b, (id * 2 + kind) * kPgRows, &full[kind]);
        };
        __syncthreads();  // the last segment's tiles and tables have been read
        if (tid == 0) {
            copy(0, 0);
            copy(0, 1);
        }
        const bool whole = w.steps == w.tile_steps && w.tile >= pre_tiles;
        const int32_t slot = w.tile < pre_tiles ? 2 * p.tile_grid + cta + w.tile * p.kh + w.head : 2 * cta + (begins ? 0 : 1);
        if (tid < kTfPairs) {
            int32_t row = -1, at = 0;
            if (tid < pairs) {
                const int32_t local = p.by_group.div(tid);
                row = s.row0 + local;
                at = s.at0 + local;
                if (s.request < 0) {
                    const int4 e = p.short_list[row];
                    row = e.x;
                    at = e.y;
                }
            }
            pair_row[tid] = row;
            pair_at[tid] = at;
        }
        const auto head_of = [&](int32_t pair) { return w.head * p.group + pair - p.by_group.div(pair) * p.group; };
        __syncthreads();
        {
            float4 v[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {  // a warp to a row of 512 bytes
                const int32_t pair = 4 * k + (tid >> 5), row = pair_row[pair];
                v[k] = row >= 0 ? ld4(static_cast<const float *>(p.q) + row * p.q_stride + head_of(pair) * kPgDim + 4 * lane)
                                : make_float4(0.f, 0.f, 0.f, 0.f);
            }
#pragma unroll
            for (int k = 0; k < 16; ++k) *tf_query(queries, 4 * k + (tid >> 5), lane) = v[k];
        }
        float o[8][8], m[8], l[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            m[i] = -INFINITY;
            l[i] = 0.0f;
#pragma unroll
            for (int d = 0; d < 8; ++d) o[i][d] = 0.0f;
        }
        __syncthreads();
#pragma unroll 1
        for (int32_t n = 0; n < w.steps; ++n) {
            const int32_t step = w.step + n, key0 = key0_of(step);
            const bool own = step >= pre_steps;
            const int32_t limit = own ? s.own_limit : p.prefix;
            ok = mbar_wait(&full[0], phase);
            if (__syncthreads_or(!ok)) {
                ok = false;
                break;
            }
            float x[8][4];
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) x[i][j] = 0.0f;
            {
                // Addresses: a row's swizzle and the piece's number join by exclusive or. The next
                // piece's loads are under way while this one is multiplied.
                uint32_t k_at[4], q_at[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) k_at[j] = smem_u32(tf_piece(tile_at[0], tx + 16 * j, 0));
#pragma unroll
                for (int i = 0; i < 8; ++i) q_at[i] = smem_u32(tf_query(queries, 8 * ty + i, 0));
                float4 k[2][4], q[2][8];
                const auto load = [&](int four, int c) {  // piece 4 four + c
                    const uint32_t turn = (four & 1) << 6, k_box = (four >> 1) * (kTfKeys * 128), q_box = (four >> 1) * 128;
#pragma unroll
                    for (int j = 0; j < 4; ++j) k[c & 1][j] = lds_f32x4(((k_at[j] ^ turn) ^ (c << 4)) + k_box);
#pragma unroll
                    for (int i = 0; i < 8; ++i) q[c & 1][i] = lds_f32x4(((q_at[i] ^ turn) ^ (c << 4)) + q_box);
                };
                load(0, 0);
#pragma unroll 1
                for (int four = 0; four < kPgDim / 16; ++four)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        if (c < 3) load(four, c + 1);
                        else if (four < kPgDim / 16 - 1) load(four + 1, 0);
#pragma unroll
                        for (int i = 0; i < 8; ++i)
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const float4 a = q[c & 1][i], b = k[c & 1][j];
                                x[i][j] = fmaf(a.w, b.w, fmaf(a.z, b.z, fmaf(a.y, b.y, fmaf(a.x, b.x, x[i][j]))));
                            }
                    }
            }
            // Keys that each pair sees, of this step's: [lo, hi).
            int32_t lo[8], hi[8];
            bool move = false;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int32_t at = pair_at[8 * ty + i], place = max(at, 0) + (own ? 0 : p.prefix);
                lo[i] = p.window ? max(place - p.window + 1 - key0, 0) : 0;
                hi[i] = at < 0 ? 0 : min((own ? min(at + 1, limit) : limit) - key0, kTfKeys);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int key = tx + 16 * j;
                    x[i][j] = key >= lo[i] && key < hi[i] ? x[i][j] * p.scale2 : -INFINITY;
                    move |= x[i][j] > m[i] + kLazy;
                }
            }
            // (the pairs of a thread are those of 16 lanes; both halves of a warp take the turn together)
            if (__any_sync(0xffffffffu, move)) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float top = fmaxf(fmaxf(fmaxf(x[i][0], x[i][1]), fmaxf(x[i][2], x[i][3])), m[i]);
#pragma unroll
                    for (int b = 1; b < 16; b <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, b));
                    const float corr = top == -INFINITY ? 1.0f : pg_exp2(m[i] - top);
                    m[i] = top;
                    l[i] *= corr;
#pragma unroll
                    for (int d = 0; d < 8; ++d) o[i][d] *= corr;
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float y[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    y[i] = pg_exp2(x[i][j] - (m[i] == -INFINITY ? 0.0f : m[i]));
                    l[i] += y[i];
                }
                *tf_weight(weights, tx + 16 * j, 2 * ty) = make_float4(y[0], y[1], y[2], y[3]);
                *tf_weight(weights, tx + 16 * j, 2 * ty + 1) = make_float4(y[4], y[5], y[6], y[7]);
            }
            ok = mbar_wait(&full[1], phase);
            // A weight of zero leaves a value out only if that is finite: where keys are hidden from
            // some pair, the values are looked over.
            bool masked, odd = false;
            const int32_t valid = min(limit - key0, kTfKeys);  // keys that exist
            step_is_mended(p, s, step, &masked);
            if (masked) {
#pragma unroll 4
                for (int k = tid; k < valid * (kPgDim / 4); k += kTfThreads) {
                    const float4 v = *tf_piece(tile_at[1], k >> 5, k & 31);
                    odd |= !(isfinite(v.x) && isfinite(v.y) && isfinite(v.z) && isfinite(v.w));
                }
                odd = __syncthreads_or(odd);
            }
            if (__syncthreads_or(!ok)) {  // the weights are there, and the keys have been read
                ok = false;
                break;
            }
            if (tid == 0 && n + 1 < w.steps) copy(n + 1, 0);
            const auto add = [&](int key, float4 a, float4 b, float4 u, float4 v, bool all) {
                const float y[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}, z[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (all || (key >= lo[i] && key < hi[i])) {
#pragma unroll
                        for (int d = 0; d < 8; ++d) o[i][d] = fmaf(y[i], z[d], o[i][d]);
                    }
            };
            // Eights of keys at full speed; the rest, and all where a value is odd, for the pairs that
            // see them only.
            const int eights = odd ? 0 : valid / 8;
            if (eights) {
                const uint32_t w_at = smem_u32(tf_weight(weights, 0, 2 * ty)), v_at = smem_u32(tf_piece(tile_at[1], 0, tx));
                float4 a[2], b[2], u[2], v[2];
                const auto load = [&](int eight, int key) {  // key 8 eight + key
                    const uint32_t wa = ((w_at ^ ((eight & 1) << 7)) ^ (key << 4)) + (8 * eight + key) * (kTfPairs * 4);
                    const uint32_t va = (v_at ^ (key << 4)) + (8 * eight + key) * 128;
                    a[key & 1] = lds_f32x4(wa);
                    b[key & 1] = lds_f32x4(wa ^ 16);
                    u[key & 1] = lds_f32x4(va);
                    v[key & 1] = lds_f32x4(va + 2 * kTfKeys * 128);
                };
                load(0, 0);
#pragma unroll 1
                for (int eight = 0; eight < eights; ++eight)
#pragma unroll
                    for (int key = 0; key < 8; ++key) {
                        if (key < 7) load(eight, key + 1);
                        else if (eight < eights - 1) load(eight + 1, 0);
                        add(key, a[key & 1], b[key & 1], u[key & 1], v[key & 1], true);
                    }
            }
#pragma unroll 1
            for (int key = 8 * eights; key < valid; ++key)
                add(key, *tf_weight(weights, key, 2 * ty), *tf_weight(weights, key, 2 * ty + 1), *tf_piece(tile_at[1], key, tx),
                    *tf_piece(tile_at[1], key, 16 + tx), false);
            __syncthreads();  // values and weights have been read
            if (tid == 0 && n + 1 < w.steps) copy(n + 1, 1);
            phase ^= 1u;
        }
        if (!ok) break;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float sum = l[i];
#pragma unroll
            for (int b = 1; b < 16; b <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, b);
            const int pair = 8 * ty + i;
            const int32_t row = pair_row[pair];
            if (row < 0) continue;
            const uint64_t to = whole ? row * p.out_stride + head_of(pair) * kPgDim : (static_cast<uint64_t>(slot) * kTfPairs + pair) * kPgDim;
            const float2 ml = pg_ml(m[i], sum);
            const float inv = whole ? pg_inverse(pair_at[pair], sum) : 1.0f;
            float *dst = (whole ? static_cast<float *>(p.out) : p.tile_sum) + to + 4 * tx;
            *reinterpret_cast<float4 *>(dst) = make_float4(o[i][0] * inv, o[i][1] * inv, o[i][2] * inv, o[i][3] * inv);
            *reinterpret_cast<float4 *>(dst + 64) = make_float4(o[i][4] * inv, o[i][5] * inv, o[i][6] * inv, o[i][7] * inv);
            if (!whole && tx == 0) p.tile_ml[static_cast<int64_t>(slot) * kTfPairs + pair] = ml;
        }
    }
    if (!ok && tid == 0) {  // copies in flight land before the CTA ends
        pg_flag(p.status, PLAMO_PAGED_FAILED);
        mbar_wait(&full[0], phase);
        mbar_wait(&full[1], phase);
    }
}

}  // namespace plamo

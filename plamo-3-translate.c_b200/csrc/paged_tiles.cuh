// Attention of a paged batch step on the tensor cores: BF16, 256 (row, head)
// pairs to a tile. Serves the prefix, whose queries are all of the batch's
// short requests' rows at once, and the prompts among the requests.
#pragma once
#include "paged_attention.cuh"

namespace plamo {

// A tile is two halves of 128 pairs (the M of one MMA), each with its own
// scores, weights and sums in tensor memory and four warps of softmax; both
// read the same keys and values, 128 at a time. Tensor memory (512 columns):
// scores of half i at 128 i (FP32; the weights replace them as BF16, 64
// columns), sums at 256 + 128 i. Per 128 keys each half needs 2 x 512 cycles
// of the tensor pipe (128 x 128 x 128 at 4096 multiply-adds a cycle) and
// 1024 cycles of exponentials (16 a cycle): the halves run half a step apart,
// so that one's exponentials cover the other's products.
constexpr int kTlKeys = 128;
constexpr int kTlThreads = 384;                 // copy, MMA, 2 mending, 8 softmax warps
constexpr int kTlUnitBytes = kTlKeys * kPgDim * 2;  // keys or values of a step
constexpr int kTlUnits = 5;
constexpr int kTlQBytes = kTlPairs * kPgDim * 2;
constexpr int kTlSmem = 1024 + kTlQBytes + kTlUnits * kTlUnitBytes;

// Tile t of a prompt (its rows [t * tile_rows, ...)).
__device__ __forceinline__ TileShape prompt_tile(const PagedAttnParams &p, int32_t request, const OwnShape &o, int32_t t) {
    TileShape s{};
    const int32_t first = t * static_cast<int32_t>(p.tile_rows);
    s.request = request;
    s.row0 = o.row0 + first;
    s.rows = min(static_cast<int32_t>(p.tile_rows), o.rows - first);
    s.at0 = static_cast<int32_t>(o.at0) + first;
    const int64_t last = static_cast<int64_t>(s.at0) + s.rows - 1;
    if (last < 0) return s;  // rows before own row 0 see nothing
    const int64_t held = max(s.at0, 0);
    const int64_t lo = p.window ? max(held - p.window + 1, static_cast<int64_t>(0)) : 0;
    const int64_t pre = p.window ? max(p.prefix + held - p.window + 1, static_cast<int64_t>(0)) : 0;
    s.pre1 = static_cast<int32_t>((p.prefix + kTlKeys - 1) / kTlKeys);
    s.pre0 = static_cast<int32_t>(min(pre / kTlKeys, static_cast<int64_t>(s.pre1)));
    s.own_limit = static_cast<int32_t>(min(last + 1, static_cast<int64_t>(o.length)));
    s.own1 = (s.own_limit + kTlKeys - 1) / kTlKeys;
    s.own0 = min(static_cast<int32_t>(lo / kTlKeys), s.own1);
    return s;
}

// ---- the schedule ---------------------------------------------------------------------
// One CTA sorts the requests into short ones (their own rows are the row
// kernel's, their rows join the list that shares the prefix's tiles) and
// prompts (tiles of their own over prefix and own rows), and numbers the key
// steps of all tiles. A step of a tile and KV head is the unit of work: the
// tile kernel's CTAs take equal runs of consecutive ones.
constexpr int kScThreads = 1024;

__global__ void __launch_bounds__(kScThreads) paged_schedule_kernel(const PagedAttnParams p) {
    __shared__ int64_t sums[kScThreads / 32];
    __shared__ int32_t first_at;
    pdl_launch_dependents();
    const int tid = threadIdx.x;
    const int64_t R = p.requests, per = (R + kScThreads - 1) / kScThreads;
    const int64_t r0 = min(R, tid * per), r1 = min(R, r0 + per);
    if (tid == 0) first_at = INT32_MAX;
    __syncthreads();
    int64_t counts = 0, steps = 0;  // short rows | prompts' tiles << 32; the tiles' key steps
    int32_t lowest = INT32_MAX;
    for (int64_t r = r0; r < r1; ++r) {
        const OwnShape s = own_shape(p, r);
        if (!s.rows) continue;
        if (request_is_short(p, s)) {
            counts += s.rows;
            lowest = min(lowest, static_cast<int32_t>(max(s.at0, static_cast<int64_t>(0))));
        } else {
            const int32_t n = static_cast<int32_t>((s.rows + p.tile_rows - 1) / p.tile_rows);
            counts += static_cast<int64_t>(n) << 32;
            for (int32_t t = 0; t < n; ++t) steps += prompt_tile(p, static_cast<int32_t>(r), s, t).steps();
        }
    }
    lowest = __reduce_min_sync(0xffffffffu, lowest);
    if ((tid & 31) == 0) atomicMin(&first_at, lowest);
    int64_t all_counts, all_steps;
    const int64_t before = pg_block_scan<kScThreads>(counts, sums, &all_counts);
    int64_t step_at = pg_block_scan<kScThreads>(steps, sums, &all_steps);
    int64_t short_at = before & 0xffffffff, tile_at = before >> 32;
    int64_t all_short = all_counts & 0xffffffff, all_tiles = all_counts >> 32;
    // Ranges that overlap (starts that decrease) could ask for more than there is.
    if (all_short > p.rows) all_short = p.rows;
    int64_t pre_tiles = 0, pre_steps = 0;
    TileShape pre{};
    if (p.tile_rows && p.prefix) {
        pre_tiles = (all_short + p.tile_rows - 1) / p.tile_rows;
        pre.request = -1;
        pre.pre1 = static_cast<int32_t>((p.prefix + kTlKeys - 1) / kTlKeys);
        if (p.window && first_at != INT32_MAX) {
            const int64_t lo = max(p.prefix + first_at - p.window + 1, static_cast<int64_t>(0));
            pre.pre0 = static_cast<int32_t>(min(lo / kTlKeys, static_cast<int64_t>(pre.pre1)));
        }
        pre_steps = pre.steps();
    }
    const bool fits = !p.tile_rows || (pre_tiles + all_tiles <= p.tile_cap && pre_tiles * pre_steps + all_steps <= INT32_MAX);
    if (!fits) {  // only starts or lengths that no pool holds ask for this
        if (tid == 0) pg_flag(p.status, PLAMO_PAGED_BATCH_ROWS);
        pre_tiles = all_tiles = 0;
    }
    for (int64_t r = r0; r < r1; ++r) {
        const OwnShape s = own_shape(p, r);
        if (!s.rows) continue;
        if (request_is_short(p, s)) {
            for (int32_t i = 0; i < s.rows; ++i, ++short_at)
                if (short_at < all_short)
                    p.short_list[short_at] = make_int4(s.row0 + i, static_cast<int32_t>(max(s.at0 + i, static_cast<int64_t>(-1))),
                                                       static_cast<int32_t>(r), i);
        } else if (fits) {
            const int32_t n = static_cast<int32_t>((s.rows + p.tile_rows - 1) / p.tile_rows);
            for (int32_t t = 0; t < n; ++t, ++tile_at) {
                const TileShape shape = prompt_tile(p, static_cast<int32_t>(r), s, t);
                p.tile_shape[pre_tiles + tile_at] = shape;
                p.tile_unit[pre_tiles + tile_at] = static_cast<uint32_t>(pre_tiles * pre_steps + step_at);
                step_at += shape.steps();
            }
        }
    }
    for (int64_t t = tid; t < pre_tiles; t += kScThreads) {
        pre.row0 = static_cast<int32_t>(t * p.tile_rows);
        pre.rows = static_cast<int32_t>(min(static_cast<int64_t>(p.tile_rows), all_short - pre.row0));
        p.tile_shape[t] = pre;
        p.tile_unit[t] = static_cast<uint32_t>(t * pre_steps);
    }
    if (tid == 0) {
        p.header[kTlShortRows] = static_cast<int32_t>(all_short);
        if (p.tile_rows) {
            const int64_t n = pre_tiles + all_tiles, total = fits ? pre_tiles * pre_steps + all_steps : 0;
            p.tile_unit[n] = static_cast<uint32_t>(total);
            p.header[kTlTiles] = static_cast<int32_t>(n);
            p.header[kTlPreTiles] = static_cast<int32_t>(pre_tiles);
            p.header[kTlCtas] = static_cast<int32_t>(
                min(static_cast<int64_t>(p.tile_grid), (total * p.kh + kTlMinUnits - 1) / kTlMinUnits));
        }
    }
}

// ---- the tile kernel ---------------------------------------------------------------------
// A wait that ends when the phase completes, after about two seconds, or when
// another warp gave up.
__device__ __forceinline__ bool tl_wait(uint64_t *bar, uint32_t parity, volatile int *gave_up) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t start = global_ns();
    while (!mbar_try_wait(bar, parity)) {
        if (*gave_up) return false;
        if (global_ns() - start > 2000000000ull) {
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
    const int64_t key0 = own ? static_cast<int64_t>(s.own0 + step - (s.pre1 - s.pre0)) * kTlKeys
                             : static_cast<int64_t>(s.pre0 + step) * kTlKeys;
    const int64_t limit = own ? s.own_limit : p.prefix, end = min(key0 + kTlKeys, limit);
    bool m = s.request >= 0 && s.at0 < 0;
    if (own) m |= s.at0 + 1 < end || (p.window && s.at0 + s.rows - p.window > key0);
    else if (p.window) m |= s.request < 0 || p.prefix + s.at0 + s.rows - p.window > key0;
    *masked = m;
    return m || key0 + kTlKeys > limit;
}

// The segments of a CTA: runs of steps of one (tile, KV head).
struct TileWalk {
    int64_t unit, end;  // of this CTA
    int32_t tile, head, step, steps;  // current segment: first step and count
    int32_t tile_steps;
};
__device__ __forceinline__ bool walk_next(const PagedAttnParams &p, TileWalk &w) {
    if (w.unit >= w.end) return false;
    for (;;) {
        const int64_t u0 = static_cast<int64_t>(p.tile_unit[w.tile]) * p.kh, u1 = static_cast<int64_t>(p.tile_unit[w.tile + 1]) * p.kh;
        if (w.unit < u1) {
            w.tile_steps = static_cast<int32_t>((u1 - u0) / p.kh);
            const int64_t x = w.unit - u0;
            w.head = static_cast<int32_t>(x / w.tile_steps);
            w.step = static_cast<int32_t>(x % w.tile_steps);
            w.steps = static_cast<int32_t>(min(static_cast<int64_t>(w.tile_steps - w.step), w.end - w.unit));
            return true;
        }
        ++w.tile;
    }
}

__global__ void __launch_bounds__(kTlThreads, 1)
    paged_tile_kernel(const __grid_constant__ CUtensorMap map, const PagedAttnParams p) {
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
            mbar_init(&empty[s], 3);  // the MMAs, and the two mending warps
            mbar_init(&mended[s], 2);
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
    if (warp == 1) {
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
    int64_t all_units = 0;
    if (cta < ctas) {
        all_units = static_cast<int64_t>(p.tile_unit[tiles]) * p.kh;
        w.unit = tile_cta_start(all_units, ctas, cta);
        w.end = tile_cta_start(all_units, ctas, cta + 1);
        // Last tile that starts at or before the first unit.
        w.tile = pg_owner(reinterpret_cast<const int32_t *>(p.tile_unit), static_cast<uint32_t>(tiles),
                          static_cast<int32_t>(w.unit / p.kh));
        while (w.tile > 0 && static_cast<int64_t>(p.tile_unit[w.tile]) * p.kh > w.unit) --w.tile;
    }
    volatile int *quit = &gave_up;
    bool ok = true;

    if (warp == 0) {
        // ---- copies: keys and values of each step alternate in the ring
        uint32_t q = 0;
        for (; ok && walk_next(p, w); w.unit += w.steps) {
            const TileShape s = p.tile_shape[w.tile];
            const int32_t pre_steps = s.pre1 - s.pre0;
            const int32_t *own_table = p.tables + static_cast<uint64_t>(max(s.request, 0)) * p.table_stride;
            const int32_t pre_pages = static_cast<int32_t>((p.prefix + kPgRows - 1) / kPgRows);
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
                if (there && (id < 0 || id >= static_cast<int32_t>(p.pages))) {
                    pg_flag(p.status, PLAMO_PAGED_PAGE);
                    id = static_cast<int32_t>(p.pages);  // past the pool: reads as zeros
                }
                const uint32_t present = __ballot_sync(0xffffffffu, there);
                for (int32_t k = 0; k < 16 && base_step + k < w.steps && ok; ++k) {
                    const int32_t id0 = __shfl_sync(0xffffffffu, id, 2 * k), id1 = __shfl_sync(0xffffffffu, id, 2 * k + 1);
                    const bool two = (present >> (2 * k + 1)) & 1;
                    if (lane == 0) {
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
    } else if (warp == 1) {
        // ---- products: one lane issues
        if (lane == 0) {
            constexpr uint32_t idesc_s = tc_idesc(128, kTlKeys), idesc_o = tc_idesc(128, kPgDim) | kTcIdescMnB;
            // Phases: a bit per half or unit, flipped by each wait.
            uint32_t q = 0, queries = 0, done = 0, weights = 0, mends = 0;
            auto turn = [](uint32_t &phases, uint32_t x) {
                const uint32_t parity = (phases >> x) & 1u;
                phases ^= 1u << x;
                return parity;
            };
            const uint32_t qs = smem_u32(base), us = smem_u32(units_at);
            auto scores = [&](int i, uint32_t unit) {
                const uint32_t a = qs + i * (kTlQBytes / 2), b = us + (unit % kTlUnits) * kTlUnitBytes;
#pragma unroll
                for (int k = 0; k < kPgDim / 16; ++k) {
                    const uint32_t off = (k / 4) * (kTlKeys * 128) + (k % 4) * 32;
                    tc_mma(tmem + 128 * i, smem_desc_sw128(a + off), smem_desc_sw128(b + off), idesc_s, k ? 1u : 0u);
                }
                tc_commit(&s_full[i]);
            };
            for (; ok && walk_next(p, w); w.unit += w.steps) {
                const TileShape s = p.tile_shape[w.tile];
                const int halves = s.rows * static_cast<int32_t>(p.group) > 128 ? 2 : 1;
                ok = tl_wait(&full[q % kTlUnits], (q / kTlUnits) & 1u, quit);
                for (int i = 0; i < halves && ok; ++i) {
                    ok = tl_wait(&q_full[i], turn(queries, i), quit);
                    if (!ok) break;
                    tc_fence_after();
                    scores(i, q);
                }
                if (!ok) break;
                tc_commit(&empty[q % kTlUnits]);
                for (int32_t n = 0; n < w.steps && ok; ++n) {
                    const uint32_t v = q + 2 * n + 1, next = v + 1;
                    ok = tl_wait(&full[v % kTlUnits], (v / kTlUnits) & 1u, quit);
                    bool masked;
                    if (ok && step_is_mended(p, s, w.step + n, &masked))
                        ok = tl_wait(&mended[v % kTlUnits], turn(mends, v % kTlUnits), quit);
                    for (int i = 0; i < halves && ok; ++i) {
                        ok = tl_wait(&p_full[i], turn(weights, i), quit);
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t b = us + (v % kTlUnits) * kTlUnitBytes;
#pragma unroll
                        for (int k = 0; k < kTlKeys / 16; ++k)
                            tc_mma_ts(tmem + 256 + 128 * i, tmem + 128 * i + 8 * k,
                                      smem_desc_mn_sw128(b + k * 16 * 128, kTlKeys * 128), idesc_o, n || k ? 1u : 0u);
                        tc_commit(&pv_done[i]);
                        if (i == halves - 1) tc_commit(&empty[v % kTlUnits]);
                        const uint32_t products = turn(done, i);
                        if (n + 1 < w.steps) {
                            // The next scores replace the weights just read.
                            ok = tl_wait(&full[next % kTlUnits], (next / kTlUnits) & 1u, quit) &&
                                 tl_wait(&pv_done[i], products, quit);
                            if (!ok) break;
                            tc_fence_after();
                            scores(i, next);
                            if (i == halves - 1) tc_commit(&empty[next % kTlUnits]);
                        }
                    }
                }
                q += 2 * w.steps;
            }
        }
    } else if (warp < 4) {
        // ---- mending: values that no weight may touch become zero before the products read them
        uint32_t q = 0;
        const int mt = tid - 64;
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
                        const int64_t key0 = static_cast<int64_t>(own ? s.own0 + step - pre_steps : s.pre0 + step) * kTlKeys;
                        const int64_t limit = own ? s.own_limit : p.prefix;
                        unsigned char *unit = units_at + st * kTlUnitBytes;
                        bool odd = false;
                        for (int c = mt; c < kTlUnitBytes / 16; c += 64) {  // 16-byte pieces, row by row
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
        const int i = (warp - 4) >> 2;  // half
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t scol = tmem + lanes + 128 * i, ocol = tmem + lanes + 256 + 128 * i;
        const int pair = 128 * i + (warp & 3) * 32 + lane;
        uint32_t n_scores = 0, n_sums = 0;
        for (bool begins = true; ok && walk_next(p, w); w.unit += w.steps, begins = false) {
            const TileShape s = p.tile_shape[w.tile];
            const int32_t pairs = s.rows * static_cast<int32_t>(p.group), pre_steps = s.pre1 - s.pre0;
            const bool active = i == 0 || pairs > 128;
            const int32_t local = pair / static_cast<int32_t>(p.group);
            const bool there = pair < pairs;
            int64_t row = 0, at = -1;
            if (there) {
                if (s.request < 0) {
                    const int4 e = p.short_list[s.row0 + local];
                    row = e.x;
                    at = e.y;
                } else {
                    row = s.row0 + local;
                    at = s.at0 + local;
                }
            }
            const uint32_t head = static_cast<uint32_t>(w.head) * p.group + pair % p.group;
            // Queries into shared memory as an MMA operand.
            if (active) {
                unsigned char *dst = base + i * (kTlQBytes / 2) + (pair & 127) * 128;
                const uint4 *src = reinterpret_cast<const uint4 *>(static_cast<const uint16_t *>(p.q) + row * p.q_stride + static_cast<uint64_t>(head) * kPgDim);
                const uint32_t flip = p.scale2 < 0.0f ? 0x80008000u : 0u;
#pragma unroll
                for (int c0 = 0; c0 < 16; c0 += 8) {  // eight loads in flight
                    uint4 v[8];
#pragma unroll
                    for (int c = 0; c < 8; ++c) v[c] = there ? src[c0 + c] : make_uint4(0, 0, 0, 0);
#pragma unroll
                    for (int c = 0; c < 8; ++c)
                        *reinterpret_cast<uint4 *>(dst + (c0 >> 3) * (kTlKeys * 128) + ((c ^ (pair & 7)) << 4)) =
                            make_uint4(v[c].x ^ flip, v[c].y ^ flip, v[c].z ^ flip, v[c].w ^ flip);
                }
                fence_async_shared();
            }
            if (!active) continue;
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[i]);

            const float scale2 = fabsf(p.scale2);
            // Keys this row sees, prefix and own: [lo, hi).
            const int32_t pre_hi = at < 0 ? 0 : static_cast<int32_t>(p.prefix), own_hi = at < 0 ? 0 : static_cast<int32_t>(min(at + 1, static_cast<int64_t>(s.own_limit)));
            const int32_t pre_lo = p.window ? static_cast<int32_t>(min(max(p.prefix + at - p.window + 1, static_cast<int64_t>(0)), p.prefix)) : 0;
            const int32_t own_lo = p.window ? static_cast<int32_t>(max(at - p.window + 1, static_cast<int64_t>(0))) : 0;
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
                // 64 scores at a time: the second half is read first, for the maximum, and again
                // after the first half's weights have gone.
                float x[64];
                const auto load = [&](int half) {
                    uint32_t r0[32], r1[32];
                    tmem_ld32_async(scol + 64 * half, r0);
                    tmem_ld32_async(scol + 64 * half + 32, r1);
                    tmem_wait_ld();
#pragma unroll
                    for (int c = 0; c < 32; ++c) {
                        x[c] = __uint_as_float(r0[c]);
                        x[32 + c] = __uint_as_float(r1[c]);
                    }
                    if (partial) {
#pragma unroll
                        for (int c = 0; c < 64; ++c)
                            if (c + 64 * half < lo || c + 64 * half >= hi) x[c] = -INFINITY;
                    }
                };
                const auto largest = [&]() {
                    float t0 = x[0], t1 = x[1], t2 = x[2], t3 = x[3];
#pragma unroll
                    for (int c = 4; c < 64; c += 4) {
                        t0 = fmaxf(t0, x[c]);
                        t1 = fmaxf(t1, x[c + 1]);
                        t2 = fmaxf(t2, x[c + 2]);
                        t3 = fmaxf(t3, x[c + 3]);
                    }
                    return fmaxf(fmaxf(t0, t1), fmaxf(t2, t3));
                };
                load(1);
                float top = largest();
                load(0);
                top = fmaxf(top, largest()) * scale2;
                // The reference point moves only when passed by 2^8: the weights stay below 2^8,
                // FP32 sums and BF16 weights lose nothing by it, and the sums in tensor memory are
                // rarely touched.
                const bool move = top > m + kLazy;
                if (__any_sync(0xffffffffu, move)) {
                    const float factor = move ? pg_exp2(m - top) : 1.0f;
                    if (move) m = top;
                    l *= factor;
                    if (n) {  // this half's last products are done: the scores came after them
                        for (int c = 0; c < kPgDim; c += 32) {
                            uint32_t r[32];
                            tmem_ld32_async(ocol + c, r);
                            tmem_wait_ld();
#pragma unroll
                            for (int k = 0; k < 32; ++k) r[k] = __float_as_uint(__uint_as_float(r[k]) * factor);
                            tmem_st32(ocol + c, r);
                        }
                    }
                }
                const float shift = m == -INFINITY ? 0.0f : -m;
                float l0 = 0.0f, l1 = 0.0f;
                const auto weigh = [&](int half) {
                    uint32_t r[32];
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        const float a = pg_exp2(fmaf(x[2 * k], scale2, shift)), b = pg_exp2(fmaf(x[2 * k + 1], scale2, shift));
                        l0 += a;
                        l1 += b;
                        r[k] = pg_pack(a, b);
                    }
                    tmem_st32(scol + 32 * half, r);
                };
                weigh(0);
                load(1);
                weigh(1);
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
            const uint64_t slot = w.tile < pre_tiles ? 2ull * p.tile_grid + cta + static_cast<uint64_t>(w.tile) * p.kh + w.head
                                                     : 2ull * cta + (begins ? 0 : 1);
            const bool odd = *reinterpret_cast<volatile int *>(&odd_values);
            const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
            for (int c = 0; c < kPgDim; c += 32) {
                uint32_t r[32];
                tmem_ld32_async(ocol + c, r);
                tmem_wait_ld();
                float o[32];
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = __uint_as_float(r[k]);
                if (odd && there) {
                    // Values that are not finite left the products of steps with masked keys: the
                    // rows that see them get them here (a weight times one of them is itself).
                    for (int32_t n = 0; n < w.steps; ++n) {
                        const int32_t step = w.step + n;
                        bool masked;
                        step_is_mended(p, s, step, &masked);
                        if (!masked) continue;
                        const bool own = step >= pre_steps;
                        const int64_t key0 = static_cast<int64_t>(own ? s.own0 + step - pre_steps : s.pre0 + step) * kTlKeys;
                        const int64_t hi = at < 0 ? 0 : min(key0 + kTlKeys, own ? min(at + 1, static_cast<int64_t>(s.own_limit)) : p.prefix);
                        const int64_t lo = max(key0, p.window ? (own ? at : p.prefix + at) - p.window + 1 : static_cast<int64_t>(0));
                        for (int64_t key = lo; key < hi; ++key) {
                            const int32_t id = own ? p.tables[static_cast<uint64_t>(s.request) * p.table_stride + key / kPgRows]
                                                   : p.prefix_pages[key / kPgRows];
                            if (id < 0 || id >= static_cast<int32_t>(p.pages)) continue;
                            const uint16_t *v = static_cast<const uint16_t *>(p.pool) +
                                                ((static_cast<uint64_t>(id) * 2 + 1) * kPgRows + key % kPgRows) * p.kh * kPgDim +
                                                static_cast<uint64_t>(w.head) * kPgDim + c;
#pragma unroll
                            for (int k = 0; k < 32; ++k) {
                                const float x = bf16_to_f32(v[k]);
                                if (!isfinite(x)) o[k] += x;
                            }
                        }
                    }
                }
                if (whole && there) {
                    uint16_t *dst = static_cast<uint16_t *>(p.out) + row * p.out_stride + static_cast<uint64_t>(head) * kPgDim + c;
#pragma unroll
                    for (int k = 0; k < 32; k += 8)
                        *reinterpret_cast<uint4 *>(dst + k) =
                            make_uint4(pg_pack(o[k] * inv, o[k + 1] * inv), pg_pack(o[k + 2] * inv, o[k + 3] * inv),
                                       pg_pack(o[k + 4] * inv, o[k + 5] * inv), pg_pack(o[k + 6] * inv, o[k + 7] * inv));
                } else if (there) {
                    float *dst = p.tile_sum + (slot * kTlPairs + pair) * kPgDim + c;
#pragma unroll
                    for (int k = 0; k < 32; k += 4)
                        *reinterpret_cast<float4 *>(dst + k) = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
                }
                __syncwarp();
            }
            if (there && !whole) p.tile_ml[slot * kTlPairs + pair] = make_float2(m, l);
            tc_fence_before();
        }
    }
    if (!ok && lane == 0) pg_flag(p.status, PLAMO_PAGED_FAILED);
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

}  // namespace plamo

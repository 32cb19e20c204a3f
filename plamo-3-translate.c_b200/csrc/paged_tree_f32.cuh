// Attention of draft trees on the tensor cores: FP32, tiles of up to 128 (row, head)
// pairs by steps of 64 keys, a page.
#pragma once
#include "paged_tree_tiles.cuh"

namespace plamo {

// Queries, keys, weights and values each enter as three BF16 terms x1 + x2 + x3 (24
// bits), and of the nine products of two those six are made whose size is above 2^-24
// of the whole: (3,1) (1,3) (2,2) (2,1) (1,2) (1,1), the small ones first. Tensor cores
// cut what they add up, by 1e-5 of the sum over some thousand keys; so a step's value
// products start from zero and are added to FP32 registers, and nothing is cut by more
// than a few products of 2^-24. 128 pairs by 64 keys are some 3,100 cycles of the tensor pipe;
// as many multiply-adds of the CUDA cores are 16,384.
//  - Sixteen warps have the softmax and the sums. Warp w has the rows of tensor-memory lanes
//    32 (w % 4) up; its quarter w / 4 has 16 of a step's keys and 32 of the dimensions. In
//    each step a thread makes its keys' weights and adds its dimensions' sums of the step
//    before to its registers. Eight more turn keys and values into terms in shared memory,
//    as far ahead as there is room: 5,700 cycles a step, the 12 trees of 24 rows in a window 97 us
//    (9,000 and 148 where the sixteen did that, too; four warps for it 178).
//  - Tensor memory (512 columns): the queries' terms 3 x 64, a step's sums 128, and two
//    places by turns of 96 for a step's scores (64), then its weights' terms (3 x 32).
//  - Shared memory: two steps' terms of keys and of values, 4 x 48 KB.
// Values that are not finite leave the products, and rows that see them get them at the
// end of a segment; a key that has such a number gets its scores one by one.
constexpr int kTqPairs = 128, kTqKeys = 64, kTqWarps = 16, kTqTurning = 8, kTqThreads = 32 * (kTqWarps + kTqTurning + 2);
constexpr int kTqWalk = 24, kTqProducts = 25;  // warps; 0-15 softmax, 16-23 turn keys and values into terms
constexpr int kTqTerm = kTqKeys * kPgDim * 2, kTqBlock = kTqKeys * 128;  // bytes: a term of keys or values, its block of 64 dimensions
constexpr int kTqSmem = 1024 + 4 * 3 * kTqTerm;
constexpr uint32_t kTqQueries = 0, kTqSums = 192, kTqPlaces = 320, kTqPlace = 96;  // columns

// A pair of finite numbers as terms: the upper halves, what is left rounded, and what is left then rounded.
__device__ __forceinline__ void tq_split(uint32_t a, uint32_t b, uint32_t (&t)[3]) {
    const uint64_t less = pair_of(-1.0f, -1.0f);
    t[0] = __byte_perm(a, b, 0x7632);
    uint64_t left = fma_pair(pair_of(a & 0xffff0000u, b & 0xffff0000u), less, pair_of(a, b));
    t[1] = pg_pack(low_of(left), high_of(left));
    left = fma_pair(pair_of(t[1] << 16, t[1] & 0xffff0000u), less, left);
    t[2] = pg_pack(low_of(left), high_of(left));
}
__device__ __forceinline__ void tq_split(float a, float b, uint32_t (&t)[3]) { tq_split(__float_as_uint(a), __float_as_uint(b), t); }
__device__ __forceinline__ float tq_or_zero(float x) { return isfinite(x) ? x : 0.0f; }

__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
__device__ __forceinline__ void tmem_ld16_async(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
// A barrier of the sixteen warps that says whether any thread asks.
__device__ __forceinline__ bool tq_any(bool ask) {
    uint32_t any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "barrier.cta.red.or.pred q, 1, %2, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(any)
        : "r"(static_cast<uint32_t>(ask)), "n"(32 * kTqWarps)
        : "memory");
    return any != 0;
}

// Values that are not finite, for a row that sees them (a weight times one of them is itself): dimensions c to c + 31.
__device__ __noinline__ void tq_add_odd_values(const PagedAttnParams &p, const TreeSegment &t, int32_t row, int32_t held, int32_t added,
                                               const TreeSees &sees, int32_t from, int c, float (&o)[32]) {
    const TileShape s = p.tile_shape[t.tile];
#pragma unroll 1
    for (int32_t n = 0; n < t.steps; ++n) {
        const int32_t step = t.step + n;
        const bool own = step >= t.pre_steps;
        const int32_t key0 = (own ? t.own0 + step - t.pre_steps : t.pre0 + step) * kTqKeys, hi = min(key0 + kTqKeys, own ? s.own_limit : p.prefix);
        const int32_t id = own ? p.tables[static_cast<uint64_t>(s.request) * p.table_stride + key0 / kPgRows] : p.prefix_pages[key0 / kPgRows];
        if (id < 0 || id >= p.pages) continue;
#pragma unroll 1
        for (int32_t key = max(key0, own ? sees.lo : sees.pre); key < hi; ++key) {
            if (own && key >= held && !(tree_bits(p, row, added, from, key - held) & 1u)) continue;
            const float *v = static_cast<const float *>(p.pool) +
                             (((static_cast<uint64_t>(id) * 2 + 1) * kPgRows + key % kPgRows) * p.kh + t.head) * static_cast<uint64_t>(kPgDim) + c;
#pragma unroll 1
            for (int k = 0; k < 32; ++k)
                if (!isfinite(v[k])) o[k] += v[k];
        }
    }
}

__global__ void __launch_bounds__(kTqThreads, 1) paged_tree_f32_kernel(const __grid_constant__ PagedAttnParams p) {
    extern __shared__ __align__(128) unsigned char tq_smem[];
    __shared__ __align__(8) uint64_t seg_full[kTsSegments], seg_empty[kTsSegments];
    __shared__ __align__(8) uint64_t q_ready, k_ready[2], k_free[2], v_ready[2], v_free[2], s_full[2], p_ready[2], o_full, o_free;
    __shared__ TreeSegment segments[kTsSegments];
    __shared__ float tops[4][kTqPairs];
    __shared__ __align__(8) unsigned char odd_keys[4][kTqKeys / 8];  // of step s, at s % 4: keys with a number that is not finite
    __shared__ uint32_t tmem_base;
    __shared__ int gave_up, odd_values;
    unsigned char *base = reinterpret_cast<unsigned char *>(
        (reinterpret_cast<uintptr_t>(tq_smem) + 1023) & ~static_cast<uintptr_t>(1023));
    unsigned char *const keys_at = base, *const values_at = base + 2 * 3 * kTqTerm;  // two steps' each
    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    if (tid == 0) {
        for (int s = 0; s < kTsSegments; ++s) {
            mbar_init(&seg_full[s], 1);
            mbar_init(&seg_empty[s], kTqWarps + kTqTurning + 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_ready[i], kTqTurning);
            mbar_init(&v_ready[i], kTqTurning);
            mbar_init(&p_ready[i], kTqWarps);
            mbar_init(&k_free[i], 1);
            mbar_init(&v_free[i], 1);
            mbar_init(&s_full[i], 1);
        }
        mbar_init(&q_ready, kTqWarps);
        mbar_init(&o_full, 1);
        mbar_init(&o_free, kTqWarps);
        gave_up = odd_values = 0;
        fence_barrier_init();
    }
    if (warp == kTqProducts) {
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
    volatile int *quit = &gave_up;
    bool ok = true;
    const auto wait = [&](uint64_t *bar, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_try_wait(bar, parity)) || __all_sync(0xffffffffu, ts_wait(bar, parity, quit));
    };

    if (warp == kTqWalk) {
        // ---- the work's segments
        pdl_wait();
        const int32_t ctas = p.header[kTlCtas], cta = static_cast<int32_t>(blockIdx.x);
        const int32_t first_row = p.header[kTlFirst];
        TileWalk w{};
        if (cta < ctas) {
            const Runs runs = tile_runs(p);
            w.unit = runs.start(cta);
            w.end = runs.start(cta + 1);
            w.tile = pg_owner(reinterpret_cast<const int32_t *>(p.tile_unit), static_cast<uint32_t>(p.header[kTlTiles]), p.by_kh.div(w.unit));
        }
        uint32_t seg = 0;
        for (bool more = true; more && ok; ++seg) {
            more = tree_walk_next(p, w);
            TileShape s{};
            if (more) s = p.tile_shape[w.tile];
            const uint32_t e = seg % kTsSegments;
            ok = seg < kTsSegments || wait(&seg_empty[e], (seg / kTsSegments - 1) & 1u);
            if (ok && lane == 0) {
                TreeSegment t{};
                if (more)
                    t = TreeSegment{w.steps, 0, w.tile, w.head, w.step, w.tile_steps, s.request < 0 ? first_row + s.row0 : s.row0, s.rows * p.group,
                                    s.request < 0 ? -1 : s.at0, s.added, s.pre0, s.pre1 - s.pre0, s.own0, s.request, s.own_limit, 0};
                segments[e] = t;
                mbar_arrive(&seg_full[e]);
            }
            __syncwarp();
        }
    } else if (warp == kTqProducts) {
        // ---- products
        constexpr uint32_t idesc_s = tc_idesc(128, kTqKeys), idesc_o = tc_idesc(128, kPgDim) | kTcIdescMnB;
        constexpr int kOf[6][2] = {{2, 0}, {0, 2}, {1, 1}, {1, 0}, {0, 1}, {0, 0}};  // terms of the first and second operand
        const bool leader = elect_one();
        const uint64_t k_desc = smem_desc_sw128(smem_u32(keys_at)), v_desc = smem_desc_mn_sw128(smem_u32(values_at), kTqBlock);
        uint32_t c = 0;  // steps before the segment's
        for (uint32_t seg = 0; ok; ++seg) {
            ok = wait(&seg_full[seg % kTsSegments], (seg / kTsSegments) & 1u);
            if (!ok) break;
            const int32_t steps = __shfl_sync(0xffffffffu, segments[seg % kTsSegments].steps, 0);
            __syncwarp();
            if (leader) mbar_arrive(&seg_empty[seg % kTsSegments]);
            if (!steps) break;
            // Of step s: its place is free when the value products of step s - 2 are done. (Of a segment's
            // first step they are, and those of s - 1: the queries were put there behind them.)
            const auto scores = [&](uint32_t s, bool first) {
                const uint32_t i = s & 1;
                if (!wait(&k_ready[i], (s >> 1) & 1u) || (!first && s >= 2 && !wait(&o_full, (s - 2) & 1u))) return false;
                tc_fence_after();
                if (leader) {
                    const uint32_t d = tmem + kTqPlaces + i * kTqPlace;
                    const uint64_t b = k_desc + i * (3 * kTqTerm / 16);
#pragma unroll
                    for (int y = 0; y < 6; ++y)
#pragma unroll
                        for (int k = 0; k < kPgDim / 16; ++k)
                            tc_mma_ts(d, tmem + kTqQueries + 64 * kOf[y][0] + 8 * k, b + (kOf[y][1] * kTqTerm + (k / 4) * kTqBlock + (k % 4) * 32) / 16,
                                      idesc_s, y || k ? 1u : 0u);
                    tc_commit(&s_full[i]);
                    tc_commit(&k_free[i]);
                }
                __syncwarp();
                return true;
            };
            ok = wait(&q_ready, seg & 1u) && scores(c, true);
#pragma unroll 1
            for (int32_t n = 0; n < steps && ok; ++n) {
                const uint32_t s = c + n, i = s & 1;
                if (n + 1 < steps) ok = scores(s + 1, false);
                ok = ok && wait(&p_ready[i], (s >> 1) & 1u) && wait(&v_ready[i], (s >> 1) & 1u) && (!s || wait(&o_free, (s - 1) & 1u));
                if (!ok) break;
                tc_fence_after();
                if (leader) {
                    const uint32_t a = tmem + kTqPlaces + i * kTqPlace;
                    const uint64_t b = v_desc + i * (3 * kTqTerm / 16);
#pragma unroll
                    for (int y = 0; y < 6; ++y)
#pragma unroll
                        for (int k = 0; k < kTqKeys / 16; ++k)
                            tc_mma_ts(tmem + kTqSums, a + 32 * kOf[y][0] + 8 * k, b + (kOf[y][1] * kTqTerm + k * 16 * 128) / 16, idesc_o, y || k ? 1u : 0u);
                    tc_commit(&o_full);
                    tc_commit(&v_free[i]);
                }
                __syncwarp();
            }
            c += steps;
        }
    } else if (warp >= kTqWarps && warp < kTqWalk) {
        // ---- keys and values into terms: eight rows of a step to a warp, 16 bytes of each to a lane; four
        // are turned while four are on their way
        pdl_wait();
        const int turning = warp - kTqWarps;
        unsigned char *const put_at = base + (lane >> 4) * kTqBlock + 8 * turning * 128 + (lane & 1) * 8;
        const uint64_t row_size = static_cast<uint64_t>(p.kh) * kPgDim;
        uint32_t c = 0;  // steps before the segment's
        for (uint32_t seg = 0; ok; ++seg) {
            ok = wait(&seg_full[seg % kTsSegments], (seg / kTsSegments) & 1u);
            if (!ok) break;
            const TreeSegment t = segments[seg % kTsSegments];
            __syncwarp();
            if (lane == 0) mbar_arrive(&seg_empty[seg % kTsSegments]);
            if (!t.steps) break;
            const auto page_id = [&](int32_t n) {
                const int32_t step = t.step + n;
                const bool own = step >= t.pre_steps;
                const int32_t *table = own ? p.tables + static_cast<uint64_t>(max(t.request, 0)) * p.table_stride + t.own0 - t.pre_steps : p.prefix_pages + t.pre0;
                return n < t.steps ? table[step] : -1;
            };
            // The first of this warp's rows of page `id`; and how many of them step n has.
            const auto rows_at = [&](int32_t id) {
                const bool good = id >= 0 && id < p.pages;
                return static_cast<const float *>(p.pool) + (static_cast<uint64_t>(good ? id : 0) * 2 * kPgRows + 8 * turning) * row_size + t.head * kPgDim;
            };
            const auto rows_of = [&](int32_t n, int32_t id) {
                const int32_t step = t.step + n;
                const bool own = step >= t.pre_steps;
                const int32_t left = own ? t.own_limit - (t.own0 + step - t.pre_steps) * kTqKeys : p.prefix - (t.pre0 + step) * kTqKeys;
                return id >= 0 && id < p.pages ? left - 8 * turning : 0;
            };
            float4 raw[2][4];
            const auto load = [&](int i, const float *from, int32_t rows) {
#pragma unroll
                for (int y = 0; y < 4; ++y) raw[i][y] = 4 * i + y < rows ? ld4(from + (4 * i + y) * row_size + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
            };
            // A line of 128 bytes to a lane: they are in L2 when their turn comes.
            const auto ahead = [&](const float *from, int32_t rows) {
                if ((lane >> 2) < rows) asm volatile("prefetch.global.L2 [%0];" ::"l"(from + (lane >> 2) * row_size + 32 * (lane & 3)));
            };
            const auto put = [&](int i, uint32_t to, uint32_t s) {  // says which rows had a number that is not finite
                uint64_t z = pair_of(0.0f, 0.0f);  // no number where one of them is none
                uint32_t odd = 0;
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    z = fma_pair(pair_of(raw[i][y].x, raw[i][y].y), pair_of(0.0f, 0.0f), z);
                    z = fma_pair(pair_of(raw[i][y].z, raw[i][y].w), pair_of(0.0f, 0.0f), z);
                }
                if (__any_sync(0xffffffffu, low_of(z) + high_of(z) != 0.0f)) {
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        const float4 v = raw[i][y];
                        raw[i][y] = make_float4(tq_or_zero(v.x), tq_or_zero(v.y), tq_or_zero(v.z), tq_or_zero(v.w));
                        if (__any_sync(0xffffffffu, !(isfinite(v.x) && isfinite(v.y) && isfinite(v.z) && isfinite(v.w)))) odd |= 1u << y;
                    }
                }
                unsigned char *const at0 = put_at + to + (s & 1) * 3 * kTqTerm + 4 * i * 128;
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    uint32_t a[3], b[3];
                    tq_split(raw[i][y].x, raw[i][y].y, a);
                    tq_split(raw[i][y].z, raw[i][y].w, b);
                    unsigned char *const at = at0 + y * 128 + ((((lane & 15) >> 1) ^ (4 * i + y)) << 4);
#pragma unroll
                    for (int x = 0; x < 3; ++x) *reinterpret_cast<uint2 *>(at + x * kTqTerm) = make_uint2(a[x], b[x]);
                }
                return odd;
            };
            const auto ready = [&](uint64_t *bar) {
                fence_async_shared();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar);
            };
            int32_t id = page_id(0), id_next = page_id(1);
            const float *keys = rows_at(id);
            load(0, keys, rows_of(0, id));
            load(1, keys, rows_of(0, id));
            ahead(keys + kPgRows * row_size, rows_of(0, id));
#pragma unroll 1
            for (int32_t n = 0; n < t.steps && ok; ++n) {
                const uint32_t s = c + n;
                const int32_t rows = rows_of(n, id), rows_next = n + 1 < t.steps ? rows_of(n + 1, id_next) : 0, id_after = page_id(n + 2);
                const float *const values = keys + kPgRows * row_size, *const keys_next = rows_at(id_next);
                if ((id < 0 || id >= p.pages) && turning == 0 && lane == 0) pg_flag(p.status, PLAMO_PAGED_PAGE);
                ahead(keys_next, rows_next);
                ahead(keys_next + kPgRows * row_size, rows_next);
                ok = s < 2 || wait(&k_free[s & 1], ((s >> 1) - 1) & 1u);
                if (!ok) break;
                uint32_t odd = 0;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    odd |= put(i, 0, s) << 4 * i;
                    load(i, values, rows);
                }
                if (lane == 0) odd_keys[s & 3][turning] = static_cast<unsigned char>(odd);
                ready(&k_ready[s & 1]);
                ok = s < 2 || wait(&v_free[s & 1], ((s >> 1) - 1) & 1u);
                if (!ok) break;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (put(i, 2 * 3 * kTqTerm, s) && lane == 0) odd_values = 1;
                    load(i, keys_next, rows_next);
                }
                ready(&v_ready[s & 1]);
                id = id_next;
                id_next = id_after;
                keys = keys_next;
            }
            c += t.steps;
        }
    } else if (warp < kTqWarps) {
        // ---- softmax, sums
        pdl_wait();
        const int quarter = warp >> 2, pair = (warp & 3) * 32 + lane;
        const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const int32_t cta = static_cast<int32_t>(blockIdx.x), pre_tiles = p.header[kTlPreTiles];
        const float scale2 = fabsf(p.scale2);
        const uint32_t flip = p.scale2 < 0.0f ? 0x80000000u : 0u;
        uint32_t c = 0;  // steps before the segment's
        // (The sixteen warps meet at barriers, so none leaves alone: a wait that runs out is asked for.)
        for (uint32_t seg = 0;; ++seg) {
            ok = wait(&seg_full[seg % kTsSegments], (seg / kTsSegments) & 1u);
            if (tq_any(!ok)) {
                ok = false;
                break;
            }
            const TreeSegment t = segments[seg % kTsSegments];
            __syncwarp();
            if (lane == 0) mbar_arrive(&seg_empty[seg % kTsSegments]);
            if (!t.steps) break;
            const int32_t request = t.request;
            const bool there = pair < t.pairs;
            const int32_t local = p.by_group.div(pair), row = t.row0 + local, head = t.head * p.group + pair - local * p.group;
            const float *const query = static_cast<const float *>(p.q) + static_cast<int64_t>(there ? row : t.row0) * static_cast<int64_t>(p.q_stride) + (there ? head : 0) * kPgDim;
            // 32 dimensions of this row's query into tensor memory; the last segment's products are done with it.
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t term[3][8];
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const float4 v = there ? ld4(query + 32 * quarter + 16 * half + 4 * y) : make_float4(0.f, 0.f, 0.f, 0.f);
                    uint32_t a[3], b[3];
                    tq_split(v.x, v.y, a);
                    tq_split(v.z, v.w, b);
#pragma unroll
                    for (int x = 0; x < 3; ++x) term[x][2 * y] = a[x], term[x][2 * y + 1] = b[x];
                }
#pragma unroll
                for (int x = 0; x < 3; ++x) tmem_st8(lanes + kTqQueries + 64 * x + 16 * quarter + 8 * half, term[x]);
            }
            tmem_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_ready);
            int32_t held = t.held, added = t.added, from = 0;  // `from`: bits of the mask below it are outside the window
            TreeSees sees{0, 0, 0};
            if (p.window && there) {
                if (held < 0) {  // rows of many requests
                    const int4 e = p.short_list[row - p.header[kTlFirst]];
                    held = max(e.y, 0);
                    added = listed_added(p, e);
                }
                sees = tree_sees(p, tree_skip(p, row, held, added), held);
                from = tree_first(p, row, added, sees.drop);
            }
            float o[32], m = -INFINITY, l = 0.0f, later = 1.0f;  // `later`: what the step's sums on their way are multiplied with
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = 0.0f;
            const auto fold = [&](uint32_t s) {  // adds step s's sums
                if (!wait(&o_full, s & 1u)) return false;
                tc_fence_after();
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    uint32_t x[16];
                    tmem_ld16_async(lanes + kTqSums + 32 * quarter + 16 * half, x);
                    tmem_wait_ld();
#pragma unroll
                    for (int k = 0; k < 16; ++k) o[16 * half + k] = fmaf(__uint_as_float(x[k]), later, o[16 * half + k]);
                }
                later = 1.0f;
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&o_free);
                return true;
            };
#pragma unroll 1
            for (int32_t n = 0; n < t.steps; ++n) {
                const uint32_t s = c + n;
                const int32_t step = t.step + n;
                const bool own = step >= t.pre_steps;
                // ---- this thread's 16 keys of the step: which of them the row sees
                const int32_t key0 = (own ? t.own0 + step - t.pre_steps : t.pre0 + step) * kTqKeys + 16 * quarter;
                const int32_t hi = min(max((own ? held : p.prefix) - key0, 0), 16);
                const int32_t lo = min(max((own ? sees.lo : sees.pre) - key0, 0), 16);
                uint32_t see = 0;
                if (there) {
                    see = tl_bits(lo, hi);
                    if (own && key0 + 16 > held) see |= tree_bits(p, row, added, from, key0 - held);
                }
                ok = ok && wait(&s_full[s & 1], (s >> 1) & 1u);
                const uint32_t at = lanes + kTqPlaces + (s & 1) * kTqPlace;
                uint32_t x[16];
                float top = -INFINITY;
#pragma unroll
                for (int k = 0; k < 16; ++k) x[k] = 0xff800000u;  // -inf
                if (ok) {
                    tc_fence_after();
                    tmem_ld16_async(at + 16 * quarter, x);
                    tmem_wait_ld();
                    if (flip) {
#pragma unroll
                        for (int k = 0; k < 16; ++k) x[k] ^= flip;
                    }
                    const uint32_t odd = *reinterpret_cast<const uint16_t *>(&odd_keys[s & 3][2 * quarter]) & see;
                    if (__any_sync(0xffffffffu, see != 0xffffu || odd)) {
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            if (!((see >> k) & 1u)) x[k] = 0xff800000u;
                        if (odd) {
                            // Keys with a number that is not finite: their scores one by one.
                            const int32_t page = key0 / kTqKeys;
                            const int32_t id = own ? p.tables[static_cast<uint64_t>(max(request, 0)) * p.table_stride + page] : p.prefix_pages[page];
#pragma unroll
                            for (int k = 0; k < 16; ++k) {
                                if (!((odd >> k) & 1u)) continue;
                                const float *key = static_cast<const float *>(p.pool) +
                                                   ((static_cast<uint64_t>(id) * 2 * kPgRows + 16 * quarter + k) * p.kh + t.head) * static_cast<uint64_t>(kPgDim);
                                float dot = 0.0f;
#pragma unroll 1
                                for (int d = 0; d < kPgDim; ++d) dot = fmaf(query[d], key[d], dot);
                                x[k] = __float_as_uint(dot) ^ flip;
                            }
                        }
                    }
                    float y[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int k = 0; k < 16; k += 4)
#pragma unroll
                        for (int z = 0; z < 2; ++z) y[z] = fmaxf(fmaxf(y[z], __uint_as_float(x[k + 2 * z])), __uint_as_float(x[k + 2 * z + 1]));
                    top = fmaxf(y[0], y[1]) * scale2;
                    tc_fence_before();
                }
                // The reference point of a row moves when some key passes it by 2^8, for all four quarters
                // alike. The barrier also says that all have read the scores, which the weights replace.
                if (tq_any(top > m + kLazy || !ok)) {
                    tops[quarter][pair] = top;
                    if (tq_any(!ok)) {  // (all leave together)
                        ok = false;
                        break;
                    }
                    const float all = fmaxf(fmaxf(tops[0][pair], tops[1][pair]), fmaxf(tops[2][pair], tops[3][pair]));
                    if (all > m + kLazy) {
                        const float factor = pg_exp2(m - all);
                        m = all;
                        l *= factor;
                        if (n) later = factor;
#pragma unroll
                        for (int k = 0; k < 32; ++k) o[k] *= factor;
                    }
                    tq_any(false);  // before the next step's
                }
                tc_fence_after();
                {
                    const float shift = m == -INFINITY ? 0.0f : -m;
                    uint64_t sums = pair_of(0.0f, 0.0f);
                    uint32_t term[3][8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const uint64_t y = fma_pair(pair_of(x[2 * k], x[2 * k + 1]), pair_of(scale2, scale2), pair_of(shift, shift));
                        const uint32_t a = __float_as_uint(pg_exp2(low_of(y))), b = __float_as_uint(pg_exp2(high_of(y)));
                        sums = add_pair(sums, pair_of(a, b));
                        uint32_t w[3];
                        tq_split(a, b, w);
#pragma unroll
                        for (int z = 0; z < 3; ++z) term[z][k] = w[z];
                    }
                    l += low_of(sums) + high_of(sums);
#pragma unroll
                    for (int y = 0; y < 3; ++y) tmem_st8(at + 32 * y + 8 * quarter, term[y]);
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&p_ready[s & 1]);
                }
                if (n) ok = ok && fold(s - 1);
            }
            ok = ok && fold(c + t.steps - 1);
            c += t.steps;
            // ---- the segment's sums
            tops[quarter][pair] = l;
            if (tq_any(!ok)) {
                ok = false;
                break;
            }
            l = (tops[0][pair] + tops[1][pair]) + (tops[2][pair] + tops[3][pair]);
            if (*reinterpret_cast<volatile int *>(&odd_values) && there) {
                float with[32];
#pragma unroll
                for (int k = 0; k < 32; ++k) with[k] = o[k];
                tq_add_odd_values(p, t, row, held, added, sees, from, 32 * quarter, with);
#pragma unroll
                for (int k = 0; k < 32; ++k) o[k] = with[k];
            }
            const bool whole = t.steps == t.tile_steps && t.tile >= pre_tiles && !p.share;
            const int64_t place = static_cast<int64_t>(2 * p.tile_grid + cta + t.tile * p.kh + t.head) * kTqPairs + pair;
            if (whole) {
                if (there) {
                    const float inv = tree_inverse(p, row, held, added, l);
                    float *to = static_cast<float *>(p.out) + row * p.out_stride + head * kPgDim + 32 * quarter;
#pragma unroll
                    for (int k = 0; k < 32; k += 4) *reinterpret_cast<float4 *>(to + k) = make_float4(o[k] * inv, o[k + 1] * inv, o[k + 2] * inv, o[k + 3] * inv);
                }
            } else {
                // Four lanes write 128 bytes of one row at a time: a line is written once.
                uint32_t v[32];
#pragma unroll
                for (int k = 0; k < 32; ++k) v[k] = __float_as_uint(o[k]);
                transpose_blocks(v);
                float *to = p.tile_sum + (place - (lane & 3)) * kPgDim + 32 * quarter + 8 * (lane & 3);
#pragma unroll
                for (int y = 0; y < 4; ++y)
                    if (pair - (lane & 3) + y < t.pairs) store_256(to + y * kPgDim, v + 8 * y);
                if (there && quarter == 0) p.tile_ml[place] = pg_ml(m, l);
            }
            tq_any(false);  // before the next segment's tops
        }
    }
    if (!ok && lane == 0) pg_flag(p.status, PLAMO_PAGED_FAILED);
    tc_fence_before();
    __syncthreads();
    if (warp == kTqProducts) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

}  // namespace plamo

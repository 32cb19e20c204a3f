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

// x / d for x < 2^31 by a multiplication: the kernels run for microseconds, in
// which the code of divisions would take longer to fetch than to execute.
struct FastDiv {
    uint32_t d, mul, shift;
    __host__ static FastDiv of(uint32_t d) {
        FastDiv f{d, 0, 0};
        if (d > 1) {
            uint32_t bits = 0;
            while ((1ull << bits) < d) ++bits;
            f.shift = bits - 1;
            f.mul = static_cast<uint32_t>(((1ull << (31 + bits)) + d - 1) / d);
        }
        return f;
    }
    __device__ __forceinline__ int32_t div(int32_t x) const {
        return d == 1 ? x : static_cast<int32_t>(__umulhi(static_cast<uint32_t>(x), mul) >> shift);
    }
};

// All lengths and positions are below 2^31, requests and (row, head) pairs at
// most 2^30 (checked by the host).
struct PagedAttnParams {
    const void *q;
    void *out;
    const int32_t *starts, *lengths, *tables, *prefix_pages;
    uint64_t q_stride, out_stride, table_stride;
    uint32_t *status;
    int32_t rows, requests, pages, qh, kh, group;
    FastDiv by_group, by_kh;
    int32_t prefix, window;  // window: rows seen, 0 for all
    int32_t max_length;      // own rows a page table holds
    float scale2;            // scale * log2(e)
    // The row kernel's partial results, unnormalised: [slot][kRtPairs][128] sums and [slot][kRtPairs] {m, l}.
    float *row_sum;
    float2 *row_ml;
    int4 *row_record;      // [requests + 1] where a request's units begin, its pages, its first strip, tiles; last: the prefix
    int32_t row_slots;     // capacity
    int32_t workers;       // CTAs that take work
    int32_t prefix_tiles;  // row tiles over the prefix, 0: the tile kernel's
    // The schedule (paged_tiles.cuh).
    int32_t *header;   // [kTlHeader]
    int4 *short_list;  // [rows] {batch row, own row, request, row of it} of the short requests' rows
    // The tile kernel's share; tile_rows 0: it has none.
    const void *pool;
    int32_t tile_rows;   // batch rows to a tile
    int32_t tile_pairs;  // pairs to a tile: 256 in BF16, 64 in FP32
    int32_t tile_keys;   // keys to a step: 128, 64
    FastDiv by_tile_rows;
    int32_t tile_grid, tile_cap;
    struct TileShape *tile_shape;  // [tile_cap]
    uint32_t *tile_unit;           // [tile_cap + 1] key steps before each tile
    float *tile_sum;               // [slot][tile_pairs][128], [slot][tile_pairs] {m, l}
    float2 *tile_ml;
};
enum { kTlShortRows, kTlTiles, kTlPreTiles, kTlCtas, kTlRun, kTlLonger, kTlFirst, kTlTaken, kRtRun, kRtLonger, kTlHeader };
// Requests of up to so many pairs keep their own rows in the row kernel and share
// the prefix's tiles. Over 4 to 64 requests of 300 and 2,000 rows: with a bound of 16,
// requests of 17 to 32 pairs take 1.41 times as long behind 4,096 rows (BF16; FP32
// 1.60), 0.96 (1.11) behind 455; with one of 64, those of 33 to 64 pairs 0.97
// (0.97) behind 4,096, 1.28 (1.15) behind 455, 1.19 (1.05) behind none.
constexpr int kTlShortPairs = 32;
constexpr int kTlMinUnits = 2;     // least key steps worth a CTA
// Units of the row kernel, strips times pages, that the tile kernel is worth: prompts', a prefix's.
constexpr uint64_t kTlPromptUnits = 2000, kTlPrefixUnits = 3000;

// The row kernel works on slabs of 16 keys, the M of one mma.sync, against
// tiles of 8 (row, head-in-group) pairs, its N. Tiles of 16 for more pairs than
// that to a request read its keys half as often, in twice the code, which a CTA's
// few slabs do not pay for: 61 requests of 1,000 rows and 16 heads 47 us against
// 23, 8 of 450 rows and two rows of eight heads 28 against 14; only one request
// of four rows over 131,072, 32 pairs whose keys outlast the L2 cache, gained
// (135 against 177).
constexpr int kRtKeys = 16;
constexpr int kRtPairs = 8;
constexpr int kRtWarps = 6;                      // computing warps, a slab each in turn
constexpr int kRtThreads = 32 * (kRtWarps + 1);  // and the copying warp
constexpr int kRtMinPages = 1;                   // least pages worth a CTA (8 requests of 450 FP32 rows: 18.5 us; 22.6 with 2)
constexpr int kRtBatch = 8;                      // items laid out at a time
template <bool F32>
__host__ __device__ constexpr int rt_slab_bytes() {  // keys, then values
    return 2 * kRtKeys * kPgDim * (F32 ? 4 : 2);
}
// A ring of slabs and, behind it, the queries or the warps' joined sums; two
// CTAs to an SM. The ring's places are a multiple of the warps, so that within
// an item a place serves one warp, which has seen each of its phases before the
// next (and between items all warps meet): a wait by parity could not tell a
// phase from the one before the last.
constexpr int kRtRing = 98304;
constexpr int kRtSmem = 1024 + kRtRing + 16 * kPgDim * 4;

// A request's new rows and visible own keys.
struct OwnShape {
    int32_t row0, rows;  // batch rows
    int32_t at0;         // own row of the first one (negative: not held)
    int32_t length;      // own rows held
    int32_t page0, pages;
    int32_t tiles;
};
__device__ __forceinline__ OwnShape own_shape(const PagedAttnParams &p, int32_t r) {
    OwnShape s;
    s.row0 = min(max(p.starts[r], 0), p.rows);
    s.rows = min(max(p.starts[r + 1], s.row0), p.rows) - s.row0;
    s.length = min(max(p.lengths[r], 0), p.max_length);
    s.at0 = s.length - s.rows;
    const int32_t first = p.window ? max(max(s.at0, 0) - p.window + 1, 0) : 0;
    s.page0 = first / kPgRows;
    s.pages = s.rows ? max((s.length + kPgRows - 1) / kPgRows - s.page0, 0) : 0;
    s.tiles = (s.rows * p.group + kRtPairs - 1) / kRtPairs;
    return s;
}
// Short requests' own rows go through the row kernel, eight pairs at a time;
// the others are the tile kernel's, where there is one.
__device__ __forceinline__ bool request_is_short(const PagedAttnParams &p, const OwnShape &s) {
    return !p.tile_rows || s.rows * p.group <= kTlShortPairs;
}
__device__ __forceinline__ OwnShape short_shape(const PagedAttnParams &p, int32_t r) {
    OwnShape s = own_shape(p, r);
    if (!request_is_short(p, s)) s.tiles = s.pages = 0;
    return s;
}

// What one tile covers, as the schedule lays it down.
struct __align__(16) TileShape {
    int32_t request;     // -1: rows of the short list, prefix only
    int32_t row0, rows;  // in the batch, or in that list
    int32_t at0;         // own row of its first batch row
    int32_t pre0, pre1;  // prefix key steps
    int32_t own0, own1;  // own key steps
    int32_t own_limit;   // own keys from here on are seen by none
    int32_t unused[3];
    __device__ int32_t steps() const { return pre1 - pre0 + own1 - own0; }
};

// Work comes in strips, the keys of one tile and KV head, of so many units
// (pages in the row kernel, key steps in the tile kernel). CTAs take equal runs
// of all units, whatever strips they cut: the first `longer` of them run + 1,
// the others run. Strip x's part in CTA c has slot c + x, its own since each
// part begins with the next CTA or the next strip.
struct Runs {
    int32_t run, longer;
    __device__ __forceinline__ int32_t start(int32_t cta) const { return cta * run + min(cta, longer); }
    __device__ __forceinline__ int32_t cta_of(int32_t unit) const {
        const int32_t cut = longer * (run + 1);
        return unit < cut ? unit / (run + 1) : longer + (unit - cut) / run;
    }
};
__device__ __forceinline__ Runs tile_runs(const PagedAttnParams &p) { return Runs{p.header[kTlRun], p.header[kTlLonger]}; }
__device__ __forceinline__ Runs row_runs(const PagedAttnParams &p) { return Runs{p.header[kRtRun], p.header[kRtLonger]}; }

struct RowItem {
    int32_t request;  // -1: prefix
    int32_t tile, head;
    int32_t page0, pages;  // of the request's table or the prefix's
    int32_t limit;         // keys from here on hold nothing
    int32_t row0, rows;    // batch rows of the tile's source
    int32_t at0;
    int32_t slot;
    int32_t direct;  // the only part of its rows: normalise and write the result
};

// 32-way search for the last request whose first row is at or before `row`
// (the one that holds it, since starts never decrease); whole warp.
__device__ __noinline__ int32_t pg_owner(const int32_t *starts, uint32_t requests, int32_t row) {
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
// A part's {m, l}: m of -inf says that it saw no score above that and has no say,
// so a part that saw scores of which none is a number (no maximum, l not a
// number) gets another.
__device__ __forceinline__ float2 pg_ml(float m, float l) { return make_float2(l != l && m == -INFINITY ? 0.0f : m, l); }
// What the sums of a row at own row `at` are multiplied with. A row that is held
// sees itself at least: where l is zero all the same, every score is -inf, and
// the result is none (0 / 0). One that is not held sees nothing: zero.
__device__ __forceinline__ float pg_inverse(int32_t at, float l) { return at < 0 ? 0.0f : 1.0f / l; }
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
// The 8x8 transpose of a matrix of 16-bit elements held two to a lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void rt_bar() { asm volatile("bar.sync 1, %0;" ::"n"(32 * kRtWarps) : "memory"); }
// Two weights as two BF16 terms each: the upper half of each's bits, and what is
// left of the weight and 2^-22 of it more, which is never zero or negative beside a first
// term that is not (a zero times an infinite value, or infinities of two signs,
// would be no number; weights below 2^-104 aside). Of a weight of zero both are zero.
__device__ __forceinline__ void pg_split(float a, float b, uint32_t &first, uint32_t &rest) {
    const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
    constexpr float kMore = 1.0f + 0x1p-22f;
    first = __byte_perm(x, y, 0x7632);
    rest = pg_pack(fmaf(a, kMore, -__uint_as_float(x & 0xffff0000u)), fmaf(b, kMore, -__uint_as_float(y & 0xffff0000u)));
}
constexpr float kLazy = 8.0f;  // a maximum is renewed when passed by 2^8

// Byte offset of a 16-byte chunk in a slab's [boxes][16][128 bytes] rows with
// the copy engine's 128-byte swizzle.
__device__ __forceinline__ uint32_t rt_chunk(uint32_t row, uint32_t chunk) {
    return (chunk >> 3) * (kRtKeys * 128) + row * 128 + (((chunk & 7) ^ (row & 7)) << 4);
}

// A CTA's shared state, as its computing warps use it.
struct RowCta {
    uint64_t *full, *empty;
    const unsigned char *slabs;
    float *joined;              // [2][kRtPairs][128]: the sums of half of the warps each
    float2 (*warp_ml)[kRtPairs];  // [warps]
};

// The keys that a pair of an item sees, [lo, hi); lo -1 where there is no such pair.
__device__ __noinline__ int2 rt_sees(const PagedAttnParams &p, const RowItem &it, int32_t pair) {
    if (pair >= it.rows * p.group) return make_int2(-1, 0);
    const int32_t i = p.by_group.div(pair);
    if (it.request >= 0) {
        const int32_t at = it.at0 + i;
        return make_int2(p.window ? max(max(at, 0) - p.window + 1, 0) : 0, max(at + 1, 0));
    }
    int32_t lo = 0;
    if (p.window && p.requests) {  // its request's length decides: the last one to start at or before row i
        int32_t r = 0, n = p.requests;
        while (n > 1) {
            const int32_t half = n / 2;
            const bool below = p.starts[r + half] <= i;
            r = below ? r + half : r;
            n = below ? n - half : half;
        }
        const OwnShape s = own_shape(p, r);
        lo = min(max(p.prefix + max(s.at0 + i - s.row0, 0) - p.window + 1, 0), p.prefix);
    }
    return make_int2(lo, p.prefix);
}
// Where a pair's query starts (in elements), or -1.
__device__ __forceinline__ int64_t rt_query(const PagedAttnParams &p, const RowItem &it, int32_t pair) {
    if (pair >= it.rows * p.group) return -1;
    const int32_t i = p.by_group.div(pair);
    return static_cast<int64_t>(it.row0 + i) * static_cast<int64_t>(p.q_stride) + (it.head * p.group + pair - i * p.group) * kPgDim;
}

__device__ __forceinline__ void rt_item_bf16(const PagedAttnParams &p, const RowItem &it, const RowCta &cta, int32_t begin, int32_t end,
                                             int32_t slabs, uint32_t ring, bool &dead) {
    constexpr int SLAB = rt_slab_bytes<false>(), SLABS = kRtRing / SLAB;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int32_t pair0 = it.tile * kRtPairs;
    // This thread's pairs, 2 t + c: which keys they see.
    int32_t see_lo[2], see_hi[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const int2 sees = rt_sees(p, it, pair0 + 2 * t + c);
        see_lo[c] = sees.x;
        see_hi[c] = sees.y;
    }
    // Queries as MMA operands.
    uint32_t qf[kPgDim / 16][2];
    {
        const int64_t at = rt_query(p, it, pair0 + g);
        const uint16_t *src = static_cast<const uint16_t *>(p.q) + at;
#pragma unroll
        for (int ks = 0; ks < kPgDim / 16; ++ks)
#pragma unroll
            for (int x = 0; x < 2; ++x) qf[ks][x] = at >= 0 ? *reinterpret_cast<const uint32_t *>(src + 16 * ks + 2 * t + 8 * x) : 0u;
    }
    float o[8][4];  // dims 16 j + g (+ 8) x pairs 2 t (+ 1)
    float mx[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int x = 0; x < 4; ++x) o[j][x] = 0.0f;

    for (int32_t n = warp; n < slabs && !dead; n += kRtWarps) {
        const uint32_t q = ring + n, st = q % SLABS;
        if (!mbar_wait(&cta.full[st], (q / SLABS) & 1u)) dead = true;
        dead = __any_sync(0xffffffffu, dead);
        if (dead) break;
        const int32_t key0 = begin + n * kRtKeys;
        const uint32_t kbase = smem_u32(cta.slabs + st * SLAB), vbase = kbase + SLAB / 2;
        // ---- scores: key g (x = 0, 1) and g + 8 (2, 3) of pairs 2 t, 2 t + 1
        float s[4], c1[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) s[x] = c1[x] = 0.0f;
        {
            const uint32_t r = lane & 15, half = lane >> 4;
#pragma unroll
            for (int ks = 0; ks < kPgDim / 16; ++ks) {
                uint32_t a[4];
                ldsm4(kbase + rt_chunk(r, 2 * ks + half), a);
                mma_bf16(ks & 1 ? c1 : s, a, qf[ks][0], qf[ks][1]);
            }
        }
        // ---- masks; a key that exists and that some pair does not see?
        const int32_t left = min(end - key0, kRtKeys);
        bool hidden = false, move = false;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int c = x & 1, key = g + 8 * (x >> 1);
            const bool seen = key0 + key >= see_lo[c] && key0 + key < see_hi[c] && key < left;
            hidden |= !seen && key < left && see_lo[c] >= 0;
            s[x] = seen ? (s[x] + c1[x]) * p.scale2 : -INFINITY;
            move |= s[x] > mx[c] + kLazy;
        }
        // The reference point moves when a score passes it by 2^8 (the first one always does):
        // weights stay below 2^8, and the sums are rarely scaled.
        if (__any_sync(0xffffffffu, move)) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float top = fmaxf(mx[c], fmaxf(s[c], s[2 + c]));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                const float corr = top == -INFINITY ? 1.0f : pg_exp2(mx[c] - top);
                mx[c] = top;
                sum[c] *= corr;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    o[j][c] *= corr;
                    o[j][2 + c] *= corr;
                }
            }
        }
        // ---- weights, transposed into the product's operand as two BF16 terms (16 bits together:
        // the values are BF16 and both operands have one type). Keys bound the kernel: one request
        // over 131,072 rows takes 59.3 us, 58.9 with one term, 256 requests of 500 rows 142 and 139;
        // one term's results are 2.28e-3 from 64 bits where their own rounding makes 1.69e-3.
        uint32_t pf[2], pr[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float &e = s[2 * h + c];
                e = pg_exp2(e - (mx[c] == -INFINITY ? 0.0f : mx[c]));
                sum[c] += e;
            }
            uint32_t first, rest;
            pg_split(s[2 * h], s[2 * h + 1], first, rest);
            pf[h] = transpose8(first);
            pr[h] = transpose8(rest);
        }
        // ---- sums. A weight of zero times a value that is not finite would be NaN: such values
        // leave the products and are added where they are seen. Only slabs with masked keys are
        // looked over; keys past the end are zeroed in any case.
        const bool careful = __any_sync(0xffffffffu, hidden) || left < kRtKeys;
        bool odd = false;
        const uint32_t r = (lane & 7) + ((lane >> 4) << 3), half = (lane >> 3) & 1;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            uint32_t a[4];
            ldsm4_t(vbase + rt_chunk(r, 2 * j + half), a);
            if (careful) {
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const int key = 2 * t + 8 * (x >> 1);
                    const bool bad0 = (a[x] & 0x7f80u) == 0x7f80u, bad1 = (a[x] & 0x7f800000u) == 0x7f800000u;
                    odd |= (bad0 && key < left) || (bad1 && key + 1 < left);
                    if (bad0 || key >= left) a[x] &= 0xffff0000u;
                    if (bad1 || key + 1 >= left) a[x] &= 0x0000ffffu;
                }
            }
            mma_bf16(o[j], a, pf[0], pf[1]);
            mma_bf16(o[j], a, pr[0], pr[1]);
        }
        if (careful && __any_sync(0xffffffffu, odd)) {
#pragma unroll 1
            for (int key = 0; key < left; ++key) {
                float w[2];
                bool seen[2];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int src = (key & 7) * 4 + t;
                    const float a = __shfl_sync(0xffffffffu, s[c], src), b = __shfl_sync(0xffffffffu, s[2 + c], src);
                    w[c] = key < 8 ? a : b;
                    seen[c] = key0 + key >= see_lo[c] && key0 + key < see_hi[c];
                }
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t dim = 16 * j + 8 * x + g;
                        const float v = __uint_as_float(lds_u16(vbase + rt_chunk(key, dim / 8) + 2 * (dim & 7)) << 16);
                        if (!isfinite(v)) {
                            if (seen[0]) o[j][2 * x] += w[0] * v;
                            if (seen[1]) o[j][2 * x + 1] += w[1] * v;
                        }
                    }
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&cta.empty[st]);
    }

    // ---- join the warps: {m, l} of each pair, then the sums, half of the warps' beside the others'
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        float l = sum[c];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        if (g == 0) cta.warp_ml[warp][2 * t + c] = pg_ml(mx[c], l);
    }
    rt_bar();
    float factor[2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < kRtWarps; ++w) top = fmaxf(top, cta.warp_ml[w][2 * t + c].x);
        factor[c] = mx[c] == -INFINITY ? 0.0f : pg_exp2(mx[c] - top);
    }
#pragma unroll 1
    for (int w = 0; w < kRtWarps / 2; ++w) {
        if (w == warp / 2) {
            float *dst = cta.joined + (warp & 1) * kRtPairs * kPgDim;
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    float *to = dst + (2 * t + (x & 1)) * kPgDim + 16 * j + 8 * (x >> 1) + g;
                    const float v = o[j][x] * factor[x & 1];
                    *to = w ? *to + v : v;
                }
        }
        rt_bar();
    }
}

// FP32: lane l holds dimensions 4l..4l+3 of all eight pairs' queries and sums.
// Four keys' scores are 32 numbers, partial over the lanes: a butterfly leaves
// lane l the score of key l / 8 and pair l % 8. Each step of it keeps half of
// the numbers and sends the other; with key and pair of a register chosen by
// the lane's own number (key ^ l / 8, pair ^ l % 8) it is always the same half
// of the registers, and nothing is selected.
__device__ __forceinline__ void rt_item_f32(const PagedAttnParams &p, const RowItem &it, const RowCta &cta, float *weights,
                                            int32_t begin, int32_t end, int32_t slabs, uint32_t ring, bool &dead) {
    constexpr int SLAB = rt_slab_bytes<true>(), SLABS = kRtRing / SLAB;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int32_t pair0 = it.tile * 8;
    const int2 sees = rt_sees(p, it, pair0 + (lane & 7));
    float4 q[8], o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t at = rt_query(p, it, pair0 + (i ^ (lane & 7)));
        q[i] = at >= 0 ? ld4(static_cast<const float *>(p.q) + at + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
        o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float m = -INFINITY, l = 0.0f;  // of pair lane % 8, l over this lane's keys
    const uint32_t box = (lane >> 3) * (kRtKeys * 128);
    for (int32_t n = warp; n < slabs && !dead; n += kRtWarps) {
        const uint32_t x = ring + n, st = x % SLABS;
        if (!mbar_wait(&cta.full[st], (x / SLABS) & 1u)) dead = true;
        dead = __any_sync(0xffffffffu, dead);
        if (dead) break;
        const int32_t key0 = begin + n * kRtKeys;
        const unsigned char *keys = cta.slabs + st * SLAB + box, *values = keys + SLAB / 2;
        const auto piece = [&](const unsigned char *base, int row) {
            return *reinterpret_cast<const float4 *>(base + row * 128 + (((lane & 7) ^ (row & 7)) << 4));
        };
        float s[4];
#pragma unroll 1
        for (int four = 0; four < 4; ++four) {  // (rolled: the kernel's code is mostly run once)
            float v[4][8];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float4 kv = piece(keys, 4 * four + (k ^ (lane >> 3)));
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    v[k][i] = fmaf(q[i].w, kv.w, fmaf(q[i].z, kv.z, fmaf(q[i].y, kv.y, __fmul_rn(q[i].x, kv.x))));
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                v[0][i] += __shfl_xor_sync(0xffffffffu, v[2][i], 16);
                v[1][i] += __shfl_xor_sync(0xffffffffu, v[3][i], 16);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) v[0][i] += __shfl_xor_sync(0xffffffffu, v[1][i], 8);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[0][i] += __shfl_xor_sync(0xffffffffu, v[0][i + 4], 4);
            v[0][0] += __shfl_xor_sync(0xffffffffu, v[0][2], 2);
            v[0][1] += __shfl_xor_sync(0xffffffffu, v[0][3], 2);
            weights[32 * four + lane] = v[0][0] + __shfl_xor_sync(0xffffffffu, v[0][1], 1);
        }
#pragma unroll
        for (int four = 0; four < 4; ++four) s[four] = weights[32 * four + lane];  // this lane's own
        const int32_t left = min(end - key0, kRtKeys);
        bool hidden = false, move = false;
        uint32_t seen_by[4];  // bit 8 * key + pair of four keys
#pragma unroll
        for (int four = 0; four < 4; ++four) {
            const int key = 4 * four + (lane >> 3);
            const bool seen = key0 + key >= sees.x && key0 + key < sees.y && key < left;
            hidden |= !seen && sees.x >= 0;
            seen_by[four] = __ballot_sync(0xffffffffu, seen);
            s[four] = seen ? s[four] * p.scale2 : -INFINITY;
            move |= s[four] > m + kLazy;
        }
        if (__any_sync(0xffffffffu, move)) {
            float top = fmaxf(fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])), m);
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
            const float corr = top == -INFINITY ? 1.0f : pg_exp2(m - top);
            m = top;
            l *= corr;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float f = __shfl_sync(0xffffffffu, corr, i);
                o[i] = make_float4(o[i].x * f, o[i].y * f, o[i].z * f, o[i].w * f);
            }
        }
#pragma unroll
        for (int four = 0; four < 4; ++four) {
            const float w = pg_exp2(s[four] - (m == -INFINITY ? 0.0f : m));
            l += w;
            weights[32 * four + lane] = w;  // [key][pair]
        }
        __syncwarp();
        if (__any_sync(0xffffffffu, hidden)) {
            // Keys that some pair does not see, or that do not exist: their values, whatever they
            // are, are added for the pairs that see them only.
#pragma unroll 1
            for (int key = 0; key < left; ++key) {
                const float4 v = piece(values, key);
                const uint32_t by = key < 8 ? (key < 4 ? seen_by[0] : seen_by[1]) : (key < 12 ? seen_by[2] : seen_by[3]);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float w = weights[8 * key + i];
                    if ((by >> (8 * (key & 3) + i)) & 1u)
                        o[i] = make_float4(fmaf(w, v.x, o[i].x), fmaf(w, v.y, o[i].y), fmaf(w, v.z, o[i].z), fmaf(w, v.w, o[i].w));
                }
            }
        } else {
#pragma unroll 4
            for (int key = 0; key < kRtKeys; ++key) {
                const float4 v = piece(values, key);
                const float4 a = ld4(weights + 8 * key), b = ld4(weights + 8 * key + 4);
                const float w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    o[i] = make_float4(fmaf(w[i], v.x, o[i].x), fmaf(w[i], v.y, o[i].y), fmaf(w[i], v.z, o[i].z), fmaf(w[i], v.w, o[i].w));
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&cta.empty[st]);
    }
    l += __shfl_xor_sync(0xffffffffu, l, 8);
    l += __shfl_xor_sync(0xffffffffu, l, 16);
    if (lane < 8) cta.warp_ml[warp][lane] = pg_ml(m, l);
    rt_bar();
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < kRtWarps; ++w) top = fmaxf(top, cta.warp_ml[w][lane & 7].x);
    const float factor = m == -INFINITY ? 0.0f : pg_exp2(m - top);
#pragma unroll 1
    for (int w = 0; w < kRtWarps / 2; ++w) {
        if (w == warp / 2) {
            float *dst = cta.joined + (warp & 1) * 8 * kPgDim + 4 * lane;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float f = __shfl_sync(0xffffffffu, factor, i);
                float4 v = make_float4(o[i].x * f, o[i].y * f, o[i].z * f, o[i].w * f);
                if (w) {
                    const float4 u = ld4(dst + i * kPgDim);
                    v = make_float4(v.x + u.x, v.y + u.y, v.z + u.z, v.w + u.w);
                }
                *reinterpret_cast<float4 *>(dst + i * kPgDim) = v;
            }
        }
        rt_bar();
    }
}

// ---- the row kernel ---------------------------------------------------------------
// Items are parts of strips: one tile of pairs over a run of pages. CTAs take
// equal runs of all pages, whatever requests they cut, so ragged lengths cost
// no waiting (whole chunks of a request to a CTA left the last ones alone with
// their work). Own keys are read once per tile and the products are far below
// the tensor pipe's rate, so this is a streaming kernel: one warp copies slabs
// of 16 keys into a ring, two CTAs to an SM, and six warps take a slab each in
// turn, with a running maximum and sums of their own that are joined at the end
// of the item. Scores are computed transposed, keys x pairs: a group of up to
// eight heads then fills the N of an MMA instead of half its M, and the value
// sums (dimensions x pairs) take 32 registers a thread instead of 64, which
// leaves room for 14 warps on an SM.
// FP32 pools take the CUDA cores: 32 multiply-adds a lane for each key's
// scores and as many for its values are 350 issue cycles of an SM per slab,
// half of what the slab's 16 KB take to arrive, and lose nothing to splitting.
// (TF32 mma.sync with two terms to an operand took 5 us per slab and warp; this
// takes 2 to 3, BF16 0.7.)
// Bound: HBM on long runs (one request over 131,072 rows of 1 KB: 53 us cold, 5.1
// TB/s); on short items their ends, about 4 us each (256 requests of 500 rows
// and eight KV heads: 133 us, 4.0 TB/s). The FP32 kernel spills (48 bytes
// stored, 112 loaded) at the 128 registers that two CTAs to an SM leave a thread.
__device__ void paged_schedule(const PagedAttnParams &p, int64_t *sums);  // paged_tiles.cuh

// Request r's work, or the prefix's (r == requests) from page pp0 on.
__device__ __forceinline__ OwnShape row_work(const PagedAttnParams &p, int32_t r, int32_t pp0) {
    if (r < p.requests) {
        OwnShape s = short_shape(p, r);
        if (!s.pages) s.tiles = 0;
        return s;
    }
    OwnShape s{};
    s.rows = p.rows;
    s.length = p.prefix;
    s.page0 = pp0;
    s.pages = (p.prefix + kPgRows - 1) / kPgRows - pp0;
    s.tiles = s.pages ? p.prefix_tiles : 0;
    return s;
}

template <bool F32>
__global__ void __launch_bounds__(kRtThreads, 2)
    paged_rows_kernel(const __grid_constant__ CUtensorMap map, const __grid_constant__ PagedAttnParams p) {
    constexpr int SLAB = rt_slab_bytes<F32>(), SLABS = kRtRing / SLAB;
    static_assert(SLABS % kRtWarps == 0, "a place of the ring serves one warp");
    constexpr int PER = kPgRows / kRtKeys;  // slabs per page
    extern __shared__ __align__(128) unsigned char rt_raw[];
    __shared__ __align__(8) uint64_t full[SLABS], empty[SLABS];
    __shared__ int64_t scan[kRtThreads / 32];
    __shared__ RowItem items[kRtBatch];
    __shared__ float2 warp_ml[kRtWarps][kRtPairs];
    __shared__ __align__(16) float weights[F32 ? kRtWarps : 1][F32 ? kRtKeys * 8 : 4];
    __shared__ int32_t first_strip, last_strip, lowest_at;
    unsigned char *base = reinterpret_cast<unsigned char *>(
        (reinterpret_cast<uintptr_t>(rt_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    float *joined = reinterpret_cast<float *>(base + kRtRing);  // [2][kRtPairs][128]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_launch_dependents();
    if (blockIdx.x == 0) {  // for the kernels that follow, while the others work
        paged_schedule(p, scan);
        return;
    }
    const int32_t worker = static_cast<int32_t>(blockIdx.x) - 1;
    const RowCta cta{full, empty, base, joined, warp_ml};
    if (tid == 0) {
        for (int s = 0; s < SLABS; ++s) {
            mbar_init(&full[s], 1);
            mbar_init(&empty[s], 1);
        }
        fence_barrier_init();
        prefetch_tensormap(&map);
        lowest_at = INT32_MAX;
        first_strip = 0;
        last_strip = -1;
    }

    // Every CTA lays the work out by itself from the requests' lengths: thread
    // t's share of the requests, and the prefix after the last one's.
    const int32_t per = (p.requests + kRtThreads - 1) / kRtThreads;
    const int32_t r0 = min(p.requests, tid * per);
    const int32_t r1 = min(p.requests, r0 + per) + (tid == kRtThreads - 1 && p.prefix_tiles);
    int32_t pp0 = 0;  // first prefix page that some row sees
    if (p.window && p.prefix_tiles) {
        __syncthreads();
        int32_t lowest = INT32_MAX;
        for (int32_t r = r0; r < min(r1, p.requests); ++r) {
            const OwnShape s = own_shape(p, r);
            if (s.rows) lowest = min(lowest, max(s.at0, 0));
        }
        lowest = __reduce_min_sync(0xffffffffu, lowest);
        if (lane == 0) atomicMin(&lowest_at, lowest);
        __syncthreads();
        if (lowest_at != INT32_MAX) pp0 = min(max(p.prefix + lowest_at - p.window + 1, 0), p.prefix) / kPgRows;
    }
    int64_t units = 0, strips = 0, all_units, all_strips;
#pragma unroll 1
    for (int32_t r = r0; r < r1; ++r) {
        const OwnShape s = row_work(p, r, pp0);
        strips += s.tiles * p.kh;
        units += static_cast<int64_t>(s.tiles) * s.pages * p.kh;
    }
    const int64_t unit0 = pg_block_scan<kRtThreads>(units, scan, &all_units);
    const int32_t strip0 = static_cast<int32_t>(pg_block_scan<kRtThreads>(strips, scan, &all_strips));
    if (all_units > INT32_MAX - 1024 || all_strips + p.workers > p.row_slots) {  // starts that overlap, or 2^31 units
        if (tid == 0) pg_flag(p.status, PLAMO_PAGED_BATCH_ROWS);
        all_units = 0;
    }
    const int32_t total = static_cast<int32_t>(all_units);
    const int32_t ctas = min(p.workers, (total + kRtMinPages - 1) / kRtMinPages);
    const Runs runs{ctas ? total / ctas : 1, ctas ? total % ctas : 0};
    const int32_t begin_unit = runs.start(min(worker, ctas)), end_unit = runs.start(min(worker + 1, ctas));
    // The request or prefix of this thread: its strips that this CTA has a part of, as
    // f(shape, request, first unit, first strip).
    const auto each = [&](auto f) {
        int32_t unit = static_cast<int32_t>(unit0), strip = strip0;
#pragma unroll 1
        for (int32_t r = r0; r < r1; ++r) {
            const OwnShape s = row_work(p, r, pp0);
            f(s, r, unit, strip);
            strip += s.tiles * p.kh;
            unit += s.tiles * s.pages * p.kh;
        }
    };
    if (worker == 0) {
        each([&](const OwnShape &s, int32_t r, int32_t unit, int32_t strip) {
            p.row_record[r] = total ? make_int4(unit, s.pages, strip, s.tiles) : make_int4(0, 0, 0, 0);
        });
        if (tid == 0) {
            p.header[kRtRun] = runs.run;
            p.header[kRtLonger] = runs.longer;
        }
    }
    if (begin_unit < end_unit)
        each([&](const OwnShape &s, int32_t, int32_t unit, int32_t strip) {
            const int32_t n = s.tiles * s.pages * p.kh;
            if (begin_unit >= unit && begin_unit < unit + n) first_strip = strip + (begin_unit - unit) / s.pages;
            if (end_unit > unit && end_unit <= unit + n) last_strip = strip + (end_unit - 1 - unit) / s.pages;
        });
    __syncthreads();

    uint32_t ring = 0, issued = 0;  // slabs of the items before; copied ones
    bool dead = false;
#pragma unroll 1
    for (int32_t batch = first_strip; batch <= last_strip; batch += kRtBatch) {
        __syncthreads();  // the last batch's items are done with
        each([&](const OwnShape &s, int32_t r, int32_t unit, int32_t strip) {
            const int32_t x0 = max(batch, strip), x1 = min(min(batch + kRtBatch, last_strip + 1), strip + s.tiles * p.kh);
#pragma unroll 1
            for (int32_t x = x0; x < x1; ++x) {
                const int32_t y = x - strip, from = unit + y * s.pages;  // the strip's units: [from, from + pages)
                RowItem it;
                it.request = r < p.requests ? r : -1;
                it.tile = p.by_kh.div(y);
                it.head = y - it.tile * p.kh;
                const int32_t lo = max(begin_unit - from, 0), hi = min(end_unit - from, s.pages);
                it.page0 = s.page0 + lo;
                it.pages = hi - lo;
                // Keys past the tile's last row are seen by none of its rows.
                const int32_t last = s.at0 + min(s.rows - 1, p.by_group.div(it.tile * kRtPairs + kRtPairs - 1));
                it.limit = r < p.requests ? min(max(last + 1, 0), s.length) : p.prefix;
                it.row0 = s.row0;
                it.rows = s.rows;
                it.at0 = s.at0;
                it.slot = worker + x;
                it.direct = it.pages == s.pages && p.prefix == 0;
                items[x - batch] = it;
            }
        });
        __syncthreads();
#pragma unroll 1
        for (int k = 0; k < kRtBatch; ++k) {
            if (batch + k > last_strip) break;
            const RowItem it = items[k];
            const int32_t begin = it.page0 * kPgRows, end = min(begin + it.pages * kPgRows, it.limit);
            const int32_t slabs = end > begin ? (end - begin + kRtKeys - 1) / kRtKeys : 0;
            if (warp == kRtWarps) {
                // ---- the copying warp: page ids 32 at a time, one lane issues.
                const int32_t *table = it.request < 0 ? p.prefix_pages
                                                      : p.tables + static_cast<uint64_t>(it.request) * p.table_stride;
                for (int32_t n0 = 0; n0 < slabs && !dead; n0 += 32 * PER) {
                    int32_t id = n0 / PER + lane < it.pages ? table[it.page0 + n0 / PER + lane] : 0;
                    if (n0 / PER + lane < it.pages && (id < 0 || id >= p.pages)) {
                        pg_flag(p.status, PLAMO_PAGED_PAGE);
                        id = p.pages;  // past the pool: the copy brings zeros
                    }
#pragma unroll 1
                    for (int32_t n = n0; n < min(slabs, n0 + 32 * PER); ++n) {
                        const int32_t page = __shfl_sync(0xffffffffu, id, (n / PER) & 31);
                        if (lane == 0 && !dead) {
                            const uint32_t q = ring + n, st = q % SLABS;
                            if (q >= SLABS && !mbar_wait(&empty[st], (q / SLABS - 1) & 1u)) {
                                dead = true;
                            } else {
                                unsigned char *dst = base + st * SLAB;
                                const int y = page * 2 * kPgRows + (n % PER) * kRtKeys, x = it.head * kPgDim;
                                mbar_expect_tx(&full[st], SLAB);
                                constexpr int BOX = F32 ? 32 : 64;  // elements in 128 bytes
#pragma unroll
                                for (int b = 0; b < kPgDim / BOX; ++b) {
                                    tma_load_2d(dst + b * kRtKeys * 128, &map, x + b * BOX, y, &full[st]);
                                    tma_load_2d(dst + SLAB / 2 + b * kRtKeys * 128, &map, x + b * BOX, y + kPgRows, &full[st]);
                                }
                                issued = q + 1;
                            }
                        }
                    }
                    dead = __shfl_sync(0xffffffffu, dead, 0);
                }
                ring += slabs;
                continue;
            }
            // ---- the computing warps
            if constexpr (F32) rt_item_f32(p, it, cta, weights[warp], begin, end, slabs, ring, dead);
            else rt_item_bf16(p, it, cta, begin, end, slabs, ring, dead);
            ring += slabs;
            // ---- result, or the tile's partial sums
#pragma unroll 1
            for (int x = tid; x < kRtPairs * kPgDim / 4; x += 32 * kRtWarps) {
                const int pair = x / (kPgDim / 4), d = 4 * (x % (kPgDim / 4));
                float top = -INFINITY, l = 0.0f;
#pragma unroll
                for (int w = 0; w < kRtWarps; ++w) top = fmaxf(top, warp_ml[w][pair].x);
#pragma unroll
                for (int w = 0; w < kRtWarps; ++w) {
                    const float2 ml = warp_ml[w][pair];
                    if (ml.x != -INFINITY) l += pg_exp2(ml.x - top) * ml.y;
                }
                float4 v = ld4(joined + pair * kPgDim + d);
                const float4 u = ld4(joined + (kRtPairs + pair) * kPgDim + d);
                v = make_float4(v.x + u.x, v.y + u.y, v.z + u.z, v.w + u.w);
                if (it.direct) {
                    const int32_t m = it.tile * kRtPairs + pair;
                    if (m >= it.rows * p.group) continue;
                    const int32_t i = p.by_group.div(m);
                    const float inv = pg_inverse(it.at0 + i, l);
                    v = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
                    const uint64_t at = (it.row0 + i) * p.out_stride + (it.head * p.group + m - i * p.group) * kPgDim + d;
                    if constexpr (F32) pg_store4(static_cast<float *>(p.out) + at, v);
                    else pg_store4(static_cast<uint16_t *>(p.out) + at, v);
                } else {
                    const uint64_t at = static_cast<uint64_t>(it.slot) * kRtPairs + pair;
                    *reinterpret_cast<float4 *>(p.row_sum + at * kPgDim + d) = v;
                    if (d == 0) p.row_ml[at] = make_float2(top, l);
                }
            }
            rt_bar();  // before the next item writes warp_ml or the sums
        }
    }
    if (warp == kRtWarps && lane == 0) {
        // Every copy issued has landed before the CTA can exit.
        for (uint32_t n = issued > SLABS ? issued - SLABS : 0; n < issued; ++n)
            if (!mbar_wait(&full[n % SLABS], (n / SLABS) & 1u)) break;
    }
    if (dead && lane == 0) pg_flag(p.status, PLAMO_PAGED_FAILED);
}

// ---- joining the parts ----------------------------------------------------------------
// One result (a row and head): its parts lie in two arrays, the sums of part x
// at (first + x * stride) * rows + place, joined in that order.
struct PartList {
    const float *sum;
    const float2 *ml;
    int32_t first, stride, rows, place, count;
    __device__ __forceinline__ int64_t at(int32_t x) const { return static_cast<int64_t>(first + x * stride) * rows + place; }
};
// Joins RES (2 or 8) results, lane y's lists those of result y % RES (empty
// where there is none). Warp `sub` of `warps` takes every warps-th part of each,
// 32 / RES at a time: a lane weighs one part of one result, then the parts' sums
// are loaded eight at once. Every lane returns with four dimensions of the sums
// over its warp's parts, and l and the maximum m over them of its own result.
template <int RES>
__device__ __forceinline__ void join_parts(const PartList &a, const PartList &b, int32_t sub, int32_t warps, float4 (&o)[RES], float &l,
                                           float &m) {
    const int32_t lane = threadIdx.x & 31, all = a.count + b.count;
    const int32_t most = __reduce_max_sync(0xffffffffu, all);
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < RES; ++i) o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int32_t x0 = sub; x0 < most; x0 += 32 / RES * warps) {
        const int32_t x = x0 + (lane / RES) * warps;
        float2 v = make_float2(-INFINITY, 0.0f);
        const float *from = nullptr;
        if (x < all) {
            const bool first = x < a.count;
            const int64_t at = first ? a.at(x) : b.at(x - a.count);
            v = (first ? a.ml : b.ml)[at];
            from = (first ? a.sum : b.sum) + at * kPgDim;
        }
        float top = fmaxf(m, v.x);
#pragma unroll
        for (int k = RES; k < 32; k <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, k));
        const float w = v.x == -INFINITY ? 0.0f : pg_exp2(v.x - top), corr = m == -INFINITY ? 0.0f : pg_exp2(m - top);
        m = top;
        l = fmaf(w, v.y, l * corr);
        if (x0 != sub) {
#pragma unroll
            for (int i = 0; i < RES; ++i) {
                const float f = __shfl_sync(0xffffffffu, corr, i);
                o[i] = make_float4(o[i].x * f, o[i].y * f, o[i].z * f, o[i].w * f);
            }
        }
#pragma unroll 1
        for (int k = 0; k < 32; k += 8) {
            if (x0 + k / RES * warps >= most) break;
            float4 u[8];
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                f[i] = __shfl_sync(0xffffffffu, w, k + i);
                const float *src = reinterpret_cast<const float *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(from), k + i));
                u[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (f[i] != 0.0f) u[i] = ld4(src + 4 * lane);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float4 &t = o[i % RES];
                t = make_float4(fmaf(f[i], u[i].x, t.x), fmaf(f[i], u[i].y, t.y), fmaf(f[i], u[i].z, t.z), fmaf(f[i], u[i].w, t.w));
            }
        }
    }
#pragma unroll
    for (int k = RES; k < 32; k <<= 1) l += __shfl_xor_sync(0xffffffffu, l, k);
}
template <bool F32>
__device__ __forceinline__ void join_store(const PagedAttnParams &p, int32_t row, int32_t at, int32_t head, float4 o, float l) {
    const float inv = pg_inverse(at, l);
    o = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    const uint64_t to = row * p.out_stride + head * kPgDim + 4 * (threadIdx.x & 31);
    if constexpr (F32) pg_store4(static_cast<float *>(p.out) + to, o);
    else pg_store4(static_cast<uint16_t *>(p.out) + to, o);
}

// Joins the short requests' rows, the prompts' tiles that two or more CTAs
// shared (a warp to RES pairs), and zeroes the rows that see nothing. FEW: a
// block to RES results, its warps sharing their parts; else a warp to RES.
constexpr int kJoinThreads = 256, kJoinWarps = kJoinThreads / 32;
template <bool F32, int RES, bool FEW>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const __grid_constant__ PagedAttnParams p) {
    __shared__ float4 warp_sums[FEW ? kJoinWarps : 1][RES][32];
    __shared__ float2 warp_ml[FEW ? kJoinWarps : 1][RES];
    const int32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    pdl_wait();
    const int32_t tiles = p.tile_rows ? p.header[kTlTiles] : 0, pre_tiles = p.tile_rows ? p.header[kTlPreTiles] : 0;
    const int32_t ctas = p.tile_rows ? p.header[kTlCtas] : 0;
    const int32_t first_row = p.header[kTlFirst], end_row = p.header[kTlTaken];  // of the requests'
    const Runs runs = tile_runs(p), of_rows = row_runs(p);
    PartList shared{}, own{};
    float4 o[RES];
    float l, top;
    const int32_t groups = (p.qh + RES - 1) / RES, items = p.header[kTlShortRows] * groups;
#pragma unroll 1
    for (int32_t n = FEW ? blockIdx.x : blockIdx.x * kJoinWarps + warp; n < items; n += FEW ? gridDim.x : gridDim.x * kJoinWarps) {
        const int32_t listed = n / groups, head0 = RES * (n - listed * groups), head = head0 + (lane & (RES - 1));
        const int4 e = p.short_list[listed];
        shared.count = own.count = 0;
        bool written = false;
        if (e.y >= 0 && head < p.qh) {
            const int32_t kv = p.by_group.div(head), in_group = head - kv * p.group;
            // The parts of row tile m / kRtPairs of request r (or of the prefix) for this head.
            const auto row_parts = [&](int32_t r, int32_t m) {
                const int4 rec = p.row_record[r];
                const int32_t strip = m / kRtPairs * p.kh + kv, u0 = rec.x + strip * rec.y;
                const int32_t c0 = rec.y ? of_rows.cta_of(u0) : 0;
                return PartList{p.row_sum, p.row_ml, c0 + rec.z + strip, 1, kRtPairs, m % kRtPairs,
                                rec.y ? of_rows.cta_of(u0 + rec.y - 1) - c0 + 1 : 0};
            };
            own = row_parts(e.z, e.w * p.group + in_group);
            written = own.count == 1 && p.prefix == 0;  // where it was computed
            if (p.prefix_tiles) {
                shared = row_parts(p.requests, e.x * p.group + in_group);
            } else if (pre_tiles && ctas) {
                const int32_t tile = p.by_tile_rows.div(listed);
                const int32_t unit = p.tile_unit[tile], steps = static_cast<int32_t>(p.tile_unit[tile + 1]) - unit;
                const int32_t u0 = unit * p.kh + kv * steps, c0 = runs.cta_of(u0);
                shared = PartList{p.tile_sum, p.tile_ml, 2 * p.tile_grid + c0 + tile * p.kh + kv, 1, p.tile_pairs,
                                  (listed - tile * p.tile_rows) * p.group + in_group, steps ? runs.cta_of(u0 + steps - 1) - c0 + 1 : 0};
            }
        }
        const uint32_t skip = __ballot_sync(0xffffffffu, written || head >= p.qh);  // (the same in all warps of an item)
        if (skip == 0xffffffffu) continue;
        join_parts<RES>(shared, own, FEW ? warp : 0, FEW ? kJoinWarps : 1, o, l, top);
        if constexpr (FEW) {
#pragma unroll
            for (int i = 0; i < RES; ++i) warp_sums[warp][i][lane] = o[i];
            if (lane < RES) warp_ml[warp][lane] = make_float2(top, l);
            __syncthreads();
            if (warp < RES && !((skip >> warp) & 1u)) {  // warp y puts result y together, the warps' shares in order
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                top = -INFINITY;
                l = 0.0f;
#pragma unroll
                for (int i = 0; i < kJoinWarps; ++i) top = fmaxf(top, warp_ml[i][warp].x);
#pragma unroll
                for (int i = 0; i < kJoinWarps; ++i) {
                    const float2 ml = warp_ml[i][warp];
                    const float f = ml.x == -INFINITY ? 0.0f : pg_exp2(ml.x - top);
                    const float4 u = warp_sums[i][warp][lane];
                    if (f != 0.0f) v = make_float4(fmaf(f, u.x, v.x), fmaf(f, u.y, v.y), fmaf(f, u.z, v.z), fmaf(f, u.w, v.w));
                    l = fmaf(f, ml.y, l);
                }
                join_store<F32>(p, e.x, e.y, head0 + warp, v, l);
            }
            __syncthreads();
        } else {
#pragma unroll
            for (int i = 0; i < RES; ++i) {
                const float li = __shfl_sync(0xffffffffu, l, i);
                if (!((skip >> i) & 1u)) join_store<F32>(p, e.x, e.y, head0 + i, o[i], li);
            }
        }
    }
    // Prompts' tiles that a CTA's end cuts: the first such end does the tile.
    const int32_t blocks = p.tile_pairs / (RES * kJoinWarps);  // to a tile
#pragma unroll 1
    for (int32_t n = blockIdx.x; n < blocks * (ctas - 1); n += gridDim.x) {
        const int32_t c = n / blocks + 1, pair0 = ((n - (c - 1) * blocks) * kJoinWarps + warp) * RES, cut = runs.start(c);
        const int32_t tile = pg_owner(reinterpret_cast<const int32_t *>(p.tile_unit), static_cast<uint32_t>(tiles), p.by_kh.div(cut));
        if (tile < pre_tiles) continue;
        const int32_t unit = p.tile_unit[tile], steps = static_cast<int32_t>(p.tile_unit[tile + 1]) - unit;
        const int32_t kv = (cut - unit * p.kh) / steps, u0 = unit * p.kh + kv * steps, before = runs.start(c - 1);
        const int32_t row0 = p.tile_shape[tile].row0, pairs = p.tile_shape[tile].rows * p.group;
        if (cut == u0 || before > u0 || pair0 >= pairs) continue;
        // CTA c - 1 has this tile as its last run unless it begins with it; the others begin with it.
        const int32_t pair = pair0 + (lane & (RES - 1)), there = pair < pairs;
        shared = PartList{p.tile_sum, p.tile_ml, 2 * (c - 1) + (before == u0 ? 0 : 1), 0, p.tile_pairs, pair, there};
        own = PartList{p.tile_sum, p.tile_ml, 2 * c, 2, p.tile_pairs, pair, there * (runs.cta_of(u0 + steps - 1) - c + 1)};
        join_parts<RES>(shared, own, 0, 1, o, l, top);
#pragma unroll
        for (int i = 0; i < RES; ++i) {
            const float li = __shfl_sync(0xffffffffu, l, i);
            if (pair0 + i >= pairs) break;
            const int32_t row = p.by_group.div(pair0 + i);
            join_store<F32>(p, row0 + row, p.tile_shape[tile].at0 + row, kv * p.group + pair0 + i - row * p.group, o[i], li);
        }
    }
    // Rows that no request has, and tiles without a key.
    const auto clear = [&](int32_t row) {
        for (int32_t x = threadIdx.x; x < p.qh * kPgDim / 4; x += blockDim.x) {
            if constexpr (F32) pg_store4(static_cast<float *>(p.out) + row * p.out_stride + 4 * x, make_float4(0.f, 0.f, 0.f, 0.f));
            else pg_store4(static_cast<uint16_t *>(p.out) + row * p.out_stride + 4 * x, make_float4(0.f, 0.f, 0.f, 0.f));
        }
    };
#pragma unroll 1
    for (int32_t row = blockIdx.x; row < first_row; row += gridDim.x) clear(row);
#pragma unroll 1
    for (int32_t row = end_row + blockIdx.x; row < p.rows; row += gridDim.x) clear(row);
#pragma unroll 1
    for (int32_t tile = pre_tiles + static_cast<int32_t>(blockIdx.x); tile < tiles; tile += gridDim.x)
        if (p.tile_unit[tile + 1] == p.tile_unit[tile])
            for (int32_t i = 0; i < p.tile_shape[tile].rows; ++i) clear(p.tile_shape[tile].row0 + i);
}

}  // namespace plamo

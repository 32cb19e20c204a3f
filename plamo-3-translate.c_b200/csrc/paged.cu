// Host side of the paged batch operators (include/plamo_paged.h).
#include "../../include/plamo_cuda.h"
#include "../../include/plamo_paged.h"
#include "context.h"
#include "paged.cuh"
#include "paged_attention.cuh"
#include "paged_tiles.cuh"

#include <algorithm>
#include <cmath>

using namespace plamo;

namespace {

cudaStream_t stream_of(const plamo_cuda *c, void *stream) {
    return stream ? static_cast<cudaStream_t>(stream) : context_stream(c);
}
bool aligned(const void *p, uintptr_t a) { return reinterpret_cast<uintptr_t>(p) % a == 0; }
uint64_t element_bytes(uint32_t type) { return type == PLAMO_PAGED_FP32 ? 4 : 2; }
bool type_ok(uint32_t type) { return type == PLAMO_PAGED_BF16 || type == PLAMO_PAGED_FP32; }
bool overlap(const int32_t *a, uint64_t na, const int32_t *b, uint64_t nb) { return a && b && na && nb && a < b + nb && b < a + na; }
uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

template <typename... KArgs, typename... Args>
bool launch(plamo_cuda *c, const char *what, void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem,
            cudaStream_t stream, bool dependent, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    if (dependent && context_pdl(c)) {
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
    }
    return context_launched(c, what, cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...));
}

// Shapes of an attention call; NULL when they are fine, else what is wrong.
const char *attention_shapes(const plamo_paged_attention_args *d) {
    if (!type_ok(d->type)) return "paged_attention: type must be PLAMO_PAGED_BF16 or PLAMO_PAGED_FP32";
    if (!d->kv_heads || !d->query_heads || d->query_heads % d->kv_heads || d->query_heads > 4096)
        return "paged_attention: query_heads must be a multiple of kv_heads, at most 4096";
    // (threads step through both in 32 bits, a grid past the end)
    if (d->rows > kPgMaxCount || d->requests > kPgMaxCount || d->rows * d->query_heads > kPgMaxCount)
        return "paged_attention: at most 2^30 requests, and rows times query heads";
    if (!d->pages || d->pages > static_cast<uint64_t>(kPgMaxPages) / 4)
        return "paged_attention: pages must be 1 to 2^23";
    if (d->prefix_rows > INT32_MAX / 2 || d->table_stride > INT32_MAX / 2 / kPgRows)
        return "paged_attention: the prefix and a request's page table hold at most 2^30 rows each";
    if (d->prefix_rows > d->pages * kPgRows) return "paged_attention: the prefix does not fit the pool";
    return nullptr;
}

// How an attention call is laid out: the workspace's parts and the grid.
struct AttentionLayout {
    uint32_t prefix_tiles, row_slots, workers, tile_rows, tile_grid, tile_cap;
    uint64_t record, row_sum, row_ml;
    uint64_t header, short_list, tile_shape, tile_unit, tile_sum, tile_ml, bytes;
};

AttentionLayout attention_layout(const plamo_cuda *c, const plamo_paged_attention_args *d) {
    AttentionLayout a{};
    const uint64_t group = d->query_heads / d->kv_heads, sms = static_cast<uint64_t>(context_sms(c));
    const uint64_t pairs = d->rows * group, prefix_pages = ceil_div(d->prefix_rows, kPgRows);
    // The tile kernel is for prompts, requests of more pairs than a short one has:
    // where the caller says so, or says nothing and there are more rows than
    // requests (a step whose padding or idle slots hide what it is has to say). And
    // only where the row kernel's work, a unit for eight pairs, a KV head and a page,
    // takes longer than another kernel to begin and end, with the page tables as
    // full as they can be, since lengths are on the device. Eight heads to each of
    // four KV heads: one request behind 12 rows, 320 units 14 us there and 33 with
    // tiles, 1,536 31 and 38, 3,584 64 and 40; 16 of nine rows behind 12, 2,880 units
    // 53 and 36; in FP32 six of 16 rows, 1,536 units 35 and 48, of 32, 3,072 57 and 49.
    // In BF16 it is also for a prefix that would keep the row kernel longer. A step
    // of 128 keys costs what four units do, however few of its tile's 256 pairs there
    // are, so few pairs stay there: one request behind 65,536 rows 38 us there and 71
    // with tiles, two 55 and 73, four 98 and 74; 16 behind 2,048 24 and 29, behind
    // 4,096 36 and 31; 61 behind 512 29 and 37, behind 1,024 39 and 38, behind 2,048
    // 58 and 39. In FP32 the tiles' rate is no better than the row kernel's (61 behind
    // 512 rows 76 us in it; behind 1,000, 2,000 with tiles 103, 136: the same slope,
    // 12 us more).
    const bool f32 = d->type == PLAMO_PAGED_FP32;
    const uint64_t tile_pairs = f32 ? kTfPairs : kTlPairs;
    const uint64_t strips = ceil_div(pairs, kRtPairs) * d->kv_heads;
    const uint64_t prefix_steps = ceil_div(pairs, kTlPairs) * d->kv_heads * ceil_div(d->prefix_rows, kTlKeys);
    const bool prompts = (d->most_new ? std::min(d->most_new, d->rows) * group : d->rows > d->requests ? pairs : 0) > kTlShortPairs;
    if (group <= tile_pairs && ((prompts && strips * (prefix_pages + d->table_stride) > kTlPromptUnits) ||
                                (!f32 && strips * prefix_pages > kTlPrefixUnits + 4 * prefix_steps))) {
        a.tile_rows = static_cast<uint32_t>(tile_pairs / group);
        a.tile_grid = static_cast<uint32_t>(f32 ? 2 * sms : sms);
        // Prefix tiles of the short requests' rows, and each prompt's own with a last partial one.
        a.tile_cap = static_cast<uint32_t>(2 * ceil_div(d->rows, a.tile_rows) + std::min(d->requests, d->rows));
    }
    a.prefix_tiles = prefix_pages && !a.tile_rows ? static_cast<uint32_t>(ceil_div(pairs, kRtPairs)) : 0;
    a.workers = static_cast<uint32_t>(2 * sms - 1);  // beside the schedule's CTA
    // A slot for each strip (a row tile and KV head; every request's last tile
    // may be partial), one more for each CTA. Beside the tile kernel only
    // requests of up to kTlShortPairs pairs are here.
    const uint64_t tiles = pairs / kRtPairs + std::min<uint64_t>(d->requests, d->rows);
    a.row_slots = static_cast<uint32_t>(std::min<uint64_t>(
        a.workers + d->kv_heads * (a.prefix_tiles + (a.tile_rows ? std::min<uint64_t>(tiles, kTlShortPairs / kRtPairs * d->requests) : tiles)),
        INT32_MAX));
    uint64_t at = 0;
    auto part = [&](uint64_t bytes) {
        const uint64_t here = at;
        at += (bytes + 255) / 256 * 256;
        return here;
    };
    a.header = part(kTlHeader * 4);
    a.short_list = part(d->rows * sizeof(int4));
    a.record = part((d->requests + 1) * sizeof(int4));
    a.row_sum = part(static_cast<uint64_t>(a.row_slots) * kRtPairs * kPgDim * 4);
    a.row_ml = part(static_cast<uint64_t>(a.row_slots) * kRtPairs * sizeof(float2));
    if (a.tile_rows) {
        // Two runs of a CTA may end inside a prompt's tile; every run of a prefix tile is a part.
        const uint64_t shared = prefix_pages ? a.tile_grid + ceil_div(d->rows, a.tile_rows) * d->kv_heads : 0;
        const uint64_t slots = 2ull * a.tile_grid + shared;
        a.tile_shape = part(a.tile_cap * sizeof(TileShape));
        a.tile_unit = part((a.tile_cap + 1ull) * 4);
        a.tile_sum = part(slots * tile_pairs * kPgDim * 4);
        a.tile_ml = part(slots * tile_pairs * sizeof(float2));
    }
    a.bytes = std::max<uint64_t>(at, 256);
    return a;
}

template <bool F32>
bool run_attention(plamo_cuda *c, const plamo_paged_attention_args *d, const AttentionLayout &a, cudaStream_t stream) {
    const auto pool_map = [&](CUtensorMap *map, uint32_t rows) {
        return tensor_map_2d(map, F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, F32 ? 4 : 2,
                             d->pool, d->pages * 2 * kPgRows, static_cast<uint64_t>(d->kv_heads) * kPgDim, F32 ? 32 : 64, rows);
    };
    CUtensorMap map, page_map;
    if (!pool_map(&map, kRtKeys) || (a.tile_rows && !pool_map(&page_map, kPgRows)))
        return context_launched(c, "paged_attention: tensor map", cudaErrorInvalidValue);
    char *ws = static_cast<char *>(d->workspace);
    PagedAttnParams p{};
    p.q = d->q;
    p.out = d->out;
    p.starts = d->starts;
    p.lengths = d->lengths;
    p.tables = d->tables;
    p.prefix_pages = d->prefix_pages;
    p.q_stride = d->q_stride;
    p.out_stride = d->out_stride;
    p.table_stride = d->table_stride;
    p.status = d->status ? d->status : context_paged_status(c);
    p.rows = static_cast<int32_t>(d->rows);
    p.requests = static_cast<int32_t>(d->requests);
    p.pages = static_cast<int32_t>(d->pages);
    p.qh = static_cast<int32_t>(d->query_heads);
    p.kh = static_cast<int32_t>(d->kv_heads);
    p.group = p.qh / p.kh;
    p.by_group = FastDiv::of(p.group);
    p.by_kh = FastDiv::of(p.kh);
    p.prefix = static_cast<int32_t>(d->prefix_rows);
    p.max_length = static_cast<int32_t>(d->table_stride * kPgRows);
    // A window that reaches back past every row hides nothing.
    p.window = d->window > d->prefix_rows + d->table_stride * kPgRows ? 0 : static_cast<int32_t>(d->window);
    p.scale2 = d->scale * 1.4426950408889634f;
    // The tile kernel masks before it scales: -inf must stay so.
    if (std::fabs(p.scale2) < 1e-30f) p.scale2 = std::copysign(1e-30f, p.scale2);
    p.row_record = reinterpret_cast<int4 *>(ws + a.record);
    p.header = reinterpret_cast<int32_t *>(ws + a.header);
    p.short_list = reinterpret_cast<int4 *>(ws + a.short_list);
    p.row_sum = reinterpret_cast<float *>(ws + a.row_sum);
    p.row_ml = reinterpret_cast<float2 *>(ws + a.row_ml);
    p.row_slots = static_cast<int32_t>(a.row_slots);
    p.prefix_tiles = static_cast<int32_t>(a.prefix_tiles);
    p.workers = static_cast<int32_t>(a.workers);
    if (a.tile_rows) {
        p.pool = d->pool;
        p.tile_rows = static_cast<int32_t>(a.tile_rows);
        p.by_tile_rows = FastDiv::of(a.tile_rows);
        p.tile_pairs = F32 ? kTfPairs : kTlPairs;
        p.tile_keys = F32 ? kTfKeys : kTlKeys;
        p.tile_grid = static_cast<int32_t>(a.tile_grid);
        p.tile_cap = static_cast<int32_t>(a.tile_cap);
        p.tile_shape = reinterpret_cast<TileShape *>(ws + a.tile_shape);
        p.tile_unit = reinterpret_cast<uint32_t *>(ws + a.tile_unit);
        p.tile_sum = reinterpret_cast<float *>(ws + a.tile_sum);
        p.tile_ml = reinterpret_cast<float2 *>(ws + a.tile_ml);
    }
    if (!launch(c, "paged_attention rows", paged_rows_kernel<F32>, dim3(a.workers + 1), dim3(kRtThreads), kRtSmem, stream, false, map, p) ||
        (a.tile_rows && !launch(c, "paged_attention tiles", F32 ? paged_tile_f32_kernel : paged_tile_kernel, dim3(a.tile_grid),
                                dim3(F32 ? kTfThreads : kTlThreads), F32 ? kTfSmem : kTlSmem, stream, true, page_map, p)))
        return false;
    // Two results to a block, its warps sharing their parts, while that takes two
    // blocks to an SM at most (one request over 131,072 rows, 74 parts each: 10 us
    // against 26 with eight to a block); then eight to a block, up to four blocks
    // (61 requests behind a long prefix, 19 parts: 14 us against 27 with two to a
    // warp); then eight to a warp (256 requests, 6 parts: 21 us against 39).
    const uint64_t sms = static_cast<uint64_t>(context_sms(c)), twos = d->rows * ceil_div(d->query_heads, 2);
    const uint64_t eights = d->rows * ceil_div(d->query_heads, 8);
    const auto join = twos <= 2 * sms     ? paged_join_kernel<F32, 2, true>
                      : eights <= 4 * sms ? paged_join_kernel<F32, 8, true>
                                          : paged_join_kernel<F32, 8, false>;
    const uint64_t blocks = std::min(4 * sms, std::max<uint64_t>(a.tile_rows ? 4 * sms : 1, twos <= 2 * sms ? twos : eights));
    return launch(c, "paged_attention join", join, dim3(static_cast<uint32_t>(blocks)), dim3(kJoinThreads), 0, stream, true, p);
}

template <typename In, typename Out>
bool run_store(plamo_cuda *c, const plamo_paged_store_args *d, cudaStream_t stream) {
    const uint64_t heads = d->query_heads + 2ull * d->kv_heads;
    // Eight heads to a warp once one head each would be four rounds of eight warps
    // to an SM; one to a warp for the few rows of a decode step, where latency
    // counts (8 rows: 3.7 us).
    const bool wide = d->rows * heads >= 4ull * 8 * static_cast<uint64_t>(context_sms(c));
    const uint64_t units = d->rows * ceil_div(heads, wide ? 8 : 1);
    const dim3 grid(static_cast<uint32_t>(ceil_div(units, 8)));
    plamo_paged_store_args args = *d;
    if (!args.status) args.status = context_paged_status(c);
    if (wide)
        return launch(c, "paged_store", paged_store_kernel<In, Out, 8>, grid, dim3(256), 0, stream, false, args);
    return launch(c, "paged_store", paged_store_kernel<In, Out, 1>, grid, dim3(256), 0, stream, false, args);
}

}  // namespace

namespace plamo {
cudaError_t paged_configure() {
    const auto allow = [](auto kernel, int bytes) {
        return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    };
    cudaError_t e = allow(paged_rows_kernel<false>, kRtSmem);
    if (e == cudaSuccess) e = allow(paged_rows_kernel<true>, kRtSmem);
    if (e == cudaSuccess) e = allow(paged_tile_kernel, kTlSmem);
    if (e == cudaSuccess) e = allow(paged_tile_f32_kernel, kTfSmem);
    return e;
}
}  // namespace plamo

extern "C" {

int plamo_paged_plan(struct plamo_cuda *c, const struct plamo_paged_plan_args *d) {
    if (!c || !d) return 0;
    if (!d->lengths || !d->starts || !d->summary || (d->requests && (!d->held || !d->added || (d->table_stride && !d->tables))) ||
        (d->rows && (!d->slots || !d->positions)) || (d->free_count && !d->free_pages))
        return context_decline(c, "paged_plan: a buffer is missing");
    if (d->rows > INT32_MAX - kPlanThreads || d->requests >= INT32_MAX || d->free_count > INT32_MAX ||
        d->table_stride > static_cast<uint64_t>(kPgMaxPages) || d->base < 0 || d->base > INT32_MAX)
        return context_decline(c, "paged_plan: a count is out of range");
    if (overlap(d->head, 1, d->summary, 4)) return context_decline(c, "paged_plan: head must not lie in this plan's own summary");
    // Every CTA reads the counts by itself, so none may write what another reads. Lengths that
    // replace `held` are written by a launch of their own, or by the only CTA, whose threads
    // read the entries that they write.
    const uint64_t R = d->requests;
    const bool in_place = R && d->lengths == d->held;
    const struct {
        const int32_t *at;
        uint64_t count;
    } buffers[] = {{d->lengths, R}, {d->starts, R + 1}, {d->slots, d->rows}, {d->positions, d->rows}, {d->summary, 4},
                   {d->tables, R * d->table_stride},  // (read and written)
                   {d->held, R}, {d->added, R}, {d->free_pages, d->free_count}, {d->head, 1}};
    for (int i = 0; i < 6; ++i)
        for (int j = i + 1; j < 10; ++j)
            if (!(i == 0 && j == 6 && in_place) && overlap(buffers[i].at, buffers[i].count, buffers[j].at, buffers[j].count))
                return context_decline(c, "paged_plan: buffers overlap (only lengths may be held itself)");
    ContextDevice device(c);
    const uint32_t grid = static_cast<uint32_t>(std::max<uint64_t>(1, ceil_div(d->rows, kPlanThreads)));
    const cudaStream_t stream = stream_of(c, d->stream);
    PlanParams p{*d};
    const bool apart = in_place && grid > 1;
    if (apart) p.d.lengths = nullptr;
    if (!launch(c, "paged_plan", paged_plan_kernel, dim3(grid), dim3(kPlanThreads), 0, stream, false, p)) return -1;
    if (!apart) return 1;
    return launch(c, "paged_plan lengths", paged_plan_lengths_kernel, dim3(static_cast<uint32_t>(ceil_div(R, kPlanThreads))),
                  dim3(kPlanThreads), 0, stream, false, d->lengths, d->added, d->summary, R)
               ? 1
               : -1;
}

int plamo_paged_store(struct plamo_cuda *c, const struct plamo_paged_store_args *d) {
    if (!c || !d) return 0;
    if (!type_ok(d->qkv_type) || !type_ok(d->pool_type))
        return context_decline(c, "paged_store: types must be PLAMO_PAGED_BF16 or PLAMO_PAGED_FP32");
    if (!d->kv_heads || !d->query_heads || d->query_heads % d->kv_heads || d->query_heads > 4096)
        return context_decline(c, "paged_store: query_heads must be a multiple of kv_heads, at most 4096");
    if (!d->pages || d->pages > static_cast<uint64_t>(kPgMaxPages) || d->rows > INT32_MAX / 4096)
        return context_decline(c, "paged_store: pages must be 1 to 2^25 and rows below 2^19");
    const uint64_t heads = d->query_heads + 2ull * d->kv_heads;
    if (d->qkv_stride < heads * kPgDim || d->q_stride < static_cast<uint64_t>(d->query_heads) * kPgDim)
        return context_decline(c, "paged_store: a row stride is shorter than its row");
    if (!d->rows) return 1;
    if (!d->qkv || !d->pool || !d->q || !d->slots || !d->positions || !d->q_norm || !d->k_norm ||
        (d->positions_count && !d->table))
        return context_decline(c, "paged_store: a buffer is missing");
    // Four elements at a time.
    if (!aligned(d->qkv, 4 * element_bytes(d->qkv_type)) || !aligned(d->q, 4 * element_bytes(d->pool_type)) ||
        d->qkv_stride % 4 || d->q_stride % 4 || !aligned(d->pool, 16) || !aligned(d->q_norm, 8) ||
        !aligned(d->k_norm, 8) || !aligned(d->table, 16))
        return context_decline(c, "paged_store: rows must start on four-element boundaries, pool and table on 16 bytes, norms on 8");
    ContextDevice device(c);
    const cudaStream_t stream = stream_of(c, d->stream);
    const bool in32 = d->qkv_type == PLAMO_PAGED_FP32, out32 = d->pool_type == PLAMO_PAGED_FP32;
    const bool ok = in32 ? (out32 ? run_store<float, float>(c, d, stream) : run_store<float, uint16_t>(c, d, stream))
                         : (out32 ? run_store<uint16_t, float>(c, d, stream) : run_store<uint16_t, uint16_t>(c, d, stream));
    return ok ? 1 : -1;
}

uint32_t plamo_paged_status(struct plamo_cuda *c) {
    if (!c) return 0;
    ContextDevice device(c);
    uint32_t bits = 0, *words = context_paged_status(c);
    const cudaStream_t stream = context_stream(c);
    const bool ok = launch(c, "paged_status", paged_status_kernel, dim3(1), dim3(1), 0, stream, false, words) &&
                    context_note(c, "paged_status", cudaMemcpyAsync(&bits, words + 1, 4, cudaMemcpyDeviceToHost, stream)) &&
                    context_note(c, "paged_status", cudaStreamSynchronize(stream));
    return ok ? bits : PLAMO_PAGED_FAILED;
}

uint64_t plamo_paged_attention_workspace(struct plamo_cuda *c, const struct plamo_paged_attention_args *d) {
    if (!c || !d) return 0;
    if (const char *why = attention_shapes(d)) return static_cast<uint64_t>(context_decline(c, why));
    return attention_layout(c, d).bytes;
}

int plamo_paged_attention(struct plamo_cuda *c, const struct plamo_paged_attention_args *d) {
    if (!c || !d) return 0;
    if (const char *why = attention_shapes(d)) return context_decline(c, why);
    const uint64_t width = static_cast<uint64_t>(d->query_heads) * kPgDim, per16 = 16 / element_bytes(d->type);
    if (d->q_stride < width || d->out_stride < width)
        return context_decline(c, "paged_attention: a row stride is shorter than its row");
    if (!std::isfinite(d->scale)) return context_decline(c, "paged_attention: scale must be finite");
    if (!d->rows) return 1;
    if (!d->q || !d->pool || !d->out || !d->starts || (d->requests && (!d->lengths || (d->table_stride && !d->tables))) ||
        (d->prefix_rows && !d->prefix_pages))
        return context_decline(c, "paged_attention: a buffer is missing");
    if (!aligned(d->q, 16) || !aligned(d->out, 16) || !aligned(d->pool, 16) || d->q_stride % per16 || d->out_stride % per16)
        return context_decline(c, "paged_attention: pool, queries and results must start on 16-byte boundaries, row by row");
    const AttentionLayout a = attention_layout(c, d);
    if (!d->workspace || !aligned(d->workspace, 256) || d->workspace_bytes < a.bytes)
        return context_decline(c, "paged_attention: the workspace is missing, too small or not 256-byte aligned");
    ContextDevice device(c);
    const cudaStream_t stream = stream_of(c, d->stream);
    const bool ok = d->type == PLAMO_PAGED_FP32 ? run_attention<true>(c, d, a, stream) : run_attention<false>(c, d, a, stream);
    return ok ? 1 : -1;
}

}  // extern "C"

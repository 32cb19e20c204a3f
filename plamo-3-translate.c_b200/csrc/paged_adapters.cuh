// Low-rank adapters of a batch's requests (include/plamo_paged.h):
//   out[row] = base[row] + scale * B (A x[row]),
// A [rank][columns], B [outputs][rank] those of the row's request. Two launches,
// the inner products' sums h = A x in between: h of a row needs all of A and x,
// every output all of h.
#pragma once
#include "paged_attention.cuh"

namespace plamo {

struct AdapterParams {
    const void *x, *base;
    void *out;
    const uint16_t *a, *b;
    const float *scales;
    const int32_t *ids, *starts;
    uint32_t *status;
    float *inner;  // [splits][rows][rank] sums over a share of the columns
    uint64_t x_stride, base_stride, out_stride;
    int32_t rows, columns, outputs, requests, adapters, rank;
    int32_t splits, share;  // columns to a split, a multiple of kAdColumns
};
constexpr int kAdRows = 8;       // to a tile: the N of one mma.sync
constexpr int kAdWarps = 8, kAdThreads = 32 * kAdWarps;
constexpr int kAdColumns = 64 * kAdWarps;  // a round of a CTA's warps

// FP32 as BF16 terms whose sum is the value: the upper 16 bits, and twice the upper bits of what is
// left. A value that is not finite is its first term alone (infinity less itself would be no number).
__device__ __forceinline__ uint32_t ad_top(float v) {  // (a number's upper half may not turn a NaN into an infinity)
    return v != v ? 0x7fff0000u : __float_as_uint(v) & 0xffff0000u;
}
__device__ __forceinline__ float ad_rest(float v, uint32_t top) { return isfinite(v) ? v - __uint_as_float(top) : 0.0f; }
template <int TERMS>
__device__ __forceinline__ void ad_split(float v0, float v1, uint32_t (&t)[TERMS]) {
#pragma unroll
    for (int i = 0; i < TERMS; ++i) {
        const uint32_t a = ad_top(v0), b = ad_top(v1);
        t[i] = __byte_perm(a, b, 0x7632);
        v0 = ad_rest(v0, a);
        v1 = ad_rest(v1, b);
    }
}

// The adapter of batch row `row`, -1 where it has none; whole warp.
__device__ __forceinline__ int32_t ad_row_adapter(const AdapterParams &p, int32_t row) {
    if (!p.requests || row >= p.rows || row < p.starts[0] || row >= p.starts[p.requests]) return -1;
    const int32_t id = p.ids[pg_owner(p.starts, p.requests, row)];
    if (id >= -1 && id < p.adapters) return id;
    if ((threadIdx.x & 31) == 0) pg_flag(p.status, PLAMO_PAGED_ADAPTER);
    return -1;
}
// Fills adapter[] (kAdRows entries, shared) for the tile's rows, a warp to a row.
__device__ __forceinline__ void ad_tile(const AdapterParams &p, int32_t row0, int32_t *adapter) {
    const int32_t warp = threadIdx.x >> 5;
    const int32_t id = ad_row_adapter(p, row0 + warp);
    if ((threadIdx.x & 31) == 0) adapter[warp] = id;
    __syncthreads();
}

// ---- inner products, few rows -----------------------------------------------------------
// A CTA takes eight rows, 16 of the ranks and a share of the columns; its warps
// 64 columns each in turn. A's rows are the M of an MMA, the batch's rows its N,
// so that a single row of a decode step costs no more than reading A. The
// products' order along the columns is free: lane t of four takes columns 16 t to
// 16 t + 15 of 64, so that both operands come in whole 16-byte pieces from
// global memory, A's once per run of rows with the same adapter.
template <typename X>
__global__ void __launch_bounds__(kAdThreads) paged_adapters_inner_kernel(const __grid_constant__ AdapterParams p) {
    constexpr int TERMS = sizeof(X) == 4 ? 3 : 1;
    __shared__ int32_t adapter[kAdRows];
    __shared__ float sums[kAdWarps][16][kAdRows + 1];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int32_t row0 = blockIdx.x * kAdRows, rank0 = blockIdx.z * 16;
    pdl_launch_dependents();
    ad_tile(p, row0, adapter);
    const int32_t begin = blockIdx.y * p.share, end = min(begin + p.share, p.columns);
    const bool there = row0 + g < p.rows && adapter[g] >= 0;
    const X *x = static_cast<const X *>(p.x) + static_cast<uint64_t>(there ? row0 + g : 0) * p.x_stride;
    float total[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
    for (int32_t c0 = begin + 64 * warp; c0 < end; c0 += kAdColumns) {
        const int32_t c = c0 + 16 * t;
        // x of this lane's row: pairs (2 j, 2 j + 1) of its 16 columns
        uint32_t xf[8][TERMS];
        if constexpr (sizeof(X) == 4) {
            float v[16];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4 u = there && c + 4 * j < end ? ld4(reinterpret_cast<const float *>(x) + c + 4 * j) : make_float4(0.f, 0.f, 0.f, 0.f);
                v[4 * j] = u.x, v[4 * j + 1] = u.y, v[4 * j + 2] = u.z, v[4 * j + 3] = u.w;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) ad_split<TERMS>(v[2 * j], v[2 * j + 1], xf[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint4 u = there && c + 8 * j < end ? *reinterpret_cast<const uint4 *>(reinterpret_cast<const uint16_t *>(x) + c + 8 * j)
                                                         : make_uint4(0, 0, 0, 0);
                xf[4 * j][0] = u.x, xf[4 * j + 1][0] = u.y, xf[4 * j + 2][0] = u.z, xf[4 * j + 3][0] = u.w;
            }
        }
#pragma unroll 1
        for (int first = 0; first < kAdRows;) {  // runs of rows with one adapter
            const int32_t id = adapter[first];
            int last = first + 1;
            while (last < kAdRows && adapter[last] == id) ++last;
            if (id >= 0) {
                uint4 w[2][2];
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int32_t r = rank0 + g + 8 * i;
                        w[i][j] = r < p.rank && c + 8 * j < end
                                      ? *reinterpret_cast<const uint4 *>(p.a + (static_cast<uint64_t>(id) * p.rank + r) * p.columns + c + 8 * j)
                                      : make_uint4(0, 0, 0, 0);
                    }
                float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint4 lo = w[0][j >> 1], hi = w[1][j >> 1];
                    const uint32_t m[4] = {j & 1 ? lo.z : lo.x, j & 1 ? hi.z : hi.x, j & 1 ? lo.w : lo.y, j & 1 ? hi.w : hi.y};
#pragma unroll
                    for (int term = TERMS - 1; term >= 0; --term) mma_bf16(s, m, xf[2 * j][term], xf[2 * j + 1][term]);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {  // the other rows' sums are not theirs, whatever this adapter holds
                    const int row = 2 * t + (k & 1);
                    if (row >= first && row < last) total[k] += s[k];
                }
            }
            first = last;
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) sums[warp][g + 8 * (k >> 1)][2 * t + (k & 1)] = total[k];
    __syncthreads();
    if (tid < 16 * kAdRows) {
        const int r = tid & 15, row = tid >> 4;
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < kAdWarps; ++w) s += sums[w][r][row];
        if (rank0 + r < p.rank && row0 + row < p.rows)
            p.inner[(static_cast<uint64_t>(blockIdx.y) * p.rows + row0 + row) * p.rank + rank0 + r] = s;
    }
}

// ---- outputs, few rows ----------------------------------------------------------------------
// A CTA takes eight rows and 128 outputs at a time, 16 to a warp. B's rows are the M
// of an MMA; h enters as three BF16 terms, which are all of its 24 bits.
constexpr int kAdMaxRank = 256;
constexpr int kAdOutputs = 16 * kAdWarps;

template <typename T>
__device__ __forceinline__ float ad_load(const T *p) {
    if constexpr (sizeof(T) == 4) return *p;
    else return bf16_to_f32(*p);
}
template <typename T>
__device__ __forceinline__ void ad_store(T *p, float v) {
    if constexpr (sizeof(T) == 4) *p = v;
    else *p = static_cast<uint16_t>(pg_pack(v, 0.0f));
}

template <typename T>
__global__ void __launch_bounds__(kAdThreads) paged_adapters_outer_kernel(const __grid_constant__ AdapterParams p, int32_t per) {
    __shared__ int32_t adapter[kAdRows];
    __shared__ uint32_t h[3][kAdRows][kAdMaxRank / 2 + 4];  // terms of scale * h, two ranks to a word
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    const int32_t row0 = blockIdx.x * kAdRows, pairs = p.rank / 2, steps = (p.rank + 15) / 16;
    ad_tile(p, row0, adapter);
    pdl_wait();
    for (int32_t x = tid; x < kAdRows * 8 * steps; x += kAdThreads) {
        const int32_t row = x / (8 * steps), pair = x - row * 8 * steps;
        float2 s = make_float2(0.f, 0.f);
        if (adapter[row] >= 0 && pair < pairs) {
            const float *from = p.inner + static_cast<uint64_t>(row0 + row) * p.rank + 2 * pair;
#pragma unroll 4
            for (int32_t y = 0; y < p.splits; ++y) {
                const float2 v = *reinterpret_cast<const float2 *>(from + static_cast<uint64_t>(y) * p.rows * p.rank);
                s.x += v.x;
                s.y += v.y;
            }
            const float scale = p.scales ? p.scales[adapter[row]] : 1.0f;
            s.x *= scale;
            s.y *= scale;
        }
        uint32_t terms[3];
        ad_split<3>(s.x, s.y, terms);
#pragma unroll
        for (int i = 0; i < 3; ++i) h[i][row][pair] = terms[i];
    }
    __syncthreads();
#pragma unroll 1
    for (int32_t y = 0; y < per; ++y) {
        const int32_t n0 = (blockIdx.y * per + y) * kAdOutputs + 16 * warp;
        if (n0 >= p.outputs) break;
        float total[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int first = 0; first < kAdRows;) {
            const int32_t id = adapter[first];
            int last = first + 1;
            while (last < kAdRows && adapter[last] == id) ++last;
            if (id >= 0) {
                float s[4] = {0.f, 0.f, 0.f, 0.f};
                const uint16_t *w = p.b + (static_cast<uint64_t>(id) * p.outputs + n0 + g) * p.rank + 4 * t;
                const bool lo = n0 + g < p.outputs, hi = n0 + g + 8 < p.outputs;
#pragma unroll 4
                for (int32_t k = 0; k < steps; ++k) {  // 16 ranks: lane t has 4 t to 4 t + 3 of them
                    const bool in = 16 * k + 4 * t < p.rank;
                    const uint2 a = lo && in ? *reinterpret_cast<const uint2 *>(w + 16 * k) : make_uint2(0, 0);
                    const uint2 b = hi && in ? *reinterpret_cast<const uint2 *>(w + 8ull * p.rank + 16 * k) : make_uint2(0, 0);
                    const uint32_t m[4] = {a.x, b.x, a.y, b.y};
#pragma unroll
                    for (int term = 2; term >= 0; --term) {
                        const uint2 v = *reinterpret_cast<const uint2 *>(&h[term][g][8 * k + 2 * t]);
                        mma_bf16(s, m, v.x, v.y);
                    }
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int row = 2 * t + (k & 1);
                    if (row >= first && row < last) total[k] = s[k];
                }
            }
            first = last;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int32_t row = row0 + 2 * t + (k & 1), n = n0 + g + 8 * (k >> 1);
            if (row >= p.rows || n >= p.outputs) continue;
            const T *from = static_cast<const T *>(p.base) + row * p.base_stride + n;
            T *to = static_cast<T *>(p.out) + row * p.out_stride + n;
            if (adapter[2 * t + (k & 1)] >= 0) ad_store(to, ad_load(from) + total[k]);
            else *to = *from;
        }
    }
}

}  // namespace plamo

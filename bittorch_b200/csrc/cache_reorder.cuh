// Reordering of cached states after a step of beam search: row b * W + w of every cache tensor takes the rows of its
// parent, in place, for all tensors of all layers in one launch.
//
// A permutation with repeats cannot be done row by row in place, but at one place of the cache (tensor, head, slot,
// 16 bytes) it is W values in, W values out: a thread reads the parents' values of its place and then writes the beams
// that move.  Beams whose parent is themselves are neither read nor written for that; a source that several beams
// share comes from the cache the second time.  Bound by HBM: 16 tensors of 2 x 8 beams,
// slots 1024 to 4000, 2 GB moved in 341 to 363 us, 5.5 to 5.8 TB/s.
#pragma once

#include "cache_common.cuh"

namespace bt {

constexpr int RO_THREADS = 256;
constexpr int RO_TENSORS = 64;                                     // tensors of a launch: their addresses are its arguments

struct ReorderParams {
    uint8_t* base[RO_TENSORS];
    int64_t row[RO_TENSORS], head[RO_TENSORS], slot[RO_TENSORS];   // strides in bytes
    const int64_t* parents;
    Lengths lengths;
    int W, Hkv, S, start, units, lanes_log2;
    int blocks;                                                    // CTAs per tensor, group and head
};

// (Up to eight beams: at least 48 warps an SM, 16 x 4001 slots of 8 beams 361 us instead of 405 us.)
template <typename U, int WMAX>
__global__ void __launch_bounds__(RO_THREADS, WMAX <= 8 ? 6 : 1) reorder_cache_kernel(const __grid_constant__ ReorderParams p) {
    __shared__ int s_parent[WMAX];
    const int tid = threadIdx.x;
    const int at = static_cast<int>(blockIdx.x / static_cast<unsigned>(p.blocks)), blk = static_cast<int>(blockIdx.x) - at * p.blocks;
    const int b = at / p.Hkv, h = at - b * p.Hkv, t = blockIdx.y;
    pdl_launch_dependents();
    pdl_wait();
    if (tid < WMAX) {
        int64_t from = tid < p.W ? p.parents[static_cast<int64_t>(b) * p.W + tid] : tid;
        s_parent[tid] = from < 0 || from >= p.W ? tid : static_cast<int>(from);
    }
    __syncthreads();
    int parent[WMAX];
#pragma unroll
    for (int w = 0; w < WMAX; ++w) parent[w] = s_parent[w];
    const int end = p.lengths.at(b, p.S);
    uint8_t* base = p.base[t] + static_cast<int64_t>(b) * p.W * p.row[t] + h * p.head[t];
    const int64_t row = p.row[t], slot = p.slot[t];
    const int lanes = 1 << p.lanes_log2, rows = RO_THREADS >> p.lanes_log2;
    for (int64_t n = p.start + static_cast<int64_t>(blk) * rows + (tid >> p.lanes_log2); n < end; n += static_cast<int64_t>(p.blocks) * rows)
        for (int c = tid & (lanes - 1); c < p.units; c += lanes) {
            uint8_t* place = base + n * slot + c * sizeof(U);
            U v[WMAX];
#pragma unroll
            for (int w = 0; w < WMAX; ++w)
                if (parent[w] != w) v[w] = *reinterpret_cast<const U*>(place + parent[w] * row);
#pragma unroll
            for (int w = 0; w < WMAX; ++w)
                if (parent[w] != w) *reinterpret_cast<U*>(place + w * row) = v[w];
        }
}

template <typename U>
static int launch_reorder(ReorderParams p, int64_t tensors, int64_t B, int row_bytes, void* stream) {
    p.units = row_bytes / static_cast<int>(sizeof(U));
    const int64_t heads = B * p.Hkv;
    // enough CTAs for 16 rounds of every SM over the whole launch, no more than there are places
    int64_t blocks = ceil_div<int64_t>(static_cast<int64_t>(sm_count()) * 8 * 16, heads * tensors);
    p.lanes_log2 = row_lanes_log2(p.units);
    blocks = std::min<int64_t>(blocks, ceil_div<int64_t>(p.S - p.start, RO_THREADS >> p.lanes_log2));
    p.blocks = static_cast<int>(std::max<int64_t>(1, blocks));
    const dim3 grid(static_cast<unsigned>(heads * p.blocks), static_cast<unsigned>(tensors));
    if (p.W <= 4) return launch_early(reorder_cache_kernel<U, 4>, "reorder_cache_kernel", grid, RO_THREADS, 0, stream, p);
    if (p.W <= 8) return launch_early(reorder_cache_kernel<U, 8>, "reorder_cache_kernel", grid, RO_THREADS, 0, stream, p);
    if (p.W <= 16) return launch_early(reorder_cache_kernel<U, 16>, "reorder_cache_kernel", grid, RO_THREADS, 0, stream, p);
    return launch_early(reorder_cache_kernel<U, 32>, "reorder_cache_kernel", grid, RO_THREADS, 0, stream, p);
}

}  // namespace bt

extern "C" int bt_reorder_cache(void* const* tensors, int64_t count, int dtype, int64_t B, int64_t W, int64_t Hkv, int64_t S,
                                int64_t D, const int64_t* strides, const int64_t* parents, const void* lengths,
                                int lengths_i64, int64_t lengths_stride, int64_t start, void* stream) {
    using namespace bt;
    BT_REQUIRE(tensors && strides && parents && lengths, "bt_reorder_cache: NULL pointer");
    BT_REQUIRE(valid_dtype(dtype), "bt_reorder_cache: unknown dtype %d", dtype);
    BT_REQUIRE(count > 0 && B > 0 && W > 0 && Hkv > 0 && S > 0 && D > 0, "bt_reorder_cache: empty cache");
    BT_REQUIRE(start >= 0 && lengths_stride >= 0, "bt_reorder_cache: negative start or stride");
    BT_UNSUPPORTED_IF(W > BT_REORDER_MAX_BEAMS, "bt_reorder_cache: %lld beams exceed %d", (long long)W, BT_REORDER_MAX_BEAMS);
    const int64_t most = int64_t{1} << 30;
    BT_UNSUPPORTED_IF(S > most || D > 65536 || B > most / Hkv / 65536, "bt_reorder_cache: sizes too large");
    if (start >= S) return BT_OK;
    const int64_t es = static_cast<int64_t>(dtype_size(dtype));
    for (int64_t t = 0; t < count; ++t) BT_REQUIRE(tensors[t] != nullptr, "bt_reorder_cache: NULL pointer");
    for (int64_t t0 = 0; t0 < count; t0 += RO_TENSORS) {
        const int64_t some = std::min<int64_t>(RO_TENSORS, count - t0);
        ReorderParams p = {};
        uint64_t low = static_cast<uint64_t>(D * es);
        for (int64_t t = 0; t < some; ++t) {
            p.base[t] = static_cast<uint8_t*>(tensors[t0 + t]);
            p.row[t] = strides[3 * (t0 + t)] * es; p.head[t] = strides[3 * (t0 + t) + 1] * es; p.slot[t] = strides[3 * (t0 + t) + 2] * es;
            low |= reinterpret_cast<uintptr_t>(p.base[t]) | static_cast<uint64_t>(p.row[t]) | static_cast<uint64_t>(p.head[t]) |
                   static_cast<uint64_t>(p.slot[t]);
        }
        p.parents = parents;
        p.lengths = {lengths, lengths_stride, lengths_i64};
        p.W = static_cast<int>(W); p.Hkv = static_cast<int>(Hkv); p.S = static_cast<int>(S); p.start = static_cast<int>(start);
        const int row = static_cast<int>(D * es);
        int rc;
        if (low % 16 == 0) rc = launch_reorder<uint4>(p, some, B, row, stream);
        else if (low % 4 == 0) rc = launch_reorder<uint32_t>(p, some, B, row, stream);
        else rc = launch_reorder<uint16_t>(p, some, B, row, stream);
        if (rc != BT_OK) return rc;
    }
    return BT_OK;
}

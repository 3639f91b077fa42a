// Eviction from a key/value cache by accumulated attention weight, and the gather of the slots that stay.
//
// evict_select: one CTA per sequence and key/value head finds the k-th largest weight among the slots that may go, as
// a radix selection over the 32 ordered bits of a float (four passes of 8 bits, each a histogram in shared memory:
// integer counts, so the order of the atomics does not matter), then writes the kept slots in order: a slot's place is
// the number of kept slots before it, and of slots equal to the k-th weight the first ones stay.
//
// compact: rows are copied in units of 16 bytes (less where the alignment asks for it).  Between two caches every row
// is independent.  In place, entry j goes to slot first + j <= keep[j], so a CTA takes a narrow column of one head's
// cache (up to 64 bytes of every row) and walks the entries in blocks: all reads of a block, a barrier, then its
// writes.  Reads of later blocks only touch slots that earlier writes do not reach.
#pragma once

#include "cache_common.cuh"

namespace bt {

constexpr int EV_THREADS = 1024;

struct EvictParams {
    const float* mass;
    int64_t mass_sb, mass_sh;
    Lengths lengths;
    int S, Hkv, sinks, recent;
    int64_t budget;
    int64_t* keep;
    int64_t* counts;
};

// Larger floats have larger keys; -0 equals +0; a NaN is below everything.
__device__ __forceinline__ uint32_t ordered_key(float x) {
    if (x != x) return 0u;
    const uint32_t u = __float_as_uint(x == 0.0f ? 0.0f : x);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(EV_THREADS) evict_select_kernel(const EvictParams p) {
    __shared__ int s_hist[256];
    __shared__ int s_scan[256];
    __shared__ unsigned s_warp[EV_THREADS / 32];
    __shared__ uint32_t s_prefix;
    __shared__ int s_want;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int h = static_cast<int>(blockIdx.x % p.Hkv), b = static_cast<int>(blockIdx.x / p.Hkv);
    pdl_launch_dependents();
    pdl_wait();
    const int n = p.lengths.at(b, p.S);
    int64_t* keep = p.keep + static_cast<int64_t>(blockIdx.x) * p.budget;
    if (h == 0 && tid == 0) p.counts[b] = n < p.budget ? n : p.budget;
    if (n <= p.budget) {
        for (int64_t j = tid; j < p.budget; j += EV_THREADS) keep[j] = j < n ? j : -1;
        return;
    }
    const float* mass = p.mass + b * p.mass_sb + h * p.mass_sh;
    const int lo = p.sinks, hi = n - p.recent;                     // the slots that compete
    if (tid == 0) {
        s_prefix = 0;
        s_want = static_cast<int>(p.budget) - p.sinks - p.recent;
    }
    __syncthreads();
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (s_want == 0) break;                                    // nothing of the middle stays
        if (tid < 256) s_hist[tid] = 0;
        __syncthreads();
        const uint32_t prefix = s_prefix;
        for (int i = lo + tid; i < hi; i += EV_THREADS) {
            const uint32_t key = ordered_key(mass[i]);
            if (shift == 24 || ((key ^ prefix) >> (shift + 8)) == 0) atomicAdd(&s_hist[(key >> shift) & 255u], 1);
        }
        __syncthreads();
        // s_scan[i]: how many keys of this prefix have a digit >= i
        if (tid < 256) s_scan[tid] = s_hist[tid];
        for (int step = 1; step < 256; step <<= 1) {
            __syncthreads();
            const int add = tid + step < 256 ? s_scan[tid + step] : 0;
            __syncthreads();
            if (tid < 256) s_scan[tid] += add;
        }
        __syncthreads();
        const int want = s_want;
        __syncthreads();
        if (tid < 256 && s_scan[tid] >= want && s_scan[tid] - s_hist[tid] < want) {     // one digit holds the k-th key
            s_prefix = prefix | (static_cast<uint32_t>(tid) << shift);
            s_want = want - (s_scan[tid] - s_hist[tid]);
        }
        __syncthreads();
    }
    const uint32_t edge = s_prefix;                                // the k-th largest key; s_want slots equal to it stay
    const int equal_kept = s_want;
    const bool none = p.budget - p.sinks - p.recent == 0;
    int above = 0, equal = 0;                                      // kept / equal-to-the-edge slots before this block of slots
    for (int i0 = 0; i0 < n; i0 += EV_THREADS) {
        const int i = i0 + tid;
        bool stays = i < n && (i < lo || i >= hi), ties = false;
        if (i >= lo && i < hi && !none) {
            const uint32_t key = ordered_key(mass[i]);
            stays = key > edge;
            ties = key == edge;
        }
        const unsigned ms = __ballot_sync(0xffffffffu, stays), mt = __ballot_sync(0xffffffffu, ties), below = (1u << lane) - 1;
        if (lane == 0) s_warp[warp] = static_cast<unsigned>(__popc(ms)) | (static_cast<unsigned>(__popc(mt)) << 16);
        __syncthreads();
        unsigned before = 0, total = 0;                            // both counts stay below 2^16: a block is 1024 slots
        for (int w = 0; w < EV_THREADS / 32; ++w) {
            if (w == warp) before = total;
            total += s_warp[w];
        }
        const int a = above + static_cast<int>(before & 0xffffu) + __popc(ms & below);
        const int e = equal + static_cast<int>(before >> 16) + __popc(mt & below);
        if (stays || (ties && e < equal_kept)) keep[a + min(e, equal_kept)] = i;
        above += static_cast<int>(total & 0xffffu);
        equal += static_cast<int>(total >> 16);
        __syncthreads();
    }
}

struct CompactParams {
    const uint8_t* src[2];
    uint8_t* dst[2];
    int64_t sb[2], sh[2], ss[2], db[2], dh[2], ds[2];              // strides in bytes
    const int64_t* keep;
    int64_t keep_sb, keep_sh;
    const int64_t* counts;
    const int64_t* first;
    const float* mass;
    float* mass_out;
    int64_t msb, msh, mdb, mdh;                                    // in elements
    int B, Hkv, S, S_out, units;                                   // units of a row
    int64_t n;
    int blocks;                                                    // gather: CTAs per sequence, head and tensor
};

__device__ __forceinline__ int64_t compact_count(const CompactParams& p, int b) {
    const int64_t c = p.counts[b];
    return c < 0 ? 0 : c > p.n ? p.n : c;
}

constexpr int CG_THREADS = 256;
constexpr int CG_UNITS = 4;                                        // copies in flight per thread

// Between two caches: blockIdx.y = tensor (0, 1) or the mass (2).
template <typename U>
__global__ void __launch_bounds__(CG_THREADS) compact_gather_kernel(const CompactParams p) {
    const int tid = threadIdx.x;
    const int64_t bh = blockIdx.x / p.blocks;
    const int blk = static_cast<int>(blockIdx.x % p.blocks);
    const int h = static_cast<int>(bh % p.Hkv), b = static_cast<int>(bh / p.Hkv);
    pdl_launch_dependents();
    pdl_wait();
    const int64_t count = compact_count(p, b), first = p.first ? p.first[b] : 0;
    const int64_t* keep = p.keep + b * p.keep_sb + h * p.keep_sh;
    const int which = blockIdx.y;
    if (which == 2) {
        const float* m = p.mass + b * p.msb + h * p.msh;
        float* out = p.mass_out + b * p.mdb + h * p.mdh;
        for (int64_t j = blk * static_cast<int64_t>(CG_THREADS) + tid; j < p.S_out; j += static_cast<int64_t>(p.blocks) * CG_THREADS) {
            if (j < first) continue;
            const int64_t from = j - first < count ? keep[j - first] : -1;
            if (j - first >= count) out[j] = 0.0f;
            else if (from >= 0 && from < p.S) out[j] = m[from];
        }
        return;
    }
    const uint8_t* src = p.src[which] + b * p.sb[which] + h * p.sh[which];
    uint8_t* dst = p.dst[which] + b * p.db[which] + h * p.dh[which];
    const int64_t total = count * p.units, step = static_cast<int64_t>(p.blocks) * CG_THREADS;
    for (int64_t u0 = blk * static_cast<int64_t>(CG_THREADS) + tid; u0 < total; u0 += step * CG_UNITS) {
        U v[CG_UNITS];
        U* to[CG_UNITS];
#pragma unroll
        for (int i = 0; i < CG_UNITS; ++i) {
            const int64_t u = u0 + i * step;
            to[i] = nullptr;
            if (u >= total) continue;
            const int64_t j = u / p.units, c = u - j * p.units, from = keep[j], at = first + j;
            if (from < 0 || from >= p.S || at < 0 || at >= p.S_out) continue;
            v[i] = *reinterpret_cast<const U*>(src + from * p.ss[which] + c * sizeof(U));
            to[i] = reinterpret_cast<U*>(dst + at * p.ds[which] + c * sizeof(U));
        }
#pragma unroll
        for (int i = 0; i < CG_UNITS; ++i)
            if (to[i] != nullptr) *to[i] = v[i];
    }
}

constexpr int CI_THREADS = 512;
constexpr int CI_ROWS = 8;                                         // rows staged per thread and block
constexpr int CI_COLS = 4;                                         // units of a column

// In place: blockIdx.x = sequence, head and column, blockIdx.y = tensor (0, 1) or the mass (2, one column of one unit).
template <typename U>
__device__ __forceinline__ void compact_column(uint8_t* base, int64_t stride, int c0, int cols, const int64_t* keep, int64_t count,
                                               int64_t first, int S) {
    const int tid = threadIdx.x;
    const int lanes = cols <= 1 ? 1 : cols <= 2 ? 2 : 4;           // threads of a row
    const int col = tid % lanes, per = CI_THREADS / lanes;         // rows per pass
    U v[CI_ROWS];
    int64_t at[CI_ROWS];
    for (int64_t j0 = 0; j0 < count; j0 += static_cast<int64_t>(per) * CI_ROWS) {
#pragma unroll
        for (int i = 0; i < CI_ROWS; ++i) {
            const int64_t j = j0 + static_cast<int64_t>(i) * per + tid / lanes;
            at[i] = -1;
            if (j >= count || col >= cols) continue;
            const int64_t from = keep[j], to = first + j;
            if (from < 0 || from >= S || to < 0 || to >= S || from == to) continue;
            v[i] = *reinterpret_cast<const U*>(base + from * stride + (c0 + col) * sizeof(U));
            at[i] = to;
        }
        __syncthreads();                                           // every read of this block, before its writes
#pragma unroll
        for (int i = 0; i < CI_ROWS; ++i)
            if (at[i] >= 0) *reinterpret_cast<U*>(base + at[i] * stride + (c0 + col) * sizeof(U)) = v[i];
    }
}

template <typename U>
__global__ void __launch_bounds__(CI_THREADS) compact_inplace_kernel(const CompactParams p) {
    const int columns = (p.units + CI_COLS - 1) / CI_COLS;
    const int64_t bh = blockIdx.x / columns;
    const int c0 = static_cast<int>(blockIdx.x % columns) * CI_COLS;
    const int h = static_cast<int>(bh % p.Hkv), b = static_cast<int>(bh / p.Hkv), which = blockIdx.y;
    if (which == 2 && c0 != 0) return;
    pdl_launch_dependents();
    pdl_wait();
    const int64_t count = compact_count(p, b), first = p.first ? p.first[b] : 0;
    const int64_t* keep = p.keep + b * p.keep_sb + h * p.keep_sh;
    if (which < 2) {
        compact_column<U>(p.dst[which] + b * p.db[which] + h * p.dh[which], p.ds[which], c0, min(CI_COLS, p.units - c0), keep, count, first, p.S);
        return;
    }
    float* m = p.mass_out + b * p.mdb + h * p.mdh;
    compact_column<uint32_t>(reinterpret_cast<uint8_t*>(m), 4, 0, 1, keep, count, first, p.S);
    __syncthreads();
    const int64_t tail = first + count < 0 ? 0 : first + count;
    for (int64_t j = tail + threadIdx.x; j < p.S; j += CI_THREADS) m[j] = 0.0f;
}

template <typename U>
static int launch_compact(CompactParams p, bool in_place, int row_bytes, void* stream) {
    p.units = row_bytes / static_cast<int>(sizeof(U));
    const int64_t heads = static_cast<int64_t>(p.B) * p.Hkv;
    const unsigned kinds = p.mass ? 3 : 2;
    if (in_place)
        return launch_early(compact_inplace_kernel<U>, "compact_inplace_kernel",
                            dim3(static_cast<unsigned>(heads * ceil_div(p.units, CI_COLS)), kinds), CI_THREADS, 0, stream, p);
    // as many CTAs as keep every SM at eight, each with at least one full round of copies
    int64_t blocks = ceil_div<int64_t>(p.n * p.units, CG_THREADS * CG_UNITS);
    blocks = std::min<int64_t>(blocks, std::max<int64_t>(1, ceil_div<int64_t>(static_cast<int64_t>(sm_count()) * 8, heads * 2)));
    p.blocks = static_cast<int>(std::max<int64_t>(1, blocks));
    return launch_early(compact_gather_kernel<U>, "compact_gather_kernel", dim3(static_cast<unsigned>(heads * p.blocks), kinds), CG_THREADS, 0, stream, p);
}

}  // namespace bt

extern "C" int bt_evict_select(const float* mass, int64_t mass_sb, int64_t mass_sh, int64_t B, int64_t Hkv, int64_t S,
                               const void* lengths, int lengths_i64, int64_t lengths_stride, int64_t budget, int64_t sinks,
                               int64_t recent, int64_t* keep, int64_t* counts, void* stream) {
    using namespace bt;
    BT_REQUIRE(mass && lengths && keep && counts, "bt_evict_select: NULL pointer");
    BT_REQUIRE(B > 0 && Hkv > 0 && S > 0, "bt_evict_select: empty cache");
    BT_REQUIRE(budget > 0 && sinks >= 0 && recent >= 0 && sinks <= budget && recent <= budget - sinks,
               "bt_evict_select: budget %lld must be positive and hold %lld sinks and %lld recent slots", (long long)budget,
               (long long)sinks, (long long)recent);
    BT_REQUIRE(lengths_stride >= 0, "bt_evict_select: negative stride");
    BT_UNSUPPORTED_IF(S > (int64_t{1} << 30) || B > (int64_t{1} << 30) / Hkv || budget > (int64_t{1} << 30), "bt_evict_select: sizes too large");
    EvictParams p = {};
    p.mass = mass; p.mass_sb = mass_sb; p.mass_sh = mass_sh;
    p.lengths = {lengths, lengths_stride, lengths_i64};
    p.S = static_cast<int>(S); p.Hkv = static_cast<int>(Hkv);
    p.sinks = static_cast<int>(sinks); p.recent = static_cast<int>(recent);
    p.budget = budget; p.keep = keep; p.counts = counts;
    return launch_early(evict_select_kernel, "evict_select_kernel", dim3(static_cast<unsigned>(B * Hkv)), EV_THREADS, 0, stream, p);
}

extern "C" int bt_compact_cache(const void* k, const void* v, void* k_out, void* v_out, int dtype, int64_t B, int64_t Hkv,
                                int64_t S, int64_t S_out, int64_t D, const int64_t* strides, const int64_t* keep,
                                int64_t keep_sb, int64_t keep_sh, int64_t n, const int64_t* counts, const int64_t* first,
                                const float* mass, float* mass_out, const int64_t* mass_strides, void* stream) {
    using namespace bt;
    BT_REQUIRE(k && v && k_out && v_out && strides && keep && counts, "bt_compact_cache: NULL pointer");
    BT_REQUIRE(valid_dtype(dtype), "bt_compact_cache: unknown dtype %d", dtype);
    BT_REQUIRE(B > 0 && Hkv > 0 && S > 0 && S_out > 0 && D > 0 && n > 0, "bt_compact_cache: empty cache");
    BT_REQUIRE((mass != nullptr) == (mass_out != nullptr) && (mass == nullptr || mass_strides != nullptr),
               "bt_compact_cache: mass, mass_out and mass_strides come together");
    const bool in_place = k == k_out;
    BT_REQUIRE(in_place == (v == v_out) && (mass == nullptr || in_place == (mass == mass_out)),
               "bt_compact_cache: keys, values and mass are all compacted in place, or none");
    BT_REQUIRE(!in_place || S == S_out, "bt_compact_cache: in place, both caches have the same slots");
    if (in_place) {
        for (int i = 0; i < 6; ++i) BT_REQUIRE(strides[i] == strides[6 + i], "bt_compact_cache: in place, both caches have the same strides");
        BT_REQUIRE(mass == nullptr || (mass_strides[0] == mass_strides[2] && mass_strides[1] == mass_strides[3]),
                   "bt_compact_cache: in place, both masses have the same strides");
    }
    const int64_t most = int64_t{1} << 30;
    BT_UNSUPPORTED_IF(S > most || S_out > most || n > most || D > 65536 || B > most / Hkv / 16384, "bt_compact_cache: sizes too large");
    const int64_t es = static_cast<int64_t>(dtype_size(dtype));
    CompactParams p = {};
    p.src[0] = static_cast<const uint8_t*>(k); p.src[1] = static_cast<const uint8_t*>(v);
    p.dst[0] = static_cast<uint8_t*>(k_out); p.dst[1] = static_cast<uint8_t*>(v_out);
    uint64_t low = static_cast<uint64_t>(D * es);                  // what every address is a multiple of
    for (int t = 0; t < 2; ++t) {
        p.sb[t] = strides[3 * t] * es; p.sh[t] = strides[3 * t + 1] * es; p.ss[t] = strides[3 * t + 2] * es;
        p.db[t] = strides[6 + 3 * t] * es; p.dh[t] = strides[6 + 3 * t + 1] * es; p.ds[t] = strides[6 + 3 * t + 2] * es;
        for (const int64_t s : {p.sb[t], p.sh[t], p.ss[t], p.db[t], p.dh[t], p.ds[t]}) low |= static_cast<uint64_t>(s);
        low |= reinterpret_cast<uintptr_t>(p.src[t]) | reinterpret_cast<uintptr_t>(p.dst[t]);
    }
    p.keep = keep; p.keep_sb = keep_sb; p.keep_sh = keep_sh; p.counts = counts; p.first = first;
    p.mass = mass; p.mass_out = mass_out;
    if (mass) { p.msb = mass_strides[0]; p.msh = mass_strides[1]; p.mdb = mass_strides[2]; p.mdh = mass_strides[3]; }
    p.B = static_cast<int>(B); p.Hkv = static_cast<int>(Hkv); p.S = static_cast<int>(S); p.S_out = static_cast<int>(S_out); p.n = n;
    const int row = static_cast<int>(D * es);
    if (low % 16 == 0) return launch_compact<uint4>(p, in_place, row, stream);
    if (low % 4 == 0) return launch_compact<uint32_t>(p, in_place, row, stream);
    return launch_compact<uint16_t>(p, in_place, row, stream);
}

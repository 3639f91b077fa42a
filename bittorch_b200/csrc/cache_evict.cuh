// Eviction from a key/value cache by accumulated attention weight, and the gather of the slots that stay.
//
// evict_select: one CTA per sequence and key/value head finds the k-th largest weight among the slots that may go, as
// a radix selection over the 32 ordered bits of a float (up to four passes of 8 bits), then writes the kept slots in
// order: a slot's place is the number of kept slots before it, and of slots equal to the k-th weight the first ones
// stay.  Weights have few exponents, so most slots of a warp count into the same digit: every lane has a column of the
// histogram to itself, and no two lanes ever meet in a bank.  Counts are integers, so the order of the atomics does
// not matter.  A thread holds neighbouring slots, in registers for the whole selection unless the cache is longer than
// a CTA's registers.  Bound by the instructions and barriers of four passes of one CTA, not by the 4 bytes a slot: 8 heads of
// 16387 slots 14 us, 256 heads of 8192 slots 24 us.
//
// compact: rows are copied in pieces of 16 bytes (less where the alignment asks for it), a row by neighbouring lanes.
// Between two caches every row is independent.  In place, entry j goes to slot first + j <= keep[j], so a CTA takes a
// narrow column of one head's cache (up to 64 bytes of every row) and walks the entries in blocks: all reads of a
// block, a barrier, then its writes.  Reads of later blocks only touch slots that earlier writes do not reach.  Bound by HBM:
// between two caches 32 x 8 heads x 4096 rows of 256 bytes 168 us, 6.4 TB/s.
#pragma once

#include "cache_common.cuh"

namespace bt {

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

// IPT: neighbouring slots of a thread.
template <int EV_THREADS, int IPT>
__global__ void __launch_bounds__(EV_THREADS) evict_select_kernel(const EvictParams p) {
    constexpr int BLOCK = EV_THREADS * IPT;
    __shared__ int s_hist[257 * 32];                               // [digit][lane]; the last row takes the keys with another prefix
    __shared__ int s_digit[256];
    __shared__ unsigned s_warp[EV_THREADS / 32];
    __shared__ uint32_t s_prefix;
    __shared__ int s_want, s_left;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int b = static_cast<int>(blockIdx.x / static_cast<unsigned>(p.Hkv)), h = static_cast<int>(blockIdx.x) - b * p.Hkv;
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
    const int blocks = (n + BLOCK - 1) / BLOCK;
    const bool vec = aligned(mass, 16);
    uint32_t key[IPT];
    auto load = [&](int i0) {
        if (vec && i0 + IPT <= n) {
#pragma unroll
            for (int i = 0; i < IPT; i += 4) {
                const float4 x = *reinterpret_cast<const float4*>(mass + i0 + i);
                key[i] = ordered_key(x.x); key[i + 1] = ordered_key(x.y); key[i + 2] = ordered_key(x.z); key[i + 3] = ordered_key(x.w);
            }
        } else {
#pragma unroll
            for (int i = 0; i < IPT; ++i) key[i] = i0 + i < n ? ordered_key(mass[i0 + i]) : 0;
        }
    };
    // Slots that do not compete count as the lowest key there is: they never stand above another, and where the k-th key
    // is that low (a NaN's), the last loop leaves them out.
    auto competitors = [&](int i0) {
        load(i0);
        if (i0 < lo || i0 + IPT > hi) {
#pragma unroll
            for (int i = 0; i < IPT; ++i)
                if (i0 + i < lo || i0 + i >= hi) key[i] = 0;
        }
    };
    if (blocks == 1) competitors(tid * IPT);
    uint32_t prefix = 0;                                           // the digits of the k-th largest key that are known
    int want = static_cast<int>(p.budget) - p.sinks - p.recent;    // it is the want-th largest of those with this prefix
    int shift = 32;                                                // bits not yet known
#pragma unroll 1                                                   // four copies of the code cost more to fetch than they save
    while (want > 0 && shift > 0) {
        shift -= 8;
        for (int i = tid; i < 256 * 32; i += EV_THREADS) s_hist[i] = 0;
        __syncthreads();
        for (int blk = 0; blk < blocks; ++blk) {
            if (blocks > 1) competitors(blk * BLOCK + tid * IPT);
#pragma unroll
            for (int i = 0; i < IPT; ++i) atomicAdd(&s_hist[min((key[i] ^ prefix) >> shift, 256u) * 32 + lane], 1);
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 256 / (EV_THREADS / 32); ++i) {
            const int d = warp * (256 / (EV_THREADS / 32)) + i, sum = warp_add(s_hist[d * 32 + lane]);
            if (lane == 0) s_digit[d] = sum;
        }
        __syncthreads();
        if (warp == 0) {                                           // eight digits per lane, the largest in lane 31
            int mine = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) mine += s_digit[lane * 8 + i];
            int above = mine;                                      // inclusive, from the top
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_down_sync(0xffffffffu, above, o);
                if (lane + o < 32) above += x;
            }
            above -= mine;
            if (above < want && above + mine >= want) {            // one lane
                int d = lane * 8 + 7;
                while (above + s_digit[d] < want) above += s_digit[d--];
                s_prefix = prefix | (static_cast<uint32_t>(d) << shift);
                s_want = want - above;
                s_left = s_digit[d];
            }
        }
        __syncthreads();
        prefix = s_prefix;
        want = s_want;
        if (s_left == want) break;                                 // all of them stay: the lower bits do not matter
    }
    const int equal_kept = want;                                   // so many of those that tie with the prefix stay, the first ones
    const bool none = static_cast<int>(p.budget) == p.sinks + p.recent;
    const uint32_t edge = shift < 32 ? prefix >> shift : 0;
    shift &= 31;                                                   // nothing competes where it is 32
    int above = 0, equal = 0;                                      // kept / tying slots before this block
    for (int blk = 0; blk < blocks; ++blk) {
        const int i0 = blk * BLOCK + tid * IPT;
        if (blocks > 1) competitors(i0);
        unsigned stays = 0, ties = 0;                              // a bit per slot
#pragma unroll
        for (int i = 0; i < IPT; ++i) {
            if ((key[i] >> shift) > edge) stays |= 1u << i;
            if ((key[i] >> shift) == edge) ties |= 1u << i;
        }
        // bits of the slots below x among this thread's
        auto below = [&](int x) { return x <= i0 ? 0u : x >= i0 + IPT ? ~0u : (1u << (x - i0)) - 1u; };
        const unsigned compete = below(hi) & ~below(lo), exist = below(n) & (IPT == 32 ? ~0u : (1u << (IPT & 31)) - 1u);
        stays = none ? exist & ~compete : ((stays & compete) | ~compete) & exist;
        ties = none ? 0u : ties & compete & exist;
        const unsigned mine = static_cast<unsigned>(__popc(stays)) | (static_cast<unsigned>(__popc(ties)) << 16);     // a block holds at most 2^15 of each
        unsigned upto = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        if (lane == 31) s_warp[warp] = upto;
        __syncthreads();
        unsigned all = lane < EV_THREADS / 32 ? s_warp[lane] : 0u;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned x = __shfl_up_sync(0xffffffffu, all, o);
            if (lane >= o) all += x;
        }
        const unsigned before = (warp > 0 ? __shfl_sync(0xffffffffu, all, warp > 0 ? warp - 1 : 0) : 0u) + upto - mine;
        const unsigned total = __shfl_sync(0xffffffffu, all, 31);
        int a = above + static_cast<int>(before & 0xffffu), e = equal + static_cast<int>(before >> 16);
        for (unsigned left = stays | ties; left != 0; left &= left - 1) {
            const int i = __ffs(left) - 1;
            const bool tie = (ties >> i) & 1u;
            if (!tie || e < equal_kept) keep[a + (e < equal_kept ? e : equal_kept)] = i0 + i;
            a += !tie;
            e += tie;
        }
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
    int B, Hkv, S, S_out, units, lanes_log2;                       // units of a row, threads of a row
    int64_t n;
    int blocks;                                                    // gather: CTAs per sequence, head and tensor
};

__device__ __forceinline__ int64_t compact_count(const CompactParams& p, int b) {
    const int64_t c = p.counts[b];
    return c < 0 ? 0 : c > p.n ? p.n : c;
}

constexpr int CG_THREADS = 256;
constexpr int CG_ROWS = 4;                                         // rows in flight per thread

// Between two caches: blockIdx.y = tensor (0, 1) or the mass (2).
template <typename U>
__global__ void __launch_bounds__(CG_THREADS) compact_gather_kernel(const CompactParams p) {
    const int tid = threadIdx.x;
    const int bh = static_cast<int>(blockIdx.x / static_cast<unsigned>(p.blocks)), blk = static_cast<int>(blockIdx.x) - bh * p.blocks;
    const int b = bh / p.Hkv, h = bh - b * p.Hkv, which = blockIdx.y;
    pdl_launch_dependents();
    pdl_wait();
    const int64_t count = compact_count(p, b), first = p.first ? p.first[b] : 0;
    const int64_t* keep = p.keep + b * p.keep_sb + h * p.keep_sh;
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
    const int64_t ss = p.ss[which], ds = p.ds[which];
    const int rows = CG_THREADS >> p.lanes_log2, c0 = tid & ((1 << p.lanes_log2) - 1);
    for (int64_t j0 = static_cast<int64_t>(blk) * rows * CG_ROWS + (tid >> p.lanes_log2); j0 < count; j0 += static_cast<int64_t>(p.blocks) * rows * CG_ROWS) {
        int64_t from[CG_ROWS];
#pragma unroll
        for (int i = 0; i < CG_ROWS; ++i) {
            const int64_t j = j0 + i * rows, at = first + j;
            from[i] = j < count && at >= 0 && at < p.S_out ? keep[j] : -1;
            if (from[i] >= p.S) from[i] = -1;
        }
        for (int c = c0; c < p.units; c += 1 << p.lanes_log2) {
            U v[CG_ROWS];
#pragma unroll
            for (int i = 0; i < CG_ROWS; ++i)
                if (from[i] >= 0) v[i] = *reinterpret_cast<const U*>(src + from[i] * ss + c * sizeof(U));
#pragma unroll
            for (int i = 0; i < CG_ROWS; ++i)
                if (from[i] >= 0) *reinterpret_cast<U*>(dst + (first + j0 + i * rows) * ds + c * sizeof(U)) = v[i];
        }
    }
}

// A step is a read of the entry, a read of the row, a barrier and a write, so what counts is the warps that are under way:
// 32 sequences of 8 heads, 4096 of 8192 rows of 256 bytes in place: 512 threads with 8 rows each 429 us, 1024 with 8 303 us,
// 1024 with 4 236 us, with 2 209 us (5.1 TB/s).  Columns of 32 bytes take 268 us there, of 128 bytes 232 us and twice as long
// as these for few heads.
constexpr int CI_THREADS = 1024;
constexpr int CI_ROWS = 2;                                         // rows staged per thread and block
constexpr int CI_COLS = 4;                                         // units of a column

// In place: blockIdx.x = sequence, head and column, blockIdx.y = tensor (0, 1) or the mass (2, one column of one unit).
template <typename U>
__device__ __forceinline__ void compact_column(uint8_t* base, int64_t stride, int c0, int cols, const int64_t* keep, int64_t count,
                                               int64_t first, int S) {
    const int tid = threadIdx.x;
    const int lanes = cols <= 1 ? 1 : cols <= 2 ? 2 : 4;           // threads of a row
    const int col = tid % lanes, per = CI_THREADS / lanes;         // rows per pass
    U v[CI_ROWS];
    int at[CI_ROWS];
    for (int64_t j0 = 0; j0 < count; j0 += static_cast<int64_t>(per) * CI_ROWS) {
#pragma unroll
        for (int i = 0; i < CI_ROWS; ++i) {
            const int64_t j = j0 + static_cast<int64_t>(i) * per + tid / lanes;
            at[i] = -1;
            if (j >= count || col >= cols) continue;
            const int64_t from = keep[j], to = first + j;
            if (from < 0 || from >= S || to < 0 || to >= S || from == to) continue;
            v[i] = *reinterpret_cast<const U*>(base + from * stride + (c0 + col) * sizeof(U));
            at[i] = static_cast<int>(to);
        }
        __syncthreads();                                           // every read of this block, before its writes
#pragma unroll
        for (int i = 0; i < CI_ROWS; ++i)
            if (at[i] >= 0) *reinterpret_cast<U*>(base + at[i] * stride + (c0 + col) * sizeof(U)) = v[i];
    }
}

template <typename U>
__global__ void __launch_bounds__(CI_THREADS, 2) compact_inplace_kernel(const CompactParams p) {
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
    // up to four waves of eight CTAs per SM, each with at least one full round of copies
    p.lanes_log2 = row_lanes_log2(p.units);
    int64_t blocks = ceil_div<int64_t>(p.n, (CG_THREADS >> p.lanes_log2) * CG_ROWS);
    blocks = std::min<int64_t>(blocks, std::max<int64_t>(1, ceil_div<int64_t>(static_cast<int64_t>(sm_count()) * 32, heads * 2)));
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
    const dim3 grid(static_cast<unsigned>(B * Hkv));
    // The shortest run of slots per thread that holds the cache in registers; a longer cache is read again in every pass.
    // Short caches: a CTA of 1024 threads is the fastest for one head, many heads go faster through CTAs of 256.
    if (S <= 4096 && grid.x <= static_cast<unsigned>(sm_count())) return launch_early(evict_select_kernel<1024, 4>, "evict_select_kernel", grid, 1024, 0, stream, p);
    if (S <= 4096) return launch_early(evict_select_kernel<256, 16>, "evict_select_kernel", grid, 256, 0, stream, p);
    if (S <= 16384) return launch_early(evict_select_kernel<1024, 16>, "evict_select_kernel", grid, 1024, 0, stream, p);
    return launch_early(evict_select_kernel<1024, 32>, "evict_select_kernel", grid, 1024, 0, stream, p);
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

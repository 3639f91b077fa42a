// The 16-bit kernel of bt_tree_attention for many rows per key/value head (token trees, grouped heads): both products on the
// 5th-generation tensor cores, scores, weights and output in tensor memory.
//
// The rows of a head (query heads x new tokens) are cut into tiles of 128, one thread per row.  A CTA works on two tiles
// of one sequence at a time ("streams"): while the tensor cores make one tile's scores, the other tile's threads turn
// theirs into weights.  Tiles of the same head share the keys and values that TMA brings in; the last tile of a head and
// the first of the next go together too, each with its own.  A stream's step, for 128 slots:
//   S = Q K^T   tcgen05.mma, both operands in shared memory, 128 columns of TMEM that the streams use in turn
//   weights     a row's 128 scores in its thread's registers; the reference point of the exponentials moves only when a
//               score exceeds it by 2^8 (the sums stay far from overflow, and the output is almost never rescaled);
//               the weights, rounded to the cache's type (relative 2^-8 / 2^-11 at most; in fp16 those
//               below 2^-14 by up to 2^-25), go to the stream's place in TMEM
//   O += P V    tcgen05.mma with P from TMEM, V as it lies in the cache (its columns contiguous)
//
// Work is dealt out in blocks of 128 slots: the blocks of all pairs of tiles of all sequences form one line, and every
// CTA (one per SM) takes an equal piece of it, so that ragged lengths cost nothing.  A CTA writes a pair that it has
// whole straight to the output; of the others, the first and the last of its piece, it leaves sums, maxima and
// unnormalised output in its two places of the workspace, and attn_tc_join_kernel adds the pieces of a pair up.
//
// New tokens: scores that a row does not see are masked; values in slots past the end are overwritten with zeros before
// they are multiplied, and so are infinities and NaN among the new tokens' values, which are added at the end to
// the rows that see them.
//
// 8 trees of 61 nodes over 4099 to 8190 slots, 64 heads over 8, head size 128, fp16: 126 us, 787 TFLOP/s.  A block of two tiles
// takes about 3350 cycles; its four products need 2048, the 32768 exponentials of the two streams as many (16 a cycle).
// Bound by latency: the tensor pipe is busy 50 % of the time, the exponentials' pipe 50 %, 37 % of the issue slots are used, and
// in 63 % of the cycles no warp of a scheduler can issue (11 warps an SM, one thread a row; the streams pass one buffer of
// scores between them, so that neither's products run while both wait).  Short calls: by 16 to 19 thousand cycles at the
// end of a pair (output through shared memory, the pieces' join).
#pragma once

#include "cache_attention_stream.cuh"
#include "gemm_tcgen05.cuh"

namespace bt {

constexpr int TC_ROWS = 128;                                       // rows of a tile
constexpr int TC_KEYS = 128;                                       // slots of a block
constexpr int TC_SLOTS = 4;                                        // ring of key / value tiles
constexpr int TC_THREADS = 352;                                    // warps: 0 TMA, 1 scores, 10 outputs, 2-5 and 6-9 the streams
constexpr int TC_COLS = 512;                                       // TMEM: scores at 0, weights at 128 and 192, outputs at 256 and 384
constexpr int TC_WEIGHTS = 128, TC_OUTPUT = 256;
// What finishing a pair costs, in blocks: counted when work is dealt out (8 x 61 nodes over up to 8190 slots: 0 138 us, 4 130 us,
// 8 126 us, 13 129 us).
constexpr int TC_END = 8;
constexpr float TC_LAZY = 8.0f;                                    // how far (in powers of 2) a score may exceed the reference point

template <int D> __host__ __device__ constexpr int tc_tile_bytes() { return TC_KEYS * D * 2; }
constexpr int TC_NODES = 128;                                      // trees up to this many nodes have their rows as bits in shared memory
constexpr int TC_STAGE = 32 * 64;                                  // bytes of a warp's staging buffer: 32 rows x 32 columns
template <int D> constexpr size_t tc_smem() {
    return 1024 + static_cast<size_t>(2 + TC_SLOTS) * tc_tile_bytes<D>() + 1024 /*barriers*/ + 2 * TC_NODES * 16 + 8 * TC_STAGE;
}

struct AttnTcParams {
    AttnParams a;
    int tiles;                                                     // of a head
    int items;                                                     // Hkv * tiles of a sequence
    int pairs;                                                     // pairs of tiles of a sequence
    float scale2;                                                  // scale * log2(e), not negative
    float* part_o;                                                 // [CTA][2][stream][D][128]: rows vary fastest, as the threads do
    float2* part_ml;                                               // [CTA][2][stream][128]
    int give_up;                                                   // self-test: every CTA's TMA role leaves after so many tiles, as if a wait had run out; -1: never
};

// A piece of one pair's line of blocks
struct TcPiece {
    int b, pair, k0, k1, blocks, len, end;
    int streams, own;                                              // tiles of the pair; own: they are of two heads, each with its keys and values
    uint32_t first;                                                // the piece's first tile in the ring's sequence
};
__device__ __forceinline__ int tc_blocks(const AttnTcParams& p, int b) { return (attn_end(p.a, attn_len(p.a, b)) + TC_KEYS - 1) / TC_KEYS; }

// The length of the whole line, in which every pair's blocks are followed by TC_END places without work, and where position
// `pos` lies on it.  Run by whole warps; every lane gets the result.
__device__ __forceinline__ int64_t tc_total(const AttnTcParams& p) {
    const int lane = threadIdx.x & 31;
    int64_t sum = 0;
    for (int b = lane; b < p.a.B; b += 32) sum += tc_blocks(p, b) + TC_END;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    return sum * p.pairs;
}
__device__ __forceinline__ void tc_locate(const AttnTcParams& p, int64_t pos, int& b, int& pair, int& block) {
    const int lane = threadIdx.x & 31;
    int64_t before = 0;
    b = p.a.B, pair = 0, block = 0;
    for (int b0 = 0; b0 < p.a.B; b0 += 32) {
        const int n = b0 + lane < p.a.B ? tc_blocks(p, b0 + lane) + TC_END : 0;
        int64_t upto = static_cast<int64_t>(n) * p.pairs;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t x = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += x;
        }
        const unsigned past = __ballot_sync(0xffffffffu, before + upto > pos);
        if (past != 0) {
            const int hit = __ffs(past) - 1;
            const int blocks = __shfl_sync(0xffffffffu, n, hit);
            const int64_t start = before + __shfl_sync(0xffffffffu, upto, hit) - static_cast<int64_t>(blocks) * p.pairs;
            b = b0 + hit;
            pair = static_cast<int>((pos - start) / blocks);
            block = static_cast<int>((pos - start) - static_cast<int64_t>(pair) * blocks);
            return;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
}
// Where CTA i's piece of the line begins
struct TcCuts {
    int64_t each;
    unsigned rest, ctas;
    __device__ __forceinline__ TcCuts(int64_t total, unsigned n) : each(total / n), rest(static_cast<unsigned>(total % n)), ctas(n) {}
    __device__ __forceinline__ int64_t at(unsigned i) const { return each * i + rest * i / ctas; }
};

// The place of the values of block j of n, for stream x, in the sequence of a piece's tiles (as the TMA warp brings them)
__device__ __forceinline__ uint32_t tc_value_tile(bool own, int n, int j, int x) {
    const int ahead = min(j, max(n - 2, 0));                       // keys of blocks j + 1 that came before
    if (!own) return min(2, n) + j + ahead;
    return 2 + (n > 1) + 2 * j + min(j, n - 1) + ahead + (x ? 1 + (j + 1 < n) : 0);
}

// The same for the keys
__device__ __forceinline__ uint32_t tc_key_tile(bool own, int n, int j, int x) {
    if (!own) return j < 2 ? j : tc_value_tile(own, n, j - 2, 0) + 1;
    if (x == 1) return j == 0 ? 1 : tc_value_tile(own, n, j - 1, 0) + 1;
    return j < 2 ? 2 * j : tc_value_tile(own, n, j - 2, 1) + 1;
}

struct TcWalk {
    int b, pair, block;
    int64_t left;
    uint32_t tiles;                                                // of keys and values so far
    __device__ __forceinline__ bool next(const AttnTcParams& p, TcPiece& c) {
        while (true) {
            if (left <= 0 || b >= p.a.B) return false;
            c.len = attn_len(p.a, b);
            c.end = attn_end(p.a, c.len);
            c.blocks = (c.end + TC_KEYS - 1) / TC_KEYS;
            if (block < c.blocks) break;
            left -= c.blocks + TC_END - block;                     // nothing is left of this pair
            block = 0;
            if (++pair == p.pairs) pair = 0, ++b;
        }
        c.b = b; c.pair = pair; c.k0 = block;
        c.k1 = static_cast<int>(c.blocks - block < left ? c.blocks : block + left);
        const int item = pair * 2;
        c.streams = item + 1 < p.items ? 2 : 1;
        c.own = c.streams == 2 && item / p.tiles != (item + 1) / p.tiles;
        c.first = tiles;
        tiles += (c.own ? 4 : 2) * (c.k1 - c.k0);
        left -= c.blocks + TC_END - block;
        block = 0;
        if (++pair == p.pairs) pair = 0, ++b;
        return true;
    }
};

__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
        : "memory");
}
// The products of one step as one instruction sequence (issued one by one, each costs as much to prepare as it runs):
// STEPS k16 steps with both operands in shared memory, K-major, the second 64 columns `BOX >> 4` further.
template <int STEPS>
__device__ __forceinline__ void umma_f16_ss_steps(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
    static_assert(STEPS == 4 || STEPS == 8, "head sizes 64 and 128");
#define BT_SS(off, pred) "add.s64 ta, %1, " #off ";\n\tadd.s64 tb, %2, " #off ";\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], ta, tb, %3, " pred ";\n\t"
    if (STEPS == 4)
        asm volatile("{\n\t.reg .pred p0, p1;\n\t.reg .b64 ta, tb;\n\tsetp.ne.b32 p0, 0, 0;\n\tsetp.eq.b32 p1, 0, 0;\n\t"
                     BT_SS(0, "p0") BT_SS(2, "p1") BT_SS(4, "p1") BT_SS(6, "p1") "}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc) : "memory");
    else
        asm volatile("{\n\t.reg .pred p0, p1;\n\t.reg .b64 ta, tb;\n\tsetp.ne.b32 p0, 0, 0;\n\tsetp.eq.b32 p1, 0, 0;\n\t"
                     BT_SS(0, "p0") BT_SS(2, "p1") BT_SS(4, "p1") BT_SS(6, "p1") BT_SS(1024, "p1") BT_SS(1026, "p1") BT_SS(1028, "p1") BT_SS(1030, "p1") "}"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc) : "memory");
#undef BT_SS
}
// Eight k16 steps with A from TMEM (8 words of a row per step) and B with contiguous columns (16 rows of 128 bytes per step)
__device__ __forceinline__ void umma_f16_ts_steps(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
#define BT_TS(i, pred) "add.u32 ta, %1, " #i " * 8;\n\tadd.s64 tb, %2, " #i " * 128;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [ta], tb, %3, " pred ";\n\t"
    asm volatile("{\n\t.reg .pred p0, p1;\n\t.reg .b32 ta;\n\t.reg .b64 tb;\n\tsetp.ne.b32 p0, %4, 0;\n\tsetp.eq.b32 p1, 0, 0;\n\t"
                 BT_TS(0, "p0") BT_TS(1, "p1") BT_TS(2, "p1") BT_TS(3, "p1") BT_TS(4, "p1") BT_TS(5, "p1") BT_TS(6, "p1") BT_TS(7, "p1") "}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
#undef BT_TS
}
__device__ __forceinline__ void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
                   "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, int (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
          "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(taddr)
        : "memory");
}
// Two float32 operations in one instruction
__device__ __forceinline__ float2 fma_f32x2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, c, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
        "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ float2 add_f32x2(float2 a, float2 b) {
    float2 d;
    asm("{\n\t.reg .b64 a, b, d;\n\tmov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tadd.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// Which of the 32 slots from n0 on a row of token t sees.  `bits`: the row of the tree, 128 nodes, or NULL where the
// tree is read itself (more nodes than that).
__device__ __forceinline__ uint32_t tc_seen_word(const AttnParams& p, int b, int len, int end, int t, int n0, const uint4* bits) {
    if (n0 + 32 <= len) return ~0u;
    if (n0 >= end) return 0u;
    const int node = n0 - len, exist = min(end - n0, 32);          // the first slot's node, negative: committed slots come first
    const uint32_t there = exist >= 32 ? ~0u : (1u << exist) - 1u;
    if (p.tree == nullptr) {                                       // slots up to its own
        const int seen = t + 1 - node;
        return seen <= 0 ? 0u : seen >= 32 ? there : ((1u << seen) - 1u) & there;
    }
    if (bits != nullptr) {
        const uint4 w = bits[t];
        const int i = node >> 5;                                   // rounds down
        auto word = [&](int j) { return j < 0 ? ~0u : j == 0 ? w.x : j == 1 ? w.y : j == 2 ? w.z : j == 3 ? w.w : 0u; };
        return __funnelshift_r(word(i), word(i + 1), node & 31) & there;
    }
    uint32_t seen = 0;
#pragma unroll 8
    for (int e = 0; e < 32; ++e)
        if (e < exist && attn_sees(p, b, len, t, n0 + e)) seen |= 1u << e;
    return seen;
}

// Operand whose columns (not the summed dimension) are contiguous, 128-byte swizzle: 64 columns x 8 rows per 1024 bytes,
// row groups 1024 bytes apart, groups of 64 columns a tile of 128 rows apart
__device__ __forceinline__ uint64_t umma_desc_sw128_mn(uint32_t smem_addr) {
    uint64_t d = 0;
    d |= static_cast<uint64_t>((smem_addr & 0x3ffffu) >> 4);
    d |= static_cast<uint64_t>((TC_KEYS * 128) >> 4) << 16;
    d |= static_cast<uint64_t>(1024 >> 4) << 32;
    d |= static_cast<uint64_t>(1) << 46;
    d |= static_cast<uint64_t>(2) << 61;
    return d;
}
// D = f32, A and B both f16 or both bf16, M = 128
template <typename T>
__device__ __forceinline__ constexpr uint32_t tc_idesc(int n, bool b_columns_contiguous) {
    const uint32_t fmt = sizeof(T) == 2 && exponent_mask<T>() == 0x7f80u ? 1u : 0u;
    return (1u << 4) | (fmt << 7) | (fmt << 10) | ((b_columns_contiguous ? 1u : 0u) << 16) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(TC_ROWS >> 4) << 24);
}

struct TcBars {
    uint64_t full[TC_SLOTS];                                       // TMA -> products
    uint64_t empty[TC_SLOTS];                                      // products -> TMA
    uint64_t q_full[2];                                            // stream -> scores: the queries of a piece lie in shared memory
    uint64_t s_full[2];                                            // scores -> stream: they are there
    uint64_t s_read[2];                                            // stream -> scores: they are in registers, the buffer is free
    uint64_t p_full[2];                                            // stream -> outputs: weights are in place, output rescaled
    // First stream -> second: values that both multiply have been looked through.  Two, by turns: the scores of the first
    // stream's next block need the second only to have read its own, so it may look through the values of that block
    // before a warp of the second has waited for those of this one; with one barrier both phases would have passed then,
    // and a wait by parity would not see it.  No further: the block after that one needs the second stream's next scores
    // to have been read, which every warp does after this wait.
    uint64_t v_checked[2];
    uint64_t pv_done[2];                                           // outputs -> stream: they have been multiplied
    uint64_t bits[2];                                              // among the threads of a stream, twice a piece: its tree's old bits are free, the new ones there
    uint64_t drained[2];                                           // at the end: the products that a warp has issued have been made
};

// Copies the queries of a tile into shared memory, asynchronously: each warp its own 32 rows, neighbouring lanes a row.
// (A function of its own: it runs once per piece and must not cost the loop over the blocks its registers.)
template <typename T, int D>
__device__ __noinline__ void tc_fetch_queries(const AttnTcParams& p, int b, int item, int row, uint32_t base) {
    constexpr int LANES = D / 8, PER = 32 / LANES, BOX = TC_KEYS * 128;          // lanes of a row, rows at a time
    const int lane = threadIdx.x & 31, h = item / p.tiles, r = (item - h * p.tiles) * TC_ROWS + row;
    const long long mine = r < p.a.rows ? static_cast<long long>(attn_q_row<T>(p.a, b, h, r) - static_cast<const T*>(p.a.q)) : -1;
    const int chunk = lane % LANES, row0 = row - lane;
#pragma unroll 4
    for (int i = 0; i < 32 / PER; ++i) {
        const int rr = i * PER + lane / LANES, at = row0 + rr;
        const long long from = __shfl_sync(0xffffffffu, mine, rr);
        cp_async16(base + chunk / 8 * BOX + at * 128 + (((chunk & 7) ^ (at & 7)) << 4), static_cast<const T*>(p.a.q) + (from < 0 ? 0 : from) + chunk * 8, from >= 0);
    }
    cp_async_commit();
}

// What a stream leaves of the pieces that it cannot finish because a wait has run out, the one that it is in and all after it:
// NaN, in the output or in the workspace (from where the join carries them on), so that nothing that was never written
// passes for a result.  `two`: the piece that the warp is in, at `turn`, and at the other place the one after it if that has
// been looked up (else the one before, or the first one's empty place, with no more tiles before it).
// (A function of its own, for the registers of the loop over the blocks: 8 x 64/8 heads, 5 tokens, 4000 slots 50.8 us, 51.3 us
// inside the kernel, 50.2 us without it.)
template <typename T, int D>
__device__ __noinline__ void tc_leave_nan(const AttnTcParams& p, const TcWalk& after, const TcPiece* two, int turn, int x, int row) {
    TcWalk at = after;
    TcPiece c = two[turn];
    const bool ahead = two[turn ^ 1].b < 0 || two[turn ^ 1].first > c.first;
    for (bool next = ahead, more = true; more; ) {
        const int item = c.pair * 2 + x, h = item / p.tiles, r = (item - h * p.tiles) * TC_ROWS + row;
        const float nan = __int_as_float(0x7fffffff);
        if (item >= p.items) {                                     // no tile of this stream
        } else if (c.k0 > 0 || c.k1 < c.blocks) {
            p.part_ml[((static_cast<int64_t>(blockIdx.x) * 2 + (c.k0 > 0 ? 0 : 1)) * 2 + x) * TC_ROWS + row] = make_float2(nan, nan);
        } else if (r < p.a.rows) {
            T* out = attn_out_row<T>(p.a, c.b, h, r);
            for (int d = 0; d < D; ++d) out[d] = from_float<T>(nan);
        }
        if (next) {
            next = false;
            c = two[turn ^ 1];
            more = c.b >= 0;
        } else {
            more = at.next(p, c);
        }
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(TC_THREADS, 1)
attn_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ AttnTcParams p) {
    static_assert(TC_KEYS * 128 >> 4 == 1024, "umma_f16_ss_steps");
    constexpr int TILE = tc_tile_bytes<D>(), BOXES = D / 64, BOX = TC_KEYS * 128;      // a box: 128 rows of 64 columns
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* s_q = smem;                                           // [2] queries
    uint8_t* s_kv = smem + 2 * TILE;                               // [TC_SLOTS]
    TcBars& bar = *reinterpret_cast<TcBars*>(s_kv + TC_SLOTS * TILE);
    uint4* s_bits = reinterpret_cast<uint4*>(s_kv + TC_SLOTS * TILE + 1024);           // [2][TC_NODES]
    uint8_t* s_stage = reinterpret_cast<uint8_t*>(s_bits + 2 * TC_NODES);
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort_storage, s_odd;
    __shared__ int s_start[3];
    __shared__ int64_t s_left;
    __shared__ TcWalk s_walk[8];                                   // per warp of the streams
    __shared__ TcPiece s_piece[8][2];                              // the piece that the warp is in and the one after it
    volatile int* s_abort = &s_abort_storage;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < TC_SLOTS; ++s) {
            mbar_init(&bar.full[s], 1);
            mbar_init(&bar.empty[s], 1);
        }
        for (int x = 0; x < 2; ++x) {
            mbar_init(&bar.q_full[x], TC_ROWS);
            mbar_init(&bar.s_full[x], 1);
            mbar_init(&bar.s_read[x], TC_ROWS);
            mbar_init(&bar.p_full[x], TC_ROWS);
            mbar_init(&bar.pv_done[x], 1);
            mbar_init(&bar.v_checked[x], TC_ROWS);
            mbar_init(&bar.bits[x], TC_ROWS);
            mbar_init(&bar.drained[x], 1);
        }
        s_abort_storage = 0;
        s_odd = 0;
        mbar_fence_init();
    }
    if (warp == 1) tmem_alloc(&s_tmem, TC_COLS);
    pdl_launch_dependents();
    pdl_wait();
    if (warp == 0) {
        const TcCuts cuts(tc_total(p), gridDim.x);
        const int64_t from = cuts.at(blockIdx.x);
        int b, pair, block;
        tc_locate(p, from, b, pair, block);
        if (lane == 0) {
            s_start[0] = b; s_start[1] = pair; s_start[2] = block;
            s_left = cuts.at(blockIdx.x + 1) - from;
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    TcWalk walk = {s_start[0], s_start[1], s_start[2], s_left, 0};
    TcPiece c;

    if (warp == 0) {
        // ================= TMA: tiles in the order in which the products use them =================
        if (lane == 0) {
            uint32_t pos = 0;
            auto load = [&](const CUtensorMap* map, int head, int block) {
                const uint32_t s = pos % TC_SLOTS;
                if (pos == static_cast<uint32_t>(p.give_up)) {
                    report_wait_timeout();
                    *s_abort = 1;
                    return false;
                }
                if (!wait_or_abort(&bar.empty[s], ((pos / TC_SLOTS) & 1) ^ 1, s_abort)) return false;
                mbar_expect_tx(&bar.full[s], TILE);
#pragma unroll
                for (int i = 0; i < BOXES; ++i) tma_load_4d(s_kv + s * TILE + i * BOX, map, i * 64, block * TC_KEYS, head, c.b, &bar.full[s]);
                ++pos;
                return true;
            };
            bool ok = true;
            while (ok && walk.next(p, c)) {
                const int item = c.pair * 2, loads = c.own ? 2 : 1;                    // tiles of each kind and block
                const int head[2] = {item / p.tiles, (item + 1) / p.tiles};
                for (int x = 0; x < loads && ok; ++x) ok = load(&map_k, head[x], c.k0);
                if (ok && c.k0 + 1 < c.k1) ok = load(&map_k, head[0], c.k0 + 1);
                for (int k = c.k0; k < c.k1 && ok; ++k) {
                    ok = load(&map_v, head[0], k);
                    if (loads == 2) {
                        if (ok && k + 1 < c.k1) ok = load(&map_k, head[1], k + 1);
                        if (ok) ok = load(&map_v, head[1], k);
                    }
                    if (ok && k + 2 < c.k1) ok = load(&map_k, head[0], k + 2);
                }
            }
            // after a wait that ran out: the copies under way must land before the shared memory is someone else's
            for (uint32_t i = pos < TC_SLOTS ? 0 : pos - TC_SLOTS; *s_abort && i < pos; ++i)
                mbar_wait_bounded(&bar.full[i % TC_SLOTS], (i / TC_SLOTS) & 1);
        }
    } else if (warp == 1 || warp == 10) {
        // ================= products: warp 1 the scores of both streams, warp 10 their outputs =================
        // Two warps, because a product is issued no faster than the tensor cores take it: weights that are ready must not
        // wait behind scores.  Everything that the products go by is made provably the same in all lanes: the compiler then
        // keeps descriptors and addresses in uniform registers, where the instruction wants them.
        const bool values = __shfl_sync(0xffffffffu, warp, 0) == 10;
        const uint32_t tmem_u = __shfl_sync(0xffffffffu, tmem, 0);
        const uint64_t q_desc = umma_desc_sw128(smem_u32(s_q)), k_desc = umma_desc_sw128(smem_u32(s_kv)), v_desc = umma_desc_sw128_mn(smem_u32(s_kv));
        uint32_t n_q[2] = {0, 0}, n_p[2] = {0, 0}, n_read[2] = {0, 0};               // phases
        int unread = -1;                                           // the stream whose scores the buffer holds
        bool ok = true;
        auto tile_there = [&](uint32_t tile) { ok = ok && wait_or_abort_warp(&bar.full[tile % TC_SLOTS], (tile / TC_SLOTS) & 1, s_abort); };
        while (ok && __all_sync(0xffffffffu, walk.next(p, c))) {
            const int blocks = __shfl_sync(0xffffffffu, c.k1 - c.k0, 0), streams = __shfl_sync(0xffffffffu, c.streams, 0);
            const bool own = __shfl_sync(0xffffffffu, c.own, 0) != 0;
            const uint32_t first = __shfl_sync(0xffffffffu, c.first, 0);
            for (int j = 0; j < blocks && ok; ++j)
                for (int x = 0; x < streams && ok; ++x) {
                    const bool last_use = own || x == streams - 1;
                    if (!values) {
                        const uint32_t tile = first + tc_key_tile(own, blocks, j, x), slot = tile % TC_SLOTS;
                        if (x == 0 || own) tile_there(tile);
                        if (j == 0) ok = ok && wait_or_abort_warp(&bar.q_full[x], n_q[x]++ & 1, s_abort);
                        if (unread >= 0) ok = ok && wait_or_abort_warp(&bar.s_read[unread], n_read[unread]++ & 1, s_abort);
                        unread = x;
                        if (!ok) break;
                        tc_fence_after();
                        if (elect_one_lane()) {
                            umma_f16_ss_steps<D / 16>(tmem_u, q_desc + x * (TILE >> 4), k_desc + slot * (TILE >> 4), tc_idesc<T>(TC_KEYS, false));
                            umma_commit(&bar.s_full[x]);
                            if (last_use) umma_commit(&bar.empty[slot]);
                        }
                    } else {
                        const uint32_t tile = first + tc_value_tile(own, blocks, j, x), slot = tile % TC_SLOTS;
                        if (x == 0 || own) tile_there(tile);
                        ok = ok && wait_or_abort_warp(&bar.p_full[x], n_p[x]++ & 1, s_abort);
                        if (!ok) break;
                        tc_fence_after();
                        if (elect_one_lane()) {
                            umma_f16_ts_steps(tmem_u + TC_OUTPUT + x * 128, tmem_u + TC_WEIGHTS + x * 64, v_desc + slot * (TILE >> 4), tc_idesc<T>(D, true), j > 0);
                            umma_commit(&bar.pv_done[x]);
                            if (last_use) umma_commit(&bar.empty[slot]);
                        }
                    }
                    __syncwarp();
                }
        }
        // What was issued must end before the tensor memory is freed, whichever role gave up (else it has, or is about to).
        if (elect_one_lane()) umma_commit(&bar.drained[values]);
        __syncwarp();
        mbar_wait_bounded(&bar.drained[values], 0);
    } else {
        // ================= streams: one thread per row =================
        const int x = (warp - 2) >> 2, row = (warp & 3) * 32 + lane;   // a warp can reach the TMEM lanes of its number mod 4
        const uint32_t quarter = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t t_s = tmem + quarter, t_p = t_s + TC_WEIGHTS + x * 64, t_o = t_s + TC_OUTPUT + x * 128;
        uint32_t n_s = 0, n_pv = 0, n_checked = 0;                     // n_checked: blocks whose values the streams look through together
        bool ok = true;
        uint8_t* stage = s_stage + (warp - 2) * TC_STAGE;
        uint4* bits = s_bits + x * TC_NODES;
        auto fetch_queries = [&](const volatile TcPiece& w) { tc_fetch_queries<T, D>(p, w.b, w.pair * 2 + x, row, smem_u32(s_q + x * TILE)); };
        auto queries_there = [&]() {
            cp_async_wait<0>();
            fence_proxy_async_smem();
            mbar_arrive(&bar.q_full[x]);
        };
        // Every wait of the streams is one that gives up when another role has, their own barrier among them: a warp that
        // has left does not come to it.
        auto stream_together = [&](uint32_t parity) {
            mbar_arrive(&bar.bits[x]);
            return wait_or_abort_warp(&bar.bits[x], parity, s_abort);
        };
        int turn = 0;
        // Where the stream is lives in shared memory: the registers are for the scores.
        auto advance = [&]() {                                     // to the next piece that has a tile for this stream
            __syncwarp();
            if (lane == 0) {
                TcWalk at = s_walk[warp - 2];
                TcPiece to;
                bool found = false;
                while (!found && at.next(p, to)) found = to.pair * 2 + x < p.items;
                if (!found) to.b = -1;
                s_piece[warp - 2][turn ^ 1] = to;
                s_walk[warp - 2] = at;
            }
            __syncwarp();
            return s_piece[warp - 2][turn ^ 1].b >= 0;
        };
        if (lane == 0) {
            s_walk[warp - 2] = walk;
            s_piece[warp - 2][0].b = 0;                            // no piece yet
            s_piece[warp - 2][0].first = 0;
        }
        bool more = advance();
        if (more) {
            fetch_queries(s_piece[warp - 2][turn ^ 1]);
            queries_there();
        }
        while (ok && more) {
            turn ^= 1;
            const volatile TcPiece& c = s_piece[warp - 2][turn];
            const int item = c.pair * 2 + x, h = item / p.tiles, r = (item - h * p.tiles) * TC_ROWS + row;
            const bool real = r < p.a.rows;
            const int t = real ? r % p.a.T : 0;
            const bool table = p.a.tree != nullptr && p.a.T <= TC_NODES;
            if (table && c.k1 * TC_KEYS > c.len) {                 // this piece reaches the new tokens: a tree row as 128 bits
                const uint8_t* tree = p.a.tree + c.b * p.a.tree_sb;
                if (!stream_together(0)) { ok = false; break; }    // the last piece's bits are no longer needed
#pragma unroll 4
                for (int i = row >> 5; i < p.a.T; i += 4) {
                    uint32_t w[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int node = j * 32 + lane;
                        w[j] = __ballot_sync(0xffffffffu, node < p.a.T && tree[static_cast<int64_t>(i) * p.a.T + (node < p.a.T ? node : 0)] != 0);
                    }
                    if (lane == 0) bits[i] = make_uint4(w[0], w[1], w[2], w[3]);
                }
                if (!stream_together(1)) { ok = false; break; }
            }
            float m = -INFINITY, l = 0.0f;
            for (int k = c.k0; k < c.k1; ++k) {
                if (!wait_or_abort_warp(&bar.s_full[x], n_s++ & 1, s_abort)) { ok = false; break; }
                tc_fence_after();
                const int n0 = k * TC_KEYS;
                const bool tail = n0 + TC_KEYS > c.len;            // new tokens or slots past the end: what is not seen counts as -infinity
                uint32_t sees[4] = {~0u, ~0u, ~0u, ~0u};
                if (tail) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) sees[i] = tc_seen_word(p.a, c.b, c.len, c.end, t, n0 + i * 32, table ? bits : nullptr);
                    __syncwarp();
                }
                int s[4][32];
#pragma unroll
                for (int i = 0; i < 4; ++i) tmem_ld_32x32b_x32(t_s + i * 32, s[i]);
                tmem_ld_wait();
                tc_fence_before();
                mbar_arrive(&bar.s_read[x]);
                if (tail) {
#pragma unroll
                    for (int i = 0; i < 4; ++i)
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            if (!((sees[i] >> e) & 1u)) s[i][e] = __float_as_int(-INFINITY);
                }
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e = 0; e < 32; e += 2)
#pragma unroll
                    for (int i = 0; i < 4; ++i) top[i] = fmaxf(top[i], fmaxf(__int_as_float(s[i][e]), __int_as_float(s[i][e + 1])));
                if (k > c.k0) {                                    // the weights before these have been multiplied
                    if (!wait_or_abort_warp(&bar.pv_done[x], n_pv++ & 1, s_abort)) { ok = false; break; }
                    tc_fence_after();
                }
                const float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * p.scale2;
                if (__any_sync(0xffffffffu, high > m + TC_LAZY)) {
                    const float m_new = fmaxf(m, high), alpha = m_new == -INFINITY ? 1.0f : exp2_fast(m - m_new);
                    m = m_new;
                    l *= alpha;
                    if (k > c.k0) {
#pragma unroll 1
                        for (int i = 0; i < D; i += 16) {
                            int o[16];
                            tmem_ld_32x32b_x16(t_o + i, o);
                            tmem_ld_wait();
                            uint32_t f[16];
#pragma unroll
                            for (int e = 0; e < 16; ++e) f[e] = __float_as_uint(__int_as_float(o[e]) * alpha);
                            tmem_st_32x32b_x16(t_o + i, f);
                        }
                    }
                }
                const float ref = m == -INFINITY ? 0.0f : m;
                float2 sum[4] = {};
                const float2 scale = make_float2(p.scale2, p.scale2), minus = make_float2(-ref, -ref);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    uint32_t w[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        float2 y = fma_f32x2(make_float2(__int_as_float(s[i][2 * e]), __int_as_float(s[i][2 * e + 1])), scale, minus);
                        y.x = exp2_fast(y.x);
                        y.y = exp2_fast(y.y);
                        sum[e & 3] = add_f32x2(sum[e & 3], y);
                        w[e] = pack2<T>(y.x, y.y);
                    }
                    tmem_st_32x32b_x16(t_p + i * 16, w);
                }
                l += ((sum[0].x + sum[0].y) + (sum[1].x + sum[1].y)) + ((sum[2].x + sum[2].y) + (sum[3].x + sum[3].y));
                if (tail && (c.own || x == 0)) {                   // the values of this block, before anything is multiplied by them
                    const uint32_t tile = c.first + tc_value_tile(c.own, c.k1 - c.k0, k - c.k0, x), slot = tile % TC_SLOTS;
                    if (!wait_or_abort_warp(&bar.full[slot], (tile / TC_SLOTS) & 1, s_abort)) { ok = false; break; }
                    auto at = [&](int i) {                         // 16-byte piece i of the tile's rows
                        const int n = i / (D / 8), chunk = i % (D / 8);
                        return reinterpret_cast<uint4*>(s_kv + slot * TILE + chunk / 8 * BOX + n * 128 + (((chunk & 7) ^ (n & 7)) << 4));
                    };
                    const int from = max(0, c.len - n0), to = min(TC_KEYS, c.end - n0);
                    bool bad = false;
                    for (int i = to * (D / 8) + row; i < TC_KEYS * (D / 8); i += TC_ROWS) *at(i) = make_uint4(0, 0, 0, 0);
                    for (int i = from * (D / 8) + row; i < to * (D / 8); i += TC_ROWS) {
                        const uint4 v = *at(i);
                        if (any_nonfinite<T>(v.x) || any_nonfinite<T>(v.y) || any_nonfinite<T>(v.z) || any_nonfinite<T>(v.w)) {
                            bad = true;
                            *at(i) = make_uint4(finite_only<T>(v.x), finite_only<T>(v.y), finite_only<T>(v.z), finite_only<T>(v.w));
                        }
                    }
                    if (bad) *reinterpret_cast<volatile int*>(&s_odd) = 1;
                    fence_proxy_async_smem();
                    __syncwarp();
                    if (c.streams == 2 && !c.own) {
                        mbar_arrive(&bar.v_checked[n_checked & 1]);
                        ++n_checked;
                    }
                } else if (tail) {
                    if (!wait_or_abort_warp(&bar.v_checked[n_checked & 1], (n_checked >> 1) & 1, s_abort)) { ok = false; break; }
                    ++n_checked;
                }
                tmem_st_wait();
                tc_fence_before();
                mbar_arrive(&bar.p_full[x]);
            }
            if (!ok) break;
            more = advance();                                      // the last product with these queries is done
            if (more) {
                fetch_queries(s_piece[warp - 2][turn ^ 1]);
                queries_there();
            }
            if (!ok || !wait_or_abort_warp(&bar.pv_done[x], n_pv++ & 1, s_abort)) { ok = false; break; }
            tc_fence_after();
            const bool whole = c.k0 == 0 && c.k1 == c.blocks, odd = *reinterpret_cast<volatile int*>(&s_odd) != 0;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            const int64_t place = (static_cast<int64_t>(blockIdx.x) * 2 + (c.k0 > 0 ? 0 : 1)) * 2 + x;
            const long long out_row = real ? static_cast<long long>(attn_out_row<T>(p.a, c.b, h, r) - static_cast<T*>(p.a.out)) : -1;
            if (!whole) p.part_ml[place * TC_ROWS + row] = make_float2(m, l);
#pragma unroll 1
            for (int i = 0; i < D; i += 32) {
                int o[32];
                tmem_ld_32x32b_x32(t_o + i, o);
                tmem_ld_wait();
                float f[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) f[e] = l == 0.0f ? 0.0f : __int_as_float(o[e]);
                if (odd && real) {                                 // infinities and NaN of the new tokens that this row sees
                    for (int n = max(c.len, c.k0 * TC_KEYS); n < min(c.end, c.k1 * TC_KEYS); ++n) {
                        if (!attn_sees(p.a, c.b, c.len, t, n)) continue;
                        const T* val = static_cast<const T*>(p.a.v) + c.b * p.a.vb + h * p.a.vh + n * p.a.vs + i;
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            const float y = to_float<T>(val[e]);
                            if (y - y != 0.0f) f[e] += y;
                        }
                    }
                }
                __syncwarp();
                if (whole) {                                       // through the warp's buffer, so that four lanes write 64 bytes of a row
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        uint4 y;
                        y.x = pack2<T>(f[e] * inv, f[e + 1] * inv); y.y = pack2<T>(f[e + 2] * inv, f[e + 3] * inv);
                        y.z = pack2<T>(f[e + 4] * inv, f[e + 5] * inv); y.w = pack2<T>(f[e + 6] * inv, f[e + 7] * inv);
                        *reinterpret_cast<uint4*>(stage + lane * 64 + (((e >> 3) ^ ((lane >> 1) & 3)) << 4)) = y;
                    }
                    __syncwarp();
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int rr = j * 8 + (lane >> 2), q = lane & 3;
                        const uint4 y = *reinterpret_cast<const uint4*>(stage + rr * 64 + ((q ^ ((rr >> 1) & 3)) << 4));
                        const long long to = __shfl_sync(0xffffffffu, out_row, rr);
                        if (to >= 0) *reinterpret_cast<uint4*>(static_cast<T*>(p.a.out) + to + i + q * 8) = y;
                    }
                    __syncwarp();
                } else {
                    float* to = p.part_o + (place * D + i) * TC_ROWS + row;
#pragma unroll
                    for (int e = 0; e < 32; ++e) to[e * TC_ROWS] = f[e];
                }
            }
            tc_fence_before();                                     // before the next piece's weights, which say that the output may be overwritten
        }
        if (!ok) tc_leave_nan<T, D>(p, s_walk[warp - 2], s_piece[warp - 2], turn, x, row);
        __syncwarp();
        tmem_st_wait();                                            // weights on their way when a wait ran out
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem, TC_COLS);
    }
}

// Adds up the pieces of the pairs that the CTAs' cuts went through: blockIdx.x = the CTA that has such a pair's first
// piece, blockIdx.y = the stream and 16 columns; one thread per row, as the pieces were written.
constexpr int TJ_COLS = 16;

template <typename T, int D>
__global__ void __launch_bounds__(TC_ROWS) attn_tc_join_kernel(const __grid_constant__ AttnTcParams p, const int ctas) {
    const int row = threadIdx.x, x = blockIdx.y / (D / TJ_COLS), d0 = blockIdx.y % (D / TJ_COLS) * TJ_COLS;
    pdl_launch_dependents();
    pdl_wait();
    const int64_t total = tc_total(p);
    const int i = blockIdx.x;
    const TcCuts cuts(total, ctas);
    const int64_t from = cuts.at(i), to = cuts.at(i + 1);
    int b, pair, block;
    if (to >= total || to == from) return;
    tc_locate(p, to, b, pair, block);
    if (block == 0 || block >= tc_blocks(p, b) || to - block < from) return;       // the cut lies between pairs, or the pair begins in an earlier CTA
    const int64_t end = to - block + tc_blocks(p, b);
    int last = i + 1;                                              // the CTA with the pair's last piece
    while (cuts.at(last + 1) < end) ++last;
    const int item = pair * 2 + x;
    if (item >= p.items) return;
    const int h = item / p.tiles, r = (item - h * p.tiles) * TC_ROWS + row;
    auto place = [&](int cta) { return (static_cast<int64_t>(cta) * 2 + (cta == i ? 1 : 0)) * 2 + x; };
    auto there = [&](int cta) { return cuts.each > 0 || cuts.at(cta) < cuts.at(cta + 1); };      // a CTA may have no blocks at all
    float m = -INFINITY;
#pragma unroll 4
    for (int cta = i; cta <= last; ++cta)
        if (there(cta)) m = fmaxf(m, p.part_ml[place(cta) * TC_ROWS + row].x);
    const float ref = m == -INFINITY ? 0.0f : m;
    float l = 0.0f, o[TJ_COLS];
#pragma unroll
    for (int e = 0; e < TJ_COLS; ++e) o[e] = 0.0f;
    for (int cta = i; cta <= last; ++cta) {
        if (!there(cta)) continue;
        const float2 ml = p.part_ml[place(cta) * TC_ROWS + row];
        const float* src = p.part_o + (place(cta) * D + d0) * TC_ROWS + row;
        float v[TJ_COLS];
#pragma unroll
        for (int e = 0; e < TJ_COLS; ++e) v[e] = src[e * TC_ROWS];
        const float w = ml.y == 0.0f ? 0.0f : exp2f(ml.x - ref);
        l += w * ml.y;
#pragma unroll
        for (int e = 0; e < TJ_COLS; ++e) o[e] = ml.y == 0.0f ? o[e] : fmaf(w, v[e], o[e]);
    }
    if (r >= p.a.rows) return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    uint32_t packed[TJ_COLS / 2];
#pragma unroll
    for (int e = 0; e < TJ_COLS; e += 2) packed[e / 2] = pack2<T>(l == 0.0f ? 0.0f : o[e] * inv, l == 0.0f ? 0.0f : o[e + 1] * inv);
    uint4* out = reinterpret_cast<uint4*>(attn_out_row<T>(p.a, b, h, r) + d0);
    out[0] = make_uint4(packed[0], packed[1], packed[2], packed[3]);
    out[1] = make_uint4(packed[4], packed[5], packed[6], packed[7]);
}

// ---- host side ----------------------------------------------------------------------------------------------------

// Whether a call's sizes are for this kernel (the workspace goes by them).  The kernel for few rows takes more rows 16 at a
// time and reads the cache again for each tile, out of L2; what speaks for it is that a call of it costs 8 us at least,
// one of this kernel 25 us (tensor memory, barriers, the joining of pieces).  Measured, in us, that kernel / this one
// (batch x heads / key heads, new tokens, filled slots; head size 128, bf16):
//   1 x 20/20, 32, 517: 16.7 / 28.0   1 x 64/8, 5, 900: 14.7 / 31.2     1 x 64/8, 5, 16000: 56.6 / 68.0   1 x 32/8, 24, 4000: 41.8 / 54.3
//   8 x 64/8, 5, 900: 41.0 / 29.5     8 x 32/8, 24, 400: 48.5 / 28.3    1 x 64/8, 61, 400: 32.9 / 29.4    8 x 64/8, 5, 4000: 90.6 / 50.0
// so the other one where there are few tiles of few rows, or little work in all (the slots are the cache's: how many are
// filled only the device knows).
static bool attn_tc_sizes(int64_t B, int64_t H, int64_t Hkv, int64_t T, int64_t S, int64_t D, int dtype, bool want_mass) {
    const int64_t rows = H / Hkv * T, tiles = ceil_div<int64_t>(rows, AT_ROWS), all = B * Hkv * tiles;
    if (dtype == BT_F32 || (D != 64 && D != 128) || want_mass || tiles == 1) return false;
    if (rows <= TC_ROWS && all <= 64) return false;
    return static_cast<double>(all) * static_cast<double>(S) * static_cast<double>(D) > 1.3e7;
}
static size_t attn_tc_bytes(int64_t D) {
    return static_cast<size_t>(sm_count()) * 4 * TC_ROWS * (static_cast<size_t>(D) * sizeof(float) + sizeof(float2));
}
// Whether TMA can read the cache: every row on a 16-byte boundary, no stride that it cannot express.
static bool attn_tc_ok(const AttnParams& p) {
    if (!attn_stream_ok(p) || p.scale2 < 0.0f) return false;       // a row's largest score would be its smallest product
    const int64_t sizes[3] = {p.S, p.Hkv, p.B}, ks[3] = {p.ks, p.kh, p.kb}, vs[3] = {p.vs, p.vh, p.vb};
    for (int i = 0; i < 3; ++i)
        if (sizes[i] > 1 && (ks[i] <= 0 || vs[i] <= 0 || ks[i] >= (int64_t{1} << 38) || vs[i] >= (int64_t{1} << 38))) return false;
    for (int i = 0; i < 3; ++i)
        if (p.ob % 8 != 0 || p.oh % 8 != 0 || p.ot % 8 != 0) return false;
    return aligned(p.out, 16);
}

static int encode_cache_map(EncodeTiledFn encode, const void* base, int dtype, const AttnParams& p, int64_t sb, int64_t sh, int64_t ss,
                            CUtensorMap* map) {
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(p.D), static_cast<cuuint64_t>(p.S), static_cast<cuuint64_t>(p.Hkv), static_cast<cuuint64_t>(p.B)};
    const int64_t s[3] = {ss, sh, sb};
    cuuint64_t strides[3];
    for (int i = 0; i < 3; ++i) strides[i] = dims[i + 1] == 1 ? 16 : static_cast<cuuint64_t>(s[i]) * 2;      // of no meaning for a single one
    const cuuint32_t box[4] = {64, TC_KEYS, 1, 1}, step[4] = {1, 1, 1, 1};
    const CUresult cr = encode(map, dtype == BT_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base),
                               dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (cr != CUDA_SUCCESS) {
        set_error("bt_tree_attention: cuTensorMapEncodeTiled failed with code %d", static_cast<int>(cr));
        return BT_ERR_CUDA;
    }
    return BT_OK;
}

template <typename T, int D>
static int launch_attn_tc(const AttnParams& a, int dtype, float scale, void* workspace, void* stream) {
    EncodeTiledFn encode = get_encode_tiled();
    if (encode == nullptr) {
        set_error("bt_tree_attention: cuTensorMapEncodeTiled is not available from the driver");
        return BT_ERR_CUDA;
    }
    CUtensorMap map_k, map_v;
    if (const int rc = encode_cache_map(encode, a.k, dtype, a, a.kb, a.kh, a.ks, &map_k)) return rc;
    if (const int rc = encode_cache_map(encode, a.v, dtype, a, a.vb, a.vh, a.vs, &map_v)) return rc;
    AttnTcParams p = {};
    p.a = a;
    p.tiles = ceil_div(a.rows, TC_ROWS);
    p.items = a.Hkv * p.tiles;
    p.pairs = ceil_div(p.items, 2);
    p.scale2 = std::max(scale * 1.4426950408889634f, 1e-30f);      // not 0: masked scores are -infinity
    const int ctas = sm_count();
    p.give_up = tuning(BT_TUNE_ATTENTION_GIVE_UP);
    p.part_o = static_cast<float*>(workspace);
    p.part_ml = reinterpret_cast<float2*>(p.part_o + static_cast<size_t>(ctas) * 4 * TC_ROWS * D);
    static std::atomic<size_t> granted[BT_MAX_DEVICES];
    if (const int rc = ensure_dynamic_smem(attn_tc_kernel<T, D>, tc_smem<D>(), granted)) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(ctas));
    cfg.blockDim = dim3(TC_THREADS);
    cfg.dynamicSmemBytes = tc_smem<D>();
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    BT_CUDA_OK(cudaLaunchKernelEx(&cfg, attn_tc_kernel<T, D>, map_k, map_v, p));
    cfg.gridDim = dim3(static_cast<unsigned>(ctas), 2 * D / TJ_COLS);
    cfg.blockDim = dim3(TC_ROWS);
    cfg.dynamicSmemBytes = 0;
    BT_CUDA_OK(cudaLaunchKernelEx(&cfg, attn_tc_join_kernel<T, D>, p, ctas));
    return BT_OK;
}

static int launch_attn_tc_for(const AttnParams& a, int dtype, float scale, void* workspace, void* stream) {
    if (dtype == BT_F16) return a.D == 64 ? launch_attn_tc<__half, 64>(a, dtype, scale, workspace, stream) : launch_attn_tc<__half, 128>(a, dtype, scale, workspace, stream);
    return a.D == 64 ? launch_attn_tc<__nv_bfloat16, 64>(a, dtype, scale, workspace, stream) : launch_attn_tc<__nv_bfloat16, 128>(a, dtype, scale, workspace, stream);
}

}  // namespace bt

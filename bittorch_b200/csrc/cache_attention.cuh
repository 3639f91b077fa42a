// Attention of a few new tokens per sequence (a tree of drafted tokens, or one token) over a key/value cache.
//
//   s[r,n] = scale q_r . k_n,  p[r,n] = exp(s[r,n] - max) over the slots n that row r sees,  o_r = sum_n p[r,n] v_n / sum_n p[r,n]
//
// The rows of one key/value head are its query heads x the new tokens (row r = g * T + t), so the keys and values of a
// head are read once for all of them.  The slots of a sequence are cut into `nsplit` runs of whole 64-slot units,
// from the length that the device knows: every CTA takes one run with the running maximum and sum of a softmax, and
// attn_merge joins the runs (exp2 of the difference of the maxima as weights).  A run that is empty leaves sum 0.
//
// This file: the kernel for every type, head size and alignment (attn_split_kernel), in float32 on the CUDA cores,
// and the join.  16 rows x 32 slots per step: each thread owns the scores of one slot for four rows, then four
// rows x four columns of the output.  Bound by shared-memory reads of the two products; the kernels of the files beside it
// take the calls whose rows can be read in vectors, this one what is left.
//
// With mass every score is kept in float32 and read once more by attn_merge, which needs the row's sum over all runs first:
// 4 sequences of 32776 slots, 64 heads over 8, one token 118 us, 22 us of them for that; 32 tokens over 8190 slots (256 rows a head,
// 16 at a time, the scores 268 MB) 488 us.
#pragma once

#include "cache_common.cuh"

namespace bt {

constexpr int AT_THREADS = 128;
constexpr int AT_ROWS = 16;                      // rows of a CTA
constexpr int AT_KEYS = 32;                      // slots of a step
constexpr int AT_UNIT = 64;                      // runs are multiples of this many slots
constexpr int AT_MAX_SPLIT = 64;
// CTAs an SM that the runs are made for (32 sequences of 601 to 2303 slots, 20 heads: 4 90.2 us, 8 90.5 us, 16 101 us; ragged lengths and few
// sequences want more).
constexpr int AT_PER_SM = 8;

struct AttnParams {
    const void *q, *k, *v;
    void* out;
    int64_t qb, qh, qt, kb, kh, ks, vb, vh, vs, ob, oh, ot;    // strides in elements
    Lengths lengths;
    const uint8_t* tree;                         // [T,T] per tree_sb, or NULL: causal
    int64_t tree_sb;
    int B, H, Hkv, T, S, D;
    int group, rows;                             // H / Hkv, group * T
    int row_tiles, nsplit;
    float scale2;                                // scale * log2(e): scores are kept as exponents of 2
    float* mass;
    int64_t mass_sb, mass_sh;
    float* part_o;                               // [B][Hkv][rows][nsplit][D] sums not yet divided
    float2* part_ml;                             // [B][Hkv][rows][nsplit] (maximum, sum)
    float* scores;                               // mass only: [B][Hkv][rows][S]
    int vec;                                     // rows of q, k and v can be read four elements at a time
};

// Slots that exist for sequence b, committed and new ones, and the committed ones alone.
__device__ __forceinline__ int attn_len(const AttnParams& p, int b) { return p.lengths.at(b, p.S); }
__device__ __forceinline__ int attn_end(const AttnParams& p, int len) { return len + p.T < p.S ? len + p.T : p.S; }
// The run of split `i`: [first, last)
__device__ __forceinline__ void attn_run(int end, int nsplit, int i, int& first, int& last) {
    const int units = (end + AT_UNIT - 1) / AT_UNIT, per = (units + nsplit - 1) / nsplit;
    const int64_t lo = static_cast<int64_t>(i) * per * AT_UNIT, hi = lo + static_cast<int64_t>(per) * AT_UNIT;
    first = static_cast<int>(lo < end ? lo : end);
    last = static_cast<int>(hi < end ? hi : end);
}
// What a CTA of the split kernels works on: splits vary fastest, so that a head's runs are read at the same time
__device__ __forceinline__ void attn_place(const AttnParams& p, int& split, int& r0, int& h, int& b) {
    unsigned at = blockIdx.x, next = at / p.nsplit;
    split = static_cast<int>(at - next * p.nsplit);
    at = next, next = at / p.row_tiles;
    r0 = static_cast<int>(at - next * p.row_tiles) * AT_ROWS;
    b = static_cast<int>(next / p.Hkv);
    h = static_cast<int>(next - b * p.Hkv);
}
// Does token t of sequence b see slot n (n < end)?
__device__ __forceinline__ bool attn_sees(const AttnParams& p, int b, int len, int t, int n) {
    const int node = n - len;
    if (node < 0) return true;
    return p.tree ? p.tree[b * p.tree_sb + static_cast<int64_t>(t) * p.T + node] != 0 : node <= t;
}
__device__ __forceinline__ int64_t attn_row_index(const AttnParams& p, int b, int h, int r) {
    return (static_cast<int64_t>(b) * p.Hkv + h) * p.rows + r;
}
template <typename T>
__device__ __forceinline__ T* attn_out_row(const AttnParams& p, int b, int h, int r) {
    return static_cast<T*>(p.out) + b * p.ob + static_cast<int64_t>(h * p.group + r / p.T) * p.oh + static_cast<int64_t>(r % p.T) * p.ot;
}
template <typename T>
__device__ __forceinline__ const T* attn_q_row(const AttnParams& p, int b, int h, int r) {
    return static_cast<const T*>(p.q) + b * p.qb + static_cast<int64_t>(h * p.group + r / p.T) * p.qh + static_cast<int64_t>(r % p.T) * p.qt;
}

__host__ __device__ inline int attn_pitch(int D) { return (D + 3) / 4 * 4 + 4; }
inline size_t attn_smem(int D) { return sizeof(float) * (static_cast<size_t>(AT_ROWS + 2 * AT_KEYS) * attn_pitch(D) + AT_KEYS * AT_ROWS + 2 * AT_ROWS); }

template <typename T>
__global__ void __launch_bounds__(AT_THREADS) attn_split_kernel(const AttnParams p) {
    BT_DYNAMIC_SMEM(smem, 16);
    const int pitch = attn_pitch(p.D), nq = (p.D + 3) / 4;
    float* s_q = reinterpret_cast<float*>(smem);                   // [rows][pitch]
    float* s_k = s_q + AT_ROWS * pitch;                            // [slots][pitch]
    float* s_v = s_k + AT_KEYS * pitch;                            // [slots][pitch]
    float* s_p = s_v + AT_KEYS * pitch;                            // [slots][rows]; -1: the row does not see the slot
    float* s_alpha = s_p + AT_KEYS * AT_ROWS;                      // [rows]
    float* s_l = s_alpha + AT_ROWS;                                // [rows]
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    int split, r0, h, b;
    attn_place(p, split, r0, h, b);
    pdl_launch_dependents();
    pdl_wait();
    const int len = attn_len(p, b), end = attn_end(p, len);
    int first, last;
    attn_run(end, p.nsplit, split, first, last);

    for (int i = tid; i < AT_ROWS * nq; i += AT_THREADS) {
        const int r = i / nq, d = i % nq * 4;
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (r0 + r < p.rows) load4<T>(attn_q_row<T>(p, b, h, r0 + r) + d, p.vec, min(4, p.D - d), v);
        *reinterpret_cast<float4*>(s_q + r * pitch + d) = make_float4(v[0], v[1], v[2], v[3]);
    }
    const T* kbase = static_cast<const T*>(p.k) + b * p.kb + h * p.kh;
    const T* vbase = static_cast<const T*>(p.v) + b * p.vb + h * p.vh;
    float m[4], l[4], acc[2][4][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) m[j] = -INFINITY, l[j] = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[i][j][c] = 0.0f;

    for (int n0 = first; n0 < last; n0 += AT_KEYS) {
        for (int i = tid; i < AT_KEYS * nq; i += AT_THREADS) {
            const int n = i / nq, d = i % nq * 4;
            float kv[4] = {0.0f, 0.0f, 0.0f, 0.0f}, vv[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (n0 + n < last) {
                load4<T>(kbase + (n0 + n) * p.ks + d, p.vec, min(4, p.D - d), kv);
                load4<T>(vbase + (n0 + n) * p.vs + d, p.vec, min(4, p.D - d), vv);
            }
            *reinterpret_cast<float4*>(s_k + n * pitch + d) = make_float4(kv[0], kv[1], kv[2], kv[3]);
            *reinterpret_cast<float4*>(s_v + n * pitch + d) = make_float4(vv[0], vv[1], vv[2], vv[3]);
        }
        __syncthreads();
        {   // scores: lane = slot, warp = four rows
            float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            const float* kr = s_k + lane * pitch;
            const float* qr = s_q + warp * 4 * pitch;
            for (int d = 0; d < nq * 4; d += 4) {
                const float4 kv = *reinterpret_cast<const float4*>(kr + d);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float4 qv = *reinterpret_cast<const float4*>(qr + j * pitch + d);
                    s[j] = fmaf(qv.x, kv.x, fmaf(qv.y, kv.y, fmaf(qv.z, kv.z, fmaf(qv.w, kv.w, s[j]))));
                }
            }
            const int n = n0 + lane;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = r0 + warp * 4 + j;
                const bool sees = n < last && r < p.rows && attn_sees(p, b, len, r % p.T, n);
                const float x = sees ? s[j] * p.scale2 : -INFINITY;
                if (p.scores && n < last && r < p.rows) p.scores[attn_row_index(p, b, h, r) * p.S + n] = x;
                const float m_new = fmaxf(m[j], warp_max(x));
                const float ref = m_new == -INFINITY ? 0.0f : m_new;
                const float e = sees ? exp2f(x - ref) : 0.0f, alpha = exp2f(m[j] - ref);
                l[j] = l[j] * alpha + warp_add(e);
                m[j] = m_new;
                s_p[lane * AT_ROWS + warp * 4 + j] = sees ? e : -1.0f;
                if (lane == 0) s_alpha[warp * 4 + j] = alpha;
            }
        }
        __syncthreads();
        // output: item = four columns x four rows.  What a row does not see is left out of its sum, not multiplied by
        // zero: an infinity or a NaN there must not reach it.
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int item = tid + i * AT_THREADS;
            if (item >= nq * 4) break;
            const int d = item % nq * 4, rg = item / nq * 4;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float a = s_alpha[rg + j];
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[i][j][c] *= a;
            }
            const int slots = min(AT_KEYS, last - n0);
            for (int n = 0; n < slots; ++n) {
                const float4 vv = *reinterpret_cast<const float4*>(s_v + n * pitch + d);
                const float4 pv = *reinterpret_cast<const float4*>(s_p + n * AT_ROWS + rg);
                const float w[4] = {pv.x, pv.y, pv.z, pv.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if (w[j] < 0.0f) continue;
                    acc[i][j][0] = fmaf(w[j], vv.x, acc[i][j][0]);
                    acc[i][j][1] = fmaf(w[j], vv.y, acc[i][j][1]);
                    acc[i][j][2] = fmaf(w[j], vv.z, acc[i][j][2]);
                    acc[i][j][3] = fmaf(w[j], vv.w, acc[i][j][3]);
                }
            }
        }
        __syncthreads();
    }

    if (lane == 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = r0 + warp * 4 + j;
            s_l[warp * 4 + j] = l[j];
            if (r < p.rows && p.part_ml) p.part_ml[attn_row_index(p, b, h, r) * p.nsplit + split] = make_float2(m[j], l[j]);
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int item = tid + i * AT_THREADS;
        if (item >= nq * 4) break;
        const int d = item % nq * 4, rg = item / nq * 4, valid = min(4, p.D - d);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int r = r0 + rg + j;
            if (r >= p.rows) continue;
            if (p.nsplit > 1) {
                if (first >= last) continue;                       // the join does not read it
                float* o = p.part_o + (attn_row_index(p, b, h, r) * p.nsplit + split) * p.D + d;
                for (int c = 0; c < 4; ++c)
                    if (c < valid) o[c] = acc[i][j][c];
            } else {
                T* o = attn_out_row<T>(p, b, h, r) + d;
                const float lr = s_l[rg + j];
                for (int c = 0; c < 4; ++c)
                    if (c < valid) o[c] = from_float<T>(lr == 0.0f ? 0.0f : acc[i][j][c] / lr);
            }
        }
    }
}

// What a row's runs add up to: the lanes of a warp share them out.  Returns the common maximum (0 for a row that sees
// nothing), the sum in `l`, and leaves every run's weight exp2(its maximum - the common one) in weight[0 .. nsplit).
__device__ __forceinline__ float attn_row_stats(const float2* ml, int nsplit, float* weight, float& l) {
    const int lane = threadIdx.x & 31;
    float2 mine[AT_MAX_SPLIT / 32];
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < AT_MAX_SPLIT / 32; ++i) {
        mine[i] = lane + 32 * i < nsplit ? ml[lane + 32 * i] : make_float2(-INFINITY, 0.0f);
        m = fmaxf(m, mine[i].x);
    }
    m = warp_max(m);
    if (m == -INFINITY) m = 0.0f;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < AT_MAX_SPLIT / 32; ++i) {
        const float w = exp2f(mine[i].x - m);
        l += w * mine[i].y;
        if (weight != nullptr && lane + 32 * i < nsplit) weight[lane + 32 * i] = mine[i].y == 0.0f ? 0.0f : w;    // 0: wrote nothing
    }
    l = warp_add(l);
    return m;
}

constexpr int AM_THREADS = 256;
constexpr int AM_WARPS = AM_THREADS / 32;
constexpr int AM_ROWS = 64;                      // rows whose statistics a mass CTA holds at a time

// Joins the runs of a row: one warp per row, four columns per lane, the runs' loads independent of one another.  CTAs past
// the rows add the rows' weights to the mass, one thread per slot.
template <typename T>
__global__ void __launch_bounds__(AM_THREADS) attn_merge_kernel(const AttnParams p) {
    __shared__ float s_weight[AM_WARPS][AT_MAX_SPLIT];
    __shared__ float s_m[AM_ROWS], s_inv[AM_ROWS];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const unsigned rows = static_cast<unsigned>(p.B) * p.Hkv * p.rows;
    const unsigned row_blocks = p.nsplit > 1 ? (rows + AM_WARPS - 1) / AM_WARPS : 0;
    pdl_launch_dependents();
    pdl_wait();
    if (blockIdx.x < row_blocks) {
        const unsigned row = blockIdx.x * AM_WARPS + warp;
        if (row >= rows) return;                                   // a whole warp
        const unsigned bh = row / p.rows;
        const int r = static_cast<int>(row - bh * p.rows), h = static_cast<int>(bh % p.Hkv), b = static_cast<int>(bh / p.Hkv);
        float l;
        attn_row_stats(p.part_ml + static_cast<int64_t>(row) * p.nsplit, p.nsplit, s_weight[warp], l);
        __syncwarp();
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        const float* part = p.part_o + static_cast<int64_t>(row) * p.nsplit * p.D;
        T* out = attn_out_row<T>(p, b, h, r);
        const bool wide = p.D % 4 == 0;
        for (int d = lane * 4; d < p.D; d += 128) {
            float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 8
            for (int i = 0; i < p.nsplit; ++i) {
                const float w = s_weight[warp][i];
                if (w == 0.0f) continue;                           // nothing was written there, or it counts for nothing
                if (wide) {
                    const float4 x = *reinterpret_cast<const float4*>(part + static_cast<int64_t>(i) * p.D + d);
                    o[0] = fmaf(w, x.x, o[0]); o[1] = fmaf(w, x.y, o[1]); o[2] = fmaf(w, x.z, o[2]); o[3] = fmaf(w, x.w, o[3]);
                } else {
                    for (int e = 0; e < 4; ++e)
                        if (d + e < p.D) o[e] = fmaf(w, part[static_cast<int64_t>(i) * p.D + d + e], o[e]);
                }
            }
            for (int e = 0; e < 4; ++e)
                if (d + e < p.D) out[d + e] = from_float<T>(l == 0.0f ? 0.0f : o[e] * inv);
        }
        return;
    }
    // mass[n] += sum over the rows of exp2(score - row's log-sum)
    const unsigned slot_blocks = (p.S + AM_THREADS - 1) / AM_THREADS;
    const unsigned at = blockIdx.x - row_blocks, bh = at / slot_blocks;
    const int h = static_cast<int>(bh % p.Hkv), b = static_cast<int>(bh / p.Hkv);
    const int n0 = static_cast<int>(at - bh * slot_blocks) * AM_THREADS;
    const int end = attn_end(p, attn_len(p, b));
    if (n0 >= end) return;                                         // for every thread of the CTA
    const int n = n0 + tid;
    float sum = 0.0f;
    for (int r0 = 0; r0 < p.rows; r0 += AM_ROWS) {
        const int count = min(AM_ROWS, p.rows - r0);
        __syncthreads();
        for (int i = warp; i < count; i += AM_WARPS) {
            float l;
            const float m = attn_row_stats(p.part_ml + attn_row_index(p, b, h, r0 + i) * p.nsplit, p.nsplit, nullptr, l);
            if (lane == 0) {
                s_m[i] = m;
                s_inv[i] = l == 0.0f ? 0.0f : 1.0f / l;
            }
        }
        __syncthreads();
        if (n < end) {
            const float* s = p.scores + attn_row_index(p, b, h, r0) * p.S + n;
#pragma unroll 8
            for (int i = 0; i < count; ++i) sum += exp2f(s[static_cast<int64_t>(i) * p.S] - s_m[i]) * s_inv[i];
        }
    }
    if (n < end) p.mass[b * p.mass_sb + h * p.mass_sh + n] += sum;
}

// ---- host side ----------------------------------------------------------------------------------------------------

// How a call is cut up; the workspace size follows from it.
struct AttnPlan {
    int row_tiles, nsplit;
    size_t o_bytes, ml_bytes, score_bytes, tc_bytes;
    size_t bytes() const { return std::max(o_bytes + ml_bytes + score_bytes, tc_bytes); }
};

// cache_attention_tcgen05.cuh
static bool attn_tc_sizes(int64_t B, int64_t H, int64_t Hkv, int64_t T, int64_t S, int64_t D, int dtype, bool want_mass);
static size_t attn_tc_bytes(int64_t D);
static bool attn_tc_ok(const AttnParams& p);
static int launch_attn_tc_for(const AttnParams& a, int dtype, float scale, void* workspace, void* stream);

static AttnPlan attn_plan(int64_t B, int64_t H, int64_t Hkv, int64_t T, int64_t S, int64_t D, int dtype, bool want_mass) {
    AttnPlan a;
#ifdef BT_SIMT_HOST
    a.tc_bytes = 0;
    (void)dtype;
#else
    a.tc_bytes = attn_tc_sizes(B, H, Hkv, T, S, D, dtype, want_mass) ? attn_tc_bytes(D) : 0;
#endif
    const int64_t rows = H / Hkv * T;
    a.row_tiles = static_cast<int>(ceil_div<int64_t>(rows, AT_ROWS));
    const int64_t units = B * Hkv * a.row_tiles;
    // no run shorter than one unit of a full cache
    int64_t split = ceil_div<int64_t>(static_cast<int64_t>(sm_count()) * AT_PER_SM, units);
    split = std::min<int64_t>(split, ceil_div<int64_t>(S, AT_UNIT));
    a.nsplit = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(split, AT_MAX_SPLIT)));
    const size_t all = static_cast<size_t>(B) * Hkv * rows;
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    a.o_bytes = a.nsplit > 1 ? up(all * a.nsplit * D * sizeof(float)) : 0;
    a.ml_bytes = a.nsplit > 1 || want_mass ? up(all * a.nsplit * sizeof(float2)) : 0;
    a.score_bytes = want_mass ? up(all * S * sizeof(float)) : 0;
    return a;
}

// cache_attention_float.cuh, cache_attention_stream.cuh
static bool attn_float_ok(const AttnParams& p);
static int launch_attn_float(const AttnParams& p, void* stream);
static bool attn_stream_ok(const AttnParams& p);
template <typename T> static int launch_attn_stream_for(const AttnParams& p, void* stream);

template <typename T>
static int launch_attn_split(const AttnParams& p, void* stream) {
    if constexpr (sizeof(T) == 4)
        if (attn_float_ok(p)) return launch_attn_float(p, stream);
#ifndef BT_SIMT_HOST
    if constexpr (sizeof(T) == 2)
        if (attn_stream_ok(p)) return launch_attn_stream_for<T>(p, stream);
#endif
    const size_t smem = attn_smem(p.D);
    static std::atomic<size_t> granted[BT_MAX_DEVICES];
    if (const int rc = ensure_dynamic_smem(attn_split_kernel<T>, smem, granted)) return rc;
    const int64_t ctas = static_cast<int64_t>(p.B) * p.Hkv * p.row_tiles * p.nsplit;
    return launch_early(attn_split_kernel<T>, "attn_split_kernel", dim3(static_cast<unsigned>(ctas)), AT_THREADS, smem, stream, p);
}

template <typename T>
static int launch_attention(const AttnParams& p, const AttnPlan& plan, void* stream) {
    if (const int rc = launch_attn_split<T>(p, stream)) return rc;
    if (plan.ml_bytes == 0) return BT_OK;
    const int64_t rows = static_cast<int64_t>(p.B) * p.Hkv * p.rows;
    int64_t blocks = p.nsplit > 1 ? ceil_div<int64_t>(rows, AM_WARPS) : 0;
    if (p.mass) blocks += static_cast<int64_t>(p.B) * p.Hkv * ceil_div(p.S, AM_THREADS);
    return launch_early(attn_merge_kernel<T>, "attn_merge_kernel", dim3(static_cast<unsigned>(blocks)), AM_THREADS, 0, stream, p);
}

static bool attn_sizes_ok(int64_t B, int64_t H, int64_t Hkv, int64_t T, int64_t S, int64_t D) {
    return B > 0 && H > 0 && Hkv > 0 && T > 0 && S > 0 && D > 0 && H % Hkv == 0;
}
// Grid sizes and the 32-bit slot, row and head arithmetic of the kernels
static bool attn_sizes_supported(int64_t B, int64_t H, int64_t Hkv, int64_t T, int64_t S, int64_t D) {
    const int64_t most = int64_t{1} << 30;
    if (D > BT_ATTENTION_MAX_D || S > most || T > most || H > most || B > most || H / Hkv > most / T) return false;
    const int64_t tiles = ceil_div<int64_t>(H / Hkv * T, AT_ROWS);
    return B <= most / Hkv && B * Hkv <= most / tiles / AT_MAX_SPLIT && B * Hkv <= most / (S / AT_THREADS + H / Hkv * T + 1);
}

}  // namespace bt

extern "C" size_t bt_tree_attention_workspace(int64_t B, int64_t H, int64_t Hkv, int64_t T, int64_t S, int64_t D, int dtype,
                                              int want_mass) {
    using namespace bt;
    if (!attn_sizes_ok(B, H, Hkv, T, S, D) || !attn_sizes_supported(B, H, Hkv, T, S, D) || !valid_dtype(dtype)) return 0;
    return attn_plan(B, H, Hkv, T, S, D, dtype, want_mass != 0).bytes();
}

extern "C" int bt_tree_attention(const void* q, const void* k, const void* v, int dtype, int64_t B, int64_t H, int64_t Hkv,
                                 int64_t T, int64_t S, int64_t D, const int64_t* strides, const void* lengths, int lengths_i64,
                                 int64_t lengths_stride, const uint8_t* tree, int64_t tree_stride_b, float scale, float* mass,
                                 int64_t mass_sb, int64_t mass_sh, void* out, void* workspace, size_t workspace_bytes,
                                 void* stream) {
    using namespace bt;
    BT_REQUIRE(q && k && v && out && strides && lengths, "bt_tree_attention: NULL pointer");
    BT_REQUIRE(valid_dtype(dtype), "bt_tree_attention: unknown dtype %d", dtype);
    BT_REQUIRE(attn_sizes_ok(B, H, Hkv, T, S, D), "bt_tree_attention: empty input, or H is not a multiple of Hkv");
    BT_REQUIRE(lengths_stride >= 0 && tree_stride_b >= 0, "bt_tree_attention: negative stride");
    BT_REQUIRE(scale == scale && scale - scale == 0.0f, "bt_tree_attention: scale must be finite");
    BT_UNSUPPORTED_IF(!attn_sizes_supported(B, H, Hkv, T, S, D), "bt_tree_attention: sizes too large (head size at most %d)",
                      BT_ATTENTION_MAX_D);
    const AttnPlan plan = attn_plan(B, H, Hkv, T, S, D, dtype, mass != nullptr);
    BT_REQUIRE(workspace_bytes >= plan.bytes(), "bt_tree_attention: workspace of %zu bytes, %zu needed", workspace_bytes, plan.bytes());
    BT_REQUIRE(plan.bytes() == 0 || (workspace != nullptr && aligned(workspace, 16)), "bt_tree_attention: workspace must be 16-byte aligned");
    AttnParams p = {};
    p.q = q; p.k = k; p.v = v; p.out = out;
    p.qb = strides[0]; p.qh = strides[1]; p.qt = strides[2];
    p.kb = strides[3]; p.kh = strides[4]; p.ks = strides[5];
    p.vb = strides[6]; p.vh = strides[7]; p.vs = strides[8];
    p.ob = strides[9]; p.oh = strides[10]; p.ot = strides[11];
    p.lengths = {lengths, lengths_stride, lengths_i64};
    p.tree = tree; p.tree_sb = tree_stride_b;
    p.B = static_cast<int>(B); p.H = static_cast<int>(H); p.Hkv = static_cast<int>(Hkv); p.T = static_cast<int>(T);
    p.S = static_cast<int>(S); p.D = static_cast<int>(D);
    p.group = p.H / p.Hkv; p.rows = p.group * p.T;
    p.row_tiles = plan.row_tiles; p.nsplit = plan.nsplit;
    p.scale2 = scale * 1.4426950408889634f;
    p.mass = mass; p.mass_sb = mass_sb; p.mass_sh = mass_sh;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    if (plan.o_bytes) p.part_o = reinterpret_cast<float*>(ws);
    if (plan.ml_bytes) p.part_ml = reinterpret_cast<float2*>(ws + plan.o_bytes);
    if (plan.score_bytes) p.scores = reinterpret_cast<float*>(ws + plan.o_bytes + plan.ml_bytes);
    const size_t four = 4 * dtype_size(dtype);
    p.vec = D % 4 == 0 && aligned(q, four) && aligned(k, four) && aligned(v, four);
    for (int i = 0; i < 9; ++i) p.vec = p.vec && strides[i] % 4 == 0;
#ifndef BT_SIMT_HOST
    if (plan.tc_bytes != 0 && attn_tc_ok(p)) return launch_attn_tc_for(p, dtype, scale, workspace, stream);
#endif
    if (dtype == BT_F32) return launch_attention<float>(p, plan, stream);
    if (dtype == BT_F16) return launch_attention<__half>(p, plan, stream);
    return launch_attention<__nv_bfloat16>(p, plan, stream);
}

#include "cache_attention_float.cuh"

// The float32 kernel of bt_tree_attention for head sizes up to 128 whose rows can be read 16 bytes at a time: no tensor core
// takes float32 without rounding it, so the products are made on the CUDA cores, out of registers.
//
// Eight lanes share a slot: each holds every eighth 16 bytes of a key, of the warp's rows of queries and of the output, so
// that keys and values go from the cache straight into registers, once each for all of the warp's rows (RPW, four at
// most: a lane keeps D / 8 columns of queries and of output for each).  A slot's scores take three shuffles a row; the
// four groups of a warp keep maxima and sums of their own until the end.  A CTA's four warps share its tile of up to 16
// rows as rows ask for it: all slots by one to four warps at the same time, whose common reads meet in L1, and the other warps
// take other slots.  Measured against the kernel that stages the cache in shared memory (8 sequences, 8 key/value heads of
// size 128, 4091 slots): one row 50 us instead of 185 us (5.3 TB/s: HBM), 20 rows 247 us instead of 324 us (10.9 TFLOP/s: the eight
// warps that fit an SM at 252 registers a thread do not cover the way of the loads; more slots a step and loads a step ahead
// were slower, 286 us and 277 us).  Many rows read the cache again for every 16 of them: 8 sequences of 4000 slots, 64 heads over 8,
// size 128: 64 rows 736 us, 488 rows 4.4 ms, 14.9 TFLOP/s of 74; two library products with the scores written out between them take
// 733 us and 3.4 ms.
#pragma once

#include "cache_attention.cuh"

namespace bt {

constexpr int AF_WARPS = 4;
constexpr int AF_SLOTS = 2;                                        // slots of a group's step

// P: 16-byte pieces of a lane; FULL: there are no columns behind the head size
template <int P, int RPW, bool FULL>
__global__ void __launch_bounds__(AF_WARPS * 32, RPW == 1 ? 4 : 2) attn_float_kernel(const AttnParams p) {
    constexpr int D = P * 32;                                      // the columns of a row, with those behind p.D
    __shared__ __align__(16) float s_o[AF_WARPS * RPW * D];        // [warps][rows][D]
    __shared__ float2 s_ml[AF_WARPS * RPW];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 3, c = lane & 7;
    int split, r0, h, b;
    attn_place(p, split, r0, h, b);
    pdl_launch_dependents();
    pdl_wait();
    const int len = attn_len(p, b), end = attn_end(p, len);
    int first, last;
    attn_run(end, p.nsplit, split, first, last);
    const int count = min(AT_ROWS, p.rows - r0);
    const int wr = count <= RPW ? 1 : count <= 2 * RPW ? 2 : 4;    // warps along the rows; AF_WARPS / wr along the slots
    const int rw = r0 + warp % wr * RPW, sw = warp / wr, step = AF_WARPS / wr * 4 * AF_SLOTS;
    const float* kbase = static_cast<const float*>(p.k) + b * p.kb + h * p.kh;
    const float* vbase = static_cast<const float*>(p.v) + b * p.vb + h * p.vh;

    const float4 zero = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float4 q[RPW][P], o[RPW][P];
    int token[RPW];
    float m[RPW], l[RPW];
#pragma unroll
    for (int j = 0; j < RPW; ++j) {
        const bool on = rw + j < p.rows;
        token[j] = on ? (rw + j) % p.T : -1;
        m[j] = -INFINITY;
        l[j] = 0.0f;
        const float* row = attn_q_row<float>(p, b, h, on ? rw + j : 0);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const int d = (c + 8 * i) * 4;
            q[j][i] = on && d < p.D ? *reinterpret_cast<const float4*>(row + d) : zero;
            o[j][i] = zero;
        }
    }
    for (int n0 = first + sw * 4 * AF_SLOTS; n0 < last; n0 += step) {
        float4 k[AF_SLOTS][P], v[AF_SLOTS][P];
#pragma unroll
        for (int u = 0; u < AF_SLOTS; ++u) {
            const int64_t n = min(n0 + u * 4 + g, last - 1);       // what lies behind the run is read twice and seen by no row
            const float *kn = kbase + n * p.ks + c * 4, *vn = vbase + n * p.vs + c * 4;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const bool on = FULL || (c + 8 * i) * 4 < p.D;
                k[u][i] = on ? *reinterpret_cast<const float4*>(kn + i * 32) : zero;
                v[u][i] = on ? *reinterpret_cast<const float4*>(vn + i * 32) : zero;
            }
        }
        float s[AF_SLOTS][RPW];
#pragma unroll
        for (int u = 0; u < AF_SLOTS; ++u)
#pragma unroll
            for (int j = 0; j < RPW; ++j) {
                float x = 0.0f;
#pragma unroll
                for (int i = 0; i < P; ++i)
                    x = fmaf(q[j][i].x, k[u][i].x, fmaf(q[j][i].y, k[u][i].y, fmaf(q[j][i].z, k[u][i].z, fmaf(q[j][i].w, k[u][i].w, x))));
                x += __shfl_xor_sync(0xffffffffu, x, 1);
                x += __shfl_xor_sync(0xffffffffu, x, 2);
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                s[u][j] = x * p.scale2;
            }
        // What a row does not see is left out of its sums, not multiplied by zero: an infinity or a NaN there must not reach it.
        const bool all = n0 + 4 * AF_SLOTS <= min(len, last);      // committed slots
        unsigned sees = 0xffffffffu;
        if (!all) {
            sees = 0;
#pragma unroll
            for (int u = 0; u < AF_SLOTS; ++u)
#pragma unroll
                for (int j = 0; j < RPW; ++j) {
                    const int n = n0 + u * 4 + g;
                    if (n < last && token[j] >= 0 && attn_sees(p, b, len, token[j], n)) sees |= 1u << (u * RPW + j);
                    else s[u][j] = -INFINITY;
                }
        }
        if (p.scores != nullptr && c == 0) {
#pragma unroll
            for (int u = 0; u < AF_SLOTS; ++u)
#pragma unroll
                for (int j = 0; j < RPW; ++j)
                    if (n0 + u * 4 + g < last && token[j] >= 0) p.scores[attn_row_index(p, b, h, rw + j) * p.S + n0 + u * 4 + g] = s[u][j];
        }
#pragma unroll
        for (int j = 0; j < RPW; ++j) {
            float x = s[0][j];
#pragma unroll
            for (int u = 1; u < AF_SLOTS; ++u) x = fmaxf(x, s[u][j]);
            if (x > m[j]) {                                        // rare once the maximum has been met
                const float f = exp2f(m[j] - x);
                m[j] = x;
                l[j] *= f;
#pragma unroll
                for (int i = 0; i < P; ++i) o[j][i].x *= f, o[j][i].y *= f, o[j][i].z *= f, o[j][i].w *= f;
            }
            const float ref = m[j] == -INFINITY ? 0.0f : m[j];
#pragma unroll
            for (int u = 0; u < AF_SLOTS; ++u) {
                if (!((sees >> (u * RPW + j)) & 1u)) continue;
                const float w = exp2f(s[u][j] - ref);
                l[j] += w;
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    o[j][i].x = fmaf(w, v[u][i].x, o[j][i].x);
                    o[j][i].y = fmaf(w, v[u][i].y, o[j][i].y);
                    o[j][i].z = fmaf(w, v[u][i].z, o[j][i].z);
                    o[j][i].w = fmaf(w, v[u][i].w, o[j][i].w);
                }
            }
        }
    }

    // the four groups of the warp become one, then the warps of the same rows
#pragma unroll
    for (int j = 0; j < RPW; ++j) {
        const float top = fmaxf(m[j], __shfl_xor_sync(0xffffffffu, m[j], 8));
        const float all = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
        const float f = m[j] == -INFINITY ? 0.0f : exp2f(m[j] - all);   // times a sum of NaN stays NaN
        float sum = l[j] * f;
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        if (lane == 0) s_ml[warp * RPW + j] = make_float2(all, sum);
#pragma unroll
        for (int i = 0; i < P; ++i) {
            float x[4] = {o[j][i].x * f, o[j][i].y * f, o[j][i].z * f, o[j][i].w * f};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] += __shfl_xor_sync(0xffffffffu, x[e], 8);
                x[e] += __shfl_xor_sync(0xffffffffu, x[e], 16);
            }
            if (g == 0) *reinterpret_cast<float4*>(s_o + (warp * RPW + j) * D + (c + 8 * i) * 4) = make_float4(x[0], x[1], x[2], x[3]);
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < count * (D / 4); i += AF_WARPS * 32) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        if (d >= p.D) continue;
        const int w0 = r / RPW, j = r % RPW;                       // the first of the row's warps, and its place there
        float top = -INFINITY, sum = 0.0f;
        for (int w = w0; w < AF_WARPS; w += wr) top = fmaxf(top, s_ml[w * RPW + j].x);
        float4 x = zero;
        for (int w = w0; w < AF_WARPS; w += wr) {
            const float2 ml = s_ml[w * RPW + j];
            const float f = ml.x == -INFINITY ? 0.0f : exp2f(ml.x - top);
            const float4 part = *reinterpret_cast<const float4*>(s_o + (w * RPW + j) * D + d);
            sum = fmaf(ml.y, f, sum);
            x.x = fmaf(part.x, f, x.x); x.y = fmaf(part.y, f, x.y); x.z = fmaf(part.z, f, x.z); x.w = fmaf(part.w, f, x.w);
        }
        const int64_t row = attn_row_index(p, b, h, r0 + r);
        if (p.part_ml != nullptr && d == 0) p.part_ml[row * p.nsplit + split] = make_float2(top, sum);
        if (p.nsplit > 1) {
            if (first < last) *reinterpret_cast<float4*>(p.part_o + (row * p.nsplit + split) * p.D + d) = x;     // else the join does not read it
        } else {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            float* out = attn_out_row<float>(p, b, h, r0 + r) + d;
            out[0] = sum == 0.0f ? 0.0f : x.x * inv;
            out[1] = sum == 0.0f ? 0.0f : x.y * inv;
            out[2] = sum == 0.0f ? 0.0f : x.z * inv;
            out[3] = sum == 0.0f ? 0.0f : x.w * inv;
        }
    }
}

static bool attn_float_ok(const AttnParams& p) { return p.vec && p.D <= 128; }

template <int P>
static int launch_attn_float_for(const AttnParams& p, void* stream) {
    const dim3 grid(static_cast<unsigned>(static_cast<int64_t>(p.B) * p.Hkv * p.row_tiles * p.nsplit));
    if (p.rows == 1)
        return launch_early(p.D == 32 * P ? attn_float_kernel<P, 1, true> : attn_float_kernel<P, 1, false>, "attn_float_kernel", grid, AF_WARPS * 32, 0, stream, p);
    return launch_early(p.D == 32 * P ? attn_float_kernel<P, 4, true> : attn_float_kernel<P, 4, false>, "attn_float_kernel", grid, AF_WARPS * 32, 0, stream, p);
}
static int launch_attn_float(const AttnParams& p, void* stream) {
    if (p.D <= 32) return launch_attn_float_for<1>(p, stream);
    if (p.D <= 64) return launch_attn_float_for<2>(p, stream);
    if (p.D <= 96) return launch_attn_float_for<3>(p, stream);
    return launch_attn_float_for<4>(p, stream);
}

}  // namespace bt

// The 16-bit kernel of bt_tree_attention for few rows per key/value head, 16 at a time (one token with grouped heads, small trees):
// bound by HBM, so it is built around the loads.
//
// A CTA is four warps, and every warp is a pipeline of its own: it copies 16 slots of keys and values at a time into its
// private ring in shared memory (cp.async, two steps in flight while it works on the third), so that nothing but the end
// of the CTA waits for another warp.  Scores and output are m16n8k16 products on the warp's registers:
//   scores  rows x slots: the sum over D may run in any order, so a thread takes 16 contiguous bytes of a key for two
//           products instead of the four 4-byte pieces the instruction's own order would ask for;
//   output  rows x D: a thread takes 16 contiguous bytes of four slots' values and pairs the slots up with byte
//           permutes; the columns of the product are numbered to match.
// Both come from shared memory without bank conflicts by exchanging 16-byte pieces of a row by the row's number.
// The weights are rounded to the cache's type for the second product (relative 2^-8 / 2^-11 at most each, their sum is
// taken before the rounding; in fp16 a weight below 2^-14 of the largest is off by up to 2^-25 of that instead); everything
// else stays float32.
//
// 32 sequences of 601 to 2303 slots, 20 heads, head size 128, bf16: 90 us with the join, 5.3 TB/s (a plain copy: 6.53).  Head
// sizes between those it is built for are padded with zeros in the ring: 8 x 4090 slots, 32 heads over 8, head size 80: 38 us,
// on the CUDA cores 143 us.  Many rows of a head size other than 64 and 128 are this kernel's too, and the cache is read again, out of
// L2, for every 16 of them: 8 trees of 61 nodes, 64 heads over 8, up to 8190 slots, bf16: size 80 789 us, 96 764 us, 256 2649 us,
// 75 to 97 TFLOP/s (size 128 on the tensor-memory kernel 135 us).
#pragma once

#include "cache_attention.cuh"

namespace bt {

constexpr int AS_WARPS = 4;
constexpr int AS_STAGES = 3;
constexpr int AS_SLOTS = 16;                                       // slots of a warp's step

template <int D> __host__ __device__ constexpr int as_pitch() { return (D * 2 + 127) / 128 * 128; }       // bytes of a row in the ring
template <int D> __host__ __device__ constexpr int as_stage_bytes() { return 2 * AS_SLOTS * as_pitch<D>(); }
template <int D> constexpr size_t as_smem() { return static_cast<size_t>(AS_WARPS) * AS_STAGES * as_stage_bytes<D>() + AS_WARPS * AT_ROWS * sizeof(float2); }

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool on) {
    const int bytes = on ? 16 : 0;                                 // the rest of the 16 bytes is filled with zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
    return v;
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
template <> __device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
// Exponent bits of the two halves of a word; all ones: an infinity or a NaN
template <typename T> __device__ __forceinline__ constexpr uint32_t exponent_mask() { return 0; }
template <> __device__ __forceinline__ constexpr uint32_t exponent_mask<__nv_bfloat16>() { return 0x7f80u; }
template <> __device__ __forceinline__ constexpr uint32_t exponent_mask<__half>() { return 0x7c00u; }
template <typename T>
__device__ __forceinline__ bool any_nonfinite(uint32_t w) {
    constexpr uint32_t m = exponent_mask<T>();
    return (w & m) == m || ((w >> 16) & m) == m;
}
template <typename T>
__device__ __forceinline__ uint32_t finite_only(uint32_t w) {      // infinities and NaN replaced by zero
    constexpr uint32_t m = exponent_mask<T>();
    if ((w & m) == m) w &= 0xffff0000u;
    if (((w >> 16) & m) == m) w &= 0x0000ffffu;
    return w;
}

// FULL: the head size is D; otherwise it is a smaller multiple of 8, and the columns behind it are zeros in the ring.
template <typename T, int D, bool FULL>
__global__ void __launch_bounds__(AS_WARPS * 32, D <= 128 ? 2 : 1) attn_stream_kernel(const AttnParams p) {
    constexpr int PITCH = as_pitch<D>(), STAGE = as_stage_bytes<D>(), CHUNKS = D / 8, V_AT = AS_SLOTS * PITCH;
    constexpr int TILES = D / 8;                                   // n8 tiles of the output
    static_assert(D % 32 == 0 && D <= 256, "head sizes of this kernel");
    const int width = FULL ? D : p.D;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    float2* s_ml = reinterpret_cast<float2*>(smem + AS_WARPS * AS_STAGES * STAGE);       // [warps][rows]
    const uint32_t ring = smem_u32(smem) + warp * AS_STAGES * STAGE;
    int split, r0, h, b;
    attn_place(p, split, r0, h, b);
    pdl_launch_dependents();
    pdl_wait();
    const int len = attn_len(p, b), end = attn_end(p, len);
    int first, last;
    attn_run(end, p.nsplit, split, first, last);
    if (first >= last && p.nsplit > 1) {                           // a run that this length does not have
        const int r = r0 + threadIdx.x;
        if (threadIdx.x < AT_ROWS && r < p.rows) p.part_ml[attn_row_index(p, b, h, r) * p.nsplit + split] = make_float2(-INFINITY, 0.0f);
        return;
    }
    const T* kbase = static_cast<const T*>(p.k) + b * p.kb + h * p.kh;
    const T* vbase = static_cast<const T*>(p.v) + b * p.vb + h * p.vh;

    const int n_first = first + warp * AS_SLOTS;
    const int steps = n_first < last ? (last - n_first + AS_WARPS * AS_SLOTS - 1) / (AS_WARPS * AS_SLOTS) : 0;
    auto load = [&](int step) {
        if (step < steps) {
            const int n0 = n_first + step * AS_WARPS * AS_SLOTS;
            const uint32_t stage = ring + step % AS_STAGES * STAGE;
#pragma unroll
            for (int i = 0; i < AS_SLOTS * CHUNKS / 32; ++i) {
                const int idx = i * 32 + lane, row = idx / CHUNKS, chunk = idx % CHUNKS;
                const bool on = n0 + row < last && chunk * 8 < width;
                const int64_t n = on ? n0 + row : first;           // a valid address for what is only zeros
                const int col = FULL || on ? chunk * 8 : 0;
                cp_async16(stage + row * PITCH + ((chunk ^ ((row & 1) << 2)) << 4), kbase + n * p.ks + col, on);
                cp_async16(stage + V_AT + row * PITCH + ((chunk ^ (((row >> 1) & 3) << 1)) << 4), vbase + n * p.vs + col, on);
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < AS_STAGES - 1; ++s) load(s);

    // queries: rows g and g + 8, the 16-byte pieces c + 4j, in the order in which the keys are taken
    uint32_t qa[D / 32][2][4];
    const int ra = r0 + g, rb = r0 + g + 8;
    const int ta = ra % p.T, tb = rb % p.T;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
        const uint4 zero = make_uint4(0, 0, 0, 0);
        const uint4 qx = ra < p.rows && (c + 4 * j) * 8 < width ? *reinterpret_cast<const uint4*>(attn_q_row<T>(p, b, h, ra) + (c + 4 * j) * 8) : zero;
        const uint4 qy = rb < p.rows && (c + 4 * j) * 8 < width ? *reinterpret_cast<const uint4*>(attn_q_row<T>(p, b, h, rb) + (c + 4 * j) * 8) : zero;
        qa[j][0][0] = qx.x; qa[j][0][1] = qy.x; qa[j][0][2] = qx.y; qa[j][0][3] = qy.y;
        qa[j][1][0] = qx.z; qa[j][1][1] = qy.z; qa[j][1][2] = qx.w; qa[j][1][3] = qy.w;
    }
    float o[TILES][4];
#pragma unroll
    for (int t = 0; t < TILES; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[t][i] = 0.0f;
    float ma = -INFINITY, mb = -INFINITY, la = 0.0f, lb = 0.0f;

    for (int step = 0; step < steps; ++step) {
        cp_async_wait<AS_STAGES - 2>();
        __syncwarp();                                              // every lane's copies have landed, and the last step's reads are over
        load(step + AS_STAGES - 1);
        const uint32_t stage = ring + step % AS_STAGES * STAGE;
        const int n0 = n_first + step * AS_WARPS * AS_SLOTS;
        float s[2][4];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
            s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.0f;
            const uint32_t krow = stage + (nt * 8 + g) * PITCH;
#pragma unroll
            for (int j = 0; j < D / 32; ++j) {
                const uint4 kv = lds128(krow + (((c + 4 * j) ^ ((g & 1) << 2)) << 4));
                mma16816<T>(s[nt], qa[j][0], kv.x, kv.y);
                mma16816<T>(s[nt], qa[j][1], kv.z, kv.w);
            }
        }
        const bool tail = n0 + AS_SLOTS > len;                     // new tokens, or slots past the end, are among these
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[nt][i] *= p.scale2;
                if (tail) {
                    const int n = n0 + nt * 8 + 2 * c + (i & 1), r = i < 2 ? ra : rb;
                    const bool sees = n < last && r < p.rows && attn_sees(p, b, len, i < 2 ? ta : tb, n);
                    if (!sees) s[nt][i] = -INFINITY;
                }
            }
        if (p.scores != nullptr) {
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int n = n0 + nt * 8 + 2 * c + (i & 1), r = i < 2 ? ra : rb;
                    if (n < last && r < p.rows) p.scores[attn_row_index(p, b, h, r) * p.S + n] = s[nt][i];
                }
        }
        float xa = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[1][0], s[1][1]));
        float xb = fmaxf(fmaxf(s[0][2], s[0][3]), fmaxf(s[1][2], s[1][3]));
        xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, 1));
        xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, 1));
        xa = fmaxf(xa, __shfl_xor_sync(0xffffffffu, xa, 2));
        xb = fmaxf(xb, __shfl_xor_sync(0xffffffffu, xb, 2));
        if (__any_sync(0xffffffffu, xa > ma || xb > mb)) {         // rare once the maximum has been met
            const float na = fmaxf(ma, xa), nb = fmaxf(mb, xb);
            const float fa = na == -INFINITY ? 1.0f : exp2_fast(ma - na), fb = nb == -INFINITY ? 1.0f : exp2_fast(mb - nb);
            ma = na; mb = nb; la *= fa; lb *= fb;
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                o[t][0] *= fa; o[t][1] *= fa; o[t][2] *= fb; o[t][3] *= fb;
            }
        }
        const float refa = ma == -INFINITY ? 0.0f : ma, refb = mb == -INFINITY ? 0.0f : mb;
        float w[2][4];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
            w[nt][0] = exp2_fast(s[nt][0] - refa); w[nt][1] = exp2_fast(s[nt][1] - refa);
            w[nt][2] = exp2_fast(s[nt][2] - refb); w[nt][3] = exp2_fast(s[nt][3] - refb);
            la += w[nt][0] + w[nt][1];
            lb += w[nt][2] + w[nt][3];
        }
        const uint32_t pa[4] = {pack2<T>(w[0][0], w[0][1]), pack2<T>(w[0][2], w[0][3]), pack2<T>(w[1][0], w[1][1]), pack2<T>(w[1][2], w[1][3])};
        // values: slots 2c, 2c+1, 2c+8, 2c+9; all four rows exchange their pieces by c
        const uint32_t vrow = stage + V_AT + 2 * c * PITCH;
        bool odd = false;
        if (tail && n0 + AS_SLOTS > len) {                         // an infinity or NaN in a new token that some do not see?
            bool bad = false;
#pragma unroll
            for (int i = 0; i < AS_SLOTS * CHUNKS / 32; ++i) {
                const int idx = i * 32 + lane;
                const uint4 v = lds128(stage + V_AT + idx / CHUNKS * PITCH + ((idx % CHUNKS) << 4 ^ (((idx / CHUNKS >> 1) & 3) << 5)));
                bad = bad || any_nonfinite<T>(v.x) || any_nonfinite<T>(v.y) || any_nonfinite<T>(v.z) || any_nonfinite<T>(v.w);
            }
            odd = __any_sync(0xffffffffu, bad);
        }
#pragma unroll
        for (int j = 0; j < D / 64; ++j) {
            const uint32_t piece = ((g + 8 * j) ^ (c << 1)) << 4;
            uint4 v0 = lds128(vrow + piece), v1 = lds128(vrow + PITCH + piece);
            uint4 v2 = lds128(vrow + 8 * PITCH + piece), v3 = lds128(vrow + 9 * PITCH + piece);
            uint32_t x0[4] = {v0.x, v0.y, v0.z, v0.w}, x1[4] = {v1.x, v1.y, v1.z, v1.w};
            uint32_t x2[4] = {v2.x, v2.y, v2.z, v2.w}, x3[4] = {v3.x, v3.y, v3.z, v3.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (odd) {
                    x0[e] = finite_only<T>(x0[e]); x1[e] = finite_only<T>(x1[e]);
                    x2[e] = finite_only<T>(x2[e]); x3[e] = finite_only<T>(x3[e]);
                }
                mma16816<T>(o[j * 8 + 2 * e], pa, __byte_perm(x0[e], x1[e], 0x5410), __byte_perm(x2[e], x3[e], 0x5410));
                mma16816<T>(o[j * 8 + 2 * e + 1], pa, __byte_perm(x0[e], x1[e], 0x7632), __byte_perm(x2[e], x3[e], 0x7632));
            }
        }
        if constexpr (D % 64 == 32) {                              // the last 32 columns: four of them per thread
            constexpr int J = D / 64;
            const uint32_t piece = (((8 * J + (g >> 1)) ^ (c << 1)) << 4) + ((g & 1) << 3);
            const uint2 v0 = lds64(vrow + piece), v1 = lds64(vrow + PITCH + piece);
            const uint2 v2 = lds64(vrow + 8 * PITCH + piece), v3 = lds64(vrow + 9 * PITCH + piece);
            uint32_t x0[2] = {v0.x, v0.y}, x1[2] = {v1.x, v1.y}, x2[2] = {v2.x, v2.y}, x3[2] = {v3.x, v3.y};
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (odd) {
                    x0[e] = finite_only<T>(x0[e]); x1[e] = finite_only<T>(x1[e]);
                    x2[e] = finite_only<T>(x2[e]); x3[e] = finite_only<T>(x3[e]);
                }
                mma16816<T>(o[J * 8 + 2 * e], pa, __byte_perm(x0[e], x1[e], 0x5410), __byte_perm(x2[e], x3[e], 0x5410));
                mma16816<T>(o[J * 8 + 2 * e + 1], pa, __byte_perm(x0[e], x1[e], 0x7632), __byte_perm(x2[e], x3[e], 0x7632));
            }
        }
        if (odd) {                                                 // add the infinities and NaN to the rows that see their slot
            for (int n = 0; n < AS_SLOTS; ++n) {
                const int from = (g << 2) | ((n & 7) >> 1);        // the lane of this quad that holds slot n's weights
                const float w0 = n < 8 ? ((n & 1) ? w[0][1] : w[0][0]) : ((n & 1) ? w[1][1] : w[1][0]);
                const float w1 = n < 8 ? ((n & 1) ? w[0][3] : w[0][2]) : ((n & 1) ? w[1][3] : w[1][2]);
                const float pa_n = __shfl_sync(0xffffffffu, w0, from), pb_n = __shfl_sync(0xffffffffu, w1, from);
                const int slot = n0 + n;
                const bool sa = slot < last && ra < p.rows && attn_sees(p, b, len, ta, slot);
                const bool sb = slot < last && rb < p.rows && attn_sees(p, b, len, tb, slot);
#pragma unroll
                for (int t = 0; t < TILES; ++t)
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int per = t < D / 64 * 8 ? 8 : 4, base = t < D / 64 * 8 ? t / 8 * 64 : D / 64 * 64, e = t < D / 64 * 8 ? t % 8 : t - D / 64 * 8;
                        const int col = base + (2 * c + half) * per + e;
                        const uint32_t addr = stage + V_AT + n * PITCH + (((col >> 3) ^ (((n >> 1) & 3) << 1)) << 4) + (col & 7) * 2;
                        unsigned short bits;
                        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(bits) : "r"(addr));
                        if ((bits & exponent_mask<T>()) != exponent_mask<T>()) continue;
                        const float v = to_float<T>(*reinterpret_cast<const T*>(&bits));
                        if (sa) o[t][half] += pa_n * v;
                        if (sb) o[t][2 + half] += pb_n * v;
                    }
            }
        }
    }
    cp_async_wait<0>();

    // the four warps' runs become one
    la += __shfl_xor_sync(0xffffffffu, la, 1);
    lb += __shfl_xor_sync(0xffffffffu, lb, 1);
    la += __shfl_xor_sync(0xffffffffu, la, 2);
    lb += __shfl_xor_sync(0xffffffffu, lb, 2);
    if (c == 0) {
        s_ml[warp * AT_ROWS + g] = make_float2(ma, la);
        s_ml[warp * AT_ROWS + g + 8] = make_float2(mb, lb);
    }
    __syncthreads();                                               // every ring is free
    float* s_o = reinterpret_cast<float*>(smem);                   // [warps][rows][D]
    float m_all[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < AS_WARPS; ++i) {
        m_all[0] = fmaxf(m_all[0], s_ml[i * AT_ROWS + g].x);
        m_all[1] = fmaxf(m_all[1], s_ml[i * AT_ROWS + g + 8].x);
    }
    // A thread holds 16 (last 32 columns of 96: 8) neighbouring columns of its rows.  Pieces of four columns change places
    // within groups of four, by row and place, so that a store meets no bank twice.
    const float f_ab[2] = {exp2_fast(ma - m_all[0]), exp2_fast(mb - m_all[1])};     // of no meaning where the sum is 0
    auto place = [](int r, int f) { return f ^ ((f >> 3) & 1) ^ ((r & 1) << 1); };
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        if ((half ? rb : ra) >= p.rows || (half ? lb : la) == 0.0f) continue;
        const int r = g + 8 * half;
        float4* row = reinterpret_cast<float4*>(s_o + (warp * AT_ROWS + r) * D);
        const float f = f_ab[half];
#pragma unroll
        for (int t = 0; t < TILES; t += 4) {
            const bool whole = t < D / 64 * 8;
            const int at0 = whole ? t / 8 * 16 + 4 * c + t % 8 / 4 : D / 64 * 16 + 2 * c, step = whole ? 2 : 1;
            row[place(r, at0)] = make_float4(o[t][2 * half] * f, o[t + 1][2 * half] * f, o[t + 2][2 * half] * f, o[t + 3][2 * half] * f);
            row[place(r, at0 + step)] = make_float4(o[t][2 * half + 1] * f, o[t + 1][2 * half + 1] * f, o[t + 2][2 * half + 1] * f, o[t + 3][2 * half + 1] * f);
        }
    }
    __syncthreads();
    const int rows = min(AT_ROWS, p.rows - r0);
    for (int i = threadIdx.x; i < rows * (D / 4); i += AS_WARPS * 32) {
        const int r = i / (D / 4), d = i % (D / 4) * 4;
        if (d >= width) continue;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        float m = -INFINITY, l = 0.0f;
        float2 ml[AS_WARPS];
#pragma unroll
        for (int k = 0; k < AS_WARPS; ++k) {
            ml[k] = s_ml[k * AT_ROWS + r];
            m = fmaxf(m, ml[k].x);
        }
#pragma unroll
        for (int k = 0; k < AS_WARPS; ++k) {
            if (ml[k].y == 0.0f) continue;                         // that warp saw nothing and wrote nothing
            const float4 x = reinterpret_cast<const float4*>(s_o + (k * AT_ROWS + r) * D)[place(r, d >> 2)];
            v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
            l += ml[k].y * exp2_fast(ml[k].x - m);
        }
        const int64_t row = attn_row_index(p, b, h, r0 + r);
        if (p.part_ml != nullptr && d == 0) p.part_ml[row * p.nsplit + split] = make_float2(m, l);
        if (p.nsplit > 1) {
            *reinterpret_cast<float4*>(p.part_o + (row * p.nsplit + split) * width + d) = v;
        } else {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            T* out = attn_out_row<T>(p, b, h, r0 + r) + d;
            out[0] = from_float<T>(l == 0.0f ? 0.0f : v.x * inv);
            out[1] = from_float<T>(l == 0.0f ? 0.0f : v.y * inv);
            out[2] = from_float<T>(l == 0.0f ? 0.0f : v.z * inv);
            out[3] = from_float<T>(l == 0.0f ? 0.0f : v.w * inv);
        }
    }
}

template <typename T, int D, bool FULL>
static int launch_attn_stream(const AttnParams& p, void* stream) {
    static std::atomic<size_t> granted[BT_MAX_DEVICES];
    if (const int rc = ensure_dynamic_smem(attn_stream_kernel<T, D, FULL>, as_smem<D>(), granted)) return rc;
    const int64_t ctas = static_cast<int64_t>(p.B) * p.Hkv * p.row_tiles * p.nsplit;
    return launch_early(attn_stream_kernel<T, D, FULL>, "attn_stream_kernel", dim3(static_cast<unsigned>(ctas)), AS_WARPS * 32, as_smem<D>(), stream, p);
}

// Whether this kernel can take the call: 16-bit rows, every one on a 16-byte boundary and a multiple of 16 bytes long.
static bool attn_stream_ok(const AttnParams& p) {
    if (p.D % 8 != 0) return false;
    const int64_t s[9] = {p.qb, p.qh, p.qt, p.kb, p.kh, p.ks, p.vb, p.vh, p.vs};
    for (const int64_t x : s)
        if (x % 8 != 0) return false;
    return aligned(p.q, 16) && aligned(p.k, 16) && aligned(p.v, 16);
}

template <typename T>
static int launch_attn_stream_for(const AttnParams& p, void* stream) {
    if (p.D == 64) return launch_attn_stream<T, 64, true>(p, stream);
    if (p.D == 96) return launch_attn_stream<T, 96, true>(p, stream);
    if (p.D == 128) return launch_attn_stream<T, 128, true>(p, stream);
    if (p.D < 64) return launch_attn_stream<T, 64, false>(p, stream);
    if (p.D < 128) return p.D < 96 ? launch_attn_stream<T, 96, false>(p, stream) : launch_attn_stream<T, 128, false>(p, stream);
    return launch_attn_stream<T, 256, false>(p, stream);
}

}  // namespace bt

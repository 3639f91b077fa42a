// Beam search's selection: the n best of beams x vocabulary by score + log softmax(logits).
//
// Within a beam the candidates rank by their logits, so one pass over the logits is enough: beam_scan gives every CTA
// one piece of a row, held in registers, and leaves the piece's maximum, its sum of exponentials and its n largest
// logits; beam_join makes the log-sums and ranks the survivors of all beams in float64.  32 x 8 rows of 100003 16-bit logits:
// scan 30 us, join 11 us (a copy's time for the logits is 7.8 us): bound by the selection's instructions in the scan and by
// the float64 exponentials and logarithms in the join.
//
// The n largest of a piece: 16 or 64 groups of threads have a maximum each, and the n-th of those bounds the
// n-th of the piece from below.  What is not below it is collected and ranked by counting: with independent logits a
// little more than n.  A logit and its place make one 64-bit key (larger logit first, then the lower place), so that no
// two are equal.  A plateau of equal logits can pass the bound in any number; a list that overflows is abandoned for n
// searches of the largest key below the last.
//
// A row's elements go to threads by their place in the row, whatever the row's alignment (a misaligned row is read in
// aligned 16-byte words and shifted): equal rows have equal sums, so that ties between beams are ties.  Exponentials and
// their sums within a warp are float32, float64 from there.  With u = 2^-24 a log-sum is off by at most 54 u = 3.3e-6: an
// exponent y by 3 u |y| (difference, factor, product), which over a warp's 1024 terms, the largest at y = 0, is worth 13 u of
// their sum (the mean of |y| by weight is at most 6.4); an exponential by 2 ulp, 4 u; a term goes through at most 36 additions
// (31 of its thread one after the other, 5 of the warp).  Seen on a B200: 2.1e-7 (rows of one to five large logits,
// flat and random rows).  Within a beam the order is exact, between beams it is that of candidates with such an error.
#pragma once

#include "cache_common.cuh"
#include "cache_evict.cuh"   // ordered_key

namespace bt {

constexpr int BS_THREADS = 256;
constexpr int BS_WARPS = BS_THREADS / 32;
constexpr int BS_WORDS = 4;                                        // 16-byte words of a thread
constexpr int BS_LIST = 1024;
// Groups of neighbouring threads whose maxima bound the n-th largest of a piece: at least n, and as few as that allows,
// since all are compared with all.
constexpr int BS_FEW_GROUPS = 16, BS_GROUPS = 64;
static_assert(BS_GROUPS >= BT_BEAM_MAX_SELECT, "the n-th group maximum must exist");
template <typename T> __host__ __device__ constexpr int bs_per_word() { return 16 / static_cast<int>(sizeof(T)); }
template <typename T> __host__ __device__ constexpr int bs_piece() { return BS_THREADS * BS_WORDS * bs_per_word<T>(); }
constexpr int BJ_LIST = 1024;                                      // candidates that beam_join ranks by counting

struct BeamParams {
    const void* logits;
    int64_t ld_b, ld_w;
    const float* scores;
    const uint8_t* finished;
    int64_t end_token, V;
    int W, n, pieces;
    unsigned long long* keys;                                      // [B * W][pieces][n], largest first, 0: none
    float* piece_max;                                              // [B * W][pieces]
    double* piece_sum;
    float* out_scores;
    int64_t* out_tokens;
    int64_t* out_parents;
};

__device__ __forceinline__ float key_value(uint32_t u) { return __uint_as_float((u & 0x80000000u) ? u & 0x7fffffffu : ~u); }
__device__ __forceinline__ bool beam_live(const BeamParams& p, int64_t row) {
    const float s = p.scores[row];
    return !(p.finished && p.finished[row]) && s - s == 0.0f;
}
__device__ __forceinline__ double warp_add_double(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const long long bits = __double_as_longlong(v);
        const int lo = __shfl_xor_sync(0xffffffffu, static_cast<int>(bits & 0xffffffffll), o);
        const int hi = __shfl_xor_sync(0xffffffffu, static_cast<int>(bits >> 32), o);
        v += __longlong_as_double((static_cast<long long>(hi) << 32) | static_cast<unsigned int>(lo));
    }
    return v;
}

// The 16 bytes from `shift` (bytes, even) of the 32 in lo, hi
__device__ __forceinline__ uint4 shifted_word(uint4 lo, uint4 hi, int shift) {
    uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    if (shift & 8) {
#pragma unroll
        for (int i = 0; i < 6; ++i) w[i] = w[i + 2];
    }
    if (shift & 4) {
#pragma unroll
        for (int i = 0; i < 5; ++i) w[i] = w[i + 1];
    }
    if (shift & 2) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (w[i] >> 16) | (w[i + 1] << 16);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
template <typename T>
__device__ __forceinline__ void widen_word(uint4 w, float* x);
template <>
__device__ __forceinline__ void widen_word<float>(uint4 w, float* x) {
    x[0] = __uint_as_float(w.x); x[1] = __uint_as_float(w.y); x[2] = __uint_as_float(w.z); x[3] = __uint_as_float(w.w);
}
template <>
__device__ __forceinline__ void widen_word<__nv_bfloat16>(uint4 w, float* x) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = __uint_as_float(v[i] << 16);
        x[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    }
}
template <>
__device__ __forceinline__ void widen_word<__half>(uint4 w, float* x) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = *reinterpret_cast<const __half2*>(&v[i]);
        x[2 * i] = __low2float(h);
        x[2 * i + 1] = __high2float(h);
    }
}
// Largest element of a word so far; a NaN is dropped.  16-bit types: two at a time, `acc` holds the even and odd places.
template <typename T> struct WordMax;
template <> struct WordMax<float> {
    float m = -INFINITY;
    __device__ __forceinline__ void add(uint4 w) {
        m = fmaxf(fmaxf(m, __uint_as_float(w.x)), fmaxf(__uint_as_float(w.y), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w))));
    }
    __device__ __forceinline__ float get() const { return m; }
};
#ifdef BT_SIMT_HOST
template <typename T> struct WordMax {
    float m = -INFINITY;
    void add(uint4 w) {
        float x[8];
        widen_word<T>(w, x);
        for (int e = 0; e < 8; ++e) m = fmaxf(m, x[e]);
    }
    float get() const { return m; }
};
#else
template <> struct WordMax<__nv_bfloat16> {
    __nv_bfloat162 m = __float2bfloat162_rn(-INFINITY);
    __device__ __forceinline__ void add(uint4 w) {
        const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w);
        m = __hmax2(__hmax2(m, h[0]), __hmax2(__hmax2(h[1], h[2]), h[3]));
    }
    __device__ __forceinline__ float get() const { return fmaxf(__low2float(m), __high2float(m)); }
};
template <> struct WordMax<__half> {
    __half2 m = __float2half2_rn(-INFINITY);
    __device__ __forceinline__ void add(uint4 w) {
        const __half2* h = reinterpret_cast<const __half2*>(&w);
        m = __hmax2(__hmax2(m, h[0]), __hmax2(__hmax2(h[1], h[2]), h[3]));
    }
    __device__ __forceinline__ float get() const { return fmaxf(__low2float(m), __high2float(m)); }
};
#endif
// A word of which elements [0, valid) come from memory and the rest are -infinity
template <typename T>
__device__ __forceinline__ uint4 partial_word(const T* x, int64_t valid) {
    union { T e[bs_per_word<T>()]; uint4 w; } u;
    for (int i = 0; i < bs_per_word<T>(); ++i) u.e[i] = i < valid ? x[i] : from_float<T>(-INFINITY);
    return u.w;
}
// Words as the row has them, whatever its alignment: word `wi` is elements [wi * PER, +PER).  This form for the row's ends.
template <typename T>
__device__ __noinline__ uint4 row_word_at_end(const T* x0, int64_t V, int64_t wi) {
    const int64_t v = wi * bs_per_word<T>();
    return v < V ? partial_word<T>(x0 + v, V - v) : partial_word<T>(x0, 0);
}
// Makes the compiler forget what it derived from the word: keeping 32 widened values instead of 16 packed ones would
// halve the warps of an SM.
__device__ __forceinline__ void keep_packed(uint4& w) {
#ifndef BT_SIMT_HOST
    asm volatile("" : "+r"(w.x), "+r"(w.y), "+r"(w.z), "+r"(w.w));
#endif
}
__device__ __forceinline__ unsigned long long logit_key(float x, int64_t v) {
    return (static_cast<unsigned long long>(ordered_key(x != x ? -INFINITY : x)) << 32) | (0xffffffffu - static_cast<uint32_t>(v));
}

template <typename T, int GROUPS>
__global__ void __launch_bounds__(BS_THREADS, 6) beam_scan_kernel(const BeamParams p) {
    constexpr int PER = bs_per_word<T>(), PIECE = bs_piece<T>();
    __shared__ unsigned long long s_list[BS_LIST];
    __shared__ float s_sum[BS_WARPS];
    __shared__ float s_max[BS_WARPS], s_group[GROUPS];
    __shared__ unsigned long long s_best[BS_WARPS];
    __shared__ float s_edge;
    __shared__ int s_count;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t row = blockIdx.x / static_cast<unsigned>(p.pieces);
    const int piece = static_cast<int>(blockIdx.x - static_cast<unsigned>(row) * p.pieces);
    if (tid == 0) s_count = 0;
    pdl_launch_dependents();
    pdl_wait();
    const bool live = beam_live(p, row);
    const int b = static_cast<int>(row) / p.W;
    const T* x0 = static_cast<const T*>(p.logits) + b * p.ld_b + (static_cast<int>(row) - b * p.W) * p.ld_w;
    const int64_t v0 = static_cast<int64_t>(piece) * PIECE;
    const int64_t w0 = v0 / PER + tid;                             // this thread's first word; the others follow at BS_THREADS

    const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(x0) & 15);
    const uint4* words = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(x0) - shift);
    uint4 word[BS_WORDS];
#pragma unroll
    for (int i = 0; i < BS_WORDS; ++i) {
        const int64_t wi = w0 + i * BS_THREADS;
        // a shifted word takes bytes of two aligned ones, all of which have to lie in the row
        if (shift == 0 && (wi + 1) * PER <= p.V) word[i] = words[wi];
        else if (wi > 0 && (wi + 2) * PER <= p.V) word[i] = shifted_word(words[wi], words[wi + 1], shift);
        else word[i] = row_word_at_end<T>(x0, p.V, wi);
    }
    if (!live) return;                                             // for every thread of the CTA; beam_join knows
    WordMax<T> top;
#pragma unroll
    for (int i = 0; i < BS_WORDS; ++i) top.add(word[i]);
    const float mine = top.get();
    constexpr int MEMBERS = BS_THREADS / GROUPS;
    float mx = mine;
#pragma unroll
    for (int o = 1; o < MEMBERS; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if ((lane & (MEMBERS - 1)) == 0) s_group[tid / MEMBERS] = mx;
    mx = warp_max(mx);
    __syncthreads();
    {   // the n-th largest group maximum: a group's threads compare it with all, GROUPS / MEMBERS each
        const float a = s_group[tid / MEMBERS];
        int above = 0, level = 0;
#pragma unroll
        for (int i = 0; i < GROUPS / MEMBERS; ++i) {
            const float x = s_group[(tid & (MEMBERS - 1)) * (GROUPS / MEMBERS) + i];
            above += x > a;
            level += x >= a;
        }
#pragma unroll
        for (int o = 1; o < MEMBERS; o <<= 1) {
            above += __shfl_xor_sync(0xffffffffu, above, o);
            level += __shfl_xor_sync(0xffffffffu, level, o);
        }
        if (above < p.n && level >= p.n) s_edge = a;               // groups that tie here write the same value
    }
    float sum = 0.0f;
    if (mx - mx == 0.0f) {                                         // finite
#pragma unroll
        for (int i = 0; i < BS_WORDS; ++i) {
            float x[PER];
            keep_packed(word[i]);
            widen_word<T>(word[i], x);
#pragma unroll
            for (int e = 0; e < PER; ++e) sum += exp2_fast((fmaxf(x[e], -INFINITY) - mx) * 1.4426950408889634f);     // a NaN adds 0
        }
    }
    sum = warp_add(sum);
    if (lane == 0) {
        s_sum[warp] = sum;
        s_max[warp] = mx;
    }
    __syncthreads();
    const float edge = s_edge;
    if (mine >= edge && mine > -INFINITY) {
#pragma unroll
        for (int i = 0; i < BS_WORDS; ++i) {
            keep_packed(word[i]);
            WordMax<T> here;
            here.add(word[i]);
            if (!(here.get() >= edge)) continue;
            float x[PER];
            widen_word<T>(word[i], x);
#pragma unroll
            for (int e = 0; e < PER; ++e)
                if (x[e] >= edge && x[e] > -INFINITY) {
                    const int at = atomicAdd(&s_count, 1);
                    if (at < BS_LIST) s_list[at] = logit_key(x[e], (w0 + i * BS_THREADS) * PER + e);
                }
        }
    }
    __syncthreads();
    const int count = s_count;
    unsigned long long* out = p.keys + (row * p.pieces + piece) * p.n;
    if (warp == 0) {                                               // the warps' sums become one, a lane per warp
        const float m_w = lane < BS_WARPS ? s_max[lane] : -INFINITY, m = warp_max(m_w);
        double all = 0.0;
        if (lane < BS_WARPS && m - m == 0.0f && s_sum[lane] > 0.0)
            all = static_cast<double>(s_sum[lane]) * exp2(1.4426950408889634 * (static_cast<double>(m_w) - static_cast<double>(m)));
        all = warp_add_double(all);
        if (lane == 0) {
            p.piece_max[row * p.pieces + piece] = m;
            p.piece_sum[row * p.pieces + piece] = all;
        }
    }
    if (count <= BS_LIST) {
        for (int i = tid; i < count; i += BS_THREADS) {
            const unsigned long long key = s_list[i];
            int rank = 0;
            for (int j = 0; j < count; ++j) rank += s_list[j] > key;
            if (rank < p.n) out[rank] = key;
        }
        // Fewer than n numbers above -infinity: the lowest places among the others come next, and as only `count` places
        // hold a number, they are found among the first n.
        if (count < p.n && warp == BS_WARPS - 1) {
            int at = count;
            for (int i0 = 0; i0 < p.n; i0 += 32) {
                const int64_t v = v0 + i0 + lane;
                const float x = i0 + lane < p.n && v < p.V ? to_float<T>(x0[v]) : 0.0f;
                const bool low = !(x > -INFINITY);
                const unsigned mask = __ballot_sync(0xffffffffu, low);
                const int to = at + __popc(mask & ((1u << lane) - 1));
                if (low && to < p.n) out[to] = logit_key(x, v);
                at += __popc(mask);
            }
            for (int i = at + lane; i < p.n; i += 32) out[i] = 0;  // the row ends before that
        }
        return;
    }
    unsigned long long last = ~0ull;
    for (int k = 0; k < p.n; ++k) {
        unsigned long long best = 0;
#pragma unroll
        for (int i = 0; i < BS_WORDS; ++i) {
            float x[PER];
            keep_packed(word[i]);
            widen_word<T>(word[i], x);
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                const int64_t v = (w0 + i * BS_THREADS) * PER + e;
                const unsigned long long key = v < p.V ? logit_key(x[e], v) : 0;
                if (key < last && key > best) best = key;
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned hi = __shfl_xor_sync(0xffffffffu, static_cast<unsigned>(best >> 32), o);
            const unsigned lo = __shfl_xor_sync(0xffffffffu, static_cast<unsigned>(best), o);
            const unsigned long long other = (static_cast<unsigned long long>(hi) << 32) | lo;
            if (other > best) best = other;
        }
        if (lane == 0) s_best[warp] = best;
        __syncthreads();
        last = s_best[0];
        for (int i = 1; i < BS_WARPS; ++i) last = s_best[i] > last ? s_best[i] : last;
        if (tid == 0) out[k] = last;
        __syncthreads();
    }
}

struct Candidate {
    double score;
    int64_t place;                                                 // w * V + v, or -1: none
    __device__ __forceinline__ bool better(const Candidate& o) const {
        if (place < 0 || o.place < 0) return place >= 0 && o.place < 0;
        return score > o.score || (score == o.score && place < o.place);
    }
};

// Entry e of the list that piece `piece` of beam w left.  (One copy of the code: what a kernel this short spends most of its
// time on is fetching its instructions.)
__device__ __noinline__ Candidate beam_candidate(const BeamParams& p, int64_t b, int w, int piece, int e, const double* s_base,
                                                    const uint8_t* s_kind) {
    Candidate c = {-INFINITY, -1};
    int64_t token;
    if (s_kind[w] == 0) {                                          // live: what beam_scan left
        const unsigned long long key = p.keys[((b * p.W + w) * p.pieces + piece) * p.n + e];
        if (key == 0) return c;
        token = 0xffffffffu - static_cast<uint32_t>(key);
        c.score = s_base[w] + static_cast<double>(key_value(static_cast<uint32_t>(key >> 32)));
    } else {                                                       // no ranking of its own: its lowest tokens, at -infinity
        if (piece != 0) return c;
        token = e;
        if (s_kind[w] == 1) {                                      // finished: the end token first, at the beam's score
            token = e == 0 ? p.end_token : e - 1 < p.end_token ? e - 1 : e;
            if (e == 0) c.score = s_base[w];
        }
        if (token >= p.V) return c;
    }
    c.place = w * p.V + token;
    return c;
}

constexpr int BJ_THREADS = 256;

__global__ void __launch_bounds__(BJ_THREADS) beam_join_kernel(const __grid_constant__ BeamParams p) {
    __shared__ double s_base[BT_BEAM_MAX_BEAMS];                   // score - log-sum
    __shared__ uint8_t s_kind[BT_BEAM_MAX_BEAMS];                  // 0 live, 1 finished, 2 nothing but -infinity
    __shared__ Candidate s_best[BJ_THREADS];
    __shared__ Candidate s_list[BJ_LIST];
    __shared__ Candidate s_edge;
    __shared__ int s_count;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, b = blockIdx.x;
    if (tid == 0) s_count = 0, s_edge = {-INFINITY, -1};
    pdl_launch_dependents();
    pdl_wait();
    for (int w = warp; w < p.W; w += BJ_THREADS / 32) {
        const int64_t row = static_cast<int64_t>(b) * p.W + w;
        const float score = p.scores[row];
        if (!beam_live(p, row)) {
            if (lane == 0) {
                s_base[w] = score;
                s_kind[w] = p.finished && p.finished[row] && score == score ? 1 : 2;
            }
            continue;
        }
        float m = -INFINITY;
        for (int i = lane; i < p.pieces; i += 32) m = fmaxf(m, p.piece_max[row * p.pieces + i]);
        m = warp_max(m);
        double sum = 0.0;
        if (m - m == 0.0f)
            for (int i = lane; i < p.pieces; i += 32) {
                const double s = p.piece_sum[row * p.pieces + i];
                if (s > 0.0) sum += s * exp(static_cast<double>(p.piece_max[row * p.pieces + i]) - static_cast<double>(m));
            }
        sum = warp_add_double(sum);
        if (lane == 0) {
            s_kind[w] = m - m == 0.0f ? 0 : 2;
            s_base[w] = static_cast<double>(score) - (static_cast<double>(m) + log(sum));
        }
    }
    __syncthreads();
    // Lists are sorted, so a thread that owns some of them knows its best from their heads.  With at least n threads, the
    // n-th best of those bounds the n-th best of all from below.
    const unsigned lists = static_cast<unsigned>(p.W) * p.pieces;
    Candidate best = {-INFINITY, -1};
    for (unsigned i = tid; i < lists; i += BJ_THREADS) {
        const Candidate c = beam_candidate(p, b, i / p.pieces, i % p.pieces, 0, s_base, s_kind);
        if (c.better(best)) best = c;
    }
    s_best[tid] = best;
    __syncthreads();
    if (best.place >= 0) {
        const int heads = lists < BJ_THREADS ? lists : BJ_THREADS;
        int above = 0;
        for (int i = 0; i < heads; ++i) above += s_best[i].better(best);
        if (above == p.n - 1) s_edge = best;
    }
    __syncthreads();
    const Candidate edge = s_edge;
    for (unsigned i = tid; i < lists * p.n; i += BJ_THREADS) {
        const unsigned list = i / p.n, w = list / p.pieces;
        const Candidate c = beam_candidate(p, b, w, list - w * p.pieces, i - list * p.n, s_base, s_kind);
        if (c.place < 0 || edge.better(c)) continue;
        const int at = atomicAdd(&s_count, 1);
        if (at < BJ_LIST) s_list[at] = c;
    }
    __syncthreads();
    const int64_t out = static_cast<int64_t>(b) * p.n;
    const int count = s_count;
    if (count <= BJ_LIST) {
        for (int i = tid; i < count; i += BJ_THREADS) {
            const Candidate c = s_list[i];
            int rank = 0;
            for (int j = 0; j < count; ++j) rank += s_list[j].better(c);
            if (rank < p.n) {
                p.out_scores[out + rank] = static_cast<float>(c.score);
                const int64_t w = c.place / p.V;
                p.out_tokens[out + rank] = c.place - w * p.V;
                p.out_parents[out + rank] = w;
            }
        }
        return;
    }
    // More candidates above the edge than the list holds (fewer lists than n, or many whose best are all in a few): the
    // best below the last one, n times.
    Candidate last = {INFINITY, -1};
    for (int k = 0; k < p.n; ++k) {
        Candidate mine = {-INFINITY, -1};
        for (unsigned i = tid; i < lists; i += BJ_THREADS)
            for (int e = 0; e < p.n; ++e) {
                const Candidate c = beam_candidate(p, b, i / p.pieces, i % p.pieces, e, s_base, s_kind);
                if (c.place < 0) break;
                if (k > 0 && !last.better(c)) continue;            // taken already
                if (c.better(mine)) mine = c;
                break;
            }
        __syncthreads();
        s_best[tid] = mine;
        __syncthreads();
        last = s_best[0];
        for (int i = 1; i < BJ_THREADS; ++i)
            if (s_best[i].better(last)) last = s_best[i];
        if (tid == 0) {
            p.out_scores[out + k] = static_cast<float>(last.score);
            p.out_tokens[out + k] = last.place % p.V;
            p.out_parents[out + k] = last.place / p.V;
        }
    }
}

struct BeamPlan {
    int pieces;
    size_t keys, sums, maxima;
    size_t bytes() const { return keys + sums + maxima; }
};
static BeamPlan beam_plan(int64_t B, int64_t W, int64_t V, int dtype, int64_t n) {
    BeamPlan a;
    a.pieces = static_cast<int>(ceil_div<int64_t>(V, dtype == BT_F32 ? bs_piece<float>() : bs_piece<__half>()));
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    const size_t all = static_cast<size_t>(B) * W * a.pieces;
    a.keys = up(all * n * 8);
    a.sums = up(all * 8);
    a.maxima = up(all * 4);
    return a;
}
template <typename T>
static int launch_beam_scan(const BeamParams& p, dim3 grid, void* stream) {
    if (p.n <= BS_FEW_GROUPS) return launch_early(beam_scan_kernel<T, BS_FEW_GROUPS>, "beam_scan_kernel", grid, BS_THREADS, 0, stream, p);
    return launch_early(beam_scan_kernel<T, BS_GROUPS>, "beam_scan_kernel", grid, BS_THREADS, 0, stream, p);
}
static bool beam_sizes_ok(int64_t B, int64_t W, int64_t V, int64_t n) {
    return B > 0 && W > 0 && V > 0 && n > 0 && (V >= n || n <= W * V);
}
static bool beam_sizes_supported(int64_t B, int64_t W, int64_t V, int64_t n) {
    return W <= BT_BEAM_MAX_BEAMS && n <= BT_BEAM_MAX_SELECT && V <= (int64_t{1} << 30) && B <= (int64_t{1} << 30) / W / (V / 4096 + 1);
}

}  // namespace bt

extern "C" size_t bt_beam_select_workspace(int64_t B, int64_t W, int64_t V, int dtype, int64_t n) {
    using namespace bt;
    if (!valid_dtype(dtype) || !beam_sizes_ok(B, W, V, n) || !beam_sizes_supported(B, W, V, n)) return 0;
    return beam_plan(B, W, V, dtype, n).bytes();
}

extern "C" int bt_beam_select(const void* logits, int dtype, int64_t B, int64_t W, int64_t V, int64_t ld_b, int64_t ld_w,
                              const float* scores, const uint8_t* finished, int64_t end_token, int64_t n, float* out_scores,
                              int64_t* out_tokens, int64_t* out_parents, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace bt;
    BT_REQUIRE(logits && scores && out_scores && out_tokens && out_parents && workspace, "bt_beam_select: NULL pointer");
    BT_REQUIRE(valid_dtype(dtype), "bt_beam_select: unknown dtype %d", dtype);
    BT_REQUIRE(beam_sizes_ok(B, W, V, n), "bt_beam_select: empty input, or more selected than there are candidates");
    BT_REQUIRE(finished == nullptr || (end_token >= 0 && end_token < V), "bt_beam_select: end token %lld outside the vocabulary", (long long)end_token);
    BT_UNSUPPORTED_IF(!beam_sizes_supported(B, W, V, n), "bt_beam_select: at most %d beams and %d selected", BT_BEAM_MAX_BEAMS, BT_BEAM_MAX_SELECT);
    BT_REQUIRE(aligned(logits, dtype_size(dtype)) && aligned(workspace, 16), "bt_beam_select: misaligned pointer");
    const BeamPlan plan = beam_plan(B, W, V, dtype, n);
    BT_REQUIRE(workspace_bytes >= plan.bytes(), "bt_beam_select: workspace of %zu bytes, %zu needed", workspace_bytes, plan.bytes());
    BeamParams p = {};
    p.logits = logits; p.ld_b = ld_b; p.ld_w = ld_w; p.scores = scores; p.finished = finished; p.end_token = end_token; p.V = V;
    p.W = static_cast<int>(W); p.n = static_cast<int>(n); p.pieces = plan.pieces;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    p.keys = reinterpret_cast<unsigned long long*>(ws);
    p.piece_sum = reinterpret_cast<double*>(ws + plan.keys);
    p.piece_max = reinterpret_cast<float*>(ws + plan.keys + plan.sums);
    p.out_scores = out_scores; p.out_tokens = out_tokens; p.out_parents = out_parents;
    const dim3 grid(static_cast<unsigned>(B * W * plan.pieces));
    int rc;
    if (dtype == BT_F32) rc = launch_beam_scan<float>(p, grid, stream);
    else if (dtype == BT_F16) rc = launch_beam_scan<__half>(p, grid, stream);
    else rc = launch_beam_scan<__nv_bfloat16>(p, grid, stream);
    if (rc != BT_OK) return rc;
    return launch_early(beam_join_kernel, "beam_join_kernel", dim3(static_cast<unsigned>(B)), BJ_THREADS, 0, stream, p);
}

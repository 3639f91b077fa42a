// Beam search's selection: the n best of beams x vocabulary by score + log softmax(logits).
//
// Within a beam the candidates rank by their logits, so one pass over the logits is enough: beam_scan gives every CTA
// one piece of a row, held in registers, and leaves the piece's maximum, its sum of exponentials and its n largest
// logits; beam_join makes the log-sums and ranks the survivors of all beams in float64.  Bound by HBM (the logits).
//
// The n largest of a piece: a logit and its place make one 64-bit key (larger logit first, then the lower place), so no
// two are equal.  Every thread's largest key is compared with all others; the n-th of those bounds the n-th of the
// piece from below, and only the n threads above it can hold more: at most n x 32 keys are collected and ranked by
// counting, usually little more than n.
//
// A row's elements go to threads by their place in the row, whatever the row's alignment (a misaligned row is read in
// aligned 16-byte words and shifted): equal rows have equal sums, so that ties between beams are ties.
#pragma once

#include "cache_common.cuh"
#include "cache_evict.cuh"   // ordered_key

namespace bt {

constexpr int BS_THREADS = 256;
constexpr int BS_WORDS = 4;                                        // 16-byte words of a thread
template <typename T> __host__ __device__ constexpr int bs_per_word() { return 16 / static_cast<int>(sizeof(T)); }
template <typename T> __host__ __device__ constexpr int bs_piece() { return BS_THREADS * BS_WORDS * bs_per_word<T>(); }
constexpr int BJ_LIST = 2048;                                      // candidates that beam_join ranks by counting

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

template <typename T>
__global__ void __launch_bounds__(BS_THREADS) beam_scan_kernel(const BeamParams p) {
    constexpr int PER = bs_per_word<T>(), E = BS_WORDS * PER, PIECE = bs_piece<T>();
    __shared__ unsigned long long s_best[BS_THREADS];
    __shared__ unsigned long long s_list[BT_BEAM_MAX_SELECT * E];
    __shared__ double s_sum[BS_THREADS / 32];
    __shared__ float s_max[BS_THREADS / 32];
    __shared__ unsigned long long s_edge;
    __shared__ int s_count;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int64_t row = blockIdx.x / p.pieces;
    const int piece = static_cast<int>(blockIdx.x % p.pieces);
    if (tid == 0) s_count = 0, s_edge = 0;
    pdl_launch_dependents();
    pdl_wait();
    if (!beam_live(p, row)) return;                                // for every thread of the CTA; beam_join knows
    const T* x0 = static_cast<const T*>(p.logits) + row / p.W * p.ld_b + row % p.W * p.ld_w;
    const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(x0) & 15);
    const uint4* words = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(x0) - shift);
    const int64_t v0 = static_cast<int64_t>(piece) * PIECE;

    float x[E];
    unsigned long long best = 0;
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < BS_WORDS; ++i) {
        const int64_t v = v0 + (static_cast<int64_t>(i) * BS_THREADS + tid) * PER;     // first element of the word
        const int64_t wi = v / PER;
        if (v + PER <= p.V && (shift == 0 || (wi > 0 && v + 2 * PER <= p.V))) {         // all bytes read lie in the row
            const uint4 lo = words[wi];
            widen_word<T>(shift == 0 ? lo : shifted_word(lo, words[wi + 1], shift), x + i * PER);
        } else {
#pragma unroll
            for (int e = 0; e < PER; ++e) x[i * PER + e] = v + e < p.V ? to_float<T>(x0[v + e]) : -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            float& f = x[i * PER + e];
            if (f != f) f = -INFINITY;                             // a NaN is never better than a number
            mx = fmaxf(mx, f);
            if (v + e < p.V) {
                const unsigned long long key = (static_cast<unsigned long long>(ordered_key(f)) << 32) | (0xffffffffu - static_cast<uint32_t>(v + e));
                if (key > best) best = key;
            }
        }
    }
    s_best[tid] = best;
    mx = warp_max(mx);
    if (lane == 0) s_max[warp] = mx;
    __syncthreads();
    mx = s_max[0];
#pragma unroll
    for (int i = 1; i < BS_THREADS / 32; ++i) mx = fmaxf(mx, s_max[i]);
    float sum = 0.0f;
    if (mx - mx == 0.0f) {                                         // finite
#pragma unroll
        for (int e = 0; e < E; ++e) sum += expf(x[e] - mx);
    }
    const double total = warp_add_double(static_cast<double>(sum));
    if (lane == 0) s_sum[warp] = total;
    // the n-th largest of the threads' best keys
    int above = 0;
    for (int i = 0; i < BS_THREADS; ++i) above += s_best[i] > best;
    if (above == p.n - 1 && best != 0) s_edge = best;
    __syncthreads();
    const unsigned long long edge = s_edge;                        // 0: fewer than n threads hold anything
    if (best >= edge && best != 0) {
#pragma unroll
        for (int i = 0; i < BS_WORDS; ++i)
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                const int64_t v = v0 + (static_cast<int64_t>(i) * BS_THREADS + tid) * PER + e;
                const unsigned long long key = (static_cast<unsigned long long>(ordered_key(x[i * PER + e])) << 32) | (0xffffffffu - static_cast<uint32_t>(v));
                if (v < p.V && key >= edge) s_list[atomicAdd(&s_count, 1)] = key;
            }
    }
    __syncthreads();
    const int count = s_count;
    unsigned long long* out = p.keys + (row * p.pieces + piece) * p.n;
    for (int i = tid; i < count; i += BS_THREADS) {
        const unsigned long long key = s_list[i];
        int rank = 0;
        for (int j = 0; j < count; ++j) rank += s_list[j] > key;
        if (rank < p.n) out[rank] = key;
    }
    for (int i = count + tid; i < p.n; i += BS_THREADS) out[i] = 0;
    if (tid == 0) {
        double all = 0.0;
#pragma unroll
        for (int i = 0; i < BS_THREADS / 32; ++i) all += s_sum[i];
        p.piece_max[row * p.pieces + piece] = mx;
        p.piece_sum[row * p.pieces + piece] = all;
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

// Survivor `i` of a sequence: entry i % n of piece i / n % pieces of beam i / n / pieces
__device__ __forceinline__ Candidate beam_candidate(const BeamParams& p, int b, int64_t i, const double* s_base, const uint8_t* s_kind) {
    const int e = static_cast<int>(i % p.n), piece = static_cast<int>(i / p.n % p.pieces), w = static_cast<int>(i / p.n / p.pieces);
    Candidate c = {-INFINITY, -1};
    int64_t token;
    if (s_kind[w] == 0) {                                          // live: what beam_scan left
        const unsigned long long key = p.keys[((static_cast<int64_t>(b) * p.W + w) * p.pieces + piece) * p.n + e];
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

__global__ void __launch_bounds__(BJ_THREADS) beam_join_kernel(const BeamParams p) {
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
    const int64_t total = static_cast<int64_t>(p.W) * p.pieces * p.n;
    Candidate best = {-INFINITY, -1};
    for (int64_t i = tid; i < total; i += BJ_THREADS) {
        const Candidate c = beam_candidate(p, b, i, s_base, s_kind);
        if (c.better(best)) best = c;
    }
    s_best[tid] = best;
    __syncthreads();
    int above = 0;
    for (int i = 0; i < BJ_THREADS; ++i) above += s_best[i].better(best);
    if (above == p.n - 1 && best.place >= 0) s_edge = best;
    __syncthreads();
    const Candidate edge = s_edge;
    for (int64_t i = tid; i < total; i += BJ_THREADS) {
        const Candidate c = beam_candidate(p, b, i, s_base, s_kind);
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
                p.out_tokens[out + rank] = c.place % p.V;
                p.out_parents[out + rank] = c.place / p.V;
            }
        }
        return;
    }
    // More candidates above the edge than the list holds (many pieces whose best are all in a few of them): the best
    // below the last one, n times.
    Candidate last = {INFINITY, -1};
    for (int k = 0; k < p.n; ++k) {
        Candidate mine = {-INFINITY, -1};
        for (int64_t i = tid; i < total; i += BJ_THREADS) {
            const Candidate c = beam_candidate(p, b, i, s_base, s_kind);
            if ((k == 0 || last.better(c)) && c.better(mine)) mine = c;
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
    if (dtype == BT_F32) rc = launch_early(beam_scan_kernel<float>, "beam_scan_kernel", grid, BS_THREADS, 0, stream, p);
    else if (dtype == BT_F16) rc = launch_early(beam_scan_kernel<__half>, "beam_scan_kernel", grid, BS_THREADS, 0, stream, p);
    else rc = launch_early(beam_scan_kernel<__nv_bfloat16>, "beam_scan_kernel", grid, BS_THREADS, 0, stream, p);
    if (rc != BT_OK) return rc;
    return launch_early(beam_join_kernel, "beam_join_kernel", dim3(static_cast<unsigned>(B)), BJ_THREADS, 0, stream, p);
}

/*
 * bittorch_b200 - C ABI of the operators over a decoder's key/value cache.
 *
 * Same library and conventions as bittorch_b200.h (device pointers, sizes, a stream,
 * an integer status with bt_last_error(); nothing allocates, synchronises, throws or
 * traps).  A cache tensor is [B, Hkv, S, D] with contiguous D and any other strides,
 * which are given in ELEMENTS; arrays marked "host" are read before the call returns.
 * No counterpart in the reference, whose runtime attends over plain arrays
 * (js/src/models/TernaryTransformer.ts:366-464).
 *
 * Lengths: int32 or int64 device vectors (`*_i64` says which); element b is read at
 * index b * stride, stride 0 gives every sequence the same length.  Values outside
 * [0, S] are clamped to it.
 */
#ifndef BITTORCH_B200_CACHE_H
#define BITTORCH_B200_CACHE_H

#include "bittorch_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Most candidates that bt_beam_select returns per sequence, and most beams. */
#define BT_BEAM_MAX_SELECT 64
#define BT_BEAM_MAX_BEAMS 64
/* Most beams per group of bt_reorder_cache. */
#define BT_REORDER_MAX_BEAMS 32
/* Largest head size of bt_tree_attention. */
#define BT_ATTENTION_MAX_D 256

/*
 * Attention of T new tokens per sequence over a cache that already holds their keys and
 * values: sequence b has len = lengths[b] committed slots, and the new tokens sit in
 * slots len .. len+T-1 (slots from S on do not exist).  New token i sees slots < len and
 * the new tokens j with tree[b][i][j] != 0 (tree NULL: j <= i).
 *   s = scale * q . k;  p = softmax of s over the slots that are seen;  out = sum p v
 * Query head h reads key/value head h / (H / Hkv).  A token that sees nothing gives
 * zeros.  Slots that no token sees are never read into a result, whatever they hold.
 * Sums and softmax statistics are float32; with 16-bit types the weights are rounded to
 * that type for the product with the values.  Should a wait of the kernel run out (2 s), what
 * it could not write is NaN and bt_device_status() says BT_ERR_DEVICE_WAIT.
 *
 * q [B,H,T,D], k and v [B,Hkv,S,D], out [B,H,T,D], all of `dtype`;
 * strides  host int64[12]: q (b,h,t), k (b,h,s), v (b,h,s), out (b,h,t)
 * tree     uint8 [T,T] (tree_stride_b 0) or [B][T,T], or NULL
 * mass     float32 [B,Hkv,S] with strides (mass_sb, mass_sh, 1), or NULL:
 *          mass[b,h,n] += sum of p over the query heads of group h and the T tokens
 * workspace: bt_tree_attention_workspace() bytes, 16-byte aligned, not shared with a
 * call that may run at the same time; no initial contents needed.
 */
size_t bt_tree_attention_workspace(int64_t B, int64_t H, int64_t Hkv, int64_t T, int64_t S,
                                   int64_t D, int dtype, int want_mass);
int bt_tree_attention(const void* q, const void* k, const void* v, int dtype, int64_t B,
                      int64_t H, int64_t Hkv, int64_t T, int64_t S, int64_t D,
                      const int64_t* strides, const void* lengths, int lengths_i64,
                      int64_t lengths_stride, const uint8_t* tree, int64_t tree_stride_b,
                      float scale, float* mass, int64_t mass_sb, int64_t mass_sh, void* out,
                      void* workspace, size_t workspace_bytes, void* stream);

/*
 * Which slots of a cache to keep: for every sequence and key/value head the first
 * `sinks` slots, the last `recent` of its lengths[b] slots, and of the others those with
 * the largest mass (equal mass: the lowest slot; a NaN ranks below everything), `budget`
 * slots in all, in slot order.  A sequence of at most `budget` slots keeps them all.
 * mass float32 [B,Hkv,S], strides (mass_sb, mass_sh, 1)
 * keep int64 [B,Hkv,budget] (-1 from counts[b] on);  counts int64 [B] = min(length, budget)
 */
int bt_evict_select(const float* mass, int64_t mass_sb, int64_t mass_sh, int64_t B, int64_t Hkv,
                    int64_t S, const void* lengths, int lengths_i64, int64_t lengths_stride,
                    int64_t budget, int64_t sinks, int64_t recent, int64_t* keep,
                    int64_t* counts, void* stream);

/*
 * Gathers cache slots: destination slot first[b] + j takes source slot keep[b,h,j] for
 * j < counts[b], j < n (first NULL: 0); all other destination slots of k_out and v_out
 * stay as they are.  With k_out == k and v_out == v the cache is compacted in place;
 * then keep must ascend and keep[b,h,j] >= first[b] + j.  An entry outside [0, S) and a
 * destination outside [0, S_out) are skipped.
 * strides host int64[12]: k (b,h,s), v (b,h,s), k_out (b,h,s), v_out (b,h,s)
 * keep int64, strides (keep_sb, keep_sh, 1)
 * mass / mass_out (both or none): float32 [B,Hkv,S] / [B,Hkv,S_out], mass_strides host
 * int64[4]: mass (b,h), mass_out (b,h); gathered like the rows, and the slots of
 * mass_out from first[b] + counts[b] on are set to zero.
 */
int bt_compact_cache(const void* k, const void* v, void* k_out, void* v_out, int dtype, int64_t B,
                     int64_t Hkv, int64_t S, int64_t S_out, int64_t D, const int64_t* strides,
                     const int64_t* keep, int64_t keep_sb, int64_t keep_sh, int64_t n,
                     const int64_t* counts, const int64_t* first, const float* mass,
                     float* mass_out, const int64_t* mass_strides, void* stream);

/*
 * One step of beam search: of the candidates (beam w, token v) of sequence b with
 *   score = scores[b,w] + logits[b,w,v] - log(sum_u exp(logits[b,w,u]))
 * the `n` best, best first (equal scores: the lowest w * V + v).  The sums are ranked in
 * float64; the log is off by 3.3e-6 at most (float32 exponentials), so candidates of
 * different beams that are closer than this may change places.  A beam with finished[b,w] != 0 has one candidate, `end_token` with its score
 * unchanged; its others count as -infinity, as do those of a beam whose score is not
 * finite or whose logits have no finite maximum, and NaN logits.
 * logits [B,W,V] of `dtype`, strides (ld_b, ld_w, 1); scores float32 [B,W];
 * finished uint8 [B,W] or NULL
 * out_scores float32, out_tokens int64, out_parents int64, each [B,n]; n <= W * V
 */
size_t bt_beam_select_workspace(int64_t B, int64_t W, int64_t V, int dtype, int64_t n);
int bt_beam_select(const void* logits, int dtype, int64_t B, int64_t W, int64_t V, int64_t ld_b,
                   int64_t ld_w, const float* scores, const uint8_t* finished, int64_t end_token,
                   int64_t n, float* out_scores, int64_t* out_tokens, int64_t* out_parents,
                   void* workspace, size_t workspace_bytes, void* stream);

/*
 * Gives every beam its parent's cache rows, in place: slots [start, lengths[b]) of row
 * b * W + w become those that row b * W + parents[b,w] had before the call.  A parent
 * outside [0, W) leaves its beam as it is.  All `count` tensors [B*W, Hkv, S, D] have
 * the same sizes and type; none may overlap another.
 * tensors host array of device pointers; strides host int64[3 * count]: (row, head, slot)
 * parents int64 [B,W]
 */
int bt_reorder_cache(void* const* tensors, int64_t count, int dtype, int64_t B, int64_t W,
                     int64_t Hkv, int64_t S, int64_t D, const int64_t* strides,
                     const int64_t* parents, const void* lengths, int lengths_i64,
                     int64_t lengths_stride, int64_t start, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* BITTORCH_B200_CACHE_H */

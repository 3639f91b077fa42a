// libbt_simt_cache.so: the kernels over a key/value cache compiled for the CPU (see simt_host.h).  TEST INFRASTRUCTURE ONLY.
//
// Includes the real kernel files, so bt_tree_attention (the float32 kernel and the join), bt_evict_select,
// bt_compact_cache, bt_beam_select and bt_reorder_cache are exported with their usual signatures and take HOST pointers.
// Not built here: the tensor-core kernels of bt_tree_attention.
#include "simt_host.h"

// ---- primitives that simt_host.h does not have ---------------------------------------------------
inline int atomicAdd(int* p, int v) {
    static std::mutex mu;
    std::lock_guard<std::mutex> lock(mu);
    const int old = *p;
    *p = old + v;
    return old;
}
inline int __ffs(int v) { return __builtin_ffs(v); }
inline int __popc(unsigned v) { return __builtin_popcount(v); }
inline unsigned __ballot_sync(unsigned, bool on) {
    simt::Warp& w = simt::my_warp();
    w.xchg[simt::my_lane()] = on ? 1u : 0u;
    pthread_barrier_wait(&w.bar);
    unsigned r = 0;
    for (int i = 0; i < 32; ++i) r |= w.xchg[i] << i;
    pthread_barrier_wait(&w.bar);
    return r;
}
template <typename T> inline T __shfl_sync(unsigned, T v, int src) { return ::simt::shfl(v, src); }
template <typename T> inline T __shfl_up_sync(unsigned, T v, int by) { return ::simt::shfl(v, ::simt::my_lane() >= by ? ::simt::my_lane() - by : ::simt::my_lane()); }
template <typename T> inline T __shfl_down_sync(unsigned, T v, int by) { return ::simt::shfl(v, ::simt::my_lane() + by < 32 ? ::simt::my_lane() + by : ::simt::my_lane()); }
#ifndef __grid_constant__
#define __grid_constant__
#endif
#ifndef __noinline__
#define __noinline__ __attribute__((noinline))
#endif

#include <cstdarg>

#include "../../bittorch_b200/csrc/common.cuh"

namespace bt {

static thread_local char g_error[512] = "";

void set_error(const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_error, sizeof(g_error), fmt, ap);
    va_end(ap);
}

static int g_sm_count = 1;
int sm_count() { return g_sm_count; }
int tuning(int) { return -1; }

}  // namespace bt

#include "../../bittorch_b200/csrc/cache_attention.cuh"
#include "../../bittorch_b200/csrc/cache_evict.cuh"
#include "../../bittorch_b200/csrc/cache_reorder.cuh"
#include "../../bittorch_b200/csrc/beam_select.cuh"

extern "C" const char* bt_last_error(void) { return bt::g_error; }
extern "C" void simt_set_sm_count(int n) { bt::g_sm_count = n > 0 ? n : 1; }
extern "C" int simt_take_errors(char* text, size_t size) {
    std::lock_guard<std::mutex> lock(simt::error_mutex());
    const int n = simt::error_count().exchange(0);
    if (text != nullptr && size > 0) snprintf(text, size, "%s", simt::error_text());
    simt::error_text()[0] = 0;
    return n;
}

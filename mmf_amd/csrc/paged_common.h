// mmf_amd :: what the kernels over the paged cache share.
#pragma once
#include <atomic>

#include "common.h"
#include "mmf_amd.h"

// Set where a page, slot, parent or row index points outside its table; the access is left out.  One flag per source file;
// mmf_amd_take_index_error() reports and clears them all.
static __device__ int g_page_error = 0;
DEVI void flag_page_error() { atomicOr(&g_page_error, 1); }

// Whether this file's kernels were ever launched or captured: until then its flag cannot be set, and who asks for errors between steps (the embedding gathers' callers, that
// use no paged cache) does not pay for a copy from the device that can only bring 0: 12 us each.  (Not cleared again: a captured launch runs at every replay.)
static std::atomic<bool> g_page_used{false};
static inline void page_kernels_used() { g_page_used.store(true, std::memory_order_relaxed); }
static inline int take_page_error() {
    if (!g_page_used.load(std::memory_order_relaxed)) return 0;
    int v = 0;
    if (hipMemcpyFromSymbol(&v, HIP_SYMBOL(g_page_error), sizeof(int)) != hipSuccess) { mmf_amd_set_error("take_index_error: copy failed"); return -1; }
    if (v) { const int z = 0; (void)hipMemcpyToSymbol(HIP_SYMBOL(g_page_error), &z, sizeof(int)); }
    return v;
}

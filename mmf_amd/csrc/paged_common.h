// mmf_amd :: what the kernels over the paged cache share.
#pragma once
#include "common.h"

// Set where a page, slot, parent or row index points outside its table; the access is left out.  One flag per source file;
// mmf_amd_take_index_error() reports and clears them all.
static __device__ int g_page_error = 0;
DEVI void flag_page_error() { atomicOr(&g_page_error, 1); }

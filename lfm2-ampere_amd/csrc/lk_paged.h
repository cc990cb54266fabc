// lk_paged.h - what the kernels over a paged cache share (paged.hip, paged_attn.hip):
// bounded reads of a step's tables, and the host's checks of its descriptions.
#pragma once
#include "lk_types.h"

// A sequence's rows [r0, r0 + n) of the step and its positions before it, every value
// brought into its range.
struct LkSeq { int r0, n, len; };
__device__ __forceinline__ int lk_clamp(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }
__device__ __forceinline__ LkSeq lk_seq(int f0, int f1, int len, int rows, int cap) {
    LkSeq s;
    s.r0 = lk_clamp(f0, 0, rows);
    s.n = lk_clamp(f1, s.r0, rows) - s.r0;
    s.len = lk_clamp(len, 0, cap);
    return s;
}

// The largest width * page: slots, and a slot plus a step's rows, stay far inside an int.
#define LK_PAGED_MAX_SLOTS (1 << 30)

// Checks that all three entry points make; 0 or an error code (lk_host.cpp's lk_fail).
int lk_paged_check(const char * what, const lk_pages * p, const lk_step * s);
int lk_paged_check_type(const char * what, const lk_pages * p, int type);
int lk_paged_check_pages(const char * what, const lk_pages * p);
static inline int lk_log2(int v) { return 31 - __builtin_clz((unsigned) v); }

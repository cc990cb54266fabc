// lk_q81.h - the arithmetic of planar Q8_1 quants and scales, shared by the
// prefill attention's epilogue, the stand-alone quantiser (prefill.hip) and the
// norm's 8-bit outputs (norm.hip).
#pragma once
#include "lk_common.h"

// Reference k_pf_quant_rows / pf_quant_warp (prefill.cu:1574-1580, 90-103): per
// 32-value block am = max|x| (exact), sum = xor-butterfly over the block's
// dims with strides 16, 8, 4, 2, 1, d = am/127 (IEEE), q = roundf(x/d) (0 when
// am = 0), scale plane (float(fp16(d)), 8 * float(fp16(sum))).  Layout:
// qs int8 [rows][2048] (block b of a row at 32b), sc float2 [rows][64].
__device__ __forceinline__ float2 lk_q81_scales(float d, float sum) {
    return make_float2((float) (_Float16) d, 8.0f * (float) (_Float16) sum);
}
__device__ __forceinline__ int8_t lk_q81_q(float x, float am, float d) {
    return (am == 0.0f) ? (int8_t) 0 : (int8_t) roundf(x / d);
}
// The same q for the many values of one block with one division per block:
// with r = RN(1/d'), q0 = RN(x*r) is within an ulp of x/d' and
// RN(q0 + RN(x - q0*d')*r) (two fmas, the remainder exact) is RN(x/d')
// (Markstein's correction theorem), so roundf sees the bits of x / d.  The
// theorem needs x/d' and 1/d' in the normal range: blocks with am < 2^-64
// scale x and d by 2^64 (exact, the quotient unchanged); quotients that are
// subnormal may differ, but roundf gives 0 for both.  am = 0 (all x = 0)
// divides by 1.  tests/test_q81_division.py runs this arithmetic on the host
// against x / d over am in [2^-140, 2^100], ties and quotients next to .5
// included.
struct LkQ81Div { float s, d, r; };
__device__ __forceinline__ LkQ81Div lk_q81_div(float am, float d) {
    LkQ81Div q;
    q.s = am < 0x1p-64f ? 0x1p64f : 1.0f;
    q.d = am == 0.0f ? 1.0f : d * q.s;
    q.r = 1.0f / q.d;
    return q;
}
__device__ __forceinline__ int8_t lk_q81_qd(const LkQ81Div & q, float x) {
#pragma clang fp contract(off)
    const float xs = x * q.s;
    const float q0 = xs * q.r;
    const float e = __builtin_fmaf(-q0, q.d, xs);
    return (int8_t) roundf(__builtin_fmaf(e, q.r, q0));
}

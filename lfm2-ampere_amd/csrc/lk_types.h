// lk_types.h - element types, unaligned pieces and wave reductions shared by the
// norm, int8 product and mixture-of-experts kernels (norm.hip, gemm_i8.hip,
// moe.hip).
#pragma once
#include "lk_common.h"

typedef int lk_i16v __attribute__((ext_vector_type(16)));                // a tile of v_mfma_i32_32x32x32_i8, a lane's part

// ---- 16- and 32-bit float elements (LK_F32, LK_F16, LK_BF16) --------------------
template <int TYPE> struct LkElem;
template <> struct LkElem<LK_F32>  { typedef float type; };
template <> struct LkElem<LK_F16>  { typedef _Float16 type; };
template <> struct LkElem<LK_BF16> { typedef __bf16 type; };
static inline int lk_type_size(int type) { return type == LK_F32 ? 4 : 2; }
static inline bool lk_type_ok(int type) { return type == LK_F32 || type == LK_F16 || type == LK_BF16; }

// N consecutive elements at p as fp32, and back (rounded to nearest).  Element
// alignment is enough: rows of odd length put every second row off any wider
// alignment, and gfx950 loads and stores 16 bytes at any address, so that one
// form serves both.
template <int N, typename T>
__device__ __forceinline__ void lk_load(const T * p, float (&v)[N]) {
    struct { T e[N]; } b;
    __builtin_memcpy(&b, p, sizeof b);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (float) b.e[i];
}
template <int N, typename T>
__device__ __forceinline__ void lk_store(T * p, const float (&v)[N]) {
    struct { T e[N]; } b;
#pragma unroll
    for (int i = 0; i < N; ++i) b.e[i] = (T) v[i];
    __builtin_memcpy(p, &b, sizeof b);
}

// The same, past the caches' order (non-temporal): for outputs that the kernel does not read again,
// which otherwise wait in the L2s to be written back when it ends.
template <int N, typename T>
__device__ __forceinline__ void lk_store_nt(T * p, const float (&v)[N]) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4), aligned(2)));       // the elements' alignment
    static_assert(N * sizeof(T) % 16 == 0, "whole 16-byte stores");
    union { T e[N]; u4 q[N * sizeof(T) / 16]; } b;
#pragma unroll
    for (int i = 0; i < N; ++i) b.e[i] = (T) v[i];
#pragma unroll
    for (int i = 0; i < (int) (N * sizeof(T) / 16); ++i) __builtin_nontemporal_store(b.q[i], (u4 *) p + i);
}

// ---- reductions over the 64 lanes of a wave, every lane left with the same bits --
__device__ __forceinline__ float lk_wave_sum(float v) { return lk_xrow_sum(lk_row_sum16(v)); }
template <int CTRL>
__device__ __forceinline__ double lk_dpp64(double v) {
    const uint64_t u = __builtin_bit_cast(uint64_t, v);
    const float lo = lk_dpp<CTRL>(__builtin_bit_cast(float, (uint32_t) u));
    const float hi = lk_dpp<CTRL>(__builtin_bit_cast(float, (uint32_t) (u >> 32)));
    return __builtin_bit_cast(double, (uint64_t) __builtin_bit_cast(uint32_t, hi) << 32 | __builtin_bit_cast(uint32_t, lo));
}
__device__ __forceinline__ double lk_wave_sum64(double v) {
    v += lk_dpp64<LK_DPP_QP_XOR1>(v);
    v += lk_dpp64<LK_DPP_QP_XOR2>(v);
    v += lk_dpp64<LK_DPP_HMIRROR>(v);
    v += lk_dpp64<LK_DPP_MIRROR>(v);
    v += __shfl_xor(v, 16, 64);
    v += __shfl_xor(v, 32, 64);
    return v;
}
// The larger of two bit patterns of non-negative floats is that of the larger
// float, infinities above every number and NaN above infinities.
__device__ __forceinline__ uint32_t lk_umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
template <int CTRL>
__device__ __forceinline__ uint32_t lk_dpp_u(uint32_t v) {
    return __builtin_bit_cast(uint32_t, lk_dpp<CTRL>(__builtin_bit_cast(float, v)));
}
__device__ __forceinline__ uint32_t lk_wave_umax(uint32_t v) {
    v = lk_umax(v, lk_dpp_u<LK_DPP_QP_XOR1>(v));
    v = lk_umax(v, lk_dpp_u<LK_DPP_QP_XOR2>(v));
    v = lk_umax(v, lk_dpp_u<LK_DPP_HMIRROR>(v));
    v = lk_umax(v, lk_dpp_u<LK_DPP_MIRROR>(v));
    v = lk_umax(v, (uint32_t) __shfl_xor((int) v, 16, 64));
    v = lk_umax(v, (uint32_t) __shfl_xor((int) v, 32, 64));
    return v;
}

// norm.hip - the step between a projection and the product that follows it: the
// residual addition, the RMS norm and the quantisation of the normed row to 8
// bits, in one pass over the rows.
//
// Per row of n values (contraction off, so every fp32 step rounds as written):
//     h = x + delta                       (fp32; delta absent: h = x)
//     r = (float) (1 / sqrt(sum (double) h^2 / n + eps))
//     y = (h * r) * w
// and of y either one scale a row (the int8 product's operand, gemm_i8.hip):
//     a = max |y|, scale = a / 127, q = rint(y * (127 / a))
// or Q8_1 blocks of 32 (lk_q81.h), planar for the Q4_0 GEMM or as lk_block_q8_1
// for the Q4_0 GEMV, the bytes lk_pf_quant_rows and the decode combine make of y.
// h and y are also stored where the caller asks, rounded once to the rows' type;
// the norm goes on from the unrounded h.
// The sum of squares is taken in 64 bits: q is a rounding of y, and fp32 partial sums of
// 2048 squares differ in their last bits with the number of lanes, which moved 1 of
// about 10^5 quants by one.  The orders of 64-bit sums differ by about 2^-50, so the launch
// shapes agree but where 1 / sqrt lies that close to the middle of two fp32 numbers: one row
// of some 10^8.
// A row of h with a value that is not finite gets the scale NaN and zeros (row form),
// and NaN in h * r, so that everything computed from it is NaN and no other row
// is touched (with eps 0, a row of zeros too: 0 / 0); a row whose largest |y| is below
// 2^-120 gets scale and quants 0 (127 / a would overflow).
#include "lk_types.h"
#include "lk_q81.h"

#define LK_NORM_TINY 0x1p-120f

struct LkNormArgs {
    const void * x;
    const void * delta;
    const float * w;
    void * res;
    void * y;
    int8_t * q;
    float * sc;
    int ldx, ldd, ldr, ldy, ldq, rows, n;
    float eps;
};

// Rows of h and y, which the next kernel does not need (q it does: with q past the caches' order
// too, the int8 product that follows lost what was gained and more, 4096 x 2048 x 2048 35.1 us
// together for 32.5): 16-bit rows go past the caches' order, 4096 x 2048 bf16 11.7 us for 13.0, 1024 x
// 16384 21.3 for 22.9; fp32 rows gain and lose (4096 x 1024 9.6 for 11.1, 2048 x 8192 38.1 for 35.1)
// and stay.
template <typename T>
__device__ __forceinline__ void lk_norm_store(T * o, const float (&v)[8]) {
    if constexpr (sizeof(T) == 2) lk_store_nt<8>(o, v);
    else                          lk_store<8>(o, v);
}

// NW waves hold a row, 8 consecutive values per lane and chunk, C chunks; a workgroup
// has 4 waves or one row's, whichever is more.  One pass: the row stays in registers
// between the sum of squares, the largest value and the quants, and w is asked for along
// with x and delta.  What bounds it: one row, the launch and one load's latency (2.5 us a
// call in a graph, 1 x 2048); many rows, memory: 4096 x 2048 with delta and res, bf16, 59 MB
// in 11.7 us (5.0 TB/s), fp32, 109 MB in 18.2 us (6.0), next to 5.15 TB/s of a 1 GiB copy.
template <int TYPE, int FORM, int NW, int C>
__global__ void __launch_bounds__(NW > 4 ? 64 * NW : 256)
lk_k_norm_q8(const LkNormArgs a) {
#pragma clang fp contract(off)
    typedef typename LkElem<TYPE>::type T;
    constexpr int RW = NW > 4 ? 1 : 4 / NW;              // rows per workgroup
    __shared__ double s_ss[NW > 1 ? NW * RW : 1];
    __shared__ uint32_t s_am[NW > 1 ? NW * RW : 1];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int wr = wv % NW;                              // the wave's part of its row
    const long row0 = (long) blockIdx.x * RW + wv / NW;
    const bool live = row0 < a.rows;
    const long row = live ? row0 : a.rows - 1;           // clamped: loads stay in bounds, nothing is stored
    const int n = a.n;
    const T * x = (const T *) a.x + row * a.ldx;
    const T * dl = a.delta ? (const T *) a.delta + row * a.ldd : nullptr;

    float h[C][8];
    double ss = 0.0;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = ((c * NW + wr) * 64 + lane) * 8;
        if (i + 8 <= n) {
            lk_load<8>(x + i, h[c]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) h[c][e] = i + e < n ? (float) x[i + e] : 0.0f;
        }
    }
    if (dl) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int i = ((c * NW + wr) * 64 + lane) * 8;
            float d[8];
            if (i + 8 <= n) {
                lk_load<8>(dl + i, d);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) d[e] = i + e < n ? (float) dl[i + e] : 0.0f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) h[c][e] += d[e];
        }
    }
    float w[C][8];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = ((c * NW + wr) * 64 + lane) * 8;
        if (i + 8 <= n) {
            lk_load<8>(a.w + i, w[c]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) w[c][e] = i + e < n ? a.w[i + e] : 0.0f;
        }
    }
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = __builtin_fma((double) h[c][e], (double) h[c][e], ss);
    if (a.res && live) {
        T * o = (T *) a.res + row * a.ldr;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int i = ((c * NW + wr) * 64 + lane) * 8;
            if (i + 8 <= n) lk_norm_store(o + i, h[c]);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) if (i + e < n) o[i + e] = (T) h[c][e];
        }
    }
    ss = lk_wave_sum64(ss);
    if constexpr (NW > 1) {
        if (lane == 0) s_ss[wv] = ss;
        __syncthreads();
        ss = 0.0;
#pragma unroll
        for (int k = 0; k < NW; ++k) ss += s_ss[wv / NW * NW + k];
    }
    float r = (float) (1.0 / sqrt(ss / (double) n + (double) a.eps));
    if (!(ss < __builtin_inf())) r = __builtin_nanf("");   // an infinite or NaN h: the whole row is NaN
    uint32_t am = 0;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = ((c * NW + wr) * 64 + lane) * 8;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            h[c][e] = (h[c][e] * r) * w[c][e];           // y from here on
            if (i + e < n) am = lk_umax(am, __builtin_bit_cast(uint32_t, h[c][e]) & 0x7FFFFFFFu);
        }
    }
    if (a.y && live) {
        T * o = (T *) a.y + row * a.ldy;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int i = ((c * NW + wr) * 64 + lane) * 8;
            if (i + 8 <= n) lk_norm_store(o + i, h[c]);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) if (i + e < n) o[i + e] = (T) h[c][e];
        }
    }
    if constexpr (FORM == LK_Q8_ROW) {
        am = lk_wave_umax(am);
        if constexpr (NW > 1) {
            if (lane == 0) s_am[wv] = am;
            __syncthreads();
#pragma unroll
            for (int k = 0; k < NW; ++k) am = lk_umax(am, s_am[wv / NW * NW + k]);
        }
        const float amax = __builtin_bit_cast(float, am);
        const bool fin = am < 0x7F800000u, some = fin && amax >= LK_NORM_TINY;
        const float id = some ? 127.0f / amax : 0.0f;
        if (!live) return;
        if (wr == 0 && lane == 0) a.sc[row] = fin ? (some ? amax / 127.0f : 0.0f) : __builtin_nanf("");
        int8_t * o = a.q + row * a.ldq;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int i = ((c * NW + wr) * 64 + lane) * 8;
            uint32_t q[2] = { 0, 0 };
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float v = some ? __builtin_rintf(h[c][e] * id) : 0.0f;
                q[e / 4] |= (uint32_t) (uint8_t) (int8_t) (int) v << (8 * (e % 4));
            }
            if (i + 8 <= n) __builtin_memcpy(o + i, q, 8);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) if (i + e < n) o[i + e] = (int8_t) (q[e / 4] >> (8 * (e % 4)));
        }
    } else {
        // a block's 32 values are on four consecutive lanes; its sum is the butterfly
        // with strides 16 and 8 (lanes xor 2 and 1), then 4, 2 and 1 in the lane
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int i = ((c * NW + wr) * 64 + lane) * 8;
            float bm = fabsf(h[c][0]), t[8];             // not from 0: a block of NaN alone keeps a NaN scale
#pragma unroll
            for (int e = 1; e < 8; ++e) bm = fmaxf(bm, fabsf(h[c][e]));
            bm = fmaxf(bm, lk_dpp<LK_DPP_QP_XOR1>(bm));
            bm = fmaxf(bm, lk_dpp<LK_DPP_QP_XOR2>(bm));
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] = h[c][e] + lk_dpp<LK_DPP_QP_XOR2>(h[c][e]);
#pragma unroll
            for (int e = 0; e < 8; ++e) t[e] += lk_dpp<LK_DPP_QP_XOR1>(t[e]);
            const float sum = ((t[0] + t[4]) + (t[2] + t[6])) + ((t[1] + t[5]) + (t[3] + t[7]));
            const float d = bm / 127.0f;
            const LkQ81Div qd = lk_q81_div(bm, d);
            uint32_t q[2] = { 0, 0 };
            if (d == 0.0f) {                             // the largest value is up to 63 units of 2^-149: y / d is infinite
#pragma unroll
                for (int e = 0; e < 8; ++e) q[e / 4] |= (uint32_t) (uint8_t) lk_q81_q(h[c][e], bm, d) << (8 * (e % 4));
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) q[e / 4] |= (uint32_t) (uint8_t) lk_q81_qd(qd, h[c][e]) << (8 * (e % 4));
            }
            if (i >= n || !live) continue;               // whole blocks: n is a multiple of 32
            const long b = row * (n / 32) + i / 32;
            if constexpr (FORM == LK_Q81_PLANAR) {
                __builtin_memcpy(a.q + row * n + i, q, 8);
                if ((lane & 3) == 0) ((float2 *) a.sc)[b] = lk_q81_scales(d, sum);
            } else {
                uint32_t * o = (uint32_t *) a.q + b * 9;
                o[1 + 2 * (lane & 3)] = q[0];
                o[2 + 2 * (lane & 3)] = q[1];
                if ((lane & 3) == 0)
                    o[0] = (uint32_t) __builtin_bit_cast(uint16_t, (_Float16) d) |
                           (uint32_t) __builtin_bit_cast(uint16_t, (_Float16) sum) << 16;
            }
        }
    }
}

template <int TYPE, int FORM, int NW, int C>
static void lk_norm_launch(const LkNormArgs & a, hipStream_t st) {
    constexpr int RW = NW > 4 ? 1 : 4 / NW;
    hipLaunchKernelGGL((lk_k_norm_q8<TYPE, FORM, NW, C>), dim3((unsigned) ((a.rows - 1) / RW + 1)),
                       dim3(NW > 4 ? 64 * NW : 256), 0, st, a);
}
// As many waves as a row has runs of 512 values, so that all lanes have work and a lane one
// chunk.  Measured, row form, us (<NW, C>):
//   4096 x 1024 bf16   <2,1>  7.1   <1,2>  6.6   <4,1> 10.8 (half of the lanes idle)
//   1 x 2048 fp32      <4,1>  2.6   <2,2>  3.3   <1,4>  4.1
//   333 x 2048 bf16    <4,1>  3.5   <2,2>  3.9   <1,4>  5.0
//   4096 x 2048 bf16   <4,1> 12.7   <2,2> 12.6   <1,4> 12.2
//   1 x 4096 bf16      <8,1>  3.0   <4,2>  3.3   <4,4>  5.8
//   4096 x 4096 bf16   <8,1> 21.4   <4,2> 21.8   <4,4> 31.3
//   64 x 8192 bf16     <16,1> 4.2   <8,2>  4.3   <4,4>  5.1
//   1024 x 16384 bf16  <16,2> 23.0  <8,4> 23.8   <16,4> 40.6
template <int TYPE, int FORM>
static void lk_norm_shape(const LkNormArgs & a, hipStream_t st) {
    if (a.n <= 512)        lk_norm_launch<TYPE, FORM, 1, 1>(a, st);
    else if (a.n <= 1024)  lk_norm_launch<TYPE, FORM, 2, 1>(a, st);
    else if (a.n <= 2048)  lk_norm_launch<TYPE, FORM, 4, 1>(a, st);
    else if (a.n <= 4096)  lk_norm_launch<TYPE, FORM, 8, 1>(a, st);
    else if (a.n <= 8192)  lk_norm_launch<TYPE, FORM, 16, 1>(a, st);
    else if (a.n <= 16384) lk_norm_launch<TYPE, FORM, 16, 2>(a, st);
    else                   lk_norm_launch<TYPE, FORM, 16, 4>(a, st);
}
template <int TYPE>
static void lk_norm_form(int form, const LkNormArgs & a, hipStream_t st) {
    if (form == LK_Q8_ROW)          lk_norm_shape<TYPE, LK_Q8_ROW>(a, st);
    else if (form == LK_Q81_PLANAR) lk_norm_shape<TYPE, LK_Q81_PLANAR>(a, st);
    else                            lk_norm_shape<TYPE, LK_Q81_BLOCK>(a, st);
}

extern "C" int lk_norm_q8(int type, const void * x, int ldx, const void * delta, int ldd, const float * w, float eps,
                          int rows, int n, void * res, int ldr, void * y, int ldy, int form, int8_t * q, int ldq,
                          float * sc, void * stream) {
    if (!lk_type_ok(type) || form < LK_Q8_ROW || form > LK_Q81_BLOCK)
        return lk_fail(hipErrorInvalidValue, "lk_norm_q8: type %d / form %d", type, form);
    if (rows < 0 || n < 1 || n > LK_NORM_MAX_N)
        return lk_fail(hipErrorInvalidValue, "lk_norm_q8: rows %d, n %d (1..%d)", rows, n, LK_NORM_MAX_N);
    if (!(eps >= 0.0f)) return lk_fail(hipErrorInvalidValue, "lk_norm_q8: eps %g", (double) eps);
    if (form != LK_Q8_ROW && n % 32 != 0)
        return lk_fail(hipErrorInvalidValue, "lk_norm_q8: n %d must be a multiple of 32 for Q8_1 blocks", n);
    if (rows == 0) return 0;
    // a grid has fewer than 2^32 threads, a workgroup 256 or more (1024 above 4096 values)
    if ((n > 4096 ? 1024l : n > 2048 ? 512l : n > 1024 ? 256l : n > 512 ? 128l : 64l) * rows > 0xFFFFFE00l)
        return lk_fail(hipErrorInvalidValue, "lk_norm_q8: %d rows of %d", rows, n);
    if (!x || !w || !q || (form != LK_Q81_BLOCK && !sc))
        return lk_fail(hipErrorInvalidValue, "lk_norm_q8: null pointer argument");
    if (ldx < n || (delta && ldd < n) || (res && ldr < n) || (y && ldy < n) || (form == LK_Q8_ROW && ldq < n) ||
        (form != LK_Q8_ROW && ldq != n))
        return lk_fail(hipErrorInvalidValue, "lk_norm_q8: row strides x %d, delta %d, res %d, y %d, q %d for n %d (Q8_1: q %d)",
                       ldx, ldd, ldr, ldy, ldq, n, n);
    const uintptr_t em = (uintptr_t) lk_type_size(type) - 1;
    if (((uintptr_t) x & em) || ((uintptr_t) delta & em) || ((uintptr_t) res & em) || ((uintptr_t) y & em) ||
        ((uintptr_t) w & 3) || ((uintptr_t) sc & (form == LK_Q81_PLANAR ? 7 : 3)) ||
        (form == LK_Q81_BLOCK && ((uintptr_t) q & 3)))
        return lk_fail(hipErrorInvalidValue, "lk_norm_q8: misaligned argument (rows by their element, w 4 B, sc 4 B (planar 8), blocks 4 B)");
    const LkNormArgs a = { x, delta, w, res, y, q, sc, ldx, ldd, ldr, ldy, ldq, rows, n, eps };
    const hipStream_t st = lk_stream(stream);
    if (type == LK_F32)      lk_norm_form<LK_F32>(form, a, st);
    else if (type == LK_F16) lk_norm_form<LK_F16>(form, a, st);
    else                     lk_norm_form<LK_BF16>(form, a, st);
    return lk_launch_status("lk_norm_q8");
}

// gemm_i8.hip - the matrix product of 8-bit integer rows with a scale for each
// token (row of x) and each channel (row of w):
//     out[t][r] = (res ? res[t][r] : 0) + ((float) S * sx[t]) * sw[r]
//     S = sum over k of x[t][k] * w[r][k], exact in int32 (K <= 131071)
// with fp32 scales and fp32, fp16 or bf16 out and res: the sum is converted once,
// multiplied and added in fp32 with every step rounded as written, and rounded once
// to the output's type.  x is what lk_norm_q8 writes in row form.
//
// Rows of x and w are multiples of 16 bytes apart and 16-byte aligned; what lies
// between K and the next multiple of 16 is read but does not count: the last piece
// of each x row is masked, and 0 times anything is 0.
#include "lk_types.h"

typedef int lk_i16v __attribute__((ext_vector_type(16)));

// The result of one output: every step rounded as written.
__device__ __forceinline__ float lk_i8_out(int s, float sx, float sw) {
#pragma clang fp contract(off)
    const float v = (float) s * sx;
    return v * sw;
}
// Bytes k0 .. k0+15 of a row of K: those at K and beyond as zero.
__device__ __forceinline__ lk_i4 lk_i8_mask(lk_i4 v, int k0, int K) {
    const int left = K - k0;
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const int b = left - 4 * d;                      // bytes of this dword that count
        v[d] = b >= 4 ? v[d] : b <= 0 ? 0 : (int) ((uint32_t) v[d] & (0xFFFFFFFFu >> (32 - 8 * b)));
    }
    return v;
}

struct LkI8Args {
    const int8_t * x;
    const int8_t * w;
    const float * sx;
    const float * sw;
    const void * res;
    void * out;
    int ldx, ldw, ldr, ldo, M, N, K;
};

// ---- few tokens -------------------------------------------------------------------
// 16 weight rows per workgroup against TT tiles of 16 tokens
// (v_mfma_i32_16x16x64_i8); the NW waves take 128-byte pieces of K in turn and
// load them straight into the operand layout (lane: row or token l % 16, 16
// bytes at 16 * (l / 16) of a 64-byte step), so that nothing waits for anything
// but its own loads.  The int32 parts meet in LDS; integer sums have no order.
template <int TYPE, int TT, int NW>
__global__ void __launch_bounds__(64 * NW)
lk_k_gemm_i8_few(const LkI8Args a) {
    typedef typename LkElem<TYPE>::type T;
    constexpr int U = TT > 2 ? 2 : 4;                    // 64-byte steps in flight per wave
    __shared__ __attribute__((aligned(16))) lk_i4 part[NW][TT][64];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4;
    const int r0 = blockIdx.x * 16, t0 = blockIdx.y * (16 * TT);
    const int8_t * wp = a.w + (size_t) (r0 + c < a.N ? r0 + c : a.N - 1) * a.ldw;
    const int8_t * xp[TT];
#pragma unroll
    for (int j = 0; j < TT; ++j) {
        const int t = t0 + 16 * j + c;
        xp[j] = a.x + (size_t) (t < a.M ? t : a.M - 1) * a.ldx;
    }
    lk_i4 acc[TT];
#pragma unroll
    for (int j = 0; j < TT; ++j) acc[j] = lk_i4{ 0, 0, 0, 0 };
    const int K = a.K, nst = (K + 63) / 64;
    for (int s0 = 2 * wv; s0 < nst; s0 += U * NW) {
        lk_i4 wv4[U], xv[U][TT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k0 = (s0 + (u / 2) * 2 * NW + u % 2) * 64 + 16 * g;
            const int kc = k0 < K ? k0 : 0;              // in bounds; masked below
            wv4[u] = *(const lk_i4 *) (wp + kc);
#pragma unroll
            for (int j = 0; j < TT; ++j) xv[u][j] = *(const lk_i4 *) (xp[j] + kc);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int st = s0 + (u / 2) * 2 * NW + u % 2;
            if (st * 64 + 64 > K) {                      // wave-uniform: the last step, or past it
#pragma unroll
                for (int j = 0; j < TT; ++j) xv[u][j] = lk_i8_mask(xv[u][j], st * 64 + 16 * g, K);
            }
#pragma unroll
            for (int j = 0; j < TT; ++j) acc[j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv4[u], xv[u][j], acc[j], 0, 0, 0);
        }
    }
#pragma unroll
    for (int j = 0; j < TT; ++j) part[wv][j][lane] = acc[j];
    __syncthreads();
    // output (token tc of tile j, row r): lane r / 4 * 16 + tc holds it in r % 4
    const T * res = (const T *) a.res;
    T * out = (T *) a.out;
    for (int i = threadIdx.x; i < TT * 256; i += 64 * NW) {
        const int r = i & 15, tt = i >> 4, j = tt >> 4, tc = tt & 15;
        int s = 0;
#pragma unroll
        for (int k = 0; k < NW; ++k) s += part[k][j][(r >> 2) * 16 + tc][r & 3];
        const int t = t0 + tt, rr = r0 + r;
        if (t < a.M && rr < a.N) {
            float v = lk_i8_out(s, a.sx[t], a.sw[rr]);
            if (res) v = (float) res[(size_t) t * a.ldr + rr] + v;
            out[(size_t) t * a.ldo + rr] = (T) v;
        }
    }
}

// ---- tiles ------------------------------------------------------------------------
// A wave covers TM x TN tiles of v_mfma_i32_32x32x32_i8 (TM along the weight rows, TN
// along the tokens), WM x WN waves a workgroup; K in stages of KC bytes, a ring of
// NB of them in LDS, filled by LDS DMA.
template <int TM_, int TN_, int WM_, int WN_, int KC_, int NB_, int OCC_>
struct LkI8Shape {
    static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, KC = KC_, NB = NB_, OCC = OCC_;   // OCC: waves per SIMD
    static constexpr int NW = WM * WN, BM = 32 * TM * WM, BN = 32 * TN * WN, PC = KC / 16;
    static constexpr int BYTES = (BM + BN) * KC;         // a stage: BM weight rows, then BN token rows
    static constexpr int NA = BM * PC / 64, NI = (BM + BN) * PC / 64, PW = NI / NW;
    static_assert(NI % NW == 0 && BM * PC % 64 == 0 && BN * PC % 64 == 0, "whole DMA instructions, the same for every wave");
    static_assert((NB - 2) * PW < 64, "vmcnt range");
};
// 16-byte slot of piece p of a row of n pieces: XOR-permuted so that the same piece
// of 16 consecutive rows lies in 16 different slots modulo 256 bytes (all banks).
__device__ __forceinline__ constexpr int lk_i8_slot(int n, int row, int p) { return row * n + (p ^ (row / (16 / n) % n)); }

template <class SH, int TYPE>
__global__ void __launch_bounds__(64 * SH::NW, SH::OCC)
lk_k_gemm_i8(const LkI8Args a) {
    typedef typename LkElem<TYPE>::type T;
    constexpr int TM = SH::TM, TN = SH::TN, KC = SH::KC, NB = SH::NB, NW = SH::NW, PC = SH::PC, PW = SH::PW, NQ = KC / 32;
    __shared__ __attribute__((aligned(16))) uint8_t stg[NB * SH::BYTES];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    // XCD-aware tile order: workgroups go round-robin over the 8 XCDs (id % 8), so
    // consecutive tiles L are given to one XCD; L runs through groups of 8 row tiles,
    // row tiles first, so that the tiles an XCD works on at a time form a patch
    // whose operands its L2 holds once.
    const int nrt = (a.N + SH::BM - 1) / SH::BM, ntt = (a.M + SH::BN - 1) / SH::BN, ntile = nrt * ntt;
    const int id = blockIdx.x, x8 = id & 7, rem = ntile & 7;
    const int L = x8 * (ntile >> 3) + (x8 < rem ? x8 : rem) + (id >> 3);
    const int gr = L / (8 * ntt), gw = nrt - 8 * gr < 8 ? nrt - 8 * gr : 8, li = L - gr * 8 * ntt;
    const int row0 = (8 * gr + li % gw) * SH::BM, tok0 = (li / gw) * SH::BN;
    const int wr = (w % SH::WM) * 32 * TM, wt = (w / SH::WM) * 32 * TN;
    const int lm = lane & 31, h = lane >> 5;
    const int K = a.K, nst = (K + KC - 1) / KC;

    // DMA instruction i of this wave: slots 64 * (i * NW + w) + lane of a stage
    uint32_t roff[PW], pc[PW];
#pragma unroll
    for (int i = 0; i < PW; ++i) {
        const int j = i * NW + w;
        const bool isa = j < SH::NA;
        const int slot = 64 * (isa ? j : j - SH::NA) + lane, r = slot / PC;
        pc[i] = (uint32_t) (lk_i8_slot(PC, r, slot % PC) % PC * 16);
        const int lim = isa ? a.N - 1 - row0 : a.M - 1 - tok0;
        roff[i] = (uint32_t) (r < lim ? r : lim) * (uint32_t) (isa ? a.ldw : a.ldx);       // clamped: in bounds
    }
    const int8_t * wb = a.w + (size_t) row0 * a.ldw, * xb = a.x + (size_t) tok0 * a.ldx;
    const uint32_t lds0 = lk_lds_addr(stg);
    auto fetch = [&](int s) {
        const uint32_t sb = lds0 + (uint32_t) (s % NB * SH::BYTES);
        const int k0 = s * KC;
        if (k0 + KC <= K) {
#pragma unroll
            for (int i = 0; i < PW; ++i) {
                const int j = i * NW + w;
                lk_dma16c_so((j < SH::NA ? wb : xb) + k0, roff[i] + pc[i], sb + (uint32_t) (1024 * j));
            }
        } else {                                         // pieces past the row: its first piece instead
#pragma unroll
            for (int i = 0; i < PW; ++i) {
                const int j = i * NW + w;
                const uint32_t k = (uint32_t) k0 + pc[i];
                lk_dma16c_so(j < SH::NA ? wb : xb, roff[i] + (k < (uint32_t) K ? k : 0u), sb + (uint32_t) (1024 * j));
            }
        }
    };
    lk_i16v acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
    lk_i4 av[2][TM], bv[2][TN];
    auto load = [&](int s, int q, int u) {               // operands of step q of stage s
        const uint8_t * S = stg + s % NB * SH::BYTES;
#pragma unroll
        for (int i = 0; i < TM; ++i) av[u][i] = *(const lk_i4 *) (S + lk_i8_slot(PC, wr + 32 * i + lm, 2 * q + h) * 16);
#pragma unroll
        for (int j = 0; j < TN; ++j) bv[u][j] = *(const lk_i4 *) (S + SH::BM * KC + lk_i8_slot(PC, wt + 32 * j + lm, 2 * q + h) * 16);
    };
    // all of this wave's LDS reads are in registers, stage s + 1 of every wave has
    // landed; afterwards the buffer of stage s may be overwritten
    auto turn = [&](int s) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (s + NB - 1 < nst) lk_wait_vm<(NB - 2) * PW>();
        else lk_wait_vm<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    for (int s = 0; s < NB - 1 && s < nst; ++s) fetch(s);
    if (nst > NB - 2) lk_wait_vm<(NB - 2) * PW>();
    else lk_wait_vm<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    load(0, 0, 0);
    for (int s = 0; s < nst; ++s) {
        if (s + NB - 1 < nst) fetch(s + NB - 1);
        const bool whole = (s + 1) * KC <= K;
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            const int u = q & 1;
            if (q + 1 < NQ) load(s, q + 1, u ^ 1);
            else if (s + 1 < nst) { turn(s); load(s + 1, 0, u ^ 1); }
            if (!whole) {
#pragma unroll
                for (int j = 0; j < TN; ++j) bv[u][j] = lk_i8_mask(bv[u][j], s * KC + 32 * q + 16 * h, K);
            }
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(av[u][i], bv[u][j], acc[i][j], 0, 0, 0);
        }
    }
    // lane: token lm of a tile, rows 8 * e4 + 4 * h .. +3
    const T * res = (const T *) a.res;
    T * out = (T *) a.out;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        const int t = tok0 + wt + 32 * j + lm;
        if (t >= a.M) continue;
        const float sx = a.sx[t];
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int e4 = 0; e4 < 4; ++e4) {
                const int r = row0 + wr + 32 * i + 8 * e4 + 4 * h;
                float v[4], s4[4], r4[4];
                if (r + 4 <= a.N) {
                    lk_load<4>(a.sw + r, s4);
                    if (res) lk_load<4>(res + (size_t) t * a.ldr + r, r4);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        v[e] = lk_i8_out(acc[i][j][4 * e4 + e], sx, s4[e]);
                        if (res) v[e] = r4[e] + v[e];
                    }
                    lk_store<4>(out + (size_t) t * a.ldo + r, v);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) if (r + e < a.N) {
                        float u = lk_i8_out(acc[i][j][4 * e4 + e], sx, a.sw[r + e]);
                        if (res) u = (float) res[(size_t) t * a.ldr + r + e] + u;
                        out[(size_t) t * a.ldo + r + e] = (T) u;
                    }
                }
            }
    }
}

template <int TYPE, int TT, int NW>
static void lk_i8_few(const LkI8Args & a, hipStream_t st) {
    hipLaunchKernelGGL((lk_k_gemm_i8_few<TYPE, TT, NW>), dim3((a.N + 15) / 16, (a.M + 16 * TT - 1) / (16 * TT)), dim3(64 * NW), 0, st, a);
}
template <class SH, int TYPE>
static int lk_i8_tiles(const LkI8Args & a, hipStream_t st) {
    const long n = (long) ((a.N + SH::BM - 1) / SH::BM) * ((a.M + SH::BN - 1) / SH::BN);
    if (n > 0x7FFFFFFF) return lk_fail(hipErrorInvalidValue, "lk_gemm_i8: %d x %d outputs", a.M, a.N);
    hipLaunchKernelGGL((lk_k_gemm_i8<SH, TYPE>), dim3((unsigned) n), dim3(64 * SH::NW), 0, st, a);
    return 0;
}
template <int TYPE>
static int lk_i8_shape(const LkI8Args & a, hipStream_t st) {
    if (a.M <= 16) { lk_i8_few<TYPE, 1, 8>(a, st); return 0; }
    if (a.M <= 32) { lk_i8_few<TYPE, 2, 8>(a, st); return 0; }
    const long t256 = (long) ((a.N + 255) / 256) * ((a.M + 255) / 256);
    if (t256 >= 256) return lk_i8_tiles<LkI8Shape<4, 4, 2, 2, 64, 4, 1>, TYPE>(a, st);
    const long t128 = (long) ((a.N + 127) / 128) * ((a.M + 127) / 128);
    if (t128 >= 256) return lk_i8_tiles<LkI8Shape<2, 2, 2, 2, 64, 4, 2>, TYPE>(a, st);
    return lk_i8_tiles<LkI8Shape<1, 1, 2, 2, 128, 4, 2>, TYPE>(a, st);
}

extern "C" int lk_gemm_i8(const int8_t * x, int ldx, const float * sx, const int8_t * w, int ldw, const float * sw,
                          int M, int N, int K, int type, const void * res, int ldr, void * out, int ldo, void * stream) {
    if (!lk_type_ok(type)) return lk_fail(hipErrorInvalidValue, "lk_gemm_i8: type %d", type);
    if (M < 0 || N < 0 || K < 1 || K > LK_GEMM_I8_MAX_K)
        return lk_fail(hipErrorInvalidValue, "lk_gemm_i8: M %d / N %d / K %d (1..%d)", M, N, K, LK_GEMM_I8_MAX_K);
    if (M == 0 || N == 0) return 0;
    if (!x || !sx || !w || !sw || !out) return lk_fail(hipErrorInvalidValue, "lk_gemm_i8: null pointer argument");
    if (ldx < K || ldx % 16 || ldw < K || ldw % 16 || ldo < N || (res && ldr < N))
        return lk_fail(hipErrorInvalidValue, "lk_gemm_i8: row strides x %d, w %d (multiples of 16, >= K %d), out %d, res %d (>= N %d)",
                       ldx, ldw, K, ldo, ldr, N);
    // the kernels address the rows of a tile (up to 256) with 32-bit byte offsets
    if (ldx > LK_GEMM_I8_MAX_LD || ldw > LK_GEMM_I8_MAX_LD)
        return lk_fail(hipErrorInvalidValue, "lk_gemm_i8: row strides x %d, w %d (at most %d)", ldx, ldw, LK_GEMM_I8_MAX_LD);
    const uintptr_t em = (uintptr_t) lk_type_size(type) - 1;
    if (((uintptr_t) x & 15) || ((uintptr_t) w & 15) || ((uintptr_t) sx & 3) || ((uintptr_t) sw & 3) || ((uintptr_t) out & em) ||
        ((uintptr_t) res & em))
        return lk_fail(hipErrorInvalidValue, "lk_gemm_i8: misaligned argument (x, w 16 B; sx, sw 4 B; out, res by their element)");
    const LkI8Args a = { x, w, sx, sw, res, out, ldx, ldw, ldr, ldo, M, N, K };
    const hipStream_t st = lk_stream(stream);
    int rc;
    if (type == LK_F32)      rc = lk_i8_shape<LK_F32>(a, st);
    else if (type == LK_F16) rc = lk_i8_shape<LK_F16>(a, st);
    else                     rc = lk_i8_shape<LK_BF16>(a, st);
    return rc ? rc : lk_launch_status("lk_gemm_i8");
}

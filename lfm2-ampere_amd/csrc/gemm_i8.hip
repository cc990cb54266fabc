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
// 16 weight rows per workgroup against up to 16 tokens (v_mfma_i32_16x16x64_i8); the
// NW waves take 128-byte pieces of K in turn, two at a time, and load them straight into
// the operand layout (lane: row or token l % 16, 16 bytes at 16 * (l / 16) of a 64-byte
// step), so that nothing waits for anything but its own loads.  The int32 parts meet in
// LDS; integer sums have no order.  Bound by the latency of one round of loads and the
// launch for short rows (1 x 4096 x 1024: 3.0 us with 4 waves, 3.7 with 8, of which half
// find no piece), by the weights' way from the cache for long ones (1 x 4096 x 8192, 34 MB:
// 7.1 us with 8 waves, 4.7 TB/s; 8.0 with 4).
template <int TYPE, int NW>
__global__ void __launch_bounds__(64 * NW)
lk_k_gemm_i8_few(const LkI8Args a) {
    typedef typename LkElem<TYPE>::type T;
    constexpr int U = 4;                                 // 64-byte steps in flight per wave
    __shared__ __attribute__((aligned(16))) lk_i4 part[NW][64];
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, g = lane >> 4, r0 = blockIdx.x * 16;
    const int8_t * wp = a.w + (size_t) (r0 + c < a.N ? r0 + c : a.N - 1) * a.ldw;
    const int8_t * xp = a.x + (size_t) (c < a.M ? c : a.M - 1) * a.ldx;
    lk_i4 acc = { 0, 0, 0, 0 };
    const int K = a.K, nst = (K + 63) / 64;
    for (int s0 = 2 * wv; s0 < nst; s0 += U * NW) {
        lk_i4 wv4[U], xv[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k0 = (s0 + (u / 2) * 2 * NW + u % 2) * 64 + 16 * g;
            const int kc = k0 < K ? k0 : 0;              // in bounds; masked below
            wv4[u] = *(const lk_i4 *) (wp + kc);
            xv[u] = *(const lk_i4 *) (xp + kc);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int st = s0 + (u / 2) * 2 * NW + u % 2;
            if (st * 64 + 64 > K) xv[u] = lk_i8_mask(xv[u], st * 64 + 16 * g, K);      // wave-uniform: the last step, or past it
            acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wv4[u], xv[u], acc, 0, 0, 0);
        }
    }
    part[wv][lane] = acc;
    __syncthreads();
    // output (token t, row r): lane r / 4 * 16 + t holds it in r % 4
    const T * res = (const T *) a.res;
    T * out = (T *) a.out;
    if (threadIdx.x >= 256) return;
    const int r = threadIdx.x & 15, t = threadIdx.x >> 4, rr = r0 + r;
    int s = 0;
#pragma unroll
    for (int k = 0; k < NW; ++k) s += part[k][(r >> 2) * 16 + t][r & 3];
    if (t < a.M && rr < a.N) {
        float v = lk_i8_out(s, a.sx[t], a.sw[rr]);
        if (res) v = (float) res[(size_t) t * a.ldr + rr] + v;
        out[(size_t) t * a.ldo + rr] = (T) v;
    }
}

// ---- tiles ------------------------------------------------------------------------
// A wave covers TM x TN tiles of v_mfma_i32_32x32x32_i8 (TM along the weight rows, TN
// along the tokens), WM x WN of them a workgroup, or WK times as many that share K: each takes
// its part of every stage, and integer sums have no order.  K in stages of KC bytes, a ring of
// NB of them in LDS, filled by LDS DMA.
// What bounds it.  Large: the matrix instructions at the clock that the power leaves: 8192^3 in
// 441 and 459 us in a row of ten or more on two cards (2400 to 2490 TOPS), 517 and 523 for a call alone after a
// wait; the library's int8 product with int32 out, in turn with it, 448 and 463, and 505 and 528 (earlier: 4
// waves of 4 x 4 tiles, which read less from LDS, 5 % slower, a ring of 4 stages of 64 bytes 5 to 10 %).
// 4096 x 8192 x 2048, two rounds of tiles: 70 to 72 us (1930 TOPS; the library 78), of which the outputs, 34
// MB of every unit's at once, are a part that nothing hides.  Small: the latency of the ring's
// start, of a stage and of the launch (333 x 2048 x 2048: 6.1 us).
template <int TM_, int TN_, int WM_, int WN_, int WK_, int KC_, int NB_, int OCC_>
struct LkI8Shape {
    static constexpr int TM = TM_, TN = TN_, WM = WM_, WN = WN_, WK = WK_, KC = KC_, NB = NB_, OCC = OCC_;   // OCC: waves per SIMD
    static constexpr int NW = WM * WN * WK, BM = 32 * TM * WM, BN = 32 * TN * WN, PC = KC / 16;
    static constexpr int BYTES = (BM + BN) * KC;         // a stage: BM weight rows, then BN token rows
    static constexpr int NA = BM * PC / 64, NI = (BM + BN) * PC / 64, PW = NI / NW;
    static_assert(NI % NW == 0 && BM * PC % 64 == 0 && BN * PC % 64 == 0, "whole DMA instructions, the same for every wave");
    static_assert((NB - 2) * PW < 64, "vmcnt range");
    // Rings of two stages go on from tile to tile (MORE): the outputs leave by way of the last
    // stage's buffer while the next tile's first stage is in the other (a workgroup a tile, us:
    // 8192 x 8192 x 2048 146, so 136; 4096 x 8192 x 2048 77 and 73; 8192^3 462 and 448).
    static constexpr bool MORE = NB == 2;
    static constexpr int RS = TM < 2 ? TM : 2, STG = 32 * 32 * RS * 4;       // MFMA tiles of outputs on their way at a time; bytes of a wave
    // the ring, or the parts of K and the outputs where those are more
    static constexpr int PARTS = WM * WN * (WK - 1) * TM * TN * 4096, OUTS = PARTS + WM * WN * STG;
    static constexpr int LDS = NB * BYTES > OUTS ? NB * BYTES : OUTS;
    static_assert(!MORE || (WK == 1 && NW * STG <= BYTES), "the outputs' room");
    static_assert(KC % (32 * WK) == 0 && 16 % PC == 0, "whole steps; a row's pieces divide the 16 slots of all banks");
};
// 16-byte slot of piece p of a row of n pieces: XOR-permuted so that the same piece
// of 16 consecutive rows lies in 16 different slots modulo 256 bytes (all banks).
__device__ __forceinline__ constexpr int lk_i8_slot(int n, int row, int p) { return row * n + (p ^ (row / (16 / n) % n)); }

template <class SH, int TYPE>
__global__ void __launch_bounds__(64 * SH::NW, SH::OCC)
lk_k_gemm_i8(const LkI8Args a) {
    typedef typename LkElem<TYPE>::type T;
    constexpr int TM = SH::TM, TN = SH::TN, KC = SH::KC, NB = SH::NB, NW = SH::NW, PC = SH::PC, PW = SH::PW;
    constexpr bool MORE = SH::MORE;
    constexpr int WMN = SH::WM * SH::WN, NQ = KC / 32 / SH::WK;        // a wave's steps of a stage
    __shared__ __attribute__((aligned(16))) uint8_t stg[SH::LDS];
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    // XCD-aware tile order: workgroups go round-robin over the 8 XCDs (id % 8), so
    // consecutive tiles L are given to one XCD; L runs through groups of 8 row tiles,
    // row tiles first, so that the tiles an XCD works on at a time form a patch
    // whose operands its L2 holds once.
    const int nrt = (a.N - 1) / SH::BM + 1, ntt = (a.M - 1) / SH::BN + 1, ntile = nrt * ntt;
    auto place = [&](int id, int & row0, int & tok0) {
        const int x8 = id & 7, rem = ntile & 7;
        const int L = x8 * (ntile >> 3) + (x8 < rem ? x8 : rem) + (id >> 3);
        const int gr = L / (8 * ntt), gw = nrt - 8 * gr < 8 ? nrt - 8 * gr : 8, li = L - gr * 8 * ntt;
        row0 = (8 * gr + li % gw) * SH::BM;
        tok0 = (li / gw) * SH::BN;
    };
    int row0, tok0;
    place(blockIdx.x, row0, tok0);
    const int kw = w / WMN;                              // the wave's part of every stage
    const int wr = (w % SH::WM) * 32 * TM, wt = (w % WMN / SH::WM) * 32 * TN;
    const int lm = lane & 31, h = lane >> 5;
    const int K = a.K, nst = (K + KC - 1) / KC;

    // DMA instruction i of this wave: slots 64 * (i * NW + w) + lane of a stage
    uint32_t roff[PW];
    const uint32_t pc = (uint32_t) (lk_i8_slot(PC, (64 * w + lane) / PC, lane % PC) % PC * 16);   // the same for all i
    static_assert(4 * NW % PC == 0 && SH::BM % 16 == 0, "a permutation that the wave's instructions share");
    const int8_t * wb, * xb;
    auto aim = [&](int row0, int tok0) {                 // at a tile
#pragma unroll
        for (int i = 0; i < PW; ++i) {
            const int j = i * NW + w;
            const bool isa = j < SH::NA;
            const int r = (64 * (isa ? j : j - SH::NA) + lane) / PC;
            const int lim = isa ? a.N - 1 - row0 : a.M - 1 - tok0;
            roff[i] = (uint32_t) (r < lim ? r : lim) * (uint32_t) (isa ? a.ldw : a.ldx);   // clamped: in bounds
        }
        wb = a.w + (size_t) row0 * a.ldw;
        xb = a.x + (size_t) tok0 * a.ldx;
    };
    const uint32_t lds0 = lk_lds_addr(stg);
    int sb = 0;                                          // the ring's place of the tile's stage 0
    auto fetch = [&](int s, int at, int i) {             // stage s into place at; pieces past the row: its first piece instead
        const int j = i * NW + w;
        const uint32_t k = (uint32_t) (s * KC) + pc;
        lk_dma16c_so(j < SH::NA ? wb : xb, roff[i] + (k < (uint32_t) K ? k : 0u), lds0 + (uint32_t) (at % NB * SH::BYTES + 1024 * j));
    };
    lk_i16v acc[TM][TN];
    lk_i4 av[2][TM], bv[2][TN];
    auto read = [&](int s, int q, int u, int k) {        // operand k of step q of stage s
        const uint8_t * S = stg + (s + sb) % NB * SH::BYTES;
        if (k < TM) av[u][k] = *(const lk_i4 *) (S + lk_i8_slot(PC, wr + 32 * k + lm, 2 * (kw * NQ + q) + h) * 16);
        else bv[u][k - TM] = *(const lk_i4 *) (S + SH::BM * KC + lk_i8_slot(PC, wt + 32 * (k - TM) + lm, 2 * (kw * NQ + q) + h) * 16);
    };
    auto meet = [&] {                                    // the next stage of every wave has landed
        lk_wait_vm<(NB - 2) * PW>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    // A stage: NQ steps of TM x TN MFMAs, in TM groups of TN.  Before each group come its share
    // of the next step's operand reads and of the DMA of stage s + NB - 1 (the ring's free
    // buffer), pinned there: issued all at once at the start of a stage, the DMAs of 8 waves
    // kept the address unit, and with it every wave's MFMAs, waiting.  Before the last step's
    // reads, which are of the next stage, the waves meet: each has its reads of this stage in
    // registers, and its part of the next has landed.
    auto stage = [&](int s, bool last) {
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
            const int u = q & 1;
            if (q + 1 == NQ && !last) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                meet();
            }
            if (last) {
#pragma unroll
                for (int j = 0; j < TN; ++j) bv[u][j] = lk_i8_mask(bv[u][j], s * KC + 32 * (kw * NQ + q) + 16 * h, K);
            }
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                constexpr int ND = TM * (NQ > 1 ? NQ / 2 : 1);       // groups that the DMAs are spread over
#pragma unroll
                for (int k = (TM + TN) * i / TM; k < (TM + TN) * (i + 1) / TM; ++k) {
                    if (q + 1 < NQ) read(s, q + 1, u ^ 1, k);
                    else if (!last) read(s + 1, 0, u ^ 1, k);
                }
                const int g = q * TM + i;
                if (g < ND)
#pragma unroll
                    for (int k = PW * g / ND; k < PW * (g + 1) / ND; ++k) fetch(MORE && last ? 0 : s + NB - 1, s + sb + NB - 1, k);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int j = 0; j < TN; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(av[u][i], bv[u][j], acc[i][j], 0, 0, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    };
    aim(row0, tok0);
#pragma unroll
    for (int s = 0; s < NB - 1; ++s)
#pragma unroll
        for (int i = 0; i < PW; ++i) fetch(s, s, i);     // those past the end: the rows' first pieces, not used
    meet();
    for (int id = blockIdx.x;;) {
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int j = 0; j < TN; ++j)
#pragma unroll
                for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
#pragma unroll
        for (int k = 0; k < TM + TN; ++k) read(0, 0, 0, k);
#pragma unroll 1
        for (int s = 0; s + 1 < nst; ++s) stage(s, false);
        // the last stage brings the next tile's first; after the last tile, its own again
        int row1 = row0, tok1 = tok0;
        if (MORE) {
            id += gridDim.x;
            if (id < ntile) place(id, row1, tok1);
            aim(row1, tok1);
        }
        stage(nst - 1, true);
        // What is on its way lands before LDS is used otherwise (MORE: so that the next tile's first stage
        // needs no wait that the stores below would be part of), and every wave has read its last operands.
        lk_wait_vm<0>();
        // Outputs by way of LDS, 32 tokens and 32 RS rows of the wave at a time: a lane has token
        // lm and rows 8 * e4 + 4 * h .. +3 of every MFMA tile, 8 bytes of 32 output rows per store;
        // from LDS it takes 16 bytes of one token, whole runs of 64 * RS bytes (fp32 128).  They go
        // past the caches' order, which the L2s need for the operands (4096 x 8192 x 2048 bf16 73 us, so
        // 67; 2000 x 4096 x 2048 23.5 and 19.5), and 16 bytes of neighbouring lanes side by side (fp32, 32
        // bytes a lane in two stores: 103 us for 80, and in the caches' order 86).
        // A token's 16-byte pieces are XOR-permuted so that writes and reads use all banks alike.
        constexpr int RS = SH::RS, RW = 32 * RS;
        __syncthreads();
        if constexpr (SH::WK > 1) {                          // the parts of K meet: integer sums have no order
            lk_i16v * pt = (lk_i16v *) stg;
            if (kw > 0) {
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j) pt[((w - WMN) * TM * TN + i * TN + j) * 64 + lane] = acc[i][j];
            }
            __syncthreads();
            if (kw > 0) return;
#pragma unroll
            for (int k = 1; k < SH::WK; ++k)
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int j = 0; j < TN; ++j) acc[i][j] += pt[((k * WMN + w - WMN) * TM * TN + i * TN + j) * 64 + lane];
        }
        // (behind the parts of K, which other waves may still be reading)
        uint8_t * st = stg + (MORE ? (nst - 1 + sb) % NB * SH::BYTES : SH::PARTS) + (w % WMN) * SH::STG;
        auto piece = [&](int t, int p) { return st + t * (RW * 4) + (p ^ (RS == 2 ? t & 15 : t >> 1 & 7)) * 16; };
        const T * res = (const T *) a.res;
        T * out = (T *) a.out;
        constexpr int VL = 16 / sizeof(T), LT = RW / VL, TP = 64 / LT;       // rows a lane, lanes a token, tokens a step
#pragma unroll
        for (int i0 = 0; i0 < TM; i0 += RS) {
            float sw[RS][4][4];
#pragma unroll
            for (int i = 0; i < RS; ++i)
#pragma unroll
                for (int e4 = 0; e4 < 4; ++e4) {
                    const int r = row0 + wr + 32 * (i0 + i) + 8 * e4 + 4 * h;
                    if (r + 4 <= a.N) lk_load<4>(a.sw + r, sw[i][e4]);
                    else
#pragma unroll
                        for (int e = 0; e < 4; ++e) sw[i][e4][e] = r + e < a.N ? a.sw[r + e] : 0.0f;
                }
            const int rl = lane % LT, r = row0 + wr + 32 * i0 + VL * rl;
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const int t0 = tok0 + wt + 32 * j;           // wave-uniform
                const float sx = a.sx[t0 + lm < a.M ? t0 + lm : a.M - 1];
#pragma unroll
                for (int i = 0; i < RS; ++i)
#pragma unroll
                    for (int e4 = 0; e4 < 4; ++e4) {
                        lk_f4 v;
#pragma unroll
                        for (int e = 0; e < 4; ++e) v[e] = lk_i8_out(acc[i0 + i][j][4 * e4 + e], sx, sw[i][e4][e]);
                        *(lk_f4 *) piece(lm, 8 * i + 2 * e4 + h) = v;
                    }
                __builtin_amdgcn_wave_barrier();
                float vv[32 / TP][VL];                       // all of them asked for before the first is stored
#pragma unroll
                for (int k = 0; k < 32 / TP; ++k)
#pragma unroll
                    for (int p = 0; p < VL / 4; ++p) *(lk_f4 *) (vv[k] + 4 * p) = *(const lk_f4 *) piece(k * TP + lane / LT, VL / 4 * rl + p);
#pragma unroll
                for (int k = 0; k < 32 / TP; ++k) {
                    float (&v)[VL] = vv[k];
                    const int t = t0 + k * TP + lane / LT;
                    if (t >= a.M || r >= a.N) continue;
                    if (r + VL <= a.N) {
                        if (res) {
                            float o[VL];
                            lk_load<VL>(res + (size_t) t * a.ldr + r, o);
#pragma unroll
                            for (int e = 0; e < VL; ++e) v[e] = o[e] + v[e];
                        }
                        lk_store_nt<VL>(out + (size_t) t * a.ldo + r, v);
                    } else {
#pragma unroll
                        for (int e = 0; e < VL; ++e) if (r + e < a.N) {
                            float u = v[e];
                            if (res) u = (float) res[(size_t) t * a.ldr + r + e] + u;
                            out[(size_t) t * a.ldo + r + e] = (T) u;
                        }
                    }
                }
                __builtin_amdgcn_wave_barrier();
            }
        }
        if (!MORE || id >= ntile) return;
        row0 = row1;
        tok0 = tok1;
        sb = (sb + nst) % NB;
        __syncthreads();                                     // every wave has left the outputs' room
    }
}

template <int TYPE, int NW>
static void lk_i8_few(const LkI8Args & a, hipStream_t st) {
    hipLaunchKernelGGL((lk_k_gemm_i8_few<TYPE, NW>), dim3((a.N + 15) / 16), dim3(64 * NW), 0, st, a);
}
template <int BM, int BN>
static long lk_i8_ntile(const LkI8Args & a) { return (long) ((a.N - 1) / BM + 1) * ((a.M - 1) / BN + 1); }        // M, N >= 1
template <class SH, int TYPE>
static int lk_i8_tiles(const LkI8Args & a, hipStream_t st) {
    const long n = lk_i8_ntile<SH::BM, SH::BN>(a);       // a grid has fewer than 2^32 threads
    if (n * 64 * SH::NW >= 1l << 32) return lk_fail(hipErrorInvalidValue, "lk_gemm_i8: %d x %d outputs", a.M, a.N);
    // rings that go on: as many workgroups as the units hold (a multiple of the XCDs)
    const long most = SH::MORE ? 256 * ((160 << 10) / SH::LDS) : n;
    hipLaunchKernelGGL((lk_k_gemm_i8<SH, TYPE>), dim3((unsigned) (n < most ? n : most)), dim3(64 * SH::NW), 0, st, a);
    return 0;
}
// Which kernel.  What counts is how many rounds of 256 units the tiles take: the smallest
// tile that fits one round is the best, for a larger one leaves units idle and has fewer waves
// to share K, and a smaller one takes a second round.
// Measured (bf16 out, operands in the cache, ten calls in a graph, us each; * is what the rule takes):
//   M x N x K          few   32x32  64x32  64x64  128x64  128x128  2/unit  256x256
//   1 x 4096 x 4096    4.8*   5.3    6.6    7.4
//   16 x 4096 x 4096   6.1    5.3*
//   1 x 8192 x 2048    4.4*   4.5    5.3    5.6
//   8 x 8192 x 2048    5.0    4.5*   5.4    5.7
//   1 x 8192 x 8192   13.5   12.3*  13.0   15.1    23.1
//   128 x 2048 x 2048         4.7*   5.6    5.8     8.4
//   192 x 2048 x 2048         6.5    5.7*   5.9     8.5     10.0
//   333 x 2048 x 2048         9.0    9.6    6.1*    8.6      9.9
//   640 x 2048 x 2048        13.2   13.7    9.3     8.9*    10.3    12.5
//   1000 x 4096 x 2048                     17.8    15.6     13.7*   15.8    27.9
//   1500 x 4096 x 2048                     26.8    22.5     23.3    20.2*   28.4
//   2048 x 4096 x 2048                     35.8    29.3     27.4    22.5*   29.3
//   2600 x 4096 x 2048                     46.6    40.9     37.8    34.1    30.4*
//   2600 x 8192 x 2048                             73.2     75.3    55.8*   60.3
//   3000 x 8192 x 2048                             80.8     83.6    60.2*   61.3
//   4096 x 8192 x 2048                            107.5    110.8    79.2    70.3*
// Few tokens: 16 rows a workgroup read every token's row again, so that their time grows with M K where
// that of 32x32 does not (few / 32x32; 1, 4, 16 tokens): 4096 x 2048 3.6, 3.7, 4.1 / 4.5; 4096 x 4096 4.8, 5.1,
// 6.1 / 5.3; 4096 x 8192 7.1, 7.8, 9.7 / 8.6 to 9.2; 2048 x 8192 6.8, 7.5, 9.5 / 7.0; 8192 x 1024 3.5, 3.7, 4.2 /
// 4.1; 8192 x 2048 4.4, 4.7, 5.8 / 4.5.
// A round of 256 256x256 tiles takes about 5 / 3 of one of 512 128x128 tiles.
// 64x32 has two forms: K over four waves in stages of 256 bytes (4096 x 128 x 8192 12.2 us, 13.9 with two
// waves and 128), and over two in stages of 128 where K is short (8192 x 64 x 512 4.0, 4.6).
// Up to 32 tokens, wider tiles have nothing to share: many weight rows take the second
// form too, three workgroups a unit: 1 x 32000 x 2048 11.9 (64x64 12.3, 128x64 12.8,
// few 11.3), 32 x 65536 x 2048 22.3 (24.4, 22.9), 16 x 128256 x 4096 92 (96, 98; 5.7 TB/s of weights).
template <int TYPE>
static int lk_i8_shape(const LkI8Args & a, hipStream_t st) {
    const long mk = (long) a.M * a.K;
    if (a.M <= 16 && ((a.N <= 4096 && (a.K <= 2048 || mk <= 16384)) || (a.N <= 8192 && a.K <= 2048 && mk <= 8192))) {
        if (a.K <= 2048) lk_i8_few<TYPE, 4>(a, st);
        else lk_i8_few<TYPE, 8>(a, st);
        return 0;
    }
    if (lk_i8_ntile<32, 32>(a) <= 256) return lk_i8_tiles<LkI8Shape<1, 1, 1, 1, 4, 256, 4, 2>, TYPE>(a, st);
    const bool one = lk_i8_ntile<64, 32>(a) <= 256;      // round
    if (one && a.K >= 2048) return lk_i8_tiles<LkI8Shape<1, 1, 2, 1, 4, 256, 4, 2>, TYPE>(a, st);
    if (one || a.M <= 32) return lk_i8_tiles<LkI8Shape<1, 1, 2, 1, 2, 128, 4, 2>, TYPE>(a, st);
    if (lk_i8_ntile<64, 64>(a) <= 256) return lk_i8_tiles<LkI8Shape<1, 1, 2, 2, 2, 128, 4, 2>, TYPE>(a, st);
    if (lk_i8_ntile<128, 64>(a) <= 256) return lk_i8_tiles<LkI8Shape<2, 1, 2, 2, 2, 128, 3, 2>, TYPE>(a, st);
    const long t128 = lk_i8_ntile<128, 128>(a), t256 = lk_i8_ntile<256, 256>(a);
    if (t128 <= 256) return lk_i8_tiles<LkI8Shape<2, 1, 2, 4, 1, 128, 3, 2>, TYPE>(a, st);
    if (5 * ((t256 + 255) / 256) > 3 * ((t128 + 511) / 512)) return lk_i8_tiles<LkI8Shape<2, 2, 2, 2, 1, 128, 2, 2>, TYPE>(a, st);
    return lk_i8_tiles<LkI8Shape<4, 2, 2, 4, 1, 128, 2, 2>, TYPE>(a, st);
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

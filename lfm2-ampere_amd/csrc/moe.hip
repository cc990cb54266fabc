// moe.hip - a whole mixture-of-experts layer for a few tokens: router, choice of
// experts, their Q4_0 gate / up / down products with SwiGLU, and the weighted sum.
//
// Per token t, in fp32 unless stated:
//     l_e = R_e . x                                          (router rows R, fp32)
//     s_e = sigmoid(l_e), or softmax over the experts
//     the k experts of the largest s_e + bias_e (without a bias: the largest l_e,
//     the same order); of equals the lowest index, NaN below every number
//     w_j = s_j, divided by their sum + 1e-20 when renorm; times scale
//     h_j = silu(G_j x) * (U_j x),  silu(g) = g / (1 + exp(-g))
//     out = res + sum over j, in the order of choice, of w_j * (D_j h_j)
// A Q4_0 block of 32 weights is (n - 8) * d, n = 0..15 (byte i of its 16: element i
// low, element 16 + i high), d fp16.
//
// Exactness: the products run on v_mfma_f32_16x16x32_bf16 with operands that are
// exact.  The weight enters as the bf16 number 16 + n (one AND-OR on two nibbles:
// n at the top of the mantissa of 16.0); the -24 it is too large by is
// -24 * (sum of the block's x), put into the accumulator first.  x and h enter as
// bf16 terms that add up to the value: three (24 bits, all of fp32) for fp32 rows, two
// (16 bits; fp16 and bf16 rows exact, h to 2^-17) for 16-bit rows.  A block's sum is scaled
// by d in fp32 and added in fp32.
#include "lk_types.h"

typedef __bf16 lk_b8 __attribute__((ext_vector_type(8)));
typedef uint32_t lk_u4 __attribute__((ext_vector_type(4)));

#define LK_MOE_THREADS 256
static_assert(LK_MOE_THREADS == LK_MOE_MAX_EXPERTS, "lk_moe_slot: a thread per expert");

struct LkMoeArgs {
    const void * x;
    const void * res;
    void * out;
    const float * router;
    const float * bias;
    const uint8_t * qs[3];               // gate, up, down: [E][rows][bpr] 16-byte blocks
    const _Float16 * d[3];
    int32_t * ids_out;
    float * wts_out;
    // workspace
    float * logits;                      // [T][E]
    __bf16 * xp;                         // [T][NP][hidden] terms of x, permuted within blocks
    float * xs;                          // [T][hidden / 16] -24 * sums of half blocks
    __bf16 * hp;                         // [T * k][NP][ffn]
    float * hs;                          // [T * k][ffn / 16]
    float * y;                           // [T * k][hidden]
    int32_t * ids;                       // [T * k]
    float * wts;                         // [T * k]
    int ldx, ldr, ldo, T, E, k, hidden, ffn, score, renorm;
    float scale;
};

// Position of element m of a block in its plane: lane group g of an MFMA holds the
// eight weights of dword g of the block, in the order in which lk_moe_dequant takes
// them out of it (bytes 0, 2 low, 0, 2 high, 1, 3 low, 1, 3 high).
__device__ __forceinline__ constexpr int lk_moe_pos(int m) {
    return 8 * ((m & 15) >> 2) + 4 * (m & 1) + 2 * (m >> 4) + ((m & 3) >> 1);
}
// The 8 weights of a dword as bf16 16 + n.
__device__ __forceinline__ lk_b8 lk_moe_dequant(uint32_t w) {
    constexpr uint32_t M = 0x00780078u, S = 0x41804180u;
    const lk_u4 v = { ((w << 3) & M) | S, ((w >> 1) & M) | S, ((w >> 5) & M) | S, ((w >> 9) & M) | S };
    return __builtin_bit_cast(lk_b8, v);
}
// v as NP bf16 terms by truncation: every remainder is exact, and no term
// overflows.
template <int NP>
__device__ __forceinline__ void lk_moe_split(float v, uint16_t (&t)[NP]) {
#pragma unroll
    for (int p = 0; p < NP; ++p) {
        const uint32_t u = __builtin_bit_cast(uint32_t, v);
        if (p + 1 == NP && NP == 2) {                    // the last of two: rounded
            t[p] = __builtin_bit_cast(uint16_t, (__bf16) v);
        } else {
            t[p] = (uint16_t) (u >> 16);
            v -= __builtin_bit_cast(float, u & 0xFFFF0000u);
        }
    }
}
// Dwords j of lane groups g (16 lanes each) transposed: afterwards register j of
// group g is what register g of group j was.
__device__ __forceinline__ void lk_moe_transpose(lk_u4 & w) {
#ifdef __HIP_DEVICE_COMPILE__
    uint32_t a = w[0], b = w[1], c = w[2], d = w[3];
    asm("s_nop 1\n\tv_permlane32_swap_b32 %0, %2\n\tv_permlane32_swap_b32 %1, %3\n\ts_nop 1\n\t"
        "v_permlane16_swap_b32 %0, %1\n\tv_permlane16_swap_b32 %2, %3\n\ts_nop 1"
        : "+v"(a), "+v"(b), "+v"(c), "+v"(d));
    w = lk_u4{ a, b, c, d };
#endif
}

// ---- router scores, and the terms of x -------------------------------------------
// Workgroups 0 .. nE-1 (of blockIdx.x): one expert per wave, four tokens; the rest:
// the terms and half-block sums of four tokens, four threads per block of 32.
template <int TYPE, int NP>
__global__ void __launch_bounds__(LK_MOE_THREADS)
lk_k_moe_router(const LkMoeArgs a, int nE) {
    typedef typename LkElem<TYPE>::type T;
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6;
    const int t0 = blockIdx.y * 4, H = a.hidden;
    const T * x = (const T *) a.x;
    if ((int) blockIdx.x < nE) {
        const int e = blockIdx.x * 4 + wv;
        if (e >= a.E) return;
        const float * r = a.router + (size_t) e * H;
        float s[4] = { 0.0f, 0.0f, 0.0f, 0.0f };
        for (int i = lane * 8; i < H; i += 512) {        // H is a multiple of 32: whole pieces
            float w[8];
            lk_load<8>(r + i, w);
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int t = t0 + k < a.T ? t0 + k : a.T - 1;
                float v[8];
                lk_load<8>(x + (size_t) t * a.ldx + i, v);
#pragma unroll
                for (int j = 0; j < 8; ++j) s[k] = __builtin_fmaf(w[j], v[j], s[k]);
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            s[k] = lk_wave_sum(s[k]);
            if (lane == 0 && t0 + k < a.T) a.logits[(size_t) (t0 + k) * a.E + e] = s[k];
        }
        return;
    }
    const int u = (blockIdx.x - nE) * LK_MOE_THREADS + threadIdx.x, b = u >> 2, g = u & 3, bpr = H / 32;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int t = t0 + k;
        const bool ok = t < a.T && b < bpr;              // the same for the four threads of a block
        float lo[4] = { 0 }, hi[4] = { 0 };
        if (ok) {
            lk_load<4>(x + (size_t) t * a.ldx + 32 * b + 4 * g, lo);
            lk_load<4>(x + (size_t) t * a.ldx + 32 * b + 16 + 4 * g, hi);
        }
        float s0 = (lo[0] + lo[1]) + (lo[2] + lo[3]), s1 = (hi[0] + hi[1]) + (hi[2] + hi[3]);
        s0 += lk_dpp<LK_DPP_QP_XOR1>(s0);
        s0 += lk_dpp<LK_DPP_QP_XOR2>(s0);
        s1 += lk_dpp<LK_DPP_QP_XOR1>(s1);
        s1 += lk_dpp<LK_DPP_QP_XOR2>(s1);
        if (!ok) continue;
        uint16_t q[8][NP];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            lk_moe_split<NP>(lo[j], q[lk_moe_pos(j)]);
            lk_moe_split<NP>(hi[j], q[lk_moe_pos(16 + j)]);
        }
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            lk_u16x8 v;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[j] = q[j][p];
            *(lk_u16x8 *) (a.xp + ((size_t) (t * NP + p) * bpr + b) * 32 + 8 * g) = v;
        }
        if (g == 0) *(float2 *) (a.xs + ((size_t) t * bpr + b) * 2) = make_float2(-24.0f * s0, -24.0f * s1);
    }
}

// ---- choice of experts --------------------------------------------------------------
// 16 lanes per token: lane i holds experts i, i + 16, ...; a round finds the best that
// is left over the 16 lanes.
__device__ __forceinline__ uint32_t lk_moe_key(float r) {    // orderable bits; NaN lowest, -0 as 0
    const uint32_t u = __builtin_bit_cast(uint32_t, r + 0.0f);
    return r != r ? 0u : (u >> 31) ? ~u : u | 0x80000000u;
}
template <int CTRL>
__device__ __forceinline__ void lk_moe_better(uint32_t & key, uint32_t & e) {
    const uint32_t k2 = lk_dpp_u<CTRL>(key), e2 = lk_dpp_u<CTRL>(e);
    const bool take = k2 > key || (k2 == key && e2 < e);
    key = take ? k2 : key;
    e = take ? e2 : e;
}
// The experts of every token and their weights into LDS (ids, wts: [T * k]); all
// threads of the workgroup, a barrier at the end.
__device__ __forceinline__ void lk_moe_choose(const LkMoeArgs & a, int * ids, float * wts) {
    constexpr int NL = LK_MOE_MAX_EXPERTS / 16;
    const int i16 = threadIdx.x & 15;
    for (int t = threadIdx.x >> 4; t < a.T; t += LK_MOE_THREADS / 16) {
        float l[NL];
        uint32_t key[NL];
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int e = 16 * i + i16;
            l[i] = 16 * i < a.E && e < a.E ? a.logits[(size_t) t * a.E + e] : -__builtin_inff();
        }
        float m = -__builtin_inff(), z = 0.0f;
        if (a.score == LK_MOE_SOFTMAX) {
#pragma unroll
            for (int i = 0; i < NL; ++i) if (16 * i < a.E) m = fmaxf(m, l[i]);
            m = lk_row_max16(m);
#pragma unroll
            for (int i = 0; i < NL; ++i) if (16 * i < a.E) z += 16 * i + i16 < a.E ? expf(l[i] - m) : 0.0f;
            z = lk_row_sum16(z);
        }
        auto score = [&](float v) {
            return a.score == LK_MOE_SOFTMAX ? expf(v - m) / z : 1.0f / (1.0f + expf(-v));
        };
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int e = 16 * i + i16;
            key[i] = 0;
            if (16 * i < a.E && e < a.E) key[i] = lk_moe_key(a.bias ? score(l[i]) + a.bias[e] : l[i]);
        }
        uint32_t used = 0;
        float sum = 0.0f, mine = 0.0f;
        for (int j = 0; j < a.k; ++j) {
            uint32_t bk = 0, be = 0xFFFFu;
            float bl = 0.0f;
#pragma unroll
            for (int i = 0; i < NL; ++i) if (16 * i < a.E) {
                const uint32_t e = 16 * i + i16;
                const bool take = (int) e < a.E && !(used >> i & 1) && (be == 0xFFFFu || key[i] > bk);
                bk = take ? key[i] : bk;
                bl = take ? l[i] : bl;
                be = take ? e : be;
            }
            const uint32_t own = be;
            lk_moe_better<LK_DPP_QP_XOR1>(bk, be);
            lk_moe_better<LK_DPP_QP_XOR2>(bk, be);
            lk_moe_better<LK_DPP_HMIRROR>(bk, be);
            lk_moe_better<LK_DPP_MIRROR>(bk, be);
            if (own == be) used |= 1u << (be / 16);
            // the chosen expert's logit, from the lane that holds it (j < k <= E: there is one)
            const float s = score(__shfl(bl, (threadIdx.x & 48) + (int) (be & 15), 64));
            sum += s;
            if (i16 == j) mine = s;
            if (i16 == 0) ids[t * a.k + j] = (int) be;
        }
        if (a.renorm) mine = mine / (sum + 1e-20f);
        if (i16 < a.k) wts[t * a.k + i16] = mine * a.scale;
    }
    __syncthreads();
}

// The expert of a slot (the slot-th of those that any token chose, by index) and the
// assignments t * k + j that chose it, in order, into list; returns the expert or
// -1, their number in count.  All threads, barriers inside.
__device__ __forceinline__ int lk_moe_slot(const LkMoeArgs & a, const int * ids, int slot, int * list, int & count) {
    __shared__ uint8_t met[LK_MOE_MAX_EXPERTS];
    __shared__ uint64_t words[LK_MOE_MAX_EXPERTS / 64];
    __shared__ int s_e, s_n;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6, na = a.T * a.k;
    if (tid < LK_MOE_MAX_EXPERTS) met[tid] = 0;
    if (tid == 0) s_e = -1;
    __syncthreads();
    for (int i = tid; i < na; i += LK_MOE_THREADS) met[ids[i]] = 1;
    __syncthreads();
    const bool m = met[tid] != 0;                        // LK_MOE_THREADS == LK_MOE_MAX_EXPERTS
    const uint64_t word = __ballot(m);
    if (lane == 0) words[wv] = word;
    __syncthreads();
    int before = __popcll(word & ((1ull << lane) - 1));
    for (int i = 0; i < wv; ++i) before += __popcll(words[i]);
    if (m && before == slot) s_e = tid;
    __syncthreads();
    const int e = s_e;
    if (e >= 0 && wv == 0) {
        int n = 0;
        for (int i0 = 0; i0 < na; i0 += 64) {
            const bool hit = i0 + lane < na && ids[i0 + lane] == e;
            const uint64_t b = __ballot(hit);
            if (hit) list[n + __popcll(b & ((1ull << lane) - 1))] = i0 + lane;
            n += __popcll(b);
        }
        if (lane == 0) s_n = n;
    }
    __syncthreads();
    count = e >= 0 ? s_n : 0;
    return e;
}

// ---- the products -------------------------------------------------------------------
// 16 weight rows of NM matrices times 4 rows of terms, over the block groups
// (4 blocks) g0, g0 + gs, ... below (bpr + 3) / 4.  Lane (c = l % 16, g = l / 16)
// loads block g of a group of its weight row c, whole (16 bytes); the transpose gives it
// dword g of each of the four.  The A operand has row 4b + t = block b of term row
// t, so that one register serves all four blocks: in the product with block j's
// weights only rows 4j + t mean something, and those arrive in lane group j.  Lane
// group g takes its four results of block g there, times its own row's d.
// acc[m][t]: the part of this lane's block column; the sum over the four lane groups
// is the caller's.
template <int NP, int NM, int U>
__device__ __forceinline__ void lk_moe_rows(const uint8_t * const (&qs)[NM], const _Float16 * const (&d)[NM],
                                            const __bf16 * planes, const float * seeds, int bpr, int arow,
                                            const int (&trow)[4], int g0, int gs, float (&acc)[NM][4]) {
    const int lane = threadIdx.x & 63, g = lane >> 4, ab = (lane & 15) >> 2;
    const int ng = (bpr + 3) / 4;
    const __bf16 * ap = planes + (size_t) arow * NP * bpr * 32 + 8 * g;
    const float * sp[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) sp[r] = seeds + (size_t) trow[r] * bpr * 2;
    for (int gi = g0; gi < ng; gi += gs * U) {
        lk_u4 w[U][NM];
        _Float16 dw[U][NM];
        lk_b8 av[U][NP];
        float2 sd[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = gi + u * gs < ng ? gi + u * gs : ng - 1;
            const int bw = 4 * i + g < bpr ? 4 * i + g : bpr - 1, ba = 4 * i + ab < bpr ? 4 * i + ab : bpr - 1;   // in bounds
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                w[u][m] = *(const lk_u4 *) (qs[m] + (size_t) bw * 16);
                dw[u][m] = d[m][bw];
            }
#pragma unroll
            for (int p = 0; p < NP; ++p) av[u][p] = *(const lk_b8 *) (ap + ((size_t) p * bpr + ba) * 32);
#pragma unroll
            for (int r = 0; r < 4; ++r) sd[u][r] = *(const float2 *) (sp[r] + 2 * bw);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (gi + u * gs >= ng) break;                // wave-uniform
            const bool in = 4 * (gi + u * gs) + g < bpr; // a block of the last, ragged group that is not there: d 0
            lk_f4 seed;
#pragma unroll
            for (int r = 0; r < 4; ++r) seed[r] = sd[u][r].x + sd[u][r].y;
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                lk_moe_transpose(w[u][m]);
                lk_f4 D[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const lk_b8 b = lk_moe_dequant(w[u][m][j]);
                    D[j] = seed;
#pragma unroll
                    for (int p = NP - 1; p >= 0; --p) D[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av[u][p], b, D[j], 0, 0, 0);
                }
                const float dv = in ? (float) dw[u][m] : 0.0f;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float s = g == 0 ? D[0][r] : g == 1 ? D[1][r] : g == 2 ? D[2][r] : D[3][r];
                    acc[m][r] = __builtin_fmaf(dv, s, acc[m][r]);
                }
            }
        }
    }
}

template <int NP>
__global__ void __launch_bounds__(LK_MOE_THREADS)
lk_k_moe_up(const LkMoeArgs a) {
    __shared__ int ids[LK_MOE_MAX_TOKENS * LK_MOE_MAX_TOP_K];
    __shared__ float wts[LK_MOE_MAX_TOKENS * LK_MOE_MAX_TOP_K];
    __shared__ int list[LK_MOE_MAX_TOKENS];
    __shared__ float part[4][2][4][16];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    lk_moe_choose(a, ids, wts);
    if (blockIdx.x == 0 && blockIdx.y == 0)
        for (int i = tid; i < a.T * a.k; i += LK_MOE_THREADS) {
            a.ids[i] = ids[i];
            a.wts[i] = wts[i];
            if (a.ids_out) a.ids_out[i] = ids[i];
            if (a.wts_out) a.wts_out[i] = wts[i];
        }
    int n;
    const int e = __builtin_amdgcn_readfirstlane(lk_moe_slot(a, ids, blockIdx.y, list, n));
    if (e < 0) return;
    const int bpr = a.hidden / 32, F = a.ffn, r0 = blockIdx.x * 16;
    const size_t row = (size_t) e * F + r0 + c;          // F is a multiple of 32: whole tiles
    const uint8_t * const qs[2] = { a.qs[0] + row * bpr * 16, a.qs[1] + row * bpr * 16 };
    const _Float16 * const d[2] = { a.d[0] + row * bpr, a.d[1] + row * bpr };
    for (int n0 = 0; n0 < n; n0 += 4) {
        int trow[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) trow[r] = list[n0 + r < n ? n0 + r : n0] / a.k;
        const int arow = list[n0 + (lane & 3) < n ? n0 + (lane & 3) : n0] / a.k;
        float acc[2][4] = {};
        lk_moe_rows<NP, 2, 4>(qs, d, a.xp, a.xs, bpr, arow, trow, wv, 4, acc);
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float v = lk_xrow_sum(acc[m][r]);
                if (g == r) part[wv][m][r][c] = v;
            }
        __syncthreads();
        if (tid < 64) {                                  // token g of the four, row c
            const float gt = (part[0][0][g][c] + part[1][0][g][c]) + (part[2][0][g][c] + part[3][0][g][c]);
            const float up = (part[0][1][g][c] + part[1][1][g][c]) + (part[2][1][g][c] + part[3][1][g][c]);
            const float h = gt / (1.0f + expf(-gt)) * up;
            const float s = -24.0f * lk_row_sum16(h);
            if (n0 + g < n) {
                const int as = list[n0 + g], f = r0 + c;
                uint16_t q[NP];
                lk_moe_split<NP>(h, q);
#pragma unroll
                for (int p = 0; p < NP; ++p)
                    ((uint16_t *) a.hp)[(size_t) (as * NP + p) * F + (f & ~31) + lk_moe_pos(f & 31)] = q[p];
                if (c == 0) a.hs[(size_t) as * (F / 16) + r0 / 16] = s;
            }
        }
        __syncthreads();
    }
}

template <int NP>
__global__ void __launch_bounds__(LK_MOE_THREADS)
lk_k_moe_down(const LkMoeArgs a) {
    __shared__ int ids[LK_MOE_MAX_TOKENS * LK_MOE_MAX_TOP_K];
    __shared__ int list[LK_MOE_MAX_TOKENS];
    __shared__ float part[4][4][16];
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    for (int i = tid; i < a.T * a.k; i += LK_MOE_THREADS) ids[i] = a.ids[i];
    __syncthreads();
    int n;
    const int e = __builtin_amdgcn_readfirstlane(lk_moe_slot(a, ids, blockIdx.y, list, n));
    if (e < 0) return;
    const int bpr = a.ffn / 32, H = a.hidden, r0 = blockIdx.x * 16;
    const size_t row = (size_t) e * H + r0 + c;
    const uint8_t * const qs[1] = { a.qs[2] + row * bpr * 16 };
    const _Float16 * const d[1] = { a.d[2] + row * bpr };
    for (int n0 = 0; n0 < n; n0 += 4) {
        int trow[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) trow[r] = list[n0 + r < n ? n0 + r : n0];
        const int arow = list[n0 + (lane & 3) < n ? n0 + (lane & 3) : n0];
        float acc[1][4] = {};
        lk_moe_rows<NP, 1, 4>(qs, d, a.hp, a.hs, bpr, arow, trow, wv, 4, acc);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float v = lk_xrow_sum(acc[0][r]);
            if (g == r) part[wv][r][c] = v;
        }
        __syncthreads();
        if (tid < 64 && n0 + g < n)
            a.y[(size_t) list[n0 + g] * H + r0 + c] = (part[0][g][c] + part[1][g][c]) + (part[2][g][c] + part[3][g][c]);
        __syncthreads();
    }
}

template <int TYPE>
__global__ void __launch_bounds__(LK_MOE_THREADS)
lk_k_moe_sum(const LkMoeArgs a) {
    typedef typename LkElem<TYPE>::type T;
    const int t = blockIdx.y, i = (blockIdx.x * LK_MOE_THREADS + threadIdx.x) * 4;
    if (i >= a.hidden) return;
    float o[4] = {};
    for (int j = 0; j < a.k; ++j) {
        const int as = t * a.k + j;
        const float w = a.wts[as];
        const float4 y = *(const float4 *) (a.y + (size_t) as * a.hidden + i);
        o[0] = __builtin_fmaf(w, y.x, o[0]);
        o[1] = __builtin_fmaf(w, y.y, o[1]);
        o[2] = __builtin_fmaf(w, y.z, o[2]);
        o[3] = __builtin_fmaf(w, y.w, o[3]);
    }
    if (a.res) {
        float r[4];
        lk_load<4>((const T *) a.res + (size_t) t * a.ldr + i, r);
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = r[k] + o[k];
    }
    lk_store<4>((T *) a.out + (size_t) t * a.ldo + i, o);
}

// ---- host ---------------------------------------------------------------------------
static int lk_moe_check(const lk_moe * m) {
    if (!m) return lk_fail(hipErrorInvalidValue, "lk_moe: null description");
    if (m->n_experts < 1 || m->n_experts > LK_MOE_MAX_EXPERTS || m->top_k < 1 || m->top_k > LK_MOE_MAX_TOP_K || m->top_k > m->n_experts)
        return lk_fail(hipErrorInvalidValue, "lk_moe: %d experts (1..%d), top_k %d (1..%d, at most the experts)", m->n_experts,
                       LK_MOE_MAX_EXPERTS, m->top_k, LK_MOE_MAX_TOP_K);
    if (m->hidden < 32 || m->hidden % 32 || m->hidden > LK_MOE_MAX_DIM || m->ffn < 32 || m->ffn % 32 || m->ffn > LK_MOE_MAX_DIM)
        return lk_fail(hipErrorInvalidValue, "lk_moe: hidden %d, ffn %d must be multiples of 32 up to %d", m->hidden, m->ffn, LK_MOE_MAX_DIM);
    if ((m->score != LK_MOE_SIGMOID && m->score != LK_MOE_SOFTMAX))
        return lk_fail(hipErrorInvalidValue, "lk_moe: score %d", m->score);
    return 0;
}
// The workspace's parts, every one at a multiple of 16 bytes.
static size_t lk_moe_layout(const lk_moe * m, int T, void * work, LkMoeArgs * a) {
    size_t at = 0;
    const size_t k = m->top_k, H = m->hidden, F = m->ffn, NP = 3;
    auto take = [&](size_t bytes) {
        char * p = work ? (char *) work + at : nullptr;
        at += (bytes + 15) & ~(size_t) 15;
        return (void *) p;
    };
    LkMoeArgs b = {};
    LkMoeArgs * o = a ? a : &b;
    o->logits = (float *) take(4 * (size_t) T * m->n_experts);
    o->xp = (__bf16 *) take(2 * T * NP * H);
    o->xs = (float *) take(4 * T * (H / 16));
    o->hp = (__bf16 *) take(2 * T * k * NP * F);
    o->hs = (float *) take(4 * T * k * (F / 16));
    o->y = (float *) take(4 * T * k * H);
    o->ids = (int32_t *) take(4 * T * k);
    o->wts = (float *) take(4 * T * k);
    return at;
}
extern "C" size_t lk_moe_work_bytes(const lk_moe * moe, int T) {
    if (lk_moe_check(moe) || T < 0 || T > LK_MOE_MAX_TOKENS) return 0;
    return lk_moe_layout(moe, T, nullptr, nullptr);
}

template <int TYPE>
static void lk_moe_go(const LkMoeArgs & a, hipStream_t st) {
    constexpr int NP = TYPE == LK_F32 ? 3 : 2;
    const int nE = (a.E + 3) / 4, slots = a.T * a.k < a.E ? a.T * a.k : a.E;
    hipLaunchKernelGGL((lk_k_moe_router<TYPE, NP>), dim3(nE + (a.hidden / 8 + LK_MOE_THREADS - 1) / LK_MOE_THREADS, (a.T + 3) / 4),
                       dim3(LK_MOE_THREADS), 0, st, a, nE);
    hipLaunchKernelGGL((lk_k_moe_up<NP>), dim3(a.ffn / 16, slots), dim3(LK_MOE_THREADS), 0, st, a);
    hipLaunchKernelGGL((lk_k_moe_down<NP>), dim3(a.hidden / 16, slots), dim3(LK_MOE_THREADS), 0, st, a);
    hipLaunchKernelGGL((lk_k_moe_sum<TYPE>), dim3((a.hidden / 4 + LK_MOE_THREADS - 1) / LK_MOE_THREADS, a.T), dim3(LK_MOE_THREADS), 0, st, a);
}

extern "C" int lk_moe_q4_0(const lk_moe * moe, int type, const void * x, int ldx, int T, const void * res, int ldr,
                           void * out, int ldo, int32_t * ids, float * weights, void * work, size_t work_bytes,
                           void * stream) {
    const int rc = lk_moe_check(moe);
    if (rc) return rc;
    if (!lk_type_ok(type) || T < 0 || T > LK_MOE_MAX_TOKENS)
        return lk_fail(hipErrorInvalidValue, "lk_moe_q4_0: type %d / %d tokens (0..%d)", type, T, LK_MOE_MAX_TOKENS);
    if (T == 0) return 0;
    if (!x || !out || !work || !moe->router || !moe->gate_qs || !moe->gate_d || !moe->up_qs || !moe->up_d || !moe->down_qs || !moe->down_d)
        return lk_fail(hipErrorInvalidValue, "lk_moe_q4_0: null pointer argument");
    if (ldx < moe->hidden || ldo < moe->hidden || (res && ldr < moe->hidden))
        return lk_fail(hipErrorInvalidValue, "lk_moe_q4_0: row strides x %d, out %d, res %d for hidden %d", ldx, ldo, ldr, moe->hidden);
    const uintptr_t em = (uintptr_t) lk_type_size(type) - 1;
    if (((uintptr_t) x & em) || ((uintptr_t) out & em) || ((uintptr_t) res & em) || ((uintptr_t) moe->router & 3) ||
        ((uintptr_t) moe->bias & 3) || ((uintptr_t) ids & 3) || ((uintptr_t) weights & 3) || ((uintptr_t) work & 15) ||
        ((uintptr_t) moe->gate_qs & 15) || ((uintptr_t) moe->up_qs & 15) || ((uintptr_t) moe->down_qs & 15) ||
        ((uintptr_t) moe->gate_d & 1) || ((uintptr_t) moe->up_d & 1) || ((uintptr_t) moe->down_d & 1))
        return lk_fail(hipErrorInvalidValue, "lk_moe_q4_0: misaligned argument (blocks and workspace 16 B, block scales 2 B, rows by their element, the rest 4 B)");
    LkMoeArgs a = {};
    const size_t need = lk_moe_layout(moe, T, work, &a);
    if (work_bytes < need)
        return lk_fail(hipErrorInvalidValue, "lk_moe_q4_0: workspace of %zu bytes, %zu needed for %d tokens", work_bytes, need, T);
    a.x = x; a.res = res; a.out = out;
    a.router = moe->router; a.bias = moe->bias;
    a.qs[0] = (const uint8_t *) moe->gate_qs; a.qs[1] = (const uint8_t *) moe->up_qs; a.qs[2] = (const uint8_t *) moe->down_qs;
    a.d[0] = (const _Float16 *) moe->gate_d; a.d[1] = (const _Float16 *) moe->up_d; a.d[2] = (const _Float16 *) moe->down_d;
    a.ids_out = ids; a.wts_out = weights;
    a.ldx = ldx; a.ldr = ldr; a.ldo = ldo; a.T = T; a.E = moe->n_experts; a.k = moe->top_k;
    a.hidden = moe->hidden; a.ffn = moe->ffn; a.score = moe->score; a.renorm = moe->renorm; a.scale = moe->scale;
    const hipStream_t st = lk_stream(stream);
    if (type == LK_F32)      lk_moe_go<LK_F32>(a, st);
    else if (type == LK_F16) lk_moe_go<LK_F16>(a, st);
    else                     lk_moe_go<LK_BF16>(a, st);
    return lk_launch_status("lk_moe_q4_0");
}

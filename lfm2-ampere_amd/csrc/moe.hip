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
// The products are integer dot products (v_dot4_i32_i8): a block of 32 values of x or h
// becomes whole numbers i = rint(v * 2^p), the largest just inside the range, in NP
// int8 digits of base 256: three for fp32 rows (24 bits of the block's largest value), two
// for fp16 and bf16 rows (16 bits).  sum (n - 8) i is exact in int32 digit by digit
// (-8 * the digits' sum is where the sum starts), the digits are put together and scaled by
// d * 2^-p in fp32, and blocks are added in fp32.  A block that holds a value
// that is not finite gets the scale NaN; one whose largest value is under 2^-100 counts as
// zero.
#include "lk_types.h"

typedef uint32_t lk_u4 __attribute__((ext_vector_type(4)));

// Up to this many tokens every workgroup chooses the experts itself, a wave per
// token, and the down product adds the experts up itself (three launches); above it a
// launch of one workgroup chooses once and sorts the tokens by expert, and another
// adds up (five).
#define LK_MOE_FEW 8
#define LK_MOE_THREADS 256                // router and sum
#define LK_MOE_NW 8                       // waves of a gate/up or down workgroup
#define LK_MOE_NWF 16                     // of a down workgroup for few tokens

// The assignments (token * k + j) sorted by expert: expert e[s] of slot s has those of
// list[from[s]] .. list[from[s + 1] - 1].
struct LkMoeTab {
    int32_t slots;
    int32_t e[LK_MOE_MAX_EXPERTS];
    int32_t from[LK_MOE_MAX_EXPERTS + 1];
    int32_t list[LK_MOE_MAX_TOKENS * LK_MOE_MAX_TOP_K];
};

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
    uint8_t * xr;                        // [T][hidden / 32] records (LkMoeRec) of x
    uint8_t * hr;                        // [T * k][ffn / 32] records of h
    float * y;                           // [T * k][hidden]
    int32_t * ids;                       // [T * k]
    float * wts;                         // [T * k]
    int32_t * tab;                       // LkMoeTab, for more than LK_MOE_FEW tokens
    int ldx, ldr, ldo, T, E, k, hidden, ffn, score, renorm;
    float scale;
};

// ---- whole numbers of a block -------------------------------------------------------
// A block's record: NP planes of 32 int8 digits, highest first, then int32 -8 * sum of
// each plane (0 for a third of two) and the fp32 scale 2^-p.
template <int NP>
struct LkMoeRec {
    static constexpr int PIECES = 2 * NP + 1, BYTES = 16 * PIECES;
};
// 2^p for a block whose largest |v| has the bits am; 0 for a block of zeros and for one
// that is not finite.  The digits reach 127 * (1 + 256 (+ 65536)): the largest value
// goes to the top binade where its leading bits allow, else one below.
template <int NP>
__device__ __forceinline__ float lk_moe_up2(uint32_t am) {
    constexpr float TOP = NP == 3 ? 8355711.0f : 32639.0f;
    constexpr int B = NP == 3 ? 22 : 14;
    if (am >= 0x7F800000u || am < (27u << 23)) return 0.0f;                       // not finite; under 2^-100
    // 2^(B - E), E the exponent of am, by way of two factors: the exponent of one may leave the range
    const int E = (int) (am >> 23) - 127;
    const float f = ldexpf(1.0f, B - E);
    return __builtin_bit_cast(float, am) * f > TOP ? 0.5f * f : f;
}
__device__ __forceinline__ float lk_moe_scale(uint32_t am, float up) {            // 2^-p; NaN for what is not finite
    return am >= 0x7F800000u ? __builtin_nanf("") : up == 0.0f ? 0.0f : 1.0f / up; // a power of two: exact
}
template <int NP>
__device__ __forceinline__ void lk_moe_digits(float v, float up, int (&q)[NP]) {
    int i = up == 0.0f ? 0 : (int) __builtin_rintf(v * up);
#pragma unroll
    for (int p = NP - 1; p > 0; --p) {
        q[p] = (int) (int8_t) i;
        i = (i - q[p]) >> 8;
    }
    q[0] = i;
}

// ---- router scores, and the records of x -------------------------------------------
// Workgroups 0 .. nE-1 (of blockIdx.x): one expert per wave, four tokens; the rest:
// the records of four tokens, four threads per block of 32.
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
    constexpr int REC = LkMoeRec<NP>::BYTES;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int t = t0 + k;
        const bool ok = t < a.T && b < bpr;              // the same for the four threads of a block
        float v[8] = { 0 };
        if (ok) lk_load<8>(x + (size_t) t * a.ldx + 32 * b + 8 * g, v);
        uint32_t am = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) am = lk_umax(am, __builtin_bit_cast(uint32_t, v[j]) & 0x7FFFFFFFu);
        am = lk_umax(am, lk_dpp_u<LK_DPP_QP_XOR1>(am));
        am = lk_umax(am, lk_dpp_u<LK_DPP_QP_XOR2>(am));
        const float up = lk_moe_up2<NP>(am);
        uint32_t w[NP][2] = {};
        int s[3] = { 0, 0, 0 };
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            int q[NP];
            lk_moe_digits<NP>(v[j], up, q);
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                w[p][j / 4] |= (uint32_t) (uint8_t) q[p] << (8 * (j % 4));
                s[p] += q[p];
            }
        }
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            s[p] += (int) lk_dpp_u<LK_DPP_QP_XOR1>((uint32_t) s[p]);
            s[p] += (int) lk_dpp_u<LK_DPP_QP_XOR2>((uint32_t) s[p]);
        }
        if (!ok) continue;
        uint8_t * r = a.xr + ((size_t) t * bpr + b) * REC;
#pragma unroll
        for (int p = 0; p < NP; ++p) *(uint2 *) (r + 32 * p + 8 * g) = make_uint2(w[p][0], w[p][1]);
        if (g == 0)
            *(lk_i4 *) (r + 32 * NP) = lk_i4{ -8 * s[0], -8 * s[1], -8 * s[2], __builtin_bit_cast(int, lk_moe_scale(am, up)) };
    }
}

// ---- choice of experts --------------------------------------------------------------
// A wave per token: lane i holds experts i, i + 64, ...  A round takes the largest key
// that is left; the first register and then the first lane that holds it are the
// lowest index.
__device__ __forceinline__ uint32_t lk_moe_key(float r) {    // orderable bits; 0: taken, 1: NaN; -0 as 0
    const uint32_t u = __builtin_bit_cast(uint32_t, r + 0.0f);
    return r != r ? 1u : (u >> 31) ? ~u : u | 0x80000000u;
}
// Token t's experts and weights into ids[0 .. k-1] and wts[0 .. k-1] (LDS).
__device__ __forceinline__ void lk_moe_choose(const LkMoeArgs & a, int t, int * ids, float * wts) {
    constexpr int NL = LK_MOE_MAX_EXPERTS / 64;
    const int lane = threadIdx.x & 63;
    float l[NL];
    uint32_t key[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const int e = 64 * i + lane;
        l[i] = e < a.E ? a.logits[(size_t) t * a.E + e] : -__builtin_inff();
    }
    float m = -__builtin_inff(), z = 1.0f;
    if (a.score == LK_MOE_SOFTMAX) {
#pragma unroll
        for (int i = 0; i < NL; ++i) m = fmaxf(m, l[i]);
        m = lk_xrow_max(lk_row_max16(m));
        z = 0.0f;
#pragma unroll
        for (int i = 0; i < NL; ++i) if (64 * i < a.E) z += 64 * i + lane < a.E ? expf(l[i] - m) : 0.0f;
        z = lk_wave_sum(z);
    }
    auto score = [&](float v) {
        return a.score == LK_MOE_SOFTMAX ? expf(v - m) / z : 1.0f / (1.0f + expf(-v));
    };
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const int e = 64 * i + lane;
        key[i] = 0;
        if (64 * i < a.E) {
            const float r = a.bias ? score(l[i]) + a.bias[e < a.E ? e : 0] : l[i];
            key[i] = e < a.E ? lk_moe_key(r) : 0;
        }
    }
    float mine = 0.0f;                                   // lane j: the logit of choice j
    int id = 0;
    for (int j = 0; j < a.k; ++j) {
        uint32_t best = key[0];
#pragma unroll
        for (int i = 1; i < NL; ++i) best = lk_umax(best, key[i]);
        best = (uint32_t) __builtin_amdgcn_readfirstlane((int) lk_wave_umax(best));
        int e = -1;
        float v = 0.0f;
#pragma unroll
        for (int i = NL - 1; i >= 0; --i) {
            const uint64_t b = __ballot(key[i] == best);
            if (b) {                                     // at least one: k <= E
                e = 64 * i + __builtin_ctzll(b);
                v = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, l[i]), e & 63));
            }
        }
#pragma unroll
        for (int i = 0; i < NL; ++i) key[i] = 64 * i + lane == e ? 0 : key[i];
        mine = lane == j ? v : mine;
        id = lane == j ? e : id;
    }
    const float s = lane < a.k ? score(mine) : 0.0f;
    float w = s;
    if (a.renorm) w = s / (lk_row_sum16(s) + 1e-20f);    // k <= 8: the first row of 16 lanes
    if (lane < a.k) {
        ids[lane] = id;
        wts[lane] = w * a.scale;
    }
}
// The choices of all tokens for the caller and the launches that follow.
__device__ __forceinline__ void lk_moe_publish(const LkMoeArgs & a, const int * ids, const float * wts) {
    for (int i = threadIdx.x; i < a.T * a.k; i += blockDim.x) {
        a.ids[i] = ids[i];
        a.wts[i] = wts[i];
        if (a.ids_out) a.ids_out[i] = ids[i];
        if (a.wts_out) a.wts_out[i] = wts[i];
    }
}

// More than LK_MOE_FEW tokens: one workgroup of 16 waves chooses for all of them and
// sorts the assignments by expert (counting sort; a wave per expert keeps their order).
__global__ void __launch_bounds__(1024)
lk_k_moe_route(const LkMoeArgs a) {
    __shared__ int ids[LK_MOE_MAX_TOKENS * LK_MOE_MAX_TOP_K];
    __shared__ float wts[LK_MOE_MAX_TOKENS * LK_MOE_MAX_TOP_K];
    __shared__ int cnt[LK_MOE_MAX_EXPERTS], from[LK_MOE_MAX_EXPERTS];
    __shared__ uint64_t words[LK_MOE_MAX_EXPERTS / 64];
    __shared__ int sums[LK_MOE_MAX_EXPERTS / 64];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), na = a.T * a.k;
    LkMoeTab & tab = *(LkMoeTab *) a.tab;
    if (tid < LK_MOE_MAX_EXPERTS) cnt[tid] = 0;
    for (int t = wv; t < a.T; t += 16) lk_moe_choose(a, t, ids + t * a.k, wts + t * a.k);
    __syncthreads();
    lk_moe_publish(a, ids, wts);
    if (tid < na) atomicAdd(&cnt[ids[tid]], 1);          // na <= 512; counts have no order
    __syncthreads();
    int c = 0, before = 0, slot = 0;
    if (tid < LK_MOE_MAX_EXPERTS) {                      // waves 0 .. 3: exclusive sums over the experts
        c = cnt[tid];
        int s = c;
        for (int o = 1; o < 64; o <<= 1) {
            const int u = __shfl_up(s, o, 64);
            if (lane >= o) s += u;
        }
        before = s - c;
        const uint64_t b = __ballot(c > 0);
        slot = __popcll(b & ((1ull << lane) - 1));
        if (lane == 63) { words[wv] = b; sums[wv] = s; }
    }
    __syncthreads();
    if (tid < LK_MOE_MAX_EXPERTS) {
        for (int i = 0; i < wv; ++i) { before += sums[i]; slot += __popcll(words[i]); }
        from[tid] = before;
        if (c > 0) {
            tab.e[slot] = tid;
            tab.from[slot] = before;
        }
        if (tid == LK_MOE_MAX_EXPERTS - 1) {
            slot += c > 0;
            tab.slots = slot;
            tab.from[slot] = na;
        }
    }
    __syncthreads();
    for (int e = wv; e < a.E; e += 16) {
        if (cnt[e] == 0) continue;
        int n = from[e];
        for (int i0 = 0; i0 < na; i0 += 64) {
            const bool hit = i0 + lane < na && ids[i0 + lane] == e;
            const uint64_t b = __ballot(hit);
            if (hit) tab.list[n + __popcll(b & ((1ull << lane) - 1))] = i0 + lane;
            n += __popcll(b);
        }
    }
}

// ---- the products -------------------------------------------------------------------
// R weight rows of NM matrices (qs, d: the first of the rows) times TK rows of records
// (rec + trow[t] * bpr records), over the groups of 64 / R blocks of a row,
// U consecutive ones at a time, of which this is part g0 of gs.  Lane (c = l % R, g = l /
// R) takes block g of a group of weight row c, whole: 16 bytes, its scale, and of every
// record row the block's digits.  Those are the same for the R lanes of a block: the
// wave copies them, one run of memory, into its own part of LDS (xs) and every lane reads
// them there.
// acc[t][m]: this lane's blocks; the sum over the lanes of a row is the caller's.
// Every address is a wave-uniform base and a 32-bit offset: an expert's planes are below
// 4 GiB (LK_MOE_MAX_DIM).
template <typename V>
__device__ __forceinline__ V lk_moe_ld(const void * base, uint32_t off) { return *(const V *) ((const char *) base + off); }
template <int NP, int R, int U>
struct LkMoeX {                                          // one row's digits of a step: Z pieces of 16 bytes
    static constexpr int NB = 64 / R, Z = U * NB * LkMoeRec<NP>::PIECES, NZ = (Z + 63) / 64;
    lk_u4 x[64 * NZ];
};
template <int NP, int NM, int R, int U, int TK>
__device__ __forceinline__ void lk_moe_rows(const uint8_t * const (&qs)[NM], const _Float16 * const (&d)[NM],
                                            const uint8_t * rec, int bpr, const int (&trow)[TK], int g0, int gs,
                                            LkMoeX<NP, R, U> * xs, float (&acc)[TK][NM]) {
    typedef LkMoeX<NP, R, U> X;
    constexpr int NB = X::NB, PC = LkMoeRec<NP>::PIECES, NZ = X::NZ;
    const int lane = threadIdx.x & 63, c = lane % R, g = lane / R;
    const int ng = (bpr + NB - 1) / NB;
#pragma unroll 1
    for (int gi = g0 * U; gi < ng; gi += gs * U) {
        lk_u4 xv[TK][NZ], w[U][NM];
        _Float16 dw[U][NM];
        const int end = bpr * PC - gi * NB * PC;         // pieces from here to the row's end
#pragma unroll
        for (int t = 0; t < TK; ++t)
#pragma unroll
            for (int z = 0; z < NZ; ++z)
                xv[t][z] = lk_moe_ld<lk_u4>(rec + ((size_t) trow[t] * bpr + gi * NB) * (PC * 16),
                                            64 * z + lane < end ? 16u * (64 * z + lane) : 0u);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int b = (gi + u) * NB + g;
            const uint32_t wb = (uint32_t) (c * bpr + (b < bpr ? b : bpr - 1));                  // in bounds
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                w[u][m] = lk_moe_ld<lk_u4>(qs[m], wb * 16u);
                dw[u][m] = lk_moe_ld<_Float16>(d[m], wb * 2u);
            }
        }
#pragma unroll
        for (int t = 0; t < TK; ++t)
#pragma unroll
            for (int z = 0; z < NZ; ++z) xs[t].x[64 * z + lane] = xv[t][z];        // past the row's end: its first piece here
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (gi + u >= ng) break;                     // wave-uniform
            const bool in = (gi + u) * NB + g < bpr;
            uint32_t lo[NM][4], hi[NM][4];
            float dv[NM];
#pragma unroll
            for (int m = 0; m < NM; ++m) {
                dv[m] = (float) dw[u][m];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    lo[m][k] = w[u][m][k] & 0x0F0F0F0Fu;
                    hi[m][k] = (w[u][m][k] >> 4) & 0x0F0F0F0Fu;
                }
            }
#pragma unroll
            for (int t = 0; t < TK; ++t) {
                asm volatile("" ::: "memory");           // one token's digits at a time: all at once spill
                const lk_u4 * x = xs[t].x + (u * NB + g) * PC;
                lk_u4 q[2 * NP];
#pragma unroll
                for (int p = 0; p < 2 * NP; ++p) q[p] = x[p];
                const lk_i4 meta = __builtin_bit_cast(lk_i4, x[2 * NP]);
                const int m3 = meta[3];                  // a copy: bit_cast of a vector's element takes element 0
                const float sc = in ? __builtin_bit_cast(float, m3) : 0.0f;        // a block past the row's end counts nothing
#pragma unroll
                for (int m = 0; m < NM; ++m) {
                    float f = 0.0f;
#pragma unroll
                    for (int p = 0; p < NP; ++p) {
                        int s = meta[p];
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            s = __builtin_amdgcn_sdot4((int) lo[m][k], (int) q[2 * p][k], s, false);
                            s = __builtin_amdgcn_sdot4((int) hi[m][k], (int) q[2 * p + 1][k], s, false);
                        }
                        f = p ? __builtin_fmaf(f, 256.0f, (float) s) : (float) s;
                    }
                    acc[t][m] = __builtin_fmaf(dv[m] * sc, f, acc[t][m]);
                }
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}
// The sum over the lanes that hold blocks of one row (64 / R of them), in every lane.
template <int R>
__device__ __forceinline__ float lk_moe_lanes(float v) {
    if constexpr (R == 8) v += lk_dpp<LK_DPP_ROR8>(v);
    return lk_xrow_sum(v);
}

// 32 rows of one expert's gate and up products for N assignments (as[0 .. N-1]), and
// what follows of them: the records of h.  N is known at compile time: with branches on
// it the compiler keeps the digits of all tokens at once and spills.
template <int NP>
struct LkMoeUp {
    static constexpr int U = 2, TK = 4;
    LkMoeX<NP, 16, U> xs[LK_MOE_NW][TK];
    float part[LK_MOE_NW][4][TK][16];
};
template <int NP, int N>
__device__ __forceinline__ void lk_moe_up_tile(const LkMoeArgs & a, int e, const int * as, LkMoeUp<NP> & sh) {
    constexpr int U = LkMoeUp<NP>::U, REC = LkMoeRec<NP>::BYTES;
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int bpr = a.hidden / 32, F = a.ffn, r0 = blockIdx.x * 32;
    const size_t row = (size_t) e * F + r0;              // F is a multiple of 32: whole tiles
    const uint8_t * qs[4];
    const _Float16 * d[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
        qs[m] = a.qs[m >> 1] + (row + 16 * (m & 1)) * bpr * 16;
        d[m] = a.d[m >> 1] + (row + 16 * (m & 1)) * bpr;
    }
    int trow[N];
#pragma unroll
    for (int r = 0; r < N; ++r) trow[r] = __builtin_amdgcn_readfirstlane(as[r] / a.k);
    float acc[N][4] = {};
    lk_moe_rows<NP, 4, 16, U, N>(qs, d, a.xr, bpr, trow, wv, LK_MOE_NW, sh.xs[wv], acc);
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const float v = lk_moe_lanes<16>(acc[t][m]);
            if (g == m) sh.part[wv][m][t][c] = v;
        }
    __syncthreads();
    if (tid < 32 * N) {                                  // token t, row r of the 32
        const int t = tid >> 5, r = tid & 31;
        float gt = 0.0f, up = 0.0f;
#pragma unroll
        for (int k = 0; k < LK_MOE_NW; ++k) {
            gt += sh.part[k][r >> 4][t][r & 15];
            up += sh.part[k][2 + (r >> 4)][t][r & 15];
        }
        const float h = gt / (1.0f + expf(-gt)) * up;
        uint32_t am = __builtin_bit_cast(uint32_t, h) & 0x7FFFFFFFu;
        for (int o = 16; o > 0; o >>= 1) am = lk_umax(am, (uint32_t) __shfl_xor((int) am, o, 32));
        const float p2 = lk_moe_up2<NP>(am);
        int q[NP], s[3] = { 0, 0, 0 };
        lk_moe_digits<NP>(h, p2, q);
#pragma unroll
        for (int p = 0; p < NP; ++p) {
            s[p] = q[p];
            for (int o = 16; o > 0; o >>= 1) s[p] += __shfl_xor(s[p], o, 32);
        }
        uint8_t * rc = a.hr + ((size_t) as[t] * (F / 32) + blockIdx.x) * REC;
#pragma unroll
        for (int p = 0; p < NP; ++p) rc[32 * p + r] = (uint8_t) q[p];
        if (r == 0)
            *(lk_i4 *) (rc + 32 * NP) = lk_i4{ -8 * s[0], -8 * s[1], -8 * s[2], __builtin_bit_cast(int, lk_moe_scale(am, p2)) };
    }
}

// n assignments, four at a time.
template <int NP>
__device__ __forceinline__ void lk_moe_up_tiles(const LkMoeArgs & a, int e, const int * as, int n, LkMoeUp<NP> & sh) {
    for (; n > 0; n -= 4, as += 4) {
        if (n >= 4)      lk_moe_up_tile<NP, 4>(a, e, as, sh);
        else if (n == 3) lk_moe_up_tile<NP, 3>(a, e, as, sh);
        else if (n == 2) lk_moe_up_tile<NP, 2>(a, e, as, sh);
        else             lk_moe_up_tile<NP, 1>(a, e, as, sh);
        if (n > 4) __syncthreads();                      // part has been read
    }
}

// Up to LK_MOE_FEW tokens; grid (ffn / 32, T * k): the workgroups of an assignment
// whose expert an earlier one has end at once.
template <int NP>
__global__ void __launch_bounds__(64 * LK_MOE_NW, 4)
lk_k_moe_up_few(const LkMoeArgs a) {
    __shared__ int ids[LK_MOE_FEW * LK_MOE_MAX_TOP_K], as[LK_MOE_FEW];
    __shared__ float wts[LK_MOE_FEW * LK_MOE_MAX_TOP_K];
    __shared__ LkMoeUp<NP> sh;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), na = a.T * a.k;
    if (wv < a.T) lk_moe_choose(a, wv, ids + wv * a.k, wts + wv * a.k);
    __syncthreads();
    if (blockIdx.x == 0 && blockIdx.y == 0) lk_moe_publish(a, ids, wts);
    const int mine = lane < na ? ids[lane] : -1;
    const int e = __builtin_amdgcn_readlane(mine, blockIdx.y);
    const uint64_t hits = __ballot(mine == e);
    if (__builtin_ctzll(hits) != (int) blockIdx.y) return;
    if (wv == 0 && mine == e) as[__popcll(hits & ((1ull << lane) - 1))] = lane;
    __syncthreads();
    lk_moe_up_tiles<NP>(a, e, as, __popcll(hits), sh);
}

template <int NP>
__global__ void __launch_bounds__(64 * LK_MOE_NW, 4)
lk_k_moe_up(const LkMoeArgs a) {
    __shared__ int as[LK_MOE_MAX_TOKENS];
    __shared__ LkMoeUp<NP> sh;
    const LkMoeTab & tab = *(const LkMoeTab *) a.tab;
    if ((int) blockIdx.y >= tab.slots) return;
    const int e = tab.e[blockIdx.y], from = tab.from[blockIdx.y], n = tab.from[blockIdx.y + 1] - from;
    if ((int) threadIdx.x < n) as[threadIdx.x] = tab.list[from + threadIdx.x];
    __syncthreads();
    lk_moe_up_tiles<NP>(a, e, as, n, sh);
}

// Up to LK_MOE_FEW tokens: a workgroup of 16 waves has 8 rows of every expert that was
// chosen (at most 64), and adds them up itself.  The waves share the experts, Q = 16 /
// experts of them (at least one) to each, taking its block groups in turn.
template <int TYPE, int NP>
__global__ void __launch_bounds__(64 * LK_MOE_NWF, 4)
lk_k_moe_down_few(const LkMoeArgs a) {
    typedef typename LkElem<TYPE>::type T;
    constexpr int R = 8, U = 2, TK = 2, MAXA = LK_MOE_FEW * LK_MOE_MAX_TOP_K;
    __shared__ LkMoeX<NP, R, U> xs[LK_MOE_NWF][TK];
    // [q][assignment][row]: q * assignments is at most 16 / experts * (experts * LK_MOE_FEW), or MAXA
    __shared__ float part[LK_MOE_NWF * LK_MOE_FEW][R];
    static_assert(LK_MOE_NWF * LK_MOE_FEW >= MAXA, "part");
    const int tid = threadIdx.x, lane = tid & 63, c = lane % R, g = lane / R;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6), na = a.T * a.k, r0 = blockIdx.x * R, bpr = a.ffn / 32;
    const int mine = lane < na ? a.ids[lane] : -1;
    // what the sum at the end needs, asked for now (T * R <= 64: the first wave)
    const int ot = tid / R, orow = r0 + tid % R;
    const bool sums = tid < a.T * R;
    float wt[LK_MOE_MAX_TOP_K], rs = 0.0f;
#pragma unroll
    for (int j = 0; j < LK_MOE_MAX_TOP_K; ++j) wt[j] = sums && j < a.k ? a.wts[ot * a.k + j] : 0.0f;
    if (sums && a.res) rs = (float) ((const T *) a.res)[(size_t) ot * a.ldr + orow];
    uint64_t first = 0;                                  // the assignments that are their expert's first
    for (int i = 0; i < na; ++i) {
        const uint64_t b = __ballot(mine == __builtin_amdgcn_readlane(mine, i));
        first |= (uint64_t) (__builtin_ctzll(b) == i) << i;
    }
    const int nd = __popcll(first), Q = nd >= LK_MOE_NWF ? 1 : LK_MOE_NWF / nd;
    for (int item = wv; item < nd * Q; item += LK_MOE_NWF) {       // expert item / Q, part item % Q
        uint64_t left = first;
        for (int i = item / Q; i > 0; --i) left &= left - 1;
        const int e = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left)), q = item % Q;
        const size_t row = (size_t) e * a.hidden + r0;   // hidden is a multiple of 32: whole tiles
        const uint8_t * const qs[1] = { a.qs[2] + row * bpr * 16 };
        const _Float16 * const d[1] = { a.d[2] + row * bpr };
        uint64_t hits = __ballot(mine == e);
        while (hits) {                                   // two assignments at a time
            const int t0 = __builtin_ctzll(hits);
            hits &= hits - 1;
            if (hits) {
                const int trow[2] = { t0, __builtin_ctzll(hits) };
                hits &= hits - 1;
                float acc[2][1] = {};
                lk_moe_rows<NP, 1, R, U, 2>(qs, d, a.hr, bpr, trow, q, Q, xs[wv], acc);
                const float v0 = lk_moe_lanes<R>(acc[0][0]), v1 = lk_moe_lanes<R>(acc[1][0]);
                if (g < 2) part[q * na + trow[g]][c] = g ? v1 : v0;
            } else {
                const int trow[1] = { t0 };
                float acc[1][1] = {};
                lk_moe_rows<NP, 1, R, U, 1>(qs, d, a.hr, bpr, trow, q, Q, xs[wv], acc);
                const float v0 = lk_moe_lanes<R>(acc[0][0]);
                if (g == 0) part[q * na + t0][c] = v0;
            }
        }
    }
    __syncthreads();
    if (sums) {
        float o = 0.0f;
#pragma unroll
        for (int j = 0; j < LK_MOE_MAX_TOP_K; ++j) {
            if (j >= a.k) break;
            float y = 0.0f;
            for (int q = 0; q < Q; ++q) y += part[q * na + ot * a.k + j][tid % R];
            o = __builtin_fmaf(wt[j], y, o);
        }
        if (a.res) o = rs + o;
        ((T *) a.out)[(size_t) ot * a.ldo + orow] = (T) o;
    }
}

// 32 rows of one expert's down product for N assignments.
template <int NP>
struct LkMoeDown {
    static constexpr int U = 2, TK = 4;
    LkMoeX<NP, 16, U> xs[LK_MOE_NW][TK];
    float part[LK_MOE_NW][2][TK][16];
};
template <int NP, int N>
__device__ __forceinline__ void lk_moe_down_tile(const LkMoeArgs & a, int e, const int * as, LkMoeDown<NP> & sh) {
    constexpr int U = LkMoeDown<NP>::U;
    const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6), r0 = blockIdx.x * 32, bpr = a.ffn / 32;
    const size_t row = (size_t) e * a.hidden + r0;
    const uint8_t * const qs[2] = { a.qs[2] + row * bpr * 16, a.qs[2] + (row + 16) * bpr * 16 };
    const _Float16 * const d[2] = { a.d[2] + row * bpr, a.d[2] + (row + 16) * bpr };
    int trow[N];
#pragma unroll
    for (int r = 0; r < N; ++r) trow[r] = __builtin_amdgcn_readfirstlane(as[r]);
    float acc[N][2] = {};
    lk_moe_rows<NP, 2, 16, U, N>(qs, d, a.hr, bpr, trow, wv, LK_MOE_NW, sh.xs[wv], acc);
#pragma unroll
    for (int t = 0; t < N; ++t)
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const float v = lk_moe_lanes<16>(acc[t][m]);
            if (g == m) sh.part[wv][m][t][c] = v;
        }
    __syncthreads();
    if (tid < 32 * N) {
        const int t = tid >> 5, r = tid & 31;
        float y = 0.0f;
#pragma unroll
        for (int k = 0; k < LK_MOE_NW; ++k) y += sh.part[k][r >> 4][t][r & 15];
        a.y[(size_t) as[t] * a.hidden + r0 + r] = y;
    }
}

template <int NP>
__global__ void __launch_bounds__(64 * LK_MOE_NW, 4)
lk_k_moe_down(const LkMoeArgs a) {
    __shared__ int as[LK_MOE_MAX_TOKENS];
    __shared__ LkMoeDown<NP> sh;
    const LkMoeTab & tab = *(const LkMoeTab *) a.tab;
    if ((int) blockIdx.y >= tab.slots) return;
    const int e = tab.e[blockIdx.y], from = tab.from[blockIdx.y], n = tab.from[blockIdx.y + 1] - from;
    if ((int) threadIdx.x < n) as[threadIdx.x] = tab.list[from + threadIdx.x];
    __syncthreads();
    const int * p = as;
    for (int left = n; left > 0; left -= 4, p += 4) {
        if (left >= 4)      lk_moe_down_tile<NP, 4>(a, e, p, sh);
        else if (left == 3) lk_moe_down_tile<NP, 3>(a, e, p, sh);
        else if (left == 2) lk_moe_down_tile<NP, 2>(a, e, p, sh);
        else                lk_moe_down_tile<NP, 1>(a, e, p, sh);
        if (left > 4) __syncthreads();                   // part has been read
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
    const size_t k = m->top_k, H = m->hidden, F = m->ffn, REC = LkMoeRec<3>::BYTES;        // of two digits: less
    auto take = [&](size_t bytes) {
        char * p = work ? (char *) work + at : nullptr;
        at += (bytes + 15) & ~(size_t) 15;
        return (void *) p;
    };
    LkMoeArgs b = {};
    LkMoeArgs * o = a ? a : &b;
    o->logits = (float *) take(4 * (size_t) T * m->n_experts);
    o->xr = (uint8_t *) take(T * (H / 32) * REC);
    o->hr = (uint8_t *) take(T * k * (F / 32) * REC);
    o->y = (float *) take(4 * T * k * H);
    o->ids = (int32_t *) take(4 * T * k);
    o->wts = (float *) take(4 * T * k);
    o->tab = (int32_t *) take(sizeof(LkMoeTab));
    return at;
}
extern "C" size_t lk_moe_work_bytes(const lk_moe * moe, int T) {
    if (lk_moe_check(moe) || T < 0 || T > LK_MOE_MAX_TOKENS) return 0;
    return lk_moe_layout(moe, T, nullptr, nullptr);
}

template <int TYPE>
static void lk_moe_go(const LkMoeArgs & a, hipStream_t st) {
    constexpr int NP = TYPE == LK_F32 ? 3 : 2;
    const int nE = (a.E + 3) / 4, na = a.T * a.k, slots = na < a.E ? na : a.E;
    hipLaunchKernelGGL((lk_k_moe_router<TYPE, NP>), dim3(nE + (a.hidden / 8 + LK_MOE_THREADS - 1) / LK_MOE_THREADS, (a.T + 3) / 4),
                       dim3(LK_MOE_THREADS), 0, st, a, nE);
    if (a.T <= LK_MOE_FEW) {
        hipLaunchKernelGGL((lk_k_moe_up_few<NP>), dim3(a.ffn / 32, na), dim3(64 * LK_MOE_NW), 0, st, a);
        hipLaunchKernelGGL((lk_k_moe_down_few<TYPE, NP>), dim3(a.hidden / 8), dim3(64 * LK_MOE_NWF), 0, st, a);
        return;
    }
    hipLaunchKernelGGL(lk_k_moe_route, dim3(1), dim3(1024), 0, st, a);
    hipLaunchKernelGGL((lk_k_moe_up<NP>), dim3(a.ffn / 32, slots), dim3(64 * LK_MOE_NW), 0, st, a);
    hipLaunchKernelGGL((lk_k_moe_down<NP>), dim3(a.hidden / 32, slots), dim3(64 * LK_MOE_NW), 0, st, a);
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

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
// int8 digits of base 256: four for fp32 rows (32 bits of the block's largest value), three
// for fp16 and bf16 rows (24 bits).  sum (n - 8) i is exact in int32 digit by digit
// (-8 * the digits' sum is where the sum starts), the digits are put together and scaled by
// d * 2^-p in fp32, and blocks are added in fp32.  A block that holds a value
// that is not finite gets the scale NaN; one whose largest value is under 2^-100 counts as
// zero.
// Why that many: a channel, of x or of h, that is 1000 times the others leaves its 31 neighbours
// 10 bits fewer.  With a digit less a row whose large channels meet weights of zero
// was off by 2e-2 to 4e-2 (16-bit rows) and 1.7e-4 (fp32), so 2e-4 and 6e-7.
#include "lk_types.h"

typedef uint32_t lk_u4 __attribute__((ext_vector_type(4)));

// For a few tokens (at most this many) every workgroup chooses the experts itself, a wave
// per token, and the down product adds the experts up itself (three launches); for more a
// launch of one workgroup chooses once and sorts the tokens by expert, and another
// adds up (five).  us with three / five launches, bf16 and fp32 rows; the rule (lk_moe_few)
// takes three for up to 5 tokens, and 8 of up to 28 choices in all (fp32 rows: 16):
//   tokens                           2        4        5        6        7        8
//   64 experts, 4 of 2048 x 1536   20/26    29/32    33/36    37/38    42/41    47/45
//                            fp32  21/27    29/33    35/37    39/39    44/42    50/47
//   128 experts, 8 of 2048 x 768   21/30    33/37    37/41    45/44    50/48    55/51
//                            fp32  22/31    34/38    39/42    46/46    52/50    58/53
//   16 experts, 4 of 1280 x 1184   17/22    21/26    24/27    25/27    27/28    29/29
//                            fp32  17/23    22/27    25/28    27/28    30/29    31/30
//   32 experts, 2 of 2048 x 1792   15/22    20/27    21/28    25/31    27/32    29/34
//                            fp32  16/23    21/28    22/29    27/32    30/33    32/35
#define LK_MOE_FEW 8
#define LK_MOE_THREADS 256
#define LK_MOE_NW 8                       // waves of a gate/up workgroup for few tokens
#define LK_MOE_NWF 16                     // of a down workgroup
template <int N> struct LkInt { static constexpr int value = N; };

// The experts by the number of their assignments (token * k + j), most first, equals by
// index: slot s has expert e with n assignments, list[s][0 .. n-1] in order.
struct LkMoeTab {
    struct { int32_t e, n, pad[2]; } slot[LK_MOE_MAX_EXPERTS];
    int32_t list[LK_MOE_MAX_EXPERTS][LK_MOE_MAX_TOKENS];
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
    int32_t * tab;                       // LkMoeTab, for more than a few tokens
    int ldx, ldr, ldo, T, E, k, hidden, ffn, score, renorm, kinv;
    float scale;
};

// ---- whole numbers of a block -------------------------------------------------------
// A block's record: NP planes of 32 int8 digits, highest first, then a piece of int32 -8 * the
// sums of the planes, two planes put together (the first * 256 + the second; the third of
// three alone), 0, and the fp32 scale 2^-p.  A plane holds elements 0 .. 7, 16 .. 23, then 8 .. 15, 24
// .. 31: dwords 2 h, 2 h + 1 of a weight block are the elements of piece h.
template <int NP>
struct LkMoeRec {
    static constexpr int PIECES = 2 * NP + 1, BYTES = 16 * PIECES;
};
// 2^p for a block whose largest |v| has the bits am; 0 for a block of zeros and for one
// that is not finite.  The digits reach 127 * (1 + 256 + 65536 (+ 2^24)): the largest value
// goes to the top binade where its leading bits allow, else one below.
template <int NP>
__device__ __forceinline__ float lk_moe_up2(uint32_t am) {
    constexpr float TOP = NP == 4 ? 2139062016.0f : 8355711.0f;                   // 24 bits of the four digits' end
    constexpr int B = NP == 4 ? 30 : 22;
    if (am >= 0x7F800000u || am < (27u << 23)) return 0.0f;                       // not finite; under 2^-100
    // 2^(B - E), E the exponent of am, up to 2^126, whose inverse is normal (four digits: blocks of 2^-96 to
    // 2^-100 have 30 to 26 bits)
    const int e = B + 254 - (int) (am >> 23);
    const float f = __builtin_bit_cast(float, (uint32_t) (e < 253 ? e : 253) << 23);
    return __builtin_bit_cast(float, am) * f > TOP ? 0.5f * f : f;
}
__device__ __forceinline__ float lk_moe_scale(uint32_t am, float up) {            // 2^-p; NaN for what is not finite
    return am >= 0x7F800000u ? __builtin_nanf("") : up == 0.0f ? 0.0f : __builtin_bit_cast(float, (254u << 23) - __builtin_bit_cast(uint32_t, up));
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

// The token of an assignment: as / k, as < 512, k <= 8, by a multiplication (kinv = 65536 / k + 1).
__device__ __forceinline__ int lk_moe_token(const LkMoeArgs & a, int as) { return (int) ((uint32_t) (as * a.kinv) >> 16); }

// ---- small helpers --------------------------------------------------------------------
// exp(-|x|) on v_exp_f32 with the product's rounding error put back (about one unit of
// 2^-23): expf's branches cost more than they are worth in kernels of a microsecond.
__device__ __forceinline__ float lk_moe_expn(float x) {
    const float y = fmaxf(-fabsf(x), -104.0f);           // 0 from there on; NaN too (the callers see to it)
    const float t = y * LK_LOG2E_F, r = __builtin_fmaf(y, LK_LOG2E_F, -t) + y * 1.925963033500e-8f;
    const float z = lk_exp2(t);
    return __builtin_fmaf(z, r * 0.6931471805599453f, z);
}
__device__ __forceinline__ float lk_moe_sigmoid(float x) {   // of a NaN: 0 or NaN
    const float z = lk_moe_expn(x), q = __builtin_amdgcn_rcpf(1.0f + z);
    return x >= 0.0f ? q : z * q;
}
__device__ __forceinline__ float lk_moe_h(float g, float u) { return g * lk_moe_sigmoid(g) * u; }   // NaN * 0 is NaN
// Largest of a wave's unsigned values, wave-uniform.
__device__ __forceinline__ uint32_t lk_moe_top(uint32_t v) {
    v = lk_umax(v, lk_dpp_u<LK_DPP_QP_XOR1>(v));
    v = lk_umax(v, lk_dpp_u<LK_DPP_QP_XOR2>(v));
    v = lk_umax(v, lk_dpp_u<LK_DPP_HMIRROR>(v));
    v = lk_umax(v, lk_dpp_u<LK_DPP_MIRROR>(v));
    const uint32_t a = (uint32_t) __builtin_amdgcn_readlane((int) v, 0), b = (uint32_t) __builtin_amdgcn_readlane((int) v, 16);
    const uint32_t c = (uint32_t) __builtin_amdgcn_readlane((int) v, 32), d = (uint32_t) __builtin_amdgcn_readlane((int) v, 48);
    return lk_umax(lk_umax(a, b), lk_umax(c, d));
}
// Sum over each half of a wave.
__device__ __forceinline__ int lk_moe_sum32(int v) {
    float x = __builtin_bit_cast(float, v), y = x;
    lk_swap16(x, y);
    v = __builtin_bit_cast(int, x) + __builtin_bit_cast(int, y);
    v += (int) lk_dpp_u<LK_DPP_ROR8>((uint32_t) v);
    v += (int) lk_dpp_u<LK_DPP_ROR4>((uint32_t) v);
    v += (int) lk_dpp_u<LK_DPP_QP_XOR2>((uint32_t) v);
    v += (int) lk_dpp_u<LK_DPP_QP_XOR1>((uint32_t) v);
    return v;
}
__device__ __forceinline__ constexpr int lk_moe_place(int i) { return 16 * (i / 8 % 2) + 8 * (i / 16) + i % 8; }    // of element i
// The record of a block whose 32 values h lie on the 32 lanes of a half-wave (r: the
// lane's place); nothing is stored where !ok.
template <int NP>
__device__ __forceinline__ void lk_moe_record(float h, int r, bool ok, uint8_t * rec) {
    const float m = lk_bfly32_max(h == h ? fabsf(h) : __builtin_inff());
    const uint32_t am = __builtin_bit_cast(uint32_t, m);
    const float up = lk_moe_up2<NP>(am);
    int q[NP];
    lk_moe_digits<NP>(h, up, q);
    const int s01 = lk_moe_sum32(q[0] * 256 + q[1]), s23 = lk_moe_sum32(NP == 4 ? q[2] * 256 + q[NP - 1] : q[2]);
    if (!ok) return;
#pragma unroll
    for (int p = 0; p < NP; ++p) rec[32 * p + lk_moe_place(r)] = (uint8_t) q[p];
    if (r == 0)
        *(lk_i4 *) (rec + 32 * NP) = lk_i4{ -8 * s01, -8 * s23, 0, __builtin_bit_cast(int, lk_moe_scale(am, up)) };
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
        // H is a multiple of 32: whole pieces of 8.  U pieces of the row and of NT tokens are asked
        // for before the first is used: a piece at a time each took a round trip
        auto go = [&](auto tokens, auto pieces) {
            constexpr int NT = decltype(tokens)::value, U = decltype(pieces)::value;
            float s[NT] = {};
            for (int i0 = lane * 8; i0 < H; i0 += 512 * U) {
                float w[U][8], v[U][NT][8];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int i = i0 + 512 * u < H ? i0 + 512 * u : i0;                          // past the end: not used
                    lk_load<8>(r + i, w[u]);
#pragma unroll
                    for (int k = 0; k < NT; ++k) lk_load<8>(x + (size_t) (t0 + k < a.T ? t0 + k : a.T - 1) * a.ldx + i, v[u][k]);
                }
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    if (i0 + 512 * u >= H) break;
#pragma unroll
                    for (int k = 0; k < NT; ++k)
#pragma unroll
                        for (int j = 0; j < 8; ++j) s[k] = __builtin_fmaf(w[u][j], v[u][k][j], s[k]);
                }
            }
#pragma unroll
            for (int k = 0; k < NT; ++k) {
                s[k] = lk_wave_sum(s[k]);
                if (lane == 0 && t0 + k < a.T) a.logits[(size_t) (t0 + k) * a.E + e] = s[k];
            }
        };
        if (a.T == 1) go(LkInt<1>{}, LkInt<4>{});
        else          go(LkInt<4>{}, LkInt<2>{});
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
        int s[2] = { 0, 0 };
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            int q[NP];
            lk_moe_digits<NP>(v[j], up, q);
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                w[p][j / 4] |= (uint32_t) (uint8_t) q[p] << (8 * (j % 4));
                s[p / 2] += p == 0 || (NP == 4 && p == 2) ? q[p] * 256 : q[p];
            }
        }
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            s[p] += (int) lk_dpp_u<LK_DPP_QP_XOR1>((uint32_t) s[p]);
            s[p] += (int) lk_dpp_u<LK_DPP_QP_XOR2>((uint32_t) s[p]);
        }
        if (!ok) continue;
        uint8_t * r = a.xr + ((size_t) t * bpr + b) * REC;
#pragma unroll
        for (int p = 0; p < NP; ++p) *(uint2 *) (r + 32 * p + lk_moe_place(8 * g)) = make_uint2(w[p][0], w[p][1]);
        if (g == 0)
            *(lk_i4 *) (r + 32 * NP) = lk_i4{ -8 * s[0], -8 * s[1], 0, __builtin_bit_cast(int, lk_moe_scale(am, up)) };
    }
}

// ---- choice of experts --------------------------------------------------------------
// A wave per token: lane i holds experts i, i + 64, ... (NL registers, for up to 64 *
// NL experts).  A round takes the largest key that is left; the first register and then the
// first lane that holds it are the lowest index.
__device__ __forceinline__ uint32_t lk_moe_key(float r) {    // orderable bits; 0: taken, 1: NaN; -0 as 0
    const uint32_t u = __builtin_bit_cast(uint32_t, r + 0.0f);
    return r != r ? 1u : (u >> 31) ? ~u : u | 0x80000000u;
}
// A token's logits and the biases, as a lane holds them (past the experts: expert 0's).
template <int NL>
__device__ __forceinline__ void lk_moe_logits(const LkMoeArgs & a, int t, float (&l)[NL]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < NL; ++i) l[i] = a.logits[(size_t) t * a.E + (64 * i + lane < a.E ? 64 * i + lane : 0)];
}
template <int NL>
__device__ __forceinline__ void lk_moe_bias(const LkMoeArgs & a, float (&b)[NL]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < NL; ++i) b[i] = a.bias ? a.bias[64 * i + lane < a.E ? 64 * i + lane : 0] : 0.0f;
}
// Of TW tokens, one after the other in every step, the choice j and its weight in lane j < k; the
// other lanes hold -1.
template <int NL, int TW>
__device__ __forceinline__ void lk_moe_choose(const LkMoeArgs & a, const float (&l)[TW][NL], const float (&b)[NL], int (&id)[TW], float (&w)[TW]) {
    const int lane = threadIdx.x & 63;
    uint32_t key[TW][NL];
    float m[TW], zi[TW], mine[TW];                       // mine: lane j: the logit of choice j
    auto score = [&](int t, float v) {                   // v - v: 0, or NaN for what is not finite
        return a.score == LK_MOE_SOFTMAX ? (lk_moe_expn(v - m[t]) + (v - v)) * zi[t] : v == v ? lk_moe_sigmoid(v) : v;
    };
#pragma unroll
    for (int t = 0; t < TW; ++t) {
        m[t] = 0.0f, zi[t] = 1.0f, mine[t] = 0.0f, id[t] = -1;
        if (a.score == LK_MOE_SOFTMAX) {
            m[t] = l[t][0];
#pragma unroll
            for (int i = 1; i < NL; ++i) m[t] = fmaxf(m[t], l[t][i]);
            m[t] = lk_xrow_max(lk_row_max16(m[t]));      // lanes past the experts repeat expert 0
            float z = 0.0f;
#pragma unroll
            for (int i = 0; i < NL; ++i) z += 64 * i + lane < a.E ? lk_moe_expn(l[t][i] - m[t]) + (l[t][i] - l[t][i]) : 0.0f;
            zi[t] = 1.0f / lk_wave_sum(z);
        }
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const float r = a.bias ? score(t, l[t][i]) + b[i] : l[t][i];
            key[t][i] = 64 * i + lane < a.E ? lk_moe_key(r) : 0;
        }
    }
    for (int j = 0; j < a.k; ++j)
#pragma unroll
        for (int t = 0; t < TW; ++t) {
            uint32_t best = key[t][0];
#pragma unroll
            for (int i = 1; i < NL; ++i) best = lk_umax(best, key[t][i]);
            best = lk_moe_top(best);
            int e = 0;
            float v = 0.0f;
#pragma unroll
            for (int i = NL - 1; i >= 0; --i) {
                const uint64_t at = __ballot(key[t][i] == best);
                if (NL == 1 || at) {                     // in one register at least: k <= E
                    e = 64 * i + __builtin_ctzll(at);
                    v = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, l[t][i]), e & 63));
                }
            }
#pragma unroll
            for (int i = 0; i < NL; ++i) key[t][i] = 64 * i + lane == e ? 0 : key[t][i];
            mine[t] = lane == j ? v : mine[t];
            id[t] = lane == j ? e : id[t];
        }
#pragma unroll
    for (int t = 0; t < TW; ++t) {
        w[t] = lane < a.k ? score(t, mine[t]) : 0.0f;
        if (a.renorm) w[t] = w[t] / (lk_row_sum16(w[t]) + 1e-20f);         // k <= 8: the first row of 16 lanes
        w[t] *= a.scale;
    }
}
// More than a few tokens: one workgroup of 16 waves chooses for all of them and
// sorts the assignments by expert: TW tokens a wave, whose steps fill each other's waits, and
// several lanes to an expert's rank among the counts (64 tokens 9.0 us, 19 tokens 5.6; a token, an
// expert and a count at a time 11.1 and 6.1; 64 tokens: 1 us of it the logits' way, 4 the choice, the
// instructions of 16 tokens on each SIMD).
template <int NL, int TW>
__global__ void __launch_bounds__(1024)
lk_k_moe_route(const LkMoeArgs a) {
    __shared__ int ids[LK_MOE_MAX_TOKENS * LK_MOE_MAX_TOP_K], cnt[LK_MOE_MAX_EXPERTS], slot[LK_MOE_MAX_EXPERTS];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), na = a.T * a.k;
    LkMoeTab & tab = *(LkMoeTab *) a.tab;
    if (tid < LK_MOE_MAX_EXPERTS) cnt[tid] = 0;
    __syncthreads();
    float l[TW][NL], b[NL];
#pragma unroll
    for (int i = 0; i < TW; ++i) lk_moe_logits<NL>(a, wv + 16 * i < a.T ? wv + 16 * i : a.T - 1, l[i]);
    lk_moe_bias<NL>(a, b);
    int id[TW];
    float w[TW];
    lk_moe_choose<NL, TW>(a, l, b, id, w);               // past the last token: the last again, not used
#pragma unroll
    for (int i = 0; i < TW; ++i) {
        const int t = wv + 16 * i;
        if (t < a.T && id[i] >= 0) {
            const int at = t * a.k + lane;
            ids[at] = id[i];
            a.wts[at] = w[i];
            if (a.ids_out) a.ids_out[at] = id[i];
            if (a.wts_out) a.wts_out[at] = w[i];
            atomicAdd(&cnt[id[i]], 1);                   // counts have no order
        }
    }
    __syncthreads();
    constexpr int NS = NL == 1 ? 16 : 4;                 // lanes that share an expert's comparisons
    {
        const int e = tid / NS, c = e < a.E ? cnt[e] : 0;
        int s = 0;
#pragma unroll 4
        for (int o = tid % NS; o < a.E; o += NS) s += cnt[o] > c || (cnt[o] == c && o < e);
#pragma unroll
        for (int x = 1; x < NS; x *= 2) s += __shfl_xor(s, x);
        if (e < a.E && tid % NS == 0) {
            slot[e] = s;
            tab.slot[s].e = e;
            tab.slot[s].n = c;
        }
    }
    __syncthreads();
    constexpr int NC = LK_MOE_MAX_TOKENS * LK_MOE_MAX_TOP_K / 64;
    int mine[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) mine[i] = 64 * i + lane < na ? ids[64 * i + lane] : -1;
    for (int e = wv; e < a.E; e += 16) {                 // a wave per expert keeps the order
        if (cnt[e] == 0) continue;
        int32_t * list = tab.list[slot[e]];
        int n = 0;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            if (64 * i >= na) break;
            const uint64_t b = __ballot(mine[i] == e);
            if (mine[i] == e) list[n + __popcll(b & ((1ull << lane) - 1))] = 64 * i + lane;
            n += __popcll(b);
        }
    }
}

// ---- the products -------------------------------------------------------------------
// 8 weight rows of NM matrices (qs, d: the first of the rows) times TK rows of records
// (rec + trow[t] * bpr records), over the steps of 8 blocks of a row, U consecutive ones at
// a time, of which this is part g0 of gs.  Lane (c = l / 8, g = l % 8) takes block g of a
// step of weight row c, whole: 16 bytes, its scale, and of every record row the block's
// digits.  So eight lanes in a row load a whole 128-byte line of a weight row, and 16 bytes
// of its scales: with c = l % 8, another row in every lane, the scales' loads took as long
// again as the weights' (64 tokens, gate and up, 226 MB: 70 us, so 63).  The digits are the
// same for the 8 lanes of a block: the wave copies them, one run of memory, into its own
// part of LDS (xs) and every lane reads them there.
// acc[t][m]: this lane's blocks; the sum over the lanes of a row is the caller's.
// Every address is a wave-uniform base and a 32-bit offset: an expert's planes are below
// 4 GiB (LK_MOE_MAX_DIM).
template <typename V>
__device__ __forceinline__ V lk_moe_ld(const void * base, uint32_t off) { return *(const V *) ((const char *) base + off); }
// The digits' sums of a block put together: two at a time exactly (below 2^24, or 16 times
// that where all are multiples of 16), and one rounding.
template <int NP, typename V>
__device__ __forceinline__ float lk_moe_digits_sum(const V & s) {
    const float f = (float) (s[0] * 256 + s[1]);
    return NP == 4 ? __builtin_fmaf(f, 65536.0f, (float) (s[2] * 256 + s[3])) : __builtin_fmaf(f, 256.0f, (float) s[2]);
}
// A block's record x times the lane's block of NM weight rows (its 32 nibbles: lo, hi).
template <int NP, int NM>
__device__ __forceinline__ void lk_moe_token_dots(const lk_u4 * x, bool in, const uint32_t (&lo)[NM][4], const uint32_t (&hi)[NM][4],
                                                  const float (&dv)[NM], float (&acc)[NM]) {
    const lk_i4 meta = __builtin_bit_cast(lk_i4, x[2 * NP]);
    const int m3 = meta[3];                              // a copy: bit_cast of a vector's element takes element 0
    const float sc = in ? __builtin_bit_cast(float, m3) : 0.0f;                    // a block past the row's end counts nothing
    // of four planes two at a time: all their digits take 32 registers (1 token fp32 15.9 us, so 15.3; three
    // planes in two steps 15.2, at once 14.8)
    constexpr int P = NP == 4 ? 2 : NP;
    int s[NP][NM];
#pragma unroll
    for (int a = 0; a < NP; a += P) {
        lk_u4 q[2 * P];
#pragma unroll
        for (int i = 0; i < 2 * P; ++i) q[i] = x[2 * a + i];
#pragma unroll
        for (int m = 0; m < NM; ++m)
#pragma unroll
            for (int p = 0; p < P; ++p) {
                int v = a + p == 1 ? meta[0] : a + p == NP - 1 ? meta[1] : 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    v = __builtin_amdgcn_sdot4((int) lo[m][k], (int) q[2 * p + k / 2][k % 2], v, false);
                    v = __builtin_amdgcn_sdot4((int) hi[m][k], (int) q[2 * p + k / 2][2 + k % 2], v, false);
                }
                s[a + p][m] = v;                         // at most 32 * 8 * 128 = 2^15 without meta
            }
        // done here: left to itself the compiler reads the digits of all tokens first and spills
#pragma unroll
        for (int m = 0; m < NM; ++m)
#pragma unroll
            for (int p = 0; p < P; ++p) asm volatile("" : "+v"(s[a + p][m]) :: "memory");
    }
#pragma unroll
    for (int m = 0; m < NM; ++m) {
        const int s4[4] = { s[0][m], s[1][m], s[2][m], s[NP - 1][m] };
        acc[m] = __builtin_fmaf(dv[m] * sc, lk_moe_digits_sum<NP>(s4), acc[m]);
        asm volatile("" : "+v"(acc[m]) :: "memory");
    }
}
template <int NP, int U>
struct LkMoeX {                                          // one row's digits of U steps: Z pieces of 16 bytes
    static constexpr int Z = U * 8 * LkMoeRec<NP>::PIECES, NZ = (Z + 63) / 64;
    lk_u4 x[64 * NZ];
};
template <int NP, int NM, int U, int TK>
__device__ __forceinline__ void lk_moe_rows(const uint8_t * const (&qs)[NM], const _Float16 * const (&d)[NM],
                                            const uint8_t * rec, int bpr, const int (&trow)[TK], int g0, int gs,
                                            LkMoeX<NP, U> * xs, float (&acc)[TK][NM]) {
    constexpr int PC = LkMoeRec<NP>::PIECES, NZ = LkMoeX<NP, U>::NZ, NB = 8;
    const int lane = threadIdx.x & 63, c = lane >> 3, g = lane & 7;
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
                lk_moe_token_dots<NP, NM>(xs[t].x + (u * NB + g) * PC, in, lo, hi, dv, acc[t]);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}
// The sum over the eight lanes that hold blocks of one row, in every lane.
__device__ __forceinline__ float lk_moe_lanes(float v) {
    v += lk_dpp<LK_DPP_QP_XOR1>(v);
    v += lk_dpp<LK_DPP_QP_XOR2>(v);
    return v + lk_dpp<LK_DPP_HMIRROR>(v);
}

// Where a wave of a gate/up workgroup finds its 16 + 16 of the tile's 32 rows (half:
// 0 or 1): matrices 0, 1 the gate's rows 16 half .. +15, eight each, 2, 3 the up's.
__device__ __forceinline__ void lk_moe_up_rows(const LkMoeArgs & a, int e, int half, const uint8_t * (&qs)[4], const _Float16 * (&d)[4]) {
    const int bpr = a.hidden / 32;
    const size_t row = (size_t) e * a.ffn + blockIdx.x * 32 + 16 * half;        // ffn is a multiple of 32: whole tiles
#pragma unroll
    for (int m = 0; m < 4; ++m) {
        qs[m] = a.qs[m >> 1] + (row + 8 * (m & 1)) * bpr * 16;
        d[m] = a.d[m >> 1] + (row + 8 * (m & 1)) * bpr;
    }
}

// More tokens: a workgroup of 4 waves has 32 rows (up: of gate and up) or 64 (down) of
// one expert and up to TG of its assignments at a time.  Wave w has half w & 1 of the rows
// (four matrices of 8 rows) and every second step of 8 blocks of K; it copies a step's
// digits into its own part of LDS while the step's weights are on their way, which are
// asked for before the products of the step before.
// One assignment: the dots above.  More: v_mfma_i32_32x32x32_i8, a block of 32 weight rows (the
// second operand) against the digits of TG assignments (the first: row 4 t + p is digit p of
// t; of three, p = 3 is the last digit again), for which the weights go by way of LDS: they
// come as whole blocks a lane, and lane (row l % 32, h = l / 32) multiplies dwords 2 h and 2 h + 1 of a
// block, nibbles as 16 (n - 8).  It pays from two assignments on: with matrix instructions for one as
// well 12 tokens 59.3 us for 53.3, 19 tokens 74.0 for 71.0, 64 tokens (four an expert) 105.9 for 106.2.
// TG: what LDS holds of four workgroups a unit.  16-bit rows (three digits) with TG 4, 6, 8 (8: three
// workgroups): 12 tokens 52.6, 52.8, 55.4, 19 tokens 70.7, 70.8, 72.4, 48 tokens 105, 96, 99, 64 tokens 122,
// 106, 105; fp32 rows (four digits) with 4 and 8 (two workgroups): 19 tokens 72.7, 83.5, 64 tokens 129, 130.
// Bound by memory: 64 tokens at 64 experts, bf16, read 226 MB (gate, up) in 54.7 us and 113 MB in 28.2, 4.1
// TB/s (a 1 GiB copy 5.15); about a tenth is the third digit's, its copies and products (with two
// digits, which do not hold enough, 50.0 and 26.4).
template <int NP, int TG_>
struct LkMoeShare {
    static constexpr int Z = 8 * LkMoeRec<NP>::PIECES, NZ = (Z + 63) / 64;      // pieces of a step's digits
    static constexpr int TG = TG_;                       // assignments at a time
    // the digits of assignment t, so far apart that the 16 rows' reads use all banks alike
    static __device__ __forceinline__ constexpr int at(int t) { return t * Z + t / 2; }
    struct Wave {
        lk_u4 x[TG * Z + (TG - 1) / 2];
        lk_u4 w[32][8];                                  // rows' blocks, block b of row r in slot b ^ r / 2 % 8; of rows 16 .. 31
                                                         // the halves changed over, so that 32 lanes' reads use all banks
        lk_u4 d[32];                                     // their scales
    };
    union {
        Wave wave[4];
        float part[2][TG][64];                           // [part of K][assignment][row of 32 gate and 32 up, or of 64]
    };
};
template <int NP, int TG>
__device__ __forceinline__ void lk_moe_many_dots(const uint8_t * const (&qs)[4], const _Float16 * const (&d)[4], const uint8_t * rec,
                                                 int bpr, int trow, LkMoeShare<NP, TG> & sh, float (&acc)[4]) {
    constexpr int PC = LkMoeRec<NP>::PIECES, Z = LkMoeShare<NP, TG>::Z, NZ = LkMoeShare<NP, TG>::NZ;
    const int lane = threadIdx.x & 63, c = lane >> 3, g = lane & 7, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ns = (bpr + 7) / 8;                        // steps; this wave's are s0, s0 + 2, ...
    typename LkMoeShare<NP, TG>::Wave & me = sh.wave[wv];
    const uint32_t lds = lk_lds_addr(me.x);
    lk_u4 w[4];
    _Float16 dw[4];
    auto load = [&](int s) {
        const int b = 8 * s + g;
        const uint32_t wb = (uint32_t) (c * bpr + (b < bpr ? b : bpr - 1));                      // in bounds
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            // read once: past the caches' order, so that the lines of scales stay (10 tokens 53 us, so 50)
            w[m] = __builtin_nontemporal_load((const lk_u4 *) ((const char *) qs[m] + wb * 16u));
            dw[m] = lk_moe_ld<_Float16>(d[m], wb * 2u);
        }
    };
    auto copy = [&](int s) {
        const int left = (bpr - 8 * s) * PC;             // pieces to the row's end; none: the row's first
        const uint8_t * src = rec + ((size_t) trow * bpr + (left > 0 ? 8 * s : 0)) * (PC * 16);
#pragma unroll
        for (int z = 0; z < NZ; ++z) {
            const int i = 64 * z + lane;
            if (i < Z) lk_dma16c_so(src, 16u * (i < left ? i : 0), lds + 1024u * z);
        }
    };
    load(wv >> 1);
    copy(wv >> 1);
#pragma unroll 1
    for (int s = wv >> 1; s < ns; s += 2) {
        const bool in = 8 * s + g < bpr;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // the copies; the weights, asked for before, come with them
        uint32_t lo[4][4], hi[4][4];
        float dv[4];
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            dv[m] = (float) dw[m];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                lo[m][k] = w[m][k] & 0x0F0F0F0Fu;
                hi[m][k] = (w[m][k] >> 4) & 0x0F0F0F0Fu;
            }
        }
        load(s + 2);                                     // past the last: in bounds, not used
        lk_moe_token_dots<NP, 4>(me.x + g * PC, in, lo, hi, dv, acc);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");          // the digits have been read
        copy(s + 2);
    }
    // the last copies, not used, end before LDS is given to another workgroup
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// The same for n of up to TG assignments, over the steps s0, s0 + 2, ..., or of PAIRS, s0, s0 + 1, s0 + 8,
// s0 + 9, ....  sum[i]: the 32 rows of the four matrices, row l % 32; assignment 2 i + l / 32.  The
// blocks of a step are summed apart over the steps and joined as the dots' lanes are, so that a
// token's result does not depend, by a bit, on how many others chose its expert.
template <bool PAIRS, int NP, int TG>
__device__ __forceinline__ void lk_moe_mfma(const uint8_t * const (&qs)[4], const _Float16 * const (&d)[4], const uint8_t * rec, int bpr,
                                            const int (&trow)[TG], int n, int s0, typename LkMoeShare<NP, TG>::Wave & me, float (&sum)[TG / 2]) {
    typedef LkMoeShare<NP, TG> Share;
    constexpr int PC = LkMoeRec<NP>::PIECES, Z = Share::Z, NZ = Share::NZ, NE = TG / 2;
    const int lane = threadIdx.x & 63, c = lane >> 3, g = lane & 7;
    const int r = lane & 31, h = lane >> 5, ns = (bpr + 7) / 8;
    const uint32_t lds = lk_lds_addr(me.x);
    const int p = (r & 3) < NP ? r & 3 : NP - 1;
    const lk_i4 * xa = (const lk_i4 *) (me.x + Share::at(r / 4 % TG) + 2 * p + h);       // + PC b: the row's digits
    const float * xs[NE];                                // + 4 PC b: the scales
#pragma unroll
    for (int e = 0; e < NE; ++e) xs[e] = (const float *) (me.x + Share::at(2 * e + h) + 2 * NP) + 3;
    lk_u4 w[4];
    _Float16 dw[4];
    auto load = [&](int s) {
        const int b = 8 * s + g;
        const uint32_t wb = (uint32_t) (c * bpr + (b < bpr ? b : bpr - 1));                      // in bounds
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            w[m] = lk_moe_ld<lk_u4>(qs[m], wb * 16u);
            dw[m] = lk_moe_ld<_Float16>(d[m], wb * 2u);
        }
    };
    auto copy = [&](int s) {
        if (s >= ns) return;                             // wave-uniform, as the next two
        const int left = (bpr - 8 * s) * PC;             // pieces to the row's end
#pragma unroll
        for (int t = 0; t < TG; ++t) {
            if (t >= n) break;
            const uint8_t * src = rec + ((size_t) trow[t] * bpr + 8 * s) * (PC * 16);
#pragma unroll
            for (int z = 0; z < NZ; ++z) {
                const int i = 64 * z + lane;
                if (i < Z && i < left) lk_dma16c_so(src, 16u * i, lds + 16u * Share::at(t) + 1024u * z);
                if (left < Z && i >= left && i < Z) me.x[Share::at(t) + i] = lk_u4{ 0, 0, 0, 0 };
            }
        }
    };
    float acc[8][NE] = {};
    auto next = [](int s) { return !PAIRS ? s + 2 : s & 1 ? s + 7 : s + 1; };
    load(s0);
    copy(s0);
#pragma unroll 1
    for (int s = s0; s < ns; s = next(s)) {
        const bool in = 8 * s + g < bpr;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); // the copies; the weights, asked for before, come with them
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            me.w[8 * m + c][g ^ (4 * (m & 1) + (c >> 1))] = m < 2 ? w[m] : lk_u4{ w[m][2], w[m][3], w[m][0], w[m][1] };
            ((_Float16 *) &me.d[8 * m + c])[g] = in ? dw[m] : (_Float16) 0.0f;
        }
        __builtin_amdgcn_wave_barrier();
        load(next(s));                                   // past the last: in bounds, not used
        union { lk_u4 q; _Float16 h[8]; } dv;
        dv.q = me.d[r];
        lk_i4 x[2];
        float sc[2][NE];
        uint64_t v[2];
        auto read = [&](int b) {
            x[b & 1] = xa[PC * b];
#pragma unroll
            for (int e = 0; e < NE; ++e) sc[b & 1][e] = xs[e][4 * PC * b];
            v[b & 1] = ((const uint64_t *) &me.w[r][b ^ (r >> 1 & 7)])[h ^ r >> 4];
        };
        read(0);
#pragma unroll
        for (int b = 0; b < 8; ++b) {                    // a block's operands are read before the products of the one before
            if (b < 7) read(b + 1);
            asm volatile("" ::: "memory");
            const uint32_t u0 = (uint32_t) v[b & 1], u1 = (uint32_t) (v[b & 1] >> 32);
            const lk_i4 wv = { (int) ((u0 << 4 & 0xF0F0F0F0u) ^ 0x80808080u), (int) ((u1 << 4 & 0xF0F0F0F0u) ^ 0x80808080u),
                               (int) ((u0 & 0xF0F0F0F0u) ^ 0x80808080u), (int) ((u1 & 0xF0F0F0F0u) ^ 0x80808080u) };
            lk_i16v zero = {};
            const lk_i16v sv = __builtin_amdgcn_mfma_i32_32x32x32_i8(x[b & 1], wv, zero, 0, 0, 0);
            const float dd = (float) dv.h[b] * 0.0625f;  // the nibbles are 16 times theirs
#pragma unroll
            for (int e = 0; e < NE; ++e) {
                if (2 * e >= n) break;                   // wave-uniform
                // a plane's products: at most 32 * 128 * 128 = 2^19
                const int s4[4] = { sv[4 * e], sv[4 * e + 1], sv[4 * e + 2], sv[4 * e + 3] };
                acc[b][e] = __builtin_fmaf(dd * sc[b & 1][e], lk_moe_digits_sum<NP>(s4), acc[b][e]);
            }
#pragma unroll
            for (int e = 0; e < NE; ++e) asm volatile("" : "+v"(acc[b][e]) :: "memory");
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");          // the digits have been read
        copy(next(s));
    }
#pragma unroll
    for (int e = 0; e < NE; ++e)
        sum[e] = ((acc[0][e] + acc[1][e]) + (acc[2][e] + acc[3][e])) + ((acc[4][e] + acc[5][e]) + (acc[6][e] + acc[7][e]));
}

// 32 rows of one expert's gate and up products for n of its assignments (as, in LDS; the only one:
// as0), all in all `of` them, and what follows: the records of h.  Wave w has half w & 1 of the rows
// and of K the pairs of steps w >> 1, + 4, ...  One assignment by dots, more by matrix instructions;
// both add the blocks in the same order.
template <int NP>
struct LkMoeUp {
    static constexpr int U = 2, TG = 4;
    struct One {
        LkMoeX<NP, U> xs[LK_MOE_NW][1];
        float part[LK_MOE_NW / 2][64];                   // [part of K][row of 32 gate and 32 up]
    };
    union {
        One one;
        typename LkMoeShare<NP, TG>::Wave wave[LK_MOE_NW];
        float part[LK_MOE_NW / 2][TG][64];               // of more: [part of K][assignment][row], where the digits were
    };
};
template <int NP>
__device__ __forceinline__ void lk_moe_up_few(const LkMoeArgs & a, int e, const int * as, int as0, int n, int of, LkMoeUp<NP> & sh) {
    constexpr int TG = LkMoeUp<NP>::TG;
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), half = wv & 1, kp = wv >> 1, F = a.ffn;
    const uint8_t * qs[4];
    const _Float16 * d[4];
    lk_moe_up_rows(a, e, half, qs, d);
    if (n == 1) {
        const int c = lane >> 3, g = lane & 7, trow[1] = { lk_moe_token(a, of == 1 ? as0 : __builtin_amdgcn_readfirstlane(as[0])) };
        float acc[1][4] = {};
        lk_moe_rows<NP, 4, LkMoeUp<NP>::U, 1>(qs, d, a.xr, a.hidden / 32, trow, kp, LK_MOE_NW / 2, sh.one.xs[wv], acc);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const float v = lk_moe_lanes(acc[0][m]);
            if (g == m) sh.one.part[kp][32 * (m >> 1) + 16 * half + 8 * (m & 1) + c] = v;
        }
    } else {
        int trow[TG];
#pragma unroll
        for (int t = 0; t < TG; ++t) trow[t] = lk_moe_token(a, __builtin_amdgcn_readfirstlane(as[t < n ? t : 0]));
        float acc[TG / 2];
        lk_moe_mfma<true, NP, TG>(qs, d, a.xr, a.hidden / 32, trow, n, 2 * kp, sh.wave[wv], acc);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TG / 2; ++i) sh.part[kp][2 * i + (lane >> 5)][2 * (lane & 16) + 16 * half + (lane & 15)] = acc[i];
    }
    __syncthreads();
    const int t = tid >> 5, r = tid & 31;
    if (t < n) {                                         // whole halves of waves
        float gt = 0.0f, up = 0.0f;
#pragma unroll
        for (int k = 0; k < LK_MOE_NW / 2; ++k) {
            const float * p = n == 1 ? sh.one.part[k] : sh.part[k][t];
            gt += p[r];
            up += p[32 + r];
        }
        lk_moe_record<NP>(lk_moe_h(gt, up), r, true,
                          a.hr + ((size_t) (of == 1 ? as0 : as[t]) * (F / 32) + blockIdx.x) * LkMoeRec<NP>::BYTES);
    }
}

// A few tokens; grid (ffn / 32, T * k): the workgroups of an assignment
// whose expert an earlier one has end at once.
template <int NP, int NL>
__global__ void __launch_bounds__(64 * LK_MOE_NW, 4)
lk_k_moe_up_few(const LkMoeArgs a) {
    __shared__ int ids[LK_MOE_FEW * LK_MOE_MAX_TOP_K], as[LK_MOE_FEW];
    __shared__ LkMoeUp<NP> sh;
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), na = a.T * a.k;
    const bool tells = blockIdx.x == 0 && blockIdx.y == 0;          // the one that writes the choices down
    int mine = -1;
    if (a.T == 1 || wv < a.T) {                          // one token: every wave for itself
        const int t = a.T == 1 ? 0 : wv;
        int id[1];
        float l[1][NL], b[NL], w[1];
        lk_moe_logits<NL>(a, t, l[0]);
        lk_moe_bias<NL>(a, b);
        lk_moe_choose<NL, 1>(a, l, b, id, w);
        mine = id[0];
        if (mine >= 0) {
            if (a.T > 1) ids[t * a.k + lane] = mine;
            if (tells && (a.T > 1 || wv == 0)) {
                const int i = t * a.k + lane;
                a.ids[i] = mine;
                a.wts[i] = w[0];
                if (a.ids_out) a.ids_out[i] = mine;
                if (a.wts_out) a.wts_out[i] = w[0];
            }
        }
    }
    if (a.T > 1) {
        __syncthreads();
        mine = lane < na ? ids[lane] : -1;
    }
    const int e = __builtin_amdgcn_readlane(mine, blockIdx.y);
    const uint64_t hits = __ballot(mine == e);
    if (__builtin_ctzll(hits) != (int) blockIdx.y) return;
    const int n = __popcll(hits);
    if (n > 1) {
        if (wv == 0 && mine == e) as[__popcll(hits & ((1ull << lane) - 1))] = lane;
        __syncthreads();
    }
    constexpr int TG = LkMoeUp<NP>::TG;
    for (int at = 0; at < n; at += TG) {
        if (at) __syncthreads();                         // part has been read
        lk_moe_up_few<NP>(a, e, as + at, blockIdx.y, n - at < TG ? n - at : TG, n, sh);
    }
}

// n of up to TG assignments (as, the rows of records trow) of an expert: the sums of the
// workgroup's 64 rows over each part of K, into sh.part.
template <bool UP, int NP, int TG>
__device__ __forceinline__ void lk_moe_many_part(const uint8_t * const (&qs)[4], const _Float16 * const (&d)[4], const uint8_t * rec,
                                                 int bpr, const int (&trow)[TG], int n, LkMoeShare<NP, TG> & sh) {
    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = wv & 1, kp = wv >> 1;
    if (n == 1) {
        const int c = lane >> 3, g = lane & 7;
        float acc[4] = {};
        lk_moe_many_dots<NP, TG>(qs, d, rec, bpr, trow[0], sh, acc);
        __syncthreads();                                 // part lies where the digits were
#pragma unroll
        for (int m = 0; m < 4; ++m) {
            const float v = lk_moe_lanes(acc[m]);
            if (g == m) sh.part[kp][0][UP ? 32 * (m >> 1) + 16 * half + 8 * (m & 1) + c : 32 * half + 8 * m + c] = v;
        }
    } else {
        float acc[TG / 2];
        lk_moe_mfma<false, NP, TG>(qs, d, rec, bpr, trow, n, kp, sh.wave[wv], acc);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TG / 2; ++i)
            sh.part[kp][2 * i + (lane >> 5)][UP ? 2 * (lane & 16) + 16 * half + (lane & 15) : 32 * half + (lane & 31)] = acc[i];
    }
    __syncthreads();
}
template <int NP, int TG>
__device__ __forceinline__ void lk_moe_up_many(const LkMoeArgs & a, int e, const int (&as)[TG], int n, LkMoeShare<NP, TG> & sh) {
    const int F = a.ffn, tid = threadIdx.x;
    const uint8_t * qs[4];
    const _Float16 * d[4];
    lk_moe_up_rows(a, e, __builtin_amdgcn_readfirstlane(tid >> 6) & 1, qs, d);
    int trow[TG];
#pragma unroll
    for (int t = 0; t < TG; ++t) trow[t] = lk_moe_token(a, as[t]);
    lk_moe_many_part<true, NP, TG>(qs, d, a.xr, a.hidden / 32, trow, n, sh);
    const int t = tid >> 5, r = tid & 31;
    if (t < n) {                                         // whole halves of waves
        const float gt = sh.part[0][t][r] + sh.part[1][t][r], up = sh.part[0][t][32 + r] + sh.part[1][t][32 + r];
        int at = as[0];
#pragma unroll
        for (int k = 1; k < TG; ++k) at = t == k ? as[k] : at;
        lk_moe_record<NP>(lk_moe_h(gt, up), r, true, a.hr + ((size_t) at * (F / 32) + blockIdx.x) * LkMoeRec<NP>::BYTES);
    }
}
template <int NP, int TG>
__device__ __forceinline__ void lk_moe_down_many(const LkMoeArgs & a, int e, const int (&as)[TG], int n, LkMoeShare<NP, TG> & sh) {
    const int bpr = a.ffn / 32, H = a.hidden, r0 = blockIdx.x * 64, tid = threadIdx.x, lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6), half = wv & 1;
    const uint8_t * qs[4];
    const _Float16 * d[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {                        // a last tile of 32 rows: those twice
        const size_t row = (size_t) e * H + (r0 + 32 * half < H ? r0 + 32 * half : r0) + 8 * m;
        qs[m] = a.qs[2] + row * bpr * 16;
        d[m] = a.d[2] + row * bpr;
    }
    lk_moe_many_part<false, NP, TG>(qs, d, a.hr, bpr, as, n, sh);
#pragma unroll
    for (int t = 0; t < TG; ++t)         // a wave per assignment
        if ((t & 3) == wv && t < n && r0 + lane < H)
            a.y[(size_t) as[t] * H + r0 + lane] = sh.part[0][t][lane] + sh.part[1][t][lane];
}

// grid (row tiles, slots, groups of TG assignments that an expert may have).  An expert of many
// assignments has a workgroup for each group, which finds the weights in the cache: 64 tokens, all 8
// experts of 2048 x 768 chosen, 62 us, fp32 rows 76 (one workgroup for all groups of an expert, when
// rows had a digit less: 112 for 58 and 162 for 74).  The workgroups of groups that an expert has not
// got cost less than they save.
template <int NP, int TG, bool UP>
__global__ void __launch_bounds__(LK_MOE_THREADS, 4)
lk_k_moe_many(const LkMoeArgs a) {
    __shared__ LkMoeShare<NP, TG> sh;
    // written by the launch before: read as constants, by scalar loads
    typedef const __attribute__((address_space(4))) LkMoeTab Tab;
    Tab & tab = *(Tab *) (uintptr_t) a.tab;
    const int slot = blockIdx.y, at = TG * blockIdx.z, e = tab.slot[slot].e, left = tab.slot[slot].n - at, n = left < TG ? left : TG;
    if (n <= 0) return;
    int as[TG];
#pragma unroll
    for (int t = 0; t < TG; ++t) as[t] = tab.list[slot][at + (t < n ? t : 0)];
    if constexpr (UP) lk_moe_up_many<NP, TG>(a, e, as, n, sh);
    else              lk_moe_down_many<NP, TG>(a, e, as, n, sh);
}

// A few tokens: a workgroup of 16 waves has 8 rows of every expert that was
// chosen (at most 64), and adds them up itself.  The waves share the experts, Q = 16 /
// experts of them (at least one) to each, taking its block groups in turn.
template <int TYPE, int NP>
__global__ void __launch_bounds__(64 * LK_MOE_NWF, 4)
lk_k_moe_down_few(const LkMoeArgs a) {
    typedef typename LkElem<TYPE>::type T;
    constexpr int R = 8, U = 2, TK = 2, MAXA = LK_MOE_FEW * LK_MOE_MAX_TOP_K;
    __shared__ LkMoeX<NP, U> xs[LK_MOE_NWF][TK];
    // [q][assignment][row]: q * assignments is at most 16 / experts * (experts * LK_MOE_FEW), or MAXA
    __shared__ float part[LK_MOE_NWF * LK_MOE_FEW][R];
    static_assert(LK_MOE_NWF * LK_MOE_FEW >= MAXA, "part");
    const int tid = threadIdx.x, lane = tid & 63, c = lane >> 3, g = lane & 7;
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
                lk_moe_rows<NP, 1, U, 2>(qs, d, a.hr, bpr, trow, q, Q, xs[wv], acc);
                const float v0 = lk_moe_lanes(acc[0][0]), v1 = lk_moe_lanes(acc[1][0]);
                if (g < 2) part[q * na + trow[g]][c] = g ? v1 : v0;
            } else {
                const int trow[1] = { t0 };
                float acc[1][1] = {};
                lk_moe_rows<NP, 1, U, 1>(qs, d, a.hr, bpr, trow, q, Q, xs[wv], acc);
                const float v0 = lk_moe_lanes(acc[0][0]);
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
    const size_t k = m->top_k, H = m->hidden, F = m->ffn, REC = LkMoeRec<4>::BYTES;        // of three digits: less
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
    if (lk_moe_check(moe)) return 0;
    if (T < 0 || T > LK_MOE_MAX_TOKENS) {
        lk_fail(hipErrorInvalidValue, "lk_moe_work_bytes: %d tokens (0..%d)", T, LK_MOE_MAX_TOKENS);
        return 0;
    }
    return lk_moe_layout(moe, T, nullptr, nullptr);
}

static bool lk_moe_few(const LkMoeArgs & a, int type) { return a.T <= 5 || (a.T <= LK_MOE_FEW && a.T * a.k <= (type == LK_F32 ? 16 : 28)); }

template <int TYPE>
static void lk_moe_go(const LkMoeArgs & a, hipStream_t st) {
    constexpr int NP = TYPE == LK_F32 ? 4 : 3, TG = NP == 4 ? 4 : 6;
    const bool few = lk_moe_few(a, TYPE);
    const int nE = (a.E + 3) / 4, na = a.T * a.k, slots = na < a.E ? na : a.E;
    hipLaunchKernelGGL((lk_k_moe_router<TYPE, NP>), dim3(nE + (a.hidden / 8 + LK_MOE_THREADS - 1) / LK_MOE_THREADS, (a.T + 3) / 4),
                       dim3(LK_MOE_THREADS), 0, st, a, nE);
    auto route = [&](auto regs) {
        constexpr int NL = decltype(regs)::value;
        if (a.T <= 16)      hipLaunchKernelGGL((lk_k_moe_route<NL, 1>), dim3(1), dim3(1024), 0, st, a);
        else if (a.T <= 32) hipLaunchKernelGGL((lk_k_moe_route<NL, 2>), dim3(1), dim3(1024), 0, st, a);
        else                hipLaunchKernelGGL((lk_k_moe_route<NL, 4>), dim3(1), dim3(1024), 0, st, a);
    };
    auto go = [&](auto regs) {                           // registers of 64 experts a choosing wave holds
        constexpr int NL = decltype(regs)::value;
        if (few)
            hipLaunchKernelGGL((lk_k_moe_up_few<NP, NL>), dim3(a.ffn / 32, na), dim3(64 * LK_MOE_NW), 0, st, a);
        else
            route(LkInt<NL>{});
    };
    if (a.E <= 64) go(LkInt<1>{});
    else           go(LkInt<LK_MOE_MAX_EXPERTS / 64>{});
    if (few) {
        hipLaunchKernelGGL((lk_k_moe_down_few<TYPE, NP>), dim3(a.hidden / 8), dim3(64 * LK_MOE_NWF), 0, st, a);
        return;
    }
    const int groups = (a.T - 1) / TG + 1;
    hipLaunchKernelGGL((lk_k_moe_many<NP, TG, true>), dim3(a.ffn / 32, slots, groups), dim3(LK_MOE_THREADS), 0, st, a);
    hipLaunchKernelGGL((lk_k_moe_many<NP, TG, false>), dim3((a.hidden + 63) / 64, slots, groups), dim3(LK_MOE_THREADS), 0, st, a);
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
    a.hidden = moe->hidden; a.ffn = moe->ffn; a.score = moe->score; a.renorm = moe->renorm; a.kinv = 65536 / moe->top_k + 1; a.scale = moe->scale;
    const hipStream_t st = lk_stream(stream);
    if (type == LK_F32)      lk_moe_go<LK_F32>(a, st);
    else if (type == LK_F16) lk_moe_go<LK_F16>(a, st);
    else                     lk_moe_go<LK_BF16>(a, st);
    return lk_launch_status("lk_moe_q4_0");
}

// paged_attn.hip - attention of a batch's new tokens over its sequences' pages: single
// tokens, trees of drafted tokens, causal runs (lk_paged_attn).
//
//     x_ij = scale * q_i . k_j;  x = cap * tanh(x / cap);  x += slope_h * (position of j - position of i)
//     out_i = sum_j exp(x_ij) v_j / sum_j exp(x_ij)      over the j that i sees
//
// The work is one line of key tiles: per sequence, chunk of its new tokens and group of kv
// heads ("item") the tiles of the keys that the chunk sees.  Each of a fixed number of workgroups
// takes an equal run of that line, whatever the lengths are: it finds its place from the
// lengths on the device, walks on from item to item, and its DMA runs ahead over the
// borders.  An item inside one run is finished there; one that is cut leaves partials
// (max, sum, unnormalised rows), which a second kernel joins in order.  A workgroup has at
// most two cut items, one at each end of its run, so the workspace does not depend on the
// batch.
//
// In a workgroup a tile (16 KB of K rows and 16 KB of V rows of the group's heads, fetched by LDS DMA into a
// ring) is shared by waves that differ in kv head, in the query columns they hold, and, where
// there are too few heads and columns, in the keys they take.  A wave computes S^T = K.Q^T and
// O^T += V^T.P^T on 16x16 tiles of the matrix cores: a score tile leaves the matrix core as the
// operand the second product takes, so P stays in registers.  Columns are (token, query head)
// pairs of one kv head.
// The sum of the weights comes from the same product (a row of ones), so weights and sum are
// rounded alike.
#include "lk_paged.h"

#define LK_PA_TILEB 32768          // a tile: K rows, then V rows
// Weights are 2^(score - offset).  The offset is set so that the largest weight is 2^LIFT, and raised when one passes
// 2^HEADROOM.  In fp16, whose steps below 2^-14 are 2^-24 whatever the value, the largest is 2^7 to 2^15, so that
// a weight keeps its 11 bits down to 2^-21 of the row's first maximum.  In bf16, whose values reach the end of fp32,
// it is 2^-8 to 1: a weight times a value stays finite.
#define LK_PA_NONE  3.0e38f        // minus the offset of no score: 2^(offset - any score in sight) is 0 against it
#define LK_PA_SOME  2.0e38f        // the same for a column that sees keys, none of which had a weight yet

// Two kinds of workgroup.  For up to 16 columns a kv head (STEP 16) the cache's bytes bound it: one workgroup a
// CU, a ring of four tiles, so that 96 KB are on their way (64 sequences of up to 8192, 32 / 8 heads of 128, bf16: 212 us,
// 6.6 TB/s; one of 131072 in 42 us, 6.3 TB/s, the pieces' sum 6 more).  For more (STEP 32) the products and
// exponentials do: two workgroups a CU of one wave a SIMD each, which wait at barriers of their own, and two tiles
// (2 x 4096 new tokens 238 us, 493 TFLOP/s, and their join; of 586 thousand cycles a SIMD issues matrix
// instructions for 201 and others for 284, which hardly overlap).  Between the two, 8 tokens of 4 heads a kv head, STEP 32
// too: one sequence at 30000 22.4 us against 28.6, 16 at 1000 15.1 against 19.9.  DMA and products of short runs wait
// for each other: 13 trees of up to 64 at 4096 45 us, where a SIMD issues for 60 of 126 thousand cycles.
__host__ __device__ constexpr int lk_pa_waves(int d, int step) { return step == 16 && d == 64 ? 8 : 4; }
__host__ __device__ constexpr int lk_pa_bufs(int step) { return step == 16 ? 4 : 2; }
__host__ __device__ constexpr int lk_pa_wgs(int step) { return step == 16 ? 256 : 512; }
#define LK_PA_MAX_WGS 512

typedef short lk_s4 __attribute__((ext_vector_type(4)));
typedef __bf16 lk_b8 __attribute__((ext_vector_type(8)));
typedef __bf16 lk_b4 __attribute__((ext_vector_type(4)));

template <int CTYPE> struct LkMm;
template <> struct LkMm<LK_F16> {
    typedef _Float16 T;
    typedef lk_h8 V8;
    typedef lk_h4 V4;
#ifdef __HIP_DEVICE_COMPILE__
    static __device__ __forceinline__ lk_f4 k32(V8 a, V8 b, lk_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ lk_f4 k16(V4 a, V4 b, lk_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0); }
#else
    static __device__ __forceinline__ lk_f4 k32(V8, V8, lk_f4 c) { return c; }
    static __device__ __forceinline__ lk_f4 k16(V4, V4, lk_f4 c) { return c; }
#endif
    static constexpr uint16_t INF = 0x7C00;
    static constexpr uint32_t LEAD = 0xFFFFE000;               // the bits of an fp32 number that the type holds
    static constexpr float LIFT = 7.0f, HEADROOM = 15.0f;
};
template <> struct LkMm<LK_BF16> {
    typedef __bf16 T;
    typedef lk_b8 V8;
    typedef lk_b4 V4;
#ifdef __HIP_DEVICE_COMPILE__
    static __device__ __forceinline__ lk_f4 k32(V8 a, V8 b, lk_f4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ lk_f4 k16(V4 a, V4 b, lk_f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(lk_s4, a), __builtin_bit_cast(lk_s4, b), c, 0, 0, 0);
    }
#else
    static __device__ __forceinline__ lk_f4 k32(V8, V8, lk_f4 c) { return c; }
    static __device__ __forceinline__ lk_f4 k16(V4, V4, lk_f4 c) { return c; }
#endif
    static constexpr uint16_t INF = 0x7F80;
    static constexpr uint32_t LEAD = 0xFFFF0000;
    static constexpr float LIFT = -8.0f, HEADROOM = 0.0f;
};

struct LkPaArgs {
    const void * q;
    void * out;
    const char * kp, * vp;
    const int32_t * first, * lens, * table, * pos;
    const uint64_t * mask;
    const float * slopes;
    float * acc;                   // partials: [2 * run + end][block of columns][D / 16][column][4][4 dims]
    float2 * ml;                   // and their (max, sum; lk_pa_factor): [..][..][16]
    int4 * cut;                    // per run the cut item that begins in it: (pieces, first row, rows, kv head group)
    int ldq, ldo, n_seqs, rows, ldt, width, page_sh, n_pages;
    int hkv, g;                    // g = query heads a kv head
    int nhg, hg_sh, qw_sh, kw_sh;  // groups of 2^hg_sh kv heads; a workgroup's waves = heads x column groups x key shares
    int qc;                        // tokens a chunk, a power of two up to 64
    int extra;                     // places of the line an item takes in front of its tiles
    float sc, scale, cap, inv_cap; // sc = scale * log2(e), inv_cap = 1 / cap
};

// What keys that no row sees are fetched from; never written.
static __device__ __align__(1024) char lk_pa_zeros[1024];

// Wave-uniform loads of the tables by the scalar unit: they are counted apart from the DMA in flight,
// which a vector load would be waited for together with.
__device__ __forceinline__ int lk_sld(const int32_t * p, long i) {
#ifdef __HIP_DEVICE_COMPILE__
    return ((const __attribute__((address_space(4))) int32_t *) (uintptr_t) p)[i];
#else
    return p[i];
#endif
}

// The arguments where the launch left them.  What is needed once an item or less is read there again each time
// (args() below): kept for the whole kernel, the fifty values would take the scalar registers that a tile's
// loops need.  These are free of spilled scalars but for a few reads; around them, where tiles are fetched and
// items begin and end, 180 to 360 scalars of an instance pass through lanes of vector registers.
#ifdef __HIP_DEVICE_COMPILE__
typedef __attribute__((address_space(4))) LkPaArgs LkPaC;
__device__ __forceinline__ const LkPaC * lk_pa_kernarg() { return (const LkPaC *) __builtin_amdgcn_kernarg_segment_ptr(); }
#else
typedef LkPaArgs LkPaC;
__device__ __forceinline__ const LkPaC * lk_pa_kernarg() { return nullptr; }
#endif

// ---- the line of tiles: every item has a.extra places, for what it costs to begin and end one, and then
// its tiles ------------------------------------------------------------
// Tiles of chunk c of a sequence: the keys up to the last one that a row of the chunk sees.
__device__ __forceinline__ int lk_pa_vis(const LkPaC & a, const LkSeq & s, int c) {
    int e = a.mask ? ((c * a.qc) & ~63) + 64 : (c + 1) * a.qc;
    e = s.len + (e < s.n ? e : s.n);
    const int cap = a.width << a.page_sh;
    return e < cap ? e : cap;
}
__device__ __forceinline__ int lk_pa_tiles(int vis, int tk_sh) {
    const int t = (vis + (1 << tk_sh) - 1) >> tk_sh;
    return t > 0 ? t : 1;                                  // a chunk that sees nothing still has its zeros to write
}
__device__ __forceinline__ LkSeq lk_pa_seq(const LkPaC & a, int b) {     // by a lane
    return lk_seq(a.first[b], a.first[b + 1], a.lens[b], a.rows, a.width << a.page_sh);
}
__device__ __forceinline__ long lk_pa_seq_tiles(const LkPaC & a, const LkSeq & s, int tk_sh) {
    long n = 0;
    for (int c = 0; c * a.qc < s.n; ++c) n += lk_pa_tiles(lk_pa_vis(a, s, c), tk_sh) + a.extra;
    return n * a.nhg;
}

__device__ __forceinline__ long lk_shfl64(long v, int src) {
    const int lo = __shfl((int) v, src, 64), hi = __shfl((int) (v >> 32), src, 64);
    return (long) ((unsigned long) (unsigned) hi << 32 | (unsigned) lo);
}
__device__ __forceinline__ long lk_uniform64(long v) {
    const unsigned lo = __builtin_amdgcn_readfirstlane((int) v), hi = __builtin_amdgcn_readfirstlane((int) (v >> 32));
    return (long) ((unsigned long) hi << 32 | lo);
}

// Sum of a value over the lanes up to each, by lane shifts where the sums fit 32 bits.
__device__ __forceinline__ long lk_pa_scan(long v) {
    const int lane = threadIdx.x & 63;
    if (__ballot(v >> 25) == 0) {
        uint32_t s = (uint32_t) v;
#ifdef __HIP_DEVICE_COMPILE__
        s += __builtin_amdgcn_update_dpp(0, (int) s, 0x111, 0xF, 0xF, false);      // row_shr 1, 2, 4, 8: within 16 lanes
        s += __builtin_amdgcn_update_dpp(0, (int) s, 0x112, 0xF, 0xF, false);
        s += __builtin_amdgcn_update_dpp(0, (int) s, 0x114, 0xF, 0xF, false);
        s += __builtin_amdgcn_update_dpp(0, (int) s, 0x118, 0xF, 0xF, false);
        s += __builtin_amdgcn_update_dpp(0, (int) s, 0x142, 0xA, 0xF, false);      // lane 15 of a row to the next, for rows 1 and 3
        s += __builtin_amdgcn_update_dpp(0, (int) s, 0x143, 0xC, 0xF, false);      // lane 31 to rows 2 and 3
#endif
        return s;
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const long t = lk_shfl64(v, (lane - o) & 63);
        if (lane >= o) v += t;
    }
    return v;
}

// A place on the line: tile t of the nt tiles of (sequence b, chunk c, head group h).
struct LkPaAt {
    int b, c, h, t, nt, vis;
    LkSeq s;
    const int32_t * row;           // the sequence's pages
};
__device__ __forceinline__ void lk_pa_item(const LkPaC & a, LkPaAt & p, int tk_sh) {
    p.vis = lk_pa_vis(a, p.s, p.c);
    p.nt = lk_pa_tiles(p.vis, tk_sh);
}
// The next item's first tile; behind the last one b is n_seqs.
__device__ __forceinline__ void lk_pa_next(const LkPaC & a, LkPaAt & p, int tk_sh) {
    p.t = 0;
    if (++p.h < a.nhg) return;
    p.h = 0;
    ++p.c;
    while (p.c * a.qc >= p.s.n) {
        p.c = 0;
        if (++p.b >= a.n_seqs) return;
        p.s = lk_seq(lk_sld(a.first, p.b), lk_sld(a.first, p.b + 1), lk_sld(a.lens, p.b), a.rows, a.width << a.page_sh);
        p.row = a.table + (long) p.b * a.ldt;
    }
    lk_pa_item(a, p, tk_sh);
}

// v, for what is worked out of it to be worked out here: values that hold for the whole kernel and are used
// once a tile or less would otherwise take registers from the start.
__device__ __forceinline__ int lk_here(int v) {
#ifdef __HIP_DEVICE_COMPILE__
    asm volatile("" : "+v"(v));
#endif
    return v;
}

// The factor f of a piece's rows where they are joined, l its sum of weights: with the sign bit set (which the
// joins take off) there are infinities among the rows, and the factor is above 0, as their weights are.
__device__ __forceinline__ float lk_pa_factor(float f, float l) { return signbit(l) ? fmaxf(f, 0x1p-149f) : f; }

// 1 / the sum l of the weights, m their offset.  Without any weight a row that sees nothing gets zeros, one that
// sees keys of score -inf alone is no number.
__device__ __forceinline__ float lk_pa_inverse(float l, float m) {
    return l != 0.0f ? 1.0f / l : m > -LK_PA_NONE ? NAN : 0.0f;
}

// tanh of t: below 1/2 by its series (the difference of two numbers near 1 would lose what is
// left), the first term left out below 2^-26 of the value; above by the exponential, with the hardware's
// reciprocal (1 ulp): three half steps of the value, where an IEEE division costs ten instructions more.
__device__ __forceinline__ float lk_tanh(float t) {
    const float u = fabsf(t), z = t * t;
    float p = 929569.0f / 638512875.0f;
    p = __builtin_fmaf(-p, z, 21844.0f / 6081075.0f);
    p = __builtin_fmaf(-p, z, 1382.0f / 155925.0f);
    p = __builtin_fmaf(-p, z, 62.0f / 2835.0f);
    p = __builtin_fmaf(-p, z, 17.0f / 315.0f);
    p = __builtin_fmaf(-p, z, 2.0f / 15.0f);
    p = __builtin_fmaf(-p, z, 1.0f / 3.0f);
    const float small = __builtin_fmaf(-p * z, u, u);
    const float e = lk_exp2(u * (-2.0f * LK_LOG2E_F));
#if defined(__HIP_DEVICE_COMPILE__)
    const float large = (1.0f - e) * __builtin_amdgcn_rcpf(1.0f + e);
#else
    const float large = (1.0f - e) / (1.0f + e);
#endif
    return copysignf(u < 0.5f ? small : large, t);
}

// D: head_dim.  RT: rows (LK_F32: q as two parts).  CT: pools.  CB: blocks of 16
// columns a wave holds.  STEP: keys a wave takes at once, 32 by K = 32 products of both kinds, 16 by
// K = 16 for P.V.  MOD: capped or biased scores.
// The weights enter P.V as two parts of the pools' type, a second product for what the first part leaves,
// so that the result is off by its own rounding alone, whatever kernel `max_new` chose (bf16 1.7e-3 relative,
// fp16 2.1e-4; one part 2.3e-3 and 2.9e-4).  Where memory bounds the kernel that costs nothing; 2 x 4096 new
// tokens take 254 us so, 197 with one part, 13 trees of up to 64 at 4096 51 and 45.
template <int D, int RT, int CT, int CB, int STEP, bool MOD>
__global__ void __launch_bounds__(64 * lk_pa_waves(D, STEP), STEP == 16 && D == 128 ? 1 : 2)
lk_k_paged_attn(const LkPaArgs) {
    const LkPaC * const karg = lk_pa_kernarg();
    auto args = [&]() -> const LkPaC & {
        const LkPaC * p = karg;
#ifdef __HIP_DEVICE_COMPILE__
        asm volatile("" : "+s"(p));
#endif
        return *p;
    };
    typedef LkMm<CT> M;
    typedef typename M::T T;
    typedef typename M::V8 V8;
    typedef typename M::V4 V4;
    typedef typename LkElem<RT>::type RowT;
    constexpr bool TWO = RT == LK_F32;
    constexpr int NW = lk_pa_waves(D, STEP), NBUF = lk_pa_bufs(STEP), NB = STEP / 16;
    constexpr int KS = D / 32, DB = D / 16, DC = D / 8;        // steps of q.k, blocks of output dims, 16-byte pieces of a head's row
    constexpr int NF = 16 / NW;                                // pieces of 1 KB a wave fetches of a tile's K, and of its V
    constexpr int AHEAD = NBUF - 1;
    __shared__ __attribute__((aligned(16))) unsigned char s_tile[NBUF][LK_PA_TILEB];
    __shared__ lk_f4 s_x[2][NW][64];                           // key shares' rows on their way to one wave
    __shared__ float2 s_ml[NW][16];
    __shared__ uint64_t s_see[NW][CB][16];                     // which of the 64 tokens from `base` on a column sees
    __shared__ int s_left[NW], s_start[NW][4];                 // a wave's left_out; the run's first item and tile
    __shared__ long s_places[NW];                              // and its places from there on, of which each wave keeps a copy

    const int lane = threadIdx.x & 63, col = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const LkPaC & a0 = args();
    const int kw_sh = a0.kw_sh, kw = w & ((1 << kw_sh) - 1), qw = (w >> kw_sh) & ((1 << a0.qw_sh) - 1), hh = w >> (kw_sh + a0.qw_sh);
    const int rb_sh = a0.hg_sh + (D == 64 ? 7 : 8);             // bytes of a position's piece: its group's heads
    const int rb = 1 << rb_sh;
    const int tk_sh = 14 - rb_sh;                              // keys a tile: 16 KB of K rows
    const int kpw = (1 << tk_sh) >> kw_sh;                   // of them the wave's

    // ---- this workgroup's run of the line ---------------------------------------------
    long total = 0, mine = 0, sum = 0, before = 0;             // sum: of the sequences up to the lane's
    LkSeq ls = { 0, 0, 0 };
    for (int b = lane; b < a0.n_seqs; b += 64) {
        ls = lk_pa_seq(a0, b);
        mine = lk_pa_seq_tiles(a0, ls, tk_sh);
        total += mine;
    }
    const bool one_pass = a0.n_seqs <= 64;
    if (one_pass) {
        sum = lk_pa_scan(mine);
        total = lk_uniform64(lk_shfl64(sum, 63));
    } else {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) total += lk_shfl64(total, lane ^ o);
        total = lk_uniform64(total);
    }
    const long share = (total + lk_pa_wgs(STEP) - 1) / lk_pa_wgs(STEP);
    // Workgroups go round the eight XCDs; runs side by side, whose chunks read the same keys, are given to one XCD and
    // its L2 (13 trees 52.5 -> 51.4 us, 2 x 4096 new tokens, which the products bound, 260 -> 262), but for short runs, which
    // may be fewer than the workgroups and would then be on few XCDs (a tree of 16 at 32768 28.4 that way, 27.1 round).
    const int wgi = share >= 8 ? (blockIdx.x & 7) * (lk_pa_wgs(STEP) / 8) + (blockIdx.x >> 3) : blockIdx.x;
    const long f0 = share * wgi, f1 = f0 + share < total ? f0 + share : total;
    if (f0 >= f1) {
        if (threadIdx.x == 0) args().cut[wgi] = make_int4(0, 0, 0, 0);
        return;
    }
    LkPaAt at;
    for (int b0 = 0;; b0 += 64) {                              // ends: f0 is below the total
        if (!one_pass) {
            const int b = b0 + lane;
            mine = 0;
            if (b < a0.n_seqs) {
                ls = lk_pa_seq(a0, b);
                mine = lk_pa_seq_tiles(a0, ls, tk_sh);
            }
            sum = lk_pa_scan(mine);
        }
        const uint64_t here = __ballot(before + sum > f0);
        if (here) {
            const int src = __builtin_ctzll(here);
            long rem = lk_uniform64(lk_shfl64(f0 - before - (sum - mine), src));
            at.b = b0 + src;
            at.row = a0.table + (long) at.b * a0.ldt;
            at.s.r0 = __builtin_amdgcn_readlane(ls.r0, src);
            at.s.n = __builtin_amdgcn_readlane(ls.n, src);
            at.s.len = __builtin_amdgcn_readlane(ls.len, src);
            for (at.c = 0;; ++at.c) {                          // ends: rem is below the sequence's places
                lk_pa_item(a0, at, tk_sh);
                const long u = (long) (at.nt + a0.extra) * a0.nhg;
                if (rem < u) break;
                rem -= u;
            }
            for (at.h = 0; rem >= at.nt + a0.extra; ++at.h) rem -= at.nt + a0.extra;
            at.t = (int) rem - a0.extra;                       // below 0: in front of the first tile
            break;
        }
        before += lk_uniform64(lk_shfl64(sum, 63));
    }

    // ---- fetch: wave w brings the 1 KB pieces w, w + NW, .. of a tile's K and of its V -----
    // Piece i holds the keys i * rpp .. of the tile, all in one page (a page is a multiple of 16).
    // Within a row its 16-byte pieces are permuted by the key, so that the lanes' reads below meet
    // different ones of the 64 banks: 16 keys of a K piece, 8 keys of two V pieces, over 256 bytes.
    // The pages of the next tile are asked for a tile ahead.
    const int rpp_sh = 10 - rb_sh, rpp = 1 << rpp_sh;
    const uint32_t lds0 = lk_lds_addr(&s_tile[0][0]);
    const uint32_t row_bytes = (uint32_t) a0.hkv * D * 2;
    const char * const kp = a0.kp, * const vp = a0.vp;
    const int page_sh = a0.page_sh, n_pages = a0.n_pages, extra = a0.extra;
    auto swk = [&](int key) -> int { return rb == 128 ? (key >> 1) & 7 : key & 15; };
    auto swv = [&](int key) -> int { return (rb == 128 ? (key >> 1) & 3 : key & 7) << 1; };
    int pg[NF];
    auto ask = [&](const LkPaAt & p) {
#pragma unroll
        for (int i = 0; i < NF; ++i) {
            const int p0 = (p.t << tk_sh) + ((w + NW * i) << rpp_sh);
            pg[i] = lk_sld(p.row, (p0 < p.vis ? p0 : 0) >> page_sh);
        }
    };
    auto fetch = [&](const LkPaAt & p, int slot) {
        const int ln = lk_here(lane), frow = ln >> (6 - rpp_sh), part = ln & ((1 << (6 - rpp_sh)) - 1);
        const uint32_t base = lds0 + (uint32_t) slot * LK_PA_TILEB;
#pragma unroll
        for (int i = 0; i < NF; ++i) {
            const int piece = w + NW * i, p0 = (p.t << tk_sh) + (piece << rpp_sh);
            const bool ok = pg[i] >= 0 && pg[i] < n_pages;
            const size_t off = (((size_t) (ok ? pg[i] : 0) << page_sh) + (p0 & ((1 << page_sh) - 1))) * row_bytes +
                               ((size_t) p.h << rb_sh);
            // the lane's bytes from the piece's first row on
            const int key = (piece << rpp_sh) + frow;
            const uint32_t ko = frow * row_bytes + 16 * (part ^ swk(key)), vo = frow * row_bytes + 16 * (part ^ swv(key));
            const uint32_t lk = base + piece * 1024, lv = lk + LK_PA_TILEB / 2;
            if (ok && p0 + rpp <= p.vis) {
                if constexpr (STEP == 16) {                    // up to 16 columns a head: few others read the tile
                    lk_dma16_so(kp + off, ko, lk);
                    lk_dma16_so(vp + off, vo, lv);
                } else {
                    lk_dma16c_so(kp + off, ko, lk);
                    lk_dma16c_so(vp + off, vo, lv);
                }
            } else {
                // rows that nobody sees are zeros: what lies there must not meet weights of 0 as an infinity or NaN
                // (zeros written to LDS instead cost 4 to 15%: the branch over the lanes)
                const bool live = ok && p0 + frow < p.vis;
                const char * zs = lk_pa_zeros + 16 * ln;
                lk_dma16c(live ? kp + off + ko : zs, lk);
                lk_dma16c(live ? vp + off + vo : zs, lv);
            }
        }
    };

    // ---- a column's state ----------------------------------------------------------------
    V8 qh[CB][KS], ql[TWO ? CB : 1][KS];
    lk_f4 acc[CB][DB], accl[CB];
    float mneg[CB], fac[TWO ? CB : 1];                          // minus the weights' offset (units of log2); score factor of a scaled q
    float slope[MOD ? CB : 1];
    int qpos[MOD ? CB : 1];
    int base = 0;                                               // keys below it are seen by all of the chunk's rows
    bool busy = false;                                          // the wave has columns
    bool left_out = false;                                      // the run met infinities or NaN of V
    // column block cb: the token of the chunk, its row of the step, its query head; false: there is none
    auto column = [&](const LkPaC & a, int cb, int & i, int & row, int & head) -> bool {
        const int c = (qw * CB + cb) * 16 + lk_here(col), i0 = at.c * a.qc, m = at.s.n - i0 < a.qc ? at.s.n - i0 : a.qc;
        i = c / a.g;
        const int h = c - i * a.g;
        const bool live = i < m;
        i = live ? i : 0;
        row = at.s.r0 + i0 + i;
        head = ((at.h << a.hg_sh) + hh) * a.g + (live ? h : 0);
        return live;
    };
    float sc = 0.0f, cap = 0.0f, inv_cap = 0.0f;                // scale (times log2(e) but for MOD), cap
    bool biased = false;
    // the item's `base`, and the tokens from it on that a column sees
    auto set_base = [&](const LkPaC & a) {
        const int blk = (at.c * a.qc) & ~63, slots = a.width << a.page_sh;
        base = at.s.len + blk < slots ? at.s.len + blk : slots;
    };
    auto seen = [&](const LkPaC & a, int i, int row) -> uint64_t {
        const int limit = at.vis - base;                        // of the 64 tokens from base on the ones that have a slot
        const uint64_t lim = limit >= 64 ? ~0ull : limit > 0 ? (1ull << limit) - 1 : 0;
        return (a.mask ? a.mask[row] : ~0ull >> (63 - ((at.c * a.qc + i) & 63))) & lim;
    };
    auto begin = [&]() {
        const LkPaC & a = args();
        sc = MOD ? a.scale : a.sc;
        if constexpr (MOD) {
            cap = a.cap;
            inv_cap = a.inv_cap;
            biased = a.slopes != nullptr;
        }
        set_base(a);
        busy = false;
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
            int i, row, head;
            const bool live = column(a, cb, i, row, head);
            busy |= __ballot(live) != 0;                        // wave-uniform
            if constexpr (MOD) {
                slope[cb] = a.slopes ? a.slopes[head] * LK_LOG2E_F : 0.0f;
                qpos[cb] = a.pos ? a.pos[row] : at.s.len + (row - at.s.r0);
            }
            const RowT * src = (const RowT *) a.q + (size_t) row * a.ldq + (size_t) head * D + 8 * g;
            if constexpr (TWO) {
                // a head is scaled by a power of two to a largest value of 2^14 to 2^15, so that both parts are
                // finite and 22 bits of it count whatever its size is, and its scores back
                float v[KS][8], am = 0.0f;
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    lk_load<8>(src + 32 * ks, v[ks]);
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        v[ks][e] = live ? v[ks][e] : 0.0f;
                        am = fmaxf(am, fabsf(v[ks][e]));
                    }
                }
                am = lk_xrow_max(am);
                int e2 = 0;
                if (am > 0.0f && am < INFINITY) {
                    (void) frexpf(am, &e2);
                    e2 -= 15;
                }
                fac[cb] = fmaxf(ldexpf(sc, e2), 0x1p-126f);     // (smaller, it could be 0 against an infinity)
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const float x = ldexpf(v[ks][e], -e2);
                        const T h = (T) x;
                        qh[cb][ks][e] = h;
                        ql[cb][ks][e] = (T) (x - (float) h);
                    }
            } else {
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    V8 v;
                    __builtin_memcpy(&v, src + 32 * ks, 16);
                    qh[cb][ks] = live ? v : V8{};
                }
            }
            const uint64_t see = seen(a, i, row);               // (a wave reads its own words only)
            if (g == 0) s_see[w][cb][col] = see;
            mneg[cb] = base > 0 || see != 0 ? LK_PA_SOME : LK_PA_NONE;
            accl[cb] = (lk_f4){ 0.f, 0.f, 0.f, 0.f };
#pragma unroll
            for (int db = 0; db < DB; ++db) acc[cb][db] = (lk_f4){ 0.f, 0.f, 0.f, 0.f };
        }
    };

    // ---- keys ---------------------------------------------------------------------------------
    // (a head's pieces start at a multiple of DC, so the parts of a piece's number do not overlap)
    const int kadr = col * rb, ksw = (hh * DC | g) ^ swk(col);
    const int vadr = (4 * g + (col >> 2)) * rb + 8 * (col & 1), vsw = (hh * DC | ((col >> 1) & 1)) ^ swv(4 * g + (col >> 2));
    auto kload = [&](const unsigned char * kt, V8 (&kf)[NB][KS]) {
#pragma unroll
        for (int n = 0; n < NB; ++n)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) kf[n][ks] = *(const V8 *) (kt + kadr + ((16 * n) << rb_sh) + ((ksw ^ (4 * ks)) << 4));
    };
    auto vload = [&](const unsigned char * vt, int n, int db) -> V4 {
        return __builtin_bit_cast(V4, lk_ds_tr4(vt + vadr + ((16 * n) << rb_sh) + ((vsw ^ (2 * db)) << 4)));
    };
    auto scores = [&](const V8 (&kf)[KS], int cb) -> lk_f4 {
        lk_f4 c = { 0.f, 0.f, 0.f, 0.f };
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            c = M::k32(kf[ks], qh[cb][ks], c);
            if constexpr (TWO) c = M::k32(kf[ks], ql[cb][ks], c);
        }
        return c;
    };
    // fp32 rows: an infinity among the keys times a query's second part, which is 0 or of either sign, is no number, and
    // the first part of a small value is 0.  Scores that are not finite are formed again from the signs of the
    // query's finite values and its other values.
    auto endless_scores = [&](const V8 (&kf)[NB][KS], lk_f4 (&c)[CB][NB]) {
        const LkPaC & a = args();
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
            int i, row, head;
            const bool live = column(a, cb, i, row, head);
            const RowT * src = (const RowT *) a.q + (size_t) row * a.ldq + (size_t) head * D + 8 * g;
            lk_f4 o[NB];
#pragma unroll
            for (int n = 0; n < NB; ++n) o[n] = (lk_f4){ 0.f, 0.f, 0.f, 0.f };
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                float v[8];
                V8 q;
                lk_load<8>(src + 32 * ks, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = live ? v[e] : 0.0f;
                    q[e] = (T) (x != 0.0f && fabsf(x) < INFINITY ? copysignf(1.0f, x) : x);
                }
#pragma unroll
                for (int n = 0; n < NB; ++n) o[n] = M::k32(kf[n][ks], q, o[n]);
            }
#pragma unroll
            for (int n = 0; n < NB; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) c[cb][n][r] = fabsf(c[cb][n][r]) < INFINITY ? c[cb][n][r] : o[n][r];
        }
    };
    auto factor = [&](int cb) -> float { return TWO ? fac[cb] : sc; };
    // capped and biased scores in units of log2, of keys k0 .. k0 + 3 (k0: the lane's first)
    auto shaped = [&](lk_f4 & c, int cb, int k0) {
        c *= factor(cb);
        if (cap > 0.0f) {
#pragma unroll
            for (int r = 0; r < 4; ++r) c[r] = cap * lk_tanh(c[r] * inv_cap);
        }
        c *= LK_LOG2E_F;
        if (biased) {
            const int32_t * pos = args().pos;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                int kp = k0 + r;
                if (pos && kp >= at.s.len && kp < at.vis) kp = pos[at.s.r0 + kp - at.s.len];
                c[r] = __builtin_fmaf(slope[cb], (float) (kp - qpos[cb]), c[r]);
            }
        }
    };
    // raises the offset of column block cb to cover a lane's largest score (units of log2)
    auto raise = [&](int cb, float top) {
        if (__ballot(top + mneg[cb] > M::HEADROOM)) {        // wave-uniform (a difference: exact for large scores)
            const float mx = lk_xrow_max(top);
            if (mx + mneg[cb] > M::HEADROOM) {
                const float to = M::LIFT - mx, f = lk_exp2(to - mneg[cb]);
                mneg[cb] = to;
#pragma unroll
                for (int db = 0; db < DB; ++db) acc[cb][db] *= f;
                accl[cb] *= f;
            }
        }
    };
    // weights of four scores in two parts: the leading bits that the type holds, cut off by a mask, and the rest,
    // rounded: 2^-22 of the weight is lost in fp16, 2^-16 in bf16.  (The first part rounded to nearest has to be
    // converted back: a prompt of 4096 with heads of 128, bf16, 279 us for 264, 2 x 4096 in fp16 259 for 262.)
    auto weights = [&](const lk_f4 & c, int cb, V4 & ph, V4 & pl) {
        lk_f4 p, h;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float x = lk_exp2(MOD ? c[r] + mneg[cb] : __builtin_fmaf(c[r], factor(cb), mneg[cb]));
            h[r] = __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & M::LEAD);
            p[r] = x;
        }
        ph = __builtin_convertvector(h, V4);
        p -= h;
        pl = __builtin_convertvector(p, V4);
    };
    // (of fp32 rows' scores NaN is the largest)
    auto larger = [](float x, float y) -> float {
        if constexpr (TWO) return __builtin_elementwise_maximum(x, y);
        else               return fmaxf(x, y);
    };
    auto top4 = [&](const lk_f4 & c) -> float { return larger(larger(c[0], c[1]), larger(c[2], c[3])); };
    auto units = [&](float top, int cb) -> float { return MOD ? top : top * factor(cb); };
    auto join = [](const V4 & x, const V4 & y) -> V8 { return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7); };
    V4 ones4;
#pragma unroll
    for (int i = 0; i < 4; ++i) ones4[i] = (T) 1.0f;

    // whether the column of block cb sees the lane's keys 4g .. 4g + 3 of the 16 from key0 on: four bits
    auto sees = [&](int cb, int key0) -> uint32_t {
        const int d = key0 + 4 * g - base;
        const uint64_t e = s_see[w][cb][col];
        return (uint32_t) (d >= 0 ? (d < 64 ? e >> d : 0) : d > -4 ? e << -d | ((1 << -d) - 1) : 15) & 15;
    };
    // STEP keys, the first of them key0, kf their K rows; `more`: the rows of the STEP keys behind are
    // asked for.  From `base` on there are keys that only some of the rows see.
    auto step = [&](const unsigned char * kt, const unsigned char * vt, int key0, V8 (&kf)[NB][KS], bool more) {
        V4 ph[CB][NB], pl[CB][NB], vf[DB][NB];
        lk_f4 c[CB][NB];
        const bool some = key0 + STEP > base;                   // wave-uniform
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int n = 0; n < NB; ++n) vf[db][n] = vload(vt, n, db);
#pragma unroll
        for (int cb = 0; cb < CB; ++cb)
#pragma unroll
            for (int n = 0; n < NB; ++n) c[cb][n] = scores(kf[n], cb);
        if (more) kload(kt + (STEP << rb_sh), kf);
        auto shape = [&]() {
            if constexpr (MOD) {
#pragma unroll
                for (int cb = 0; cb < CB; ++cb)
#pragma unroll
                    for (int n = 0; n < NB; ++n) shaped(c[cb][n], cb, key0 + 16 * n + 4 * g);
            }
        };
        auto hide = [&]() {
#pragma unroll
            for (int cb = 0; cb < CB; ++cb)
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    const uint32_t bits = sees(cb, key0 + 16 * n);
#pragma unroll
                    for (int r = 0; r < 4; ++r) c[cb][n][r] = (bits >> r) & 1 ? c[cb][n][r] : -INFINITY;
                }
        };
        shape();
        // the softmax first: of the two waves of a SIMD one then multiplies while the other forms weights (2 x 4096 new
        // tokens 271 -> 262 us; no other order of the two parts' instructions within a wave gained anything)
        if constexpr (STEP == 32) __builtin_amdgcn_s_setprio(1);
        if (some) {
            hide();
            // 0 times an infinity is NaN: such values are left out of the product, which would spoil the rows that
            // do not see them, and added at the run's end
            bool odd = false;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int n = 0; n < NB; ++n) {
                    lk_u16x4 u = __builtin_bit_cast(lk_u16x4, vf[db][n]);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const bool o = (u[r] & M::INF) == M::INF;
                        odd |= o;
                        u[r] = o ? 0 : u[r];
                    }
                    vf[db][n] = __builtin_bit_cast(V4, u);
                }
            left_out |= __ballot(odd) != 0;                     // wave-uniform
        }
        // one test for all blocks of columns says whether a max has to be raised
        float top[CB], over;
        auto tops = [&]() {
            over = -INFINITY;
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) {
                top[cb] = top4(c[cb][0]);
                if constexpr (NB == 2) top[cb] = larger(top[cb], top4(c[cb][1]));
                over = larger(over, MOD ? top[cb] + mneg[cb] : __builtin_fmaf(top[cb], factor(cb), mneg[cb]));
            }
        };
        tops();
        if constexpr (TWO) {
            if (__ballot(over != over)) {                       // wave-uniform
                V8 kx[NB][KS];
                kload(kt, kx);
#pragma unroll
                for (int cb = 0; cb < CB; ++cb)
#pragma unroll
                    for (int n = 0; n < NB; ++n) c[cb][n] = scores(kx[n], cb);
                endless_scores(kx, c);
                shape();
                if (some) hide();
                tops();
            }
        }
        if (__ballot(!(over <= M::HEADROOM))) {                 // wave-uniform (NaN of one column hides no other's)
#pragma unroll
            for (int cb = 0; cb < CB; ++cb) raise(cb, units(top[cb], cb));
        }
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
#pragma unroll
            for (int n = 0; n < NB; ++n) weights(c[cb][n], cb, ph[cb][n], pl[cb][n]);
            auto product = [&](const V4 (&v)[NB], lk_f4 o) -> lk_f4 {
                if constexpr (NB == 2) {
                    o = M::k32(join(v[0], v[1]), join(ph[cb][0], ph[cb][1]), o);
                    o = M::k32(join(v[0], v[1]), join(pl[cb][0], pl[cb][1]), o);
                } else {
                    o = M::k16(v[0], ph[cb][0], o);
                    o = M::k16(v[0], pl[cb][0], o);
                }
                return o;
            };
            V4 ones[NB];
#pragma unroll
            for (int n = 0; n < NB; ++n) ones[n] = ones4;
            accl[cb] = product(ones, accl[cb]);
#pragma unroll
            for (int db = 0; db < DB; ++db) acc[cb][db] = product(vf[db], acc[cb][db]);
        }
        if constexpr (STEP == 32) __builtin_amdgcn_s_setprio(0);
    };

    // ---- an item's end, or the run's ----------------------------------------------------------
    // The key shares of a head and its columns meet in the wave with the first of them.
    auto join_shares = [&]() {
        const int kws = 1 << kw_sh;
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
            if (g == 0) s_ml[w][col] = make_float2(-mneg[cb], accl[cb][0]);
            if (lane == 0) s_left[w] = left_out;
            __syncthreads();
            int met = 0;
            for (int k = 0; k < kws; ++k) met |= s_left[w - kw + k];
            left_out = __builtin_amdgcn_readfirstlane(met) != 0;
            float mx = -mneg[cb];
            for (int k = 0; k < kws; ++k) mx = fmaxf(mx, s_ml[w - kw + k][col].x);
            const float f = lk_exp2(-mneg[cb] - mx);
            float l = 0.0f;
            for (int k = 0; k < kws; ++k) {
                const float2 o = s_ml[w - kw + k][col];
                l += o.y * lk_exp2(o.x - mx);
            }
            mneg[cb] = -mx;
            accl[cb][0] = l;
#pragma unroll
            for (int db = 0; db < DB; db += 2) {
                s_x[0][w][lane] = acc[cb][db] * f;
                s_x[1][w][lane] = acc[cb][db + 1] * f;
                __syncthreads();
                if (kw == 0) {
                    lk_f4 o0 = s_x[0][w][lane], o1 = s_x[1][w][lane];
                    for (int k = 1; k < kws; ++k) {
                        o0 += s_x[0][w + k][lane];
                        o1 += s_x[1][w + k][lane];
                    }
                    acc[cb][db] = o0;
                    acc[cb][db + 1] = o1;
                }
                __syncthreads();
            }
        }
    };
    auto finish = [&](bool whole, bool from_first) {
        if (kw_sh) join_shares();
        if (kw != 0) return;
        // infinities or NaN among the sums of a column that are not its scores'
        bool odd = false;
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
            lk_f4 all = { 0.f, 0.f, 0.f, 0.f };
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int r = 0; r < 4; ++r) all[r] = __builtin_fmaf(acc[cb][db][r], 0.0f, all[r]);
            odd |= (all[0] + all[1]) + (all[2] + all[3]) != 0.0f && accl[cb][0] == accl[cb][0];
        }
        left_out |= __ballot(odd) != 0;                         // wave-uniform
        const LkPaC & a = args();
        const int nblk = CB << (a.qw_sh + a.hg_sh);
        const int slot = 2 * wgi + from_first;
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
            int i, row, head;
            if (!column(a, cb, i, row, head)) continue;
            if (whole) {
                const float il = lk_pa_inverse(accl[cb][0], -mneg[cb]);
                RowT * o = (RowT *) a.out + (size_t) row * a.ldo + (size_t) head * D + 4 * g;
#pragma unroll
                for (int db = 0; db < DB; ++db) {
                    float v[4] = { acc[cb][db][0] * il, acc[cb][db][1] * il, acc[cb][db][2] * il, acc[cb][db][3] * il };
                    if (left_out || il != il) {                 // NaN by the values is marked, by its sign, for the run's end
#pragma unroll
                        for (int r = 0; r < 4; ++r) v[r] = v[r] == v[r] ? v[r] : il == il ? -NAN : NAN;
                    }
                    lk_store<4>(o + 16 * db, v);
                }
            } else {
                const size_t blk = (size_t) slot * nblk + ((hh << a.qw_sh) + qw) * CB + cb;
#pragma unroll
                for (int db = 0; db < DB; ++db) *(lk_f4 *) (a.acc + ((blk * DB + db) * 64 + col * 4 + g) * 4) = acc[cb][db];
                if (g == 0) a.ml[blk * 16 + col] = make_float2(-mneg[cb], accl[cb][0]);
            }
        }
    };

    // ---- the run: item by item, in each the tiles that all rows see whole, then the others -------
    // Places of the run behind the current one; an item's last piece may end in front of its first tile.
    long left = f1 - f0;
    if (at.t < 0) {
        left += at.t;
        at.t = 0;
        if (left <= 0) {
            if (threadIdx.x == 0) args().cut[wgi] = make_int4(0, 0, 0, 0);
            return;
        }
    }
    if (lane == 0) {
        s_start[w][0] = at.b, s_start[w][1] = at.c, s_start[w][2] = at.h, s_start[w][3] = at.t;
        s_places[w] = left;
    }
    LkPaAt ft = at;                                             // the next tile to fetch
    long ft_left = left;                                        // places of the run from it on
    int slot = 0, ahead = 0;                                    // the awaited tile's buffer; tiles fetched and not yet taken
    auto fetch_next = [&]() {
        fetch(ft, (slot + ahead) & (NBUF - 1));
        ++ahead;
        if (++ft.t == ft.nt) {
            ft_left -= extra;
            lk_pa_next(args(), ft, tk_sh);
        }
        --ft_left;
        if (ft_left > 0) ask(ft);
    };
    ask(ft);
    for (int i = 0; i < AHEAD && ft_left > 0; ++i) fetch_next();
    int4 cut = make_int4(0, 0, 0, 0);
    while (left > 0) {
        begin();
        const bool from_first = at.t == 0;
        const int t_end = left < at.nt - at.t ? at.t + (int) left : at.nt;        // of this item in this run
        for (; at.t < t_end; ++at.t) {
            // waits for the tile in `slot`, then asks for the tile AHEAD further, into the buffer that every
            // wave has read before the barrier
            if constexpr (AHEAD == 3) {
                if (ahead > 2)       lk_wait_vm<4 * NF>();
                else if (ahead == 2) lk_wait_vm<2 * NF>();
                else                 lk_wait_vm<0>();
            } else {
                static_assert(AHEAD == 1 || AHEAD == 3, "tiles that may stay in flight behind the awaited one: none, or two");
                lk_wait_vm<0>();
            }
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
            if (ft_left > 0) fetch_next();
            const int k0 = (at.t << tk_sh) + kw * kpw;
            if (k0 < at.vis && busy) {                          // the wave's share may lie behind the last key
                const unsigned char * kt = s_tile[slot] + ((kw * kpw) << rb_sh), * vt = kt + LK_PA_TILEB / 2;
                const int n = k0 + kpw < at.vis ? kpw : at.vis - k0;
                V8 kf[NB][KS];
                kload(kt, kf);
                for (int k = 0; k < n; k += STEP) {
                    step(kt + (k << rb_sh), vt + (k << rb_sh), k0 + k, kf, STEP == 32 && k + STEP < n);
                }
            }
            slot = (slot + 1) & (NBUF - 1);
            --ahead;
            --left;
        }
        const bool ends = t_end == at.nt;
        finish(ends && from_first, from_first);
        if (!ends && from_first) {
            // the workgroups that the rest of the item falls to, this one counted
            const long end = f1 + (at.nt - t_end);              // behind the item's last tile
            const int qc = args().qc, m = at.s.n - at.c * qc;
            const long last = end - 1 - f0;                     // its last place, counted from this workgroup's first
            const int more = last >> 31 ? (int) (last / share) : (int) ((uint32_t) last / (uint32_t) share);
            cut = make_int4(more + 1, at.s.r0 + at.c * qc, m < qc ? m : qc, at.h);
        }
        left -= extra;
        if (left > 0) lk_pa_next(args(), at, tk_sh);
    }
    if (threadIdx.x == 0) args().cut[wgi] = cut;

    // ---- infinities and NaN of V, where the run met any ---------------------------------------
    // In the products above they were left out, or met a second part of a weight, which may be 0 or of either sign, a weight
    // that is 0 in the pools' type, or a factor of 0.  The results of the dims in which a column sees some are formed
    // again here from them alone, since nothing finite is left beside them: each counts as it is, its weight
    // being above 0, but for a score of -inf, whose weight is 0 and 0 times it NaN.  (Such a key has an infinite value itself and
    // its score no cap; an infinite query makes its whole row NaN anyway.)  The run's V is scanned once more, behind all
    // that the usual call does (at each item's end these lines took scalar registers from the products' loop:
    // 64 sequences of up to 8192 323 us for 222).  With an infinite value in one of the sequences: 64 of up to 8192
    // 342 us for 229, 2 x 4096 new tokens 495 for 292.
    if (kw != 0 || !left_out) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");      // what the wave's lanes wrote is read and written again
    const LkPaC & a = args();
    at.b = __builtin_amdgcn_readfirstlane(s_start[w][0]);
    at.c = __builtin_amdgcn_readfirstlane(s_start[w][1]);
    at.h = __builtin_amdgcn_readfirstlane(s_start[w][2]);
    at.t = __builtin_amdgcn_readfirstlane(s_start[w][3]);
    left = lk_uniform64(s_places[w]);
    at.s = lk_seq(lk_sld(a.first, at.b), lk_sld(a.first, at.b + 1), lk_sld(a.lens, at.b), a.rows, a.width << a.page_sh);
    at.row = a.table + (long) at.b * a.ldt;
    lk_pa_item(a, at, tk_sh);
    auto endless = [](uint16_t u) -> bool { return (u & M::INF) == M::INF; };
    while (left > 0) {
        const int t0 = at.t, t1 = left < at.nt - t0 ? t0 + (int) left : at.nt;
        const int end = (t1 << tk_sh) < at.vis ? t1 << tk_sh : at.vis, m = (1 << a.page_sh) - 1;
        set_base(a);
        uint64_t see[CB];
        lk_f4 sum[CB][DB];
        uint32_t found[CB];                                     // a bit for each of the lane's dims
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
            int i, row, head;
            (void) column(a, cb, i, row, head);
            see[cb] = seen(a, i, row);
            found[cb] = 0;
#pragma unroll
            for (int db = 0; db < DB; ++db) sum[cb][db] = (lk_f4){ 0.f, 0.f, 0.f, 0.f };
        }
        // 32 keys at a time, some in each of D / 16 loads, 16 bytes a lane; then one by one those that have any
        constexpr int LPK = D / 8, KPL = 64 / LPK, NL = D / 16;
        const size_t head0 = ((size_t) at.h << rb_sh) + hh * (D * 2);
#pragma clang loop unroll(disable)
        for (int k0 = t0 << tk_sh; k0 < end; k0 += KPL * NL) {
            uint64_t odd[NL];
            size_t row0[NL];                                    // of each load's first key (all in a page)
            lk_u16x8 u8[NL];
#pragma unroll
            for (int j = 0; j < NL; ++j) {
                const int k = k0 + KPL * j, page = lk_sld(at.row, (k < end ? k : k0) >> a.page_sh);
                const bool ok = k < end && page >= 0 && page < a.n_pages;
                row0[j] = (((size_t) (ok ? page : 0) << a.page_sh) + (k & m)) * row_bytes + head0;
                u8[j] = lk_u16x8{};
                if (ok) u8[j] = *(const lk_u16x8 *) (a.vp + row0[j] + (size_t) (lane / LPK) * row_bytes + 16 * (lane % LPK));
            }
            uint64_t any = 0;
#pragma unroll
            for (int j = 0; j < NL; ++j) {
                bool o = false;
#pragma unroll
                for (int e = 0; e < 8; ++e) o |= endless(u8[j][e]);
                odd[j] = __ballot(o);
                any |= odd[j];
            }
            if (any == 0) continue;                             // wave-uniform
#pragma unroll
            for (int j = 0; j < NL; ++j)
#pragma clang loop unroll(disable)
                while (odd[j]) {
                    const int f = __builtin_ctzll(odd[j]) / LPK, k = k0 + KPL * j + f;
                    odd[j] &= ~(((1ull << LPK) - 1) << (f * LPK));
                    if (k >= end) break;
                    const size_t at0 = row0[j] + (size_t) f * row_bytes;
                    bool none = false;                          // the key's score is -inf, if it is not +inf or NaN
                    if (!(a.cap > 0.0f)) {
                        const uint16_t * key = (const uint16_t *) (a.kp + at0);
#pragma unroll
                        for (int e = 0; e < D / 64; ++e) none |= endless(key[lane + 64 * e]);
                        none = __ballot(none) != 0;
                    }
                    const int d = k - base;
#pragma unroll
                    for (int db = 0; db < DB; ++db) {
                        const lk_u16x4 u = *(const lk_u16x4 *) (a.vp + at0 + 32 * db + 8 * g);
                        const V4 v = __builtin_bit_cast(V4, u);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            if (!endless(u[r])) continue;
#pragma unroll
                            for (int cb = 0; cb < CB; ++cb)
                                if (d < 0 || (d < 64 && ((see[cb] >> d) & 1))) {
                                    sum[cb][db][r] += none ? NAN : (float) v[r];
                                    found[cb] |= 1u << (4 * db + r);
                                }
                        }
                    }
                }
        }
        const bool whole = t0 == 0 && t1 == at.nt;
#pragma unroll
        for (int cb = 0; cb < CB; ++cb) {
            int i, row, head;
            if (!column(a, cb, i, row, head) || found[cb] == 0) continue;
            RowT * o = (RowT *) a.out + (size_t) row * a.ldo + (size_t) head * D + 4 * g;
            const size_t blk = (size_t) (2 * wgi + (t0 == 0)) * (CB << (a.qw_sh + a.hg_sh)) + ((hh << a.qw_sh) + qw) * CB + cb;
            if (!whole) {                                       // (lanes of a column write the same)
                float * const l = &a.ml[blk * 16 + col].y;
                *l = copysignf(*l, -1.0f);
            }
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (((found[cb] >> (4 * db + r)) & 1) == 0) continue;
                    if (whole) {                                // but for rows that the scores made NaN
                        const float was = (float) o[16 * db + r];
                        if (was == was || signbit(was)) o[16 * db + r] = (RowT) sum[cb][db][r];
                    } else {
                        a.acc[((blk * DB + db) * 64 + col * 4 + g) * 4 + r] = sum[cb][db][r];
                    }
                }
        }
        left -= t1 - t0 + extra;
        if (left > 0) lk_pa_next(a, at, tk_sh);
    }
}

// ---- joining cut items ------------------------------------------------------------------------
// A block of 16 columns of a cut item: where its output goes, and which of its columns are there.
struct LkPaBlock {
    int c0, hh, live;              // first column of the chunk, kv head of the group, columns
    __device__ __forceinline__ LkPaBlock(const LkPaArgs & a, const int4 & it, int blk, int cb_n) {
        const int cb = blk % cb_n, qw = (blk / cb_n) & ((1 << a.qw_sh) - 1);
        hh = (blk / cb_n) >> a.qw_sh;
        c0 = (qw * cb_n + cb) * 16;
        live = lk_clamp(it.z * a.g - c0, 0, 16);            // columns are (token, head) in order: the live ones come first
    }
    // value e of dims 16 db ..: column e / 4, its dims 4 (e % 4) ..
    template <int D, typename RowT>
    __device__ __forceinline__ void store(const LkPaArgs & a, const int4 & it, int db, int e, const lk_f4 & r, float l, float m) const {
        const int c = c0 + (e >> 2), t = c / a.g, head = ((it.w << a.hg_sh) + hh) * a.g + (c - t * a.g);
        const float il = lk_pa_inverse(l, m), v[4] = { r[0] * il, r[1] * il, r[2] * il, r[3] * il };
        lk_store<4>((RowT *) a.out + (size_t) (it.y + t) * a.ldo + (size_t) head * D + 16 * db + 4 * (e & 3), v);
    }
};

// Many items, cut into few pieces each: workgroup (x, blk) joins block blk of the item that begins in
// run x, each wave some of its dims.  A load of each piece is all it does: eight are asked for at once, so
// that their latencies overlap (in place of two: 16 sequences at up to 1000 18.0 -> 15.2 us as a whole, 19 at up
// to 5003 20.0 -> 17.9).  Of 2 x 4096 new tokens it takes 11.7 us for at most 64 MB, 5.5 TB/s.
template <int D, int RT>
__global__ void __launch_bounds__(256)
lk_k_paged_join(const LkPaArgs a, int cb_n) {
    constexpr int DB = D / 16, W = DB / 4;
    const int4 it = a.cut[blockIdx.x];
    if (it.x == 0) return;
    const int lane = threadIdx.x & 63, db0 = (threadIdx.x >> 6) * W;
    const int blk = blockIdx.y, nblk = gridDim.y;
    const LkPaBlock B(a, it, blk, cb_n);
    if (lane >= 4 * B.live) return;
    float m = -LK_PA_NONE, l = 0.0f, odd = 0.0f;               // odd: its sign, of the pieces so far
    lk_f4 o[W];
#pragma unroll
    for (int i = 0; i < W; ++i) o[i] = (lk_f4){ 0.f, 0.f, 0.f, 0.f };
    constexpr int NP = 8 / W;                                  // pieces asked for at once
    for (int k0 = 0; k0 < it.x; k0 += NP) {
        float2 ml[NP];
        lk_f4 x[NP][W];
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            ml[j] = make_float2(-LK_PA_NONE, 0.0f);
#pragma unroll
            for (int i = 0; i < W; ++i) x[j][i] = (lk_f4){ 0.f, 0.f, 0.f, 0.f };
            const int k = k0 + j;
            if (k < it.x) {                                    // the same for every thread
                const size_t p = (size_t) (2 * (blockIdx.x + k) + (k == 0)) * nblk + blk;
                ml[j] = a.ml[p * 16 + (lane >> 2)];
#pragma unroll
                for (int i = 0; i < W; ++i) x[j][i] = ((const lk_f4 *) a.acc)[(p * DB + db0 + i) * 64 + lane];
            }
        }
        float mx = m;
#pragma unroll
        for (int j = 0; j < NP; ++j) mx = fmaxf(mx, ml[j].x);
        const float f = lk_exp2(m - mx);
        m = mx;
        const float fo = lk_pa_factor(f, odd);
        l *= f;
#pragma unroll
        for (int i = 0; i < W; ++i) o[i] *= fo;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const float fj = lk_exp2(ml[j].x - mx);
            l = __builtin_fmaf(fabsf(ml[j].y), fj, l);
            const float fx = lk_pa_factor(fj, ml[j].y);
            odd = signbit(ml[j].y) ? ml[j].y : odd;
#pragma unroll
            for (int i = 0; i < W; ++i) o[i] += x[j][i] * fx;
        }
    }
#pragma unroll
    for (int i = 0; i < W; ++i) B.template store<D, typename LkElem<RT>::type>(a, it, db0 + i, lane, o[i], l, m);
}

// Few items, cut into many pieces: workgroup (x, y) joins 16 dims of a block of the cut items number x,
// x + gridDim.x, ..  All pieces' (max, sum) first give their weights; then the threads are divided over the
// block's live values and as many pieces at once as fit, and their sums are added in order.  Latency bounds it: the
// list of cut items, one round of loads, two barriers of the weights, three of the sums (256 pieces of one token,
// 32 heads of 64: 5.5 us).
template <int D, int RT>
__global__ void __launch_bounds__(1024)
lk_k_paged_spread(const LkPaArgs a, int cb_n, int wgs) {
    constexpr int DB = D / 16, NT = 1024, NV = NT / 64, MW = LK_PA_MAX_WGS / 64;
    __shared__ int4 s_item[LK_PA_MAX_WGS];
    __shared__ int s_from[LK_PA_MAX_WGS], s_count[MW];
    __shared__ float s_w[LK_PA_MAX_WGS][16], s_r[2][NV][16];
    __shared__ lk_f4 s_o[NT];
    const int tid = threadIdx.x, lane = tid & 63, v = __builtin_amdgcn_readfirstlane(tid >> 6);
    static_assert(NT >= LK_PA_MAX_WGS, "a thread for every workgroup's entry");
    // the items that are cut, in order
    int4 mine = make_int4(0, 0, 0, 0);
    if (tid < wgs) mine = a.cut[tid];
    const uint64_t has = __ballot(mine.x > 0);
    if (lane == 0 && v < MW) s_count[v] = __builtin_popcountll(has);
    __syncthreads();
    int n = 0, off = 0;
#pragma unroll
    for (int k = 0; k < MW; ++k) {
        if (k < v) off += s_count[k];
        n += s_count[k];
    }
    if (mine.x > 0) {
        off += __builtin_popcountll(has & ((1ull << lane) - 1));
        s_item[off] = mine;
        s_from[off] = tid;
    }
    __syncthreads();

    const int blk = blockIdx.y / DB, db = blockIdx.y % DB, nblk = gridDim.y / DB, col = tid & 15;
    for (int x = blockIdx.x; x < n; x += gridDim.x) {
        const int4 it = s_item[x];
        const int w0 = s_from[x];
        const LkPaBlock B(a, it, blk, cb_n);
        if (B.live == 0) continue;                             // the same for every thread
        auto piece = [&](int k) -> size_t { return (size_t) (2 * (w0 + k) + (k == 0)) * nblk + blk; };
        // all that is needed is asked for at once: the thread's (max, sum) pairs, and its rows of up to 8 pieces
        constexpr int NP = LK_PA_MAX_WGS * 16 / NT, NR = 8;
        const int e_sh = B.live > 8 ? 6 : B.live > 4 ? 5 : 4, e = tid & ((1 << e_sh) - 1), p0 = tid >> e_sh, pp = NT >> e_sh;
        auto rows = [&](int k) -> lk_f4 { return ((const lk_f4 *) a.acc)[(piece(k) * DB + db) * 64 + e]; };
        float2 ml[NP];
        lk_f4 x4[NR];
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int k = (tid >> 4) + j * (NT / 16);
            ml[j] = make_float2(-LK_PA_NONE, 0.0f);
            if (k < it.x && col < B.live) ml[j] = a.ml[piece(k) * 16 + col];
        }
#pragma unroll
        for (int j = 0; j < NR; ++j) {
            x4[j] = (lk_f4){ 0.f, 0.f, 0.f, 0.f };
            if (p0 + j * pp < it.x && e < 4 * B.live) x4[j] = rows(p0 + j * pp);
        }
        float m = -LK_PA_NONE, l = 0.0f;
#pragma unroll
        for (int j = 0; j < NP; ++j) m = fmaxf(m, ml[j].x);
        m = lk_xrow_max(m);
        if (lane < 16) s_r[0][v][col] = m;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NV; ++k) m = fmaxf(m, s_r[0][k][col]);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int k = (tid >> 4) + j * (NT / 16);
            const float f = lk_exp2(ml[j].x - m);
            if (k < it.x) s_w[k][col] = lk_pa_factor(f, ml[j].y);
            l = __builtin_fmaf(fabsf(ml[j].y), f, l);
        }
        l = lk_xrow_sum(l);
        if (lane < 16) s_r[1][v][col] = l;
        __syncthreads();
        lk_f4 o = { 0.f, 0.f, 0.f, 0.f };
        if (e < 4 * B.live) {
#pragma unroll
            for (int j = 0; j < NR; ++j)
                if (p0 + j * pp < it.x) o += x4[j] * s_w[p0 + j * pp][e >> 2];
#pragma unroll 8
            for (int k = p0 + NR * pp; k < it.x; k += pp) o += rows(k) * s_w[k][e >> 2];
        }
        s_o[tid] = o;
        __syncthreads();
        // eight threads' sums at a time, then those
        if ((tid >> e_sh) % 8 == 0) {
            lk_f4 r = s_o[tid];
#pragma unroll
            for (int k = 1; k < 8; ++k) r += s_o[tid + (k << e_sh)];
            s_o[tid] = r;
        }
        __syncthreads();
        if (tid < 4 * B.live) {
            lk_f4 r = s_o[tid];
            for (int k = 8; k < pp; k += 8) r += s_o[(k << e_sh) + tid];
            float sum = 0.0f, mx = -LK_PA_NONE;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                sum += s_r[1][k][tid >> 2];
                mx = fmaxf(mx, s_r[0][k][tid >> 2]);
            }
            B.template store<D, typename LkElem<RT>::type>(a, it, db, tid, r, sum, mx);
        }
        __syncthreads();
    }
}

// ---- host ---------------------------------------------------------------------------------------
// How a workgroup's waves divide a tile, for chunks of `want` tokens of g query heads a kv head.
struct LkPaShape { int cb, step, hg_sh, qw_sh, kw_sh, qc, extra; };
// Column blocks a wave of the STEP 32 kernels holds, its columns being spread over up to four waves first: with
// more than one chunk a sequence (max_new above 64) as many as the registers take, so that a tile is read from
// LDS once for all of them; for up to 64 rows, whose items are cut into many pieces, one or two, since what a
// workgroup leaves behind grows with its columns; one for chunks of four blocks in all until there are enough
// of them to go round.  Measured, us, 32 / 8 heads of 64 (1, 2, 4 blocks):
//   one tree of 16 at 2000      13.1  16.0  21.1     four of 24 at 2000            17.6  20.0  23.9
//   one of 16 at 32768          27.2  30.1  35.8     one of 64 at 8000             27.0  28.5  42.4
//   one of 16 at 131072         62.9  63.9  68.4     13 of up to 64 at 4096        57.7  51.9  57.9
//   2 x 4096 new tokens          390   308   271     one of 64 at 131072            191   161   156
//   8 x up to 512 new tokens    43.0  36.4  38.2     5 x up to 500 behind 500      55.0  46.7  58.8
// (the last two have few chunks, which this rule does not see); fp32 rows 13 trees 63.6, 56.2, 2 x 4096 new tokens
// 452, 346; heads of 128, bf16, 13 trees 90.8, 73.9, a prompt of 4096 415, 273; 16 / 16 heads of 64 5 x 500 behind 500
// 36.3, 36.8, 42.1; 2 x 4096 behind 4096 433, 408, 404.
constexpr int lk_pa_cb32(int d, int type, int max_new, int nb) {
    return (nb <= 4 && max_new < 1024) || (d == 128 && type == LK_F32) ? 1 : d == 64 && type != LK_F32 && max_new > 64 ? 4 : 2;
}
static LkPaShape lk_pa_shape(const lk_pages * p, int type, int max_new) {
    const int g = p->n_heads / p->n_kv_heads, d = p->head_dim;
    const int want = max_new < 1 ? 1 : max_new > 64 ? 64 : max_new;
    LkPaShape s;
    const int nb = (want * g + 15) / 16;                       // blocks of columns
    s.step = nb > 1 ? 32 : 16;
    s.cb = nb > 1 ? lk_pa_cb32(d, type, max_new, nb) : 1;
    const int nw = lk_pa_waves(d, s.step);
    s.qw_sh = s.step == 32 && d == 128 ? 1 : 0;                // (a wave's share of a tile is 16 * 2^qw_sh keys and more)
    while ((s.cb << s.qw_sh) < nb && (1 << s.qw_sh) < nw) ++s.qw_sh;
    const int qw = 1 << s.qw_sh;
    s.hg_sh = 0;
    // few heads a group where the columns are many: what a cut item leaves behind is 16 KB a wave and more
    while ((2 << s.hg_sh) * qw <= nw && p->n_kv_heads % (2 << s.hg_sh) == 0 && (s.step == 16 || s.hg_sh < 1)) ++s.hg_sh;
    s.kw_sh = lk_log2(nw / qw) - s.hg_sh;
    int qc = s.cb * 16 * qw / g;
    if (qc > 64) qc = 64;
    if (qc < 1) qc = 1;
    s.qc = 1 << lk_log2(qc);
    s.extra = s.step == 32 ? 5 : 2;
    return s;
}
static int lk_pa_blocks(const LkPaShape & s) { return s.cb << (s.qw_sh + s.hg_sh); }

template <int D, int RT, int CT, int CB, int STEP>
static void lk_pa_run(const LkPaArgs & a, bool mod, hipStream_t st) {
    const dim3 grid(lk_pa_wgs(STEP)), block(64 * lk_pa_waves(D, STEP));
    if (mod) hipLaunchKernelGGL((lk_k_paged_attn<D, RT, CT, CB, STEP, true>), grid, block, 0, st, a);
    else     hipLaunchKernelGGL((lk_k_paged_attn<D, RT, CT, CB, STEP, false>), grid, block, 0, st, a);
}
template <int D, int RT, int CT>
static void lk_pa_launch(const LkPaShape & s, const LkPaArgs & a, bool mod, hipStream_t st) {
    if (s.step == 32) {
        if (s.cb == 1) lk_pa_run<D, RT, CT, 1, 32>(a, mod, st);
        if constexpr (D == 64 || RT != LK_F32) {
            if (s.cb == 2) lk_pa_run<D, RT, CT, 2, 32>(a, mod, st);
        }
        if constexpr (D == 64 && RT != LK_F32) {
            if (s.cb == 4) lk_pa_run<D, RT, CT, 4, 32>(a, mod, st);
        }
        return;
    }
    lk_pa_run<D, RT, CT, 1, 16>(a, mod, st);
}

template <int D, int RT>
static void lk_pa_join(const LkPaArgs & a, long items, int nblk, const LkPaShape & s, hipStream_t st) {
    // attention and its join, us, spread and join: one token at 131072 50, 86; one at 4096 13.1, 33; a tree of 16
    // at 32768 27.1, 30.6; 16 of up to 1000 23.2, 15.4; 64 of up to 8192 293, 231; 13 trees of up to 64 123, 51
    const int wgs = lk_pa_wgs(s.step);
    if (items <= wgs / 32)
        hipLaunchKernelGGL((lk_k_paged_spread<D, RT>), dim3((unsigned) items, nblk * (D / 16)), dim3(1024), 0, st, a, s.cb, wgs);
    else
        hipLaunchKernelGGL((lk_k_paged_join<D, RT>), dim3(wgs - 1, nblk), dim3(256), 0, st, a, s.cb);
}

extern "C" size_t lk_paged_attn_work_bytes(const lk_pages * pages, int type, int max_new) {
    static const char * const W = "lk_paged_attn_work_bytes";
    if (lk_paged_check_pages(W, pages) || lk_paged_check_type(W, pages, type)) return 0;
    if (max_new < 0) {
        lk_fail(hipErrorInvalidValue, "%s: max_new %d", W, max_new);
        return 0;
    }
    const LkPaShape s = lk_pa_shape(pages, type, max_new);
    const size_t blocks = (size_t) 2 * lk_pa_wgs(s.step) * lk_pa_blocks(s);
    return blocks * (16 * pages->head_dim * 4 + 16 * 8) + lk_pa_wgs(s.step) * 16;
}

extern "C" int lk_paged_attn(const lk_pages * pages, const lk_step * step, int type, const void * q, int ldq, float scale, float cap,
                             const float * slopes, void * out, int ldo, void * work, size_t work_bytes, void * stream) {
    static const char * const W = "lk_paged_attn";
    if (const int e = lk_paged_check(W, pages, step)) return e;
    if (const int e = lk_paged_check_type(W, pages, type)) return e;
    const int d = pages->head_dim, hq = pages->n_heads;
    if (!(scale > 0.0f) || !(scale < __builtin_inff()) || !(cap == 0.0f || cap >= 0x1p-100f) ||
        !(cap < __builtin_inff()))
        return lk_fail(hipErrorInvalidValue, "%s: scale %g, cap %g (0: none)", W, (double) scale, (double) cap);
    if (step->rows == 0 || step->n_seqs == 0) return 0;
    if (!q || !out || !work) return lk_fail(hipErrorInvalidValue, "%s: null pointer argument", W);
    if (ldq < hq * d || ldo < hq * d)
        return lk_fail(hipErrorInvalidValue, "%s: row strides q %d, out %d for %d heads of %d", W, ldq, ldo, hq, d);
    if (q == out && ldq != ldo && step->rows > 1)
        return lk_fail(hipErrorInvalidValue, "%s: output over queries %d apart in rows %d apart", W, ldq, ldo);
    const uintptr_t em = (uintptr_t) lk_type_size(type) - 1;
    if ((((uintptr_t) q | (uintptr_t) out) & em) || ((uintptr_t) slopes & 3) || ((uintptr_t) work & 15))
        return lk_fail(hipErrorInvalidValue, "%s: misaligned argument (rows by their element, slopes 4 B, work 16 B)", W);
    // max_new 0: the mean, where the workspace has room for its kernel (a prompt of 4096: 190 us, as single tokens 798)
    int most = step->max_new;
    if (most == 0) {
        most = (step->rows - 1) / step->n_seqs + 1;
        if (work_bytes < lk_paged_attn_work_bytes(pages, type, most)) most = 1;
    }
    const size_t need = lk_paged_attn_work_bytes(pages, type, most);
    if (work_bytes < need) return lk_fail(hipErrorInvalidValue, "%s: workspace of %zu bytes, %zu needed", W, work_bytes, need);
    const LkPaShape s = lk_pa_shape(pages, type, most);
    const int nblk = lk_pa_blocks(s), g = hq / pages->n_kv_heads, nhg = pages->n_kv_heads >> s.hg_sh;
    const size_t blocks = (size_t) 2 * lk_pa_wgs(s.step) * nblk;
    float * acc = (float *) work;
    float2 * ml = (float2 *) (acc + blocks * 16 * d);
    const LkPaArgs a = { q, out, (const char *) pages->k, (const char *) pages->v, step->first, step->lens, step->table, step->pos,
                         step->mask, slopes, acc, ml, (int4 *) (ml + blocks * 16), ldq, ldo, step->n_seqs, step->rows, step->ldt,
                         step->width, lk_log2(pages->page), pages->n_pages, pages->n_kv_heads, g, nhg, s.hg_sh, s.qw_sh, s.kw_sh, s.qc, s.extra,
                         scale * LK_LOG2E_F, scale, cap, 1.0f / cap };
    const hipStream_t st = lk_stream(stream);
    const bool mod = cap > 0.0f || slopes;
    if (d == 64) {
        if (type == LK_F32)      lk_pa_launch<64, LK_F32, LK_F16>(s, a, mod, st);
        else if (type == LK_F16) lk_pa_launch<64, LK_F16, LK_F16>(s, a, mod, st);
        else                     lk_pa_launch<64, LK_BF16, LK_BF16>(s, a, mod, st);
    } else {
        if (type == LK_F32)      lk_pa_launch<128, LK_F32, LK_F16>(s, a, mod, st);
        else if (type == LK_F16) lk_pa_launch<128, LK_F16, LK_F16>(s, a, mod, st);
        else                     lk_pa_launch<128, LK_BF16, LK_BF16>(s, a, mod, st);
    }
    if (const int e = lk_launch_status(W)) return e;
    const long items = ((long) step->rows / s.qc + step->n_seqs) * nhg;       // at most
    if (d == 64) {
        if (type == LK_F32)      lk_pa_join<64, LK_F32>(a, items, nblk, s, st);
        else if (type == LK_F16) lk_pa_join<64, LK_F16>(a, items, nblk, s, st);
        else                     lk_pa_join<64, LK_BF16>(a, items, nblk, s, st);
    } else {
        if (type == LK_F32)      lk_pa_join<128, LK_F32>(a, items, nblk, s, st);
        else if (type == LK_F16) lk_pa_join<128, LK_F16>(a, items, nblk, s, st);
        else                     lk_pa_join<128, LK_BF16>(a, items, nblk, s, st);
    }
    return lk_launch_status(W);
}

// paged.hip - what writes a paged cache: the append of a step's keys and values with the
// head norms and the rotation (lk_paged_append), and the commit of accepted drafts
// (lk_paged_commit).
//
// Append, per row t (token i of sequence b, slot lens[b] + i) and head row x of D values:
//     y = x * inv * w,  inv = 1 / sqrt(sum x^2 / D + eps)                  (fp32)
//     a_i = position * freq_i                                             (fp64, exact below position 2^29)
//     (u, v) -> (u cos a - v sin a, u sin a + v cos a)                     (fp32; cos and sin fp64, rounded once)
// q to its rows, k and v to the slot's page, each rounded once.  An angle in fp32 would be
// off by 2^-24 of itself: 0.008 at position 131072, far above the rounding of 16-bit rows.
#include "lk_paged.h"

int lk_paged_check_pages(const char * what, const lk_pages * p) {
    if (!p) return lk_fail(hipErrorInvalidValue, "%s: pages is null", what);
    if (p->type != LK_F16 && p->type != LK_BF16)
        return lk_fail(hipErrorInvalidValue, "%s: pools of type %d (fp16 or bf16)", what, p->type);
    if (p->head_dim != 64 && p->head_dim != 128)
        return lk_fail(hipErrorInvalidValue, "%s: head_dim %d (64 or 128)", what, p->head_dim);
    if (p->n_kv_heads < 1 || p->n_heads < p->n_kv_heads || p->n_heads > LK_PAGED_MAX_HEADS ||
        p->n_heads % p->n_kv_heads != 0 || p->n_heads / p->n_kv_heads > LK_PAGED_MAX_GROUP)
        return lk_fail(hipErrorInvalidValue, "%s: %d heads over %d kv heads (a multiple, up to %d, up to %d a kv head)", what,
                       p->n_heads, p->n_kv_heads, LK_PAGED_MAX_HEADS, LK_PAGED_MAX_GROUP);
    if (p->page < 16 || p->page > 65536 || (p->page & (p->page - 1)))
        return lk_fail(hipErrorInvalidValue, "%s: %d positions a page (a power of two, 16 .. 65536)", what, p->page);
    return 0;
}

int lk_paged_check_type(const char * what, const lk_pages * p, int type) {
    if (!lk_type_ok(type) || (type == LK_BF16) != (p->type == LK_BF16))
        return lk_fail(hipErrorInvalidValue, "%s: rows of type %d with pools of type %d (fp32 or fp16 with fp16, bf16 with bf16)",
                       what, type, p->type);
    return 0;
}

int lk_paged_check(const char * what, const lk_pages * p, const lk_step * s) {
    if (const int e = lk_paged_check_pages(what, p)) return e;
    if (p->n_pages < 1 || !p->k || !p->v || (((uintptr_t) p->k | (uintptr_t) p->v) & 15))
        return lk_fail(hipErrorInvalidValue, "%s: pools of %d pages, null or not 16-byte aligned", what, p->n_pages);
    if (!s) return lk_fail(hipErrorInvalidValue, "%s: step is null", what);
    if (s->n_seqs < 0 || s->rows < 0 || s->max_new < 0)
        return lk_fail(hipErrorInvalidValue, "%s: %d sequences, %d rows, max_new %d", what, s->n_seqs, s->rows, s->max_new);
    // every sequence and row is a workgroup or a part of one; a count times any width used stays in an int
    if (s->n_seqs > (1 << 20) || s->rows > (1 << 24))
        return lk_fail(hipErrorInvalidValue, "%s: %d sequences (up to 2^20), %d rows (up to 2^24)", what, s->n_seqs, s->rows);
    if (s->width < 1 || s->ldt < s->width || (long) s->width * p->page > LK_PAGED_MAX_SLOTS)
        return lk_fail(hipErrorInvalidValue, "%s: a table of %d pages a sequence (1 .. %d of %d positions), %d apart", what, s->width,
                       LK_PAGED_MAX_SLOTS / p->page, p->page, s->ldt);
    if (s->n_seqs == 0) return 0;
    if (!s->first || !s->lens || !s->table)
        return lk_fail(hipErrorInvalidValue, "%s: null pointer in step", what);
    if ((((uintptr_t) s->first | (uintptr_t) s->lens | (uintptr_t) s->table | (uintptr_t) s->pos) & 3) || ((uintptr_t) s->mask & 7))
        return lk_fail(hipErrorInvalidValue, "%s: misaligned table (first, lens, table, pos 4 B, mask 8 B)", what);
    return 0;
}

// ---- append -----------------------------------------------------------------------
struct LkAppendArgs {
    const void * q, * k, * v;
    const float * qn, * kn, * freq;
    void * qo;
    char * kp, * vp;
    const int32_t * first, * lens, * table, * pos;
    int ldq, ldk, ldv, ldqo, n_seqs, rows, ldt, width, page_sh, n_pages, hq, hkv, rot, pairs;
    float eps;
};

// 1 / sqrt(a): the hardware's estimate (1 ulp) and one step of Newton's method on it.
// (fp64 square root and division instead cost as much time as the rows' traffic.)
__device__ __forceinline__ float lk_rsqrt(float a) {
#if defined(__HIP_DEVICE_COMPILE__)
    const float r = __builtin_amdgcn_rsqf(a);
#else
    const float r = 1.0f / sqrtf(a);
#endif
    const float e = __builtin_fmaf(-a * r, r, 1.0f);
    return __builtin_fmaf(r * 0.5f, e, r);
}

// Sum over the 4 or 8 lanes of a head row.
template <int LPH>
__device__ __forceinline__ float lk_head_sum(float v) {
    v += lk_dpp<LK_DPP_QP_XOR1>(v);
    v += lk_dpp<LK_DPP_QP_XOR2>(v);
    if constexpr (LPH == 8) v += lk_dpp<LK_DPP_HMIRROR>(v);
    return v;
}

// A workgroup has R rows and (of grid.y parts) a share of their head rows (q, k, then v heads),
// LPH lanes a head row.  A lane holds the two runs of eight values that the rotation pairs: 8j and
// rot/2 + 8j with halves, 16j and 16j + 8 with pairs or behind `rot`, so that nothing is exchanged between
// lanes.  The rows are asked for first; meanwhile the lanes look for the rows' sequences, all of
// `first` at once, and one lane an angle forms the sines and cosines.
// Bound by latency for few rows (three loads one behind the other: bounds, page, and the launch; one row of
// 32 + 8 + 8 heads of 64 in fp32 3.2 us in a graph) and by memory for many: 8192 rows of fp16 19.6 us, 4.3 TB/s,
// next to 5.15 of a large copy.  Eight values a run: with four (twice the lanes, loads of 8 bytes) the
// instructions bound it, 23.8 us.
#define LK_APPEND_ROWS 2           // per workgroup, where there are many; 1: 21.1 us, 4: 20.7 us
template <int TYPE, int CTYPE, int LPH, int R>
__global__ void __launch_bounds__(512)
lk_k_paged_append(const LkAppendArgs a) {
    typedef typename LkElem<TYPE>::type T;
    typedef typename LkElem<CTYPE>::type C;
    constexpr int D = LPH * 16;
    __shared__ __attribute__((aligned(16))) float s_c[R][D / 2], s_s[R][D / 2];
    __shared__ unsigned long long s_seq[R];
    const int t0 = blockIdx.x * R, tid = threadIdx.x;
    const int unit = blockIdx.y * blockDim.x + tid;
    const int head = unit / LPH, j = unit % LPH;
    const int nq = a.q ? a.hq : 0;
    const bool isq = head < nq, isk = !isq && head < nq + a.hkv, isv = !isq && !isk && head < nq + 2 * a.hkv;
    const int hh = isq ? head : isk ? head - nq : isv ? head - nq - a.hkv : 0;
    const bool split = !a.pairs && 16 * j < a.rot && !isv;
    const int lo = split ? 8 * j : 16 * j, hi = split ? a.rot / 2 + 8 * j : 16 * j + 8;

    const T * src = (const T *) (isq ? a.q : isk ? a.k : a.v) + hh * D;
    const size_t ld = isq ? a.ldq : isk ? a.ldk : a.ldv;
    const float * w = isq ? a.qn : isk ? a.kn : nullptr;
    float x0[R][8], x1[R][8], w0[8], w1[8];
    if (isq | isk | isv) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int t = t0 + r < a.rows ? t0 + r : a.rows - 1;
            lk_load<8>(src + t * ld + lo, x0[r]);
            lk_load<8>(src + t * ld + hi, x1[r]);
        }
        if (w) {
            lk_load<8>(w + lo, w0);
            lk_load<8>(w + hi, w1);
        }
    }
    // the rows' sequences (of those that name a row the first) and slots
    const int slots = a.width << a.page_sh;
    if (tid < R) s_seq[tid] = ~0ull;
    __syncthreads();
    for (int b = tid; b < a.n_seqs; b += blockDim.x) {
        const LkSeq s = lk_seq(a.first[b], a.first[b + 1], a.lens[b], a.rows, slots);
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int i = t0 + r - s.r0;
            if (i >= 0 && i < s.n) atomicMin(&s_seq[r], (unsigned long long) b << 32 | (unsigned) (s.len + i));
        }
    }
    __syncthreads();
    int page[R], slot[R];                                     // page -2: padding, nothing is written
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const unsigned b = __builtin_amdgcn_readfirstlane((int) (s_seq[r] >> 32));
        slot[r] = b == ~0u ? 0 : __builtin_amdgcn_readfirstlane((int) s_seq[r]);
        page[r] = a.table[(size_t) (b == ~0u ? 0 : b) * a.ldt + ((slot[r] < slots ? slot[r] : 0) >> a.page_sh)];
        page[r] = b == ~0u ? -2 : slot[r] < slots && page[r] >= 0 ? page[r] : -1;
    }
    for (int i = tid; i < R * (a.rot / 2); i += blockDim.x) {
        const int r = i / (a.rot / 2), k = i - r * (a.rot / 2);
        int pos = 0;
#pragma unroll
        for (int u = 0; u < R; ++u) pos = u == r ? slot[u] : pos;
        if (a.pos && t0 + r < a.rows) pos = a.pos[t0 + r];
        double sn, cs;
        lk_sincos((double) pos * (double) a.freq[k], sn, cs);
        s_c[r][k] = (float) cs;
        s_s[r][k] = (float) sn;
    }
    __syncthreads();
    if (!(isq | isk | isv)) return;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        if (page[r] == -2) continue;
        float (&y0)[8] = x0[r], (&y1)[8] = x1[r];
        if (w) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(y0[i], y0[i], ss);
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(y1[i], y1[i], ss);
            ss = lk_head_sum<LPH>(ss);
            const float inv = lk_rsqrt(__builtin_fmaf(ss, 1.0f / D, a.eps));
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                y0[i] = y0[i] * inv * w0[i];
                y1[i] = y1[i] * inv * w1[i];
            }
        }
        if (!isv && 16 * j < a.rot) {
            float c[8], sn[8];
            lk_load<8>(s_c[r] + 8 * j, c);
            lk_load<8>(s_s[r] + 8 * j, sn);
            auto turn = [&](float & u, float & v, int i) {
                const float p = u;
                u = p * c[i] - v * sn[i];
                v = p * sn[i] + v * c[i];
            };
            if (split) {
#pragma unroll
                for (int i = 0; i < 8; ++i) turn(y0[i], y1[i], i);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    turn(y0[2 * i], y0[2 * i + 1], i);
                    turn(y1[2 * i], y1[2 * i + 1], 4 + i);
                }
            }
        }
        if (isq) {
            T * o = (T *) a.qo + (size_t) (t0 + r) * a.ldqo + hh * D;
            lk_store<8>(o + lo, y0);
            lk_store<8>(o + hi, y1);
        } else if (page[r] >= 0 && page[r] < a.n_pages) {
            const size_t at = ((size_t) page[r] << a.page_sh) + (slot[r] & ((1 << a.page_sh) - 1));
            C * o = (C *) (isk ? a.kp : a.vp) + (at * a.hkv + hh) * D;
            lk_store<8>(o + lo, y0);
            lk_store<8>(o + hi, y1);
        }
    }
}

template <int TYPE, int CTYPE, int LPH>
static void lk_append_launch(const LkAppendArgs & a, hipStream_t st) {
    const int units = ((a.q ? a.hq : 0) + 2 * a.hkv) * LPH;
    const int ny = (units + 511) / 512, nt = ((units + ny - 1) / ny + 63) / 64 * 64;    // whole head rows a workgroup
    // several rows a workgroup where that still fills the GPU
    if ((long) a.rows * ny >= 2048)
        hipLaunchKernelGGL((lk_k_paged_append<TYPE, CTYPE, LPH, LK_APPEND_ROWS>), dim3((a.rows - 1) / LK_APPEND_ROWS + 1, ny), dim3(nt), 0, st, a);
    else
        hipLaunchKernelGGL((lk_k_paged_append<TYPE, CTYPE, LPH, 1>), dim3(a.rows, ny), dim3(nt), 0, st, a);
}
template <int TYPE, int CTYPE>
static void lk_append_launch(const LkAppendArgs & a, int d, hipStream_t st) {
    if (d == 64) lk_append_launch<TYPE, CTYPE, 4>(a, st);
    else         lk_append_launch<TYPE, CTYPE, 8>(a, st);
}

extern "C" int lk_paged_append(const lk_pages * pages, const lk_step * step, int type, const void * q, int ldq, const void * k,
                               int ldk, const void * v, int ldv, const float * qn, const float * kn, float eps,
                               const float * freq, int rot, int style, void * qo, int ldqo, void * stream) {
    static const char * const W = "lk_paged_append";
    if (const int e = lk_paged_check(W, pages, step)) return e;
    if (const int e = lk_paged_check_type(W, pages, type)) return e;
    const int d = pages->head_dim, hq = pages->n_heads, hkv = pages->n_kv_heads;
    if (style != LK_ROPE_HALVES && style != LK_ROPE_PAIRS) return lk_fail(hipErrorInvalidValue, "%s: style %d", W, style);
    if (rot < 0 || rot > d || rot % 16 != 0 || (rot > 0) != (freq != nullptr))
        return lk_fail(hipErrorInvalidValue, "%s: rot %d (a multiple of 16 up to %d; 0 without freq)", W, rot, d);
    if (!(eps >= 0.0f)) return lk_fail(hipErrorInvalidValue, "%s: eps %g", W, (double) eps);
    if (step->rows == 0 || step->n_seqs == 0) return 0;
    if (!k || !v || (q != nullptr) != (qo != nullptr))
        return lk_fail(hipErrorInvalidValue, "%s: null pointer argument (k and v; q and qo both or neither)", W);
    if ((q && (ldq < hq * d || ldqo < hq * d)) || ldk < hkv * d || ldv < hkv * d)
        return lk_fail(hipErrorInvalidValue, "%s: row strides q %d, k %d, v %d, qo %d for %d and %d heads of %d", W, ldq, ldk, ldv, ldqo,
                       hq, hkv, d);
    if (q && q == qo && ldq != ldqo && step->rows > 1)
        return lk_fail(hipErrorInvalidValue, "%s: output over queries %d apart in rows %d apart", W, ldq, ldqo);
    const uintptr_t em = (uintptr_t) lk_type_size(type) - 1;
    if ((((uintptr_t) q | (uintptr_t) k | (uintptr_t) v | (uintptr_t) qo) & em) ||
        (((uintptr_t) qn | (uintptr_t) kn | (uintptr_t) freq) & 15))
        return lk_fail(hipErrorInvalidValue, "%s: misaligned argument (rows by their element; qn, kn, freq 16 B)", W);
    const LkAppendArgs a = { q, k, v, qn, kn, freq, qo, (char *) pages->k, (char *) pages->v, step->first, step->lens, step->table,
                             step->pos, ldq, ldk, ldv, ldqo, step->n_seqs, step->rows, step->ldt, step->width, lk_log2(pages->page),
                             pages->n_pages, hq, hkv, rot, style == LK_ROPE_PAIRS, eps };
    const hipStream_t st = lk_stream(stream);
    if (type == LK_F32)      lk_append_launch<LK_F32, LK_F16>(a, d, st);
    else if (type == LK_F16) lk_append_launch<LK_F16, LK_F16>(a, d, st);
    else                     lk_append_launch<LK_BF16, LK_BF16>(a, d, st);
    return lk_launch_status(W);
}

// ---- commit -----------------------------------------------------------------------
struct LkCommitArgs {
    char * kp, * vp;
    const int32_t * first, * lens, * table, * path, * count;
    int32_t * new_lens;
    int n_seqs, rows, ldt, width, page_sh, n_pages, ldp, row16;      // row16: 16-byte pieces of a position's row
};

// One workgroup a sequence (so that new_lens may be lens).  The first wave checks the list and
// leaves the rows' places in LDS; then every thread has one 16-byte column of the K or V rows
// and moves it in order: the list is strictly increasing, so path[j] >= j, and a place is written
// only after it was read (the loads of eight rows go out before their stores).
// Bound by latency, three loads one behind the other: lengths and list, pages, rows (a launch in a kernel trace:
// one sequence 3.0 us, 128 of up to 64 drafted tokens and 3.2 MB 4.0).
__global__ void __launch_bounds__(1024)
lk_k_paged_commit(const LkCommitArgs a) {
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    __shared__ long s_src[LK_PAGED_MAX_PATH], s_dst[LK_PAGED_MAX_PATH];
    __shared__ int s_n;
    const int b = blockIdx.x, tid = threadIdx.x;
    if (tid < 64) {
        const int cap = a.width << a.page_sh;
        const LkSeq s = lk_seq(a.first[b], a.first[b + 1], a.lens[b], a.rows, cap);
        const int most = s.n < cap - s.len ? s.n : cap - s.len;         // new tokens that have a slot
        int n = lk_clamp(a.count[b], 0, a.path ? a.ldp : most);
        if (a.path) {
            const int p = tid < n ? a.path[(size_t) b * a.ldp + tid] : -1;
            int before = __shfl_up(p, 1, 64);
            if (tid == 0) before = -1;
            const int32_t * row = a.table + (size_t) b * a.ldt;
            bool ok = tid < n && p > before && p < most;
            long src = 0, dst = 0;
            if (ok) {
                const int ss = s.len + p, sd = s.len + tid;
                const int ps = row[ss >> a.page_sh], pd = row[sd >> a.page_sh], m = (1 << a.page_sh) - 1;
                ok = ps >= 0 && ps < a.n_pages && pd >= 0 && pd < a.n_pages;
                src = ((long) ps << a.page_sh) + (ss & m);
                dst = ((long) pd << a.page_sh) + (sd & m);
            }
            const uint64_t bad = ~__ballot(ok);
            n = bad ? __builtin_ctzll(bad) : 64;                // the places before the first that is not in order
            s_src[tid] = src;
            s_dst[tid] = dst;
        }
        if (tid == 0) {
            s_n = n;
            a.new_lens[b] = s.len + n;
        }
    }
    if (!a.path) return;
    __syncthreads();
    const int n = s_n;
    for (int c = tid; c < 2 * a.row16; c += blockDim.x) {
        u4 * base = (u4 *) (c < a.row16 ? a.kp : a.vp) + (c < a.row16 ? c : c - a.row16);
        for (int j0 = 0; j0 < n; j0 += 8) {
            u4 v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (j0 + i < n && s_src[j0 + i] != s_dst[j0 + i]) v[i] = base[s_src[j0 + i] * a.row16];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (j0 + i < n && s_src[j0 + i] != s_dst[j0 + i]) base[s_dst[j0 + i] * a.row16] = v[i];
        }
    }
}

extern "C" int lk_paged_commit(const lk_pages * pages, const lk_step * step, const int32_t * path, int ldp, const int32_t * count,
                               int32_t * new_lens, void * stream) {
    static const char * const W = "lk_paged_commit";
    if (const int e = lk_paged_check(W, pages, step)) return e;
    if (path && (ldp < 1 || ldp > LK_PAGED_MAX_PATH))
        return lk_fail(hipErrorInvalidValue, "%s: lists of %d (1 .. %d)", W, ldp, LK_PAGED_MAX_PATH);
    if (step->n_seqs == 0) return 0;
    if (!count || !new_lens) return lk_fail(hipErrorInvalidValue, "%s: null pointer argument", W);
    if (((uintptr_t) path | (uintptr_t) count | (uintptr_t) new_lens) & 3)
        return lk_fail(hipErrorInvalidValue, "%s: misaligned argument (path, count, new_lens 4 B)", W);
    const int row16 = pages->n_kv_heads * pages->head_dim / 8;
    const LkCommitArgs a = { (char *) pages->k, (char *) pages->v, step->first, step->lens, step->table, path, count, new_lens,
                             step->n_seqs, step->rows, step->ldt, step->width, lk_log2(pages->page), pages->n_pages, ldp, row16 };
    const int nt = !path ? 64 : 2 * row16 < 1024 ? (2 * row16 + 63) / 64 * 64 : 1024;
    hipLaunchKernelGGL(lk_k_paged_commit, dim3(step->n_seqs), dim3(nt), 0, lk_stream(stream), a);
    return lk_launch_status(W);
}

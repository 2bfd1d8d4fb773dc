/*
 * kq_linattn_chunk.hip — linear attention with a decay for each head on
 * gfx950, the chunked form (include/kq_hip.h, kq_hip_linear_attention_f32).
 *
 * For the 64 rows of a chunk that starts from the state S, with log decays
 * summed from its start G_i (inclusive), rows of k, q, v as matrices, norms
 * taken out of the rows of k = n k', the e_i = n_i d_i of the recurrent form
 * solve
 *   (1 + L) E = diag(b) (diag(n) V - diag(n^2 e^G) K' S),
 *                                     L_ij = b_i n_i^2 e^(G_i - G_j) k'_i.k'_j  (j < i)
 * so that with T = (1 + L)^-1 diag(b), B = T diag(n), W = T diag(n^2 e^G) K'
 *   E = B V - W S
 *   O = diag(e^G) Q S + M E,          M_ij = e^(G_i - G_j) q_i.k'_j      (j <= i)
 *   S' = e^(G_64) S + sum_j e^(G_64 - G_j) k'_j e_j^T
 * and what hangs on the chunk before is four products with S and E. e^(G_64)
 * is kept as kq::Decay has it: rounded to 32 bits it would be off the same way
 * chunk after chunk, 8e-6 of a state after 256 of them.
 * Without the delta correction E = diag(n) V.
 *
 * Three launches:
 *   linattn_rows  the recurrent form over the short sequences, which also cuts
 *                 the others into chunks (on the device: the lengths are there;
 *                 not for a call's only sequence)
 *   linattn_prep  a workgroup for each chunk and key head: Q, K'^T as operands
 *                 of the matrix cores, and for each of its value heads M, W, B
 *   linattn_scan  a workgroup for each sequence, head and 32 columns of v:
 *                 S in registers from the first chunk to the last; without the
 *                 delta correction and with few such workgroups three launches
 *                 over all chunks instead (linattn_sums, _states, _outs)
 *
 * A lane's eight values of an operand's long axis are 4 g .. 4 g + 3 of one 16
 * and the same four of the next (g = lane / 16), for both sides of a product:
 * these are the rows that a lane holds of two results, so that S, E and F
 * become operands, and M, W (formed transposed) too, without an exchange.
 *
 * Operands are two fp16 numbers hi + lo (22 bits) in three products
 * hi hi + hi lo + lo hi with binary32 sums: off by at most 2^-22 of a
 * product, 2.5 times the rate of binary32 products (8192^3 in the vendor
 * library: 1134 TFLOP/s in 16 bits, a third of which is 378, against 154 in 32).
 * The ranges that fp16 lacks are kept outside: a row of k or q is scaled by a
 * power of two to below 1 and its norm becomes a factor of the row; T and W
 * carry a power of two, V, E, F and S one for each column. Log decays are summed
 * in 64 bits, since their differences are what counts.
 *
 * 16,384 rows of one sequence, 16 key and 48 value heads of 128 x 128: 852 us,
 * 105 TFLOP/s of the recurrent form's operations, which at 1.2 us a row would
 * take 20 ms for them. 690 us are the scan's, whose 256 steps hang on each
 * other: 2.6 us a step, two LDS round trips through a barrier with 24 matrix
 * instructions a wave behind each (2.07 us with a third of the heads: the L2s
 * give a workgroup 120 KB a step). 265 are linattn_prep's, bound by the bytes
 * it writes. (Launches overlap; U = B V formed there as well made its writes,
 * not the scan, the bound.) 513 rows: 43.7 us.
 */
#include <type_traits>

#include "kq_linattn.h"

namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kC = kChunkRows;
constexpr uint32_t kHeads = 3;    /* value heads that linattn_prep takes at a time */
constexpr uint32_t kBlk = 20;     /* floats of an LDS row of a 16 x 16 block */
constexpr uint32_t kMat = 12288;  /* bytes of a lower 64 x 64 operand, hi and lo */
constexpr uint32_t kRowF = 5 * kC; /* floats of a value head's factors */

constexpr float kUnit = 0x1p10f;   /* of the rows of k and q */
/* W from its product T K' with T at 2^14 .. 2^15: |W| <= 64 x 2 max |T| */
constexpr int kWDown = 7;
constexpr float kMixUnit = 0x1p6f; /* of M: |q.k| <= 512 of such rows (128 values, below 2) */

/* where the parts of the scratch lie */
struct Work {
    kq_linattn_plan plan;
    kq_launch_seqs one; /* a call of one sequence, which needs no plan; else count 0 */
    char *data;       /* operands of the chunks of a window */
    uint32_t window;  /* chunks */
    uint64_t chunk_bytes;
    uint32_t key_bytes, value_at, value_bytes;
};

/* chunk c of the call; one without rows behind the last */
__device__ __forceinline__ kq_linattn_chunk chunk_at(const Work &w, uint32_t c) {
    if (w.one.count == 0u) return c < w.plan.chunks ? w.plan.chunk[c] : kq_linattn_chunk{};
    bool bad = false;
    const kq::SeqSpan sp = kq::seq_span(w.one, 0u, bad);
    kq_linattn_chunk r = {};
    if (sp.live && c * kC < sp.rows) {
        r.row = sp.begin + c * kC;
        r.ahead = sp.rows - c * kC;
        r.rows = r.ahead < kC ? r.ahead : kC;
        r.number = c;
        r.left = (r.ahead + kC - 1u) / kC;
        r.slot = sp.slot;
        r.fresh = sp.fresh ? 1u : 0u;
    }
    return r;
}

/* Whether chunk c, which has no rows, is the first of a call's only sequence,
 * without rows: its state is passed on. Says so if the sequence is refused. */
__device__ __forceinline__ bool passes(const Work &w, uint32_t c, kq::SeqSpan &sp,
                                       uint32_t *status) {
    if (w.one.count == 0u || c != 0u) return false;
    bool bad = false;
    sp = kq::seq_span(w.one, 0u, bad);
    if (bad) kq_flag(status, KQ_DEV_SEQUENCE);
    return sp.live;
}

__device__ __forceinline__ f4 mfma(h8 a, h8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
/* (ah + al) (bh + bl) without the smallest product */
__device__ __forceinline__ f4 mfma3(h8 ah, h8 al, h8 bh, h8 bl, f4 c) {
    c = mfma(al, bh, c);
    c = mfma(ah, bl, c);
    return mfma(ah, bh, c);
}

/* x s in two fp16 numbers: hi rounded from x s, lo from what is left */
template <int N, typename H>
__device__ __forceinline__ void split(const float *x, float s, H &hi, H &lo) {
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const h2 h = __builtin_convertvector(f2{x[i] * s, x[i + 1] * s}, h2);
        hi[i] = h.x;
        hi[i + 1] = h.y;
        lo[i] = (_Float16)fmaf(x[i], s, -(float)h.x);
        lo[i + 1] = (_Float16)fmaf(x[i + 1], s, -(float)h.y);
    }
}

/* Of a lower 64 x 64 operand the pieces (row tile rt, 32 columns from 32 ks)
 * that are not zeros, 2048 bytes each: rt 0 and 1 have ks 0 only */
__device__ __forceinline__ constexpr uint32_t piece(uint32_t rt, uint32_t ks) {
    return (rt < 2u ? rt : 2u * rt - 2u + ks) * 2048u;
}

/* the power of two that brings m to 2^14 .. 2^15 */
__device__ __forceinline__ int scale_exp(float m) {
    const int e = 15 - __builtin_amdgcn_frexp_expf(m);
    return e > 126 ? 126 : e;
}
__device__ __forceinline__ float pow2(int e) { return ldexpf(1.0f, e); }

/* ------------------------------------------------------------------ */

/* A lane's part x[ks][8] of a row in the order of an operand; its four lanes
 * differ in bits 4 and 5. Scales the
 * row to below 1 by a power of two and gives the factor that makes it the
 * row (over its norm) again. */
template <int KS>
__device__ __forceinline__ float unit_row(float (&x)[KS][8], uint32_t normalize, float eps,
                                          bool &badin) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            badin |= !kq_isfinite(x[i][e]);
            m = fmaxf(m, fabsf(x[i][e]));
        }
    m = kq::lanes_max<48>(m);
    int p = __builtin_amdgcn_frexp_expf(m);
    p = p > 127 ? 127 : p < -126 ? -126 : p;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            x[i][e] = ldexpf(x[i][e], -p);
            s = fmaf(x[i][e], x[i][e], s);
        }
    s = kq::lanes_sum<48>(s);
    if (m == 0.0f) return 0.0f; /* 1 / sqrt(eps) would make the others' share of a scale small */
    if (normalize == 0u) return pow2(p);
    /* 2^p / sqrt(2^2p s + eps) */
    return (float)(1.0 / sqrt((double)s + ldexp((double)eps, -2 * p)));
}

/* the lower blocks of a 64 x 64 matrix, 16 x 16 each, in LDS */
typedef float Lower[10][16][kBlk];
__device__ __forceinline__ constexpr int blk(int i, int j) { return i * (i + 1) / 2 + j; }

/* C + A B in binary32, where a lane has A[r16][4 g4 ..] and B[4 g4 ..][r16],
 * the layout of C itself */
__device__ __forceinline__ f4 mfma_f32(f4 a, f4 b, f4 c) {
#pragma unroll
    for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], c, 0, 0, 0);
    return c;
}

/* The inverse of 1 + L by one wave, L's lower blocks (below the diagonal) in
 * `m`, into x (a lane: rows 4 g4 .., column r16 of each block). The diagonal
 * blocks by forward substitution, a lane for each column of each; the others
 * from X_ij = -X_ii sum_k L_ik X_kj. */
__device__ __forceinline__ void invert(Lower &m, uint32_t lane, f4 (&x)[10]) {
    const uint32_t r16 = lane & 15u, g4 = lane >> 4;
    {
        const int d[4] = {blk(0, 0), blk(1, 1), blk(2, 2), blk(3, 3)};
        const float(*l)[kBlk] = m[g4 == 0u ? d[0] : g4 == 1u ? d[1] : g4 == 2u ? d[2] : d[3]];
        float t[16];
        t[0] = r16 == 0u ? 1.0f : 0.0f;
        auto rows = [&](auto from, auto to) { /* all of their reads in flight at once */
            f4 row[to - from][(to + 2) / 4];
#pragma unroll
            for (int i = from; i < to; ++i)
#pragma unroll
                for (int k = 0; 4 * k < i; ++k) row[i - from][k] = *(const f4 *)&l[i][4 * k];
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = from; i < to; ++i) {
                float s[2] = {(int)r16 == i ? 1.0f : 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < i; ++j)
                    s[j & 1] = fmaf(-row[i - from][j / 4][j % 4], t[j], s[j & 1]);
                t[i] = s[0] + s[1];
            }
        };
        rows(std::integral_constant<int, 1>{}, std::integral_constant<int, 9>{});
        rows(std::integral_constant<int, 9>{}, std::integral_constant<int, 16>{});
        __builtin_amdgcn_wave_barrier();
        float(*o)[kBlk] = m[g4 == 0u ? d[0] : g4 == 1u ? d[1] : g4 == 2u ? d[2] : d[3]];
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i][r16] = t[i];
        __builtin_amdgcn_wave_barrier();
    }
    f4 diag[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        diag[i] = *(const f4 *)&m[blk(i, i)][r16][4u * g4];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[blk(i, i)][r] = m[blk(i, i)][4u * g4 + r][r16];
    }
#pragma unroll
    for (int d = 1; d < 4; ++d)
#pragma unroll
        for (int j = 0; j + d < 4; ++j) {
            const int i = j + d;
            f4 p = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = j; k < i; ++k)
                p = mfma_f32(*(const f4 *)&m[blk(i, k)][r16][4u * g4], x[blk(k, j)], p);
            x[blk(i, j)] = -mfma_f32(diag[i], p, f4{0.0f, 0.0f, 0.0f, 0.0f});
        }
}

template <int DK, bool DELTA>
__global__ __launch_bounds__(256, 2) void linattn_prep(kq_launch_linattn a, Work w,
                                                       uint32_t base, uint32_t *status) {
    constexpr int KS = DK / 32, NT = DK / 64; /* dk tiles of a wave */
    constexpr uint32_t kKeyImage = 256u * DK, kSolve = DELTA ? kHeads * sizeof(Lower) : 0u;
    /* K' as an operand, then the triangles of the heads */
    __shared__ __attribute__((aligned(16))) char pool[kKeyImage > kSolve ? kKeyImage : kSolve];
    /* T diag(n^2 e^G) as an operand */
    __shared__ __attribute__((aligned(16))) char tri[DELTA ? kMat : 16];
    __shared__ __attribute__((aligned(16))) double sum[kHeads][kC];
    __shared__ __attribute__((aligned(16))) float cw[kHeads][kC], cu[kHeads][kC];
    __shared__ float bet[kHeads][kC], nks[kC], nqs[kC];
    __shared__ int pw[kHeads], pu[kHeads];
    const uint32_t c = base + blockIdx.x, kh = blockIdx.y;
    const kq_linattn_chunk ch = chunk_at(w, c);
    if (ch.rows == 0u) return;
    const uint32_t lane = threadIdx.x & 63u, r16 = lane & 15u, g4 = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t per = a.value_heads / a.key_heads;
    char *cb = w.data + (uint64_t)blockIdx.x * w.chunk_bytes;
    char *kb = cb + (uint64_t)kh * w.key_bytes;
    bool badin = false;

    /* the gates of head h0 + wave, row `lane`: loaded first, formed while
     * nothing else is under way that a wait for them would wait for too */
    float g_rate = 0.0f, g_bias = 0.0f, g_alpha = 0.0f, g_beta = 0.0f, g_b = 0.0f;
    double g_sum = 0.0, g_end = 0.0;
    auto load_gates = [&](uint32_t h) {
        const uint64_t t = (uint64_t)ch.row + (lane < ch.rows ? lane : 0u);
        g_rate = a.rate[h];
        if (a.bias != nullptr) g_bias = a.bias[h];
        if (a.alpha != nullptr) g_alpha = a.alpha[t * a.as + h];
        if (DELTA) g_beta = a.beta[t * a.bs + h];
    };
    auto form_gates = [&]() {
        badin |= !kq_isfinite(g_rate) || g_rate > 0.0f || !kq_isfinite(g_bias) ||
                 !kq_isfinite(g_alpha) || !kq_isfinite(g_beta);
        const float g = lane < ch.rows ? kq::log_decay(a, g_alpha, g_rate, g_bias) : 0.0f;
        if (DELTA) g_b = lane < ch.rows ? kq::sigmoid(g_beta) : 0.0f;
        g_sum = kq_wave_scan_f64((double)g);
        g_end = kq_readlane_f64(g_sum, 63);
    };
    if (wave < kHeads && wave < per) load_gates(kh * per + wave);

    /* rows 16 wave + r16 of k and q as operands */
    f4 kk[4], qk[4];
    {
        h8 kh8[KS], kl8[KS], qh8[KS], ql8[KS];
        const uint32_t i = 16u * wave + r16;
        float x[KS][8], y[KS][8];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int e = 0; e < 8; ++e) x[ks][e] = y[ks][e] = 0.0f;
        if (i < ch.rows) {
            const uint64_t t = (uint64_t)ch.row + i;
            const float4 *kp = (const float4 *)(a.k + t * a.ks + kh * DK + 4u * g4);
            const float4 *qp = (const float4 *)(a.q + t * a.qs + kh * DK + 4u * g4);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float4 u = kp[8 * ks + 4 * k], v = qp[8 * ks + 4 * k];
                    x[ks][4 * k] = u.x; x[ks][4 * k + 1] = u.y;
                    x[ks][4 * k + 2] = u.z; x[ks][4 * k + 3] = u.w;
                    y[ks][4 * k] = v.x; y[ks][4 * k + 1] = v.y;
                    y[ks][4 * k + 2] = v.z; y[ks][4 * k + 3] = v.w;
                }
        }
        if (wave < kHeads && wave < per) form_gates();
        const float nk = unit_row<KS>(x, a.normalize, a.epsilon, badin);
        const float nq = unit_row<KS>(y, a.normalize, a.epsilon, badin) * a.scale;
        if (g4 == 0u) {
            nks[i] = nk;
            nqs[i] = nq;
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            split<8>(x[ks], kUnit, kh8[ks], kl8[ks]);
            split<8>(y[ks], kUnit, qh8[ks], ql8[ks]);
            const uint32_t at = ((wave * KS + ks) * 2u) * 1024u + lane * 16u;
            *(h8 *)(pool + at) = kh8[ks];
            *(h8 *)(pool + at + 1024u) = kl8[ks];
            *(h8 *)(kb + at) = qh8[ks];
            *(h8 *)(kb + at + 1024u) = ql8[ks];
        }
        __syncthreads();
        /* k_j.k_i and k_j.q_i, times kUnit^2: row j = 16 jt + 4 g4 + r, column
         * i = 16 wave + r16 */
#pragma unroll
        for (int jt = 0; jt < 4; ++jt) {
            kk[jt] = qk[jt] = f4{0.0f, 0.0f, 0.0f, 0.0f};
            if (jt <= (int)wave)
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const uint32_t at = ((jt * KS + ks) * 2u) * 1024u + lane * 16u;
                    const h8 ah = *(const h8 *)(pool + at), al = *(const h8 *)(pool + at + 1024u);
                    if (DELTA) kk[jt] = mfma3(ah, al, kh8[ks], kl8[ks], kk[jt]);
                    qk[jt] = mfma3(ah, al, qh8[ks], ql8[ks], qk[jt]);
                }
        }
    }
    /* K'^T: row 16 (NT wave + t) + r16 of DK, 8 of the 64 columns */
    h8 kth[NT][2], ktl[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const uint32_t tile = NT * wave + t;
        const uint32_t from = (tile >> 1) * 2048u + (tile & 1u) * 8u + (r16 >> 2) * 256u +
                              (r16 & 3u) * 2u + 4u * g4 * 16u;
#pragma unroll
        for (uint32_t ks = 0; ks < 2u; ++ks) {
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e) { /* row 32 ks + 16 (e / 4) + 4 g4 + e % 4 of K' */
                const uint32_t at = from + (2u * ks + e / 4u) * (KS * 2048u) + (e & 3u) * 16u;
                kth[t][ks][e] = *(const _Float16 *)(pool + at);
                ktl[t][ks][e] = *(const _Float16 *)(pool + at + 1024u);
            }
            char *to = kb + kKeyImage + ((tile * 2u + ks) * 2u) * 1024u + lane * 16u;
            *(h8 *)to = kth[t][ks];
            *(h8 *)(to + 1024u) = ktl[t][ks];
        }
    }
    __syncthreads(); /* the image of k is free */

    Lower *solve = (Lower *)pool;
    for (uint32_t h0 = 0; h0 < per; h0 += kHeads) {
        const uint32_t nh = per - h0 < kHeads ? per - h0 : kHeads;
        char *vb0 = cb + w.value_at + (uint64_t)(kh * per + h0) * w.value_bytes;
        if (wave < nh) { /* a wave for each head, a lane for each row */
            if (h0 != 0u) {
                load_gates(kh * per + h0 + wave);
                form_gates();
            }
            const double G = g_sum, end = g_end;
            const float from = kq::exp_of(G), n = nks[lane], b = g_b;
            sum[wave][lane] = G;
            bet[wave][lane] = b * n * n;
            cw[wave][lane] = b * n * n * from;
            cu[wave][lane] = b * n;
            float *f = (float *)(vb0 + wave * w.value_bytes + kMat);
            f[lane] = n;
            f[kC + lane] = kq::exp_of(end - G);
            f[2 * kC + lane] = nqs[lane];
            f[3 * kC + lane] = from * nqs[lane];
            const kq::Decay e = kq::decay_of(end);
            if (lane == 0u) *(f2 *)&f[4 * kC] = f2{e.c0, e.c1};
        }
        __syncthreads();
        for (uint32_t hh = 0; hh < nh; ++hh) {
            char *vb = vb0 + hh * w.value_bytes;
            const double gi = sum[hh][16u * wave + r16];
            const float bi = bet[hh][16u * wave + r16] * (1.0f / kUnit / kUnit);
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                float x[8];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const int jt = 2 * ks + half;
                    f4 l = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int r = 0; r < 4; ++r) x[4 * half + r] = 0.0f;
                    if (jt <= (int)wave) {
                        double gj[4];
#pragma unroll
                        for (int r = 0; r < 4; ++r) gj[r] = sum[hh][16 * jt + 4u * g4 + r];
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            float fall = kq::exp_of(gi - gj[r]);
                            /* rows of the diagonal tile past column i: zeros */
                            fall = jt == (int)wave && 4u * g4 + r > r16 ? 0.0f : fall;
                            x[4 * half + r] = qk[jt][r] * fall;
                            l[r] = bi * fall * kk[jt][r];
                        }
                    }
                    if (DELTA && jt <= (int)wave)
                        *(f4 *)&solve[hh][blk((int)wave, 0) + jt][r16][4u * g4] = l;
                }
                if (2 * ks > (int)wave) continue;
                h8 hi, lo;
                split<8>(x, kMixUnit / kUnit / kUnit, hi, lo);
                char *to = vb + piece(wave, ks) + lane * 16u;
                *(h8 *)to = hi;
                *(h8 *)(to + 1024u) = lo;
            }
        }
        __syncthreads();
        if constexpr (!DELTA) continue;
        if (wave < nh) {
            f4 x[10];
            invert(solve[wave], lane, x);
            float mw = 0.0f, mu = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j <= i; ++j) {
                    const float fw = cw[wave][16 * j + r16], fu = cu[wave][16 * j + r16];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float t = x[blk(i, j)][r];
                        mw = fmaxf(mw, fabsf(t * fw));
                        mu = fmaxf(mu, fabsf(t * fu));
                        if (i != j) solve[wave][blk(i, j)][4u * g4 + r][r16] = t;
                    }
                }
            mw = kq::lanes_max<63>(mw);
            mu = kq::lanes_max<63>(mu);
            if (lane == 0u) {
                const int p = scale_exp(mw);
                pw[wave] = p;
                pu[wave] = scale_exp(mu);
                float *f = (float *)(vb0 + wave * w.value_bytes + kMat) + 4 * kC;
                f[2] = pow2(kWDown - p);
                f[3] = pow2(-pu[wave]);
            }
        }
        __syncthreads();
        for (uint32_t hh = 0; hh < nh; ++hh) {
            char *vb = vb0 + hh * w.value_bytes + kMat + kRowF * 4u;
            /* T's rows 16 wave + r16 with the two factors of its columns, as operands */
            const float sw = pow2(pw[hh]), su = pow2(pu[hh]);
#pragma unroll
            for (uint32_t ks = 0; ks < 2u; ++ks) {
                if (ks > wave >> 1) continue;
                float xw[8], xu[8];
#pragma unroll
                for (uint32_t half = 0; half < 2u; ++half) {
                    const uint32_t jb = 2u * ks + half;
                    f4 t = f4{0.0f, 0.0f, 0.0f, 0.0f};
                    if (jb <= wave) t = *(const f4 *)&solve[hh][blk((int)wave, 0) + jb][r16][4u * g4];
                    const f4 fw = *(const f4 *)&cw[hh][16u * jb + 4u * g4],
                             fu = *(const f4 *)&cu[hh][16u * jb + 4u * g4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        xw[4 * half + r] = t[r] * fw[r];
                        xu[4 * half + r] = t[r] * fu[r];
                    }
                }
                h8 hi, lo;
                char *to = tri + piece(wave, ks) + lane * 16u;
                split<8>(xw, sw, hi, lo);
                *(h8 *)to = hi;
                *(h8 *)(to + 1024u) = lo;
                to = vb + kKeyImage + piece(wave, ks) + lane * 16u;
                split<8>(xu, su, hi, lo);
                *(h8 *)to = hi;
                *(h8 *)(to + 1024u) = lo;
            }
            kq_lds_barrier();
            /* W's rows 16 rt .., the wave's columns, transposed */
#pragma unroll
            for (int rt = 0; rt < 4; ++rt) {
                f4 x[NT];
#pragma unroll
                for (int t = 0; t < NT; ++t) x[t] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int ks = 0; ks <= rt >> 1; ++ks) {
                    const char *p = tri + piece(rt, ks) + lane * 16u;
                    const h8 wh = *(const h8 *)p, wl = *(const h8 *)(p + 1024);
#pragma unroll
                    for (int t = 0; t < NT; ++t)
                        x[t] = mfma3(kth[t][ks], ktl[t][ks], wh, wl, x[t]);
                }
                /* as an operand: half of a lane's eight values from each tile */
                h8 hi, lo;
                float y[4 * NT];
#pragma unroll
                for (int k = 0; k < 4 * NT; ++k) y[k] = x[k / 4][k % 4];
                const uint32_t tile = NT * wave;
                char *to = vb + ((rt * KS + (tile >> 1)) * 2u) * 1024u + lane * 16u;
                if constexpr (NT == 2) {
                    split<8>(y, 1.0f / kUnit / (1 << kWDown), hi, lo);
                    *(h8 *)to = hi;
                    *(h8 *)(to + 1024u) = lo;
                } else {
                    h4 hi4, lo4;
                    split<4>(y, 1.0f / kUnit / (1 << kWDown), hi4, lo4);
                    *(h4 *)(to + (tile & 1u) * 8u) = hi4;
                    *(h4 *)(to + (tile & 1u) * 8u + 1024u) = lo4;
                }
            }
            kq_lds_barrier();
        }
    }
    if (badin) kq_flag(status, KQ_DEV_INPUT);
}

/* ------------------------------------------------------------------ */

constexpr uint32_t kTile = 32; /* columns of v that a workgroup holds */

/* a lane's part of an operand, hi and lo, N pieces 2048 bytes apart */
template <int N>
struct Frag {
    h8 hi[N], lo[N];
    __device__ __forceinline__ void load1(KqBuf b, uint32_t lane16, uint32_t at, int i) {
        hi[i] = __builtin_bit_cast(h8, kq_ld128(b, lane16, at + i * 2048u));
        lo[i] = __builtin_bit_cast(h8, kq_ld128(b, lane16, at + i * 2048u + 1024u));
    }
    __device__ __forceinline__ void load(KqBuf b, uint32_t lane16, uint32_t at) {
#pragma unroll
        for (int i = 0; i < N; ++i) load1(b, lane16, at, i);
    }
    __device__ __forceinline__ void read1(const char *p, int i) {
        hi[i] = *(const h8 *)p;
        lo[i] = *(const h8 *)(p + 1024);
    }
    __device__ __forceinline__ void read(const char *p, int step) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            hi[i] = *(const h8 *)(p + i * step);
            lo[i] = *(const h8 *)(p + i * step + 1024);
        }
    }
};

/* A lane's four rows of row tile `tile`, column tile ct of a result, times s,
 * as part of the right operand at p */
__device__ __forceinline__ void put(char *p, uint32_t tile, uint32_t ct, uint32_t lane16,
                                    const f4 &x, float s) {
    const float y[4] = {x[0], x[1], x[2], x[3]};
    h4 hi, lo;
    split<4>(y, s, hi, lo);
    char *to = p + (((tile >> 1) * 2u + ct) * 2u) * 1024u + lane16 + (tile & 1u) * 8u;
    *(h4 *)to = hi;
    *(h4 *)(to + 1024u) = lo;
}

__device__ __forceinline__ float largest(float m, const f4 &x) {
    return fmaxf(fmaxf(m, fmaxf(fabsf(x[0]), fabsf(x[1]))), fmaxf(fabsf(x[2]), fabsf(x[3])));
}

/* The largest values of column r16 over a wave's rows, for sets of 16 columns:
 * row g4 of the lanes has set g4 & 1 of two, set g4 of four. Rows of lanes are
 * exchanged between two sets, so that each step halves what is left. */
__device__ __forceinline__ float swap_max16(float a, float b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false,
                                                    false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float swap_max32(float a, float b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false,
                                                    false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float tops(float m0, float m1) {
    const float x = swap_max16(m0, m1);
    return swap_max32(x, x);
}
__device__ __forceinline__ float tops(float m0, float m1, float m2, float m3) {
    return swap_max16(swap_max32(m0, m2), swap_max32(m1, m3));
}
/* over the four waves that hold the rows */
__device__ __forceinline__ float top_of(const f4 &a) {
    return fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3]));
}

/* of a power of two */
__device__ __forceinline__ float inverse(float power) {
    return __uint_as_float((254u << 23) - __float_as_uint(power));
}

/* The scales of an operand's columns, which all waves hold from one chunk to
 * the next: a lane for each column, of two or four sets (`tops`). A column has
 * its own, since what one column of v is multiplied by says nothing of its
 * neighbours': under one scale for 32 a column 2^-k of the largest would be
 * off by 2^(k - 35) of itself. They hold while every column's largest value
 * lies between `low` and 2^15, or is zero. Values from 2^-2 on keep 22 bits,
 * smaller ones an error of 2^-25: 2^-31 of the column's largest for E, whose
 * rows are in the outputs one by one. For S and F, which are in sums over all
 * rows, 2^-27 will do: decays that leave a chunk's last few rows move their
 * largest values far (each time a barrier more: 64 steps of four heads 118 us
 * with E's limits, 111 with these).
 */
struct Scales {
    float s, low;
    int back; /* from 2^14 .. 2^15 to where a largest value is set */
    __device__ __forceinline__ Scales(bool sums)
        : s(1.0f), low(sums ? 4.0f : 64.0f), back(sums ? 7 : 5) {}
    /* the same in all waves */
    __device__ __forceinline__ bool hold(float m) const {
        const float y = m * s;
        return __ballot(!(y < 32768.0f) || (y < low && m > 0.0f)) == 0ull;
    }
    __device__ __forceinline__ void set(float m) { s = pow2(scale_exp(m) - back); }
    /* of column r16 of a set */
    __device__ __forceinline__ float of(uint32_t set, uint32_t r16) const {
        return __shfl(s, (int)(16u * set + r16), KQ_WAVE);
    }
};

/*
 * Waves 0 .. 3 (the solvers) run the chain S -> E -> S': W S and E for 16 rows
 * of the chunk each, then K'^T F for a fourth of S's rows, which they hold.
 * Waves 4 .. 7 (the writers) form Q S and M E for 16 rows each and store the
 * output. Waves 8 .. 11, with the delta correction, split V and form B V. So
 * an operand is loaded by one wave, for both column tiles, and what no other
 * step waits for runs beside the chain. Two phases a chunk with a barrier each:
 *   1  S's operand is there: W S, E, F | M E of the chunk before, its output |
 *                            B V of the next
 *   2  E's and F's are there: S' | Q S | V of the chunk after as an operand
 * (Q S beside W S would have both wait for the same LDS reads). All loads of
 * a role's loop are straight-line code: behind a branch the compiler could
 * not tell how many are under way, and would wait for too many.
 */
constexpr int scan_waves(bool delta) { return delta ? 12 : 8; }

template <int DK, bool DELTA>
__global__ __launch_bounds__(64 * scan_waves(DELTA)) void linattn_scan(kq_launch_linattn a,
                                                                Work w, uint32_t base,
                                                                uint32_t *status) {
    constexpr int KS = DK / 32, NR = DK / 64; /* steps over S's rows; row tiles of a solver */
    constexpr uint32_t kKeyImage = 256u * DK;
    __shared__ __attribute__((aligned(16))) char sbufs[2][KS * 4096], ebufs[2][8192], fbuf[8192],
        vbuf[DELTA ? 8192 : 16], ubufs[2][DELTA ? 8192 : 16]; /* V; B V in 32 bits */
    /* the columns' largest values in each solver's rows, of S; of E, then F */
    __shared__ __attribute__((aligned(16))) float top_s[kTile][4], top_ef[2 * kTile][4];
    __shared__ float vscale[2][kTile]; /* of V's columns, by 32 rows */
    /* the chunks of one sequence that lie in the window: from the window's
     * first chunk, or the sequence's */
    const kq_linattn_chunk ch = chunk_at(w, base + blockIdx.y);
    if (ch.rows == 0u) {
        kq::SeqSpan sp;
        if (passes(w, base + blockIdx.y, sp, status)) {
            const uint32_t at = blockIdx.x * (DK * kTile); /* a part of the state each */
            const size_t from = (size_t)sp.slot * a.value_heads * DK * a.value_width + at;
            bool odd = false;
            for (uint32_t i = threadIdx.x; i < DK * kTile; i += blockDim.x) {
                const float x = sp.fresh ? 0.0f : a.state[from + i];
                odd |= !kq_isfinite(x);
                a.state_out[from + i] = x;
            }
            if (odd) kq_flag(status, KQ_DEV_NUMERIC);
        }
        return;
    }
    if (blockIdx.y != 0u && ch.number != 0u) return;
    const uint32_t left_here = w.window - blockIdx.y;
    const uint32_t last = (left_here < ch.left ? left_here : ch.left) - 1u;
    bool bad = false, badin = false;
    const uint32_t rows = ch.ahead; /* from the first chunk on */
    const float *state = ch.number == 0u ? a.state : a.state_out; /* as the last window left it */
    const bool fresh = ch.fresh != 0u && ch.number == 0u;
    const uint32_t lane = threadIdx.x & 63u, r16 = lane & 15u, g4 = lane >> 4, lane16 = lane * 16u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t rt = wave & 3u, fr = 16u * rt + 4u * g4; /* rows of the chunk */
    /* workgroups go round the 8 XCDs: those of a head, which read the same
     * operands, to one of them */
    uint32_t b = blockIdx.x;
    if (gridDim.x % 8u == 0u) b = (b % 8u) * (gridDim.x / 8u) + b / 8u;
    const uint32_t tiles = a.value_width / kTile;
    const uint32_t h = b / tiles, tile = b % tiles, col = tile * kTile + r16;
    const uint32_t kh = h / (a.value_heads / a.key_heads);

    const char *data = w.data + (uint64_t)blockIdx.y * w.chunk_bytes;
    const uint32_t kat = kh * w.key_bytes, vat = w.value_at + h * w.value_bytes; /* Q; M */
    const uint32_t fat = vat + kMat;           /* the rows' factors */
    const uint32_t wat = fat + kRowF * 4u;     /* W, then B */
    auto chunk = [&](uint32_t n) {
        return kq_buf(data + (uint64_t)n * w.chunk_bytes, (uint32_t)w.chunk_bytes);
    };
    auto factors = [&](KqBuf c, uint32_t i) {
        return __builtin_bit_cast(f4, kq_ld128(c, fr * 4u, fat + i * kC * 4u));
    };
    auto scalar = [&](KqBuf c, uint32_t i) {
        return __uint_as_float(kq_ld32(c, i * 4u, fat + 4u * kC * 4u));
    };
    /* lower operands: the piece that rows 0 .. 31 lack lies past the buffer */
    const uint32_t lane_k1 = rt < 2u ? 0x7fffff00u : lane16;
    auto load_lower = [&](Frag<2> &x, KqBuf c, uint32_t at, int ks) {
        x.hi[ks] = __builtin_bit_cast(
            h8, kq_ld128(c, ks == 0 ? lane16 : lane_k1, at + piece(rt, rt < 2u ? 0u : ks)));
        x.lo[ks] = __builtin_bit_cast(
            h8, kq_ld128(c, ks == 0 ? lane16 : lane_k1, at + piece(rt, rt < 2u ? 0u : ks) + 1024u));
    };
    auto zero = [](f4(&x)[2]) { x[0] = x[1] = f4{0.0f, 0.0f, 0.0f, 0.0f}; };
    /* rows of v or of the output of chunk n, the call's column tile */
    auto rows_at = [&](const float *p, uint64_t stride, uint32_t n) {
        const uint32_t left = rows - n * kC; /* rows past it are past the buffer */
        return kq_buf(p + ((uint64_t)ch.row + n * kC) * stride + h * a.value_width,
                      (left < kC ? left : kC) * (uint32_t)stride * 4u);
    };
    /* of S, of E and F; and of the lane's columns, by column tile: */
    Scales own_s(true), own_ef(lane >= kTile);
    float ss[2] = {1.0f, 1.0f}, se[2] = {1.0f, 1.0f}, sf[2] = {1.0f, 1.0f};
    /* From the largest values that a phase left behind its barrier: whether the
     * scales are set anew, which all waves find alike, so that all of them take
     * the barrier more behind which the operand is there again. */
    auto moved_s = [&](f4 t) {
        const float m = top_of(t);
        if (own_s.hold(m)) return false;
        own_s.set(m);
        for (uint32_t ct = 0; ct < 2u; ++ct) ss[ct] = own_s.of(ct, r16);
        return true;
    };
    auto moved_ef = [&](f4 t) {
        const float m = top_of(t);
        if (own_ef.hold(m)) return false;
        own_ef.set(m);
        for (uint32_t ct = 0; ct < 2u; ++ct) {
            se[ct] = own_ef.of(ct, r16);
            sf[ct] = own_ef.of(2u + ct, r16);
        }
        return true;
    };

    if (wave < 4u) {
        __builtin_amdgcn_s_setprio(3); /* the chain first */
        const uint32_t srow = 16u * NR * rt + 4u * g4;
        const size_t sat = (((size_t)ch.slot * a.value_heads + h) * DK + srow) * a.value_width + col;
        f4 S[NR][2];
#pragma unroll
        for (int t = 0; t < NR; ++t)
#pragma unroll
            for (int ct = 0; ct < 2; ++ct)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    S[t][ct][r] =
                        fresh ? 0.0f
                              : state[sat + (size_t)(16 * t + r) * a.value_width + 16u * ct];
        Frag<KS> W;
        Frag<2> T[NR];
        f4 V[2], f0, f1; /* B V, or V with the factors n; e^(G_64 - G) */
        float iw = 0.0f, c0, c1;
        uint32_t io[4]; /* the wave's rows of v, in bytes */
        if (!DELTA)
#pragma unroll
            for (int r = 0; r < 4; ++r) io[r] = ((fr + r) * (uint32_t)a.vs + col) * 4u;
        auto load_w = [&](KqBuf c) {
            if (DELTA) W.load(c, lane16, wat + rt * KS * 2048u);
        };
        auto load_v = [&](KqBuf c, uint32_t n) {
            if (DELTA) {
                iw = scalar(c, 2u);
            } else {
                f0 = factors(c, 0u);
                const KqBuf v = rows_at(a.v, a.vs, n);
#pragma unroll
                for (int ct = 0; ct < 2; ++ct)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        V[ct][r] = __uint_as_float(kq_ld32(v, io[r], 64u * ct));
            }
            f1 = factors(c, 1u);
        };
        auto load_decay = [&](KqBuf c) {
            const f2 e = __builtin_bit_cast(f2, kq_ld64(c, 0u, fat + 4u * kC * 4u));
            c0 = e.x;
            c1 = e.y;
        };
        auto load_t = [&](KqBuf c) {
#pragma unroll
            for (int t = 0; t < NR; ++t)
                T[t].load(c, lane16, kat + kKeyImage + (NR * rt + t) * 4096u);
            load_decay(c);
        };
        /* S as an operand */
        char *sbuf = sbufs[0];
        auto put_s = [&]() {
#pragma unroll
            for (int t = 0; t < NR; ++t)
#pragma unroll
                for (int ct = 0; ct < 2; ++ct) put(sbuf, NR * rt + t, ct, lane16, S[t][ct], ss[ct]);
        };
        auto share_s = [&]() {
            float m[2] = {0.0f, 0.0f};
#pragma unroll
            for (int t = 0; t < NR; ++t)
#pragma unroll
                for (int ct = 0; ct < 2; ++ct) m[ct] = largest(m[ct], S[t][ct]);
            const float top = tops(m[0], m[1]);
            if (lane < kTile) top_s[lane][rt] = top;
            put_s();
        };
        const KqBuf first = chunk(0u);
        load_w(first);
        load_v(first, 0u);
        load_t(first);
        share_s();
        if (DELTA) { /* the writers' V and B V of the first chunk */
            kq_lds_barrier();
            kq_lds_barrier();
        }
        for (uint32_t n = 0; n <= last; ++n) {
            const uint32_t more = n < last ? n + 1u : n; /* the last loads again */
            const KqBuf next = chunk(more);
            char *ebuf = ebufs[n & 1u];
            kq_lds_barrier();
            /* 1: E, and F with the decay to the chunk's end */
            f4 E[2], F[2];
            zero(E);
            Frag<2> B[2]; /* two steps' at a time */
            auto read_s = [&]() {
                if (DELTA)
#pragma unroll
                    for (int ct = 0; ct < 2; ++ct) B[ct].read(sbuf + ct * 2048u + lane16, 4096);
            };
            {
                const f4 t = *(const f4 *)top_s[lane & 31u];
                read_s(); /* under way meanwhile */
                if (moved_s(t)) {
                    put_s();
                    kq_lds_barrier();
                    read_s();
                }
            }
            if (DELTA) {
#pragma unroll
                for (int ct = 0; ct < 2; ++ct)
                    V[ct] = *(const f4 *)(ubufs[n & 1u] + (ct * 4u + rt) * 1024u + lane16);
                __builtin_amdgcn_sched_barrier(0); /* all in flight, then the products */
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                    for (int ct = 0; ct < 2; ++ct)
                        E[ct] = mfma3(W.hi[ks], W.lo[ks], B[ct].hi[ks & 1], B[ct].lo[ks & 1],
                                      E[ct]);
                    if (ks + 2 < KS)
#pragma unroll
                        for (int ct = 0; ct < 2; ++ct)
                            B[ct].read1(sbuf + ct * 2048u + lane16 + (ks + 2) * 4096, ks & 1);
                    W.load1(next, lane16, wat + rt * KS * 2048u, ks); /* of the next chunk */
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            const float is[2] = {inverse(ss[0]) * iw, inverse(ss[1]) * iw};
#pragma unroll
            for (int ct = 0; ct < 2; ++ct)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (!DELTA) badin |= !kq_isfinite(V[ct][r]);
                    E[ct][r] = DELTA ? fmaf(-is[ct], E[ct][r], V[ct][r]) : f0[r] * V[ct][r];
                    F[ct][r] = E[ct][r] * f1[r];
                }
            top_ef[lane][rt] = tops(largest(0.0f, E[0]), largest(0.0f, E[1]), largest(0.0f, F[0]),
                                    largest(0.0f, F[1]));
            auto put_ef = [&]() {
#pragma unroll
                for (int ct = 0; ct < 2; ++ct) {
                    put(fbuf, rt, ct, lane16, F[ct], sf[ct]);
                    put(ebuf, rt, ct, lane16, E[ct], se[ct]);
                }
            };
            put_ef();
            kq_lds_barrier();
            /* 2: S' = e^G S + K'^T F, e^G in two parts (kq::Decay) */
            f4 x[NR][2];
            {
                Frag<2> B[2];
                auto read_f = [&]() {
#pragma unroll
                    for (int ct = 0; ct < 2; ++ct) B[ct].read(fbuf + ct * 2048u + lane16, 4096);
                };
                const f4 t = *(const f4 *)top_ef[lane];
                read_f();
                if (moved_ef(t)) {
                    put_ef();
                    kq_lds_barrier();
                    read_f();
                }
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int t = 0; t < NR; ++t) zero(x[t]);
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
                    for (int t = 0; t < NR; ++t)
#pragma unroll
                        for (int ct = 0; ct < 2; ++ct) {
                            x[t][ct] = mfma3(T[t].hi[ks], T[t].lo[ks], B[ct].hi[ks], B[ct].lo[ks],
                                             x[t][ct]);
                            if (ks == 1) /* beside the products */
#pragma unroll
                                for (int r = 0; r < 4; ++r)
                                    S[t][ct][r] = fmaf(c1, S[t][ct][r], c0 * S[t][ct][r]);
                        }
#pragma unroll
                    for (int t = 0; t < NR; ++t)
                        T[t].load1(next, lane16, kat + kKeyImage + (NR * rt + t) * 4096u, ks);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            load_v(next, more);
            const float jf[2] = {inverse(sf[0]) * (1.0f / kUnit), inverse(sf[1]) * (1.0f / kUnit)};
#pragma unroll
            for (int t = 0; t < NR; ++t)
#pragma unroll
                for (int ct = 0; ct < 2; ++ct)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        S[t][ct][r] = fmaf(x[t][ct][r], jf[ct], S[t][ct][r]);
            load_decay(next);
            sbuf = sbufs[(n + 1u) & 1u];
            share_s();
        }
        kq_lds_barrier();
#pragma unroll
        for (int t = 0; t < NR; ++t)
#pragma unroll
            for (int ct = 0; ct < 2; ++ct)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    bad |= !kq_isfinite(S[t][ct][r]);
                    a.state_out[sat + (size_t)(16 * t + r) * a.value_width + 16u * ct] =
                        S[t][ct][r];
                }
    } else if (wave < 8u) {
        Frag<KS> Q;
        Frag<2> M;
        f4 f0, f1; /* the factors of q, and with e^G */
        uint32_t io[4]; /* the wave's rows of the output, in bytes */
#pragma unroll
        for (int r = 0; r < 4; ++r) io[r] = ((fr + r) * (uint32_t)a.ys + col) * 4u;
        f4 P[2];
        float ps[2] = {0.0f, 0.0f};
        zero(P);
        /* M E and the output of chunk n; the operands of chunk n + 1 */
        auto write = [&](uint32_t n, KqBuf next) {
            f4 O[2];
            zero(O);
            Frag<2> B[2];
#pragma unroll
            for (int ct = 0; ct < 2; ++ct)
                B[ct].read(ebufs[n & 1u] + ct * 2048u + lane16, 4096);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
                for (int ct = 0; ct < 2; ++ct)
                    O[ct] = mfma3(M.hi[ks], M.lo[ks], B[ct].hi[ks], B[ct].lo[ks], O[ct]);
                load_lower(M, next, vat, ks);
                __builtin_amdgcn_sched_barrier(0);
            }
            const float pe[2] = {inverse(se[0]) * (1.0f / kMixUnit),
                                 inverse(se[1]) * (1.0f / kMixUnit)};
            const KqBuf y = rows_at(a.y, a.ys, n);
#pragma unroll
            for (int ct = 0; ct < 2; ++ct)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float o = fmaf(f1[r], P[ct][r] * ps[ct], f0[r] * (O[ct][r] * pe[ct]));
                    bad |= !kq_isfinite(o);
                    __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(o), y.r, (int)io[r],
                                                          64 * ct, 0);
                }
            f0 = factors(next, 2u);
            f1 = factors(next, 3u);
        };
        {
            const KqBuf first = chunk(0u);
            Q.load(first, lane16, kat + rt * KS * 2048u);
            load_lower(M, first, vat, 0);
            load_lower(M, first, vat, 1);
            f0 = factors(first, 2u);
            f1 = factors(first, 3u);
        }
        if (DELTA) {
            kq_lds_barrier();
            kq_lds_barrier();
        }
        auto check_s = [&]() {
            kq_lds_barrier();
            if (moved_s(*(const f4 *)top_s[lane & 31u])) kq_lds_barrier();
        };
        /* 2: Q S */
        auto second = [&](uint32_t n) {
            kq_lds_barrier();
            if (moved_ef(*(const f4 *)top_ef[lane])) kq_lds_barrier();
            const KqBuf next = chunk(n < last ? n + 1u : n);
            const char *sb = sbufs[n & 1u] + lane16;
            Frag<2> B[2];
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) B[ct].read(sb + ct * 2048u, 4096);
            zero(P);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
                for (int ct = 0; ct < 2; ++ct)
                    P[ct] = mfma3(Q.hi[ks], Q.lo[ks], B[ct].hi[ks & 1], B[ct].lo[ks & 1], P[ct]);
                if (ks + 2 < KS)
#pragma unroll
                    for (int ct = 0; ct < 2; ++ct)
                        B[ct].read1(sb + ct * 2048u + (ks + 2) * 4096, ks & 1);
                Q.load1(next, lane16, kat + rt * KS * 2048u, ks);
                __builtin_amdgcn_sched_barrier(0);
            }
            for (int ct = 0; ct < 2; ++ct) ps[ct] = inverse(ss[ct]) * (1.0f / kUnit);
        };
        check_s();
        second(0u);
        for (uint32_t n = 1; n <= last; ++n) {
            check_s();
            write(n - 1u, chunk(n));
            second(n);
        }
        kq_lds_barrier();
        write(last, chunk(last));
    } else if constexpr (DELTA) {
        /* what a wait for a miss in every cache would hold up the chain for:
         * two chunks on their way */
        Frag<2> B2[2];
        float ib[2], v[2][8];
        /* V of a chunk: a wave has the 32 rows ks of column tile ct, in the
         * order of an operand, a power of two for each column */
        const uint32_t ct = rt & 1u, ks = rt >> 1;
        auto load_v = [&](float(&v)[8], uint32_t n) {
            const KqBuf vr = rows_at(a.v, a.vs, n < last ? n : last);
            /* the row in the lane's offset, which alone is held against the buffer's end */
            const uint32_t at = ((32u * ks + 4u * g4) * (uint32_t)a.vs + col) * 4u;
#pragma unroll
            for (uint32_t e = 0; e < 8u; ++e)
                v[e] = __uint_as_float(
                    kq_ld32(vr, at + (16u * (e / 4u) + e % 4u) * (uint32_t)a.vs * 4u, 64u * ct));
        };
        auto put_v = [&](float(&v)[8]) {
            float m = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                badin |= !kq_isfinite(v[e]);
                m = fmaxf(m, fabsf(v[e]));
            }
            const int p = scale_exp(kq::lanes_max<48>(m));
            if (g4 == 0u) vscale[ks][16u * ct + r16] = pow2(-p);
            h8 hi, lo;
            split<8>(v, pow2(p), hi, lo);
            char *to = vbuf + ((ks * 2u + ct) * 2u) * 1024u + lane16;
            *(h8 *)to = hi;
            *(h8 *)(to + 1024u) = lo;
        };
        auto load_b = [&](int i, uint32_t n) {
            const KqBuf c = chunk(n < last ? n : last);
            load_lower(B2[i], c, wat + kKeyImage, 0);
            load_lower(B2[i], c, wat + kKeyImage, 1);
            ib[i] = scalar(c, 3u);
        };
        /* B V of chunk n from vbuf; then B of chunk n + 2 */
        auto times_v = [&](int i, uint32_t n) {
            f4 U[2][2];
            Frag<2> B[2];
            float sc[2][2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                zero(U[t]);
                B[t].read(vbuf + t * 2048u + lane16, 4096);
                sc[t][0] = vscale[0][16 * t + r16] * ib[i];
                sc[t][1] = vscale[1][16 * t + r16] * ib[i];
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    U[t][k] = mfma3(B2[i].hi[k], B2[i].lo[k], B[t].hi[k], B[t].lo[k], U[t][k]);
#pragma unroll
            for (int t = 0; t < 2; ++t)
                *(f4 *)(ubufs[n & 1u] + (4u * t + rt) * 1024u + lane16) =
                    U[t][0] * sc[t][0] + U[t][1] * sc[t][1];
            __builtin_amdgcn_sched_barrier(0);
            load_b(i, n + 2u);
        };
        load_v(v[0], 0u);
        load_v(v[1], 1u);
        load_b(0, 0u);
        load_b(1, 1u);
        put_v(v[0]);
        load_v(v[0], 2u);
        kq_lds_barrier();
        times_v(0, 0u);
        kq_lds_barrier();
        put_v(v[1]);
        load_v(v[1], 3u);
        /* chunk n, with the registers of B of chunk n + 1 and of V of chunk n + 2 */
        auto body = [&](int ib1, int iv, uint32_t n) {
            kq_lds_barrier();
            if (moved_s(*(const f4 *)top_s[lane & 31u])) kq_lds_barrier();
            /* 1 (behind the last chunk, B V of it again) */
            times_v(ib1, n + 1u);
            kq_lds_barrier();
            if (moved_ef(*(const f4 *)top_ef[lane])) kq_lds_barrier();
            /* 2 */
            put_v(v[iv]);
            load_v(v[iv], n + 4u);
        };
        for (uint32_t n = 0; n <= last; n += 2u) {
            body(1, 0, n);
            if (n == last) break;
            body(0, 1, n + 1u);
        }
        kq_lds_barrier();
    }
    if (badin) kq_flag(status, KQ_DEV_INPUT);
    if (bad) kq_flag(status, KQ_DEV_NUMERIC);
}

/* ------------------------------------------------------------------ */

/*
 * Without the delta correction a chunk's rows add to the state what does not
 * hang on it. Where the scan would have few workgroups, the work is split
 * over the chunks instead:
 *   linattn_sums    U = sum_j e^(G_64 - G_j) k'_j e_j^T of every chunk
 *   linattn_states  S from chunk to chunk, into U's place
 *   linattn_outs    the outputs of every chunk
 * for a state read and written more a chunk.
 */

/* a workgroup's chunk, value head and 32 columns; four waves with 16 rows of
 * the chunk each */
struct Place {
    kq_linattn_chunk ch;
    uint32_t h, col, fr;
    char *data;
    uint32_t kat, vat, fat, uat; /* Q, M, the factors, U */
    KqBuf buf;
    __device__ __forceinline__ Place(const kq_launch_linattn &a, const Work &w, uint32_t base,
                                     uint32_t wave, uint32_t lane) {
        ch = chunk_at(w, base + blockIdx.y);
        uint32_t b = blockIdx.x; /* a head's to one XCD, as in the scan */
        if (gridDim.x % 8u == 0u) b = (b % 8u) * (gridDim.x / 8u) + b / 8u;
        const uint32_t tiles = a.value_width / kTile;
        h = b / tiles;
        col = (b % tiles) * kTile + (lane & 15u);
        fr = 16u * wave + 4u * (lane >> 4);
        data = w.data + (uint64_t)blockIdx.y * w.chunk_bytes;
        kat = h / (a.value_heads / a.key_heads) * w.key_bytes;
        vat = w.value_at + h * w.value_bytes;
        fat = vat + kMat;
        uat = fat + kRowF * 4u;
        buf = kq_buf(data, (uint32_t)w.chunk_bytes);
    }
    __device__ __forceinline__ f4 factors(uint32_t i) const {
        return __builtin_bit_cast(f4, kq_ld128(buf, fr * 4u, fat + i * kC * 4u));
    }
    /* the chunk's rows of v or of the output; rows past it are past the buffer */
    __device__ __forceinline__ KqBuf rows(const float *p, uint64_t stride, uint32_t width) const {
        return kq_buf(p + (uint64_t)ch.row * stride + h * width, ch.rows * (uint32_t)stride * 4u);
    }
    __device__ __forceinline__ void load_v(const kq_launch_linattn &a, f4 (&V)[2]) const {
        const KqBuf v = rows(a.v, a.vs, a.value_width);
#pragma unroll
        for (int ct = 0; ct < 2; ++ct)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                V[ct][r] = __uint_as_float(
                    kq_ld32(v, ((fr + r) * (uint32_t)a.vs + col) * 4u, 64u * ct));
    }
};

template <int DK>
__global__ __launch_bounds__(256) void linattn_sums(kq_launch_linattn a, Work w,
                                                    uint32_t base, uint32_t *status) {
    constexpr int NR = DK / 64;
    __shared__ __attribute__((aligned(16))) char fbuf[8192];
    __shared__ __attribute__((aligned(16))) float top[kTile][4]; /* of each wave's rows */
    const uint32_t lane = threadIdx.x & 63u, lane16 = lane * 16u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Place p(a, w, base, wave, lane);
    if (p.ch.rows == 0u) return;
    f4 V[2];
    p.load_v(a, V);
    const f4 f0 = p.factors(0u), f1 = p.factors(1u);
    Frag<2> T[NR];
#pragma unroll
    for (int t = 0; t < NR; ++t)
        T[t].load(p.buf, lane16, p.kat + 256u * DK + (NR * wave + t) * 4096u);
    bool badin = false;
#pragma unroll
    for (int ct = 0; ct < 2; ++ct)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            badin |= !kq_isfinite(V[ct][r]);
            V[ct][r] = f0[r] * V[ct][r] * f1[r];
        }
    const float m = tops(largest(0.0f, V[0]), largest(0.0f, V[1]));
    if (lane < kTile) top[lane][wave] = m;
    kq_lds_barrier();
    float s[2]; /* of the lane's columns */
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) {
        s[ct] = pow2(scale_exp(top_of(*(const f4 *)top[16 * ct + (lane & 15u)])));
        put(fbuf, wave, ct, lane16, V[ct], s[ct]);
    }
    kq_lds_barrier();
    float *u = (float *)(p.data + p.uat) +
               (16u * NR * wave + 4u * (lane >> 4)) * a.value_width + p.col;
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) {
        Frag<2> B;
        B.read(fbuf + ct * 2048u + lane16, 4096);
#pragma unroll
        for (int t = 0; t < NR; ++t) {
            f4 x = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
                x = mfma3(T[t].hi[ks], T[t].lo[ks], B.hi[ks], B.lo[ks], x);
#pragma unroll
            for (int r = 0; r < 4; ++r)
                u[(uint32_t)(16 * t + r) * a.value_width + 16u * ct] =
                    x[r] * (inverse(s[ct]) * (1.0f / kUnit));
        }
    }
    if (badin) kq_flag(status, KQ_DEV_INPUT);
}

/* grid (1024 values of the states, window): the first chunk of a sequence in
 * the window goes on to its last there */
__global__ __launch_bounds__(256) void linattn_states(kq_launch_linattn a, Work w,
                                                      uint32_t base, uint32_t *status) {
    constexpr uint32_t kAhead = 8;
    kq_linattn_chunk ch = chunk_at(w, base + blockIdx.y);
    uint32_t n = 0u;
    if (ch.rows == 0u) {
        kq::SeqSpan sp;
        if (!passes(w, base + blockIdx.y, sp, status)) return;
        ch.slot = sp.slot;
        ch.fresh = sp.fresh ? 1u : 0u;
    } else {
        if (blockIdx.y != 0u && ch.number != 0u) return;
        const uint32_t left_here = w.window - blockIdx.y;
        n = left_here < ch.left ? left_here : ch.left;
    }
    bool bad = false;
    const uint32_t size = a.key_width * a.value_width; /* a multiple of 1024 */
    const uint32_t at = blockIdx.x * 1024u, h = at / size, i = at % size + 4u * threadIdx.x;
    const size_t sat = ((size_t)ch.slot * a.value_heads + h) * size + i;
    f4 S = f4{0.0f, 0.0f, 0.0f, 0.0f};
    if (ch.number != 0u)
        S = *(const f4 *)(a.state_out + sat);
    else if (ch.fresh == 0u)
        S = *(const f4 *)(a.state + sat);
    char *f = w.data + (uint64_t)blockIdx.y * w.chunk_bytes + w.value_at + h * w.value_bytes + kMat;
    for (uint32_t c = 0; c < n; c += kAhead) {
        f4 u[kAhead];
        f2 e[kAhead]; /* e^G in two parts */
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k) { /* the last again behind it */
            const char *p = f + (uint64_t)(c + k < n ? c + k : n - 1u) * w.chunk_bytes;
            u[k] = *(const f4 *)(p + kRowF * 4u + i * 4u);
            e[k] = *(const f2 *)(p + 4u * kC * 4u);
        }
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k) {
            if (c + k >= n) break;
            *(f4 *)(f + (uint64_t)(c + k) * w.chunk_bytes + kRowF * 4u + i * 4u) = S;
#pragma unroll
            for (int r = 0; r < 4; ++r) S[r] = fmaf(e[k].x, S[r], fmaf(e[k].y, S[r], u[k][r]));
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) bad |= !kq_isfinite(S[r]);
    *(f4 *)(a.state_out + sat) = S;
    if (bad) kq_flag(status, KQ_DEV_NUMERIC);
}

template <int DK>
__global__ __launch_bounds__(256) void linattn_outs(kq_launch_linattn a, Work w,
                                                    uint32_t base, uint32_t *status) {
    constexpr int KS = DK / 32, NR = DK / 64;
    __shared__ __attribute__((aligned(16))) char sbuf[KS * 4096], ebuf[8192];
    __shared__ __attribute__((aligned(16))) float top[2 * kTile][4]; /* of S, then E */
    const uint32_t lane = threadIdx.x & 63u, lane16 = lane * 16u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Place p(a, w, base, wave, lane);
    if (p.ch.rows == 0u) return;
    f4 S[NR][2], V[2];
    const float *s = (const float *)(p.data + p.uat) +
                     (16u * NR * wave + 4u * (lane >> 4)) * a.value_width + p.col;
#pragma unroll
    for (int t = 0; t < NR; ++t)
#pragma unroll
        for (int ct = 0; ct < 2; ++ct)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                S[t][ct][r] = s[(uint32_t)(16 * t + r) * a.value_width + 16u * ct];
    p.load_v(a, V);
    const f4 f0 = p.factors(0u), f2 = p.factors(2u), f3 = p.factors(3u);
    Frag<KS> Q;
    Frag<2> M;
    Q.load(p.buf, lane16, p.kat + wave * KS * 2048u);
    M.load(p.buf, lane16, p.vat + piece(wave, 0u)); /* rows 0 .. 31 have one piece */
    float ms[2] = {0.0f, 0.0f}, me[2];
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) {
#pragma unroll
        for (int t = 0; t < NR; ++t) ms[ct] = largest(ms[ct], S[t][ct]);
#pragma unroll
        for (int r = 0; r < 4; ++r) V[ct][r] *= f0[r];
        me[ct] = largest(0.0f, V[ct]);
    }
    top[lane][wave] = tops(ms[0], ms[1], me[0], me[1]);
    kq_lds_barrier();
    float ss[2], se[2]; /* of the lane's columns */
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) {
        ss[ct] = pow2(scale_exp(top_of(*(const f4 *)top[16 * ct + (lane & 15u)])));
        se[ct] = pow2(scale_exp(top_of(*(const f4 *)top[kTile + 16 * ct + (lane & 15u)])));
#pragma unroll
        for (int t = 0; t < NR; ++t) put(sbuf, NR * wave + t, ct, lane16, S[t][ct], ss[ct]);
        put(ebuf, wave, ct, lane16, V[ct], se[ct]);
    }
    kq_lds_barrier();
    const KqBuf y = p.rows(a.y, a.ys, a.value_width);
    bool bad = false;
#pragma unroll
    for (int ct = 0; ct < 2; ++ct) {
        f4 P = f4{0.0f, 0.0f, 0.0f, 0.0f}, O = P;
        const float ps = inverse(ss[ct]) * (1.0f / kUnit), pe = inverse(se[ct]) * (1.0f / kMixUnit);
        Frag<KS> B;
        B.read(sbuf + ct * 2048u + lane16, 4096);
        Frag<2> E;
        E.read(ebuf + ct * 2048u + lane16, 4096);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
            P = mfma3(Q.hi[ks], Q.lo[ks], B.hi[ks], B.lo[ks], P);
        O = mfma3(M.hi[0], M.lo[0], E.hi[0], E.lo[0], O);
        if (wave >= 2u) O = mfma3(M.hi[1], M.lo[1], E.hi[1], E.lo[1], O);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float o = fmaf(f3[r], P[r] * ps, f2[r] * (O[r] * pe));
            bad |= !kq_isfinite(o);
            __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(o), y.r,
                                                  (int)(((p.fr + r) * (uint32_t)a.ys + p.col) * 4u),
                                                  64 * ct, 0);
        }
    }
    if (bad) kq_flag(status, KQ_DEV_NUMERIC);
}

/* Whether a call without the delta correction is split over the chunks: if the
 * scan's workgroups, those of 128 rows of S counted twice, are 64 at most.
 * The scan and the three launches (4099 rows): 32 of 64 rows 99 and 44 us, 48
 * of 64 (three sequences) 42 and 26; 64 of 128 125 and 112; 192 of 128 148
 * and 268. */
bool over_chunks(const kq_launch_linattn &a, uint32_t count) {
    return a.beta == nullptr &&
           (uint64_t)a.value_heads * (a.value_width / kTile) * (a.key_width / 64u) * count <= 64u;
}

uint64_t up256(uint64_t n) { return (n + 255u) & ~(uint64_t)255u; }

/* chunks that sequences of more than max_rows rows can have at most */
uint64_t most_chunks(uint64_t tokens, uint32_t count, uint32_t max_rows) {
    const uint64_t n = tokens / (max_rows + 1u);
    return (tokens + (kC - 1u) * (n < count ? n : count)) / kC;
}

/* The operands are made and used a window of chunks at a time, so that they
 * stay in the memory-side cache between the two launches and are overwritten
 * there. */
constexpr uint64_t kWindowBytes = 160u << 20;

Work carve(const kq_launch_linattn &a, uint64_t tokens, uint32_t count, uint32_t max_rows,
           void *scratch, uint64_t *bytes) {
    Work w = {};
    const uint64_t n = most_chunks(tokens, count, max_rows);
    const bool delta = a.beta != nullptr;
    char *p = (char *)(((uintptr_t)scratch + 255u) & ~(uintptr_t)255u);
    w.plan.chunk = (kq_linattn_chunk *)p;
    w.plan.chunks = (uint32_t)n;
    w.data = p + up256(sizeof(kq_linattn_chunk) * n);
    w.key_bytes = 512u * a.key_width;
    w.value_at = w.key_bytes * a.key_heads;
    const uint32_t least = kMat + kRowF * 4u;
    const uint32_t solved = least + 256u * a.key_width + kMat;
    const uint32_t states = least + 4u * a.key_width * a.value_width;
    w.value_bytes = delta ? solved : over_chunks(a, count) ? states : least;
    w.chunk_bytes = w.value_at + (uint64_t)w.value_bytes * a.value_heads;
    /* room for any form: the sizes alone do not tell which */
    const uint64_t most =
        w.value_at + (uint64_t)(solved > states ? solved : states) * a.value_heads;
    const uint64_t fit = kWindowBytes / most < 8u ? 8u : kWindowBytes / most;
    /* whole rounds of linattn_prep's workgroups, two on each of 256 CUs */
    const uint64_t round = a.key_heads < 512u ? 512u / a.key_heads : 1u;
    const uint64_t whole = fit > round ? fit / round * round : fit;
    w.window = (uint32_t)(whole < n ? whole : n);
    *bytes = 256u + up256(sizeof(kq_linattn_chunk) * n) + w.window * most;
    return w;
}

template <int DK, bool DELTA>
hipError_t run(const kq_launch_linattn &a, uint32_t count, const Work &w, uint32_t *status,
               hipStream_t s) {
    for (uint32_t base = 0u; base < w.plan.chunks; base += w.window) {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(linattn_prep<DK, DELTA>),
                           dim3(w.window, a.key_heads), dim3(256), 0, s, a, w, base, status);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        if constexpr (!DELTA) {
            if (over_chunks(a, count)) {
                const dim3 grid(a.value_heads * (a.value_width / kTile), w.window);
                hipLaunchKernelGGL(HIP_KERNEL_NAME(linattn_sums<DK>), grid, dim3(256), 0, s, a,
                                   w, base, status);
                hipLaunchKernelGGL(linattn_states,
                                   dim3(a.value_heads * a.key_width * a.value_width / 1024u,
                                        w.window),
                                   dim3(256), 0, s, a, w, base, status);
                hipLaunchKernelGGL(HIP_KERNEL_NAME(linattn_outs<DK>), grid, dim3(256), 0, s, a,
                                   w, base, status);
                e = hipGetLastError();
                if (e != hipSuccess) return e;
                continue;
            }
        }
        hipLaunchKernelGGL(HIP_KERNEL_NAME(linattn_scan<DK, DELTA>),
                           dim3(a.value_heads * (a.value_width / kTile), w.window),
                               dim3(64 * scan_waves(DELTA)), 0, s, a, w, base, status);
        e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace

uint64_t kq_linattn_chunked_scratch(const kq_launch_linattn &a, uint64_t tokens, uint32_t count,
                                    uint32_t max_rows) {
    uint64_t bytes;
    (void)carve(a, tokens, count, max_rows, nullptr, &bytes);
    return bytes;
}

hipError_t kq_linattn_chunked(const kq_launch_linattn &a, const kq_launch_seqs &q,
                              uint32_t max_rows, void *scratch, uint32_t *status, hipStream_t s) {
    uint64_t bytes;
    Work w = carve(a, q.tokens, q.count, max_rows, scratch, &bytes);
    if (q.count == 1u) { /* a prompt of its own: no launch for its plan, 4.5 us */
        w.one = q;
    } else {
        const hipError_t e = kq_linattn_recurrent(a, q, max_rows, w.plan, status, s);
        if (e != hipSuccess) return e;
    }
    const bool delta = a.beta != nullptr;
    if (a.key_width == 128u)
        return delta ? run<128, true>(a, q.count, w, status, s)
                     : run<128, false>(a, q.count, w, status, s);
    return delta ? run<64, true>(a, q.count, w, status, s)
                 : run<64, false>(a, q.count, w, status, s);
}

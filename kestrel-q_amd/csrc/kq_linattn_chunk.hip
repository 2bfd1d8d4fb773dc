/*
 * kq_linattn_chunk.hip — linear attention with a decay for each head on
 * gfx950, the chunked form (include/kq_hip.h, kq_hip_linear_attention_f32).
 *
 * For the 64 rows of a chunk that starts from the state S, with log decays
 * summed from its start G_i (inclusive), rows of k, q, v as matrices, and
 * K~ = diag(e^G) K, the d of the recurrent form solve
 *   (1 + L) D = diag(b) (V - K~ S),   L_ij = b_i e^(G_i - G_j) k_i.k_j  (j < i)
 *   O = diag(e^G) Q S + M D,          M_ij = e^(G_i - G_j) q_i.k_j      (j <= i)
 *   S' = e^(G_64) S + sum_j e^(G_64 - G_j) k_j d_j^T
 * so that everything but three products with S is independent of it, and a
 * chunk costs seven matrix products instead of 64 dependent steps.
 *
 * Three launches:
 *   linattn_plan  cuts the sequences into chunks (on the device: the lengths
 *                 are there)
 *   linattn_prep  a workgroup for each chunk and key head: K, Q as operands
 *                 of the matrix cores, and for each of its value heads
 *                 A = (1 + L)^-1 diag(b) and M
 *   linattn_scan  a workgroup for each sequence, head and 32 columns of v:
 *                 S in registers from the first chunk to the last,
 *                 D = A (V - K~ S), O, S'
 *
 * Operands are two fp16 numbers hi + lo (22 bits) in three products
 * hi hi + hi lo + lo hi with binary32 sums: off by at most 2^-22 of a
 * product, 5 times the rate of binary32 products on these cores. The ranges
 * that fp16 lacks are kept outside: a row of k or q is scaled by a power of
 * two to below 1 and its norm becomes a factor of the row, A, the right-hand
 * sides, D and S carry a power of two for each workgroup (its largest value
 * at 2^14 .. 2^15: values down to 2^-17 of it keep all 22 bits, the rest an
 * error of 2^-40 of it). Log decays are summed in 64 bits, since their
 * differences are what counts.
 */
#include "kq_linattn.h"

namespace {

typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));

constexpr uint32_t kC = 64;       /* rows of a chunk */
constexpr uint32_t kHeads = 3;    /* value heads that linattn_prep takes at a time */
constexpr uint32_t kPitch = 68;   /* floats of an LDS row of 64 */
constexpr uint32_t kMat = 16384;  /* bytes of a 64 x 64 operand, hi and lo */
constexpr uint32_t kRowF = 6 * kC; /* floats of a value head's row factors */

constexpr float kUnit = 0x1p10f;   /* of the rows of k and q */
constexpr float kMixUnit = 0x1p6f; /* of M: |q.k| <= 512 of such rows (128 values, below 2) */

/* where the parts of the scratch lie */
struct Work {
    uint32_t *total;  /* chunks */
    uint2 *seq;       /* of each sequence: its first chunk and their number */
    uint4 *chunk;     /* first row, rows, sequence, 0 */
    char *data;
    uint64_t chunk_bytes;
    uint32_t key_bytes, value_at, value_bytes;
};

__device__ __forceinline__ f4 mfma(h8 a, h8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
/* (ah + al) (bh + bl) without the smallest product */
__device__ __forceinline__ f4 mfma3(h8 ah, h8 al, h8 bh, h8 bl, f4 c) {
    c = mfma(al, bh, c);
    c = mfma(ah, bl, c);
    return mfma(ah, bh, c);
}

template <int N, typename H>
__device__ __forceinline__ void split(const float *x, H &hi, H &lo) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        hi[i] = (_Float16)x[i];
        lo[i] = (_Float16)(x[i] - (float)hi[i]);
    }
}

/* the power of two that brings m to 2^14 .. 2^15 */
__device__ __forceinline__ int scale_exp(float m) {
    const int e = 15 - __builtin_amdgcn_frexp_expf(m);
    return e > 126 ? 126 : e;
}
__device__ __forceinline__ float pow2(int e) { return ldexpf(1.0f, e); }

/* ------------------------------------------------------------------ */

constexpr int kPlanThreads = 1024;

__global__ __launch_bounds__(kPlanThreads) void linattn_plan(kq_launch_seqs q, uint32_t max_rows,
                                                             Work w) {
    __shared__ uint32_t first[kPlanThreads], number[kPlanThreads], begin[kPlanThreads],
        rows[kPlanThreads], sums[kPlanThreads / 64];
    __shared__ uint32_t refused;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    if (tid == 0u) refused = 0u;
    __syncthreads();
    bool bad = false;
    for (uint32_t s = tid; s < q.count; s += kPlanThreads) kq::seq_span(q, s, bad);
    if (bad) refused = 1u; /* the recurrent form's launch reports it */
    __syncthreads();
    const bool none = refused != 0u;
    uint32_t at = 0u;
    for (uint32_t base = 0u; base < q.count; base += kPlanThreads) {
        const uint32_t s = base + tid;
        uint32_t n = 0u;
        if (s < q.count) {
            const kq::SeqSpan sp = kq::seq_span(q, s, bad);
            begin[tid] = sp.begin;
            rows[tid] = sp.rows;
            if (!none && sp.live && sp.rows > max_rows) n = (sp.rows + kC - 1u) / kC;
        }
        uint32_t x = n; /* inclusive sum over the workgroup */
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t y = __shfl_up(x, o, KQ_WAVE);
            if (lane >= (uint32_t)o) x += y;
        }
        if (lane == 63u) sums[wave] = x;
        __syncthreads();
        uint32_t before = at, all = at;
        for (uint32_t k = 0; k < kPlanThreads / 64u; ++k) {
            if (k < wave) before += sums[k];
            all += sums[k];
        }
        first[tid] = before + x - n;
        number[tid] = n;
        if (s < q.count) w.seq[s] = make_uint2(before + x - n, n);
        __syncthreads();
        for (uint32_t i = wave; i < kPlanThreads && base + i < q.count; i += kPlanThreads / 64u)
            for (uint32_t k = lane; k < number[i]; k += 64u) {
                const uint32_t left = rows[i] - k * kC;
                w.chunk[first[i] + k] =
                    make_uint4(begin[i] + k * kC, left < kC ? left : kC, base + i, 0u);
            }
        at = all;
        __syncthreads();
    }
    if (tid == 0u) *w.total = at;
}

/* ------------------------------------------------------------------ */

/* A lane's part of a row x in the order of an operand, x[ks][8] the values
 * 32 ks + 8 (lane >> 4) ..; its four lanes differ in bits 4 and 5. Scales the
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
    if (normalize == 0u) return pow2(p);
    /* 2^p / sqrt(2^2p s + eps) */
    return (float)(1.0 / sqrt((double)s + ldexp((double)eps, -2 * p)));
}

template <int DK, bool DELTA>
__global__ __launch_bounds__(256) void linattn_prep(kq_launch_linattn a, Work w,
                                                    uint32_t *status) {
    constexpr int KS = DK / 32;
    constexpr uint32_t kKeyImage = 256u * DK, kSolve = DELTA ? kHeads * kC * kPitch * 4u : 0u;
    __shared__ __attribute__((aligned(16))) char pool[kKeyImage > kSolve ? kKeyImage : kSolve];
    __shared__ __attribute__((aligned(16))) float mixbuf[4][16][kPitch];
    __shared__ double sum[kHeads][kC];
    __shared__ float beta[kHeads][kC], nks[kC], nqs[kC];
    const uint32_t c = blockIdx.x, kh = blockIdx.y;
    if (c >= *w.total) return;
    const uint4 ch = w.chunk[c];
    const uint32_t lane = threadIdx.x & 63u, r16 = lane & 15u, g4 = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    char *kb = w.data + (uint64_t)c * w.chunk_bytes + (uint64_t)kh * w.key_bytes;
    bool badin = false;

    /* rows 16 wave + r16 of k and q as operands */
    h8 kh8[KS], kl8[KS], qh8[KS], ql8[KS];
    {
        const uint32_t i = 16u * wave + r16;
        float x[KS][8], y[KS][8];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int e = 0; e < 8; ++e) x[ks][e] = y[ks][e] = 0.0f;
        if (i < ch.y) {
            const uint64_t t = (uint64_t)ch.x + i;
            const float4 *kp = (const float4 *)(a.k + t * a.ks + kh * DK + 8u * g4);
            const float4 *qp = (const float4 *)(a.q + t * a.qs + kh * DK + 8u * g4);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float4 u = kp[8 * ks + k], v = qp[8 * ks + k];
                    x[ks][4 * k] = u.x; x[ks][4 * k + 1] = u.y;
                    x[ks][4 * k + 2] = u.z; x[ks][4 * k + 3] = u.w;
                    y[ks][4 * k] = v.x; y[ks][4 * k + 1] = v.y;
                    y[ks][4 * k + 2] = v.z; y[ks][4 * k + 3] = v.w;
                }
        }
        const float nk = unit_row<KS>(x, a.normalize, a.epsilon, badin);
        const float nq = unit_row<KS>(y, a.normalize, a.epsilon, badin) * a.scale;
        if (g4 == 0u) {
            nks[i] = nk;
            nqs[i] = nq;
        }
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[ks][e] *= kUnit;
                y[ks][e] *= kUnit;
            }
            split<8>(x[ks], kh8[ks], kl8[ks]);
            split<8>(y[ks], qh8[ks], ql8[ks]);
            const uint32_t at = ((wave * KS + ks) * 2u) * 1024u + lane * 16u;
            *(h8 *)(pool + at) = kh8[ks];
            *(h8 *)(pool + at + 1024u) = kl8[ks];
            if (DELTA) {
                *(h8 *)(kb + at) = kh8[ks];
                *(h8 *)(kb + at + 1024u) = kl8[ks];
            }
            *(h8 *)(kb + kKeyImage + at) = qh8[ks];
            *(h8 *)(kb + kKeyImage + at + 1024u) = ql8[ks];
        }
    }
    __syncthreads();

    /* k_i.k_j and q_i.k_j, times kUnit^2: row 16 wave + 4 g4 + r, column 16 jt + r16 */
    f4 kk[4], qk[4];
#pragma unroll
    for (int jt = 0; jt < 4; ++jt) {
        kk[jt] = qk[jt] = f4{0.0f, 0.0f, 0.0f, 0.0f};
        if (jt <= (int)wave)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const uint32_t at = ((jt * KS + ks) * 2u) * 1024u + lane * 16u;
                const h8 bh = *(const h8 *)(pool + at), bl = *(const h8 *)(pool + at + 1024u);
                if (DELTA) kk[jt] = mfma3(kh8[ks], kl8[ks], bh, bl, kk[jt]);
                qk[jt] = mfma3(qh8[ks], ql8[ks], bh, bl, qk[jt]);
            }
    }
    /* k transposed: row 16 rt + r16 of DK, 8 of the 64 columns */
    for (uint32_t rt = wave; rt < DK / 16u; rt += 4u) {
        const uint32_t d = 16u * rt + r16;
        const uint32_t from = (d >> 5) * 2048u + ((d & 31u) >> 3) * 256u + (d & 7u) * 2u;
#pragma unroll
        for (uint32_t ks = 0; ks < 2u; ++ks)
#pragma unroll
            for (uint32_t plane = 0; plane < 2u; ++plane) {
                h8 v;
#pragma unroll
                for (uint32_t e = 0; e < 8u; ++e) {
                    const uint32_t t = 32u * ks + 8u * g4 + e;
                    v[e] = *(const _Float16 *)(pool + from + plane * 1024u +
                                               (t >> 4) * (KS * 2048u) + (t & 15u) * 16u);
                }
                *(h8 *)(kb + 2u * kKeyImage + ((rt * 2u + ks) * 2u + plane) * 1024u +
                        lane * 16u) = v;
            }
    }
    /* columns of M that no tile below writes */
#pragma unroll
    for (int k = 0; k < 16; ++k) mixbuf[wave][k][lane] = 0.0f;
    __syncthreads(); /* the image of k is free */

    float(*solve)[kC][kPitch] = (float(*)[kC][kPitch])pool;
    const uint32_t per = a.value_heads / a.key_heads;
    for (uint32_t h0 = 0; h0 < per; h0 += kHeads) {
        const uint32_t nh = per - h0 < kHeads ? per - h0 : kHeads;
        if (wave < nh) { /* a wave for each head, a lane for each row */
            const uint32_t h = kh * per + h0 + wave;
            const float rate = a.rate[h], bias = a.bias != nullptr ? a.bias[h] : 0.0f;
            badin |= !kq_isfinite(rate) || rate > 0.0f || !kq_isfinite(bias);
            float g = 0.0f, b = 0.0f;
            if (lane < ch.y) {
                const uint64_t t = (uint64_t)ch.x + lane;
                g = kq::log_decay(a, t, h, rate, bias, badin);
                if (DELTA) {
                    const float x = a.beta[t * a.bs + h];
                    badin |= !kq_isfinite(x);
                    b = kq::sigmoid(x);
                }
            }
            const double G = kq_wave_scan_f64((double)g);
            const double end = kq_readlane_f64(G, 63);
            sum[wave][lane] = G;
            beta[wave][lane] = b;
            const float from = kq::exp_of(G), to = kq::exp_of(end - G);
            float *f = (float *)(w.data + (uint64_t)c * w.chunk_bytes + w.value_at +
                                 (uint64_t)h * w.value_bytes + kMat);
            f[lane] = from * nks[lane];
            f[kC + lane] = nks[lane];
            f[2 * kC + lane] = to * nks[lane];
            f[3 * kC + lane] = nqs[lane];
            f[4 * kC + lane] = from * nqs[lane];
            const kq::Decay d = kq::decay_of((float)end);
            if (lane == 0u) {
                f[5 * kC] = d.c0;
                f[5 * kC + 1] = d.c1;
            }
        }
        __syncthreads();
        for (uint32_t hh = 0; hh < nh; ++hh) {
            char *vb = w.data + (uint64_t)c * w.chunk_bytes + w.value_at +
                       (uint64_t)(kh * per + h0 + hh) * w.value_bytes;
            double gi[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) gi[r] = sum[hh][16u * wave + 4u * g4 + r];
#pragma unroll
            for (int jt = 0; jt < 4; ++jt) {
                if (jt > (int)wave) continue;
                const uint32_t j = 16u * jt + r16;
                const double gj = sum[hh][j];
                const float nkj = nks[j];
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const uint32_t i = 16u * wave + 4u * g4 + r;
                    const float fall = j <= i ? kq::exp_of(gi[r] - gj) : 0.0f;
                    mixbuf[wave][4u * g4 + r][j] = qk[jt][r] * fall * (kMixUnit / kUnit / kUnit);
                    if (DELTA && j < i)
                        solve[hh][i][j] = beta[hh][i] * nks[i] * nkj * fall *
                                          (kk[jt][r] * (1.0f / kUnit / kUnit));
                }
            }
            /* the wave's own rows: its LDS operations complete in order */
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                float x[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = mixbuf[wave][r16][32u * ks + 8u * g4 + e];
                h8 hi, lo;
                split<8>(x, hi, lo);
                char *to = vb + ((wave * 2u + ks) * 2u) * 1024u + lane * 16u;
                *(h8 *)to = hi;
                *(h8 *)(to + 1024u) = lo;
            }
            __builtin_amdgcn_wave_barrier();
        }
        if constexpr (!DELTA) {
            __syncthreads();
            continue;
        }
        __syncthreads();
        if (wave < nh) {
            /* column `lane` of (1 + L)^-1, row after row */
            float t[kC];
#pragma unroll
            for (uint32_t i = 0; i < kC; ++i) {
                float s[4] = {lane == i ? 1.0f : 0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (uint32_t j = 0; j < i; ++j)
                    s[j & 3u] = fmaf(-solve[wave][i][j], t[j], s[j & 3u]);
                t[i] = (s[0] + s[1]) + (s[2] + s[3]);
            }
            const float b = beta[wave][lane];
            float m = 0.0f;
#pragma unroll
            for (uint32_t i = 0; i < kC; ++i) {
                t[i] *= b;
                m = fmaxf(m, fabsf(t[i]));
            }
            m = kq::lanes_max<63>(m);
            const int p = scale_exp(m);
            char *vb = w.data + (uint64_t)c * w.chunk_bytes + w.value_at +
                       (uint64_t)(kh * per + h0 + wave) * w.value_bytes;
            if (lane == 0u) *(float *)(vb + kMat + (5 * kC + 2) * 4u) = pow2(-p);
            __builtin_amdgcn_wave_barrier(); /* the rows of L have been read */
#pragma unroll
            for (uint32_t i = 0; i < kC; ++i) solve[wave][i][lane] = ldexpf(t[i], p);
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
            __builtin_amdgcn_wave_barrier();
            vb += kMat + kRowF * 4u;
#pragma unroll
            for (uint32_t rt = 0; rt < 4u; ++rt)
#pragma unroll
                for (uint32_t ks = 0; ks < 2u; ++ks) {
                    float x[8];
#pragma unroll
                    for (uint32_t e = 0; e < 8u; ++e)
                        x[e] = solve[wave][16u * rt + r16][32u * ks + 8u * g4 + e];
                    h8 hi, lo;
                    split<8>(x, hi, lo);
                    char *to = vb + ((rt * 2u + ks) * 2u) * 1024u + lane * 16u;
                    *(h8 *)to = hi;
                    *(h8 *)(to + 1024u) = lo;
                }
        }
        __syncthreads();
    }
    if (badin) kq_flag(status, KQ_DEV_INPUT);
}

/* ------------------------------------------------------------------ */

constexpr uint32_t kTile = 32; /* columns of v that a workgroup holds */

/* a lane's part of an operand, hi and lo, N pieces 1024 bytes apart */
template <int N>
struct Frag {
    h8 hi[N], lo[N];
    __device__ __forceinline__ void load(const char *p) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            hi[i] = *(const h8 *)(p + i * 2048);
            lo[i] = *(const h8 *)(p + i * 2048 + 1024);
        }
    }
};

/* Four values of consecutive rows (of which `row` is the first, in fours) of
 * column r16 of column tile ct, as part of the right operand at p */
__device__ __forceinline__ void put(char *p, uint32_t row, uint32_t ct, uint32_t r16, const f4 &x,
                                    float s) {
    float y[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) y[r] = x[r] * s;
    h4 hi, lo;
    split<4>(y, hi, lo);
    char *to = p + (((row >> 5) * 2u + ct) * 2u) * 1024u + (((row & 31u) >> 3) * 16u + r16) * 16u +
               (row & 7u) * 2u;
    *(h4 *)to = hi;
    *(h4 *)(to + 1024u) = lo;
}

__device__ __forceinline__ float largest(float m, const f4 &x) {
#pragma unroll
    for (int r = 0; r < 4; ++r) m = fmaxf(m, fabsf(x[r]));
    return m;
}

template <int DK, bool DELTA>
__global__ __launch_bounds__(256) void linattn_scan(kq_launch_linattn a, kq_launch_seqs q, Work w,
                                                    uint32_t *status) {
    constexpr int KS = DK / 32, RT = DK / 64;
    __shared__ __attribute__((aligned(16))) char sbuf[KS * 4096], rbuf[8192], ebuf[8192],
        fbuf[8192];
    __shared__ float top[4][4]; /* largest values: of S, the right-hand sides, E, F by wave */
    const uint32_t s = blockIdx.y;
    const uint2 mine = w.seq[s];
    if (mine.y == 0u) return;
    bool badseq = false, bad = false, badin = false;
    const kq::SeqSpan sp = kq::seq_span(q, s, badseq);
    if (!sp.live) return;
    const uint32_t lane = threadIdx.x & 63u, r16 = lane & 15u, g4 = lane >> 4;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    /* workgroups go round the 8 XCDs: those of a head, which read the same
     * operands, to one of them */
    uint32_t b = blockIdx.x;
    if (gridDim.x % 8u == 0u) b = (b % 8u) * (gridDim.x / 8u) + b / 8u;
    const uint32_t tiles = a.value_width / kTile;
    const uint32_t h = b / tiles, col = (b % tiles) * kTile + r16;
    const uint32_t kh = h / (a.value_heads / a.key_heads);
    const size_t sat = ((size_t)sp.slot * a.value_heads + h) * DK * a.value_width + col;

    f4 S[RT][2];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int ct = 0; ct < 2; ++ct)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t d = (wave * RT + rt) * 16u + 4u * g4 + r;
                S[rt][ct][r] = sp.fresh ? 0.0f
                                        : a.state[sat + (size_t)d * a.value_width + 16u * ct];
            }

    const char *kb = w.data + (uint64_t)mine.x * w.chunk_bytes + (uint64_t)kh * w.key_bytes;
    const char *vb = w.data + (uint64_t)mine.x * w.chunk_bytes + w.value_at +
                     (uint64_t)h * w.value_bytes;
    constexpr uint32_t kKeyImage = 256u * DK;
    Frag<KS> K, Q;
    Frag<2> A, M, T[RT];
    f4 V[2];
    auto load_kq = [&](uint32_t n) {
        const char *p = kb + (uint64_t)n * w.chunk_bytes + wave * KS * 2048u + lane * 16u;
        if (DELTA) K.load(p);
        Q.load(p + kKeyImage);
    };
    auto load_v = [&](uint32_t n) {
#pragma unroll
        for (int ct = 0; ct < 2; ++ct)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t i = n * kC + 16u * wave + 4u * g4 + r;
                V[ct][r] = i < sp.rows ? a.v[((uint64_t)sp.begin + i) * a.vs +
                                             h * a.value_width + col + 16u * ct]
                                       : 0.0f;
            }
    };
    auto load_a = [&](uint32_t n) {
        A.load(vb + (uint64_t)n * w.chunk_bytes + kMat + kRowF * 4u + wave * 4096u + lane * 16u);
    };
    auto load_mt = [&](uint32_t n) {
        M.load(vb + (uint64_t)n * w.chunk_bytes + wave * 4096u + lane * 16u);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
            T[rt].load(kb + (uint64_t)n * w.chunk_bytes + 2u * kKeyImage +
                       (wave * RT + rt) * 4096u + lane * 16u);
    };
    load_kq(0u);
    load_v(0u);
    if (DELTA) load_a(0u);
    load_mt(0u);

    for (uint32_t n = 0; n < mine.y; ++n) {
        const uint32_t more = n + 1u < mine.y ? n + 1u : n; /* the last loads again */
        const float *f = (const float *)(vb + (uint64_t)n * w.chunk_bytes + kMat);
        const uint32_t fr = 16u * wave + 4u * g4;
        const f4 fk = *(const f4 *)(f + fr), fe = *(const f4 *)(f + kC + fr),
                 ff = *(const f4 *)(f + 2 * kC + fr), fq = *(const f4 *)(f + 3 * kC + fr),
                 fp = *(const f4 *)(f + 4 * kC + fr);
        const float c0 = f[5 * kC], c1 = f[5 * kC + 1], ia = DELTA ? f[5 * kC + 2] : 0.0f;

        /* S as an operand */
        float m = 0.0f;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) m = largest(m, S[rt][ct]);
        m = kq::lanes_max<63>(m);
        if (lane == 0u) top[0][wave] = m;
        kq_lds_barrier();
        const int es = scale_exp(fmaxf(fmaxf(top[0][0], top[0][1]), fmaxf(top[0][2], top[0][3])));
        const float ss = pow2(es), is = ldexpf(1.0f / kUnit, -es);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int ct = 0; ct < 2; ++ct)
                put(sbuf, (wave * RT + rt) * 16u + 4u * g4, ct, r16, S[rt][ct], ss);
        kq_lds_barrier();

        /* K S and Q S for the wave's 16 rows */
        f4 X[2], P[2];
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) X[ct] = P[ct] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) {
                const char *p = sbuf + ((ks * 2 + ct) * 2) * 1024 + lane * 16u;
                const h8 bh = *(const h8 *)p, bl = *(const h8 *)(p + 1024);
                if (DELTA) X[ct] = mfma3(K.hi[ks], K.lo[ks], bh, bl, X[ct]);
                P[ct] = mfma3(Q.hi[ks], Q.lo[ks], bh, bl, P[ct]);
            }
        load_kq(more);

        f4 D[2];
#pragma unroll
        for (int ct = 0; ct < 2; ++ct)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                badin |= !kq_isfinite(V[ct][r]);
                D[ct][r] = DELTA ? V[ct][r] - fk[r] * (X[ct][r] * is) : V[ct][r];
            }
        load_v(more);
        if (DELTA) {
            /* D = A (V - K~ S) */
            m = kq::lanes_max<63>(largest(largest(0.0f, D[0]), D[1]));
            if (lane == 0u) top[1][wave] = m;
            kq_lds_barrier();
            const int er =
                scale_exp(fmaxf(fmaxf(top[1][0], top[1][1]), fmaxf(top[1][2], top[1][3])));
            const float sr = pow2(er);
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) put(rbuf, fr, ct, r16, D[ct], sr);
            kq_lds_barrier();
            const float ir = ia * pow2(-er);
#pragma unroll
            for (int ct = 0; ct < 2; ++ct) {
                f4 x = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    const char *p = rbuf + ((ks * 2 + ct) * 2) * 1024 + lane * 16u;
                    x = mfma3(A.hi[ks], A.lo[ks], *(const h8 *)p, *(const h8 *)(p + 1024), x);
                }
                D[ct] = x * ir;
            }
            load_a(more);
        }
        /* E: rows of D times the norm of k; F: and the decay to the chunk's end */
        f4 E[2], F[2];
        float me = 0.0f, mf = 0.0f;
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) {
            E[ct] = D[ct] * fe;
            F[ct] = D[ct] * ff;
            me = largest(me, E[ct]);
            mf = largest(mf, F[ct]);
        }
        me = kq::lanes_max<63>(me);
        mf = kq::lanes_max<63>(mf);
        if (lane == 0u) {
            top[2][wave] = me;
            top[3][wave] = mf;
        }
        kq_lds_barrier();
        const int ee = scale_exp(fmaxf(fmaxf(top[2][0], top[2][1]), fmaxf(top[2][2], top[2][3])));
        const int ef = scale_exp(fmaxf(fmaxf(top[3][0], top[3][1]), fmaxf(top[3][2], top[3][3])));
        const float se = pow2(ee), sf = pow2(ef);
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) {
            put(ebuf, fr, ct, r16, E[ct], se);
            put(fbuf, fr, ct, r16, F[ct], sf);
        }
        kq_lds_barrier();
        const float ie = ldexpf(1.0f / kMixUnit, -ee), jf = ldexpf(1.0f / kUnit, -ef);
        /* O = Q~ S + M E and S' = e^G S + K^T F */
        f4 O[2];
#pragma unroll
        for (int ct = 0; ct < 2; ++ct) {
            O[ct] = f4{0.0f, 0.0f, 0.0f, 0.0f};
            f4 x[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) x[rt] = O[ct];
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                const uint32_t at = ((ks * 2 + ct) * 2) * 1024 + lane * 16u;
                const h8 eh = *(const h8 *)(ebuf + at), el = *(const h8 *)(ebuf + at + 1024);
                const h8 fh = *(const h8 *)(fbuf + at), fl = *(const h8 *)(fbuf + at + 1024);
                O[ct] = mfma3(M.hi[ks], M.lo[ks], eh, el, O[ct]);
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) x[rt] = mfma3(T[rt].hi[ks], T[rt].lo[ks], fh, fl, x[rt]);
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    S[rt][ct][r] = fmaf(x[rt][r], jf, fmaf(c1, S[rt][ct][r], c0 * S[rt][ct][r]));
        }
        load_mt(more);
#pragma unroll
        for (int ct = 0; ct < 2; ++ct)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t i = n * kC + fr + r;
                const float o = fmaf(fp[r], P[ct][r] * is, fq[r] * (O[ct][r] * ie));
                bad |= !kq_isfinite(o);
                if (i < sp.rows)
                    a.y[((uint64_t)sp.begin + i) * a.ys + h * a.value_width + col + 16u * ct] = o;
            }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int ct = 0; ct < 2; ++ct)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t d = (wave * RT + rt) * 16u + 4u * g4 + r;
                bad |= !kq_isfinite(S[rt][ct][r]);
                a.state_out[sat + (size_t)d * a.value_width + 16u * ct] = S[rt][ct][r];
            }
    if (badin) kq_flag(status, KQ_DEV_INPUT);
    if (bad) kq_flag(status, KQ_DEV_NUMERIC);
}

uint64_t up256(uint64_t n) { return (n + 255u) & ~(uint64_t)255u; }

/* chunks that sequences of more than max_rows rows can have at most */
uint64_t most_chunks(uint64_t tokens, uint32_t count, uint32_t max_rows) {
    const uint64_t n = tokens / (max_rows + 1u);
    return (tokens + (kC - 1u) * (n < count ? n : count)) / kC;
}

Work carve(const kq_launch_linattn &a, uint64_t tokens, uint32_t count, uint32_t max_rows,
           void *scratch, uint64_t *bytes) {
    Work w;
    const uint64_t n = most_chunks(tokens, count, max_rows);
    const bool delta = a.beta != nullptr;
    char *p = (char *)(((uintptr_t)scratch + 255u) & ~(uintptr_t)255u);
    w.total = (uint32_t *)p;
    w.seq = (uint2 *)(p + 256u);
    w.chunk = (uint4 *)((char *)w.seq + up256(8u * (uint64_t)count));
    w.data = (char *)w.chunk + up256(16u * n);
    w.key_bytes = 768u * a.key_width;
    w.value_at = w.key_bytes * a.key_heads;
    w.value_bytes = kMat * (delta ? 2u : 1u) + kRowF * 4u;
    w.chunk_bytes = w.value_at + (uint64_t)w.value_bytes * a.value_heads;
    /* room for the delta form, which the sizes alone do not tell */
    *bytes = 512u + up256(8u * (uint64_t)count) + up256(16u * n) +
             n * (w.value_at + (uint64_t)(2u * kMat + kRowF * 4u) * a.value_heads);
    return w;
}

template <int DK, bool DELTA>
hipError_t run(const kq_launch_linattn &a, const kq_launch_seqs &q, const Work &w, uint32_t chunks,
               uint32_t *status, hipStream_t s) {
    hipLaunchKernelGGL(HIP_KERNEL_NAME(linattn_prep<DK, DELTA>), dim3(chunks, a.key_heads),
                       dim3(256), 0, s, a, w, status);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(linattn_scan<DK, DELTA>),
                       dim3(a.value_heads * (a.value_width / kTile), q.count), dim3(256), 0, s, a,
                       q, w, status);
    return hipGetLastError();
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
    const Work w = carve(a, q.tokens, q.count, max_rows, scratch, &bytes);
    const uint32_t chunks = (uint32_t)most_chunks(q.tokens, q.count, max_rows);
    hipLaunchKernelGGL(linattn_plan, dim3(1), dim3(kPlanThreads), 0, s, q, max_rows, w);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const bool delta = a.beta != nullptr;
    if (a.key_width == 128u)
        return delta ? run<128, true>(a, q, w, chunks, status, s)
                     : run<128, false>(a, q, w, chunks, status, s);
    return delta ? run<64, true>(a, q, w, chunks, status, s)
                 : run<64, false>(a, q, w, chunks, status, s);
}

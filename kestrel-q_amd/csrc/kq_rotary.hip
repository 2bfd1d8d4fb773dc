/*
 * kq_rotary.hip — rotary positions, and rows appended to a paged cache, on
 * gfx950 (include/kq_hip.h, kq_hip_rotary_f32 and kq_hip_cache_append_f32).
 *
 *   y_i = m (x_i cos a - x_j sin a),  y_j = m (x_i sin a + x_j cos a)
 *
 * a = position x frequency. The angle's quarter turns are formed in binary64
 * (a position of 2^20 has 2^-33 of a turn left then, where binary32 would
 * have 2^-4), their fraction, at most 1/2, is rounded once to binary32, and
 * sine and cosine of the eighth turn are their series, 2^-27 off.
 *
 * Bound by memory: 3 operations a value of 8 bytes moved. A workgroup forms
 * the cosines and sines of its tokens once, in LDS, for all heads; a thread
 * takes the same 8 values of a head (4 pairs) of kTokens tokens at once, so
 * that their loads are under way together.
 */
#include "kq_device.h"
#include "kq_launch.h"
#include "kq_paged.h"

namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kTokens = 4; /* of a workgroup: a wave looks up each */
constexpr uint32_t kMaxHalf = 512;

struct Turn {
    float c, s;
};

/* cos and sin of position x frequency radians, times m */
__device__ __forceinline__ Turn turn_of(uint32_t position, double frequency, float m) {
    const double quarters = (double)position * (frequency * 0.63661977236758134308);
    const double whole = rint(quarters);
    const float r = (float)((quarters - whole) * 1.57079632679489661923); /* -pi/4 .. pi/4 */
    const float z = r * r;
    /* the series of sine and cosine; the next terms are below 2^-29 */
    float s = fmaf(z, 2.755731922e-6f, -1.984126984e-4f);
    s = fmaf(z, s, 8.333333333e-3f);
    s = fmaf(z, s, -1.666666667e-1f);
    s = fmaf(z * r, s, r);
    float c = fmaf(z, -2.755731922e-7f, 2.480158730e-5f);
    c = fmaf(z, c, -1.388888889e-3f);
    c = fmaf(z, c, 4.166666667e-2f);
    c = fmaf(z * z, c, fmaf(z, -0.5f, 1.0f));
    /* whole quarters modulo 4: of up to 2^32 positions and any frequency */
    const int n = (int)(whole - 4.0 * floor(whole * 0.25));
    Turn t;
    t.c = (n & 1) ? s : c;
    t.s = (n & 1) ? c : s;
    t.c = (n == 1 || n == 2) ? -t.c : t.c;
    t.s = (n >= 2) ? -t.s : t.s;
    t.c *= m;
    t.s *= m;
    return t;
}

/* V neighbouring values */
template <int V>
struct Vec {
    float v[V];
    __device__ __forceinline__ void load(const float *p) {
        if constexpr (V == 4) {
            const float4 q = *(const float4 *)p;
            v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
        } else {
            v[0] = *p;
        }
    }
    __device__ __forceinline__ bool finite() const {
        bool ok = true;
#pragma unroll
        for (int i = 0; i < V; ++i) ok &= kq_isfinite(v[i]);
        return ok;
    }
};

/* where results go: fp32 rows */
struct ToRows {
    template <int V>
    __device__ __forceinline__ void store(float *p, const Vec<V> &x, bool &bad) const {
        if constexpr (V == 4)
            *(float4 *)p = make_float4(x.v[0], x.v[1], x.v[2], x.v[3]);
        else
            *p = x.v[0];
        bad |= !x.finite();
    }
};

/* or a page, rounded to its type */
template <typename T>
struct ToPage {
    template <int V>
    __device__ __forceinline__ void store(T *p, const Vec<V> &x, bool &bad) const {
        typedef T tv __attribute__((ext_vector_type(V)));
        tv r;
        bool ok = true;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            r[i] = (T)x.v[i];
            ok &= kq_isfinite((float)r[i]);
        }
        bad |= !ok;
        *(tv *)p = r;
    }
};

/* The cosines and sines of tokens [0, n) of the workgroup at their positions */
__device__ __forceinline__ void make_turns(const kq_launch_rotary &r, uint32_t n,
                                           const uint32_t *position, float (*co)[kMaxHalf],
                                           float (*si)[kMaxHalf], bool &badin) {
    const uint32_t half = r.dims / 2u;
    for (uint32_t i = threadIdx.x; i < half; i += kThreads) {
        const double f = r.frequencies[i];
        badin |= !isfinite(f);
        for (uint32_t t = 0; t < n; ++t) {
            const Turn c = turn_of(position[t], f, r.magnitude);
            co[t][i] = c.c;
            si[t][i] = c.s;
        }
    }
}

/* Heads of up to kTokens rows, turned: from[t] a row's heads, to(t, head) where
 * the head goes; NULL rows are left out. A unit is V pairs (2 V values), or V
 * values that are passed on. */
template <int V, typename Out, typename To>
__device__ __forceinline__ void turn_heads(const kq_launch_rotary &r, uint32_t heads,
                                           uint32_t width, const float *const (&from)[kTokens],
                                           const Out &out, To to, const float (*co)[kMaxHalf],
                                           const float (*si)[kMaxHalf], bool &badin, bool &bad) {
    const uint32_t half = r.dims / 2u;
    const uint32_t turned = half / V, units = turned + (width - r.dims) / V;
    for (uint32_t u = threadIdx.x; u < heads * units; u += kThreads) {
        const uint32_t head = u / units, k = u - head * units;
        const uint32_t base = head * width;
        if (k < turned) {
            const uint32_t a = r.pairs ? 2u * V * k : V * k;
            const uint32_t b = r.pairs ? a + V : a + half;
            Vec<V> x[kTokens], y[kTokens];
#pragma unroll
            for (uint32_t t = 0; t < kTokens; ++t)
                if (from[t] != nullptr) {
                    x[t].load(from[t] + base + a);
                    y[t].load(from[t] + base + b);
                }
#pragma unroll
            for (uint32_t t = 0; t < kTokens; ++t) {
                if (from[t] == nullptr) continue;
                badin |= !x[t].finite() || !y[t].finite();
                Vec<V> c, s, p, q;
                c.load(&co[t][V * k]);
                s.load(&si[t][V * k]);
                if (r.pairs && V > 1) {
                    /* x, y: pairs side by side */
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float e = i < V / 2 ? x[t].v[(2 * i) % V] : y[t].v[(2 * i) % V];
                        const float o = i < V / 2 ? x[t].v[(2 * i + 1) % V] : y[t].v[(2 * i + 1) % V];
                        const float re = fmaf(e, c.v[i], -(o * s.v[i]));
                        const float im = fmaf(e, s.v[i], o * c.v[i]);
                        if (i < V / 2) {
                            p.v[(2 * i) % V] = re;
                            p.v[(2 * i + 1) % V] = im;
                        } else {
                            q.v[(2 * i) % V] = re;
                            q.v[(2 * i + 1) % V] = im;
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        p.v[i] = fmaf(x[t].v[i], c.v[i], -(y[t].v[i] * s.v[i]));
                        q.v[i] = fmaf(x[t].v[i], s.v[i], y[t].v[i] * c.v[i]);
                    }
                }
                out.store(to(t, head) + a, p, bad);
                out.store(to(t, head) + b, q, bad);
            }
        } else {
            const uint32_t a = r.dims + (k - turned) * V;
            Vec<V> x[kTokens];
#pragma unroll
            for (uint32_t t = 0; t < kTokens; ++t)
                if (from[t] != nullptr) x[t].load(from[t] + base + a);
#pragma unroll
            for (uint32_t t = 0; t < kTokens; ++t) {
                if (from[t] == nullptr) continue;
                badin |= !x[t].finite();
                out.store(to(t, head) + a, x[t], bad);
            }
        }
    }
}

template <int V>
__global__ __launch_bounds__(kThreads) void rotary_rows(kq_launch_rotary r, uint32_t heads,
                                                        uint32_t width, uint32_t tokens,
                                                        const uint32_t *__restrict__ positions,
                                                        const float *x, uint64_t xs, float *y,
                                                        uint64_t ys, uint32_t *status) {
    __shared__ __attribute__((aligned(16))) float co[kTokens][kMaxHalf], si[kTokens][kMaxHalf];
    const uint32_t t0 = blockIdx.x * kTokens;
    const uint32_t n = tokens - t0 < kTokens ? tokens - t0 : kTokens;
    uint32_t at[kTokens];
    const float *from[kTokens];
    bool badin = false, bad = false;
#pragma unroll
    for (uint32_t t = 0; t < kTokens; ++t) {
        at[t] = t < n ? (positions != nullptr ? positions[t0 + t] : t0 + t) : 0u;
        from[t] = t < n ? x + (size_t)(t0 + t) * xs : nullptr;
    }
    make_turns(r, n, at, co, si, badin);
    __syncthreads();
    turn_heads<V>(
        r, heads, width, from, ToRows{},
        [&](uint32_t t, uint32_t head) { return y + (size_t)(t0 + t) * ys + head * width; }, co, si,
        badin, bad);
    if (badin) kq_flag(status, KQ_DEV_INPUT);
    if (bad) kq_flag(status, KQ_DEV_NUMERIC);
}

template <typename T, int V>
__global__ __launch_bounds__(kThreads) void append_rows(kq_launch_paged c, kq_launch_seqs q,
                                                        kq_launch_append a, kq_launch_rotary r,
                                                        uint32_t *status) {
    __shared__ __attribute__((aligned(16))) float co[kTokens][kMaxHalf], si[kTokens][kMaxHalf];
    __shared__ uint32_t pos_of[kTokens], page_of[kTokens];
    const uint32_t t0 = blockIdx.x * kTokens, tokens = (uint32_t)q.tokens;
    const uint32_t n = tokens - t0 < kTokens ? tokens - t0 : kTokens;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u);
    bool badin = false, bad = false, badseq = false;
    /* wave w: where row t0 + w goes */
    if (wave < kTokens) {
        uint32_t page = ~0u, pos = 0u;
        const uint32_t t = t0 + wave;
        if (wave < n) {
            const uint32_t s = q.offsets != nullptr ? kq::wave_find(q.offsets, q.count, t) : t;
            const kq::PagedSeq sp = kq::paged_seq(q, c, s, badseq);
            if (sp.live && t >= sp.begin && t - sp.begin < sp.rows) {
                pos = sp.past + (t - sp.begin);
                page = c.table[(size_t)sp.slot * c.table_pages + (pos >> c.page_shift)];
                if (page >= c.page_count) {
                    badseq = true;
                    page = ~0u;
                }
            }
        }
        if ((threadIdx.x & 63u) == 0u) {
            pos_of[wave] = pos;
            page_of[wave] = page;
        }
    }
    __syncthreads();
    uint32_t at[kTokens];
    size_t place[kTokens];
    const float *from[kTokens];
    const uint32_t mask = (1u << c.page_shift) - 1u;
    const size_t head_values = (size_t)c.width << c.page_shift;
#pragma unroll
    for (uint32_t t = 0; t < kTokens; ++t) {
        at[t] = pos_of[t];
        const uint32_t page = page_of[t];
        from[t] = page != ~0u ? a.k + (size_t)(t0 + t) * a.ks : nullptr;
        place[t] = page != ~0u ? page * c.heads * head_values + (size_t)(at[t] & mask) * c.width : 0u;
    }
    if (r.dims != 0u) make_turns(r, n, at, co, si, badin);
    __syncthreads();
    turn_heads<V>(
        r, c.heads, c.width, from, ToPage<T>{},
        [&](uint32_t t, uint32_t head) { return (T *)c.keys + place[t] + head * head_values; }, co,
        si, badin, bad);
    if (a.query_heads != 0u) {
#pragma unroll
        for (uint32_t t = 0; t < kTokens; ++t)
            if (from[t] != nullptr) from[t] = a.q + (size_t)(t0 + t) * a.qs;
        turn_heads<V>(
            r, a.query_heads, c.width, from, ToRows{},
            [&](uint32_t t, uint32_t head) {
                return a.qo + (size_t)(t0 + t) * a.qos + head * c.width;
            },
            co, si, badin, bad);
    }
#pragma unroll
    for (uint32_t t = 0; t < kTokens; ++t)
        if (from[t] != nullptr) from[t] = a.v + (size_t)(t0 + t) * a.vs;
    r.dims = 0u;
    turn_heads<4>(
        r, c.heads, c.width, from, ToPage<T>{},
        [&](uint32_t t, uint32_t head) { return (T *)c.values + place[t] + head * head_values; }, co,
        si, badin, bad);
    /* every sequence is looked at, those without rows too, and its slot */
    for (uint32_t s = blockIdx.x; s < q.count; s += gridDim.x) {
        const kq::PagedSeq sp = kq::paged_seq(q, c, s, badseq);
        if (sp.live) badseq |= kq::seq_slot_taken<kThreads>(q, s, sp.slot);
    }
    if (badseq) kq_flag(status, KQ_DEV_SEQUENCE);
    if (badin) kq_flag(status, KQ_DEV_INPUT);
    if (bad) kq_flag(status, KQ_DEV_NUMERIC);
}

}  // namespace

extern "C" hipError_t kq_launch_rotary_rows(const kq_launch_rotary *r, uint32_t heads,
                                            uint32_t width, uint64_t tokens,
                                            const uint32_t *positions, const float *x, uint64_t xs,
                                            float *y, uint64_t ys, uint32_t *status,
                                            hipStream_t s) {
    const bool v4 = r->dims % 8u == 0u && width % 4u == 0u && xs % 4u == 0u && ys % 4u == 0u &&
                    (((uintptr_t)x | (uintptr_t)y) & 15u) == 0u;
    const dim3 grid((uint32_t)((tokens + kTokens - 1u) / kTokens));
    if (v4)
        hipLaunchKernelGGL(HIP_KERNEL_NAME(rotary_rows<4>), grid, dim3(kThreads), 0, s, *r, heads,
                           width, (uint32_t)tokens, positions, x, xs, y, ys, status);
    else
        hipLaunchKernelGGL(HIP_KERNEL_NAME(rotary_rows<1>), grid, dim3(kThreads), 0, s, *r, heads,
                           width, (uint32_t)tokens, positions, x, xs, y, ys, status);
    return hipGetLastError();
}

extern "C" hipError_t kq_launch_cache_append(const kq_launch_paged *c, const kq_launch_seqs *q,
                                             const kq_launch_append *a, const kq_launch_rotary *r,
                                             uint32_t *status, hipStream_t s) {
    const dim3 grid((uint32_t)((q->tokens + kTokens - 1u) / kTokens));
    const bool v4 = r->dims % 8u == 0u;
#define KQ_APPEND(T, V)                                                                          \
    hipLaunchKernelGGL(HIP_KERNEL_NAME(append_rows<T, V>), grid, dim3(kThreads), 0, s, *c, *q, *a, \
                       *r, status)
    if (c->bf16) {
        if (v4)
            KQ_APPEND(__bf16, 4);
        else
            KQ_APPEND(__bf16, 1);
    } else {
        if (v4)
            KQ_APPEND(_Float16, 4);
        else
            KQ_APPEND(_Float16, 1);
    }
#undef KQ_APPEND
    return hipGetLastError();
}

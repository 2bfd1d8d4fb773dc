/*
 * kq_rotary.hip — rotary positions, and rows appended to a paged cache, on
 * gfx950 (include/kq_hip.h, kq_hip_rotary_f32 and kq_hip_cache_append_f32).
 *
 *   y_i = m (x_i cos a - x_j sin a),  y_j = m (x_i sin a + x_j cos a)
 *
 * a = position x frequency. The angle's quarter turns are formed in binary64
 * (a position of 2^20 has 2^-33 of a turn left then, where binary32 would
 * have 2^-4), and their fraction, pi/4 at most in radians, goes on as two
 * binary32 numbers: one alone would be 2^-25 off. Sine and cosine are their
 * series, below 2^-27 off and rounded once.
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
constexpr int kTokens = 4; /* of a workgroup: a wave looks up each */
constexpr uint32_t kMaxHalf = 512;

struct Turn {
    float c, s;
};

/* cos and sin of position x frequency radians, times m */
__device__ __forceinline__ Turn turn_of(uint32_t position, double frequency, float m) {
    const double quarters = (double)position * (frequency * 0.63661977236758134308);
    const double whole = rint(quarters);
    const double x = (quarters - whole) * 1.57079632679489661923; /* -pi/4 .. pi/4 */
    const float r = (float)x, d = (float)(x - (double)r);
    const float z = r * r, e = fmaf(r, r, -z); /* r^2 = z + e */
    /* the series of sine and cosine; the next terms are below 2^-29 */
    float s = fmaf(z, 2.755731922e-6f, -1.984126984e-4f);
    s = fmaf(z, s, 8.333333333e-3f);
    s = fmaf(z, s, -1.666666667e-1f);
    const float h = fmaf(z, -0.5f, 1.0f); /* its rounding is put back */
    s = r + fmaf(z * r, s, h * d);
    float c = fmaf(z, -2.755731922e-7f, 2.480158730e-5f);
    c = fmaf(z, c, -1.388888889e-3f);
    c = fmaf(z, c, 4.166666667e-2f);
    c = h + fmaf(z * z, c, fmaf(-r, d, fmaf(e, -0.5f, fmaf(z, -0.5f, 1.0f - h))));
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
    typedef float fv __attribute__((ext_vector_type(V)));
    float v[V];
    __device__ __forceinline__ void load(const float *p) {
        *this = __builtin_bit_cast(Vec<V>, *(const fv *)p);
    }
    __device__ __forceinline__ bool finite() const {
        bool ok = true;
#pragma unroll
        for (int i = 0; i < V; ++i) ok &= kq_isfinite(v[i]);
        return ok;
    }
};

/* Results go past the caches: what reads them next runs on other XCDs, and the
 * call's inputs would make room for them (8191 rows of 24 heads of 128: 56 us
 * where ordinary stores took 71). Rows are fp32, pages of the cache's type. */
template <int V, typename T>
__device__ __forceinline__ void store(T *p, const Vec<V> &x, bool &bad) {
    typedef T tv __attribute__((ext_vector_type(V)));
    tv r;
    bool ok = true;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        r[i] = (T)x.v[i];
        ok &= kq_isfinite((float)r[i]);
    }
    bad |= !ok;
    __builtin_nontemporal_store(r, (tv *)p);
}

/* The cosines and sines of n tokens at their positions */
template <int TOK>
struct Turns {
    float c[TOK][kMaxHalf], s[TOK][kMaxHalf];

    template <typename At>
    __device__ __forceinline__ void make(const kq_launch_rotary &r, uint32_t n, At position,
                                         bool &badin) {
        const uint32_t half = r.dims / 2u;
        for (uint32_t i = threadIdx.x; i < n * half; i += kThreads) {
            const uint32_t t = TOK == 1 ? 0u : i / half, k = i - t * half;
            const double f = r.frequencies[k];
            badin |= !isfinite(f);
            const Turn x = turn_of(position(t), f, r.magnitude);
            c[t][k] = x.c;
            s[t][k] = x.s;
        }
    }
};

/* Heads of rows that turn, or are passed on (dims 0), in units: V pairs of two
 * vectors (HALVES), or one vector of V values. The lanes' vectors of a load lie
 * side by side, and the stores' too, which go past the caches. */
struct Heads {
    const float *rows;
    uint64_t stride;
    uint32_t count, width, dims, pairs;
};

/* values that turn in a unit */
template <int V>
__device__ __forceinline__ uint32_t unit_turns(const Heads &h) {
    return V == 1 || !h.pairs ? 2u * V : V;
}
template <int V>
__device__ __forceinline__ uint32_t units_of(const Heads &h) {
    return h.dims / unit_turns<V>(h) + (h.width - h.dims) / V;
}

template <int V>
struct Unit {
    uint32_t head, a, b, turn; /* turn: its first pair, ~0: passed on */
    bool two;

    __device__ __forceinline__ Unit(const Heads &h, uint32_t u) {
        const uint32_t each = units_of<V>(h), values = unit_turns<V>(h), turned = h.dims / values;
        head = u / each;
        const uint32_t k = u - head * each;
        if (k < turned) {
            turn = k * (values / 2u);
            two = values == 2u * V;
            a = h.pairs ? values * k : V * k;
            b = h.pairs ? a + 1u : a + h.dims / 2u;
        } else {
            turn = ~0u;
            two = false;
            a = b = h.dims + (k - turned) * V;
        }
    }
};

template <int V, int TOK>
struct Values {
    Vec<V> a[TOK], b[TOK];

    __device__ __forceinline__ void load(const Heads &h, const Unit<V> &u, uint32_t t0,
                                         uint32_t n) {
        const float *p = h.rows + (size_t)t0 * h.stride + u.head * h.width;
#pragma unroll
        for (uint32_t t = 0; t < TOK; ++t) {
            if (t >= n) break;
            a[t].load(p + t * h.stride + u.a);
            if (u.two) b[t].load(p + t * h.stride + u.b);
        }
    }

    /* the turned values of token t */
    __device__ __forceinline__ void turned(const Unit<V> &u, const Turns<TOK> &turns, uint32_t t,
                                           Vec<V> &p, Vec<V> &q) const {
        if (V > 1 && !u.two) { /* V / 2 pairs side by side */
            Vec<(V + 1) / 2> c, s;
            c.load(&turns.c[t][u.turn]);
            s.load(&turns.s[t][u.turn]);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                const float e = a[t].v[2 * i], o = a[t].v[(2 * i + 1) % V];
                p.v[2 * i] = fmaf(e, c.v[i], -(o * s.v[i]));
                p.v[(2 * i + 1) % V] = fmaf(e, s.v[i], o * c.v[i]);
            }
        } else {
            Vec<V> c, s;
            c.load(&turns.c[t][u.turn]);
            s.load(&turns.s[t][u.turn]);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                p.v[i] = fmaf(a[t].v[i], c.v[i], -(b[t].v[i] * s.v[i]));
                q.v[i] = fmaf(a[t].v[i], s.v[i], b[t].v[i] * c.v[i]);
            }
        }
    }

    /* unit u's values of the n tokens, those that `some` names, to to(t) */
    template <typename Some, typename To>
    __device__ __forceinline__ void put(const Heads &h, const Unit<V> &u, const Turns<TOK> &turns,
                                        uint32_t n, Some some, To to, bool &badin,
                                        bool &bad) const {
#pragma unroll
        for (uint32_t t = 0; t < TOK; ++t) {
            if (t >= n) break;
            if (!some(t)) continue;
            badin |= !a[t].finite() || (u.two && !b[t].finite());
            Vec<V> p = a[t], q = b[t];
            if (u.turn != ~0u) turned(u, turns, t, p, q);
            auto *at = to(t) + (size_t)u.head * h.width;
            store(at + u.a, p, bad);
            if (u.two) store(at + u.b, q, bad);
        }
    }
};

template <int V, int TOK>
__global__ __launch_bounds__(kThreads) void rotary_rows(kq_launch_rotary r, Heads h,
                                                        uint32_t tokens,
                                                        const uint32_t *__restrict__ positions,
                                                        float *y, uint64_t ys, uint32_t *status) {
    __shared__ __attribute__((aligned(16))) Turns<TOK> turns;
    const uint32_t t0 = blockIdx.x * TOK;
    const uint32_t n = tokens - t0 < TOK ? tokens - t0 : TOK;
    const uint32_t units = h.count * units_of<V>(h);
    bool badin = false, bad = false;
    uint32_t at = blockIdx.y * kThreads + threadIdx.x;
    const uint32_t step = gridDim.y * kThreads;
    Values<V, TOK> x;
    /* the first values are under way while the turns are formed */
    if (at < units) x.load(h, Unit<V>(h, at), t0, n);
    turns.make(
        r, n, [&](uint32_t t) { return positions != nullptr ? positions[t0 + t] : t0 + t; }, badin);
    __syncthreads();
    while (at < units) {
        const Unit<V> u(h, at);
        x.put(
            h, u, turns, n, [](uint32_t) { return true; },
            [&](uint32_t t) { return y + (size_t)(t0 + t) * ys; }, badin, bad);
        at += step;
        if (at < units) x.load(h, Unit<V>(h, at), t0, n);
    }
    if (badin) kq_flag(status, KQ_DEV_INPUT);
    if (bad) kq_flag(status, KQ_DEV_NUMERIC);
}

/* Keys, then queries, then values of a row. Where a row goes hangs on its
 * sequence, slot, length and page, one load after the other: the first values
 * are asked for before. */
template <typename T, int V, int TOK>
__global__ __launch_bounds__(kThreads) void append_rows(kq_launch_paged c, kq_launch_seqs q,
                                                        kq_launch_append a, kq_launch_rotary r,
                                                        uint32_t *status) {
    __shared__ __attribute__((aligned(16))) Turns<TOK> turns;
    __shared__ uint32_t pos_of[TOK], page_of[TOK];
    const uint32_t t0 = blockIdx.x * TOK, tokens = (uint32_t)q.tokens;
    const uint32_t n = tokens - t0 < TOK ? tokens - t0 : TOK;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u);
    const Heads keys = {a.k, a.ks, c.heads, c.width, r.dims, r.pairs};
    const Heads queries = {a.q, a.qs, a.query_heads, c.width, r.dims, r.pairs};
    const Heads values = {a.v, a.vs, c.heads, c.width, 0u, 0u};
    const uint32_t nk = c.heads * units_of<V>(keys), nq = nk + a.query_heads * units_of<V>(queries);
    const uint32_t units = nq + c.heads * units_of<V>(values);
    bool badin = false, bad = false, badseq = false;
    uint32_t at = blockIdx.y * kThreads + threadIdx.x;
    const uint32_t step = gridDim.y * kThreads;
    Values<V, TOK> x;
    auto load = [&]() {
        if (at < nk)
            x.load(keys, Unit<V>(keys, at), t0, n);
        else if (at < nq)
            x.load(queries, Unit<V>(queries, at - nk), t0, n);
        else if (at < units)
            x.load(values, Unit<V>(values, at - nq), t0, n);
    };
    load();
    /* wave w: where row t0 + w goes */
    if (wave < TOK) {
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
    if (r.dims != 0u) turns.make(r, n, [&](uint32_t t) { return pos_of[t]; }, badin);
    __syncthreads();
    const uint32_t mask = (1u << c.page_shift) - 1u;
    const size_t head_values = (size_t)c.width << c.page_shift;
    auto some = [&](uint32_t t) { return page_of[t] != ~0u; };
    while (at < units) {
        if (at < nk || at >= nq) {
            const Heads &h = at < nk ? keys : values;
            const Unit<V> u(h, at < nk ? at : at - nq);
            T *pool = (T *)(at < nk ? c.keys : c.values) + u.head * (head_values - c.width);
            x.put(
                h, u, turns, n, some,
                [&](uint32_t t) {
                    return pool + (size_t)page_of[t] * c.heads * head_values +
                           (size_t)(pos_of[t] & mask) * c.width;
                },
                badin, bad);
        } else {
            x.put(
                queries, Unit<V>(queries, at - nk), turns, n, some,
                [&](uint32_t t) { return a.qo + (size_t)(t0 + t) * a.qos; }, badin, bad);
        }
        at += step;
        load();
    }
    /* every sequence is looked at, those without rows too, and its slot */
    if (blockIdx.y == 0u)
        for (uint32_t s = blockIdx.x; s < q.count; s += gridDim.x) {
            const kq::PagedSeq sp = kq::paged_seq(q, c, s, badseq);
            if (sp.live) badseq |= kq::seq_slot_taken<kThreads>(q, s, sp.slot);
        }
    if (badseq) kq_flag(status, KQ_DEV_SEQUENCE);
    if (badin) kq_flag(status, KQ_DEV_INPUT);
    if (bad) kq_flag(status, KQ_DEV_NUMERIC);
}

/* Tokens of a workgroup: one while that does not fill the device (61 rows of 20
 * heads: 4.6 us, 10.2 with four), then four, whose turns are formed together.
 * Beside each other in y, workgroups for the row's values, so that a thread has
 * few to walk through: 8191 rows of 24 heads take 38.2 us, 5.3 TB/s, where one
 * workgroup for them took 43; 4099 rows of 48 heads into pages 40.3, 4.6 TB/s,
 * and 46. */
struct Shape {
    bool one;
    dim3 grid;
};
Shape shape_of(uint64_t tokens, uint64_t units) {
    Shape s;
    s.one = tokens < 1024u;
    const uint64_t across = (units + kThreads - 1u) / kThreads, most = s.one ? 8u : 4u;
    s.grid = dim3((uint32_t)(s.one ? tokens : (tokens + kTokens - 1u) / kTokens),
                  (uint32_t)(across < most ? across : most));
    return s;
}

/* Whether the turned part is made of units of four values, of which a thread takes
 * one, in HALVES one of each half. Others go value by value: 8191 rows of 24 heads
 * of 128 with 58 turned 58.5 us (in pairs 54.5), with 64 47.5 (38.8); 4099 rows of 48
 * heads into pages with 58 turned 60.4 (60.8), with 128 41.5. */
bool whole_vectors(const kq_launch_rotary &r) { return r.dims % (r.pairs ? 4u : 8u) == 0u; }

}  // namespace

extern "C" hipError_t kq_launch_rotary_rows(const kq_launch_rotary *r, uint32_t heads,
                                            uint32_t width, uint64_t tokens,
                                            const uint32_t *positions, const float *x, uint64_t xs,
                                            float *y, uint64_t ys, uint32_t *status,
                                            hipStream_t s) {
    const bool v4 = whole_vectors(*r) && width % 4u == 0u && xs % 4u == 0u && ys % 4u == 0u &&
                    (((uintptr_t)x | (uintptr_t)y) & 15u) == 0u;
    const Heads h = {x, xs, heads, width, r->dims, r->pairs};
    const Shape g = shape_of(tokens, (uint64_t)heads * width / (v4 ? 4u : 1u));
#define KQ_ROTARY(V, TOK)                                                                          \
    hipLaunchKernelGGL(HIP_KERNEL_NAME(rotary_rows<V, TOK>), g.grid, dim3(kThreads), 0, s, *r, h,  \
                       (uint32_t)tokens, positions, y, ys, status)
    if (g.one) {
        if (v4)
            KQ_ROTARY(4, 1);
        else
            KQ_ROTARY(1, 1);
    } else {
        if (v4)
            KQ_ROTARY(4, kTokens);
        else
            KQ_ROTARY(1, kTokens);
    }
#undef KQ_ROTARY
    return hipGetLastError();
}

namespace {

template <typename T>
hipError_t append(const kq_launch_paged &c, const kq_launch_seqs &q, const kq_launch_append &a,
                  const kq_launch_rotary &r, uint32_t *status, hipStream_t s) {
    const bool v4 = whole_vectors(r);
    const Shape g =
        shape_of(q.tokens, (uint64_t)(2u * c.heads + a.query_heads) * c.width / (v4 ? 4u : 1u));
#define KQ_APPEND(V, TOK)                                                                         \
    hipLaunchKernelGGL(HIP_KERNEL_NAME(append_rows<T, V, TOK>), g.grid, dim3(kThreads), 0, s, c,  \
                       q, a, r, status)
    if (g.one) {
        if (v4)
            KQ_APPEND(4, 1);
        else
            KQ_APPEND(1, 1);
    } else {
        if (v4)
            KQ_APPEND(4, kTokens);
        else
            KQ_APPEND(1, kTokens);
    }
#undef KQ_APPEND
    return hipGetLastError();
}

}  // namespace

extern "C" hipError_t kq_launch_cache_append(const kq_launch_paged *c, const kq_launch_seqs *q,
                                             const kq_launch_append *a, const kq_launch_rotary *r,
                                             uint32_t *status, hipStream_t s) {
    return c->bf16 ? append<__bf16>(*c, *q, *a, *r, status, s)
                   : append<_Float16>(*c, *q, *a, *r, status, s);
}

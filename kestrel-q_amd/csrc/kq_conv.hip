/*
 * kq_conv.hip — causal depthwise convolution of sequences on gfx950
 * (include/kq_hip.h, kq_hip_causal_conv_f32).
 *
 *   y_t[c] = act(bias[c] + sum_j w[c][j] x_(t - (K-1) + j)[c]),  K taps,
 *
 * the rows before a sequence's first from its state, oldest first. A thread
 * holds V neighbouring channels and walks a block of rows with the last K-1
 * inputs in registers, so that each input is read once (plus K-1 rows at a
 * walk's start, from a cache). Bound by memory: 2 K operations and a sigmoid
 * for a value of 8 bytes moved. 4097 rows of 10,240 channels take 66 us, 5.1
 * TB/s, what a large copy reaches; walks of 32 rows 5 us more, of 64 rows 9
 * (fewer loads under way). One row a sequence, 32 x 10,240: 4.4 us, mostly the
 * launch.
 *
 * A state may be written in place. Everything that reads it is therefore
 * done by the workgroup that also writes it: those of a sequence take its
 * first K-1 rows and write the state behind its last (inputs, or what is left
 * of the old state). Those of a block of rows take all others, whatever
 * sequences they belong to, and read inputs only. One launch has both, the
 * sequences' first, so that many short sequences run side by side.
 */
#include "kq_device.h"
#include "kq_launch.h"
#include "kq_seq.h"

namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 8; /* rows that a walk reads at a time */
constexpr uint32_t kRows = 16; /* rows of a walk */
constexpr uint32_t kParts = 1u << 15;

typedef float f4 __attribute__((ext_vector_type(4)));

template <int V>
struct Vec {
    float v[V];
};

template <int V>
__device__ __forceinline__ Vec<V> load(const float *p) {
    Vec<V> r;
    if constexpr (V == 4) {
        const float4 q = *(const float4 *)p;
        r.v[0] = q.x; r.v[1] = q.y; r.v[2] = q.z; r.v[3] = q.w;
    } else {
        r.v[0] = *p;
    }
    return r;
}

template <int V>
__device__ __forceinline__ void store(float *p, const Vec<V> &r) {
    if constexpr (V == 4)
        *(float4 *)p = make_float4(r.v[0], r.v[1], r.v[2], r.v[3]);
    else
        *p = r.v[0];
}

/* the next launch reads these rows, from other XCDs' caches as a rule: not
 * kept in this one's (for 4097 rows of 10,240 channels 7 us less) */
template <int V>
__device__ __forceinline__ void store_nt(float *p, const Vec<V> &r) {
    if constexpr (V == 4)
        __builtin_nontemporal_store(__builtin_bit_cast(f4, r), (f4 *)p);
    else
        __builtin_nontemporal_store(r.v[0], p);
}

template <int V>
__device__ __forceinline__ bool finite(const Vec<V> &r) {
    bool ok = true;
#pragma unroll
    for (int i = 0; i < V; ++i) ok &= kq_isfinite(r.v[i]);
    return ok;
}

/* the weights and the bias of V channels */
template <int K, int V>
struct Taps {
    float w[K][V], b[V];
    __device__ __forceinline__ bool load(const kq_launch_conv &c, uint32_t ch) {
        bool ok = true;
#pragma unroll
        for (int i = 0; i < V; ++i) {
#pragma unroll
            for (int j = 0; j < K; ++j) {
                w[j][i] = c.weight[(size_t)(ch + i) * K + j];
                ok &= kq_isfinite(w[j][i]);
            }
            b[i] = c.bias != nullptr ? c.bias[ch + i] : 0.0f;
            ok &= kq_isfinite(b[i]);
        }
        return ok;
    }
    /* hist: the K-1 inputs before x, oldest first */
    __device__ __forceinline__ Vec<V> apply(const Vec<V> (&hist)[K - 1], const Vec<V> &x,
                                            bool silu) const {
        Vec<V> y;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float s = b[i];
#pragma unroll
            for (int j = 0; j < K - 1; ++j) s = fmaf(w[j][i], hist[j].v[i], s);
            s = fmaf(w[K - 1][i], x.v[i], s);
            y.v[i] = silu ? s * kq::sigmoid(s) : s;
        }
        return y;
    }
};

/* the state behind n rows from x on: entry n + j of [the old state, the rows] */
template <int K, int V>
__device__ __forceinline__ void write_state(const Vec<V> (&old)[K - 1], const float *x,
                                            uint64_t xs, uint32_t n, float *to, uint32_t channels) {
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
        Vec<V> v = old[j];
        if (n + j >= (uint32_t)(K - 1)) {
            v = load<V>(x + (size_t)(n + j - (K - 1)) * xs);
        } else {
#pragma unroll
            for (int k = 0; k < K - 1; ++k)
                if (n + j == (uint32_t)k) v = old[k];
        }
        store(to + (size_t)j * channels, v);
    }
}

template <int K, int V>
__device__ __forceinline__ void read_state(Vec<V> (&old)[K - 1], bool fresh, const float *from,
                                           uint32_t channels) {
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
        if (fresh) {
#pragma unroll
            for (int i = 0; i < V; ++i) old[j].v[i] = 0.0f;
        } else {
            old[j] = load<V>(from + (size_t)j * channels);
        }
    }
}

/* the first K-1 rows of a sequence (or what it has), and its state */
template <int K, int V>
__device__ __forceinline__ void head_rows(const kq_launch_conv &c, const kq::SeqSpan &sp,
                                          uint32_t ch, const float *x, uint64_t xs,
                                          const float *state, float *state_out, float *y,
                                          uint64_t ys, const Taps<K, V> &w, bool &badin,
                                          bool &bad) {
    const size_t at = (size_t)sp.slot * (K - 1) * c.channels + ch;
    x += (size_t)sp.begin * xs + ch;
    y += (size_t)sp.begin * ys + ch;
    Vec<V> in[K - 1], hist[K - 1];
    read_state<K, V>(hist, sp.fresh, state + at, c.channels);
    if (sp.rows != 0u)
#pragma unroll
        for (int j = 0; j < K - 1; ++j)
            in[j] = load<V>(x + (j < (int)sp.rows ? (size_t)j * xs : 0u));
#pragma unroll
    for (int j = 0; j < K - 1; ++j) badin |= !finite(hist[j]); /* passed on, without rows */
    write_state<K, V>(hist, x, xs, sp.rows, state_out + at, c.channels);
#pragma unroll
    for (int t = 0; t < K - 1; ++t) {
        if (t >= (int)sp.rows) break;
        badin |= !finite(in[t]);
        const Vec<V> out = w.apply(hist, in[t], c.silu != 0u);
        bad |= !finite(out);
        store(y + (size_t)t * ys, out);
#pragma unroll
        for (int j = 0; j + 1 < K - 1; ++j) hist[j] = hist[j + 1];
        hist[K - 2] = in[t];
    }
}

/* grid: channel groups x (sequences, then blocks of kRows rows of the token
 * array), the latter in y and z, kParts of them in y */
template <int K, int V>
__global__ __launch_bounds__(kThreads) void conv_rows(kq_launch_conv c, kq_launch_seqs q,
                                                      const float *__restrict__ x, uint64_t xs,
                                                      const float *state, float *state_out,
                                                      float *__restrict__ y, uint64_t ys,
                                                      uint32_t *status) {
    const uint32_t part = blockIdx.z * kParts + blockIdx.y;
    const uint32_t ch = (blockIdx.x * kThreads + threadIdx.x) * V;
    const bool mine = ch < c.channels;
    bool badin = false, bad = false, badseq = false;
    Taps<K, V> w;
    if (mine) badin |= !w.load(c, ch);
    if (part < q.count) {
        const kq::SeqSpan sp = kq::seq_span(q, part, badseq);
        if (sp.live && mine)
            head_rows<K, V>(c, sp, ch, x, xs, state, state_out, y, ys, w, badin, bad);
        if (sp.live && blockIdx.x == 0u) badseq |= kq::seq_slot_taken<kThreads>(q, part, sp.slot);
    } else {
        const uint32_t tokens = (uint32_t)q.tokens;
        const uint32_t t0 = (part - q.count) * kRows; /* past the rows: none to do */
        const uint32_t t1 = t0 + kRows < tokens ? t0 + kRows : tokens;
        /* the last sequence that begins before t0: each wave counts them */
        uint32_t s = 0u;
        const uint32_t lane = threadIdx.x & 63u;
        for (uint32_t base = 0u; base < q.count; base += 64u) {
            const uint64_t m = __ballot(base + lane < q.count && q.offsets[base + lane] < t0);
            s += (uint32_t)__popcll(m);
            if (m != ~0ull) break;
        }
        s = __builtin_amdgcn_readfirstlane(s > 0u ? s - 1u : 0u);
        for (; mine && s < q.count && q.offsets[s] < t1; ++s) {
            bool skip = false; /* its own workgroups say so */
            const kq::SeqSpan sp = kq::seq_span(q, s, skip);
            if (!sp.live || sp.rows < (uint32_t)K) continue;
            const uint32_t from = sp.begin + (uint32_t)(K - 1), to = sp.begin + sp.rows;
            const uint32_t first = from > t0 ? from : t0, end = to < t1 ? to : t1;
            if (first >= end) continue;
            Vec<V> hist[K - 1];
#pragma unroll
            for (int j = 0; j < K - 1; ++j)
                hist[j] = load<V>(x + (size_t)(first - (K - 1) + j) * xs + ch);
            for (uint32_t t = first; t < end; t += kBatch) {
                Vec<V> in[kBatch]; /* all under way before the first is used */
#pragma unroll
                for (int i = 0; i < kBatch; ++i)
                    in[i] = load<V>(x + (size_t)(t + i < end ? t + i : end - 1u) * xs + ch);
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    if (t + i >= end) break;
                    badin |= !finite(in[i]);
                    const Vec<V> out = w.apply(hist, in[i], c.silu != 0u);
                    bad |= !finite(out);
                    store_nt(y + (size_t)(t + i) * ys + ch, out);
#pragma unroll
                    for (int j = 0; j + 1 < K - 1; ++j) hist[j] = hist[j + 1];
                    hist[K - 2] = in[i];
                }
            }
        }
    }
    if (badseq) kq_flag(status, KQ_DEV_SEQUENCE);
    if (badin) kq_flag(status, KQ_DEV_INPUT);
    if (bad) kq_flag(status, KQ_DEV_NUMERIC);
}

/* grid (channel groups, sequences): one row a sequence */
template <int K, int V>
__global__ __launch_bounds__(kThreads) void conv_step(kq_launch_conv c, kq_launch_seqs q,
                                                      const float *__restrict__ x, uint64_t xs,
                                                      const float *state, float *state_out,
                                                      float *__restrict__ y, uint64_t ys,
                                                      uint32_t *status) {
    const uint32_t s = blockIdx.y;
    bool badseq = false, badin = false, bad = false;
    const kq::SeqSpan sp = kq::seq_span(q, s, badseq);
    const uint32_t ch = (blockIdx.x * kThreads + threadIdx.x) * V;
    if (sp.live && ch < c.channels) {
        const size_t at = (size_t)sp.slot * (K - 1) * c.channels + ch;
        const Vec<V> in = load<V>(x + (size_t)sp.begin * xs + ch);
        Vec<V> hist[K - 1];
        read_state<K, V>(hist, sp.fresh, state + at, c.channels);
        Taps<K, V> w;
        badin |= !w.load(c, ch);
        badin |= !finite(in);
#pragma unroll
        for (int j = 0; j < K - 1; ++j) badin |= !finite(hist[j]);
        const Vec<V> out = w.apply(hist, in, c.silu != 0u);
        bad |= !finite(out);
        store(y + (size_t)sp.begin * ys + ch, out);
#pragma unroll
        for (int j = 0; j < K - 1; ++j)
            store(state_out + at + (size_t)j * c.channels, j + 1 < K - 1 ? hist[j + 1] : in);
    }
    if (sp.live && blockIdx.x == 0u) badseq |= kq::seq_slot_taken<kThreads>(q, s, sp.slot);
    if (badseq) kq_flag(status, KQ_DEV_SEQUENCE);
    if (badin) kq_flag(status, KQ_DEV_INPUT);
    if (bad) kq_flag(status, KQ_DEV_NUMERIC);
}

template <int K, int V>
hipError_t run(const kq_launch_conv &c, const kq_launch_seqs &q, const float *x, uint64_t xs,
               const float *state, float *state_out, float *y, uint64_t ys, uint32_t *status,
               hipStream_t s) {
    const uint32_t groups = (c.channels / V + kThreads - 1) / kThreads;
    if (q.offsets == nullptr) {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(conv_step<K, V>), dim3(groups, q.count),
                           dim3(kThreads), 0, s, c, q, x, xs, state, state_out, y, ys, status);
        return hipGetLastError();
    }
    const uint32_t parts = q.count + (uint32_t)((q.tokens + kRows - 1) / kRows);
    const dim3 grid(groups, parts < kParts ? parts : kParts, (parts + kParts - 1) / kParts);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(conv_rows<K, V>), grid, dim3(kThreads), 0, s, c, q, x, xs,
                       state, state_out, y, ys, status);
    return hipGetLastError();
}

}  // namespace

extern "C" hipError_t kq_launch_causal_conv(const kq_launch_conv *c, const kq_launch_seqs *q,
                                            const float *x, uint64_t xs, const float *state,
                                            float *state_out, float *y, uint64_t ys,
                                            uint32_t *status, hipStream_t s) {
    const bool v4 = c->channels % 4u == 0u && xs % 4u == 0u && ys % 4u == 0u &&
                    (((uintptr_t)x | (uintptr_t)state | (uintptr_t)state_out | (uintptr_t)y) &
                     15u) == 0u;
    switch (c->taps) {
#define KQ_TAPS(K)                                                                             \
    case K:                                                                                    \
        return v4 ? run<K, 4>(*c, *q, x, xs, state, state_out, y, ys, status, s)               \
                  : run<K, 1>(*c, *q, x, xs, state, state_out, y, ys, status, s);
        KQ_TAPS(2)
        KQ_TAPS(3)
        KQ_TAPS(4)
        KQ_TAPS(5)
        KQ_TAPS(6)
        KQ_TAPS(7)
        KQ_TAPS(8)
#undef KQ_TAPS
    default: return hipErrorInvalidValue;
    }
}

/*
 * kq_conv.hip — causal depthwise convolution of sequences on gfx950
 * (include/kq_hip.h, kq_hip_causal_conv_f32).
 *
 *   y_t[c] = act(bias[c] + sum_j w[c][j] x_(t - (K-1) + j)[c]),  K taps,
 *
 * the rows before a sequence's first from its state, oldest first. A thread
 * holds V neighbouring channels and walks kRows rows with the last K-1
 * inputs in registers, so that each input is read once (plus K-1 rows at a
 * walk's start). Bound by memory: 4 (K+1) operations a value of 8 bytes.
 *
 * The states are written by a second launch: a state that is updated in
 * place is read by the walk that holds the sequence's first row, which may
 * run behind the one that holds its last. With one row a sequence the same
 * thread reads and writes it, and one launch does both.
 */
#include "kq_device.h"
#include "kq_launch.h"
#include "kq_seq.h"

namespace {

constexpr int kThreads = 256;

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

/* grid (channel groups, row blocks): rows [blockIdx.y * rows, + rows) of the
 * token array, whatever sequences they belong to */
template <int K, int V>
__global__ __launch_bounds__(kThreads) void conv_rows(kq_launch_conv c, kq_launch_seqs q,
                                                      const float *__restrict__ x, uint64_t xs,
                                                      const float *state, float *__restrict__ y,
                                                      uint64_t ys, uint32_t rows,
                                                      uint32_t *status) {
    const uint32_t t0 = blockIdx.y * rows;
    const uint32_t t1 = t0 + rows < (uint32_t)q.tokens ? t0 + rows : (uint32_t)q.tokens;
    /* the last sequence that begins at or before t0: each wave counts */
    uint32_t s = 0u;
    {
        const uint32_t lane = threadIdx.x & 63u;
        for (uint32_t base = 0u; base < q.count; base += 64u) {
            const bool le = base + lane < q.count && q.offsets[base + lane] <= t0;
            const uint64_t m = __ballot(le);
            s += (uint32_t)__popcll(m);
            if (m != ~0ull) break;
        }
        if (s > 0u) s -= 1u;
        s = __builtin_amdgcn_readfirstlane(s);
    }
    const uint32_t ch = (blockIdx.x * kThreads + threadIdx.x) * V;
    if (ch >= c.channels) return;
    Taps<K, V> w;
    bool badin = !w.load(c, ch), bad = false, badseq = false;
    Vec<V> hist[K - 1];
    for (; s < q.count; ++s) {
        if (q.offsets[s] >= t1) break;
        const kq::SeqSpan sp = kq::seq_span(q, s, badseq);
        if (!sp.live) continue;
        const uint32_t end = sp.begin + sp.rows < t1 ? sp.begin + sp.rows : t1;
        const uint32_t first = sp.begin > t0 ? sp.begin : t0;
        if (first >= end) continue;
#pragma unroll
        for (int j = 0; j < K - 1; ++j) {
            /* the sequence's row that tap j of row `first` reads */
            const int32_t at = (int32_t)(first - sp.begin) - (K - 1) + j;
            if (at >= 0) {
                hist[j] = load<V>(x + (size_t)(sp.begin + at) * xs + ch);
            } else if (sp.fresh) {
#pragma unroll
                for (int i = 0; i < V; ++i) hist[j].v[i] = 0.0f;
            } else {
                hist[j] = load<V>(state + ((size_t)sp.slot * (K - 1) + (size_t)(at + K - 1)) *
                                              c.channels + ch);
                badin |= !finite(hist[j]);
            }
        }
        for (uint32_t t = first; t < end; ++t) {
            const Vec<V> in = load<V>(x + (size_t)t * xs + ch);
            badin |= !finite(in);
            const Vec<V> out = w.apply(hist, in, c.silu != 0u);
            bad |= !finite(out);
            store(y + (size_t)t * ys + ch, out);
#pragma unroll
            for (int j = 0; j + 1 < K - 1; ++j) hist[j] = hist[j + 1];
            hist[K - 2] = in;
        }
    }
    if (badin) kq_flag(status, KQ_DEV_INPUT);
    if (bad) kq_flag(status, KQ_DEV_NUMERIC);
}

/* grid (channel groups, sequences). ROWS: one row a sequence, its output
 * formed here too; otherwise only the state behind the last row. Checks the
 * sequences of the call. */
template <int K, int V, bool ROWS>
__global__ __launch_bounds__(kThreads) void conv_states(kq_launch_conv c, kq_launch_seqs q,
                                                        const float *__restrict__ x, uint64_t xs,
                                                        const float *state, float *state_out,
                                                        float *__restrict__ y, uint64_t ys,
                                                        uint32_t *status) {
    const uint32_t s = blockIdx.y;
    bool badseq = false, badin = false, bad = false;
    const kq::SeqSpan sp = kq::seq_span(q, s, badseq);
    if (blockIdx.x == 0u) {
        if (sp.live) badseq |= kq::seq_slot_taken<kThreads>(q, s, sp.slot);
        if (badseq) kq_flag(status, KQ_DEV_SEQUENCE);
    }
    const uint32_t ch = (blockIdx.x * kThreads + threadIdx.x) * V;
    if (ch >= c.channels || !sp.live) return;
    const size_t at = (size_t)sp.slot * (K - 1) * c.channels + ch;
    Vec<V> hist[K - 1];
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
        if (sp.fresh) {
#pragma unroll
            for (int i = 0; i < V; ++i) hist[j].v[i] = 0.0f;
        } else {
            hist[j] = load<V>(state + at + (size_t)j * c.channels);
        }
    }
    if constexpr (ROWS) {
        Taps<K, V> w;
        badin |= !w.load(c, ch);
        const Vec<V> in = load<V>(x + (size_t)sp.begin * xs + ch);
        badin |= !finite(in);
#pragma unroll
        for (int j = 0; j < K - 1; ++j) badin |= !finite(hist[j]);
        const Vec<V> out = w.apply(hist, in, c.silu != 0u);
        bad |= !finite(out);
        store(y + (size_t)sp.begin * ys + ch, out);
    }
    const uint32_t n = sp.rows;
#pragma unroll
    for (int j = 0; j < K - 1; ++j) {
        /* entry n + j of [the old state, the rows] */
        Vec<V> v;
        if (n + j >= (uint32_t)(K - 1)) {
            v = load<V>(x + (size_t)(sp.begin + (n + j - (K - 1))) * xs + ch);
        } else {
            v = hist[j];
#pragma unroll
            for (int k = 0; k < K - 1; ++k)
                if (n + j == (uint32_t)k) v = hist[k];
        }
        store(state_out + at + (size_t)j * c.channels, v);
    }
    if (badin) kq_flag(status, KQ_DEV_INPUT);
    if (bad) kq_flag(status, KQ_DEV_NUMERIC);
}

template <int K, int V>
hipError_t run(const kq_launch_conv &c, const kq_launch_seqs &q, const float *x, uint64_t xs,
               const float *state, float *state_out, float *y, uint64_t ys, uint32_t *status,
               hipStream_t s) {
    const uint32_t groups = (c.channels / V + kThreads - 1) / kThreads;
    if (q.offsets == nullptr) {
        hipLaunchKernelGGL(HIP_KERNEL_NAME(conv_states<K, V, true>), dim3(groups, q.count),
                           dim3(kThreads), 0, s, c, q, x, xs, state, state_out, y, ys, status);
        return hipGetLastError();
    }
    const uint32_t rows = 16u;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(conv_rows<K, V>),
                       dim3(groups, (uint32_t)((q.tokens + rows - 1) / rows)), dim3(kThreads), 0,
                       s, c, q, x, xs, state, y, ys, rows, status);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(conv_states<K, V, false>), dim3(groups, q.count),
                       dim3(kThreads), 0, s, c, q, x, xs, state, state_out, y, ys, status);
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

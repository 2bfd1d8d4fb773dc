/*
 * kq_norm.hip — norms around a block with its gate and its residual on
 * gfx950 (include/kq_hip.h, kq_hip_gated_norm_f32 and kq_hip_block_join_f32).
 *
 *   rms(x) = x / sqrt(sum x^2 / n + epsilon)
 *
 * Both kernels hold a row in registers between its sum of squares and its
 * scaling, so that memory is read once and written once; a few operations a
 * value leave them bound by memory (or, for few rows, by the launch). Groups
 * of up to 256 values share a workgroup: 4099 rows of 48 heads of 128 with a
 * SiLU gate take 55 us, 5.5 TB/s (a large copy: 5.1). 2499 tokens of 4
 * branches of 2560, gated and with both norms, take 83.5 us: 4.3 TB/s, of
 * which 4 bytes in 7 are written (two branches a workgroup 89 us, the next
 * branch's loads during the norm before it 84.5, a thread for 4 x 4 values in
 * place of 2 x 4 at this width 87.4).
 */
#include "kq_device.h"
#include "kq_launch.h"
#include "kq_seq.h"

namespace {

enum : uint32_t { kNone = 0u, kSigmoid = 1u, kSilu = 2u };

__device__ __forceinline__ float act(uint32_t kind, float g) {
    const float s = kq::sigmoid(g);
    return kind == kSilu ? g * s : s;
}

/* 1 / sqrt(sum / n + eps) where the sum of squares lies in the middle of the
 * type's range. Elsewhere (values so large or small that their squares are
 * not) the squares are formed of x 2^-96 or x 2^96 and the rest in 64 bits.
 * Every thread of a row has the same sum, so all of them take the same way. */
__device__ __forceinline__ bool in_range(float sum) { return sum < 3.0e38f && sum > 1.0e-30f; }

template <int V>
__device__ __forceinline__ void ld(const float *p, float *v) {
    if constexpr (V == 4) {
        const float4 q = *(const float4 *)p;
        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
    } else {
        v[0] = *p;
    }
}
template <int V>
__device__ __forceinline__ void st(float *p, const float *v) {
    if constexpr (V == 4)
        *(float4 *)p = make_float4(v[0], v[1], v[2], v[3]);
    else
        *p = v[0];
}

/* sum over the L threads of a row: L <= 64 neighbouring lanes, or the whole
 * workgroup of L threads */
template <int L>
__device__ __forceinline__ float row_sum(float v, float *red) {
    if constexpr (L <= 64) {
        return kq::lanes_sum<L - 1>(v);
    } else {
        v = kq::lanes_sum<63>(v);
        __syncthreads(); /* earlier readers of red are done */
        if ((threadIdx.x & 63u) == 0u) red[threadIdx.x >> 6] = v;
        __syncthreads();
        float s = 0.0f;
#pragma unroll
        for (int w = 0; w < L / 64; ++w) s += red[w];
        return s;
    }
}

/* the sum of squares of a row's values x[0 .. n) and its inverse root */
template <int L, int N>
__device__ __forceinline__ float row_inverse(const float (&x)[N], uint32_t width, float eps,
                                             float *red) {
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fmaf(x[i], x[i], s);
    s = row_sum<L>(s, red);
    if (in_range(s)) return 1.0f / sqrtf(s / (float)width + eps);
    const float down = s > 1.0f ? 0x1p-96f : 0x1p96f;
    const double up = s > 1.0f ? 0x1p192 : 0x1p-192;
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) s = fmaf(x[i] * down, x[i] * down, s);
    s = row_sum<L>(s, red);
    return (float)(1.0 / sqrt((double)s * up / (double)width + (double)eps));
}

/* A row of `width` values on L threads, P pieces of V values each: thread l
 * has pieces l, l + L, ... */
template <int L, int V, int P>
__global__ __launch_bounds__(L <= 64 ? 256 : L) void gated_norm(kq_launch_norm a, uint64_t rows,
                                                                const float *x, uint64_t xs,
                                                                const float *gate, uint64_t gs,
                                                                float *y, uint64_t ys,
                                                                uint32_t *status) {
    __shared__ float red[L <= 64 ? 1 : L / 64];
    constexpr int kRows = L <= 64 ? 256 / L : 1;
    const uint32_t l = threadIdx.x % L;
    bool badin = false, bad = false;
    for (uint64_t row = (uint64_t)blockIdx.x * kRows + (L <= 64 ? threadIdx.x / L : 0u);
         row < rows; row += (uint64_t)gridDim.x * kRows) { /* the threads of a row together */
        const uint64_t t = row / a.groups;
        const uint32_t g = (uint32_t)(row - t * a.groups);
        const size_t at = (size_t)g * a.width;
        const float *xr = x + (size_t)t * xs + at;
        const float *gr = gate + (a.gate != kNone ? (size_t)t * gs + at : 0u);
        const float *w = a.weight != nullptr ? a.weight + (a.per_group != 0u ? at : 0u) : nullptr;
        float *yr = y + (size_t)t * ys + at;
        float v[P * V], m[P * V], gv[P * V];
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const uint32_t i = (l + p * L) * V;
#pragma unroll
            for (int k = 0; k < V; ++k) v[p * V + k] = 0.0f, m[p * V + k] = 0.0f, gv[p * V + k] = 0.0f;
            if (i < a.width) {
                ld<V>(xr + i, v + p * V);
                if (a.gate != kNone) ld<V>(gr + i, gv + p * V);
                if (w != nullptr) ld<V>(w + i, m + p * V);
            }
        }
#pragma unroll
        for (int k = 0; k < P * V; ++k)
            badin |= !(kq_isfinite(v[k]) && kq_isfinite(m[k]) && kq_isfinite(gv[k]));
        const float inv = row_inverse<L>(v, a.width, a.epsilon, red);
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const uint32_t i = (l + p * L) * V;
            if (i < a.width) {
                float o[V];
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const int j = p * V + k;
                    o[k] = v[j] * inv;
                    if (w != nullptr) o[k] *= a.offset + m[j];
                    if (a.gate != kNone) o[k] *= act(a.gate, gv[j]);
                    bad |= !kq_isfinite(o[k]);
                }
                st<V>(yr + i, o);
            }
        }
    }
    if (badin) kq_flag(status, KQ_DEV_INPUT);
    if (bad) kq_flag(status, KQ_DEV_NUMERIC);
}

/* grid (tokens, branch groups of `per`): a workgroup of L threads forms the
 * block's output y of a token in registers and takes `per` branches to it */
template <int L, int V, int P>
__global__ __launch_bounds__(L) void block_join(kq_launch_join a, uint32_t per,
                                                uint32_t *status) {
    __shared__ float red[L / 64];
    const size_t t = blockIdx.x;
    const uint32_t H = a.hidden, l = threadIdx.x;
    float y[P * V];
    bool badin = false, bad = false;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const uint32_t i = (l + p * L) * V;
#pragma unroll
        for (int k = 0; k < V; ++k) y[p * V + k] = 0.0f;
        if (i < H) ld<V>(a.block + t * H + i, y + p * V);
    }
#pragma unroll
    for (int k = 0; k < P * V; ++k) badin |= !kq_isfinite(y[k]);
    float inv = 1.0f;
    if (a.post != nullptr) inv = row_inverse<L>(y, H, a.epsilon, red);
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const uint32_t i = (l + p * L) * V;
        if (i < H) {
            float m[V], g[V];
            if (a.post != nullptr) {
                ld<V>(a.post + i, m);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    badin |= !kq_isfinite(m[k]);
                    y[p * V + k] = y[p * V + k] * inv * (a.post_offset + m[k]);
                }
            }
            if (a.gate_kind != kNone) {
                ld<V>(a.gate + t * H + i, g);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    badin |= !kq_isfinite(g[k]);
                    y[p * V + k] *= act(a.gate_kind, g[k]);
                }
            }
        }
    }
    for (uint32_t b = blockIdx.y * per; b < a.branches && b < (blockIdx.y + 1u) * per; ++b) {
        const size_t at = (t * a.branches + b) * H;
        const float c = a.branch_gate != nullptr ? a.branch_gate[t * a.branches + b] : 1.0f;
        badin |= !kq_isfinite(c);
        const float cs = a.scale * c;
        float r[P * V];
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const uint32_t i = (l + p * L) * V;
#pragma unroll
            for (int k = 0; k < V; ++k) r[p * V + k] = 0.0f;
            if (i < H) {
                ld<V>(a.residual + at + i, r + p * V);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    badin |= !kq_isfinite(r[p * V + k]);
                    /* a rounded product and a sum: gr_write's bits */
                    r[p * V + k] = r[p * V + k] + cs * y[p * V + k];
                    bad |= !kq_isfinite(r[p * V + k]);
                }
                st<V>(a.residual_out + at + i, r + p * V);
            }
        }
        if (a.pre == nullptr) continue;
        const float rinv = row_inverse<L>(r, H, a.epsilon, red);
        const float *w = a.pre + (size_t)b * H;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const uint32_t i = (l + p * L) * V;
            if (i < H) {
                float m[V], o[V];
                ld<V>(w + i, m);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    badin |= !kq_isfinite(m[k]);
                    o[k] = r[p * V + k] * rinv * (a.pre_offset + m[k]);
                    bad |= !kq_isfinite(o[k]);
                }
                st<V>(a.normalized + at + i, o);
            }
        }
    }
    if (badin) kq_flag(status, KQ_DEV_INPUT);
    if (bad) kq_flag(status, KQ_DEV_NUMERIC);
}

constexpr uint64_t kMaxGrid = 1u << 20; /* workgroups, threads of a launch below 2^32 */

bool by16(const void *p) { return ((uintptr_t)p & 15u) == 0u; }

}  // namespace

extern "C" hipError_t kq_launch_gated_norm(const kq_launch_norm *a, uint64_t tokens,
                                           const float *x, uint64_t xs, const float *gate,
                                           uint64_t gs, float *y, uint64_t ys, uint32_t *status,
                                           hipStream_t s) {
    const uint64_t rows = tokens * a->groups;
    const uint32_t w = a->width;
    const bool gated = a->gate != kNone;
    const bool v4 = w % 4u == 0u && xs % 4u == 0u && ys % 4u == 0u && (!gated || gs % 4u == 0u) &&
                    by16(x) && by16(y) && (!gated || by16(gate)) && by16(a->weight);
#define KQ_NORM(L, V, P)                                                                         \
    do {                                                                                         \
        const uint32_t per = L <= 64 ? 256 / L : 1;                                              \
        const uint64_t need = (rows + per - 1) / per;                                            \
        hipLaunchKernelGGL(HIP_KERNEL_NAME(gated_norm<L, V, P>),                                 \
                           dim3((uint32_t)(need < kMaxGrid ? need : kMaxGrid)),                  \
                           dim3(L <= 64 ? 256 : L), 0,                                           \
                           s, *a, rows, x, xs, gate, gs, y, ys, status);                         \
        return hipGetLastError();                                                                \
    } while (0)
    if (v4) {
        if (w <= 64u) KQ_NORM(16, 4, 1);
        if (w <= 128u) KQ_NORM(32, 4, 1);
        if (w <= 256u) KQ_NORM(64, 4, 1);
        if (w <= 1024u) KQ_NORM(64, 4, 4);
        if (w <= 4096u) KQ_NORM(256, 4, 4);
        KQ_NORM(1024, 4, 4);
    }
    if (w <= 64u) KQ_NORM(64, 1, 1);
    if (w <= 256u) KQ_NORM(64, 1, 4);
    if (w <= 1024u) KQ_NORM(256, 1, 4);
    if (w <= 4096u) KQ_NORM(1024, 1, 4);
    KQ_NORM(1024, 1, 16);
#undef KQ_NORM
}

extern "C" hipError_t kq_launch_block_join(const kq_launch_join *a, uint64_t tokens,
                                           uint32_t *status, hipStream_t s) {
    const uint32_t h = a->hidden;
    const bool v4 = h % 4u == 0u && by16(a->block) && by16(a->post) &&
                    (a->gate_kind == kNone || by16(a->gate)) && by16(a->residual) &&
                    by16(a->residual_out) && by16(a->pre) && by16(a->normalized);
    /* Few tokens: a workgroup for each branch, which forms the block's norm for
     * itself. 4 branches of 2560 with both norms and a gate, a workgroup a
     * branch and one for all of them: 64 tokens 5.6 and 9.8 us, 256 9.8 and 13.5,
     * 384 14.0 and 15.4, 500 18.0 and 15.9, 512 17.1 and 16.0, 1024 41.6 and
     * 33.2. */
    const uint32_t per = tokens >= 512u ? a->branches : 1u;
    const dim3 grid((uint32_t)tokens, (a->branches + per - 1u) / per);
#define KQ_JOIN(L, V, P)                                                                         \
    do {                                                                                         \
        hipLaunchKernelGGL(HIP_KERNEL_NAME(block_join<L, V, P>), grid, dim3(L), 0, s, *a, per,   \
                           status);                                                              \
        return hipGetLastError();                                                                \
    } while (0)
    if (v4) {
        /* 2499 tokens of 4 branches, 256 and 320 threads: 1536 values 56 and 67 us,
         * 2048 65 and 72, 2304 80.5 and 77.9, 2560 87.5 and 83.6 */
        if (h <= 1024u) KQ_JOIN(256, 4, 1);
        if (h <= 2048u) KQ_JOIN(256, 4, 2);
        if (h <= 2560u) KQ_JOIN(320, 4, 2);
        if (h <= 4096u) KQ_JOIN(256, 4, 4);
        KQ_JOIN(1024, 4, 4);
    }
    if (h <= 1024u) KQ_JOIN(256, 1, 4);
    if (h <= 4096u) KQ_JOIN(1024, 1, 4);
    KQ_JOIN(1024, 1, 16);
#undef KQ_JOIN
}

/*
 * kq_linattn.hip — linear attention with a decay for each head on gfx950,
 * the recurrent form (include/kq_hip.h, kq_hip_linear_attention_f32): single
 * rows and short sequences.
 *
 * For a row with query q, key k, value v, log decay g and beta b, the state
 * S [dk][dv] of a value head becomes
 *   S' = e^g S + k d^T,  d = b (v - e^g S^T k),  o = S'^T q = e^g S^T q + (q.k) d,
 * so S^T k and S^T q are formed in one pass over S, which stays in registers
 * from the first row to the last.
 *
 * A wave holds 4 CG columns of one head's state: lane = rg CG + cg has rows
 * rg R .. rg R + R - 1 of columns 4 cg .. 4 cg + 3, and every sum over the rows
 * is finished by lane exchanges, without LDS or a barrier. For one row a
 * sequence the state's read and write are the bound: 131,072 bytes a head of
 * 128 x 128, against 100 KFLOP. 61 sequences of 48 such heads take 74 us, 5.2
 * TB/s (a large copy: 5.1).
 *
 * Sequences of up to 16 rows run here too, a row after the other in 1.2 us
 * each; longer ones have chunks (kq_linattn_chunk.hip).
 */
#include "kq_linattn.h"

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));

/* one row of a lane: its part of q and k, its columns of v */
template <int R>
struct Row {
    float q[R], k[R], v[4];
    __device__ __forceinline__ void load(const kq_launch_linattn &a, uint64_t t, uint32_t qk,
                                         uint32_t vc) {
        const float4 *qp = (const float4 *)(a.q + t * a.qs + qk);
        const float4 *kp = (const float4 *)(a.k + t * a.ks + qk);
#pragma unroll
        for (int i = 0; i < R / 4; ++i) {
            const float4 x = qp[i], y = kp[i];
            q[4 * i] = x.x; q[4 * i + 1] = x.y; q[4 * i + 2] = x.z; q[4 * i + 3] = x.w;
            k[4 * i] = y.x; k[4 * i + 1] = y.y; k[4 * i + 2] = y.z; k[4 * i + 3] = y.w;
        }
        const float4 x = *(const float4 *)(a.v + t * a.vs + vc);
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    }
};

/* x = scale x / n(x) for a lane's part of x, where SUM are the bits of the lanes
 * that hold the rest. Where squares leave the type's range x is taken 2^-96
 * times: 1 / n(x) itself could be a number of fewer bits. */
template <int R, int SUM>
__device__ __forceinline__ void normalize(float (&x)[R], float eps, float scale) {
    auto squares = [&]() {
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < R; ++i) s = fmaf(x[i], x[i], s);
        return kq::lanes_sum<SUM>(s);
    };
    float s = squares();
    float f = kq::inverse_root(s + eps);
    if (!(s < 3.0e38f)) { /* the same way in every lane */
#pragma unroll
        for (int i = 0; i < R; ++i) x[i] *= 0x1p-96f;
        f = 1.0f / sqrtf(squares());
    }
#pragma unroll
    for (int i = 0; i < R; ++i) x[i] = x[i] * f * scale;
}

/* the plan, by one workgroup of NT threads */
template <int NT>
__device__ __forceinline__ void cut(const kq_launch_seqs &q, uint32_t max_rows,
                                    const kq_linattn_plan &w) {
    __shared__ uint32_t number[NT], sums[NT / 64];
    __shared__ uint32_t refused;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    if (tid == 0u) refused = 0u;
    __syncthreads();
    bool bad = false;
    for (uint32_t s = tid; s < q.count; s += NT) kq::seq_span(q, s, bad);
    if (bad) refused = 1u; /* each sequence's own workgroups report it */
    __syncthreads();
    const bool none = refused != 0u;
    /* the longest first, so that their scans, a workgroup after the other where
     * there are more than the device holds, do not end last */
    const bool sorted = q.count <= (uint32_t)NT;
    uint32_t at = 0u;
    for (uint32_t base = 0u; base < q.count; base += NT) {
        const uint32_t s = base + tid;
        uint32_t n = 0u;
        kq::SeqSpan sp = {};
        if (s < q.count) {
            sp = kq::seq_span(q, s, bad);
            if (!none && sp.live && sp.rows > max_rows)
                n = (sp.rows + kChunkRows - 1u) / kChunkRows;
        }
        uint32_t x = n; /* inclusive sum over the workgroup */
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t y = __shfl_up(x, o, KQ_WAVE);
            if (lane >= (uint32_t)o) x += y;
        }
        if (lane == 63u) sums[wave] = x;
        number[tid] = n;
        __syncthreads();
        uint32_t first = at + x - n, all = at;
        for (uint32_t k = 0; k < NT / 64u; ++k) {
            if (k < wave) first += sums[k];
            all += sums[k];
        }
        if (sorted) {
            first = 0u;
            for (uint32_t j = 0; j < q.count; ++j)
                first += number[j] > n || (number[j] == n && j < tid) ? number[j] : 0u;
        }
        /* the wave's sequences one after the other, a lane for a chunk */
        for (uint64_t todo = __ballot(n != 0u); todo != 0ull; todo &= todo - 1ull) {
            const int i = __builtin_ctzll(todo);
            auto of = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, i); };
            const uint32_t to = of(first), chunks = of(n), begin = of(sp.begin), rows = of(sp.rows);
            const uint32_t slot = of(sp.slot), fresh = of(sp.fresh ? 1u : 0u);
            for (uint32_t k = lane; k < chunks && to + k < w.chunks; k += 64u) {
                const uint32_t ahead = rows - k * kChunkRows;
                w.chunk[to + k] = kq_linattn_chunk{begin + k * kChunkRows,
                                                   ahead < kChunkRows ? ahead : kChunkRows,
                                                   k, chunks - k, slot, fresh, ahead, 0u};
            }
        }
        at = all;
        __syncthreads();
    }
    for (uint32_t i = at + tid; i < w.chunks; i += NT) w.chunk[i] = kq_linattn_chunk{};
}

/* grid (waves of columns of all heads / waves a workgroup, sequences): the
 * sequences of at most max_rows (64) rows. With a plan (CUT) one workgroup more in
 * x, the first of which cuts the others into chunks: a launch of its own for
 * that takes 5 us. */
template <int DK, int CG, int NT, bool CUT>
__global__ __launch_bounds__(NT) void linattn_rows(kq_launch_linattn a, kq_launch_seqs q,
                                                   uint32_t max_rows, kq_linattn_plan plan,
                                                   uint32_t *status) {
    if (CUT && blockIdx.x == gridDim.x - 1u) {
        if (blockIdx.y == 0u) cut<NT>(q, max_rows, plan);
        return;
    }
    constexpr int RG = 64 / CG, R = DK / RG, SUM = 63 & ~(CG - 1);
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t s = blockIdx.y;
    constexpr uint32_t kTile = 4u * CG; /* columns of a wave */
    const uint32_t shift = (a.value_width == 128u ? 7u : 6u) - (kTile == 32u ? 5u : 4u);
    const uint32_t w = __builtin_amdgcn_readfirstlane(blockIdx.x * (NT / 64) +
                                                      (threadIdx.x >> 6));
    const uint32_t h = w >> shift;
    const uint32_t col = (w & ((1u << shift) - 1u)) * kTile + (lane % CG) * 4u;
    const uint32_t row0 = (lane / CG) * R;
    const uint32_t qk = h / (a.value_heads / a.key_heads) * DK + row0;
    const uint32_t vc = h * a.value_width + col;
    /* where each sequence has one row, its loads do not wait for its slot */
    const bool single = q.offsets == nullptr;
    float alpha = 0.0f, beta = 0.0f;
    Row<R> next;
    auto load_gates = [&](uint64_t t) {
        if (a.alpha != nullptr) alpha = a.alpha[t * a.as + h];
        if (a.beta != nullptr) beta = a.beta[t * a.bs + h];
    };
    if (single && h < a.value_heads) {
        load_gates(s);
        next.load(a, s, qk, vc);
    }
    bool badseq = false;
    const kq::SeqSpan sp = kq::seq_span(q, s, badseq);
    /* by a workgroup of the sequence, every thread, behind its loads */
    auto check_slot = [&]() {
        if (blockIdx.x != 0u) return;
        if (sp.live && q.slots != nullptr)
            for (uint32_t j = threadIdx.x; j < s; j += NT) badseq |= q.slots[j] == sp.slot;
        if (badseq) kq_flag(status, KQ_DEV_SEQUENCE);
    };
    if (!sp.live || sp.rows > max_rows || h >= a.value_heads) {
        check_slot();
        return;
    }
    const size_t at = (((size_t)sp.slot * a.value_heads + h) * DK + row0) * a.value_width + col;
    if (!single && sp.rows != 0u) /* the gates: a lane for each row */
        load_gates((uint64_t)sp.begin + (lane < sp.rows ? lane : 0u));
    const float rate = a.rate[h], bias = a.bias != nullptr ? a.bias[h] : 0.0f;
    float S[R][4];
    if (!sp.fresh) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const float4 x = *(const float4 *)(a.state + at + (size_t)i * a.value_width);
            S[i][0] = x.x; S[i][1] = x.y; S[i][2] = x.z; S[i][3] = x.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < R; ++i) S[i][0] = S[i][1] = S[i][2] = S[i][3] = 0.0f;
    }
    if (!single && sp.rows != 0u) next.load(a, sp.begin, qk, vc);
    bool badin = !kq_isfinite(rate) || rate > 0.0f || !kq_isfinite(bias), bad = false;
    badin |= !kq_isfinite(alpha) || !kq_isfinite(beta);
    const kq::Decay e = kq::decay_of(kq::log_decay(a, alpha, rate, bias));
    const float part = kq::sigmoid(beta);
    for (uint32_t n = 0; n < sp.rows; ++n) {
        Row<R> r = next;
        const uint64_t t = (uint64_t)sp.begin + n;
        if (n + 1u < sp.rows) next.load(a, t + 1u, qk, vc);
        auto of = [&](float x) {
            return __uint_as_float(
                (uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x), (int)n));
        };
        const float c0 = of(e.c0), c1 = of(e.c1), b = of(part);
        /* sums over the rows of S, of q and k as they are: all exchanges side by
         * side, then the norms as factors */
        float q2, k2, qkv, sk[4], sq[4];
        auto sums = [&]() {
            q2 = k2 = qkv = 0.0f;
#pragma unroll
            for (int c = 0; c < 4; ++c) sk[c] = sq[c] = 0.0f;
#pragma unroll
            for (int i = 0; i < R; ++i) {
                q2 = fmaf(r.q[i], r.q[i], q2);
                k2 = fmaf(r.k[i], r.k[i], k2);
                qkv = fmaf(r.q[i], r.k[i], qkv);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    sk[c] = fmaf(r.k[i], S[i][c], sk[c]);
                    sq[c] = fmaf(r.q[i], S[i][c], sq[c]);
                }
            }
            q2 = kq::lanes_sum<SUM>(q2);
            k2 = kq::lanes_sum<SUM>(k2);
            qkv = kq::lanes_sum<SUM>(qkv);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                sk[c] = kq::lanes_sum<SUM>(sk[c]);
                sq[c] = kq::lanes_sum<SUM>(sq[c]);
            }
        };
        sums();
        float nq = a.scale, nk = 1.0f;
        /* sums with S may leave the range before their norm divides them */
        const float most = ((fabsf(sk[0]) + fabsf(sk[1])) + (fabsf(sk[2]) + fabsf(sk[3]))) +
                           ((fabsf(sq[0]) + fabsf(sq[1])) + (fabsf(sq[2]) + fabsf(sq[3])));
        const bool fits = most < 3.0e38f && q2 > 1e-24f && q2 < 1e12f && k2 > 1e-24f && k2 < 1e12f;
        if (a.normalize != 0u && __ballot(!fits) == 0ull) { /* the same way in every lane */
            nq *= kq::inverse_root(q2 + a.epsilon);
            nk = kq::inverse_root(k2 + a.epsilon);
        } else {
#pragma unroll
            for (int i = 0; i < R; ++i) badin |= !kq_isfinite(r.q[i]) || !kq_isfinite(r.k[i]);
            if (a.normalize != 0u) { /* sums as they are could leave the type's range */
                normalize<R, SUM>(r.q, a.epsilon, a.scale);
                normalize<R, SUM>(r.k, a.epsilon, 1.0f);
                sums();
                nq = nk = 1.0f;
            }
        }
        qkv *= nq * nk;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            sk[c] *= nk;
            sq[c] *= nq;
        }
        float d[4], o[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            badin |= !kq_isfinite(r.v[c]);
            d[c] = r.v[c];
            if (a.beta != nullptr) d[c] = b * (r.v[c] - fmaf(c1, sk[c], c0 * sk[c]));
            o[c] = fmaf(qkv, d[c], fmaf(c1, sq[c], c0 * sq[c]));
            bad |= !kq_isfinite(o[c]);
        }
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c)
                S[i][c] = fmaf(r.k[i], d[c] * nk, fmaf(c1, S[i][c], c0 * S[i][c]));
        if (lane < CG)
            *(float4 *)(a.y + t * a.ys + vc) = make_float4(o[0], o[1], o[2], o[3]);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        /* not kept in the caches, which other states need: 61 sequences' single
         * rows 86.4 -> 80.8 us */
        __builtin_nontemporal_store(f4{S[i][0], S[i][1], S[i][2], S[i][3]},
                                    (f4 *)(a.state_out + at + (size_t)i * a.value_width));
#pragma unroll
        for (int c = 0; c < 4; ++c) bad |= !kq_isfinite(S[i][c]);
    }
    check_slot();
    if (badin) kq_flag(status, KQ_DEV_INPUT);
    if (bad) kq_flag(status, KQ_DEV_NUMERIC);
}

template <int DK, int CG, int NT, bool CUT>
hipError_t launch(const kq_launch_linattn &a, const kq_launch_seqs &q, uint32_t max_rows,
                  const kq_linattn_plan &plan, uint32_t *status, hipStream_t s) {
    const uint32_t waves = a.value_heads * a.value_width / (4u * CG), per = NT / 64;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(linattn_rows<DK, CG, NT, CUT>),
                       dim3((waves + per - 1u) / per + (CUT ? 1u : 0u), q.count), dim3(NT), 0, s, a,
                       q, max_rows, plan, status);
    return hipGetLastError();
}

/* Workgroups of four waves with 32 columns each. For few sequences 16 columns
 * and, for the fewest, one wave a workgroup, so that they spread over the
 * device. 48 heads of 128 x 128, in us, with 16 columns and one wave, 16 and
 * four, 32 and four: one sequence 5.4, 5.6, 6.7; two 7.3, 6.1, 7.0; four 9.5,
 * 8.1, 9.0; six 12.5, 10.1, 11.5; eight 14.0, 12.4, 12.0; 32 55, 48, 39.
 * With a plan 32 columns always, since what takes long there are many rows:
 * 16 and 32 columns for 32 sequences of one row 41 and 36, 61 of one 92 and 79,
 * 32 of four 46 and 41, but two of 16 rows 26 and 32. */
template <int DK>
hipError_t launch(const kq_launch_linattn &a, const kq_launch_seqs &q, uint32_t max_rows,
                  const kq_linattn_plan &plan, uint32_t *status, hipStream_t s) {
    const uint64_t tiles = (uint64_t)a.value_heads * a.value_width / 32u * q.count;
    if (plan.chunk != nullptr) return launch<DK, 8, 256, true>(a, q, max_rows, plan, status, s);
    if (tiles <= 256u) return launch<DK, 4, 64, false>(a, q, max_rows, plan, status, s);
    if (tiles <= 1280u) return launch<DK, 4, 256, false>(a, q, max_rows, plan, status, s);
    return launch<DK, 8, 256, false>(a, q, max_rows, plan, status, s);
}

}  // namespace

hipError_t kq_linattn_recurrent(const kq_launch_linattn &a, const kq_launch_seqs &q,
                                uint32_t max_rows, const kq_linattn_plan &plan, uint32_t *status,
                                hipStream_t s) {
    return a.key_width == 128u ? launch<128>(a, q, max_rows, plan, status, s)
                               : launch<64>(a, q, max_rows, plan, status, s);
}

/* Sequences up to this long (64: a lane for each row) run in the recurrent form:
 * 1.2 us a row, against a chunk's launches. In the recurrent form and in chunks,
 * in us, 48 heads of 128 x 128: one sequence of 17 rows 24 and 24, of 24 32 and 25;
 * eight of 17 48 and 61, of 24 63 and 62, of 32 82 and 62; 32 of 17 120 and 209, of
 * 24 163 and 212, of 32 223 and 215. So 16 is the limit of one sequence; many
 * would gain from twice that, which a call's counts alone, with the lengths on
 * the device, do not tell. */
constexpr uint32_t kShort = 16u;

extern "C" uint64_t kq_launch_linattn_scratch(const kq_launch_linattn *a, uint64_t tokens,
                                              uint32_t count) {
    return tokens <= kShort ? 0u : kq_linattn_chunked_scratch(*a, tokens, count, kShort);
}

extern "C" hipError_t kq_launch_linattn_run(const kq_launch_linattn *a, const kq_launch_seqs *q,
                                            void *scratch, uint32_t *status, hipStream_t s) {
    if (q->offsets == nullptr || q->tokens <= kShort)
        return kq_linattn_recurrent(*a, *q, kShort, kq_linattn_plan{}, status, s);
    return kq_linattn_chunked(*a, *q, kShort, scratch, status, s);
}

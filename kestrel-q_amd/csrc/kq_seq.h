/*
 * kq_seq.h — sequences on the device: where a sequence's rows and its state
 * lie, checked before anything is indexed with them (include/kq_hip.h,
 * "Sequences").
 */
#ifndef KQ_SEQ_H
#define KQ_SEQ_H

#include "kq_device.h"
#include "kq_launch.h"

#define KQ_NO_SLOT 0xffffffffu

namespace kq {

struct SeqSpan {
    uint32_t begin, rows, slot;
    bool fresh;
    bool live; /* false: taken out of the call, or refused */
};

/* Sequence s of the call. A span or slot that breaks the rules is not live
 * and sets `bad`, so nothing is read or written through it. */
__device__ __forceinline__ SeqSpan seq_span(const kq_launch_seqs &q, uint32_t s, bool &bad) {
    SeqSpan r;
    r.begin = s;
    r.rows = 1u;
    r.slot = q.slots != nullptr ? q.slots[s] : s;
    r.live = r.slot != KQ_NO_SLOT;
    if (q.offsets != nullptr) {
        const uint32_t a = q.offsets[s], b = q.offsets[s + 1u];
        r.begin = a;
        r.rows = b - a;
        if (a > b || b > q.tokens) {
            bad = true;
            r.live = false;
        }
    }
    if (r.live && r.slot >= q.slot_count) {
        bad = true;
        r.live = false;
    }
    r.fresh = q.fresh != nullptr && q.fresh[s] != 0u;
    return r;
}

/* Whether a sequence before s names s's slot too. All NT threads of a
 * workgroup look at a part; each returns its own finding. */
template <int NT>
__device__ __forceinline__ bool seq_slot_taken(const kq_launch_seqs &q, uint32_t s,
                                               uint32_t slot) {
    bool taken = false;
    if (q.slots != nullptr && slot != KQ_NO_SLOT)
        for (uint32_t j = threadIdx.x; j < s; j += NT) taken |= q.slots[j] == slot;
    return taken;
}

/* e^x, x <= 0, to about one unit in the last place: x log2(e) as a rounded
 * product t and its error r, 2^t of the hardware, and 1 + r ln 2. Below
 * -150 it is 0 in 32 bits. */
__device__ __forceinline__ float exp_neg(float x) {
    x = fmaxf(x, -150.0f);
    const float t = x * 0x1.715476p+0f;
    const float r = fmaf(x, 0x1.4ae0cp-26f, fmaf(x, 0x1.715476p+0f, -t));
    const float e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, r * 0x1.62e43p-1f, e);
}

/* e^x, x <= 0 in 64 bits (a difference of sums of log decays): rounding the
 * base-2 exponent to 32 bits costs at most |x| 2^-24 of a value e^x, 0.37
 * 2^-24 of 1 */
__device__ __forceinline__ float exp_of(double x) {
    return __builtin_amdgcn_exp2f((float)(x * 1.4426950408889634));
}

/* 1 / d, d in [1, 2]: the hardware's reciprocal and one Newton step */
__device__ __forceinline__ float inverse_of(float d) {
    const float r = __builtin_amdgcn_rcpf(d);
    return fmaf(fmaf(-d, r, 1.0f), r, r);
}

/* 1 / sqrt(x), x normal: the hardware's and one Newton step */
__device__ __forceinline__ float inverse_root(float x) {
    const float r = __builtin_amdgcn_rsqf(x);
    return fmaf(0.5f * r, fmaf(-x * r, r, 1.0f), r);
}

/* ln(1 + e^x) of a finite sum x that may have left the range */
__device__ __forceinline__ float softplus(float x) {
    x = fminf(x, 0x1.fffffep127f);
    return fmaxf(x, 0.0f) + log1pf(exp_neg(-fabsf(x)));
}

__device__ __forceinline__ float sigmoid(float x) {
    const float e = exp_neg(-fabsf(x));
    const float r = inverse_of(1.0f + e);
    return x >= 0.0f ? r : e * r;
}

/* x of lane l ^ BIT, bits below 16: DPP controls, for bit 4 the half-row
 * mirror where the lanes of a quad hold the same already (QUAD) */
template <int BIT, bool QUAD>
__device__ __forceinline__ float lane_xor(float x) {
    if constexpr (BIT == 4 && !QUAD) return __shfl_xor(x, 4, KQ_WAVE);
    constexpr int ctrl = BIT == 1 ? 0xB1 : BIT == 2 ? 0x4E : BIT == 4 ? 0x141 : 0x128;
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), ctrl,
                                                                 0xf, 0xf, false));
}

/* v over the lanes that differ in the bits of MASK, by an operation that does
 * not look at the order of its two operands; rows of 16 lanes are swapped
 * (bits 16 and 32), so that nothing goes through LDS */
template <int MASK, int BIT = 1, typename Op>
__device__ __forceinline__ float lanes_all(float v, Op op) {
    if constexpr (BIT < 64) {
        if constexpr ((MASK & BIT) != 0) {
            if constexpr (BIT == 16 || BIT == 32) {
                const uint32_t u = __float_as_uint(v);
                auto r = BIT == 16 ? __builtin_amdgcn_permlane16_swap(u, u, false, false)
                                   : __builtin_amdgcn_permlane32_swap(u, u, false, false);
                v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
            } else {
                v = op(v, lane_xor<BIT, (MASK & 3) == 3>(v));
            }
        }
        return lanes_all<MASK, BIT * 2>(v, op);
    } else {
        return v;
    }
}
template <int MASK>
__device__ __forceinline__ float lanes_sum(float v) {
    return lanes_all<MASK>(v, [](float a, float b) { return a + b; });
}
template <int MASK>
__device__ __forceinline__ float lanes_max(float v) {
    return lanes_all<MASK>(v, [](float a, float b) { return fmaxf(a, b); });
}

}  // namespace kq

#endif

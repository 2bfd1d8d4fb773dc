/*
 * kq_linattn.h — the two forms of the linear attention (kq_linattn.hip,
 * kq_linattn_chunk.hip).
 */
#ifndef KQ_LINATTN_H
#define KQ_LINATTN_H

#include "kq_device.h"
#include "kq_launch.h"
#include "kq_seq.h"

namespace kq {

/* A row's log decay g <= 0 of a head. From -104 on e^g is 0 in binary32; held
 * at -1024, a decay is as strong as any, and 64 of them summed in 64 bits leave
 * the decays of the rows between them to 2^-33: a difference of the sums that
 * does not span a strong row would otherwise have lost its own terms. */
__device__ __forceinline__ float log_decay(const kq_launch_linattn &a, float alpha, float rate,
                                           float bias) {
    return fmaxf(a.alpha != nullptr ? rate * softplus(alpha + bias) : rate, -1024.0f);
}

/* S e^g as c0 S + c1 S. A decay near 1 that is rounded to 32 bits is off by
 * up to 2^-25 in the same direction row after row, which a memory of many
 * rows adds up; e^g - 1 has its own 24 bits. Where much of S is lost the
 * sum would cancel, and e^g itself is exact enough. */
struct Decay {
    float c0, c1;
};
__device__ __forceinline__ Decay decay_of(float g) {
    Decay d;
    d.c0 = g > -0.5f ? 1.0f : 0.0f;
    d.c1 = g > -0.5f ? expm1f(g) : exp_neg(g);
    return d;
}
/* of many rows, g their sum. e^g - 1 is Taylor's sum to g^8, whose rest is
 * 2^-26 of it at -1/2. */
__device__ __forceinline__ Decay decay_of(double g) {
    const float x = fmaxf((float)g, -0.5f);
    float s = 1.0f / 40320.0f;
    s = fmaf(s, x, 1.0f / 5040.0f);
    s = fmaf(s, x, 1.0f / 720.0f);
    s = fmaf(s, x, 1.0f / 120.0f);
    s = fmaf(s, x, 1.0f / 24.0f);
    s = fmaf(s, x, 1.0f / 6.0f);
    s = fmaf(s, x, 0.5f);
    s = fmaf(s * x, x, x);
    Decay d;
    d.c0 = g > -0.5 ? 1.0f : 0.0f;
    d.c1 = g > -0.5 ? s : exp_of(g);
    return d;
}

}  // namespace kq

/* A chunk of a sequence that the chunked form runs: all that a workgroup has
 * to know before its first loads, which a record of its own for the sequence
 * would have wait for one more. */
struct alignas(32) kq_linattn_chunk {
    uint32_t row, rows;    /* its first, their number (0: no chunk) */
    uint32_t number, left; /* which of its sequence; chunks from it to the last */
    uint32_t slot, fresh;  /* the sequence's */
    uint32_t ahead;        /* rows from its first to the sequence's end */
    uint32_t none;
};
struct kq_linattn_plan {
    kq_linattn_chunk *chunk; /* in device memory; NULL for no plan */
    uint32_t chunks;         /* what the sizes of a call allow */
};
constexpr uint32_t kChunkRows = 64;

/* the recurrent form over the sequences of at most max_rows rows; checks all
 * sequences, and writes the plan of the others */
hipError_t kq_linattn_recurrent(const kq_launch_linattn &a, const kq_launch_seqs &q,
                                uint32_t max_rows, const kq_linattn_plan &plan, uint32_t *status,
                                hipStream_t s);
/* both forms: the chunked one over the sequences of more rows */
uint64_t kq_linattn_chunked_scratch(const kq_launch_linattn &a, uint64_t tokens, uint32_t count,
                                    uint32_t max_rows);
hipError_t kq_linattn_chunked(const kq_launch_linattn &a, const kq_launch_seqs &q,
                              uint32_t max_rows, void *scratch, uint32_t *status, hipStream_t s);

#endif

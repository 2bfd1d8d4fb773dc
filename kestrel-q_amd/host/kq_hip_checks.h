/*
 * kq_hip_checks.h — the checks of arguments that the operators over sequences
 * share (kq_hip_gdn.c, kq_hip_paged.c).
 */
#ifndef KQ_HIP_CHECKS_H
#define KQ_HIP_CHECKS_H

#include <stdint.h>

#include "kq_hip.h"
#include "kq_launch.h"
#include "kq_status_internal.h"

#define KQ_MAX_TOKENS 262144u
#define KQ_MAX_SEQUENCES 65535u
#define KQ_MAX_WIDTH 16384u

static inline int on(const void *p, uintptr_t a) { return ((uintptr_t)p % a) == 0u; }

/* a buffer of `floats` values at p, for the overlap checks */
typedef struct span {
    const void *p;
    uint64_t floats;
} span;

static inline int overlap(span a, span b) {
    const uintptr_t a0 = (uintptr_t)a.p, b0 = (uintptr_t)b.p;
    if (a.p == NULL || b.p == NULL || a.floats == 0u || b.floats == 0u) return 0;
    return a0 < b0 + b.floats * 4u && b0 < a0 + a.floats * 4u;
}

/* floats from the first value of `rows` rows to the last one's end */
static inline uint64_t rows_span(uint64_t rows, uint64_t stride, uint64_t width) {
    return rows == 0u ? 0u : (rows - 1u) * stride + width;
}

/* Outputs against everything else; NULL buffers overlap nothing. The first
 * output may be the first input, which lies there alone: any other one is
 * read where something else is written. */
static inline int aliased(const span *outs, uint32_t n, const span *ins, uint32_t m) {
    for (uint32_t i = 0; i < n; ++i) {
        for (uint32_t j = i + 1u; j < n; ++j)
            if (overlap(outs[i], outs[j])) return 1;
        for (uint32_t j = 0; j < m; ++j) {
            if (i == 0u && j == 0u && outs[0].p == ins[0].p) continue;
            if (overlap(outs[i], ins[j])) return 1;
        }
    }
    return 0;
}

/* a row stride in floats: at least the row; 64 rows within 32-bit offsets */
static inline int stride_ok(uint64_t stride, uint64_t width) {
    return stride >= width && stride <= (UINT64_C(1) << 22);
}

static inline kq_status sequences_ok(const kq_hip_sequences *q, kq_diagnostic *diag) {
    if (q == NULL || q->token_count == 0u || q->sequence_count == 0u || q->slot_count == 0u)
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT, "tokens, sequences and slots are required");
    if (q->token_count > KQ_MAX_TOKENS || q->sequence_count > KQ_MAX_SEQUENCES)
        return kq_fail(diag, KQ_STATUS_LIMIT_EXCEEDED,
                       "at most %u tokens and %u sequences a call", KQ_MAX_TOKENS,
                       KQ_MAX_SEQUENCES);
    if (q->offsets == NULL && q->token_count != q->sequence_count)
        return kq_fail(diag, KQ_STATUS_DIMENSION_MISMATCH,
                       "without offsets each sequence has one token");
    if (q->slots == NULL && q->sequence_count > q->slot_count)
        return kq_fail(diag, KQ_STATUS_DIMENSION_MISMATCH,
                       "without slots there are as many as sequences at least");
    if (!on(q->offsets, 4u) || !on(q->slots, 4u) || !on(q->fresh, 4u))
        return kq_fail(diag, KQ_STATUS_INVALID_ALIGNMENT, "offsets, slots and fresh need 4-byte alignment");
    return KQ_STATUS_OK;
}

static inline kq_launch_seqs launch_seqs(const kq_hip_sequences *q) {
    kq_launch_seqs s;
    s.tokens = q->token_count;
    s.count = q->sequence_count;
    s.slot_count = q->slot_count;
    s.offsets = q->offsets;
    s.slots = q->slots;
    s.fresh = q->fresh;
    return s;
}

#endif

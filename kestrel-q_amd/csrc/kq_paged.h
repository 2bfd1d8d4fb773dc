/*
 * kq_paged.h — sequences whose tokens lie in the pages of a cache: where a
 * sequence's rows stand, and which page holds a token, checked before
 * anything is indexed with them (include/kq_hip.h, kq_hip_paged_cache).
 */
#ifndef KQ_PAGED_H
#define KQ_PAGED_H

#include "kq_device.h"
#include "kq_launch.h"
#include "kq_seq.h"

namespace kq {

struct PagedSeq {
    uint32_t begin, rows, past, slot;
    bool live; /* false: taken out of the call, or refused */
};

/* Sequence s of the call and the tokens that the cache holds of it */
__device__ __forceinline__ PagedSeq paged_seq(const kq_launch_seqs &q, const kq_launch_paged &c,
                                              uint32_t s, bool &bad) {
    const SeqSpan sp = seq_span(q, s, bad);
    PagedSeq r;
    r.begin = sp.begin;
    r.rows = sp.rows;
    r.slot = sp.slot;
    r.live = sp.live;
    r.past = 0u;
    if (r.live && !sp.fresh) r.past = c.lengths[r.slot];
    if (r.live && (uint64_t)r.past + r.rows > (uint64_t)c.table_pages << c.page_shift) {
        bad = true;
        r.live = false;
    }
    return r;
}

/* The last s of [0, count) with sorted[s] <= x, 0 if there is none: each wave
 * looks at 64 entries at a time. Entries that are not in order give some s of
 * the range. All lanes get the same. */
__device__ __forceinline__ uint32_t wave_find(const uint32_t *sorted, uint32_t count, uint32_t x) {
    const uint32_t lane = threadIdx.x & 63u;
    uint32_t lo = 0u, range = count;
    while (range > 1u) {
        const uint32_t step = (range + 63u) / 64u;
        const uint32_t at = lane * step;
        const uint64_t m = __ballot(at < range && sorted[lo + at] <= x);
        const uint32_t k = m == 0ull ? 0u : 63u - (uint32_t)__clzll(m);
        lo += k * step;
        range = range - k * step < step ? range - k * step : step;
    }
    return __builtin_amdgcn_readfirstlane(lo);
}

}  // namespace kq

#endif

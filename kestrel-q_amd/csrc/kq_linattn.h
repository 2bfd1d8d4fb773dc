/*
 * kq_linattn.h — the two forms of the linear attention (kq_linattn.hip,
 * kq_linattn_chunk.hip).
 */
#ifndef KQ_LINATTN_H
#define KQ_LINATTN_H

#include "kq_launch.h"

/* the recurrent form over the sequences of at most max_rows rows; checks all
 * sequences */
hipError_t kq_linattn_recurrent(const kq_launch_linattn &a, const kq_launch_seqs &q,
                                uint32_t max_rows, uint32_t *status, hipStream_t s);

#endif

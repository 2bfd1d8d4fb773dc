/*
 * kq_hip_gdn.c — host side of the operators between a GDN layer's
 * projections and its residual (include/kq_hip.h: sequences, the causal
 * convolution, linear attention, the norms around a block).
 *
 * C17. Everything that the host can see is checked before any device work:
 * the descriptions, then limits, alignment and overlaps. What lies in
 * device memory (the offsets and slots of the sequences) is checked by the
 * kernels before they index with it.
 */
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "kq_hip.h"
#include "kq_hip_internal.h"
#include "kq_launch.h"
#include "kq_status_internal.h"

#define KQ_MAX_TOKENS 262144u
#define KQ_MAX_SEQUENCES 65535u
#define KQ_MAX_WIDTH 16384u

static int on(const void *p, uintptr_t a) { return ((uintptr_t)p % a) == 0u; }

/* a buffer of `floats` values at p, for the overlap checks */
typedef struct span {
    const void *p;
    uint64_t floats;
} span;

static int overlap(span a, span b) {
    const uintptr_t a0 = (uintptr_t)a.p, b0 = (uintptr_t)b.p;
    if (a.p == NULL || b.p == NULL || a.floats == 0u || b.floats == 0u) return 0;
    return a0 < b0 + b.floats * 4u && b0 < a0 + a.floats * 4u;
}

/* floats from the first value of `rows` rows to the last one's end */
static uint64_t rows_span(uint64_t rows, uint64_t stride, uint64_t width) {
    return rows == 0u ? 0u : (rows - 1u) * stride + width;
}

/* Outputs against everything else; NULL buffers overlap nothing. The first
 * output may be the first input, which lies there alone: any other one is
 * read where something else is written. */
static int aliased(const span *outs, uint32_t n, const span *ins, uint32_t m) {
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
static int stride_ok(uint64_t stride, uint64_t width) {
    return stride >= width && stride <= (UINT64_C(1) << 22);
}

static kq_status sequences_ok(const kq_hip_sequences *q, kq_diagnostic *diag) {
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

static kq_launch_seqs launch_seqs(const kq_hip_sequences *q) {
    kq_launch_seqs s;
    s.tokens = q->token_count;
    s.count = q->sequence_count;
    s.slot_count = q->slot_count;
    s.offsets = q->offsets;
    s.slots = q->slots;
    s.fresh = q->fresh;
    return s;
}

/* ------------------------------------------------------------------ */

kq_status kq_hip_causal_conv_f32(kq_hip_context *c, const kq_hip_causal_conv *v,
                                 const kq_hip_sequences *q, const float *x, uint64_t xs,
                                 const float *state, float *state_out, float *y, uint64_t ys,
                                 kq_diagnostic *diag) {
    kq_launch_conv l;
    kq_launch_seqs s;
    uint64_t state_floats;
    kq_status st;
    kq_diagnostic_clear(diag);
    if (c == NULL || v == NULL || x == NULL || state == NULL || state_out == NULL || y == NULL ||
        v->weight == NULL || v->channels == 0u)
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT, "complete convolution arguments are required");
    if (v->activation != KQ_HIP_ACTIVATION_NONE && v->activation != KQ_HIP_ACTIVATION_SILU)
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT, "the convolution's activation is none or SiLU");
    if (v->taps < 2u || v->taps > 8u || v->channels > (1u << 20))
        return kq_fail(diag, KQ_STATUS_LIMIT_EXCEEDED, "2 .. 8 taps and at most 2^20 channels");
    st = sequences_ok(q, diag);
    if (st != KQ_STATUS_OK) return st;
    if (!stride_ok(xs, v->channels) || !stride_ok(ys, v->channels))
        return kq_fail(diag, KQ_STATUS_DIMENSION_MISMATCH, "row strides hold the channels and at most 2^22 floats");
    if (!on(x, 4u) || !on(y, 4u) || !on(state, 4u) || !on(state_out, 4u) || !on(v->weight, 4u) ||
        !on(v->bias, 4u))
        return kq_fail(diag, KQ_STATUS_INVALID_ALIGNMENT, "convolution buffers need 4-byte alignment");
    state_floats = (uint64_t)q->slot_count * (v->taps - 1u) * v->channels;
    {
        const span outs[2] = {{state_out, state_floats},
                              {y, rows_span(q->token_count, ys, v->channels)}};
        const span ins[7] = {{state, state_floats},
                             {x, rows_span(q->token_count, xs, v->channels)},
                             {v->weight, (uint64_t)v->channels * v->taps},
                             {v->bias, v->channels},
                             {q->offsets, (uint64_t)q->sequence_count + 1u},
                             {q->slots, q->sequence_count},
                             {q->fresh, q->sequence_count}};
        if (aliased(outs, 2u, ins, 7u))
            return kq_fail(diag, KQ_STATUS_ALIASING_VIOLATION,
                           "convolution outputs overlap; state_out may only be the state itself");
    }
    st = kqi_context_begin(c, diag);
    if (st == KQ_STATUS_OK) {
        void *const outs[2] = {state_out, y};
        const uint64_t lens[2] = {state_floats * 4u, rows_span(q->token_count, ys, v->channels) * 4u};
        st = kqi_context_snapshot(c, 2u, outs, lens, diag);
    }
    if (st != KQ_STATUS_OK) return st;
    l.channels = v->channels;
    l.taps = v->taps;
    l.weight = v->weight;
    l.bias = v->bias;
    l.silu = v->activation == KQ_HIP_ACTIVATION_SILU;
    s = launch_seqs(q);
    return kqi_context_finish(c,
                              (int)kq_launch_causal_conv(&l, &s, x, xs, state, state_out, y, ys,
                                                         kqi_context_status_word(c),
                                                         (hipStream_t)kqi_context_stream_ptr(c)),
                              "convolution launch", diag);
}

/* ------------------------------------------------------------------ */

static kq_status attention_ok(const kq_hip_linear_attention *a, kq_diagnostic *diag) {
    if (a == NULL || a->key_heads == 0u || a->value_heads == 0u || a->normalize > 1u ||
        !isfinite(a->scale) ||
        (a->normalize != 0u && !(isfinite(a->epsilon) && a->epsilon >= 1e-20f)))
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT,
                       "linear attention needs heads, a finite scale and, to normalize, an epsilon "
                       "of at least 1e-20");
    if (a->value_heads % a->key_heads != 0u)
        return kq_fail(diag, KQ_STATUS_DIMENSION_MISMATCH,
                       "the value heads are a multiple of the key heads");
    if (a->value_heads > 256u || (a->key_width != 64u && a->key_width != 128u) ||
        (a->value_width != 64u && a->value_width != 128u))
        return kq_fail(diag, KQ_STATUS_LIMIT_EXCEEDED,
                       "linear attention: at most 256 value heads, of width 64 or 128");
    return KQ_STATUS_OK;
}

static kq_launch_linattn launch_attention(const kq_hip_linear_attention *a) {
    kq_launch_linattn l;
    memset(&l, 0, sizeof l);
    l.key_heads = a->key_heads;
    l.value_heads = a->value_heads;
    l.key_width = a->key_width;
    l.value_width = a->value_width;
    l.scale = a->scale;
    l.normalize = a->normalize;
    l.epsilon = a->epsilon;
    l.rate = a->rate;
    l.bias = a->bias;
    return l;
}

uint64_t kq_hip_linear_attention_scratch_bytes(const kq_hip_linear_attention *a,
                                               const kq_hip_sequences *q) {
    kq_launch_linattn l;
    if (attention_ok(a, NULL) != KQ_STATUS_OK || sequences_ok(q, NULL) != KQ_STATUS_OK ||
        q->offsets == NULL)
        return 0u;
    l = launch_attention(a);
    return kq_launch_linattn_scratch(&l, q->token_count, q->sequence_count);
}

kq_status kq_hip_linear_attention_f32(kq_hip_context *c, const kq_hip_linear_attention *a,
                                      const kq_hip_sequences *q,
                                      const kq_hip_linear_attention_inputs *in,
                                      const float *state, float *state_out, float *y, uint64_t ys,
                                      void *scratch, uint64_t scratch_bytes, kq_diagnostic *diag) {
    kq_launch_linattn l;
    kq_launch_seqs s;
    uint64_t kw, vw, need, state_floats, n;
    kq_status st;
    kq_diagnostic_clear(diag);
    if (c == NULL || a == NULL || in == NULL || in->query == NULL || in->key == NULL ||
        in->value == NULL || a->rate == NULL || state == NULL || state_out == NULL || y == NULL)
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT,
                       "complete linear attention arguments are required");
    st = attention_ok(a, diag);
    if (st == KQ_STATUS_OK) st = sequences_ok(q, diag);
    if (st != KQ_STATUS_OK) return st;
    kw = (uint64_t)a->key_heads * a->key_width;
    vw = (uint64_t)a->value_heads * a->value_width;
    n = q->token_count;
    if (!stride_ok(in->query_stride, kw) || !stride_ok(in->key_stride, kw) ||
        !stride_ok(in->value_stride, vw) || !stride_ok(ys, vw) ||
        (in->alpha != NULL && !stride_ok(in->alpha_stride, a->value_heads)) ||
        (in->beta != NULL && !stride_ok(in->beta_stride, a->value_heads)))
        return kq_fail(diag, KQ_STATUS_DIMENSION_MISMATCH, "row strides hold the heads and at most 2^22 floats");
    need = kq_hip_linear_attention_scratch_bytes(a, q);
    if (need != 0u && scratch == NULL)
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT, "linear attention scratch is required");
    if (scratch_bytes < need)
        return kq_fail(diag, KQ_STATUS_BUFFER_TOO_SMALL, "linear attention scratch needs %llu bytes",
                       (unsigned long long)need);
    if (!on(in->query, 16u) || !on(in->key, 16u) || !on(in->value, 16u) || !on(y, 16u) ||
        !on(state, 16u) || !on(state_out, 16u) || (need != 0u && !on(scratch, 16u)) ||
        in->query_stride % 4u != 0u || in->key_stride % 4u != 0u || in->value_stride % 4u != 0u ||
        ys % 4u != 0u)
        return kq_fail(diag, KQ_STATUS_INVALID_ALIGNMENT,
                       "linear attention rows, states and scratch need 16-byte alignment");
    if (!on(in->alpha, 4u) || !on(in->beta, 4u) || !on(a->rate, 4u) || !on(a->bias, 4u))
        return kq_fail(diag, KQ_STATUS_INVALID_ALIGNMENT, "gates need 4-byte alignment");
    state_floats = (uint64_t)q->slot_count * a->value_heads * a->key_width * a->value_width;
    {
        const span outs[3] = {{state_out, state_floats},
                              {y, rows_span(n, ys, vw)},
                              {scratch, need / 4u}};
        const span ins[11] = {{state, state_floats},
                              {in->query, rows_span(n, in->query_stride, kw)},
                              {in->key, rows_span(n, in->key_stride, kw)},
                              {in->value, rows_span(n, in->value_stride, vw)},
                              {in->alpha, rows_span(n, in->alpha_stride, a->value_heads)},
                              {in->beta, rows_span(n, in->beta_stride, a->value_heads)},
                              {a->rate, a->value_heads},
                              {a->bias, a->value_heads},
                              {q->offsets, (uint64_t)q->sequence_count + 1u},
                              {q->slots, q->sequence_count},
                              {q->fresh, q->sequence_count}};
        if (aliased(outs, 3u, ins, 11u))
            return kq_fail(diag, KQ_STATUS_ALIASING_VIOLATION,
                           "linear attention outputs or scratch overlap; state_out may only be the "
                           "state itself");
    }
    st = kqi_context_begin(c, diag);
    if (st == KQ_STATUS_OK) {
        void *const outs[2] = {state_out, y};
        const uint64_t lens[2] = {state_floats * 4u, rows_span(n, ys, vw) * 4u};
        st = kqi_context_snapshot(c, 2u, outs, lens, diag);
    }
    if (st != KQ_STATUS_OK) return st;
    l = launch_attention(a);
    l.q = in->query;
    l.k = in->key;
    l.v = in->value;
    l.alpha = in->alpha;
    l.beta = in->beta;
    l.qs = in->query_stride;
    l.ks = in->key_stride;
    l.vs = in->value_stride;
    l.as = in->alpha_stride;
    l.bs = in->beta_stride;
    l.state = state;
    l.state_out = state_out;
    l.y = y;
    l.ys = ys;
    s = launch_seqs(q);
    return kqi_context_finish(c,
                              (int)kq_launch_linattn_run(&l, &s, need != 0u ? scratch : NULL,
                                                         kqi_context_status_word(c),
                                                         (hipStream_t)kqi_context_stream_ptr(c)),
                              "linear attention launch", diag);
}

/* ------------------------------------------------------------------ */

kq_status kq_hip_gated_norm_f32(kq_hip_context *c, const kq_hip_gated_norm *v, uint64_t tokens,
                                const float *x, uint64_t xs, const float *gate, uint64_t gs,
                                float *y, uint64_t ys, kq_diagnostic *diag) {
    kq_launch_norm l;
    uint64_t w;
    int gated;
    kq_status st;
    kq_diagnostic_clear(diag);
    if (c == NULL || v == NULL || x == NULL || y == NULL || v->groups == 0u || v->width == 0u ||
        v->gate_activation > KQ_HIP_ACTIVATION_SILU || v->weight_per_group > 1u || tokens == 0u)
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT, "complete norm arguments are required");
    gated = v->gate_activation != KQ_HIP_ACTIVATION_NONE;
    if (gated && gate == NULL)
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT, "the norm's gate is required");
    if (!isfinite(v->epsilon) || !(v->epsilon > 0.0f) || !isfinite(v->weight_offset))
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT,
                       "the norm needs a positive epsilon and a finite weight offset");
    if (v->width > KQ_MAX_WIDTH || (uint64_t)v->groups * v->width > (1u << 22) || tokens > KQ_MAX_TOKENS)
        return kq_fail(diag, KQ_STATUS_LIMIT_EXCEEDED,
                       "norm: groups of at most %u, rows of 2^22, %u tokens", KQ_MAX_WIDTH,
                       KQ_MAX_TOKENS);
    w = (uint64_t)v->groups * v->width;
    if (!stride_ok(xs, w) || !stride_ok(ys, w) || (gated && !stride_ok(gs, w)))
        return kq_fail(diag, KQ_STATUS_DIMENSION_MISMATCH, "row strides hold the groups and at most 2^22 floats");
    if (!on(x, 4u) || !on(y, 4u) || (gated && !on(gate, 4u)) || !on(v->weight, 4u))
        return kq_fail(diag, KQ_STATUS_INVALID_ALIGNMENT, "norm buffers need 4-byte alignment");
    {
        const span out = {y, rows_span(tokens, ys, w)};
        const span xi = {x, rows_span(tokens, xs, w)};
        const span gi = {gated ? gate : NULL, rows_span(tokens, gs, w)};
        const span wi = {v->weight, v->weight_per_group ? w : v->width};
        if ((overlap(out, xi) && !(x == y && xs == ys)) ||
            (overlap(out, gi) && !(gate == y && gs == ys)) || overlap(out, wi))
            return kq_fail(diag, KQ_STATUS_ALIASING_VIOLATION,
                           "the norm's output may only be its input or its gate, row for row");
    }
    st = kqi_context_begin(c, diag);
    if (st == KQ_STATUS_OK) {
        void *const outs[1] = {y};
        const uint64_t lens[1] = {rows_span(tokens, ys, w) * 4u};
        st = kqi_context_snapshot(c, 1u, outs, lens, diag);
    }
    if (st != KQ_STATUS_OK) return st;
    l.groups = v->groups;
    l.width = v->width;
    l.epsilon = v->epsilon;
    l.offset = v->weight_offset;
    l.weight = v->weight;
    l.per_group = v->weight_per_group;
    l.gate = v->gate_activation;
    return kqi_context_finish(c,
                              (int)kq_launch_gated_norm(&l, tokens, x, xs, gated ? gate : NULL, gs,
                                                        y, ys, kqi_context_status_word(c),
                                                        (hipStream_t)kqi_context_stream_ptr(c)),
                              "norm launch", diag);
}

kq_status kq_hip_block_join_f32(kq_hip_context *c, const kq_hip_block_join *v, uint64_t tokens,
                                const float *block, const float *gate, const float *residual,
                                const float *branch_gate, float *residual_out, float *normalized,
                                kq_diagnostic *diag) {
    kq_launch_join l;
    uint64_t hf, bf;
    int gated;
    kq_status st;
    kq_diagnostic_clear(diag);
    if (c == NULL || v == NULL || block == NULL || residual == NULL || residual_out == NULL ||
        v->branch_count == 0u || v->hidden_size == 0u || tokens == 0u ||
        v->gate_activation > KQ_HIP_ACTIVATION_SILU)
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT, "complete block join arguments are required");
    gated = v->gate_activation != KQ_HIP_ACTIVATION_NONE;
    if (gated && gate == NULL)
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT, "the block join's gate is required");
    if ((v->pre_weight == NULL) != (normalized == NULL))
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT,
                       "the next norm's weight and its output go together");
    if (!isfinite(v->residual_scale) || !isfinite(v->post_offset) || !isfinite(v->pre_offset) ||
        ((v->post_weight != NULL || v->pre_weight != NULL) &&
         !(isfinite(v->epsilon) && v->epsilon > 0.0f)))
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT,
                       "the block join needs finite scales and, for a norm, a positive epsilon");
    if (v->hidden_size > KQ_MAX_WIDTH || v->branch_count > 64u || tokens > KQ_MAX_TOKENS)
        return kq_fail(diag, KQ_STATUS_LIMIT_EXCEEDED,
                       "block join: hidden at most %u, 64 branches, %u tokens", KQ_MAX_WIDTH,
                       KQ_MAX_TOKENS);
    if (!on(block, 4u) || (gated && !on(gate, 4u)) || !on(residual, 4u) || !on(branch_gate, 4u) ||
        !on(residual_out, 4u) || !on(normalized, 4u) || !on(v->post_weight, 4u) ||
        !on(v->pre_weight, 4u))
        return kq_fail(diag, KQ_STATUS_INVALID_ALIGNMENT, "block join buffers need 4-byte alignment");
    hf = tokens * v->hidden_size;
    bf = hf * v->branch_count;
    {
        const span outs[2] = {{residual_out, bf}, {normalized, bf}};
        const span ins[6] = {{residual, bf},
                             {block, hf},
                             {gated ? gate : NULL, hf},
                             {branch_gate, tokens * v->branch_count},
                             {v->post_weight, v->hidden_size},
                             {v->pre_weight, (uint64_t)v->branch_count * v->hidden_size}};
        if (aliased(outs, 2u, ins, 6u))
            return kq_fail(diag, KQ_STATUS_ALIASING_VIOLATION,
                           "block join outputs overlap; residual_out may only be the residual");
    }
    st = kqi_context_begin(c, diag);
    if (st == KQ_STATUS_OK) {
        void *const outs[2] = {residual_out, normalized};
        const uint64_t lens[2] = {bf * 4u, bf * 4u};
        st = kqi_context_snapshot(c, 2u, outs, lens, diag);
    }
    if (st != KQ_STATUS_OK) return st;
    l.branches = v->branch_count;
    l.hidden = v->hidden_size;
    l.epsilon = v->epsilon;
    l.post = v->post_weight;
    l.post_offset = v->post_offset;
    l.gate_kind = v->gate_activation;
    l.scale = v->residual_scale;
    l.pre = v->pre_weight;
    l.pre_offset = v->pre_offset;
    l.block = block;
    l.gate = gated ? gate : NULL;
    l.residual = residual;
    l.branch_gate = branch_gate;
    l.residual_out = residual_out;
    l.normalized = normalized;
    return kqi_context_finish(c,
                              (int)kq_launch_block_join(&l, tokens, kqi_context_status_word(c),
                                                        (hipStream_t)kqi_context_stream_ptr(c)),
                              "block join launch", diag);
}

/*
 * kq_hip_paged.c — host side of softmax attention over a paged cache
 * (include/kq_hip.h: rotary positions, the cache, the attention).
 *
 * C17. Everything that the host can see is checked before any device work;
 * what lies in device memory (offsets, slots, lengths, page numbers) is
 * checked by the kernels before they index with it.
 */
#include <math.h>
#include <stdint.h>
#include <string.h>

#include "kq_gguf.h"
#include "kq_hip.h"
#include "kq_hip_checks.h"
#include "kq_hip_internal.h"

#define KQ_MAX_HEAD 1024u
#define KQ_MAX_HEADS 256u
#define KQ_MAX_CONTEXT (UINT64_C(1) << 24)

/* Rows of `width` floats, a stride apart */
typedef struct rows_of {
    const float *p;
    uint64_t stride, width;
} rows_of;

/* Whether n rows of a and of b share a value: as spans, unless both have one
 * stride and lie beside each other in its rows (a projection's parts). */
static int rows_overlap(rows_of a, rows_of b, uint64_t n) {
    const span sa = {a.p, rows_span(n, a.stride, a.width)};
    const span sb = {b.p, rows_span(n, b.stride, b.width)};
    if (!overlap(sa, sb)) return 0;
    if (a.stride == b.stride && on(a.p, 4u) && on(b.p, 4u)) {
        const uint64_t d = ((uintptr_t)b.p - (uintptr_t)a.p) / 4u;
        /* b's column in a's rows; a's addresses may be the higher ones */
        const uint64_t col = (uintptr_t)b.p >= (uintptr_t)a.p
                                 ? d % a.stride
                                 : (a.stride - ((uintptr_t)a.p - (uintptr_t)b.p) / 4u % a.stride) %
                                       a.stride;
        return !(col >= a.width && col + b.width <= a.stride);
    }
    return 1;
}

static int rows_on_span(rows_of a, uint64_t n, span b) {
    const span sa = {a.p, rows_span(n, a.stride, a.width)};
    return overlap(sa, b);
}

/* ------------------------------------------------------------------ */

kq_status kq_hip_rotary_frequencies(const kq_hip_rotary_scaling *v, uint32_t dims, double *out,
                                    float *magnitude, kq_diagnostic *diag) {
    const double turn = 6.283185307179586476925;
    double low = 0.0, high = 0.0;
    kq_diagnostic_clear(diag);
    if (v == NULL || out == NULL || magnitude == NULL)
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT, "a scaling and places for its results are required");
    if (dims == 0u || dims % 2u != 0u || dims > KQ_MAX_HEAD)
        return kq_fail(diag, KQ_STATUS_LIMIT_EXCEEDED, "rotary dims are even, 2 .. %u", KQ_MAX_HEAD);
    if (!isfinite(v->base) || !(v->base > 1.0) || v->kind > KQ_HIP_ROTARY_SCALING_BANDS ||
        (v->kind != KQ_HIP_ROTARY_SCALING_NONE && !(isfinite(v->factor) && v->factor >= 1.0)))
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT,
                       "rotary frequencies need a base above 1, a known scaling and a factor of at "
                       "least 1");
    if (v->kind == KQ_HIP_ROTARY_SCALING_BANDS &&
        (!isfinite(v->original_context) || !(v->original_context >= 1.0) || !isfinite(v->fast) ||
         !(v->slow > 0.0) || !(v->fast > v->slow)))
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT,
                       "bands need the original context and fast > slow > 0");
    if (v->divisors != NULL)
        for (uint32_t i = 0; i < dims / 2u; ++i)
            if (!isfinite(v->divisors[i]) || !(v->divisors[i] > 0.0f))
                return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT,
                               "rotary divisors are finite and above 0");
    if (v->kind == KQ_HIP_ROTARY_SCALING_BANDS) {
        /* the index whose plain frequency turns `fast` (`slow`) times in the
         * original context: base^(-2 i / dims) context = 2 pi turns */
        const double per = (double)dims / (2.0 * log(v->base));
        low = floor(per * log(v->original_context / (turn * v->fast)));
        high = ceil(per * log(v->original_context / (turn * v->slow)));
        if (high <= 0.0) low = -1.0; /* none turns more than `slow` times */
        else if (low < 0.0) low = 0.0;
        if (high > (double)dims - 1.0) high = (double)dims - 1.0;
        if (high - low < 0.001) high = low + 0.001;
    }
    for (uint32_t i = 0; i < dims / 2u; ++i) {
        double f = pow(v->base, -2.0 * (double)i / (double)dims);
        if (v->divisors != NULL) f /= (double)v->divisors[i];
        if (v->kind == KQ_HIP_ROTARY_SCALING_LINEAR) f /= v->factor;
        if (v->kind == KQ_HIP_ROTARY_SCALING_BANDS) {
            double slow = ((double)i - low) / (high - low);
            slow = slow < 0.0 ? 0.0 : slow > 1.0 ? 1.0 : slow;
            f = f * (1.0 - slow) + f / v->factor * slow;
        }
        out[i] = f;
    }
    *magnitude = v->kind == KQ_HIP_ROTARY_SCALING_BANDS ? (float)(0.1 * log(v->factor) + 1.0) : 1.0f;
    return KQ_STATUS_OK;
}

static kq_status rotary_ok(const kq_hip_rotary *r, uint32_t width, kq_diagnostic *diag) {
    if (r == NULL || r->frequencies == NULL || r->layout > KQ_HIP_ROTARY_PAIRS ||
        !isfinite(r->magnitude))
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT,
                       "a rotation needs frequencies, a layout and a finite magnitude");
    if (r->dims == 0u || r->dims % 2u != 0u || r->dims > KQ_MAX_HEAD)
        return kq_fail(diag, KQ_STATUS_LIMIT_EXCEEDED, "rotary dims are even, 2 .. %u", KQ_MAX_HEAD);
    if (r->dims > width)
        return kq_fail(diag, KQ_STATUS_DIMENSION_MISMATCH, "a head has the values that turn");
    if (!on(r->frequencies, 8u))
        return kq_fail(diag, KQ_STATUS_INVALID_ALIGNMENT, "rotary frequencies need 8-byte alignment");
    return KQ_STATUS_OK;
}

static kq_launch_rotary launch_rotary(const kq_hip_rotary *r) {
    kq_launch_rotary l;
    memset(&l, 0, sizeof l);
    if (r == NULL) return l;
    l.dims = r->dims;
    l.pairs = r->layout == KQ_HIP_ROTARY_PAIRS;
    l.magnitude = r->magnitude;
    l.frequencies = r->frequencies;
    return l;
}

kq_status kq_hip_rotary_f32(kq_hip_context *c, const kq_hip_rotary *r, uint32_t heads,
                            uint32_t width, uint64_t tokens, const uint32_t *positions,
                            const float *x, uint64_t xs, float *y, uint64_t ys,
                            kq_diagnostic *diag) {
    kq_launch_rotary l;
    uint64_t w;
    kq_status st;
    kq_diagnostic_clear(diag);
    if (c == NULL || r == NULL || x == NULL || y == NULL || heads == 0u || width == 0u ||
        tokens == 0u)
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT, "complete rotary arguments are required");
    if (width > KQ_MAX_HEAD || (uint64_t)heads * width > (1u << 22) || tokens > KQ_MAX_TOKENS)
        return kq_fail(diag, KQ_STATUS_LIMIT_EXCEEDED,
                       "rotary: heads of at most %u, rows of 2^22, %u tokens", KQ_MAX_HEAD,
                       KQ_MAX_TOKENS);
    st = rotary_ok(r, width, diag);
    if (st != KQ_STATUS_OK) return st;
    w = (uint64_t)heads * width;
    if (!stride_ok(xs, w) || !stride_ok(ys, w))
        return kq_fail(diag, KQ_STATUS_DIMENSION_MISMATCH, "row strides hold the heads and at most 2^22 floats");
    if (!on(x, 4u) || !on(y, 4u) || !on(positions, 4u))
        return kq_fail(diag, KQ_STATUS_INVALID_ALIGNMENT, "rotary buffers need 4-byte alignment");
    {
        const rows_of out = {y, ys, w}, in = {x, xs, w};
        const span f = {r->frequencies, r->dims}; /* doubles: two floats each, half as many */
        const span p = {positions, tokens};
        if ((!(x == y && xs == ys) && rows_overlap(out, in, tokens)) ||
            rows_on_span(out, tokens, f) || rows_on_span(out, tokens, p))
            return kq_fail(diag, KQ_STATUS_ALIASING_VIOLATION,
                           "the rotation's output may only be its input, row for row");
    }
    st = kqi_context_begin(c, diag);
    if (st == KQ_STATUS_OK) {
        void *const outs[1] = {y};
        const uint64_t lens[1] = {rows_span(tokens, ys, w) * 4u};
        st = kqi_context_snapshot(c, 1u, outs, lens, diag);
    }
    if (st != KQ_STATUS_OK) return st;
    l = launch_rotary(r);
    return kqi_context_finish(c,
                              (int)kq_launch_rotary_rows(&l, heads, width, tokens, positions, x, xs,
                                                         y, ys, kqi_context_status_word(c),
                                                         (hipStream_t)kqi_context_stream_ptr(c)),
                              "rotary launch", diag);
}

/* ------------------------------------------------------------------ */

static uint64_t pool_values(const kq_hip_paged_cache *v) {
    return (uint64_t)v->page_count * v->heads * v->page_tokens * v->width;
}

static kq_status cache_shape_ok(const kq_hip_paged_cache *v, kq_diagnostic *diag) {
    if (v == NULL || v->heads == 0u || v->page_count == 0u || v->table_pages == 0u)
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT, "a cache needs heads, pages and a table");
    if (v->type_id != KQ_HIP_TYPE_F16 && v->type_id != KQ_GGUF_TYPE_BF16)
        return kq_fail(diag, KQ_STATUS_UNSUPPORTED_TENSOR_TYPE, "a cache is F16 or BF16");
    if (v->heads > KQ_MAX_HEADS || (v->width != 64u && v->width != 128u && v->width != 256u) ||
        v->page_tokens < 16u || v->page_tokens > 256u ||
        (v->page_tokens & (v->page_tokens - 1u)) != 0u ||
        (uint64_t)v->table_pages * v->page_tokens > KQ_MAX_CONTEXT)
        return kq_fail(diag, KQ_STATUS_LIMIT_EXCEEDED,
                       "cache: at most %u heads of width 64, 128 or 256, pages of 16, 32, 64, 128 "
                       "or 256 tokens, lines of at most 2^24 tokens", KQ_MAX_HEADS);
    return KQ_STATUS_OK;
}

static kq_status cache_ok(const kq_hip_paged_cache *v, kq_diagnostic *diag) {
    const kq_status st = cache_shape_ok(v, diag);
    if (st != KQ_STATUS_OK) return st;
    if (v->keys == NULL || v->values == NULL || v->table == NULL || v->lengths == NULL)
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT,
                       "a cache needs keys, values, a table and lengths");
    if (!on(v->keys, 16u) || !on(v->values, 16u) || !on(v->table, 4u) || !on(v->lengths, 4u))
        return kq_fail(diag, KQ_STATUS_INVALID_ALIGNMENT,
                       "keys and values need 16-byte alignment, the table and lengths 4");
    return KQ_STATUS_OK;
}

static kq_launch_paged launch_cache(const kq_hip_paged_cache *v) {
    kq_launch_paged l;
    l.bf16 = v->type_id == KQ_GGUF_TYPE_BF16;
    l.heads = v->heads;
    l.width = v->width;
    l.page_shift = 0u;
    while ((1u << l.page_shift) < v->page_tokens) ++l.page_shift;
    l.page_count = v->page_count;
    l.table_pages = v->table_pages;
    l.keys = v->keys;
    l.values = v->values;
    l.table = v->table;
    l.lengths = v->lengths;
    return l;
}

/* what the device reads to find a sequence's rows and pages */
#define KQ_INDEX_SPANS 5u
static void index_spans(const kq_hip_paged_cache *v, const kq_hip_sequences *q,
                        span out[KQ_INDEX_SPANS]) {
    out[0] = (span){v->table, (uint64_t)q->slot_count * v->table_pages};
    out[1] = (span){v->lengths, q->slot_count};
    out[2] = (span){q->offsets, (uint64_t)q->sequence_count + 1u};
    out[3] = (span){q->slots, q->sequence_count};
    out[4] = (span){q->fresh, q->sequence_count};
}

kq_status kq_hip_cache_append_f32(kq_hip_context *c, const kq_hip_paged_cache *v,
                                  const kq_hip_sequences *q, const kq_hip_cache_rows *in,
                                  const kq_hip_rotary *r, kq_diagnostic *diag) {
    kq_launch_paged lc;
    kq_launch_seqs ls;
    kq_launch_append la;
    kq_launch_rotary lr;
    uint64_t w, qw = 0u, n;
    int turned;
    kq_status st;
    kq_diagnostic_clear(diag);
    if (c == NULL || v == NULL || in == NULL || in->key == NULL || in->value == NULL)
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT, "complete cache arguments are required");
    turned = in->query_heads != 0u;
    if (turned && (in->query == NULL || in->query_output == NULL))
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT, "the queries and their output are required");
    st = cache_ok(v, diag);
    if (st == KQ_STATUS_OK) st = sequences_ok(q, diag);
    if (st == KQ_STATUS_OK && r != NULL) st = rotary_ok(r, v->width, diag);
    if (st != KQ_STATUS_OK) return st;
    if (in->query_heads > KQ_MAX_HEADS)
        return kq_fail(diag, KQ_STATUS_LIMIT_EXCEEDED, "at most %u query heads", KQ_MAX_HEADS);
    n = q->token_count;
    w = (uint64_t)v->heads * v->width;
    qw = (uint64_t)in->query_heads * v->width;
    if (!stride_ok(in->key_stride, w) || !stride_ok(in->value_stride, w) ||
        (turned && (!stride_ok(in->query_stride, qw) || !stride_ok(in->query_output_stride, qw))))
        return kq_fail(diag, KQ_STATUS_DIMENSION_MISMATCH, "row strides hold the heads and at most 2^22 floats");
    if (!on(in->key, 16u) || !on(in->value, 16u) || in->key_stride % 4u != 0u ||
        in->value_stride % 4u != 0u ||
        (turned && (!on(in->query, 16u) || !on(in->query_output, 16u) ||
                    in->query_stride % 4u != 0u || in->query_output_stride % 4u != 0u)))
        return kq_fail(diag, KQ_STATUS_INVALID_ALIGNMENT,
                       "keys, values and queries need 16-byte alignment");
    {
        const span pools[2] = {{v->keys, pool_values(v) / 2u}, {v->values, pool_values(v) / 2u}};
        const rows_of key = {in->key, in->key_stride, w}, value = {in->value, in->value_stride, w};
        const rows_of query = {turned ? in->query : NULL, in->query_stride, qw};
        const rows_of out = {turned ? in->query_output : NULL, in->query_output_stride, qw};
        const span f = {r != NULL ? r->frequencies : NULL, r != NULL ? r->dims : 0u};
        span index[KQ_INDEX_SPANS];
        int bad = overlap(pools[0], pools[1]);
        index_spans(v, q, index);
        for (uint32_t i = 0; i < 2u; ++i) {
            bad |= rows_on_span(key, n, pools[i]) || rows_on_span(value, n, pools[i]) ||
                   overlap(f, pools[i]);
            if (turned) bad |= rows_on_span(query, n, pools[i]) || rows_on_span(out, n, pools[i]);
            for (uint32_t j = 0; j < KQ_INDEX_SPANS; ++j) bad |= overlap(pools[i], index[j]);
        }
        if (turned) {
            bad |= rows_overlap(out, key, n) || rows_overlap(out, value, n) ||
                   (!(query.p == out.p && query.stride == out.stride) &&
                    rows_overlap(out, query, n)) ||
                   rows_on_span(out, n, f);
            for (uint32_t j = 0; j < KQ_INDEX_SPANS; ++j) bad |= rows_on_span(out, n, index[j]);
        }
        if (bad)
            return kq_fail(diag, KQ_STATUS_ALIASING_VIOLATION,
                           "the pages or the turned queries overlap; query_output may only be the "
                           "query, row for row");
    }
    st = kqi_context_begin(c, diag);
    if (st == KQ_STATUS_OK && turned) {
        void *const outs[1] = {in->query_output};
        const uint64_t lens[1] = {rows_span(n, in->query_output_stride, qw) * 4u};
        st = kqi_context_snapshot(c, 1u, outs, lens, diag);
    } else if (st == KQ_STATUS_OK) {
        st = kqi_context_snapshot(c, 0u, NULL, NULL, diag);
    }
    if (st != KQ_STATUS_OK) return st;
    lc = launch_cache(v);
    ls = launch_seqs(q);
    lr = launch_rotary(r);
    la.k = in->key;
    la.v = in->value;
    la.q = in->query;
    la.qo = in->query_output;
    la.ks = in->key_stride;
    la.vs = in->value_stride;
    la.qs = in->query_stride;
    la.qos = in->query_output_stride;
    la.query_heads = in->query_heads;
    return kqi_context_finish(c,
                              (int)kq_launch_cache_append(&lc, &ls, &la, &lr,
                                                          kqi_context_status_word(c),
                                                          (hipStream_t)kqi_context_stream_ptr(c)),
                              "cache append launch", diag);
}

/* ------------------------------------------------------------------ */

static kq_status attention_ok(const kq_hip_paged_attention *a, const kq_hip_paged_cache *v,
                              kq_diagnostic *diag) {
    if (a == NULL || a->query_heads == 0u || a->causal > 1u || !isfinite(a->scale) ||
        (a->gate_activation != KQ_HIP_ACTIVATION_NONE &&
         a->gate_activation != KQ_HIP_ACTIVATION_SIGMOID))
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT,
                       "attention needs query heads, a finite scale and no gate or a sigmoid");
    if (a->query_heads > KQ_MAX_HEADS)
        return kq_fail(diag, KQ_STATUS_LIMIT_EXCEEDED, "at most %u query heads", KQ_MAX_HEADS);
    if (a->query_heads % v->heads != 0u)
        return kq_fail(diag, KQ_STATUS_DIMENSION_MISMATCH,
                       "the query heads are a multiple of the cache's");
    return KQ_STATUS_OK;
}

static kq_launch_pattn launch_pattn(const kq_hip_paged_attention *a) {
    kq_launch_pattn l;
    memset(&l, 0, sizeof l);
    l.query_heads = a->query_heads;
    l.scale = a->scale;
    l.causal = a->causal;
    l.window = a->window;
    l.sinks = a->sinks;
    l.gated = a->gate_activation == KQ_HIP_ACTIVATION_SIGMOID;
    return l;
}

uint64_t kq_hip_paged_attention_scratch_bytes(const kq_hip_paged_attention *a,
                                              const kq_hip_paged_cache *v,
                                              const kq_hip_sequences *q) {
    kq_launch_pattn l;
    kq_launch_paged lc;
    kq_launch_seqs ls;
    if (cache_shape_ok(v, NULL) != KQ_STATUS_OK || attention_ok(a, v, NULL) != KQ_STATUS_OK ||
        sequences_ok(q, NULL) != KQ_STATUS_OK)
        return 0u;
    l = launch_pattn(a);
    lc = launch_cache(v);
    ls = launch_seqs(q);
    return kq_launch_pattn_scratch(&l, &lc, &ls);
}

kq_status kq_hip_paged_attention_f32(kq_hip_context *c, const kq_hip_paged_attention *a,
                                     const kq_hip_paged_cache *v, const kq_hip_sequences *q,
                                     const float *query, uint64_t qs, const float *gate,
                                     uint64_t gs, float *y, uint64_t ys, void *scratch,
                                     uint64_t scratch_bytes, kq_diagnostic *diag) {
    kq_launch_pattn l;
    kq_launch_paged lc;
    kq_launch_seqs ls;
    uint64_t w, need, n;
    int gated;
    kq_status st;
    kq_diagnostic_clear(diag);
    if (c == NULL || a == NULL || v == NULL || query == NULL || y == NULL)
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT, "complete attention arguments are required");
    st = cache_ok(v, diag);
    if (st == KQ_STATUS_OK) st = attention_ok(a, v, diag);
    if (st == KQ_STATUS_OK) st = sequences_ok(q, diag);
    if (st != KQ_STATUS_OK) return st;
    gated = a->gate_activation != KQ_HIP_ACTIVATION_NONE;
    if (gated && gate == NULL)
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT, "the attention's gate is required");
    n = q->token_count;
    w = (uint64_t)a->query_heads * v->width;
    if (!stride_ok(qs, w) || !stride_ok(ys, w) || (gated && !stride_ok(gs, w)))
        return kq_fail(diag, KQ_STATUS_DIMENSION_MISMATCH, "row strides hold the heads and at most 2^22 floats");
    need = kq_hip_paged_attention_scratch_bytes(a, v, q);
    if (need != 0u && scratch == NULL)
        return kq_fail(diag, KQ_STATUS_INVALID_ARGUMENT, "attention scratch is required");
    if (scratch_bytes < need)
        return kq_fail(diag, KQ_STATUS_BUFFER_TOO_SMALL, "attention scratch needs %llu bytes",
                       (unsigned long long)need);
    if (!on(query, 16u) || !on(y, 16u) || (gated && !on(gate, 16u)) || !on(scratch, 16u) ||
        qs % 4u != 0u || ys % 4u != 0u || (gated && gs % 4u != 0u) || !on(a->sinks, 4u))
        return kq_fail(diag, KQ_STATUS_INVALID_ALIGNMENT,
                       "queries, gate, output and scratch need 16-byte alignment, sinks 4");
    {
        const rows_of out = {y, ys, w}, in = {query, qs, w}, ga = {gated ? gate : NULL, gs, w};
        const span work = {scratch, need / 4u};
        span index[KQ_INDEX_SPANS];
        const span other[3] = {{v->keys, pool_values(v) / 2u}, {v->values, pool_values(v) / 2u},
                               {a->sinks, a->query_heads}};
        int bad = rows_overlap(out, in, n) || (gated && rows_overlap(out, ga, n)) ||
                  rows_on_span(out, n, work) || rows_on_span(in, n, work) ||
                  (gated && rows_on_span(ga, n, work));
        index_spans(v, q, index);
        for (uint32_t i = 0; i < 3u; ++i)
            bad |= rows_on_span(out, n, other[i]) || overlap(work, other[i]);
        for (uint32_t i = 0; i < KQ_INDEX_SPANS; ++i)
            bad |= rows_on_span(out, n, index[i]) || overlap(work, index[i]);
        if (bad)
            return kq_fail(diag, KQ_STATUS_ALIASING_VIOLATION,
                           "the attention's output or scratch overlaps what it reads");
    }
    st = kqi_context_begin(c, diag);
    if (st == KQ_STATUS_OK) {
        void *const outs[1] = {y};
        const uint64_t lens[1] = {rows_span(n, ys, w) * 4u};
        st = kqi_context_snapshot(c, 1u, outs, lens, diag);
    }
    if (st != KQ_STATUS_OK) return st;
    l = launch_pattn(a);
    l.q = query;
    l.qs = qs;
    l.gate = gated ? gate : NULL;
    l.gs = gs;
    l.y = y;
    l.ys = ys;
    lc = launch_cache(v);
    ls = launch_seqs(q);
    return kqi_context_finish(c,
                              (int)kq_launch_pattn_run(&l, &lc, &ls, scratch,
                                                       kqi_context_status_word(c),
                                                       (hipStream_t)kqi_context_stream_ptr(c)),
                              "attention launch", diag);
}

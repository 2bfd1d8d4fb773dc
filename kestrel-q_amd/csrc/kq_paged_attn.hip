/*
 * kq_paged_attn.hip — softmax attention of a call's rows over a paged cache
 * on gfx950 (include/kq_hip.h, kq_hip_paged_attention_f32).
 */
#include "kq_device.h"
#include "kq_dma.h"
#include "kq_launch.h"
#include "kq_paged.h"

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) char lds_char;

constexpr int kThreads = 256, kWaves = 4;
constexpr uint32_t kTile = 64;       /* keys of a tile */
constexpr uint32_t kFew = 16;        /* rows of an item whose waves share out its keys */
constexpr uint32_t kMany = 128;      /* rows of an item whose waves share out its rows */
constexpr uint32_t kLeast = 2;       /* tiles of a part */
constexpr uint32_t kTarget = 1024;   /* parts that the device is filled with */
constexpr uint32_t kSlots = 2u * kTarget;
constexpr uint32_t kByLane = 64;     /* sequences that each wave plans by itself */
constexpr float kSlack = 8.0f;       /* by which a row's largest exponent may pass its stand-in */
constexpr float kLowest = -0x1.fffffep127f;

struct Args {
    kq_launch_pattn a;
    kq_launch_paged c;
    kq_launch_seqs q;
    uint32_t group;     /* query heads of a key head */
    uint32_t slot_rows; /* rows that a slot of the partial results holds */
    uint32_t slots;
    double exponent;    /* scale log2(e) */
    float *partial;     /* slots of [slot_rows][width] sums, then tops, then totals */
    uint32_t *plan;     /* [0]: tiles a part, [1]: parts; then first parts, then first slots of
                           the sequences */
};

/* ---------------------------------------------------------------- the plan */

/* What a sequence asks for: its items (blocks of rows, for each key head) and
 * the tiles of keys that an item reads at most. */
struct Need {
    uint32_t blocks, tiles;
};

__device__ __forceinline__ uint32_t rows_of_block(const Args &g, uint32_t rows) {
    return (uint64_t)rows * g.group <= kFew ? kFew : kMany;
}

__device__ __forceinline__ Need need_of(const Args &g, const kq::PagedSeq &s) {
    Need n = {0u, 0u};
    if (!s.live || s.rows == 0u) return n;
    const uint32_t rows = s.rows * g.group, block = rows_of_block(g, s.rows);
    n.blocks = (rows + block - 1u) / block;
    n.tiles = (s.past + s.rows + kTile - 1u) / kTile;
    if (g.a.window != 0u && g.a.causal != 0u) {
        /* keys from the first token's window to the last token of a block */
        const uint32_t span = (rows < block ? rows - 1u : block - 1u) / g.group + 1u;
        const uint64_t keys = (uint64_t)g.a.window + span;
        const uint64_t most = (keys + kTile - 1u) / kTile + 1u;
        if (most < n.tiles) n.tiles = (uint32_t)most;
    }
    return n;
}

__device__ __forceinline__ uint64_t cost_of(const Args &g, const Need &n) {
    return (uint64_t)n.blocks * g.c.heads * n.tiles;
}

/* tiles a part, of all sequences' cost: kTarget parts, not too short ones */
__device__ __forceinline__ uint32_t part_tiles(uint64_t cost) {
    const double t = ceil((double)cost * (1.0 / (double)kTarget));
    return t < (double)kLeast ? kLeast : (uint32_t)t;
}

__device__ __forceinline__ uint32_t parts_of(const Need &n, uint32_t length) {
    return n.tiles == 0u ? 0u : (n.tiles + length - 1u) / length;
}

/* One part of the work */
struct Part {
    kq::PagedSeq seq;
    uint32_t row0, rows;  /* of the sequence's rows x group */
    uint32_t block;       /* kFew or kMany */
    uint32_t head;
    uint32_t part, parts; /* this one, and how many the item really has */
    uint32_t t0, t1;      /* its tiles */
    uint32_t key0, key1;  /* keys that any of the item's rows sees */
    uint32_t slot, step;  /* of the item's first part, and between two parts */
    bool live;
};

__device__ __forceinline__ Part part_of(const Args &g, const kq::PagedSeq &s, const Need &n,
                                        uint32_t length, uint32_t u, uint32_t first_slot) {
    Part p;
    p.seq = s;
    p.block = rows_of_block(g, s.rows);
    const uint32_t parts = parts_of(n, length);
    p.head = u % g.c.heads;
    u /= g.c.heads;
    p.part = u % parts;
    u /= parts;
    /* the last rows, which see the most keys, first */
    p.row0 = (n.blocks - 1u - u) * p.block;
    const uint32_t all = s.rows * g.group;
    p.rows = all - p.row0 < p.block ? all - p.row0 : p.block;
    const uint32_t ta = p.row0 / g.group, tb = (p.row0 + p.rows - 1u) / g.group;
    p.key1 = g.a.causal ? s.past + tb + 1u : s.past + s.rows;
    p.key0 = 0u;
    if (g.a.window != 0u && s.past + ta + 1u > g.a.window) p.key0 = s.past + ta + 1u - g.a.window;
    const uint32_t a = p.key0 / kTile, tiles = (p.key1 + kTile - 1u) / kTile - a;
    p.parts = (tiles + length - 1u) / length;
    const uint32_t each = (tiles + p.parts - 1u) / p.parts;
    p.t0 = a + p.part * each;
    p.t1 = p.t0 + each < a + tiles ? p.t0 + each : a + tiles;
    p.slot = first_slot + u * parts * g.c.heads + p.head;
    p.step = g.c.heads;
    /* offsets that overlap could ask for more slots than there are */
    p.live = p.part < p.parts &&
             (p.parts == 1u || p.slot + (p.parts - 1u) * p.step < g.slots);
    return p;
}

__device__ __forceinline__ uint64_t lanes_add(uint64_t v) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d, KQ_WAVE);
    return v;
}
__device__ __forceinline__ uint32_t lanes_before(uint32_t v) {
    uint32_t sum = v;
    const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t o = __shfl_up(sum, d, KQ_WAVE);
        if (lane >= (uint32_t)d) sum += o;
    }
    return sum - v;
}

/* Part `index` of the call, the same in all lanes. Up to kByLane sequences:
 * a lane looks at each, and every wave adds up for itself. More: plan_many
 * has done so. */
template <bool MANY>
__device__ __forceinline__ Part find_part(const Args &g, uint32_t index, bool report,
                                          uint32_t *status) {
    Part p;
    p.live = false;
    bool bad = false;
    if constexpr (!MANY) {
        const uint32_t lane = threadIdx.x & 63u;
        kq::PagedSeq s = {0u, 0u, 0u, 0u, false};
        if (lane < g.q.count) s = kq::paged_seq(g.q, g.c, lane, bad);
        if (report && bad) kq_flag(status, KQ_DEV_SEQUENCE);
        const Need n = need_of(g, s);
        const uint32_t length = part_tiles(lanes_add(cost_of(g, n)));
        const uint32_t each = parts_of(n, length), mine = n.blocks * g.c.heads * each;
        const uint32_t first = lanes_before(mine);
        const uint32_t first_slot = lanes_before(each > 1u ? mine : 0u);
        const uint64_t m = __ballot(index >= first && index - first < mine);
        if (m == 0ull) return p;
        const int at = __builtin_amdgcn_readfirstlane((int)__builtin_ctzll(m));
        kq::PagedSeq w;
        w.begin = __builtin_amdgcn_readlane(s.begin, at);
        w.rows = __builtin_amdgcn_readlane(s.rows, at);
        w.past = __builtin_amdgcn_readlane(s.past, at);
        w.slot = __builtin_amdgcn_readlane(s.slot, at);
        w.live = true;
        return part_of(g, w, need_of(g, w), __builtin_amdgcn_readfirstlane(length),
                       index - __builtin_amdgcn_readlane(first, at),
                       __builtin_amdgcn_readlane(first_slot, at));
    } else {
        if (index >= g.plan[1]) return p;
        const uint32_t *first = g.plan + 2u, *slots = first + g.q.count + 1u;
        const uint32_t s = kq::wave_find(first, g.q.count, index);
        const kq::PagedSeq w = kq::paged_seq(g.q, g.c, s, bad);
        const Need n = need_of(g, w);
        const uint32_t length = g.plan[0], u = index - first[s];
        if (u >= n.blocks * g.c.heads * parts_of(n, length)) return p; /* offsets not in order */
        return part_of(g, w, n, length, u, slots[s]);
    }
}

/* One workgroup: the plan of more sequences than a wave has lanes */
__global__ __launch_bounds__(1024) void plan_many(Args g, uint32_t *status) {
    __shared__ uint64_t sums[16];
    __shared__ uint32_t parts[16], slots[16];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x / 64u;
    uint64_t cost = 0u;
    bool bad = false;
    for (uint32_t s = threadIdx.x; s < g.q.count; s += 1024u)
        cost += cost_of(g, need_of(g, kq::paged_seq(g.q, g.c, s, bad)));
    if (bad) kq_flag(status, KQ_DEV_SEQUENCE);
    cost = lanes_add(cost);
    if (lane == 0u) sums[wave] = cost;
    __syncthreads();
    cost = 0u;
    for (int w = 0; w < 16; ++w) cost += sums[w];
    const uint32_t length = part_tiles(cost);
    uint32_t *first = g.plan + 2u, *slot = first + g.q.count + 1u;
    uint32_t parts_before = 0u, slots_before = 0u;
    for (uint32_t base = 0u; base < g.q.count; base += 1024u) {
        const uint32_t s = base + threadIdx.x;
        uint32_t mine = 0u, held = 0u;
        if (s < g.q.count) {
            const Need n = need_of(g, kq::paged_seq(g.q, g.c, s, bad));
            const uint32_t each = parts_of(n, length);
            mine = n.blocks * g.c.heads * each;
            held = each > 1u ? mine : 0u;
        }
        const uint32_t p = lanes_before(mine), h = lanes_before(held);
        if (lane == 63u) {
            parts[wave] = p + mine;
            slots[wave] = h + held;
        }
        __syncthreads();
        uint32_t pw = 0u, hw = 0u, pa = 0u, ha = 0u;
        for (uint32_t w = 0; w < 16u; ++w) {
            if (w < wave) {
                pw += parts[w];
                hw += slots[w];
            }
            pa += parts[w];
            ha += slots[w];
        }
        if (s < g.q.count) {
            first[s] = parts_before + pw + p;
            slot[s] = slots_before + hw + h;
        }
        parts_before += pa;
        slots_before += ha;
        __syncthreads();
    }
    if (threadIdx.x == 0u) {
        g.plan[0] = length;
        g.plan[1] = parts_before;
        first[g.q.count] = parts_before;
        slot[g.q.count] = slots_before;
    }
}

/* ------------------------------------------------------------- arithmetic */

/* The cache's type as operands. A factor that is not of that type, a query or
 * a weight, is TERMS values of it: two fp16 numbers hold 22 bits, three bf16
 * numbers 24, so that the product is binary32's. */
template <bool BF>
struct Type {
    typedef _Float16 e;
    static constexpr int TERMS = 2;
    /* fp16's own range is short: a row's largest query is brought to 2^13, and
     * weights are held times 2^7, at most 2^15 with the slack */
    static constexpr int TOP = 13;
    static constexpr float LIFT = 7.0f;
};
template <>
struct Type<true> {
    typedef __bf16 e;
    static constexpr int TERMS = 3;
    static constexpr int TOP = 0;
    static constexpr float LIFT = 0.0f;
};

template <bool BF>
using e8 = typename Type<BF>::e __attribute__((ext_vector_type(8)));
template <bool BF>
using e2 = typename Type<BF>::e __attribute__((ext_vector_type(2)));

__device__ __forceinline__ f4 mma(e8<false> a, e8<false> b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f4 mma(e8<true> a, e8<true> b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f16v mma(e8<false> a, e8<false> b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f16v mma(e8<true> a, e8<true> b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

/* x[0..7] as TERMS operands whose sum it is */
template <bool BF>
__device__ __forceinline__ void split(const float (&x)[8], e8<BF> (&t)[Type<BF>::TERMS]) {
    typedef typename Type<BF>::e E;
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        float a = x[i], b = x[i + 1];
#pragma unroll
        for (int k = 0; k < Type<BF>::TERMS; ++k) {
            const E p = (E)a, q = (E)b;
            t[k][i] = p;
            t[k][i + 1] = q;
            a -= (float)p;
            b -= (float)q;
        }
    }
}

/* A row's queries, as operands: the exponent's factor put in in binary64, and
 * the row's largest value brought to 2^TOP by a power of two. */
template <bool BF, int STEPS>
struct Query {
    e8<BF> x[STEPS][Type<BF>::TERMS];
    float unscale;
};

/* at(step): 8 values of the row from there on; LANES: the lanes that share a row */
template <bool BF, int STEPS, int LANES, typename At>
__device__ __forceinline__ void load_query(Query<BF, STEPS> &q, bool some, double factor, At at,
                                           bool &badin) {
    float v[STEPS][8], top = 0.0f;
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        if (some) {
            const float4 a = *(const float4 *)at(s), b = *(const float4 *)(at(s) + 4);
            v[s][0] = a.x; v[s][1] = a.y; v[s][2] = a.z; v[s][3] = a.w;
            v[s][4] = b.x; v[s][5] = b.y; v[s][6] = b.z; v[s][7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[s][i] = 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            badin |= !kq_isfinite(v[s][i]);
            top = fmaxf(top, fabsf(v[s][i]));
        }
    }
    top = kq::lanes_max<LANES>(top);
    /* the largest value's exponent, 0 for a row of zeros */
    int e = 0;
    if (top > 0.0f && kq_isfinite(top)) e = ilogb((double)top * fabs(factor));
    e = e < -100 ? -100 : e > 126 ? 126 : e;
    const double scale = __builtin_ldexp(factor, Type<BF>::TOP - e);
    q.unscale = __builtin_ldexpf(1.0f, e - Type<BF>::TOP);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = (float)((double)v[s][i] * scale);
        split<BF>(x, q.x[s]);
    }
}

/* four values of V's column `lane & 15` in a block of 16: rows r .. r + 3 */
__device__ __forceinline__ s4 transposed(uint32_t at) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (__attribute__((address_space(3))) s4 *)(uintptr_t)at);
}

template <bool BF>
__device__ __forceinline__ e8<BF> join8(s4 a, s4 b) {
    return __builtin_bit_cast(e8<BF>, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

/* ------------------------------------------------------------ the results */

/* A piece of four values of a row, all keys in: the sink, the division and the
 * gate, and where it goes */
__device__ __forceinline__ void put(const Args &g, const kq::PagedSeq &s, uint32_t head,
                                    uint32_t row, uint32_t d, uint32_t width, f4 o, float top,
                                    float total, bool &badin, bool &bad) {
    const uint32_t h = head * g.group + row % g.group;
    const size_t token = s.begin + row / g.group;
    if (g.a.sinks != nullptr)
        total += __builtin_amdgcn_exp2f((float)((double)g.a.sinks[h] * 1.4426950408889634 - top));
    const float inv = total > 0.0f ? 1.0f / total : total; /* a NaN stays one */
    o *= inv;
    const size_t at = (size_t)h * width + d;
    if (g.a.gated) {
        const float4 e = *(const float4 *)(g.a.gate + token * g.a.gs + at);
        badin |= !kq_isfinite(e.x) || !kq_isfinite(e.y) || !kq_isfinite(e.z) || !kq_isfinite(e.w);
        o[0] *= kq::sigmoid(e.x);
        o[1] *= kq::sigmoid(e.y);
        o[2] *= kq::sigmoid(e.z);
        o[3] *= kq::sigmoid(e.w);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) bad |= !kq_isfinite(o[i]);
    *(f4 *)(g.a.y + token * g.a.ys + at) = o;
}

__device__ __forceinline__ float *slot_at(const Args &g, uint32_t slot) {
    return g.partial + (size_t)slot * g.slot_rows * (g.c.width + 2u);
}

/* a part's sums of a row, for the join */
__device__ __forceinline__ void keep(const Args &g, float *slot, uint32_t row, uint32_t d,
                                     uint32_t width, f4 o, float top, float total) {
    *(f4 *)(slot + (size_t)row * width + d) = o;
    if (d == 0u) {
        float *m = slot + (size_t)g.slot_rows * width;
        m[row] = top;
        m[g.slot_rows + row] = total;
    }
}

/* ------------------------------------------------------------------ pages */

/* 16 keys from key `at` on (a multiple of 16) of the item's head: a descriptor
 * of the page's part, and the byte where the keys begin in it. `some`: whether
 * any of them is asked for; otherwise, and for a page that is none, nothing can
 * be read through it. */
struct Place {
    const char *kp, *vp;
    uint32_t bytes, off;
    __device__ __forceinline__ kq_i4v k() const { return dma_rsrc(kp, bytes); }
    __device__ __forceinline__ kq_i4v v() const { return dma_rsrc(vp, bytes); }
};

template <int D>
__device__ __forceinline__ Place place_of(const Args &g, const Part &p, uint32_t at, bool some,
                                          bool &bad) {
    Place r;
    uint32_t page = 0u, bytes = (D * 2u) << g.c.page_shift;
    if (some) page = g.c.table[(size_t)p.seq.slot * g.c.table_pages + (at >> g.c.page_shift)];
    if (page >= g.c.page_count) {
        bad = true;
        some = false;
        page = 0u;
    }
    page = __builtin_amdgcn_readfirstlane(page);
    const uint64_t off = ((uint64_t)page * g.c.heads + p.head) * bytes;
    if (!some) bytes = 0u;
    bytes = __builtin_amdgcn_readfirstlane(bytes);
    r.kp = (const char *)g.c.keys + off;
    r.vp = (const char *)g.c.values + off;
    r.bytes = bytes;
    r.off = (at & ((1u << g.c.page_shift) - 1u)) * (D * 2u);
    return r;
}

constexpr uint32_t kOut = 0xfffffff0u; /* an offset that no page has */

/* ------------------------------------------------- few rows: keys shared out */

/* where the 16-byte piece c of V's row r lies: a transposing read takes the
 * same 32 bytes of 16 rows, which 64 banks hold 8 of at a time */
template <int D>
__device__ __forceinline__ uint32_t few_piece(uint32_t r, uint32_t c) {
    return D == 64 ? c ^ (2u * ((r >> 1) & 3u)) : c ^ (2u * (r & 7u));
}

template <int D>
constexpr uint32_t lds_bytes() {
    return 512u * D; /* 4 waves x 2 x 32 rows of V, or 2 x 64 rows of K and V */
}

/* Up to 16 rows: a wave takes every fourth 32 keys, S' = K Q' and O' = V' P' of
 * 16 x 16 x 32 products, and the waves' results are joined in LDS. */
template <bool BF, int D>
__device__ __forceinline__ void few_rows(const Args &g, const Part &p, char *lds, bool &badin,
                                         bool &bad, bool &badseq) {
    constexpr int STEPS = D / 32, BLOCKS = D / 16, TERMS = Type<BF>::TERMS;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u);
    const uint32_t n = lane & 15u, quarter = lane >> 4;
    const bool some = n < p.rows;
    const uint32_t row = p.row0 + n, token = some ? row / g.group : 0u;
    const uint32_t h = p.head * g.group + (some ? row % g.group : 0u);
    const uint32_t last = g.a.causal ? p.seq.past + token + 1u : p.seq.past + p.seq.rows;
    const uint32_t from = g.a.window != 0u && p.seq.past + token + 1u > g.a.window
                              ? p.seq.past + token + 1u - g.a.window : 0u;

    Query<BF, STEPS> q;
    const float *qp = g.a.q + (size_t)(p.seq.begin + token) * g.a.qs + (size_t)h * D + 8u * quarter;
    load_query<BF, STEPS, 48>(q, some, g.exponent, [&](int s) { return qp + 32 * s; }, badin);

    f4 o[BLOCKS];
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) o[b] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    float top = kLowest, total = 0.0f;

    const uint32_t mine = lds_addr(lds) + wave * (128u * D); /* 2 x 32 rows of V */
    e8<BF> k[2][2][STEPS];
    uint32_t key = p.t0 * kTile + wave * 32u;
    const uint32_t end = p.t1 * kTile < p.key1 ? p.t1 * kTile : p.key1;

    auto load = [&](uint32_t at, uint32_t buf, e8<BF> (&kk)[2][STEPS]) {
#pragma unroll
        for (uint32_t b = 0; b < 2u; ++b) {
            const uint32_t a16 = at + 16u * b;
            const Place pl = place_of<D>(g, p, a16, a16 < p.key1 && a16 + 16u > p.key0, badseq);
            /* V's 16 rows: D / 32 pieces of 1 KiB */
#pragma unroll
            for (uint32_t j = 0; j < D / 32u; ++j) {
                const uint32_t o16 = j * 64u + lane, r = o16 / (D / 8u), c = o16 % (D / 8u);
                const bool in = a16 + r < p.key1 && a16 + r >= p.key0;
                dma16(pl.v(), in ? pl.off + r * (2u * D) + few_piece<D>(r, c) * 16u : kOut,
                      mine + buf * (64u * D) + b * (32u * D) + j * 1024u);
            }
            const bool in = a16 + n < p.key1 && a16 + n >= p.key0;
            const auto keys = __builtin_amdgcn_make_buffer_rsrc((void *)pl.kp, 0, pl.bytes, 0x00020000);
#pragma unroll
            for (int s = 0; s < STEPS; ++s) {
                const auto w = __builtin_amdgcn_raw_buffer_load_b128(
                    keys, in ? pl.off + n * (2u * D) + 64u * s + 16u * quarter : kOut, 0, 0);
                kk[b][s] = __builtin_bit_cast(e8<BF>, w);
            }
        }
    };
    auto compute = [&](uint32_t at, uint32_t buf, const e8<BF> (&kk)[2][STEPS]) {
        f4 s[2];
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            s[b] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int t = 0; t < STEPS; ++t)
#pragma unroll
                for (int m = 0; m < TERMS; ++m) s[b] = mma(kk[b][t], q.x[t][m], s[b]);
        }
        float w[8];
        float peak = kLowest;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t key = at + 16u * (i / 4) + 4u * quarter + i % 4;
            w[i] = key < last && key >= from ? s[i / 4][i % 4] * q.unscale : -INFINITY;
            peak = fmaxf(peak, w[i]);
        }
        peak = kq::lanes_max<48>(peak) - Type<BF>::LIFT;
        if (__any(peak > top + kSlack)) {
            const float next = fmaxf(top, peak);
            const float f = __builtin_amdgcn_exp2f(top - next);
            top = next;
            total *= f;
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) o[b] *= f;
        }
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            w[i] = __builtin_amdgcn_exp2f(w[i] - top);
            sum += w[i];
        }
        total += sum;
        e8<BF> pw[TERMS];
        split<BF>(w, pw);
#pragma unroll
        for (uint32_t b = 0; b < BLOCKS; ++b) {
            const uint32_t r = 4u * quarter + n / 4u;
            const uint32_t a = mine + buf * (64u * D) + r * (2u * D) +
                               few_piece<D>(r, 2u * b + (n % 4u) / 2u) * 16u + (n & 1u) * 8u;
            const e8<BF> v = join8<BF>(transposed(a), transposed(a + 32u * D));
#pragma unroll
            for (int m = 0; m < TERMS; ++m) o[b] = mma(v, pw[m], o[b]);
        }
    };

    if (key < end) {
        load(key, 0u, k[0]);
        for (;;) {
            wait_vm<0>();
            if (key + 128u < end) load(key + 128u, 1u, k[1]);
            compute(key, 0u, k[0]);
            key += 128u;
            if (key >= end) break;
            wait_lgkm0();
            wait_vm<0>();
            if (key + 128u < end) load(key + 128u, 0u, k[0]);
            compute(key, 1u, k[1]);
            key += 128u;
            if (key >= end) break;
            wait_lgkm0();
        }
    }
    total = kq::lanes_sum<48>(total);

    /* the waves' tops, totals and sums [wave][row][d], then 16 rows by all */
    float *tops = (float *)lds, *totals = tops + kWaves * 16, *sums = totals + kWaves * 16;
    constexpr uint32_t kRow = D + 4u; /* rows 16 bytes apart in the banks */
    __syncthreads();
    if (quarter == 0u) {
        tops[wave * 16u + n] = top;
        totals[wave * 16u + n] = total;
    }
#pragma unroll
    for (uint32_t b = 0; b < BLOCKS; ++b)
        *(f4 *)(sums + (wave * 16u + n) * kRow + 16u * b + 4u * quarter) = o[b];
    __syncthreads();
    float *slot = p.parts > 1u ? slot_at(g, p.slot + p.part * p.step) : nullptr;
    for (uint32_t i = threadIdx.x; i < p.rows * (D / 4u); i += kThreads) {
        const uint32_t r = i / (D / 4u), d = i % (D / 4u) * 4u;
        float t = tops[r];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) t = fmaxf(t, tops[w * 16 + r]);
        f4 v = f4{0.0f, 0.0f, 0.0f, 0.0f};
        float l = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(tops[w * 16 + r] - t);
            l = fmaf(totals[w * 16 + r], f, l);
            const f4 x = *(const f4 *)(sums + (w * 16u + r) * kRow + d);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = fmaf(x[e], f, v[e]);
        }
        if (slot != nullptr)
            keep(g, slot, r, d, D, v, t, l);
        else
            put(g, p.seq, p.head, p.row0 + r, d, D, v, t, l, badin, bad);
    }
}

/* ------------------------------------------------ many rows: rows shared out */

/* where the 16-byte piece c of a row of K (read down 16 rows), or of V (read
 * 64 bytes of 8 rows, transposed) lies */
template <int D>
__device__ __forceinline__ uint32_t k_piece(uint32_t r, uint32_t c) {
    return D == 64 ? c ^ ((r >> 1) & 7u) : c ^ (r & 15u);
}
template <int D>
__device__ __forceinline__ uint32_t v_piece(uint32_t r, uint32_t c) {
    return D == 64 ? c ^ (((r >> 1) & 1u) << 2) : c ^ ((r & 3u) << 2);
}

/* Up to 128 rows, 32 of them a wave: K and V come into LDS once for all, two
 * buffers of 64 keys; S' = K Q' and O' = V' P' of 32 x 32 x 16 products. */
template <bool BF, int D>
__device__ __forceinline__ void many_rows(const Args &g, const Part &p, char *lds, bool &badin,
                                          bool &bad, bool &badseq) {
    constexpr int STEPS = D / 16, BLOCKS = D / 32, TERMS = Type<BF>::TERMS;
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u);
    const uint32_t n = lane & 31u, half = lane >> 5;
    const uint32_t r0 = wave * 32u;
    const bool some = r0 + n < p.rows;
    const uint32_t row = p.row0 + r0 + n, token = some ? row / g.group : 0u;
    const uint32_t h = p.head * g.group + (some ? row % g.group : 0u);
    const uint32_t last = g.a.causal ? p.seq.past + token + 1u : p.seq.past + p.seq.rows;
    const uint32_t from = g.a.window != 0u && p.seq.past + token + 1u > g.a.window
                              ? p.seq.past + token + 1u - g.a.window : 0u;
    /* the wave's rows: whether there are any, and what they see */
    const bool awake = r0 < p.rows;
    uint32_t see0 = 0u, see1 = 0u, all0 = 0u, all1 = 0u; /* any row; every row */
    if (awake) {
        const uint32_t rl = (r0 + 32u < p.rows ? r0 + 31u : p.rows - 1u) + p.row0;
        const uint32_t ta = (p.row0 + r0) / g.group, tb = rl / g.group;
        const uint32_t pa = p.seq.past + ta + 1u, pb = p.seq.past + tb + 1u;
        see1 = g.a.causal ? pb : p.seq.past + p.seq.rows;
        all1 = g.a.causal ? pa : p.seq.past + p.seq.rows;
        if (g.a.window != 0u) {
            see0 = pa > g.a.window ? pa - g.a.window : 0u;
            all0 = pb > g.a.window ? pb - g.a.window : 0u;
        }
    }

    Query<BF, STEPS> q;
    const float *qp = g.a.q + (size_t)(p.seq.begin + token) * g.a.qs + (size_t)h * D + 8u * half;
    load_query<BF, STEPS, 32>(q, some, g.exponent, [&](int s) { return qp + 16 * s; }, badin);

    f16v o[BLOCKS];
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[b][i] = 0.0f;
    float top = kLowest, total = 0.0f;

    const uint32_t base = lds_addr(lds);
    /* the wave's 16 keys of a tile, K and V: D / 32 pieces of 1 KiB each */
    auto load = [&](uint32_t t, uint32_t buf) {
        const uint32_t a16 = t * kTile + wave * 16u;
        const Place pl = place_of<D>(g, p, a16, a16 < p.key1 && a16 + 16u > p.key0, badseq);
        const uint32_t to = base + buf * (256u * D) + wave * (32u * D);
#pragma unroll
        for (uint32_t j = 0; j < D / 32u; ++j) {
            const uint32_t o16 = j * 64u + lane, r = o16 / (D / 8u), c = o16 % (D / 8u);
            const bool in = a16 + r < p.key1 && a16 + r >= p.key0;
            const uint32_t a = pl.off + r * (2u * D);
            dma16(pl.k(), in ? a + k_piece<D>(r, c) * 16u : kOut, to + j * 1024u);
            dma16(pl.v(), in ? a + v_piece<D>(r, c) * 16u : kOut, to + 128u * D + j * 1024u);
        }
    };
    auto compute = [&](uint32_t t, uint32_t buf) {
        const uint32_t kb = base + buf * (256u * D), vb = kb + 128u * D, at = t * kTile;
        f16v s[2];
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[b][i] = 0.0f;
#pragma unroll
        for (uint32_t st = 0; st < STEPS; ++st)
#pragma unroll
            for (uint32_t b = 0; b < 2u; ++b) {
                const uint32_t r = 32u * b + n;
                const u4 w = *(__attribute__((address_space(3))) u4 *)(uintptr_t)(
                    kb + r * (2u * D) + k_piece<D>(r, 2u * st + half) * 16u);
                const e8<BF> k = __builtin_bit_cast(e8<BF>, w);
#pragma unroll
                for (int m = 0; m < TERMS; ++m) s[b] = mma(k, q.x[st][m], s[b]);
            }
        if (at + kTile > all1 || at < all0) {
#pragma unroll
            for (uint32_t b = 0; b < 2u; ++b)
#pragma unroll
                for (uint32_t i = 0; i < 16u; ++i) {
                    const uint32_t key = at + 32u * b + 8u * (i / 4u) + 4u * half + i % 4u;
                    s[b][i] = key < last && key >= from ? s[b][i] : -INFINITY;
                }
        }
        float peak = s[0][0];
#pragma unroll
        for (int i = 1; i < 32; ++i) peak = fmaxf(peak, s[i / 16][i % 16]);
        peak = fmaxf(kq::lanes_max<32>(peak) * q.unscale, kLowest) - Type<BF>::LIFT;
        if (__any(peak > top + kSlack)) {
            const float next = fmaxf(top, peak);
            const float f = __builtin_amdgcn_exp2f(top - next);
            top = next;
            total *= f;
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) o[b] *= f;
        }
        float sum = 0.0f;
#pragma unroll
        for (uint32_t c = 0; c < 4u; ++c) { /* 16 keys */
            float w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                w[i] = __builtin_amdgcn_exp2f(fmaf(s[c / 2u][8u * (c % 2u) + i], q.unscale, -top));
                sum += w[i];
            }
            e8<BF> pw[TERMS];
            split<BF>(w, pw);
#pragma unroll
            for (uint32_t b = 0; b < BLOCKS; ++b) {
                const uint32_t r = 16u * c + 4u * half + (n % 16u) / 4u;
                const uint32_t a = vb + r * (2u * D) +
                                   v_piece<D>(r, 4u * b + 2u * (n / 16u) + (n % 4u) / 2u) * 16u +
                                   (n & 1u) * 8u;
                const e8<BF> v = join8<BF>(transposed(a), transposed(a + 16u * D));
#pragma unroll
                for (int m = 0; m < TERMS; ++m) o[b] = mma(v, pw[m], o[b]);
            }
        }
        total += sum;
    };

    load(p.t0, 0u);
    for (uint32_t t = p.t0; t < p.t1; ++t) {
        const uint32_t buf = (t - p.t0) & 1u;
        wait_vm<0>();
        __syncthreads(); /* the tile is there; the other buffer is read */
        if (t + 1u < p.t1) load(t + 1u, buf ^ 1u);
        if (awake && t * kTile < see1 && t * kTile + kTile > see0) compute(t, buf);
    }
    if (!some) return;
    total = kq::lanes_sum<32>(total);
    float *slot = p.parts > 1u ? slot_at(g, p.slot + p.part * p.step) : nullptr;
#pragma unroll
    for (uint32_t b = 0; b < BLOCKS; ++b)
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            const f4 v = f4{o[b][4 * i], o[b][4 * i + 1], o[b][4 * i + 2], o[b][4 * i + 3]};
            const uint32_t d = 32u * b + 8u * i + 4u * half;
            if (slot != nullptr)
                keep(g, slot, r0 + n, d, D, v, top, total);
            else
                put(g, p.seq, p.head, row, d, D, v, top, total, badin, bad);
        }
}

template <bool BF, int D, bool MANY>
__global__ __launch_bounds__(kThreads, D == 256 ? 1 : 2) void attend(Args g, uint32_t *status) {
    __shared__ __attribute__((aligned(16))) char lds[lds_bytes<D>()];
    const Part p = find_part<MANY>(g, blockIdx.x, blockIdx.x == 0u, status);
    if (!p.live) return;
    bool badin = false, bad = false, badseq = false;
    if (p.block == kFew)
        few_rows<BF, D>(g, p, lds, badin, bad, badseq);
    else
        many_rows<BF, D>(g, p, lds, badin, bad, badseq);
    if (badseq) kq_flag(status, KQ_DEV_SEQUENCE);
    if (badin) kq_flag(status, KQ_DEV_INPUT);
    if (bad) kq_flag(status, KQ_DEV_NUMERIC);
}

/* The parts of items that have several, joined: the workgroup of each part
 * takes its share of the item's values over all parts. */
template <bool MANY>
__global__ __launch_bounds__(kThreads) void join_parts(Args g, uint32_t *status) {
    __shared__ f4 sums[kThreads];
    __shared__ float tops[kThreads], totals[kThreads];
    const Part p = find_part<MANY>(g, blockIdx.x, false, status);
    if (!p.live || p.parts < 2u) return;
    bool badin = false, bad = false;
    const uint32_t width = g.c.width, pieces = p.rows * (width / 4u);
    const uint32_t a = (uint32_t)((uint64_t)pieces * p.part / p.parts);
    const uint32_t b = (uint32_t)((uint64_t)pieces * (p.part + 1u) / p.parts);
    /* side by side: pieces in the threads' low bits, parts in the high ones */
    uint32_t wide = 1u;
    while (wide < b - a && wide < (uint32_t)kThreads) wide *= 2u;
    const uint32_t groups = kThreads / wide;
    const uint32_t mine = threadIdx.x % wide, group = threadIdx.x / wide;
    for (uint32_t at = a; at < b; at += wide) {
        const uint32_t i = at + mine;
        const uint32_t row = i / (width / 4u), d = i % (width / 4u) * 4u;
        f4 v = f4{0.0f, 0.0f, 0.0f, 0.0f};
        float top = kLowest, total = 0.0f;
        if (i < b)
            for (uint32_t k = group; k < p.parts; k += groups) {
                const float *slot = slot_at(g, p.slot + k * p.step);
                const float *m = slot + (size_t)g.slot_rows * width;
                const float t = m[row], l = m[g.slot_rows + row];
                const f4 x = *(const f4 *)(slot + (size_t)row * width + d);
                const float next = fmaxf(top, t);
                const float f = __builtin_amdgcn_exp2f(top - next), e = __builtin_amdgcn_exp2f(t - next);
                top = next;
                total = fmaf(total, f, l * e);
#pragma unroll
                for (int c = 0; c < 4; ++c) v[c] = fmaf(v[c], f, x[c] * e);
            }
        for (uint32_t step = groups / 2u; step != 0u; step /= 2u) {
            __syncthreads();
            sums[threadIdx.x] = v;
            tops[threadIdx.x] = top;
            totals[threadIdx.x] = total;
            __syncthreads();
            if (group < step) {
                const uint32_t o = threadIdx.x + step * wide;
                const float t = tops[o], next = fmaxf(top, t);
                const float f = __builtin_amdgcn_exp2f(top - next), e = __builtin_amdgcn_exp2f(t - next);
                top = next;
                total = fmaf(total, f, totals[o] * e);
                const f4 x = sums[o];
#pragma unroll
                for (int c = 0; c < 4; ++c) v[c] = fmaf(v[c], f, x[c] * e);
            }
        }
        if (group == 0u && i < b)
            put(g, p.seq, p.head, p.row0 + row, d, width, v, top, total, badin, bad);
    }
    if (badin) kq_flag(status, KQ_DEV_INPUT);
    if (bad) kq_flag(status, KQ_DEV_NUMERIC);
}

/* ------------------------------------------------------------------ host */

struct Sizes {
    uint64_t items, parts, slots;
    uint32_t slot_rows;
    uint64_t plan_bytes, bytes;
};

/* What a call can need, whatever the device holds */
Sizes sizes_of(const kq_launch_pattn &a, const kq_launch_paged &c, const kq_launch_seqs &q) {
    Sizes z;
    const uint64_t group = a.query_heads / c.heads, rows = q.tokens * group;
    const bool single = q.offsets == nullptr;
    z.slot_rows = (single ? group : rows) <= kFew ? kFew : kMany;
    z.items = c.heads * (single ? q.count * ((group + z.slot_rows - 1u) / z.slot_rows)
                                : rows / kMany + q.count);
    z.parts = kTarget + z.items;
    /* an item of w tiles has at most w / kLeast + 1 parts */
    const uint64_t tiles = (((uint64_t)c.table_pages << c.page_shift) + kTile - 1u) / kTile;
    const uint64_t most = z.items * (tiles / kLeast + 1u);
    z.slots = most < kSlots ? most : kSlots;
    z.plan_bytes = q.count > kByLane ? ((2u + 2u * (q.count + 1u)) * 4u + 255u) / 256u * 256u : 0u;
    z.bytes = z.plan_bytes + z.slots * z.slot_rows * (c.width + 2u) * 4u;
    return z;
}

template <bool MANY>
hipError_t launch(const Args &g, uint32_t parts, uint32_t *status, hipStream_t s) {
    if (MANY) {
        hipLaunchKernelGGL(plan_many, dim3(1), dim3(1024), 0, s, g, status);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
#define KQ_ATTEND(BF, D)                                                                    \
    hipLaunchKernelGGL(HIP_KERNEL_NAME(attend<BF, D, MANY>), dim3(parts), dim3(kThreads), 0, s, g, \
                       status)
    switch (g.c.width * 2u + (g.c.bf16 ? 1u : 0u)) {
    case 128u: KQ_ATTEND(false, 64); break;
    case 129u: KQ_ATTEND(true, 64); break;
    case 256u: KQ_ATTEND(false, 128); break;
    case 257u: KQ_ATTEND(true, 128); break;
    case 512u: KQ_ATTEND(false, 256); break;
    case 513u: KQ_ATTEND(true, 256); break;
    default: return hipErrorInvalidValue;
    }
#undef KQ_ATTEND
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(join_parts<MANY>), dim3(parts), dim3(kThreads), 0, s, g,
                       status);
    return hipGetLastError();
}

}  // namespace

extern "C" uint64_t kq_launch_pattn_scratch(const kq_launch_pattn *a, const kq_launch_paged *c,
                                            const kq_launch_seqs *q) {
    return sizes_of(*a, *c, *q).bytes;
}

extern "C" hipError_t kq_launch_pattn_run(const kq_launch_pattn *a, const kq_launch_paged *c,
                                          const kq_launch_seqs *q, void *scratch, uint32_t *status,
                                          hipStream_t s) {
    const Sizes z = sizes_of(*a, *c, *q);
    Args g;
    g.a = *a;
    g.c = *c;
    g.q = *q;
    g.group = a->query_heads / c->heads;
    g.slot_rows = z.slot_rows;
    g.slots = (uint32_t)z.slots;
    g.exponent = (double)a->scale * 1.4426950408889634;
    g.plan = (uint32_t *)scratch;
    g.partial = (float *)((char *)scratch + z.plan_bytes);
    return q->count > kByLane ? launch<true>(g, (uint32_t)z.parts, status, s)
                              : launch<false>(g, (uint32_t)z.parts, status, s);
}

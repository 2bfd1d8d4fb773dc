/*
 * kq_paged_attn.hip — softmax attention of a call's rows over a paged cache
 * on gfx950 (include/kq_hip.h, kq_hip_paged_attention_f32).
 *
 * One pass over a row's keys with the largest exponent so far, M, and the sum of
 * weights, both binary32:
 *   s_t = scale log2(e) q . k_t,  w_t = 2^(s_t - M),  l = sum w_t,
 *   y = (sum w_t v_t) / (l + 2^(sink log2(e) - M))
 * M follows a row's largest s only when that has passed it by SLACK, so that
 * the sums are rarely scaled; what they are held by cancels in the end. Partial
 * sums (of waves, of parts of a long context) are added by their M.
 *
 * Products run on the matrix cores with keys and values as they lie in the cache.
 * The queries and the weights, which are binary32, are two fp16 (three bf16)
 * numbers each, whose products add up in one accumulator: twice (three times) the
 * matrix work buys results off by 2-9 x 10^-7 of their 2-norm, as those of
 * binary32 products are, where one fp16 term would leave 2 x 10^-4. Weights too small
 * for fp16's exponents are multiplied at a scale of their own (kRest). S' = K Q'
 * and O' = V' P': a lane has one row's scores, whose weights are the next product's
 * operand as they stand (its keys in the order that the first product left them),
 * and V comes transposed out of LDS (ds_read_b64_tr_b16).
 *
 * Few rows (up to 16 for a key head: decoding) are bound by the pages' bytes: a
 * workgroup's waves take 32 keys in turn each, K straight into registers, V
 * through LDS of the wave's own, with no barrier before the end. 61 sequences of
 * 500 to 32,000 tokens, 504 MB: 94 us, 5.4 TB/s, and 6 for the join; one of
 * 130,002 tokens, 133 MB: 28 us (4 of them until the first keys are there: length,
 * page and key hang on each other) and 6.
 * Many rows (128 for a key head) are bound by the matrix cores, whose clock falls
 * to 1.9 GHz under it: 8192 rows over themselves with 16 heads of 128 take 473 -
 * 514 us on different cards, 1070 - 1163 TFLOP/s of products, where a library
 * product of 8192^3 fp16 reached 1159 on one; 3 terms and heads of 256, 2049 rows:
 * 216 - 221 us, 925 - 945 TFLOP/s.
 */
#include <math.h>

#include "kq_device.h"
#include "kq_dma.h"
#include "kq_launch.h"
#include "kq_paged.h"

namespace {

typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;
constexpr uint32_t kTile = 64;       /* keys of a tile */
constexpr uint32_t kFew = 16;        /* rows of an item whose waves share out its keys */
constexpr uint32_t kMany = 128;      /* rows of an item whose waves share out its rows */
constexpr uint32_t kMid = 64;        /* the same, where 128 would not fill the device */
/* Parts that a call's items are cut into. Of few rows 1024, three to four rounds
 * of the device's waves that follow each other: 61 sequences 102 us, with 512
 * parts 116, with 2048 111. But parts of fewer than 8 tiles are not worth a
 * second round: one sequence of 130,002 tokens takes 34 us in parts of 8 tiles
 * (512), 38 in parts of 4. Of many rows 512, whose partial results are 64 KB or
 * more each (32 KB of 64 rows): 509 rows over 65,509 keys 464 us, 2049 rows of
 * 256-wide heads 215; with 1024 parts 475 and 231, with 256 505 and 224. */
constexpr uint32_t kParts = 1024;
constexpr uint32_t kShort = 8;       /* tiles */
constexpr uint32_t kLeast = 2;       /* tiles */
constexpr uint32_t kSmall = 512;     /* tiles in all of items of many rows (rows_of_items) */
constexpr uint32_t kSmallWide = 48;
constexpr uint32_t kMiddle = 2560;
constexpr uint32_t kFill = 448;      /* parts (plan_holds) */
constexpr uint32_t kEven = 700;
/* Items of few rows are a workgroup's each, of as many waves as a CU holds, where
 * there are CUs for all of them and the table's lines are short: 6 tiles of 128,
 * 196 KB of keys and values, which those waves bring in at once. There is nothing
 * to join then. 8 sequences of 30 to 318 keys 7.0 - 9.9 us, in parts of two tiles
 * and a join 7.7 - 10.8; heads of 64 of 30 to 700 keys 5.9 - 9.8, 7.8 - 9.9. Behind
 * that a CU alone is slow, 47 GB/s: 2000 keys 23.7, 11.2. And 512 items, two to a
 * CU one after the other, 15.3, 13.9. */
constexpr uint32_t kWholeItems = 256;
constexpr uint32_t kWhole = 768; /* tiles times width */
/* Calls of many rows over short lines have items of one part too: 7 tiles of 128
 * (97 rows of 24 heads over themselves 8.1 us, 9.8 with parts and a join; 1000 rows
 * of 9 sequences 22.6, 31.3; 500 of one, 9 tiles, would take 23.4, 22.7, and in bf16
 * 30.6, 24.8), 14 of 64, of which 12 measured 19.5, 22.5. */
constexpr uint32_t kWholeMany = 896;
/* Workgroups of a launch, which has fewer than 2^32 threads, up to 512 a workgroup: 65,535
 * sequences of 256 key heads have 16.8 million */
constexpr uint32_t kLaunch = 1u << 22;
constexpr uint32_t kPlan = 5;        /* words of the plan before the sequences' */
constexpr uint32_t kSlots = (4u * kParts + 2u) / 3u;
constexpr uint32_t kByLane = 64;     /* sequences that each wave plans by itself */
constexpr float kLowest = -0x1.fffffep127f;

struct Args {
    kq_launch_pattn a;
    kq_launch_paged c;
    kq_launch_seqs q;
    uint32_t group;     /* query heads of a key head */
    uint32_t slot_rows; /* rows that a slot of the partial results holds */
    uint32_t slots;     /* partial results that there is room for */
    uint32_t parts;     /* workgroups */
    uint32_t first;     /* of this launch */
    bool whole;         /* each item is one part */
    float factor_high, factor_low; /* scale log2(e), 1 .. 2 and its exponent */
    int factor_exponent;
    struct Item *items; /* of the slots, for the join */
    float *partial;     /* slots of [slot_rows][width] sums, then tops, then totals */
    uint32_t *plan;     /* tiles a part of few rows, parts, tiles a part of many rows, slots; with
                           more sequences than kByLane their first parts, then first slots */
};

/* ---------------------------------------------------------------- the plan */

/* Tiles a part, of items of few and of more rows. */
struct Lengths {
    uint32_t few, many;
};

/* Rows of a sequence's items. 17 to 32 rows are one wave of an item of 128, two of one
 * of 64: 4 rows of each of 61 sequences of 500 to 32,000 tokens, 32 for a key head, 116 us
 * (bf16 120), 128 (139) in items of 128. 33 to 64 rows keep items of 128: 488 rows spread
 * unevenly over sequences of up to 16,000 tokens 133 us (155), 138 (157) in items of 64; where
 * all have so many items of 64 would be faster: 8 rows of each 119 (120), now 128 (157). */
__device__ __forceinline__ uint32_t block_of(const Args &g, uint32_t rows, uint32_t most) {
    if (rows <= kFew) return kFew;
    return most == kMany && rows <= kMid / 2u && g.c.width != 256u ? kMid : most;
}

/* What a sequence asks for: its items (blocks of rows, for each key head) and
 * the tiles of keys that an item reads at most. */
struct Need {
    uint32_t blocks, tiles, block;
};

__device__ __forceinline__ Need need_of(const Args &g, const kq::PagedSeq &s, uint32_t most) {
    const uint32_t rows = s.rows * g.group, block = block_of(g, rows, most);
    Need n = {0u, 0u, block};
    if (!s.live || s.rows == 0u) return n;
    n.blocks = (rows + block - 1u) / block;
    n.tiles = (s.past + s.rows + kTile - 1u) / kTile;
    if (g.a.window != 0u && g.a.causal != 0u) {
        /* keys from the first token's window to the last token of a block */
        const uint32_t span = (rows < block ? rows - 1u : block - 1u) / g.group + 1u;
        const uint64_t keys = (uint64_t)g.a.window + span;
        const uint64_t seen = (keys + kTile - 1u) / kTile + 1u;
        if (seen < n.tiles) n.tiles = (uint32_t)seen;
    }
    return n;
}

/* all its items' tiles */
__device__ __forceinline__ uint64_t cost_of(const Args &g, const Need &n) {
    return (uint64_t)n.blocks * g.c.heads * n.tiles;
}

/* the tiles of its items of many rows, as many as their rows see on the average */
__device__ __forceinline__ uint64_t seen_by_many(const Args &g, const kq::PagedSeq &s,
                                                 const Need &n) {
    if (n.block == kFew) return 0u;
    const uint32_t mean = (s.past + s.rows / 2u + kTile - 1u) / kTile;
    return (uint64_t)n.blocks * g.c.heads * (g.a.causal && mean < n.tiles ? mean : n.tiles);
}

/* Rows of the items of a call whose items of 128 rows would see so many tiles in all.
 * A workgroup of 128 rows begins with 3 us of queries (64 KB, at what a CU alone reads)
 * and takes 2 us a tile where it has its CU to itself. So small calls have items of
 * 16 rows, which read their keys eight times: 97 rows of 24 heads over themselves (48
 * tiles) 8.1 us, 19.4 in items of 128; 500 of 16 heads (256) 17.4, 22.8; but 300 over
 * 1300 keys (684) 37, 27. Those in the middle have items of 64, which begin sooner and
 * are joined from fewer parts: 300 rows over 1300 keys 24.5, 27; 1200 rows of 8
 * sequences (1364) 30, 39; but they read LDS twice as often for a product: 2003 ragged
 * rows of heads of 64 (3300) 53, 49. Where one sequence's rows stand behind many keys
 * the sides cross later than kMiddle: 500 rows of 2 key heads over 1500 keys more (1792)
 * 35, 38, over 2000 (2304) 39.5, 40.7, over 2500 (2752) 43, 44, over 5500 (5760) 63, 66
 * (bf16 73, 80). Heads of 256,
 * whose workgroups have no room beside each other, have no such form, and items of 16
 * rows up to 48 tiles (116 rows of 32 heads, 32 tiles, 13.2, 18.7; 250 of 16, 64 tiles,
 * 29.7, 27). */
__device__ __forceinline__ uint32_t rows_of_items(const Args &g, uint64_t seen) {
    if (g.c.width == 256u) return seen < kSmallWide ? kFew : kMany;
    return seen >= kMiddle ? kMany : seen < kSmall ? kFew : kMid;
}

/* Whether a plan of items of `most` rows with so many parts holds; otherwise `most`
 * becomes what is planned next. Items of 64 rows also take the place of items of 128
 * that are planned fewer parts than the 512 workgroups that have room at once (3000
 * rows over themselves, 376 parts: 83 us, 105), or fewer than 700 that are uneven, as
 * the rows see three quarters or less of the most (2500 rows, 628 parts: 66, 87; 4096,
 * 512: 148, 155, bf16 186, 208; 2048, 512: 54, 63). With even parts items of 128 are
 * faster: 300 rows over 10,300 keys 67, 88; 509 over 65,509 474, 509. A plan of smaller
 * items that has more parts than the call has workgroups falls back to larger ones. */
__device__ __forceinline__ bool plan_holds(const Args &g, uint32_t &most, bool &last,
                                           uint32_t parts, uint64_t seen, uint64_t cost) {
    if (most == kMany) {
        const bool uneven = parts < kEven && seen * 4u <= cost * 3u;
        if (last || g.c.width == 256u || !(parts < kFill || uneven)) return true;
        most = kMid;
    } else {
        if (parts <= g.parts) return true;
        most = g.c.width == 256u || most == kMid ? kMany : kMid;
    }
    last = true;
    return false;
}

__device__ __forceinline__ Lengths part_tiles(const Args &g, uint64_t cost) {
    if (g.whole) return Lengths{1u << 24, 1u << 24};
    const uint32_t fine = (uint32_t)((cost + kParts - 1u) / kParts);
    const uint32_t coarse = (uint32_t)((cost + kParts / 2u - 1u) / (kParts / 2u));
    Lengths l;
    l.few = coarse < kShort ? coarse : fine > kShort ? fine : kShort;
    l.few = l.few < kLeast ? kLeast : l.few;
    l.many = coarse < kLeast ? kLeast : coarse;
    return l;
}

__device__ __forceinline__ uint32_t length_of(const Lengths &l, const Need &n) {
    return n.block == kFew ? l.few : l.many;
}

/* parts of so many tiles, the nearest number: an item a little longer than a part
 * stays whole, up to 1.5 times `length`; several parts have 0.75 to 1.25 times
 * `length` on the average, to whole tiles (3 tiles by 2: one of 2, one of 1). */
__device__ __forceinline__ uint32_t parts_of(uint32_t tiles, uint32_t length) {
    if (tiles == 0u) return 0u;
    const uint32_t n = (tiles + length / 2u) / length;
    return n == 0u ? 1u : n;
}

/* One part of the work */
struct Part {
    kq::PagedSeq seq;
    uint32_t row0, rows;  /* of the sequence's rows x group */
    uint32_t block;       /* kFew, kMid or kMany */
    uint32_t head;
    uint32_t part, parts; /* this one, and how many the item really has */
    uint32_t t0, t1;      /* its tiles */
    uint32_t key0, key1;  /* keys that any of the item's rows sees */
    uint32_t slot, step;  /* of the item's first part, and between two parts */
    bool slotted;         /* whether the sequence's parts have slots */
    bool live;

    /* what all lanes hold alike goes into scalar registers, as the descriptors
     * of the loads into LDS need it */
    __device__ __forceinline__ void pin() {
        uint32_t *const all[] = {&seq.begin, &seq.rows, &seq.past, &seq.slot, &row0, &rows, &block,
                                 &head, &part, &parts, &t0, &t1, &key0, &key1, &slot, &step};
#pragma unroll
        for (uint32_t *x : all) *x = __builtin_amdgcn_readfirstlane(*x);
    }
};

/* What the join has to know of a part that has a slot: its item's rows, and
 * where its item's partial results lie. The part's workgroup leaves it, by slot;
 * plan[3] says how many slots there are. */
struct __attribute__((aligned(16))) Item {
    uint32_t begin, row0, rows, head_kind; /* rows 0: nothing to join; kind: the upper half */
    uint32_t part, parts, slot, step;
};

__device__ __forceinline__ void leave(const Args &g, const Part &p) {
    if (threadIdx.x != 0u || !p.slotted) return;
    const uint32_t at = p.slot + p.part * p.step;
    if (at < g.slots) {
        const uint32_t kind = p.block == kFew ? 1u : p.block == kMid || g.c.width == 256u ? 2u : 0u;
        Item t = {p.seq.begin, p.row0, p.rows, p.head | kind << 16,
                  p.part, p.parts, p.slot, p.step};
        if (!p.live || p.parts == 1u) t.rows = 0u;
        g.items[at] = t;
    }
}

__device__ __forceinline__ void part_of(Part &p, const Args &g, const kq::PagedSeq &s,
                                        const Need &n, uint32_t length, uint32_t u,
                                        uint32_t first_slot) {
    p.seq = s;
    p.block = n.block;
    /* Workgroups go to the XCDs in turn, so neighbours in number should have
     * work alike: heads, then blocks, whose last rows see the most keys and go
     * first, then parts, of which an item may have fewer than its sequence. (With
     * the parts before the blocks 2049 rows of 4 heads of 256 took 323 us in place
     * of 224: one half of the XCDs had the second parts, most of them none.) */
    const uint32_t items = n.blocks * g.c.heads, all = s.rows * g.group;
    uint32_t item = u % items, ta = 0u, tb = s.rows - 1u;
    p.part = u / items;
    p.head = item;
    p.row0 = 0u;
    p.rows = all;
    if (n.blocks != 1u) {
        p.head = item % g.c.heads;
        p.row0 = (n.blocks - 1u - item / g.c.heads) * p.block;
        p.rows = all - p.row0 < p.block ? all - p.row0 : p.block;
        ta = p.row0 / g.group;
        tb = (p.row0 + p.rows - 1u) / g.group;
    }
    p.key1 = g.a.causal ? s.past + tb + 1u : s.past + s.rows;
    p.key0 = 0u;
    if (g.a.window != 0u && s.past + ta + 1u > g.a.window) p.key0 = s.past + ta + 1u - g.a.window;
    const uint32_t a = p.key0 / kTile, tiles = (p.key1 + kTile - 1u) / kTile - a;
    p.parts = parts_of(tiles, length);
    const uint32_t each = tiles / p.parts, more = tiles % p.parts;
    p.t0 = a + p.part * each + (p.part < more ? p.part : more);
    p.t1 = p.t0 + each + (p.part < more ? 1u : 0u);
    p.slot = first_slot + item;
    p.step = items;
    p.slotted = parts_of(n.tiles, length) > 1u;
    p.live = p.part < p.parts &&
             (p.parts == 1u || p.slot + (p.parts - 1u) * p.step < g.slots);
}

/* x of the lane that CTRL (a DPP control) names, 0 where there is none or ROWS
 * leaves the row of 16 lanes out */
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t lane_from(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t lane_add(uint32_t x) {
    return x + lane_from<CTRL, ROWS>(x);
}
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t lane_add(uint64_t x) {
    return x + ((uint64_t)lane_from<CTRL, ROWS>((uint32_t)(x >> 32)) << 32 |
                lane_from<CTRL, ROWS>((uint32_t)x));
}
/* v of the lanes up to and with this one: within rows of 16, then row 0's end to
 * row 1 and 2's to 3, then the lower half's end to the upper half */
template <typename T>
__device__ __forceinline__ T lanes_through(T v) {
    v = lane_add<0x111, 0xf>(v);
    v = lane_add<0x112, 0xf>(v);
    v = lane_add<0x114, 0xf>(v);
    v = lane_add<0x118, 0xf>(v);
    v = lane_add<0x142, 0xa>(v);
    return lane_add<0x143, 0xc>(v);
}
__device__ __forceinline__ uint32_t lanes_before(uint32_t v) { return lanes_through(v) - v; }
/* v of all lanes */
__device__ __forceinline__ uint64_t lanes_add(uint64_t v) {
    v = lanes_through(v);
    return (uint64_t)__builtin_amdgcn_readlane((uint32_t)(v >> 32), 63) << 32 |
           __builtin_amdgcn_readlane((uint32_t)v, 63);
}

/* Part `index` of the call, the same in all lanes. Up to kByLane sequences:
 * a lane looks at each, and every wave adds up for itself. More: plan_many
 * has done so. Offsets, slots and lengths that break the rules leave no part at
 * all: where they hold, the rows of all sequences are at most the call's tokens,
 * which the host's sizes go by. */
template <bool MANY>
__device__ __forceinline__ Part find_part(const Args &g, uint32_t index, uint32_t *status) {
    Part p;
    p.live = p.slotted = false;
    bool bad = false;
    if constexpr (!MANY) {
        const uint32_t lane = threadIdx.x & 63u;
        kq::PagedSeq s = {0u, 0u, 0u, 0u, false};
        if (lane < g.q.count) s = kq::paged_seq(g.q, g.c, lane, bad);
        if (__any(bad)) { /* refused: nothing runs, and there is nothing to join */
            if (index == 0u) {
                if (bad) kq_flag(status, KQ_DEV_SEQUENCE);
                g.plan[3] = 0u;
            }
            return p;
        }
        uint32_t most = kFew;
        uint64_t seen = 0u;
        if (g.slot_rows == kMany) {
            seen = lanes_add(seen_by_many(g, s, need_of(g, s, kMany)));
            most = rows_of_items(g, seen);
        }
        Need n;
        Lengths length;
        uint32_t each, mine, through, total;
        bool last = false;
        for (;;) {
            n = need_of(g, s, most);
            const uint64_t cost = lanes_add(cost_of(g, n));
            length = part_tiles(g, cost);
            each = parts_of(n.tiles, length_of(length, n));
            mine = n.blocks * g.c.heads * each;
            through = lanes_through(mine);
            total = __builtin_amdgcn_readlane(through, 63);
            if (plan_holds(g, most, last, total, seen, cost)) break;
        }
        const uint32_t first = through - mine;
        const uint32_t held = each > 1u ? mine : 0u, slots = lanes_through(held);
        const uint32_t first_slot = slots - held;
        if (index == 0u && lane == 63u) g.plan[3] = slots; /* for the join */
        const uint64_t m = __ballot(index >= first && index - first < mine);
        if (m == 0ull) return p;
        const int at = __builtin_amdgcn_readfirstlane((int)__builtin_ctzll(m));
        kq::PagedSeq w;
        w.begin = __builtin_amdgcn_readlane(s.begin, at);
        w.rows = __builtin_amdgcn_readlane(s.rows, at);
        w.past = __builtin_amdgcn_readlane(s.past, at);
        w.slot = __builtin_amdgcn_readlane(s.slot, at);
        w.live = true;
        const Need need = need_of(g, w, most);
        part_of(p, g, w, need, length_of(length, need),
                index - __builtin_amdgcn_readlane(first, at),
                __builtin_amdgcn_readlane(first_slot, at));
        return p;
    } else {
        if (index >= g.plan[1]) return p;
        const uint32_t *first = g.plan + kPlan, *slots = first + g.q.count + 1u;
        const uint32_t s = kq::wave_find(first, g.q.count, index);
        const kq::PagedSeq w = kq::paged_seq(g.q, g.c, s, bad);
        const Lengths length = {g.plan[0], g.plan[2]};
        const Need need = need_of(g, w, g.plan[4]);
        part_of(p, g, w, need, length_of(length, need), index - first[s], slots[s]);
        return p;
    }
}

/* One workgroup: the plan of more sequences than a wave has lanes */
__global__ __launch_bounds__(1024) void plan_many(Args g, uint32_t *status) {
    __shared__ uint64_t sums[16];
    __shared__ uint32_t parts[16], slots[16];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x / 64u;
    bool bad = false;
    /* a value of every sequence, added up */
    auto sum = [&](auto of) {
        uint64_t v = 0u;
        for (uint32_t s = threadIdx.x; s < g.q.count; s += 1024u)
            v += of(kq::paged_seq(g.q, g.c, s, bad));
        v = lanes_add(v);
        if (lane == 0u) sums[wave] = v;
        __syncthreads();
        v = 0u;
        for (int w = 0; w < 16; ++w) v += sums[w];
        __syncthreads();
        return v;
    };
    const uint64_t seen = sum([&](const kq::PagedSeq &s) {
        return seen_by_many(g, s, need_of(g, s, kMany));
    });
    uint32_t most = g.slot_rows == kFew ? kFew : rows_of_items(g, seen);
    bool last = false;
    if (bad) kq_flag(status, KQ_DEV_SEQUENCE);
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0u) g.plan[1] = g.plan[3] = 0u;
        return;
    }
    uint32_t *first = g.plan + kPlan, *slot = first + g.q.count + 1u;
    for (;;) {
        const uint64_t cost =
            sum([&](const kq::PagedSeq &s) { return cost_of(g, need_of(g, s, most)); });
        const Lengths length = part_tiles(g, cost);
        uint32_t parts_before = 0u, slots_before = 0u;
        for (uint32_t base = 0u; base < g.q.count; base += 1024u) {
            const uint32_t s = base + threadIdx.x;
            uint32_t mine = 0u, held = 0u;
            if (s < g.q.count) {
                const Need n = need_of(g, kq::paged_seq(g.q, g.c, s, bad), most);
                const uint32_t each = parts_of(n.tiles, length_of(length, n));
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
        if (!plan_holds(g, most, last, parts_before, seen, cost)) continue;
        if (threadIdx.x == 0u) {
            g.plan[0] = length.few;
            g.plan[1] = parts_before;
            g.plan[2] = length.many;
            g.plan[3] = slots_before;
            g.plan[4] = most;
        }
        return;
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
    /* fp16's own range is short: a row's largest query is brought to 2^12 .. 2^14, and
     * the largest of its weights so far to 2^13, 2^15 with what its exponent may pass its
     * stand-in by, the slack */
    static constexpr int TOP = 12;
    static constexpr float LIFT = 13.0f, SLACK = 2.0f;
};
template <>
struct Type<true> {
    typedef __bf16 e;
    static constexpr int TERMS = 3;
    static constexpr int TOP = 0;
    static constexpr float LIFT = 0.0f, SLACK = 8.0f;
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

/* x[0..7] as TERMS operands whose sum it is: pairs at a time, which one
 * instruction rounds and packs */
template <bool BF>
__device__ __forceinline__ void split(const float (&x)[8], e8<BF> (&t)[Type<BF>::TERMS]) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    e2<BF> p[Type<BF>::TERMS][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        f2 v = f2{x[2 * i], x[2 * i + 1]};
#pragma unroll
        for (int k = 0; k < Type<BF>::TERMS; ++k) {
            p[k][i] = __builtin_convertvector(v, e2<BF>);
            if constexpr (BF) {
                const uint32_t u = __builtin_bit_cast(uint32_t, p[k][i]);
                v -= f2{__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u)};
            } else {
                /* x less its rounded value, without converting that back */
                const uint32_t u = __builtin_bit_cast(uint32_t, p[k][i]);
                if (k + 1 < Type<BF>::TERMS) {
                    f2 r;
                    asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel_hi:[1,0,0]"
                        : "=v"(r.x) : "v"(u), "v"(v.x));
                    asm("v_fma_mix_f32 %0, -%1, 1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]"
                        : "=v"(r.y) : "v"(u), "v"(v.y));
                    v = r;
                }
            }
        }
    }
#pragma unroll
    for (int k = 0; k < Type<BF>::TERMS; ++k) t[k] = __builtin_bit_cast(e8<BF>, p[k]);
}

/* fp16 ends at 2^-24, so that two terms hold 22 bits of a weight of 2^-2 or more: 2^-15
 * of a row's largest, 10 nats. Behind a key that leads by more, smaller ones can be the
 * whole sum (its own value may be next to nothing). Where a wave has any, what their two
 * terms leave, at most 2^-25, is multiplied as well, times 2^40 and with the sums times
 * 2^40 for as long: powers of two, which change no bit, and the sums of 2^24 keys, below
 * 2^55, have room. That holds 22 bits down to 2^-55 of the largest, 38 nats. bf16 has
 * binary32's exponents and needs none of it. 61 sequences decoding take 107 us where
 * all waves have such weights, 104 where none has. */
constexpr float kHeld = 0x1p-2f, kHeldLog2 = -2.0f;
constexpr float kRest = 0x1p40f;
/* Of many rows it is left out where it could not be told from the sums' own roundings:
 * of a tile's 64 keys it is at most 2^-25 8 times the 2-norm of all their values, by
 * Cauchy and Schwarz, and where the square of a row's sums is 2^4 times that of the values,
 * below 2^-24 of the sums, to which the tile is added in eight or more roundings. So
 * scores that are merely wide cost a look at the values: 8192 rows with scores 4 nats
 * wide 582 us, with all rests 865, without small weights 478. Squares below fp16's normal
 * numbers may be taken for 0: kNoSquare stands for more of them than a lane has. */
constexpr float kRestMatters = 0x1p4f;
constexpr float kNoSquare = 0x1p-20f;

__device__ __forceinline__ void rest_of(float (&w)[8]) {
    e8<false> t[2];
    split<false>(w, t);
#pragma unroll
    for (int i = 0; i < 8; ++i)
        w[i] = w[i] < kHeld ? (w[i] - (float)t[0][i] - (float)t[1][i]) * kRest : 0.0f;
}

/* sums and the squares of fp16 values */
__device__ __forceinline__ f4 squares(f4 sums, u4 v) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const h2 x = __builtin_bit_cast(h2, (uint32_t)v[i]);
        sums[i] = __builtin_amdgcn_fdot2(x, x, sums[i], false);
    }
    return sums;
}

/* x as a value that is not known: what comes of it is formed again, not held */
template <typename T>
__device__ __forceinline__ T again(T x) {
    asm volatile("" : "+v"(x));
    return x;
}
/* the lane's number, likewise */
__device__ __forceinline__ uint32_t lane_again() {
    const uint32_t all = again(~0u);
    return __builtin_amdgcn_mbcnt_hi(all, __builtin_amdgcn_mbcnt_lo(all, 0u));
}

/* A row's queries, as operands: the exponent's factor put in to 48 bits, and
 * the row's largest value brought to 2^TOP .. 2^(TOP + 2) by a power of two. */
template <bool BF, int STEPS>
struct Query {
    e8<BF> x[STEPS][Type<BF>::TERMS];
    float unscale;
};

template <int STEPS>
struct Raw {
    float4 v[STEPS][2];
};

/* at(step): 8 values of the row from there on */
template <int STEPS, typename At>
__device__ __forceinline__ void fetch_query(Raw<STEPS> &r, bool some, At at) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int i = 0; i < 2; ++i)
            r.v[s][i] =
                some ? *(const float4 *)(at(s) + 4 * i) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
}

/* LANES: the lanes that share a row */
template <bool BF, int STEPS, int LANES>
__device__ __forceinline__ void split_query(const Args &g, const Raw<STEPS> &r, Query<BF, STEPS> &q,
                                            bool &badin) {
    constexpr int TOP = Type<BF>::TOP;
    uint32_t most = 0u; /* of the values' bits without the sign: orders them, and finds a NaN */
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const uint32_t b = __float_as_uint((&r.v[s][i].x)[c]) & 0x7fffffffu;
                most = b > most ? b : most;
            }
    badin |= __any(most >= 0x7f800000u);
    const float top = kq::lanes_max<LANES>(__uint_as_float(most < 0x7f800000u ? most : 0u));
    /* the largest value's exponent, 0 for a row of zeros */
    int e = (int)(__float_as_uint(top) >> 23) - 127;
    e = top == 0.0f ? 0 : e < -114 ? -114 : e; /* the factor's scale stays finite */
    /* the factor as two numbers: its own rounding would be the same for all keys */
    const float high = __builtin_ldexpf(g.factor_high, TOP - e);
    const float low = __builtin_ldexpf(g.factor_low, TOP - e);
    /* at least 2^-126, where scores are 0 to any precision: a masked -inf times 0 is none */
    const int back = e + g.factor_exponent - TOP;
    q.unscale = __builtin_ldexpf(1.0f, back < -126 ? -126 : back);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = (&r.v[s][i / 4].x)[i % 4];
            x[i] = fmaf(v, high, v * low);
        }
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

/* What a row's sums are divided by, all keys in and the sink, whose exponent has
 * its factor in 48 bits as the queries have */
__device__ __forceinline__ float inverse_of_row(const Args &g, uint32_t h, float top, float total,
                                                bool &bad) {
    if (g.a.sinks != nullptr) {
        const float sink = g.a.sinks[h];
        const float e = fmaf(sink, 0x1.715476p+0f, fmaf(sink, 0x1.4ae0cp-26f, -top));
        if (e > 64.0f) { /* by the sink's weight, in halves: it may be beyond the range */
            const float half = __builtin_amdgcn_exp2f(-0.5f * e);
            return half * (half / fmaf(total * half, half, 1.0f));
        }
        total += __builtin_amdgcn_exp2f(e);
    }
    bad |= !(total > 0.0f); /* of a row's keys one at least has a weight of its slack */
    return 1.0f / total;
}

/* Four values of a row, at d of head h: its gate, and where they go */
__device__ __forceinline__ void put(const Args &g, uint32_t token, uint32_t h, uint32_t d, f4 o,
                                    float inverse, bool &badin, bool &bad) {
    const size_t at = (size_t)h * g.c.width + d;
    o *= inverse;
    if (g.a.gated) {
        const f4 e = *(const f4 *)(g.a.gate + (size_t)token * g.a.gs + at);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            badin |= !kq_isfinite(e[i]);
            o[i] *= kq::sigmoid(e[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) bad |= !kq_isfinite(o[i]);
    *(f4 *)(g.a.y + (size_t)token * g.a.ys + at) = o;
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

/* Pages of KEYS keys from key `at` on (16 or 8, a multiple of that), by scalar
 * loads: the vector loads under way are not waited for. `some`: whether any of the keys is
 * asked for; otherwise, and for a page that is none, the descriptor that comes
 * of it lets nothing be read. */
template <uint32_t KEYS>
__device__ __forceinline__ uint32_t page_at(const Args &g, const Part &p, uint32_t at) {
    typedef const __attribute__((address_space(4))) uint32_t *scalar_ptr;
    const bool some = at < p.key1 && at + KEYS > p.key0;
    return some ? ((scalar_ptr)g.c.table)[(size_t)p.seq.slot * g.c.table_pages +
                                          (at >> g.c.page_shift)]
                : ~0u;
}

struct Place {
    const char *kp, *vp;
    uint32_t bytes, off;
};

template <int D, uint32_t KEYS>
__device__ __forceinline__ Place place_of(const Args &g, const Part &p, uint32_t at, uint32_t page,
                                          bool &bad) {
    Place r;
    const uint32_t bytes = (D * 2u) << g.c.page_shift;
    const bool there = page < g.c.page_count;
    bad |= !there && at < p.key1 && at + KEYS > p.key0;
    const uint64_t off = ((uint64_t)(there ? page : 0u) * g.c.heads + p.head) * bytes;
    r.kp = (const char *)g.c.keys + off;
    r.vp = (const char *)g.c.values + off;
    r.bytes = there ? bytes : 0u;
    r.off = (at & ((1u << g.c.page_shift) - 1u)) * (D * 2u);
    return r;
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const char *p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, bytes, 0x00020000);
}

constexpr uint32_t kOut = 0x80000000u; /* an offset that no page has, nor what is added to it */

/* ------------------------------------------------- few rows: keys shared out */

/* where the 16-byte piece c of V's row r lies: a transposing read takes the
 * same 32 bytes of 16 rows, which 64 banks hold 8 of at a time */
template <int D>
__device__ __forceinline__ uint32_t few_piece(uint32_t r, uint32_t c) {
    return D == 64 ? c ^ (2u * ((r >> 1) & 3u)) : c ^ (2u * (r & 7u));
}

/* 32 rows of V a wave, or what the waves hand each other: sums of 16 rows, tops, totals */
template <int D, int W>
constexpr uint32_t few_bytes() {
    return W * (16u * (D + 4u) * 4u + 128u);
}
template <int D>
constexpr uint32_t many_bytes() {
    return 512u * D; /* 2 x 64 rows of K and V */
}
/* Waves a SIMD that registers are given for. Heads of 128 in fp16 need 150: three
 * (61 sequences 109 us; four, at 128 with 24 of them in memory, 136). */
template <int D>
constexpr int few_side() {
    return D == 256 ? 2 : D == 128 ? 3 : 4;
}

/* Up to 16 rows: a wave takes every W-th 32 keys, S' = K Q' and O' = V' P' of
 * 16 x 16 x 32 products, and the waves' results are joined in LDS. One set of
 * registers and one buffer a wave: three workgroups a CU hide the loads better
 * than a second set would (two workgroups then: 115 us for the 61 sequences). */
template <bool BF, int D, int W>
__device__ __forceinline__ void few_rows(const Args &g, const Part &p, char *lds, bool &badin,
                                         bool &bad, bool &badseq) {
    constexpr int STEPS = D / 32, BLOCKS = D / 16, TERMS = Type<BF>::TERMS;
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u);
    const uint32_t n = lane & 15u, quarter = lane >> 4;
    const bool some = n < p.rows;
    const uint32_t row = p.row0 + n, token = some ? row / g.group : 0u;
    const uint32_t h = p.head * g.group + (some ? row % g.group : 0u);
    const uint32_t last = g.a.causal ? p.seq.past + token + 1u : p.seq.past + p.seq.rows;
    const uint32_t from = g.a.window != 0u && p.seq.past + token + 1u > g.a.window
                              ? p.seq.past + token + 1u - g.a.window : 0u;

    Query<BF, STEPS> q;
    const float *qp = g.a.q + (size_t)(p.seq.begin + token) * g.a.qs + (size_t)h * D + 8u * quarter;

    f4 o[BLOCKS];
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b) o[b] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    float top = kLowest, total = 0.0f;

    char *const mine = lds + wave * (64u * D); /* 32 rows of V */
    const uint32_t mine_at = lds_addr(mine);
    uint32_t key = p.t0 * kTile + wave * 32u;
    const uint32_t end = p.t1 * kTile < p.key1 ? p.t1 * kTile : p.key1;
    const bool any = key < end;
    e8<BF> k[2][STEPS];
    uint32_t page[2];
    Place place[2];

    auto pages = [&](uint32_t at) {
#pragma unroll
        for (uint32_t b = 0; b < 2u; ++b) page[b] = page_at<16u>(g, p, at + 16u * b);
    };
    auto places = [&](uint32_t at) {
#pragma unroll
        for (uint32_t b = 0; b < 2u; ++b)
            place[b] = place_of<D, 16u>(g, p, at + 16u * b, page[b], badseq);
    };
    auto load_k = [&](uint32_t at) {
#pragma unroll
        for (uint32_t b = 0; b < 2u; ++b) {
            const uint32_t r = at + 16u * b + n;
            const uint32_t off = r < p.key1 && r >= p.key0
                                     ? place[b].off + n * (2u * D) + 16u * quarter : kOut;
            const auto keys = buffer_of(place[b].kp, place[b].bytes);
#pragma unroll
            for (uint32_t s = 0; s < STEPS; ++s)
                k[b][s] = __builtin_bit_cast(
                    e8<BF>, __builtin_amdgcn_raw_buffer_load_b128(keys, off + 64u * s, 0, 0));
        }
    };
    auto load_v = [&](uint32_t at) {
#pragma unroll
        for (uint32_t b = 0; b < 2u; ++b) {
            const auto values = buffer_of(place[b].vp, place[b].bytes);
#pragma unroll
            for (uint32_t j = 0; j < D / 32u; ++j) { /* pieces of 1 KiB */
                const uint32_t o16 = j * 64u + lane, r = o16 / (D / 8u), c = o16 % (D / 8u);
                const uint32_t key = at + 16u * b + r;
                const uint32_t off = key < p.key1 && key >= p.key0
                                         ? place[b].off + r * (2u * D) + few_piece<D>(r, c) * 16u
                                         : kOut;
                __builtin_amdgcn_raw_ptr_buffer_load_lds(
                    values,
                    (__attribute__((address_space(3))) void *)(mine + b * (32u * D) + j * 1024u),
                    16, off, 0, 0, 0);
            }
        }
    };
    auto scores = [&](f4 (&s)[2]) {
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            s[b] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int t = 0; t < STEPS; ++t)
#pragma unroll
                for (int m = 0; m < TERMS; ++m) s[b] = mma(k[b][t], q.x[t][m], s[b]);
        }
    };
    /* whether any is too small for its terms */
    auto weights = [&](uint32_t at, const f4 (&s)[2], float (&w)[8]) {
        float peak = kLowest;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t key = at + 16u * (i / 4) + 4u * quarter + i % 4;
            w[i] = key < last && key >= from ? s[i / 4][i % 4] * q.unscale : -INFINITY;
            peak = fmaxf(peak, w[i]);
        }
        peak = kq::lanes_max<48>(peak) - Type<BF>::LIFT;
        if (__any(peak > top + Type<BF>::SLACK)) {
            const float next = fmaxf(top, peak);
            const float f = __builtin_amdgcn_exp2f(top - next);
            top = next;
            total *= f;
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) o[b] *= f;
        }
        float sum = 0.0f;
        bool small = false;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            w[i] = __builtin_amdgcn_exp2f(w[i] - top);
            sum += w[i];
            small |= !BF && w[i] > 0.0f && w[i] < kHeld;
        }
        total += sum;
        return !BF && __any(small);
    };
    auto gather = [&](const e8<BF> (&pw)[TERMS], uint32_t lane) {
        const uint32_t n = lane & 15u, r = lane / 4u; /* 4 a quarter, and n / 4 */
#pragma unroll
        for (uint32_t b = 0; b < BLOCKS; ++b) {
            const uint32_t a = mine_at + r * (2u * D) +
                               few_piece<D>(r, 2u * b + (n % 4u) / 2u) * 16u + (n & 1u) * 8u;
            const e8<BF> v = join8<BF>(transposed(a), transposed(a + 32u * D));
#pragma unroll
            for (int m = 0; m < TERMS; ++m) o[b] = mma(v, pw[m], o[b]);
        }
    };

    /* the first keys are under way while the queries are split, if registers hold both */
    constexpr bool AHEAD = !(BF && D == 256);
    auto begin = [&]() {
        if (!any) return;
        places(key);
        load_k(key);
        load_v(key);
        if (key + 32u * W < end) pages(key + 32u * W);
    };
    if (any) pages(key);
    Raw<STEPS> raw;
    fetch_query(raw, some, [&](int s) { return qp + 32 * s; });
    if (AHEAD) begin();
    split_query<BF, STEPS, 48>(g, raw, q, badin);
    if (!AHEAD) begin();
    /* K of the next keys is asked for when this one's is used, V likewise: while
     * one waits the CU's other workgroups read */
    while (key < end) {
        const uint32_t next = key + 32u * W;
        f4 s[2];
        float w[8];
        e8<BF> pw[TERMS];
        scores(s);
        if (next < end) {
            places(next);
            load_k(next);
            if (next + 32u * W < end) pages(next + 32u * W);
        }
        const bool small = weights(key, s, w);
        /* V is there: loads return in order, and only the next K's come behind it */
        auto wait = [&]() {
            if (next < end)
                wait_vm<2 * STEPS>();
            else
                wait_vm<0>();
        };
        if constexpr (!BF)
            if (small) {
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = again(w[i]);
                rest_of(x);
                split<BF>(x, pw);
                wait();
#pragma unroll
                for (int b = 0; b < BLOCKS; ++b) o[b] *= kRest;
                gather(pw, lane_again());
#pragma unroll
                for (int b = 0; b < BLOCKS; ++b) o[b] *= 1.0f / kRest;
            }
        split<BF>(w, pw);
        wait();
        gather(pw, lane);
        if (next < end) {
            wait_lgkm0(); /* V is read */
            load_v(next);
        }
        key = next;
    }
    total = kq::lanes_sum<48>(total);

    /* the waves' tops, totals and sums [wave][row][d], then 16 rows by all */
    float *tops = (float *)lds, *totals = tops + W * 16, *sums = totals + W * 16;
    constexpr uint32_t kRow = D + 4u; /* rows 16 bytes apart in the banks */
    __syncthreads();
    const uint32_t l = lane_again(), at = wave * 16u + l % 16u;
    if (l < 16u) {
        tops[at] = top;
        totals[at] = total;
    }
#pragma unroll
    for (uint32_t b = 0; b < BLOCKS; ++b)
        *(f4 *)(sums + at * kRow + 16u * b + 4u * (l / 16u)) = o[b];
    __syncthreads();
    float *slot = p.parts > 1u ? slot_at(g, p.slot + p.part * p.step) : nullptr;
    const uint32_t group = again(g.group); /* its reciprocal is not held either */
    for (uint32_t i = 64u * wave + l; i < p.rows * (D / 4u); i += 64u * W) {
        const uint32_t r = i / (D / 4u), d = i % (D / 4u) * 4u;
        float t = tops[r];
#pragma unroll
        for (int w = 1; w < W; ++w) t = fmaxf(t, tops[w * 16 + r]);
        f4 v = f4{0.0f, 0.0f, 0.0f, 0.0f};
        float l = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const float f = __builtin_amdgcn_exp2f(tops[w * 16 + r] - t);
            l = fmaf(totals[w * 16 + r], f, l);
            const f4 x = *(const f4 *)(sums + (w * 16u + r) * kRow + d);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = fmaf(x[e], f, v[e]);
        }
        if (slot != nullptr)
            keep(g, slot, r, d, D, v, t, l);
        else {
            const uint32_t row = p.row0 + r, h = p.head * g.group + row % group;
            put(g, p.seq.begin + row / group, h, d, v, inverse_of_row(g, h, t, l, bad), badin, bad);
        }
    }
}

/* ------------------------------------------------ many rows: rows shared out */

/* Up to 128 rows: M of them a wave, whose K and V come into LDS once for all,
 * two buffers of 64 keys. S' = K Q' and O' = V' P' of products of M x M: 32 (4
 * waves) moves half the bytes out of LDS that 16 (8 waves) does, and 16 holds a
 * head of 256 in the registers of two waves a SIMD, one of which multiplies
 * while the other forms exponentials (2049 rows of bf16 heads: 282 us, with 32
 * and one wave 429). Heads of 64 leave room for three (19 ragged sequences 47,
 * with two 54). MID: up to 64 rows, four waves of 16. */
template <int D, bool MID = false>
struct Many {
    static constexpr int M = MID || D == 256 ? 16 : 32;
    static constexpr int W = (MID ? kMid : kMany) / M, THREADS = 64 * W;
    static constexpr int KEYS = 64 / W;         /* that a wave brings in */
    static constexpr int REGS = M * M / 64;     /* values of a block that a lane holds */
    static constexpr int STEPS = D * M / 512;   /* products along a head */
    static constexpr int BLOCKS = D / M;        /* of O */
    static constexpr uint32_t ROW = 2 * D;      /* bytes */
    static constexpr uint32_t LDS = 4u * kTile * ROW;
    typedef float acc __attribute__((ext_vector_type(REGS)));

    /* 16-byte pieces of a row's bytes are held at piece c ^ these: K's are read
     * down 16 rows, V's 64 (32) bytes of 8 (16) rows at a time, transposed */
    static __device__ __forceinline__ uint32_t k_swap(uint32_t r) {
        return D == 64 ? (r >> 1) & 7u : r & 15u;
    }
    static __device__ __forceinline__ uint32_t v_swap(uint32_t r) {
        if (M == 16) return few_piece<D>(r, 0u);
        return D == 64 ? ((r >> 1) & 1u) << 2 : (r & 3u) << 2;
    }
    /* where a lane's piece `at` (of four values) of a partial result's rows lies */
    static __device__ __forceinline__ uint32_t column(uint32_t piece, uint32_t lane) {
        return M == 16 ? 16u * piece + 4u * (lane / 16u)
                       : 32u * (piece / 4u) + 8u * (piece % 4u) + 4u * (lane / 32u);
    }
};

template <uint32_t I>
struct Buffer {
    static constexpr uint32_t value = I;
};

template <bool BF, int D, bool MID>
__device__ __forceinline__ void many_rows(const Args &g, const Part &p, char *lds, bool &badin,
                                          bool &bad, bool &badseq) {
    typedef Many<D, MID> T;
    typedef typename T::acc acc;
    constexpr int M = T::M, REGS = T::REGS, STEPS = T::STEPS, BLOCKS = T::BLOCKS;
    constexpr int TERMS = Type<BF>::TERMS, SETS = kTile / M, LANES = M == 32 ? 32 : 48;
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64u);
    const uint32_t n = lane % M, part = lane / M;
    const uint32_t r0 = wave * M;
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
        const uint32_t rl = (r0 + M < p.rows ? r0 + M - 1u : p.rows - 1u) + p.row0;
        const uint32_t ta = (p.row0 + r0) / g.group, tb = rl / g.group;
        const uint32_t pa = p.seq.past + ta + 1u, pb = p.seq.past + tb + 1u;
        see1 = g.a.causal ? pb : p.seq.past + p.seq.rows;
        all1 = g.a.causal ? pa : p.seq.past + p.seq.rows;
        if (g.a.window != 0u) {
            see0 = pa > g.a.window ? pa - g.a.window : 0u;
            all0 = pb > g.a.window ? pb - g.a.window : 0u;
        }
    }

    const uint32_t base = lds_addr(lds);
    /* the wave's keys of a tile, K and V: pieces of 1 KiB */
    auto load = [&](uint32_t t, uint32_t buf) {
        const uint32_t at = t * kTile + wave * T::KEYS;
        const Place pl = place_of<D, T::KEYS>(g, p, at, page_at<T::KEYS>(g, p, at), badseq);
        const kq_i4v keys = dma_rsrc(pl.kp, pl.bytes), values = dma_rsrc(pl.vp, pl.bytes);
        const uint32_t to = base + buf * (2u * kTile * T::ROW) + wave * (T::KEYS * T::ROW);
#pragma unroll
        for (uint32_t j = 0; j < T::KEYS * T::ROW / 1024u; ++j) {
            const uint32_t o16 = j * 64u + lane, r = o16 / (D / 8u), c = o16 % (D / 8u);
            const uint32_t rt = wave * T::KEYS + r; /* of the tile */
            const bool in = at + r < p.key1 && at + r >= p.key0;
            const uint32_t a = pl.off + r * T::ROW;
            dma16(keys, in ? a + (c ^ T::k_swap(rt)) * 16u : kOut, to + j * 1024u);
            dma16(values, in ? a + (c ^ T::v_swap(rt)) * 16u : kOut,
                  to + kTile * T::ROW + j * 1024u);
        }
    };
    load(p.t0, 0u);

    Query<BF, STEPS> q;
    const float *qp = g.a.q + (size_t)(p.seq.begin + token) * g.a.qs + (size_t)h * D + 8u * part;
    Raw<STEPS> raw;
    fetch_query(raw, some, [&](int s) { return qp + 512 / M * s; });
    split_query<BF, STEPS, LANES>(g, raw, q, badin);

    acc o[BLOCKS];
#pragma unroll
    for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
        for (int i = 0; i < REGS; ++i) o[b][i] = 0.0f;
    float top = kLowest, total = 0.0f;

    /* K: row n of a block, 16 bytes; V: row `vr` of 16 (M 32: of 8), 8 bytes */
    const uint32_t k_at = base + n * T::ROW + (T::k_swap(n) ^ part) * 16u;
    const uint32_t vr = 4u * part + n % 16u / 4u;
    const uint32_t v_at = base + kTile * T::ROW + vr * T::ROW +
                          (T::v_swap(vr) ^ (n / 16u * 2u) ^ (n % 4u / 2u)) * 16u + (n & 1u) * 8u;
    auto compute = [&](uint32_t t, auto buffer) {
        constexpr uint32_t BUF = decltype(buffer)::value * 2u * kTile * T::ROW;
        const uint32_t at = t * kTile;
        acc s[SETS];
#pragma unroll
        for (int b = 0; b < SETS; ++b)
#pragma unroll
            for (int i = 0; i < REGS; ++i) s[b][i] = 0.0f;
#pragma unroll
        for (uint32_t st = 0; st < STEPS; ++st) {
            e8<BF> k[SETS];
#pragma unroll
            for (uint32_t b = 0; b < SETS; ++b)
                k[b] = __builtin_bit_cast(
                    e8<BF>, *(__attribute__((address_space(3))) u4 *)(uintptr_t)(
                                (k_at ^ (64u / M * st * 16u)) + BUF + b * M * T::ROW));
#pragma unroll
            for (int m = 0; m < TERMS; ++m)
#pragma unroll
                for (uint32_t b = 0; b < SETS; ++b) s[b] = mma(k[b], q.x[st][m], s[b]);
        }
        float lowest = INFINITY; /* of the keys that the row sees */
        if (at + kTile > all1 || at < all0) {
#pragma unroll
            for (uint32_t b = 0; b < SETS; ++b)
#pragma unroll
                for (uint32_t i = 0; i < REGS; ++i) {
                    const uint32_t key = at + M * b + 256u / M * (i / 4u) + 4u * part + i % 4u;
                    const bool seen = key < last && key >= from;
                    if (!BF) lowest = fminf(lowest, seen ? s[b][i] : INFINITY);
                    s[b][i] = seen ? s[b][i] : -INFINITY;
                }
        } else if (!BF) {
#pragma unroll
            for (int i = 0; i < SETS * REGS; ++i) lowest = fminf(lowest, s[i / REGS][i % REGS]);
        }
        float peak = s[0][0];
#pragma unroll
        for (int i = 1; i < SETS * REGS; ++i) peak = fmaxf(peak, s[i / REGS][i % REGS]);
        peak = fmaxf(kq::lanes_max<LANES>(peak) * q.unscale, kLowest) - Type<BF>::LIFT;
        if (__any(peak > top + Type<BF>::SLACK)) {
            const float next = fmaxf(top, peak);
            const float f = __builtin_amdgcn_exp2f(top - next);
            top = next;
            total *= f;
#pragma unroll
            for (int b = 0; b < BLOCKS; ++b) o[b] *= f;
        }
        constexpr uint32_t CHUNK = 512u / M; /* keys of a product */
        /* M 32: half of a block; M 16: four values of each of two */
        auto weights = [&](uint32_t c, float (&w)[8], float top) {
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) {
                const uint32_t x = 8u * c + i;
                w[i] = __builtin_amdgcn_exp2f(fmaf(s[x / REGS][x % REGS], q.unscale, -top));
            }
        };
        auto gather = [&](uint32_t c, const float (&w)[8], uint32_t v_at) {
            e8<BF> pw[TERMS];
            split<BF>(w, pw);
#pragma unroll
            for (uint32_t b = 0; b < BLOCKS; ++b) {
                const uint32_t a = (v_at ^ (b * M * 2u)) + BUF + c * CHUNK * T::ROW;
                const e8<BF> v = join8<BF>(transposed(a), transposed(a + CHUNK / 2u * T::ROW));
#pragma unroll
                for (int m = 0; m < TERMS; ++m) o[b] = mma(v, pw[m], o[b]);
            }
        };
        if constexpr (!BF) {
            const bool small = fmaf(lowest, q.unscale, -top) < kHeldLog2;
            bool rest = __any(small);
            if (rest) {
                f4 vv = f4{kNoSquare, 0.0f, 0.0f, 0.0f}, oo = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
                for (uint32_t i = 0; i < D / 8u; ++i)
                    vv = squares(vv, *(__attribute__((address_space(3))) u4 *)(uintptr_t)(
                                         again(base) + kTile * T::ROW + BUF + 1024u * i +
                                         16u * lane));
#pragma unroll
                for (int b = 0; b < BLOCKS; ++b)
#pragma unroll
                    for (int i = 0; i < REGS; ++i) oo[i % 4] = fmaf(o[b][i], o[b][i], oo[i % 4]);
                const float mine = kq::lanes_sum<LANES>(oo[0] + oo[1] + (oo[2] + oo[3]));
                const float tile = kq::lanes_sum<63>(vv[0] + vv[1] + (vv[2] + vv[3]));
                rest = __any(small && !(mine >= kRestMatters * tile));
            }
            if (rest) {
#pragma unroll
                for (int b = 0; b < BLOCKS; ++b) o[b] *= kRest;
#pragma unroll
                for (uint32_t c = 0; c < kTile / CHUNK; ++c) {
                    float w[8];
                    weights(c, w, again(top));
                    rest_of(w);
                    gather(c, w, again(v_at));
                }
#pragma unroll
                for (int b = 0; b < BLOCKS; ++b) o[b] *= 1.0f / kRest;
            }
        }
        float sum = 0.0f;
#pragma unroll
        for (uint32_t c = 0; c < kTile / CHUNK; ++c) {
            float w[8];
            weights(c, w, top);
#pragma unroll
            for (int i = 0; i < 8; ++i) sum += w[i];
            gather(c, w, v_at);
        }
        total += sum;
    };
    auto step = [&](uint32_t t, auto buffer) {
        wait_vm<0>();
        __syncthreads(); /* the tile is there; the other buffer is read */
        if (t + 1u < p.t1) load(t + 1u, 1u - decltype(buffer)::value);
        if (t * kTile < see1 && t * kTile + kTile > see0) compute(t, buffer);
    };
    /* two tiles a round, so that the buffers' places are constants (8192 rows: 4%) */
    uint32_t t = p.t0;
    for (; t + 1u < p.t1; t += 2u) {
        step(t, Buffer<0u>{});
        step(t + 1u, Buffer<1u>{});
    }
    if (t < p.t1) step(t, Buffer<0u>{});
    total = kq::lanes_sum<LANES>(total);
    if (p.parts > 1u) {
        /* lane by lane, as join_parts reads it */
        float *slot = slot_at(g, p.slot + p.part * p.step);
        f4 *to = (f4 *)slot + wave * (M * D / 4u) + lane;
#pragma unroll
        for (uint32_t k = 0; k < BLOCKS * REGS / 4u; ++k) {
            const uint32_t b = k / (REGS / 4u), i = k % (REGS / 4u) * 4u;
            to[k * 64u] = f4{o[b][i], o[b][i + 1], o[b][i + 2], o[b][i + 3]};
        }
        if (part == 0u) {
            float *m = slot + (size_t)kMany * D;
            m[r0 + n] = top;
            m[kMany + r0 + n] = total;
        }
        return;
    }
    if (!some) return;
    const float inverse = inverse_of_row(g, h, top, total, bad);
#pragma unroll
    for (uint32_t k = 0; k < BLOCKS * REGS / 4u; ++k) {
        const uint32_t b = k / (REGS / 4u), i = k % (REGS / 4u) * 4u;
        put(g, p.seq.begin + token, h, T::column(k, lane),
            f4{o[b][i], o[b][i + 1], o[b][i + 2], o[b][i + 3]}, inverse, badin, bad);
    }
}

/* calls whose items all have few rows, as where every sequence decodes */
template <bool BF, int D, bool MANY>
__global__ __launch_bounds__(kThreads, (few_side<D>())) void attend_few(Args g,
                                                                        uint32_t *status) {
    __shared__ __attribute__((aligned(16))) char lds[few_bytes<D, 4>()];
    Part p = find_part<MANY>(g, g.first + blockIdx.x, status);
    leave(g, p);
    if (!p.live) return;
    p.pin();
    bool badin = false, bad = false, badseq = false;
    few_rows<BF, D, 4>(g, p, lds, badin, bad, badseq);
    if (badseq) kq_flag(status, KQ_DEV_SEQUENCE);
    if (badin) kq_flag(status, KQ_DEV_INPUT);
    if (bad) kq_flag(status, KQ_DEV_NUMERIC);
}

/* calls of few rows that need no join: an item is a workgroup's */
template <bool BF, int D>
__global__ __launch_bounds__((256 * few_side<D>()), (few_side<D>())) void attend_whole(
    Args g, uint32_t *status) {
    constexpr int W = 4 * few_side<D>();
    __shared__ __attribute__((aligned(16))) char lds[few_bytes<D, W>()];
    Part p = find_part<false>(g, blockIdx.x, status);
    if (!p.live) return;
    p.pin();
    bool badin = false, bad = false, badseq = false;
    few_rows<BF, D, W>(g, p, lds, badin, bad, badseq);
    if (badseq) kq_flag(status, KQ_DEV_SEQUENCE);
    if (badin) kq_flag(status, KQ_DEV_INPUT);
    if (bad) kq_flag(status, KQ_DEV_NUMERIC);
}

/* The first 256 workgroups, which begin on a CU each, in reverse: items come longest
 * first, so that the longest of the next 256 lie beside the shortest of these. 8192 rows
 * over themselves 496 us, 515 without (bf16 643, 668); 4096 151, 155 (177, 186). Where all
 * items are long there is nothing to even out, and it costs: 2000 rows of 8 key heads over
 * 4000 more keys 188, 181 (bf16 246, 231), 4096 rows of heads of 64 94, 89. By eights,
 * which leaves a head's workgroups on their XCD. */
__device__ __forceinline__ uint32_t in_turn(uint32_t u) {
    return u < 256u && gridDim.x >= 256u ? (u & 7u) | (248u - (u & ~7u)) : u;
}

template <bool BF, int D, bool MANY>
__global__ __launch_bounds__(Many<D>::THREADS, D == 64 ? 3 : 2) void attend(Args g,
                                                                            uint32_t *status) {
    constexpr int W = Many<D>::W;
    constexpr uint32_t BYTES = Many<D>::LDS > few_bytes<D, W>() ? Many<D>::LDS : few_bytes<D, W>();
    /* a row's pieces are found by flipping address bits below its size */
    __shared__ __attribute__((aligned(1024))) char lds[BYTES];
    bool badin = false, bad = false, badseq = false;
    Part p = find_part<MANY>(g, g.first + in_turn(blockIdx.x), status);
    leave(g, p);
    if (!p.live) return;
    p.pin();
    if (p.block == kFew)
        few_rows<BF, D, W>(g, p, lds, badin, bad, badseq);
    else if (D != 256 && p.block == kMid)
        many_rows<BF, D, D != 256>(g, p, lds, badin, bad, badseq);
    else
        many_rows<BF, D, false>(g, p, lds, badin, bad, badseq);
    if (badseq) kq_flag(status, KQ_DEV_SEQUENCE);
    if (badin) kq_flag(status, KQ_DEV_INPUT);
    if (bad) kq_flag(status, KQ_DEV_NUMERIC);
}

/* four values of a row over some keys, with the exponent they are held by and
 * the weights' sum */
struct Sum {
    f4 v;
    float top, total;

    __device__ __forceinline__ void clear() {
        v = f4{0.0f, 0.0f, 0.0f, 0.0f};
        top = kLowest;
        total = 0.0f;
    }
    __device__ __forceinline__ void add(const Sum &o) {
        const float next = fmaxf(top, o.top);
        const float f = __builtin_amdgcn_exp2f(top - next);
        const float e = __builtin_amdgcn_exp2f(o.top - next);
        top = next;
        total = fmaf(total, f, o.total * e);
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = fmaf(v[c], f, o.v[c] * e);
    }
};
constexpr uint32_t kAtOnce = 4;

/* The parts of items that have several, joined: the workgroup of each part
 * takes its share of the item's values over all parts. */
__global__ __launch_bounds__(kThreads) void join_parts(Args g, uint32_t *status) {
    __shared__ Sum sums[kThreads];
    const Item p = g.items[blockIdx.x]; /* behind the last slot, whatever lies there */
    if (blockIdx.x >= g.plan[3] || p.rows == 0u) return;
    bool badin = false, bad = false;
    /* pieces of four values, in the slots' order: by rows, or by waves and lanes */
    const uint32_t width = g.c.width, tall = p.head_kind >> 16 == 2u ? Many<256>::M : Many<128>::M;
    const bool by_rows = p.head_kind >> 16 == 1u;
    const uint32_t pieces =
        (by_rows ? p.rows : (p.rows + tall - 1u) / tall * tall) * (width / 4u);
    const uint32_t share = p.part * gridDim.y + blockIdx.y, shares = p.parts * gridDim.y;
    const uint32_t a = (uint32_t)((uint64_t)pieces * share / shares);
    const uint32_t b = (uint32_t)((uint64_t)pieces * (share + 1u) / shares);
    /* side by side: pieces in the threads' low bits, parts in the high ones */
    uint32_t wide = 1u;
    while (wide < b - a && wide < (uint32_t)kThreads) wide *= 2u;
    const uint32_t groups = kThreads / wide;
    const uint32_t mine = threadIdx.x % wide, group = threadIdx.x / wide;
    /* kAtOnce pieces of a thread have their loads under way together */
    for (uint32_t at = a; at < b; at += wide * kAtOnce) {
        uint32_t i[kAtOnce], row[kAtOnce], d[kAtOnce];
        bool have[kAtOnce];
        Sum v[kAtOnce];
#pragma unroll
        for (uint32_t u = 0; u < kAtOnce; ++u) {
            i[u] = at + u * wide + mine;
            row[u] = i[u] / (width / 4u);
            d[u] = i[u] % (width / 4u) * 4u;
            if (!by_rows) {
                const uint32_t lane = i[u] % 64u, piece = i[u] / 64u % (tall * width / 256u);
                row[u] = i[u] / (tall * width / 4u) * tall + lane % tall;
                d[u] = tall == 16u ? Many<256>::column(piece, lane)
                                   : Many<128>::column(piece, lane);
            }
            have[u] = i[u] < b && row[u] < p.rows;
            v[u].clear();
        }
        for (uint32_t k = group; k < p.parts; k += groups) {
            const float *slot = slot_at(g, p.slot + k * p.step);
            const float *m = slot + (size_t)g.slot_rows * width;
            Sum x[kAtOnce];
#pragma unroll
            for (uint32_t u = 0; u < kAtOnce; ++u)
                if (have[u]) {
                    x[u].top = m[row[u]];
                    x[u].total = m[g.slot_rows + row[u]];
                    x[u].v = *((const f4 *)slot + i[u]);
                }
#pragma unroll
            for (uint32_t u = 0; u < kAtOnce; ++u)
                if (have[u]) v[u].add(x[u]);
        }
        for (uint32_t step = groups / 2u; step != 0u; step /= 2u) { /* then kAtOnce 1 is enough */
            __syncthreads();
            sums[threadIdx.x] = v[0];
            __syncthreads();
            if (group < step) v[0].add(sums[threadIdx.x + step * wide]);
        }
#pragma unroll
        for (uint32_t u = 0; u < kAtOnce; ++u)
            if (group == 0u && have[u]) {
                const uint32_t r = p.row0 + row[u];
                const uint32_t h = (p.head_kind & 0xffffu) * g.group + r % g.group;
                put(g, p.begin + r / g.group, h, d[u], v[u].v,
                    inverse_of_row(g, h, v[u].top, v[u].total, bad), badin, bad);
            }
    }
    if (badin) kq_flag(status, KQ_DEV_INPUT);
    if (bad) kq_flag(status, KQ_DEV_NUMERIC);
}

/* ------------------------------------------------------------------ host */

struct Sizes {
    uint64_t items, parts, slots;
    uint32_t slot_rows;
    bool whole, wide; /* each item is one part; and a workgroup's of many waves */
    uint64_t plan_bytes, item_bytes, bytes;
};

/* What a call can need, whatever the device holds */
Sizes sizes_of(const kq_launch_pattn &a, const kq_launch_paged &c, const kq_launch_seqs &q) {
    Sizes z;
    const uint64_t group = a.query_heads / c.heads, rows = q.tokens * group;
    const bool single = q.offsets == nullptr;
    z.slot_rows = (single ? group : rows) <= kFew ? kFew : kMany;
    z.items = c.heads * (single ? q.count * ((group + z.slot_rows - 1u) / z.slot_rows)
                                : rows / kMany + q.count);
    /* An item of w tiles has at most w / kLeast + 1/2 parts, at least one. All
     * tiles by the tiles a part are at most kParts. Only sequences whose items may
     * have two parts or more have slots: of w tiles, at least 3/2 parts long,
     * which makes at most 4/3 of their length by a part's. */
    const uint64_t tiles = (((uint64_t)c.table_pages << c.page_shift) + kTile - 1u) / kTile;
    uint64_t sees = tiles; /* that an item reads at most */
    if (a.window != 0u && a.causal != 0u) {
        const uint64_t keys = (uint64_t)a.window + z.slot_rows;
        sees = (keys + kTile - 1u) / kTile + 1u < tiles ? (keys + kTile - 1u) / kTile + 1u : tiles;
    }
    z.wide = z.slot_rows == kFew && q.count <= kByLane && z.items <= kWholeItems &&
             sees * c.width <= (uint64_t)kWhole;
    z.whole = z.wide || sees < kLeast * 3u / 2u ||
              (z.slot_rows == kMany && sees * c.width <= (uint64_t)kWholeMany);
    /* where a call is small, items of many rows are kMany / kFew of few, if there
     * are workgroups for them */
    const uint64_t finest = z.slot_rows == kFew ? z.items : z.items * (kMany / kFew);
    const uint64_t most = finest * (z.whole ? 1u : (tiles + kLeast / 2u) / kLeast + 1u);
    z.parts = most < kParts + z.items ? most : kParts + z.items;
    z.slots = z.whole ? 0u : most < kSlots ? most : kSlots;
    const uint64_t firsts = q.count > kByLane ? 2u * (q.count + 1u) : 0u;
    z.plan_bytes = ((kPlan + firsts) * 4u + 255u) / 256u * 256u;
    /* a call that joins nothing asks for what one of single rows would: scratch of the
     * largest call is enough for all */
    const uint64_t few = c.heads * q.count * ((tiles + kLeast / 2u) / kLeast + 1u);
    const uint64_t held =
        !z.whole ? z.slots : sees < kLeast * 3u / 2u ? 0u : few < kSlots ? few : kSlots;
    z.item_bytes = (held * sizeof(Item) + 255u) / 256u * 256u;
    z.bytes = z.plan_bytes + z.item_bytes +
              held * (z.whole ? kFew : z.slot_rows) * (c.width + 2u) * 4u;
    return z;
}

template <bool MANY>
hipError_t launch_parts(const Args &g, uint32_t parts, bool wide, uint32_t *status, hipStream_t s) {
#define KQ_ATTEND(BF, D)                                                                       \
    if (wide)                                                                                  \
        hipLaunchKernelGGL(HIP_KERNEL_NAME(attend_whole<BF, D>), dim3(parts),                  \
                           dim3(256 * few_side<D>()), 0, s, g, status);                        \
    else if (g.slot_rows == kFew)                                                              \
        hipLaunchKernelGGL(HIP_KERNEL_NAME(attend_few<BF, D, MANY>), dim3(parts),              \
                           dim3(kThreads), 0, s, g, status);                                   \
    else                                                                                       \
        hipLaunchKernelGGL(HIP_KERNEL_NAME(attend<BF, D, MANY>), dim3(parts),                  \
                           dim3(Many<D>::THREADS), 0, s, g, status)
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
    return hipGetLastError();
}

template <bool MANY>
hipError_t launch(Args &g, bool wide, uint32_t *status, hipStream_t s) {
    hipError_t e = hipSuccess;
    if (MANY) {
        hipLaunchKernelGGL(plan_many, dim3(1), dim3(1024), 0, s, g, status);
        e = hipGetLastError();
    }
    for (g.first = 0u; e == hipSuccess && g.first < g.parts; g.first += kLaunch)
        e = launch_parts<MANY>(g, g.parts - g.first < kLaunch ? g.parts - g.first : kLaunch, wide,
                               status, s);
    if (e != hipSuccess || g.slots == 0u) return e; /* nothing to join */
    /* where rows are many, a part's share is shared out again: kAtOnce pieces a thread */
    hipLaunchKernelGGL(join_parts, dim3(g.slots, g.slot_rows == kFew ? 1u : g.c.width / 64u),
                       dim3(kThreads), 0, s, g, status);
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
    g.parts = (uint32_t)z.parts;
    g.first = 0u;
    g.whole = z.whole;
    int exponent = 0;
    const double factor = 2.0 * frexp((double)a->scale * 1.4426950408889634, &exponent);
    g.factor_high = (float)factor;
    g.factor_low = (float)(factor - (double)g.factor_high);
    g.factor_exponent = exponent - 1;
    g.plan = (uint32_t *)scratch;
    g.items = (Item *)((char *)scratch + z.plan_bytes);
    g.partial = (float *)((char *)scratch + z.plan_bytes + z.item_bytes);
    return q->count > kByLane ? launch<true>(g, z.wide, status, s)
                              : launch<false>(g, z.wide, status, s);
}

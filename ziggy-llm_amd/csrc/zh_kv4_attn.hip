// zh_kv4_attn.hip -- attention of a batch of sequences over the paged cache held in 4 bits.
//
// o = sum_t w_t v_t / sum_t w_t, w_t = 2^(s_t - max), s_t = qscale q.k_t, in one pass with the running
// maximum and sum.  A code times its power-of-two scale is exact in bf16, whose exponents are binary32's, so K
// and V enter the matrix cores exactly and no scale is left over to weigh scores or outputs by.  A query and a
// weight enter as three bf16 pieces, cut off by truncation, whose sum they are to the bit.  Products accumulate in
// binary32, maximum and sum are binary32.
//
// Two kernels.  Few columns (a sequence's rows times the query heads of a kv head, up to 64; 32 of head size 256): every
// wavefront streams blocks of 32 positions from memory straight into the products' operands, and the batch's blocks are
// spread over the card, so that long contexts are split and joined.  Many: four wavefronts share pages widened into LDS.
// (48 columns, 7 sequences of 2000 positions, 8 kv heads of 128: 28.2 us by the first, 33.8 by the second; 64 columns, one
// of 9000, heads of 64: 17.0 and 19.3.)
//
// What bounds it (32 heads over 8 kv heads of 128; kernel times under the profiler).  A query at 131071 positions: memory,
// 30.7 us for 143 MB, and the join 4.8.  At 4113: the chain launch, lengths, page, codes, products, exchange 7.0, and the
// join's 3.6.  48 sequences of up to 16384 positions: memory and the last workgroups of uneven sequences, 76 us for 311 MB,
// and 6.4.  2048 queries at 16384: the matrix cores, 1.03 to 1.09 ms by card for three pieces of both products, 1.42 to 1.51
// PFLOP/s (library products of bf16 reach 1.34).
#include <algorithm>

#include "zh_serving.h"

namespace zh {

namespace {

typedef unsigned long long u64;
typedef __bf16 fb2 __attribute__((ext_vector_type(2)));
typedef __bf16 fb8 __attribute__((ext_vector_type(8)));
typedef float ff4 __attribute__((ext_vector_type(4)));

constexpr int kBlock = 32;  // positions of a product
// The running maximum stays where it is while scores pass it by no more than this many powers of two: the outputs are
// scaled again only where one does (with every new maximum of 32 columns, 200 of 480 blocks of a prompt).  Sums of 2^30
// weights of 2^3 and values of 6 2^92 end below 2^128.
constexpr float kSlack = 3.f;
// Scores in powers of two from which on the maximum, rounded, is off by more than an eighth.  Below it s qscale - max is one
// fused step, whose exact result holds the maximum's rounding too, alike in all weights of a column.  From 2^31 on that
// would pass the exponents there are (a lone key at a score of 10^10 had a weight of 0, or an infinite one), so past this
// one the score is rounded as the maximum was: the largest comes to 0 whatever it is.
constexpr float kFar = 0x1p22f;

struct Kv4Params {
    Kv4Layer c;
    Batch b;
    const float *q;
    size_t q_stride;
    float *out;
    int heads, group, q_aligned;
    uint32_t window;
    float qscale, qsign;
    uint32_t few;       // columns up to which a sequence is the few-column kernel's (0: none is)
    uint32_t wgs;       // few: workgroups to spread the blocks over, at most
    uint32_t cus;       // many: workgroups to spread the tiles over, two for each
    uint32_t splits;    // of each tile's positions, at most
    uint32_t *plan;     // of more than 64 sequences: see Plan
    float *part;        // few: partial outputs, and {maximum, sum} of each
    float2 *part_ml;
    float *many_part;   // many: theirs
    float2 *many_part_ml;
};

// The positions that columns first .. last of a sequence see: some of them (first .. last) and all (full_first ..
// full_last), and the blocks of 32 that hold the former.
struct Range {
    int first, last, full_first, full_last;
    int begin, end;
};
__device__ __forceinline__ int first_seen(int pos, uint32_t window) {
    return window && (int64_t)pos >= (int64_t)window ? pos + 1 - (int)window : 0;
}
__device__ __forceinline__ Range range_of(const Kv4Params &p, const Sequence &q, uint32_t first_row, uint32_t last_row) {
    Range r;
    const int a = q.first + (int)first_row, z = q.first + (int)last_row, top = (int)p.b.cap - 1;
    r.first = first_seen(a, p.window), r.full_first = first_seen(z, p.window);
    r.last = min(z, top), r.full_last = min(a, top);
    r.begin = r.first / kBlock;
    r.end = r.last < r.first ? r.begin : r.last / kBlock + 1;
    return r;
}

// the z-th of `parts` shares of begin .. end - 1, the first of them one longer where they are not alike
__device__ __forceinline__ void share(int &begin, int &end, uint32_t parts, uint32_t z) {
    const uint32_t n = (uint32_t)(end - begin), each = n / parts, more = n - each * parts;
    begin += (int)(each * z + min(z, more));
    end = begin + (int)(each + (z < more ? 1u : 0u));
}

// What every lane has alike, in scalar registers.
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
__device__ __forceinline__ Sequence uniform(const Sequence &q) {
    return {uniform(q.index), uniform(q.row0), uniform(q.rows), (int)uniform((uint32_t)q.first)};
}

// Of more than 64 sequences a kernel of its own makes a table, which the others search: for each sequence the end of its
// items among the few-column kernel's and of its tiles among the other's, and the slot of its first split.  Up to 64 every
// wavefront has a sequence a lane, and a table would cost a launch, 4.6 us.  The border is where the lanes end, not where
// the table begins to pay: with every wavefront going through all sequences, 64 at a time, and with the table 2048 sequences
// of 512 positions took 828 us and 302, 512 of 512 127 and 88, but 128 of 1024 40 and 43, 65 of 2048 45 and 49.  A third form
// for those in between would have to take two sequences a lane; without it they pay up to 4 us.
struct Plan {
    const uint32_t *quota, *items, *tiles, *slots;
    __host__ __device__ static size_t words(uint32_t sequences) { return 4 + 3 * (size_t)sequences; }
    __device__ __forceinline__ explicit Plan(const Kv4Params &p)
        : quota(p.plan), items(p.plan + 4), tiles(items + p.b.sequences), slots(tiles + p.b.sequences) {}
};
constexpr uint32_t kLanes = 64;

// The work of the many-column kernel: tiles of columns (a sequence's rows' heads of one kv head, row by row) of the
// sequences with more than `few` columns, times the kv heads, times the splits of their positions that fill the card.
template <int COLUMNS> __device__ __forceinline__ uint32_t tiles_of(const Kv4Params &p, uint32_t columns) {
    return columns > p.few ? (columns + COLUMNS - 1) / COLUMNS : 0u;
}
// How many splits, from the number of tiles that the batch turns out to have.  (A chunk of 400 rows beside 47 sequences of
// one: 57 us and the join 8, from as many as it may have 133.)
__device__ __forceinline__ uint32_t splits_of(const Kv4Params &p, uint32_t tiles) {
    return max(1u, min(p.splits, 2 * p.cus / max(tiles * p.c.nkv, 1u)));
}
// Of these a sequence has as many as leave each two pages of what its rows see, whatever room it has besides: the parts that
// its sums are taken in follow from its tables.  (8 heads over 2 kv heads of 128, with the join: 64 rows of a fresh prompt
// with room for 131072 positions 15.2 us, of all splits that might be 18.8; 180 rows at 1000 positions 19.0 and 21.3; 100 rows
// at 100000 with a window of 1024 20.1 and 22.3.  Of four pages each, 180 rows at 1000: 23.8.)
__device__ __forceinline__ uint32_t splits_of(const Kv4Params &p, const Sequence &q, uint32_t splits) {
    const Range r = range_of(p, q, 0, q.rows - 1);
    return max(1u, min(splits, (uint32_t)((r.end + 1) / 2 - r.begin / 2) / 2));
}
template <int COLUMNS> __device__ __forceinline__ uint32_t all_tiles(const Kv4Params &p) {
    if (p.b.sequences > kLanes) return uniform(Plan(p).tiles[p.b.sequences - 1]);
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t n = lane < p.b.sequences ? tiles_of<COLUMNS>(p, sequence_of(p.b, lane).rows * p.group) : 0u;
    return (uint32_t)__builtin_amdgcn_readlane((int)running_sum(n), 63);
}
// A workgroup's item, the last tiles, which see most, first; count 0: none.  Every lane of a wavefront takes part.
struct Tile {
    Sequence q;
    uint32_t first, count;  // columns
    uint32_t split, splits;
    int head;
};
template <int COLUMNS> __device__ __forceinline__ Tile tile_of(const Kv4Params &p, uint32_t block) {
    Tile t{};
    const uint32_t lane = threadIdx.x & 63, group = (uint32_t)p.group, nkv = (uint32_t)p.c.nkv;
    uint32_t before, number;
    auto item = [&](uint32_t tiles) {
        t.splits = splits_of(p, tiles);
        const uint32_t items = tiles * nkv * t.splits, i = items - 1 - block;
        t.head = (int)(i % nkv), t.split = i / nkv % t.splits, number = i / nkv / t.splits;
        return block < items;
    };
    if (p.b.sequences > kLanes) {
        const Plan plan(p);
        if (!item(uniform(plan.tiles[p.b.sequences - 1]))) return t;
        const uint32_t s = count_up_to(plan.tiles, p.b.sequences, number);
        if (s >= p.b.sequences) return t;
        t.q = uniform(sequence_of(p.b, s));
        before = s ? uniform(plan.tiles[s - 1]) : 0u;
    } else {
        Sequence q{};
        if (lane < p.b.sequences) q = sequence_of(p.b, lane);
        const uint32_t n = tiles_of<COLUMNS>(p, q.rows * group), sum = running_sum(n);
        if (!item((uint32_t)__builtin_amdgcn_readlane((int)sum, 63))) return t;
        const u64 past = __ballot(sum > number);
        if (!past) return t;
        const int at = __ffsll(past) - 1;
        auto of = [&](uint32_t v) { return (uint32_t)__builtin_amdgcn_readlane((int)v, at); };
        t.q = {of(q.index), of(q.row0), of(q.rows), (int)of((uint32_t)q.first)};
        before = of(sum - n);
    }
    t.first = (number - before) * COLUMNS;
    const uint32_t all = t.q.rows * group;  // (tables that don't ascend may pass 32 bits in the sums)
    t.count = number >= before && t.first < all ? min((uint32_t)COLUMNS, all - t.first) : 0u;
    if (t.count) t.splits = splits_of(p, t.q, t.splits);
    if (t.split >= t.splits) t.count = 0;
    return t;
}

// How the few-column kernel spreads a batch: each sequence's tiles of columns, times the kv heads, go through the
// sequence's blocks of 32 positions; together they are spread over p.wgs workgroups, `quota` blocks each at most.  A
// tile's blocks are split evenly; its items follow each other, the kv heads side by side.  Splits that are to be joined
// have slots in the workspace, at most 2 p.wgs of them: a tile has two splits only where it has more than a quota.
struct Share {
    Sequence q;
    uint32_t splits, tiles; // 0: none
    uint32_t index;         // item: within the sequence's
    uint32_t slot;          // of the sequence's first split
};
constexpr uint32_t kFewWaves = 4, kLeastBlocks = kFewWaves;  // of a workgroup: one for each wavefront (16: 4113 positions 9.2 us, not 7.8)

// A sequence's tiles, and its blocks (of all columns: a tile's own are no more).
template <int COLUMNS> __device__ __forceinline__ void load_of(const Kv4Params &p, const Sequence &q, uint32_t &tiles, uint32_t &blocks) {
    const uint32_t columns = q.rows * p.group;
    tiles = blocks = 0;
    if (columns == 0 || columns > p.few) return;
    const Range r = range_of(p, q, 0, q.rows - 1);
    tiles = (columns + COLUMNS - 1) / COLUMNS;
    blocks = max((uint32_t)(r.end - r.begin), 1u);  // rows that see nothing have an item, which writes zeros
}
// One workgroup a CU while that leaves it up to 8 blocks a wavefront, two past that.  (One and two, 8 kv heads of 128: a
// query at 4113 positions 6.65 us and 7.35, 16000 8.9 and 10.1, 32000 12.8 and 13.1, 131071 34.8 and 30.2; 48 sequences 85
// and 76, with three 76.)  Where it is one, half a workgroup is kept for every tile, as its blocks rarely are whole quotas:
// a few items more than CUs take another round (three sequences of 3000 positions, 264 items: 9.4 us).
__device__ __forceinline__ uint32_t quota_of(const Kv4Params &p, u64 total, uint32_t tiles) {
    const double blocks = (double)total * p.c.nkv, cus = 0.5 * p.wgs, one = ceil(blocks / (cus - 0.5 * fmin((double)tiles * p.c.nkv, cus)));
    return max(kLeastBlocks, (uint32_t)fmin(one <= 8 * kFewWaves ? one : ceil(blocks / p.wgs), 0x1p31));
}

// The item with this number, or (BY_SEQUENCE) the sequence.  Every lane of a wavefront takes part.
template <bool BY_SEQUENCE, int COLUMNS> __device__ __forceinline__ Share share_of(const Kv4Params &p, uint32_t number) {
    const uint32_t lane = threadIdx.x & 63, nkv = (uint32_t)p.c.nkv;
    Share t{};
    if (p.b.sequences > kLanes) {
        const Plan plan(p);
        const uint32_t s = BY_SEQUENCE ? number : count_up_to(plan.items, p.b.sequences, number);
        if (s >= p.b.sequences) return t;
        t.q = uniform(sequence_of(p.b, s));
        uint32_t blocks;
        load_of<COLUMNS>(p, t.q, t.tiles, blocks);
        const uint32_t quota = uniform(plan.quota[0]);
        t.splits = (blocks + quota - 1) / quota;
        t.index = number - (s ? uniform(plan.items[s - 1]) : 0u);
        if (!BY_SEQUENCE && t.index >= t.splits * t.tiles * nkv) t.splits = 0;  // (tables that changed on the way)
        t.slot = uniform(plan.slots[s]);
        return t;
    }
    auto of = [](uint32_t v, int at) { return (uint32_t)__builtin_amdgcn_readlane((int)v, at); };
    Sequence q{};  // a lane's
    uint32_t tiles = 0, blocks = 0;
    if (lane < p.b.sequences) q = sequence_of(p.b, lane), load_of<COLUMNS>(p, q, tiles, blocks);
    u64 total = running_sum((u64)blocks * tiles);
    total = (u64)of((uint32_t)(total >> 32), 63) << 32 | of((uint32_t)total, 63);
    const uint32_t quota = uniform(quota_of(p, total, of(running_sum(tiles), 63))), splits = (blocks + quota - 1) / quota, n = splits * tiles * nkv;
    const uint32_t sum = running_sum(n), slot_sum = running_sum(splits > 1 ? n : 0u);
    const u64 past = __ballot(BY_SEQUENCE ? lane == number : sum > number);
    if (!past) return t;
    const int at = __ffsll(past) - 1;
    t.q = {of(q.index, at), of(q.row0, at), of(q.rows, at), (int)of((uint32_t)q.first, at)};
    t.splits = of(splits, at), t.tiles = of(tiles, at);
    t.index = number - of(sum - n, at);
    t.slot = of(slot_sum, at) - (t.splits > 1 ? t.splits * t.tiles * nkv : 0u);
    return t;
}

// The table of more than 64 sequences: one workgroup, 1024 sequences at a time.
template <int FEW, int MANY> __global__ void __launch_bounds__(1024) kv4_plan_kernel(Kv4Params p) {
    __shared__ u64 totals[16];
    __shared__ uint32_t all_tiles[16], sums[3][16];
    const Plan plan(p);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t tiles, blocks;
    auto look = [&](uint32_t s, Sequence &q) {
        q.rows = tiles = blocks = 0;
        if (s < p.b.sequences) q = sequence_of(p.b, s), load_of<FEW>(p, q, tiles, blocks);
    };
    u64 total = 0;
    uint32_t count = 0;
    for (uint32_t s = threadIdx.x; s < p.b.sequences; s += 1024) {
        Sequence q;
        look(s, q);
        total += (u64)blocks * tiles;
        count += tiles;
    }
    total = running_sum(total), count = running_sum(count);
    if (lane == 63) totals[wave] = total, all_tiles[wave] = count;
    __syncthreads();
    total = count = 0;
    for (int i = 0; i < 16; i++) total += totals[i], count += all_tiles[i];
    const uint32_t quota = quota_of(p, total, count);
    if (threadIdx.x == 0) p.plan[0] = quota;
    uint32_t before[3] = {};
    for (uint32_t from = 0; from < p.b.sequences; from += 1024) {
        const uint32_t s = from + threadIdx.x;
        Sequence q;
        look(s, q);
        const uint32_t splits = (blocks + quota - 1) / quota, n = splits * tiles * p.c.nkv;
        const uint32_t own[3] = {n, tiles_of<MANY>(p, q.rows * p.group), splits > 1 ? n : 0u};
        uint32_t sum[3];
        for (int k = 0; k < 3; k++) {
            sum[k] = running_sum(own[k]);
            if (lane == 63) sums[k][wave] = sum[k];
        }
        __syncthreads();
        for (int k = 0; k < 3; k++) {
            uint32_t all = 0, ahead = 0;
            for (int i = 0; i < 16; i++) ahead += i < wave ? sums[k][i] : 0u, all += sums[k][i];
            sum[k] += before[k] + ahead;
            before[k] += all;
        }
        if (s < p.b.sequences) {
            const_cast<uint32_t *>(plan.items)[s] = sum[0];
            const_cast<uint32_t *>(plan.tiles)[s] = sum[1];
            const_cast<uint32_t *>(plan.slots)[s] = sum[2] - own[2];
        }
        __syncthreads();
    }
}

__device__ __forceinline__ uint32_t cut(float v) { return __float_as_uint(v) & 0xFFFF0000u; }
// the upper halves of two words
__device__ __forceinline__ uint32_t upper(uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }
__device__ __forceinline__ uint32_t upper(float a, float b) { return upper(__float_as_uint(a), __float_as_uint(b)); }

// Three bf16 pieces of eight values, exact: each takes the eight leading bits of what the ones before leave.
__device__ __forceinline__ void pieces(const float (&v)[8], fb8 (&to)[3]) {
    uint32_t w[3][4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float a = v[2 * i], b = v[2 * i + 1];
#pragma unroll
        for (int k = 0; k < 3; k++) {
            w[k][i] = upper(a, b);
            a -= __uint_as_float(cut(a)), b -= __uint_as_float(cut(b));
        }
    }
#pragma unroll
    for (int k = 0; k < 3; k++) __builtin_memcpy(&to[k], w[k], 16);
}

template <int SEL> __device__ __forceinline__ uint32_t widen(uint32_t w, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
}
// 2^(byte - 127) as far as the conversion looks: it takes the scale's exponent alone, whatever sign and fraction are
// (every byte with 256 of them: the same), so a shift brings the byte there and nothing is masked.
__device__ __forceinline__ float scale_of(uint32_t w, int byte) { return __uint_as_float(byte < 3 ? w << (23 - 8 * byte) : w >> 1); }

// v f - m, the product rounded
__device__ __forceinline__ float product_less(float v, float f, float m) {
#pragma clang fp contract(off)
    const float z = v * f;
    return z - m;
}

__device__ __forceinline__ float finite(float v) { return v == -INFINITY ? 0.f : v; }
// the sum over four lanes side by side
__device__ __forceinline__ float four(float v) {
    v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xF, 0xF, false));
    return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xF, 0xF, false));
}

// A lane's part of 32 positions: lane (i, g) holds K rows 8 (i / 4) + 4 pt + i % 4 of both halves pt (its words g of
// every 32 dims), and V's dims 32 t + i and 32 t + 16 + i of positions 8 g .. 8 g + 7.
template <int HD> struct Lane4 {
    static constexpr int G = HD / 32;
    uint32_t k[2][G], v[2 * G], ks[2][(G + 3) / 4], vs[2 * G];
    __device__ __forceinline__ void load_k(const Kv4Layer &c, uint32_t page, int head, int half) {
        const uint32_t i = threadIdx.x & 15, g = threadIdx.x >> 4 & 3, row = 8 * (i >> 2) + (i & 3);
        const uint8_t *codes = c.kc + c.codes(page, head) + half * (kBlock / 2 * HD), *scales = c.ks + c.scales(page, head) + half * (kBlock * G);
#pragma unroll
        for (int pt = 0; pt < 2; pt++) {
            __builtin_memcpy(k[pt], codes + (row * (HD / 2) + g * 4 * G) + pt * (2 * HD), 4 * G);
            if constexpr (G % 4) ks[pt][0] = 0;
            __builtin_memcpy(ks[pt], scales + row * G + pt * (4 * G), G);
        }
    }
    __device__ __forceinline__ void load_v(const Kv4Layer &c, uint32_t page, int head, int half) {
        const uint32_t i = threadIdx.x & 15, g = threadIdx.x >> 4 & 3;
        const uint8_t *codes = c.vc + c.codes(page, head) + half * (kBlock / 2 * HD), *scales = c.vs + c.scales(page, head) + half * (kBlock * G);
        __builtin_memcpy(v, codes + (g * 16 + i) * (8 * G), 8 * G);
        __builtin_memcpy(vs, scales + g * (8 * G), 8 * G);
    }
    // V's positions outside first .. last of the block as zeros: what was never stored may read as NaN
    __device__ __forceinline__ void clear_v(int first, int last) {
        const int g = threadIdx.x >> 4 & 3;
#pragma unroll
        for (int w = 0; w < 2 * G; w++) {
            uint32_t keep = 0;
#pragma unroll
            for (int b = 0; b < 4; b++) {
                const int pos = 8 * g + (4 * w + b) / G;
                if (pos >= first && pos <= last) keep |= 255u << 8 * b;
            }
            v[w] &= keep, vs[w] &= keep;
        }
    }
    // K's 16 rows of half pt, dims 32 t ..: the left operand of scores
    __device__ __forceinline__ fb8 key(int t, int pt) const {
        const float scale = scale_of(ks[pt][t / 4], t % 4);
        const uint32_t w[4] = {widen<0>(k[pt][t], scale), widen<1>(k[pt][t], scale), widen<2>(k[pt][t], scale), widen<3>(k[pt][t], scale)};
        fb8 a;
        __builtin_memcpy(&a, w, 16);
        return a;
    }
    // V's dims 32 t + i and 32 t + 16 + i: the left operands of two tiles of outputs
    __device__ __forceinline__ void values(int t, fb8 (&b)[2]) const {
        uint32_t a[2][4];
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
            uint32_t y[2];
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int n = (j + e) * G + t;  // byte of this position's dims
                const float scale = scale_of(vs[n >> 2], n & 3);
                const uint32_t word = v[n >> 2];
                y[e] = (n & 3) == 0   ? widen<0>(word, scale)
                       : (n & 3) == 1 ? widen<1>(word, scale)
                       : (n & 3) == 2 ? widen<2>(word, scale)
                                      : widen<3>(word, scale);
            }
            a[0][j / 2] = __builtin_amdgcn_perm(y[1], y[0], 0x05040100u);
            a[1][j / 2] = __builtin_amdgcn_perm(y[1], y[0], 0x07060302u);
        }
        __builtin_memcpy(b, a, 32);
    }
};

// One wavefront's columns: their queries, running maxima and sums, and outputs.  Scores S^T[position][column] = K Q^T on
// 16x16x32 products, outputs O^T[dim][column] = V^T P^T: what a lane gets of S^T, positions 8 g .. 8 g + 7 of column i,
// is what it gives of P^T.
// PACKED (CT 1): four columns at most, whose three pieces, and a fourth of zeros, are sixteen: lane i holds piece i % 4 of
// column i / 4, so that a product of all pieces is one instead of three.  Scores of the pieces add up across four lanes,
// outputs once at the end.  (A query at 131071 positions 30.7 us, without 38.6; 48 sequences 75 and 95.)
template <int HD, int CT, int AWAY, bool PACKED = false> struct Columns {
    static constexpr int G = HD / 32, DT = HD / 16, P = PACKED ? 1 : 3, NEAR = P - AWAY;
    fb8 q[CT][G][NEAR];
    const fb8 *away;  // the queries' other pieces, [CT][G][AWAY][64] in LDS
    ff4 o[CT][DT];
    float m[CT], l[CT];
    float base[CT];  // what comes off the scores: the maximum (none yet: 0), or 0 where it already is (see kFar)
    bool far;        // some column's maximum is kFar or more either way
    int lo[CT], hi[CT];  // the positions that a column sees, both included

    // Columns first .. first + count - 1 of a sequence: their queries on the way, then in pieces.
    struct Raw {
        float v[CT][G][8];
    };
    __device__ __forceinline__ void fetch(const Kv4Params &p, const Sequence &t, uint32_t first, uint32_t count, int head, Raw &raw) {
        const int i = threadIdx.x & 15, g = threadIdx.x >> 4 & 3;
#pragma unroll
        for (int c = 0; c < CT; c++) {
            const uint32_t column = first + min((uint32_t)(PACKED ? i >> 2 : 16 * c + i), count - 1), row = column / p.group;
            const float *src = p.q + (size_t)(t.row0 + row) * p.q_stride + (size_t)(head * p.group + (int)(column - row * p.group)) * HD;
            hi[c] = t.first + (int)row;
            lo[c] = first_seen(hi[c], p.window);
            hi[c] = min(hi[c], (int)p.b.cap - 1);
#pragma unroll
            for (int k = 0; k < G; k++) {
                const float *from = src + 32 * k + 8 * g;
                if (p.q_aligned) {
                    *reinterpret_cast<float4 *>(raw.v[c][k]) = *reinterpret_cast<const float4 *>(from);
                    *reinterpret_cast<float4 *>(raw.v[c][k] + 4) = *reinterpret_cast<const float4 *>(from + 4);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) raw.v[c][k][e] = from[e];
                }
            }
        }
    }
    __device__ __forceinline__ void begin(const Kv4Params &p, const Raw &raw, fb8 *lds) {
        const int i = threadIdx.x & 15;
        away = lds, far = false;
#pragma unroll
        for (int c = 0; c < CT; c++) {
#pragma unroll
            for (int k = 0; k < G; k++) {
                float v[8];
                fb8 all[3];
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = raw.v[c][k][e] * p.qsign;
                pieces(v, all);
                if constexpr (PACKED) {
                    const fb8 none = {};
                    all[0] = i & 2 ? (i & 1 ? none : all[2]) : i & 1 ? all[1] : all[0];
                }
#pragma unroll
                for (int e = 0; e < P; e++) {
                    if (e < NEAR) q[c][k][e] = all[e];
                    else lds[((c * G + k) * AWAY + e - NEAR) * 64 + (threadIdx.x & 63)] = all[e];
                }
            }
            m[c] = -INFINITY, l[c] = base[c] = 0.f;
#pragma unroll
            for (int d = 0; d < DT; d++) o[c][d] = ff4{0.f, 0.f, 0.f, 0.f};
        }
    }

    // 32 H positions from `at` on, key(h, t, pt) and values(h, t, b) their operands.  edge: some columns may not see all of
    // them (hidden: their page is none).  after_w: runs when the scores are through.
    template <int H, bool HOLD, class K, class V, class B>
    __device__ __forceinline__ void take(float qscale, int at, bool edge, bool hidden, K key, V values, B after_w) {
        const int g = threadIdx.x >> 4 & 3;
        // of a weight, lane i % 4 = 1 takes off the first piece, 2 the second too (3 as well: its outputs are left out)
        const float second = PACKED && (threadIdx.x & 3) > 0 ? -1.f : 0.f, third = PACKED && (threadIdx.x & 3) > 1 ? -1.f : 0.f;
        int lane = threadIdx.x & 63;
        if constexpr (AWAY > 0) __asm__ volatile("" : "+v"(lane));  // (the pieces in LDS are read where they are used, not ahead of the loop)
        ff4 s[H][CT][2];
#pragma unroll
        for (int h = 0; h < H; h++) {
#pragma unroll
            for (int c = 0; c < CT; c++) s[h][c][0] = s[h][c][1] = ff4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < G; t++) {
                fb8 a[2], far[CT][AWAY ? AWAY : 1];
#pragma unroll
                for (int c = 0; c < CT; c++)
#pragma unroll
                    for (int k = 0; k < AWAY; k++) far[c][k] = away[((c * G + t) * AWAY + k) * 64 + lane];
                a[0] = key(h, t, 0), a[1] = key(h, t, 1);
#pragma unroll
                for (int k = 0; k < P; k++)
#pragma unroll
                    for (int c = 0; c < CT; c++)
#pragma unroll
                        for (int pt = 0; pt < 2; pt++)
                            s[h][c][pt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                a[pt], k < NEAR ? q[c][t][k < NEAR ? k : 0] : far[c][k < NEAR ? 0 : k - NEAR], s[h][c][pt], 0, 0, 0);
                if constexpr (HOLD) __builtin_amdgcn_sched_barrier(0);  // (or the operands of all steps take registers at once)
            }
        }
        if constexpr (PACKED) {
#pragma unroll
            for (int h = 0; h < H; h++)
#pragma unroll
                for (int e = 0; e < 8; e++) s[h][0][e >> 2][e & 3] = four(s[h][0][e >> 2][e & 3]);
        }
        if (edge) {
#pragma unroll
            for (int h = 0; h < H; h++)
#pragma unroll
                for (int c = 0; c < CT; c++)
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const int pos = at + kBlock * h + 8 * g + e;
                        if (hidden || pos < lo[c] || pos > hi[c]) s[h][c][e >> 2][e & 3] = -INFINITY;
                    }
        }
        float next[CT];
        bool grows = false;
#pragma unroll
        for (int c = 0; c < CT; c++) {
            float top = s[0][c][0][0];
#pragma unroll
            for (int e = 1; e < 8 * H; e++) top = fmaxf(top, s[e >> 3][c][e >> 2 & 1][e & 3]);
            next[c] = fmaxf(m[c], xmax<32>(xmax<16>(top)) * qscale);
            grows = grows || next[c] > m[c] + kSlack;  // (-infinity: the first)
        }
        if (__any(grows)) {
#pragma unroll
            for (int c = 0; c < CT; c++) {
                const float was = __builtin_amdgcn_exp2f(m[c] - finite(next[c]));
                m[c] = next[c];
                l[c] *= was;
#pragma unroll
                for (int d = 0; d < DT; d++) o[c][d] *= was;
            }
            bool some = false;
#pragma unroll
            for (int c = 0; c < CT; c++) {
                const bool is = fabsf(finite(m[c])) >= kFar;
                base[c] = is ? 0.f : finite(m[c]);
                some = some || is;
            }
            far = __any(some);
        }
        if (far) {
            const float inverse = 1.f / qscale;  // (scores are below 2^128: qscale is above 2^-106)
#pragma unroll
            for (int c = 0; c < CT; c++) {
                if (fabsf(finite(m[c])) < kFar) continue;
#pragma unroll
                for (int h = 0; h < H; h++)
#pragma unroll
                    for (int e = 0; e < 8; e++) s[h][c][e >> 2][e & 3] = product_less(s[h][c][e >> 2][e & 3], qscale, m[c]) * inverse;
            }
        }
#pragma unroll
        for (int h = 0; h < H; h++) {
            fb8 w[CT][P];
#pragma unroll
            for (int c = 0; c < CT; c++) {
                float v[8], sum = 0.f;
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] = __builtin_amdgcn_exp2f(fmaf(s[h][c][e >> 2][e & 3], qscale, -base[c])), sum += v[e];
                l[c] += sum;
                if constexpr (PACKED) {
                    uint32_t own[4];
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        v[e] = fmaf(second, __uint_as_float(cut(v[e])), v[e]);
                        v[e] = fmaf(third, __uint_as_float(cut(v[e])), v[e]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) own[e] = upper(v[2 * e], v[2 * e + 1]);
                    __builtin_memcpy(&w[c][0], own, 16);
                } else {
                    pieces(v, w[c]);
                }
            }
            if (h == H - 1) after_w();
#pragma unroll
            for (int t = 0; t < G; t++) {
                fb8 b[2];
                values(h, t, b);
#pragma unroll
                for (int k = 0; k < P; k++)
#pragma unroll
                    for (int c = 0; c < CT; c++)
#pragma unroll
                        for (int d = 0; d < 2; d++)
                            o[c][2 * t + d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[d], w[c][k], o[c][2 * t + d], 0, 0, 0);
                if constexpr (HOLD) __builtin_amdgcn_sched_barrier(0);
            }
        }
    }

    // The blocks begin, begin + step .. below end, the next one's loads under way during the work on one.
    // ready: what else has to be done before, behind the first loads.
    template <bool HOLD, class F>
    __device__ __forceinline__ void run(const Kv4Params &p, const Range &r, uint32_t sequence, int head, int begin, int end, int step, F ready) {
        if (begin >= end) {
            ready();
            return;
        }
        const int lane = threadIdx.x & 63;
        uint32_t pages = 0;  // of the next 64 blocks, one a lane; those that the pool doesn't have: 0, not seen
        u64 missing = 0;
        auto look = [&](int b) {
            const int at = b + step * lane;
            pages = 0xFFFFFFFFu;
            if (at < end) pages = page_of(p.b, sequence, (uint32_t)at * kBlock);
            const bool none = pages >= p.b.pool;
            if (none) pages = 0;
            missing = __ballot(none);
        };
        look(begin);
        const int n = (end - begin + step - 1) / step;
        auto page = [&](int i) { return (uint32_t)__builtin_amdgcn_readlane((int)pages, i & 63); };
        auto half = [&](int i) { return (begin + step * i) & 1; };
        int i = 0;
        auto at = [&](int j) { return (begin + step * j) * kBlock; };
        auto inner = [&](int j) { return at(j) >= r.full_first && at(j) + kBlock - 1 <= r.full_last && !(missing >> (j & 63) & 1); };
        Lane4<HD> x, y;
        x.load_k(p.c, page(0), head, half(0)), x.load_v(p.c, page(0), head, half(0));
        __builtin_amdgcn_sched_barrier(0);
        ready();
        auto both = [&](Lane4<HD> &now, Lane4<HD> &after) {
            const bool hidden = missing >> (i & 63) & 1, edge = !inner(i);
            if ((i & 63) == 63) look(begin + step * (i + 1));
            const int j = min(i + 1, n - 1);
            const uint32_t next = page(j);
            after.load_k(p.c, next, head, half(j)), after.load_v(p.c, next, head, half(j));
            if (edge) now.clear_v(r.first - at(i), hidden ? -1 : r.last - at(i));
            take<1, HOLD>(p.qscale, at(i), edge, hidden, [&](int, int t, int pt) { return now.key(t, pt); },
                          [&](int, int t, fb8(&b)[2]) { now.values(t, b); }, [] {});
            i++;
        };
        while (i < n) {
            both(x, y);
            if (i < n) both(y, x);
        }
    }
};

__device__ __forceinline__ float *column_of(float *out, const Kv4Params &p, const Sequence &q, int head, uint32_t column, int hd) {
    const uint32_t row = column / p.group;
    return out + ((size_t)(q.row0 + row) * p.heads + head * p.group + (column - row * p.group)) * hd;
}

// Few columns (decoding): a workgroup takes an item, its wavefronts blocks in turn, joined in LDS.  (Eight wavefronts: a
// batch of 48 103 us instead of 84.  One workgroup a share of exactly as many blocks, sequences cut wherever it ends: 79
// instead of 75, 4113 positions 10.1 instead of 7.5, for the registers and the chain of loads of every unit in a row.)
template <int HD, int CT, bool PACKED> struct FewItem {
    static constexpr int N = PACKED ? 4 : 16 * CT, AWAY = !PACKED && HD * CT > 128 ? 2 : 0;
    static constexpr int PIECES = CT * (HD / 32) * AWAY * 64;  // of a wavefront (16 bytes each)
    static constexpr int OUTPUTS = kFewWaves * N * (HD + 4), HELD = kFewWaves * PIECES * 4;
    static constexpr int LDS = (OUTPUTS > HELD ? OUTPUTS : HELD) + 2 * kFewWaves * N;
};
// lds: the queries' pieces, then the wavefronts' outputs, and their maxima and sums.  SLOT: columns of a slot.
template <int HD, int CT, bool PACKED, int SLOT>
__device__ __forceinline__ void few_item(const Kv4Params &p, const Share &t, int head, const Range &r, int begin, int end, uint32_t first,
                                         uint32_t count, float *lds) {
    typedef FewItem<HD, CT, PACKED> I;
    constexpr int N = I::N, C = HD / 4, AWAY = I::AWAY, PIECES = I::PIECES;
    float(*os)[N][HD + 4] = reinterpret_cast<float(*)[N][HD + 4]>(lds);
    float(*ms)[N] = reinterpret_cast<float(*)[N]>(lds + (I::LDS - 2 * kFewWaves * N)), (*ls)[N] = ms + kFewWaves;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), i = tid & 15, g = tid >> 4 & 3;
    Columns<HD, CT, AWAY, PACKED> x;
    typename Columns<HD, CT, AWAY, PACKED>::Raw raw;
    x.fetch(p, t.q, first, count, head, raw);
    x.template run<(HD * CT > 128)>(p, r, t.q.index, head, begin + wave, end, kFewWaves,
                                    [&] { x.begin(p, raw, reinterpret_cast<fb8 *>(lds) + wave * PIECES); });
    if (AWAY) __syncthreads();
#pragma unroll
    for (int c = 0; c < CT; c++) {
        if ((uint32_t)(16 * c) >= count) break;
        const float l = xsum<32>(xsum<16>(x.l[c]));
        const int column = PACKED ? i >> 2 : 16 * c + i;
        if (g == 0 && !(PACKED && (i & 3))) ms[wave][column] = x.m[c], ls[wave][column] = l;
#pragma unroll
        for (int d = 0; d < HD / 16; d++) {
            float4 v = make_float4(x.o[c][d][0], x.o[c][d][1], x.o[c][d][2], x.o[c][d][3]);
            if (PACKED) {
                if ((i & 3) == 3) v = make_float4(0.f, 0.f, 0.f, 0.f);  // (the third piece's once more)
                v = make_float4(four(v.x), four(v.y), four(v.z), four(v.w));
            }
            if (!(PACKED && (i & 3))) *reinterpret_cast<float4 *>(&os[wave][column][16 * d + 4 * g]) = v;
        }
    }
    __syncthreads();
    for (uint32_t u = tid; u < count * C; u += 64 * kFewWaves) {
        const uint32_t column = u / C;
        const int d = 4 * (int)(u % C);
        float m = ms[0][column];
#pragma unroll
        for (int w = 1; w < (int)kFewWaves; w++) m = fmaxf(m, ms[w][column]);
        const float mf = finite(m);
        float l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < (int)kFewWaves; w++) {
            const float f = __builtin_amdgcn_exp2f(ms[w][column] - mf);
            const float4 v = *reinterpret_cast<const float4 *>(&os[w][column][d]);
            l = fmaf(f, ls[w][column], l);
            o.x = fmaf(f, v.x, o.x), o.y = fmaf(f, v.y, o.y), o.z = fmaf(f, v.z, o.z), o.w = fmaf(f, v.w, o.w);
        }
        if (t.splits > 1) {
            const size_t at = ((size_t)t.slot + t.index) * SLOT + column;
            *reinterpret_cast<float4 *>(p.part + at * HD + d) = o;
            if (d == 0) p.part_ml[at] = make_float2(m, l);
        } else {
            const float inv = l == 0.f ? 0.f : 1.f / l;  // (rows that see nothing: zeros)
            *reinterpret_cast<float4 *>(column_of(p.out, p, t.q, head, first + column, HD) + d) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        }
    }
}

// Items of up to 16 CT columns (4: PACKED), each at its own width: beside a prompt's chunk or drafts to verify most
// sequences of a batch have one row.  (47 of a row beside one of 6: 60 us, all at that one's width 111.)
template <int HD, int CT, bool PACKED> __global__ void __launch_bounds__(64 * kFewWaves, 2) kv4_few_kernel(Kv4Params p) {
    constexpr int N = FewItem<HD, CT, PACKED>::N;
    __shared__ __align__(16) float lds[FewItem<HD, CT, PACKED>::LDS];
    const Share t = share_of<false, N>(p, blockIdx.x);
    if (t.splits == 0) return;
    const int head = (int)(t.index % p.c.nkv);
    const uint32_t z = t.index / p.c.nkv % t.splits, first = t.index / p.c.nkv / t.splits * N, count = min(t.q.rows * p.group - first, (uint32_t)N);
    const Range r = range_of(p, t.q, first / p.group, (first + count - 1) / p.group);
    int begin = r.begin, end = r.end;
    share(begin, end, t.splits, z);
    if (PACKED || count <= 4) few_item<HD, 1, true, N>(p, t, head, r, begin, end, first, count, lds);
    if constexpr (!PACKED) {
        if (count > 4 && (CT == 1 || count <= 16)) few_item<HD, 1, false, N>(p, t, head, r, begin, end, first, count, lds);
        if constexpr (CT > 1)
            if (count > 16 && (CT == 2 || count <= 32)) few_item<HD, 2, false, N>(p, t, head, r, begin, end, first, count, lds);
        if constexpr (CT > 2)
            if (count > 32 && (CT == 3 || count <= 48)) few_item<HD, 3, false, N>(p, t, head, r, begin, end, first, count, lds);
        if constexpr (CT > 3)
            if (count > 48) few_item<HD, 4, false, N>(p, t, head, r, begin, end, first, count, lds);
    }
}

// Joins the splits of a sequence's kv head, a column at a time: a float4 of every N-th split a thread, four under way.
template <int HD, int COLUMNS> __device__ __forceinline__ void join_few(const Kv4Params &p, uint32_t unit, uint32_t from, uint32_t step) {
    constexpr int C = HD / 4, N = 256 / C, Z = 4;
    __shared__ float4 os[N][C];
    __shared__ float ls[N], ms[N];
    const Share t = share_of<true, COLUMNS>(p, unit / p.c.nkv);
    if (t.splits < 2) return;
    const int head = (int)(unit % p.c.nkv), tid = threadIdx.x, c = tid % C, n = tid / C;
    const uint32_t count = t.q.rows * p.group;
    for (uint32_t column = from; column < count; column += step) {
        const uint32_t tile = column / COLUMNS, within = column - tile * COLUMNS;
        auto at = [&](uint32_t z) { return ((size_t)t.slot + (tile * t.splits + min(z, t.splits - 1)) * p.c.nkv + head) * COLUMNS + within; };
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        float m = -INFINITY, l = 0.f;
        if (n < N)
            for (uint32_t z = n; z < t.splits; z += N * Z) {
                float2 ml[Z];
                float4 v[Z];
                float top = m;
#pragma unroll
                for (int e = 0; e < Z; e++) {
                    ml[e] = p.part_ml[at(z + e * N)];
                    v[e] = *reinterpret_cast<const float4 *>(p.part + at(z + e * N) * HD + 4 * c);
                }
#pragma unroll
                for (int e = 0; e < Z; e++) top = fmaxf(top, ml[e].x);
                const float mf = finite(top), was = __builtin_amdgcn_exp2f(m - mf);
                m = top;
                l *= was, o.x *= was, o.y *= was, o.z *= was, o.w *= was;
#pragma unroll
                for (int e = 0; e < Z; e++) {
                    const float f = z + e * N < t.splits ? __builtin_amdgcn_exp2f(ml[e].x - mf) : 0.f;
                    l = fmaf(f, ml[e].y, l);
                    o.x = fmaf(f, v[e].x, o.x), o.y = fmaf(f, v[e].y, o.y), o.z = fmaf(f, v[e].z, o.z), o.w = fmaf(f, v[e].w, o.w);
                }
            }
        if (n < N) {
            os[n][c] = o;
            if (c == 0) ls[n] = l, ms[n] = m;
        }
        __syncthreads();
        if (n == 0) {
            for (int k = 1; k < N; k++) m = fmaxf(m, ms[k]);
            const float mf = finite(m);
            o = make_float4(0.f, 0.f, 0.f, 0.f), l = 0.f;
            for (int k = 0; k < N; k++) {
                const float f = __builtin_amdgcn_exp2f(ms[k] - mf);
                const float4 v = os[k][c];
                l = fmaf(f, ls[k], l);
                o.x = fmaf(f, v.x, o.x), o.y = fmaf(f, v.y, o.y), o.z = fmaf(f, v.z, o.z), o.w = fmaf(f, v.w, o.w);
            }
            const float inv = l == 0.f ? 0.f : 1.f / l;
            *reinterpret_cast<float4 *>(column_of(p.out, p, t.q, head, column, HD) + 4 * c) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        }
        __syncthreads();
    }
}
template <int HD, int COLUMNS> __global__ void __launch_bounds__(256) kv4_few_join_kernel(Kv4Params p) {
    join_few<HD, COLUMNS>(p, blockIdx.x, blockIdx.y, gridDim.y);
}

// Many columns (prompts): a workgroup takes a tile of 64 CT columns, a wavefront 16 CT of them, through a split of its
// pages.  A page's operands are widened once, a quarter by each wavefront, into LDS, in the order in which the
// products take them; two pages' room, so that one barrier a page is enough.  (2048 queries at 16384: CT 2 1.04 ms, CT 1
// 1.28; every wavefront widening all for itself 1.62.)
template <int HD> struct Quarter {  // wavefront (half h, pt): K rows of half h, its 16 of pt; V of half h, every second t from pt on
    static constexpr int G = HD / 32, T = (G + 1) / 2;
    Lane4<HD> x;
    __device__ __forceinline__ void load(const Kv4Layer &c, uint32_t page, int head, int wave) {
        const uint32_t i = threadIdx.x & 15, g = threadIdx.x >> 4 & 3, row = 8 * (i >> 2) + (i & 3);
        const int half = wave >> 1, pt = wave & 1;
        const uint8_t *codes = c.kc + c.codes(page, head) + half * (kBlock / 2 * HD) + pt * (2 * HD);
        const uint8_t *scales = c.ks + c.scales(page, head) + half * (kBlock * G) + pt * (4 * G);
        __builtin_memcpy(x.k[0], codes + (row * (HD / 2) + g * 4 * G), 4 * G);
        if constexpr (G % 4) x.ks[0][0] = 0;
        __builtin_memcpy(x.ks[0], scales + row * G, G);
        x.load_v(c, page, head, half);
    }
    // to: K's chunks [half][pt][t], V's [half][dim tile], of 64 lanes each
    __device__ __forceinline__ void store(fb8 *to, int wave) const {
        const int lane = threadIdx.x & 63;
#pragma unroll
        for (int t = 0; t < G; t++) to[(wave * G + t) * 64 + lane] = x.key(t, 0);
        fb8 *v = to + 4 * G * 64 + (wave >> 1) * (2 * G * 64) + lane;
        auto put = [&](int t) {
            fb8 b[2];
            x.values(t, b);
            v[2 * t * 64] = b[0], v[(2 * t + 1) * 64] = b[1];
        };
        if (wave & 1) {
#pragma unroll
            for (int t = 1; t < G; t += 2) put(t);
        } else {
#pragma unroll
            for (int t = 0; t < G; t += 2) put(t);
        }
    }
};

template <int HD, int CT> __global__ void __launch_bounds__(256, 2) kv4_many_kernel(Kv4Params p) {
    constexpr int G = HD / 32, PAGE = 8 * G * 64;  // a page's operands
    __shared__ fb8 pages[2][PAGE];
    const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), i = threadIdx.x & 15, g = threadIdx.x >> 4 & 3, lane = threadIdx.x & 63;
    const Tile t = tile_of<64 * CT>(p, blockIdx.x);
    if (t.count == 0) return;
    const int head = t.head;
    const Range r = range_of(p, t.q, t.first / p.group, (t.first + t.count - 1) / p.group);
    int begin = r.begin / 2, end = r.end > r.begin ? (r.end + 1) / 2 : r.begin / 2;
    share(begin, end, t.splits, t.split);
    Columns<HD, CT, 0> x;
    const uint32_t first = t.first + 16 * CT * wave;
    typename Columns<HD, CT, 0>::Raw raw;
    x.fetch(p, t.q, min(first, t.first + t.count - 1), first < t.first + t.count ? t.first + t.count - first : 1, head, raw);
    uint32_t ids = 0;  // of the next 64 pages, one a lane; those that the pool doesn't have: 0, not seen
    u64 missing = 0;
    auto look = [&](int b) {
        ids = 0xFFFFFFFFu;
        if (b + lane < end) ids = page_of(p.b, t.q.index, (uint32_t)(b + lane) * kPage);
        const bool none = ids >= p.b.pool;
        if (none) ids = 0;
        missing = __ballot(none);
    };
    auto id = [&](int n) { return (uint32_t)__builtin_amdgcn_readlane((int)ids, (n - begin) & 63); };
    Quarter<HD> y;
    if (begin < end) {
        look(begin);
        y.load(p.c, id(begin), head, wave);
    }
    x.begin(p, raw, nullptr);
    for (int n = begin; n < end; n++) {
        const int at = n * kPage;
        const bool hidden = missing >> ((n - begin) & 63) & 1, edge = hidden || at < r.full_first || at + kPage - 1 > r.full_last;
        fb8 *page = pages[n & 1];
        if (edge) {
            const int from = at + kBlock * (wave >> 1);
            y.x.clear_v(r.first - from, hidden ? -1 : r.last - from);
        }
        y.store(page, wave);
        if (n + 1 < end && ((n - begin) & 63) == 63) look(n + 1);
        __syncthreads();
        x.template take<2, false>(p.qscale, at, edge, hidden, [&](int h, int t, int pt) { return page[((2 * h + pt) * G + t) * 64 + lane]; },
                                  [&](int h, int t, fb8(&b)[2]) {
                                      const fb8 *v = page + (4 * G + 2 * G * h + 2 * t) * 64 + lane;
                                      b[0] = v[0], b[1] = v[64];
                                  },
                                  [&] { y.load(p.c, id(min(n + 1, end - 1)), head, wave); });
    }
#pragma unroll
    for (int c = 0; c < CT; c++) {
        const float l = xsum<32>(xsum<16>(x.l[c])), inv = l == 0.f ? 0.f : 1.f / l;
        const uint32_t column = first + 16 * c + i;
        if (column >= t.first + t.count) continue;
        float *out = t.splits > 1 ? p.many_part + (size_t)t.split * p.b.rows * p.heads * HD : p.out;
        float *to = column_of(out, p, t.q, head, column, HD);
#pragma unroll
        for (int d = 0; d < HD / 16; d++)
            *reinterpret_cast<float4 *>(to + 16 * d + 4 * g) = make_float4(x.o[c][d][0] * inv, x.o[c][d][1] * inv, x.o[c][d][2] * inv, x.o[c][d][3] * inv);
        if (t.splits > 1 && g == 0) p.many_part_ml[(to - p.many_part) / HD] = make_float2(x.m[c], l);
    }
}
// The splits of a row's heads joined, a thread four dims.
template <int HD, int COLUMNS> __device__ __forceinline__ void join_many(const Kv4Params &p, uint32_t row, uint32_t block) {
    const uint32_t most = splits_of(p, all_tiles<COLUMNS>(p));
    if (most == 1) return;
    const Sequence q = sequence_of_row(p.b, row);
    if (q.rows * p.group <= p.few) return;  // (none's, or the other kernel's)
    const int splits = (int)splits_of(p, q, most);
    if (splits == 1) return;
    const uint32_t u = block * 256 + threadIdx.x;
    if (u < (uint32_t)p.heads * (HD / 4)) {
        const size_t at = (size_t)row * p.heads + u / (HD / 4), each = (size_t)p.b.rows * p.heads;
        const int d = 4 * (int)(u % (HD / 4));
        constexpr int Z = 8;  // under way at once
        float m = -INFINITY, l = 0.f;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int z = 0; z < splits; z += Z) {
            float2 ml[Z];
            float4 v[Z];
            float top = m;
#pragma unroll
            for (int e = 0; e < Z; e++) {
                const size_t from = min(z + e, splits - 1) * each + at;
                ml[e] = p.many_part_ml[from];
                v[e] = *reinterpret_cast<const float4 *>(p.many_part + from * HD + d);
            }
#pragma unroll
            for (int e = 0; e < Z; e++) top = fmaxf(top, ml[e].x);
            const float mf = finite(top), was = __builtin_amdgcn_exp2f(m - mf);
            m = top;
            l *= was, o.x *= was, o.y *= was, o.z *= was, o.w *= was;
#pragma unroll
            for (int e = 0; e < Z; e++) {
                const float f = z + e < splits ? __builtin_amdgcn_exp2f(ml[e].x - mf) * ml[e].y : 0.f;
                l += f;
                o.x = fmaf(f, v[e].x, o.x), o.y = fmaf(f, v[e].y, o.y), o.z = fmaf(f, v[e].z, o.z), o.w = fmaf(f, v[e].w, o.w);
            }
        }
        const float inv = l == 0.f ? 0.f : 1.f / l;
        *reinterpret_cast<float4 *>(p.out + at * HD + d) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    }
}
template <int HD, int COLUMNS> __global__ void __launch_bounds__(256) kv4_many_join_kernel(Kv4Params p) {
    join_many<HD, COLUMNS>(p, blockIdx.x, blockIdx.y);
}
// Both joins in one launch (a small batch's time is its launches').  x: `units` of the one, then the rows of the other; y:
// few_y and many_y of them.
template <int HD, int FEW, int MANY>
__global__ void __launch_bounds__(256) kv4_both_join_kernel(Kv4Params p, uint32_t units, uint32_t few_y, uint32_t many_y) {
    if (blockIdx.x < units) {
        if (blockIdx.y < few_y) join_few<HD, FEW>(p, blockIdx.x, blockIdx.y, few_y);
    } else if (blockIdx.y < many_y) {
        join_many<HD, MANY>(p, blockIdx.x - units, blockIdx.y);
    }
}

}  // namespace

hipError_t launch_kv4_attention(const Kv4Attn &a, int cus, hipStream_t s) {
    Kv4Params p{};
    p.c = a.c, p.b = a.b, p.q = a.q, p.q_stride = a.q_stride, p.out = a.out;
    p.heads = a.heads, p.group = a.heads / a.c.nkv, p.q_aligned = a.q_aligned;
    p.window = a.window, p.qscale = a.qscale, p.qsign = a.qsign;
    const uint64_t nkv = a.c.nkv, most = (uint64_t)a.b.max_rows * p.group, all = (uint64_t)a.b.rows * p.group;
    const uint64_t blocks = (a.b.cap + kBlock - 1) / kBlock;  // of a sequence, at most
    const uint32_t limit = a.c.hd <= 128 ? 64 : 32;
    // a batch of one sequence is one kernel's; others may hold sequences of both kinds
    p.few = a.b.sequences == 1 && most > limit ? 0 : limit;
    const bool planned = a.b.sequences > kLanes;
    p.plan = (uint32_t *)a.part;
    const size_t plan_floats = planned ? (Plan::words(a.b.sequences) + 3) / 4 * 4 : 0;
    if (a.part_floats < plan_floats + 4 * 64 * 260) return hipErrorInvalidValue;
    auto go = [&](auto h, auto ct_few, auto ct_many) {
        constexpr int HD = decltype(h)::value, FEW = decltype(ct_few)::value, MANY = decltype(ct_many)::value;
        constexpr uint64_t M = 64 * MANY;
        const bool several = a.b.sequences > 1, many = most > p.few;
        const uint64_t units = a.b.sequences * nkv, columns = std::min<uint64_t>(most, limit);
        const uint64_t n = many || most > 16 ? 16 * FEW : most > 4 ? 16 : 4;  // columns of a few-column item
        const uint64_t per = (blocks + kLeastBlocks - 1) / kLeastBlocks;      // its splits, at most
        uint64_t few_items = 0, many_items = 0;
        float *part = a.part + plan_floats;
        size_t part_floats = a.part_floats - plan_floats;
        if (p.few) {
            p.wgs = 2 * cus;
            while (p.wgs > 1 && 2 * p.wgs * n * (HD + 2) > part_floats / 2) p.wgs /= 2;
            const uint64_t tiles = units * ((columns + n - 1) / n), slots = 2 * (uint64_t)p.wgs * n;
            few_items = std::min(p.wgs + tiles, tiles * per);
            p.part = part, p.part_ml = (float2 *)(part + slots * HD);
            part += slots * (HD + 2), part_floats -= slots * (HD + 2);
        }
        if (many) {
            // tiles of a sequence alone; of several, at most and at least as many, however the rows are theirs
            const uint64_t few_columns = (uint64_t)p.few * a.b.sequences;
            const uint64_t most_tiles = several ? all / M + std::min<uint64_t>(a.b.sequences, all / (p.few + 1)) : (most + M - 1) / M;
            const uint64_t least_tiles = several ? std::max<uint64_t>(1, all > few_columns ? (all - few_columns) / M : 1) : most_tiles;
            const uint64_t each = (uint64_t)a.b.rows * a.heads * (HD + 2);
            p.cus = (uint32_t)cus;
            // of the positions that a tile's rows see, two pages a split at least, and 32 splits at most
            const uint64_t tile_rows = std::min<uint64_t>(a.b.max_rows, (M - 1) / p.group + 2), pages = (a.b.cap + kPage - 1) / kPage;
            const uint64_t seen = a.window ? std::min(pages, (a.window + tile_rows - 2) / kPage + 2) : pages;
            p.splits = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>({2 * (uint64_t)cus / (least_tiles * nkv), seen / 2, 32,
                                                                           part_floats / each}));
            p.many_part = part, p.many_part_ml = (float2 *)(part + (size_t)p.splits * a.b.rows * a.heads * HD);
            many_items = p.splits > 1 ? std::max<uint64_t>(most_tiles * nkv, 2 * (uint64_t)cus) : most_tiles * nkv;
        }
        // what is resident at once, 8 workgroups a CU (40 sequences of up to 4 rows: 7.0 us, of half as many 9.1, of twice 8.5)
        const unsigned few_y = (unsigned)std::min<uint64_t>(columns, std::max<uint64_t>(1, 8 * (uint64_t)cus / units));
        const unsigned many_y = (unsigned)((a.heads * (HD / 4) + 255) / 256);
        auto plan = [&](auto f) {
            if (planned) hipLaunchKernelGGL((kv4_plan_kernel<decltype(f)::value, (int)M>), dim3(1), dim3(1024), 0, s, p);
        };
        auto few = [&](auto ct, auto packed) {
            constexpr int CT = decltype(ct)::value, N = FewItem<HD, CT, decltype(packed)::value>::N;
            plan(std::integral_constant<int, N>{});
            hipLaunchKernelGGL((kv4_few_kernel<HD, CT, decltype(packed)::value>), dim3((unsigned)few_items), dim3(64 * kFewWaves), 0, s, p);
            if (per > 1 && !many) hipLaunchKernelGGL((kv4_few_join_kernel<HD, N>), dim3((unsigned)units, few_y), dim3(256), 0, s, p);
        };
        if (!p.few) {
            hipLaunchKernelGGL((kv4_many_kernel<HD, MANY>), dim3((unsigned)many_items), dim3(256), 0, s, p);
            if (p.splits > 1) hipLaunchKernelGGL((kv4_many_join_kernel<HD, (int)M>), dim3(a.b.rows, many_y), dim3(256), 0, s, p);
        } else if (many) {
            few(ct_few, std::false_type{});
            hipLaunchKernelGGL((kv4_many_kernel<HD, MANY>), dim3((unsigned)many_items), dim3(256), 0, s, p);
            const unsigned rows = p.splits > 1 ? a.b.rows : 0;
            if (per > 1)
                hipLaunchKernelGGL((kv4_both_join_kernel<HD, 16 * FEW, (int)M>),
                                   dim3((unsigned)units + rows, rows ? std::max(few_y, many_y) : few_y), dim3(256), 0, s, p, (uint32_t)units,
                                   few_y, many_y);
        } else if (most <= 4) {
            few(std::integral_constant<int, 1>{}, std::true_type{});
        } else if (most <= 16) {
            few(std::integral_constant<int, 1>{}, std::false_type{});
        } else {
            few(ct_few, std::false_type{});
        }
    };
    switch (a.c.hd) {
    case 64: go(std::integral_constant<int, 64>{}, std::integral_constant<int, 4>{}, std::integral_constant<int, 2>{}); break;
    case 96: go(std::integral_constant<int, 96>{}, std::integral_constant<int, 2>{}, std::integral_constant<int, 2>{}); break;
    case 128: go(std::integral_constant<int, 128>{}, std::integral_constant<int, 2>{}, std::integral_constant<int, 2>{}); break;
    case 256: go(std::integral_constant<int, 256>{}, std::integral_constant<int, 1>{}, std::integral_constant<int, 1>{}); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace zh

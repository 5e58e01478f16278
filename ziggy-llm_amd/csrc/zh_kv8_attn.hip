// zh_kv8_attn.hip -- attention over the cache held in 8 bits.
//
// o = sum_t w_t v_t / sum_t w_t, w_t = 2^(s_t - max), s_t = qscale q.k_t, in one pass with the running
// maximum and sum.  The codes are integers of at most 127, exact in binary16, and enter the matrix
// cores as they are; a block's scales multiply its scores and its weights.  A query enters as two
// binary16 pieces of q 2^e (the power of two that brings the row's largest value to [2^14, 2^15)), a
// weight as two of 2^14 w, each rounded to nearest: q to 2^-22, w to 2^-22 of itself or 2^-37 of the
// largest (see pieces).  Products accumulate in binary32, maximum and sum are binary32.
//
// Two kernels.  Few (query, head) rows of a kv head (decoding): a wavefront streams blocks of 32
// positions, K and V straight from memory into operands.  Many (prompts): a workgroup's 128 rows share
// tiles of 64 positions in LDS.  Both split the positions over workgroups where rows alone leave CUs
// idle; a second launch joins the splits in their order, so results don't change from run to run.
//
// What bounds them (32 heads of 128 over 8 kv heads; mean and least of 60 launches): one query of 131071
// positions memory, 268 MB in 49.9 (47.9) us, 5.4 TB/s, and 4.8 (4.3) of the join; of 4113 positions the chain
// of loads, products and exchange, 7.4 (7.0), of which 1.5 are its one block, and 3.1 (2.4) of the join; 9 queries
// of 16398 positions vector issue and memory about alike, 22.7 (22.0) and 4.5 (3.8); 2048 queries of 14336 to 16384
// positions the matrix cores, 992 (958), 1.04 PFLOP/s with both pieces counted.
#include <algorithm>
#include <cmath>

#include "zh_longctx.h"

namespace zh {

namespace {

typedef _Float16 kh2 __attribute__((ext_vector_type(2)));
typedef _Float16 kh8 __attribute__((ext_vector_type(8)));
typedef float kf4 __attribute__((ext_vector_type(4)));
typedef float kf16 __attribute__((ext_vector_type(16)));

constexpr int kMaxSplits = 256;  // one a thread when they are joined
constexpr float kWeight = 16384.f;  // of the largest weight: its pieces below binary16's 65504

__device__ __forceinline__ uint32_t first_seen(uint32_t pos, uint32_t window) {
    return window && pos >= window ? pos + 1 - window : 0u;
}

// four codes -> binary16: 0x64XX is 1024 + XX, XX = code + 128
__device__ __forceinline__ void widen4(uint32_t w, uint32_t &a, uint32_t &b) {
    const uint32_t u = w ^ 0x80808080u;
    const kh2 off = {(_Float16)-1152.f, (_Float16)-1152.f};
    a = __builtin_bit_cast(uint32_t, __builtin_bit_cast(kh2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + off);
    b = __builtin_bit_cast(uint32_t, __builtin_bit_cast(kh2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + off);
}
__device__ __forceinline__ kh8 widen8(uint32_t x, uint32_t y) {
    uint4 r;
    widen4(x, r.x, r.y);
    widen4(y, r.z, r.w);
    return __builtin_bit_cast(kh8, r);
}

// The power of two that brings a row's largest value to [2^14, 2^15), and its inverse.
__device__ __forceinline__ void row_power(float largest, float &up, float &down) {
    const uint32_t e = max(__float_as_uint(largest) >> 23 & 255u, 15u);
    const bool fine = e < 255u;  // (an infinity or NaN: as it is)
    up = fine ? __uint_as_float((268u - e) << 23) : 1.f;
    down = fine ? __uint_as_float((e - 14u) << 23) : 1.f;
}

// eight values of a query row, the row's start on 16 bytes or not
__device__ __forceinline__ void load8(const float *q, int aligned, float (&v)[8]) {
    if (aligned) {
        const float4 a = *reinterpret_cast<const float4 *>(q), b = *reinterpret_cast<const float4 *>(q + 4);
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
        for (int e = 0; e < 8; e++) v[e] = q[e];
    }
}

// the z-th of `parts` shares of 0 .. n - 1, the first n % parts of them one longer
__device__ __forceinline__ void share(uint32_t n, uint32_t parts, uint32_t z, uint32_t &begin, uint32_t &end) {
    if (parts == 1) {
        begin = 0, end = n;
        return;
    }
    const uint32_t each = n / parts, more = n - each * parts;
    begin = each * z + min(z, more);
    end = begin + each + (z < more ? 1u : 0u);
}

__device__ __forceinline__ float uniform(float v) { return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(v))); }
__device__ __forceinline__ float finite(float v) { return v == -INFINITY ? 0.f : v; }

// Two weights' pieces.  A weight below 2^-14 is rounded in binary16's denormal range first, to 2^-25, and
// what that leaves, times 2^14 up to 2^-11, to 2^-23: 2^-37 of the largest weight.  (2^14 w rounded
// instead, by products ahead or in the exponential's argument: 2^-39, and 2048 queries after 14336 positions 1000
// to 1030 us against 980: the lesser pieces hold bits where these are 0, and the matrix cores draw more power.)
__device__ __forceinline__ void pieces(float a, float b, uint32_t &hi, uint32_t &lo) {
    const kh2 h = kh2{(_Float16)a, (_Float16)b} * (_Float16)kWeight;  // (exact)
    const kh2 l = {(_Float16)fmaf(a, kWeight, -(float)h[0]), (_Float16)fmaf(b, kWeight, -(float)h[1])};
    hi = __builtin_bit_cast(uint32_t, h), lo = __builtin_bit_cast(uint32_t, l);
}

// A block's V scale as a share of the largest: its log2 goes into the weights' exponent, w = 2^(s +
// log2 share - max), and the weights over the share add to the sum.  (A multiplication of a block's
// outputs instead would be an FMA per output and block.)  An all-zero block, whose codes are 0, counts as
// a share of 2^-60: the sum keeps its weights.  Other shares are at least 2^-32 here (their log2 is held
// to 2^-19): see far_apart.
__device__ __forceinline__ void share_of(float scale, float big, float &log_share, float &inverse) {
    const float share = scale / big;
    log_share = big > 0.f ? __builtin_amdgcn_logf(share < 0x1p-60f ? 0x1p-60f : share) : 0.f * scale;
    inverse = __builtin_amdgcn_exp2f(-log_share);
}

// Four dims' sums of weighted outputs, in 64 bits: the mean of values lies within binary32, their sum may not, nor
// the products with weights below 1.
struct Wide4 {
    double x, y, z, w;
    __device__ __forceinline__ void add(double f, const float4 &v) {
        x = fma(f, (double)v.x, x), y = fma(f, (double)v.y, y), z = fma(f, (double)v.z, z), w = fma(f, (double)v.w, w);
    }
    __device__ __forceinline__ void shrink(double f) { x *= f, y *= f, z *= f, w *= f; }
    __device__ __forceinline__ float4 over(double n) const { return make_float4((float)(x * n), (float)(y * n), (float)(z * n), (float)(w * n)); }
};

struct Kv8Params {
    Kv8Layer c;
    const float *q;
    size_t q_stride;
    float *out, *part, *part_ml;  // splits > 1: row r of split z at part + (z rows + r) hd, {max, sum} at part_ml + ...2
    uint32_t position, queries, window;
    int heads, group, splits, q_aligned;
    uint32_t per_group;  // ceil(2^16 / group): rows / group of the few and of a workgroup (both below 128) by a product
    __device__ __forceinline__ uint32_t query_of(uint32_t row) const { return row * per_group >> 16; }
    float qscale;
};

// Scales of V, the largest and the smallest that is not 0, too far apart for weights that hold them in
// their exponent: a row may see the small ones only, or give the large ones next to no weight.
__device__ __forceinline__ bool far_apart(float largest, float smallest) { return !(smallest >= largest * 0x1p-32f); }
constexpr float kNoScale = INFINITY;  // the smallest of none
__device__ __forceinline__ float wave_min_scale(float scale) { return -wave_max_f32(scale > 0.f ? -scale : -kNoScale); }

// For such scales alone: a block's weights are of its own largest, w = 2^(s - block max), their outputs t a
// product by themselves, which 2^(block max - max) and the scale multiply on their way into the row's:
// o = o 2^(was - max) + (t 2^(block max - max)) scale.  The pieces then hold what counts of each block.  Sums of
// 2^31 values past 2^87 would leave binary32: they are taken in units of 2^32, which costs values below 2^-94 bits.
// (A pass where the first block's values are 2^-40 of the others': 2048 queries after 14336 positions 1779 us against
// 994, 9 queries after 16389 36.3 against 26.4, one after 4112 11.3 against 10.3.  A row at a time without matrix
// cores: 288 ms, 1106 and 57 us.)
__device__ __forceinline__ float far_unit(float largest) { return largest >= 0x1p80f ? 0x1p32f : 1.f; }

// One block of a row: its largest score `top` (-infinity: none in sight) in scores' unit f, the row's running
// maximum m (updated); `was`: what the row's sums shrink by, the result: what the block's do, -1 of a block out of
// sight, which gives nothing whatever its scale.
__device__ __forceinline__ float take_block(float top, float f, float &block_max, float &m, float &was) {
    const bool seen = top > -INFINITY;
    block_max = seen ? top * f : 0.f;
    const float mn = seen ? fmaxf(m, block_max) : m;
    was = __builtin_amdgcn_exp2f(m - finite(mn));
    m = mn;
    return seen ? __builtin_amdgcn_exp2f(block_max - mn) : -1.f;
}

// ---- few rows ----
//
// A wavefront takes blocks of 32 positions (4 wavefronts of a workgroup in turn).  Scores on
// 16x16x32 products, S[position][column] = K Q^T; lane (i, g) holds K row 8 (i / 4) + 4 pt + i % 4 of
// its half pt, so that the 8 scores it gets back are of positions 8 g .. 8 g + 7, in order: what the
// value products O[column][dim] = P V take as their left operand, and what its 8 bytes of a V dim
// hold.  Up to 8 rows (NR 8): 16 columns are their two pieces.  More: CT tiles of 16 rows, each piece
// a product, which share the blocks' loads and widening.
template <int HD, int NR> struct Few {
    static constexpr bool PAIRED = NR == 8;
    static constexpr int CT = PAIRED ? 1 : NR / 16;    // column tiles
    static constexpr int P = PAIRED ? 1 : 2;           // products of a step: both pieces in one, or one for each
    static constexpr int KS = HD / 32, DT = HD / 16;   // k-steps, dim tiles
    static constexpr int KB = HD % 64 ? 8 : 16;        // bytes of a lane's K load
    static constexpr int KL = HD / 4 / KB;             // K loads of a row
    static constexpr int KW = KB / 4;
};
template <int HD> struct Block8 {
    uint32_t k[2][HD / 16], v[HD / 16][2];
};

template <int HD, int NR>
__global__ void __launch_bounds__(256, 1) kv8_few_kernel(Kv8Params p) {
    using F = Few<HD, NR>;
    constexpr int CT = F::CT, P = F::P;
    __shared__ __align__(16) float os[4][NR][HD + 4];
    __shared__ float ms[4][NR], ls[4][NR], unit[4];  // unit: of a wavefront's outputs
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, i16 = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.x % p.c.nkv, z = blockIdx.y;
    const uint32_t rows = p.queries * (uint32_t)p.group, r0 = blockIdx.x / p.c.nkv * NR;
    const uint32_t rlast = min(r0 + NR, rows) - 1;
    // the blocks that any of the rows sees, and this split's share of them
    const uint32_t pos_min = p.position + p.query_of(r0), pos_max = p.position + p.query_of(rlast);
    const uint32_t lo_min = first_seen(pos_min, p.window), lo_max = first_seen(pos_max, p.window);
    const uint32_t b_first = lo_min / kKv8Block, nb_all = pos_max / kKv8Block - b_first + 1;
    uint32_t b0, b1;
    share(nb_all, (uint32_t)p.splits, (uint32_t)z, b0, b1);
    b0 += b_first, b1 += b_first;
    const int nb = (int)(b1 - b0) > wave ? (int)((b1 - b0 - wave + 3) / 4) : 0;  // of this wavefront: b0 + wave + 4 t

    const size_t head0 = (size_t)kvh * p.c.blocks;
    const int8_t *kl = p.c.kc + head0 * (kKv8Block * HD) + (size_t)(8 * (i16 >> 2) + (i16 & 3)) * HD + F::KB * g;
    const int8_t *vl = p.c.vc + head0 * (kKv8Block * HD) + (size_t)i16 * kKv8Block + 8 * g;
    auto block_of = [&](int t) { return b0 + wave + 4 * (uint32_t)min(t, nb - 1); };
    auto load = [&](Block8<HD> &r, int t) {
        const size_t at = (size_t)block_of(t) * (kKv8Block * HD);
#pragma unroll
        for (int pt = 0; pt < 2; pt++)
#pragma unroll
            for (int j = 0; j < F::KL; j++)
                __builtin_memcpy(&r.k[pt][F::KW * j], kl + at + 4 * pt * HD + 4 * F::KB * j, F::KB);
#pragma unroll
        for (int d = 0; d < F::DT; d++) __builtin_memcpy(r.v[d], vl + at + d * (16 * kKv8Block), 8);
    };
    // of the wavefront's next 64 blocks, one a lane: the K scale, log2 of the V scale's share of `big` (the
    // largest V scale so far), and the share's inverse
    float ksl = 0.f, vsl = 0.f, lvl = 0.f, inl = 0.f, big = 0.f, small = kNoScale;
    auto load_scales = [&](int t) {
        const uint32_t b = block_of(t + lane);
        ksl = p.c.ks[head0 + b], vsl = p.c.vs[head0 + b];
    };
    Block8<HD> x, y;

    // this lane's column of tile c: a row, and of paired ones a piece of it
    auto row_of = [&](int c, int column) { return min(r0 + (uint32_t)(F::PAIRED ? column >> 1 : 16 * c + column), rlast); };
    // first dim of step s: byte 8 s of a lane's row
    auto dim_of = [&](int s) { return 4 * F::KB * (8 * s / F::KB) + F::KB * g + 8 * s % F::KB; };
    kh8 qb[CT][P][F::KS];
    float down[CT];
    {
        float qv[CT][F::KS][8];
#pragma unroll
        for (int c = 0; c < CT; c++) {
            const uint32_t row = row_of(c, i16), qi = p.query_of(row);
            const float *q = p.q + (size_t)qi * p.q_stride + (size_t)(kvh * p.group + (int)(row - qi * p.group)) * HD;
#pragma unroll
            for (int s = 0; s < F::KS; s++) load8(q + dim_of(s), p.q_aligned, qv[c][s]);
        }
        // the queries' loads go first, K and V right behind them: all are under way while the queries are cut
        if (nb > 0) {
            load_scales(0);
            load(x, 0);
            load(y, 1);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int c = 0; c < CT; c++) {
            float top = 0.f, up;
#pragma unroll
            for (int s = 0; s < F::KS; s++)
#pragma unroll
                for (int e = 0; e < 8; e++) qv[c][s][e] *= p.qscale, top = fmaxf(top, fabsf(qv[c][s][e]));
            top = xmax<32>(xmax<16>(top));
            row_power(top, up, down[c]);
#pragma unroll
            for (int s = 0; s < F::KS; s++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float v = qv[c][s][e] * up;
                    const _Float16 h = (_Float16)v, l = (_Float16)(v - (float)h);
                    if constexpr (F::PAIRED) qb[c][0][s][e] = i16 & 1 ? l : h;
                    else qb[c][0][s][e] = h, qb[c][1][s][e] = l;
                }
        }
    }
    kf4 o[CT][F::DT];
    float m[CT], l[CT];
#pragma unroll
    for (int c = 0; c < CT; c++) {
        m[c] = -INFINITY, l[c] = 0.f;
#pragma unroll
        for (int d = 0; d < F::DT; d++) o[c][d] = kf4{0.f, 0.f, 0.f, 0.f};
    }
    // the next 64 blocks' scales against the largest so far: outputs are in its unit, maxima hold its log2
    auto take_scales = [&]() {
        const float next = fmaxf(big, wave_max_f32(vsl));
        if (next > big) {
            const float r = big > 0.f ? next / big : 1.f, lg = __builtin_amdgcn_logf(r);
#pragma unroll
            for (int c = 0; c < CT; c++) {
                l[c] *= r, m[c] -= lg;
#pragma unroll
                for (int d = 0; d < F::DT; d++)
                    if (big == 0.f) o[c][d] = kf4{0.f, 0.f, 0.f, 0.f};  // (of zeros alone)
            }
            big = next;
        }
        small = fminf(small, wave_min_scale(vsl));
        share_of(vsl, big, lvl, inl);
        return !far_apart(big, small);
    };

    // a block's scores, in units of ks down[c]
    auto scores = [&](const Block8<HD> &r, kf4 (&s)[CT][2]) {
#pragma unroll
        for (int pt = 0; pt < 2; pt++) {
#pragma unroll
            for (int c = 0; c < CT; c++) s[c][pt] = kf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < F::KS; k++) {
                const kh8 a = widen8(r.k[pt][2 * k], r.k[pt][2 * k + 1]);
#pragma unroll
                for (int c = 0; c < CT; c++)
#pragma unroll
                    for (int j = 0; j < P; j++) s[c][pt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, qb[c][j][k], s[c][pt], 0, 0, 0);
            }
        }
    };
    // this lane's 8 scores of tile c, those out of sight -infinity; which are in sight
    auto column = [&](const kf4 (&s)[CT][2], int c, bool edge, uint32_t first, float (&w)[8]) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            w[e] = s[c][e >> 2][e & 3];
            if constexpr (F::PAIRED)  // the other piece's column
                w[e] += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(w[e]), 0xB1, 0xF, 0xF, false));
        }
        uint32_t keep = 255;
        if (edge) {
            const uint32_t pos = p.position + p.query_of(row_of(c, i16)), lo = first_seen(pos, p.window);
            keep = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const uint32_t at = first + 8 * g + e;
                const bool in = at >= lo && at <= pos;
                keep |= (uint32_t)in << e;
                if (!in) w[e] = -INFINITY;
            }
        }
        return keep;
    };
    // the column's weights' pieces, and their sum
    auto weigh = [&](const float (&w)[8], kh8 (&ph)[P]) {
        float sum = 0.f;
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int e = 0; e < 4; e++) {
            sum += w[2 * e] + w[2 * e + 1];
            pieces(w[2 * e], w[2 * e + 1], hi[e], lo[e]);
            if constexpr (F::PAIRED) hi[e] = i16 & 1 ? lo[e] : hi[e];
        }
        ph[0] = __builtin_bit_cast(kh8, uint4{hi[0], hi[1], hi[2], hi[3]});
        if constexpr (!F::PAIRED) ph[1] = __builtin_bit_cast(kh8, uint4{lo[0], lo[1], lo[2], lo[3]});
        return sum;
    };
    auto compute = [&](const Block8<HD> &r, int t) {
        const uint32_t first = block_of(t) * kKv8Block;
        auto of_block = [&](float v) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), t & 63)); };
        const float ks = of_block(ksl), lv = of_block(lvl), inv = of_block(inl);
        const bool edge = first < lo_max || first + kKv8Block - 1 > pos_min;
        kf4 s[CT][2];
        scores(r, s);
        kh8 ph[CT][P];
#pragma unroll
        for (int c = 0; c < CT; c++) {
            float w[8], mx = -INFINITY;
            const float f = ks * down[c];
            const uint32_t keep = column(s, c, edge, first, w);
#pragma unroll
            for (int e = 0; e < 8; e++) mx = fmaxf(mx, w[e]);
            mx = fmaf(xmax<32>(xmax<16>(mx)), f, lv);
            if (__any(mx > m[c])) {
                const float mn = fmaxf(m[c], mx), al = __builtin_amdgcn_exp2f(m[c] - finite(mn));
                m[c] = mn;
                l[c] *= al;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float a = __shfl(al, 4 * g + j);
#pragma unroll
                    for (int d = 0; d < F::DT; d++) o[c][d][j] *= a;
                }
            }
            const float to = lv - finite(m[c]);
#pragma unroll
            for (int e = 0; e < 8; e++) w[e] = __builtin_amdgcn_exp2f(fmaf(w[e], f, to));
            if (edge)
#pragma unroll
                for (int e = 0; e < 8; e++)
                    if (!(keep >> e & 1u)) w[e] = 0.f;
            const float sum = weigh(w, ph[c]);
            // (a row with none of the block in sight takes nothing from it, whatever its scale)
            l[c] += sum == 0.f ? 0.f : sum * inv;
        }
#pragma unroll
        for (int d = 0; d < F::DT; d++) {
            const kh8 v = widen8(r.v[d][0], r.v[d][1]);
#pragma unroll
            for (int c = 0; c < CT; c++)
#pragma unroll
                for (int j = 0; j < P; j++) o[c][d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[c][j], v, o[c][d], 0, 0, 0);
        }
    };

    // the same where scales are far apart
    auto compute_far = [&](const Block8<HD> &r, int t) {
        const uint32_t first = block_of(t) * kKv8Block;
        auto of_block = [&](float v) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(v), t & 63)); };
        const float ks = of_block(ksl), vs = of_block(vsl) / big;
        kf4 s[CT][2];
        scores(r, s);
        kh8 ph[CT][P];
        float was[CT][4], now[CT][4];  // of the rows that this lane holds outputs of
#pragma unroll
        for (int c = 0; c < CT; c++) {
            float w[8], top = -INFINITY, block_max, shrink;
            const float f = ks * down[c];
            const uint32_t keep = column(s, c, true, first, w);
#pragma unroll
            for (int e = 0; e < 8; e++) top = fmaxf(top, w[e]);
            const float share = take_block(xmax<32>(xmax<16>(top)), f, block_max, m[c], shrink);
#pragma unroll
            for (int e = 0; e < 8; e++) {
                w[e] = __builtin_amdgcn_exp2f(fmaf(w[e], f, -block_max));
                if (!(keep >> e & 1u)) w[e] = 0.f;
            }
            const float sum = weigh(w, ph[c]);
            l[c] = fmaf(l[c], shrink, sum == 0.f ? 0.f : sum * fmaxf(share, 0.f));
#pragma unroll
            for (int j = 0; j < 4; j++) was[c][j] = __shfl(shrink, 4 * g + j), now[c][j] = __shfl(share * (1.f / kWeight), 4 * g + j);
        }
#pragma unroll
        for (int d = 0; d < F::DT; d++) {
            const kh8 v = widen8(r.v[d][0], r.v[d][1]);
#pragma unroll
            for (int c = 0; c < CT; c++) {
                kf4 b = kf4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < P; j++) b = __builtin_amdgcn_mfma_f32_16x16x32_f16(ph[c][j], v, b, 0, 0, 0);
#pragma unroll
                for (int j = 0; j < 4; j++)
                    o[c][d][j] = now[c][j] < 0.f ? o[c][d][j] * was[c][j] : fmaf(b[j] * now[c][j], vs, o[c][d][j] * was[c][j]);
            }
        }
    };

    bool together = true;
    float weight_unit = 1.f / kWeight;  // of the outputs' weights
    if (nb > 0) {
        together = take_scales();
        for (int t = 0; t < nb && together; t += 2) {
            if (t && (t & 63) == 0) {
                load_scales(t);
                together = take_scales();
            }
            compute(x, t);
            load(x, t + 2);
            if (t + 1 < nb) compute(y, t + 1);
            load(y, t + 3);
        }
    }
    if (!together) {  // from the first block again
#pragma unroll
        for (int c = 0; c < CT; c++) {
            m[c] = -INFINITY, l[c] = 0.f;
#pragma unroll
            for (int d = 0; d < F::DT; d++) o[c][d] = kf4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll 1
        for (int t = 0; t < nb; t += 64) {
            load_scales(t);
            big = fmaxf(big, wave_max_f32(vsl));
        }
        big = far_unit(big), weight_unit = 1.f;
#pragma unroll 1
        for (int t = 0; t < nb; t++) {
            if ((t & 63) == 0) load_scales(t);
            load(x, t);
            compute_far(x, t);
        }
    }
    // the wavefront's rows: both pieces' outputs, the sum over its lanes
    const uint32_t live = rlast - r0 + 1;
#pragma unroll
    for (int c = 0; c < CT; c++) {
        const float sum = xsum<32>(xsum<16>(l[c]));
#pragma unroll
        for (int d = 0; d < F::DT; d++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if constexpr (F::PAIRED) {
                    if (j % 2 == 0) os[wave][2 * g + j / 2][16 * d + i16] = (o[c][d][j] + o[c][d][j + 1]) * weight_unit;
                } else
                    os[wave][16 * c + 4 * g + j][16 * d + i16] = o[c][d][j] * weight_unit;
            }
        if (lane < 16 && (!F::PAIRED || lane % 2 == 0)) {
            const int r = F::PAIRED ? lane / 2 : 16 * c + lane;
            ms[wave][r] = m[c], ls[wave][r] = sum;
        }
    }
    if (lane == 0) unit[wave] = big;
    __syncthreads();
    for (int u = tid; u < (int)live * (HD / 4); u += 256) {
        const int r = u / (HD / 4), d = 4 * (u % (HD / 4));
        const float mx = fmaxf(fmaxf(ms[0][r], ms[1][r]), fmaxf(ms[2][r], ms[3][r])), mf = finite(mx);
        float sum = 0.f;
        Wide4 a = {};
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float al = __builtin_amdgcn_exp2f(ms[w][r] - mf);
            sum = fmaf(al, ls[w][r], sum);
            a.add((double)al * unit[w], *reinterpret_cast<const float4 *>(&os[w][r][d]));
        }
        const uint32_t gr = r0 + r, qi = p.query_of(gr);
        const size_t to = (size_t)qi * p.heads + kvh * p.group + (gr - qi * p.group), at = (size_t)z * p.queries * p.heads + to;
        // a split's outputs are those of its own positions (0 where it has none in sight)
        const float n = p.splits > 1 && mx == -INFINITY && sum == 0.f ? 0.f : 1.f / sum;
        *reinterpret_cast<float4 *>(p.splits > 1 ? p.part + at * HD + d : p.out + to * HD + d) = a.over(n);
        if (p.splits > 1 && d == 0) *reinterpret_cast<float2 *>(p.part_ml + 2 * at) = make_float2(mx, sum);
    }
}

// ---- many rows ----
//
// A workgroup takes 128 (query, head) rows of one kv head, 32 a wavefront, over tiles of 64 positions
// (two blocks), widened to binary16 on their way into LDS, two tiles deep.  S[position][row] = K Q^T
// and O[dim][row] = V^T P^T on 32x32x16 products.  K rows are read with bits 2 and 3 of their index
// exchanged, so that a lane's weights are of positions 16 k + 8 h .. + 7: 16 bytes of a V dim in LDS.
template <int HD> constexpr int kManyPerCu = HD <= 128 ? 2 : 1;

template <int HD> __global__ void __launch_bounds__(256, kManyPerCu<HD>) kv8_many_kernel(Kv8Params p) {
    constexpr int KT = HD / 16, DT = HD / 32;
    constexpr int KST = 2 * HD + 16, VST = 2 * 64 + 16;      // bytes of a K row and of a V dim: 16 rows in distinct banks
    constexpr int BUF = 64 * KST + HD * VST;
    constexpr int UN = 4 * HD, NU = (UN + 255) / 256;         // 16-byte pieces of a K or V tile, of a thread
    __shared__ __align__(16) char lds[2 * BUF];
    __shared__ float top_scale[4], low_scale[4];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, l32 = lane & 31, lh = lane >> 5;
    const int kvh = blockIdx.x % p.c.nkv, z = blockIdx.y;
    const int qn = 128 / p.group, nqb = ((int)p.queries + qn - 1) / qn, qb = nqb - 1 - (int)blockIdx.x / p.c.nkv;
    const int q0 = qb * qn, qlast = min(q0 + qn, (int)p.queries) - 1;
    const uint32_t kv_last = p.position + qlast, kv_first = first_seen(p.position + q0, p.window);
    const int t_first = (int)(kv_first >> 6), nt_all = (int)(kv_last >> 6) + 1 - t_first;
    uint32_t s0, s1;
    share((uint32_t)nt_all, (uint32_t)p.splits, (uint32_t)z, s0, s1);
    const int t0 = t_first + (int)s0, t1 = t_first + (int)s1;
    const int v = wave * 32 + l32, vq = (int)p.query_of(v), qi = q0 + vq, vh = v - vq * p.group, head = kvh * p.group + vh;
    const bool valid = v < qn * p.group && qi <= qlast;
    const int qc = min(qi, qlast);
    const uint32_t qpos = p.position + qc, qlo = first_seen(qpos, p.window);
    // the wavefront's earliest query, and the latest one's first position: tiles between need no mask
    const uint32_t wave_first = p.position + min(q0 + wave * 32 / p.group, qlast);
    const uint32_t wave_lo = first_seen(p.position + min(q0 + (wave * 32 + 31) / p.group, qlast), p.window);
    const size_t head0 = (size_t)kvh * p.c.blocks;
    const uint32_t last_block = kv_last / kKv8Block, first_block = kv_first / kKv8Block;

    uint4 kr[NU], vr[NU];
    auto load = [&](int t) {
        const uint32_t ba = 2 * (uint32_t)t, bb = min(ba + 1, last_block);
        const int8_t *ka = p.c.kc + (head0 + ba) * (kKv8Block * HD), *kb = p.c.kc + (head0 + bb) * (kKv8Block * HD);
        const int8_t *va = p.c.vc + (head0 + ba) * (kKv8Block * HD), *vb = p.c.vc + (head0 + bb) * (kKv8Block * HD);
#pragma unroll
        for (int i = 0; i < NU; i++) {
            const int u = min(tid + 256 * i, UN - 1);
            const bool second = u >= UN / 2;
            const int at = 16 * (second ? u - UN / 2 : u);
            kr[i] = *reinterpret_cast<const uint4 *>((second ? kb : ka) + at);
            vr[i] = *reinterpret_cast<const uint4 *>((second ? vb : va) + at);
        }
    };
    auto put = [&](int t) {
        char *ks = lds + (t & 1) * BUF, *vs = ks + 64 * KST;
#pragma unroll
        for (int i = 0; i < NU; i++) {
            const int u = tid + 256 * i;
            if (UN % 256 && u >= UN) break;
            constexpr int R = HD / 16;  // 16-code pieces of a K row
            uint4 a, b;
            auto widen = [&](const uint4 &x) {
                widen4(x.x, a.x, a.y), widen4(x.y, a.z, a.w), widen4(x.z, b.x, b.y), widen4(x.w, b.z, b.w);
            };
            widen(kr[i]);
            uint4 *kd = reinterpret_cast<uint4 *>(ks + u / R * KST + u % R * 32);
            kd[0] = a, kd[1] = b;
            widen(vr[i]);
            const int w = u % (2 * HD), half = u / (2 * HD);  // a block's dims hold two pieces each
            uint4 *vd = reinterpret_cast<uint4 *>(vs + w / 2 * VST + half * 64 + w % 2 * 32);
            vd[0] = a, vd[1] = b;
        }
    };

    // the largest V scale in this workgroup's range, and the smallest
    float big = 0.f, small = kNoScale;
    for (int b = 2 * t0 + tid; b < 2 * t1; b += 256)
        if ((uint32_t)b >= first_block && (uint32_t)b <= last_block) {
            const float scale = p.c.vs[head0 + b];
            big = fmaxf(big, scale);
            if (scale > 0.f) small = fminf(small, scale);
        }
    big = wave_max_f32(big), small = wave_min_scale(small);
    if (lane == 0) top_scale[wave] = big, low_scale[wave] = small;
    if (t0 < t1) load(t0);

    kh8 qh[KT], ql[KT];
    float down;
    {
        const float *q = p.q + (size_t)qc * p.q_stride + (size_t)(kvh * p.group + (valid ? vh : 0)) * HD + 8 * lh;
        float qv[KT][8], top = 0.f, up;
#pragma unroll
        for (int t = 0; t < KT; t++) load8(q + 16 * t, p.q_aligned, qv[t]);
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int e = 0; e < 8; e++) qv[t][e] *= p.qscale, top = fmaxf(top, fabsf(qv[t][e]));
        top = xmax<32>(top);
        row_power(top, up, down);
#pragma unroll
        for (int t = 0; t < KT; t++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float x = qv[t][e] * up;
                qh[t][e] = (_Float16)x;
                ql[t][e] = (_Float16)(x - (float)qh[t][e]);
            }
    }
    kf16 o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) o[d][r] = 0.f;
    float m = -INFINITY, l = 0.f;
    if (t0 < t1) put(t0);
    __syncthreads();
    const bool rows_here = wave * 32 < (qlast - q0 + 1) * p.group;  // else the wavefront only fills LDS
    big = uniform(fmaxf(fmaxf(top_scale[0], top_scale[1]), fmaxf(top_scale[2], top_scale[3])));
    small = uniform(fminf(fminf(low_scale[0], low_scale[1]), fminf(low_scale[2], low_scale[3])));
    const int krow = (l32 & 0x13) | (l32 & 4) << 1 | (l32 & 8) >> 1;

    // a tile's scores, in units of its blocks' K scales times down
    auto scores = [&](int t, kf16 (&s)[2]) {
        const char *ks = lds + (t & 1) * BUF + krow * KST + 16 * lh;
#pragma unroll
        for (int pt = 0; pt < 2; pt++) {
#pragma unroll
            for (int r = 0; r < 16; r++) s[pt][r] = 0.f;
#pragma unroll
            for (int k = 0; k < KT; k++) {
                const kh8 a = *reinterpret_cast<const kh8 *>(ks + pt * 32 * KST + 32 * k);
                s[pt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, qh[k], s[pt], 0, 0, 0);
                s[pt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ql[k], s[pt], 0, 0, 0);
            }
        }
    };
    // those out of this row's sight -infinity; which are in sight
    auto mask = [&](int t, kf16 (&s)[2]) {
        uint32_t keep = 0;
#pragma unroll
        for (int pt = 0; pt < 2; pt++)
#pragma unroll
            for (int r = 0; r < 16; r++) {
                const uint32_t at = 64 * (uint32_t)t + 32 * pt + 16 * (r >> 3) + 8 * lh + (r & 7);
                const bool in = at >= qlo && at <= qpos;
                keep |= (uint32_t)in << (16 * pt + r);
                if (!in) s[pt][r] = -INFINITY;
            }
        return keep;
    };
    // a block's weights' pieces, and their sum
    auto weigh = [&](const kf16 &w, kh8 (&ph)[2], kh8 (&pl)[2]) {
        float sum = 0.f;
        uint32_t hi[8], lo[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const float a = w[2 * i], b = w[2 * i + 1];
            sum += a + b;
            pieces(a, b, hi[i], lo[i]);
        }
#pragma unroll
        for (int k = 0; k < 2; k++) {
            ph[k] = __builtin_bit_cast(kh8, uint4{hi[4 * k], hi[4 * k + 1], hi[4 * k + 2], hi[4 * k + 3]});
            pl[k] = __builtin_bit_cast(kh8, uint4{lo[4 * k], lo[4 * k + 1], lo[4 * k + 2], lo[4 * k + 3]});
        }
        return sum;
    };
    const bool apart = __builtin_amdgcn_readfirstlane(far_apart(big, small));
    const float weight_unit = apart ? 1.f : kWeight;  // of the outputs' weights
    if (apart) {
        big = far_unit(big);
#pragma unroll 1
        for (int t = t0; t < t1; t++) {
            const uint32_t ba = 2 * (uint32_t)t, bb = min(ba + 1, last_block);
            if (t + 1 < t1) load(t + 1);
            if (rows_here) {
                const char *vs = lds + (t & 1) * BUF + 64 * KST + l32 * VST + 16 * lh;
                kf16 s[2];
                scores(t, s);
                const uint32_t keep = mask(t, s);
#pragma unroll
                for (int pt = 0; pt < 2; pt++) {
                    const float f = p.c.ks[head0 + (pt ? bb : ba)] * down, vscale = p.c.vs[head0 + (pt ? bb : ba)] / big;
                    float top = s[pt][0], block_max, was;
#pragma unroll
                    for (int r = 1; r < 16; r++) top = fmaxf(top, s[pt][r]);
                    const float share = take_block(xmax<32>(top), f, block_max, m, was), out_share = share * (1.f / kWeight);
#pragma unroll
                    for (int r = 0; r < 16; r++) {
                        s[pt][r] = __builtin_amdgcn_exp2f(fmaf(s[pt][r], f, -block_max));
                        if (!(keep >> (16 * pt + r) & 1u)) s[pt][r] = 0.f;
                    }
                    kh8 ph[2], pl[2];
                    const float sum = weigh(s[pt], ph, pl);
                    l = fmaf(l, was, sum == 0.f ? 0.f : sum * fmaxf(share, 0.f));
#pragma unroll
                    for (int d = 0; d < DT; d++) {
                        kf16 b;
#pragma unroll
                        for (int r = 0; r < 16; r++) b[r] = 0.f;
#pragma unroll
                        for (int k = 0; k < 2; k++) {
                            const kh8 a = *reinterpret_cast<const kh8 *>(vs + d * 32 * VST + pt * 64 + 32 * k);
                            b = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ph[k], b, 0, 0, 0);
                            b = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pl[k], b, 0, 0, 0);
                        }
#pragma unroll
                        for (int r = 0; r < 16; r++) o[d][r] = share < 0.f ? o[d][r] * was : fmaf(b[r] * out_share, vscale, o[d][r] * was);
                    }
                }
            }
            if (t + 1 < t1) put(t + 1);
            __syncthreads();
        }
    }
    for (int t = apart ? t1 : t0; t < t1; t++) {
        const uint32_t ba = 2 * (uint32_t)t, bb = min(ba + 1, last_block);
        // (a block ahead of every row's window holds any bytes: its scale counts as 0)
        const float kscale[2] = {ba < first_block ? 0.f : p.c.ks[head0 + ba], p.c.ks[head0 + bb]}, vscale[2] = {p.c.vs[head0 + ba], p.c.vs[head0 + bb]};
        if (t + 1 < t1) load(t + 1);
        __builtin_amdgcn_sched_barrier(0);
        if (rows_here) {
            const char *vs = lds + (t & 1) * BUF + 64 * KST + l32 * VST + 16 * lh;
            kf16 s[2];
            scores(t, s);
            const bool edge = 64 * (uint32_t)t + 63 > wave_first || 64 * (uint32_t)t < wave_lo;
            uint32_t keep = 0xFFFFFFFFu;
            if (edge) keep = mask(t, s);
            float f[2], lv[2], inv[2], mx = -INFINITY;
#pragma unroll
            for (int pt = 0; pt < 2; pt++) {
                f[pt] = kscale[pt] * down;
                share_of(vscale[pt], big, lv[pt], inv[pt]);
                float a = s[pt][0];
#pragma unroll
                for (int r = 1; r < 16; r++) a = fmaxf(a, s[pt][r]);
                mx = fmaxf(mx, fmaf(a, f[pt], lv[pt]));
            }
            mx = xmax<32>(mx);
            if (__any(mx > m)) {
                const float mn = fmaxf(m, mx), al = __builtin_amdgcn_exp2f(m - finite(mn));
                m = mn;
                l *= al;
#pragma unroll
                for (int d = 0; d < DT; d++)
#pragma unroll
                    for (int r = 0; r < 16; r++) o[d][r] *= al;
            }
            const float mf = finite(m);
#pragma unroll
            for (int pt = 0; pt < 2; pt++) {
                const float c = lv[pt] - mf;
#pragma unroll
                for (int r = 0; r < 16; r++) s[pt][r] = __builtin_amdgcn_exp2f(fmaf(s[pt][r], f[pt], c));
                if (edge)
#pragma unroll
                    for (int r = 0; r < 16; r++)
                        if (!(keep >> (16 * pt + r) & 1u)) s[pt][r] = 0.f;
                kh8 ph[2], pl[2];
                const float sum = weigh(s[pt], ph, pl);
                // (a row with none of the block in sight takes nothing from it, whatever its scale)
                l += sum == 0.f ? 0.f : sum * inv[pt];
#pragma unroll
                for (int k = 0; k < 2; k++)
#pragma unroll
                    for (int d = 0; d < DT; d++) {
                        const kh8 a = *reinterpret_cast<const kh8 *>(vs + d * 32 * VST + pt * 64 + 32 * k);
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ph[k], o[d], 0, 0, 0);
                        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pl[k], o[d], 0, 0, 0);
                    }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (t + 1 < t1) put(t + 1);
        __syncthreads();
    }
    l = xsum<32>(l);
    if (!valid) return;
    // a split's outputs are those of its own positions (0 where it has none in sight)
    const float inv = p.splits > 1 && m == -INFINITY && l == 0.f ? 0.f : 1.f / (l * weight_unit);
    const size_t row = (size_t)qi * p.heads + head, at = (size_t)z * p.queries * p.heads + row;
    float *dst = (p.splits > 1 ? p.part + at * HD : p.out + row * HD) + 4 * lh;
#pragma unroll
    for (int d = 0; d < DT; d++)
#pragma unroll
        for (int g = 0; g < 4; g++)
            *reinterpret_cast<float4 *>(dst + 32 * d + 8 * g) =
                make_float4(o[d][4 * g] * inv * big, o[d][4 * g + 1] * inv * big, o[d][4 * g + 2] * inv * big, o[d][4 * g + 3] * inv * big);
    if (p.splits > 1 && lh == 0) *reinterpret_cast<float2 *>(p.part_ml + 2 * at) = make_float2(m, l);
}

// The splits' partial results of a row joined in their order, a workgroup per row: the splits' maxima and
// sums a thread each, and a float4 of every N-th split, eight of them under way at once.
template <int HD> __global__ void __launch_bounds__(256) kv8_join_kernel(const float *__restrict__ part, const float2 *__restrict__ ml,
                                                                       float *__restrict__ out, size_t rows, int splits) {
    constexpr int C = HD / 4, N = 256 / C, Z = 8;  // float4s of a row; splits side by side
    __shared__ Wide4 acc[N][C];
    __shared__ float weight[kMaxSplits], tops[4], sums[4];
    const size_t row = blockIdx.x;
    const int tid = threadIdx.x, c = tid % C, n = tid / C;
    const float2 own = ml[(size_t)min(tid, splits - 1) * rows + row];
    float4 v[Z];
    auto load = [&](int from) {
#pragma unroll
        for (int i = 0; i < Z; i++)
            v[i] = *reinterpret_cast<const float4 *>(part + ((size_t)min(from + n + N * i, splits - 1) * rows + row) * HD + 4 * c);
    };
    load(0);
    float m = wave_max_f32(own.x);
    if ((tid & 63) == 0) tops[tid >> 6] = m;
    __syncthreads();
    m = finite(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])));
    float w = tid < splits ? __builtin_amdgcn_exp2f(own.x - m) * own.y : 0.f;
    weight[tid] = w;
    for (int d = 1; d < 64; d <<= 1) w += __shfl_xor(w, d);
    if ((tid & 63) == 0) sums[tid >> 6] = w;
    __syncthreads();
    w = (sums[0] + sums[1]) + (sums[2] + sums[3]);
    Wide4 a = {};
    for (int from = 0; from < splits; from += N * Z) {
        if (from) load(from);
#pragma unroll
        for (int i = 0; i < Z; i++)
            if (from + n + N * i < splits) a.add(weight[from + n + N * i], v[i]);
    }
    if (n < N) acc[n][c] = a;
    __syncthreads();
    if (n) return;
    for (int k = 1; k < N; k++) {
        const Wide4 o = acc[k][c];
        a.x += o.x, a.y += o.y, a.z += o.z, a.w += o.w;
    }
    *reinterpret_cast<float4 *>(out + row * HD + 4 * c) = a.over(1.f / w);
}

// The same for many rows: a thread takes four dims of a row through the splits, four of them under way.
template <int HD> __global__ void __launch_bounds__(256) kv8_join_rows_kernel(const float *__restrict__ part, const float2 *__restrict__ ml,
                                                                            float *__restrict__ out, size_t rows, int splits) {
    constexpr int C = HD / 4, Z = 4;
    const size_t u = (size_t)blockIdx.x * 256 + threadIdx.x, row = u / C;
    const int d = 4 * (int)(u % C);
    if (row >= rows) return;
    float m = -INFINITY, l = 0.f;
    Wide4 a = {};
    for (int z = 0; z < splits; z += Z) {
        float2 w[Z];
        float4 v[Z];
        float top = m;
#pragma unroll
        for (int i = 0; i < Z; i++) {
            const size_t at = (size_t)min(z + i, splits - 1) * rows + row;
            w[i] = ml[at];
            v[i] = *reinterpret_cast<const float4 *>(part + at * HD + d);
        }
#pragma unroll
        for (int i = 0; i < Z; i++) top = fmaxf(top, w[i].x);
        const float mf = finite(top), al = __builtin_amdgcn_exp2f(m - mf);
        m = top;
        a.shrink(al), l *= al;
#pragma unroll
        for (int i = 0; i < Z; i++) {
            const float f = z + i < splits ? __builtin_amdgcn_exp2f(w[i].x - mf) * w[i].y : 0.f;
            if (z + i < splits) a.add(f, v[i]);
            l += f;
        }
    }
    *reinterpret_cast<float4 *>(out + row * HD + d) = a.over(1.f / l);
}

}  // namespace

hipError_t launch_kv8_attention(const Kv8Attn &a, int cus, hipStream_t s) {
    Kv8Params p{};
    p.c = a.c, p.q = a.q, p.q_stride = a.q_stride, p.out = a.out;
    p.position = a.position, p.queries = a.queries, p.window = a.window;
    p.heads = a.heads, p.group = a.heads / a.c.nkv, p.qscale = a.qscale;
    p.per_group = (65536u + p.group - 1) / p.group;
    p.q_aligned = (uintptr_t)a.q % 16 == 0 && a.q_stride % 4 == 0;
    const uint64_t rows = (uint64_t)a.queries * p.group;  // of a kv head
    // (9 queries x 4 heads over 16k positions: 25.8 us here, 27.3 by the other kernel; 16 x 4: 33.1 and 30.3.
    // Of head size 256 more than 16 rows don't fit a wavefront's registers.)
    const bool many = rows > (a.c.hd <= 128 ? 48 : 16);
    const int nr = rows <= 8 ? 8 : (int)(rows + 15) / 16 * 16, qn = 128 / p.group;
    const uint64_t wgs = p.c.nkv * (many ? (a.queries + (uint64_t)qn - 1) / qn : 1);
    if (wgs > 0x7FFFFFFFu) return hipErrorInvalidValue;
    const uint64_t total = (uint64_t)a.queries * a.heads;
    uint64_t splits = 1;
    if (!many) {
        // one workgroup a CU, a block for each of its wavefronts at least (131071 positions, 8 kv heads: 32 splits
        // 52.1 us, 48 57.9, 64 52.5; 4113 positions: 16 splits 10.3, 32 9.5, 64 10.2)
        const uint32_t seen = a.window && a.window <= a.position ? a.window : a.position + 1;  // of the first query
        splits = std::min({(uint64_t)cus / wgs, (uint64_t)seen / (4 * kKv8Block), (uint64_t)kMaxSplits});
    } else {
        // The split count whose estimated time is least, in us: the longest workgroup's tiles (2.2 of head size 128,
        // 3.4 where two workgroups share a CU), in rounds of as many workgroups as are resident, and the join's launch
        // and traffic.  (Longest range: the splits of a workgroup with a shorter one are shorter, or empty.  300 queries
        // of 32 heads, 8 of them kv heads, after 4000: 1 split 158 us, 3 70.6, 6 62.9, 16 77.2; taken: 6.)
        const uint64_t last = (uint64_t)a.position + a.queries, range = a.window ? std::min(last, (uint64_t)a.window + qn) : last;
        const double tiles = (double)(range / 64 + 1), size = 0.25 + 0.75 * a.c.hd / 128;
        const uint64_t per_cu = a.c.hd <= 128 ? 2 : 1;
        double best = 1e300;
        for (uint64_t n = 1; n <= (uint64_t)kMaxSplits && n <= (uint64_t)tiles; n++) {
            const double tile = size * (wgs * n > (uint64_t)cus && per_cu == 2 ? 3.4 : 2.2);
            const double t = (double)((wgs * n + per_cu * cus - 1) / (per_cu * cus)) * std::ceil(tiles / n) * tile +
                             (n > 1 ? 2.5 + n * (double)total * a.c.hd * 8 / 4e6 : 0.0);
            if (t < best * 0.98) best = t, splits = n;
        }
    }
    while (splits > 1 && splits * total * (a.c.hd + 2) > a.part_floats) splits--;
    p.splits = splits > 1 ? (int)splits : 1;
    p.part = a.part, p.part_ml = a.part + (size_t)p.splits * total * a.c.hd;
    const dim3 grid((unsigned)wgs, (unsigned)p.splits);
    auto go = [&](auto h) {
        constexpr int HD = decltype(h)::value;
        if (many) hipLaunchKernelGGL(kv8_many_kernel<HD>, grid, dim3(256), 0, s, p);
        else if (nr == 8) hipLaunchKernelGGL((kv8_few_kernel<HD, 8>), grid, dim3(256), 0, s, p);
        else if (nr == 16) hipLaunchKernelGGL((kv8_few_kernel<HD, 16>), grid, dim3(256), 0, s, p);
        else if constexpr (HD <= 128) {
            if (nr == 32) hipLaunchKernelGGL((kv8_few_kernel<HD, 32>), grid, dim3(256), 0, s, p);
            else hipLaunchKernelGGL((kv8_few_kernel<HD, 48>), grid, dim3(256), 0, s, p);
        }
        if (p.splits == 1) return;
        const float2 *ml = (const float2 *)p.part_ml;
        if (total < 1024)  // (860 queries x 6 heads, 5 splits: 23.3 us a pass with a workgroup per row, 17.8 with a thread per four dims)
            hipLaunchKernelGGL(kv8_join_kernel<HD>, dim3((unsigned)total), dim3(256), 0, s, p.part, ml, p.out, (size_t)total, p.splits);
        else
            hipLaunchKernelGGL(kv8_join_rows_kernel<HD>, dim3((unsigned)((total * (HD / 4) + 255) / 256)), dim3(256), 0, s, p.part, ml,
                               p.out, (size_t)total, p.splits);
    };
    switch (a.c.hd) {
    case 64: go(std::integral_constant<int, 64>{}); break;
    case 96: go(std::integral_constant<int, 96>{}); break;
    case 128: go(std::integral_constant<int, 128>{}); break;
    case 256: go(std::integral_constant<int, 256>{}); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace zh

// zh_kv4_attn.hip -- attention of a batch of sequences over the paged cache held in 4 bits.
//
// o = sum_t w_t v_t / sum_t w_t, w_t = 2^(s_t - max), s_t = qscale q.k_t, in one pass with the running
// maximum and sum.  A code times its power-of-two scale is exact in bf16, whose exponents are binary32's, so K
// and V enter the matrix cores exactly and no scale is left over to weigh scores or outputs by.  A query and a
// weight enter as three bf16 pieces, cut off by truncation, whose sum they are to the bit.  Products accumulate in
// binary32, maximum and sum are binary32.
#include "zh_serving.h"

namespace zh {

namespace {

typedef unsigned long long u64;
typedef __bf16 fb2 __attribute__((ext_vector_type(2)));
typedef __bf16 fb8 __attribute__((ext_vector_type(8)));
typedef float ff4 __attribute__((ext_vector_type(4)));

constexpr int kBlock = 32;  // positions of a product

struct Kv4Params {
    Kv4Layer c;
    Batch b;
    const float *q;
    size_t q_stride;
    float *out;
    int heads, group, q_aligned;
    uint32_t window;
    float qscale, qsign;
};

// A sequence's tile of columns (its rows' heads of one kv head, row by row) by the tile's number in the batch;
// count 0: none.  Every lane of a wavefront takes part.
struct Tile {
    Sequence q;
    uint32_t first, count;  // columns
};
template <int COLUMNS> __device__ __forceinline__ Tile tile_of(const Batch &b, uint32_t group, uint32_t number) {
    Tile t{};
    const uint32_t lane = threadIdx.x & 63;
    uint32_t before = 0;
    for (uint32_t from = 0; from < b.sequences; from += 64) {
        uint32_t n = 0;
        if (from + lane < b.sequences) n = (sequence_of(b, from + lane).rows * group + COLUMNS - 1) / COLUMNS;
        uint32_t sum = n;  // of this lane and those before it
        for (int d = 1; d < 64; d <<= 1) {
            const uint32_t o = (uint32_t)__shfl_up((int)sum, d);
            if ((int)lane >= d) sum += o;
        }
        const u64 past = __ballot(before + sum > number);
        if (past) {
            const int at = __ffsll(past) - 1;
            t.q = sequence_of(b, from + at);
            t.first = (number - before - (uint32_t)__shfl((int)(sum - n), at)) * COLUMNS;
            const uint32_t all = t.q.rows * group;  // (tables that don't ascend may pass 32 bits in the sums)
            t.count = t.first < all ? min((uint32_t)COLUMNS, all - t.first) : 0u;
            return t;
        }
        before += (uint32_t)__shfl((int)sum, 63);
    }
    return t;
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
__device__ __forceinline__ float scale_of(uint32_t w, int byte) { return __uint_as_float((w >> (8 * byte) & 255u) << 23); }

__device__ __forceinline__ float finite(float v) { return v == -INFINITY ? 0.f : v; }

// A lane's part of 32 positions: lane (i, g) holds K rows 8 (i / 4) + 4 pt + i % 4 of both halves pt (its words g of
// every 32 dims), and V's dims 32 t + i and 32 t + 16 + i of positions 8 g .. 8 g + 7.
template <int HD> struct Lane4 {
    static constexpr int G = HD / 32;
    uint32_t k[2][G], v[2 * G];
    uint8_t ks[2][G];
    uint32_t vs[2 * G];
    __device__ __forceinline__ void load(const Kv4Layer &c, uint32_t page, int head, int half) {
        const int i = threadIdx.x & 15, g = threadIdx.x >> 4 & 3;
        const size_t codes = c.codes(page, head), scales = c.scales(page, head);
#pragma unroll
        for (int pt = 0; pt < 2; pt++) {
            const int pos = kBlock * half + 8 * (i >> 2) + 4 * pt + (i & 3);
            __builtin_memcpy(k[pt], c.kc + codes + (size_t)pos * (HD / 2) + g * 4 * G, 4 * G);
            __builtin_memcpy(ks[pt], c.ks + scales + (size_t)pos * G, G);
        }
        __builtin_memcpy(v, c.vc + codes + (size_t)half * (16 * HD) + (g * 16 + i) * 8 * G, 8 * G);
        __builtin_memcpy(vs, c.vs + scales + (size_t)(kBlock * half + 8 * g) * G, 8 * G);
    }
};

// One wavefront's columns: their queries, running maxima and sums, and outputs.  Scores S^T[position][column] = K Q^T on
// 16x16x32 products, outputs O^T[dim][column] = V^T P^T: what a lane gets of S^T, positions 8 g .. 8 g + 7 of column i,
// is what it gives of P^T.
template <int HD, int CT> struct Columns {
    static constexpr int G = HD / 32, DT = HD / 16;
    fb8 q[CT][G][3];
    ff4 o[CT][DT];
    float m[CT], l[CT];
    int lo[CT], hi[CT];  // the positions that a column sees, both included

    __device__ __forceinline__ void begin(const Kv4Params &p, const Tile &t, uint32_t first, int head) {
        const int i = threadIdx.x & 15, g = threadIdx.x >> 4 & 3;
#pragma unroll
        for (int c = 0; c < CT; c++) {
            const uint32_t column = min(first + 16 * c + i, t.first + t.count - 1), row = column / p.group;
            const float *src = p.q + (size_t)(t.q.row0 + row) * p.q_stride + (size_t)(head * p.group + (int)(column - row * p.group)) * HD;
            hi[c] = t.q.first + (int)row;
            lo[c] = p.window && (int64_t)hi[c] - p.window >= 0 ? hi[c] + 1 - (int)p.window : 0;
            hi[c] = min(hi[c], (int)p.b.cap - 1);
#pragma unroll
            for (int k = 0; k < G; k++) {
                float v[8];
                const float *from = src + 32 * k + 8 * g;
                if (p.q_aligned) {
                    *reinterpret_cast<float4 *>(v) = *reinterpret_cast<const float4 *>(from);
                    *reinterpret_cast<float4 *>(v + 4) = *reinterpret_cast<const float4 *>(from + 4);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) v[e] = from[e];
                }
#pragma unroll
                for (int e = 0; e < 8; e++) v[e] *= p.qsign;
                pieces(v, q[c][k]);
            }
            m[c] = -INFINITY, l[c] = 0.f;
#pragma unroll
            for (int d = 0; d < DT; d++) o[c][d] = ff4{0.f, 0.f, 0.f, 0.f};
        }
    }

    // 32 positions from `at` on; of these only first .. last are any column's to see
    __device__ __forceinline__ void take(const Kv4Params &p, const Lane4<HD> &x, int at, int first, int last) {
        const int g = threadIdx.x >> 4 & 3;
        const bool edge = at < first || at + kBlock - 1 > last;
        ff4 s[CT][2];
#pragma unroll
        for (int pt = 0; pt < 2; pt++) {
#pragma unroll
            for (int c = 0; c < CT; c++) s[c][pt] = ff4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = 0; t < G; t++) {
                const float scale = __uint_as_float((uint32_t)x.ks[pt][t] << 23);
                uint32_t w[4] = {widen<0>(x.k[pt][t], scale), widen<1>(x.k[pt][t], scale), widen<2>(x.k[pt][t], scale), widen<3>(x.k[pt][t], scale)};
                fb8 a;
                __builtin_memcpy(&a, w, 16);
#pragma unroll
                for (int c = 0; c < CT; c++)
#pragma unroll
                    for (int k = 0; k < 3; k++) s[c][pt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, q[c][t][k], s[c][pt], 0, 0, 0);
            }
        }
        fb8 w[CT][3];
#pragma unroll
        for (int c = 0; c < CT; c++) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int pos = at + 8 * g + e;
                v[e] = pos >= lo[c] && pos <= hi[c] && pos >= first && pos <= last ? s[c][e >> 2][e & 3] : -INFINITY;
            }
            float top = v[0];
#pragma unroll
            for (int e = 1; e < 8; e++) top = fmaxf(top, v[e]);
            top = xmax<32>(xmax<16>(top)) * p.qscale;
            const float next = fmaxf(m[c], top), nf = finite(next), was = __builtin_amdgcn_exp2f(m[c] - nf);
            m[c] = next;
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = __builtin_amdgcn_exp2f(fmaf(v[e], p.qscale, -nf)), sum += v[e];
            l[c] = fmaf(l[c], was, sum);
#pragma unroll
            for (int d = 0; d < DT; d++) o[c][d] *= was;
            pieces(v, w[c]);
        }
#pragma unroll
        for (int t = 0; t < G; t++) {
            uint32_t a[2][4];
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                uint32_t y[2];
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const int n = (j + e) * G + t;  // byte of this position's dims
                    const bool out = edge && (at + 8 * g + j + e < first || at + 8 * g + j + e > last);
                    const float scale = scale_of(x.vs[n >> 2], n & 3);
                    const uint32_t word = x.v[n >> 2];
                    const uint32_t u = (n & 3) == 0 ? widen<0>(word, scale) : (n & 3) == 1 ? widen<1>(word, scale) : (n & 3) == 2 ? widen<2>(word, scale) : widen<3>(word, scale);
                    y[e] = out ? 0u : u;  // (what was never stored may read as NaN)
                }
                a[0][j / 2] = __builtin_amdgcn_perm(y[1], y[0], 0x05040100u);
                a[1][j / 2] = __builtin_amdgcn_perm(y[1], y[0], 0x07060302u);
            }
#pragma unroll
            for (int h = 0; h < 2; h++) {
                fb8 b;
                __builtin_memcpy(&b, a[h], 16);
#pragma unroll
                for (int c = 0; c < CT; c++)
#pragma unroll
                    for (int k = 0; k < 3; k++) o[c][2 * t + h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, w[c][k], o[c][2 * t + h], 0, 0, 0);
            }
        }
    }
};

// A wavefront takes 16 columns through all of their positions.
template <int HD> __global__ void __launch_bounds__(64) kv4_simple_kernel(Kv4Params p) {
    const int head = blockIdx.x % p.c.nkv, i = threadIdx.x & 15, g = threadIdx.x >> 4;
    const Tile t = tile_of<16>(p.b, (uint32_t)p.group, blockIdx.x / p.c.nkv);
    if (t.count == 0) return;
    Columns<HD, 1> x;
    x.begin(p, t, t.first, head);
    const int row0 = (int)(t.first / p.group), row1 = (int)((t.first + t.count - 1) / p.group);
    const int last = min(t.q.first + row1, (int)p.b.cap - 1);
    const int first = p.window && (int64_t)t.q.first + row0 - p.window >= 0 ? t.q.first + row0 + 1 - (int)p.window : 0;
    for (int at = first / kBlock * kBlock; at <= last; at += kBlock) {
        const uint32_t page = page_of(p.b, t.q.index, (uint32_t)at);
        if (page >= p.b.pool) continue;
        Lane4<HD> y;
        y.load(p.c, page, head, at / kBlock & 1);
        x.take(p, y, at, first, last);
    }
    const float l = xsum<32>(xsum<16>(x.l[0])), inv = l == 0.f ? 0.f : 1.f / l;
    if ((uint32_t)i >= t.count) return;
    const uint32_t column = t.first + i, row = column / p.group;
    float *to = p.out + ((size_t)(t.q.row0 + row) * p.heads + head * p.group + (column - row * p.group)) * HD + 4 * g;
#pragma unroll
    for (int d = 0; d < HD / 16; d++)
        *reinterpret_cast<float4 *>(to + 16 * d) = make_float4(x.o[0][d][0] * inv, x.o[0][d][1] * inv, x.o[0][d][2] * inv, x.o[0][d][3] * inv);
}

}  // namespace

hipError_t launch_kv4_attention(const Kv4Attn &a, int cus, hipStream_t s) {
    Kv4Params p{};
    p.c = a.c, p.b = a.b, p.q = a.q, p.q_stride = a.q_stride, p.out = a.out;
    p.heads = a.heads, p.group = a.heads / a.c.nkv, p.q_aligned = a.q_aligned;
    p.window = a.window, p.qscale = a.qscale, p.qsign = a.qsign;
    const uint64_t wgs = a.c.nkv * ((uint64_t)a.b.rows * p.group / 16 + a.b.sequences);  // at most
    if (wgs > 0x7FFFFFFFu) return hipErrorInvalidValue;
    const dim3 grid((unsigned)wgs);
    switch (a.c.hd) {
    case 64: hipLaunchKernelGGL(kv4_simple_kernel<64>, grid, dim3(64), 0, s, p); break;
    case 96: hipLaunchKernelGGL(kv4_simple_kernel<96>, grid, dim3(64), 0, s, p); break;
    case 128: hipLaunchKernelGGL(kv4_simple_kernel<128>, grid, dim3(64), 0, s, p); break;
    case 256: hipLaunchKernelGGL(kv4_simple_kernel<256>, grid, dim3(64), 0, s, p); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace zh

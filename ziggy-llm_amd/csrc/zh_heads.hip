// zh_heads.hip -- norms of query and key heads with the position rotation in one pass, and keys and values into the
// paged cache of 4 bits on the way.
//
// y = R(p) (x (w + o) / sqrt(mean x^2 + eps)), R(p) turning pair i by p base^(-2 i / rd).  Sums of squares, angles, sines
// and a key's whole way are 64 bits, so that its codes do not hang on binary32's roundings; a query's or an f32 key's
// factors are rounded once and applied in binary32, the normalised value ahead of its weight.
//
// What bounds it: memory where there are many rows (4095 rows of 40 heads of 128: 33.3 us, 5.0 TB/s read and written), the
// chain launch, tables, page, sines, norm where there are few (one row 4.3 us, 32 rows appended 6.4, read back 4.9).  Between
// the two lie prompts' chunks on their way into the cache and back, 3012 rows of four with 32 query and 8 kv heads: appended
// in 32 us for 129 MB by the counters (126.6 have to move), 4.0 TB/s, as every row's bytes wait for its sequence, page and
// sines; read back in 9.3 us for 32 MB, 3.4 TB/s, of which 28.0 have to move: a position's V codes are four bytes of every
// 32, so a row fetches 2.3 times its codes.  A wavefront a row: its sines are shared by all its heads, and there is nothing to
// wait for but its own loads (a workgroup a row, with barriers: 43 to 50 us).
#include "zh_serving.h"

namespace zh {

namespace {

typedef unsigned long long u64;

// the scale byte (its exponent + 127) of 32 values whose largest magnitude has these bits
__device__ __forceinline__ uint32_t scale_byte(uint32_t bits) {
    const uint32_t e = (bits >> 23) + ((bits & 0x7FFFFFu) > 0x600000u ? 1u : 0u);  // 7 2^x is 1.75 2^(x + 2)
    return min(max(e, 33u) - 2u, 219u);
}

// 1 / sqrt(x) to a step or two of 64 bits: the hardware's estimate, and two steps of Newton's
__device__ __forceinline__ double inverse_root(double x) {
    double y = __builtin_amdgcn_rsq(x);
    if (!(x > 0.0 && x < INFINITY)) return y;  // (0: infinity, an infinity: 0)
    y = fma(0.5 * y, fma(-x * y, y, 1.0), y);
    return fma(0.5 * y, fma(-x * y, y, 1.0), y);
}

// A lane's eight values of a head, two vectors: which of them turn with which.
//   SPLIT   a[j] with b[j] (halves, all of the head turning): values 4 u and hd / 2 + 4 u on
//   PAIRS   neighbours, of the same values
//   MIXED   halves of part of the head, neighbours behind: 16-byte loads, but not of whole lines
//   LOOSE   any of these, value by value
enum Layout { SPLIT, PAIRS, MIXED, LOOSE };

constexpr int kAhead = 2;  // heads of a team whose loads are under way ahead of the one at work

struct HeadPlan {
    int units, team;        // lanes of a head: those with values, rounded up to a power of two
    int chunks;             // wavefronts that share a row's heads
    int wave_bytes;         // of LDS
    int streams;            // the output is more than the caches hold
};

// streams: past the caches (4095 rows of 40 heads of 128: 41 us without, 34 with; of parts of lines it costs time)
__device__ __forceinline__ void put(float *to, float4 v, int streams) {
    typedef float f4 __attribute__((ext_vector_type(4)));
    if (streams) __builtin_nontemporal_store(f4{v.x, v.y, v.z, v.w}, reinterpret_cast<f4 *>(to));
    else *reinterpret_cast<float4 *>(to) = v;
}

// A wavefront takes a row's heads (or every chunks-th team of them): its sines and cosines once, a pair a lane, then
// a head a team of lanes.
template <int LAYOUT, bool CACHE> __global__ void __launch_bounds__(256) head_rows_kernel(HeadRows p, HeadPlan plan) {
    extern __shared__ __align__(16) char lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const int team = plan.team, u = lane % team, slot = lane / team;
    const uint32_t unit = blockIdx.x * 4 + wave, r = unit / plan.chunks, chunk = unit - r * plan.chunks;
    if (r >= p.rows) return;
    const int half = p.rotates ? p.rd / 2 : 0, i0 = 4 * u, hp = 64 / team;
    double2 *table = reinterpret_cast<double2 *>(lds + wave * plan.wave_bytes);
    // pair i: halves (i, i + half), neighbours (2 i, 2 i + 1) of interleaved ones and of what does not turn
    auto pair = [&](int j) { return LAYOUT == PAIRS ? 2 * u + (j & 1) + (j >> 1) * (p.hd / 4) : i0 + j; };
    auto turns = [&](int j) { return pair(j) < half; };
    auto split = [&](int j) { return LAYOUT == SPLIT || (LAYOUT != PAIRS && p.style && turns(j)); };
    auto first_of = [&](int j) { return split(j) ? pair(j) : 2 * pair(j); };
    auto second_of = [&](int j) { return split(j) ? pair(j) + half : 2 * pair(j) + 1; };
    auto in = [&](int j) { return u < plan.units && 2 * pair(j) < p.hd; };
    const int d0 = split(0) ? i0 : LAYOUT == PAIRS ? 4 * u : 2 * i0, d1 = split(0) ? i0 + half : LAYOUT == PAIRS ? p.hd / 2 + 4 * u : 2 * i0 + 4;
    const bool some = u < plan.units, whole = some && d1 < p.hd;
    // x[0][j], x[1][j]: pair j
    auto load = [&](const float *src, float (&x)[2][4]) {
        if constexpr (LAYOUT == LOOSE) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                x[0][j] = in(j) ? src[first_of(j)] : 0.f;
                x[1][j] = in(j) ? src[second_of(j)] : 0.f;
            }
        } else {
            float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
            if (some) a = *reinterpret_cast<const float4 *>(src + d0);
            if (whole) b = *reinterpret_cast<const float4 *>(src + d1);
            const bool halves = split(0);
            x[0][0] = a.x, x[1][3] = b.w;
            x[0][1] = halves ? a.y : a.z, x[0][2] = halves ? a.z : b.x, x[0][3] = halves ? a.w : b.z;
            x[1][0] = halves ? b.x : a.y, x[1][1] = halves ? b.y : a.w, x[1][2] = halves ? b.z : b.y;
        }
    };
    auto store = [&](float *dst, const float (&y)[2][4]) {
        if constexpr (LAYOUT == LOOSE) {
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (in(j)) dst[first_of(j)] = y[0][j], dst[second_of(j)] = y[1][j];
        } else {
            const bool halves = split(0);
            const float4 a = make_float4(y[0][0], halves ? y[0][1] : y[1][0], halves ? y[0][2] : y[0][1], halves ? y[0][3] : y[1][1]);
            const float4 b = make_float4(halves ? y[1][0] : y[0][2], halves ? y[1][1] : y[1][2], halves ? y[1][2] : y[0][3], y[1][3]);
            if (some) put(dst + d0, a, plan.streams);
            if (whole) put(dst + d1, b, plan.streams);
        }
    };
    const int f32_heads = p.q_heads + p.k_heads, step = plan.chunks * hp, h0 = (int)chunk * hp + slot;
    const float *row = p.src + r * p.src_stride;
    float x[kAhead + 1][2][4];  // of this head and the next ones
#pragma unroll
    for (int b = 0; b < kAhead; b++)
        if (h0 + b * step < f32_heads) load(row + (size_t)(h0 + b * step) * p.hd, x[b]);
    float wq[2][4], wk[2][4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int d[2] = {first_of(j), second_of(j)};
#pragma unroll
        for (int e = 0; e < 2; e++) {
            wq[e][j] = p.q_norm && in(j) ? p.q_norm[d[e]] + p.weight_offset : 0.f;
            wk[e][j] = p.k_norm && in(j) ? p.k_norm[d[e]] : 0.f;
        }
    }
    double at;
    int pos = 0;
    uint32_t page = 0;
    bool stored = false;
    if constexpr (CACHE) {
        const Sequence q = sequence_of_row(p.b, r);
        pos = q.first + (int)(r - q.row0);
        if (q.rows == 0 || pos < 0) return;
        stored = (uint32_t)pos < p.b.cap;
        if (stored) page = page_of(p.b, q.index, (uint32_t)pos);
        stored = stored && page < p.b.pool;
        at = (double)pos;
    } else {
        at = (double)(p.positions ? p.positions[r] : p.first + r);
    }
    for (int i = lane; i < half; i += 64) {
        const double t = at * p.freq.turns_per_position(i, p.factors);
        double s, c;
        sincospi(2.0 * (t - rint(t)), &s, &c);
        table[i] = make_double2(c * (double)p.magnitude, s * (double)p.magnitude);
    }
    wave_fence();
    double cs[4], sn[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const double2 v = turns(j) ? table[pair(j)] : make_double2(1.0, 0.0);
        cs[j] = v.x, sn[j] = v.y;
    }
    auto norm_of = [&](const float (&v)[2][4]) {
        double ss = 0.0;
#pragma unroll
        for (int j = 0; j < 4; j++) ss = fma((double)v[0][j], (double)v[0][j], fma((double)v[1][j], (double)v[1][j], ss));
        return inverse_root(team_sum(ss, team) / p.hd + (double)p.eps);
    };
    auto turn = [&](int h, const float (&v)[2][4]) {
        const bool key = h >= p.q_heads, normed = key ? p.k_norm : p.q_norm;
        // The factor 1 / rms as a power of two and a binary32 number of .5 to 1: where all values are denormal, or next to the
        // largest, it is itself no binary32 number, nor is its product with a weight.  What it makes of a value is.
        const double inv = normed ? norm_of(v) : 1.0;
        const int power = __builtin_amdgcn_frexp_exp(inv);
        const float part = (float)__builtin_amdgcn_frexp_mant(inv);
        float y[2][4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float a = v[0][j], c = v[1][j];
            if (normed) {
                a = ldexpf(a, power) * part * (key ? wk[0][j] + p.weight_offset : wq[0][j]);
                c = ldexpf(c, power) * part * (key ? wk[1][j] + p.weight_offset : wq[1][j]);
            }
            const float fc = (float)cs[j], fs = (float)sn[j];
            const bool t = LAYOUT == SPLIT || turns(j);
            y[0][j] = t ? a * fc - c * fs : a, y[1][j] = t ? a * fs + c * fc : c;
        }
        store(p.dst + r * p.dst_stride + (size_t)h * p.hd, y);
    };
    for (int h = h0; h < f32_heads; h += (kAhead + 1) * step) {
#pragma unroll
        for (int b = 0; b <= kAhead; b++) {
            const int now = h + b * step, next = now + kAhead * step;
            if (next < f32_heads) load(row + (size_t)next * p.hd, x[(b + kAhead) % (kAhead + 1)]);
            if (now < f32_heads) turn(now, x[b]);
        }
    }
    if constexpr (CACHE) {
        if (!stored) return;
        const int g_n = p.hd / 32, c = u, g = c & 3, t = c >> 2, at64 = pos % kPage;
        const bool holds = c < 4 * g_n;
        float *key_at = reinterpret_cast<float *>(table + half) + lane / team * 8 * team, *value_at = key_at + 512;
        float *scale_at = key_at - lane / team * 8 * team + 1024 + lane / team * team;
        // keys and values behind the other heads, so that few rows' are spread over wavefronts too
        for (int h = (h0 + step - f32_heads % step) % step; h < p.c.nkv; h += step) {
            load(p.k + r * p.src_stride + (size_t)h * p.hd, x[0]);
            const float *vs = p.v + r * p.src_stride + (size_t)h * p.hd;
            float k8[8] = {}, v8[8] = {};
            if (holds) {
                if constexpr (LAYOUT != LOOSE) {
                    *reinterpret_cast<float4 *>(v8) = *reinterpret_cast<const float4 *>(vs + 8 * c);
                    *reinterpret_cast<float4 *>(v8 + 4) = *reinterpret_cast<const float4 *>(vs + 8 * c + 4);
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++) v8[e] = vs[8 * c + e];
                }
            }
            const double inv = p.k_norm ? norm_of(x[0]) : 1.0;
#pragma unroll
            for (int j = 0; j < 4; j++) {
                double a = (double)x[0][0][j], b = (double)x[0][1][j];
                if (p.k_norm) {
                    a *= ((double)wk[0][j] + (double)p.weight_offset) * inv;
                    b *= ((double)wk[1][j] + (double)p.weight_offset) * inv;
                }
                if (turns(j)) {
                    const double y = a * cs[j] - b * sn[j];
                    b = a * sn[j] + b * cs[j], a = y;
                }
                if (in(j)) key_at[first_of(j)] = (float)a, key_at[second_of(j)] = (float)b;
            }
            if (holds) {
                *reinterpret_cast<float4 *>(value_at + 8 * c) = make_float4(v8[0], v8[1], v8[2], v8[3]);
                *reinterpret_cast<float4 *>(value_at + 8 * c + 4) = make_float4(v8[4], v8[5], v8[6], v8[7]);
            }
            wave_fence();
            uint32_t kmax = 0, vmax = 0;
            if (holds) {
                *reinterpret_cast<float4 *>(k8) = *reinterpret_cast<const float4 *>(key_at + 8 * c);
                *reinterpret_cast<float4 *>(k8 + 4) = *reinterpret_cast<const float4 *>(key_at + 8 * c + 4);
#pragma unroll
                for (int e = 0; e < 8; e++)
                    kmax = max(kmax, __float_as_uint(k8[e]) & 0x7FFFFFFFu), vmax = max(vmax, __float_as_uint(v8[e]) & 0x7FFFFFFFu);
            }
            kmax = max(kmax, moved<0xB1, 0xF>(kmax)), vmax = max(vmax, moved<0xB1, 0xF>(vmax));
            kmax = max(kmax, moved<0x4E, 0xF>(kmax)), vmax = max(vmax, moved<0x4E, 0xF>(vmax));
            const u64 lanes = team == 64 ? ~0ull : ((1ull << team) - 1) << (slot * team);
            const bool marked = __ballot(max(kmax, vmax) >= 0x7F800000u) & lanes;
            const uint32_t kb = scale_byte(kmax), vb = marked ? 127u : scale_byte(vmax);
            const float ks = __uint_as_float(kb << 23);
            uint32_t w = 0;
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, k8[0], k8[1], ks, 0);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, k8[2], k8[3], ks, 1);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, k8[4], k8[5], ks, 2);
            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, k8[6], k8[7], ks, 3);
            const size_t codes = p.c.codes(page, h), scales = p.c.scales(page, h) + (size_t)at64 * g_n;
            if (holds) {
                *reinterpret_cast<uint32_t *>(p.c.kc + codes + (size_t)at64 * (p.hd / 2) + (g * g_n + t) * 4) = marked ? 0u : w;
                if (g == 0) {
                    p.c.ks[scales + t] = (uint8_t)(marked ? 255u : kb);
                    p.c.vs[scales + t] = (uint8_t)vb;
                    scale_at[t] = __uint_as_float(vb << 23);
                }
            }
            wave_fence();
            if (holds) {
                // four bytes of the position's, dim by dim: of one dim where it has that many
                uint8_t *to = p.c.vc + codes + (size_t)(at64 / 8) * (128 * g_n) + at64 % 8 * g_n;
                uint32_t bytes[4];
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const int n4 = 4 * c + e, d = n4 / g_n, tt = n4 % g_n;
                    const uint32_t two = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, value_at[32 * tt + d], value_at[32 * tt + 16 + d], scale_at[tt], 0);
                    bytes[e] = marked ? 0u : two & 255u;
                }
                if (g_n % 4 == 0) {
                    const int d = 4 * c / g_n, tt = 4 * c % g_n;
                    *reinterpret_cast<uint32_t *>(to + d * 8 * g_n + tt) = bytes[0] | bytes[1] << 8 | bytes[2] << 16 | bytes[3] << 24;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int n4 = 4 * c + e;
                        to[n4 / g_n * 8 * g_n + n4 % g_n] = (uint8_t)bytes[e];
                    }
                }
            }
            wave_fence();
        }
    }
}

// what a code (bits 3 .. 0) stands for
__device__ __forceinline__ float value_of(uint32_t code) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 v = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(code, 1.f, 0);
    return v[0];
}

// A wavefront reads a row back, 1024 / HD heads at a time: a lane eight dims of a key, then the dims 32 t + d and
// 32 t + 16 + d of a value, which go through LDS to be written in order.
template <int HD> __global__ void __launch_bounds__(256) kv4_load_kernel(Kv4Layer c, Batch b, float *k, float *v) {
    constexpr int G = HD / 32, EACH = HD / 8, SOME = 1024 / HD, HELD = HD + 4;
    __shared__ __align__(16) float lds[4][SOME * HELD];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const uint32_t r = blockIdx.x * 4 + wave;
    if (r >= b.rows) return;
    const Sequence q = sequence_of_row(b, r);
    const int pos = q.first + (int)(r - q.row0);
    if (q.rows == 0 || pos < 0 || (uint32_t)pos >= b.cap) return;
    const uint32_t page = page_of(b, q.index, (uint32_t)pos);
    if (page >= b.pool) return;
    const int at64 = pos % kPage;
    const float nan = __uint_as_float(0x7FC00000u);
    float *held = lds[wave];
    for (int from = 0; from < c.nkv; from += SOME) {
        const int heads = min(SOME, c.nkv - from);
        const size_t to = ((size_t)r * c.nkv + from) * HD;
#pragma unroll
        for (int e = 0; e < SOME * 16; e += 64) {
            const int i = e + lane, head = i / 16, d = i % 16;
            if (i >= heads * 16) break;
            uint8_t bytes[G], ks[G], vs[G];
            __builtin_memcpy(bytes, c.vc + c.codes(page, from + head) + (size_t)(at64 / 8) * (128 * G) + d * 8 * G + at64 % 8 * G, G);
            __builtin_memcpy(ks, c.ks + c.scales(page, from + head) + (size_t)at64 * G, G);
            __builtin_memcpy(vs, c.vs + c.scales(page, from + head) + (size_t)at64 * G, G);
#pragma unroll
            for (int t = 0; t < G; t++) {
                const float scale = ks[t] == 255u ? nan : __uint_as_float((uint32_t)vs[t] << 23);
                held[head * HELD + 32 * t + d] = value_of(bytes[t]) * scale;
                held[head * HELD + 32 * t + 16 + d] = value_of(bytes[t] >> 4) * scale;
            }
        }
#pragma unroll
        for (int e = 0; e < SOME * EACH; e += 64) {
            const int i = e + lane, head = from + i / EACH, n = i % EACH, t = n / 4, g = n % 4;
            if (i >= heads * EACH) break;
            const uint32_t w = *reinterpret_cast<const uint32_t *>(c.kc + c.codes(page, head) + (size_t)at64 * (HD / 2) + (g * G + t) * 4);
            const uint32_t byte = c.ks[c.scales(page, head) + (size_t)at64 * G + t];
            const float scale = byte == 255u ? nan : __uint_as_float(byte << 23);
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] = value_of(w >> 4 * j) * scale;
            *reinterpret_cast<float4 *>(k + to + 8 * i) = make_float4(x[0], x[1], x[2], x[3]);
            *reinterpret_cast<float4 *>(k + to + 8 * i + 4) = make_float4(x[4], x[5], x[6], x[7]);
        }
        wave_fence();
        for (int i = lane; i < heads * (HD / 4); i += 64)
            *reinterpret_cast<float4 *>(v + to + 4 * i) = *reinterpret_cast<const float4 *>(held + i / (HD / 4) * HELD + 4 * (i % (HD / 4)));
        wave_fence();
    }
}

}  // namespace

hipError_t launch_head_rows(const HeadRows &p, int cus, hipStream_t s) {
    HeadPlan plan{};
    plan.units = (p.hd + 7) / 8;
    plan.team = 8;
    while (plan.team < plan.units) plan.team *= 2;  // at most 64: hd is at most 512
    const bool cache = p.c.kc != nullptr;
    const int hp = 64 / plan.team, heads = p.q_heads + p.k_heads + (cache ? p.c.nkv : 0), passes = (heads + hp - 1) / hp;
    // Few rows: their heads over wavefronts, up to 16 a CU.  (A row of 40 heads by one wavefront is ten passes in a row; 4 and
    // 64 a CU are within 0.5 us of this at 1 to 200 rows.)
    const uint32_t want = 16u * (uint32_t)cus / p.rows;
    plan.chunks = want < 1 ? 1 : want < (uint32_t)passes ? (int)want : passes;
    const int half = p.rotates ? p.rd / 2 : 0;
    plan.wave_bytes = half * 16 + (cache ? 2 * 512 * 4 + 64 * 4 : 0);
    const dim3 grid((unsigned)(((uint64_t)p.rows * plan.chunks + 3) / 4));
    const bool aligned = p.aligned && p.hd % 8 == 0, pairs = !p.rotates || !p.style;
    const Layout layout = !aligned ? LOOSE : pairs ? PAIRS : p.rd == p.hd ? SPLIT : p.rd % 8 == 0 ? MIXED : LOOSE;
    plan.streams = layout <= PAIRS && (uint64_t)p.rows * (p.q_heads + p.k_heads) * p.hd * 4 > (16u << 20);
    auto go = [&](auto l) {
        constexpr int L = decltype(l)::value;
        if (cache) hipLaunchKernelGGL((head_rows_kernel<L, true>), grid, dim3(256), 4 * plan.wave_bytes, s, p, plan);
        else hipLaunchKernelGGL((head_rows_kernel<L, false>), grid, dim3(256), 4 * plan.wave_bytes, s, p, plan);
    };
    switch (layout) {
    case SPLIT: go(std::integral_constant<int, SPLIT>{}); break;
    case PAIRS: go(std::integral_constant<int, PAIRS>{}); break;
    case MIXED: go(std::integral_constant<int, MIXED>{}); break;
    default: go(std::integral_constant<int, LOOSE>{});
    }
    return hipGetLastError();
}

hipError_t launch_kv4_load(const Kv4Layer &c, const Batch &b, float *k, float *v, hipStream_t s) {
    const dim3 grid((b.rows + 3) / 4);
    switch (c.hd) {
    case 64: hipLaunchKernelGGL(kv4_load_kernel<64>, grid, dim3(256), 0, s, c, b, k, v); break;
    case 96: hipLaunchKernelGGL(kv4_load_kernel<96>, grid, dim3(256), 0, s, c, b, k, v); break;
    case 128: hipLaunchKernelGGL(kv4_load_kernel<128>, grid, dim3(256), 0, s, c, b, k, v); break;
    default: hipLaunchKernelGGL(kv4_load_kernel<256>, grid, dim3(256), 0, s, c, b, k, v);
    }
    return hipGetLastError();
}

}  // namespace zh

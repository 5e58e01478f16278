// zh_heads.hip -- norms of query and key heads with the position rotation in one pass, and keys and values into the
// paged cache of 4 bits on the way.
#include "zh_serving.h"

namespace zh {

namespace {

typedef unsigned long long u64;

__device__ __forceinline__ double turns_per_position(const HeadRows &p, int i) {
    double f = exp2((double)i * p.freq.exponent) * 0.15915494309189533577;
    const double g = fmin(fmax(p.freq.a + p.freq.b * (p.freq.by_turns ? f : (double)i), 0.0), 1.0);
    f *= g + (1.0 - g) * p.freq.inv_factor;
    return p.factors ? f / (double)p.factors[i] : f;
}

// LDS of a wavefront's own lanes: what they wrote is what they read behind this
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// the scale byte (its exponent + 127) of 32 values whose largest magnitude has these bits
__device__ __forceinline__ uint32_t scale_byte(uint32_t bits) {
    const uint32_t e = (bits >> 23) + ((bits & 0x7FFFFFu) > 0x600000u ? 1u : 0u);  // 7 2^x is 1.75 2^(x + 2)
    return min(max(e, 33u) - 2u, 219u);
}

// A team of lanes takes a head, a lane four pairs of it.
template <bool ALIGNED, bool CACHE> __global__ void __launch_bounds__(256) head_rows_kernel(HeadRows p, int units, int team) {
    __shared__ double2 table[256];
    __shared__ __align__(16) float held[CACHE ? 2 : 1][CACHE ? 2048 : 1];  // of each team: a key, and a value
    __shared__ float held_scale[CACHE ? 256 : 1];
    const int tid = threadIdx.x, u = tid % team, slot = tid / team, hp = 256 / team;
    const int half = p.rotates ? p.rd / 2 : 0, i0 = 4 * u;
    // pair i: halves (i, i + half), neighbours (2 i, 2 i + 1) of interleaved ones and of what does not turn
    auto turns = [&](int j) { return i0 + j < half; };
    auto split = [&](int j) { return p.style && turns(j); };
    auto first_of = [&](int j) { return split(j) ? i0 + j : 2 * (i0 + j); };
    auto second_of = [&](int j) { return split(j) ? i0 + j + half : 2 * (i0 + j) + 1; };
    auto in = [&](int j) { return u < units && 2 * (i0 + j) < p.hd; };
    // ALIGNED: a unit's pairs are alike, and lie in two float4
    const int d0 = split(0) ? i0 : 2 * i0, d1 = split(0) ? i0 + half : 2 * i0 + 4;
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
    const double f = tid < half ? turns_per_position(p, tid) : 0.0;
    const int f32_heads = p.q_heads + p.k_heads, heads = f32_heads + (CACHE ? p.c.nkv : 0);
    for (uint32_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        int pos = 0;
        double at;
        uint32_t page = 0;
        bool stored = false;
        if constexpr (CACHE) {
            const Sequence q = sequence_of_row(p.b, r);
            pos = q.first + (int)(r - q.row0);
            if (q.rows == 0 || pos < 0) continue;  // (the workgroup's wavefronts alike)
            stored = (uint32_t)pos < p.b.cap;
            if (stored) page = page_of(p.b, q.index, (uint32_t)pos);
            stored = stored && page < p.b.pool;
            at = (double)pos;
        } else {
            at = (double)(p.positions ? p.positions[r] : p.first + r);
        }
        __syncthreads();  // the row before is done with the table
        if (tid < half) {
            const double t = at * f;
            double sn, cs;
            sincospi(2.0 * (t - rint(t)), &sn, &cs);
            table[tid] = make_double2(cs * (double)p.magnitude, sn * (double)p.magnitude);
        }
        __syncthreads();
        for (int h = blockIdx.y * hp + slot; h < heads; h += gridDim.y * hp) {
            const bool cached = CACHE && h >= f32_heads, key = cached || h >= p.q_heads;
            const float *src = cached ? p.k + r * p.src_stride + (size_t)(h - f32_heads) * p.hd : p.src + r * p.src_stride + (size_t)h * p.hd;
            float x[2][4] = {};
            if (ALIGNED) {
                if (u < units) {
                    const float4 a = *reinterpret_cast<const float4 *>(src + d0);
                    const float4 b = d1 < p.hd ? *reinterpret_cast<const float4 *>(src + d1) : make_float4(0.f, 0.f, 0.f, 0.f);
                    if (split(0)) {
                        x[0][0] = a.x, x[0][1] = a.y, x[0][2] = a.z, x[0][3] = a.w;
                        x[1][0] = b.x, x[1][1] = b.y, x[1][2] = b.z, x[1][3] = b.w;
                    } else {
                        x[0][0] = a.x, x[1][0] = a.y, x[0][1] = a.z, x[1][1] = a.w;
                        x[0][2] = b.x, x[1][2] = b.y, x[0][3] = b.z, x[1][3] = b.w;
                    }
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    if (in(j)) x[0][j] = src[first_of(j)];
                    if (in(j)) x[1][j] = src[second_of(j)];
                }
            }
            const bool normed = key ? p.k_norm : p.q_norm;
            double inv = 1.0;
            if (normed) {
                double ss = 0.0;
#pragma unroll
                for (int j = 0; j < 4; j++) ss = fma((double)x[0][j], (double)x[0][j], fma((double)x[1][j], (double)x[1][j], ss));
                for (int m = 1; m < team; m <<= 1) ss += __shfl_xor(ss, m);
                inv = 1.0 / sqrt(ss / p.hd + (double)p.eps);
            }
            if (!cached) {
                float *dst = p.dst + r * p.dst_stride + (size_t)h * p.hd, y[2][4];
                const float fi = (float)inv;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    float a = x[0][j], b = x[1][j];
                    if (normed) {
                        a *= (key ? wk[0][j] + p.weight_offset : wq[0][j]) * fi;
                        b *= (key ? wk[1][j] + p.weight_offset : wq[1][j]) * fi;
                    }
                    y[0][j] = a, y[1][j] = b;
                    if (turns(j)) {
                        const double2 cs = table[i0 + j];
                        const float c = (float)cs.x, s = (float)cs.y;
                        y[0][j] = a * c - b * s, y[1][j] = a * s + b * c;
                    }
                }
                if (ALIGNED) {
                    if (u < units) {
                        *reinterpret_cast<float4 *>(dst + d0) = split(0) ? make_float4(y[0][0], y[0][1], y[0][2], y[0][3]) : make_float4(y[0][0], y[1][0], y[0][1], y[1][1]);
                        if (d1 < p.hd)
                            *reinterpret_cast<float4 *>(dst + d1) = split(0) ? make_float4(y[1][0], y[1][1], y[1][2], y[1][3]) : make_float4(y[0][2], y[1][2], y[0][3], y[1][3]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        if (in(j)) dst[first_of(j)] = y[0][j];
                        if (in(j)) dst[second_of(j)] = y[1][j];
                    }
                }
            }
            if constexpr (CACHE) {
                if (!cached || !stored) continue;
                const int kvh = h - f32_heads, g_n = p.hd / 32, c = u, g = c & 3, t = c >> 2;
                float *key_at = held[0] + slot * 8 * team, *value_at = held[1] + slot * 8 * team, *scale_at = held_scale + slot * team;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    double a = (double)x[0][j], b = (double)x[1][j];
                    if (normed) {
                        a *= ((double)wk[0][j] + (double)p.weight_offset) * inv;
                        b *= ((double)wk[1][j] + (double)p.weight_offset) * inv;
                    }
                    if (turns(j)) {
                        const double2 cs = table[i0 + j];
                        const double y = a * cs.x - b * cs.y;
                        b = a * cs.y + b * cs.x, a = y;
                    }
                    if (in(j)) key_at[first_of(j)] = (float)a;
                    if (in(j)) key_at[second_of(j)] = (float)b;
                }
                const float *vs = p.v + r * p.src_stride + (size_t)kvh * p.hd;
                const bool holds = c < 4 * g_n;
                float k8[8] = {}, v8[8] = {};
                if (holds) {
                    if (ALIGNED) {
                        *reinterpret_cast<float4 *>(v8) = *reinterpret_cast<const float4 *>(vs + 8 * c);
                        *reinterpret_cast<float4 *>(v8 + 4) = *reinterpret_cast<const float4 *>(vs + 8 * c + 4);
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; e++) v8[e] = vs[8 * c + e];
                    }
#pragma unroll
                    for (int e = 0; e < 8; e++) value_at[8 * c + e] = v8[e];
                }
                wave_fence();
                uint32_t kmax = 0, vmax = 0;
                if (holds) {
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        k8[e] = key_at[8 * c + e];
                        kmax = max(kmax, __float_as_uint(k8[e]) & 0x7FFFFFFFu), vmax = max(vmax, __float_as_uint(v8[e]) & 0x7FFFFFFFu);
                    }
                }
                for (int m = 1; m < 4; m <<= 1) kmax = max(kmax, (uint32_t)__shfl_xor((int)kmax, m)), vmax = max(vmax, (uint32_t)__shfl_xor((int)vmax, m));
                const u64 lanes = team == 64 ? ~0ull : ((1ull << team) - 1) << ((tid & 63) / team * team);
                const bool marked = __ballot(max(kmax, vmax) >= 0x7F800000u) & lanes;
                const uint32_t kb = scale_byte(kmax), vb = marked ? 127u : scale_byte(vmax);
                const float ks = __uint_as_float(kb << 23);
                uint32_t w = 0;
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, k8[0], k8[1], ks, 0);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, k8[2], k8[3], ks, 1);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, k8[4], k8[5], ks, 2);
                w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, k8[6], k8[7], ks, 3);
                const int at64 = pos % kPage;
                const size_t codes = p.c.codes(page, kvh), scales = p.c.scales(page, kvh) + (size_t)at64 * g_n;
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
                    uint8_t *to = p.c.vc + codes + (size_t)(at64 / 8) * (128 * g_n) + at64 % 8 * g_n;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int n = 4 * c + e, d = n / g_n, tt = n % g_n;
                        const float a = value_at[32 * tt + d], b = value_at[32 * tt + 16 + d];
                        const uint32_t byte = marked ? 0u : __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, a, b, scale_at[tt], 0);
                        to[d * 8 * g_n + tt] = (uint8_t)byte;
                    }
                }
                wave_fence();
            }
        }
    }
}

__device__ __forceinline__ float value_of(uint32_t code) {
    const uint32_t m = code & 7u;
    const float v = m < 4 ? 0.5f * (float)m : m < 6 ? (float)m - 2.f : 2.f * (float)m - 8.f;
    return code & 8u ? -v : v;
}

// A workgroup reads a row back, a thread eight dims of a key and of a value at a time.
__global__ void __launch_bounds__(256) kv4_load_kernel(Kv4Layer c, Batch b, float *k, float *v) {
    const uint32_t r = blockIdx.x;
    const Sequence q = sequence_of_row(b, r);
    const int pos = q.first + (int)(r - q.row0), gn = c.hd / 32;
    if (q.rows == 0 || pos < 0 || (uint32_t)pos >= b.cap) return;
    const uint32_t page = page_of(b, q.index, (uint32_t)pos);
    if (page >= b.pool) return;
    const int at64 = pos % kPage, each = c.hd / 8;
    for (int i = threadIdx.x; i < c.nkv * each; i += 256) {
        const int head = i / each, n = i % each, t = n / 4, g = n % 4;
        const size_t codes = c.codes(page, head), scales = c.scales(page, head) + (size_t)at64 * gn + t;
        const uint32_t w = *reinterpret_cast<const uint32_t *>(c.kc + codes + (size_t)at64 * (c.hd / 2) + (g * gn + t) * 4);
        const uint32_t kb = c.ks[scales], vb = c.vs[scales];
        const float ks = kb == 255u ? __uint_as_float(0x7FC00000u) : __uint_as_float(kb << 23);
        const float vs = kb == 255u ? ks : __uint_as_float(vb << 23);
        const uint8_t *from = c.vc + codes + (size_t)(at64 / 8) * (128 * gn) + at64 % 8 * gn + t;
        const size_t to = (size_t)r * c.nkv * c.hd + (size_t)head * c.hd + 8 * n;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            k[to + e] = value_of(w >> 4 * e) * ks;
            const int d = (8 * n + e) % 32;
            v[to + e] = value_of((uint32_t)from[d % 16 * 8 * gn] >> (d < 16 ? 0 : 4)) * vs;
        }
    }
}

}  // namespace

hipError_t launch_head_rows(const HeadRows &p, int cus, hipStream_t s) {
    const int units = (p.hd + 7) / 8;
    int team = 8;
    while (team < units) team *= 2;  // at most 64: hd is at most 512
    const bool cache = p.c.kc != nullptr;
    const int hp = 256 / team, heads = p.q_heads + p.k_heads + (cache ? p.c.nkv : 0);
    // few rows: their heads over workgroups; many: a workgroup takes every head of several rows
    const uint32_t passes = (uint32_t)(heads + hp - 1) / hp, want = 8u * (uint32_t)cus;
    const uint32_t spread = want / p.rows < 1 ? 1 : want / p.rows, gy = passes < spread ? passes : spread;
    const dim3 grid(p.rows < want / gy ? p.rows : want / gy, gy);
    const bool aligned = p.aligned && p.hd % 4 == 0 && (!p.rotates || p.rd % 8 == 0);
    if (cache && aligned) hipLaunchKernelGGL((head_rows_kernel<true, true>), grid, dim3(256), 0, s, p, units, team);
    else if (cache) hipLaunchKernelGGL((head_rows_kernel<false, true>), grid, dim3(256), 0, s, p, units, team);
    else if (aligned) hipLaunchKernelGGL((head_rows_kernel<true, false>), grid, dim3(256), 0, s, p, units, team);
    else hipLaunchKernelGGL((head_rows_kernel<false, false>), grid, dim3(256), 0, s, p, units, team);
    return hipGetLastError();
}

hipError_t launch_kv4_load(const Kv4Layer &c, const Batch &b, float *k, float *v, hipStream_t s) {
    hipLaunchKernelGGL(kv4_load_kernel, dim3(b.rows), dim3(256), 0, s, c, b, k, v);
    return hipGetLastError();
}

}  // namespace zh

// zh_rope.hip -- rotary positions of many rows, with frequencies scaled for long contexts.
//
// (x0, x1) -> m (x0 cos t - x1 sin t, x0 sin t + x1 cos t), t = position * f_i.  The angle is taken in
// turns and in 64 bits, f_i / 2 pi = 2^(i exponent) / 2 pi, and reduced to half a turn either way
// before it is rounded to 32 bits (at position 10^6 a 32-bit angle would be off by 0.06 rad); what the
// rounding leaves off enters sine and cosine to first order.
//
// What bounds it: memory for a prompt (4096 rows of 40 heads of 128, 168 MB: 34.0 us, 4.9 TB/s; 59.4 with
// 4-byte accesses, a head and a row's angles at a time), the launch for a step (40 heads of 128: 3.1-3.5 us).
#include "zh_longctx.h"

namespace zh {

namespace {

constexpr int kPairs = 4;  // pairs of a thread: two float4 of every head it takes
constexpr int kBatch = 3;  // heads whose loads go out together

// A thread takes four pairs (or eight values behind the rotated ones) of every hp-th head of its rows.
template <bool ALIGNED> __global__ void __launch_bounds__(256) rope_rows_kernel(RopeRows p, int units, int hp) {
    const int u = threadIdx.x % units, h0 = threadIdx.x / units, half = p.rd / 2, turning = (half + kPairs - 1) / kPairs;
    if (h0 >= hp) return;
    const bool rotates = u < turning;
    const int i0 = rotates ? kPairs * u : p.rd + 8 * (u - turning);
    const int n = rotates ? min(kPairs, half - i0) : min(8, p.hd - i0);
    double f[kPairs];
    if (rotates)
        for (int j = 0; j < kPairs; j++) f[j] = p.freq.turns_per_position(min(i0 + j, half - 1), p.factors);
    for (size_t r = blockIdx.x; r < p.rows; r += gridDim.x) {
        const float *src = p.src + r * p.src_stride;
        float *dst = p.dst + r * p.dst_stride;
        float c[kPairs], s[kPairs];
        if (rotates) {
            const double at = (double)(p.positions ? p.positions[r] : p.first + (uint32_t)r);
            for (int j = 0; j < kPairs; j++) {
                const double t = at * f[j], half_turns = 2.0 * (t - rint(t));
                const float near = (float)half_turns, rest = (float)(half_turns - (double)near) * 3.14159265f;
                float sn, cs;  // of the angle rounded, then of the angle
                sincospif(near, &sn, &cs);
                c[j] = fmaf(-rest, sn, cs) * p.magnitude, s[j] = fmaf(rest, cs, sn) * p.magnitude;
            }
        }
        if constexpr (ALIGNED) {
            // this thread's two float4: the pairs' (interleaved: side by side), or what is copied
            const int a0 = rotates && !p.style ? 2 * i0 : i0, a1 = rotates && p.style ? i0 + half : a0 + 4;
            const bool two = rotates || n > 4;
            for (int h = blockIdx.y * hp + h0; h < p.heads; h += kBatch * gridDim.y * hp) {
                float4 x[kBatch], y[kBatch];
#pragma unroll
                for (int j = 0; j < kBatch; j++) {
                    const float *at = src + (size_t)min(h + j * (int)gridDim.y * hp, p.heads - 1) * p.hd;
                    x[j] = *reinterpret_cast<const float4 *>(at + a0);
                    y[j] = *reinterpret_cast<const float4 *>(at + (two ? a1 : a0));
                }
#pragma unroll
                for (int j = 0; j < kBatch; j++) {
                    const int g = h + j * (int)gridDim.y * hp;
                    if (g >= p.heads) break;
                    float *at = dst + (size_t)g * p.hd;
                    float4 u = x[j], v = y[j];
                    if (rotates && p.style) {
                        u = make_float4(x[j].x * c[0] - y[j].x * s[0], x[j].y * c[1] - y[j].y * s[1],
                                        x[j].z * c[2] - y[j].z * s[2], x[j].w * c[3] - y[j].w * s[3]);
                        v = make_float4(x[j].x * s[0] + y[j].x * c[0], x[j].y * s[1] + y[j].y * c[1],
                                        x[j].z * s[2] + y[j].z * c[2], x[j].w * s[3] + y[j].w * c[3]);
                    } else if (rotates) {
                        u = make_float4(x[j].x * c[0] - x[j].y * s[0], x[j].x * s[0] + x[j].y * c[0],
                                        x[j].z * c[1] - x[j].w * s[1], x[j].z * s[1] + x[j].w * c[1]);
                        v = make_float4(y[j].x * c[2] - y[j].y * s[2], y[j].x * s[2] + y[j].y * c[2],
                                        y[j].z * c[3] - y[j].w * s[3], y[j].z * s[3] + y[j].w * c[3]);
                    }
                    *reinterpret_cast<float4 *>(at + a0) = u;
                    if (two) *reinterpret_cast<float4 *>(at + a1) = v;
                }
            }
            continue;
        }
        for (int h = blockIdx.y * hp + h0; h < p.heads; h += gridDim.y * hp) {
            const float *x = src + (size_t)h * p.hd;
            float *y = dst + (size_t)h * p.hd;
            if (!rotates) {
                for (int j = 0; j < n; j++) y[i0 + j] = x[i0 + j];
                continue;
            }
            for (int j = 0; j < n; j++) {
                const int a = p.style ? i0 + j : 2 * (i0 + j), b = p.style ? a + half : a + 1;
                const float xa = x[a], xb = x[b];
                y[a] = xa * c[j] - xb * s[j];
                y[b] = xa * s[j] + xb * c[j];
            }
        }
    }
}

}  // namespace

hipError_t launch_rope_rows(const RopeRows &p, int cus, hipStream_t s) {
    const int units = (p.rd / 2 + kPairs - 1) / kPairs + (p.hd - p.rd + 7) / 8, hp = 256 / units;
    // few rows: their heads over workgroups; many: a workgroup takes every head of several rows, whose
    // frequencies it computes once
    const uint32_t passes = (uint32_t)(p.heads + hp - 1) / hp, want = 8u * (uint32_t)cus;
    const uint32_t spread = want / p.rows < 1 ? 1 : want / p.rows, gy = passes < spread ? passes : spread;
    const dim3 grid(p.rows < want / gy ? p.rows : want / gy, gy);
    if (p.aligned && p.hd % 4 == 0 && p.rd % 8 == 0)
        hipLaunchKernelGGL(rope_rows_kernel<true>, grid, dim3(256), 0, s, p, units, hp);
    else
        hipLaunchKernelGGL(rope_rows_kernel<false>, grid, dim3(256), 0, s, p, units, hp);
    return hipGetLastError();
}

}  // namespace zh

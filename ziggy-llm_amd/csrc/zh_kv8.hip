// zh_kv8.hip -- K/V rows into and out of the cache held in 8 bits, a scale per block of 32 positions and
// kv head.
//
// scale = max|x| / 127 of the block's rows, code = x / scale to the nearest integer (ties to even),
// decided on the exact quotient: the product with the reciprocal is at most one off next to a tie, and
// x - code * scale is exact there (the difference of near values), so one comparison with scale / 2
// mends it.  The maximum is taken of the bits of |x|, in which infinities and NaN are the largest.
#include "zh_longctx.h"

namespace zh {

namespace {

// x / s to the nearest integer, ties to even, within [-127, 127]; s > 0
__device__ __forceinline__ int code_of(float x, float s, float inv) {
    float c = fminf(fmaxf(rintf(x * inv), -127.f), 127.f);
    const float r = fmaf(-c, s, x), h = 0.5f * s, over = fabsf(r) - h;
    if (over > 0.f || (over == 0.f && ((int)c & 1))) c += r > 0.f ? 1.f : -1.f;
    return (int)fminf(fmaxf(c, -127.f), 127.f);
}

// an earlier row's code under a larger scale
__device__ __forceinline__ int recode(int c, float was, float now) {
    if (!(now > 0.f)) return 0;
    return (int)fmin(fmax(rint((double)c * (double)was / (double)now), -127.0), 127.0);
}

__device__ __forceinline__ uint32_t pack4(int a, int b, int c, int d) {
    return (uint32_t)(a & 255) | (uint32_t)(b & 255) << 8 | (uint32_t)(c & 255) << 16 | (uint32_t)d << 24;
}

// A workgroup takes one block of one kv head, K (z 0) or V (z 1).
template <int HD>
__global__ void __launch_bounds__(256) kv8_store_kernel(Kv8Layer c, const float *k, const float *v, size_t stride,
                                                        uint32_t position, uint32_t rows, int aligned) {
    constexpr int NU = HD / 32, Q = HD / 4;  // float4s of a thread, of a row
    constexpr int LD = 36;                   // bytes of a dim's 32 positions in LDS
    __shared__ uint32_t amax[4];
    __shared__ __align__(4) int8_t tile[HD * LD];
    const int tid = threadIdx.x, head = blockIdx.y;
    const bool is_v = blockIdx.z;
    const uint32_t block = position / kKv8Block + blockIdx.x, p0 = block * kKv8Block;
    const int lo = position > p0 ? (int)(position - p0) : 0, hi = (int)min(32u, position + rows - p0);
    const float *src = (is_v ? v : k) + (size_t)head * HD;
    float x[NU][4];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NU; i++) {
        const int unit = tid + 256 * i, row = unit / Q, d = 4 * (unit % Q);
#pragma unroll
        for (int j = 0; j < 4; j++) x[i][j] = 0.f;
        if (row >= lo && row < hi) {
            const float *at = src + (size_t)(p0 + row - position) * stride + d;
            if (aligned) {
                const float4 f = *reinterpret_cast<const float4 *>(at);
                x[i][0] = f.x, x[i][1] = f.y, x[i][2] = f.z, x[i][3] = f.w;
            } else {
                for (int j = 0; j < 4; j++) x[i][j] = at[j];
            }
        }
#pragma unroll
        for (int j = 0; j < 4; j++) top = max(top, __float_as_uint(x[i][j]) & 0x7FFFFFFFu);
    }
    for (int d = 32; d; d >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, d));
    if ((tid & 63) == 0) amax[tid >> 6] = top;
    float *scale = (is_v ? c.vs : c.ks) + (size_t)head * c.blocks + block;
    const float was = lo ? *scale : 0.f;
    __syncthreads();
    top = max(max(amax[0], amax[1]), max(amax[2], amax[3]));
    float now = top < 0x7F800000u ? __uint_as_float(top) / 127.f : __uint_as_float(0x7FC00000u);
    if (was > now || was != was) now = was;
    if (tid == 0) *scale = now;
    // (scales below the reciprocal's range: both sides times a power of two)
    const float up = now < 1e-30f ? 1.2676506e30f : 1.f, s = now * up, inv = 1.f / s;
    const bool live = now > 0.f, again = lo && !(now == was);
    auto code = [&](float f) { return live ? code_of(f * up, s, inv) : 0; };
    int8_t *codes = (is_v ? c.vc : c.kc) + ((size_t)head * c.blocks + block) * (kKv8Block * HD);
#pragma unroll
    for (int i = 0; i < NU; i++) {
        const int unit = tid + 256 * i, row = unit / Q, d = 4 * (unit % Q);
        if (!is_v) {
            uint32_t *at = reinterpret_cast<uint32_t *>(codes + row * HD + d);
            if (row >= lo && row < hi)
                *at = pack4(code(x[i][0]), code(x[i][1]), code(x[i][2]), code(x[i][3]));
            else if (row < lo && again) {
                const uint32_t o = *at;
                *at = pack4(recode((int8_t)o, was, now), recode((int8_t)(o >> 8), was, now),
                            recode((int8_t)(o >> 16), was, now), recode((int8_t)(o >> 24), was, now));
            }
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) tile[(d + j) * LD + row] = (int8_t)code(x[i][j]);
        }
    }
    if (!is_v) return;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NU; i++) {
        const int unit = tid + 256 * i, d = unit / 8, row = 4 * (unit % 8);
        uint32_t *at = reinterpret_cast<uint32_t *>(codes + d * kKv8Block + row);
        const uint32_t fresh = *reinterpret_cast<const uint32_t *>(tile + d * LD + row);
        if (row >= lo && row + 4 <= hi) {
            *at = fresh;
        } else if ((row < hi && row + 4 > lo) || (row < lo && again)) {
            const uint32_t o = *at;
            uint32_t w = 0;
            for (int j = 0; j < 4; j++) {
                uint32_t b = o >> (8 * j);
                if (row + j >= lo && row + j < hi) b = fresh >> (8 * j);
                else if (row + j < lo && again) b = (uint32_t)recode((int8_t)b, was, now);
                w |= (b & 255u) << (8 * j);
            }
            *at = w;
        }
    }
}

template <int HD>
__global__ void __launch_bounds__(256) kv8_load_kernel(Kv8Layer c, float *k, float *v, uint32_t position, uint32_t rows) {
    constexpr int NU = HD / 32, Q = HD / 4, LD = HD + 4;
    __shared__ __align__(4) int8_t tile[32 * LD];
    const int tid = threadIdx.x, head = blockIdx.y;
    const bool is_v = blockIdx.z;
    const uint32_t block = position / kKv8Block + blockIdx.x, p0 = block * kKv8Block;
    const int lo = position > p0 ? (int)(position - p0) : 0, hi = (int)min(32u, position + rows - p0);
    const float s = (is_v ? c.vs : c.ks)[(size_t)head * c.blocks + block];
    const int8_t *codes = (is_v ? c.vc : c.kc) + ((size_t)head * c.blocks + block) * (kKv8Block * HD);
    if (is_v) {
#pragma unroll
        for (int i = 0; i < NU; i++) {
            const int unit = tid + 256 * i, d = unit / 8, row = 4 * (unit % 8);
            const uint32_t o = *reinterpret_cast<const uint32_t *>(codes + d * kKv8Block + row);
            for (int j = 0; j < 4; j++) tile[(row + j) * LD + d] = (int8_t)(o >> (8 * j));
        }
        __syncthreads();
    }
    float *dst = (is_v ? v : k) + (size_t)head * HD;
#pragma unroll
    for (int i = 0; i < NU; i++) {
        const int unit = tid + 256 * i, row = unit / Q, d = 4 * (unit % Q);
        if (row < lo || row >= hi) continue;
        const uint32_t o = *reinterpret_cast<const uint32_t *>(is_v ? tile + row * LD + d : codes + row * HD + d);
        *reinterpret_cast<float4 *>(dst + (size_t)(p0 + row - position) * ((size_t)c.nkv * HD) + d) =
            make_float4((float)(int8_t)o * s, (float)(int8_t)(o >> 8) * s, (float)(int8_t)(o >> 16) * s,
                        (float)(int8_t)(o >> 24) * s);
    }
}

template <class F> hipError_t by_head_dim(int hd, F f) {
    switch (hd) {
    case 64: f(std::integral_constant<int, 64>{}); break;
    case 96: f(std::integral_constant<int, 96>{}); break;
    case 128: f(std::integral_constant<int, 128>{}); break;
    case 256: f(std::integral_constant<int, 256>{}); break;
    default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

dim3 block_grid(const Kv8Layer &c, uint32_t position, uint32_t rows) {
    return dim3((position + rows - 1) / kKv8Block - position / kKv8Block + 1, (unsigned)c.nkv, 2);
}

}  // namespace

hipError_t launch_kv8_store(const Kv8Layer &c, const float *k, const float *v, size_t row_stride, uint32_t position,
                            uint32_t rows, hipStream_t s) {
    const int aligned = !(((uintptr_t)k | (uintptr_t)v) % 16) && row_stride % 4 == 0;
    return by_head_dim(c.hd, [&](auto hd) {
        hipLaunchKernelGGL(kv8_store_kernel<decltype(hd)::value>, block_grid(c, position, rows), dim3(256), 0, s, c, k, v,
                           row_stride, position, rows, aligned);
    });
}

hipError_t launch_kv8_load(const Kv8Layer &c, float *k, float *v, uint32_t position, uint32_t rows, hipStream_t s) {
    return by_head_dim(c.hd, [&](auto hd) {
        hipLaunchKernelGGL(kv8_load_kernel<decltype(hd)::value>, block_grid(c, position, rows), dim3(256), 0, s, c, k, v,
                           position, rows);
    });
}

}  // namespace zh

// zh_kv8.hip -- K/V rows into and out of the cache held in 8 bits, a scale per block of 32 positions and
// kv head.
//
// scale = max|x| times 1/127, a product in binary32, of the block's rows; code = x / scale to the nearest
// integer (ties to even), decided on the exact quotient.  The product with the reciprocal, rounded to an
// integer, is that unless it lies next to a tie (within 3e-5; a wavefront in twenty has such a value):
// then every code of the thread is decided by x - code * scale, which is exact there (the difference of
// near values), against half the scale.  The maximum is taken of the bits of |x|, in which infinities and
// NaN are the largest.
//
// What bounds it: memory for a prompt (4095 rows of 8 heads of 128, K and V, 42 MB: mean 13.8 us, least 12.4, 3.0-3.4
// TB/s; the read-back of as many 7.4 and 6.5), the chain of load, maximum, scale and store for one row (3.5
// us, least 3.1; 5.7 with the exact decision and the rescaling unrolled in line, 2000 instructions more to fetch).
// Tried and slower: two blocks a workgroup (17.7 us), V's words from four rows per thread without LDS
// (17.0), workgroups ordered heads first (15.4; all against 14.7 then).
#include "zh_longctx.h"

namespace zh {

namespace {

// x / s to the nearest integer, ties to even, within [-127, 127]; s > 0
__device__ __forceinline__ int exact_code(float x, float s, float inv) {
    float c = fminf(fmaxf(rintf(x * inv), -127.f), 127.f);
    const float r = fmaf(-c, s, x), over = fabsf(r) - 0.5f * s;
    if (over > 0.f || (over == 0.f && ((int)c & 1))) c += r > 0.f ? 1.f : -1.f;
    return (int)fminf(fmaxf(c, -127.f), 127.f);
}

// an earlier row's code under a larger scale
__device__ __forceinline__ int recode(int c, float was, float now) {
    if (!(now > 0.f)) return 0;
    return (int)fmin(fmax(rint((double)c * (double)was / (double)now), -127.0), 127.0);
}

// the low bytes of four words
__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0C0C0400u), __builtin_amdgcn_perm(b, a, 0x0C0C0400u), 0x05040100u);
}

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
    auto dpp = [](uint32_t x, auto ctrl) {
        return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xF, 0xF, false);
    };
    v = max(v, dpp(v, std::integral_constant<int, 0xB1>{}));
    v = max(v, dpp(v, std::integral_constant<int, 0x4E>{}));
    v = max(v, dpp(v, std::integral_constant<int, 0x141>{}));
    v = max(v, dpp(v, std::integral_constant<int, 0x140>{}));
    uint32_t x, y;
    lane_pair<16>(v, x, y);
    v = max(x, y);
    lane_pair<32>(v, x, y);
    return max(x, y);
}

// A workgroup takes one block of one kv head, K (z 0) or V (z 1).  V goes through LDS, rows in and dims
// out.
template <int HD>
__global__ void __launch_bounds__(256) kv8_store_kernel(Kv8Layer c, const float *k, const float *v, size_t stride,
                                                        uint32_t position, uint32_t rows, int aligned) {
    constexpr int NU = HD / 32, Q = HD / 4;  // float4s of a thread, of a row
    constexpr int LD = 36;                   // bytes of a dim's 32 positions in LDS
    __shared__ uint32_t amax[4];
    __shared__ __align__(4) uint8_t tile[HD * LD];
    const int tid = threadIdx.x, head = blockIdx.y;
    const bool is_v = blockIdx.z;
    const uint32_t block = position / kKv8Block + blockIdx.x, p0 = block * kKv8Block;
    // the block's rows lo .. hi - 1 are new
    const int lo = position > p0 ? (int)(position - p0) : 0, hi = (int)min(32u, position + rows - p0);
    const bool part = lo > 0 || hi < 32;
    const float *src = (is_v ? v : k) + (size_t)head * HD;
    float *scale = (is_v ? c.vs : c.ks) + (size_t)head * c.blocks + block;
    uint32_t *codes = reinterpret_cast<uint32_t *>((is_v ? c.vc : c.kc) + ((size_t)head * c.blocks + block) * (kKv8Block * HD));
    float x[NU][4];
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
    }
    const float was = lo ? *scale : 0.f;
    uint32_t old[NU];  // V words of a block stored in part
    if (is_v && part)
#pragma unroll
        for (int i = 0; i < NU; i++) old[i] = codes[tid + 256 * i];
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < NU; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) top = max(top, __float_as_uint(x[i][j]) & 0x7FFFFFFFu);
    top = wave_max_u32(top);
    if ((tid & 63) == 0) amax[tid >> 6] = top;
    __syncthreads();
    top = max(max(amax[0], amax[1]), max(amax[2], amax[3]));
    float now = top < 0x7F800000u ? __uint_as_float(top) * (1.f / 127.f) : __uint_as_float(0x7FC00000u);
    if (was > now || was != was) now = was;
    if (tid == 0) *scale = now;

    if (lo && !(now == was)) {  // the earlier rows' codes under the new scale
#pragma unroll 1
        for (int u = tid; u < NU * 256; u += 256) {
            const int first = is_v ? 4 * (u % 8) : u / Q;  // row of byte 0; of byte j: j rows on (V), the same (K)
            if (first >= lo) continue;
            uint32_t w = codes[u], r = 0;
#pragma unroll 1
            for (int j = 0; j < 4; j++, w >>= 8) {
                const int b = is_v && first + j >= lo ? (int8_t)w : recode((int8_t)w, was, now);
                r |= (uint32_t)(b & 255) << (8 * j);
            }
            codes[u] = r;
        }
        if (is_v)  // (a thread's own words)
#pragma unroll
            for (int i = 0; i < NU; i++) old[i] = codes[tid + 256 * i];
    }

    // u's low byte is the code: the integer in the low bits of 1.5 2^23 + x / s.  A scale of 0 or NaN: codes 0
    const bool live = now > 0.f, tiny = live && now < 1e-30f;
    float inv = live ? 1.f / now : 0.f, near = 0.f;
    constexpr float kRound = 12582912.f;
    uint32_t u[NU][4];
#pragma unroll
    for (int i = 0; i < NU; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float t = fmaf(x[i][j], inv, kRound);
            u[i][j] = __float_as_uint(t);
            near = fmaxf(near, fabsf(fmaf(x[i][j], inv, kRound - t)));
        }
    if (tiny || near > 0.49997f) {
        // (scales below the reciprocal's range: both sides times a power of two)
        const float up = tiny ? 1.2676506e30f : 1.f, s = now * up;
        inv = 1.f / s;
#pragma unroll
        for (int i = 0; i < NU; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) u[i][j] = (uint32_t)exact_code(x[i][j] * up, s, inv);
    }
#pragma unroll
    for (int i = 0; i < NU; i++) {
        const int unit = tid + 256 * i, row = unit / Q, d = 4 * (unit % Q);
        if (is_v) {
#pragma unroll
            for (int j = 0; j < 4; j++) tile[(d + j) * LD + row] = (uint8_t)u[i][j];
        } else if (row >= lo && row < hi) {
            codes[unit] = pack4(u[i][0], u[i][1], u[i][2], u[i][3]);
        }
    }
    if (!is_v) return;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NU; i++) {
        const int unit = tid + 256 * i, d = unit / 8, row = 4 * (unit % 8);
        uint32_t w = *reinterpret_cast<const uint32_t *>(tile + d * LD + row);
        if (part) {
            const int a = min(max(lo - row, 0), 4), b = min(max(hi - row, 0), 4);  // bytes a .. b - 1 are new
            if (a >= b) continue;
            const uint32_t upto_b = b == 4 ? 0xFFFFFFFFu : (1u << (8 * b)) - 1u, mask = upto_b & ~((1u << (8 * a)) - 1u);
            w = (w & mask) | (old[i] & ~mask);
        }
        codes[unit] = w;
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

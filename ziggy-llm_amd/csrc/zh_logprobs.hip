// zh_logprobs.hip -- log probabilities of given tokens, the rows' entropy and their best tokens.
#include "zh_serving.h"

namespace zh {

namespace {

typedef unsigned long long u64;

// orders by value, the highest first, then by index, the lowest first; NaN as -infinity, the zeros equal
__device__ __forceinline__ u64 key_of(float v, uint32_t i) {
    const uint32_t b = __float_as_uint(v != v ? -INFINITY : v + 0.f);
    return (u64)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (0xFFFFFFFFu - i);
}
__device__ __forceinline__ float value_of_key(u64 k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}

// A workgroup per row.
__global__ void __launch_bounds__(1024) logprobs_kernel(TokenLogprobs p) {
    __shared__ u64 best[16];
    __shared__ double sums[2][16];
    const uint32_t r = blockIdx.x, tid = threadIdx.x, wave = tid >> 6;
    const float *x = p.x + (size_t)r * p.stride;
    auto top_below = [&](u64 limit) {
        u64 k = 0;
        for (uint32_t i = tid; i < p.vocab; i += 1024) {
            const u64 n = key_of(x[i], i);
            if (n < limit && n > k) k = n;
        }
        k = wave_max_key(k);
        if ((tid & 63) == 0) best[wave] = k;
        __syncthreads();
        k = 0;
        for (int w = 0; w < 16; w++) k = best[w] > k ? best[w] : k;
        __syncthreads();
        return k;
    };
    u64 k = top_below(~0ull);
    const float m = value_of_key(k);
    const uint32_t at = 0xFFFFFFFFu - (uint32_t)k;  // its own weight, 1, stays out of the sum, which may be next to nothing
    double s = 0, t = 0;
    for (uint32_t i = tid; i < p.vocab; i += 1024) {
        if (i == at) continue;
        const float v = x[i], d = v != v ? -INFINITY : v - m, e = expf(d);
        s += (double)e;
        if (e > 0.f) t += (double)e * (double)d;
    }
    for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d), t += __shfl_xor(t, d);
    if ((tid & 63) == 0) sums[0][wave] = s, sums[1][wave] = t;
    __syncthreads();
    s = t = 0;
    for (int w = 0; w < 16; w++) s += sums[0][w], t += sums[1][w];
    const double nan = (double)__uint_as_float(0x7FC00000u), log_s = isfinite(m) ? log1p(s) : nan;
    if (tid == 0) {
        const uint32_t token = p.tokens[r];
        double y = nan;
        if (token < p.vocab) {
            const float v = x[token];
            y = ((double)(v != v ? -INFINITY : v) - (double)m) - log_s;
        }
        p.out[r] = (float)y;
        if (p.entropy) p.entropy[r] = (float)(log_s - t / (1.0 + s));
    }
    for (int i = 0; i < p.k; i++) {
        if (tid == 0) {
            p.top_tokens[(size_t)r * p.k + i] = 0xFFFFFFFFu - (uint32_t)k;
            p.top[(size_t)r * p.k + i] = (float)(((double)value_of_key(k) - (double)m) - log_s);
        }
        if (i + 1 < p.k) k = top_below(k);
    }
}

}  // namespace

hipError_t launch_token_logprobs(const TokenLogprobs &p, int cus, hipStream_t s) {
    hipLaunchKernelGGL(logprobs_kernel, dim3(p.rows), dim3(1024), 0, s, p);
    return hipGetLastError();
}

}  // namespace zh

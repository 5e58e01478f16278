// zh_draw.hip -- sampling from the logits on the device: temperature, top-k, top-p, min-p and repeat
// penalty, with given random numbers.
//
// Every limit keeps a beginning of the candidates in some order, and the draw is the first candidate
// whose running sum reaches a target.  So all of it is one search: the first element, in descending
// order of a key, whose running sum of weights (or count) reaches a target, found digit by digit of
// the key from histograms of the sums.  Weights are exp((a - max) / T) in 64 bits, rounded to integers
// of 2^-s, so that sums are exact whatever their order.
#include "zh_longctx.h"

namespace zh {

namespace {

constexpr int kThreads = 1024;

// float -> an integer that orders as it does; NaN as -infinity, the zeros equal
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t b = __float_as_uint(v != v ? -INFINITY : v + 0.f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

struct Key {
    uint32_t w[3];
};
__device__ __forceinline__ bool at_least(const Key &a, const Key &b) {
    return a.w[0] != b.w[0] ? a.w[0] > b.w[0] : a.w[1] != b.w[1] ? a.w[1] > b.w[1] : a.w[2] >= b.w[2];
}

struct Shared {
    unsigned long long hist[256], sum;
    uint32_t digit;
    uint32_t seen[262144 / 32];
    Key best;
    unsigned long long red[kThreads / 64];
    Key redk[kThreads / 64];
};

// The first element, in descending order of key(i), at which the sum of weight(i) reaches target (1 ..
// the whole sum); *before: the sum of those ahead of it.
template <class K, class W>
__device__ Key reach(Shared &sh, uint32_t n, unsigned long long target, unsigned long long *before, K key, W weight) {
    Key b{};
    unsigned long long done = 0;
    for (int d = 0; d < 12; d++) {
        const int word = d / 4, shift = 24 - 8 * (d % 4);
        __syncthreads();
        if (threadIdx.x < 256) sh.hist[threadIdx.x] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
            const unsigned long long w = weight(i);
            if (w == 0) continue;
            const Key k = key(i);
            bool in = true;
            for (int j = 0; j < 3; j++) {
                const uint32_t mask = j < word ? 0xFFFFFFFFu : j > word || shift == 24 ? 0u : 0xFFFFFFFFu << (shift + 8);
                in = in && ((k.w[j] ^ b.w[j]) & mask) == 0;
            }
            if (in) atomicAdd(&sh.hist[k.w[word] >> shift & 255u], w);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            unsigned long long sum = done;
            uint32_t last = 0, at = 256;
            for (int g = 255; g >= 0 && at == 256; g--) {
                if (!sh.hist[g]) continue;
                last = g;
                if (sum + sh.hist[g] >= target) at = g;
                else sum += sh.hist[g];
            }
            sh.digit = at < 256 ? at : last;
            sh.sum = sum;
        }
        __syncthreads();
        b.w[word] |= sh.digit << shift;
        done = sh.sum;
    }
    *before = done;
    return b;
}

template <class K> __device__ Key largest(Shared &sh, uint32_t n, K key) {
    Key k{};
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        const Key c = key(i);
        if (at_least(c, k)) k = c;
    }
    for (int d = 32; d; d >>= 1) {
        Key o;
        for (int j = 0; j < 3; j++) o.w[j] = (uint32_t)__shfl_xor((int)k.w[j], d);
        if (at_least(o, k)) k = o;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.redk[threadIdx.x >> 6] = k;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int j = 1; j < kThreads / 64; j++)
            if (at_least(sh.redk[j], k)) k = sh.redk[j];
        sh.best = k;
    }
    __syncthreads();
    return sh.best;
}

__device__ unsigned long long block_sum(Shared &sh, unsigned long long v) {
    for (int d = 32; d; d >>= 1) {
        const uint32_t lo = (uint32_t)__shfl_xor((int)(uint32_t)v, d), hi = (uint32_t)__shfl_xor((int)(uint32_t)(v >> 32), d);
        v += (unsigned long long)hi << 32 | lo;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
    for (int j = 0; j < kThreads / 64; j++) v += sh.red[j];
    return v;
}

__device__ unsigned long long target_of(double share, unsigned long long total) {
    const double t = ceil(share * (double)total);
    const unsigned long long c = t >= 1.0 ? (unsigned long long)t : 1ull;
    return c < total ? c : total;
}

// A workgroup takes one row.
__global__ void __launch_bounds__(kThreads) draw_simple_kernel(SampleRows p, unsigned long long *weights, size_t ld) {
    __shared__ Shared sh;
    const uint32_t n = p.vocab;
    const float *x = p.x + blockIdx.x * p.stride;
    unsigned long long *w = weights + blockIdx.x * ld;
    auto raw = [&](uint32_t i) { return x[i]; };
    if (p.o.temperature <= 0.f) {
        const Key k = largest(sh, n, [&](uint32_t i) { return Key{{ordered(raw(i)), ~i, 0}}; });
        if (threadIdx.x == 0) p.out[blockIdx.x] = ~k.w[1];
        return;
    }
    if (p.recent) {
        for (uint32_t i = threadIdx.x; i < (n + 31) / 32; i += kThreads) sh.seen[i] = 0;
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < p.recent_count; i += kThreads) {
            const uint32_t id = p.recent[(size_t)blockIdx.x * p.recent_count + i];
            if (id < n) atomicOr(&sh.seen[id / 32], 1u << (id % 32));
        }
        __syncthreads();
    }
    auto logit = [&](uint32_t i) {
        const float v = x[i], r = p.o.repeat_penalty;
        if (!p.recent || !(sh.seen[i / 32] >> (i % 32) & 1u)) return v;
        return v < 0.f ? v * r : v / r;
    };
    const uint32_t top_k = p.o.top_k == 0 ? n : min(p.o.top_k, n);
    const bool limited = top_k < n, sorted = p.o.top_p < 1.f;
    unsigned long long before;
    auto by_raw = [&](uint32_t i) { return Key{{ordered(raw(i)), ~i, 0}}; };
    Key last{};
    if (limited) last = reach(sh, n, top_k, &before, by_raw, [&](uint32_t) { return 1ull; });
    auto in = [&](uint32_t i) { return !limited || at_least(by_raw(i), last); };
    auto by_logit = [&](uint32_t i) { return Key{{ordered(logit(i)), limited ? ordered(raw(i)) : 0u, ~i}}; };
    const Key best = largest(sh, n, [&](uint32_t i) { return in(i) ? by_logit(i) : Key{}; });
    const float mx = logit(~best.w[2]);
    if (!(fabsf(mx) < INFINITY)) {
        if (threadIdx.x == 0) p.out[blockIdx.x] = ~best.w[2];
        return;
    }
    int bits = 0;
    while ((1u << bits) < top_k) bits++;
    const double unit = ldexp(1.0, 62 - bits), t = (double)p.o.temperature, least = (double)p.o.min_p;
    unsigned long long total = 0;
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        const float a = logit(i);
        unsigned long long v = 0;
        if (a > -INFINITY && in(i)) {
            const double e = exp(((double)a - (double)mx) / t);
            if (e >= least) v = (unsigned long long)rint(e * unit);
        }
        w[i] = v;
        total += v;
    }
    total = block_sum(sh, total);
    auto weight = [&](uint32_t i) { return w[i]; };
    if (sorted) {
        const Key end = reach(sh, n, target_of((double)p.o.top_p, total), &before, by_logit, weight);
        total = before + w[~end.w[2]];
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < n; i += kThreads)
            if (!at_least(by_logit(i), end)) w[i] = 0;
        __syncthreads();
    }
    const double given = p.uniforms[blockIdx.x], u = given >= 0.0 ? fmin(given, 1.0) : 0.0;
    const unsigned long long target = target_of(u, total);
    uint32_t id;
    if (sorted) id = ~reach(sh, n, target, &before, by_logit, weight).w[2];
    else if (limited) id = ~reach(sh, n, target, &before, by_raw, weight).w[1];
    else id = ~reach(sh, n, target, &before, [&](uint32_t i) { return Key{{~i, 0, 0}}; }, weight).w[0];
    if (threadIdx.x == 0) p.out[blockIdx.x] = id;
}

}  // namespace

size_t sample_rows_bytes(uint32_t vocab) { return ((size_t)vocab * 8 + 255) / 256 * 256; }

hipError_t launch_sample_rows(const SampleRows &p, hipStream_t s) {
    hipLaunchKernelGGL(draw_simple_kernel, dim3(p.rows), dim3(kThreads), 0, s, p, (unsigned long long *)p.work,
                       sample_rows_bytes(p.vocab) / 8);
    return hipGetLastError();
}

}  // namespace zh

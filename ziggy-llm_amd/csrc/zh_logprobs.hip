// zh_logprobs.hip -- log probabilities of given tokens, the rows' entropy and their best tokens.
//
// ln p_t = (x_t - m) - ln S, S = sum e^(x - m), m the largest logit; the entropy is ln S - T / S, T = sum e^d d of
// d = x - m.  The largest's own weight, 1, stays out of the sums (others as large are counted), so that ln S = log1p(S')
// keeps its digits where one token takes nearly everything.
//
// Two launches, one pass over the logits:
//   slices  a workgroup per 2048 logits (8192 where rows alone fill the device), held in registers: the largest, the
//           sums relative to it, and its k best in order;
//   rows    a workgroup per row joins its slices.
// The k best: a value that at least k others of the slice reach (the k-th of 64 columns' largest) leaves few
// candidates, and a candidate's place is the count of those above it: no sort, no dependence on the order of arrival.
#include <algorithm>

#include "zh_serving.h"

namespace zh {

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 256, kCandidates = 1024, kMaxSlices = 128, kTop = ZIGGY_HIP_MAX_TOP_LOGPROBS;

struct SliceSums {
    float top;       // the largest
    uint32_t count;  // logits that are
    double s, t;     // of the others' weights relative to it, and of those times their logits less its own
};
struct LogprobsWork {
    SliceSums *sums;  // [row][slice]
    u64 *top;         // [row][slice][k]
    uint32_t slices;
};

// orders by value, the highest first, then by index, the lowest first; NaN as -infinity, the zeros equal; above 0
__device__ __forceinline__ u64 key_of(float v, uint32_t i) {
    const uint32_t b = __float_as_uint(v != v ? -INFINITY : v + 0.f);
    return (u64)(b & 0x80000000u ? ~b : b | 0x80000000u) << 32 | (0xFFFFFFFFu - i);
}
__device__ __forceinline__ float value_of_key(u64 k) {
    const uint32_t o = (uint32_t)(k >> 32);
    return __uint_as_float(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}
__device__ __forceinline__ uint32_t index_of_key(u64 k) { return 0xFFFFFFFFu - (uint32_t)k; }

// e^d for d <= 0 to about a step and a half of binary32: what the exponent's rounding leaves off comes back to first
// order.  -infinity (and NaN) as -150: 0 all the same.
__device__ __forceinline__ float exp_of(float d) {
    const float t = d * 1.44269504f, r = fmaf(t, 1.90465421e-9f, fmaf(t, -0.693147182f, d)), e = __builtin_amdgcn_exp2f(t);
    return fmaf(e, r, e);
}

__device__ __forceinline__ double wave_sum(double v) {
    auto add = [](double x, u64 y) { return x + __longlong_as_double((long long)y); };
    v = add(v, dpp_u64<0xB1>((u64)__double_as_longlong(v)));
    v = add(v, dpp_u64<0x4E>((u64)__double_as_longlong(v)));
    v = add(v, dpp_u64<0x141>((u64)__double_as_longlong(v)));
    v = add(v, dpp_u64<0x140>((u64)__double_as_longlong(v)));
    auto far = [](double x, auto d) {
        const u64 u = (u64)__double_as_longlong(x);
        uint32_t a0, b0, a1, b1;
        lane_pair<decltype(d)::value>((uint32_t)u, a0, b0);
        lane_pair<decltype(d)::value>((uint32_t)(u >> 32), a1, b1);
        return __longlong_as_double((long long)((u64)a1 << 32 | a0)) + __longlong_as_double((long long)((u64)b1 << 32 | b0));
    };
    v = far(v, std::integral_constant<int, 16>{});
    return far(v, std::integral_constant<int, 32>{});
}

// candidates' places by counting: those of rank below k go to `to`
__device__ __forceinline__ void place(const u64 *candidates, int n, int k, u64 *to) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const u64 own = candidates[i];
        int rank = 0;
        for (int j = 0; j < n; j++) rank += candidates[j] > own;
        if (rank < k) to[rank] = own;
    }
}

// A workgroup per slice of 256 V logits.
template <int V> __global__ void __launch_bounds__(kThreads) logprobs_slice_kernel(TokenLogprobs p, LogprobsWork w) {
    __shared__ u64 columns[4][64], candidates[kCandidates];
    __shared__ double sums[2][4];
    __shared__ float tops[4];
    __shared__ uint32_t counts[4];
    __shared__ int ranks[64], found;
    const uint32_t row = blockIdx.x / w.slices, slice = blockIdx.x % w.slices, first = slice * (kThreads * V);
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const float *x = p.x + (size_t)row * p.stride + first;
    const uint32_t n = min((uint32_t)(kThreads * V), p.vocab - first);
    float v[V];
    auto at = [&](int j) { return (uint32_t)((j / 4 * kThreads + tid) * 4 + j % 4); };
#pragma unroll
    for (int j = 0; j < V; j += 4) {
        if (at(j) + 4 <= n) {
            __builtin_memcpy(&v[j], x + at(j), 16);
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) v[j + e] = at(j) + e < n ? x[at(j) + e] : -INFINITY;
        }
    }
    float top = -INFINITY;  // (fmaxf passes over NaN)
#pragma unroll
    for (int j = 0; j < V; j++) top = fmaxf(top, v[j]);
    u64 own = 0;  // this thread's best, while the best are asked for
    if (p.k) {
        uint32_t best = 0;
#pragma unroll
        for (int j = V - 1; j >= 0; j--) {
            if (v[j] != v[j]) v[j] = -INFINITY;
            if (v[j] == top) best = at(j);
        }
        if (best < n) own = key_of(top, first + best);  // (-infinity: the first of its own or none's)
        columns[wave][lane] = own;
        if (wave == 0) ranks[lane] = 0;
    }
    top = wave_max_f32(top);
    if (lane == 0) tops[wave] = top;
    if (tid == 0) found = 0;
    __syncthreads();
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    double s = 0.0, t = 0.0;
    uint32_t count = 0;
#pragma unroll
    for (int j = 0; j < V; j += 8) {  // eight at a time in binary32
        float e[8], d[8];
#pragma unroll
        for (int i = 0; i < 8; i++) {
            d[i] = fmaxf(v[j + i] - top, -150.f);
            const bool largest = v[j + i] == top;
            count += largest;
            e[i] = largest ? 0.f : exp_of(d[i]);
        }
        s += (double)(((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7])));
        t += (double)((fmaf(e[0], d[0], e[1] * d[1]) + fmaf(e[2], d[2], e[3] * d[3])) + (fmaf(e[4], d[4], e[5] * d[5]) + fmaf(e[6], d[6], e[7] * d[7])));
    }
    s = wave_sum(s), t = wave_sum(t);
    for (int d = 1; d < 64; d <<= 1) count += (uint32_t)__shfl_xor((int)count, d);
    if (lane == 0) sums[0][wave] = s, sums[1][wave] = t, counts[wave] = count;
    u64 column = 0;
    if (p.k) {
        // ranks of the columns' largest, each wavefront against sixteen of them
        column = max(max(columns[0][lane], columns[1][lane]), max(columns[2][lane], columns[3][lane]));
        int rank = 0;
#pragma unroll
        for (int i = 0; i < 16; i++) {
            const u64 other = (u64)(uint32_t)__builtin_amdgcn_readlane((int)(column >> 32), 16 * wave + i) << 32 |
                              (uint32_t)__builtin_amdgcn_readlane((int)column, 16 * wave + i);
            rank += other > column;
        }
        atomicAdd(&ranks[lane], rank);
    }
    __syncthreads();
    const size_t out = (size_t)row * w.slices + slice;
    if (tid == 0)
        w.sums[out] = {top, counts[0] + counts[1] + counts[2] + counts[3], (sums[0][0] + sums[0][1]) + (sums[0][2] + sums[0][3]),
                       (sums[1][0] + sums[1][1]) + (sums[1][2] + sums[1][3])};
    if (p.k == 0) return;
    // the k-th of the columns' largest, which k logits reach
    const u64 here = __ballot(ranks[lane] == p.k - 1 && column);
    u64 least = 1;
    if (here) {
        const int i = __ffsll(here) - 1;
        least = (u64)(uint32_t)__builtin_amdgcn_readlane((int)(column >> 32), i) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)column, i);
    }
    if (own >= least) {
#pragma unroll
        for (int j = 0; j < V; j++) {
            const u64 k = key_of(v[j], first + at(j));
            if (at(j) < n && k >= least) {
                const int i = atomicAdd(&found, 1);
                if (i < kCandidates) candidates[i] = k;
            }
        }
    }
    __syncthreads();
    u64 *to = w.top + out * p.k;
    const int c = found;
    if (c <= kCandidates) {
        for (int i = c + tid; i < p.k; i += kThreads) to[i] = 0;  // (fewer logits than that)
        place(candidates, c, p.k, to);
        return;
    }
    // the best crowd a few columns (their places in the slice alike to a multiple of 256): one after the other
    u64 last = ~0ull;
    for (int i = 0; i < p.k; i++) {
        u64 k = 0;
#pragma unroll
        for (int j = 0; j < V; j++) {
            const u64 o = key_of(v[j], first + at(j));
            if (at(j) < n && o > k && o < last) k = o;
        }
        k = wave_max_key(k);
        __syncthreads();
        if (lane == 0) columns[0][wave] = k;
        __syncthreads();
        last = max(max(columns[0][0], columns[0][1]), max(columns[0][2], columns[0][3]));
        if (tid == 0) to[i] = last;
    }
}

// A workgroup per row.
__global__ void __launch_bounds__(1024) logprobs_row_kernel(TokenLogprobs p, LogprobsWork w) {
    __shared__ __align__(16) u64 heads[8][kMaxSlices], candidates[kTop * kMaxSlices], placed[kTop], limits[8];
    __shared__ double sums[3][2];
    __shared__ float tops[2];
    __shared__ int found;
    const uint32_t row = blockIdx.x, n = w.slices;
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const SliceSums *from = w.sums + (size_t)row * n;
    const u64 *top = w.top + (size_t)row * n * p.k;
    SliceSums own{-INFINITY, 0, 0.0, 0.0};
    if ((uint32_t)tid < n) own = from[tid];
    const uint32_t token = p.tokens[row];
    const float given = token < p.vocab ? p.x[(size_t)row * p.stride + token] : 0.f;
    // For each j of 1, 2, 4 .. k: of the slices' j-th best the ceil(k / j)-th largest is a value that k logits reach.
    const int group = tid >> 7, j = 1 << group, i = tid & 127;
    if (p.k) {
        heads[group][i] = (uint32_t)i < n && j <= p.k ? top[(size_t)i * p.k + j - 1] : 0ull;
        if (i == 0) limits[group] = 1;
    }
    if (tid == 0) found = 0;
    if (tid < 64 * 2) {
        const float m = wave_max_f32(own.top);
        if (lane == 0) tops[wave] = m;
    }
    __syncthreads();
    const float largest = fmaxf(tops[0], tops[1]);
    if (tid < 64 * 2) {
        // slices that have the largest give its count, the others their weights
        double s = own.s, t = own.t, count = own.top == largest ? (double)own.count : 0.0;
        if (own.top != largest) {
            const double d = fmax((double)own.top - (double)largest, -1000.0), f = exp(d), all = own.count + own.s;
            s = f * all, t = f * (own.t + d * all);
        }
        s = wave_sum(s), t = wave_sum(t), count = wave_sum(count);
        if (lane == 0) sums[0][wave] = s, sums[1][wave] = t, sums[2][wave] = count;
    }
    if (j <= p.k) {
        const u64 mine = heads[group][i];
        int rank = 0;
        for (uint32_t o = 0; o < n; o += 2) {  // (those behind the last are 0)
            const ulonglong2 other = *reinterpret_cast<const ulonglong2 *>(&heads[group][o]);
            rank += (other.x > mine) + (other.y > mine);
        }
        if (mine && rank == (p.k + j - 1) / j - 1) limits[group] = mine;
    }
    __syncthreads();
    const double s = (sums[0][0] + sums[0][1]) + (sums[2][0] + sums[2][1] - 1.0), t = sums[1][0] + sums[1][1], nan = (double)__uint_as_float(0x7FC00000u);
    const double log_s = isfinite(largest) ? log1p(s) : nan;
    auto logprob = [&](float v) { return (float)(((double)(v != v ? -INFINITY : v) - (double)largest) - log_s); };
    if (tid == 0) {
        p.out[row] = token < p.vocab ? logprob(given) : (float)nan;
        if (p.entropy) p.entropy[row] = (float)(log_s - t / (1.0 + s));
    }
    if (p.k == 0) return;
    u64 least = 1;
#pragma unroll
    for (int g = 0; g < 8; g++) least = max(least, limits[g]);
    // a slice's are in order: an eighth of a wavefront takes a slice until one falls below
    for (uint32_t a = (uint32_t)tid / 8; a < n; a += 128)
        for (int b = tid & 7; b < p.k; b += 8) {
            const u64 k = top[(size_t)a * p.k + b];
            if (k < least) break;
            candidates[atomicAdd(&found, 1)] = k;
        }
    __syncthreads();
    place(candidates, found, p.k, placed);
    __syncthreads();
    if (tid < p.k) {
        p.top_tokens[(size_t)row * p.k + tid] = index_of_key(placed[tid]);
        p.top[(size_t)row * p.k + tid] = logprob(value_of_key(placed[tid]));
    }
}

}  // namespace

hipError_t launch_token_logprobs(const TokenLogprobs &a, int cus, hipStream_t s) {
    // slices of 2048 logits fill the device while there are up to 16 workgroups a CU of them
    const bool wide = (uint64_t)a.rows * ((a.vocab + 2047) / 2048) > 16ull * cus;
    LogprobsWork w{};
    w.slices = wide ? (a.vocab + 8191) / 8192 : (a.vocab + 2047) / 2048;
    const size_t each = w.slices * (sizeof(SliceSums) + 8 * (size_t)a.k);
    const uint32_t most = (uint32_t)std::min<size_t>(a.work_bytes / each, 0x7FFFFFFFu / w.slices);
    TokenLogprobs p = a;
    for (uint32_t r = 0; r < a.rows; r += p.rows) {  // as many rows at a time as the workspace holds
        p.rows = std::min(a.rows - r, most);
        p.x = a.x + (size_t)r * a.stride, p.tokens = a.tokens + r, p.out = a.out + r;
        p.entropy = a.entropy ? a.entropy + r : nullptr;
        if (a.k) p.top = a.top + (size_t)r * a.k, p.top_tokens = a.top_tokens + (size_t)r * a.k;
        w.sums = (SliceSums *)a.work, w.top = (u64 *)(w.sums + (size_t)p.rows * w.slices);
        const dim3 grid(p.rows * w.slices);
        if (wide) hipLaunchKernelGGL(logprobs_slice_kernel<32>, grid, dim3(kThreads), 0, s, p, w);
        else hipLaunchKernelGGL(logprobs_slice_kernel<8>, grid, dim3(kThreads), 0, s, p, w);
        hipLaunchKernelGGL(logprobs_row_kernel, dim3(p.rows), dim3(1024), 0, s, p, w);
    }
    return hipGetLastError();
}

}  // namespace zh

// zh_logprobs.hip -- log probabilities of given tokens, the rows' entropy and their best tokens.
//
// ln p_t = (x_t - m) - ln S, S = sum e^(x - m), m the largest logit; the entropy is ln S - T / S, T = sum e^d d of
// d = x - m.  The largest's own weight, 1, stays out of the sums (others as large are counted), so that ln S = log1p(S')
// keeps its digits where one token takes nearly everything.
//
// Two launches, one pass over the logits:
//   slices  a workgroup per 4096 logits (8192 where those fill the device), held in registers: the largest, the
//           sums relative to it, and its k best in order;
//   rows    a workgroup per row joins its slices (rows of up to 8192 logits: one slice, which is the answer).
// The k best of a slice: a value that k logits reach leaves few candidates, and a candidate's place is the count of those
// above it: no sort, no dependence on the order of arrival.
//
// What bounds it: 511 rows of 151936 memory (56 us for 311 MB, 5.5 TB/s); 33 of 128256 the loads and the sums 7.6 us, 20
// alternatives of each slice 4, the rows 3.9 (17 MB are 3.3 us of memory); one row the chain of two launches, load,
// exchange and join (4.7 + 3.7).
#include <algorithm>

#include "zh_serving.h"

namespace zh {

namespace {

typedef unsigned long long u64;

constexpr int kThreads = 256, kCandidates = 1024, kMaxSlices = 64, kTop = ZIGGY_HIP_MAX_TOP_LOGPROBS;

struct SliceSums {
    float top;       // the largest
    uint32_t count;  // logits that are
    double s, t;     // of the others' weights relative to it, and of those times their logits less its own
};
struct LogprobsWork {
    SliceSums *sums;  // [row][slice]
    u64 *top;         // [row][slice][k]
    uint32_t slices, logits;  // of a row, and (all but the last) of a slice: a multiple of 4
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

// candidates' places by counting: to(rank, candidate) for those of rank below k
template <class F> __device__ __forceinline__ void place(const u64 *candidates, int n, int k, F to) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const u64 own = candidates[i];
        int rank = 0, j = 0;
        for (; j + 8 <= n; j += 8) {
            ulonglong2 o[4];
#pragma unroll
            for (int e = 0; e < 4; e++) o[e] = *reinterpret_cast<const ulonglong2 *>(candidates + j + 2 * e);
#pragma unroll
            for (int e = 0; e < 4; e++) rank += (o[e].x > own) + (o[e].y > own);
        }
        for (; j < n; j++) rank += candidates[j] > own;
        if (rank < k) to(rank, own);
    }
}

// lanes of this one's row of 16 with a larger value
__device__ __forceinline__ int above_in_row(float v) {
    int above = 0;
    auto turn = [&](auto by) {  // the lane so many on within the row
        const float other = __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + decltype(by)::value, 0xF, 0xF, false));
        above += other > v;
    };
    turn(std::integral_constant<int, 1>{}), turn(std::integral_constant<int, 2>{}), turn(std::integral_constant<int, 3>{});
    turn(std::integral_constant<int, 4>{}), turn(std::integral_constant<int, 5>{}), turn(std::integral_constant<int, 6>{});
    turn(std::integral_constant<int, 7>{}), turn(std::integral_constant<int, 8>{}), turn(std::integral_constant<int, 9>{});
    turn(std::integral_constant<int, 10>{}), turn(std::integral_constant<int, 11>{}), turn(std::integral_constant<int, 12>{});
    turn(std::integral_constant<int, 13>{}), turn(std::integral_constant<int, 14>{}), turn(std::integral_constant<int, 15>{});
    return above;
}
// the largest of four lanes, and of a row of 16
template <int CTRL> __device__ __forceinline__ float max_moved(float v) {
    return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false)));
}
__device__ __forceinline__ float quad_max(float v) { return max_moved<0x4E>(max_moved<0xB1>(v)); }
__device__ __forceinline__ float row_max(float v) { return max_moved<0x140>(max_moved<0x141>(quad_max(v))); }

__device__ __forceinline__ float logprob_of(float v, float largest, double log_s) {
    return (float)(((double)(v != v ? -INFINITY : v) - (double)largest) - log_s);
}
// A row's log probability and entropy, by the first lane: s the weights beside one of the largest, t = sum e^d d.
__device__ __forceinline__ double finish_row(const TokenLogprobs &p, uint32_t row, float largest, double s, double t, uint32_t token,
                                             float given, bool first) {
    const double nan = (double)__uint_as_float(0x7FC00000u), log_s = isfinite(largest) ? log1p(s) : nan;
    if (first) {
        p.out[row] = token < p.vocab ? logprob_of(given, largest, log_s) : (float)nan;
        if (p.entropy) p.entropy[row] = (float)(log_s - t / (1.0 + s));
    }
    return log_s;
}
__device__ __forceinline__ void put_best(const TokenLogprobs &p, uint32_t row, int rank, uint32_t token, float v, float largest, double log_s) {
    p.top_tokens[(size_t)row * p.k + rank] = token;
    p.top[(size_t)row * p.k + rank] = logprob_of(v, largest, log_s);
}
// Fewer finite logits than k: `have` are placed, all of them, +infinities too; the first of the others follow.
template <int THREADS>
__device__ __forceinline__ void put_others(const TokenLogprobs &p, uint32_t row, uint32_t have, float largest, double log_s, uint32_t *taken) {
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    for (uint32_t at = 0; have < (uint32_t)p.k && at < p.vocab; at += THREADS) {
        const float v = at + tid < p.vocab ? p.x[(size_t)row * p.stride + at + tid] : 0.f;
        const bool none = at + tid < p.vocab && (v != v || v == -INFINITY);
        const u64 which = __ballot(none);
        __syncthreads();
        if (lane == 0) taken[wave] = (uint32_t)__popcll(which);
        __syncthreads();
        uint32_t rank = have + (uint32_t)__popcll(which & ((1ull << lane) - 1)), all = 0;
        for (int i = 0; i < THREADS / 64; i++) rank += i < wave ? taken[i] : 0u, all += taken[i];
        if (none && rank < (uint32_t)p.k) put_best(p, row, (int)rank, at + tid, -INFINITY, largest, log_s);
        have += all;
    }
}

// A workgroup per slice of 256 V logits.  Its k best are of the finite ones alone.  WHOLE: the slice is the row.
template <int V, bool WHOLE> __global__ void __launch_bounds__(kThreads) logprobs_slice_kernel(TokenLogprobs p, LogprobsWork w) {
    __shared__ __align__(16) u64 candidates[kCandidates];
    __shared__ u64 best[4];
    __shared__ double sums[2][4];
    __shared__ float rows[16], quads[64];
    __shared__ uint32_t counts[4];
    __shared__ int found[4], ranks[64];
    const uint32_t row = blockIdx.x / w.slices, slice = blockIdx.x % w.slices, first = slice * w.logits;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const float *x = p.x + (size_t)row * p.stride + first;
    const uint32_t n = min(w.logits, p.vocab - first);
    uint32_t token = 0;
    float given = 0.f;
    if (WHOLE && wave == 0) {
        token = p.tokens[row];
        if (token < p.vocab) given = x[token];
    }
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
    float own = -INFINITY;  // (fmaxf passes over NaN)
#pragma unroll
    for (int j = 0; j < V; j++) own = fmaxf(own, v[j]);
    // A value that k logits reach: up to 12 the k-th largest of the 16 rows' (of 16 lanes) largest, up to 48 that of the
    // 64 quads' largest, past that the least of the rows' ceil(k / 16)-th.  (The finer, the fewer candidates and the more to
    // compare.  33 x 128256 logits, by rows and by quads: 12 tokens 10.3 and 11.3 us, 16 tokens 12.0 and 11.4; the last
    // leaves 50 to 140 candidates: 20 tokens 14.5 us, 50 tokens 22.)
    const float row_top = row_max(own);
    const bool by_quads = p.k > 12 && p.k <= 48;
    if (lane % 16 == 0) rows[wave * 4 + lane / 16] = row_top;
    if (by_quads) {
        const float quad = quad_max(own);
        if (lane % 4 == 0) quads[wave * 16 + lane / 4] = quad;
    } else if (p.k > 48) {
        const float low = -row_max(above_in_row(own) < (p.k + 15) / 16 ? -own : -INFINITY);
        if (lane % 16 == 0) quads[wave * 4 + lane / 16] = low;
    }
    if (tid < 64) ranks[tid] = 0;
    __syncthreads();
    const float of_row = rows[lane % 16], top = row_max(of_row);
    float least = -INFINITY;
    if (by_quads) {
        const float quad = quads[lane];
        int above = 0;
#pragma unroll
        for (int i = 0; i < 64; i++) above += __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(quad), i)) > quad;
        least = -wave_max_f32(above < p.k ? -quad : -INFINITY);
    } else if (p.k > 48) {
        least = -row_max(-quads[lane % 16]);
    } else if (p.k) {
        least = -row_max(above_in_row(of_row) < p.k ? -of_row : -INFINITY);
    }
    least = fmaxf(least, -3.402823466e38f);  // finite ones (all of them where a row has none)
    constexpr int EACH = kCandidates / 4;
    int have = 0;  // of this wavefront
    if (p.k && __any(own >= least)) {
#pragma unroll
        for (int j = 0; j < V; j++) {
            const u64 which = __ballot(v[j] >= least);
            if (!which) continue;
            const int to = have + __popcll(which & ((1ull << lane) - 1));
            if (v[j] >= least && to < EACH) candidates[wave * EACH + to] = key_of(v[j], first + at(j));
            have += __popcll(which);
        }
    }
    if (lane == 0) found[wave] = have;
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
        t += (double)((fmaf(e[0], d[0], e[1] * d[1]) + fmaf(e[2], d[2], e[3] * d[3])) +
                      (fmaf(e[4], d[4], e[5] * d[5]) + fmaf(e[6], d[6], e[7] * d[7])));
    }
    s = team_sum(s, 64), t = team_sum(t, 64);
    count = running_sum(count);
    if (lane == 63) sums[0][wave] = s, sums[1][wave] = t, counts[wave] = count;
    __syncthreads();
    const size_t out = (size_t)row * w.slices + slice;
    const SliceSums all = {top, counts[0] + counts[1] + counts[2] + counts[3], (sums[0][0] + sums[0][1]) + (sums[0][2] + sums[0][3]),
                           (sums[1][0] + sums[1][1]) + (sums[1][2] + sums[1][3])};
    double log_s = 0.0;
    if constexpr (WHOLE) log_s = finish_row(p, row, top, all.s + ((double)all.count - 1.0), all.t, token, given, tid == 0);
    else if (tid == 0) w.sums[out] = all;
    if (p.k == 0) return;
    auto put = [&](int rank, u64 key) {
        if constexpr (WHOLE) put_best(p, row, rank, index_of_key(key), value_of_key(key), top, log_s);
        else w.top[out * p.k + rank] = key;
    };
    const int c0 = found[0], c1 = c0 + found[1], c2 = c1 + found[2], c = c2 + found[3];
    // the i-th of the wavefronts' candidates
    auto candidate = [&](int i) { return candidates[i < c0 ? i : i < c1 ? EACH + i - c0 : i < c2 ? 2 * EACH + i - c1 : 3 * EACH + i - c2]; };
    if (max(max(found[0], found[1]), max(found[2], found[3])) <= EACH) {
        if constexpr (WHOLE) put_others<kThreads>(p, row, (uint32_t)c, top, log_s, counts);
        else for (int i = c + tid; i < p.k; i += kThreads) put(i, 0);  // (fewer than that)
        if (c <= 64) {  // a lane each, every wavefront against its own
            const u64 mine = lane < c ? candidate(lane) : 0ull;
            int rank = 0;
            for (int j = 0; j < found[wave]; j += 4) {
                u64 o[4];
#pragma unroll
                for (int e = 0; e < 4; e++) o[e] = candidates[wave * EACH + min(j + e, EACH - 1)];
#pragma unroll
                for (int e = 0; e < 4; e++) rank += j + e < found[wave] && o[e] > mine;
            }
            atomicAdd(&ranks[lane], rank);
            __syncthreads();
            if (wave == 0 && lane < c && ranks[lane] < p.k) put(ranks[lane], mine);
            return;
        }
        for (int i = tid; i < c; i += kThreads) {
            const u64 mine = candidate(i);
            int rank = 0;
            for (int q = 0; q < 4; q++)
                for (int j = 0; j < found[q]; j += 8) {
                    ulonglong2 o[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) o[e] = *reinterpret_cast<const ulonglong2 *>(candidates + q * EACH + j + 2 * e);
#pragma unroll
                    for (int e = 0; e < 4; e++) rank += (j + 2 * e < found[q] && o[e].x > mine) + (j + 2 * e + 1 < found[q] && o[e].y > mine);
                }
            if (rank < p.k) put(rank, mine);
        }
        return;
    }
    // many are equal, or the best crowd a few rows of lanes: one after the other
    u64 last = ~0ull;
    int i = 0;
    for (; i < p.k; i++) {
        u64 k = 0;
#pragma unroll
        for (int j = 0; j < V; j++) {
            const u64 o = key_of(v[j], first + at(j));
            if (v[j] >= least && o > k && o < last) k = o;
        }
        k = wave_max_key(k);
        __syncthreads();
        if (lane == 0) best[wave] = k;
        __syncthreads();
        last = max(max(best[0], best[1]), max(best[2], best[3]));
        if (WHOLE && last == 0) break;
        if (tid == 0) put(i, last);
    }
    if constexpr (WHOLE) put_others<kThreads>(p, row, (uint32_t)i, top, log_s, counts);
}

// A workgroup per row: the last wavefront joins the slices' sums, a lane each, while the others find the best.
constexpr int kRowThreads = 512, kLists = 7;
__global__ void __launch_bounds__(kRowThreads) logprobs_row_kernel(TokenLogprobs p, LogprobsWork w) {
    __shared__ __align__(16) u64 heads[kLists][kMaxSlices], candidates[kTop * kMaxSlices];
    __shared__ uint32_t taken[kRowThreads / 64];
    __shared__ u64 limits[kLists];
    __shared__ double shared_log;
    __shared__ float shared_largest;
    __shared__ int found;
    const uint32_t row = blockIdx.x, n = w.slices;
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const u64 *top = w.top + (size_t)row * n * p.k;
    if (tid == 0) found = 0;
    // For each j of 1, 2, 4 .. k: of the slices' j-th best the ceil(k / j)-th largest is a value that k logits reach.
    const int j = 1 << wave;
    if (wave < kLists && p.k) {
        const u64 mine = (uint32_t)lane < n && j <= p.k ? top[(size_t)lane * p.k + j - 1] : 0ull;
        if (lane == 0) limits[wave] = 1;
        heads[wave][lane] = mine;
        wave_fence();
        int rank = 0;
        for (uint32_t o = 0; o < n; o += 8) {  // (those behind the last are 0)
            ulonglong2 other[4];
#pragma unroll
            for (int e = 0; e < 4; e++) other[e] = *reinterpret_cast<const ulonglong2 *>(&heads[wave][o + 2 * e]);
#pragma unroll
            for (int e = 0; e < 4; e++) rank += (other[e].x > mine) + (other[e].y > mine);
        }
        if (mine && rank == (p.k + j - 1) / j - 1) limits[wave] = mine;
    }
    SliceSums own{-INFINITY, 0, 0.0, 0.0};
    float given = 0.f;
    uint32_t token = 0;
    if (wave == kLists) {
        token = p.tokens[row];
        if ((uint32_t)lane < n) own = w.sums[(size_t)row * n + lane];
        if (token < p.vocab) given = p.x[(size_t)row * p.stride + token];
    }
    __syncthreads();
    if (wave < kLists && p.k) {
        u64 least = 1;
#pragma unroll
        for (int g = 0; g < kLists; g++) least = max(least, limits[g]);
        // a slice's are in order: eight lanes take a slice until one falls below
        for (uint32_t a = (uint32_t)tid / 8; a < n; a += 64 * kLists / 8)
            for (int b = tid & 7; b < p.k; b += 8) {
                const u64 k = top[(size_t)a * p.k + b];
                if (k < least) break;
                candidates[atomicAdd(&found, 1)] = k;
            }
    }
    if (wave == kLists) {  // meanwhile the sums
        const float largest = wave_max_f32(own.top);
        // slices that have the largest give its count, the others their weights
        double s = own.s, t = own.t, count = own.top == largest ? (double)own.count : 0.0;
        if (own.top != largest) {
            const double d = fmax((double)own.top - (double)largest, -1000.0), f = exp(d), all = own.count + own.s;
            s = f * all, t = f * (own.t + d * all);
        }
        s = team_sum(s, 64) + (team_sum(count, 64) - 1.0), t = team_sum(t, 64);
        const double log_s = finish_row(p, row, largest, s, t, token, given, lane == 0);
        if (lane == 0) shared_log = log_s, shared_largest = largest;
    }
    if (p.k == 0) return;
    __syncthreads();
    const double log_s = shared_log;
    const float largest = shared_largest;
    place(candidates, found, p.k, [&](int rank, u64 k) { put_best(p, row, rank, index_of_key(k), value_of_key(k), largest, log_s); });
    put_others<kRowThreads>(p, row, (uint32_t)found, largest, log_s, taken);
}

}  // namespace

hipError_t launch_token_logprobs(const TokenLogprobs &a, int cus, hipStream_t s) {
    // The fewer workgroups the rows make, the smaller their slices.  (Of 4096 logits and of 8192: a row of 151936 4.7 us and
    // 5.5, 8 rows 6.3 and 6.8, 33 of 128256 12.0 and 10.8, 511 of 151936 67 and 57.)
    // A row that is one slice needs no second launch (200 rows of 1500 logits, 20 tokens: 6.3 us, with it 5.9 and 4.1).
    const bool whole = a.vocab <= 8192;
    const uint32_t slice = a.vocab <= 4096 || (!whole && (uint64_t)a.rows * ((a.vocab + 4095) / 4096) <= 2ull * cus) ? 4096 : 8192;
    LogprobsWork w{};
    w.slices = (a.vocab + slice - 1) / slice;
    w.logits = ((a.vocab + w.slices - 1) / w.slices + 3) / 4 * 4;  // alike, so that the last one's lanes aren't mostly empty
    w.slices = (a.vocab + w.logits - 1) / w.logits;
    const size_t each = w.slices * (sizeof(SliceSums) + 8 * (size_t)a.k);
    // as many rows at a time as the workspace holds; rows that are one slice need none of it, but a launch has less than 2^32 threads
    const uint32_t most = whole ? 0xFFFFFFFFu / kThreads : (uint32_t)std::min<size_t>(a.work_bytes / each, 0x7FFFFFFFu / w.slices);
    TokenLogprobs p = a;
    for (uint32_t r = 0; r < a.rows; r += p.rows) {
        p.rows = std::min(a.rows - r, most);
        p.x = a.x + (size_t)r * a.stride, p.tokens = a.tokens + r, p.out = a.out + r;
        p.entropy = a.entropy ? a.entropy + r : nullptr;
        if (a.k) p.top = a.top + (size_t)r * a.k, p.top_tokens = a.top_tokens + (size_t)r * a.k;
        w.sums = (SliceSums *)a.work, w.top = (u64 *)(w.sums + (size_t)p.rows * w.slices);
        const dim3 grid(p.rows * w.slices);
        if (whole) {
            if (slice == 8192) hipLaunchKernelGGL((logprobs_slice_kernel<32, true>), grid, dim3(kThreads), 0, s, p, w);
            else hipLaunchKernelGGL((logprobs_slice_kernel<16, true>), grid, dim3(kThreads), 0, s, p, w);
            continue;
        }
        if (slice == 8192) hipLaunchKernelGGL((logprobs_slice_kernel<32, false>), grid, dim3(kThreads), 0, s, p, w);
        else hipLaunchKernelGGL((logprobs_slice_kernel<16, false>), grid, dim3(kThreads), 0, s, p, w);
        hipLaunchKernelGGL(logprobs_row_kernel, dim3(p.rows), dim3(kRowThreads), 0, s, p, w);
    }
    return hipGetLastError();
}

}  // namespace zh

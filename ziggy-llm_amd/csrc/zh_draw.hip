// zh_draw.hip -- sampling from the logits on the device: temperature, top-k, top-p, min-p and repeat
// penalty, with given random numbers.
//
// Every limit keeps a beginning of the candidates in some order, and the draw is the first candidate
// whose running sum reaches a target.  Weights are exp((a - max) / T) in 64 bits, rounded to integers
// of 2^-s, so that sums are exact whatever their order and a row's token depends on its inputs alone.
//
// Three launches, none of which sorts the row:
//   stats   slices of 2048 logits: maximum, minimum and mean, from which a linear scale of 256 bins
//           is laid over the values, the largest in bin 0;
//   bins    per slice the bins' sums of weights (with top-k, which comes first: counts of the logits that may
//           have a weight), and its logits in the order of their bins;
//   finish  a workgroup per row: the bin in which a target lies, then 1024 finer bins of that bin's
//           logits, then the few logits of the finer bin in order.  With top-k the bins above the k-th
//           logit are sorted instead (in registers; through LDS what lies in different wavefronts), and
//           everything else is prefix sums of at most 1024.
// What is left of a row at the end, up to 64 logits, is a wavefront's work without a barrier.  Where a
// finer bin holds more than 1024 logits, equal ones or nearly, their values go digit by digit, and equal
// ones by the counts of their slices.  (128256 logits rounded to quarters, nucleus of 0.9: 29 us; all
// equal: 0.51 ms, top-k 0.31.)
//
// What bounds it: three dependent launches, each a chain of memory round trips, barriers and LDS.  One row
// of 128256 logits, top-k 40 of 0.9: 16.2 us a pass (the launches' least of 60: 1.8, 5.4 and 6.1); 16 rows of 151936,
// nucleus of 0.95: 23.7 (3.0, 6.2 and 12.9; the logits' 9.7 MB are 2.1 us of it).  Of the finish, 3 us were barriers
// of 16 wavefronts in the sums and sorts that a wavefront does now, 2 the tables of all bins where a top-k
// lies in the first quarter.  A row whole in one workgroup, in one launch: 42 us at 32000 logits, these 21.
#include "zh_longctx.h"

namespace zh {

namespace {

constexpr int kSliceLogits = 2048, kBins = 256, kFine = 1024, kThreads = 1024, kMaxSlices = 262144 / kSliceLogits;

typedef unsigned long long u64;

// a row's part of the workspace
struct RowHead {
    float max, per_bin;  // of the binned logits; bins per unit
};
struct SliceStats {
    float max, min, sum, count;  // of what is finite and no mask (above -1e30)
};
__host__ __device__ constexpr size_t up256(size_t n) { return (n + 255) / 256 * 256; }
__host__ __device__ constexpr uint32_t slices_of(uint32_t vocab) { return (vocab + kSliceLogits - 1) / kSliceLogits; }
__host__ __device__ constexpr size_t row_bytes(uint32_t vocab) {
    return 256 + up256(slices_of(vocab) * sizeof(SliceStats)) +
           slices_of(vocab) * (kBins * (sizeof(u64) + 4) + sizeof(u64) + kSliceLogits * (sizeof(float) + 2)) + 256;
}
struct RowWork {
    RowHead *head;
    SliceStats *stats;
    u64 *sums;       // [slice][kBins] (without top-k)
    uint32_t *run;   // [slice][kBins]: where the bin's logits begin in the slice's order, and (high half) end
    float *value;    // [slice][kSliceLogits], in the order of their bins
    uint16_t *from;  // [slice][kSliceLogits]: of which logit of the slice
    u64 *whole;      // [slice]
};
__device__ __forceinline__ RowWork row_work(const SampleRows &p, uint32_t row) {
    char *at = (char *)p.work + row * up256(row_bytes(p.vocab));
    RowWork w;
    const uint32_t n = slices_of(p.vocab);
    w.head = (RowHead *)at, at += 256;
    w.stats = (SliceStats *)at, at += up256(n * sizeof(SliceStats));
    w.sums = (u64 *)at, at += (size_t)n * kBins * sizeof(u64);
    w.value = (float *)at, at += (size_t)n * kSliceLogits * sizeof(float);
    w.run = (uint32_t *)at, at += (size_t)n * kBins * 4;
    w.from = (uint16_t *)at, at += (size_t)n * kSliceLogits * 2;
    w.whole = (u64 *)at;
    return w;
}

// float -> an integer that orders as it does; NaN as -infinity, the zeros equal
__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t b = __float_as_uint(v != v ? -INFINITY : v + 0.f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) { return __uint_as_float((o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o); }

__device__ __forceinline__ float penalised(float v, float r) { return v < 0.f ? v * r : v / r; }

// What a row's limits come to.
struct Policy {
    bool limited, sorted;
    uint32_t top_k;
    double per_t, least, unit;  // unit 2^s
    float none;                 // exponents below it surely come to a weight of 0
    __device__ explicit Policy(const SampleRows &p) {
        top_k = p.o.top_k == 0 ? p.vocab : min(p.o.top_k, p.vocab);
        limited = top_k < p.vocab, sorted = p.o.top_p < 1.f;
        per_t = 1.0 / (double)p.o.temperature, least = (double)p.o.min_p;
        const int bits = top_k > 1 ? 32 - __clz((int)top_k - 1) : 0;
        unit = __longlong_as_double((long long)(1023 + 62 - bits) << 52);
        none = fmaxf(logf(p.o.min_p), -0.6931472f * (float)(63 - bits)) - 0.01f;
    }
    // With top-k: logits below it have a weight of 0, penalised or not, and are no candidates.  (The largest weight's
    // logit is at least the largest logit penalised; a penalty raises none.)
    __device__ float least_logit(const SampleRows &p, float largest) const {
        const float base = p.recent ? penalised(largest, p.o.repeat_penalty) : largest;
        return base + 1.001f * none * p.o.temperature - 1e-6f * fabsf(base);
    }
    // (the same operations wherever it is called: the sums of the bins and of their logits agree)
    __device__ __forceinline__ u64 weight(float a, float mx) const {
#pragma clang fp contract(off)
        const double x = ((double)a - (double)mx) * per_t;
        if (!(x > (double)none)) return 0;  // (-infinity, NaN too)
        const double e = exp(x);
        return e >= least ? (u64)rint(e * unit) : 0;
    }
};

__device__ __forceinline__ int bin_of(float a, float mx, float per_bin, float &t) {
    t = fmaxf((mx - a) * per_bin, 0.f);  // (0 times infinity: 0)
    return (int)fminf(t, (float)(kBins - 1));
}
__device__ __forceinline__ int fine_of(float t, int bin) {
    return (int)fminf(fmaxf((t - (float)bin) * (float)kFine, 0.f), (float)(kFine - 1));
}

// The bits of the row's recent tokens with ids first .. first + 32 words - 1, into LDS.
__device__ __forceinline__ void mark_recent(const SampleRows &p, uint32_t row, uint32_t *bits, uint32_t words, uint32_t first) {
    constexpr int N = 4;  // of a thread under way at once
    const uint32_t *recent = p.recent + (size_t)row * p.recent_count;
    uint32_t id[N];
    auto load = [&](size_t i) {
#pragma unroll
        for (int k = 0; k < N; k++) {
            id[k] = 0xFFFFFFFFu;
            if (i + k * blockDim.x < p.recent_count) id[k] = recent[i + k * blockDim.x];
        }
    };
    load(threadIdx.x);
    for (uint32_t i = threadIdx.x; i < words; i += blockDim.x) bits[i] = 0;
    __syncthreads();
    for (size_t i = threadIdx.x;;) {
#pragma unroll
        for (int k = 0; k < N; k++)
            if (id[k] < p.vocab && id[k] >= first && id[k] - first < 32 * words) atomicOr(&bits[(id[k] - first) / 32], 1u << (id[k] % 32));
        if ((i += N * blockDim.x) >= p.recent_count) break;
        load(i);
    }
    __syncthreads();
}

// The logits that the bins order: penalised, or, with top-k (which comes first), as they are.
struct Slice {
    uint32_t first, n;
    float a[kSliceLogits / 256];
    __device__ Slice(const SampleRows &p, uint32_t row, bool penalise, uint32_t *bits) {
        first = blockIdx.x * kSliceLogits, n = min(p.vocab - first, (uint32_t)kSliceLogits);
        const float *x = p.x + row * p.stride + first;
#pragma unroll
        for (int i = 0; i < kSliceLogits / 256; i++) {
            const uint32_t j = threadIdx.x + 256 * i;
            const float v = x[min(j, n - 1)];
            a[i] = j < n && v == v ? v : -INFINITY;
        }
        if (!penalise) return;
        mark_recent(p, row, bits, kSliceLogits / 32, first);
#pragma unroll
        for (int i = 0; i < kSliceLogits / 256; i++) {
            const uint32_t j = threadIdx.x + 256 * i;
            if (bits[j / 32] >> (j % 32) & 1u) a[i] = penalised(a[i], p.o.repeat_penalty);
        }
    }
};

// Inclusive prefix sum over the wavefront on the vector ALU: within rows of 16 by row shifts, then the
// rows' ends broadcast to the rows behind.
template <int CTRL, int ROWS> __device__ __forceinline__ u64 add_dpp(u64 v) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xF, false);
    return v + ((u64)hi << 32 | lo);
}
__device__ __forceinline__ u64 wave_prefix(u64 v) {
    v = add_dpp<0x111, 0xF>(v);  // row_shr:1, 2, 4, 8 (lanes before the row's start: 0)
    v = add_dpp<0x112, 0xF>(v);
    v = add_dpp<0x114, 0xF>(v);
    v = add_dpp<0x118, 0xF>(v);
    v = add_dpp<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
    return add_dpp<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
}
// The sum over the wavefront, in every lane.
__device__ __forceinline__ float wave_sum(float v) {
    auto add = [&](auto ctrl) {
        v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xF, 0xF, false));
    };
    add(std::integral_constant<int, 0xB1>{});
    add(std::integral_constant<int, 0x4E>{});
    add(std::integral_constant<int, 0x141>{});
    add(std::integral_constant<int, 0x140>{});
    return xsum<32>(xsum<16>(v));
}

__global__ void __launch_bounds__(256) draw_stats_kernel(SampleRows p) {
    __shared__ uint32_t bits[kSliceLogits / 32];
    __shared__ float4 red[4];
    const uint32_t row = blockIdx.y;
    const Slice s(p, row, p.recent && !Policy(p).limited, bits);
    float mx = -INFINITY, mn = INFINITY, sum = 0.f, count = 0.f;
#pragma unroll
    for (int i = 0; i < kSliceLogits / 256; i++) {
        mx = fmaxf(mx, s.a[i]);
        if (s.a[i] > -1e30f && s.a[i] < INFINITY) mn = fminf(mn, s.a[i]), sum += s.a[i], count += 1.f;
    }
    mx = wave_max_f32(mx), mn = -wave_max_f32(-mn), sum = wave_sum(sum), count = wave_sum(count);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = make_float4(mx, mn, sum, count);
    __syncthreads();
    if (threadIdx.x) return;
    for (int w = 1; w < 4; w++) mx = fmaxf(mx, red[w].x), mn = fminf(mn, red[w].y), sum += red[w].z, count += red[w].w;
    row_work(p, row).stats[blockIdx.x] = SliceStats{mx, mn, sum, count};
}

__global__ void __launch_bounds__(256) draw_bins_kernel(SampleRows p) {
    __shared__ uint32_t bits[kSliceLogits / 32];
    __shared__ float4 all[kMaxSlices];
    __shared__ u64 sums[kBins], red[4];
    __shared__ uint32_t count[kBins], begin[kBins], wave_count[4];
    __shared__ float value[kSliceLogits];
    __shared__ uint16_t from[kSliceLogits];
    const uint32_t row = blockIdx.y, slices = slices_of(p.vocab);
    const RowWork w = row_work(p, row);
    const Policy policy(p);
    if (threadIdx.x < slices) all[threadIdx.x] = *reinterpret_cast<const float4 *>(w.stats + threadIdx.x);
    sums[threadIdx.x] = 0, count[threadIdx.x] = 0;
    const Slice s(p, row, p.recent && !policy.limited, bits);
    __syncthreads();
    float mx = -INFINITY, mn = INFINITY, sum = 0.f, known = 0.f;
    for (uint32_t i = threadIdx.x & 63; i < slices; i += 64)
        mx = fmaxf(mx, all[i].x), mn = fminf(mn, all[i].y), sum += all[i].z, known += all[i].w;
    mx = wave_max_f32(mx), mn = -wave_max_f32(-mn), sum = wave_sum(sum), known = wave_sum(known);
    // the scale: with top-k down to the mean, or to where weights are surely 0 (which a logit of -10000 or one far
    // above the others would take the mean past); else to the lowest, or to where weights are 0, or, where few lie
    // far below the others, as far below the mean as half again the largest is above it
    const float above = mx - sum / known, least = policy.limited ? policy.least_logit(p, mx) : -INFINITY;
    float range = policy.limited ? fminf(above, mx - least) : fminf(fminf(43.7f * p.o.temperature, mx - mn), 2.5f * above);
    const float per_bin = range > 0.f && fabsf(mx) < INFINITY ? (float)kBins / range : 0.f;
    if (blockIdx.x == 0 && threadIdx.x == 0) w.head->max = mx, w.head->per_bin = per_bin;
    const bool ordering = policy.limited || policy.sorted;  // else the draw goes by the ids: the slice's sum is all
    u64 whole = 0;
    uint32_t at[kSliceLogits / 256];  // bin, and the logit's place in it (in no order: their sums are exact)
#pragma unroll
    for (int i = 0; i < kSliceLogits / 256; i++) {
        float t;
        const int b = bin_of(s.a[i], mx, per_bin, t);
        const u64 v = !(fabsf(mx) < INFINITY) ? 0ull : policy.limited ? (s.a[i] > -INFINITY && s.a[i] >= least ? 1ull : 0ull) : policy.weight(s.a[i], mx);
        at[i] = 0xFFFFFFFFu;  // no candidate: in no bin
        if (v && ordering) {
            if (!policy.limited) atomicAdd(&sums[b], v);
            at[i] = (uint32_t)b << 16 | atomicAdd(&count[b], 1u);
        }
        whole += v;
    }
    whole = wave_prefix(whole);
    if ((threadIdx.x & 63) == 63) red[threadIdx.x >> 6] = whole;
    __syncthreads();
    if (threadIdx.x == 0) w.whole[blockIdx.x] = red[0] + red[1] + red[2] + red[3];
    if (!ordering) return;
    const uint32_t mine = count[threadIdx.x];
    uint32_t upto = (uint32_t)wave_prefix(mine);
    if ((threadIdx.x & 63) == 63) wave_count[threadIdx.x >> 6] = upto;
    __syncthreads();
    for (uint32_t k = 0; k < threadIdx.x >> 6; k++) upto += wave_count[k];
    begin[threadIdx.x] = upto - mine;
    const size_t slice = blockIdx.x;
    w.run[slice * kBins + threadIdx.x] = (upto - mine) | upto << 16;
    if (!policy.limited) w.sums[slice * kBins + threadIdx.x] = sums[threadIdx.x];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSliceLogits / 256; i++)
        if (at[i] != 0xFFFFFFFFu) {
            const uint32_t to = begin[at[i] >> 16] + (at[i] & 0xFFFFu);
            value[to] = s.a[i], from[to] = (uint16_t)(threadIdx.x + 256 * i);
        }
    __syncthreads();
    const uint32_t held = wave_count[0] + wave_count[1] + wave_count[2] + wave_count[3];
    for (uint32_t i = threadIdx.x; i < held; i += 256)
        w.value[slice * kSliceLogits + i] = value[i], w.from[slice * kSliceLogits + i] = from[i];
}

// ---- finish: a workgroup of 1024 per row ----

struct Finish {
    u64 list[2 * kThreads];       // logits' keys; the bins' sums of several slices; keys being sorted
    u64 sums[kFine];              // the fine bins' sums
    u64 runs[kBins];              // the bins' running sums
    u64 wave[kThreads / 64];
    uint32_t seen[262144 / 32];   // recent tokens
    u64 value, key;
    uint32_t found, count, least, most;
};

// Inclusive prefix sum over the workgroup; *total: the whole.
__device__ u64 prefix(Finish &f, u64 v, u64 *total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    v = wave_prefix(v);
    __syncthreads();
    if (lane == 63) f.wave[wave] = v;
    __syncthreads();
    u64 before = 0, all = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 64; i++) {
        const u64 w = f.wave[i];
        before += i < wave ? w : 0;
        all += w;
    }
    *total = all;
    return v + before;
}
// The thread whose running sum `run` (of its own v) reaches target, 1 .. the whole sum; *before: the sum
// ahead of it.
__device__ uint32_t first_reaching(Finish &f, u64 run, u64 v, u64 target, u64 *before) {
    __syncthreads();
    if (v && run >= target && run - v < target) f.found = threadIdx.x, f.value = run - v;
    __syncthreads();
    *before = f.value;
    return f.found;
}

// The two in one: the thread at which the running sum of v reaches target.
__device__ uint32_t reach(Finish &f, u64 v, u64 target, u64 *before) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    u64 run = wave_prefix(v);
    if (lane == 63) f.wave[wave] = run;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 64 - 1; i++) run += i < wave ? f.wave[i] : 0;
    if (v && run >= target && run - v < target) f.found = threadIdx.x, f.value = run - v;
    __syncthreads();
    *before = f.value;
    return f.found;
}

__device__ u64 target_of(double share, u64 total) {
    const double t = ceil(share * (double)total);
    const u64 c = t >= 1.0 ? (u64)t : 1ull;
    return c < total ? c : total;
}

// The keys of lanes 0 .. n - 1 of the first wavefront (they differ) in descending order, 0 in the lanes
// behind: a key's place is the count of larger ones.  Takes f.list's first 64 places.
__device__ __forceinline__ u64 wave_sorted(Finish &f, u64 key, uint32_t n) {
    constexpr int N = 16;
    const uint32_t lane = threadIdx.x;
    f.list[lane] = lane < n ? key : 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    uint32_t place = 0;
    for (uint32_t i = 0; i < n; i += N) {
        u64 other[N];
#pragma unroll
        for (int j = 0; j < N; j++) other[j] = f.list[i + j];
#pragma unroll
        for (int j = 0; j < N; j++) place += other[j] > key;
    }
    const int to = 4 * (int)(lane < n ? place : lane);
    const u64 r = (u64)(uint32_t)__builtin_amdgcn_ds_permute(to, (int)(key >> 32)) << 32 | (uint32_t)__builtin_amdgcn_ds_permute(to, (int)key);
    return lane < n ? r : 0;
}

// The larger or the smaller of a key and that of the lane whose number differs in bit S.
template <int S> __device__ __forceinline__ u64 exchanged(u64 key, bool larger) {
    u64 a = key, b;
    if constexpr (S >= 4) {
        uint32_t al, bl, ah, bh;
        lane_pair<1 << S>((uint32_t)key, al, bl), lane_pair<1 << S>((uint32_t)(key >> 32), ah, bh);
        a = (u64)ah << 32 | al, b = (u64)bh << 32 | bl;
    } else if constexpr (S == 3) {
        b = dpp_u64<0x128>(key);  // row_ror:8
    } else if constexpr (S == 2) {
        b = dpp_u64<0x1B>(dpp_u64<0x141>(key));  // lane ^ 7, then ^ 3
    } else {
        b = dpp_u64<S == 1 ? 0x4E : 0xB1>(key);
    }
    return (a > b) == larger ? a : b;
}

// The workgroup's keys in descending order, thread i the i-th: n keys that differ, of threads 0 .. n - 1, 0
// behind.  A bitonic sort: in registers up to 32 lanes apart, through LDS beyond.
__device__ u64 sorted(Finish &f, u64 key, uint32_t n) {
    const uint32_t tid = threadIdx.x;
    if (tid >= n) key = 0;
    uint32_t steps = 6, half = 0;
    while (1u << steps < n) steps++;
    for (uint32_t r = 1; r <= steps; r++) {
        const uint32_t down = tid >> r;  // bit 0: whether this block ascends
        for (uint32_t s = r - 1; s >= 6 && s < r; s--) {
            f.list[half + tid] = key;
            __syncthreads();
            const u64 o = f.list[half + (tid ^ 1u << s)];
            half ^= kThreads;
            key = (key > o) == (((tid >> s ^ down) & 1) == 0) ? key : o;
        }
        auto larger = [&](int s) { return ((tid >> s ^ down) & 1) == 0; };
        switch (r < 6 ? r : 6) {
        case 6: key = exchanged<5>(key, larger(5)); [[fallthrough]];
        case 5: key = exchanged<4>(key, larger(4)); [[fallthrough]];
        case 4: key = exchanged<3>(key, larger(3)); [[fallthrough]];
        case 3: key = exchanged<2>(key, larger(2)); [[fallthrough]];
        case 2: key = exchanged<1>(key, larger(1)); [[fallthrough]];
        default: key = exchanged<0>(key, larger(0));
        }
    }
    return key;
}

// The id of the first of the largest of logits begin .. end - 1.
template <class V> __device__ uint32_t first_of_largest(Finish &f, uint32_t begin, uint32_t end, V value) {
    u64 k = 0;
    for (uint32_t i = begin + threadIdx.x; i < end; i += kThreads) {
        const u64 c = (u64)ordered(value(i)) << 32 | (uint32_t)~i;
        k = c > k ? c : k;
    }
    k = wave_max_key(k);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) f.wave[threadIdx.x >> 6] = k;
    __syncthreads();
    for (int j = 0; j < kThreads / 64; j++) k = f.wave[j] > k ? f.wave[j] : k;
    return ~(uint32_t)k;
}

// The row's logits of bins first .. last, 8 lanes a slice: the first 64 of a slice in registers, the
// others read again each time.
struct OfBins {
    static constexpr int N = 8;
    const float *value;
    const uint16_t *from;
    uint32_t base, begin, end;
    float a[N];
    uint32_t id[N];
    __device__ __forceinline__ OfBins(const RowWork &w, uint32_t slices, uint32_t first, uint32_t last) {
        const uint32_t slice = threadIdx.x / 8;
        base = slice * kSliceLogits, begin = end = 0;
        value = w.value + base, from = w.from + base;
        if (slice < slices) begin = (w.run[slice * kBins + first] & 0xFFFFu) + threadIdx.x % 8, end = w.run[slice * kBins + last] >> 16;
        if (begin < end) load(begin);
    }
    __device__ __forceinline__ void load(uint32_t e) {
#pragma unroll
        for (int k = 0; k < N; k++) {
            const uint32_t at = min(e + 8 * k, end - 1);
            a[k] = value[at], id[k] = from[at];
        }
    }
    // take(logit, its id) of each
    template <class T> __device__ __forceinline__ void each(T take) {
        for (uint32_t e = begin; e < end; e += 8 * N) {
            if (end - begin > 8 * N) load(e);
#pragma unroll
            for (int k = 0; k < N; k++)
                if (e + 8 * k < end) take(a[k], base + id[k]);
        }
    }
};
static_assert(kThreads / 8 >= kMaxSlices, "8 lanes for every slice");

__global__ void __launch_bounds__(kThreads) draw_finish_kernel(SampleRows p) {
    __shared__ Finish f;
    const uint32_t row = blockIdx.x, n = p.vocab, tid = threadIdx.x;
    const float *x = p.x + row * p.stride;
    auto answer = [&](uint32_t id) {
        if (tid == 0) p.out[row] = id;
    };
    const RowWork w = row_work(p, row);
    if (p.o.temperature <= 0.f) {  // the first slice with the largest logit
        auto key = [&](uint32_t slice) { return slice < slices_of(n) ? (u64)ordered(w.stats[slice].max) << 32 | (uint32_t)~slice : 0; };
        const u64 a = key(tid & 63), b = key((tid & 63) + 64);
        const uint32_t first = ~(uint32_t)wave_max_key(a > b ? a : b) * kSliceLogits;
        return answer(first_of_largest(f, first, min(first + kSliceLogits, n), [&](uint32_t i) { return x[i]; }));
    }
    const Policy policy(p);
    // the slices' tables of bins, 16 bytes of a slice a thread, under way while the recent tokens are marked: two bins'
    // sums of every eighth slice; with top-k the runs of four of the first quarter's bins of every 64th
    const uint32_t slices = slices_of(n);
    constexpr int kAhead = 12;
    ulonglong2 part[kAhead];
    uint32_t quarters = 0;  // of the bins whose sums are known
    auto load_counts = [&]() {
#pragma unroll
        for (uint32_t k = 0; k < 2; k++) {
            const uint32_t slice = tid / 16 + 64 * k;
            part[k] = make_ulonglong2(0, 0);
            if (slice < slices) part[k] = reinterpret_cast<const ulonglong2 *>(w.run)[slice * 64 + quarters * 16 + tid % 16];
        }
    };
    auto load_sums = [&](uint32_t from) {
#pragma unroll
        for (uint32_t k = 0; k < kAhead; k++) {
            const uint32_t slice = from + tid / 128 + 8 * k;
            part[k] = make_ulonglong2(0, 0);
            if (slice < slices) part[k] = reinterpret_cast<const ulonglong2 *>(w.sums)[slice * 128 + tid % 128];
        }
    };
    static_assert(kMaxSlices <= 128 && kThreads == 1024 && kBins == 256, "a thread's pieces of the tables");
    if (policy.limited) load_counts();
    else if (policy.sorted) load_sums(0);
    const uint32_t lane = tid & 63;
    const u64 mass = (lane < slices ? w.whole[lane] : 0) + (lane + 64 < slices ? w.whole[lane + 64] : 0);
    // (the bins hold penalised logits, but for top-k's)
    if (p.recent) mark_recent(p, row, f.seen, (n + 31) / 32, 0);
    auto logit_of = [&](uint32_t i, float v) {
        return p.recent && (f.seen[i / 32] >> (i % 32) & 1u) ? penalised(v, p.o.repeat_penalty) : v;
    };
    auto logit = [&](uint32_t i) { return logit_of(i, x[i]); };
    const double given = p.uniforms[row], u = given >= 0.0 ? fmin(given, 1.0) : 0.0;
    const float top = w.head->max, per_bin = w.head->per_bin;
    if (!(fabsf(top) < INFINITY))  // no largest number: the first of the largest logits (of the binned ones)
        return answer(first_of_largest(f, 0, n, [&](uint32_t i) { return policy.limited ? x[i] : logit(i); }));

    const u64 mass_upto = wave_prefix(mass);
    u64 total = (u64)(uint32_t)__builtin_amdgcn_readlane((int)(mass_upto >> 32), 63) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)mass_upto, 63), before;
    // f.runs of the loaded bins: their running sums
    auto run_counts = [&]() {
        uint32_t c[4] = {};
#pragma unroll
        for (int k = 0; k < 2; k++) {
            const uint32_t run[4] = {(uint32_t)part[k].x, (uint32_t)(part[k].x >> 32), (uint32_t)part[k].y, (uint32_t)(part[k].y >> 32)};
            for (int j = 0; j < 4; j++) c[j] += (run[j] >> 16) - (run[j] & 0xFFFFu);
        }
        uint32_t *counts = reinterpret_cast<uint32_t *>(f.list);  // [wavefront][64]
        for (int j = 0; j < 4; j++) {
            uint32_t a, b;
            lane_pair<16>(c[j], a, b);
            lane_pair<32>(a + b, a, b);
            c[j] = a + b;
        }
        if (lane < 16) *reinterpret_cast<uint4 *>(counts + (tid & ~63u) + 4 * lane) = make_uint4(c[0], c[1], c[2], c[3]);
        __syncthreads();
        if (tid < 64) {
            uint32_t v = 0;
#pragma unroll
            for (int k = 0; k < kThreads / 64; k++) v += counts[64 * k + tid];
            f.runs[64 * quarters + tid] = wave_prefix(v) + (quarters ? f.runs[64 * quarters - 1] : 0);
        }
        quarters++;
        __syncthreads();
    };
    auto run_sums = [&]() {
        u64 x = 0, y = 0;
        for (uint32_t from = 0;;) {
#pragma unroll
            for (int k = 0; k < kAhead; k++) x += part[k].x, y += part[k].y;
            if ((from += 8 * kAhead) >= slices) break;
            load_sums(from);
        }
        f.list[2 * tid] = x, f.list[2 * tid + 1] = y;  // [8][kBins]
        __syncthreads();
        if (tid < 64) {
            u64 v[4] = {};
#pragma unroll
            for (int k = 0; k < 8; k++)
                for (int j = 0; j < 4; j++) v[j] += f.list[k * kBins + 4 * tid + j];
            v[1] += v[0], v[2] += v[1], v[3] += v[2];
            const u64 ahead = wave_prefix(v[3]) - v[3];
            for (int j = 0; j < 4; j++) f.runs[4 * tid + j] = ahead + v[j];
        }
        quarters = 4;
        __syncthreads();
    };
    // the bin in which the sum reaches target (every wavefront by itself); *ahead: the sum of the bins before
    auto bin_reaching = [&](u64 target, u64 *ahead) {
        uint32_t bin = 0;
        for (uint32_t k = 0; k < quarters; k++) bin += (uint32_t)__popcll(__ballot(f.runs[64 * k + lane] < target));
        *ahead = bin ? f.runs[bin - 1] : 0;
        return (int)bin;
    };

    // The logit at which the sum of weights reaches target, in descending order (equal logits: of ascending ids), as
    // its key, value and complement of the id; *upto: the sum with it.  It lies in the given bin, ahead of which the sum
    // is `ahead`.
    auto find = [&](auto weight, int bin, u64 ahead, u64 target, u64 *upto) {
        u64 fine_ahead;
        f.sums[tid] = 0;  // (each thread's own, until here)
        if (tid == 0) f.count = 0, f.least = 0xFFFFFFFFu, f.most = 0;
        OfBins logits(w, slices, bin, bin);
        __syncthreads();
        logits.each([&](float a, uint32_t) {
            float t;
            bin_of(a, top, per_bin, t);
            atomicAdd(&f.sums[fine_of(t, bin)], weight(a));
        });
        __syncthreads();
        const int fine = (int)reach(f, f.sums[tid], target - ahead, &fine_ahead);
        // take(value, id) for the logits of the finer bin
        auto of_fine = [&](auto take) {
            logits.each([&](float a, uint32_t i) {
                float t;
                bin_of(a, top, per_bin, t);
                if (fine_of(t, bin) == fine) take(ordered(a), i);
            });
        };
        uint32_t lo = 0xFFFFFFFFu, hi = 0;
        of_fine([&](uint32_t o, uint32_t i) {
            lo = min(lo, o), hi = max(hi, o);
            const uint32_t at = atomicAdd(&f.count, 1u);
            if (at < kThreads) f.list[at] = (u64)o << 32 | (uint32_t)~i;
        });
        __syncthreads();
        const uint32_t m = f.count;
        u64 need = target - ahead - fine_ahead, last;
        *upto = ahead + fine_ahead;
        if (m <= 64) {  // by a wavefront
            if (tid < 64) {
                const u64 key = wave_sorted(f, tid < m ? f.list[tid] : 0, m);
                const u64 wt = tid < m ? weight(unordered((uint32_t)(key >> 32))) : 0, run = wave_prefix(wt);
                if (wt && run >= need && run - wt < need) f.value = run, f.key = key;
            }
            __syncthreads();
            *upto += f.value;
            return f.key;
        }
        if (m <= kThreads) {
            const u64 mine = sorted(f, tid < m ? f.list[tid] : 0, m);
            const u64 wt = tid < m ? weight(unordered((uint32_t)(mine >> 32))) : 0;
            if (tid == reach(f, wt, need, &last)) f.key = mine;
            __syncthreads();
            *upto += last + weight(unordered((uint32_t)(f.key >> 32)));
            return f.key;
        }
        // the value: its digits, but for those that all of them share
        atomicMin(&f.least, lo);
        atomicMax(&f.most, hi);
        __syncthreads();
        uint32_t value = f.most;
        const uint32_t differ = f.least ^ f.most;
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (differ >> shift == 0) continue;  // (uniform)
            value = value >> (shift + 8 < 32 ? shift + 8 : 31) >> (shift + 8 < 32 ? 0 : 1);  // the digits above
            __syncthreads();
            f.sums[tid] = 0;
            __syncthreads();
            of_fine([&](uint32_t o, uint32_t) {
                const uint32_t above = shift == 24 ? 0 : o >> (shift + 8);
                if (above == value) atomicAdd(&f.sums[255 - (o >> shift & 255u)], weight(unordered(o)));
            });
            __syncthreads();
            value = (value << 8 | (255 - reach(f, f.sums[tid], need, &last))) << shift;
            need -= last, *upto += last;
        }
        // equal logits: the rank among them, by the slices' counts and then the ids of one slice
        const u64 one = weight(unordered(value)), rank = (need + one - 1) / one;
        __syncthreads();
        f.sums[tid] = 0;
        __syncthreads();
        of_fine([&](uint32_t o, uint32_t i) {
            if (o == value) atomicAdd(&f.sums[i / kSliceLogits], 1ull);
        });
        __syncthreads();
        const uint32_t slice = reach(f, f.sums[tid], rank, &last);
        uint32_t *bits = reinterpret_cast<uint32_t *>(f.list);
        __syncthreads();
        if (tid < kSliceLogits / 32) bits[tid] = 0;
        __syncthreads();
        of_fine([&](uint32_t o, uint32_t i) {
            if (o == value && i / kSliceLogits == slice) atomicOr(&bits[i % kSliceLogits / 32], 1u << (i % 32));
        });
        __syncthreads();
        uint32_t word = tid < kSliceLogits / 32 ? bits[tid] : 0;
        u64 ahead_of_word;
        const uint32_t at = reach(f, __popc(word), rank - last, &ahead_of_word);
        word = bits[at];
        for (u64 k = rank - last - ahead_of_word; k > 1; k--) word &= word - 1;
        *upto += rank * one;
        __syncthreads();
        return (u64)value << 32 | (uint32_t)~(slice * kSliceLogits + 32 * at + (uint32_t)__ffs((int)word) - 1);
    };

    if (policy.limited) {
        const uint32_t k = (uint32_t)(total < policy.top_k ? total : policy.top_k);  // (the binned ones)
        if (tid == 0) f.count = 0;
        for (run_counts(); f.runs[64 * quarters - 1] < k; run_counts()) load_counts();
        const int last = bin_reaching(k, &before);
        OfBins logits(w, slices, 0, last);
        logits.each([&](float v, uint32_t i) {
            const uint32_t at = atomicAdd(&f.count, 1u);
            if (at < kThreads) f.list[at] = (u64)ordered(v) << 32 | (uint32_t)~i;
        });
        __syncthreads();
        uint32_t m = f.count;
        __syncthreads();
        if (m > kThreads) {  // many logits about the k-th: those down to it alone
            u64 upto;
            const u64 end = find([](float) { return 1ull; }, last, before, k, &upto);
            __syncthreads();
            if (tid == 0) f.count = 0;
            __syncthreads();
            logits.each([&](float v, uint32_t i) {
                const u64 key = (u64)ordered(v) << 32 | (uint32_t)~i;
                if (key >= end) f.list[atomicAdd(&f.count, 1u)] = key;
            });
            __syncthreads();
            m = k;
        }
        if (m <= 64) {  // as below, by a wavefront
            if (tid >= 64) return;
            const u64 mine = wave_sorted(f, tid < m ? f.list[tid] : 0, m);
            const bool in = tid < k;
            uint32_t token = ~(uint32_t)mine;
            float b = in ? logit_of(token, unordered((uint32_t)(mine >> 32))) : -INFINITY;
            const u64 key = in ? (u64)ordered(b) << 32 | (uint32_t)~tid : 0, best = wave_max_key(key);
            const float mx = unordered((uint32_t)(best >> 32));
            if (!(fabsf(mx) < INFINITY)) {
                if (tid == ~(uint32_t)best) p.out[row] = token;
                return;
            }
            if (policy.sorted && p.recent) {
                const u64 next = wave_sorted(f, key, k);
                b = in ? unordered((uint32_t)(next >> 32)) : -INFINITY;
                token = (uint32_t)__shfl((int)token, (int)(~(uint32_t)next & 63));
            }
            const u64 v = policy.weight(b, mx), sum = wave_prefix(v);
            auto sum_at = [&](int lane) { return (u64)__shfl((long long)sum, lane); };
            auto reaching = [&](u64 target) { return __ffsll(__ballot(v && sum >= target && sum - v < target)) - 1; };
            u64 all = sum_at(63);
            if (policy.sorted) all = sum_at(reaching(target_of((double)p.o.top_p, all)));
            if ((int)tid == reaching(target_of(u, all))) p.out[row] = token;
            return;
        }
        // this thread's candidate: rank tid in the order of the logits
        u64 mine = sorted(f, tid < m ? f.list[tid] : 0, m);
        const uint32_t id = ~(uint32_t)mine;
        const float a = tid < k ? logit_of(id, unordered((uint32_t)(mine >> 32))) : -INFINITY;
        u64 best = wave_max_key(tid < k ? (u64)ordered(a) << 32 | (uint32_t)~tid : 0);  // of equal ones the first
        __syncthreads();
        if ((tid & 63) == 0) f.wave[tid >> 6] = best;
        __syncthreads();
        for (int j = 0; j < kThreads / 64; j++) best = f.wave[j] > best ? f.wave[j] : best;
        const float mx = unordered((uint32_t)(best >> 32));
        if (!(fabsf(mx) < INFINITY)) {
            if (tid == ~(uint32_t)best) p.out[row] = id;
            return;
        }
        float b = a;
        uint32_t token = id;
        if (policy.sorted && p.recent) {  // by weight: the penalised logits, ties as they stand
            uint32_t *ids = reinterpret_cast<uint32_t *>(f.sums);
            ids[tid] = id;
            __syncthreads();
            mine = sorted(f, (u64)ordered(a) << 32 | (uint32_t)~tid, k);
            b = tid < k ? unordered((uint32_t)(mine >> 32)) : -INFINITY;
            token = tid < k ? ids[~(uint32_t)mine] : 0;
        }
        const u64 v = policy.weight(b, mx), sum = prefix(f, v, &total);
        if (policy.sorted) {
            const uint32_t end = first_reaching(f, sum, v, target_of((double)p.o.top_p, total), &before);
            __syncthreads();
            if (tid == end) f.value = sum;
            __syncthreads();
            total = f.value;
        }
        const uint32_t at = first_reaching(f, sum, v, target_of(u, total), &before);
        if (tid == at) p.out[row] = token;
        return;
    }

    if (!policy.sorted) {  // in the order of the ids: the slice, then the logit
        const u64 s = tid < slices ? w.whole[tid] : 0, run = prefix(f, s, &total), target = target_of(u, total);
        const uint32_t slice = first_reaching(f, run, s, target, &before);
        u64 v[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const uint32_t i = slice * kSliceLogits + 2 * tid + j;
            v[j] = i < n ? policy.weight(logit(i), top) : 0;
        }
        const u64 pair = prefix(f, v[0] + v[1], &total);
        u64 ahead;
        const uint32_t at = first_reaching(f, pair, v[0] + v[1], target - before, &ahead);
        if (tid == at) p.out[row] = slice * kSliceLogits + 2 * tid + (v[0] && ahead + v[0] >= target - before ? 0u : 1u);
        return;
    }

    run_sums();
    u64 upto, key = 0, target = target_of((double)p.o.top_p, total);
    for (int i = 0; i < 2; i++) {  // where the nucleus ends, the draw in it
        const int bin = bin_reaching(target, &before);
        key = find([&](float a) { return policy.weight(a, top); }, bin, before, target, &upto);
        target = target_of(u, upto);
    }
    answer(~(uint32_t)key);
}

}  // namespace

size_t sample_rows_bytes(uint32_t vocab) { return up256(row_bytes(vocab)); }

hipError_t launch_sample_rows(const SampleRows &p, hipStream_t s) {
    const dim3 grid(slices_of(p.vocab), p.rows);
    hipLaunchKernelGGL(draw_stats_kernel, grid, dim3(256), 0, s, p);
    if (p.o.temperature > 0.f) hipLaunchKernelGGL(draw_bins_kernel, grid, dim3(256), 0, s, p);
    hipLaunchKernelGGL(draw_finish_kernel, dim3(p.rows), dim3(kThreads), 0, s, p);
    return hipGetLastError();
}

}  // namespace zh

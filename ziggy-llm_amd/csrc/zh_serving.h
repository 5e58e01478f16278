// zh_serving.h -- launchers of the operators that serve several sequences (norms with the rotation, the paged
// 4-bit cache and its attention, log probabilities); their arguments are checked in zh_serving.cpp.
#pragma once

#include "zh_longctx.h"

namespace zh {

constexpr int kPage = ZIGGY_HIP_KV_PAGE_POSITIONS;

// A batch whose tables the host can't see: what a kernel takes from them goes through the members below, which stay
// in bounds whatever they hold.
struct Batch {
    const uint32_t *pages, *starts, *lengths;
    uint32_t sequences, per_seq, rows, max_rows;
    uint32_t cap;   // positions that a sequence may have
    uint32_t pool;  // pages of the cache
};
// One sequence's share of a batch.
struct Sequence {
    uint32_t index, row0, rows;
    int first;  // position of row0 (below 0 where there are more rows than positions)
};
__device__ __forceinline__ Sequence sequence_of(const Batch &b, uint32_t s) {
    Sequence q;
    const uint32_t a = b.starts[s], z = b.starts[s + 1], n = b.lengths[s];
    q.index = s;
    q.row0 = a < b.rows ? a : b.rows;
    const uint32_t end = z < b.rows ? z : b.rows, all = end > q.row0 ? end - q.row0 : 0u;
    q.rows = all < b.max_rows ? all : b.max_rows;
    q.first = (int)(n < 0x7FFFFFFFu ? n : 0x7FFFFFFFu) - (int)all;
    return q;
}
// How many of the ascending values at ends[0 .. n - 1] are at most r, 64 probes at a time.  Every lane takes part; what
// does not ascend gives some number from 0 to n.
__device__ __forceinline__ uint32_t count_up_to(const uint32_t *ends, uint32_t n, uint32_t r) {
    const uint32_t lane = threadIdx.x & 63;
    uint32_t base = 0;
    while (n > 0) {
        const uint32_t step = (n + 63) / 64, at = (lane + 1) * step;  // the lane's probe is the last of its step
        const uint32_t c = (uint32_t)__popcll(__ballot(at <= n && ends[base + min(at, n) - 1] <= r));
        if (step == 1) return base + c;
        base += c * step;
        n = min(step, n - c * step);
    }
    return base;
}

// The sequence that row r belongs to; rows 0: none.  Every lane of a wavefront takes part.
__device__ __forceinline__ Sequence sequence_of_row(const Batch &b, uint32_t r) {
    Sequence q{};
    const int lane = threadIdx.x & 63;
    auto of = [&](uint32_t v, int at) { return (uint32_t)__builtin_amdgcn_readlane((int)v, at); };
    if (b.sequences <= 64) {  // every lane a sequence, one round of loads
        Sequence own{};
        uint32_t end = 0xFFFFFFFFu;
        if ((uint32_t)lane < b.sequences) own = sequence_of(b, lane), end = b.starts[lane + 1];
        const unsigned long long below = __ballot(end <= r);  // sequences that end ahead of r: the first ones
        if (!~below) return q;
        const int at = __popcll(below);
        if (at < 64) q = {of(own.index, at), of(own.row0, at), of(own.rows, at), (int)of((uint32_t)own.first, at)};
    } else {
        const uint32_t s = count_up_to(b.starts + 1, b.sequences, r);
        if (s < b.sequences) q = sequence_of(b, s);
        q = {of(q.index, 0), of(q.row0, 0), of(q.rows, 0), (int)of((uint32_t)q.first, 0)};
    }
    if (r < q.row0 || r - q.row0 >= q.rows) q.rows = 0;
    return q;
}
// the pool's page that position t < cap lies in; `pool` or above: none
__device__ __forceinline__ uint32_t page_of(const Batch &b, uint32_t s, uint32_t t) {
    return b.pages[(size_t)s * b.per_seq + t / kPage];
}

// Inclusive sums over a wavefront on the vector ALU: within rows of 16 by row shifts, then the rows' ends broadcast to
// the rows behind.  Every lane takes part.
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t moved(uint32_t v) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false);
}
template <int CTRL, int ROWS, class T> __device__ __forceinline__ T add_moved(T v) {
    if constexpr (sizeof(T) == 4) return v + (T)moved<CTRL, ROWS>((uint32_t)v);
    else return v + ((T)moved<CTRL, ROWS>((uint32_t)((unsigned long long)v >> 32)) << 32 | (T)moved<CTRL, ROWS>((uint32_t)v));
}
template <class T> __device__ __forceinline__ T running_sum(T v) {
    v = add_moved<0x111, 0xF>(v);  // row_shr:1, 2, 4, 8 (lanes before the row's start: 0)
    v = add_moved<0x112, 0xF>(v);
    v = add_moved<0x114, 0xF>(v);
    v = add_moved<0x118, 0xF>(v);
    v = add_moved<0x142, 0xA>(v);  // row_bcast:15 into rows 1 and 3
    return add_moved<0x143, 0xC>(v);  // row_bcast:31 into rows 2 and 3
}

// The sum over a team of 8 .. 64 lanes, in each of them.
__device__ __forceinline__ double team_sum(double v, int team) {
    auto add = [&](unsigned long long o) { v += __longlong_as_double((long long)o); };
    add(dpp_u64<0xB1>((unsigned long long)__double_as_longlong(v)));
    add(dpp_u64<0x4E>((unsigned long long)__double_as_longlong(v)));
    add(dpp_u64<0x141>((unsigned long long)__double_as_longlong(v)));
    if (team > 8) add(dpp_u64<0x140>((unsigned long long)__double_as_longlong(v)));
    auto far = [&](auto d) {
        const unsigned long long u = (unsigned long long)__double_as_longlong(v);
        uint32_t a0, b0, a1, b1;
        lane_pair<decltype(d)::value>((uint32_t)u, a0, b0);
        lane_pair<decltype(d)::value>((uint32_t)(u >> 32), a1, b1);
        v = __longlong_as_double((long long)((unsigned long long)a1 << 32 | a0)) + __longlong_as_double((long long)((unsigned long long)b1 << 32 | b0));
    };
    if (team > 16) far(std::integral_constant<int, 16>{});
    if (team > 32) far(std::integral_constant<int, 32>{});
    return v;
}

// LDS of a wavefront's own lanes: what they wrote is what they read behind this
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// One layer of a 4-bit cache.
struct Kv4Layer {
    uint8_t *kc, *vc, *ks, *vs;
    int nkv, hd;
    // a page's and kv head's first code byte, and scale byte
    __device__ __forceinline__ size_t codes(uint32_t page, int head) const { return ((size_t)page * nkv + head) * (kPage / 2 * hd); }
    __device__ __forceinline__ size_t scales(uint32_t page, int head) const { return ((size_t)page * nkv + head) * (kPage / 32 * hd); }
};

struct HeadRows {
    RopeFreq freq;
    int rotates, hd, rd, style;
    float magnitude;
    const float *factors, *q_norm, *k_norm;
    float eps, weight_offset;
    // f32 rows: q_heads heads, then k_heads
    const float *src;
    float *dst;
    size_t src_stride, dst_stride;
    int q_heads, k_heads;
    const uint32_t *positions;  // without a cache: null: first + row
    uint32_t first, rows;
    // rows that go into a cache (c.kc not null): heads c.nkv, the rows and positions of the batch
    Kv4Layer c;
    Batch b;
    const float *k, *v;
    int aligned;  // every row and head starts on 16 bytes
};
hipError_t launch_head_rows(const HeadRows &p, int cus, hipStream_t s);
hipError_t launch_kv4_load(const Kv4Layer &c, const Batch &b, float *k, float *v, hipStream_t s);

struct Kv4Attn {
    Kv4Layer c;
    Batch b;
    const float *q;
    size_t q_stride;
    float *out;  // [rows][heads * hd]
    int heads;
    uint32_t window;      // 0: none
    float qscale, qsign;  // score scale x log2 e, above 0; -1, 0 or 1: what the queries are multiplied by ahead
    int q_aligned;
    float *part;          // workspace
    size_t part_floats;
};
hipError_t launch_kv4_attention(const Kv4Attn &p, int cus, hipStream_t s);

struct TokenLogprobs {
    const float *x;
    size_t stride;
    const uint32_t *tokens;
    float *out, *entropy, *top;
    uint32_t *top_tokens;
    uint32_t rows, vocab;
    int k;
    void *work;
    size_t work_bytes;
};
hipError_t launch_token_logprobs(const TokenLogprobs &p, int cus, hipStream_t s);

}  // namespace zh

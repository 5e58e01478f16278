// zh_longctx.h -- launchers of a long-context step's operators (rotary rows, the 8-bit cache and its
// attention, sampling on the device); their arguments are checked in zh_longctx.cpp.
#pragma once

#include "zh_args.h"

namespace zh {

// Scaled rotary frequencies in turns a position (radians / 2 pi): 2^(i exponent) / 2 pi, blended.
struct RopeFreq {
    double exponent;   // -2 log2(base) / rope_dim
    double inv_factor; // 1 / factor (1: no scaling)
    double a, b;       // g_i = clamp(a + b x, 0, 1), x the pair (YARN) or the turns a position (BANDS); LINEAR: 0, 0
    int by_turns;
    // of pair i; factors (or null) divide the frequencies
    __device__ __forceinline__ double turns_per_position(int i, const float *factors) const {
        double f = exp2((double)i * exponent) * 0.15915494309189533577;
        const double g = fmin(fmax(a + b * (by_turns ? f : (double)i), 0.0), 1.0);
        f *= g + (1.0 - g) * inv_factor;
        return factors ? f / (double)factors[i] : f;
    }
};
// why a rope description is not served (null: it is), and its frequencies
const char *rope_refusal(const ZiggyHipRopeDesc &d);
RopeFreq rope_freq(const ZiggyHipRopeDesc &d);
struct RopeRows {
    RopeFreq freq;
    const float *src;
    float *dst;
    size_t src_stride, dst_stride;
    const uint32_t *positions;
    const float *factors;
    uint32_t first, rows;
    int heads, hd, rd, style;
    float magnitude;
    int aligned;  // every row and head starts on 16 bytes
};
hipError_t launch_rope_rows(const RopeRows &p, int cus, hipStream_t s);

constexpr int kKv8Block = ZIGGY_HIP_KV8_BLOCK;
// One layer of an 8-bit cache: head h's codes start h * blocks * 32 * hd on, its scales h * blocks on.
struct Kv8Layer {
    int8_t *kc, *vc;
    float *ks, *vs;
    int nkv, hd;
    uint32_t blocks;
};
hipError_t launch_kv8_store(const Kv8Layer &c, const float *k, const float *v, size_t row_stride, uint32_t position,
                            uint32_t rows, hipStream_t s);
hipError_t launch_kv8_load(const Kv8Layer &c, float *k, float *v, uint32_t position, uint32_t rows, hipStream_t s);

struct Kv8Attn {
    Kv8Layer c;
    const float *q;
    size_t q_stride;
    float *out;  // [queries][heads * hd]
    int heads;
    uint32_t position, queries, window;  // window 0: none
    float qscale;                        // score scale x log2 e
    float *part;                         // workspace
    size_t part_floats;
};
hipError_t launch_kv8_attention(const Kv8Attn &p, int cus, hipStream_t s);

struct SampleRows {
    const float *x;
    size_t stride;
    const uint32_t *recent;
    uint32_t recent_count;
    const double *uniforms;
    uint32_t *out;
    uint32_t rows, vocab;
    ZiggyHipSamplingOptions o;
    void *work;  // sample_rows_bytes(vocab) a row
};
size_t sample_rows_bytes(uint32_t vocab);
// why options or a vocabulary are not sampled on the device (null: they are)
const char *sample_refusal(const ZiggyHipSamplingOptions &o, uint32_t vocab);
hipError_t launch_sample_rows(const SampleRows &p, hipStream_t s);

}  // namespace zh

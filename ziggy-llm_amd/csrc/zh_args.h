// zh_args.h -- checks of arguments that the entry points over several rows share.
#pragma once

#include "zh_internal.h"

#define ZH_REFUSE(cond, ...)                      \
    if (cond) {                                   \
        set_err(err, err_len, __VA_ARGS__);       \
        return ZIGGY_HIP_INVALID_ARGUMENT;        \
    }

namespace zh {

// The context's device current for a call, the caller's again after it.
struct OnDevice {
    int before = -1;
    explicit OnDevice(int device) {
        int now = -1;
        if (hipGetDevice(&now) == hipSuccess && now != device) {
            before = now;
            hipSetDevice(device);
        }
    }
    ~OnDevice() {
        if (before >= 0) hipSetDevice(before);
    }
};

// a * b + c, or SIZE_MAX where it does not fit
inline size_t span(size_t a, size_t b, size_t c = 0) {
    size_t r;
    return __builtin_mul_overflow(a, b, &r) || __builtin_add_overflow(r, c, &r) ? SIZE_MAX : r;
}

// `need` bytes of b from `off` on, on the context's device
inline bool in_buffer(const ZiggyHipContext *ctx, const ZiggyHipBuffer *b, size_t need, size_t off = 0) {
    return b && b->ptr && b->device == ctx->device && off <= b->len && need <= b->len - off;
}

// the bytes of `rows` rows of `width` floats, `stride` floats apart
inline size_t rows_bytes(size_t rows, size_t width, size_t stride) {
    const size_t floats = span(rows - 1, stride, width);
    return span(floats, 4);
}

inline bool overlap(const void *a, size_t na, const void *b, size_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y ? y - x < na : x - y < nb;
}

}  // namespace zh

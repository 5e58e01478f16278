// zh_longctx.cpp -- entry points of a long-context step's operators: their arguments are checked here,
// on the host, so that the kernels (zh_rope.hip, zh_kv8.hip, zh_kv8_attn.hip, zh_draw.hip) index in bounds.
#include <math.h>

#include <new>

#include "zh_longctx.h"

using namespace zh;

namespace {

#define ZH_REFUSE(cond, ...)                      \
    if (cond) {                                   \
        set_err(err, err_len, __VA_ARGS__);       \
        return ZIGGY_HIP_INVALID_ARGUMENT;        \
    }

// a * b + c, or SIZE_MAX where it does not fit
size_t span(size_t a, size_t b, size_t c = 0) {
    size_t r;
    return __builtin_mul_overflow(a, b, &r) || __builtin_add_overflow(r, c, &r) ? SIZE_MAX : r;
}

// `need` bytes of b from `off` on, on the context's device
bool in_buffer(const ZiggyHipContext *ctx, const ZiggyHipBuffer *b, size_t need, size_t off = 0) {
    return b && b->ptr && b->device == ctx->device && off <= b->len && need <= b->len - off;
}

// the bytes of `rows` rows of `width` floats, `stride` floats apart
size_t rows_bytes(size_t rows, size_t width, size_t stride) {
    const size_t floats = span(rows - 1, stride, width);
    return span(floats, 4);
}

bool overlap(const void *a, size_t na, const void *b, size_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return x < y ? y - x < na : x - y < nb;
}

bool kv8_shape(uint32_t layers, uint32_t nkv, uint32_t hd, uint32_t context) {
    return layers && nkv && nkv <= 1024 && context && context <= 0x7FFFFFE0u && (hd == 64 || hd == 96 || hd == 128 || hd == 256);
}

size_t kv8_blocks(uint32_t context) { return ((size_t)context + kKv8Block - 1) / kKv8Block; }

// the layer of a cache whose buffers hold it; null: why not
const char *kv8_layer(const ZiggyHipContext *ctx, const ZiggyHipKv8Cache *c, uint32_t layer, Kv8Layer *out) {
    if (!c || !kv8_shape(c->layers, c->head_count_kv, c->head_dim, c->context_length)) return "unsupported 8-bit cache shape";
    if (layer >= c->layers) return "layer out of range";
    const size_t nc = ziggy_hip_kv8_codes_length(c->layers, c->head_count_kv, c->head_dim, c->context_length),
                 ns = ziggy_hip_kv8_scales_length(c->layers, c->head_count_kv, c->head_dim, c->context_length);
    if (nc == 0 || !in_buffer(ctx, c->k_codes, nc) || !in_buffer(ctx, c->v_codes, nc) || !in_buffer(ctx, c->k_scales, ns) ||
        !in_buffer(ctx, c->v_scales, ns))
        return "8-bit cache buffers too small, or of another device";
    const ZiggyHipBuffer *b[4] = {c->k_codes, c->v_codes, c->k_scales, c->v_scales};
    const size_t n[4] = {nc, nc, ns, ns};
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < i; j++)
            if (overlap(b[i]->ptr, n[i], b[j]->ptr, n[j])) return "8-bit cache buffers overlap";
    const size_t blocks = kv8_blocks(c->context_length), heads = (size_t)layer * c->head_count_kv;
    out->kc = (int8_t *)c->k_codes->ptr + heads * blocks * kKv8Block * c->head_dim;
    out->vc = (int8_t *)c->v_codes->ptr + heads * blocks * kKv8Block * c->head_dim;
    out->ks = (float *)c->k_scales->ptr + heads * blocks;
    out->vs = (float *)c->v_scales->ptr + heads * blocks;
    out->nkv = (int)c->head_count_kv;
    out->hd = (int)c->head_dim;
    out->blocks = (uint32_t)blocks;
    return nullptr;
}

// whether [p, p + n) meets one of the cache's buffers
bool meets_cache(const ZiggyHipKv8Cache *c, const void *p, size_t n) {
    for (const ZiggyHipBuffer *b : {c->k_codes, c->v_codes, c->k_scales, c->v_scales})
        if (overlap(b->ptr, b->len, p, n)) return true;
    return false;
}

}  // namespace

namespace zh {

const char *sample_refusal(const ZiggyHipSamplingOptions &o, uint32_t vocab) {
    if (vocab == 0 || vocab > 262144) return "sampling takes rows of 1 to 262144 logits";
    if (o.top_k > 1024 && o.top_k < vocab) return "top_k is neither at most 1024 nor the whole vocabulary";
    if (!isfinite(o.temperature) || !isfinite(o.repeat_penalty) || !(o.top_p >= 0.f && o.top_p <= 1.f) ||
        !(o.min_p >= 0.f && o.min_p <= 1.f))
        return "invalid sampling options";
    return nullptr;
}

}  // namespace zh

extern "C" {

int ziggy_hip_wrap_buffer(ZiggyHipContext *ctx, void *device_memory, size_t length, ZiggyHipBuffer **out, char *err,
                          size_t err_len) {
    if (out) *out = nullptr;
    ZH_REFUSE(!ctx || !out || !device_memory || length == 0, "invalid buffer request");
    ZH_REFUSE((uintptr_t)device_memory % 16, "wrapped memory must be 16-byte aligned");
    OnDevice on(ctx->device);
    hipPointerAttribute_t at{};
    hipDeviceptr_t base = nullptr;
    size_t size = 0;
    if (hipPointerGetAttributes(&at, device_memory) != hipSuccess || at.type != hipMemoryTypeDevice ||
        at.device != ctx->device || hipMemGetAddressRange(&base, &size, (hipDeviceptr_t)device_memory) != hipSuccess) {
        hipGetLastError();  // the refusal is this call's alone
        ZH_REFUSE(true, "not device memory of device %d", ctx->device);
    }
    const size_t into = (size_t)((const char *)device_memory - (const char *)base);
    ZH_REFUSE(into > size || length > size - into, "wrapped memory ends past its allocation");
    ZiggyHipBuffer *b = new (std::nothrow) ZiggyHipBuffer();
    if (!b) {
        set_err(err, err_len, "out of host memory");
        return ZIGGY_HIP_BUFFER_FAILED;
    }
    b->ctx = ctx;
    b->device = ctx->device;
    b->ptr = device_memory;
    b->len = length;
    b->owned = false;
    *out = b;
    return ZIGGY_HIP_OK;
}

int ziggy_hip_rope_rows_f32(ZiggyHipContext *ctx, const ZiggyHipRopeDesc *d, const ZiggyHipBuffer *src, size_t soff,
                            size_t sstride, ZiggyHipBuffer *dst, size_t doff, size_t dstride,
                            const ZiggyHipBuffer *positions, uint32_t first, const ZiggyHipBuffer *factors, uint32_t rows,
                            uint32_t heads, char *err, size_t err_len) {
    ZH_REFUSE(!ctx || !d, "null context or rope description");
    ZH_REFUSE(d->head_dim == 0 || d->head_dim % 2 || d->head_dim > 512 || d->rope_dim < 2 || d->rope_dim % 2 ||
                  d->rope_dim > d->head_dim || d->rope_style > 1 || d->scaling > ZIGGY_HIP_ROPE_BANDS,
              "unsupported rope shape");
    ZH_REFUSE(!(d->freq_base > 0) || !isfinite(d->freq_base) || !isfinite(d->magnitude), "invalid rope frequencies");
    ZH_REFUSE(d->scaling != ZIGGY_HIP_ROPE_NONE && (!(d->factor > 0) || !isfinite(d->factor)), "invalid rope factor");
    ZH_REFUSE(d->scaling >= ZIGGY_HIP_ROPE_YARN &&
                  (d->original_context == 0 || !(d->low > 0) || !(d->high > d->low) || !isfinite(d->high)),
              "invalid rope blend");
    ZH_REFUSE(d->scaling == ZIGGY_HIP_ROPE_YARN && !(d->freq_base > 1), "the YaRN blend needs a base above 1");
    ZH_REFUSE(rows == 0 || heads == 0 || heads > 65536, "rope needs rows and heads (at most 65536)");
    const size_t width = (size_t)heads * d->head_dim;
    if (sstride == 0) sstride = width;
    if (dstride == 0) dstride = width;
    const size_t ns = rows_bytes(rows, width, sstride), nd = rows_bytes(rows, width, dstride);
    ZH_REFUSE(soff % 4 || doff % 4 || sstride < width || dstride < width || !in_buffer(ctx, src, ns, soff) ||
                  !in_buffer(ctx, dst, nd, doff) || (positions && !in_buffer(ctx, positions, (size_t)rows * 4)) ||
                  (factors && !in_buffer(ctx, factors, (size_t)d->rope_dim * 2)),
              "rope buffers too small, misaligned or of another device");
    ZH_REFUSE(!positions && first + (uint64_t)rows > (1ull << 32), "rope positions past 32 bits");
    RopeRows p{};
    p.src = (const float *)((const char *)src->ptr + soff);
    p.dst = (float *)((char *)dst->ptr + doff);
    ZH_REFUSE(overlap(p.src, ns, p.dst, nd) && !(p.src == p.dst && sstride == dstride), "rope rows overlap");
    ZH_REFUSE((positions && overlap(p.dst, nd, positions->ptr, (size_t)rows * 4)) ||
                  (factors && overlap(p.dst, nd, factors->ptr, (size_t)d->rope_dim * 2)),
              "rope rows overlap their positions or factors");
    p.src_stride = sstride, p.dst_stride = dstride;
    p.positions = positions ? (const uint32_t *)positions->ptr : nullptr;
    p.factors = factors ? (const float *)factors->ptr : nullptr;
    p.first = first, p.rows = rows;
    p.heads = (int)heads, p.hd = (int)d->head_dim, p.rd = (int)d->rope_dim, p.style = (int)d->rope_style;
    p.magnitude = d->magnitude;
    p.aligned = !(((uintptr_t)p.src | (uintptr_t)p.dst) % 16) && sstride % 4 == 0 && dstride % 4 == 0;
    RopeFreq &f = p.freq;
    const double base = d->freq_base, dim = d->rope_dim, turns = 6.283185307179586476925;
    f.exponent = -2.0 * log2(base) / dim;
    f.inv_factor = d->scaling == ZIGGY_HIP_ROPE_NONE ? 1.0 : 1.0 / (double)d->factor;
    if (d->scaling == ZIGGY_HIP_ROPE_YARN) {
        auto pair_of = [&](double t) { return dim * log(d->original_context / (turns * t)) / (2.0 * log(base)); };
        const double lo = fmax(0.0, floor(pair_of(d->high))), hi = fmin(dim - 1.0, ceil(pair_of(d->low)));
        const double run = fmax(0.001, hi - lo);
        f.a = 1.0 + lo / run, f.b = -1.0 / run;
    } else if (d->scaling == ZIGGY_HIP_ROPE_BANDS) {
        const double run = (double)d->high - (double)d->low;
        f.a = -(double)d->low / run, f.b = (double)d->original_context / run;
        f.by_turns = 1;
    }
    OnDevice on(ctx->device);
    ZH_TRY(launch_rope_rows(p, (int)ctx->info.compute_units, ctx->stream), "rope_rows");
    return finish_op(ctx, "rope_rows", err, err_len);
}

size_t ziggy_hip_kv8_codes_length(uint32_t layers, uint32_t nkv, uint32_t hd, uint32_t context) {
    if (!kv8_shape(layers, nkv, hd, context)) return 0;
    const size_t n = span(span((size_t)layers * nkv, kv8_blocks(context)), (size_t)kKv8Block * hd);
    return n == SIZE_MAX ? 0 : n;
}

size_t ziggy_hip_kv8_scales_length(uint32_t layers, uint32_t nkv, uint32_t hd, uint32_t context) {
    return ziggy_hip_kv8_codes_length(layers, nkv, hd, context) / ((size_t)kKv8Block * (hd ? hd : 1)) * 4;
}

int ziggy_hip_kv8_store(ZiggyHipContext *ctx, const ZiggyHipKv8Cache *cache, const ZiggyHipBuffer *k, size_t koff,
                        const ZiggyHipBuffer *v, size_t voff, size_t stride, uint32_t layer, uint32_t position,
                        uint32_t rows, char *err, size_t err_len) {
    ZH_REFUSE(!ctx, "null context");
    Kv8Layer c{};
    const char *why = kv8_layer(ctx, cache, layer, &c);
    ZH_REFUSE(why, "%s", why);
    ZH_REFUSE(rows == 0 || position >= cache->context_length || rows > cache->context_length - position,
              "rows %u at position %u outside the context of %u", rows, position, cache->context_length);
    const size_t width = (size_t)c.nkv * c.hd;
    if (stride == 0) stride = width;
    const size_t n = rows_bytes(rows, width, stride);
    ZH_REFUSE(stride < width || koff % 4 || voff % 4 || !in_buffer(ctx, k, n, koff) || !in_buffer(ctx, v, n, voff),
              "K/V rows too small, misaligned or of another device");
    const float *kp = (const float *)((const char *)k->ptr + koff), *vp = (const float *)((const char *)v->ptr + voff);
    ZH_REFUSE(meets_cache(cache, kp, n) || meets_cache(cache, vp, n), "K/V rows overlap the cache");
    OnDevice on(ctx->device);
    ZH_TRY(launch_kv8_store(c, kp, vp, stride, position, rows, ctx->stream), "kv8_store");
    return finish_op(ctx, "kv8_store", err, err_len);
}

int ziggy_hip_kv8_load_f32(ZiggyHipContext *ctx, const ZiggyHipKv8Cache *cache, ZiggyHipBuffer *k, ZiggyHipBuffer *v,
                           uint32_t layer, uint32_t position, uint32_t rows, char *err, size_t err_len) {
    ZH_REFUSE(!ctx, "null context");
    Kv8Layer c{};
    const char *why = kv8_layer(ctx, cache, layer, &c);
    ZH_REFUSE(why, "%s", why);
    ZH_REFUSE(rows == 0 || position >= cache->context_length || rows > cache->context_length - position,
              "rows %u at position %u outside the context of %u", rows, position, cache->context_length);
    const size_t width = (size_t)c.nkv * c.hd, n = rows_bytes(rows, width, width);
    ZH_REFUSE(!in_buffer(ctx, k, n) || !in_buffer(ctx, v, n), "K/V outputs too small or of another device");
    ZH_REFUSE(overlap(k->ptr, n, v->ptr, n) || meets_cache(cache, k->ptr, n) || meets_cache(cache, v->ptr, n),
              "K/V outputs overlap each other or the cache");
    OnDevice on(ctx->device);
    ZH_TRY(launch_kv8_load(c, (float *)k->ptr, (float *)v->ptr, position, rows, ctx->stream), "kv8_load");
    return finish_op(ctx, "kv8_load", err, err_len);
}

int ziggy_hip_kv8_attention_f32(ZiggyHipContext *ctx, const ZiggyHipKv8Cache *cache, const ZiggyHipBuffer *q,
                                size_t q_stride, ZiggyHipBuffer *out, uint32_t heads, uint32_t layer, uint32_t position,
                                uint32_t queries, uint32_t window, float scale, char *err, size_t err_len) {
    ZH_REFUSE(!ctx, "null context");
    Kv8Attn p{};
    const char *why = kv8_layer(ctx, cache, layer, &p.c);
    ZH_REFUSE(why, "%s", why);
    ZH_REFUSE(heads == 0 || heads % p.c.nkv || heads / p.c.nkv > 64, "unsupported query heads %u over %d kv heads", heads,
              p.c.nkv);
    ZH_REFUSE(queries == 0 || position >= cache->context_length || queries > cache->context_length - position,
              "queries %u at position %u outside the context of %u", queries, position, cache->context_length);
    const float qscale = scale * 1.44269504088896340736f;  // scores as powers of two
    ZH_REFUSE(!isfinite(qscale), "invalid score scale");
    const size_t width = (size_t)heads * p.c.hd;
    if (q_stride == 0) q_stride = width;
    const size_t nq = rows_bytes(queries, width, q_stride), no = rows_bytes(queries, width, width);
    ZH_REFUSE(q_stride < width || !in_buffer(ctx, q, nq) || !in_buffer(ctx, out, no),
              "attention buffers too small or of another device");
    ZH_REFUSE(overlap(q->ptr, nq, out->ptr, no) || meets_cache(cache, out->ptr, no),
              "the attention's output overlaps its inputs");
    p.q = (const float *)q->ptr;
    p.q_stride = q_stride;
    p.out = (float *)out->ptr;
    p.heads = (int)heads;
    p.position = position, p.queries = queries, p.window = window;
    p.qscale = qscale;
    p.part = (float *)ctx->scratch;
    p.part_floats = ctx->scratch_len / 4;
    OnDevice on(ctx->device);
    ZH_TRY(launch_kv8_attention(p, (int)ctx->info.compute_units, ctx->stream), "kv8_attention");
    return finish_op(ctx, "kv8_attention", err, err_len);
}

int ziggy_hip_sample_rows_f32(ZiggyHipContext *ctx, const ZiggyHipBuffer *logits, size_t stride,
                              const ZiggyHipBuffer *recent, uint32_t recent_count, const ZiggyHipSamplingOptions *o,
                              const ZiggyHipBuffer *uniforms, ZiggyHipBuffer *out, uint32_t rows, uint32_t vocab, char *err,
                              size_t err_len) {
    ZH_REFUSE(!ctx || !o, "null context or sampling options");
    ZH_REFUSE(rows == 0, "sampling needs rows");
    const char *why = sample_refusal(*o, vocab);
    ZH_REFUSE(why, "%s", why);
    if (stride == 0) stride = vocab;
    const bool penalty = o->repeat_penalty > 1.f && recent_count > 0 && o->temperature > 0;
    ZH_REFUSE(stride < vocab || !in_buffer(ctx, logits, rows_bytes(rows, vocab, stride)) ||
                  !in_buffer(ctx, out, (size_t)rows * 4) || !in_buffer(ctx, uniforms, (size_t)rows * 8) ||
                  (recent_count && !in_buffer(ctx, recent, span((size_t)rows * 4, recent_count))),
              "sampling buffers too small or of another device");
    ZH_REFUSE(overlap(out->ptr, (size_t)rows * 4, logits->ptr, rows_bytes(rows, vocab, stride)) ||
                  overlap(out->ptr, (size_t)rows * 4, uniforms->ptr, (size_t)rows * 8) ||
                  (recent_count && overlap(out->ptr, (size_t)rows * 4, recent->ptr, span((size_t)rows * 4, recent_count))),
              "the tokens overlap the sampling inputs");
    SampleRows p{};
    p.stride = stride;
    p.vocab = vocab;
    p.o = *o;
    p.work = ctx->scratch;
    OnDevice on(ctx->device);
    // as many rows at a time as the context's workspace holds
    const uint32_t most = (uint32_t)(ctx->scratch_len / sample_rows_bytes(vocab) < 65535 ? ctx->scratch_len / sample_rows_bytes(vocab) : 65535);
    for (uint32_t r = 0; r < rows; r += p.rows) {
        p.rows = rows - r < most ? rows - r : most;
        p.x = (const float *)logits->ptr + (size_t)r * stride;
        p.recent = penalty ? (const uint32_t *)recent->ptr + (size_t)r * recent_count : nullptr;
        p.recent_count = penalty ? recent_count : 0;
        p.uniforms = (const double *)uniforms->ptr + r;
        p.out = (uint32_t *)out->ptr + r;
        ZH_TRY(launch_sample_rows(p, ctx->stream), "sample_rows");
    }
    return finish_op(ctx, "sample_rows", err, err_len);
}

}  // extern "C"

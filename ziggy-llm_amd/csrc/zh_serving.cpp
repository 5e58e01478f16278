// zh_serving.cpp -- entry points of the operators that serve several sequences: their arguments are checked here, on
// the host, so that the kernels (zh_heads.hip, zh_kv4_attn.hip, zh_logprobs.hip) index in bounds.
#include <math.h>

#include "zh_args.h"
#include "zh_serving.h"

using namespace zh;

namespace {

bool kv4_shape(uint32_t layers, uint32_t nkv, uint32_t hd, uint32_t pages) {
    return layers && nkv && nkv <= 1024 && pages && pages <= (1u << 24) && (hd == 64 || hd == 96 || hd == 128 || hd == 256);
}

// the layer of a cache whose buffers hold it; null: why not
const char *kv4_layer(const ZiggyHipContext *ctx, const ZiggyHipKv4Cache *c, uint32_t layer, Kv4Layer *out) {
    if (!c || !kv4_shape(c->layers, c->head_count_kv, c->head_dim, c->pages)) return "unsupported 4-bit cache shape";
    if (layer >= c->layers) return "layer out of range";
    const size_t nc = ziggy_hip_kv4_codes_length(c->layers, c->head_count_kv, c->head_dim, c->pages), ns = nc / 16;
    if (nc == 0 || !in_buffer(ctx, c->k_codes, nc) || !in_buffer(ctx, c->v_codes, nc) || !in_buffer(ctx, c->k_scales, ns) ||
        !in_buffer(ctx, c->v_scales, ns))
        return "4-bit cache buffers too small, or of another device";
    const ZiggyHipBuffer *b[4] = {c->k_codes, c->v_codes, c->k_scales, c->v_scales};
    const size_t n[4] = {nc, nc, ns, ns};
    for (int i = 0; i < 4; i++)
        for (int j = 0; j < i; j++)
            if (overlap(b[i]->ptr, n[i], b[j]->ptr, n[j])) return "4-bit cache buffers overlap";
    const size_t each = nc / c->layers * layer;
    out->kc = (uint8_t *)c->k_codes->ptr + each, out->vc = (uint8_t *)c->v_codes->ptr + each;
    out->ks = (uint8_t *)c->k_scales->ptr + each / 16, out->vs = (uint8_t *)c->v_scales->ptr + each / 16;
    out->nkv = (int)c->head_count_kv;
    out->hd = (int)c->head_dim;
    return nullptr;
}

// whether [p, p + n) meets one of the cache's arrays
bool meets_cache(const ZiggyHipKv4Cache *c, const void *p, size_t n) {
    const size_t nc = ziggy_hip_kv4_codes_length(c->layers, c->head_count_kv, c->head_dim, c->pages), ns = nc / 16;
    return overlap(c->k_codes->ptr, nc, p, n) || overlap(c->v_codes->ptr, nc, p, n) || overlap(c->k_scales->ptr, ns, p, n) ||
           overlap(c->v_scales->ptr, ns, p, n);
}

// Rows of one call: a wavefront has one, and a launch less than 2^32 threads.
constexpr uint32_t kMostRows = 1u << 25;

// a batch whose tables lie in their buffers; null: why not
const char *batch_of(const ZiggyHipContext *ctx, const ZiggyHipBatch *d, const ZiggyHipKv4Cache *c, Batch *out) {
    if (!d || d->sequences == 0 || d->sequences > 65536 || d->pages_per_sequence == 0 || d->pages_per_sequence > (1u << 24) ||
        d->rows == 0 || d->rows > kMostRows)
        return "unsupported batch";
    const size_t np = (size_t)d->sequences * d->pages_per_sequence * 4, n = (size_t)d->sequences * 4;
    if (!in_buffer(ctx, d->page_table, np) || !in_buffer(ctx, d->row_starts, n + 4) || !in_buffer(ctx, d->lengths, n))
        return "batch tables too small, or of another device";
    if (meets_cache(c, d->page_table->ptr, np) || meets_cache(c, d->row_starts->ptr, n + 4) || meets_cache(c, d->lengths->ptr, n))
        return "batch tables overlap the cache";
    out->pages = (const uint32_t *)d->page_table->ptr;
    out->starts = (const uint32_t *)d->row_starts->ptr;
    out->lengths = (const uint32_t *)d->lengths->ptr;
    out->sequences = d->sequences, out->per_seq = d->pages_per_sequence, out->rows = d->rows;
    out->max_rows = d->max_rows && d->max_rows < d->rows ? d->max_rows : d->rows;
    const uint32_t held = d->pages_per_sequence * kPage;  // at most 2^30
    out->cap = d->max_length && d->max_length < held ? d->max_length : held;
    out->pool = c->pages;
    return nullptr;
}

// whether [p, p + n) meets one of the batch's tables
bool meets_batch(const ZiggyHipBatch *d, const void *p, size_t n) {
    return overlap(d->page_table->ptr, (size_t)d->sequences * d->pages_per_sequence * 4, p, n) ||
           overlap(d->row_starts->ptr, (size_t)d->sequences * 4 + 4, p, n) || overlap(d->lengths->ptr, (size_t)d->sequences * 4, p, n);
}

// norms and rotation of heads of `hd` values; null: why not
const char *heads_of(const ZiggyHipContext *ctx, const ZiggyHipHeadsDesc *d, uint32_t hd, HeadRows *out) {
    if (!(d->eps >= 0) || !isfinite(d->eps) || !isfinite(d->weight_offset)) return "invalid norm";
    for (const ZiggyHipBuffer *w : {d->q_norm, d->k_norm})
        if (w && !in_buffer(ctx, w, (size_t)hd * 4)) return "norm weights too small, or of another device";
    out->q_norm = d->q_norm ? (const float *)d->q_norm->ptr : nullptr;
    out->k_norm = d->k_norm ? (const float *)d->k_norm->ptr : nullptr;
    out->eps = d->eps, out->weight_offset = d->weight_offset;
    if (!d->rope) return nullptr;
    const char *why = rope_refusal(*d->rope);
    if (why) return why;
    if (d->rope->head_dim != hd) return "the rotation's head size is another than the heads'";
    if (d->freq_factors && !in_buffer(ctx, d->freq_factors, (size_t)d->rope->rope_dim * 2))
        return "frequency factors too small, or of another device";
    out->rotates = 1, out->rd = (int)d->rope->rope_dim, out->style = (int)d->rope->rope_style;
    out->magnitude = d->rope->magnitude;
    out->factors = d->freq_factors ? (const float *)d->freq_factors->ptr : nullptr;
    out->freq = rope_freq(*d->rope);
    return nullptr;
}

// whether [p, p + n) meets what heads of `hd` values are turned by
bool meets_heads(const HeadRows &h, const void *p, size_t n) {
    return (h.q_norm && overlap(h.q_norm, (size_t)h.hd * 4, p, n)) || (h.k_norm && overlap(h.k_norm, (size_t)h.hd * 4, p, n)) ||
           (h.factors && overlap(h.factors, (size_t)h.rd * 2, p, n));
}

}  // namespace

extern "C" {

int ziggy_hip_norm_rope_rows_f32(ZiggyHipContext *ctx, const ZiggyHipHeadsDesc *d, const ZiggyHipBuffer *src, size_t soff,
                                 size_t sstride, ZiggyHipBuffer *dst, size_t doff, size_t dstride,
                                 const ZiggyHipBuffer *positions, uint32_t first, uint32_t rows, uint32_t q_heads,
                                 uint32_t k_heads, char *err, size_t err_len) {
    ZH_REFUSE(!ctx || !d || !d->rope, "null context, heads or rope description");
    HeadRows p{};
    p.hd = (int)d->rope->head_dim;
    const char *why = heads_of(ctx, d, d->rope->head_dim, &p);
    ZH_REFUSE(why, "%s", why);
    ZH_REFUSE(rows == 0 || rows > kMostRows || q_heads > 65536 || k_heads > 65536 || q_heads + k_heads == 0,
              "1 to 33554432 rows of 1 to 65536 heads are served");
    const size_t width = (size_t)(q_heads + k_heads) * p.hd;
    if (sstride == 0) sstride = width;
    if (dstride == 0) dstride = width;
    const size_t ns = rows_bytes(rows, width, sstride), nd = rows_bytes(rows, width, dstride), np = positions ? (size_t)rows * 4 : 0;
    ZH_REFUSE(soff % 4 || doff % 4 || sstride < width || dstride < width || !in_buffer(ctx, src, ns, soff) ||
                  !in_buffer(ctx, dst, nd, doff) || (positions && !in_buffer(ctx, positions, np)),
              "head rows too small, misaligned or of another device");
    ZH_REFUSE(!positions && first + (uint64_t)rows > (1ull << 32), "positions past 32 bits");
    p.src = (const float *)((const char *)src->ptr + soff);
    p.dst = (float *)((char *)dst->ptr + doff);
    ZH_REFUSE(overlap(p.src, ns, p.dst, nd) && !(p.src == p.dst && sstride == dstride), "head rows overlap");
    ZH_REFUSE((positions && overlap(p.dst, nd, positions->ptr, np)) || meets_heads(p, p.dst, nd),
              "head rows overlap their positions, weights or factors");
    p.src_stride = sstride, p.dst_stride = dstride;
    p.q_heads = (int)q_heads, p.k_heads = (int)k_heads;
    p.positions = positions ? (const uint32_t *)positions->ptr : nullptr;
    p.first = first, p.rows = rows;
    p.aligned = !(((uintptr_t)p.src | (uintptr_t)p.dst) % 16) && sstride % 4 == 0 && dstride % 4 == 0;
    OnDevice on(ctx->device);
    ZH_TRY(launch_head_rows(p, (int)ctx->info.compute_units, ctx->stream), "norm_rope_rows");
    return finish_op(ctx, "norm_rope_rows", err, err_len);
}

size_t ziggy_hip_kv4_codes_length(uint32_t layers, uint32_t nkv, uint32_t hd, uint32_t pages) {
    if (!kv4_shape(layers, nkv, hd, pages)) return 0;
    const size_t n = span(span((size_t)layers * nkv, pages), (size_t)kPage / 2 * hd);
    return n == SIZE_MAX ? 0 : n;
}

size_t ziggy_hip_kv4_scales_length(uint32_t layers, uint32_t nkv, uint32_t hd, uint32_t pages) {
    return ziggy_hip_kv4_codes_length(layers, nkv, hd, pages) / 16;  // a byte for 32 halves of a byte
}

int ziggy_hip_kv4_append(ZiggyHipContext *ctx, const ZiggyHipKv4Cache *cache, uint32_t layer, const ZiggyHipBatch *batch,
                         const ZiggyHipHeadsDesc *d, const ZiggyHipBuffer *src, size_t koff, size_t voff, size_t stride,
                         uint32_t q_heads, size_t qoff, ZiggyHipBuffer *q_out, size_t ooff, size_t ostride, char *err,
                         size_t err_len) {
    ZH_REFUSE(!ctx, "null context");
    HeadRows p{};
    const char *why = kv4_layer(ctx, cache, layer, &p.c);
    if (!why) why = batch_of(ctx, batch, cache, &p.b);
    p.hd = p.c.hd;
    if (!why && d) why = heads_of(ctx, d, (uint32_t)p.hd, &p);
    ZH_REFUSE(why, "%s", why);
    const size_t kv_width = (size_t)p.c.nkv * p.hd, q_width = (size_t)q_heads * p.hd;
    ZH_REFUSE(q_heads > 65536, "too many query heads");
    if (stride == 0) stride = kv_width;
    if (ostride == 0) ostride = q_width;
    const uint32_t rows = batch->rows;
    const size_t nkv = rows_bytes(rows, kv_width, stride);
    ZH_REFUSE(stride < kv_width || koff % 4 || voff % 4 || !in_buffer(ctx, src, nkv, koff) || !in_buffer(ctx, src, nkv, voff),
              "K/V rows too small, misaligned or of another device");
    p.k = (const float *)((const char *)src->ptr + koff), p.v = (const float *)((const char *)src->ptr + voff);
    ZH_REFUSE(meets_cache(cache, p.k, nkv) || meets_cache(cache, p.v, nkv), "K/V rows overlap the cache");
    ZH_REFUSE((p.q_norm && meets_cache(cache, p.q_norm, p.hd * 4)) || (p.k_norm && meets_cache(cache, p.k_norm, p.hd * 4)) ||
                  (p.factors && meets_cache(cache, p.factors, (size_t)p.rd * 2)),
              "weights or factors overlap the cache");
    p.aligned = !(((uintptr_t)p.k | (uintptr_t)p.v) % 16) && stride % 4 == 0;
    p.src_stride = stride;
    if (q_heads) {
        const size_t nq = rows_bytes(rows, q_width, stride), no = rows_bytes(rows, q_width, ostride);
        ZH_REFUSE(stride < q_width || ostride < q_width || qoff % 4 || ooff % 4 || !in_buffer(ctx, src, nq, qoff) ||
                      !in_buffer(ctx, q_out, no, ooff),
                  "query rows too small, misaligned or of another device");
        p.src = (const float *)((const char *)src->ptr + qoff);
        p.dst = (float *)((char *)q_out->ptr + ooff);
        ZH_REFUSE(overlap(p.src, nq, p.dst, no) && !(p.src == p.dst && stride == ostride), "query rows overlap");
        // in place, their heads lie beside the keys' and values' in the same rows
        auto beside = [&](const float *kv) {
            const size_t apart = kv < p.dst ? (size_t)(p.dst - kv) : (size_t)(kv - p.dst), of = apart % stride;
            return ostride == stride && (kv < p.dst ? of >= kv_width && of + q_width <= stride : of >= q_width && of + kv_width <= stride);
        };
        ZH_REFUSE((overlap(p.k, nkv, p.dst, no) && !beside(p.k)) || (overlap(p.v, nkv, p.dst, no) && !beside(p.v)),
                  "the query output overlaps the K/V rows");
        ZH_REFUSE(meets_cache(cache, p.dst, no) || meets_batch(batch, p.dst, no) || meets_heads(p, p.dst, no),
                  "the query output overlaps the cache, the batch's tables, weights or factors");
        p.dst_stride = ostride;
        p.q_heads = (int)q_heads;
        p.aligned = p.aligned && !(((uintptr_t)p.src | (uintptr_t)p.dst) % 16) && ostride % 4 == 0;
    }
    p.rows = rows;
    OnDevice on(ctx->device);
    ZH_TRY(launch_head_rows(p, (int)ctx->info.compute_units, ctx->stream), "kv4_append");
    return finish_op(ctx, "kv4_append", err, err_len);
}

int ziggy_hip_kv4_load_f32(ZiggyHipContext *ctx, const ZiggyHipKv4Cache *cache, uint32_t layer, const ZiggyHipBatch *batch,
                           ZiggyHipBuffer *k, ZiggyHipBuffer *v, char *err, size_t err_len) {
    ZH_REFUSE(!ctx, "null context");
    Kv4Layer c{};
    Batch b{};
    const char *why = kv4_layer(ctx, cache, layer, &c);
    if (!why) why = batch_of(ctx, batch, cache, &b);
    ZH_REFUSE(why, "%s", why);
    const size_t width = (size_t)c.nkv * c.hd, n = rows_bytes(b.rows, width, width);
    ZH_REFUSE(!in_buffer(ctx, k, n) || !in_buffer(ctx, v, n), "K/V outputs too small or of another device");
    ZH_REFUSE(overlap(k->ptr, n, v->ptr, n) || meets_cache(cache, k->ptr, n) || meets_cache(cache, v->ptr, n) ||
                  meets_batch(batch, k->ptr, n) || meets_batch(batch, v->ptr, n),
              "K/V outputs overlap each other, the cache or the batch's tables");
    OnDevice on(ctx->device);
    ZH_TRY(launch_kv4_load(c, b, (float *)k->ptr, (float *)v->ptr, ctx->stream), "kv4_load");
    return finish_op(ctx, "kv4_load", err, err_len);
}

int ziggy_hip_kv4_attention_f32(ZiggyHipContext *ctx, const ZiggyHipKv4Cache *cache, uint32_t layer, const ZiggyHipBatch *batch,
                                const ZiggyHipBuffer *q, size_t qoff, size_t q_stride, ZiggyHipBuffer *out, uint32_t heads,
                                uint32_t window, float scale, char *err, size_t err_len) {
    ZH_REFUSE(!ctx, "null context");
    Kv4Attn p{};
    const char *why = kv4_layer(ctx, cache, layer, &p.c);
    if (!why) why = batch_of(ctx, batch, cache, &p.b);
    ZH_REFUSE(why, "%s", why);
    ZH_REFUSE(heads == 0 || heads % p.c.nkv || heads / p.c.nkv > 64, "unsupported query heads %u over %d kv heads", heads, p.c.nkv);
    ZH_REFUSE((uint64_t)p.b.sequences * p.c.nkv > (1u << 21) || (uint64_t)p.b.rows * heads > (1u << 29), "too many sequences or rows for one call");
    // scores as powers of two; the scale's sign goes to the queries
    p.qscale = fabsf(scale) * 1.44269504088896340736f, p.qsign = scale > 0 ? 1.f : scale < 0 ? -1.f : 0.f;
    ZH_REFUSE(!isfinite(p.qscale), "invalid score scale");
    if (p.qscale == 0) p.qscale = 1.f, p.qsign = 0.f;
    const size_t width = (size_t)heads * p.c.hd;
    if (q_stride == 0) q_stride = width;
    const size_t nq = rows_bytes(p.b.rows, width, q_stride), no = rows_bytes(p.b.rows, width, width);
    ZH_REFUSE(q_stride < width || qoff % 4 || !in_buffer(ctx, q, nq, qoff) || !in_buffer(ctx, out, no),
              "attention buffers too small, misaligned or of another device");
    p.q = (const float *)((const char *)q->ptr + qoff);
    ZH_REFUSE(overlap(p.q, nq, out->ptr, no) || meets_cache(cache, out->ptr, no) || meets_batch(batch, out->ptr, no),
              "the attention's output overlaps its inputs");
    p.q_stride = q_stride;
    p.out = (float *)out->ptr;
    p.heads = (int)heads;
    p.window = window;
    p.q_aligned = (uintptr_t)p.q % 16 == 0 && q_stride % 4 == 0;
    p.part = (float *)ctx->scratch;
    p.part_floats = ctx->scratch_len / 4;
    OnDevice on(ctx->device);
    ZH_TRY(launch_kv4_attention(p, (int)ctx->info.compute_units, ctx->stream), "kv4_attention");
    return finish_op(ctx, "kv4_attention", err, err_len);
}

int ziggy_hip_token_logprobs_f32(ZiggyHipContext *ctx, const ZiggyHipBuffer *logits, size_t stride, const ZiggyHipBuffer *tokens,
                                 ZiggyHipBuffer *out, ZiggyHipBuffer *entropy, uint32_t k, ZiggyHipBuffer *top_tokens,
                                 ZiggyHipBuffer *top, uint32_t rows, uint32_t vocab, char *err, size_t err_len) {
    ZH_REFUSE(!ctx, "null context");
    ZH_REFUSE(rows == 0 || vocab == 0 || vocab > 262144, "log probabilities take rows of 1 to 262144 logits");
    ZH_REFUSE(k > ZIGGY_HIP_MAX_TOP_LOGPROBS || k > vocab, "at most %d top tokens, and no more than the vocabulary",
              ZIGGY_HIP_MAX_TOP_LOGPROBS);
    if (stride == 0) stride = vocab;
    const size_t nx = rows_bytes(rows, vocab, stride), n = (size_t)rows * 4, nk = n * k;
    ZH_REFUSE(stride < vocab || !in_buffer(ctx, logits, nx) || !in_buffer(ctx, tokens, n) || !in_buffer(ctx, out, n) ||
                  (entropy && !in_buffer(ctx, entropy, n)) || (k && (!in_buffer(ctx, top_tokens, nk) || !in_buffer(ctx, top, nk))),
              "log probability buffers too small or of another device");
    const ZiggyHipBuffer *outs[4] = {out, entropy, k ? top_tokens : nullptr, k ? top : nullptr};
    const size_t sizes[4] = {n, n, nk, nk};
    for (int i = 0; i < 4; i++) {
        if (!outs[i]) continue;
        bool meets = overlap(outs[i]->ptr, sizes[i], logits->ptr, nx) || overlap(outs[i]->ptr, sizes[i], tokens->ptr, n);
        for (int j = 0; j < i; j++) meets = meets || (outs[j] && overlap(outs[i]->ptr, sizes[i], outs[j]->ptr, sizes[j]));
        ZH_REFUSE(meets, "the log probabilities overlap each other or their inputs");
    }
    TokenLogprobs p{};
    p.x = (const float *)logits->ptr, p.stride = stride;
    p.tokens = (const uint32_t *)tokens->ptr;
    p.out = (float *)out->ptr, p.entropy = entropy ? (float *)entropy->ptr : nullptr;
    p.top = k ? (float *)top->ptr : nullptr, p.top_tokens = k ? (uint32_t *)top_tokens->ptr : nullptr;
    p.rows = rows, p.vocab = vocab, p.k = (int)k;
    p.work = ctx->scratch, p.work_bytes = ctx->scratch_len;
    OnDevice on(ctx->device);
    ZH_TRY(launch_token_logprobs(p, (int)ctx->info.compute_units, ctx->stream), "token_logprobs");
    return finish_op(ctx, "token_logprobs", err, err_len);
}

}  // extern "C"

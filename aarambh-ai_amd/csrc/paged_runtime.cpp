// C ABI of the paged-cache operators and the logits processor: argument checks and launches.
// Nothing here allocates device memory, waits for the device or reads a device array, so every entry may
// be captured into a graph.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <exception>
#include <string>

#include "../../include/aarambh_hip.h"
#include "paged.hpp"

using namespace aarh;

namespace aarh {
int ctx_fail(aarh_ctx* c, int code, const char* msg);
int ctx_device(const aarh_ctx* c);
int host_fail(int code, const char* msg);
int rope_scaling_check(int head_dim, int max_seq_len, const aarh_rope_scaling* s, std::string& err);
}  // namespace aarh

namespace {

int fail(aarh_ctx* c, int code, const char* fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof(buf), fmt, ap);
    va_end(ap);
    return ctx_fail(c, code, buf);
}

// The context's device for the length of a call.
struct DeviceScope {
    int before = -1;
    bool ok = true;
    explicit DeviceScope(int device) {
        if (hipGetDevice(&before) != hipSuccess) before = -1;
        if (before != device) ok = hipSetDevice(device) == hipSuccess;
        else before = -1;
    }
    ~DeviceScope() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

hipStream_t stream_of(aarh_ctx* c, void* stream) {
    if (stream == AARH_DEFAULT_STREAM) return nullptr;
    return stream ? (hipStream_t)stream : (hipStream_t)aarh_stream(c);
}

bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

int check_pool(aarh_ctx* c, const aarh_page_pool* p, PagePool* out) {
    if (p->kv_format != AARH_KV_F16 && p->kv_format != AARH_KV_INT8 && p->kv_format != AARH_KV_BF16)
        return fail(c, AARH_ERR_UNSUPPORTED, "page pools hold AARH_KV_F16, AARH_KV_BF16 or AARH_KV_INT8, not format %d",
                    p->kv_format);
    if (p->head_dim != 64 && p->head_dim != 128)
        return fail(c, AARH_ERR_UNSUPPORTED, "page pools need head_dim 64 or 128, not %d", p->head_dim);
    int shift = 5;
    while (shift <= 8 && (1 << shift) != p->page_tokens) shift++;
    if (shift > 8) return fail(c, AARH_ERR_UNSUPPORTED, "page_tokens must be 32, 64, 128 or 256, not %d", p->page_tokens);
    if (p->n_pages <= 0 || p->n_kv_heads <= 0 || p->n_kv_heads > 32768)
        return fail(c, AARH_ERR_SHAPE, "bad page pool: %d pages of %d kv heads", p->n_pages, p->n_kv_heads);
    if (!p->k || !p->v || (p->kv_format == AARH_KV_INT8 && (!p->k_scale || !p->v_scale)))
        return fail(c, AARH_ERR_CONFIG, "null page pool array");
    if (!aligned(p->k) || !aligned(p->v) || !aligned(p->k_scale) || !aligned(p->v_scale))
        return fail(c, AARH_ERR_UNSUPPORTED, "page pool arrays must be 16-byte aligned");
    out->fmt = p->kv_format;
    out->n_kv = p->n_kv_heads;
    out->hd = p->head_dim;
    out->page_shift = shift;
    out->n_pages = p->n_pages;
    out->k = p->k;
    out->v = p->v;
    out->ks = p->k_scale;
    out->vs = p->v_scale;
    return 0;
}

// shapes: no pointer is looked at (workspace queries)
int check_batch(aarh_ctx* c, const aarh_page_batch* b, const PagePool& pool, bool shapes, PageBatch* out) {
    if (b->nseq < 0 || b->nseq > 65535 || b->rows < 0 || b->max_rows < 0 || b->max_kv < 0)
        return fail(c, AARH_ERR_SHAPE, "bad page batch: %d sequences, %d rows, at most %d rows and %d tokens each", b->nseq,
                    b->rows, b->max_rows, b->max_kv);
    if (b->max_kv > (1 << 30) || b->rows > (1 << 30))
        return fail(c, AARH_ERR_SHAPE, "page batch of %d rows and %d tokens: at most 2^30", b->rows, b->max_kv);
    if (!shapes && b->nseq) {
        if (!b->row_off || !b->kv_len || !b->tables) return fail(c, AARH_ERR_CONFIG, "null page batch array");
        if (b->table_ld < (((int64_t)b->max_kv + (1 << pool.page_shift) - 1) >> pool.page_shift))
            return fail(c, AARH_ERR_SHAPE, "page tables of %lld entries cannot hold %d tokens", (long long)b->table_ld,
                        b->max_kv);
    }
    out->nseq = b->nseq;
    out->rows = b->rows;
    // a sequence has no more rows than the buffers, and no more than cached tokens
    out->max_rows = b->max_rows < b->rows ? b->max_rows : b->rows;
    if (out->max_rows > b->max_kv) out->max_rows = b->max_kv;
    out->max_kv = b->max_kv;
    out->row_off = b->row_off;
    out->kv_len = b->kv_len;
    out->tables = b->tables;
    out->table_ld = b->table_ld;
    out->status = b->status;
    return 0;
}

int check_act(aarh_ctx* c, int act, int fmt) {
    const bool ok = (act == AARH_A_F32 && (fmt == AARH_KV_F16 || fmt == AARH_KV_INT8)) ||
                    (act == AARH_A_F16 && (fmt == AARH_KV_F16 || fmt == AARH_KV_INT8)) ||
                    (act == AARH_A_BF16 && fmt == AARH_KV_BF16);
    if (!ok)
        return fail(c, AARH_ERR_UNSUPPORTED,
                    "activation type %d over page format %d (f32 and fp16 go with fp16 and INT8 pages, bf16 with bf16)", act, fmt);
    return 0;
}

int check_rows(aarh_ctx* c, const char* what, const void* p, int64_t ld, int64_t width, int act) {
    const int64_t esz = act == AARH_A_F32 ? 4 : 2;
    if (!p) return fail(c, AARH_ERR_CONFIG, "null %s", what);
    if (ld < width) return fail(c, AARH_ERR_SHAPE, "%s rows of %lld elements are %lld apart", what, (long long)width, (long long)ld);
    if (!aligned(p) || ld * esz % 16) return fail(c, AARH_ERR_UNSUPPORTED, "%s rows must be 16-byte aligned", what);
    return 0;
}

int attn_args(aarh_ctx* c, const aarh_page_pool* pool, const aarh_page_batch* batch, const aarh_paged_attn_args* args,
              bool shapes, PagedAttnArgs* a) {
    int r;
    *a = PagedAttnArgs{};
    if ((r = check_pool(c, pool, &a->pool)) || (r = check_batch(c, batch, a->pool, shapes, &a->bt)) ||
        (r = check_act(c, args->act, pool->kv_format)))
        return r;
    if (args->n_heads <= 0 || args->n_heads > 65535 || args->n_heads % pool->n_kv_heads)
        return fail(c, AARH_ERR_SHAPE, "%d query heads over %d kv heads", args->n_heads, pool->n_kv_heads);
    const int64_t rows = (int64_t)a->bt.max_rows * (args->n_heads / pool->n_kv_heads);
    if (rows > (1 << 30) || (int64_t)batch->nseq * pool->n_kv_heads * (rows / 128 + 1) > (1 << 23))  // workgroups of a grid
        return fail(c, AARH_ERR_SHAPE, "%d sequences of up to %d rows are too much for one call", batch->nseq, a->bt.max_rows);
    if (!shapes && (!std::isfinite(args->scale) || !(args->softcap >= 0.f) || !std::isfinite(args->softcap)))
        return fail(c, AARH_ERR_CONFIG, "scale must be finite, softcap finite and not negative");
    if (args->window < 0) return fail(c, AARH_ERR_CONFIG, "negative attention window %d", args->window);
    a->act = args->act;
    a->n_heads = args->n_heads;
    a->grouped = args->grouped ? 1 : 0;
    a->q = args->q;
    a->q_ld = args->q_ld;
    a->out = args->out;
    a->out_ld = args->out_ld;
    a->scale = args->scale;
    a->softcap = args->softcap;
    a->window = args->window;
    a->slopes = args->slopes;
    a->prefix = args->prefix;
    a->workspace = args->workspace;
    return 0;
}

}  // namespace

extern "C" {

int aarh_rope_frequencies(int32_t R, double theta, int32_t max_seq_len, const aarh_rope_scaling* s, double* inv,
                          float* attn) {
    try {
        if (!inv || !attn) return host_fail(AARH_ERR_CONFIG, "null output");
        if (R <= 0 || R % 2 || R > 65536) return host_fail(AARH_ERR_SHAPE, "rot_dim must be positive and even");
        if (!(theta > 0.0) || !std::isfinite(theta)) return host_fail(AARH_ERR_CONFIG, "rope_theta must be finite and positive");
        std::string err;
        if (s) {
            const int r = rope_scaling_check(R, max_seq_len, s, err);
            if (r) return host_fail(r, err.c_str());
        }
        const int how = s ? s->method : AARH_ROPE_NONE, half = R / 2;
        *attn = how == AARH_ROPE_NONE ? 1.0f : (float)s->attn_factor;
        const double base = how == AARH_ROPE_NTK ? theta * std::pow(s->factor, (double)R / ((double)R - 2.0)) : theta;
        double low = 0, high = 0;
        if (how == AARH_ROPE_YARN) {
            // dimension indices between which the frequency goes over from its own to the interpolated one
            auto dim = [&](double turns) {
                return (double)R * std::log((double)s->original_max_seq_len / (turns * 2.0 * 3.14159265358979323846)) /
                       (2.0 * std::log(theta));
            };
            low = std::fmin(std::fmax(std::floor(dim(s->beta_fast)), 0.0), half - 1.0);
            high = std::fmin(std::fmax(std::ceil(dim(s->beta_slow)), 0.0), half - 1.0);
            if (high == low) high += 0.001;
        }
        for (int i = 0; i < half; i++) {
            inv[i] = 1.0 / std::pow(base, 2.0 * i / R);
            if (how == AARH_ROPE_LINEAR) inv[i] /= s->factor;
            if (how == AARH_ROPE_YARN) {
                const double ramp = std::fmin(std::fmax((i - low) / (high - low), 0.0), 1.0);
                inv[i] = inv[i] / s->factor * ramp + inv[i] * (1.0 - ramp);
            }
        }
        return 0;
    } catch (const std::exception& e) {
        return host_fail(AARH_ERR_CONFIG, e.what());
    }
}

int aarh_rope_append(aarh_ctx* c, const aarh_page_pool* pool, const aarh_page_batch* batch, const aarh_rope_args* args,
                     void* stream) {
    if (!c || !pool || !batch || !args) return c ? fail(c, AARH_ERR_CONFIG, "null argument block") : AARH_ERR_CONFIG;
    RopeAppendArgs a{};
    int r;
    if ((r = check_pool(c, pool, &a.pool)) || (r = check_batch(c, batch, a.pool, false, &a.bt)) ||
        (r = check_act(c, args->act, pool->kv_format)))
        return r;
    const int hd = pool->head_dim;
    if (args->n_heads < 0 || args->n_heads > 32768) return fail(c, AARH_ERR_SHAPE, "bad query head count %d", args->n_heads);
    if (args->rot_dim < 0 || args->rot_dim > hd || args->rot_dim % 16)
        return fail(c, AARH_ERR_UNSUPPORTED, "rot_dim %d is not a multiple of 16 up to head_dim %d", args->rot_dim, hd);
    if (args->rot_dim && !args->inv_freq) return fail(c, AARH_ERR_CONFIG, "null inv_freq");
    if (batch->nseq == 0 || batch->rows == 0) return 0;
    const int64_t kw = (int64_t)pool->n_kv_heads * hd, qw = (int64_t)args->n_heads * hd;
    if ((r = check_rows(c, "k", args->k, args->k_ld, kw, args->act)) ||
        (r = check_rows(c, "v", args->v, args->v_ld, kw, args->act)))
        return r;
    if (args->n_heads && ((r = check_rows(c, "q", args->q, args->q_ld, qw, args->act)) ||
                          (r = check_rows(c, "q_out", args->q_out, args->q_out_ld, qw, args->act))))
        return r;
    a.act = args->act;
    a.n_heads = args->n_heads;
    a.q = args->q;
    a.k = args->k;
    a.v = args->v;
    a.q_ld = args->q_ld;
    a.k_ld = args->k_ld;
    a.v_ld = args->v_ld;
    a.q_out = args->q_out;
    a.q_out_ld = args->q_out_ld;
    a.inv_freq = args->inv_freq;
    a.rot = args->rot_dim;
    a.interleaved = args->interleaved ? 1 : 0;
    a.attn = args->attn_factor;
    DeviceScope dev(ctx_device(c));
    if (!dev.ok) return fail(c, AARH_ERR_DEVICE, "hipSetDevice(%d) failed", ctx_device(c));
    if (launch_rope_append(a, stream_of(c, stream)))
        return fail(c, AARH_ERR_DEVICE, "rope append launch failed: %s", last_launch_error());
    return 0;
}

int aarh_paged_attention_workspace(aarh_ctx* c, const aarh_page_pool* pool, const aarh_page_batch* batch,
                                   const aarh_paged_attn_args* args, int64_t* bytes) {
    if (!c || !pool || !batch || !args || !bytes) return c ? fail(c, AARH_ERR_CONFIG, "null argument block") : AARH_ERR_CONFIG;
    PagedAttnArgs a;
    const int r = attn_args(c, pool, batch, args, true, &a);
    if (r) return r;
    *bytes = batch->nseq && batch->rows ? paged_attention_workspace(a) : 0;
    return 0;
}

int aarh_paged_attention(aarh_ctx* c, const aarh_page_pool* pool, const aarh_page_batch* batch,
                         const aarh_paged_attn_args* args, void* stream) {
    if (!c || !pool || !batch || !args) return c ? fail(c, AARH_ERR_CONFIG, "null argument block") : AARH_ERR_CONFIG;
    PagedAttnArgs a;
    int r = attn_args(c, pool, batch, args, false, &a);
    if (r) return r;
    if (batch->nseq == 0 || batch->rows == 0 || a.bt.max_rows == 0) return 0;
    const int64_t w = (int64_t)args->n_heads * pool->head_dim;
    if ((r = check_rows(c, "q", args->q, args->q_ld, w, args->act)) ||
        (r = check_rows(c, "out", args->out, args->out_ld, w, args->act)))
        return r;
    const long long need = paged_attention_workspace(a);
    if (need && (!args->workspace || args->workspace_bytes < need))
        return fail(c, AARH_ERR_SHAPE, "attention workspace of %lld bytes, %lld needed", (long long)args->workspace_bytes, need);
    if (need && !aligned(args->workspace)) return fail(c, AARH_ERR_UNSUPPORTED, "attention workspace must be 16-byte aligned");
    DeviceScope dev(ctx_device(c));
    if (!dev.ok) return fail(c, AARH_ERR_DEVICE, "hipSetDevice(%d) failed", ctx_device(c));
    if (launch_paged_attention(a, stream_of(c, stream)))
        return fail(c, AARH_ERR_DEVICE, "paged attention launch failed: %s", last_launch_error());
    return 0;
}

int aarh_process_logits(aarh_ctx* c, const aarh_logits_args* g, void* stream) {
    if (!c || !g) return c ? fail(c, AARH_ERR_CONFIG, "null argument block") : AARH_ERR_CONFIG;
    if (g->nseq < 0 || g->nseq > 65535 || g->rows_per_seq < 0 || g->vocab < 0)
        return fail(c, AARH_ERR_SHAPE, "bad logits shape: %d sequences x %d rows x %d", g->nseq, g->rows_per_seq, g->vocab);
    if (g->nseq == 0 || g->rows_per_seq == 0 || g->vocab == 0) return 0;
    if (!g->logits || !g->out) return fail(c, AARH_ERR_CONFIG, "null logits");
    if (g->ld < g->vocab || g->out_ld < g->vocab)
        return fail(c, AARH_ERR_SHAPE, "logits rows of %d are %lld and %lld apart", g->vocab, (long long)g->ld, (long long)g->out_ld);
    if (((uintptr_t)g->logits & 3) || ((uintptr_t)g->out & 3)) return fail(c, AARH_ERR_UNSUPPORTED, "logits must be 4-byte aligned");
    if (g->logits == g->out && g->ld != g->out_ld)
        return fail(c, AARH_ERR_SHAPE, "logits processed in place need one row stride, not %lld and %lld", (long long)g->ld,
                    (long long)g->out_ld);
    if (g->history && (g->history_ld < 0 || !g->history_len)) return fail(c, AARH_ERR_CONFIG, "a history needs its lengths");
    if (g->draft && g->draft_ld < g->rows_per_seq - 1)
        return fail(c, AARH_ERR_SHAPE, "%d rows need %d proposals, got %lld", g->rows_per_seq, g->rows_per_seq - 1,
                    (long long)g->draft_ld);
    if (g->bias_off && (g->n_bias < 0 || (g->n_bias && (!g->bias_ids || !g->bias_vals))))
        return fail(c, AARH_ERR_CONFIG, "bias offsets without bias ids and values");
    if (g->masks && (g->n_masks < 0 || !g->mask_of_row || g->mask_ld < ((int64_t)g->vocab + 31) / 32))
        return fail(c, AARH_ERR_SHAPE, "%d masks of %lld words for a vocabulary of %d", g->n_masks, (long long)g->mask_ld, g->vocab);
    LogitsArgs a{};
    a.nseq = g->nseq;
    a.R = g->rows_per_seq;
    a.V = g->vocab;
    a.x = g->logits;
    a.ld = g->ld;
    a.out = g->out;
    a.out_ld = g->out_ld;
    a.hist = g->history;
    a.hist_ld = g->history_ld;
    a.hist_len = g->history_len;
    a.prompt_len = g->prompt_len;
    a.pen = g->penalties;
    a.draft = g->draft;
    a.draft_ld = g->draft_ld;
    a.bias_off = g->bias_off;
    a.bias_ids = g->bias_ids;
    a.bias_vals = g->bias_vals;
    a.n_bias = g->n_bias;
    a.masks = g->masks;
    a.mask_ld = g->mask_ld;
    a.n_masks = g->n_masks;
    a.mask_of_row = g->mask_of_row;
    DeviceScope dev(ctx_device(c));
    if (!dev.ok) return fail(c, AARH_ERR_DEVICE, "hipSetDevice(%d) failed", ctx_device(c));
    if (launch_process_logits(a, stream_of(c, stream)))
        return fail(c, AARH_ERR_DEVICE, "logits processing launch failed: %s", last_launch_error());
    return 0;
}

}  // extern "C"

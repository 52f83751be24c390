// attn_api.hip -- the attention part of the extern "C" boundary: handle, checks, launches.
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <new>

#include "attn_internal.hpp"
#include "moe_internal.hpp"

using namespace moe;

struct moe_attn {
    int device = 0;
    moe_attn_config cfg{};
    int page_shift = 0;
    void *arena = nullptr;     // one device allocation, carved below
    uint32_t *flags = nullptr; // sticky device flags
    float *part = nullptr;     // partial rows: [part_rows][head_dim]
    float *part_ml = nullptr;  // ... and each one's maximum and sum: [part_rows][2]
    int64_t part_rows = 0;
    Piece *piece = nullptr;    // [n_wg]
    int n_wg = 0;              // workgroups of a decode launch
    int n_cu = 0;              // compute units of the device
};

namespace {

moe_status fail(moe_status st, const char *fmt, ...) {
    char buf[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(buf, sizeof buf, fmt, ap);
    va_end(ap);
    return set_error(st, buf);
}

moe_status ok() { return set_error(MOE_OK, ""); }

bool aligned(const void *p, unsigned n) { return ((uintptr_t)p & (n - 1)) == 0; }

// Makes a device current for a call and the caller's one again after it.
struct OnDevice {
    int before = -1;
    hipError_t he;
    explicit OnDevice(int device) {
        he = hipGetDevice(&before);
        if (he == hipSuccess && before != device) he = hipSetDevice(device);
        else before = -1;
    }
    ~OnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

// The checks that every call shares; fills the sequences and the cache.
moe_status common_args(const char *fn, moe_attn *a, const moe_kv_cache *kv, const moe_seq_batch *s, AttnArgs *c) {
    if (!a || !kv || !s) return fail(MOE_EINVAL, "%s: null argument", fn);
    const moe_attn_config &g = a->cfg;
    if (s->n_seqs < 0 || s->n_seqs > g.max_seqs)
        return fail(MOE_EINVAL, "%s: %d sequences outside 0..max_seqs=%d", fn, s->n_seqs, g.max_seqs);
    if (s->n_rows < 0 || s->n_rows > (1 << 22)) // (rows * heads) are counted in 31 bits
        return fail(MOE_EINVAL, "%s: %d rows outside 0..2^22", fn, s->n_rows);
    if (!s->row_start && s->n_rows != s->n_seqs)
        return fail(MOE_EINVAL, "%s: %d rows of %d sequences without row_start", fn, s->n_rows, s->n_seqs);
    if (s->max_pages < 1 || s->max_pages > ((1 << 30) >> a->page_shift))
        return fail(MOE_EINVAL, "%s: page lists of %d pages of %d tokens (1 page to 2^30 tokens)", fn, s->max_pages,
                    g.page_tokens);
    if (s->pages_stride < s->max_pages)
        return fail(MOE_EINVAL, "%s: pages_stride %lld below max_pages %d", fn, (long long)s->pages_stride, s->max_pages);
    if (kv->n_pages < 1) return fail(MOE_EINVAL, "%s: a cache of %d pages", fn, kv->n_pages);
    const int64_t strides[3] = {kv->page_stride, kv->head_stride, kv->token_stride};
    for (int64_t v : strides)
        if (v < g.head_dim || (v & 7) || v > ((int64_t)1 << 40) || kv->token_stride > (1 << 22)) // (bytes in 24 bits)
            return fail(MOE_EINVAL, "%s: cache stride %lld (multiples of 8, head_dim=%d at least; token_stride at most 2^22)", fn,
                        (long long)v, g.head_dim);
    if (kv->n_pages > ((int64_t)1 << 46) / kv->page_stride)
        return fail(MOE_EINVAL, "%s: %d pages %lld elements apart", fn, kv->n_pages, (long long)kv->page_stride);
    // steps of 32 tokens, of every sequence and head, are counted in 32 bits
    const int64_t blocks = (int64_t)g.n_kv_heads * ((g.n_q_heads / g.n_kv_heads + DEC_HEADS - 1) / DEC_HEADS);
    if ((((int64_t)s->max_pages << a->page_shift) / 32 + 1) * s->n_seqs * blocks >= ((int64_t)1 << 31))
        return fail(MOE_EINVAL, "%s: %d page lists of %d pages of %d tokens are too long together", fn, s->n_seqs,
                    s->max_pages, g.page_tokens);
    *c = AttnArgs{};
    if (s->n_seqs == 0 || s->n_rows == 0) return MOE_OK; // nothing to do: no other pointer is needed
    if (!kv->k || !kv->v || !s->pages || !s->kv_len) return fail(MOE_EINVAL, "%s: null argument", fn);
    if (!aligned(kv->k, 16) || !aligned(kv->v, 16)) return fail(MOE_EINVAL, "%s: cache not 16-byte aligned", fn);
    if (!aligned(s->pages, 4) || !aligned(s->kv_len, 4) || !aligned(s->row_start, 4))
        return fail(MOE_EINVAL, "%s: misaligned sequence arrays", fn);
    c->k = (uint8_t *)kv->k;
    c->v = (uint8_t *)kv->v;
    c->page_stride = kv->page_stride;
    c->head_stride = kv->head_stride;
    c->token_stride = kv->token_stride;
    c->n_pages = kv->n_pages;
    c->pages = s->pages;
    c->pages_stride = s->pages_stride;
    c->max_pages = s->max_pages;
    c->page_shift = a->page_shift;
    c->kv_len = s->kv_len;
    c->row_start = s->row_start;
    c->n_seqs = s->n_seqs;
    c->n_rows = s->n_rows;
    c->hq = g.n_q_heads;
    c->hkv = g.n_kv_heads;
    c->group = g.n_q_heads / g.n_kv_heads;
    c->flags = a->flags;
    return MOE_OK;
}

moe_status attn_call(const char *fn, moe_attn *a, const moe_kv_cache *kv, const moe_seq_batch *s, const void *q,
                     int64_t q_stride, float scale, void *o, int64_t o_stride, float *lse, void *stream) {
    AttnArgs c;
    moe_status rc = common_args(fn, a, kv, s, &c);
    if (rc != MOE_OK) return rc;
    const int64_t row = (int64_t)a->cfg.n_q_heads * a->cfg.head_dim;
    if (q_stride < row || (q_stride & 7) || o_stride < row || (o_stride & 7))
        return fail(MOE_EINVAL, "%s: row strides %lld and %lld (multiples of 8, %lld at least)", fn,
                    (long long)q_stride, (long long)o_stride, (long long)row);
    c.scale_log2 = (float)(scale * 1.4426950408889634);
    if (!std::isfinite(c.scale_log2)) return fail(MOE_EINVAL, "%s: scale %g", fn, (double)scale);
    if (s->n_seqs == 0 || s->n_rows == 0) return ok();
    if (!q || !o) return fail(MOE_EINVAL, "%s: null argument", fn);
    if (!aligned(q, 16) || !aligned(o, 16) || !aligned(lse, 4))
        return fail(MOE_EINVAL, "%s: misaligned pointer (q and o need 16 bytes)", fn);
    if (q == o && q_stride != o_stride) return fail(MOE_EINVAL, "%s: o is q with another row stride", fn);
    if (c.row_start && prompt_places(c) >= 1 << 24) // 256 threads each: below 2^32
        return fail(MOE_EINVAL, "%s: %d rows of %d heads in %d sequences are too many", fn, s->n_rows, c.hq, s->n_seqs);
    c.q = q;
    c.q_stride = q_stride;
    c.o = o;
    c.o_stride = o_stride;
    c.lse = lse;
    c.part = a->part;
    c.part_ml = a->part_ml;
    c.part_rows = a->part_rows;
    c.piece = a->piece;
    c.n_wg = a->n_wg;
    c.n_cu = a->n_cu;
    OnDevice on(a->device);
    hipError_t he = on.he;
    if (he == hipSuccess)
        he = c.row_start ? launch_attn_prompt(c, a->cfg.type, a->cfg.head_dim, (hipStream_t)stream)
                         : launch_attn_decode(c, a->cfg.type, a->cfg.head_dim, (hipStream_t)stream);
    if (he != hipSuccess) return fail(MOE_EHIP, "%s: launch: %s", fn, hipGetErrorString(he));
    return ok();
}

} // namespace

extern "C" {

moe_status moe_attn_create(int device, const moe_attn_config *cfg, moe_attn **out) {
    static const char *fn = "moe_attn_create";
    if (!cfg || !out) return fail(MOE_EINVAL, "%s: null argument", fn);
    *out = nullptr;
    const moe_attn_config &g = *cfg;
    if (g.head_dim != 64 && g.head_dim != 128 && g.head_dim != 256)
        return fail(MOE_EUNSUPPORTED, "%s: head_dim=%d not compiled (64, 128, 256)", fn, g.head_dim);
    if (g.type != MOE_T_F16 && g.type != MOE_T_BF16)
        return fail(MOE_EUNSUPPORTED, "%s: type %d (F16 %d and BF16 %d)", fn, g.type, MOE_T_F16, MOE_T_BF16);
    if (g.n_q_heads < 1 || g.n_q_heads > 256 || g.n_kv_heads < 1 || g.n_q_heads % g.n_kv_heads)
        return fail(MOE_EINVAL, "%s: %d query heads (1..256) over %d key-value heads", fn, g.n_q_heads, g.n_kv_heads);
    if (g.page_tokens < 16 || g.page_tokens > 1024 || (g.page_tokens & (g.page_tokens - 1)))
        return fail(MOE_EINVAL, "%s: page_tokens=%d (a power of two, 16..1024)", fn, g.page_tokens);
    if (g.max_seqs < 1 || g.max_seqs > 65535)
        return fail(MOE_EINVAL, "%s: max_seqs=%d outside 1..65535", fn, g.max_seqs);
    int ndev = 0;
    hipError_t he = hipGetDeviceCount(&ndev);
    if (he != hipSuccess) return fail(MOE_EHIP, "%s: hipGetDeviceCount: %s", fn, hipGetErrorString(he));
    if (device < 0 || device >= ndev) return fail(MOE_EINVAL, "%s: device %d of %d", fn, device, ndev);
    OnDevice on(device);
    if (on.he != hipSuccess) return fail(MOE_EHIP, "%s: hipSetDevice: %s", fn, hipGetErrorString(on.he));
    moe_attn *a = new (std::nothrow) moe_attn();
    if (!a) return fail(MOE_ENOMEM, "%s: host allocation", fn);
    a->device = device;
    a->cfg = g;
    while ((1 << a->page_shift) < g.page_tokens) ++a->page_shift;
    int ncu = 0;
    if (hipDeviceGetAttribute(&ncu, hipDeviceAttributeMultiprocessorCount, device) != hipSuccess || ncu < 1) ncu = 1;
    a->n_cu = ncu;
    a->n_wg = 2 * ncu < DEC_MAX_WG ? 2 * ncu : DEC_MAX_WG;
    // decode: two slots a workgroup; prompt: a piece for each workgroup on the card (prompt_d)
    const int64_t dec_rows = (int64_t)a->n_wg * 2 * DEC_HEADS;
    const int64_t prompt_rows = (int64_t)ncu * (g.head_dim == 256 ? 1 : 2) * PR_ROWS;
    a->part_rows = dec_rows > prompt_rows ? dec_rows : prompt_rows;
    struct Part {
        void **dst;
        size_t bytes;
    } parts[] = {
        {(void **)&a->flags, 256},
        {(void **)&a->piece, (size_t)a->n_wg * sizeof(Piece)},
        {(void **)&a->part_ml, (size_t)a->part_rows * 2 * 4},
        {(void **)&a->part, (size_t)a->part_rows * g.head_dim * 4},
    };
    size_t total = 0;
    for (auto &p : parts) total += (p.bytes + 255) / 256 * 256;
    he = hipMalloc(&a->arena, total);
    if (he != hipSuccess) {
        (void)hipGetLastError();
        delete a;
        return fail(MOE_ENOMEM, "%s: hipMalloc(%zu): %s", fn, total, hipGetErrorString(he));
    }
    size_t off = 0;
    for (auto &p : parts) {
        *p.dst = (char *)a->arena + off;
        off += (p.bytes + 255) / 256 * 256;
    }
    he = hipMemset(a->arena, 0, total);
    if (he == hipSuccess) he = hipDeviceSynchronize();
    if (he != hipSuccess) {
        (void)hipFree(a->arena);
        delete a;
        return fail(MOE_EHIP, "%s: clearing workspace: %s", fn, hipGetErrorString(he));
    }
    *out = a;
    return ok();
}

moe_status moe_attn_destroy(moe_attn *a) {
    if (!a) return fail(MOE_EINVAL, "moe_attn_destroy: null handle");
    OnDevice on(a->device);
    (void)hipDeviceSynchronize();
    const hipError_t he = hipFree(a->arena);
    delete a;
    if (he != hipSuccess) return fail(MOE_EHIP, "moe_attn_destroy: hipFree: %s", hipGetErrorString(he));
    return ok();
}

moe_status moe_kv_append(moe_attn *a, const moe_kv_cache *kv, const moe_seq_batch *seqs, const void *k, const void *v,
                         int in_type, int64_t k_row_stride, int64_t v_row_stride, void *stream) {
    static const char *fn = "moe_kv_append";
    AppendArgs p;
    moe_status rc = common_args(fn, a, kv, seqs, &p.c);
    if (rc != MOE_OK) return rc;
    if (in_type != a->cfg.type && in_type != MOE_T_F32)
        return fail(MOE_EUNSUPPORTED, "%s: rows of type %d (the cache's %d, or F32)", fn, in_type, a->cfg.type);
    const int el = in_type == MOE_T_F32 ? 4 : 2;
    const int64_t row = (int64_t)a->cfg.n_kv_heads * a->cfg.head_dim;
    if (k_row_stride < row || v_row_stride < row || (k_row_stride * el & 15) || (v_row_stride * el & 15))
        return fail(MOE_EINVAL, "%s: row strides %lld and %lld (multiples of 16 bytes, %lld elements at least)", fn,
                    (long long)k_row_stride, (long long)v_row_stride, (long long)row);
    if (seqs->n_seqs == 0 || seqs->n_rows == 0) return ok();
    if (!k || !v) return fail(MOE_EINVAL, "%s: null argument", fn);
    if (!aligned(k, 16) || !aligned(v, 16)) return fail(MOE_EINVAL, "%s: k and v must be 16-byte aligned", fn);
    p.src[0] = (const uint8_t *)k;
    p.src[1] = (const uint8_t *)v;
    p.src_stride[0] = k_row_stride * el;
    p.src_stride[1] = v_row_stride * el;
    p.dst[0] = p.c.k;
    p.dst[1] = p.c.v;
    OnDevice on(a->device);
    hipError_t he = on.he;
    if (he == hipSuccess) he = launch_kv_append(p, a->cfg.type, in_type, a->cfg.head_dim, (hipStream_t)stream);
    if (he != hipSuccess) return fail(MOE_EHIP, "%s: launch: %s", fn, hipGetErrorString(he));
    return ok();
}

moe_status moe_attn_decode(moe_attn *a, const moe_kv_cache *kv, const moe_seq_batch *seqs, const void *q,
                           int64_t q_row_stride, float scale, void *o, int64_t o_row_stride, float *lse,
                           void *stream) {
    if (seqs && seqs->row_start)
        return fail(MOE_EINVAL, "moe_attn_decode: row_start given (one row a sequence; others: moe_attn_prompt)");
    return attn_call("moe_attn_decode", a, kv, seqs, q, q_row_stride, scale, o, o_row_stride, lse, stream);
}

moe_status moe_attn_prompt(moe_attn *a, const moe_kv_cache *kv, const moe_seq_batch *seqs, const void *q,
                           int64_t q_row_stride, float scale, void *o, int64_t o_row_stride, float *lse,
                           void *stream) {
    return attn_call("moe_attn_prompt", a, kv, seqs, q, q_row_stride, scale, o, o_row_stride, lse, stream);
}

moe_status moe_attn_flags(moe_attn *a, void *stream, uint32_t *flags) {
    static const char *fn = "moe_attn_flags";
    if (!a || !flags) return fail(MOE_EINVAL, "%s: null argument", fn);
    OnDevice on(a->device);
    hipError_t he = on.he;
    if (he == hipSuccess) he = hipStreamSynchronize((hipStream_t)stream);
    uint32_t v = 0;
    if (he == hipSuccess) he = hipMemcpy(&v, a->flags, 4, hipMemcpyDeviceToHost);
    if (he == hipSuccess && v) he = hipMemset(a->flags, 0, 4);
    if (he == hipSuccess && v) he = hipDeviceSynchronize();
    if (he != hipSuccess) return fail(MOE_EHIP, "%s: %s", fn, hipGetErrorString(he));
    *flags = v;
    return ok();
}

moe_status moe_attn_flags_async(moe_attn *a, uint32_t *dst, void *stream) {
    static const char *fn = "moe_attn_flags_async";
    if (!a || !dst) return fail(MOE_EINVAL, "%s: null argument", fn);
    if (!aligned(dst, 4)) return fail(MOE_EINVAL, "%s: dst not 4-byte aligned", fn);
    OnDevice on(a->device);
    hipError_t he = on.he;
    if (he == hipSuccess) he = launch_attn_flags(a->flags, dst, (hipStream_t)stream);
    if (he != hipSuccess) return fail(MOE_EHIP, "%s: launch: %s", fn, hipGetErrorString(he));
    return ok();
}

} // extern "C"

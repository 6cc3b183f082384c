// C entry points of the cache operators: argument checks and the views the
// kernels take (xattn_rope.h, xattn_cache_attend.h).  Host code only.
#pragma once

#include <math.h>

#include <algorithm>

#include "xattn_cache_attend.h"
#include "xattn_rope.h"

namespace xattn {
namespace cache {

static bool refuse(const char* who, const char* why) {
    set_error(XATTN_ERR_INVALID_VALUE, "%s: %s", who, why);
    return false;
}

static int type_size(int dtype) { return dtype == XATTN_F32 ? 4 : 2; }

static bool check_type(const char* who, int dtype) {
    if (dtype == XATTN_F32 || dtype == XATTN_F16 || dtype == XATTN_BF16) return true;
    set_error(XATTN_ERR_INVALID_VALUE, "%s: unknown element type %d", who, dtype);
    return false;
}

// A token tensor of `heads` heads of `dim`: rows stride elements apart, every
// address a multiple of `align` bytes.
static bool check_rows(const char* who, const char* name, const void* p, long long stride,
                       int heads, int dim, int size, int align) {
    if (!p) {
        set_error(XATTN_ERR_INVALID_VALUE, "%s: NULL %s", who, name);
        return false;
    }
    if (stride < (long long)heads * dim) {
        set_error(XATTN_ERR_INVALID_VALUE, "%s: %s rows %lld elements apart hold no %d x %d", who,
                  name, stride, heads, dim);
        return false;
    }
    if ((uintptr_t)p % align != 0 || (stride % align * size) % align != 0) {
        set_error(XATTN_ERR_INVALID_VALUE, "%s: %s at %p, rows %lld elements apart, is not "
                  "%d-byte aligned", who, name, p, stride, align);
        return false;
    }
    return true;
}

static bool view_rope(const char* who, const xattn_rope* rope, int dim, int inverse, Rope* out) {
    *out = Rope{nullptr, 1.0f, 0, false, inverse != 0};
    if (!rope) return true;
    if (rope->rot_dim < 0 || rope->rot_dim % 2 != 0 || rope->rot_dim > dim) {
        set_error(XATTN_ERR_INVALID_VALUE, "%s: rot_dim %d is not an even number of 0..%d", who,
                  rope->rot_dim, dim);
        return false;
    }
    if (rope->rot_dim > kMaxRot) {
        set_error(XATTN_ERR_UNSUPPORTED, "%s: rot_dim %d over %d", who, rope->rot_dim, kMaxRot);
        return false;
    }
    if (rope->rot_dim > 0 && !rope->freqs) return refuse(who, "NULL frequencies");
    if ((uintptr_t)rope->freqs % sizeof(double) != 0)
        return refuse(who, "frequencies are not 8-byte aligned");
    if (!isfinite(rope->amplitude)) return refuse(who, "the amplitude is not finite");
    out->freqs = rope->freqs;
    out->amplitude = rope->amplitude;
    out->rot = rope->rot_dim;
    out->interleaved = rope->interleaved != 0;
    return true;
}

static bool view_pages(const char* who, const xattn_kv_cache* c, Pages* out) {
    if (!c) return refuse(who, "NULL cache");
    if (!check_type(who, c->dtype)) return false;
    if (c->num_pages < 0 || c->kv_heads < 1 || c->page_size < 1 || c->dim < 1) {
        set_error(XATTN_ERR_INVALID_VALUE,
                  "%s: a cache of num_pages=%d kv_heads=%d page_size=%d dim=%d", who,
                  c->num_pages, c->kv_heads, c->page_size, c->dim);
        return false;
    }
    const unsigned __int128 rows =
        (unsigned __int128)c->num_pages * (unsigned)c->kv_heads * (unsigned)c->page_size;
    if (rows > 0xffffffffu || (long long)c->kv_heads * c->page_size > 0x7fffffffLL ||
        (long long)c->kv_heads * c->dim > 0x7ffffff) {
        set_error(XATTN_ERR_UNSUPPORTED, "%s: a cache of over 2^32 - 1 rows, a page of over 2^31 "
                  "or a token of over 2^27 elements", who);
        return false;
    }
    if (c->num_pages > 0 && (!c->k || !c->v)) return refuse(who, "NULL pages");
    if ((uintptr_t)c->k % 16 != 0 || (uintptr_t)c->v % 16 != 0)
        return refuse(who, "pages are not 16-byte aligned");
    *out = Pages{(char*)c->k, (char*)c->v, (unsigned)c->num_pages, (unsigned)c->kv_heads,
                 FastDiv::of((unsigned)c->page_size), c->dim};
    return true;
}

static bool view_batch(const char* who, const xattn_batch* b, int page_size, bool sizes_only,
                       Batch* out) {
    if (!b) return refuse(who, "NULL batch");
    if (b->batch < 0 || b->table_width < 0 || b->tokens < 0 || b->max_q_len < 0 ||
        b->max_kv_len < 0) {
        set_error(XATTN_ERR_INVALID_VALUE,
                  "%s: a batch of batch=%d table_width=%d tokens=%d max_q_len=%d max_kv_len=%d",
                  who, b->batch, b->table_width, b->tokens, b->max_q_len, b->max_kv_len);
        return false;
    }
    if (!sizes_only && b->batch > 0 &&
        (!b->q_starts || !b->kv_lens || (b->table_width > 0 && !b->page_table)))
        return refuse(who, "NULL q_starts, kv_lens or page_table");
    if (((uintptr_t)b->q_starts | (uintptr_t)b->kv_lens | (uintptr_t)b->page_table) % 4 != 0)
        return refuse(who, "q_starts, kv_lens or page_table is not 4-byte aligned");
    if ((long long)b->table_width * page_size > kMaxKeys) {
        set_error(XATTN_ERR_UNSUPPORTED, "%s: rows of page_table for over 2^30 keys", who);
        return false;
    }
    *out = Batch{b->q_starts, b->kv_lens, b->page_table, b->batch, b->table_width, b->tokens,
                 (long long)b->table_width * page_size};
    return true;
}

// The checks that the scratch query and the launchers share; heads 64-bit
// products stay within 32 bits.
static bool view_attention(const char* who, const xattn_kv_cache* cache, const xattn_batch* batch,
                           const xattn_prefix* prefix, int heads, bool sizes_only,
                           Attention* a) {
    *a = Attention{};
    if (!view_pages(who, cache, &a->pages)) return false;
    if (!view_batch(who, batch, cache->page_size, sizes_only, &a->batch)) return false;
    if (cache->dim != 64 && cache->dim != 128 && cache->dim != 256 && cache->dim != kDim) {
        set_error(XATTN_ERR_UNSUPPORTED, "%s: dim=%d unsupported (64, 128, 256 or %d)", who,
                  cache->dim, kDim);
        return false;
    }
    if (heads < 1 || heads % cache->kv_heads != 0) {
        set_error(XATTN_ERR_INVALID_VALUE, "%s: %d heads over %d kv heads", who, heads,
                  cache->kv_heads);
        return false;
    }
    if ((long long)heads * std::max(std::max(batch->tokens, batch->batch), 1) > 0x1fffffff) {
        set_error(XATTN_ERR_UNSUPPORTED, "%s: %d tokens of %d heads in one call", who,
                  batch->tokens, heads);
        return false;
    }
    if (prefix) {
        if (prefix->len < 0 || prefix->num_listed < 0 ||
            (long long)prefix->num_listed * cache->page_size < prefix->len) {
            set_error(XATTN_ERR_INVALID_VALUE, "%s: a prefix of %d keys on %d pages of %d", who,
                      prefix->len, prefix->num_listed, cache->page_size);
            return false;
        }
        if (prefix->len > kMaxKeys) {
            set_error(XATTN_ERR_UNSUPPORTED, "%s: a prefix of over 2^30 keys", who);
            return false;
        }
        if (!sizes_only && prefix->len > 0 && !prefix->pages)
            return refuse(who, "NULL prefix pages");
        if ((uintptr_t)prefix->pages % 4 != 0)
            return refuse(who, "prefix pages are not 4-byte aligned");
        a->prefix_pages = prefix->pages;
        a->prefix_listed = prefix->num_listed;
        a->prefix_len = prefix->len;
    }
    a->dtype = cache->dtype;
    a->heads = heads;
    a->max_q = std::min(batch->max_q_len, batch->tokens);
    a->max_kv = (int)std::min<long long>(batch->max_kv_len, a->batch.capacity);
    return true;
}

static void attention(const char* who, const xattn_kv_cache* cache, const xattn_batch* batch,
                      const xattn_prefix* prefix, const void* q, long long q_stride, void* out,
                      long long out_stride, int heads, float scale, int causal, void* scratch,
                      size_t scratch_bytes, hipStream_t stream) {
    Attention a;
    if (!view_attention(who, cache, batch, prefix, heads, false, &a)) return;
    if (!isfinite(scale)) {
        refuse(who, "the scale is not finite");
        return;
    }
    if (a.batch.batch == 0 || a.batch.tokens == 0 || a.max_q == 0) return;
    const int size = type_size(a.dtype);
    if (!check_rows(who, "q", q, q_stride, heads, cache->dim, size, 16)) return;
    if (!check_rows(who, "out", out, out_stride, heads, cache->dim, size, 16)) return;
    if (out == q) {
        refuse(who, "out may not be q");
        return;
    }
    const size_t need = attention_scratch(a);
    if (need > 0 && (!scratch || scratch_bytes < need || (uintptr_t)scratch % 16 != 0)) {
        set_error(XATTN_ERR_INVALID_VALUE,
                  "%s: scratch of %zu bytes at %p; %zu are needed, 16-byte aligned", who,
                  scratch ? scratch_bytes : (size_t)0, scratch, need);
        return;
    }
    a.q = q;
    a.out = out;
    a.qs = q_stride;
    a.os = out_stride;
    a.scale = scale;
    a.causal = causal != 0;
    launch_attention(a, scratch, stream);
}

extern "C" {

int xattn_rope_frequencies(double* freqs, int rot_dim, double base, int scaling, double factor,
                           int trained_len, double slow_turns, double fast_turns) {
    const char* who = "xattn_rope_frequencies";
    const char* why = nullptr;
    if (rot_dim < 0 || rot_dim % 2 != 0 || (rot_dim > 0 && !freqs))
        why = "rot_dim is not an even number, or there is no array";
    else if (!(base > 0 && isfinite(base) && factor > 0 && isfinite(factor)))
        why = "base and factor have to be positive and finite";
    else if (scaling < XATTN_ROPE_PLAIN || scaling > XATTN_ROPE_PARTS)
        why = "unknown scaling";
    else if (scaling == XATTN_ROPE_BASE && rot_dim == 2)
        why = "a single pair has no base to scale";
    else if (scaling == XATTN_ROPE_PARTS &&
             !(trained_len >= 1 && slow_turns >= 0 && slow_turns < fast_turns &&
               isfinite(fast_turns)))
        why = "the blend needs a trained length and 0 <= slow_turns < fast_turns";
    if (why) {
        refuse(who, why);
        return XATTN_ERR_INVALID_VALUE;
    }
    if (scaling == XATTN_ROPE_BASE) base *= pow(factor, (double)rot_dim / (rot_dim - 2));
    for (int i = 0; i < rot_dim / 2; ++i) {
        double f = pow(base, -2.0 * i / rot_dim) / (2.0 * M_PI);
        if (scaling == XATTN_ROPE_LINEAR) f /= factor;
        if (scaling == XATTN_ROPE_PARTS) {
            const double keep = (f * trained_len - slow_turns) / (fast_turns - slow_turns);
            const double g = keep < 0 ? 0 : keep > 1 ? 1 : keep;
            f = f * g + f / factor * (1 - g);
        }
        freqs[i] = f;
    }
    return XATTN_OK;
}

void launch_rope_kernel(const void* x, void* y, const int* positions, const xattn_rope* rope,
                        int dtype, int tokens, int heads, int dim, long long x_stride,
                        long long y_stride, int inverse, hipStream_t stream) {
    const char* who = "launch_rope_kernel";
    if (!check_type(who, dtype)) return;
    if (tokens < 0 || heads < 0 || dim < 1) {
        set_error(XATTN_ERR_INVALID_VALUE, "%s: tokens=%d heads=%d dim=%d", who, tokens, heads,
                  dim);
        return;
    }
    if ((long long)heads * dim > 0x7ffffff) {
        set_error(XATTN_ERR_UNSUPPORTED, "%s: a token of over 2^27 elements", who);
        return;
    }
    if (!rope) {
        refuse(who, "NULL rotation");
        return;
    }
    Rope r;
    if (!view_rope(who, rope, dim, inverse, &r)) return;
    if (tokens == 0 || heads == 0) return;
    const int size = type_size(dtype);
    if (!check_rows(who, "x", x, x_stride, heads, dim, size, size)) return;
    if (!check_rows(who, "y", y, y_stride, heads, dim, size, size)) return;
    if (x == y && x_stride != y_stride) {
        refuse(who, "in place, both strides have to be the same");
        return;
    }
    if (r.rot > 0 && (!positions || (uintptr_t)positions % 4 != 0)) {
        refuse(who, "NULL or unaligned positions");
        return;
    }
    launch_rope(x, y, positions, r, dtype, tokens, heads, dim, x_stride, y_stride, stream);
}

void launch_cache_append_kernel(const xattn_kv_cache* cache, const xattn_batch* batch,
                                const void* k, long long k_stride, const void* v,
                                long long v_stride, const void* q, long long q_stride,
                                void* q_out, long long q_out_stride, int heads,
                                const int* positions, const xattn_rope* rope,
                                hipStream_t stream) {
    const char* who = "launch_cache_append_kernel";
    Pages pages;
    Batch b;
    Rope r;
    if (!view_pages(who, cache, &pages)) return;
    if (!view_batch(who, batch, cache->page_size, false, &b)) return;
    if (!view_rope(who, rope, cache->dim, 0, &r)) return;
    if (q && (heads < 1 || (long long)heads * cache->dim > 0x7ffffff)) {
        set_error(XATTN_ERR_INVALID_VALUE, "%s: %d query heads of %d", who, heads, cache->dim);
        return;
    }
    if (b.batch == 0 || b.tokens == 0) return;
    const int size = type_size(cache->dtype), dim = cache->dim;
    if (!check_rows(who, "k", k, k_stride, cache->kv_heads, dim, size, size)) return;
    if (!check_rows(who, "v", v, v_stride, cache->kv_heads, dim, size, size)) return;
    if (q) {
        if (!check_rows(who, "q", q, q_stride, heads, dim, size, size)) return;
        if (!check_rows(who, "q_out", q_out, q_out_stride, heads, dim, size, size)) return;
        if (q == q_out && q_stride != q_out_stride) {
            refuse(who, "in place, both strides have to be the same");
            return;
        }
    }
    if ((uintptr_t)positions % 4 != 0) {
        refuse(who, "positions are not 4-byte aligned");
        return;
    }
    launch_append(pages, b, r, cache->dtype, k, k_stride, v, v_stride, q, q_stride, q_out,
                  q_out_stride, heads, positions, stream);
}

size_t xattn_cache_attention_scratch(const xattn_kv_cache* cache, const xattn_batch* batch,
                                     const xattn_prefix* prefix, int heads) {
    Attention a;
    if (!view_attention("xattn_cache_attention_scratch", cache, batch, prefix, heads, true, &a))
        return 0;
    return a.batch.batch == 0 || a.batch.tokens == 0 || a.max_q == 0 ? 0 : attention_scratch(a);
}

void launch_cache_attention_kernel(const xattn_kv_cache* cache, const xattn_batch* batch,
                                   const void* q, long long q_stride, void* out,
                                   long long out_stride, int heads, float scale, int causal,
                                   void* scratch, size_t scratch_bytes, hipStream_t stream) {
    attention("launch_cache_attention_kernel", cache, batch, nullptr, q, q_stride, out,
              out_stride, heads, scale, causal, scratch, scratch_bytes, stream);
}

void launch_prefix_attention_kernel(const xattn_kv_cache* cache, const xattn_batch* batch,
                                    const xattn_prefix* prefix, const void* q,
                                    long long q_stride, void* out, long long out_stride,
                                    int heads, float scale, int causal, void* scratch,
                                    size_t scratch_bytes, hipStream_t stream) {
    const char* who = "launch_prefix_attention_kernel";
    if (!prefix) {
        set_error(XATTN_ERR_INVALID_VALUE, "%s: NULL prefix", who);
        return;
    }
    attention(who, cache, batch, prefix, q, q_stride, out, out_stride, heads, scale, causal,
              scratch, scratch_bytes, stream);
}

}  // extern "C"

}  // namespace cache
}  // namespace xattn

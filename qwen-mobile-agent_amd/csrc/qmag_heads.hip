// qmag_heads.hip -- host checks of the attention entries' descriptors.
#include "qmag_attn.h"

namespace qmag {

DeviceScope::DeviceScope()
{
    int cur = -1;
    hipError_t e = hipGetDevice(&cur);
    if (e == hipSuccess && cur != ctx().dev) {
        e = hipSetDevice(ctx().dev);
        if (e == hipSuccess) was = cur;
    }
    if (e != hipSuccess) st = hip_fail(e, "device of the library", __FILE__, __LINE__);
}

DeviceScope::~DeviceScope()
{
    if (was >= 0) (void)hipSetDevice(was);
}

// values from the first one to behind the last
static int64_t extent(const qmag_heads *h, int dim, int64_t n_tok)
{
    if (h->n_head == 0 || n_tok == 0) return 0;
    return (n_tok - 1) * h->token_stride + (h->n_head - 1) * h->head_stride + dim;
}

int check_heads(const char *what, const qmag_heads *h, int type, int dim, int64_t n_tok, bool written)
{
    const int size = attn_type_size(type);
    if (!size) return fail(QMAG_ERR_ARG, "%s: type %d", what, type);
    if (h->n_head < 0 || h->n_head > QMAG_MAX_HEADS) return fail(QMAG_ERR_ARG, "%s: %d heads", what, h->n_head);
    if (h->n_head == 0 || n_tok == 0) return QMAG_OK;
    if (!h->ptr) return fail(QMAG_ERR_ARG, "%s: null pointer", what);
    if ((uintptr_t)h->ptr % (unsigned)size) return fail(QMAG_ERR_ARG, "%s: not aligned to its values", what);
    // 2^59 values at most: no place, in bytes either, leaves 64 bits
    const int64_t most = (int64_t)1 << 58;
    if (h->token_stride < 0 || h->head_stride < 0 || h->token_stride > most / n_tok || h->head_stride > most / h->n_head)
        return fail(QMAG_ERR_ARG, "%s: strides %lld, %lld", what, (long long)h->token_stride, (long long)h->head_stride);
    if (!written) return QMAG_OK;
    const int64_t ts = h->token_stride, hs = h->head_stride;
    const bool by_token = (h->n_head == 1 || hs >= dim) && (n_tok == 1 || ts >= (h->n_head - 1) * hs + dim);
    const bool by_head = (n_tok == 1 || ts >= dim) && (h->n_head == 1 || hs >= (n_tok - 1) * ts + dim);
    if (!by_token && !by_head)
        return fail(QMAG_ERR_ARG, "%s: strides %lld, %lld put two of its values in one place", what, (long long)ts,
                    (long long)hs);
    return QMAG_OK;
}

bool heads_aligned(const qmag_heads *h, int type)
{
    const int64_t v = 16 / attn_type_size(type);
    return h->n_head == 0 || ((uintptr_t)h->ptr % 16 == 0 && h->token_stride % v == 0 && h->head_stride % v == 0);
}

// whether ranges of ea and eb values, repeated every `stride` values from
// places `apart` values from one another, never meet
static bool side_by_side(int64_t apart, int64_t stride, int64_t ea, int64_t eb)
{
    if (stride <= 0 || ea > stride || eb > stride) return false;
    const int64_t d = ((apart % stride) + stride) % stride;
    return d >= eb && d + ea <= stride;
}

bool heads_overlap(const qmag_heads *a, const qmag_heads *b, int size, int dim, int64_t n_tok)
{
    const int64_t na = extent(a, dim, n_tok), nb = extent(b, dim, n_tok);
    if (na == 0 || nb == 0) return false;
    const intptr_t pa = (intptr_t)a->ptr, pb = (intptr_t)b->ptr;
    if (pa + na * size <= pb || pb + nb * size <= pa) return false;
    if ((pa - pb) % size) return true;
    const int64_t apart = (pa - pb) / size;
    if (a->token_stride == b->token_stride &&
        side_by_side(apart, a->token_stride, extent(a, dim, 1), extent(b, dim, 1)))
        return false;
    const int64_t hs = a->n_head > 1 ? a->head_stride : b->head_stride;
    const bool heads_alike = (a->n_head == 1 || a->head_stride == hs) && (b->n_head == 1 || b->head_stride == hs);
    if (heads_alike && side_by_side(apart, hs, (n_tok - 1) * a->token_stride + dim, (n_tok - 1) * b->token_stride + dim)) return false;
    const bool whole = hs > 0 && a->token_stride % hs == 0 && b->token_stride % hs == 0;
    if (whole && heads_alike && side_by_side(apart, hs, dim, dim))
        return false;
    return true;
}

bool heads_meet(const qmag_heads *h, int size, int dim, int64_t n_tok, const void *p, size_t bytes)
{
    const int64_t all = extent(h, dim, n_tok);
    const uintptr_t a = (uintptr_t)h->ptr, b = (uintptr_t)p;
    if (all == 0 || bytes == 0 || a + (uintptr_t)(all * size) <= b || b + bytes <= a) return false;
    // bytes from h's first value: rows of `row` bytes, inner ones within outer ones
    const int64_t row = (int64_t)dim * size, lo = (int64_t)(b - a), hi = lo + (int64_t)bytes;
    int64_t so = h->token_stride * size, si = h->head_stride * size, no = n_tok, ni = h->n_head;
    if (so < si) {
        const int64_t s = so, n = no;
        so = si, no = ni, si = s, ni = n;
    }
    if (so == 0) return true;                      // a single row, and it lies there
    if (si == 0) ni = 1;
    // the first outer one that begins at or behind lo, then those before it that reach behind lo
    const int64_t first = lo <= 0 ? 0 : (lo + so - 1) / so;
    if (first < no && first * so < hi) return true;
    for (int64_t o = (first < no ? first : no) - 1; o >= 0 && o * so + (ni - 1) * si + row > lo; o--) {
        const int64_t d = lo - row - o * so, j = d < 0 || si == 0 ? 0 : d / si + 1;      // the first inner row that ends behind lo
        if (j < ni && o * so + j * si + row > lo && o * so + j * si < hi) return true;
    }
    return false;
}

int check_kv4(const qmag_kv4 *c)
{
    if (!c) return fail(QMAG_ERR_ARG, "kv4: null cache");
    if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
        return fail(QMAG_ERR_ARG, "kv4: head_dim %d (64, 128 or 256)", c->head_dim);
    if (c->block_size < 16 || c->block_size > 256 || (c->block_size & (c->block_size - 1)))
        return fail(QMAG_ERR_ARG, "kv4: block_size %d (a power of two from 16 to 256)", c->block_size);
    if (c->n_kv < 1 || c->n_kv > QMAG_MAX_HEADS) return fail(QMAG_ERR_ARG, "kv4: n_kv %d", c->n_kv);
    if (c->n_block < 1 || c->n_block > INT32_MAX / c->block_size)
        return fail(QMAG_ERR_ARG, "kv4: %d blocks of %d tokens", c->n_block, c->block_size);
    if (!c->data || (uintptr_t)c->data % 16) return fail(QMAG_ERR_ARG, "kv4: data is null or not 16-byte aligned");
    return QMAG_OK;
}

}  // namespace qmag

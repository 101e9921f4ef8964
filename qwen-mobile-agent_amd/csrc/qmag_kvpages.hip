// qmag_kvpages.hip -- the bookkeeping of a paged cache on the device: blocks
// given back by ended sequences, blocks for new tokens, the slot and position
// of every new token.  Lengths stay on the device, so a step needs no copy to
// the host.
//
// Every workgroup forms both prefix sums over the sequences (new tokens, new
// blocks) for itself in LDS and then writes its share of the tokens and of the
// table: no workgroup waits for another, and a step is one launch.  The k-th
// block taken in a call is free_list[n_free - 1 - k], so a token's slot does
// not need the table entry another workgroup writes.  Bound by the launch and the
// chain lengths - sums - search - table: 48 sequences, one token each, 3.5 us given
// back and 4.7 assigned; 509 sequences and 262,144 tokens 5.0 and 6.6.
#include "qmag_attn.h"

namespace qmag {

constexpr int PG_WG = 256;
constexpr int PG_TOK = 4;                  // consecutive tokens of a thread and step

// Exclusive prefix sums over the workgroup of one count per thread; the totals
// come back too.  In 64 bits: lengths are the caller's data.
struct PgScan {
    long long tok, blk;
    int bad;                               // bits of any thread
};
__device__ __forceinline__ PgScan pg_scan(PgScan v, PgScan *total, PgScan *wave_sum)
{
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const PgScan in = {wave_scan(v.tok), wave_scan(v.blk), (__any(v.bad & 1) ? 1 : 0) | (__any(v.bad & 2) ? 2 : 0)};
    if (lane == 63) wave_sum[w] = in;
    __syncthreads();
    PgScan base = {0, 0, 0}, all = {0, 0, 0};
#pragma unroll
    for (int i = 0; i < PG_WG / 64; i++) {
        if (i < w) {
            base.tok += wave_sum[i].tok;
            base.blk += wave_sum[i].blk;
        }
        all.tok += wave_sum[i].tok;
        all.blk += wave_sum[i].blk;
        all.bad |= wave_sum[i].bad;
    }
    *total = all;
    return {base.tok + in.tok - v.tok, base.blk + in.blk - v.blk, 0};
}

// the last i in [0, n) with off[i] <= k (off ascending, off[0] = 0, k < off[n])
__device__ __forceinline__ int pg_find(const int *off, int n, int k)
{
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (off[mid] <= k) lo = mid;
        else hi = mid;
    }
    return lo;
}

struct PgArgs {
    int n_seq, max_blocks, shift, n_block, T;
    int *table, *free_list;
    const int *len, *what, *n_free;        // what: new tokens, or ended flags
    int *slot, *pos, *cu, *len_next, *n_free_next, *status;
};

// blocks of n tokens (n >= 0)
__device__ __forceinline__ int pg_blocks(int n, int shift) { return (int)(((unsigned)n + (1u << shift) - 1u) >> shift); }

// What both kernels begin with.  ASSIGN: tok[i] and blk[i] become the tokens and
// blocks of the sequences before i, held[i] its length; otherwise blk[i] the blocks given back
// before i.  Returns the status every workgroup agrees on.
template <bool ASSIGN>
__device__ __forceinline__ int pg_plan(const PgArgs &A, int *tok, int *blk, int *held, PgScan *wave_sum, int n_free, PgScan *total)
{
    const int per = (A.n_seq + PG_WG - 1) / PG_WG, a = min(A.n_seq, (int)threadIdx.x * per), b = min(A.n_seq, a + per);
    PgScan mine = {0, 0, 0};
    int bad = 0;
    for (int i = a; i < b; i++) {
        const int len = A.len[i], w = A.what[i];
        int n = 0, t = 0;
        if (ASSIGN) {
            if (len < 0 || w < 0 || w > INT32_MAX - len) bad |= 1;
            else {
                const int after = pg_blocks(len + w, A.shift);
                if (after > A.max_blocks) bad |= 2;
                n = after - pg_blocks(len, A.shift);
                t = w;
            }
        } else if (w) {
            if (len < 0) bad |= 1;
            else if ((n = pg_blocks(len, A.shift)) > A.max_blocks) bad |= 2;
        }
        if (ASSIGN) tok[i] = t, held[i] = len;
        blk[i] = n;
        mine.tok += t;
        mine.blk += n;
    }
    mine.bad = bad;
    PgScan at = pg_scan(mine, total, wave_sum);
    if ((total->bad & 1) || total->tok > (ASSIGN ? A.T : 0)) return QMAG_KV_LENGTH;
    if (total->bad & 2) return QMAG_KV_ROW;
    if (n_free < 0 || n_free > A.n_block) return QMAG_KV_LIST;
    if (ASSIGN ? total->blk > n_free : total->blk > A.n_block - n_free) return ASSIGN ? QMAG_KV_FULL : QMAG_KV_LIST;
    for (int i = a; i < b; i++) {
        const int n = blk[i];
        blk[i] = (int)at.blk;
        at.blk += n;
        if (ASSIGN) {
            const int t = tok[i];
            tok[i] = (int)at.tok;
            at.tok += t;
        }
    }
    if (threadIdx.x == 0) {
        blk[A.n_seq] = (int)total->blk;
        if (ASSIGN) tok[A.n_seq] = (int)total->tok;
    }
    __syncthreads();
    return QMAG_KV_OK;
}

__global__ void __launch_bounds__(PG_WG) kv_assign_kernel(PgArgs A)
{
    __shared__ int tok[QMAG_KV_MAX_SEQ + 1], blk[QMAG_KV_MAX_SEQ + 1], held[QMAG_KV_MAX_SEQ];
    __shared__ PgScan wave_sum[PG_WG / 64];
    const int n_free = *A.n_free;
    PgScan total;
    const int st = pg_plan<true>(A, tok, blk, held, wave_sum, n_free, &total);
    const int tid = threadIdx.x;
    if (blockIdx.x == 0) {
        for (int i = tid; i < A.n_seq; i += PG_WG) {
            A.cu[i] = st ? 0 : tok[i];
            A.len_next[i] = held[i] + (st ? 0 : A.what[i]);
        }
        if (tid == 0) {
            A.cu[A.n_seq] = st ? 0 : tok[A.n_seq];
            *A.n_free_next = st ? n_free : n_free - (int)total.blk;
            *A.status = st;
        }
    }
    const int n_tok = st ? 0 : (int)total.tok;
    const int step = (int)gridDim.x * PG_WG;
    if (!st)
        for (int k = (int)blockIdx.x * PG_WG + tid; k < total.blk; k += step) {
            const int i = pg_find(blk, A.n_seq, k);
            const int64_t col = pg_blocks(held[i], A.shift) + k - blk[i];
            A.table[i * (int64_t)A.max_blocks + col] = A.free_list[n_free - 1 - k];
        }
    const bool vec = ((uintptr_t)A.slot | (uintptr_t)A.pos) % 16 == 0;
    for (int64_t t0 = ((int64_t)blockIdx.x * PG_WG + tid) * PG_TOK; t0 < A.T; t0 += (int64_t)step * PG_TOK) {
        int sl[PG_TOK], ps[PG_TOK];
        int i = t0 < n_tok ? pg_find(tok, A.n_seq, (int)t0) : 0;
#pragma unroll
        for (int j = 0; j < PG_TOK; j++) {
            const int t = (int)t0 + j;
            sl[j] = -1;
            ps[j] = 0;
            if (t0 + j >= n_tok) continue;
            while (tok[i + 1] <= t) i++;
            const int len = held[i], had = pg_blocks(len, A.shift);
            const int p = len + t - tok[i], col = p >> A.shift;
            const int id = col < had ? A.table[i * (int64_t)A.max_blocks + col]
                                     : A.free_list[n_free - 1 - (blk[i] + col - had)];
            if (id >= 0 && id < A.n_block) sl[j] = (id << A.shift) + (p & ((1 << A.shift) - 1));
            ps[j] = p;
        }
        if (vec && t0 + PG_TOK <= A.T) {
            *reinterpret_cast<int4 *>(A.slot + t0) = make_int4(sl[0], sl[1], sl[2], sl[3]);
            *reinterpret_cast<int4 *>(A.pos + t0) = make_int4(ps[0], ps[1], ps[2], ps[3]);
        } else {
            for (int j = 0; j < PG_TOK && t0 + j < A.T; j++) {
                A.slot[t0 + j] = sl[j];
                A.pos[t0 + j] = ps[j];
            }
        }
    }
}

__global__ void __launch_bounds__(PG_WG) kv_release_kernel(PgArgs A)
{
    __shared__ int blk[QMAG_KV_MAX_SEQ + 1];
    __shared__ PgScan wave_sum[PG_WG / 64];
    const int n_free = *A.n_free;
    PgScan total;
    const int st = pg_plan<false>(A, nullptr, blk, nullptr, wave_sum, n_free, &total);
    const int tid = threadIdx.x;
    if (blockIdx.x == 0) {
        for (int i = tid; i < A.n_seq; i += PG_WG) A.len_next[i] = !st && A.what[i] ? 0 : A.len[i];
        if (tid == 0) {
            *A.n_free_next = st ? n_free : n_free + (int)total.blk;
            *A.status = st;
        }
    }
    if (st) return;
    for (int k = (int)blockIdx.x * PG_WG + tid; k < total.blk; k += (int)gridDim.x * PG_WG) {
        const int i = pg_find(blk, A.n_seq, k);
        A.free_list[n_free + k] = A.table[i * (int64_t)A.max_blocks + (k - blk[i])];
    }
}

static int check_table(const qmag_kv_table *t)
{
    if (!t || !t->table || !t->free_list) return fail(QMAG_ERR_ARG, "kv table: null pointer");
    if (t->n_seq < 0 || t->n_seq > QMAG_KV_MAX_SEQ || t->max_blocks < 1)
        return fail(QMAG_ERR_ARG, "kv table: n_seq=%d max_blocks=%d", t->n_seq, t->max_blocks);
    if (t->block_size < 16 || t->block_size > 256 || (t->block_size & (t->block_size - 1)))
        return fail(QMAG_ERR_ARG, "kv table: block_size %d (a power of two from 16 to 256)", t->block_size);
    if (t->n_block < 1 || t->n_block > INT32_MAX / t->block_size)
        return fail(QMAG_ERR_ARG, "kv table: %d blocks of %d tokens", t->n_block, t->block_size);
    return QMAG_OK;
}

struct Range {
    const int *p;
    int64_t n;
};

static bool ranges_meet(const Range &x, const Range &y)
{
    const uintptr_t a = (uintptr_t)x.p, b = (uintptr_t)y.p;
    return x.n > 0 && y.n > 0 && a < b + (uintptr_t)y.n * sizeof(int) && b < a + (uintptr_t)x.n * sizeof(int);
}

// The first n_out ranges are written, the others read: aligned, and none of the
// written ones meets another.
static int check_ranges(const char *what, const Range *r, int n_out, int n)
{
    for (int i = 0; i < n; i++) {
        if ((uintptr_t)r[i].p % sizeof(int)) return fail(QMAG_ERR_ARG, "%s: a pointer is not aligned", what);
        for (int j = 0; j < n_out && j < i; j++)
            if (ranges_meet(r[i], r[j])) return fail(QMAG_ERR_ARG, "%s: what is written goes to places of its own", what);
    }
    return QMAG_OK;
}

// The table and the free list, of which a call writes one, against what else it
// takes.  (A descriptor with the two in one place holds no blocks yet and is not
// looked into.)
static int check_lists(const char *what, const qmag_kv_table *t, bool table_written, const Range *r, int n_out, int n)
{
    const Range table = {t->table, (int64_t)t->n_seq * t->max_blocks}, list = {t->free_list, t->n_block};
    if ((uintptr_t)table.p % sizeof(int) || (uintptr_t)list.p % sizeof(int))
        return fail(QMAG_ERR_ARG, "%s: the table or the free list is not aligned", what);
    if (table.p == list.p) return QMAG_OK;
    if (ranges_meet(table, list)) return fail(QMAG_ERR_ARG, "%s: the table and the free list overlap", what);
    for (int i = 0; i < n; i++)
        if (i < n_out ? ranges_meet(r[i], table) || ranges_meet(r[i], list) : ranges_meet(r[i], table_written ? table : list))
            return fail(QMAG_ERR_ARG, "%s: the table or the free list overlaps another argument", what);
    return QMAG_OK;
}

static int log2_of(int v)
{
    int s = 0;
    while ((1 << s) < v) s++;
    return s;
}

}  // namespace qmag

using namespace qmag;

extern "C" int qmag_kv_release_dev(const qmag_kv_table *t, const int *len, const int *ended, const int *n_free,
                                   int *len_next, int *n_free_next, int *status)
{
    int st = check_table(t);
    if (st) return st;
    if (!len || !ended || !n_free || !len_next || !n_free_next || !status)
        return fail(QMAG_ERR_ARG, "kv_release: null pointer");
    const int64_t n = t->n_seq;
    const Range r[] = {{len_next, n}, {n_free_next, 1}, {status, 1}, {len, n}, {ended, n}, {n_free, 1}};
    if ((st = check_ranges("kv_release", r, 3, 6))) return st;
    if ((st = check_lists("kv_release", t, false, r, 3, 6))) return st;
    if ((st = require_ready())) return st;
    DeviceScope dev;
    if (dev.st) return dev.st;
    PgArgs A = {t->n_seq, t->max_blocks, log2_of(t->block_size), t->n_block, 0, t->table, t->free_list, len, ended, n_free,
                nullptr, nullptr, nullptr, len_next, n_free_next, status};
    const int64_t most = (int64_t)t->n_seq * t->max_blocks;
    const int64_t wgs = (most + 16 * PG_WG - 1) / (16 * PG_WG);
    hipStream_t s = ctx().stream;
    prof_begin(PROF_KV, s);
    kv_release_kernel<<<dim3((unsigned)(wgs < 1 ? 1 : wgs > 256 ? 256 : wgs)), PG_WG, 0, s>>>(A);
    prof_end(PROF_KV, s);
    QMAG_HIP(hipGetLastError());
    return QMAG_OK;
}

extern "C" int qmag_kv_assign_dev(const qmag_kv_table *t, const int *len, const int *n_new, const int *n_free, int T,
                                  int *slot, int *pos, int *cu, int *len_next, int *n_free_next, int *status)
{
    int st = check_table(t);
    if (st) return st;
    if (T < 0 || !len || !n_new || !n_free || !cu || !len_next || !n_free_next || !status || (T > 0 && (!slot || !pos)))
        return fail(QMAG_ERR_ARG, "kv_assign: T=%d or a null pointer", T);
    const int64_t n = t->n_seq;
    const Range r[] = {{len_next, n}, {n_free_next, 1}, {status, 1}, {cu, n + 1}, {slot, T},
                       {pos, T},      {len, n},         {n_new, n},  {n_free, 1}};
    if ((st = check_ranges("kv_assign", r, 6, 9))) return st;
    if ((st = check_lists("kv_assign", t, true, r, 6, 9))) return st;
    if ((st = require_ready())) return st;
    DeviceScope dev;
    if (dev.st) return dev.st;
    PgArgs A = {t->n_seq, t->max_blocks, log2_of(t->block_size), t->n_block, T, t->table, t->free_list, len, n_new, n_free,
                slot, pos, cu, len_next, n_free_next, status};
    const int64_t wgs = ((int64_t)T + PG_WG * PG_TOK - 1) / (PG_WG * PG_TOK);
    hipStream_t s = ctx().stream;
    prof_begin(PROF_KV, s);
    kv_assign_kernel<<<dim3((unsigned)(wgs < 1 ? 1 : wgs > 1024 ? 1024 : wgs)), PG_WG, 0, s>>>(A);
    prof_end(PROF_KV, s);
    QMAG_HIP(hipGetLastError());
    return QMAG_OK;
}

/*
 * pages.c -- the paged KV cache and its attention (kv_pages.h): handles, argument checks and the
 * workspace of the launches (pages.cu, pages_attn.cu, pages_attn_tc.cu).
 *
 * The reference's cache is one block per request (kernel/kv_cache.c:15-34) and is copied whole where
 * two requests share a document; here requests name the same pages.  All of it is queued work on
 * device memory: nothing here reads the device back.
 */
#include <cuda_runtime_api.h>
#include <pthread.h>
#include <stdlib.h>
#include <string.h>

#include "attn_ext.h"
#include "host_internal.h"
#include "kv_pages.h"
#include "pages_shim.h"

#define TYB_PAGES_MAGIC 0x54594250u /* "TYBP" */

enum { WS_SCRATCH, WS_TICKETS, WS_KINDS }; /* tickets: tyb_pages_ticket_bytes, the same for every call of a pool */

typedef struct tyb_pages_s {
    KVPages pub; /* first: the KVPages* handed out converts back */
    uint32_t magic;
    int owned;
    tyb_pages_env env;
    pthread_mutex_t lock; /* held from a call's workspace to its last launch */
    struct {
        void *p;
        size_t bytes;
        int captured; /* a captured call was given it */
    } ws[WS_KINDS];
    struct tyb_pages_s *next; /* in g_pools */
    _Alignas(64) unsigned char maps[TYB_PAGES_MAPS_BYTES];
} tyb_pages;

/* ---- workspace ----------------------------------------------------------------------------
 * A pool has its own, since a pool is driven from one stream at a time: work queued by its calls, and
 * the graphs captured from them, use it in turn, and calls on other pools never touch it.  Its lock is held
 * until a call's last launch, so that host threads that share the stream queue whole calls, and none loses
 * to another's growth the buffer that it was just given.  It grows on
 * demand (after waiting for the device), but not while the stream is captured, where an allocation
 * would spoil the capture.  A buffer that a captured call was given is never freed or handed on: a graph
 * may name it for as long as the process lives.  (Each is at least half as large again as the one it
 * replaced, so those kept are at most twice the largest.) */

static int capturing(void)
{
    enum cudaStreamCaptureStatus state = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing((cudaStream_t)tyb_stream(), &state) != cudaSuccess) {
        cudaGetLastError(); /* the default stream beside another's capture: the launch will say so */
        return 0;
    }
    return state != cudaStreamCaptureStatusNone;
}

/* Buffers that no pool has any more, for the next one that needs such (an allocation and its return cost
 * a new pool's first call about a millisecond).  No work uses them. */
#define TYB_PAGES_SPARES 16
#define TYB_PAGES_SPARE_BYTES ((size_t)256 << 20) /* in all */
static pthread_mutex_t g_spare_lock = PTHREAD_MUTEX_INITIALIZER;
static struct {
    int device, kind;
    void *p;
    size_t bytes;
} g_spare[TYB_PAGES_SPARES];
static int g_spares;
static size_t g_spare_bytes;

static void give_back(tyb_pages *t, int kind)
{
    void *p = t->ws[kind].p;
    if (p && !t->ws[kind].captured) {
        cudaDeviceSynchronize(); /* it may still be in use */
        pthread_mutex_lock(&g_spare_lock);
        if (g_spares < TYB_PAGES_SPARES && g_spare_bytes + t->ws[kind].bytes <= TYB_PAGES_SPARE_BYTES) {
            g_spare[g_spares].device = t->env.device;
            g_spare[g_spares].kind = kind;
            g_spare[g_spares].p = p;
            g_spare[g_spares++].bytes = t->ws[kind].bytes;
            g_spare_bytes += t->ws[kind].bytes;
            p = NULL;
        }
        pthread_mutex_unlock(&g_spare_lock);
        cudaFree(p);
    }
    memset(&t->ws[kind], 0, sizeof t->ws[kind]);
}

/* The smallest spare buffer of `bytes` to eight times as many for the pool; 0: there is none. */
static int take_spare(tyb_pages *t, int kind, size_t bytes)
{
    int at = -1;
    pthread_mutex_lock(&g_spare_lock);
    for (int i = 0; i < g_spares; i++)
        if (g_spare[i].device == t->env.device && g_spare[i].kind == kind && g_spare[i].bytes >= bytes && g_spare[i].bytes / 8 <= bytes &&
            (at < 0 || g_spare[i].bytes < g_spare[at].bytes))
            at = i;
    if (at >= 0) {
        t->ws[kind].p = g_spare[at].p;
        t->ws[kind].bytes = g_spare[at].bytes;
        g_spare_bytes -= g_spare[at].bytes;
        g_spare[at] = g_spare[--g_spares];
    }
    pthread_mutex_unlock(&g_spare_lock);
    return at >= 0;
}

/* Frees the current device's spare buffers; 0: there were none. */
static int free_spares(int device)
{
    int freed = 0;
    pthread_mutex_lock(&g_spare_lock);
    for (int i = g_spares - 1; i >= 0; i--)
        if (g_spare[i].device == device) {
            cudaFree(g_spare[i].p);
            g_spare_bytes -= g_spare[i].bytes;
            g_spare[i] = g_spare[--g_spares];
            freed = 1;
        }
    pthread_mutex_unlock(&g_spare_lock);
    return freed;
}

/* A buffer of `bytes` for a pool that has none of the kind.  (What is spare may be what an allocation lacks.) */
static int fetch(tyb_pages *t, int kind, size_t bytes, const char *what)
{
    if (take_spare(t, kind, bytes)) return 1;
    if (!tyb_dev_alloc(&t->ws[kind].p, bytes, what) && !(free_spares(t->env.device) && tyb_dev_alloc(&t->ws[kind].p, bytes, what))) return 0;
    t->ws[kind].bytes = bytes;
    return 1;
}

/* The pool's buffer of a kind, its lock being held; tickets are zero to begin with.  NULL on failure (error
 * set). */
static void *workspace(tyb_pages *t, int kind, size_t bytes, const char *what)
{
    void *p = NULL;
    const int in_graph = capturing();
    if (t->ws[kind].bytes < bytes) {
        if (in_graph) {
            tyb_set_error("%s: the pool's workspace is too small for this call, and cannot grow while the stream is captured: "
                          "make a call of these sizes before", what);
        } else {
            size_t want = t->ws[kind].bytes ? t->ws[kind].bytes : 1 << 18;
            while (want < bytes) want += want / 2;
            give_back(t, kind);
            if (fetch(t, kind, want, what) && kind == WS_TICKETS &&
                !tyb_cuda_ok(cudaMemsetAsync(t->ws[kind].p, 0, t->ws[kind].bytes, (cudaStream_t)tyb_stream()), what))
                give_back(t, kind);
        }
    }
    if (t->ws[kind].bytes >= bytes) p = t->ws[kind].p;
    if (p && in_graph) t->ws[kind].captured = 1;
    return p;
}

/* The pools that there are, for tyb_pages_after_timeout. */
static pthread_mutex_t g_pools_lock = PTHREAD_MUTEX_INITIALIZER;
static tyb_pages *g_pools;

/* A kernel whose wait ran out leaves tickets half counted, and says so in their first word; until that is
 * zero again, kernels that would use them raise the same status instead.  Called when the status has been
 * reported: clears those tickets, and of the other pools nothing (they may be in use on other streams).  The
 * word goes last: a launch that is on its way meanwhile finds it set in some of its CTAs, which set it
 * again, or in none, and then the tickets are all zero. */
void tyb_pages_after_timeout(void)
{
    int dev = -1;
    if (cudaGetDevice(&dev) != cudaSuccess) return;
    pthread_mutex_lock(&g_pools_lock);
    for (tyb_pages *t = g_pools; t; t = t->next) {
        pthread_mutex_lock(&t->lock);
        char *tickets = (char *)t->ws[WS_TICKETS].p;
        unsigned int gave_up = 0;
        if (tickets && t->env.device == dev && cudaDeviceSynchronize() == cudaSuccess &&
            cudaMemcpy(&gave_up, tickets, sizeof gave_up, cudaMemcpyDeviceToHost) == cudaSuccess && gave_up) {
            const size_t head = TYB_PAGES_TICKET_HEAD;
            if (cudaMemset(tickets + head, 0, t->ws[WS_TICKETS].bytes - head) == cudaSuccess && cudaDeviceSynchronize() == cudaSuccess &&
                cudaMemset(tickets, 0, head) == cudaSuccess)
                cudaDeviceSynchronize();
        }
        pthread_mutex_unlock(&t->lock);
    }
    pthread_mutex_unlock(&g_pools_lock);
}

/* ---- handles ------------------------------------------------------------------------------- */

/* The pool behind a KVPages*, with its device current; NULL (error set) otherwise. */
static tyb_pages *pages_from(const KVPages *p, const char *what)
{
    tyb_pages *t = (tyb_pages *)p;
    if (!p) {
        tyb_set_error("%s: KVPages is NULL", what);
        return NULL;
    }
    if (t->magic != TYB_PAGES_MAGIC) {
        tyb_set_error("%s: KVPages was not made by kv_pages_alloc or kv_pages_attach", what);
        return NULL;
    }
    int dev = -1;
    if (!tyb_cuda_ok(cudaGetDevice(&dev), what)) return NULL;
    if (dev != t->env.device) {
        tyb_set_error("%s: the pool is on device %d, the current device is %d", what, t->env.device, dev);
        return NULL;
    }
    return t;
}

/* Memory of `device` (TYB_CURRENT: the current one), `align` bytes aligned; 1 when so.  (Another device's would be a fault, or a way over the
 * link for every access.) */
#define TYB_CURRENT (-1)
static int on_device(const void *p, size_t align, int device, const char *name, const char *what)
{
    if (!p) {
        tyb_set_error("%s: NULL %s", what, name);
        return 0;
    }
    if ((uintptr_t)p % align) {
        tyb_set_error("%s: %s %p is not %zu-byte aligned", what, name, p, align);
        return 0;
    }
    if (device == TYB_CURRENT && !tyb_cuda_ok(cudaGetDevice(&device), what)) return 0;
    struct cudaPointerAttributes at;
    const cudaError_t e = cudaPointerGetAttributes(&at, p);
    if (e != cudaSuccess) {
        cudaGetLastError(); /* not for later calls */
        tyb_set_error("%s: %s: %s", what, name, cudaGetErrorString(e));
        return 0;
    }
    if (at.type != cudaMemoryTypeDevice && at.type != cudaMemoryTypeManaged) {
        tyb_set_error("%s: %s is not device memory", what, name);
        return 0;
    }
    if (at.type == cudaMemoryTypeDevice && at.device != device) {
        tyb_set_error("%s: %s is on device %d, the pool on device %d", what, name, at.device, device);
        return 0;
    }
    return 1;
}

static int check_dims(const KVPages *p, const char *what)
{
    const char *bad = NULL;
    if (p->num_layers < 1) bad = "num_layers";
    else if (p->num_pages < 1 || p->num_pages > 1 << 20) bad = "num_pages";
    else if (p->page_size != 16 && p->page_size != 32 && p->page_size != 64 && p->page_size != 128) bad = "page_size";
    else if (p->kv_heads < 1 || p->kv_heads > 1024) bad = "kv_heads";
    else if (p->head_dim != 64 && p->head_dim != 128) bad = "head_dim";
    else if (p->max_seqs < 1 || p->max_seqs > TYB_PAGES_MAX_SEQS) bad = "max_seqs";
    else if (p->max_pages < 1 || p->max_pages > 1 << 20) bad = "max_pages";
    else if (p->kv_dtype != ATTN_KV_F32 && p->kv_dtype != ATTN_KV_BF16) bad = "kv_dtype";
    else if ((long long)p->num_layers * p->num_pages > (1LL << 31) / ((long long)p->kv_heads * p->page_size) - 1)
        bad = "num_layers * num_pages * kv_heads * page_size";
    if (bad) tyb_set_error("%s: %s is outside the supported range", what, bad);
    return !bad;
}

static size_t slab_bytes(const KVPages *p)
{
    return (size_t)p->num_layers * p->num_pages * p->kv_heads * p->page_size * p->head_dim *
           (p->kv_dtype == ATTN_KV_BF16 ? 2 : 4);
}

static void destroy(tyb_pages *t)
{
    pthread_mutex_lock(&g_pools_lock);
    for (tyb_pages **at = &g_pools; *at; at = &(*at)->next)
        if (*at == t) {
            *at = t->next;
            break;
        }
    pthread_mutex_unlock(&g_pools_lock);
    if (t->owned) {
        cudaFree(t->pub.k);
        cudaFree(t->pub.v);
        cudaFree(t->pub.table); /* table, len and ref are one allocation */
    }
    for (int k = 0; k < WS_KINDS; k++) give_back(t, k);
    pthread_mutex_destroy(&t->lock);
    t->magic = 0;
    free(t);
}

static tyb_pages *make(const KVPages *dims, int owned, const char *what)
{
    tyb_pages *t = (tyb_pages *)aligned_alloc(64, sizeof *t); /* the maps' alignment */
    if (!t) {
        tyb_set_error("%s: out of host memory", what);
        return NULL;
    }
    memset(t, 0, sizeof *t);
    t->pub = *dims;
    t->magic = TYB_PAGES_MAGIC;
    t->owned = owned;
    pthread_mutex_init(&t->lock, NULL);
    if (!tyb_cuda_ok(cudaGetDevice(&t->env.device), what)) {
        destroy(t);
        return NULL;
    }
    if (tyb_status_mirror_setup() != 0) cudaGetLastError(); /* as in kv_cache_alloc_ex */
    t->env.status = tyb_status_word();
    t->env.mirror = tyb_status_mirror_device();
    if (!t->env.status) {
        tyb_set_error("%s: no status word on device %d", what, t->env.device);
        destroy(t);
        return NULL;
    }
    pthread_mutex_lock(&g_pools_lock);
    t->next = g_pools;
    g_pools = t;
    pthread_mutex_unlock(&g_pools_lock);
    return t;
}

KVPages *kv_pages_alloc(int num_layers, int num_pages, int page_size, int kv_heads, int head_dim, int max_seqs,
                        int max_pages, int kv_dtype)
{
    const char *what = "kv_pages_alloc";
    const KVPages d = {NULL, NULL, NULL, NULL, NULL, num_layers, num_pages, page_size, kv_heads, head_dim, max_seqs,
                       max_pages, kv_dtype};
    if (!check_dims(&d, what)) return NULL;
    tyb_pages *t = make(&d, 1, what);
    if (!t) return NULL;
    const size_t entries = (size_t)max_seqs * max_pages, ints = entries + max_seqs + num_pages;
    int ok = tyb_dev_alloc(&t->pub.k, slab_bytes(&d), what) && tyb_dev_alloc(&t->pub.v, slab_bytes(&d), what) &&
             tyb_dev_alloc((void **)&t->pub.table, ints * sizeof(int), what);
    if (ok) {
        t->pub.len = t->pub.table + entries;
        t->pub.ref = t->pub.len + max_seqs;
        ok = tyb_cuda_ok(cudaMemset(t->pub.table, 0xff, entries * sizeof(int)), what) &&
             tyb_cuda_ok(cudaMemset(t->pub.len, 0, (ints - entries) * sizeof(int)), what) &&
             tyb_cuda_ok(cudaDeviceSynchronize(), what) && /* the pool may be used on any stream next */
             tyb_cuda_ok(tyb_pages_maps(&t->pub, t->maps), what);
    }
    if (!ok) {
        destroy(t);
        return NULL;
    }
    return &t->pub;
}

KVPages *kv_pages_attach(void *k, void *v, int *table, int *len, int *ref, int num_layers, int num_pages, int page_size,
                         int kv_heads, int head_dim, int max_seqs, int max_pages, int kv_dtype)
{
    const char *what = "kv_pages_attach";
    const KVPages d = {k, v, table, len, ref, num_layers, num_pages, page_size, kv_heads, head_dim, max_seqs, max_pages,
                       kv_dtype};
    if (!check_dims(&d, what) || !on_device(k, 16, TYB_CURRENT, "k", what) || !on_device(v, 16, TYB_CURRENT, "v", what) ||
        !on_device(table, 4, TYB_CURRENT, "table", what) || !on_device(len, 4, TYB_CURRENT, "len", what) ||
        !on_device(ref, 4, TYB_CURRENT, "ref", what))
        return NULL;
    tyb_pages *t = make(&d, 0, what);
    if (t && !tyb_cuda_ok(tyb_pages_maps(&t->pub, t->maps), what)) {
        destroy(t);
        t = NULL;
    }
    return t ? &t->pub : NULL;
}

void kv_pages_release(KVPages *p)
{
    if (!p) return;
    tyb_pages *t = pages_from(p, "kv_pages_release");
    if (!t) return;
    cudaStreamSynchronize((cudaStream_t)tyb_stream());
    destroy(t);
}

/* ---- maintenance --------------------------------------------------------------------------- */

/* A list of n device ints; 1 when there is one to work on, 0 when the call is done (*rc says how). */
static int list_ready(const tyb_pages *t, const int *list, int n, const char *name, int *rc, const char *what)
{
    *rc = 1;
    if (n < 0) {
        tyb_set_error("%s: negative count %d", what, n);
        return 0;
    }
    if (n == 0) {
        *rc = 0;
        return 0;
    }
    return on_device(list, 4, t->env.device, name, what);
}

/* Ends a call that holds the pool's lock. */
static int launched(tyb_pages *t, int err, const char *what)
{
    pthread_mutex_unlock(&t->lock);
    return tyb_cuda_ok(err, what) ? 0 : 1;
}

/* The same for a call that was not given its workspace (error set). */
static int not_launched(tyb_pages *t)
{
    pthread_mutex_unlock(&t->lock);
    return 1;
}

int kv_pages_extend(KVPages *p, const int *seqs, const int *counts, int n)
{
    const char *what = "kv_pages_extend";
    int rc;
    tyb_pages *t = pages_from(p, what);
    if (!t) return 1;
    if (!list_ready(t, seqs, n, "seqs", &rc, what)) return rc;
    if (!on_device(counts, 4, t->env.device, "counts", what)) return 1;
    pthread_mutex_lock(&t->lock);
    void *ws = workspace(t, WS_SCRATCH, tyb_pages_plan_bytes(p, n), what);
    return ws ? launched(t, tyb_pages_extend_launch(p, &t->env, seqs, counts, n, ws, tyb_stream()), what) : not_launched(t);
}

static int fork_or_copy(KVPages *p, const int *src, const int *dst, int n, int deep, const char *what)
{
    int rc;
    tyb_pages *t = pages_from(p, what);
    if (!t) return 1;
    if (!list_ready(t, src, n, "src", &rc, what)) return rc;
    if (!on_device(dst, 4, t->env.device, "dst", what)) return 1;
    pthread_mutex_lock(&t->lock);
    void *ws = workspace(t, WS_SCRATCH, tyb_pages_plan_bytes(p, n), what);
    return ws ? launched(t, tyb_pages_fork_launch(p, &t->env, src, dst, n, deep, ws, tyb_stream()), what) : not_launched(t);
}

int kv_pages_fork(KVPages *p, const int *src, const int *dst, int n) { return fork_or_copy(p, src, dst, n, 0, "kv_pages_fork"); }

int kv_pages_copy(KVPages *p, const int *src, const int *dst, int n) { return fork_or_copy(p, src, dst, n, 1, "kv_pages_copy"); }

int kv_pages_free(KVPages *p, const int *seqs, int n)
{
    const char *what = "kv_pages_free";
    int rc;
    tyb_pages *t = pages_from(p, what);
    if (!t) return 1;
    if (!list_ready(t, seqs, n, "seqs", &rc, what)) return rc;
    pthread_mutex_lock(&t->lock);
    const size_t bytes = tyb_pages_release_bytes(n);
    void *ws = bytes ? workspace(t, WS_SCRATCH, bytes, what) : NULL;
    if (bytes && !ws) return not_launched(t);
    return launched(t, tyb_pages_free_launch(p, &t->env, seqs, n, ws, tyb_stream()), what);
}

int kv_pages_trim(KVPages *p, const int *seqs, int n, int window, int sinks)
{
    const char *what = "kv_pages_trim";
    int rc;
    tyb_pages *t = pages_from(p, what);
    if (!t) return 1;
    if (window < 1 || sinks < 0) {
        tyb_set_error("%s: window %d must be at least 1 and sinks %d not negative", what, window, sinks);
        return 1;
    }
    if (!list_ready(t, seqs, n, "seqs", &rc, what)) return rc;
    /* more than a sequence can have keeps it all; the kernel rounds it up to pages in 32 bits */
    if (sinks > p->max_pages * p->page_size) sinks = p->max_pages * p->page_size;
    pthread_mutex_lock(&t->lock);
    const size_t bytes = tyb_pages_release_bytes(n);
    void *ws = bytes ? workspace(t, WS_SCRATCH, bytes, what) : NULL;
    if (bytes && !ws) return not_launched(t);
    return launched(t, tyb_pages_trim_launch(p, &t->env, seqs, n, window, sinks, ws, tyb_stream()), what);
}

int kv_pages_compact(KVPages *p, int *live_out)
{
    const char *what = "kv_pages_compact";
    tyb_pages *t = pages_from(p, what);
    if (!t || (live_out && !on_device(live_out, 4, t->env.device, "live_out", what))) return 1;
    pthread_mutex_lock(&t->lock);
    void *ws = workspace(t, WS_SCRATCH, tyb_pages_plan_bytes(p, 0), what);
    return ws ? launched(t, tyb_pages_compact_launch(p, live_out, ws, tyb_stream()), what) : not_launched(t);
}

static int check_layer(const KVPages *p, int layer, const char *what)
{
    if (layer >= 0 && layer < p->num_layers) return 1;
    tyb_set_error("%s: layer %d out of range [0, %d)", what, layer, p->num_layers);
    return 0;
}

/* Rows of `width` elements, `stride` apart, in dtype: 16-byte accesses have to fit. */
static int check_rows(const tyb_pages *t, const void *x, int dtype, long long stride, long long width, const char *name, const char *what)
{
    if (dtype != ATTN_DT_F32 && dtype != ATTN_DT_BF16) {
        tyb_set_error("%s: unknown element type %d", what, dtype);
        return 0;
    }
    if (stride < width || stride % (dtype == ATTN_DT_BF16 ? 8 : 4)) {
        tyb_set_error("%s: %s rows are %lld elements apart: at least %lld, and a multiple of 16 bytes, are wanted", what, name,
                      stride, width);
        return 0;
    }
    return on_device(x, 16, t->env.device, name, what);
}

int kv_pages_write(KVPages *p, int layer, const int *seqs, const int *starts, int n, int rows, const void *k_new,
                   const void *v_new, int in_dtype, long long stride)
{
    const char *what = "kv_pages_write";
    int rc;
    tyb_pages *t = pages_from(p, what);
    if (!t || !check_layer(p, layer, what)) return 1;
    if (rows < 0 || rows > 1 << 28) {
        tyb_set_error("%s: rows %d out of range", what, rows);
        return 1;
    }
    if (!list_ready(t, seqs, n, "seqs", &rc, what)) return rc;
    if (rows == 0) return 0;
    const long long width = (long long)p->kv_heads * p->head_dim;
    if (!on_device(starts, 4, t->env.device, "starts", what) || !check_rows(t, k_new, in_dtype, stride, width, "k_new", what) ||
        !check_rows(t, v_new, in_dtype, stride, width, "v_new", what))
        return 1;
    pthread_mutex_lock(&t->lock);
    return launched(t, tyb_pages_write_launch(p, &t->env, layer, seqs, starts, n, rows, k_new, v_new, in_dtype == ATTN_DT_BF16, stride,
                                           tyb_stream()),
                    what);
}

int kv_pages_import(KVPages *p, int seq, const KVCache *cache)
{
    const char *what = "kv_pages_import";
    tyb_pages *t = pages_from(p, what);
    if (!t) return 1;
    tyb_cache *c = tyb_cache_from(cache);
    if (!c) return 1;
    if (p->num_layers != KV_NUM_LAYERS || p->kv_heads != KV_NUM_KV_HEADS || p->head_dim != KV_HEAD_DIM ||
        p->kv_dtype != kv_cache_dtype(cache) || c->device != t->env.device) {
        tyb_set_error("%s: the pool's layers, heads, element type and device have to be the cache's", what);
        return 1;
    }
    if (seq < 0 || seq >= p->max_seqs) {
        tyb_set_error("%s: sequence %d out of range [0, %d)", what, seq, p->max_seqs);
        return 1;
    }
    const int rows = cache->seq_len;
    if (rows < 0 || rows > cache->max_seq_len) {
        tyb_set_error("%s: seq_len %d out of range [0, %d]", what, rows, cache->max_seq_len);
        return 1;
    }
    for (int l = 0; l < KV_NUM_LAYERS; l++)
        if (!tyb_flush_pending(c, l, what)) return 1;
    if (rows == 0) return 0;
    pthread_mutex_lock(&t->lock);
    void *ws = workspace(t, WS_SCRATCH, tyb_pages_plan_bytes(p, 1), what);
    if (!ws) return not_launched(t);
    return launched(t, tyb_pages_import_launch(p, &t->env, seq, c->k_slab, c->v_slab, cache->max_seq_len, rows, ws, tyb_stream()), what);
}

/* ---- attention ------------------------------------------------------------------------------ */

static int attend(const KVPages *p, tyb_pages_attn *a, const char *what)
{
    tyb_pages *t = pages_from(p, what);
    if (!t || !check_layer(p, a->layer, what)) return 1;
    if (a->q_heads < 1 || a->q_heads % p->kv_heads || a->q_heads / p->kv_heads > TYB_PAGES_MAX_GROUP) {
        tyb_set_error("%s: q_heads %d is not 1 .. %d times the %d KV heads", what, a->q_heads, TYB_PAGES_MAX_GROUP, p->kv_heads);
        return 1;
    }
    if (a->batch < 0 || a->batch > 65535 || a->rows < 0 || a->rows > (1 << 30) / a->q_heads) {
        tyb_set_error("%s: batch %d or rows %d out of range", what, a->batch, a->rows);
        return 1;
    }
    if (a->max_new < 0 || a->max_len < 0 || a->window < 0 || a->sinks < 0) {
        tyb_set_error("%s: negative max_new, max_len, window or sinks", what);
        return 1;
    }
    if (!(a->scale > 0.f) || a->scale > 3.0e38f) {
        tyb_set_error("%s: scale %g is not a positive number", what, (double)a->scale);
        return 1;
    }
    if (a->batch == 0 || a->rows == 0) return 0;
    if (!check_rows(t, a->q, a->io_bf16 ? ATTN_DT_BF16 : ATTN_DT_F32, a->q_stride, (long long)a->q_heads * p->head_dim, "q", what) ||
        !on_device(a->out, 16, t->env.device, "output", what) || !on_device(a->seqs, 4, t->env.device, "seqs", what))
        return 1;
    const int tokens = a->max_new == 1 && a->rows == a->batch; /* one each: no starts */
    if (!tokens && !on_device(a->starts, 4, t->env.device, "starts", what)) return 1;
    /* The shared pass takes whole pages: each sequence has its own copy of a partly filled one. */
    a->prefix -= a->prefix % p->page_size;
    a->p = *p;
    a->maps = t->maps;
    a->env = t->env;
    int uses_tickets;
    const size_t bytes = tyb_pages_attn_bytes(a, &uses_tickets);
    pthread_mutex_lock(&t->lock);
    void *ws = bytes ? workspace(t, WS_SCRATCH, bytes, what) : NULL;
    void *tickets = uses_tickets ? workspace(t, WS_TICKETS, tyb_pages_ticket_bytes(p), what) : NULL;
    if ((bytes && !ws) || (uses_tickets && !tickets)) return not_launched(t);
    return launched(t, tyb_pages_attn_launch(a, ws, tickets, tyb_stream()), what);
}

static int io_type(int io_dtype, const char *what)
{
    if (io_dtype == ATTN_DT_F32 || io_dtype == ATTN_DT_BF16) return 1;
    tyb_set_error("%s: unknown element type %d", what, io_dtype);
    return 0;
}

int attention_pages_prefix_gqa(const void *q, long long q_stride, const KVPages *p, int layer, const int *seqs, int batch,
                               int q_heads, int prefix_len, int max_len, void *output, int io_dtype, float scale)
{
    const char *what = "attention_pages_prefix_gqa";
    if (!io_type(io_dtype, what)) return 1;
    if (prefix_len < 0 || prefix_len > max_len) {
        tyb_set_error("%s: prefix_len %d out of range [0, max_len = %d]", what, prefix_len, max_len);
        return 1;
    }
    tyb_pages_attn a = {.layer = layer, .q = q, .q_stride = q_stride, .out = output, .io_bf16 = io_dtype == ATTN_DT_BF16,
                        .q_heads = q_heads, .seqs = seqs, .batch = batch, .rows = batch, .max_new = 1, .max_len = max_len,
                        .scale = scale};
    a.prefix = batch == 1 ? 0 : prefix_len; /* one alone has nothing to share */
    return attend(p, &a, what);
}

int attention_pages_window_gqa(const void *q, long long q_stride, const KVPages *p, int layer, const int *seqs,
                               const int *starts, int batch, int rows, int q_heads, int max_new, int max_len, int window,
                               int sinks, void *output, int io_dtype, float scale)
{
    const char *what = "attention_pages_window_gqa";
    if (!io_type(io_dtype, what)) return 1;
    tyb_pages_attn a = {.layer = layer, .q = q, .q_stride = q_stride, .out = output, .io_bf16 = io_dtype == ATTN_DT_BF16,
                        .q_heads = q_heads, .seqs = seqs, .starts = starts, .batch = batch, .rows = rows,
                        .max_new = max_new, .max_len = max_len, .window = window, .sinks = sinks, .scale = scale};
    return attend(p, &a, what);
}

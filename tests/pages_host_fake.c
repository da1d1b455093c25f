/*
 * pages_host_fake.c -- what csrc/pages.c calls, for tests of its host side without a GPU: a CUDA runtime
 * that only keeps books (allocations, captures, what device a pointer is on) and launches that note what
 * they were given.  Compiled together with pages.c by test_pages_host_cpu.py.
 */
#include <cuda_runtime_api.h>
#include <stdarg.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>
#include <unistd.h>

#include "attn_ext.h"
#include "host_internal.h"
#include "kv_pages.h"
#include "pages_shim.h"

/* ---- set and read by the tests ---- */
int fake_device, fake_capturing;     /* the current device; whether the current stream is captured */
int fake_foreign_device = 1;         /* device of pointers in fake_foreign */
char fake_foreign[64];
int fake_syncs, fake_mallocs, fake_memsets, fake_launches;
void *fake_ws, *fake_tickets;        /* what the last launch was given */
int fake_window, fake_sinks;         /* of the last trim or attention launch */
int fake_launch_us;                  /* how long a launch takes */
int fake_overlaps, fake_lost;        /* launches while another one was on its way; that found their workspace freed */
static void *g_stream;
static char g_err[512];

#define FAKE_MAX 4096
static void *g_live[FAKE_MAX];
static int g_nlive;
int fake_is_live(const void *p)
{
    for (int i = 0; i < g_nlive; i++)
        if (g_live[i] == p) return 1;
    return 0;
}
int fake_live(void) { return g_nlive; }
const char *fake_error(void) { return g_err; }
void fake_stream(void *s) { g_stream = s; }

/* ---- the CUDA runtime ---- */
cudaError_t cudaGetDevice(int *d)
{
    *d = fake_device;
    return cudaSuccess;
}
cudaError_t cudaGetLastError(void) { return cudaSuccess; }
const char *cudaGetErrorString(cudaError_t e) { return e == cudaSuccess ? "no error" : "an error"; }
cudaError_t cudaMalloc(void **p, size_t n)
{
    if (fake_capturing || g_nlive == FAKE_MAX) return cudaErrorStreamCaptureUnsupported;
    fake_mallocs++;
    *p = g_live[g_nlive++] = calloc(1, n < 65536 ? n : 65536);
    return cudaSuccess;
}
cudaError_t cudaFree(void *p)
{
    for (int i = 0; i < g_nlive; i++)
        if (g_live[i] == p) {
            free(p);
            g_live[i] = g_live[--g_nlive];
            break;
        }
    return cudaSuccess;
}
cudaError_t cudaMemset(void *p, int v, size_t n)
{
    fake_memsets++;
    memset(p, v, n < 4096 ? n : 4096);
    return cudaSuccess;
}
cudaError_t cudaMemsetAsync(void *p, int v, size_t n, cudaStream_t s) { return fake_memsets++, cudaSuccess; }
cudaError_t cudaMemcpy(void *d, const void *s, size_t n, enum cudaMemcpyKind k) { return memcpy(d, s, n), cudaSuccess; }
cudaError_t cudaDeviceSynchronize(void) { return fake_syncs++, cudaSuccess; }
cudaError_t cudaStreamSynchronize(cudaStream_t s) { return fake_syncs++, cudaSuccess; }
cudaError_t cudaStreamIsCapturing(cudaStream_t s, enum cudaStreamCaptureStatus *state)
{
    *state = fake_capturing ? cudaStreamCaptureStatusActive : cudaStreamCaptureStatusNone;
    return cudaSuccess;
}
cudaError_t cudaPointerGetAttributes(struct cudaPointerAttributes *a, const void *p)
{
    memset(a, 0, sizeof *a);
    a->type = cudaMemoryTypeDevice;
    a->device = (const char *)p >= fake_foreign && (const char *)p < fake_foreign + sizeof fake_foreign ? fake_foreign_device : fake_device;
    return cudaSuccess;
}

/* ---- the library's other files ---- */
void tyb_set_error(const char *fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof g_err, fmt, ap);
    va_end(ap);
}
int tyb_cuda_ok(int err, const char *what)
{
    if (err) tyb_set_error("%s: %s", what, cudaGetErrorString((cudaError_t)err));
    return err == 0;
}
void *tyb_stream(void) { return g_stream; }
int tyb_is_device_ptr(const void *p)
{
    struct cudaPointerAttributes a;
    cudaPointerGetAttributes(&a, p);
    return a.type == cudaMemoryTypeDevice;
}
int tyb_dev_alloc(void **p, size_t bytes, const char *what)
{
    *p = NULL;
    return tyb_cuda_ok(cudaMalloc(p, bytes), what);
}
static unsigned int g_word;
int tyb_status_mirror_setup(void) { return 0; }
unsigned int *tyb_status_word(void) { return &g_word; }
unsigned int *tyb_status_mirror_device(void) { return &g_word; }
tyb_cache *tyb_cache_from(const KVCache *c) { return NULL; }
int kv_cache_dtype(const KVCache *c) { return 0; }
int tyb_flush_pending(tyb_cache *t, int layer, const char *what) { return 1; }

/* ---- the launches ---- */
int tyb_pages_maps(const KVPages *p, void *maps) { return 0; }
size_t tyb_pages_plan_bytes(const KVPages *p, int n) { return 64 + 4u * (size_t)n + 16u * (size_t)p->num_pages; }
static int launch(void *ws, void *tickets)
{
    static int inside;
    if (__atomic_add_fetch(&inside, 1, __ATOMIC_SEQ_CST) > 1) __atomic_add_fetch(&fake_overlaps, 1, __ATOMIC_SEQ_CST);
    if (fake_launch_us) usleep(fake_launch_us);
    if ((ws && !fake_is_live(ws)) || (tickets && !fake_is_live(tickets))) __atomic_add_fetch(&fake_lost, 1, __ATOMIC_SEQ_CST);
    __atomic_sub_fetch(&inside, 1, __ATOMIC_SEQ_CST);
    fake_ws = ws;
    fake_tickets = tickets;
    fake_launches++;
    return 0;
}
int tyb_pages_extend_launch(const KVPages *p, const tyb_pages_env *env, const int *seqs, const int *counts, int n, void *ws, void *stream) { return launch(ws, 0); }
int tyb_pages_fork_launch(const KVPages *p, const tyb_pages_env *env, const int *src, const int *dst, int n, int deep, void *ws, void *stream) { return launch(ws, 0); }
size_t tyb_pages_release_bytes(int n) { return n > 256 ? 1024 : 0; }
int tyb_pages_free_launch(const KVPages *p, const tyb_pages_env *env, const int *seqs, int n, void *ws, void *stream) { return launch(ws, 0); }
int tyb_pages_trim_launch(const KVPages *p, const tyb_pages_env *env, const int *seqs, int n, int window, int sinks, void *ws, void *stream)
{
    fake_window = window;
    fake_sinks = sinks;
    return launch(0, 0);
}
int tyb_pages_compact_launch(const KVPages *p, int *live_out, void *ws, void *stream) { return launch(ws, 0); }
int tyb_pages_write_launch(const KVPages *p, const tyb_pages_env *env, int layer, const int *seqs, const int *starts, int n, int rows,
                           const void *k_new, const void *v_new, int in_bf16, long long stride, void *stream) { return launch(0, 0); }
int tyb_pages_import_launch(const KVPages *p, const tyb_pages_env *env, int seq, const void *k_slab, const void *v_slab, int row_capacity,
                            int rows, void *ws, void *stream) { return launch(ws, 0); }
/* as much scratch as there are rows */
size_t tyb_pages_ticket_bytes(const KVPages *p) { return 4096; }
size_t tyb_pages_attn_bytes(const tyb_pages_attn *a, int *uses_tickets)
{
    *uses_tickets = 1;
    return 65536u * (size_t)a->rows;
}
int tyb_pages_attn_launch(const tyb_pages_attn *a, void *ws, void *tickets, void *stream)
{
    fake_window = a->window;
    fake_sinks = a->sinks;
    return launch(ws, tickets);
}

/*
 * pages_shim.h -- the thin C interface between pages.c and its sm_100a kernels (pages.cu,
 * pages_attn.cu, pages_attn_tc.cu).  Launchers take DEVICE pointers, enqueue on `stream` and
 * return a cudaError_t value (0 = success), as in attn_shim.h.
 */
#ifndef TYB_PAGES_SHIM_H
#define TYB_PAGES_SHIM_H

#include <stddef.h>
#include <stdint.h>

#include "attn_shim.h"
#include "kv_pages.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Largest max_seqs: the duplicate check keeps a bit per sequence in shared memory. */
#define TYB_PAGES_MAX_SEQS (1 << 20)
/* Largest q_heads / kv_heads: the query rows of one tensor-core row tile. */
#define TYB_PAGES_MAX_GROUP 16

/* What a handle looks up once for its launches: its device, and there the status word and its mirror. */
typedef struct {
    int device;
    unsigned int *status, *mirror;
} tyb_pages_env;

/* ---- maintenance (pages.cu); ws: tyb_pages_plan_bytes bytes of workspace ----------------- */
size_t tyb_pages_plan_bytes(const KVPages *p, int n);
int tyb_pages_extend_launch(const KVPages *p, const tyb_pages_env *env, const int *seqs, const int *counts, int n, void *ws, void *stream);
int tyb_pages_fork_launch(const KVPages *p, const tyb_pages_env *env, const int *src, const int *dst, int n, int deep, void *ws, void *stream);
size_t tyb_pages_release_bytes(int n); /* workspace of the next two */
int tyb_pages_free_launch(const KVPages *p, const tyb_pages_env *env, const int *seqs, int n, void *ws, void *stream);
int tyb_pages_trim_launch(const KVPages *p, const tyb_pages_env *env, const int *seqs, int n, int window, int sinks, void *ws, void *stream);
int tyb_pages_compact_launch(const KVPages *p, int *live_out, void *ws, void *stream);
int tyb_pages_write_launch(const KVPages *p, const tyb_pages_env *env, int layer, const int *seqs, const int *starts, int n, int rows,
                           const void *k_new, const void *v_new, int in_bf16, long long stride, void *stream);
/* Sequence `seq` (a host number) takes `rows` tokens: kv_pages_extend's plan for one sequence, then
 * the rows of a static cache (k_slab, v_slab: [28][8][row_capacity][128] of the pool's type). */
int tyb_pages_import_launch(const KVPages *p, const tyb_pages_env *env, int seq, const void *k_slab, const void *v_slab, int row_capacity,
                            int rows, void *ws, void *stream);

/* ---- attention ---------------------------------------------------------------------------- */
/* TMA tensor maps of a pool's K and V (64-byte aligned room), built once per handle. */
#define TYB_PAGES_MAPS_BYTES (6 * 128)
int tyb_pages_maps(const KVPages *p, void *maps);

typedef struct {
    KVPages p;
    tyb_pages_env env;
    const void *maps;
    int layer;
    const void *q;
    long long q_stride;
    void *out;
    int io_bf16;
    int q_heads;
    const int *seqs;
    const int *starts; /* NULL: one query per sequence */
    int batch;
    int rows;
    int max_new;
    int max_len;
    int prefix; /* leading rows computed once for all (whole pages); 0: none */
    int window; /* 0: unlimited */
    int sinks;
    float scale;
} tyb_pages_attn;

/* Bytes of workspace of a call, and whether it uses the pool's tickets. */
size_t tyb_pages_attn_bytes(const tyb_pages_attn *a, int *uses_tickets);
/* Tickets of a pool: a head, whose first word is set by a kernel that gave up (its tickets may then be half
 * counted: tyb_pages_after_timeout), then words that are zero between launches. */
#define TYB_PAGES_TICKET_HEAD 64
size_t tyb_pages_ticket_bytes(const KVPages *p);
int tyb_pages_attn_launch(const tyb_pages_attn *a, void *ws, void *tickets, void *stream);

#ifdef __cplusplus
}
#endif
#endif

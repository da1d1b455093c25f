// pages_attn.cuh -- what the attention kernels over the paged cache share: the visibility of a query
// row, the list of key tiles a set of rows can see, and the layout of the split records.
#pragma once

#include "common.cuh"
#include "pages_shim.h"

namespace tyb {

struct Status {
    unsigned int* word;
    unsigned int* mirror;
};

__device__ __forceinline__ void raise(const Status& s, unsigned int bits)
{
    atomicOr(s.word, bits);
    flag_mirror(s.mirror);
}

// The kernels of the paged cache are launched as programmatic dependents (launch_after): a kernel may start while
// its predecessor in the stream ends, sets itself up, and reads or writes nothing global before this wait.
// Only then it lets the next one start, as the library's other kernels do and rely on.
__device__ __forceinline__ void after_predecessor()
{
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

// The two halves apart, for a kernel that runs beside its predecessor (which has itself waited, before it let this
// one start, for all that came before).
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_predecessor() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// In clusters of `cluster` CTAs.
template <typename... P, typename... A>
int launch_after_in(int cluster, void (*kernel)(P...), dim3 grid, int threads, size_t shared, cudaStream_t stream, A... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = shared;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    return (int)cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}
template <typename... P, typename... A>
int launch_after(void (*kernel)(P...), dim3 grid, int threads, size_t shared, cudaStream_t stream, A... args)
{
    return launch_after_in(1, kernel, grid, threads, shared, stream, args...);
}

// Waits for phase `parity` of an mbarrier, at most limit_ns; false (and the status raised) when that ran
// out.
__device__ __forceinline__ bool wait_for(uint64_t* bar, uint32_t parity, uint64_t limit_ns, const Status& s)
{
    return mbar_wait_bounded_to(bar, parity, limit_ns, TYB_STATUS_WAIT_TIMEOUT, s.word, s.mirror);
}

// The same by all lanes of a warp, with one answer.
__device__ __forceinline__ bool warp_wait_for(uint64_t* bar, uint32_t parity, uint64_t limit_ns, const Status& s)
{
    return !__any_sync(0xffffffffu, !wait_for(bar, parity, limit_ns, s));
}

// The limit of the waits for a kernel's own copies and products in flight, at its end: a CTA whose other waits ran
// out (whatever the limit set for those) must not leave before them.
constexpr uint64_t kDrainNs = 500000000ull;
__device__ __forceinline__ uint64_t drain_ns(uint64_t limit_ns) { return limit_ns > kDrainNs ? limit_ns : kDrainNs; }

// One arrival for the warp, after all its lanes have come here.
__device__ __forceinline__ void warp_arrive(uint64_t* bar)
{
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// A query row at position `pos` sees key j when j <= pos and (j >= lo or j < sinks).  The four uses:
//   prefix      pos = P - 1,   lo = 0
//   own rows    pos = len - 1, lo = P
//   window      pos = its position, lo = max(0, pos - window + 1)
//   causal      the same with lo = 0
// A row that is not there has pos = -1: it sees nothing.

// The key tiles (of `kt` rows) that rows with positions up to pos_max and lower bounds from lo_min
// on can see: [0, na) for the sinks, then [b0, b0 + nb).
struct Tiles {
    int na, b0, nb;
    __device__ __forceinline__ int count() const { return na + nb; }
    __device__ __forceinline__ int at(int i) const { return i < na ? i : b0 + i - na; }
};

__device__ __forceinline__ Tiles tiles_of(int pos_max, int lo_min, int sinks, int kt)
{
    Tiles t;
    pos_max = max(pos_max, -1);
    const int end = (pos_max + kt) / kt;  // tiles up to pos_max
    t.na = (min(sinks, pos_max + 1) + kt - 1) / kt;
    t.b0 = max(lo_min / kt, t.na);
    t.nb = max(0, end - t.b0);
    return t;
}

// Split record s of output row R (= token * q_heads + head): the unnormalised output in FP32 at
// o[(s * rows + R) * D], the running maximum (base-2 exponent) and sum at ml[s * rows + R].
struct Records {
    float* o;
    float2* ml;
    int rows;
    int slots;
};

// Length of sequence s as the kernels may use it: within its table, 0 when s is no sequence.
__device__ __forceinline__ int checked_len(const KVPages& p, int s, const Status& st)
{
    if (s < 0 || s >= p.max_seqs) {
        raise(st, TYB_STATUS_BAD_ARGUMENT);
        return 0;
    }
    const int len = p.len[s];
    if (len < 0 || len > p.max_pages * p.page_size) {
        raise(st, TYB_STATUS_BAD_ARGUMENT);
        return 0;
    }
    return len;
}

struct AttnArgs {
    KVPages p;
    const void* q;
    long long q_stride;
    void* out;
    int io_bf16;
    int q_heads, group;
    const int* seqs;
    const int* starts;
    int batch, rows;
    int prefix;      // leading rows left to (or handled by) the shared pass
    int window, sinks;
    float scale_log2;
    int splits;   // a record slot each
    Records rec;  // slots == 1: the output is written directly
    Status st;
    int device;
};

// The tcgen05 form (pages_attn_tc.cu) for the query rows of a BF16 pool, `items` row tiles: tall, of at
// most 128 rows each, with two record slots a split; else of 256 rows.
constexpr int kTcTall = 128, kTcWide = 256;
int tc_launch(const AttnArgs& a, int layer, bool tall, bool shared_pass, bool beside, int items, const void* maps, cudaStream_t stream);

// The row form (pages_rows.cu) for the prompt chunks of an FP32 pool, row tiles of kRowsTile rows.
constexpr int kRowsTile = 64;
// CTAs on an SM: what the registers allow.  (40 chunks of 200 .. 900 tokens with heads of 64: 412 us, with two 455 us.)
__host__ __device__ constexpr int rows_ctas(int head_dim) { return head_dim == 64 ? 3 : 2; }
int rows_launch(const AttnArgs& a, int layer, int items, const void* maps, cudaStream_t stream);

// Item x of a list of row tiles: sequence b's queries starts[b] .. starts[b + 1] in tiles of `per` tokens.
// found: b (-1: no such item), its first query, its queries, and that query's place before the sequence's end
// (its position is the length plus this).  By one warp.
__device__ __forceinline__ void find_item(const AttnArgs& a, int x, int per, int* found)
{
    const int lane = threadIdx.x & 31;
    int before = 0;
    if (lane == 0) found[0] = -1;
    __syncwarp();
    for (int base = 0; base < a.batch && before <= x; base += 32) {
        const int b = base + lane;
        const int q0 = b < a.batch ? a.starts[b] : 0, q1 = b < a.batch ? a.starts[b + 1] : 0;
        const int cnt = q1 > q0 ? (q1 - q0 + per - 1) / per : 0;
        int sum = cnt;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += y;
        }
        const int lo = before + sum - cnt;
        if (x >= lo && x < lo + cnt) {
            if (q0 < 0 || q1 > a.rows) {
                raise(a.st, TYB_STATUS_BAD_ARGUMENT);
            } else {
                found[0] = b;
                found[1] = q0 + (x - lo) * per;
                found[2] = min(per, q1 - q0 - (x - lo) * per);
                found[3] = (x - lo) * per - (q1 - q0);
            }
        }
        before += __shfl_sync(0xffffffffu, sum, 31);
    }
}

// The streaming form (pages_stream.cu): the single tokens of sequences first .. first + count (at most
// kStreamSeqs) of the call, with the shared pass over a.prefix rows in the same launch (`shared`); the
// results are the output, or (out_slot >= 0) record slot out_slot of a.rec.  beside: 0, or the SMs that the
// shared pass launched just before keeps busy: the launch then runs on the others at the same time, and waits for the
// pass (which has waited for all before it) only at its end.  (A kernel that another host thread queues between the two
// changes nothing of that: it has itself waited for the pass before it lets this launch start, and this one ends after
// it.)  ws: stream_bytes; tickets: the pool's, its head
// first (zero between launches unless one gave up).
constexpr int kStreamSeqs = 1024;
// An item's start and end (its query, the join of the warps) cost a CTA about as much as this many stages:
// runs are cut by stages plus this for each item.  Measured with 256 sequences of 1 .. 512 rows (4.6 stages on
// average): 61 us against 84 us of runs with equal stages, whose run of one-stage items took twice the others.
constexpr int kItemUnits = 2;
size_t stream_bytes(const AttnArgs& a, int count, bool shared);
int launch_stream(const AttnArgs& a, int layer, int first, int count, bool shared, int out_slot, int beside, int max_len, const void* maps, void* ws,
                  unsigned int* tickets, cudaStream_t stream);

constexpr int kSms = 148;
// Rows of a TMA box of the pool's maps: a page, or the part of it that a stage holds.
__host__ __device__ inline int box_rows(const KVPages& p)
{
    const int most = p.kv_dtype == TYB_BF16 ? 64 : 32;
    return p.page_size < most ? p.page_size : most;
}

// log2 of the page size (16 .. 128)
__device__ __forceinline__ int page_shift(int page_size) { return __ffs(page_size) - 1; }

// A box of a page pool's map: columns from c0, rows from c1.
__device__ __forceinline__ void tma_load_2d(void* dst, const void* map, int c0, int c1, uint64_t* bar)
{
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(smem_u32(bar))
        : "memory");
}

// Rows from c1 of its column boxes from c2.
__device__ __forceinline__ void tma_load_3d(void* dst, const void* map, int c1, int c2, uint64_t* bar)
{
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(0), "r"(c1), "r"(c2), "r"(smem_u32(bar))
        : "memory");
}

__device__ __forceinline__ float fast_exp2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

}  // namespace tyb

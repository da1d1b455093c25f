// pages.cu -- maintenance of the paged KV cache (kv_pages.h): taking, sharing, copying, moving and
// freeing pages, and writing rows into them.
//
// The bookkeeping lives on the device (table, len, ref), so a call needs no read-back.  A call that
// takes pages runs as two kernels: a plan kernel of one CTA checks the whole request, ranks the new
// pages (prefix sums over the list, then over the free pages in rising order: the result depends on
// nothing but the state) and writes the page copies to do into the workspace; an apply kernel over
// the whole GPU writes tables and counts and moves the rows.  A request that fails a check leaves
// the plan's `ok` at 0 and the apply kernel does nothing.
//
// The row copies are bound by memory: each row is read once and written once, by 16-byte accesses,
// a (page, layer, tensor, head) block of consecutive rows per warp and turn.
#define TYB_WHOLE_PROGRAM
#include "pages_attn.cuh"

namespace tyb {

constexpr int kPlanThreads = 1024;
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kApplyThreads = 256;


// One copy of a plan: the first `rows` rows of page `from` (every layer, K and V) go to page `to`.
struct Move {
    int from, to, rows;
};

// The workspace: header, then first[n] (rank of list item i's first new page), fresh[num_pages] (the
// new pages in rank order; in a compaction, where page p goes), moves[num_pages].
struct PlanHead {
    int ok, moves, live, pad;
};
struct Plan {
    PlanHead* head;
    int* first;
    int* fresh;
    Move* moves;
};

__host__ __device__ inline size_t plan_bytes(int n, int num_pages)
{
    return sizeof(PlanHead) + ((size_t)n + num_pages) * sizeof(int) + (size_t)num_pages * sizeof(Move);
}

__host__ __device__ inline Plan plan_at(void* ws, int n, int num_pages)
{
    Plan p;
    p.head = static_cast<PlanHead*>(ws);
    p.first = reinterpret_cast<int*>(p.head + 1);
    p.fresh = p.first + n;
    p.moves = reinterpret_cast<Move*>(p.fresh + num_pages);
    return p;
}

// Exclusive prefix sum over the CTA's threads; *total receives the sum.  Every thread calls it.
__device__ __forceinline__ int block_scan(int x, int* total)
{
    __shared__ int part[kPlanWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int sum = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += y;
    }
    __syncthreads();  // part may still be read by the previous call
    if (lane == 31) part[warp] = sum;
    __syncthreads();
    if (warp == 0) {
        int w = lane < kPlanWarps ? part[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, w, o);
            if (lane >= o) w += y;
        }
        part[lane] = w;
    }
    __syncthreads();
    *total = part[kPlanWarps - 1];
    return sum - x + (warp ? part[warp - 1] : 0);
}

// Writes the numbers of the first `want` pages in [lo, hi) whose use (ref > 0) is `used` to out[0],
// out[stride] .. in rising order; returns how many there are (at most `want`).  Every thread of the CTA calls it.
__device__ int list_pages(const int* ref, int lo, int hi, bool used, int want, int* out,
                          int stride = 1)
{
    int found = 0;
    for (int base = lo; base < hi && found < want; base += kPlanThreads) {
        const int p = base + (int)threadIdx.x;
        const int hit = p < hi && (ref[p] > 0) == used;
        int total;
        const int at = found + block_scan(hit, &total);
        if (hit && at < want) out[at * stride] = p;
        found += total;
    }
    return found < want ? found : want;
}

// Marks sequence s in the bit set; false where it was there already.
__device__ __forceinline__ bool mark(unsigned int* bits, int s)
{
    const unsigned int b = 1u << (s & 31);
    return !(atomicOr(&bits[s >> 5], b) & b);
}

__device__ __forceinline__ void clear_marks(unsigned int* bits, int max_seqs)
{
    for (int i = threadIdx.x; i < (max_seqs + 31) / 32; i += kPlanThreads) bits[i] = 0u;
    __syncthreads();
}

// Ends a plan: records the outcome, raises what went wrong.
__device__ void plan_done(PlanHead* head, bool bad, bool short_of, int moves, const Status& st)
{
    if (threadIdx.x == 0) {
        head->ok = !bad && !short_of;
        head->moves = bad || short_of ? 0 : moves;
        if (bad) raise(st, TYB_STATUS_BAD_ARGUMENT);
        else if (short_of) raise(st, TYB_STATUS_OUT_OF_PAGES);
    }
}

// ---- extend ------------------------------------------------------------------------------------

// Plan and apply in one CTA (a step takes few pages).  seqs == NULL: the one sequence `seq0`, which
// has to be empty, grows by count0.
__global__ void __launch_bounds__(kPlanThreads)
    pages_extend_kernel(const KVPages p, const int* seqs, const int* counts, int n, int seq0, int count0, void* ws, Status st)
{
    extern __shared__ unsigned int marks[];
    const Plan plan = plan_at(ws, n, p.num_pages);
    const int cap = p.max_pages * p.page_size;
    after_predecessor();
    clear_marks(marks, p.max_seqs);
    int need = 0, s = 0, len = 0, mine = 0, at = 0;  // the thread's item of the last turn: the only one of most calls
    bool bad = false;
    for (int base = 0; base < n; base += kPlanThreads) {
        const int i = base + (int)threadIdx.x;
        mine = 0;
        if (i < n) {
            const int c = counts ? counts[i] : count0;
            s = seqs ? seqs[i] : seq0;
            if (s < 0 || s >= p.max_seqs || c < 0 || !mark(marks, s)) {
                bad = true;
            } else {
                len = p.len[s];
                if (len < 0 || len > cap || c > cap - len || (!seqs && len != 0)) bad = true;
                else mine = (len + c + p.page_size - 1) / p.page_size - (len + p.page_size - 1) / p.page_size;
                len += c;
            }
        }
        // no list of valid items needs more pages than the pool has: the sum stays far below 2^31
        if (mine > p.num_pages) mine = p.num_pages + 1;
        if (__syncthreads_or(bad)) break;
        int total;
        at = need + block_scan(mine, &total);
        if (i < n && n > kPlanThreads) plan.first[i] = at;
        need += total;
        if (need > p.num_pages) break;
    }
    bad = __syncthreads_or(bad);
    bool short_of = need > p.num_pages;
    if (!bad && !short_of) short_of = list_pages(p.ref, 0, p.num_pages, false, need, plan.fresh) < need;
    plan_done(plan.head, bad, short_of, 0, st);
    __syncthreads();
    if (bad || short_of) return;
    for (int base = 0; base < n; base += kPlanThreads) {
        const int i = base + (int)threadIdx.x;
        if (n > kPlanThreads && i < n) {  // not the thread's last item
            s = seqs[i];
            at = plan.first[i];
            const int c = counts[i], old = p.len[s];
            len = old + c;
            mine = (len + p.page_size - 1) / p.page_size - (old + p.page_size - 1) / p.page_size;
        }
        if (i >= n) mine = 0;
        const int e0 = (len + p.page_size - 1) / p.page_size - mine;
        // a few pages by the sequence's own thread, many by its warp
        const bool many = mine > 8;
        for (int k = 0; !many && k < mine; k++) {
            const int page = plan.fresh[at + k];
            p.table[(size_t)s * p.max_pages + e0 + k] = page;
            p.ref[page] = 1;
        }
        for (unsigned int left = __ballot_sync(0xffffffffu, many); left; left &= left - 1) {
            const int l = __ffs(left) - 1;
            const int s1 = __shfl_sync(0xffffffffu, s, l), at1 = __shfl_sync(0xffffffffu, at, l), e1 = __shfl_sync(0xffffffffu, e0, l),
                      n1 = __shfl_sync(0xffffffffu, mine, l);
            for (int k = threadIdx.x & 31; k < n1; k += 32) {
                const int page = plan.fresh[at1 + k];
                p.table[(size_t)s1 * p.max_pages + e1 + k] = page;
                p.ref[page] = 1;
            }
        }
        if (i < n) p.len[s] = len;
    }
}

// ---- fork and copy -----------------------------------------------------------------------------

// Entries of sequence s that become pages of the new sequence's own, from entry `e0` on: all of a
// copy (e0 = 0), a partly filled last one of a fork.
__device__ __forceinline__ int first_own_entry(const KVPages& p, int len, bool deep) { return deep ? 0 : len / p.page_size; }
__device__ __forceinline__ int entries_of(const KVPages& p, int len) { return (len + p.page_size - 1) / p.page_size; }

__global__ void __launch_bounds__(kPlanThreads)
    pages_fork_plan_kernel(const KVPages p, const int* src, const int* dst, int n, int deep, void* ws, Status st)
{
    extern __shared__ unsigned int marks[];
    const Plan plan = plan_at(ws, n, p.num_pages);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int cap = p.max_pages * p.page_size;
    after_predecessor();
    clear_marks(marks, p.max_seqs);
    bool bad = false;
    for (int i = threadIdx.x; i < n; i += kPlanThreads) {
        const int s = src[i], d = dst[i];
        if (s < 0 || s >= p.max_seqs || d < 0 || d >= p.max_seqs || !mark(marks, d)) bad = true;
        else if (p.len[d] != 0 || p.len[s] < 0 || p.len[s] > cap) bad = true;
    }
    bad = __syncthreads_or(bad);
    for (int i = threadIdx.x; !bad && i < n; i += kPlanThreads)
        if (marks[src[i] >> 5] >> (src[i] & 31) & 1u) bad = true;  // a source that the call also makes
    bad = __syncthreads_or(bad);
    // How many pages each item takes (a warp per item), then where its first one stands.  Entries that a branch shares are
    // looked at too, once where a warp's items have the same source: they are to name pages that the pool has.
    for (int i = warp, before = -1; !bad && i < n; i += kPlanWarps) {
        const int s = src[i], len = p.len[s], e1 = entries_of(p, len), own = first_own_entry(p, len, deep);
        const int* row = p.table + (size_t)s * p.max_pages;
        int mine = 0;
        bool off = false;
#pragma unroll 4
        for (int e = (s == before ? own : 0) + lane; e < e1; e += 32) {
            const int page = row[e];
            mine += page >= 0 && e >= own;
            off |= page >= p.num_pages;
        }
        before = s;
        bad |= __any_sync(0xffffffffu, off);
        mine = __reduce_add_sync(0xffffffffu, mine);
        if (lane == 0) plan.first[i] = mine;
    }
    bad = __syncthreads_or(bad);
    int need = 0;
    for (int base = 0; !bad && base < n && need <= p.num_pages; base += kPlanThreads) {
        const int i = base + (int)threadIdx.x;
        int total;
        const int at = block_scan(i < n ? plan.first[i] : 0, &total);
        if (i < n) plan.first[i] = need + at;
        need += total;
    }
    __syncthreads();
    bool short_of = need > p.num_pages;
    if (!bad && !short_of) short_of = list_pages(p.ref, 0, p.num_pages, false, need, plan.fresh) < need;
    __syncthreads();
    plan_done(plan.head, bad, short_of, need, st);
    if (bad || short_of) return;
    for (int i = warp; i < n; i += kPlanWarps) {
        const int s = src[i], len = p.len[s], e1 = entries_of(p, len);
        const int* row = p.table + (size_t)s * p.max_pages;
        int at = plan.first[i];
        for (int e0 = first_own_entry(p, len, deep); e0 < e1; e0 += 32) {
            const int e = e0 + lane, page = e < e1 ? row[e] : -1;
            const unsigned int have = __ballot_sync(0xffffffffu, page >= 0);
            const int m = at + __popc(have & ((1u << lane) - 1u));
            if (page >= 0) plan.moves[m] = {page, plan.fresh[m], min(p.page_size, len - e * p.page_size)};
            at += __popc(have);
        }
    }
}

// A block of `bytes` consecutive bytes (a multiple of 16, up to 64 KB) by one warp, eight 16-byte accesses a lane
// requested at a time.  kAgain: other blocks are copied from the same bytes, which had better stay in L2.
template <bool kAgain>
__device__ __forceinline__ void copy_block(char* to, const char* from, int bytes, int lane)
{
    const uint4* f = reinterpret_cast<const uint4*>(from);
    uint4* t = reinterpret_cast<uint4*>(to);
    const int n = bytes / 16;
    for (int i = lane; i < n; i += 8 * 32) {
        uint4 x[8];
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (i + j * 32 < n) x[j] = kAgain ? __ldg(f + i + j * 32) : __ldcs(f + i + j * 32);
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (i + j * 32 < n) __stcs(t + i + j * 32, x[j]);
    }
}

// The rows of a plan's moves: a (move, layer, tensor, head) block per warp and turn.  Neighbouring warps have
// neighbouring heads of a page; with kAgain (branches: several moves from one page) neighbouring moves of a head, so
// that the page's rows are read from memory once.  (A block per CTA and turn left two accesses a thread in flight:
// 113 us for 350 MB.  The rows read as if for the only time, page by page: 88 us.)
template <bool kAgain>
__device__ void copy_rows(const KVPages& p, const Plan& plan, int row_bytes)
{
    const int lane = threadIdx.x & 31;
    const unsigned int lt = p.num_layers * 2, per_move = lt * p.kv_heads;  // no pool has 2^32 blocks: it has fewer rows
    const unsigned int moves = plan.head->moves, units = moves * per_move, warps = gridDim.x * (kApplyThreads / 32);
    const size_t block = (size_t)p.page_size * row_bytes;
    for (unsigned int u = blockIdx.x * (kApplyThreads / 32) + (threadIdx.x >> 5); u < units; u += warps) {
        const unsigned int major = u / (kAgain ? moves : per_move), minor = u - major * (kAgain ? moves : per_move);
        const unsigned int move = kAgain ? minor : major, in_move = kAgain ? major : minor, q = in_move / p.kv_heads, h = in_move - q * p.kv_heads;
        const Move m = plan.moves[move];
        char* slab = static_cast<char*>((q & 1) ? p.v : p.k) + ((size_t)(q >> 1) * p.num_pages * p.kv_heads + h) * block;
        copy_block<kAgain>(slab + (size_t)m.to * p.kv_heads * block, slab + (size_t)m.from * p.kv_heads * block, m.rows * row_bytes, lane);
    }
}

__global__ void __launch_bounds__(kApplyThreads)
    pages_fork_apply_kernel(const KVPages p, const int* src, const int* dst, int n, int deep, int row_bytes, void* ws)
{
    const Plan plan = plan_at(ws, n, p.num_pages);
    after_predecessor();
    if (!plan.head->ok) return;
    const int lane = threadIdx.x & 31;
    // Tables and counts: a warp per item.
    for (int i = (int)(blockIdx.x * (kApplyThreads / 32) + (threadIdx.x >> 5)); i < n; i += (int)gridDim.x * (kApplyThreads / 32)) {
        const int s = src[i], d = dst[i], len = p.len[s];
        const int own = first_own_entry(p, len, deep), e1 = entries_of(p, len);
        const int* from = p.table + (size_t)s * p.max_pages;
        int* to = p.table + (size_t)d * p.max_pages;
        int at = plan.first[i];
        for (int e0 = 0; e0 < p.max_pages; e0 += 32) {
            const int e = e0 + lane;
            int page = e < e1 ? from[e] : -1;
            const unsigned int fresh = __ballot_sync(0xffffffffu, page >= 0 && e >= own);
            if (page >= 0) {
                if (e >= own) {
                    page = plan.fresh[at + __popc(fresh & ((1u << lane) - 1u))];
                    p.ref[page] = 1;
                } else {
                    atomicAdd(&p.ref[page], 1);
                }
            }
            at += __popc(fresh);
            if (e < p.max_pages) to[e] = page;
        }
        if (lane == 0) p.len[d] = len;
    }
    copy_rows<true>(p, plan, row_bytes);
}

// ---- free and trim -----------------------------------------------------------------------------

// What a call takes of each sequence's table row.  trim: only entries wholly in rows [sinks, len - window); else all,
// and the sequence ends (whatever its length says: a row can be freed in any state).
struct Release {
    int trim, window, sinks;
    __device__ __forceinline__ int begin(const KVPages& p) const { return trim ? (sinks + p.page_size - 1) / p.page_size : 0; }
    __device__ __forceinline__ int end(const KVPages& p, int s) const { return trim ? min(p.max_pages, max(0, p.len[s] - window) / p.page_size) : p.max_pages; }
    // Both by lanes of which each has every `step`-th entry from its `first` on, kAtOnce of them at a time.
    static constexpr int kAtOnce = 8;
    __device__ __forceinline__ void read(const int* row, int e, int step, int e1, int (&page)[kAtOnce]) const
    {
#pragma unroll
        for (int i = 0; i < kAtOnce; i++) page[i] = e + i * step < e1 ? row[e + i * step] : -1;
    }
    // Whether sequence s is one, of a length that its table has, and its entries name pages that the pool has.
    __device__ __forceinline__ bool right(const KVPages& p, int s, int first, int step) const
    {
        if (s < 0 || s >= p.max_seqs) return false;
        if (trim && (p.len[s] < 0 || p.len[s] > p.max_pages * p.page_size)) return false;
        const int* row = p.table + (size_t)s * p.max_pages;
        const int e1 = end(p, s);
        bool ok = true;
        for (int e = begin(p) + first; e < e1; e += kAtOnce * step) {
            int page[kAtOnce];
            read(row, e, step, e1, page);
#pragma unroll
            for (int i = 0; i < kAtOnce; i++) ok &= page[i] < p.num_pages;
        }
        return ok;
    }
    // Each entry is taken out with an exchange, so that a sequence named twice gives its pages back once.
    __device__ __forceinline__ void take(const KVPages& p, int s, int first, int step) const
    {
        int* row = p.table + (size_t)s * p.max_pages;
        const int e1 = end(p, s);
        for (int e = begin(p) + first; e < e1; e += kAtOnce * step) {
            int page[kAtOnce];
            read(row, e, step, e1, page);
#pragma unroll
            for (int i = 0; i < kAtOnce; i++)
                if (page[i] >= 0) page[i] = atomicExch(&row[e + i * step], -1);
#pragma unroll
            for (int i = 0; i < kAtOnce; i++)
                if (page[i] >= 0) atomicSub(&p.ref[page[i]], 1);
        }
        if (!trim && first == 0) p.len[s] = 0;
    }
};

// A short list by one cluster: the CTAs look at all of it, tell each other whether it is right, and only then change
// anything.  `team` warps to a sequence.  Up to as many sequences as it has warps; in one launch / in two, in microseconds
// on the device: trim of 4, 32 and 256 sequences that has nothing to take 2.6, 2.8, 2.6 / 3.5, 3.6, 3.9; free of 32 and of 256
// with up to 64 pages 2.9, 3.6 / 3.3, 4.0, of one with 4,096 3.3 / 6.0, of 256 with up to 512 6.0 / 4.0.
constexpr int kTogether = 256;  // sequences, at most
constexpr int kClusterCtas = 8, kClusterThreads = kTogether / kClusterCtas * 32;
__global__ void __launch_bounds__(kClusterThreads) pages_release_kernel(const KVPages p, const int* seqs, int n, int team, const Release what, Status st)
{
    __shared__ int wrong[kClusterCtas];
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // this CTA's shared memory is there
    after_predecessor();
    const int warp = (int)((blockIdx.x * kClusterThreads + threadIdx.x) >> 5), item = warp / team, first = warp % team * 32 + (int)(threadIdx.x & 31);
    const int s = item < n ? seqs[item] : -1;
    const int bad = __syncthreads_or(item < n && !what.right(p, s, first, team * 32));
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // and so is the others'
    if (threadIdx.x < kClusterCtas) {  // into every CTA's array
        uint32_t at;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(&wrong[blockIdx.x])), "r"(threadIdx.x));
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(bad) : "memory");
    }
    __syncwarp();  // (the barrier's aligned form wants the warp together)
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    int any = 0;
#pragma unroll
    for (int i = 0; i < kClusterCtas; i++) any |= wrong[i];
    if (any) {
        if (blockIdx.x == 0 && threadIdx.x == 0) raise(st, TYB_STATUS_BAD_ARGUMENT);
        return;
    }
    if (item < n) what.take(p, s, first, team * 32);
}

// A long one in two launches: what each CTA of the first found, a warp to a sequence, stands in the workspace.
constexpr int kLookCtas = 2 * kSms, kLookThreads = 128;
__global__ void __launch_bounds__(kLookThreads) pages_release_look_kernel(const KVPages p, const int* seqs, int n, const Release what, int* wrong)
{
    after_predecessor();
    bool bad = false;
    for (int i = (int)(blockIdx.x * kLookThreads + threadIdx.x) >> 5; i < n; i += (int)gridDim.x * (kLookThreads / 32))
        bad |= !what.right(p, seqs[i], threadIdx.x & 31, 32);
    bad = __syncthreads_or(bad);
    if (threadIdx.x == 0) wrong[blockIdx.x] = bad;
}
__global__ void __launch_bounds__(kLookThreads) pages_release_apply_kernel(const KVPages p, const int* seqs, const Release what, const int* wrong, Status st)
{
    after_predecessor();
    int any = 0;
    for (int i = threadIdx.x; i < kLookCtas; i += kLookThreads) any |= wrong[i];
    if (__syncthreads_or(any)) {
        if (blockIdx.x == 0 && threadIdx.x == 0) raise(st, TYB_STATUS_BAD_ARGUMENT);
        return;
    }
    what.take(p, seqs[blockIdx.x], threadIdx.x, kLookThreads);
}

// ---- compact -----------------------------------------------------------------------------------

__global__ void __launch_bounds__(kPlanThreads) pages_compact_plan_kernel(const KVPages p, int* live_out, void* ws)
{
    const Plan plan = plan_at(ws, 0, p.num_pages);
    after_predecessor();
    int live = 0;
    for (int i = threadIdx.x; i < p.num_pages; i += kPlanThreads) live += p.ref[i] > 0;
    int total;
    block_scan(live, &total);
    live = total;
    // As many pages in use lie at or past `live` as free ones below it: the k-th goes to the k-th.
    const int moves = list_pages(p.ref, live, p.num_pages, true, p.num_pages, &plan.moves->from, 3);
    list_pages(p.ref, 0, live, false, moves, &plan.moves->to, 3);
    __syncthreads();
    for (int k = threadIdx.x; k < moves; k += kPlanThreads) {
        const int a = plan.moves[k].from, b = plan.moves[k].to;
        plan.moves[k].rows = p.page_size;
        plan.fresh[a] = b;
        p.ref[b] = p.ref[a];
        p.ref[a] = 0;
    }
    if (threadIdx.x == 0) {
        plan.head->ok = 1;
        plan.head->moves = moves;
        plan.head->live = live;
        if (live_out) *live_out = live;
    }
}

__global__ void __launch_bounds__(kApplyThreads) pages_compact_apply_kernel(const KVPages p, int row_bytes, void* ws)
{
    const Plan plan = plan_at(ws, 0, p.num_pages);
    after_predecessor();
    const int live = plan.head->live;
    const long long entries = (long long)p.max_seqs * p.max_pages;
    for (long long i = (long long)blockIdx.x * kApplyThreads + threadIdx.x; i < entries; i += (long long)gridDim.x * kApplyThreads) {
        const int page = p.table[i];
        if (page >= live && page < p.num_pages) p.table[i] = plan.fresh[page];
    }
    copy_rows<false>(p, plan, row_bytes);
}

// ---- rows --------------------------------------------------------------------------------------

// Token t of the list belongs to the sequence i with starts[i] <= t < starts[i + 1].
__device__ __forceinline__ int item_of(const int* starts, int n, int t)
{
    int lo = 0, hi = n;  // starts[lo] <= t < starts[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= t) lo = mid;
        else hi = mid;
    }
    return lo;
}

// A warp per (token, tensor): its row of all KV heads, eight elements per lane and turn.
template <typename In, typename T>
__global__ void __launch_bounds__(kApplyThreads)
    pages_write_kernel(const KVPages p, int layer, const int* seqs, const int* starts, int n, int rows, const In* k_new,
                       const In* v_new, long long stride, Status st)
{
    const int lane = threadIdx.x & 31;
    after_predecessor();
    const int row_vecs = p.kv_heads * p.head_dim / 8, head_vecs = p.head_dim / 8;
    for (int w = (int)(blockIdx.x * (kApplyThreads / 32) + (threadIdx.x >> 5)); w < 2 * rows; w += (int)gridDim.x * (kApplyThreads / 32)) {
        const int t = w >> 1;
        const int i = item_of(starts, n, t);
        const int s = seqs[i];
        int page = -1, at = 0;
        if (s >= 0 && s < p.max_seqs && t >= starts[i] && t < starts[i + 1]) {
            at = p.len[s] - starts[i + 1] + t;
            if (at >= 0 && at < p.max_pages * p.page_size) page = p.table[(size_t)s * p.max_pages + at / p.page_size];
        }
        if (page < 0 || page >= p.num_pages) {
            if (lane == 0) raise(st, TYB_STATUS_BAD_ARGUMENT);
            continue;
        }
        const In* from = (w & 1 ? v_new : k_new) + (size_t)t * stride;
        T* to = static_cast<T*>(w & 1 ? p.v : p.k) +
                (((size_t)layer * p.num_pages + page) * p.kv_heads * p.page_size + at % p.page_size) * p.head_dim;
        for (int c = lane; c < row_vecs; c += 32) {
            float x[8];
            load8(from + 8 * c, x);
            store8(to + (size_t)(c / head_vecs) * p.page_size * p.head_dim + 8 * (c % head_vecs), x);
        }
    }
}

// Rows of a static cache into a sequence that pages_extend_kernel has just given its pages: a block
// of consecutive rows per (entry, layer, tensor, head).
__global__ void __launch_bounds__(kApplyThreads)
    pages_import_kernel(const KVPages p, int seq, const char* k_slab, const char* v_slab, int row_capacity, int rows,
                        int row_bytes, const void* ws)
{
    after_predecessor();
    if (!static_cast<const PlanHead*>(ws)->ok) return;
    const int lane = threadIdx.x & 31;
    const unsigned int lt = p.num_layers * 2, per_entry = lt * p.kv_heads, warps = gridDim.x * (kApplyThreads / 32);
    const unsigned int units = (unsigned int)((rows + p.page_size - 1) / p.page_size) * per_entry;
    const size_t block = (size_t)p.page_size * row_bytes;
    for (unsigned int u = blockIdx.x * (kApplyThreads / 32) + (threadIdx.x >> 5); u < units; u += warps) {
        const unsigned int e = u / per_entry, in_entry = u - e * per_entry, q = in_entry / p.kv_heads, h = in_entry - q * p.kv_heads;
        const int page = p.table[(size_t)seq * p.max_pages + e];
        const char* from = ((q & 1) ? v_slab : k_slab) + (((size_t)(q >> 1) * p.kv_heads + h) * row_capacity + (size_t)e * p.page_size) * row_bytes;
        char* to = static_cast<char*>((q & 1) ? p.v : p.k) + (((size_t)(q >> 1) * p.num_pages + page) * p.kv_heads + h) * block;
        copy_block<false>(to, from, min(p.page_size, rows - (int)e * p.page_size) * row_bytes, lane);
    }
}

// ---- launches ----------------------------------------------------------------------------------

static int row_bytes_of(const KVPages* p) { return p->head_dim * (p->kv_dtype == TYB_BF16 ? 2 : 4); }

static Status status_of(const tyb_pages_env* env) { return {env->status, env->mirror}; }

// Shared memory of the duplicate check, above the default limit for pools of many sequences.
template <typename K>
static int marks_bytes(K* kernel, const KVPages* p, size_t* bytes)
{
    *bytes = (size_t)(p->max_seqs + 31) / 32 * sizeof(unsigned int);
    if (*bytes <= 40 * 1024) return 0;
    return (int)cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)*bytes);
}

}  // namespace tyb

using namespace tyb;

extern "C" size_t tyb_pages_plan_bytes(const KVPages* p, int n) { return plan_bytes(n, p->num_pages); }

extern "C" int tyb_pages_extend_launch(const KVPages* p, const tyb_pages_env* env, const int* seqs, const int* counts, int n, void* ws,
                                       void* stream)
{
    size_t marks;
    const int e = marks_bytes(pages_extend_kernel, p, &marks);
    if (e) return e;
    return launch_after(pages_extend_kernel, dim3(1), kPlanThreads, marks, (cudaStream_t)stream, *p, seqs, counts, n, 0, 0, ws, status_of(env));
}

extern "C" int tyb_pages_fork_launch(const KVPages* p, const tyb_pages_env* env, const int* src, const int* dst, int n, int deep, void* ws,
                                     void* stream)
{
    size_t marks;
    int e = marks_bytes(pages_fork_plan_kernel, p, &marks);
    if (!e) e = launch_after(pages_fork_plan_kernel, dim3(1), kPlanThreads, marks, (cudaStream_t)stream, *p, src, dst, n, deep, ws, status_of(env));
    if (e) return e;
    return launch_after(pages_fork_apply_kernel, dim3(kSms * 8), kApplyThreads, 0, (cudaStream_t)stream, *p, src, dst, n, deep, row_bytes_of(p), ws);
}

static int launch_release(const KVPages* p, const tyb_pages_env* env, const int* seqs, int n, const Release& what, void* ws, cudaStream_t stream)
{
    if (n <= kTogether) {
        int team = 1;
        while (2 * team * n <= kTogether) team *= 2;
        return launch_after_in(kClusterCtas, pages_release_kernel, dim3(kClusterCtas), kClusterThreads, 0, stream, *p, seqs, n, team, what, status_of(env));
    }
    int* wrong = static_cast<int*>(ws);
    const int e = launch_after(pages_release_look_kernel, dim3(kLookCtas), kLookThreads, 0, stream, *p, seqs, n, what, wrong);
    return e ? e : launch_after(pages_release_apply_kernel, dim3(n), kLookThreads, 0, stream, *p, seqs, what, wrong, status_of(env));
}

extern "C" size_t tyb_pages_release_bytes(int n) { return n <= kTogether ? 0 : kLookCtas * sizeof(int); }

extern "C" int tyb_pages_free_launch(const KVPages* p, const tyb_pages_env* env, const int* seqs, int n, void* ws, void* stream)
{
    return launch_release(p, env, seqs, n, Release{0, 0, 0}, ws, (cudaStream_t)stream);
}

extern "C" int tyb_pages_trim_launch(const KVPages* p, const tyb_pages_env* env, const int* seqs, int n, int window, int sinks, void* ws, void* stream)
{
    return launch_release(p, env, seqs, n, Release{1, window, sinks}, ws, (cudaStream_t)stream);
}

extern "C" int tyb_pages_compact_launch(const KVPages* p, int* live_out, void* ws, void* stream)
{
    const int e = launch_after(pages_compact_plan_kernel, dim3(1), kPlanThreads, 0, (cudaStream_t)stream, *p, live_out, ws);
    if (e) return e;
    return launch_after(pages_compact_apply_kernel, dim3(kSms * 8), kApplyThreads, 0, (cudaStream_t)stream, *p, row_bytes_of(p), ws);
}

template <typename In, typename T>
static int launch_write(const KVPages* p, const tyb_pages_env* env, int layer, const int* seqs, const int* starts, int n, int rows,
                        const void* k_new, const void* v_new, long long stride, cudaStream_t stream)
{
    const int per_cta = kApplyThreads / 32;
    const long long ctas = (2LL * rows + per_cta - 1) / per_cta;
    return launch_after(pages_write_kernel<In, T>, dim3((unsigned)(ctas < kSms * 16 ? ctas : kSms * 16)), kApplyThreads, 0, stream, *p, layer,
                        seqs, starts, n, rows, static_cast<const In*>(k_new), static_cast<const In*>(v_new), stride, status_of(env));
}

extern "C" int tyb_pages_write_launch(const KVPages* p, const tyb_pages_env* env, int layer, const int* seqs, const int* starts, int n,
                                      int rows, const void* k_new, const void* v_new, int in_bf16, long long stride, void* stream)
{
    typedef __nv_bfloat16 bf;
    auto* launch = p->kv_dtype == TYB_BF16 ? (in_bf16 ? launch_write<bf, bf> : launch_write<float, bf>)
                                           : (in_bf16 ? launch_write<bf, float> : launch_write<float, float>);
    return launch(p, env, layer, seqs, starts, n, rows, k_new, v_new, stride, (cudaStream_t)stream);
}

extern "C" int tyb_pages_import_launch(const KVPages* p, const tyb_pages_env* env, int seq, const void* k_slab, const void* v_slab,
                                       int row_capacity, int rows, void* ws, void* stream)
{
    size_t marks;
    int e = marks_bytes(pages_extend_kernel, p, &marks);
    if (!e)
        e = launch_after(pages_extend_kernel, dim3(1), kPlanThreads, marks, (cudaStream_t)stream, *p, nullptr, nullptr, 1, seq, rows, ws,
                         status_of(env));
    if (e) return e;
    return launch_after(pages_import_kernel, dim3(kSms * 8), kApplyThreads, 0, (cudaStream_t)stream, *p, seq, static_cast<const char*>(k_slab),
                        static_cast<const char*>(v_slab), row_capacity, rows, row_bytes_of(p), ws);
}

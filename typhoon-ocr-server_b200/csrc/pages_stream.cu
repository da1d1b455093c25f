// pages_stream.cu -- single-token attention over the paged cache: every sequence's own rows (all of
// them, those behind a shared prefix, or those in a window with sinks) and, for batches too small for
// the tcgen05 form, the shared prefix itself.
//
// The work is memory traffic: each K and V element meets q_heads / kv_heads query rows (a prefix
// element at most 16) once.  So the kernel is two CTAs per SM that stream equal shares of all the call's
// rows, whatever the lengths: the key tiles of all (sequence, KV head) items, laid end to end,
// are cut into gridDim.x equal runs.  One warp requests a run's tiles with TMA into a ring of stages,
// crossing from item to item without a pause (item starts bring their query rows along).  Two teams of
// two warps take the stages in turn, a warp 32 (BF16) or 16 (FP32) of its rows, with the running maximum
// and sum of an online softmax in base 2; at an item's end each leaves its rows in shared memory and goes on, and
// the last to do so joins the four.  (A stage is a chain of dependent steps, about a microsecond: few keys per
// warp make it no shorter, so four of them at a time per SM keep up with the memory, two do not.)
// An item that a run boundary cuts is joined by the CTA that finishes it last (records in the workspace, a
// ticket per item); the order of that sum is by run, not by arrival, so results repeat exactly.
//
// Long items: 512 windows of 2,048 rows and 16 sinks in 610 us, 4.2 GB at the rate of a copy.  Short ones are bound by
// the stage's round trip (request, arrival, two warps' products, release) over a ring of three: 1.0 us a stage,
// 256 x 8 items of 4.6 stages in 60 us on 116 SMs.
//
// The products (pages_mma.cuh) are mma.sync, with up to 16 query rows as columns.
#define TYB_WHOLE_PROGRAM
#include "pages_attn.cuh"
#include "pages_mma.cuh"
#include "tcgen05.cuh"

namespace tyb {

constexpr int kTeam = 2;                         // warps that share a stage
constexpr int kTakers = 2 * kTeam;               // warps that consume stages: two teams, in turn
constexpr int kTakerThreads = 32 * kTakers;
constexpr int kStreamThreads = kTakerThreads + 32;  // + the requesting warp
constexpr int kMaxStages = 10;
constexpr int kItemRing = 16;                    // > kMaxStages: a taker reads of an item while that many stages follow
constexpr int kStreamRuns = 2 * kSms;            // CTAs, at most

template <typename T, int D>
struct Stream {
    static constexpr int kKeys = sizeof(T) == 2 ? 32 : 16;  // of a warp
    static constexpr int kRows = kTeam * kKeys;             // of a stage
    static constexpr int kBoxCols = 128 / (int)sizeof(T);   // columns of a 128-byte box
    static constexpr int kBoxes = D / kBoxCols;
    static constexpr int kBox = kRows * 128;                // bytes
    static constexpr int kHalf = kBoxes * kBox;             // K (or V) of a stage
    static constexpr int kStage = 2 * kHalf;
    static constexpr int kPitch = D + 4;                    // floats; joins and FP32 queries
};

// What the requesting warp tells the takers: about an item,
struct Item {
    int shared;       // of the shared pass
    int tok0, ntok, kvh;
    int pos, lo, sinks;
    int c0, c1, s0;   // the runs that have part of it, and which record of run c0 is its
};
// about a stage: its first row's key, a bit per 8 rows whose page is there, and
struct __align__(16) Stage {
    int k0;
    unsigned int seen;
    int flags;
    int more;
};
constexpr int kFirst = 1, kLast = 2, kEnd = 4;  // of its item (in this run), of its item, of the run

// Where the records of a (token, KV head) lie: in runs sh0 .. sh1 those of its shared item (none: sh1 < sh0), in runs
// own0 .. own1 its own; *_second: whether that of the first such run is the run's second record.
struct Parts {
    int sh0, sh1, sh_second, own0, own1, own_second;
};

struct Maps {
    CUtensorMap m[4];  // K, V; K, V in boxes of 16 rows by 128 bytes
};

struct StreamArgs {
    AttnArgs a;
    int layer;
    int tok_base;      // token (row of q) of this launch's first sequence
    int shared_tiles;  // row tiles of the shared pass in this launch (0: none)
    int shared_units;  // units of each: kItemUnits and the stages of its rows
    int out_slot;      // record slot of a.rec that receives the results; -1: they are the output
    int beside;        // runs at the same time as the kernel before
    int max_len;
    int stages, q_bytes, item_rows;
    // Records of this launch: [2 * kStreamRuns][16] rows of items cut by a run boundary; with a shared pass, uncut
    // items too: [batch * q_heads] own rows, then [shared_tiles * kv_heads][16] shared ones.
    float* rec_o;
    float2* rec_ml;
    unsigned int* gave_up;  // not zero: a wait ran out in a launch before, whose tickets may be half counted
    unsigned int* tickets;  // [batch * kv_heads], zero between launches
    unsigned long long wait_ns;
};

// `total` units in `runs` runs whose sizes differ by at most one (runs <= total < 2^31: no run is empty,
// and 32-bit arithmetic will do).
struct Runs {
    unsigned int runs, base, more;  // the first `more` runs have base + 1
    __device__ __forceinline__ Runs(unsigned int total, unsigned int n) : runs(n), base(total / n), more(total % n) {}
    __device__ __forceinline__ unsigned int start(unsigned int run) const { return run * base + min(run, more); }
    __device__ __forceinline__ unsigned int of(unsigned int u) const
    {
        const unsigned int split = more * (base + 1);
        return u < split ? u / (base + 1) : more + (u - split) / base;
    }
    // The runs c0 .. c1 that have stages of the item of units [u0, u1), and which record of run c0 is the item's
    // (0: its first item's, 1: its last's, an earlier item having ended in the run; in the later runs it comes
    // first).
    __device__ __forceinline__ void span(unsigned int u0, unsigned int u1, int& c0, int& c1, int& s0) const
    {
        c0 = (int)of(u0 + kItemUnits);
        c1 = (int)of(u1 - 1);
        s0 = start(c0) < u0;
    }
};

// Four output columns joined over several records: maximum (base 2), sum, values.
struct Gather {
    float m = -INFINITY, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    __device__ __forceinline__ void add(float2 ml, float4 x)
    {
        // a record that saw nothing has l = 0, o = 0 and m = -inf: its factor is 0
        const float top = fmaxf(m, ml.x), f = m == -INFINITY ? 0.f : fast_exp2(m - top), e = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - top);
        m = top;
        // (which product is rounded is spelled out, so that every place where this is inlined gives the same bits)
        l = fmaf(l, f, __fmul_rn(ml.y, e));
        o.x = fmaf(o.x, f, __fmul_rn(x.x, e));
        o.y = fmaf(o.y, f, __fmul_rn(x.y, e));
        o.z = fmaf(o.z, f, __fmul_rn(x.z, e));
        o.w = fmaf(o.w, f, __fmul_rn(x.w, e));
    }
};

template <typename T, int D, int kBlocks, bool kDup>
__global__ void __launch_bounds__(kStreamThreads, 2)
    pages_stream_kernel(const __grid_constant__ Maps maps, const StreamArgs sa)
{
    using S = Stream<T, D>;
    const AttnArgs& a = sa.a;
    extern __shared__ __align__(1024) unsigned char raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    unsigned char* ring = smem;
    float* joins = reinterpret_cast<float*>(ring + sa.stages * S::kStage);  // [kTakers][item_rows][kPitch]
    float* split_q = joins + kTakers * sa.item_rows * S::kPitch;  // FP32: hi and lo, [split_rows][kPitch] each
    constexpr int split_rows = sizeof(T) == 4 && !kDup ? 8 * kBlocks : 0;
    unsigned char* qs = reinterpret_cast<unsigned char*>(split_q + 2 * split_rows * S::kPitch);  // [stages][q_bytes]
    int* cum = reinterpret_cast<int*>(qs + sa.stages * sa.q_bytes);        // units before each sequence
    int* lens = cum + a.batch + 1;

    __shared__ uint64_t full[kMaxStages], empty[kMaxStages], met, joined;
    __shared__ int left_rows;  // warps whose rows of the item lie in the join rows
    __shared__ Stage stages_of[kMaxStages];
    __shared__ Item items[kItemRing];
    __shared__ float2 join_mls[kTakers][16];
    __shared__ int scan[kStreamThreads / 32];
    __shared__ unsigned int last_of;  // tokens whose join is this CTA's
    __shared__ Parts parts_of[16];    // and where their records lie

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int heads = a.p.kv_heads, run = blockIdx.x;

    if (tid == 0) {
        for (int i = 0; i < sa.stages; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], kTakers);
        }
        mbar_init(&met, kTakers);
        mbar_init(&joined, 1);
        left_rows = 0;
        fence_barrier_init();
    }
    if (sa.beside) {
        let_next_start();
        __threadfence();  // nothing read before by this SM is taken for the page table's or the lengths' state
    } else {
        after_predecessor();
    }
    unsigned int gave_up = __ldcg(sa.gave_up);  // (wanted further down, with the lengths)
    // Units of each sequence's own rows: kItemUnits, then its stages, of which it has one at least, so that every
    // output row has an owner.
    auto own_lo = [&](int len) { return a.window ? max(0, len - a.window) : min(a.prefix, len); };
    // A thread takes consecutive sequences, so that all loads are in flight at once and one scan will do.
    long long before = 0;
    {
        constexpr int kPer = (kStreamSeqs + kStreamThreads - 1) / kStreamThreads;
        const int each = (a.batch + kStreamThreads - 1) / kStreamThreads, b0 = tid * each;
        int len[kPer], n = 0;
#pragma unroll
        for (int i = 0; i < kPer; i++) len[i] = i < each && b0 + i < a.batch ? a.seqs[b0 + i] : -1;
#pragma unroll
        for (int i = 0; i < kPer; i++)
            if (i < each && b0 + i < a.batch) len[i] = checked_len(a.p, len[i], a.st);
#pragma unroll
        for (int i = 0; i < kPer; i++)
            if (i < each && b0 + i < a.batch) {
                // too long for the call's split, or without all of the shared rows (a sequence not in use aside, whose row means
                // nothing, unless the shared rows are to be found by it)
                if (len[i] > sa.max_len || (len[i] < a.prefix && (len[i] > 0 || b0 + i == 0))) {
                    raise(a.st, TYB_STATUS_BAD_ARGUMENT);
                    len[i] = 0;
                }
                lens[b0 + i] = len[i];
                len[i] = kItemUnits + max(1, tiles_of(len[i] - 1, own_lo(len[i]), a.sinks, S::kRows).count());
                n += len[i];
            }
        int sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += y;
        }
        if (lane == 31) scan[warp] = sum;
        gave_up = __syncthreads_or((int)gave_up);
        int at = sum - n;
#pragma unroll
        for (int w = 0; w < kStreamThreads / 32; w++) {
            if (w < warp) at += scan[w];
            before += scan[w];
        }
#pragma unroll
        for (int i = 0; i < kPer; i++)
            if (i < each && b0 + i < a.batch) {
                cum[b0 + i] = at;
                at += len[i];
            }
    }
    if (tid == 0) cum[a.batch] = (int)before;
    __syncthreads();
    if (gave_up) {
        if (tid == 0) {
            atomicOr(sa.gave_up, 1u);
            raise(a.st, TYB_STATUS_WAIT_TIMEOUT);
        }
        if (sa.beside) wait_for_predecessor();
        return;
    }
    const unsigned long long all = ((unsigned long long)sa.shared_tiles * sa.shared_units + before) * heads;
    if (all >= 1ull << 31) {  // only tables that name pages over and over
        if (tid == 0) raise(a.st, TYB_STATUS_BAD_ARGUMENT);
        if (sa.beside) wait_for_predecessor();
        return;
    }
    const Runs cuts((unsigned int)all, min(gridDim.x, (unsigned int)all));
    if (run >= (int)cuts.runs) return;
    const unsigned int shared_all = (unsigned int)sa.shared_tiles * sa.shared_units * heads;
    const unsigned int begin = cuts.start(run), end = cuts.start(run + 1);
    const int per = 16 / a.group;  // tokens of a shared row tile

    // A wait, by all lanes of a warp.  (The mark is left where the wait itself gives up: behind the vote it was in the way of
    // every wait, 256 questions 70.3 us for 69.5.)
    auto waited = [&](uint64_t* bar, uint32_t parity, uint64_t limit_ns) {
        bool out = false;
        if (!wait_for(bar, parity, limit_ns, a.st)) {
            atomicOr(sa.gave_up, 1u);
            out = true;
        }
        return !__any_sync(0xffffffffu, out);
    };

    if (warp == kTakers) {
        // ---- requests
        // Lane (part, box, K or V): a stage's rows come as one copy of whole rows, or in 2 or 4 parts (pages; 16 rows
        // each where not all of the stage is in sight, so that no more is read than that), each 128-byte column box
        // of each as a copy.
        const int shift = page_shift(a.p.page_size), whole = max(0, page_shift(S::kRows) - shift);
        struct Lane {
            int parts, rows, part, box, which, to;
            uint32_t bytes;
        };
        auto lane_of = [&](int parts_log2, bool all_boxes) {
            Lane l;
            const int other = lane >> parts_log2;  // lane / parts
            l.parts = 1 << parts_log2;
            l.rows = S::kRows >> parts_log2;
            l.part = lane & (l.parts - 1);
            l.box = all_boxes ? 0 : other % S::kBoxes;
            l.which = all_boxes ? other : other / S::kBoxes;
            l.to = l.which * S::kHalf + l.box * S::kBox + l.part * l.rows * 128;
            l.bytes = (uint32_t)(l.rows * 128 * (all_boxes ? S::kBoxes : 1));
            return l;
        };
        const Lane coarse = lane_of(whole, whole == 0), finer = lane_of(page_shift(S::kRows) - 4, false);
        Lane mine = coarse;
        bool fine = false;
        const uint32_t q_row = (uint32_t)(a.group * D * (a.io_bf16 ? 2 : 4));
        const int max_page = a.p.num_pages;
        Item item = {};
        Tiles list = {};
        const int* table = a.p.table;
        unsigned int u = begin, u0 = 0, u1 = 0, sent = 0;  // u0, u1: the current item's units
        int b = 0, st = 0, page = -1, item_at = kItemRing - 1, k0 = 0, flags = 0;
        uint32_t phase = 0;
        bool ok = true, more = true;
        // The next stage: what it holds, and the lane's page of it (requested here, so that its way from memory
        // passes while the stage before waits for its place).  kEnd: none follows.
        auto next = [&]() {
            const bool first = u == begin || u >= u1;
            if (first) {  // the item that unit u lies in
                if (u < shared_all) {
                    const unsigned int n = u / sa.shared_units;
                    u0 = n * sa.shared_units;
                    u1 = u0 + sa.shared_units;
                    item.shared = 1;
                    item.kvh = (int)(n % heads);
                    item.tok0 = (int)(n / heads) * per;
                    item.ntok = min(per, a.batch - item.tok0);
                    item.sinks = 0;
                    item.lo = 0;
                    item.pos = min(a.prefix, lens[0]) - 1;
                    table = a.p.table + (size_t)(lens[0] ? a.seqs[0] : 0) * a.p.max_pages;
                } else {
                    bool other = true;
                    if (u == begin) {  // which sequence: cum[b] * heads <= u - shared_all
                        int lo = 0, hi = a.batch;
                        while (hi - lo > 1) {
                            const int mid = (lo + hi) >> 1;
                            if ((unsigned int)(cum[mid] * heads) <= u - shared_all) lo = mid;
                            else hi = mid;
                        }
                        b = lo;
                    } else if (u - shared_all >= (unsigned int)(cum[b + 1] * heads)) {
                        b++;
                    } else {
                        other = item.shared;
                    }
                    const unsigned int units = cum[b + 1] - cum[b];
                    if (u == begin) {
                        const unsigned int at = u - shared_all - cum[b] * heads;
                        item.kvh = (int)(at / units);
                        u0 = u - at % units;
                    } else {
                        item.kvh = other ? 0 : item.kvh + 1;
                        u0 = u;
                    }
                    u1 = u0 + units;
                    if (other) {
                        item.shared = 0;
                        item.tok0 = b;
                        item.ntok = 1;
                        item.sinks = a.sinks;
                        item.pos = lens[b] - 1;
                        item.lo = own_lo(lens[b]);
                        table = a.p.table + (size_t)(lens[b] ? a.seqs[b] : 0) * a.p.max_pages;
                    }
                }
                // items inside the run are whole: only its first and last may lie in others too
                item.c0 = item.c1 = run;
                item.s0 = 0;
                if (u == begin || u1 > end) cuts.span(u0, u1, item.c0, item.c1, item.s0);
                list = tiles_of(item.pos, item.lo, item.sinks, S::kRows);
                if (u < u0 + kItemUnits) u = min(u0 + kItemUnits, end);
            }
            const bool none = u == end;  // the run ends before the item's first stage
            flags = (none ? 0 : (first ? kFirst : 0) | (u + 1 == u1 || u + 1 == end ? kLast : 0)) |
                    (none || (u + 1 == u1 ? u1 + kItemUnits : u + 1) >= end ? kEnd : 0);
            const int i = none ? list.count() : (int)(u - u0 - kItemUnits);
            const bool real = i < list.count();
            k0 = real ? list.at(i) * S::kRows : item.pos + 1;
            fine = k0 + S::kRows - 1 > item.pos || (k0 < item.lo && k0 + S::kRows > item.sinks);
            mine = fine ? finer : coarse;
            const int key = k0 + mine.part * mine.rows;
            page = real && mine.which < 2 && key <= item.pos && (key + mine.rows > item.lo || key < item.sinks) ? table[key >> shift] : -1;
            u++;
        };
        next();
        while (more) {
            if (sent >= (unsigned int)sa.stages) {
                ok = waited(&empty[st], phase ^ 1u, sa.wait_ns);
                if (!ok) break;
            }
            if (page >= max_page) {
                raise(a.st, TYB_STATUS_BAD_ARGUMENT);
                page = -1;
            }
            const unsigned int have = __ballot_sync(0xffffffffu, page >= 0);
            if (flags & kFirst) {
                if (++item_at == kItemRing) item_at = 0;
                if (lane == 0) items[item_at] = item;
            }
            if (lane == 0) {
                unsigned int seen = 0;
                for (int l = 0; l < mine.parts; l++)
                    if (have >> l & 1u) seen |= (0xffu >> (8 - mine.rows / 8)) << (l * (mine.rows / 8));
                stages_of[st] = Stage{k0, seen, flags, 0};
                mbar_arrive_expect_tx(&full[st], __popc(have) * mine.bytes + (flags & kFirst ? q_row * (uint32_t)item.ntok : 0u));
            }
            __syncwarp();
            if (page >= 0) {
                const int row = ((sa.layer * a.p.num_pages + page) * heads + item.kvh) * a.p.page_size + ((k0 + mine.part * mine.rows) & (a.p.page_size - 1));
                tma_load_3d(ring + st * S::kStage + mine.to, &maps.m[2 * fine + mine.which], row, mine.box, &full[st]);
            }
            if ((flags & kFirst) && lane < item.ntok)
                bulk_g2s(qs + st * sa.q_bytes + lane * q_row,
                         static_cast<const char*>(a.q) + ((size_t)(sa.tok_base + item.tok0 + lane) * a.q_stride + (size_t)item.kvh * a.group * D) *
                                                             (a.io_bf16 ? 2 : 4),
                         q_row, &full[st]);
            sent++;
            if (++st == sa.stages) {
                st = 0;
                phase ^= 1u;
            }
            more = !(flags & kEnd);
            if (more) next();
        }
        // The copies requested have landed before this warp, and with it the CTA, ends.
        const unsigned int all_stages = sa.stages;
        for (unsigned int n = sent > all_stages ? sent - all_stages : 0; n < sent; n++)
            waited(&full[n % all_stages], n / all_stages & 1u, drain_ns(sa.wait_ns));
        if (sa.beside) wait_for_predecessor();  // so that the end of this kernel is the end of that one as well
        return;
    }

    // ---- takers
    const int g = lane >> 2, t = lane & 3, team = warp / kTeam, r0 = warp % kTeam * S::kKeys;
    Rows<T, D, kBlocks, kDup> w;
    w.clear();
    int st = 0, turn = 0;  // turn: whose stage it is
    uint32_t phase = 0;
    int item_at = kItemRing - 1;
    bool one_item = true;  // no item has ended in this run yet
    int direct_items = 0;
    // Rows of the records: of a cut item's part in a run, of uncut own rows, of an uncut shared item.
    auto part_row = [&](int run_of, int second) { return (2 * run_of + second) * 16; };
    auto own_row = [&](int tok, int kvh) { return 2 * kStreamRuns * 16 + tok * a.q_heads + kvh * a.group; };
    auto shared_row = [&](int tok, int kvh) {
        return 2 * kStreamRuns * 16 + a.batch * a.q_heads + (tok / per * heads + kvh) * 16;
    };
    // The takers meet at an mbarrier rather than a CTA barrier: its wait is bounded, so that a warp whose
    // wait ran out and left does not leave the others waiting.
    uint32_t meeting = 0;
    auto meet = [&]() {
        warp_arrive(&met);
        const bool ok = waited(&met, meeting, sa.wait_ns);
        meeting ^= 1u;
        return ok;
    };
    // A finished row block: the output, or its record for the join kernel.
    auto deliver = [&](size_t R, int c, const Gather& x) {
        if (sa.out_slot < 0) {
            put_out(a, R * D + c, x.o, x.l);
        } else {
            const size_t at = (size_t)sa.out_slot * a.rec.rows + R;
            *reinterpret_cast<float4*>(a.rec.o + at * D + c) = x.o;
            if (c == 0) a.rec.ml[at] = make_float2(x.m, x.l);
        }
    };
    // Four columns of a row, joined over the warps' shares in shared memory.
    auto over_warps = [&](int row, int c) {
        Gather sum;
#pragma unroll
        for (int x = 0; x < kTakers; x++)
            sum.add(join_mls[x][row], *reinterpret_cast<const float4*>(joins + (x * sa.item_rows + row) * S::kPitch + c));
        return sum;
    };
    for (bool more = true; more;) {
        if (!waited(&full[st], phase, sa.wait_ns)) return;
        const Stage stage = stages_of[st];
        if ((stage.flags & kFirst) && ++item_at == kItemRing) item_at = 0;
        const Item& tile = items[item_at];
        const int nrows = tile.ntok * a.group;
        more = !(stage.flags & kEnd);
        if (stage.flags & kFirst) {
            w.load_q(qs + st * sa.q_bytes, nrows, a.io_bf16, g, t, split_q, tid, kTakerThreads);
            if (split_rows && !meet()) return;
        }
        const int j0 = stage.k0 + r0;
        unsigned char* rows_k = ring + st * S::kStage;
        unsigned char* rows_v = rows_k + S::kHalf;
        const unsigned int want = (1u << (S::kKeys / 8)) - 1u, seen = stage.seen >> (r0 / 8) & want;
        // the other team's stage, or none of the warp's rows in sight: nothing to do
        const bool any = turn == team && seen && j0 <= tile.pos && (j0 + S::kKeys > tile.lo || j0 < tile.sinks);
        if (any) {
            unsigned int see = 0xffffffffu >> (32 - S::kKeys);  // bit i: row j0 + i
            if (seen != want || j0 + S::kKeys - 1 > tile.pos || (j0 < tile.lo && j0 + S::kKeys > tile.sinks)) {
                auto under = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };
                unsigned int pages = 0;
#pragma unroll
                for (int i = 0; i < S::kKeys / 8; i++)
                    if (seen >> i & 1u) pages |= 0xffu << (8 * i);
                see &= pages & under(tile.pos + 1 - j0) & (~under(tile.lo - j0) | under(tile.sinks - j0));
                // what lies in rows out of sight may be anything, and 0 * NaN is not 0
                for (int i = 0; i < S::kKeys; i++)
                    if (!(see >> i & 1u) && lane < D * (int)sizeof(T) / 16)
                        *reinterpret_cast<uint4*>(rows_v + (lane >> 3) * S::kBox + (r0 + i) * 128 + (lane & 7) * 16) = make_uint4(0, 0, 0, 0);
                fence_proxy_async_smem();
                __syncwarp();
            }
            w.step(rows_k, rows_v, S::kBox, r0, SameSight<S::kKeys>{see}, a.scale_log2, split_q, g, t, lane);
        }
        warp_arrive(&empty[st]);
        turn ^= 1;
        if (++st == sa.stages) {
            st = 0;
            phase ^= 1u;
        }
        if (!(stage.flags & kLast)) continue;
        const bool first_item = one_item;
        one_item = false;

        // ---- the item's end in this run: join the warps
        const bool cut = tile.c0 != tile.c1, direct = !cut && !sa.shared_tiles;
        if (direct && !split_rows) {
            // An item to itself: each warp leaves its rows and goes on to the next item; the last to do so joins them.
            if (direct_items > 0 && !waited(&joined, (uint32_t)(direct_items - 1) & 1u, sa.wait_ns)) return;
            direct_items++;
            w.put(joins + warp * sa.item_rows * S::kPitch, S::kPitch, join_mls[warp], nrows, g, t);
            w.clear();
            __syncwarp();
            int before_me = 0;
            if (lane == 0) {
                __threadfence_block();
                before_me = atomicAdd(&left_rows, 1);
                __threadfence_block();
            }
            before_me = __shfl_sync(0xffffffffu, before_me, 0);
            __syncwarp();
            if (before_me != kTakers - 1) continue;
            if (lane == 0) left_rows = 0;
            for (int i = lane; i < nrows * (D / 4); i += 32) {
                const int row = i / (D / 4), c = i % (D / 4) * 4;
                deliver((size_t)(sa.tok_base + tile.tok0) * a.q_heads + tile.kvh * a.group + row, c, over_warps(row, c));
            }
            warp_arrive(&joined);
            continue;
        }
        // Others by all four together, once nobody needs the join rows.
        if (!first_item && !meet()) return;
        w.put(joins + warp * sa.item_rows * S::kPitch, S::kPitch, join_mls[warp], nrows, g, t);
        w.clear();  // (and so not kept through what follows)
        if (!meet()) return;
        const int record = cut ? part_row(run, first_item ? 0 : 1) : tile.shared ? shared_row(tile.tok0, tile.kvh) : own_row(tile.tok0, tile.kvh);
        for (int i = tid; i < nrows * (D / 4); i += kTakerThreads) {
            const int row = i / (D / 4), c = i % (D / 4) * 4;
            const Gather sum = over_warps(row, c);
            if (direct) {
                deliver((size_t)(sa.tok_base + tile.tok0) * a.q_heads + tile.kvh * a.group + row, c, sum);
            } else {
                *reinterpret_cast<float4*>(sa.rec_o + (size_t)(record + row) * D + c) = sum.o;
                if (c == 0) sa.rec_ml[record + row] = make_float2(sum.m, sum.l);
            }
        }
        if (direct) continue;

        // Tickets: of each sequence that the item has rows of, this run's record is there; the last to come
        // joins that sequence's rows.
        if (tid == 0) last_of = 0;
        if (!meet()) return;
        if (tid < tile.ntok) {
            const int tok = tile.tok0 + tid;
            Parts p = {0, -1, 0, tile.c0, tile.c1, tile.s0};
            if (tile.shared) {
                p.sh0 = tile.c0, p.sh1 = tile.c1, p.sh_second = tile.s0;
                const unsigned int units = cum[tok + 1] - cum[tok], v0 = shared_all + cum[tok] * heads + tile.kvh * units;
                cuts.span(v0, v0 + units, p.own0, p.own1, p.own_second);
            } else if (sa.shared_tiles) {
                const unsigned int v0 = ((unsigned int)(tok / per) * heads + tile.kvh) * sa.shared_units;
                cuts.span(v0, v0 + sa.shared_units, p.sh0, p.sh1, p.sh_second);
            }
            const unsigned int count = (unsigned int)(p.own1 - p.own0 + 1 + p.sh1 - p.sh0 + 1);
            unsigned int* ticket = sa.tickets + (size_t)tok * heads + tile.kvh;
            // releases what all the CTA's threads wrote before they met, and acquires what the others released
            unsigned int before_me;
            asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before_me) : "l"(ticket) : "memory");
            if (before_me == count - 1u) {
                *ticket = 0u;
                parts_of[tid] = p;
                atomicOr(&last_of, 1u << tid);
            }
        }
        if (!meet()) return;
        const unsigned int mine = last_of;
        if (!mine) continue;  // (and the join rows were read before the meeting)
        // The rows of all those sequences at once: a row's records in `shares`, each a dozen (statistics and columns)
        // requested at a time; then the shares are joined.  Few rows: a warp per share, else all of a row's by one warp.
        // (The shares depend on the group alone: how many sequences come together here is a matter of timing, and must not
        // change the order of a sum.)
        const int rows = __popc(mine) * a.group, shares = a.group >= kTakers ? 1 : kTakers / a.group;
        const bool spread = shares > 1 && rows < kTakers;
        auto token_of = [&](int k) {  // of the k-th sequence to join
            unsigned int left = mine;
            for (; k > 0; k--) left &= left - 1;
            return __ffs(left) - 1;
        };
        constexpr int kDozen = 12;
        // (with 64 columns a row needs half a warp: two at a time)
        constexpr int kLanes = D / 4, kAtOnce = 32 / kLanes;
        const int half = kAtOnce > 1 ? lane / kLanes : 0, in_half = lane - half * kLanes, c = in_half * 4, jobs = spread ? rows * shares : rows;
        auto of_half = [&](auto x, int from) { return __shfl_sync(0xffffffffu, x, half * kLanes + from); };
#pragma unroll 1
        for (int j0 = warp * kAtOnce; j0 < jobs; j0 += kTakers * kAtOnce) {
            const int j = min(j0 + half, jobs - 1), row = spread ? j / shares : j, seq_of = row / a.group, in_head = row - seq_of * a.group;
            const int k = token_of(seq_of), tok = tile.tok0 + k;
            const Parts p = parts_of[k];
            const int ns = p.sh1 - p.sh0 + 1, n = ns + p.own1 - p.own0 + 1;
            const int part0 = spread ? j - row * shares : 0, parts = spread ? 1 : shares;
            Gather sum;
#pragma unroll 1
            for (int part = part0; part < part0 + parts; part++) {
                const int mine_n = (n - part + shares - 1) / shares, most_n = max(mine_n, __shfl_xor_sync(0xffffffffu, mine_n, 16));
                Gather share;
#pragma unroll 1
                for (int base = 0; base < most_n; base += kDozen) {
                    const int here = min(kDozen, mine_n - base);  // (0 or less: only the other half of the warp has any)
                    // lane y: record base + y of the share
                    const int x = min(part + (base + min(in_half, max(here, 1) - 1)) * shares, n - 1), y = x - ns;
                    int at;
                    if (x < ns) at = (ns == 1 ? shared_row(tok, tile.kvh) : part_row(p.sh0 + x, x ? 0 : p.sh_second)) + (tok - tok / per * per) * a.group;
                    else at = p.own0 == p.own1 ? own_row(tok, tile.kvh) : part_row(p.own0 + y, y ? 0 : p.own_second);
                    at += in_head;
                    float2 ml = __ldcg(&sa.rec_ml[at]);
                    float4 v[kDozen];
#pragma unroll
                    for (int i = 0; i < kDozen; i++) v[i] = __ldcg(reinterpret_cast<const float4*>(sa.rec_o + (size_t)of_half(at, i) * D + c));
                    if (in_half >= here) ml = make_float2(-INFINITY, 0.f);
                    float top = ml.x;
#pragma unroll
                    for (int d = 8; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                    top = of_half(top, 0);
                    const float f = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - top);
                    float l = ml.y * f;
#pragma unroll
                    for (int d = 8; d; d >>= 1) l += __shfl_xor_sync(0xffffffffu, l, d);
                    l = of_half(l, 0);
                    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int i = 0; i < kDozen; i++) {
                        const float fi = of_half(f, i);
                        if (i < here) {
                            o.x = fmaf(v[i].x, fi, o.x);
                            o.y = fmaf(v[i].y, fi, o.y);
                            o.z = fmaf(v[i].z, fi, o.z);
                            o.w = fmaf(v[i].w, fi, o.w);
                        }
                    }
                    if (here > 0) share.add(make_float2(top, l), o);
                }
                sum.add(make_float2(share.m, share.l), share.o);
            }
            if (j0 + half >= jobs) continue;
            if (spread) {
                *reinterpret_cast<float4*>(joins + (part0 * sa.item_rows + row) * S::kPitch + c) = sum.o;
                if (c == 0) join_mls[part0][row] = make_float2(sum.m, sum.l);
            } else {
                deliver((size_t)(sa.tok_base + tok) * a.q_heads + tile.kvh * a.group + in_head, c, sum);
            }
        }
        if (spread) {
            if (!meet()) return;
            for (int i = tid; i < rows * (D / 4); i += kTakerThreads) {
                const int row = i / (D / 4), c = i % (D / 4) * 4, tok = tile.tok0 + token_of(row / a.group);
                Gather sum;
                for (int x = 0; x < shares; x++)
                    sum.add(join_mls[x][row], *reinterpret_cast<const float4*>(joins + (x * sa.item_rows + row) * S::kPitch + c));
                deliver((size_t)(sa.tok_base + tok) * a.q_heads + tile.kvh * a.group + row % a.group, c, sum);
            }
        }
        // (these join rows, and parts_of, are written again only after another meeting, or by a direct item:)
        if (more && !meet()) return;
    }
}

// ---- host --------------------------------------------------------------------------------------

constexpr int kSmemMax = 227 * 1024, kSmemSm = 228 * 1024, kStaticMax = 2048;  // the kernel's own shared arrays: at most this

static int shared_tiles_of(const AttnArgs& a, int count) { return (count + 16 / a.group - 1) / (16 / a.group); }

template <typename T, int D, int kBlocks, bool kDup>
static int launch_rows_t(StreamArgs sa, const void* maps, cudaStream_t stream)
{
    using S = Stream<T, D>;
    static bool ready[64];
    const int dev = sa.a.device;
    if (dev < 0 || dev >= 64) return (int)cudaErrorInvalidDevice;
    cudaError_t e;
    sa.q_bytes = (sa.item_rows * D * (sa.a.io_bf16 ? 2 : 4) + 127) / 128 * 128;
    // Two CTAs per SM where that leaves each two stages or more, else one.
    const int fixed = kTakers * sa.item_rows * S::kPitch * 4 + (2 * sa.a.batch + 1) * 4 + 1024 +  // + alignment
                      (sizeof(T) == 4 && !kDup ? 2 * 8 * kBlocks * S::kPitch * 4 : 0);
    int ctas = 2, most = kSmemSm / 2 - 1024 - kStaticMax;
    if ((most - fixed) / (S::kStage + sa.q_bytes) < 2) {
        ctas = 1;
        most = kSmemMax - kStaticMax;
    }
    sa.stages = (most - fixed) / (S::kStage + sa.q_bytes);
    if (sa.stages > kMaxStages) sa.stages = kMaxStages;
    const int bytes = sa.stages * (S::kStage + sa.q_bytes) + fixed;
    if (!ready[dev]) {
        e = cudaFuncSetAttribute(pages_stream_kernel<T, D, kBlocks, kDup>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax - kStaticMax);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(pages_stream_kernel<T, D, kBlocks, kDup>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        if (e != cudaSuccess) return (int)e;
        ready[dev] = true;
    }
    return launch_after(pages_stream_kernel<T, D, kBlocks, kDup>, dim3(ctas * (kSms - sa.beside)), kStreamThreads, bytes, stream, *reinterpret_cast<const Maps*>(static_cast<const CUtensorMap*>(maps) + 2), sa);
}

template <typename T, int D>
static int launch_stream_t(StreamArgs sa, const void* maps, cudaStream_t stream)
{
    const int tokens = sa.shared_tiles ? min(sa.a.batch, 16 / sa.a.group) : 1;  // of an item, at most
    sa.item_rows = tokens * sa.a.group;
    if (sa.item_rows <= 4) return launch_rows_t<T, D, 1, true>(sa, maps, stream);
    if (sa.item_rows <= 8) return launch_rows_t<T, D, 1, false>(sa, maps, stream);
    return launch_rows_t<T, D, 2, false>(sa, maps, stream);
}

// Record rows of one launch for `count` sequences.
static size_t record_rows(const AttnArgs& a, int count, bool shared)
{
    return (size_t)2 * kStreamRuns * 16 + (shared ? (size_t)count * a.q_heads + (size_t)shared_tiles_of(a, count) * a.p.kv_heads * 16 : 0);
}

size_t stream_bytes(const AttnArgs& a, int count, bool shared)
{
    return record_rows(a, count, shared) * (a.p.head_dim * sizeof(float) + sizeof(float2));
}

int launch_stream(const AttnArgs& a, int layer, int first, int count, bool shared, int out_slot, int beside, int max_len, const void* maps, void* ws,
                  unsigned int* tickets, cudaStream_t stream)
{
    const int D = a.p.head_dim;
    StreamArgs sa = {};
    sa.a = a;
    sa.a.seqs = a.seqs + first;
    sa.a.batch = count;
    sa.layer = layer;
    sa.tok_base = first;
    const int rows = a.p.kv_dtype == TYB_BF16 ? 64 : 32;  // of a stage
    sa.shared_tiles = shared ? shared_tiles_of(a, count) : 0;
    sa.shared_units = shared ? kItemUnits + (a.prefix + rows - 1) / rows : 0;
    sa.out_slot = out_slot;
    sa.max_len = max_len;
    sa.beside = beside;
    sa.rec_o = static_cast<float*>(ws);
    sa.rec_ml = reinterpret_cast<float2*>(sa.rec_o + record_rows(a, count, shared) * D);
    sa.gave_up = tickets;
    sa.tickets = tickets + TYB_PAGES_TICKET_HEAD / sizeof(unsigned int);
    sa.wait_ns = tyb_wait_limit_of(a.device);
    if (a.p.kv_dtype == TYB_BF16)
        return D == 128 ? launch_stream_t<__nv_bfloat16, 128>(sa, maps, stream) : launch_stream_t<__nv_bfloat16, 64>(sa, maps, stream);
    return D == 128 ? launch_stream_t<float, 128>(sa, maps, stream) : launch_stream_t<float, 64>(sa, maps, stream);
}

}  // namespace tyb

// pages_attn.cu -- attention over the paged cache: which kernels a call runs on, and the join of split
// records.  Single tokens run on the streaming form (pages_stream.cu), prompt chunks on the tcgen05 form
// (BF16, pages_attn_tc.cu) or the row form (FP32, pages_rows.cu); a prefix that a batch shares runs on the
// tcgen05 form when the batch has enough rows for it, else inside the streaming form.
#define TYB_WHOLE_PROGRAM
#include "pages_mma.cuh"

#include <type_traits>

namespace tyb {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;

// Joins the split records of each output row: a warp per row, four records (statistics and values) requested at a time.
template <int D>
__global__ void __launch_bounds__(kThreads) pages_join_kernel(const AttnArgs a)
{
    const int lane = threadIdx.x & 31;
    const int R = (int)(blockIdx.x * kWarps + (threadIdx.x >> 5));
    after_predecessor();
    if (R >= a.rec.rows) return;
    constexpr int kPer = D / 32, kAtOnce = 4;
    using Values = typename std::conditional<kPer == 4, float4, float2>::type;
    float top = -INFINITY, acc[kPer] = {}, l = 0.f;
    for (int s0 = 0; s0 < a.rec.slots; s0 += kAtOnce) {
        float2 ml[kAtOnce];
        Values o[kAtOnce];
#pragma unroll
        for (int i = 0; i < kAtOnce; i++) {
            const size_t at = (size_t)min(s0 + i, a.rec.slots - 1) * a.rec.rows + R;
            ml[i] = a.rec.ml[at];
            o[i] = *reinterpret_cast<const Values*>(a.rec.o + at * D + lane * kPer);
        }
        const float before = top;
#pragma unroll
        for (int i = 0; i < kAtOnce; i++) {
            if (s0 + i >= a.rec.slots) ml[i] = make_float2(-INFINITY, 0.f);
            top = fmaxf(top, ml[i].x);
        }
        const float g = before == -INFINITY ? 0.f : fast_exp2(before - top);
        l *= g;
#pragma unroll
        for (int x = 0; x < kPer; x++) acc[x] *= g;
#pragma unroll
        for (int i = 0; i < kAtOnce; i++) {
            const float f = ml[i].x == -INFINITY ? 0.f : fast_exp2(ml[i].x - top);
            l = fmaf(ml[i].y, f, l);
            const float* v = reinterpret_cast<const float*>(&o[i]);
#pragma unroll
            for (int x = 0; x < kPer; x++) acc[x] = ml[i].x == -INFINITY ? acc[x] : fmaf(v[x], f, acc[x]);
            // (what lies in a record of nothing does not matter; in one that only weighs nothing, rows may not be finite)
        }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int i = 0; i < kPer; i += 2) {
        const size_t at = (size_t)R * D + lane * kPer + i;
        if (a.io_bf16) *reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(a.out) + at) = pack2(acc[i] * inv, acc[i + 1] * inv);
        else *reinterpret_cast<float2*>(static_cast<float*>(a.out) + at) = make_float2(acc[i] * inv, acc[i + 1] * inv);
    }
}

// ---- launches ----------------------------------------------------------------------------------

static int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

// How a call is laid out.
struct Layout {
    bool tokens;  // single tokens: the streaming form
    bool tiles;   // row tiles: prompt chunks, or a shared prefix on the tcgen05 form
    bool shared;  // the streaming form takes the shared prefix along
    bool tc, tall;
    int row_tiles, splits, slots;
    int beside;   // SMs of a shared pass that the own rows run beside; 0: after it
};

// Query rows of a KV head, and their product with the shared keys, from which a shared prefix runs on the tcgen05 form
// rather than in the streaming one.  With 2 rows a sequence and up to 50 own rows, streaming / tcgen05 in microseconds:
// 48 rows x 200 keys 20.5 / 23.5, 96 x 200 21.5 / 25.6; 16 x 1,024 20.1 / 17.4, 32 x 1,024 21.9 / 19.3, 96 x 1,024 28.2 /
// 20.0; 32 x 4,096 25.8 / 24.2, 96 x 4,096 38.9 / 24.8; 12 x 16,384 34.6 / 38.7, 32 x 16,384 42.1 / 42.2, 48 x 16,384 59.9 / 42.5.
// (The rule takes the shorter of the two everywhere but at 16 x 1,024.)
constexpr int kTcSharedRows = 32, kTcSharedWork = 24576;

// A shared pass on the tensor cores and the streaming of the sequences' own rows are bound by different things: they
// run at the same time where that is estimated to be shorter.  In microseconds: a split of the pass its tiles; the
// own rows (taken to be half of what max_len allows) what a CTA needs for a stage (an item's start and end take as
// long as kItemUnits of them), or what the memory can deliver; each of the two 10 for its start and end.  Of the splits
// tried, that picked the fastest or one within 1 % of it.  (The prices are those of heads of 128 with two rows a sequence;
// for others the split may not be the best.)  Measured, in turn / at the same time: 256 sequences behind 4,096
// shared rows with up to 512 own ones 94 / 72, with up to 64 own ones 55 / 41, behind 1,024 85 / 68; 64 behind 4,096
// 61 / 35; 512 behind 2,048 with up to 128 91 / 77; 128 behind 4,096 with up to 1,500 110 / 82.
static void share_sms(const tyb_pages_attn* c, int tiles, int ctas, Layout* l)
{
    const double tile_us = l->tall ? 0.7 : 1.0, unit_us = 1.0, fixed_us = 10.0, memory = 6.4e6;
    const double rows = 0.5 * (c->max_len - c->prefix), items = (double)c->batch * c->p.kv_heads;
    const double bytes = rows * items * c->p.head_dim * 4.0, units = items * (kItemUnits + 0.5 + rows / 64);  // K and V in BF16
    auto pass_us = [&](int splits) { return fixed_us + (tiles + splits - 1) / splits * tile_us; };
    auto own_us = [&](int sms) {
        const double busy = units / (2 * sms) * unit_us, read = bytes / memory;
        return fixed_us + (busy > read ? busy : read);
    };
    double best = pass_us(l->splits) + own_us(kSms);
    for (int s = 1; s <= tiles / 4 && s * ctas <= kSms / 2; s++) {
        const double us = pass_us(s) > own_us(kSms - s * ctas) ? pass_us(s) : own_us(kSms - s * ctas);
        if (us < best) {
            best = us;
            l->splits = s;
            l->beside = (s * ctas + 1) / 2 * 2;
        }
    }
}

static Layout layout_of(const tyb_pages_attn* c)
{
    Layout l = {};
    const bool bf16 = c->p.kv_dtype == TYB_BF16;
    const int group = c->q_heads / c->p.kv_heads;
    l.tokens = c->max_new == 1 && c->rows == c->batch;
    const bool prefix = l.tokens && c->prefix > 0;
    const long long shared_rows = (long long)c->batch * group;
    l.tiles = !l.tokens || (prefix && bf16 && shared_rows >= kTcSharedRows && shared_rows * c->prefix >= kTcSharedWork);
    l.shared = prefix && !l.tiles;
    if (!l.tiles) return l;
    l.tc = bf16;
    l.tall = l.tc && (long long)(l.tokens ? c->batch : c->max_new) * group <= kTcTall;
    const int per = (l.tall ? kTcTall : l.tc ? kTcWide : kRowsTile) / group;
    // Each of the sequences of a call ends in a tile of its own; no list has more tiles than this.
    l.row_tiles = l.tokens ? ceil_div(c->batch, per) : (int)((c->rows + (long long)c->batch * (per - 1)) / per);
    const long long in_view = c->window ? (long long)c->window + c->sinks : c->max_len;
    const long long keys = l.tokens ? c->prefix : in_view < c->max_len ? in_view : c->max_len;
    const int tiles = ceil_div(keys, l.tc ? 64 : 32);
    const long long ctas = (long long)l.row_tiles * c->p.kv_heads;
    if (l.tc) {
        l.splits = (int)(kSms / ctas);  // one CTA fits an SM; a split has at least four tiles
        if (l.splits > tiles / 4) l.splits = tiles / 4;
    } else {
        // Splits for twice as many CTAs as fit, each of at least 64 keys.  As many as fit, twice, three times as many: 3 chunks of
        // 37 .. 733 tokens through 301, heads of 64, 42, 44, 44 us; with heads of 128 80, 68, 75; 12 of up to 300 through 1,200,
        // heads of 64, 204, 141, 131; one of 400 with 32 heads of 128 on 4 71, 72, 77.
        l.splits = (int)(2 * rows_ctas(c->p.head_dim) * kSms / ctas);
        if (l.splits > tiles / 2) l.splits = tiles / 2;
    }
    if (l.splits < 1) l.splits = 1;
    if (l.tokens) share_sms(c, tiles, (int)ctas, &l);
    l.slots = l.splits * (l.tall ? 2 : 1) + l.tokens;  // the last one of a shared pass's call: the own rows
    return l;
}

static AttnArgs args_of(const tyb_pages_attn* c, const Layout& l)
{
    AttnArgs a = {};
    a.p = c->p;
    a.q = c->q;
    a.q_stride = c->q_stride;
    a.out = c->out;
    a.io_bf16 = c->io_bf16;
    a.q_heads = c->q_heads;
    a.group = c->q_heads / c->p.kv_heads;
    a.seqs = c->seqs;
    a.starts = c->starts;
    a.batch = c->batch;
    a.rows = c->rows;
    a.prefix = c->prefix;
    a.window = c->window;
    a.sinks = c->window ? c->sinks : 0;
    a.scale_log2 = c->scale * kLog2e;
    a.splits = l.splits;
    a.rec.rows = c->rows * c->q_heads;
    a.rec.slots = l.slots;
    return a;
}

static bool records(const Layout& l) { return l.slots > 1; }
static size_t record_bytes(const AttnArgs& a, const Layout& l)
{
    return records(l) ? (size_t)l.slots * a.rec.rows * (a.p.head_dim * sizeof(float) + sizeof(float2)) : 0;
}

}  // namespace tyb

using namespace tyb;

extern "C" size_t tyb_pages_ticket_bytes(const KVPages* p) { return TYB_PAGES_TICKET_HEAD + (size_t)kStreamSeqs * p->kv_heads * sizeof(unsigned int); }

extern "C" size_t tyb_pages_attn_bytes(const tyb_pages_attn* c, int* uses_tickets)
{
    const Layout l = layout_of(c);
    const AttnArgs a = args_of(c, l);
    const int count = c->batch < kStreamSeqs ? c->batch : kStreamSeqs;
    *uses_tickets = l.tokens;
    return (record_bytes(a, l) + 255) / 256 * 256 + (l.tokens ? stream_bytes(a, count, l.shared) : 0);
}

extern "C" int tyb_pages_attn_launch(const tyb_pages_attn* c, void* ws, void* tickets, void* stream)
{
    cudaStream_t st = (cudaStream_t)stream;
    const Layout l = layout_of(c);
    AttnArgs a = args_of(c, l);
    a.st.word = c->env.status;
    a.st.mirror = c->env.mirror;
    a.device = c->env.device;
    const int D = a.p.head_dim;
    if (records(l)) {
        a.rec.o = static_cast<float*>(ws);
        a.rec.ml = reinterpret_cast<float2*>(a.rec.o + (size_t)l.slots * a.rec.rows * D);
    }
    void* more = static_cast<char*>(ws) + (record_bytes(a, l) + 255) / 256 * 256;
    if (l.tiles) {
        const int e = l.tc ? tc_launch(a, c->layer, l.tall, l.tokens, l.beside > 0, l.row_tiles, c->maps, st)
                           : rows_launch(a, c->layer, l.row_tiles, c->maps, st);
        if (e) return e;
    }
    if (l.tokens) {
        for (int first = 0; first < c->batch; first += kStreamSeqs) {
            const int count = c->batch - first < kStreamSeqs ? c->batch - first : kStreamSeqs;
            const int e = launch_stream(a, c->layer, first, count, l.shared, l.tiles ? l.slots - 1 : -1, first ? 0 : l.beside, c->max_len, c->maps, more,
                                        static_cast<unsigned int*>(tickets), st);
            if (e) return e;
        }
    }
    if (records(l)) {
        const int grid = ceil_div(a.rec.rows, kWarps);
        return launch_after(D == 128 ? pages_join_kernel<128> : pages_join_kernel<64>, dim3(grid), kThreads, 0, st, a);
    }
    return 0;
}

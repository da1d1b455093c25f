// pages_attn.cu -- attention over the paged cache by warps that read keys and values straight into
// tensor-core fragments: single tokens of a sequence (whole, or behind a shared prefix, or through a
// window with sinks), and the general form for up to 64 query rows per CTA.
//
// One warp holds 16 query rows (q_heads / kv_heads heads of one token, or several tokens) and walks
// key tiles of 16 rows (BF16) or 8 rows (FP32) with the running maximum and sum of an online softmax
// in base 2.  Nothing passes through shared memory on the way in: the contraction over the head
// dimension may run in any order as long as Q and K agree, so lane (g, t) of a fragment takes 16
// consecutive bytes of key row g instead of four scattered words, and the value rows' columns are
// likewise dealt out 16 bytes per lane; each 16-byte access then carries whole sectors.  The next
// tile's K is requested as soon as this tile's scores are formed, its V as soon as P.V is.
//   BF16: mma.sync m16n8k16; P as a BF16 pair (value and remainder), so that the only roundings are
//         the operands' own and the output's.  The step is memory-bound: the second P.V is free.
//   FP32: mma.sync m16n8k8 on TF32 halves, x = hi + lo, hi.hi + hi.lo + lo.hi: relative error about
//         2^-21 per product, FP32 sums.
// Decode is bound by memory (each K and V element is used by q_heads / kv_heads rows once), so what
// matters is bytes in flight: four warps a CTA, each with one tile of K and of V (8 KB) requested.
#define TYB_WHOLE_PROGRAM
#include "pages_mma.cuh"

namespace tyb {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;

__device__ __forceinline__ uint4 ldg16(const void* p)
{
    uint4 v;
    asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// Where key row `tile * KT` lies, as an element offset into the layer's pages of KV head h; -1 when the
// page is not there.
__device__ __forceinline__ int tile_page(const KVPages& p, const int* table, int tile, int kt, const Status& st)
{
    const int page = table[(tile * kt) >> page_shift(p.page_size)];
    if (page >= p.num_pages) {
        raise(st, TYB_STATUS_BAD_ARGUMENT);
        return -1;
    }
    return page;
}

// What one warp's 16 rows have gathered: O fragments, and per lane the statistics of rows g and g + 8.
template <typename T, int D>
struct Warp {
    static constexpr int kVec = 16 / (int)sizeof(T);     // elements of a 16-byte access
    static constexpr int kTile = sizeof(T) == 2 ? 16 : 8;  // keys of a tile
    static constexpr int kKeysK = kTile / 8;             // key rows per lane of K
    static constexpr int kKeysV = kTile / 4;             // and of V
    static constexpr int kChunkK = D / (4 * kVec);       // 16-byte chunks of a K row per lane
    static constexpr int kChunkV = D / (8 * kVec);       // and of a V row
    static constexpr int kOut = D / 8;                   // 8-column fragments of O
    float o[kOut][4];
    float m[2], l[2];
    uint4 k[kKeysK][kChunkK];
    uint4 v[kKeysV][kChunkV];

    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int i = 0; i < kOut; i++) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
    }

    // Column of O fragment i, register r (0 or 1; 2 and 3 are the same columns of row g + 8).
    static __device__ __forceinline__ int column(int i, int r, int t)
    {
        return (i / kVec) * 8 * kVec + kVec * (2 * t + r) + i % kVec;
    }
    // Key (within the tile) of V row e of lane t: the rows that meet its P columns.
    static __device__ __forceinline__ int v_key(int e, int t) { return kTile == 16 ? 2 * t + (e & 1) + 8 * (e >> 1) : 2 * t + e; }

    __device__ __forceinline__ void load_k(const T* rows, int g, int t)
    {
#pragma unroll
        for (int e = 0; e < kKeysK; e++)
#pragma unroll
            for (int j = 0; j < kChunkK; j++) k[e][j] = ldg16(rows + (size_t)(8 * e + g) * D + (4 * j + t) * kVec);
    }
    __device__ __forceinline__ void load_v(const T* rows, int g, int t)
    {
#pragma unroll
        for (int e = 0; e < kKeysV; e++)
#pragma unroll
            for (int j = 0; j < kChunkV; j++) v[e][j] = ldg16(rows + (size_t)v_key(e, t) * D + (8 * j + g) * kVec);
    }
    __device__ __forceinline__ void none_k()
    {
#pragma unroll
        for (int e = 0; e < kKeysK; e++)
#pragma unroll
            for (int j = 0; j < kChunkK; j++) k[e][j] = make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void none_v(int e)
    {
#pragma unroll
        for (int j = 0; j < kChunkV; j++) v[e][j] = make_uint4(0, 0, 0, 0);
    }
};

// The query fragments of a warp.  BF16: in registers.  FP32: the rows stay in shared memory
// (kPitch floats apart: conflict-free 16-byte reads) and are split as they are used.
template <typename T, int D>
struct Query;

template <int D>
struct Query<float, D> {
    static constexpr int kPitch = D + 16;
    static constexpr int kSharedFloats = 16 * kPitch;
    const float* rows;
    __device__ __forceinline__ void load(const void* row0, const void* row1, bool bf16, int t, float* shared, int g)
    {
        rows = shared;
        for (int j = 0; j < D / 32; j++)
            for (int r = 0; r < 2; r++) {
                const void* row = r ? row1 : row0;
                float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                const int at = (4 * j + t) * 8;
                if (row && bf16) load8(static_cast<const __nv_bfloat16*>(row) + at, x);
                else if (row) load8(static_cast<const float*>(row) + at, x);
                store8(shared + (g + 8 * r) * kPitch + at, x);
            }
        __syncwarp();
    }
    __device__ __forceinline__ void scores(const Warp<float, D>& w, float (&s)[1][4], int g, int t) const
    {
        // hi.hi and the two cross terms in accumulators of their own: shorter chains, and the small
        // terms are not rounded away one by one.
        float c[2][4] = {};
#pragma unroll
        for (int j = 0; j < D / 16; j++) {
            const float4 q0 = *reinterpret_cast<const float4*>(rows + g * kPitch + (4 * j + t) * 4);
            const float4 q1 = *reinterpret_cast<const float4*>(rows + (g + 8) * kPitch + (4 * j + t) * 4);
            const float* kf = reinterpret_cast<const float*>(&w.k[0][j]);
#pragma unroll
            for (int u = 0; u < 2; u++) {
                uint32_t ah[4], al[4], bh[2], bl[2];
                split_tf32(u ? q0.z : q0.x, ah[0], al[0]);
                split_tf32(u ? q1.z : q1.x, ah[1], al[1]);
                split_tf32(u ? q0.w : q0.y, ah[2], al[2]);
                split_tf32(u ? q1.w : q1.y, ah[3], al[3]);
                split_tf32(kf[2 * u], bh[0], bl[0]);
                split_tf32(kf[2 * u + 1], bh[1], bl[1]);
                mma_tf32(c[1], al, bh[0], bh[1]);
                mma_tf32(c[1], ah, bl[0], bl[1]);
                mma_tf32(c[0], ah, bh[0], bh[1]);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; i++) s[0][i] = c[0][i] + c[1][i];
    }
};

// O += P . V for the tile; P in the score layout.
template <int D>
__device__ __forceinline__ void accumulate(Warp<float, D>& w, const float (&p)[1][4])
{
    // columns k = t and t + 4 of the P operand are keys 2t and 2t + 1
    uint32_t ph[4], pl[4];
    split_tf32(p[0][0], ph[0], pl[0]);
    split_tf32(p[0][2], ph[1], pl[1]);
    split_tf32(p[0][1], ph[2], pl[2]);
    split_tf32(p[0][3], ph[3], pl[3]);
    const float(&v)[2][Warp<float, D>::kChunkV][4] = reinterpret_cast<const float(&)[2][Warp<float, D>::kChunkV][4]>(w.v);
#pragma unroll
    for (int j = 0; j < Warp<float, D>::kChunkV; j++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t bh[2], bl[2];
            split_tf32(v[0][j][i], bh[0], bl[0]);
            split_tf32(v[1][j][i], bh[1], bl[1]);
            // The tile's contribution in an accumulator of its own, joined by an FP32 addition: the
            // tensor core's own sums round towards zero, which over thousands of keys would add up.
            float c[4] = {};
            mma_tf32(c, pl, bh[0], bh[1]);
            mma_tf32(c, ph, bl[0], bl[1]);
            mma_tf32(c, ph, bh[0], bh[1]);
#pragma unroll
            for (int r = 0; r < 4; r++) w.o[4 * j + i][r] += c[r];
        }
}

// What the rows of a warp (or CTA) can see, and where the keys are.
struct View {
    const int* table;
    int kvh;
    int pos[2], lo[2];                     // of rows g and g + 8
    int pos_min, pos_max, lo_min, lo_max;  // over the rows that share the tiles (those that are there)
    int sinks;
};

// Tiles first, first + step, .. of `tiles` below `end`.
template <typename T, int D>
__device__ __forceinline__ void walk(Warp<T, D>& w, const Query<T, D>& q, const AttnArgs& a, const View& view, const Tiles& tiles,
                                     int first, int end, int step, int g, int t, int lane)
{
    using W = Warp<T, D>;
    constexpr int kTile = W::kTile;
    const size_t head = (size_t)view.kvh * a.p.page_size * D, page_elems = (size_t)a.p.kv_heads * a.p.page_size * D;
    const T* kb = static_cast<const T*>(a.k) + head;
    const T* vb = static_cast<const T*>(a.v) + head;
    const int in_page = a.p.page_size - 1;
    int pages = -1;  // lane l: page of the walk's tile 32 x + l
    const int n = end > first ? (end - first + step - 1) / step : 0;
    auto page_at = [&](int i) {
        if ((i & 31) == 0 && i < n) {
            const int mine = first + (i + lane) * step;
            pages = mine < end ? tile_page(a.p, view.table, tiles.at(mine), kTile, a.st) : -1;
        }
        return i < n ? __shfl_sync(0xffffffffu, pages, i & 31) : -1;
    };
    auto offset = [&](int page, int tile) { return (size_t)page * page_elems + (size_t)((tile * kTile) & in_page) * D; };

    int page = page_at(0), tile = n ? tiles.at(first) : 0;
    if (page >= 0) {
        w.load_k(kb + offset(page, tile), g, t);
        w.load_v(vb + offset(page, tile), g, t);
    }
    for (int i = 0; i < n; i++) {
        const int j0 = tile * kTile;
        const bool there = page >= 0;
        // A tile wholly seen by every row needs no mask; else each score is tested, and value rows that no
        // row of the call's tile set sees are cleared (what lies there may be anything, NaN included).
        const bool whole = there && j0 + kTile - 1 <= view.pos_min && (j0 >= view.lo_max || j0 + kTile <= view.sinks);
        float s[W::kKeysK][4];
        if (there) q.scores(w, s, g, t);
        const int next_page = page_at(i + 1);
        const int next_tile = i + 1 < n ? tiles.at(first + (i + 1) * step) : 0;
        const bool visible = there;
        if (next_page >= 0) w.load_k(kb + offset(next_page, next_tile), g, t);
        if (visible) {
            if (!whole) {
#pragma unroll
                for (int e = 0; e < W::kKeysK; e++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const int j = j0 + 8 * e + 2 * t + (r & 1), row = r >> 1;
                        if (j > view.pos[row] || (j < view.lo[row] && j >= view.sinks)) s[e][r] = -INFINITY;
                    }
#pragma unroll
                for (int e = 0; e < W::kKeysV; e++) {
                    const int j = j0 + W::v_key(e, t);
                    if (j > view.pos_max || (j < view.lo_min && j >= view.sinks)) w.none_v(e);
                }
            }
            float top[2];
#pragma unroll
            for (int r = 0; r < 2; r++) {
                top[r] = fmaxf(s[0][2 * r], s[0][2 * r + 1]);
#pragma unroll
                for (int e = 1; e < W::kKeysK; e++) top[r] = fmaxf(top[r], fmaxf(s[e][2 * r], s[e][2 * r + 1]));
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
                top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
                top[r] = fmaxf(w.m[r], top[r] * a.scale_log2);
            }
            if (__any_sync(0xffffffffu, top[0] > w.m[0] || top[1] > w.m[1])) {
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    const float f = w.m[r] == -INFINITY ? 0.f : fast_exp2(w.m[r] - top[r]);
                    w.l[r] *= f;
                    w.m[r] = top[r];
#pragma unroll
                    for (int c = 0; c < W::kOut; c++) {
                        w.o[c][2 * r] *= f;
                        w.o[c][2 * r + 1] *= f;
                    }
                }
            }
            const float neg[2] = {w.m[0] == -INFINITY ? 0.f : -w.m[0], w.m[1] == -INFINITY ? 0.f : -w.m[1]};
#pragma unroll
            for (int e = 0; e < W::kKeysK; e++)
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    s[e][r] = fast_exp2(fmaf(s[e][r], a.scale_log2, neg[r >> 1]));
                    w.l[r >> 1] += s[e][r];
                }
            accumulate(w, s);
        }
        if (next_page >= 0) w.load_v(vb + offset(next_page, next_tile), g, t);
        page = next_page;
        tile = next_tile;
    }
    // the row sums of the four lanes of a row
#pragma unroll
    for (int r = 0; r < 2; r++) {
        w.l[r] += __shfl_xor_sync(0xffffffffu, w.l[r], 1);
        w.l[r] += __shfl_xor_sync(0xffffffffu, w.l[r], 2);
    }
}

// Four values of output row R, columns c .. c + 3: the finished output, or split record `slot`.
__device__ __forceinline__ void put4(const AttnArgs& a, int D, int slot, size_t R, int c, float4 x, float l)
{
    if (a.rec.slots == 1) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        x.x *= inv; x.y *= inv; x.z *= inv; x.w *= inv;
        if (a.io_bf16)
            *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + R * D + c) = make_uint2(pack2(x.x, x.y), pack2(x.z, x.w));
        else
            *reinterpret_cast<float4*>(static_cast<float*>(a.out) + R * D + c) = x;
    } else {
        *reinterpret_cast<float4*>(a.rec.o + ((size_t)slot * a.rec.rows + R) * D + c) = x;
    }
}

// Rows of a CTA tile: `per` tokens x `group` heads, token-major.  The prefix pass takes the batch's
// single tokens as its rows.
constexpr int kRowsCta = 16 * kWarps;

// CTA (row tile, KV head, split): each warp has 16 rows of its own and walks all the split's tiles.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) pages_rows_kernel(const AttnArgs a)
{
    using W = Warp<T, D>;
    extern __shared__ float4 shared4[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int kvh = blockIdx.y, split = blockIdx.z;
    const int per = kRowsCta / a.group;
    int seq = 0, tok0, ntok, pos0;  // first token (row of q) of the tile, tokens, position of the first
    after_predecessor();
    __shared__ int found[4];
    {
        // which sequence's tile this is: a warp scans the sequences' tile counts
        if (warp == 0) {
            int before = 0;
            if (lane == 0) found[0] = -1;
            __syncwarp();
            for (int base = 0; base < a.batch; base += 32) {
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
                if ((int)blockIdx.x >= lo && (int)blockIdx.x < lo + cnt) {
                    const int i = (int)blockIdx.x - lo;
                    if (q0 < 0 || q1 > a.rows) {
                        raise(a.st, TYB_STATUS_BAD_ARGUMENT);
                    } else {
                        found[0] = b;
                        found[1] = q0 + i * per;
                        found[2] = min(per, q1 - q0 - i * per);
                        found[3] = i * per - (q1 - q0);
                    }
                }
                before += __shfl_sync(0xffffffffu, sum, 31);
                if (before > (int)blockIdx.x) break;
            }
        }
        __syncthreads();
        if (found[0] < 0) return;
        seq = a.seqs[found[0]];
        tok0 = found[1];
        ntok = found[2];
        pos0 = checked_len(a.p, seq, a.st) + found[3];
        if (pos0 < 0 && threadIdx.x == 0) raise(a.st, TYB_STATUS_BAD_ARGUMENT);  // more queries than tokens
    }
    View view;
    view.table = a.p.table + (size_t)(seq < 0 || seq >= a.p.max_seqs ? 0 : seq) * a.p.max_pages;
    view.kvh = kvh;
    view.sinks = a.sinks;
    auto lo_of_pos = [&](int pos) { return a.window ? max(0, pos - a.window + 1) : 0; };
    view.pos_min = pos0;
    view.pos_max = pos0 + ntok - 1;
    view.lo_min = lo_of_pos(view.pos_min);
    view.lo_max = lo_of_pos(view.pos_max);
    const char* qrow[2];
    size_t R[2];
    bool here[2];
    const size_t esize = a.io_bf16 ? 2 : 4;
#pragma unroll
    for (int r = 0; r < 2; r++) {
        const int row = 16 * warp + g + 8 * r, tk = row / a.group, hh = row - tk * a.group;
        here[r] = tk < ntok;
        view.pos[r] = here[r] ? pos0 + tk : -1;
        view.lo[r] = lo_of_pos(view.pos[r]);
        qrow[r] = here[r] ? static_cast<const char*>(a.q) + ((size_t)(tok0 + tk) * a.q_stride + (size_t)(kvh * a.group + hh) * D) * esize : nullptr;
        R[r] = (size_t)(tok0 + tk) * a.q_heads + kvh * a.group + hh;
    }
    const Tiles tiles = tiles_of(view.pos_max, view.lo_min, view.sinks, W::kTile);
    const int n = tiles.count();
    const int first = (int)((long long)n * split / a.splits), end = (int)((long long)n * (split + 1) / a.splits);
    Query<T, D> q;
    float* shared = reinterpret_cast<float*>(shared4);
    q.load(qrow[0], qrow[1], a.io_bf16, t, shared + warp * Query<T, D>::kSharedFloats, g);
    W w;
    w.clear();
    walk(w, q, a, view, tiles, first, end, 1, g, t, lane);
    // The warp's rows through its part of shared memory, then out in whole rows.
    constexpr int kPitch = D + 4;
    static_assert(Query<float, D>::kSharedFloats >= 16 * kPitch, "the query rows' room holds the output rows");
    float* so = shared + warp * Query<float, D>::kSharedFloats;
    __syncwarp();
#pragma unroll
    for (int r = 0; r < 2; r++)
#pragma unroll
        for (int c = 0; c < W::kOut; c++) {
            so[(g + 8 * r) * kPitch + W::column(c, 0, t)] = w.o[c][2 * r];
            so[(g + 8 * r) * kPitch + W::column(c, 1, t)] = w.o[c][2 * r + 1];
        }
    __syncwarp();
#pragma unroll
    for (int r = 0; r < 2; r++) {
        if (!here[r]) continue;
        for (int c = 4 * t; c < D; c += 16)
            put4(a, D, a.slot0 + split, R[r], c, *reinterpret_cast<const float4*>(so + (g + 8 * r) * kPitch + c), w.l[r]);
        if (a.rec.slots > 1 && t == 0) a.rec.ml[(size_t)(a.slot0 + split) * a.rec.rows + R[r]] = make_float2(w.m[r], w.l[r]);
    }
}

// Joins the split records of each output row: a warp per row.
template <int D>
__global__ void __launch_bounds__(kThreads) pages_join_kernel(const AttnArgs a)
{
    const int lane = threadIdx.x & 31;
    const int R = (int)(blockIdx.x * kWarps + (threadIdx.x >> 5));
    after_predecessor();
    if (R >= a.rec.rows) return;
    constexpr int kPer = D / 32;
    float top = -INFINITY;
    for (int s = lane; s < a.rec.slots; s += 32) top = fmaxf(top, a.rec.ml[(size_t)s * a.rec.rows + R].x);
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float acc[kPer] = {}, l = 0.f;
#pragma unroll 4
    for (int s = 0; s < a.rec.slots; s++) {
        const float2 ml = a.rec.ml[(size_t)s * a.rec.rows + R];
        const float f = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - top);
        l = fmaf(ml.y, f, l);
        const float* o = a.rec.o + ((size_t)s * a.rec.rows + R) * D + lane * kPer;
        if (f != 0.f) {
#pragma unroll
            for (int i = 0; i < kPer; i++) acc[i] = fmaf(o[i], f, acc[i]);
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
};

// Query rows of a KV head from which the shared prefix runs on the tcgen05 form.
constexpr int kTcSharedRows = 65;

static Layout layout_of(const tyb_pages_attn* c)
{
    Layout l = {};
    const bool bf16 = c->p.kv_dtype == TYB_BF16;
    const int group = c->q_heads / c->p.kv_heads;
    l.tokens = c->max_new == 1 && c->rows == c->batch;
    const bool prefix = l.tokens && c->prefix > 0;
    l.tiles = !l.tokens || (prefix && bf16 && (long long)c->batch * group >= kTcSharedRows);
    l.shared = prefix && !l.tiles;
    if (!l.tiles) return l;
    l.tc = bf16;
    l.tall = l.tc && (long long)(l.tokens ? c->batch : c->max_new) * group <= kTcTall;
    const int per = (l.tall ? kTcTall : l.tc ? kTcWide : kRowsCta) / group;
    // Each of the sequences of a call ends in a tile of its own; no list has more tiles than this.
    l.row_tiles = l.tokens ? ceil_div(c->batch, per) : (int)((c->rows + (long long)c->batch * (per - 1)) / per);
    const long long keys = l.tokens ? c->prefix : c->window && c->window < c->max_len ? c->window + c->sinks : c->max_len;
    const int tiles = ceil_div(keys, l.tc ? 64 : 8);
    const long long ctas = (long long)l.row_tiles * c->p.kv_heads;
    if (l.tc) {
        l.splits = (int)(kSms / ctas);  // one CTA fits an SM; a split has at least four tiles
        if (l.splits > tiles / 4) l.splits = tiles / 4;
    } else {
        l.splits = ceil_div(3LL * kSms, ctas);
        if (l.splits > ceil_div(tiles, 8)) l.splits = ceil_div(tiles, 8);
    }
    if (l.splits < 1) l.splits = 1;
    l.slots = l.splits * (l.tall ? 2 : 1) + l.tokens;  // the last one of a shared pass's call: the own rows
    return l;
}

static AttnArgs args_of(const tyb_pages_attn* c, const Layout& l)
{
    AttnArgs a = {};
    a.p = c->p;
    const size_t layer = (size_t)c->layer * c->p.num_pages * c->p.kv_heads * c->p.page_size * c->p.head_dim *
                         (c->p.kv_dtype == TYB_BF16 ? 2 : 4);
    a.k = static_cast<const char*>(c->p.k) + layer;
    a.v = static_cast<const char*>(c->p.v) + layer;
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

template <int D>
static int launch_rows(const AttnArgs& a, int row_tiles, cudaStream_t stream)
{
    static bool ready[64];
    const int dev = a.device;
    if (dev < 0 || dev >= 64) return (int)cudaErrorInvalidDevice;
    cudaError_t e;
    const size_t rows = kWarps * (size_t)Query<float, D>::kSharedFloats * sizeof(float);
    if (!ready[dev]) {
        e = cudaFuncSetAttribute(pages_rows_kernel<float, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)rows);
        if (e != cudaSuccess) return (int)e;
        ready[dev] = true;
    }
    return launch_after(pages_rows_kernel<float, D>, dim3(row_tiles, a.p.kv_heads, a.splits), kThreads, rows, stream, a);
}

}  // namespace tyb

using namespace tyb;

extern "C" void tyb_pages_attn_bytes(const tyb_pages_attn* c, size_t* ws, size_t* tickets)
{
    const Layout l = layout_of(c);
    const AttnArgs a = args_of(c, l);
    const int count = c->batch < kStreamSeqs ? c->batch : kStreamSeqs;
    *ws = (record_bytes(a, l) + 255) / 256 * 256 + (l.tokens ? stream_bytes(a, count, l.shared) : 0);
    *tickets = l.tokens ? (size_t)count * c->p.kv_heads * sizeof(unsigned int) : 0;
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
        const int e = l.tc ? tc_launch(a, c->layer, l.tall, l.tokens, l.row_tiles, c->maps, st)
                           : D == 128 ? launch_rows<128>(a, l.row_tiles, st) : launch_rows<64>(a, l.row_tiles, st);
        if (e) return e;
    }
    if (l.tokens) {
        for (int first = 0; first < c->batch; first += kStreamSeqs) {
            const int count = c->batch - first < kStreamSeqs ? c->batch - first : kStreamSeqs;
            const int e = launch_stream(a, c->layer, first, count, l.shared, l.tiles ? l.slots - 1 : -1, c->max_len, c->maps, more,
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

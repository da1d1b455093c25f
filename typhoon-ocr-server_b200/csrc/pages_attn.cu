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
#include "pages_attn.cuh"

namespace tyb {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;

__device__ __forceinline__ uint4 ldg16(const void* p)
{
    uint4 v;
    asm("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ float lo_of(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float hi_of(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x = hi + lo in TF32, the remainder below 2^-22 |x|.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo)
{
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(x - __uint_as_float(hi)));
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
struct Query<__nv_bfloat16, D> {
    static constexpr int kSharedFloats = 0;
    uint32_t a[D / 16][4];
    // Row r of the warp at q[r] (NULL: absent, zeros), FP32 or BF16.
    __device__ __forceinline__ void load(const void* row0, const void* row1, bool bf16, int t, float*, int)
    {
#pragma unroll
        for (int j = 0; j < D / 32; j++)
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const void* row = r ? row1 : row0;
                float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
                const int at = (4 * j + t) * 8;
                if (row && bf16) load8(static_cast<const __nv_bfloat16*>(row) + at, x);
                else if (row) load8(static_cast<const float*>(row) + at, x);
                a[2 * j][r] = pack2(x[0], x[1]);
                a[2 * j][2 + r] = pack2(x[2], x[3]);
                a[2 * j + 1][r] = pack2(x[4], x[5]);
                a[2 * j + 1][2 + r] = pack2(x[6], x[7]);
            }
    }
    // Scores of the 16 rows against the tile: s[e] keys 8e .. 8e + 8 (rows g, g + 8; keys 2t, 2t + 1).
    __device__ __forceinline__ void scores(const Warp<__nv_bfloat16, D>& w, float (&s)[2][4], int, int) const
    {
#pragma unroll
        for (int e = 0; e < 2; e++) {
            s[e][0] = s[e][1] = s[e][2] = s[e][3] = 0.f;
#pragma unroll
            for (int j = 0; j < D / 32; j++) {
                mma_bf16(s[e], a[2 * j][0], a[2 * j][1], a[2 * j][2], a[2 * j][3], w.k[e][j].x, w.k[e][j].y);
                mma_bf16(s[e], a[2 * j + 1][0], a[2 * j + 1][1], a[2 * j + 1][2], a[2 * j + 1][3], w.k[e][j].z, w.k[e][j].w);
            }
        }
    }
};

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
__device__ __forceinline__ void accumulate(Warp<__nv_bfloat16, D>& w, const float (&p)[2][4])
{
    uint32_t h[4], r[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const float x = p[i >> 1][2 * (i & 1)], y = p[i >> 1][2 * (i & 1) + 1];
        h[i] = pack2(x, y);
        r[i] = pack2(x - lo_of(h[i]), y - hi_of(h[i]));
    }
    const uint32_t(&v)[4][Warp<__nv_bfloat16, D>::kChunkV][4] =
        reinterpret_cast<const uint32_t(&)[4][Warp<__nv_bfloat16, D>::kChunkV][4]>(w.v);
#pragma unroll
    for (int j = 0; j < Warp<__nv_bfloat16, D>::kChunkV; j++)
#pragma unroll
        for (int i = 0; i < 8; i++) {
            // element i of the chunk of two key rows as a pair
            const uint32_t sel = i & 1 ? 0x7632 : 0x5410;
            const uint32_t b0 = __byte_perm(v[0][j][i / 2], v[1][j][i / 2], sel);
            const uint32_t b1 = __byte_perm(v[2][j][i / 2], v[3][j][i / 2], sel);
            mma_bf16(w.o[8 * j + i], h[0], h[1], h[2], h[3], b0, b1);
            mma_bf16(w.o[8 * j + i], r[0], r[1], r[2], r[3], b0, b1);
        }
}

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

template <typename T, int D>
constexpr size_t solo_shared_floats()
{
    const size_t join = (size_t)kWarps * 16 * (D + 4) + 2 * kWarps * 16;
    return Query<T, D>::kSharedFloats > join ? Query<T, D>::kSharedFloats : join;
}

// Single tokens: CTA (split, KV head, sequence); the four warps share the head's query rows and deal
// out the split's tiles in turn; their results are joined in shared memory.
template <typename T, int D>
__global__ void __launch_bounds__(kThreads) pages_token_kernel(const AttnArgs a)
{
    using W = Warp<T, D>;
    extern __shared__ float4 shared4[];
    float* shared = reinterpret_cast<float*>(shared4);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
    const int s = a.seqs[b];
    const int len = checked_len(a.p, s, a.st);
    View view;
    view.table = a.p.table + (size_t)(len ? s : 0) * a.p.max_pages;
    view.kvh = kvh;
    view.sinks = a.sinks;
    view.pos_min = view.pos_max = len - 1;
    view.lo_min = view.lo_max = a.window ? max(0, len - a.window) : min(a.prefix, len);
    view.pos[0] = view.pos[1] = view.pos_max;
    view.lo[0] = view.lo[1] = view.lo_min;
    const Tiles tiles = tiles_of(view.pos_max, view.lo_min, view.sinks, W::kTile);
    const int n = tiles.count();
    const int first = (int)((long long)n * split / a.splits), end = (int)((long long)n * (split + 1) / a.splits);

    Query<T, D> q;
    const size_t esize = a.io_bf16 ? 2 : 4;
    const char* q0 = static_cast<const char*>(a.q) + ((size_t)b * a.q_stride + (size_t)kvh * a.group * D) * esize;
    q.load(g < a.group ? q0 + (size_t)g * D * esize : nullptr, g + 8 < a.group ? q0 + (size_t)(g + 8) * D * esize : nullptr, a.io_bf16, t,
           shared, g);
    if (Query<T, D>::kSharedFloats) __syncthreads();  // every warp wrote the same rows

    W w;
    w.clear();
    walk(w, q, a, view, tiles, first + warp, end, kWarps, g, t, lane);

    // Join the warps: maximum, then everything scaled to it.
    if (Query<T, D>::kSharedFloats) __syncthreads();  // the query rows are no longer needed
    constexpr int kPitch = D + 4;
    float* so = shared;                          // [warp][16][kPitch]
    float* sm = shared + kWarps * 16 * kPitch;   // [warp][16]
    float* sl = sm + kWarps * 16;
    if (t == 0)
        for (int r = 0; r < 2; r++) {
            sm[warp * 16 + g + 8 * r] = w.m[r];
            sl[warp * 16 + g + 8 * r] = w.l[r];
        }
#pragma unroll
    for (int r = 0; r < 2; r++) {
        if (g + 8 * r >= a.group) continue;
#pragma unroll
        for (int c = 0; c < W::kOut; c++) {
            so[(warp * 16 + g + 8 * r) * kPitch + W::column(c, 0, t)] = w.o[c][2 * r];
            so[(warp * 16 + g + 8 * r) * kPitch + W::column(c, 1, t)] = w.o[c][2 * r + 1];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < a.group * (D / 4); i += kThreads) {
        const int row = i / (D / 4), c = i % (D / 4) * 4;
        float top = -INFINITY, l = 0.f;
        for (int x = 0; x < kWarps; x++) top = fmaxf(top, sm[x * 16 + row]);
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int x = 0; x < kWarps; x++) {
            const float mx = sm[x * 16 + row];
            const float f = mx == -INFINITY ? 0.f : fast_exp2(mx - top);
            const float4 y = *reinterpret_cast<const float4*>(so + (x * 16 + row) * kPitch + c);
            l += sl[x * 16 + row] * f;
            o.x = fmaf(y.x, f, o.x);
            o.y = fmaf(y.y, f, o.y);
            o.z = fmaf(y.z, f, o.z);
            o.w = fmaf(y.w, f, o.w);
        }
        const size_t R = (size_t)b * a.q_heads + kvh * a.group + row;
        put4(a, D, a.slot0 + split, R, c, o, l);
        if (a.rec.slots > 1 && c == 0) a.rec.ml[(size_t)(a.slot0 + split) * a.rec.rows + R] = make_float2(top, l);
    }
}

// Rows of a CTA tile: `per` tokens x `group` heads, token-major.  The prefix pass takes the batch's
// single tokens as its rows.
constexpr int kRowsCta = 16 * kWarps;

// CTA (row tile, KV head, split): each warp has 16 rows of its own and walks all the split's tiles.
template <typename T, int D, bool kPrefix>
__global__ void __launch_bounds__(kThreads) pages_rows_kernel(const AttnArgs a)
{
    using W = Warp<T, D>;
    extern __shared__ float4 shared4[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int kvh = blockIdx.y, split = blockIdx.z;
    const int per = kRowsCta / a.group;
    int seq = 0, tok0, ntok, pos0;  // first token (row of q) of the tile, tokens, position of the first
    __shared__ int found[4];
    if (kPrefix) {
        tok0 = blockIdx.x * per;
        ntok = min(per, a.batch - tok0);
        seq = a.seqs[0];
        const int len = checked_len(a.p, seq, a.st);
        pos0 = min(a.prefix, len) - 1;
    } else {
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
    view.sinks = kPrefix ? 0 : a.sinks;
    auto lo_of_pos = [&](int pos) { return !kPrefix && a.window ? max(0, pos - a.window + 1) : 0; };
    view.pos_min = pos0;
    view.pos_max = kPrefix ? pos0 : pos0 + ntok - 1;
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
        view.pos[r] = !here[r] ? -1 : kPrefix ? pos0 : pos0 + tk;
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

constexpr int kSms = 148;

// How a call is laid out: its row tiles and splits.
struct Layout {
    bool tokens;  // the token kernel handles (all or the own rows of) the call
    bool shared;  // the row tiles are the shared pass over a prefix
    bool tc;      // the row tiles run on the tcgen05 form
    bool tall;
    int token_splits, row_tiles, row_splits, row_slots, slots;
};

static int ceil_div(long long a, long long b) { return (int)((a + b - 1) / b); }

static Layout layout_of(const tyb_pages_attn* c)
{
    Layout l = {};
    const int kt = c->p.kv_dtype == TYB_BF16 ? 16 : 8;
    const int group = c->q_heads / c->p.kv_heads;
    l.tokens = c->max_new == 1 && c->rows == c->batch;
    l.shared = l.tokens && c->prefix > 0;
    if (l.tokens) {
        long long own = c->window && c->window < c->max_len ? c->window + c->sinks : c->max_len - c->prefix;
        const int tiles = ceil_div(own, kt) + 1;
        // enough CTAs for four on every SM, and at least a tile for each warp of a split
        int s = ceil_div(4LL * kSms, (long long)c->batch * c->p.kv_heads);
        if (s > ceil_div(tiles, kWarps)) s = ceil_div(tiles, kWarps);
        l.token_splits = s < 1 ? 1 : s;
    }
    if (!l.tokens || l.shared) {
        l.tc = c->p.kv_dtype == TYB_BF16;
        l.tall = l.tc && (long long)(l.shared ? c->batch : c->max_new) * group <= kTcTall;
        const int per = (l.tall ? kTcTall : l.tc ? kTcWide : kRowsCta) / group;
        // Each of the sequences of a call ends in a tile of its own; no list has more tiles than this.
        l.row_tiles = l.shared ? ceil_div(c->batch, per) : (int)((c->rows + (long long)c->batch * (per - 1)) / per);
        const long long keys = l.shared ? c->prefix : c->window && c->window < c->max_len ? c->window + c->sinks : c->max_len;
        const int tiles = ceil_div(keys, l.tc ? 128 : kt);
        const long long ctas = (long long)l.row_tiles * c->p.kv_heads;
        int s;
        if (l.tc) {
            s = (int)(kSms / ctas);  // one CTA fits an SM; a split has at least two tiles
            if (s > tiles / 2) s = tiles / 2;
        } else {
            s = ceil_div(3LL * kSms, ctas);
            if (s > ceil_div(tiles, 8)) s = ceil_div(tiles, 8);
        }
        l.row_splits = s < 1 ? 1 : s;
    }
    l.row_slots = l.row_splits * (l.tall ? 2 : 1);
    l.slots = l.token_splits + l.row_slots;
    return l;
}

}  // namespace tyb

extern "C" size_t tyb_pages_attn_bytes(const tyb_pages_attn* c)
{
    const tyb::Layout l = tyb::layout_of(c);
    if (l.slots <= 1) return 0;
    return (size_t)l.slots * c->rows * c->q_heads * (c->p.head_dim * sizeof(float) + sizeof(float2));
}

namespace tyb {

template <typename T, int D>
static int launch(const tyb_pages_attn* c, void* ws, cudaStream_t stream)
{
    const Layout l = layout_of(c);
    AttnArgs a = {};
    a.p = c->p;
    const size_t layer = (size_t)c->layer * c->p.num_pages * c->p.kv_heads * c->p.page_size * D;
    a.k = static_cast<const T*>(c->p.k) + layer;
    a.v = static_cast<const T*>(c->p.v) + layer;
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
    a.rec.rows = c->rows * c->q_heads;
    a.rec.slots = l.slots;
    a.rec.o = static_cast<float*>(ws);
    a.rec.ml = reinterpret_cast<float2*>(static_cast<float*>(ws) + (size_t)l.slots * a.rec.rows * D);
    a.st.word = tyb_status_word();
    a.st.mirror = tyb_status_mirror_device();
    if (!a.st.word) return (int)cudaErrorInvalidSymbol;
    static bool ready[64];
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    if (dev < 0 || dev >= 64) return (int)cudaErrorInvalidDevice;
    const size_t solo = solo_shared_floats<T, D>() * sizeof(float);
    const size_t rows = kWarps * (size_t)Query<float, D>::kSharedFloats * sizeof(float);
    if (!ready[dev]) {
        e = cudaFuncSetAttribute(pages_token_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)solo);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(pages_rows_kernel<T, D, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)rows);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(pages_rows_kernel<T, D, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)rows);
        if (e != cudaSuccess) return (int)e;
        ready[dev] = true;
    }
    if (l.tokens) {
        a.splits = l.token_splits;
        a.slot0 = l.row_slots;
        pages_token_kernel<T, D><<<dim3(l.token_splits, c->p.kv_heads, c->batch), kThreads, solo, stream>>>(a);
        if ((e = cudaGetLastError()) != cudaSuccess) return (int)e;
    }
    if (l.row_splits) {
        a.splits = l.row_splits;
        a.slot0 = 0;
        const dim3 grid(l.row_tiles, c->p.kv_heads, l.row_splits);
        if (l.tc) {
            const int rc = tc_launch(a, c->layer, l.tall, l.shared, l.row_tiles, c->maps, stream);
            if (rc) return rc;
        } else if (l.shared) pages_rows_kernel<T, D, true><<<grid, kThreads, rows, stream>>>(a);
        else pages_rows_kernel<T, D, false><<<grid, kThreads, rows, stream>>>(a);
        if ((e = cudaGetLastError()) != cudaSuccess) return (int)e;
    }
    if (l.slots > 1) {
        pages_join_kernel<D><<<ceil_div(a.rec.rows, kWarps), kThreads, 0, stream>>>(a);
        if ((e = cudaGetLastError()) != cudaSuccess) return (int)e;
    }
    return 0;
}

}  // namespace tyb

using namespace tyb;

extern "C" int tyb_pages_attn_launch(const tyb_pages_attn* c, void* ws, void* stream)
{
    cudaStream_t st = (cudaStream_t)stream;
    if (c->p.kv_dtype == TYB_BF16)
        return c->p.head_dim == 128 ? launch<__nv_bfloat16, 128>(c, ws, st) : launch<__nv_bfloat16, 64>(c, ws, st);
    return c->p.head_dim == 128 ? launch<float, 128>(c, ws, st) : launch<float, 64>(c, ws, st);
}

// pages_rows.cu -- prompt chunks over an FP32 paged cache, through a window with sinks: 64 query rows a CTA
// (the q_heads / kv_heads heads of a KV head folded into the rows) against key tiles of 32 or 16.
//
// A requesting warp brings the tiles by TMA into a ring of stages; four warps with 16 query rows each take
// every tile, with the running maximum and sum of an online softmax in base 2 (pages_mma.cuh: products on
// TF32 halves, a relative error of about 2^-21 each, FP32 sums).  The products bound it: three TF32
// products for each FP32 one, issued by mma.sync; the K and V halves are split by each warp as it uses them.
#define TYB_WHOLE_PROGRAM
#include "pages_mma.cuh"
#include "tcgen05.cuh"

namespace tyb {

constexpr int kRowWarps = kRowsTile / 16;
constexpr int kRowThreads = 32 * (kRowWarps + 1);
constexpr int kRowStagesMax = 6;

template <int D>
struct RowTile {
    // Heads of 128: tiles of 16 keys, with which two CTAs fit an SM (3 chunks of 37 .. 733 tokens through 301: 68 us, with
    // tiles of 32 96; 20 of 200 .. 900: 390 and 552).  Heads of 64, of which three fit either way: tiles of 32 (3 chunks
    // 44 us, with 16 42; 40 chunks 409 and 411; 12 through 1,200 rows 140 and 141).
    static constexpr int kKeys = D == 64 ? 32 : 16;
    static constexpr unsigned int kAll = 0xffffffffu >> (32 - kKeys);
    static constexpr int kBoxes = D / 32, kBox = kKeys * 128, kHalf = kBoxes * kBox, kStage = 2 * kHalf;
    static constexpr int kPitch = D + 4;
    static constexpr int kSplit = 2 * 16 * kPitch * 4;  // a warp's query rows, hi and lo; at the end its output rows
};

struct RowMaps {
    CUtensorMap m[2];  // K, V; for tiles of 16 keys in boxes of 16 rows
};

// A lane's four columns of query rows: where they stand, and what of the tile at j0 they see.
struct ColumnSight {
    int pos[2][2], lo[2][2];
    int j0, sinks;
    unsigned int seen;  // keys whose page is there
    bool whole;
    __device__ __forceinline__ bool all() const { return whole; }
    __device__ __forceinline__ bool operator()(int n, int c, int i) const
    {
        const int j = j0 + i;
        return j <= pos[n][c] && (j >= lo[n][c] || j < sinks) && (seen >> i & 1u);
    }
};

template <int D>
__global__ void __launch_bounds__(kRowThreads, rows_ctas(D)) pages_rows_kernel(const __grid_constant__ RowMaps maps, const AttnArgs a, int layer, int stages,
                                                                   unsigned long long wait_ns)
{
    using R = RowTile<D>;
    extern __shared__ __align__(1024) unsigned char raw[];
    unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    float* splits = reinterpret_cast<float*>(ring + stages * R::kStage);
    __shared__ uint64_t full[kRowStagesMax], empty[kRowStagesMax];
    __shared__ unsigned int seen_of[kRowStagesMax];
    __shared__ float2 out_ml[kRowWarps][16];
    __shared__ int found[4];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int kvh = blockIdx.y, split = blockIdx.z, per = kRowsTile / a.group;
    if (tid == 0) {
        for (int i = 0; i < stages; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], kRowWarps);
        }
        fence_barrier_init();
    }
    after_predecessor();
    if (warp == kRowWarps) find_item(a, (int)(gridDim.x - 1 - blockIdx.x), per, found);  // the last items, with the most keys, first
    __syncthreads();
    if (found[0] < 0) return;
    const int seq = a.seqs[found[0]], tok0 = found[1], ntok = found[2];
    const int pos0 = checked_len(a.p, seq, a.st) + found[3], pos_max = pos0 + ntok - 1;
    if (pos0 < 0 && tid == 0) raise(a.st, TYB_STATUS_BAD_ARGUMENT);  // more queries than tokens
    auto lo_of_pos = [&](int pos) { return a.window ? max(0, pos - a.window + 1) : 0; };
    const int lo_min = lo_of_pos(pos0);
    const Tiles tiles = tiles_of(pos_max, lo_min, a.sinks, R::kKeys);
    const int all = tiles.count(), first = (int)((long long)all * split / a.splits), nt = (int)((long long)all * (split + 1) / a.splits) - first;

    if (warp == kRowWarps) {
        // ---- requests: lane (part, 128-byte column box, K or V)
        const int part_rows = min(box_rows(a.p), R::kKeys), parts = R::kKeys / part_rows, shift = page_shift(a.p.page_size);
        const int part = lane & (parts - 1), box = lane / parts & (R::kBoxes - 1), which = lane / (parts * R::kBoxes);
        const int* table = a.p.table + (size_t)max(0, min(seq, a.p.max_seqs - 1)) * a.p.max_pages;
        int st = 0, t = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (; t < nt; t++) {
            const int key = tiles.at(first + t) * R::kKeys + part * part_rows;
            int page = which < 2 && key <= pos_max ? table[key >> shift] : -1;
            if (page >= a.p.num_pages) {
                raise(a.st, TYB_STATUS_BAD_ARGUMENT);
                page = -1;
            }
            const unsigned int have = __ballot_sync(0xffffffffu, page >= 0);
            if (t >= stages) ok = warp_wait_for(&empty[st], phase ^ 1u, wait_ns, a.st);
            if (!ok) break;
            if (lane == 0) {
                unsigned int seen = 0;
                for (int l = 0; l < parts; l++)
                    if (have >> l & 1u) seen |= (part_rows == 32 ? 0xffffffffu : 0xffffu) << (l * part_rows);
                seen_of[st] = seen;
                mbar_arrive_expect_tx(&full[st], (uint32_t)(__popc(have) * part_rows * 128));
            }
            __syncwarp();
            if (page >= 0) {
                const int row = ((layer * a.p.num_pages + page) * a.p.kv_heads + kvh) * a.p.page_size + (key & (a.p.page_size - 1));
                unsigned char* to = ring + st * R::kStage + which * R::kHalf + box * R::kBox + part * part_rows * 128;
                if (R::kKeys == 16) tma_load_3d(to, &maps.m[which], row, box, &full[st]);
                else tma_load_2d(to, &maps.m[which], box * 32, row, &full[st]);
            }
            if (++st == stages) {
                st = 0;
                phase ^= 1u;
            }
        }
        // The copies requested have landed before this warp, and with it the CTA, ends.
        for (int n = max(0, t - stages); n < t; n++) warp_wait_for(&full[n % stages], (uint32_t)(n / stages) & 1u, drain_ns(wait_ns), a.st);
        return;
    }

    // ---- rows 16 warp .. + 16 of the tile, token-major; those that are not there repeat the last token's, and nobody
    // takes their results
    const int g = lane >> 2, t = lane & 3;
    float* mine = splits + warp * (R::kSplit / 4);
    Rows<float, D, 2, false> w;
    w.clear();
    auto token = [&](int row, int& head) {
        const int flat = 16 * warp + row, tk = flat / a.group;
        head = flat - tk * a.group;
        return tk;
    };
    {
        // two lanes a row, 16 bytes at a time in turn
        int head;
        const int row = lane >> 1, tk = min(token(row, head), ntok - 1);
        const size_t at = (size_t)(tok0 + tk) * a.q_stride + (size_t)(kvh * a.group + head) * D;
#pragma unroll
        for (int c = 8 * (lane & 1); c < D; c += 16) {
            float x[8];
            if (a.io_bf16) load8(static_cast<const __nv_bfloat16*>(a.q) + at + c, x);
            else load8(static_cast<const float*>(a.q) + at + c, x);
#pragma unroll
            for (int i = 0; i < 8; i++) {
                uint32_t hi, lo;
                split_tf32(x[i], hi, lo);
                mine[row * R::kPitch + c + i] = __uint_as_float(hi);
                mine[(16 + row) * R::kPitch + c + i] = __uint_as_float(lo);
            }
        }
        __syncwarp();
    }
    ColumnSight sight;
    sight.sinks = a.sinks;
#pragma unroll
    for (int n = 0; n < 2; n++)
#pragma unroll
        for (int c = 0; c < 2; c++) {
            int head;
            sight.pos[n][c] = pos0 + min(token(8 * n + 2 * t + c, head), ntok - 1);
            sight.lo[n][c] = lo_of_pos(sight.pos[n][c]);
        }
    int head;
    const int wpos_min = pos0 + min(token(0, head), ntok - 1), wpos_max = pos0 + min(token(15, head), ntok - 1);
    const int wlo_min = lo_of_pos(wpos_min), wlo_max = lo_of_pos(wpos_max);
    int st = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int i = 0; i < nt; i++) {
        ok = warp_wait_for(&full[st], phase, wait_ns, a.st);
        if (!ok) break;
        const int k0 = tiles.at(first + i) * R::kKeys;
        const unsigned int seen = seen_of[st];
        unsigned char *rows_k = ring + st * R::kStage, *rows_v = rows_k + R::kHalf;
        // Rows that no query of the CTA sees may hold anything, and 0 * NaN is not 0.  (Every warp clears them for
        // itself: the others write the same zeros.)
        if (seen != R::kAll || k0 + R::kKeys - 1 > pos_max || (k0 < lo_min && k0 + R::kKeys > a.sinks)) {
#pragma unroll 4
            for (int x = lane; x < R::kKeys * (D / 4); x += 32) {
                const int r = x / (D / 4), c = x % (D / 4), j = k0 + r;
                if (!((seen >> r & 1u) && j <= pos_max && (j >= lo_min || j < a.sinks)))
                    *reinterpret_cast<uint4*>(rows_v + (c >> 3) * R::kBox + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
        }
#pragma unroll 1
        for (int r0 = 0; r0 < R::kKeys; r0 += 16) {
            sight.j0 = k0 + r0;
            sight.seen = seen >> r0 & 0xffffu;
            if (!sight.seen || sight.j0 > wpos_max || (sight.j0 + 16 <= wlo_min && sight.j0 >= a.sinks)) continue;  // nothing in sight
            sight.whole = sight.seen == 0xffffu && sight.j0 + 15 <= wpos_min && (sight.j0 >= wlo_max || sight.j0 + 16 <= a.sinks);
            w.step(rows_k, rows_v, R::kBox, r0, sight, a.scale_log2, mine, g, t, lane);
        }
        warp_arrive(&empty[st]);
        if (++st == stages) {
            st = 0;
            phase ^= 1u;
        }
    }
    if (!ok) return;
    // ---- out, in whole rows, through the warp's part of shared memory
    __syncwarp();
    w.put(mine, R::kPitch, out_ml[warp], 16, g, t);
    __syncwarp();
    for (int x = lane; x < 16 * (D / 4); x += 32) {
        const int row = x / (D / 4), c = x % (D / 4) * 4, tk = token(row, head);
        if (tk >= ntok) continue;
        const size_t out = (size_t)(tok0 + tk) * a.q_heads + kvh * a.group + head;
        const float4 v = *reinterpret_cast<const float4*>(mine + row * R::kPitch + c);
        const float2 ml = out_ml[warp][row];
        if (a.rec.slots == 1) {
            put_out(a, out * D + c, v, ml.y);
        } else {
            const size_t at = (size_t)split * a.rec.rows + out;
            *reinterpret_cast<float4*>(a.rec.o + at * D + c) = v;
            if (c == 0) a.rec.ml[at] = ml;
        }
    }
}

template <int D>
static int launch(const AttnArgs& a, int layer, int items, const void* maps, cudaStream_t stream)
{
    using R = RowTile<D>;
    static bool ready[64];
    const int dev = a.device;
    if (dev < 0 || dev >= 64) return (int)cudaErrorInvalidDevice;
    // as many stages as leave room for rows_ctas(D) CTAs on the SM, or two
    const int fixed = kRowWarps * R::kSplit + 1024;
    int stages = (228 * 1024 / rows_ctas(D) - 1024 - 1024 - fixed) / R::kStage;
    stages = stages < 2 ? 2 : stages > kRowStagesMax ? kRowStagesMax : stages;
    const int bytes = stages * R::kStage + fixed;
    if (!ready[dev]) {
        cudaError_t e = cudaFuncSetAttribute(pages_rows_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(pages_rows_kernel<D>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
        if (e != cudaSuccess) return (int)e;
        ready[dev] = true;
    }
    return launch_after(pages_rows_kernel<D>, dim3(items, a.p.kv_heads, a.splits), kRowThreads, bytes, stream, *reinterpret_cast<const RowMaps*>(static_cast<const CUtensorMap*>(maps) + (R::kKeys == 16 ? 4 : 0)), a,
                        layer, stages, tyb_wait_limit_of(dev));
}

int rows_launch(const AttnArgs& a, int layer, int items, const void* maps, cudaStream_t stream)
{
    return a.p.head_dim == 128 ? launch<128>(a, layer, items, maps, stream) : launch<64>(a, layer, items, maps, stream);
}

}  // namespace tyb

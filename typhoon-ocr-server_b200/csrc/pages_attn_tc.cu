// pages_attn_tc.cu -- attention of many query rows over the paged BF16 cache on the 5th-generation
// tensor cores (tcgen05 + TMEM): prompt chunks through a window with sinks, and the shared prefix of a
// decode batch.
//
// A CTA has query rows of one KV head (its q_heads / kv_heads query heads folded into the rows, so
// that one K/V tile feeds them all) and a run of key tiles of 64.  Two streams of 128 rows alternate on
// the tensor core, one's softmax overlapping the other's products:
//   wide   256 rows, both streams take every tile (each K/V tile is loaded once for 256 rows);
//   tall   at most 128 rows: the streams have the same rows and take the tiles in turn, and their results
//          are joined like those of two splits.  Half the tensor work of a wide item that would be half empty.
// A tile comes page by page: one TMA tensor copy per page and 64 columns, the 128-byte-swizzled
// layout building up in shared memory as if it were one copy; the pages of a tile are issued by as
// many lanes of the producer warp.  Rows of the tile that no row of the item sees (behind the
// sequence's end, a page that is not there, before the window) may hold anything: their scores are
// masked, and their V rows are cleared in shared memory before P.V, since 0 * NaN is not 0.
//
// Roles (12 warps): 0-3 and 4-7 the streams' softmax (one row per thread), 8 issues Q.K^T, 11 P.V, 9 the
// copies, 10 clears V rows.  TMEM: S0 | S1 (64 columns each) | P of each stream, two buffers (32 each) |
// O0 | O1.  Tiles of 64 keys are what makes room for two P buffers beside an S for each stream: the softmax of a
// tile waits for neither the P.V of the one before nor the other stream, only for its own S, which is computed
// while it works on the tile before: 256 rows x 64 keys of 128 dimensions in 1.0 us.  (With tiles of 128, one S for
// both streams and one P each, 256 rows x 128 keys took 2.6 us; their products alone take 1.1 us and their
// exponentials as much.)
// Every wait is bounded; a CTA whose wait ran out raises the status word, leaves its loops, frees its
// TMEM and returns.
#define TYB_WHOLE_PROGRAM
#include "pages_attn.cuh"
#include "tcgen05.cuh"

#include <type_traits>

namespace tyb {

constexpr int kRows = 128;   // rows of a stream (tensor-core M)
constexpr int kKeys = 64;    // keys of a tile: N of S, K of P.V
constexpr int kSoftThreads = 256;
constexpr int kTcThreads = kSoftThreads + 128;
// Register split, as in the fused prefill: launched at kLaunchRegs, the issue warpgroup drops to
// kIssueRegs and the softmax warpgroups rise to kSoftRegs; the shares fit the launch's registers.
constexpr int kLaunchRegs = 168, kIssueRegs = 112, kSoftRegs = 192;
static_assert(kSoftThreads * kSoftRegs + 128 * kIssueRegs <= kTcThreads * kLaunchRegs, "register split");
static_assert(2 * kSoftRegs + kIssueRegs <= 512, "register split of a sub-partition");
constexpr int kBoxQ = kTcBox;        // 128 rows x 64 columns of BF16
constexpr int kBox = kKeys * 128;    // a tile's rows x 64 columns
constexpr int kStages = 5;           // of the K and V rings: 32 KB of 128-wide tiles each, all that fits beside Q
constexpr int kSeen = 16;  // ring of page masks, one per tile: more than the tiles in flight

struct TcArgs {
    AttnArgs a;
    int layer;
    int tall;        // the streams share their rows
    int row_tiles;
    int shared_pass; // the rows are the batch's single tokens against the first sequence's leading rows
    unsigned long long wait_ns;
};

template <int D>
struct Smem {
    static constexpr int kTileQ = (D / 64) * kBoxQ, kTile = (D / 64) * kBox;
    static constexpr int kQ = 0, kK = 2 * kTileQ, kV = kK + kStages * kTile, kBars = kV + kStages * kTile;
    static constexpr size_t kBytes = (size_t)kBars + 512 + 1024;  // + barriers + alignment slack
};

// Instruction descriptor, kind::f16: BF16 operands, FP32 accumulator, M = 128.
__host__ __device__ constexpr uint32_t idesc(int n, bool b_mn_major)
{
    return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}

// D[tmem] (+)= A . B^T, kind::f16, A from shared memory (mma_ss) or TMEM (mma_ts).  Issued by one elected lane of a
// converged warp, so that descriptors and addresses stay in uniform registers: issued from a branch of one
// lane, each product cost about 150 cycles in moving its operands there, more than twice its execution.
__device__ __forceinline__ bool elect_one()
{
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a),
                 "l"(b), "r"(id), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
                 "r"(a), "l"(b), "r"(id), "r"(accumulate)
                 : "memory");
}

__device__ __forceinline__ float max3(float a, float b, float c)
{
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

// Columns [0, n) of 32, n clamped.
__device__ __forceinline__ uint32_t below(int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; }

// Which of a tile's columns a row sees, 32 per word.
struct Mask {
    uint32_t w[kKeys / 32];
};

template <bool kMask>
__device__ __forceinline__ float row_max(const float (&s)[kKeys], const Mask& mk)
{
    float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int c = 0; c < kKeys; c += 2) {
        const float a = (!kMask || (mk.w[c >> 5] >> (c & 31) & 1u)) ? s[c] : -INFINITY;
        const float b = (!kMask || (mk.w[c >> 5] >> ((c + 1) & 31) & 1u)) ? s[c + 1] : -INFINITY;
        m[(c >> 1) & 3] = max3(m[(c >> 1) & 3], a, b);
    }
    return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}

// p = exp2(s * scale + neg) on the visible columns (0 on the others) as BF16 pairs into the row's TMEM
// columns at p_addr; returns the FP32 sum.  kTrack: *top receives the largest exponent.
template <bool kMask, bool kTrack, typename Ready>
__device__ __forceinline__ float row_exp(const float (&s)[kKeys], const Mask& mk, float scale, float neg, uint32_t p_addr, float* top,
                                         Ready ready)
{
    const float2 sc = make_float2(scale, scale), nm = make_float2(neg, neg);
    float2 acc0 = make_float2(0.f, 0.f), acc1 = make_float2(0.f, 0.f);
    float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
    for (int q = 0; q < kKeys / 32; q++) {
        uint32_t pk[16];
#pragma unroll
        for (int c = 0; c < 32; c += 4) {
            const int k = q * 32 + c;
            float2 x0 = __ffma2_rn(make_float2(s[k], s[k + 1]), sc, nm);
            float2 x1 = __ffma2_rn(make_float2(s[k + 2], s[k + 3]), sc, nm);
            if (kMask) {
                if (!(mk.w[q] >> c & 1u)) x0.x = -INFINITY;
                if (!(mk.w[q] >> (c + 1) & 1u)) x0.y = -INFINITY;
                if (!(mk.w[q] >> (c + 2) & 1u)) x1.x = -INFINITY;
                if (!(mk.w[q] >> (c + 3) & 1u)) x1.y = -INFINITY;
            }
            if (kTrack) {
                t0 = max3(t0, x0.x, x0.y);
                t1 = max3(t1, x1.x, x1.y);
            }
            const float2 e0 = make_float2(pt_exp2(x0.x), pt_exp2(x0.y)), e1 = make_float2(pt_exp2(x1.x), pt_exp2(x1.y));
            acc0 = __fadd2_rn(acc0, e0);
            acc1 = __fadd2_rn(acc1, e1);
            pk[c / 2] = pack_bf16x2(e0.x, e0.y);
            pk[c / 2 + 1] = pack_bf16x2(e1.x, e1.y);
        }
        if (q == 0) ready();
        tmem_st16u(p_addr + q * 16, pk);
    }
    tmem_wait_st();
    if (kTrack) *top = fmaxf(t0, t1);
    return (acc0.x + acc0.y) + (acc1.x + acc1.y);
}

template <int D>
__global__ void __launch_bounds__(kTcThreads, 1)
    pages_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const TcArgs ta)
{
    using S = Smem<D>;
    const AttnArgs& a = ta.a;
    extern __shared__ __align__(1024) unsigned char raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    unsigned char *sQ = smem + S::kQ, *sK = smem + S::kK, *sV = smem + S::kV;
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::kBars);
    uint64_t *k_full = bars, *k_free = k_full + kStages, *v_full = k_free + kStages, *v_free = v_full + kStages,
             *v_clear = v_free + kStages;                         // [stage]
    uint64_t *s_full = v_clear + kStages, *s_free = s_full + 2;   // [stream]
    uint64_t *p_full = s_free + 2, *pv_done = p_full + 4;         // [stream][buffer]
    uint64_t *q_full = pv_done + 4, *drain = q_full + 1;          // drain: [2]
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 2);
    int* found = reinterpret_cast<int*>(drain + 3);                       // [4]
    volatile uint32_t* present = reinterpret_cast<uint32_t*>(drain + 5);  // [kSeen] a bit per 16 rows of the tile

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    // CTA: a row tile's KV heads next to each other, then its splits (16,384 tokens through 4,096 in 485 us, with
    // a head's row tiles next to each other 505 us).
    const int kvh = (int)blockIdx.x % a.p.kv_heads, split = (int)blockIdx.x / a.p.kv_heads % a.splits,
              row_tile = (int)blockIdx.x / (a.p.kv_heads * a.splits);
    if (row_tile >= ta.row_tiles) return;  // (one CTA, of a grid rounded up to pairs)
    const int rows_item = ta.tall ? kRows : 2 * kRows;
    const int per = rows_item / a.group;  // tokens of an item

    if (warp == 8) {
        if (lane == 0) {
            for (int i = 0; i < kStages; i++) {
                mbar_init(&k_full[i], 1);
                mbar_init(&k_free[i], 1);
                mbar_init(&v_full[i], 1);
                mbar_init(&v_free[i], 1);
                mbar_init(&v_clear[i], 1);
            }
            for (int i = 0; i < 2; i++) {
                mbar_init(&s_full[i], 1);
                mbar_init(&s_free[i], kRows / 32);
            }
            for (int i = 0; i < 4; i++) {
                mbar_init(&p_full[i], kRows / 32);
                mbar_init(&pv_done[i], 1);
            }
            mbar_init(q_full, kSoftThreads / 32);
            mbar_init(&drain[0], 1);
            mbar_init(&drain[1], 1);
            fence_barrier_init();
            fence_proxy_async_smem();
        }
        __syncwarp();
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(tmem_slot)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        tc_fence_before();
    }
    after_predecessor();
    if (warp == 0 && !ta.shared_pass) find_item(a, ta.row_tiles - 1 - row_tile, per, found);  // the last items, with the most keys, first
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    int tok0 = 0, ntok = 0;
    if (ta.shared_pass) {
        tok0 = row_tile * per;
        ntok = min(per, a.batch - tok0);
    } else if (found[0] >= 0) {
        tok0 = found[1];
        ntok = found[2];
    }
    // ---- queries, BF16, into the swizzled layout: a warp per 32 rows, D / 8 lanes a row
    // (rows that are not there repeat the last token's: nobody takes their results).  All of a warp's loads are in
    // flight at once.
    if (warp < 8 && ntok > 0 && (!ta.tall || warp < 4)) {
        const int h = warp >> 2;
        constexpr int kLanes = D / 8, kAtOnce = 32 / kLanes, kLoads = 32 / kAtOnce;
        unsigned char* tile = sQ + h * S::kTileQ;
        const int c = lane % kLanes * 8;
        size_t off[kLoads];
        // row 32 (warp & 3) + lane / kLanes, then kAtOnce further each time; in flat rows twice that when wide
        const int row0 = 32 * (warp & 3) + lane / kLanes, flat0 = ta.tall ? row0 : 2 * row0 + h, ahead = ta.tall ? kAtOnce : 2 * kAtOnce;
        int tk = flat0 / a.group, hh = flat0 - tk * a.group;
        const int tk_ahead = ahead / a.group, hh_ahead = ahead - tk_ahead * a.group;
#pragma unroll
        for (int i = 0; i < kLoads; i++) {
            off[i] = (size_t)(tok0 + min(tk, ntok - 1)) * a.q_stride + (size_t)(kvh * a.group + hh) * D + c;
            tk += tk_ahead;
            hh += hh_ahead;
            if (hh >= a.group) {
                hh -= a.group;
                tk++;
            }
        }
        uint4 x[kLoads];
        if (a.io_bf16) {
#pragma unroll
            for (int i = 0; i < kLoads; i++) x[i] = *reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.q) + off[i]);
        } else {
#pragma unroll
            for (int i = 0; i < kLoads; i++) {
                float f[8];
                load8(static_cast<const float*>(a.q) + off[i], f);
                x[i] = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
            }
        }
#pragma unroll
        for (int i = 0; i < kLoads; i++)
            *reinterpret_cast<uint4*>(tile + sw128_offset(row0 + i * kAtOnce, c)) = x[i];
    }
    if (warp < 8) {
        fence_proxy_async_smem();
        warp_arrive(q_full);
    }

    // (after the queries' loads are out: the length is two loads deep)
    int seq = -1, pos0 = -1;
    if (ta.shared_pass) {
        seq = a.seqs[0];
        pos0 = min(a.prefix, checked_len(a.p, seq, a.st)) - 1;
    } else if (ntok > 0) {
        seq = a.seqs[found[0]];
        pos0 = checked_len(a.p, seq, a.st) + found[3];
        if (pos0 < 0 && tid == 0) raise(a.st, TYB_STATUS_BAD_ARGUMENT);  // more queries than tokens
    }
    const int sinks = ta.shared_pass ? 0 : a.sinks;
    const bool windowed = !ta.shared_pass && a.window;
    const int pos_max = ta.shared_pass ? pos0 : pos0 + ntok - 1;
    const int lo_min = windowed ? max(0, pos0 - a.window + 1) : 0, lo_max = windowed ? max(0, pos_max - a.window + 1) : 0;
    const Tiles tiles = tiles_of(ntok > 0 ? pos_max : -1, lo_min, sinks, kKeys);
    const int all = tiles.count();
    const int first = (int)((long long)all * split / a.splits), nt = (int)((long long)all * (split + 1) / a.splits) - first;
    constexpr uint32_t kTile16 = S::kTile >> 4, kTileQ16 = S::kTileQ >> 4;  // in units of the operand descriptors
    // Step i of both streams is stream i & 1's; its tile:
    const int steps = ta.tall ? nt : 2 * nt;
    auto tile_of = [&](int i) { return ta.tall ? i : i >> 1; };
    // Whether some row of the item does not see the whole tile (its pages aside), and whether the tile
    // has rows that none sees.
    auto edge = [&](int k0) { return k0 + kKeys - 1 > pos0 || (k0 < lo_max && k0 + kKeys > sinks); };
    auto loose = [&](int k0) { return k0 + kKeys - 1 > pos_max || (k0 < lo_min && k0 + kKeys > sinks); };
    auto warp_drain = [&](uint64_t* bar, uint32_t parity) { return warp_wait_for(bar, parity & 1u, drain_ns(ta.wait_ns), a.st); };
    auto warp_wait = [&](uint64_t* bar, uint32_t parity) { return warp_wait_for(bar, parity & 1u, ta.wait_ns, a.st); };

    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
        if (warp == 9) {
            // ---- copies: lane l < parts of a tile has the page (or its part) at rows l * part
            const int part = box_rows(a.p), shift = page_shift(a.p.page_size), per_tile = kKeys / part;
            const int* table = a.p.table + (size_t)max(0, min(seq, a.p.max_seqs - 1)) * a.p.max_pages;
            const uint32_t part_bits = (1u << (part / 16)) - 1u;
            const int part_bytes = part * 128;  // of a 64-column box
            bool ok = true;
            int k_sent = 0, v_sent = 0;  // tiles requested
            int st = 0;
            uint32_t phase = 1;  // of the last use of the stage
            for (int t = 0; t < nt && ok; t++) {
                const int key = tiles.at(first + t) * kKeys + lane * part;
                int page = -1;
                if (lane < per_tile && key <= pos_max) {
                    page = table[key >> shift];
                    if (page >= a.p.num_pages) {
                        raise(a.st, TYB_STATUS_BAD_ARGUMENT);
                        page = -1;
                    }
                }
                const uint32_t have = __ballot_sync(0xffffffffu, page >= 0);
                const int row = page < 0 ? 0
                                         : ((ta.layer * a.p.num_pages + page) * a.p.kv_heads + kvh) * a.p.page_size + (key & (a.p.page_size - 1));
                const uint32_t bytes = (uint32_t)__popc(have) * (uint32_t)(part_bytes * (D / 64));
                if (t >= kStages) ok = warp_wait(&k_free[st], phase);
                if (!ok) break;
                if (lane == 0) {
                    uint32_t seen = 0;
                    for (int l = 0; l < per_tile; l++)
                        if (have >> l & 1u) seen |= part_bits << (l * (part / 16));
                    present[t & (kSeen - 1)] = seen;
                    mbar_arrive_expect_tx(&k_full[st], bytes);
                }
                __syncwarp();
                if (page >= 0)
#pragma unroll
                    for (int c = 0; c < D / 64; c++)
                        tma_load_2d(sK + st * S::kTile + c * kBox + lane * part_bytes, &map_k, 64 * c, row, &k_full[st]);
                k_sent = t + 1;
                if (t >= kStages) ok = warp_wait(&v_free[st], phase);
                if (!ok) break;
                if (lane == 0) mbar_arrive_expect_tx(&v_full[st], bytes);
                __syncwarp();
                if (page >= 0)
#pragma unroll
                    for (int c = 0; c < D / 64; c++)
                        tma_load_2d(sV + st * S::kTile + c * kBox + lane * part_bytes, &map_v, 64 * c, row, &v_full[st]);
                v_sent = t + 1;
                if (++st == kStages) {
                    st = 0;
                    phase ^= 1u;
                }
            }
            // The copies requested have landed before this warp, and with it the CTA, ends.
            for (int t = max(0, k_sent - kStages); t < k_sent; t++) warp_drain(&k_full[t % kStages], (uint32_t)(t / kStages));
            for (int t = max(0, v_sent - kStages); t < v_sent; t++) warp_drain(&v_full[t % kStages], (uint32_t)(t / kStages));
        } else if (warp == 8) {
            // ---- S = Q . K^T: a stream's next one goes out as soon as its S has been read
            const uint64_t dq = umma_desc(smem_u32(sQ), 16), dk = umma_desc(smem_u32(sK), 16);
            bool ok = steps == 0 || warp_wait(q_full, 0);
            int st = 0;
            uint32_t phase = 0;
            for (int i = 0; i < steps && ok; i++) {
                const int h = i & 1;
                if (i >= 2) ok = warp_wait(&s_free[h], (uint32_t)(i >> 1) - 1u);
                if (ok && (ta.tall || h == 0)) ok = warp_wait(&k_full[st], phase);
                if (!ok) break;
                tc_fence_after();
                const uint64_t q = dq + (ta.tall ? 0u : h * kTileQ16), k = dk + st * kTile16;
                const bool last = ta.tall || h == 1;  // use of the tile
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < D / 16; kk++)
                        mma_ss(tmem + h * kKeys, q + (((kk >> 2) * kBoxQ + (kk & 3) * 32) >> 4), k + (((kk >> 2) * kBox + (kk & 3) * 32) >> 4),
                               idesc(kKeys, false), kk > 0);
                    tc_commit(&s_full[h]);
                    if (last) tc_commit(&k_free[st]);
                }
                __syncwarp();
                if (last && ++st == kStages) {
                    st = 0;
                    phase ^= 1u;
                }
            }
            // The products issued have ended before this warp does, and TMEM is given back.
            if (elect_one()) tc_commit(&drain[0]);
            __syncwarp();
            warp_drain(&drain[0], 0);
        } else if (warp == 11) {
            // ---- O += P . V, from a warp of its own: one warp's waits and issue for both took longer than the products
            const uint64_t dv = umma_desc(smem_u32(sV), kBox);
            bool ok = true;
            int st = 0;
            uint32_t phase = 0;
            for (int i = 0; i < steps && ok; i++) {
                const int h = i & 1, buf = i >> 1 & 1;
                if (ta.tall || h == 0) ok = warp_wait(&v_full[st], phase) && warp_wait(&v_clear[st], phase);
                if (ok) ok = warp_wait(&p_full[2 * h + buf], (uint32_t)(i >> 2));
                if (!ok) break;
                tc_fence_after();
                const uint64_t v = dv + st * kTile16;
                const bool last = ta.tall || h == 1;  // use of the tile
                if (elect_one()) {
#pragma unroll
                    for (int kk = 0; kk < kKeys / 16; kk++)
                        mma_ts(tmem + 256 + h * D, tmem + 128 + (2 * h + buf) * 32 + kk * 8, v + ((kk * 16 * 128) >> 4), idesc(D, true),
                               i > 1 || kk > 0);
                    tc_commit(&pv_done[2 * h + buf]);
                    if (last) tc_commit(&v_free[st]);
                }
                __syncwarp();
                if (last && ++st == kStages) {
                    st = 0;
                    phase ^= 1u;
                }
            }
            if (elect_one()) tc_commit(&drain[1]);
            __syncwarp();
            warp_drain(&drain[1], 0);
        } else if (warp == 10) {
            // ---- V rows that no row of the item sees.  Every tile passes here, so that this warp and the MMAs
            // stay within one phase of each other.
            int st = 0;
            uint32_t phase = 0;
            for (int t = 0; t < nt; t++) {
                const int k0 = tiles.at(first + t) * kKeys;
                if (!warp_wait(&v_full[st], phase)) break;
                const uint32_t seen = present[t & (kSeen - 1)];
                if (loose(k0) || seen != 0xfu) {
#pragma unroll 4
                    for (int i = lane; i < kKeys * (D / 8); i += 32) {
                        const int r = i / (D / 8), c = i % (D / 8), j = k0 + r;
                        if (!((seen >> (r >> 4) & 1u) && j <= pos_max && (j >= lo_min || j < sinks)))
                            *reinterpret_cast<uint4*>(sV + st * S::kTile + (c >> 3) * kBox + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async_smem();
                }
                warp_arrive(&v_clear[st]);
                if (++st == kStages) {
                    st = 0;
                    phase ^= 1u;
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftRegs));
        // Row r of stream h is flat row 2 r + h of the item (r when tall), token-major: both streams reach
        // over the same tokens.
        const int h = warp >> 2, r = 32 * (warp & 3) + lane;
        // ---- softmax: a row per thread
        const int flat = ta.tall ? r : 2 * r + h;
        const int tk = flat / a.group, hh = flat - tk * a.group;
        const bool here = tk < ntok;
        const int pos = ta.shared_pass ? pos0 : pos0 + min(tk, ntok - 1);
        const int lo = windowed ? max(0, pos - a.window + 1) : 0;
        const uint32_t lanes = (uint32_t)(32 * (warp & 3)) << 16;
        const uint32_t s_addr = tmem + lanes + h * kKeys, p_addr = tmem + lanes + 128 + h * 64, o_addr = tmem + lanes + 256 + h * D;
        const int mine = (steps + 1 - h) >> 1;  // steps of this stream
        float m_run = -INFINITY, l_run = 0.f;
        bool ok = true;
        auto pv_wait = [&](int j) { return warp_wait(&pv_done[2 * h + (j & 1)], (uint32_t)(j >> 1)); };
        for (int j = 0; j < mine; j++) {
            const int i = 2 * j + h, t = tile_of(i);
            if (!warp_wait(&s_full[h], (uint32_t)j)) {
                ok = false;
                break;
            }
            tc_fence_after();
            float sv[kKeys];
            tmem_ld64(s_addr, sv);
            tc_fence_before();
            const uint32_t seen = present[t & (kSeen - 1)];
            warp_arrive(&s_free[h]);
            const int k0 = tiles.at(first + t) * kKeys;
            const bool masked = edge(k0) || seen != 0xfu;
            Mask mk;
            if (masked) {
#pragma unroll
                for (int q = 0; q < kKeys / 32; q++) {
                    const int c0 = k0 + 32 * q;
                    const uint32_t pages = (seen >> (2 * q) & 1u ? 0xffffu : 0u) | (seen >> (2 * q) & 2u ? 0xffff0000u : 0u);
                    mk.w[q] = below(pos + 1 - c0) & (~below(lo - c0) | below(sinks - c0)) & pages;
                }
            }
            // The P buffer is the operand of P.V two steps back until that is done: looked at when the first half of the
            // exponentials is on its way.
            auto ready = [&]() {
                if (j > 1) {
                    ok = ok && pv_wait(j - 2);
                    tc_fence_after();
                }
            };
            const uint32_t p = p_addr + (j & 1) * 32;
            // The running maximum moves only when a step's exceeds it by more than 2^8 (P stays within BF16's
            // range and the FP32 sums do not mind), which spares most rescalings of O: exponentials against the
            // running maximum, tracking the largest exponent, and again if some row's passed 8.  Rows that have
            // seen nothing yet take their step's maximum first.
            float rowsum, alpha = 1.f;
            if (__any_sync(0xffffffffu, m_run == -INFINITY)) {
                float m_new = m_run;
                const float top = (masked ? row_max<true>(sv, mk) : row_max<false>(sv, mk)) * a.scale_log2;
                if (m_run == -INFINITY) m_new = top;
                else if (top > m_run + 8.f) m_new = top;
                alpha = m_run == -INFINITY ? 1.f : pt_exp2(m_run - m_new);  // nothing gathered: nothing to scale
                m_run = m_new;
                const float neg = m_run == -INFINITY ? 0.f : -m_run;
                rowsum = masked ? row_exp<true, false>(sv, mk, a.scale_log2, neg, p, nullptr, ready)
                                : row_exp<false, false>(sv, mk, a.scale_log2, neg, p, nullptr, ready);
            } else {
                float top;
                rowsum = masked ? row_exp<true, true>(sv, mk, a.scale_log2, -m_run, p, &top, ready)
                                : row_exp<false, true>(sv, mk, a.scale_log2, -m_run, p, &top, ready);
                const bool move = top > 8.f;
                if (__any_sync(0xffffffffu, move)) {
                    float m_new = m_run;
                    if (move) {
                        m_new = m_run + top;
                        alpha = pt_exp2(m_run - m_new);
                    }
                    m_run = m_new;
                    rowsum = masked ? row_exp<true, false>(sv, mk, a.scale_log2, -m_run, p, nullptr, ready)
                                    : row_exp<false, false>(sv, mk, a.scale_log2, -m_run, p, nullptr, ready);
                }
            }
            if (!ok) break;
            if (j > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                if (!pv_wait(j - 1)) {  // O is at rest
                    ok = false;
                    break;
                }
                tc_fence_after();
#pragma unroll
                for (int q = 0; q < D / 32; q++) {
                    float ov[32];
                    tmem_ld32(o_addr + q * 32, ov);
#pragma unroll
                    for (int c = 0; c < 32; c++) ov[c] *= alpha;
                    tmem_st32(o_addr + q * 32, ov);
                }
                tmem_wait_st();
            }
            l_run = l_run * alpha + rowsum;
            tc_fence_before();
            warp_arrive(&p_full[2 * h + (j & 1)]);
        }
        // ---- the rows' outputs, or their records: some columns at a time through shared memory (the stream's query
        // tile, no longer needed), so that they leave in whole lines instead of 16 bytes of 32 rows at a time
        const int slot = ta.tall ? 2 * split + h : split;
        const bool direct = a.rec.slots == 1;
        if (ok && mine > 0) ok = pv_wait(mine - 1);
        if (ta.tall) asm volatile("bar.sync 1, %0;" ::"n"(kSoftThreads) : "memory");  // the other stream is done with the queries too
        const size_t R = (size_t)(tok0 + tk) * a.q_heads + kvh * a.group + hh;
        const float mul = !direct ? 1.f : l_run == 0.f ? 0.f : 1.f / l_run;
        if (!direct && here && ok) a.rec.ml[(size_t)slot * a.rec.rows + R] = make_float2(m_run, l_run);
        tc_fence_after();
        unsigned char* stage = sQ + h * S::kTileQ + (warp & 3) * (S::kTileQ / 4);
        static_assert(S::kTileQ / 4 >= 32 * 128, "room for 32 rows");
        constexpr int kWide = S::kTileQ / 4 >= 32 * 256 ? 64 : 32;  // columns that fit as FP32
        auto leave = [&](auto as_half) {
            constexpr bool kHalf = decltype(as_half)::value;
            constexpr int kCols = kHalf ? 64 : kWide, kPitch = kCols * (kHalf ? 2 : 4), kPieces = kPitch / 16, kSwap = kPieces < 8 ? kPieces - 1 : 7;
#pragma unroll 1
            for (int c0 = 0; c0 < D; c0 += kCols) {
                if (ok) {
#pragma unroll
                    for (int c = 0; c < kCols; c += 32) {
                        float v[32];
                        if (mine > 0) {
                            tmem_ld32(o_addr + c0 + c, v);
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; i++) v[i] = 0.f;
                        }
#pragma unroll
                        for (int i = 0; i < 32; i++) v[i] = mul == 0.f ? 0.f : v[i] * mul;
                        // piece p of a row lies at p ^ (row % 8): no two rows' pieces of a phase in the same banks
                        if (kHalf) {
#pragma unroll
                            for (int i = 0; i < 32; i += 8)
                                *reinterpret_cast<uint4*>(stage + lane * kPitch + ((((c + i) >> 3) ^ (lane & kSwap)) << 4)) =
                                    make_uint4(pack_bf16x2(v[i], v[i + 1]), pack_bf16x2(v[i + 2], v[i + 3]), pack_bf16x2(v[i + 4], v[i + 5]),
                                               pack_bf16x2(v[i + 6], v[i + 7]));
                        } else {
#pragma unroll
                            for (int i = 0; i < 32; i += 4)
                                *reinterpret_cast<float4*>(stage + lane * kPitch + ((((c + i) >> 2) ^ (lane & kSwap)) << 4)) =
                                    make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                        }
                    }
                }
                __syncwarp();
                // a row's pieces by neighbouring lanes; the row's address from the lane that has the row
                constexpr int kAtOnce = 32 / kPieces;
#pragma unroll
                for (int r0 = 0; r0 < 32; r0 += kAtOnce) {
                    const int row = r0 + lane / kPieces, piece = lane % kPieces;
                    const long long to = __shfl_sync(0xffffffffu, here && ok ? (long long)R : -1ll, row);
                    const uint4 x = *reinterpret_cast<const uint4*>(stage + row * kPitch + ((piece ^ (row & kSwap)) << 4));
                    if (to < 0) continue;
                    if (kHalf) *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + to * D + c0 + piece * 8) = x;
                    else if (direct) *reinterpret_cast<uint4*>(static_cast<float*>(a.out) + to * D + c0 + piece * 4) = x;
                    else *reinterpret_cast<uint4*>(a.rec.o + ((size_t)slot * a.rec.rows + to) * D + c0 + piece * 4) = x;
                }
                __syncwarp();
            }
        };
        if (direct && a.io_bf16) leave(std::true_type());
        else leave(std::false_type());
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 8) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// ---- host --------------------------------------------------------------------------------------

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

template <int D>
static int launch_tc(const TcArgs& ta, const void* maps, int grid, int pair, cudaStream_t stream)
{
    static bool ready[64];
    const int dev = ta.a.device;
    if (dev < 0 || dev >= 64) return (int)cudaErrorInvalidDevice;
    cudaError_t e;
    if (!ready[dev]) {
        // a register split above the launch's registers would never be granted
        cudaFuncAttributes fa;
        e = cudaFuncGetAttributes(&fa, pages_tc_kernel<D>);
        if (e != cudaSuccess) return (int)e;
        if (fa.numRegs != kLaunchRegs || fa.maxThreadsPerBlock < kTcThreads) return (int)cudaErrorInvalidConfiguration;
        e = cudaFuncSetAttribute(pages_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)Smem<D>::kBytes);
        if (e != cudaSuccess) return (int)e;
        ready[dev] = true;
    }
    const CUtensorMap* m = static_cast<const CUtensorMap*>(maps);
    return launch_after_in(pair, pages_tc_kernel<D>, dim3(grid), kTcThreads, Smem<D>::kBytes, stream, m[0], m[1], ta);
}

int tc_launch(const AttnArgs& a, int layer, bool tall, bool shared_pass, bool beside, int items, const void* maps, cudaStream_t stream)
{
    TcArgs ta;
    ta.a = a;
    ta.layer = layer;
    ta.tall = tall;
    ta.shared_pass = shared_pass;
    ta.wait_ns = tyb_wait_limit_of(a.device);
    ta.row_tiles = items;
    // Beside the own rows in pairs, which lie on the two SMs of a TPC: one of these CTAs and one of the streaming form's
    // on the two slowed the latter (256 questions: the run there took 68 us on average, the others 53).
    const int pair = beside ? 2 : 1, ctas = items * a.p.kv_heads * a.splits, grid = (ctas + pair - 1) / pair * pair;
    return a.p.head_dim == 128 ? launch_tc<128>(ta, maps, grid, pair, stream) : launch_tc<64>(ta, maps, grid, pair, stream);
}

}  // namespace tyb

using namespace tyb;

extern "C" int tyb_pages_maps(const KVPages* p, void* maps)
{
    static EncodeTiledFn fn = nullptr;
    if (!fn) {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
            return (int)cudaErrorNotSupported;
        fn = reinterpret_cast<EncodeTiledFn>(f);
    }
    // Every row of every layer, page and head.  K, V: as a 2-D tensor, a box is 128 bytes of a page's rows (at most a
    // stage's).  For the streaming form as a 3-D one, columns in a box by rows by column boxes: K, V with boxes of those
    // rows, all their columns where they fill a stage; K, V with boxes of 16 rows by 128 bytes.
    const bool bf16 = p->kv_dtype == TYB_BF16;
    const cuuint32_t cols = bf16 ? 64 : 32, boxes = (cuuint32_t)p->head_dim / cols, rows = (cuuint32_t)box_rows(*p);
    const cuuint64_t all = (cuuint64_t)p->num_layers * p->num_pages * p->kv_heads * p->page_size, pitch = (cuuint64_t)p->head_dim * (bf16 ? 2 : 4);
    const cuuint64_t dims2[2] = {(cuuint64_t)p->head_dim, all}, dims3[3] = {cols, all, boxes}, strides[2] = {pitch, 128};
    const cuuint32_t estr[3] = {1, 1, 1}, box[3][3] = {{cols, rows, 1}, {cols, rows, rows == (bf16 ? 64u : 32u) ? boxes : 1u}, {cols, 16, 1}};
    for (int i = 0; i < 6; i++)
        if (fn(static_cast<CUtensorMap*>(maps) + i, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, i < 2 ? 2 : 3,
               i & 1 ? p->v : p->k, i < 2 ? dims2 : dims3, strides, box[i / 2], estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return (int)cudaErrorInvalidValue;
    return 0;
}

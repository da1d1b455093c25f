// pages_mma.cuh -- a few query rows of one warp against key tiles in shared memory, on warp-level matrix
// products (mma.sync): the running softmax and output of pages_stream.cu.  Tiles lie as TMA writes them
// with the 128-byte swizzle: boxes of 128-byte rows, 16-byte chunks XORed with row % 8.
//
// Few rows meet many keys, so the keys (and in P.V the head dimensions) are the 16 rows of the product and
// the queries its 8 columns: S^T = K Q^T, O^T = V^T P^T.  A product costs the same whether its columns are
// used or not, and for at most four query rows the other four columns carry what would be a second product:
//   BF16  the weights' remainders: columns 0-3 of P^T the weights rounded to BF16, columns 4-7 what that
//         left (the queries are repeated, so those lanes have the scores as well); O is the columns' sum.
//         So the only roundings are the operands' own and the output's.
//   FP32  the TF32 remainders: x = hi + lo in every operand; columns 0-3 of Q^T and P^T hi, 4-7 lo; two
//         products (hi and lo of K or V) give all four terms.  A relative error of about 2^-21 per product.
// That makes 32 products for 32 BF16 keys of 128 dimensions, against 96 of the usual form (queries as rows,
// remainders by a second product): mma.sync issues one per 16 cycles here, and the usual form was bound by it.
#pragma once

#include "pages_attn.cuh"

namespace tyb {

__device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ float lo_of(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float hi_of(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }

__device__ __forceinline__ void mma_bf16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1)
{
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// x = hi + lo in TF32 to within 2^-22 |x|: hi the leading 11 significant bits, lo the exact rest, rounded (to nearest,
// by half a unit of the last bit that the product reads: it ignores the 13 below).  In integer and FP32 operations of
// full rate; the conversions to TF32 have a fraction of it.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo)
{
    hi = __float_as_uint(x) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi)) + 0x1000u;
}

__device__ __forceinline__ void ldsm(uint32_t (&r)[4], uint32_t at)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t (&r)[4], uint32_t at)
{
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(at)
                 : "memory");
}

// The 8x8 matrix of 16-bit values whose row g lane (g, t) has columns 2 t, 2 t + 1 of, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x)
{
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

// Four finished output values at element `at`.
__device__ __forceinline__ void put_out(const AttnArgs& a, size_t at, float4 x, float l)
{
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (a.io_bf16)
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + at) = make_uint2(pack2(x.x * inv, x.y * inv), pack2(x.z * inv, x.w * inv));
    else
        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
}

// What a tile's keys look like to rows that all see the same: bit i, key i.
template <int kKeys>
struct SameSight {
    unsigned int see;
    __device__ __forceinline__ bool all() const { return see == 0xffffffffu >> (32 - kKeys); }
    __device__ __forceinline__ bool operator()(int, int, int i) const { return see >> i & 1u; }
};

// Column q of block n of the products is query row 8 n + q; with kDup (rows up to 4, one block) columns 4-7
// are rows 0-3 again.  Lane (g, t) = (lane / 4, lane % 4).
// O^T fragments: o[n][i][c] is dimension 16 i + g + 8 (c / 2) of column 2 t + c % 2; statistics per column.
template <int D, int kBlocks, bool kDup>
struct Running {
    float o[kBlocks][D / 16][4];
    float m[kBlocks][2], l[kBlocks][2];

    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int n = 0; n < kBlocks; n++) {
#pragma unroll
            for (int i = 0; i < D / 16; i++) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
            m[n][0] = m[n][1] = -INFINITY;
            l[n][0] = l[n][1] = 0.f;
        }
    }

    // Scores s[n][e][c] (key 16 e + g + 8 (c / 2) of column 2 t + c % 2) become weights.  sight.all(): every key
    // is in sight of every row; else sight(n, c, i): key i is in sight of column 2 t + c of block n.
    template <int E, typename Sight>
    __device__ __forceinline__ void weigh(float (&s)[kBlocks][E][4], const Sight& sight, float scale, int g)
    {
        if (!sight.all()) {
#pragma unroll
            for (int e = 0; e < E; e++)
#pragma unroll
                for (int hf = 0; hf < 2; hf++)
#pragma unroll
                    for (int n = 0; n < kBlocks; n++)
#pragma unroll
                        for (int c = 0; c < 2; c++)
                            if (!sight(n, c, 16 * e + g + 8 * hf)) s[n][e][2 * hf + c] = -INFINITY;
        }
        float top[kBlocks][2];
        bool rise = false;
#pragma unroll
        for (int n = 0; n < kBlocks; n++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                float x = fmaxf(s[n][0][c], s[n][0][2 + c]);
#pragma unroll
                for (int e = 1; e < E; e++) x = fmaxf(x, fmaxf(s[n][e][c], s[n][e][2 + c]));
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
                top[n][c] = fmaxf(m[n][c], x * scale);
                rise |= top[n][c] > m[n][c];
            }
        if (__any_sync(0xffffffffu, rise)) {
#pragma unroll
            for (int n = 0; n < kBlocks; n++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    const float f = m[n][c] == -INFINITY ? 0.f : fast_exp2(m[n][c] - top[n][c]);
                    l[n][c] *= f;
                    m[n][c] = top[n][c];
#pragma unroll
                    for (int i = 0; i < D / 16; i++) {
                        o[n][i][c] *= f;
                        o[n][i][2 + c] *= f;
                    }
                }
        }
#pragma unroll
        for (int n = 0; n < kBlocks; n++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const float neg = m[n][c] == -INFINITY ? 0.f : -m[n][c];
#pragma unroll
                for (int e = 0; e < E; e++)
#pragma unroll
                    for (int hf = 0; hf < 2; hf++) {
                        float& x = s[n][e][2 * hf + c];
                        x = fast_exp2(fmaf(x, scale, neg));
                        l[n][c] += x;
                    }
            }
    }

    // The warp's rows, to be joined: output rows at rows[r * pitch], statistics at ml[r].
    __device__ __forceinline__ void put(float* rows, int pitch, float2* ml, int nrows, int g, int t)
    {
#pragma unroll
        for (int n = 0; n < kBlocks; n++)
#pragma unroll
            for (int c = 0; c < 2; c++) {
#pragma unroll
                for (int d = 4; d < 32; d <<= 1) l[n][c] += __shfl_xor_sync(0xffffffffu, l[n][c], d);
                const int row = 8 * n + 2 * t + c;
                if (g == 0 && row < nrows) ml[row] = make_float2(m[n][c], l[n][c]);
#pragma unroll
                for (int i = 0; i < D / 16; i++)
#pragma unroll
                    for (int hf = 0; hf < 2; hf++) {
                        float x = o[n][i][2 * hf + c];
                        if (kDup) x += __shfl_xor_sync(0xffffffffu, x, 2);
                        if (row < nrows) rows[row * pitch + 16 * i + g + 8 * hf] = x;
                    }
            }
    }
};

template <typename T, int D, int kBlocks, bool kDup>
struct Rows;

template <int D, int kBlocks, bool kDup>
struct Rows<__nv_bfloat16, D, kBlocks, kDup> : Running<D, kBlocks, kDup> {
    uint32_t q[kBlocks][D / 16][2];

    // n >= 1 query rows at `at` (shared memory, [n][D] BF16 or FP32); further columns repeat the last one:
    // theirs are results that nobody takes.
    __device__ __forceinline__ void load_q(const unsigned char* at, int n, bool bf16, int g, int t, float*, int, int)
    {
#pragma unroll
        for (int b = 0; b < kBlocks; b++) {
            const int first = min(8 * b + (kDup ? g & 3 : g), n - 1) * D + 2 * t;
            if (bf16) {
#pragma unroll
                for (int k = 0; k < D / 16; k++)
#pragma unroll
                    for (int i = 0; i < 2; i++) q[b][k][i] = *reinterpret_cast<const uint32_t*>(at + (first + 16 * k + 8 * i) * 2);
            } else {
#pragma unroll
                for (int k = 0; k < D / 16; k++)
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        const float2 f = *reinterpret_cast<const float2*>(at + (first + 16 * k + 8 * i) * 4);
                        q[b][k][i] = pack2(f.x, f.y);
                    }
            }
        }
    }

    // Rows r0 .. r0 + 32 of the tile.
    template <typename Sight>
    __device__ __forceinline__ void step(const unsigned char* kt, const unsigned char* vt, int box, int r0, const Sight& see, float scale,
                                         const float*, int g, int t, int lane)
    {
        float s[kBlocks][2][4];
#pragma unroll
        for (int b = 0; b < kBlocks; b++)
#pragma unroll
            for (int e = 0; e < 2; e++) s[b][e][0] = s[b][e][1] = s[b][e][2] = s[b][e][3] = 0.f;
        {
            const int row = r0 + (lane & 15), half = lane >> 4;
            const uint32_t at = smem_u32(kt) + row * 128;
#pragma unroll
            for (int k = 0; k < D / 16; k++) {
                const int chunk = 2 * k + half;
                const uint32_t off = at + (chunk >> 3) * box + (((chunk & 7) ^ (row & 7)) << 4);
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    uint32_t x[4];
                    ldsm(x, off + e * 16 * 128);
#pragma unroll
                    for (int b = 0; b < kBlocks; b++) mma_bf16(s[b][e], x, q[b][k][0], q[b][k][1]);
                }
            }
        }
        this->template weigh<2>(s, see, scale, g);
        const int row = r0 + (lane & 7) + (lane >> 4) * 8, half = lane >> 3 & 1;
        const uint32_t at = smem_u32(vt) + row * 128;
#pragma unroll
        for (int e = 0; e < 2; e++) {  // 16 keys
            uint32_t h[kBlocks][2], r[kBlocks][2];
#pragma unroll
            for (int b = 0; b < kBlocks; b++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const float x = s[b][e][2 * i], y = s[b][e][2 * i + 1];
                    h[b][i] = pack2(x, y);
                    r[b][i] = pack2(x - lo_of(h[b][i]), y - hi_of(h[b][i]));
                    if (kDup) h[b][i] = t < 2 ? h[b][i] : r[b][i];
                    h[b][i] = transpose8(h[b][i]);
                    if (!kDup) r[b][i] = transpose8(r[b][i]);
                }
#pragma unroll
            for (int i = 0; i < D / 16; i++) {
                const int chunk = 2 * i + half;
                uint32_t x[4];
                ldsm_t(x, at + e * 16 * 128 + (chunk >> 3) * box + (((chunk & 7) ^ (row & 7)) << 4));
#pragma unroll
                for (int b = 0; b < kBlocks; b++) {
                    mma_bf16(this->o[b][i], x, h[b][0], h[b][1]);
                    if (!kDup) mma_bf16(this->o[b][i], x, r[b][0], r[b][1]);
                }
            }
        }
    }
};

template <int D, int kBlocks, bool kDup>
struct Rows<float, D, kBlocks, kDup> : Running<D, kBlocks, kDup> {
    static constexpr int kPitch = D + 4;
    uint32_t q[kDup ? D / 8 : 1][2];  // kDup: hi of rows 0-3 in columns 0-3, lo in columns 4-7

    // The rows as TF32 halves: into registers (kDup), or by `threads` threads together into `split` (hi, then
    // lo: [8 kBlocks][kPitch] each).
    __device__ __forceinline__ void load_q(const unsigned char* at, int n, bool bf16, int g, int t, float* split, int tid, int threads)
    {
        auto value = [&](int row, int c) {
            const int i = min(row, n - 1) * D + c;
            return bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(at)[i]) : reinterpret_cast<const float*>(at)[i];
        };
        if constexpr (kDup) {
#pragma unroll
            for (int k = 0; k < D / 8; k++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    uint32_t hi, lo;
                    split_tf32(value(g & 3, 8 * k + 4 * i + t), hi, lo);
                    q[k][i] = g < 4 ? hi : lo;
                }
        } else {
            for (int i = tid; i < 8 * kBlocks * D; i += threads) {
                const int row = i / D, c = i % D;
                uint32_t hi, lo;
                split_tf32(value(row, c), hi, lo);
                split[row * kPitch + c] = __uint_as_float(hi);
                split[(8 * kBlocks + row) * kPitch + c] = __uint_as_float(lo);
            }
        }
    }

    // Rows r0 .. r0 + 16 of the tile.
    template <typename Sight>
    __device__ __forceinline__ void step(const unsigned char* kt, const unsigned char* vt, int box, int r0, const Sight& see, float scale,
                                         const float* split, int g, int t, int lane)
    {
        // The terms hi.hi, lo.hi and hi.lo in accumulators of their own: shorter chains, and the small terms are not
        // rounded away one by one.
        float s[kBlocks][1][4], s2[kBlocks][4], s3[kBlocks][4];
#pragma unroll
        for (int b = 0; b < kBlocks; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[b][0][i] = s2[b][i] = s3[b][i] = 0.f;
        {
            const int row = r0 + (lane & 15), half = lane >> 4;
            const uint32_t at = smem_u32(kt) + row * 128;
            const uint32_t* qh = reinterpret_cast<const uint32_t*>(split) + g * kPitch + t;
#pragma unroll
            for (int k = 0; k < D / 8; k++) {
                const int chunk = 2 * k + half;
                uint32_t x[4], hi[4], lo[4];
                ldsm(x, at + (chunk >> 3) * box + (((chunk & 7) ^ (row & 7)) << 4));
#pragma unroll
                for (int i = 0; i < 4; i++) split_tf32(__uint_as_float(x[i]), hi[i], lo[i]);
#pragma unroll
                for (int b = 0; b < kBlocks; b++) {
                    if constexpr (kDup) {
                        mma_tf32(s[b][0], hi, q[k][0], q[k][1]);
                        mma_tf32(s2[b], lo, q[k][0], q[k][1]);
                    } else {
                        const uint32_t* p = qh + 8 * b * kPitch + 8 * k;
                        const uint32_t h0 = p[0], h1 = p[4], l0 = p[8 * kBlocks * kPitch], l1 = p[8 * kBlocks * kPitch + 4];
                        mma_tf32(s[b][0], hi, h0, h1);
                        mma_tf32(s2[b], lo, h0, h1);
                        mma_tf32(s3[b], hi, l0, l1);
                    }
                }
            }
        }
#pragma unroll
        for (int b = 0; b < kBlocks; b++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[b][0][i] += s2[b][i] + s3[b][i];
                if (kDup) s[b][0][i] += __shfl_xor_sync(0xffffffffu, s[b][0][i], 2);  // the columns of hi and of lo
            }
        this->template weigh<1>(s, see, scale, g);
        // P^T as the products' second operand: lane (g, t) has column g of keys 2 t and 2 t + 1 (of 8; the
        // order of the keys is the same in V^T).
        uint32_t ph[kBlocks][2][2], pl[kBlocks][2][2];
#pragma unroll
        for (int b = 0; b < kBlocks; b++)
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int from = (2 * t + i) * 4 + (g >> 1);
                    const float x = __shfl_sync(0xffffffffu, s[b][0][2 * e], from), y = __shfl_sync(0xffffffffu, s[b][0][2 * e + 1], from);
                    split_tf32(g & 1 ? y : x, ph[b][e][i], pl[b][e][i]);
                    if (kDup && g >= 4) ph[b][e][i] = pl[b][e][i];
                }
        const unsigned char* v0 = vt + (r0 + 2 * t) * 128 + (g & 3) * 4;
#pragma unroll
        for (int i = 0; i < D / 16; i++) {
            // The tile's contribution in accumulators of its own, joined by an FP32 addition: the tensor core's
            // own sums round towards zero, which over thousands of keys would add up.
            float x[kBlocks][4], y[kBlocks][4];
#pragma unroll
            for (int b = 0; b < kBlocks; b++)
#pragma unroll
                for (int c = 0; c < 4; c++) x[b][c] = y[b][c] = 0.f;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                uint32_t hi[4], lo[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {  // dimension + 8 (j & 1), key 2 t + (j >> 1)
                    const int chunk = 4 * i + 2 * (j & 1) + (g >> 2), key = 2 * t + (j >> 1);
                    split_tf32(*reinterpret_cast<const float*>(v0 + (chunk >> 3) * box + (8 * e + (j >> 1)) * 128 + (((chunk & 7) ^ key) << 4)),
                               hi[j], lo[j]);
                }
#pragma unroll
                for (int b = 0; b < kBlocks; b++) {
                    mma_tf32(x[b], hi, ph[b][e][0], ph[b][e][1]);
                    mma_tf32(y[b], lo, ph[b][e][0], ph[b][e][1]);
                    if (!kDup) mma_tf32(y[b], hi, pl[b][e][0], pl[b][e][1]);
                }
            }
#pragma unroll
            for (int b = 0; b < kBlocks; b++)
#pragma unroll
                for (int c = 0; c < 4; c++) this->o[b][i][c] += x[b][c] + y[b][c];
        }
    }
};

}  // namespace tyb

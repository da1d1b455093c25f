// pages_mma.cuh -- 16 query rows of one warp against key tiles in shared memory, on warp-level matrix
// products (mma.sync): the running softmax and output of pages_stream.cu.  Tiles lie as TMA writes
// them with the 128-byte swizzle: boxes of 128-byte rows, 16-byte chunks XORed with row % 8.
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

// x = hi + lo in TF32, the remainder below 2^-22 |x|.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo)
{
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(hi) : "f"(x));
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(lo) : "f"(x - __uint_as_float(hi)));
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

// Four finished output values at element `at`.
__device__ __forceinline__ void put_out(const AttnArgs& a, size_t at, float4 x, float l)
{
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (a.io_bf16)
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(a.out) + at) = make_uint2(pack2(x.x * inv, x.y * inv), pack2(x.z * inv, x.w * inv));
    else
        *reinterpret_cast<float4*>(static_cast<float*>(a.out) + at) = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
}

// Output fragments and statistics; lane (g, t) = (lane / 4, lane % 4) has columns 8 c + 2 t, + 1 of rows g
// (o[c][0..1]) and g + 8 (o[c][2..3]).
template <int D>
struct Running {
    float o[D / 8][4];
    float m[2], l[2];

    __device__ __forceinline__ void clear()
    {
#pragma unroll
        for (int c = 0; c < D / 8; c++) o[c][0] = o[c][1] = o[c][2] = o[c][3] = 0.f;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = 0.f;
    }

    // Scores s[e][..] (keys 8 e + 2 t, + 1 of rows g and g + 8) become weights; bit i of `see`: key i is in
    // sight of the rows.
    template <int E>
    __device__ __forceinline__ void weigh(float (&s)[E][4], unsigned int see, float scale, int t)
    {
        if (see != (1u << (8 * E)) - 1u) {
#pragma unroll
            for (int e = 0; e < E; e++)
#pragma unroll
                for (int r = 0; r < 2; r++)
                    if (!(see >> (8 * e + 2 * t + r) & 1u)) s[e][r] = s[e][2 + r] = -INFINITY;
        }
        float top[2];
#pragma unroll
        for (int r = 0; r < 2; r++) {
            top[r] = fmaxf(s[0][2 * r], s[0][2 * r + 1]);
#pragma unroll
            for (int e = 1; e < E; e++) top[r] = fmaxf(top[r], fmaxf(s[e][2 * r], s[e][2 * r + 1]));
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
            top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
            top[r] = fmaxf(m[r], top[r] * scale);
        }
        if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
#pragma unroll
            for (int r = 0; r < 2; r++) {
                const float f = m[r] == -INFINITY ? 0.f : fast_exp2(m[r] - top[r]);
                l[r] *= f;
                m[r] = top[r];
#pragma unroll
                for (int c = 0; c < D / 8; c++) {
                    o[c][2 * r] *= f;
                    o[c][2 * r + 1] *= f;
                }
            }
        }
        const float neg[2] = {m[0] == -INFINITY ? 0.f : -m[0], m[1] == -INFINITY ? 0.f : -m[1]};
#pragma unroll
        for (int e = 0; e < E; e++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                s[e][r] = fast_exp2(fmaf(s[e][r], scale, neg[r >> 1]));
                l[r >> 1] += s[e][r];
            }
    }

    // The lanes' shares of the row sums.
    __device__ __forceinline__ void finish()
    {
#pragma unroll
        for (int r = 0; r < 2; r++) {
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
            l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        }
    }
};

template <typename T, int D>
struct Rows;

template <int D>
struct Rows<__nv_bfloat16, D> : Running<D> {
    uint32_t q[D / 16][4];

    // n query rows at `at` (shared memory, [n][D] BF16 or FP32; the others are zeros).
    __device__ __forceinline__ void load_q(const unsigned char* at, int n, bool bf16, int g, int t, float*, int, int, int)
    {
#pragma unroll
        for (int k = 0; k < D / 16; k++)
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const int row = g + 8 * (i & 1), c = 16 * k + 8 * (i >> 1) + 2 * t;
                uint32_t x = 0;
                if (row < n) {
                    if (bf16) {
                        x = *reinterpret_cast<const uint32_t*>(at + (row * D + c) * 2);
                    } else {
                        const float2 f = *reinterpret_cast<const float2*>(at + (row * D + c) * 4);
                        x = pack2(f.x, f.y);
                    }
                }
                q[k][i] = x;
            }
    }

    // Rows r0 .. r0 + 16 of the tile.
    __device__ __forceinline__ void step(const unsigned char* kt, const unsigned char* vt, int box, int r0, unsigned int see, float scale,
                                         const float*, int, int t, int lane)
    {
        const uint32_t kb = smem_u32(kt), vb = smem_u32(vt);
        float s[2][4], s2[2][4];
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[e][i] = s2[e][i] = 0.f;
        {
            const int row = r0 + (lane & 7) + (lane >> 4) * 8, half = lane >> 3 & 1;
            const uint32_t at = kb + row * 128;
#pragma unroll
            for (int k = 0; k < D / 16; k++) {
                uint32_t b[4];
                const int chunk = 2 * k + half;
                ldsm(b, at + (chunk >> 3) * box + (((chunk & 7) ^ (row & 7)) << 4));
                mma_bf16(k & 1 ? s2[0] : s[0], q[k], b[0], b[1]);
                mma_bf16(k & 1 ? s2[1] : s[1], q[k], b[2], b[3]);
            }
        }
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int i = 0; i < 4; i++) s[e][i] += s2[e][i];
        this->template weigh<2>(s, see, scale, t);
        uint32_t h[4], r[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float x = s[i >> 1][2 * (i & 1)], y = s[i >> 1][2 * (i & 1) + 1];
            h[i] = pack2(x, y);
            r[i] = pack2(x - lo_of(h[i]), y - hi_of(h[i]));
        }
        const int row = r0 + (lane & 7) + (lane >> 3 & 1) * 8, half = lane >> 4;
        const uint32_t at = vb + row * 128;
#pragma unroll
        for (int c = 0; c < D / 16; c++) {
            uint32_t b[4];
            const int chunk = 2 * c + half;
            ldsm_t(b, at + (chunk >> 3) * box + (((chunk & 7) ^ (row & 7)) << 4));
            mma_bf16(this->o[2 * c], h, b[0], b[1]);
            mma_bf16(this->o[2 * c + 1], h, b[2], b[3]);
            mma_bf16(this->o[2 * c], r, b[0], b[1]);
            mma_bf16(this->o[2 * c + 1], r, b[2], b[3]);
        }
    }
};

template <int D>
struct Rows<float, D> : Running<D> {
    static constexpr int kPitch = D + 4;

    // The rows as TF32 halves into `split` (hi, then lo: [rows][kPitch] each, rows 8 or 16), by `threads`
    // threads together.
    int rows;
    __device__ __forceinline__ void load_q(const unsigned char* at, int n, bool bf16, int, int, float* split, int padded, int tid, int threads)
    {
        rows = padded;
        for (int i = tid; i < rows * D; i += threads) {
            const int row = i / D, c = i % D;
            float x = 0.f;
            if (row < n) x = bf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(at)[row * D + c]) : reinterpret_cast<const float*>(at)[row * D + c];
            uint32_t hi, lo;
            split_tf32(x, hi, lo);
            split[row * kPitch + c] = __uint_as_float(hi);
            split[(rows + row) * kPitch + c] = __uint_as_float(lo);
        }
    }

    // Rows r0 .. r0 + 8 of the tile.
    __device__ __forceinline__ void step(const unsigned char* kt, const unsigned char* vt, int box, int r0, unsigned int see, float scale,
                                         const float* split, int g, int t, int lane)
    {
        const uint32_t kb = smem_u32(kt);
        const uint32_t* qh = reinterpret_cast<const uint32_t*>(split) + g * kPitch + t;
        const uint32_t* ql = qh + rows * kPitch;
        const int low = rows == 16 ? 8 * kPitch : 0;  // of 8 rows, g + 8 repeats g: not used
        // hi.hi and the cross terms in accumulators of their own: shorter chains, and the small terms are
        // not rounded away one by one
        float c0[4] = {}, c1[4] = {}, c2[4] = {};
        const int row = r0 + (lane & 7);
#pragma unroll
        for (int k = 0; k < D / 16; k++) {
            uint32_t b[4];
            const int chunk = 4 * k + (lane >> 3);
            ldsm(b, kb + (chunk >> 3) * box + row * 128 + (((chunk & 7) ^ (row & 7)) << 4));
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int d = 16 * k + 8 * u;
                const uint32_t ah[4] = {qh[d], qh[d + low], qh[d + 4], qh[d + 4 + low]};
                const uint32_t al[4] = {ql[d], ql[d + low], ql[d + 4], ql[d + 4 + low]};
                uint32_t bh[2], bl[2];
                split_tf32(__uint_as_float(b[2 * u]), bh[0], bl[0]);
                split_tf32(__uint_as_float(b[2 * u + 1]), bh[1], bl[1]);
                mma_tf32(c0, ah, bh[0], bh[1]);
                mma_tf32(c1, al, bh[0], bh[1]);
                mma_tf32(c2, ah, bl[0], bl[1]);
            }
        }
        float s[1][4];
#pragma unroll
        for (int i = 0; i < 4; i++) s[0][i] = c0[i] + (c1[i] + c2[i]);
        this->template weigh<1>(s, see, scale, t);
        // columns k = t and t + 4 of the P operand are keys 2 t and 2 t + 1
        uint32_t ph[4], pl[4];
        split_tf32(s[0][0], ph[0], pl[0]);
        split_tf32(s[0][2], ph[1], pl[1]);
        split_tf32(s[0][1], ph[2], pl[2]);
        split_tf32(s[0][3], ph[3], pl[3]);
        const int v0 = r0 + 2 * t, v1 = v0 + 1;
#pragma unroll
        for (int c = 0; c < D / 8; c++) {
            const int chunk = 2 * c + (g >> 2);
            const unsigned char* at = vt + (chunk >> 3) * box + (g & 3) * 4;
            uint32_t bh[2], bl[2];
            split_tf32(*reinterpret_cast<const float*>(at + v0 * 128 + (((chunk & 7) ^ (v0 & 7)) << 4)), bh[0], bl[0]);
            split_tf32(*reinterpret_cast<const float*>(at + v1 * 128 + (((chunk & 7) ^ (v1 & 7)) << 4)), bh[1], bl[1]);
            // The tile's contribution in an accumulator of its own, joined by an FP32 addition: the tensor
            // core's own sums round towards zero, which over thousands of keys would add up.
            float x[4] = {};
            mma_tf32(x, pl, bh[0], bh[1]);
            mma_tf32(x, ph, bl[0], bl[1]);
            mma_tf32(x, ph, bh[0], bh[1]);
#pragma unroll
            for (int i = 0; i < 4; i++) this->o[c][i] += x[i];
        }
    }
};

}  // namespace tyb

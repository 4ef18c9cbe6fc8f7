// Decode attention over the 4-bit paged cache (kv4.cuh), one query position per take, optionally with the newest
// position's rope, quantisation and cache write in the same launch.
//
// The mathematics. With value = s n + z for each group of 32 channels,
//   score_j = sum_g s_jg (q . n_j)_g + sum_g z_jg Q_g,    Q_g = the sum of q over group g,
//   out     = [ sum_j (p_j s_jg) n_jc + sum_j p_j z_jg ] / sum_j p_j    for channel c of group g,
// so the matrix instructions multiply by the codes themselves: fp16 subnormals n 2^-24, exact, masked out of the
// packed words. q is scaled by a power of two of its own for each head so that it is exact in fp16; the zeros' term of
// the scores is one more instruction, bf16 zeros times Q split into three bf16 parts (24 bits). p_j s_jg is rounded to
// fp16 (2^-12 relative): its running reference M keeps the largest near 2^10, far from fp16's limits at both ends,
// and moves only when a product passes 2^15. Sums, p, the zeros' term of the output and M are fp32.
// The tensor cores cut their sums off instead of rounding them, a bias that grows with the number of positions while
// the result, an average of values of either sign, shrinks: codes 0..15 of one sign left 6e-3 relative error at 65536
// positions. So an odd position's value is taken as s (n - 15) + (z + 15 s): the codes of even and odd positions then
// have opposite signs and the sums stay near the size of the result (1.7e-3, the rounding of the bf16 output).
#pragma once
#include "common.cuh"
#include "kv4.cuh"

namespace d4 {

using kv4::Fmt;
using kv4::HALF;
using kv4::Words;

constexpr int GMAX = 8;      // q heads per kv head handled by one mma column block
constexpr float SMIN = 8.6736174e-19f;  // 2^-60: groups of smaller scale count as this when M is set

__device__ __forceinline__ void mma_f16(float *d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// 8 codes of a word as fp16 pairs: n 2^-24 (even nibbles) and 16 n 2^-24 (odd ones)
__device__ __forceinline__ uint32_t code_even(uint32_t w) { return w & 0x000f000fu; }
__device__ __forceinline__ uint32_t code_odd(uint32_t w) { return w & 0x00f000f0u; }
// The same with the high halves (V: the odd positions) as n - 15
__device__ __forceinline__ uint32_t flip_even(uint32_t w) { return (w & 0x000f000fu) ^ 0x800f0000u; }
__device__ __forceinline__ uint32_t flip_odd(uint32_t w) { return (w & 0x00f000f0u) ^ 0x80f00000u; }

struct Params {
    const bf16 *qkv;
    uint8_t *pool;               // written only by the fused form, at the newest position
    const int *table;
    bf16 *out, *held;            // held: fused form, may be null
    float *part;                 // partial records
    int *cnt;                    // [B * nk], zero between launches
    const int *pos, *lens;
    const float *cos_t, *sin_t;  // fused form: rotary tables, or null (no rope)
    int B, nq, nk, npages, maxpages;
    float sl2;                   // scale * log2(e)
};

// q of one (take, kv head) as B fragments: lane 4g + t holds head g, channels 32w + 8t .. + 7 of every group w, in fp16
// times 2^e (the pairs of odd nibbles also / 16), and the sums of its groups in three bf16 parts.
template <int HD>
struct Query {
    static constexpr int W = Fmt<HD>::W;
    uint32_t q[W][4];
    uint32_t z0, z1;   // B fragment of the zeros' instruction
    float mul0, mul1;  // heads 2t, 2t + 1: raw score -> base-2 logit
    __device__ void load(const Params &P, int s, int kh, int p, int lane) {
        const int g = lane >> 2, t = lane & 3, G = P.nq / P.nk;
        float x[W][8];
        const bf16 *row = P.qkv + static_cast<long>(s) * (P.nq + 2 * P.nk) * HD + (kh * G + g) * HD;
#pragma unroll
        for (int w = 0; w < W; w++) {
            const uint4 u = g < G ? *reinterpret_cast<const uint4 *>(row + 32 * w + 8 * t) : make_uint4(0, 0, 0, 0);
            const uint32_t *v = reinterpret_cast<const uint32_t *>(&u);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 f = unpack_bf16x2(v[i]);
                x[w][2 * i] = f.x;
                x[w][2 * i + 1] = f.y;
            }
        }
        if (P.cos_t) {
#pragma unroll
            for (int w = 0; w < W / 2; w++) {
                const long at = static_cast<long>(p) * (HD / 2) + 32 * w + 8 * t;
#pragma unroll
                for (int i = 0; i < 8; i += 4) {
                    const float4 c = *reinterpret_cast<const float4 *>(P.cos_t + at + i);
                    const float4 sn = *reinterpret_cast<const float4 *>(P.sin_t + at + i);
                    const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {sn.x, sn.y, sn.z, sn.w};
#pragma unroll
                    for (int j = 0; j < 4; j++) {  // the arithmetic and rounding of oumu_rope
                        const float a = x[w][i + j], b = x[w + W / 2][i + j];
                        x[w][i + j] = bf2f(f2bf(a * cc[j] - b * ss[j]));
                        x[w + W / 2][i + j] = bf2f(f2bf(b * cc[j] + a * ss[j]));
                    }
                }
            }
        }
        float mx = 0.f;
#pragma unroll
        for (int w = 0; w < W; w++)
#pragma unroll
            for (int i = 0; i < 8; i++) mx = fmaxf(mx, fabsf(x[w][i]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // the largest |q| of the head lands in [2^14, 2^15): fp16 keeps a bf16 exactly down to 2^-28 of it
        int e = 14 - (static_cast<int>(__float_as_uint(mx) >> 23) - 127);
        e = e > 100 ? 100 : e < -90 ? -90 : e;
        const float f = __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
        float sum[W];
#pragma unroll
        for (int w = 0; w < W; w++) {
            sum[w] = 0.f;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                x[w][i] *= f;
                sum[w] += x[w][i];
            }
            sum[w] += __shfl_xor_sync(0xffffffffu, sum[w], 1);
            sum[w] += __shfl_xor_sync(0xffffffffu, sum[w], 2);
            sum[w] *= 5.9604645e-08f;  // 2^-24, the codes' unit
            q[w][0] = pack_f16x2(x[w][0], x[w][1]);
            q[w][1] = pack_f16x2(x[w][2] * 0.0625f, x[w][3] * 0.0625f);
            q[w][2] = pack_f16x2(x[w][4], x[w][5]);
            q[w][3] = pack_f16x2(x[w][6] * 0.0625f, x[w][7] * 0.0625f);
        }
        // k index of the zeros' instruction: the row's zeros W wide, three times over, against the three parts
        uint32_t part[3][W / 2];
#pragma unroll
        for (int w = 0; w < W; w += 2) {
            float a = sum[w], b = sum[w + 1];
#pragma unroll
            for (int k = 0; k < 3; k++) {
                part[k][w / 2] = pack_bf16x2(a, b);
                const float2 r = unpack_bf16x2(part[k][w / 2]);
                a -= r.x;
                b -= r.y;
            }
        }
        if constexpr (W == 4) {
            z0 = t < 2 ? part[0][t & 1] : part[1][t & 1];
            z1 = t < 2 ? part[2][t & 1] : 0u;
        } else {
            z0 = t == 0 ? part[0][0] : t == 1 ? part[1][0] : t == 2 ? part[2][0] : 0u;
            z1 = 0u;
        }
        const float m = __uint_as_float(static_cast<uint32_t>(24 - e + 127) << 23) * P.sl2;
        mul0 = __shfl_sync(0xffffffffu, m, 8 * t);
        mul1 = __shfl_sync(0xffffffffu, m, 8 * t + 4);
    }
};

// The running state of one (take, kv head): lane 4g + t holds heads 2t and 2t + 1.
template <int HD>
struct State {
    static constexpr int W = Fmt<HD>::W;
    float M[2], l[2];          // reference exponent; this lane's positions' share of the sum
    float acc[2 * W][4];       // numerator / 2^24 of channels 32w + 4g + {0 | 1 (x 16)}, {2 | 3 (x 16)}
    float z[W][2];             // this lane's positions' share of the zeros' term
    __device__ void clear() {
        M[0] = M[1] = -INFINITY;
        l[0] = l[1] = 0.f;
#pragma unroll
        for (int i = 0; i < 2 * W; i++) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
#pragma unroll
        for (int w = 0; w < W; w++) z[w][0] = z[w][1] = 0.f;
    }

    // One tile of 32 positions at `half`, the first `n` of them valid (what lies behind is never used: its codes are
    // finite whatever they hold, its scales and zeros are replaced).
    __device__ __forceinline__ void tile(const uint8_t *half, int n, const Query<HD> &Q, int lane) {
        using F = Fmt<HD>;
        const int g = lane >> 2, t = lane & 3;
        const float c15 = g & 1 ? 15.f : 0.f;
        float x[2][4];
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const Words<W> k0 = kv4::ld_words<W>(half + (2 * h) * F::BLOCK + lane * 4 * W);
            const Words<W> k1 = kv4::ld_words<W>(half + (2 * h + 1) * F::BLOCK + lane * 4 * W);
            const Words<W> m0 = kv4::ld_words<W>(half + F::KMETA + (16 * h + g) * F::ROW);
            const Words<W> m1 = kv4::ld_words<W>(half + F::KMETA + (16 * h + 8 + g) * F::ROW);
            float d[4] = {0.f, 0.f, 0.f, 0.f};
            const uint32_t a0 = W == 4 ? (t & 1 ? m0.v[W - 1] : m0.v[W / 2]) : m0.v[W - 1];
            const uint32_t a1 = W == 4 ? (t & 1 ? m1.v[W - 1] : m1.v[W / 2]) : m1.v[W - 1];
            mma_bf16_16816(d, a0, a1, a0, a1, Q.z0, Q.z1);
#pragma unroll
            for (int w = 0; w < W; w++) {
                float a[4] = {0.f, 0.f, 0.f, 0.f};
                mma_f16(a, code_even(k0.v[w]), code_even(k1.v[w]), code_odd(k0.v[w]), code_odd(k1.v[w]), Q.q[w][0],
                        Q.q[w][1]);
                mma_f16(a, code_even(k0.v[w] >> 8), code_even(k1.v[w] >> 8), code_odd(k0.v[w] >> 8),
                        code_odd(k1.v[w] >> 8), Q.q[w][2], Q.q[w][3]);
                const float s0 = kv4::row_scale<W>(m0, w), s1 = kv4::row_scale<W>(m1, w);
                d[0] = fmaf(s0, a[0], d[0]);
                d[1] = fmaf(s0, a[1], d[1]);
                d[2] = fmaf(s1, a[2], d[2]);
                d[3] = fmaf(s1, a[3], d[3]);
            }
            x[h][0] = d[0] * Q.mul0;
            x[h][1] = d[1] * Q.mul1;
            x[h][2] = d[2] * Q.mul0;
            x[h][3] = d[3] * Q.mul1;
        }
        Words<W> vm[2][2];
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int r = 0; r < 2; r++) vm[h][r] = kv4::ld_words<W>(half + F::VMETA + (16 * h + 8 * r + g) * F::ROW);
        if (n < HALF) {
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int r = 0; r < 2; r++)
                    if (16 * h + 8 * r + g >= n) {
                        x[h][2 * r] = x[h][2 * r + 1] = -INFINITY;
#pragma unroll
                        for (int i = 0; i < W; i++) vm[h][r].v[i] = 0u;
                    }
        }
        float p[2][4];
        uint32_t pv[2][W][2];
        auto weights = [&]() -> bool {  // p and p s; true where M is too low for them
            uint32_t top = 0;
            float big = 0.f;
#pragma unroll
            for (int h = 0; h < 2; h++) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    p[h][i] = fast_exp2(x[h][i] - M[i & 1]);
                    big = fmaxf(big, p[h][i]);
                }
#pragma unroll
                for (int w = 0; w < W; w++)
#pragma unroll
                    for (int r = 0; r < 2; r++) {
                        const float s = kv4::row_scale<W>(vm[h][r], w);
                        pv[h][w][r] = pack_f16x2(p[h][2 * r] * s, p[h][2 * r + 1] * s);
                        top = __vmaxu2(top, pv[h][w][r]);
                    }
            }
            // 2^15 in fp16 is 0x7800 (infinities and NaN lie above); p itself may reach 2^75 where every scale is tiny
            return (top & 0xffffu) > 0x7800u || top >> 16 > 0x7800u || !(big <= 3.7778932e22f);
        };
        if (__any_sync(0xffffffffu, weights())) {
            rescale(x, vm, lane);
            weights();
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            l[0] += p[h][0] + p[h][2];
            l[1] += p[h][1] + p[h][3];
            const Words<W> v0 = kv4::ld_words<W>(half + F::CODES + (2 * h) * F::BLOCK + lane * 4 * W);
            const Words<W> v1 = kv4::ld_words<W>(half + F::CODES + (2 * h + 1) * F::BLOCK + lane * 4 * W);
#pragma unroll
            for (int w = 0; w < W; w++) {
                const float z0 = fmaf(c15, kv4::row_scale<W>(vm[h][0], w), kv4::row_zero<W>(vm[h][0], w));
                const float z1 = fmaf(c15, kv4::row_scale<W>(vm[h][1], w), kv4::row_zero<W>(vm[h][1], w));
                z[w][0] = fmaf(p[h][0], z0, fmaf(p[h][2], z1, z[w][0]));
                z[w][1] = fmaf(p[h][1], z0, fmaf(p[h][3], z1, z[w][1]));
                const uint32_t b0 = movmatrix_t(pv[h][w][0]), b1 = movmatrix_t(pv[h][w][1]);
                mma_f16(acc[2 * w], flip_even(v0.v[w]), flip_odd(v0.v[w]), flip_even(v1.v[w]), flip_odd(v1.v[w]), b0,
                        b1);
                mma_f16(acc[2 * w + 1], flip_even(v0.v[w] >> 8), flip_odd(v0.v[w] >> 8), flip_even(v1.v[w] >> 8),
                        flip_odd(v1.v[w] >> 8), b0, b1);
            }
        }
    }

    // Raise M so that the largest p s of this tile is 2^10, and bring the sums along. The first tile of a state always
    // comes here (M = -inf); later ones when a logit rises by more than 5 over everything before.
    __device__ __forceinline__ void rescale(const float (&x)[2][4], const Words<W> (&vm)[2][2], int lane) {
        float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int r = 0; r < 2; r++) {
                float s = SMIN;
#pragma unroll
                for (int w = 0; w < W; w++) s = fmaxf(s, kv4::row_scale<W>(vm[h][r], w));
                const float ls = __log2f(s);
                top[0] = fmaxf(top[0], x[h][2 * r] + ls);
                top[1] = fmaxf(top[1], x[h][2 * r + 1] + ls);
            }
#pragma unroll
        for (int c = 0; c < 2; c++) {
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], o));
            float m = fmaxf(M[c], top[c] - 10.f);
            if (m == -INFINITY) m = 0.f;
            const float f = fast_exp2(M[c] - m);
            M[c] = m;
            l[c] *= f;
#pragma unroll
            for (int i = 0; i < 2 * W; i++) {
                acc[i][c] *= f;
                acc[i][c + 2] *= f;
            }
#pragma unroll
            for (int w = 0; w < W; w++) z[w][c] *= f;
        }
    }

    // The state as a record: m[8], l[8], o[8][HD] (o with the zeros' term, in the values' own unit).
    __device__ __forceinline__ void record(float *R, int lane) {
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) {
                l[c] += __shfl_xor_sync(0xffffffffu, l[c], o);
#pragma unroll
                for (int w = 0; w < W; w++) z[w][c] += __shfl_xor_sync(0xffffffffu, z[w][c], o);
            }
        if (g == 0) {
            R[2 * t] = M[0];
            R[2 * t + 1] = M[1];
            R[GMAX + 2 * t] = l[0];
            R[GMAX + 2 * t + 1] = l[1];
        }
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int w = 0; w < W; w++) {
                const float u = 16777216.f, u16 = 1048576.f;  // 2^24, and / 16 for the odd nibbles
                *reinterpret_cast<float4 *>(R + 2 * GMAX + (2 * t + c) * HD + 32 * w + 4 * g) =
                    make_float4(fmaf(acc[2 * w][c], u, z[w][c]), fmaf(acc[2 * w][c + 2], u16, z[w][c]),
                                fmaf(acc[2 * w + 1][c], u, z[w][c]), fmaf(acc[2 * w + 1][c + 2], u16, z[w][c]));
            }
    }
};

// Fused form: the newest position's k (rotated) and v, quantised by one warp into position p of the take's cache, in
// global memory and in `tile`, the copy of that half in shared memory (null: none). Lane l has channels 4l .. 4l + 3.
template <int HD>
__device__ __forceinline__ void newest(const Params &P, int s, int kh, int p, int lane, uint8_t *half, uint8_t *tile) {
    using F = Fmt<HD>;
    constexpr int W = F::W;
    const bool on = lane < HD / 4;
    const int w = lane >> 3, j = lane & 7, r = p % HALF, c4 = 4 * (on ? lane : 0);
    const bf16 *row = P.qkv + static_cast<long>(s) * (P.nq + 2 * P.nk) * HD;
#pragma unroll
    for (int kv = 0; kv < 2; kv++) {
        const uint2 u = *reinterpret_cast<const uint2 *>(row + (P.nq + kv * P.nk + kh) * HD + c4);
        float2 a = unpack_bf16x2(u.x), b = unpack_bf16x2(u.y);
        float x[4] = {a.x, a.y, b.x, b.y};
        if (kv == 0 && P.cos_t) {
            const int i = c4 % (HD / 2);
            const float4 c = *reinterpret_cast<const float4 *>(P.cos_t + static_cast<long>(p) * (HD / 2) + i);
            const float4 sn = *reinterpret_cast<const float4 *>(P.sin_t + static_cast<long>(p) * (HD / 2) + i);
            const float cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {sn.x, sn.y, sn.z, sn.w};
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; e++) y[e] = __shfl_xor_sync(0xffffffffu, x[e], HD / 8);
#pragma unroll
            for (int e = 0; e < 4; e++)  // low half: a c - b s; high half: b c + a s
                x[e] = bf2f(f2bf(c4 < HD / 2 ? x[e] * cc[e] - y[e] * ss[e] : x[e] * cc[e] + y[e] * ss[e]));
        }
        const uint32_t u0 = pack_bf16x2(x[0], x[1]), u1 = pack_bf16x2(x[2], x[3]);
        uint32_t rg = kv4::range_of(kv4::as_u32(__hmax2_nan(kv4::as_bf2(u0), kv4::as_bf2(u1))),
                                    kv4::as_u32(__hmin2_nan(kv4::as_bf2(u0), kv4::as_bf2(u1))));
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) rg = kv4::range_max(rg, __shfl_xor_sync(0xffffffffu, rg, o));
        const kv4::Quant q = kv4::quant_of(rg);
        uint32_t n[4];
#pragma unroll
        for (int e = 0; e < 4; e++) n[e] = kv4::quant_code(x[e], q);
        if (P.held && on) {
            uint2 o;
            o.x = pack_bf16x2(fmaf(q.s, n[0], q.z), fmaf(q.s, n[1], q.z));
            o.y = pack_bf16x2(fmaf(q.s, n[2], q.z), fmaf(q.s, n[3], q.z));
            *reinterpret_cast<uint2 *>(P.held + (static_cast<long>(s) * 2 * P.nk + kv * P.nk + kh) * HD + c4) = o;
        }
        // K: this lane's codes are two bytes of the word of lanes (j, j ^ 1); V: one half of a word
        uint32_t kw = (n[0] | n[2] << 4 | (n[1] | n[3] << 4) << 16) << (8 * (j & 1));
        kw |= __shfl_xor_sync(0xffffffffu, kw, 1);
        const int at = kv == 0 ? r / 8 * F::BLOCK + ((r % 8 * 4 + j / 2) * W + w) * 4
                               : F::CODES + r / 8 * F::BLOCK + ((j * 4 + r % 8 / 2) * W + w) * 4 + 2 * (r & 1);
        const int meta = (kv ? F::VMETA : F::KMETA) + r * F::ROW + 2 * w;
#pragma unroll
        for (int k = 0; k < 2; k++) {
            uint8_t *base = k ? tile : half;
            if (!base || !on) continue;
            if (kv) *reinterpret_cast<uint16_t *>(base + at) = static_cast<uint16_t>(n[0] | n[1] << 4 | n[2] << 8 | n[3] << 12);
            else if (!(j & 1)) *reinterpret_cast<uint32_t *>(base + at) = kw;
            if (j == 0) {
                *reinterpret_cast<uint16_t *>(base + meta) = static_cast<uint16_t>(__float_as_uint(q.s) >> 16);
                *reinterpret_cast<uint16_t *>(base + meta + 2 * W) = static_cast<uint16_t>(__float_as_uint(q.z) >> 16);
            }
        }
    }
}

// Length of take s: lens[s] or *pos + 1, cut to what its table row can hold (recorded).
__device__ __forceinline__ int take_len(const Params &P, int s) {
    int L = P.lens ? P.lens[s] : *P.pos + 1;
    const int room = P.maxpages * kv4::PAGE;
    if (L < 0 || L > room) {
        record_error(OUMU_DEVERR_LENGTH);
        L = L < 0 ? 0 : room;
    }
    return L;
}

constexpr int NW = 8;  // warps of a CTA

// One CTA per (take, kv head): its warps take the tiles in turn, each with a state of its own, merged at the end.
template <int HD, bool FUSED>
__global__ void __launch_bounds__(NW * 32) k_attn_decode_kv4(Params P) {
    using F = Fmt<HD>;
    constexpr int REC = 2 * GMAX + GMAX * HD;
    extern __shared__ __align__(16) float recs[];
    const int s = blockIdx.x / P.nk, kh = blockIdx.x % P.nk, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int G = P.nq / P.nk;
    pdl_trigger();
    pdl_wait();
    const int L = take_len(P, s);
    bf16 *out = P.out + (static_cast<long>(s) * P.nq + kh * G) * HD;
    if (L == 0) {
        for (int i = threadIdx.x; i < G * HD; i += NW * 32) out[i] = f2bf(0.f);
        if (FUSED && P.held)
            for (int i = threadIdx.x; i < 2 * HD; i += NW * 32)
                P.held[(static_cast<long>(s) * 2 * P.nk + i / HD * P.nk + kh) * HD + i % HD] = f2bf(0.f);
        return;
    }
    Query<HD> Q;
    Q.load(P, s, kh, L - 1, lane);
    State<HD> S;
    S.clear();
    const int tiles = (L + HALF - 1) / HALF;
    for (int j = warp; j < tiles; j += NW) {
        int page = P.table[static_cast<long>(s) * P.maxpages + j / 2];
        if (page < 0 || page >= P.npages) {
            if (lane == 0) record_error(OUMU_DEVERR_PAGE);
            continue;
        }
        uint8_t *half = P.pool + (static_cast<long>(page) * P.nk + kh) * F::UNIT + (j & 1) * F::HALFB;
        if (FUSED && j == tiles - 1) {
            newest<HD>(P, s, kh, L - 1, lane, half, nullptr);
            __syncwarp();
        }
        S.tile(half, L - j * HALF, Q, lane);
    }
    S.record(recs + warp * REC, lane);
    __syncthreads();
    for (int i = threadIdx.x; i < G * HD; i += NW * 32) {
        const int h = i / HD;
        float M = -INFINITY, l = 0.f, o = 0.f;
        for (int w = 0; w < NW; w++) M = fmaxf(M, recs[w * REC + h]);
        for (int w = 0; w < NW; w++) {
            const float m = recs[w * REC + h];
            const float f = m == -INFINITY ? 0.f : fast_exp2(m - M);
            l = fmaf(f, recs[w * REC + GMAX + h], l);
            o = fmaf(f, recs[w * REC + 2 * GMAX + i], o);
        }
        out[i] = f2bf(l > 0.f || l != l ? o / l : 0.f);
    }
}

}  // namespace d4

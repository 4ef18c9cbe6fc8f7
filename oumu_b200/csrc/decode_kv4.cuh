// Decode attention over the 4-bit paged cache (kv4.cuh), one query position per take, optionally with the newest
// position's rope, quantisation and cache write in the same launch.
//
// Measured (one B200, back to back in a graph, 16 q and 2 kv heads of 128): 256 takes of 330..4096 positions, 184 MB,
// 49 us (3.8 TB/s; the copies alone take 32); 64 takes 21.2 us; 32 takes 17.6; 2 takes of 65536 positions 21.7; one of
// 512 8.4. 64 takes of 24576 positions, 504 MB, take 92.4 us (5.5 TB/s), of 8192 41.1 (4.1): 6.5 TB/s between the two,
// the rest is fixed: 3 us to the first tile, 3 to 4 from a CTA's last tile to the end (merge, counter, the last one's
// sum), 2 of launch, and what the warps' ends differ by.
//
// The mathematics. With value = s n + z for each group of 32 channels,
//   score_j = sum_g s_jg (q . n_j)_g + sum_g z_jg Q_g,    Q_g = the sum of q over group g,
//   out     = [ sum_j (p_j s_jg) n_jc + sum_j p_j z_jg ] / sum_j p_j    for channel c of group g,
// so the matrix instructions multiply by the codes themselves: fp16 subnormals n 2^-24, exact, masked out of the
// packed words. q is scaled by a power of two of its own for each head so that it is exact in fp16; the zeros' term of
// the scores is one more instruction, bf16 zeros times Q split into three bf16 parts (24 bits). p_j s_jg is rounded to
// fp16 (2^-11 relative, at most). The head's running reference M, a raw score, keeps the largest p at 2^-12: no sum of p z
// leaves fp32, and M is exact however large the scores are. A power of two of each channel group's own, its gain, keeps the
// group's largest scale at 2^21 or more: the largest products are near 2^9, V may be of any size, and one group's size
// costs another nothing. Both move only when p or a product rises by more than 2^5. A scale keeps all bits of p s down to
// 2^-23 of its group's largest. Sums, p, the zeros' term of the output and M are fp32.
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
constexpr uint32_t GAIN_MAX = 0x7e807e80u;  // a pair of 2^126: for groups whose scales have all been 0 (and subnormal ones)

// Not volatile (nor the transposition below): the compiler may interleave these with other work as it likes.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// d = a * b, with nothing added
__device__ __forceinline__ void mma_f16_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                            uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_bf16_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose8(uint32_t a) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// 8 codes of a word as fp16 pairs: n 2^-24 (even nibbles) and 16 n 2^-24 (odd ones)
__device__ __forceinline__ uint32_t code_even(uint32_t w) { return w & 0x000f000fu; }
__device__ __forceinline__ uint32_t code_odd(uint32_t w) { return w & 0x00f000f0u; }
// The same with the high halves (V: the odd positions) as n - 15: (w & mask) ^ flip in one instruction
__device__ __forceinline__ uint32_t and_xor(uint32_t w, uint32_t mask, uint32_t flip) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(r) : "r"(w), "r"(mask), "r"(flip));
    return r;
}
__device__ __forceinline__ uint32_t flip_even(uint32_t w) { return and_xor(w, 0x000f000fu, 0x800f0000u); }
__device__ __forceinline__ uint32_t flip_odd(uint32_t w) { return and_xor(w, 0x00f000f0u, 0x80f00000u); }
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t min_u16x2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("min.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
    return kv4::as_u32(__hmul2(kv4::as_bf2(a), kv4::as_bf2(b)));
}

struct Params {
    const bf16 *qkv;
    uint8_t *pool;               // written only by the fused form, at the newest position
    const int *table;
    bf16 *out, *held;            // held: fused form, may be null
    float *part;                 // partial records
    int *cnt;                    // [B * nk], zero between launches
    const int *pos, *lens;
    const float *cos_t, *sin_t;  // fused form: rotary tables, or null (no rope)
    int rot_rows;                // rows of cos_t and sin_t
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
        // the largest |q| of the head lands in [2^14, 2^15): fp16 keeps a bf16 exactly down to 2^-27 of it
        int e = mx > 0.f ? 14 + 127 - static_cast<int>(__float_as_uint(mx) >> 23) : 14;
        e = e > 127 ? 127 : e;
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
            z0 = t & 1 ? (t < 2 ? part[0][W / 2 - 1] : part[1][W / 2 - 1]) : (t < 2 ? part[0][0] : part[1][0]);
            z1 = t < 2 ? (t & 1 ? part[2][W / 2 - 1] : part[2][0]) : 0u;
        } else {
            z0 = t == 0 ? part[0][0] : t == 1 ? part[1][0] : t == 2 ? part[2][0] : 0u;
            z1 = 0u;
        }
        // 2^(24 - e), by the units of q and of the codes, in two factors. Kept inside fp32, where products with 0 and infinity
        // have a value (the upper end is met where |q| scale reaches 2^117)
        float m = __uint_as_float(static_cast<uint32_t>((24 - e) / 2 + 127) << 23);
        m = m * P.sl2 * m * (e & 1 ? e < 24 ? 2.f : 0.5f : 1.f);
        m = fminf(fmaxf(m, 1.17549435e-38f), 3.40282347e38f);
        mul0 = __shfl_sync(0xffffffffu, m, 8 * t);
        mul1 = __shfl_sync(0xffffffffu, m, 8 * t + 4);
    }
};

// The running state of one (take, kv head): lane 4g + t holds heads 2t and 2t + 1. What goes with the codes beside them,
// the zeros' term and the sum of p: for hd 128 by the matrix instructions too, the meta rows of 8 positions being an 8 x 8
// matrix whose transpose (ldmatrix) is their operand, p in two bf16 parts (17 bits); for hd 64 by each lane for its
// positions.
template <int HD>
struct State {
    static constexpr int W = Fmt<HD>::W;
    static constexpr bool SIDE = W == 4;
    float M[2];                // the reference: the largest raw score, or a little less
    uint32_t gain[W / 2];      // the groups' powers of two, as bf16 pairs like a meta row's scales
    float acc[2 * W][4];       // numerator * gain / 2^24 of channels 32w + 4g + {0 | 1 (x 16)}, {2 | 3 (x 16)}
    // SIDE: [0..1] row g: sum p s_g (g < 4, not used) | sum p z of group g - 4; [2..3] row 8 + g: sum over odd positions
    // of p s_g (g < 4) | sum p. Otherwise: [2w + c] this lane's share of the zeros' term, [2W + c] of the sum.
    float side[SIDE ? 4 : 2 * W + 2];
    __device__ void clear() {
        M[0] = M[1] = -INFINITY;
#pragma unroll
        for (uint32_t &f : gain) f = GAIN_MAX;
#pragma unroll
        for (int i = 0; i < 2 * W; i++) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.f;
#pragma unroll
        for (float &f : side) f = 0.f;
    }

    // One tile of 32 positions in shared memory, the first `n` of them valid (what lies behind is never used: its codes
    // are finite whatever they hold, the scales and zeros of its V are cleared here).
    __device__ __forceinline__ void tile(uint8_t *half, int n, const Query<HD> &Q, int lane) {
        using F = Fmt<HD>;
        const int g = lane >> 2, t = lane & 3;
        float x[2][4];
        {
            // the instructions of all groups and halves side by side: two dependent ones a group, 2 W independent chains
            Words<W> k[2][2], m[2][2];
            float a[2][W][4];
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    k[h][r] = kv4::ld_words<W>(half + (2 * h + r) * F::BLOCK + lane * 4 * W);
                    m[h][r] = kv4::ld_words<W>(half + F::KMETA + (16 * h + 8 * r + g) * F::ROW);
                }
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int w = 0; w < W; w++)
                    mma_f16_new(a[h][w], code_even(k[h][0].v[w]), code_even(k[h][1].v[w]), code_odd(k[h][0].v[w]),
                                code_odd(k[h][1].v[w]), Q.q[w][0], Q.q[w][1]);
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t a0 = W == 4 && !(t & 1) ? m[h][0].v[W / 2] : m[h][0].v[W - 1];
                const uint32_t a1 = W == 4 && !(t & 1) ? m[h][1].v[W / 2] : m[h][1].v[W - 1];
                mma_bf16_new(x[h], a0, a1, a0, a1, Q.z0, Q.z1);
            }
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int w = 0; w < W; w++)
                    mma_f16(a[h][w], code_even(k[h][0].v[w] >> 8), code_even(k[h][1].v[w] >> 8),
                            code_odd(k[h][0].v[w] >> 8), code_odd(k[h][1].v[w] >> 8), Q.q[w][2], Q.q[w][3]);
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int w = 0; w < W; w++)
#pragma unroll
                    for (int i = 0; i < 4; i++) x[h][i] = fmaf(kv4::row_scale<W>(m[h][i >> 1], w), a[h][w][i], x[h][i]);
        }
        if (n < HALF) {
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (16 * h + 8 * (i >> 1) + g >= n) x[h][i] = -INFINITY;
            if (lane >= n) kv4::st_words<W>(half + F::VMETA + lane * F::ROW, Words<W>{});
            fence_proxy_async_smem();  // before the stage's next copy
            __syncwarp();
        }
        Words<W> vm[2][2];
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int r = 0; r < 2; r++) vm[h][r] = kv4::ld_words<W>(half + F::VMETA + (16 * h + 8 * r + g) * F::ROW);
        float p[2][4];
        uint32_t pv[2][W][2];
        // p and p s, again where M turns out too low for them
        for (bool again = false;; again = true) {
            uint32_t top = 0;
            float big = 0.f;
#pragma unroll
            for (int h = 0; h < 2; h++) {
#pragma unroll
                for (int i = 0; i < 4; i++) p[h][i] = fast_exp2(fmaf(x[h][i] - M[i & 1], i & 1 ? Q.mul1 : Q.mul0, -12.f));
                big = fmax3(fmax3(big, p[h][0], p[h][1]), p[h][2], p[h][3]);
#pragma unroll
                for (int r = 0; r < 2; r++) {
                    Words<W> sg;
#pragma unroll
                    for (int i = 0; i < W / 2; i++) sg.v[i] = mul_bf16x2(vm[h][r].v[i], gain[i]);  // exact
#pragma unroll
                    for (int w = 0; w < W; w++) {
                        const float s = kv4::row_scale<W>(sg, w);
                        pv[h][w][r] = pack_f16x2(p[h][2 * r] * s, p[h][2 * r + 1] * s);
                        top = max_u16x2(top, pv[h][w][r]);
                    }
                }
            }
            // 2^-7, and 2^15 in fp16 (0x7800; infinities and NaN lie above)
            const bool over = (top & 0xffffu) > 0x7800u || top > 0x7800ffffu || !(big <= 0.0078125f);
            if (again || !__any_sync(0xffffffffu, over)) break;
            rescale(x, vm, Q);
        }
        if constexpr (SIDE) {
            uint32_t r[4];
            ldsm_x4_t(smem_u32(half + F::VMETA + lane * F::ROW), r[0], r[1], r[2], r[3]);
            const uint32_t keep = g < 4 ? 0xffff0000u : 0u, one = g < 4 ? 0u : 0x3f803f80u;
            float d[4];
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const uint32_t u0 = pack_bf16x2(p[h][0], p[h][1]), u1 = pack_bf16x2(p[h][2], p[h][3]);
                const float2 f0 = unpack_bf16x2(u0), f1 = unpack_bf16x2(u1);
                const uint32_t v0 = pack_bf16x2(p[h][0] - f0.x, p[h][1] - f0.y);
                const uint32_t v1 = pack_bf16x2(p[h][2] - f1.x, p[h][3] - f1.y);
                const uint32_t a0 = r[2 * h], a2 = r[2 * h + 1], a1 = (a0 & keep) | one, a3 = (a2 & keep) | one;
                if (h == 0) mma_bf16_new(d, a0, a1, a2, a3, transpose8(u0), transpose8(u1));
                else mma_bf16(d, a0, a1, a2, a3, transpose8(u0), transpose8(u1));
                mma_bf16(d, a0, a1, a2, a3, transpose8(v0), transpose8(v1));
            }
#pragma unroll
            for (int i = 0; i < 4; i++) side[i] += d[i];  // rounded, not cut: these sums keep one sign
        } else {
            const float c15 = g & 1 ? 15.f : 0.f;
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    side[2 * W + c] += p[h][c] + p[h][2 + c];
#pragma unroll
                    for (int w = 0; w < W; w++)
#pragma unroll
                        for (int r = 0; r < 2; r++)
                            side[2 * w + c] = fmaf(
                                p[h][2 * r + c],
                                fmaf(c15, kv4::row_scale<W>(vm[h][r], w), kv4::row_zero<W>(vm[h][r], w)), side[2 * w + c]);
                }
        }
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const Words<W> v0 = kv4::ld_words<W>(half + F::CODES + (2 * h) * F::BLOCK + lane * 4 * W);
            const Words<W> v1 = kv4::ld_words<W>(half + F::CODES + (2 * h + 1) * F::BLOCK + lane * 4 * W);
#pragma unroll
            for (int w = 0; w < W; w++) {
                const uint32_t b0 = transpose8(pv[h][w][0]), b1 = transpose8(pv[h][w][1]);
                mma_f16(acc[2 * w], flip_even(v0.v[w]), flip_odd(v0.v[w]), flip_even(v1.v[w]), flip_odd(v1.v[w]), b0,
                        b1);
                mma_f16(acc[2 * w + 1], flip_even(v0.v[w] >> 8), flip_odd(v0.v[w] >> 8), flip_even(v1.v[w] >> 8),
                        flip_odd(v1.v[w] >> 8), b0, b1);
            }
        }
    }

    // Raise M to the largest score of this tile, lower the gains so that no scale passes 2^22, and bring the sums along. The
    // first tile of a state always comes here (M = -inf); later ones when a logit rises by more than 5 over everything
    // before, or a scale by more than 2^5.
    __device__ __forceinline__ void rescale(const float (&x)[2][4], const Words<W> (&vm)[2][2], const Query<HD> &Q) {
        float top[2];
#pragma unroll
        for (int c = 0; c < 2; c++) {
            top[c] = fmaxf(fmaxf(x[0][c], x[0][2 + c]), fmaxf(x[1][c], x[1][2 + c]));
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], o));
            top[c] = fmaxf(M[c], top[c]);
            if (top[c] == -INFINITY) top[c] = 0.f;
        }
        uint32_t now[W / 2];
#pragma unroll
        for (int i = 0; i < W / 2; i++) {
            const uint32_t m = max_u16x2(max_u16x2(vm[0][0].v[i], vm[0][1].v[i]), max_u16x2(vm[1][0].v[i], vm[1][1].v[i]));
            const uint32_t lo = __reduce_max_sync(0xffffffffu, m << 16), hi = __reduce_max_sync(0xffffffffu, m);
            // exponent fields: 2^(21 - e) for a scale in [2^e, 2^(e + 1)), e + 127 being the scale's own (0: GAIN_MAX)
            now[i] = min_u16x2(gain[i], 0x89808980u - (__byte_perm(lo, hi, 0x7632) & 0x7f807f80u));
        }
        if (M[0] != -INFINITY) {  // some sums there are
            float g[W];  // now / gain, 0 below 2^-149
#pragma unroll
            for (int w = 0; w < W; w++) g[w] = pick(now, w) * __uint_as_float(0x7f000000u - __float_as_uint(pick(gain, w)));
#pragma unroll
            for (int c = 0; c < 2; c++) {
                const float f = fast_exp2((M[c] - top[c]) * (c ? Q.mul1 : Q.mul0));
#pragma unroll
                for (int i = 0; i < 2 * W; i++) {
                    acc[i][c] *= f * g[i / 2];
                    acc[i][c + 2] *= f * g[i / 2];
                }
#pragma unroll
                for (int i = c; i < (SIDE ? 4 : 2 * W + 2); i += 2) side[i] *= f;
            }
        }
        M[0] = top[0];
        M[1] = top[1];
#pragma unroll
        for (int i = 0; i < W / 2; i++) gain[i] = now[i];
    }
    // Group w's of pairs of bf16
    __device__ __forceinline__ static float pick(const uint32_t (&v)[W / 2], int w) {
        return __uint_as_float(w & 1 ? v[w / 2] & 0xffff0000u : v[w / 2] << 16);
    }

    // The sums of p and the zeros' terms of heads 2t and 2t + 1 over all positions, in every lane.
    __device__ __forceinline__ void reduce(float (&l)[2], float (&z)[W][2], int lane) const {
#pragma unroll
        for (int c = 0; c < 2; c++) {
            if constexpr (SIDE) {
                const int t = lane & 3;
                l[c] = __shfl_sync(0xffffffffu, side[2 + c], 16 + t);
#pragma unroll
                for (int w = 0; w < W; w++)
                    z[w][c] = fmaf(15.f, __shfl_sync(0xffffffffu, side[2 + c], 4 * w + t),
                                   __shfl_sync(0xffffffffu, side[c], 16 + 4 * w + t));
            } else {
                l[c] = side[2 * W + c];
#pragma unroll
                for (int w = 0; w < W; w++) z[w][c] = side[2 * w + c];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) {
                    l[c] += __shfl_xor_sync(0xffffffffu, l[c], o);
#pragma unroll
                    for (int w = 0; w < W; w++) z[w][c] += __shfl_xor_sync(0xffffffffu, z[w][c], o);
                }
            }
        }
    }
    // Numerators of head 2t + c, channels 32w + 4g .. + 3, with the zeros' term, in the values' own unit.
    __device__ __forceinline__ float4 numerators(const float (&z)[W][2], int w, int c) const {
        const float u = 16777216.f, u16 = 1048576.f;  // 2^24, and / 16 for the odd nibbles
        const float r = __uint_as_float(0x7f000000u - __float_as_uint(pick(gain, w)));  // 1 / gain
        return make_float4(fmaf(acc[2 * w][c] * u, r, z[w][c]), fmaf(acc[2 * w][c + 2] * u16, r, z[w][c]),
                           fmaf(acc[2 * w + 1][c] * u, r, z[w][c]), fmaf(acc[2 * w + 1][c + 2] * u16, r, z[w][c]));
    }
    // The output of a segment that this warp has seen whole; out: its first head's row.
    __device__ __forceinline__ void finish(bf16 *out, int G, int lane) {
        const int g = lane >> 2, t = lane & 3;
        float l[2], z[W][2];
        reduce(l, z, lane);
#pragma unroll
        for (int c = 0; c < 2; c++) {
            if (2 * t + c >= G) continue;
            const float r = 1.f / l[c];
#pragma unroll
            for (int w = 0; w < W; w++) {
                const float4 o = numerators(z, w, c);
                uint2 u;
                u.x = pack_bf16x2(o.x * r, o.y * r);
                u.y = pack_bf16x2(o.z * r, o.w * r);
                *reinterpret_cast<uint2 *>(out + (2 * t + c) * HD + 32 * w + 4 * g) = u;
            }
        }
    }
    // The state as a record: m[8] (base-2 logits), l[8], o[8][HD].
    __device__ __forceinline__ void record(float *R, const Query<HD> &Q, int lane) {
        const int g = lane >> 2, t = lane & 3;
        float l[2], z[W][2];
        reduce(l, z, lane);
        if (g == 0) {
            R[2 * t] = M[0] * Q.mul0;
            R[2 * t + 1] = M[1] * Q.mul1;
            R[GMAX + 2 * t] = l[0];
            R[GMAX + 2 * t + 1] = l[1];
        }
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
            for (int w = 0; w < W; w++)
                *reinterpret_cast<float4 *>(R + 2 * GMAX + (2 * t + c) * HD + 32 * w + 4 * g) = numerators(z, w, c);
    }
};

// Fused form: the newest position's k (rotated) and v, quantised by the warp that has the segment's last tile. Lane l has
// channels 4l .. 4l + 3. `make` writes them into the take's page (`half`; null: not at all) and `held` as soon as q
// arrives; `patch` into the copy of that half in shared memory, which was on its way already.
template <int HD>
struct Newest {
    static constexpr int W = Fmt<HD>::W;
    uint32_t code[2], meta[2];  // K word | V half word; scale | zero << 16
    __device__ __forceinline__ static int code_at(int kv, int r, int lane) {
        using F = Fmt<HD>;
        const int w = lane >> 3, j = lane & 7;
        return kv == 0 ? r / 8 * F::BLOCK + ((r % 8 * 4 + j / 2) * W + w) * 4
                       : F::CODES + r / 8 * F::BLOCK + ((j * 4 + r % 8 / 2) * W + w) * 4 + 2 * (r & 1);
    }
    __device__ __forceinline__ void patch(uint8_t *half, int r, int lane) const {
        using F = Fmt<HD>;
        if (lane >= HD / 4) return;
        if (!(lane & 1)) *reinterpret_cast<uint32_t *>(half + code_at(0, r, lane)) = code[0];
        *reinterpret_cast<uint16_t *>(half + code_at(1, r, lane)) = static_cast<uint16_t>(code[1]);
        if ((lane & 7) == 0) {
#pragma unroll
            for (int kv = 0; kv < 2; kv++) {
                uint8_t *m = half + (kv ? F::VMETA : F::KMETA) + r * F::ROW + 2 * (lane >> 3);
                *reinterpret_cast<uint16_t *>(m) = static_cast<uint16_t>(meta[kv]);
                *reinterpret_cast<uint16_t *>(m + 2 * W) = static_cast<uint16_t>(meta[kv] >> 16);
            }
        }
    }
    __device__ __forceinline__ void make(const Params &P, int s, int kh, int p, int lane, uint8_t *half) {
        const bool on = lane < HD / 4;
        const int j = lane & 7, c4 = 4 * (on ? lane : 0);
        const bf16 *row = P.qkv + static_cast<long>(s) * (P.nq + 2 * P.nk) * HD;
        uint2 u[2];
#pragma unroll
        for (int kv = 0; kv < 2; kv++) u[kv] = *reinterpret_cast<const uint2 *>(row + (P.nq + kv * P.nk + kh) * HD + c4);
        if (P.cos_t) {
            const float2 a = unpack_bf16x2(u[0].x), b = unpack_bf16x2(u[0].y);
            const int i = c4 % (HD / 2);
            const float4 c = *reinterpret_cast<const float4 *>(P.cos_t + static_cast<long>(p) * (HD / 2) + i);
            const float4 sn = *reinterpret_cast<const float4 *>(P.sin_t + static_cast<long>(p) * (HD / 2) + i);
            const float x[4] = {a.x, a.y, b.x, b.y}, cc[4] = {c.x, c.y, c.z, c.w}, ss[4] = {sn.x, sn.y, sn.z, sn.w};
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {  // low half: a c - b s; high half: b c + a s
                const float o = __shfl_xor_sync(0xffffffffu, x[e], HD / 8);
                y[e] = c4 < HD / 2 ? x[e] * cc[e] - o * ss[e] : x[e] * cc[e] + o * ss[e];
            }
            u[0].x = pack_bf16x2(y[0], y[1]);
            u[0].y = pack_bf16x2(y[2], y[3]);
        }
#pragma unroll
        for (int kv = 0; kv < 2; kv++) {
            uint32_t rg = kv4::range_of(kv4::as_u32(__hmax2_nan(kv4::as_bf2(u[kv].x), kv4::as_bf2(u[kv].y))),
                                        kv4::as_u32(__hmin2_nan(kv4::as_bf2(u[kv].x), kv4::as_bf2(u[kv].y))));
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) rg = kv4::range_max(rg, __shfl_xor_sync(0xffffffffu, rg, o));
            const kv4::Quant q = kv4::quant_of(rg);
            const uint32_t pr[2] = {u[kv].x, u[kv].y};
            uint32_t marks = 0, c = kv4::quant_pairs<2>(pr, q, marks);  // low half: channels 0, 2; high half: 1, 3
            if (marks & 1u && kv4::quant_marked<2>(pr, q.s, q.z, c)) {
                const float2 f0 = unpack_bf16x2(pr[0]), f1 = unpack_bf16x2(pr[1]);
                c = kv4::quant_exact(f0.x, q.z, q.s) | kv4::quant_exact(f0.y, q.z, q.s) << 16 |
                    kv4::quant_exact(f1.x, q.z, q.s) << 4 | kv4::quant_exact(f1.y, q.z, q.s) << 20;
            }
            const uint32_t n[4] = {c & 15u, c >> 16 & 15u, c >> 4 & 15u, c >> 20 & 15u};
            if (P.held && on) {
                uint2 o;
                o.x = pack_bf16x2(fmaf(q.s, n[0], q.z), fmaf(q.s, n[1], q.z));
                o.y = pack_bf16x2(fmaf(q.s, n[2], q.z), fmaf(q.s, n[3], q.z));
                *reinterpret_cast<uint2 *>(P.held + (static_cast<long>(s) * 2 * P.nk + kv * P.nk + kh) * HD + c4) = o;
            }
            if (kv == 0) {  // two bytes of the word that lanes j and j ^ 1 share
                const uint32_t kw = (c & 0x00ff00ffu) << (8 * (j & 1));
                code[0] = kw | __shfl_xor_sync(0xffffffffu, kw, 1);
            } else {
                code[1] = kv4::in_order(c);
            }
            meta[kv] = kv4::meta_bits(q.s, q.z);
        }
        if (half) patch(half, p % HALF, lane);
    }
};

// Work is counted in tiles (5 KB: 32 positions of one take and kv head, a "segment", at hd 128, 64 at hd 64), laid end to
// end take by take and cut into equal contiguous ranges: one per CTA, and that into one per warp. A warp streams its range
// through a ring of its own in shared memory (one bulk copy per tile, nothing shared, no producer warp), so no warp waits
// for another before the range's end. A segment that lies inside a warp's range is finished by it alone; the parts of one
// that crosses warps meet in shared memory, of one that crosses CTAs in records in global memory, where the last to arrive
// adds them up in CTA order: the result does not depend on timing.
//
// NW warps and ST tiles in flight for each. 12 warps keep three per scheduler, which hides more of the instructions'
// latencies (5 KB of cache take about 660 instructions): between 64 takes of 8192 and of 24576 positions they stream at
// 6.3 TB/s against 5.2 with 8, of 7.1 for the copies alone. 8 warps have less to merge at the end (the launch's rule has both sides' times).
template <int HD>
constexpr int TP = HD == 128 ? kv4::HALF : kv4::PAGE;  // positions per tile
template <int NW>
constexpr int ST = NW == 8 ? 4 : 2;
// tiles per CTA at least: one a warp
template <int NW>
constexpr int MIN_TILES = NW;
// CTA boundaries do not cut segments of up to so many tiles, three per warp: adding up records across CTAs costs about
// 3 us, as long as a CTA's work growing by that many tiles (one take of 512 positions 8.4 us against 9.4, 19 takes at hd 64
// 9.4 against 9.7; long segments are cut either way).
template <int NW>
constexpr int SNAP = 3 * NW;

// A segment that a boundary cuts: take * nk + kv head (-1: none), its tiles.
struct Cut {
    int id, start, end;
};

template <int HD, int NW>
struct Lay {
    static_assert(NW <= 16, "a half warp holds a reference per warp");
    static constexpr int REC = 2 * GMAX + GMAX * HD;  // floats of a record: m[8], l[8], o[8][HD]
    static constexpr int TILE = TP<HD> / kv4::HALF * Fmt<HD>::HALFB;
    static constexpr int RING = ST<NW> * TILE;
    static_assert(REC * 4 <= RING, "a warp's last record lies in its own ring");
    static constexpr int FIRST = NW * RING;           // records of segments that end inside a warp's range
    static constexpr int BAR = FIRST + NW * REC * 4;
    static constexpr int CUTS = BAR + NW * ST<NW> * 8;    // segments cut by the warps' boundaries
    static constexpr int MISC = CUTS + (NW + 1) * static_cast<int>(sizeof(Cut));
    static constexpr int PRE = MISC + 128;            // pre[B + 1], lens[B]
    static __host__ __device__ int bytes(int B) { return PRE + (2 * B + 1) * 4; }
};

// The warp's first lane announces and starts a copy (predicated: no branch in the loop).
__device__ __forceinline__ void bulk_load_first_lane(uint32_t dst, unsigned long long src, uint32_t bytes, uint32_t bar,
                                                     int lane) {
    asm volatile(
        "{\n .reg .pred p;\n .reg .b64 st;\n setp.eq.s32 p, %4, 0;\n"
        " @p mbarrier.arrive.expect_tx.shared::cta.b64 st, [%3], %2;\n"
        " @p cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n}" ::"r"(dst),
        "l"(src), "r"(bytes), "r"(bar), "r"(lane)
        : "memory");
}

// Take s's length: lens[s] or *pos + 1, cut to what its table row, and the rotary tables, can hold (recorded).
__device__ __forceinline__ int take_len(const Params &P, int s) {
    int L = P.lens ? P.lens[s] : *P.pos + 1;
    int room = P.maxpages * kv4::PAGE;
    if (P.cos_t) room = min(room, P.rot_rows);
    if (L < 0 || L > room) {
        record_error(OUMU_DEVERR_LENGTH);
        L = L < 0 ? 0 : room;
    }
    return L;
}
template <int HD>
__device__ __forceinline__ int tiles_of(int L) { return (L + TP<HD> - 1) / TP<HD>; }

// The take whose tiles hold tile t: the last s with pre[s] <= t (takes without tiles are passed over).
__device__ __forceinline__ int take_of(const int *pre, int B, int t) {
    int lo = 0, hi = B - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (pre[mid] <= t) lo = mid; else hi = mid - 1;
    }
    return lo;
}
// W tiles in n parts, the first W % n of them one tile longer: where part i starts, and the part that has tile t.
struct Parts {
    int q, r;
    __device__ Parts(int W, int n) : q(W / n), r(W % n) {}
    __device__ int start(int i) const { return i * q + min(i, r); }
    __device__ int of(int t) const {
        const int a = r * (q + 1);
        return t < a ? t / (q + 1) : r + (t - a) / q;
    }
};

template <int HD, int NW, bool FUSED>
__global__ void __launch_bounds__(NW * 32, 1) k_attn_decode_kv4(Params P) {
    using F = Fmt<HD>;
    using Y = Lay<HD, NW>;
    constexpr int NT = NW * 32, ST = d4::ST<NW>, TP = d4::TP<HD>;
    extern __shared__ __align__(128) uint8_t sm[];
    int *pre = reinterpret_cast<int *>(sm + Y::PRE), *Ls = pre + P.B + 1;
    int *misc = reinterpret_cast<int *>(sm + Y::MISC);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int B = P.B, nk = P.nk, G = P.nq / P.nk, c = blockIdx.x;
    const uint32_t ring = smem_u32(sm) + warp * Y::RING, bars = smem_u32(sm) + Y::BAR + warp * ST * 8;

    if (lane < ST) mbar_init(bars + 8 * lane, 1);
    mbar_fence_init();
    pdl_trigger();
    // tiles before every take
    {
        int run = 0;
        for (int s0 = 0; s0 < B; s0 += NT) {
            const int s = s0 + threadIdx.x, L = s < B ? take_len(P, s) : 0, n = tiles_of<HD>(L) * nk;
            int x = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            if (lane == 31) misc[warp] = x;
            __syncthreads();
            int before = run, all = run;
#pragma unroll
            for (int w = 0; w < NW; w++) {
                before += w < warp ? misc[w] : 0;
                all += misc[w];
            }
            if (s < B) {
                pre[s] = before + x - n;
                Ls[s] = L;
            }
            run = all;
            __syncthreads();
        }
        if (threadIdx.x == 0) pre[B] = run;
    }
    __syncthreads();
    const int W = pre[B];
    const int want = (W + MIN_TILES<NW> - 1) / MIN_TILES<NW>, Gc = want < static_cast<int>(gridDim.x) ? want : gridDim.x;
    int ta = 0, tb = 0;
    const Parts ctas(W, Gc > 0 ? Gc : 1);
    if (c < Gc) {
        // a boundary inside a short segment moves to the segment's nearer end: lanes 0 and 1 find this CTA's two
        int t = ctas.start(min(c + (lane & 1), Gc));
        if (t < W) {
            const int s = take_of(pre, B, t), T = tiles_of<HD>(Ls[s]), j = (t - pre[s]) % T;
            if (T <= SNAP<NW>) t += 2 * j < T ? -j : T - j;
        }
        ta = __shfl_sync(0xffffffffu, t, 0);
        tb = __shfl_sync(0xffffffffu, t, 1);
    }
    auto after_predecessor = [&] {  // what the preceding kernel may write is read, and memory written, from here on
        pdl_wait();
        for (int s = c; s < B; s += gridDim.x) {  // takes that hold nothing
            if (Ls[s] > 0) continue;
            const uint4 zero = make_uint4(0, 0, 0, 0);
            for (int i = threadIdx.x; i < P.nq * HD / 8; i += NT)
                reinterpret_cast<uint4 *>(P.out + static_cast<long>(s) * P.nq * HD)[i] = zero;
            if (FUSED && P.held)
                for (int i = threadIdx.x; i < 2 * nk * HD / 8; i += NT)
                    reinterpret_cast<uint4 *>(P.held + static_cast<long>(s) * 2 * nk * HD)[i] = zero;
        }
    };
    if (ta >= tb) {
        after_predecessor();
        return;
    }
    const Parts parts(tb - ta, NW);
    // by way of a shuffle: the loop then takes 3 to 12 registers fewer (6.26 TB/s between 64 takes of
    // 8192 and of 24576 positions, 6.05 without)
    const int bound = ta + parts.start(warp + (lane & 1));
    const int wa = __shfl_sync(0xffffffffu, bound, 0), wb = __shfl_sync(0xffffffffu, bound, 1), n = wb - wa;

    // Boundary b of the CTA's range (b < nb: where warp b starts; nb, the number of warps with tiles: the range's end) and
    // the segment it cuts, each found by the warp that has it at hand; id -1 where a segment ends there.
    Cut *cuts = reinterpret_cast<Cut *>(sm + Y::CUTS);
    const int nb = min(NW, tb - ta);
    // ---- this warp's tiles ----
    if (n > 0) {
        const uint8_t *src = nullptr;  // lane i: tile base + i
        int s, T, kh, j;               // its take, tiles of a segment, kv head, tile of the segment
        auto look_up = [&](int base) {
            const int t = min(wa + base + lane, wb - 1);
            s = take_of(pre, B, t);
            T = tiles_of<HD>(Ls[s]);
            kh = (t - pre[s]) / T;
            j = t - pre[s] - kh * T;
            constexpr int per = kv4::PAGE / TP;  // tiles of a page
            int page = P.table[static_cast<long>(s) * P.maxpages + j / per];
            if (page < 0 || page >= P.npages) {
                record_error(OUMU_DEVERR_PAGE);
                page = 0;  // read in its place: the take's output is unspecified
            }
            src = P.pool + (static_cast<long>(page) * nk + kh) * F::UNIT + j % per * Y::TILE;
        };
        auto issue = [&](int k) {  // tile k into its stage
            const unsigned long long a = __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), k & 31);
            bulk_load_first_lane(ring + (k % ST) * Y::TILE, a, Y::TILE, bars + 8 * (k % ST), lane);
        };
        // Fused, a copy may come before the preceding kernel's end: that kernel writes no page, and the newest position is
        // patched in. Otherwise it may be the write of the newest position.
        if (!FUSED) after_predecessor();
        auto look_up_later = [&](int base) {  // with s .. j kept: they are the warp's place by then
            const int s0 = s, T0 = T, kh0 = kh, j0 = j;
            look_up(base);
            s = s0, T = T0, kh = kh0, j = j0;
        };
        look_up(0);
        issue(0);
        if (FUSED) after_predecessor();
        s = __shfl_sync(0xffffffffu, s, 0);
        T = __shfl_sync(0xffffffffu, T, 0);
        kh = __shfl_sync(0xffffffffu, kh, 0);
        j = __shfl_sync(0xffffffffu, j, 0);
        if (lane == 0) cuts[warp] = Cut{j > 0 ? s * nk + kh : -1, wa - j, wa - j + T};
        int k = 0, issued = 1;
        while (k < n) {
            // ---- this warp's part of a segment: tiles j .. of take s, kv head kh ----
            const int L = Ls[s], Sg = wa + k - j, stop = min(n, k + T - j);
            Query<HD> Q;
            State<HD> S;
            Newest<HD> N;
            Q.load(P, s, kh, L - 1, lane);
            S.clear();
            const bool ends = stop == k + T - j;  // its last tile is this warp's
            if (FUSED && ends) {
                // a length that take_len has cut is not this position's: what the page holds there, for other takes too,
                // stays
                const int page = P.table[static_cast<long>(s) * P.maxpages + (L - 1) / kv4::PAGE];
                const bool write = page >= 0 && page < P.npages && (P.lens ? P.lens[s] : *P.pos + 1) == L;
                N.make(P, s, kh, L - 1, lane,
                       write ? P.pool + (static_cast<long>(page) * nk + kh) * F::UNIT +
                                   (L - 1) % kv4::PAGE / HALF * F::HALFB
                             : nullptr);
            }
            for (; issued < ST && issued < n; issued++) issue(issued);  // behind every warp's first tile
            int left = L - j * TP;  // positions from this tile on
            for (; k < stop; k++, left -= TP) {
                const uint32_t bar = bars + 8 * (k % ST), phase = (k / ST) & 1;
                if (!__all_sync(0xffffffffu, mbar_try_wait(bar, phase)) &&
                    !__all_sync(0xffffffffu, mbar_wait(bar, phase)))
                    break;
                uint8_t *half = sm + warp * Y::RING + (k % ST) * Y::TILE;
                if (FUSED && ends && k == stop - 1) {
                    N.patch(half + (L - 1) % TP / HALF * F::HALFB, (L - 1) % HALF, lane);
                    fence_proxy_async_smem();  // before the stage's next copy
                    __syncwarp();
                }
#pragma unroll 1
                for (int h = 0; h < TP / HALF && left > h * HALF; h++)
                    S.tile(half + h * F::HALFB, left - h * HALF, Q, lane);
                __syncwarp();
                if (issued < n) {
                    if ((issued & 31) == 0) look_up_later(issued);
                    issue(issued++);
                }
            }
            if (k < stop) {
                // A wait ran out (recorded): nothing more is computed or started; the outputs are unspecified, but no
                // copy may still be on its way when the CTA leaves (bounded again).
                for (int i = k; i < issued; i++) mbar_wait(bars + 8 * (i % ST), (i / ST) & 1);
                if (warp == nb - 1 && lane == 0) {  // what this warp would have found at its end
                    const int s1 = take_of(pre, B, tb - 1), T1 = tiles_of<HD>(Ls[s1]), h1 = (tb - 1 - pre[s1]) / T1;
                    const int g1 = pre[s1] + h1 * T1;
                    cuts[nb] = Cut{g1 + T1 > tb ? s1 * nk + h1 : -1, g1, g1 + T1};
                }
                break;
            }
            if (ends && Sg >= wa) {
                S.finish(P.out + (static_cast<long>(s) * P.nq + kh * G) * HD, G, lane);
            } else {
                S.record(k == n ? reinterpret_cast<float *>(sm + warp * Y::RING)
                                : reinterpret_cast<float *>(sm + Y::FIRST) + warp * Y::REC,
                         Q, lane);
            }
            if (k == n && warp == nb - 1 && lane == 0) cuts[nb] = Cut{ends ? -1 : s * nk + kh, Sg, Sg + T};
            j = 0;
            if (++kh == nk) {
                kh = 0;
                do ++s; while (s < B && Ls[s] == 0);
                T = s < B ? tiles_of<HD>(Ls[s]) : 1;
            }
        }
    } else {
        after_predecessor();
    }
    __syncthreads();

    // ---- segments that cross a boundary between warps, or the CTA's ends ----
    // The loops here are not unrolled: run once per launch, they cost their instruction fetches.
    constexpr int LPH = HD / 4;  // threads per head, 4 channels each
    const int d4 = threadIdx.x % LPH;
    const unsigned mates = LPH == 32 ? 0xffffffffu : 0xffffu << (lane & 16);  // a head's threads in this warp
    auto store = [&](int id, int h, float l, float4 o) {
        const float r = 1.f / l;
        uint2 u;
        u.x = pack_bf16x2(o.x * r, o.y * r);
        u.y = pack_bf16x2(o.z * r, o.w * r);
        *reinterpret_cast<uint2 *>(P.out + (static_cast<long>(id / nk) * P.nq + id % nk * G + h) * HD + 4 * d4) = u;
    };
    // which cut segments reach into other CTAs. Bit 0: the one cut by the range's start, bit 1: by its end only
    int crossing = cuts[0].id >= 0;
    if (cuts[nb].id >= 0 && cuts[nb].start >= ta) crossing |= 2;
    {
        // boundaries that cut a segment for the first time, and those that cut the one before's again (a lane per boundary)
        const int mine = lane <= nb ? cuts[lane].id : -1, left_one = __shfl_up_sync(0xffffffffu, mine, 1);
        const bool again = lane > 0 && mine == left_one;
        unsigned todo = __ballot_sync(0xffffffffu, mine >= 0 && !again);
        const unsigned more = __ballot_sync(0xffffffffu, mine >= 0 && again);
        constexpr int PER = GMAX / 2;  // a warp takes two heads of a segment
        int done = 0;
#pragma unroll 1
        for (int unit = warp;; unit += NW) {
            for (; done < unit / PER; done++) todo &= todo - 1;
            if (!todo) break;
            const int i = __ffs(todo) - 1;
            const Cut x = cuts[i];
            // the warps that have some of it: from the one before its first boundary to the one behind its last
            const int first = max(i - 1, 0), last = min(i + __ffs(~(more >> i >> 1)) - 1, nb - 1);
            auto at = [&](int w) {  // warp w's record of it: its last one if the segment goes on to the range's end
                return x.end >= ta + parts.start(w + 1) ? reinterpret_cast<const float *>(sm + w * Y::RING)
                                                        : reinterpret_cast<const float *>(sm + Y::FIRST) + w * Y::REC;
            };
            const bool has = first + d4 <= last;  // the head's threads take a record's reference and sum each
            const float *own = at(has ? first + d4 : first);
#pragma unroll
            for (int hh = 0; hh < (LPH == 32 ? 2 : 1); hh++) {
                const int h = unit % PER * 2 + (LPH == 32 ? hh : lane >> 4);
                if (h >= G) continue;
                const float m = has ? own[h] : -INFINITY;
                float M = m;
#pragma unroll
                for (int e = 1; e < 16; e <<= 1) M = fmaxf(M, __shfl_xor_sync(mates, M, e, 16));
                M = __shfl_sync(mates, M, 0, LPH);
                const float fm = fast_exp2(m - M);
                float l = has ? fm * own[GMAX + h] : 0.f;
#pragma unroll
                for (int e = 1; e < 16; e <<= 1) l += __shfl_xor_sync(mates, l, e, 16);
                l = __shfl_sync(mates, l, 0, LPH);
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
                for (int w = first; w <= last; w++) {
                    const float f = __shfl_sync(mates, fm, w - first, LPH);
                    const float4 v = *reinterpret_cast<const float4 *>(at(w) + 2 * GMAX + h * HD + 4 * d4);
                    o = make_float4(fmaf(f, v.x, o.x), fmaf(f, v.y, o.y), fmaf(f, v.z, o.z), fmaf(f, v.w, o.w));
                }
                if (x.start >= ta && x.end <= tb) {
                    store(x.id, h, l, o);
                } else {  // record 1 of a CTA is of a segment that starts in it
                    float *rec = P.part + (static_cast<long>(c) * 2 + (x.start >= ta)) * Y::REC;
                    if (d4 == 0) {
                        rec[h] = M;
                        rec[GMAX + h] = l;
                    }
                    *reinterpret_cast<float4 *>(rec + 2 * GMAX + h * HD + 4 * d4) = o;
                }
            }
        }
    }
    if (!crossing) return;
    // the counts of the (at most two) segments that reach into other CTAs; whoever completes one adds it up
    __syncthreads();
    if (threadIdx.x < 2 && crossing >> threadIdx.x & 1) {
        const Cut x = cuts[threadIdx.x ? nb : 0];
        const int others = ctas.of(x.end - 1) - ctas.of(x.start);
        const bool done = atomic_add_acq_rel(P.cnt + x.id, 1) == others;
        if (done) P.cnt[x.id] = 0;
        misc[1 + threadIdx.x] = done;
    }
    __syncthreads();
    const int h = threadIdx.x / LPH;
#pragma unroll 1
    for (int k = 0; k < 2; k++) {
        if (!(crossing >> k & 1) || !misc[1 + k] || h >= G) continue;
        const Cut x = cuts[k ? nb : 0];
        const int cf = ctas.of(x.start), cl = ctas.of(x.end - 1);
        auto at = [&](int cc) { return P.part + (static_cast<long>(cc) * 2 + (cc == cf)) * Y::REC + h; };
        auto numer = [&](int cc) {
            return __ldcg(reinterpret_cast<const float4 *>(at(cc) - h + 2 * GMAX + h * HD + 4 * d4));
        };
        // up to 16 records' numerators on their way while the head's LPH threads take a record's reference and sum each
        constexpr int N = 16;
        float4 v[N];
#pragma unroll
        for (int e = 0; e < N; e++) v[e] = cf + e <= cl ? numer(cf + e) : make_float4(0.f, 0.f, 0.f, 0.f);
        float m = cf + d4 <= cl ? __ldcg(at(cf + d4)) : -INFINITY;
        float lw = cf + d4 <= cl ? __ldcg(at(cf + d4) + GMAX) : 0.f;
        float M = m, l = 0.f;
        constexpr float DOWN = 8.f;  // 2^-8 of everything: sums over a take's positions stay inside fp32
        for (int cc = cf + d4 + LPH; cc <= cl; cc += LPH) M = fmaxf(M, __ldcg(at(cc)));
#pragma unroll
        for (int e = 1; e < LPH; e <<= 1) M = fmaxf(M, __shfl_xor_sync(mates, M, e, LPH));  // a head's threads come together
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        float f = fast_exp2(m - M - DOWN);
        l = f * lw;
#pragma unroll 1
        for (int c0 = cf;;) {
#pragma unroll
            for (int e = 0; e < N; e++) {
                const float fe = __shfl_sync(mates, f, (c0 - cf + e) % LPH, LPH);
                o = make_float4(fmaf(fe, v[e].x, o.x), fmaf(fe, v[e].y, o.y), fmaf(fe, v[e].z, o.z), fmaf(fe, v[e].w, o.w));
            }
            c0 += N;
            if (c0 > cl) break;
#pragma unroll
            for (int e = 0; e < N; e++) v[e] = c0 + e <= cl ? numer(c0 + e) : make_float4(0.f, 0.f, 0.f, 0.f);
            if ((c0 - cf) % LPH == 0) {  // the next LPH records' references
                const bool in = c0 + d4 <= cl;
                f = in ? fast_exp2(__ldcg(at(c0 + d4)) - M - DOWN) : 0.f;
                l = in ? fmaf(f, __ldcg(at(c0 + d4) + GMAX), l) : l;
            }
        }
#pragma unroll
        for (int e = 1; e < LPH; e <<= 1) l += __shfl_xor_sync(mates, l, e, LPH);
        store(x.id, h, l, o);
    }
}

}  // namespace d4

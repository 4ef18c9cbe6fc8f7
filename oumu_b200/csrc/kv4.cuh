// The 4-bit paged KV cache: its format, the quantiser, prompt writes and reads back to bf16 (include/oumu_attn.h).
//
// Format. A page holds 64 positions of every kv head; a unit is one kv head of a page: two halves of 32 positions, each
//   [K codes 16 hd bytes][V codes 16 hd bytes][K meta 32 rows][V meta 32 rows],
// a meta row being the position's hd/32 group scales, then its hd/32 group zeros, in bf16 (a group is 32 channels of
// one position). Codes lie in blocks of 8 positions (4 hd bytes) in the order the decode kernel's warps hold them:
// lane 4g + t of a warp finds its words w = 0 .. hd/32-1 of a block at (4g + t) * hd/8 bytes, one 16-byte (hd 128)
// or 8-byte load. A word is 8 codes of group w, nibble i of its low and high half being
//   K: position g, channels 32w + 8t + 2i and 32w + 8t + 2i + 1 (pairs of channels: the k index of q . K)
//   V: positions 2t and 2t + 1, channel 32w + 4g + i             (pairs of positions: the k index of P . V)
// so `word & 0x000f000f` is a pair of fp16 numbers n * 2^-24 (subnormals: exact, no offset to take away) and
// `word & 0x00f000f0` the next pair times 16: the fragments of mma.sync.m16n8k16, in 5 operations per 8 codes.
//
// Quantiser of a group: z = min (a bf16 input, exact), s = the smallest bf16 >= (max - min) / 15, n = (x - z) / s to
// the nearest whole number, half to even, so |s n + z - x| <= s / 2 and n <= 15 without a clamp. A group that holds a
// NaN or an infinity (or whose spread overflows fp32) reads back as NaN.
#pragma once
#include "common.cuh"

namespace kv4 {

constexpr int PAGE = 64;   // positions per page
constexpr int HALF = 32;   // positions per half: one tile of the decode kernel
constexpr int GROUP = 32;  // channels per scale and zero

template <int HD>
struct Fmt {
    static constexpr int W = HD / GROUP;          // groups per position, words per lane and block
    static constexpr int BLOCK = 4 * HD;          // bytes of codes of 8 positions
    static constexpr int CODES = 4 * BLOCK;       // bytes of K (or V) codes of a half
    static constexpr int ROW = 4 * W;             // bytes of a meta row
    static constexpr int META = HALF * ROW;       // bytes of K (or V) meta of a half
    static constexpr int KMETA = 2 * CODES, VMETA = KMETA + META;
    static constexpr int HALFB = VMETA + META;    // bytes of a half: 5120 (hd 128), 2560 (hd 64)
    static constexpr int UNIT = 2 * HALFB;
};

// hd/32 32-bit words, loaded and stored whole
template <int W>
struct Words {
    uint32_t v[W];
};
template <int W>
__device__ __forceinline__ Words<W> ld_words(const void *p) {
    Words<W> r;
    if constexpr (W == 4) {
        const uint4 u = *static_cast<const uint4 *>(p);
        r.v[0] = u.x, r.v[1] = u.y, r.v[2] = u.z, r.v[3] = u.w;
    } else {
        const uint2 u = *static_cast<const uint2 *>(p);
        r.v[0] = u.x, r.v[1] = u.y;
    }
    return r;
}
template <int W>
__device__ __forceinline__ void st_words(void *p, const Words<W> &r) {
    if constexpr (W == 4) *static_cast<uint4 *>(p) = make_uint4(r.v[0], r.v[1], r.v[2], r.v[3]);
    else *static_cast<uint2 *>(p) = make_uint2(r.v[0], r.v[1]);
}

// Group w's scale and zero of a meta row (bf16 pairs in words; a bf16 is the upper half of an fp32).
template <int W>
__device__ __forceinline__ float row_bf16(const Words<W> &m, int i) {
    return __uint_as_float(i & 1 ? m.v[i >> 1] & 0xffff0000u : m.v[i >> 1] << 16);
}
template <int W>
__device__ __forceinline__ float row_scale(const Words<W> &m, int w) { return row_bf16<W>(m, w); }
template <int W>
__device__ __forceinline__ float row_zero(const Words<W> &m, int w) { return row_bf16<W>(m, W + w); }

// ---- the quantiser -------------------------------------------------------------------------------------------

// (max, -min) of a bf16 pair's two values and of two such results: NaN propagates, negation is exact, so one packed
// maximum (and one shuffle) reduces both.
__device__ __forceinline__ __nv_bfloat162 as_bf2(uint32_t u) { return *reinterpret_cast<__nv_bfloat162 *>(&u); }
__device__ __forceinline__ uint32_t as_u32(__nv_bfloat162 b) { return *reinterpret_cast<uint32_t *>(&b); }
__device__ __forceinline__ uint32_t range_of(uint32_t mx2, uint32_t mn2) {  // packed maxima and minima -> (max, -min)
    const uint32_t a = __byte_perm(mx2, mn2 ^ 0x80008000u, 0x5410), b = __byte_perm(mx2, mn2 ^ 0x80008000u, 0x7632);
    return as_u32(__hmax2_nan(as_bf2(a), as_bf2(b)));
}
__device__ __forceinline__ uint32_t range_max(uint32_t a, uint32_t b) { return as_u32(__hmax2_nan(as_bf2(a), as_bf2(b))); }

struct Quant {
    float s, z, rinv;  // rinv: 1 / s, its last bit a mark (see quant_of); 0 for a scale of 0 or NaN
};
constexpr float TINY = 0.000244140625f;  // 2^-12
// s, the smallest bf16 >= D / 15 with D = max - min rounded up in fp32 (15 s has 12 bits, so rounding D up to fp32 does
// not change which s is enough): D times a float a little above 1 / 15, cut to bf16, is it or the one before it, and
// 15 s >= D, exact, tells. A scale that is not finite becomes NaN.
__device__ __forceinline__ Quant quant_of(uint32_t range) {
    const float2 r = unpack_bf16x2(range);  // max, -min
    Quant q;
    q.z = -r.y;
    const float D = __fadd_ru(r.x, r.y);
    const uint32_t b = __float_as_uint(D * __uint_as_float(0x3d88888au)) & 0xffff0000u;
    q.s = __uint_as_float(15.f * __uint_as_float(b) >= D ? b : b + 0x10000u);
    if (!(D < INFINITY)) q.s = __uint_as_float(0x7fc00000u);
    q.rinv = __fdividef(1.f, q.s);
    // quant_pairs takes x - z as fp32 has it, which is exact for ordinary groups: where z is 0 or at least 2^-12 s, and x
    // too, both are multiples of 2^-19 of the power of two at or below s, and the difference is below 2^5 of it. Where x
    // is smaller, but not 0, x - z is far from every border unless 0 itself lies on one. The last bit of 1 / s marks
    // groups that may be other than that, and scales without a normal reciprocal.
    const float n = __fadd_rn(fmaf(-q.z, q.rinv, 12582912.f), -12582912.f);
    const bool odd = fabsf(fmaf(-n, q.s, -q.z)) == 0.5f * q.s || (q.z != 0.f && fabsf(q.z) < q.s * TINY) || q.s < 7.9e-31f;
    q.rinv = q.s > 0.f ? __uint_as_float((__float_as_uint(q.rinv) & ~1u) | odd) : 0.f;
    return q;
}
// The nearest multiple decided exactly: x - z = d + e (two-sum), r = d - n s (n s has 12 bits, n is at most one off), all
// times a power of two where 1 / s would not be a normal number.
__device__ __forceinline__ uint32_t quant_exact(float x, float z, float s) {
    if (!(s > 0.f)) return 0u;
    const float up = s < 9.1e-13f ? 1.2676506e30f : 1.f;  // 2^100 for scales below 2^-40
    const float dx = __fsub_rn(x, z), bb = __fsub_rn(dx, x);
    const float e = __fadd_rn(__fsub_rn(x, __fsub_rn(dx, bb)), __fsub_rn(-z, bb));
    const float d = dx * up, sc = s * up, h = 0.5f * sc;
    float n = fminf(fmaxf(rintf(d * __fdividef(1.f, sc)), 0.f), 15.f);
    const float r = fmaf(-n, sc, d);
    const bool odd = static_cast<int>(n) & 1;
    if (r > h || (r == h && (e > 0.f || (e == 0.f && odd)))) n += 1.f;
    else if (r < -h || (r == -h && (e < 0.f || (e == 0.f && odd)))) n -= 1.f;
    return static_cast<uint32_t>(n);
}
// The codes of NP bf16 pairs, nibble i of the low and high half being pair i's two values. The quotient (x - z) / s is
// corrected to the nearest float, so a tie among whole numbers is one exactly (among bf16 numbers ties are common: one
// value in 370 of normal ones) and nothing else becomes one, being 2^-20 or more off; adding 1.5 * 2^23 rounds it, ties to
// even, and leaves n in the low bits. `marks` collects 1 / s: where its last bit is set, quant_marked has to look at these
// codes. (Checks behind each group would cost as much as the codes.)
template <int NP>
__device__ __forceinline__ uint32_t quant_pairs(const uint32_t (&x)[NP], const Quant &q, uint32_t &marks) {
    const float magic = 12582912.f;
    const float2 rv = make_float2(q.rinv, q.rinv), ms = make_float2(-q.s, -q.s);
    const float2 mz = make_float2(-q.z, -q.z), mg = make_float2(magic, magic);
    uint32_t lo = 0, hi = 0;
#pragma unroll
    for (int i = NP - 1; i >= 0; i--) {
        const float2 d = add2(make_float2(__uint_as_float(x[i] << 16), __uint_as_float(x[i] & 0xffff0000u)), mz);
        const float2 t = mul2(d, rv);
        const float2 a = add2(fma2(fma2(t, ms, d), rv, t), mg);
        lo = lo * 16u + __float_as_uint(a.x);  // the magic number's own bits leave the low 16
        hi = hi * 16u + __float_as_uint(a.y);
    }
    marks |= __float_as_uint(q.rinv);
    return __byte_perm(lo, hi, 0x5410);
}
// What a mark stands for, in the codes of quant_pairs: where 0 lies on a border, -z = (m + 1/2) s, a value tiny beside s
// has m + 1 or m by its sign. True where the codes have to be made by quant_exact instead.
template <int NP>
__device__ __forceinline__ bool quant_marked(const uint32_t (&x)[NP], float s, float z, uint32_t &code) {
    const float n = rintf(-z * __fdividef(1.f, s)), r = fmaf(-n, s, -z), tiny = s * TINY;
    if (fabsf(r) == 0.5f * s) {
        const uint32_t m = static_cast<uint32_t>(r > 0.f ? n : n - 1.f);
#pragma unroll
        for (int i = 0; i < NP; i++) {
            const float2 f = unpack_bf16x2(x[i]);
            if (f.x != 0.f && fabsf(f.x) < tiny) code = (code & ~(15u << (4 * i))) | (m + (f.x > 0.f)) << (4 * i);
            if (f.y != 0.f && fabsf(f.y) < tiny)
                code = (code & ~(15u << (4 * i + 16))) | (m + (f.y > 0.f)) << (4 * i + 16);
        }
    }
    return (z != 0.f && fabsf(z) < tiny) || (s > 0.f && s < 7.9e-31f);
}
// Four nibbles of two pairs' codes (the low half's two, the high half's two) in the order of the four values
__device__ __forceinline__ uint32_t in_order(uint32_t c) {
    return (c & 0xfu) | (c >> 12 & 0xf0u) | (c << 4 & 0xf00u) | (c >> 8 & 0xf000u);
}
__device__ __forceinline__ uint32_t meta_bits(float a, float b) {  // two bf16-valued floats as a bf16 pair
    return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
}
__device__ __forceinline__ float scale_of(uint32_t meta) { return __uint_as_float(meta << 16); }
__device__ __forceinline__ float zero_of(uint32_t meta) { return __uint_as_float(meta & 0xffff0000u); }
__device__ __forceinline__ Quant quant_from(uint32_t meta, float rinv) {  // of meta_bits(s, z)
    Quant q;
    q.s = __uint_as_float(meta << 16);
    q.z = __uint_as_float(meta & 0xffff0000u);
    q.rinv = rinv;
    return q;
}

// The page of position p of take s: its unit of kv head h, or null (recorded) where the table names no page.
__device__ __forceinline__ uint8_t *unit_of(uint8_t *pool, const int *table, int s, int p, int h, int nk, int npages,
                                            int maxpages, int unit) {
    const int pi = p / PAGE;
    const int page = pi < maxpages ? table[static_cast<long>(s) * maxpages + pi] : -1;
    if (page < 0 || page >= npages) {
        record_error(OUMU_DEVERR_PAGE);
        return nullptr;
    }
    return pool + (static_cast<long>(page) * nk + h) * unit;
}

// ---- prompt writes and reads -----------------------------------------------------------------------------------

// Work of one warp: `per` blocks of 8 positions of one (take, kv head, K or V), aligned inside a page; the next block's
// rows are on their way while one is worked on.
struct Part {
    int s, h, v, block;  // v: 0 for K, 1 for V; the first block
    __device__ Part(long item, int parts, int nk) {
        const int hv = static_cast<int>(item % (2 * nk));
        const long sp = item / (2 * nk);
        h = hv >> 1;
        v = hv & 1;
        s = static_cast<int>(sp / parts);
        block = static_cast<int>(sp % parts);
    }
};

// A part's rows, where they go, and the work on one of its blocks: true where the codes have to be made again.
template <int HD>
struct WriteTo {
    using F = Fmt<HD>;
    static constexpr int W = F::W;
    const bf16 *src;  // row of position p of this head's k or v: src + p * pitch
    long pitch;
    uint8_t *u;       // the page's unit
    int p0, n, lane;  // rows of positions p0 .. p0 + n - 1
    __device__ __forceinline__ bool ok(int p) const { return p >= p0 && p < p0 + n; }

    __device__ __forceinline__ void load(int b, uint4 (&x)[W]) const {
        const int p = b * 8 + (lane >> 2);
#pragma unroll
        for (int w = 0; w < W; w++)
            x[w] = ok(p) ? __ldcs(reinterpret_cast<const uint4 *>(src + p * pitch + 32 * w + 8 * (lane & 3)))
                         : make_uint4(0, 0, 0, 0);
    }
    __device__ __forceinline__ void load(int b, uint2 (&x)[2][W]) const {
#pragma unroll
        for (int e = 0; e < 2; e++) {
            const int p = b * 8 + 2 * (lane & 3) + e;
#pragma unroll
            for (int w = 0; w < W; w++)
                x[e][w] = ok(p) ? __ldcs(reinterpret_cast<const uint2 *>(src + p * pitch + 32 * w + 4 * (lane >> 2)))
                                : make_uint2(0, 0);
        }
    }

    // K: lane 4g + t has channels 32w + 8t .. + 7 of position g
    __device__ __forceinline__ bool k_block(int b, const uint4 (&x)[W]) const {
        const int g = lane >> 2, t = lane & 3;
        Words<W> code, meta;
        uint32_t sz[W], marks = 0;
#pragma unroll
        for (int w = 0; w < W; w++) {
            const uint32_t xu[4] = {x[w].x, x[w].y, x[w].z, x[w].w};
            uint32_t mx = xu[0], mn = xu[0];
#pragma unroll
            for (int i = 1; i < 4; i++) {
                mx = as_u32(__hmax2_nan(as_bf2(mx), as_bf2(xu[i])));
                mn = as_u32(__hmin2_nan(as_bf2(mn), as_bf2(xu[i])));
            }
            uint32_t rg = range_of(mx, mn);
            rg = range_max(rg, __shfl_xor_sync(0xffffffffu, rg, 1));
            rg = range_max(rg, __shfl_xor_sync(0xffffffffu, rg, 2));
            const Quant q = quant_of(rg);
            code.v[w] = quant_pairs<4>(xu, q, marks);
            sz[w] = meta_bits(q.s, q.z);
        }
        if (!ok(b * 8 + g)) return false;
        bool open = false;
        if (marks & 1u) {
#pragma unroll
            for (int w = 0; w < W; w++) {
                const uint32_t xu[4] = {x[w].x, x[w].y, x[w].z, x[w].w};
                open = quant_marked<4>(xu, scale_of(sz[w]), zero_of(sz[w]), code.v[w]) || open;
            }
        }
        uint8_t *half = u + (b & 7) / 4 * F::HALFB;
        st_words<W>(half + (b & 3) * F::BLOCK + lane * 4 * W, code);
        if (t == 0) {
#pragma unroll
            for (int w = 0; w < W; w += 2) {
                meta.v[w / 2] = __byte_perm(sz[w], sz[w + 1], 0x5410);
                meta.v[W / 2 + w / 2] = __byte_perm(sz[w], sz[w + 1], 0x7632);
            }
            st_words<W>(half + F::KMETA + ((b & 3) * 8 + g) * F::ROW, meta);
        }
        return open;
    }

    // V: lane 4g + t has channels 32w + 4g .. + 3 of positions 2t and 2t + 1
    __device__ __forceinline__ bool v_block(int b, const uint2 (&x)[2][W]) const {
        const int g = lane >> 2, t = lane & 3;
        // ranges of the 2 W groups over the 8 lanes of a position pair: each exchange halves what a lane holds, until
        // lane g has one group's and works out its scale, which then goes to all
        uint32_t rg[2 * W];
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int w = 0; w < W; w++)
                rg[e * W + w] = range_of(as_u32(__hmax2_nan(as_bf2(x[e][w].x), as_bf2(x[e][w].y))),
                                         as_u32(__hmin2_nan(as_bf2(x[e][w].x), as_bf2(x[e][w].y))));
#pragma unroll
        for (int m = W, o = 16; m >= 1; m >>= 1, o >>= 1) {
            const bool up = lane & o;
#pragma unroll
            for (int i = 0; i < m; i++) {
                const uint32_t send = up ? rg[i] : rg[i + m], keep = up ? rg[i + m] : rg[i];
                rg[i] = range_max(keep, __shfl_xor_sync(0xffffffffu, send, o));
            }
        }
        if (W == 2) rg[0] = range_max(rg[0], __shfl_xor_sync(0xffffffffu, rg[0], 4));
        const Quant mine = quant_of(rg[0]);
        const uint32_t mine_sz = meta_bits(mine.s, mine.z);
        Words<W> code, meta;
        uint32_t sz[2][W], c[2][W], marks = 0;
#pragma unroll
        for (int w = 0; w < W; w++) {
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int from = (e * W + w) * (16 / W) + t;
                sz[e][w] = __shfl_sync(0xffffffffu, mine_sz, from);
                const Quant q = quant_from(sz[e][w], __shfl_sync(0xffffffffu, mine.rinv, from));
                const uint32_t pr[2] = {x[e][w].x, x[e][w].y};
                c[e][w] = quant_pairs<2>(pr, q, marks);
            }
        }
        const bool ok0 = ok(b * 8 + 2 * t), ok1 = ok(b * 8 + 2 * t + 1);
        bool open = false;
        if (marks & 1u) {
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int w = 0; w < W; w++) {
                    const uint32_t pr[2] = {x[e][w].x, x[e][w].y};
                    open = (quant_marked<2>(pr, scale_of(sz[e][w]), zero_of(sz[e][w]), c[e][w]) && (e ? ok1 : ok0)) || open;
                }
        }
#pragma unroll
        for (int w = 0; w < W; w++) code.v[w] = __byte_perm(in_order(c[0][w]), in_order(c[1][w]), 0x5410);
        uint8_t *half = u + (b & 7) / 4 * F::HALFB;
        uint8_t *dst = half + F::CODES + (b & 3) * F::BLOCK + lane * 4 * W;
        if (ok0 && ok1) {
            st_words<W>(dst, code);
        } else {  // one of the word's two positions belongs to this write: its halves only
#pragma unroll
            for (int w = 0; w < W; w++) {
                if (ok0) reinterpret_cast<uint16_t *>(dst)[2 * w] = static_cast<uint16_t>(code.v[w]);
                if (ok1) reinterpret_cast<uint16_t *>(dst)[2 * w + 1] = static_cast<uint16_t>(code.v[w] >> 16);
            }
        }
        if (g == 0) {
#pragma unroll
            for (int e = 0; e < 2; e++) {
                if (!(e ? ok1 : ok0)) continue;
#pragma unroll
                for (int w = 0; w < W; w += 2) {
                    meta.v[w / 2] = __byte_perm(sz[e][w], sz[e][w + 1], 0x5410);
                    meta.v[W / 2 + w / 2] = __byte_perm(sz[e][w], sz[e][w + 1], 0x7632);
                }
                st_words<W>(half + F::VMETA + ((b & 3) * 8 + 2 * t + e) * F::ROW, meta);
            }
        }
        return open;
    }

    // A block's codes once more, each by quant_exact, from the scales and zeros that stand in the page by now. For groups
    // that real caches hardly have: short rather than fast.
    __device__ __forceinline__ void exact(int b, int v) const {
        __syncwarp();
        uint8_t *half = u + (b & 7) / 4 * F::HALFB;
        const int g = lane >> 2, t = lane & 3;
        uint8_t *dst = half + v * F::CODES + (b & 3) * F::BLOCK + lane * 4 * W;
#pragma unroll 1
        for (int i = 0; i < 2 * W; i++) {  // 16-bit halves of the lane's words
            const int w = i >> 1, e = i & 1;
            const int p = b * 8 + (v ? 2 * t + e : g), c0 = 32 * w + (v ? 4 * g : 8 * t + e), step = v ? 1 : 2;
            if (!ok(p)) continue;
            const bf16 *row = reinterpret_cast<const bf16 *>(half + (v ? F::VMETA : F::KMETA) + p % HALF * F::ROW);
            const float s = bf2f(row[w]), z = bf2f(row[W + w]);
            uint32_t code = 0;
#pragma unroll 1
            for (int k = 0; k < 4; k++) code |= quant_exact(bf2f(src[p * pitch + c0 + k * step]), z, s) << (4 * k);
            reinterpret_cast<uint16_t *>(dst)[i] = static_cast<uint16_t>(code);
        }
    }
};

// 512 bytes are read and 160 written per position and kv head at hd 128; the quantiser's instructions (69 % of the issue
// slots) bound it as much as HBM. The lanes load row chunks in the order of the block's words, so a block's 512 bytes of
// codes leave in one 16-byte store per lane. 48 prompts of 427..4048 positions, 145 MB: 42.5 us (3.4 TB/s); one prompt of
// 1024: 4.0 us. At hd 128 the 80 registers that three CTAs an SM leave spill 24 bytes a thread.
template <int HD>
__global__ void __launch_bounds__(256, 3) k_kv4_write(const bf16 *qkv, uint8_t *pool, const int *table, const int *start,
                                                   const int *count, int B, int rows, int nq, int nk, int npages,
                                                   int maxpages, int parts, int per) {
    using F = Fmt<HD>;
    constexpr int W = F::W;
    const int lane = threadIdx.x & 31;
    const Part it(static_cast<long>(blockIdx.x) * 8 + (threadIdx.x >> 5), parts, nk);
    if (it.s >= B) return;
    const int p0 = start ? start[it.s] : 0, n = count ? min(count[it.s], rows) : rows;
    if (n <= 0) return;
    if (p0 < 0 || static_cast<long>(p0) + n > static_cast<long>(maxpages) * PAGE) {
        if (lane == 0 && it.block == 0) record_error(OUMU_DEVERR_LENGTH);
        return;
    }
    const int b0 = (p0 / (8 * per) + it.block) * per;
    const int first = max(b0, p0 / 8), last = min(b0 + per - 1, (p0 + n - 1) / 8);  // blocks with rows to write
    if (first > last) return;
    uint8_t *u = unit_of(pool, table, it.s, b0 * 8, it.h, nk, npages, maxpages, F::UNIT);
    if (!u) return;
    const long pitch = static_cast<long>(nq + 2 * nk) * HD;
    const WriteTo<HD> to{qkv + (static_cast<long>(it.s) * rows - p0) * pitch + (nq + it.v * nk + it.h) * HD, pitch, u, p0, n,
                         lane};
    unsigned again = 0;  // blocks, from the first, to be made again
    if (it.v == 0) {
        uint4 x[W], y[W];
        to.load(first, y);
        for (int b = first; b <= last; b++) {
#pragma unroll
            for (int w = 0; w < W; w++) x[w] = y[w];
            if (b < last) to.load(b + 1, y);
            if (to.k_block(b, x)) again |= 1u << (b - first);
        }
    } else {
        uint2 x[2][W], y[2][W];
        to.load(first, y);
        for (int b = first; b <= last; b++) {
#pragma unroll
            for (int e = 0; e < 2; e++)
#pragma unroll
                for (int w = 0; w < W; w++) x[e][w] = y[e][w];
            if (b < last) to.load(b + 1, y);
            if (to.v_block(b, x)) again |= 1u << (b - first);
        }
    }
    again = __reduce_or_sync(0xffffffffu, again);
    for (int b = first; again; b++, again >>= 1)
        if (again & 1) to.exact(b, it.v);
}

// The 4 codes of nibbles 0..3 of a 16-bit half, as values rounded once to bf16 (s n is exact, the sum rounds once
// in fp32 and once to bf16).
__device__ __forceinline__ float value_of(uint32_t half, int i, float s, float z) {
    // n from its bits: 2^23 + n, minus 2^23
    return fmaf(s, __uint_as_float(((half >> (4 * i)) & 15u) | 0x4b000000u) - 8388608.f, z);
}

// The write's order backwards; a part's codes and meta rows are all loaded before the first value is stored. Bound by HBM:
// the 48 prompts above, with 77 positions before each 150 MB, in 27.4 us (5.5 TB/s).
template <int HD, int PER>
__global__ void __launch_bounds__(256) k_kv4_read(uint8_t *pool, const int *table, const int *lens, const int *pos,
                                                  bf16 *kc, bf16 *vc, int B, int nk, int npages, int maxpages,
                                                  int maxlen, int parts) {
    using F = Fmt<HD>;
    constexpr int W = F::W;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const Part it(static_cast<long>(blockIdx.x) * 8 + (threadIdx.x >> 5), parts, nk);
    if (it.s >= B) return;
    int L = lens ? lens[it.s] : *pos + 1;
    const long room = min(static_cast<long>(maxlen), static_cast<long>(maxpages) * PAGE);
    if (L < 0 || L > room) {
        if (lane == 0 && it.block == 0) record_error(OUMU_DEVERR_LENGTH);
        L = L < 0 ? 0 : static_cast<int>(room);
    }
    const int b0 = it.block * PER;
    if (b0 * 8 >= L) return;
    const uint8_t *u = unit_of(pool, table, it.s, b0 * 8, it.h, nk, npages, maxpages, F::UNIT);
    if (!u) return;
    bf16 *dst = (it.v ? vc : kc) + ((static_cast<long>(it.s) * nk + it.h) * maxlen + b0 * 8) * HD;
    const int left = L - b0 * 8;
    Words<W> code[PER], m[PER][2];
#pragma unroll
    for (int i = 0; i < PER; i++) {
        if (i * 8 >= left) break;
        const uint8_t *half = u + ((b0 + i) & 7) / 4 * F::HALFB;
        code[i] = ld_words<W>(half + it.v * F::CODES + ((b0 + i) & 3) * F::BLOCK + lane * 4 * W);
        const uint8_t *rows = half + (it.v ? F::VMETA : F::KMETA) + ((b0 + i) & 3) * 8 * F::ROW;
        m[i][0] = ld_words<W>(rows + (it.v ? 2 * t : g) * F::ROW);
        if (it.v) m[i][1] = ld_words<W>(rows + (2 * t + 1) * F::ROW);
    }
#pragma unroll
    for (int i = 0; i < PER; i++) {
        if (i * 8 >= left) break;
        if (it.v == 0) {
            if (i * 8 + g >= left) continue;
#pragma unroll
            for (int w = 0; w < W; w++) {
                const float sc = row_scale<W>(m[i][0], w), z = row_zero<W>(m[i][0], w);
                const uint32_t lo = code[i].v[w] & 0xffffu, hi = code[i].v[w] >> 16;
                uint4 o;
                o.x = pack_bf16x2(value_of(lo, 0, sc, z), value_of(hi, 0, sc, z));
                o.y = pack_bf16x2(value_of(lo, 1, sc, z), value_of(hi, 1, sc, z));
                o.z = pack_bf16x2(value_of(lo, 2, sc, z), value_of(hi, 2, sc, z));
                o.w = pack_bf16x2(value_of(lo, 3, sc, z), value_of(hi, 3, sc, z));
                __stcs(reinterpret_cast<uint4 *>(dst + (i * 8 + g) * HD + 32 * w + 8 * t), o);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 2; e++) {
                if (i * 8 + 2 * t + e >= left) continue;
#pragma unroll
                for (int w = 0; w < W; w++) {
                    const float sc = row_scale<W>(m[i][e], w), z = row_zero<W>(m[i][e], w);
                    const uint32_t hf = code[i].v[w] >> (16 * e) & 0xffffu;
                    uint2 o;
                    o.x = pack_bf16x2(value_of(hf, 0, sc, z), value_of(hf, 1, sc, z));
                    o.y = pack_bf16x2(value_of(hf, 2, sc, z), value_of(hf, 3, sc, z));
                    __stcs(reinterpret_cast<uint2 *>(dst + (i * 8 + 2 * t + e) * HD + 32 * w + 4 * g), o);
                }
            }
        }
    }
}

}  // namespace kv4

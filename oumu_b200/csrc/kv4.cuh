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
    float s, z, rinv;
};
// Rounding up twice in fp32 (x - y, then / 15) and then to bf16 gives the smallest bf16 >= (max - min) / 15 itself:
// if a bf16 b is >= it, 15 b is >= max - min and has 12 bits, so neither step rounds past it.
__device__ __forceinline__ Quant quant_of(uint32_t range) {
    const float2 r = unpack_bf16x2(range);  // max, -min
    Quant q;
    q.z = -r.y;
    const float d = __fdiv_ru(__fadd_ru(r.x, r.y), 15.f);
    q.s = d != d ? d : __uint_as_float((__float_as_uint(d) + 0xffffu) & 0xffff0000u);
    q.rinv = __fdividef(1.f, q.s);
    return q;
}
// Nearest multiple near a border: x - z = d + e exactly (two-sum), r = d - n s exactly (n s has 12 bits).
__device__ __noinline__ int quant_exact(float x, float z, float s) {
    if (!(s > 0.f) || !(s < INFINITY)) return 0;
    const float d = __fsub_rn(x, z);
    const float bb = __fsub_rn(d, x);
    const float e = __fadd_rn(__fsub_rn(x, __fsub_rn(d, bb)), __fsub_rn(-z, bb));
    float n = rintf(__fdiv_rn(d, s));
    const float r = fmaf(-n, s, d), h = 0.5f * s;
    const bool odd = static_cast<int>(n) & 1;
    if (r > h || (r == h && (e > 0.f || (e == 0.f && odd)))) n += 1.f;
    else if (r < -h || (r == -h && (e < 0.f || (e == 0.f && odd)))) n -= 1.f;
    return static_cast<int>(fminf(fmaxf(n, 0.f), 15.f));
}
// The product with 1 / s is within 2^-21 of the quotient (at most 15): away from a border by more, rounding it is right.
__device__ __forceinline__ int quant_code(float x, const Quant &q) {
    const float t = __fsub_rn(x, q.z) * q.rinv;
    const float n = rintf(t);
    if (fabsf(t - n) < 0.4999f) return static_cast<int>(n);
    return quant_exact(x, q.z, q.s);  // NaN and infinities of the product come here too
}
__device__ __forceinline__ uint32_t meta_bits(float a, float b) {  // two bf16-valued floats as a bf16 pair
    return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632);
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

// One warp per (take, block of 8 positions, kv head, K or V). Bound by HBM (512 bytes read and 160 written per
// position and kv head at hd 128); the lanes load q-row chunks in the order of the block's words, so the block's
// 512 bytes of codes leave in one 16-byte store per lane.
template <int HD>
__global__ void __launch_bounds__(256) k_kv4_write(const bf16 *qkv, uint8_t *pool, const int *table, const int *start,
                                                   const int *count, int B, int rows, int nq, int nk, int npages,
                                                   int maxpages, int blocks) {
    using F = Fmt<HD>;
    constexpr int W = F::W;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const long item = static_cast<long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int hv = static_cast<int>(item % (2 * nk)), h = hv >> 1;
    const long sb = item / (2 * nk);
    const int s = static_cast<int>(sb / blocks), b = static_cast<int>(sb % blocks);
    if (s >= B) return;
    const int p0 = start ? start[s] : 0, n = count ? min(count[s], rows) : rows;
    if (n <= 0) return;
    if (p0 < 0 || static_cast<long>(p0) + n > static_cast<long>(maxpages) * PAGE) {
        if (lane == 0 && b == 0) record_error(OUMU_DEVERR_LENGTH);
        return;
    }
    const int pb = (p0 / 8 + b) * 8;  // the block's first position
    if (pb >= p0 + n) return;
    uint8_t *u = unit_of(pool, table, s, pb, h, nk, npages, maxpages, F::UNIT);
    if (!u) return;
    u += (pb % PAGE) / HALF * F::HALFB;
    const int r0 = pb % HALF;
    const long pitch = static_cast<long>(nq + 2 * nk) * HD;
    const bf16 *src = qkv + (static_cast<long>(s) * rows + pb - p0) * pitch + (nq + (hv & 1) * nk + h) * HD;
    auto ok = [&](int i) { return pb + i >= p0 && pb + i < p0 + n; };
    Words<W> code, meta;
    if (!(hv & 1)) {  // K: lane 4g + t has channels 32w + 8t .. + 7 of position g
        uint4 x[W];
#pragma unroll
        for (int w = 0; w < W; w++)
            x[w] = ok(g) ? *reinterpret_cast<const uint4 *>(src + g * pitch + 32 * w + 8 * t) : make_uint4(0, 0, 0, 0);
        uint32_t sc[W], zc[W];
#pragma unroll
        for (int w = 0; w < W; w++) {
            const uint32_t *xu = reinterpret_cast<const uint32_t *>(&x[w]);
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
            uint32_t c = 0;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 f = unpack_bf16x2(xu[i]);
                c |= static_cast<uint32_t>(quant_code(f.x, q)) << (4 * i);
                c |= static_cast<uint32_t>(quant_code(f.y, q)) << (4 * i + 16);
            }
            code.v[w] = c;
            sc[w] = __float_as_uint(q.s) >> 16;
            zc[w] = __float_as_uint(q.z) >> 16;
        }
        if (!ok(g)) return;
        st_words<W>(u + r0 / 8 * F::BLOCK + lane * 4 * W, code);
#pragma unroll
        for (int w = 0; w < W; w += 2) {
            meta.v[w / 2] = sc[w] | sc[w + 1] << 16;
            meta.v[W / 2 + w / 2] = zc[w] | zc[w + 1] << 16;
        }
        if (t == 0) st_words<W>(u + F::KMETA + (r0 + g) * F::ROW, meta);
    } else {  // V: lane 4g + t has channels 32w + 4g .. + 3 of positions 2t and 2t + 1
        uint2 x[2][W];
#pragma unroll
        for (int e = 0; e < 2; e++)
#pragma unroll
            for (int w = 0; w < W; w++)
                x[e][w] = ok(2 * t + e) ? *reinterpret_cast<const uint2 *>(src + (2 * t + e) * pitch + 32 * w + 4 * g)
                                        : make_uint2(0, 0);
        uint32_t sc[2][W], zc[2][W];
#pragma unroll
        for (int w = 0; w < W; w++) {
            code.v[w] = 0;
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const uint2 y = x[e][w];
                uint32_t rg = range_of(as_u32(__hmax2_nan(as_bf2(y.x), as_bf2(y.y))),
                                       as_u32(__hmin2_nan(as_bf2(y.x), as_bf2(y.y))));
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) rg = range_max(rg, __shfl_xor_sync(0xffffffffu, rg, o));
                const Quant q = quant_of(rg);
                const float2 a = unpack_bf16x2(y.x), c = unpack_bf16x2(y.y);
                const uint32_t n4 = quant_code(a.x, q) | quant_code(a.y, q) << 4 | quant_code(c.x, q) << 8 |
                                    quant_code(c.y, q) << 12;
                code.v[w] |= n4 << (16 * e);
                sc[e][w] = __float_as_uint(q.s) >> 16;
                zc[e][w] = __float_as_uint(q.z) >> 16;
            }
        }
        uint8_t *dst = u + F::CODES + r0 / 8 * F::BLOCK + lane * 4 * W;
        if (ok(2 * t) && ok(2 * t + 1)) {
            st_words<W>(dst, code);
        } else {  // one of the word's two positions belongs to this write: its halves only
#pragma unroll
            for (int e = 0; e < 2; e++)
                if (ok(2 * t + e))
#pragma unroll
                    for (int w = 0; w < W; w++)
                        reinterpret_cast<uint16_t *>(dst)[2 * w + e] = static_cast<uint16_t>(code.v[w] >> (16 * e));
        }
        if (g == 0) {
#pragma unroll
            for (int e = 0; e < 2; e++) {
                if (!ok(2 * t + e)) continue;
#pragma unroll
                for (int w = 0; w < W; w += 2) {
                    meta.v[w / 2] = sc[e][w] | sc[e][w + 1] << 16;
                    meta.v[W / 2 + w / 2] = zc[e][w] | zc[e][w + 1] << 16;
                }
                st_words<W>(u + F::VMETA + (r0 + 2 * t + e) * F::ROW, meta);
            }
        }
    }
}

// The 4 codes of nibbles 0..3 of a 16-bit half, as values rounded once to bf16 (s n is exact, the sum rounds once
// in fp32 and once to bf16).
__device__ __forceinline__ float value_of(uint32_t half, int i, float s, float z) {
    return fmaf(s, static_cast<float>((half >> (4 * i)) & 15u), z);
}

// One warp per (take, block of 8 positions, kv head, K or V), the write's order backwards.
template <int HD>
__global__ void __launch_bounds__(256) k_kv4_read(uint8_t *pool, const int *table, const int *lens, const int *pos,
                                                  bf16 *kc, bf16 *vc, int B, int nk, int npages, int maxpages,
                                                  int maxlen, int blocks) {
    using F = Fmt<HD>;
    constexpr int W = F::W;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const long item = static_cast<long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int hv = static_cast<int>(item % (2 * nk)), h = hv >> 1;
    const long sb = item / (2 * nk);
    const int s = static_cast<int>(sb / blocks), b = static_cast<int>(sb % blocks);
    if (s >= B) return;
    int L = lens ? lens[s] : *pos + 1;
    const long room = min(static_cast<long>(maxlen), static_cast<long>(maxpages) * PAGE);
    if (L < 0 || L > room) {
        if (lane == 0 && b == 0) record_error(OUMU_DEVERR_LENGTH);
        L = L < 0 ? 0 : static_cast<int>(room);
    }
    const int pb = b * 8;
    if (pb >= L) return;
    const uint8_t *u = unit_of(pool, table, s, pb, h, nk, npages, maxpages, F::UNIT);
    if (!u) return;
    u += (pb % PAGE) / HALF * F::HALFB;
    const int r0 = pb % HALF;
    const Words<W> code = ld_words<W>(u + (hv & 1) * F::CODES + r0 / 8 * F::BLOCK + lane * 4 * W);
    bf16 *dst = (hv & 1 ? vc : kc) + ((static_cast<long>(s) * nk + h) * maxlen + pb) * HD;
    if (!(hv & 1)) {
        if (pb + g >= L) return;
        const Words<W> m = ld_words<W>(u + F::KMETA + (r0 + g) * F::ROW);
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float sc = row_scale<W>(m, w), z = row_zero<W>(m, w);
            const uint32_t lo = code.v[w] & 0xffffu, hi = code.v[w] >> 16;
            uint4 o;
            o.x = pack_bf16x2(value_of(lo, 0, sc, z), value_of(hi, 0, sc, z));
            o.y = pack_bf16x2(value_of(lo, 1, sc, z), value_of(hi, 1, sc, z));
            o.z = pack_bf16x2(value_of(lo, 2, sc, z), value_of(hi, 2, sc, z));
            o.w = pack_bf16x2(value_of(lo, 3, sc, z), value_of(hi, 3, sc, z));
            *reinterpret_cast<uint4 *>(dst + g * HD + 32 * w + 8 * t) = o;
        }
    } else {
#pragma unroll
        for (int e = 0; e < 2; e++) {
            if (pb + 2 * t + e >= L) continue;
            const Words<W> m = ld_words<W>(u + F::VMETA + (r0 + 2 * t + e) * F::ROW);
#pragma unroll
            for (int w = 0; w < W; w++) {
                const float sc = row_scale<W>(m, w), z = row_zero<W>(m, w);
                const uint32_t hf = code.v[w] >> (16 * e) & 0xffffu;
                uint2 o;
                o.x = pack_bf16x2(value_of(hf, 0, sc, z), value_of(hf, 1, sc, z));
                o.y = pack_bf16x2(value_of(hf, 2, sc, z), value_of(hf, 3, sc, z));
                *reinterpret_cast<uint2 *>(dst + (2 * t + e) * HD + 32 * w + 4 * g) = o;
            }
        }
    }
}

}  // namespace kv4

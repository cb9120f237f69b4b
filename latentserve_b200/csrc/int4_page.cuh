// The page record of the 4-bit KV cache, and one token's way into it.
//
// A value is held as a code 0..15 with value = lo + step * code; lo and step are fp16, one
// pair per (token, head, group of 32, 64 or 128 channels), G = 128 / group. All a page (16
// tokens) holds of one KV head is ONE contiguous record of 2048 + 128 G bytes, so that the
// attention kernel fetches a page-head with one bulk copy and a page is forked or moved as
// plain bytes:
//
//   [0, 1024)         K codes, token t at 64 t: [j 4][q 4] words; nibble i of word (q, j) is
//                     channel 32 q + 8 j + i
//   [1024, 2048)      V codes: [c 2][lane 32][i 4] words, lane = 4 g + j. The word's byte
//                     2 e + f belongs to token 8 f + 2 j + e and holds channel 64 c + 16 i + g
//                     in its low nibble, that channel + 8 in its high one
//   [2048, +64 G)     K scales fp16 [16 tokens][G steps, G lows]
//   [.., +32 G)       V steps fp16 [j 4][G][f 2][e 2]
//   [.., +32 G)       V lows, the same order
//
// The orders are those of the tensor-core fragments (see Int4State in paged_decode_int4.cu):
// a lane gets what it feeds to the MMAs of a whole page with two 16-byte loads for K and two
// for V. No byte is shared by two tokens, so tokens are written in any order, by any thread,
// without reading the record first.
#pragma once

#include "ls_common.cuh"

namespace ls {

constexpr int kI4V = 1024;                 // byte offsets inside a record
constexpr int kI4Scales = 2048;
__host__ __device__ constexpr int int4_record_bytes(int G) { return 2048 + 128 * G; }
__host__ __device__ constexpr int int4_v_steps(int G) { return kI4Scales + 64 * G; }
__host__ __device__ constexpr int int4_v_lows(int G) { return kI4Scales + 96 * G; }

// Index (in fp16 units, from the start of the V steps) of token t's entry of group `grp`.
__device__ __forceinline__ int int4_v_scale_index(int G, int t, int grp) {
    return ((t & 7) >> 1) * 4 * G + 4 * grp + 2 * (t >> 3) + (t & 1);
}

// What the quantiser makes of a lane's eight channels: their codes, nibble i channel i, and the
// group's step and lo.
struct Int4Fit {
    uint32_t codes;
    __half step, lo;
};

// The quantiser as its formula reads. Out of line: the usual row does not come here.
template <int G>
static __device__ __noinline__ Int4Fit int4_fit_divided(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3) {
    const uint32_t raw[4] = {c0, c1, c2, c3};            // (as words: a uint4 would go through memory)
    const __half2* h2 = reinterpret_cast<const __half2*>(raw);
    Int4Fit fit;
    float x[8], lo = 65504.f, hi = -65504.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(h2[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = isnan(x[i]) ? 0.f : fminf(fmaxf(x[i], -65504.f), 65504.f);
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
    }
#pragma unroll
    for (int off = 1; off < 16 / G; off <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(LS_FULL_MASK, lo, off));
        hi = fmaxf(hi, __shfl_xor_sync(LS_FULL_MASK, hi, off));
    }
    fit.step = __float2half_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f));
    fit.lo = __float2half_rn(lo);
    const float t = __half2float(fit.step);
    fit.codes = 0;
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
        float v = x[0];                                   // (no indexing by i: x stays in registers)
#pragma unroll
        for (int k = 1; k < 8; ++k) v = i == k ? x[k] : v;
        const float u = t > 0.f ? rintf(__fdiv_rn(__fsub_rn(v, lo), t)) : 0.f;
        fit.codes |= (uint32_t)fminf(fmaxf(u, 0.f), 15.f) << (4 * i);
    }
    return fit;
}

// Eight neighbouring channels a lane, 16 / G lanes a group, a row in 16 lanes; all lanes of the warp
// take part. lo = min x, step = fp16((max - lo) / 15), code = rne((x - lo) / step), at most 15.
// NaN counts as 0 and infinities as +-65504: what is stored is always finite, and a step is at
// most 131008 / 15.
//
// Computing bounds this, so the usual row goes without a division per channel, two channels an
// instruction: with y the correctly rounded 1 / step, u = d y, the quotient d / step correctly
// rounded is u + (d - u step) y (Markstein; the fused residual is exact), and adding 1.5 2^23
// rounds it to an integer, halves to even. A warp with a value that is not finite, or with
// quotients past 15 (subnormal steps), divides.
template <int G>
__device__ __forceinline__ Int4Fit int4_fit(const uint4& raw) {
    const __half2* h2 = reinterpret_cast<const __half2*>(&raw);
    // Minimum and negated maximum side by side, NaN passing through.
    const __half2 mn = __hmin2_nan(__hmin2_nan(h2[0], h2[1]), __hmin2_nan(h2[2], h2[3]));
    const __half2 mx = __hmax2_nan(__hmax2_nan(h2[0], h2[1]), __hmax2_nan(h2[2], h2[3]));
    __half2 both = __hmin2_nan(__halves2half2(__low2half(mn), __hneg(__low2half(mx))),
                               __halves2half2(__high2half(mn), __hneg(__high2half(mx))));
#pragma unroll
    for (int off = 1; off < 16 / G; off <<= 1) {
        const uint32_t o = __shfl_xor_sync(LS_FULL_MASK, *reinterpret_cast<const uint32_t*>(&both), off);
        both = __hmin2_nan(both, *reinterpret_cast<const __half2*>(&o));
    }
    float lo = __low2float(both);
    const float range = -__high2float(both) - lo;
    // range / 15, correctly rounded: the quotient by the rounded reciprocal, corrected once.
    const float fifteenth = 1.f / 15.f, q0 = range * fifteenth;
    Int4Fit fit;
    fit.step = __float2half_rn(fmaf(fmaf(-15.f, q0, range), fifteenth, q0));
    fit.lo = __low2half(both);
    const float s = __half2float(fit.step);
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(s));
    y = s > 0.f ? fmaf(fmaf(-s, y, 1.f), y, y) : 0.f;     // a group of one value has step 0: codes 0
    const float magic = 12582912.f;
    const f32x2 lo2 = pack2(-lo, -lo), y2 = pack2(y, y), up = pack2(magic, magic), down = pack2(-magic, -magic), s2 = pack2(-s, -s);
    f32x2 z[4];                                           // codes as floats, two neighbours each
    float r_first[2];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 x = __half22float2(h2[i]);
        const f32x2 d = add2(pack2(x.x, x.y), lo2), u = mul2(d, y2), r = add2(fma2(fma2(u, s2, d), y2, u), up);
        z[i] = add2(r, down);
        float skip;
        if (i % 2 == 0) unpack2(r, r_first[i / 2], skip);
    }
    // Four codes make sixteen bits on top of 1.5 2^23, exactly.
    uint32_t quad[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float z1, z2, z3, skip;
        unpack2(z[2 * i], skip, z1);
        unpack2(z[2 * i + 1], z2, z3);
        quad[i] = __float_as_uint(fmaf(fmaf(z3, 256.f, z1), 16.f, fmaf(z2, 256.f, r_first[i])));
    }
    fit.codes = prmt(quad[0], quad[1], 0x5410);
    const bool plain = range <= 131008.f && range * y < 15.4f;
    if (__all_sync(LS_FULL_MASK, plain)) return fit;

    return int4_fit_divided<G>(raw.x, raw.y, raw.z, raw.w);
}

// Bytes k of four words next to one another: out[k] = {w0.k, w1.k, w2.k, w3.k}.
__device__ __forceinline__ void transpose_bytes(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, uint32_t (&out)[4]) {
    const uint32_t a = prmt(w0, w1, 0x5140), b = prmt(w2, w3, 0x5140);     // {w0.0, w1.0, w0.1, w1.1}
    const uint32_t c = prmt(w0, w1, 0x7362), d = prmt(w2, w3, 0x7362);
    out[0] = prmt(a, b, 0x5410);
    out[1] = prmt(a, b, 0x7632);
    out[2] = prmt(c, d, 0x5410);
    out[3] = prmt(c, d, 0x7632);
}

__device__ __forceinline__ uint32_t half_pair(__half lo, __half hi) {
    const __half2 h = __halves2half2(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// One token's K codes and scales, lane hl of its sixteen.
template <int G>
__device__ __forceinline__ void int4_put_k(uint8_t* rec, int t, const Int4Fit& fit, int hl) {
    *reinterpret_cast<uint32_t*>(rec + 64 * t + 16 * (hl & 3) + 4 * (hl >> 2)) = fit.codes;
    if (hl % (16 / G) == 0) {
        __half* at = reinterpret_cast<__half*>(rec + kI4Scales) + 2 * G * t + hl / (16 / G);
        at[0] = fit.step;
        at[G] = fit.lo;
    }
}

template <int G>
__device__ __forceinline__ void int4_put_v_scales(uint8_t* rec, int t, const Int4Fit& fit, int hl) {
    if (hl % (16 / G) == 0) {
        __half* at = reinterpret_cast<__half*>(rec + int4_v_steps(G)) + int4_v_scale_index(G, t, hl / (16 / G));
        at[0] = fit.step;
        at[16 * G] = fit.lo;
    }
}

// A V byte holds channel c of a token in its low nibble and channel c + 8, the neighbouring lane's,
// in its high one. Of the pair's eight bytes the even lane gets the first four, the odd lane the rest.
__device__ __forceinline__ uint32_t int4_v_bytes(uint32_t codes, int odd) {
    const uint32_t other = __shfl_xor_sync(LS_FULL_MASK, codes, 1);
    // Nibbles a0 a1 a2 a3 b0 b1 b2 b3 (a: the even lane's), then shuffled to a0 b0 a1 b1 a2 b2 a3 b3.
    uint32_t x = odd ? prmt(other, codes, 0x7632) : prmt(codes, other, 0x5410);
    uint32_t t = (x ^ (x >> 8)) & 0x0000ff00u;
    x ^= t ^ (t << 8);
    t = (x ^ (x >> 4)) & 0x00f000f0u;
    return x ^ t ^ (t << 4);
}

// Byte address of row 0 of a lane's V words: tile hl / 2, lanes 4 g + j of the record.
__device__ __forceinline__ int int4_v_word(int j, int hl) {
    return kI4V + (hl >> 3) * 512 + (16 * (hl & 1) + j) * 16 + ((hl >> 1) & 3) * 4;
}

template <int G>
__device__ __forceinline__ void int4_put_v(uint8_t* rec, int t, const Int4Fit& fit, uint32_t bytes, int hl) {
    uint8_t* dst = rec + int4_v_word((t & 7) >> 1, hl) + 2 * (t & 1) + (t >> 3);
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[i * 64] = (uint8_t)(bytes >> (8 * i));
    int4_put_v_scales<G>(rec, t, fit, hl);
}

// One token's K row (lanes 0-15) and V row (lanes 16-31), lane hl of a half holding channels
// 8 hl .. 8 hl + 7, quantised by one warp into the record `rec`: only that token's bytes.
template <int G>
__device__ __forceinline__ void int4_put_token(uint8_t* rec, int t, const uint4& raw, int lane) {
    const Int4Fit fit = int4_fit<G>(raw);
    const uint32_t bytes = int4_v_bytes(fit.codes, lane & 1);
    if (lane < 16) int4_put_k<G>(rec, t, fit, lane);
    else int4_put_v<G>(rec, t, fit, bytes, lane & 15);
}

// A whole page's rows in a CTA of four warps: warps 0, 1 have K, 2, 3 V, four tokens a half-warp.
// V tokens 2j, 2j + 1, 2j + 8, 2j + 9 share words of codes, so they are one half-warp's.
__device__ __forceinline__ int page_token(int warp, int lane, int k) {
    const int j = 2 * (warp & 1) + (lane >> 4);
    return warp < 2 ? 4 * j + k : 2 * j + (k & 1) + 8 * (k >> 1);
}

template <int G>
__device__ __forceinline__ void int4_put_page(uint8_t* rec, const uint4 (&raw)[4], int warp, int lane) {
    const int hl = lane & 15;
    if (warp < 2) {
#pragma unroll
        for (int k = 0; k < 4; ++k) int4_put_k<G>(rec, page_token(warp, lane, k), int4_fit<G>(raw[k]), hl);
        return;
    }
    uint32_t bytes[4], words[4];
    __half steps[4], lows[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const Int4Fit fit = int4_fit<G>(raw[k]);
        bytes[k] = int4_v_bytes(fit.codes, lane & 1);
        steps[k] = fit.step;
        lows[k] = fit.lo;
    }
    const int j = 2 * (warp & 1) + (lane >> 4);
    if (hl % (16 / G) == 0) {                                 // [f][e] of the four tokens lie side by side
        uint8_t* at = rec + int4_v_steps(G) + 8 * G * j + 8 * (hl / (16 / G));
        *reinterpret_cast<uint2*>(at) = make_uint2(half_pair(steps[0], steps[1]), half_pair(steps[2], steps[3]));
        *reinterpret_cast<uint2*>(at + 32 * G) = make_uint2(half_pair(lows[0], lows[1]), half_pair(lows[2], lows[3]));
    }
    transpose_bytes(bytes[0], bytes[2], bytes[1], bytes[3], words);      // byte 2 e + f: tokens 2j, 2j+8, 2j+1, 2j+9
    uint8_t* dst = rec + int4_v_word(j, hl);
#pragma unroll
    for (int i = 0; i < 4; ++i) *reinterpret_cast<uint32_t*>(dst + i * 64) = words[i];
}

// Eight codes, one a byte, as fp16 values lo + step * code, each rounded once.
__device__ __forceinline__ uint4 int4_values(uint32_t b0, uint32_t b1, __half step, __half lo) {
    const __half2 s2 = __half2half2(step), l2 = __half2half2(lo), off = __float2half2_rn(1024.f);
    uint4 out;
    uint32_t* o = reinterpret_cast<uint32_t*>(&out);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t n = prmt(i < 2 ? b0 : b1, 0x64646464u, (i & 1) ? 0x4342 : 0x4140);   // 1024 + code
        const __half2 v = __hfma2(s2, __hsub2(*reinterpret_cast<const __half2*>(&n), off), l2);
        o[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
    return out;
}

// The inverse of int4_put_page: channels 8 hl .. 8 hl + 7 of page_token(warp, lane, k) into out[k].
template <int G>
__device__ __forceinline__ void int4_get_page(const uint8_t* rec, int warp, int lane, uint4 (&out)[4]) {
    const int hl = lane & 15, odd = lane & 1, grp = hl / (16 / G), j = 2 * (warp & 1) + (lane >> 4);
    uint32_t words[4];
    __half steps[4], lows[4];
    if (warp < 2) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int t = page_token(warp, lane, k);
            const __half* sc = reinterpret_cast<const __half*>(rec + kI4Scales) + 2 * G * t + grp;
            words[k] = *reinterpret_cast<const uint32_t*>(rec + 64 * t + 16 * (hl & 3) + 4 * (hl >> 2));
            steps[k] = sc[0];
            lows[k] = sc[G];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t even = words[k] & 0x0f0f0f0fu, uneven = (words[k] >> 4) & 0x0f0f0f0fu;
            out[k] = int4_values(prmt(even, uneven, 0x5140), prmt(even, uneven, 0x7362), steps[k], lows[k]);
        }
        return;
    }
    uint32_t bytes[4];
    const uint8_t *src = rec + int4_v_word(j, hl), *at = rec + int4_v_steps(G) + 8 * G * j + 8 * grp;
#pragma unroll
    for (int i = 0; i < 4; ++i) words[i] = *reinterpret_cast<const uint32_t*>(src + i * 64);
    *reinterpret_cast<uint2*>(steps) = *reinterpret_cast<const uint2*>(at);
    *reinterpret_cast<uint2*>(lows) = *reinterpret_cast<const uint2*>(at + 32 * G);
    transpose_bytes(words[0], words[1], words[2], words[3], bytes);      // bytes[k]: token (0, 8, 1, 9)[k] of the four
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t mine = bytes[(k & 1) * 2 + (k >> 1)], other = __shfl_xor_sync(LS_FULL_MASK, mine, 1);
        out[k] = int4_values(((odd ? other : mine) >> (4 * odd)) & 0x0f0f0f0fu,
                             ((odd ? mine : other) >> (4 * odd)) & 0x0f0f0f0fu, steps[k], lows[k]);
    }
}

}  // namespace ls

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

// Eight neighbouring channels a lane, 16 / G lanes a group, a row in 16 lanes; all lanes of the warp
// take part. lo = min x, step = fp16((max - lo) / 15), code = rne((x - lo) / step), at most 15.
// NaN counts as 0 and infinities as +-65504: what is stored is always finite, and a step is at
// most 131008 / 15.
//
// Computing bounds this, so the usual row goes without a division per channel: code = rne(d y) with
// y within 2^-23 of 1 / step, by adding and subtracting 1.5 2^23, two channels an instruction. That
// is the rounded quotient unless it lies within 15 2^-22 of a half; then what the code leaves of
// d is half a step up to 2^-17 of it. A warp with such a channel, a value that is not finite or a
// quotient past 15 (subnormal steps) divides.
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
    const float magic = 12582912.f;
    const f32x2 lo2 = pack2(-lo, -lo), y2 = pack2(y, y), up = pack2(magic, magic), down = pack2(-magic, -magic), s2 = pack2(-s, -s);
    uint32_t w = 0;
    float off_most = 0.f;
#pragma unroll
    for (int i = 3; i >= 0; --i) {
        const float2 x = __half22float2(h2[i]);
        const f32x2 d = add2(pack2(x.x, x.y), lo2), r = fma2(d, y2, up), e = fma2(add2(r, down), s2, d);
        float r0, r1, e0, e1;
        unpack2(r, r0, r1);
        unpack2(e, e0, e1);
        off_most = fmaxf(off_most, fmaxf(fabsf(e0), fabsf(e1)));
        w = (w * 16 + __float_as_uint(r1)) * 16 + __float_as_uint(r0);
    }
    fit.codes = w - 0x3f400000u;                          // 8 nibbles of 0x4b400000, the bits of 1.5 2^23
    const bool plain = range <= 131008.f && range * y < 15.4f && off_most < 0.49999f * s;
    if (__all_sync(LS_FULL_MASK, plain)) return fit;

    float x[8], hi = -65504.f;
    lo = 65504.f;
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

// Nibbles 4 n .. 4 n + 3 of w in the low halves of four bytes.
__device__ __forceinline__ uint32_t spread_nibbles(uint32_t w, int n) {
    uint32_t x = n ? w >> 16 : w & 0xffffu;
    x = (x | (x << 8)) & 0x00ff00ffu;
    return (x | (x << 4)) & 0x0f0f0f0fu;
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

// The K codes and the scales of one token, K in lanes 0-15, V in lanes 16-31.
template <int G>
__device__ __forceinline__ void int4_put_scales(uint8_t* rec, int t, const Int4Fit& fit, int lane) {
    const int hl = lane & 15, grp = hl / (16 / G);
    if (lane < 16) *reinterpret_cast<uint32_t*>(rec + 64 * t + 16 * (hl & 3) + 4 * (hl >> 2)) = fit.codes;
    if (hl % (16 / G) != 0) return;
    __half* at = reinterpret_cast<__half*>(rec + (lane < 16 ? kI4Scales : int4_v_steps(G)));
    at += lane < 16 ? 2 * G * t + grp : int4_v_scale_index(G, t, grp);
    at[0] = fit.step;
    at[lane < 16 ? G : 16 * G] = fit.lo;
}

// One token's K row (lanes 0-15) and V row (lanes 16-31), lane hl of a half holding channels
// 8 hl .. 8 hl + 7, quantised by one warp into the record `rec`: only that token's bytes.
template <int G>
__device__ __forceinline__ void int4_put_token(uint8_t* rec, int t, const uint4& raw, int lane) {
    const int hl = lane & 15;
    const Int4Fit fit = int4_fit<G>(raw);
    // The V byte of channel c is shared with channel c + 8, the neighbouring lane's.
    const uint32_t other = __shfl_xor_sync(LS_FULL_MASK, fit.codes, 1);
    int4_put_scales<G>(rec, t, fit, lane);
    if (lane < 16) return;
    const int odd = hl & 1, tile = hl >> 1;
    const uint32_t bytes = spread_nibbles(odd ? other : fit.codes, odd) | (spread_nibbles(odd ? fit.codes : other, odd) << 4);
    uint8_t* dst = rec + kI4V + (tile >> 2) * 512 + ((t & 7) >> 1) * 16 + (tile & 3) * 4 + 2 * (t & 1) + (t >> 3);
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[(4 * odd + i) * 64] = (uint8_t)(bytes >> (8 * i));
}

// Tokens 2j, 2j + 1, 2j + 8, 2j + 9 of a page, rows as above: the four that share V words.
template <int G>
__device__ __forceinline__ void int4_put_tokens(uint8_t* rec, int j, const uint4 (&raw)[4], int lane) {
    const int hl = lane & 15, odd = hl & 1, tile = hl >> 1;
    uint32_t bytes[4];                                    // of token k: channels of rows 4 odd .. 4 odd + 3 of the tile
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const Int4Fit fit = int4_fit<G>(raw[k]);
        const uint32_t other = __shfl_xor_sync(LS_FULL_MASK, fit.codes, 1);
        int4_put_scales<G>(rec, 2 * j + (k & 1) + 8 * (k >> 1), fit, lane);
        bytes[k] = spread_nibbles(odd ? other : fit.codes, odd) | (spread_nibbles(odd ? fit.codes : other, odd) << 4);
    }
    if (lane < 16) return;
    uint32_t words[4];
    transpose_bytes(bytes[0], bytes[2], bytes[1], bytes[3], words);      // byte 2 e + f: tokens 2j, 2j+8, 2j+1, 2j+9
    uint8_t* dst = rec + kI4V + (tile >> 2) * 512 + (16 * odd + j) * 16 + (tile & 3) * 4;
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

// The inverse of int4_put_tokens: channels 8 hl .. 8 hl + 7 of the four tokens, K in lanes 0-15, V in 16-31.
template <int G>
__device__ __forceinline__ void int4_get_tokens(const uint8_t* rec, int j, int lane, uint4 (&out)[4]) {
    const int hl = lane & 15, odd = hl & 1, tile = hl >> 1, grp = hl / (16 / G);
    uint32_t words[4], bytes[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int t = 2 * j + (i & 1) + 8 * (i >> 1);
        words[i] = *reinterpret_cast<const uint32_t*>(
            lane < 16 ? rec + 64 * t + 16 * (hl & 3) + 4 * (hl >> 2)
                      : rec + kI4V + (tile >> 2) * 512 + (16 * odd + j) * 16 + (tile & 3) * 4 + i * 64);
    }
    transpose_bytes(words[0], words[1], words[2], words[3], bytes);      // V: byte k = token (0, 8, 1, 9)[k]
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t mine = bytes[(k & 1) * 2 + (k >> 1)], other = __shfl_xor_sync(LS_FULL_MASK, mine, 1);
        const int t = 2 * j + (k & 1) + 8 * (k >> 1);
        const __half* sc = reinterpret_cast<const __half*>(rec + (lane < 16 ? kI4Scales : int4_v_steps(G)));
        sc += lane < 16 ? 2 * G * t + grp : int4_v_scale_index(G, t, grp);
        uint32_t b0, b1;
        if (lane < 16) {
            b0 = spread_nibbles(words[k], 0);
            b1 = spread_nibbles(words[k], 1);
        } else {
            b0 = ((odd ? other : mine) >> (4 * odd)) & 0x0f0f0f0fu;
            b1 = ((odd ? mine : other) >> (4 * odd)) & 0x0f0f0f0fu;
        }
        out[k] = int4_values(b0, b1, sc[0], sc[lane < 16 ? G : 16 * G]);
    }
}

}  // namespace ls

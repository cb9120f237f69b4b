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

// One token's K row (lanes 0-15) and V row (lanes 16-31) quantised by one warp and put into
// `rec` (shared or global memory). Lane hl of a half holds channels 8 hl .. 8 hl + 7 in x.
// step = fp16((max - lo) / 15), code = rne((x - lo) / step) clamped to 15; the divisions are
// IEEE ones, so the codes are those of the formula in fp32. NaN counts as 0 and infinities as
// +-65504: what is stored is always finite, and a step is at most 131008 / 15.
template <int G>
__device__ __forceinline__ void int4_put_token(uint8_t* rec, int t, const uint4& raw, int lane) {
    const int hl = lane & 15, side = lane >> 4;
    const __half2* h2 = reinterpret_cast<const __half2*>(&raw);
    float x[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(h2[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
    }
    float lo = 65504.f, hi = -65504.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        x[i] = isnan(x[i]) ? 0.f : fminf(fmaxf(x[i], -65504.f), 65504.f);
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
    }
#pragma unroll
    for (int off = 1; off < 16 / G; off <<= 1) {         // 16 / G lanes hold a group
        lo = fminf(lo, __shfl_xor_sync(LS_FULL_MASK, lo, off));
        hi = fmaxf(hi, __shfl_xor_sync(LS_FULL_MASK, hi, off));
    }
    const __half step = __float2half_rn(__fdiv_rn(__fsub_rn(hi, lo), 15.f));
    const float s = __half2float(step);
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float u = s > 0.f ? rintf(__fdiv_rn(__fsub_rn(x[i], lo), s)) : 0.f;
        w |= (uint32_t)fminf(fmaxf(u, 0.f), 15.f) << (4 * i);
    }
    // The V byte of channel c is shared with channel c + 8, the neighbouring lane's.
    const uint32_t other = __shfl_xor_sync(LS_FULL_MASK, w, 1);
    const int grp = hl / (16 / G);
    const bool first = hl % (16 / G) == 0;
    if (side == 0) {
        *reinterpret_cast<uint32_t*>(rec + 64 * t + 16 * (hl & 3) + 4 * (hl >> 2)) = w;
        if (first) {
            __half* sc = reinterpret_cast<__half*>(rec + kI4Scales) + 2 * G * t + grp;
            sc[0] = step;
            sc[G] = __float2half_rn(lo);
        }
    } else {
        const uint32_t low = (hl & 1) ? other : w, high = (hl & 1) ? w : other;
        const int tile = hl >> 1, g0 = (hl & 1) * 4;
        uint8_t* dst = rec + kI4V + (tile >> 2) * 512 + ((t & 7) >> 1) * 16 + (tile & 3) * 4 + 2 * (t & 1) + (t >> 3);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int g = g0 + i;
            dst[g * 64] = (uint8_t)(((low >> (4 * g)) & 15u) | (((high >> (4 * g)) & 15u) << 4));
        }
        if (first) {
            const int at = int4_v_scale_index(G, t, grp);
            reinterpret_cast<__half*>(rec + int4_v_steps(G))[at] = step;
            reinterpret_cast<__half*>(rec + int4_v_lows(G))[at] = __float2half_rn(lo);
        }
    }
}

// Channels 8 hl .. 8 hl + 7 of token t's K row (side 0) or V row (side 1) as fp16 values.
template <int G>
__device__ __forceinline__ uint4 int4_get(const uint8_t* rec, int t, int side, int hl) {
    uint32_t w = 0;
    float step, lo;
    const int grp = hl / (16 / G);
    if (side == 0) {
        w = *reinterpret_cast<const uint32_t*>(rec + 64 * t + 16 * (hl & 3) + 4 * (hl >> 2));
        const __half* sc = reinterpret_cast<const __half*>(rec + kI4Scales) + 2 * G * t + grp;
        step = __half2float(sc[0]);
        lo = __half2float(sc[G]);
    } else {
        const int tile = hl >> 1, up = (hl & 1) * 4;
        const uint8_t* src = rec + kI4V + (tile >> 2) * 512 + ((t & 7) >> 1) * 16 + (tile & 3) * 4 + 2 * (t & 1) + (t >> 3);
#pragma unroll
        for (int g = 0; g < 8; ++g) w |= (uint32_t)((src[g * 64] >> up) & 15) << (4 * g);
        const int at = int4_v_scale_index(G, t, grp);
        step = __half2float(reinterpret_cast<const __half*>(rec + int4_v_steps(G))[at]);
        lo = __half2float(reinterpret_cast<const __half*>(rec + int4_v_lows(G))[at]);
    }
    uint4 out;
    uint32_t* o = reinterpret_cast<uint32_t*>(&out);
#pragma unroll
    for (int i = 0; i < 4; ++i)
        o[i] = pack_half2(fmaf(step, (float)((w >> (8 * i)) & 15u), lo), fmaf(step, (float)((w >> (8 * i + 4)) & 15u), lo));
    return out;
}

}  // namespace ls

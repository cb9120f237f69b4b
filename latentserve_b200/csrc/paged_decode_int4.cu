// Paged GQA decode attention over a cache held in 4 bits (record layout: int4_page.cuh).
//
// Measured on one B200 (copy peak 6.54 TB/s), launches back to back: 64 x 16 384 tokens, 2 KV
// heads, 6 query rows, groups of 32: 71 us (4.7 TB/s; a page more per SM costs 64 ns = 5.9 TB/s);
// 64 x 16 384, 8 KV heads, 4 rows, groups of 64: 210 us (5.75 TB/s). What is left over the bytes is
// a fixed 10 us (launch 2, lengths and tables 2, first pages 1, the last states' way out 4) and, in
// the loop, instruction issue about as much as memory: 269 instructions and 27 MMAs a page at six
// rows (a word of eight codes is one shift and four ANDs), issue slots 48 % used, the tensor pipe 38 %.
//
// Mathematics, per page of 16 tokens and one KV head, n = codes, step / lo = fp16 scales per
// (token t, group y of channels):
//   score[t, r]  = sum_y step[t, y] (sum_{c in y} q[r, c] n[t, c]) + sum_y lo[t, y] qsum[r, y]
//   out[c, r]   += sum_t (w[t, r] step[t, y]) n[t, c] + sum_t w[t, r] lo[t, y]
// Codes go to the tensor cores as they are: a nibble masked out of its word IS an fp16 number
// (n 2^-24, or n 2^-20 four bits higher up: subnormals, which the MMA takes exactly), so a word
// of eight codes costs one shift and four ANDs and nothing is ever dequantised. K: the query
// channels that meet the low nibbles carry a factor 16, so both kinds add up in one accumulator;
// V: low and high nibbles are different output channels, told apart at the end. The lows enter
// through one MMA each (A = the page's lows, B = the query's group sums, or the weights).
//
// Precision: q is scaled by a power of two per row; q, codes, lows are exact in fp16, group sums are
// split into two fp16 numbers; steps multiply in fp32. The weights w and their products with the V
// steps are split into high and low fp16 halves: one fp16 rounding of the product alone (2^-11 of a
// weight at most, 2e-4 on average, as much as rounding the output) would put outputs of random
// values 1.4 times as far from the exact ones as they are now.
// The reference of the online softmax lags by at most 2 (log2), so w <= 4 and w * step <= 4 * 8734,
// inside fp16 for every step the writer can store.
#include "decode_core.cuh"
#include "int4_page.cuh"

namespace ls {

// A warp takes kInt4Group pages of a sequence at a time: one wait, one decision on the softmax
// reference and one loop's bookkeeping for all of them, and the pages' chains of dependent
// instructions overlap. Two groups of each warp are in flight or being worked on. (16 x 16 384 tokens:
// a page at a time in the INT8 kernel's loop 33.0 us, groups of four 30.9; groups of two or three with
// three blocks an SM the same within 1 us, a third stage costs the second block and 15 us.)
#ifndef LS_INT4_GROUP
#define LS_INT4_GROUP 4
#endif
#ifndef LS_INT4_STAGES
#define LS_INT4_STAGES 2
#endif
#ifndef LS_INT4_CTAS
#define LS_INT4_CTAS 2
#endif
constexpr int kInt4Group = LS_INT4_GROUP, kInt4Stages = LS_INT4_STAGES;
constexpr float kInt4Margin = 2.f;         // log2 units the softmax reference may lag

__device__ __forceinline__ uint2 lds64(uint32_t addr) {
    uint2 r;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];\n" : "=r"(r.x), "=r"(r.y) : "r"(addr));
    return r;
}
__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
    uint32_t r;
    asm volatile("ld.shared.u32 %0, [%1];\n" : "=r"(r) : "r"(addr));
    return r;
}
__device__ __forceinline__ uint32_t hfma2_u32(uint32_t a, uint32_t b, uint32_t c) {
    const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b),
                              *reinterpret_cast<const __half2*>(&c));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hneg2_u32(uint32_t a) {
    const __half2 r = __hneg2(*reinterpret_cast<const __half2*>(&a));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ float half_lo(uint32_t x) { return __low2float(*reinterpret_cast<const __half2*>(&x)); }
__device__ __forceinline__ float half_hi(uint32_t x) { return __high2float(*reinterpret_cast<const __half2*>(&x)); }

// D = A(16x8, fp16, row) * B(8x8, fp16, col).
__device__ __forceinline__ void mma_1688_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0, const float (&z)[4]) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%8,%9,%10};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(b0), "f"(z[0]), "f"(z[1]), "f"(z[2]), "f"(z[3]));
}
// D = A(16x16) * B(16x8): an accumulator that starts here is not cleared first.
__device__ __forceinline__ void mma_16816_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                              uint32_t b0, uint32_t b1, const float (&z)[4]) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(z[0]), "f"(z[1]), "f"(z[2]), "f"(z[3]));
}

// The state of one warp. Lane (g = lane / 4, j = lane % 4).
//
// TWICE (at most four query rows): an MMA has eight columns of rows, so columns 4-7 hold rows 0-3
// again. The scores come out twice, and where the weights go into the MMAs, columns 0-3 carry
// their high halves and 4-7 the low ones: one MMA per tile does what takes two otherwise (18
// MMAs a page instead of 27), and the two sums meet at the end.
template <int G, bool TWICE>
struct Int4State {
    static constexpr uint32_t kLow = 0x000f000fu, kHigh = 0x00f000f0u;
    static constexpr int kRecord = int4_record_bytes(G);
    uint32_t qb[4][4];         // B fragments of channels 32 w + 8 j ..: low-nibble channels (x16), high-nibble ones
    uint32_t qs;               // B fragment of the query's group sums (high and low fp16 parts)
    float o[9][4];             // O^T tile i < 8: channel 16 i + g of rows 2j, 2j+1 (in 2^-24), channel 16 i + 8 + g
                               // (in 2^-20); tile 8: lanes g < G the sum of w * lo of group g, lanes g = G the sum of w
    float m[2];                // reference of rows 2j, 2j+1 (log2)
    float zero[4];             // what a new accumulator starts from, in registers of its own
    float f[2];                // softmax scale (log2) over the query's power of two, rows 2j, 2j+1

    // This lane's share of the query: row g, channels 32 w + 8 j .. of word w.
    static __device__ __forceinline__ void load_query(const DecodeParams& p, int b, int h, int lane, uint4 (&raw)[4]) {
        const int row = TWICE ? (lane >> 2) & 3 : lane >> 2, j = lane & 3;
        const __half* src = p.q + b * p.sq_b + h * p.sq_h + row * p.sq_m + 8 * j;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            raw[w] = make_uint4(0, 0, 0, 0);
            if (row < p.n_rep) raw[w] = *reinterpret_cast<const uint4*>(src + 32 * w);
        }
    }

    __device__ __forceinline__ void begin(const DecodeParams& p, const uint4 (&raw)[4], int lane) {
        m[0] = m[1] = neg_inf();
#pragma unroll
        for (int i = 0; i < 4; ++i) asm volatile("mov.f32 %0, 0f00000000;\n" : "=f"(zero[i]));
#pragma unroll
        for (int i = 0; i < 9; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) o[i][k] = 0.f;
        const int j = lane & 3;
        float top = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const uint32_t* x = reinterpret_cast<const uint32_t*>(&raw[w]);
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(fabsf(half_lo(x[i])), fabsf(half_hi(x[i]))));
        }
        top = fmaxf(top, __shfl_xor_sync(LS_FULL_MASK, top, 1));
        top = fmaxf(top, __shfl_xor_sync(LS_FULL_MASK, top, 2));
        // The row is multiplied by the power of two that brings its largest value into [8, 16), and by
        // the sign of the softmax scale, so that larger scores are larger weights.
        const int e = top > 0.f ? 130 - (__float_as_int(top) >> 23) : 0;
        const float up = copysignf(__int_as_float((127 + e) << 23), p.scale_log2);
        // (Never zero: a masked score is -inf times this.)
        const float back = fmaxf(fabsf(p.scale_log2) * __int_as_float((127 - e) << 23), 1e-37f);
        f[0] = __shfl_sync(LS_FULL_MASK, back, 8 * j);
        f[1] = __shfl_sync(LS_FULL_MASK, back, 8 * j + 4);
        float sum[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const uint32_t* x = reinterpret_cast<const uint32_t*>(&raw[w]);
            float c[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                c[2 * i] = half_lo(x[i]) * up;
                c[2 * i + 1] = half_hi(x[i]) * up;
            }
            qb[w][0] = pack_half2(16.f * c[0], 16.f * c[4]);
            qb[w][1] = pack_half2(16.f * c[2], 16.f * c[6]);
            qb[w][2] = pack_half2(c[1], c[5]);
            qb[w][3] = pack_half2(c[3], c[7]);
            sum[w] = ((c[0] + c[1]) + (c[2] + c[3])) + ((c[4] + c[5]) + (c[6] + c[7]));
            sum[w] += __shfl_xor_sync(LS_FULL_MASK, sum[w], 1);
            sum[w] += __shfl_xor_sync(LS_FULL_MASK, sum[w], 2);
        }
        // Columns 2j, 2j+1 of the lows' A fragment: lanes j < 2 meet the sums' high parts, j >= 2
        // their low parts; see scores() for which lows a lane's register holds.
        float s0, s1;
        if (G == 4) {
            s0 = (j & 1) ? sum[2] : sum[0];
            s1 = (j & 1) ? sum[3] : sum[1];
        } else if (G == 2) {
            s0 = (j & 1) ? 0.f : sum[0] + sum[1];
            s1 = (j & 1) ? 0.f : sum[2] + sum[3];
        } else {
            s0 = 0.f;
            s1 = (j & 1) ? 0.f : (sum[0] + sum[1]) + (sum[2] + sum[3]);
        }
        const uint32_t top2 = pack_half2(s0, s1);
        qs = j < 2 ? top2 : pack_half2(s0 - half_lo(top2), s1 - half_hi(top2));
    }

    // One page's scores, before the factor f: s[0], s[1] = token g, rows 2j, 2j+1; s[2], s[3] = token g + 8.
    __device__ __forceinline__ void scores(uint32_t page, int lane, float (&s)[4]) const {
        const int g = lane >> 2, j = lane & 3;
        const uint4 w0 = lds128(page + 64 * g + 16 * j), w1 = lds128(page + 64 * (g + 8) + 16 * j);
        const uint32_t* k0 = reinterpret_cast<const uint32_t*>(&w0);
        const uint32_t* k1 = reinterpret_cast<const uint32_t*>(&w1);
        uint32_t low0, low1;                    // this lane's column pair of the lows, tokens g and g + 8
        float st0[G], st1[G];                   // steps of tokens g and g + 8
        if (G == 4) {
            const uint4 c0 = lds128(page + kI4Scales + 16 * g), c1 = lds128(page + kI4Scales + 16 * (g + 8));
            low0 = (j & 1) ? c0.w : c0.z;
            low1 = (j & 1) ? c1.w : c1.z;
            st0[0] = half_lo(c0.x); st0[1 % G] = half_hi(c0.x); st0[2 % G] = half_lo(c0.y); st0[3 % G] = half_hi(c0.y);
            st1[0] = half_lo(c1.x); st1[1 % G] = half_hi(c1.x); st1[2 % G] = half_lo(c1.y); st1[3 % G] = half_hi(c1.y);
        } else if (G == 2) {
            const uint2 c0 = lds64(page + kI4Scales + 8 * g), c1 = lds64(page + kI4Scales + 8 * (g + 8));
            low0 = c0.y;
            low1 = c1.y;
            st0[0] = half_lo(c0.x); st0[1 % G] = half_hi(c0.x);
            st1[0] = half_lo(c1.x); st1[1 % G] = half_hi(c1.x);
        } else {
            low0 = lds32(page + kI4Scales + 4 * g);              // (step, lo): the step meets a zero
            low1 = lds32(page + kI4Scales + 4 * (g + 8));
            st0[0] = half_lo(low0);
            st1[0] = half_lo(low1);
        }
        float base[4], acc[G][4];
        mma_1688_new(base, low0, low1, qs, zero);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const int y = w * G / 4;
            const uint32_t x0 = k0[w], x1 = k1[w], z0 = x0 >> 8, z1 = x1 >> 8;
            if (w * G % 4 == 0) mma_16816_new(acc[y], x0 & kLow, x1 & kLow, z0 & kLow, z1 & kLow, qb[w][0], qb[w][1], zero);
            else mma_16816(acc[y], x0 & kLow, x1 & kLow, z0 & kLow, z1 & kLow, qb[w][0], qb[w][1]);
            mma_16816(acc[y], x0 & kHigh, x1 & kHigh, z0 & kHigh, z1 & kHigh, qb[w][2], qb[w][3]);
        }
        s[0] = st0[0] * acc[0][0];
        s[1] = st0[0] * acc[0][1];
        s[2] = st1[0] * acc[0][2];
        s[3] = st1[0] * acc[0][3];
#pragma unroll
        for (int y = 1; y < G; ++y) {
            s[0] = fmaf(st0[y], acc[y][0], s[0]);
            s[1] = fmaf(st0[y], acc[y][1], s[1]);
            s[2] = fmaf(st1[y], acc[y][2], s[2]);
            s[3] = fmaf(st1[y], acc[y][3], s[3]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) s[i] = fmaf(s[i], 1048576.f, base[i]);       // codes are in 2^-20
    }

    // One page's share of the output, s = its weights.
    template <bool FULL>
    __device__ __forceinline__ void values(uint32_t page, int valid, int lane, const float (&s)[4]) {
        const int g = lane >> 2, j = lane & 3;
        // Weights as B fragments (rows g, tokens 2j, 2j+1 | 2j+8, 2j+9), high and low halves.
        const uint32_t p0 = pack_half2(s[0], s[1]), p1 = pack_half2(s[2], s[3]);
        const uint32_t w0h = movmatrix_trans(p0), w1h = movmatrix_trans(p1);
        const uint32_t w0l = movmatrix_trans(pack_half2(s[0] - half_lo(p0), s[1] - half_hi(p0)));
        const uint32_t w1l = movmatrix_trans(pack_half2(s[2] - half_lo(p1), s[3] - half_hi(p1)));
        // Scales of tokens past the end may hold anything, NaN included: they are cleared.
        uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
        if (!FULL) {
            keep0 = (2 * j < valid ? 0xffffu : 0u) | (2 * j + 1 < valid ? 0xffff0000u : 0u);
            keep1 = (2 * j + 8 < valid ? 0xffffu : 0u) | (2 * j + 9 < valid ? 0xffff0000u : 0u);
        }
        {
            // Rows g < G of this tile's A: the lows of group g; row G: ones, which sum the weights.
            uint2 lows = lds64(page + int4_v_lows(G) + 8 * G * j + 8 * (g < G ? g : 0));
            const uint32_t mine = g < G ? 0xffffffffu : 0u, one = g == G ? 0x3c003c00u : 0u;
            lows.x = (lows.x & mine & keep0) | one;
            lows.y = (lows.y & mine & keep1) | one;
            if (TWICE) {
                mma_16816(o[8], lows.x, 0u, lows.y, 0u, g < 4 ? w0h : w0l, g < 4 ? w1h : w1l);
            } else {
                mma_16816(o[8], lows.x, 0u, lows.y, 0u, w0h, w1h);
                mma_16816(o[8], lows.x, 0u, lows.y, 0u, w0l, w1l);
            }
        }
        uint32_t st[2 * G];                          // V steps [group][half]
        if (G == 1) {
            const uint2 c = lds64(page + int4_v_steps(G) + 8 * j);
            st[0] = c.x; st[1] = c.y;
        } else {
#pragma unroll
            for (int y = 0; y < G; y += 2) {
                const uint4 c = lds128(page + int4_v_steps(G) + 8 * G * j + 8 * y);
                st[2 * y] = c.x; st[2 * y + 1] = c.y; st[(2 * y + 2) % (2 * G)] = c.z; st[(2 * y + 3) % (2 * G)] = c.w;
            }
        }
        // w * step in two halves: the rounded product, and what it and the weight's low half left.
        uint32_t b[2 * G], e[2 * G];
#pragma unroll
        for (int y = 0; y < G; ++y) {
            const uint32_t t0 = FULL ? st[2 * y] : st[2 * y] & keep0, t1 = FULL ? st[2 * y + 1] : st[2 * y + 1] & keep1;
            b[2 * y] = hmul2_u32(w0h, t0);
            b[2 * y + 1] = hmul2_u32(w1h, t1);
            e[2 * y] = hfma2_u32(w0l, t0, hfma2_u32(w0h, t0, hneg2_u32(b[2 * y])));
            e[2 * y + 1] = hfma2_u32(w1l, t1, hfma2_u32(w1h, t1, hneg2_u32(b[2 * y + 1])));
            if (TWICE && g >= 4) {
                b[2 * y] = e[2 * y];
                b[2 * y + 1] = e[2 * y + 1];
            }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const uint4 v4 = lds128(page + kI4V + 512 * c + 16 * lane);
            const uint32_t* v = reinterpret_cast<const uint32_t*>(&v4);
            // Two tiles at a time, so that an accumulator's two MMAs are not next to each other.
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const int tile = 4 * c + i, y0 = tile * G / 8, y1 = (tile + 1) * G / 8;
                const uint32_t x0 = v[i], z0 = x0 >> 8, x1 = v[i + 1], z1 = x1 >> 8;
                const uint32_t a0 = x0 & kLow, a1 = x0 & kHigh, a2 = z0 & kLow, a3 = z0 & kHigh;
                const uint32_t c0 = x1 & kLow, c1 = x1 & kHigh, c2 = z1 & kLow, c3 = z1 & kHigh;
                mma_16816(o[tile], a0, a1, a2, a3, b[2 * y0], b[2 * y0 + 1]);
                mma_16816(o[tile + 1], c0, c1, c2, c3, b[2 * y1], b[2 * y1 + 1]);
                if (!TWICE) {
                    mma_16816(o[tile], a0, a1, a2, a3, e[2 * y0], e[2 * y0 + 1]);
                    mma_16816(o[tile + 1], c0, c1, c2, c3, e[2 * y1], e[2 * y1 + 1]);
                }
            }
        }
    }

    // N pages. FULL: all their tokens exist. Otherwise N = 1 and the first `valid` do.
    template <int N, bool FULL>
    __device__ __forceinline__ void pages(uint32_t stage, int valid, int lane) {
        const int g = lane >> 2;
        float s[N][4];
#pragma unroll
        for (int i = 0; i < N; ++i) scores(stage + i * kRecord, lane, s[i]);
        if (!FULL) {
            if (g >= valid) s[0][0] = s[0][1] = neg_inf();
            if (g + 8 >= valid) s[0][2] = s[0][3] = neg_inf();
        }
        float top0 = neg_inf(), top1 = neg_inf();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            top0 = fmaxf(top0, fmaxf(s[i][0], s[i][2]));
            top1 = fmaxf(top1, fmaxf(s[i][1], s[i][3]));
        }
        top0 *= f[0];
        top1 *= f[1];
        // Usually no score rises more than the margin above the reference, which then stays as it
        // is: one vote instead of the shuffles and the rescaling.
        const bool ok = top0 <= m[0] + kInt4Margin && top1 <= m[1] + kInt4Margin && m[0] != neg_inf() && m[1] != neg_inf();
        if (!__all_sync(LS_FULL_MASK, ok)) {
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) {
                top0 = fmaxf(top0, __shfl_xor_sync(LS_FULL_MASK, top0, off));
                top1 = fmaxf(top1, __shfl_xor_sync(LS_FULL_MASK, top1, off));
            }
            const float n0 = fmaxf(m[0], top0), n1 = fmaxf(m[1], top1);
            const float a0 = ex2(m[0] - (n0 == neg_inf() ? 0.f : n0)), a1 = ex2(m[1] - (n1 == neg_inf() ? 0.f : n1));
            m[0] = n0;
            m[1] = n1;
#pragma unroll
            for (int i = 0; i < 9; ++i) {
                o[i][0] *= a0;
                o[i][1] *= a1;
                o[i][2] *= a0;
                o[i][3] *= a1;
            }
        }
        // A row that has seen no token yet keeps -inf; zero stands in for it.
        const float m0 = m[0] == neg_inf() ? 0.f : m[0], m1 = m[1] == neg_inf() ? 0.f : m[1];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            s[i][0] = ex2(fmaf(s[i][0], f[0], -m0));
            s[i][1] = ex2(fmaf(s[i][1], f[1], -m1));
            s[i][2] = ex2(fmaf(s[i][2], f[0], -m0));
            s[i][3] = ex2(fmaf(s[i][3], f[1], -m1));
            values<FULL>(stage + i * kRecord, valid, lane, s[i]);
        }
    }

    __device__ __forceinline__ void finish(float* mo, float* mm, float* ml, int n_rep, int lane) {
        const int g = lane >> 2, j = lane & 3;
        const int r0 = 2 * j, r1 = r0 + 1;
        if (TWICE) {
#pragma unroll
            for (int i = 0; i < 9; ++i)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[i][k] += __shfl_xor_sync(LS_FULL_MASK, o[i][k], 2);
        }
#pragma unroll
        for (int y = 0; y < G; ++y) {
            const float low0 = __shfl_sync(LS_FULL_MASK, o[8][0], 4 * y + j);
            const float low1 = __shfl_sync(LS_FULL_MASK, o[8][1], 4 * y + j);
#pragma unroll
            for (int tile = y * (8 / G); tile < (y + 1) * (8 / G); ++tile) {
                const int c = 16 * tile + g;
                if (r0 < n_rep) {
                    mo[r0 * kMergeStride + c] = fmaf(o[tile][0], 16777216.f, low0);
                    mo[r0 * kMergeStride + c + 8] = fmaf(o[tile][2], 1048576.f, low0);
                }
                if (r1 < n_rep) {
                    mo[r1 * kMergeStride + c] = fmaf(o[tile][1], 16777216.f, low1);
                    mo[r1 * kMergeStride + c + 8] = fmaf(o[tile][3], 1048576.f, low1);
                }
            }
        }
        if (g == G) {
            if (r0 < n_rep) { mm[r0] = m[0]; ml[r0] = o[8][0]; }
            if (r1 < n_rep) { mm[r1] = m[1]; ml[r1] = o[8][1]; }
        }
    }
};

// How the batch is cut. Every sequence takes its pages plus kInt4Begin units on one axis, and the
// axis is cut into even chunks, one per CTA: a CTA that goes from one sequence to the next gets
// that many pages fewer, for the time that summing up the one and starting the other takes (16 x
// 16 384 tokens: 30.6 us with none, 29.1 with 12, 26.5 with 24, 26.6 with 40). A
// sequence's pages begin behind its extra units, so a chunk that ends inside those has none of it.
#ifndef LS_INT4_BEGIN
#define LS_INT4_BEGIN 24
#endif
constexpr int kInt4Begin = LS_INT4_BEGIN;

template <int THREADS>
__device__ __forceinline__ int int4_prefix(const DecodeParams& p, int* cum, int* scratch) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ipt = (p.batch + THREADS - 1) / THREADS, base = tid * ipt;
    auto units = [&](int b) {
        const int n = seq_units<LS_MODE_DENSE>(p, b);
        return n > 0 ? n + kInt4Begin : 0;
    };
    int own = 0, s = 0;
    for (int i = 0; i < ipt; ++i)
        if (base + i < p.batch) s += own = units(base + i);
    int inc = s;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
        const int o = __shfl_up_sync(LS_FULL_MASK, inc, off);
        if (lane >= off) inc += o;
    }
    if (lane == 31) scratch[warp] = inc;
    __syncthreads();
    int run = inc - s;
    for (int w = 0; w < warp; ++w) run += scratch[w];
    for (int i = 0; i < ipt; ++i)
        if (base + i < p.batch) {
            cum[base + i] = run;
            run += ipt == 1 ? own : units(base + i);
        }
    if (tid == THREADS - 1) cum[p.batch] = run;
    __syncthreads();
    return cum[p.batch];
}

// Units of one chunk: even shares, but not fewer than `min_chunk` pages of a long sequence: below
// that the partial states cost more to merge than the pages to read. Sequences shorter than that
// are not lumped together to make up for it.
__device__ __forceinline__ int int4_chunk_size(const DecodeParams& p, int total) {
    const int even = (total + p.num_chunks - 1) / p.num_chunks, mean = (total + p.batch - 1) / p.batch;
    return max(max(even, min(p.min_chunk, mean)), 1);
}

// Pages [lo, hi) of sequence b that lie in the chunk [g0, g1) of the axis (none: hi <= lo).
__device__ __forceinline__ void int4_piece(const int* cum, int b, int g0, int g1, int& lo, int& hi) {
    lo = max(g0 - cum[b] - kInt4Begin, 0);
    hi = min(g1, cum[b + 1]) - cum[b] - kInt4Begin;
}

// The next sequence after b with pages in a chunk that ends at g1; `batch` if there is none.
__device__ __forceinline__ int int4_next(const int* cum, int batch, int b, int g1) {
    do ++b; while (b < batch && cum[b + 1] == cum[b]);
    return b < batch && cum[b] + kInt4Begin < g1 ? b : batch;
}

// Warp w's share of a segment's pages [lo, hi): an even, contiguous part.
__device__ __forceinline__ int warp_share(int lo, int hi, int w) { return lo + (hi - lo) * w / kWarps; }

// The load side of one warp: its share of every segment of the chunk, in order, kInt4Group pages
// at a time. Lane l of a window holds the block id of the window's page l, so the lanes of a group
// issue its copies side by side; the next window's ids are requested while this one is handed out.
template <int G>
struct GroupLoader {
    static constexpr int PG = kInt4Group, kWindow = 32 / PG * PG;
    static constexpr int kRecord = int4_record_bytes(G);
    struct Window {
        int u, n, len, id;          // first page, pages, tokens of the sequence, this lane's block
    };
    int b, u, hi, g1;               // where the window after the next one starts
    bool done;
    Window cur, nxt;
    int i;                          // pages of `cur` handed out
    uint32_t there;                 // lanes of `cur` whose block lies inside the pool

    __device__ __forceinline__ void normalize(const int* cum, int batch, int warp) {
        while (!done && u >= hi) {                       // bounded: every pass moves to a later sequence
            b = int4_next(cum, batch, b, g1);
            done = b == batch;
            if (!done) {
                int lo, end;
                int4_piece(cum, b, 0, g1, lo, end);
                u = warp_share(0, end, warp);
                hi = warp_share(0, end, warp + 1);
            }
        }
    }

    __device__ __forceinline__ Window fetch(const DecodeParams& p, const int* cum, int warp, int lane) {
        Window w = {0, 0, 0, -1};
        if (done) return w;
        w.n = min(kWindow, hi - u);
        w.u = u;
        w.len = p.seq_lens[b];
        if (lane < w.n) w.id = p.block_tables[(long long)b * p.max_pages + u + lane];
        u += w.n;
        normalize(cum, p.batch, warp);
        return w;
    }

    __device__ __forceinline__ void promote(const DecodeParams& p, const int* cum, int warp, int lane) {
        cur = nxt;
        i = 0;
        const bool in = lane < cur.n, ok = in && cur.id >= 0 && cur.id < p.num_blocks;
        if (in && !ok) p.seg_range[2 * p.batch] = 1;     // corrupt table: read nothing, flag it
        there = __ballot_sync(LS_FULL_MASK, ok);
        nxt = fetch(p, cum, warp, lane);
    }

    __device__ __forceinline__ void begin(const DecodeParams& p, const int* cum, int b0, int lo, int top, int end, int warp,
                                          int lane) {
        b = b0;
        g1 = end;
        u = warp_share(lo, top, warp);
        hi = warp_share(lo, top, warp + 1);
        done = false;
        normalize(cum, p.batch, warp);
        nxt = fetch(p, cum, warp, lane);
        promote(p, cum, warp, lane);
    }

    // Request the next group into `stage`; what the compute side has to know goes to `meta`: its
    // tokens, and from bit 16 which of its pages are not there. `wait` is called before a
    // sequence's last page is requested.
    template <class Wait>
    __device__ __forceinline__ void issue(const DecodeParams& p, const int* cum, int h, int warp, int lane, uint32_t stage,
                                          uint32_t mbar, uint32_t meta, uint64_t policy, Wait wait) {
        if (i >= cur.n) {
            if (cur.n == 0) return;
            promote(p, cum, warp, lane);
            if (cur.n == 0) return;
        }
        const int first = cur.u + i, n = min(PG, cur.n - i);
        const uint32_t present = (1u << n) - 1, here = (there >> i) & present;
        const int tokens = min(n * LS_PAGE, cur.len - first * LS_PAGE);
        if ((first + n) * LS_PAGE >= cur.len) wait();
        if (lane == 0) {
            asm volatile("st.shared.u32 [%0], %1;\n" ::"r"(meta), "r"(tokens | ((present & ~here) << 16)) : "memory");
            mbar_expect_tx(mbar, __popc(here) * kRecord);
        }
        __syncwarp();
        if (lane >= i && lane < i + n && ((there >> lane) & 1))
            bulk_load_hint(stage + (lane - i) * kRecord,
                           static_cast<const uint8_t*>(p.k_pool) + cur.id * p.sk_b + h * p.sk_h, kRecord, mbar, policy);
        i += PG;
    }
};

// A partial state: [8] maxima, [8] sums, then n_rep rows of 128 sums, all fp32. The states of one
// KV head lie behind one another, so those of a sequence are one run of memory.
constexpr int kStateHead = 2 * kRP;
__device__ __forceinline__ int state_floats(const DecodeParams& p) { return kStateHead + p.n_rep * LS_HEAD_DIM; }
__device__ __forceinline__ float* state_of(const DecodeParams& p, int slot, int h) {
    return p.part_acc + ((long long)h * (p.batch + p.num_chunks) + slot) * state_floats(p);
}

// Merge of a sequence's `count` partial states (slots first ..) by the whole CTA, into `out`:
//   out = sum_s acc_s 2^(m_s - M) / sum_s l_s 2^(m_s - M).
// The states come in by one bulk copy of as many as fit `room` (per-thread loads took a round trip
// for the maxima, one for the sums and one for each few rows; a copy each for 64 states, 5 us). Every warp
// works out all weights by itself, lane 4 r + k row r of states k, k + 4, ..; warp w then sums states
// w, w + 4, .., a lane four channels of all rows, and the warps' sums meet in `rows` (kWarps x n_rep
// x kMergeStride floats). States that do not fit at once are weighed against the maximum so far.
__device__ __forceinline__ void int4_merge(const DecodeParams& p, int first, int count, int b, int h, unsigned char* room,
                                           int room_bytes, float* rows, uint32_t mbar, uint32_t& phase, int tid) {
    const int warp = tid >> 5, lane = tid & 31, r4 = lane >> 2, k4 = lane & 3, n_rep = p.n_rep;
    const int stride = state_floats(p);
    // [warp][state][8] weights behind the states.
    const int fit = room_bytes / (stride * 4 + kWarps * kRP * 4);
    const float* states = reinterpret_cast<const float*>(room);
    float* wgt = reinterpret_cast<float*>(room) + fit * stride + warp * fit * kRP;
    float4 a[kRP];
#pragma unroll
    for (int r = 0; r < kRP; ++r) a[r] = make_float4(0.f, 0.f, 0.f, 0.f);
    float top = neg_inf(), sum = 0.f;                         // of row r4
    for (int s0 = 0; s0 < count; s0 += fit) {
        const int n = min(fit, count - s0);
        if (tid == 0) {
            // What other CTAs stored, and this one's reads of the room, come before the copy.
            asm volatile("fence.proxy.async;\n" ::: "memory");
            mbar_expect_tx(mbar, n * stride * 4);
            bulk_load(smem_u32(room), state_of(p, first + s0, h), n * stride * 4, mbar);
        }
        if (!mbar_wait_bounded(mbar, phase, kMbarSpinLimit) && tid == 0) p.seg_range[2 * p.batch] = 2;
        phase ^= 1u;
        float t = top;
        for (int s = k4; s < n; s += 4) t = fmaxf(t, states[s * stride + r4]);
        t = fmaxf(t, __shfl_xor_sync(LS_FULL_MASK, t, 1));
        t = fmaxf(t, __shfl_xor_sync(LS_FULL_MASK, t, 2));
        const float ref = t == neg_inf() ? 0.f : t, shrink = ex2(top - ref);
        sum *= shrink;
        top = t;
        for (int s = k4; s < n; s += 4) {
            const float w = ex2(states[s * stride + r4] - ref);
            wgt[s * kRP + r4] = w;
            sum = fmaf(w, states[s * stride + kRP + r4], sum);
        }
        __syncwarp();
        if (s0 > 0) {
#pragma unroll
            for (int r = 0; r < kRP; ++r) {
                const float by = __shfl_sync(LS_FULL_MASK, shrink, 4 * r);
                a[r].x *= by; a[r].y *= by; a[r].z *= by; a[r].w *= by;
            }
        }
        // (Rows past n_rep repeat the last one into sums that nobody reads: no branches.)
#pragma unroll 2
        for (int s = warp; s < n; s += kWarps) {
            const float4 w0 = *reinterpret_cast<const float4*>(wgt + s * kRP), w1 = *reinterpret_cast<const float4*>(wgt + s * kRP + 4);
            const float w[kRP] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
            const float* x = states + s * stride + kStateHead + 4 * lane;
#pragma unroll
            for (int r = 0; r < kRP; ++r) {
                const float4 v = *reinterpret_cast<const float4*>(x + min(r, n_rep - 1) * LS_HEAD_DIM);
                a[r].x = fmaf(w[r], v.x, a[r].x);
                a[r].y = fmaf(w[r], v.y, a[r].y);
                a[r].z = fmaf(w[r], v.z, a[r].z);
                a[r].w = fmaf(w[r], v.w, a[r].w);
            }
        }
        if (s0 + fit < count) __syncthreads();                // the room is free again
    }
    sum += __shfl_xor_sync(LS_FULL_MASK, sum, 1);
    sum += __shfl_xor_sync(LS_FULL_MASK, sum, 2);
    const float inv = 1.f / fmaxf(sum, 1e-20f);
#pragma unroll
    for (int r = 0; r < kRP; ++r)
        if (r < n_rep) *reinterpret_cast<float4*>(rows + (warp * n_rep + r) * kMergeStride + 4 * lane) = a[r];
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRP; ++r) {
        const float scale = __shfl_sync(LS_FULL_MASK, inv, 4 * r);
        const float* x = rows + min(r, n_rep - 1) * kMergeStride + tid;
        const int step = n_rep * kMergeStride;
        const float all = (x[0] + x[step]) + (x[2 * step] + x[3 * step]);
        if (r < n_rep) p.out[b * p.so_b + h * p.so_h + r * p.so_m + tid] = __float2half_rn(all * scale);
    }
    __syncthreads();                                          // room and rows are free again
}

template <int G, bool TWICE>
__global__ void __launch_bounds__(kThreads, LS_INT4_CTAS)
int4_decode_kernel(const __grid_constant__ DecodeParams p) {
    extern __shared__ __align__(1024) unsigned char smem[];
    constexpr int PG = kInt4Group, STAGES = kInt4Stages, STAGE_BYTES = PG * int4_record_bytes(G);
    static_assert(kThreads == LS_HEAD_DIM, "a thread per channel where warps' states are summed");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int chunk_id = blockIdx.x, h = blockIdx.y;

    const uint32_t ring = smem_u32(smem + warp * (STAGES * STAGE_BYTES));
    unsigned char* after = smem + kWarps * STAGES * STAGE_BYTES;
    const uint32_t mbar0 = smem_u32(after) + warp * STAGES * 8;
    const uint32_t meta0 = smem_u32(after + kWarps * STAGES * 8) + warp * STAGES * 4;
    const uint32_t merge_bar = smem_u32(after + kWarps * STAGES * 12);
    float* merge_o = reinterpret_cast<float*>(after + kWarps * STAGES * 16);
    float* merge_m = merge_o + kWarps * p.n_rep * kMergeStride;
    float* merge_l = merge_m + kWarps * kRP;
    int* scan = reinterpret_cast<int*>(merge_l + kWarps * kRP);   // [kWarps]
    int* flag = scan + kWarps;                                    // [2]
    int* cum = flag + 2;                                          // [batch + 1]

    // Programmatic dependent launch as in decode_kernel: lengths and tables are read at once,
    // pages with LS_EARLY_PAGES except each sequence's last one.
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    if (lane == 0) {
#pragma unroll
        for (int s = 0; s < STAGES; ++s) mbar_init(mbar0 + 8 * s, 1);
        if (warp == 0) mbar_init(merge_bar, 1);
        mbar_init_fence();
    }
    __syncwarp();
    const int total = int4_prefix<kThreads>(p, cum, scan);
    const int chunk = int4_chunk_size(p, total);
    const int g0 = chunk_id * chunk, g1 = min(total, g0 + chunk);
    // The first sequence with pages in this chunk, and which.
    int b0 = g0 < total ? find_seq(cum, p.batch, g0) : p.batch, lo = 0, hi = 0;
    if (b0 < p.batch) int4_piece(cum, b0, g0, g1, lo, hi);
    if (b0 < p.batch && hi <= lo) {
        b0 = int4_next(cum, p.batch, b0, g1);
        if (b0 < p.batch) int4_piece(cum, b0, g0, g1, lo, hi);
    }
    const bool has_work = b0 < p.batch;
    GroupLoader<G> load;
    if (has_work) load.begin(p, cum, b0, lo, hi, g1, warp, lane);
    bool waited = false;
    auto dep_wait = [&]() {
        if (!waited) asm volatile("griddepcontrol.wait;\n" ::: "memory");
        waited = true;
    };
    const uint64_t policy = l2_policy_evict_first();      // pages are read once per step
    auto issue = [&](int slot) {
        load.issue(p, cum, h, warp, lane, ring + slot * STAGE_BYTES, mbar0 + 8 * slot, meta0 + 4 * slot, policy, dep_wait);
    };
    if (!p.early) dep_wait();
    if (has_work) {
#pragma unroll 1
        for (int s = 0; s < STAGES; ++s) issue(s);
    }
    dep_wait();

    if (chunk_id == 0) {
        // Sequences with nothing to attend produce zeros (nobody else writes them).
        for (int b = 0; b < p.batch; ++b)
            if (cum[b + 1] == cum[b])
                for (int r = 0; r < p.n_rep; ++r)
                    p.out[b * p.so_b + h * p.so_h + r * p.so_m + tid] = __float2half_rn(0.f);
    }
    if (!has_work) return;

    Int4State<G, TWICE> st;
    uint4 query[4];
    Int4State<G, TWICE>::load_query(p, b0, h, lane, query);
    int stage = 0, b = b0;
    uint32_t phase = 0;                                   // parity of the stage's mbarrier
    bool refill = false;                                  // whether the slot before this one has been consumed
    // Only a chunk's first and last sequence can have pages in other chunks as well.
    int shared_b0 = -1, shared_b1 = -1;
    for (int guard = 0; guard <= p.batch; ++guard) {
        const int end_u = warp_share(lo, hi, warp + 1);
        st.begin(p, query, lane);
        for (int u = warp_share(lo, hi, warp); u < end_u; u += PG) {
            if (!mbar_wait_bounded(mbar0 + 8 * stage, phase, kMbarSpinLimit) && lane == 0) p.seg_range[2 * p.batch] = 2;
            __syncwarp();
            const uint32_t meta = lds32(meta0 + 4 * stage), page = ring + stage * STAGE_BYTES;
            if (refill) issue(stage == 0 ? STAGES - 1 : stage - 1);      // the slot consumed one group ago
            refill = true;
            if (meta == PG * LS_PAGE) {
                st.template pages<PG, true>(page, LS_PAGE, lane);
            } else {
                // A segment's end, a sequence's last page, a page outside the pool: one by one.
                const int tokens = meta & 0xffff;
#pragma unroll 1
                for (int i = 0; i * LS_PAGE < tokens; ++i)
                    if (!((meta >> (16 + i)) & 1))
                        st.template pages<1, false>(page + i * int4_record_bytes(G), min(tokens - i * LS_PAGE, LS_PAGE), lane);
            }
            if (++stage == STAGES) {
                stage = 0;
                phase ^= 1u;
            }
        }
        const int next = int4_next(cum, p.batch, b, g1);
        const bool more = next < p.batch;
        if (more) Int4State<G, TWICE>::load_query(p, next, h, lane, query);
        if (guard > 0) __syncthreads();                   // the last sequence's sums have been read
        st.finish(merge_o + warp * p.n_rep * kMergeStride, merge_m + warp * kRP, merge_l + warp * kRP, p.n_rep, lane);
        __syncthreads();
        // The warps' states summed, a thread per channel: the output itself where the sequence lies
        // in this chunk alone, else one partial state. Lane 4 r + w works out warp w's weight of row r.
        const int c_lo = (cum[b] + kInt4Begin) / chunk, c_hi = (cum[b + 1] - 1) / chunk;
        float* state = state_of(p, chunk_id + b, h);
        const float mine = merge_m[(lane & 3) * kRP + (lane >> 2)];
        float top = fmaxf(mine, __shfl_xor_sync(LS_FULL_MASK, mine, 1));
        top = fmaxf(top, __shfl_xor_sync(LS_FULL_MASK, top, 2));
        const float f = ex2(mine - (top == neg_inf() ? 0.f : top));
        float l = f * merge_l[(lane & 3) * kRP + (lane >> 2)];
        l += __shfl_xor_sync(LS_FULL_MASK, l, 1);
        l += __shfl_xor_sync(LS_FULL_MASK, l, 2);
        const float inv = 1.f / fmaxf(l, 1e-20f);
        if (c_lo != c_hi && warp == 0 && (lane & 3) == 0) {
            state[lane >> 2] = top;
            state[kRP + (lane >> 2)] = l;
        }
#pragma unroll
        for (int r = 0; r < kRP; ++r) {
            float a = 0.f;
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float fw = __shfl_sync(LS_FULL_MASK, f, 4 * r + w);
                a = fmaf(fw, merge_o[(w * p.n_rep + min(r, p.n_rep - 1)) * kMergeStride + tid], a);
            }
            const float scale = __shfl_sync(LS_FULL_MASK, inv, 4 * r);
            if (r < p.n_rep) {
                if (c_lo == c_hi) p.out[b * p.so_b + h * p.so_h + r * p.so_m + tid] = __float2half_rn(a * scale);
                else state[kStateHead + r * LS_HEAD_DIM + tid] = a;
            }
        }
        if (c_lo != c_hi) {
            if (b == b0) shared_b0 = b;
            else shared_b1 = b;
        }
        if (!more) break;
        b = next;
        int4_piece(cum, b, 0, g1, lo, hi);
    }
    // Whoever brings a sequence's last partial merges them all. Arrival is counted with one
    // atomic per partial; nobody waits for anybody.
    if (shared_b0 < 0 && shared_b1 < 0) return;
    __syncthreads();                                      // the CTA's partials are written
    const int sb_mine = tid == 0 ? shared_b0 : shared_b1;
    if (tid < 2 && sb_mine >= 0) {
        const int sb = sb_mine;
        const int others = (cum[sb + 1] - 1) / chunk - (cum[sb] + kInt4Begin) / chunk;
        int* counter = p.seg_range + 2 * p.batch + 2 + sb * p.heads + h;
        int seen;
        // Releases the CTA's partial (ordered before this by the barrier) and acquires the others'.
        asm volatile("atom.add.acq_rel.gpu.s32 %0, [%1], 1;\n" : "=r"(seen) : "l"(counter) : "memory");
        flag[tid] = seen == others;
        if (seen == others) *counter = 0;                 // ready for the next launch
    }
    __syncthreads();
    uint32_t merge_phase = 0;
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
        const int sb = i == 0 ? shared_b0 : shared_b1;
        if (sb < 0 || !flag[i]) continue;
        const int c_lo = (cum[sb] + kInt4Begin) / chunk, count = (cum[sb + 1] - 1) / chunk - c_lo + 1;
        // Into the ring: every page that was requested has been consumed.
        int4_merge(p, c_lo + sb, count, sb, h, smem, kWarps * STAGES * STAGE_BYTES, merge_o, merge_bar,
                   merge_phase, tid);
    }
}

template <int G>
static int launch_int4(const DecodeParams& p, cudaStream_t stream, bool programmatic) {
    const size_t ring = (size_t)kWarps * kInt4Stages * kInt4Group * int4_record_bytes(G);
    const size_t smem = ring + kWarps * kInt4Stages * 16 +
                        sizeof(float) * ((size_t)kWarps * p.n_rep * kMergeStride + 2 * kWarps * kRP) +
                        sizeof(int) * ((size_t)kWarps + 2 + p.batch + 1);
    auto kern = p.n_rep <= 4 ? int4_decode_kernel<G, true> : int4_decode_kernel<G, false>;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return (int)e;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.num_chunks, p.heads);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = programmatic ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, kern, p);
    if (e != cudaSuccess) return (int)e;
    return (int)cudaGetLastError();
}

}  // namespace ls

extern "C" {

int ls_paged_decode_int4(const void* q, const void* kv_pool, const int32_t* block_tables, const int32_t* seq_lens,
                         float* part, int32_t* seg_range, void* out, int batch, int kv_heads, int n_rep, int groups,
                         int head_dim, int page, int max_pages, int num_blocks, int num_chunks, int min_chunk, int flags,
                         int64_t sq_b, int64_t sq_h, int64_t sq_m, int64_t sp_b, int64_t sp_h, int64_t so_b, int64_t so_h,
                         int64_t so_m, float softmax_scale, void* stream) {
    if (head_dim != LS_HEAD_DIM || page != LS_PAGE) return LS_ERR_UNSUPPORTED;
    if (groups != 1 && groups != 2 && groups != 4) return LS_ERR_UNSUPPORTED;
    if (flags & ~(LS_LAUNCH_PROGRAMMATIC | LS_EARLY_PAGES)) return LS_ERR_UNSUPPORTED;
    ls::DecodeParams p = {};
    p.q = static_cast<const __half*>(q);
    p.k_pool = p.v_pool = kv_pool;
    p.block_tables = block_tables;
    p.seq_lens = seq_lens;
    p.part_acc = p.part_m = p.part_l = part;             // states of its own layout: see state_of
    p.seg_range = seg_range;
    p.out = static_cast<__half*>(out);
    p.so_b = so_b; p.so_h = so_h; p.so_m = so_m;
    p.batch = batch;
    p.heads = kv_heads;
    p.n_rep = n_rep;
    p.max_pages = max_pages;
    p.num_blocks = num_blocks;
    p.num_res_rows = 1;
    p.num_chunks = num_chunks;
    p.min_chunk = min_chunk;
    p.sq_b = sq_b; p.sq_h = sq_h; p.sq_m = sq_m;
    p.sk_b = sp_b; p.sk_h = sp_h;
    p.early = (flags & LS_EARLY_PAGES) != 0;
    p.scale_log2 = softmax_scale * 1.4426950408889634f;
    if (!out) return LS_ERR_NULL_POINTER;
    const int rc = ls::validate_common(p);
    if (rc != LS_OK) return rc;
    if ((reinterpret_cast<uintptr_t>(kv_pool) & 15) || (reinterpret_cast<uintptr_t>(part) & 15) || (sp_b % 16) || (sp_h % 16)) return LS_ERR_MISALIGNED;
    if (sp_b < ls::int4_record_bytes(groups) || sp_h < ls::int4_record_bytes(groups)) return LS_ERR_BAD_STRIDE;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool pdl = (flags & LS_LAUNCH_PROGRAMMATIC) != 0;
    if (groups == 4) return ls::launch_int4<4>(p, s, pdl);
    if (groups == 2) return ls::launch_int4<2>(p, s, pdl);
    return ls::launch_int4<1>(p, s, pdl);
}

}  // extern "C"

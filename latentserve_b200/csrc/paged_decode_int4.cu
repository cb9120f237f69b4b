// Paged GQA decode attention over a cache held in 4 bits (record layout: int4_page.cuh). The
// split, the walk over the pages and the merge are those of the other pools (decode_core.cuh).
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
// steps are split into high and low fp16 halves, two MMAs per tile: with one fp16 rounding of the
// product alone, random values of V give outputs 1.4 times as far off as rounding the output is.
// The reference of the online softmax lags by at most 2 (log2), so w <= 4 and w * step <= 4 * 8734,
// inside fp16 for every step the writer can store.
#include "decode_core.cuh"
#include "int4_page.cuh"

namespace ls {

#ifndef LS_INT4_STAGES
#define LS_INT4_STAGES 4
#endif
#ifndef LS_INT4_CTAS
#define LS_INT4_CTAS 3
#endif
constexpr int kInt4Margin = 2;

// A page-head is one record: one bulk copy by one lane, completion counted on the stage's mbarrier.
template <int G>
struct PoolInt4 {
    static constexpr bool kTma = true;
    static constexpr int STAGE_BYTES = int4_record_bytes(G);

    static __device__ __forceinline__ int issue(const DecodeParams& p, const TmaMaps&, int, int h, const PageItem& it,
                                                uint32_t stage, uint32_t mbar, int lane, uint64_t pol) {
        if (lane == 0) {
            if (it.valid == 0) {
                mbar_arrive(mbar);                     // nothing to load: the phase completes at once
            } else {
                mbar_expect_tx(mbar, STAGE_BYTES);
                bulk_load_hint(stage, static_cast<const uint8_t*>(p.k_pool) + it.blk * p.sk_b + h * p.sk_h, STAGE_BYTES,
                               mbar, pol);
            }
        }
        return it.valid;
    }
};

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
__device__ __forceinline__ float half_lo(uint32_t x) { return __low2float(*reinterpret_cast<const __half2*>(&x)); }
__device__ __forceinline__ float half_hi(uint32_t x) { return __high2float(*reinterpret_cast<const __half2*>(&x)); }

// D += A(16x8, fp16, row) * B(8x8, fp16, col).
__device__ __forceinline__ void mma_1688(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm volatile(
        "mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(b0));
}

// Lane (g = lane / 4, j = lane % 4).
template <int G>
struct Int4State {
    using Pool = PoolInt4<G>;
    static constexpr int kMinCtas = LS_INT4_CTAS;
    static constexpr uint32_t kLow = 0x000f000fu, kHigh = 0x00f000f0u;
    uint32_t qb[4][4];         // B fragments of channels 32 w + 8 j ..: low-nibble channels (x16), high-nibble ones
    uint32_t qs;               // B fragment of the query's group sums (high and low fp16 parts)
    float o[9][4];             // O^T tile i < 8: channel 16 i + g of rows 2j, 2j+1 (in 2^-24), channel 16 i + 8 + g
                               // (in 2^-20); tile 8, lanes g < G: sum of w * lo of group g
    float m[2], l[2];
    float f[2];                // rows 2j, 2j+1: softmax scale (log2) over the query's power of two

    __device__ __forceinline__ void begin(const DecodeParams& p, int b, int h, int lane) {
        m[0] = m[1] = neg_inf();
        l[0] = l[1] = 0.f;
#pragma unroll
        for (int i = 0; i < 9; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) o[i][k] = 0.f;
        const int g = lane >> 2, j = lane & 3;
        const __half* src = p.q + b * p.sq_b + h * p.sq_h + g * p.sq_m + 8 * j;
        uint4 raw[4];
        float top = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            raw[w] = make_uint4(0, 0, 0, 0);
            if (g < p.n_rep) raw[w] = *reinterpret_cast<const uint4*>(src + 32 * w);
            const uint32_t* x = reinterpret_cast<const uint32_t*>(&raw[w]);
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(fabsf(half_lo(x[i])), fabsf(half_hi(x[i]))));
        }
        top = fmaxf(top, __shfl_xor_sync(LS_FULL_MASK, top, 1));
        top = fmaxf(top, __shfl_xor_sync(LS_FULL_MASK, top, 2));
        // The row is multiplied by the power of two that brings its largest value into [8, 16).
        const int e = top > 0.f ? 130 - (__float_as_int(top) >> 23) : 0;
        const float up = __int_as_float((127 + e) << 23);
        const float back = p.scale_log2 * __int_as_float((127 - e) << 23);
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
        // their low parts; see compute_page for which lows a lane's register holds.
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

    __device__ __forceinline__ void compute(const DecodeParams& p, uint32_t stage, int meta, int lane, uint32_t) {
        if (meta == LS_PAGE) compute_page<true>(p, stage, meta, lane);
        else compute_page<false>(p, stage, meta, lane);
    }

    template <bool FULL>
    __device__ __forceinline__ void compute_page(const DecodeParams& p, uint32_t stage, int valid, int lane) {
        const int g = lane >> 2, j = lane & 3;
        // Scores.
        float s[4];
        {
            const uint4 w0 = lds128(stage + 64 * g + 16 * j), w1 = lds128(stage + 64 * (g + 8) + 16 * j);
            const uint32_t* k0 = reinterpret_cast<const uint32_t*>(&w0);
            const uint32_t* k1 = reinterpret_cast<const uint32_t*>(&w1);
            uint32_t low0, low1;                    // this lane's column pair of the lows, tokens g and g + 8
            float st0[G], st1[G];                   // steps of tokens g and g + 8
            if (G == 4) {
                const uint4 c0 = lds128(stage + kI4Scales + 16 * g), c1 = lds128(stage + kI4Scales + 16 * (g + 8));
                low0 = (j & 1) ? c0.w : c0.z;
                low1 = (j & 1) ? c1.w : c1.z;
                st0[0] = half_lo(c0.x); st0[1 % G] = half_hi(c0.x); st0[2 % G] = half_lo(c0.y); st0[3 % G] = half_hi(c0.y);
                st1[0] = half_lo(c1.x); st1[1 % G] = half_hi(c1.x); st1[2 % G] = half_lo(c1.y); st1[3 % G] = half_hi(c1.y);
            } else if (G == 2) {
                const uint2 c0 = lds64(stage + kI4Scales + 8 * g), c1 = lds64(stage + kI4Scales + 8 * (g + 8));
                low0 = c0.y;
                low1 = c1.y;
                st0[0] = half_lo(c0.x); st0[1 % G] = half_hi(c0.x);
                st1[0] = half_lo(c1.x); st1[1 % G] = half_hi(c1.x);
            } else {
                low0 = lds32(stage + kI4Scales + 4 * g);         // (step, lo): the step meets a zero
                low1 = lds32(stage + kI4Scales + 4 * (g + 8));
                st0[0] = half_lo(low0);
                st1[0] = half_lo(low1);
            }
            float base[4] = {0.f, 0.f, 0.f, 0.f};
            mma_1688(base, low0, low1, qs);
            s[0] = s[1] = s[2] = s[3] = 0.f;
#pragma unroll
            for (int y = 0; y < G; ++y) {
                float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int w = y * (4 / G); w < (y + 1) * (4 / G); ++w) {
                    const uint32_t x0 = k0[w], x1 = k1[w], z0 = x0 >> 8, z1 = x1 >> 8;
                    mma_16816(acc, x0 & kLow, x1 & kLow, z0 & kLow, z1 & kLow, qb[w][0], qb[w][1]);
                    mma_16816(acc, x0 & kHigh, x1 & kHigh, z0 & kHigh, z1 & kHigh, qb[w][2], qb[w][3]);
                }
                s[0] = fmaf(st0[y], acc[0], s[0]);
                s[1] = fmaf(st0[y], acc[1], s[1]);
                s[2] = fmaf(st1[y], acc[2], s[2]);
                s[3] = fmaf(st1[y], acc[3], s[3]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] = fmaf(s[i], 1048576.f, base[i]) * f[i & 1];       // codes in 2^-20
        }
        if (!FULL) {
            if (g >= valid) s[0] = s[1] = neg_inf();
            if (g + 8 >= valid) s[2] = s[3] = neg_inf();
        }
        float a0, a1;
        softmax_update<9, kInt4Margin>(s, m, l, o, a0, a1);
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
            uint2 lows = make_uint2(0, 0);
            if (g < G) lows = lds64(stage + int4_v_lows(G) + 8 * G * j + 8 * g);
            if (!FULL) {
                lows.x &= keep0;
                lows.y &= keep1;
            }
            mma_16816(o[8], lows.x, 0u, lows.y, 0u, w0h, w1h);
            mma_16816(o[8], lows.x, 0u, lows.y, 0u, w0l, w1l);
        }
        uint32_t st[2 * G];                          // V steps [group][half]
        if (G == 1) {
            const uint2 c = lds64(stage + int4_v_steps(G) + 8 * j);
            st[0] = c.x; st[1] = c.y;
        } else {
#pragma unroll
            for (int y = 0; y < G; y += 2) {
                const uint4 c = lds128(stage + int4_v_steps(G) + 8 * G * j + 8 * y);
                st[2 * y] = c.x; st[2 * y + 1] = c.y; st[(2 * y + 2) % (2 * G)] = c.z; st[(2 * y + 3) % (2 * G)] = c.w;
            }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const uint4 v4 = lds128(stage + kI4V + 512 * c + 16 * lane);
            const uint32_t* v = reinterpret_cast<const uint32_t*>(&v4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int tile = 4 * c + i, y = tile * G / 8;
                uint32_t t0 = st[2 * y], t1 = st[2 * y + 1];
                if (!FULL) {
                    t0 &= keep0;
                    t1 &= keep1;
                }
                // w * step in two halves: the rounded product, and what it and the weight's low half left.
                const uint32_t b0 = hmul2_u32(w0h, t0), b1 = hmul2_u32(w1h, t1);
                const uint32_t e0 = hfma2_u32(w0l, t0, hfma2_u32(w0h, t0, b0 ^ 0x80008000u));
                const uint32_t e1 = hfma2_u32(w1l, t1, hfma2_u32(w1h, t1, b1 ^ 0x80008000u));
                const uint32_t x = v[i], z = x >> 8;
                mma_16816(o[tile], x & kLow, x & kHigh, z & kLow, z & kHigh, b0, b1);
                mma_16816(o[tile], x & kLow, x & kHigh, z & kLow, z & kHigh, e0, e1);
            }
        }
    }

    __device__ __forceinline__ void finish(float* mo, float* mm, float* ml, int n_rep, int lane) {
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) {
            l[0] += __shfl_xor_sync(LS_FULL_MASK, l[0], off);
            l[1] += __shfl_xor_sync(LS_FULL_MASK, l[1], off);
        }
        const int g = lane >> 2, j = lane & 3;
        const int r0 = 2 * j, r1 = r0 + 1;
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
        if (g == 0) {
            if (r0 < n_rep) { mm[r0] = m[0]; ml[r0] = l[0]; }
            if (r1 < n_rep) { mm[r1] = m[1]; ml[r1] = l[1]; }
        }
    }
};

}  // namespace ls

extern "C" {

int ls_paged_decode_int4(const void* q, const void* kv_pool, const int32_t* block_tables, const int32_t* seq_lens,
                         float* part_acc, float* part_m, float* part_l, int32_t* seg_range, void* out, int batch,
                         int kv_heads, int n_rep, int groups, int head_dim, int page, int max_pages, int num_blocks,
                         int num_chunks, int min_chunk, int flags, int64_t sq_b, int64_t sq_h, int64_t sq_m, int64_t sp_b,
                         int64_t sp_h, int64_t so_b, int64_t so_h, int64_t so_m, float softmax_scale, void* stream) {
    if (head_dim != LS_HEAD_DIM || page != LS_PAGE) return LS_ERR_UNSUPPORTED;
    if (groups != 1 && groups != 2 && groups != 4) return LS_ERR_UNSUPPORTED;
    if (flags & ~(LS_LAUNCH_PROGRAMMATIC | LS_EARLY_PAGES)) return LS_ERR_UNSUPPORTED;
    ls::DecodeParams p = {};
    p.q = static_cast<const __half*>(q);
    p.k_pool = p.v_pool = kv_pool;
    p.block_tables = block_tables;
    p.seq_lens = seq_lens;
    p.part_acc = part_acc;
    p.part_m = part_m;
    p.part_l = part_l;
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
    const int rc = ls::validate_common(p);
    if (rc != LS_OK) return rc;
    if ((reinterpret_cast<uintptr_t>(kv_pool) & 15) || (sp_b % 16) || (sp_h % 16)) return LS_ERR_MISALIGNED;
    if (sp_b < ls::int4_record_bytes(groups) || sp_h < ls::int4_record_bytes(groups)) return LS_ERR_BAD_STRIDE;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool pdl = (flags & LS_LAUNCH_PROGRAMMATIC) != 0;
    if (groups == 4) return ls::launch_decode<ls::Int4State<4>, LS_MODE_DENSE, LS_INT4_STAGES>(p, s, pdl);
    if (groups == 2) return ls::launch_decode<ls::Int4State<2>, LS_MODE_DENSE, LS_INT4_STAGES>(p, s, pdl);
    return ls::launch_decode<ls::Int4State<1>, LS_MODE_DENSE, LS_INT4_STAGES>(p, s, pdl);
}

}  // extern "C"

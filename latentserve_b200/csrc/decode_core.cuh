// The split-KV decode kernel and what its variants share: the walk of a warp over its pages,
// the online softmax on MMA fragments, the merge of partial states, and the launch. A variant
// is a State class (how one page is computed) with a Pool class (how one page is fetched);
// see paged_decode.cu (fp16, INT8, page-sparse) and paged_decode_int4.cu.
#pragma once

#include <cuda.h>

#include "decode_sched.cuh"

#include <type_traits>

namespace ls {

constexpr int kWarps = 4;
// Tensor maps of the TMA-loading variants (unused and zero for the others).
struct TmaMaps {
    CUtensorMap k, v, ks, kz;
    CUtensorMap kv;                 // INT8: K and V pools as one 5-d tensor (see build_int8_maps)
};
constexpr int kMbarSpinLimit = 1 << 22;   // probes of an mbarrier phase before a warp gives up
constexpr int kThreads = kWarps * 32;
constexpr int kMergeStride = LS_HEAD_DIM + 4;   // floats per merged row (bank-conflict pad)
constexpr int kRP = 8;                          // query rows held per partial


// What the load side knows about the page it is about to fetch.
struct PageItem {
    int blk;
    int valid;      // tokens of the page that exist (0 = skip)
    int last;       // bit 0: the sequence's last page; bit 1: a page the step before this
                    // launch may still be writing (never requested ahead of the dependency wait)
    int vl;         // valid | last << 8: equals LS_PAGE for a full page of a sequence's interior
};

// Lookahead over a warp's page sequence. Lane j of the warp holds the block id
// and extent of the j-th upcoming page of the current segment (up to 32 pages),
// fetched with one round of independent loads (two for the sparse kernel:
// selection entry, then block-table entry) instead of a dependent scalar load
// per page. The next window is fetched while the last two pages of the current
// one are still being handed out, so its latency hides behind compute.
template <int MODE>
struct PageWindow {
    Cursor c;                       // first page of the current window
    int n, i;                       // pages in the window, next one to hand out
    int blk, vl;                    // lane j: page j's block id, and valid tokens | last-page bits << 8
    Cursor nc;                      // the window after this one
    int nn, nblk, nvl;
    bool have_next;
    int cached_b, cached_len;

    __device__ __forceinline__ void fill(const DecodeParams& p, const Cursor& cur, int h, int lane,
                                         int& cnt, int& b_, int& vl_) {
        cnt = 0; b_ = 0; vl_ = 0;
        if (cur.done) return;
        if (cur.b != cached_b) {
            cached_b = cur.b;
            cached_len = max(p.seq_lens[cur.b], 0);
        }
        const int np = min((cached_len + LS_PAGE - 1) / LS_PAGE, p.max_pages);
        cnt = min(32, (cur.hi - cur.u + kWarps - 1) / kWarps);
        const int u = cur.u + kWarps * lane;
        const bool in = lane < cnt;
        int page = u;
        if (MODE == LS_MODE_SPARSE && in) page = p.sel[cur.b * p.sl_b + h * p.sl_h + u];
        if (in && page >= 0 && page < np) {
            const int id = p.block_tables[(long long)cur.b * p.max_pages + page];
            if (id >= 0 && id < p.num_blocks) {
                b_ = id;
                // INT8 pools: the page before the last is rewritten (K bytes and K scales,
                // by the page-finalize kernel) in the step whose new token opened the last
                // page, so it counts as mutable too; every earlier page is final.
                const int last = (page == np - 1 ? 1 : 0) | ((p.k_scale != nullptr && page >= np - 2) ? 2 : 0);
                vl_ = min(LS_PAGE, cached_len - page * LS_PAGE) | (last << 8);
            } else {
                p.seg_range[2 * p.batch] = 1;      // corrupt table: read nothing, flag it
            }
        }
    }

    __device__ __forceinline__ void begin(const DecodeParams& p, const Cursor& first, int h,
                                          int lane) {
        cached_b = -1;
        cached_len = 0;
        c = first;
        fill(p, c, h, lane, n, blk, vl);
        i = 0;
        have_next = false;
    }

    __device__ __forceinline__ void prefetch(const DecodeParams& p, const int* cum, int h, int warp,
                                             int lane) {
        nc = c;
        nc.u += kWarps * n;
        cursor_normalize<kWarps>(nc, cum, p.batch, warp);
        fill(p, nc, h, lane, nn, nblk, nvl);
        have_next = true;
    }

    // Next page of this warp; false when the chunk is exhausted. `b` is its sequence.
    __device__ __forceinline__ bool next(const DecodeParams& p, const int* cum, int h, int warp,
                                         int lane, PageItem& it, int& b) {
        if (i == n) {
            // The window after this one was fetched when its last pages were handed out
            // (below): every non-empty window reaches i + 2 >= n before it reaches i == n.
            if (n == 0 || !have_next) return false;
            c = nc; n = nn; blk = nblk; vl = nvl;
            have_next = false;
            i = 0;
            if (n == 0) return false;
        }
        it.blk = __shfl_sync(LS_FULL_MASK, blk, i);
        const int v = __shfl_sync(LS_FULL_MASK, vl, i);
        it.vl = v;
        it.valid = v & 255;
        it.last = v >> 8;
        b = c.b;
        ++i;
        // Once per window, when its last two pages are about to be handed out (i + 2 >= n
        // for the first time): one compare instead of three tests per page.
        if (i == max(n - 2, 1)) prefetch(p, cum, h, warp, lane);
        return true;
    }
};

// ---------------------------------------------------------------------------
// Online softmax on MMA accumulator fragments. Lane (g = lane / 4, t = lane % 4)
// holds scores of tokens g and g + 8 for query rows 2t and 2t + 1:
// s[0] = (g, 2t), s[1] = (g, 2t+1), s[2] = (g+8, 2t), s[3] = (g+8, 2t+1).
// On return s holds the weights 2^(s - m_new); m, l and the output
// accumulators o[8][4] are rescaled. Scores are in the log2 domain.
// The reference may lag the scores by MARGIN (log2 units): weights stay below 2^MARGIN.
template <int TILES, int MARGIN = 8>
__device__ __forceinline__ void softmax_update(float (&s)[4], float (&m)[2], float (&l)[2],
                                               float (&o)[TILES][4], float& a0, float& a1) {
    // Usual case after a segment's first pages: no score of the page rises more
    // than 2^MARGIN above the running reference m. Then m is kept as it is
    // (any shared reference gives the same normalised result; weights stay below
    // 2^MARGIN, well inside fp16) and one vote replaces the six shuffles and
    // the rescale test. The choice depends on the data only, so results are
    // reproducible.
    {
        const float lim0 = m[0] + (float)MARGIN, lim1 = m[1] + (float)MARGIN;
        const bool ok = (m[0] != neg_inf()) & (m[1] != neg_inf()) & (s[0] <= lim0) & (s[2] <= lim0) &
                        (s[1] <= lim1) & (s[3] <= lim1);
        if (__all_sync(LS_FULL_MASK, ok)) {
            a0 = a1 = 1.f;
            s[0] = ex2(s[0] - m[0]);
            s[1] = ex2(s[1] - m[1]);
            s[2] = ex2(s[2] - m[0]);
            s[3] = ex2(s[3] - m[1]);
            l[0] += s[0] + s[2];
            l[1] += s[1] + s[3];
            return;
        }
    }
    float mx0 = fmaxf(s[0], s[2]);
    float mx1 = fmaxf(s[1], s[3]);
#pragma unroll
    for (int off = 4; off < 32; off <<= 1) {
        mx0 = fmaxf(mx0, __shfl_xor_sync(LS_FULL_MASK, mx0, off));
        mx1 = fmaxf(mx1, __shfl_xor_sync(LS_FULL_MASK, mx1, off));
    }
    const float mn0 = fmaxf(m[0], mx0), mn1 = fmaxf(m[1], mx1);
    // A row that has seen no valid token keeps m = -inf; subtracting a finite
    // stand-in keeps exp2 away from (-inf) - (-inf).
    const float ms0 = (mn0 == neg_inf()) ? 0.f : mn0;
    const float ms1 = (mn1 == neg_inf()) ? 0.f : mn1;
    a0 = ex2(m[0] - ms0);
    a1 = ex2(m[1] - ms1);
    s[0] = ex2(s[0] - ms0);
    s[1] = ex2(s[1] - ms1);
    s[2] = ex2(s[2] - ms0);
    s[3] = ex2(s[3] - ms1);
    m[0] = mn0;
    m[1] = mn1;
    l[0] = l[0] * a0 + (s[0] + s[2]);
    l[1] = l[1] * a1 + (s[1] + s[3]);
    // Once a row's running maximum has settled (the usual case after the first
    // few pages) the factors are exactly 1 and the rescale is skipped.
    if (a0 != 1.f || a1 != 1.f) {
#pragma unroll
        for (int mt = 0; mt < TILES; ++mt) {
            o[mt][0] *= a0;
            o[mt][1] *= a1;
            o[mt][2] *= a0;
            o[mt][3] *= a1;
        }
    }
}

__device__ __forceinline__ void mask_and_scale(float (&s)[4], int valid, float scale_log2, int lane) {
    const int g = lane >> 2;
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] *= scale_log2;
    if (g >= valid) s[0] = s[1] = neg_inf();
    if (g + 8 >= valid) s[2] = s[3] = neg_inf();
}

__device__ __forceinline__ uint32_t hmul2_u32(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
    uint4 r;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
                 : "r"(addr));
    return r;
}
__device__ __forceinline__ float lds32f(uint32_t addr) {
    float r;
    asm volatile("ld.shared.f32 %0, [%1];\n" : "=f"(r) : "r"(addr));
    return r;
}

// ---------------------------------------------------------------------------
// Merge of a sequence's partials:
//   out = sum_s acc_s 2^(m_s - M) / max(sum_s l_s 2^(m_s - M), 1e-20),
// the reference combine (kernels/gqa/paged_decode.py:421-471, torch form
// :689-706) with m held in the log2 domain. Called by the 4 warps of a CTA:
// warp w takes query rows w, w + 4; lane s holds partial s's (m, l) and weight,
// and the 32 lanes cover the 128 dims as float4, so a row of one partial is one
// coalesced 512-byte load and the loads of a row's partials are independent
// (issued back to back, not one L2 round trip after another). Loads bypass L1
// because other CTAs of the same launch may have written the partials.
__device__ __forceinline__ void merge_partials(const float* part_acc, const float* part_m,
                                               const float* part_l, int first, int count,
                                               __half* out, int heads, int n_rep, int b, int h,
                                               int tid, long long so_b, long long so_h,
                                               long long so_m) {
    constexpr int kBatch = 8;                                // partial rows loaded per round
    const int warp = tid >> 5, lane = tid & 31;
    const long long step = (long long)heads * kRP;           // rows between partials
    // Warp w merges rows w and w + 4 together, so both rows' loads are in flight at once.
    const int r0 = warp, r1 = warp + kWarps;
    const bool has0 = r0 < n_rep, has1 = r1 < n_rep;
    if (!has0) return;
    const long long base0 = ((long long)first * heads + h) * kRP + r0;
    const long long base1 = base0 + kWarps;
    const float4* src0 = reinterpret_cast<const float4*>(part_acc + base0 * LS_HEAD_DIM) + lane;
    const float4* src1 = src0 + kWarps * (LS_HEAD_DIM / 4);
    const long long pstep = step * (LS_HEAD_DIM / 4);

    // One round trip for everything the usual case needs: lane s's (m, l) of partial s,
    // and the accumulator rows of the first kBatch partials (which do not depend on m).
    float pm0 = neg_inf(), pm1 = neg_inf(), pl0 = 0.f, pl1 = 0.f;
    if (lane < count) {
        pm0 = __ldcg(part_m + base0 + lane * step);
        pl0 = __ldcg(part_l + base0 + lane * step);
        if (has1) {
            pm1 = __ldcg(part_m + base1 + lane * step);
            pl1 = __ldcg(part_l + base1 + lane * step);
        }
    }
    float4 v0[kBatch], v1[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
        const bool ok = j < count;
        v0[j] = ok ? __ldcg(src0 + j * pstep) : make_float4(0.f, 0.f, 0.f, 0.f);
        v1[j] = (ok && has1) ? __ldcg(src1 + j * pstep) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float mg0 = pm0, mg1 = pm1;
    for (int s = lane + 32; s < count; s += 32) {            // more than 32 partials: rare
        mg0 = fmaxf(mg0, __ldcg(part_m + base0 + s * step));
        if (has1) mg1 = fmaxf(mg1, __ldcg(part_m + base1 + s * step));
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        mg0 = fmaxf(mg0, __shfl_xor_sync(LS_FULL_MASK, mg0, off));
        mg1 = fmaxf(mg1, __shfl_xor_sync(LS_FULL_MASK, mg1, off));
    }
    const float ms0 = (mg0 == neg_inf()) ? 0.f : mg0;
    const float ms1 = (mg1 == neg_inf()) ? 0.f : mg1;
    float ls0 = 0.f, ls1 = 0.f;
    float4 a0 = make_float4(0.f, 0.f, 0.f, 0.f), a1 = a0;
    for (int s0 = 0; s0 < count; s0 += 32) {
        const int s = s0 + lane;
        float w0 = 0.f, w1 = 0.f;
        if (s < count) {
            if (s0 > 0) {
                pm0 = __ldcg(part_m + base0 + s * step);
                pl0 = __ldcg(part_l + base0 + s * step);
                if (has1) {
                    pm1 = __ldcg(part_m + base1 + s * step);
                    pl1 = __ldcg(part_l + base1 + s * step);
                }
            }
            w0 = ex2(pm0 - ms0);
            ls0 += w0 * pl0;
            if (has1) {
                w1 = ex2(pm1 - ms1);
                ls1 += w1 * pl1;
            }
        }
        const int n = min(32, count - s0);
        for (int j0 = 0; j0 < n; j0 += kBatch) {
            if (s0 + j0 > 0) {                               // the first batch is already here
#pragma unroll
                for (int j = 0; j < kBatch; ++j) {
                    const bool ok = j0 + j < n;
                    v0[j] = ok ? __ldcg(src0 + (s0 + j0 + j) * pstep) : make_float4(0.f, 0.f, 0.f, 0.f);
                    v1[j] = (ok && has1) ? __ldcg(src1 + (s0 + j0 + j) * pstep)
                                         : make_float4(0.f, 0.f, 0.f, 0.f);
                }
            }
#pragma unroll
            for (int j = 0; j < kBatch; ++j) {
                const float x0 = __shfl_sync(LS_FULL_MASK, w0, (j0 + j) & 31);
                const float x1 = __shfl_sync(LS_FULL_MASK, w1, (j0 + j) & 31);
                a0.x += x0 * v0[j].x; a0.y += x0 * v0[j].y; a0.z += x0 * v0[j].z; a0.w += x0 * v0[j].w;
                a1.x += x1 * v1[j].x; a1.y += x1 * v1[j].y; a1.z += x1 * v1[j].z; a1.w += x1 * v1[j].w;
            }
        }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) {
        ls0 += __shfl_xor_sync(LS_FULL_MASK, ls0, off);
        ls1 += __shfl_xor_sync(LS_FULL_MASK, ls1, off);
    }
    const float i0 = 1.f / fmaxf(ls0, 1e-20f), i1 = 1.f / fmaxf(ls1, 1e-20f);
    uint2 packed;
    packed.x = pack_half2(a0.x * i0, a0.y * i0);
    packed.y = pack_half2(a0.z * i0, a0.w * i0);
    *reinterpret_cast<uint2*>(out + b * so_b + h * so_h + r0 * so_m + lane * 4) = packed;
    if (has1) {
        packed.x = pack_half2(a1.x * i1, a1.y * i1);
        packed.y = pack_half2(a1.z * i1, a1.w * i1);
        *reinterpret_cast<uint2*>(out + b * so_b + h * so_h + r1 * so_m + lane * 4) = packed;
    }
}

// ---------------------------------------------------------------------------
template <class State, int MODE, int STAGES>
__global__ void __launch_bounds__(kThreads, State::kMinCtas)
decode_kernel(const DecodeParams p, const __grid_constant__ TmaMaps maps) {
    extern __shared__ __align__(1024) unsigned char smem[];
    using Pool = typename State::Pool;
    constexpr int STAGE_BYTES = Pool::STAGE_BYTES;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int chunk_id = blockIdx.x, h = blockIdx.y;

    // After the ring: one mbarrier per (warp, stage) for the TMA-loading variants.
    const uint32_t mbar0 = smem_u32(smem + kWarps * STAGES * STAGE_BYTES) + warp * STAGES * 8;
    float* merge_o = reinterpret_cast<float*>(smem + kWarps * STAGES * STAGE_BYTES + kWarps * STAGES * 8);
    float* merge_m = merge_o + kWarps * p.n_rep * kMergeStride;
    float* merge_l = merge_m + kWarps * kRP;
    int* scan = reinterpret_cast<int*>(merge_l + kWarps * kRP);   // [kWarps]
    int* flag = scan + kWarps;                                    // [1]
    int* cum = flag + 1;                                          // [batch + 1]

    // Programmatic dependent launch: let the next kernel of the stream be
    // scheduled as this one drains, and -- when this launch was itself made
    // with the attribute -- do the part of the prologue that reads only
    // seq_lens and block_tables while the previous kernel is still finishing.
    // Without the attribute both instructions are no-ops.
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
    if (Pool::kTma) {
        if (lane == 0) {
#pragma unroll
            for (int s = 0; s < STAGES; ++s) mbar_init(mbar0 + 8 * s, 1);
            mbar_init_fence();
        }
        __syncwarp();
    }
    const int total = build_prefix<MODE, kThreads>(p, cum, scan);
    const int chunk = chunk_size(p, total);
    const int g0 = chunk_id * chunk;
    const int g1 = min(total, g0 + chunk);
    const bool has_work = g0 < total;
    const int b0 = has_work ? find_seq(cum, p.batch, g0) : 0;
    const uint32_t ring = smem_u32(smem + warp * (STAGES * STAGE_BYTES));
    const uint32_t warp_scratch = smem_u32(merge_o + warp * p.n_rep * kMergeStride);   // free while pages are walked

    // Load side. The dense walk needs nothing the previous kernel may have
    // written; the sparse walk reads the selection, which it usually did write.
    // With LS_EARLY_PAGES the first pages are requested before the dependency
    // wait as well: a decode step's predecessor (the KV append) writes only the
    // newest token, which lies in its sequence's last page, so every other page
    // is immutable; a warp waits before it requests a last page. An INT8 cache also
    // rewrites the page before the last one (its K page is quantised, by a kernel that
    // precedes the append, in the step after it filled up), so there the wait comes
    // before either of a sequence's two last pages.
    PageWindow<MODE> win;
    const bool early = MODE == LS_MODE_DENSE && p.early != 0;
    if (MODE == LS_MODE_DENSE && has_work)
        win.begin(p, cursor_begin<kWarps>(cum, p.batch, b0, g0, g1, warp), h, lane);
    bool waited = false;
    auto dep_wait = [&]() {
        if (!waited) asm volatile("griddepcontrol.wait;\n" ::: "memory");
        waited = true;
    };
    // KV pages are read once per step: evict-first keeps tables, lengths, queries and
    // partials in L2.
    const uint64_t pol = l2_policy_evict_first();
    // What the load side knows about the page in each ring slot (valid tokens, flags):
    // warp-uniform, indexed by compile-time slot numbers only, so it lives in registers.
    int slot_meta[STAGES];
#pragma unroll
    for (int s = 0; s < STAGES; ++s) slot_meta[s] = 0;
    auto issue = [&](int slot) {
        PageItem item;
        int lb;
        if (win.next(p, cum, h, warp, lane, item, lb)) {
            if (item.vl != LS_PAGE && item.last) dep_wait();
            int mt;
            if constexpr (Pool::kTma)
                mt = Pool::issue(p, maps, lb, h, item, ring + slot * STAGE_BYTES, mbar0 + 8 * slot, lane, pol);
            else
                mt = Pool::issue(p, lb, h, item, ring + slot * STAGE_BYTES, lane, pol);
#pragma unroll
            for (int q = 0; q < STAGES; ++q) slot_meta[q] = slot == q ? mt : slot_meta[q];
        }
        if (!Pool::kTma) cp_async_commit();
    };
    auto issue_first = [&]() {                               // STAGES - 1 pages ahead
#pragma unroll 1
        for (int s = 0; s < STAGES - 1; ++s) issue(s);       // one copy of the code, not STAGES - 1
    };
    if (early && has_work) issue_first();
    dep_wait();

    if (chunk_id == 0 && h == 0) write_seg_ranges<kThreads>(p, cum, chunk);
    if (chunk_id == 0 && p.out != nullptr) {
        // Sequences with nothing to attend produce zeros (nobody else writes them).
        for (int b = 0; b < p.batch; ++b) {
            if (cum[b + 1] != cum[b]) continue;
            for (int i = tid; i < p.n_rep * LS_HEAD_DIM; i += kThreads)
                p.out[b * p.so_b + h * p.so_h + (i >> 7) * p.so_m + (i & 127)] = __float2half_rn(0.f);
        }
    }
    if (!has_work) return;
    if (MODE != LS_MODE_DENSE)
        win.begin(p, cursor_begin<kWarps>(cum, p.batch, b0, g0, g1, warp), h, lane);
    if (!early) issue_first();

    // Compute side: segment by segment. One page step: wait for the slot, refill the slot
    // consumed one page ago, compute. (A copy of the step per ring slot, with the slot a
    // compile-time constant, was measured: the larger code cost more than the immediates saved.)
    State st;
    int stage = 0;         // ring slot of the page being consumed
    uint32_t phase = 0;    // parity of that slot's mbarrier phase (TMA variants)
    int b = b0;
    int first_u = g0 - cum[b0];
    for (int guard = 0; guard <= p.batch; ++guard) {
        const int hi = min(g1, cum[b + 1]) - cum[b];
        st.begin(p, b, h, lane);
        for (int u = first_u + warp; u < hi; u += kWarps) {
            {
                const uint32_t bar = mbar0 + 8 * stage;
                if constexpr (Pool::kTma) {
                    if (!mbar_wait_bounded(bar, phase, kMbarSpinLimit)) {
                        if (lane == 0) p.seg_range[2 * p.batch] = 2;
                    }
                } else {
                    cp_async_wait<STAGES - 2>();
                }
                __syncwarp();
                int meta_now = slot_meta[0];
#pragma unroll
                for (int q = 1; q < STAGES; ++q) meta_now = stage == q ? slot_meta[q] : meta_now;
                issue(stage == 0 ? STAGES - 1 : stage - 1);          // the slot consumed one page ago
#ifndef LS_LOADS_ONLY
                st.compute(p, ring + stage * STAGE_BYTES, meta_now, lane, warp_scratch);
#else
                (void)meta_now;                          // build flag: pages land, nothing is computed
#endif
            }
            if (++stage == STAGES) {
                stage = 0;
                phase ^= 1u;
            }
        }
        st.finish(merge_o + warp * p.n_rep * kMergeStride, merge_m + warp * kRP,
                  merge_l + warp * kRP, p.n_rep, lane);
        __syncthreads();
        const int slot = chunk_id + b;
        {
            // CTA merge: thread = one of the 128 dims, all rows.
            float* pa = p.part_acc + ((long long)slot * p.heads + h) * kRP * LS_HEAD_DIM;
            float* pm = p.part_m + ((long long)slot * p.heads + h) * kRP;
            float* pl = p.part_l + ((long long)slot * p.heads + h) * kRP;
            for (int r = 0; r < p.n_rep; ++r) {
                float mg = neg_inf();
#pragma unroll
                for (int w = 0; w < kWarps; ++w) mg = fmaxf(mg, merge_m[w * kRP + r]);
                const float ms = (mg == neg_inf()) ? 0.f : mg;
                float lsum = 0.f;
                float wgt[kWarps];
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    wgt[w] = ex2(merge_m[w * kRP + r] - ms);
                    lsum += wgt[w] * merge_l[w * kRP + r];
                }
                for (int d = tid; d < LS_HEAD_DIM; d += kThreads) {
                    float a = 0.f;
#pragma unroll
                    for (int w = 0; w < kWarps; ++w)
                        a += wgt[w] * merge_o[(w * p.n_rep + r) * kMergeStride + d];
                    pa[r * LS_HEAD_DIM + d] = a;
                }
                if (tid == 0) {
                    pm[r] = mg;
                    pl[r] = lsum;
                }
            }
        }
        if (p.out != nullptr) {
            // Whoever brings a sequence's last partial merges them all. Arrival is
            // counted with one atomic per segment; nobody waits for anybody.
            const int c_lo = cum[b] / chunk, c_hi = (cum[b + 1] - 1) / chunk;
            const int nseg = c_hi - c_lo + 1;
            int* counter = p.seg_range + 2 * p.batch + 2 + b * p.heads + h;
            __syncthreads();                                  // the CTA's partial is written
            if (tid == 0) {
                int last = 1;
                if (nseg > 1) {
                    // Release the CTA's partial (ordered before this by the barrier) and
                    // acquire the others' in one atomic; the merge reads them from L2.
                    int seen;
                    asm volatile("atom.add.acq_rel.gpu.s32 %0, [%1], 1;\n" : "=r"(seen) : "l"(counter) : "memory");
                    last = seen == nseg - 1;
                    if (last) *counter = 0;                  // ready for the next launch
                }
                *flag = last;
            }
            __syncthreads();
            if (*flag) {
                merge_partials(p.part_acc, p.part_m, p.part_l, c_lo + b, nseg, p.out, p.heads,
                               p.n_rep, b, h, tid, p.so_b, p.so_h, p.so_m);
            }
        }
        if (cum[b + 1] >= g1) break;
        __syncthreads();
        ++b;
        while (b < p.batch - 1 && cum[b + 1] == cum[b]) ++b;
        first_u = 0;
    }
    cp_async_wait<0>();
}

// ---------------------------------------------------------------------------
static int validate_common(const DecodeParams& p) {
    if (!p.q || !p.k_pool || !p.v_pool || !p.block_tables || !p.seq_lens || !p.part_acc ||
        !p.part_m || !p.part_l || !p.seg_range)
        return LS_ERR_NULL_POINTER;
    if (p.batch <= 0 || p.heads <= 0 || p.n_rep <= 0 || p.max_pages <= 0 || p.num_chunks <= 0 ||
        p.num_blocks <= 0 || p.min_chunk <= 0)
        return LS_ERR_BAD_SHAPE;
    if (p.batch > LS_MAX_BATCH || p.heads > 65535) return LS_ERR_TOO_LARGE;
    if (p.n_rep > kRP) return LS_ERR_UNSUPPORTED;
    if ((reinterpret_cast<uintptr_t>(p.q) & 15) || (p.sq_b % 8) || (p.sq_h % 8) || (p.sq_m % 8))
        return LS_ERR_MISALIGNED;
    if (p.out && ((reinterpret_cast<uintptr_t>(p.out) & 7) || (p.so_b % 4) || (p.so_h % 4) || (p.so_m % 4)))
        return LS_ERR_MISALIGNED;
    return LS_OK;
}

template <class State, int MODE, int STAGES>
static int launch_decode(const DecodeParams& p, cudaStream_t stream, bool programmatic = false,
                         const TmaMaps* maps = nullptr) {
    static const TmaMaps no_maps = {};
    const size_t smem = (size_t)kWarps * STAGES * State::Pool::STAGE_BYTES + kWarps * STAGES * 8 +
                        sizeof(float) * ((size_t)kWarps * p.n_rep * kMergeStride + 2 * kWarps * kRP) +
                        sizeof(int) * ((size_t)kWarps + 1 + p.batch + 1);
    auto kern = decode_kernel<State, MODE, STAGES>;
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
    e = cudaLaunchKernelEx(&cfg, kern, p, maps ? *maps : no_maps);
    if (e != cudaSuccess) return (int)e;
    return (int)cudaGetLastError();
}

}  // namespace ls

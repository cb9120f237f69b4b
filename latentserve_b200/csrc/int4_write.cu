// Writing into the 4-bit KV cache, and reading it back (record layout: int4_page.cuh).
//
//   ls_int4_write          new K / V rows of a decode step or a prompt, quantised into the pages
//   ls_int4_read           a window of positions of each sequence expanded to fp16 rows
//   ls_rope_append_int4    a decode step's RoPE of q and k, with k and v quantised and appended
//
// Mathematics: int4_page.cuh. A token's K and V row of a head are 512 B of fp16 and 128 + 8 G B of
// record. Measured on 8 sequences x 8197 tokens x 8 heads, groups of 32: reading back 59 us (5.9
// TB/s of the measured 6.5; memory bound), writing 82 us (4.3 TB/s): the quantiser's instructions
// bound it, 532 a warp for eight rows, issue slots 80 % used (both together, with a division per
// channel and the page put together in shared memory: 412 us; now 139).
#include "int4_page.cuh"

namespace ls {

constexpr int kWriteThreads = 128;

struct Int4Rows {
    const int* block_tables;
    const int* seq_lens;
    int heads, max_pages, num_blocks, tokens;
    long long sp_b, sp_h;                  // pool strides, bytes
};

// grid (pages a window of `tokens` positions can touch, H, B), one page of one head per CTA: two
// warps have its K rows, two its V rows (page_token). The last new_lens[b] (or `tokens`) positions of
// sequence b, [L - m, L), are written from rows 0 .. m - 1. Of a page that the new rows cover whole
// every store fills 32-byte sectors, straight from registers (through shared memory it was a barrier
// more and no faster); of any other page only the new tokens' own bytes are stored.
template <int G>
__global__ void __launch_bounds__(kWriteThreads)
int4_write_kernel(const __half* __restrict__ k, const __half* __restrict__ v, uint8_t* __restrict__ pool,
                  const int* __restrict__ new_lens, Int4Rows r, long long sk_b, long long sk_h, long long sk_t,
                  long long sv_b, long long sv_h, long long sv_t) {
    const int h = blockIdx.y, b = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int len = r.seq_lens[b];
    const int m = new_lens != nullptr ? min(max(new_lens[b], 0), r.tokens) : r.tokens;
    const int start = len - m;                           // position of row 0; may be negative
    const int first = max(start, 0);
    const int page = first / LS_PAGE + blockIdx.x;
    if (page >= r.max_pages || (long long)page * LS_PAGE >= len) return;
    const int blk = r.block_tables[(long long)b * r.max_pages + page];
    const int t0 = max(first - page * LS_PAGE, 0), t1 = min(len - page * LS_PAGE, LS_PAGE);
    const __half* src = (warp < 2 ? k + b * sk_b + h * sk_h : v + b * sv_b + h * sv_h) + (lane & 15) * 8;
    const long long st = warp < 2 ? sk_t : sv_t, row0 = (long long)page * LS_PAGE - start;
    const bool there = blk >= 0 && blk < r.num_blocks;   // never write outside the pool
    uint8_t* rec = pool + blk * r.sp_b + h * r.sp_h;
    if (t0 == 0 && t1 == LS_PAGE) {
        uint4 raw[4];
        src += (row0 + page_token(warp, lane, 0)) * st;
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[i] = *reinterpret_cast<const uint4*>(src + (page_token(warp, 0, i) - page_token(warp, 0, 0)) * st);
        if (there) int4_put_page<G>(rec, raw, warp, lane);
        return;
    }
    if (!there) return;
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
        const int t = page_token(warp, lane, i);
        const bool mine = t >= t0 && t < t1;
        if (!__any_sync(LS_FULL_MASK, mine)) continue;
        uint4 raw = make_uint4(0, 0, 0, 0);
        if (mine) raw = *reinterpret_cast<const uint4*>(src + (row0 + t) * st);
        const Int4Fit fit = int4_fit<G>(raw);
        const uint32_t bytes = int4_v_bytes(fit.codes, lane & 1);
        if (!mine) continue;
        if (warp < 2) int4_put_k<G>(rec, t, fit, lane & 15);
        else int4_put_v<G>(rec, t, fit, bytes, lane & 15);
    }
}

// grid as above for the window [start[b], start[b] + tokens). Rows at or past the sequence's
// end, or of a page whose block id is outside the pool, are zeros.
template <int G>
__global__ void __launch_bounds__(kWriteThreads)
int4_read_kernel(const uint8_t* __restrict__ pool, __half* __restrict__ k, __half* __restrict__ v,
                 const int* __restrict__ starts, Int4Rows r, long long sk_b, long long sk_h, long long sk_t,
                 long long sv_b, long long sv_h, long long sv_t) {
    const int h = blockIdx.y, b = blockIdx.z;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int len = r.seq_lens[b];
    const int start = starts != nullptr ? max(starts[b], 0) : 0;
    const int page = start / LS_PAGE + blockIdx.x;
    int blk = -1;
    if ((long long)page * LS_PAGE < len && page < r.max_pages) blk = r.block_tables[(long long)b * r.max_pages + page];
    const bool there = blk >= 0 && blk < r.num_blocks;
    uint4 out[4] = {};
    if (there) int4_get_page<G>(pool + blk * r.sp_b + h * r.sp_h, warp, lane, out);
    __half* dst = (warp < 2 ? k + b * sk_b + h * sk_h : v + b * sv_b + h * sv_h) + (lane & 15) * 8;
    const long long st = warp < 2 ? sk_t : sv_t, row0 = (long long)page * LS_PAGE - start;
    const int end = there ? min(len - page * LS_PAGE, LS_PAGE) : 0;      // tokens of the page that exist
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int t = page_token(warp, lane, i);
        if (row0 + t < 0 || row0 + t >= r.tokens) continue;
        *reinterpret_cast<uint4*>(dst + (row0 + t) * st) = t < end ? out[i] : make_uint4(0, 0, 0, 0);
    }
}

__device__ __forceinline__ float round_half(float x) { return __half2float(__float2half_rn(x)); }

// grid (ceil(B * (HQ + HK) / 4)), block 128. One warp per query head (rotated into q_out), and
// one per KV head: lanes 0-15 hold the K row (rotated), 16-31 the V row, both put into the
// page of flat slot slots[b]. The rotation rounds to fp16 where ls_rope_append_fp16 does.
template <int G>
__global__ void __launch_bounds__(128)
rope_append_int4_kernel(const __half* __restrict__ qkv, const __half* __restrict__ cos_t,
                        const __half* __restrict__ sin_t, const long long* __restrict__ positions,
                        const long long* __restrict__ slots, __half* __restrict__ q_out,
                        uint8_t* __restrict__ pool, int batch, int hq, int hk, long long max_pos,
                        long long num_blocks, long long s_qkv, long long s_cos, long long sq_b, long long sp_b,
                        long long sp_h) {
    asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");   // let a programmatic successor start its prologue
    const int heads = hq + hk;
    const int item = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (item >= batch * heads) return;
    const int b = item / heads, head = item % heads;
    const long long pos = positions[b];
    if (pos < 0 || pos >= max_pos) return;
    // A query head spans 16 lanes as well: the upper half of the warp repeats the lower one's work.
    const int hl = lane & 15;
    const bool is_q = head < hq, is_v = !is_q && lane >= 16;
    const int src_head = is_q ? head : (is_v ? head + hk : head);
    uint4 raw = *reinterpret_cast<const uint4*>(qkv + b * s_qkv + (long long)src_head * LS_HEAD_DIM + hl * 8);
    uint4 mate;                                          // the channels 64 away, eight lanes over
    mate.x = __shfl_xor_sync(LS_FULL_MASK, raw.x, 8);
    mate.y = __shfl_xor_sync(LS_FULL_MASK, raw.y, 8);
    mate.z = __shfl_xor_sync(LS_FULL_MASK, raw.z, 8);
    mate.w = __shfl_xor_sync(LS_FULL_MASK, raw.w, 8);
    if (!is_v) {
        const uint4 cr = *reinterpret_cast<const uint4*>(cos_t + pos * s_cos + hl * 8);
        const uint4 sr = *reinterpret_cast<const uint4*>(sin_t + pos * s_cos + hl * 8);
        __half* x = reinterpret_cast<__half*>(&raw);
        const __half* y = reinterpret_cast<const __half*>(&mate);
        const __half* c = reinterpret_cast<const __half*>(&cr);
        const __half* s = reinterpret_cast<const __half*>(&sr);
        const float sign = hl < 8 ? -1.f : 1.f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x[i] = __float2half_rn(round_half(__half2float(x[i]) * __half2float(c[i])) +
                                   sign * round_half(__half2float(y[i]) * __half2float(s[i])));
    }
    if (is_q) {
        if (lane < 16) *reinterpret_cast<uint4*>(q_out + b * sq_b + (long long)head * LS_HEAD_DIM + hl * 8) = raw;
        return;
    }
    const long long slot = slots[b];
    if (slot < 0 || slot >= num_blocks * LS_PAGE) return;
    int4_put_token<G>(pool + (slot / LS_PAGE) * sp_b + (head - hq) * sp_h, (int)(slot % LS_PAGE), raw, lane);
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

static int check_int4_pool(const void* pool, int groups, int64_t sp_b, int64_t sp_h) {
    if (!pool) return LS_ERR_NULL_POINTER;
    if (groups != 1 && groups != 2 && groups != 4) return LS_ERR_UNSUPPORTED;
    if (!aligned16(pool) || (sp_b % 16) || (sp_h % 16)) return LS_ERR_MISALIGNED;
    if (sp_h < int4_record_bytes(groups) || sp_b < int4_record_bytes(groups)) return LS_ERR_BAD_STRIDE;
    return LS_OK;
}

static int check_rows(const void* k, const void* v, int batch, int heads, int tokens, int max_pages, int num_blocks,
                      int64_t sk_b, int64_t sk_h, int64_t sk_t, int64_t sv_b, int64_t sv_h, int64_t sv_t) {
    if (!k || !v) return LS_ERR_NULL_POINTER;
    if (batch <= 0 || heads <= 0 || tokens <= 0 || max_pages <= 0 || num_blocks <= 0) return LS_ERR_BAD_SHAPE;
    if (batch > 65535 || heads > 65535 || tokens > (1 << 30)) return LS_ERR_TOO_LARGE;
    if (!aligned16(k) || !aligned16(v) || (sk_b % 8) || (sk_h % 8) || (sk_t % 8) || (sv_b % 8) || (sv_h % 8) || (sv_t % 8))
        return LS_ERR_MISALIGNED;
    return LS_OK;
}

}  // namespace ls

extern "C" {

int ls_int4_write(const void* k, const void* v, void* pool, const int32_t* block_tables, const int32_t* seq_lens,
                  const int32_t* new_lens, int batch, int kv_heads, int tokens, int groups, int head_dim, int page,
                  int max_pages, int num_blocks, int64_t sk_b, int64_t sk_h, int64_t sk_t, int64_t sv_b, int64_t sv_h,
                  int64_t sv_t, int64_t sp_b, int64_t sp_h, void* stream) {
    if (head_dim != LS_HEAD_DIM || page != LS_PAGE) return LS_ERR_UNSUPPORTED;
    if (!block_tables || !seq_lens) return LS_ERR_NULL_POINTER;
    int rc = ls::check_int4_pool(pool, groups, sp_b, sp_h);
    if (rc == LS_OK)
        rc = ls::check_rows(k, v, batch, kv_heads, tokens, max_pages, num_blocks, sk_b, sk_h, sk_t, sv_b, sv_h, sv_t);
    if (rc != LS_OK) return rc;
    const ls::Int4Rows r = {block_tables, seq_lens, kv_heads, max_pages, num_blocks, tokens, sp_b, sp_h};
    auto kern = groups == 4 ? ls::int4_write_kernel<4> : groups == 2 ? ls::int4_write_kernel<2> : ls::int4_write_kernel<1>;
    const dim3 grid((tokens + 2 * LS_PAGE - 2) / LS_PAGE, kv_heads, batch);
    kern<<<grid, ls::kWriteThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const __half*>(k), static_cast<const __half*>(v), static_cast<uint8_t*>(pool), new_lens, r, sk_b, sk_h,
        sk_t, sv_b, sv_h, sv_t);
    return (int)cudaGetLastError();
}

int ls_int4_read(const void* pool, void* k, void* v, const int32_t* block_tables, const int32_t* seq_lens,
                 const int32_t* start, int batch, int kv_heads, int tokens, int groups, int head_dim, int page,
                 int max_pages, int num_blocks, int64_t sk_b, int64_t sk_h, int64_t sk_t, int64_t sv_b, int64_t sv_h,
                 int64_t sv_t, int64_t sp_b, int64_t sp_h, void* stream) {
    if (head_dim != LS_HEAD_DIM || page != LS_PAGE) return LS_ERR_UNSUPPORTED;
    if (!block_tables || !seq_lens) return LS_ERR_NULL_POINTER;
    int rc = ls::check_int4_pool(pool, groups, sp_b, sp_h);
    if (rc == LS_OK)
        rc = ls::check_rows(k, v, batch, kv_heads, tokens, max_pages, num_blocks, sk_b, sk_h, sk_t, sv_b, sv_h, sv_t);
    if (rc != LS_OK) return rc;
    const ls::Int4Rows r = {block_tables, seq_lens, kv_heads, max_pages, num_blocks, tokens, sp_b, sp_h};
    auto kern = groups == 4 ? ls::int4_read_kernel<4> : groups == 2 ? ls::int4_read_kernel<2> : ls::int4_read_kernel<1>;
    // A window that starts at a page boundary touches one page less than one that does not.
    const dim3 grid((tokens + (start ? 2 * LS_PAGE - 2 : LS_PAGE - 1)) / LS_PAGE, kv_heads, batch);
    kern<<<grid, ls::kWriteThreads, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const uint8_t*>(pool), static_cast<__half*>(k), static_cast<__half*>(v), start, r, sk_b, sk_h, sk_t,
        sv_b, sv_h, sv_t);
    return (int)cudaGetLastError();
}

int ls_rope_append_int4(const void* qkv, const void* cos, const void* sin, const int64_t* positions,
                        const int64_t* slots, void* q_out, void* pool, int batch, int q_heads, int kv_heads, int groups,
                        int head_dim, int page, int64_t max_pos, int64_t num_blocks, int64_t s_qkv, int64_t s_cos,
                        int64_t sq_b, int64_t sp_b, int64_t sp_h, void* stream) {
    if (!qkv || !cos || !sin || !positions || !slots || !q_out) return LS_ERR_NULL_POINTER;
    if (head_dim != LS_HEAD_DIM || page != LS_PAGE) return LS_ERR_UNSUPPORTED;
    if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || max_pos <= 0 || num_blocks <= 0) return LS_ERR_BAD_SHAPE;
    if ((int64_t)batch * (q_heads + kv_heads) > (1 << 30)) return LS_ERR_TOO_LARGE;
    const int rc = ls::check_int4_pool(pool, groups, sp_b, sp_h);
    if (rc != LS_OK) return rc;
    if (!ls::aligned16(qkv) || !ls::aligned16(cos) || !ls::aligned16(sin) || !ls::aligned16(q_out) || (s_qkv % 8) ||
        (s_cos % 8) || (sq_b % 8))
        return LS_ERR_MISALIGNED;
    auto kern = groups == 4   ? ls::rope_append_int4_kernel<4>
                : groups == 2 ? ls::rope_append_int4_kernel<2>
                              : ls::rope_append_int4_kernel<1>;
    const int items = batch * (q_heads + kv_heads);
    kern<<<(items + 3) / 4, 128, 0, static_cast<cudaStream_t>(stream)>>>(
        static_cast<const __half*>(qkv), static_cast<const __half*>(cos), static_cast<const __half*>(sin),
        reinterpret_cast<const long long*>(positions), reinterpret_cast<const long long*>(slots),
        static_cast<__half*>(q_out), static_cast<uint8_t*>(pool), batch, q_heads, kv_heads, max_pos, num_blocks, s_qkv,
        s_cos, sq_b, sp_b, sp_h);
    return (int)cudaGetLastError();
}

}  // extern "C"

// Copying pages inside the pools of a cache: pool[dst[i]] = pool[src[i]] for every pool, all
// layers, one launch. What forking a sequence (its partly filled last page) and compacting a
// pool (live pages moved to the lowest ids) do on the device.
//
// Plain bytes, bound by memory: each byte is read and written once. The page ids and the pools'
// addresses travel in the kernel's parameters (up to 32 KB), so a call needs no staging buffer,
// no host-to-device copy and no lifetime of either. 512 pages of 8 KB in 56 pools: 74 us (6.3 TB/s
// of the measured 6.5); three pages: 4.2 us, the launch.
#include <stdlib.h>

#include "ls_common.cuh"
#include "../../include/latentserve_b200.h"

namespace ls {

constexpr int kCopyThreads = 128;
constexpr int kCopyPiece = kCopyThreads * 64;      // bytes a CTA moves: four 16-byte loads a thread in flight
constexpr int kCopyPools = 64;

struct CopyPool {
    uint8_t* base;
    long long layer_stride, page_stride;
    int bytes, layers;
};

template <int PAIRS>
struct CopyArgs {
    CopyPool pool[kCopyPools];
    int2 pair[PAIRS];                              // src, dst
    int pieces;                                    // grid.x = pairs x pieces; grid.y = all pools' layers
};

// Whole units of W bytes: 16, or 4 / 1 where a pool's addresses or sizes are not multiples of 16.
template <class W>
__device__ __forceinline__ void copy_piece(uint8_t* dst, const uint8_t* src, int bytes) {
    const int n = bytes / (int)sizeof(W);
    for (int at = threadIdx.x; at < n; at += 4 * kCopyThreads) {
        W v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (at + i * kCopyThreads < n) v[i] = reinterpret_cast<const W*>(src)[at + i * kCopyThreads];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (at + i * kCopyThreads < n) reinterpret_cast<W*>(dst)[at + i * kCopyThreads] = v[i];
    }
}

template <int PAIRS>
__global__ void __launch_bounds__(kCopyThreads)
copy_pages_kernel(const __grid_constant__ CopyArgs<PAIRS> a) {
    const int pair = blockIdx.x / a.pieces, piece = blockIdx.x % a.pieces;
    int layer = blockIdx.y, which = 0;
    while (layer >= a.pool[which].layers) layer -= a.pool[which++].layers;      // grid.y = sum of the layers: ends
    const CopyPool& p = a.pool[which];
    const int at = piece * kCopyPiece;
    if (at >= p.bytes) return;
    const int bytes = min(kCopyPiece, p.bytes - at);
    uint8_t* base = p.base + layer * p.layer_stride + at;
    const uint8_t* src = base + a.pair[pair].x * p.page_stride;
    uint8_t* dst = base + a.pair[pair].y * p.page_stride;
    const unsigned odd = (unsigned)(reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst)) | (unsigned)bytes;
    if (!(odd & 15)) copy_piece<uint4>(dst, src, bytes);
    else if (!(odd & 3)) copy_piece<uint32_t>(dst, src, bytes);
    else copy_piece<uint8_t>(dst, src, bytes);
}

template <int PAIRS>
static int launch_copies(CopyArgs<PAIRS>& a, const int32_t* src, const int32_t* dst, int count, int layers, int pieces,
                         cudaStream_t stream) {
    a.pieces = pieces;
    for (int done = 0; done < count; done += PAIRS) {
        const int n = count - done < PAIRS ? count - done : PAIRS;
        for (int i = 0; i < n; ++i) a.pair[i] = make_int2(src[done + i], dst[done + i]);
        copy_pages_kernel<PAIRS><<<dim3(n * pieces, layers), kCopyThreads, 0, stream>>>(a);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return (int)e;
    }
    return LS_OK;
}

// Every id inside the pool; no page written twice, none both read and written.
static int check_pairs(const int32_t* src, const int32_t* dst, int count, int num_blocks) {
    for (int i = 0; i < count; ++i)
        if (src[i] < 0 || src[i] >= num_blocks || dst[i] < 0 || dst[i] >= num_blocks) return LS_ERR_PAGE_ID;
    unsigned char* written = static_cast<unsigned char*>(calloc((size_t)num_blocks / 8 + 1, 1));
    if (written == nullptr) return (int)cudaErrorMemoryAllocation;
    int rc = LS_OK;
    for (int i = 0; i < count && rc == LS_OK; ++i) {
        unsigned char& byte = written[dst[i] / 8];
        if (byte & (1 << (dst[i] % 8))) rc = LS_ERR_OVERLAP;
        byte |= (unsigned char)(1 << (dst[i] % 8));
    }
    for (int i = 0; i < count && rc == LS_OK; ++i)
        if (written[src[i] / 8] & (1 << (src[i] % 8))) rc = LS_ERR_OVERLAP;
    free(written);
    return rc;
}

}  // namespace ls

extern "C" int ls_copy_pages(const ls_page_pool* pools, int num_pools, const int32_t* src, const int32_t* dst, int count,
                             int num_blocks, void* stream) {
    if (!pools || (count > 0 && (!src || !dst))) return LS_ERR_NULL_POINTER;
    if (num_pools <= 0 || count < 0 || num_blocks <= 0) return LS_ERR_BAD_SHAPE;
    for (int i = 0; i < num_pools; ++i) {
        if (!pools[i].base) return LS_ERR_NULL_POINTER;
        if (pools[i].page_bytes <= 0 || pools[i].layers <= 0) return LS_ERR_BAD_SHAPE;
        if (pools[i].page_bytes > (1 << 24) || pools[i].layers > 65535) return LS_ERR_TOO_LARGE;
        if (pools[i].page_stride < pools[i].page_bytes || (pools[i].layers > 1 && pools[i].layer_stride < pools[i].page_bytes))
            return LS_ERR_BAD_STRIDE;
    }
    const int rc = ls::check_pairs(src, dst, count, num_blocks);
    if (rc != LS_OK || count == 0) return rc;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    // Few pairs: the small parameter block (a launch copies all of it).
    ls::CopyArgs<128> few;
    ls::CopyArgs<3584> many;
    static_assert(sizeof(many) <= 32764, "kernel parameters end at 32 764 bytes");
    for (int first = 0; first < num_pools;) {
        int n = 0, layers = 0, pieces = 1;
        ls::CopyPool* to = count <= 128 ? few.pool : many.pool;
        while (first + n < num_pools && n < ls::kCopyPools && layers + pools[first + n].layers <= 65535) {
            const ls_page_pool& p = pools[first + n];
            to[n] = {static_cast<uint8_t*>(p.base), p.layer_stride, p.page_stride, p.page_bytes, p.layers};
            const int need = (p.page_bytes + ls::kCopyPiece - 1) / ls::kCopyPiece;
            pieces = need > pieces ? need : pieces;
            layers += p.layers;
            ++n;
        }
        const int e = count <= 128 ? ls::launch_copies(few, src, dst, count, layers, pieces, s)
                                   : ls::launch_copies(many, src, dst, count, layers, pieces, s);
        if (e != LS_OK) return e;
        first += n;
    }
    return LS_OK;
}

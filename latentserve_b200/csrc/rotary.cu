// Rotary positions for queries and keys, out of place or in place.
//
//   (a, b) -> (a cos - b sin, b cos + a sin), pair i < rot / 2 of a head being channels
//   (i, i + rot / 2) in the half layout and (2 i, 2 i + 1) in the interleaved one; channels past
//   `rot` are copied. cos / sin come from fp32 tables [max_pos, rot / 2] (made in 64 bits by the
//   caller: a far position times a frequency has no room in 32), arithmetic is fp32, one
//   rounding to the tensor's type at the end.
//
// Bound by memory: each element is read and written once. A thread owns 16 bytes of the same channels in
// up to kHeads heads of one token, so that a token's table row is read once for several heads.
#include <cuda_bf16.h>

#include "ls_common.cuh"

namespace ls {

struct RotaryArgs {
    const void* x[2];                  // queries, keys
    void* y[2];
    long long sx_t[2], sx_h[2], sy_t[2], sy_h[2];
    int heads[2];
    const float* cos_t;
    const float* sin_t;
    const long long* positions;
    long long max_pos, s_tab;
    int tokens, dim, rot, splits;      // splits: threads that share a token's heads
    float sign;                        // -1: the inverse rotation
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

constexpr int kRotaryThreads = 256;

// V channels of one run in registers: 16 bytes, or a single channel where rows are not aligned for that.
template <class T, int V>
struct alignas(V * sizeof(T)) Run {
    T v[V];
};

// Rows are read and written once: past L1, which the tables' rows are better left in.
template <class T, int V>
__device__ __forceinline__ Run<T, V> load_run(const T* p) {
    Run<T, V> r;
    if constexpr (sizeof(r) == 16) {
        uint4 x;
        asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];\n" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w) : "l"(p));
        r = *reinterpret_cast<Run<T, V>*>(&x);
    } else {
        r.v[0] = *p;
    }
    return r;
}

template <int V>
__device__ __forceinline__ void load_angles(const float* p, float (&out)[V]) {
    if constexpr (V % 4 == 0) {
#pragma unroll
        for (int k = 0; k < V; k += 4) {
            const float4 x = *reinterpret_cast<const float4*>(p + k);
            out[k] = x.x; out[k + 1] = x.y; out[k + 2] = x.z; out[k + 3] = x.w;
        }
    } else {
        out[0] = *p;
    }
}

// Two neighbouring channels at once where the type packs them.
__device__ __forceinline__ void store2(float* d, float a, float b) { d[0] = a; d[1] = b; }
__device__ __forceinline__ void store2(__half* d, float a, float b) { *reinterpret_cast<__half2*>(d) = __floats2half2_rn(a, b); }
__device__ __forceinline__ void store2(__nv_bfloat16* d, float a, float b) {
    *reinterpret_cast<__nv_bfloat162*>(d) = __floats2bfloat162_rn(a, b);
}

// UNIT = what one thread owns of a head: in the half layout a run of V channels and the run rot / 2
// further on; interleaved two neighbouring runs; or a run of the channels that are not rotated.
template <class T, int V, bool INTERLEAVED, int HEADS>
__global__ void __launch_bounds__(kRotaryThreads, 5)
rotary_kernel(const __grid_constant__ RotaryArgs a) {
    using R = Run<T, V>;
    const unsigned rot_units = a.rot / 2 / V, units = rot_units + (a.dim - a.rot) / V;
    const unsigned idx = blockIdx.x * kRotaryThreads + threadIdx.x;
    const unsigned rest = idx / units, unit = idx - rest * units;
    const unsigned tok = rest / a.splits, split = rest - tok * a.splits;
    if (tok >= (unsigned)a.tokens) return;
    const long long pos = a.positions[tok];
    const bool turn = unit < rot_units;
    const int c0 = turn ? (INTERLEAVED ? 2 * V : V) * unit : a.rot + V * (unit - rot_units);
    const int c1 = turn ? (INTERLEAVED ? c0 + V : c0 + a.rot / 2) : c0;
    const int total = a.heads[0] + a.heads[1];
    R lo[HEADS], hi[HEADS];
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        const int head = split + i * a.splits;
        if (head >= total) continue;
        const int w = head >= a.heads[0];
        const T* src = static_cast<const T*>(a.x[w]) + tok * a.sx_t[w] + (head - (w ? a.heads[0] : 0)) * a.sx_h[w];
        lo[i] = load_run<T, V>(src + c0);
        if (turn) hi[i] = load_run<T, V>(src + c1);
    }
    if (turn) {
        const bool known = pos >= 0 && pos < a.max_pos;
        float c[V], s[V];
        load_angles<V>(a.cos_t + (known ? pos : 0) * a.s_tab + V * unit, c);
        load_angles<V>(a.sin_t + (known ? pos : 0) * a.s_tab + V * unit, s);
        // A position that the tables do not have comes out as NaN.
        const float mul = known ? a.sign : __int_as_float(0x7fffffff);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            s[k] *= mul;
            if (!known) c[k] = mul;
        }
#pragma unroll
        for (int i = 0; i < HEADS; ++i) {
            T* const u = lo[i].v;
            T* const v = hi[i].v;
            if constexpr (V == 1) {
                const float p = to_f(u[0]), q = to_f(v[0]);
                u[0] = from_f<T>(p * c[0] - q * s[0]);
                v[0] = from_f<T>(q * c[0] + p * s[0]);
            } else if constexpr (INTERLEAVED) {
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    T* const at = 2 * k < V ? u + 2 * k : v + (2 * k - V);
                    const float p = to_f(at[0]), q = to_f(at[1]);
                    store2(at, p * c[k] - q * s[k], q * c[k] + p * s[k]);
                }
            } else {
#pragma unroll
                for (int k = 0; k < V; k += 2) {
                    const float p0 = to_f(u[k]), p1 = to_f(u[k + 1]), q0 = to_f(v[k]), q1 = to_f(v[k + 1]);
                    store2(u + k, p0 * c[k] - q0 * s[k], p1 * c[k + 1] - q1 * s[k + 1]);
                    store2(v + k, q0 * c[k] + p0 * s[k], q1 * c[k + 1] + p1 * s[k + 1]);
                }
            }
        }
    }
#pragma unroll
    for (int i = 0; i < HEADS; ++i) {
        const int head = split + i * a.splits;
        if (head >= total) continue;
        const int w = head >= a.heads[0];
        T* dst = static_cast<T*>(a.y[w]) + tok * a.sy_t[w] + (head - (w ? a.heads[0] : 0)) * a.sy_h[w];
        *reinterpret_cast<R*>(dst + c0) = lo[i];
        if (turn) *reinterpret_cast<R*>(dst + c1) = hi[i];
    }
}

template <class T, int V, int HEADS>
static int launch_rotary(const RotaryArgs& a, bool interleaved, cudaStream_t stream) {
    const long long units = a.rot / 2 / V + (a.dim - a.rot) / V;
    const long long threads = units * a.splits * a.tokens;
    if (threads > 0x7fffff00LL) return LS_ERR_TOO_LARGE;
    const unsigned grid = (unsigned)((threads + kRotaryThreads - 1) / kRotaryThreads);
    if (interleaved) rotary_kernel<T, V, true, HEADS><<<grid, kRotaryThreads, 0, stream>>>(a);
    else rotary_kernel<T, V, false, HEADS><<<grid, kRotaryThreads, 0, stream>>>(a);
    return (int)cudaGetLastError();
}

// Two heads a thread and five blocks an SM: 32 768 tokens x 40 heads of bf16 in 119 us (5.8 TB/s of the
// measured 6.5); one head 131 us, four heads (fewer threads fit) 123 us, streaming stores no better.
constexpr int kHeads = 2;

template <class T>
static int run_rotary(RotaryArgs& a, bool interleaved, cudaStream_t stream) {
    constexpr int V = 16 / sizeof(T);
    bool wide = (a.rot / 2) % V == 0 && (a.dim - a.rot) % V == 0 && a.s_tab % 4 == 0 &&
                !((reinterpret_cast<uintptr_t>(a.cos_t) | reinterpret_cast<uintptr_t>(a.sin_t)) & 15);
    for (int w = 0; w < 2; ++w)
        if (a.heads[w])
            wide = wide && !(reinterpret_cast<uintptr_t>(a.x[w]) & 15) && !(reinterpret_cast<uintptr_t>(a.y[w]) & 15) &&
                   a.sx_t[w] % V == 0 && a.sx_h[w] % V == 0 && a.sy_t[w] % V == 0 && a.sy_h[w] % V == 0;
    const int total = a.heads[0] + a.heads[1];
    const long long units = wide ? a.rot / 2 / V + (a.dim - a.rot) / V : a.dim - a.rot / 2;
    // Several heads a thread once there are threads enough to fill the GPU all the same.
    const bool many = units * a.tokens * total >= (long long)kHeads * 148 * 2048;
    a.splits = many ? (total + kHeads - 1) / kHeads : total;
    if (wide)
        return many ? launch_rotary<T, V, kHeads>(a, interleaved, stream) : launch_rotary<T, V, 1>(a, interleaved, stream);
    a.splits = total;
    return launch_rotary<T, 1, 1>(a, interleaved, stream);
}

}  // namespace ls

extern "C" int ls_rotary(const void* q, const void* k, void* q_out, void* k_out, const float* cos, const float* sin,
                         const int64_t* positions, int tokens, int q_heads, int k_heads, int dim, int rot, int dtype,
                         int interleaved, int inverse, int64_t max_pos, int64_t s_tab, int64_t sq_t, int64_t sq_h,
                         int64_t sk_t, int64_t sk_h, int64_t sqo_t, int64_t sqo_h, int64_t sko_t, int64_t sko_h,
                         void* stream) {
    if (!cos || !sin || !positions || (q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out))) return LS_ERR_NULL_POINTER;
    if (tokens <= 0 || q_heads < 0 || k_heads < 0 || q_heads + (int64_t)k_heads <= 0 || max_pos <= 0) return LS_ERR_BAD_SHAPE;
    if (dim <= 0 || rot <= 0 || rot > dim || rot % 2 || s_tab < rot / 2) return LS_ERR_BAD_SHAPE;
    if (dim > 65536 || q_heads > 65536 || k_heads > 65536) return LS_ERR_TOO_LARGE;
    ls::RotaryArgs a = {};
    a.x[0] = q; a.x[1] = k;
    a.y[0] = q_out; a.y[1] = k_out;
    a.sx_t[0] = sq_t; a.sx_h[0] = sq_h; a.sx_t[1] = sk_t; a.sx_h[1] = sk_h;
    a.sy_t[0] = sqo_t; a.sy_h[0] = sqo_h; a.sy_t[1] = sko_t; a.sy_h[1] = sko_h;
    a.heads[0] = q_heads; a.heads[1] = k_heads;
    a.cos_t = cos; a.sin_t = sin;
    a.positions = reinterpret_cast<const long long*>(positions);
    a.max_pos = max_pos; a.s_tab = s_tab;
    a.tokens = tokens; a.dim = dim; a.rot = rot;
    a.sign = inverse ? -1.f : 1.f;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == 0) return ls::run_rotary<__half>(a, interleaved != 0, s);
    if (dtype == 1) return ls::run_rotary<__nv_bfloat16>(a, interleaved != 0, s);
    if (dtype == 2) return ls::run_rotary<float>(a, interleaved != 0, s);
    return LS_ERR_UNSUPPORTED;
}

// hx_readout.cuh -- building blocks of the readout-row kernels: element types,
// teams of threads that own a row, the row in shared memory.
//
// A row is worked on by a team: one warp (several rows per block), one block,
// or a cluster of blocks that share the row in equal slices.  Each member block
// keeps its slice in shared memory, so that a row is read from memory once
// whatever the number of passes over it.
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "heliox_b200.h"

namespace hxr {

namespace cg = cooperative_groups;

// Order-preserving integer keys (equal values, +0 and -0 among them, have equal keys).
__device__ __forceinline__ unsigned long long key_of(double x) {
    const unsigned long long b = (unsigned long long)__double_as_longlong(x + 0.0);
    return b ^ ((b >> 63) ? ~0ull : 0x8000000000000000ull);
}
__device__ __forceinline__ double value_of(unsigned long long k) {
    return __longlong_as_double((long long)(k ^ ((k >> 63) ? 0x8000000000000000ull : ~0ull)));
}
__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned b = __float_as_uint(x + 0.0f);
    return b ^ ((b >> 31) ? ~0u : 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : ~0u)); }

// Element type -> compute and statistics type W, key type K, elements of a 16-byte vector.
template <typename T>
struct Ty {  // float, __half, __nv_bfloat16
    using W = float;
    using K = unsigned;
    static constexpr int VEC = 16 / (int)sizeof(T);
};
template <>
struct Ty<double> {
    using W = double;
    using K = unsigned long long;
    static constexpr int VEC = 2;
};

__device__ __forceinline__ double wide(double x) { return x; }
__device__ __forceinline__ float wide(float x) { return x; }
__device__ __forceinline__ float wide(__half x) { return __half2float(x); }
__device__ __forceinline__ float wide(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T narrow(typename Ty<T>::W v);
template <>
__device__ __forceinline__ double narrow<double>(double v) { return v; }
template <>
__device__ __forceinline__ float narrow<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T>
struct alignas(16) Vec {
    T e[Ty<T>::VEC];
};

__device__ __forceinline__ double load_any(const void* p, int dtype, size_t i) {
    switch (dtype) {
        case HX_DT_F64: return ((const double*)p)[i];
        case HX_DT_F32: return (double)((const float*)p)[i];
        case HX_DT_F16: return (double)__half2float(((const __half*)p)[i]);
        default: return (double)__bfloat162float(((const __nv_bfloat16*)p)[i]);
    }
}

// exp(d / T) for d <= 0: fp64 by the library's exp, fp32 by the hardware's 2^x
// (about 2 steps of 2^-23; results below 2^-126 are 0).
struct Scaler64 {
    double inv;
    __device__ explicit Scaler64(double temperature) : inv(1.0 / temperature) {}
    __device__ __forceinline__ double operator()(double d) const { return exp(d * inv); }
};
struct Scaler32 {
    float inv;
    __device__ explicit Scaler32(double temperature) : inv((float)(1.4426950408889634 / temperature)) {}
    __device__ __forceinline__ float operator()(float d) const {
        float r;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d * inv));
        return r;
    }
};
__device__ __forceinline__ Scaler64 scaler(double, double temperature) { return Scaler64(temperature); }
__device__ __forceinline__ Scaler32 scaler(float, double temperature) { return Scaler32(temperature); }

__device__ __forceinline__ double max_num(double a, double b) { return fmax(a, b); }  // the number, where one is NaN
__device__ __forceinline__ float max_num(float a, float b) { return fmaxf(a, b); }

constexpr int kRedBytes = 2 * 16 * 32 + 2 * 32;  // two buffers of 16 warps' partials and of the block's

// The threads that own a row.  NT = 32: a warp, kWarpRows rows per block;
// otherwise a block of NT threads, CL: a cluster of such blocks.
constexpr int kWarpRows = 4;
template <int NT_, bool CL_>
struct Team {
    static constexpr int NT = NT_, NW = NT_ / 32;
    static constexpr bool CL = CL_;
    int t;            // thread within this block's part of the team
    int part, parts;  // block within the cluster
    int parity = 0, parity_all = 0;
    char* red;  // kRedBytes of shared memory

    __device__ explicit Team(char* scratch) : red(scratch) {
        t = NT == 32 ? threadIdx.x & 31 : threadIdx.x;
        part = CL ? (int)cg::this_cluster().block_rank() : 0;
        parts = CL ? (int)cg::this_cluster().num_blocks() : 1;
    }
    static __device__ __forceinline__ size_t row_of_block(int parts) {
        return NT == 32 ? (size_t)blockIdx.x * kWarpRows + (threadIdx.x >> 5) : CL ? (size_t)blockIdx.x / parts : (size_t)blockIdx.x;
    }
    __device__ __forceinline__ void sync() const {
        if constexpr (NT == 32)
            __syncwarp();
        else
            __syncthreads();
    }
    __device__ __forceinline__ void sync_all() const {
        if constexpr (CL)
            cg::this_cluster().sync();
        else
            sync();
    }
    template <typename V>
    __device__ __forceinline__ V* of(V* p, int rank) const {  // p in another member's shared memory
        if constexpr (CL) return cg::this_cluster().map_shared_rank(p, rank);
        return p;
    }
    // Reductions: butterflies within warps, then over the warps' and the
    // blocks' partials in a fixed order, so that every thread holds the same
    // bits and no timing shows.  One barrier each (two buffers in turn); all
    // threads of the block, with ALL of the cluster, take part.
    template <bool ALL, typename V, typename F>
    __device__ __forceinline__ V reduce(V v, F op) {
        static_assert(sizeof(V) <= 32, "partials are 32 bytes");
        v = warp(v, op);
        if constexpr (NW > 1) {
            char* buf = red + parity * 16 * 32;
            if ((t & 31) == 0) *(V*)(buf + (t >> 5) * 32) = v;
            __syncthreads();
            v = *(const V*)(buf + ((t & 31) % NW) * 32);
            for (int o = NW / 2; o > 0; o >>= 1) v = op(v, shfl(v, o));
        }
        if constexpr (CL && ALL) {
            V* mine = (V*)(red + 2 * 16 * 32 + parity_all * 32);
            parity_all ^= 1;
            if (t == 0) *mine = v;
            cg::this_cluster().sync();
            v = *of(mine, 0);
            for (int r = 1; r < parts; r++) v = op(v, *of(mine, r));
        }
        parity ^= 1;
        return v;
    }
    template <typename V>
    static __device__ __forceinline__ V shfl(const V& v, int o) {
        static_assert(sizeof(V) % 4 == 0, "");
        V r;
        const int* a = (const int*)&v;
        int* b = (int*)&r;
#pragma unroll
        for (int i = 0; i < (int)(sizeof(V) / 4); i++) b[i] = __shfl_xor_sync(~0u, a[i], o);
        return r;
    }
    template <typename V, typename F>
    static __device__ __forceinline__ V warp(V v, F op) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v = op(v, shfl(v, o));
        return v;
    }
    __device__ __forceinline__ bool any(bool p) const {  // of this block's part; a barrier
        if constexpr (NT == 32) {
            __syncwarp();
            return __any_sync(~0u, p);
        } else {
            return __syncthreads_or(p);
        }
    }
};

// This block's slice of a row in shared memory, in 16-byte vectors aligned as
// in global memory: element i of the slice is e[phase + i].  What the first
// and the last vector hold besides is -inf.
template <typename T>
struct Slice {
    static constexpr int VEC = Ty<T>::VEC;
    T* e;
    const T* src;
    int first;  // position of element 0 in the row
    int n, phase, nv;

    __device__ Slice(T* smem, const T* row, int ncol, int part, int parts) : e(smem) {
        const int per = (ncol + parts - 1) / parts;
        first = min(part * per, ncol);
        n = min(per, ncol - first);
        src = row + first;
        phase = n > 0 ? (int)(((size_t)src & 15) / sizeof(T)) : 0;
        nv = (phase + n + VEC - 1) / VEC;
    }
    static size_t bytes(int ncol, int parts) {  // of shared memory (host)
        const int per = (ncol + parts - 1) / parts;
        return (size_t)(per / VEC + 2) * 16;
    }
    __device__ __forceinline__ bool whole(int v) const {
        return v * VEC >= phase && (v + 1) * VEC <= phase + n;
    }
    // Starts the copy into shared memory: 16 bytes at a time, elementwise at
    // the edges, so that nothing outside the row is read.
    template <int NT>
    __device__ void load(int t) const {
        for (int v = t; v < nv; v += NT) {
            if (whole(v)) {
                const unsigned d = (unsigned)__cvta_generic_to_shared(e + v * VEC);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src + (v * VEC - phase)) : "memory");
            } else {
                for (int u = v * VEC; u < (v + 1) * VEC; u++)
                    e[u] = u >= phase && u < phase + n ? src[u - phase] : narrow<T>((typename Ty<T>::W)-INFINITY);
            }
        }
    }
    static __device__ __forceinline__ void wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }
    __device__ __forceinline__ Vec<T> get(int v) const { return *(const Vec<T>*)(e + v * VEC); }
    __device__ __forceinline__ void set(int v, const Vec<T>& x) const { *(Vec<T>*)(e + v * VEC) = x; }
    // Writes f(v)'s elements to a row of global memory, vectors where it is aligned like the source.
    template <int NT, typename F>
    __device__ void store(int t, T* row, F f) const {
        T* dst = row + first;
        const bool aligned = (((size_t)dst ^ (size_t)src) & 15) == 0;
        for (int v = t; v < nv; v += NT) {
            const Vec<T> x = f(v);
            if (aligned && whole(v)) {
                *(Vec<T>*)(dst + (v * VEC - phase)) = x;
            } else {
#pragma unroll
                for (int u = 0; u < VEC; u++) {
                    const int i = v * VEC + u - phase;
                    if (i >= 0 && i < n) dst[i] = x.e[u];
                }
            }
        }
    }
};

}  // namespace hxr

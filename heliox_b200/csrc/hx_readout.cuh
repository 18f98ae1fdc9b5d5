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

#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <type_traits>

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

// exp((x - m) / T), m a readout near the largest.
//
// fp64: the table-driven method of P. T. P. Tang (ACM TOMS 15, 1989): with
// d = x - m and s = 16 d log2(e) / T = 16 k + j + f, |f| <= 1/2, the result is
// 2^k 2^(j/16) 2^(f/16), the last factor by a polynomial through the Chebyshev
// nodes of degree 6 (relative error 1.5e-17).  The table holds 2^(j/16) less
// j 2^-4 in the exponent's place, so that one addition of the whole number
// 16 k + j puts the power of two in.  11 fp64 operations and one table entry:
// 16 doubles are one entry per pair of shared-memory banks, so lanes never
// wait for one another; 64 entries would save two operations and cost four
// more conflicts.  Below 2^-1018 it is 0; above 2^1000 it is about 2^1000, for
// NaN that (sign bit clear) or NaN, which the caller sees in the sum.
// fp32: the hardware's 2^x (about 3 half steps); results below 2^-126 are 0.
constexpr int kPowBytes = 16 * 8;
__constant__ unsigned long long kPow16[16] = {
    0x3ff0000000000000, 0x3fefb5586cf9890f, 0x3fef72b83c7d517b, 0x3fef387a6e756238, 0x3fef06fe0a31b715, 0x3feedea64c123422,
    0x3feebfdad5362a27, 0x3feeab07dd485429, 0x3feea09e667f3bcd, 0x3feea11473eb0187, 0x3feeace5422aa0db, 0x3feec49182a3f090,
    0x3feee89f995ad3ad, 0x3fef199bdd85529c, 0x3fef5818dcfba487, 0x3fefa4afa2a490da};
struct Heat {  // a temperature, worked out on the host
    double t, inv, c;  // c = 16 log2(e) / T
    int high;          // high word of the largest d that is taken as it is
    unsigned low, span;  // and of the d below which the result is 0; from there to -inf's, NaN's being beyond
    float cf;          // log2(e) / T
};
struct Scaler64 {
    double c, m, inv;
    int high;
    unsigned low, span;
    const int2* pow16;  // kPow16 in shared memory
    __device__ __forceinline__ Scaler64(const Heat& h, double m_, const char* table)
        : c(h.c), m(m_), inv(h.inv), high(h.high), low(h.low), span(h.span), pow16((const int2*)table) {}
    __device__ __forceinline__ double operator()(double x) const {
        const double d0 = x - m;
        const double d = __hiloint2double(min(__double2hiint(d0), high), __double2loint(d0));
        const double y = __fma_rn(d, c, 6755399441055744.0);  // 1.5 2^52: the sum's low bits are s to the nearest whole number
        const int k = __double2loint(y);
        const double f = __fma_rn(d, c, 6755399441055744.0 - y);
        double q = 0x1.430a1d08ec681p-37;
        q = __fma_rn(q, f, 0x1.5d897e525c216p-30);
        q = __fma_rn(q, f, 0x1.3b2ab6fb41213p-23);
        q = __fma_rn(q, f, 0x1.c6b08d6f2a289p-17);
        q = __fma_rn(q, f, 0x1.ebfbdff82c590p-11);
        q = __fma_rn(q, f, 0x1.62e42fefa39f3p-5);
        q = q * f;
        const int2 t = pow16[k & 15];
        const double p = __hiloint2double(t.y + (k << 16), t.x);
        const double e = __fma_rn(p, q, p);
        return (unsigned)__double2hiint(d) - low <= span ? 0.0 : e;
    }
    __device__ __forceinline__ double z(double x) const { return (x - m) * inv; }  // of which it is the exponential
    static constexpr double most = 0x1p500;  // a sum up to here has left no readout out
};
struct Scaler32 {
    float c, m;
    double inv;
    __device__ __forceinline__ Scaler32(const Heat& h, float m_, const char*) : c(h.cf), m(m_), inv(h.inv) {}
    __device__ __forceinline__ float operator()(float x) const {
        float r;
        asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"((x - m) * c));
        return r;
    }
    __device__ __forceinline__ double z(double x) const { return (x - (double)m) * inv; }
    static constexpr double most = 0x1p40;
};
__device__ __forceinline__ Scaler64 scaler(double m, const Heat& h, const char* table) { return Scaler64(h, m, table); }
__device__ __forceinline__ Scaler32 scaler(float m, const Heat& h, const char* table) { return Scaler32(h, m, table); }

// The larger of a and b; a where b is NaN.
__device__ __forceinline__ double larger(double a, double b) { return b > a ? b : a; }
__device__ __forceinline__ float larger(float a, float b) { return fmaxf(a, b); }

// A team's scratch: two buffers of 16 warps' partials and of the block's, the
// table of powers, numbers that one warp leaves for the others.
constexpr int kPartials = 2 * 16 * 32 + 2 * 32;
constexpr int kRedBytes = kPartials + kPowBytes + 16 * 8;

// The threads that own a row.  NT = 32: a warp, kWarpRows rows per block;
// otherwise the first NT threads of a block, CL: of each block of a cluster.
// HELP: the block has one more warp, the helper, which meets the others at
// every barrier of sync_block() and reduce().
constexpr int kWarpRows = 4;
__device__ __forceinline__ void bar_sync(int id, int n) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(n) : "memory"); }
__device__ __forceinline__ void bar_arrive(int id, int n) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(n) : "memory"); }
template <int NT_, bool CL_, bool HELP_>
struct Team {
    static constexpr int NT = NT_, NW = NT_ / 32, THREADS = NT_ + (HELP_ ? 32 : 0);
    static constexpr bool CL = CL_, HELP = HELP_;
    int t;            // thread within this block's part of the team; the helper's are NT .. NT+31
    int part, parts;  // block within the cluster
    int parity = 0, parity_all = 0;
    char* red;  // kRedBytes of shared memory

    // The table of powers is ready after the next barrier.
    __device__ explicit Team(char* scratch) : red(scratch) {
        t = NT == 32 ? threadIdx.x & 31 : threadIdx.x;
        if (t < 16) ((unsigned long long*)(red + kPartials))[t] = kPow16[t];
        part = CL ? (int)cg::this_cluster().block_rank() : 0;
        parts = CL ? (int)cg::this_cluster().num_blocks() : 1;
    }
    // rows are dealt to the teams of the grid in turn
    __device__ __forceinline__ long long first_row() const {
        return NT == 32 ? (long long)blockIdx.x * kWarpRows + (threadIdx.x >> 5) : CL ? blockIdx.x / parts : blockIdx.x;
    }
    __device__ __forceinline__ long long row_step() const {
        return NT == 32 ? (long long)gridDim.x * kWarpRows : CL ? gridDim.x / parts : gridDim.x;
    }
    __device__ __forceinline__ void sync_block() const {
        if constexpr (NT == 32)
            __syncwarp();
        else
            __syncthreads();
    }
    __device__ __forceinline__ void sync_all() const {
        if constexpr (CL)
            cg::this_cluster().sync();
        else
            sync_block();
    }
    __device__ __forceinline__ const char* table() const { return red + kPartials; }
    __device__ __forceinline__ double* notes() const { return (double*)(red + kPartials + kPowBytes); }
    template <typename V>
    __device__ __forceinline__ V* of(V* p, int rank) const {  // p in another member's shared memory
        if constexpr (CL) return cg::this_cluster().map_shared_rank(p, rank);
        return p;
    }
    // Reductions: butterflies within warps, then over the warps' and the
    // blocks' partials in a fixed order, so that every thread holds the same
    // bits and no timing shows.  reduce(): over the block, one barrier;
    // across(): over the cluster's blocks, one cluster barrier.  Two buffers in
    // turn: a buffer is written again only after a barrier that follows its
    // last reading.  The helper listens: it passes no value.
    template <typename V, typename F>
    __device__ __forceinline__ V reduce(V v, F op) {
        static_assert(sizeof(V) <= 32, "partials are 32 bytes");
        if (!HELP || t < NT) v = warp(v, op);
        if constexpr (NW > 1) {
            char* buf = red + parity * 16 * 32;
            if ((t & 31) == 0 && (!HELP || t < NT)) *(V*)(buf + (t >> 5) * 32) = v;
            __syncthreads();
            v = *(const V*)(buf + ((t & 31) % NW) * 32);
#pragma unroll
            for (int o = NW / 2; o > 0; o >>= 1) v = op(v, shfl(v, o));
            parity ^= 1;
        }
        return v;
    }
    template <typename V, typename F>
    __device__ __forceinline__ V across(V v, F op) {
        static_assert(sizeof(V) <= 32, "partials are 32 bytes");
        if constexpr (CL) {
            V* mine = (V*)(red + 2 * 16 * 32 + parity_all * 32);
            parity_all ^= 1;
            if (t == 0) *mine = v;
            cg::this_cluster().sync();
            v = *of(mine, 0);
            for (int r = 1; r < parts; r++) v = op(v, *of(mine, r));
        }
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
};

// Asynchronous copies into shared memory; wait_copies() waits for the thread's
// own: a barrier of the warp follows it before other lanes' copies are read.
__device__ __forceinline__ void copy8(void* d, const void* g) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"((unsigned)__cvta_generic_to_shared(d)), "l"(g) : "memory");
}
__device__ __forceinline__ void copy4(void* d, const void* g) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"((unsigned)__cvta_generic_to_shared(d)), "l"(g) : "memory");
}
template <int GROUPS = 0>  // all but the latest GROUPS groups
__device__ __forceinline__ void wait_copies() {
    if constexpr (GROUPS == 0)
        asm volatile("cp.async.wait_all;" ::: "memory");
    else
        asm volatile("cp.async.wait_group %0;" ::"n"(GROUPS) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }

// Bulk copies out of shared memory, by one thread for a warp: the warp's writes
// are fenced first; bulk_read() waits until the memory has been read and may be
// written again.  They pass the load-store unit by, which global stores of a
// whole row would fill for thousands of cycles: shared-memory traffic and
// shuffles of every warp on the SM would wait behind them.
__device__ __forceinline__ void fence_bulk() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void bulk_store(void* g, const void* s, unsigned bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(g), "r"((unsigned)__cvta_generic_to_shared(s)), "r"(bytes)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void bulk_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }

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
    int lo, wholes;  // the vectors that the slice fills
    int room;        // vectors that any row's slice may have

    __device__ Slice(T* smem, const T* row, int ncol, int part, int parts) : e(smem) {
        const int per = (ncol + parts - 1) / parts;
        first = min(part * per, ncol);
        n = min(per, ncol - first);
        room = per / VEC + 2;
        src = row + first;
        phase = n > 0 ? (int)(((size_t)src & 15) / sizeof(T)) : 0;
        nv = (phase + n + VEC - 1) / VEC;
        lo = phase > 0;
        wholes = max((phase + n) / VEC - lo, 0);
    }
    static size_t bytes(int ncol, int parts) {  // of shared memory (host)
        const int per = (ncol + parts - 1) / parts;
        return (size_t)(per / VEC + 2) * 16;
    }
    // Starts the copy of vectors v0 .. v1-1 into shared memory, by a warp: 16
    // bytes at a time, elementwise at the slice's edges, so that nothing
    // outside the row is read.
    __device__ __forceinline__ void load(int v0, int v1, int lane) const {
        const int a = max(v0, lo), b = min(v1, lo + wholes);
        const T* from = src + ((a + lane) * VEC - phase);
        unsigned to = (unsigned)__cvta_generic_to_shared(e + (a + lane) * VEC);
#pragma unroll 4
        for (int v = a + lane; v < b; v += 32, from += 32 * VEC, to += 32 * 16)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
        edges(v0, v1, lane, [&](int u) { e[u] = u >= phase && u < phase + n ? src[u - phase] : narrow<T>((typename Ty<T>::W)-INFINITY); });
    }
    // Vectors v0 .. v1-1 into L2.
    __device__ __forceinline__ void prefetch(int v0, int v1) const {
        const int a = max(v0, lo), b = min(v1, lo + wholes);
        if (a < b) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(src + (a * VEC - phase)), "r"((unsigned)(b - a) * 16) : "memory");
    }
    // f(u) for the elements (from the first vector's start) of partial vectors among v0 .. v1-1
    template <typename F>
    __device__ __forceinline__ void edges(int v0, int v1, int lane, F f) const {
        if (lane < 2) {
            const int v = lane == 0 ? 0 : nv - 1;
            if (v >= v0 && v < v1 && (unsigned)(v - lo) >= (unsigned)wholes && (lane == 0 || nv > 1))
                for (int u = v * VEC; u < (v + 1) * VEC; u++) f(u);
        }
    }
    // The vectors of a warp, a run of them: the same places in shared memory
    // for every row of a call, however the rows are aligned.
    template <int NW>
    __device__ __forceinline__ int run(int warp) const {
        return min(warp * ((room + NW - 1) / NW), nv);
    }
    __device__ __forceinline__ Vec<T> get(int v) const { return *(const Vec<T>*)(e + v * VEC); }
    __device__ __forceinline__ void set(int v, const Vec<T>& x) const { *(Vec<T>*)(e + v * VEC) = x; }
    // Vectors v0 .. v1-1 to this slice's place in a row of global memory, by a
    // warp: in one bulk copy where the place is aligned like the source.
    __device__ __forceinline__ void store(int v0, int v1, int lane, T* row) const {
        T* const dst = row + first;
        if ((((size_t)dst ^ (size_t)src) & 15) == 0) {
            fence_bulk();
            __syncwarp();
            const int a = max(v0, lo), b = min(v1, lo + wholes);
            if (lane == 0 && a < b) bulk_store(dst + (a * VEC - phase), e + a * VEC, (unsigned)(b - a) * 16);
            edges(v0, v1, lane, [&](int u) {
                if (u >= phase && u < phase + n) dst[u - phase] = e[u];
            });
            if (lane == 0) bulk_read();
            __syncwarp();
        } else {
            for (int v = v0 + lane; v < v1; v += 32) {
                const Vec<T> x = get(v);
#pragma unroll
                for (int u = 0; u < VEC; u++) {
                    const int i = v * VEC + u - phase;
                    if (i >= 0 && i < n) dst[i] = x.e[u];
                }
            }
            __syncwarp();  // every lane has read its vectors
        }
    }
};

// ---------------------------------------------------------------- host side

inline Heat heat_of(double t) {
    Heat h;
    h.t = t;
    h.inv = 1.0 / t;
    h.c = 16.0 * 1.4426950408889634 * h.inv;
    h.cf = (float)(1.4426950408889634 * h.inv);
    const auto high_word = [](double x) {
        unsigned long long b;
        memcpy(&b, &x, 8);
        return (unsigned)(b >> 32);
    };
    h.high = (int)high_word(16000.0 / h.c);
    h.low = high_word(-16300.0 / h.c) + 1;
    h.span = 0xfff00000u - h.low;
    return h;
}

// How a call's rows are dealt to threads.
struct Deal {
    int nt, help, parts, blocks;  // threads of a team (32: a warp) and its helper's, blocks of a team, of the grid
    size_t slice, team;  // bytes of shared memory: of a slice, of a team's part
};
constexpr size_t kSmemBlock = 227 * 1024, kSmemSM = 228 * 1024;

// Warps take short rows (where what they need besides is at most warp_extra
// bytes), blocks of 128 and 256 threads longer ones.  A row
// that no block can hold is shared by a cluster of blocks, and one of few rows
// too, so that the card is not left idle.
template <typename T>
Deal deal(const hx_readout& r, size_t extra, size_t warp_extra, int block, int blocks, int help, int sms) {
    Deal d{};
    d.help = help;
    d.parts = 1;
    if (r.ncol <= 512 && extra <= warp_extra) {
        d.nt = 32;
    } else {
        while (d.parts < 8 && kRedBytes + Slice<T>::bytes(r.ncol, d.parts) + extra > kSmemBlock) d.parts *= 2;
        while (d.parts < 8 && (long long)r.nrow * d.parts * 2 <= sms && r.ncol / d.parts >= 4096) d.parts *= 2;
        d.nt = d.parts == 1 && r.ncol <= 2048 ? 128 : block;
    }
    d.slice = Slice<T>::bytes(r.ncol, d.parts);
    d.team = kRedBytes + d.slice + (extra + 15) / 16 * 16;
    // as many blocks as are resident at once: each takes rows in turn
    const int rows = d.nt == 32 ? kWarpRows : 1;
    const int per_sm = (int)std::min<size_t>(d.nt == block ? blocks : 6, kSmemSM / (d.team * rows + 1024));
    const long long all = ((long long)r.nrow + rows - 1) / rows * d.parts, most = (long long)sms * std::max(per_sm, 1) / d.parts * d.parts;
    d.blocks = (int)std::min(all, most);
    return d;
}

template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), const Deal& d, cudaStream_t st, A... args) {
    cudaLaunchConfig_t c{};
    c.dynamicSmemBytes = d.nt == 32 ? d.team * kWarpRows : d.team;
    // the limit is the kernel's, for every thread and context: always the same one, so that no call takes it from another
    if (c.dynamicSmemBytes > 48 * 1024)
        if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSmemBlock)) return e;
    c.gridDim = dim3((unsigned)d.blocks);
    c.blockDim = dim3(d.nt == 32 ? 32 * kWarpRows : d.nt + d.help);
    c.stream = st;
    cudaLaunchAttribute a;
    a.id = cudaLaunchAttributeClusterDimension;
    a.val.clusterDim.x = d.parts;
    a.val.clusterDim.y = a.val.clusterDim.z = 1;
    if (d.parts > 1) {
        c.attrs = &a;
        c.numAttrs = 1;
    }
    return cudaLaunchKernelEx(&c, kernel, P(args)...);
}

inline int sm_count(int device) {  // asked once a device
    static std::atomic<int> known[64];
    std::atomic<int>* const k = device >= 0 && device < 64 ? known + device : nullptr;
    int n = k ? k->load(std::memory_order_relaxed) : 0;
    if (n > 0) return n;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return 1;
    if (k) k->store(n, std::memory_order_relaxed);
    return n;
}

template <typename F>
auto by_type(int dtype, F f) {
    switch (dtype) {
        case HX_DT_F64: return f((double*)nullptr);
        case HX_DT_F32: return f((float*)nullptr);
        case HX_DT_F16: return f((__half*)nullptr);
        default: return f((__nv_bfloat16*)nullptr);
    }
}

// hx_select.cu
cudaError_t launch_top(const hx_readout& rows, int k, const Heat& heat, int* idx, void* val, void* lse, int sms, cudaStream_t st);
cudaError_t launch_sample(const hx_readout& rows, const hx_sample_rule& rule, const hx_sample_rule* rules, const double* u, int bits,
                          int* idx, void* logp, int sms, cudaStream_t st);

}  // namespace hxr

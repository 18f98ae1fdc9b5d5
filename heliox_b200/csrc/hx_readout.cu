// hx_readout.cu -- operators over readout rows: a teacher's top logits, the
// distillation loss of a student's rows with its gradient, sampled choices.
//
// One thread block per row; the row is read from global memory once per pass.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdio>
#include <string>

#include "heliox_b200.h"
#include "hx_ctx.hpp"

namespace {

constexpr int kThreads = 256;

// Compute and statistics type W and the order-preserving integer key of each
// element type (equal values, +0 and -0 among them, have equal keys).
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

template <typename T>
struct Ty {  // float, __half, __nv_bfloat16
    using W = float;
    using K = unsigned;
};
template <>
struct Ty<double> {
    using W = double;
    using K = unsigned long long;
};

__device__ __forceinline__ double wide(double x) { return x; }
__device__ __forceinline__ float wide(float x) { return x; }
__device__ __forceinline__ float wide(__half x) { return __half2float(x); }
__device__ __forceinline__ float wide(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void put(double* p, double v) { *p = v; }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ double load_any(const void* p, int dtype, size_t i) {
    switch (dtype) {
        case HX_DT_F64: return ((const double*)p)[i];
        case HX_DT_F32: return (double)((const float*)p)[i];
        case HX_DT_F16: return (double)__half2float(((const __half*)p)[i]);
        default: return (double)__bfloat162float(((const __nv_bfloat16*)p)[i]);
    }
}

template <typename V, typename F>
__device__ V block_reduce(V v, V* red, F op) {  // the same order whatever the timing
    __syncthreads();
    red[threadIdx.x] = v;
    __syncthreads();
    for (int s = kThreads / 2; s > 0; s >>= 1) {
        if ((int)threadIdx.x < s) red[threadIdx.x] = op(red[threadIdx.x], red[threadIdx.x + s]);
        __syncthreads();
    }
    return red[0];
}
template <typename V>
__device__ V block_sum(V v, V* red) {
    return block_reduce(v, red, [](V a, V b) { return a + b; });
}
template <typename V>
__device__ V block_max(V v, V* red) {
    return block_reduce(v, red, [](V a, V b) { return a > b ? a : b; });
}

// The border of the row's descending order at which a running measure (1 or
// the mass of each element) first exceeds `target`: the border's key, and the
// measure of everything above that key.  The caller makes sure that the whole
// row's measure exceeds the target.
template <typename T, typename M>
__device__ typename Ty<T>::K select_border(const T* __restrict__ x, int n, unsigned long long target, M measure,
                                           unsigned long long* above_out) {
    using K = typename Ty<T>::K;
    using W = typename Ty<T>::W;
    __shared__ unsigned long long hist[256];
    __shared__ int s_digit;
    __shared__ unsigned long long s_above;
    K prefix = 0, mask = 0;
    unsigned long long above = 0;
    for (int shift = (int)sizeof(K) * 8 - 8; shift >= 0; shift -= 8) {
        __syncthreads();
        hist[threadIdx.x] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const W v = wide(x[i]);
            if (v == -INFINITY) continue;
            const K k = key_of(v);
            if ((k & mask) != prefix) continue;
            const unsigned long long m = measure(v);
            if (m) atomicAdd(&hist[(int)((k >> shift) & 255)], m);
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            unsigned long long a = above;
            int d = 255;
            while (d > 0 && a + hist[d] <= target) a += hist[d--];
            s_digit = d;
            s_above = a;
        }
        __syncthreads();
        above = s_above;
        prefix |= (K)s_digit << shift;
        mask |= (K)255 << shift;
    }
    *above_out = above;
    return prefix;
}

// Calls take(i) for the first `want` elements of the row with this key, by position.
template <typename T, typename F>
__device__ void first_of_key(const T* __restrict__ x, int n, typename Ty<T>::K key, unsigned long long want, F take) {
    __shared__ int wsum[kThreads / 32];
    unsigned long long seen = 0;
    for (int i0 = 0; i0 < n && seen < want; i0 += kThreads) {
        const int i = i0 + threadIdx.x;
        const bool hit = i < n && wide(x[i]) != -INFINITY && key_of(wide(x[i])) == key;
        const unsigned b = __ballot_sync(~0u, hit);
        if ((threadIdx.x & 31) == 0) wsum[threadIdx.x >> 5] = __popc(b);
        __syncthreads();
        unsigned long long at = seen + __popc(b & ((1u << (threadIdx.x & 31)) - 1));
        int all = 0;
        for (int w = 0; w < kThreads / 32; w++) {
            if (w < (int)(threadIdx.x >> 5)) at += wsum[w];
            all += wsum[w];
        }
        if (hit && at < want) take(i, at);
        seen += all;
        __syncthreads();
    }
}

// ---------------------------------------------------------------- top logits

template <typename T>
__global__ void __launch_bounds__(kThreads) top_kernel(const T* __restrict__ xs, int ncol, long long ld, int k, double temperature,
                                                       int* __restrict__ idx, T* __restrict__ val,
                                                       typename Ty<T>::W* __restrict__ lse) {
    using W = typename Ty<T>::W;
    using K = typename Ty<T>::K;
    __shared__ double red[kThreads];
    __shared__ K skey[HX_READOUT_MAX_K];
    __shared__ int sidx[HX_READOUT_MAX_K];
    __shared__ int nabove;
    const T* x = xs + (size_t)blockIdx.x * ld;
    idx += (size_t)blockIdx.x * k;
    val += (size_t)blockIdx.x * k;
    W mx = -INFINITY;
    int open = 0, bad = 0;
    for (int i = threadIdx.x; i < ncol; i += kThreads) {
        const W v = wide(x[i]);
        if (v > mx) mx = v;
        open += v > -INFINITY;
        bad |= v != v;
    }
    mx = (W)block_max((double)mx, red);
    open = block_sum(open, (int*)red);
    bad = block_max(bad, (int*)red);
    const W nan = (W)NAN;
    if (lse) {
        const W inv = (W)(1.0 / temperature);
        W s = 0;
        for (int i = threadIdx.x; i < ncol; i += kThreads) s += exp((wide(x[i]) - mx) * inv);
        s = block_sum(s, (W*)red);
        if (threadIdx.x == 0)
            lse[blockIdx.x] = bad ? nan : mx == -INFINITY || mx == INFINITY ? mx : (W)((double)mx / temperature + log((double)s));
    }
    const int kk = bad ? 0 : min(k, open);
    for (int j = kk + threadIdx.x; j < k; j += kThreads) {
        idx[j] = -1;
        put(&val[j], bad ? nan : (W)-INFINITY);
    }
    if (kk == 0) return;
    unsigned long long above;
    const K border = select_border(x, ncol, (unsigned long long)(kk - 1), [](W) { return 1ull; }, &above);
    __syncthreads();
    if (threadIdx.x == 0) nabove = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < ncol; i += kThreads) {
        const W v = wide(x[i]);
        if (v > -INFINITY && key_of(v) > border) {
            const int at = atomicAdd(&nabove, 1);
            skey[at] = key_of(v);
            sidx[at] = i;
        }
    }
    __syncthreads();
    first_of_key(x, ncol, border, (unsigned long long)kk - above, [&](int i, unsigned long long at) {
        skey[above + at] = border;
        sidx[above + at] = i;
    });
    int p2 = 1;
    while (p2 < kk) p2 <<= 1;
    for (int j = kk + threadIdx.x; j < p2; j += kThreads) {
        skey[j] = 0;
        sidx[j] = INT_MAX;
    }
    for (int w = 2; w <= p2; w <<= 1) {
        for (int d = w >> 1; d > 0; d >>= 1) {
            __syncthreads();
            for (int j = threadIdx.x; j < p2; j += kThreads) {
                const int o = j ^ d;
                if (o > j) {
                    const K a = skey[j], b = skey[o];
                    const int ia = sidx[j], ib = sidx[o];
                    const bool first = a > b || (a == b && ia < ib);
                    if (first != ((j & w) == 0)) {
                        skey[j] = b;
                        skey[o] = a;
                        sidx[j] = ib;
                        sidx[o] = ia;
                    }
                }
            }
        }
    }
    __syncthreads();
    for (int j = threadIdx.x; j < kk; j += kThreads) {
        idx[j] = sidx[j];
        val[j] = x[sidx[j]];
    }
}

// ---------------------------------------------------------------- distillation

template <typename T>
__global__ void __launch_bounds__(kThreads) distill_kernel(const T* xs, int ncol, long long ld, hx_teacher te, double temperature,
                                                           double scale, const double* __restrict__ weight, T* gs,
                                                           long long ldg, typename Ty<T>::W* __restrict__ row_loss) {
    using W = typename Ty<T>::W;
    extern __shared__ unsigned inside[];  // one bit per column: in a slot
    __shared__ double red[kThreads];
    __shared__ double sq[HX_READOUT_MAX_K], sx[HX_READOUT_MAX_K];
    __shared__ int si[HX_READOUT_MAX_K];
    const size_t row = blockIdx.x;
    const T* x = xs + row * ld;
    T* g = gs ? gs + row * ldg : nullptr;
    const int k = te.k;
    const double w = weight ? weight[row] : 1.0;
    const double inv = 1.0 / temperature;
    for (int i = threadIdx.x; i < (ncol + 31) / 32; i += kThreads) inside[i] = 0;
    for (int j = threadIdx.x; j < k; j += kThreads) {
        const int i = te.idx[row * k + j];
        const double v = load_any(te.val, te.dtype, row * k + j);
        si[j] = i >= 0 && i < ncol && v != -INFINITY ? i : -1;
        sq[j] = v;
    }
    __syncthreads();
    int used = 0;
    for (int j = threadIdx.x; j < k; j += kThreads) {
        bool twice = false;
        for (int l = 0; l < j; l++) twice |= si[l] == si[j];
        sx[j] = twice ? 1.0 : 0.0;
    }
    __syncthreads();
    for (int j = threadIdx.x; j < k; j += kThreads) {
        if (sx[j] != 0.0) si[j] = -1;
        if (si[j] >= 0) {
            used = 1;
            atomicOr(&inside[si[j] >> 5], 1u << (si[j] & 31));
        }
    }
    used = block_max(used, (int*)red);
    W mx = -INFINITY;
    int bad = 0;
    if (w != 0.0 && used)
        for (int i = threadIdx.x; i < ncol; i += kThreads) {
            const W v = wide(x[i]);
            if (v > mx) mx = v;
            bad |= v != v;
        }
    mx = (W)block_max((double)mx, red);
    bad = block_max(bad, (int*)red);
    if (w == 0.0 || !used || (mx == -INFINITY && !bad)) {
        if (threadIdx.x == 0) row_loss[row] = 0;
        if (g)
            for (int i = threadIdx.x; i < ncol; i += kThreads) put(&g[i], (W)0);
        return;
    }
    if (bad) mx = NAN;
    const W winv = (W)inv;
    W s_in = 0, s_out = 0;
    for (int i = threadIdx.x; i < ncol; i += kThreads) {
        const W e = exp((wide(x[i]) - mx) * winv);
        if (inside[i >> 5] >> (i & 31) & 1)
            s_in += e;
        else
            s_out += e;
    }
    const double sum_in = (double)block_sum(s_in, (W*)red), sum_out = (double)block_sum(s_out, (W*)red);
    const double total = sum_in + sum_out, log_total = log(total);
    // the teacher's q in the slots
    double norm;
    if (te.lse) {
        norm = load_any(te.lse, te.dtype == HX_DT_F64 ? HX_DT_F64 : HX_DT_F32, row);
    } else {
        double tm = -INFINITY;
        for (int j = threadIdx.x; j < k; j += kThreads)
            if (si[j] >= 0) tm = sq[j] > tm || sq[j] != sq[j] ? sq[j] : tm;
        tm = block_reduce(tm, red, [](double a, double b) { return a > b || a != a ? a : b; });
        double ts = 0;
        for (int j = threadIdx.x; j < k; j += kThreads)
            if (si[j] >= 0) ts += exp((sq[j] - tm) * inv);
        ts = block_sum(ts, red);
        norm = tm * inv + log(ts);
    }
    double qs = 0, loss = 0;
    for (int j = threadIdx.x; j < k; j += kThreads) {
        if (si[j] < 0) continue;
        const double lq = sq[j] * inv - norm, q = exp(lq);
        const double lp = ((double)wide(x[si[j]]) - (double)mx) * inv - log_total;
        sx[j] = lp;
        sq[j] = q;
        qs += q;
        loss += q == 0.0 ? 0.0 : q * (lq - lp);
    }
    qs = block_sum(qs, red);
    loss = block_sum(loss, red);
    double qr = te.lse ? (qs == qs ? fmax(0.0, 1.0 - qs) : qs) : 0.0;
    const double pr = sum_out / total;
    if (qr > 0.0 && sum_out > 0.0)
        loss += qr * (log(qr) - log(pr));
    else if (qr == qr)
        qr = 0.0;
    if (threadIdx.x == 0) row_loss[row] = (W)(temperature * temperature * loss);
    if (!g) return;
    const double c = scale * w * temperature, mass = te.lse ? qs + qr : 1.0;
    const W a_in = (W)(c * mass / total), a_out = qr == 0.0 ? a_in : (W)(c * (mass - qr / pr) / total);
    __syncthreads();
    for (int i = threadIdx.x; i < ncol; i += kThreads) {
        const W e = exp((wide(x[i]) - mx) * winv);
        if (!(inside[i >> 5] >> (i & 31) & 1)) put(&g[i], a_out * e);
    }
    for (int j = threadIdx.x; j < k; j += kThreads)
        if (si[j] >= 0) put(&g[si[j]], (W)(c * (mass * exp(sx[j]) - sq[j])));
}

template <typename W>
__global__ void __launch_bounds__(kThreads) loss_kernel(const W* __restrict__ row_loss, const double* __restrict__ weight, int nrow,
                                                        double scale, W* __restrict__ loss) {
    __shared__ double red[kThreads];
    double s = 0;
    for (int r = threadIdx.x; r < nrow; r += kThreads) {
        const double w = weight ? weight[r] : 1.0;
        if (w != 0.0) s += w * (double)row_loss[r];
    }
    s = block_sum(s, red);
    if (threadIdx.x == 0) *loss = (W)(scale * s);
}

// ---------------------------------------------------------------- sampling

struct Rule {
    double temperature;
    int top_k;
    double top_p, min_p;
};
__device__ __forceinline__ Rule clean(const hx_sample_rule& r, int ncol) {
    Rule o;
    const bool greedy = r.temperature <= 0.0;
    o.temperature = greedy ? 1.0 : r.temperature;
    o.top_k = greedy ? 1 : r.top_k >= 1.0 ? (r.top_k < (double)ncol ? (int)r.top_k : ncol) : ncol;
    o.top_p = r.top_p < 1.0 ? fmax(r.top_p, 0.0) : 1.0;
    o.min_p = r.min_p > 0.0 ? fmin(r.min_p, 1.0) : 0.0;
    return o;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const T* __restrict__ xs, int ncol, long long ld, hx_sample_rule rule,
                                                          const hx_sample_rule* __restrict__ rules,
                                                          const double* __restrict__ us, int bits, int* __restrict__ idx,
                                                          typename Ty<T>::W* __restrict__ logp) {
    using W = typename Ty<T>::W;
    using K = typename Ty<T>::K;
    __shared__ double red[kThreads];
    __shared__ int s_at;
    const T* x = xs + (size_t)blockIdx.x * ld;
    const Rule r = clean(rules ? rules[blockIdx.x] : rule, ncol);
    W mxw = -INFINITY;
    int open = 0, bad = r.temperature != r.temperature;
    for (int i = threadIdx.x; i < ncol; i += kThreads) {
        const W v = wide(x[i]);
        if (v > mxw) mxw = v;
        open += v > -INFINITY;
        bad |= v != v || v == INFINITY;
    }
    const double mx = block_max((double)mxw, red);
    open = block_sum(open, (int*)red);
    bad = block_max(bad, (int*)red);
    if (bad || open == 0) {
        if (threadIdx.x == 0) {
            idx[blockIdx.x] = bad ? -2 : -1;
            if (logp) logp[blockIdx.x] = bad ? (W)NAN : (W)-INFINITY;
        }
        return;
    }
    const double inv = 1.0 / r.temperature, unit = ldexp(1.0, bits);
    auto weight = [&](W v) { return exp(((double)v - mx) * inv); };
    auto mass = [&](W v) { return __double2ull_rn(weight(v) * unit); };
    unsigned long long total, above;
    const int top_k = min(r.top_k, open);
    auto mass_above = [&](K key) {
        unsigned long long s = 0;
        for (int i = threadIdx.x; i < ncol; i += kThreads) {
            const W v = wide(x[i]);
            if (v > -INFINITY && key_of(v) > key) s += mass(v);
        }
        return block_sum(s, (unsigned long long*)red);
    };
    if (top_k < open) {
        const K key = select_border(x, ncol, (unsigned long long)(top_k - 1), [](W) { return 1ull; }, &above);
        total = mass_above(key) + ((unsigned long long)top_k - above) * mass(value_of(key));
    } else {
        total = mass_above(0);
    }
    double floor_ = r.min_p;  // kept: weight at least this
    if (r.top_p < 1.0) {
        const double want = ceil(r.top_p * (double)total);
        unsigned long long target = want < 1.0 ? 1 : (unsigned long long)want;
        if (target > total) target = total;
        const K key = select_border(x, ncol, target - 1, mass, &above);
        const W v = value_of(key);
        const unsigned long long m = mass(v);
        total = above + (target - above + m - 1) / m * m;
        if (weight(v) >= floor_) floor_ = 0.0;
    } else if (top_k < open) {
        const K key = select_border(x, ncol, total - 1, mass, &above);
        if (weight(value_of(key)) >= floor_) floor_ = 0.0;
    }
    if (floor_ > 0.0) {
        unsigned long long s = 0;
        for (int i = threadIdx.x; i < ncol; i += kThreads) {
            const W v = wide(x[i]);
            if (v > -INFINITY && weight(v) >= floor_) s += mass(v);
        }
        s = block_sum(s, (unsigned long long*)red);
        total = s < total ? s : total;
    }
    double u = us[blockIdx.x];
    u = u > 0.0 ? u : 0.0;
    const double want = u < 1.0 ? floor(u * (double)total) : (double)total;
    unsigned long long target = (unsigned long long)want;
    if (target >= total) target = total - 1;
    const K key = select_border(x, ncol, target, mass, &above);
    const W v = value_of(key);
    first_of_key(x, ncol, key, (target - above) / mass(v) + 1, [&](int i, unsigned long long at) {
        if (at == (target - above) / mass(v)) s_at = i;
    });
    __syncthreads();
    if (threadIdx.x == 0) {
        idx[blockIdx.x] = s_at;
        if (logp) logp[blockIdx.x] = (W)(((double)v - mx) * inv - log((double)total / unit));
    }
}

// ---------------------------------------------------------------- host side

int type_size(int dtype) { return dtype == HX_DT_F64 ? 8 : dtype == HX_DT_F32 ? 4 : 2; }
int stat_size(int dtype) { return dtype == HX_DT_F64 ? 8 : 4; }
bool off(const void* p, int align) { return (size_t)p % (size_t)align != 0; }

const char* check_rows(const hx_readout* r) {
    if (!r) return "null rows";
    if (r->dtype < HX_DT_F64 || r->dtype > HX_DT_BF16) return "rows: unknown dtype";
    if (r->nrow < 0 || r->ncol < 0) return "rows: nrow and ncol must not be negative";
    if (r->ld < r->ncol) return "rows: ld must be at least ncol";
    if ((long long)r->ncol * type_size(r->dtype) > HX_READOUT_MAX_ROW_BYTES) return "rows: a row is longer than HX_READOUT_MAX_ROW_BYTES";
    if (r->nrow > 1 && r->ld > (1ll << 60) / r->nrow) return "rows: ld is out of range";
    if (r->nrow > 0 && r->ncol > 0 && !r->x) return "rows: null x";
    if (off(r->x, type_size(r->dtype))) return "rows: x is not aligned to its type";
    return nullptr;
}
const char* check_temperature(double t) {
    return t >= 1e-30 && t <= 1e30 ? nullptr : "temperature must be between 1e-30 and 1e30";
}

const char* check_top(const hx_readout* r, int k, double t, const void* idx, const void* val, const void* lse) {
    if (const char* e = check_rows(r)) return e;
    if (k < 1 || k > HX_READOUT_MAX_K) return "k must be 1 .. HX_READOUT_MAX_K";
    if (const char* e = check_temperature(t)) return e;
    if (r->nrow > 0 && (!idx || !val)) return "null idx or val";
    if (off(idx, 4) || off(val, type_size(r->dtype)) || off(lse, stat_size(r->dtype))) return "an output is not aligned to its type";
    return nullptr;
}

const char* check_distill(const hx_readout* r, const hx_teacher* t, double temperature, double scale, const void* weight,
                          const void* grad, long long ldg, const void* row_loss, const void* loss) {
    if (const char* e = check_rows(r)) return e;
    if (!t) return "null teacher";
    if (t->dtype < HX_DT_F64 || t->dtype > HX_DT_BF16) return "teacher: unknown dtype";
    if (t->k < 1 || t->k > HX_READOUT_MAX_K) return "teacher: k must be 1 .. HX_READOUT_MAX_K";
    if (r->nrow > 0 && (!t->idx || !t->val)) return "teacher: null idx or val";
    if (off(t->idx, 4) || off(t->val, type_size(t->dtype)) || off(t->lse, stat_size(t->dtype))) return "teacher: an array is not aligned to its type";
    if (const char* e = check_temperature(temperature)) return e;
    if (!std::isfinite(scale)) return "scale must be finite";
    if (!loss || (r->nrow > 0 && !row_loss)) return "null loss or row_loss";
    if (off(weight, 8) || off(grad, type_size(r->dtype)) || off(row_loss, stat_size(r->dtype)) || off(loss, stat_size(r->dtype)))
        return "an array is not aligned to its type";
    if (!grad || r->nrow == 0 || r->ncol == 0) return nullptr;
    if (ldg < r->ncol) return "ld_grad must be at least ncol";
    if (r->nrow > 1 && ldg > (1ll << 60) / r->nrow) return "ld_grad is out of range";
    if (grad == r->x) return r->nrow == 1 || ldg == r->ld ? nullptr : "grad in place of x needs the same ld";
    // other overlaps: rows between rows are apart, everything else is refused
    const long long es = type_size(r->dtype);
    const long long x0 = (long long)(size_t)r->x, g0 = (long long)(size_t)grad;
    const long long x1 = x0 + ((r->nrow - 1) * r->ld + r->ncol) * es, g1 = g0 + ((r->nrow - 1) * ldg + r->ncol) * es;
    if (g0 >= x1 || x0 >= g1) return nullptr;
    if (ldg == r->ld) {
        const long long pitch = r->ld * es, d = ((g0 - x0) % pitch + pitch) % pitch;
        if (d >= r->ncol * es && pitch - d >= r->ncol * es) return nullptr;
    }
    return "grad overlaps x";
}

const char* check_sample(const hx_readout* r, const hx_sample_rule* rule, const void* rules, const void* u, const void* idx,
                         const void* logp) {
    if (const char* e = check_rows(r)) return e;
    if (!rules) {
        if (!rule) return "null rule";
        if (rule->temperature != 0.0)
            if (const char* e = check_temperature(rule->temperature)) return e;
        if (!(rule->top_k >= 0.0)) return "top_k must not be negative";
        if (!(rule->top_p >= 0.0 && rule->top_p <= 1.0)) return "top_p must be between 0 and 1";
        if (!(rule->min_p >= 0.0 && rule->min_p <= 1.0)) return "min_p must be between 0 and 1";
    }
    if (r->nrow > 0 && (!u || !idx)) return "null u or idx";
    if (off(rules, 8) || off(u, 8) || off(idx, 4) || off(logp, stat_size(r->dtype))) return "an array is not aligned to its type";
    return nullptr;
}

int told(const char* e, char* msg, int cap) {
    if (e && msg && cap > 0) snprintf(msg, (size_t)cap, "%s", e);
    return e ? -1 : 0;
}

// The context's device for the length of a call.
struct OnDevice {
    int before = -1;
    cudaError_t e;
    explicit OnDevice(int device) {
        e = cudaGetDevice(&before);
        if (e == cudaSuccess && before != device)
            e = cudaSetDevice(device);
        else
            before = -1;
    }
    ~OnDevice() {
        if (before >= 0) cudaSetDevice(before);
    }
};

template <typename F>
int by_type(int dtype, F f) {
    switch (dtype) {
        case HX_DT_F64: return f((double*)nullptr);
        case HX_DT_F32: return f((float*)nullptr);
        case HX_DT_F16: return f((__half*)nullptr);
        default: return f((__nv_bfloat16*)nullptr);
    }
}

}  // namespace

#define HXC(call)                                                                                       \
    do {                                                                                                \
        cudaError_t _e = (call);                                                                        \
        if (_e != cudaSuccess) return hx_fail(ctx, std::string(#call) + ": " + cudaGetErrorString(_e)); \
    } while (0)

extern "C" {

int hx_top_logits_check(const hx_readout* rows, int k, double temperature, const int32_t* idx_dev, const void* val_dev,
                        const void* lse_dev, char* msg, int cap) {
    return told(check_top(rows, k, temperature, idx_dev, val_dev, lse_dev), msg, cap);
}
int hx_distill_check(const hx_readout* rows, const hx_teacher* teacher, double temperature, double scale,
                     const double* row_weight_dev, const void* grad_dev, long long ld_grad, const void* row_loss_dev,
                     const void* loss_dev, char* msg, int cap) {
    return told(check_distill(rows, teacher, temperature, scale, row_weight_dev, grad_dev, ld_grad, row_loss_dev, loss_dev), msg, cap);
}
int hx_sample_check(const hx_readout* rows, const hx_sample_rule* rule, const hx_sample_rule* rules_dev,
                    const double* u_dev, const int32_t* idx_dev, const void* logp_dev, char* msg, int cap) {
    return told(check_sample(rows, rule, rules_dev, u_dev, idx_dev, logp_dev), msg, cap);
}

int hx_top_logits_dev(hx_ctx* ctx, const hx_readout* rows, int k, double temperature, int32_t* idx_dev, void* val_dev,
                      void* lse_dev) {
    if (!ctx) return -1;
    if (const char* e = check_top(rows, k, temperature, idx_dev, val_dev, lse_dev)) return hx_fail(ctx, e);
    if (rows->nrow == 0) return 0;
    OnDevice on(ctx->device);
    HXC(on.e);
    return by_type(rows->dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        top_kernel<T><<<rows->nrow, kThreads, 0, ctx->st>>>((const T*)rows->x, rows->ncol, rows->ld, k, temperature, idx_dev,
                                                            (T*)val_dev, (typename Ty<T>::W*)lse_dev);
        HXC(cudaGetLastError());
        return 0;
    });
}

int hx_distill_loss_grad_dev(hx_ctx* ctx, const hx_readout* rows, const hx_teacher* teacher, double temperature,
                             double scale, const double* row_weight_dev, void* grad_dev, long long ld_grad,
                             void* row_loss_dev, void* loss_dev) {
    if (!ctx) return -1;
    if (const char* e = check_distill(rows, teacher, temperature, scale, row_weight_dev, grad_dev, ld_grad, row_loss_dev, loss_dev))
        return hx_fail(ctx, e);
    OnDevice on(ctx->device);
    HXC(on.e);
    return by_type(rows->dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        using W = typename Ty<T>::W;
        const size_t smem = (size_t)(rows->ncol + 31) / 32 * 4;
        HXC(cudaFuncSetAttribute(distill_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        if (rows->nrow > 0) {
            distill_kernel<T><<<rows->nrow, kThreads, smem, ctx->st>>>((const T*)rows->x, rows->ncol, rows->ld, *teacher, temperature,
                                                                       scale, row_weight_dev, (T*)grad_dev, ld_grad, (W*)row_loss_dev);
            HXC(cudaGetLastError());
        }
        loss_kernel<W><<<1, kThreads, 0, ctx->st>>>((const W*)row_loss_dev, row_weight_dev, rows->nrow, scale, (W*)loss_dev);
        HXC(cudaGetLastError());
        return 0;
    });
}

int hx_sample_dev(hx_ctx* ctx, const hx_readout* rows, const hx_sample_rule* rule, const hx_sample_rule* rules_dev,
                  const double* u_dev, int32_t* idx_dev, void* logp_dev) {
    if (!ctx) return -1;
    if (const char* e = check_sample(rows, rule, rules_dev, u_dev, idx_dev, logp_dev)) return hx_fail(ctx, e);
    if (rows->nrow == 0) return 0;
    int lg = 0;
    while ((1ll << lg) < rows->ncol) lg++;
    const int bits = lg <= 10 ? 52 : 62 - lg;
    const hx_sample_rule none{1.0, 0.0, 1.0, 0.0};
    OnDevice on(ctx->device);
    HXC(on.e);
    return by_type(rows->dtype, [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        sample_kernel<T><<<rows->nrow, kThreads, 0, ctx->st>>>((const T*)rows->x, rows->ncol, rows->ld, rules_dev ? none : *rule,
                                                               rules_dev, u_dev, bits, idx_dev, (typename Ty<T>::W*)logp_dev);
        HXC(cudaGetLastError());
        return 0;
    });
}

}  // extern "C"

// hx_readout.cu -- operators over readout rows: a teacher's top logits, the
// distillation loss of a student's rows with its gradient, sampled choices.
//
// One thread block per row; the row is read from global memory once per pass.
#include <cuda_runtime.h>

#include <climits>
#include <cmath>
#include <cstdio>
#include <string>
#include <type_traits>

#include "heliox_b200.h"
#include "hx_ctx.hpp"
#include "hx_readout.cuh"

namespace {

using namespace hxr;

constexpr int kThreads = 256;

__device__ __forceinline__ void put(double* p, double v) { *p = v; }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

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
//
// One pass over memory: the row waits in shared memory while its maximum, the
// sum of its exponentials and then the gradient are taken.  The slots' readouts
// are lifted out of the row first (-inf stands in their places), so that the
// sum over the rest is a sum of its own and not a difference.  The teacher's
// side is worked out while the row is on its way.

constexpr int kScanSlots = 128;  // up to here a slot looks for earlier ones of its position one by one, above in a hash table
constexpr int kHash = 2048;

static_assert(HX_READOUT_MAX_ROW_BYTES / 2 <= 1 << 20 && HX_READOUT_MAX_K <= 1 << 10, "a position and a slot share 32 bits in the hash table");

size_t distill_extra(int k) { return ((size_t)k * (8 + 8 + 4) + 15) / 16 * 16 + (k > kScanSlots ? kHash * 4 : 0); }

template <typename T, int NT, bool CL>
__global__ void __launch_bounds__(NT == 32 ? 32 * kWarpRows : NT, NT == 512 ? 2 : 1)
    distill_kernel(const T* xs, int nrow, int ncol, long long ld, hx_teacher te, double temperature, double scale,
                   const double* __restrict__ weight, T* gs, long long ldg, typename Ty<T>::W* __restrict__ row_loss,
                   int team_bytes, int slice_bytes) {
    using W = typename Ty<T>::W;
    constexpr int VEC = Ty<T>::VEC;
    extern __shared__ __align__(16) char smem[];
    char* mine = smem + (NT == 32 ? (threadIdx.x >> 5) * team_bytes : 0);
    Team<NT, CL> team(mine);
    const size_t row = team.row_of_block(team.parts);
    if (NT == 32 && row >= (size_t)nrow) return;
    const int t = team.t, k = te.k;
    const Slice<T> sl((T*)(mine + kRedBytes), xs + row * ld, ncol, team.part, team.parts);
    double* sq = (double*)(mine + kRedBytes + slice_bytes);  // the slots: value, then probability
    double* sx = sq + k;                                     // the row's readout there
    int* si = (int*)(sx + k);                                // position, -1: not used
    unsigned* hash = (unsigned*)(mine + kRedBytes + slice_bytes + ((size_t)k * 20 + 15) / 16 * 16);
    T* g = gs ? gs + row * ldg : nullptr;
    const double w = weight ? weight[row] : 1.0;
    const double inv = 1.0 / temperature;
    if (w != 0.0) sl.template load<NT>(t);

    // the slots
    if (k > kScanSlots)
        for (int j = t; j < kHash; j += NT) hash[j] = ~0u;
    for (int j = t; j < k; j += NT) {
        const int i = te.idx[row * k + j];
        const double v = load_any(te.val, te.dtype, row * k + j);
        si[j] = i >= 0 && i < ncol && v != -INFINITY ? i : -1;
        sq[j] = v;
    }
    team.sync();
    if (k > kScanSlots) {
        for (int j = t; j < k; j += NT) {
            const int i = si[j];
            if (i < 0) continue;
            const unsigned both = (unsigned)i << 10 | (unsigned)j;
            int h = (int)(((unsigned)i * 2654435761u) >> 21);
            for (int step = 0; step < kHash; step++, h = (h + 1) & (kHash - 1)) {  // at most kHash / 2 places are taken
                const unsigned o = atomicCAS(&hash[h], ~0u, both);
                if (o == ~0u) break;
                if (o >> 10 == (unsigned)i) {
                    atomicMin(&hash[h], both);
                    break;
                }
            }
        }
        team.sync();
    }
    double tm = -INFINITY;
    bool used = false;
    for (int j = t; j < k; j += NT) {
        const int i = si[j];
        bool first = i >= 0;
        if (k > kScanSlots) {
            if (first) {
                int h = (int)(((unsigned)i * 2654435761u) >> 21);
                for (int step = 0; step < kHash && hash[h] >> 10 != (unsigned)i; step++) h = (h + 1) & (kHash - 1);
                first = (hash[h] & 1023) == (unsigned)j;
            }
        } else {
            for (int l = 0; l < j; l++) first &= si[l] != i;
        }
        sx[j] = first ? 1.0 : 0.0;
        used |= first;
        if (first) tm = sq[j] > tm || sq[j] != sq[j] ? sq[j] : tm;
    }
    used = team.any(used) && w != 0.0;
    if (used) {
        for (int j = t; j < k; j += NT)
            if (sx[j] == 0.0) si[j] = -1;
    } else {  // the same in every block of a cluster
        if (t == 0 && team.part == 0) row_loss[row] = 0;
        sl.wait();
        if (g) sl.template store<NT>(t, g, [](int) {
            Vec<T> z;
#pragma unroll
            for (int u = 0; u < VEC; u++) z.e[u] = narrow<T>((W)0);
            return z;
        });
        return;
    }
    double norm;
    if (te.lse) {
        norm = load_any(te.lse, te.dtype == HX_DT_F64 ? HX_DT_F64 : HX_DT_F32, row);
    } else {
        tm = team.template reduce<false>(tm, [](double a, double b) { return a > b || a != a ? a : b; });
        double ts = 0;
        for (int j = t; j < k; j += NT)
            if (si[j] >= 0) ts += exp((sq[j] - tm) * inv);
        ts = team.template reduce<false>(ts, [](double a, double b) { return a + b; });
        norm = tm * inv + log(ts);
    }
    struct Pair {
        double a, b;
    } qa{0, 0};  // sum of q, sum of q log q
    for (int j = t; j < k; j += NT) {
        if (si[j] < 0) continue;
        const double lq = sq[j] * inv - norm, q = exp(lq);
        sq[j] = q;
        qa.a += q;
        qa.b += q == 0.0 ? 0.0 : q * lq;
    }
    qa = team.template reduce<false>(qa, [](Pair x, Pair y) { return Pair{x.a + y.a, x.b + y.b}; });

    // the row is here: lift the slots' readouts out of it
    sl.wait();
    team.sync();
    W mx = -INFINITY;
    for (int j = t; j < k; j += NT) {
        const int i = si[j] - sl.first;
        if (si[j] >= 0 && i >= 0 && i < sl.n) {
            const W v = wide(sl.e[sl.phase + i]);
            sx[j] = (double)v;
            mx = max_num(mx, v);
            sl.e[sl.phase + i] = narrow<T>((W)-INFINITY);
        }
    }
    team.sync();
    for (int v = t; v < sl.nv; v += NT) {
        const Vec<T> x = sl.get(v);
#pragma unroll
        for (int u = 0; u < VEC; u++) mx = max_num(mx, wide(x.e[u]));
    }
    mx = team.template reduce<true>(mx, [](W a, W b) { return max_num(a, b); });
    const W m0 = mx == -INFINITY ? (W)0 : mx;
    const auto ex = scaler((W)0, temperature);
    struct Sums {
        double out, in, qz;
    } s{0, 0, 0};
    {
        W part[2] = {0, 0};
        for (int v = t; v < sl.nv; v += NT) {
            Vec<T> x = sl.get(v);
#pragma unroll
            for (int u = 0; u < VEC; u++) {
                const W e = ex(wide(x.e[u]) - m0);
                part[u & 1] += e;
                if constexpr (sizeof(T) == sizeof(W)) x.e[u] = e;
            }
            if constexpr (sizeof(T) == sizeof(W)) sl.set(v, x);
        }
        s.out = (double)part[0] + (double)part[1];
    }
    for (int j = t; j < k; j += NT) {
        const int i = si[j] - sl.first;
        if (si[j] >= 0 && i >= 0 && i < sl.n) {
            const double z = (sx[j] - (double)m0) * inv;
            s.in += exp(z);
            s.qz += sq[j] == 0.0 ? 0.0 : sq[j] * z;
        }
    }
    s = team.template reduce<true>(s, [](Sums a, Sums b) { return Sums{a.out + b.out, a.in + b.in, a.qz + b.qz}; });
    const double total = s.in + s.out;
    const bool empty = mx == -INFINITY && total == 0.0;  // NaN in the row makes the sums NaN
    double qr = te.lse ? (qa.a == qa.a ? fmax(0.0, 1.0 - qa.a) : qa.a) : 0.0;
    const double pr = s.out / total;
    double loss = qa.b - s.qz + qa.a * log(total);
    if (qr > 0.0 && s.out > 0.0)
        loss += qr * (log(qr) - log(pr));
    else if (qr == qr && s.out == s.out)
        qr = 0.0;
    if (t == 0 && team.part == 0) row_loss[row] = empty ? (W)0 : (W)(temperature * temperature * loss);
    if (g) {
        const double c = empty ? 0.0 : scale * w * temperature;
        const double mass = te.lse || qa.a != qa.a ? qa.a + qr : 1.0;
        const W a_out = empty ? (W)0 : (W)(c * (qr == 0.0 ? mass : mass - qr / pr) / total);
        sl.template store<NT>(t, g, [&](int v) {
            Vec<T> x = sl.get(v);
#pragma unroll
            for (int u = 0; u < VEC; u++) {
                if constexpr (sizeof(T) == sizeof(W))
                    x.e[u] = x.e[u] * a_out;
                else
                    x.e[u] = narrow<T>(ex(wide(x.e[u]) - m0) * a_out);
            }
            return x;
        });
        team.sync();
        for (int j = t; j < k; j += NT) {
            const int i = si[j] - sl.first;
            if (si[j] >= 0 && i >= 0 && i < sl.n) {
                const double p = exp((sx[j] - (double)m0) * inv) / total;
                g[si[j]] = narrow<T>(empty ? (W)0 : (W)(c * (mass * p - sq[j])));
            }
        }
    }
    if constexpr (CL) team.sync_all();  // a block stays while others may read its partials
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

// How a call's rows are dealt to threads.
struct Deal {
    int nt, parts;
    size_t slice, team;  // bytes of shared memory: of a slice, of a team's part
};
constexpr size_t kSmemBlock = 227 * 1024;

// Warps take short rows, blocks of 128 and 512 threads longer ones.  A row
// that no block can hold is shared by a cluster of blocks, and one of few rows
// too, so that the card is not left idle.
template <typename T>
Deal deal(const hx_readout* r, size_t extra, int sms) {
    Deal d{};
    d.parts = 1;
    if (r->ncol <= 512 && extra <= 6144) {
        d.nt = 32;
    } else {
        while (d.parts < 8 && kRedBytes + Slice<T>::bytes(r->ncol, d.parts) + extra > kSmemBlock) d.parts *= 2;
        while (d.parts < 8 && (long long)r->nrow * d.parts * 2 <= sms && r->ncol / d.parts >= 4096) d.parts *= 2;
        d.nt = d.parts == 1 && r->ncol <= 2048 ? 128 : 512;
    }
    d.slice = Slice<T>::bytes(r->ncol, d.parts);
    d.team = kRedBytes + d.slice + (extra + 15) / 16 * 16;
    return d;
}

template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), const Deal& d, int nrow, cudaStream_t st, A... args) {
    cudaLaunchConfig_t c{};
    c.dynamicSmemBytes = d.nt == 32 ? d.team * kWarpRows : d.team;
    if (c.dynamicSmemBytes > 48 * 1024)
        if (cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)c.dynamicSmemBytes)) return e;
    c.gridDim = dim3(d.nt == 32 ? (unsigned)((nrow + kWarpRows - 1) / kWarpRows) : (unsigned)nrow * d.parts);
    c.blockDim = dim3(d.nt == 32 ? 32 * kWarpRows : d.nt);
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

int sm_count(int device) {
    int n = 0;
    return cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) == cudaSuccess ? n : 1;
}

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
        if (rows->nrow > 0) {
            const Deal d = deal<T>(rows, distill_extra(teacher->k), sm_count(ctx->device));
            auto go = [&](auto* kernel) {
                return launch(kernel, d, rows->nrow, ctx->st, (const T*)rows->x, rows->nrow, rows->ncol, rows->ld, *teacher, temperature,
                              scale, row_weight_dev, (T*)grad_dev, ld_grad, (W*)row_loss_dev, (int)d.team, (int)d.slice);
            };
            HXC(d.nt == 32 ? go(distill_kernel<T, 32, false>) : d.parts > 1 ? go(distill_kernel<T, 512, true>)
                : d.nt == 128 ? go(distill_kernel<T, 128, false>) : go(distill_kernel<T, 512, false>));
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

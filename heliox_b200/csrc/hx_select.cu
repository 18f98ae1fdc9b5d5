// hx_select.cu -- operators over readout rows that select: a teacher's top
// logits, and sampled choices.
//
// A team keeps a row (or its blocks' slices of it) in shared memory.  Neither
// operator sorts the row: a histogram narrows it down to a handful of
// candidates, which are gathered and put in order.
#include "hx_readout.cuh"

namespace {

using namespace hxr;

using u64 = unsigned long long;

constexpr int kWide = 256;  // threads of a block that has a row, or a slice of one, to itself (short rows: 128)
template <typename T>
constexpr int kWides = sizeof(T) == 8 ? 2 : 3;  // such blocks on an SM, where their shared memory lets them


// What a team needs besides the row, in its leading block's shared memory.
template <typename K>
struct Bag {   // candidates
    K* key;
    int* pos;
    int* count;
    int cap;
};
// Distances d = largest - x >= 0 are counted in bins from below 2^-16 to above
// 2^16: 32 of an octave for a block, 16 for a warp, which has fewer readouts.
template <int NT>
constexpr int kBins = NT == 32 ? 512 : 1024;
template <int NT>
constexpr int kMantissa = NT == 32 ? 4 : 5;  // bits of a distance's mantissa that number its bin
template <int NT>
__device__ __forceinline__ int bin_of(float d) {
    return min(max((int)(__float_as_uint(d) >> (23 - kMantissa<NT>)) - (111 << kMantissa<NT>), 0), kBins<NT> - 1);
}
template <int NT>
__device__ __forceinline__ float bin_end(int b) {
    return b >= kBins<NT> - 1 ? INFINITY : __uint_as_float((unsigned)((111 << kMantissa<NT>) + 1 + b) << (23 - kMantissa<NT>));
}
template <typename W>
__device__ __forceinline__ float distance(W top, W x) {  // also where both are +inf
    return x == top ? 0.0f : (float)(top - x);
}

// whether one candidate comes before another (without branches)
__device__ __forceinline__ bool before(u64 ka, int pa, u64 kb, int pb) { return (ka > kb) | ((ka == kb) & (pa < pb)); }
__device__ __forceinline__ bool before(unsigned ka, int pa, unsigned kb, int pb) {
    return ((u64)ka << 32 | (unsigned)~pa) > ((u64)kb << 32 | (unsigned)~pb);
}

__device__ __forceinline__ u64 scan(u64 v, int lane) {  // inclusive, over a warp
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 a = __shfl_up_sync(~0u, v, o);
        if (lane >= o) v += a;
    }
    return v;
}

// The larger of two; NaN where one is NaN (fp64: b where a is NaN).
__device__ __forceinline__ double larger_nan(double a, double b) { return b > a ? b : a; }
__device__ __forceinline__ float larger_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// The largest of a vector's elements, NaN where one is NaN (but not in fp64): 16-bit types two at a time.
__device__ __forceinline__ double of_vector(const Vec<double>& x) { return larger_nan(x.e[0], x.e[1]); }
__device__ __forceinline__ float of_vector(const Vec<float>& x) {
    return larger_nan(larger_nan(x.e[0], x.e[1]), larger_nan(x.e[2], x.e[3]));
}
__device__ __forceinline__ float of_vector(const Vec<__half>& x) {
    const __half2* p = (const __half2*)x.e;
    const __half2 m = __hmax2_nan(__hmax2_nan(p[0], p[1]), __hmax2_nan(p[2], p[3]));
    return larger_nan(__low2float(m), __high2float(m));
}
__device__ __forceinline__ float of_vector(const Vec<__nv_bfloat16>& x) {
    const __nv_bfloat162* p = (const __nv_bfloat162*)x.e;
    const __nv_bfloat162 m = __hmax2_nan(__hmax2_nan(p[0], p[1]), __hmax2_nan(p[2], p[3]));
    return larger_nan(__low2float(m), __high2float(m));
}

// The row's largest readout, and whether a readout is NaN (odd 1) or +inf (odd 2; also 1 alone where one is NaN).
template <typename W>
struct Top {
    W mx;
    int odd;
};
template <typename T, typename G>
__device__ __forceinline__ Top<typename Ty<T>::W> largest(G& team, const Slice<T>& sl, int v0, int v1, int lane) {
    using W = typename Ty<T>::W;
    W mx = -INFINITY;
    bool fine = true;
#pragma unroll 4
    for (int v = v0 + lane; v < v1; v += 32) {
        const Vec<T> x = sl.get(v);
        if constexpr (sizeof(W) == 8) {
            fine &= (x.e[0] == x.e[0]) & (x.e[1] == x.e[1]);
            mx = larger(mx, larger(x.e[0], x.e[1]));  // one step of the dependent chain a vector
        } else {
            mx = larger_nan(mx, of_vector(x));
        }
    }
    Top<W> t{mx, (mx == mx && fine ? 0 : 1) | (mx == (W)INFINITY ? 2 : 0)};
    if (mx != mx) t.mx = -INFINITY;
    const auto op = [](Top<W> a, Top<W> b) { return Top<W>{larger(a.mx, b.mx), a.odd | b.odd}; };
    t = team.across(team.reduce(t, op), op);
    return t;
}

// ---------------------------------------------------------------- the k largest
//
// The k-th largest of the maxima of at least 2 k groups of readouts is a lower
// bound of the k-th largest readout, and few readouts besides the k reach it
// (1.15 k of them where the groups are 4 k).  The maxima are counted by their
// distance from the largest; what is as near as the bin that the k-th falls
// into is gathered.

// Measured (B200): 4000 x 10000 fp64, k 64, with log-sum-exp: 155 us (2.1 TB/s;
// 74 candidates a row); 1024 x 32000 fp16, k 100: 45 us; 8001 x 302 fp64, a warp
// a row: 28 us.  Bound by the latency of the passes over shared memory, with two
// to three rows an SM.  Bins of an eighth of an octave let in more candidates
// than the list holds where a few readouts stand far above the others (5000
// columns: 189 us for 1184 rows, 55 with a thirty-second).  So do these where one
// stands 95 mV above a bulk of sd 2.5 mV: 8000 x 3000, k 64, 0.9 ms against 0.19,
// by find_border().

// Each lane's vectors in groups; each group's maximum is counted in the
// leading block's histogram.  f(vector) sees every vector.
template <typename T, typename G, typename F>
__device__ __forceinline__ void count_groups(G& team, const Slice<T>& sl, int v0, int v1, int lane, int ncol, int k,
                                             typename Ty<T>::W top, unsigned* hist, F f) {
    using W = typename Ty<T>::W;
    constexpr int VEC = Ty<T>::VEC;
    unsigned* const h = team.of(hist, 0);
    if (ncol < 2 * k * VEC) {  // too few vectors: every readout is a group
        for (int v = v0 + lane; v < v1; v += 32) {
            const Vec<T> x = sl.get(v);
            f(x);
#pragma unroll
            for (int u = 0; u < VEC; u++) {
                const W y = wide(x.e[u]);
                if (y > (W)-INFINITY) atomicAdd(h + bin_of<G::NT>(distance(top, y)), 1u);
            }
        }
        return;
    }
    const int per = max(1, ncol / (4 * k * VEC));  // vectors of a group
    for (int v = v0 + lane; v < v1;) {
        W g = -INFINITY;
        const int end = min(v1, v + 32 * per);
#pragma unroll 4
        for (; v < end; v += 32) {
            const Vec<T> x = sl.get(v);
            f(x);
            g = larger(g, of_vector(x));
        }
        if (g > (W)-INFINITY) atomicAdd(h + bin_of<G::NT>(distance(top, g)), 1u);
    }
}

// The bin that the k-th group falls into (the last bin where there are fewer), by the leading block's threads.
template <typename G>
__device__ __forceinline__ void find_bin(G& team, const unsigned* hist, int k, int* bin) {
    constexpr int PER = kBins<G::NT> / G::NT;
    static_assert(PER * G::NT == kBins<G::NT>, "");
    const int t = team.t;
    unsigned c[PER], s = 0;
#pragma unroll
    for (int i = 0; i < PER; i++) s += c[i] = hist[t * PER + i];
    unsigned a = (unsigned)scan(s, t & 31) - s;  // in the bins before, of this warp
    if constexpr (G::NW > 1) {
        unsigned* w = (unsigned*)team.notes();
        if ((t & 31) == 31) w[t >> 5] = a + s;
        team.sync_block();
        for (int i = 0; i < (t >> 5); i++) a += w[i];
    }
#pragma unroll
    for (int i = 0; i < PER; i++) {
        if (a < (unsigned)k && a + c[i] >= (unsigned)k) *bin = t * PER + i;
        a += c[i];
    }
}

// Puts every readout of this block's slice for which want(value) into the
// leading block's bag; vectors for which maybe(vector) is false have none.
// Hits are rare: lanes first mark the vectors that may have some, then count
// theirs, and the warp takes its places in the bag with one atomic addition.
template <typename T, typename G, typename K, typename P, typename F>
__device__ __forceinline__ void gather(G& team, const Slice<T>& sl, int v0, int v1, int lane, const Bag<K>& bag, P maybe, F want) {
    constexpr int VEC = Ty<T>::VEC;
    K* const key = team.of(bag.key, 0);
    int *const pos = team.of(bag.pos, 0), *const count = team.of(bag.count, 0);
    const int at = sl.first - sl.phase;
    for (int first = v0; first < v1; first += 32 * 32) {
        const int mine = min(32, (v1 - first - lane + 31) >> 5);  // vectors of this lane
        unsigned marks = 0;
#pragma unroll 4
        for (int i = 0; i < mine; i++)
            if (maybe(sl.get(first + lane + 32 * i))) marks |= 1u << i;
        if (!__any_sync(~0u, marks)) continue;
        int hits = 0;
        for (unsigned m = marks; m; m &= m - 1) {
            const T* const x = sl.e + (first + lane + 32 * (__ffs(m) - 1)) * VEC;
#pragma unroll 2
            for (int u = 0; u < VEC; u++) hits += want(wide(x[u]));
        }
        int upto = hits;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int h = __shfl_up_sync(~0u, upto, o);
            if (lane >= o) upto += h;
        }
        int p = 0;
        if (lane == 31) p = atomicAdd(count, upto);
        p = __shfl_sync(~0u, p, 31) + upto - hits;
        for (unsigned m = hits ? marks : 0u; m; m &= m - 1) {
            const int v = first + lane + 32 * (__ffs(m) - 1);
            const T* const x = sl.e + v * VEC;
#pragma unroll 1
            for (int u = 0; u < VEC; u++) {
                const auto y = wide(x[u]);
                if (want(y)) {
                    if (p < bag.cap) {
                        key[p] = key_of(y);
                        pos[p] = at + v * VEC + u;
                    }
                    p++;
                }
            }
        }
    }
}
// Those in the bins up to b.  What reaches the least value of these bins, or
// comes a rounding short of it, is taken: a few too many do no harm.
template <typename T, typename G, typename K>
__device__ __forceinline__ void gather_bins(G& team, const Slice<T>& sl, int v0, int v1, int lane, const Bag<K>& bag, int b, typename Ty<T>::W top) {
    using W = typename Ty<T>::W;
    W least = top - (W)bin_end<G::NT>(b) * (W)1.000001;
    const W lowest = sizeof(W) == 8 ? (W)-1.7976931348623157e308 : (W)-3.4028234663852886e38f;
    if (b >= kBins<G::NT> - 1 || !(least > lowest)) least = lowest;
    if (top == (W)INFINITY && b < kBins<G::NT> - 1) least = top;
    gather<T>(team, sl, v0, v1, lane, bag, [&](const Vec<T>& x) {
        if constexpr (sizeof(W) == 8) return (bool)((x.e[0] >= least) | (x.e[1] >= least));
        return of_vector(x) >= least;
    }, [&](W y) { return y >= least; });
}

// The n candidates in order: put(rank, key, position) for the first `want`, by
// one block's threads.  Few are ranked by comparing each with all others (with
// ranks, kRanks zeroed numbers, by all threads of a block), more by a bitonic
// network in place.
constexpr int kRanks = 128;
template <typename G, typename K, typename F>
__device__ __forceinline__ void in_order(G& team, const Bag<K>& bag, int n, int want, int* ranks, F put) {
    constexpr int NT = G::NT;
    const int t = team.t;
    if constexpr (NT > 32) {
        if (ranks && n > 32 && n <= kRanks) {  // each by several threads
            int p2 = 64;
            while (p2 < n) p2 <<= 1;
            const int j = t & (p2 - 1), groups = NT / p2, each = (n + groups - 1) / groups;
            const int l0 = (t / p2) * each, l1 = min(l0 + each, n);
            K k = 0;
            int p = 0, r = 0;
            if (j < n) {
                k = bag.key[j];
                p = bag.pos[j];
#pragma unroll 8
                for (int l = l0; l < l1; l++) r += before(bag.key[l], bag.pos[l], k, p);
                if (r) atomicAdd(ranks + j, r);
            }
            team.sync_block();
            if (t < n && ranks[t] < want) put(ranks[t], k, p);
            return;
        }
    }
    if (n <= (NT == 32 ? 64 : 128)) {
        for (int j = t; j < n; j += NT) {
            const K k = bag.key[j];
            const int p = bag.pos[j];
            int r = 0;
#pragma unroll 4
            for (int l = 0; l < n; l++) r += before(bag.key[l], bag.pos[l], k, p);
            if (r < want) put(r, k, p);
        }
        return;
    }
    int p2 = 1;
    while (p2 < n) p2 <<= 1;  // at most the bag's room, which is a power of two
    for (int j = n + t; j < p2; j += NT) {
        bag.key[j] = 0;
        bag.pos[j] = INT_MAX;
    }
    for (int w = 2; w <= p2; w <<= 1) {
        for (int d = w >> 1; d > 0; d >>= 1) {
            team.sync_block();
            for (int i = t; i < p2 / 2; i += NT) {
                const int j = 2 * i - (i & (d - 1)), o = j + d;
                const K a = bag.key[j], b = bag.key[o];
                const int pa = bag.pos[j], pb = bag.pos[o];
                if (before(a, pa, b, pb) != ((j & w) == 0)) {
                    bag.key[j] = b;
                    bag.key[o] = a;
                    bag.pos[j] = pb;
                    bag.pos[o] = pa;
                }
            }
        }
    }
    team.sync_block();
    for (int j = t; j < min(n, want); j += NT) put(j, bag.key[j], bag.pos[j]);
}

// ---------------------------------------------------------------- rows of many equal readouts
//
// Where more readouts share a border's bin than the bag holds (resting cells
// with one voltage, 16-bit logits), the leading block finds the border from
// global memory: at once if all of them are equal, else by 8-bit digits of the
// keys from the first that differs.

struct Border {
    u64 key, above;  // the border's key; the measure of everything before it
};
// The border at which the running measure of the readouts in(value) first
// exceeds target, `above` being the measure of everything before them.
template <typename T, typename G, typename I, typename M>
__device__ Border find_border(G& team, const T* __restrict__ x, int n, u64* hist, u64 target, u64 above, I in, M measure) {
    using K = typename Ty<T>::K;
    constexpr int NT = G::NT;
    const int t = team.t;
    struct Span {
        u64 lo, hi;
    } s{~0ull, 0};
    for (int i = t; i < n; i += NT) {
        const auto v = wide(x[i]);
        if (!in(v)) continue;
        const u64 k = key_of(v);
        s.lo = min(s.lo, k);
        s.hi = max(s.hi, k);
    }
    s = team.reduce(s, [](Span a, Span b) { return Span{min(a.lo, b.lo), max(a.hi, b.hi)}; });
    if (s.lo == s.hi) return Border{s.lo, above};
    int shift = max(64 - __clzll((long long)(s.lo ^ s.hi)) - 8, 0);
    u64 mask = shift + 8 >= 64 ? 0 : ~0ull << (shift + 8), prefix = s.hi & mask;
    int* const digit = (int*)(hist + 256);
    for (;;) {
        team.sync_block();
        for (int b = t; b < 256; b += NT) hist[b] = 0;
        team.sync_block();
        for (int i = t; i < n; i += NT) {
            const auto v = wide(x[i]);
            if (!in(v)) continue;
            const u64 k = (u64)(K)key_of(v);
            if ((k & mask) != prefix) continue;
            const u64 m = measure(v);
            if (m) atomicAdd(hist + ((k >> shift) & 255), m);
        }
        team.sync_block();
        if (t == 0) {
            u64 a = above;
            int d = 255;
            while (d > 0 && a + hist[d] <= target) a += hist[d--];
            *digit = d;
            hist[257] = a;
        }
        team.sync_block();
        above = hist[257];
        prefix |= (u64)*digit << shift;
        mask |= 255ull << shift;
        if (shift == 0) return Border{prefix, above};
        shift = max(shift - 8, 0);
    }
}
constexpr int kSlowBytes = 258 * 8;

// take(position, number) for the first `want` readouts with this key, by position.
template <typename T, typename G, typename F>
__device__ void first_of_key(G& team, const T* __restrict__ x, int n, u64 key, u64 want, F take) {
    constexpr int NT = G::NT;
    const int t = team.t, lane = t & 31;
    int* const w = (int*)team.notes();
    u64 seen = 0;
    for (int i0 = 0; i0 < n && seen < want; i0 += NT) {
        const int i = i0 + t;
        const bool hit = i < n && (u64)key_of(wide(x[i])) == key;
        const unsigned b = __ballot_sync(~0u, hit);
        u64 at = seen + __popc(b & ((1u << lane) - 1));
        int all = __popc(b);
        if constexpr (G::NW > 1) {
            team.sync_block();
            if (lane == 0) w[t >> 5] = all;
            team.sync_block();
            all = 0;
            for (int j = 0; j < G::NW; j++) {
                if (j < (t >> 5)) at += w[j];
                all += w[j];
            }
        }
        if (hit && at < want) take(i, at);
        seen += all;
    }
    team.sync_block();
}

// ---------------------------------------------------------------- top logits

template <int NT>
constexpr int kCountBytes = kBins<NT> * 4 > kSlowBytes ? kBins<NT> * 4 : kSlowBytes;
size_t top_extra(int nt, int cap, size_t key) { return (nt == 32 ? kCountBytes<32> : kCountBytes<kWide>) + 16 + (size_t)cap * (key + 4); }
int top_cap(int k) {  // room for the candidates: a power of two
    int c = 128;
    while (c < 3 * k && c < 2 * HX_READOUT_MAX_K) c *= 2;
    return c;
}

template <typename T, int NT, bool CL>
__global__ void __launch_bounds__(NT == 32 ? 32 * kWarpRows : NT, NT == kWide ? kWides<T> : 6)
    top_kernel(const T* __restrict__ xs, int nrow, int ncol, long long ld, int k, Heat heat, int* __restrict__ idx, T* __restrict__ val,
               typename Ty<T>::W* __restrict__ lse, int cap, int team_bytes, int slice_bytes) {
    using W = typename Ty<T>::W;
    using K = typename Ty<T>::K;
    constexpr int NW = NT / 32;
    extern __shared__ __align__(16) char smem[];
    char* const mine = smem + (NT == 32 ? (threadIdx.x >> 5) * team_bytes : 0);
    Team<NT, CL, false> team(mine);
    const int t = team.t, lane = t & 31, warp = NT == 32 ? 0 : t >> 5;
    T* const row_mem = (T*)(mine + kRedBytes);
    char* const extra = mine + kRedBytes + slice_bytes;
    unsigned* const hist = (unsigned*)extra;  // and the digits of find_border()
    int* const count = (int*)(extra + kCountBytes<NT>);
    int* const bin = count + 1;
    const Bag<K> bag{(K*)(extra + kCountBytes<NT> + 16), (int*)((K*)(extra + kCountBytes<NT> + 16) + cap), count, cap};
    const bool lead = team.part == 0;
    const long long step = team.row_step();
    long long row = team.first_row();
    if (row >= nrow) return;
    const auto ask = [&](long long r) {
        const Slice<T> s(row_mem, xs + r * ld, ncol, team.part, team.parts);
        s.load(s.template run<NW>(warp), s.template run<NW>(warp + 1), lane);
    };
    const auto prefetch = [&](long long r) {
        const Slice<T> s(row_mem, xs + r * ld, ncol, team.part, team.parts);
        if (lane == 0) s.prefetch(s.template run<NW>(warp), s.template run<NW>(warp + 1));
    };
    ask(row);
    for (;;) {
        const T* const x = xs + row * ld;
        const Slice<T> sl(row_mem, x, ncol, team.part, team.parts);
        const int v0 = sl.template run<NW>(warp), v1 = sl.template run<NW>(warp + 1);
        const long long next = row + step;
        for (int b = t; b < kBins<NT>; b += NT) hist[b] = 0;
        if (t == 0) {
            *count = 0;
            *bin = kBins<NT> - 1;
        }
        wait_copies();
        __syncwarp();  // the lanes' copies are the warp's from here on
        if (next < nrow) prefetch(next);
        const Top<W> top = largest<T>(team, sl, v0, v1, lane);
        if (NT == 32) __syncwarp();
        int* const out_idx = idx + row * k;
        T* const out_val = val + row * k;
        int n = 0;
        const bool odd = top.odd & 1;
        if (!odd && top.mx > (W)-INFINITY) {
            double sum = 0;
            if (lse) {
                const auto ex = scaler(top.mx, heat, team.table());
                W part = 0;
                count_groups<T>(team, sl, v0, v1, lane, ncol, k, top.mx, hist, [&](const Vec<T>& xv) {
#pragma unroll
                    for (int q = 0; q < Ty<T>::VEC; q++) part += ex(wide(xv.e[q]));
                });
                sum = team.reduce((double)part, [](double a, double b) { return a + b; });
            } else {
                count_groups<T>(team, sl, v0, v1, lane, ncol, k, top.mx, hist, [](const Vec<T>&) {});
            }
            sum = team.across(sum, [](double a, double b) { return a + b; });
            if (!CL) team.sync_block();
            if (lead) find_bin(team, hist, k, bin);
            team.sync_all();
            const int b = *team.of(bin, 0);
            for (int j = t; j < kRanks; j += NT) hist[j] = 0;  // ranks from here on
            gather_bins<T>(team, sl, v0, v1, lane, bag, b, top.mx);
            team.sync_all();
            if (next < nrow) ask(next);
            if (lead) {
                n = *count;
                if (n > cap) {
                    // the bin's readouts are too many: what is before its border, and the first of the border's
                    const Border br = find_border(team, x, ncol, (u64*)hist, (u64)(k - 1), 0ull, [](W y) { return y > (W)-INFINITY; }, [](W) { return 1ull; });
                    team.sync_block();
                    if (t == 0) *count = 0;
                    team.sync_block();
                    for (int i = t; i < ncol; i += NT) {
                        const W y = wide(x[i]);
                        if (y > (W)-INFINITY && (u64)key_of(y) > br.key) {
                            const int p = atomicAdd(count, 1);
                            bag.key[p] = key_of(y);
                            bag.pos[p] = i;
                        }
                    }
                    first_of_key(team, x, ncol, br.key, (u64)k - br.above, [&](int i, u64 at) {
                        bag.key[br.above + at] = (K)br.key;
                        bag.pos[br.above + at] = i;
                    });
                    n = k;
                    for (int j = t; j < kRanks; j += NT) hist[j] = 0;
                    team.sync_block();
                }
                in_order(team, bag, n, k, (int*)hist, [&](int r, K key, int p) {
                    out_idx[r] = p;
                    out_val[r] = narrow<T>(value_of(key));
                });
                if (lse && t == 0) lse[row] = top.mx == (W)INFINITY ? (W)INFINITY : (W)((double)top.mx * heat.inv + log(sum));
            }
        } else {
            if (next < nrow) ask(next);
            if (lse && lead && t == 0) lse[row] = odd ? (W)NAN : (W)-INFINITY;
        }
        if (lead)
            for (int j = min(n, k) + t; j < k; j += NT) {
                out_idx[j] = -1;
                out_val[j] = narrow<T>(odd ? (W)NAN : (W)-INFINITY);
            }
        if (next >= nrow) break;
        row = next;
        team.sync_block();
    }
    if constexpr (CL) team.sync_all();
}

// ---------------------------------------------------------------- sampling
//
// Every weight e = exp((x - max) / T) counts as the whole number of 2^-bits
// nearest to it, its mass: sums of masses are exact, so that no result depends
// on the order or the number of the threads, and rounding moves a border by no
// more than n / 2 units.  In the order of descending readouts top_k, top_p and
// min_p each keep a first run, so that the shortest of the three is known by
// its mass, and the choice is the first readout whose running mass exceeds
// u times that.
//
// Measured (B200): 2000 x 10000 fp64, top_p: 140 us (two gathers; one without
// top_p); 64 x 32000 fp32 with rules of their own: 13 us, a row two blocks;
// 8001 x 302 fp64, a warp a row: 33 us.  Ranking a whole bin's candidates (208
// of 10000 columns) instead of one of its 128 parts took 225 us.
//
// With top_k the candidates are the k largest, in order.  Without it the
// masses are summed up in bins of a sixteenth of an octave (the whole part of
// the exponential's argument); a running mass is first followed over the bins
// and then over the readouts of one bin, gathered and put in order.

struct Rule {
    double temperature;
    int top_k;
    double top_p, min_p;
};
__device__ __forceinline__ Rule clean(const hx_sample_rule& r, int ncol) {
    Rule o;
    const bool greedy = r.temperature < 1e-30;
    o.temperature = greedy ? 1.0 : r.temperature < 1e30 ? r.temperature : 1e30;
    o.top_k = greedy ? 1 : r.top_k >= 1.0 ? (r.top_k < (double)ncol ? (int)r.top_k : ncol) : ncol;
    o.top_p = r.top_p < 1.0 ? larger(0.0, r.top_p) : 1.0;
    o.min_p = r.min_p > 0.0 ? (r.min_p < 1.0 ? r.min_p : 1.0) : 0.0;
    return o;
}

// Weights and masses of one row.
struct Scale {
    double m, c, unit, least;  // largest readout; 16 log2(e) / T; 2^bits; arguments below `least` have no mass
    const int2* pow16;
    // 2^(s / 16), s = 16 (x - m) log2(e) / T = k + f
    __device__ __forceinline__ double arg(double x) const { return (x - m) * c; }
    static __device__ __forceinline__ double rounded(double s) { return s + 6755399441055744.0; }
    __device__ __forceinline__ double weight(double s) const {
        const double y = rounded(s);
        const int k = __double2loint(y);
        const double f = s - (y - 6755399441055744.0);
        double q = 0x1.430a1d08ec681p-37;
        q = __fma_rn(q, f, 0x1.5d897e525c216p-30);
        q = __fma_rn(q, f, 0x1.3b2ab6fb41213p-23);
        q = __fma_rn(q, f, 0x1.c6b08d6f2a289p-17);
        q = __fma_rn(q, f, 0x1.ebfbdff82c590p-11);
        q = __fma_rn(q, f, 0x1.62e42fefa39f3p-5);
        q = q * f;
        const int2 t = pow16[k & 15];
        const double p = __hiloint2double(t.y + (k << 16), t.x);
        return __fma_rn(p, q, p);
    }
    // e 2^bits to the nearest whole number: the low bits of its sum with 2^52
    __device__ __forceinline__ u64 mass_of(double e) const {
        return (u64)__double_as_longlong(__fma_rn(e, unit, 4503599627370496.0)) - 0x4330000000000000ull;
    }
    __device__ __forceinline__ u64 mass(double x) const {
        const double s = arg(x);
        return s > least ? mass_of(weight(s)) : 0ull;
    }
    __device__ __forceinline__ double weight_at(double x) const {
        const double s = arg(x);
        return s > least ? weight(s) : 0.0;
    }
};

constexpr int kParts = 128;  // of a bin, where it has many readouts
constexpr int kMassBins = 896;  // 16 * (52 + 2) and more
template <int NT>
constexpr int kCoarse = NT == 32 ? 2 : 0;  // a warp's bins are four times as wide
template <int NT>
constexpr int kRowBins = kMassBins >> kCoarse<NT>;

template <int NT>
constexpr int kMassBytes = kRowBins<NT> * 8 > kCountBytes<NT> ? kRowBins<NT> * 8 : kCountBytes<NT>;
static_assert(128 * (8 + 4 + 4 + 4) >= kSlowBytes, "find_border() has the candidates' place");
size_t sample_extra(int nt, int cap, size_t key) {
    const size_t lists = (size_t)cap * (key + 4) + (size_t)cap * (8 + 4);
    return nt == 32 ? kMassBytes<32> + 64 + lists : kMassBytes<kWide> + 64 + lists + (size_t)cap * (key + 4) + kParts * 8;
}

// Adds a mass to a bin (two words) in shared memory: the carry goes with the high word.
__device__ __forceinline__ void add_mass(unsigned at, u64 m) {
    const unsigned lo = (unsigned)m;
    unsigned was;
    asm volatile("atom.shared.add.u32 %0, [%1], %2;" : "=r"(was) : "r"(at), "r"(lo) : "memory");
    asm volatile("red.shared.add.u32 [%0], %1;" ::"r"(at + 4), "r"((unsigned)(m >> 32) + (was + lo < was ? 1u : 0u)) : "memory");
}

// The first of n masses in order (running sums cum) whose running mass exceeds target; by a warp.
__device__ __forceinline__ int past(const u64* cum, int n, u64 target, int lane) {
    int c = 0;
    for (int j0 = 0; j0 < n; j0 += 32) {
        const unsigned b = __ballot_sync(~0u, j0 + lane < n && cum[j0 + lane] <= target);
        c += __popc(b);
        if (b != ~0u) break;
    }
    return min(c, n - 1);
}

template <typename T, int NT, bool CL>
__global__ void __launch_bounds__(NT == 32 ? 32 * kWarpRows : NT, NT == kWide ? kWides<T> : 6)
    sample_kernel(const T* __restrict__ xs, int nrow, int ncol, long long ld, hx_sample_rule rule, const hx_sample_rule* __restrict__ rules,
                  const double* __restrict__ us, int bits, int* __restrict__ idx, typename Ty<T>::W* __restrict__ logp, int cap,
                  int team_bytes, int slice_bytes) {
    using W = typename Ty<T>::W;
    using K = typename Ty<T>::K;
    using G = Team<NT, CL, false>;
    constexpr int NW = NT / 32, NB = kRowBins<NT>, PER = (NB + NT - 1) / NT;
    extern __shared__ __align__(16) char smem[];
    char* const mine = smem + (NT == 32 ? (threadIdx.x >> 5) * team_bytes : 0);
    G team(mine);
    const int t = team.t, lane = t & 31, warp = NT == 32 ? 0 : t >> 5;
    T* const row_mem = (T*)(mine + kRedBytes);
    char* const extra = mine + kRedBytes + slice_bytes;
    unsigned* const hist = (unsigned*)extra;  // counting bins, or
    uint2* const bins = (uint2*)extra;        // masses of the bins (low and high words), then the masses before each, or
    u64* const digits = (u64*)extra;          // of find_border()
    char* const rest = extra + kMassBytes<NT>;
    u64* const found = (u64*)rest;  // [0] mass before the bin, [1] its number, [2] total mass, [3] key of the choice
    int* const count = (int*)(found + 4);
    int* const bin = count + 1;
    int *const choice = count + 2, *const count2 = count + 3;
    u64* const cum = (u64*)(rest + 64);  // running masses of the candidates in order
    const Bag<K> bag{(K*)(cum + cap), (int*)((K*)(cum + cap) + cap), count, cap};
    int* const pos = bag.pos + cap;  // positions in order; keys in order: in cum's place until the masses are
    uint2* const parts = (uint2*)(pos + cap);  // NT > 32: masses of the parts of a bin, and the readouts of one part
    const Bag<K> fine{(K*)(parts + kParts), (int*)((K*)(parts + kParts) + cap), count2, cap};
    const bool lead = team.part == 0;
    const long long step = team.row_step();
    long long row = team.first_row();
    if (row >= nrow) return;
    const auto ask = [&](long long r) {
        const Slice<T> s(row_mem, xs + r * ld, ncol, team.part, team.parts);
        s.load(s.template run<NW>(warp), s.template run<NW>(warp + 1), lane);
    };
    const auto prefetch = [&](long long r) {
        const Slice<T> s(row_mem, xs + r * ld, ncol, team.part, team.parts);
        if (lane == 0) s.prefetch(s.template run<NW>(warp), s.template run<NW>(warp + 1));
    };
    ask(row);
    for (;;) {
        const T* const x = xs + row * ld;
        const Slice<T> sl(row_mem, x, ncol, team.part, team.parts);
        const int v0 = sl.template run<NW>(warp), v1 = sl.template run<NW>(warp + 1);
        const long long next = row + step;
        const hx_sample_rule given = rules ? rules[row] : rule;
        double u = us[row];
        const Rule r = clean(given, ncol);
        const bool few = r.top_k < ncol && r.top_k <= cap / 2, by_mass = r.top_k >= ncol;
        for (int b = t; b < NB * 2 || b < kBins<NT>; b += NT) hist[b] = 0;
        if (t == 0) {
            *count = 0;
            *bin = kBins<NT> - 1;
        }
        wait_copies();
        __syncwarp();  // the lanes' copies are the warp's from here on
        if (next < nrow) prefetch(next);
        const Top<W> top = largest<T>(team, sl, v0, v1, lane);
        if (NT == 32) __syncwarp();
        const bool odd = top.odd || given.temperature != given.temperature;
        if (odd || top.mx == (W)-INFINITY) {
            if (next < nrow) ask(next);
            if (lead && t == 0) {
                idx[row] = odd ? -2 : -1;
                if (logp) logp[row] = odd ? (W)NAN : (W)-INFINITY;
            }
        } else {
            const double inv = 1.0 / r.temperature;
            Scale sc;
            sc.m = (double)top.mx;
            sc.c = 16.0 * 1.4426950408889634 * inv;
            sc.unit = __hiloint2double((1023 + bits) << 20, 0);
            sc.least = -16.0 * (bits + 1.5);
            sc.pow16 = (const int2*)team.table();
            u = u > 0.0 ? u : 0.0;
            const auto share = [](double f, u64 total) {  // floor of f times total, below total
                const double w = floor(f * (double)total);
                const u64 v = w > 0.0 ? (u64)w : 0ull;
                return f >= 1.0 || v >= total ? total - 1 : v;
            };
            const auto write = [&](int p, double v, u64 total) {
                idx[row] = p;
                if (logp) logp[row] = (W)((v - sc.m) * inv - log((double)total / sc.unit));
            };
            // mass of the readouts of weight min_p and more
            const auto floor_mass = [&](auto each) {
                u64 s = 0;
                each([&](double y) {
                    const double e = sc.weight_at(y);
                    if (e >= r.min_p) s += sc.mass_of(e);
                });
                return s;
            };
            if (few) {
                count_groups<T>(team, sl, v0, v1, lane, ncol, r.top_k, top.mx, hist, [](const Vec<T>&) {});
                team.sync_all();
                if (lead) find_bin(team, hist, r.top_k, bin);
                team.sync_all();
                const int b = *team.of(bin, 0);
                for (int j = t; j < kRanks; j += NT) hist[j] = 0;  // ranks from here on
                gather_bins<T>(team, sl, v0, v1, lane, bag, b, top.mx);
                team.sync_all();
                if (next < nrow) ask(next);
                if (lead) {
                    int n = *count;
                    if (n > cap) {
                        const Border br = find_border(team, x, ncol, digits, (u64)(r.top_k - 1), 0ull, [](W y) { return y > (W)-INFINITY; }, [](W) { return 1ull; });
                        team.sync_block();
                        if (t == 0) *count = 0;
                        team.sync_block();
                        for (int i = t; i < ncol; i += NT) {
                            const W y = wide(x[i]);
                            if (y > (W)-INFINITY && (u64)key_of(y) > br.key) {
                                const int p = atomicAdd(count, 1);
                                bag.key[p] = key_of(y);
                                bag.pos[p] = i;
                            }
                        }
                        first_of_key(team, x, ncol, br.key, (u64)r.top_k - br.above, [&](int i, u64 at) {
                            bag.key[br.above + at] = (K)br.key;
                            bag.pos[br.above + at] = i;
                        });
                        n = r.top_k;
                        for (int j = t; j < kRanks; j += NT) hist[j] = 0;
                        team.sync_block();
                    }
                    in_order(team, bag, n, r.top_k, (int*)hist, [&](int j, K key, int p) {
                        cum[j] = (u64)key;
                        pos[j] = p;
                    });
                    n = min(n, r.top_k);
                    team.sync_block();
                    if (t < 32) {  // one warp: running masses, the cuts, the choice
                        u64 a = 0, atleast = 0;
                        double pick = 0;
                        for (int j0 = 0; j0 < n; j0 += 32) {
                            const int j = j0 + lane;
                            double e = 0;
                            if (j < n) e = sc.weight_at((double)value_of((K)cum[j]));
                            const u64 s = a + scan(e > 0.0 ? sc.mass_of(e) : 0ull, lane);
                            const unsigned keep = __ballot_sync(~0u, j < n && e >= r.min_p);
                            if (keep) atleast = __shfl_sync(~0u, s, 31 - __clz(keep));
                            if (j < n) cum[j] = s;
                            a = __shfl_sync(~0u, s, 31);
                        }
                        __syncwarp();
                        u64 total = a;
                        if (r.top_p < 1.0) {
                            const double w = ceil(r.top_p * (double)total);
                            const u64 want = w < 1.0 ? 1ull : min((u64)w, total);
                            total = cum[past(cum, n, want - 1, lane)];
                        }
                        if (r.min_p > 0.0) total = min(total, atleast);
                        const int at = past(cum, n, share(u, total), lane);
                        if (lane == 0) {
                            pick = (double)wide(x[pos[at]]);
                            write(pos[at], pick, total);
                        }
                    }
                }
            } else if (by_mass) {
                u64 atleast = 0;
                const unsigned bins_at = (unsigned)__cvta_generic_to_shared(bins);
#pragma unroll 2
                for (int v = v0 + lane; v < v1; v += 32) {
                    const Vec<T> xv = sl.get(v);
#pragma unroll
                    for (int q = 0; q < Ty<T>::VEC; q++) {
                        const double s = sc.arg((double)wide(xv.e[q]));
                        if (s > sc.least) {
                            const double e = sc.weight(s);
                            const u64 m = sc.mass_of(e);
                            add_mass(bins_at + (-__double2loint(Scale::rounded(s)) >> kCoarse<NT>) * 8, m);
                            if (r.min_p > 0.0 && e >= r.min_p) atleast += m;
                        }
                    }
                }
                if (r.min_p > 0.0) {
                    const auto op = [](u64 a, u64 b) { return a + b; };
                    atleast = team.across(team.reduce(atleast, op), op);
                }
                team.sync_all();
                if (lead) {  // masses before each bin
                    u64 m[PER], s = 0;
#pragma unroll
                    for (int i = 0; i < PER; i++) {
                        const int b = t * PER + i;
                        m[i] = 0;
                        if (b < NB)
                            for (int p = 0; p < team.parts; p++) {
                                const uint2 w = *team.of(bins + b, p);
                                m[i] += (u64)w.y << 32 | w.x;
                            }
                        s += m[i];
                    }
                    u64 a = scan(s, lane) - s;
                    if constexpr (NW > 1) {
                        u64* const w = (u64*)team.notes();
                        if (lane == 31) w[warp] = a + s;
                        team.sync_block();
                        for (int i = 0; i < warp; i++) a += w[i];
                    } else {
                        __syncwarp();
                    }
#pragma unroll
                    for (int i = 0; i < PER; i++) {
                        const int b = t * PER + i;
                        if (b < NB) *(u64*)(bins + b) = a;
                        a += m[i];
                    }
                    if (t == NT - 1) found[2] = a;
                    team.sync_block();
                }
                // the readout at which the running mass first exceeds target: its key, position and running mass
                struct At {
                    u64 key, through;
                    int pos;
                };
                const auto follow = [&](u64 target, bool last) {
                    At at{0, 0, 0};
                    if (lead) {
                        for (int b = t; b < NB; b += NT) {
                            const u64 a = *(u64*)(bins + b), e = b + 1 < NB ? *(u64*)(bins + b + 1) : found[2];
                            if (a <= target && target < e) {
                                found[0] = a;
                                *bin = b;
                            }
                        }
                        if (t == 0) *count = 0;
                        if (NW > 1 && t < kParts) parts[t] = make_uint2(0, 0);
                    }
                    team.sync_all();
                    const int b = *team.of(bin, 0);
                    const auto in = [&](W y) {
                        const double s = sc.arg((double)y);
                        return s > sc.least && -__double2loint(Scale::rounded(s)) >> kCoarse<NT> == b;
                    };
                    // every readout of the bin lies between these
                    const double width = (double)(1 << kCoarse<NT>) / sc.c, half = 0.5 / (1 << kCoarse<NT>);
                    const W hi = (W)(sc.m - ((double)b - 1.001 * half) * width), lo = (W)(sc.m - ((double)(b + 1) - 0.999 * half) * width);
                    gather<T>(team, sl, v0, v1, lane, bag,
                              [&](const Vec<T>& xv) {
                                  bool some = false;
#pragma unroll
                                  for (int q = 0; q < Ty<T>::VEC; q++) some |= (wide(xv.e[q]) <= hi) & (wide(xv.e[q]) >= lo);
                                  return some;
                              },
                              [&](W y) { return NW > 1 ? (y <= hi) & (y >= lo) : in(y); });  // a block sorts out the few too many below
                    team.sync_all();
                    if (last && next < nrow) ask(next);
                    if (lead) {
                        int n = *count;
                        u64 above = found[0];
                        Bag<K> list = bag;
                        team.sync_block();
                        if constexpr (NW > 1) {
                            if (n <= cap) {  // by the fraction of the argument: one of kParts parts of the bin
                                const auto part_of = [&](double v) {
                                    const double s = sc.arg(v), y = Scale::rounded(s);
                                    if (!(s > sc.least) || -__double2loint(y) != b) return -1;
                                    return min(max((int)((0.5 - (s - (y - 6755399441055744.0))) * kParts), 0), kParts - 1);
                                };
                                const unsigned parts_at = (unsigned)__cvta_generic_to_shared(parts);
                                for (int j = t; j < n; j += NT) {
                                    const double v = (double)value_of(bag.key[j]);
                                    const int p = part_of(v);
                                    if (p >= 0) add_mass(parts_at + p * 8, sc.mass(v));
                                }
                                team.sync_block();
                                if (t < 32) {
                                    constexpr int P = kParts / 32;
                                    u64 m[P], s = 0;
#pragma unroll
                                    for (int i = 0; i < P; i++) {
                                        const uint2 w = parts[lane * P + i];
                                        s += m[i] = (u64)w.y << 32 | w.x;
                                    }
                                    u64 a = above + scan(s, lane) - s;
#pragma unroll
                                    for (int i = 0; i < P; i++) {
                                        if (a <= target && target < a + m[i]) {
                                            found[0] = a;
                                            *choice = lane * P + i;
                                        }
                                        a += m[i];
                                    }
                                    if (lane == 0) *count2 = 0;
                                }
                                team.sync_block();
                                const int one = *choice;
                                above = found[0];
                                for (int j = t; j < n; j += NT)
                                    if (part_of((double)value_of(bag.key[j])) == one) {
                                        const int p = atomicAdd(count2, 1);
                                        fine.key[p] = bag.key[j];
                                        fine.pos[p] = bag.pos[j];
                                    }
                                team.sync_block();
                                n = *count2;
                                list = fine;
                            }
                        }
                        if (n > cap) {
                            const Border br = find_border(team, x, ncol, cum, target, above, in, [&](W y) { return sc.mass((double)y); });
                            const u64 m = sc.mass((double)value_of((K)br.key)), nth = (target - br.above) / m;
                            first_of_key(team, x, ncol, br.key, nth + 1, [&](int i, u64 j) {
                                if (j == nth) *choice = i;
                            });
                            at.key = br.key;
                            at.through = br.above + (nth + 1) * m;
                            at.pos = *choice;
                        } else {
                            in_order(team, list, n, n, nullptr, [&](int j, K key, int p) {
                                cum[j] = (u64)key;
                                pos[j] = p;
                            });
                            team.sync_block();
                            if (t < 32) {
                                u64 a = above;
                                for (int j0 = 0; j0 < n; j0 += 32) {
                                    const int j = j0 + lane;
                                    const u64 s = a + scan(j < n ? sc.mass((double)value_of((K)cum[j])) : 0ull, lane);
                                    const unsigned over = __ballot_sync(~0u, j < n && s > target);
                                    if (over) {
                                        if (lane == __ffs(over) - 1) {
                                            found[3] = cum[j];
                                            found[0] = s;
                                            *choice = pos[j];
                                        }
                                        break;
                                    }
                                    a = __shfl_sync(~0u, s, 31);
                                }
                            }
                            team.sync_block();
                            at.key = found[3];
                            at.through = found[0];
                            at.pos = *choice;
                        }
                        team.sync_block();
                    }
                    return at;
                };
                u64 total = lead ? found[2] : 0;
                if (r.top_p < 1.0) {
                    const double w = ceil(r.top_p * (double)total);
                    const u64 want = w < 1.0 ? 1ull : min((u64)w, total);
                    total = follow(want - 1, false).through;
                }
                if (r.min_p > 0.0) total = min(total, atleast);
                const At at = follow(share(u, total), true);
                if (lead && t == 0) write(at.pos, (double)value_of((K)at.key), total);
            } else {  // a long run of the largest: from global memory, by digits
                if (next < nrow) ask(next);
                if (lead) {
                    const auto open = [](W y) { return y > (W)-INFINITY; };
                    const auto mass = [&](W y) { return sc.mass((double)y); };
                    const auto sum = [&](auto f) {
                        u64 s = 0;
                        for (int i = t; i < ncol; i += NT) s += f(wide(x[i]));
                        return team.reduce(s, [](u64 a, u64 b) { return a + b; });
                    };
                    const u64 opened = sum([](W y) { return (u64)(y > (W)-INFINITY); });
                    u64 total;
                    if ((u64)r.top_k < opened) {
                        const Border br = find_border(team, x, ncol, digits, (u64)(r.top_k - 1), 0ull, open, [](W) { return 1ull; });
                        total = sum([&](W y) { return open(y) && (u64)key_of(y) > br.key ? mass(y) : 0ull; }) +
                                ((u64)r.top_k - br.above) * sc.mass((double)value_of((K)br.key));
                    } else {
                        total = sum(mass);
                    }
                    if (r.top_p < 1.0) {
                        const double w = ceil(r.top_p * (double)total);
                        const u64 want = w < 1.0 ? 1ull : min((u64)w, total);
                        const Border br = find_border(team, x, ncol, digits, want - 1, 0ull, open, mass);
                        const u64 m = sc.mass((double)value_of((K)br.key));
                        total = br.above + ((want - 1 - br.above) / m + 1) * m;
                    }
                    if (r.min_p > 0.0)
                        total = min(total, sum([&](W y) {
                                        const double e = sc.weight_at((double)y);
                                        return e >= r.min_p ? sc.mass_of(e) : 0ull;
                                    }));
                    const u64 target = share(u, total);
                    const Border br = find_border(team, x, ncol, digits, target, 0ull, open, mass);
                    const double v = (double)value_of((K)br.key);
                    const u64 nth = (target - br.above) / sc.mass(v);
                    first_of_key(team, x, ncol, br.key, nth + 1, [&](int i, u64 j) {
                        if (j == nth) write(i, v, total);
                    });
                }
            }
        }
        if (next >= nrow) break;
        row = next;
        team.sync_all();
    }
    if constexpr (CL) team.sync_all();
}

}  // namespace

namespace hxr {

cudaError_t launch_top(const hx_readout& rows, int k, const Heat& heat, int* idx, void* val, void* lse, int sms, cudaStream_t st) {
    return by_type(rows.dtype, [&](auto* tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        const int cap = top_cap(k);
        const size_t key = sizeof(typename Ty<T>::K);
        const bool warps = rows.ncol <= 512 && cap <= 512;
        const size_t ex = top_extra(warps ? 32 : kWide, cap, key);
        const Deal d = deal<T>(rows, ex, warps ? ex : 0, kWide, kWides<T>, 0, sms);
        const auto go = [&](auto* kernel) {
            return launch(kernel, d, st, (const T*)rows.x, rows.nrow, rows.ncol, rows.ld, k, heat, idx, (T*)val, (typename Ty<T>::W*)lse, cap,
                          (int)d.team, (int)d.slice);
        };
        return d.nt == 32 ? go(top_kernel<T, 32, false>) : d.parts > 1 ? go(top_kernel<T, kWide, true>)
               : d.nt == 128 ? go(top_kernel<T, 128, false>) : go(top_kernel<T, kWide, false>);
    });
}

cudaError_t launch_sample(const hx_readout& rows, const hx_sample_rule& rule, const hx_sample_rule* rules, const double* u, int bits,
                          int* idx, void* logp, int sms, cudaStream_t st) {
    return by_type(rows.dtype, [&](auto* tag) {
        using T = std::remove_pointer_t<decltype(tag)>;
        const size_t key = sizeof(typename Ty<T>::K);
        // room for twice top_k where it is known and small; per-row rules: up to 256
        int cap = rows.ncol <= 512 ? 128 : 512;
        if (!rules)
            while (cap < 1024 && rule.top_k >= 1.0 && 2.0 * rule.top_k > cap &&
                   kRedBytes + Slice<T>::bytes(rows.ncol, 8) + sample_extra(kWide, 2 * cap, key) <= kSmemBlock)
                cap *= 2;
        const bool warps = rows.ncol <= 512 && cap <= 256;
        const size_t ex = sample_extra(warps ? 32 : kWide, cap, key);
        const Deal d = deal<T>(rows, ex, warps ? ex : 0, kWide, kWides<T>, 0, sms);
        const auto go = [&](auto* kernel) {
            return launch(kernel, d, st, (const T*)rows.x, rows.nrow, rows.ncol, rows.ld, rule, rules, u, bits, idx, (typename Ty<T>::W*)logp, cap,
                          (int)d.team, (int)d.slice);
        };
        return d.nt == 32 ? go(sample_kernel<T, 32, false>) : d.parts > 1 ? go(sample_kernel<T, kWide, true>)
               : d.nt == 128 ? go(sample_kernel<T, 128, false>) : go(sample_kernel<T, kWide, false>);
    });
}

}  // namespace hxr

// hx_readout.cu -- operators over readout rows: the distillation loss of a
// student's rows with its gradient, and the C entries of all three.
#include <cuda_runtime.h>

#include <string>

#include "heliox_b200.h"
#include "hx_ctx.hpp"
#include "hx_readout.cuh"

namespace {

using namespace hxr;

// ---------------------------------------------------------------- distillation
//
// One pass over memory, and as few instructions as it takes: the row waits in
// shared memory, is replaced there by its exponentials, these by the gradient,
// and leaves in bulk copies.  Every warp has a run of the row's vectors of its
// own, for which it waits, and asks for that run of the team's next row when
// the bulk copy has read the last.  The warps of a row meet twice: before it,
// when the teacher's side is ready, and for the sum.
//
// The exponentials are taken relative to the readout in the first slot, which
// the teacher holds for likely, not to the row's largest: only where the sum
// then shows that some other readout is far above it (e^28 times in fp32,
// e^346 in fp64), or NaN, is the row read again and its largest found.
//
// The slots' readouts are lifted out of the row before the sum (-inf stands in
// their places), so that the sum over the rest is a sum of its own and not a
// difference.  A rest that the record gives a share, but that lies e^-44 or more
// below, is summed up again relative to its own largest readout, so that its
// logarithm and its readouts' shares of it are right at any distance.  The
// teacher's side of the next row is worked out meanwhile: in a block of many
// warps by a helper, which has no run, so that its chain of dependent
// exponentials and reductions is waited for by nobody.

constexpr int kBlock = 256;  // threads of a block that has a row, or a slice of one, to itself (short rows: 128)
template <typename T>
constexpr int kBlocks = sizeof(T) == 8 ? 2 : 3;  // such blocks on an SM, where their shared memory lets them

// Measured (B200): 4000 x 10000 fp64 rows, 64 slots: 168 us, 3.8 TB/s of reads
// and writes, with two 80 KB rows an SM in flight and the warps' dependent
// chains between them as the bound; 1021 x 32003 bf16 51 us; 8000 x 302 fp64,
// a warp a row, 28 us, about 900 instructions a row besides its readouts.
// Blocks of 512 threads: 199 us for the first, 62 for the second (each warp has
// its share of reductions and divisions once a row); 3 blocks of 256 an SM
// against 2: 50 and 55 us for the second.  Without copying the next row to L2
// ahead: 174 us against 167 for the first, 219 against 211 at 8000 x 3000.
constexpr double kFar = 0x1p-64;  // a sum from here on has lost nothing that counts to the exponentials' range (2^-126 in fp32)
constexpr int kFewSlots = 128;  // up to here the next row's slots are worked out into lists of their own

__host__ __device__ constexpr int slot_list(int k) { return (k + 3) / 4 * 4; }
__host__ __device__ constexpr int hash_bits(int k) {  // a table at most half full
    int b = 5;
    while ((1 << b) < 2 * k) b++;
    return b;
}
static_assert(HX_READOUT_MAX_ROW_BYTES / 2 <= 1 << 20 && HX_READOUT_MAX_K <= 1 << 10, "a position and a slot share 32 bits in the hash table");
size_t distill_extra(int k) { return (size_t)slot_list(k) * 20 * (k <= kFewSlots ? 2 : 1) + ((size_t)4 << hash_bits(k)); }

// The slots of a row, in shared memory, and the warp that works on them
// (lane l has slots l, l + 32, ...).
struct Slots {
    double* q;  // value, then probability
    double* x;  // the row's readout there, then its exponential
    int* at;    // position, -1: not used
    double* notes;  // [0] log-sum-exp of the record, [1] sum of q, [2] sum of q log q, [3] 1: a slot is used, [4] a readout there, [5], [6] of lifted(), [7] the largest value
    int lane;
    __device__ Slots(char* lists, double* all_notes, int k, int set, int thread) : lane(thread & 31) {
        q = (double*)(lists + (k <= kFewSlots ? set * slot_list(k) * 20 : 0));
        x = q + slot_list(k);
        at = (int*)(x + slot_list(k));
        notes = all_notes + set * 8;
    }
    static __device__ __forceinline__ double sum(double v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
        return v;
    }
    // Starts the copy of a row's record; narrow values are widened at once.
    __device__ __forceinline__ void load(const hx_teacher& te, size_t row) const {
        const int k = te.k;
        for (int j = lane; j < k; j += 32) {
            copy4(at + j, te.idx + row * k + j);
            if (te.dtype == HX_DT_F64)
                copy8(q + j, (const double*)te.val + row * k + j);
            else if (te.dtype == HX_DT_F32)
                copy4(q + j, (const float*)te.val + row * k + j);
            else
                q[j] = load_any(te.val, te.dtype, row * k + j);
        }
        if (te.lse && lane == 0) {
            if (te.dtype == HX_DT_F64)
                copy8(notes, (const double*)te.lse + row);
            else
                copy4(notes, (const float*)te.lse + row);
        }
    }
    // The slots in use, from the copied record; GROUPS of later copies may be on their way.
    template <int GROUPS, typename T>
    __device__ __forceinline__ void sift(const hx_teacher& te, const T* row, int ncol, unsigned* hash) const {
        const int k = te.k, bits = hash_bits(k), most = 1 << bits;
        wait_copies<GROUPS>();
        if (k > 32)
            for (int h = lane; h < most; h += 32) hash[h] = ~0u;
        __syncwarp();
        for (int j = lane; j < k; j += 32) {
            const double v = te.dtype == HX_DT_F32 ? (double)*(const float*)(q + j) : q[j];
            int i = at[j];
            q[j] = v;
            if (i < 0 || i >= ncol || v == -INFINITY) i = -1;
            at[j] = i;
            if (k <= 32 || i < 0) continue;
            const unsigned both = (unsigned)i << 10 | (unsigned)j;
            unsigned h = ((unsigned)i * 2654435761u) >> (32 - bits);
            for (int step = 0; step < most; step++, h = (h + 1) & (most - 1)) {
                const unsigned o = atomicCAS(&hash[h], ~0u, both);
                if (o == ~0u) break;
                if (o >> 10 == (unsigned)i) {
                    atomicMin(&hash[h], both);
                    break;
                }
            }
        }
        __syncwarp();
        // a position that an earlier slot has is dropped
        double tm = -INFINITY;
        bool used = false;
        if (k <= 32) {
            const int i = lane < k ? at[lane] : -1;
            const unsigned same = __match_any_sync(~0u, i);
            if (i >= 0 && __ffs(same) - 1 == lane) {
                used = true;
                tm = larger(tm, q[lane]);
            } else if (lane < k) {
                at[lane] = -1;
            }
        } else {
            for (int j = lane; j < k; j += 32) {
                const int i = at[j];
                if (i < 0) continue;
                unsigned h = ((unsigned)i * 2654435761u) >> (32 - bits);
                for (int step = 0; step < most && hash[h] >> 10 != (unsigned)i; step++) h = (h + 1) & (most - 1);
                if ((hash[h] & 1023) == (unsigned)j) {
                    used = true;
                    tm = larger(tm, q[j]);
                } else {
                    at[j] = -1;
                }
            }
        }
        __syncwarp();
        const unsigned lanes = __ballot_sync(~0u, used);
        double ref = 0;
        if (lanes) {
            int j = __ffs(lanes) - 1;
            while (j < k && at[j] < 0) j += 32;  // that lane's first slot in use
            if (j < k) ref = (double)wide(row[at[j]]);
        }
        if (!te.lse) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) tm = larger(tm, __shfl_xor_sync(~0u, tm, o));
        }
        if (lane == 0) {
            notes[3] = lanes ? 1.0 : 0.0;
            notes[4] = ref;
            notes[7] = tm;
        }
    }
    // Their probabilities and sums.
    __device__ __forceinline__ void weigh(const hx_teacher& te, double inv) const {
        const int k = te.k;
        __syncwarp();
        const double tm = te.lse ? 0.0 : notes[7];
        const double shift = !te.lse ? 0.0 : te.dtype == HX_DT_F64 ? notes[0] : (double)*(const float*)notes;
        double s = 0, qv = 0;
        for (int j = lane; j < k; j += 32) {
            if (at[j] < 0) continue;
            const double lq = (q[j] - tm) * inv - shift, e = exp(lq);
            q[j] = e;
            s += e;
            qv += e == 0.0 ? 0.0 : e * lq;
        }
        s = sum(s);
        qv = sum(qv);
        if (!te.lse) {  // over the slots alone: divide by their sum
            const double f = 1.0 / s;
            for (int j = lane; j < k; j += 32)
                if (at[j] >= 0) q[j] *= f;
            qv = qv * f - log(s);
            s = s == s ? 1.0 : s;
        }
        if (lane == 0) {
            notes[1] = s;
            notes[2] = qv;
        }
    }
    // The exponentials of the readouts that have been lifted out of this
    // block's slice, and the sums of those and of q z.
    template <typename T, typename E>
    __device__ __forceinline__ void lifted(const Slice<T>& sl, int k, const E& ex) const {
        double in = 0, qz = 0;
        for (int j = lane; j < k; j += 32) {
            if (at[j] < 0 || (unsigned)(at[j] - sl.first) >= (unsigned)sl.n) continue;
            const double z = ex.z(x[j]), e = exp(z);
            x[j] = e;
            in += e;
            qz += q[j] == 0.0 ? 0.0 : q[j] * z;
        }
        in = sum(in);
        qz = sum(qz);
        if (lane == 0) {
            notes[5] = in;
            notes[6] = qz;
        }
    }
    // f(j, cell) for the slots whose readouts are in vectors v0 .. v1-1 of the slice.
    template <typename T, typename F>
    __device__ __forceinline__ void each(const Slice<T>& sl, int k, int v0, int v1, F f) const {
        const int a = max(v0 * Ty<T>::VEC, sl.phase), n = min(v1 * Ty<T>::VEC, sl.phase + sl.n) - a, shift = sl.phase - sl.first;
        for (int j = lane; j < k; j += 32) {
            const int p = at[j];
            if (p >= 0 && (unsigned)(p + shift - a) < (unsigned)max(n, 0)) f(j, sl.e + (p + shift));
        }
    }
};

template <typename T, int NT, bool CL>
__global__ void __launch_bounds__(NT == 32 ? 32 * kWarpRows : NT + 32, NT == kBlock ? kBlocks<T> : 6)
    distill_kernel(const T* xs, int nrow, int ncol, long long ld, hx_teacher te, Heat heat, double scale,
                   const double* __restrict__ weight, T* gs, long long ldg, typename Ty<T>::W* __restrict__ row_loss,
                   int team_bytes, int slice_bytes) {
    using W = typename Ty<T>::W;
    constexpr int VEC = Ty<T>::VEC;
    constexpr bool ONE = NT == 32;  // one warp does it all
    constexpr int UNROLL = VEC == 8 ? 1 : 2;
    extern __shared__ __align__(16) char smem[];
    char* const mine = smem + (ONE ? (threadIdx.x >> 5) * team_bytes : 0);
    Team<NT, CL, !ONE> team(mine);
    const int t = team.t, k = te.k;
    const bool few = ONE || k <= kFewSlots;  // a warp's record is copied ahead of its row: deal() gives warps no more slots
    const bool helper = ONE || t >= NT, worker = ONE || t < NT;
    T* const row_mem = (T*)(mine + kRedBytes);
    char* const lists = mine + kRedBytes + slice_bytes;
    unsigned* const hash = (unsigned*)(lists + slot_list(k) * 20 * (few ? 2 : 1));
    const long long step = team.row_step();
    long long row = team.first_row();
    if (row >= nrow) return;  // a whole team
    double w = weight ? weight[row] : 1.0;
    int set = 0;
    const int lane = t & 31, warp = ONE ? 0 : t >> 5;
    constexpr int NW = NT / 32;
    const auto ask = [&](const Slice<T>& s) {  // for this warp's run
        s.load(s.template run<NW>(warp), s.template run<NW>(warp + 1), lane);
    };
    if (w != 0.0) {
        const Slots slots(lists, team.notes(), k, 0, t);
        const T* const x = xs + row * ld;
        if (helper) slots.load(te, row);
        if (ONE) commit_copies();
        if (worker) ask(Slice<T>(row_mem, x, ncol, team.part, team.parts));
        if (ONE) commit_copies();
        if (helper) {
            slots.template sift<ONE ? 1 : 0>(te, x, ncol, hash);
            slots.weigh(te, heat.inv);
        }
    }
    for (;;) {
        const Slice<T> sl(row_mem, xs + row * ld, ncol, team.part, team.parts);
        const int v0 = sl.template run<NW>(warp), v1 = sl.template run<NW>(warp + 1);
        T* const g = gs ? gs + row * ldg : nullptr;
        const long long next = row + step;
        const double wn = next < nrow ? (weight ? weight[next] : 1.0) : 0.0;
        const Slots slots(lists, team.notes(), k, set, t), ahead(lists, team.notes(), k, set ^ 1, t);
        bool live = w != 0.0;
        if (worker) wait_copies();
        team.sync_block();  // the slots are ready, and those of the row before are free
        live = live && slots.notes[3] != 0.0;
        // the next row into L2, its record into shared memory, before this row's own traffic
        if (worker && wn != 0.0) {
            const Slice<T> nx(row_mem, xs + next * ld, ncol, team.part, team.parts);
            if (lane == 0) nx.prefetch(nx.template run<NW>(warp), nx.template run<NW>(warp + 1));
        }
        if (helper && few && wn != 0.0) ahead.load(te, next);
        if (ONE) commit_copies();
        if (live) {
            struct Sums {
                double out, in, qz;
            } s;
            // the exponentials of this warp's run, in the readouts' place where they fit, and the lanes' sums
            const auto sum_up = [&](const auto& ex) {
                W part[2] = {0, 0};
#pragma unroll UNROLL
                for (int v = v0 + lane; v < v1; v += 32) {
                    Vec<T> x = sl.get(v);
#pragma unroll
                    for (int u = 0; u < VEC; u++) {
                        const W e = ex(wide(x.e[u]));
                        part[u & 1] += e;
                        if constexpr (sizeof(T) == sizeof(W)) x.e[u] = e;
                    }
                    if constexpr (sizeof(T) == sizeof(W)) sl.set(v, x);
                }
                return (double)part[0] + (double)part[1];
            };
            const auto add = [](double a, double b) { return a + b; };
            const auto close = [](int, T* cell) { *cell = narrow<T>((W)-INFINITY); };
            W m = (W)slots.notes[4];
            bool odd = false, empty = false;  // NaN or +inf in the row; no readout is open
            for (bool sure = false;; sure = true) {
                if (sure) {  // the row's largest readout
                    struct Top {
                        W mx;
                        int odd;
                    } top{(W)-INFINITY, 0};
                    if (worker) {
                        __syncwarp();
                        ask(sl);
                        wait_copies();
                        __syncwarp();
                        for (int v = v0 + lane; v < v1; v += 32) {
                            const Vec<T> x = sl.get(v);
#pragma unroll
                            for (int u = 0; u < VEC; u++) {
                                const W y = wide(x.e[u]);
                                top.mx = larger(top.mx, y);
                                top.odd |= !(y < (W)INFINITY);
                            }
                        }
                        __syncwarp();
                    }
                    const auto op = [](Top a, Top b) { return Top{larger(a.mx, b.mx), a.odd | b.odd}; };
                    top = team.across(team.reduce(top, op), op);
                    odd = top.odd;
                    empty = top.mx == (W)-INFINITY && !odd;
                    m = odd || empty ? (W)0 : top.mx;
                }
                const auto ex = scaler(m, heat, team.table());
                double out = 0;
                if (worker) {
                    slots.each(sl, k, v0, v1, [&](int j, T* cell) {
                        slots.x[j] = (double)wide(*cell);
                        close(j, cell);
                    });
                    __syncwarp();
                    if (!ONE) bar_arrive(2, NT + 32);
                    out = sum_up(ex);
                }
                if (helper) {
                    if (!ONE) bar_sync(2, NT + 32);
                    slots.lifted(sl, k, ex);
                    if (!ONE && few && wn != 0.0 && !sure) ahead.template sift<0>(te, xs + next * ld, ncol, hash);
                }
                out = team.reduce(out, add);
                if (ONE) __syncwarp();
                s = team.across(Sums{out, slots.notes[5], slots.notes[6]},
                                [](Sums a, Sums b) { return Sums{a.out + b.out, a.in + b.in, a.qz + b.qz}; });
                if (sure || (s.in + s.out <= decltype(ex)::most && s.in + s.out > 0.0)) break;
            }
            const double sum_q = slots.notes[1], sum_qlq = slots.notes[2];
            const double total = odd ? (double)NAN : s.in + s.out;
            double qr = te.lse ? (sum_q == sum_q ? larger(0.0, 1.0 - sum_q) : sum_q) : 0.0;
            // a rest far below: once more, relative to its own largest readout
            W m_out = m;
            if (qr > 0.0 && s.out < kFar && !odd && !empty) {
                W mx = -INFINITY;
                if (worker) {
                    if constexpr (sizeof(T) == sizeof(W)) {
                        __syncwarp();
                        ask(sl);
                        wait_copies();
                        __syncwarp();
                        slots.each(sl, k, v0, v1, close);
                        __syncwarp();
                    }
                    for (int v = v0 + lane; v < v1; v += 32) {
                        const Vec<T> x = sl.get(v);
#pragma unroll
                        for (int u = 0; u < VEC; u++) mx = larger(mx, wide(x.e[u]));
                    }
                }
                const auto op = [](W a, W b) { return larger(a, b); };
                mx = team.across(team.reduce(mx, op), op);
                if (mx > (W)-INFINITY) m_out = mx;  // else all of it is closed, and stays 0
                const auto ex = scaler(m_out, heat, team.table());
                s.out = team.across(team.reduce(worker ? sum_up(ex) : 0.0, add), add);
            }
            const double z_out = ((double)m_out - (double)m) * heat.inv;  // log of what s.out is a multiple of
            if (!(qr > 0.0 && s.out > 0.0) && qr == qr && s.out == s.out) qr = 0.0;
            if (worker && g) {
                const double one_over = 1.0 / total, mass = sum_q + qr, c = empty ? 0.0 : scale * w * heat.t;
                double a = c * mass * one_over;
                const double a_in = empty ? 0.0 : a;
                if (z_out != 0.0) a *= exp(z_out);
                if (qr != 0.0) a -= c * qr / s.out;
                if (empty) a = 0.0;
                const auto ex = scaler(m_out, heat, team.table());
                const auto times = [&](const auto by) {  // the exponentials times a, in the type of `by`
#pragma unroll UNROLL
                    for (int v = v0 + lane; v < v1; v += 32) {
                        Vec<T> x = sl.get(v);
#pragma unroll
                        for (int u = 0; u < VEC; u++) {
                            if constexpr (sizeof(T) == sizeof(W))
                                x.e[u] = (W)(x.e[u] * by);
                            else
                                x.e[u] = narrow<T>((W)(ex(wide(x.e[u])) * by));
                        }
                        sl.set(v, x);
                    }
                };
                // a large or a tiny scale's factor may be beyond fp32 where the products are not
                if (sizeof(W) == 8 || a == 0.0 || !(fabs(a) < 0x1p-126 || fabs(a) > 0x1p127))
                    times((W)a);
                else
                    times(a);
                __syncwarp();
                slots.each(sl, k, v0, v1, [&](int j, T* cell) { *cell = narrow<T>((W)(a_in * slots.x[j] - c * slots.q[j])); });
            }
            if (helper && lane == 0 && team.part == 0) {
                double loss = sum_qlq - s.qz + sum_q * log(total);
                if (qr != 0.0) loss += qr * (log(qr * total / s.out) - z_out);
                row_loss[row] = empty ? (W)0 : (W)(heat.t * heat.t * loss);
            }
        } else {  // for every block of a cluster alike
            if (helper && lane == 0 && team.part == 0) row_loss[row] = 0;
            if (worker && g)
                for (int v = v0 + lane; v < v1; v += 32) {
                    Vec<T> z;
#pragma unroll
                    for (int u = 0; u < VEC; u++) z.e[u] = narrow<T>((W)0);
                    sl.set(v, z);
                }
        }
        if (!few && wn != 0.0) team.sync_block();  // the slots have been read
        if (worker) {
            __syncwarp();
            if (g) sl.store(v0, v1, lane, g);
            if (wn != 0.0) ask(Slice<T>(row_mem, xs + next * ld, ncol, team.part, team.parts));
            if (ONE) commit_copies();  // the row's; the slots' are the group before
        }
        if (helper && wn != 0.0) {
            if (!few) ahead.load(te, next);  // by a helper, which has no copies besides
            if (ONE || !few || !live) ahead.template sift<ONE ? 1 : 0>(te, xs + next * ld, ncol, hash);
            ahead.weigh(te, heat.inv);
        }
        if (next >= nrow) break;
        row = next;
        w = wn;
        set ^= 1;
    }
    if constexpr (CL) team.sync_all();  // a block stays while others may read its partials
}

// scale sum_r w_r L_r in one block, each thread over rows of its own, then a tree: one order.
constexpr int kLossThreads = 1024;
template <typename W>
__global__ void __launch_bounds__(kLossThreads) loss_kernel(const W* __restrict__ row_loss, const double* __restrict__ weight, int nrow,
                                                            double scale, W* __restrict__ loss) {
    __shared__ double red[32];
    double s = 0;
#pragma unroll 8
    for (unsigned r = threadIdx.x; r < (unsigned)nrow; r += kLossThreads) {  // up to 2^31 - 1 of them
        const double w = weight ? weight[r] : 1.0, l = (double)row_loss[r];
        s += w != 0.0 ? w * l : 0.0;
    }
    s = Slots::sum(s);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x < 32) {
        s = Slots::sum(red[threadIdx.x]);
        if (threadIdx.x == 0) *loss = (W)(scale * s);
    }
}

// ---------------------------------------------------------------- host side

int type_size(int dtype) { return dtype == HX_DT_F64 ? 8 : dtype == HX_DT_F32 ? 4 : 2; }
int stat_size(int dtype) { return dtype == HX_DT_F64 ? 8 : 4; }
bool off(const void* p, int align) { return (size_t)p % (size_t)align != 0; }

constexpr long long kMostElements = 1ll << 56;  // of rows and what lies between them: no address space has more, and byte offsets fit 64 bits

const char* check_rows(const hx_readout* r) {
    if (!r) return "null rows";
    if (r->dtype < HX_DT_F64 || r->dtype > HX_DT_BF16) return "rows: unknown dtype";
    if (r->nrow < 0 || r->ncol < 0) return "rows: nrow and ncol must not be negative";
    if (r->ld < r->ncol) return "rows: ld must be at least ncol";
    if ((long long)r->ncol * type_size(r->dtype) > HX_READOUT_MAX_ROW_BYTES) return "rows: a row is longer than HX_READOUT_MAX_ROW_BYTES";
    if (r->nrow > 1 && r->ld > kMostElements / r->nrow) return "rows: ld is out of range";
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
    if (r->nrow > 1 && ldg > kMostElements / r->nrow) return "ld_grad is out of range";
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
    HXC(launch_top(*rows, k, heat_of(temperature), idx_dev, val_dev, lse_dev, sm_count(ctx->device), ctx->st));
    return 0;
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
            const size_t extra = distill_extra(teacher->k);
            const Deal d = deal<T>(*rows, extra, teacher->k <= kFewSlots ? extra : 0, kBlock, kBlocks<T>, 32, sm_count(ctx->device));
            auto go = [&](auto* kernel) {
                return launch(kernel, d, ctx->st, (const T*)rows->x, rows->nrow, rows->ncol, rows->ld, *teacher, heat_of(temperature),
                              scale, row_weight_dev, (T*)grad_dev, ld_grad, (W*)row_loss_dev, (int)d.team, (int)d.slice);
            };
            HXC(d.nt == 32 ? go(distill_kernel<T, 32, false>) : d.parts > 1 ? go(distill_kernel<T, kBlock, true>)
                : d.nt == 128 ? go(distill_kernel<T, 128, false>) : go(distill_kernel<T, kBlock, false>));
        }
        loss_kernel<W><<<1, kLossThreads, 0, ctx->st>>>((const W*)row_loss_dev, row_weight_dev, rows->nrow, scale, (W*)loss_dev);
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
    const int bits = lg <= 10 ? 52 : 62 - lg;  // a row's masses add up to less than 2^62
    const hx_sample_rule none{1.0, 0.0, 1.0, 0.0};
    OnDevice on(ctx->device);
    HXC(on.e);
    HXC(launch_sample(*rows, rules_dev ? none : *rule, rules_dev, u_dev, bits, idx_dev, logp_dev, sm_count(ctx->device), ctx->st));
    return 0;
}

}  // extern "C"

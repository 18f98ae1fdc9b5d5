"""GPU: the readout-row entries against plain numpy in 64 bits.

Tolerances, with u = 2^-53 (fp64 rows) or 2^-24 (others) the half step of the
statistics' type and h that of the rows' type (fp16 2^-11, bf16 2^-8):

* a scaled readout z = (x - max) / T takes two or three roundings, 3 u |z|;
  exp adds 2 steps (4 u); a sum of n positive terms, split over at least 32
  threads, adds at most (n / 32 + 10) u.  So a probability, and the log of a
  sum, carry at most E = u (3 Z + n / 32 + 24) relative (absolute for the log),
  Z the largest |z| that matters: 104 for fp32, where exp is 0 below, else the
  row's own spread up to 746.
* row losses: in 64 bits log q = v / T - norm is off by up to 2^-50 (k + 8 +
  |v| / T) =: N (two roundings at |v| / T, two at |norm| <= |v| / T + log k, a
  sum of k), on both sides, so q is off by q N, and a term q (log q - log p)
  by q (|log q - log p| N + N + E + 2^-50 (|log p| + |log q| + 1)); the rest's
  q_r is off by N, its term by N (|log q_r| + |log p_r| + 2) + 2 q_r E (a
  teacher's log-sum-exp is the same input on both sides); then one rounding.
* gradients: c (Q p - q) carries |c| (p E + (p + q) (k + 40) 2^-52), the rest's
  c p (Q - q_r / p_r) carries |c| p (2 E (1 + q_r / p_r) + 2^-50 (k + 8) / p_r),
  then one rounding to the rows' type (an absolute 2^-25 for subnormal fp16).
* a choice may differ only where u times the run's mass is nearer to a border
  than the masses' own rounding: n units of 2^-s.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DT = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF = {"f64": 2.0**-53, "f32": 2.0**-24, "f16": 2.0**-11, "bf16": 2.0**-8}
# exponentials below 2^-1018 (fp64) and 2^-126 (fp32) of one whose sum is at least 1 are 0, here times a factor below 2^10; fp16: half a subnormal step
TINY = {"f64": 2.0**-1000, "f32": 2.0**-116, "f16": 2.0**-25, "bf16": 2.0**-116}
STAT = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float32, "bf16": torch.float32}


def stat_u(dtype):
    return 2.0**-53 if dtype == "f64" else 2.0**-24


@pytest.fixture(scope="module")
def sim():
    from heliox_b200.runtime import Sim

    s = Sim(0)
    s.set_stream(torch.cuda.current_stream().cuda_stream)
    yield s
    s.close()


def place(a, dtype, pad=0, offset=0):
    """Rows of ``a`` on the GPU, ``pad`` NaN elements between them, ``offset`` elements into their buffer."""
    nrow, ncol = a.shape
    ld = ncol + pad
    buf = torch.full((offset + nrow * ld + 1,), math.nan, dtype=DT[dtype], device="cuda")
    view = buf[offset:offset + nrow * ld].view(nrow, ld)[:, :ncol] if nrow * ld else torch.empty((nrow, ncol), dtype=DT[dtype], device="cuda")
    if a.size:
        view.copy_(torch.from_numpy(a).to(DT[dtype]))
    return buf, view, ld


def wide(t):
    return t.double().cpu().numpy()


def readouts(rng, nrow, ncol, dtype, closed=0.0):
    x = rng.standard_normal((nrow, ncol)) * 2.5 + (-65.0 if dtype == "f64" else 0.0)
    x[rng.random(x.shape) < 0.02] += 8.0
    if closed:
        x[rng.random(x.shape) < closed] = -math.inf
    return x


# ------------------------------------------------------------------ plain forms, row by row

def plain_top(x, k, T):
    n = len(x)
    if np.isnan(x).any():
        return np.full(k, -1), np.full(k, np.nan), np.nan
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf][:k]
    idx, val = np.full(k, -1), np.full(k, -np.inf)
    idx[:len(order)], val[:len(order)] = order, x[order]
    if not len(order) or x.max() == np.inf:
        return idx, val, x.max() if n else -np.inf
    with np.errstate(over="ignore"):
        return idx, val, x.max() / T + math.log(np.exp((x - x.max()) / T).sum())


def spread(x, T, dtype):
    f = x[np.isfinite(x)]
    with np.errstate(over="ignore"):
        z = (f.max() - f.min()) / T if len(f) else 0.0
    return min(z, 746.0 if dtype == "f64" else 104.0)


def row_error(x, T, dtype):
    return stat_u(dtype) * (3 * spread(x, T, dtype) + len(x) / 32 + 24)


def plain_distill(x, idx, val, lse, T, w, scale, dtype):
    """(loss, its bound, gradient, its bound) of one row."""
    n, E = len(x), row_error(x, T, dtype)
    zero = (0.0, 0.0, np.zeros(n), np.zeros(n))
    slots = {}
    for i, v in zip(idx, val):
        if 0 <= i < n and v != -np.inf and int(i) not in slots:
            slots[int(i)] = float(v)
    if w == 0 or not slots:
        return zero
    if np.isnan(x).any():
        return np.nan, 0.0, np.full(n, np.nan), np.zeros(n)
    if not (x > -np.inf).any():
        return zero
    at, v = np.array(list(slots)), np.array(list(slots.values()))
    k = len(idx)
    z = (x - x.max()) / T
    e = np.exp(z)
    S = e.sum()
    p, logp = e / S, z - math.log(S)
    if lse is None:
        tm = v.max()
        lq = (v - tm) / T - math.log(np.exp((v - tm) / T).sum())
    else:
        lq = v / T - lse
    q = np.exp(lq)
    live = q > 0
    with np.errstate(invalid="ignore"):
        L = (q * (lq - logp[at]))[live].sum()
        noise = 2.0**-50 * (k + 8 + np.abs(v).max() / T)
        dL = (q * (E + noise * (1 + np.abs(lq - logp[at])) + (np.abs(lq) + np.abs(logp[at]) + 1) * 2.0**-50))[live].sum()
    Q, c = q.sum(), scale * w * T
    full = np.zeros(n)
    full[at] = q
    out = np.ones(n, bool)
    out[at] = False
    if lse is None:
        g = c * (p - full)
        dg = abs(c) * (p * E + (p + full) * (k + 40 + np.abs(v).max() / T) * 2.0**-52)
    else:
        qr, pr = max(0.0, 1.0 - Q), e[out].sum() / S
        if qr == 0 or pr == 0:
            qr = 0.0
        ratio = 0.0
        if qr > 0:
            L += qr * (math.log(qr) - math.log(pr))
            dL += qr * 2 * E + noise * (abs(math.log(qr)) + abs(math.log(pr)) + 2)
            ratio = qr / pr
        g = c * np.where(out, p * (Q + qr - ratio), (Q + qr) * p - full)
        dg = abs(c) * (p * E * (1 + 2 * ratio) * 2 + (p + full) * noise * 2 + (p * noise * 2 / pr if pr > 0 else 0))
    h = HALF[dtype]
    with np.errstate(invalid="ignore"):
        return T * T * L, T * T * dL + abs(T * T * L) * stat_u(dtype) * 2, g, dg + np.abs(g) * h * (1 + 2.0**-20) + TINY[dtype] * (1 + 2.0**-8)


def plain_sample(x, T, top_k, top_p, min_p, u):
    """(position, log-probability, the positions that rounding of the masses may also choose)."""
    n = len(x)
    if math.isnan(T) or np.isnan(x).any() or (x == np.inf).any():
        return -2, math.nan, {-2}
    order = np.argsort(-x, kind="stable")
    order = order[x[order] > -np.inf]
    if not len(order):
        return -1, -math.inf, {-1}
    if T <= 0:
        T, top_k = 1.0, 1
    z = (x[order] - x[order[0]]) / T
    e = np.exp(z)
    L = len(order)
    if top_k >= 1:
        L = min(L, int(min(top_k, n)))
    bits = min(52, 62 - math.ceil(math.log2(n)) if n > 1 else 62)
    slack = (n + 2) * 2.0**-bits + 2.0**-50 * e[:L].sum() * 4
    run = np.cumsum(e[:L])

    def lengths(target):  # prefixes that reach the target within the slack
        lo = int(np.searchsorted(run, target - slack)) + 1
        hi = int(np.searchsorted(run, target + slack)) + 1
        return range(min(lo, L), min(hi, L) + 1)

    cuts = lengths(max(top_p, 0.0) * run[-1]) if top_p < 1 else [L]
    m3 = int((e[:L] >= min(max(min_p, 0.0), 1.0)).sum()) if min_p > 0 else L
    near = 0 < min_p < 1 and (np.abs(e[:L] - min_p) <= 2.0**-50 * min_p).any()
    may, best = set(), None
    uu = min(max(u, 0.0), 1.0)
    for cut in cuts:
        K = max(1, min(cut, m3))
        target = uu * run[K - 1]
        lo = min(int(np.searchsorted(run[:K], target - slack, side="right")), K - 1)
        hi = min(int(np.searchsorted(run[:K], target + slack, side="right")), K - 1)
        may |= {int(order[j]) for j in range(lo, hi + 1)}
        j = min(int(np.searchsorted(run[:K], target, side="right")), K - 1)
        best = best or (int(order[j]), z[j] - math.log(run[K - 1]))
    assert not near, "a weight on the border of min_p"
    return best[0], best[1], may


# ------------------------------------------------------------------ calls

def call_top(sim, view, ld, k, T, dtype, lse=True):
    nrow, ncol = view.shape
    idx = torch.full((nrow + 1, k), 77, dtype=torch.int32, device="cuda")
    val = torch.full((nrow + 1, k), 77.0, dtype=DT[dtype], device="cuda")
    ls = torch.full((nrow + 1,), 77.0, dtype=STAT[dtype], device="cuda")
    sim.top_logits_dev(view.data_ptr(), nrow, ncol, k, idx.data_ptr(), val.data_ptr(), lse_ptr=ls.data_ptr() if lse else 0,
                       temperature=T, dtype=dtype, ld=ld)
    torch.cuda.synchronize()
    assert (idx[nrow] == 77).all() and (val[nrow] == 77).all() and ls[nrow] == 77  # nothing behind the last row
    return idx[:nrow].cpu().numpy(), wide(val[:nrow]), wide(ls[:nrow])


def check_top(sim, x, k, T, dtype, pad=0, offset=0):
    buf, view, ld = place(x, dtype, pad, offset)
    idx, val, lse = call_top(sim, view, ld, k, T, dtype)
    xx = wide(view)
    for r in range(x.shape[0]):
        i, v, l = plain_top(xx[r], k, T)
        if abs(l) > torch.finfo(STAT[dtype]).max:  # beyond the statistics' type: max / T of lowest values
            l = math.copysign(math.inf, l)
        assert np.array_equal(idx[r], i), (r, idx[r], i)
        assert np.array_equal(val[r], v, equal_nan=True), r
        if np.isfinite(l):
            with np.errstate(over="ignore"):
                most = abs(l) + np.abs(xx[r][np.isfinite(xx[r])]).max() / T
            assert abs(lse[r] - l) <= row_error(xx[r], T, dtype) + 3 * stat_u(dtype) * most, (r, lse[r], l)
        else:
            assert np.array_equal(lse[r], l, equal_nan=True), (r, lse[r], l)


def call_distill(sim, view, ld, rec, T, dtype, t_dtype, w=None, scale=1.0, grad_ld=None, in_place=False, grad=True):
    nrow, ncol = view.shape
    ti, tv, tl = rec
    gl = ncol if grad_ld is None else grad_ld
    g = torch.full((nrow * gl + 5,), 77.0, dtype=DT[dtype], device="cuda")
    rl = torch.full((nrow + 1,), 77.0, dtype=STAT[dtype], device="cuda")
    lo = torch.full((2,), 77.0, dtype=STAT[dtype], device="cuda")
    wt = None if w is None else torch.from_numpy(np.asarray(w, dtype=np.float64)).cuda()
    sim.distill_loss_grad_dev(view.data_ptr(), nrow, ncol, ti.shape[1], ti.data_ptr(), tv.data_ptr(),
                              view.data_ptr() if in_place else g.data_ptr() if grad else 0, rl.data_ptr(), lo.data_ptr(),
                              t_lse_ptr=0 if tl is None else tl.data_ptr(), temperature=T, scale=scale,
                              row_weight_ptr=0 if wt is None else wt.data_ptr(), dtype=dtype, t_dtype=t_dtype, ld=ld,
                              ld_grad=ld if in_place else gl)
    torch.cuda.synchronize()
    assert rl[nrow] == 77 and lo[1] == 77
    if in_place or not grad:
        assert (g == 77).all()
        return (view.clone() if in_place else None), wide(rl[:nrow]), float(lo[0])
    assert (g[nrow * gl:] == 77).all()
    full = g[:nrow * gl].view(nrow, gl) if nrow * gl else g[:0].view(nrow, 0)
    assert (full[:, ncol:] == 77).all()  # between the rows
    return full[:, :ncol], wide(rl[:nrow]), float(lo[0])


def record(idx, val, lse, t_dtype):
    return (torch.from_numpy(np.ascontiguousarray(idx, dtype=np.int32)).cuda(), torch.from_numpy(val).to(DT[t_dtype]).cuda(),
            None if lse is None else torch.from_numpy(lse).to(STAT[t_dtype]).cuda())


def check_distill(sim, x, idx, val, lse, T, dtype, t_dtype, w=None, scale=0.25, pad=0, offset=0, **kw):
    buf, view, ld = place(x, dtype, pad, offset)
    xx = wide(view)
    rec = record(idx, val, lse, t_dtype)
    g, rl, lo = call_distill(sim, view, ld, rec, T, dtype, t_dtype, w, scale, **kw)
    vv, ll = wide(rec[1]), None if lse is None else wide(rec[2])
    total, slack = 0.0, 0.0
    for r in range(x.shape[0]):
        wr = 1.0 if w is None else w[r]
        L, dL, G, dG = plain_distill(xx[r], idx[r], vv[r], None if ll is None else ll[r], T, wr, scale, dtype)
        if np.isfinite(L):
            assert abs(rl[r] - L) <= dL, (r, rl[r], L, dL)
        else:
            assert np.array_equal(rl[r], L, equal_nan=True), (r, rl[r], L)
        if g is not None:
            got = wide(g[r])
            bad = ~(np.abs(got - G) <= dG) & ~(np.isnan(got) & np.isnan(G))
            assert not bad.any(), (r, np.flatnonzero(bad)[:5], got[bad][:5], G[bad][:5], dG[bad][:5])
        if wr != 0:
            total += wr * L
            slack += abs(wr) * dL
    total *= scale
    if np.isfinite(total):
        assert abs(lo - total) <= abs(scale) * slack + abs(total) * stat_u(dtype) * 2 + 2.0**-50 * abs(total) * (x.shape[0] + 8), (lo, total)
    else:
        assert np.array_equal(lo, total, equal_nan=True)
    return view, rec


def call_sample(sim, view, ld, u, dtype, rules=None, **rule):
    nrow, ncol = view.shape
    idx = torch.full((nrow + 1,), 77, dtype=torch.int32, device="cuda")
    lp = torch.full((nrow + 1,), 77.0, dtype=STAT[dtype], device="cuda")
    ut = torch.from_numpy(np.asarray(u, dtype=np.float64)).cuda()
    rt = None if rules is None else torch.from_numpy(np.asarray(rules, dtype=np.float64)).cuda()
    sim.sample_dev(view.data_ptr(), nrow, ncol, ut.data_ptr(), idx.data_ptr(), logp_ptr=lp.data_ptr(),
                   rules_ptr=0 if rt is None else rt.data_ptr(), dtype=dtype, ld=ld, **rule)
    torch.cuda.synchronize()
    assert idx[nrow] == 77 and lp[nrow] == 77
    return idx[:nrow].cpu().numpy(), wide(lp[:nrow])


def check_sample(sim, x, u, dtype, pad=0, offset=0, rules=None, **rule):
    buf, view, ld = place(x, dtype, pad, offset)
    idx, lp = call_sample(sim, view, ld, u, dtype, rules, **rule)
    xx = wide(view)
    for r in range(x.shape[0]):
        T, tk, tp, mp = rules[r] if rules is not None else (rule.get("temperature", 1.0), rule.get("top_k", 0),
                                                            rule.get("top_p", 1.0), rule.get("min_p", 0.0))
        i, l, may = plain_sample(xx[r], T, tk, tp, mp, u[r])
        assert idx[r] in may, (r, idx[r], i, may)
        if idx[r] == i and np.isfinite(l):
            n = len(xx[r])
            bits = min(52, 62 - math.ceil(math.log2(n)) if n > 1 else 62)
            assert abs(lp[r] - l) <= 2.0**-48 * (1 + abs(l)) + (n + 2) * 2.0**-bits + stat_u(dtype) * abs(l), (r, lp[r], l)
        elif idx[r] == i:
            assert np.array_equal(lp[r], l, equal_nan=True)
    return idx


# ------------------------------------------------------------------ top logits

SIZES = [(1, 1), (3, 2), (2, 31), (5, 33), (4, 257), (3, 1000), (2, 4099)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("nrow,ncol", SIZES)
def test_top_sizes(sim, dtype, nrow, ncol):
    rng = np.random.default_rng(nrow * 7919 + ncol)
    for k in sorted({1, 2, min(16, ncol), min(ncol, 1024), min(ncol + 3, 1024)}):
        check_top(sim, readouts(rng, nrow, ncol, dtype, 0.2 if k == 2 else 0.0), k, 1.7, dtype)


@pytest.mark.parametrize("dtype,ncol,k", [("f64", 60001, 300), ("f64", 196608, 1024), ("f32", 120007, 64), ("f16", 50001, 1024), ("bf16", 500009, 17)])
def test_top_long_rows(sim, dtype, ncol, k):
    rng = np.random.default_rng(ncol)
    check_top(sim, readouts(rng, 2, ncol, dtype, 0.1), k, 1.0, dtype)


@pytest.mark.parametrize("dtype", list(DT))
def test_top_strides_and_alignment(sim, dtype):
    rng = np.random.default_rng(5)
    for pad, offset in ((1, 0), (0, 1), (7, 3), (64, 8)):
        for ncol in (37, 302, 2050):
            check_top(sim, readouts(rng, 4, ncol, dtype), 9, 2.0, dtype, pad, offset)


@pytest.mark.parametrize("dtype", list(DT))
def test_top_hard_rows(sim, dtype):
    low = float(torch.finfo(DT[dtype]).min)
    rng = np.random.default_rng(3)
    for n in (40, 700, 9000):
        rows = [np.full(n, -np.inf), np.full(n, 1.5), np.full(n, low), np.zeros(n), rng.integers(0, 3, n).astype(float),
                np.where(rng.random(n) < 0.5, low, rng.standard_normal(n)), np.where(np.arange(n) == n - 1, 2.0, -np.inf),
                np.where(np.arange(n) % 2 == 0, 0.0, -0.0), np.linspace(5, -5, n), np.linspace(-5, 5, n),
                np.where(np.arange(n) == 3, np.inf, 1.0), np.where(np.arange(n) == n // 2, np.nan, 1.0), np.full(n, np.nan),
                1e-4 * rng.standard_normal(n), np.where(np.arange(n) == 0, 3e4, 1e-3 * rng.standard_normal(n)),
                np.where(np.arange(n) < 30, 1.0, -1.0)]
        for k in (1, 31, 64):
            check_top(sim, np.stack(rows), k, 0.9, dtype)


def test_top_many_distinct_close_values(sim):
    # distinct fp64 values whose differences from the row's largest round together in fp32, and in fp64
    n = 5000
    a = 1.0 + np.arange(n) * 2.0**-52
    b = np.where(np.arange(n) == 7, 1e6, -1.0 - np.random.default_rng(0).permutation(n) * 2.0**-52)
    c = np.where(np.arange(n) == 7, 1.0, np.random.default_rng(1).permutation(n) * 1e-300)
    check_top(sim, np.stack([a, a[::-1], b, c]), 1000, 1.0, "f64")


def test_top_empty_shapes(sim):
    check_top(sim, np.zeros((3, 0)), 4, 1.0, "f64")
    check_top(sim, np.zeros((0, 5)), 4, 1.0, "bf16")


def test_top_without_lse(sim):
    x = readouts(np.random.default_rng(0), 3, 100, "f32")
    buf, view, ld = place(x, "f32")
    idx, val, lse = call_top(sim, view, ld, 5, 1.0, "f32", lse=False)
    assert (lse == 77).all()
    assert np.array_equal(idx, np.argsort(-wide(view), axis=1, kind="stable")[:, :5])


# ------------------------------------------------------------------ distillation

def teacher(rng, x, k, T, rest, spread_=1.5):
    t = np.where(np.isfinite(x), x, 0.0) + spread_ * rng.standard_normal(x.shape)
    order = np.argsort(-t, axis=1, kind="stable")[:, :k]
    if order.shape[1] < k:  # more slots than readouts
        order = np.concatenate([order, np.full((len(x), k - order.shape[1]), -1)], 1)
    val = np.where(order >= 0, np.take_along_axis(t, np.maximum(order, 0), 1), -np.inf) if x.shape[1] else np.full(order.shape, -np.inf)
    m = t.max(1, keepdims=True) if x.shape[1] else np.zeros((len(x), 1))
    lse = (m[:, 0] / T + np.log(np.exp((t - m) / T).sum(1))) if rest and x.shape[1] else (np.zeros(len(x)) if rest else None)
    return order, val, lse


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("nrow,ncol", SIZES)
def test_distill_sizes(sim, dtype, nrow, ncol, rest):
    rng = np.random.default_rng(nrow * 31 + ncol)
    for k in sorted({1, min(16, ncol), min(40, ncol + 3)}):
        x = readouts(rng, nrow, ncol, dtype)
        check_distill(sim, x, *teacher(rng, x, k, 1.7, rest), 1.7, dtype, "f64" if dtype == "f64" else "f32")


@pytest.mark.parametrize("dtype,ncol,k", [("f64", 60001, 300), ("f64", 196608, 1024), ("f32", 120007, 64), ("f16", 50001, 1024), ("bf16", 500009, 17)])
def test_distill_long_rows(sim, dtype, ncol, k):
    rng = np.random.default_rng(ncol)
    x = readouts(rng, 2, ncol, dtype)
    for rest in (False, True):
        check_distill(sim, x, *teacher(rng, x, k, 1.0, rest), 1.0, dtype, dtype, scale=100.0)


@pytest.mark.parametrize("t_dtype", list(DT))
@pytest.mark.parametrize("dtype", list(DT))
def test_distill_types(sim, dtype, t_dtype):
    rng = np.random.default_rng(8)
    x = readouts(rng, 3, 400, dtype)
    for rest in (False, True):
        check_distill(sim, x, *teacher(rng, x, 20, 2.0, rest), 2.0, dtype, t_dtype, w=[0.5, -2.0, 1.0])


@pytest.mark.parametrize("dtype", list(DT))
def test_distill_strides_alignment_in_place(sim, dtype):
    rng = np.random.default_rng(5)
    for pad, offset, gpad in ((1, 0, 2), (0, 1, 0), (7, 3, 1), (64, 8, 64)):
        for ncol in (37, 302, 2050):
            x = readouts(rng, 4, ncol, dtype)
            rec = teacher(rng, x, 9, 2.0, True)
            view, r = check_distill(sim, x, *rec, 2.0, dtype, "f32", pad=pad, offset=offset, grad_ld=ncol + gpad)
            g, rl, lo = call_distill(sim, view, ncol + pad, r, 2.0, dtype, "f32", scale=0.25)
            n, rl1, lo1 = call_distill(sim, view, ncol + pad, r, 2.0, dtype, "f32", scale=0.25, grad=False)
            assert n is None and np.array_equal(rl, rl1) and lo == lo1
            p, rl2, lo2 = call_distill(sim, view, ncol + pad, r, 2.0, dtype, "f32", scale=0.25, in_place=True)
            assert torch.equal(p, g) and np.array_equal(rl, rl2) and lo == lo2


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("dtype", list(DT))
def test_distill_hard_rows(sim, dtype, rest):
    low = float(torch.finfo(DT[dtype]).min)
    rng = np.random.default_rng(4)
    for n in (33, 900):
        k = 12
        base = readouts(rng, 1, n, dtype)[0]
        rows = [np.full(n, -np.inf), np.full(n, 1.0), np.full(n, low), base, base, base, base,
                np.where(np.arange(n) == 5, np.nan, base), np.where(np.arange(n) == 5, np.nan, base),
                np.where(np.arange(n) % 3 == 0, -np.inf, base), np.where(np.arange(n) % 3 == 0, low, base)]
        x = np.stack(rows)
        order, val, lse = teacher(rng, x[[3]], k, 1.5, True)
        order, val, lse = np.repeat(order, len(x), 0), np.repeat(val, len(x), 0), np.repeat(lse, len(x), 0)
        order[3] = -1  # no slot used
        order[4, 1:] = order[4, 0]  # the same position in every slot
        val[5, 3:7] = -np.inf  # slots without mass
        order[6, 2], order[6, 4], order[6, 5] = n, 2**31 - 1, -(2**31)  # positions outside the row
        order[9] = np.array([i for i in range(n) if i % 3][:k])  # no slot on a closed readout
        w = np.ones(len(x))
        w[7] = 0.0  # a padded row that holds NaN
        check_distill(sim, x, order, val, lse if rest else None, 1.5, dtype, "f64", w=w)


def test_distill_closed_readout_in_a_slot(sim):
    # a teacher that wants a closed readout: infinite loss, finite gradients
    x = np.array([[0.0, -np.inf, 1.0, 2.0]])
    rec = record(np.array([[1, 3]]), np.array([[0.5, 0.25]]), None, "f64")
    buf, view, ld = place(x, "f64")
    g, rl, lo = call_distill(sim, view, ld, rec, 1.0, "f64", "f64")
    q = np.exp([0.5, 0.25])
    q /= q.sum()
    p = np.exp([0.0, -np.inf, 1.0, 2.0])
    p /= p.sum()
    assert rl[0] == np.inf and lo == np.inf
    assert np.allclose(wide(g[0]), p - np.array([0, q[0], 0, q[1]]), rtol=0, atol=2.0**-48)


def test_distill_all_positions_in_slots(sim):
    # no readout is outside the slots: the rest's term is left out
    rng = np.random.default_rng(6)
    for n in (2, 33, 600):
        x = readouts(rng, 2, n, "f64")
        check_distill(sim, x, *teacher(rng, x, n, 1.0, True), 1.0, "f64", "f64")


def test_distill_slots_without_mass(sim):
    # values far below the rest: q of 0 leaves a term out, whatever the readout
    x = np.array([[0.0, -np.inf, 1.0, 2.0]])
    check_distill(sim, x, np.array([[1, 3]]), np.array([[-5000.0, 0.25]]), None, 1.0, "f64", "f64")


@pytest.mark.parametrize("dtype", list(DT))
def test_distill_slots_far_from_the_largest(sim, dtype):
    # the readouts in the slots far below, or far above, nearly all of the row, by more than the types' exponents hold
    rng = np.random.default_rng(7)
    for n in (33, 700, 9000):
        x = rng.integers(-40, 40, (6, n)) * (0.25 if dtype in ("f16", "bf16") else 1.0)
        x[4] -= 500.0
        x[5] = np.where(np.arange(n) % 5 == 1, -np.inf, x[5])
        order = np.argsort(x, axis=1, kind="stable")[:, :6]
        order[3] = np.argsort(-x[3], kind="stable")[:6]
        order[5, :3] = [1, 6, 11]  # closed readouts in the first slots
        val = rng.standard_normal(order.shape)
        val[5, :3] = -5e5  # of no probability
        for T in (1.0, 0.04, 1e-4):
            check_distill(sim, x, order, val * T, None, T, dtype, "f64", scale=1.0 / T)


def test_distill_empty_shapes(sim):
    check_distill(sim, np.zeros((3, 0)), np.full((3, 2), 0), np.zeros((3, 2)), None, 1.0, "f64", "f64")
    check_distill(sim, np.zeros((0, 5)), np.zeros((0, 2)), np.zeros((0, 2)), np.zeros(0), 1.0, "f16", "f32")


def test_distill_many_rows_and_a_label(sim):
    # one slot, renormalised: the cross entropy with a label
    rng = np.random.default_rng(12)
    x = readouts(rng, 2000, 10, "f32")
    check_distill(sim, x, rng.integers(0, 10, (2000, 1)), np.full((2000, 1), 123.0), None, 1.0, "f32", "f32", scale=1 / 2000)


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("ncol", [7, 302, 5000])
def test_distill_gradient_by_differences(sim, rest, ncol):
    """Central differences of the loss: the error of step h is h^2 |L'''| / 6 + 2^-50 |L| / h, with |L'''| <= 6 / T."""
    rng = np.random.default_rng(ncol)
    T, h = 1.3, 1e-4
    x = readouts(rng, 1, ncol, "f64") + 65.0
    order, val, lse = teacher(rng, x, 5, T, rest)
    rec = record(order, val, lse, "f64")
    buf, view, ld = place(x, "f64")
    g, rl, lo = call_distill(sim, view, ld, rec, T, "f64", "f64")
    g = wide(g)[0]
    for i in [int(order[0, 0]), int(order[0, 3]), int(x[0].argmin()), int(x[0].argsort()[ncol // 2])]:
        side = []
        for s in (1, -1):
            y = x.copy()
            y[0, i] += s * h
            b, v, l = place(y, "f64")
            side.append(call_distill(sim, v, l, rec, T, "f64", "f64")[2])
        d = (side[0] - side[1]) / (2 * h)
        assert abs(d - g[i]) <= h * h / T + 2.0**-44 * abs(lo) / h, (i, d, g[i])


# ------------------------------------------------------------------ sampling

RULES = [dict(), dict(temperature=0.0), dict(temperature=0.6), dict(top_k=1), dict(top_k=5), dict(top_k=50, top_p=0.9),
         dict(top_p=0.5), dict(top_p=0.99, temperature=1.7), dict(top_p=0.0), dict(min_p=0.05), dict(min_p=1.0),
         dict(temperature=2.0, top_k=700, top_p=0.95, min_p=0.01), dict(top_k=100000), dict(top_p=0.97, min_p=0.2)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("ncol", [1, 2, 31, 33, 302, 1025, 4099])
def test_sample_sizes_and_rules(sim, dtype, ncol):
    rng = np.random.default_rng(ncol)
    for j, rule in enumerate(RULES):
        nrow = 1 + j % 4
        check_sample(sim, readouts(rng, nrow, ncol, dtype, 0.2 if j % 2 else 0.0), rng.random(nrow), dtype, **rule)


@pytest.mark.parametrize("dtype,ncol", [("f64", 60001), ("f64", 196608), ("f32", 120007), ("f16", 50001), ("bf16", 500009)])
def test_sample_long_rows(sim, dtype, ncol):
    rng = np.random.default_rng(ncol)
    x = readouts(rng, 2, ncol, dtype)
    for rule in (dict(temperature=1.2), dict(top_k=40, top_p=0.9), dict(top_k=5000, top_p=0.8), dict(top_p=0.9), dict(min_p=0.001)):
        check_sample(sim, x, rng.random(2), dtype, **rule)


@pytest.mark.parametrize("dtype", list(DT))
def test_sample_strides_and_alignment(sim, dtype):
    rng = np.random.default_rng(5)
    for pad, offset in ((1, 0), (0, 1), (7, 3), (64, 8)):
        for ncol in (37, 302, 2050):
            check_sample(sim, readouts(rng, 4, ncol, dtype), rng.random(4), dtype, pad, offset, temperature=1.5, top_p=0.9)


def test_sample_rules_per_row(sim):
    rng = np.random.default_rng(9)
    rules = [(1.0, 0, 1.0, 0.0), (0.0, 0, 1.0, 0.0), (-1.0, 0, 0.5, 0.0), (0.7, 3.9, 1.0, 0.0), (1.0, -5.0, 2.0, -1.0),
             (1.0, 0.5, 0.3, 0.0), (1.0, math.inf, 0.9, 0.0), (2.0, 10.0, -1.0, 0.0), (2.0, 0, 1.0, 7.0), (1.5, 20, 0.9, 0.05),
             (math.nan, 0, 1.0, 0.0), (1.0, 1e30, 0.99, 0.3)]
    for dtype in DT:
        for ncol in (20, 302, 3001):
            x = readouts(rng, len(rules), ncol, dtype)
            check_sample(sim, x, rng.random(len(rules)), dtype, rules=rules)
    # NaN in a switch turns it off
    x = readouts(rng, 1, 500, "f64")
    u = [0.7]
    buf, view, ld = place(x, "f64")
    a = call_sample(sim, view, ld, u, "f64", rules=[(1.0, math.nan, math.nan, math.nan)])
    b = call_sample(sim, view, ld, u, "f64")
    assert a[0][0] == b[0][0] and a[1][0] == b[1][0]


@pytest.mark.parametrize("dtype", list(DT))
def test_sample_hard_rows(sim, dtype):
    low = float(torch.finfo(DT[dtype]).min)
    rng = np.random.default_rng(3)
    for n in (40, 700, 9000):
        rows = [np.full(n, -np.inf), np.full(n, 1.5), np.full(n, low), rng.integers(0, 3, n).astype(float),
                np.where(rng.random(n) < 0.5, low, rng.standard_normal(n)), np.where(np.arange(n) == n - 1, 2.0, -np.inf),
                np.where(np.arange(n) % 2 == 0, 0.0, -0.0), np.where(np.arange(n) == 3, np.inf, 1.0),
                np.where(np.arange(n) == n // 2, np.nan, 1.0), 1e-4 * rng.standard_normal(n),
                np.where(np.arange(n) == 0, 3e4, 1e-3 * rng.standard_normal(n)), np.where(np.arange(n) < 30, 1.0, -1.0)]
        # fractions that keep the borders of equal weights away from top_p and u times the mass
        for rule in (dict(), dict(top_k=7), dict(top_p=0.6180339), dict(top_k=33, top_p=0.6180339), dict(min_p=0.017), dict(temperature=0.0)):
            check_sample(sim, np.stack(rows), rng.random(len(rows)), dtype, **rule)


def test_sample_of_extreme_numbers(sim):
    x = np.tile(np.array([[0.0, 1.0, 2.0, 3.0, 4.0]]), (6, 1))
    u = [0.0, 1.0 - 2.0**-53, 1.0, -3.0, math.nan, 7.0]
    buf, view, ld = place(x, "f64")
    idx, lp = call_sample(sim, view, ld, u, "f64")
    assert list(idx) == [4, 0, 0, 4, 4, 0]
    assert check_sample(sim, np.zeros((3, 0)), [0.1, 0.2, 0.3], "f32").tolist() == [-1, -1, -1]
    check_sample(sim, np.zeros((0, 4)), [], "f64")


def test_sample_ties_by_position(sim):
    # equal readouts are drawn in order of position: u walks through them
    n = 1000
    for dtype in DT:
        x = np.zeros((n, n))
        u = (np.arange(n) + 0.5) / n
        buf, view, ld = place(x, dtype)
        idx, lp = call_sample(sim, view, ld, u, dtype)
        assert np.array_equal(idx, np.arange(n))
        idx, lp = call_sample(sim, view, ld, u, dtype, top_k=100)
        assert np.array_equal(idx, np.arange(n) // 10)


def test_sample_frequencies(sim):
    """Counts of N draws: each is binomial, so 6 standard deviations hold a bin with 1 - 2e-9."""
    rng = np.random.default_rng(1)
    x = rng.standard_normal(13) * 1.5
    N = 40000
    buf, view, ld = place(np.tile(x, (N, 1)), "f32")
    idx, lp = call_sample(sim, view, ld, rng.random(N), "f32", temperature=0.8, top_k=9)
    xx = wide(view[0])
    p = np.exp(xx / 0.8) * (np.argsort(np.argsort(-xx)) < 9)
    p /= p.sum()
    got = np.bincount(idx, minlength=13)
    assert (np.abs(got - N * p) <= 6 * np.sqrt(N * p * (1 - p)) + 1e-9).all()
    assert np.abs(lp - np.log(p[idx])).max() <= 1e-6


# ------------------------------------------------------------------ calls as programs make them

@pytest.mark.parametrize("dtype", ["f64", "bf16"])
@pytest.mark.parametrize("nrow", [8, 90])
def test_long_rows_of_equal_readouts(sim, dtype, nrow):
    # rows shared by several blocks (few rows) and rows of a block (many): more equal readouts than any list of candidates holds
    rng = np.random.default_rng(17)
    n = 20011
    a = np.stack([np.full(n, -65.0), rng.integers(0, 3, n) * 1.0, np.where(rng.random(n) < 0.9, -np.inf, 0.0),
                  np.where(np.arange(n) < 40, rng.permutation(n) * 1e-3, -65.0), np.where(np.arange(n) % 2, -65.0, -65.5),
                  rng.standard_normal(n), np.full(n, -np.inf), np.where(np.arange(n) == n - 1, np.nan, 1.0)])
    x = np.concatenate([a, np.tile(rng.standard_normal((1, n)), (nrow - 8, 1))]) if nrow > 8 else a
    check_top(sim, x, 100, 1.0, dtype)
    u = rng.random(nrow)
    for rule in (dict(), dict(top_p=0.6180339), dict(top_k=64, top_p=0.6180339), dict(top_k=3000), dict(temperature=0.01, min_p=0.017), dict(temperature=0.0)):
        check_sample(sim, x, u, dtype, **rule)
    order, val, lse = teacher(rng, np.where(np.isfinite(x), x, 0.0), 30, 1.0, True)
    check_distill(sim, x, order, val, lse, 1.0, dtype, "f64", scale=10.0)


@pytest.mark.parametrize("dtype,nrow,ncol,k", [("f64", 2000, 700, 200), ("bf16", 2000, 700, 200), ("f64", 700, 2500, 130), ("f32", 700, 2500, 130),
                                               ("f64", 80, 60001, 300), ("f16", 90, 300007, 40), ("f64", 9000, 33, 40)])
def test_more_rows_than_the_card_holds_at_once(sim, dtype, nrow, ncol, k):
    # teams take several rows in turn: rows without weight, without slots, with NaN and closed ones among them, in every order
    rng = np.random.default_rng(nrow + ncol)
    x = readouts(rng, nrow, ncol, dtype)
    kind = rng.integers(0, 8, nrow)
    x[kind == 1, 0] = np.nan
    x[kind == 2] = -np.inf
    check_top(sim, x, min(k, ncol), 1.0, dtype)
    check_sample(sim, x, rng.random(nrow), dtype, temperature=1.3, top_p=0.9)
    rules = np.stack([0.5 + rng.random(nrow), rng.integers(0, 2 * k, nrow) * (rng.random(nrow) < 0.6), 0.3 + 0.6 * rng.random(nrow),
                      0.1 * rng.random(nrow) * (rng.random(nrow) < 0.5)], 1)
    check_sample(sim, x, rng.random(nrow), dtype, rules=rules)
    order, val, lse = teacher(rng, np.where(np.isfinite(x), x, 0.0), k, 1.0, True)
    order[kind == 3] = -1
    w = np.where((kind == 4) | (kind == 5), 0.0, 1.0)
    for rest in (False, True):
        check_distill(sim, x, order, val, lse if rest else None, 1.0, dtype, dtype, w=w, scale=1.0)


def test_offsets_beyond_32_bits(sim):
    ncol, ld = 1001, 2**31 + 24
    a = readouts(np.random.default_rng(3), 2, ncol, "f16")
    buf = torch.empty(ld + ncol, dtype=torch.float16, device="cuda")
    view = buf.as_strided((2, ncol), (ld, 1))
    view.copy_(torch.from_numpy(a).half())
    xx = wide(view)
    idx, val, lse = call_top(sim, view, ld, 5, 1.0, "f16")
    for r in range(2):
        i, v, l = plain_top(xx[r], 5, 1.0)
        assert np.array_equal(idx[r], i) and np.array_equal(val[r], v)
    c, lp = call_sample(sim, view, ld, [0.3, 0.8], "f16")
    assert all(c[r] in plain_sample(xx[r], 1.0, 0, 1.0, 0.0, [0.3, 0.8][r])[2] for r in range(2))
    rec = record(idx, val, lse, "f32")
    # rows of the same alignment: another one may add a row's terms up in another order
    near, near_view, near_ld = place(a, "f16", pad=7)
    assert torch.equal(near_view, view) and near_ld * 2 % 16 == ld * 2 % 16 == 0
    want, rl, lo = call_distill(sim, near_view, near_ld, rec, 1.0, "f16", "f32")
    got, rl2, lo2 = call_distill(sim, view, ld, rec, 1.0, "f16", "f32", in_place=True)
    assert torch.equal(got, want) and np.array_equal(rl, rl2) and lo == lo2


def test_two_contexts_at_once():
    # calls of two contexts on streams of their own, from two threads
    import threading

    from heliox_b200.runtime import Sim

    rng = np.random.default_rng(4)
    want, got, sims = [], [None, None], []
    data = [readouts(rng, 60, 9001, "f64") for _ in range(2)]
    for j in range(2):
        s = Sim(0)
        s.set_stream(torch.cuda.Stream().cuda_stream)
        sims.append(s)
        buf, view, ld = place(data[j], "f64")
        want.append((view, call_top(s, view, ld, 20, 1.0, "f64")))

    def work(j):
        for _ in range(5):
            got[j] = call_top(sims[j], want[j][0], 9001, 20, 1.0, "f64")

    ts = [threading.Thread(target=work, args=(j,)) for j in range(2)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    for j in range(2):
        assert all(np.array_equal(a, b) for a, b in zip(got[j], want[j][1]))
        sims[j].close()


def test_same_bits_twice_and_whatever_the_batch(sim):
    rng = np.random.default_rng(2)
    for dtype, n in (("f64", 302), ("f64", 9001), ("bf16", 30011), ("f32", 120)):
        x = readouts(rng, 9, n, dtype)
        order, val, lse = teacher(rng, x, 30, 1.0, True)
        u = rng.random(9)
        buf, view, ld = place(x, dtype)
        rec = record(order, val, lse, "f32")
        one = (call_top(sim, view, ld, 30, 1.0, dtype), call_distill(sim, view, ld, rec, 1.0, dtype, "f32"), call_sample(sim, view, ld, u, dtype, top_p=0.9))
        two = (call_top(sim, view, ld, 30, 1.0, dtype), call_distill(sim, view, ld, rec, 1.0, dtype, "f32"), call_sample(sim, view, ld, u, dtype, top_p=0.9))
        for a, b in zip(one, two):
            for p, q in zip(a, b):
                assert torch.equal(p, q) if isinstance(p, torch.Tensor) else np.array_equal(p, q)


def test_another_stream_capture_and_two_graphs(sim):
    """The three as one captured run, replayed on new inputs; two graphs of one context side by side."""
    from heliox_b200.runtime import Sim

    rng = np.random.default_rng(20)
    nrow, ncol, k = 50, 302, 8
    s = Sim(0)
    before = torch.cuda.current_device()
    sets = []
    for j in range(2):
        st = torch.cuda.Stream()
        d = dict(st=st, t=torch.empty((nrow, ncol), dtype=torch.float64, device="cuda"), x=torch.empty((nrow, ncol), dtype=torch.float64, device="cuda"),
                 u=torch.empty(nrow, dtype=torch.float64, device="cuda"), i=torch.empty((nrow, k), dtype=torch.int32, device="cuda"),
                 v=torch.empty((nrow, k), dtype=torch.float64, device="cuda"), l=torch.empty(nrow, dtype=torch.float64, device="cuda"),
                 g=torch.empty((nrow, ncol), dtype=torch.float64, device="cuda"), rl=torch.empty(nrow, dtype=torch.float64, device="cuda"),
                 lo=torch.empty(1, dtype=torch.float64, device="cuda"), c=torch.empty(nrow, dtype=torch.int32, device="cuda"),
                 lp=torch.empty(nrow, dtype=torch.float64, device="cuda"))

        def calls(d=d):
            s.top_logits_dev(d["t"].data_ptr(), nrow, ncol, k, d["i"].data_ptr(), d["v"].data_ptr(), lse_ptr=d["l"].data_ptr(), temperature=2.0)
            s.distill_loss_grad_dev(d["x"].data_ptr(), nrow, ncol, k, d["i"].data_ptr(), d["v"].data_ptr(), d["g"].data_ptr(),
                                    d["rl"].data_ptr(), d["lo"].data_ptr(), t_lse_ptr=d["l"].data_ptr(), temperature=2.0)
            s.sample_dev(d["x"].data_ptr(), nrow, ncol, d["u"].data_ptr(), d["c"].data_ptr(), logp_ptr=d["lp"].data_ptr(), temperature=2.0, top_p=0.9)

        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):  # the first call of all is a captured one
            s.set_stream(st.cuda_stream)
            calls()
        d["graph"], d["calls"] = graph, calls
        sets.append(d)
    for rep in range(3):
        ins = []
        for d in sets:
            t, x, u = readouts(rng, nrow, ncol, "f64"), readouts(rng, nrow, ncol, "f64"), rng.random(nrow)
            ins.append((t, x, u))
            for name, a in (("t", t), ("x", x), ("u", u)):
                d[name].copy_(torch.from_numpy(a))
        torch.cuda.synchronize()
        for d in sets:
            with torch.cuda.stream(d["st"]):
                d["graph"].replay()
        torch.cuda.synchronize()
        for d, (t, x, u) in zip(sets, ins):
            got = {n: d[n].clone() for n in ("i", "v", "l", "g", "rl", "lo", "c", "lp")}
            for r in range(nrow):
                i, v, l = plain_top(t[r], k, 2.0)
                assert np.array_equal(wide(got["i"][r]), i)
                L, dL, G, dG = plain_distill(x[r], i, v, float(got["l"][r]), 2.0, 1.0, 1.0 / nrow, "f64")
                assert abs(float(got["rl"][r]) - L) <= dL and (np.abs(wide(got["g"][r]) - G) <= dG).all()
                assert int(got["c"][r]) in plain_sample(x[r], 2.0, 0, 0.9, 0.0, u[r])[2]
            for n in ("i", "v", "l", "g", "rl", "lo", "c", "lp"):
                d[n].zero_()
            s.set_stream(torch.cuda.current_stream().cuda_stream)
            d["calls"]()
            torch.cuda.synchronize()
            assert all(torch.equal(got[n], d[n]) for n in got)  # eager and captured give the same bits
    assert torch.cuda.current_device() == before
    s.close()


def test_refusals_leave_the_context_usable(sim):
    from heliox_b200.runtime import HxError

    x = torch.zeros((2, 4), dtype=torch.float64, device="cuda")
    i = torch.zeros((2, 4), dtype=torch.int32, device="cuda")
    with pytest.raises(HxError, match="k must"):
        sim.top_logits_dev(x.data_ptr(), 2, 4, 0, i.data_ptr(), x.data_ptr())
    with pytest.raises(HxError, match="overlaps"):
        sim.distill_loss_grad_dev(x.data_ptr(), 2, 4, 1, i.data_ptr(), x.data_ptr(), x.data_ptr() + 8, x.data_ptr(), x.data_ptr())
    with pytest.raises(HxError, match="top_p"):
        sim.sample_dev(x.data_ptr(), 2, 4, x.data_ptr(), i.data_ptr(), top_p=1.5)
    check_top(sim, np.eye(4), 2, 1.0, "f64")


@pytest.mark.parametrize("ncol,k,dtype,t_dtype,rest", [(302, 129, "f64", "f64", True), (302, 150, "f64", "f32", False), (302, 204, "f64", "bf16", True),
                                                       (302, 205, "f64", "f64", False), (512, 128, "f64", "f64", True), (512, 129, "f32", "f32", True),
                                                       (512, 150, "bf16", "bf16", False), (512, 204, "f64", "f32", True), (512, 205, "f16", "f64", True)])
def test_distill_many_slots_on_many_short_rows(sim, ncol, k, dtype, t_dtype, rest):
    # each team takes several rows, whose records differ: dropped and doubled positions, other ones in every row
    rng = np.random.default_rng(ncol * 1000 + k)
    nrow = 8000
    x = readouts(rng, nrow, ncol, dtype)
    order, val, lse = teacher(rng, x, k, 2.0, rest)
    mix = rng.permuted(np.tile(np.arange(k), (nrow, 1)), axis=1)
    order, val = np.take_along_axis(order, mix, 1), np.take_along_axis(val, mix, 1)
    r = np.arange(nrow)
    order[r, rng.integers(0, k, nrow)] = order[r, rng.integers(0, k, nrow)]
    order[rng.random(order.shape) < 0.1] = -1
    check_distill(sim, x, order, val, lse, 2.0, dtype, t_dtype, scale=1.0)


@pytest.mark.parametrize("dtype,nrow,ncol", [("f64", 700, 2051), ("f32", 1200, 2053), ("bf16", 1200, 4099), ("f16", 1300, 611), ("f64", 40, 20001), ("f64", 5000, 37)])
def test_edges_of_unaligned_rows(sim, dtype, nrow, ncol):
    # rows that start inside a vector, NaN between them: the largest readouts stand at the row's ends, which lanes copy for one another
    rng = np.random.default_rng(nrow + ncol)
    x = readouts(rng, nrow, ncol, dtype)
    at = np.where(rng.random(nrow) < 0.5, rng.integers(0, 9, nrow), ncol - 1 - rng.integers(0, 9, nrow))
    r = np.arange(nrow)
    x[r, at] = (-65.0 if dtype == "f64" else 0.0) + 60.0 + rng.integers(0, 30, nrow)
    for pad, offset in ((1, 1), (3, 0)):
        check_top(sim, x, 5, 1.0, dtype, pad, offset)
        assert np.array_equal(check_sample(sim, x, rng.random(nrow), dtype, pad, offset, top_k=3), at)
        assert np.array_equal(check_sample(sim, x, rng.random(nrow), dtype, pad, offset), at)
        # the slots' readouts are the smallest: the loss reads the row again and seeks its largest
        order = np.argsort(x, axis=1, kind="stable")[:, :4]
        check_distill(sim, x, order, rng.standard_normal(order.shape), None, 0.25, dtype, "f64", scale=4.0, pad=pad, offset=offset, grad_ld=ncol + 2)


def test_two_threads_with_rows_of_other_lengths():
    # the same kernel with more and with less shared memory, from two threads that call without a pause
    import ctypes as C
    import os
    import subprocess

    from heliox_b200 import _lib
    from heliox_b200.runtime import Sim

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    out = os.path.join(root, "tests", "capi", "_build")
    os.makedirs(out, exist_ok=True)
    so = os.path.join(out, "two_threads.so")
    subprocess.run(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-I" + os.path.join(root, "include"),
                    os.path.join(root, "tests", "capi", "two_threads.cpp"), "-o", so, "-L" + os.path.join(root, "heliox_b200"), "-lhx_b200",
                    "-Wl,-rpath," + os.path.join(root, "heliox_b200"), "-pthread"], check=True)
    nrow, k, rng = 2, 8, np.random.default_rng(6)
    sims, views, idx, val = [], [], [], []
    for n in (60000, 45000):
        sims.append(Sim(0))
        views.append(place(rng.standard_normal((nrow, n)), "f64")[1])
        idx.append(torch.empty((nrow, k), dtype=torch.int32, device="cuda"))
        val.append(torch.empty((nrow, k), dtype=torch.float64, device="cuda"))
    torch.cuda.synchronize()
    two = C.CDLL(so).two_threads
    two.argtypes = [C.c_void_p, C.c_void_p, C.c_int, C.c_void_p, C.c_void_p, C.c_int]
    ptrs = [(C.c_void_p * 2)(*a) for a in ([s._ctx for s in sims], [t.data_ptr() for t in idx], [t.data_ptr() for t in val])]
    rows = (_lib.Readout * 2)(*[_lib.Readout(v.data_ptr(), 0, nrow, v.shape[1], v.shape[1]) for v in views])
    assert two(ptrs[0], rows, k, ptrs[1], ptrs[2], 20000) == 0
    torch.cuda.synchronize()
    for j in range(2):
        assert np.array_equal(idx[j].cpu().numpy(), np.argsort(-wide(views[j]), axis=1, kind="stable")[:, :k])
        sims[j].close()


def test_calls_of_other_lengths_in_one_graph(sim):
    # a long row's call keeps its shared memory when shorter rows follow, in a graph that is put together after both
    from heliox_b200.runtime import Sim

    rng = np.random.default_rng(7)
    s, st = Sim(0), torch.cuda.Stream()
    parts = []
    for n in (20001, 7001, 9001):
        buf, view, ld = place(rng.standard_normal((150, n)), "f64")
        parts.append((n, view, torch.empty((150, 4), dtype=torch.int32, device="cuda"), torch.empty((150, 4), dtype=torch.float64, device="cuda")))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        s.set_stream(st.cuda_stream)
        for n, view, i, v in parts:
            s.top_logits_dev(view.data_ptr(), 150, n, 4, i.data_ptr(), v.data_ptr())
    graph.replay()
    torch.cuda.synchronize()
    for n, view, i, v in parts:
        assert np.array_equal(i.cpu().numpy(), np.argsort(-wide(view), axis=1, kind="stable")[:, :4])
    s.close()


@pytest.mark.parametrize("dtype", list(DT))
def test_nan_of_either_sign(sim, dtype):
    # a NaN outside the slots, with its sign bit set (as the host's and the device's invalid operations make it) and clear
    bits = {"f64": (0xFFF8 << 48, torch.int64, 64), "f32": (0xFFC0 << 16, torch.int32, 32), "f16": (0xFE00, torch.int16, 16), "bf16": (0xFFC0, torch.int16, 16)}
    word, itype, size = bits[dtype]
    rng = np.random.default_rng(11)
    for nrow, n in ((3, 40), (3, 700), (200, 9000), (3, 60001)):
        x = readouts(rng, nrow, n, dtype)
        order, val, lse = teacher(rng, x, 6, 1.0, True)
        free = [next(i for i in range(n - 1, 0, -1) if i not in order[r]) for r in (0, 1)]
        buf, view, ld = place(x, dtype)
        view.view(itype)[0, free[0]] = word - (1 << size)
        view.view(itype)[1, free[1]] = word - (1 << (size - 1))
        xx = wide(view)
        assert np.isnan(xx[0, free[0]]) and np.isnan(xx[1, free[1]])
        idx, v, ls = call_top(sim, view, ld, 6, 1.0, dtype)
        assert (idx[:2] == -1).all() and np.isnan(v[:2]).all() and np.isnan(ls[:2]).all() and (idx[2:] >= 0).all()
        c, lp = call_sample(sim, view, ld, rng.random(nrow), dtype)
        assert (c[:2] == -2).all() and np.isnan(lp[:2]).all() and (c[2:] >= 0).all()
        for rest in (False, True):
            g, rl, lo = call_distill(sim, view, ld, record(order, val, lse if rest else None, "f64"), 1.0, dtype, "f64")
            assert np.isnan(rl[:2]).all() and np.isnan(wide(g[:2])).all() and math.isnan(lo)
            assert np.isfinite(rl[2:]).all() and torch.isfinite(g[2:]).all()


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("nrow,n", [(3, 40), (3, 700), (200, 5003), (3, 60001), (4000, 120)])
def test_distill_rest_far_below_the_slots(sim, dtype, nrow, n):
    """Rows whose readouts outside the slots lie further below than the types' exponents reach, in logarithms:
    log p_r = max / T + log S' - log S is off by E (of S' and S) + 2^-50 |log p_r|; a share e' / S' by 2 E and 3 u |z|
    (within E); q_r by N as above."""
    rng = np.random.default_rng(n)
    k, T, scale = 3, 0.5, 2.0
    x = rng.integers(0, 8, (nrow, n)) * 0.25
    gap = rng.choice([10.0, 21.0, 24.0, 40.0, 47.0, 60.0, 174.0, 360.0, 375.0, 1000.0], nrow)
    order = np.argsort(rng.random((nrow, n)), axis=1)[:, :k]
    r = np.arange(nrow)[:, None]
    x[rng.random(x.shape) < 0.1] = -np.inf
    x[r, order] = gap[:, None] + [2.0, 0.0, 1.0]
    x[0, np.setdiff1d(np.arange(n), order[0])] = -np.inf  # nothing is open outside: no term
    val = np.tile([1.0, 0.25, 0.5], (nrow, 1))
    lse = val.max(1) / T + 1.0
    buf, view, ld = place(x, dtype)
    xx, rec = wide(view), record(order, val, lse, "f64")
    g, rl, lo = call_distill(sim, view, ld, rec, T, dtype, "f64", scale=scale)
    g = wide(g)
    noise = 2.0**-50 * (k + 8 + np.abs(val).max() / T)
    with np.errstate(divide="ignore", invalid="ignore", over="ignore"):
        for i in range(nrow):
            a = np.zeros(n, bool)
            a[order[i]] = True
            z = (xx[i] - xx[i].max()) / T
            logS = math.log(np.exp(z).sum())
            lq = val[i] / T - lse[i]
            q, lp = np.exp(lq), z[order[i]] - logS
            qr = 1.0 - q.sum()
            top = z[~a].max()
            E = row_error(xx[i][a], T, dtype) + (row_error(xx[i][~a], T, dtype) if top > -np.inf else 0.0)
            L, dL = (q * (lq - lp)).sum(), (q * (E + noise * (2 + np.abs(lq - lp) + np.abs(lp)))).sum()
            if top > -np.inf:
                e = np.where(a, 0.0, np.exp(z - top))
                share, lpr = e / e.sum(), top + math.log(e.sum()) - logS
                L += qr * (math.log(qr) - lpr)
                dL += 2 * E * qr + noise * (abs(math.log(qr)) + 2 * abs(lpr) + 2)
            else:
                share, qr = np.zeros(n), 0.0
            c, p = scale * T, np.exp(z - logS)
            G = c * ((q.sum() + qr) * p - qr * share)
            G[order[i]] -= c * q
            dG = c * ((p + share) * (2 * E + 3 * noise) + np.where(a, noise, 0.0)) + np.abs(G) * HALF[dtype] * (1 + 2.0**-20) + TINY[dtype] * (1 + 2.0**-8)
            assert abs(rl[i] - T * T * L) <= T * T * (dL + 2 * stat_u(dtype) * abs(L)), (i, gap[i], rl[i], T * T * L)
            assert (np.abs(g[i] - G) <= dG).all(), (i, gap[i], np.abs(g[i] - G).max())


@pytest.mark.parametrize("dtype", ["f64", "f32", "bf16"])
@pytest.mark.parametrize("n", [40, 700, 9000])
def test_distill_factors_beyond_fp32(sim, dtype, n):
    # products within the type's range whose factors are not: a loss scale of 1e27 with a rest e^-41 below, one of 1e-32 with
    # slots e^-25 below; errors as for every gradient, relative to the shares
    rng = np.random.default_rng(n)
    h = HALF[dtype]
    x = np.full((1, n), 1.0) + rng.integers(0, 4, (1, n)) * 0.25
    x[0, 3], x[0, 7] = 42.0, -np.inf
    buf, view, ld = place(x, dtype)
    g, rl, lo = call_distill(sim, view, ld, record(np.array([[3]]), np.zeros((1, 1)), np.array([0.5]), "f64"), 1.0, dtype, "f64", scale=1e27)
    z = wide(view)[0] - 42.0
    out, qr = np.where(np.arange(n) == 3, 0.0, np.exp(z)), 1.0 - math.exp(-0.5)
    p = np.exp(z) / np.exp(z).sum()
    G = 1e27 * np.where(np.arange(n) == 3, p - math.exp(-0.5), p - qr * out / out.sum())
    got = wide(g[0])
    assert got[7] == 0.0 and (np.abs(got - G) <= (h + 2 * row_error(wide(view)[0], 1.0, dtype)) * (np.abs(G) + 1e27 * p)).all()

    x = rng.integers(0, 8, (1, n)) * 0.25
    x[0, 5] = -25.0
    buf, view, ld = place(x, dtype)
    g, rl, lo = call_distill(sim, view, ld, record(np.array([[5]]), np.zeros((1, 1)), None, "f64"), 1.0, dtype, "f64", scale=1e-32)
    z = wide(view)[0] - wide(view)[0].max()
    p = np.exp(z) / np.exp(z).sum()
    G = 1e-32 * (p - (np.arange(n) == 5))
    got = wide(g[0])
    assert (np.abs(got - G) <= (h + 2 * row_error(wide(view)[0], 1.0, dtype)) * np.abs(G)).all()


def test_distill_as_many_rows_as_an_int_counts(sim):
    # 30 GB: every row's loss is log 2, the last one's log(1 + e)
    nrow = 2**31 - 1
    x = torch.zeros((nrow, 2), dtype=torch.bfloat16, device="cuda")
    x[-1, 1] = 1.0
    ti, tv = torch.zeros((nrow, 1), dtype=torch.int32, device="cuda"), torch.zeros((nrow, 1), dtype=torch.bfloat16, device="cuda")
    rl, lo = torch.zeros(nrow, dtype=torch.float32, device="cuda"), torch.zeros(1, dtype=torch.float32, device="cuda")
    sim.distill_loss_grad_dev(x.data_ptr(), nrow, 2, 1, ti.data_ptr(), tv.data_ptr(), 0, rl.data_ptr(), lo.data_ptr(), dtype="bf16")
    torch.cuda.synchronize()
    u = 2.0**-24
    assert abs(float(rl[-1]) - math.log(1 + math.e)) <= 40 * u
    assert abs(float(rl[:-1].min()) - math.log(2)) <= 40 * u and abs(float(rl[:-1].max()) - math.log(2)) <= 40 * u
    assert abs(float(lo[0]) - math.log(2)) <= 40 * u  # their mean
    del x, ti, tv, rl
    torch.cuda.empty_cache()

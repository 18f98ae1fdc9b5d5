"""Operators over readout rows: what is measured, with their plain forms.

A probe trace is a matrix of readouts, one row per step and one column per
probe.  Three operators work on such rows (of fp64 traces, or of fp32, fp16 and
bf16 logits of another model):

* ``top``: a teacher's record -- each row's k largest readouts with their
  positions, and the row's log-sum-exp at a temperature;
* ``distill``: the loss of a student's rows against such a record, with its
  gradient with respect to every readout;
* ``sample``: one choice per row from given uniform numbers, with temperature,
  top-k, top-p and min-p, and its log-probability.

``own`` False: plain torch; True: the framework's entry points.
"""
import math

import torch

own = False

DTYPES = {"f64": torch.float64, "f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BYTES = {"f64": 8, "f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # one decision of a 302-cell network: a single row, latency counts
        {"name": "sample_one_302_f64", "op": "sample", "dtype": "f64", "nrow": 1, "ncol": 302, "temperature": 2.0, "top_k": 0, "top_p": 0.9, "min_p": 0.0, "rules": False, "masked": False},
        # a decision at every step of a 200 ms trial of the 302-cell network, some choices closed
        {"name": "sample_trial_302_f64", "op": "sample", "dtype": "f64", "nrow": 8001, "ncol": 302, "temperature": 2.0, "top_k": 0, "top_p": 0.95, "min_p": 0.02, "rules": False, "masked": True},
        # answers of a batch, each row with settings of its own
        {"name": "sample_batch_32000_f32", "op": "sample", "dtype": "f32", "nrow": 64, "ncol": 32000, "temperature": 0.8, "top_k": 50, "top_p": 0.95, "min_p": 0.0, "rules": True, "masked": False},
        # sampled labels over every cell of the 10,000-cell network
        {"name": "sample_cells_10000_f64", "op": "sample", "dtype": "f64", "nrow": 2000, "ncol": 10000, "temperature": 3.0, "top_k": 0, "top_p": 0.9, "min_p": 0.0, "rules": False, "masked": False},
        # the record of one teacher row with a long output, latency counts
        {"name": "top_one_50001_bf16", "op": "top", "dtype": "bf16", "nrow": 1, "ncol": 50001, "temperature": 1.0, "k": 32, "masked": False},
        # a teacher trial of the 302-cell network
        {"name": "top_trial_302_f64", "op": "top", "dtype": "f64", "nrow": 8001, "ncol": 302, "temperature": 2.0, "k": 16, "masked": False},
        # a teacher trial of the 10,000-cell network (100 ms)
        {"name": "top_cells_10000_f64", "op": "top", "dtype": "f64", "nrow": 4000, "ncol": 10000, "temperature": 3.0, "k": 64, "masked": False},
        # the record of another model's batch of outputs
        {"name": "top_batch_32000_f16", "op": "top", "dtype": "f16", "nrow": 1024, "ncol": 32000, "temperature": 1.0, "k": 100, "masked": False},
        # labels (one slot) on a handful of rows
        {"name": "distill_label_10_f32", "op": "distill", "dtype": "f32", "t_dtype": "f32", "nrow": 60, "ncol": 10, "temperature": 1.0, "k": 1, "tail": False, "masked": False},
        # a student trial of the 302-cell network, rows before the stimulus without weight
        {"name": "distill_trial_302_f64", "op": "distill", "dtype": "f64", "t_dtype": "f64", "nrow": 8000, "ncol": 302, "temperature": 2.0, "k": 16, "tail": True, "masked": True},
        # a student trial of the 10,000-cell network (100 ms)
        {"name": "distill_cells_10000_f64", "op": "distill", "dtype": "f64", "t_dtype": "f64", "nrow": 4000, "ncol": 10000, "temperature": 3.0, "k": 64, "tail": True, "masked": False},
        # a 16-bit student with a long output, renormalised top logits
        {"name": "distill_batch_32003_bf16", "op": "distill", "dtype": "bf16", "t_dtype": "bf16", "nrow": 1021, "ncol": 32003, "temperature": 1.5, "k": 50, "tail": False, "masked": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["sample", "top", "distill"])
    dtype = rng.choice(["f64", "f64", "f32", "f16", "bf16"])
    ncol = _log_int(rng, 2, 60000)
    most = 20_000_000 if op == "sample" else 40_000_000
    nrow = _log_int(rng, 1, max(1, min(9000, most // ncol)))
    c = {"op": op, "dtype": dtype, "nrow": nrow, "ncol": ncol, "masked": rng.random() < 0.3,
         "temperature": round(rng.uniform(1.0, 4.0) if dtype == "f64" else rng.uniform(0.5, 2.0), 3)}
    if op == "sample":
        c["top_k"] = rng.choice([0, 0, _log_int(rng, 1, 1000)])
        c["top_p"] = rng.choice([1.0, round(rng.uniform(0.1, 0.99), 3)])
        c["min_p"] = rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.3), 4)])
        c["rules"] = rng.random() < 0.3
    else:
        c["k"] = _log_int(rng, 1, min(512, ncol))
    if op == "distill":
        c["t_dtype"] = rng.choice([dtype, "f32"])
        c["tail"] = rng.random() < 0.5
    return c


def _readouts(case, gen):
    """Membrane potentials (mV) with a few depolarised probes for fp64 rows, logits with a spread of a few units for the others."""
    shape = (case["nrow"], case["ncol"])
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float64 if case["dtype"] == "f64" else torch.float32)
    if case["dtype"] == "f64":
        up = torch.rand(shape, generator=gen, device="cuda", dtype=torch.float32) < 0.01
        x.mul_(2.5).sub_(65.0)
        x += up * (10.0 + 5.0 * torch.rand(shape, generator=gen, device="cuda", dtype=torch.float32))
    else:
        x.mul_(2.0)
        x += 3.0 * (torch.rand(shape, generator=gen, device="cuda", dtype=torch.float32) < 0.002)
    return x


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    nrow, ncol, dt = case["nrow"], case["ncol"], DTYPES[case["dtype"]]
    stat = torch.float64 if case["dtype"] == "f64" else torch.float32
    x = _readouts(case, gen)
    s = {"case": case}
    if case["op"] == "distill":
        k, tdt = case["k"], DTYPES[case["t_dtype"]]
        tstat = torch.float64 if case["t_dtype"] == "f64" else torch.float32
        # the teacher: the student's readouts and differences of its own; its record as a program keeps it
        t = (x + 1.5 * torch.randn((nrow, ncol), generator=gen, device="cuda", dtype=x.dtype)).to(tdt)
        v, i = torch.topk(t.to(x.dtype), k, dim=1)
        s["t_idx"], s["t_val"] = i.to(torch.int32).contiguous(), v.to(tdt).contiguous()
        s["t_lse"] = torch.logsumexp(t.to(x.dtype) / case["temperature"], 1).to(tstat) if case["tail"] else None
        s["w"] = None
        if case["masked"]:  # rows without weight, and slots that are not used
            s["w"] = (torch.rand(nrow, generator=gen, device="cuda") < 0.8).double() * 0.5
            gone = torch.rand((nrow, k), generator=gen, device="cuda") < 0.1
            s["t_idx"][gone] = -1
        s["grad"] = torch.empty((nrow, ncol), device="cuda", dtype=dt)
        s["row_loss"] = torch.empty(nrow, device="cuda", dtype=stat)
        s["loss"] = torch.empty(1, device="cuda", dtype=stat)
    elif case["masked"]:  # closed choices
        x.masked_fill_(torch.rand((nrow, ncol), generator=gen, device="cuda", dtype=torch.float32) < 0.15, -math.inf)
    s["x"] = x.to(dt)
    if case["op"] == "top":
        s["idx"] = torch.empty((nrow, case["k"]), device="cuda", dtype=torch.int32)
        s["val"] = torch.empty((nrow, case["k"]), device="cuda", dtype=dt)
        s["lse"] = torch.empty(nrow, device="cuda", dtype=stat)
    if case["op"] == "sample":
        s["u"] = torch.rand(nrow, generator=gen, device="cuda", dtype=torch.float64)
        s["rules"] = None
        if case["rules"]:  # each row's temperature, top_k, top_p, min_p
            f = 0.5 + torch.rand((nrow, 4), generator=gen, device="cuda", dtype=torch.float64)
            r = torch.empty((nrow, 4), device="cuda", dtype=torch.float64)
            r[:, 0] = case["temperature"] * f[:, 0]
            r[:, 1] = torch.floor(case["top_k"] * f[:, 1])
            r[:, 2] = torch.clamp(case["top_p"] * f[:, 2], max=1.0)
            r[:, 3] = torch.clamp(case["min_p"] * f[:, 3], max=1.0)
            s["rules"] = r
        s["idx"] = torch.empty(nrow, device="cuda", dtype=torch.int32)
        s["logp"] = torch.empty(nrow, device="cuda", dtype=stat)
    return s


# ------------------------------------------------------------------ plain forms

def _plain_top(s):
    c = s["case"]
    x = s["x"] if c["dtype"] == "f64" else s["x"].float()
    v, i = torch.sort(x, dim=1, descending=True, stable=True)
    k = c["k"]
    v, i = v[:, :k], i[:, :k].to(torch.int32)
    i = torch.where(v == -math.inf, torch.full_like(i, -1), i)
    z = x / c["temperature"]
    m = z.amax(1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    lse = m[:, 0] + torch.log(torch.exp(z - m).sum(1))
    return {"idx": i, "val": v.to(s["x"].dtype), "lse": lse}


def _plain_distill(s):
    c = s["case"]
    wide = torch.float64 if c["dtype"] == "f64" else torch.float32
    tau = c["temperature"]
    z = s["x"].to(wide) / tau
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(1, keepdim=True)
    p = e / total
    logp = (z - m) - torch.log(total)
    used = s["t_idx"] >= 0
    at = s["t_idx"].clamp(min=0).long()
    tz = torch.where(used, s["t_val"].to(wide) / tau, torch.full((), -math.inf, device=z.device, dtype=wide))
    logp_k = torch.gather(logp, 1, at)
    inside = torch.zeros_like(z).scatter_add_(1, at, used.to(wide))
    if s["t_lse"] is None:
        tm = tz.amax(1, keepdim=True)
        tm = torch.where(tm == -math.inf, torch.zeros_like(tm), tm)
        te = torch.exp(tz - tm)
        logq = (tz - tm) - torch.log(te.sum(1, keepdim=True))
    else:
        logq = tz - s["t_lse"].to(wide)[:, None]
    q = torch.where(used, torch.exp(logq), torch.zeros_like(logq))
    terms = torch.where(used, q * (logq - logp_k), torch.zeros_like(q))
    loss = terms.sum(1)
    full = torch.zeros_like(z).scatter_add_(1, at, q)
    if s["t_lse"] is None:
        grad = p - full
    else:
        qr = (1.0 - q.sum(1)).clamp(min=0)
        pr = (p * (1.0 - inside)).sum(1)
        some = (pr > 0) & (qr > 0)
        qr = torch.where(some, qr, torch.zeros_like(qr))
        one = torch.ones_like(qr)
        loss = loss + qr * (torch.log(torch.where(some, qr, one)) - torch.log(torch.where(some, pr, one)))
        mass = (q.sum(1) + qr)[:, None]
        share = (qr / torch.where(some, pr, one))[:, None]
        grad = mass * p - full - (1.0 - inside) * p * share
    any_used = used.any(1)
    w = any_used.to(wide) if s["w"] is None else any_used.to(wide) * s["w"].to(wide)
    row_loss = torch.where(w != 0, tau * tau * loss, torch.zeros_like(loss))
    scale = 1.0 / c["nrow"]
    grad = torch.where((w != 0)[:, None], (scale * tau) * w[:, None] * grad, torch.zeros_like(grad))
    return {"grad": grad.to(s["x"].dtype), "row_loss": row_loss, "loss": (scale * (w * row_loss).sum()).reshape(1)}


def _plain_sample(s):
    c = s["case"]
    x = s["x"].double()  # in 64 bits: a choice next to a border has to fall on its side
    nrow, ncol = x.shape
    v, i = torch.sort(x, dim=1, descending=True, stable=True)
    if s["rules"] is None:
        tau = torch.full((nrow, 1), c["temperature"], device=x.device, dtype=x.dtype)
        top_k = torch.full((nrow, 1), float(c["top_k"]), device=x.device, dtype=x.dtype)
        top_p = torch.full((nrow, 1), c["top_p"], device=x.device, dtype=x.dtype)
        min_p = torch.full((nrow, 1), c["min_p"], device=x.device, dtype=x.dtype)
    else:
        tau, top_k, top_p, min_p = (s["rules"][:, j:j + 1] for j in range(4))
    z = (v - v[:, :1]) / tau
    e = torch.exp(z)
    place = torch.arange(ncol, device=x.device)[None, :]
    e = torch.where((top_k < 1) | (place < top_k), e, torch.zeros_like(e))
    run_ = torch.cumsum(e, 1)
    total = run_[:, -1:]
    # the shortest prefix whose mass reaches top_p of the total: all whose mass before them does not
    keep = ((run_ - e) < top_p * total) | (top_p >= 1)
    keep &= e >= min_p
    keep[:, 0] = True
    e = torch.where(keep, e, torch.zeros_like(e))
    run_ = torch.cumsum(e, 1)
    total = run_[:, -1:]
    at = (run_ <= s["u"][:, None] * total).sum(1, keepdim=True).clamp(max=ncol - 1)
    idx = torch.gather(i, 1, at)[:, 0].to(torch.int32)
    logp = torch.gather(z, 1, at)[:, 0] - torch.log(total[:, 0])
    none = v[:, 0] == -math.inf
    idx = torch.where(none, torch.full_like(idx, -1), idx)
    logp = torch.where(none, torch.full_like(logp, -math.inf), logp)
    return {"idx": idx, "logp": logp.to(s["logp"].dtype)}


# ------------------------------------------------------------------ the framework's calls

_sims = {}


def _sim():
    """The runtime handle that a program keeps, on torch's current stream."""
    if 0 not in _sims:
        from heliox_b200.runtime import Sim

        _sims[0] = Sim(0)
        _sims[0].set_stream(torch.cuda.current_stream().cuda_stream)
    return _sims[0]


def _own_top(s):
    c = s["case"]
    _sim().top_logits_dev(s["x"].data_ptr(), c["nrow"], c["ncol"], c["k"], s["idx"].data_ptr(), s["val"].data_ptr(),
                          lse_ptr=s["lse"].data_ptr(), temperature=c["temperature"], dtype=c["dtype"])
    return {"idx": s["idx"], "val": s["val"], "lse": s["lse"]}


def _own_distill(s):
    c = s["case"]
    _sim().distill_loss_grad_dev(
        s["x"].data_ptr(), c["nrow"], c["ncol"], c["k"], s["t_idx"].data_ptr(), s["t_val"].data_ptr(),
        s["grad"].data_ptr(), s["row_loss"].data_ptr(), s["loss"].data_ptr(),
        t_lse_ptr=0 if s["t_lse"] is None else s["t_lse"].data_ptr(), temperature=c["temperature"],
        scale=1.0 / c["nrow"], row_weight_ptr=0 if s["w"] is None else s["w"].data_ptr(),
        dtype=c["dtype"], t_dtype=c["t_dtype"])
    return {"grad": s["grad"], "row_loss": s["row_loss"], "loss": s["loss"]}


def _own_sample(s):
    c = s["case"]
    _sim().sample_dev(s["x"].data_ptr(), c["nrow"], c["ncol"], s["u"].data_ptr(), s["idx"].data_ptr(),
                      logp_ptr=s["logp"].data_ptr(), temperature=c["temperature"], top_k=c["top_k"], top_p=c["top_p"],
                      min_p=c["min_p"], rules_ptr=0 if s["rules"] is None else s["rules"].data_ptr(), dtype=c["dtype"])
    return {"idx": s["idx"], "logp": s["logp"]}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"top": _own_top, "distill": _own_distill, "sample": _own_sample}[op](state)
    return {"top": _plain_top, "distill": _plain_distill, "sample": _plain_sample}[op](state)


def work(case):
    n, b = case["nrow"] * case["ncol"], BYTES[case["dtype"]]
    stat = 8 if case["dtype"] == "f64" else 4
    if case["op"] == "top":  # each readout read once; compared, scaled, exponentiated, summed
        return {"bytes": n * b + case["nrow"] * (case["k"] * (4 + b) + stat), "flops": 4 * n}
    if case["op"] == "sample":
        return {"bytes": n * b + case["nrow"] * (8 + 4 + stat + (32 if case["rules"] else 0)), "flops": 4 * n}
    rec = case["k"] * (4 + BYTES[case["t_dtype"]]) + (8 if case["tail"] else 0) + (8 if case["masked"] else 0)
    return {"bytes": 2 * n * b + case["nrow"] * (rec + stat), "flops": 7 * n}


# ------------------------------------------------------------------ from the definitions, in 64 bits

def _exact_distill(s):
    """The loss written as a Kullback-Leibler divergence over the slots and the rest, its gradient by automatic differentiation."""
    c = s["case"]
    tau = c["temperature"]
    x = s["x"].double().requires_grad_(True)
    ls = torch.log_softmax(x / tau, 1)
    used = s["t_idx"] >= 0
    at = torch.where(used, s["t_idx"], torch.zeros_like(s["t_idx"])).long()
    t = s["t_val"].double() / tau
    lp = torch.gather(ls, 1, at)
    if s["t_lse"] is None:
        lq = torch.log_softmax(torch.where(used, t, torch.full_like(t, -1e300)), 1)
    else:
        lq = t - s["t_lse"].double()[:, None]
    q = torch.exp(lq) * used
    kl = torch.where(used, q * (lq - lp), 0.0).sum(1)
    if s["t_lse"] is not None:
        hole = torch.zeros(ls.shape, dtype=torch.bool, device=ls.device).scatter_(1, at[:, :1], used[:, :1])
        hole.scatter_(1, torch.where(used, at, at.gather(1, used.int().argmax(1, keepdim=True))), True)
        rest = torch.logsumexp(ls.masked_fill(hole, -math.inf), 1)
        q_rest = 1.0 - q.sum(1)
        ok = (q_rest > 0) & (rest > -math.inf)
        kl = kl + torch.where(ok, torch.xlogy(q_rest.clamp(min=0), q_rest.clamp(min=0)) - q_rest * torch.where(ok, rest, 0.0), 0.0)
    live = used.any(1)
    w = live.double() if s["w"] is None else live * s["w"]
    row = torch.where(w != 0, tau * tau * kl, 0.0)
    loss = (w * row).sum() / c["nrow"]
    loss.backward()
    return {"grad": x.grad, "row_loss": row.detach(), "loss": loss.detach().reshape(1)}


def _exact_sample(s):
    """By a threshold on each row: the set that is kept is {x above the last one kept}, with ties by position; the choice is left to whole-number comparison."""
    c = s["case"]
    x = s["x"].double()
    nrow, ncol = x.shape
    rules = s["rules"]
    if rules is None:
        rules = torch.tensor([[c["temperature"], float(c["top_k"]), c["top_p"], c["min_p"]]], dtype=torch.float64, device=x.device).expand(nrow, 4)
    tau, top_k, top_p, min_p = (rules[:, j] for j in range(4))
    prob = torch.softmax(x / tau[:, None], 1)
    order = torch.argsort(-x, dim=1, stable=True)
    prob = prob.gather(1, order)
    length = torch.where(top_k >= 1, top_k.clamp(max=ncol), torch.full_like(top_k, ncol)).long()
    rank = torch.arange(1, ncol + 1, device=x.device)
    prob = prob * (rank[None] <= length[:, None])
    prob = prob / prob.sum(1, keepdim=True)
    reach = (prob.cumsum(1) < top_p[:, None]).sum(1) + 1
    length = torch.where(top_p < 1, torch.minimum(length, reach), length)
    length = torch.minimum(length, (prob >= min_p[:, None] * prob[:, :1]).sum(1)).clamp(min=1)
    prob = prob * (rank[None] <= length[:, None])
    prob = prob / prob.sum(1, keepdim=True)
    at = torch.searchsorted(prob.cumsum(1), s["u"][:, None], right=True).clamp(max=ncol - 1)
    at = torch.minimum(at, length[:, None] - 1)
    picked = order.gather(1, at)
    z = (x.gather(1, picked) - x.gather(1, order[:, :1]))[:, 0] / tau
    kept = (torch.exp((x.gather(1, order) - x.gather(1, order[:, :1])) / tau[:, None]) * (rank[None] <= length[:, None])).sum(1)
    empty = x.amax(1) == -math.inf
    return {"idx": None, "logp": torch.where(empty, torch.full_like(z, -math.inf), z - torch.log(kept))}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "top":
        x = s["x"].double()
        return {"idx": None, "val": torch.topk(x, case["k"], dim=1).values, "lse": torch.logsumexp(x / case["temperature"], 1)}
    return _exact_distill(s) if case["op"] == "distill" else _exact_sample(s)

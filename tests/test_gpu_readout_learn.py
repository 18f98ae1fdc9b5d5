"""GPU: the readout-row operators together, as training uses them: a teacher's
record, the distillation loss of a student network, the adjoint, Adam, choices."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

from heliox_b200 import synth  # noqa: E402
from test_gpu_readout import plain_distill, plain_sample, plain_top, wide  # noqa: E402

T, TEMP, K = 400, 3.0, 4
KEYS = ("hh.gnabar", "hh.gkbar", "pas.g")


def student_and_teacher():
    g = synth.random_tree_batch(7, seed0=31, nmin=60, nmax=90)
    return g, synth.perturb_conductances(g, 0.2, seed=4)


def plain_loss_and_grad(trace, rec, w):
    loss, g = 0.0, np.zeros_like(trace)
    for t in range(T):
        L, _, G, _ = plain_distill(trace[t + 1], wide(rec.idx[t]).astype(int), wide(rec.val[t]),
                                   None if rec.lse is None else float(rec.lse[t]), TEMP, w[t], 1.0 / T, "f64")
        loss += w[t] * L / T
        g[t + 1] = G
    return loss, g


@pytest.mark.parametrize("rest", [True, False])
def test_teacher_record_loss_and_adjoint(rest):
    from heliox_b200.learn import AdjointRuntime, record_teacher, train_distill
    from oracle import oracle as O

    g, gt = student_and_teacher()
    rt = AdjointRuntime(gt)
    rec = record_teacher(rt, T, K, TEMP, rest=rest)
    trace = rt.sim.forward_capture(T)
    for t in range(0, T, 7):
        i, v, l = plain_top(trace[t + 1], K, TEMP)
        assert np.array_equal(wide(rec.idx[t]), i) and np.array_equal(wide(rec.val[t]), v)
        assert not rest or abs(float(rec.lse[t]) - l) <= 2.0**-48 * (abs(l) + 50)
    assert (rec.lse is None) == (not rest) and rec.total_steps == T and rec.k == K
    rt.close()

    st = AdjointRuntime(g)
    w = np.ones(T)
    w[:40] = 0.0  # before the stimulus
    ref_trace, _ = O.forward(g, T)
    loss, dl = plain_loss_and_grad(ref_trace, rec, w)
    _, ref = O.adjoint(g, T, dl)
    h = [st.handle("hh", "gnabar", i) for i in range(0, g.hh.n, 5)]
    w0 = st.sim.get_variables(h)
    seen = []
    hist = train_distill(st, h, rec, epochs=1, lr=1e-3, row_weight=w, on_epoch=lambda e, x: seen.append(x))
    assert seen == hist and abs(hist[0] - loss) <= 1e-9 * abs(loss)  # the traces agree within 1e-9
    # the step that Adam takes first: lr * grad / (|grad| + eps)
    gr = ref["hh.gnabar"][::5]
    np.testing.assert_allclose(st.sim.get_variables(h), w0 - 1e-3 * gr / (np.abs(gr) + 1e-8), rtol=0, atol=1e-7 * 1e-3)
    st.close()

    # the gradient itself, for every kind
    st = AdjointRuntime(g)
    tr = torch.zeros((T + 1, rec.ncol), dtype=torch.float64, device="cuda")
    dLdv = torch.zeros_like(tr)
    rl, lo = torch.empty(T, dtype=torch.float64, device="cuda"), torch.empty(1, dtype=torch.float64, device="cuda")
    wt = torch.from_numpy(w).cuda()
    torch.cuda.synchronize()
    s = st.sim
    s.forward_capture_dev(T, tr.data_ptr())
    s.distill_loss_grad_dev(tr[1:].data_ptr(), T, rec.ncol, K, rec.idx.data_ptr(), rec.val.data_ptr(), dLdv[1:].data_ptr(),
                            rl.data_ptr(), lo.data_ptr(), t_lse_ptr=rec.lse.data_ptr() if rest else 0, temperature=TEMP,
                            row_weight_ptr=wt.data_ptr())
    s.synchronize()
    grads = s.backward(wide(dLdv), keys=KEYS)
    for key in KEYS:
        assert np.abs(grads[key] - ref[key]).max() <= 1e-7 * np.abs(ref[key]).max(), key
    st.close()


def test_distill_gradient_of_a_conductance_by_differences():
    """Central differences through simulation and loss: truncation falls with
    h^2, the loss's rounding (2^-44 of it through 400 steps) with 1 / h; two
    steps a factor of four apart bound the truncation by their distance."""
    from heliox_b200.learn import AdjointRuntime, record_teacher

    g, gt = student_and_teacher()
    rt = AdjointRuntime(gt)
    rec = record_teacher(rt, T, K, TEMP)
    rt.close()
    st = AdjointRuntime(g)
    w = np.ones(T)
    trace = st.sim.forward_capture(T)
    loss, dl = plain_loss_and_grad(trace, rec, w)
    grad = st.sim.backward(dl, keys=("hh.gnabar",))["hh.gnabar"]
    for i in (0, int(np.abs(grad).argmax())):
        h = st.handle("hh", "gnabar", i)
        x0 = st.sim.get_variables([h])[0]
        d = []
        for rel in (4e-5, 1e-5):
            side = []
            for sgn in (1, -1):
                st.sim.set_variables([h], [x0 * (1 + sgn * rel)])
                side.append(plain_loss_and_grad(st.sim.simulate(T), rec, w)[0])
            d.append((side[0] - side[1]) / (2 * x0 * rel))
        st.sim.set_variables([h], [x0])
        assert abs(d[1] - grad[i]) <= abs(d[1] - d[0]) + 2.0**-40 * loss / (x0 * 1e-5) + 1e-6 * abs(grad[i]), (i, d, grad[i])
    st.close()


def test_choices_of_a_network():
    from heliox_b200.learn import AdjointRuntime, sample_choices

    g, _ = student_and_teacher()
    rt = AdjointRuntime(g)
    rng = np.random.default_rng(0)
    u = rng.random(100)
    idx, logp = sample_choices(rt, T, u, temperature=TEMP, top_k=5, top_p=0.95, min_p=0.01)
    trace = rt.sim.forward_capture(T)[T + 1 - 100:]
    for r in range(100):
        i, l, may = plain_sample(trace[r], TEMP, 5, 0.95, 0.01, u[r])
        assert idx[r] in may and (idx[r] != i or abs(logp[r] - l) <= 1e-12)
    one, _ = sample_choices(rt, T, [0.5], temperature=0.0)
    assert one[0] == trace[-1].argmax()
    with pytest.raises(ValueError, match="at most"):
        sample_choices(rt, 3, np.zeros(4))
    rt.close()


def test_train_distill_refuses_other_shapes():
    from heliox_b200.learn import AdjointRuntime, record_teacher, train_distill

    g, _ = student_and_teacher()
    rt = AdjointRuntime(g)
    rec = record_teacher(rt, 20, 2, TEMP, probes=[0, 1, 2])
    h = [rt.handle("hh", "gnabar", 0)]
    with pytest.raises(ValueError, match="probes"):
        train_distill(rt, h, rec, 1)
    with pytest.raises(ValueError, match="row_weight"):
        train_distill(rt, h, rec, 1, probes=[0, 1, 2], row_weight=np.ones(3))
    hist = train_distill(rt, h, rec, 3, probes=[0, 1, 2])
    assert len(hist) == 3 and np.isfinite(hist).all()
    rt.close()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_narrow_teachers_record_trains(dtype):
    from heliox_b200.learn import AdjointRuntime, TeacherRecord, record_teacher, train_distill

    g, gt = student_and_teacher()
    rt = AdjointRuntime(gt)
    rec = record_teacher(rt, T, K, TEMP)
    rt.close()
    val = rec.val.to(getattr(torch, dtype))
    narrow = TeacherRecord(rec.idx, val, torch.zeros((T, 2), device="cuda", dtype=torch.float32).add_(rec.lse.float()[:, None])[:, 0], rec.ncol, TEMP)
    st = AdjointRuntime(g)
    trace = st.sim.forward_capture(T)
    loss, _ = plain_loss_and_grad(trace, narrow, np.ones(T))
    hist = train_distill(st, [st.handle("hh", "gnabar", 0)], narrow, 1)
    assert abs(hist[0] - loss) <= 1e-9 * abs(loss)
    st.close()

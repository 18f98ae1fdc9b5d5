"""CPU: the host side of recording a teacher, distilling it and choosing, on a
runtime that only notes what is asked of it."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from heliox_b200 import learn  # noqa: E402


class Sim:
    def __init__(self, refuse=None):
        self.device, self.refuse, self.calls, self.kw, self.sharded = 0, refuse, [], {}, False

    def __getattr__(self, name):
        def call(*args, **kw):
            self.calls.append(name)
            self.kw[name] = (args, kw)
            if name == self.refuse:
                raise RuntimeError(name)
            return 0

        return call


class Runtime:
    def __init__(self, refuse=None):
        self.sim = Sim(refuse)


@pytest.fixture(autouse=True)
def on_the_host(monkeypatch):
    monkeypatch.setattr(learn, "_device_trace", lambda runtime, T, n: torch.zeros((T + 1, n), dtype=torch.float64))
    monkeypatch.setattr(torch.cuda, "current_stream", lambda dev=None: Sim())


def a_record(T=5, k=2, n=3, rest=True):
    return learn.TeacherRecord(torch.zeros((T, k), dtype=torch.int32), torch.zeros((T, k), dtype=torch.float64),
                               torch.zeros(T, dtype=torch.float64) if rest else None, n, 2.0)


RUNS = {
    "record_teacher": lambda rt: learn.record_teacher(rt, 5, 2, probes=[0, 1, 2]),
    "train_distill": lambda rt: learn.train_distill(rt, [0], a_record(), 2, probes=[0, 1, 2]),
    "sample_choices": lambda rt: learn.sample_choices(rt, 5, np.zeros(3), probes=[0, 1, 2]),
}


@pytest.mark.parametrize("run,refuse", [("record_teacher", "top_logits_dev"), ("record_teacher", "forward_capture_dev"),
                                        ("train_distill", "distill_loss_grad_dev"), ("train_distill", "backward_dev"),
                                        ("sample_choices", "sample_dev")])
def test_a_refused_call_leaves_no_work_behind(run, refuse):
    # the forward that was started writes to a torch buffer, which the exception gives back
    rt = Runtime(refuse)
    with pytest.raises(RuntimeError, match=refuse):
        RUNS[run](rt)
    assert rt.sim.calls[-2:] == [refuse, "synchronize"]


@pytest.mark.parametrize("run", list(RUNS))
def test_work_is_done_at_the_end(run):
    rt = Runtime()
    RUNS[run](rt)
    assert rt.sim.calls[-1] == "synchronize"


I32, F64, F32, F16, BF16 = torch.int32, torch.float64, torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("change,error,word", [
    (dict(idx=torch.zeros((5, 2), dtype=torch.int64)), TypeError, "int32"),
    (dict(val=torch.zeros((5, 2), dtype=torch.int32)), TypeError, "float64"),
    (dict(val=torch.zeros((5, 2), dtype=F32)), TypeError, "lse must be torch.float32"),
    (dict(lse=torch.zeros(5, dtype=F32)), TypeError, "lse must be torch.float64"),
    (dict(val=torch.zeros((5, 2), dtype=BF16), lse=torch.zeros(5, dtype=BF16)), TypeError, "lse must be torch.float32"),
    (dict(val=torch.zeros((5, 1), dtype=F64)), ValueError, r"\(T, k\)"),
    (dict(val=torch.zeros((4, 2), dtype=F64)), ValueError, r"\(T, k\)"),
    (dict(idx=torch.zeros(5, dtype=I32), val=torch.zeros(5, dtype=F64)), ValueError, r"\(T, k\)"),
    (dict(lse=torch.zeros(4, dtype=F64)), ValueError, r"\(T,\)"),
    (dict(lse=torch.zeros((5, 1), dtype=F64)), ValueError, r"\(T,\)"),
    (dict(lse=torch.zeros(5, dtype=F64, device="meta")), ValueError, "is on meta"),
])
def test_records_that_the_library_would_misread(change, error, word):
    rec = a_record()
    for name, x in change.items():
        setattr(rec, name, x)
    rt = Runtime()
    with pytest.raises(error, match=word):
        learn.train_distill(rt, [0], rec, 1, probes=[0, 1, 2])
    assert "distill_loss_grad_dev" not in rt.sim.calls


@pytest.mark.parametrize("dtype,name", [(F64, "f64"), (F32, "f32"), (F16, "f16"), (BF16, "bf16")])
def test_records_of_narrow_teachers_and_strided_ones(dtype, name):
    rec = learn.TeacherRecord(torch.arange(10, dtype=I32).reshape(2, 5).T, torch.arange(20, dtype=dtype).reshape(5, 4)[:, ::2],
                              torch.zeros((5, 2), dtype=F64 if dtype == F64 else F32)[:, 0], 3, 2.0)
    idx, val, lse, got = learn._record_arrays(rec, torch.device("cpu"))
    assert got == name and torch.equal(idx, rec.idx) and torch.equal(val, rec.val) and torch.equal(lse, rec.lse)
    assert idx.is_contiguous() and val.is_contiguous() and lse.is_contiguous()
    rt = Runtime()
    learn.train_distill(rt, [0], rec, 1, probes=[0, 1, 2])
    args, kw = rt.sim.kw["distill_loss_grad_dev"]
    assert kw["t_dtype"] == name and args[3] == 2 and kw["t_lse_ptr"]


@pytest.mark.parametrize("run", list(RUNS))
def test_a_sharded_network_is_refused(run):
    rt = Runtime()
    rt.sim.sharded = True
    with pytest.raises(ValueError, match="sharded network"):
        RUNS[run](rt)
    assert rt.sim.calls == []


def test_what_counts_as_sharded():
    from heliox_b200 import _lib, runtime, shard, synth

    s = runtime.Sim.__new__(runtime.Sim)
    s.group = None
    assert not s.sharded
    g = synth.spiking_network(6)
    s.group, s._bound = g, _lib.BoundGroup(g)
    assert not s.sharded
    part, base, nsrc = shard.shard(g, 2, 1)
    s.group, s._bound = part, _lib.BoundGroup(part, gid_base=base, nsrc_cells=nsrc)
    assert s.sharded
    whole, base, nsrc = shard.shard(g, 1, 0)
    s.group, s._bound = whole, _lib.BoundGroup(whole, gid_base=base, nsrc_cells=nsrc)
    assert not s.sharded

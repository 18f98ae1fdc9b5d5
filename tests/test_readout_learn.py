"""CPU: the host side of recording a teacher, distilling it and choosing, on a
runtime that only notes what is asked of it."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

from heliox_b200 import learn  # noqa: E402


class Sim:
    def __init__(self, refuse=None):
        self.device, self.refuse, self.calls, self.kw = 0, refuse, [], {}

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

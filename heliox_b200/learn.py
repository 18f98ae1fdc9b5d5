"""``heliox_learn``-compatible surface for the exact adjoint.

The reference's learning package defines a gradient-method plugin slot
(``GradientMethod``: ``spec``, ``capture(runtime, state)``,
``backward(runtime, captured, dL_dprobe)``, python_lib/heliox_learn/method.py:
15-32), column mappings of runtime handles (``MappedSignal``, signals.py:9-37)
and the result type ``ReplayGrads(dw_out_n, dx_lr_it)`` (signals.py:94-99).
``AdjointMethod`` plugs the exact discrete adjoint into that slot: ``capture``
runs the forward with tape, ``backward`` runs the reverse sweep and reduces the
per-instance gradients into the N columns of a ``MappedSignal`` on the device
(the reference's batch_scatter_add, src/runtime_api/core/kernels/
batch_scatter_add.cu:4-27).  ``train_adam`` is the loop the reference drives
through ``Sim.optimizer_*`` (SimWrapper.cpp:284-451), run on the device.
"""
from __future__ import annotations

from contextlib import contextmanager
from dataclasses import dataclass, field
from typing import Any, Callable, Dict, List, Optional, Protocol, Sequence, Tuple, runtime_checkable

import numpy as np

from .model import CellGroup
from .runtime import Sim


try:
    # The reference's own plugin types, when its package is installed beside
    # this one: AdjointMethod then satisfies heliox_learn.GradientMethod,
    # accepts heliox_learn.MappedSignal and returns heliox_learn.ReplayGrads.
    from heliox_learn.method import GradientMethod, MethodSpec  # type: ignore
    from heliox_learn.signals import MappedSignal, ReplayGrads  # type: ignore

    REFERENCE_TYPES = True
except ImportError:
    # The same types restated (field names, validation and messages of
    # python_lib/heliox_learn/method.py:7-32 and signals.py:9-37, 94-99) for
    # hosts without the reference package.
    REFERENCE_TYPES = False

    @dataclass(frozen=True)
    class MethodSpec:  # type: ignore[no-redef]
        name: str
        precise: bool = True

    @runtime_checkable
    class GradientMethod(Protocol):  # type: ignore[no-redef]
        @property
        def spec(self) -> MethodSpec: ...

        def capture(self, runtime: Any, *, state: Any) -> Any: ...

        def backward(self, runtime: Any, *, captured: Any, dL_dprobe: Any) -> Any: ...

    @dataclass(frozen=True)
    class MappedSignal:  # type: ignore[no-redef]
        """Handles gathered and scatter-added into N columns: out[dest[j]] += scale[j] * x[handles[j]]."""

        name: str
        handles: Sequence[int]
        dest: np.ndarray  # int32 (len(handles),)
        scale: np.ndarray  # float32 (len(handles),)

        def __post_init__(self) -> None:
            if self.dest.ndim != 1 or self.scale.ndim != 1:
                raise ValueError(f"MappedSignal({self.name}): dest/scale must be 1D arrays")
            if int(self.dest.shape[0]) != len(self.handles) or int(self.scale.shape[0]) != len(self.handles):
                raise ValueError(f"MappedSignal({self.name}): size mismatch")
            if self.dest.dtype != np.int32:
                raise TypeError(f"MappedSignal({self.name}): dest must be int32 (got {self.dest.dtype})")
            if self.scale.dtype != np.float32:
                raise TypeError(f"MappedSignal({self.name}): scale must be float32 (got {self.scale.dtype})")

    @dataclass(frozen=True)
    class ReplayGrads:  # type: ignore[no-redef]
        dw_out_n: np.ndarray  # float32 (N,)
        dx_lr_it: Optional[np.ndarray] = None


def n_columns(p: MappedSignal) -> int:
    """Columns N of a mapping: 1 + the largest destination column."""
    return int(p.dest.max()) + 1 if p.dest.size else 0


@dataclass(frozen=True)
class AdjointCaptureSpec:
    """Forward capture: voltages at probe nodes over ``total_steps`` steps."""

    probe_nodes: Sequence[int]
    total_steps: int
    v_init: Optional[float] = None


@dataclass
class CapturedTrace:
    output_vs_tn: np.ndarray  # float64 (total_steps+1, n_output)

    @property
    def total_steps(self) -> int:
        return int(self.output_vs_tn.shape[0]) - 1

    @property
    def n_output(self) -> int:
        return int(self.output_vs_tn.shape[1])


class AdjointRuntime:
    """A loaded cell group on one GPU (the counterpart of heliox_learn.Runtime)."""

    def __init__(self, group: CellGroup, device: int = 0, **sim_kwargs):
        self.group = group
        self.sim = Sim(device, **sim_kwargs)
        self.sim.load_group(group)

    @property
    def loaded(self) -> bool:
        return True

    @property
    def dt_ms(self) -> float:
        return float(self.group.dt)

    @property
    def v_init(self) -> float:
        return float(self.group.v_init)

    def handle(self, mech: str, var: str, idx: int) -> int:
        return self.sim.get_variable_handle(mech, var, idx)

    def close(self) -> None:
        self.sim.close()


@dataclass
class AdjointState:
    spec: AdjointCaptureSpec
    params: MappedSignal


class AdjointMethod:
    """Exact discrete adjoint in the GradientMethod slot."""

    @property
    def spec(self) -> MethodSpec:
        return MethodSpec("adjoint", precise=True)

    def capture(self, runtime: AdjointRuntime, *, state: AdjointState) -> CapturedTrace:
        sp = state.spec
        tr = runtime.sim.forward_capture(int(sp.total_steps), v_init=sp.v_init,
                                         probes=np.asarray(sp.probe_nodes, dtype=np.int32))
        return CapturedTrace(tr)

    def backward(self, runtime: AdjointRuntime, *, captured: CapturedTrace, dL_dprobe: np.ndarray,
                 state: Optional[AdjointState] = None) -> ReplayGrads:
        if state is None:
            raise ValueError("AdjointMethod.backward needs the state with the parameter mapping")
        runtime.sim.backward(np.asarray(dL_dprobe, dtype=np.float64), keys=())
        p = state.params
        dw = runtime.sim.reduce_grads_f32(list(p.handles), p.dest, p.scale, n_columns(p))
        return ReplayGrads(dw_out_n=dw, dx_lr_it=None)


def mse_objective(trace: np.ndarray, target: np.ndarray) -> Tuple[float, np.ndarray]:
    """Soma-voltage MSE over steps 1..T and its gradient dL/dtrace (row 0 is the initial state)."""
    err = trace[1:] - target[1:]
    n = err.size
    loss = float(np.sum(err * err) / n)
    g = np.zeros_like(trace)
    g[1:] = (2.0 / n) * err
    return loss, g


def train_adam(runtime: AdjointRuntime, handles: Sequence[int], target: np.ndarray, epochs: int,
               lr: float = 1e-3, probes: Optional[Sequence[int]] = None, total_steps: Optional[int] = None,
               allreduce: Optional[Callable[[int, int, int], None]] = None,
               on_epoch: Optional[Callable[[int, float], None]] = None) -> List[float]:
    """Fit the parameters behind ``handles`` to ``target`` with the device Adam.

    Each epoch: forward capture, MSE against ``target`` on the host, reverse
    sweep, gradients of the bound parameters copied into the optimizer's slots
    on the device, one Adam step.  With data-parallel replicas (one trial or
    teacher per rank) ``allreduce`` is the optimizer's all-reduce hook
    (``shard.allreduce_sum()``): each step first sums the slot gradients over
    the ranks on the library's stream.  Returns the loss history.
    """
    sim = runtime.sim
    probes = runtime.group.soma_nodes() if probes is None else np.asarray(probes, dtype=np.int32)
    T = int(total_steps if total_steps is not None else target.shape[0] - 1)
    opt = sim.create_optimizer("adam")
    sim.optimizer_add_external_grads(opt, list(handles), impedance=1.0)
    if allreduce is not None:
        sim.optimizer_set_allreduce(opt, allreduce)
    hist = []
    for ep in range(int(epochs)):
        tr = sim.forward_capture(T, probes=probes)
        loss, g = mse_objective(tr, target)
        sim.backward(g, keys=())
        sim.optimizer_grads_from_backward(opt)
        sim.optimizer_step_with_inv_record_steps(opt, lr, 1.0)
        hist.append(loss)
        if on_epoch:
            on_epoch(ep, loss)
    sim.synchronize()
    return hist


@dataclass
class TeacherRecord:
    """A teacher's top readouts of the steps 1..T of a trial (device tensors):
    what ``train_distill`` fits a student to.  ``record_teacher`` keeps those of a
    network; those of another model, or labels, may be put together by hand."""

    idx: Any  # int32 (T, k): probe columns in descending order, -1 where unused
    val: Any  # float64, float32, float16 or bfloat16 (T, k): their voltages (or logits)
    lse: Any  # (T,) log-sum-exp of the whole row at ``temperature`` (float64, float32 beside narrower val), or None
    ncol: int
    temperature: float

    @property
    def total_steps(self) -> int:
        return int(self.idx.shape[0])

    @property
    def k(self) -> int:
        return int(self.idx.shape[1])


def _whole_network(sim: Sim, what: str) -> Sim:
    if sim.sharded:
        raise ValueError(f"{what} of a sharded network: the choice is among the probes of one rank's shard, not of the network")
    return sim


def _device_trace(runtime: AdjointRuntime, total_steps: int, ncol: int):
    """A zeroed (T+1, ncol) float64 buffer on the runtime's device, safe to use on the runtime's stream."""
    import torch

    dev = torch.device("cuda", runtime.sim.device)
    buf = torch.zeros((int(total_steps) + 1, int(ncol)), dtype=torch.float64, device=dev)
    torch.cuda.current_stream(dev).synchronize()
    return buf


@contextmanager
def _settled(sim: Sim):
    """Leaves the block, also by an exception, with the context's work done: until
    then it uses torch's buffers, which torch would give to others."""
    try:
        yield
    finally:
        sim.synchronize()


def record_teacher(runtime: AdjointRuntime, total_steps: int, k: int, temperature: float = 1.0, rest: bool = True,
                   probes: Optional[Sequence[int]] = None) -> TeacherRecord:
    """Run a teacher and keep the ``k`` largest readouts of every step.

    The probes are the choices: step t's probabilities are softmax(v[t] /
    temperature) (temperature in mV).  ``rest`` also keeps each row's
    log-sum-exp, so that the loss counts what the k readouts leave out as one
    more class; without it the k are renormalised.  A row is the readouts of one
    ``Sim``: a network that is sharded by cell over ranks is refused, here and
    in ``train_distill`` and ``sample_choices``.  A full float64 trace of
    10,000 probes over 8,000 steps is 640 MB, 64 readouts of each step 6 MB."""
    import torch

    sim = _whole_network(runtime.sim, "the record")
    p = runtime.group.soma_nodes() if probes is None else np.asarray(probes, dtype=np.int32)
    T, n = int(total_steps), int(len(p))
    trace = _device_trace(runtime, T, n)
    idx = torch.empty((T, int(k)), dtype=torch.int32, device=trace.device)
    val = torch.empty((T, int(k)), dtype=torch.float64, device=trace.device)
    lse = torch.empty(T, dtype=torch.float64, device=trace.device) if rest else None
    with _settled(sim):
        sim.forward_capture_dev(T, trace.data_ptr(), probes=p)
        sim.top_logits_dev(trace[1:].data_ptr(), T, n, int(k), idx.data_ptr(), val.data_ptr(),
                           lse_ptr=0 if lse is None else lse.data_ptr(), temperature=temperature)
    return TeacherRecord(idx, val, lse, n, float(temperature))


def _record_arrays(teacher: TeacherRecord, device):
    """(idx, val, lse, type name of val) of a record as the library reads it."""
    import torch

    names = {torch.float64: "f64", torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}
    idx, val, lse = teacher.idx, teacher.val, teacher.lse
    for what, x in (("idx", idx), ("val", val), ("lse", lse)):
        if x is not None and x.device != device:
            raise ValueError(f"the teacher's record is on {x.device} ({what}), the student on {device}")
    if idx.dtype != torch.int32:
        raise TypeError(f"the record's idx must be int32 (got {idx.dtype})")
    if val.dtype not in names:
        raise TypeError(f"the record's val must be float64, float32, float16 or bfloat16 (got {val.dtype})")
    if idx.ndim != 2 or val.shape != idx.shape:
        raise ValueError(f"the record's idx and val must both be (T, k) (got {tuple(idx.shape)} and {tuple(val.shape)})")
    if lse is not None:
        stat = torch.float64 if val.dtype == torch.float64 else torch.float32
        if lse.dtype != stat:
            raise TypeError(f"the record's lse must be {stat} beside {val.dtype} val (got {lse.dtype})")
        if lse.shape != idx.shape[:1]:
            raise ValueError(f"the record's lse must be (T,) (got {tuple(lse.shape)} beside {tuple(idx.shape)})")
        lse = lse.contiguous()
    return idx.contiguous(), val.contiguous(), lse, names[val.dtype]


def train_distill(runtime: AdjointRuntime, handles: Sequence[int], teacher: TeacherRecord, epochs: int,
                  lr: float = 1e-3, probes: Optional[Sequence[int]] = None, row_weight: Optional[np.ndarray] = None,
                  allreduce: Optional[Callable[[int, int, int], None]] = None,
                  on_epoch: Optional[Callable[[int, float], None]] = None) -> List[float]:
    """Fit the parameters behind ``handles`` so that the probes choose as the teacher's do.

    ``train_adam`` with the distillation loss in place of the trace's MSE, the
    mean over the teacher's steps: forward capture, loss and gradient, reverse
    sweep and Adam all stay on the device.  ``row_weight`` (T): the weight of
    each step, 0 leaves one out.  ``allreduce``: of data-parallel replicas, as in
    ``train_adam``.  Returns the loss history."""
    import torch

    sim = _whole_network(runtime.sim, "distillation")
    p = runtime.group.soma_nodes() if probes is None else np.asarray(probes, dtype=np.int32)
    T, n = teacher.total_steps, teacher.ncol
    if len(p) != n:
        raise ValueError(f"the teacher's record has {n} readouts a step, the student {len(p)} probes")
    if row_weight is not None and np.shape(row_weight) != (T,):
        raise ValueError(f"row_weight must have shape ({T},)")
    trace, dLdv = _device_trace(runtime, T, n), _device_trace(runtime, T, n)  # row 0, the initial state, has no loss
    t_idx, t_val, t_lse, t_dtype = _record_arrays(teacher, trace.device)
    row_loss = torch.empty(T, dtype=torch.float64, device=trace.device)
    losses = torch.zeros(max(int(epochs), 1), dtype=torch.float64, device=trace.device)
    w = None if row_weight is None else torch.from_numpy(np.ascontiguousarray(row_weight, dtype=np.float64)).to(trace.device)
    torch.cuda.current_stream(trace.device).synchronize()
    opt = sim.create_optimizer("adam")
    sim.optimizer_add_external_grads(opt, list(handles), impedance=1.0)
    if allreduce is not None:
        sim.optimizer_set_allreduce(opt, allreduce)
    with _settled(sim):
        for ep in range(int(epochs)):
            sim.forward_capture_dev(T, trace.data_ptr(), probes=p)
            sim.distill_loss_grad_dev(trace[1:].data_ptr(), T, n, teacher.k, t_idx.data_ptr(), t_val.data_ptr(),
                                      dLdv[1:].data_ptr(), row_loss.data_ptr(), losses[ep:].data_ptr(),
                                      t_lse_ptr=0 if t_lse is None else t_lse.data_ptr(), t_dtype=t_dtype,
                                      temperature=teacher.temperature, row_weight_ptr=0 if w is None else w.data_ptr())
            sim.backward_dev(dLdv.data_ptr(), {})
            sim.optimizer_grads_from_backward(opt)
            sim.optimizer_step_with_inv_record_steps(opt, lr, 1.0)
            if on_epoch:
                sim.synchronize()
                on_epoch(ep, float(losses[ep]))
    return [float(x) for x in losses[:int(epochs)].cpu()]


def sample_choices(runtime: AdjointRuntime, total_steps: int, u: np.ndarray, temperature: float = 1.0, top_k: int = 0,
                   top_p: float = 1.0, min_p: float = 0.0, probes: Optional[Sequence[int]] = None) -> Tuple[np.ndarray, np.ndarray]:
    """Run the network and draw one choice among its probes at each of the last
    len(u) steps, from the uniform numbers ``u``: (probe columns int32,
    log-probabilities float64)."""
    import torch

    sim = _whole_network(runtime.sim, "choices")
    p = runtime.group.soma_nodes() if probes is None else np.asarray(probes, dtype=np.int32)
    T, n = int(total_steps), int(len(p))
    uu = np.ascontiguousarray(u, dtype=np.float64)
    m = int(uu.shape[0])
    if uu.ndim != 1 or m > T:
        raise ValueError(f"u must be one-dimensional with at most {T} entries")
    trace = _device_trace(runtime, T, n)
    ud = torch.from_numpy(uu).to(trace.device)
    idx = torch.empty(m, dtype=torch.int32, device=trace.device)
    logp = torch.empty(m, dtype=torch.float64, device=trace.device)
    torch.cuda.current_stream(trace.device).synchronize()
    with _settled(sim):
        sim.forward_capture_dev(T, trace.data_ptr(), probes=p)
        sim.sample_dev(trace[T + 1 - m:].data_ptr(), m, n, ud.data_ptr(), idx.data_ptr(), logp_ptr=logp.data_ptr(),
                       temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    return idx.cpu().numpy(), logp.cpu().numpy()

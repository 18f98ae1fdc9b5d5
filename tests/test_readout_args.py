"""CPU: what the readout-row entries refuse, and what they accept."""
import ctypes as C

import pytest

from heliox_b200 import _lib
from heliox_b200.runtime import Sim, _readout

P = 0x7F0000000000  # a well aligned address that nothing here follows


def rows(x=P, dtype=0, nrow=4, ncol=10, ld=10):
    return _lib.Readout(x or None, dtype, nrow, ncol, ld)


def top(r, k=3, t=1.0, idx=P, val=P, lse=P):
    msg = C.create_string_buffer(200)
    rc = _lib.load().hx_top_logits_check(C.byref(r) if r is not None else None, k, t, idx, val, lse, msg, 200)
    return rc, msg.value.decode()


def distill(r, t=1.0, scale=1.0, weight=None, grad=P + (1 << 30), ldg=10, row_loss=P, loss=P, tidx=P, tval=P, tlse=None,
            tdtype=0, k=3, teacher=True):
    te = _lib.Teacher(tidx or None, tval or None, tlse, tdtype, k)
    msg = C.create_string_buffer(200)
    rc = _lib.load().hx_distill_check(C.byref(r), C.byref(te) if teacher else None, t, scale, weight, grad or None, ldg,
                                      row_loss or None, loss or None, msg, 200)
    return rc, msg.value.decode()


def sample(r, rule=(1.0, 0.0, 1.0, 0.0), rules=None, u=P, idx=P, logp=None):
    ru = C.byref(_lib.SampleRule(*rule)) if rule is not None else None
    msg = C.create_string_buffer(200)
    rc = _lib.load().hx_sample_check(C.byref(r), ru, rules, u or None, idx or None, logp, msg, 200)
    return rc, msg.value.decode()


def test_accepted():
    for r in (rows(), rows(nrow=0, x=0), rows(ncol=0, ld=0, x=0), rows(ld=1000), rows(dtype=3, x=P + 2), rows(ncol=1, ld=1),
              rows(ncol=196608, ld=196608), rows(dtype=3, ncol=786432, ld=786432), rows(nrow=1 << 30, ld=1 << 20)):
        assert top(r) == (0, "")
        assert distill(r, ldg=r.ld, grad=0) == (0, "")
        assert sample(r) == (0, "")
    assert top(rows(), k=1024, lse=None)[0] == 0
    assert distill(rows(), tlse=P)[0] == 0
    assert distill(rows(), grad=P)[0] == 0  # in place
    assert distill(rows(ld=40), grad=P + 10 * 8, ldg=40)[0] == 0  # rows between rows
    assert sample(rows(), rule=None, rules=P)[0] == 0
    assert sample(rows(), rule=(0.0, 0.0, 1.0, 0.0))[0] == 0  # greedy
    assert sample(rows(), rule=(1.0, 1e9, 0.0, 1.0))[0] == 0


BAD_ROWS = [(dict(x=0), "null x"), (dict(dtype=4), "dtype"), (dict(dtype=-1), "dtype"), (dict(nrow=-1), "negative"),
            (dict(ncol=-1), "negative"), (dict(ld=9), "ld"), (dict(ncol=196609, ld=196609), "MAX_ROW"),
            (dict(dtype=2, ncol=786433, ld=786433), "MAX_ROW"), (dict(x=P + 4), "aligned"), (dict(dtype=1, x=P + 2), "aligned"),
            (dict(dtype=3, x=P + 1), "aligned"), (dict(nrow=1 << 30, ld=1 << 40), "ld")]


@pytest.mark.parametrize("kw,word", BAD_ROWS)
def test_bad_rows(kw, word):
    for rc, msg in (top(rows(**kw)), distill(rows(**kw), grad=0), sample(rows(**kw))):
        assert rc == -1 and word in msg


NAN, INF = float("nan"), float("inf")


@pytest.mark.parametrize("kw,word", [(dict(k=0), "k must"), (dict(k=1025), "k must"), (dict(t=0.0), "temperature"),
                                     (dict(t=-1.0), "temperature"), (dict(t=NAN), "temperature"), (dict(t=INF), "temperature"),
                                     (dict(t=1e-31), "temperature"), (dict(idx=None), "null"), (dict(val=None), "null"),
                                     (dict(idx=P + 2), "aligned"), (dict(val=P + 4), "aligned"), (dict(lse=P + 4), "aligned")])
def test_top_refuses(kw, word):
    rc, msg = top(rows(), **kw)
    assert rc == -1 and word in msg


@pytest.mark.parametrize("kw,word", [(dict(teacher=False), "null teacher"), (dict(k=0), "k must"), (dict(k=1025), "k must"),
                                     (dict(tdtype=9), "dtype"), (dict(tidx=0), "null"), (dict(tval=0), "null"),
                                     (dict(tval=P + 4), "aligned"), (dict(tlse=P + 4), "aligned"),
                                     (dict(tdtype=1, tlse=P + 2), "aligned"), (dict(t=0.0), "temperature"),
                                     (dict(t=NAN), "temperature"), (dict(scale=NAN), "scale"), (dict(scale=INF), "scale"),
                                     (dict(loss=0), "null"), (dict(row_loss=0), "null"), (dict(weight=P + 4), "aligned"),
                                     (dict(grad=P + 4), "aligned"), (dict(ldg=9), "ld_grad"),
                                     (dict(grad=P, ldg=11), "same ld"), (dict(grad=P + 8), "overlaps"),
                                     (dict(grad=P - 80), "overlaps"), (dict(grad=P + 30 * 8, ldg=10), "overlaps")])
def test_distill_refuses(kw, word):
    rc, msg = distill(rows(), **kw)
    assert rc == -1 and word in msg


def test_distill_refuses_interleaved_overlap():
    assert distill(rows(ld=15), grad=P + 10 * 8, ldg=15)[0] == -1  # its row reaches into the next row
    assert distill(rows(ld=40), grad=P + 10 * 8, ldg=41)[0] == -1


@pytest.mark.parametrize("kw,word", [(dict(rule=None), "null rule"), (dict(u=0), "null"), (dict(idx=0), "null"),
                                     (dict(u=P + 4), "aligned"), (dict(rule=None, rules=P + 4), "aligned"),
                                     (dict(logp=P + 4), "aligned"), (dict(rule=(-1.0, 0, 1, 0)), "temperature"),
                                     (dict(rule=(NAN, 0, 1, 0)), "temperature"), (dict(rule=(1, -1, 1, 0)), "top_k"),
                                     (dict(rule=(1, NAN, 1, 0)), "top_k"), (dict(rule=(1, 0, 1.1, 0)), "top_p"),
                                     (dict(rule=(1, 0, -0.1, 0)), "top_p"), (dict(rule=(1, 0, NAN, 0)), "top_p"),
                                     (dict(rule=(1, 0, 1, 1.1)), "min_p"), (dict(rule=(1, 0, 1, NAN)), "min_p")])
def test_sample_refuses(kw, word):
    rc, msg = sample(rows(), **kw)
    assert rc == -1 and word in msg


def test_null_context_and_message_bounds():
    L = _lib.load()
    r = rows()
    assert L.hx_top_logits_dev(None, C.byref(r), 1, 1.0, P, P, None) == -1
    assert L.hx_sample_dev(None, C.byref(r), None, P, P, P, None) == -1
    te = _lib.Teacher(P, P, None, 0, 1)
    assert L.hx_distill_loss_grad_dev(None, C.byref(r), C.byref(te), 1.0, 1.0, None, None, 0, P, P) == -1
    assert top(None)[1] == "null rows"
    msg = C.create_string_buffer(b"zzzzzzzz", 8)
    assert L.hx_top_logits_check(None, 1, 1.0, None, None, None, msg, 5) == -1
    assert msg.raw[:5] == b"null\0" and msg.raw[5:7] == b"zz"
    assert L.hx_top_logits_check(None, 1, 1.0, None, None, None, None, 0) == -1


def test_python_dtype_names():
    assert _readout(0, 1, 2, "bf16", None).ld == 2
    with pytest.raises(ValueError, match="dtype"):
        _readout(0, 1, 2, "float64", None)
    assert {"top_logits_dev", "distill_loss_grad_dev", "sample_dev"} <= set(dir(Sim))


def test_python_numbers_that_do_not_fit():
    # a descriptor's int would cut 2^32 + 3 rows to 3, and answer for those
    for kw, word in ((dict(nrow=2**32 + 3), "nrow"), (dict(nrow=2**31), "nrow"), (dict(ncol=2**32 + 2), "ncol"), (dict(ld=2**64 + 2), "ld"),
                     (dict(nrow=-(2**32) + 1), "nrow")):
        with pytest.raises(ValueError, match=word):
            _readout(**{**dict(ptr=P, nrow=1, ncol=2, dtype="f64", ld=None), **kw})
    assert _readout(P, 2**31 - 1, 2, "f64", 2**40).ld == 2**40

    class Lib:
        def __getattr__(self, name):
            def called(*args):
                raise AssertionError(name)

            return called

    s = Sim.__new__(Sim)
    s._L, s._ctx = Lib(), None
    with pytest.raises(ValueError, match="^k ="):
        s.top_logits_dev(P, 1, 2, 2**32 + 1, P, P)
    with pytest.raises(ValueError, match="^k ="):
        s.distill_loss_grad_dev(P, 1, 2, 2**32 + 1, P, P, P, P, P)
    with pytest.raises(ValueError, match="ld_grad"):
        s.distill_loss_grad_dev(P, 1, 2, 1, P, P, P, P, P, ld_grad=2**64 + 2)
    with pytest.raises(ValueError, match="nrow"):
        s.sample_dev(P, 2**32 + 1, 2, P, P)


def test_offsets_beyond_any_address():
    # nrow * ld elements whose bytes do not fit 64 bits, in the rows and in the gradient
    for nrow, ld in ((1 << 20, 1 << 40), (1 << 16, 1 << 42), (2, 1 << 59)):
        for rc, msg in (top(rows(nrow=nrow, ld=ld)), distill(rows(nrow=nrow, ld=ld), ldg=ld), sample(rows(nrow=nrow, ld=ld))):
            assert rc == -1 and "ld is out of range" in msg
        rc, msg = distill(rows(nrow=nrow), ldg=ld)
        assert rc == -1 and "ld_grad is out of range" in msg
    assert distill(rows(nrow=1 << 16, ld=1 << 40), ldg=1 << 40, grad=P + 80)[0] == 0

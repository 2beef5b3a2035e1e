"""CPU: the row operators' definitions (oracle/rows.py) against differences and brute force, and the refusals that need no device."""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import rows as orow


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("index", [[1, 4, 0], [2, 2, 5], [-1, 3, 9], [-1, 7, 9]])
def test_distill_gradient_is_the_loss_s_slope(rest, index):
    rng = np.random.default_rng(3)
    s = torch.tensor(rng.normal(size=7))
    values = torch.tensor(rng.normal(size=3))
    lse = 2.0 if rest else None
    _, grad = orow.distill_row(s, values, index, lse, 1.7)
    h = 1e-6
    for j in range(7):
        up, dn = s.clone(), s.clone()
        up[j] += h
        dn[j] -= h
        slope = (orow.distill_row(up, values, index, lse, 1.7)[0] - orow.distill_row(dn, values, index, lse, 1.7)[0]) / (2 * h)
        assert abs(slope - float(grad[j])) < 1e-8      # h^2 times a third derivative of order 1, and 1e-16 / h


def test_distill_is_zero_where_the_student_is_the_teacher():
    x = torch.tensor(np.random.default_rng(0).normal(size=9))
    lse = float(torch.logsumexp(x / 2.0, 0))
    loss, grad = orow.distill_row(x, x[[3, 1, 5]], [3, 1, 5], lse, 2.0)
    assert abs(loss) < 1e-13 and float(grad.abs().max()) < 1e-13


def test_order():
    row = np.array([0.0, -0.0, 3.0, np.nan, -np.inf, 3.0, np.inf, np.nan], np.float32)
    assert orow.order(row).tolist() == [3, 7, 6, 2, 5, 0, 1, 4]


def test_sample_definition_by_hand():
    row = np.log(np.array([0.1, 0.4, 0.2, 0.3]))
    assert orow.sample_row(row, 0.0, 1.0, 0, 1.0, 0.0)[0] == 1
    assert orow.sample_row(row, 0.41, 1.0, 0, 1.0, 0.0)[0] == 3
    assert orow.sample_row(row, 0.95, 1.0, 0, 1.0, 0.0)[0] == 0
    assert orow.sample_row(row, 0.99, 1.0, 2, 1.0, 0.0)[0] == 3
    assert orow.sample_row(row, 0.99, 1.0, 0, 0.65, 0.0)[0] == 3       # 0.4 + 0.3 holds 0.65
    assert orow.sample_row(row, 0.99, 1.0, 0, 1.0, 0.45)[0] == 2       # 0.1 < 0.45 * 0.4
    assert orow.sample_row(row, 0.99, 0.0, 0, 1.0, 0.0)[0] == 1
    tok, logp, _, share = orow.sample_row(row, 0.5, 1.0, 2, 1.0, 0.0)
    assert tok == 1 and math.isclose(logp, math.log(0.4 / 0.7)) and len(share) == 2


def test_ops_refuse_host_tensors():
    from mucon_amd import _lib, ops

    x = torch.zeros(2, 8)
    for call in (lambda: ops.top_logits(x, 2), lambda: ops.sample_logits(x, torch.zeros(2)),
                 lambda: ops.distill_loss(x, torch.zeros(2, 2), torch.zeros(2, 2, dtype=torch.int32)),
                 lambda: ops.distill_loss_and_grad(x, torch.zeros(2, 2), torch.zeros(2, 2, dtype=torch.int32))):
        with pytest.raises(_lib.MuconHipError, match="no CPU fallback"):
            call()


def _cfg(**kw):
    from mucon_amd import _lib

    d = dict(rows=4, row_stride=8, vocab=8, k=3, type=0, teacher_type=0, reduction=2, reserved=0, temperature=1.0)
    d.update(kw)
    return _lib.DistillCfg(**d)


@pytest.mark.parametrize("bad", [dict(rows=0), dict(rows=1 << 31), dict(rows=1 << 22, vocab=65, row_stride=65), dict(rows=1 << 26), dict(row_stride=7), dict(vocab=0), dict(vocab=(1 << 18) + 1, row_stride=1 << 19), dict(k=0),
                                 dict(k=1025), dict(type=3), dict(teacher_type=-1), dict(reduction=3), dict(temperature=0.0), dict(temperature=math.nan),
                                 dict(temperature=math.inf)])
def test_distill_refuses(bad):
    from mucon_amd import _lib

    lib = _lib.load()
    cfg = _cfg(**bad)
    assert lib.mucon_distill_workspace_bytes(ctypes.byref(cfg)) == 0
    assert lib.mucon_distill_fwd(ctypes.byref(cfg), 64, 64, 64, 0, 0, 64, 64, 1 << 30, None) == _lib.E_ARG
    assert lib.mucon_distill_bwd(ctypes.byref(cfg), 64, 64, 64, 0, 0, 64, 64, 64, 1 << 30, None) == _lib.E_ARG
    assert lib.mucon_distill_fwd_bwd(ctypes.byref(cfg), 64, 64, 64, 0, 0, 1.0, 64, 64, 64, 1 << 30, None) == _lib.E_ARG
    assert lib.mucon_last_error().startswith(b"distill")


def test_distill_refuses_null_pointers_and_a_small_workspace():
    from mucon_amd import _lib

    lib = _lib.load()
    cfg = _cfg()
    need = lib.mucon_distill_workspace_bytes(ctypes.byref(cfg))
    assert need > 0
    assert lib.mucon_distill_fwd(ctypes.byref(cfg), 0, 64, 64, 0, 0, 64, 64, need, None) == _lib.E_ARG
    assert lib.mucon_distill_fwd(ctypes.byref(cfg), 64, 64, 64, 0, 0, 64, 64, need - 1, None) == _lib.E_WORKSPACE
    assert lib.mucon_distill_bwd(ctypes.byref(cfg), 64, 64, 64, 0, 0, 0, 64, 64, need, None) == _lib.E_ARG
    assert lib.mucon_distill_fwd_bwd(ctypes.byref(cfg), 64, 64, 64, 0, 0, 1.0, 64, 0, 64, need, None) == _lib.E_ARG


@pytest.mark.parametrize("bad", [dict(type=3), dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 18) + 1), dict(stride=7), dict(k=0), dict(k=9), dict(k=1025, vocab=2000, stride=2000),
                                 dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=math.nan), dict(x=0)])
def test_top_logits_refuses(bad):
    from mucon_amd import _lib

    lib = _lib.load()
    d = dict(type=0, rows=2, vocab=8, stride=8, k=2, temperature=1.0, x=64)
    d.update(bad)
    assert lib.mucon_top_logits(d["type"], d["rows"], d["vocab"], d["stride"], d["k"], d["temperature"], d["x"], 64, 64, 64, 0, 0, None) == _lib.E_ARG


@pytest.mark.parametrize("bad", [dict(temperature=-0.5), dict(temperature=math.nan), dict(temperature=math.inf), dict(top_p=0.0), dict(top_p=math.nan), dict(min_p=-0.1),
                                 dict(min_p=1.5), dict(min_p=math.nan), dict(top_k=-1)])
def test_sample_logits_refuses(bad):
    from mucon_amd import _lib

    lib = _lib.load()
    d = dict(temperature=1.0, top_p=1.0, min_p=0.0, top_k=0)
    d.update(bad)
    p = _lib.SampleParams(**d)
    assert lib.mucon_sample_logits(0, 2, 8, 8, 64, 64, ctypes.byref(p), 64, 64, None) == _lib.E_ARG
    good = _lib.SampleParams(temperature=1.0, top_p=1.0)
    assert lib.mucon_sample_logits(0, 2, 8, 8, 0, 64, ctypes.byref(good), 64, 64, None) == _lib.E_ARG
    assert lib.mucon_sample_logits(0, 2, 8, 4, 64, 64, ctypes.byref(good), 64, 64, None) == _lib.E_ARG
    assert lib.mucon_sample_logits(0, 0, 8, 8, 0, 0, ctypes.byref(good), 0, 0, None) == _lib.OK


def test_few_long_rows_need_their_workspace():
    from mucon_amd import _lib

    lib = _lib.load()
    need = lib.mucon_top_logits_workspace_bytes(0, 2, 100000, 50)
    assert need > 0 and lib.mucon_top_logits_workspace_bytes(0, 4096, 100000, 50) == 0 and lib.mucon_top_logits_workspace_bytes(0, 2, 1000, 50) == 0
    assert lib.mucon_top_logits(0, 2, 100000, 100000, 50, 1.0, 64, 64, 64, 64, 64, need - 1, None) == _lib.E_WORKSPACE
    assert lib.mucon_top_logits(0, 2, 100000, 100000, 50, 1.0, 64, 64, 64, 64, 0, need, None) == _lib.E_WORKSPACE


def test_more_rows_than_a_launch_holds():
    from mucon_amd import _lib

    lib = _lib.load()
    p = _lib.SampleParams(temperature=1.0, top_p=1.0)
    for rows, vocab in ((1 << 22, 65), (1 << 26, 64)):
        assert lib.mucon_top_logits(0, rows, vocab, vocab, 3, 1.0, 64, 64, 64, 64, 0, 0, None) == _lib.E_ARG
        assert lib.mucon_sample_logits(0, rows, vocab, vocab, 64, 64, ctypes.byref(p), 64, 64, None) == _lib.E_ARG
    cfg = _cfg(rows=1 << 20, vocab=1 << 18, row_stride=1 << 18, type=1)       # 1 M rows in 32 pieces each
    need = lib.mucon_distill_workspace_bytes(ctypes.byref(cfg))
    assert lib.mucon_distill_bwd(ctypes.byref(cfg), 64, 64, 64, 0, 0, 64, 64, 64, need, None) == _lib.E_ARG


def test_every_argument_may_be_given_by_name():
    """On host tensors: refused for being there, not for a missing argument."""
    from mucon_amd import _lib, ops

    x, listed = torch.zeros(2, 8), dict(teacher_values=torch.zeros(2, 2), teacher_index=torch.zeros(2, 2, dtype=torch.int32))
    for fn, kw in ((ops.top_logits, dict(logits=x, k=2)), (ops.sample_logits, dict(logits=x, uniform=torch.zeros(2))), (ops.distill_loss, dict(student=x, **listed)),
                   (ops.distill_loss_and_grad, dict(student=x, **listed))):
        with pytest.raises(_lib.MuconHipError, match="no CPU fallback"):
            fn(**kw)
        with pytest.raises(TypeError, match="logits|student"):
            fn(**{name: v for name, v in kw.items() if v is not x})


@pytest.mark.parametrize("temperature", [1e-300, 1e-46, 9e-31, 1.1e30, 1e46, 1e300])
def test_temperatures_whose_inverse_leaves_fp32_are_refused(temperature):
    """log2(e) / T is infinite or 0 in fp32 at the outer ones: 0 times infinity, a row of NaN."""
    from mucon_amd import _lib

    lib = _lib.load()
    assert lib.mucon_top_logits(0, 2, 8, 8, 2, temperature, 64, 64, 64, 64, 0, 0, None) == _lib.E_ARG
    assert b"temperature" in lib.mucon_last_error()
    cfg = _cfg(temperature=temperature)
    assert lib.mucon_distill_workspace_bytes(ctypes.byref(cfg)) == 0 and b"temperature" in lib.mucon_last_error()
    for inside in (1e-30, 1e30):
        assert lib.mucon_distill_workspace_bytes(ctypes.byref(_cfg(temperature=inside))) > 0

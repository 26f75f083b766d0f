"""not-gpu: what the head losses refuse, through ops (values and shapes before devices) and through the C ABI."""
import ctypes

import pytest
import torch

from neuron_interpolation_model_fusion_amd import _lib, ops

H, W, B = torch.zeros(6, 8), torch.zeros(5, 8), torch.zeros(5)
Y = torch.zeros(6, dtype=torch.int64)
V, I = torch.zeros(6, 3), torch.zeros(6, 3, dtype=torch.int32)
Z = torch.zeros(6, 5)


@pytest.mark.parametrize('call, error', [
    (lambda: ops.linear_cross_entropy(H, W, Y), _lib.NifError),  # host tensors
    (lambda: ops.linear_cross_entropy(H, W.bfloat16(), Y), TypeError),
    (lambda: ops.linear_cross_entropy(H.double(), W.double(), Y), TypeError),
    (lambda: ops.linear_cross_entropy(H, W, Y, B.half()), TypeError),
    (lambda: ops.linear_cross_entropy(H, W[:, :7], Y), ValueError),
    (lambda: ops.linear_cross_entropy(H, W[:0], Y), ValueError),
    (lambda: ops.linear_cross_entropy(H, W, Y, B[:4]), ValueError),
    (lambda: ops.linear_cross_entropy(H, W, Y[:5]), ValueError),
    (lambda: ops.linear_cross_entropy(H, W, Y.float()), ValueError),
    (lambda: ops.linear_cross_entropy(H, W, Y.bool()), ValueError),
    (lambda: ops.linear_cross_entropy(H, W, Y, reduction='batchmean'), ValueError),
    (lambda: ops.linear_topk_distillation(H, W, V, I), _lib.NifError),
    (lambda: ops.linear_topk_distillation(H, W, V, I[:, :2]), ValueError),
    (lambda: ops.linear_topk_distillation(H, W, V[:5], I[:5]), ValueError),
    (lambda: ops.linear_topk_distillation(H, W, V[:, :0], I[:, :0]), ValueError),
    (lambda: ops.linear_topk_distillation(H, W, V.int(), I), TypeError),
    (lambda: ops.linear_topk_distillation(H, W, V, I.float()), TypeError),
    (lambda: ops.linear_topk_distillation(H, W, V, I, temperature=0.0), ValueError),
    (lambda: ops.linear_topk_distillation(H, W, V, I, temperature=float('nan')), ValueError),
    (lambda: ops.linear_topk_distillation(H, W, V, I, top_lse=V), ValueError),
    (lambda: ops.topk_distillation(Z, V, I), _lib.NifError),
    (lambda: ops.topk_distillation(Z[:, :0], V, I), ValueError),
    (lambda: ops.topk_distillation(Z, V, I, temperature=-1.0), ValueError),
    (lambda: ops.topk_distillation(Z, torch.zeros(6, 1025), torch.zeros(6, 1025, dtype=torch.int32)), ValueError),
    (lambda: ops.top_logits(Z, 2), _lib.NifError),
    (lambda: ops.top_logits(Z, 6), ValueError),
    (lambda: ops.top_logits(Z, 0), ValueError),
    (lambda: ops.top_logits(Z.int(), 2), TypeError),
])
def test_ops_refuse(call, error):
    with pytest.raises(error):
        call()


def _desc(**kw):
    d = _lib.HeadDesc()
    p = ctypes.c_void_p(4096)  # never read: every call below returns before a launch
    values = dict(hidden=p, ldh=8, weight=p, ldw=8, bias=None, rows=6, features=8, classes=5, dtype=_lib.NIF_F32,
                  reduction=_lib.NIF_REDUCE_MEAN, labels=p, ignore_index=-100, top_indices=None, top_values=None, top_lse=None,
                  top=0, temperature=1.0)
    for key, value in {**values, **kw}.items():
        setattr(d, key, value)
    return ctypes.byref(d)


@pytest.mark.parametrize('change', [
    dict(rows=-1), dict(features=0), dict(classes=0), dict(dtype=_lib.NIF_F64), dict(dtype=9), dict(reduction=3),
    dict(ldh=7), dict(ldw=7), dict(hidden=None), dict(weight=None), dict(labels=None), dict(top=2),
    dict(labels=None, top_indices=ctypes.c_void_p(4096), top_values=ctypes.c_void_p(4096), top=0),
    dict(labels=None, top_indices=ctypes.c_void_p(4096), top_values=None, top=2),
    dict(labels=None, top_indices=ctypes.c_void_p(4096), top_values=ctypes.c_void_p(4096), top=2, temperature=0.0),
    dict(labels=None, top_indices=ctypes.c_void_p(4096), top_values=ctypes.c_void_p(4096), top=2000),
    dict(top_indices=ctypes.c_void_p(4096)), dict(rows=1 << 40),
])
def test_c_abi_refuses_bad_head_problems(change):
    p = ctypes.c_void_p(4096)
    assert _lib.lib.nif_head_forward(_desc(**change), p, p, 1 << 40, p, 1 << 40, None) == -1
    assert _lib.lib.nif_head_backward(_desc(**change), p, p, 1 << 40, p, 8, p, 8, None, p, 1 << 40, None) == -1


def test_c_abi_refuses_small_buffers_and_null_outputs():
    p, lib = ctypes.c_void_p(4096), _lib.lib
    d = _desc()
    state, fwd, bwd = (f(d) for f in (lib.nif_head_state_bytes, lib.nif_head_forward_workspace_bytes,
                                      lib.nif_head_backward_workspace_bytes))
    assert min(state, fwd, bwd) > 0
    assert lib.nif_head_forward(d, None, p, state, p, fwd, None) == -1
    assert lib.nif_head_forward(d, p, p, state - 1, p, fwd, None) == -2
    assert lib.nif_head_forward(d, p, p, state, p, fwd - 1, None) == -2
    assert lib.nif_head_forward(d, p, None, state, p, fwd, None) == -2
    assert lib.nif_head_backward(d, None, p, state, p, 8, p, 8, None, p, bwd, None) == -1
    assert lib.nif_head_backward(d, p, p, state, p, 7, None, 8, None, p, bwd, None) == -1
    assert lib.nif_head_backward(d, p, p, state, p, 8, p, 8, None, p, bwd - 1, None) == -2
    assert lib.nif_head_backward(d, p, p, state, None, 8, None, 8, None, p, bwd, None) == 0  # nothing asked for
    assert lib.nif_head_state_bytes(_desc(features=-1)) == 0
    for none in (_desc(rows=0), _desc(rows=0, hidden=None, labels=None)):  # no rows is a problem like any other
        assert lib.nif_head_state_bytes(none) > 0 and lib.nif_head_backward_workspace_bytes(none) > 0

    n, k = 6, 3
    state, ws = lib.nif_distill_state_bytes(n, k), lib.nif_distill_workspace_bytes(n)
    args = lambda ld=5, rows=n, classes=5, dt=0, top=k, tau=1.0, red=1: (  # noqa: E731
        p, ld, rows, classes, dt, p, p, None, top, tau, red, p)
    f = lib.nif_distill_forward
    for bad in (dict(ld=4), dict(rows=-1), dict(classes=0), dict(dt=1), dict(top=0), dict(top=1025), dict(tau=0.0),
                dict(tau=float('inf')), dict(red=7)):
        assert f(*args(**bad), p, 1 << 30, p, 1 << 30, None) == -1
    assert f(*args(), p, state - 1, p, ws, None) == -2
    assert f(*args(), p, state, p, ws - 1, None) == -2
    assert lib.nif_distill_backward(p, 5, n, 5, 0, k, 1.0, 1, p, p, state, p, 4, None) == -1
    assert lib.nif_distill_backward(p, 5, n, 5, 0, k, 1.0, 1, None, p, state, p, 5, None) == -1
    assert lib.nif_distill_backward(p, 5, n, 5, 0, k, 1.0, 1, p, p, state - 1, p, 5, None) == -2
    assert lib.nif_distill_backward(p, 5, 0, 5, 0, k, 1.0, 1, p, p, state, p, 5, None) == 0
    assert lib.nif_top_logits(p, 5, n, 5, 0, 6, 1.0, p, p, p, None) == -1
    assert lib.nif_top_logits(p, 4, n, 5, 0, 2, 1.0, p, p, p, None) == -1
    assert lib.nif_top_logits(p, 5, n, 5, 0, 2, 1.0, p, None, p, None) == -1
    assert lib.nif_top_logits(p, 5, 0, 5, 0, 2, 1.0, p, p, p, None) == 0

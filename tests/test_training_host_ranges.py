"""Refusals of the training operators' later arguments and entry points, on a CPU."""
import ctypes as C

import pytest
import torch

from cognitive_aim_depth_estimation_amd import _lib
from cognitive_aim_depth_estimation_amd import training as T

P = 4096          # an address that no refused call follows


def t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def raw(name, *args):
    return getattr(_lib.lib(), name)(*args)


@pytest.mark.parametrize("fn,error,match", [
    (lambda: T.activation_backward(t(2, 3), t(2, 3), "gelu"), RuntimeError, "no CPU path"),
    (lambda: T.linear_forward(t(2, 3), t(4, 3), pre_activation=True), RuntimeError, "no CPU path"),
    (lambda: T.activation_backward(t(2, 3), t(2, 4), "gelu"), ValueError, "shape"),
    (lambda: T.activation_backward(t(2, 3), t(2, 3, dtype=torch.int8), "gelu"), TypeError, "bf16, fp16 or fp32"),
    (lambda: T.activation_backward(t(2, 3), t(2, 3), "none"), ValueError, "relu"),
    (lambda: T.activation_backward(t(2, 3), None, "relu"), TypeError, "Checkpoint8"),
    (lambda: T.linear_forward(t(2, 3), t(4, 3), checkpoint=True, pre_activation=True), ValueError, "two ways"),
    (lambda: T.linear(t(2, 3), t(4, 3, dtype=torch.float64)), TypeError, "weight must be"),
    (lambda: T._ops().scale_unit(t(4, dtype=torch.float32)), RuntimeError, "no CPU path"),
    (lambda: T._ops().scale_unit(t(4)), ValueError, "float32"),
    (lambda: T._ops().scale_unit(t(0, dtype=torch.float32)), ValueError, "vector"),
])
def test_refusals(fn, error, match):
    with pytest.raises(error, match=match):
        fn()


def test_entry_points_refuse():
    bad = -22
    assert raw("cogaim_scale_unit", P, P, None, 4, None) == bad and raw("cogaim_scale_unit", P, P, P, 0, None) == bad
    assert raw("cogaim_scale_unit", None, P, P, 4, None) == bad
    act = lambda dy=P, dt=0, ld=8, u=P, ut=2, ldu=8, du=P, dut=0, lddu=8, a=1, M=1, D=8: raw("cogaim_activation_bwd_from", dy, dt, ld, u, ut, ldu, du, dut, lddu, a, M, D, None)  # noqa: E731
    for k in (dict(dy=None), dict(dt=3), dict(ld=7), dict(u=None), dict(ut=-1), dict(ldu=7), dict(u=P + 2), dict(du=None), dict(dut=3), dict(lddu=7),
              dict(a=0), dict(a=3), dict(M=0), dict(D=0), dict(dy=P + 1)):
        assert act(**k) == bad, k


def test_pre_activation_descriptor():
    d = dict(x=P, w=P, y=P, ldx=64, ldw=64, ldy=32, M=4, N=32, K=64, dtype=0, y_dtype=0)
    size = lambda **k: raw("cogaim_linear_fwd_workspace_bytes", C.byref(_lib.LinearFwdDesc(**d, **k)))  # noqa: E731
    assert size(extended=1, pre=P) >= 0 and size(extended=1, pre=P + 1) == -22
    assert size(extended=0, pre=P + 1) >= 0            # a shorter descriptor has no such field


def test_layer_norm_backward_workspace_is_its_partial_rows():
    size = lambda M, D: raw("cogaim_layernorm_bwd_workspace_bytes", M, D)  # noqa: E731
    assert size(1, 8) == 2 * 8 * 4 and size(4, 768) == 2 * 768 * 4 and size(5, 768) == 2 * 2 * 768 * 4
    assert size(10 ** 6, 768) == 768 * 2 * 768 * 4 and size(10 ** 6, 16384) == 512 * 2 * 16384 * 4 and size(100, 4096) == 100 * 2 * 4096 * 4

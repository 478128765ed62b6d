"""Refusals of the training operators: arguments are checked before a device is needed, so all of this runs on a CPU."""
import ctypes as C

import pytest
import torch

from training_reference import decode, quantise

from cognitive_aim_depth_estimation_amd import _lib
from cognitive_aim_depth_estimation_amd import training as T

B = torch.bfloat16


def t(*shape, dtype=B):
    return torch.zeros(*shape, dtype=dtype)


def ck(*shape):
    return T.Checkpoint8(torch.zeros(*shape, dtype=torch.int8), torch.zeros(*shape[:-1], -(-shape[-1] // 32), dtype=torch.uint8))


f32 = torch.float32


@pytest.mark.parametrize("fn", [
    lambda: T.pack8(t(2, 3)),
    lambda: T.unpack8(ck(2, 3)),
    lambda: T.activation_backward(t(2, 3), ck(2, 3), "gelu"),
    lambda: T.layer_norm_forward(t(2, 3), t(3, dtype=f32), t(3, dtype=f32)),
    lambda: T.layer_norm_backward(t(2, 3), ck(2, 3), None, t(2, dtype=f32), t(3, dtype=f32)),
    lambda: T.linear_forward(t(2, 3), t(4, 3)),
    lambda: T.linear_backward_input(t(2, 4), t(4, 3)),
    lambda: T.linear_backward_weight(t(2, 4), t(2, 3)),
])
def test_no_cpu_path(fn):
    with pytest.raises(RuntimeError, match="no CPU path"):
        fn()


@pytest.mark.parametrize("fn,error", [
    (lambda: T.pack8(t(2, 3, dtype=torch.float64)), TypeError),
    (lambda: T.pack8(t(2, 0)), ValueError),
    (lambda: T.pack8([1.0]), TypeError),
    (lambda: T.unpack8(t(2, 3)), TypeError),
    (lambda: T.unpack8(ck(2, 3), torch.float64), TypeError),
    (lambda: T.unpack8(T.Checkpoint8(t(2, 40), t(2, 2))), TypeError),
    (lambda: T.unpack8(T.Checkpoint8(ck(2, 40).codes, ck(2, 32).exponents)), ValueError),
    (lambda: T.activation_backward(t(2, 3), ck(2, 3), "none"), ValueError),
    (lambda: T.activation_backward(t(2, 3), ck(2, 4), "gelu"), ValueError),
    (lambda: T.activation_backward(t(2, 3), ck(2, 3), "silu"), ValueError),
    (lambda: T.layer_norm_forward(t(2, 3), t(4, dtype=f32), t(3, dtype=f32)), ValueError),
    (lambda: T.layer_norm_forward(t(2, 3), t(3), t(3, dtype=f32)), ValueError),
    (lambda: T.layer_norm_forward(t(2, 3), None, t(3, dtype=f32)), ValueError),
    (lambda: T.layer_norm_forward(t(2, 3), t(3, dtype=f32), t(3, dtype=f32), eps=-1.0), ValueError),
    (lambda: T.layer_norm_forward(t(1, 16385), t(16385, dtype=f32), t(16385, dtype=f32)), ValueError),
    (lambda: T.layer_norm_forward(t(2, 3), t(3, dtype=f32), t(3, dtype=f32), out_dtype=torch.int32), TypeError),
    (lambda: T.layer_norm_backward(t(2, 3), t(2, 4), t(2, dtype=f32), t(2, dtype=f32), t(3, dtype=f32)), ValueError),
    (lambda: T.layer_norm_backward(t(2, 3), t(2, 3), None, t(2, dtype=f32), t(3, dtype=f32)), TypeError),
    (lambda: T.layer_norm_backward(t(2, 3), t(2, 3), t(2, dtype=f32), t(3, dtype=f32), t(3, dtype=f32)), ValueError),
    (lambda: T.layer_norm_backward(t(2, 3), ck(2, 3), None, t(2, dtype=f32), t(3, dtype=f32), add=t(1, 3)), ValueError),
    (lambda: T.linear_forward(t(2, 3, dtype=f32), t(4, 3)), TypeError),
    (lambda: T.linear_forward(t(2, 3), t(4, 3, dtype=torch.float16)), ValueError),
    (lambda: T.linear_forward(t(2, 3), t(4, 5)), ValueError),
    (lambda: T.linear_forward(t(2, 3), t(3)), ValueError),
    (lambda: T.linear_forward(t(2, 3), t(4, 3), t(3, dtype=f32)), ValueError),
    (lambda: T.linear_forward(t(2, 3), t(4, 3), activation="tanh"), ValueError),
    (lambda: T.linear_forward(t(2, 3), t(4, 3), activation="gelu", scale=t(4, dtype=f32)), ValueError),
    (lambda: T.linear_forward(t(2, 3), t(4, 3), residual=t(2, 3)), ValueError),
    (lambda: T.linear_backward_input(t(2, 3), t(4, 3)), ValueError),
    (lambda: T.linear_backward_input(t(2, 4), t(4, 3), "gelu"), ValueError),
    (lambda: T.linear_backward_input(t(2, 4), t(4, 3), "none", ck(2, 3)), ValueError),
    (lambda: T.linear_backward_input(t(2, 4), t(4, 3), "gelu", ck(2, 4)), ValueError),
    (lambda: T.linear_backward_input(t(2, 4), t(4, 3), "gelu", t(2, 3)), TypeError),
    (lambda: T.linear_backward_input(t(2, 4), t(4, 3), want_activation=True), ValueError),
    (lambda: T.linear_backward_input(t(2, 4), t(4, 3), scale=t(3, dtype=f32)), ValueError),
    (lambda: T.linear_backward_weight(t(2, 4), t(3, 3)), ValueError),
    (lambda: T.linear_backward_weight(t(2, 4), t(2, 3, dtype=torch.float16)), TypeError),
    (lambda: T.linear_backward_weight(t(2, 4), t(2, 3), x_scale=t(3, dtype=f32)), ValueError),
    (lambda: T.linear_backward_weight(t(2, 4), ck(2, 3), x_scale=t(4, dtype=f32)), ValueError),
    (lambda: T.linear_backward_weight(t(2, 4), t(2, 3), scale=t(4, dtype=f32)), ValueError),
    (lambda: T.linear_backward_weight(t(2, 4), t(2, 3), weight=t(4, 3)), ValueError),
    (lambda: T.linear_backward_weight(t(2, 4), t(2, 3), weight=t(3, 4), scale=t(4, dtype=f32)), ValueError),
    (lambda: T.mlp_half(t(2, 3), *[t(3, dtype=f32)] * 2, t(4, 3), t(4, dtype=f32), t(3, 5), t(3, dtype=f32)), ValueError),
    (lambda: T.mlp_half(t(2, 3), *[t(3, dtype=f32)] * 2, t(4, 3), t(4, dtype=f32), t(3, 4), t(3, dtype=f32), compute_dtype=f32), TypeError),
])
def test_refusals(fn, error):
    with pytest.raises(error):
        fn()


def raw(name, *args):
    return getattr(_lib.lib(), name)(*args)


P = 4096          # an address that no refused call follows


def test_entry_points_refuse():
    """-22 from the C entry points, before anything is launched."""
    bad = -22
    assert raw("cogaim_pack8", P, 3, 8, P, P, 1, 8, None) == bad
    assert raw("cogaim_pack8", P, 0, 7, P, P, 1, 8, None) == bad
    assert raw("cogaim_pack8", P + 1, 0, 8, P, P, 1, 8, None) == bad
    assert raw("cogaim_pack8", P, 0, 8, P, None, 1, 8, None) == bad
    assert raw("cogaim_pack8", P, 0, 8, P, P, 0, 8, None) == bad
    assert raw("cogaim_pack8", P, 0, 1 << 31, P, P, 1, (1 << 30) + 1, None) == bad
    assert raw("cogaim_unpack8", P, P, P, 0, 8, 1, 8, 7, None) == bad
    assert raw("cogaim_unpack8", P, P, P, 0, 7, 1, 8, 8, None) == bad
    assert raw("cogaim_activation_bwd", P, 0, 8, P, P, P, 0, 8, 0, 1, 8, None) == bad
    assert raw("cogaim_activation_bwd", P, 0, 8, P, P, P, 0, 8, 3, 1, 8, None) == bad
    assert raw("cogaim_layernorm_train_fwd", P, 2, 8, P, P, P, 0, 8, P, P, P, None, 1, 8, 1e-6, None) == bad
    assert raw("cogaim_layernorm_train_fwd", P, 2, 8, P, P, P, 0, 8, P, P, None, None, 1, 8, -1e-6, None) == bad
    assert raw("cogaim_layernorm_train_fwd", P, 2, 20000, P, P, P, 0, 20000, P, P, None, None, 1, 20000, 1e-6, None) == bad
    need = raw("cogaim_layernorm_bwd_workspace_bytes", 5, 8)
    assert need > 0 and raw("cogaim_layernorm_bwd_workspace_bytes", 0, 8) == bad
    ln = lambda x, codes, mean, n: raw("cogaim_layernorm_bwd", P, 0, 8, x, 2, 8, codes, codes, mean, P, P, None, 0, 0, P, 2, 8, P, P, 5, 8, P, n, None)  # noqa: E731
    assert ln(P, P, P, need) == bad and ln(None, None, P, need) == bad and ln(P, None, None, need) == bad and ln(P, None, P, need - 1) == bad


def test_descriptors_refuse():
    def fwd(**k):
        a = dict(x=P, w=P, y=P, ldx=64, ldw=64, ldy=32, M=4, N=32, K=64, dtype=0, y_dtype=0)
        a.update(k)
        return raw("cogaim_linear_fwd_workspace_bytes", C.byref(_lib.LinearFwdDesc(**a)))
    assert fwd() >= 0
    for k in (dict(x=None), dict(M=0), dict(M=0x7fffffff), dict(N=-1), dict(K=0), dict(dtype=2), dict(y_dtype=3), dict(ldx=63), dict(ldw=1 << 22), dict(ldy=31),
              dict(activation=3), dict(activation=2, scale=P), dict(codes=P), dict(residual=P, ldr=31), dict(residual=P, ldr=32, residual_dtype=5),
              dict(x=P + 1)):
        assert fwd(**k) == -22, k
    assert raw("cogaim_linear_fwd_workspace_bytes", None) == -22
    d = _lib.LinearFwdDesc(x=P, w=P, y=P, ldx=61, ldw=64, ldy=32, M=4, N=32, K=61, dtype=0)
    assert raw("cogaim_linear_fwd_workspace_bytes", C.byref(d)) == 0    # few rows are read where they lie
    d.M = 64
    need = raw("cogaim_linear_fwd_workspace_bytes", C.byref(d))
    assert need > 0                                                     # rows that 16-byte loads cannot address are copied
    assert raw("cogaim_linear_fwd", C.byref(d), P, need - 1, None) == -22 and raw("cogaim_linear_fwd", C.byref(d), None, need, None) == -22

    def inp(**k):
        a = dict(dy=P, w=P, dx=P, lddy=32, ldw=64, lddx=64, M=4, N=32, K=64, dtype=0, dx_dtype=0)
        a.update(k)
        return raw("cogaim_linear_bwd_input_workspace_bytes", C.byref(_lib.LinearBwdInputDesc(**a)))
    assert inp() >= 0 and inp(activation=2, codes=P, exponents=P, a=P, lda=64) >= 0
    for k in (dict(dy=None), dict(activation=1), dict(codes=P, exponents=P), dict(a=P, lda=64), dict(lddx=63), dict(dtype=2),
              dict(activation=2, codes=P), dict(activation=2, codes=P, exponents=P, a=P, lda=8)):
        assert inp(**k) == -22, k

    def wgt(**k):
        a = dict(dy=P, x=P, dw=P, db=P, lddy=32, ldx=64, lddw=64, M=4, N=32, K=64, dtype=0, dw_dtype=2)
        a.update(k)
        return raw("cogaim_linear_bwd_weight_workspace_bytes", C.byref(_lib.LinearBwdWeightDesc(**a)))
    assert wgt() >= 0 and wgt(x=None, codes=P, exponents=P, x_scale=P) > 0 and wgt(scale=P, ds=P, w=P, ldw=64) > 0
    for k in (dict(x=None), dict(codes=P, exponents=P), dict(x_scale=P), dict(scale=P), dict(ds=P), dict(scale=P, ds=P), dict(db=None), dict(lddw=8)):
        assert wgt(**k) == -22, k


def test_reference_quantiser_is_within_half_a_step():
    x = torch.randn(7, 100) * torch.exp(3 * torch.randn(7, 1))
    codes, exps = quantise(x)
    step = torch.exp2(exps.double() - 127).repeat_interleave(32, 1)[:, :100]
    assert bool(((decode(codes, exps) - x.double()).abs() <= step / 2).all())
    top = torch.stack([codes[:, g:g + 32].abs().amax(1) for g in range(0, 100, 32)], 1)
    assert bool((top >= 63).all())

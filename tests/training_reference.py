"""Plain float64 statements of the training operators and the error bounds their fp32 arithmetic is held to.

U32 = 2^-24 is fp32's half step; a sum whose longest chain has n additions is off by at most n U32 times the sum of the
magnitudes.  An output rounded to a type t adds finfo(t).eps / 2 of its value."""
import math

import torch

U32 = 2.0 ** -24
GROUP = 32


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    """Half the spacing of the type's subnormal numbers."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def quantise(x):
    """(codes int8, exponents uint8) of a 2-D tensor, in float64 / integer arithmetic on the host's terms."""
    x = x.double().cpu()
    M, D = x.shape
    G = -(-D // GROUP)
    codes = torch.zeros(M, D, dtype=torch.int8)
    exps = torch.zeros(M, G, dtype=torch.uint8)
    for g in range(G):
        v = x[:, g * GROUP:(g + 1) * GROUP]
        top = v.abs().amax(1)
        bad = ~torch.isfinite(v).all(1)
        m, p = torch.frexp(torch.where(bad, torch.ones_like(top), top))        # top = m 2^p, m in [0.5, 1)
        e = torch.where(m == 0, torch.full_like(p, -126), p - 7 + (m * 128 >= 127.5).to(p.dtype)).clamp(min=-126)
        q = torch.round(torch.where(bad[:, None], torch.zeros_like(v), v) * torch.exp2(-e.double())[:, None])
        assert int(q.abs().max()) <= 127
        q = torch.where(e[:, None] == 122, q.clamp(-63, 63), q)                # 64 * 2^122 is no finite fp32 number
        codes[:, g * GROUP:(g + 1) * GROUP] = q.to(torch.int8)
        exps[:, g] = torch.where(bad, torch.full_like(e, 255), e + 127).to(torch.uint8)
    return codes, exps


def decode(codes, exps):
    """float64 values of an 8-bit copy; NaN where the exponent says so."""
    e = exps.double() - 127
    step = torch.where(exps == 255, torch.full_like(e, float("nan")), torch.exp2(e))
    return codes.double() * step.repeat_interleave(GROUP, -1)[..., : codes.shape[-1]]


def steps(exps, D):
    return torch.exp2(exps.double() - 127).repeat_interleave(GROUP, -1)[..., :D]


def act(u, name):
    if name == "relu":
        return u.clamp(min=0)
    return u * torch.special.ndtr(u) if name == "gelu" else u


def slope(u, name):
    if name == "relu":
        return (u > 0).double()
    return torch.special.ndtr(u) + u * torch.exp(-u * u / 2) / math.sqrt(2 * math.pi)


def within(got, want, bound, what=""):
    """got within bound of want, element by element; the same elements infinite or NaN."""
    got, want = got.double(), want.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got)), what
    off = torch.where(fine, (got - want).abs() - bound, torch.zeros_like(want))
    worst = float(off.max()) if off.numel() else 0.0
    at = int(off.argmax()) if off.numel() else 0
    assert worst <= 0, (what, "over its bound by", worst, "got", float(got.flatten()[at]), "want", float(want.flatten()[at]))

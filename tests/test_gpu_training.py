"""The training operators (layer norm, linear layers, 8-bit activations) against float64, at the sizes, types, strides and
values where they can go wrong, and together as one MLP half of an encoder layer."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

from training_reference import U32, act, decode, half_step, least, quantise, slope, steps, within  # noqa: E402

from cognitive_aim_depth_estimation_amd import training as T  # noqa: E402

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


@pytest.fixture(autouse=True)
def _dev():
    assert torch.cuda.is_available(), "these tests need the MI355X"
    torch.manual_seed(0)
    with torch.enable_grad():            # other test modules switch gradients off for the whole process
        yield
    torch.cuda.synchronize()


def rnd(*shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, device="cuda") * scale).to(dtype)


def laid(t, how):
    """The same values in another layout: rows further apart, or a base off the 16-byte grid."""
    if how == "plain":
        return t
    M, D = t.shape
    pad = {"padded": 8, "odd": 3, "offset": 8}[how]
    first = 1 if how == "offset" else 0
    big = torch.full((M, D + pad), float("nan"), device=t.device, dtype=t.dtype)
    big[:, first:first + D] = t
    return big[:, first:first + D]


# ---- 8 bits ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("M,D", [(1, 1), (3, 31), (2, 32), (5, 33), (7, 577), (300, 768), (3, 4104), (1, 100000)])
def test_pack8_is_the_definition(dtype, M, D):
    x = (rnd(M, D) * torch.exp(2 * rnd(M, 1))).to(DT[dtype])
    for how in ("plain", "padded", "odd", "offset"):
        got = T.pack8(laid(x, how))
        codes, exps = quantise(x)
        assert torch.equal(got.codes.cpu(), codes) and torch.equal(got.exponents.cpu(), exps), how
        want = decode(codes, exps)
        for out in DT.values():
            back = T.unpack8(got, out)
            assert back.dtype == out
            exact = want.clamp(-65504, 65504).to(out) if out == torch.float16 else want.to(out)
            assert torch.equal(back.cpu(), exact), (how, out)


def test_pack8_special_groups():
    """Zeros, the largest and the smallest numbers, magnitudes around the step's border, infinities and NaN: group by group."""
    top = torch.finfo(torch.float32).max
    rows = [
        [0.0] * 32, [-0.0] * 32, [top, -top] + [1.0] * 30, [2.0 ** -149] * 32, [2.0 ** -126, 2.0 ** -133] * 16,
        [127.5] + [0.5, 1.5, 2.5, -0.5, -1.5] * 6 + [0.0], [127.49999] + [1.0] * 31, [63.75] * 32, [63.749996] * 32,
        [255.0] + [1.0] * 31, [float("inf")] + [1.0] * 31, [-float("inf")] * 32, [float("nan")] + [3.0] * 31, [1.0] * 31 + [float("nan")],
    ]
    x = torch.tensor(rows, device="cuda")
    got = T.pack8(x)
    codes, exps = quantise(x)
    assert torch.equal(got.exponents.cpu(), exps) and torch.equal(got.codes.cpu(), codes)
    back = T.unpack8(got)
    bad = torch.tensor([not all(math.isfinite(v) for v in r) for r in rows])
    assert bool(torch.isnan(back.cpu()[bad]).all()) and bool(torch.isfinite(back.cpu()[~bad]).all())
    # one bad group does not reach its neighbours
    y = rnd(4, 96)
    y[1, 40] = float("nan")
    b = T.unpack8(T.pack8(y)).cpu()
    assert torch.isnan(b).sum() == 32 and bool(torch.isnan(b[1, 32:64]).all())
    # fp16's largest value rounds up past it in 8 bits and is held
    z = torch.full((1, 32), 65504.0, device="cuda", dtype=torch.float16)
    assert torch.equal(T.unpack8(T.pack8(z), torch.float16), z)


def test_unpack_leaves_what_lies_behind_the_rows():
    from cognitive_aim_depth_estimation_amd._lib import call, stream_ptr
    x = rnd(5, 40)
    p = T.pack8(x)
    out = torch.full((7, 64), 9.0, device="cuda", dtype=torch.bfloat16)
    call("cogaim_unpack8", p.codes.data_ptr(), p.exponents.data_ptr(), out.data_ptr(), 0, 64, 5, 40, 48, stream_ptr())
    assert torch.equal(out[:5, :40].cpu(), decode(*[t.cpu() for t in p]).to(torch.bfloat16))
    assert bool((out[:5, 40:48] == 0).all()) and bool((out[:5, 48:] == 9).all()) and bool((out[5:] == 9).all())


# ---- layer norm --------------------------------------------------------------------------------------------------
WIDTHS = [1, 5, 31, 64, 255, 577, 768, 1000, 1024, 2048, 2056, 3000, 4096, 4100, 8192, 12000, 16384]
CHAIN = 128         # additions on the longest chain of a row's sum: at most 32 in a thread, 6 in a wave, 16 waves; twice for two sums


def ln_case(M, D, x_dtype, how="plain"):
    x = rnd(M, D) * (0.5 + torch.rand(M, 1, device="cuda") * 3) + 0.7
    if D > 8:
        x[:, D // 2] += 30
    x = laid(x.to(x_dtype), how)
    return x, 1 + 0.2 * rnd(D), 0.1 * rnd(D)


def ln_reference(x, w, b, eps):
    """y, mean, rstd, rows and the bound on the rows' error: the mean's error over the spread, and the statistics' own."""
    d = x.double()
    mean = d.mean(1, keepdim=True)
    var = (d - mean).square().mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    h = (d - mean) * rstd
    off = CHAIN * U32 * d.abs().mean(1, keepdim=True) * rstd
    bound = off + h.abs() * (CHAIN * U32 + off * off + 2 * off * CHAIN * U32)
    return h * w.double() + b.double(), mean, rstd, h, bound


@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("x_dtype,y_dtype", [("fp32", "bf16"), ("bf16", "bf16"), ("fp16", "fp32"), ("fp32", "fp16")])
def test_layer_norm_forward(D, x_dtype, y_dtype):
    eps = 1e-6
    for M, how in ((1, "plain"), (6, "plain"), (3, "padded"), (5, "odd"), (2, "offset")):
        x, w, b = ln_case(M, D, DT[x_dtype], how)
        y, mean, rstd, saved = T.layer_norm_forward(x, w, b, eps, out_dtype=DT[y_dtype], checkpoint=True)
        want, m, r, h, hb = ln_reference(x, w, b, eps)
        if D > 1:
            within(mean, m[:, 0], CHAIN * U32 * x.double().abs().mean(1), "mean")
            spread = CHAIN * U32 * x.double().abs().mean(1) * r[:, 0]
            within(rstd, r[:, 0], r[:, 0] * (CHAIN * U32 + spread * spread), "rstd")
        yb = hb * w.double().abs() + 2 * U32 * (h * w).abs() + U32 * b.double().abs()
        within(y, want, yb + half_step(DT[y_dtype]) * (want.abs() + yb) + least(DT[y_dtype]), ("y", M, how))
        kept = decode(saved.codes, saved.exponents)
        within(kept, h, 0.5 * steps(saved.exponents, D) + hb, ("saved", M, how))
        for g in range(0, D, 32):                       # no step larger than the group needs
            top = saved.codes[:, g:g + 32].abs().amax(1)
            assert bool((top[(saved.exponents[:, g // 32] > 1)] >= 63).all())


@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("dy_dtype,x_dtype,dx_dtype", [("bf16", "fp32", "fp32"), ("fp16", "fp16", "fp16"), ("fp32", "bf16", "bf16")])
@pytest.mark.parametrize("kept", [False, True])
def test_layer_norm_backward(D, dy_dtype, x_dtype, dx_dtype, kept):
    for M, how in ((1, "plain"), (9, "plain"), (5, "padded"), (4, "odd"), (6, "offset")):
        x, w, b = ln_case(M, D, DT[x_dtype], how)
        _, mean, rstd, saved = T.layer_norm_forward(x, w, b, 1e-6, checkpoint=True)
        dy = laid(rnd(M, D, dtype=DT[dy_dtype], scale=0.1), how)
        add = laid(rnd(M, D, dtype=DT[dx_dtype], scale=0.1), how) if M % 2 else None
        dx, dw, db = T.layer_norm_backward(dy, saved if kept else x, None if kept else mean, rstd, w, add=add, out_dtype=DT[dx_dtype])
        r, d = rstd.double()[:, None], dy.double()
        h = decode(saved.codes, saved.exponents) if kept else (x.double() - mean.double()[:, None]) * r
        g = d * w.double()
        want = r * (g - g.mean(1, keepdim=True) - h * (g * h).mean(1, keepdim=True))
        bound = CHAIN * U32 * r * (g.abs() + g.abs().mean(1, keepdim=True) + h.abs() * (g * h).abs().mean(1, keepdim=True))
        if add is not None:
            want = want + add.double()
            bound = bound + U32 * want.abs()
        within(dx, want, bound + half_step(DT[dx_dtype]) * (want.abs() + bound) + least(DT[dx_dtype]), ("dx", M, how))
        within(dw, (d * h).sum(0), CHAIN * U32 * (d * h).abs().sum(0), ("dw", M, how))
        within(db, d.sum(0), CHAIN * U32 * d.abs().sum(0), ("db", M, how))


@pytest.mark.parametrize("D,M", [(768, 5000), (577, 4100), (4096, 1500), (96, 20000)])
def test_layer_norm_backward_many_rows(D, M):
    """Rows past one per thread group: the reduction of the weight's gradient, its chain a block's rows and the blocks'."""
    x, w, b = ln_case(M, D, torch.float32)
    _, mean, rstd, _ = T.layer_norm_forward(x, w, b)
    dy = rnd(M, D, dtype=torch.bfloat16)
    dx, dw, db = T.layer_norm_backward(dy, x, mean, rstd, w)
    h, d = (x.double() - mean.double()[:, None]) * rstd.double()[:, None], dy.double()
    chain = M // 1024 + 80                     # rows of a block, its 4 waves, 32 blocks a thread, 32 threads
    within(dw, (d * h).sum(0), chain * U32 * (d * h).abs().sum(0), "dw")
    within(db, d.sum(0), chain * U32 * d.abs().sum(0), "db")
    again = T.layer_norm_backward(dy, x, mean, rstd, w)
    assert all(torch.equal(p, q) for p, q in zip((dx, dw, db), again))


def test_layer_norm_non_finite_rows_stay_in_their_row():
    x, w, b = ln_case(6, 768, torch.float32)
    x[2, 5] = float("inf")
    x[4, 700] = float("nan")
    y, _, _, saved = T.layer_norm_forward(x, w, b, checkpoint=True)
    kept = T.unpack8(saved)
    for r in range(6):
        assert bool(torch.isnan(y[r]).all()) == (r in (2, 4)) and bool(torch.isnan(kept[r]).all()) == (r in (2, 4))


# ---- linear layers -----------------------------------------------------------------------------------------------
SHAPES = [(1, 1, 1), (1, 8, 8), (5, 64, 64), (3, 577, 588), (65, 129, 72), (130, 256, 768), (64, 200, 8), (257, 1000, 264),
          (31, 24, 4096), (1000, 96, 100), (9, 2048, 1024), (300, 1544, 520), (16, 2052, 1000), (17, 100, 72), (32, 333, 1001),
          (33, 333, 1001), (2, 7, 30), (40, 333, 5001)]
LARGE = [(2600, 4096, 264), (11000, 1000, 200), (2100, 2048, 4160), (700, 5000, 136), (20000, 520, 264), (2600, 264, 4096)]


def product_bound(A, B, K):
    """|A| |B|^T in float64 times the chain: K products, each exact in fp32, added in any order."""
    return (K + 8) * 2 * U32 * (A.double().abs() @ B.double().abs().t())


def check_forward(M, N, K, dtype, activation, with_scale, residual, out_dtype, layout="plain", bias=True):
    t = DT[dtype]
    x, w = laid(rnd(M, K, dtype=t), layout), laid(rnd(N, K, dtype=t, scale=K ** -0.5), layout)
    b = rnd(N) if bias else None
    s = 0.5 + torch.rand(N, device="cuda") if with_scale else None
    r = laid(rnd(M, N, dtype=DT[residual]), layout) if residual else None
    y, saved = T.linear_forward(x, w, b, activation=activation, scale=s, residual=r, out_dtype=DT[out_dtype], checkpoint=True)
    u = x.double() @ w.double().t() + (b.double() if bias else 0)
    ub = product_bound(x, w, K) + 2 * U32 * u.abs()
    want = act(u, activation)
    # |gelu'| <= 1.13; the tail's polynomial and the last operations: 2e-7 and two roundings
    yb = (1.13 * ub + 2e-7 + 4 * U32 * u.abs()) if activation == "gelu" else ub
    if with_scale:
        want, yb = want * s.double(), yb * s.double() + U32 * (want * s.double()).abs()
    if residual:
        want = want + r.double()
        yb = yb + U32 * want.abs()
    within(y, want, yb + half_step(DT[out_dtype]) * (want.abs() + yb) + least(DT[out_dtype]), "y")
    within(decode(saved.codes, saved.exponents), u, 0.5 * steps(saved.exponents, N) + ub, "saved")
    for g in range(0, N, 32):
        top = saved.codes[:, g:g + 32].abs().amax(1)
        assert bool((top[saved.exponents[:, g // 32] > 1] >= 63).all())
    plain, none = T.linear_forward(x, w, b, activation=activation, scale=s, residual=r, out_dtype=DT[out_dtype])
    assert none is None and torch.equal(plain, y)


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype,activation,scale,residual,out", [
    ("bf16", "none", False, None, "bf16"), ("fp16", "gelu", False, None, "fp16"), ("bf16", "relu", False, "fp32", "fp32"),
    ("fp16", "none", True, "fp32", "fp32"), ("bf16", "gelu", False, "bf16", "bf16"), ("fp16", "none", True, "fp16", "bf16")])
def test_linear_forward(M, N, K, dtype, activation, scale, residual, out):
    check_forward(M, N, K, dtype, activation, scale, residual, out)


@pytest.mark.parametrize("M,N,K", LARGE)
def test_linear_forward_large(M, N, K):
    check_forward(M, N, K, "bf16", "gelu", False, None, "bf16")
    check_forward(M, N, K, "fp16", "none", True, "fp32", "fp32", bias=False)


@pytest.mark.parametrize("layout", ["padded", "odd", "offset"])
def test_linear_forward_layouts(layout):
    check_forward(150, 136, 264, "bf16", "gelu", False, "bf16", "bf16", layout)
    check_forward(70, 33, 41, "fp16", "none", True, "fp32", "fp32", layout, bias=False)


def check_input(M, N, K, dtype, activation, with_scale, out_dtype, layout="plain"):
    t = DT[dtype]
    dy, w = laid(rnd(M, N, dtype=t, scale=0.1), layout), laid(rnd(N, K, dtype=t, scale=N ** -0.5), layout)
    s = 0.5 + torch.rand(N, device="cuda") if with_scale else None
    saved = T.pack8(1.4 * rnd(M, K)) if activation != "none" else None
    dx, a = T.linear_backward_input(dy, w, activation=activation, saved=saved, scale=s, out_dtype=DT[out_dtype], want_activation=activation != "none")
    # with a scale the matrix cores take W * scale, or (few rows) dy * scale, rounded to 16 bits: half a step of each product
    ws = w.double() * s.double()[:, None] if with_scale else w.double()
    want = dy.double() @ ws
    bound = (N + 8) * 2 * U32 * (dy.double().abs() @ ws.abs())
    if with_scale:
        bound = bound + 1.01 * dy.double().abs() @ (half_step(t) * ws.abs() + least(t)) + least(t) * w.double().abs().sum(0)
    if activation != "none":
        u = decode(saved.codes, saved.exponents)
        f = slope(u, activation)
        want, bound = want * f, bound * f.abs() + want.abs() * (3e-7 + 4 * U32) + U32 * (want * f).abs()
        value = act(u, activation)
        within(a, value, 2e-7 + (half_step(t) + 4 * U32) * value.abs() + least(t), "a")
        assert a.dtype == t
    else:
        assert a is None
    within(dx, want, bound + half_step(DT[out_dtype]) * (want.abs() + bound) + least(DT[out_dtype]), "dx")


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("dtype,activation,scale,out", [("bf16", "none", False, "bf16"), ("fp16", "gelu", True, "fp16"),
                                                        ("bf16", "relu", True, "fp32"), ("fp16", "gelu", False, "fp32")])
def test_linear_backward_input(M, N, K, dtype, activation, scale, out):
    check_input(M, N, K, dtype, activation, scale, out)


@pytest.mark.parametrize("M,N,K", [(1, 64, 40), (20, 333, 72), (150, 520, 264), (70, 33, 41), (300, 4096, 128)])
@pytest.mark.parametrize("size", [1e-5, 1.0, 3e4, 1e-30])
def test_linear_backward_input_fp16_scales(M, N, K, size):
    """fp16 with scales far from one.  Scale times an operand is rounded with the largest scale brought into [0.5, 1): by half
    a step of the product, or half of fp16's least number in units of at most twice the largest scale."""
    t = torch.float16
    dy, w = rnd(M, N, dtype=t, scale=0.1), rnd(N, K, dtype=t, scale=N ** -0.5)
    s = size * (0.5 + torch.rand(N, device="cuda"))
    dx, _ = T.linear_backward_input(dy, w, scale=s, out_dtype=torch.float32)
    ws, top = w.double() * s.double()[:, None], float(s.max())
    want, wide = dy.double() @ ws, dy.double().abs() @ ws.abs()
    bound = (N + 8) * 2 * U32 * wide + 1.01 * half_step(t) * wide
    bound = bound + 2.0 ** -24 * top * (dy.double().abs().sum(1, keepdim=True) + w.double().abs().sum(0)) + least(torch.float32)
    within(dx, want, bound + U32 * want.abs(), "dx")


@pytest.mark.parametrize("scales", ["zeros", "inf", "nan"])
@pytest.mark.parametrize("M", [3, 80])
def test_linear_backward_input_fp16_special_scales(M, scales):
    N, K = 64, 72
    dy, w = rnd(M, N, dtype=torch.float16), rnd(N, K, dtype=torch.float16)
    s = torch.zeros(N, device="cuda")
    if scales != "zeros":
        s[5] = float(scales)
    dx, _ = T.linear_backward_input(dy, w, scale=s, out_dtype=torch.float32)
    want = dy.double() @ (w.double() * s.double()[:, None])
    assert torch.equal(torch.isfinite(dx), torch.isfinite(want))
    if scales == "zeros":
        assert int(dx.count_nonzero()) == 0


@pytest.mark.parametrize("M,K,N", LARGE)
def test_linear_backward_input_large(M, K, N):
    check_input(M, N, K, "bf16", "gelu", False, "bf16")


@pytest.mark.parametrize("M,N,K", [(200, 128, 264), (2600, 264, 4096)])
def test_linear_backward_input_any_step(M, N, K):
    """Pre-activations whose groups span many steps: those the GELU table holds, smaller and larger ones, zeros and NaN,
    in one matrix; a group's result does not depend on the others of its wave."""
    u = rnd(M, K) * torch.exp2(torch.randint(-14, 8, (M, 1), device="cuda").float()) * torch.exp2(torch.randint(-2, 3, (1, K), device="cuda").float())
    u[5] = 0
    u[7, 40] = float("nan")
    saved = T.pack8(u)
    dy, w = rnd(M, N, dtype=torch.bfloat16), rnd(N, K, dtype=torch.bfloat16, scale=N ** -0.5)
    dx, a = T.linear_backward_input(dy, w, "gelu", saved, out_dtype=torch.float32, want_activation=True)
    v = decode(saved.codes, saved.exponents)
    ok = torch.isfinite(v)
    assert torch.equal(torch.isnan(dx), ~ok) and torch.equal(torch.isnan(a), ~ok) and int((~ok).sum()) == 32
    v = torch.where(ok, v, torch.zeros_like(v))
    G, f = dy.double() @ w.double(), slope(v, "gelu")
    bound = (N + 8) * 2 * U32 * (dy.double().abs() @ w.double().abs()) * f.abs() + G.abs() * (3e-7 + 4 * U32) + 2 * U32 * (G * f).abs()
    within(torch.where(ok, dx.double(), torch.zeros_like(v)), torch.where(ok, G * f, torch.zeros_like(v)), bound, "dx")
    value = act(v, "gelu")
    within(torch.where(ok, a.double(), torch.zeros_like(v)), torch.where(ok, value, torch.zeros_like(v)), 2e-7 + (half_step(torch.bfloat16) + 4 * U32) * value.abs() + least(torch.bfloat16), "a")


@pytest.mark.parametrize("layout", ["padded", "odd", "offset"])
def test_linear_backward_input_layouts(layout):
    check_input(150, 136, 264, "bf16", "gelu", True, "bf16", layout)
    check_input(70, 33, 41, "fp16", "relu", False, "fp32", layout)


def check_weight(M, N, K, dtype, kept, affine, with_scale, out_dtype="fp32", layout="plain"):
    t = DT[dtype]
    dy = laid(rnd(M, N, dtype=t, scale=0.1), layout)
    xs, xt = (1 + 0.2 * rnd(K), 0.1 * rnd(K)) if affine else (None, None)
    if kept:
        x = T.pack8(rnd(M, K))
        v = decode(x.codes, x.exponents)
        if affine:
            v = v * xs.double() + xt.double()
    else:
        x = laid(rnd(M, K, dtype=t), layout)
        v = x.double()
    more = {}
    if with_scale:
        more = {"weight": laid(rnd(N, K, dtype=t, scale=K ** -0.5), layout), "bias": rnd(N), "scale": 0.5 + torch.rand(N, device="cuda")}
    dW, db, ds = T.linear_backward_weight(dy, x, x_scale=xs, x_shift=xt, out_dtype=DT[out_dtype], **more)
    d = dy.double()
    G, total = d.t() @ v, d.sum(0)
    raw = (decode(x.codes, x.exponents) if kept else v).abs()
    Gb = (M + 8) * 2 * U32 * (d.abs().t() @ raw)
    tb = (M + 8) * 2 * U32 * d.abs().sum(0)
    if affine:
        Gb = Gb * xs.double().abs() + tb[:, None] * xt.double().abs() + 4 * U32 * ((d.abs().t() @ raw) * xs.double().abs() + d.abs().sum(0)[:, None] * xt.double().abs())
    if kept and t == torch.float16:          # values of an 8-bit copy below fp16's normal numbers are rounded to its grid
        Gb = Gb + d.abs().sum(0)[:, None] * least(t) * (xs.double().abs() if affine else 1)
    want, wb, wt, wtb = G, Gb, total, tb
    if with_scale:
        s = more["scale"].double()
        W = more["weight"].double()
        wds = (W * G).sum(1) + total * more["bias"].double()
        sb = (W.abs() * Gb).sum(1) + (K + 8) * U32 * (W * G).abs().sum(1) + (tb + 2 * U32 * total.abs()) * more["bias"].double().abs()
        within(ds, wds, sb + 2 * U32 * wds.abs(), "ds")
        want, wb = G * s[:, None], Gb * s[:, None] + U32 * (G * s[:, None]).abs()
        wt, wtb = total * s, tb * s + U32 * (total * s).abs()
    else:
        assert ds is None
    o = DT[out_dtype]
    within(dW, want, wb + half_step(o) * (want.abs() + wb) + least(o), "dW")
    within(db, wt, wtb + U32 * wt.abs(), "db")


@pytest.mark.parametrize("M,N,K", [(m, n, k) for n, k, m in SHAPES] + [(4096, 40, 24), (1370, 768, 768)])
@pytest.mark.parametrize("dtype,kept,affine,scale,out", [("bf16", False, False, False, "fp32"), ("fp16", True, True, False, "fp32"),
                                                         ("bf16", True, False, True, "bf16"), ("fp16", False, False, True, "fp16"),
                                                         ("bf16", True, True, True, "fp32")])
def test_linear_backward_weight(M, N, K, dtype, kept, affine, scale, out):
    check_weight(M, N, K, dtype, kept, affine, scale, out)


@pytest.mark.parametrize("M,N,K", [(264, 2600, 4096), (200, 11000, 1000), (4160, 2100, 2048), (136, 700, 5000), (20000, 520, 264), (11000, 1000, 200)])
def test_linear_backward_weight_large(M, N, K):
    check_weight(M, N, K, "bf16", False, False, False)
    check_weight(M, N, K, "fp16", True, True, True)


@pytest.mark.parametrize("layout", ["padded", "odd", "offset"])
def test_linear_backward_weight_layouts(layout):
    check_weight(150, 136, 264, "bf16", False, False, True, "bf16", layout)
    check_weight(70, 33, 41, "fp16", False, False, False, "fp32", layout)


def test_products_keep_rows_apart():
    """A NaN or an infinity in one row, column or (past the rows) behind a matrix reaches nothing else."""
    t = torch.bfloat16
    x, w = rnd(70, 88, dtype=t), rnd(40, 88, dtype=t)
    x[3, 87] = float("nan")
    y, _ = T.linear_forward(x, w)
    assert bool(torch.isnan(y[3]).all()) and int(torch.isnan(y).sum()) == 40
    dy = rnd(70, 40, dtype=t)
    dy[69, 39] = float("inf")
    dx, _ = T.linear_backward_input(dy, w)
    assert bool(torch.isfinite(dx[:69]).all()) and not bool(torch.isfinite(dx[69]).any())
    dW, db, _ = T.linear_backward_weight(dy, rnd(70, 88, dtype=t))
    assert bool(torch.isfinite(dW[:39]).all()) and not bool(torch.isfinite(dW[39]).any())
    assert bool(torch.isfinite(db[:39]).all()) and bool(torch.isinf(db[39]))


def test_a_group_that_overflowed_gives_nan_gradients():
    u = rnd(4, 64)
    u[1, 3] = float("inf")
    dy, w = rnd(4, 48, dtype=torch.bfloat16), rnd(48, 64, dtype=torch.bfloat16)
    for name in ("relu", "gelu"):
        dx, a = T.linear_backward_input(dy, w, activation=name, saved=T.pack8(u), want_activation=True)
        du = T.activation_backward(rnd(4, 64, dtype=torch.bfloat16), T.pack8(u), name)
        for t in (dx, a, du):
            bad = torch.isnan(t)
            assert bool(bad[1, :32].all()) and int(bad.sum()) == 32


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
@pytest.mark.parametrize("M,D", [(1, 1), (7, 33), (40, 1024)])
@pytest.mark.parametrize("name", ["relu", "gelu"])
def test_activation_backward(dtype, M, D, name):
    t = DT[dtype]
    u = T.pack8(2 * rnd(M, D))
    v = decode(u.codes, u.exponents)
    dy = rnd(M, D, dtype=t)
    want = dy.double() * slope(v, name)
    bound = dy.double().abs() * 3e-7 + 4 * U32 * want.abs()
    within(T.activation_backward(dy, u, name), want, bound + half_step(t) * want.abs() + least(t))
    assert T.activation_backward(dy, u, name, torch.float16).dtype == torch.float16


def test_residual_in_place_and_rows_behind_the_last():
    """y written over the residual, and nothing past the rows or the columns of a wider matrix."""
    import ctypes as C
    from cognitive_aim_depth_estimation_amd import _lib
    for M, N, K in ((77, 72, 64), (77, 75, 64), (700, 520, 72)):
        x, w = rnd(M, K, dtype=torch.bfloat16), rnd(N, K, dtype=torch.bfloat16, scale=K ** -0.5)
        big = torch.full((M + 3, N + 8), 5.0, device="cuda")
        big[:M, :N] = rnd(M, N)
        before = big.clone()
        d = _lib.LinearFwdDesc(x.data_ptr(), w.data_ptr(), None, None, big.data_ptr(), big.data_ptr(), None, None, K, K, N + 8, N + 8, M, N, K, 0, 2, 2, 0, 0)
        n = _lib.call("cogaim_linear_fwd_workspace_bytes", C.byref(d))
        ws = torch.empty(max(n, 1), device="cuda", dtype=torch.uint8)
        _lib.call("cogaim_linear_fwd", C.byref(d), ws.data_ptr(), n, _lib.stream_ptr())
        want = before[:M, :N].double() + x.double() @ w.double().t()
        within(big[:M, :N], want, product_bound(x, w, K) + 2 * U32 * want.abs())
        assert torch.equal(big[M:], before[M:]) and torch.equal(big[:, N:], before[:, N:])


def test_no_rows():
    e = lambda *s, dtype=torch.bfloat16: torch.empty(*s, device="cuda", dtype=dtype)  # noqa: E731
    w, g = rnd(24, 16, dtype=torch.bfloat16), rnd(16)
    y, mean, rstd, saved = T.layer_norm_forward(e(2, 0, 16), g, g, checkpoint=True)
    assert y.shape == (2, 0, 16) and mean.shape == (2, 0) and saved.codes.shape == (2, 0, 16) and saved.exponents.shape == (2, 0, 1)
    dx, dw, db = T.layer_norm_backward(e(2, 0, 16), saved, None, rstd, g)
    assert dx.shape == (2, 0, 16) and not bool(dw.any()) and not bool(db.any())
    y, saved = T.linear_forward(e(0, 16), w, checkpoint=True)
    assert y.shape == (0, 24) and saved.codes.shape == (0, 24)
    dx, a = T.linear_backward_input(e(0, 24), w, "gelu", T.pack8(e(0, 16)), want_activation=True)
    assert dx.shape == a.shape == (0, 16)
    dW, db, ds = T.linear_backward_weight(e(0, 24), e(0, 16), weight=w, scale=rnd(24))
    assert dW.shape == (24, 16) and not bool(dW.any()) and not bool(db.any()) and not bool(ds.any())
    assert T.unpack8(T.pack8(e(0, 5))).shape == (0, 5)
    assert T.activation_backward(e(0, 5), T.pack8(e(0, 5)), "gelu").shape == (0, 5)


# ---- together ----------------------------------------------------------------------------------------------------
def mlp_tensors(M, D, H, x_dtype=torch.float32):
    p = [rnd(M, D) * 1.5 + 0.2, 1 + 0.2 * rnd(D), 0.1 * rnd(D), rnd(H, D, scale=D ** -0.5), 0.1 * rnd(H), rnd(D, H, scale=H ** -0.5),
         0.1 * rnd(D), 0.5 + 0.5 * torch.rand(D, device="cuda")]
    p[0] = p[0].to(x_dtype)
    return [t.requires_grad_() for t in p]


def mlp_plain(x, g, b, w1, b1, w2, b2, s, eps=1e-6):
    h = torch.nn.functional.layer_norm(x, (x.shape[-1],), g, b, eps)
    u = h @ w1.t() + b1
    return x + s * ((u * torch.special.ndtr(u)) @ w2.t() + b2)


@pytest.mark.parametrize("M,D,H,dtype,x_dtype", [(37, 64, 256, "bf16", "fp32"), (300, 768, 520, "fp16", "fp32"), (70, 100, 130, "bf16", "bf16"), (1, 32, 48, "fp16", "fp16")])
def test_mlp_half_gradients(M, D, H, dtype, x_dtype):
    """All of a layer's MLP half in one step against float64 autograd.  The backward pass sees activations that are off by
    up to half a step of 8 bits, 1/127.5 of their group's largest magnitude (about 3 of their rms over 32 columns: 0.024 at
    most, uniform, so 0.0136 rms at the worst step), in the normalised rows and in the pre-activation, and its operands are
    rounded to 16 bits.  A gradient is a sum over many such independent errors, so in the 2-norm it is off by no more
    than the sum of the sources: 0.0136 (1 + max |gelu''| = 0.8) + five roundings of 2^-8, doubled for the fewest terms."""
    t = DT[dtype]
    p = mlp_tensors(M, D, H, DT[x_dtype])
    y = T.mlp_half(*p, compute_dtype=t)
    dy = rnd(M, D).to(y.dtype)
    grads = torch.autograd.grad(y, p, dy)
    q = [v.detach().double().requires_grad_() for v in p]
    ref = mlp_plain(*q)
    want = torch.autograd.grad(ref, q, dy.double())
    # forward: LN(x), W1, gelu, W2 rounded once each, the last two sums over many terms
    assert float((y.detach().double() - ref.detach()).norm() / ref.detach().norm()) <= 4 * half_step(t) + half_step(y.dtype)
    bound = 2 * (0.0136 * 1.8 + 5 * half_step(torch.bfloat16))
    for name, a, r, v in zip("x g b w1 b1 w2 b2 s".split(), grads, want, p):
        assert a.dtype == v.dtype and a.shape == v.shape
        off = float((a.double() - r.detach()).norm() / r.detach().norm())
        assert off <= bound, (name, off, bound)


def test_mlp_half_is_its_operators():
    """The fused step against the separate differentiable functions: the same kernels on the same values."""
    p = mlp_tensors(90, 96, 160)
    y = T.mlp_half(*p)
    x, g, b, w1, b1, w2, b2, s = p
    h = T.layer_norm(x, g, b, out_dtype=torch.bfloat16, checkpoint=True)
    a = T.linear(h, w1, b1, "gelu")
    z = T.linear(a, w2, b2, scale=s, residual=x, out_dtype=torch.float32)
    assert torch.equal(y, z)
    dy = rnd(90, 96)
    one, two = torch.autograd.grad(y, p, dy), torch.autograd.grad(z, p, dy)
    for u, v in zip(one, two):                     # recomputed operands differ in 8-bit steps
        assert float((u - v).norm() / v.norm()) < 0.05


def test_gradients_against_differences():
    """linear and layer_norm without 8-bit copies: directional differences of the forward in fp32 outputs."""
    torch.manual_seed(3)
    x, w, b = rnd(33, 72, dtype=torch.float16).requires_grad_(), rnd(40, 72, dtype=torch.float16, scale=0.1).requires_grad_(), rnd(40).requires_grad_()
    s, r = (0.5 + torch.rand(40, device="cuda")).requires_grad_(), rnd(33, 40).requires_grad_()
    f = lambda x, w, b, s, r: T.linear(x, w, b, scale=s, residual=r, out_dtype=torch.float32)  # noqa: E731
    dy = rnd(33, 40).half().float()                # what the products take of it is exact
    grads = torch.autograd.grad(f(x, w, b, s, r), (x, w, b, s, r), dy)
    args = [x, w, b, s, r]
    for i, g in enumerate(grads):
        # y is linear in each argument on its own: a difference over any distance is the derivative, to rounding
        step = torch.randint(-2, 3, args[i].shape, device="cuda").to(args[i].dtype) * 0.25
        moved = [(a + step).detach() if j == i else a.detach() for j, a in enumerate(args)]
        real = (moved[i].double() - args[i].detach().double())
        change = ((f(*moved).double() - f(*[a.detach() for a in args]).double()) * dy.double()).sum()
        want = (g.double() * real).sum()
        size = float((g.double() * real).norm()) + 1e-3
        # 16-bit gradients: half a step of each term; the scaled weight another; sums of independent roundings
        assert abs(float(change - want)) <= 8 * 2 * half_step(torch.float16) * size + 2e-3, (i, float(change), float(want))
    x = (rnd(11, 48) * 2 + 1).requires_grad_()
    g, b = (1 + 0.1 * rnd(48)).requires_grad_(), rnd(48).requires_grad_()
    dy = rnd(11, 48)
    grads = torch.autograd.grad(T.layer_norm(x, g, b), (x, g, b), dy)
    args = [x.detach(), g.detach(), b.detach()]
    for i, gr in enumerate(grads):
        v = rnd(*args[i].shape)
        e = 2.0 ** -6
        val = [float((T.layer_norm(*[a + k * e * v if j == i else a for j, a in enumerate(args)]).double() * dy.double()).sum()) for k in (-1, 1)]
        want = float((gr.double() * v.double()).sum())
        # e^2 / 6 of the third derivative (under 10 of the first's size here), and fp32 rounding over 2 e
        size = float(gr.norm() * v.norm())
        assert abs((val[1] - val[0]) / (2 * e) - want) <= size * (10 * e * e / 6 + 64 * U32 / e), (i, val, want)


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_encoder_mlp_trains_a_layer(dtype):
    """The model's own entry: value and gradients of one layer's MLP half on a residual stream, and the forward that follows
    an in-place step sees the new weights."""
    from util import default_exif, synth_model_and_sd
    model, _ = synth_model_and_sd(layers=2, native_grid=4, dtype=dtype)
    D = model.feature_dim
    x = rnd(2, 17, D, scale=1.5).requires_grad_()
    layer = getattr(model.backbone.encoder.layer, "1")
    named = [layer.norm2.weight, layer.norm2.bias, layer.mlp.fc1.weight, layer.mlp.fc1.bias, layer.mlp.fc2.weight, layer.mlp.fc2.bias, layer.layer_scale2.lambda1]
    for p in named:
        p.requires_grad_()
    y = model.encoder_mlp(1, x)
    assert y.shape == x.shape and y.dtype == torch.float32
    dy = rnd(2, 17, D)
    grads = torch.autograd.grad(y, [x] + named, dy)
    q = [v.detach().double().requires_grad_() for v in [x] + named]
    ref = mlp_plain(q[0], q[1], q[2], q[3], q[4], q[5], q[6], q[7], model.layer_norm_eps)
    want = torch.autograd.grad(ref, q, dy.double())
    assert float((y.detach().double() - ref.detach()).norm() / ref.detach().norm()) <= 4 * half_step(DT[dtype])
    bound = 2 * (0.0136 * 1.8 + 5 * half_step(torch.bfloat16))          # as in test_mlp_half_gradients
    for g, r in zip(grads, want):
        assert float((g.double() - r).norm() / r.norm()) <= bound
    images, exif = torch.randn(2, 3, 56, 56, device="cuda"), default_exif(2, "cuda")
    with torch.no_grad():
        before = model(images, exif)[0].clone()
        for p, g in zip(named, grads[1:]):
            p.add_(g, alpha=-0.05)
        after = model(images, exif)[0]
    assert bool(torch.isfinite(after).all()) and not torch.equal(before, after)
    with pytest.raises(IndexError):
        model.encoder_mlp(2, x)
    with pytest.raises(ValueError):
        model.encoder_mlp(0, x[..., :64])


def test_only_wanted_gradients_and_leading_dims():
    p = mlp_tensors(2 * 15, 64, 96)
    x = p[0].detach().view(2, 15, 64)
    y = T.mlp_half(x, *[v.detach() if i not in (4,) else v for i, v in enumerate(p[1:], 1)])
    assert y.shape == (2, 15, 64)
    y.sum().backward()
    assert p[4].grad is not None and all(v.grad is None for i, v in enumerate(p) if i != 4)
    y, mean, rstd, saved = T.layer_norm_forward(x, p[1].detach(), p[2].detach(), checkpoint=True)
    assert mean.shape == (2, 15) and saved.exponents.shape == (2, 15, 2)
    dx, dw, db = T.layer_norm_backward(x, saved, None, rstd, p[1].detach())
    flat = T.layer_norm_backward(x.view(30, 64), T.Checkpoint8(saved.codes.view(30, 64), saved.exponents.view(30, 2)), None, rstd.view(30), p[1].detach())
    assert torch.equal(dx.view(30, 64), flat[0]) and torch.equal(dw, flat[1])


def test_transposed_and_broadcast_inputs():
    """Views whose columns are not contiguous and rows that repeat are taken as the values they show."""
    x = rnd(64, 40, dtype=torch.bfloat16).t()
    w = rnd(64, 24, dtype=torch.bfloat16).t()
    y, _ = T.linear_forward(x, w)
    assert torch.equal(y, T.linear_forward(x.contiguous(), w.contiguous())[0])
    one = rnd(1, 64, dtype=torch.bfloat16).expand(9, 64)
    assert torch.equal(T.linear_forward(one, w)[0], T.linear_forward(one.contiguous(), w)[0])
    g = rnd(64)
    dx, dw, db = T.layer_norm_backward(one, one, torch.zeros(9, device="cuda"), torch.ones(9, device="cuda"), g)
    same = T.layer_norm_backward(one.contiguous(), one.contiguous(), torch.zeros(9, device="cuda"), torch.ones(9, device="cuda"), g)
    assert torch.equal(dx, same[0]) and torch.equal(dw, same[1]) and torch.equal(db, same[2])


@pytest.mark.parametrize("D", [1, 3, 5, 33, 577, 767, 1022, 2047, 4095, 8191, 12001])
@pytest.mark.parametrize("gap", [0, 3])
def test_a_row_ignores_what_lies_behind_it(D, gap):
    """NaN in every second row and between the rows: the others' results are those of the same rows alone."""
    M = 41
    def among(t):
        wide = torch.full((2 * M, D + gap), float("nan"), device="cuda", dtype=t.dtype)
        wide[::2, :D] = t
        return wide[:, :D]
    x, dy = rnd(M, D), rnd(M, D, dtype=torch.bfloat16)
    g, b = 1 + 0.1 * rnd(D), rnd(D)
    for t in (x, dy):
        p, q = T.pack8(among(t)), T.pack8(t)
        assert torch.equal(p.codes[::2], q.codes) and torch.equal(p.exponents[::2], q.exponents)
        assert bool((p.exponents[1::2] == 255).all())
        for o in (torch.bfloat16, torch.float32):
            assert torch.equal(T.unpack8(p, o)[::2], T.unpack8(q, o)) and bool(T.unpack8(p, o)[1::2].isnan().all())
        assert torch.equal(T.activation_backward(among(dy), p, "gelu")[::2], T.activation_backward(dy, q, "gelu"))
        y, mean, rstd, s = T.layer_norm_forward(among(t), g, b, out_dtype=torch.bfloat16, checkpoint=True)
        y2, mean2, rstd2, s2 = T.layer_norm_forward(t, g, b, out_dtype=torch.bfloat16, checkpoint=True)
        assert torch.equal(y[::2], y2) and torch.equal(mean[::2], mean2) and torch.equal(rstd[::2], rstd2)
        assert torch.equal(s.codes[::2], s2.codes) and torch.equal(s.exponents[::2], s2.exponents)
        assert torch.equal(T.layer_norm_backward(among(dy), among(t), mean, rstd, g, add=among(x))[0][::2],
                           T.layer_norm_backward(dy, t, mean2, rstd2, g, add=x)[0])
        assert torch.equal(T.layer_norm_backward(among(dy), s, None, rstd, g)[0][::2], T.layer_norm_backward(dy, s2, None, rstd2, g)[0])
        # a gradient that is zero in the other rows leaves the sums to these ones
        near = torch.zeros(2 * M, D, device="cuda", dtype=torch.bfloat16)
        near[::2] = dy
        full = torch.zeros(2 * M, D, device="cuda", dtype=t.dtype)
        full[::2] = t
        _, m3, r3, s3 = T.layer_norm_forward(full, g, b, checkpoint=True)
        h = (t.double() - mean2.double()[:, None]) * rstd2.double()[:, None]
        dg, db = T.layer_norm_backward(near, full, m3, r3, g)[1:]
        within(db, dy.double().sum(0), 4 * M * U32 * dy.double().abs().sum(0))
        within(dg, (dy.double() * h).sum(0), 4 * M * U32 * (dy.double() * h).abs().sum(0) + 8 * U32 * (dy.double().abs() * (h.abs() + mean2.double().abs()[:, None] * rstd2.double()[:, None])).sum(0))


def test_offsets_past_32_bits():
    """Matrices of more than 2^31 elements: their last rows against the same rows alone."""
    M, D = 600_000, 4096
    x = torch.empty(M, D, device="cuda", dtype=torch.bfloat16)
    x[-70:] = rnd(70, D, dtype=torch.bfloat16)
    x[:-70] = 1.0
    last = x[-70:].clone()
    p, q = T.pack8(x), T.pack8(last)
    assert torch.equal(p.codes[-70:], q.codes) and torch.equal(p.exponents[-70:], q.exponents)
    assert torch.equal(T.unpack8(p, torch.bfloat16)[-70:], T.unpack8(q, torch.bfloat16))
    g, b = 1 + 0.1 * rnd(D), rnd(D)
    y, mean, rstd, _ = T.layer_norm_forward(x, g, b)
    y2, mean2, rstd2, _ = T.layer_norm_forward(last, g, b)
    assert torch.equal(y[-70:], y2) and torch.equal(mean[-70:], mean2) and torch.equal(rstd[-70:], rstd2)
    dx = T.layer_norm_backward(x, p, None, rstd, g)[0]
    assert torch.equal(dx[-70:], T.layer_norm_backward(last, q, None, rstd2, g)[0])
    del y, dx
    w = rnd(64, D, dtype=torch.bfloat16, scale=D ** -0.5)
    z, s = T.linear_forward(x, w, activation="gelu", checkpoint=True)              # offsets of the operand
    dx, a = T.linear_backward_input(z, w, "gelu", p, want_activation=True)           # of the results and of the codes
    u = last.double() @ w.double().t()
    within(z[-70:], act(u, "gelu"), 1.13 * product_bound(last, w, D) + 2e-7 + 6 * U32 * u.abs() + half_step(z.dtype) * (1.01 * u.abs() + 1e-6))
    v = decode(q.codes, q.exponents)
    G, f = z[-70:].double() @ w.double(), slope(v, "gelu")
    within(dx[-70:], G * f, 80 * 2 * U32 * (z[-70:].double().abs() @ w.double().abs()) * f.abs() + G.abs() * 4e-7 + 1.01 * half_step(dx.dtype) * (G * f).abs())
    within(a[-70:], act(v, "gelu"), 2e-7 + 1.01 * half_step(a.dtype) * act(v, "gelu").abs())
    del dx, a
    # the weight's gradient walks down the rows: only the last 70 have a gradient, so it is theirs alone
    dy = torch.zeros(M, 64, device="cuda", dtype=torch.bfloat16)
    dy[-70:] = z[-70:]
    want, wide = dy[-70:].double().t() @ last.double(), dy[-70:].double().abs().t() @ last.double().abs()
    dw, db, _ = T.linear_backward_weight(dy, x)
    within(dw, want, 80 * 2 * U32 * wide)
    within(db, dy[-70:].double().sum(0), 80 * 2 * U32 * dy[-70:].double().abs().sum(0))
    dw = T.linear_backward_weight(dy, p)[0]
    within(dw, dy[-70:].double().t() @ v, 80 * 2 * U32 * (dy[-70:].double().abs().t() @ v.abs()))


def step_functions(p, dy):
    x, g, b, w1, b1, w2, b2, s = [v.detach() for v in p]
    v1, v2 = w1.bfloat16(), w2.bfloat16()
    h, _, rstd, rows = T.layer_norm_forward(x, g, b, out_dtype=torch.bfloat16, checkpoint=True)
    a, pre = T.linear_forward(h, v1, b1, "gelu", checkpoint=True)
    y, _ = T.linear_forward(a, v2, b2, scale=s, residual=x, out_dtype=x.dtype)
    d = dy.to(torch.bfloat16)
    du, a2 = T.linear_backward_input(d, v2, "gelu", pre, scale=s, want_activation=True)
    dw2, db2, ds = T.linear_backward_weight(d, a2, weight=v2, bias=b2, scale=s)
    dw1, db1, _ = T.linear_backward_weight(du, rows, x_scale=g, x_shift=b)
    dx, dg, db = T.layer_norm_backward(T.linear_backward_input(du, v1)[0], rows, None, rstd, g, add=dy, out_dtype=x.dtype)
    return y, dx, dg, db, dw1, db1, dw2, db2, ds


def test_captured_step_replays():
    """A training step in a graph, replayed on new inputs with eager work in between, against the eager step bit for bit;
    two graphs in turn (each has its own workspaces)."""
    graphs = []
    for M, D, H in ((150, 96, 200), (64, 768, 264)):
        p = [v.detach() for v in mlp_tensors(M, D, H)]
        dy = rnd(M, D)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step_functions(p, dy)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step_functions(p, dy)
        graphs.append((graph, p, dy, out))
    for turn in range(4):
        for graph, p, dy, out in graphs:
            with torch.no_grad():
                for v in p:
                    v.mul_(0.9).add_(0.01)
                dy.normal_()
            graph.replay()
        for graph, p, dy, out in graphs:
            want = step_functions(p, dy)
            torch.cuda.synchronize()
            for i, (a, r) in enumerate(zip(out, want)):
                assert torch.equal(a, r), (turn, i)


def test_two_streams_at_once():
    ps = [mlp_tensors(200, 128, 264), mlp_tensors(333, 96, 136)]
    dys = [rnd(200, 128), rnd(333, 96)]
    want = [step_functions(p, d) for p, d in zip(ps, dys)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = [None, None]
    for _ in range(5):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i] = step_functions(ps[i], dys[i])
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(a, r) for a, r in zip(got[i], want[i]))

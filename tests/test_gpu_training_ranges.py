"""The training operators at the ends of their types' ranges: results in fp16 near its largest and smallest numbers, results
that keep fp32's precision, the GELU's tails, ReLU's border, and more rows than one launch takes."""
import pytest
import torch

pytestmark = pytest.mark.gpu

from training_reference import U32, act, decode, half_step, least, slope, steps, within  # noqa: E402

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


def in_fp16(v):
    """What fp16 makes of decoded values: 64 steps of 1024 are what an 8-bit code makes of a finite fp16 number of 65024 or
    more, and are held at the largest finite one; anything larger is an infinity."""
    return torch.where(v.abs() <= 65536, v.clamp(-65504, 65504), v).to(torch.float16)


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_unpack8_to_fp16_overflows(dtype):
    x = torch.tensor([65504.0, 65536.0, 7e4, 1e6, 1e30, 3e38], device="cuda")
    x = torch.cat([x, -x])[:, None] * torch.linspace(0.01, 1, 41, device="cuda")
    saved = T.pack8(x.to(DT[dtype]))
    v = decode(saved.codes, saved.exponents)
    assert bool((v.abs() > 65536).any()) and bool((v.abs() == 65536).any())
    assert torch.equal(T.unpack8(saved, torch.float16), in_fp16(v))


@pytest.mark.parametrize("M", [3, 80])
@pytest.mark.parametrize("name", ["relu", "gelu"])
def test_activation_again_at_the_top_of_fp16(M, name):
    """The layer's input, made again from its 8-bit copy, is finite where it was in the forward."""
    N, K = 40, 72
    u = torch.full((M, K), 65500.0, device="cuda")
    u[1] = -65500.0
    u[2, 32:] = 1e6
    dy, w = rnd(M, N, dtype=torch.float16), rnd(N, K, dtype=torch.float16)
    saved = T.pack8(u)
    _, a = T.linear_backward_input(dy, w, name, saved, want_activation=True)
    want = in_fp16(act(decode(saved.codes, saved.exponents), name))
    assert torch.equal(torch.isinf(a), u > 1e5) and bool((a[0] == 65504).all())
    assert torch.equal(a[0], want[0]) and torch.equal(a[2], want[2]) and float(a[1].abs().max()) < 1e-6

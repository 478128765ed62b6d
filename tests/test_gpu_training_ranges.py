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

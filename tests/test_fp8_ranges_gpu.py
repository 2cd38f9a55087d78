"""Linear layers in 8 bits where numbers or sizes are at the ends of their ranges, and where a value that is missing would look like one that is
right: a NaN is neither above nor below a tolerance, so every comparison here asks for what has to hold and not for what must not."""
import pytest
import torch

from tests.fp8_util import BF, F8, blocks_of, held_close, product, product_off, random_held, unit, unit_off

pytestmark = pytest.mark.gpu
TYPES = {"bf16": BF, "f32": torch.float32}


@pytest.fixture
def mode():
    """sets the kernel that products take, and puts it back"""
    from llmq_b200 import lib
    yield lib.gemm_fp8_set_mode
    lib.gemm_fp8_set_mode(0)
    torch.cuda.synchronize()
    assert lib.load().b200q_wait_failures() == 0


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def held(code, scales, x, off, what=""):
    """held_close of finite codes and scales of rows"""
    assert torch.isfinite(code.float()).all() and torch.isfinite(scales).all(), f"{what}: not finite"
    held_close(code, scales, x, off, what=what)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("eps", [1e-12, 0.0])
@pytest.mark.parametrize("size", [1e-7, 1e-15])
@pytest.mark.parametrize("add", [True, False])
def test_norm_of_small_rows(cuda, dtype, eps, size, add):
    """rows whose factor 1 / sqrt(mean + eps) is a million or more: zeros stay zeros, as whole rows (a padded batch; with eps = 0 such a row is 0 x
    infinity) and as blocks, and blocks whose weights are next to nothing keep their codes.  Squares stay above 2^-126 but for those of row 3's
    smallest block, which are less than 2^-80 of the row's; everything else as in test_fp8_gpu.py's test_norm: 2^-17"""
    from llmq_b200 import lib
    T, H, t, g = 4, 640, TYPES[dtype], gen(11)
    x = torch.randn(T, H, generator=g, device="cuda") * size
    x[0] = 0.0 if eps else x[0]
    x[1, 128:256] = 0.0
    x[3, 256:384] *= 2.0 ** -40
    w = 1 + 0.3 * torch.randn(H, generator=g, device="cuda")
    w[384:512] *= 2.0 ** -105
    x, w = x.to(t), w.to(t)
    r = (0.5 * x.float()).to(t) if add else None
    v = ((x.float() + r.float()).to(t) if add else x).double()
    y, s = torch.empty(T, H, dtype=F8, device="cuda"), lib.fp8_row_scales(T, H)
    lib.rmsnorm_fp8(x, w, y, s, eps, residual=r)
    n = v * torch.rsqrt(v.square().mean(1, keepdim=True) + eps) * w.double()
    held(y, s[:, :T], n, n.abs() * 2.0 ** -17, what="norm")
    assert (y[1, 128:256].float() == 0.0).all() and (eps == 0.0 or (y[0].float() == 0.0).all())

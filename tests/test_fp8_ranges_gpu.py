"""Linear layers in 8 bits where numbers or sizes are at the ends of their ranges, and where a value that is missing would look like one that is
right: a NaN is neither above nor below a tolerance, so every comparison here asks for what has to hold and not for what must not."""
import pytest
import torch

from tests.fp8_util import BF, F8, blocks_of, held_close, product, product_off, random_held

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


@pytest.mark.parametrize("which", [1, 2, 3, "experts"])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_units_of_gates_that_next_to_nothing_is_left_of(cuda, mode, which, act):
    """act(gate) as little of the gate as 2^-127.6, less than the least reciprocal that fp32 has in full, and what it gates as large as 2^117, so that
    the product counts; a block whose exponentials pass fp32's range lets nothing through.  One code of each operand and scales of few bits to a sum:
    sums are exact."""
    from llmq_b200 import lib
    M, K = 6, 128
    a = torch.zeros(M, K, device="cuda")
    a[:, 0] = 1.0
    a, sa = a.to(F8), torch.ones(1, 8, device="cuda")
    sa[0, :M] = 1 + torch.arange(M, device="cuda") / 1024
    w = torch.zeros(768, K, device="cuda")
    gate = 88.0 if act == "silu" else 10.0
    w[:128, 0] = -gate
    w[256:384, 0] = -gate * torch.tensor([1.0, 0.5, 0.25, 0.125], device="cuda").repeat_interleave(32)
    w[512:640, 0] = -2.0 * gate
    w.view(3, 2, 128, K)[:, 1, :, 0] = torch.arange(128, device="cuda") % 4 + 1.0
    w, sw = w.to(F8), torch.ones(6, 1, device="cuda")
    sw[1::2] = 2.0 ** 115
    y, ys = torch.zeros(M, 384, dtype=F8, device="cuda"), lib.fp8_row_scales(M, 384)
    if which == "experts":
        tab, n = torch.tensor([[0, 0, M, 0]], dtype=torch.int32, device="cuda"), torch.ones(1, dtype=torch.int32, device="cuda")
        lib.gemm_grouped_gated_fp8(a, sa, w[None], sw[None], y, ys, tab, n, act)
    else:
        mode(which)
        lib.gemm_gated_fp8(a, sa, w, sw, y, ys, act)
    sums, _ = product(a, sa, w, sw)
    gate, up = (sums.view(M, 3, 2, 128)[:, :, i].flatten(1) for i in range(2))
    # (tanh GELU as gate x sigmoid, since 1 + tanh is 0 in 64 bits here, in unit_off too, whose share of the value for the unit's own arithmetic
    # is taken: 2^-19 (1 + |t|))
    t = gate if act == "silu" else 1.5957691216057308 * (gate + 0.044715 * gate ** 3)
    want = gate * torch.sigmoid(t) * up
    want[:, 256:] = 0.0
    held(y, ys[:, :M], want, want.abs() * 2.0 ** -19 * (1 + t.abs()) + 1e-30, what=str(which))
    assert (want[:, :256].abs() > 2.0 ** -10).all() and (y[:, :128].float() != 0.0).all()


@pytest.mark.parametrize("M", [1, 40])
def test_more_columns_than_small_tiles_go_round(cuda, M):
    """65536 tiles of 128 columns and eight columns more: small tiles are counted in a grid's second direction, which ends at 65535"""
    from llmq_b200 import lib
    N, K, g = 65536 * 128 + 8, 16, gen(M)
    a, sa = random_held(g, M, K, 1)
    w, sw = random_held(g, N, K, 128)
    c = torch.full((M, N), float("nan"), device="cuda")
    lib.gemm_fp8(a, sa, w, sw, c)
    ref, size = product(a, sa, w, sw)
    assert ((c.double() - ref).abs() <= product_off(size, K) + 1e-30).all()

"""Linear layers in 8 bits: what the documentation says of them and no other test asks.  Outputs are finite where inputs are (a comparison that asks
whether something is above a tolerance lets NaN pass), NaN and infinity stay in their rows and columns behind units and experts too, a row's bits in the
batch-invariant mode do not depend on its neighbours, tensors of more than 2^32 values, block counts that are no powers of two."""
import pytest
import torch

from tests import test_fp8_gpu as base
from tests.fp8_util import BF, F8, blocks_of, held_close, random_held, tile_table, values
from tests.test_fp8_gpu import mode  # noqa: F401

pytestmark = pytest.mark.gpu


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def held(code, scales, x, off, **kw):
    """held_close of finite codes and scales"""
    assert torch.isfinite(code.float()).all() and torch.isfinite(scales).all()
    held_close(code, scales, x, off, **kw)


# ---- finite ------------------------------------------------------------------------------------------------------------------
OUTPUTS = {"rmsnorm_fp8": lambda a: (a[2], a[3][:, :len(a[2])]), "quantize_fp8": lambda a: (a[1], a[2][:, :len(a[1])]), "quantize_fp8_weight": lambda a: a[1:3],
           "gemm_fp8": lambda a: a[4:5], "gemm_gated_fp8": lambda a: (a[4], a[5][:, :len(a[4])]), "gemm_grouped_fp8": lambda a: a[4:5],
           "gemm_grouped_gated_fp8": lambda a: (a[4], a[5][:, :len(a[4])])}


@pytest.fixture
def finite(monkeypatch):
    """every call's outputs are finite"""
    from llmq_b200 import lib

    def looked_at(name, call):
        def f(*args, **kw):
            call(*args, **kw)
            for t in OUTPUTS[name](args):
                assert torch.isfinite(t.float()).all(), f"{name}: not finite"
        return f

    for name in OUTPUTS:
        monkeypatch.setattr(lib, name, looked_at(name, getattr(lib, name)))


@pytest.mark.parametrize("M,N,K", base.SHAPES)
def test_products_are_finite(cuda, mode, finite, M, N, K):
    for which in (0, 1, 2, 3, 22, 32, 33, 204, 304, 804, 224, 524, 334, 205, 405):
        for out in ("bf16", "f32"):
            base.test_product(cuda, mode, M, N, K, which, out)


@pytest.mark.parametrize("M,N,K", [(1, 256, 16), (7, 2048, 144), (48, 4608, 2304), (129, 768, 640), (1001, 512, 400)])
def test_units_are_finite(cuda, mode, finite, M, N, K):
    for which in (0, 1, 2, 3):
        for act in ("silu", "gelu"):
            base.test_gated(cuda, mode, M, N, K, which, act)


@pytest.mark.parametrize("loads", list(base.LOADS))
def test_experts_are_finite(cuda, mode, finite, loads):
    for N, K in ((256, 128), (136, 272), (2048, 1024)):
        for out in ("bf16", "f32"):
            base.test_grouped(cuda, mode, loads, N, K, 0, out)
    for N, K in ((256, 128), (1024, 400), (2048, 2048)):
        base.test_grouped_gated(cuda, mode, loads, N, K, 0)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_rows_weights_and_norms_are_finite(cuda, finite, dtype):
    for T, K in ((1, 16), (7, 144), (33, 2048), (300, 400), (2, 16384)):
        base.test_quantize(cuda, dtype, T, K)
        for add in (True, False):
            base.test_norm(cuda, dtype, T, K, add)
    base.test_quantize_gathered(cuda, dtype)
    for shape in ((1, 16), (300, 2048), (3, 136, 272)):
        base.test_quantize_weight(cuda, dtype, shape)


# ---- NaN and infinity ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("which", [1, 2, 3, "experts"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_nan_and_infinity_behind_units(cuda, mode, which, bad):
    """a row with a bad block leaves NaN in all of its blocks and nowhere else, a bad square of weights in the units of its columns"""
    from llmq_b200 import lib
    M, N, K, g = 40, 768, 512, gen(3)
    x, w = torch.randn(M, K, generator=g, device="cuda"), torch.randn(N, K, generator=g, device="cuda") * K ** -0.5

    def run(x, w):
        a, sa = torch.empty(M, K, dtype=F8, device="cuda"), lib.fp8_row_scales(M, K)
        q, qs = torch.empty(N, K, dtype=F8, device="cuda"), torch.empty(blocks_of(N), blocks_of(K), device="cuda")
        lib.quantize_fp8(x, a, sa)
        lib.quantize_fp8_weight(w, q, qs)
        y, ys = torch.empty(M, N // 2, dtype=F8, device="cuda"), lib.fp8_row_scales(M, N // 2)
        if which == "experts":          # (rows 0 .. 16 and 17 .. 39 are two experts' with the same weights)
            tab, n = tile_table([17, M - 17])
            lib.gemm_grouped_gated_fp8(a, sa, torch.stack([q.view(torch.uint8)] * 2).view(F8), torch.stack([qs] * 2), y, ys, tab, n)
        else:
            mode(which)
            lib.gemm_gated_fp8(a, sa, q, qs, y, ys)
        return values(y, ys[:, :M])

    good = run(x, w)
    assert torch.isfinite(good).all()
    x[16, 200], x[17, 0] = bad, -bad
    v = run(x, w)
    assert torch.isnan(v[16:18]).all()
    kept = [r for r in range(M) if r not in (16, 17)]
    assert torch.equal(v[kept], good[kept])
    w[256 + 130, 300] = bad             # (the second block's units: what is gated)
    v = run(x, w)
    assert torch.isnan(v[:, 128:256]).all() and torch.equal(v[kept][:, :128], good[kept][:, :128]) and torch.equal(v[kept][:, 256:], good[kept][:, 256:])


@pytest.mark.parametrize("out", [BF, torch.float32])
def test_nan_and_infinity_behind_experts(cuda, out):
    """rows beside those of an expert whose rows or weights are bad, in one tile's box"""
    from llmq_b200 import lib
    loads, N, K, g = [5, 30, 140, 3], 264, 272, gen(4)
    a, sa = random_held(g, sum(loads), K, 1)
    held = [random_held(g, N, K, 128) for _ in loads]
    w, sw = torch.stack([h[0].view(torch.uint8) for h in held]).view(F8), torch.stack([h[1] for h in held])
    tab, n = tile_table(loads)
    good, bad = (torch.empty(sum(loads), N, dtype=out, device="cuda") for _ in range(2))
    lib.gemm_grouped_fp8(a, sa, w, sw, good, tab, n)
    sa[1, 20] = float("nan")
    sw[2, 0, 0] = float("inf")
    lib.gemm_grouped_fp8(a, sa, w, sw, bad, tab, n)
    assert torch.isfinite(good).all() and torch.isnan(bad[20]).all() and not torch.isfinite(bad[35:175, :128]).any()
    good[20] = bad[20] = 0.0
    good[35:175, :128] = bad[35:175, :128] = 0.0
    assert torch.equal(good, bad)


# ---- the batch-invariant mode ------------------------------------------------------------------------------------------------
@pytest.fixture
def invariant(cuda):
    """the hook that stands for B200Q_BATCH_INVARIANT"""
    from llmq_b200 import lib
    lib.check(lib.load().b200q_gemm_set_splitk(1))
    yield
    lib.check(lib.load().b200q_gemm_set_splitk(0))


ROWS = (1, 7, 33, 40, 64, 65, 129, 300, 700)


@pytest.mark.parametrize("N,K", [(1024, 2048), (4096, 4096), (2304, 9216), (136, 400)])
@pytest.mark.parametrize("out", [BF, torch.float32])
def test_products_in_the_batch_invariant_mode(invariant, N, K, out):
    from llmq_b200 import lib
    g = gen(N + K)
    (a, sa), (w, sw) = random_held(g, max(ROWS), K, 1), random_held(g, N, K, 128)
    want = None
    for M in ROWS[::-1]:
        c = torch.empty(M, N, dtype=out, device="cuda")
        lib.gemm_fp8(a[:M], sa, w, sw, c)
        want = c if want is None else want
        assert torch.equal(c, want[:M]), M


@pytest.mark.parametrize("N,K", [(512, 2048), (16384, 2048), (4608, 2304), (512, 400)])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_units_in_the_batch_invariant_mode(invariant, N, K, act):
    from llmq_b200 import lib
    g = gen(N + K)
    (a, sa), (w, sw) = random_held(g, max(ROWS), K, 1), random_held(g, N, K, 128)
    sa, sw = sa / 60, sw * (2.0 / 60 * K ** -0.5)
    want = None
    for M in ROWS[::-1]:
        y, ys = torch.empty(M, N // 2, dtype=F8, device="cuda"), lib.fp8_row_scales(M, N // 2)
        lib.gemm_gated_fp8(a[:M], sa, w, sw, y, ys, act)
        if want is None:
            want = y, ys
        assert torch.equal(y.view(torch.uint8), want[0][:M].view(torch.uint8)) and torch.equal(ys[:, :M], want[1][:, :M]), M


@pytest.mark.parametrize("gated", [False, True])
def test_experts_in_the_batch_invariant_mode(invariant, gated):
    """an expert's rows alone, and behind another's that shift them within their tiles"""
    from llmq_b200 import lib
    N, K, mine, g = 512, 1024, 150, gen(6)
    (a, sa), held = random_held(g, 800, K, 1), [random_held(g, N, K, 128) for _ in range(2)]
    sa = sa / 60
    w, sw = torch.stack([h[0].view(torch.uint8) for h in held]).view(F8), torch.stack([h[1] for h in held]) * (2.0 / 60 * K ** -0.5)
    want = None
    for before in (0, 1, 77, 128, 650):
        T, (tab, n) = before + mine, tile_table([before, mine])
        rows = torch.cat([torch.arange(800 - before, 800), torch.arange(mine)]).cuda()
        part, s = a.view(torch.uint8)[rows].view(F8), lib.fp8_row_scales(T, K)
        s[:, :T] = sa[:, rows]
        if gated:
            y, ys = torch.empty(T, N // 2, dtype=F8, device="cuda"), lib.fp8_row_scales(T, N // 2)
            lib.gemm_grouped_gated_fp8(part, s, w, sw, y, ys, tab, n)
            have = torch.cat([y[before:].float(), ys[:, before:T].t()], 1)
        else:
            c = torch.empty(T, N, device="cuda")
            lib.gemm_grouped_fp8(part, s, w, sw, c, tab, n)
            have = c[before:]
        want = have if want is None else want
        assert torch.equal(have, want), before


# ---- sizes -----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("K", [16 * 17, 128 * 5, 128 * 7 - 16, 128 * 11, 128 * 96, 128 * 127])
@pytest.mark.parametrize("gather", [False, True])
def test_rows_of_any_number_of_blocks(cuda, K, gather):
    """every block's scale tells its row and its place: they are numbered up to 300000, which is fewer than scales of 24 bits tell apart"""
    from llmq_b200 import lib
    n = blocks_of(K)
    T = 300000 // n
    number = torch.arange(1, T * n + 1, device="cuda", dtype=torch.float32).view(T, n)
    x = number.repeat_interleave(128, 1)[:, :K].contiguous()
    rows = torch.randperm(T, generator=gen(K), device="cuda").to(torch.int32) if gather else None
    y, s = torch.empty(T, K, dtype=F8, device="cuda"), lib.fp8_row_scales(T, K)
    lib.quantize_fp8(x, y, s, rows=rows)
    want = number[rows.long()] if gather else number
    assert (y.float() == 448.0).all()
    assert ((s[:, :T].t().double() * 448 - want.double()).abs() <= want.double() * 2.0 ** -22).all()


def some(T):
    return torch.cat([torch.arange(3), torch.arange(T // 2, T // 2 + 3), torch.arange(T - 3, T)]).cuda()


def test_rows_of_more_than_2_32_values(cuda):
    from llmq_b200 import lib
    T, K = 270000, 16384
    at, part = some(T), base.hard_rows(9, K, gen(7), BF)
    x = torch.zeros(T, K, dtype=BF, device="cuda")
    x[at] = part
    y, s = torch.empty(T, K, dtype=F8, device="cuda"), lib.fp8_row_scales(T, K)
    lib.quantize_fp8(x, y, s)
    held(y[at], s[:, at], part, 0.0, what="rows")
    assert (y[3:T // 2:997].float() == 0.0).all() and (y[T // 2 + 3:T - 3:997].float() == 0.0).all()
    del y
    torch.cuda.empty_cache()
    y, s = torch.empty(9, K, dtype=F8, device="cuda"), lib.fp8_row_scales(9, K)
    lib.quantize_fp8(x, y, s, rows=at.to(torch.int32))
    held(y, s[:, :9], part, 0.0, what="gathered")


def test_weights_of_more_than_2_32_values(cuda):
    from llmq_b200 import lib
    E, N, K = 3, 1400 * 64, 16384
    w = torch.zeros(E, N, K, dtype=BF, device="cuda")
    part = base.hard_rows(128, K, gen(8), BF)
    w[0, :128], w[1, 128:256], w[2, N - 128:] = part, part, part
    q, s = torch.empty(E, N, K, dtype=F8, device="cuda"), torch.empty(E, N // 128, K // 128, device="cuda")
    lib.quantize_fp8_weight(w, q, s)
    for e, n in ((0, 0), (1, 128), (2, N - 128)):
        held(q[e, n:n + 128], s[e, n // 128:n // 128 + 1], part, 0.0, tall=128, what=f"expert {e}")
    assert (q[:, 256:N - 128:997].float() == 0.0).all()


def test_norm_of_more_than_2_32_values(cuda):
    from llmq_b200 import lib
    T, H = 270000, 16384
    at = some(T)
    part, more = (torch.randn(9, H, generator=gen(9 + i), device="cuda").to(BF) for i in range(2))
    w = (1 + 0.3 * torch.randn(H, generator=gen(11), device="cuda")).to(BF)
    x, r = torch.zeros(T, H, dtype=BF, device="cuda"), torch.zeros(T, H, dtype=BF, device="cuda")
    x[at], r[at] = part, more
    y, s = torch.empty(T, H, dtype=F8, device="cuda"), lib.fp8_row_scales(T, H)
    lib.rmsnorm_fp8(x, w, y, s, 1e-5, residual=r)
    v = (part.float() + more.float()).to(BF)
    assert torch.equal(r[at], v)
    n = v.double() * torch.rsqrt(v.double().square().mean(1, keepdim=True) + 1e-5) * w.double()
    held(y[at], s[:, at], n, n.abs() * 2.0 ** -17, what="norm")
    assert (y[3:T // 2:997].float() == 0.0).all() and (r[3:T // 2:997] == 0).all()

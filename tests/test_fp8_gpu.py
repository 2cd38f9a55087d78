"""Linear layers in 8 bits (csrc/fp8_ops.cu, csrc/gemm_fp8.cu) through the C ABI, against plain 64-bit forms (tests/fp8_util.py)."""
import threading

import pytest
import torch

from tests.fp8_util import (BF, F8, blocks_of, held_close, product, product_off, random_held, spread, tile_table, unit, unit_off, values)

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


def hard_rows(T, K, g, dtype):
    """rows whose blocks are ordinary, zeros, tiny, huge, or full of values on the borders between two codes"""
    n = blocks_of(K)
    x = torch.randn(T, n, 128, generator=g, device="cuda")
    kind = torch.randint(0, 6, (T, n), generator=g, device="cuda")
    x = x * torch.exp2(torch.randint(-20, 18, (T, n, 1), generator=g, device="cuda").float())
    border = torch.tensor([448.0, 17.0, -19.0, 232.0, -0.0009765625, 0.0029296875, 1.0625, -3.75], device="cuda").repeat(16)
    x[kind == 1] = 0.0
    x[kind == 2] = 1e-36
    x[kind == 3] = border * 0.5
    x[kind == 4] = x[kind == 4] * 1e30
    return x.view(T, -1)[:, :K].contiguous().to(dtype)


def rows_of(scales, T):
    return scales[:, :T]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T,K", [(1, 128), (1, 16), (7, 144), (33, 2048), (300, 400), (1001, 4096), (2, 16384)])
def test_quantize(cuda, dtype, T, K):
    from llmq_b200 import lib
    x = hard_rows(T, K, gen(T + K), TYPES[dtype])
    y, s = torch.empty(T, K, dtype=F8, device="cuda"), lib.fp8_row_scales(T, K)
    s.fill_(-5.0)
    lib.quantize_fp8(x, y, s)
    held_close(y, rows_of(s, T), x, 0.0, what="rows")
    assert (s[:, T:] == -5.0).all()   # (behind the last row)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_quantize_gathered(cuda, dtype):
    """rows in any order, some twice; rows of wider rows"""
    from llmq_b200 import lib
    g = gen(5)
    wide = hard_rows(50, 1024, g, TYPES[dtype])
    rows = torch.randint(0, 50, (333,), generator=g, device="cuda").to(torch.int32)
    for x in (wide, wide[:, 128:128 + 272], wide[:, 8:8 + 16]):
        x = x if x.data_ptr() % 16 == 0 else x
        y, s = torch.empty(333, x.shape[1], dtype=F8, device="cuda"), lib.fp8_row_scales(333, x.shape[1])
        lib.quantize_fp8(x, y, s, rows=rows)
        held_close(y, rows_of(s, 333), x[rows.long()], 0.0, what="gathered")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("shape", [(128, 128), (1, 16), (8, 400), (300, 2048), (3, 136, 272), (5, 256, 128)])
def test_quantize_weight(cuda, dtype, shape):
    from llmq_b200 import lib
    g = gen(sum(shape))
    w = hard_rows(shape[-2] * (shape[0] if len(shape) == 3 else 1), shape[-1], g, TYPES[dtype]).view(shape)
    q = torch.empty(shape, dtype=F8, device="cuda")
    s = torch.empty(*shape[:-2], blocks_of(shape[-2]), blocks_of(shape[-1]), device="cuda")
    lib.quantize_fp8_weight(w, q, s)
    for i in range(shape[0] if len(shape) == 3 else 1):
        a, b, c = (w[i], q[i], s[i]) if len(shape) == 3 else (w, q, s)
        held_close(b, c, a, 0.0, tall=128, what="weights")


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("T,H", [(1, 2048), (1, 16), (5, 144), (64, 2304), (129, 3584), (300, 4096), (3, 16384)])
@pytest.mark.parametrize("add", [True, False])
def test_norm(cuda, dtype, T, H, add):
    from llmq_b200 import lib
    g, t = gen(T + H), TYPES[dtype]
    x = torch.randn(T, H, generator=g, device="cuda").to(t)
    r = (4 * torch.randn(T, H, generator=g, device="cuda")).to(t)
    w = (1 + 0.3 * torch.randn(H, generator=g, device="cuda")).to(t)
    if T > 2:
        x[1], r[1] = 0.0, 0.0
        x[2], r[2] = x[2] * 1e-4, r[2] * 1e-4
    kept = x.clone()
    v = (x.float() + r.float()).to(t) if add else x   # (the sum of two bf16 is exact in fp32, or rounded to bf16 as it would be from more bits
    #   but for ties that fp32 made: what the kernel wrote is what counts below)
    y, s = torch.empty(T, H, dtype=F8, device="cuda"), lib.fp8_row_scales(T, H)
    lib.rmsnorm_fp8(x, w, y, s, 1e-5, residual=r if add else None)
    assert torch.equal(x, kept)
    if add:
        assert torch.equal(r, v)
    d = v.double()
    n = d * torch.rsqrt(d.square().mean(1, keepdim=True) + 1e-5) * w.double()
    # sums of up to H squares in fp32 by threads, warps and blocks: at most 64 + 13 additions on a path, of like sign; square root, products
    held_close(y, rows_of(s, T), n, n.abs() * 2.0 ** -17, what="norm")


def test_nan_and_infinity(cuda):
    """a block with a NaN or an infinity reads back as NaN, its neighbours as they are"""
    from llmq_b200 import lib
    x = torch.ones(4, 384, device="cuda", dtype=BF)
    x[1, 130], x[2, 255], x[3, 128] = float("nan"), float("inf"), float("-inf")
    y, s = torch.empty(4, 384, dtype=F8, device="cuda"), lib.fp8_row_scales(4, 384)
    lib.quantize_fp8(x, y, s)
    v = values(y, s)
    assert torch.isnan(v[1:, 128:256]).all()
    assert torch.allclose(v[:, :128], torch.ones_like(v[:, :128]), rtol=2.0 ** -22) and not torch.isnan(v[0]).any() and not torch.isnan(v[:, 256:]).any()
    q, qs = torch.empty(256, 384, dtype=F8, device="cuda"), torch.empty(2, 3, device="cuda")
    w = torch.ones(256, 384, device="cuda")
    w[200, 383] = float("nan")
    lib.quantize_fp8_weight(w, q, qs)
    assert torch.isnan(values(q, qs, 128)).sum() == 128 * 128
    # a row's NaN stays in its row
    for m in (1, 2, 3):
        lib.gemm_fp8_set_mode(m)
        c = torch.empty(4, 256, dtype=BF, device="cuda")
        lib.quantize_fp8_weight(torch.ones(256, 384, device="cuda"), q, qs)
        lib.gemm_fp8(y, s, q, qs, c)
        assert torch.isfinite(c[0]).all() and torch.isnan(c[1:]).all()
    lib.gemm_fp8_set_mode(0)


SHAPES = [(1, 8, 16), (1, 4096, 4096), (5, 136, 144), (16, 256, 128), (33, 1000, 1024), (64, 2048, 2048), (100, 4096, 2064), (128, 384, 14336), (129, 512, 512),
          (200, 2304, 1152), (257, 264, 272), (300, 8192, 384), (513, 2048, 2048), (1001, 3584, 640), (2100, 1024, 256)]


@pytest.mark.parametrize("M,N,K", SHAPES)
@pytest.mark.parametrize("which", [0, 1, 2, 3])
@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_product(cuda, mode, M, N, K, which, out):
    from llmq_b200 import lib
    mode(which)
    g = gen(M + N + K)
    (a, sa), (w, sw) = random_held(g, M, K, 1, wild=M % 2 == 0), random_held(g, N, K, 128, wild=N % 16 == 0)
    c = torch.full((M + 1, N), 7.0, dtype=TYPES[out], device="cuda")
    lib.gemm_fp8(a, sa, w, sw, c[:M])
    ref, size = product(a, sa, w, sw)
    tol = product_off(size, K) + (ref.abs() * 2.0 ** -8 if out == "bf16" else 0.0) + 1e-30
    bad = (c[:M].double() - ref).abs() > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {((c[:M].double() - ref).abs() / tol).max().item():.3g}"
    assert (c[M] == 7.0).all()


# large tiles of 128 and 192 columns, and parts of the reduction: the test hook's mode is parts * 100 + columns / 64 * 10 + kernel
@pytest.mark.parametrize("M,N,K", [(1, 8, 16), (1, 4096, 4096), (100, 200, 272), (128, 384, 14336), (129, 512, 512), (200, 2304, 1152), (257, 264, 272),
                                   (300, 1000, 2064), (513, 2048, 2048), (1001, 3584, 640)])
@pytest.mark.parametrize("which", [22, 32, 33, 204, 304, 804, 224, 524, 334, 205, 405])
@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_product_of_other_tiles(cuda, mode, M, N, K, which, out):
    test_product(cuda, mode, M, N, K, which, out)


@pytest.mark.parametrize("M,N,K", [(3, 264, 400), (300, 520, 512), (1001, 768, 1024)])
@pytest.mark.parametrize("which", [22, 32, 33, 204, 804, 324, 305])
def test_whole_numbers_of_other_tiles(cuda, mode, M, N, K, which):
    test_whole_numbers(cuda, mode, M, N, K, which)


@pytest.mark.parametrize("M,N,K", [(3, 264, 400), (70, 1024, 2048), (128, 256, 1040), (300, 520, 512), (1001, 768, 1024)])
@pytest.mark.parametrize("which", [0, 1, 2, 3])
def test_whole_numbers(cuda, mode, M, N, K, which):
    """small whole codes and scales that are powers of two: every sum is exact in fp32, whatever the order"""
    from llmq_b200 import lib
    mode(which)
    g = gen(M * N)
    a = torch.randint(-4, 5, (M, K), generator=g, device="cuda").float().to(F8)
    w = torch.randint(-4, 5, (N, K), generator=g, device="cuda").float().to(F8)
    sa = torch.exp2(torch.randint(0, 3, (blocks_of(K), (M + 3) // 4 * 4 + 8), generator=g, device="cuda").float())
    sw = torch.exp2(torch.randint(0, 3, (blocks_of(N), blocks_of(K)), generator=g, device="cuda").float())
    c = torch.empty(M, N, device="cuda")
    lib.gemm_fp8(a, sa, w, sw, c)
    assert torch.equal(c.double(), product(a, sa, w, sw)[0])


@pytest.mark.parametrize("M,N,K", [(1, 256, 16), (1, 16384, 2048), (7, 2048, 144), (32, 512, 1024), (48, 4608, 2304), (128, 1024, 4096), (129, 768, 640),
                                   (300, 2048, 1024), (1001, 512, 400)])
@pytest.mark.parametrize("which", [0, 1, 2, 3])
@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_gated(cuda, mode, M, N, K, which, act):
    from llmq_b200 import lib
    mode(which)
    g = gen(M + N + K)
    (a, sa), (w, sw) = random_held(g, M, K, 1), random_held(g, N, K, 128)
    sa, sw = sa / 60, sw * (2.0 / 60 * K ** -0.5)   # (sums of a few units)
    y, ys = torch.zeros(M + 1, N // 2, dtype=F8, device="cuda"), lib.fp8_row_scales(M, N // 2)
    ys.fill_(-3.0)
    lib.gemm_gated_fp8(a, sa, w, sw, y[:M], ys, act)
    sums, size = product(a, sa, w, sw)
    held_close(y[:M], ys[:, :M], unit(sums, act), unit_off(sums, product_off(size, K), act), what="gated")
    assert (ys[:, M:] == -3.0).all() and (y[M].float() == 0.0).all()


LOADS = {"one": [1], "few": [0, 3, 0, 17, 1, 0], "even": [32] * 8, "uneven": [200, 0, 5, 128, 129, 31, 0, 64], "many": [700, 1, 333, 0, 256]}


@pytest.mark.parametrize("loads", list(LOADS))
@pytest.mark.parametrize("N,K", [(256, 128), (136, 272), (2048, 1024)])
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("out", ["bf16", "f32"])
def test_grouped(cuda, mode, loads, N, K, which, out):
    from llmq_b200 import lib
    mode(which)
    loads = LOADS[loads]
    T, E, g = sum(loads), len(loads), gen(N + K)
    a, sa = random_held(g, T, K, 1)
    held = [random_held(g, N, K, 128) for _ in loads]
    w, sw = torch.stack([h[0].view(torch.uint8) for h in held]).view(F8), torch.stack([h[1] for h in held])
    tab, n = tile_table(loads, T // 128 + E + 3)
    c = torch.full((T + 2, N), 7.0, dtype=TYPES[out], device="cuda")
    wide = torch.zeros(T + 2, K, dtype=F8, device="cuda")   # (two rows that no expert has: they stay)
    wide[:T] = a
    s = lib.fp8_row_scales(T + 2, K)
    s.fill_(float("nan"))
    s[:, :T] = sa[:, :T]
    lib.gemm_grouped_fp8(wide, s, w, sw, c, tab, n)
    at = 0
    for e, load in enumerate(loads):
        if load:
            ref, size = product(a[at:at + load], sa[:, at:at + load], w[e], sw[e])
            tol = product_off(size, K) + (ref.abs() * 2.0 ** -8 if out == "bf16" else 0.0) + 1e-30
            bad = (c[at:at + load].double() - ref).abs() > tol
            assert not bad.any(), f"expert {e}: {int(bad.sum())} off"
        at += load
    assert (c[T:] == 7.0).all()


@pytest.mark.parametrize("loads", list(LOADS))
@pytest.mark.parametrize("N,K", [(256, 128), (1024, 400), (2048, 2048)])
@pytest.mark.parametrize("which", [0, 1, 2])
def test_grouped_gated(cuda, mode, loads, N, K, which):
    from llmq_b200 import lib
    mode(which)
    loads = LOADS[loads]
    T, E, g = sum(loads), len(loads), gen(N + K)
    a, sa = random_held(g, T, K, 1)
    sa = sa / 60
    held = [random_held(g, N, K, 128) for _ in loads]
    w, sw = torch.stack([h[0].view(torch.uint8) for h in held]).view(F8), torch.stack([h[1] for h in held]) * (2.0 / 60 * K ** -0.5)
    tab, n = tile_table(loads)
    y, ys = torch.zeros(T, N // 2, dtype=F8, device="cuda"), lib.fp8_row_scales(T, N // 2)
    ys.fill_(-3.0)
    act = "gelu" if N == 1024 else "silu"
    lib.gemm_grouped_gated_fp8(a, sa, w, sw, y, ys, tab, n, act)
    at = 0
    for e, load in enumerate(loads):
        if load:
            sums, size = product(a[at:at + load], sa[:, at:at + load], w[e], sw[e])
            held_close(y[at:at + load], ys[:, at:at + load], unit(sums, act), unit_off(sums, product_off(size, K), act), what=f"expert {e}")
        at += load
    assert (ys[:, T:] == -3.0).all()


def test_no_rows(cuda):
    from llmq_b200 import lib
    w, sw = random_held(gen(1), 256, 128, 128)
    a, s = torch.empty(0, 128, dtype=F8, device="cuda"), lib.fp8_row_scales(0, 128)
    lib.gemm_fp8(a, s, w, sw, torch.empty(0, 256, dtype=BF, device="cuda"))
    lib.quantize_fp8(torch.empty(0, 128, dtype=BF, device="cuda"), a, s)
    lib.rmsnorm_fp8(torch.empty(0, 128, dtype=BF, device="cuda"), torch.ones(128, dtype=BF, device="cuda"), a, s, 1e-5)
    tab, n = torch.zeros(3, 4, dtype=torch.int32, device="cuda"), torch.zeros(1, dtype=torch.int32, device="cuda")
    full = torch.empty(5, 128, dtype=F8, device="cuda"), torch.ones(1, 8, device="cuda")
    c = torch.full((5, 256), 3.0, device="cuda")
    lib.gemm_grouped_fp8(*full, w[None], sw[None], c, tab, n)   # (a table of no tiles)
    assert (c == 3.0).all()


class Layer:
    """normed rows, one fused product, a quantised row of its output, a gated unit and the product down: a layer without its attention"""

    def __init__(self, T, H, I, seed):
        from llmq_b200 import lib
        g = gen(seed)
        self.x, self.residual = torch.randn(T, H, generator=g, device="cuda").to(BF), torch.randn(T, H, generator=g, device="cuda").to(BF)
        self.norm = torch.ones(H, dtype=BF, device="cuda")
        self.w = []
        for N, K in ((H, H), (2 * I, H), (H, I)):
            w = (torch.randn(N, K, generator=g, device="cuda") * K ** -0.5).to(BF)
            q, s = torch.empty(N, K, dtype=F8, device="cuda"), torch.empty(blocks_of(N), blocks_of(K), device="cuda")
            lib.quantize_fp8_weight(w, q, s)
            self.w.append((q, s))
        e = lambda n: torch.empty(T, n, dtype=F8, device="cuda")
        self.a, self.sa, self.b, self.sb = e(H), lib.fp8_row_scales(T, H), e(I), lib.fp8_row_scales(T, I)
        self.mid, self.out = torch.empty(T, H, dtype=BF, device="cuda"), torch.empty(T, H, dtype=BF, device="cuda")

    def run(self, stream=None):
        from llmq_b200 import lib
        lib.rmsnorm_fp8(self.x, self.norm, self.a, self.sa, 1e-5, residual=self.residual, stream=stream)
        lib.gemm_fp8(self.a, self.sa, *self.w[0], self.mid, stream=stream)
        lib.rmsnorm_fp8(self.mid, self.norm, self.a, self.sa, 1e-5, residual=self.residual, stream=stream)
        lib.gemm_gated_fp8(self.a, self.sa, *self.w[1], self.b, self.sb, stream=stream)
        lib.gemm_fp8(self.b, self.sb, *self.w[2], self.out, stream=stream)

    def plain(self):
        """the same from the kernels' own codes step by step: what each leaves is checked against 64 bits"""
        from llmq_b200 import lib
        r0 = self.residual.clone()
        lib.rmsnorm_fp8(self.x, self.norm, self.a, self.sa, 1e-5, residual=self.residual)
        v = (self.x.float() + r0.float()).to(BF).double()
        n = v * torch.rsqrt(v.square().mean(1, keepdim=True) + 1e-5)
        T = v.shape[0]
        held_close(self.a, self.sa[:, :T], n, n.abs() * 2.0 ** -17)
        lib.gemm_fp8(self.a, self.sa, *self.w[0], self.mid)
        ref, size = product(self.a, self.sa, *self.w[0])
        assert ((self.mid.double() - ref).abs() <= ref.abs() * 2.0 ** -8 + product_off(size, n.shape[1])).all()
        r1 = self.residual.clone()
        lib.rmsnorm_fp8(self.mid, self.norm, self.a, self.sa, 1e-5, residual=self.residual)
        assert torch.equal(self.residual, (self.mid.float() + r1.float()).to(BF))
        lib.gemm_gated_fp8(self.a, self.sa, *self.w[1], self.b, self.sb)
        sums, size = product(self.a, self.sa, *self.w[1])
        held_close(self.b, self.sb[:, :T], unit(sums, "silu"), unit_off(sums, product_off(size, n.shape[1]), "silu"))
        lib.gemm_fp8(self.b, self.sb, *self.w[2], self.out)
        ref, size = product(self.b, self.sb, *self.w[2])
        assert ((self.out.double() - ref).abs() <= ref.abs() * 2.0 ** -8 + product_off(size, self.b.shape[1])).all()


@pytest.mark.parametrize("T", [1, 40, 300])
def test_layer(cuda, T):
    Layer(T, 512, 768, 3).plain()


@pytest.mark.parametrize("T", [1, 40, 300])
def test_layer_captured(cuda, T):
    """captured and replayed, on a stream of its own: the same bits as called one by one"""
    layer = Layer(T, 1024, 1024, 4)
    first = layer.residual.clone()
    layer.run()
    torch.cuda.synchronize()
    want = [layer.out.clone(), layer.residual.clone(), layer.b.clone()]
    stream = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        layer.run()
    for _ in range(3):
        layer.residual.copy_(first)
        layer.out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(layer.out, want[0]) and torch.equal(layer.residual, want[1]) and torch.equal(layer.b.view(torch.uint8), want[2].view(torch.uint8))


def test_two_threads(cuda):
    """two layers at once, each on a stream and a thread of its own"""
    layers = [Layer(T, 1024, 1024, T) for T in (24, 280)]
    want, first = [], [layer.residual.clone() for layer in layers]
    for layer, r in zip(layers, first):
        layer.run()
        torch.cuda.synchronize()
        want.append(layer.out.clone())
        layer.residual.copy_(r)
    torch.cuda.synchronize()

    def work(layer, r, stream):
        for _ in range(20):
            with torch.cuda.stream(stream):
                layer.residual.copy_(r)
            layer.run(stream)

    threads = [threading.Thread(target=work, args=(layer, r, torch.cuda.Stream())) for layer, r in zip(layers, first)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    for layer, w in zip(layers, want):
        assert torch.equal(layer.out, w)


@pytest.mark.parametrize("T", [9, 300])
def test_routed_layer(cuda, T):
    """router, rows sorted by expert in 8 bits, both products, weighted sum: the framework's own calls on either side"""
    from llmq_b200 import lib
    g, E, top, H, I = gen(T), 8, 2, 512, 256
    x = torch.randn(T, H, generator=g, device="cuda").to(BF)
    logits = torch.randn(T, E, generator=g, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    idx, wts, off, perm, pair = (torch.empty(T * top, **i32), torch.empty(T * top, device="cuda"), torch.empty(E + 1, **i32),
                                 torch.empty(T * top, **i32), torch.empty(T * top, **i32))
    room = T * top // 128 + E
    tab, n = torch.zeros(room, 4, **i32), torch.zeros(1, **i32)
    L, s = lib.load(), torch.cuda.current_stream().cuda_stream
    lib.check(L.b200q_moe_route(logits.data_ptr(), T, E, top, idx.data_ptr(), wts.data_ptr(), off.data_ptr(), perm.data_ptr(), pair.data_ptr(),
                                tab.data_ptr(), n.data_ptr(), s))
    held = []
    for N, K in ((2 * I, H), (H, I)):
        w = (torch.randn(E, N, K, generator=g, device="cuda") * K ** -0.5).to(BF)
        q, qs = torch.empty(E, N, K, dtype=F8, device="cuda"), torch.empty(E, blocks_of(N), blocks_of(K), device="cuda")
        lib.quantize_fp8_weight(w, q, qs)
        held.append((q, qs))
    a, sa = torch.empty(T * top, H, dtype=F8, device="cuda"), lib.fp8_row_scales(T * top, H)
    b, sb = torch.empty(T * top, I, dtype=F8, device="cuda"), lib.fp8_row_scales(T * top, I)
    down, total = torch.empty(T * top, H, dtype=BF, device="cuda"), torch.zeros(T, H, device="cuda")
    zeros = torch.zeros(T, H, dtype=BF, device="cuda")
    lib.quantize_fp8(x, a, sa, rows=perm)
    lib.gemm_grouped_gated_fp8(a, sa, *held[0], b, sb, tab, n)
    lib.gemm_grouped_fp8(b, sb, *held[1], down, tab, n)
    lib.check(L.b200q_layer_sum(total.data_ptr(), zeros.data_ptr(), None, down.data_ptr(), pair.data_ptr(), wts.data_ptr(), top, None, None, T, H, 0, s))
    torch.cuda.synchronize()
    # what each token's experts give, from the codes that the kernels left
    want, off_by = torch.zeros(T, H, dtype=torch.float64, device="cuda"), torch.zeros(T, H, dtype=torch.float64, device="cuda")
    weight = torch.softmax(torch.gather(logits.double(), 1, idx.view(T, top).long()), 1)
    for t in range(T):
        for k in range(top):
            e, r = int(idx[t * top + k]), int(pair[t * top + k])
            held_close(a[r:r + 1], sa[:, r:r + 1], x[t:t + 1], 0.0)
            sums, size = product(a[r:r + 1], sa[:, r:r + 1], held[0][0][e], held[0][1][e])
            held_close(b[r:r + 1], sb[:, r:r + 1], unit(sums, "silu"), unit_off(sums, product_off(size, H), "silu"))
            ref, size = product(b[r:r + 1], sb[:, r:r + 1], held[1][0][e], held[1][1][e])
            want[t] += weight[t, k] * ref[0]
            off_by[t] += weight[t, k] * (product_off(size, I)[0] + ref[0].abs() * (2.0 ** -8 + 2.0 ** -20))
    assert ((total.double() - want).abs() <= off_by + 1e-6).all()


def test_order_of_sums_in_the_batch_invariant_mode(cuda, mode):
    """the hook that stands for B200Q_BATCH_INVARIANT: a row gives the same bits whatever the number of rows beside it"""
    from llmq_b200 import lib
    g = gen(8)
    (a, sa), (w, sw) = random_held(g, 700, 2048, 1), random_held(g, 1024, 2048, 128)
    lib.check(lib.load().b200q_gemm_set_splitk(1))
    try:
        outs = []
        for M in (1, 40, 129, 700):
            c = torch.empty(M, 1024, device="cuda")
            lib.gemm_fp8(a[:M], sa, w, sw, c)
            outs.append(c[0].clone())
        for o in outs[1:]:
            assert torch.equal(o, outs[0])
    finally:
        lib.check(lib.load().b200q_gemm_set_splitk(0))


def test_offsets_beyond_32_bits(cuda):
    """codes of a matrix of more than 2^32 bytes, and an output of more than 2^31 elements"""
    from llmq_b200 import lib
    g = gen(2)
    M, N, K = 280000, 8192, 16384
    w, sw = random_held(g, N, K, 128)
    rows = torch.cat([torch.arange(3), torch.arange(M // 2, M // 2 + 3), torch.arange(M - 3, M)])
    a = torch.zeros(M, K, dtype=torch.uint8, device="cuda").view(F8)
    sa = torch.ones(blocks_of(K), M, device="cuda")
    part, _ = random_held(g, 9, K, 1)
    a.view(torch.uint8)[rows.cuda()] = part.view(torch.uint8)
    c = torch.empty(M, N, dtype=BF, device="cuda")
    lib.gemm_fp8(a, sa, w, sw, c)
    ref, size = product(part, torch.ones(blocks_of(K), 9, device="cuda"), w, sw)
    assert ((c[rows.cuda()].double() - ref).abs() <= product_off(size, K) + ref.abs() * 2.0 ** -8).all()
    assert (c[3:M // 2:997] == 0).all()


def test_rule_reaches_every_kernel(cuda):
    """over the matrices of the built-in models every kernel and tile is taken somewhere"""
    from llmq_b200 import lib
    L = lib.load()
    shapes = ((6144, 4096), (4096, 4096), (4096, 14336), (2048, 2048), (2048, 8192), (8192, 3584), (3584, 4096), (3584, 14336), (4096, 2304), (2304, 9216))
    taken = {L.b200q_gemm_fp8_choice(m, N, K, 0) for N, K in shapes for m in range(1, 4609, 13)}
    assert {1, 22, 42, 33, 43} <= taken and {24, 34, 45} <= {t % 100 for t in taken if t > 100}, sorted(taken)
    assert {L.b200q_gemm_fp8_choice(m, 16384, 2048, 1) % 10 for m in range(1, 4609, 7)} == {1, 2, 3}


def test_first_call_in_a_capture(cuda):
    """a process whose first product is captured"""
    import subprocess
    import sys
    code = """
import torch
from llmq_b200 import lib
from tests.fp8_util import random_held, product, product_off
g = torch.Generator(device="cuda").manual_seed(0)
(a, sa), (w, sw) = random_held(g, 300, 1024, 1), random_held(g, 512, 1024, 128)
c = torch.zeros(300, 512, device="cuda")
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    lib.gemm_fp8(a, sa, w, sw, c)
graph.replay()
torch.cuda.synchronize()
ref, size = product(a, sa, w, sw)
assert ((c.double() - ref).abs() <= product_off(size, 1024)).all()
print("fine")
"""
    import os
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, cwd=root, timeout=120)
    assert r.returncode == 0 and "fine" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("act", ["silu", "gelu"])
def test_units_far_from_zero(cuda, mode, act):
    """gates of hundreds, of either sign, and of next to nothing: what a row of 128 is held as stays right"""
    from llmq_b200 import lib
    for which in (1, 2, 3):
        mode(which)
        a = torch.zeros(6, 128, device="cuda")
        a[:, 0] = torch.tensor([1.0, -1.0, 0.25, -0.25, 2.0 ** -9, 0.0])
        a, sa = a.to(F8), torch.ones(1, 8, device="cuda")
        w = torch.zeros(256, 128, device="cuda")
        w[:128, 0] = torch.linspace(-448, 448, 128)
        w[128:, 0] = torch.linspace(1, 3, 128)
        w, sw = w.to(F8), torch.ones(2, 1, device="cuda")
        y, ys = torch.empty(6, 128, dtype=F8, device="cuda"), lib.fp8_row_scales(6, 128)
        lib.gemm_gated_fp8(a, sa, w, sw, y, ys, act)
        sums, size = product(a, sa, w, sw)
        held_close(y, ys[:, :6], unit(sums, act), unit_off(sums, product_off(size, 128), act) + 1e-13, what=f"mode {which}")


def test_repeated_rows_and_layers_in_place(cuda):
    """the same row many times in a gather; a residual that is normed again and again"""
    from llmq_b200 import lib
    g = gen(3)
    x = torch.randn(7, 256, generator=g, device="cuda").to(BF)
    rows = torch.full((500,), 6, dtype=torch.int32, device="cuda")
    y, s = torch.empty(500, 256, dtype=F8, device="cuda"), lib.fp8_row_scales(500, 256)
    lib.quantize_fp8(x, y, s, rows=rows)
    assert (y.view(torch.uint8) == y.view(torch.uint8)[0]).all() and (s[:, :500] == s[:, :1]).all()
    r, w = torch.zeros(7, 256, dtype=BF, device="cuda"), torch.ones(256, dtype=BF, device="cuda")
    y, s = torch.empty(7, 256, dtype=F8, device="cuda"), lib.fp8_row_scales(7, 256)
    want = r.clone()
    for _ in range(5):
        lib.rmsnorm_fp8(x, w, y, s, 1e-5, residual=r)
        want = (x.float() + want.float()).to(BF)
    assert torch.equal(r, want)


@pytest.mark.parametrize("gated", [False, True])
def test_rows_of_a_table_stay_within_the_matrices(cuda, gated):
    """entries whose rows lie far outside are no rows at all, in whichever quarter of a tile their sum with the first row would turn over"""
    from llmq_b200 import lib
    g = gen(5)
    (a, sa), (w, sw) = random_held(g, 130, 256, 1), random_held(g, 256, 256, 128)
    last = 2 ** 31 - 1
    tab = torch.tensor([[0, last, last, 0], [0, last - 40, last, 0], [0, last - 100, 130, 0], [0, 130, last, 0], [0, 64, 100, 0]], dtype=torch.int32, device="cuda")
    n = torch.tensor([5], dtype=torch.int32, device="cuda")
    w, sw = w[None], sw[None]
    if gated:
        y, ys = torch.zeros(130, 128, dtype=F8, device="cuda"), lib.fp8_row_scales(130, 128)
        ys.fill_(-3.0)
        lib.gemm_grouped_gated_fp8(a, sa / 60, w, sw, y, ys, tab, n)
        out, none = ys[0, :130], -3.0
        assert (y[:64].float() == 0.0).all() and (y[100:].float() == 0.0).all()
    else:
        c = torch.full((130, 256), 7.0, device="cuda")
        lib.gemm_grouped_fp8(a, sa, w, sw, c, tab, n)
        out, none = c[:, 0], 7.0
        assert (c[:64] == 7.0).all() and (c[100:] == 7.0).all()
    assert (out[:64] == none).all() and (out[100:130] == none).all() and (out[64:100] != none).all()


def test_unknown_units_are_refused(cuda):
    from llmq_b200 import lib
    (a, sa), (w, sw) = random_held(gen(1), 4, 128, 1), random_held(gen(2), 256, 128, 128)
    y, ys = torch.zeros(4, 128, dtype=F8, device="cuda"), lib.fp8_row_scales(4, 128)
    with pytest.raises(lib.B200QError, match="act=-1"):
        lib.gemm_gated_fp8(a, sa, w, sw, y, ys, act="relu")
    assert (y.float() == 0.0).all()

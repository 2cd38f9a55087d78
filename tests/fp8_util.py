"""Values in 8 bits with a scale for each block of 128, in plain 64-bit arithmetic."""
import torch

BF, F8 = torch.bfloat16, torch.float8_e4m3fn
LEAST = 2.0 ** -100


def blocks_of(n):
    return (n + 127) // 128


def spread(scales, rows, K, tall=1):
    """scales [blocks down, blocks across] as one for each value [rows, K]"""
    return scales.double().repeat_interleave(tall, 0)[:rows].repeat_interleave(128, 1)[:, :K]


def values(code, scales, tall=1):
    """what codes [rows, K] stand for; scales of rows are [blocks, rows or more]"""
    rows, K = code.shape
    s = scales if tall > 1 else scales[:, :rows].t()
    return code.double() * spread(s, rows, K, tall)


def largest(x, tall=1):
    """largest magnitude of each block of x [rows, K]: [blocks down, blocks across]"""
    rows, K = x.shape
    down = (rows + tall - 1) // tall
    p = torch.zeros(down * tall, blocks_of(K) * 128, dtype=torch.float64, device=x.device)
    p[:rows, :K] = x.double().abs()
    return p.view(down, tall, -1, 128).amax((1, 3))


def half_step(r):
    """half the distance between neighbouring e4m3 numbers at |r|"""
    e = torch.frexp(r.abs().clamp(min=2.0 ** -6))[1].double()     # |r| < 2^e
    return torch.exp2(e - 5)


def held_close(code, scales, x, off, tall=1, what=""):
    """codes and scales (of weights, or of rows cut to [blocks, rows]) are those of x, of which the kernel knew values that were `off` away (a
    tensor or number).  The scale is a product with 1 / 448: the constant off by 0.38 x 2^-23, the product by 2^-24, 0.88 x 2^-23 together, for which
    2^-23 is allowed.  The code is a product with the reciprocal of the scale that is given here: 2^-23 and 2^-24, for which 2^-22 is allowed; behind
    them a rounding of half a step of e4m3.  (What a norm multiplies by beforehand is part of `off`.)"""
    rows, K = x.shape
    x = x.double()
    off = torch.as_tensor(off, dtype=torch.float64, device=x.device).expand(x.shape)
    scale = scales.double() if tall > 1 else scales.double().t()
    want, slack = largest(x, tall).clamp(min=LEAST) / 448, largest(off, tall) / 448
    bad = (scale - want).abs() > slack + want * 2.0 ** -23
    assert not bad.any(), f"{what}: {int(bad.sum())} scales of {bad.numel()} off"
    s = spread(scale, rows, K, tall)
    r, c = x / s, code.double()
    tol = half_step(torch.maximum(r.abs() + off / s, c.abs())) + off / s + r.abs() * 2.0 ** -22
    bad = (c - r).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} codes of {bad.numel()} off, worst {((c - r).abs() / tol).max().item():.3g} of the tolerance"


def random_held(g, rows, K, tall, wild=False, device="cuda"):
    """random codes and scales; wild: scales that differ by up to 2^20"""
    code = torch.randn(rows, K, generator=g, device=device).mul(60).clamp(-448, 448).to(F8)
    shape = (blocks_of(rows), blocks_of(K)) if tall > 1 else (blocks_of(K), (rows + 3) // 4 * 4)
    s = torch.rand(shape, generator=g, device=device) + 0.5
    if wild:
        s = s * torch.exp2(torch.randint(-10, 11, shape, generator=g, device=device).float())
    return code, s


def product(a, a_scales, w, w_scales):
    """(sums, sums of magnitudes) in 64 bits"""
    x, y = values(a, a_scales), values(w, w_scales, 128)
    return x @ y.t(), x.abs() @ y.abs().t()


def product_off(size, K):
    """How far a kernel's fp32 sums may be: 128 products are exact in fp32 (two 4-bit mantissas) and are added with one rounding or cut of up to
    2^-23 of the sum of magnitudes each; the product of two scales, its product with the block's sum and the running total are rounded once a
    block, 2^-24 each, which with the order of parts of the reduction counts as three for each block."""
    return size * (128 + 3 * blocks_of(K) + 8) * 2.0 ** -23


def unit(sums, act):
    """the gated unit of sums whose columns are gate and up in turns of 128"""
    pairs = sums.view(sums.shape[0], -1, 2, 128)
    gate, up = pairs[:, :, 0].flatten(1), pairs[:, :, 1].flatten(1)
    if act == "silu":
        return gate * torch.sigmoid(gate) * up
    return torch.nn.functional.gelu(gate, approximate="tanh") * up


def unit_off(sums, off, act):
    """How far the unit may be where the sums are `off`: both units' slopes are below 1.13 in size, |act(g)| <= |g|.  Its own arithmetic: the
    exponential's argument t has a few roundings, 2^-22 of its size together, which the exponential turns into a share of its value, as t e^-t
    is below 1 / (1 - share) there; with the exponential's own 2^-21, the division's 2^-22 and the product's: 2^-19 (1 + |t|) of the value."""
    pairs = lambda v: v.view(v.shape[0], -1, 2, 128)
    gate, up = (pairs(sums)[:, :, i].flatten(1) for i in range(2))
    dg, du = (pairs(off)[:, :, i].flatten(1) for i in range(2))
    t = gate.abs() if act == "silu" else 1.5957691216057308 * (gate + 0.044715 * gate ** 3).abs()
    y = unit(sums, act).abs()
    return 1.13 * dg * (up.abs() + du) + gate.abs() * du + y * 2.0 ** -19 * (1 + t) + 1e-30


def tile_table(loads, room=None, device="cuda"):
    """the tiles of rows that are sorted by expert, as moe_route writes them, and their number"""
    first, tiles = 0, []
    for e, n in enumerate(loads):
        tiles += [[e, first + i, first + n, 0] for i in range(0, n, 128)]
        first += n
    room = room or first // 128 + len(loads)
    return (torch.tensor(tiles + [[0, 0, 0, 0]] * (room - len(tiles)), dtype=torch.int32, device=device).view(-1, 4),
            torch.tensor([len(tiles)], dtype=torch.int32, device=device))

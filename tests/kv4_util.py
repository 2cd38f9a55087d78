"""The 4-bit cache in plain 64-bit arithmetic: quantisation by search, pages byte by byte, attention over what they stand for."""

import torch

BF = torch.bfloat16
BS = 16
CODES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)
# scale bytes 0 .. 226: five bits of exponent, three of mantissa
SCALES = torch.tensor([(b % 8) * 2.0 ** -17 if b < 8 else (8 + b % 8) * 2.0 ** (b // 8 - 18) for b in range(227)], dtype=torch.float64)


def nearest_even(x, ladder):
    """index of the nearest entry of an ascending ladder, of two equally near ones the even one"""
    hi = torch.searchsorted(ladder, x).clamp(1, len(ladder) - 1)
    lo = hi - 1
    up, down = ladder[hi] - x, x - ladder[lo]
    return torch.where(up < down, hi, torch.where(up > down, lo, torch.where(hi % 2 == 0, hi, lo)))


def quantise(x):
    """codes [..., D] (0 .. 15) and scale bytes [..., D / 16] of values [..., D]"""
    g = x.double().unflatten(-1, (-1, 16))
    nan = torch.isnan(g).any(-1)
    most = torch.nan_to_num(g.abs(), nan=0.0, posinf=float("inf")).amax(-1)
    b = nearest_even((most / 6).clamp(max=10240.0), SCALES).clamp(min=1)
    r = (torch.nan_to_num(g.abs(), nan=0.0, posinf=1e300) / SCALES[b].unsqueeze(-1)).clamp(max=6.0)
    code = nearest_even(r, CODES) + 8 * torch.signbit(g).long()
    return code.flatten(-2), torch.where(nan, 255, b)


def dequantise(code, b):
    size = torch.where(b == 255, float("nan"), SCALES[b.clamp(max=226)])
    v = CODES[code % 8] * torch.where(code >= 8, -1.0, 1.0)
    return (v.unflatten(-1, (-1, 16)) * size.unsqueeze(-1)).flatten(-2)


def held(x):
    """what a row of values is held as"""
    return dequantise(*quantise(x))


def places(D):
    """[16][D / 16] byte offsets in a head's page: keys' codes (8 bytes of a group), scale, values' codes, scale"""
    out = ([], [], [], [])
    for token in range(16):
        t, j = token % 4, token // 4
        row = 2 * t + j % 2 + 8 * (j // 2)
        lines = ([], [], [], [])
        for p in range(D // 16):
            lane, deep = (row % 8) * 4, row // 8
            if D == 64:
                line = (row * 32 + p * 8, (lane + p) * 2 + deep, token * 32 + p * 8, (p * 4 + t) * 4 + j)
            elif D == 128:
                line = (row * 64 + p * 8, (lane + p // 2) * 4 + deep * 2 + p % 2, token * 64 + (p ^ (token // 2 % 2 * 4)) * 8, (p * 4 + t) * 4 + j)
            else:
                line = (row * 128 + ((p // 2) ^ (row % 2 * 4)) * 16 + p % 2 * 8, (lane + p % 8 // 2) * 8 + deep * 4 + p // 8 * 2 + p % 2,
                        token * 128 + ((p // 2) ^ (token % 4 * 2)) * 16 + p % 2 * 8, (p // 2 * 4 + t) * 8 + p % 2 * 4 + j)
            for part, at in zip(lines, line):
                part.append(at)
        for part, at in zip(out, lines):
            part.append(at)
    at = [torch.tensor(p) for p in out]
    return at[0], at[1] + 8 * D, at[2] + 9 * D, at[3] + 17 * D


def page_index(D):
    """[16, D / 2] bytes of codes, [16, D / 16] of scales, for keys and for values"""
    kc, ks, vc, vs = places(D)
    return [(c.unsqueeze(-1) + torch.arange(8)).flatten(-2) for c in (kc, vc)], [ks, vs]


def write_rows(cache, slots, k, v, D):
    """rows k, v [T, heads, D] into cache uint8 [blocks, heads, 18 D] (CPU); slots < 0 are left out"""
    codes_at, scales_at = page_index(D)
    for which, x in enumerate((k, v)):
        code, b = quantise(x)
        byte = (code[..., ::2] | (code[..., 1::2] << 4)).to(torch.uint8)
        for i, s in enumerate(slots.tolist()):
            if s >= 0:
                page = cache[s // 16]
                page[:, codes_at[which][s % 16]] = byte[i]
                page[:, scales_at[which][s % 16]] = b[i].to(torch.uint8)


def read_pages(pages, D):
    """keys and values fp64 [..., 16, D] of pages uint8 [..., 18 D] (CPU)"""
    codes_at, scales_at = page_index(D)
    out = []
    for which in range(2):
        byte = pages[..., codes_at[which].flatten()].unflatten(-1, (16, D // 2)).long()
        code = torch.stack([byte % 16, byte // 16], -1).flatten(-2)
        b = pages[..., scales_at[which].flatten()].unflatten(-1, (16, D // 16)).long()
        out.append(dequantise(code, torch.where(b > 226, 255, b)))
    return out


def make_cache(ctxs, n_kv, D, seed, fill=0xFF, spread=1.0):
    """(cache uint8 [blocks, n_kv, 18 D], table int32 [n, columns], [(k, v) fp64 [n_kv, ctx, D]]): scattered pages; bytes that no token has
    are `fill` (0xFF: scales that read as NaN)"""
    g = torch.Generator().manual_seed(seed)
    needs = [(c + 15) // 16 for c in ctxs]
    blocks = sum(needs) + 2
    perm = torch.randperm(blocks, generator=g).tolist()
    cache = torch.full((blocks, n_kv, 18 * D), fill, dtype=torch.uint8)
    table = torch.zeros(len(ctxs), max(needs + [1]), dtype=torch.int32)
    rows, at = [], 0
    for i, (c, need) in enumerate(zip(ctxs, needs)):
        pages = perm[at:at + need]
        at += need
        table[i, :need] = torch.tensor(pages, dtype=torch.int32)
        k, v = (spread * torch.randn(c, n_kv, D, generator=g) for _ in range(2))
        slots = torch.tensor([pages[j // 16] * 16 + j % 16 for j in range(c)], dtype=torch.long)
        write_rows(cache, slots, k.to(BF), v.to(BF), D)
        rows.append((held(k.to(BF)).transpose(0, 1), held(v.to(BF)).transpose(0, 1)))
    return cache, table, rows


def attention(q, k, v, positions, scale, cap=0.0, window=0):
    """q [T, n_q, D], k, v [n_kv, J, D] in 64 bits: outputs, sum_j p_j |v_j|, largest sum_d |q k| scale of a row's keys (each per row, head)"""
    T, n_q, D = q.shape
    n_kv, J, _ = k.shape
    G = n_q // n_kv
    qh = q.double().view(T, n_kv, G, D)
    s = torch.einsum("tngd,njd->tngj", qh, k) * scale
    size = torch.einsum("tngd,njd->tngj", qh.abs(), k.abs()) * abs(scale)
    if cap > 0:
        s = cap * torch.tanh(s / cap)
    j = torch.arange(J)
    seen = j[None] <= positions[:, None]
    if window > 0:
        seen &= j[None] > positions[:, None] - window
    seen = seen[:, None, None, :]
    s = s.masked_fill(~seen, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), 0.0, top))
    p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
    size = (size * seen).amax(-1)
    flat = lambda x: x.reshape(T, n_q, -1).squeeze(-1) if x.dim() == 3 else x.reshape(T, n_q, D)
    return flat(torch.einsum("tngj,njd->tngd", p, v)), flat(torch.einsum("tngj,njd->tngd", p, v.abs())), size.reshape(T, n_q)


def attention_close(got, ref, weight, size, D, p_half_step, what=""):
    """The output's rounding to bf16 (2^-8 of the value), a probability's rounding (p_half_step of sum p |v|), and the score's: D products
    summed in fp32, each sum off by at most 2^-23 of sum |q k|, to which the exponential's own 2^-21 come; numerator and sum both feel it."""
    got = got.double().cpu()
    assert torch.isfinite(got).all(), what
    tol = 2.0 ** -8 * ref.abs() + weight * (p_half_step + 2 * (D * 2.0 ** -23 * size.unsqueeze(-1) + 2.0 ** -21)) + 1e-30
    bad = (got - ref).abs() > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off; worst {((got - ref).abs() / tol).max().item():.3g} of the tolerance"


def rope_rows(qkv, cos_sin, positions, n_q, n_kv, D):
    """rotated q and k with a bf16 rounding behind every operation, v; each [T, heads, D] (64 bits)"""
    T = qkv.shape[0]
    x = qkv.view(T, n_q + 2 * n_kv, D).double()
    cs = cos_sin[positions.long()].double().unsqueeze(1)
    c, s = cs[..., : D // 2], cs[..., D // 2:]
    r = lambda v: v.float().to(BF).double()
    a, b = x[:, : n_q + n_kv, : D // 2], x[:, : n_q + n_kv, D // 2:]
    y = torch.cat([r(r(a * c) - r(b * s)), r(r(b * c) + r(a * s))], -1)
    return y[:, :n_q], y[:, n_q:], x[:, n_q + n_kv:]



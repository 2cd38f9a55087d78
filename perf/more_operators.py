"""Linear layers in 8 bits with a scale for each block of 128: what the operators cost and what they compute.

A worker that serves a model whose weights are held in 8 bits does in every layer: normalise the residual stream and hand it on in 8 bits,
multiply it by the fused query / key / value matrix, quantise what attention gives and multiply that by the output matrix, normalise again, one
product for gate and up whose unit leaves in 8 bits again, and the product down.  Experts do the last two over rows that are sorted by expert.
Weights are quantised once, when they are loaded.

A value in 8 bits is e4m3 (sign, four bits of exponent, three of mantissa, up to 448) times an fp32 scale.  Activations [T, K] have one scale for
each 128 neighbouring values of a row, laid out [ceil(K / 128), rows]; weights [N, K] one for each square of 128 x 128, [ceil(N / 128), ceil(K / 128)].
A scale is a 448th of its block's largest magnitude.

All tensors are made on the GPU from the seed: activations are unit normal, weights normal with a deviation of K^-1/2."""
import math
import random

import torch

own = False   # set from outside: True runs the framework's operators, False the plain forms

BF, F8 = torch.bfloat16, torch.float8_e4m3fn
BLOCK = 128
EPS = 1e-5
#           columns of the output, length of the reduction
PRODUCTS = {"llama-3-8b qkv": (6144, 4096), "llama-3-8b o": (4096, 4096), "llama-3-8b down": (4096, 14336), "llama-3.2-1b o": (2048, 2048),
            "llama-3.2-1b down": (2048, 8192), "gemma-2-9b qkv": (8192, 3584), "gemma-2-9b o": (3584, 4096), "gemma-2-9b down": (3584, 14336),
            "gemma-2-2b qkv": (4096, 2304), "gemma-2-2b down": (2304, 9216)}
#        gate and up together, length of the reduction, unit
GATED = {"llama-3-8b": (28672, 4096, "silu"), "llama-3.2-1b": (16384, 2048, "silu"), "gemma-2-9b": (28672, 3584, "gelu"),
         "gemma-2-2b": (18432, 2304, "gelu")}
#          width, an expert's inner size, experts, how many of them a token goes to
EXPERTS = {"fimilorn-1b": (2048, 1024, 16, 4), "noridra-1b": (2048, 1024, 16, 4), "wide": (4096, 1536, 64, 6)}


def listed():
    return [
        # one token of the small model: the smallest call there is
        {"name": "norm 1b 1 row", "kind": "norm", "rows": 1, "width": 2048, "dtype": "bf16"},
        # a full step of prompts
        {"name": "norm 8b 4608 rows", "kind": "norm", "rows": 4608, "width": 4096, "dtype": "bf16"},
        # tokens of a step sorted by expert, four times each
        {"name": "rows 1001 x 4 sorted", "kind": "rows", "rows": 4004, "width": 2048, "tokens": 1001, "dtype": "bf16"},
        # the largest matrix of a layer when the weights are loaded
        {"name": "weights 8b gate up", "kind": "weights", "columns": 28672, "width": 4096, "dtype": "bf16"},
        # one user
        {"name": "product 8b o 1 row", "kind": "product", "matrix": "llama-3-8b o", "rows": 1},
        # a decode step of a small batch
        {"name": "product 8b down 48 rows", "kind": "product", "matrix": "llama-3-8b down", "rows": 48},
        # a ragged step of the translation model
        {"name": "product 9b qkv 1001 rows", "kind": "product", "matrix": "gemma-2-9b qkv", "rows": 1001},
        # a full step of prompts
        {"name": "product 8b down 4608 rows", "kind": "product", "matrix": "llama-3-8b down", "rows": 4608},
        # a decode step of a handful of sequences on the small model
        {"name": "gated 1b 7 rows", "kind": "gated", "model": "llama-3.2-1b", "rows": 7},
        # a full step of prompts: the largest product of a layer
        {"name": "gated 8b 4608 rows", "kind": "gated", "model": "llama-3-8b", "rows": 4608},
        # a decode step of routed experts
        {"name": "experts gate up 64", "kind": "experts", "model": "fimilorn-1b", "tokens": 64, "gated": True},
        # a step of prompts over many experts of uneven loads
        {"name": "experts down 4096", "kind": "experts", "model": "wide", "tokens": 4096, "gated": False},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("norm", "rows", "weights", "product", "product", "product", "gated", "gated", "experts", "experts"))
    if kind in ("norm", "rows"):
        case = {"kind": kind, "rows": _log(rng, 1, 4608), "width": 16 * _log(rng, 8, 512), "dtype": rng.choice(("bf16", "bf16", "f32"))}
        return {**case, "tokens": _log(rng, 1, case["rows"])} if kind == "rows" else case
    if kind == "weights":
        return {"kind": kind, "columns": 8 * _log(rng, 16, 3584), "width": 16 * _log(rng, 8, 256), "dtype": rng.choice(("bf16", "f32"))}
    if kind == "product":
        return {"kind": kind, "matrix": rng.choice(tuple(PRODUCTS)), "rows": _log(rng, 1, 4608)}
    if kind == "gated":
        return {"kind": kind, "model": rng.choice(tuple(GATED)), "rows": _log(rng, 1, 4608)}
    return {"kind": kind, "model": rng.choice(tuple(EXPERTS)), "tokens": _log(rng, 1, 4096), "gated": rng.random() < 0.5}


# ---- inputs --------------------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape, dtype=BF, by=1.0):
    return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * by).to(dtype)


def _type(case):
    return BF if case["dtype"] == "bf16" else torch.float32


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def _padded(x, rows, columns):
    """x with zeros behind its last row and column"""
    out = torch.zeros(rows, columns, dtype=x.dtype, device=x.device)
    out[: x.shape[0], : x.shape[1]] = x
    return out


def _scales(rows, K):
    """room for the scales of `rows` rows of K values: [ceil(K / 128), rows rounded up to 4]"""
    return torch.zeros(_blocks(K), (rows + 3) // 4 * 4, device="cuda")


def _held(x, tall):
    """codes and scales of a matrix in blocks of `tall` x 128; scales [blocks down, blocks across]"""
    rows, K = x.shape
    p = _padded(x.float(), (rows + tall - 1) // tall * tall, _blocks(K) * BLOCK).view(-1, tall, _blocks(K), BLOCK)
    scale = p.abs().amax((1, 3)).clamp(min=2.0 ** -100) / 448.0
    code = (p / scale[:, None, :, None]).to(F8)
    return code.view(-1, _blocks(K) * BLOCK)[:rows, :K].contiguous(), scale


def _activations(g, rows, K):
    code, scale = _held(_normal(g, rows, K), 1)
    out = _scales(rows, K)
    out[:, :rows] = scale.t()
    return code, out


def _loads(case):
    """rows of each expert: uneven, some without any where tokens are few; the case alone decides"""
    _, _, E, top = EXPERTS[case["model"]]
    r, count = random.Random(case["tokens"]), [0] * E
    liked = [1.0 + 3.0 * (e % 5 == 0) for e in range(E)]
    for _ in range(case["tokens"]):
        left = list(range(E))
        for _ in range(top):
            e = r.choices(left, [liked[i] for i in left])[0]
            left.remove(e)
            count[e] += 1
    return count


def prepare(case, seed):
    k, g, st = case["kind"], _gen(seed), {"case": case}
    if k in ("norm", "rows"):
        T, H = case["rows"], case["width"]
        st["x"] = _normal(g, case.get("tokens", T), H, dtype=_type(case))
        if k == "norm":
            st["residual"] = _normal(g, T, H, dtype=_type(case), by=3.0)
            st["w"] = (1.0 + 0.2 * _normal(g, H, dtype=torch.float32)).to(_type(case))
        else:
            st["at"] = torch.randint(0, case["tokens"], (T,), generator=g, device="cuda").to(torch.int32)
        st["y"], st["scales"] = torch.empty(T, H, dtype=F8, device="cuda"), _scales(T, H)
        st["told"] = st["scales"][:, :T]
    elif k == "weights":
        N, K = case["columns"], case["width"]
        st["w"] = _normal(g, N, K, dtype=_type(case), by=K ** -0.5)
        st["y"], st["told"] = torch.empty(N, K, dtype=F8, device="cuda"), torch.empty(_blocks(N), _blocks(K), device="cuda")
    elif k in ("product", "gated"):
        T = case["rows"]
        N, K = (PRODUCTS[case["matrix"]] if k == "product" else GATED[case["model"]])[:2]
        st["a"], st["as"] = _activations(g, T, K)
        st["w"], st["ws"] = _held(_normal(g, N, K, by=K ** -0.5), BLOCK)
        if k == "product":
            st["c"] = torch.empty(T, N, dtype=BF, device="cuda")
        else:   # (rows of gate and up in turns of 128, as the 16-bit product has them)
            st["act"] = GATED[case["model"]][2]
            st["y"], st["ys"] = torch.empty(T, N // 2, dtype=F8, device="cuda"), _scales(T, N // 2)
            st["told"] = st["ys"][:, :T]
    else:
        width, inner, E, top = EXPERTS[case["model"]]
        N, K = (2 * inner, width) if case["gated"] else (width, inner)
        loads = _loads(case)
        T = sum(loads)
        st["a"], st["as"] = _activations(g, T, K)
        w, ws = _held(_normal(g, E * N, K, by=K ** -0.5), BLOCK)
        st["w"], st["ws"] = w.view(E, N, K), ws.view(E, N // BLOCK, K // BLOCK)
        first, tiles = 0, []
        for e, n in enumerate(loads):   # the router's table of tiles: {expert, first row, end of the expert's rows, 0}
            tiles += [[e, first + i, first + n, 0] for i in range(0, n, 128)]
            first += n
        room = T // 128 + E
        st["tiles"] = torch.tensor(tiles + [[0, 0, 0, 0]] * (room - len(tiles)), dtype=torch.int32, device="cuda")
        st["n_tiles"] = torch.tensor([len(tiles)], dtype=torch.int32, device="cuda")
        st["expert"] = torch.cat([torch.full((n,), e) for e, n in enumerate(loads)]).cuda()
        st["loads"] = loads
        if case["gated"]:
            st["act"] = "silu"
            st["y"], st["ys"] = torch.empty(T, inner, dtype=F8, device="cuda"), _scales(T, inner)
            st["told"] = st["ys"][:, :T]
        else:
            st["c"] = torch.empty(T, N, dtype=BF, device="cuda")
    return st


# ---- one pass --------------------------------------------------------------------------------------------------------------
def _quantised(x):
    """codes and scales [blocks, rows] of fp32 rows"""
    code, scale = _held(x, 1)
    return {"y": code, "scales": scale.t()}


def _values(code, scale, tall):
    """what codes [rows, K] stand for, scales [blocks down, blocks across]"""
    rows, K = code.shape
    return code.float() * scale.repeat_interleave(tall, 0)[:rows].repeat_interleave(BLOCK, 1)[:, :K]


def _unit(x, act):
    """the gated unit of sums whose columns are gate and up in turns of 128"""
    pairs = x.view(x.shape[0], -1, 2, BLOCK)
    gate, up = pairs[:, :, 0].flatten(1), pairs[:, :, 1].flatten(1)
    if act == "silu":
        return gate / (1.0 + torch.exp(-gate)) * up
    return 0.5 * gate * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (gate + 0.044715 * gate * gate * gate))) * up


def _norm(st):
    x, r = st["x"].float(), st["residual"]
    r.copy_(x + r.float())
    v = r.float()
    inv = 1.0 / torch.sqrt((v * v).mean(-1, keepdim=True) + EPS)
    return {**_quantised(v * inv * st["w"].float()), "residual": r}


def _experts(st):
    """every expert's product over all rows of the largest load: rows that it has not are zeros"""
    E, N, K = st["w"].shape
    a = _values(st["a"], st["as"][:, : st["a"].shape[0]].t(), 1)
    most = max(st["loads"])
    first = torch.cumsum(torch.tensor([0] + st["loads"][:-1], device=a.device), 0)
    place = torch.arange(a.shape[0], device=a.device) - first[st["expert"]]
    by_expert = torch.zeros(E, most, K, device=a.device)
    by_expert[st["expert"], place] = a
    w = _values(st["w"].view(E * N, K), st["ws"].view(-1, K // BLOCK), BLOCK).view(E, N, K)
    return torch.matmul(by_expert, w.transpose(1, 2))[st["expert"], place]


def run(st):
    k = st["case"]["kind"]
    if own:
        return _run_own(st, k)
    if k == "norm":
        return _norm(st)
    if k == "rows":
        return _quantised(st["x"].float()[st["at"].long()])
    if k == "weights":
        code, scale = _held(st["w"], BLOCK)
        return {"y": code, "scales": scale}
    if k == "experts":
        sums = _experts(st)
    else:
        a = _values(st["a"], st["as"][:, : st["a"].shape[0]].t(), 1)
        sums = torch.matmul(a, _values(st["w"], st["ws"], BLOCK).t())
    return _quantised(_unit(sums, st["act"])) if "act" in st else sums.to(BF)


def _run_own(st, k):
    from llmq_b200 import lib as L

    if k == "norm":
        L.rmsnorm_fp8(st["x"], st["w"], st["y"], st["scales"], EPS, residual=st["residual"])
        return {"y": st["y"], "scales": st["told"], "residual": st["residual"]}
    if k == "rows":
        L.quantize_fp8(st["x"], st["y"], st["scales"], rows=st["at"])
    elif k == "weights":
        L.quantize_fp8_weight(st["w"], st["y"], st["told"])
    elif k == "product":
        L.gemm_fp8(st["a"], st["as"], st["w"], st["ws"], st["c"])
        return st["c"]
    elif k == "gated":
        L.gemm_gated_fp8(st["a"], st["as"], st["w"], st["ws"], st["y"], st["ys"], st["act"])
    elif st["case"]["gated"]:
        L.gemm_grouped_gated_fp8(st["a"], st["as"], st["w"], st["ws"], st["y"], st["ys"], st["tiles"], st["n_tiles"], st["act"])
    else:
        L.gemm_grouped_fp8(st["a"], st["as"], st["w"], st["ws"], st["c"], st["tiles"], st["n_tiles"])
        return st["c"]
    return {"y": st["y"], "scales": st["told"]}


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------
def _bytes8(rows, K, tall=1):
    return rows * K + 4.0 * ((rows + tall - 1) // tall) * _blocks(K)


def work(case):
    k = case["kind"]
    if k in ("norm", "rows"):
        size, T, H = 2 if case["dtype"] == "bf16" else 4, case["rows"], case["width"]
        if k == "norm":
            return {"bytes": 3.0 * size * T * H + size * H + _bytes8(T, H), "flops": 8.0 * T * H}
        return {"bytes": 1.0 * size * min(T, case["tokens"]) * H + 4.0 * T + _bytes8(T, H), "flops": 3.0 * T * H}
    if k == "weights":
        N, K = case["columns"], case["width"]
        return {"bytes": (2.0 if case["dtype"] == "bf16" else 4.0) * N * K + _bytes8(N, K, BLOCK), "flops": 3.0 * N * K}
    if k == "experts":
        width, inner, E, top = EXPERTS[case["model"]]
        N, K = (2 * inner, width) if case["gated"] else (width, inner)
        T, used, gated = case["tokens"] * top, sum(n > 0 for n in _loads(case)), case["gated"]
    else:
        T, used, gated = case["rows"], 1, k == "gated"
        N, K = (GATED[case["model"]] if gated else PRODUCTS[case["matrix"]])[:2]
    out = _bytes8(T, N // 2) if gated else 2.0 * T * N
    return {"bytes": _bytes8(T, K) + used * _bytes8(N, K, BLOCK) + out, "flops": 2.0 * T * N * K}


# ---- the definition, in 64 bits -----------------------------------------------------------------------------------------
def _nearest(r):
    """the nearest e4m3 number, of two equally near ones the one with an even mantissa; |r| up to 448"""
    low = [m * 2.0 ** -9 for m in range(8)]
    ladder = torch.tensor(low + [(8 + m) * 2.0 ** (e - 10) for e in range(1, 16) for m in range(8)][:-1], dtype=torch.float64, device=r.device)
    middle = (ladder[1:] + ladder[:-1]) / 2
    out = torch.empty_like(r)
    for at in range(0, r.shape[0], 4096):
        size = r[at: at + 4096].abs()
        a, b = torch.searchsorted(middle, size, right=False), torch.searchsorted(middle, size, right=True)
        out[at: at + 4096] = ladder[torch.where(a % 2 == 0, a, b)] * torch.sign(r[at: at + 4096])
    return out


def _exact_blocks(x, tall):
    """(values of the codes, scales) of rows in 64 bits, block by block of 128 columns"""
    codes, scales = [], []
    for at in range(0, x.shape[1], BLOCK):
        part = x[:, at: at + BLOCK]
        most = part.abs().amax(1)
        if tall > 1:
            most = torch.stack([piece.max() for piece in most.split(tall)])
        scale = most.clamp(min=2.0 ** -100) / 448
        scales.append(scale)
        by = scale if tall == 1 else scale.repeat_interleave(tall)[: x.shape[0]]
        codes.append(_nearest(part / by[:, None]))
    return torch.cat(codes, 1), torch.stack(scales)


def _exact_product(a, a_scales, w, w_scales):
    """[rows, N] sums in 64 bits, a block of 128 of the reduction at a time"""
    out = torch.zeros(a.shape[0], w.shape[0], dtype=torch.float64, device=a.device)
    for b in range(w_scales.shape[1]):
        part = slice(b * BLOCK, (b + 1) * BLOCK)
        down = w_scales[:, b].double().repeat_interleave(BLOCK)[: w.shape[0]]
        out += (a[:, part].double() @ w[:, part].double().t()) * a_scales[b, : a.shape[0], None].double() * down
    return out


def _exact_unit(sums, act):
    gate = torch.cat([sums[:, i: i + BLOCK] for i in range(0, sums.shape[1], 2 * BLOCK)], 1)
    up = torch.cat([sums[:, i: i + BLOCK] for i in range(BLOCK, sums.shape[1], 2 * BLOCK)], 1)
    if act == "silu":
        value = gate * torch.sigmoid(gate) * up
    else:
        value = torch.nn.functional.gelu(gate, approximate="tanh") * up
    code, scale = _exact_blocks(value, 1)
    return {"y": code, "scales": scale}


def exact(case, seed):
    k, st = case["kind"], prepare(case, seed)
    if k == "norm":
        v = (st["x"].double() + st["residual"].double()).to(_type(case)).double()   # (the residual stream is held in its own type)
        y, scale = _exact_blocks(v * torch.rsqrt(v.square().mean(1, keepdim=True) + EPS) * st["w"].double(), 1)
        return {"y": y, "scales": scale, "residual": v}
    if k in ("rows", "weights"):
        y, scale = _exact_blocks(st["x"][st["at"].long()].double() if k == "rows" else st["w"].double(), 1 if k == "rows" else BLOCK)
        return {"y": y, "scales": scale if k == "rows" else scale.t()}
    if k == "experts":
        out, at = [], 0
        for e, n in enumerate(st["loads"]):
            if n:
                out.append(_exact_product(st["a"][at: at + n], st["as"][:, at: at + n], st["w"][e], st["ws"][e]))
            at += n
        sums = torch.cat(out)
    else:
        sums = _exact_product(st["a"], st["as"], st["w"], st["ws"])
    return _exact_unit(sums, st["act"]) if "act" in st else sums

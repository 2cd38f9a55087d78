"""Decoding with beams over a paged cache that is held in 4 bits: what the operators cost and what they compute.

A worker that searches with beams does in every step: choose the best continuations of each sequence, give every beam the pages of
its parent and one of its own to write to, rotate the new queries and keys and put keys and values into their pages, and attend over
the pages.  Prompts come as portions; now and then the pages in use are moved together so that memory behind them can be given back.

The cache.  Sixteen neighbouring values of a head share a scale of eight bits, five of exponent and three of mantissa (the upper byte
of a half without its sign); a value is sign, two bits of exponent and one of mantissa: 0, .5, 1, 1.5, 2, 3, 4, 6 times the scale.  A
page holds 16 tokens of one layer, per head the keys' codes, their scales, the values' codes, their scales.  Where each lies in its part
is what `places` computes.

All tensors are made on the GPU from the seed: activations and cached rows are unit normal, pages are scattered, contexts are ragged."""
import math
import random

import torch

own = False   # set from outside: True runs the framework's operators, False the plain forms

PAGE = 16
BF = torch.bfloat16
#         layers, query heads, heads, head size, scale, soft cap, window, rotation base, vocabulary
MODELS = {"llama-3-8b": (32, 32, 8, 128, 128 ** -0.5, 0.0, 0, 500000.0, 128256),
          "llama-3.2-1b": (16, 32, 8, 64, 64 ** -0.5, 0.0, 0, 500000.0, 128256),
          "gemma-2-9b": (42, 16, 8, 256, 256 ** -0.5, 50.0, 4096, 10000.0, 256000),
          "gemma-2-2b": (26, 8, 4, 256, 256 ** -0.5, 50.0, 4096, 10000.0, 256000)}


def listed():
    return [
        # a decode step of a handful of sequences on the small model: the smallest call there is
        {"name": "write 1b 7 rows", "kind": "write", "model": "llama-3.2-1b", "rows": 7, "together": False},
        # a full step of prompts: rows of one sequence behind each other
        {"name": "write 8b 4608 rows", "kind": "write", "model": "llama-3-8b", "rows": 4608, "together": True},
        # three users with long documents on the small model
        {"name": "decode 1b 3 long seqs", "kind": "decode", "model": "llama-3.2-1b", "seqs": 3, "lo": 9001, "hi": 16001},
        # a large ragged batch
        {"name": "decode 8b 700 seqs", "kind": "decode", "model": "llama-3-8b", "seqs": 700, "lo": 33, "hi": 1000},
        # a step of ragged prompts
        {"name": "prompts 8b 9 ragged", "kind": "prompt", "model": "llama-3-8b", "prompts": 9, "lo": 65, "hi": 1021, "past": 0},
        # later portions of two long prompts on the translation model: large heads, soft cap, sliding window, an odd number of keys before
        {"name": "prompts gemma 9b 2 long", "kind": "prompt", "model": "gemma-2-9b", "prompts": 2, "lo": 1500, "hi": 3001, "past": 1111},
        # one sentence with the usual four beams
        {"name": "beams 1 x 4", "kind": "beam", "vocab": 128256, "groups": 1, "beams": 4, "stops": 1},
        # a batch of translations over the translation model's vocabulary
        {"name": "beams 48 x 8 gemma", "kind": "beam", "vocab": 256000, "groups": 48, "beams": 8, "stops": 2},
        # the pages of one search with five beams
        {"name": "fork 1 x 5", "kind": "fork", "model": "llama-3.2-1b", "layers": 16, "groups": 1, "beams": 5, "lo": 77, "hi": 77},
        # the pages of a batch of searches
        {"name": "fork 24 x 6", "kind": "fork", "model": "llama-3-8b", "layers": 16, "groups": 24, "beams": 6, "lo": 50, "hi": 900},
        # a small pool, half empty after its sequences ended in any order
        {"name": "compact 300 pages", "kind": "compact", "model": "llama-3.2-1b", "layers": 4, "pages": 300, "live": 0.4, "hi": 200},
        # a large pool of which little is in use
        {"name": "compact 20000 pages", "kind": "compact", "model": "llama-3-8b", "layers": 2, "pages": 20000, "live": 0.3, "hi": 1500},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(("write", "decode", "decode", "decode", "prompt", "prompt", "beam", "beam", "fork", "compact"))
    model = rng.choice(tuple(MODELS))
    layers, n_q, n_kv, D = MODELS[model][:4]
    if kind == "write":
        return {"kind": kind, "model": model, "rows": _log(rng, 1, 4608), "together": rng.random() < 0.5}
    if kind == "decode":
        hi = _log(rng, 48, 16000)
        most = int(0.6e9 / (n_kv * D * hi))
        return {"kind": kind, "model": model, "seqs": _log(rng, 1, max(2, min(4608, most))), "lo": rng.randint(1, hi), "hi": hi}
    if kind == "prompt":
        hi = _log(rng, 8, 3000)
        return {"kind": kind, "model": model, "prompts": _log(rng, 1, max(1, 6000 // hi)), "lo": rng.randint(max(1, hi // 4), hi), "hi": hi,
                "past": rng.choice((0, 0, rng.randint(1, 1500)))}
    if kind == "beam":
        beams, vocab = rng.choice((1, 2, 3, 4, 5, 8, 12)), rng.choice((32000, 50257, 128256, 256000))
        return {"kind": kind, "vocab": vocab, "groups": _log(rng, 1, max(1, min(64, int(9e7 / (vocab * beams))))), "beams": beams,
                "stops": rng.randint(0, 2)}
    hi = _log(rng, 20, 1200)
    if kind == "fork":
        return {"kind": kind, "model": model, "layers": rng.randint(2, 12), "groups": _log(rng, 1, max(1, 9000 // hi)), "beams": rng.randint(2, 8),
                "lo": rng.randint(1, hi), "hi": hi}
    pages = _log(rng, 40, 9000)
    return {"kind": kind, "model": model, "layers": rng.randint(1, 2), "pages": pages, "live": rng.uniform(0.1, 0.9), "hi": min(hi, 2 * pages)}


# ---- the layout of a page ----------------------------------------------------------------------------------------------------
def places(D):
    """where a page of one head (18 D bytes) has what belongs to token i and value d of it, as [16, D] tables: the byte of a key's code, of its
    scale, of a value's code, of its scale.  A byte holds two neighbouring codes, the even one in its lower half."""
    i, d = torch.arange(16).view(16, 1).expand(16, D), torch.arange(D).view(1, D).expand(16, D)
    t, j = i % 4, i // 4                                  # token i = t + 4 j
    row = 2 * t + (j & 1) + 8 * (j >> 1)                  # keys: tokens are rows of a matrix product's tile in this order
    group, byte = d // 16, d // 2
    if D == 256:
        kc = row * 128 + ((byte // 16) ^ ((row & 1) * 4)) * 16 + byte % 16
        vc = i * 128 + ((byte // 16) ^ ((i & 3) * 2)) * 16 + byte % 16
    elif D == 128:
        kc = row * 64 + byte
        vc = i * 64 + ((byte // 8) ^ (((i >> 1) & 1) * 4)) * 8 + byte % 8
    else:
        kc, vc = row * 32 + byte, i * 32 + byte
    if D == 256:
        ks = ((row & 7) * 4 + group % 8 // 2) * 8 + (row >> 3) * 4 + group // 8 * 2 + group % 2
        vs = (group // 2 * 4 + t) * 8 + group % 2 * 4 + j
    elif D == 128:
        ks = ((row & 7) * 4 + group // 2) * 4 + (row >> 3) * 2 + group % 2
        vs = (group * 4 + t) * 4 + j
    else:
        ks = ((row & 7) * 4 + group) * 2 + (row >> 3)
        vs = (group * 4 + t) * 4 + j
    return kc, 8 * D + ks, 9 * D + vc, 17 * D + vs


def _values(pages, code_at, scale_at, D):
    """what the codes and scales at these places of pages [..., 18 D] stand for, fp32 [..., 16, D]"""
    byte = pages[..., code_at.reshape(-1)]
    odd = (torch.arange(D, device=pages.device) % 2).repeat(16).bool()
    code = torch.where(odd, byte >> 4, byte & 15).to(torch.int16)
    value = (((code & 8) << 12) | ((code & 7) << 9)).view(torch.float16).float() * 16384.0
    scale = (pages[..., scale_at.reshape(-1)].to(torch.int16) << 7).view(torch.float16).float()
    return (value * scale).view(*pages.shape[:-1], 16, D)


def _codes(x):
    """codes and scale bytes of groups of 16 along the last axis of x (values of a 16-bit float): uint8 [..., D], uint8 [..., D / 16].  In 64
    bits: borders between two codes are met exactly by many values."""
    g = x.double().unflatten(-1, (-1, 16))
    want = g.abs().amax(-1, keepdim=True) / torch.full((), 6.0, dtype=torch.float64, device=x.device)
    step = torch.exp2((torch.frexp(want)[1] - 4).clamp(min=-17).double())
    scale = (torch.round(want / step) * step).clamp(2.0 ** -17, 10240.0)
    r = g.abs() / scale
    code = ((r > 0.25).to(torch.uint8) + (r >= 0.75) + (r > 1.25) + (r >= 1.75) + (r > 2.5) + (r >= 3.5) + (r > 5.0)).to(torch.uint8)
    code = code | (torch.signbit(g).to(torch.uint8) << 3)
    bits = scale.squeeze(-1).to(torch.float16).view(torch.int16) >> 7
    return code.flatten(-2), bits.to(torch.uint8)


def _pages_of(k, v, at, D):
    """pages [..., 18 D] of keys and values [..., 16, D]"""
    out = torch.zeros(*k.shape[:-2], 18 * D, dtype=torch.uint8, device=k.device)
    for x, code_at, scale_at in ((k, at[0], at[1]), (v, at[2], at[3])):
        code, scale = _codes(x)
        out[..., code_at[:, ::2].reshape(-1)] = (code[..., ::2] | (code[..., 1::2] << 4)).flatten(-2)
        out[..., scale_at[:, ::16].reshape(-1)] = scale.flatten(-2)
    return out


# ---- inputs --------------------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _normal(g, *shape, dtype=BF):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(dtype)


def _lengths(n, lo, hi, seed):
    """n lengths spread evenly over [lo, hi], in any order"""
    lens = [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]
    random.Random(int(seed)).shuffle(lens)
    return lens


def _fork_lengths(case):
    """(passes do not make the sequences longer, so a page that a pass began would be given back by none: no length ends with its page)"""
    return [n - (n % PAGE == 0) for n in _lengths(case["groups"], case["lo"], case["hi"], 0)]


def _table(g, needs):
    """a block table over a scattered pool: int32 [n, columns], pages of the pool"""
    total, columns = sum(needs) + 3, max(needs)
    perm = torch.randperm(total, generator=g, device="cuda").to(torch.int32).tolist()
    rows, at = [], 0
    for k in needs:
        rows.append(perm[at:at + k] + [0] * (columns - k))
        at += k
    return torch.tensor(rows, dtype=torch.int32, device="cuda"), total


def _cache4(g, blocks, n_kv, D, at):
    """a layer's pages, uint8 [blocks, n_kv, 18 D]: 256 pages of normal rows, each at many places"""
    base = _pages_of(_normal(g, 256, 16, D), _normal(g, 256, 16, D), at, D)
    return base[torch.randint(0, 256, (blocks, n_kv), generator=g, device="cuda")]


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    k, g, st = case["kind"], _gen(seed), {"case": case}
    if k in ("write", "decode", "prompt"):
        _, n_q, n_kv, D, scale, cap, window, base, _ = MODELS[case["model"]]
        st["at"] = at = [p.cuda() for p in places(D)]
        st["heads"] = (n_q, n_kv, D)
    if k == "write":
        T = case["rows"]
        st["qkv"] = _normal(g, T, (n_q + 2 * n_kv) * D)
        pos = list(range(T)) if case["together"] else _lengths(T, 5, 8000, seed)
        angle = torch.outer(torch.arange(max(8001, T), device="cuda").float(), base ** (-torch.arange(0, D, 2, device="cuda").float() / D))
        st["cos_sin"] = torch.cat([angle.cos(), angle.sin()], -1).to(BF)
        blocks = (T + 15) // 16 if case["together"] else T
        page = torch.randperm(blocks, generator=g, device="cuda").tolist()
        slots = [page[i // 16] * 16 + i % 16 for i in range(T)] if case["together"] else [page[i] * 16 + pos[i] % 16 for i in range(T)]
        st["pos"], st["slots"], st["pages"] = _ints(pos), _ints(slots), _ints(sorted(page))
        st["kv"] = _cache4(g, blocks, n_kv, D, at)
        st["back"] = torch.empty(blocks, 2, n_kv, PAGE, D, dtype=BF, device="cuda")
    elif k in ("decode", "prompt"):
        past = case.get("past", 0)
        lens = _lengths(case["seqs"] if k == "decode" else case["prompts"], case["lo"], case["hi"], seed)
        st["lens"] = lens
        st["bt"], blocks = _table(g, [(past + n + PAGE - 1) // PAGE for n in lens])
        st["kv"] = _cache4(g, blocks, n_kv, D, at)
        T = len(lens)
        if k == "decode":
            st["ctx"] = _ints(lens)
        else:
            tiles, T = [], 0
            for i, n in enumerate(lens):
                tiles += [[i, T + j, min(16, n - j), past + j] for j in range(0, n, 16)]
                T += n
            st["tiles"] = _ints(tiles)
            own_row = torch.cat([torch.full((n,), i) for i, n in enumerate(lens)])
            st["row"], st["pos"] = own_row.cuda(), torch.cat([torch.arange(n) for n in lens]).cuda()
            blocks_of = st["bt"].shape[0] * st["bt"].shape[1]   # the 16-bit pages that a portion's keys are spread out to, and a few bytes
            st["work"] = torch.empty(blocks_of * (4 * n_kv * PAGE * D + 4) + 4096, dtype=torch.uint8, device="cuda")
        st["qkv"] = _normal(g, T, (n_q + 2 * n_kv) * D)
        st["out"] = torch.empty(T, n_q * D, dtype=BF, device="cuda")
        st["scale"], st["cap"], st["window"] = scale, cap, window
    elif k == "beam":
        B, W, V = case["groups"], case["beams"], case["vocab"]
        st["logits"] = torch.empty(B * W, V, dtype=BF, device="cuda").normal_(0.0, 2.5, generator=g)
        st["scores"] = -torch.rand(B * W, generator=g, device="cuda") * 3.0 - 10.0
        st["stops"] = torch.randperm(V, generator=g, device="cuda")[: case["stops"]].to(torch.int32)
        if case["stops"]:   # (some sentences end here)
            st["logits"][::5, st["stops"][0].long()] = 14.0
        i32 = dict(dtype=torch.int32, device="cuda")
        K = 2 * W
        st["cand"] = (torch.empty(B, K, device="cuda"), torch.empty(B, K, **i32), torch.empty(B, K, **i32))
        st["work"] = torch.empty(B * W * (V // 2048 + 2) * (16 + 8 * K), dtype=torch.uint8, device="cuda")   # (what pieces of the rows have found)
        st["next"] = (torch.empty(B, W, device="cuda"), torch.empty(B, W, **i32), torch.empty(B, W, **i32))
    else:
        _, _, n_kv, D = MODELS[case["model"]][:4]
        r, fixed = random.Random(int(seed)), random.Random(0)   # (how much there is follows from the case alone, where it lies from the seed)
        groups, held = [], 0
        if k == "fork":
            B, W = case["groups"], case["beams"]
            for n in _fork_lengths(case):   # a group's beams share pages up to some place, and hold the rest themselves
                pages = (n + PAGE - 1) // PAGE
                shared = max(0, pages - fixed.randint(1, 4))
                own_pages = [held + shared + i * (pages - shared) for i in range(W + 1)]
                common = list(range(held, held + shared))
                groups.append([(n, common + list(range(own_pages[i], own_pages[i + 1]))) for i in range(W)])
                held = own_pages[W]
            spare, columns = 2 * B * W + 5, max(n // PAGE + 1 for n in _fork_lengths(case))
            st["parents"] = _ints([b * W + r.randrange(W) for b in range(B) for _ in range(W)])
        else:
            while held < case["live"] * case["pages"]:
                n = fixed.randint(1, case["hi"])
                pages = min((n + PAGE - 1) // PAGE, case["pages"] - held)
                groups.append([(min(n, pages * PAGE), list(range(held, held + pages)))])
                held += pages
            spare, columns = case["pages"] - held, max(len(g[0][1]) for g in groups)
        r.shuffle(groups)
        lens, rows = [n for group in groups for n, _ in group], [row for group in groups for _, row in group]
        blocks = held + spare
        perm = torch.randperm(blocks, generator=g, device="cuda").tolist()
        refs = [0] * blocks
        for row in rows:
            for p in row:
                refs[perm[p]] += 1
        st["table"] = _ints([[perm[p] for p in row] + [0] * (columns - len(row)) for row in rows])
        st["table_out"], st["lens"], st["refs"] = torch.zeros_like(st["table"]), _ints(lens), _ints(refs)
        st["slots"], st["status"] = torch.zeros(len(rows), dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
        st["pairs"] = torch.zeros(len(rows) if k == "fork" else blocks // 2 + 1, 2, dtype=torch.int32, device="cuda")
        st["refs_out"], st["map"] = torch.empty_like(st["refs"]), torch.empty_like(st["refs"])
        st["kv"] = torch.empty(case["layers"], blocks, 2 * n_kv * PAGE * D, dtype=BF, device="cuda").normal_(generator=g)
    return st


# ---- one pass --------------------------------------------------------------------------------------------------------------
def _rotated(x, cos, sin):
    """a rounding to 16 bits behind every operation, as the 16-bit path has them"""
    a, b = x.float().chunk(2, -1)
    r = lambda v: v.to(BF).float()
    return torch.cat([r(r(a * cos) - r(b * sin)), r(r(b * cos) + r(a * sin))], -1).to(BF)


def _as_16bit_pages(k, v):
    """keys and values [blocks, heads, 16, D] as the 16-bit cache holds them: 16-byte pieces of a row permuted by its place in the page"""
    D = k.shape[-1]
    i, c = torch.arange(16, device=k.device).view(16, 1), torch.arange(D, device=k.device).view(1, D)
    source = ((c // 8) ^ (i & 7)) * 8 + c % 8
    both = torch.stack([k, v], 1)
    return both.gather(-1, source.expand(both.shape)).to(BF)


def _write(st):
    n_q, n_kv, D = st["heads"]
    T = st["qkv"].shape[0]
    x = st["qkv"].view(T, n_q + 2 * n_kv, D)
    cs = st["cos_sin"][st["pos"].long()].float().unsqueeze(1)
    turned = _rotated(x[:, : n_q + n_kv], cs[..., : D // 2], cs[..., D // 2:])
    x[:, :n_q] = turned[:, :n_q]
    slot = st["slots"].long()
    kc, ks, vc, vs = st["at"]
    flat = st["kv"].view(st["kv"].shape[0], n_kv, 18 * D)
    page, off = slot // 16, slot % 16
    head = torch.arange(n_kv, device=slot.device).view(1, n_kv, 1)
    for val, code_at, scale_at in ((turned[:, n_q:], kc, ks), (x[:, n_q + n_kv:], vc, vs)):
        code, scale = _codes(val)
        flat[page.view(T, 1, 1), head, code_at[off][:, None, ::2]] = code[..., ::2] | (code[..., 1::2] << 4)
        flat[page.view(T, 1, 1), head, scale_at[off][:, None, ::16]] = scale
    got = flat[st["pages"].long()]
    return {"q": st["qkv"][:, : n_q * D], "cache": _as_16bit_pages(_values(got, kc, ks, D), _values(got, vc, vs, D))}


def _rows_of(st):
    """cached keys and values of every sequence, fp32 [sequences, heads, tokens, D]"""
    n_q, n_kv, D = st["heads"]
    kc, ks, vc, vs = st["at"]
    got = st["kv"].view(-1, n_kv, 18 * D)[st["bt"].long()]
    k, v = _values(got, kc, ks, D), _values(got, vc, vs, D)
    join = lambda x: x.transpose(1, 2).flatten(2, 3)
    return join(k), join(v)


def _softmax_rows(s, seen, v):
    s = s.masked_fill(~seen, float("-inf"))
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))


def _scores(st, q, k):
    s = torch.matmul(q, k.transpose(-1, -2)) * st["scale"]
    return st["cap"] * torch.tanh(s / st["cap"]) if st["cap"] > 0 else s


def _decode(st):
    n_q, n_kv, D = st["heads"]
    k, v = _rows_of(st)
    S = k.shape[0]
    q = st["qkv"][:, : n_q * D].float().view(S, n_kv, n_q // n_kv, D)
    j, ctx = torch.arange(k.shape[2], device=k.device).view(1, 1, 1, -1), st["ctx"].view(S, 1, 1, 1)
    seen = (j < ctx) & (j >= ctx - st["window"]) if st["window"] else j < ctx
    return _softmax_rows(_scores(st, q, k), seen, v).reshape(S, n_q * D).to(BF)


def _prompt(st):
    n_q, n_kv, D = st["heads"]
    k, v = _rows_of(st)
    S, G, past = k.shape[0], n_q // n_kv, st["case"]["past"]
    row, pos = st["row"], st["pos"]
    n = max(st["lens"])
    q = torch.zeros(S, n, n_kv, G, D, device=k.device)
    q[row, pos] = st["qkv"][:, : n_q * D].float().view(-1, n_kv, G, D)
    q = q.permute(0, 2, 3, 1, 4).reshape(S, n_kv, G * n, D)
    at = (torch.arange(n, device=k.device) + past).repeat(G).view(1, 1, -1, 1)
    j = torch.arange(k.shape[2], device=k.device).view(1, 1, 1, -1)
    seen = (j <= at) & (j > at - st["window"]) if st["window"] else j <= at
    out = _softmax_rows(_scores(st, q, k), seen, v).view(S, n_kv, G, n, D).permute(0, 3, 1, 2, 4)
    return out[row, pos].reshape(-1, n_q * D).to(BF)


def _beam(st):
    B, W, V = st["case"]["groups"], st["case"]["beams"], st["case"]["vocab"]
    x = st["logits"].double()
    top = x.amax(-1, keepdim=True)
    t = st["scores"].double().unsqueeze(1) + (x - (top + torch.log(torch.exp(x - top).sum(-1, keepdim=True))))
    best, at = torch.sort(t.view(B, W * V), dim=1, descending=True, stable=True)
    best, at = best[:, : 2 * W], at[:, : 2 * W]
    token, row = at % V, at // V + torch.arange(B, device=at.device).view(B, 1) * W
    stop = (token.unsqueeze(-1) == st["stops"].view(1, 1, -1)).any(-1)
    go = torch.sort(stop.to(torch.int32), dim=1, stable=True)[1][:, :W]   # the first that do not end
    left = stop.logical_not().sum(1, keepdim=True) > torch.arange(W, device=at.device).view(1, W)
    first = torch.arange(B, device=at.device).view(B, 1) * W
    none = torch.full_like(best[:, :W], float("-inf"))
    go_on = (torch.where(left, best.gather(1, go), none), torch.where(left, token.gather(1, go), 0 * first),
             torch.where(left, row.gather(1, go), first))
    return _told(best.float(), token, row, go_on[0].float(), *go_on[1:])


def _told(score, token, row, next_score, next_token, next_row):
    i = torch.int32
    return {"score": score, "token": token.to(i), "row": row.to(i), "next_score": next_score, "next_token": next_token.to(i),
            "next_row": next_row.to(i)}


def _fork(st):
    table, lens, parents, refs = st["table"], st["lens"].long(), st["parents"].long(), st["refs"]
    rows, columns = table.shape
    c = torch.arange(columns, device=table.device).view(1, columns)
    held = c < ((lens + 15) // 16).view(rows, 1)
    n, old = lens[parents], table[parents]
    kept = held[parents]
    part, last = n % 16 != 0, n // 16
    last_page = old.gather(1, last.view(-1, 1)).squeeze(1).long()
    i = torch.arange(rows, device=table.device)
    first = torch.full((rows,), rows, device=table.device).scatter_reduce(0, parents, i, "amin")[parents] == i
    fresh = ~(part & first & (refs[torch.where(part, last_page, 0 * last_page)] == 1))
    free = torch.nonzero(refs == 0).squeeze(1)
    page = free[(torch.cumsum(fresh, 0) - 1).clamp(min=0)]
    out = torch.where(kept, old, st["table_out"])
    mine = (c == last.view(-1, 1))
    out = torch.where(mine & fresh.view(-1, 1), page.view(-1, 1).to(torch.int32), out)
    one = torch.ones(rows * columns, dtype=torch.int32, device=table.device)
    refs.index_add_(0, table.long().flatten()[held.flatten()], -one[: int(held.sum())])
    now = kept | mine
    refs.index_add_(0, out.long().flatten()[now.flatten()], one[: int(now.sum())])
    moved = fresh & part
    st["kv"][:, page[moved]] = st["kv"][:, last_page[moved]]
    st["table_out"].copy_(out)
    slots = out.gather(1, last.view(-1, 1)).squeeze(1) * 16 + (n % 16).to(torch.int32)
    return slots


def _compact(st):
    refs, table, lens = st["refs"], st["table"], st["lens"].long()
    rows, columns = table.shape
    live = refs > 0
    n = int(live.sum())
    ids = torch.arange(refs.numel(), device=refs.device)
    to, source = ids[~live & (ids < n)], ids[live & (ids >= n)]
    where = torch.where(live, ids, -torch.ones_like(ids))
    where[source] = to
    st["kv"][:, to] = st["kv"][:, source]
    held = torch.arange(columns, device=table.device).view(1, columns) < ((lens + 15) // 16).view(rows, 1)
    out = torch.where(held, where[table.long()].to(torch.int32), st["table_out"])
    counts = torch.zeros_like(refs)
    counts[where[live]] = refs[live]
    return out, counts, where.to(torch.int32), _ints([n, to.numel()])


def run(st):
    k = st["case"]["kind"]
    if own:
        return _run_own(st, k)
    if k == "write":
        return _write(st)
    if k == "decode":
        return _decode(st)
    if k == "prompt":
        return _prompt(st)
    if k == "beam":
        return _beam(st)
    if k == "fork":
        slots = _fork(st)
        st["table"], st["table_out"] = st["table_out"], st["table"]
        return {"table": st["table"], "slots": slots, "refs": st["refs"], "kv": st["kv"]}
    table, refs, where, status = _compact(st)
    return {"table": table, "refs": refs, "map": where, "status": status, "kv": st["kv"]}


def _run_own(st, k):
    from llmq_b200 import lib as L

    if k == "write":
        n_q, n_kv, D = st["heads"]
        L.rope_kvwrite_q4(st["qkv"], st["cos_sin"], st["pos"], st["slots"], st["kv"], n_q, n_kv, D, PAGE)
        L.kv4_unpack(st["kv"], st["pages"], st["back"], n_kv, D, PAGE)
        return {"q": st["qkv"][:, : n_q * D], "cache": st["back"]}
    if k == "decode":
        L.decode_attn_q4(st["qkv"], st["out"], st["kv"], st["bt"], st["ctx"], *st["heads"], PAGE, st["scale"], softcap=st["cap"],
                         window=st["window"])
        return st["out"]
    if k == "prompt":
        L.prefill_attn_q4(st["qkv"], st["out"], st["kv"], st["bt"], st["tiles"], *st["heads"], PAGE, st["scale"], st["work"], softcap=st["cap"],
                          window=st["window"])
        return st["out"]
    if k == "beam":
        L.beam_select(st["logits"], st["scores"], st["case"]["beams"], st["stops"], *st["cand"], *st["next"], st["work"])
        names = ("score", "token", "row", "next_score", "next_token", "next_row")
        return dict(zip(names, st["cand"] + st["next"]))
    if k == "fork":
        L.pages_fork(st["table"], st["lens"], st["parents"], st["refs"], st["table_out"], st["slots"], st["pairs"], st["status"])
        L.pages_copy(st["kv"], st["pairs"])
        st["table"], st["table_out"] = st["table_out"], st["table"]
        return {"table": st["table"], "slots": st["slots"], "refs": st["refs"], "kv": st["kv"]}
    L.pages_compact(st["table"], st["lens"], st["refs"], st["table_out"], st["refs_out"], st["map"], st["pairs"], st["status"])
    L.pages_copy(st["kv"], st["pairs"], st["status"][1:])
    return {"table": st["table_out"], "refs": st["refs_out"], "map": st["map"], "status": st["status"], "kv": st["kv"]}


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------
def _span(n, window):
    return min(n, window) if window else n


def work(case):
    k = case["kind"]
    if k in ("write", "decode", "prompt"):
        _, n_q, n_kv, D, _, _, window, _, _ = MODELS[case["model"]]
        token = 2 * n_kv * D * 9 / 16          # bytes of a cached token
    if k == "write":
        T, blocks = case["rows"], (case["rows"] + 15) // 16 if case["together"] else case["rows"]
        row = (2 * n_q + 2 * n_kv) * D * 2 + 2 * D   # queries in and out, keys and values in, its angles
        return {"bytes": T * (row + token) + blocks * PAGE * (token + 4 * n_kv * D), "flops": 20.0 * T * (n_q + 2 * n_kv) * D}
    if k == "decode":
        S = case["seqs"]
        keys = sum(_span(n, window) for n in _lengths(S, case["lo"], case["hi"], 0))
        return {"bytes": keys * token + 4 * S * n_q * D, "flops": 4.0 * keys * n_q * D}
    if k == "prompt":
        lens, past = _lengths(case["prompts"], case["lo"], case["hi"], 0), case["past"]
        pairs = sum(_span(past + i + 1, window) for n in lens for i in range(n))
        keys = sum(min(past + n, n + window - 1) if window else past + n for n in lens)
        return {"bytes": keys * token + 4 * sum(lens) * n_q * D, "flops": 4.0 * pairs * n_q * D}
    if k == "beam":
        n = case["groups"] * case["beams"] * case["vocab"]
        return {"bytes": 2.0 * n + 60.0 * case["groups"] * case["beams"], "flops": 4.0 * n}
    _, _, n_kv, D = MODELS[case["model"]][:4]
    page = 4.0 * n_kv * PAGE * D * case["layers"]
    if k == "fork":   # beams beyond the first of a parent get a copy of its last page
        r, copies, entries = random.Random(0), 0, 0
        for n in _fork_lengths(case):
            chosen = {r.randrange(case["beams"]) for _ in range(case["beams"])}
            copies += case["beams"] - len(chosen)
            entries += case["beams"] * ((n + PAGE - 1) // PAGE)
        return {"bytes": 2.0 * page * copies + 16.0 * entries, "flops": 1.0 * entries}
    live = case["live"] * case["pages"]
    return {"bytes": 2.0 * page * live * (1 - case["live"]) + 12.0 * case["pages"], "flops": 1.0 * case["pages"]}


# ---- the definition, in 64 bits -----------------------------------------------------------------------------------------
_STEPS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def _read(pages, D, keys):
    """rows [..., 16, D] of pages [..., 18 D] in 64 bits, token by token"""
    steps = torch.cat([_STEPS, -_STEPS]).to(pages.device)
    part = pages[..., : 9 * D] if keys else pages[..., 9 * D:]
    codes, scales = part[..., : 8 * D], part[..., 8 * D:].long()
    size = torch.where(scales < 8, (scales % 8).double() * 2.0 ** -17, (8 + scales % 8).double() * torch.exp2((scales // 8 - 18).double()))
    rows = []
    for token in range(16):
        at = (2 * (token % 4) + (token // 4) % 2 + 8 * (token // 8)) if keys else token
        line = codes[..., at * D // 2: (at + 1) * D // 2]
        piece = D // 2 // 8                                       # bytes that are permuted together, and by what
        turn = 0
        if D == 256:
            turn = 4 * (at % 2) if keys else 2 * (token % 4)
        elif D == 128 and not keys:
            turn = 4 * (token // 2 % 2)
        line = torch.cat([line[..., (p ^ turn) * piece: ((p ^ turn) + 1) * piece] for p in range(8)], -1).long()
        value = torch.stack([steps[line % 16], steps[line // 16]], -1).flatten(-2)
        by_group = []
        for group in range(D // 16):
            if keys:
                lane, deep = (at % 8) * 4, at // 8
                where = {64: (lane + group) * 2 + deep, 128: (lane + group // 2) * 4 + 2 * deep + group % 2,
                         256: (lane + group % 8 // 2) * 8 + 4 * deep + group // 8 * 2 + group % 2}[D]
            else:
                t, j = token % 4, token // 4
                where = (group // 2 * 4 + t) * 8 + group % 2 * 4 + j if D == 256 else (group * 4 + t) * 4 + j
            by_group.append(size[..., where: where + 1].expand(*size.shape[:-1], 16))
        rows.append(value * torch.cat(by_group, -1))
    return torch.stack(rows, -2)


def _exact_write(st):
    n_q, n_kv, D = st["heads"]
    T, half = st["qkv"].shape[0], D // 2
    x = st["qkv"].view(T, -1, D).double()
    angle = st["cos_sin"][st["pos"].long()].double()[:, None]
    cos, sin = angle[..., :half], angle[..., half:]
    rounded = lambda v: v.to(torch.float32).to(BF).double()       # (products of two 16-bit numbers are exact in 32 bits, sums nearly always)
    lo, hi = x[:, : n_q + n_kv, :half], x[:, : n_q + n_kv, half:]
    turned = torch.cat([rounded(rounded(lo * cos) - rounded(hi * sin)), rounded(rounded(hi * cos) + rounded(lo * sin))], -1)
    steps = _STEPS.to(x.device)

    def held(v):
        g = v.unflatten(-1, (-1, 16))
        most = g.abs().amax(-1, keepdim=True)
        ladder = torch.cat([torch.arange(1, 8).double() * 2.0 ** -17] + [torch.arange(8, 16).double() * 2.0 ** (e - 3) for e in range(-14, 14)])
        ladder = ladder[ladder <= 10240.0].to(v.device)
        between = (ladder[1:] + ladder[:-1]) * 3.0                # six times the middle of two neighbours; the even one takes a tie
        up = torch.searchsorted(between, most, right=False)
        tie = (up < between.numel()) & (between[up.clamp(max=between.numel() - 1)] == most)
        scale = ladder[torch.where(tie & (up % 2 == 0), up + 1, up)]   # (entry i has mantissa i + 1 modulo 8)
        r = g.abs() / scale
        middle = (steps[1:] + steps[:-1]) / 2
        low, high = torch.searchsorted(middle, r, right=False), torch.searchsorted(middle, r, right=True)
        code = torch.where(low % 2 == 0, low, high)
        return (steps[code] * scale * torch.sign(g)).flatten(-2)

    D16 = st["kv"].view(-1, n_kv, 18 * D)
    k, v = _read(D16, D, True), _read(D16, D, False)
    page, off = st["slots"].long() // 16, st["slots"].long() % 16
    k[page, :, off], v[page, :, off] = held(turned[:, n_q:]), held(x[:, n_q + n_kv:])
    cache = torch.stack([k, v], 1)[st["pages"].long()]
    pieces = cache.unflatten(-1, (-1, 8))
    turned_pieces = torch.stack([pieces[..., i, [p ^ (i % 8) for p in range(D // 8)], :] for i in range(16)], -3)
    return {"q": turned[:, :n_q].reshape(T, n_q * D), "cache": turned_pieces.flatten(-2)}


def _exact_attention(st):
    n_q, n_kv, D = st["heads"]
    past, out = st["case"].get("past", 0), []
    at = 0
    for i, n in enumerate(st["lens"]):
        total, first = past + n, past if "tiles" in st else past + n - 1
        pages = st["kv"].view(-1, n_kv, 18 * D)[st["bt"][i, : (total + 15) // 16].long()]
        k, v = (_read(pages, D, keys).transpose(0, 1).flatten(1, 2)[:, :total] for keys in (True, False))
        q = st["qkv"][at: at + total - first, : n_q * D].double().view(-1, n_kv, n_q // n_kv, D)
        at += total - first
        answer = torch.empty(total - first, n_kv, n_q // n_kv, D, dtype=torch.float64, device=k.device)
        for a in range(0, total - first, 512):
            pos = torch.arange(first + a, min(first + a + 512, total), device=k.device)
            s = torch.einsum("ahgd,hjd->hgaj", q[a: a + 512], k) * st["scale"]
            if st["cap"]:
                s = st["cap"] * torch.tanh(s / st["cap"])
            far = pos[:, None] - torch.arange(total, device=k.device)
            hidden = (far < 0) | (far >= (st["window"] or total + 1))
            answer[a: a + 512] = torch.einsum("hgaj,hjd->ahgd", torch.softmax(s.masked_fill(hidden, float("-inf")), -1), v)
        out.append(answer.reshape(-1, n_q * D))
    return torch.cat(out)


def _exact_beam(st):
    W = st["case"]["beams"]
    scores, next_scores = [], []
    for b in range(st["case"]["groups"]):
        x = st["logits"][b * W: (b + 1) * W].double()
        t = (torch.log_softmax(x, -1) + st["scores"][b * W: (b + 1) * W].double().unsqueeze(1)).flatten()
        best, at = torch.topk(t, 2 * W)
        going = [s for s, token in zip(best.tolist(), (at % x.shape[1]).tolist()) if token not in st["stops"].tolist()][:W]
        scores.append(best)
        next_scores.append(torch.tensor(going + [float("-inf")] * (W - len(going)), dtype=torch.float64, device=x.device))
    return {"score": torch.stack(scores), "token": None, "row": None, "next_score": torch.stack(next_scores), "next_token": None, "next_row": None}


def exact(case, seed):
    k = case["kind"]
    if k in ("fork", "compact"):
        return None       # whole numbers, and pages that are moved as they are
    if k == "prompt" and work(case)["flops"] > 4e11:
        return None
    st = prepare(case, seed)
    return _exact_write(st) if k == "write" else _exact_beam(st) if k == "beam" else _exact_attention(st)

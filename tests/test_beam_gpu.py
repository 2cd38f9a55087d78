"""The selection of beams (csrc/beam.cu) against a plain 64-bit form, and a whole search over a 4-bit cache: selection, forked pages, writes
and attention, beside the same search over rows that are copied instead of shared."""
import math

import pytest
import torch

from tests.kv4_util import BF, BS, attention, attention_close, held, read_pages, rope_rows

pytestmark = pytest.mark.gpu


def select_rules(logits, scores, W, K, stops):
    """(cand scores, tokens, rows), (next ...): every candidate's value in 64 bits, sorted"""
    x = logits.double()
    x = torch.where(torch.isnan(x), -math.inf, x)
    top = x.amax(-1, keepdim=True)
    t = scores.double().unsqueeze(1) + (x - (top + (x - top).exp().sum(-1, keepdim=True).log()))
    dead = ~torch.isfinite(top) | ~torch.isfinite(scores.double()).unsqueeze(1)
    t = torch.where(dead | torch.isnan(t), -math.inf, t)
    B, V = logits.shape[0] // W, logits.shape[1]
    cand, nxt = ([], [], []), ([], [], [])
    for b in range(B):
        best, at = torch.sort(t[b * W: (b + 1) * W].flatten(), descending=True, stable=True)
        best, at = best[:K].tolist(), at[:K].tolist()
        picked = [(s, i % V, b * W + i // V) for s, i in zip(best, at)]
        going = ([p for p in picked if p[1] not in stops] + [(-math.inf, 0, b * W)] * W)[:W]
        for lists, rows in ((cand, picked), (nxt, going)):
            for column, part in zip(lists, zip(*rows)):
                column.append(list(part))
    return cand, nxt


def select(lib, cuda, logits, scores, W, K, stops):
    B, V = logits.shape[0] // W, logits.shape[1]
    i32 = dict(dtype=torch.int32, device=cuda)
    cand = (torch.empty(B, K, device=cuda), torch.empty(B, K, **i32), torch.empty(B, K, **i32))
    nxt = (torch.empty(B, W, device=cuda), torch.empty(B, W, **i32), torch.empty(B, W, **i32))
    work = torch.full((lib.beam_select_workspace(B, W, V, K),), 0xFF, dtype=torch.uint8, device=cuda)
    lib.beam_select(logits.to(cuda), scores.to(cuda), W, torch.tensor(stops, **i32), *cand, *nxt, work)
    return [c.cpu() for c in cand], [c.cpu() for c in nxt]


def check(lib, cuda, logits, scores, W, K, stops):
    want, got = select_rules(logits, scores, W, K, stops), select(lib, cuda, logits, scores, W, K, stops)
    for w, g in zip(want, got):
        assert g[1].tolist() == w[1] and g[2].tolist() == w[2]
        ref = torch.tensor(w[0], dtype=torch.float64)
        inf = torch.isinf(ref)
        assert torch.equal(torch.isinf(g[0]), inf) and (g[0][inf] < 0).all()
        # rounding to fp32 (2^-24), and the logarithm of a sum that keeps 2^-20 at the very least
        tol = 2.0 ** -24 * ref.abs() + 2.0 ** -20
        assert ((g[0].double() - ref).abs()[~inf] <= tol[~inf]).all()


@pytest.mark.parametrize("V", [64, 97, 1000, 2048, 2049, 32000, 50257, 128256, 256000])
@pytest.mark.parametrize("B,W,K", [(1, 1, 1), (1, 4, 8), (3, 5, 10), (2, 32, 64), (9, 2, 7)])
def test_select(cuda, V, B, W, K):
    from llmq_b200 import lib
    g = torch.Generator().manual_seed(V + K)
    logits = (2.5 * torch.randn(B * W, V, generator=g)).to(BF)
    scores = -3 * torch.rand(B * W, generator=g)
    check(lib, cuda, logits, scores, W, K, [])
    check(lib, cuda, logits, scores, W, K, logits.float().argmax(-1)[:3].tolist())


@pytest.mark.parametrize("V", [3001, 50257, 256000])
@pytest.mark.parametrize("W,K", [(2, 4), (8, 16), (3, 64)])
def test_few_tokens_allowed(cuda, V, W, K):
    """rows of which a mask leaves none, one, about K or some hundred tokens, anywhere in them, and rows of which it leaves the second half"""
    from llmq_b200 import lib
    g = torch.Generator().manual_seed(V + W)
    for left in (0, 1, K - 1, K, K + 1, 300):
        logits = torch.full((2 * W, V), -math.inf)
        for row in logits:
            at = torch.randperm(V, generator=g)[:left]
            row[at] = torch.randn(left, generator=g)
        check(lib, cuda, logits.to(BF), -torch.rand(2 * W, generator=g), W, K, [])
    half = torch.randn(2 * W, V, generator=g)
    half[:, :V // 2] = -math.inf
    half[-1, V // 2: V // 2 + 40] = math.nan
    check(lib, cuda, half.to(BF), -torch.rand(2 * W, generator=g), W, K, [])


@pytest.mark.parametrize("V", [9000, 50257, 128256])
@pytest.mark.parametrize("W,K", [(1, 1), (8, 16), (2, 64)])
def test_logits_in_order(cuda, V, W, K):
    """rows that rise, fall, rise in steps, and random ones whose largest logits lie side by side"""
    from llmq_b200 import lib
    g = torch.Generator().manual_seed(V + K)
    x = (2.5 * torch.randn(2 * W, V, generator=g)).to(BF)
    scores = -torch.rand(2 * W, generator=g)
    check(lib, cuda, x.sort(-1)[0], scores, W, K, [])
    check(lib, cuda, x.sort(-1, descending=True)[0], scores, W, K, [])
    steps = torch.arange(V).div(997, rounding_mode="floor").to(BF).expand(2 * W, V).contiguous()
    check(lib, cuda, steps, scores, W, K, [])
    x[:, V // 3: V // 3 + 700] = x.float().sort(-1, descending=True)[0][:, :700].to(BF)
    check(lib, cuda, x, scores, W, K, [])


def test_whatever_the_batch(cuda):
    """in the batch-invariant mode a group's scores are the same bits alone and beside others"""
    from llmq_b200 import lib
    g = torch.Generator().manual_seed(5)
    W, K, V = 4, 8, 50257
    logits, scores = (2.5 * torch.randn(90 * W, V, generator=g)).to(BF), -torch.rand(90 * W, generator=g)
    lib.load().b200q_gemm_set_splitk(1)   # (stands for B200Q_BATCH_INVARIANT)
    try:
        many = select(lib, cuda, logits, scores, W, K, [])
        for b in (0, 57, 89):
            alone = select(lib, cuda, logits[b * W: (b + 1) * W], scores[b * W: (b + 1) * W], W, K, [])
            for x, y in zip(many, alone):
                assert torch.equal(x[0][b], y[0][0]) and torch.equal(x[1][b], y[1][0]) and torch.equal(x[2][b] - b * W, y[2][0])
    finally:
        lib.load().b200q_gemm_set_splitk(0)


# A row's logarithm: terms off by at most 2^-22 (the exponential) and 1.5 x 2^-24 (the rounding of its exponent, which is taken relative to the
# row's own largest logits), five additions in fp32 on a term's way into a sum of 64 bits: (4 + 1.5 + 5) 2^-24, and a result rounded to fp32.
LOG_SUM = 10.5 * 2.0 ** -24


@pytest.mark.parametrize("V", [64, 3001, 128256])
def test_one_logit(cuda, V):
    """rows of which a mask leaves one token, and rows whose largest logit has all but 2^-20 of the sum: the token's probability is 1 within what
    a row's logarithm may be off by, whatever the logit's size, and never above 1"""
    from llmq_b200 import lib
    sizes = [15.3125, 23.0, 30.625, 31.875, -15.3125, -30.625, -31.5, 0.0, 100.0, -100.0, 599.0, -640.0, 1e4, -1e4, 1e30, -1e30]
    for rest in (-math.inf, -30.0):
        x = torch.full((len(sizes), V), -math.inf, dtype=torch.float64)
        for i, size in enumerate(sizes):
            if rest > -math.inf and abs(size) < 1000:
                x[i] = size + rest
            x[i, V * i // len(sizes)] = size
        x, scores = x.to(BF), -torch.rand(len(sizes), generator=torch.Generator().manual_seed(V))
        cand, _ = select(lib, cuda, x, scores, 1, 1, [])
        want, _ = select_rules(x, scores, 1, 1, [])
        assert cand[1].tolist() == want[1]
        ref = torch.tensor(want[0], dtype=torch.float64).flatten()
        got = cand[0].double().flatten()
        assert ((got - ref).abs() <= LOG_SUM + 2.0 ** -24 * ref.abs()).all(), (got - ref) * 2 ** 24
        assert (got <= scores.double()).all()


@pytest.mark.parametrize("V,R", [(128256, 740), (50257, 740), (256000, 384), (256000, 4)])
def test_peak_over_a_flat_tail(cuda, V, R):
    """rows of one large logit, wherever it is, and a tail whose terms lie below half of its last place each: they count"""
    from llmq_b200 import lib
    tail, peak = -2.875, 14.0
    x = torch.full((R, V), tail, dtype=BF)
    at = [(0, V - 1, V // 2, 1, 8, 4096, V // 3, 7919)[i % 8] + 2 * (i // 8) * (-1 if i % 8 in (1, 2) else 1) for i in range(R)]
    x[torch.arange(R), torch.tensor(at)] = peak
    scores = torch.zeros(R)
    cand, _ = select(lib, cuda, x, scores, 1, 1, [])
    ref = -math.log1p((V - 1) * math.exp(tail - peak))
    assert cand[1].flatten().tolist() == at
    assert ((cand[0].double() - ref).abs() <= LOG_SUM + 2.0 ** -24 * abs(ref)).all(), (cand[0].double() - ref).abs().max() * 2 ** 24


@pytest.mark.parametrize("V,R", [(128256, 740), (256000, 384), (50257, 300)])
def test_sums_of_rows_with_too_many_near_the_bound(cuda, V, R):
    """rows of hundreds of equal largest logits, of any size, with and without larger ones behind them"""
    from llmq_b200 import lib
    sizes = [-500.0, -556.0, -598.0, -37.0, -3.0, 0.0, 5.0, 41.0, 300.0, 556.0]
    x = torch.empty(R, V, dtype=BF)
    ref = []
    for i in range(R):
        size, more = sizes[i % 10], (0.0, 1.0, 4.0, 12.0)[i // 10 % 4]
        x[i] = size
        at = V - 1 - 97 * (i % 5)
        x[i, at] = size + more
        y = float(x[i, at]) - float(x[i, 0])   # (sizes are rounded to bf16)
        ref.append(-math.log1p((V - 1) * math.exp(-y)))
    cand, _ = select(lib, cuda, x, torch.zeros(R), 1, 1, [])
    ref = torch.tensor(ref, dtype=torch.float64)
    e = (cand[0].flatten().double() - ref).abs()
    assert (e <= LOG_SUM + 2.0 ** -24 * ref.abs()).all(), (e * 2 ** 24).max()


def test_many_groups(cuda):
    from llmq_b200 import lib
    g = torch.Generator().manual_seed(1)
    check(lib, cuda, (2.5 * torch.randn(600, 5000, generator=g)).to(BF), -torch.rand(600, generator=g), 3, 6, [5])
    check(lib, cuda, (2.5 * torch.randn(70000, 64, generator=g)).to(BF), -torch.rand(70000, generator=g), 1, 2, [])   # more rows than a grid dimension takes


@pytest.mark.parametrize("V", [80, 5000, 40001])
@pytest.mark.parametrize("W,K", [(1, 4), (4, 8), (6, 64)])
def test_equal_and_hidden_logits(cuda, V, W, K):
    """all logits equal, few different ones, most at -infinity, fewer than K that are not, NaN, rows with none, rows that do not take part"""
    from llmq_b200 import lib
    g = torch.Generator().manual_seed(V)
    B = 2
    R = B * W
    scores = -torch.rand(R, generator=g)
    check(lib, cuda, torch.zeros(R, V).to(BF), torch.zeros(R), W, K, [0, 3])
    check(lib, cuda, torch.randint(0, 3, (R, V), generator=g).to(BF), scores, W, K, [])
    few = torch.full((R, V), -math.inf)
    few[:, [3, V // 2, V - 1]] = torch.randn(R, 3, generator=g)
    check(lib, cuda, few.to(BF), scores, W, K, [3])
    nan = torch.randn(R, V, generator=g)
    nan[:, ::3] = math.nan
    check(lib, cuda, nan.to(BF), scores, W, K, [])
    nan[:, :] = math.nan
    nan[0, 7] = 1.0
    check(lib, cuda, nan.to(BF), scores, W, K, [])
    check(lib, cuda, torch.full((R, V), -math.inf).to(BF), scores, W, K, [0])
    first = torch.full((R,), -math.inf)   # a search's first step: one beam takes part
    first[::W] = 0.0
    check(lib, cuda, torch.randn(R, V, generator=g).to(BF), first, W, K, [])
    first[0] = math.nan
    big = torch.randn(R, V, generator=g)
    big[R - 1, 5] = math.inf
    check(lib, cuda, big.to(BF), first, W, K, [])
    check(lib, cuda, (1e5 * torch.randn(R, V, generator=g)).to(BF), 1e4 * scores, W, K, [])
    close = torch.randn(R, V, generator=g).to(BF)
    close[1:] = close[0]   # beams with the same logits and the same score: the lower row first
    check(lib, cuda, close, torch.full((R,), -1.25), W, K, [])


@pytest.mark.parametrize("V", [64, 3001, 40001])
@pytest.mark.parametrize("W,K", [(1, 4), (4, 8), (3, 64)])
def test_zeros_of_either_sign(cuda, V, W, K):
    """a logit or a score of -0 is as large as one of 0: the lower row and token first"""
    from llmq_b200 import lib
    g = torch.Generator().manual_seed(V)
    R = 2 * W
    zeros = torch.where(torch.rand(R, V, generator=g) < 0.5, -0.0, 0.0)
    scores = -torch.rand(R, generator=g)
    check(lib, cuda, zeros.to(BF), scores, W, K, [])                       # all equal
    few = torch.where(torch.rand(R, V, generator=g) < 40 / V, zeros, torch.tensor(-5.0))
    check(lib, cuda, few.to(BF), scores, W, K, [])
    few[:, V // 2] = 1.0
    check(lib, cuda, few.to(BF), scores, W, K, [])
    one = torch.full((R, V), -math.inf)                                    # certain tokens: scores of -0 and 0
    one[torch.arange(R), torch.arange(R) * 7 % V] = torch.where(torch.arange(R) % 2 == 0, -0.0, 0.0)
    check(lib, cuda, one.to(BF), torch.where(torch.arange(R) % 2 == 0, -0.0, 0.0), W, K, [])


@pytest.mark.parametrize("D,n_q,n_kv", [(64, 4, 2), (128, 8, 2), (256, 4, 1)])
def test_search(cuda, D, n_q, n_kv):
    """A model of one layer whose queries, keys and values are rows of a table and whose logits are its attention's outputs times another:
    two groups of four beams over pages that are shared, forked, written and read, captured once and replayed.  Beside it the same on the
    CPU with a cache of its own for each beam, fed with the GPU's choices; its attention has to be the GPU's within rounding, and the
    choices those that the GPU's own logits give."""
    from llmq_b200 import lib
    B, W, V, steps, stride, blocks = 2, 4, 320, 40, 6, 80
    R, width = B * W, (n_q + 2 * n_kv) * D
    g = torch.Generator().manual_seed(D)
    embed = torch.randn(V, width, generator=g).to(BF)
    head = torch.randn(V, n_q * D, generator=g).to(BF)
    angle = torch.outer(torch.arange(200).float(), 10000.0 ** (-torch.arange(0, D, 2).float() / D))
    cos_sin = torch.cat([angle.cos(), angle.sin()], -1).to(BF)
    i32 = dict(dtype=torch.int32, device=cuda)
    emb, hd, cs = embed.to(cuda), head.to(cuda), cos_sin.to(cuda)
    tables = [torch.zeros(R, stride, **i32) for _ in range(2)]
    refs, slots, pairs, status = torch.zeros(blocks, **i32), torch.zeros(R, **i32), torch.zeros(R, 2, **i32), torch.zeros(2, **i32)
    kv = torch.full((1, blocks, n_kv, 18 * D), 0xFF, dtype=torch.uint8, device=cuda)
    lens, new_lens = torch.zeros(R, **i32), torch.zeros(R, **i32)
    K = 2 * W
    cand = (torch.empty(B, K, device=cuda), torch.empty(B, K, **i32), torch.empty(B, K, **i32))
    nxt = (torch.zeros(B, W, device=cuda), torch.zeros(B, W, **i32), torch.zeros(B, W, **i32))
    scores, tokens, parents = nxt[0].view(-1), nxt[1].view(-1), nxt[2].view(-1)
    scores.fill_(-math.inf)
    scores[::W] = 0.0
    tokens.fill_(1)
    parents.copy_(torch.arange(R))
    stops = torch.tensor([2], **i32)
    work = torch.empty(lib.beam_select_workspace(B, W, V, K), dtype=torch.uint8, device=cuda)
    out, logits = torch.zeros(R, n_q * D, dtype=BF, device=cuda), torch.zeros(R, V, dtype=BF, device=cuda)

    def step(k):   # the beams' last tokens, chosen before, are written and attended to; then the next ones are chosen
        table, other = tables[k % 2], tables[1 - k % 2]
        lib.pages_fork(table, lens, parents, refs, other, slots, pairs, status)
        lib.pages_copy(kv, pairs)
        new_lens.copy_(lens[parents.long()] + 1)
        lens.copy_(new_lens)
        qkv = emb[tokens.long()]
        lib.rope_kvwrite_q4(qkv, cs, lens - 1, slots, kv, n_q, n_kv, D, BS)
        lib.decode_attn_q4(qkv, out, kv, other, lens, n_q, n_kv, D, BS, D ** -0.5)
        lib.gemm_bf16(out, hd, logits)
        lib.beam_select(logits, scores, W, stops, *cand, *nxt, work)

    history = [[] for _ in range(R)]   # the tokens that each row stands for
    k_rows = [torch.zeros(0, n_kv, D, dtype=torch.float64) for _ in range(R)]
    v_rows = [torch.zeros(0, n_kv, D, dtype=torch.float64) for _ in range(R)]
    graphs = None
    for k in range(steps):
        before = (parents.cpu().tolist(), tokens.cpu(), scores.cpu())
        if k < 2 or graphs is None:
            step(k)
        else:
            graphs[k % 2].replay()
        if k == 1:   # two graphs, because the two tables take turns
            torch.cuda.synchronize()
            keep = [t.clone() for t in (*tables, refs, slots, pairs, status, kv, lens, new_lens, *nxt, out, logits)]
            graphs = []
            for i in range(2):
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph):
                    step(i)
                graphs.append(graph)
            for t, s in zip((*tables, refs, slots, pairs, status, kv, lens, new_lens, *nxt, out, logits), keep):
                t.copy_(s)
        torch.cuda.synchronize()
        assert status.cpu().tolist() == [0, 0] and lib.load().b200q_wait_failures() == 0
        rows, token, score = before
        history = [history[p] + [int(t)] for p, t in zip(rows, token)]
        q, kk, vv = rope_rows(embed[token.long()], cos_sin, torch.full((R,), k), n_q, n_kv, D)
        k_rows = [torch.cat([k_rows[p], held(kk[i: i + 1])]) for i, p in enumerate(rows)]
        v_rows = [torch.cat([v_rows[p], held(vv[i: i + 1])]) for i, p in enumerate(rows)]
        for i in range(R):
            ref, weight, size = attention(q[i: i + 1], k_rows[i].transpose(0, 1), v_rows[i].transpose(0, 1), torch.tensor([k]), D ** -0.5)
            attention_close(out[i].view(1, n_q, D), ref, weight, size, D, 2.0 ** -11, f"step {k} row {i}")
        want = select_rules(logits.cpu(), score, W, K, [2])
        assert nxt[1].cpu().tolist() == want[1][1] and nxt[2].cpu().tolist() == want[1][2]
    # the pages hold each row's tokens; nobody holds a page that no row names
    table, count = tables[steps % 2].cpu(), [0] * blocks
    for i in range(R):
        pages = table[i, : (steps + BS - 1) // BS].long()
        for p in pages.tolist():
            count[p] += 1
        k_held, v_held = read_pages(kv[0].cpu()[pages], D)
        for got, ref in ((k_held, k_rows[i]), (v_held, v_rows[i])):
            assert torch.equal(got.transpose(1, 2).flatten(0, 1)[:steps], ref)
    assert refs.cpu().tolist() == count
    # moved to the front, everything is as it was
    moved, refs_out, page_map = tables[1 - steps % 2], torch.zeros_like(refs), torch.zeros_like(refs)
    moves = torch.zeros(blocks // 2 + 1, 2, **i32)
    again = torch.zeros_like(out)
    lib.pages_compact(tables[steps % 2], lens, refs, moved, refs_out, page_map, moves, status)
    lib.pages_copy(kv, moves, status[1:])
    qkv = emb[before[1].to(cuda).long()]
    lib.rope_kvwrite_q4(qkv, cs, lens - 1, torch.full_like(slots, -1), kv, n_q, n_kv, D, BS)
    lib.decode_attn_q4(qkv, again, kv, moved, lens, n_q, n_kv, D, BS, D ** -0.5)
    assert torch.equal(again, out)
    lib.pages_free(moved, lens, refs_out)
    assert int(refs_out.abs().max()) == 0

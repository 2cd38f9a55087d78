"""The 4-bit paged cache (csrc/kv4_ops.cu, csrc/kv4_attn.cu) through the C ABI: what is written, what is read back, and attention over
it for single tokens and for prompts, against plain 64-bit forms (tests/kv4_util.py)."""
import pytest
import torch

from tests.kv4_util import BF, BS, attention, attention_close, held, make_cache, read_pages, rope_rows, write_rows

pytestmark = pytest.mark.gpu


def same(a, b):
    return torch.equal(torch.nan_to_num(a.double().cpu(), nan=1e30), torch.nan_to_num(b.double().cpu(), nan=1e30))


def hard_rows(T, n, g):
    """rows whose groups are zeros, tiny, subnormal, huge, infinite, NaN or full of values on the borders between two codes"""
    x = torch.randn(T, n, generator=g) * torch.exp2(torch.randint(-20, 18, (T, n // 16), generator=g).float()).repeat_interleave(16, 1)
    x = x.to(BF).view(T, n // 16, 16)
    border = torch.tensor([6.0, 0.25, -0.75, 1.25, -1.75, 2.5, -3.5, 5.0, 0.0, -0.0, 0.5, 1.5, 3.0, -4.0, 2.0, -6.0])
    scale = torch.exp2(torch.randint(-12, 11, (T, n // 16, 1), generator=g).float()) * (1 + torch.randint(0, 8, (T, n // 16, 1), generator=g) / 8)
    kind = torch.randint(0, 10, (T, n // 16), generator=g)
    x[kind == 1] = (border * scale)[kind == 1].to(BF)
    x[kind == 2] = 0.0
    x[kind == 3] = 1e-7
    x[kind == 4] = (border * scale)[kind == 4].to(BF) * 1.5   # largest magnitudes of 9, 10.5, ...: scales on borders
    x[(kind == 5), 3] = float("inf")
    x[(kind == 6), 7] = float("nan")
    x[(kind == 7), 0] = -3e38
    return x.reshape(T, n)


@pytest.mark.parametrize("D,n_q,n_kv", [(64, 4, 2), (128, 3, 3), (128, 8, 1), (256, 4, 2), (64, 0, 1)])
@pytest.mark.parametrize("T", [1, 7, 333])
@pytest.mark.parametrize("hard", [False, True])
def test_write(cuda, D, n_q, n_kv, T, hard):
    from llmq_b200 import lib
    g = torch.Generator().manual_seed(T + D)
    n = (n_q + 2 * n_kv) * D
    qkv = hard_rows(T, n, g) if hard else torch.randn(T, n, generator=g).to(BF)
    positions = torch.randint(0, 5000, (T,), generator=g).to(torch.int32)
    cos_sin = torch.randn(5000, D, generator=g).to(BF) if not hard else torch.cat([torch.ones(5000, D // 2), torch.zeros(5000, D // 2)], 1).to(BF)
    blocks = T // 16 + 4
    slots = torch.randperm(blocks * 16, generator=g)[:T].to(torch.int32)
    if T > 2:
        slots[1] = -1
    start = torch.randint(0, 256, (blocks, n_kv, 18 * D), generator=g).to(torch.uint8)
    q, k, v = rope_rows(qkv, cos_sin, positions, n_q, n_kv, D)
    ref = start.clone()
    write_rows(ref, slots, k, v, D)
    x, cache = qkv.to(cuda), start.to(cuda)
    lib.rope_kvwrite_q4(x, cos_sin.to(cuda), positions.to(cuda), slots.to(cuda), cache, n_q, n_kv, D, BS)
    got = cache.cpu()
    if n_q:
        assert same(x[:, : n_q * D], q.reshape(T, -1))
    assert torch.equal(x[:, n_q * D:].view(torch.int16).cpu(), qkv[:, n_q * D:].view(torch.int16))   # keys and values stay as they were
    for a, b in zip(read_pages(got, D), read_pages(ref, D)):
        assert same(a, b)
    # (codes of a NaN's group say nothing; all other bytes are the same ones)
    if not hard:
        assert torch.equal(got, ref)


@pytest.mark.parametrize("D,n_kv", [(64, 3), (128, 2), (256, 1)])
@pytest.mark.parametrize("n", [1, 5, 700])
def test_unpack(cuda, D, n_kv, n):
    from llmq_b200 import lib
    g = torch.Generator().manual_seed(n)
    cache = torch.randint(0, 256, (900, n_kv, 18 * D), generator=g).to(torch.uint8)
    pages = torch.randint(0, 900, (n,), generator=g).to(torch.int32)   # (pages may be named twice)
    out = torch.full((n + 1, 2, n_kv, BS, D), 7.0, dtype=BF, device=cuda)
    cache[:, :, 8 * D: 9 * D].clamp_(max=226)
    cache[:, :, 17 * D:].clamp_(max=226)
    lib.kv4_unpack(cache.to(cuda), pages.to(cuda), out, n_kv, D, BS)
    k, v = read_pages(cache[pages.long()], D)
    got = out.cpu()
    assert (got[n] == 7).all()
    i, c = torch.arange(16).view(16, 1), torch.arange(D).view(1, D)
    at = ((c // 8) ^ (i & 7)) * 8 + c % 8
    for which, x in ((0, k), (1, v)):
        assert same(got[:n, which].gather(-1, at.expand(n, n_kv, 16, D)), x)


CASES = [[1], [0, 1, 15, 16, 17], [31, 32, 33, 63, 64, 65, 100], [700, 3, 129], [4097], list(range(1, 80))]


@pytest.mark.parametrize("D,n_q,n_kv", [(64, 8, 2), (64, 7, 1), (128, 8, 8), (128, 8, 1), (128, 6, 2), (256, 8, 2), (256, 8, 1)])
@pytest.mark.parametrize("ctxs", CASES, ids=lambda c: f"{len(c)}x{max(c)}")
@pytest.mark.parametrize("cap,window", [(0.0, 0), (20.0, 100), (0.0, 1), (0.0, 50)])
def test_decode(cuda, D, n_q, n_kv, ctxs, cap, window):
    from llmq_b200 import lib
    cache, table, rows = make_cache(ctxs, n_kv, D, seed=len(ctxs) + D)
    B = len(ctxs)
    qkv = torch.randn(B, (n_q + 2 * n_kv) * D, generator=torch.Generator().manual_seed(7)).to(BF)
    out = torch.full((B + 1, n_q * D), float("nan"), dtype=BF, device=cuda)
    args = (cache.to(cuda), table.to(cuda), torch.tensor(ctxs, dtype=torch.int32, device=cuda), n_q, n_kv, D, BS, D ** -0.5)
    for whole in (0, 1):
        out.fill_(float("nan"))
        lib.decode_attn_q4_set_whole(whole)
        try:
            lib.decode_attn_q4(qkv.to(cuda), out, *args, softcap=cap, window=window)
        finally:
            lib.decode_attn_q4_set_whole(-1)
        got = out.cpu()
        assert torch.isnan(got[B].float()).all()
        for i, c in enumerate(ctxs):
            if c == 0:
                assert (got[i] == 0).all()
                continue
            q = qkv[i: i + 1, : n_q * D].view(1, n_q, D)
            ref, weight, size = attention(q, *rows[i], torch.tensor([c - 1]), D ** -0.5, cap, window)
            attention_close(got[i].view(1, n_q, D), ref, weight, size, D, 2.0 ** -11, f"ctx {c}, whole {whole}")
    assert lib.load().b200q_wait_failures() == 0


@pytest.mark.parametrize("D,n_q,n_kv", [(64, 4, 1), (128, 8, 2), (256, 2, 1)])
@pytest.mark.parametrize("q_size,kv_size,scale", [(1e4, 1.0, 1e-5), (1e-6, 30.0, 1e4), (1.0, 1e-3, 100.0), (3.0, 5000.0, 1e-5), (1.0, 1.0, -0.2), (1.0, 1.0, 0.0)])
def test_decode_sizes_of_values(cuda, D, n_q, n_kv, q_size, kv_size, scale):
    """queries beyond and below what a half holds, scales of keys and values at both ends, scores that fall instead of rise"""
    from llmq_b200 import lib
    ctxs = [300, 77]
    cache, table, rows = make_cache(ctxs, n_kv, D, seed=3, spread=kv_size)
    qkv = (q_size * torch.randn(2, (n_q + 2 * n_kv) * D, generator=torch.Generator().manual_seed(9))).to(BF)
    out = torch.empty(2, n_q * D, dtype=BF, device=cuda)
    lib.decode_attn_q4(qkv.to(cuda), out, cache.to(cuda), table.to(cuda), torch.tensor(ctxs, dtype=torch.int32, device=cuda), n_q, n_kv, D, BS, scale)
    for i, c in enumerate(ctxs):
        ref, weight, size = attention(qkv[i: i + 1, : n_q * D].view(1, n_q, D), *rows[i], torch.tensor([c - 1]), scale)
        attention_close(out[i].view(1, n_q, D), ref, weight, size, D, 2.0 ** -11, f"ctx {c}")


@pytest.mark.parametrize("D", [64, 128, 256])
def test_decode_growing_scores(cuda, D):
    """each page's scores beyond the ones before it: the running maximum moves all the way, by less and by more than its step"""
    from llmq_b200 import lib
    ctx, n_kv, n_q = 600, 1, 4
    for step in (0.05, 0.3, 3.0):
        g = torch.Generator().manual_seed(1)
        k = (torch.randn(ctx, 1, D, generator=g) * 0.1 + step * torch.arange(ctx).view(ctx, 1, 1) / 16).to(BF)
        v = torch.randn(ctx, 1, D, generator=g).to(BF)
        cache = torch.zeros((ctx + 15) // 16, 1, 18 * D, dtype=torch.uint8)
        write_rows(cache, torch.arange(ctx), k, v, D)
        table = torch.arange((ctx + 15) // 16, dtype=torch.int32).view(1, -1)
        qkv = (torch.rand(1, 6 * D, generator=g) + 0.5).to(BF)
        out = torch.empty(1, n_q * D, dtype=BF, device=cuda)
        lib.decode_attn_q4(qkv.to(cuda), out, cache.to(cuda), table.to(cuda), torch.tensor([ctx], dtype=torch.int32, device=cuda), n_q, n_kv, D, BS, 1 / D)
        ref, weight, size = attention(qkv[:, : n_q * D].view(1, n_q, D), held(k).transpose(0, 1), held(v).transpose(0, 1), torch.tensor([ctx - 1]), 1 / D)
        attention_close(out.view(1, n_q, D), ref, weight, size, D, 2.0 ** -11, f"step {step}")


def test_decode_far_pages_and_many_rows(cuda):
    """pages beyond 2^31 bytes of the cache; more sequences than one grid dimension takes, most of them empty"""
    from llmq_b200 import lib
    D, n_kv, n_q = 64, 8, 8
    page = lib.kv4_page_bytes(n_kv, D)
    blocks = 2 ** 31 // page + 300
    ctxs = [200, 90]
    small, table, rows = make_cache(ctxs, n_kv, D, seed=5)
    cache = torch.zeros(blocks, n_kv, 18 * D, dtype=torch.uint8, device=cuda)
    cache[blocks - small.shape[0]:] = small.to(cuda)
    B = 65535 + 9
    far = torch.zeros(B, table.shape[1], dtype=torch.int32)
    far[0], far[B - 1] = table[0] + blocks - small.shape[0], table[1] + blocks - small.shape[0]
    lens = torch.zeros(B, dtype=torch.int32)
    lens[0], lens[B - 1] = 200, 90
    qkv = torch.randn(B, (n_q + 2 * n_kv) * D, generator=torch.Generator().manual_seed(7)).to(BF)
    out = torch.full((B, n_q * D), float("nan"), dtype=BF, device=cuda)
    lib.decode_attn_q4(qkv.to(cuda), out, cache, far.to(cuda), lens.to(cuda), n_q, n_kv, D, BS, D ** -0.5)
    got = out.cpu()
    assert (got[1: B - 1] == 0).all()
    for i, r in ((0, 0), (B - 1, 1)):
        ref, weight, size = attention(qkv[i: i + 1, : n_q * D].view(1, n_q, D), *rows[r], torch.tensor([ctxs[r] - 1]), D ** -0.5)
        attention_close(got[i].view(1, n_q, D), ref, weight, size, D, 2.0 ** -11)
    # writing there
    positions, slots = torch.tensor([3], dtype=torch.int32), torch.tensor([blocks * 16 - 1], dtype=torch.int32)
    cos_sin = torch.cat([torch.ones(8, D // 2), torch.zeros(8, D // 2)], 1).to(BF)
    lib.rope_kvwrite_q4(qkv[:1].to(cuda), cos_sin.to(cuda), positions.to(cuda), slots.to(cuda), cache, n_q, n_kv, D, BS)
    k, v = read_pages(cache[-1].cpu(), D)
    assert same(k[:, 15], held(qkv[0].view(-1, D)[n_q: n_q + n_kv])) and same(v[:, 15], held(qkv[0].view(-1, D)[n_q + n_kv:]))


def tiles_of(portions):
    tiles, row = [], 0
    for i, (n, past) in enumerate(portions):
        tiles += [[i, row + j, min(16, n - j), past + j] for j in range(0, n, 16)]
        row += n
    return torch.tensor(tiles, dtype=torch.int32), row


@pytest.mark.parametrize("D,n_q,n_kv", [(64, 8, 2), (128, 8, 1), (128, 3, 3), (256, 8, 2)])
@pytest.mark.parametrize("portions", [[(1, 0)], [(16, 0), (3, 40)], [(5, 11), (33, 0), (17, 100)], [(700, 0)], [(300, 77), (40, 1000)], [(12, 3)] * 40],
                         ids=lambda p: f"{len(p)}x{max(n for n, _ in p)}")
@pytest.mark.parametrize("cap,window", [(0.0, 0), (30.0, 90), (0.0, 7)])
def test_prompts(cuda, D, n_q, n_kv, portions, cap, window):
    from llmq_b200 import lib
    cache, table, rows = make_cache([n + past for n, past in portions], n_kv, D, seed=len(portions) + D)
    table = torch.cat([table, torch.zeros(table.shape[0], 3, dtype=torch.int32)], 1).contiguous()
    tiles, T = tiles_of(portions)
    qkv = torch.randn(T, (n_q + 2 * n_kv) * D, generator=torch.Generator().manual_seed(7)).to(BF)
    out = torch.full((T + 1, n_q * D), float("nan"), dtype=BF, device=cuda)
    size = lib.prefill_attn_q4_workspace(*table.shape, n_kv, D)
    work = torch.full((size + 256,), 0xFF, dtype=torch.uint8, device=cuda)
    lib.prefill_attn_q4(qkv.to(cuda), out, cache.to(cuda), table.to(cuda), tiles.to(cuda), n_q, n_kv, D, BS, D ** -0.5, work[:size], softcap=cap, window=window)
    got = out.cpu()
    assert torch.isnan(got[T].float()).all() and (work[size:] == 0xFF).all()
    at = 0
    for i, (n, past) in enumerate(portions):
        q = qkv[at: at + n, : n_q * D].view(n, n_q, D)
        ref, weight, sz = attention(q, *rows[i], torch.arange(past, past + n), D ** -0.5, cap, window)
        # probabilities are bf16 here, a half step 2^-8
        attention_close(got[at: at + n].view(n, n_q, D), ref, weight, sz, D, 2.0 ** -8, f"portion {i}")
        at += n
    assert lib.load().b200q_wait_failures() == 0


@pytest.mark.parametrize("route", [-1, 0, 1, 2])
@pytest.mark.parametrize("D,n_q,n_kv", [(64, 8, 2), (128, 8, 1), (256, 8, 2)])
@pytest.mark.parametrize("window", [0, 50])
def test_padded_lists_of_tiles(cuda, D, n_q, n_kv, window, route):
    """tiles of no rows between the others and behind them, at positions whose pages nobody sees: as if they were not there"""
    from llmq_b200 import lib
    portions = [(5, 11), (333, 0), (170, 100)]
    cache, table, rows = make_cache([n + past for n, past in portions], n_kv, D, seed=D)
    table = torch.cat([table, torch.zeros(2, table.shape[1], dtype=torch.int32)]).contiguous()   # (two rows of no portion)
    tiles, T = tiles_of(portions)
    padded = []
    for i, t in enumerate(tiles.tolist()):
        padded += [[4, t[1], 0, 300], [t[0], t[1], 0, t[3]], t][i % 3:]
    padded += [[3, T, 0, 37], [0, T, 0, 300], [2, T, 0, 271], [1, 0, -1, 20]] * 3
    qkv = torch.randn(T, (n_q + 2 * n_kv) * D, generator=torch.Generator().manual_seed(7)).to(BF)
    out = torch.full((T + 1, n_q * D), float("nan"), dtype=BF, device=cuda)
    work = torch.full((lib.prefill_attn_q4_workspace(*table.shape, n_kv, D),), 0xFF, dtype=torch.uint8, device=cuda)
    lib.check(lib.load().b200q_prefill_attn_set_route(route))
    try:
        lib.prefill_attn_q4(qkv.to(cuda), out, cache.to(cuda), table.to(cuda), torch.tensor(padded, dtype=torch.int32, device=cuda), n_q, n_kv, D, BS,
                            D ** -0.5, work, window=window)
    finally:
        lib.check(lib.load().b200q_prefill_attn_set_route(-1))
    got, at = out.cpu(), 0
    assert torch.isnan(got[T].float()).all()
    for i, (n, past) in enumerate(portions):
        q = qkv[at: at + n, : n_q * D].view(n, n_q, D)
        ref, weight, sz = attention(q, *rows[i], torch.arange(past, past + n), D ** -0.5, 0.0, window)
        attention_close(got[at: at + n].view(n, n_q, D), ref, weight, sz, D, 2.0 ** -8, f"portion {i}")
        at += n
    assert lib.load().b200q_wait_failures() == 0


def test_captured_and_on_another_stream(cuda):
    """a write and the attention behind it, captured once and replayed over other inputs, beside the same on a stream of its own"""
    from llmq_b200 import lib
    D, n_q, n_kv, B = 128, 8, 2, 3
    ctxs = [40, 17, 300]
    cache, table, _ = make_cache(ctxs, n_kv, D, seed=11)
    table = torch.cat([table, torch.zeros(B, 1, dtype=torch.int32)], 1).contiguous()
    cos_sin = torch.randn(400, D, generator=torch.Generator().manual_seed(2)).to(BF).to(cuda)
    g = torch.Generator().manual_seed(4)
    steps = [torch.randn(B, (n_q + 2 * n_kv) * D, generator=g).to(BF) for _ in range(3)]

    def state():
        return {"cache": cache.to(cuda), "table": table.to(cuda), "qkv": torch.zeros(B, (n_q + 2 * n_kv) * D, dtype=BF, device=cuda),
                "ctx": torch.tensor(ctxs, dtype=torch.int32, device=cuda), "pos": torch.zeros(B, dtype=torch.int32, device=cuda),
                "slot": torch.zeros(B, dtype=torch.int32, device=cuda), "out": torch.zeros(B, n_q * D, dtype=BF, device=cuda)}

    def call(s, **kw):
        lib.rope_kvwrite_q4(s["qkv"], cos_sin, s["pos"], s["slot"], s["cache"], n_q, n_kv, D, BS, **kw)
        lib.decode_attn_q4(s["qkv"], s["out"], s["cache"], s["table"], s["ctx"], n_q, n_kv, D, BS, D ** -0.5, **kw)

    def place(s, x, lens):   # a token in the place of the last one
        s["qkv"].copy_(x)
        s["ctx"].copy_(torch.tensor(lens, dtype=torch.int32))
        s["pos"].copy_(torch.tensor([n - 1 for n in lens], dtype=torch.int32))
        s["slot"].copy_(torch.tensor([int(table[i, (n - 1) // 16]) * 16 + (n - 1) % 16 for i, n in enumerate(lens)], dtype=torch.int32))

    a, b = state(), state()
    place(a, steps[0], ctxs)
    call(a)
    torch.cuda.synchronize()
    a = state()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(a)
    other = torch.cuda.Stream()
    for k, x in enumerate(steps):
        lens = [n - k for n in ctxs]
        place(a, x, lens)
        place(b, x, lens)
        torch.cuda.synchronize()
        graph.replay()
        call(b, stream=other)
        torch.cuda.synchronize()
        for name in ("out", "cache", "qkv"):
            assert torch.equal(a[name].view(torch.uint8), b[name].view(torch.uint8)), name


@pytest.mark.parametrize("window", [-1, 2 ** 31 - 1, 5000, 4999])
def test_wide_windows(cuda, window):
    """windows that hide nothing, or one key"""
    from llmq_b200 import lib
    D, n_q, n_kv, ctxs = 128, 4, 1, [5000, 3, 0]
    cache, table, rows = make_cache(ctxs, n_kv, D, seed=8)
    qkv = torch.randn(3, (n_q + 2 * n_kv) * D, generator=torch.Generator().manual_seed(7)).to(BF)
    out = torch.full((3, n_q * D), float("nan"), dtype=BF, device=cuda)
    lib.decode_attn_q4(qkv.to(cuda), out, cache.to(cuda), table.to(cuda), torch.tensor(ctxs, dtype=torch.int32, device=cuda), n_q, n_kv, D, BS, D ** -0.5,
                       window=window)
    got = out.cpu()
    assert (got[2] == 0).all()
    for i in (0, 1):
        ref, weight, size = attention(qkv[i: i + 1, : n_q * D].view(1, n_q, D), *rows[i], torch.tensor([ctxs[i] - 1]), D ** -0.5, 0.0, max(window, 0))
        attention_close(got[i].view(1, n_q, D), ref, weight, size, D, 2.0 ** -11)


@pytest.mark.parametrize("D,n_q,n_kv", [(64, 8, 2), (256, 4, 1)])
def test_two_calls_at_once(cuda, D, n_q, n_kv):
    """long contexts, whose pieces lie in scratch: two threads on streams of their own, then two graphs replayed side by side, each time
    beside the same calls one after the other"""
    import threading
    from llmq_b200 import lib
    sets = [[5000, 33, 9000], [12000, 700]]
    args = []
    for k, ctxs in enumerate(sets):
        cache, table, _ = make_cache(ctxs, n_kv, D, seed=k)
        qkv = torch.randn(len(ctxs), (n_q + 2 * n_kv) * D, generator=torch.Generator().manual_seed(k)).to(BF)
        args.append((qkv.to(cuda), cache.to(cuda), table.to(cuda), torch.tensor(ctxs, dtype=torch.int32, device=cuda)))

    def call(k, out, stream=None):
        q, cache, table, ctx = args[k]
        lib.decode_attn_q4(q, out, cache, table, ctx, n_q, n_kv, D, BS, D ** -0.5, stream=stream)

    def outs():
        return [[torch.zeros(len(c), n_q * D, dtype=BF, device=cuda) for _ in range(20)] for c in sets]

    alone = [o[0] for o in outs()]
    for k in (0, 1):
        call(k, alone[k])
        torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], outs()
    torch.cuda.synchronize()
    threads = [threading.Thread(target=lambda k=k: [call(k, o, streams[k]) for o in got[k]]) for k in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for k in (0, 1):
        assert all(torch.equal(o, alone[k]) for o in got[k])
    graphs, got = [torch.cuda.CUDAGraph() for _ in sets], outs()
    for k in (0, 1):
        with torch.cuda.graph(graphs[k]):
            for o in got[k]:
                call(k, o)
    for _ in range(2):
        for k in (0, 1):
            for o in got[k]:
                o.zero_()
        torch.cuda.synchronize()
        for k in (0, 1):
            with torch.cuda.stream(streams[k]):
                graphs[k].replay()
        torch.cuda.synchronize()
        for k in (0, 1):
            assert all(torch.equal(o, alone[k]) for o in got[k])


def test_portions_of_one_sequence(cuda):
    """a prompt whose portions are apart in the step: each sees the keys up to its own tokens, the same as in a step of its own"""
    from llmq_b200 import lib
    D, n_q, n_kv = 128, 8, 2
    cache, table, rows = make_cache([400, 90], n_kv, D, seed=3)
    portions = [(0, 0, 33), (1, 40, 50), (0, 33, 100), (0, 300, 100)]   # sequence, past, tokens
    tiles, T = [], 0
    for s, past, n in portions:
        tiles += [[s, T + j, min(16, n - j), past + j] for j in range(0, n, 16)]
        T += n
    qkv = torch.randn(T, (n_q + 2 * n_kv) * D, generator=torch.Generator().manual_seed(7)).to(BF)
    out = torch.full((T, n_q * D), float("nan"), dtype=BF, device=cuda)
    work = torch.full((lib.prefill_attn_q4_workspace(*table.shape, n_kv, D),), 0xFF, dtype=torch.uint8, device=cuda)
    for window in (0, 20):
        lib.prefill_attn_q4(qkv.to(cuda), out, cache.to(cuda), table.to(cuda), torch.tensor(tiles, dtype=torch.int32, device=cuda), n_q, n_kv, D, BS,
                            D ** -0.5, work, window=window)
        got, at = out.cpu(), 0
        for s, past, n in portions:
            q = qkv[at: at + n, : n_q * D].view(n, n_q, D)
            ref, weight, sz = attention(q, *rows[s], torch.arange(past, past + n), D ** -0.5, 0.0, window)
            attention_close(got[at: at + n].view(n, n_q, D), ref, weight, sz, D, 2.0 ** -8, f"portion at {past}")
            at += n


@pytest.mark.parametrize("D,n_q,n_kv", [(64, 8, 2), (64, 7, 1), (128, 8, 8), (128, 8, 1), (128, 6, 2), (256, 8, 2), (256, 8, 1)])
@pytest.mark.parametrize("ctxs", CASES + [[300, 0, 5000], [7001]], ids=lambda c: f"{len(c)}x{max(c)}")
@pytest.mark.parametrize("cap,window", [(0.0, 0), (20.0, 100), (0.0, 1), (0.0, 3000)])
def test_decode_clusters(cuda, D, n_q, n_kv, ctxs, cap, window):
    """few sequences, a cluster to each head: any number of CTAs and pages, tables wider than the lengths"""
    from llmq_b200 import lib
    cache, table, rows = make_cache(ctxs, n_kv, D, seed=len(ctxs) + D)
    B = len(ctxs)
    qkv = torch.randn(B, (n_q + 2 * n_kv) * D, generator=torch.Generator().manual_seed(9)).to(BF)
    wide = torch.cat([table, torch.full((B, 60), 2 ** 30, dtype=torch.int32)], 1).contiguous()   # (numbers that no length counts)
    for bt in (table, wide):
        out = torch.full((B + 1, n_q * D), float("nan"), dtype=BF, device=cuda)
        lib.decode_attn_q4_set_whole(-2)
        try:
            lib.decode_attn_q4(qkv.to(cuda), out, cache.to(cuda), bt.to(cuda), torch.tensor(ctxs, dtype=torch.int32, device=cuda), n_q, n_kv, D, BS,
                               D ** -0.5, softcap=cap, window=window)
        finally:
            lib.decode_attn_q4_set_whole(-1)
        got = out.cpu()
        assert torch.isnan(got[B].float()).all()
        for i, c in enumerate(ctxs):
            if c == 0:
                assert (got[i] == 0).all()
                continue
            ref, weight, size = attention(qkv[i: i + 1, : n_q * D].view(1, n_q, D), *rows[i], torch.tensor([c - 1]), D ** -0.5, cap, window)
            attention_close(got[i].view(1, n_q, D), ref, weight, size, D, 2.0 ** -11, f"ctx {c}")


@pytest.mark.parametrize("way", [-2, 0, 1])
def test_ways_of_sharing(cuda, way):
    """sizes and growth of scores, NaN, far pages and two calls at once, whichever way the work is shared"""
    from llmq_b200 import lib
    lib.decode_attn_q4_set_whole(way)
    try:
        test_decode_sizes_of_values(cuda, 128, 8, 2, 1e4, 1.0, 1e-5)
        test_decode_sizes_of_values(cuda, 256, 2, 1, 1e-6, 30.0, 1e4)
        for D in (64, 128, 256):
            test_decode_growing_scores(cuda, D)
        test_decode_far_pages_and_many_rows(cuda)
        test_two_calls_at_once(cuda, 64, 8, 2)
        test_wide_windows(cuda, 4999)
    finally:
        lib.decode_attn_q4_set_whole(-1)


@pytest.mark.parametrize("what", ["attention", "products"])
def test_each_threads_own_stream(cuda, what):
    """cudaStreamPerThread is one handle and a stream for each thread: pieces and parts of two threads do not meet"""
    import threading
    from types import SimpleNamespace
    from llmq_b200 import lib
    own = SimpleNamespace(cuda_stream=2)   # (the handle)
    g = torch.Generator().manual_seed(2)
    if what == "attention":
        D, n_q, n_kv, args = 64, 8, 2, []
        for k, ctxs in enumerate([[5000, 33, 9000], [12000, 700]]):
            cache, table, _ = make_cache(ctxs, n_kv, D, seed=k)
            qkv = torch.randn(len(ctxs), (n_q + 2 * n_kv) * D, generator=g).to(BF)
            args.append((qkv.to(cuda), cache.to(cuda), table.to(cuda), torch.tensor(ctxs, dtype=torch.int32, device=cuda)))
        shape = [(len(a[0]), n_q * D) for a in args]

        def call(k, out, stream=None):
            q, cache, table, ctx = args[k]
            lib.decode_attn_q4(q, out, cache, table, ctx, n_q, n_kv, D, BS, D ** -0.5, stream=stream)
    else:
        args = [(torch.randn(256, 8192, generator=g).to(BF).to(cuda), torch.randn(512, 8192, generator=g).to(BF).to(cuda)) for _ in range(2)]
        assert lib.gemm_bf16_splitk(*args[0])[1] > 1
        shape = [(256, 512)] * 2

        def call(k, out, stream=None):
            lib.gemm_bf16(*args[k], out, stream=stream)
    alone, got = ([[torch.zeros(*s, dtype=BF, device=cuda) for _ in range(n)] for s in shape] for n in (1, 20))
    lib.decode_attn_q4_set_whole(0)
    try:
        for k in (0, 1):
            call(k, alone[k][0])
            torch.cuda.synchronize()
        threads = [threading.Thread(target=lambda k=k: [call(k, o, own) for o in got[k]]) for k in (0, 1)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
    finally:
        lib.decode_attn_q4_set_whole(-1)
    for k in (0, 1):
        assert all(torch.equal(o, alone[k][0]) for o in got[k])


@pytest.mark.parametrize("D,n_q,n_kv", [(64, 8, 2), (128, 8, 1), (256, 4, 1)])
def test_without_memory_for_pieces(cuda, D, n_q, n_kv):
    """items go to warps whole where scratch is refused, in a call and in a capture, and are shared again in the next call"""
    from llmq_b200 import lib
    ctxs = [5000, 33, 0, 900]
    cache, table, rows = make_cache(ctxs, n_kv, D, seed=D)
    qkv = torch.randn(len(ctxs), (n_q + 2 * n_kv) * D, generator=torch.Generator().manual_seed(7)).to(BF)
    args = (cache.to(cuda), table.to(cuda), torch.tensor(ctxs, dtype=torch.int32, device=cuda), n_q, n_kv, D, BS, D ** -0.5)
    q = qkv.to(cuda)
    outs = [torch.full((len(ctxs), n_q * D), float("nan"), dtype=BF, device=cuda) for _ in range(4)]
    graph = torch.cuda.CUDAGraph()
    try:
        for way, out in ((1, outs[0]), (-3, outs[1]), (0, outs[2])):
            lib.decode_attn_q4_set_whole(way)
            lib.decode_attn_q4(q, out, *args)
        lib.decode_attn_q4_set_whole(-3)
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            lib.decode_attn_q4(q, outs[3], *args)
        graph.replay()
        torch.cuda.synchronize()
    finally:
        lib.decode_attn_q4_set_whole(-1)
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[3])
    for i, c in enumerate(ctxs):
        if c == 0:
            assert all((o[i] == 0).all() for o in outs)
            continue
        ref, weight, size = attention(qkv[i: i + 1, : n_q * D].view(1, n_q, D), *rows[i], torch.tensor([c - 1]), D ** -0.5)
        for o in outs:
            attention_close(o[i].view(1, n_q, D), ref, weight, size, D, 2.0 ** -11, f"ctx {c}")


@pytest.mark.parametrize("D,n_q,n_kv", [(64, 8, 2), (256, 4, 1)])
def test_pieces_of_calls_at_once(cuda, D, n_q, n_kv):
    """calls whose pieces lie in scratch: on streams of their own and in graphs, then from two threads on one stream"""
    import threading
    from llmq_b200 import lib
    lib.decode_attn_q4_set_whole(0)
    try:
        test_two_calls_at_once(cuda, D, n_q, n_kv)
        args = []
        for k, ctxs in enumerate([[5000, 33, 9000], [12000, 700]]):
            cache, table, _ = make_cache(ctxs, n_kv, D, seed=k)
            qkv = torch.randn(len(ctxs), (n_q + 2 * n_kv) * D, generator=torch.Generator().manual_seed(k)).to(BF)
            args.append((qkv.to(cuda), cache.to(cuda), table.to(cuda), torch.tensor(ctxs, dtype=torch.int32, device=cuda)))
        stream = torch.cuda.Stream()

        def call(k, out):
            q, cache, table, ctx = args[k]
            lib.decode_attn_q4(q, out, cache, table, ctx, n_q, n_kv, D, BS, D ** -0.5, stream=stream)

        alone, got = ([[torch.zeros(len(a[0]), n_q * D, dtype=BF, device=cuda) for _ in range(n)] for a in args] for n in (1, 40))
        torch.cuda.synchronize()
        for k in (0, 1):
            call(k, alone[k][0])
            torch.cuda.synchronize()
        threads = [threading.Thread(target=lambda k=k: [call(k, o) for o in got[k]]) for k in (0, 1)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        for k in (0, 1):
            assert all(torch.equal(o, alone[k][0]) for o in got[k])
    finally:
        lib.decode_attn_q4_set_whole(-1)


@pytest.mark.parametrize("D,n_q,n_kv", [(64, 8, 2), (256, 4, 1)])
@pytest.mark.parametrize("window", [0, 40])
def test_prompts_of_few_rows_of_a_large_table(cuda, D, n_q, n_kv, window):
    """an engine's table: a row for every slot and columns up to the model's length, of which the step's portions see a few; the others hold
    whatever they do"""
    from llmq_b200 import lib
    portions, at_rows = [(5, 11), (133, 0), (70, 900)], [63, 5, 40]
    cache, small, rows = make_cache([n + past for n, past in portions], n_kv, D, seed=D)
    table = torch.full((64, 512), 2 ** 30, dtype=torch.int32)
    for i, r in enumerate(at_rows):
        held_pages = (sum(portions[i]) + 15) // 16
        table[r, :held_pages] = small[i, :held_pages]
    tiles, T = tiles_of(portions)
    tiles[:, 0] = torch.tensor(at_rows, dtype=torch.int32)[tiles[:, 0].long()]
    qkv = torch.randn(T, (n_q + 2 * n_kv) * D, generator=torch.Generator().manual_seed(7)).to(BF)
    out = torch.full((T, n_q * D), float("nan"), dtype=BF, device=cuda)
    work = torch.full((lib.prefill_attn_q4_workspace(*table.shape, n_kv, D),), 0xFF, dtype=torch.uint8, device=cuda)
    lib.prefill_attn_q4(qkv.to(cuda), out, cache.to(cuda), table.to(cuda), tiles.to(cuda), n_q, n_kv, D, BS, D ** -0.5, work, window=window)
    got, at = out.cpu(), 0
    for i, (n, past) in enumerate(portions):
        q = qkv[at: at + n, : n_q * D].view(n, n_q, D)
        ref, weight, sz = attention(q, *rows[i], torch.arange(past, past + n), D ** -0.5, 0.0, window)
        attention_close(got[at: at + n].view(n, n_q, D), ref, weight, sz, D, 2.0 ** -8, f"portion {i}")
        at += n
    assert lib.load().b200q_wait_failures() == 0


@pytest.mark.parametrize("D", [64, 256])
@pytest.mark.parametrize("way", [-1, -2, 0, 1])
def test_table_of_no_columns(cuda, D, way):
    """sequences of no tokens, and of any by a table that holds none: zeros"""
    from llmq_b200 import lib
    n_q, n_kv, B = 4, 2, 3
    qkv = torch.randn(B, (n_q + 2 * n_kv) * D, generator=torch.Generator().manual_seed(7)).to(BF).to(cuda)
    out = torch.full((B + 1, n_q * D), float("nan"), dtype=BF, device=cuda)
    cache, table = torch.zeros(0, n_kv, 18 * D, dtype=torch.uint8, device=cuda), torch.zeros(B, 0, dtype=torch.int32, device=cuda)
    lib.decode_attn_q4_set_whole(way)
    try:
        lib.decode_attn_q4(qkv, out, cache, table, torch.tensor([0, 5, 0], dtype=torch.int32, device=cuda), n_q, n_kv, D, BS, D ** -0.5)
    finally:
        lib.decode_attn_q4_set_whole(-1)
    assert (out[:B] == 0).all() and torch.isnan(out[B].float()).all()

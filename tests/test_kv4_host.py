"""What the calls of the 4-bit cache, of beams and of their pages refuse: arguments are looked at before anything is launched."""
import pytest

P = 1 << 20   # an address that nobody reads: a multiple of every alignment


def refused(rc, word):
    from llmq_b200 import lib
    assert rc == -1
    assert word in lib.load().b200q_last_error().decode()


def test_sizes():
    from llmq_b200 import lib
    assert lib.kv4_page_bytes(8, 128) == 18 * 128 * 8
    assert lib.prefill_attn_q4_workspace(3, 5, 8, 128) == 15 * 4 * 8 * 16 * 128 + 256
    assert lib.prefill_attn_q4_workspace(0, 5, 8, 128) == 0
    assert lib.beam_select_workspace(1, 4, 128256, 8) > 0
    for call in (lambda: lib.kv4_page_bytes(0, 128), lambda: lib.kv4_page_bytes(8, 96), lambda: lib.prefill_attn_q4_workspace(-1, 1, 1, 64),
                 lambda: lib.beam_select_workspace(1, 33, 100, 40), lambda: lib.beam_select_workspace(1, 4, 100, 65)):
        with pytest.raises(lib.B200QError):
            call()


@pytest.mark.parametrize("change,word", [(dict(D=96), "D=96"), (dict(block=32), "bs=32"), (dict(n_kv=0), "n_kv=0"), (dict(T=-1), "T=-1"),
                                         (dict(cache=P + 8), "aligned"), (dict(qkv=0), "null")])
def test_write(change, word):
    from llmq_b200 import lib
    a = dict(qkv=P, cos=P, pos=P, slot=P, cache=P, T=4, n_q=8, n_kv=2, D=128, block=16, **{})
    a.update(change)
    refused(lib.load().b200q_rope_kvwrite_q4(*a.values(), 0), word)


@pytest.mark.parametrize("change,word", [(dict(D=96), "D=96"), (dict(block=8), "bs=8"), (dict(out=0), "null"), (dict(out=P + 4), "aligned"), (dict(n=-1), "n_pages")])
def test_unpack(change, word):
    from llmq_b200 import lib
    a = dict(cache=P, pages=P, n=4, out=P, n_kv=2, D=64, block=16)
    a.update(change)
    refused(lib.load().b200q_kv4_unpack(*a.values(), 0), word)


@pytest.mark.parametrize("change,word", [(dict(D=32), "D=32"), (dict(n_q=18), "GQA"), (dict(n_q=7), "n_q=7"), (dict(block=32), "block"), (dict(q=P + 2), "aligned"),
                                         (dict(stride=1028), "q_stride"), (dict(stride=64), "q_stride"), (dict(ctx=0), "null"), (dict(bt=-1), "bt_stride")])
def test_decode(change, word):
    from llmq_b200 import lib
    a = dict(q=P, stride=1024, out=P, cache=P, table=P, bt=4, ctx=P, n=2, n_q=4, n_kv=2, D=128, block=16, scale=1.0, cap=0.0, window=0)
    a.update(change)
    refused(lib.load().b200q_decode_attn_q4(*a.values(), 0), word)
    assert lib.load().b200q_decode_attn_q4_set_whole(2) == -1


@pytest.mark.parametrize("n,bt,n_kv", [(64, 1 << 26, 2), (4, 1 << 26, 32), (4000, 1 << 20, 512), ((1 << 31) - 1, 1, 2)])
def test_decode_of_too_many_pages(n, bt, n_kv):
    """tables beyond what the kernel's own counts hold"""
    from llmq_b200 import lib
    refused(lib.load().b200q_decode_attn_q4(P, 128 * n_kv, P, P, P, bt, P, n, n_kv, n_kv, 128, 16, 1.0, 0.0, 0, 0), "too much at once")


@pytest.mark.parametrize("change,word", [(dict(D=256, n_q=16), "GQA"), (dict(n_q=18), "GQA"), (dict(bytes=100), "too small"), (dict(work=P + 128), "aligned"),
                                         (dict(rows=70000), "table"), (dict(work=0), "null"), (dict(block=1), "block_size=1")])
def test_prompts(change, word):
    from llmq_b200 import lib
    a = dict(q=P, stride=4096, out=P, cache=P, table=P, bt=4, rows=3, tiles=P, n_tiles=2, n_q=4, n_kv=2, D=128, block=16, scale=1.0, cap=0.0, window=0,
             work=P, bytes=1 << 30)
    a.update(change)
    refused(lib.load().b200q_prefill_attn_q4(*a.values(), 0), word)


@pytest.mark.parametrize("change,word", [(dict(beams=33), "beams=33"), (dict(K=3), "K=3"), (dict(K=65), "K=65"), (dict(V=7), "V=7"), (dict(stops=0), "null"),
                                         (dict(work=0), "null"), (dict(bytes=16), "too small"), (dict(work=P + 8), "aligned"), (dict(beams=0), "beams=0"), (dict(logits=P + 2), "aligned")])
def test_beams(change, word):
    from llmq_b200 import lib
    a = dict(logits=P, scores=P, groups=2, beams=4, V=1000, stops=P, n_stops=1, K=8, cs=P, ct=P, cr=P, ns=P, nt=P, nr=P, work=P, bytes=1 << 20)
    a.update(change)
    refused(lib.load().b200q_beam_select(*a.values(), 0), word)


@pytest.mark.parametrize("change,word", [(dict(n_old=20000), "n_old"), (dict(n_new=20000), "n_new"), (dict(block=32), "block_size"), (dict(out=P + 64), "overlap"),
                                         (dict(out=P), "overlap"), (dict(status=0), "null"), (dict(pairs=P + 4), "aligned"), (dict(blocks=0), "num_blocks")])
def test_fork(change, word):
    from llmq_b200 import lib
    a = dict(table=P, lens=P, n_old=4, parents=P, n_new=4, stride=8, refs=P, blocks=100, block=16, out=2 * P, slots=P, pairs=P, status=P)
    a.update(change)
    refused(lib.load().b200q_pages_fork(*a.values(), 0), word)


def test_free_copy_compact():
    from llmq_b200 import lib
    h = lib.load()
    refused(h.b200q_pages_free(P, P, 0, 4, 8, P, 0, 16, 0), "num_blocks")
    refused(h.b200q_pages_free(P, 0, 0, 4, 8, P, 100, 16, 0), "null")
    refused(h.b200q_pages_copy(P, P, 4, 0, 100, 2, 1600, 16, 0), "page_bytes=100")
    refused(h.b200q_pages_copy(P, P, 4, 0, 96, 2, 1500, 16, 0), "layer_stride")
    refused(h.b200q_pages_copy(P + 8, P, 4, 0, 96, 2, 1536, 16, 0), "aligned")
    refused(h.b200q_pages_copy(0, P, 4, 0, 96, 2, 1536, 16, 0), "null")
    refused(h.b200q_pages_compact(P, P, 4, 8, P, 100, 8, P, P, P, P, P, 0), "block_size")
    refused(h.b200q_pages_compact(P, P, 4, 8, P, 100, 16, P, P, 0, P, P, 0), "null")


def test_nothing_to_do():
    """calls over nothing return without a launch, whatever the pointers are"""
    from llmq_b200 import lib
    h = lib.load()
    assert h.b200q_rope_kvwrite_q4(0, 0, 0, 0, 0, 0, 8, 2, 128, 16, 0) == 0
    assert h.b200q_kv4_unpack(0, 0, 0, 0, 2, 128, 16, 0) == 0
    assert h.b200q_decode_attn_q4(0, 1024, 0, 0, 0, 4, 0, 0, 8, 2, 128, 16, 1.0, 0.0, 0, 0) == 0
    assert h.b200q_prefill_attn_q4(0, 1024, 0, 0, 0, 4, 3, 0, 0, 8, 2, 128, 16, 1.0, 0.0, 0, 0, 0, 0) == 0
    assert h.b200q_beam_select(0, 0, 0, 4, 1000, 0, 0, 8, 0, 0, 0, 0, 0, 0, 0, 0, 0) == 0
    assert h.b200q_pages_free(0, 0, 0, 0, 8, 0, 100, 16, 0) == 0
    assert h.b200q_pages_copy(0, 0, 0, 0, 96, 2, 1536, 16, 0) == 0


def test_tensors_are_looked_at():
    """types, shapes and devices of tensors, before their addresses are taken"""
    import torch

    from llmq_b200 import lib
    with pytest.raises(ValueError, match="int32"):
        lib._arg(torch.zeros(3, dtype=torch.int64), "i", "x")
    with pytest.raises(ValueError, match="CUDA"):
        lib._arg(torch.zeros(3, dtype=torch.int32), "i", "x")


def test_caches_and_outputs_are_looked_at(monkeypatch):
    """a cache that is no whole number of pages, and outputs with fewer rows than there are queries, before anything is called"""
    import torch

    from llmq_b200 import lib
    called = []

    class Calls:
        def __getattr__(self, name):
            return lambda *a: called.append(name) or 0
    monkeypatch.setattr(lib, "load", Calls)
    monkeypatch.setattr(lib, "_here", lambda stream: (0, -1))   # (tensors of the CPU are on device -1)
    n_q, n_kv, D, T = 4, 2, 64, 5
    bf = dict(dtype=torch.bfloat16)
    i32 = dict(dtype=torch.int32)
    page = 18 * n_kv * D
    qkv, cos_sin, rows = torch.zeros(T, (n_q + 2 * n_kv) * D, **bf), torch.zeros(9, D, **bf), torch.zeros(T, **i32)
    table, tiles, work = torch.zeros(T, 3, **i32), torch.zeros(2, 4, **i32), torch.zeros(8, dtype=torch.uint8)
    back = torch.zeros(T, 2 * n_kv * 16 * D, **bf)

    def write(kv):
        lib.rope_kvwrite_q4(qkv, cos_sin, rows, rows, kv, n_q, n_kv, D, 16)

    def unpack(kv):
        lib.kv4_unpack(kv, rows, back, n_kv, D, 16)

    def decode(kv, n=T):
        lib.decode_attn_q4(qkv, torch.zeros(n, n_q * D, **bf), kv, table, rows, n_q, n_kv, D, 16, 1.0)

    def prompts(kv, n=T):
        lib.prefill_attn_q4(qkv, torch.zeros(n, n_q * D, **bf), kv, table, tiles, n_q, n_kv, D, 16, 1.0, work)

    for call in (write, unpack, decode, prompts):
        for size in (page + 16, 3 * page - 1, 18 * D):
            with pytest.raises(ValueError, match="whole number of pages"):
                call(torch.zeros(size, dtype=torch.uint8))
    for call in (decode, prompts):
        with pytest.raises(ValueError, match="out"):
            call(torch.zeros(page, dtype=torch.uint8), T - 1)
    assert not called
    for call in (write, unpack, decode, prompts):
        for kv in (torch.zeros(3, n_kv, 18 * D, dtype=torch.uint8), torch.zeros(page // 4, **i32), torch.zeros(0, dtype=torch.uint8)):
            call(kv)
    decode(torch.zeros(page, dtype=torch.uint8), T + 1)
    prompts(torch.zeros(page, dtype=torch.uint8), T + 1)
    assert len(called) == 14

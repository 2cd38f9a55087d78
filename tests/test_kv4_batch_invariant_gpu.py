"""B200Q_BATCH_INVARIANT=1 over the 4-bit cache: bit for bit, a sequence's single token and a prompt's rows do not depend on what else is in the
step, nor on how wide the block table is.  The variable is read once, so the checks run in a process of their own."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.gpu
@pytest.mark.parametrize("what", ["prompts", "tokens"])
def test_same_bits_whatever_the_batch(cuda, what):
    env = dict(os.environ, B200Q_BATCH_INVARIANT="1", PYTHONPATH=ROOT + os.pathsep + os.environ.get("PYTHONPATH", ""))
    r = subprocess.run([sys.executable, os.path.abspath(__file__), what], env=env, cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "equal" in r.stdout, r.stdout + r.stderr


def prompts():
    import torch

    from llmq_b200 import lib
    from tests.kv4_util import BF, BS, make_cache
    for D, n_q, n_kv, cap, window in [(64, 8, 2, 0.0, 0), (128, 8, 8, 0.0, 100), (256, 4, 2, 20.0, 0)]:
        portions = [(0, 300), (0, 100), (40, 77), (0, 700), (500, 130), (0, 20), (0, 9)] + [(0, 33)] * 20
        cache, table, _ = make_cache([a + n for a, n in portions], n_kv, D, 5)
        cache, table = cache.cuda(), table.cuda()
        qkv = [torch.randn(n, (n_q + 2 * n_kv) * D, generator=torch.Generator().manual_seed(i)).to(BF).cuda() for i, (_, n) in enumerate(portions)]

        def run(which, columns):
            tiles, row = [], 0
            for k, i in enumerate(which):
                a, n = portions[i]
                tiles += [[k, row + j, min(16, n - j), a + j] for j in range(0, n, 16)]
                row += n
            out, bt = torch.empty(row, n_q * D, dtype=BF, device="cuda"), table[list(which), :columns].contiguous()
            work = torch.empty(lib.prefill_attn_q4_workspace(*bt.shape, n_kv, D), dtype=torch.uint8, device="cuda")
            lib.prefill_attn_q4(torch.cat([qkv[i] for i in which]), out, cache, bt, torch.tensor(tiles, dtype=torch.int32, device="cuda"), n_q, n_kv, D,
                                BS, 0.3, work, softcap=cap, window=window)
            parts, row = {}, 0
            for i in which:
                parts[i] = out[row: row + portions[i][1]].view(torch.int16)
                row += portions[i][1]
            return parts
        together, turned = run(range(len(portions)), table.shape[1]), run([6, 5, 4, 3, 2, 1, 0], table.shape[1])
        for i in range(7):
            alone = run([i], (sum(portions[i]) + 15) // 16)[i]
            assert torch.equal(alone, together[i]) and torch.equal(alone, turned[i]), (D, n_kv, window, portions[i])


def tokens():
    import torch

    from llmq_b200 import lib
    from tests.kv4_util import BF, BS, make_cache
    for D, n_q, n_kv, cap, window in [(64, 32, 8, 0.0, 0), (128, 8, 8, 0.0, 300), (128, 16, 2, 0.0, 0), (256, 16, 8, 20.0, 0)]:
        ctxs = [700, 1, 64, 130, 1500, 0] + [40] * 294
        cache, table, _ = make_cache(ctxs, n_kv, D, 6)
        cache, table = cache.cuda(), table.cuda()
        qkv = torch.randn(len(ctxs), (n_q + 2 * n_kv) * D, generator=torch.Generator().manual_seed(3)).to(BF).cuda()

        def run(lo, hi, columns):
            out = torch.empty(hi - lo, n_q * D, dtype=BF, device="cuda")
            lib.decode_attn_q4(qkv[lo:hi], out, cache, table[lo:hi, :columns].contiguous(), torch.tensor(ctxs[lo:hi], dtype=torch.int32, device="cuda"),
                               n_q, n_kv, D, BS, D ** -0.5, softcap=cap, window=window)
            return out.view(torch.int16)
        full = run(0, len(ctxs), table.shape[1])
        for i in range(6):
            assert torch.equal(run(i, i + 1, (ctxs[i] + 15) // 16)[0], full[i]), (D, ctxs[i])
        assert torch.equal(run(0, 20, table.shape[1]), full[:20])


if __name__ == "__main__":
    {"prompts": prompts, "tokens": tokens}[sys.argv[1]]()
    print("equal")

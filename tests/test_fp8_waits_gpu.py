"""Products in 8 bits whose warps of products give up: before their first block, within the ring's first round and behind it.  The call ends and says
so, large tiles leave the outputs that they have no sums for as they are, and the next calls are right."""
import os
import subprocess
import sys

import pytest
import torch

from tests.fp8_util import BF, F8, product, product_off, random_held, tile_table

pytestmark = pytest.mark.gpu
# mode (b200q_gemm_fp8_set_mode), rows, columns, length of the reduction
DENSE = [(1, 3, 256, 1024), (1, 100, 512, 4096), (2, 200, 512, 2048), (22, 200, 512, 2048), (3, 300, 512, 2048), (33, 300, 400, 2048), (204, 130, 512, 4096),
         (424, 130, 512, 4096), (334, 130, 512, 4096), (205, 300, 512, 4096), (3, 2100, 9216, 2304)]
GATED = [(1, 3, 512, 1024), (1, 48, 512, 4096), (2, 200, 512, 2048), (3, 300, 512, 2048), (3, 2100, 9216, 2304)]


def cases(wanted):
    """every product, as (call, its output, what it has to be, how far it may be off)"""
    from llmq_b200 import lib
    g = torch.Generator(device="cuda").manual_seed(1)
    for which, M, N, K in DENSE if wanted == "dense" else ():
        (a, sa), (w, sw) = random_held(g, M, K, 1), random_held(g, N, K, 128)
        c = torch.empty(M, N, dtype=BF if M % 8 else torch.float32, device="cuda")
        ref, size = product(a, sa, w, sw)
        yield f"{which}: {M} x {N} x {K}", which, lambda: lib.gemm_fp8(a, sa, w, sw, c), c, ref, product_off(size, K) + ref.abs() * 2.0 ** -8
    for which, M, N, K in GATED if wanted == "gated" else ():
        (a, sa), (w, sw) = random_held(g, M, K, 1), random_held(g, N, K, 128)
        y, ys = torch.empty(M, N // 2, dtype=F8, device="cuda"), lib.fp8_row_scales(M, N // 2)
        call = lambda: lib.gemm_gated_fp8(a, sa / 60, w, sw * (2 / 60 * K ** -0.5), y, ys)
        lib.gemm_fp8_set_mode(which)
        ys.zero_()
        call()
        yield f"gated {which}: {M} x {N} x {K}", which, call, ys[:, :M], ys[:, :M].double(), 0.0
    for gated in (False, True) if wanted == "experts" else ():
        loads, N, K = [200, 0, 5, 128, 31], 512, 2048
        a, sa = random_held(g, sum(loads), K, 1)
        held = [random_held(g, N, K, 128) for _ in loads]
        w, sw = torch.stack([h[0].view(torch.uint8) for h in held]).view(F8), torch.stack([h[1] for h in held])
        tab, n = tile_table(loads)
        out = lib.fp8_row_scales(sum(loads), N // 2) if gated else torch.empty(sum(loads), N, device="cuda")
        y = torch.empty(sum(loads), N // 2, dtype=F8, device="cuda")
        call = (lambda: lib.gemm_grouped_gated_fp8(a, sa, w, sw, y, out, tab, n)) if gated else (lambda: lib.gemm_grouped_fp8(a, sa, w, sw, out, tab, n))
        out.zero_()
        call()
        yield f"experts, gated {gated}", 0, call, out, out.double(), 0.0


def give_up(wanted):
    """in a process of its own: the flag stays set"""
    from llmq_b200 import lib
    L = lib.load()
    for name, which, call, out, ref, off in cases(wanted):
        lib.gemm_fp8_set_mode(which)
        call()
        torch.cuda.synchronize()
        for n in (1, 3, 12, 30):
            print(name, n, flush=True)
            L.b200q_gemm_fp8_set_give_up(n)
            out.fill_(7.0)
            for _ in range(3):
                call()
            torch.cuda.synchronize()
            assert L.b200q_wait_failures() != 0
            if which == 1:
                pass                    # (small tiles store what they have)
            elif n == 1:
                assert (out == 7.0).all(), f"{name}: outputs of a product that gave up at once"
            else:                       # (CTAs with fewer blocks are through before they give up; those of a cluster have as many here, or fewer)
                assert ((out == 7.0) | ((out.double() - ref).abs() <= off)).all(), f"{name}, {n}"
            L.b200q_gemm_fp8_set_give_up(0)
            call()
            torch.cuda.synchronize()
            assert ((out.double() - ref).abs() <= off).all(), f"{name}: not right again"
    print("right again")


@pytest.mark.parametrize("wanted", ["dense", "gated", "experts"])
def test_waits_that_run_out(cuda, wanted):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", f"from tests.test_fp8_waits_gpu import give_up; give_up({wanted!r})"], cwd=root, capture_output=True, text=True,
                       timeout=200)
    assert r.returncode == 0 and "right again" in r.stdout, r.stdout[-500:] + r.stderr[-2000:]

"""Whoever waits for a barrier in the products in 8 bits (csrc/gemm_fp8.cu) looks at what the wait says before it goes on: a role whose wait has
run out arms no barrier, starts no load and no product."""
import os
import re

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "llmq_b200", "csrc", "gemm_fp8.cu")


def test_no_wait_is_passed_over():
    with open(SOURCE) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    calls = [text[:m.start()].rstrip() for m in re.finditer(r"\bf8_wait\((?!uint64_t)", text)]
    assert len(calls) >= 4
    for before in calls:
        used = before[-1] in "=&" or before.endswith("(void)")   # (f8_await, whose callers look at the flag that a wait leaves)
        assert used, f"the outcome of a wait behind {before[-80:]!r} is not used"


def test_issuing_ends_with_a_wait_that_ran_out():
    """between a wait of a role that issues and what it issues stands the way out of its loop"""
    with open(SOURCE) as f:
        text = re.sub(r"//[^\n]*", "", f.read())
    found = 0
    for m in re.finditer(r"f8_a?wait\((?:empty|full) \+ stage", text):
        behind = text[m.end():]
        end = min((behind.find(w) for w in ("expect_tx(", "umma_fp8", "tmem_ld32(") if w in behind), default=-1)
        if behind[end:].startswith("tmem_ld32("):
            continue                    # (who only adds reads on, and does not store)
        assert "break;" in behind[:end], behind[:200]
        found += 1
    assert found == 4

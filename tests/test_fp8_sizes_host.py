"""Linear layers in 8 bits refuse sizes so close to 2^31 that rounding them up to whole blocks or tiles passes 32 bits.  (Their operands would
fit into memory: 2^31 rows or columns of 16 codes are 34 GB.)"""
import pytest

from tests.test_fp8_host import GATED, GEMM, GROUPED, GROUPED_GATED, ROWS, WEIGHT, call, refused

TOP = 1 << 31


@pytest.mark.parametrize("name,args,change,word", [
    ("b200q_gemm_fp8", GEMM, dict(M=TOP - 4, ld=TOP - 4, N=8, K=16), f"M={TOP - 4}"),
    ("b200q_gemm_fp8", GEMM, dict(M=TOP - 512, ld=TOP - 512, N=8, K=16), f"M={TOP - 512}"),
    ("b200q_gemm_fp8", GEMM, dict(N=TOP - 8, K=16), f"N={TOP - 8}"),
    ("b200q_gemm_fp8", GEMM, dict(K=TOP - 16), f"K={TOP - 16}"),
    ("b200q_gemm_gated_fp8", GATED, dict(N=TOP - 256, K=16), f"N={TOP - 256}"),
    ("b200q_gemm_gated_fp8", GATED, dict(K=TOP - 16), f"K={TOP - 16}"),
    ("b200q_gemm_grouped_fp8", GROUPED, dict(rows=TOP - 4, ld=TOP - 4, N=8, K=16), f"M={TOP - 4}"),
    ("b200q_gemm_grouped_fp8", GROUPED, dict(groups=(TOP - 8) // 264, N=264, K=16), f"groups={(TOP - 8) // 264}"),
    ("b200q_gemm_grouped_gated_fp8", GROUPED_GATED, dict(groups=TOP // 512 - 1, N=512, K=16), f"groups={TOP // 512 - 1}"),
    ("b200q_quantize_fp8", ROWS, dict(T=1, K=TOP - 16, ld_x=TOP), f"K={TOP - 16}"),
    ("b200q_quantize_fp8_weight", WEIGHT, dict(N=TOP - 1, K=16), f"N={TOP - 1}"),
    ("b200q_quantize_fp8_weight", WEIGHT, dict(N=1, K=TOP - 16), f"K={TOP - 16}"),
])
def test_sizes_next_to_2_31(name, args, change, word):
    refused(call(name, dict(args), change), word)

"""What the calls of linear layers in 8 bits refuse: arguments are looked at before anything is launched."""
import pytest

P = 1 << 20   # an address that nobody reads: a multiple of every alignment


def refused(rc, word):
    from llmq_b200 import lib
    assert rc == -1
    assert word in lib.load().b200q_last_error().decode()


def call(name, a, change):
    from llmq_b200 import lib
    a.update(change)
    return getattr(lib.load(), name)(*a.values(), 0)


NORM = dict(x=P, residual=P, w=P, y=P, scales=P, ld=8, T=4, H=256, eps=1e-5, dtype=0)


@pytest.mark.parametrize("change,word", [(dict(H=24), "H=24"), (dict(H=16400), "H=16400"), (dict(H=0), "H=0"), (dict(T=-1), "T=-1"), (dict(dtype=2), "dtype=2"),
                                         (dict(ld=3), "ld_scales"), (dict(x=0), "null"), (dict(scales=0), "null"), (dict(y=P + 8), "aligned"),
                                         (dict(residual=P + 4), "aligned")])
def test_norm(change, word):
    refused(call("b200q_rmsnorm_fp8", dict(NORM), change), word)
    assert call("b200q_rmsnorm_fp8", dict(NORM), dict(T=0, x=0)) == 0


ROWS = dict(x=P, ld_x=256, rows=0, y=P, scales=P, ld=8, T=4, K=256, dtype=1)


@pytest.mark.parametrize("change,word", [(dict(K=200), "K=200"), (dict(T=-2), "T=-2"), (dict(dtype=7), "dtype=7"), (dict(ld=2), "ld_scales=2"),
                                         (dict(ld_x=248), "ld_x=248"), (dict(ld_x=260), "ld_x=260"), (dict(y=0), "null"), (dict(x=P + 2), "aligned"),
                                         (dict(T=(1 << 31) - 1, ld=(1 << 31) - 1, K=4096, ld_x=4096), "too much")])
def test_rows(change, word):
    refused(call("b200q_quantize_fp8", dict(ROWS), change), word)
    assert call("b200q_quantize_fp8", dict(ROWS), dict(T=0, y=0)) == 0


WEIGHT = dict(w=P, q=P, scales=P, groups=2, N=100, K=256, dtype=0)


@pytest.mark.parametrize("change,word", [(dict(K=100), "K=100"), (dict(N=0), "N=0"), (dict(groups=-1), "groups=-1"), (dict(groups=70000), "groups=70000"),
                                         (dict(dtype=-1), "dtype=-1"), (dict(q=0), "null"), (dict(w=P + 8), "aligned"), (dict(N=1 << 24), "N=16777216")])
def test_weight(change, word):
    refused(call("b200q_quantize_fp8_weight", dict(WEIGHT), change), word)
    assert call("b200q_quantize_fp8_weight", dict(WEIGHT), dict(groups=0, w=0)) == 0


GEMM = dict(a=P, a_s=P, ld=8, w=P, w_s=P, c=P, M=5, N=264, K=272, f32=0)


@pytest.mark.parametrize("change,word", [(dict(K=264), "K=264"), (dict(N=260), "N=260"), (dict(M=-1), "M=-1"), (dict(ld=4), "ld_a_scales=4"),
                                         (dict(ld=10), "ld_a_scales=10"), (dict(w_s=0), "null"), (dict(a_s=P + 4), "aligned"), (dict(c=P + 8), "aligned")])
def test_product(change, word):
    refused(call("b200q_gemm_fp8", dict(GEMM), change), word)
    assert call("b200q_gemm_fp8", dict(GEMM), dict(M=0, a=0)) == 0


GATED = dict(a=P, a_s=P, ld=8, w=P, w_s=P, y=P, y_s=P, ld_y=8, M=5, N=512, K=272, act=0)


@pytest.mark.parametrize("change,word", [(dict(N=384), "N=384"), (dict(act=2), "act=2"), (dict(ld_y=4), "ld_y_scales=4"), (dict(y_s=0), "null"),
                                         (dict(y=P + 4), "aligned"), (dict(K=8), "K=8")])
def test_gated(change, word):
    refused(call("b200q_gemm_gated_fp8", dict(GATED), change), word)
    assert call("b200q_gemm_gated_fp8", dict(GATED), dict(M=0, y_s=0)) == 0


GROUPED = dict(a=P, rows=5, a_s=P, ld=8, w=P, w_s=P, groups=3, c=P, N=264, K=272, tab=P, n=P, mt=4, f32=0)


@pytest.mark.parametrize("change,word", [(dict(groups=0), "groups=0"), (dict(mt=-1), "max_mtiles=-1"), (dict(tab=0), "table"), (dict(n=0), "table"),
                                         (dict(tab=P + 4), "aligned"), (dict(rows=-3), "M=-3"), (dict(N=4), "N=4"), (dict(groups=1 << 26), "groups=67108864"),
                                         (dict(c=0), "null")])
def test_grouped(change, word):
    refused(call("b200q_gemm_grouped_fp8", dict(GROUPED), change), word)
    assert call("b200q_gemm_grouped_fp8", dict(GROUPED), dict(rows=0, a=0)) == 0
    assert call("b200q_gemm_grouped_fp8", dict(GROUPED), dict(mt=0, tab=0)) == 0


GROUPED_GATED = dict(a=P, rows=5, a_s=P, ld=8, w=P, w_s=P, groups=3, y=P, y_s=P, ld_y=8, N=512, K=272, tab=P, n=P, mt=4, act=0)


@pytest.mark.parametrize("change,word", [(dict(N=264), "N=264"), (dict(act=-1), "act=-1"), (dict(ld_y=0), "ld_y_scales=0"), (dict(y_s=0), "y_scales"),
                                         (dict(tab=0), "table")])
def test_grouped_gated(change, word):
    refused(call("b200q_gemm_grouped_gated_fp8", dict(GROUPED_GATED), change), word)
    assert call("b200q_gemm_grouped_gated_fp8", dict(GROUPED_GATED), dict(mt=0)) == 0


def test_mode():
    from llmq_b200 import lib
    for mode in (-1, 6, 12, 53, 4, 103, 904, 605):
        refused(lib.load().b200q_gemm_fp8_set_mode(mode), f"mode={mode}")


def test_wrappers_refuse_other_tensors():
    """types and shapes are looked at before devices, and before the library is called"""
    import torch
    from llmq_b200 import lib

    if not torch.cuda.is_available():
        lib._stream, lib._device, before = (lambda s=None: 0), (lambda: 0), (lib._stream, lib._device)
    else:
        before = None
    try:
        x, y = torch.zeros(4, 256, dtype=torch.bfloat16), torch.zeros(4, 256, dtype=torch.float8_e4m3fn)
        s = lib.fp8_row_scales(4, 256, "cpu")
        for bad in (lambda: lib.rmsnorm_fp8(x.half(), x[0], y, s, 1e-5), lambda: lib.rmsnorm_fp8(x, x[0, :128], y, s, 1e-5),
                    lambda: lib.rmsnorm_fp8(x, x[0], y[:2], s, 1e-5), lambda: lib.rmsnorm_fp8(x, x[0], y, s, 1e-5, residual=x[:2]),
                    lambda: lib.quantize_fp8(x, y[:, :128], s), lambda: lib.quantize_fp8(x[:2], y, s), lambda: lib.quantize_fp8(x, y, s),
                    lambda: lib.quantize_fp8_weight(x, y[:2], s), lambda: lib.gemm_fp8(y, s, y[:, :128], s, x),
                    lambda: lib.gemm_fp8(y, s, y, s, x), lambda: lib.gemm_fp8(y, s[:1], y, s, x[:, :4]),
                    lambda: lib.gemm_gated_fp8(y, s, y, s, y, s), lambda: lib.gemm_grouped_fp8(y, s, y[None], s, x, torch.zeros(1, 3), torch.zeros(1))):
            with pytest.raises(ValueError):
                bad()
    finally:
        if before:
            lib._stream, lib._device = before

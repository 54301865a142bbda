"""CPU-side checks of the 8-bit dense layer's and the embedding rows' entry points: what they refuse, before any HIP call."""
import os

import pytest


@pytest.fixture(scope="module")
def heads_lib():
    from phonlp_amd import _lib
    from phonlp_amd import build as B
    if not os.path.exists(_lib.LIB_PATH):
        B.build()
    return _lib.lib()


def test_e4m3_and_embedding_refusals(heads_lib):
    """The 8-bit dense layer and the embedding rows refuse bad arguments before any HIP call."""
    L, one = heads_lib, 16
    for K, kp, kb in ((1, 128, 4), (128, 128, 4), (129, 256, 4), (513, 640, 8), (868, 896, 8)):
        assert L.phonlp_e4m3_kp(K) == kp and L.phonlp_e4m3_kb(K) == kb
    assert L.phonlp_e4m3_kp(0) == 0 and L.phonlp_e4m3_kb((1 << 22) + 1) == 0

    def bad(f, good, rc=-1, **change):
        args = list(good)
        for i, v in change.items():
            args[int(i[1:])] = v
        assert f(*args) == rc, change
        assert f.__name__[len("phonlp_"):].encode() in L.phonlp_last_error()

    rows = (one, 0, 70, 4, 70, one, one, None)  # x, type, ldx, rows, K, codes, exponents
    for change in ({"_0": None}, {"_1": 3}, {"_1": -1}, {"_2": 69}, {"_3": 0}, {"_4": 0}, {"_4": (1 << 22) + 1, "_2": 1 << 23}, {"_5": None},
                   {"_6": None}, {"_0": 18}, {"_5": 24}, {"_6": 18}):
        bad(L.phonlp_e4m3_rows, rows, **change)
    values = (one, one, 4, 70, 0, one, None)
    for change in ({"_0": None}, {"_1": None}, {"_2": 0}, {"_3": 0}, {"_4": 3}, {"_5": None}, {"_5": 18}, {"_0": 24}, {"_1": 18}):
        bad(L.phonlp_e4m3_values, values, **change)
    linear = (one, one, one, one, None, one, 0, None, 4, 5, 70, 1, None)
    for change in ({"_0": None}, {"_1": None}, {"_2": None}, {"_3": None}, {"_5": None}, {"_6": 3}, {"_8": 0}, {"_9": -1}, {"_10": 0},
                   {"_0": 24}, {"_2": 24}, {"_1": 18}, {"_3": 18}, {"_4": 18}, {"_5": 18}, {"_7": 18}):
        bad(L.phonlp_linear_e4m3, linear, **change)
    bad(L.phonlp_linear_e4m3, linear, -4, _8=1 << 30, _9=1 << 20)
    back = (one, 0, 5, None, one, one, one, one, 4, 5, 70, one, one, one, one, 1 << 40, None)
    for change in ({"_0": None}, {"_1": 3}, {"_2": 4}, {"_4": None}, {"_5": None}, {"_6": None}, {"_7": None}, {"_8": 0}, {"_9": 0},
                   {"_10": 0}, {"_8": (1 << 24) + 1}, {"_9": (1 << 21) + 1, "_2": 1 << 22}, {"_10": (1 << 21) + 1}, {"_0": 18}, {"_3": 18},
                   {"_4": 24}, {"_6": 24}, {"_11": 18}, {"_12": 18}, {"_13": 18}):
        bad(L.phonlp_linear_e4m3_backward, back, **change)
    for change in ({"_14": None}, {"_14": 24}, {"_15": 16}):
        bad(L.phonlp_linear_e4m3_backward, back, -2, **change)
    assert L.phonlp_linear_e4m3_backward_ws_bytes(4, 5, 70, 3) == 0 and L.phonlp_linear_e4m3_backward_ws_bytes(4, 5, 70, 0) > 0
    emb = (one, 0, 9, one, 1, 4, 6, 9, 1.0, one, None)
    for change in ({"_0": None}, {"_1": 3}, {"_2": 8}, {"_3": None}, {"_5": 0}, {"_6": 0}, {"_7": 0}, {"_9": None}, {"_0": 18}, {"_3": 20},
                   {"_9": 18}):
        bad(L.phonlp_embedding_rows, emb, **change)
    grad = (one, 1, 9, one, 1, 4, 6, 9, 1.0, one, 1, one, 1 << 40, None)
    for change in ({"_0": None}, {"_1": 3}, {"_2": 8}, {"_3": None}, {"_5": 0}, {"_5": (1 << 30) + 1}, {"_6": 0}, {"_7": 0}, {"_9": None},
                   {"_10": 2}, {"_0": 17}, {"_3": 20}, {"_9": 17}):
        bad(L.phonlp_embedding_rows_grad, grad, **change)
    for change in ({"_11": None}, {"_11": 24}, {"_12": 16}):
        bad(L.phonlp_embedding_rows_grad, grad, -2, **change)
    assert L.phonlp_embedding_rows_grad_ws_bytes(0, 9) == 0 and L.phonlp_embedding_rows_grad_ws_bytes(4, 9) > 0


def test_e4m3_and_embedding_python_checks():
    """The Python entry points name the argument they refuse (host tensors are refused like any wrong argument)."""
    import torch

    from phonlp_amd import ops
    x = torch.zeros(4, 70)
    codes, exps = torch.zeros(4, 128, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.zeros(4, 4, dtype=torch.uint8)
    for match, call in (("x: expected a ROCm", lambda: ops.e4m3_rows(x)), ("x: expected dtype", lambda: ops.e4m3_rows(x.double())),
                        ("codes: expected float8", lambda: ops.e4m3_values(x, exps, 70)),
                        ("codes: expected a ROCm", lambda: ops.e4m3_values(codes, exps, 70)),
                        ("x_codes: expected", lambda: ops.linear_e4m3(codes, exps, codes, exps, None, 70, True)),
                        ("dY: expected dtype", lambda: ops.linear_e4m3_backward(x.double(), None, codes, exps, codes, exps, 70)),
                        ("dY: expected a ROCm", lambda: ops.linear_e4m3_backward(x, None, codes, exps, codes, exps, 70)),
                        ("table: expected a ROCm", lambda: ops.embedding_rows(x, torch.zeros(3, dtype=torch.int64))),
                        ("d_out: expected", lambda: ops.embedding_rows_grad(x, torch.zeros(3, dtype=torch.int64), 5))):
        with pytest.raises(ValueError, match=match):
            call()

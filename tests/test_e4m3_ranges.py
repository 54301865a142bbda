"""On the host: sizes past what one launch covers are refused by name, before any HIP call."""
import os

import pytest


@pytest.fixture(scope="module")
def heads_lib():
    from phonlp_amd import _lib
    from phonlp_amd import build as B
    if not os.path.exists(_lib.LIB_PATH):
        B.build()
    return _lib.lib()


@pytest.mark.parametrize("M,N", [(1 << 30, 1), (1, (1 << 30) + 1), (1 << 20, 1 << 17), (0x7FFFFFFF, 1), (16, 0x7FFFFFFF)])
def test_linear(heads_lib, M, N):
    assert heads_lib.phonlp_linear_e4m3(16, 16, 16, 16, None, 16, 0, None, M, N, 70, 1, None) == -4
    assert b"too large" in heads_lib.phonlp_last_error()


@pytest.mark.parametrize("M,N,K", [(1 << 24, 5, 1 << 12), (5, 1 << 21, 1 << 15)])
def test_backward(heads_lib, M, N, K):
    assert heads_lib.phonlp_linear_e4m3_backward_ws_bytes(M, N, K, 1) == 0
    assert heads_lib.phonlp_linear_e4m3_backward(16, 1, N, None, 16, 16, 16, 16, M, N, K, 16, 16, 16, 16, 1 << 60, None) == -1


@pytest.mark.parametrize("N,V,rc", [((1 << 30) + 1, 5, -1), (5, 0x7FFFFFFF, -1)])
def test_embedding(heads_lib, N, V, rc):
    assert heads_lib.phonlp_embedding_rows(16, 0, 4, 16, 1, N, V, 4, 1.0, 16, None) == rc
    assert heads_lib.phonlp_embedding_rows_grad(16, 0, 4, 16, 1, N, V, 4, 1.0, 16, 0, 16, 1 << 60, None) == rc

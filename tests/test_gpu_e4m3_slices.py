"""The backward of the 8-bit dense layer where its products read dY itself (bf16, no ReLU, whole steps of 32): dY as a right-hand or left-hand
slice of wider rows, inside a larger allocation.  Whole numbers, so that every sum is exact."""
import numpy as np
import pytest
import torch

from oracle import e4m3_oracle as O

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,K,wide,left", [(64, 32, 100, 64, 32), (96, 160, 300, 320, 160), (64, 160, 130, 168, 8), (256, 2464, 520, 4928, 2464),
                                             (4096, 2368, 896, 4736, 2368), (32, 384, 70, 776, 0), (2048, 96, 768, 4096, 4000)])
def test_slices_of_wider_rows(M, N, K, wide, left):
    from phonlp_amd import ops
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(M + N + K)
    draw = lambda *s: torch.randint(-3, 4, s, generator=g, device=dev).float()
    x, w, dy = draw(M, K), draw(N, K), draw(M, N).bfloat16()
    rows = torch.full((M + 8, wide), float("nan"), dtype=torch.bfloat16, device=dev)  # what is not dY must not be used
    rows[:M, left:left + N] = dy
    view = rows[:M, left:left + N]
    assert view.stride(0) == wide and view.data_ptr() % 16 == 0 and wide % 8 == 0
    xi, wi = ops.e4m3_rows(x), ops.e4m3_rows(w)
    want = [torch.from_numpy(t) for t in O.backward(*(t.double().cpu().numpy() if t is not None else None for t in (dy, None, x, w)))]
    assert max(float(t.abs().max()) for t in want[1:]) < 2 ** 24
    for dY in (view, dy):
        dX, dW, db = (t.cpu() for t in ops.linear_e4m3_backward(dY, None, *xi, *wi, K))
        assert torch.equal(dX, want[0].float().bfloat16()) and torch.equal(dW.double(), want[1]) and torch.equal(db.double(), want[2])

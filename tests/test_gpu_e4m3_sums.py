"""The sums of the 8-bit dense layer are fp32 whatever the result's type: small products beside large ones that cancel are kept, in every
form of the kernel.  Whole-number cases are exact (every partial sum in any order is a whole number under 2^24), so the results are the
roundings of the exact sums, with no tolerance.  For the others a sum of K exact products and a bias is off by at most
t = (K + 1) * 2^-23 * sum |product| (each addition by at most one step of fp32), and rounding is monotonic, so the result lies between
the roundings of want - t and want + t."""
import numpy as np
import pytest
import torch

from oracle import e4m3_oracle as O

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]
IDS = ["f32", "bf16", "f16"]


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


# one row, rows of the few-row form, rows and columns of the small tile, of the large one
@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M,N,K", [(1, 400, 300), (17, 13464, 300), (33, 33, 130), (700, 900, 300), (4096, 4096, 130), (8190, 4090, 1000)])
def test_small_products_beside_large_ones_that_cancel(dev, dtype, M, N, K):
    """Every row of x holds the pair 2^14, 2^14 at columns p and q, every row of w the pair 2^8, -2^8, the other entries are -1, 0 or 1 (exact
    beside either: 2^14 * 2^-6 and 1 * 2^-6 are codes): the pair's products are +-2^22 and leave nothing."""
    from phonlp_amd import ops
    g = torch.Generator(device=dev).manual_seed(M + N + K)
    for p, q in ((0, 1), (2, 9), (K - 1, 5), (64, 127)):
        x, w = (torch.randint(-1, 2, (rows, K), generator=g, device=dev).float() for rows in (M, N))
        x[:, [p, q]], w[:, p], w[:, q] = 2.0 ** 14, 2.0 ** 8, -2.0 ** 8
        y, _ = ops.linear_e4m3(*ops.e4m3_rows(x), *ops.e4m3_rows(w), None, K, False, dtype)
        x[:, [p, q]] = 0
        want = x @ w.t()  # whole numbers up to K
        assert torch.equal(y, want.to(dtype)), (p, q)


@pytest.mark.parametrize("dtype", TYPES, ids=IDS)
@pytest.mark.parametrize("M,N,K", [(5, 700, 4096), (900, 700, 128), (700, 900, 1024), (600, 700, 4096), (3000, 4090, 1024)])
def test_results_are_roundings_of_fp32_sums(dev, dtype, M, N, K):
    from phonlp_amd import ops
    g = torch.Generator().manual_seed(M + N + K)
    x, w, bias = torch.randn(M, K, generator=g).to(dtype), torch.randn(N, K, generator=g) / K ** 0.5, torch.randn(N, generator=g)
    xi, wi = ops.e4m3_rows(x.to(dev)), ops.e4m3_rows(w.to(dev))
    y, _ = ops.linear_e4m3(*xi, *wi, bias.to(dev), K, False, dtype)
    xv, wv = (torch.from_numpy(O.values(*O.image(t.double().numpy()), K)).to(dev) for t in (x, w))
    want = xv @ wv.t() + bias.double().to(dev)
    t = (K + 1) * 2.0 ** -23 * (xv.abs() @ wv.abs().t() + bias.double().abs().to(dev))
    assert (y >= (want - t).to(dtype)).all() and (y <= (want + t).to(dtype)).all()
    # of 16 bits' rounding alone the mean of the error is that of many half steps either way: no bias in the sums
    err = (y.double() - want) / want.square().mean().sqrt()
    limit = float(t.mean() / want.square().mean().sqrt()) + 8 * torch.finfo(dtype).eps / 2 / np.sqrt(err.numel())
    assert abs(float(err.mean())) <= limit


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("M,N,K", [(1, 40, 128), (300, 900, 200)])
def test_operands_down_to_their_smallest_step(dev, dtype, M, N, K):
    """x of up to fifteen steps of 2^-133, dY of up to fifteen (fp32: 4096), w and the kept input of whole numbers times 2^100: exact products and sums."""
    from phonlp_amd import ops
    g = torch.Generator(device=dev).manual_seed(M)
    draw = lambda most, *s: torch.randint(-most, most + 1, s, generator=g, device=dev).double()
    x, w, kept = draw(15, M, K), draw(3, N, K), draw(3, M, K)
    dY = draw(2 ** 12 if dtype == torch.float32 else 15, M, N)
    assert 2 ** 12 * 3 * max(M, N) < 2 ** 24
    small, large = lambda t, kind: (t * 2.0 ** -133).to(kind), lambda t: ops.e4m3_rows((t * 2.0 ** 100).float())
    wi = large(w)
    y, _ = ops.linear_e4m3(*ops.e4m3_rows(small(x, dtype)), *wi, None, K, False, dtype)
    assert torch.equal(y, ((x @ w.t()) * 2.0 ** -33).to(dtype))
    dX, dW, _ = ops.linear_e4m3_backward(small(dY, dtype), None, *large(kept), *wi, K)
    assert torch.equal(dX, ((dY @ w) * 2.0 ** -33).to(dtype)) and torch.equal(dW.double(), (dY.t() @ kept) * 2.0 ** -33)

"""The embedding rows at the ends of their documented ranges (N <= 2^30, V < 2^31 - 1): more tokens and rows of the table than one launch
covers.  One column of fp16, whole numbers: exact."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture()
def dev():
    yield torch.device("cuda:0")
    torch.cuda.empty_cache()


def test_the_most_tokens(dev):
    from phonlp_amd import ops
    N, V = 1 << 30, 1000
    g = torch.Generator(device=dev).manual_seed(1)
    tokens = torch.empty(N, dtype=torch.int32, device=dev).random_(-1, V + 1, generator=g)
    table = torch.arange(V, device=dev).half()[:, None]
    out = ops.embedding_rows(table, tokens, 2.0)
    for a in range(0, N, 1 << 28):  # whole numbers under 2048
        t = tokens[a:a + (1 << 28)]
        assert torch.equal(out[a:a + (1 << 28), 0], torch.where((t >= 0) & (t < V), t * 2, 0).half())
    out.fill_(1.0)
    got = ops.embedding_rows_grad(out, tokens, V, 1.0, torch.float32)
    want = torch.zeros(V + 2, dtype=torch.int64, device=dev)
    for a in range(0, N, 1 << 27):
        want += torch.bincount(tokens[a:a + (1 << 27)] + 1, minlength=V + 2)
    assert torch.equal(got[:, 0].long(), want[1:-1]) and int(want.max()) < 2 ** 24


@pytest.mark.parametrize("N", [6, 600])
@pytest.mark.parametrize("V", [(1 << 29) + 1, (1 << 30) + 70, (1 << 31) - 2])
def test_the_most_rows(dev, V, N):
    """Few tokens and sorted ones: every row is written, those of the tokens with their sums, the others with zeros."""
    from phonlp_amd import ops
    rows = [V - 1, 0, (1 << 29) - 1, 1 << 29, V - 2, V // 2]
    tokens = torch.tensor([rows[n % 6] for n in range(N)], device=dev)
    d = torch.arange(1, N + 1, device=dev).half()[:, None] % 7
    grad = ops.embedding_rows_grad(d, tokens, V, 1.0)
    assert grad.shape == (V, 1)
    want = {}
    for n in range(N):
        want[rows[n % 6]] = want.get(rows[n % 6], 0) + int(d[n])
    at = torch.tensor(list(want), device=dev)
    assert grad[at, 0].tolist() == [float(v) for v in want.values()]
    assert torch.equal(ops.embedding_rows(grad, tokens, 1.0)[:6], grad[tokens[:6]])
    grad[at] = 0
    assert not grad.view(torch.int16).any()

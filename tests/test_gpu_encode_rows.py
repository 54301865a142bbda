"""The training seam's gather of first-sub-word rows takes the index shapes that torch.gather takes, with its results, and refuses the others."""
import pytest
import torch

pytestmark = pytest.mark.gpu


class _Encoder(torch.nn.Module):
    def __init__(self, emb):
        super().__init__()
        self.emb = torch.nn.Parameter(emb)

    def forward(self, tokens):
        return None, None, (self.emb * 1.0,)


class _Model:
    def __init__(self, emb):
        self.phobert = _Encoder(emb)


@pytest.mark.parametrize("rows", [1, 2, 5])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_fewer_rows_than_sentences(rows, dtype):
    from phonlp_amd import compat
    dev = torch.device("cuda:0")
    g = torch.Generator().manual_seed(rows)
    emb = torch.randint(-8, 9, (5, 11, 24), generator=g).to(dev, dtype)
    first = torch.randint(0, 11, (rows, 7), generator=g)
    model = _Model(emb)
    got = compat._encode_train(model, torch.zeros(5, 11, dtype=torch.int64), first)
    idx = first.to(dev)[..., None].expand(-1, -1, 24)
    assert torch.equal(got, torch.gather(emb, 1, idx).float())
    d = torch.randint(-2, 3, got.shape, generator=g).float().to(dev)
    got.backward(d)
    want = torch.zeros(5, 11, 24, device=dev).scatter_add_(1, idx, d)
    assert torch.equal(model.phobert.emb.grad.float(), want)


@pytest.mark.parametrize("shape", [(7,), (6, 7), (1, 5, 7)])
def test_other_shapes_are_refused(shape):
    from phonlp_amd import compat
    model = _Model(torch.zeros(5, 11, 24, device="cuda:0"))
    with pytest.raises(ValueError, match="first_subword"):
        compat._encode_train(model, torch.zeros(5, 11, dtype=torch.int64), torch.zeros(shape, dtype=torch.int64))

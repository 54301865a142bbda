"""Tensor subclasses and traced calls of the 8-bit dense layer and the embedding rows, on the device."""
import pytest
import torch

pytestmark = pytest.mark.gpu


class Tagged(torch.Tensor):
    """An ordinary subclass."""


def _same(a, b):
    bits = lambda t: t.as_subclass(torch.Tensor).contiguous().view(torch.uint8)
    return a.shape == b.shape and a.dtype == b.dtype and torch.equal(bits(a), bits(b))


def test_subclasses_give_the_same_results():
    from phonlp_amd import ops
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(1)
    x, w = torch.randn(20, 300, generator=g, device=dev), torch.randn(40, 300, generator=g, device=dev)
    tokens = torch.randint(0, 20, (7,), generator=g, device=dev)
    tag = lambda t: t.as_subclass(Tagged)
    xi, wi = ops.e4m3_rows(x), ops.e4m3_rows(w)
    ti = ops.e4m3_rows(tag(x))
    assert all(_same(a, b) for a, b in zip(ti, xi))
    assert _same(ops.e4m3_values(tag(xi[0]), xi[1], 300), ops.e4m3_values(*xi, 300))
    want = ops.linear_e4m3(*xi, *wi, None, 300, True, torch.bfloat16, True)
    got = ops.linear_e4m3(tag(xi[0]), tag(xi[1]), *map(tag, wi), None, 300, True, torch.bfloat16, True)
    assert all(_same(a, b) for a, b in zip(got, want))
    assert ops.linear_e4m3(tag(xi[0]), xi[1], *wi, None, 300, True)[1] is None
    assert _same(ops.embedding_rows(tag(x), tokens, 2), ops.embedding_rows(x, tokens, 2.0))

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


def test_the_nodes_trace_through_their_backward():
    from torch._subclasses.fake_tensor import FakeTensorMode

    from phonlp_amd import compat
    with FakeTensorMode():
        table = torch.empty(50, 200, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        w = torch.empty(33, 200, device="cuda", requires_grad=True)
        b = torch.empty(33, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        y = compat.linear_e4m3(compat.embedding_rows(table, torch.empty(4, 7, dtype=torch.int64, device="cuda"), 2.0), w, b, True)
        assert y.shape == (4, 7, 33) and y.dtype == torch.bfloat16
        got = torch.autograd.grad(y, (table, w, b), torch.empty_like(y))
        for g, p in zip(got, (table, w, b)):
            assert g.shape == p.shape and g.dtype == p.dtype


def test_the_gradients_as_registered_ops():
    """torch.ops.phonlp_amd.* and subclasses against the functions; what is not asked for is an empty tensor there, None here."""
    from phonlp_amd import ops
    dev = torch.device("cuda:0")
    R = torch.ops.phonlp_amd
    g = torch.Generator(device=dev).manual_seed(2)
    x, w = torch.randn(20, 300, generator=g, device=dev), torch.randn(40, 300, generator=g, device=dev)
    xi, wi = ops.e4m3_rows(x), ops.e4m3_rows(w)
    bits = ops.linear_e4m3(*xi, *wi, None, 300, True, want_bits=True)[1]
    dY = torch.randn(20, 40, generator=g, device=dev)
    want = ops.linear_e4m3_backward(dY, bits, *xi, *wi, 300)
    for got in (R.linear_e4m3_backward(dY, bits, *xi, *wi, 300, True, True, True),
                ops.linear_e4m3_backward(dY.as_subclass(Tagged), bits, *xi, *wi, 300)):
        assert all(_same(a, b) for a, b in zip(got, want))
    got = R.linear_e4m3_backward(dY, bits, *xi, *wi, 300, False, True, False)
    assert got[0].numel() == 0 and _same(got[1], want[1]) and got[2].numel() == 0
    got = ops.linear_e4m3_backward(dY.as_subclass(Tagged), bits, *xi, *wi, 300, True, False, False)
    assert _same(got[0], want[0]) and got[1] is None and got[2] is None
    tokens = torch.randint(0, 9, (20,), generator=g, device=dev)
    want = ops.embedding_rows_grad(dY, tokens, 9, 2.0)
    assert _same(R.embedding_rows_grad(dY, tokens, 9, 2.0, None), want)
    assert _same(ops.embedding_rows_grad(dY.as_subclass(Tagged), tokens, 9, 2.0), want)


def test_a_compiled_step_gives_the_eager_gradients():
    """Lookup and layer under torch.compile, forward and backward traced: the eager results, bit for bit."""
    from phonlp_amd import compat
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(3)
    leaves = [t.requires_grad_(True) for t in (torch.randn(50, 200, generator=g, device=dev), torch.randn(33, 200, generator=g, device=dev),
                                               torch.randn(33, generator=g, device=dev))]
    tokens = torch.randint(-1, 50, (4, 7), generator=g, device=dev)

    def step(table, w, b):
        return compat.linear_e4m3(compat.embedding_rows(table, tokens, 2.0), w, b, True)

    y = step(*leaves)
    d = torch.randn(y.shape, generator=g, device=dev)
    want = torch.autograd.grad(y, leaves, d)
    z = torch.compile(step, backend="aot_eager")(*leaves)
    assert _same(z.detach(), y.detach())
    assert all(_same(a, b) for a, b in zip(torch.autograd.grad(z, leaves, d), want))

"""What the node of the 8-bit dense layer keeps for its backward, and the backward calls without the images that they do not read."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("need", [(1, 1, 1), (1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1)])
def test_only_what_a_gradient_reads_is_kept(need, relu):
    from phonlp_amd import compat
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(5)
    M, N, K = 300, 70, 400
    data = [torch.randn(*s, generator=g, device=dev) for s in ((M, K), (N, K), (N,))]
    d = torch.randn(M, N, generator=g, device=dev)

    def run(need):
        kept = []
        leaves = [t.clone().requires_grad_(bool(on)) for t, on in zip(data, need)]
        with torch.autograd.graph.saved_tensors_hooks(lambda t: kept.append(t.numel() * t.element_size()) or t, lambda t: t):
            y = compat.linear_e4m3(*leaves, relu)
        y.backward(d)
        return sum(kept), [t.grad for t in leaves]

    kept, grads = run(need)
    image = lambda rows: rows * (512 + 4)
    assert kept == image(M) * need[1] + image(N) * need[0] + M * 3 * 4 * relu
    for got, want, on in zip(grads, run((1, 1, 1))[1], need):
        assert torch.equal(got, want) if on else got is None


def test_images_that_are_not_read_may_be_none():
    from phonlp_amd import ops
    dev = torch.device("cuda:0")
    g = torch.Generator(device=dev).manual_seed(6)
    for dtype, M, N in ((torch.float32, 50, 33), (torch.bfloat16, 64, 96), (torch.float16, 2, 1)):
        xi, wi = ops.e4m3_rows(torch.randn(M, 200, generator=g, device=dev)), ops.e4m3_rows(torch.randn(N, 200, generator=g, device=dev))
        dY = torch.randn(M, N, generator=g, device=dev).to(dtype)
        dX, dW, db = ops.linear_e4m3_backward(dY, None, *xi, *wi, 200)
        none = (None, None)
        got = ops.linear_e4m3_backward(dY, None, *none, *wi, 200, True, False, True)
        assert torch.equal(got[0], dX) and got[1] is None and torch.equal(got[2], db)
        got = ops.linear_e4m3_backward(dY, None, *xi, *none, 200, False, True, True)
        assert got[0] is None and torch.equal(got[1], dW) and torch.equal(got[2], db)
        got = ops.linear_e4m3_backward(dY, None, *none, *none, 200, False, False, True)
        assert got[:2] == (None, None) and torch.equal(got[2], db)
        with pytest.raises(ValueError, match="x_codes: None"):
            ops.linear_e4m3_backward(dY, None, *none, *wi, 200)
        with pytest.raises(ValueError, match="w_codes: None"):
            ops.linear_e4m3_backward(dY, None, *xi, *none, 200)
        with pytest.raises(ValueError, match="go together"):
            ops.linear_e4m3_backward(dY, None, xi[0], None, *wi, 200, True, False, True)

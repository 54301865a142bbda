"""No GPU: tensor subclasses and fake tensors at the entry points of the 8-bit dense layer and the embedding rows."""
import pytest
import torch

from phonlp_amd import ops


class Tagged(torch.Tensor):
    """An ordinary subclass, as users make them to carry a name."""


def test_subclasses_meet_the_arguments_own_checks():
    x, tokens = torch.zeros(4, 70).as_subclass(Tagged), torch.zeros(3, dtype=torch.int64)
    codes, exps = torch.zeros(4, 128, dtype=torch.uint8).view(torch.float8_e4m3fn).as_subclass(Tagged), torch.zeros(4, 4, dtype=torch.uint8)
    for match, call in (("x: expected a ROCm", lambda: ops.e4m3_rows(x)), ("x: expected dtype", lambda: ops.e4m3_rows(x.double())),
                        ("codes: expected a ROCm", lambda: ops.e4m3_values(codes, exps, 70)),
                        ("x_codes: expected a ROCm", lambda: ops.linear_e4m3(codes, exps, codes, exps, None, 70, True)),
                        ("table: expected a ROCm", lambda: ops.embedding_rows(x, tokens))):
        with pytest.raises(ValueError, match=match):
            call()


def _fake_operands():
    x, w = torch.empty(28, 200, dtype=torch.bfloat16, device="cuda"), torch.empty(33, 200, device="cuda")
    return x, w, ops.e4m3_rows(x), ops.e4m3_rows(w)


def test_the_gradients_trace_on_fake_tensors():
    """Shapes and types flow through both gradients, each output asked for or not."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x, w, xi, wi = _fake_operands()
        dY, bits = torch.empty(28, 33, dtype=torch.float16, device="cuda"), torch.empty(28, 2, dtype=torch.int32, device="cuda")
        dX, dW, db = ops.linear_e4m3_backward(dY, bits, *xi, *wi, 200)
        assert dX.shape == (28, 200) and dX.dtype == torch.float16 and dX.is_cuda
        assert dW.shape == (33, 200) and db.shape == (33,) and dW.dtype == db.dtype == torch.float32
        dX, dW, db = ops.linear_e4m3_backward(dY, None, *xi, *wi, 200, False, True, False)
        assert dX is None and db is None and dW.shape == (33, 200)
        tokens = torch.empty(4, 7, dtype=torch.int32, device="cuda")
        d = torch.empty(4, 7, 100, dtype=torch.bfloat16, device="cuda")
        for dtype in (None, torch.bfloat16, torch.float32):
            g = ops.embedding_rows_grad(d, tokens, 50, 2.0, dtype)
            assert g.shape == (50, 100) and g.dtype == (dtype or torch.bfloat16) and g.is_cuda

"""What the 8-bit and embedding autograd nodes and the trainer's switch refuse, on the host."""
import pytest
import torch

from phonlp_amd import compat


def test_the_nodes_have_no_cpu_path():
    x, w = torch.randn(3, 8, requires_grad=True), torch.randn(4, 8)
    with pytest.raises(ValueError, match="device"):
        compat.linear_e4m3(x, w)
    with pytest.raises(ValueError, match="device"):
        compat.embedding_rows(w, torch.tensor([0, 1]))


def test_the_nodes_are_not_captured(monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="not captured"):
        compat.linear_e4m3(torch.randn(3, 8), torch.randn(4, 8))
    with pytest.raises(RuntimeError, match="not captured"):
        compat.embedding_rows(torch.randn(4, 8), torch.tensor([0, 1]))


def test_the_trainers_switch():
    class Trainer:
        model = None

    with pytest.raises(ValueError, match="dense"):
        compat.patch_trainer(Trainer(), train_seam=True, dense="e5m2")
    with pytest.raises(ValueError, match="training seam"):
        compat.patch_trainer(Trainer(), dense="e4m3")


def test_the_forward_operators_trace_on_fake_tensors():
    """No GPU: shapes and types flow through an image, its values, a layer and a lookup on fake device tensors."""
    from torch._subclasses.fake_tensor import FakeTensorMode

    from phonlp_amd import ops
    with FakeTensorMode():
        table, tokens = torch.empty(50, 200, dtype=torch.bfloat16, device="cuda"), torch.empty(4, 7, dtype=torch.int64, device="cuda")
        x = ops.embedding_rows(table, tokens, 2.0)
        assert x.shape == (4, 7, 200) and x.dtype == torch.bfloat16
        xi = ops.e4m3_rows(x.view(28, 200))
        wi = ops.e4m3_rows(torch.empty(33, 200, device="cuda"))
        assert xi[0].shape == (28, 256) and xi[0].dtype == torch.float8_e4m3fn and xi[1].shape == (28, 4) and xi[1].dtype == torch.uint8
        assert ops.e4m3_values(*xi, 200, torch.float16).shape == (28, 200)
        y, bits = ops.linear_e4m3(*xi, *wi, None, 200, True, torch.float16, True)
        assert y.shape == (28, 33) and y.dtype == torch.float16 and bits.shape == (28, 2) and bits.dtype == torch.int32
        assert ops.linear_e4m3(*xi, *wi, None, 200, True)[1] is None

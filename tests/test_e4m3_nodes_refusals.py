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

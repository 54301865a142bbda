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

"""What cross_attention refuses, on the CPU: every check stands in front of the look at the device."""

import pytest
import torch

import adasplash_amd as A


def _call(**change):
    a = {"q": torch.zeros(2, 8, 5, 64), "k": torch.zeros(2, 2, 7, 64), "v": torch.zeros(2, 2, 7, 64)}
    a.update(change)
    return A.cross_attention(**a)


@pytest.mark.parametrize("change, text", [
    ({"q": torch.zeros(8, 5, 64)}, "shape"),
    ({"v": torch.zeros(2, 2, 8, 64)}, "share one shape"),
    ({"q": torch.zeros(3, 8, 5, 64)}, "agree"),
    ({"q": torch.zeros(2, 8, 5, 32)}, "agree"),
    ({"q": torch.zeros(2, 8, 5, 48), "k": torch.zeros(2, 2, 7, 48), "v": torch.zeros(2, 2, 7, 48)}, "head_dim must be"),
    ({"q": torch.zeros(2, 7, 5, 64)}, "multiple"),
    ({"k": torch.zeros(2, 0, 7, 64), "v": torch.zeros(2, 0, 7, 64)}, "multiple"),
    ({"k": torch.zeros(2, 2, 7, 64, dtype=torch.float16)}, "dtype"),
    ({"alpha": 1.0}, "alpha"),
    ({"alpha": 2.01}, "alpha"),
    ({"q": torch.zeros(2, 5, 8, 64).transpose(1, 2)}, "contiguous"),
    ({"varlen_q": torch.ones(3, dtype=torch.int32)}, "varlen_q"),
    ({"varlen_k": torch.ones(2)}, "int32/int64"),
    ({"varlen_k": torch.ones(2, 1, dtype=torch.int64)}, "varlen_k"),
])
def test_cross_attention_refuses(change, text):
    with pytest.raises(AssertionError, match=text):
        _call(**change)


def test_a_cpu_tensor_is_refused_behind_the_other_checks():
    with pytest.raises(RuntimeError, match="ROCm device only"):
        _call()
    with pytest.raises(RuntimeError, match="ROCm device only"):
        _call(varlen_q=torch.ones(2, dtype=torch.int32), varlen_k=torch.ones(2, dtype=torch.int64))


def test_other_types():
    with pytest.raises(TypeError):
        _call(q=torch.zeros(2, 8, 5, 64).double(), k=torch.zeros(2, 2, 7, 64).double(), v=torch.zeros(2, 2, 7, 64).double())
    with pytest.raises(TypeError):
        _call(q=None)


def test_forward_mode_is_refused():
    from torch.autograd import forward_ad

    with forward_ad.dual_level(), pytest.raises((NotImplementedError, RuntimeError)):
        _call(q=forward_ad.make_dual(torch.zeros(2, 8, 5, 64), torch.ones(2, 8, 5, 64)))

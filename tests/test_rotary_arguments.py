"""What ``rotary`` and ``write_pages`` with a ``Rotary`` refuse, on the CPU: every check stands in front of the look at the device."""

import pytest
import torch

import adasplash_amd as A
from adasplash_amd.paged import PagedCache


def _call(**change):
    a = {"q": torch.zeros(2, 4, 6, 64), "k": torch.zeros(2, 2, 6, 64), "positions": torch.arange(6), "frequencies": torch.zeros(32, dtype=torch.float64)}
    a.update(change)
    return A.rotary(**a)


def test_a_cpu_tensor_is_refused_behind_the_other_checks():
    for change in ({}, {"k": None}, {"positions": torch.zeros(2, 6, dtype=torch.int32)}, {"q_weight": torch.ones(64), "k_weight": torch.ones(64)},
                   {"q": torch.zeros(6, 4, 64), "k": torch.zeros(6, 2, 64)}, {"frequencies": torch.zeros(0, dtype=torch.float64)}):
        with pytest.raises(RuntimeError, match="ROCm device only"):
            _call(**change)


@pytest.mark.parametrize("change, text", [
    ({"q": torch.zeros(6, 64)}, "q must have shape"),
    ({"q": torch.zeros(2, 4, 6, 48), "k": torch.zeros(2, 2, 6, 48)}, "head_dim must be"),
    ({"k": torch.zeros(2, 2, 5, 64)}, "agree"),
    ({"k": torch.zeros(1, 2, 6, 64)}, "agree"),
    ({"k": torch.zeros(2, 2, 6, 32)}, "agree"),
    ({"k": torch.zeros(6, 2, 64)}, "agree"),
    ({"k": torch.zeros(2, 2, 6, 64, dtype=torch.float16)}, "share a dtype"),
    ({"k": None, "k_weight": torch.ones(64)}, "k_weight without k"),
    ({"positions": torch.arange(5)}, "positions must have shape"),
    ({"positions": torch.zeros(1, 6, dtype=torch.int64)}, "positions must have shape"),
    ({"positions": torch.zeros(6, 2, dtype=torch.int64)}, "positions must have shape"),
    ({"positions": torch.zeros(6)}, "int32/int64"),
    ({"q": torch.zeros(6, 4, 64), "k": None, "positions": torch.zeros(1, 6, dtype=torch.int64)}, "positions must have shape"),
    ({"frequencies": torch.zeros(32)}, "float64"),
    ({"frequencies": torch.zeros(16, 2, dtype=torch.float64)}, "float64"),
    ({"frequencies": torch.zeros(36, dtype=torch.float64)}, "multiple of 8"),
    ({"frequencies": torch.zeros(6, dtype=torch.float64)}, "multiple of 8"),
    ({"q_weight": torch.ones(32)}, "q_weight"),
    ({"q_weight": torch.ones(64, dtype=torch.float16)}, "q_weight"),
    ({"k_weight": torch.ones(1, 64)}, "k_weight"),
    ({"eps": 0.0}, "eps"),
    ({"eps": float("nan")}, "eps"),
    ({"eps": 1e-50}, "eps"),
    ({"eps": 1e50}, "eps"),
    ({"factor": 1e300}, "factor"),
    ({"factor": float("inf")}, "factor"),
])
def test_rotary_refuses(change, text):
    with pytest.raises(AssertionError, match=text):
        _call(**change)


def test_names():
    from adasplash_amd import positions

    assert A.Rotary is positions.Rotary and "Rotary" in A.__all__
    with pytest.raises(AttributeError):
        A.rotary_embedding


def test_other_refusals():
    with pytest.raises(ValueError, match="layout"):
        _call(layout="both")
    with pytest.raises(ValueError, match="layout"):
        A.Rotary(torch.zeros(32, dtype=torch.float64), layout="both")
    with pytest.raises(TypeError):
        _call(q=torch.zeros(2, 4, 6, 64, dtype=torch.float64), k=None)
    with pytest.raises(TypeError):
        _call(q=[1.0])
    with pytest.raises(RuntimeError, match="frequencies"):
        _call(frequencies=torch.zeros(32, dtype=torch.float64, requires_grad=True))
    import torch.autograd.forward_ad as fwAD

    with fwAD.dual_level(), pytest.raises(NotImplementedError):
        _call(q=fwAD.make_dual(torch.zeros(2, 4, 6, 64), torch.ones(2, 4, 6, 64)))


def _write(**change):
    a = {"k": torch.zeros(5, 2, 64), "v": torch.zeros(5, 2, 64), "slots": torch.arange(5), "k_pages": torch.zeros(3, 2, 16, 64), "v_pages": torch.zeros(3, 2, 16, 64),
         "positions": torch.arange(5), "rotary": A.Rotary(torch.zeros(32, dtype=torch.float64))}
    a.update(change)
    return A.write_pages(**a)


@pytest.mark.parametrize("change", [
    {"positions": torch.arange(4)},
    {"positions": torch.zeros(5)},
    {"positions": torch.zeros(1, 5, dtype=torch.int64)},
    {"slots": torch.arange(4)},
    {"rotary": A.Rotary(torch.zeros(40, dtype=torch.float64))},
    {"rotary": A.Rotary(torch.zeros(32, dtype=torch.float64), k_weight=torch.ones(32))},
    {"k": torch.zeros(5, 2, 48), "v": torch.zeros(5, 2, 48), "k_pages": torch.zeros(3, 2, 16, 48), "v_pages": torch.zeros(3, 2, 16, 48),
     "rotary": A.Rotary(torch.zeros(8, dtype=torch.float64))},
])
def test_turned_writes_refuse(change):
    with pytest.raises(AssertionError):
        _write(**change)


def test_turned_writes_refuse_more():
    with pytest.raises(RuntimeError, match="ROCm device only"):
        _write()
    with pytest.raises(ValueError, match="together"):
        _write(rotary=None)
    with pytest.raises(ValueError, match="together"):
        _write(positions=None)
    with pytest.raises(RuntimeError, match="no gradient"):
        _write(rotary=A.Rotary(torch.zeros(32, dtype=torch.float64), k_weight=torch.ones(64, requires_grad=True)))


@pytest.mark.parametrize("rotary", [
    A.Rotary(torch.zeros(32)),
    A.Rotary(torch.zeros(36, dtype=torch.float64)),
    A.Rotary(torch.zeros(32, dtype=torch.float64), k_weight=torch.ones(32)),
])
def test_a_cache_refuses(rotary):
    cache = PagedCache(8, 16, 2, 2, 64, 100, dtype=torch.float32, device="cpu", rotary=rotary)
    with pytest.raises(AssertionError):
        cache.append(torch.zeros(2, 2, 64), torch.zeros(2, 2, 64))

"""Helpers that several operators' wrappers share, without a GPU."""
import pytest
import torch

from kernels import _ak


@pytest.mark.parametrize("shape", [(0,), (2,), (1, 3)])
def test_a_scale_of_several_elements_is_refused(monkeypatch, shape):
    monkeypatch.setattr(_ak, "require_cuda", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(_ak, "call", lambda *a: pytest.fail("launched"))
    with pytest.raises(RuntimeError, match="shape"):
        _ak.scale_by_device_scalar_(torch.zeros(4), torch.ones(shape))


@pytest.mark.parametrize("scale", [torch.tensor(2.0), torch.tensor([2.0]), torch.tensor([[2.0]]),
                                   torch.tensor(2.0, dtype=torch.bfloat16), torch.tensor([1.0, 2.0])[1:],
                                   torch.tensor(2.0, dtype=torch.float64)])
def test_a_scale_of_one_element_is_taken(monkeypatch, scale):
    seen = []
    monkeypatch.setattr(_ak, "require_cuda", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(_ak, "stream", lambda d: None)
    monkeypatch.setattr(_ak, "f32_dense", lambda t, f=_ak.f32_dense: seen.append(f(t)) or seen[-1])
    monkeypatch.setattr(_ak, "call", lambda name, *a: seen.append(a))
    _ak.scale_by_device_scalar_(torch.zeros(4), scale)
    s, args = seen
    assert s.dtype == torch.float32 and s.numel() == 1 and s.item() == 2.0
    assert args[2] == s.data_ptr() and args[1] == 4

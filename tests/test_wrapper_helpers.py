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


def test_sizes_are_remembered_for_each_device(monkeypatch):
    """A size may depend on the device's SMs: what one device was told is not the other's answer, and
    the question is put with the device of the tensors current."""
    asked = []

    def answer(device, name, *args):
        asked.append((device.index, name, args[:-1]))
        args[-1]._obj.value = 100 * (device.index or 0) + args[0]

    monkeypatch.setattr(_ak, "call_on", answer)
    _ak._size_on.cache_clear()
    try:
        for _ in range(2):
            for index in (0, 1):
                assert _ak._size_query(torch.device("cuda", index), "ak_rmsnorm_bwd_workspace_size", 7, 64) == 100 * index + 7
        assert asked == [(i, "ak_rmsnorm_bwd_workspace_size", (7, 64)) for i in (0, 1)]
    finally:
        _ak._size_on.cache_clear()


def test_sizes_come_from_the_library():
    n = _ak._size_query(torch.device("cpu"), "ak_linear_logprobs_workspace_size", 8, 64, 100, 0)
    assert n > 8 * 2 * 12
    with pytest.raises(_ak.AkError):
        _ak._size_query(torch.device("cpu"), "ak_linear_logprobs_workspace_size", 8, 0, 100, 0)

"""Arguments of the distillation loss: refusals, without a GPU."""
import ctypes

import pytest
import torch

from kernels import _ak
from kernels import distill as DT


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA"):
        DT.distill_topk(torch.zeros(2, 8), torch.zeros(2, 3, dtype=torch.long), torch.zeros(2, 3))


@pytest.mark.parametrize("bad,err", [
    (dict(logits=torch.zeros(2, 8, dtype=torch.float64)), TypeError),
    (dict(logits=torch.zeros(())), ValueError), (dict(logits=torch.zeros(2, 0)), ValueError),
    (dict(idx=torch.zeros(2, 3)), TypeError), (dict(idx=torch.zeros(3, 3, dtype=torch.long)), ValueError),
    (dict(idx=torch.zeros(2, 4, dtype=torch.long)), ValueError),
    (dict(lp=torch.zeros(2, 3, dtype=torch.float64)), TypeError),
    (dict(lp=torch.zeros(2, 3, requires_grad=True)), ValueError),
    (dict(idx=torch.zeros(2, 0, dtype=torch.long), lp=torch.zeros(2, 0)), ValueError),
    (dict(idx=torch.zeros(2, 129, dtype=torch.long), lp=torch.zeros(2, 129)), ValueError),
    (dict(mask=torch.zeros(2)), TypeError), (dict(mask=torch.zeros(3, dtype=torch.bool)), ValueError),
    (dict(temperature=0.0), ValueError), (dict(temperature=float("nan")), ValueError),
    (dict(softcap=-1.0), ValueError), (dict(mode="eager"), ValueError)])
def test_refusals(monkeypatch, bad, err):
    monkeypatch.setattr(_ak, "require_cuda", lambda *t: torch.device("cpu"))
    args = dict(logits=torch.zeros(2, 8), idx=torch.zeros(2, 3, dtype=torch.long), lp=torch.zeros(2, 3))
    args.update(bad)
    with pytest.raises(err):
        DT.distill_topk(args.pop("logits"), args.pop("idx"), args.pop("lp"), **args)


def test_library_refusals():
    lib = _ak.lib()
    fake = ctypes.c_void_p(256)  # never dereferenced: each call fails its checks first

    def fwd(loss=fake, losses=fake, inv_n=fake, grad=fake, rest=None, gk=None, logits=fake, idx=fake, mask=fake,
            rows=2, inner=2, V=64, K=3, T=1.0, cap=0.0, dt=1):
        return lib.ak_distill_topk_fwd(loss, losses, inv_n, grad, rest, gk, logits, idx, fake, mask, rows, inner, 0, V,
                                       V, K, T, cap, 0, dt, None, None)

    assert fwd(dt=7) == 2
    for kw in (dict(V=0), dict(K=0), dict(K=129), dict(rows=-1), dict(inner=0), dict(V=1 << 21), dict(V=500_000, dt=0)):
        assert fwd(**kw) == 3, kw
    for kw in (dict(loss=None), dict(losses=None), dict(inv_n=None), dict(logits=None), dict(idx=None), dict(T=0.0),
               dict(cap=float("inf")), dict(rest=fake), dict(gk=fake), dict(grad=ctypes.c_void_p(257)),
               dict(logits=ctypes.c_void_p(257))):
        assert fwd(**kw) == 1, kw
        assert lib.ak_last_error()

    def bwd(grad=fake, rest=fake, gk=fake, mask=None, inv_n=None, g_loss=fake, rows=2, K=3):
        return lib.ak_distill_topk_bwd(grad, fake, fake, rest, gk, mask, inv_n, g_loss, rows, 2, 0, 64, 64, K, 1.0, 0.0,
                                       1, None)

    for kw in (dict(grad=None), dict(rest=None), dict(gk=None), dict(g_loss=None), dict(mask=fake)):
        assert bwd(**kw) == 1, kw
    assert bwd(K=0) == 3
    assert bwd(rows=0) == 0

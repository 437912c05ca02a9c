"""Arguments at the edge of what the operators over logits take, without a GPU."""
import ctypes

import pytest
import torch

from kernels import _ak
from kernels import token_logprobs as TL


def on_gpu(monkeypatch):
    """Lets CPU tensors pass the device check, so that the checks behind it are reached."""
    monkeypatch.setattr(_ak, "require_cuda", lambda *t: torch.device("cpu"))


def test_temperatures_too_low_for_fp32_are_refused(monkeypatch):
    """Below 2^-100 products of masked logits with 1 / temperature leave fp32's range."""
    on_gpu(monkeypatch)
    lib = _ak.lib()
    fake = ctypes.c_void_p(256)  # never dereferenced: each call fails its checks first
    for T in (1e-31, 1e-39, 1e-45):
        with pytest.raises(ValueError, match="2\\^-100"):
            TL.token_logprobs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.long), temperature=T)
        with pytest.raises(ValueError, match="2\\^-100"):
            TL.linear_token_logprobs(torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(9, 8), temperature=T)
        assert lib.ak_token_logprobs_fwd(fake, None, fake, None, None, None, fake, fake, 2, 2, 0, 64, 64, 0, T, 0.0, -100,
                                         1, None) == 1
        assert lib.ak_distill_topk_fwd(fake, fake, None, None, None, None, fake, fake, fake, None, 2, 2, 0, 64, 64, 3, T,
                                       0.0, 0, 1, None, None) == 1
        assert lib.ak_linear_logprobs_fwd(None, None, fake, None, fake, 1 << 20, fake, fake, None, 8, 64, 100, T, 0.0,
                                          -100, 1, None, None) == 1


def test_forward_mode_derivatives_are_refused(monkeypatch):
    """Without requires_grad nothing else would stop a dual input, whose tangent the library drops."""
    from kernels import ce_fused
    from kernels.distill import distill_topk
    on_gpu(monkeypatch)
    monkeypatch.setattr(_ak, "call", lambda *a: pytest.fail("launched"))
    monkeypatch.setattr(_ak, "call_on", lambda *a: pytest.fail("launched"))
    ad = torch.autograd.forward_ad
    x, t = torch.randn(2, 8), torch.zeros(2, dtype=torch.long)
    h, w = torch.randn(2, 8, dtype=torch.bfloat16), torch.randn(9, 8, dtype=torch.bfloat16)
    idx, lp = torch.zeros(2, 3, dtype=torch.long), torch.full((2, 3), -1.5)
    with ad.dual_level():
        def dual(a):
            return ad.make_dual(a, torch.ones_like(a))
        for call in (lambda: TL.token_logprobs(dual(x), t), lambda: TL.token_logprobs(dual(x), top_k=2),
                     lambda: TL.linear_token_logprobs(dual(h), w, t), lambda: TL.linear_token_logprobs(h, dual(w), t),
                     lambda: distill_topk(dual(x), idx, lp), lambda: distill_topk(x, idx, dual(lp)),
                     lambda: ce_fused.kernel_fn(dual(x), t)):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="forward-mode"):
                    call()
        _ak.refuse_tangents("an input without a tangent", x, None)


def test_the_type_of_a_weight_gradient():
    lib, n = _ak.lib(), ctypes.c_size_t(0)
    fake = ctypes.c_void_p(256)  # never dereferenced: each call fails its checks first
    assert lib.ak_linear_logprobs_workspace_size(8, 64, 100, 1, ctypes.byref(n)) == 0

    def bwd(dt_dw, dt=1, rows=8, dW=fake):
        return lib.ak_linear_logprobs_bwd_ex(fake, dW, dt_dw, fake, n, fake, fake, fake, fake, fake, None, rows, 64, 100,
                                             1.0, 0.0, -100, dt, None, None)

    assert bwd(2) == 2 and bwd(1, dt=2) == 2 and bwd(7) == 2 and bwd(0, dt=0) == 2
    assert bwd(0, dW=ctypes.c_void_p(264)) == 1
    for dt_dw in (0, 1):
        assert bwd(dt_dw, rows=0) == 0


def test_softcaps_too_low_for_fp32_are_refused(monkeypatch):
    on_gpu(monkeypatch)
    lib = _ak.lib()
    fake = ctypes.c_void_p(256)  # never dereferenced: each call fails its checks first
    for cap in (1e-31, 1e-39, 1e-45):
        with pytest.raises(ValueError, match="2\\^-100"):
            TL.token_logprobs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.long), softcap=cap)
        assert lib.ak_token_logprobs_fwd(fake, None, fake, None, None, None, fake, fake, 2, 2, 0, 64, 64, 0, 1.0, cap, -100,
                                         1, None) == 1
        assert lib.ak_distill_topk_fwd(fake, fake, None, None, None, None, fake, fake, fake, None, 2, 2, 0, 64, 64, 3,
                                       1.0, cap, 0, 1, None, None) == 1
        assert lib.ak_linear_logprobs_fwd(None, None, fake, None, fake, 1 << 20, fake, fake, None, 8, 64, 100, 1.0, cap,
                                          -100, 1, None, None) == 1

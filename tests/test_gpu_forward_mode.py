"""Forward-mode derivatives: refused on every way into the operators over logits, on the GPU."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_dual_inputs_are_refused_with_and_without_requires_grad():
    from kernels import ce_fused
    from kernels.distill import distill_topk
    from kernels.token_logprobs import linear_token_logprobs, token_logprobs
    ad = torch.autograd.forward_ad
    x, t = torch.randn(4, 64, device="cuda"), torch.zeros(4, dtype=torch.long, device="cuda")
    h, w = (torch.randn(n, 16, device="cuda").bfloat16() for n in (4, 64))
    idx, lp = torch.zeros(4, 2, dtype=torch.long, device="cuda"), torch.full((4, 2), -1.0, device="cuda")
    plain = token_logprobs(x, t).logprobs
    with ad.dual_level():
        for leaf in (False, True):
            dx, dh = (ad.make_dual(a.clone().requires_grad_(leaf), torch.ones_like(a)) for a in (x, h))
            for call in (lambda: token_logprobs(dx, t, entropy=True), lambda: linear_token_logprobs(dh, w, t),
                         lambda: distill_topk(dx, idx, lp), lambda: ce_fused.kernel_fn(dx, t),
                         lambda: ce_fused.ce_full(dx, t)):
                with pytest.raises((NotImplementedError, RuntimeError)):
                    call()
        assert torch.equal(token_logprobs(x, t).logprobs, plain)  # nothing to refuse

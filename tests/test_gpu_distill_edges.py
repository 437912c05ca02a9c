"""Distillation: calls at the edges of what its documentation allows."""
import pytest
import torch

from oracle import logit_row_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"


def rows(n, v, k, dtype, seed, rest=0.2, std=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = (torch.randn(n, v, generator=g, device=DEV) * std).to(dtype)
    idx = torch.topk(torch.randn(n, v, generator=g, device=DEV), k, dim=1).indices
    tlp = torch.log_softmax(torch.randn(n, k, generator=g, device=DEV) * 2, 1) + torch.log1p(torch.tensor(-rest)).item()
    return x, idx, tlp


@pytest.mark.parametrize("n,v,k", [(12000, 4100, 128), (4000, 24000, 128)])
def test_many_rows_with_a_slow_finish(n, v, k):
    """128 entries a row after a short row: the row's end takes longer than its statistics, on CTAs
    that walk many rows.  Each row against the oracle at some, all rows against a second run."""
    from kernels import _ak
    x, idx, tlp = rows(n, v, k, torch.bfloat16, 3)
    mask = torch.rand(n, generator=torch.Generator().manual_seed(1)).to(DEV) < 0.9
    first = _ak.distill_topk_fwd(x, idx, tlp, mask, tail=True, want_grad=True)
    for _ in range(3):
        again = _ak.distill_topk_fwd(x, idx, tlp, mask, tail=True, want_grad=True)
        assert torch.equal(first[1], again[1]) and torch.equal(first[3], again[3])
    _ak.check_status(torch.device(DEV))
    at = torch.arange(0, n, n // 40, device=DEV)
    ref = O.distill_topk(x[at].double().cpu(), idx[at].cpu(), tlp[at].cpu(), mask[at].cpu(), tail=True)
    O.assert_within(first[1][at], ref["losses"], ref["tol_losses"], "losses")
    f = max(1, int(mask[at].sum())) / int(mask.sum())  # the mean is over all rows
    O.assert_within(first[3][at], ref["grad"] * f, ref["tol_grad"] * f, "grad")

"""The 64-bit oracle of the distillation checked against autograd of its own definition, on the CPU."""
import pytest
import torch

from oracle import logit_row_oracle as O


def definition(x, idx, tlp, mask, temperature, softcap, tail):
    """The mean loss, row by row from its definition."""
    total, n = torch.zeros((), dtype=torch.float64), x.shape[0]
    for r in range(n):
        if mask is not None and not mask[r]:
            continue
        live = [k for k in range(idx.shape[1]) if idx[r, k] >= 0]
        if not live:
            continue
        y = x[r]
        if softcap:
            y = torch.where(torch.isneginf(y), y, softcap * torch.tanh(y.nan_to_num(neginf=0.0) / softcap))
        y = y / temperature
        at, t = idx[r, live], tlp[r, live]
        q = t.exp() if tail else torch.softmax(t, 0)
        logp = y - torch.logsumexp(y, 0)
        total = total + (q * ((t if tail else torch.log_softmax(t, 0)) - logp[at])).sum()
        outside = torch.ones(x.shape[1], dtype=torch.bool)
        outside[at] = False
        outside &= ~torch.isneginf(x[r])
        rest = 1 - q.sum()
        # a rest far below the largest logit counts as masked
        if tail and rest > 0 and outside.any() and (y[outside].max() - y.max()) * temperature >= -3e4:
            total = total + rest * (rest.log() - torch.logsumexp(logp[outside], 0))
    return temperature ** 2 * total / max(1, n if mask is None else int(mask.sum()))


CASES = {
    "rest": dict(mass=0.7), "no rest": dict(mass=1.3), "masked rest": dict(mass=0.7, hide=-torch.inf),
    "lowest rest": dict(mass=0.7, hide=-6e4), "masked, no rest": dict(mass=1.3, hide=-torch.inf),
    "repeated": dict(mass=0.9, repeat=True), "repeated beyond one": dict(mass=1.6, repeat=True),
    "repeated, masked rest": dict(mass=0.5, repeat=True, hide=-torch.inf),
}


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("name", CASES)
def test_distillation_gradient(name, tail):
    case = CASES[name]
    g = torch.Generator().manual_seed(len(name))
    n, v, k = 4, 23, 5
    x = torch.randn(n, v, generator=g, dtype=torch.float64) * 2
    idx = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(n)])
    tlp = torch.log_softmax(torch.randn(n, k, generator=g, dtype=torch.float64), 1) + torch.log(torch.tensor(case["mass"]))
    if case.get("repeat"):
        idx[1, 3] = idx[1, 0]
        idx[2, 1:] = idx[2, 0]
    idx[3, 4] = -1
    if "hide" in case:
        hidden = torch.ones(n, v, dtype=torch.bool).scatter_(1, idx.clamp(min=0), False)
        x[hidden] = case["hide"]
    mask = torch.tensor([True, True, True, True])
    for temperature, softcap in ((1.0, 0.0), (1.7, 0.0), (0.8, 0.0 if case.get("hide") == -6e4 else 6.0)):
        leaf = x.clone().requires_grad_(True)
        loss = definition(leaf, idx, tlp, mask, temperature, softcap, tail)
        want, = torch.autograd.grad(loss, leaf)
        got = O.distill_topk(x, idx, tlp, mask, temperature, softcap, tail)
        # both in 64 bits: tens of operations of 2^-53 each on numbers of at most about 60 (gradients, 2)
        assert abs(got["loss"] - loss.detach()) <= 1e-12 * (1 + loss.detach().abs())
        assert (got["grad"] - want.nan_to_num(nan=0.0)).abs().max() <= 1e-13 * 2
        # the loss does not change when all logits that are tokens move together, without a softcap
        if not softcap:
            assert got["grad"].sum(1).abs().max() <= 1e-13 * 2

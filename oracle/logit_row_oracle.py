"""The operators over logit rows in 64 bits, with bounds of what fp32 arithmetic may be off by.

Each function works on double tensors and is written from the formulas alone; it is test
infrastructure, never imported by the product.

Error bounds.  u = 2^-24 is half a step of fp32.  An exponential is taken of (y - M) / T: the
difference, the product with log2(e) / T and that constant are each off by u relative, so the
argument a (in powers of 2) is off by at most 3 u |a| and e by 3 u |a| ln 2, plus 2^-22 for the
hardware's exponential.  A sum of n terms added one after the other, all positive, is off by n u
relative; a thread adds V / 512 of them into each of two sums, and 32 more join threads and CTAs.
With softcap, tanhf is off by 2 units in the last place: 4 u c in y, twice in a difference.
"""
import torch

U = 2.0 ** -24
LN2 = 0.6931471805599453


def squash(x, temperature=1.0, softcap=0.0):
    """(softcap(x) / temperature, its derivative)."""
    d = torch.ones_like(x)
    if softcap > 0:
        t = torch.tanh(x / softcap)
        x, d = softcap * t, 1 - t * t
    return x / temperature, d / temperature


def token_logprobs(x, targets=None, ignore_index=-100, temperature=1.0, softcap=0.0, top_k=0):
    """dict of logprobs, entropy, lse, top_logprobs, top_indices of double rows (N, V), and the fp32
    bounds tol_lse (of log S, which every result shares), tol_logprobs, tol_entropy."""
    n, v = x.shape
    y, _ = squash(x, temperature, softcap)
    m = y.amax(1, keepdim=True)
    empty = torch.isneginf(m)
    d = torch.where(empty, torch.full_like(y, -torch.inf), y - torch.where(empty, 0.0, m))
    e = torch.exp(d)
    s = e.sum(1, keepdim=True)
    logp = torch.where(empty, torch.full_like(y, -torch.inf), d - torch.log(s))
    p = torch.where(empty, torch.zeros_like(y), e / s)
    plogp = torch.where(p == 0, torch.zeros_like(p), p * logp)
    ent = -plogp.sum(1)
    lse = torch.where(empty, m, m + torch.log(s))[:, 0]
    # bounds
    a = torch.where(p == 0, torch.zeros_like(p), d / LN2).abs()
    adds = v / 512 + 32
    cap_err = 8 * U * softcap / temperature
    a1, a2 = (p * a).sum(1), (p * a * a).sum(1)
    tol_s = 3 * U * LN2 * a1 + 4 * U + adds * U + cap_err
    tol_logs = tol_s + 2 * U * torch.log(s)[:, 0].abs()
    out = {"lse": lse, "entropy": ent, "p": p, "logp": logp, "empty": empty[:, 0], "tol_logs": tol_logs,
           "tol_lse": tol_logs + 4 * U * (m[:, 0].abs() + lse.abs()) + cap_err,
           "tol_entropy": tol_logs + LN2 * (a1 * (4 + 6 + 2 * adds) * U + a2 * 3 * U * LN2) + a1 * tol_s
           + cap_err + 2 * U * ent.abs()}
    if targets is not None:
        ign = targets == ignore_index
        bad = ~ign & ((targets < 0) | (targets >= v))
        at = targets.clamp(0, v - 1)[:, None]
        lp = logp.gather(1, at)[:, 0]
        lp = torch.where(bad, torch.full_like(lp, torch.nan), lp)
        out["logprobs"] = torch.where(ign, torch.zeros_like(lp), lp)
        out["tol_logprobs"] = tol_logs + 4 * U * (lp.abs() + torch.log(s)[:, 0].abs()) + cap_err
        out["entropy"] = torch.where(ign, torch.zeros_like(ent), ent)
    if top_k:
        # NaN below every number, equal values by lowest index
        rank = torch.where(torch.isnan(x), torch.full_like(x, -torch.inf), x + 0.0)
        order = torch.sort(rank, dim=1, descending=True, stable=True).indices
        nan_last = torch.sort(torch.isnan(x).gather(1, order).to(torch.int8), dim=1, stable=True).indices
        out["top_indices"] = order.gather(1, nan_last)[:, :top_k]
        out["top_logprobs"] = logp.gather(1, out["top_indices"])
        out["tol_top"] = (tol_logs + cap_err)[:, None] + 4 * U * (
            out["top_logprobs"].abs() + torch.log(s).abs())
    return out


def token_logprobs_grad(x, targets, g_lp, g_ent, ignore_index=-100, temperature=1.0, softcap=0.0):
    """(gradient of double rows, elementwise fp32 bound) for upstream gradients (either None)."""
    n, v = x.shape
    r = token_logprobs(x, targets, ignore_index, temperature, softcap)
    p, logp = r["p"], r["logp"]
    ign = torch.zeros(n, dtype=torch.bool, device=x.device) if targets is None else targets == ignore_index
    hot = torch.zeros_like(p)
    if targets is not None:
        bad = ~ign & ((targets < 0) | (targets >= v))
        hot.scatter_(1, targets.clamp(0, v - 1)[:, None], 1.0)
    zero = torch.zeros(n, dtype=torch.float64, device=x.device)
    gl = (zero if g_lp is None else g_lp.double())[:, None]
    ge = (zero if g_ent is None else g_ent.double())[:, None]
    H = -torch.where(p == 0, torch.zeros_like(p), p * logp).sum(1, keepdim=True)
    lgp = torch.where(p == 0, torch.zeros_like(p), logp)
    g = gl * (hot - p) - ge * p * (lgp + H)
    if targets is not None:
        g = torch.where(bad[:, None], torch.full_like(g, torch.nan), g)
    y, dy = squash(x, temperature, softcap)
    none = (ign | r["empty"])[:, None]
    tol_logs, tol_h = r["tol_logs"][:, None], r["tol_entropy"][:, None]
    cap_err = 8 * U * softcap / temperature
    # p = 2^d, d = (y - M) kl - log2 S: both parts are at most |log p| + log V, three and two
    # roundings, and one of the difference
    logv = torch.log(torch.tensor(v + 1.0, dtype=torch.float64)).item()
    rel = 4 * U + (4 * lgp.abs() + 5 * logv) * U + tol_logs + cap_err
    mag = gl.abs() + ge.abs() * (lgp.abs() + H)
    tol = p * (rel * mag + ge.abs() * (tol_h + rel) + 6 * U * mag) + 4 * U * (g.abs() + hot * gl.abs())
    tol = tol * dy.abs()
    if softcap > 0:  # the slope 1 - t^2, t = tanh off by 6 u
        tol = tol + g.abs() * (16 * U) / temperature
    g = torch.where(none, torch.zeros_like(g), g * dy)
    return g, torch.where(none, torch.zeros_like(tol), tol)


def assert_within(actual, expected, tol, what=""):
    """Elementwise |actual - expected| <= tol (+ half a step of actual's type), with the same
    infinities and NaNs."""
    a, b = actual.detach().double().cpu(), expected.double().cpu()
    tol = torch.as_tensor(tol).double().cpu().expand_as(b)
    assert a.shape == b.shape, f"{what}: shape {tuple(a.shape)} != {tuple(b.shape)}"
    odd = ~torch.isfinite(b)
    same = torch.equal(torch.isnan(a), torch.isnan(b)) and torch.equal(a[odd & ~torch.isnan(b)], b[odd & ~torch.isnan(b)])
    assert same and torch.equal(~torch.isfinite(a), odd), f"{what}: infinities or NaNs differ"
    info = torch.finfo(actual.dtype)
    half = b.abs() * info.eps / 2 + info.smallest_normal * info.eps / 2
    bad = ((a - b).abs() > tol + half) & ~odd
    if bad.any():
        i = tuple(bad.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} values out of tolerance, first at {i}: {a[i].item():.9g} vs "
                             f"{b[i].item():.9g}, tolerance {(tol + half)[i].item():.3g}")

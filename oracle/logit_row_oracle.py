"""The operators over logit rows in 64 bits, with bounds of what fp32 arithmetic may be off by.

Each function works on double tensors and is written from the formulas alone; it is test
infrastructure, never imported by the product.

Error bounds.  u = 2^-24 is half a step of fp32.  An exponential is taken of (y - M) / T: the
difference, the product with log2(e) / T and that constant are each off by u relative, so the
argument a (in powers of 2) is off by at most 3 u |a| and e by 3 u |a| ln 2, plus 2^-22 for the
hardware's exponential.  A sum of n terms added one after the other, all positive, is off by n u
relative; a thread adds V / 512 of them into each of two sums, and 32 more join threads and CTAs.
With softcap c, y is formed as c (1 - E) / (1 + E), E = e^(-2 |x| / c): E's argument is off by 2 u
relative, the exponential by 4 u, so tanh by 2 E / (1 + E)^2 (4 |x / c| + 4) u <= 2.4 u; the
difference, the sum, a quotient of 2 units in the last place and the product add 6 u of tanh: 9 u c
at most, twice in a difference (CAP).
"""
import torch

U = 2.0 ** -24
FLUSH = 2.0 ** -125  # the hardware's exponential gives 0 below 2^-126 (S is in [1, 2))
LN2 = 0.6931471805599453
CAP = 18  # of a difference of two squashed logits, in u * softcap


def squash(x, temperature=1.0, softcap=0.0):
    """(softcap(x) / temperature, its derivative); -inf stays -inf."""
    d = torch.ones_like(x)
    if softcap > 0:
        t, gone = torch.tanh(x / softcap), torch.isneginf(x)
        x, d = torch.where(gone, x, softcap * t), torch.where(gone, torch.zeros_like(t), 1 - t * t)
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
    cap_err = CAP * U * softcap / temperature
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
    cap_err = CAP * U * softcap / temperature
    # p = 2^d, d = (y - M) kl - log2 S: both parts are at most |log p| + log V, three and two
    # roundings, and one of the difference
    logv = torch.log(torch.tensor(v + 1.0, dtype=torch.float64)).item()
    rel = 4 * U + (4 * lgp.abs() + 5 * logv) * U + tol_logs + cap_err
    mag = gl.abs() + ge.abs() * (lgp.abs() + H)
    tol = p * (rel * mag + ge.abs() * (tol_h + rel) + 6 * U * mag) + 4 * U * (g.abs() + hot * gl.abs())
    tol = tol + FLUSH * mag
    tol = tol * dy.abs()
    if softcap > 0:  # the slope 1 - t^2, t = tanh off by 9 u
        tol = tol + g.abs() * (20 * U) / temperature
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


def distill_topk(x, idx, tlp, mask=None, temperature=1.0, softcap=0.0, tail=False, g_loss=1.0):
    """dict of loss, losses, grad of double rows (N, V) and the fp32 bounds tol_loss, tol_losses, tol_grad.

    Student log-probabilities are off as in token_logprobs.  q: an exponential off by 4 u, its
    argument t - max by u each, K additions and a division, with a tail rounded once from 64 bits;
    1 - sum q is formed in 64 bits and rounded (sums of K terms, off by K 2^-52); losses are sums of K
    terms, and the mean one of N / 1024 + 64."""
    n, v = x.shape
    k = idx.shape[1]
    live = torch.ones(n, dtype=torch.bool, device=x.device) if mask is None else mask
    r = token_logprobs(x, None, temperature=temperature, softcap=softcap)
    p, logp, empty = r["p"], r["logp"], r["empty"]
    used = idx >= 0
    bad = (idx >= v).any(1)
    at = idx.clamp(0, v - 1)
    t = torch.where(used, tlp.double(), torch.full_like(tlp, -torch.inf, dtype=torch.float64))
    if tail:
        none = ~used.any(1)
        q, logq = torch.where(used, t.exp(), 0.0), t
        rel_q = torch.full_like(q, U)
        rest = (1 - q.sum(1)).clamp(min=0)
    else:
        tm = t.amax(1, keepdim=True)
        none = torch.isneginf(tm[:, 0])
        d = torch.where(none[:, None], torch.full_like(t, -torch.inf), t - torch.where(none[:, None], 0.0, tm))
        z = d.exp().sum(1, keepdim=True)
        q = torch.where(none[:, None], torch.zeros_like(t), d.exp() / z)
        logq = d - torch.log(z)
        rel_q = (torch.where(q > 0, d.abs(), 0.0) + 10 + k) * U
        rest = torch.zeros(n, dtype=torch.float64, device=x.device)
    lpk = logp.gather(1, at)
    diff = torch.where(q > 0, logq - lpk, torch.zeros_like(q))
    terms = q * diff
    inside = torch.zeros(n, v + 1, dtype=torch.bool, device=x.device)
    inside.scatter_(1, torch.where(used, at, v), True)
    inside = inside[:, :v]
    outside = ~inside & ~torch.isneginf(x)
    logpr = torch.logsumexp(torch.where(outside, logp, torch.full_like(logp, -torch.inf)), 1)
    # a rest that lies 30000 below the largest logit is masked
    y = squash(x, 1.0, softcap)[0]
    low = torch.where(outside, y, torch.full_like(y, -torch.inf)).amax(1) - y.amax(1)
    has_rest = outside.any(1) & ~none & (torch.tensor(tail, device=x.device)) & (low >= -3e4)
    dr = rest * U + (k + 4) * 2.0 ** -52
    tail_term = torch.where(has_rest & (rest > 0), rest * (torch.log(rest) - logpr), torch.zeros_like(rest))
    losses = terms.sum(1) + tail_term
    tol_lp = r["tol_logs"][:, None] + 8 * U * (lpk.abs().nan_to_num(0, 0, 0) + torch.log(torch.tensor(v + 1.0)).item()) + CAP * U * softcap / temperature
    absl = torch.where(q > 0, logq.abs(), 0.0)
    tol = (q * (rel_q * diff.abs().nan_to_num(0, 0, 0) + tol_lp + (4 + k) * U * (absl + 1))).sum(1)
    tol = tol + torch.where(has_rest, dr * (3 + torch.log(rest + dr).abs() + logpr.abs().nan_to_num(0, 0, 0))
                            + rest * (2 * r["tol_logs"] + 12 * U * (1 + logpr.abs().nan_to_num(0, 0, 0)) + 2 * CAP * U * softcap / temperature),
                            torch.zeros_like(rest))
    tol = tol + 24 * U * (terms.abs().nan_to_num(0, 0, 0).sum(1) + tail_term.abs())
    losses = torch.where(none, torch.zeros_like(losses), losses)
    losses = torch.where(bad, torch.full_like(losses, torch.nan), losses)
    losses, tol = torch.where(live, losses, 0.0), torch.where(live, tol, 0.0)
    cnt = max(1, int(live.sum()))
    mult = temperature ** 2 / cnt
    # gradient
    mass = torch.zeros_like(p).scatter_add_(1, at, torch.where(used, q, 0.0))
    cond = torch.where(has_rest[:, None] & outside, (logp - logpr[:, None]).exp(), torch.zeros_like(p))  # p_i / p_r
    # the mass of all terms of the loss: 1, or the entries' own where the rest has no term
    counts = has_rest & (rest > 0)
    total = torch.where(counts, torch.ones_like(rest), q.sum(1))[:, None] if tail else torch.ones_like(rest)[:, None]
    g = torch.where(inside, total * p - mass, total * p - rest[:, None] * cond)
    _, dy = squash(x, temperature, softcap)
    logv = torch.log(torch.tensor(v + 1.0)).item()
    lgp = torch.where(p > 0, logp, torch.zeros_like(p))
    lpr = torch.where(has_rest, logpr, torch.zeros_like(rest)).abs()[:, None]
    rel = 10 * U + (4 * lgp.abs() + 6 * logv + 6 * lpr) * U + 2 * r["tol_logs"][:, None] + 2 * CAP * U * softcap / temperature
    relm = torch.zeros_like(p).scatter_add_(1, at, torch.where(used, q * (rel_q + k * U), torch.zeros_like(q)))
    rel_t = (q * (rel_q + k * U)).sum(1, keepdim=True)  # of total, absolute
    tg = p * (total * rel + rel_t) + torch.where(inside, relm, cond * (rest[:, None] * rel + dr[:, None]))
    tg = tg + 6 * U * g.abs() + 2 * FLUSH
    tg = tg * dy.abs() + (g.abs() * 20 * U / temperature if softcap > 0 else 0.0)
    off = (none | empty | ~live)[:, None]
    g, tg = torch.where(off, torch.zeros_like(g), g * dy), torch.where(off, torch.zeros_like(tg), tg)
    g = torch.where((bad & live)[:, None], torch.full_like(g, torch.nan), g)
    f = mult * g_loss
    return {"losses": losses, "tol_losses": tol, "loss": losses.sum() * mult,
            "tol_loss": (tol.sum() + (n / 1024 + 64) * U * losses.abs().nan_to_num(0, 0, 0).sum()) * mult,
            "grad": g * f, "tol_grad": tg * abs(f)}

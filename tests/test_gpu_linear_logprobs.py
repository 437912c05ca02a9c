"""Token log-probabilities from hidden states (tcgen05 GEMM) against the 64-bit oracle."""
import pytest
import torch

from oracle import logit_row_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16]
# (rows, hidden size, vocabulary): one row, ragged tiles in each direction, several tiles
SHAPES = [(1, 8, 1), (1, 64, 300), (3, 72, 257), (8, 768, 4096), (65, 128, 1001), (257, 200, 515), (300, 768, 5003),
          (513, 1536, 2048)]


def problem(n, d, v, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + n + d + v)
    h = torch.randn(n, d, generator=g).to(dtype)
    w = (torch.randn(v, d, generator=g) * 2 / d ** 0.5).to(dtype)
    t = torch.randint(0, v, (n,), generator=g)
    if n > 2:
        t[1] = -100
    return h.to(DEV), w.to(DEV), t.to(DEV)


def logit_bound(h, w):
    """The accumulators' error: D products added in fp32, (D + 1) u of sum |h w| at most; a logit's
    error moves a log-probability by at most twice its largest."""
    return ((h.double().abs().cpu() @ w.double().abs().cpu().T) * (h.shape[1] + 1) * O.U).amax(1)


def check(h, w, t, r, entropy=True, **kw):
    x = h.double().cpu() @ w.double().cpu().T
    ref = O.token_logprobs(x, None if t is None else t.cpu(), **kw)
    e = logit_bound(h, w) / kw.get("temperature", 1.0)
    O.assert_within(r.lse, ref["lse"], ref["tol_lse"] + e, "lse")
    if t is not None:
        O.assert_within(r.logprobs, ref["logprobs"], ref["tol_logprobs"] + 2 * e, "logprobs")
    if entropy:
        # dH = -sum dp log p, |dp| <= 2 e p
        O.assert_within(r.entropy, ref["entropy"], ref["tol_entropy"] + 2 * e * (1 + 2 * ref["entropy"].abs()), "entropy")
    else:
        assert r.entropy is None


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d,v", SHAPES)
def test_forward(n, d, v, dtype):
    from kernels.token_logprobs import linear_token_logprobs
    h, w, t = problem(n, d, v, dtype)
    check(h, w, t, linear_token_logprobs(h, w, t, entropy=True))
    check(h, w, t, linear_token_logprobs(h, w, t), entropy=False)
    check(h, w, None, linear_token_logprobs(h, w, entropy=True))
    for kw in (dict(temperature=0.6), dict(softcap=3.0, temperature=1.5)):
        check(h, w, t, linear_token_logprobs(h, w, t, entropy=True, **kw), **kw)
        check(h, w, t, linear_token_logprobs(h, w, t, **kw), entropy=False, **kw)


def grad_reference(h, w, t, gl, ge, two=False, **kw):
    """(dH, dW) in 64 bits and their bounds: G is off by its fp32 bound, the accumulators' error and
    one rounding to 16 bits (two: the rounding's rest is rounded again and kept); the two products
    add (N or V + 1) u of their absolute sums."""
    x = h.double().cpu() @ w.double().cpu().T
    G, tol = O.token_logprobs_grad(x, t.cpu(), gl, ge, **kw)
    r = O.token_logprobs(x, t.cpu(), **kw)
    e = logit_bound(h, w)[:, None] / kw.get("temperature", 1.0)
    mag = (0 if gl is None else gl.double().abs()[:, None]) + (0 if ge is None else ge.double().abs()[:, None]) * (
        r["logp"].abs() + r["entropy"].abs()[:, None] + 1)
    info = torch.finfo(h.dtype)
    scale = 1.0 if h.dtype == torch.bfloat16 else float(((0 if gl is None else gl.abs()) + (0 if ge is None else ge.abs())).max())
    live = (t.cpu() != -100).double()[:, None]
    tol = tol + (4 * e * r["p"] * mag / kw.get("temperature", 1.0)) * live
    half = info.eps / 2
    tol = tol + (G.abs() + tol) * (half * half if two else half) + scale * info.smallest_normal * half
    W, H = w.double().cpu(), h.double().cpu()
    dH, dW = G @ W, G.T @ H
    tH = tol @ W.abs() + (G.abs() @ W.abs()) * (W.shape[0] + 1) * O.U
    tW = tol.T @ H.abs() + (G.abs().T @ H.abs()) * (H.shape[0] + 1) * O.U
    return dH, tH, dW, tW


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d,v", SHAPES)
def test_backward(n, d, v, dtype):
    from kernels.token_logprobs import linear_token_logprobs
    h, w, t = problem(n, d, v, dtype, seed=3)
    g = torch.Generator().manual_seed(n)
    for up in (1.0, 1e-6):
        gl, ge = torch.randn(n, generator=g) * up, torch.randn(n, generator=g) * 0.3 * up
        for kw in (dict(), dict(temperature=1.7), dict(softcap=4.0, temperature=0.8)):
            for use_lp, use_ent in ((True, True), (True, False), (False, True)):
                hg, wg = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
                r = linear_token_logprobs(hg, wg, t, entropy=True, **kw)
                outs = [r.logprobs] * use_lp + [r.entropy] * use_ent
                ups = [gl.to(DEV)] * use_lp + [ge.to(DEV)] * use_ent
                dh, dw = torch.autograd.grad(outs, [hg, wg], ups)
                rh, th, rw, tw = grad_reference(h, w, t, gl if use_lp else None, ge if use_ent else None, **kw)
                O.assert_within(dh, rh, th, f"dH {kw} {use_lp} {use_ent} {up}")
                O.assert_within(dw, rw, tw, f"dW {kw} {use_lp} {use_ent} {up}")
    # one operand only
    hg = h.clone().requires_grad_(True)
    a, = torch.autograd.grad(linear_token_logprobs(hg, w, t).logprobs.sum(), hg)
    wg = w.clone().requires_grad_(True)
    b, = torch.autograd.grad(linear_token_logprobs(h, wg, t).logprobs.sum(), wg)
    rh, th, rw, tw = grad_reference(h, w, t, torch.ones(n), None)
    O.assert_within(a, rh, th, "dH alone")
    O.assert_within(b, rw, tw, "dW alone")


def test_several_chunks():
    """More rows than one chunk: dW accumulates over them."""
    from kernels.token_logprobs import linear_token_logprobs, token_logprobs
    n, d, v = 16384 * 2 + 37, 64, 515
    h, w, t = problem(n, d, v, torch.bfloat16, seed=5)
    gl = torch.randn(n, generator=torch.Generator().manual_seed(1))
    hg, wg = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    r = linear_token_logprobs(hg, wg, t, entropy=True)
    check(h, w, t, type(r)(*(f.detach() if f is not None else None for f in r)))
    dh, dw = torch.autograd.grad(r.logprobs, [hg, wg], gl.to(DEV))
    rh, th, rw, tw = grad_reference(h, w, t, gl, None)
    O.assert_within(dh, rh, th, "dH")
    O.assert_within(dw, rw, tw, "dW")


def test_same_as_logit_rows():
    """The two ways to the same answer: from the stored fp32 logits and from the hidden states."""
    from kernels.token_logprobs import linear_token_logprobs, token_logprobs
    h, w, t = problem(130, 256, 3001, torch.bfloat16, seed=6)
    x = (h.float() @ w.float().T)
    a = token_logprobs(x, t, entropy=True, softcap=20.0, temperature=1.3)
    b = linear_token_logprobs(h, w, t, entropy=True, softcap=20.0, temperature=1.3)
    e = logit_bound(h, w).max().item()
    for f in ("logprobs", "entropy", "lse"):
        assert (getattr(a, f) - getattr(b, f)).abs().max().item() <= 2e-5 + 20 * e


def test_shapes_types_and_rows():
    from kernels.token_logprobs import linear_token_logprobs
    h, w, t = problem(24, 64, 500, torch.bfloat16, seed=7)
    want = linear_token_logprobs(h, w, t, entropy=True)
    got = linear_token_logprobs(h.view(2, 3, 4, 64), w, t.view(2, 3, 4), entropy=True)
    assert got.logprobs.shape == (2, 3, 4) and torch.equal(got.logprobs.reshape(-1), want.logprobs)
    one = linear_token_logprobs(h[3], w, t[3], entropy=True)
    assert one.logprobs.shape == () and torch.equal(one.logprobs, want.logprobs[3])
    # an fp32 weight is cast, its gradient comes back in fp32; strided and unaligned inputs are copied
    w32 = w.float().requires_grad_(True)
    r = linear_token_logprobs(h, w32, t)
    assert torch.equal(r.logprobs.detach(), want.logprobs)
    g, = torch.autograd.grad(r.logprobs.sum(), w32)
    assert g.dtype == torch.float32
    ht = h.t().contiguous().t()
    assert torch.equal(linear_token_logprobs(ht, w, t).logprobs, want.logprobs)
    buf = torch.empty(24 * 64 + 1, dtype=torch.bfloat16, device=DEV)
    buf[1:] = h.view(-1)
    assert torch.equal(linear_token_logprobs(buf[1:].view(24, 64), w, t).logprobs, want.logprobs)
    # targets
    tb = t.clone()
    tb[0], tb[1], tb[2], tb[3] = 500, -1, -100, 2 ** 40
    r = linear_token_logprobs(h, w, tb, entropy=True)
    assert torch.isnan(r.logprobs[[0, 1, 3]]).all() and r.logprobs[2] == 0 and r.entropy[2] == 0
    hg = h.clone().requires_grad_(True)
    dh, = torch.autograd.grad(linear_token_logprobs(hg, w, tb).logprobs, hg, torch.ones(24, device=DEV))
    assert torch.isnan(dh[0]).all() and (dh[2] == 0).all() and torch.isfinite(dh[4:]).all()
    # no rows
    h0 = torch.zeros(0, 64, dtype=torch.bfloat16, device=DEV, requires_grad=True)
    w0 = w.clone().requires_grad_(True)
    r = linear_token_logprobs(h0, w0, torch.zeros(0, dtype=torch.long, device=DEV), entropy=True)
    dh, dw = torch.autograd.grad([r.logprobs.sum(), r.entropy.sum()], [h0, w0])
    assert dh.shape == (0, 64) and (dw == 0).all()


def test_streams_and_graph():
    from kernels import _ak
    from kernels.token_logprobs import linear_token_logprobs
    h, w, t = problem(300, 128, 3001, torch.bfloat16, seed=8)
    gl = torch.randn(300, generator=torch.Generator().manual_seed(2)).to(DEV)
    hg, wg = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        torch.autograd.grad(linear_token_logprobs(hg, wg, t).logprobs, [hg, wg], gl)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = linear_token_logprobs(hg, wg, t, entropy=True)
        grads = torch.autograd.grad(r.logprobs, [hg, wg], gl)
    for seed in (9, 10):
        h2, w2, _ = problem(300, 128, 3001, torch.bfloat16, seed=seed)
        with torch.no_grad():
            hg.copy_(h2)
            wg.copy_(w2)
        graph.replay()
        a, b = h2.clone().requires_grad_(True), w2.clone().requires_grad_(True)
        e = linear_token_logprobs(a, b, t, entropy=True)
        eg = torch.autograd.grad(e.logprobs, [a, b], gl)
        assert torch.equal(r.logprobs, e.logprobs) and torch.equal(r.entropy, e.entropy)
        assert torch.equal(grads[0], eg[0]) and torch.equal(grads[1], eg[1])
    _ak.check_status(torch.device(DEV))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d,v", [(1, 200, 20011), (1, 8, 9001), (40, 768, 30001), (256, 136, 12000), (700, 520, 9000),
                                   (16384 + 5, 64, 515)])
def test_long_vocabulary_few_rows(n, d, v, dtype):
    """dH's vocabulary is cut into runs; up to 256 rows the logits' gradient is kept in two matrices,
    so that what it loses is below a 16-bit rounding of its rounding."""
    from kernels.token_logprobs import linear_token_logprobs
    h, w, t = problem(n, d, v, dtype, seed=12)
    g = torch.Generator().manual_seed(n)
    gl, ge = torch.randn(n, generator=g), torch.randn(n, generator=g) * 0.2
    hg, wg = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    r = linear_token_logprobs(hg, wg, t, entropy=True)
    dh, dw = torch.autograd.grad([r.logprobs, r.entropy], [hg, wg], [gl.to(DEV), ge.to(DEV)])
    rh, th, rw, tw = grad_reference(h, w, t, gl, ge, two=n <= 256)
    O.assert_within(dh, rh, th, "dH")
    O.assert_within(dw, rw, tw, "dW")
    only, = torch.autograd.grad(linear_token_logprobs(hg, w, t).logprobs, hg, gl.to(DEV))
    rh, th, _, _ = grad_reference(h, w, t, gl, None, two=n <= 256)
    O.assert_within(only, rh, th, "dH alone")


def test_policy_step_from_rows_and_from_hidden_states():
    """A policy-gradient loss with an entropy bonus both ways: stored bf16 logits, and none."""
    from kernels.token_logprobs import linear_token_logprobs, token_logprobs
    h, w, t = problem(96, 128, 2003, torch.bfloat16, seed=15)
    adv = torch.randn(96, generator=torch.Generator().manual_seed(4)).to(DEV)
    live = t != -100

    def loss(r):
        return -(adv * r.logprobs + 0.01 * r.entropy)[live].mean()

    hg, wg = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss(linear_token_logprobs(hg, wg, t, entropy=True)).backward()
    h2, w2 = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    loss(token_logprobs(torch.nn.functional.linear(h2.float(), w2.float()), t, entropy=True)).backward()
    # the same gradients up to bf16 roundings of the results (and of G, kept in two parts here)
    for a, b in ((hg.grad, h2.grad), (wg.grad, w2.grad)):
        assert (a.double() - b.double()).norm() <= 2 * 2.0 ** -8 * b.double().norm()


def test_huge_and_broken_hidden_states():
    from kernels.token_logprobs import linear_token_logprobs
    h, w, t = problem(70, 64, 900, torch.bfloat16, seed=16)
    h[:35] *= 1e6                                     # one token takes all
    x = h.double().cpu() @ w.double().cpu().T
    ref = O.token_logprobs(x, t.cpu())
    r = linear_token_logprobs(h, w, t, entropy=True)
    e = logit_bound(h, w)
    O.assert_within(r.logprobs, ref["logprobs"], ref["tol_logprobs"] + 2 * e, "logprobs")
    h[3, 5] = torch.nan
    h[4, 6] = torch.inf
    r = linear_token_logprobs(h, w, t, entropy=True)
    assert torch.isnan(r.logprobs[3]) and torch.isnan(r.entropy[3]) and torch.isfinite(r.logprobs[5:]).all()
    assert not torch.isfinite(r.logprobs[4])


@pytest.mark.parametrize("dtype", DTYPES)
def test_low_temperature_gradients(dtype):
    """1/T = 2^17 is beyond fp16's range, the gradients of hidden and weight are not.  Every logit is an
    exact sum (multiples of 2^-12 below 2^-5), so only the roundings of G and of the products count."""
    from kernels.token_logprobs import linear_token_logprobs
    n, d, v, T = 5, 8, 300, 2.0 ** -17
    g = torch.Generator().manual_seed(21)
    h = (torch.randint(-2, 3, (n, d), generator=g) * 2.0 ** -6).to(dtype)
    w = (torch.randint(-2, 3, (v, d), generator=g) * 2.0 ** -6).to(dtype)
    t = torch.randint(0, v, (n,), generator=g)
    gl, ge = torch.tensor([1.0, -0.5, 0.25, 1.0, -1.0]), torch.tensor([0.5, 0.25, -0.5, 0.0, 1.0])
    hg, wg = h.to(DEV).requires_grad_(True), w.to(DEV).requires_grad_(True)
    r = linear_token_logprobs(hg, wg, t.to(DEV), temperature=T, entropy=True)
    dh, dw = torch.autograd.grad([r.logprobs, r.entropy], [hg, wg], [gl.to(DEV), ge.to(DEV)])
    W, H = w.double(), h.double()
    G, tol = O.token_logprobs_grad(H @ W.T, t, gl, ge, temperature=T)
    info = torch.finfo(dtype)
    half = info.eps / 2
    # two 16-bit parts of G; subnormal steps count times the scale, at most (1 + 1) * 2^17 / 2^8
    tol = tol + (G.abs() + tol) * half * half + 2.0 ** 10 * info.smallest_normal * half
    tH = tol @ W.abs() + (G.abs() @ W.abs()) * (v + 1) * O.U
    tW = tol.T @ H.abs() + (G.abs().T @ H.abs()) * (n + 1) * O.U
    O.assert_within(dh, G @ W, tH, "dH")
    O.assert_within(dw, G.T @ H, tW, "dW")


@pytest.mark.parametrize("dtype", DTYPES)
def test_upstream_of_ignored_rows_does_not_count(dtype):
    from kernels.token_logprobs import linear_token_logprobs
    h, w, t = problem(9, 64, 515, dtype, seed=22)     # row 1 is ignored
    hg, wg = h.clone().requires_grad_(True), w.clone().requires_grad_(True)
    got = []
    for other in (0.0, 1e30):
        gl = torch.ones(9)
        gl[1] = other
        r = linear_token_logprobs(hg, wg, t)
        got.append(torch.autograd.grad(r.logprobs, [hg, wg], gl.to(DEV)))
    for a, b in zip(*got):
        assert torch.equal(a, b)

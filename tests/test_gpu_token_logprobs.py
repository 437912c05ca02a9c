"""Token log-probabilities, entropies and alternatives against the 64-bit oracle."""
import pytest
import torch

from oracle import logit_row_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]

# one element; less than a group; heads, tails and groups; a CTA per row and clusters of them
SHAPES = [(1, 1), (3, 7), (5, 31), (2, 33), (4, 1000), (33, 4097), (7, 50257), (64, 32768), (1, 50304), (700, 515),
          (2, 131073), (301, 8192)]


def rows(n, v, dtype, seed=0, std=2.0):
    g = torch.Generator().manual_seed(1000 * seed + n + v)
    x = torch.randn(n, v, generator=g) * std
    t = torch.randint(0, v, (n,), generator=g)
    if n > 2:
        t[1] = -100
    return x.to(dtype).to(DEV), t.to(DEV)


def check(x, t, r, top_k=0, entropy=True, **kw):
    ref = O.token_logprobs(x.double().cpu(), None if t is None else t.cpu(), top_k=top_k, **kw)
    if t is not None:
        O.assert_within(r.logprobs, ref["logprobs"], ref["tol_logprobs"], "logprobs")
    else:
        assert r.logprobs is None
    O.assert_within(r.lse, ref["lse"], ref["tol_lse"], "lse")
    if entropy:
        O.assert_within(r.entropy, ref["entropy"], ref["tol_entropy"], "entropy")
    else:
        assert r.entropy is None
    if top_k:
        assert torch.equal(r.top_indices.cpu(), ref["top_indices"])
        O.assert_within(r.top_logprobs, ref["top_logprobs"], ref["tol_top"], "top_logprobs")
    else:
        assert r.top_logprobs is None and r.top_indices is None


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v", SHAPES)
def test_forward(n, v, dtype):
    from kernels.token_logprobs import token_logprobs
    x, t = rows(n, v, dtype)
    for k in sorted({0, 1, min(20, v), min(128, v)}):
        check(x, t, token_logprobs(x, t, top_k=k, entropy=True), top_k=k)
    check(x, t, token_logprobs(x, t), entropy=False)
    check(x, None, token_logprobs(x, top_k=min(5, v), entropy=True), top_k=min(5, v))


@pytest.mark.parametrize("kw", [dict(temperature=0.5), dict(temperature=2.5), dict(softcap=5.0),
                                dict(softcap=30.0, temperature=0.7)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_temperature_and_softcap(dtype, kw):
    from kernels.token_logprobs import token_logprobs
    for n, v in ((3, 999), (2, 50304), (300, 2048)):
        x, t = rows(n, v, dtype, seed=1, std=6.0)
        check(x, t, token_logprobs(x, t, top_k=17, entropy=True, **kw), top_k=17, **kw)


def masked_rows(v, dtype):
    """Rows whose masks and values leave little or nothing, many of them tied."""
    low = torch.finfo(dtype).min
    g = torch.Generator().manual_seed(v)
    base = torch.randn(v, generator=g)
    out = [torch.full((v,), -torch.inf),            # nothing left
           torch.full((v,), low),                   # the type's lowest value everywhere
           torch.zeros(v),                          # constant
           torch.full((v,), 3.0)]
    one = torch.full((v,), -torch.inf)
    one[v // 2] = -4.0                              # a single token left
    out.append(one)
    few = torch.full((v,), -torch.inf)
    few[::max(1, v // 5)] = 1.25                    # a few, tied
    out.append(few)
    lowmask = base.clone()
    lowmask[v // 3:] = low                          # masked with the lowest value
    out.append(lowmask)
    out.append(torch.round(base))                   # many ties at the top
    out.append(torch.where(torch.arange(v) % 2 == 0, -0.0, 0.0))  # zeros of both signs are equal
    out.append(base - 1000.0 if dtype != torch.float16 else base - 100.0)
    out.append(base * 0 - 30000.0)
    return torch.stack(out).to(dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [5, 100, 4099, 50304, 131072])
def test_masks_and_ties(v, dtype):
    from kernels.token_logprobs import token_logprobs
    x = masked_rows(v, dtype).to(DEV)
    t = torch.full((x.shape[0],), v // 2, device=DEV)
    for k in sorted({1, min(20, v), min(128, v)}):
        check(x, t, token_logprobs(x, t, top_k=k, entropy=True), top_k=k)
    check(x, t, token_logprobs(x, t, top_k=min(20, v), entropy=True, softcap=9.0), top_k=min(20, v), softcap=9.0)
    big = x.repeat(60, 1)  # a CTA per row
    check(big, t.repeat(60), token_logprobs(big, t.repeat(60), top_k=min(9, v), entropy=True), top_k=min(9, v))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v,copies", [(40, 1), (4099, 1), (4099, 150)])
def test_nan_and_inf(v, copies, dtype):
    from kernels.token_logprobs import token_logprobs
    x = torch.randn(4, v, generator=torch.Generator().manual_seed(3)).to(dtype)
    x[0, v // 2] = torch.nan
    x[1, 3] = torch.inf
    x[2, :] = torch.nan
    x = x.repeat(copies, 1).to(DEV)
    t = torch.zeros(x.shape[0], dtype=torch.int64, device=DEV)
    r = token_logprobs(x, t, top_k=7, entropy=True)
    for i in (0, 1, 2):
        for f in (r.logprobs, r.entropy, r.lse, r.top_logprobs):
            assert torch.isnan(f[i::4]).all()
    check(x[3::4].contiguous(), t[3::4], token_logprobs(x, t, top_k=7, entropy=True)._replace(
        **{k: getattr(r, k)[3::4] for k in r._fields}), top_k=7)
    ref = O.token_logprobs(x.double().cpu(), top_k=7)["top_indices"]
    assert torch.equal(r.top_indices.cpu(), ref)  # NaN ranks below every number
    # ignored rows are 0 whatever they hold
    r = token_logprobs(x, torch.full_like(t, -100), entropy=True)
    assert (r.logprobs == 0).all() and (r.entropy == 0).all()


def test_targets():
    from kernels.token_logprobs import token_logprobs
    x, _ = rows(6, 100, torch.float32)
    t = torch.tensor([0, 99, 100, -1, 7, 2 ** 40], device=DEV)
    r = token_logprobs(x, t, ignore_index=7)
    assert torch.isnan(r.logprobs[[2, 3, 5]]).all() and torch.isfinite(r.logprobs[[0, 1, 4]]).all()
    assert r.logprobs[4] == 0
    i32 = torch.tensor([0, 99, 3, 4, 5, 6], dtype=torch.int32, device=DEV)
    assert torch.equal(token_logprobs(x, i32).logprobs, token_logprobs(x, i32.long()).logprobs)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    from kernels.token_logprobs import token_logprobs
    B, T, V = 3, 6, 1001
    full = torch.randn(B, T, V + 7, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
    views = {"contiguous": full, "shifted": full[:, :-1], "last": full[:, -1], "first rows": full[1:],
             "padded vocabulary": full[..., :V], "both": full[:, 1:, 3:V], "copied": full.transpose(1, 2),
             "one": full[1, 2], "every second row": full[:, ::2], "expanded": full[:1].expand(4, T, V + 7),
             "four": full[:, :, :1000].unflatten(2, (4, 250)).transpose(1, 2)}
    for name, x in views.items():
        v = x.shape[-1]
        t = torch.randint(0, v, x.shape[:-1], generator=torch.Generator().manual_seed(4)).to(DEV)
        a = token_logprobs(x, t, top_k=5, entropy=True)
        b = token_logprobs(x.contiguous().clone(), t, top_k=5, entropy=True)
        assert a.logprobs.shape == t.shape and a.top_indices.shape == (*t.shape, 5)
        flat = x.reshape(-1, v)
        r = type(a)(*(f.reshape(flat.shape[0], *f.shape[t.dim():]) for f in a))
        check(flat, t.reshape(-1), r, top_k=5)
        assert torch.equal(a.top_indices, b.top_indices), name
        xg = x.detach().requires_grad_(True)
        lp = token_logprobs(xg, t).logprobs
        gl = torch.randn(t.shape, generator=torch.Generator().manual_seed(5)).to(DEV)
        g, = torch.autograd.grad(lp, xg, gl)
        ref, tol = O.token_logprobs_grad(flat.double().cpu(), t.reshape(-1).cpu(), gl.reshape(-1).cpu(), None)
        O.assert_within(g.reshape(-1, v), ref, tol, name)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(), (0,), (2, 0, 3)])
def test_empty_and_single(shape, dtype):
    from kernels.token_logprobs import token_logprobs
    x = torch.randn(*shape, 50, device=DEV).to(dtype).requires_grad_(True)
    t = torch.ones(shape, dtype=torch.int64, device=DEV)
    r = token_logprobs(x, t, top_k=3, entropy=True)
    assert r.logprobs.shape == shape and r.top_indices.shape == (*shape, 3)
    (r.logprobs.sum() + r.entropy.sum()).backward()
    assert x.grad.shape == x.shape


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v", SHAPES)
def test_backward(n, v, dtype):
    from kernels.token_logprobs import token_logprobs
    x, t = rows(n, v, dtype, seed=7)
    g = torch.Generator().manual_seed(n)
    gl, ge = torch.randn(n, generator=g), torch.randn(n, generator=g)
    for kw in (dict(), dict(temperature=1.7), dict(softcap=4.0, temperature=0.8)):
        for use_lp, use_ent in ((True, False), (False, True), (True, True)):
            xg = x.clone().requires_grad_(True)
            r = token_logprobs(xg, t, entropy=True, **kw)
            outs = [r.logprobs] * use_lp + [r.entropy] * use_ent
            ups = [gl.to(DEV)] * use_lp + [ge.to(DEV)] * use_ent
            got, = torch.autograd.grad(outs, xg, ups)
            assert got.dtype == dtype and got.shape == x.shape
            ref, tol = O.token_logprobs_grad(x.double().cpu(), t.cpu(), gl if use_lp else None,
                                             ge if use_ent else None, **kw)
            O.assert_within(got, ref, tol, f"grad {kw} {use_lp} {use_ent}")


@pytest.mark.parametrize("dtype", DTYPES)
def test_backward_masked_rows(dtype):
    from kernels.token_logprobs import token_logprobs
    x = masked_rows(4099, dtype).to(DEV)
    t = torch.full((x.shape[0],), 4099 // 2, device=DEV)
    t[2] = -100
    gl, ge = torch.ones(len(t)), torch.full((len(t),), 0.5)
    xg = x.clone().requires_grad_(True)
    r = token_logprobs(xg, t, entropy=True)
    got, = torch.autograd.grad([r.logprobs, r.entropy], xg, [gl.to(DEV), ge.to(DEV)])
    ref, tol = O.token_logprobs_grad(x.double().cpu(), t.cpu(), gl, ge)
    O.assert_within(got, ref, tol, "grad")
    assert (got[0] == 0).all() and (got[2] == 0).all()
    r = token_logprobs(xg, t, entropy=True, softcap=9.0)
    got, = torch.autograd.grad([r.logprobs, r.entropy], xg, [gl.to(DEV), ge.to(DEV)])
    ref, tol = O.token_logprobs_grad(x.double().cpu(), t.cpu(), gl, ge, softcap=9.0)
    O.assert_within(got, ref, tol, "softcap grad")
    # a row of NaN that is ignored gets zeros
    xn = torch.full((2, 77), torch.nan, dtype=dtype, device=DEV, requires_grad=True)
    r = token_logprobs(xn, torch.tensor([-100, 5], device=DEV))
    g, = torch.autograd.grad(r.logprobs.sum(), xn)
    assert (g[0] == 0).all() and torch.isnan(g[1]).all()
    # a target outside the vocabulary makes its row's gradient NaN
    xb = torch.zeros(2, 77, dtype=dtype, device=DEV, requires_grad=True)
    g, = torch.autograd.grad(token_logprobs(xb, torch.tensor([77, 5], device=DEV)).logprobs.sum(), xb)
    assert torch.isnan(g[0]).all() and torch.isfinite(g[1]).all()


def test_backward_against_differences():
    """The gradient along a direction d, |d| = 1, equals the central difference of the 64-bit
    forward up to h^2 / 6 times the third derivative.  That is at most max |d - mean| * var(d) <= 2
    for a log-probability; for the entropy, with |y - mean| <= 16 here, the joint fourth cumulant is
    at most 16 * 2 + 3 * 16, and the 2 of lse."""
    from kernels.token_logprobs import token_logprobs
    x, t = rows(5, 300, torch.float32, seed=9)
    gl, ge = torch.randn(5, generator=torch.Generator().manual_seed(1)), torch.full((5,), 0.3)
    d = torch.randn(5, 300, generator=torch.Generator().manual_seed(2), dtype=torch.float64)
    d /= d.norm(dim=1, keepdim=True)
    xg = x.clone().requires_grad_(True)
    r = token_logprobs(xg, t, entropy=True)
    g, = torch.autograd.grad([r.logprobs, r.entropy], xg, [gl.to(DEV), ge.to(DEV)])

    def f(y):
        q = O.token_logprobs(y, t.cpu())
        return q["logprobs"] * gl.double() + q["entropy"] * ge.double()

    h = 1e-4
    x64 = x.double().cpu()
    diff = (f(x64 + h * d) - f(x64 - h * d)) / (2 * h)
    along = (g.double().cpu() * d).sum(1)
    _, tol = O.token_logprobs_grad(x64, t.cpu(), gl, ge)
    bound = h * h / 6 * (2 * gl.abs() + 82 * ge).double() + ((tol + O.U * g.double().cpu().abs()) * d.abs()).sum(1) + 1e-11
    assert ((diff - along).abs() <= bound).all()


def test_streams_graphs_and_repeats():
    from kernels.token_logprobs import token_logprobs
    x, t = rows(40, 50257, torch.bfloat16, seed=11)
    want = token_logprobs(x, t, top_k=20, entropy=True)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = token_logprobs(x, t, top_k=20, entropy=True)
    torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(want, other):
        assert torch.equal(a, b)
    xs, gl = x.clone().requires_grad_(True), torch.ones(40, device=DEV)
    with torch.cuda.stream(s):  # warm-up, then capture forward and backward
        torch.autograd.grad(token_logprobs(xs, t).logprobs, xs, gl)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = token_logprobs(xs, t, top_k=20, entropy=True)
        g, = torch.autograd.grad(r.logprobs, xs, gl)
    y, _ = rows(40, 50257, torch.bfloat16, seed=12)
    for src in (x, y, x):
        with torch.no_grad():
            xs.copy_(src)
        graph.replay()
        e = token_logprobs(src, t, top_k=20, entropy=True)
        for a, b in zip(r, e):
            assert torch.equal(a, b)
        sg = src.clone().requires_grad_(True)
        eg, = torch.autograd.grad(token_logprobs(sg, t).logprobs, sg, gl)
        assert torch.equal(g, eg)


def test_gradient_bookkeeping():
    from kernels.token_logprobs import token_logprobs
    x, t = rows(4, 64, torch.float32)
    x.requires_grad_(True)
    r = token_logprobs(x, t, top_k=2, entropy=True)
    assert r.logprobs.requires_grad and r.entropy.requires_grad
    assert not (r.lse.requires_grad or r.top_logprobs.requires_grad or r.top_indices.requires_grad)
    a, = torch.autograd.grad(r.logprobs.sum(), x, retain_graph=True)
    b, = torch.autograd.grad(r.logprobs.sum(), x)
    assert torch.equal(a, b)
    with torch.no_grad():
        assert not token_logprobs(x, t).logprobs.requires_grad


def test_large_offsets():
    """Rows beyond 2^31 elements."""
    from kernels.token_logprobs import token_logprobs
    n, v = 70_000, 32_768
    x = torch.zeros(n, v, dtype=torch.bfloat16, device=DEV)
    x[-1] = torch.randn(v, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(DEV)
    t = torch.full((n,), 17, device=DEV)
    r = token_logprobs(x, t, top_k=4, entropy=True)
    check(x[-1:], t[-1:], type(r)(*(f[-1:] for f in r)), top_k=4)
    xg = x.requires_grad_(True)
    g, = torch.autograd.grad(token_logprobs(xg, t).logprobs, xg, torch.ones(n, device=DEV))
    ref, tol = O.token_logprobs_grad(x[-1:].detach().double().cpu(), t[-1:].cpu(), torch.ones(1), None)
    O.assert_within(g[-1:], ref, tol, "grad")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v", [(1000, 1), (700, 13), (900, 1500), (801, 4095), (650, 4097), (601, 8192)])
def test_many_short_rows(n, v, dtype):
    from kernels.token_logprobs import token_logprobs
    x, t = rows(n, v, dtype, seed=13)
    x[3] = -torch.inf
    x[4] = torch.finfo(dtype).min
    x[5, v // 2:] = -torch.inf
    x[6] = 1.5
    for k in sorted({0, min(3, v), min(128, v)}):
        check(x, t, token_logprobs(x, t, top_k=k, entropy=True), top_k=k)
    check(x, t, token_logprobs(x, t, softcap=7.0), entropy=False, softcap=7.0)
    gl = torch.randn(n, generator=torch.Generator().manual_seed(1))
    xg = x.clone().requires_grad_(True)
    r = token_logprobs(xg, t, entropy=True)
    g, = torch.autograd.grad([r.logprobs, r.entropy], xg, [gl.to(DEV), gl.to(DEV)])
    ref, tol = O.token_logprobs_grad(x.double().cpu(), t.cpu(), gl, gl)
    O.assert_within(g, ref, tol, "grad")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("v,copies", [(37, 1), (5003, 1), (5003, 200), (900, 400)])
def test_huge_logits(v, copies, dtype):
    """Exponents beyond 2^22 are taken after a subtraction; rows that go from ordinary to huge logits
    and back change their reference on the way."""
    from kernels.token_logprobs import token_logprobs
    g = torch.Generator().manual_seed(v)
    base = torch.randn(6, v, generator=g)
    x = base * torch.tensor([1e7, 1e12, 3e30, 1.0, 1.0, 1e5])[:, None]
    x[3, v // 2] = 5e8                       # one huge logit among ordinary ones
    x[4, : v // 2] = -1e9                    # huge and negative first
    x[5] = -1e8 + base[5] * 100.0            # far from zero, close together (in fp32)
    x = x.to(dtype).repeat(copies, 1).to(DEV)
    t = torch.arange(x.shape[0], device=DEV) % v
    ref = O.token_logprobs(x[:6].double().cpu(), t[:6].cpu(), top_k=min(9, v))
    r = token_logprobs(x, t, top_k=min(9, v), entropy=True)
    assert torch.equal(r.top_indices[:6].cpu(), ref["top_indices"])
    for i in range(6):
        lp = r.logprobs[i::6][t[i::6] == t[i]]
        O.assert_within(lp, ref["logprobs"][i].expand(lp.shape[0]), ref["tol_logprobs"][i], f"logprobs {i}")
        n = r.entropy[i::6]
        O.assert_within(n, ref["entropy"][i].expand(n.shape[0]), ref["tol_entropy"][i], f"entropy {i}")
    gl, ge = torch.ones(6), torch.full((6,), 0.5)
    xg = x[:6].clone().requires_grad_(True)
    q = token_logprobs(xg, t[:6], entropy=True)
    got, = torch.autograd.grad([q.logprobs, q.entropy], xg, [gl.to(DEV), ge.to(DEV)])
    want, tol = O.token_logprobs_grad(x[:6].double().cpu(), t[:6].cpu(), gl, ge)
    O.assert_within(got, want, tol, "grad")


def test_graphs_of_the_backward_and_inference_mode():
    from kernels.token_logprobs import token_logprobs
    x, t = rows(4, 300, torch.float32)
    x.requires_grad_(True)
    lp = token_logprobs(x, t).logprobs
    g, = torch.autograd.grad(lp.sum(), x, create_graph=True, retain_graph=True)
    with pytest.raises(RuntimeError):  # a gradient is a constant to what comes after it
        torch.autograd.grad(g.sum(), x)
    u = torch.ones(4, device=DEV, requires_grad=True)
    g, = torch.autograd.grad(lp, x, u, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()
    with torch.inference_mode():
        r = token_logprobs(x, t, top_k=3, entropy=True)
    assert torch.equal(r.logprobs, lp.detach())


def test_two_streams_at_once():
    from kernels.distill import distill_topk
    from kernels.token_logprobs import token_logprobs
    a, t = rows(700, 20011, torch.bfloat16, seed=31)
    b, _ = rows(700, 20011, torch.bfloat16, seed=32)
    idx = torch.topk(a, 16, dim=1).indices
    lp = torch.log_softmax(torch.randn(700, 16, generator=torch.Generator().manual_seed(1)), 1).to(DEV)
    want = [(token_logprobs(x, t, top_k=16, entropy=True), distill_topk(x, idx, lp, tail=True)) for x in (a, b)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for s, x, out in zip(streams, (a, b), got):
            with torch.cuda.stream(s):
                out.append((token_logprobs(x, t, top_k=16, entropy=True), distill_topk(x, idx, lp, tail=True)))
    torch.cuda.synchronize()
    for w, out in zip(want, got):
        for r, loss in out:
            assert torch.equal(loss, w[1]) and all(torch.equal(p, q) for p, q in zip(r, w[0]))


@pytest.mark.parametrize("dtype", DTYPES)
def test_large_softcap(dtype):
    """Under a cap far above the logits their small differences count: each capped logit is within
    8 u of its own value (5 by the polynomial's bound), not of the cap."""
    from kernels.token_logprobs import token_logprobs
    cap = 2.0e4
    for n, v in ((3, 4001), (40, 1500)):
        x, t = rows(n, v, dtype, seed=31, std=6.0)
        ref = O.token_logprobs(x.double().cpu(), t.cpu(), softcap=cap)
        plain = O.token_logprobs(x.double().cpu(), t.cpu())  # the bounds without a cap
        e = 8 * O.U * x.double().abs().amax(1).cpu()
        r = token_logprobs(x, t, entropy=True, softcap=cap)
        O.assert_within(r.lse, ref["lse"], plain["tol_lse"] + e, "lse")
        O.assert_within(r.logprobs, ref["logprobs"], plain["tol_logprobs"] + 2 * e, "logprobs")
        O.assert_within(r.entropy, ref["entropy"], plain["tol_entropy"] + 2 * e * (1 + 2 * ref["entropy"].abs()), "entropy")


@pytest.mark.parametrize("dtype", DTYPES)
def test_softcap_with_masked_and_far_logits(dtype):
    """Groups of logits within the cap, with -inf among them, beyond the cap, and of the lowest value."""
    from kernels.token_logprobs import token_logprobs
    g = torch.Generator().manual_seed(32)
    for n, v in ((6, 2051), (200, 515)):
        x, t = rows(n, v, dtype, seed=33)
        holes = torch.rand(n, v, generator=g) < 0.1
        holes[:, ::64] = True
        x[holes.to(DEV)] = -torch.inf
        x[1, 100:400] = torch.finfo(dtype).min
        x[2, 37] = 60.0
        x[3, 200:300] *= 9.0
        gl, ge = torch.randn(n, generator=g), torch.randn(n, generator=g) * 0.3
        for kw in (dict(softcap=12.0), dict(softcap=30.0, temperature=0.6)):
            check(x, t, token_logprobs(x, t, top_k=9, entropy=True, **kw), top_k=9, **kw)
            check(x, t, token_logprobs(x, t, **kw), entropy=False, **kw)
            xg = x.clone().requires_grad_(True)
            r = token_logprobs(xg, t, entropy=True, **kw)
            got, = torch.autograd.grad([r.logprobs, r.entropy], xg, [gl.to(DEV), ge.to(DEV)])
            ref, tol = O.token_logprobs_grad(x.double().cpu(), t.cpu(), gl, ge, **kw)
            O.assert_within(got, ref, tol, "gradient")
            one, = torch.autograd.grad(token_logprobs(xg, t, **kw).logprobs, xg, gl.to(DEV))
            ref, tol = O.token_logprobs_grad(x.double().cpu(), t.cpu(), gl, None, **kw)
            O.assert_within(one, ref, tol, "gradient of the log-probability")

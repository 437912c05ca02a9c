"""Token log-probabilities: calls at the edges of what their documentation allows."""
import pytest
import torch

from oracle import logit_row_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def masked(n, v, dtype, seed, scale=1.0, share=0.3):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(n, v, generator=g) * scale
    t = torch.randint(0, v, (n,), generator=g)
    gone = torch.rand(n, v, generator=g) < share
    gone[torch.arange(n), t] = False
    x[gone] = -torch.inf
    return x.to(dtype), t, gone


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,scale,T,up", [(3, 777, 0.05, 0.01, 65536.0 * 1e4), (70, 515, 0.05, 0.01, 1e10), (2, 40000, 20.0, 0.01, 1e12),
                                            (4, 300, 1.0, 1.0, 1e25), (3, 5003, 900.0, 0.001, 1e9),
                                            (2, 1000, 1e-4, 1e-6, 1e15)])
def test_masked_tokens_under_a_large_upstream_of_the_entropy(n, v, scale, T, up, dtype):
    """A token without probability has gradient 0, however large T^-2 times the upstream gradient."""
    from kernels.token_logprobs import token_logprobs
    x, t, gone = masked(n, v, dtype, 3, scale)
    gl, ge = torch.full((n,), 0.5), torch.full((n,), up)
    if dtype == torch.float16:             # its largest value is not the subject
        ge = ge * 1e-25
    for kw in (dict(temperature=T), dict(temperature=T, softcap=scale * 5)):
        leaf = x.to(DEV).requires_grad_(True)
        r = token_logprobs(leaf, t.to(DEV), entropy=True, **kw)
        got, = torch.autograd.grad([r.logprobs, r.entropy], leaf, [gl.to(DEV), ge.to(DEV)])
        assert (got[gone.to(DEV)] == 0).all()
        ref, tol = O.token_logprobs_grad(x.double(), t, gl, ge, **kw)
        # a gradient half a step beyond the type's largest value, (2 - eps / 2) 2^e, rounds to infinity
        info = torch.finfo(dtype)
        over = ref.abs() >= info.max * (1 + info.eps / 4 / (1 - info.eps / 2))
        O.assert_within(got, torch.where(over, ref.sign() * torch.inf, ref), tol, f"grad {kw}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1e-9, 1e-20, 2.0 ** -100])
def test_masked_tokens_at_the_lowest_temperatures(T, dtype):
    """The entropy of rows whose exponents leave fp32's range where they are masked: two equal
    largest tokens, all others masked or far below."""
    from kernels.token_logprobs import token_logprobs
    for n, v in ((3, 700), (700, 64), (4, 20011)):
        x = torch.full((n, v), -torch.inf)
        x[:, 5], x[:, v - 2] = 0.0, 0.0
        x[1, 7:20] = -1.0
        x[2, :] = torch.finfo(dtype).min
        x[2, 1], x[2, 2] = 0.0, 0.0
        x = x.to(dtype).to(DEV)
        r = token_logprobs(x, torch.full((n,), 5, device=DEV), entropy=True, temperature=T)
        half = torch.log(torch.tensor(2.0)).item()
        # log 2 and 0.5 log 2 twice: a few roundings of numbers below 1
        assert ((r.entropy - half).abs() <= 8 * O.U).all()
        assert ((r.logprobs[:2] + half).abs() <= 8 * O.U).all()
        leaf = x.clone().requires_grad_(True)
        q = token_logprobs(leaf, torch.full((n,), 5, device=DEV), entropy=True, temperature=T)
        g, = torch.autograd.grad(q.entropy, leaf, torch.full((n,), T, device=DEV))
        assert (g.abs() <= 8 * O.U).all()  # p (log p + H) = 0 for both


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cap", [100.0, 2.0e4, 1e12, 1e30, 3e38])
def test_small_logits_beside_masks_of_the_lowest_value(monkeypatch, cap, dtype):
    """A warp with a logit beyond the cap takes another form of the softcap, which has to keep the
    small logits of that warp as well: within 40 u of their own value, not of the cap."""
    from kernels.token_logprobs import token_logprobs
    low = torch.finfo(dtype).min
    monkeypatch.setattr(O, "CAP", 0)       # the softcap's error is counted here
    for n, v in ((3, 4001), (700, 515), (40, 9000)):
        g = torch.Generator().manual_seed(n)
        x = (torch.randn(n, v, generator=g) * 6).to(dtype)
        x[torch.rand(n, v, generator=g) < 0.05] = low
        t = torch.randint(0, v, (n,), generator=g)
        x[torch.arange(n), t] = 1.25
        x[0, 7] = min(cap * 3, 6e4) if cap < 1e4 else 1.0
        ref = O.token_logprobs(x.double(), t, softcap=cap)
        size = torch.where(x == low, 0.0, x.double()).abs().amax(1).clamp(max=cap)
        # a masked token at -cap counts where exp(-cap) does: under 100 with an error of 8 u cap
        e = 40 * O.U * size + (8 * O.U * cap if cap <= 100 else 0.0)
        r = token_logprobs(x.to(DEV), t.to(DEV), entropy=True, softcap=cap)
        O.assert_within(r.lse, ref["lse"], ref["tol_lse"] + e, "lse")
        O.assert_within(r.logprobs, ref["logprobs"], ref["tol_logprobs"] + 2 * e, "logprobs")
        O.assert_within(r.entropy, ref["entropy"], ref["tol_entropy"] + 2 * e * (1 + 2 * ref["entropy"].abs()), "entropy")
        leaf = x.to(DEV).requires_grad_(True)
        gl = torch.randn(n, generator=g)
        got, = torch.autograd.grad(token_logprobs(leaf, t.to(DEV), softcap=cap).logprobs, leaf, gl.to(DEV))
        want, tol = O.token_logprobs_grad(x.double(), t, gl, None, softcap=cap)
        p = ref["p"]
        # p is off by 2 e relative, the slope 1 - (y / cap)^2 by 20 u
        tol = tol + p * 2 * e[:, None] * gl.abs()[:, None].double() + want.abs() * 24 * O.U
        O.assert_within(got, want, tol + 24 * O.U * gl.abs()[:, None].double() * (p + (torch.arange(v) == t[:, None])), "grad")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k", [(1, 128), (3, 7), (40, 20)])
def test_the_largest_vocabulary_with_alternatives(n, k, dtype):
    """1,048,320 tokens: eight CTAs a row, each with as many group maxima as its buffer holds; rows
    that start anywhere, ties that go through the exact selection, and the last token among the best."""
    from kernels.token_logprobs import token_logprobs
    v = 1_048_320
    g = torch.Generator(device=DEV).manual_seed(n)
    full = torch.randn(n, v + 3, generator=g, device=DEV).mul_(2).to(dtype)
    for x in (full[:, :v], full[:, 3:]):
        x[0, v - 1] = 20.0
        x[0, 0] = 20.0
        if n > 2:
            x[1] = 1.0                     # constant: the lowest indices
            x[2] = -torch.inf
            x[2, v - 5:] = 0.5
        t = torch.full((n,), v - 1, device=DEV)
        r = token_logprobs(x, t, top_k=k, entropy=True)
        for i in range(0, n, max(1, n // 5)):
            s = slice(i, i + 1)
            ref = O.token_logprobs(x[s].double().cpu(), t[s].cpu(), top_k=k)
            assert torch.equal(r.top_indices[s].cpu(), ref["top_indices"])
            for f, tol in (("logprobs", "tol_logprobs"), ("entropy", "tol_entropy"), ("lse", "tol_lse"), ("top_logprobs", "tol_top")):
                O.assert_within(getattr(r, f)[s], ref[f], ref[tol], f)
        if n > 2:
            assert torch.equal(r.top_indices[1].cpu(), torch.arange(k))
            assert torch.equal(r.top_indices[2, :min(k, 5)].cpu(), torch.arange(v - 5, v)[:k])
    with pytest.raises(RuntimeError, match="too large for top_k"):
        token_logprobs(torch.zeros(1, v + 1, dtype=dtype, device=DEV), top_k=1)
    assert token_logprobs(torch.zeros(1, v + 17, dtype=dtype, device=DEV)).lse.shape == (1,)

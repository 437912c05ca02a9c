"""Distillation from a teacher's top-K log-probabilities against the 64-bit oracle."""
import pytest
import torch

from oracle import logit_row_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
SHAPES = [(1, 1, 1), (3, 7, 3), (5, 31, 8), (2, 33, 1), (4, 1000, 128), (33, 4097, 20), (7, 50257, 33),
          (20, 50304, 64), (200, 515, 17), (2, 131073, 100), (160, 8192, 5)]


def problem(n, v, k, dtype, seed=0, std=2.0, mass=0.8):
    g = torch.Generator().manual_seed(1000 * seed + n + v + k)
    x = (torch.randn(n, v, generator=g) * std).to(dtype)
    kk = min(k, v)
    idx = torch.stack([torch.randperm(v, generator=g)[:kk] for _ in range(n)])
    tlp = torch.log_softmax(torch.randn(n, kk, generator=g) * 2, 1) + torch.log(torch.tensor(mass))
    mask = torch.rand(n, generator=g) < 0.8
    mask[0] = True
    return x.to(DEV), idx.to(DEV), tlp.to(DEV), mask.to(DEV)


def check(x, idx, tlp, mask=None, upstream=1.0, modes=("fused", "tiny"), **kw):
    from kernels import _ak
    from kernels.distill import distill_topk
    flat = (x.reshape(-1, x.shape[-1]), idx.reshape(-1, idx.shape[-1]), tlp.reshape(-1, tlp.shape[-1]))
    ref = O.distill_topk(flat[0].double().cpu(), flat[1].cpu(), flat[2].cpu(),
                         None if mask is None else mask.reshape(-1).cpu(), g_loss=upstream, **kw)
    loss = distill_topk(x, idx, tlp, mask=mask, **kw)
    O.assert_within(loss, ref["loss"], ref["tol_loss"], "loss")
    losses = _ak.distill_topk_fwd(x, idx.long().contiguous(), tlp.float().contiguous(), mask, kw.get("temperature", 1.0),
                                  kw.get("softcap", 0.0), kw.get("tail", False))[1]
    O.assert_within(losses.reshape(-1), ref["losses"], ref["tol_losses"], "losses")
    for mode in modes:
        leaf = x.detach().requires_grad_(True)
        out = distill_topk(leaf, idx, tlp, mask=mask, mode=mode, **kw)
        assert torch.equal(out.detach(), loss) or torch.isnan(loss)
        g, = torch.autograd.grad(out, leaf, torch.full((), upstream, device=DEV))
        assert g.dtype == x.dtype and g.shape == x.shape
        tol = ref["tol_grad"]
        if mode == "fused" and upstream != 1.0:  # rounded once in the forward, once when scaled
            info = torch.finfo(x.dtype)
            tol = tol + ref["grad"].abs() * info.eps / 2 + abs(upstream) * info.smallest_normal * info.eps / 2
        O.assert_within(g.reshape(flat[0].shape), ref["grad"], tol, f"grad {mode} {kw}")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,k", SHAPES)
def test_loss_and_gradient(n, v, k, dtype):
    x, idx, tlp, mask = problem(n, v, k, dtype)
    check(x, idx, tlp, mask, tail=True)
    check(x, idx, tlp, None, tail=False)
    check(x, idx, tlp, mask, tail=True, temperature=2.0)
    check(x, idx, tlp, mask, tail=False, temperature=0.7, softcap=6.0)
    check(x, idx, tlp, mask, tail=True, softcap=6.0, modes=("tiny",))


@pytest.mark.parametrize("dtype", DTYPES)
def test_upstream(dtype):
    x, idx, tlp, mask = problem(9, 3001, 12, dtype, seed=3)
    for up in (0.25, 1024.0, 0.0):
        check(x, idx, tlp, mask, upstream=up, tail=True, modes=("fused", "tiny"))


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_padding_duplicates_and_bad_entries(dtype, tail):
    x, idx, tlp, mask = problem(12, 2050, 10, dtype, seed=4)
    idx[1, 4:] = -1                       # ragged
    idx[2, :] = -7                        # no entry at all
    idx[3, 5] = idx[3, 0].clone()              # one token twice, thrice
    idx[4, [2, 6, 9]] = idx[4, 1].clone()
    idx[5, :] = 11                        # nothing but one token
    tlp[6, 3] = -torch.inf                # an entry without mass
    tlp[7, :] = -torch.inf                # all of them
    idx[8, 0], idx[8, 1], idx[8, 2] = 0, 2049, 16
    mask[:] = True
    check(x, idx, tlp, mask, tail=tail)
    check(x, idx.int(), tlp, None, tail=tail, temperature=3.0)
    idx[9, 2] = 2050                      # outside the vocabulary: NaN row
    from kernels.distill import distill_topk
    for mode in ("fused", "tiny"):
        leaf = x.clone().requires_grad_(True)
        loss = distill_topk(leaf, idx, tlp, tail=tail, mode=mode)
        assert torch.isnan(loss)
        g, = torch.autograd.grad(loss, leaf, torch.ones((), device=DEV))
        assert torch.isnan(g[9]).all() and torch.isfinite(g[:9]).all() and torch.isfinite(g[10:]).all()
        mask[9] = False
        leaf = x.clone().requires_grad_(True)
        loss = distill_topk(leaf, idx, tlp, mask=mask, tail=tail, mode=mode)
        g, = torch.autograd.grad(loss, leaf)
        assert torch.isfinite(loss) and (g[9] == 0).all()
        mask[9] = True


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("v", [100, 4099, 50304])
def test_masked_logits(v, dtype, tail):
    x, idx, tlp, mask = problem(8, v, 6, dtype, seed=5)
    low = torch.finfo(dtype).min
    keep = torch.zeros(v, dtype=torch.bool, device=DEV)
    for i in range(8):
        keep[:] = False
        keep[idx[i]] = True
        if i in (0, 1):                   # nothing left but the teacher's tokens
            x[i][~keep] = -torch.inf if i == 0 else low
        if i == 2:                        # a part masked
            x[i, v // 2:][~keep[v // 2:]] = -torch.inf
    x[3] = 0.0                            # constant
    x[4] = low
    check(x, idx, tlp, mask, tail=tail)
    check(x, idx, tlp, mask, tail=tail, softcap=8.0)
    # a masked row holds anything
    x[5] = torch.nan
    x[6] = torch.inf
    mask[:] = True
    mask[[5, 6]] = False
    tlp[5] = torch.nan
    from kernels.distill import distill_topk
    ok = [0, 1, 2, 3, 4, 7]
    for mode in ("fused", "tiny"):
        leaf = x.clone().requires_grad_(True)
        loss = distill_topk(leaf, idx, tlp, mask=mask, tail=tail, mode=mode)
        g, = torch.autograd.grad(loss, leaf)
        ref = O.distill_topk(x[ok].double().cpu(), idx[ok].cpu(), tlp[ok].cpu(), tail=tail)
        O.assert_within(loss, ref["loss"], ref["tol_loss"], "loss")
        O.assert_within(g[ok], ref["grad"], ref["tol_grad"], "grad")
        assert (g[5] == 0).all() and (g[6] == 0).all()


def test_all_rows_masked_or_none():
    from kernels.distill import distill_topk
    x, idx, tlp, _ = problem(4, 100, 5, torch.float32)
    x.requires_grad_(True)
    loss = distill_topk(x, idx, tlp, mask=torch.zeros(4, dtype=torch.bool, device=DEV))
    g, = torch.autograd.grad(loss, x)
    assert loss.item() == 0 and (g == 0).all()
    for shape in ((0,), (2, 0)):
        x0 = torch.zeros(*shape, 50, device=DEV, requires_grad=True)
        l0 = distill_topk(x0, torch.zeros(*shape, 3, dtype=torch.long, device=DEV), torch.zeros(*shape, 3, device=DEV),
                          mask=torch.ones(shape, dtype=torch.bool, device=DEV))
        g0, = torch.autograd.grad(l0, x0)
        assert l0.item() == 0 and g0.shape == x0.shape
    # one row without leading dimensions
    check(x.detach()[0], idx[0], tlp[0], tail=True)


def test_all_tokens_are_the_teachers():
    """K = V: no rest, whatever 1 - sum q rounds to."""
    x, idx, tlp, mask = problem(6, 50, 50, torch.float32, mass=1.0)
    check(x, idx, tlp, mask, tail=True)
    check(x, idx, tlp, mask, tail=False)


@pytest.mark.parametrize("dtype", DTYPES)
def test_strides(dtype):
    B, T, V, K = 2, 5, 1003, 9
    full = torch.randn(B, T, V, generator=torch.Generator().manual_seed(2)).to(dtype).to(DEV)
    for x in (full, full[:, :-1], full[:, -1], full[..., :1000], full[:, 1:, 3:], full.transpose(1, 2)):
        g = torch.Generator().manual_seed(3)
        idx = torch.randint(0, x.shape[-1], (*x.shape[:-1], K), generator=g).to(DEV)
        tlp = (torch.log_softmax(torch.randn(*x.shape[:-1], K, generator=g), -1) - 0.2).to(DEV)
        mask = (torch.rand(x.shape[:-1], generator=g) < 0.7).to(DEV)
        check(x, idx, tlp, mask, tail=True)
        check(x, idx.transpose(-1, -2).contiguous().transpose(-1, -2), tlp, None, tail=False)


def test_against_differences():
    """The gradient along d, |d| = 1, against the central difference of the 64-bit loss: each row's
    log-probabilities have third derivatives of at most 2 along d (q sums to 1, the rest's
    log-probability adds one of the restricted set and one of the whole, at most 4 together)."""
    from kernels.distill import distill_topk
    n = 5
    x, idx, tlp, mask = problem(n, 300, 11, torch.float32, seed=8)
    g_ = torch.Generator().manual_seed(2)
    d = torch.randn(n, 300, generator=g_, dtype=torch.float64)
    d /= d.norm()
    x64, args = x.double().cpu(), (idx.cpu(), tlp.cpu(), mask.cpu())
    for tail in (False, True):
        leaf = x.clone().requires_grad_(True)
        g, = torch.autograd.grad(distill_topk(leaf, idx, tlp, mask=mask, tail=tail), leaf)
        h = 1e-4
        f = [O.distill_topk(x64 + s * h * d, *args, tail=tail)["loss"] for s in (1, -1)]
        ref = O.distill_topk(x64, *args, tail=tail)
        bound = h * h / 6 * 6 + ((ref["tol_grad"] + O.U * ref["grad"].abs()) * d.abs()).sum() + 1e-11
        assert abs((f[0] - f[1]) / (2 * h) - (g.double().cpu() * d).sum()) <= bound


def test_backward_twice_streams_and_graph():
    from kernels.distill import distill_topk
    x, idx, tlp, mask = problem(40, 20011, 24, torch.bfloat16, seed=11)
    leaf = x.clone().requires_grad_(True)
    loss = distill_topk(leaf, idx, tlp, mask=mask, mode="tiny")
    a, = torch.autograd.grad(loss, leaf, retain_graph=True)
    b, = torch.autograd.grad(loss, leaf)
    assert torch.equal(a, b)
    loss = distill_topk(leaf, idx, tlp, mask=mask, mode="fused")
    c, = torch.autograd.grad(loss, leaf, retain_graph=True)
    assert torch.equal(a, c)  # the same arithmetic
    with pytest.raises(RuntimeError, match="twice"):
        torch.autograd.grad(loss, leaf)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    for mode in ("fused", "tiny"):
        leaf = x.clone().requires_grad_(True)
        with torch.cuda.stream(s):
            torch.autograd.grad(distill_topk(leaf, idx, tlp, mask=mask, tail=True, mode=mode), leaf)
        torch.cuda.current_stream().wait_stream(s)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            loss = distill_topk(leaf, idx, tlp, mask=mask, tail=True, mode=mode)
            g, = torch.autograd.grad(loss, leaf)
        for seed in (12, 13):
            y = problem(40, 20011, 24, torch.bfloat16, seed=seed)[0]
            with torch.no_grad():
                leaf.copy_(y)
            graph.replay()
            e = y.clone().requires_grad_(True)
            el = distill_topk(e, idx, tlp, mask=mask, tail=True, mode=mode)
            eg, = torch.autograd.grad(el, e)
            assert torch.equal(loss.detach(), el.detach()) and torch.equal(g, eg)


def test_teacher_to_student():
    """The two operators as they are used together: a teacher answers, a student learns from it."""
    from kernels import _ak
    from kernels.distill import distill_topk
    from kernels.token_logprobs import token_logprobs
    g = torch.Generator().manual_seed(0)
    B, T, V, K, temp = 3, 17, 5003, 32, 2.0
    teacher = (torch.randn(B, T, V, generator=g) * 3).to(torch.bfloat16).to(DEV)
    student = (torch.randn(B, T, V, generator=g)).to(torch.bfloat16).to(DEV).requires_grad_(True)
    with torch.no_grad():
        top = token_logprobs(teacher[:, :-1], top_k=K, temperature=temp)
    loss = distill_topk(student[:, :-1], top.top_indices, top.top_logprobs, temperature=temp, tail=True)
    loss.backward()
    flat = student.detach()[:, :-1].reshape(-1, V).double().cpu()
    tr = O.token_logprobs(teacher[:, :-1].reshape(-1, V).double().cpu(), temperature=temp, top_k=K)
    ref = O.distill_topk(flat, tr["top_indices"], tr["top_logprobs"], temperature=temp, tail=True)
    # the teacher's answers are off by tol_top each, which moves q by that much relative
    slack = 2 * tr["tol_top"].max().item() * temp ** 2 * (1 + 2 * torch.log(torch.tensor(float(V))).item())
    O.assert_within(loss.detach(), ref["loss"], ref["tol_loss"] + slack, "loss")
    got = student.grad[:, :-1].reshape(-1, V)
    O.assert_within(got, ref["grad"], ref["tol_grad"] + 4 * tr["tol_top"].max() * ref["grad"].abs().amax(), "grad")
    assert (student.grad[:, -1] == 0).all()
    # a student equal to its teacher has nothing to learn: every term cancels to rounding
    same = teacher.detach().requires_grad_(True)
    loss = distill_topk(same[:, :-1], top.top_indices, top.top_logprobs, temperature=temp, tail=True)
    z = O.distill_topk(teacher[:, :-1].reshape(-1, V).double().cpu(), tr["top_indices"], tr["top_logprobs"],
                       temperature=temp, tail=True)
    assert abs(loss.item()) <= z["tol_loss"].item() + slack
    _ak.check_status(torch.device(DEV))


def test_large_offsets():
    """Rows beyond 2^31 elements."""
    n, v, k = 70_000, 32_768, 4
    from kernels.distill import distill_topk
    x = torch.zeros(n, v, dtype=torch.bfloat16, device=DEV)
    x[-1] = torch.randn(v, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16).to(DEV)
    idx = torch.arange(k, device=DEV).expand(n, k).contiguous()
    tlp = torch.full((n, k), -1.5, device=DEV)
    mask = torch.zeros(n, dtype=torch.bool, device=DEV)
    mask[-1] = True
    for mode in ("fused", "tiny"):
        leaf = x.detach().requires_grad_(True)
        loss = distill_topk(leaf, idx, tlp, mask=mask, tail=True, mode=mode)
        g, = torch.autograd.grad(loss, leaf)
        ref = O.distill_topk(x[-1:].double().cpu(), idx[-1:].cpu(), tlp[-1:].cpu(), tail=True)
        O.assert_within(loss, ref["loss"], ref["tol_loss"], "loss")
        O.assert_within(g[-1:], ref["grad"], ref["tol_grad"], "grad")
        assert (g[0] == 0).all() and (g[n // 2] == 0).all()
        del g, loss, leaf


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,k", [(700, 50257, 9), (1201, 4099, 128), (310, 131073, 3), (3, 262147, 40), (450, 15, 2)])
def test_many_rows_per_cta(n, v, k, dtype):
    """More rows than the GPU takes at once, so that each CTA (or cluster) walks several, some of
    them masked; and a row that needs all eight CTAs of a cluster."""
    x, idx, tlp, mask = problem(n, v, min(k, v), dtype, seed=21)
    check(x, idx, tlp, mask, tail=True)
    mask[::2] = False
    check(x, idx, tlp, mask, tail=False, modes=("fused",))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,k", [(1000, 1, 1), (700, 13, 5), (900, 1500, 128), (1300, 2048, 9), (601, 2047, 33)])
def test_many_short_rows(n, v, k, dtype):
    x, idx, tlp, mask = problem(n, v, min(k, v), dtype, seed=22)
    idx[5, -1] = idx[5, 0]
    idx[6, 0] = -1
    idx[7] = -1
    check(x, idx, tlp, mask, tail=True)
    check(x, idx, tlp, None, tail=False, softcap=5.0, temperature=1.3)


@pytest.mark.parametrize("dtype", DTYPES)
def test_many_short_strided_rows(dtype):
    B, T, V, K = 60, 13, 1003, 6
    g = torch.Generator().manual_seed(5)
    full = torch.randn(B, T, V + 5, generator=g).to(dtype).to(DEV)
    for x in (full[:, :-1], full[..., 2:V + 1], full[:, 1:, :V]):
        idx = torch.randint(-1, x.shape[-1], (*x.shape[:-1], K), generator=g).to(DEV)
        tlp = (torch.log_softmax(torch.randn(*x.shape[:-1], K, generator=g), -1) - 0.2).to(DEV)
        mask = (torch.rand(x.shape[:-1], generator=g) < 0.7).to(DEV)
        check(x, idx, tlp, mask, tail=True)


@pytest.mark.parametrize("v,copies", [(37, 1), (5003, 1), (900, 200)])
def test_huge_logits(v, copies):
    g = torch.Generator().manual_seed(v)
    base = torch.randn(4, v, generator=g)
    x = base * torch.tensor([1e7, 1.0, 1e12, 1.0])[:, None]
    x[1, 0] = 5e8
    x[3] = -1e8 + base[3] * 100.0
    x = x.repeat(copies, 1).to(DEV)
    top = torch.topk(x, 3, dim=1).indices            # teacher's tokens the student's own
    tlp = torch.log(torch.tensor([0.7, 0.2, 0.1])).expand(x.shape[0], 3).contiguous().to(DEV)
    from kernels.distill import distill_topk
    ref = O.distill_topk(x.double().cpu(), top.cpu(), tlp.cpu(), tail=False)
    for mode in ("fused", "tiny"):
        leaf = x.clone().requires_grad_(True)
        loss = distill_topk(leaf, top, tlp, mode=mode)
        got, = torch.autograd.grad(loss, leaf)
        O.assert_within(loss, ref["loss"], ref["tol_loss"] + ref["loss"].abs() * 8 * O.U, "loss")
        O.assert_within(got, ref["grad"], ref["tol_grad"], "grad")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,v,k", [(5, 5003, 40), (64, 1500, 7)])
def test_softcap_with_masked_and_far_logits(n, v, k, dtype):
    x, idx, tlp, _ = problem(n, v, k, dtype, seed=41)
    holes = torch.rand(n, v, generator=torch.Generator().manual_seed(42)) < 0.05
    holes.scatter_(1, idx.cpu().clamp(min=0), False)
    x[holes.to(DEV)] = -torch.inf
    x[1, 64:128] *= 9.0
    for tail in (False, True):
        check(x, idx, tlp, tail=tail, softcap=10.0)
        check(x, idx, tlp, tail=tail, softcap=30.0, temperature=1.4)

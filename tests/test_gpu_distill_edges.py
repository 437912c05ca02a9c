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


def check(x, idx, tlp, mask=None, modes=("fused", "tiny"), upstream=1.0, **kw):
    from kernels.distill import distill_topk
    ref = O.distill_topk(x.double().cpu(), idx.cpu(), tlp.cpu(), None if mask is None else mask.cpu(), g_loss=upstream, **kw)
    for mode in modes:
        leaf = x.detach().requires_grad_(True)
        loss = distill_topk(leaf, idx, tlp, mask=mask, mode=mode, **kw)
        O.assert_within(loss, ref["loss"], ref["tol_loss"], "loss")
        g, = torch.autograd.grad(loss, leaf, torch.full((), upstream, device=DEV))
        O.assert_within(g, ref["grad"], ref["tol_grad"], f"grad {mode} {kw}")
    return ref


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,v,k", [(9, 300, 7), (700, 520, 40), (5, 50257, 64), (300, 20011, 5)])
def test_terms_whose_mass_is_not_one(n, v, k, dtype):
    """The rest masked by the student, or entries whose mass exceeds 1 (rounded log-probabilities,
    repeated tokens): the gradient is that of the terms left, so it sums to 0 over a row."""
    x, idx, tlp = rows(n, v, k, dtype, 5, rest=0.3)
    gone = torch.ones(n, v, dtype=torch.bool, device=DEV).scatter_(1, idx, False)
    x[1] = torch.where(gone[1], -torch.inf, x[1])
    x[2] = torch.where(gone[2], torch.finfo(dtype).min, x[2])
    tlp[3] += 0.5                          # mass 0.7 e^0.5 > 1
    idx[4, k // 2:] = idx[4, 0]            # one token many times
    tlp[4] += 0.6
    if n > 8:
        x[7] = torch.where(gone[7], -torch.inf, x[7])
        tlp[7] += 0.9
        x[8] = torch.where(gone[8], -torch.inf, x[8])
        idx[8, 1] = idx[8, 0]
    ref = check(x, idx, tlp, tail=True)
    total = ref["grad"].sum(1).abs()
    assert (total <= 1e-12).all()          # of the oracle's, in 64 bits
    check(x, idx, tlp, tail=True, temperature=1.6)
    check(x, idx, tlp, tail=True, softcap=12.0, temperature=0.9)
    check(x, idx, tlp, tail=False)


def test_masked_rest_against_differences():
    """Along d, |d| = 1, as a loss of mass Q <= 2: its third derivative is at most 2 Q, and 4 with the
    rest's own term."""
    from kernels.distill import distill_topk
    n, v, k = 6, 200, 9
    x, idx, tlp = rows(n, v, k, torch.float32, 6, rest=0.3)
    gone = torch.ones(n, v, dtype=torch.bool, device=DEV).scatter_(1, idx, False)
    x[:3] = torch.where(gone[:3], -torch.inf, x[:3])
    tlp[2:4] += 0.7
    idx[5, 1] = idx[5, 0]
    d = torch.randn(n, v, generator=torch.Generator().manual_seed(4), dtype=torch.float64)
    d /= d.norm()
    leaf = x.clone().requires_grad_(True)
    g, = torch.autograd.grad(distill_topk(leaf, idx, tlp, tail=True), leaf)
    h, args = 1e-4, (idx.cpu(), tlp.cpu())
    f = [O.distill_topk(x.double().cpu() + s * h * d, *args, tail=True)["loss"] for s in (1, -1)]
    ref = O.distill_topk(x.double().cpu(), *args, tail=True)
    bound = h * h / 6 * 8 + ((ref["tol_grad"] + O.U * ref["grad"].abs()) * d.abs()).sum() + 1e-11
    assert abs((f[0] - f[1]) / (2 * h) - (g.double().cpu() * d).sum()) <= bound


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n,v,k", [(40, 2000, 64), (700, 1500, 128), (6, 50257, 64), (300, 20011, 100)])
def test_teachers_that_leave_little(n, v, k, dtype):
    """A teacher's entries cover all but 1e-2 to 1e-7 of its mass: the rest of it, 1 - sum q, and what
    follows from it keep their leading bits.  The student's own rest is as small, so the rest's term
    and its gradient p_i (1 - r / p_r) count."""
    g = torch.Generator().manual_seed(7)
    rest = 10.0 ** -(2 + 5 * torch.rand(n, 1, generator=g, dtype=torch.float64))
    idx = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(n)])
    lp = torch.log_softmax(torch.randn(n, k, generator=g, dtype=torch.float64), 1) + torch.log1p(-rest)
    x = torch.randn(n, v, generator=g, dtype=torch.float64) + torch.log(rest / v)
    x.scatter_(1, idx, lp + 0.1 * torch.randn(n, k, generator=g, dtype=torch.float64))
    x, idx, tlp = x.to(dtype).to(DEV), idx.to(DEV), lp.float().to(DEV)
    check(x, idx, tlp, tail=True)
    check(x, idx, tlp, tail=True, upstream=2.0 ** 20, modes=("tiny",))
    check(x, idx, tlp, tail=False)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("n,v,k", [(400, 9000, 128), (60, 50257, 70), (8, 131073, 33), (700, 2000, 128)])
def test_repeated_tokens_beside_others_of_their_places(n, v, k, tail):
    """Tokens that come twice or often, within a group of 32 entries and across groups, among tokens
    that agree with them in their low 11 bits."""
    x, idx, tlp = rows(n, v, k, torch.float32, 9, rest=0.25)
    g = torch.Generator().manual_seed(10)
    idx = idx.cpu()
    for r in range(n):
        kind = r % 4
        if kind == 0:                      # one pair
            a, b = torch.randperm(k, generator=g)[:2].tolist()
            idx[r, a] = idx[r, b]
        elif kind == 1:                    # a few tokens, all often
            idx[r] = idx[r, torch.randint(0, 5, (k,), generator=g)]
        elif kind == 2:                    # pairs among tokens 2048 apart
            base = int(torch.randint(0, min(v, 2048), (1,), generator=g))
            pool = torch.arange(base, v, 2048)
            idx[r] = pool[torch.randint(0, len(pool), (k,), generator=g)]
    check(x, idx.to(DEV), tlp, tail=tail)


@pytest.mark.parametrize("sizes", [(60000, 24000), (21000, 9000), (4000, 900)])
def test_two_threads_with_different_vocabularies(sizes):
    """Calls from two host threads at once, each with its own vocabulary and stream, over kernels that
    they share: none is refused and each gives what it gives alone.  The library is called as often
    as it can be, on buffers made before."""
    import threading

    from kernels import _ak
    n, k, times = 640, 16, 6000
    device = torch.device(DEV, torch.cuda.current_device())
    mask = torch.zeros(n, dtype=torch.bool, device=DEV)
    mask[::80] = True                      # short calls: host threads meet in the library, not on the GPU
    calls, errors, start = [], [], threading.Barrier(len(sizes))
    for v in sizes:
        x, idx, tlp = rows(n, v, k, torch.bfloat16, 11)
        want = _ak.distill_topk_fwd(x, idx, tlp, mask, tail=True, want_grad=True)
        out = [torch.empty_like(t) for t in (want[0], want[1], want[2], want[3])]
        args = [_ak.ptr(t) for t in out] + [None, None, _ak.ptr(x), _ak.ptr(idx), _ak.ptr(tlp), _ak.ptr(mask), n, n, 0, v, v, k,
                                            1.0, 0.0, 1, _ak.dtype_code(x),
                                            _ak.status_ptr(device, "distill_topk")]
        calls.append((args, out, want, (x, idx, tlp)))
    torch.cuda.synchronize()

    def work(args, out, want, _):
        try:
            stream = torch.cuda.Stream()
            start.wait(timeout=60)
            for _ in range(times):
                _ak.call("ak_distill_topk_fwd", *args, stream.cuda_stream)
            stream.synchronize()
            assert torch.equal(out[1], want[1]) and torch.equal(out[3][mask], want[3][mask])
        except Exception as e:  # noqa: BLE001 - reported below
            errors.append(e)

    threads = [threading.Thread(target=work, args=c) for c in calls]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    _ak.check_status(device)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n", [1, 2, 22])
def test_the_longest_rows(n, dtype):
    """As many elements as eight CTAs' shared memory holds: 851,968 of 16 bits or 425,984 of fp32 (and
    the rest of a group); more rows than the GPU takes clusters at once; rows that start anywhere."""
    from kernels import _ak
    from kernels.distill import distill_topk
    v = (425_984 if dtype == torch.float32 else 851_968) + 15
    full, _, _ = rows(n, v + 1, 1, dtype, 12)
    g = torch.Generator().manual_seed(13)
    for x in (full[:, :v], full[:, 1:]):
        idx = torch.randint(0, v, (n, 64), generator=g).to(DEV)
        idx[:, 0], idx[:, 1] = 0, v - 1
        tlp = torch.log_softmax(torch.randn(n, 64, generator=g), 1).to(DEV) - 0.2
        if n <= 2:
            check(x, idx, tlp, tail=True)
            continue
        mask = torch.rand(n, generator=g).to(DEV) < 0.8
        mask[n - 1] = True
        loss, losses, _, grad, _, _ = _ak.distill_topk_fwd(x, idx, tlp, mask, tail=True, want_grad=True)
        at = [0, n // 2, n - 1]
        ref = O.distill_topk(x[at].double().cpu(), idx[at].cpu(), tlp[at].cpu(), mask[at].cpu(), tail=True)
        O.assert_within(losses[at], ref["losses"], ref["tol_losses"], "losses")
        f = max(1, int(mask[at].sum())) / int(mask.sum())
        O.assert_within(grad[at], ref["grad"] * f, ref["tol_grad"] * f, "grad")
    _ak.check_status(torch.device(DEV))
    with pytest.raises(RuntimeError, match="does not fit"):
        distill_topk(torch.zeros(1, v + 1 + 8 * 16, dtype=dtype, device=DEV), idx[:1], tlp[:1])

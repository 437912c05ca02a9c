"""Arguments of the token log-probabilities: refusals and row addressing, without a GPU."""
import ctypes

import pytest
import torch

from kernels import _ak
from kernels import token_logprobs as TL


def on_gpu(monkeypatch):
    """Lets CPU tensors pass the device check, so that the checks behind it are reached."""
    monkeypatch.setattr(_ak, "require_cuda", lambda *t: torch.device("cpu"))


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="CUDA"):
        TL.token_logprobs(torch.zeros(2, 8), torch.zeros(2, dtype=torch.long))


@pytest.mark.parametrize("bad,err", [
    (dict(logits=torch.zeros(2, 8, dtype=torch.float64)), TypeError),
    (dict(logits=torch.zeros(())), ValueError),
    (dict(logits=torch.zeros(2, 0)), ValueError),
    (dict(targets=torch.zeros(2)), TypeError),
    (dict(targets=torch.zeros(2, dtype=torch.bool)), TypeError),
    (dict(targets=torch.zeros(3, dtype=torch.long)), ValueError),
    (dict(targets=torch.zeros(2, 1, dtype=torch.long)), ValueError),
    (dict(top_k=-1), ValueError), (dict(top_k=9), ValueError),
    (dict(logits=torch.zeros(2, 500), top_k=129), ValueError),
    (dict(temperature=0.0), ValueError), (dict(temperature=-1.0), ValueError),
    (dict(temperature=float("inf")), ValueError), (dict(temperature=float("nan")), ValueError),
    (dict(softcap=-1.0), ValueError), (dict(softcap=float("nan")), ValueError)])
def test_refusals(monkeypatch, bad, err):
    on_gpu(monkeypatch)
    args = dict(logits=torch.zeros(2, 8), targets=torch.zeros(2, dtype=torch.long))
    args.update(bad)
    with pytest.raises(err):
        TL.token_logprobs(args.pop("logits"), args.pop("targets"), **args)


def test_library_refusals():
    lib = _ak.lib()
    fake = ctypes.c_void_p(256)  # never dereferenced: each call fails its checks first

    def fwd(rows=2, inner=2, V=64, k=0, T=1.0, cap=0.0, dt=1, logits=fake, targets=fake, lp=fake, top=fake):
        return lib.ak_token_logprobs_fwd(lp, None, None, None, top, top, logits, targets, rows, inner, 0, V, V, k, T,
                                         cap, -100, dt, None)

    assert fwd(dt=9) == 2
    for kw in (dict(V=0), dict(rows=-1), dict(inner=0), dict(k=65), dict(k=-1), dict(k=129, V=1000),
               dict(k=1, V=1 << 25), dict(rows=1 << 40)):
        assert fwd(**kw) == 3, kw
    for kw in (dict(T=0.0), dict(T=float("nan")), dict(T=float("inf")), dict(cap=-1.0), dict(logits=None),
               dict(targets=None), dict(k=3, top=None), dict(logits=ctypes.c_void_p(257))):
        assert fwd(**kw) == 1, kw
        assert lib.ak_last_error()
    assert fwd(rows=0) == 0

    def bwd(rows=2, V=64, grad=fake, stats=fake, targets=fake, gl=fake, ge=fake, T=1.0):
        return lib.ak_token_logprobs_bwd(grad, fake, targets, stats, gl, ge, rows, 2, 0, V, V, T, 0.0, -100, 1, None)

    for kw in (dict(grad=None), dict(stats=None), dict(targets=None), dict(stats=ctypes.c_void_p(264)), dict(T=-1.0),
               dict(grad=ctypes.c_void_p(257))):
        assert bwd(**kw) == 1, kw
    assert bwd(rows=0) == 0


def addresses(x):
    t, rows, inner, so, si = _ak.logit_rows(x)
    first = (t.data_ptr() - x.data_ptr()) // x.element_size() if t is x else None
    return t, rows, [(r // inner) * so + (r % inner) * si for r in range(rows)], first


def test_row_addressing():
    full = torch.arange(3 * 6 * 11).float().view(3, 6, 11)
    views = [full, full[:, :-1], full[:, -1], full[..., :9], full[:, 1:, 2:7], full[1, 2], full[:, ::2], full[::2],
             full[:1].expand(4, 6, 11), full[:, :, None, :], full[0:0], full.transpose(0, 1)]
    for x in views:
        t, rows, offs, first = addresses(x)
        assert t is x, "taken as it lies"
        want = x.reshape(-1, x.shape[-1])
        assert rows == want.shape[0]
        base = x.storage_offset()
        store = full.view(-1)
        for r, o in enumerate(offs):
            assert torch.equal(store[base + o:base + o + x.shape[-1]], want[r])


def test_rows_that_are_copied():
    full = torch.arange(2 * 3 * 4 * 5 * 6).float().view(2, 3, 4, 5, 6)
    for x in (full.transpose(-1, -2), full[:, ::2, ::3, :4], full.permute(2, 0, 1, 3, 4)[:, :, :2]):
        t, rows, offs, _ = addresses(x)
        want = x.reshape(-1, x.shape[-1])
        assert rows == want.shape[0]
        for r, o in enumerate(offs):
            assert torch.equal(torch.as_strided(t, (x.shape[-1],), (1,), t.storage_offset() + o), want[r])


@pytest.mark.parametrize("bad,err", [
    (dict(h=torch.zeros(2, 16)), TypeError),
    (dict(h=torch.zeros(2, 12, dtype=torch.bfloat16), w=torch.zeros(9, 12)), ValueError),
    (dict(h=torch.zeros(2, 0, dtype=torch.bfloat16), w=torch.zeros(9, 0)), ValueError),
    (dict(w=torch.zeros(9, 24)), ValueError), (dict(w=torch.zeros(16)), ValueError),
    (dict(w=torch.zeros(0, 16)), ValueError), (dict(w=torch.zeros(9, 16, dtype=torch.float64)), TypeError),
    (dict(t=torch.zeros(3, dtype=torch.long)), ValueError), (dict(t=torch.zeros(2)), TypeError),
    (dict(temperature=0.0), ValueError), (dict(softcap=-2.0), ValueError)])
def test_linear_refusals(monkeypatch, bad, err):
    on_gpu(monkeypatch)
    args = dict(h=torch.zeros(2, 16, dtype=torch.bfloat16), w=torch.zeros(9, 16), t=torch.zeros(2, dtype=torch.long))
    args.update(bad)
    with pytest.raises(err):
        TL.linear_token_logprobs(args.pop("h"), args.pop("w"), args.pop("t"), **args)


def test_linear_library_refusals():
    lib = _ak.lib()
    fake = ctypes.c_void_p(256)  # never dereferenced: each call fails its checks first
    n = ctypes.c_size_t(0)
    assert lib.ak_linear_logprobs_workspace_size(8, 64, 100, 0, None) == 1
    assert lib.ak_linear_logprobs_workspace_size(8, 0, 100, 0, ctypes.byref(n)) == 3
    assert lib.ak_linear_logprobs_workspace_size(8, 64, 100, 0, ctypes.byref(n)) == 0 and n.value > 8 * 2 * 12
    fwd_ws = n.value
    assert lib.ak_linear_logprobs_workspace_size(8, 64, 100, 1, ctypes.byref(n)) == 0 and n.value > 8 * 104 * 2
    bwd_ws = n.value

    def fwd(H=fake, lse=fake, lp=fake, t=fake, N=8, D=64, V=100, T=1.0, cap=0.0, dt=1, ws=fwd_ws):
        return lib.ak_linear_logprobs_fwd(lp, None, lse, None, fake, ws, H, fake, t, N, D, V, T, cap, -100, dt, None,
                                          None)

    assert fwd(dt=0) == 2
    for kw in (dict(D=12), dict(D=0), dict(V=0), dict(N=-1), dict(V=1 << 31)):
        assert fwd(**kw) == 3, kw
    for kw in (dict(H=None), dict(H=ctypes.c_void_p(258)), dict(lse=None), dict(t=None), dict(T=0.0), dict(cap=-1.0)):
        assert fwd(**kw) == 1, kw
    assert fwd(ws=fwd_ws - 1) == 6
    assert fwd(N=0) == 0

    def bwd(dH=fake, stats=fake, t=fake, gl=fake, ge=fake, ws=bwd_ws, N=8):
        return lib.ak_linear_logprobs_bwd(dH, fake, fake, ws, fake, fake, t, stats, gl, ge, N, 64, 100, 1.0, 0.0, -100,
                                          1, None, None)

    for kw in (dict(dH=ctypes.c_void_p(258)), dict(stats=None), dict(t=None), dict(stats=ctypes.c_void_p(264))):
        assert bwd(**kw) == 1, kw
    assert bwd(ws=bwd_ws - 1) == 6
    assert bwd(N=0) == 0

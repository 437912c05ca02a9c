"""Token log-probabilities from hidden states: calls at the edges of what the documentation allows."""
import pytest
import torch

from oracle import logit_row_oracle as O
from test_gpu_linear_logprobs import grad_reference, problem

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,d,v", [(3, 72, 257), (65, 128, 1001), (300, 768, 5003), (700, 520, 9000), (16384 + 5, 64, 515),
                                   (2 * 16384 + 300, 8, 70)])
@pytest.mark.parametrize("up", [1.0, 2.0 ** -24])
def test_gradient_of_an_fp32_weight(n, d, v, dtype, up):
    """It is the accumulators', never rounded to 16 bits: at 2^-24 fp16 would lose it.  The weight's
    values are of the 16-bit type here, so that its cast loses nothing."""
    from kernels.token_logprobs import linear_token_logprobs
    h, w, t = problem(n, d, v, dtype, seed=31)
    g = torch.Generator().manual_seed(n)
    gl, ge = torch.randn(n, generator=g) * up, torch.randn(n, generator=g) * 0.2 * up
    hg, wg = h.clone().requires_grad_(True), w.float().requires_grad_(True)
    r = linear_token_logprobs(hg, wg, t, entropy=True)
    dh, dw = torch.autograd.grad([r.logprobs, r.entropy], [hg, wg], [gl.to(DEV), ge.to(DEV)])
    assert dw.dtype == torch.float32
    rh, th, rw, tw = grad_reference(h, w, t, gl, ge, two=n <= 256)
    O.assert_within(dh, rh, th, "dH")
    O.assert_within(dw, rw, tw, "dW")
    only, = torch.autograd.grad(linear_token_logprobs(h, wg, t).logprobs, wg, gl.to(DEV))
    rh, th, rw, tw = grad_reference(h, w, t, gl, None, two=n <= 256)
    O.assert_within(only, rw, tw, "dW alone")


@pytest.mark.parametrize("dtype", DTYPES)
def test_gradient_of_a_weight_of_the_other_16_bit_type(dtype):
    from kernels.token_logprobs import linear_token_logprobs
    other = torch.float16 if dtype == torch.bfloat16 else torch.bfloat16
    h, _, t = problem(40, 64, 300, dtype, seed=32)
    w = (torch.randint(-4, 5, (300, 64), generator=torch.Generator().manual_seed(1)) * 0.125).to(DEV)
    gl = torch.randn(40, generator=torch.Generator().manual_seed(2))
    wg = w.to(other).requires_grad_(True)
    dw, = torch.autograd.grad(linear_token_logprobs(h, wg, t).logprobs, wg, gl.to(DEV))
    assert dw.dtype == other
    _, _, rw, tw = grad_reference(h, w.to(dtype), t, gl, None, two=True)
    O.assert_within(dw, rw, tw + rw.abs() * 2.0 ** -23, "dW")  # by way of fp32


def test_no_rows_and_an_fp32_weight():
    from kernels.token_logprobs import linear_token_logprobs
    h = torch.zeros(0, 64, dtype=torch.bfloat16, device=DEV)
    w = torch.randn(50, 64, device=DEV, requires_grad=True)
    r = linear_token_logprobs(h, w, torch.zeros(0, dtype=torch.long, device=DEV))
    dw, = torch.autograd.grad(r.logprobs.sum(), w)
    assert dw.dtype == torch.float32 and (dw == 0).all()

"""Block norm's gradients on rows far from one in size, against the formulas in 64 bits. The kernels' arithmetic is fp32, so what they
form on the way has to stay inside its range wherever the result does."""
import pytest
import torch

from maltos_b200.ops import _lib
from maltos_b200.ops.norm import block_norm

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _norm(t, w):
    return w * t * torch.rsqrt(t.square().mean(-1, keepdim=True))


SIZES = [(1e13, 1e13, 1.0), (1e15, 1e15, 1.0), (5e17, 5e17, 1.0), (5e17, 1.0, 1.0), (1.0, 5e17, 1e-6), (1e-13, 1e-13, 1.0), (1e-17, 1e-17, 1.0),
         (1e-18, 1.0, 1.0)]


@pytest.mark.parametrize("after,before,only", [(True, True, None), (True, True, "y"), (True, True, "h"), (True, False, None), (False, True, None),
                                               (False, True, "y"), (False, True, "h")])
# (in wide rows the forward's sum of squares leaves fp32 from some 1e17 on)
@pytest.mark.parametrize("dtype,H,size_x,size_r,size_g", [(dtype, H, *size) for dtype, H in ((torch.float32, 64), (torch.float32, 8192), (torch.bfloat16, 64), (torch.bfloat16, 264))
                                                          for size in SIZES if H < 1000 or max(size) < 1e16])
def test_gradients_of_huge_and_tiny_rows(size_x, size_r, size_g, after, before, only, dtype, H):
    g = torch.Generator(device=DEV).manual_seed(H)
    rnd = lambda *s: torch.randn(*s, device=DEV, generator=g)                # noqa: E731
    x, r = (size_x * rnd(5, H)).to(dtype).requires_grad_(), (size_r * rnd(5, H)).to(dtype).requires_grad_()
    w1, w2 = ((1 + 0.2 * rnd(H)).to(dtype).requires_grad_() for _ in range(2))
    scale = 0.7 if after else 0.5
    res = block_norm(x, r, w1 if after else None, w2 if before else None, scale=scale, eps=0.0)
    outs = list(res) if before else [res]
    douts = [(size_g * rnd(5, H)).to(dtype) for _ in outs]
    if only == "y":
        outs, douts = outs[:1], douts[:1]
    elif only == "h":
        outs, douts = outs[-1:], douts[-1:]
    got = torch.autograd.grad(outs, (x, r), douts)
    _lib.fetch_status()

    X, R = (t.detach().double().requires_grad_() for t in (x, r))
    h = R + scale * (_norm(X, w1.detach().double()) if after else X)
    exact = ([_norm(h, w2.detach().double())] if before else []) + [h]
    exact = exact[:1] if only == "y" else exact[-1:] if only == "h" else exact
    want = torch.autograd.grad(exact, (X, R), [d.double() for d in douts])
    # A gradient is a sum of up to three products whose sizes are that of the row's largest gradient (nothing cancels to less than a
    # tenth of it in random rows): fp32 gives 2^-16 of that, bf16 its own rounding, that of h and of h's share of the means
    tol = 2.0 ** -16 if dtype == torch.float32 else 2.0 ** -6
    for name, a, b in zip(("dx", "dresidual"), got, want):
        top = b.abs().amax(-1, keepdim=True)
        assert torch.isfinite(a).all(), name
        # below fp32's smallest normal number (and bf16's, the same) the steps stop shrinking
        assert ((a.double() - b).abs() <= tol * top + 2.0 ** -126).all(), (name, ((a.double() - b).abs() / top).max().item())

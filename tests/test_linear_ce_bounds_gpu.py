"""Gradients of the linear head's cross entropy (ops/linear_ce.py), element by element and in the 2-norm, at ordinary sizes.

d = g slope (p - [v = target]) is what both gradients sum; dw = d^T x, dx = d w.  Its error, and from it the bounds:

* a logit sums D products in blocks of 16; each block's sum is cut, not rounded, with the other terms aligned to its largest: 2^-22 of
  A = sum |x w| covers a block, (D / 16 + 2) 2^-22 A all of them (``e_x``);
* the score: e_x, since the cap's slope is at most 1, and 2^-20 of the cap (of 1 + the largest score without one) for its functions;
* p, relative: the score's error, the same once more from the row's log sum, 2^-18 for exponentials, logarithm and the sum itself;
* the slope, absolute: 2^-20 and the change over e_x (at most e_x, as |slope'| < 1 for caps of 2 and more); 0 without a cap;
* d is rounded to bf16, 2^-8, and a gradient's element once more.  A gradient's own sum is cut like a logit's.

Single elements: all of that at its largest, added up.  The 2-norm: the roundings of d are independent, so that the norm of what they
leave is at most 2^-8 of sqrt(sum d^2 |x|^2), whose mean is a third of that squared; errors of p are the same for all tokens or independent
from token to token: their bound times the norm of the softmax's part of dw, and times sqrt(sum (g slope p)^2 |x|^2)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
SIZES = [(512, 256, 1024), (1500, 512, 8192), (130, 384, 50021), (2049, 1024, 2047), (300, 512, 17003), (700, 200, 5003)]


def inputs(N, D, V, seed=0, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    x = torch.randn(N, D, generator=g, device=device).bfloat16()
    w = (torch.randn(V, D, generator=g, device=device) * (2.5 / D ** 0.5)).bfloat16()
    t = torch.randint(0, V, (N,), generator=g, device=device)
    t = torch.where(torch.rand(N, generator=g, device=device) < 0.2, torch.full_like(t, -100), t)
    return x, w, t, torch.rand(N, generator=g, device=device) + 0.5


def wanted(x, w, t, weight, cap):
    """{name: (gradient, bound of its elements, bound of its norm, the softmax's part of it)} in 64 bits."""
    x, w, g = x.double(), w.double(), weight.double()
    (N, D), V = x.shape, w.shape[0]
    z = x @ w.T
    s = cap * torch.tanh(z / cap) if cap else z
    slope = 1 - (s / cap) ** 2 if cap else torch.ones_like(z)
    p = torch.softmax(s, 1)
    counts = t >= 0
    g = torch.where(counts, g, 0.0)[:, None]
    hot = torch.zeros_like(p).scatter_(1, t.clamp(min=0)[:, None], 1.0)
    d, soft = g * slope * (p - hot), g * slope * p

    e_x = (D / 16 + 2) * 2.0 ** -22 * (x.abs() @ w.abs().T)
    e_s = e_x + 2.0 ** -20 * (cap if cap else 1 + s.abs().amax(1, keepdim=True))
    e_p = e_s + e_s.amax(1, keepdim=True) + 2.0 ** -18
    e_d = soft * e_p + g * (p - hot).abs() * ((2.0 ** -20 + e_x) if cap else 0.0) + g * hot * 2.0 ** -22
    off = 1.01 * (e_d + 2.0 ** -8 * d.abs())
    out = {}
    for name, a, b, n in (("dx", "nv,vd->nd", w, V), ("dw", "nv,nd->vd", x, N)):
        grad, part = torch.einsum(a, d, b), torch.einsum(a, soft, b)
        size = torch.einsum(a, d.abs(), b.abs())
        element = torch.einsum(a, off, b.abs()) + (n / 16 + 4) * 2.0 ** -22 * size + 2.0 ** -8 * grad.abs()
        other = b.square().sum(1)[:, None] if name == "dw" else b.square().sum(1)[None, :]
        spread, soft_spread = (math.sqrt(float((m.square() * other).sum())) for m in (d, soft))
        norm = 2.0 ** -8 * (spread + float(grad.norm())) + float(e_p.max()) * (soft_spread + float(part.norm()))
        norm += float(((g * (p - hot).abs() * (2.0 ** -20 + e_x)).square() * other).sum().sqrt()) if cap else 0.0
        out[name] = grad, element, norm, part
    return out


@pytest.mark.parametrize("N,D,V", SIZES)
@pytest.mark.parametrize("cap", [0.0, 15.0, 100.0])
def test_gradients_within_the_bounds_of_their_roundings(N, D, V, cap):
    from autoresearch_b200.ops import kernels as K
    from autoresearch_b200.ops.linear_ce import linear_cross_entropy
    x, w, t, weight = inputs(N, D, V)
    x.requires_grad_(True)
    w.requires_grad_(True)
    got = torch.autograd.grad(linear_cross_entropy(x, w, t, softcap=cap), (x, w), weight)
    K.check_err_flag()
    for a, (name, (grad, element, norm, part)) in zip(got, wanted(x.detach(), w.detach(), t, weight, cap).items()):
        # the bounds say something: a gradient without its softmax part is outside of both
        if name == "dw":
            assert float(part.norm()) > norm and float((part.abs() > element).double().mean()) > 0.5
        off = (a.double() - grad).abs()
        assert float(off.norm()) <= norm, f"{name}: {float(off.norm()):.3e} > {norm:.3e} of {float(grad.norm()):.3e}"
        assert bool((off <= element).all()), f"{name}: an element by {float((off / element).max()):.2f} of its bound"

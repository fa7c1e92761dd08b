"""Cross entropy of a linear head without its logits (ops/linear_ce.py) against the definition in 64 bits.

Tolerances.  Losses: products are exact in fp32 and summed in fp32, D terms of size at most |x||w|: a logit is off by at most
D 2^-24 |x||w| (in the worst order); the functions of the soft cap and the softmax by 2^-20 of the cap (or of the logit) each;
lse and target score differ by their sum.  Gradients: d is rounded to bf16 (2^-8 of each term), the result once more (2^-8):
2 x 2^-8 in the 2-norm over a tensor; rows of cancelling terms are held against the mean row norm.  Where the softmax is one
(a vocabulary of one id), what remains is the error of the probability: score, log sum and their difference are each rounded by
2^-20 up to 32 in size (units of log 2), so p by 3 ln 2 2^-20 < 2^-18, and more in proportion for larger scores; that times
|w| (dx), or |x| and the number of rows (dw), and the weight of at most 1.5 is allowed in every row."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _inputs(N, D, V, ignored=0.0, seed=0, scale=2.5, wide=True):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(N, D, generator=g, device="cuda").bfloat16()
    w = (torch.randn(V, D, generator=g, device="cuda") * (scale / D ** 0.5)).bfloat16()
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    t = torch.where(torch.rand(N, generator=g, device="cuda") < ignored, torch.full_like(t, -100), t)
    weight = torch.rand(N, generator=g, device="cuda") + 0.5
    return x, w, (t if wide else t.int()), weight


def _reference(x, w, t, weight, cap):
    x, w, weight = x.detach().double(), w.detach().double(), weight.double()
    z = x @ w.T
    s = cap * torch.tanh(z / cap) if cap else z
    ok = (t >= 0) & (t < w.shape[0])
    at = torch.where(ok, t, 0).long()[:, None]
    loss = torch.where(ok, torch.logsumexp(s, 1) - s.gather(1, at)[:, 0], 0.0)
    d = torch.softmax(s, 1)
    d.scatter_add_(1, at, -torch.ones_like(at, dtype=torch.float64))
    d *= torch.where(ok, weight, 0.0)[:, None]
    if cap:
        d *= 1 - (s / cap) ** 2
    return loss, d @ w, d.T @ x


def _run(x, w, t, weight, cap):
    from autoresearch_b200.ops.linear_ce import linear_cross_entropy
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = linear_cross_entropy(x, w, t, softcap=cap)
    return (loss.detach(),) + torch.autograd.grad(loss, (x, w), weight)


def _loss_bound(x, w, cap):
    D = x.shape[1]
    top = float(x.double().norm(dim=1).max() * w.double().norm(dim=1).max())
    return 2 * (D * 2.0 ** -24 * top + 2.0 ** -20 * (cap if cap else max(top, 1.0)))


def _compare(got, want, x, w, cap, what):
    loss, dx, dw = (a.double() for a in got)
    top = lambda a: float(a.double().norm(dim=1).max())  # noqa: E731
    p_off = 1.5 * 2.0 ** -18 * max(1.0, 1.45 * (cap if cap else top(x) * top(w)) / 32)
    assert float((loss - want[0]).abs().max()) <= _loss_bound(x, w, cap), what
    for name, a, b, floor in (("dx", dx, want[1], p_off * top(w)), ("dw", dw, want[2], p_off * top(x) * x.shape[0])):
        assert bool(torch.isfinite(a).all()), f"{what}: {name}"
        assert float((a - b).norm()) <= 2.0 ** -7 * float(b.norm()) + floor * b.shape[0] ** 0.5, f"{what}: {name} {float((a - b).norm() / b.norm()):.2e}"
        ref = b.norm(dim=1)
        worst = float(((a - b).norm(dim=1) - 2.0 ** -5 * torch.maximum(ref, ref.square().mean().sqrt())).max())
        assert worst <= floor, f"{what}: a row of {name} by {worst:.2e}"


def _check(N, D, V, cap, ignored=0.0, seed=0, scale=2.5, wide=True):
    from autoresearch_b200.ops import kernels as K
    x, w, t, weight = _inputs(N, D, V, ignored, seed, scale, wide)
    got = _run(x, w, t, weight, cap)
    K.check_err_flag()
    _compare(got, _reference(x, w, t, weight, cap), x, w, cap, f"{N} x {D} x {V}, cap {cap}")
    ok = (t >= 0) & (t < V)
    assert bool((got[0][~ok] == 0).all()) and bool((got[1][~ok] == 0).all())


@pytest.mark.parametrize("N,D,V", [(1, 8, 1), (1, 64, 2), (3, 8, 255), (255, 72, 256), (256, 128, 257), (257, 256, 1000), (512, 256, 1024),
                                   (700, 200, 5003), (1500, 512, 8192), (130, 384, 50021), (2049, 1024, 2047), (515, 200, 9001), (300, 512, 17003)])
@pytest.mark.parametrize("cap", [0.0, 15.0, 50.0, 100.0])
def test_linear_cross_entropy(N, D, V, cap):
    _check(N, D, V, cap, ignored=0.2 if N > 3 else 0.0)


def test_targets_of_32_bits_and_all_ignored():
    _check(300, 64, 777, 15.0, ignored=0.3, wide=False)
    x, w, t, weight = _inputs(64, 64, 100, ignored=1.1)
    loss, dx, dw = _run(x, w, t, weight, 0.0)
    for a in (loss, dx, dw):
        assert bool((a == 0).all())
    for bad in (100, 2 ** 40, -1, -2 ** 62):
        x, w, t, weight = _inputs(64, 64, 100)
        t[10] = bad
        loss, dx, _ = _run(x, w, t, weight, 0.0)
        assert float(loss[10]) == 0 and bool((dx[10] == 0).all()) and float(loss[11]) > 0


@pytest.mark.parametrize("cap", [0.0, 15.0, 50.0])
def test_logits_far_apart(cap):
    """Uncapped logits of a hundred and more: the running maximum; capped ones at the cap, where the slope vanishes."""
    _check(400, 128, 3000, cap, scale=40.0)


@pytest.mark.parametrize("cap", [2.0 ** -64, 2.0 ** -10])
def test_small_caps(cap):
    _check(257, 64, 600, cap, 0.1)


def test_pieces_of_the_vocabulary(monkeypatch):
    """Pieces that end inside a tile and a last piece of a single id give what one piece gives."""
    from autoresearch_b200.ops import linear_ce as L
    x, w, t, weight = _inputs(300, 128, 2049, 0.1)
    want = _run(x, w, t, weight, 15.0)
    monkeypatch.setattr(L, "PIECE_BYTES", 2 * 300 * 512)
    L._backward_plan.cache_clear()
    try:
        assert L._backward_plan(300, 128, 2049)[3] == 5
        got = _run(x, w, t, weight, 15.0)
    finally:
        L._backward_plan.cache_clear()
    assert torch.equal(got[0], want[0]) and torch.equal(got[2], want[2])
    _compare(got, _reference(x, w, t, weight, 15.0), x, w, 15.0, "pieces")


def test_twice_the_same_bits():
    x, w, t, weight = _inputs(1000, 256, 3001, 0.1)
    a, b = _run(x, w, t, weight, 15.0), _run(x, w, t, weight, 15.0)
    for p, q in zip(a, b):
        assert torch.equal(p, q)


def test_strides():
    x, w, t, weight = _inputs(200, 64, 301)
    want = _run(x, w, t, weight, 0.0)
    forms = [torch.zeros(200, 136, dtype=x.dtype, device="cuda")[:, 8:72], torch.zeros(200, 67, dtype=x.dtype, device="cuda")[:, 1:65],
             torch.zeros(64, 200, dtype=x.dtype, device="cuda").t(), torch.zeros(200 * 64 + 1, dtype=x.dtype, device="cuda")[1:].view(200, 64)]
    for f in forms:
        for p, q in zip(_run(f.copy_(x), w, t, weight, 0.0), want):
            assert torch.equal(p, q)
    two = torch.stack([t, t], 1)[:, 0]
    for p, q in zip(_run(x, w, two, torch.stack([weight, weight], 1)[:, 1], 0.0), want):
        assert torch.equal(p, q)
    same = torch.ones((), device="cuda").expand(200)        # the gradient of a sum
    for p, q in zip(_run(x, w, t, same, 0.0), _run(x, w, t, torch.ones(200, device="cuda"), 0.0)):
        assert torch.equal(p, q)


def test_main_gradient_takes_the_weights_share():
    from autoresearch_b200.ops.linear_ce import linear_cross_entropy
    x, w, t, weight = _inputs(500, 128, 1111)
    _, dx, dw = _run(x, w, t, weight, 15.0)
    p = torch.nn.Parameter(w.clone())
    p.main_grad = torch.full(w.shape, 0.5, device="cuda")
    x.requires_grad_(True)
    (linear_cross_entropy(x, p, t, softcap=15.0) * weight).sum().backward()
    assert p.grad is None and torch.equal(x.grad, dx)
    assert float((p.main_grad - 0.5 - dw.float()).norm()) <= 2.0 ** -8 * float(dw.float().norm()) + 2.0 ** -24 * w.numel() ** 0.5


def test_gradient_against_differences():
    """f = sum(weight loss) along its own gradient; the third-order term and the rounding of x + u to bf16 (which the difference of
    the rounded points already counts) stay below 2 %."""
    from autoresearch_b200.ops.linear_ce import linear_cross_entropy
    x, w, t, weight = _inputs(300, 128, 900, 0.1, seed=5)
    _, dx, dw = _run(x, w, t, weight, 15.0)

    def f(x, w):
        with torch.no_grad():
            return float((linear_cross_entropy(x, w, t, softcap=15.0).double() * weight.double()).sum())

    for i, g in ((0, dx), (1, dw)):
        at = (x, w)
        u = g.float() * (0.02 * float(at[i].float().square().mean().sqrt()) / float(g.float().square().mean().sqrt()))
        hi, lo = ((at[i].float() + s * u).bfloat16() for s in (1, -1))
        want = float((g.double() * (hi.double() - lo.double())).sum()) / 2
        diff = (f(*((hi, w) if i == 0 else (x, hi))) - f(*((lo, w) if i == 0 else (x, lo)))) / 2
        assert abs(diff - want) <= 0.02 * abs(want), (i, diff, want)


def test_graph_replay():
    x, w, t, weight = _inputs(400, 128, 700)
    x, w = x.requires_grad_(True), w.requires_grad_(True)
    from autoresearch_b200.ops.linear_ce import linear_cross_entropy

    def step():
        loss = linear_cross_entropy(x, w, t, softcap=15.0)
        return (loss.detach(),) + torch.autograd.grad(loss, (x, w), weight)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for shift in (0, 13):
        with torch.no_grad():
            t.copy_((t + shift) % 700)
            x.mul_(1.25)
        graph.replay()
        for p, q in zip(got, _run(x, w, t, weight, 15.0)):
            assert torch.equal(p, q)


def test_only_one_gradient_asked_for():
    from autoresearch_b200.ops.linear_ce import linear_cross_entropy
    x, w, t, weight = _inputs(100, 64, 300)
    _, dx, dw = _run(x, w, t, weight, 0.0)
    a = x.clone().requires_grad_(True)
    linear_cross_entropy(a, w, t).backward(weight)
    assert torch.equal(a.grad, dx)
    b = w.clone().requires_grad_(True)
    linear_cross_entropy(x, b, t).backward(weight)
    assert torch.equal(b.grad, dw)
    assert not linear_cross_entropy(x, w, t).requires_grad


def test_a_weight_of_more_elements_than_32_bits_count():
    """The last ids of 2.1 million: their gradient rows and a loss whose target is the very last one."""
    D, V, N = 1024, (1 << 21) + 300, 40
    g = torch.Generator(device="cuda").manual_seed(0)
    w = torch.empty(V, D, dtype=torch.bfloat16, device="cuda").normal_(0.0, 0.05, generator=g)
    x = torch.empty(N, D, dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    t = torch.randint(0, V, (N,), generator=g, device="cuda")
    t[:4] = torch.arange(V - 4, V, device="cuda")
    weight = torch.ones(N, device="cuda")
    loss, dx, dw = _run(x, w, t, weight, 15.0)
    s = 15 * torch.tanh(x.double() @ w.double().T / 15)
    lse = torch.logsumexp(s, 1)
    want = lse - s.gather(1, t[:, None])[:, 0]
    assert float((loss.double() - want).abs().max()) <= _loss_bound(x, w[-1000:], 15.0) * 4
    d = torch.exp(s[:, -300:] - lse[:, None])
    for i in range(4):
        d[i, 300 - 4 + i] -= 1
    d *= 1 - (s[:, -300:] / 15) ** 2
    rows = d.T @ x.double()
    assert float((dw[-300:].double() - rows).norm()) <= 2.0 ** -7 * float(rows.norm())
    del w, dw, s
    torch.cuda.empty_cache()


def test_second_derivatives_are_refused():
    from autoresearch_b200.ops.linear_ce import linear_cross_entropy
    x, w, t, weight = _inputs(10, 64, 300)
    x.requires_grad_(True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(linear_cross_entropy(x, w, t), x, weight, create_graph=True)


def test_hooks_may_hand_back_other_tensors():
    """What hooks on saved tensors return is read, in its layout, and not the forward call's memory; the main gradient of a
    parameter takes its share all the same."""
    from autoresearch_b200.ops.linear_ce import linear_cross_entropy
    x, w, t, weight = _inputs(300, 128, 1111, 0.2)
    _, dx, dw = _run(x, w, t, weight, 15.0)
    seen = []

    def pack(s):
        seen.append(s)
        return s.detach().clone(memory_format=torch.contiguous_format)
    for main in (False, True):
        wide = torch.cat([x, x], 1).requires_grad_(True)
        rows = wide[:, 128:]
        p = torch.nn.Parameter(w.clone())
        if main:
            p.main_grad = torch.zeros(w.shape, device="cuda")
        at = t.clone()
        with torch.autograd.graph.saved_tensors_hooks(pack, lambda s: s):
            loss = linear_cross_entropy(rows, p, at, softcap=15.0)
        for s in seen:
            s.data.fill_(float("nan") if s.is_floating_point() else -1)
        loss.backward(weight)
        assert torch.equal(wide.grad[:, 128:], dx)
        if main:
            assert p.grad is None
            assert float((p.main_grad - dw.float()).norm()) <= 2.0 ** -8 * float(dw.float().norm())
        else:
            assert torch.equal(p.grad, dw)


def test_activation_checkpointing():
    from torch.utils.checkpoint import checkpoint

    from autoresearch_b200.ops.linear_ce import linear_cross_entropy
    x, w, t, weight = _inputs(700, 64, 3001, 0.2)
    f = lambda a, b: linear_cross_entropy(a * 2, b * 0.5, t + 0, softcap=15.0)  # noqa: E731
    grads = []
    for run in (f, lambda *a: checkpoint(f, *a, use_reentrant=False)):
        a = [s.detach().requires_grad_(True) for s in (x, w)]
        loss = run(*a)
        junk = [torch.full_like(s, float("nan")) for s in (x, w)] + [torch.full_like(t, -1) for _ in range(3)]
        loss.backward(weight)
        del junk
        grads.append([s.grad for s in a])
    for a, b in zip(*grads):
        assert torch.equal(a, b)


def test_no_tokens():
    x, w, t, weight = _inputs(0, 64, 300)
    loss, dx, dw = _run(x, w, t, weight, 0.0)
    assert loss.shape == (0,) and dx.shape == (0, 64) and bool((dw == 0).all())


@pytest.mark.parametrize("cap", [0.0, 15.0, 50.0])
def test_values_that_are_not_finite_show_in_their_row_and_in_no_other(cap):
    from autoresearch_b200.ops.linear_ce import linear_cross_entropy
    x, w, t, weight = _inputs(300, 64, 1000)
    want = linear_cross_entropy(x, w, t, softcap=cap)
    x[7, 3], x[131, 0] = float("nan"), float("inf")
    got = linear_cross_entropy(x, w, t, softcap=cap)
    assert bool(torch.isnan(got[7]))
    assert not bool(torch.isfinite(got[131])) or cap > 0          # a capped logit of an infinity is the cap
    rest = [i for i in range(300) if i not in (7, 131)]
    assert torch.equal(got[rest], want[rest])


@pytest.mark.parametrize("cap", [15.0, 30.0, 40.0, 41.0])
@pytest.mark.parametrize("N,D", [(1993, 64), (256, 352)])
def test_one_id_under_caps_with_and_without_a_fixed_maximum(N, D, cap):
    """The softmax is one; what a gradient has left is the error of the log sum."""
    _check(N, D, 1, cap)

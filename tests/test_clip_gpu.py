"""Gradient norm and clipping (optim/clip.py) against 64 bits.

Tolerances: 32 squares are added in fp32 (at most 34 roundings of 2^-24 of the sum, half of that in its root), everything above
in 64 bits, the norm is rounded to fp32: 2^-19.  A clipped element is multiplied by a factor rounded to fp32 (2^-24, with the
norm's 2^-19) and rounded to its type: 2^-18 + half a step, and half of the smallest subnormal."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
SIZES = [(1,), (7, 3), (8192,), (8193,), (8191, 1), (16384,), (16385,), (49151,), (100, 333), (5, 0), (30,), (1 << 18,), (3,), (123457,), ()]


def _grads(sizes, dtype, seed=0, scale=1e-2, back_to_back=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = [(torch.randn(s, generator=g, device="cuda") * scale * (1 + i % 4)).to(dtype) for i, s in enumerate(sizes)]
    if back_to_back:
        flat, at = torch.cat([t.reshape(-1) for t in out]), 0
        views = []
        for t in out:
            views.append(flat[at:at + t.numel()].view(t.shape))
            at += t.numel()
        return views
    return out


def _norm(grads):
    return math.sqrt(math.fsum(float(t.double().square().sum()) for t in grads))


def _check_scaled(got, source, factor):
    tiny = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}
    for o, t in zip(got, source):
        want = t.double() * factor
        tol = (2.0 ** -18 + torch.finfo(o.dtype).eps / 2) * want.abs() + tiny[o.dtype]
        assert bool(((o.double() - want).abs() <= tol).all()), (tuple(t.shape), t.dtype, o.dtype)


@pytest.mark.parametrize("back_to_back", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_norm(dtype, back_to_back):
    from autoresearch_b200.optim.clip import GradSet, grad_norm
    grads = _grads(SIZES, dtype, back_to_back=back_to_back)
    want = _norm(grads)
    got = grad_norm(grads)
    assert got.dtype is torch.float32 and got.shape == () and abs(float(got) - want) <= 2.0 ** -19 * want
    assert torch.equal(grad_norm(GradSet(grads)), got) and torch.equal(grad_norm(grads[::-1][::-1]), got)


@pytest.mark.parametrize("ratio", [0.5, 1.5, 300.0])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("to", [None, torch.float32, torch.bfloat16, torch.float16])
def test_clip(dtype, to, ratio):
    from autoresearch_b200.optim.clip import clip_grad_norm
    grads = _grads(SIZES, dtype, back_to_back=True)
    source = [t.clone() for t in grads]
    want = _norm(source)
    out = None if to is None else _grads(SIZES, to, seed=1, back_to_back=True)
    norm = clip_grad_norm(grads, want / ratio, out=out)
    assert abs(float(norm) - want) <= 2.0 ** -19 * want
    _check_scaled(grads if out is None else out, source, min(1.0, 1.0 / ratio))
    if to is not None or ratio < 1:
        for a, b in zip(grads, source):
            assert torch.equal(a, b)


def test_mixed_types_and_many_tensors():
    from autoresearch_b200.optim.clip import GradSet, clip_grad_norm, grad_norm
    types = [torch.float32, torch.bfloat16, torch.float16]
    grads = [_grads([(1 + (i * 37) % 500,)], types[i % 3], seed=i)[0] for i in range(2100)]
    source = [t.clone() for t in grads]
    want = _norm(grads)
    s = GradSet(grads)
    assert abs(float(grad_norm(s)) - want) <= 2.0 ** -19 * want
    assert abs(float(clip_grad_norm(s, want / 4)) - want) <= 2.0 ** -19 * want
    _check_scaled(grads, source, 0.25)
    # the same set again sees what is in the buffers now
    now = _norm(grads)
    assert abs(float(grad_norm(s)) - now) <= 2.0 ** -19 * now


@pytest.mark.parametrize("size", [1e-38, 1e-30, 1e-18, 1e15, 1e25, 1e36])
def test_norms_beyond_the_range_of_fp32_squares(size):
    from autoresearch_b200.optim.clip import grad_norm
    g = torch.Generator(device="cuda").manual_seed(0)
    for dtype in (torch.float32, torch.bfloat16):
        t = [((torch.rand(n, generator=g, device="cuda") + 0.5) * size).to(dtype) for n in (1000, 20000)]
        want = _norm(t)
        assert abs(float(grad_norm(t)) - want) <= 2.0 ** -19 * want


def test_one_large_element_among_zeros():
    from autoresearch_b200.optim.clip import grad_norm
    t = torch.zeros(100003, device="cuda")
    t[77777] = 3e20
    assert abs(float(grad_norm([t])) - 3e20) <= 2.0 ** -19 * 3e20
    assert float(grad_norm([torch.zeros(5000, device="cuda")])) == 0.0


@pytest.mark.parametrize("bad", [float("inf"), float("nan")])
def test_norms_that_are_not_finite_scale_nothing(bad):
    from autoresearch_b200.optim.clip import clip_grad_norm
    grads = _grads([(100,), (9000,)], torch.float32)
    grads[1][4000] = bad
    source = [t.clone() for t in grads]
    norm = float(clip_grad_norm(grads, 1e-3))
    assert math.isnan(norm) if math.isnan(bad) else math.isinf(norm)
    out = [torch.zeros_like(t) for t in grads]
    clip_grad_norm(grads, 1e-3, out=out)
    for a, b, c in zip(grads, source, out):
        assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) and torch.equal(c.nan_to_num(7.0), b.nan_to_num(7.0))


def test_neighbours_in_memory_stay_as_they_were():
    from autoresearch_b200.optim.clip import clip_grad_norm
    for dtype in (torch.float32, torch.bfloat16):
        for offset in range(1, 9):
            buf = torch.full((16384 + 64,), 5.0, dtype=dtype, device="cuda")
            clip_grad_norm([buf[offset:offset + 16384 + 13]], 1.0)
            assert bool((buf[:offset] == 5).all()) and bool((buf[offset + 16384 + 13:] == 5).all())
            assert bool((buf[offset:offset + 16384 + 13] < 1).all())


def test_memory_orders():
    from autoresearch_b200.optim.clip import clip_grad_norm
    t = _grads([(40, 60)], torch.float32)[0].t()
    source = t.clone()
    want = _norm([t])
    clip_grad_norm([t], want / 2)
    _check_scaled([t], [source], 0.5)


def test_twice_the_same_bits_and_graph_replay():
    from autoresearch_b200.optim.clip import GradSet, clip_grad_norm, grad_norm
    grads = _grads([(123457,), (1000, 1000), (30,)], torch.float32)
    assert torch.equal(grad_norm(grads), grad_norm(grads))
    out = [torch.zeros_like(t, dtype=torch.bfloat16) for t in grads]
    s = GradSet(grads, out=out)
    clip_grad_norm(s, 1.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grad_norm(s, 1.0)
    for f in (1.0, 0.37):
        for t in grads:
            t.mul_(f)
        graph.replay()
        want = _norm(grads)
        assert abs(float(norm) - want) <= 2.0 ** -19 * want
        _check_scaled(out, grads, min(1.0, 1.0 / want))


def test_tensors_that_were_given_other_memory():
    from autoresearch_b200.optim.clip import GradSet, grad_norm
    grads = _grads([(1000,), (2000,)], torch.float32)
    s = GradSet(grads)
    grads[1].data = torch.full((2000,), 2.0, device="cuda")
    want = _norm(grads)
    assert abs(float(grad_norm(s)) - want) <= 2.0 ** -19 * want


def test_a_copy_of_a_set_scales_its_own_tensors():
    import copy

    from autoresearch_b200.optim.clip import GradSet, clip_grad_norm
    grads = _grads(SIZES[:6], torch.float32)
    source = [t.clone() for t in grads]
    other = copy.deepcopy(GradSet(grads))
    norm = clip_grad_norm(other, 0.25 * _norm(source))
    assert abs(float(norm) - _norm(source)) <= 2.0 ** -19 * _norm(source)
    assert all(torch.equal(a, b) for a, b in zip(grads, source))
    _check_scaled(other.tensors, source, 0.25)


def test_more_elements_than_32_bits_count():
    from autoresearch_b200.optim.clip import clip_grad_norm
    n = (1 << 31) + 4099
    t = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    t[-5:] = 3.0
    t[(1 << 31) - 2:(1 << 31) + 2] = 1.0
    assert abs(float(clip_grad_norm([t], 3.5)) - 7.0) <= 2.0 ** -16
    assert float(t[-1]) == 1.5 and float(t[1 << 31]) == 0.5 and float(t[0]) == 0.0
    del t
    torch.cuda.empty_cache()


def test_refusals():
    from autoresearch_b200.optim.clip import GradSet, clip_grad_norm, grad_norm
    t = torch.zeros(10, 10, device="cuda")
    for bad in ([t, t], [t, t[3:]], [t[:, :5]], [t.expand(3, 10, 10)]):
        with pytest.raises(ValueError):
            grad_norm(bad)
    for bad in ([t.double()], [t.cpu()], [t.int()], [None]):
        with pytest.raises(TypeError):
            grad_norm(bad)
    with pytest.raises(ValueError):
        clip_grad_norm([t], 1.0, out=[torch.zeros(5, 20, device="cuda")])
    with pytest.raises(ValueError):
        clip_grad_norm([t], 1.0, out=[torch.zeros(10, 10, device="cuda").t()])
    with pytest.raises(ValueError):
        clip_grad_norm([t[:5]], 1.0, out=[t[3:8]])
    with pytest.raises(ValueError):
        clip_grad_norm(GradSet([t]), 1.0, out=[t.clone()])
    clip_grad_norm([t, t.clone()], 1.0, out=[t, torch.zeros(10, 10, device="cuda")])      # one of them in place
    assert float(grad_norm([])) == 0.0 and float(grad_norm([torch.zeros(0, device="cuda")])) == 0.0


@pytest.mark.parametrize("size,max_norm", [(1e36, 1e-3), (3e35, 2e-6), (1e37, 1e-8), (1e30, 1e-30), (1e36, 30.0)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_factors_below_the_normal_numbers_of_fp32(dtype, size, max_norm):
    """max_norm / norm may be smaller than 2^-126 while the scaled elements are not."""
    from autoresearch_b200.optim.clip import clip_grad_norm
    g = torch.Generator(device="cuda").manual_seed(0)
    grads = [((torch.rand(n, generator=g, device="cuda") + 0.5) * size).to(dtype) for n in (1000, 20001)]
    source = [t.clone() for t in grads]
    factor = max_norm / _norm(source)
    out = [torch.zeros_like(t, dtype=torch.bfloat16 if dtype is torch.float32 else torch.float32) for t in grads]
    clip_grad_norm(grads, max_norm, out=out)
    _check_scaled(out, source, factor)
    clip_grad_norm(grads, max_norm)
    _check_scaled(grads, source, factor)
    if max_norm * 2e-3 > 2.0 ** -126:
        assert min(float(t.float().abs().min()) for t in grads + out) > 0


@pytest.mark.parametrize("bad", [None, float("inf")])
@pytest.mark.parametrize("to", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_gradients_that_are_not_scaled_are_copied_as_they_are(dtype, to, bad):
    """Subnormal elements among them: bit for bit in their own type, rounded once into another."""
    from autoresearch_b200.optim.clip import clip_grad_norm
    n = 20003
    t = torch.randn(n, dtype=torch.float64, generator=torch.Generator().manual_seed(0)) * 2.0 ** -(torch.arange(n) % 150).double()
    t = t.to(dtype)
    if bad is not None:
        t[777] = bad
    out = torch.zeros(n, dtype=to, device="cuda")
    clip_grad_norm([t.cuda()], 1e4, out=[out])
    assert torch.equal(out.cpu(), t.to(to))


def test_finite_gradients_of_a_norm_beyond_fp32_are_scaled():
    from autoresearch_b200.optim.clip import clip_grad_norm
    grads = [torch.full((5000,), 3e38, device="cuda"), torch.full((100,), -2e36, device="cuda", dtype=torch.bfloat16)]
    source = [t.clone() for t in grads]
    assert math.isinf(float(clip_grad_norm(grads, 1.0)))
    _check_scaled(grads, source, 1.0 / _norm(source))
    one = [torch.full((1,), 3.4e38, device="cuda")]
    assert math.isfinite(float(clip_grad_norm(one, 1.0))) and abs(float(one[0]) - 1.0) <= 2.0 ** -18


@pytest.mark.parametrize("how", ["resize", "data", "type"])
def test_tensors_that_kept_their_address_but_not_their_size(how):
    """All of it inside of one allocation: what lies behind the smaller tensor stays as it was."""
    from autoresearch_b200.optim.clip import GradSet, clip_grad_norm
    buf = torch.full((40000,), 2.0, device="cuda")
    t, other = buf[:40000], _grads([(500,)], torch.float32)[0]
    s = GradSet([t, other])
    if how == "resize":
        t.resize_(1000)
    elif how == "data":
        t.data = buf[:1000].view(10, 100)
    else:
        t.data = buf.view(torch.bfloat16)[:40000]
    source = [t.clone(), other.clone()]
    want = _norm(source)
    assert abs(float(clip_grad_norm(s, want / 4)) - want) <= 2.0 ** -19 * want
    _check_scaled([t, other], source, 0.25)
    assert bool((buf[20000 if how == "type" else 1000:] == 2.0).all())


def test_strides_of_dimensions_of_one_do_not_count():
    from autoresearch_b200.optim.clip import clip_grad_norm
    grads = [torch.randn(1, 300, device="cuda"), torch.randn(7, 1, 20, device="cuda")]
    out = [torch.zeros(300, 1, device="cuda").t(), torch.zeros(1, 7, 20, device="cuda", dtype=torch.bfloat16).transpose(0, 1)]
    assert all(o.shape == t.shape and o.stride() != t.stride() for t, o in zip(grads, out))
    clip_grad_norm(grads, _norm(grads) / 2, out=out)
    _check_scaled(out, grads, 0.5)
    with pytest.raises(ValueError, match="does not match"):
        clip_grad_norm([torch.zeros(3, 1, 5, device="cuda")], 1.0, out=[torch.zeros(5, 1, 3, device="cuda").permute(2, 1, 0)])

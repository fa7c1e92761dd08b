"""Attention over packed sequences (ops/packed.py) against the definition in 64 bits.

Tolerances: probabilities and dS are rounded to bf16 (2^-8 relative) before they are summed, results once more on the way out
(2^-8); dS also takes up the rounding of O through rowsum(dO o O) (2^-8).  Everything else is fp32.  That is at most 2 x 2^-8
for O and dV and 3 x 2^-8 for dQ and dK, relative to what is summed; rows are compared relative to the larger of their own
norm and the mean row norm, since sums of terms that cancel keep the terms' rounding: 2^-6 for every output.

A query that sees one key has dS = dP - rowsum(dO o O) = 0, as the difference of two fp32 sums of the same d <= 128 products in
different orders: each is off by at most d 2^-24 |dO||v|, so dS by 2^-16 |dO||v|, and the rows of dQ (dK) by that times scale |k|
(|q|, for each head of the group).  ``_floors`` gives that much to every row."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
TOL = 2.0 ** -6


def _bounds(lengths, lead=0):
    b = [lead]
    for n in lengths:
        b.append(b[-1] + n)
    return b


def _reference(q, k, v, bounds, window, scale, d_out):
    """O, dQ, dK, dV in 64 bits, sequence by sequence and head by head; zero outside of the sequences."""
    q, k, v, d_out = (t.detach().double() for t in (q, k, v, d_out))
    H, G = q.shape[1], q.shape[1] // k.shape[1]
    o, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    for a, b in zip(bounds[:-1], bounds[1:]):
        i = torch.arange(b - a, device=q.device)
        seen = (i[None, :] <= i[:, None]) & (i[None, :] >= i[:, None] - window)
        for h in range(H):
            g = h // G
            s = torch.where(seen, (q[a:b, h] @ k[a:b, g].T) * scale, -math.inf)
            p = torch.softmax(s, 1)
            o[a:b, h] = p @ v[a:b, g]
            dp = d_out[a:b, h] @ v[a:b, g].T
            ds = p * (dp - (p * dp).sum(1, keepdim=True)) * scale
            dq[a:b, h] = ds @ k[a:b, g]
            dk[a:b, g] += ds.T @ q[a:b, h]
            dv[a:b, g] += p.T @ d_out[a:b, h]
    return o, dq, dk, dv


def _inputs(rows, H, KV, d, seed=0, dtype=torch.bfloat16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    mk = lambda h: torch.randn(rows, h, d, generator=g, device="cuda").to(dtype)  # noqa: E731
    return mk(H), mk(KV), mk(KV), mk(H)


def _run(q, k, v, d_out, seqs, window=None, scale=None):
    from autoresearch_b200.ops.packed import packed_attention
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    out = packed_attention(q, k, v, seqs, window=window, scale=scale)
    return (out.detach(),) + torch.autograd.grad(out, (q, k, v), d_out)


def _floors(q, k, v, d_out, scale):
    top = lambda t: float(t.double().norm(dim=-1).max()) if t.numel() else 0.0  # noqa: E731
    ds = 2.0 ** -16 * top(d_out) * top(v) * scale
    return 0.0, ds * top(k), ds * top(q) * (q.shape[1] // k.shape[1]), 0.0


def _compare(got, want, what, floors):
    for name, x, y, floor in zip(("out", "dq", "dk", "dv"), got, want, floors):
        x = x.double()
        assert x.shape == y.shape and bool(torch.isfinite(x).all()), f"{what}: {name}"
        err, ref = (x - y).norm(dim=-1), y.norm(dim=-1)
        mean = ref.square().mean().sqrt()
        off, allowed = float((x - y).norm()), TOL * float(y.norm()) + floor * math.sqrt(err.numel())
        assert off <= allowed, f"{what}: {name} {off:.3e} > {allowed:.3e}"
        # single rows: the rounding of one term may be most of a row; four times the bound of the sum
        worst = float((err - 4 * TOL * torch.maximum(ref, mean) - floor).max())
        assert worst <= 0, f"{what}: a row of {name} is off by {worst:.3e} more than allowed"


def _check(lengths, H, KV, d, window=None, lead=0, pad=0, scale=None, seed=0):
    from autoresearch_b200.ops import kernels as K
    from autoresearch_b200.ops.packed import PackedSequences
    bounds = _bounds(lengths, lead)
    rows = bounds[-1] + pad
    q, k, v, d_out = _inputs(rows, H, KV, d, seed)
    seqs = PackedSequences(bounds, rows, H, KV)
    got = _run(q, k, v, d_out, seqs, window, scale)
    torch.cuda.synchronize()
    K.check_err_flag()
    scale = 1 / math.sqrt(d) if scale is None else scale
    want = _reference(q, k, v, bounds, rows if window is None else window, scale, d_out)
    _compare(got, want, f"{lengths} {H}/{KV} heads of {d}, window {window}", _floors(q, k, v, d_out, scale))


def _plan_lists(seqs):
    items = seqs.items[:4 * (seqs.cap_q + seqs.cap_k)].view(-1, 4).cpu()
    return items[:seqs.cap_q], items[seqs.cap_q:]


@pytest.mark.parametrize("bounds,rows,H,KV", [
    ([0, 512], 512, 2, 2), ([0, 1], 1, 1, 1), ([0], 77, 4, 2), ([5, 5, 5, 300, 300], 1000, 6, 2), ([0, 4096, 4097, 9000], 9000, 8, 1),
    (list(range(0, 3001)), 3005, 3, 1), ([0, 33000], 33000, 5, 5)])
def test_plan_covers_every_row_once(bounds, rows, H, KV):
    from autoresearch_b200.ops.packed import PackedSequences
    seqs = PackedSequences(bounds, rows, H, KV)
    for items, step in zip(_plan_lists(seqs), (128 // (H // KV), 128)):
        live = items[items[:, 1] > 0]
        seen = torch.zeros(rows, dtype=torch.int64)
        starts = {a: b - a for a, b in zip(bounds[:-1], bounds[1:]) if b > a}
        for start, n, tile, _ in live.tolist():
            if tile < 0:
                assert n <= step and (start + n <= bounds[0] or start >= bounds[-1])
                seen[start:start + n] += 1
            else:
                assert starts[start] == n
                seen[start + tile * step:start + min(n, (tile + 1) * step)] += 1
        assert bool((seen == 1).all())
        assert bool((items[len(live):, 1] == 0).all()), "live tiles come first"


@pytest.mark.parametrize("device_bounds", [[0, 300, 100, 700], [-5, 100, 2000], [900, 100], [2 ** 31 - 1, -2 ** 31, 7]])
def test_bounds_of_the_device_that_make_no_sense_stay_inside_and_are_reported(device_bounds):
    from autoresearch_b200.ops import kernels as K
    from autoresearch_b200.ops.packed import PackedSequences
    K.check_err_flag()
    rows = 777
    seqs = PackedSequences(torch.tensor(device_bounds, dtype=torch.int32, device="cuda"), rows, 2, 1)
    for items, step in zip(_plan_lists(seqs), (64, 128)):
        seen = torch.zeros(rows, dtype=torch.int64)
        for start, n, tile, _ in items.tolist():
            a, b = (start, start + n) if tile < 0 else (start + tile * step, start + min(n, (tile + 1) * step))
            assert n == 0 or 0 <= a < b <= rows
            seen[a:b] += 1
        assert bool((seen == 1).all())
    with pytest.raises(K.KernelError, match="sequence bounds"):
        K.check_err_flag()


@pytest.mark.parametrize("lengths,H,KV,d,window", [
    ([1], 1, 1, 128, None), ([128], 1, 1, 128, None), ([129], 2, 1, 128, None), ([127, 1, 1, 128, 2], 2, 2, 128, None),
    ([1, 130, 77, 304], 2, 2, 128, None), ([300, 0, 0, 41], 4, 2, 128, None), ([517], 4, 1, 64, None), ([1000, 24], 8, 2, 64, None),
    ([333, 200], 3, 1, 128, None), ([450, 61], 10, 2, 64, None), ([260], 16, 1, 128, None), ([200, 3], 128, 1, 64, None),
    ([150], 100, 1, 64, None), ([70, 1, 5], 65, 1, 128, None),
    ([900], 1, 1, 128, 0), ([900, 100], 2, 1, 128, 1), ([1200], 2, 2, 128, 100), ([1200, 333], 6, 2, 128, 256), ([1025], 5, 1, 64, 127),
    ([2100], 3, 3, 64, 128), ([1500, 700], 4, 1, 128, 1499)])
def test_packed_attention(lengths, H, KV, d, window):
    _check(lengths, H, KV, d, window)


@pytest.mark.parametrize("lead,pad", [(7, 0), (0, 300), (130, 1)])
def test_rows_of_no_sequence_are_zero(lead, pad):
    _check([200, 65], 4, 2, 128, lead=lead, pad=pad)
    _check([200, 65], 3, 1, 64, lead=lead, pad=pad, window=50)


def test_many_short_sequences():
    _check([1, 2, 3, 4, 5, 6, 7] * 60, 4, 4, 128)


@pytest.mark.parametrize("n", [200, 256, 384, 520])
def test_many_sequences_of_a_few_tiles(n):
    """Blocks that take many tiles of two to five steps each, without a pause between them: every sequence comes out as it does
    alone, three times over."""
    from autoresearch_b200.ops.packed import PackedSequences
    many, H, KV, d = 400, 2, 1, 128
    one = _inputs(n, H, KV, d)
    alone = _run(*one, PackedSequences([0, n], n, H, KV))
    all_ = [t.repeat(many, 1, 1) for t in one]
    seqs = PackedSequences([i * n for i in range(many + 1)], many * n, H, KV)
    for _ in range(3):
        for x, y in zip(_run(*all_, seqs), alone):
            assert torch.equal(x, y.repeat(many, 1, 1))


def test_scale_is_the_callers():
    _check([400], 2, 1, 128, scale=0.02)


@pytest.mark.parametrize("scale", [2.0 ** -64, 2.0 ** -30])
def test_small_scales(scale):
    """Every key counts alike."""
    _check([300, 1, 77], 4, 2, 64, window=200, scale=scale)


@pytest.mark.parametrize("H,KV,d", [(2, 2, 128), (6, 2, 64), (8, 2, 128)])
def test_a_sequence_does_not_see_its_neighbours(H, KV, d):
    """Bit for bit the same alone, beside other sequences, and beside NaN and infinities in them and in the rows behind."""
    from autoresearch_b200.ops.packed import PackedSequences
    lengths, n = [77, 200, 391], 200
    rows = sum(lengths) + 50
    q, k, v, g = _inputs(rows, H, KV, d)
    sl = slice(77, 277)
    alone = _run(q[sl], k[sl], v[sl], g[sl], PackedSequences([0, n], n, H, KV))
    beside = _run(q, k, v, g, PackedSequences(_bounds(lengths), rows, H, KV))
    for x, y in zip(beside, alone):
        assert torch.equal(x[sl], y)
    for bad in (float("nan"), float("inf"), -float("inf")):
        for t in (q, k, v, g):
            t[:77] = bad
            t[277:] = bad
        hurt = _run(q, k, v, g, PackedSequences(_bounds(lengths), rows, H, KV))
        for x, y in zip(hurt, alone):
            assert torch.equal(x[sl], y)
            assert bool((x[sum(lengths):] == 0).all())


@pytest.mark.parametrize("d,H,KV", [(64, 2, 2), (128, 2, 2), (128, 8, 2), (64, 3, 1), (128, 96, 1)])
def test_what_the_rounding_of_the_output_leaves_is_kept(d, H, KV):
    """With q = 0 every key counts alike, P is 1 without a rounding and O a mean of at most 16 values: off by 16 x 2^-22 of their mean
    size (16 sums in fp32, rounded or cut), and 2^-15 of itself for the 8 bits kept beyond bf16.  Whole and ragged tiles."""
    from autoresearch_b200.ops import packed as P
    lengths = [16] * 40 + [5, 1, 0, 9]
    bounds = _bounds(lengths)
    rows = bounds[-1]
    _, _, v, _ = _inputs(rows, H, KV, d)
    q, k = torch.zeros(rows, H, d, dtype=torch.bfloat16, device="cuda"), v.roll(1, 0).contiguous()
    out, kept = P._forward(q, k, v, (H * d, d) + (KV * d, d) * 2, P.PackedSequences(bounds, rows, H, KV), rows, 0.125, True)
    rest = kept[:rows * H * d].view(rows, H, d)
    both = ((out.view(torch.int16).int() << 16) + (rest.int() << 8)).view(torch.float32).double()
    want, size = torch.zeros_like(both), torch.zeros_like(both)
    for a, b in zip(bounds[:-1], bounds[1:]):
        n = torch.arange(1, b - a + 1, device="cuda").double()[:, None, None]
        x = v[a:b].double().repeat_interleave(H // KV, 1)
        want[a:b], size[a:b] = x.cumsum(0) / n, x.abs().cumsum(0) / n
    assert bool(((both - want).abs() <= 2.0 ** -15 * want.abs() + 2.0 ** -18 * size).all())


def test_twice_the_same_bits():
    from autoresearch_b200.ops.packed import PackedSequences
    q, k, v, g = _inputs(3000, 6, 2, 128)
    a, b = (_run(q, k, v, g, PackedSequences([0, 1100, 1117, 3000], 3000, 6, 2), window=400) for _ in range(2))
    for x, y in zip(a, b):
        assert torch.equal(x, y)


def test_strides_and_alignment():
    """Column blocks of one projection, head-major storage, storage that the copy engine cannot read, expanded heads."""
    from autoresearch_b200.ops.packed import PackedSequences
    rows, H, KV, d = 333, 4, 2, 128
    q, k, v, g = _inputs(rows, H, KV, d)
    seqs = PackedSequences([0, 200, 333], rows, H, KV)
    want = _run(q, k, v, g, seqs)
    packed = torch.cat([q, k, v], 1)
    forms = [(packed[:, :H], packed[:, H:H + KV], packed[:, H + KV:], g)]
    forms.append(tuple(t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v, g)))

    def odd(t):
        buf = torch.empty(t.numel() + t.shape[0] * t.shape[1] + 1, dtype=t.dtype, device=t.device)
        return buf[1:1 + t.shape[0] * t.shape[1] * (d + 1)].view(t.shape[0], t.shape[1], d + 1)[..., :d].copy_(t)
    forms.append(tuple(odd(t) for t in (q, k, v, g)))
    forms.append(tuple(torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape) for t in (q, k, v, g)))
    for f in forms:
        for x, y in zip(_run(*f, seqs), want):
            assert torch.equal(x, y)
    one = k[:, :1].expand(rows, KV, d)
    got = _run(q, one, one, g[:, :1].expand(rows, H, d), seqs)
    want = _run(q, one.contiguous(), one.contiguous(), g[:, :1].expand(rows, H, d).contiguous(), seqs)
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_packed_projection_form_gives_the_same_bits():
    from autoresearch_b200.ops.packed import PackedSequences, packed_qkv_attention
    rows, H, KV, d = 500, 4, 2, 64
    q, k, v, g = _inputs(rows, H, KV, d)
    seqs = PackedSequences([0, 123, 490], rows, H, KV)
    want = _run(q, k, v, g, seqs, window=99)
    qkv = torch.cat([q, k, v], 1).view(rows, -1).requires_grad_(True)
    out = packed_qkv_attention(qkv, seqs, window=99, head_dim=d)
    (dqkv,) = torch.autograd.grad(out, qkv, g.view(rows, -1))
    assert torch.equal(out.view(rows, H, d), want[0])
    assert torch.equal(dqkv.view(rows, H + 2 * KV, d), torch.cat(want[1:], 1))


def test_gradient_against_differences():
    """f = sum(w o O) along its own gradient: (f(x + u) - f(x - u)) / 2 = grad . u up to third order in u.  |u| is 2^-4 of the
    input's norm per element; O is rounded to bf16, which leaves 2^-8 of sqrt(sum (w O)^2) in f, far below grad . u; the
    third-order term and the rounding of x + u to bf16 stay below 5 %."""
    from autoresearch_b200.ops.packed import PackedSequences, packed_attention
    rows, H, KV, d = 640, 4, 2, 128
    q, k, v, g = _inputs(rows, H, KV, d, seed=3)
    seqs = PackedSequences([0, 250, 640], rows, H, KV)
    _, *grads = _run(q, k, v, g, seqs)

    def f(*x):
        with torch.no_grad():
            return float((packed_attention(*x, seqs).double() * g.double()).sum())

    for i in range(3):
        x = [q, k, v]
        u = grads[i].float()
        u = u * (2.0 ** -4 / u.square().mean().sqrt())
        hi, lo = (x[i].float() + u).to(x[i].dtype), (x[i].float() - u).to(x[i].dtype)
        step = (hi.double() - lo.double()) / 2
        want = float((grads[i].double() * step).sum())
        diff = (f(*x[:i], hi, *x[i + 1:]) - f(*x[:i], lo, *x[i + 1:])) / 2
        assert abs(diff - want) <= 0.05 * abs(want), f"input {i}: {diff} against {want}"


def test_graph_replay_follows_new_bounds_and_inputs():
    from autoresearch_b200.ops.packed import PackedSequences, packed_attention
    rows, H, KV, d = 700, 4, 2, 128
    q, k, v, g = _inputs(rows, H, KV, d)
    cu = torch.tensor([0, 100, 700], dtype=torch.int32, device="cuda")
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))

    def step():
        out = packed_attention(q, k, v, PackedSequences(cu, rows, H, KV))
        return (out.detach(),) + torch.autograd.grad(out, (q, k, v), g)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for bounds in ([0, 100, 700], [0, 640, 650]):
        cu.copy_(torch.tensor(bounds, dtype=torch.int32))
        with torch.no_grad():
            q.mul_(0.9)
        graph.replay()
        want = _run(q, k, v, g, PackedSequences(bounds, rows, H, KV))
        for x, y in zip(got, want):
            assert torch.equal(x, y)


def test_other_stream():
    from autoresearch_b200.ops.packed import PackedSequences
    q, k, v, g = _inputs(1000, 2, 1, 128)
    want = _run(q, k, v, g, PackedSequences([0, 400, 1000], 1000, 2, 1))
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = _run(q, k, v, g, PackedSequences([0, 400, 1000], 1000, 2, 1))
    s.synchronize()
    for x, y in zip(got, want):
        assert torch.equal(x, y)


def test_lists_outlive_the_work_of_another_stream():
    """A packing that is dropped while another stream still has work with it: its memory is not given away before that is done."""
    from autoresearch_b200.ops.packed import PackedSequences, packed_attention
    q, k, v, _ = _inputs(1000, 2, 1, 128)
    seqs = PackedSequences([0] * 20_000 + [1000], 1000, 2, 1)
    at, n = seqs.items.data_ptr(), seqs.items.numel()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s), torch.no_grad():
        torch.cuda._sleep(200_000_000)                     # about 0.1 s
        out = packed_attention(q, k, v, seqs)
    del seqs
    held = [torch.empty(n, dtype=torch.int32, device="cuda") for _ in range(64)]
    assert not s.query() and at not in [t.data_ptr() for t in held]
    s.synchronize()
    del out, held


def test_offsets_beyond_32_bits():
    """More than 2^31 elements of q: the last sequences come out as they do alone."""
    from autoresearch_b200.ops.packed import PackedSequences
    rows, H, KV, d = 140_000, 128, 8, 128
    assert rows * H * d > 1 << 31
    n, last = 200, 140_000 - 200
    g = torch.Generator(device="cuda").manual_seed(0)
    q, do = (torch.empty(rows, H, d, dtype=torch.bfloat16, device="cuda").normal_(generator=g) for _ in range(2))
    k, v = (torch.empty(rows, KV, d, dtype=torch.bfloat16, device="cuda").normal_(generator=g) for _ in range(2))
    bounds = list(range(0, rows + 1, n))
    got = [t[last:].clone() for t in _run(q, k, v, do, PackedSequences(bounds, rows, H, KV))]
    want = _run(q[last:], k[last:], v[last:], do[last:], PackedSequences([0, n], n, H, KV))
    for x, y in zip(got, want):
        assert torch.equal(x, y)
    del q, do, k, v, got, want
    torch.cuda.empty_cache()


def test_second_derivatives_are_refused():
    from autoresearch_b200.ops.packed import PackedSequences, packed_attention, packed_qkv_attention
    q, k, v, g = (t.requires_grad_(True) for t in _inputs(64, 2, 1, 128))
    seqs = PackedSequences([0, 64], 64, 2, 1)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(packed_attention(q, k, v, seqs), q, g, create_graph=True)
    qkv = torch.cat([q, k, v], 1).detach().view(64, -1).requires_grad_(True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(packed_qkv_attention(qkv, seqs), qkv, g.view(64, -1), create_graph=True)


def test_the_same_graph_twice_and_inputs_changed_in_between():
    from autoresearch_b200.ops.packed import PackedSequences, packed_attention
    q, k, v, g = _inputs(300, 2, 1, 128)
    q, k, v = (t.requires_grad_(True) for t in (q, k, v))
    out = packed_attention(q, k, v, PackedSequences([0, 300], 300, 2, 1))
    a = torch.autograd.grad(out, (q, k, v), g, retain_graph=True)
    b = torch.autograd.grad(out, (q, k, v), g, retain_graph=True)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    with torch.no_grad():
        k.mul_(2.0)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        torch.autograd.grad(out, (q, k, v), g)


class _Elsewhere(torch.autograd.graph.saved_tensors_hooks):
    """Keeps dense copies of what is saved; ``spoil`` overwrites all the originals."""

    def __init__(self):
        self.seen = []
        super().__init__(self._pack, lambda t: t)

    def _pack(self, t):
        self.seen.append(t)
        return t.detach().clone(memory_format=torch.contiguous_format)

    def spoil(self):
        for t in self.seen:
            t.data.fill_(math.nan if t.is_floating_point() else 77)


@pytest.mark.parametrize("form", ["separate", "projection"])
def test_hooks_may_hand_back_other_tensors(form):
    """What hooks on saved tensors return is read, in its layout, and not the forward call's memory."""
    from autoresearch_b200.ops.packed import PackedSequences, packed_attention, packed_qkv_attention
    rows, H, KV, d = 333, 4, 2, 128
    q, k, v, g = _inputs(rows, H, KV, d)
    seqs = PackedSequences([0, 200, 333], rows, H, KV)
    want = torch.cat(_run(q, k, v, g, seqs)[1:], 1)
    qkv = torch.cat([q, k, v], 1).requires_grad_(True)
    hooks = _Elsewhere()
    if form == "separate":
        parts = qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:]
        with hooks:
            out = packed_attention(*parts, seqs)
        hooks.spoil()
        got = torch.cat(torch.autograd.grad(out, parts, g), 1)
    else:
        flat = qkv.detach().view(rows, -1).requires_grad_(True)
        with hooks:
            out = packed_qkv_attention(flat, seqs)
        hooks.spoil()
        got = torch.autograd.grad(out, flat, g.view(rows, -1))[0].view(rows, -1, d)
    assert hooks.seen and torch.equal(got, want)


def test_activation_checkpointing():
    from torch.utils.checkpoint import checkpoint

    from autoresearch_b200.ops.packed import PackedSequences, packed_attention
    q, k, v, g = _inputs(700, 4, 2, 64)
    seqs = PackedSequences([0, 333, 700], 700, 4, 2)
    f = lambda a, b, c: packed_attention(a * 2, b * 0.5, c + 1, seqs)  # noqa: E731
    grads = []
    for run in (f, lambda *x: checkpoint(f, *x, use_reentrant=False), lambda *x: checkpoint(f, *x, use_reentrant=True)):
        x = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = run(*x)
        junk = [torch.full_like(t, math.nan) for t in (q, k, v, g) * 3]          # takes memory that was let go of
        grads.append(torch.autograd.grad(out, x, g) if run is f else (out.backward(g), *(t.grad for t in x))[1:])
        del junk
    for other in grads[1:]:
        for a, b in zip(other, grads[0]):
            assert torch.equal(a, b)


def test_no_rows_and_no_sequences():
    from autoresearch_b200.ops.packed import PackedSequences
    q, k, v, g = _inputs(0, 2, 1, 128)
    assert [t.shape[0] for t in _run(q, k, v, g, PackedSequences([0], 0, 2, 1))] == [0] * 4
    q, k, v, g = _inputs(40, 2, 1, 128)
    for x in _run(q, k, v, g, PackedSequences([0, 0], 40, 2, 1)):
        assert bool((x == 0).all())


def test_no_rows_in_the_projection_form():
    from autoresearch_b200.ops.packed import PackedSequences, packed_qkv_attention
    for heads, d in ((2, 64), (4, 128)):
        qkv = torch.zeros(0, (heads + 2) * d, dtype=torch.bfloat16, device="cuda", requires_grad=True)
        out = packed_qkv_attention(qkv, PackedSequences([0], 0, heads, 1), head_dim=d)
        assert out.shape == (0, heads * d)
        out.sum().backward()
        assert qkv.grad.shape == qkv.shape


def test_refusals():
    from autoresearch_b200.ops.packed import PackedSequences, packed_attention, packed_qkv_attention
    rows, H, KV, d = 64, 4, 2, 128
    q, k, v, g = _inputs(rows, H, KV, d)
    seqs = PackedSequences([0, 64], rows, H, KV)
    with pytest.raises(TypeError):
        packed_attention(q.float(), k, v, seqs)
    with pytest.raises(TypeError):
        packed_attention(q.cpu(), k, v, seqs)
    with pytest.raises(TypeError):
        packed_attention(q, k, v, torch.tensor([0, 64], device="cuda"))
    with pytest.raises(ValueError):
        packed_attention(q[:, :, :96], k[:, :, :96], v[:, :, :96], seqs)
    with pytest.raises(ValueError):
        packed_attention(q[:32], k[:32], v[:32], seqs)
    with pytest.raises(ValueError):
        packed_attention(q, k[:, :1], v[:, :1], seqs)
    with pytest.raises(ValueError):
        packed_attention(q, k, v[:32], seqs)
    with pytest.raises(ValueError):
        packed_attention(q, k, v, seqs, window=-1)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="scale"):
            packed_attention(q, k, v, seqs, scale=scale)
    with pytest.raises(ValueError):
        packed_attention(q[0], k[0], v[0], seqs)
    with pytest.raises(TypeError):
        PackedSequences(torch.tensor([0, 64], device="cuda"), rows, H, KV)      # int64 on the device
    with pytest.raises(ValueError):
        packed_qkv_attention(torch.cat([q, k, v], 1).view(rows, -1)[:, 1:], seqs)
    with pytest.raises(ValueError):
        packed_qkv_attention(q.view(rows, -1), seqs)


@pytest.mark.parametrize("kind", ["list", "int32", "int64", "pinned"])
def test_host_bounds_are_taken_up_without_waiting(kind):
    """While the stream is busy the call returns, and what the caller writes to the bounds afterwards does not count."""
    from autoresearch_b200.ops.packed import PackedSequences
    bounds = [0, 300, 301, 700]
    make = {"list": list, "int32": lambda b: torch.tensor(b, dtype=torch.int32), "int64": torch.tensor,
            "pinned": lambda b: torch.tensor(b, dtype=torch.int32).pin_memory()}[kind]
    want = PackedSequences(torch.tensor(bounds, dtype=torch.int32, device="cuda"), 777, 4, 2)
    PackedSequences(make(bounds), 777, 4, 2)
    torch.cuda.synchronize()
    torch.cuda._sleep(400_000_000)                          # about 0.2 s
    given = make(bounds)
    seqs = PackedSequences(given, 777, 4, 2)
    busy = not torch.cuda.current_stream().query()
    given[1] = 5
    assert busy, "the call waited for the stream"
    torch.cuda.synchronize()
    assert torch.equal(seqs.cu_seqlens, want.cu_seqlens)
    for a, b in zip(_plan_lists(seqs), _plan_lists(want)):
        assert torch.equal(a, b)


def test_host_bounds_are_refused_under_graph_capture():
    from autoresearch_b200.ops.packed import PackedSequences
    x = torch.zeros(8, device="cuda")
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.add_(1.0)
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            PackedSequences([0, 4], 4, 2, 1)
    graph.replay()
    assert float(x[0]) == 1.0


@pytest.mark.parametrize("many", [False, True])
def test_host_bounds_where_another_device_is_the_default(many):
    from autoresearch_b200.ops.packed import PackedSequences
    bounds = list(range(301)) if many else [0, 300]
    with torch.device("cuda"):
        got = [PackedSequences(b, 300, 2, 1) for b in (bounds, torch.tensor(bounds, device="cpu"))]
    for s in got:
        assert s.cu_seqlens.is_cuda and s.cu_seqlens.tolist() == bounds

"""Checks of packed sequences that need no device, and the backward formula of packed attention against differences."""
import math

import pytest
import torch

from autoresearch_b200.ops import kernels as K
from autoresearch_b200.ops import packed as P


@pytest.mark.parametrize("bounds,rows", [([0, 5, 3], 10), ([-1, 4], 10), ([0, 11], 10), ([4, 2], 10)])
def test_host_bounds_are_checked(bounds, rows):
    with pytest.raises(ValueError, match="ascend"):
        P.PackedSequences(bounds, rows, 2, 1)
    with pytest.raises(ValueError, match="ascend"):
        P.PackedSequences(torch.tensor(bounds), rows, 2, 1)


@pytest.mark.parametrize("heads,kv", [(3, 2), (0, 1), (4, 0), (129, 1), (-2, 1)])
def test_head_layouts_that_do_not_group(heads, kv):
    with pytest.raises(ValueError, match="group"):
        P.PackedSequences([0, 4], 4, heads, kv)


def test_empty_bounds_and_rows_out_of_range():
    with pytest.raises(ValueError):
        P.PackedSequences([], 4, 2, 1)
    for rows in (-1, P.MAX_ROWS + 1):
        with pytest.raises(ValueError, match="rows"):
            P.PackedSequences([0], rows, 2, 1)


def test_bounds_that_are_no_whole_numbers():
    for bad in (torch.tensor([0.0, 4.0]), torch.tensor([[0, 4]]), [0, 2.5], torch.tensor([False, True])):
        with pytest.raises(TypeError):
            P.PackedSequences(bad, 4, 2, 1)


@pytest.mark.parametrize("device", ["cpu", torch.device("cpu"), "meta"])
def test_packing_on_another_kind_of_device_is_refused(device):
    """Before anything is launched: the plan kernel would be given host addresses."""
    with pytest.raises(ValueError, match="CUDA device"):
        P.PackedSequences([0, 4], 4, 2, 1, device=device)


def test_cpu_tensors_are_refused():
    t = torch.zeros(4, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="CUDA"):
        P.packed_attention(t, t, t, None)
    with pytest.raises(TypeError, match="CUDA"):
        P.packed_qkv_attention(t.view(4, -1), None)


@pytest.mark.parametrize("scale", [0.0, -0.5, 5e-324, 1e-50, 2.0 ** -65, 2.0 ** 65, 1e300, math.inf, math.nan])
def test_scales_that_fp32_does_not_hold_are_refused(scale):
    seqs = object.__new__(P.PackedSequences)
    seqs.rows, seqs.device = 4, torch.device("cpu")
    assert P._common(seqs.device, 4, 64, seqs, None, 2.0 ** -64) == (4, 2.0 ** -64)
    with pytest.raises(ValueError, match="scale"):
        P._common(seqs.device, 4, 64, seqs, None, scale)


def test_strides_that_the_copy_engine_can_read():
    t = torch.zeros(6, 3, 64, dtype=torch.bfloat16)
    same, row, head = P._layout(t)
    assert same is t and (row, head) == (192, 64)
    v = t.transpose(0, 1)
    same, row, head = P._layout(v)
    assert same is v and (row, head) == (64, 192)
    for bad in (t[:, :, ::2], t[:, :1].expand(6, 3, 64), t.view(-1)[:6 * 3 * 60].view(6, 3, 60)[:, :, :32]):
        dense, row, head = P._layout(bad)
        assert dense.is_contiguous() and dense is not bad and (row, head) == (3 * bad.shape[2], bad.shape[2])
    one = torch.zeros(1, 1, 67, dtype=torch.bfloat16)[:, :, :64]
    same, row, head = P._layout(one)
    assert same is one and (row, head) == (64, 64)


def test_argument_block_matches_the_header():
    import re
    from pathlib import Path
    text = (Path(K.__file__).parent / "csrc" / "api.h").read_text()
    body = re.sub(r"//[^\n]*", "", text[text.index("typedef struct ArbPacked"):text.index("} ArbPacked;")])
    fields = [f for line in body[body.index("{") + 1:].split(";") for f in line.split(",") if f.strip()]
    fields = [re.sub(r"^(const )?(void|int|float|double|long long)", "", f.strip()).strip(" *") for f in fields]
    assert len(fields) == 32 and P._ARGS.size == 8 * len(fields)
    assert " ".join(fields) == ("q k v o o_lo lse d_o delta dq dk dv items rows KV G D window cap_q cap_k q_row q_head k_row k_head "
                                "v_row v_head o_row do_row do_head dq_row dk_row dv_row scale")


def test_backward_formula_against_differences():
    """dS = P (dP - rowsum(dO o O)) and what follows from it, in 64 bits."""
    g = torch.Generator().manual_seed(0)
    q, k, v, w = (torch.randn(9, 4, generator=g, dtype=torch.float64) for _ in range(4))
    i = torch.arange(9)
    seen = (i[None] <= i[:, None]) & (i[None] >= i[:, None] - 5)
    scale = 0.5

    def f(q, k, v):
        p = torch.softmax(torch.where(seen, q @ k.T * scale, -math.inf), 1)
        return p, p @ v

    p, o = f(q, k, v)
    ds = p * (w @ v.T - (w * o).sum(1, keepdim=True))
    grads = (scale * ds @ k, scale * ds.T @ q, p.T @ w)
    for n, (x, dx) in enumerate(zip((q, k, v), grads)):
        for idx in ((0, 0), (3, 2), (8, 3)):
            e = torch.zeros_like(x)
            e[idx] = 1e-5
            hi, lo = ([t + e * s if m == n else t for m, t in enumerate((q, k, v))] for s in (1, -1))
            diff = ((f(*hi)[1] - f(*lo)[1]) * w).sum() / 2e-5
            assert abs(float(diff - dx[idx])) < 1e-7

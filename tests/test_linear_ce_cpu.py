"""Checks of the linear head's cross entropy that need no device."""
import re
from pathlib import Path

import pytest
import torch

from autoresearch_b200.ops import kernels as K
from autoresearch_b200.ops import linear_ce as L


def test_argument_block_matches_the_header():
    text = (Path(K.__file__).parent / "csrc" / "api.h").read_text()
    body = re.sub(r"//[^\n]*", "", text[text.index("typedef struct ArbLinearCE"):text.index("} ArbLinearCE;")])
    fields = [f for line in body[body.index("{") + 1:].split(";") for f in line.split(",") if f.strip()]
    fields = [re.sub(r"^(const )?(void|float|double|long long)", "", f.strip()).strip(" *") for f in fields]
    assert len(fields) == 19 and L._ARGS.size == 8 * len(fields)
    assert " ".join(fields) == "x w targets part target_score lse loss weight d_logits rows cols dim vocab col0 targets_64 ldx ldw ldd softcap"


@pytest.mark.parametrize("rows,vocab", [(1, 1), (512, 1024), (16384, 65536), (16384, 65537), (1 << 20, 131072), (1 << 24, 300), (7, 50021)])
def test_pieces_cover_the_vocabulary_in_whole_tiles(rows, vocab):
    cols = L.piece_columns(rows, vocab)
    assert 1 <= cols <= vocab and (cols == vocab or cols % L.TILE == 0)
    assert 2 * rows * cols <= max(L.PIECE_BYTES, 2 * rows * L.TILE)
    covered = sum(min(vocab, a + cols) - a for a in range(0, vocab, cols))
    assert covered == vocab


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(5, 8, dtype=torch.bfloat16)
    with pytest.raises(TypeError, match="CUDA"):
        L.linear_cross_entropy(x, w, torch.zeros(4, dtype=torch.int64))


@pytest.fixture
def no_device_check(monkeypatch):
    monkeypatch.setattr(K, "_bf16", lambda t, name: None)


@pytest.mark.parametrize("x,w,t,cap", [((4, 8), (5, 16), 4, 0.0), ((4, 12), (5, 12), 4, 0.0), ((4, 0), (5, 0), 4, 0.0), ((4, 8), (0, 8), 4, 0.0),
                                       ((4, 8), (5, 8), 3, 0.0), ((4, 8), (5, 8), 4, -1.0), ((4, 8), (5, 8), 4, float("inf")),
                                       ((4, 8), (5, 8), 4, float("nan")), ((4, 8), (5, 8), 4, 101.0), ((4, 8), (5, 8), 4, 2.0 ** -65),
                                       ((4, 8), (5, 8), 4, 5e-324), ((4, 8), (5, 8), 4, -0.5)])
def test_shapes_and_caps_that_are_refused(no_device_check, x, w, t, cap):
    with pytest.raises(ValueError):
        L.linear_cross_entropy(torch.zeros(x, dtype=torch.bfloat16), torch.zeros(w, dtype=torch.bfloat16), torch.zeros(t, dtype=torch.int64), cap)


def test_target_types_that_are_refused(no_device_check):
    x, w = torch.zeros(4, 8, dtype=torch.bfloat16), torch.zeros(5, 8, dtype=torch.bfloat16)
    for dtype in (torch.int16, torch.float32, torch.bool):
        with pytest.raises(ValueError, match="targets"):
            L.linear_cross_entropy(x, w, torch.zeros(4, dtype=dtype))


@pytest.mark.parametrize("rows,dim,piece,want", [(4099, 384, 50021, 2), (16384, 1024, 65536, 1), (512, 256, 1024, 1), (512, 256, 20000, 4),
                                                 (1, 8, 8191, 1), (1, 8, 8192, 2), (300, 512, 17003, 4)])
def test_parts_fill_the_pairs_of_multiprocessors(rows, dim, piece, want):
    got = K.lib().arb_linear_ce_parts(rows, dim, piece)
    assert got == want
    blocks = -(-piece // 64)
    per = -(-blocks // got)
    assert -(-blocks // per) == got          # no part is empty

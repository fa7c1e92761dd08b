"""Checks of gradient sets that need no device."""
import re
from pathlib import Path

import pytest
import torch

from autoresearch_b200.ops import kernels as K
from autoresearch_b200.optim import clip as C


def test_entry_matches_the_header():
    text = (Path(K.__file__).parent / "csrc" / "api.h").read_text()
    body = text[text.index("typedef struct ArbGrad {"):text.index("} ArbGrad;")]
    assert re.sub(r"\s+", " ", body[body.index("{") + 1:]).strip() == "const void* in; void* out; long long n; int type, out_type;"
    assert C._ENTRY.size == 32


def test_dense_tensors_in_any_order():
    t = torch.zeros(4, 6, 5)
    assert C._dense(t) and C._dense(t.permute(2, 0, 1)) and C._dense(t[:, :1][:2, :, :].permute(0, 1, 2)[:1])
    assert C._dense(torch.zeros(()))
    for bad in (t[:, ::2], t[:, :, :3], t[:1].expand(4, 6, 5), t.transpose(0, 1)[::2]):
        assert not C._dense(bad)


def test_shared_memory_is_found():
    t = torch.zeros(100)
    C._apart([t[:50], t[50:]], "x")
    for bad in ([t[:51], t[50:]], [t, t], [t[10:20], t]):
        with pytest.raises(ValueError, match="share"):
            C._apart(bad, "x")


def test_cpu_tensors_and_other_types_are_refused():
    with pytest.raises(TypeError):
        C.GradSet([torch.zeros(4)])
    with pytest.raises(TypeError):
        C.GradSet([torch.zeros(4, dtype=torch.float64)])
    with pytest.raises(ValueError, match="outputs"):
        C.GradSet([torch.zeros(4)], out=[])
    for bad in (0.0, -1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            C.clip_grad_norm([], bad)

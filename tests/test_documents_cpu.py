"""Documents packed into rows, clipping and the head's loss by pieces through the model and the trainer, on the oracle backend."""
import math

import pytest
import torch

from autoresearch_b200.config import TrainConfig, model_preset
from autoresearch_b200.models.gpt import GPT
from autoresearch_b200.models.init import init_weights
from autoresearch_b200.ops import reference as R
from autoresearch_b200.ops.backend import get_backend
from autoresearch_b200.ops.packed import document_bounds
from autoresearch_b200.trainer import Trainer


def _trainer(**kw):
    cfg = model_preset("tiny")
    t = TrainConfig(device_batch_size=2, total_batch_size=2 * cfg.seq_len * 2, max_steps=4, cooldown_steps=1, synthetic_data=True,
                    synthetic_kind="zipf", impl="oracle", cooldown_trigger_file="", **kw)
    return Trainer(cfg, t, device="cpu", quiet=True)


def test_bounds_begin_at_rows_and_at_the_token():
    ids = torch.tensor([[5, 1, 2, 7], [7, 7, 3, 4]], dtype=torch.int32)
    kept = ids.clone()
    b = document_bounds(ids, 7)
    assert b.dtype is torch.int32 and b.tolist() == [0, 3, 4, 5, 8] and torch.equal(ids, kept)
    assert document_bounds(ids, 99).tolist() == [0, 4, 8]


@pytest.mark.parametrize("window", [3, 100])
def test_packed_oracle_is_attention_document_by_document(window):
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(20, h, 8, generator=g) for h in (4, 2, 2))
    out = R.packed_attention(q, k, v, [2, 9, 9, 15], window)
    assert bool((out[:2] == 0).all()) and bool((out[15:] == 0).all())
    for a, b in ((2, 9), (9, 15)):
        want = R.attention(q[None, a:b], k[None, a:b].repeat_interleave(2, 2), v[None, a:b].repeat_interleave(2, 2), window)[0]
        assert torch.equal(out[a:b], want)


def test_a_document_in_a_row_scores_as_it_does_alone():
    """Rotations are relative and attention stays inside: a document's losses do not depend on where in a row it stands."""
    cfg = model_preset("tiny")
    m = GPT(cfg, get_backend("oracle", cfg))
    init_weights(m, scheme="normal", std=0.1)
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, cfg.vocab, (1, 60), generator=g, dtype=torch.int32)
    tgt = torch.randint(0, cfg.vocab, (1, 60), generator=g, dtype=torch.int32)
    with torch.no_grad():
        _, whole = m(ids, tgt, cu_seqlens=torch.tensor([0, 23, 60], dtype=torch.int32))
        _, first = m(ids[:, :23], tgt[:, :23])
        _, second = m(ids[:, 23:], tgt[:, 23:])
        _, plain = m(ids, tgt)
    assert torch.allclose(whole[:23], first, atol=1e-5)
    assert torch.allclose(whole[23:], second, atol=1e-4)
    assert not torch.allclose(whole[23:], plain[23:], atol=1e-4)


def test_trainer_keeps_attention_inside_documents():
    tr = _trainer(doc_bos=0)
    seen = []
    forward = tr.model.forward

    def spy(ids, tgt, **kw):
        seen.append((ids.clone(), kw["cu_seqlens"]))
        return forward(ids, tgt, **kw)
    tr.model.forward = spy
    assert math.isfinite(float(tr.train_step())) and len(seen) == 2
    for ids, bounds in seen:
        assert torch.equal(bounds, document_bounds(ids, 0))
    tr.prefetch.close()


def test_trainer_clips_all_gradients_together():
    free, clipped = _trainer(), _trainer(grad_clip=1e-3)
    for tr in (free, clipped):
        tr.opt.step = lambda *a, **k: None
        tr.train_step()
        tr.prefetch.close()
    norm = float(free.layout.flat_grad.double().norm())
    assert norm > 1e-3 and free.grad_norm is None
    assert abs(float(clipped.grad_norm) - norm) < 1e-5 * norm
    assert torch.allclose(clipped.layout.flat_grad, free.layout.flat_grad * (1e-3 / norm), rtol=1e-4, atol=1e-12)


def test_what_a_trainer_cannot_do_is_refused():
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="grad_clip"):
            _trainer(grad_clip=bad)
    from autoresearch_b200.parallel.pipeline_inproc import InProcPipelineTrainer
    cfg = model_preset("tiny")
    for kw in (dict(grad_clip=1.0), dict(doc_bos=0)):
        t = TrainConfig(device_batch_size=2, total_batch_size=2 * cfg.seq_len, max_steps=1, synthetic_data=True, impl="oracle",
                        cooldown_trigger_file="", **kw)
        with pytest.raises(ValueError, match="grad_clip|doc_bos"):
            InProcPipelineTrainer(cfg, t, ["cpu", "cpu"])


def test_environment():
    t = TrainConfig.from_env({"GRAD_CLIP": "1.5", "DOC_BOS": "8191", "VOCAB_PIECES": "1"})
    assert (t.grad_clip, t.doc_bos, t.vocab_pieces) == (1.5, 8191, True)
    t = TrainConfig.from_env({})
    assert (t.grad_clip, t.doc_bos, t.vocab_pieces) == (0.0, None, False)


def test_memory_plan_counts_them():
    from autoresearch_b200.utils import memplan
    cfg = model_preset("phase2", vocab=131072)
    rows = cfg.seq_len * 2
    plain, docs = memplan.plan(cfg, 2, vocab_pieces=True), memplan.plan(cfg, 2, vocab_pieces=True, documents=True)
    more = sum(b for _, b in docs.step) - sum(b for _, b in plain.step)
    assert more == cfg.n_layer * rows * cfg.d_model          # a byte an element
    head = dict(plain.step)["vocabulary piece, row statistics"]
    assert rows * 2 * 512 * 8 < head < 3 << 30
    assert "logits chunk" in dict(memplan.plan(cfg, 2).step)


def test_clip_of_the_oracle():
    g = [torch.tensor([3.0, 4.0]), torch.tensor([[12.0]])]
    assert float(R.clip_grad_norm(g, 6.5)) == 13.0 and torch.allclose(g[0], torch.tensor([1.5, 2.0])) and float(g[1]) == 6.0
    assert float(R.clip_grad_norm(g, 100.0)) == 6.5 and float(g[1]) == 6.0
    g[0][0] = float("nan")
    assert math.isnan(float(R.clip_grad_norm(g, 1.0))) and float(g[1]) == 6.0


class _HeadByPieces(type(get_backend("oracle"))):
    """The oracle with the choice that the kernels' backend has."""
    vocab_pieces = False

    def takes_vocab_pieces(self, vocab):
        return self.vocab_pieces or vocab > 32768


@pytest.fixture
def one_process(tmp_path):
    import torch.distributed as dist
    dist.init_process_group("gloo", init_method=f"file://{tmp_path}/store", rank=0, world_size=1)
    yield
    dist.destroy_process_group()


def _of_kind(kind, cfg, **kw):
    from autoresearch_b200.parallel.pipeline import PipelineTrainer
    from autoresearch_b200.parallel.pipeline_inproc import InProcPipelineTrainer
    from autoresearch_b200.parallel.tp import TPTrainer
    t = TrainConfig(device_batch_size=2, total_batch_size=2 * cfg.seq_len, max_steps=2, cooldown_steps=1, synthetic_data=True, impl="oracle",
                    cooldown_trigger_file="", **kw)
    if kind == "data":
        return Trainer(cfg, t, device="cpu", quiet=True)
    if kind == "tensor":
        return TPTrainer(cfg, t, tp=1, device="cpu", quiet=True)
    if kind == "pipeline":
        return PipelineTrainer(cfg, t, pp=1, device="cpu", quiet=True)
    return InProcPipelineTrainer(cfg, t, ["cpu", "cpu"], quiet=True)


@pytest.mark.parametrize("kind", ["data", "tensor", "pipeline", "in one process"])
def test_every_trainer_passes_vocab_pieces_on(kind, monkeypatch, one_process):
    """To the backend and to the memory plan, also where the vocabulary alone decides."""
    import sys
    for name in ("autoresearch_b200.trainer", "autoresearch_b200.parallel.tp", "autoresearch_b200.parallel.pipeline",
                 "autoresearch_b200.parallel.pipeline_inproc"):
        __import__(name)
        monkeypatch.setattr(sys.modules[name], "get_backend", lambda impl, cfg: _HeadByPieces().configure(cfg))
    for vocab, asked, pieces in ((64, True, True), (64, False, False), (32776, False, True)):
        tr = _of_kind(kind, model_preset("tiny", vocab=vocab), vocab_pieces=asked)
        assert tr.model.backend.vocab_pieces is asked
        if kind != "in one process":             # which plans no memory
            assert ("vocabulary piece, row statistics" in dict(tr.mem_plan.step)) is pieces
            assert ("logits chunk" in dict(tr.mem_plan.step)) is not pieces
        tr.prefetch.close()


@pytest.mark.parametrize("kind", ["data", "tensor", "pipeline", "in one process"])
def test_vocab_pieces_are_refused_where_no_kernel_makes_them(kind, one_process):
    with pytest.raises(ValueError, match="vocab_pieces"):
        _of_kind(kind, model_preset("tiny"), vocab_pieces=True)


def test_the_norm_is_logged_and_written(tmp_path, capsys):
    import json
    for clip, f in ((1e-3, tmp_path / "a"), (0.0, tmp_path / "b")):
        tr = _trainer(grad_clip=clip, metrics_jsonl=str(f), diagnostic_steps=None)
        tr.quiet = False
        norms = []
        step = tr.train_step

        def spy():
            loss = step()
            norms.append(tr.grad_norm)
            return loss
        tr.train_step = spy
        tr.run()
        said = [ln for ln in capsys.readouterr().out.splitlines() if ln.startswith("clip | grad_norm")]
        rows = [json.loads(ln) for ln in f.read_text().splitlines()]
        assert len(rows) == len(norms) >= 4
        if clip:
            assert [r["grad_norm"] for r in rows] == [float(n) for n in norms] and min(r["grad_norm"] for r in rows) > 0
            assert len(said) == len(rows)
        else:
            assert not said and all("grad_norm" not in r for r in rows)


def test_a_norm_that_is_not_finite_is_said(capsys):
    tr = _trainer(grad_clip=1.0)
    tr.quiet = False
    tr._clip_gradients = lambda top: torch.tensor(math.inf)
    tr.run()
    assert "grad_norm inf | not finite" in capsys.readouterr().out

"""Documents packed into rows, the head's loss by pieces and clipping, together: operators in a chain, the model, the trainer.

Tolerances of the model are those of the model's own test against the fp32 oracle (tests/test_model_gpu.py): four layers of bf16
activations.  The chain is held against the same chain in 64 bits with bf16 roundings where the operators hand over bf16: each
hand-over and each operator's inner rounding adds at most 2^-8 of what it passes on, ten of them on the longest way to a gradient."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _models(cfg):
    from autoresearch_b200.models.gpt import GPT
    from autoresearch_b200.models.init import init_weights
    from autoresearch_b200.ops.backend import get_backend
    torch.manual_seed(0)
    ref = GPT(cfg, get_backend("oracle", cfg), dtype=torch.float32, device="cuda")
    mod = GPT(cfg, get_backend("sm100", cfg), dtype=torch.bfloat16, device="cuda")
    init_weights(mod, scheme="normal", std=0.05)
    with torch.no_grad():
        for p1, p2 in zip(ref.parameters(), mod.parameters()):
            p1.copy_(p2.float())
    return ref, mod


def _batch(cfg, B, seed=1):
    g = torch.Generator(device="cuda").manual_seed(seed)
    ids = torch.randint(0, cfg.vocab, (B, cfg.seq_len), generator=g, device="cuda", dtype=torch.int32)
    tgt = torch.randint(0, cfg.vocab, (B, cfg.seq_len), generator=g, device="cuda", dtype=torch.int32)
    ids[torch.rand(ids.shape, generator=g, device="cuda") < 0.01] = 0
    return ids, tgt


def _assert_gradients(ref, mod):
    from autoresearch_b200.ops import kernels as K
    K.check_err_flag()
    bad = []
    for (n, p1), (_, p2) in zip(ref.named_parameters(), mod.named_parameters()):
        if p1.grad is None or p2.grad is None:
            assert p1.grad is None and p2.grad is None, n
            continue
        rel = ((p1.grad - p2.grad.float()).norm() / (p1.grad.norm() + 1e-12)).item()
        if rel > 0.08:
            bad.append((n, rel))
    assert not bad, f"gradient mismatch: {bad}"


@pytest.mark.parametrize("preset", ["small", "small_moe"])
def test_model_with_documents_matches_the_oracle(preset):
    from autoresearch_b200.config import model_preset
    from autoresearch_b200.ops.packed import document_bounds
    cfg = model_preset(preset)
    ref, mod = _models(cfg)
    ids, tgt = _batch(cfg, 2)
    bounds = document_bounds(ids, 0)
    assert bounds.numel() > 6
    scale = 1.0 / ids.numel()
    l1, pt1 = ref(ids, tgt, grad_scale=scale, cu_seqlens=bounds)
    l2, pt2 = mod(ids, tgt, grad_scale=scale, cu_seqlens=bounds)
    _, plain = mod(ids, tgt, grad_scale=scale)
    assert abs(l1.item() - l2.item()) < 2e-2 * abs(l1.item())
    if preset == "small":                # with experts a token on a near tie may be routed differently
        l1.backward()
        l2.backward()
        assert (pt1 - pt2).abs().mean().item() < 5e-2
        _assert_gradients(ref, mod)
    assert float((plain - pt2).abs().max()) > 1e-2


def test_one_document_per_row_is_the_row():
    from autoresearch_b200.config import model_preset
    cfg = model_preset("small")
    _, mod = _models(cfg)
    ids, tgt = _batch(cfg, 3)
    with torch.no_grad():
        _, plain = mod(ids, tgt)
        _, docs = mod(ids, tgt, cu_seqlens=[0, 512, 1024, 1536])
    # the same products, summed in another order, and O rounded as before: one rounding of bf16 per layer and element
    assert float((plain - docs).abs().max()) < 4 * 2.0 ** -8 * float(plain.abs().max())


@pytest.mark.parametrize("vocab", [1024, 1001, 40000])
def test_head_by_pieces_matches_the_oracle(vocab):
    """1024: asked for; 1001 and 40000: vocabularies that the form with whole rows of logits does not take."""
    from autoresearch_b200.config import model_preset
    cfg = model_preset("small", vocab=vocab)
    ref, mod = _models(cfg)
    mod.backend.vocab_pieces = vocab == 1024
    assert mod.backend.takes_vocab_pieces(vocab)
    ids, tgt = _batch(cfg, 2)
    scale = 1.0 / ids.numel()
    l1, pt1 = ref(ids, tgt, grad_scale=scale)
    l2, pt2 = mod(ids, tgt, grad_scale=scale)
    l1.backward()
    l2.backward()
    assert abs(l1.item() - l2.item()) < 2e-2 * abs(l1.item()) and (pt1 - pt2).abs().mean().item() < 5e-2
    _assert_gradients(ref, mod)


def test_trainer_with_all_three():
    from autoresearch_b200.config import TrainConfig, model_preset
    from autoresearch_b200.ops import kernels as K
    from autoresearch_b200.trainer import Trainer
    cfg = model_preset("small")
    t = TrainConfig(device_batch_size=4, total_batch_size=4 * cfg.seq_len * 2, max_steps=6, cooldown_steps=2, synthetic_data=True,
                    synthetic_kind="zipf", impl="sm100", cooldown_trigger_file="", grad_clip=0.05, doc_bos=3, vocab_pieces=True)
    tr = Trainer(cfg, t, device="cuda", quiet=True)
    assert tr.backend.vocab_pieces
    step = tr.opt.step
    seen = []

    def spy(*a, **k):
        seen.append(float(tr.layout.flat_grad.double().norm()))
        return step(*a, **k)
    tr.opt.step = spy
    for _ in range(4):
        assert math.isfinite(float(tr.train_step()))
        norm = float(tr.grad_norm)
        # what the optimizer saw: the gradients scaled by a factor rounded to fp32
        assert abs(seen[-1] - min(norm, 0.05)) <= 2.0 ** -18 * norm
    assert max(seen) > 0
    K.check_err_flag()
    tr.prefetch.close()


def test_the_operators_in_a_chain():
    """Projection -> packed attention -> head's loss -> gradients -> clipping into bf16 buffers, against 64 bits."""
    from autoresearch_b200.ops import kernels as K
    from autoresearch_b200.ops.linear_ce import linear_cross_entropy
    from autoresearch_b200.ops.packed import PackedSequences, packed_qkv_attention
    from autoresearch_b200.ops.sm100 import LinearFn
    from autoresearch_b200.optim.clip import GradSet, clip_grad_norm
    g = torch.Generator(device="cuda").manual_seed(0)
    H, KV, d, V = 4, 2, 64, 1003
    bounds = [0, 130, 131, 500, 700]
    N, D = 700, H * d
    x = torch.randn(N, D, generator=g, device="cuda").bfloat16()
    wqkv = (torch.randn((H + 2 * KV) * d, D, generator=g, device="cuda") / D ** 0.5).bfloat16().requires_grad_(True)
    head = (torch.randn(V, D, generator=g, device="cuda") * (3 / D ** 0.5)).bfloat16().requires_grad_(True)
    tgt = torch.randint(0, V, (N,), generator=g, device="cuda")
    tgt[::7] = -100
    o = packed_qkv_attention(LinearFn.apply(x, wqkv), PackedSequences(bounds, N, H, KV), window=300, head_dim=d)
    losses = linear_cross_entropy(o, head, tgt, softcap=15.0)
    grads = torch.autograd.grad(losses.sum() / N, (wqkv, head))
    out = [torch.zeros_like(t) for t in grads]
    norm = clip_grad_norm(GradSet(grads, out=out), 0.01)
    K.check_err_flag()

    x64, w64, h64 = x.double(), wqkv.detach().double().requires_grad_(True), head.detach().double().requires_grad_(True)
    q, k, v = (x64 @ w64.T).view(N, H + 2 * KV, d).split([H, KV, KV], 1)
    rows = []
    for a, b in zip(bounds[:-1], bounds[1:]):
        i = torch.arange(b - a, device="cuda")
        seen = (i[None] <= i[:, None]) & (i[None] >= i[:, None] - 300)
        s = torch.einsum("ihd,jhd->hij", q[a:b], k[a:b].repeat_interleave(H // KV, 1)) / math.sqrt(d)
        p = torch.softmax(torch.where(seen, s, -math.inf), -1)
        rows.append(torch.einsum("hij,jhd->ihd", p, v[a:b].repeat_interleave(H // KV, 1)))
    z = 15 * torch.tanh(torch.cat(rows).reshape(N, D) @ h64.T / 15)
    ok = tgt >= 0
    l64 = torch.where(ok, torch.logsumexp(z, 1) - z.gather(1, tgt.clamp(min=0)[:, None])[:, 0], 0.0)
    want = torch.autograd.grad(l64.sum() / N, (w64, h64))
    assert float((losses.detach().double() - l64.detach()).abs().max()) < 0.05
    tol = 10 * 2.0 ** -8
    norm64 = math.sqrt(sum(float(t.square().sum()) for t in want))
    assert abs(float(norm) - norm64) <= tol * norm64 and norm64 > 0.01
    for got, clipped, t in zip(grads, out, want):
        assert float((got.double() - t).norm()) <= tol * float(t.norm())
        assert float((clipped.double() - t * (0.01 / norm64)).norm()) <= tol * float(t.norm()) * 0.01 / norm64


def test_a_training_step_on_documents_does_not_wait_for_the_device():
    from autoresearch_b200.config import TrainConfig, model_preset
    from autoresearch_b200.trainer import Trainer
    cfg = model_preset("small")
    t = TrainConfig(device_batch_size=4, total_batch_size=4 * cfg.seq_len * 2, max_steps=6, cooldown_steps=2, synthetic_data=True,
                    synthetic_kind="zipf", impl="sm100", cooldown_trigger_file="", grad_clip=0.05, doc_bos=3)
    tr = Trainer(cfg, t, device="cuda", quiet=True)
    for _ in range(2):
        tr.train_step()
    torch.cuda.synchronize()
    assert tr.prefetch.wait_for(2)
    torch.cuda._sleep(1_000_000_000)                        # about 0.5 s
    loss = tr.train_step()
    assert not torch.cuda.current_stream().query(), "the step waited for the stream"
    assert math.isfinite(float(loss))
    tr.prefetch.close()

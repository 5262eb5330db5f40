"""Scaled embedding, windowed attention and joined norms together, as a model of this framework runs them on the GPU: bf16 kernels
against the same weights in 64 bits, under activation checkpointing and in a recorded micro-step."""
import copy

import pytest
import torch

from maltos_b200.ops import _lib

pytestmark = pytest.mark.gpu
OPTIONS = dict(sliding_window=70, sink_tokens=3, full_attention_every=2, embedding_scale=16.0, residual_scale=0.5, residual_gate=True)


def _model(kind, checkpointing=False):
    import maltos_b200  # noqa: F401
    from maltos_b200 import models as M

    torch.manual_seed(0)
    sizes = dict(vocab_size=2048, hidden_size=256, intermediate_size=704, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2,
                 max_position_embeddings=256, rms_norm_eps=1e-5, activation_checkpointing=M.ActivationCheckpointConfig(enabled=checkpointing))
    if kind == "llama":
        model = M.LlamaForCausalLM(M.LlamaConfig(**sizes, **OPTIONS, post_block_norm=True))
    else:
        model = M.OlmoForCausalLM(M.OlmoConfig(**sizes, **OPTIONS))
    return model.cuda().bfloat16()


def _batch(packed):
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, 2048, (2, 250), generator=g).cuda()
    batch = {"input_ids": ids, "labels": ids.roll(-1, 1)}
    if packed:
        seq, pos = torch.full((2, 250), -1), torch.zeros(2, 250, dtype=torch.long)
        for b in range(2):
            at = 0
            for n, length in enumerate([90 + b, 3, 120]):
                seq[b, at:at + length], pos[b, at:at + length] = n, torch.arange(length)
                at += length
        batch |= {"sequence_ids": seq.cuda(), "position_ids": pos.cuda()}
        batch["labels"] = torch.where(batch["sequence_ids"] == -1, -100, batch["labels"])
    return batch


@pytest.mark.parametrize("kind", ["llama", "olmo"])
@pytest.mark.parametrize("packed", [False, True])
def test_model_against_64_bits(kind, packed):
    model, batch = _model(kind), _batch(packed)
    plain = copy.deepcopy(model).cpu().double()
    for m in plain.modules():                    # the angle tables stay fp32 by design
        if hasattr(m, "cos"):
            m.cos, m.sin = m.cos.double(), m.sin.double()
    before = _lib.launch_count()
    loss = model(batch)
    loss.backward()
    _lib.fetch_status()
    assert _lib.launch_count() - before > 40
    want = plain({k: v.cpu() for k, v in batch.items()})
    want.backward()
    # a mean over some 400 targets of values near 8 whose logits carry a few bf16 roundings (2^-8) each
    assert abs(float(loss) - float(want)) < 2e-2
    for (name, p), (_, q) in zip(model.named_parameters(), plain.named_parameters()):
        # bf16 activations and gradients through two layers: a dozen roundings of 2^-8 in a row, as independent errors 1.4 %
        rel = float((p.grad.double().cpu() - q.grad).norm() / q.grad.norm())
        assert rel < 0.05, (name, rel)


@pytest.mark.parametrize("kind", ["llama", "olmo"])
def test_activation_checkpointing_gives_the_same_bits(kind):
    batch, grads = _batch(True), []
    for checkpointing in (False, True):
        model = _model(kind, checkpointing)
        model(batch).backward()
        grads.append([p.grad for p in model.parameters()])
    assert all(torch.equal(a, b) for a, b in zip(*grads))


def test_recorded_micro_step():
    from maltos_b200.utils.cuda_graph import GraphedMicroStep

    model, batch = _model("llama"), _batch(False)
    params = list(model.parameters())
    loss = model(batch)
    loss.backward()
    eager, want = [p.grad.clone() for p in params], float(loss)
    del loss                                     # no eager graph of the parameters lives during the capture
    for p in params:
        p.grad = None
    step = GraphedMicroStep(lambda b: model(b), params, batch)
    got = float(step(batch))
    torch.cuda.synchronize()
    assert got == want
    for p, e in zip(params, eager):
        assert torch.equal(p.grad, e)
    _lib.fetch_status()

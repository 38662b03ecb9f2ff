"""The token model on the GPU: every logit against the same step in 64 bits, over
the weights and the stored keys and values that the model itself holds.

Each operator's output is rounded to float16 (2^-11); a layer's chain of ten such
roundings, with norms that rescale, is held to 2^-6 of a row's logits, in the
2-norm: a step that is wrong anywhere (a position, a head, a page, a mask) is off
by the order of the logits themselves."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


def dense(matrix):
    """The matrix a PackedMatrix stands for, in 64 bits: its products with the unit vectors."""
    import torch

    return matrix.multiply(torch.eye(matrix.inputs, device="cuda").half()).double().t()


def normed(x, weight):
    import torch

    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.double()


def turned(x, places, cosines, sines):
    import torch

    c, s = cosines.double()[places][:, None], sines.double()[places][:, None]
    a, b = x.chunk(2, -1)
    return torch.cat((a * c - b * s, b * c + a * s), -1)


def plain_logits(model, symbols, first):
    """Logits of `symbols` [batch, count] at places first.., over the caches as they stand now."""
    import torch

    config = model.config
    batch, count = symbols.shape
    places = torch.arange(first, first + count, device="cuda")
    hidden, out = model.embedding[symbols].double(), None
    for layer, cache in zip(model.layers, model.caches):
        x = normed(hidden, layer.before[0])
        q = (x @ dense(layer.qkv).t())[..., : config.heads * config.head_dim]
        q = q.view(batch, count, config.heads, config.head_dim)
        mixed = []
        for b in range(batch):
            here = torch.arange(first + count, device="cuda")
            slots = model.table[b].long()[here // model.page_size] * model.page_size + here % model.page_size
            keys, values = (t.double().repeat_interleave(config.heads // config.kv_heads, 1)
                            for t in cache.read(slots, torch.float32))
            scores = torch.einsum("ihd,thd->hit", turned(q[b], places, model.cosines, model.sines), keys)
            scores = scores * config.head_dim ** -0.5
            scores = scores.masked_fill(here[None, :] > places[:, None], float("-inf"))
            mixed.append(torch.einsum("hit,thd->ihd", scores.softmax(-1), values).flatten(1))
        delta = torch.stack(mixed) @ dense(layer.out).t()
        hidden = hidden + layer.gates[0].double() * normed(delta, layer.after[0])
        gate, up = (normed(hidden, layer.before[1]) @ dense(layer.gate_up).t()).chunk(2, -1)
        delta = (torch.nn.functional.silu(gate) * up) @ dense(layer.down).t()
        hidden = hidden + layer.gates[1].double() * normed(delta, layer.after[1])
    return normed(hidden, model.last_norm) @ dense(model.head).t()


def test_prompt_and_steps_follow_the_formulas(cuda):
    import torch

    from nvcr_b200.token_model import TokenModel, TokenModelConfig

    config = TokenModelConfig(layers=2, width=256, heads=8, kv_heads=2, head_dim=64, inner=384, symbols=101, group=32)
    model = TokenModel(config, batch=3, max_length=80)
    make = torch.Generator(device="cuda").manual_seed(2)
    at = 0
    for count in (37, 1, 1, 5, 1):
        symbols = torch.randint(0, config.symbols, (3, count), generator=make, device="cuda")
        logits = model.advance(symbols).double()
        want = plain_logits(model, symbols, at)
        at += count
        off = (logits - want).norm(dim=-1) / want.norm(dim=-1)
        assert float(off.max()) < 2.0 ** -6, (count, float(off.max()))
    model.check()
    assert model.lengths.tolist() == [at] * 3


def test_captured_steps_equal_eager_ones(cuda):
    import torch

    from nvcr_b200.token_model import TokenModel, TokenModelConfig

    config = TokenModelConfig(layers=1, width=256, heads=4, kv_heads=4, head_dim=64, inner=256, symbols=64)
    models = [TokenModel(config, batch=2, max_length=64, seed=5) for _ in range(2)]
    make = torch.Generator(device="cuda").manual_seed(3)
    prompt = torch.randint(0, config.symbols, (2, 9), generator=make, device="cuda")
    steps = [torch.randint(0, config.symbols, (2, 1), generator=make, device="cuda") for _ in range(4)]
    for model in models:
        model.advance(prompt)
        model.advance(steps[0])
    eager = [models[0].advance(s) for s in steps[1:]]
    entry, graph = steps[1].clone(), torch.cuda.CUDAGraph()
    before = models[1].lengths.clone()
    with torch.cuda.graph(graph):
        out = models[1].advance(entry)
    models[1].lengths.copy_(before)
    for s, want in zip(steps[1:], eager):
        entry.copy_(s)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    for model in models:
        model.check()


def test_the_command_runs(cuda, capsys, monkeypatch):
    import sys

    from nvcr_b200 import token_model

    monkeypatch.setattr(sys, "argv", ["token_model", "--batch", "2", "--prompt", "5", "--steps", "3", "--layers", "1"])
    token_model.main()
    assert "us a step" in capsys.readouterr().out


def test_steps_past_the_longest_sequence_are_told(cuda):
    """Symbols past max_length are left out and told, by a prompt and step by step; nothing stored changes."""
    import torch

    from nvcr_b200.executor import ExecutorError
    from nvcr_b200.token_model import TokenModel, TokenModelConfig

    config = TokenModelConfig(layers=1, width=128, heads=2, kv_heads=1, head_dim=64, inner=128, symbols=32)
    for counts in ((20, 12, 1, 1, 30), (20, 5, 9, 1)):
        model = TokenModel(config, batch=2, max_length=32)
        make = torch.Generator(device="cuda").manual_seed(1)
        prompt = torch.randint(0, config.symbols, (2, counts[0]), generator=make, device="cuda")
        model.advance(prompt)
        at = counts[0]
        for count in counts[1:]:
            before = [t.clone() for t in model.caches[0].tensors]
            logits = model.advance(prompt[:, :1].expand(2, count).contiguous())
            at += count
            assert logits.shape == (2, count, config.symbols) and torch.isfinite(logits).all()
            if at <= 32:
                model.check()
                continue
            with pytest.raises(ExecutorError, match="slot, length or offset"):
                model.check()
            if at - count >= 32:
                for t, old in zip(model.caches[0].tensors, before):
                    assert torch.equal(t, old)

"""The token model with 8-bit weights, experts and sampling on the GPU: its logits against the same step in 64 bits, and
a step's symbols against its logits.

A row that a product takes in 8 bits is off by up to half a step of a 127th of its largest value, evenly: in the 2-norm by
largest / (127 sqrt(12)) a value, 1.0% of a row whose largest value is 4.4 standard deviations (an activation's here,
which is a norm's output or the product of two such). A layer has four such products in a row, one of them with a factor
(gate times up) that doubles it; two layers and the head add up to 11%, and to 2^-3 with the float16 roundings. A step that
is wrong anywhere (an expert, a weight, a row) is off by the order of the logits themselves."""
from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu


def dense(matrix, expert=None):
    """The matrix in 64 bits: its products with the unit vectors."""
    import torch

    eye = torch.eye(matrix.inputs, device="cuda")
    if expert is None:
        return matrix.multiply(eye.half()).double().t()
    choices = torch.full((matrix.inputs, 1), expert, dtype=torch.int32, device="cuda")
    return matrix.multiply(eye, choices)[:, 0].double().t()


def normed(x, weight):
    import torch

    return x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * weight.double()


def plain_logits(model, symbols, first, routes):
    """Logits of `symbols` [batch, count] at places first.., over the caches as they stand now; `routes`: each layer's
    choices and weights, as the model had them."""
    import torch

    config = model.config
    batch, count = symbols.shape
    places = torch.arange(first, first + count, device="cuda")
    c, s = model.cosines.double()[places][:, None], model.sines.double()[places][:, None]
    hidden = model.embedding[symbols].double()
    for nth, (layer, cache) in enumerate(zip(model.layers, model.caches)):
        q = (normed(hidden, layer.before[0]) @ dense(layer.qkv).t())[..., : config.heads * config.head_dim]
        a, b = q.view(batch, count, config.heads, config.head_dim).chunk(2, -1)
        q = torch.cat((a * c - b * s, b * c + a * s), -1)
        mixed = []
        for i in range(batch):
            here = torch.arange(first + count, device="cuda")
            slots = model.table[i].long()[here // model.page_size] * model.page_size + here % model.page_size
            keys, values = (t.double().repeat_interleave(config.heads // config.kv_heads, 1)
                            for t in cache.read(slots, torch.float32))
            scores = torch.einsum("ihd,thd->hit", q[i], keys) * config.head_dim ** -0.5
            scores = scores.masked_fill(here[None, :] > places[:, None], float("-inf"))
            mixed.append(torch.einsum("hit,thd->ihd", scores.softmax(-1), values).flatten(1))
        delta = torch.stack(mixed) @ dense(layer.out).t()
        hidden = hidden + layer.gates[0].double() * normed(delta, layer.after[0])
        x = normed(hidden, layer.before[1])
        if config.experts:
            x = x.flatten(0, 1)
            choices, weights = routes[nth]
            # the model's experts are the best by these scores too, but for what 8 bits and float16 may hide
            scores = x @ dense(layer.scores).t()
            worst = scores.gather(1, choices.long()).amin(1)
            best_left = scores.scatter(1, choices.long(), float("-inf")).amax(1)
            assert float((best_left - worst).max()) < 2 * 2.0 ** -3 * float(scores.std())
            share = torch.zeros((len(x), config.experts), dtype=torch.float64, device="cuda")
            share.scatter_(1, choices.long(), weights.double())
            out = torch.zeros_like(x)
            for e in range(config.experts):
                gate, up = (x @ dense(layer.gate_up, e).t()).chunk(2, -1)
                out += share[:, e:e + 1] * ((torch.nn.functional.silu(gate) * up) @ dense(layer.down, e).t())
            delta = out.view_as(hidden)
        else:
            gate, up = (x @ dense(layer.gate_up).t()).chunk(2, -1)
            delta = (torch.nn.functional.silu(gate) * up) @ dense(layer.down).t()
        hidden = hidden + layer.gates[1].double() * normed(delta, layer.after[1])
    return normed(hidden, model.last_norm) @ dense(model.head).t()


@pytest.mark.parametrize("bits,experts,chosen", [(8, 0, 1), (4, 6, 2), (8, 6, 2), (8, 3, 1)])
def test_prompt_and_steps_follow_the_formulas(cuda, monkeypatch, bits, experts, chosen):
    import torch

    from nvcr_b200 import tokens
    from nvcr_b200.token_model import TokenModel, TokenModelConfig

    config = TokenModelConfig(layers=2, width=256, heads=8, kv_heads=2, head_dim=64, inner=384, symbols=101, group=32, bits=bits,
                              experts=experts, chosen=chosen)
    model = TokenModel(config, batch=3, max_length=80)
    routes, route = [], tokens.route

    def recorded(*args, **options):
        routes.append(route(*args, **options))
        return routes[-1]

    monkeypatch.setattr(tokens, "route", recorded)
    make = torch.Generator(device="cuda").manual_seed(2)
    at = 0
    for count in (37, 1, 5):
        symbols = torch.randint(0, config.symbols, (3, count), generator=make, device="cuda")
        routes.clear()
        logits = model.advance(symbols).double()
        want = plain_logits(model, symbols, at, routes)
        at += count
        off = (logits - want).norm(dim=-1) / want.norm(dim=-1)
        assert float(off.max()) < 2.0 ** -3, (count, float(off.max()))
    model.check()
    assert len(routes) == (config.layers if experts else 0)


def test_captured_steps_choose_as_eager_ones(cuda):
    """A routed model's sampled steps, captured once: the same symbols as eager ones, step by step."""
    import torch

    from nvcr_b200.token_model import TokenModel, TokenModelConfig

    config = TokenModelConfig(layers=2, width=256, heads=4, kv_heads=4, head_dim=64, inner=256, symbols=300, bits=8, experts=4)
    settings = {"temperature": 0.8, "top_k": 40, "top_p": 0.9}
    models = [TokenModel(config, batch=3, max_length=64, seed=5) for _ in range(2)]
    make = torch.Generator(device="cuda").manual_seed(3)
    prompt = torch.randint(0, config.symbols, (3, 9), generator=make, device="cuda")
    numbers = torch.rand((6, 3), generator=make, device="cuda")
    first = [model.step(prompt, numbers[0], **settings) for model in models]
    assert torch.equal(first[0], first[1]) and first[0].shape == (3, 1)
    eager = [first[0]]
    for number in numbers[1:]:
        eager.append(models[0].step(eager[-1], number, **settings))
    entry, uniforms, graph = first[1].clone(), numbers[1].clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        entry.copy_(models[1].step(entry, uniforms, **settings))
    models[1].lengths.fill_(9)
    entry.copy_(first[1])
    for number, want in zip(numbers[1:], eager[1:]):
        uniforms.copy_(number)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(entry, want)
    for model in models:
        model.check()


def test_steps_are_what_the_logits_say(cuda):
    """At temperature 0 the largest logit's symbol; at others one of the few that top_k keeps."""
    import torch

    from nvcr_b200.token_model import TokenModel, TokenModelConfig

    config = TokenModelConfig(layers=1, width=128, heads=2, kv_heads=1, head_dim=64, inner=128, symbols=64, experts=2, chosen=1)
    models = [TokenModel(config, batch=4, max_length=32, seed=1) for _ in range(3)]
    make = torch.Generator(device="cuda").manual_seed(1)
    prompt = torch.randint(0, config.symbols, (4, 7), generator=make, device="cuda")
    uniforms = torch.rand((4,), generator=make, device="cuda")
    logits = models[0].advance(prompt)[:, -1]
    assert torch.equal(models[1].step(prompt, uniforms, temperature=0.0)[:, 0], logits.argmax(-1))
    chosen = models[2].step(prompt, uniforms, temperature=2.0, top_k=3)
    assert (logits.topk(3, -1).indices == chosen).any(-1).all()


@pytest.mark.parametrize("options", [["--bits", "8"], ["--experts", "4", "--temperature", "0.8", "--top-p", "0.9"]])
def test_the_command_runs(cuda, capsys, monkeypatch, options):
    import sys

    from nvcr_b200 import token_model

    monkeypatch.setattr(sys, "argv", ["token_model", "--batch", "2", "--prompt", "5", "--steps", "3", "--layers", "1"] + options)
    token_model.main()
    assert "us a step" in capsys.readouterr().out

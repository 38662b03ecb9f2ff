"""A small token model over the token operators: what a step of a language model
looks like with 4-bit weights and a 4-bit cache, together as they are used. A
prompt and its single steps agree to rounding, not to the bit.

A layer is two blocks, each with a norm before and after it and a gate on the way
back to the residual stream::

    hidden, normed = block_norm(delta, residual=hidden, ...)   # after the last block, before this one
    q, k, v        = qkv.multiply(normed)
    q              = cache.append(k, v, slots, queries=q, ...)  # rotated, stored in 4 bits
    delta          = out.multiply(context.attend(q, cache, ...))
    hidden, normed = block_norm(delta, residual=hidden, ...)
    delta          = down.multiply(silu(gate) * up)             # gate, up = gate_up.multiply(normed)

With ``experts`` the second block is each token's own few of many, in 8 bits::

    choices, weights = route(scores.multiply(normed), chosen, renormalise=True)
    gate, up       = gate_up.multiply(normed, choices)          # [tokens, chosen, inner] each
    delta          = down.multiply(silu(gate) * up, choices, weights)

``bits=8`` holds all weights in 8 bits, for long prompts: their products run on the
tensor cores at their 8-bit rate, where those with 4-bit weights are made for a few rows.

``python -m nvcr_b200.token_model`` decodes a batch of sequences with random
weights and prints the time of a step, eager and as a captured CUDA graph;
``--experts 8``, ``--bits 8`` and ``--temperature 0.8 --top-p 0.9`` try the rest.
"""
from __future__ import annotations

import argparse
import time
from dataclasses import dataclass

import torch

from . import tokens


@dataclass(frozen=True)
class TokenModelConfig:
    layers: int = 2
    width: int = 512
    heads: int = 8
    kv_heads: int = 2
    head_dim: int = 64
    inner: int = 1024
    symbols: int = 257
    group: int = 64
    positions: int = 4096
    dtype: torch.dtype = torch.float16
    bits: int = 4  # of weights: 4 or 8
    experts: int = 0  # of the second block; 0: one block for all tokens
    chosen: int = 2  # experts of a token


def _matrix(config: TokenModelConfig, make: torch.Generator, outputs: int,
            inputs: int) -> tokens.PackedMatrix | tokens.ByteMatrix:
    weights = torch.randn((outputs, inputs), generator=make, device="cuda") * inputs ** -0.5
    return tokens.ByteMatrix.quantise(weights) if config.bits == 8 else tokens.PackedMatrix.quantise(weights, config.group)


class _Layer:
    def __init__(self, config: TokenModelConfig, make: torch.Generator) -> None:
        def matrix(outputs: int, inputs: int) -> tokens.PackedMatrix | tokens.ByteMatrix:
            return _matrix(config, make, outputs, inputs)

        def experts(outputs: int, inputs: int) -> tokens.ByteExperts:
            shape = (config.experts, outputs, inputs)
            return tokens.ByteExperts.quantise(torch.randn(shape, generator=make, device="cuda") * inputs ** -0.5)

        def vector(mean: float) -> torch.Tensor:
            return (torch.randn((config.width,), generator=make, device="cuda") * 0.1 + mean).to(config.dtype)

        heads = config.heads + 2 * config.kv_heads
        self.qkv = matrix(heads * config.head_dim, config.width)
        self.out = matrix(config.width, config.heads * config.head_dim)
        if config.experts:
            weights = torch.randn((config.experts, config.width), generator=make, device="cuda") * config.width ** -0.5
            self.scores = tokens.ByteMatrix.quantise(weights)
            self.gate_up = experts(2 * config.inner, config.width)
            self.down = experts(config.width, config.inner)
        else:
            self.gate_up = matrix(2 * config.inner, config.width)
            self.down = matrix(config.width, config.inner)
        self.before = [vector(1.0), vector(1.0)]  # weights of the norms before and after each block, and its gate
        self.after = [vector(1.0), vector(1.0)]
        self.gates = [vector(0.5), vector(0.5)]


class TokenModel:
    """Random weights from a seed, a paged cache a layer, and pages handed out as sequences grow."""

    def __init__(self, config: TokenModelConfig, batch: int, max_length: int, page_size: int = 16, seed: int = 0) -> None:
        make = torch.Generator(device="cuda").manual_seed(seed)
        self.config, self.batch, self.page_size = config, batch, page_size
        self.columns = -(-max_length // page_size)
        self.max_length = self.columns * page_size
        self.embedding = torch.randn((config.symbols, config.width), generator=make, device="cuda").to(config.dtype)
        self.layers = [_Layer(config, make) for _ in range(config.layers)]
        self.head = _matrix(config, make, config.symbols, config.width)
        self.last_norm = torch.ones((config.width,), dtype=config.dtype, device="cuda")
        self.caches = [tokens.PagedCache.empty(batch * self.columns, config.kv_heads, page_size, config.head_dim,
                                               min(config.group, config.head_dim)) for _ in range(config.layers)]
        self.context = tokens.TokenContext()
        half = torch.arange(0, config.head_dim, 2, device="cuda", dtype=torch.float64) / config.head_dim
        angles = torch.outer(torch.arange(config.positions, device="cuda", dtype=torch.float64), 10000.0 ** -half)
        self.cosines, self.sines = angles.cos().float(), angles.sin().float()
        # every sequence may use any page: they are handed out in an order that is nobody's own
        order = torch.randperm(batch * self.columns, generator=make, device="cuda")
        # the last column's page is none of a cache's: of the places past a sequence's end
        self.pages = torch.full((batch, self.columns + 1), batch * self.columns, dtype=torch.int32, device="cuda")
        self.pages[:, :-1] = order.view(batch, self.columns)
        self.table = self.pages[:, :-1]
        self.lengths = torch.zeros((batch,), dtype=torch.int32, device="cuda")

    def advance(self, symbols: torch.Tensor) -> torch.Tensor:
        """Appends int64 symbols [batch, count] to the sequences and returns the logits [batch, count, symbols] of what
        follows each. Nothing waits for the host, so that a step can be captured in a CUDA graph; symbols past
        max_length are not stored, their sequence attends to nothing from then on, and `check` tells."""
        config = self.config
        batch, count = symbols.shape
        nth = torch.arange(count, device="cuda", dtype=torch.int32)
        places = (self.lengths[:, None] + nth).flatten()
        self.lengths += count
        slots = self._slots(self.pages, places.view(batch, count), self.page_size)
        offsets = torch.arange(0, batch * count + 1, count, device="cuda", dtype=torch.int32)
        hidden, delta = self.embedding[symbols.flatten()], None
        heads = config.heads, config.kv_heads, config.kv_heads
        after = gate = None
        for layer, cache in zip(self.layers, self.caches):
            hidden, normed = self._between(hidden, delta, after, gate, layer.before[0])
            rows = layer.qkv.multiply(normed).view(batch * count, -1, config.head_dim)
            q, k, v = rows.split(heads, 1)
            q = cache.append(k, v, slots, queries=q, positions=places, cosines=self.cosines, sines=self.sines)
            mixed = self.context.attend(q, cache, self.table, self.lengths, query_offsets=offsets, max_queries=count,
                                        max_length=self.max_length)
            delta = layer.out.multiply(mixed.view(batch * count, -1))
            hidden, normed = self._between(hidden, delta, layer.after[0], layer.gates[0], layer.before[1])
            if config.experts:
                choices, weights = tokens.route(layer.scores.multiply(normed), config.chosen, renormalise=True)
                inner_gate, up = layer.gate_up.multiply(normed, choices).chunk(2, 2)
                delta = layer.down.multiply(torch.nn.functional.silu(inner_gate) * up, choices, weights)
            else:
                inner_gate, up = layer.gate_up.multiply(normed).chunk(2, 1)
                delta = layer.down.multiply(torch.nn.functional.silu(inner_gate) * up)
            after, gate = layer.after[1], layer.gates[1]
        _, normed = self._between(hidden, delta, after, gate, self.last_norm)
        return self.head.multiply(normed).view(batch, count, -1)

    def step(self, symbols: torch.Tensor, uniforms: torch.Tensor, **settings) -> torch.Tensor:
        """Appends int64 symbols [batch, count] and returns the one [batch, 1] that follows each sequence, chosen by its
        uniform number (float32 [batch]) and `tokens.sample`'s settings."""
        chosen, _ = tokens.sample(self.advance(symbols)[:, -1], uniforms, **settings)
        return chosen[:, None]

    @staticmethod
    def _slots(pages: torch.Tensor, places: torch.Tensor, page_size: int) -> torch.Tensor:
        """The slots of places [batch, count]; past the table's end all are the first one past the cache's."""
        places = places.clamp(max=(pages.shape[1] - 1) * page_size)
        return (pages.gather(1, (places // page_size).long()).long() * page_size + places % page_size).flatten()

    @staticmethod
    def _between(hidden, delta, after, gate, before):
        """The residual stream after a block (none yet: the embedding itself) and the next block's input."""
        if delta is None:
            return tokens.block_norm(hidden, pre_weight=before)
        return tokens.block_norm(delta, residual=hidden, gate=gate, post=True, post_weight=after, pre_weight=before)

    def check(self) -> None:
        """Raises if a kernel met a slot, position, page or length out of range, or a wait in one ran out."""
        for cache in self.caches:
            cache.check()
        parts = [self.head] + [part for layer in self.layers for part in vars(layer).values()]
        for part in parts:
            if isinstance(part, (tokens.ByteMatrix, tokens.ByteExperts)):
                part.check()


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    parser.add_argument("--batch", type=int, default=4)
    parser.add_argument("--prompt", type=int, default=32)
    parser.add_argument("--steps", type=int, default=64)
    parser.add_argument("--layers", type=int, default=4)
    parser.add_argument("--bits", type=int, choices=(4, 8), default=4, help="of the weights")
    parser.add_argument("--experts", type=int, default=0, help="of a layer's second block (0: one block for all)")
    parser.add_argument("--temperature", type=float, default=0.0, help="0: the symbol with the largest logit")
    parser.add_argument("--top-p", type=float, default=1.0)
    options = parser.parse_args()
    config = TokenModelConfig(layers=options.layers, bits=options.bits, experts=options.experts,
                              chosen=min(2, max(1, options.experts)))
    model = TokenModel(config, options.batch, options.prompt + 2 * options.steps + 8)
    make = torch.Generator(device="cuda").manual_seed(1)
    prompt = torch.randint(0, config.symbols, (options.batch, options.prompt), generator=make, device="cuda")
    symbols = model.advance(prompt)[:, -1:].argmax(-1)
    uniforms = torch.zeros((options.batch,), device="cuda")

    def step(x: torch.Tensor) -> torch.Tensor:
        if options.temperature <= 0:
            return model.advance(x).argmax(-1)
        return model.step(x, uniforms, temperature=options.temperature, top_p=options.top_p)

    for _ in range(4):
        symbols = step(symbols)
    torch.cuda.synchronize()
    began = time.perf_counter()
    for _ in range(options.steps):
        uniforms.uniform_(generator=make)
        symbols = step(symbols)
    torch.cuda.synchronize()
    eager = (time.perf_counter() - began) / options.steps

    graph, entry = torch.cuda.CUDAGraph(), symbols.clone()
    with torch.cuda.graph(graph):
        entry.copy_(step(entry))
    torch.cuda.synchronize()
    began = time.perf_counter()
    for _ in range(options.steps):
        uniforms.uniform_(generator=make)
        graph.replay()
    torch.cuda.synchronize()
    captured = (time.perf_counter() - began) / options.steps
    model.check()
    print(f"{options.layers} layers of {config.width}, {options.batch} sequences of {options.prompt} symbols: "
          f"{eager * 1e6:.1f} us a step, {captured * 1e6:.1f} us as a captured graph")


if __name__ == "__main__":
    main()

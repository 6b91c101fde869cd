"""A decoder over a paged KV cache, from the library's ops: the norms and SiLU-and-mul of the reference's
path, and between them rotary positions, the cache, attention over its pages and the pages' bookkeeping.

Random weights of a decoder architecture (default: small; ``--seven-b`` takes the served 7B
architecture's layer: hidden 3584, 28 query and 4 key heads of 128, intermediate 18944). It prefills a
prompt in chunks, forks it into several continuations, decodes them, releases half and compacts the
pages. The projections are plain torch matrix products.

    python inference-performance-lab_b200/examples/paged_decoder.py [--seven-b] [--layers N]
"""

from __future__ import annotations

import argparse
import sys
import time
from dataclasses import dataclass
from pathlib import Path

import torch

PACKAGE_DIR = Path(__file__).resolve().parents[1]
if str(PACKAGE_DIR) not in sys.path:
    sys.path.insert(0, str(PACKAGE_DIR))

from inference_performance_lab.kernels import extension as ops  # noqa: E402
from inference_performance_lab.kernels.rotary import rotary_cos_sin_cache  # noqa: E402


@dataclass
class Config:
    vocabulary: int = 512
    hidden: int = 256
    heads: int = 8
    kv_heads: int = 2
    head_size: int = 64
    intermediate: int = 640
    layers: int = 2
    max_position: int = 4096
    epsilon: float = 1e-6


class PagedDecoder:
    """``rows`` sequences over ``pages`` pages of ``page_size`` tokens; a row's state lies on the device."""

    def __init__(self, config: Config, rows: int = 16, pages: int = 256, page_size: int = 16, seed: int = 0) -> None:
        self.config, self.page_size = config, page_size
        generator = torch.Generator(device="cuda").manual_seed(seed)

        def weights(*shape: int) -> torch.Tensor:
            w = torch.randn(*shape, generator=generator, device="cuda") * shape[0] ** -0.5
            return w.to(torch.bfloat16)

        c = config
        self.embedding = weights(c.vocabulary, c.hidden) * c.vocabulary**0.5
        self.layers = [
            {
                "qkv": weights(c.hidden, (c.heads + 2 * c.kv_heads) * c.head_size),
                "out": weights(c.heads * c.head_size, c.hidden),
                "gate_up": weights(c.hidden, 2 * c.intermediate),
                "down": weights(c.intermediate, c.hidden),
                "norms": torch.rand(2, c.hidden, generator=generator, device="cuda").add_(0.5).to(torch.bfloat16),
            }
            for _ in range(c.layers)
        ]
        self.norm = torch.ones(c.hidden, device="cuda", dtype=torch.bfloat16)
        self.head = weights(c.hidden, c.vocabulary)
        self.table = rotary_cos_sin_cache(c.head_size, c.max_position)
        self.store = torch.zeros(
            c.layers, 2, pages, page_size, c.kv_heads, c.head_size, device="cuda", dtype=torch.bfloat16
        )
        self.caches = list(self.store.flatten(0, 1).unbind(0))
        width = -(-c.max_position // page_size)
        self.tables = torch.full((rows, width), -1, device="cuda", dtype=torch.int32)
        self.lens = torch.zeros(rows, device="cuda", dtype=torch.int32)
        self.refs = torch.zeros(pages, device="cuda", dtype=torch.int32)
        self.host_lens = [0] * rows  # the scheduler's own copy

    @staticmethod
    def _ints(values, dtype=torch.int32) -> torch.Tensor:
        return torch.tensor(values, device="cuda", dtype=dtype)

    def _succeed(self, status: torch.Tensor) -> None:
        status = int(status)
        if status != 0:
            raise RuntimeError("out of pages" if status > 0 else "invalid rows")

    def forward(self, rows: list[int], tokens: list[list[int]]) -> torch.Tensor:
        """Appends ``tokens[i]`` to ``rows[i]`` and returns the logits after each row's last token."""
        c = self.config
        new = [len(t) for t in tokens]
        total = [self.host_lens[r] + n for r, n in zip(rows, new)]
        index = self._ints(rows)
        lens = self._ints(total)
        self._succeed(ops.reserve_pages(self.tables, self.lens, self.refs, index, lens, self.page_size))
        for row, length in zip(rows, total):
            self.host_lens[row] = length
        tables = self.tables[index.long()]
        starts = [sum(new[:i]) for i in range(len(new) + 1)]
        positions = self._ints([p for n, t in zip(new, total) for p in range(t - n, t)], torch.int64)
        sequence = self._ints([s for s, n in enumerate(new) for _ in range(n)], torch.int64)
        slots = tables[sequence, positions // self.page_size].long() * self.page_size + positions % self.page_size
        query_start_loc = self._ints(starts)

        residual = self.embedding[self._ints([t for row in tokens for t in row], torch.int64)]
        x = ops.rms_norm(residual, self.layers[0]["norms"][0], c.epsilon)
        for number, layer in enumerate(self.layers):
            keys, values = self.store[number]
            qkv = (x @ layer["qkv"]).view(-1, c.heads + 2 * c.kv_heads, c.head_size)
            q, k, v = qkv.split([c.heads, c.kv_heads, c.kv_heads], dim=1)
            ops.rotary_embedding_cache(positions, q, k, v, self.table, keys, values, slots)
            x = ops.paged_attention(q, keys, values, tables, query_start_loc, lens, max(new), max(total), c.head_size**-0.5)
            x = x.flatten(1) @ layer["out"]
            ops.fused_add_rms_norm(x, residual, layer["norms"][1], c.epsilon)
            x = ops.silu_and_mul(x @ layer["gate_up"]) @ layer["down"]
            following = self.layers[number + 1]["norms"][0] if number + 1 < c.layers else self.norm
            ops.fused_add_rms_norm(x, residual, following, c.epsilon)
        return x[self._ints(starts[1:], torch.int64) - 1] @ self.head

    def fork(self, parents: list[int], children: list[int]) -> None:
        self._succeed(
            ops.fork_sequences(self.caches, self.tables, self.lens, self.refs, self._ints(parents), self._ints(children))
        )
        for parent, child in zip(parents, children):
            self.host_lens[child] = self.host_lens[parent]

    def release(self, rows: list[int]) -> None:
        ops.release_sequences(self.tables, self.lens, self.refs, self._ints(rows))
        for row in rows:
            self.host_lens[row] = 0

    def compact(self) -> int:
        """Moves the pages in use to the lowest numbers and returns how many there are."""
        self.tables, self.refs, live = ops.compact_pages(self.caches, self.tables, self.refs)
        return int(live)


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__.split("\n", 1)[0])
    parser.add_argument("--seven-b", action="store_true", help="the 7B architecture's layers (4 of them by default)")
    parser.add_argument("--layers", type=int)
    parser.add_argument("--prompt", type=int, default=1000)
    parser.add_argument("--chunk", type=int, default=512)
    parser.add_argument("--samples", type=int, default=8)
    parser.add_argument("--steps", type=int, default=32)
    args = parser.parse_args()
    config = Config()
    if args.seven_b:
        config = Config(vocabulary=4096, hidden=3584, heads=28, kv_heads=4, head_size=128, intermediate=18944, layers=4)
    if args.layers:
        config.layers = args.layers
    config.max_position = max(config.max_position, args.prompt + args.steps + 1)
    torch.set_grad_enabled(False)
    decoder = PagedDecoder(config, rows=2 * args.samples, pages=4 * (-(-args.prompt // 16) + args.samples * (2 + args.steps // 16)))

    generator = torch.Generator().manual_seed(1)
    prompt = torch.randint(0, config.vocabulary, (args.prompt,), generator=generator).tolist()
    torch.cuda.synchronize()
    began = time.perf_counter()
    for at in range(0, args.prompt, args.chunk):
        logits = decoder.forward([0], [prompt[at : at + args.chunk]])
    torch.cuda.synchronize()
    print(f"prefill: {args.prompt} tokens in chunks of {args.chunk}: {1e3 * (time.perf_counter() - began):.1f} ms")

    rows = list(range(args.samples))
    decoder.fork([0] * (args.samples - 1), rows[1:])
    tokens = logits[0].float().topk(args.samples).indices.tolist()  # each sample continues with another token
    texts = [[t] for t in tokens]
    began = time.perf_counter()
    for _ in range(args.steps):
        tokens = decoder.forward(rows, [[t] for t in tokens]).argmax(-1).tolist()
        for text, token in zip(texts, tokens):
            text.append(token)
    spent = time.perf_counter() - began
    print(f"decode: {args.samples} sequences x {args.steps} steps: {1e3 * spent / args.steps:.2f} ms a step")
    held = int((decoder.refs > 0).sum())
    decoder.release(rows[::2])
    live = decoder.compact()
    print(f"pages: {held} in use, {live} after releasing half the samples, compacted")
    print("first tokens of the samples left:", [text[:4] for text in texts[1::2]])


if __name__ == "__main__":
    main()

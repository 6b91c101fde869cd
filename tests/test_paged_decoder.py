"""The paged-cache ops together with the norms and SiLU-and-mul: the example decoder's chunked prefill,
forked decoding, release and compaction against a plain forward over the whole text in 32 bits."""

from __future__ import annotations

import importlib.util
from pathlib import Path

import pytest
import torch

from cache_reference import rotate
from inference_performance_lab.kernels import capi
from parity import require_cuda

gpu = pytest.mark.gpu

EXAMPLE = Path(__file__).resolve().parents[1] / "inference-performance-lab_b200" / "examples" / "paged_decoder.py"


def load_example():
    import sys

    spec = importlib.util.spec_from_file_location("paged_decoder_example", EXAMPLE)
    module = importlib.util.module_from_spec(spec)
    sys.modules[spec.name] = module
    spec.loader.exec_module(module)
    return module


def plain_logits(decoder, text):
    """Logits after the last token, every op in 32 bits over the whole text."""
    c = decoder.config

    def norm(x, w):
        return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + c.epsilon) * w.float()

    x = decoder.embedding[torch.tensor(text, device="cuda")].float()
    positions = torch.arange(len(text), device="cuda")
    hidden = torch.ones(len(text), len(text), dtype=torch.bool, device="cuda").triu(1)
    for layer in decoder.layers:
        y = norm(x, layer["norms"][0])
        q, k, v = (y @ layer["qkv"].float()).view(len(text), -1, c.head_size).split([c.heads, c.kv_heads, c.kv_heads], 1)
        q, k = (rotate(t, positions, decoder.table, True).float() for t in (q, k))
        group = c.heads // c.kv_heads
        scores = torch.einsum("qhd,khd->hqk", q, k.repeat_interleave(group, 1)) * c.head_size**-0.5
        weights = scores.masked_fill(hidden, -torch.inf).softmax(-1)
        y = torch.einsum("hqk,khd->qhd", weights, v.repeat_interleave(group, 1)).flatten(1)
        x = x + y @ layer["out"].float()
        gate, up = (norm(x, layer["norms"][1]) @ layer["gate_up"].float()).chunk(2, -1)
        x = x + (torch.nn.functional.silu(gate) * up) @ layer["down"].float()
    return norm(x[-1:], decoder.norm) @ decoder.head.float()


@gpu
@torch.no_grad()
def test_chunks_forks_and_compaction_match_a_plain_forward():
    """bf16 against 32 bits through two layers: each of about 20 roundings moves the hidden state by up to
    2^-8 of its size, independently; 0.03 of the logits' norm is three times what they add up to."""
    require_cuda()
    module = load_example()
    decoder = module.PagedDecoder(module.Config(), rows=8, pages=96)
    generator = torch.Generator().manual_seed(3)

    def tokens(n):
        return torch.randint(0, 512, (n,), generator=generator).tolist()

    def close(got, text):
        want = plain_logits(decoder, text)
        assert (got.float() - want).norm() <= 0.03 * want.norm()

    texts = {0: tokens(150), 5: tokens(37)}
    decoder.forward([0], [texts[0][:70]])
    # A chunk of one prompt beside a whole other one.
    logits = decoder.forward([0, 5], [texts[0][70:], texts[5]])
    close(logits[0], texts[0])
    close(logits[1], texts[5])
    decoder.fork([0, 0, 5], [1, 2, 6])
    for child, parent in ((1, 0), (2, 0), (6, 5)):
        texts[child] = list(texts[parent])
    for _ in range(20):
        rows = sorted(texts)
        added = [tokens(1) for _ in rows]
        logits = decoder.forward(rows, added)
        for row, token in zip(rows, added):
            texts[row] += token
    for i, row in enumerate(rows):
        close(logits[i], texts[row])
    decoder.release([0, 5])
    del texts[0], texts[5]
    held = decoder.compact()
    assert held == int((decoder.refs > 0).sum()) and (decoder.refs[:held] > 0).all()
    rows = sorted(texts)
    added = [tokens(3) for _ in rows]
    logits = decoder.forward(rows, added)
    for i, row in enumerate(rows):
        close(logits[i], texts[row] + added[i])
    with pytest.raises(RuntimeError, match="out of pages"):
        decoder.forward([7], [tokens(96 * 16)])
    assert capi.device_fault_flags(0) == 0

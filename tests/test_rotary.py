"""Rotary positions against the formula in 64 bits: layouts, partial heads, strides, alignments, the
fused write into the pages, skipped tokens, refusals; and the tables for long contexts."""

from __future__ import annotations

import math

import pytest
import torch

from cache_reference import rotary_bound, rotate
from inference_performance_lab.kernels import capi, extension
from inference_performance_lab.kernels.rotary import rotary_cos_sin_cache, rotary_frequencies
from parity import require_cuda

gpu = pytest.mark.gpu


def bf16(*shape, seed=0):
    generator = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(*shape, generator=generator, device="cuda").to(torch.bfloat16)


def check(got, x, positions, table, is_neox):
    expected = rotate(x, positions, table, is_neox)
    assert ((got.double() - expected).abs() <= rotary_bound(x, expected)).all()
    assert torch.equal(got[..., table.shape[1] :], x[..., table.shape[1] :])


IN_PLACE = [
    (1, 28, 4, 128, 128, True), (64, 28, 4, 128, 128, True), (333, 28, 4, 128, 128, False),
    (2049, 32, 8, 64, 32, False), (77, 32, 8, 64, 32, True), (5, 3, 1, 80, 40, True), (5, 3, 1, 80, 40, False),
    (9, 12, 2, 96, 16, True), (3, 300, 1, 8, 2, False), (3, 2, 2, 7, 6, True), (130, 1, 1, 256, 256, True),
]


@gpu
@pytest.mark.parametrize("tokens, heads, kv_heads, dim, rot, is_neox", IN_PLACE)
def test_in_place(tokens, heads, kv_heads, dim, rot, is_neox):
    require_cuda()
    table = rotary_cos_sin_cache(rot, 4096)
    positions = torch.randint(0, 4096, (tokens,), device="cuda")
    positions[0] = 4095
    q0, k0 = bf16(tokens, heads, dim, seed=1), bf16(tokens, kv_heads, dim, seed=2)
    q, k = q0.clone(), k0.clone()
    extension.rotary_embedding(positions, q, k, table, is_neox)
    check(q, q0, positions, table, is_neox)
    check(k, k0, positions, table, is_neox)
    assert capi.device_fault_flags(0) == 0


@gpu
@pytest.mark.parametrize("offset", [0, 1, 4, 8])
@pytest.mark.parametrize("is_neox", [True, False])
def test_views_of_a_projection(offset, is_neox):
    """q, k and v split from one tensor at any alignment; what lies between them stays."""
    require_cuda()
    heads, kv_heads, dim, tokens = 6, 2, 64, 41
    flat = bf16(tokens * (heads + 2 * kv_heads) * dim + offset + 5, seed=3)
    before = flat.clone()

    def views(f):
        qkv = f[offset : offset + tokens * (heads + 2 * kv_heads) * dim].view(tokens, heads + 2 * kv_heads, dim)
        return qkv.split([heads, kv_heads, kv_heads], dim=1)

    q, k, v = views(flat)
    q0, k0, v0 = views(before)
    table = rotary_cos_sin_cache(48, 100)
    positions = torch.arange(tokens, device="cuda")
    extension.rotary_embedding(positions, q, k, table, is_neox)
    check(q, q0, positions, table, is_neox)
    check(k, k0, positions, table, is_neox)
    assert torch.equal(v, v0)
    assert torch.equal(flat[:offset], before[:offset]) and torch.equal(flat[-5:], before[-5:])


CACHED = [
    # tokens, heads, kv_heads, dim, rot, is_neox, page, pages, heads before tokens in a page
    (1, 28, 4, 128, 128, True, 16, 3, False), (64, 28, 4, 128, 128, True, 16, 40, False),
    (333, 4, 4, 64, 64, False, 48, 11, True), (100, 16, 1, 96, 48, True, 128, 2, False),
    (17, 3, 1, 80, 40, True, 5, 9, True), (33, 2, 2, 7, 4, False, 3, 12, False), (9, 40, 8, 80, 16, False, 64, 1, True),
]


@gpu
@pytest.mark.parametrize("tokens, heads, kv_heads, dim, rot, is_neox, page, pages, hnd", CACHED)
def test_write_into_pages(tokens, heads, kv_heads, dim, rot, is_neox, page, pages, hnd):
    require_cuda()
    table = rotary_cos_sin_cache(rot, 2000)
    positions = torch.randint(0, 2000, (tokens,), device="cuda")
    slots = torch.randperm(pages * page, device="cuda")[:tokens].contiguous()
    slots[tokens // 2 :: 5] = -1
    q0, k, v = bf16(tokens, heads, dim, seed=1), bf16(tokens, kv_heads, dim, seed=2), bf16(tokens, kv_heads, dim, seed=3)
    store = bf16(2, pages, kv_heads, page, dim, seed=4) if hnd else bf16(2, pages, page, kv_heads, dim, seed=4)
    before = store.clone()
    view = (lambda s: s.transpose(2, 3)) if hnd else (lambda s: s)
    kc, vc = view(store).unbind(0)
    q, k0 = q0.clone(), k.clone()
    extension.rotary_embedding_cache(positions, q, k, v, table, kc, vc, slots, is_neox)
    check(q, q0, positions, table, is_neox)
    assert torch.equal(k, k0)
    kept = slots >= 0
    where = (slots[kept] // page, slots[kept] % page)
    check(kc[where], k[kept], positions[kept], table, is_neox)
    assert torch.equal(vc[where], v[kept])
    mask = torch.ones(pages, page, dtype=torch.bool, device="cuda")
    mask[where] = False
    for cache, old in zip((kc, vc), view(before).unbind(0)):
        assert torch.equal(cache[mask], old[mask])
    assert capi.device_fault_flags(0) == 0


@gpu
def test_slots_past_32_bit_offsets():
    require_cuda()
    page, kv_heads, dim = 16, 4, 128
    pages = 2**31 // (page * kv_heads * dim) + 8  # the last pages start past 2^31 elements
    kc = torch.empty(pages, page, kv_heads, dim, dtype=torch.bfloat16, device="cuda")
    table = rotary_cos_sin_cache(dim, 64)
    positions = torch.arange(8, device="cuda")
    slots = torch.arange(pages * page - 8, pages * page, device="cuda")
    q, k, v = bf16(8, 4, dim), bf16(8, kv_heads, dim, seed=1), bf16(8, kv_heads, dim, seed=2)
    vc = torch.empty_like(kc)
    extension.rotary_embedding_cache(positions, q, k, v, table, kc, vc, slots)
    check(kc[-1, 8:], k, positions, table, True)
    assert torch.equal(vc[-1, 8:], v)


@gpu
def test_indices_outside_their_range_are_skipped():
    require_cuda()
    capi.clear_device_fault_flags(0)
    table = rotary_cos_sin_cache(64, 10)
    q0, k, v = bf16(4, 2, 64), bf16(4, 1, 64, seed=1), bf16(4, 1, 64, seed=2)
    kc, vc = torch.zeros(2, 2, 16, 1, 64, device="cuda", dtype=torch.bfloat16).unbind(0)
    q = q0.clone()
    positions = torch.tensor([3, 10, -1, 9], device="cuda")
    slots = torch.tensor([5, 6, 7, 32], device="cuda")
    extension.rotary_embedding_cache(positions, q, k, v, table, kc, vc, slots)
    assert capi.device_fault_flags(0) == 8
    capi.clear_device_fault_flags(0)
    check(q[:1], q0[:1], positions[:1], table, True)
    assert torch.equal(q[1:], q0[1:])
    assert torch.equal(vc[0, 5], v[0])
    assert (vc != 0).any(-1).sum() == 1 and (kc != 0).any(-1).sum() == 1


@gpu
def test_no_tokens_streams_and_graphs():
    require_cuda()
    table = rotary_cos_sin_cache(128, 100)
    empty = torch.empty(0, 4, 128, device="cuda", dtype=torch.bfloat16)
    extension.rotary_embedding(torch.empty(0, dtype=torch.int64, device="cuda"), empty, empty.clone(), table)
    q0, k0 = bf16(50, 4, 128), bf16(50, 2, 128, seed=1)
    positions = torch.arange(50, device="cuda")
    q, k = q0.clone(), k0.clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        extension.rotary_embedding(positions, q, k, table)
    graph.replay()
    torch.cuda.synchronize()
    check(q, q0, positions, table, True)
    check(k, k0, positions, table, True)


@gpu
def test_refusals():
    require_cuda()
    table = rotary_cos_sin_cache(64, 10)
    positions = torch.arange(4, device="cuda")
    q, k = bf16(4, 2, 64), bf16(4, 1, 64)
    cache = bf16(2, 16, 1, 64)
    for args, message in [
        ((positions, q.float(), k, table), "query must be bfloat16"),
        ((positions, q, k.cpu(), table), "same device"),
        ((positions.int(), q, k, table), "positions must be contiguous int64"),
        ((positions[:3], q, k, table), "same number of tokens"),
        ((positions, q, k[..., :32], table), "same head size"),
        ((positions, q, k, table.to(torch.bfloat16)), "cos_sin_cache must be contiguous float32"),
        ((positions, q, k, rotary_cos_sin_cache(128, 10)), "at most the head size"),
        ((positions, q, k, table[:, :63].contiguous()), "must be even"),
        ((positions, q, k, table[:0]), "at least one position"),
        ((positions, q.transpose(1, 2), k, table), "contiguous last dimension"),
    ]:
        with pytest.raises(RuntimeError, match=message):
            extension.rotary_embedding(*args)
    for args, message in [
        ((k[:3], cache, cache, positions), "key and value must have identical shapes"),
        ((k, cache, cache[:1], positions), "key_cache and value_cache must have identical shapes"),
        ((k, cache[..., :32], cache[..., :32], positions), "heads and head size of key"),
        ((k, cache, cache, positions.int()), "slot_mapping must be contiguous int64"),
    ]:
        value, kc, vc, slots = args
        with pytest.raises(RuntimeError, match=message):
            extension.rotary_embedding_cache(positions, q, k, value, table, kc, vc, slots)


def rotary_args(**changes):
    base = 0x7F0000000000
    a = dict(positions=base, cos_sin_cache=base, query=base, key=base, num_tokens=1, num_heads=2, num_kv_heads=1, head_size=64,
             rotary_dim=64, max_position=8, query_token_stride=128, query_head_stride=64, key_token_stride=64,
             key_head_stride=64, is_neox=1, value=base, key_cache=base, value_cache=base, slot_mapping=base, num_pages=1,
             page_size=16)
    a.update(changes)
    return capi.RotaryArgs(**a)


@pytest.mark.parametrize("changes, status, message", [
    (dict(num_tokens=-1), capi.IPL_ERROR_INVALID_VALUE, "non-negative"),
    (dict(num_heads=0), capi.IPL_ERROR_INVALID_VALUE, "must be positive"),
    (dict(rotary_dim=66), capi.IPL_ERROR_INVALID_VALUE, "at most the head size"),
    (dict(rotary_dim=31), capi.IPL_ERROR_INVALID_VALUE, "even"),
    (dict(max_position=0), capi.IPL_ERROR_INVALID_VALUE, "at least one position"),
    (dict(query=0), capi.IPL_ERROR_INVALID_VALUE, "non-null"),
    (dict(key=1), capi.IPL_ERROR_INVALID_VALUE, "2-byte aligned"),
    (dict(positions=4), capi.IPL_ERROR_INVALID_VALUE, "aligned to their types"),
    (dict(num_tokens=2**31), capi.IPL_ERROR_TOO_LARGE, "too large"),
    (dict(slot_mapping=0), capi.IPL_ERROR_INVALID_VALUE, "non-null"),
    (dict(page_size=0), capi.IPL_ERROR_INVALID_VALUE, "page size must be positive"),
    (dict(num_pages=2**27, page_size=16), capi.IPL_ERROR_TOO_LARGE, "too many slots"),
])
def test_argument_errors(changes, status, message):
    with pytest.raises(capi.IplError, match=message) as info:
        capi.rotary_embedding_cache(rotary_args(**changes))
    assert info.value.status == status


def test_tables():
    """Rows are cos and sin of position * base^(-2i/R), to half a unit in the last place of fp32 (2^-25)
    and the rounding of a 64-bit angle of at most 131072 (2^-36)."""
    table = rotary_cos_sin_cache(64, 131072, base=1e6, device="cpu")
    assert table.shape == (131072, 64) and table.dtype == torch.float32
    for position in (0, 1, 4097, 131071):
        for i in (0, 1, 17, 31):
            angle = position * 1e6 ** (-2 * i / 64)
            assert abs(table[position, i] - math.cos(angle)) <= 2**-25 + 2**-34
            assert abs(table[position, 32 + i] - math.sin(angle)) <= 2**-25 + 2**-34
    linear = rotary_cos_sin_cache(64, 64, scaling={"type": "linear", "factor": 4.0}, device="cpu")
    assert torch.equal(linear[8], rotary_cos_sin_cache(64, 64, device="cpu")[2])


def test_scaled_frequencies():
    plain, _ = rotary_frequencies(128, 500000.0)
    scaling = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
                   original_max_position_embeddings=8192)
    scaled, factor = rotary_frequencies(128, 500000.0, scaling)
    assert factor == 1.0
    for i, f in enumerate(plain.tolist()):
        wavelength = 2 * math.pi / f
        if wavelength < 8192 / 4:
            want = f
        elif wavelength > 8192:
            want = f / 8
        else:
            smooth = (8192 / wavelength - 1.0) / 3.0
            want = (1 - smooth) * f / 8 + smooth * f
        assert scaled[i].item() == pytest.approx(want, rel=1e-12)
    plain, _ = rotary_frequencies(128, 1e6)
    scaled, factor = rotary_frequencies(128, 1e6, dict(type="yarn", factor=4.0, original_max_position_embeddings=32768))
    assert factor == pytest.approx(0.1 * math.log(4.0) + 1.0)
    turns = 32768 * plain / (2 * math.pi)
    assert torch.equal(scaled[turns > 40], plain[turns > 40])
    assert torch.allclose(scaled[turns < 0.9], plain[turns < 0.9] / 4, rtol=1e-12, atol=0)
    ratio = scaled / plain
    assert ((ratio[1:] - ratio[:-1]) <= 1e-15).all()


@pytest.mark.parametrize("args, kwargs, message", [
    ((63,), {}, "even"), ((64, 0.0), {}, "base"),
    ((64,), dict(scaling=dict(type="cubic", factor=2.0)), "unknown rope scaling"),
    ((64,), dict(scaling=dict(type="linear", factor=0.5)), "at least 1"),
])
def test_table_refusals(args, kwargs, message):
    with pytest.raises(ValueError, match=message):
        rotary_frequencies(*args, **kwargs)


def test_yarn_factor_from_two_scales():
    """The factor on cosines and sines that m(s) = 0.1 s ln(factor) + 1 gives, and its precedence."""
    yarn = dict(rope_type="yarn", factor=40.0, original_max_position_embeddings=4096)
    log = math.log(40.0)
    for more, want in (
        (dict(), 0.1 * log + 1),
        (dict(mscale=1.0, mscale_all_dim=1.0), 1.0),
        (dict(mscale=0.707, mscale_all_dim=0.707), 1.0),
        (dict(mscale=1.0, mscale_all_dim=0.0), 0.1 * log + 1),
        (dict(mscale=1, mscale_all_dim=0.5), (0.1 * log + 1) / (0.05 * log + 1)),
        (dict(mscale=1.0, mscale_all_dim=1.0, attention_factor=1.25), 1.25),
        (dict(mscale=0.5, attention_factor=1.25), 1.25),
        (dict(mscale=None, mscale_all_dim=None, attn_factor=1, extrapolation_factor=1.0), 0.1 * log + 1),
    ):
        frequencies, factor = rotary_frequencies(64, 10000.0, {**yarn, **more})
        assert factor == pytest.approx(want, rel=1e-15)
        assert torch.equal(frequencies, rotary_frequencies(64, 10000.0, yarn)[0])


def test_yarn_ramp_without_rounding():
    """truncate=False: the ramp begins and ends where a pair would turn beta_fast and beta_slow times."""
    dim, base, original, by = 64, 150000.0, 4096, 32.0
    yarn = dict(rope_type="yarn", factor=by, original_max_position_embeddings=original, beta_fast=32.0, beta_slow=1.0)
    plain, _ = rotary_frequencies(dim, base)
    scaled, _ = rotary_frequencies(dim, base, {**yarn, "truncate": False})
    # Pair i turns original / (2 pi base^(2 i / dim)) times: i as a function of the turns.
    at = [math.log(original / (2 * math.pi * turns), base) * dim / 2 for turns in (32.0, 1.0)]
    for i in range(dim // 2):
        kept = 1 - min(max((i - at[0]) / (at[1] - at[0]), 0.0), 1.0)
        assert scaled[i].item() == pytest.approx(plain[i].item() * (kept + (1 - kept) / by), rel=1e-12)
    rounded, _ = rotary_frequencies(dim, base, yarn)
    assert torch.equal(rounded, rotary_frequencies(dim, base, {**yarn, "truncate": True})[0])
    assert not torch.equal(rounded, scaled)


@pytest.mark.parametrize("more, message", [
    (dict(mscale=1.0), "given together"), (dict(mscale_all_dim=1.0), "given together"),
    (dict(attn_factor=1.2), "attn_factor"), (dict(extrapolation_factor=0.5), "extrapolation_factor"),
])
def test_yarn_refusals(more, message):
    with pytest.raises(ValueError, match=message):
        rotary_frequencies(64, 10000.0, dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=4096, **more))

"""Attention over a paged cache against the formula in 64 bits, where it can go wrong: lengths of zero
and one, rows that see nothing, windows, pages that end inside a tile, garbage (NaN, infinities) in
unused pages, rows past a length and table entries past a sequence's pages, odd group and head sizes,
strides, long offsets, streams and graphs; and its refusals."""

from __future__ import annotations

import random

import pytest
import torch

from cache_reference import attention, attention_bound
from inference_performance_lab.kernels import capi, extension
from parity import require_cuda

gpu = pytest.mark.gpu


def make(new, total, heads=28, kv_heads=4, dim=128, page=16, seed=0, spare=3, hnd=False, fill=float("nan"), width=None):
    """Inputs whose every unused place holds `fill`, and whose unused table entries are no page numbers."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    counts = [-(-t // page) for t in total]
    pages = sum(counts) + spare
    shape = (2, pages, kv_heads, page, dim) if hnd else (2, pages, page, kv_heads, dim)
    store = torch.full(shape, fill, dtype=torch.bfloat16, device="cuda")
    kc, vc = (store.transpose(2, 3) if hnd else store).unbind(0)
    width = width or max(counts + [1]) + 2
    tables = torch.full((len(new), width), 2**30, dtype=torch.int32, device="cuda")
    order = torch.randperm(pages, generator=g, device="cuda").int()
    at = 0
    for s, (c, t) in enumerate(zip(counts, total)):
        mine = order[at : at + c]
        at += c
        tables[s, :c] = mine
        for j, p in enumerate(mine.tolist()):
            rows = min(page, t - j * page)
            for cache in (kc, vc):
                cache[p, :rows] = torch.randn(rows, kv_heads, dim, generator=g, device="cuda").to(torch.bfloat16)
    q = (torch.randn(sum(new), heads, dim, generator=g, device="cuda") * 1.5).to(torch.bfloat16)
    starts = torch.tensor([sum(new[:i]) for i in range(len(new) + 1)], dtype=torch.int32, device="cuda")
    lens = torch.tensor(total, dtype=torch.int32, device="cuda")
    return q, kc, vc, tables, starts, lens


def call(inputs, new, total, window=0, scale=None):
    q = inputs[0]
    scale = scale or q.shape[2] ** -0.5
    return extension.paged_attention(*inputs, max(new), max(total), scale, window), scale


def check(inputs, new, total, window=0, scale=None):
    got, scale = call(inputs, new, total, window, scale)
    expected, size = attention(*inputs, scale, window)
    error = (got.double() - expected).abs()
    assert (error <= attention_bound(expected, size)).all(), (error - attention_bound(expected, size)).max()
    assert capi.device_fault_flags(0) == 0
    return got


SINGLE = [
    # new, total (per sequence), heads, kv_heads, dim, page, window
    ([1], [1], 28, 4, 128, 16, 0),
    ([1], [17], 28, 4, 128, 16, 0),
    ([1] * 5, [1, 16, 300, 2, 129], 28, 4, 128, 16, 0),
    ([1] * 3, [1027, 0, 513], 28, 4, 128, 16, 0),
    ([1] * 4, [40, 64, 65, 700], 32, 8, 64, 32, 0),
    ([1] * 3, [900, 31, 128], 16, 16, 64, 16, 100),
    ([1] * 2, [260, 77], 16, 1, 96, 48, 0),
    ([1] * 2, [260, 77], 40, 8, 80, 128, 33),
    ([1], [5000], 4, 4, 128, 64, 1),
    ([1, 1], [333, 90], 64, 1, 128, 16, 0),
    ([1, 1], [70, 9], 6, 3, 256, 16, 0),
    ([1, 1], [70, 9], 4, 2, 20, 7, 12),
    ([1] * 3, [4097, 4096, 4095], 8, 1, 128, 256, 0),
]
CHUNKS = [
    ([2], [2], 28, 4, 128, 16, 0),
    ([17, 1, 0, 64], [40, 300, 12, 64], 28, 4, 128, 16, 0),
    ([129], [129], 4, 4, 128, 16, 0),
    ([200, 3], [1000, 600], 28, 4, 128, 64, 0),
    ([300], [301], 32, 8, 64, 32, 70),
    ([130, 40], [700, 41], 16, 1, 96, 48, 0),
    ([50], [50], 40, 8, 80, 128, 7),
    ([511, 64], [511, 900], 8, 2, 128, 128, 256),
    ([9, 30], [70, 30], 6, 3, 256, 16, 0),
    ([9, 30], [70, 30], 4, 2, 20, 7, 12),
    ([37], [2300], 12, 2, 64, 16, 1000),
    ([260], [260], 16, 16, 8, 16, 0),
    ([5, 4, 3], [200, 190, 4], 28, 4, 128, 16, 0),
    ([1, 150, 1, 33], [2000, 150, 3, 1500], 28, 4, 128, 16, 0),
    ([90], [5000], 3, 1, 128, 32, 0),
]


@gpu
@pytest.mark.parametrize("new, total, heads, kv_heads, dim, page, window", SINGLE + CHUNKS)
def test_against_the_formula(new, total, heads, kv_heads, dim, page, window):
    require_cuda()
    inputs = make(new, total, heads, kv_heads, dim, page, seed=len(new) + dim)
    check(inputs, new, total, window)


@gpu
@pytest.mark.parametrize("fill", [float("inf"), float("-inf"), 3e38])
def test_unused_places_hold_infinities(fill):
    require_cuda()
    for new, total in (([1, 1], [37, 5]), ([20, 150], [37, 333])):
        check(make(new, total, fill=fill), new, total)


@gpu
def test_rows_that_see_nothing_are_zero():
    """More new tokens than the cache holds: the first ones sit before position 0."""
    require_cuda()
    for new, total in (([4], [2]), ([150], [20]), ([1], [0]), ([140], [0]), ([3, 1], [1, 5])):
        got = check(make(new, total), new, total)
        assert (got[: new[0] - total[0]] == 0).all()


@gpu
def test_heads_before_tokens_and_views():
    """A cache with heads before tokens, q a view of a projection, output of another layout."""
    require_cuda()
    for new, total in (([1] * 4, [65, 2, 130, 700]), ([70, 200], [100, 500])):
        q, kc, vc, tables, starts, lens = make(new, total, hnd=True)
        wide = torch.randn(q.shape[0], 36, 128, device="cuda").to(torch.bfloat16)
        wide[:, 3:31] = q
        q = wide[:, 3:31]
        check((q, kc, vc, tables, starts, lens), new, total)
        out = torch.zeros(28, q.shape[0], 128, device="cuda", dtype=torch.bfloat16).transpose(0, 1)
        torch.ops.inference_performance_lab.paged_attention(out, q, kc, vc, tables, starts, lens, max(new), max(total), 0.1, 0)
        expected, size = attention(q, kc, vc, tables, starts, lens, 0.1)
        assert ((out.double() - expected).abs() <= attention_bound(expected, size)).all()


@gpu
@pytest.mark.parametrize("offset", [1, 4])
def test_pointers_off_16_bytes(offset):
    require_cuda()
    for new, total in (([1, 1], [65, 200]), ([70], [100])):
        q, kc, vc, tables, starts, lens = make(new, total, heads=8, kv_heads=2, dim=64)

        def moved(t):
            flat = torch.empty(t.numel() + offset, dtype=t.dtype, device="cuda")[offset:]
            return flat.copy_(t.reshape(-1)).view(t.shape)

        check((moved(q), kc, vc, tables, starts, lens), new, total)
        check((q, moved(kc), moved(vc), tables, starts, lens), new, total)


@gpu
def test_peaked_and_shifted_scores():
    """Scores that grow along the keys by far more than an exponent's range, large equal offsets, and a
    single key that takes all the weight."""
    require_cuda()
    new, total = [1, 140], [900, 900]
    q, kc, vc, tables, starts, lens = make(new, total, heads=8, kv_heads=2)
    q.fill_(1.0)
    for s in range(2):
        for j, p in enumerate(tables[s, : -(-900 // 16)].tolist()):
            rows = min(16, 900 - j * 16)
            position = (torch.arange(rows, device="cuda") + j * 16).to(torch.bfloat16)
            kc[p, :rows] = (position / 64.0)[:, None, None]
    check((q, kc, vc, tables, starts, lens), new, total, scale=1.0)  # rises by 2 a key
    for s in range(2):
        for j, p in enumerate(tables[s, : -(-900 // 16)].tolist()):
            rows = min(16, 900 - j * 16)
            position = (torch.arange(rows, device="cuda") + j * 16).to(torch.bfloat16)
            kc[p, :rows] = (-position / 64.0 - 100.0)[:, None, None]
    check((q, kc, vc, tables, starts, lens), new, total, scale=1.0)  # falls from -12800


@gpu
def test_keys_at_masked_positions_never_matter():
    """NaN and infinite keys ahead of a token leave it as it is."""
    require_cuda()
    new, total = [40], [100]
    inputs = make(new, total)
    q, kc, vc, tables, starts, lens = inputs
    expected = check(inputs, new, total)
    for bad in (float("nan"), float("inf"), float("-inf")):
        page, row = int(tables[0, 6]), 3  # position 99, seen by the last token alone
        kc[page, row] = bad
        got, _ = call(inputs, new, total)
        assert torch.equal(got[:39], expected[:39])
        if bad != bad:
            assert got[39].isnan().all()


@gpu
def test_pages_outside_the_cache_contribute_nothing():
    require_cuda()
    capi.clear_device_fault_flags(0)
    new, total = [1, 20], [40, 40]
    q, kc, vc, tables, starts, lens = make(new, total, heads=4, kv_heads=2, dim=64)
    reference = [t.clone() for t in (kc, vc)]
    tables[:, 1] = torch.tensor([-5, 2**31 - 1], dtype=torch.int32, device="cuda")
    got, scale = call((q, kc, vc, tables, starts, lens), new, total)
    assert capi.device_fault_flags(0) == 8
    capi.clear_device_fault_flags(0)
    # The formula without positions 16 to 31.
    for s in range(2):
        pages = tables[s, [0, 2]].long()
        keys = torch.cat([reference[0][pages[0]], reference[0][pages[1], :8]]).double()
        values = torch.cat([reference[1][pages[0]], reference[1][pages[1], :8]]).double()
        position = torch.cat([torch.arange(16), torch.arange(32, 40)]).cuda()
        for t in range(int(starts[s]), int(starts[s + 1])):
            at = 40 - new[s] + t - int(starts[s])
            for h in range(4):
                logits = (keys[:, h // 2] @ q[t, h].double()) * scale
                w = torch.softmax(logits.masked_fill(position > at, -torch.inf), 0)
                want, size = w @ values[:, h // 2], w @ values[:, h // 2].abs()
                assert ((got[t, h].double() - want).abs() <= attention_bound(want, size)).all()


@gpu
def test_lengths_past_the_bounds_given():
    """max_query_len and max_seq_len only choose kernels: longer sequences come out right."""
    require_cuda()
    new, total = [1, 60, 1], [700, 500, 90]
    inputs = make(new, total)
    expected, size = attention(*inputs, 0.125)
    for most_new, most in ((1, 1), (1, 700), (60, 32), (2, 2), (4096, 100000)):
        got = extension.paged_attention(*inputs, most_new, most, 0.125)
        assert ((got.double() - expected).abs() <= attention_bound(expected, size)).all(), (most_new, most)


@gpu
def test_more_sequences_than_threads():
    """Hundreds of ragged sequences: single tokens, chunks and both, with lengths of zero among them."""
    require_cuda()
    rng = random.Random(7)
    for most_new, longest, count in ((1, 300, 700), (40, 250, 450), (9, 2000, 130)):
        new = [rng.choice([0, 1, 1, rng.randint(1, most_new)]) for _ in range(count)]
        total = [rng.randint(0, longest) for _ in range(count)]
        inputs = make(new, total, heads=4, kv_heads=2, dim=64, seed=count)
        check(inputs, new, total)


@gpu
def test_long_sequences_among_many_single_tokens_past_the_bounds():
    """A call that plans equal shares of single tokens meets chunks that max_query_len denies."""
    require_cuda()
    new = [60 if s % 50 == 3 else 1 for s in range(240)]
    total = [max(n, 200 + s) for s, n in enumerate(new)]
    inputs = make(new, total, heads=14, kv_heads=2, dim=64)
    expected, size = attention(*inputs, 0.125)
    got = extension.paged_attention(*inputs, 1, max(total), 0.125)
    assert ((got.double() - expected).abs() <= attention_bound(expected, size)).all()


@gpu
def test_groups_wider_than_a_tile():
    require_cuda()
    for new, total in (([1, 3], [300, 40]), ([50], [90])):
        check(make(new, total, heads=200, kv_heads=1, dim=64), new, total)


@gpu
def test_broadcast_keys():
    """One key head shown as four by a stride of 0: not mappable, computed all the same."""
    require_cuda()
    for new, total in (([1, 1], [300, 40]), ([150], [190])):
        q, kc, vc, tables, starts, lens = make(new, total, heads=8, kv_heads=1, dim=64)
        wide = [c.expand(-1, -1, 4, -1) for c in (kc, vc)]
        check((q, *wide, tables, starts, lens), new, total)


@gpu
def test_padding_rows_are_not_written():
    require_cuda()
    for new, total in (([1, 1], [33, 40]), ([30, 20], [33, 400])):
        q, kc, vc, tables, starts, lens = make(new, total)
        padded = torch.cat([q, q.new_full((9, 28, 128), float("nan"))])
        out = torch.full_like(padded, 7.0)
        torch.ops.inference_performance_lab.paged_attention(out, padded, kc, vc, tables, starts, lens, max(new), max(total), 0.1, 0)
        expected, size = attention(q, kc, vc, tables, starts, lens, 0.1)
        assert ((out[:-9].double() - expected).abs() <= attention_bound(expected, size)).all()
        assert (out[-9:] == 7.0).all()


@gpu
def test_offsets_past_32_bits():
    """A cache of more than 2^31 elements, a sequence in its last pages."""
    require_cuda()
    page, kv_heads, dim = 16, 4, 128
    pages = 2**31 // (page * kv_heads * dim) + 40
    kc = torch.empty(pages, page, kv_heads, dim, dtype=torch.bfloat16, device="cuda")
    vc = torch.empty_like(kc)
    kc[-40:].normal_()
    vc[-40:].normal_()
    tables = torch.arange(pages - 40, pages, dtype=torch.int32, device="cuda").flip(0)[None].contiguous()
    lens = torch.tensor([639], dtype=torch.int32, device="cuda")
    for n in (1, 100):
        q = torch.randn(n, 28, dim, device="cuda").to(torch.bfloat16)
        starts = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        check((q, kc, vc, tables, starts, lens), [n], [639])


@gpu
def test_repeatable_on_other_streams_and_in_graphs():
    require_cuda()
    for new, total in (([1] * 3, [5000, 31, 700]), ([1, 90], [3000, 2000])):
        inputs = make(new, total)
        expected = check(inputs, new, total)
        torch.cuda.synchronize()
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            again = [call(inputs, new, total)[0] for _ in range(3)]
        stream.synchronize()
        assert all(torch.equal(a, expected) for a in again)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured, _ = call(inputs, new, total)
        inputs[0].neg_()
        graph.replay()
        torch.cuda.synchronize()
        negated = captured.clone()
        assert torch.equal(negated, call(inputs, new, total)[0])
        inputs[0].neg_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, expected)


@gpu
def test_nothing_to_do():
    require_cuda()
    q, kc, vc, tables, starts, lens = make([1], [5])
    assert extension.paged_attention(q[:0], kc, vc, tables, starts * 0, lens, 0, 5, 0.1).shape == (0, 28, 128)
    none = extension.paged_attention(q, kc, vc, tables[:0], starts[:1], lens[:0], 0, 0, 0.1)
    assert none.shape == q.shape


@gpu
def test_refusals():
    require_cuda()
    q, kc, vc, tables, starts, lens = make([1, 2], [5, 9], heads=4, kv_heads=2, dim=64)

    def refused(message, **changes):
        a = dict(query=q, key_cache=kc, value_cache=vc, block_tables=tables, query_start_loc=starts, seq_lens=lens,
                 max_query_len=2, max_seq_len=9, scale=0.1, window=0)
        a.update(changes)
        with pytest.raises(RuntimeError, match=message):
            extension.paged_attention(**a)

    refused("query must be bfloat16", query=q.half())
    refused("key_cache must be bfloat16", key_cache=kc.float())
    refused("identical shapes", value_cache=vc[1:])
    refused("same head size", query=q[..., :32])
    refused("multiple of the number of key heads", query=q[:, :3])
    refused("same sequences", seq_lens=lens[:1])
    refused("same sequences", query_start_loc=starts[:2])
    refused("block_tables must be int32", block_tables=tables.long())
    refused("seq_lens must be contiguous int32", seq_lens=lens.long())
    refused("same device", seq_lens=lens.cpu())
    refused("scale must be positive", scale=0.0)
    refused("scale must be positive", scale=float("nan"))
    refused("non-negative", window=-1)
    refused("non-negative", max_query_len=-1)


def attention_args(**changes):
    base = 0x7F0000000000
    a = dict(output=base, query=base, key_cache=base, value_cache=base, block_tables=base, query_start_loc=base, seq_lens=base,
             num_tokens=4, num_seqs=4, num_heads=28, num_kv_heads=4, head_size=128, num_pages=100, page_size=16, table_width=64,
             table_stride=64, output_token_stride=3584, output_head_stride=128, query_token_stride=3584,
             query_head_stride=128, key_cache_page_stride=8192, key_cache_token_stride=512, key_cache_head_stride=128,
             value_cache_page_stride=8192, value_cache_token_stride=512, value_cache_head_stride=128, max_query_len=1,
             max_seq_len=1024, window=0, scale=0.088, workspace=0, workspace_bytes=0)
    a.update(changes)
    return capi.PagedAttentionArgs(**a)


@pytest.mark.parametrize("changes, status, message", [
    (dict(num_tokens=-1), capi.IPL_ERROR_INVALID_VALUE, "non-negative"),
    (dict(num_heads=0), capi.IPL_ERROR_INVALID_VALUE, "must be positive"),
    (dict(page_size=0), capi.IPL_ERROR_INVALID_VALUE, "must be positive"),
    (dict(num_heads=30), capi.IPL_ERROR_INVALID_VALUE, "multiple of the number of key heads"),
    (dict(window=-1), capi.IPL_ERROR_INVALID_VALUE, "non-negative"),
    (dict(scale=-1.0), capi.IPL_ERROR_INVALID_VALUE, "scale must be positive"),
    (dict(head_size=264), capi.IPL_ERROR_TOO_LARGE, "at most 256"),
    (dict(num_tokens=2**31), capi.IPL_ERROR_TOO_LARGE, "too large"),
    (dict(key_cache=0), capi.IPL_ERROR_INVALID_VALUE, "non-null"),
    (dict(query=3), capi.IPL_ERROR_INVALID_VALUE, "2-byte aligned"),
    (dict(seq_lens=2), capi.IPL_ERROR_INVALID_VALUE, "4-byte aligned"),
])
def test_argument_errors(changes, status, message):
    with pytest.raises(capi.IplError, match=message) as info:
        capi.paged_attention(attention_args(**changes))
    assert info.value.status == status
    assert capi.paged_attention_plan(attention_args(**changes)) == "invalid"
    with pytest.raises(capi.IplError, match=message):
        capi.paged_attention_workspace(attention_args(**changes))


def test_no_tokens_needs_no_device():
    capi.paged_attention(attention_args(num_tokens=0))
    assert capi.paged_attention_plan(attention_args(num_tokens=0)) == "none"
    assert capi.paged_attention_workspace(attention_args(num_tokens=0)) == 0


def test_plans():
    """The kernels a call would run, on a B200's 148 SMs."""
    plan = lambda **changes: capi.paged_attention_plan(attention_args(**changes))  # noqa: E731
    # Few sequences: a cluster each; many, or long ones: equal shares.
    assert plan() == "attention_short_kernel<1>"
    assert plan(num_tokens=64, num_seqs=64, max_seq_len=8192) == "attention_shared_kernel<1> + attention_join_parts_kernel"
    assert plan(max_seq_len=65536, table_width=4096) == "attention_shared_kernel<1> + attention_join_parts_kernel"
    assert plan(num_heads=64, query_token_stride=8192, output_token_stride=8192) == "attention_short_kernel<2>"
    # Chunks: the tile kernel, beside a short one where single tokens may be among them.
    chunk = dict(num_tokens=2048, num_seqs=1, max_query_len=2048, max_seq_len=16384, table_width=1024)
    assert plan(**chunk) == "attention_tile_kernel + attention_join_rows_kernel"
    mixed = {**chunk, "num_tokens": 2050, "num_seqs": 3, "max_seq_len": 32768}
    assert plan(**mixed) == ("attention_tile_kernel + attention_join_rows_kernel + attention_shared_kernel<1> + "
                             "attention_join_parts_kernel")
    # A few tokens stay with the short kernel, many sequences of a few with the tile kernel.
    assert plan(num_tokens=4, num_seqs=1, max_query_len=4) == "attention_short_kernel<2>"
    assert plan(num_tokens=256, num_seqs=64, max_query_len=4, max_seq_len=2000) == "attention_tile_kernel + attention_join_rows_kernel"
    # Anything that does not lie in 16-byte chunks and blocks of 16 keys: a warp a row.
    for odd in (dict(head_size=20), dict(page_size=24), dict(key_cache=0x7F0000000008), dict(query_head_stride=132),
                dict(head_size=256), dict(value_cache_token_stride=516)):
        assert plan(**odd) == "attention_row_kernel"
    # Broadcast keys (a stride of 0) cannot be mapped: rows of any number through the short kernel.
    assert plan(**chunk, key_cache_head_stride=0) == "attention_short_kernel<2>"
    assert capi.paged_attention_workspace(attention_args()) == 0
    parts = 2 * 148 * (256 * (128 * 4 + 8) + 16)
    assert capi.paged_attention_workspace(attention_args(**chunk)) == parts


@gpu
@pytest.mark.parametrize("new, total", [([1200], [2400]), ([1] * 64, [3000] * 64), ([1] * 8 + [500], [3000] * 9)])
def test_workspace_at_any_16_bytes(new, total):
    """Parts of cut rows in a workspace whose base is a multiple of 16 bytes and not of 32, as in one that is."""
    require_cuda()
    q, kc, vc, tables, starts, lens = make(new, total)
    outs = [torch.empty_like(q) for _ in range(2)]
    for out, offset in zip(outs, (0, 16)):
        a = capi.PagedAttentionArgs(
            output=out.data_ptr(), query=q.data_ptr(), key_cache=kc.data_ptr(), value_cache=vc.data_ptr(),
            block_tables=tables.data_ptr(), query_start_loc=starts.data_ptr(), seq_lens=lens.data_ptr(), num_tokens=q.shape[0],
            num_seqs=len(new), num_heads=28, num_kv_heads=4, head_size=128, num_pages=kc.shape[0], page_size=16,
            table_width=tables.shape[1], table_stride=tables.stride(0), output_token_stride=out.stride(0),
            output_head_stride=out.stride(1), query_token_stride=q.stride(0), query_head_stride=q.stride(1),
            key_cache_page_stride=kc.stride(0), key_cache_token_stride=kc.stride(1), key_cache_head_stride=kc.stride(2),
            value_cache_page_stride=vc.stride(0), value_cache_token_stride=vc.stride(1), value_cache_head_stride=vc.stride(2),
            max_query_len=max(new), max_seq_len=max(total), window=0, scale=128**-0.5)
        size = capi.paged_attention_workspace(a)
        assert size > 0
        workspace = torch.empty(size + 48, dtype=torch.uint8, device="cuda")
        at = -workspace.data_ptr() % 32 + offset
        workspace[at + size :] = 77
        a.workspace, a.workspace_bytes = workspace.data_ptr() + at, size
        capi.paged_attention(a, torch.cuda.current_stream().cuda_stream)
        assert (workspace[at + size :] == 77).all()
    assert torch.equal(*outs)
    expected, size = attention(q, kc, vc, tables, starts, lens, 128**-0.5)
    assert ((outs[0].double() - expected).abs() <= attention_bound(expected, size)).all()


def check_not_finite(inputs, new, total):
    """As the formula in 64 bits, NaN and infinities included."""
    got, scale = call(inputs, new, total)
    expected, size = attention(*inputs, scale)
    finite = expected.isfinite()
    assert torch.equal(got.isnan(), expected.isnan())
    assert ((got.double() - expected).abs() <= attention_bound(expected, size))[finite].all()


EVERY_KERNEL = [
    # heads, kv_heads, dim, page: the vector path, then a warp a row for its head size and its page size
    (28, 4, 128, 16), (32, 8, 64, 32), (6, 3, 256, 16), (8, 2, 64, 24),
]


@gpu
@pytest.mark.parametrize("heads, kv_heads, dim, page", EVERY_KERNEL)
@pytest.mark.parametrize("new, total", [([1, 1], [70, 200]), ([1, 1], [1, 33]), ([1] * 40, [4000] * 40), ([150, 9], [190, 9])])
def test_nan_and_infinite_inputs_reach_the_rows_that_see_them(heads, kv_heads, dim, page, new, total):
    require_cuda()
    group = heads // kv_heads
    inputs = make(new, total, heads, kv_heads, dim, page)
    q, kc, vc, tables, starts, lens = inputs
    # One head of the last token.
    q[-1, 1, dim // 2] = float("nan")
    check_not_finite(inputs, new, total)
    q[-1, 1, dim // 2] = 0.5
    # Every visible key of a first block of 32, of one head of the first sequence.
    for bad in (float("nan"), float("inf"), float("-inf")):
        kept = [kc[int(tables[0, t // page]), t % page, 1].clone() for t in range(min(32, total[0]))]
        for t in range(len(kept)):
            kc[int(tables[0, t // page]), t % page, 1, 3] = bad
        if bad == bad and total[0] <= 32:  # its one score may be -inf, of which the formula has no value
            q[0, group : 2 * group, 3] = 1.0 if bad > 0 else -1.0
        check_not_finite(inputs, new, total)
        for t, row in enumerate(kept):
            kc[int(tables[0, t // page]), t % page, 1] = row
    assert capi.device_fault_flags(0) == 0


@gpu
@pytest.mark.parametrize("dim", [64, 128])
def test_an_infinite_score_anywhere_in_a_step_gives_nan(dim):
    """Each key of a block of 32 that every row sees, in pairs of tiles that one CTA has whole (1200 of them)."""
    require_cuda()
    new, total = [60] * 150, [500] * 150
    inputs = make(new, total, 16, 8, dim)
    q, kc, _, tables = inputs[:4]
    q.abs_()
    for key in range(256, 288):
        pages, row = tables[:, key // 16].long(), key % 16
        kept = kc[pages, row]
        kc[pages, row, 1::2, 0] = float("inf")
        got, _ = call(inputs, new, total)
        wide = got.view(-1, 8, 2, dim)
        assert wide[:, 1::2].isnan().all(), key
        assert wide[:, 0::2].isfinite().all()
        kc[pages, row] = kept


@gpu
@pytest.mark.parametrize("heads, kv_heads, dim, page", EVERY_KERNEL)
def test_scores_of_minus_infinity_alone_give_zero(heads, kv_heads, dim, page):
    """As no score at all: such keys are as good as masked."""
    require_cuda()
    for new, total in (([1, 1], [70, 1]), ([1] * 40, [4000] * 40), ([150], [700]), ([60] * 150, [500] * 150)):
        q, kc, vc, tables, starts, lens = make(new, total, heads, kv_heads, dim, page)
        q.abs_()
        kc[..., 0] = float("-inf")
        got, _ = call((q, kc, vc, tables, starts, lens), new, total)
        assert (got == 0).all(), (new, total)


@gpu
@pytest.mark.parametrize("heads, kv_heads, dim", [(28, 4, 128), (11, 1, 64), (40, 8, 80), (127, 1, 128)])
def test_warps_whose_rows_differ(heads, kv_heads, dim):
    """Warps of the tile kernel with padding, tokens past the chunk's end and maxima that move in some rows only, over
    first steps that a window cuts: each of them parts a warp ahead of work that all of it does together."""
    require_cuda()
    for new, total, window in (([70], [1500], 600), ([301, 33] * 20, [301, 700] * 20, 190)):
        inputs = make(new, total, heads, kv_heads, dim)
        q = inputs[0]
        q[::3] *= 6.0  # scores of these rows spread over many times 2^8
        check(inputs, new, total, window)


def test_plans_of_bounds_without_limit():
    """Bounds past the tokens there are, and a window past the keys, plan as the ones that fit."""
    plan = lambda **changes: capi.paged_attention_plan(attention_args(**changes))  # noqa: E731
    chunk = dict(num_tokens=2048, num_seqs=1, max_query_len=2048, max_seq_len=16384, table_width=1024)
    few = dict(num_tokens=4, num_seqs=1, max_query_len=4)
    batch = dict(num_tokens=64, num_seqs=64, max_seq_len=8192)
    for call in (chunk, few, batch, {}):
        for most in (dict(window=2**63 - 1), dict(window=2**62), dict(window=2**31)):
            assert plan(**call, **most) == plan(**call)
            assert capi.paged_attention_workspace(attention_args(**call, **most)) == capi.paged_attention_workspace(attention_args(**call))
    for call in (chunk, few):
        for most in (2**63 - 1, 2**62, 2**33):
            assert plan(**{**call, "max_query_len": most}) == plan(**call)
            assert plan(**{**call, "max_query_len": most, "window": 2**63 - 1}) == plan(**call)


@gpu
def test_more_rows_of_a_group_than_31_bits_count():
    """2^24 + 1 tokens of 128 heads that share a key head: 2^31 + 128 rows, all but the last 100 tokens before
    position 0. The query's rows overlap, so that it takes little memory."""
    require_cuda()
    tokens = 2**24 + 1
    small, kc, vc, tables, starts, lens = make([100], [100], 128, 1, 8)
    flat = torch.randn(8 * (tokens + 127), device="cuda").to(torch.bfloat16)
    q = flat.as_strided((tokens, 128, 8), (8, 8, 1))
    starts[1] = tokens
    out = torch.full((tokens, 128, 8), 7.0, dtype=torch.bfloat16, device="cuda")
    extension.load_extension()
    torch.ops.inference_performance_lab.paged_attention(out, q, kc, vc, tables, starts, lens, tokens, 100, 0.35, 0)
    assert all(bool((part == 0).all()) for part in out[:-100].split(2**20))
    expected, size = attention(q[-100:], kc, vc, tables, torch.tensor([0, 100]), lens, 0.35)
    assert ((out[-100:].double() - expected).abs() <= attention_bound(expected, size)).all()
    assert capi.device_fault_flags(0) == 0
    del out
    torch.cuda.empty_cache()


def test_plan_of_more_rows_than_31_bits_count():
    """Without the tile kernel (broadcast keys), the rows of a group are counted by the kernel of a warp a row."""
    changes = dict(num_tokens=2**24 + 1, num_seqs=1, num_heads=128, num_kv_heads=1, head_size=8, max_query_len=2**24 + 1,
                   max_seq_len=100, key_cache_token_stride=0)
    assert capi.paged_attention_plan(attention_args(**changes)) == "attention_row_kernel"
    assert capi.paged_attention_plan(attention_args(**{**changes, "num_tokens": 2**24 - 1024})) == "attention_short_kernel<2>"


def test_plan_of_more_blocks_than_31_bits_count():
    """Equal shares are cut from a sum of all blocks of 16 keys; where the tables could hold 2^31 of them, clusters."""
    batch = dict(num_tokens=64, num_seqs=64, max_seq_len=8192)
    shares = "attention_shared_kernel<1> + attention_join_parts_kernel"
    assert capi.paged_attention_plan(attention_args(**batch, table_width=2**20)) == shares
    assert capi.paged_attention_plan(attention_args(**batch, table_width=2**25)) == "attention_short_kernel<1>"
    assert capi.paged_attention_plan(attention_args(**batch, table_width=2**31 - 1, page_size=2**20)) == "attention_short_kernel<1>"
    assert capi.paged_attention_workspace(attention_args(**batch, table_width=2**25)) == 0


@gpu
@pytest.mark.parametrize("heads, kv_heads, dim, new", [(28, 4, 128, 1), (28, 4, 128, 300), (32, 8, 64, 3), (6, 3, 256, 2)])
def test_lengths_at_the_end_of_32_bits(heads, kv_heads, dim, new):
    """A window at the end of the longest sequence there can be, and of a longer one, whose keys past it are left out.
    All of its pages are the same few."""
    require_cuda()
    capi.clear_device_fault_flags(0)
    page, window, pages = 16, 500, 48
    q, kc, vc, _, starts, _ = make([new], [pages * page], heads, kv_heads, dim, spare=0)
    width = 2**31 // page
    tables = (torch.arange(width, device="cuda", dtype=torch.int32) % pages)[None]
    for total in (2**31 - 256, 2**31 - 1):
        lens = torch.tensor([total], dtype=torch.int32, device="cuda")
        got = extension.paged_attention(q, kc, vc, tables, starts, lens, new, 2**30 - 1, dim**-0.5, window)
        assert capi.device_fault_flags(0) == (0 if total == 2**31 - 256 else 8)
        capi.clear_device_fault_flags(0)
        # The formula over the last 2048 places, those past the limit left out.
        place = torch.arange(2**31 - 2048, min(total, 2**31 - 256), device="cuda", dtype=torch.int64)
        keys, values = (c[(place // page % pages), place % page].double() for c in (kc, vc))
        position = total - new + torch.arange(new, device="cuda", dtype=torch.int64)
        seen = (place[None] <= position[:, None]) & (place[None] > position[:, None] - window)
        for h in range(heads):
            g = h // (heads // kv_heads)
            logits = (q[:, h].double() @ keys[:, g].T * dim**-0.5).masked_fill(~seen, -torch.inf)
            w = torch.softmax(logits, -1)
            want, size = w @ values[:, g], w @ values[:, g].abs()
            assert ((got[:, h].double() - want).abs() <= attention_bound(want, size)).all()

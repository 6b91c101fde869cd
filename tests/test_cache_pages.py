"""Pages of a KV cache: reserving, forking, releasing, copying and compacting against plain Python
bookkeeping and the pages' own bytes; pools without room, invalid entries, refusals."""

from __future__ import annotations

import random

import pytest
import torch

from cache_reference import Pool
from inference_performance_lab.kernels import capi, extension
from parity import require_cuda

gpu = pytest.mark.gpu


class Device:
    """A pool on the device beside the plain one."""

    def __init__(self, rows, width, pages, page_size, layers=2, kv_heads=2, dim=8, seed=0, hnd=False, dtype=torch.bfloat16):
        self.page = page_size
        g = torch.Generator(device="cuda").manual_seed(seed)
        shape = (2 * layers, pages, kv_heads, page_size, dim) if hnd else (2 * layers, pages, page_size, kv_heads, dim)
        self.store = torch.randint(0, 127, shape, generator=g, device="cuda").to(dtype)
        self.view = self.store.transpose(2, 3) if hnd else self.store
        self.caches = list(self.view.unbind(0))
        self.tables = torch.full((rows, width), -1, dtype=torch.int32, device="cuda")
        self.lens = torch.zeros(rows, dtype=torch.int32, device="cuda")
        self.refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
        self.pool = Pool(self.tables.tolist(), self.lens.tolist(), self.refs.tolist(), page_size)

    def ints(self, values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    def same(self):
        assert self.tables.tolist() == self.pool.tables
        assert self.lens.tolist() == self.pool.lens
        assert self.refs.tolist() == self.pool.refs
        assert capi.device_fault_flags(0) == 0

    def reserve(self, rows, lens):
        status = extension.reserve_pages(self.tables, self.lens, self.refs, self.ints(rows), self.ints(lens), self.page)
        assert status.tolist() == [self.pool.reserve(rows, lens)]
        self.same()

    def release(self, rows):
        extension.release_sequences(self.tables, self.lens, self.refs, self.ints(rows))
        self.pool.release(rows)
        self.same()

    def fork(self, parents, children):
        before = self.view.clone()
        status = extension.fork_sequences(self.caches, self.tables, self.lens, self.refs, self.ints(parents), self.ints(children))
        lacking, copies = self.pool.fork(parents, children)
        assert status.tolist() == [lacking]
        self.same()
        for source, target in copies:
            assert torch.equal(self.view[:, target], before[:, source])
        kept = torch.ones(before.shape[1], dtype=torch.bool, device="cuda")
        kept[[c[1] for c in copies]] = False
        assert torch.equal(self.view[:, kept], before[:, kept])

    def compact(self):
        before = self.view.clone()
        old = self.tables.clone(), self.refs.clone()
        tables, refs, live = extension.compact_pages(self.caches, self.tables, self.refs)
        want_tables, want_refs, want_live, moves = self.pool.compact()
        assert tables.tolist() == want_tables and refs.tolist() == want_refs and live.tolist() == [want_live]
        assert torch.equal(self.tables, old[0]) and torch.equal(self.refs, old[1])
        for source, target in moves:
            before[:, target] = before[:, source]
        assert torch.equal(self.view, before)
        self.tables, self.refs = tables, refs
        self.pool.tables, self.pool.refs = want_tables, want_refs
        self.same()


@gpu
@pytest.mark.parametrize("page_size, pages, rows, hnd, dim", [(16, 200, 12, False, 8), (1, 90, 9, False, 8), (48, 64, 20, True, 16),
                                                              (7, 3000, 40, False, 24), (16, 40, 10, True, 8)])
def test_random_traffic(page_size, pages, rows, hnd, dim):
    """A random mix of every call; the pool often has no room."""
    require_cuda()
    d = Device(rows, 40, pages, page_size, dim=dim, hnd=hnd, seed=page_size)
    rng = random.Random(page_size)
    for _ in range(60):
        kind = rng.choice(["reserve", "reserve", "fork", "release", "compact"])
        some = rng.sample(range(rows), rng.randint(0, rows // 2))
        if kind == "reserve":
            d.reserve(some, [rng.randint(0, 40 * page_size) if rng.random() < 0.3 else min(40 * page_size, d.pool.lens[r] + rng.randint(0, 30))
                             for r in some])
        elif kind == "release":
            d.release(some)
        elif kind == "fork":
            empty = [r for r in range(rows) if d.pool.lens[r] == 0 and not any(p >= 0 for p in d.pool.tables[r])]
            children = rng.sample(empty, rng.randint(0, len(empty)))
            held = [r for r in range(rows) if r not in children] or [0]
            d.fork([rng.choice(held) for _ in children], children)
        else:
            d.compact()


@gpu
def test_more_rows_and_pages_than_threads():
    require_cuda()
    d = Device(3000, 3, 5000, 4, layers=1, kv_heads=1)
    d.reserve(list(range(0, 2500)), [(i * 7) % 9 for i in range(2500)])
    d.release(list(range(0, 2500, 3)))
    parents = [i for i in range(1, 1500, 3)]
    d.fork(parents, list(range(2500, 2500 + len(parents))))
    d.compact()
    d.reserve(list(range(2999, -1, -1)), [12] * 3000)  # lacks pages: nothing changes


@gpu
def test_as_many_rows_as_a_call_takes():
    require_cuda()
    d = Device(16384, 2, 20000, 4, layers=1, kv_heads=1, dim=4)
    d.reserve(list(range(16384)), [i % 8 for i in range(16384)])
    with pytest.raises(RuntimeError, match="at most 16384"):
        extension.reserve_pages(d.tables, d.lens, d.refs, d.ints([0] * 16385), d.ints([1] * 16385), 4)


@gpu
def test_many_caches_take_several_launches():
    require_cuda()
    d = Device(4, 4, 12, 8, layers=70)
    d.reserve([0], [19])
    d.fork([0, 0], [1, 3])
    d.release([0])
    d.compact()


@gpu
def test_invalid_entries_change_nothing():
    require_cuda()
    d = Device(6, 4, 30, 16)
    d.reserve([0, 1], [20, 40])
    for rows, lens in (([6], [1]), ([-1], [1]), ([2], [65]), ([2], [-1]), ([3, 2, 3], [1, 1, 1])):
        status = extension.reserve_pages(d.tables, d.lens, d.refs, d.ints(rows), d.ints(lens), 16)
        assert status.tolist() == [-1]
        d.same()
    for parents, children in (([0], [6]), ([7], [2]), ([0], [1]), ([0, 1], [2, 2]), ([-1], [2])):
        status = extension.fork_sequences(d.caches, d.tables, d.lens, d.refs, d.ints(parents), d.ints(children))
        assert status.tolist() == [-1]
        d.same()
    d.fork([0, 3], [3, 4])  # a parent that is itself an empty child


@gpu
def test_a_row_released_twice_and_out_of_range():
    require_cuda()
    capi.clear_device_fault_flags(0)
    d = Device(4, 8, 20, 4)
    d.reserve([0, 1], [9, 30])
    extension.release_sequences(d.tables, d.lens, d.refs, d.ints([1, 1, 1]))
    d.pool.release([1])
    d.same()
    extension.release_sequences(d.tables, d.lens, d.refs, d.ints([4, -1]))
    assert capi.device_fault_flags(0) == 8
    capi.clear_device_fault_flags(0)
    d.same()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float8_e4m3fn, torch.float32])
def test_copy_pages(dtype):
    require_cuda()
    store = torch.arange(3 * 20 * 16 * 2 * 16, device="cuda").remainder(97).float().to(dtype).view(3, 20, 16, 2, 16)
    expected = store.clone()
    pairs = [(0, 5), (0, 7), (-1, 3), (4, -1), (19, 2)]
    extension.copy_pages(list(store.unbind(0)), torch.tensor(pairs, dtype=torch.int32, device="cuda"))
    for source, target in pairs:
        if min(source, target) >= 0:
            expected.view(torch.uint8)[:, target] = expected.view(torch.uint8)[:, source]
    assert torch.equal(store.view(torch.uint8), expected.view(torch.uint8))
    assert capi.device_fault_flags(0) == 0
    extension.copy_pages(list(store.unbind(0)), torch.tensor([(0, 20), (2**30, 0)], dtype=torch.int32, device="cuda"))
    assert capi.device_fault_flags(0) == 8
    capi.clear_device_fault_flags(0)
    assert torch.equal(store.view(torch.uint8), expected.view(torch.uint8))
    extension.copy_pages(list(store.unbind(0)), torch.empty(0, 2, dtype=torch.int32, device="cuda"))


@gpu
@pytest.mark.parametrize("dim", [8, 24, 1000])
def test_copy_pages_off_32_bytes(dim):
    """Pages whose size or base is a multiple of 16 bytes but not of 32; nothing beside them is written."""
    require_cuda()
    flat = torch.randint(0, 127, (2 * 9 * dim + 64,), device="cuda", dtype=torch.int32).to(torch.bfloat16)
    store = flat[8 : 8 + 2 * 9 * dim].view(2, 9, 1, dim)
    before = flat.clone()
    extension.copy_pages(list(store.unbind(0)), torch.tensor([[0, 3], [1, 8]], dtype=torch.int32, device="cuda"))
    expected = before[8 : 8 + 2 * 9 * dim].view(2, 9, 1, dim)
    expected[:, 3], expected[:, 8] = expected[:, 0], expected[:, 1]
    assert torch.equal(flat, before)


@gpu
def test_interleaved_caches_and_long_offsets():
    """Layers interleaved page by page in one buffer of more than 2^32 bytes."""
    require_cuda()
    pages, layers = 66000, 4
    store = torch.empty(pages, layers, 16, 2, 256, dtype=torch.bfloat16, device="cuda")
    store[-3:].copy_(torch.randn_like(store[-3:]))
    expected = store[-1].clone()
    extension.copy_pages(list(store.unbind(1)), torch.tensor([[pages - 1, 1], [pages - 1, pages - 3]], dtype=torch.int32, device="cuda"))
    assert torch.equal(store[1], expected) and torch.equal(store[-3], expected)


@gpu
def test_graph_replay():
    require_cuda()
    d = Device(8, 8, 40, 4)
    d.reserve([0, 1], [9, 14])
    parents, children = d.ints([0, 1]), d.ints([2, 3])
    extension.fork_sequences(d.caches, d.tables, d.lens, d.refs, parents, children)
    extension.release_sequences(d.tables, d.lens, d.refs, children)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        extension.release_sequences(d.tables, d.lens, d.refs, children)
        status = extension.fork_sequences(d.caches, d.tables, d.lens, d.refs, parents, children)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert status.tolist() == [0]
        d.pool.release([2, 3])
        d.pool.fork([0, 1], [2, 3])
        d.same()


@gpu
def test_c_abi():
    """The same calls through the C ABI, on raw pointers."""
    require_cuda()
    d = Device(4, 8, 20, 4)
    stream = torch.cuda.current_stream().cuda_stream
    state = capi.PagePool(d.tables.data_ptr(), d.lens.data_ptr(), d.refs.data_ptr(), 4, 8, 8, 20, 4)
    bytes_per_page = d.caches[0][0].numel() * 2
    store = capi.page_caches([c.data_ptr() for c in d.caches], bytes_per_page, bytes_per_page)
    status, live = d.ints([7]), d.ints([0])
    rows, lens, parents, children = d.ints([0, 2]), d.ints([9, 30]), d.ints([2]), d.ints([1])
    capi.reserve_pages(state, rows.data_ptr(), lens.data_ptr(), 2, status.data_ptr(), stream)
    assert status.tolist() == [d.pool.reserve([0, 2], [9, 30])]
    before = d.view.clone()
    capi.fork_sequences(store, state, parents.data_ptr(), children.data_ptr(), 1, status.data_ptr(), stream)
    lacking, copies = d.pool.fork([2], [1])
    assert status.tolist() == [lacking] and len(copies) == 1
    assert torch.equal(d.view[:, copies[0][1]], before[:, copies[0][0]])
    d.same()
    capi.release_sequences(state, rows.data_ptr(), 1, stream)
    d.pool.release([0])
    d.same()
    tables, refs = torch.empty_like(d.tables), torch.empty_like(d.refs)
    size = capi.compact_pages_workspace(20)
    workspace = torch.empty(size, dtype=torch.uint8, device="cuda")
    capi.compact_pages(store, state, tables.data_ptr(), refs.data_ptr(), live.data_ptr(), workspace.data_ptr(), size, stream)
    want_tables, want_refs, want_live, _ = d.pool.compact()
    assert tables.tolist() == want_tables and refs.tolist() == want_refs and live.tolist() == [want_live]
    pairs = d.ints([[0, 15]])
    capi.copy_pages(store, 20, pairs.data_ptr(), 1, stream)
    assert torch.equal(d.view[:, 15], d.view[:, 0])


@gpu
def test_refusals():
    require_cuda()
    d = Device(4, 8, 20, 4)
    rows = d.ints([0])
    with pytest.raises(RuntimeError, match="rows and new_lens must have the same length"):
        extension.reserve_pages(d.tables, d.lens, d.refs, rows, d.ints([1, 2]), 4)
    with pytest.raises(RuntimeError, match="page size positive"):
        extension.reserve_pages(d.tables, d.lens, d.refs, rows, rows, 0)
    with pytest.raises(RuntimeError, match="block_tables must be int32"):
        extension.release_sequences(d.tables.long(), d.lens, d.refs, rows)
    with pytest.raises(RuntimeError, match="a length for each row"):
        extension.release_sequences(d.tables, d.lens[:3], d.refs, rows)
    with pytest.raises(RuntimeError, match="same device"):
        extension.release_sequences(d.tables, d.lens, d.refs, rows.cpu())
    with pytest.raises(RuntimeError, match="a count for each page"):
        extension.fork_sequences(d.caches, d.tables, d.lens, d.refs[:19], rows, rows)
    with pytest.raises(RuntimeError, match="same type, shape and strides"):
        extension.fork_sequences([d.caches[0], d.caches[1].float()], d.tables, d.lens, d.refs, rows, rows)
    with pytest.raises(RuntimeError, match="must not be empty"):
        extension.compact_pages([], d.tables, d.refs)
    with pytest.raises(RuntimeError, match="must be contiguous, tokens or heads"):
        extension.copy_pages([d.caches[0][..., :4]], d.ints([[0, 1]]))
    with pytest.raises(RuntimeError, match="16-byte"):
        extension.copy_pages([torch.zeros(4, 1, 3, device="cuda")], d.ints([[0, 1]]))
    with pytest.raises(RuntimeError, match="pairs must be contiguous int32"):
        extension.copy_pages(d.caches, d.ints([0, 1]))


BASE = 0x7F0000000000


def pool(**changes):
    a = dict(block_tables=BASE, seq_lens=BASE, ref_counts=BASE, num_rows=4, width=8, table_stride=8, num_pages=20, page_size=16)
    a.update(changes)
    return capi.PagePool(**a)


def caches(stride=4096, size=4096, bases=(BASE, BASE + 4096)):
    return capi.page_caches(list(bases), stride, size)


@pytest.mark.parametrize("call, status, message", [
    (lambda: capi.reserve_pages(pool(num_rows=-1), BASE, BASE, 1, BASE), capi.IPL_ERROR_INVALID_VALUE, "non-negative"),
    (lambda: capi.reserve_pages(pool(num_pages=2**31), BASE, BASE, 1, BASE), capi.IPL_ERROR_TOO_LARGE, "too large"),
    (lambda: capi.reserve_pages(pool(), 0, BASE, 1, BASE), capi.IPL_ERROR_INVALID_VALUE, "non-null"),
    (lambda: capi.reserve_pages(pool(), BASE, BASE, 16385, BASE), capi.IPL_ERROR_TOO_LARGE, "at most 16384"),
    (lambda: capi.compact_pages(caches(), pool(), BASE + 64, BASE + 128, BASE, BASE, 16), capi.IPL_ERROR_INVALID_VALUE,
     "workspace is too small"),
    (lambda: capi.reserve_pages(pool(), BASE, BASE, 1, 0), capi.IPL_ERROR_INVALID_VALUE, "status must be non-null"),
    (lambda: capi.release_sequences(pool(ref_counts=0), BASE, 1), capi.IPL_ERROR_INVALID_VALUE, "non-null"),
    (lambda: capi.release_sequences(pool(seq_lens=BASE + 2), BASE, 1), capi.IPL_ERROR_INVALID_VALUE, "4-byte aligned"),
    (lambda: capi.copy_pages(caches(stride=2048), 20, BASE, 1), capi.IPL_ERROR_INVALID_VALUE, "must not overlap"),
    (lambda: capi.copy_pages(caches(size=4088), 20, BASE, 1), capi.IPL_ERROR_MISALIGNED, "16"),
    (lambda: capi.copy_pages(caches(bases=(BASE + 8,)), 20, BASE, 1), capi.IPL_ERROR_MISALIGNED, "16"),
    (lambda: capi.fork_sequences(caches(), pool(), BASE, 0, 1, BASE), capi.IPL_ERROR_INVALID_VALUE, "non-null"),
    (lambda: capi.compact_pages(caches(), pool(), BASE, BASE + 64, BASE, BASE, 1 << 20), capi.IPL_ERROR_INVALID_VALUE, "must not alias"),
])
def test_argument_errors(call, status, message):
    with pytest.raises(capi.IplError, match=message) as info:
        call()
    assert info.value.status == status


def test_workspace_and_empty_calls():
    assert capi.compact_pages_workspace(100) >= 4 * 300
    capi.copy_pages(caches(), 20, 0, 0)
    capi.release_sequences(pool(), 0, 0)


@gpu
@pytest.mark.parametrize("rows, width", [(1024, 2**21), (1024, 2**21 + 8), (16384, 140000)])
def test_needs_past_31_bits_change_nothing(rows, width):
    """A round of 1024 rows, or the rounds before one, that lack 2^31 pages and more (a little less in the first case).
    The rows of the tables are one row shown many times, which a call that changes nothing does not write."""
    require_cuda()
    table = torch.full((width,), -1, dtype=torch.int32, device="cuda")
    lens = torch.arange(rows, dtype=torch.int32, device="cuda") % 7
    refs = torch.zeros(100, dtype=torch.int32, device="cuda")
    index = torch.arange(rows, dtype=torch.int32, device="cuda")
    expected = lens.clone()
    status = extension.reserve_pages(table.expand(rows, -1), lens, refs, index, torch.full_like(index, width), 1)
    lacking = min(rows * width - int(expected.sum()), 2**31 - 1) - 100
    assert status.tolist() == [lacking]
    assert torch.equal(lens, expected) and not refs.any() and (table == -1).all()

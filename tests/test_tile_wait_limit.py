"""A bounded wait of the attention tile kernel that runs out: the kernel returns, records the fault and
leaves the CUDA context usable.

Runs the test-only build of the library (see test_staged_wait_limit.py): every wait limited to 1 ms, and
CTA 0 never issues its second load of keys. Its issuer, softmax warps, loaders and scheduler all wait on
what follows from that load; whichever gives up first records its bit, the others leave on the abort
flag, tensor memory is freed and no copy is left in flight. Every other CTA runs normally.
"""

from __future__ import annotations

import ctypes

import pytest
import torch

from cache_reference import attention, attention_bound
from inference_performance_lab.kernels import capi
from parity import require_cuda
from test_paged_attention import make
from test_staged_wait_limit import FAULT_EMPTY_BARRIER_TIMEOUT, FAULT_FULL_BARRIER_TIMEOUT, _flags, _library

pytestmark = pytest.mark.gpu


def call(lib, inputs, scale):
    q, kc, vc, tables, starts, lens = inputs
    out = torch.full_like(q, 7.0)
    a = capi.PagedAttentionArgs(
        output=out.data_ptr(), query=q.data_ptr(), key_cache=kc.data_ptr(), value_cache=vc.data_ptr(),
        block_tables=tables.data_ptr(), query_start_loc=starts.data_ptr(), seq_lens=lens.data_ptr(), num_tokens=q.shape[0],
        num_seqs=lens.numel(), num_heads=q.shape[1], num_kv_heads=kc.shape[2], head_size=q.shape[2], num_pages=kc.shape[0],
        page_size=kc.shape[1], table_width=tables.shape[1], table_stride=tables.stride(0), output_token_stride=out.stride(0),
        output_head_stride=out.stride(1), query_token_stride=q.stride(0), query_head_stride=q.stride(1),
        key_cache_page_stride=kc.stride(0), key_cache_token_stride=kc.stride(1), key_cache_head_stride=kc.stride(2),
        value_cache_page_stride=vc.stride(0), value_cache_token_stride=vc.stride(1), value_cache_head_stride=vc.stride(2),
        max_query_len=q.shape[0], max_seq_len=int(lens.max()), window=0, scale=scale)
    assert lib.ipl_paged_attention_plan(ctypes.byref(a)) == b"attention_tile_kernel + attention_join_rows_kernel"
    size = ctypes.c_size_t(0)
    assert lib.ipl_paged_attention_workspace(ctypes.byref(a), ctypes.byref(size)) == 0
    workspace = torch.zeros(size.value, dtype=torch.uint8, device="cuda")
    a.workspace, a.workspace_bytes = workspace.data_ptr(), size.value
    assert lib.ipl_paged_attention_bf16(ctypes.byref(a), torch.cuda.current_stream().cuda_stream) == 0, lib.ipl_last_error()
    torch.cuda.synchronize()  # the kernel returned and the context is intact
    return out


@pytest.mark.parametrize("dim", [64, 128])
def test_tile_wait_runs_out_and_the_kernel_returns(dim: int) -> None:
    require_cuda()
    torch.cuda.set_device(0)
    lib = _library()
    inputs = make([1200], [2400], 28, 4, dim)
    assert lib.ipl_clear_device_fault_flags(0) == 0
    for _ in range(2):
        out = call(lib, inputs, 0.1)
        flags = _flags(lib)
        expected = FAULT_FULL_BARRIER_TIMEOUT | FAULT_EMPTY_BARRIER_TIMEOUT
        assert flags & expected and not flags & ~expected, f"fault word {flags:#x}"  # no copy was left in flight
        # CTA 0 has the first two pairs of tiles (36 tokens each) of key head 0.
        want, size = attention(*inputs, 0.1)
        right = (out.double() - want).abs() <= attention_bound(want, size)
        assert right[72:].all() and right[:, 7:].all()
        assert not right[:72, :7].all()
        assert lib.ipl_clear_device_fault_flags(0) == 0
        assert _flags(lib) == 0
    # The product library's own fault word was never touched by any of this.
    assert capi.device_fault_flags(0) == 0

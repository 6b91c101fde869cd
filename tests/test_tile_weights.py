"""Work of the attention tile kernel that weighs more than 2^31 steps, shared out among its CTAs.

Runs a test-only build of the library (``build.py --tests``) in which each pair of tiles weighs 2^24 steps more
than it has, so that a small call's sums are those of one of millions of tokens.
"""

from __future__ import annotations

import ctypes

import pytest
import torch

from cache_reference import attention, attention_bound
from inference_performance_lab.kernels import capi
from inference_performance_lab.kernels.extension import NATIVE_DIR
from parity import require_cuda
from test_paged_attention import make
from test_tile_wait_limit import call

WEIGHT_TEST_LIBRARY = NATIVE_DIR / "test" / "libipl_b200_weighttest.so"
PAIR_WEIGHT = 2**24


@pytest.mark.gpu
@pytest.mark.parametrize("tokens", [
    140 * 36,  # each thread of a CTA has a pair at most; 140 pairs of a key head weigh 2.3e9
    500 * 36 + 5,  # several, whose sum has to be found again; 8.4e9
])
def test_shares_of_more_than_31_bits(tokens):
    require_cuda()
    if not WEIGHT_TEST_LIBRARY.exists():
        pytest.fail(f"{WEIGHT_TEST_LIBRARY} is missing: run inference-performance-lab_b200/build.py --tests")
    assert tokens // 36 * PAIR_WEIGHT > 2**31
    lib = ctypes.CDLL(str(WEIGHT_TEST_LIBRARY))
    for name, (restype, argtypes) in capi.SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = restype
        fn.argtypes = argtypes
    inputs = make([tokens], [tokens], 28, 4, 64)
    out = call(lib, inputs, 0.1)
    q, kc, vc, tables, starts, lens = inputs
    # The formula for every 97th token: a sequence each, of the keys up to it.
    some = torch.arange(0, tokens, 97)
    want, size = attention(q[some], kc, vc, tables.expand(len(some), -1), torch.arange(len(some) + 1), some + 1, 0.1)
    assert ((out[some].double() - want).abs() <= attention_bound(want, size)).all()
    assert not (out == 7.0).all(-1).any()  # every row is written
    flags = ctypes.c_uint32(0)
    assert lib.ipl_device_fault_flags(0, ctypes.byref(flags)) == 0 and flags.value == 0

"""The compiled paged-cache kernels' register budgets, from the ptxas report the build writes.

The tile kernel's 384 threads fit an SM with up to 168 registers, the shared kernel's three CTAs of 128
threads an SM with up to 168 for 8 rows, the two of the others with up to 255. None of them spills
(test_build.py checks that for every kernel).
"""

from __future__ import annotations

import pytest

from test_build import kernel_resources


@pytest.mark.parametrize(
    "name, instances, cap",
    [
        ("21attention_tile_kernel", 2, 168),
        ("23attention_shared_kernelILi128ELi1E", 1, 168),
        ("23attention_shared_kernelILi64ELi1E", 1, 168),
        ("23attention_shared_kernelILi", 4, 255),
        ("22attention_short_kernel", 4, 255),
        ("13rotary_kernel", 8, 64),
        ("16page_fork_kernel", 1, 64),
    ],
)
def test_registers(name: str, instances: int, cap: int) -> None:
    found = {n: r for n, r in kernel_resources().items() if n.startswith("_ZN3ipl" + name)}
    assert len(found) == instances, sorted(found)
    for kernel, (registers, spills) in found.items():
        assert registers <= cap and spills == 0, (kernel, registers, spills)

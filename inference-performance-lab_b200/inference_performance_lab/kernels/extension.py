"""Op loader and Python wrappers.

Mirrors ``src/inference_performance_lab/kernels/extension.py`` of the reference (load_extension at
:12-35, wrappers at :38-71): same function names, arguments, in-place behaviour and errors; the ops
of the paged KV cache at the end have no counterpart there. The
difference is the loader: instead of JIT-compiling with ``torch.utils.cpp_extension.load`` into a
cache directory, it loads the in-tree library built by ``build.py`` (building it first if it is
missing or stale and nvcc is present). There is no fallback: if the native library cannot be
loaded, every op raises.
"""

from __future__ import annotations

import importlib.util
from functools import cache
from pathlib import Path

import torch

PACKAGE_DIR = Path(__file__).resolve().parents[1]
NATIVE_DIR = PACKAGE_DIR / "_native"
TORCH_OPS_LIBRARY = NATIVE_DIR / "inference_performance_lab_cuda.so"
C_ABI_LIBRARY = NATIVE_DIR / "libipl_b200.so"


def _build_module():
    spec = importlib.util.spec_from_file_location(
        "_ipl_build", PACKAGE_DIR.parent / "build.py"
    )
    module = importlib.util.module_from_spec(spec)
    assert spec.loader is not None
    spec.loader.exec_module(module)
    return module


def ensure_built(*, verbose: bool = False) -> None:
    """Build the native libraries in-tree if they are missing or older than their sources."""
    try:
        builder = _build_module()
    except FileNotFoundError:
        builder = None
    if builder is not None:
        import shutil

        if shutil.which("nvcc") or Path("/usr/local/cuda/bin/nvcc").exists():
            builder.build(verbose=verbose)
    if not TORCH_OPS_LIBRARY.exists() or not C_ABI_LIBRARY.exists():
        raise RuntimeError(
            f"native library missing: {TORCH_OPS_LIBRARY} (run inference-performance-lab_b200/build.py)"
        )


@cache
def load_extension(*, verbose: bool = False) -> None:
    """Load the op library and register ``torch.ops.inference_performance_lab.*``."""
    ensure_built(verbose=verbose)
    torch.ops.load_library(str(TORCH_OPS_LIBRARY))


def fused_add_rms_norm(
    x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, epsilon: float
) -> None:
    """In place: ``residual := x + residual``; ``x := rmsnorm(x + residual) * weight``."""
    load_extension()

    torch.ops.inference_performance_lab.fused_add_rms_norm(x, residual, weight, epsilon)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, epsilon: float) -> torch.Tensor:
    """``rmsnorm(x) * weight`` into a new tensor (no residual; not in the reference library)."""
    load_extension()

    output = torch.empty_like(x)
    torch.ops.inference_performance_lab.rms_norm(output, x, weight, epsilon)

    return output


def fused_add_rms_norm_static_fp8_quant(
    x: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor, scale: torch.Tensor, epsilon: float
) -> torch.Tensor:
    """``residual := x + residual`` in place; returns ``e4m3(rmsnorm(x + residual) * weight / scale)``
    (x is not modified; not in the reference library)."""
    load_extension()

    output = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=x.device)
    torch.ops.inference_performance_lab.fused_add_rms_norm_static_fp8_quant(
        output, x, residual, weight, scale, epsilon
    )

    return output


def silu_and_mul(x: torch.Tensor) -> torch.Tensor:
    """``silu(x[..., :I]) * x[..., I:]`` into a new ``[..., I]`` tensor (any width/alignment)."""
    load_extension()

    if x.ndim == 0 or x.shape[-1] % 2 != 0:
        raise ValueError("the final tensor dimension must be even")

    output_shape = x.shape[:-1] + (x.shape[-1] // 2,)
    output = torch.empty(output_shape, dtype=x.dtype, device=x.device)

    torch.ops.inference_performance_lab.silu_and_mul(output, x)

    return output


def silu_and_mul_packed(x: torch.Tensor) -> torch.Tensor:
    """Same result; keeps the reference's packed contract (I % 8 == 0, 16-byte aligned)."""
    load_extension()

    if x.ndim == 0 or x.shape[-1] % 2 != 0:
        raise ValueError("the final tensor dimension must be even")

    output_shape = x.shape[:-1] + (x.shape[-1] // 2,)
    output = torch.empty(output_shape, dtype=x.dtype, device=x.device)

    torch.ops.inference_performance_lab.silu_and_mul_packed(output, x)

    return output


# ---- paged KV cache (not in the reference library) -----------------------------------------------


@cache
def _op(name: str):
    """The op's overload, looked up once: in a decode step the calls' host time counts."""
    load_extension()

    return getattr(torch.ops.inference_performance_lab, name).default


def rotary_embedding(
    positions: torch.Tensor,
    query: torch.Tensor,
    key: torch.Tensor,
    cos_sin_cache: torch.Tensor,
    is_neox: bool = True,
) -> None:
    """In place: the first ``R`` elements of every head of ``query`` ``[T, heads, D]`` and ``key``
    ``[T, kv_heads, D]`` turned by the angles of ``positions`` (int64 ``[T]``).

    ``cos_sin_cache`` is float32 ``[positions, R]`` (:func:`rotary_cos_sin_cache`). Pairs are
    ``(x[i], x[i + R/2])`` with ``is_neox``, else ``(x[2i], x[2i+1])``. Any strides with a contiguous
    last dimension.
    """
    _op("rotary_embedding")(positions, query, key, cos_sin_cache, is_neox)


def rotary_embedding_cache(
    positions: torch.Tensor,
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    cos_sin_cache: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    is_neox: bool = True,
) -> None:
    """Rotates ``query`` in place and writes rotated ``key`` and ``value`` to their slots of the caches
    ``[pages, page_size, kv_heads, D]``: slot ``s`` (int64, negative: none) is row ``s % page_size`` of
    page ``s // page_size``. ``key`` itself stays as it is."""
    _op("rotary_embedding_cache")(
        positions, query, key, value, cos_sin_cache, key_cache, value_cache, slot_mapping, is_neox
    )


def paged_attention(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_tables: torch.Tensor,
    query_start_loc: torch.Tensor,
    seq_lens: torch.Tensor,
    max_query_len: int,
    max_seq_len: int,
    scale: float,
    window: int = 0,
) -> torch.Tensor:
    """Causal attention of new tokens over a paged cache, into a new ``[T, heads, D]`` tensor.

    Sequence ``s`` owns rows ``query_start_loc[s]:query_start_loc[s + 1]`` of ``query`` and has
    ``seq_lens[s]`` tokens in the cache, those included; its pages are ``block_tables[s]`` (all int32).
    ``max_query_len`` and ``max_seq_len`` bound the lengths; ``window`` > 0 limits each token to the last
    ``window`` keys. A token that sees no key gives 0, and so does one all of whose scores are -infinity;
    rows of no sequence are left unwritten. Head sizes that are multiples of 8 up to 128 over pages of a
    multiple of 16 tokens are the fast ones; others, up to 256, are slower than plain torch operations.
    """
    output = torch.empty_like(query, memory_format=torch.contiguous_format)
    _op("paged_attention")(
        output, query, key_cache, value_cache, block_tables, query_start_loc, seq_lens, max_query_len, max_seq_len,
        scale, window
    )

    return output


def copy_pages(caches: list[torch.Tensor], pairs: torch.Tensor) -> None:
    """Copies page ``pairs[i, 0]`` to page ``pairs[i, 1]`` (int32; negative: skipped) in every cache."""
    _op("copy_pages")(caches, pairs)


def reserve_pages(
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    ref_counts: torch.Tensor,
    rows: torch.Tensor,
    new_lens: torch.Tensor,
    page_size: int,
) -> torch.Tensor:
    """Gives ``rows[i]`` pages for ``new_lens[i]`` tokens, in place. Returns an int32 ``[1]`` status on
    the device: 0, the number of free pages lacking, or -1 for an entry out of range; unless it is 0
    nothing has changed. A length lowered by hand loses the pages past it once the row grows again."""
    return _op("reserve_pages")(
        block_tables, seq_lens, ref_counts, rows, new_lens, page_size
    )


def fork_sequences(
    caches: list[torch.Tensor],
    block_tables: torch.Tensor,
    seq_lens: torch.Tensor,
    ref_counts: torch.Tensor,
    parents: torch.Tensor,
    children: torch.Tensor,
) -> torch.Tensor:
    """Makes the empty row ``children[i]`` a copy of row ``parents[i]``, in place: whole pages are
    shared, a partly filled last page is copied in every cache. Returns a status as
    :func:`reserve_pages` does."""
    return _op("fork_sequences")(
        caches, block_tables, seq_lens, ref_counts, parents, children
    )


def release_sequences(
    block_tables: torch.Tensor, seq_lens: torch.Tensor, ref_counts: torch.Tensor, rows: torch.Tensor
) -> None:
    """Empties ``rows``, in place: each of their pages loses one reference."""
    _op("release_sequences")(block_tables, seq_lens, ref_counts, rows)


def compact_pages(
    caches: list[torch.Tensor], block_tables: torch.Tensor, ref_counts: torch.Tensor
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Moves the pages in use to the lowest numbers. Returns the renumbered tables and counts and the
    number of pages in use (int32 ``[1]``); the old tables stay valid until moved pages are claimed."""
    new_tables = torch.empty_like(block_tables, memory_format=torch.contiguous_format)
    new_counts = torch.empty_like(ref_counts)
    live = ref_counts.new_empty(1)
    _op("compact_pages")(caches, block_tables, ref_counts, new_tables, new_counts, live)

    return new_tables, new_counts, live

"""ctypes binding of the C ABI (``include/ipl_b200.h``, ``_native/libipl_b200.so``).

This is the binding a non-torch caller uses: raw device pointers, sizes and a ``cudaStream_t``.
Each wrapper raises ``RuntimeError`` with the library's message when the call fails, the same
error surface as the torch ops (which raise through STD_TORCH_CHECK).
"""

from __future__ import annotations

import ctypes
from functools import cache

from inference_performance_lab.kernels.extension import C_ABI_LIBRARY, ensure_built

IPL_SUCCESS = 0
IPL_ERROR_INVALID_VALUE = 1
IPL_ERROR_MISALIGNED = 2
IPL_ERROR_TOO_LARGE = 3
IPL_ERROR_CUDA = 4



def _fields(pointers: str = "", sizes: str = "") -> list[tuple[str, object]]:
    return [(n, ctypes.c_void_p) for n in pointers.split()] + [(n, ctypes.c_int64) for n in sizes.split()]


class RotaryArgs(ctypes.Structure):
    """``ipl_rotary_args``."""

    _fields_ = [
        *_fields(
            "positions cos_sin_cache query key",
            "num_tokens num_heads num_kv_heads head_size rotary_dim max_position query_token_stride query_head_stride"
            " key_token_stride key_head_stride",
        ),
        ("is_neox", ctypes.c_int),
        *_fields(
            "value key_cache value_cache slot_mapping",
            "value_token_stride value_head_stride num_pages page_size key_cache_page_stride key_cache_token_stride"
            " key_cache_head_stride value_cache_page_stride value_cache_token_stride value_cache_head_stride",
        ),
    ]


class PagedAttentionArgs(ctypes.Structure):
    """``ipl_paged_attention_args``."""

    _fields_ = [
        *_fields(
            "output query key_cache value_cache block_tables query_start_loc seq_lens",
            "num_tokens num_seqs num_heads num_kv_heads head_size num_pages page_size table_width table_stride"
            " output_token_stride output_head_stride query_token_stride query_head_stride key_cache_page_stride"
            " key_cache_token_stride key_cache_head_stride value_cache_page_stride value_cache_token_stride"
            " value_cache_head_stride max_query_len max_seq_len window",
        ),
        ("scale", ctypes.c_double),
        ("workspace", ctypes.c_void_p),
        ("workspace_bytes", ctypes.c_size_t),
    ]


class PagePool(ctypes.Structure):
    """``ipl_page_pool``."""

    _fields_ = _fields("block_tables seq_lens ref_counts", "num_rows width table_stride num_pages page_size")


class PageCaches(ctypes.Structure):
    """``ipl_page_caches``."""

    _fields_ = [
        ("caches", ctypes.POINTER(ctypes.c_void_p)),
        *_fields("", "num_caches page_stride_bytes page_bytes"),
    ]


# name -> (restype, argtypes): every symbol include/ipl_b200.h declares.
SIGNATURES: dict[str, tuple[object, list[object]]] = {
    "ipl_fused_add_rms_norm_bf16": (
        ctypes.c_int,
        [
            ctypes.c_void_p,
            ctypes.c_void_p,
            ctypes.c_void_p,
            ctypes.c_int64,
            ctypes.c_int64,
            ctypes.c_double,
            ctypes.c_void_p,
        ],
    ),
    "ipl_rms_norm_bf16": (
        ctypes.c_int,
        [
            ctypes.c_void_p,
            ctypes.c_void_p,
            ctypes.c_void_p,
            ctypes.c_int64,
            ctypes.c_int64,
            ctypes.c_double,
            ctypes.c_void_p,
        ],
    ),
    "ipl_fused_add_rms_norm_static_fp8_quant": (
        ctypes.c_int,
        [
            ctypes.c_void_p,
            ctypes.c_void_p,
            ctypes.c_void_p,
            ctypes.c_void_p,
            ctypes.c_void_p,
            ctypes.c_int64,
            ctypes.c_int64,
            ctypes.c_double,
            ctypes.c_void_p,
        ],
    ),
    "ipl_silu_and_mul_bf16": (
        ctypes.c_int,
        [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64, ctypes.c_void_p],
    ),
    "ipl_silu_and_mul_packed_bf16": (
        ctypes.c_int,
        [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64, ctypes.c_void_p],
    ),
    "ipl_rotary_embedding_bf16": (ctypes.c_int, [ctypes.POINTER(RotaryArgs), ctypes.c_void_p]),
    "ipl_rotary_embedding_cache_bf16": (ctypes.c_int, [ctypes.POINTER(RotaryArgs), ctypes.c_void_p]),
    "ipl_paged_attention_bf16": (ctypes.c_int, [ctypes.POINTER(PagedAttentionArgs), ctypes.c_void_p]),
    "ipl_paged_attention_workspace": (
        ctypes.c_int,
        [ctypes.POINTER(PagedAttentionArgs), ctypes.POINTER(ctypes.c_size_t)],
    ),
    "ipl_paged_attention_plan": (ctypes.c_char_p, [ctypes.POINTER(PagedAttentionArgs)]),
    "ipl_compact_pages_workspace": (ctypes.c_int, [ctypes.c_int64, ctypes.POINTER(ctypes.c_size_t)]),
    "ipl_copy_pages": (
        ctypes.c_int,
        [ctypes.POINTER(PageCaches), ctypes.c_int64, ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p],
    ),
    "ipl_reserve_pages": (
        ctypes.c_int,
        [
            ctypes.POINTER(PagePool),
            ctypes.c_void_p,
            ctypes.c_void_p,
            ctypes.c_int64,
            ctypes.c_void_p,
            ctypes.c_void_p,
        ],
    ),
    "ipl_fork_sequences": (
        ctypes.c_int,
        [
            ctypes.POINTER(PageCaches),
            ctypes.POINTER(PagePool),
            ctypes.c_void_p,
            ctypes.c_void_p,
            ctypes.c_int64,
            ctypes.c_void_p,
            ctypes.c_void_p,
        ],
    ),
    "ipl_release_sequences": (
        ctypes.c_int,
        [ctypes.POINTER(PagePool), ctypes.c_void_p, ctypes.c_int64, ctypes.c_void_p],
    ),
    "ipl_compact_pages": (
        ctypes.c_int,
        [
            ctypes.POINTER(PageCaches),
            ctypes.POINTER(PagePool),
            ctypes.c_void_p,
            ctypes.c_void_p,
            ctypes.c_void_p,
            ctypes.c_void_p,
            ctypes.c_size_t,
            ctypes.c_void_p,
        ],
    ),
    "ipl_last_error": (ctypes.c_char_p, []),
    "ipl_status_string": (ctypes.c_char_p, [ctypes.c_int]),
    "ipl_abi_version": (ctypes.c_int, []),
    "ipl_device_fault_flags": (ctypes.c_int, [ctypes.c_int, ctypes.POINTER(ctypes.c_uint32)]),
    "ipl_clear_device_fault_flags": (ctypes.c_int, [ctypes.c_int]),
    "ipl_fused_add_rms_norm_plan": (
        ctypes.c_char_p,
        [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64],
    ),
    "ipl_rms_norm_plan": (
        ctypes.c_char_p,
        [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64],
    ),
    "ipl_fused_add_rms_norm_static_fp8_quant_plan": (
        ctypes.c_char_p,
        [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64],
    ),
    "ipl_silu_and_mul_plan": (
        ctypes.c_char_p,
        [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_int64, ctypes.c_int64],
    ),
}


class IplError(RuntimeError):
    """A nonzero ipl_status; ``status`` holds the code."""

    def __init__(self, status: int, message: str) -> None:
        super().__init__(message)
        self.status = status


@cache
def library() -> ctypes.CDLL:
    """Load libipl_b200.so once and attach the prototypes."""
    ensure_built()
    lib = ctypes.CDLL(str(C_ABI_LIBRARY))
    for name, (restype, argtypes) in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.restype = restype
        fn.argtypes = argtypes
    return lib


def _check(status: int) -> None:
    if status != IPL_SUCCESS:
        raise IplError(status, library().ipl_last_error().decode())


def fused_add_rms_norm(
    x_ptr: int,
    residual_ptr: int,
    weight_ptr: int,
    rows: int,
    hidden_size: int,
    epsilon: float,
    stream: int = 0,
) -> None:
    _check(
        library().ipl_fused_add_rms_norm_bf16(
            x_ptr, residual_ptr, weight_ptr, rows, hidden_size, epsilon, stream
        )
    )


def rms_norm(
    output_ptr: int,
    input_ptr: int,
    weight_ptr: int,
    rows: int,
    hidden_size: int,
    epsilon: float,
    stream: int = 0,
) -> None:
    _check(
        library().ipl_rms_norm_bf16(output_ptr, input_ptr, weight_ptr, rows, hidden_size, epsilon, stream)
    )


def fused_add_rms_norm_static_fp8_quant(
    output_ptr: int,
    input_ptr: int,
    residual_ptr: int,
    weight_ptr: int,
    scale_ptr: int,
    rows: int,
    hidden_size: int,
    epsilon: float,
    stream: int = 0,
) -> None:
    _check(
        library().ipl_fused_add_rms_norm_static_fp8_quant(
            output_ptr, input_ptr, residual_ptr, weight_ptr, scale_ptr, rows, hidden_size, epsilon, stream
        )
    )


def silu_and_mul(
    output_ptr: int, input_ptr: int, rows: int, intermediate_size: int, stream: int = 0
) -> None:
    _check(library().ipl_silu_and_mul_bf16(output_ptr, input_ptr, rows, intermediate_size, stream))


def silu_and_mul_packed(
    output_ptr: int, input_ptr: int, rows: int, intermediate_size: int, stream: int = 0
) -> None:
    _check(
        library().ipl_silu_and_mul_packed_bf16(
            output_ptr, input_ptr, rows, intermediate_size, stream
        )
    )


def rotary_embedding(args: RotaryArgs, stream: int = 0) -> None:
    _check(library().ipl_rotary_embedding_bf16(ctypes.byref(args), stream))


def rotary_embedding_cache(args: RotaryArgs, stream: int = 0) -> None:
    _check(library().ipl_rotary_embedding_cache_bf16(ctypes.byref(args), stream))


def paged_attention(args: PagedAttentionArgs, stream: int = 0) -> None:
    _check(library().ipl_paged_attention_bf16(ctypes.byref(args), stream))


def paged_attention_workspace(args: PagedAttentionArgs) -> int:
    size = ctypes.c_size_t(0)
    _check(library().ipl_paged_attention_workspace(ctypes.byref(args), ctypes.byref(size)))
    return size.value


def paged_attention_plan(args: PagedAttentionArgs) -> str:
    return library().ipl_paged_attention_plan(ctypes.byref(args)).decode()


def compact_pages_workspace(num_pages: int) -> int:
    size = ctypes.c_size_t(0)
    _check(library().ipl_compact_pages_workspace(num_pages, ctypes.byref(size)))
    return size.value


def page_caches(bases: list[int], page_stride_bytes: int, page_bytes: int) -> PageCaches:
    """The caches of a call; keeps the host array of bases alive."""
    return PageCaches((ctypes.c_void_p * len(bases))(*bases), len(bases), page_stride_bytes, page_bytes)


def copy_pages(caches: PageCaches, num_pages: int, pairs_ptr: int, count: int, stream: int = 0) -> None:
    _check(library().ipl_copy_pages(ctypes.byref(caches), num_pages, pairs_ptr, count, stream))


def reserve_pages(
    pool: PagePool, rows_ptr: int, new_lens_ptr: int, count: int, status_ptr: int, stream: int = 0
) -> None:
    _check(library().ipl_reserve_pages(ctypes.byref(pool), rows_ptr, new_lens_ptr, count, status_ptr, stream))


def fork_sequences(
    caches: PageCaches,
    pool: PagePool,
    parents_ptr: int,
    children_ptr: int,
    count: int,
    status_ptr: int,
    stream: int = 0,
) -> None:
    _check(
        library().ipl_fork_sequences(
            ctypes.byref(caches), ctypes.byref(pool), parents_ptr, children_ptr, count, status_ptr, stream
        )
    )


def release_sequences(pool: PagePool, rows_ptr: int, count: int, stream: int = 0) -> None:
    _check(library().ipl_release_sequences(ctypes.byref(pool), rows_ptr, count, stream))


def compact_pages(
    caches: PageCaches,
    pool: PagePool,
    new_tables_ptr: int,
    new_ref_counts_ptr: int,
    live_ptr: int,
    workspace_ptr: int,
    workspace_bytes: int,
    stream: int = 0,
) -> None:
    _check(
        library().ipl_compact_pages(
            ctypes.byref(caches), ctypes.byref(pool), new_tables_ptr, new_ref_counts_ptr, live_ptr, workspace_ptr,
            workspace_bytes, stream
        )
    )


def device_fault_flags(device: int) -> int:
    flags = ctypes.c_uint32(0)
    _check(library().ipl_device_fault_flags(device, ctypes.byref(flags)))
    return flags.value


def clear_device_fault_flags(device: int) -> None:
    _check(library().ipl_clear_device_fault_flags(device))


def fused_add_rms_norm_plan(
    x_ptr: int, residual_ptr: int, weight_ptr: int, rows: int, hidden_size: int
) -> str:
    return library().ipl_fused_add_rms_norm_plan(
        x_ptr, residual_ptr, weight_ptr, rows, hidden_size
    ).decode()


def rms_norm_plan(output_ptr: int, input_ptr: int, weight_ptr: int, rows: int, hidden_size: int) -> str:
    return library().ipl_rms_norm_plan(output_ptr, input_ptr, weight_ptr, rows, hidden_size).decode()


def fused_add_rms_norm_static_fp8_quant_plan(
    output_ptr: int, input_ptr: int, residual_ptr: int, weight_ptr: int, rows: int, hidden_size: int
) -> str:
    return library().ipl_fused_add_rms_norm_static_fp8_quant_plan(
        output_ptr, input_ptr, residual_ptr, weight_ptr, rows, hidden_size
    ).decode()


def silu_and_mul_plan(output_ptr: int, input_ptr: int, rows: int, intermediate_size: int) -> str:
    return library().ipl_silu_and_mul_plan(output_ptr, input_ptr, rows, intermediate_size).decode()


# Tensor-level conveniences (torch tensors on the current CUDA device, current stream).


def _stream_handle() -> int:
    import torch

    return torch.cuda.current_stream().cuda_stream


def fused_add_rms_norm_tensors(x, residual, weight, epsilon: float) -> None:
    hidden = x.shape[-1]
    rows = x.numel() // hidden if hidden else 0
    fused_add_rms_norm(
        x.data_ptr(), residual.data_ptr(), weight.data_ptr(), rows, hidden, epsilon, _stream_handle()
    )


def rms_norm_tensors(output, input_, weight, epsilon: float) -> None:
    hidden = input_.shape[-1]
    rows = input_.numel() // hidden if hidden else 0
    rms_norm(
        output.data_ptr(), input_.data_ptr(), weight.data_ptr(), rows, hidden, epsilon, _stream_handle()
    )


def silu_and_mul_tensors(output, input_, packed: bool = False) -> None:
    inter = input_.shape[-1] // 2
    rows = output.numel() // inter if inter else 0
    fn = silu_and_mul_packed if packed else silu_and_mul
    fn(output.data_ptr(), input_.data_ptr(), rows, inter, _stream_handle())

"""A paged cache whose keys and values are held in 8 bits (csrc/cache8.cu): what it is, how records are written and read back.

A record (the key or the value of one head and position) is its codes in 8-bit floating point (e4m3) and one exponent e, the smallest in
[-40, 40] with max|x| <= 448 * 2^e; entry i stands for ``codes[i] * 2^e``.  :mod:`.shared` has the attention that reads such a cache.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from .basic import status_word
from .native import KernelError, check, entry, is_bf16, require_cuda, sm_count, stream_address


class Cache8(NamedTuple):
    """``codes`` [pages, 2, kv_heads, page, d] float8_e4m3fn (keys, then values) and ``exponents`` [pages, 2, kv_heads, page] int8."""
    codes: torch.Tensor
    exponents: torch.Tensor


def supported(head_dim: int) -> bool:
    return head_dim % 8 == 0 and 8 <= head_dim <= 256


def new_cache8(pages: int, kv_heads: int, page_size: int, head_dim: int, device="cuda") -> Cache8:
    """An empty cache: every record stands for zeros.  2 * kv_heads * (head_dim + 1) bytes a position."""
    if not supported(head_dim):
        raise KernelError(f"cache8: heads of {head_dim} entries (multiples of 8 up to 256 only)")
    codes = torch.zeros((pages, 2, kv_heads, page_size, head_dim), dtype=torch.uint8, device=device).view(torch.float8_e4m3fn)
    return Cache8(codes, torch.zeros((pages, 2, kv_heads, page_size), dtype=torch.int8, device=device))


def check_cache8(cache: Cache8, what: str) -> tuple[int, int, int, int]:
    """(pages, kv_heads, page_size, head_dim) of a cache that is laid out as the kernels read it."""
    codes, exponents = cache
    shape = codes.shape
    if (codes.dtype is not torch.float8_e4m3fn or exponents.dtype is not torch.int8 or len(shape) != 5 or shape[1] != 2 or exponents.shape != shape[:4]
            or not codes.is_contiguous() or not exponents.is_contiguous()):
        raise KernelError(f"{what}: an 8-bit cache is dense codes [pages, 2, kv_heads, page, d] in float8_e4m3fn and exponents [pages, 2, kv_heads, page] in int8")
    if not (codes.is_cuda and exponents.is_cuda):
        require_cuda(codes, exponents)
    return shape[0], shape[2], shape[3], shape[4]


def _check_places(block_table, token_row, positions, what: str) -> tuple[int, int]:
    tokens, width = positions.numel(), block_table.shape[-1]
    if (block_table.dtype is not torch.int32 or token_row.dtype is not torch.int32 or positions.dtype is not torch.int32 or block_table.dim() != 2 or token_row.numel() != tokens
            or not (block_table.is_contiguous() and token_row.is_contiguous() and positions.is_contiguous())):
        raise KernelError(f"{what}: a dense int32 block table [rows, blocks], and a row and a position (dense int32) for each token")
    if not (block_table.is_cuda and token_row.is_cuda and positions.is_cuda):
        require_cuda(block_table, token_row, positions)
    return tokens, width


def cache8_store(src: torch.Tensor, k_offset: int, v_offset: int, cache: Cache8, block_table: torch.Tensor, token_row: torch.Tensor, positions: torch.Tensor) -> None:
    """Quantise each token's keys and values (columns of ``src`` [tokens, width], bfloat16 or float32) and write them to their pages, as
    :func:`.basic.kv_store` writes them as they are.  A token without a page is left out and reported (``raise_on_status``)."""
    pages, kv_heads, page_size, head_dim = check_cache8(cache, "cache8_store")
    tokens, table_width = _check_places(block_table, token_row, positions, "cache8_store")
    width, shape = kv_heads * head_dim, src.shape
    if len(shape) != 2 or shape[0] != tokens or src.stride(1) != 1 or min(k_offset, v_offset) < 0 or max(k_offset, v_offset) + width > shape[1]:
        raise KernelError(f"cache8_store: a source [tokens, width] with unit inner stride that holds {width} columns of keys and of values at their offsets")
    if not src.is_cuda:
        require_cuda(src)
    check(entry("cache8", "hb_cache8_store", "pilllpppippiiiiiipp")(
        src.data_ptr(), is_bf16(src), src.stride(0), k_offset, v_offset, cache[0].data_ptr(), cache[1].data_ptr(), block_table.data_ptr(), table_width, token_row.data_ptr(),
        positions.data_ptr(), tokens, kv_heads, head_dim, page_size, pages, sm_count(src.device), status_word(src.device).data_ptr(), stream_address()), "cache8_store")


def cache8_load(cache: Cache8, block_table: torch.Tensor, token_row: torch.Tensor, positions: torch.Tensor, dtype: torch.dtype = torch.bfloat16,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """The keys and values of ``positions`` (of the table rows ``token_row``) as [tokens, 2, kv_heads, d] in ``dtype`` (bfloat16 holds them exactly).
    A token without a page reads as zeros and is reported (``raise_on_status``)."""
    pages, kv_heads, page_size, head_dim = check_cache8(cache, "cache8_load")
    tokens, table_width = _check_places(block_table, token_row, positions, "cache8_load")
    if out is None:
        out = torch.empty(tokens, 2, kv_heads, head_dim, dtype=dtype, device=cache[0].device)
    elif out.shape != (tokens, 2, kv_heads, head_dim) or out.dtype != dtype or not out.is_contiguous() or not out.is_cuda:
        raise KernelError(f"cache8_load: the output is a dense {dtype} tensor [tokens, 2, kv_heads, d]")
    check(entry("cache8", "hb_cache8_load", "pppipppiiiiiiipp")(
        cache[0].data_ptr(), cache[1].data_ptr(), block_table.data_ptr(), table_width, token_row.data_ptr(), positions.data_ptr(), out.data_ptr(), is_bf16(out), tokens, kv_heads,
        head_dim, page_size, pages, sm_count(out.device), status_word(out.device).data_ptr(), stream_address()), "cache8_load")
    return out

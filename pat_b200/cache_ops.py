"""Cache operations around decode attention in a serving loop: the KV-cache append right before it, the
same for a cache held in 4 bits, and copies of whole pages (a request that forks, a compaction).

``reshape_and_cache_flash`` has the signature of vLLM's op of the same name, which the
reference's serving backend calls through ``torch.ops._C_cache_ops``
(``plugin/vllm/attention/backends/prefix_attn.py:828-837``).  It runs this library's kernel on
PyTorch's current stream; there is no fallback.
"""
from __future__ import annotations

import array
import ctypes as C
import struct
from typing import Optional, Sequence, Union

import torch

from . import _native as N
from ._launch import Signatures, launch, strides_of, struct_tail

_DTYPES = {torch.float16: 0, torch.bfloat16: 1}


def reshape_and_cache_flash(key: torch.Tensor, value: torch.Tensor, key_cache: torch.Tensor,
                            value_cache: torch.Tensor, slot_mapping: torch.Tensor,
                            kv_cache_dtype: str = "auto", k_scale: Optional[torch.Tensor] = None,
                            v_scale: Optional[torch.Tensor] = None) -> None:
    """Writes ``key[i]`` / ``value[i]`` (``[num_tokens, kv_heads, head_dim]``) into the paged caches
    (``[pages, page_size, kv_heads, head_dim]``) at ``slot_mapping[i] = page * page_size + row``.
    Tokens with a negative slot are skipped.  ``kv_cache_dtype`` must be ``"auto"`` (caches in the
    dtype of the keys); the scales belong to vLLM's fp8 caches and are ignored."""
    if kv_cache_dtype != "auto":
        raise RuntimeError(f"kv_cache_dtype {kv_cache_dtype!r} is not supported (16-bit caches only)")
    for name, t in (("key", key), ("value", value), ("key_cache", key_cache), ("value_cache", value_cache),
                    ("slot_mapping", slot_mapping)):
        if not t.is_cuda:
            raise RuntimeError(f"{name} must be a CUDA tensor")
    if key.dtype not in _DTYPES or value.dtype != key.dtype or key_cache.dtype != key.dtype or \
            value_cache.dtype != key.dtype:
        raise RuntimeError("key, value and both caches must share one dtype, fp16 or bf16")
    if key.dim() != 3 or value.shape != key.shape:
        raise RuntimeError("key and value must be [num_tokens, kv_heads, head_dim]")
    if key_cache.dim() != 4 or value_cache.shape != key_cache.shape:
        raise RuntimeError("caches must be [pages, page_size, kv_heads, head_dim]")
    tokens, heads, dim = key.shape
    if key_cache.shape[2] != heads or key_cache.shape[3] != dim:
        raise RuntimeError("caches and keys disagree on kv_heads / head_dim")
    for name, t in (("key", key), ("value", value), ("key_cache", key_cache), ("value_cache", value_cache)):
        if t.stride(-1) != 1:
            raise RuntimeError(f"{name} must have a contiguous last dimension")
    slots = slot_mapping.flatten()
    if slots.dtype != torch.int64:
        slots = slots.to(torch.int64)
    slots = slots.contiguous()
    if slots.numel() < tokens:
        raise RuntimeError("slot_mapping is shorter than the number of tokens")
    a = N.AppendArgs()
    a.key, a.value = key.data_ptr(), value.data_ptr()
    a.k_cache, a.v_cache = key_cache.data_ptr(), value_cache.data_ptr()
    a.slot_mapping = slots.data_ptr()
    a.key_token_stride, a.key_head_stride = key.stride(0), key.stride(1)
    a.value_token_stride, a.value_head_stride = value.stride(0), value.stride(1)
    a.k_page_stride, a.k_row_stride, a.k_head_stride = key_cache.stride(0), key_cache.stride(1), key_cache.stride(2)
    a.v_page_stride, a.v_row_stride, a.v_head_stride = (value_cache.stride(0), value_cache.stride(1),
                                                         value_cache.stride(2))
    a.num_pages = key_cache.shape[0]
    a.num_tokens, a.num_kv_heads, a.head_dim, a.page_size = tokens, heads, dim, key_cache.shape[1]
    a.dtype = _DTYPES[key.dtype]
    with torch.cuda.device(key.device):
        stream = torch.cuda.current_stream().cuda_stream
        rc = N.load().pat_b200_append_kv(C.byref(a), C.c_void_p(stream))
    if rc != 0:
        raise RuntimeError(f"reshape_and_cache_flash failed: {N.strerror(rc)} ({rc})")


# --------------------------------------------------------------------------- cache held in 4 bits
def int4_tile_bytes(head_dim: int) -> int:
    """Bytes of K and V of 16 tokens of one KV head in a 4-bit cache."""
    n = int(N.load().pat_b200_int4_tile_bytes(int(head_dim)))
    if n == 0:
        raise RuntimeError("head_dim must be 64 / 128 currently")
    return n


def int4_cache_shape(num_pages: int, page_size: int, kv_heads: int, head_dim: int):
    """Shape of the uint8 tensor that holds ``num_pages`` pages of K and V in 4 bits.

    Every (token, KV head) row of K and of V is stored as codes ``c`` in 0..15 with a scale and an
    offset of its own in the model's 16-bit type: ``lo = min x``, ``s = round16((max x - lo) / 15)``,
    ``c = rint((x - lo) / s)``; its values are ``lo + s * c``.  That is ``head_dim + 8`` bytes per token
    and KV head instead of ``4 * head_dim``.  Allocate it zeroed or not: only slots that were written are
    ever read."""
    if page_size < 16 or page_size % 16 != 0 or page_size > 256:
        raise RuntimeError("page_size must be a multiple of 16, at most 256")
    return (int(num_pages), int(kv_heads), int(page_size) // 16, int4_tile_bytes(head_dim))


def _check_int4_cache(kv_cache: torch.Tensor, heads: int, dim: int) -> None:
    if kv_cache.dtype != torch.uint8 or kv_cache.dim() != 4:
        raise RuntimeError("kv_cache must be uint8 [pages, kv_heads, page_size / 16, tile bytes]")
    tile = int4_tile_bytes(dim)
    if kv_cache.shape[1] != heads or kv_cache.shape[3] != tile:
        raise RuntimeError("kv_cache disagrees with the rows on kv_heads / head_dim")
    if kv_cache.stride(3) != 1 or (kv_cache.shape[2] > 1 and kv_cache.stride(2) != tile):
        raise RuntimeError("the tiles of a page and head must be contiguous in kv_cache")


_ROW_POINTERS = struct.Struct("4P")
_row_calls = Signatures()


def _check_int4_rows(key, value, kv_cache, slots):
    """(argument bytes behind the pointers, or None when there is nothing to do; device; whether
    ``slots`` can be used as it is)."""
    for n, t in (("key", key), ("value", value), ("kv_cache", kv_cache), ("slot_mapping", slots)):
        if not t.is_cuda:
            raise RuntimeError(f"{n} must be a CUDA tensor")
        if t.device != key.device:
            raise RuntimeError(f"{n} must be on the device of key")
    if key.dtype not in _DTYPES or value.dtype != key.dtype:
        raise RuntimeError("key and value must share one dtype, fp16 or bf16")
    if key.dim() != 3 or value.shape != key.shape:
        raise RuntimeError("key and value must be [num_tokens, kv_heads, head_dim]")
    tokens, heads, dim = key.shape
    _check_int4_cache(kv_cache, heads, dim)
    for n, t in (("key", key), ("value", value)):
        if t.stride(-1) != 1:
            raise RuntimeError(f"{n} must have a contiguous last dimension")
    if slots.dtype.is_floating_point or slots.dtype.is_complex or slots.dtype == torch.bool:
        raise RuntimeError("slot_mapping must hold integers")
    if slots.numel() < tokens:
        raise RuntimeError("slot_mapping is shorter than the number of tokens")
    as_is = slots.dtype == torch.int64 and slots.is_contiguous()
    if kv_cache.shape[0] == 0 or tokens == 0 or heads == 0:
        return None, key.get_device(), as_is
    a = N.Int4RowsArgs()
    (a.key_token_stride, a.key_head_stride, _), (a.value_token_stride, a.value_head_stride, _) = strides_of(key), strides_of(value)
    a.page_stride, a.head_stride = strides_of(kv_cache)[:2]
    a.num_pages = kv_cache.shape[0]
    a.num_tokens, a.num_kv_heads, a.head_dim, a.page_size = tokens, heads, dim, kv_cache.shape[2] * 16
    a.dtype = _DTYPES[key.dtype]
    return struct_tail(a, _ROW_POINTERS.size), key.get_device(), as_is


def _int4_rows(name: str, fn, key, value, kv_cache, slots) -> None:
    sig = (key.dtype, key.shape, key.stride(), key.get_device(), value.dtype, value.shape, value.stride(), value.get_device(),
           kv_cache.dtype, kv_cache.shape, kv_cache.stride(), kv_cache.get_device(),
           slots.dtype, slots.shape, slots.stride(), slots.get_device())
    known = _row_calls.get(sig)
    if known is None:
        known = _row_calls.remember(sig, _check_int4_rows(key, value, kv_cache, slots))
    tail, index, as_is = known
    if tail is None:
        return
    if not as_is:
        slots = slots.flatten().to(torch.int64).contiguous()
    rc = launch(fn, _ROW_POINTERS.pack(key.data_ptr(), value.data_ptr(), kv_cache.data_ptr(), slots.data_ptr()) + tail, index)
    if rc != 0:
        raise RuntimeError(f"{name} failed: {N.strerror(rc)} ({rc})")


def reshape_and_cache_int4(key: torch.Tensor, value: torch.Tensor, kv_cache: torch.Tensor,
                           slot_mapping: torch.Tensor) -> None:
    """Quantises ``key[i]`` / ``value[i]`` (``[num_tokens, kv_heads, head_dim]``, fp16 or bf16) into the 4-bit
    cache (``int4_cache_shape``) at ``slot_mapping[i] = page * page_size + row``.  Tokens with a
    negative slot, or one beyond the cache, are skipped; slots must be distinct.  A row that holds a NaN or an
    infinity is stored as NaN.  All rows of a cache have one dtype (its scales are stored in it)."""
    _int4_rows("reshape_and_cache_int4", N.load().pat_b200_append_int4, key, value, kv_cache, slot_mapping)


def gather_cache_int4(kv_cache: torch.Tensor, slot_mapping: torch.Tensor, key: torch.Tensor, value: torch.Tensor) -> None:
    """Reads the tokens at ``slot_mapping`` back from a 4-bit cache into ``key`` / ``value``
    (``[num_tokens, kv_heads, head_dim]``, the dtype that was appended), e.g. a cached prefix for a
    prefill that runs on 16-bit keys.  Rows of skipped slots (see ``reshape_and_cache_int4``) keep what they hold."""
    _int4_rows("gather_cache_int4", N.load().pat_b200_gather_int4, key, value, kv_cache, slot_mapping)


# --------------------------------------------------------------------------- moving pages
def _page_geometry(cache: torch.Tensor):
    """(rows, row_stride, row_bytes) of one page of ``cache``: runs of contiguous bytes at one stride."""
    item = cache.element_size()
    run, rows, row_stride = item, 1, 0
    for size, stride in zip(reversed(cache.shape[1:]), reversed(cache.stride()[1:])):
        if size == 1:
            continue
        stride *= item
        if rows == 1 and stride == run:
            run *= size
        elif rows == 1:
            rows, row_stride = size, stride
        elif stride == rows * row_stride:
            rows *= size
        else:
            return None
    return rows, row_stride or run, run


def copy_pages(caches: Union[torch.Tensor, Sequence[torch.Tensor]], mapping) -> None:
    """Copies page ``from`` over page ``to`` in every tensor of ``caches``, for every pair ``(from, to)`` of
    ``mapping``.

    ``caches``: paged caches of any kind (K and V of all layers, 16-bit or 4-bit), all of one shape,
    dtype and strides; dimension 0 counts pages.  ``mapping``: ``[n, 2]``, a list or an integer CPU tensor
    (what ``PagePool.fork`` and ``PagePool.compact`` return; checked: pages inside the cache, and no page that is the target
    of one pair may occur in another), or an int64 CUDA tensor with the same contract, which is not
    checked; pairs with a page outside the cache are then skipped.  A host mapping travels in the
    launch itself: a CUDA graph captured around the call repeats that mapping."""
    caches = [caches] if isinstance(caches, torch.Tensor) else caches
    on_device = isinstance(mapping, torch.Tensor) and mapping.is_cuda
    if not on_device:
        mapping = torch.as_tensor(mapping)
        if mapping.numel() == 0:
            mapping = mapping.reshape(0, 2)
        elif mapping.is_floating_point() or mapping.is_complex() or mapping.dtype == torch.bool:
            raise RuntimeError("mapping must hold integers")
        mapping = mapping.to(torch.int64).contiguous()
    if mapping.dim() != 2 or mapping.shape[1] != 2:
        raise RuntimeError("mapping must be [n, 2]: pairs (from, to)")
    if on_device and (mapping.dtype != torch.int64 or not mapping.is_contiguous()):
        raise RuntimeError("a CUDA mapping must be contiguous int64")
    if not caches:
        return
    first = caches[0]
    shape, strides, dtype, index = first.shape, first.stride(), first.dtype, first.get_device()
    for t in caches:
        if t.get_device() < 0:
            raise RuntimeError("caches must be CUDA tensors")
        if t.get_device() != index or t.dtype != dtype or t.shape != shape or t.stride() != strides:
            raise RuntimeError("caches must share device, dtype, shape and strides")
    if on_device and mapping.get_device() != index:
        raise RuntimeError("mapping must be on the device of the caches, or on the host")
    sig = (shape, strides, dtype)
    geometry = _copy_geometries.get(sig)
    if geometry is None:
        geometry = _copy_geometries.remember(sig, _copy_geometry(first))
    n = mapping.shape[0]
    if geometry is _NO_BYTES:
        if n and shape[0] == 0:
            raise RuntimeError("mapping names a page outside the cache (0 pages)")
        return
    pointers = array.array("Q", [t.data_ptr() for t in caches])
    address = mapping.data_ptr() if n else 0
    rc = launch(N.load().pat_b200_copy_pages,
                _COPY_ARGS.pack(pointers.buffer_info()[0], 0 if on_device else address, address if on_device else 0, *geometry,
                                len(pointers), n, 0), index)
    if rc == -10:
        _explain_mapping(mapping, shape[0])
    if rc != 0:
        raise RuntimeError(f"copy_pages failed: {N.strerror(rc)} ({rc})")


_COPY_ARGS = struct.Struct("3P4q4i")        # pat_copy_args, `rows` first of the int32
_copy_geometries = Signatures()
_NO_BYTES = ()


def _copy_geometry(cache: torch.Tensor):
    """(page_stride, row_stride, row_bytes, num_pages, rows) of the argument structure."""
    if cache.dim() < 2:
        raise RuntimeError("caches must be [pages, ...]")
    if cache.numel() == 0:
        return _NO_BYTES
    geometry = _page_geometry(cache)
    if geometry is None:
        raise RuntimeError("a page must consist of equally long contiguous runs at one stride")
    rows, row_stride, row_bytes = geometry
    page_stride = cache.stride(0) * cache.element_size() if cache.shape[0] > 1 else rows * row_stride
    return page_stride, row_stride, row_bytes, cache.shape[0], rows


def _explain_mapping(mapping: torch.Tensor, pages: int) -> None:
    """Says what is wrong with a mapping the library refused."""
    if int(mapping.min()) < 0 or int(mapping.max()) >= pages:
        raise RuntimeError(f"mapping names a page outside the cache ({pages} pages)")
    if mapping[:, 1].unique().numel() != mapping.shape[0]:
        raise RuntimeError("a page is the target of two pairs")
    raise RuntimeError("a page is both a source and a target")

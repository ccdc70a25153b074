"""K / V pages held in 8 bits: written from dense rows, and read back."""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _lib
from ._check import (check_cuda, check_dim, check_dtype, check_input, check_same_device, dtype_code, fine_rows,
                     stream_and_switch)
from .attention import _cache_strides

_ROW_TYPES = {torch.float16: _lib.TWL_F16, torch.bfloat16: _lib.TWL_BF16}
KV_FORMATS = {torch.int8: _lib.TWL_I8, torch.float8_e4m3fn: _lib.TWL_E4M3}


def kv_format_code(dt: torch.dtype, name: str) -> int:
    """Library code of an 8-bit page format."""
    if dt not in KV_FORMATS:
        raise RuntimeError(f"{name}: 8-bit pages are int8 or float8_e4m3fn, got {dt}")
    return KV_FORMATS[dt]


def check_quant_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                      v_scale: torch.Tensor):
    """Checks of the four tensors of an 8-bit cache: ``(format, cache strides, scale strides)``."""
    ks = _cache_strides(k_cache, "k_cache")
    if _cache_strides(v_cache, "v_cache") != ks or v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype:
        raise RuntimeError("k_cache and v_cache must share shape, dtype and strides")
    fmt = kv_format_code(k_cache.dtype, "k_cache")
    for name, t in (("k_scale", k_scale), ("v_scale", v_scale)):
        check_cuda(t, name); check_dtype(t, torch.float32, name)
        if tuple(t.shape) != tuple(k_cache.shape[:3]):
            raise RuntimeError(f"{name} must be [pages, 16, kv_heads] like the cache")
    if k_scale.stride() != v_scale.stride():
        raise RuntimeError("k_scale and v_scale must share strides")
    check_same_device(k_cache, ("v_cache", v_cache), ("k_scale", k_scale), ("v_scale", v_scale))
    return fmt, ks, k_scale.stride()


def check_page_table(ref: torch.Tensor, batch: int, indices: torch.Tensor, indptr: torch.Tensor,
                     last: torch.Tensor, prefix: str = "kv") -> None:
    """Checks of a CSR page table of ``batch`` lists."""
    names = (f"{prefix}_page_indices", f"{prefix}_page_indptr", f"{prefix}_last_page_len")
    for name, t in zip(names, (indices, indptr, last)):
        check_input(t, name); check_dtype(t, torch.int32, name)
    if indptr.numel() != batch + 1 or last.numel() != batch:
        raise RuntimeError(f"{names[1]} must have {batch + 1} and {names[2]} {batch} elements")
    check_same_device(ref, *zip(names, (indices, indptr, last)))


def _check_tokens(k_cache, token_indptr, kv_page_indices, kv_page_indptr, kv_last_page_len) -> int:
    check_input(token_indptr, "token_indptr"); check_dtype(token_indptr, torch.int32, "token_indptr")
    batch = token_indptr.numel() - 1
    if batch < 1:
        raise RuntimeError("token_indptr must have batch + 1 elements")
    check_same_device(k_cache, ("token_indptr", token_indptr))
    check_page_table(k_cache, batch, kv_page_indices, kv_page_indptr, kv_last_page_len)
    return batch


def _fine(k_cache, v_cache, k_scale, v_scale, token_indptr, kv_page_indices, kv_page_indptr, kv_last_page_len) -> bool:
    """Whether a cache and its tables are plainly right; if not, the checks above find out what is wrong."""
    try:
        dev, cs, batch = k_cache.get_device(), k_cache.stride(), token_indptr.numel() - 1
        shape = k_cache.shape
        return (dev >= 0 and len(cs) == 4 and cs[3] == 1 and shape[1] == _lib.PAGE and shape[3] == _lib.HEAD_DIM
                and k_cache.dtype in KV_FORMATS and v_cache.dtype is k_cache.dtype
                and v_cache.stride() == cs and v_cache.shape == shape and v_cache.get_device() == dev
                and k_scale.dtype is torch.float32 and v_scale.dtype is torch.float32
                and k_scale.shape == shape[:3] and v_scale.shape == k_scale.shape
                and k_scale.stride() == v_scale.stride() and k_scale.get_device() == dev
                and v_scale.get_device() == dev
                and batch >= 1 and kv_page_indptr.numel() == batch + 1 and kv_last_page_len.numel() == batch
                and fine_rows(dev, torch.int32, token_indptr, kv_page_indices, kv_page_indptr, kv_last_page_len))
    except AttributeError:                    # no tensor
        return False


def row_strides(rows: torch.Tensor) -> Tuple[int, int]:
    """Token and head stride of [T,Hkv,128] rows, 0 where there is one token or head and the tensor's own stride
    means nothing."""
    T, Hkv, _ = rows.shape
    t, h, _ = rows.stride()
    return t if T > 1 else 0, h if Hkv > 1 else 0


def kv_quant_append(k_new: torch.Tensor, v_new: torch.Tensor, token_indptr: torch.Tensor,
                    k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                    v_scale: torch.Tensor, kv_page_indices: torch.Tensor,
                    kv_page_indptr: torch.Tensor, kv_last_page_len: torch.Tensor) -> None:
    """Quantise the rows of ``k_new`` / ``v_new`` [T,Hkv,128] (fp16 / bf16, head_dim contiguous, the other
    strides the same for both and multiples of 8, 16-byte aligned) into 8-bit pages in one launch.

    ``k_cache`` / ``v_cache`` [pages,16,Hkv,128] int8 or float8_e4m3fn (page / token / head strides
    that are multiples of 8; attention over them takes multiples of 16), ``k_scale`` / ``v_scale`` fp32
    [pages,16,Hkv] of any strides. Every (token, kv head) row is scaled by its
    own largest magnitude: ``scale = max(max|x| / T, 2**-126)`` with T = 127 or 448, code = x / scale
    rounded to nearest even. Rows ``token_indptr[b]`` to ``token_indptr[b + 1]`` (int32 [B+1]) are the
    last tokens of request b: the page table counts them already. Rows from ``token_indptr[B]`` on are
    ignored; rows that have no place in the table are skipped. A page that is written must belong
    to one request only. A row with a non-finite element reads back as NaN."""
    if not _fine(k_cache, v_cache, k_scale, v_scale, token_indptr, kv_page_indices, kv_page_indptr, kv_last_page_len):
        check_quant_cache(k_cache, v_cache, k_scale, v_scale)
        _check_tokens(k_cache, token_indptr, kv_page_indices, kv_page_indptr, kv_last_page_len)
    if not (isinstance(k_new, torch.Tensor) and isinstance(v_new, torch.Tensor)):
        check_cuda(k_new, "k_new"); check_cuda(v_new, "v_new")
    dev, Hkv, ns = k_cache.get_device(), k_cache.size(2), k_new.stride()
    if not (k_new.shape[1:] == (Hkv, _lib.HEAD_DIM) and len(ns) == 3 and ns[2] == 1 and k_new.dtype in _ROW_TYPES
            and v_new.shape == k_new.shape and v_new.stride() == ns and v_new.dtype is k_new.dtype
            and k_new.get_device() == dev and v_new.get_device() == dev):
        for name, t in (("k_new", k_new), ("v_new", v_new)):
            check_cuda(t, name); check_dim(3, t, name)
            if t.size(1) != Hkv or t.size(2) != _lib.HEAD_DIM or t.stride(2) != 1:
                raise RuntimeError(f"{name} must be [T, {Hkv}, {_lib.HEAD_DIM}] with contiguous head_dim")
            if t.dtype not in _ROW_TYPES:
                raise RuntimeError(f"{name} must be float16 or bfloat16")
        if v_new.shape != k_new.shape or row_strides(v_new) != row_strides(k_new) or v_new.dtype != k_new.dtype:
            raise RuntimeError("k_new and v_new must share shape, dtype and strides")
        check_same_device(k_cache, ("k_new", k_new), ("v_new", v_new))
    T = k_new.size(0)
    if T == 0 or kv_page_indices.numel() == 0:
        return                                # no row, or none that has a place
    stream, switch = stream_and_switch(dev)
    if switch:
        with torch.cuda.device(dev):
            return kv_quant_append(k_new, v_new, token_indptr, k_cache, v_cache, k_scale, v_scale, kv_page_indices,
                                   kv_page_indptr, kv_last_page_len)
    if T == 1 or Hkv == 1:
        ns = row_strides(k_new)
    cs, ss = k_cache.stride(), k_scale.stride()
    rc = _lib.lib().twl_kv_quant_append(
        k_new.data_ptr(), v_new.data_ptr(), _ROW_TYPES[k_new.dtype], ns[0], ns[1], token_indptr.data_ptr(),
        T, k_cache.data_ptr(), v_cache.data_ptr(), KV_FORMATS[k_cache.dtype], cs[0], cs[1], cs[2],
        k_scale.data_ptr(), v_scale.data_ptr(), *ss, k_cache.size(0), kv_page_indices.data_ptr(),
        kv_page_indptr.data_ptr(), kv_last_page_len.data_ptr(), token_indptr.numel() - 1, Hkv, stream)
    if rc:
        _lib.check(rc, "KvQuantAppend")


def kv_quant_read(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                  v_scale: torch.Tensor, kv_page_indices: torch.Tensor, kv_page_indptr: torch.Tensor,
                  kv_last_page_len: torch.Tensor, token_indptr: torch.Tensor, tokens: int,
                  dtype: torch.dtype = torch.bfloat16, k_out: Optional[torch.Tensor] = None,
                  v_out: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The values 8-bit pages hold, as dense rows ``(k, v)`` [tokens,Hkv,128] in ``dtype`` (fp16, bf16
    or fp32): rows ``token_indptr[b]`` to ``token_indptr[b + 1]`` are the last tokens of request b (all
    of them when ``token_indptr`` adds up the requests' lengths). Arguments as in
    :func:`kv_quant_append`. Rows from ``token_indptr[B]`` on are left as they were (undefined in
    outputs this call allocates); rows that have no place in the table are zeros."""
    if not _fine(k_cache, v_cache, k_scale, v_scale, token_indptr, kv_page_indices, kv_page_indptr, kv_last_page_len):
        check_quant_cache(k_cache, v_cache, k_scale, v_scale)
        _check_tokens(k_cache, token_indptr, kv_page_indices, kv_page_indptr, kv_last_page_len)
    dev, Hkv, tokens = k_cache.get_device(), k_cache.size(2), int(tokens)
    if tokens < 0:
        raise RuntimeError("tokens must not be negative")
    code = dtype_code(dtype, "dtype")
    stream, switch = stream_and_switch(dev)
    if switch:
        with torch.cuda.device(dev):
            return kv_quant_read(k_cache, v_cache, k_scale, v_scale, kv_page_indices, kv_page_indptr, kv_last_page_len,
                                 token_indptr, tokens, dtype, k_out, v_out)
    shape = (tokens, Hkv, _lib.HEAD_DIM)
    for name, t in (("k_out", k_out), ("v_out", v_out)):
        if t is not None:
            check_input(t, name); check_same_device(k_cache, (name, t))
            if tuple(t.shape) != shape or t.dtype != dtype:
                raise RuntimeError(f"{name} must be {list(shape)} of {dtype}")
    if k_out is None:
        k_out = torch.empty(shape, dtype=dtype, device=dev)
    if v_out is None:
        v_out = torch.empty(shape, dtype=dtype, device=dev)
    if tokens == 0:
        return k_out, v_out
    if kv_page_indices.numel() == 0:          # no list holds a page, and the tensor has no address
        kv_page_indices, kv_page_indptr = kv_page_indptr, torch.zeros_like(kv_page_indptr)
    cs, ss = k_cache.stride(), k_scale.stride()
    rc = _lib.lib().twl_kv_quant_read(
        k_out.data_ptr(), v_out.data_ptr(), code, token_indptr.data_ptr(), tokens, k_cache.data_ptr(),
        v_cache.data_ptr(), KV_FORMATS[k_cache.dtype], cs[0], cs[1], cs[2], k_scale.data_ptr(), v_scale.data_ptr(),
        *ss, k_cache.size(0), kv_page_indices.data_ptr(), kv_page_indptr.data_ptr(), kv_last_page_len.data_ptr(),
        token_indptr.numel() - 1, Hkv, stream)
    if rc:
        _lib.check(rc, "KvQuantRead")
    return k_out, v_out

"""Dense paged decode attention over 8-bit pages and for requests that share a prefix."""
from __future__ import annotations

import math
from typing import Optional

import torch

from .. import _lib
from ._check import (check_dim, check_dtype, check_input, check_same_device, fine_rows, ptr,
                     stream_and_switch)
from .attention import _cache_strides
from .quant_cache import KV_FORMATS, check_page_table, check_quant_cache

_QUERY_TYPES = {torch.float16: _lib.TWL_F16, torch.bfloat16: _lib.TWL_BF16}


def prefix_attention_workspace_bytes(batch: int, num_q_heads: int, num_kv_heads: int, groups: int,
                                     max_prefix_tokens: int, max_group_size: int,
                                     max_tokens: int) -> int:
    """Bytes of scratch :func:`prefix_paged_decode_attention` needs, or (``groups`` = 0)
    :func:`quant_paged_decode_attention`."""
    return int(_lib.lib().twl_prefix_attn_workspace_bytes(batch, num_q_heads, num_kv_heads, groups,
                                                          max_prefix_tokens, max_group_size, max_tokens))


def _bound(value, name: str, least: int) -> int:
    value = int(value)
    if value < least or value > 1 << 24:
        raise RuntimeError(f"{name} must be in [{least}, 2**24], got {value}")
    return value


def _fine(q, k_cache, v_cache, k_scale, v_scale, kv_page_indices, kv_page_indptr, kv_last_page_len) -> bool:
    """Whether the operands are plainly right; if not, :func:`_check` finds out what is wrong."""
    try:
        dev, cs = q.get_device(), k_cache.stride()
        if not (dev >= 0 and q.dim() == 3 and q.is_contiguous() and q.dtype in _QUERY_TYPES and len(cs) == 4
                and v_cache.stride() == cs and cs[3] == 1 and v_cache.shape == k_cache.shape
                and v_cache.dtype is k_cache.dtype and k_cache.get_device() == dev and v_cache.get_device() == dev):
            return False
        B, H, D = q.shape
        pages, page, Hkv, Dk = k_cache.shape
        if not (D == Dk == _lib.HEAD_DIM and page == _lib.PAGE and B and H and pages and Hkv and H % Hkv == 0
                and kv_page_indptr.numel() == B + 1 and kv_last_page_len.numel() == B
                and fine_rows(dev, torch.int32, kv_page_indices, kv_page_indptr, kv_last_page_len)):
            return False
        if k_scale is None:
            return v_scale is None and k_cache.dtype is q.dtype
        return (v_scale is not None and k_cache.dtype in KV_FORMATS and k_scale.dtype is torch.float32
                and v_scale.dtype is torch.float32 and k_scale.shape == k_cache.shape[:3]
                and v_scale.shape == k_scale.shape and k_scale.stride() == v_scale.stride()
                and k_scale.get_device() == dev and v_scale.get_device() == dev)
    except AttributeError:                    # no tensor
        return False


def _check(q, k_cache, v_cache, k_scale, v_scale, kv_page_indices, kv_page_indptr, kv_last_page_len) -> None:
    check_input(q, "q"); check_dim(3, q, "q")
    B, H, D = q.shape
    if D != _lib.HEAD_DIM:
        raise RuntimeError(f"head_dim must be {_lib.HEAD_DIM}, got {D}")
    if B == 0 or H == 0:
        raise RuntimeError("q must not be empty")
    if q.dtype not in _QUERY_TYPES:
        raise RuntimeError("q must be float16 or bfloat16")
    if (k_scale is None) != (v_scale is None):
        raise RuntimeError("k_scale and v_scale go together")
    if k_scale is None:
        cs = _cache_strides(k_cache, "k_cache")
        if _cache_strides(v_cache, "v_cache") != cs or k_cache.shape != v_cache.shape:
            raise RuntimeError("k_cache and v_cache must share shape and strides")
        if k_cache.dtype != q.dtype or v_cache.dtype != q.dtype:
            raise RuntimeError("q, k_cache and v_cache must share one dtype (8-bit pages need k_scale and v_scale)")
    else:
        check_quant_cache(k_cache, v_cache, k_scale, v_scale)
    Hkv = k_cache.size(2)
    if Hkv == 0 or H % Hkv != 0:
        raise RuntimeError(f"num_q_heads {H} must be a multiple of num_kv_heads {Hkv}")
    if k_cache.size(0) == 0:
        raise RuntimeError("the cache must hold a page")
    check_same_device(q, ("k_cache", k_cache), ("v_cache", v_cache))
    check_page_table(q, B, kv_page_indices, kv_page_indptr, kv_last_page_len)


def _attend(q, k_cache, v_cache, k_scale, v_scale, prefix, kv_page_indices, kv_page_indptr,
            kv_last_page_len, max_tokens, sm_scale, return_lse, out, workspace, what):
    """The launch; the operands have been checked."""
    B, H, D = q.shape
    Hkv, dev, dtype = k_cache.size(2), q.get_device(), q.dtype
    cs = k_cache.stride()
    if k_scale is None:
        ss, fmt = (0, 0, 0), _QUERY_TYPES[dtype]
    else:
        ss, fmt = k_scale.stride(), KV_FORMATS[k_cache.dtype]
    stream, switch = stream_and_switch(dev)
    if switch:
        with torch.cuda.device(dev):
            return _attend(q, k_cache, v_cache, k_scale, v_scale, prefix, kv_page_indices, kv_page_indptr,
                           kv_last_page_len, max_tokens, sm_scale, return_lse, out, workspace, what)
    if out is None:
        out = torch.empty_like(q)
    else:
        check_input(out, "out"); check_same_device(q, ("out", out))
        if out.shape != q.shape or out.dtype != dtype:
            raise RuntimeError("out must match q")
    lse = torch.empty((B, H), dtype=torch.float32, device=dev) if return_lse else None
    scale = 1.0 / math.sqrt(D) if sm_scale is None else float(sm_scale)
    p_ids, p_ptr, p_last, g_ptr, groups, max_prefix, max_group = prefix
    if kv_page_indices.numel() == 0:          # no list holds a page, and the tensor has no address
        max_tokens = 0
    if groups and p_ids.numel() == 0:
        max_prefix = 0
    L = _lib.lib()
    need = L.twl_prefix_attn_workspace_bytes(B, H, Hkv, groups, max_prefix, max_group, max_tokens)
    if workspace is None:
        workspace = torch.empty(need, dtype=torch.uint8, device=dev) if need else None
    else:
        check_input(workspace, "workspace"); check_dtype(workspace, torch.uint8, "workspace")
        if workspace.numel() < need or workspace.get_device() != dev:
            raise RuntimeError(f"workspace must hold {need} bytes on {q.device}")
    rc = L.twl_prefix_attn(
        q.data_ptr(), out.data_ptr(), _QUERY_TYPES[dtype], k_cache.data_ptr(), v_cache.data_ptr(), fmt, cs[0], cs[1],
        cs[2], ptr(k_scale), ptr(v_scale), *ss, k_cache.size(0), ptr(p_ids), ptr(p_ptr), ptr(p_last), ptr(g_ptr),
        groups, max_prefix, max_group, kv_page_indices.data_ptr(), kv_page_indptr.data_ptr(),
        kv_last_page_len.data_ptr(), max_tokens, B, H, Hkv, scale, ptr(lse), ptr(workspace), need, stream)
    if rc:
        _lib.check(rc, what)
    return (out, lse) if return_lse else out


def quant_paged_decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                                 k_scale: torch.Tensor, v_scale: torch.Tensor,
                                 kv_page_indices: torch.Tensor, kv_page_indptr: torch.Tensor,
                                 kv_last_page_len: torch.Tensor, max_tokens: int,
                                 sm_scale: Optional[float] = None, return_lse: bool = False,
                                 out: Optional[torch.Tensor] = None,
                                 workspace: Optional[torch.Tensor] = None):
    """Softmax attention of one decode token per request over every token of 8-bit pages
    (:func:`kv_quant_append` writes them), the 8-bit form of the dense
    :func:`group_paged_decode_attention`.

    ``q`` [B,H,128] fp16 / bf16; ``k_cache`` / ``v_cache`` [pages,16,Hkv,128] int8 or float8_e4m3fn with
    ``k_scale`` / ``v_scale`` fp32 [pages,16,Hkv]; any H that is a multiple of Hkv,
    up to 65535 rows B * H. ``max_tokens`` bounds
    the requests' lengths (tokens beyond it are not attended to). Returns ``out`` [B,H,128] in q's
    dtype (and ``lse`` fp32 [B,H]); a request without tokens gives zeros and -inf. ``workspace``: a
    uint8 tensor of :func:`prefix_attention_workspace_bytes` (..., 0, 0, 0, max_tokens) bytes that
    calls on one stream may share; by default a fresh one is allocated."""
    if k_scale is None or v_scale is None:
        raise RuntimeError("8-bit pages need k_scale and v_scale")
    operands = (q, k_cache, v_cache, k_scale, v_scale, kv_page_indices, kv_page_indptr, kv_last_page_len)
    if not _fine(*operands):
        _check(*operands)
    return _attend(q, k_cache, v_cache, k_scale, v_scale, (None, None, None, None, 0, 0, 0),
                   kv_page_indices, kv_page_indptr, kv_last_page_len, _bound(max_tokens, "max_tokens", 1),
                   sm_scale, return_lse, out, workspace, "QuantPagedDecodeAttention")


def prefix_paged_decode_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                                  prefix_page_indices: torch.Tensor,
                                  prefix_page_indptr: torch.Tensor,
                                  prefix_last_page_len: torch.Tensor, group_indptr: torch.Tensor,
                                  kv_page_indices: torch.Tensor, kv_page_indptr: torch.Tensor,
                                  kv_last_page_len: torch.Tensor, max_prefix_tokens: int,
                                  max_group_size: int, max_tokens: int,
                                  k_scale: Optional[torch.Tensor] = None,
                                  v_scale: Optional[torch.Tensor] = None,
                                  sm_scale: Optional[float] = None, return_lse: bool = False,
                                  out: Optional[torch.Tensor] = None,
                                  workspace: Optional[torch.Tensor] = None):
    """Softmax attention of one decode token per request, for requests in groups that share a prefix
    (several samples of one prompt): K / V of a prefix are read once per group and kv head and
    multiplied with the queries of all its requests.

    Requests ``group_indptr[g]`` to ``group_indptr[g + 1]`` (int32 [groups+1]) see the tokens of prefix
    list g (``prefix_page_indices`` / ``prefix_page_indptr`` [groups+1] / ``prefix_last_page_len``
    [groups], pages of the same cache) and then those of their own list (``kv_page_*``, which may be
    empty); a request outside every group sees its own only. ``q`` [B,H,128] fp16 / bf16; the cache in
    q's dtype, or int8 / float8_e4m3fn with ``k_scale`` / ``v_scale`` as in
    :func:`quant_paged_decode_attention`. ``max_prefix_tokens``, ``max_group_size`` and ``max_tokens``
    are upper bounds that size the launch: tokens beyond them are not attended to, members of a
    group beyond the second do not see its prefix. Returns ``out`` (and ``lse``) as there."""
    operands = (q, k_cache, v_cache, k_scale, v_scale, kv_page_indices, kv_page_indptr, kv_last_page_len)
    if not _fine(*operands):
        _check(*operands)
    batch = q.size(0)
    try:
        groups = group_indptr.numel() - 1
        fine = (1 <= groups <= batch and prefix_page_indptr.numel() == groups + 1
                and prefix_last_page_len.numel() == groups
                and fine_rows(q.get_device(), torch.int32, group_indptr, prefix_page_indices, prefix_page_indptr,
                              prefix_last_page_len))
    except AttributeError:                    # no tensor
        fine = False
    if not fine:
        check_input(group_indptr, "group_indptr"); check_dtype(group_indptr, torch.int32, "group_indptr")
        if groups < 1 or groups > batch:
            raise RuntimeError("group_indptr must have groups + 1 elements, with 1 to batch groups")
        check_same_device(q, ("group_indptr", group_indptr))
        check_page_table(q, groups, prefix_page_indices, prefix_page_indptr, prefix_last_page_len, "prefix")
    max_group = _bound(max_group_size, "max_group_size", 1)
    if max_group > batch:
        raise RuntimeError("max_group_size must not exceed the batch")
    prefix = (prefix_page_indices, prefix_page_indptr, prefix_last_page_len, group_indptr, groups,
              _bound(max_prefix_tokens, "max_prefix_tokens", 0), max_group)
    return _attend(q, k_cache, v_cache, k_scale, v_scale, prefix, kv_page_indices, kv_page_indptr,
                   kv_last_page_len, _bound(max_tokens, "max_tokens", 0), sm_scale, return_lse, out,
                   workspace, "PrefixPagedDecodeAttention")

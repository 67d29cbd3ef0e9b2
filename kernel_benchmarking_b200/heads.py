"""Operators on the heads of a projection's output: query/key norm with rotation, and the e4m3 cache of keys and values.

They stand between `rmsnorm_linear` (which writes q, k and v side by side in the rows of one matrix) and whatever
attention the caller runs; views into those rows go in as they are.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .ops import _index_devices, _on_device, _stream_ptr

_INDEX_TYPES = (torch.int64, torch.int32)


def _check_heads(name: str, t: torch.Tensor, like: Optional[torch.Tensor] = None) -> None:
    """[tokens, heads, channels] bf16 on the GPU, channels contiguous; the strides of tokens and heads are free."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (this operator has no CPU path)")
    if t.dtype != torch.bfloat16:
        raise ValueError(f"{name} must be torch.bfloat16, got {t.dtype}")
    if t.dim() != 3 or t.stride(2) != 1:
        raise ValueError(f"{name} must be [tokens, heads, channels] with contiguous channels, got {tuple(t.shape)}")
    if like is not None and t.device != like.device:
        raise ValueError(f"{name} must be on {like.device}, got {t.device}")


def _check_index(name: str, t: torch.Tensor, n: int, like: torch.Tensor, types=_INDEX_TYPES) -> None:
    if (not isinstance(t, torch.Tensor) or t.dtype not in types or t.dim() != 1 or t.shape[0] != n
            or t.device != like.device or (n > 1 and t.stride(0) != 1)):
        raise ValueError(f"{name} must be a contiguous vector of {n} {' or '.join(str(x) for x in types)} on {like.device}")


def rope_table(positions: int, rotary_dim: int, base: float = 10000.0, device: Optional[torch.device] = None) -> torch.Tensor:
    """The table `qk_norm_rope` reads: [positions, rotary_dim] fp32, rotary_dim / 2 cosines of p * base^(-2i / rotary_dim),
    then the sines, computed in 64 bits (an angle of a far position has lost its fraction in 32)."""
    if positions <= 0 or rotary_dim <= 0 or rotary_dim % 2:
        raise ValueError("rope_table needs a positive number of positions and a positive even rotary_dim")
    inv = float(base) ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64) / rotary_dim)
    angle = torch.arange(positions, dtype=torch.float64)[:, None] * inv
    return torch.cat([angle.cos(), angle.sin()], dim=1).float().to(device or "cuda")


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, q_gamma: Optional[torch.Tensor], k_gamma: Optional[torch.Tensor],
                 table: torch.Tensor, positions: torch.Tensor, eps: float = 1e-6, *, interleaved: bool = False,
                 out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMSNorm over each head of q [T, Hq, D] and k [T, Hk, D] and the rotation by position, in one kernel; fp32 between
    the load and the one rounding to bf16.

    `q_gamma`, `k_gamma` [D] bf16 or None (= ones).  `table` [P, rotary_dim] fp32 as `rope_table` makes it; the first
    rotary_dim channels are rotated, in halves (i, i + rotary_dim / 2) or, `interleaved`, in neighbours (2i, 2i + 1).
    `positions` [T] int64 or int32; one outside the table leaves its token's rows unwritten and `check_status` raises.
    D a multiple of 8 up to 256, rotary_dim of 16 (interleaved: 8).  `out`: a pair of tensors to write, q and k
    themselves for an update in place; they may share no other memory with the inputs or each other."""
    _check_heads("q", q)
    _check_heads("k", k, q)
    T, Hq, D = q.shape
    Hk = k.shape[1]
    if k.shape[0] != T or k.shape[2] != D:
        raise ValueError(f"q is [{T}, {Hq}, {D}]: k must be [{T}, Hk, {D}], got {tuple(k.shape)}")
    for name, g in (("q_gamma", q_gamma), ("k_gamma", k_gamma)):
        if g is not None and (not isinstance(g, torch.Tensor) or g.dtype != torch.bfloat16 or g.device != q.device
                              or g.shape != (D,) or (D > 1 and g.stride(0) != 1)):
            raise ValueError(f"{name} must be a contiguous bf16 vector of length D={D} on q's device")
    if (not isinstance(table, torch.Tensor) or table.dtype != torch.float32 or table.dim() != 2 or table.device != q.device
            or table.stride(1) != 1):
        raise ValueError("table must be [positions, rotary_dim] fp32, row-major, on q's device")
    _check_index("positions", positions, T, q)
    if out is None:
        qo = torch.empty((T, Hq, D), dtype=torch.bfloat16, device=q.device)
        ko = torch.empty((T, Hk, D), dtype=torch.bfloat16, device=q.device)
    else:
        qo, ko = out
        _check_heads("out[0]", qo, q)
        _check_heads("out[1]", ko, q)
        if qo.shape != q.shape or ko.shape != k.shape:
            raise ValueError(f"out must be {tuple(q.shape)} and {tuple(k.shape)}, got {tuple(qo.shape)} and {tuple(ko.shape)}")
    if T == 0:
        return qo, ko
    with _on_device(q.device):
        rc = _lib.load().rl_qk_norm_rope_bf16(
            q.data_ptr(), k.data_ptr(), None if q_gamma is None else q_gamma.data_ptr(),
            None if k_gamma is None else k_gamma.data_ptr(), table.data_ptr(), positions.data_ptr(),
            positions.dtype == torch.int64, qo.data_ptr(), ko.data_ptr(), T, Hq, Hk, D, table.shape[1], table.shape[0],
            table.stride(0), q.stride(0), q.stride(1), k.stride(0), k.stride(1), qo.stride(0), qo.stride(1), ko.stride(0),
            ko.stride(1), eps, interleaved, _stream_ptr(q.device))
    _lib.check(rc, "rl_qk_norm_rope_bf16")
    _index_devices.add(q.device.index)
    return qo, ko


def _check_cache(k_codes, k_scale, v_codes, v_scale) -> None:
    for name, t, dtype, nd in (("k_codes", k_codes, torch.float8_e4m3fn, 4), ("v_codes", v_codes, torch.float8_e4m3fn, 4),
                               ("k_scale", k_scale, torch.float32, 3), ("v_scale", v_scale, torch.float32, 3)):
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor (this operator has no CPU path)")
        if t.dtype != dtype or t.dim() != nd or t.device != k_codes.device:
            raise ValueError(f"{name} must be {nd}-D {dtype} on {k_codes.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    if k_codes.stride(3) != 1:
        raise ValueError("the codes' channels must be contiguous")
    if v_codes.shape != k_codes.shape or v_codes.stride() != k_codes.stride():
        raise ValueError("v_codes must have the shape and strides of k_codes")
    if k_scale.shape != k_codes.shape[:3] or v_scale.shape != k_scale.shape or v_scale.stride() != k_scale.stride():
        raise ValueError(f"k_scale and v_scale must both be {tuple(k_codes.shape[:3])}, with the same strides")


def kv_cache_write(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_codes: torch.Tensor, k_scale: torch.Tensor,
                   v_codes: torch.Tensor, v_scale: torch.Tensor) -> None:
    """Write keys and values k, v [T, H, D] bf16 into a paged e4m3 cache, quantised as they are written with one scale per
    token and head: scale = max(max|x|, 2^-100) / 448, code = e4m3(448 x / max|x|), exactly rounded.

    Codes [pages, page_size, H, D] float8_e4m3fn and scales [pages, page_size, H] fp32, any strides with contiguous
    channels, the same for keys and values.  `slots` [T] int64 or int32: page * page_size + place in the page.  Negative:
    a padding token, left out.  Beyond the cache: left out, and `check_status` raises.  The slots of one call must differ.
    A NaN stays NaN; a row with an infinity reads back as NaN throughout.  D a multiple of 8 up to 256."""
    _check_cache(k_codes, k_scale, v_codes, v_scale)
    _check_heads("k", k, k_codes)
    _check_heads("v", v, k_codes)
    T, H, D = k.shape
    pages, page_size = k_codes.shape[:2]
    if v.shape != k.shape or k_codes.shape[2:] != (H, D):
        raise ValueError(f"k and v must be [T, {k_codes.shape[2]}, {k_codes.shape[3]}], got {tuple(k.shape)} and {tuple(v.shape)}")
    _check_index("slots", slots, T, k)
    if T == 0:
        return
    c, s = k_codes.stride(), k_scale.stride()
    with _on_device(k.device):
        rc = _lib.load().rl_kv_cache_write_e4m3(
            k.data_ptr(), v.data_ptr(), slots.data_ptr(), slots.dtype == torch.int64, k_codes.data_ptr(), k_scale.data_ptr(),
            v_codes.data_ptr(), v_scale.data_ptr(), T, H, D, pages, page_size, k.stride(0), k.stride(1), v.stride(0),
            v.stride(1), c[0], c[1], c[2], s[0], s[1], s[2], _stream_ptr(k.device))
    _lib.check(rc, "rl_kv_cache_write_e4m3")
    _index_devices.add(k.device.index)


def kv_cache_read(k_codes: torch.Tensor, k_scale: torch.Tensor, v_codes: torch.Tensor, v_scale: torch.Tensor,
                  page_table: torch.Tensor, cu_seqlens: torch.Tensor, total: int, *,
                  out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The cache `kv_cache_write` filled, back as bf16(code * scale): (k, v) [total, H, D], the sequences packed one behind
    the other.  Token i of sequence b comes from page `page_table[b, i // page_size]` and goes to row cu_seqlens[b] + i.

    `page_table` [B, max_pages] int32, `cu_seqlens` [B + 1] int32, not decreasing, from 0; both stay on the device, so
    `total` is the caller's: rows from cu_seqlens[B] on are zero in a fresh output and left as they are in `out`,
    tokens beyond `total` are not read.  A page outside the cache (or a sequence longer than its table row) leaves the
    row as it is, unspecified in a fresh output, and `check_status` raises."""
    _check_cache(k_codes, k_scale, v_codes, v_scale)
    pages, page_size, H, D = k_codes.shape
    if (not isinstance(page_table, torch.Tensor) or page_table.dtype != torch.int32 or page_table.dim() != 2
            or page_table.device != k_codes.device or (page_table.shape[1] > 1 and page_table.stride(1) != 1)):
        raise ValueError("page_table must be [B, max_pages] int32, row-major, on the cache's device")
    B = page_table.shape[0]
    _check_index("cu_seqlens", cu_seqlens, B + 1, k_codes, (torch.int32,))
    if total < 0:
        raise ValueError("total must not be negative")
    if out is None:
        ko = torch.empty((total, H, D), dtype=torch.bfloat16, device=k_codes.device)
        vo = torch.empty((total, H, D), dtype=torch.bfloat16, device=k_codes.device)
    else:
        ko, vo = out
        _check_heads("out[0]", ko, k_codes)
        _check_heads("out[1]", vo, k_codes)
        if ko.shape != (total, H, D) or vo.shape != ko.shape:
            raise ValueError(f"out must be two tensors [{total}, {H}, {D}], got {tuple(ko.shape)} and {tuple(vo.shape)}")
    if total == 0:
        return ko, vo
    c, s = k_codes.stride(), k_scale.stride()
    with _on_device(k_codes.device):
        rc = _lib.load().rl_kv_cache_read_e4m3(
            k_codes.data_ptr(), k_scale.data_ptr(), v_codes.data_ptr(), v_scale.data_ptr(), page_table.data_ptr(),
            cu_seqlens.data_ptr(), ko.data_ptr(), vo.data_ptr(), total, out is None, B, page_table.shape[1],
            page_table.stride(0), H, D, pages, page_size, c[0], c[1], c[2], s[0], s[1], s[2], ko.stride(0), ko.stride(1),
            vo.stride(0), vo.stride(1), _stream_ptr(k_codes.device))
    _lib.check(rc, "rl_kv_cache_read_e4m3")
    _index_devices.add(k_codes.device.index)
    return ko, vo

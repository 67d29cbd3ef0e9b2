"""Operators on the heads of a projection's output: query/key norm with rotation, and the e4m3 cache of keys and values.

They stand between `rmsnorm_linear` (which writes q, k and v side by side in the rows of one matrix) and whatever
attention the caller runs; views into those rows go in as they are.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib
from .ops import _raw_stream, _status_devices

_BF16, _E4M3 = torch.bfloat16, torch.float8_e4m3fn


# The checks sit on the path of every decode step, whose kernels run for a few microseconds: each call makes them as one
# plain condition first and looks for what is wrong, and the words for it, only when that fails.

def _explain_heads(name: str, t: torch.Tensor, like: Optional[torch.Tensor] = None) -> None:
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


def _heads_ok(t: torch.Tensor, dev: int) -> bool:
    if not isinstance(t, torch.Tensor):
        return False
    strides = t.stride()
    return t.dtype is _BF16 and t.get_device() == dev and len(strides) == 3 and strides[2] == 1


def _index_ok(t: torch.Tensor, n: int, dev: int) -> bool:
    """A contiguous vector of n int64 or int32."""
    return (isinstance(t, torch.Tensor) and (t.dtype is torch.int64 or t.dtype is torch.int32) and t.get_device() == dev
            and t.shape == (n,) and t.is_contiguous())


def _gamma_ok(g: torch.Tensor, D: int, dev: int) -> bool:
    return (isinstance(g, torch.Tensor) and g.dtype is _BF16 and g.get_device() == dev and g.shape == (D,)
            and g.is_contiguous())


_NEEDS = "heads of a multiple of 8 channels up to 256, strides of multiples of 8 elements, 16-byte aligned"
_NEEDS_HALVES = _NEEDS + "; rotary_dim a multiple of 16 up to the head's"
_NEEDS_NEIGHBOURS = _NEEDS + "; rotary_dim a multiple of 8 up to the head's"


def _call(what: str, fn, args: bytes, dev: int, needs: str = _NEEDS) -> None:
    """The C function on the device, and on its current stream."""
    if dev == torch.cuda.current_device():
        rc = fn(args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            rc = fn(args, _raw_stream(dev))
    if rc:
        _lib.check(rc, f"{what} (needs {needs})" if rc in (_lib.RL_ERR_BAD_SHAPE, _lib.RL_ERR_ALIGNMENT) else what)
    _status_devices.add(dev)


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
    dev = q.get_device() if isinstance(q, torch.Tensor) else -1
    if dev < 0 or not _heads_ok(q, dev) or not _heads_ok(k, dev):
        _explain_heads("q", q)
        _explain_heads("k", k, q)
    T, Hq, D = q.shape
    Tk, Hk, Dk = k.shape
    if Tk != T or Dk != D:
        raise ValueError(f"q is [{T}, {Hq}, {D}]: k must be [{T}, Hk, {D}], got {tuple(k.shape)}")
    if (q_gamma is not None and not _gamma_ok(q_gamma, D, dev)) or (k_gamma is not None and not _gamma_ok(k_gamma, D, dev)):
        raise ValueError(f"q_gamma and k_gamma must be contiguous bf16 vectors of length D={D} on q's device")
    table_strides = table.stride() if isinstance(table, torch.Tensor) else ()
    if len(table_strides) != 2 or table_strides[1] != 1 or table.dtype is not torch.float32 or table.get_device() != dev:
        raise ValueError("table must be [positions, rotary_dim] fp32, row-major, on q's device")
    if not _index_ok(positions, T, dev):
        raise ValueError(f"positions must be a contiguous vector of {T} int64 or int32 on q's device")
    if out is None:
        qo = torch.empty_like(q, memory_format=torch.contiguous_format)
        ko = torch.empty_like(k, memory_format=torch.contiguous_format)
    else:
        qo, ko = out
        if not (_heads_ok(qo, dev) and _heads_ok(ko, dev)):
            _explain_heads("out[0]", qo, q)
            _explain_heads("out[1]", ko, q)
        if qo.shape != q.shape or ko.shape != k.shape:
            raise ValueError(f"out must be {tuple(q.shape)} and {tuple(k.shape)}, got {tuple(qo.shape)} and {tuple(ko.shape)}")
    if T == 0:
        return qo, ko
    P, rot = table.shape
    q_t, q_h, _ = q.stride()
    k_t, k_h, _ = k.stride()
    qo_t, qo_h, _ = qo.stride()
    ko_t, ko_h, _ = ko.stride()
    _call("rl_qk_norm_rope_bf16", _lib.load().rl_qk_norm_rope_bf16, _lib.QK_NORM_ROPE_ARGS.pack(
        q.data_ptr(), k.data_ptr(), 0 if q_gamma is None else q_gamma.data_ptr(), 0 if k_gamma is None else k_gamma.data_ptr(),
        table.data_ptr(), positions.data_ptr(), qo.data_ptr(), ko.data_ptr(), T, Hq, Hk, D, rot, P, table_strides[0], q_t, q_h,
        k_t, k_h, qo_t, qo_h, ko_t, ko_h, positions.dtype is torch.int64, interleaved, eps), dev,
        _NEEDS_NEIGHBOURS if interleaved else _NEEDS_HALVES)
    return qo, ko


def _check_cache(k_codes, k_scale, v_codes, v_scale) -> Tuple[int, tuple]:
    """The cache's device index, and its part of the C structures."""
    if (isinstance(k_codes, torch.Tensor) and isinstance(k_scale, torch.Tensor) and isinstance(v_codes, torch.Tensor)
            and isinstance(v_scale, torch.Tensor)):
        dev, shape, c, scales, s = k_codes.get_device(), k_codes.shape, k_codes.stride(), k_scale.shape, k_scale.stride()
        if (dev >= 0 and len(c) == 4 and c[3] == 1 and shape[:3] == scales and k_codes.dtype is _E4M3 and v_codes.dtype is _E4M3
                and k_scale.dtype is torch.float32 and v_scale.dtype is torch.float32 and v_codes.get_device() == dev
                and k_scale.get_device() == dev and v_scale.get_device() == dev and v_codes.shape == shape
                and v_codes.stride() == c and v_scale.shape == scales and v_scale.stride() == s):
            return dev, (k_codes.data_ptr(), v_codes.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), *shape, c[0], c[1],
                         c[2], *s)
    named = (("k_codes", k_codes), ("k_scale", k_scale), ("v_codes", v_codes), ("v_scale", v_scale))
    for name, t in named:
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
    for name, t in named:
        dtype, nd = (_E4M3, 4) if name.endswith("codes") else (torch.float32, 3)
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor (this operator has no CPU path)")
        if t.dtype != dtype or t.dim() != nd or t.device != k_codes.device:
            raise ValueError(f"{name} must be {nd}-D {dtype} on {k_codes.device}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    if k_codes.stride(3) != 1:
        raise ValueError("the codes' channels must be contiguous")
    if v_codes.shape != k_codes.shape or v_codes.stride() != k_codes.stride():
        raise ValueError("v_codes must have the shape and strides of k_codes")
    raise ValueError(f"k_scale and v_scale must both be {tuple(k_codes.shape[:3])}, with the same strides")


def kv_cache_write(k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, k_codes: torch.Tensor, k_scale: torch.Tensor,
                   v_codes: torch.Tensor, v_scale: torch.Tensor) -> None:
    """Write keys and values k, v [T, H, D] bf16 into a paged e4m3 cache, quantised as they are written with one scale per
    token and head: scale = max(max|x|, 2^-100) / 448, code = e4m3(448 x / max|x|), exactly rounded.

    Codes [pages, page_size, H, D] float8_e4m3fn and scales [pages, page_size, H] fp32, any strides with contiguous
    channels, the same for keys and values.  `slots` [T] int64 or int32: page * page_size + place in the page.  Negative:
    a padding token, left out.  Beyond the cache: left out, and `check_status` raises.  The slots of one call must differ.
    A NaN stays NaN; a row with an infinity reads back as NaN throughout.  D a multiple of 8 up to 256."""
    dev, cache = _check_cache(k_codes, k_scale, v_codes, v_scale)
    if not (_heads_ok(k, dev) and _heads_ok(v, dev)):
        _explain_heads("k", k, k_codes)
        _explain_heads("v", v, k_codes)
    T, H, D = k.shape
    if v.shape != k.shape or cache[6] != H or cache[7] != D:
        raise ValueError(f"k and v must be [T, {cache[6]}, {cache[7]}], got {tuple(k.shape)} and {tuple(v.shape)}")
    if not _index_ok(slots, T, dev):
        raise ValueError(f"slots must be a contiguous vector of {T} int64 or int32 on the cache's device")
    if T == 0:
        return
    k_t, k_h, _ = k.stride()
    v_t, v_h, _ = v.stride()
    _call("rl_kv_cache_write_e4m3", _lib.load().rl_kv_cache_write_e4m3, _lib.KV_CACHE_WRITE_ARGS.pack(
        *cache, k.data_ptr(), v.data_ptr(), slots.data_ptr(), T, k_t, k_h, v_t, v_h, slots.dtype is torch.int64), dev)


def kv_cache_read(k_codes: torch.Tensor, k_scale: torch.Tensor, v_codes: torch.Tensor, v_scale: torch.Tensor,
                  page_table: torch.Tensor, cu_seqlens: torch.Tensor, total: int, *,
                  out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The cache `kv_cache_write` filled, back as bf16(code * scale): (k, v) [total, H, D], the sequences packed one behind
    the other.  Token i of sequence b comes from page `page_table[b, i // page_size]` and goes to row cu_seqlens[b] + i.

    `page_table` [B, max_pages] int32, `cu_seqlens` [B + 1] int32, not decreasing, from 0; both stay on the device, so
    `total` is the caller's: rows from cu_seqlens[B] on are zero in a fresh output and left as they are in `out`,
    tokens beyond `total` are not read.  A row whose page lies outside the cache (or beyond its sequence's table row) is
    left as it is, zero in a fresh output, and `check_status` raises."""
    dev, cache = _check_cache(k_codes, k_scale, v_codes, v_scale)
    H, D = cache[6], cache[7]
    strides = page_table.stride() if isinstance(page_table, torch.Tensor) else ()
    if (len(strides) != 2 or page_table.dtype is not torch.int32 or page_table.get_device() != dev
            or (strides[1] != 1 and page_table.shape[1] > 1)):
        raise ValueError("page_table must be [B, max_pages] int32, row-major, on the cache's device")
    B, max_pages = page_table.shape
    if not _index_ok(cu_seqlens, B + 1, dev) or cu_seqlens.dtype is not torch.int32:
        raise ValueError(f"cu_seqlens must be a contiguous vector of {B + 1} int32 on the cache's device")
    if total < 0:
        raise ValueError("total must not be negative")
    if out is None:
        ko = k_codes.new_empty((total, H, D), dtype=_BF16)
        vo = torch.empty_like(ko)
    else:
        ko, vo = out
        if not (_heads_ok(ko, dev) and _heads_ok(vo, dev)):
            _explain_heads("out[0]", ko, k_codes)
            _explain_heads("out[1]", vo, k_codes)
        if ko.shape != (total, H, D) or vo.shape != ko.shape:
            raise ValueError(f"out must be two tensors [{total}, {H}, {D}], got {tuple(ko.shape)} and {tuple(vo.shape)}")
    if total == 0:
        return ko, vo
    ko_t, ko_h, _ = ko.stride()
    vo_t, vo_h, _ = vo.stride()
    _call("rl_kv_cache_read_e4m3", _lib.load().rl_kv_cache_read_e4m3, _lib.KV_CACHE_READ_ARGS.pack(
        *cache, page_table.data_ptr(), cu_seqlens.data_ptr(), ko.data_ptr(), vo.data_ptr(), total, out is None, B, max_pages,
        strides[0], ko_t, ko_h, vo_t, vo_h), dev)
    return ko, vo

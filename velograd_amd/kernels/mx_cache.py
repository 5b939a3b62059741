"""A paged cache of keys and values in the OCP MX block formats, and attention over it.

The formats are those of `fused_rmsnorm_residual_forward_mx`: elements of 4 bits (fmt "e2m1") or 8 bits
("e4m3") and one E8M0 power-of-two scale for 32 elements of a head vector.  A cache is an `MXCache`, or any
tuple of the same four tensors (one layer's slice of a larger allocation, say):

    k_codes, v_codes    [pages, kv_heads, page_size, head_dim / 2]  torch.float4_e2m1fn_x2, or
                        [pages, kv_heads, page_size, head_dim]      torch.float8_e4m3fn
    k_scales, v_scales  [pages, kv_heads, head_dim / 32, page_size] torch.float8_e8m0fnu

contiguous, on one ROCm device; head_dim 64, 128 or 256, page_size a power of two from 16.  A token's place
is its slot, page * page_size + place in the page; a sequence's pages are listed in a block table.

  mx_cache(pages, page_size, kv_heads, head_dim, fmt, device)         an empty cache
  rope_table(positions, head_dim, theta, device)                      cosines and sines for the rotation
  mx_cache_write(k, v, cache, slots)                                  quantise tokens into their slots
  rope_mx_cache_write(q, k, v, cos_sin, positions, cache, slots)      the same with q and k rotated
  mx_cache_read(cache, slots, dtype)                                  tokens back as (k, v)
  mx_cache_attention(q, cache, block_table, lengths, q_starts, ...)   attention of new tokens

Inputs are torch tensors on the cache's device; the calls run on torch's current stream of that device and
do not synchronise.  The reference has no counterpart (its paged cache, python/velograd/paged_attn.py,
holds full-precision lists on the host).
"""

from __future__ import annotations

import math
from typing import NamedTuple, Optional, Tuple, Union

import torch

from .. import _lib

__all__ = ["MXCache", "mx_cache", "rope_table", "mx_cache_write", "rope_mx_cache_write",
           "mx_cache_read", "mx_cache_attention"]

_CODE_DTYPES = {"e4m3": torch.float8_e4m3fn, "e2m1": torch.float4_e2m1fn_x2}
HEAD_DIMS = (64, 128, 256)
BLOCK = 32


class MXCache(NamedTuple):
    k_codes: torch.Tensor
    k_scales: torch.Tensor
    v_codes: torch.Tensor
    v_scales: torch.Tensor


def mx_cache(pages: int, page_size: int, kv_heads: int, head_dim: int, fmt: str = "e2m1",
             device: Optional[Union[str, torch.device]] = None) -> MXCache:
    """A cache of `pages` pages; every slot reads as zeros until it is written."""
    if fmt not in _CODE_DTYPES:
        raise ValueError(f"fmt must be 'e4m3' or 'e2m1', got {fmt!r}")
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"head_dim must be 64, 128 or 256, got {head_dim}")
    if not (16 <= page_size <= 32768) or page_size & (page_size - 1):
        raise ValueError(f"page_size must be a power of two from 16 to 32768, got {page_size}")
    if pages < 0 or kv_heads < 1:
        raise ValueError(f"invalid cache shape: pages={pages}, kv_heads={kv_heads}")
    device = torch.device("cuda") if device is None else torch.device(device)
    size = head_dim // 2 if fmt == "e2m1" else head_dim

    def bytes_(*shape):
        return torch.zeros(shape, dtype=torch.uint8, device=device)

    parts = []
    for _ in range(2):
        parts.append(bytes_(pages, kv_heads, page_size, size).view(_CODE_DTYPES[fmt]))
        parts.append(bytes_(pages, kv_heads, head_dim // BLOCK, page_size).view(torch.float8_e8m0fnu))
    return MXCache(*parts)


def rope_table(positions: int, head_dim: int, theta: float = 10000.0,
               device: Optional[Union[str, torch.device]] = None) -> torch.Tensor:
    """Cosines and sines of positions 0 .. positions - 1 for `rope_mx_cache_write`: float32
    [positions, head_dim], head_dim / 2 cosines of position * theta^(-2j / head_dim), then the sines.
    The angles are formed in 64 bits, so far positions keep their precision (fused_rope forms them in
    float32, as its reference does)."""
    if positions < 0 or head_dim < 2 or head_dim % 2 or not theta > 0:
        raise ValueError(f"invalid table: positions={positions}, head_dim={head_dim}, theta={theta}")
    device = torch.device("cuda") if device is None else torch.device(device)
    j = torch.arange(head_dim // 2, device=device, dtype=torch.float64)
    at = torch.arange(positions, device=device, dtype=torch.float64)
    angle = at[:, None] * float(theta) ** (-2.0 * j / head_dim)
    return torch.cat((angle.cos(), angle.sin()), -1).float()


class _Shape(NamedTuple):
    pages: int
    kv_heads: int
    page_size: int
    head_dim: int
    fmt: int


def _check_tensor(t, name: str, device: torch.device, dtype=None, dims: Optional[int] = None) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch tensor, got {type(t).__name__}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, the cache on {device}")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if dims is not None and t.dim() != dims:
        raise ValueError(f"{name} must have {dims} dimensions, got shape {tuple(t.shape)}")


def _check_cache(cache) -> Tuple[_Shape, torch.device]:
    if not isinstance(cache, tuple) or len(cache) != 4:
        raise TypeError("cache must be an MXCache: (k_codes, k_scales, v_codes, v_scales)")
    kc, ks, vc, vs = cache
    if not isinstance(kc, torch.Tensor):
        raise TypeError("the cache must be torch tensors")
    device = kc.device
    if kc.dtype == torch.float4_e2m1fn_x2:
        fmt, per = _lib.MX_E2M1, 2
    elif kc.dtype == torch.float8_e4m3fn:
        fmt, per = _lib.MX_E4M3, 1
    else:
        raise TypeError(f"k_codes must be float4_e2m1fn_x2 or float8_e4m3fn, got {kc.dtype}")
    _check_tensor(kc, "k_codes", device, None, 4)
    pages, kv_heads, page_size, size = kc.shape
    head_dim = size * per
    if head_dim not in HEAD_DIMS:
        raise ValueError(f"the cache's head_dim must be 64, 128 or 256, got {head_dim}")
    _check_tensor(vc, "v_codes", device, kc.dtype)
    scales = (pages, kv_heads, head_dim // BLOCK, page_size)
    for t, name in ((ks, "k_scales"), (vs, "v_scales")):
        _check_tensor(t, name, device, torch.float8_e8m0fnu)
        if tuple(t.shape) != scales:
            raise ValueError(f"{name} has shape {tuple(t.shape)}, expected {scales}")
    if vc.shape != kc.shape:
        raise ValueError(f"v_codes has shape {tuple(vc.shape)}, k_codes {tuple(kc.shape)}")
    if not all(t.is_contiguous() for t in cache):
        raise ValueError("the cache's tensors must be contiguous")
    return _Shape(pages, kv_heads, page_size, head_dim, fmt), device


def _check_rows(t, name: str, device: torch.device, heads: Optional[int], head_dim: int) -> int:
    _check_tensor(t, name, device, None, 3)
    if t.dtype not in _lib.TORCH_DTYPE_CODES:
        raise TypeError(f"{name}: unsupported dtype {t.dtype}; use float32, float16 or bfloat16")
    if t.shape[2] != head_dim or (heads is not None and t.shape[1] != heads):
        want = f"[tokens, {'heads' if heads is None else heads}, {head_dim}]"
        raise ValueError(f"{name} must be {want}, got {tuple(t.shape)}")
    return _lib.TORCH_DTYPE_CODES[t.dtype]


def _on_gpu(device: torch.device) -> None:
    if device.type != "cuda":
        raise TypeError(f"the cache is on {device}: these functions compute on a ROCm device only")


def _unit(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(-1) == 1 else t.contiguous()


def _stream(device: torch.device) -> int:
    from . import _stream as current
    return current(device)


def _fast(cache, *given):
    """The C++ fast path, where the arguments are tensors; it returns nothing for a call that it leaves to
    the general path below."""
    if isinstance(cache, tuple) and len(cache) == 4 and all(isinstance(t, torch.Tensor) for t in cache) \
            and all(isinstance(t, torch.Tensor) for t in given):
        return _lib.fastpath()
    return None


def _write(q, k, v, cos_sin, positions, cache, slots):
    fp = _fast(cache, k, v, slots, *(t for t in (q, cos_sin, positions) if t is not None))
    if fp is not None:
        done = fp.mx_write(q, k, v, cos_sin, positions, *cache, slots)
        if done:
            return done[0]
    shape, device = _check_cache(cache)
    code = _check_rows(k, "k", device, shape.kv_heads, shape.head_dim)
    _check_rows(v, "v", device, shape.kv_heads, shape.head_dim)
    if v.dtype != k.dtype:
        raise TypeError(f"v is {v.dtype}, k {k.dtype}")
    tokens = k.shape[0]
    if v.shape[0] != tokens:
        raise ValueError(f"v has {v.shape[0]} tokens, k {tokens}")
    _check_tensor(slots, "slots", device, torch.int64, 1)
    if slots.shape[0] != tokens:
        raise ValueError(f"slots has {slots.shape[0]} entries for {tokens} tokens")
    q_out = None
    max_positions = 0
    if positions is not None:
        _check_tensor(positions, "positions", device, torch.int64, 1)
        if positions.shape[0] != tokens:
            raise ValueError(f"positions has {positions.shape[0]} entries for {tokens} tokens")
        _check_tensor(cos_sin, "cos_sin", device, torch.float32, 2)
        if cos_sin.shape[1] != shape.head_dim:
            raise ValueError(f"cos_sin must be [positions, {shape.head_dim}], got {tuple(cos_sin.shape)}")
        positions, cos_sin = positions.contiguous(), cos_sin.contiguous()
        max_positions = cos_sin.shape[0]
    if q is not None:
        _check_rows(q, "q", device, None, shape.head_dim)
        if q.dtype != k.dtype:
            raise TypeError(f"q is {q.dtype}, k {k.dtype}")
        if q.shape[0] != tokens:
            raise ValueError(f"q has {q.shape[0]} tokens, k {tokens}")
    _on_gpu(device)
    if q is not None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=device)
    if tokens == 0:
        return q_out
    k, v, slots = _unit(k), _unit(v), slots.contiguous()
    q = None if q is None else _unit(q)
    with torch.cuda.device(device):
        rc = _lib.load().velograd_mx_cache_write(
            None if q is None else q.data_ptr(), k.data_ptr(), v.data_ptr(),
            None if q_out is None else q_out.data_ptr(),
            None if positions is None else cos_sin.data_ptr(),
            None if positions is None else positions.data_ptr(), slots.data_ptr(),
            *(t.data_ptr() for t in cache), tokens, 0 if q is None else q.shape[1], shape.kv_heads,
            shape.head_dim, 0 if q is None else q.stride(0), 0 if q is None else q.stride(1),
            k.stride(0), k.stride(1), v.stride(0), v.stride(1), max_positions, shape.pages,
            shape.page_size, code, shape.fmt, _stream(device))
    _lib.check(rc, "velograd_mx_cache_write")
    return q_out


def mx_cache_write(k: torch.Tensor, v: torch.Tensor, cache: MXCache, slots: torch.Tensor) -> None:
    """Quantise tokens' keys and values into their slots of the cache.

    k, v are [tokens, kv_heads, head_dim] (float32, float16 or bfloat16; slices of a larger projection are
    taken as they are), slots int64 [tokens].  A slot outside the cache (-1 marks padding rows) is not
    written.  The slots must differ: of two tokens with the same one, either may be kept, block by block.
    """
    _write(None, k, v, None, None, cache, slots)


def rope_mx_cache_write(q: Optional[torch.Tensor], k: torch.Tensor, v: torch.Tensor,
                        cos_sin: torch.Tensor, positions: torch.Tensor, cache: MXCache,
                        slots: torch.Tensor) -> Optional[torch.Tensor]:
    """Rotate q and k at the tokens' positions and write k and v into the cache, in one launch.

    The rotation is fused_rope's (rotate half, over the whole head_dim) at positions[t] (int64 [tokens]) of
    the table `cos_sin` (`rope_table`); the rotated k is rounded to its dtype and then quantised, so the
    cache holds what rotating first and mx_cache_write then would give.  Returns the rotated q
    [tokens, heads, head_dim] (of every token, those without a slot included), or None without q.  A
    position outside the table gives NaN.  k, v and slots as mx_cache_write.
    """
    if positions is None or cos_sin is None:
        raise TypeError("rope_mx_cache_write needs cos_sin and positions")
    return _write(q, k, v, cos_sin, positions, cache, slots)


def mx_cache_read(cache: MXCache, slots: torch.Tensor,
                  dtype: torch.dtype = torch.bfloat16) -> Tuple[torch.Tensor, torch.Tensor]:
    """The keys and values that the slots (int64 [tokens], any order) hold: (k, v), each
    [tokens, kv_heads, head_dim] in `dtype`.  Exact in float32 and bfloat16; float16 rounds, and overflows
    to infinity past its range.  A slot outside the cache reads as zeros."""
    fp = _fast(cache, slots)
    if fp is not None and dtype in _lib.TORCH_DTYPE_CODES:
        done = fp.mx_read(*cache, slots, _lib.TORCH_DTYPE_CODES[dtype])
        if done:
            return done[0], done[1]
    shape, device = _check_cache(cache)
    _check_tensor(slots, "slots", device, torch.int64, 1)
    if dtype not in _lib.TORCH_DTYPE_CODES:
        raise TypeError(f"unsupported dtype {dtype}; use float32, float16 or bfloat16")
    _on_gpu(device)
    out = (slots.shape[0], shape.kv_heads, shape.head_dim)
    k = torch.empty(out, dtype=dtype, device=device)
    v = torch.empty(out, dtype=dtype, device=device)
    if slots.shape[0] == 0:
        return k, v
    slots = slots.contiguous()
    with torch.cuda.device(device):
        rc = _lib.load().velograd_mx_cache_read(
            *(t.data_ptr() for t in cache), slots.data_ptr(), k.data_ptr(), v.data_ptr(), slots.shape[0],
            shape.kv_heads, shape.head_dim, shape.pages, shape.page_size, _lib.TORCH_DTYPE_CODES[dtype],
            shape.fmt, _stream(device))
    _lib.check(rc, "velograd_mx_cache_read")
    return k, v


def mx_cache_attention(q: torch.Tensor, cache: MXCache, block_table: torch.Tensor,
                       lengths: torch.Tensor, q_starts: Optional[torch.Tensor] = None,
                       scale: Optional[float] = None, causal: bool = True, return_lse: bool = False):
    """Attention of new tokens over all that their sequences hold in the cache (write them first).

    q is [tokens, heads, head_dim] (rotated as the keys are), heads a multiple of the cache's kv_heads:
    query head h reads kv head h // (heads // kv_heads).  block_table, int32 [sequences, pages], lists each
    sequence's pages in order, lengths, int32 [sequences], the tokens it holds, its new ones included.
    q_starts, int32 [sequences + 1] rising from 0, says which rows of q are its new tokens
    (q_starts[b] .. q_starts[b + 1] - 1; where it falls, rows are left unset); None: one each.  With causal, the i-th of n new tokens of a
    sequence of L sees the first L - n + i + 1 keys, without, all L.  scale defaults to
    1 / sqrt(head_dim).

    Returns out like q (contiguous), or (out, lse) with return_lse: lse float32 [tokens, heads], the log of
    the sum of exp(scale q.k) over the keys seen (to join with attention over other keys).  A row that sees
    no key, and a row of q past the last sequence, gives 0 and -inf.  Keys on a page outside the cache are
    not seen.

    Scores, sums and outputs are held in float32.  Of a call with many rows in bfloat16 the probabilities are
    rounded to bfloat16 (2^-8) before they multiply the values, elsewhere to 2^-16 or less.
    """
    fp = _fast(cache, q, block_table, lengths, *(() if q_starts is None else (q_starts,)))
    if fp is not None and q.dim() == 3:
        done = fp.mx_attention(q, *cache, block_table, lengths, q_starts,
                               1.0 / math.sqrt(max(1, q.shape[2])) if scale is None else float(scale),
                               bool(causal), bool(return_lse))
        if done:
            return (done[0], done[1]) if return_lse else done[0]
    shape, device = _check_cache(cache)
    code = _check_rows(q, "q", device, None, shape.head_dim)
    tokens, heads = q.shape[0], q.shape[1]
    if heads == 0 or heads % shape.kv_heads:
        raise ValueError(f"q has {heads} heads, not a multiple of the cache's {shape.kv_heads}")
    _check_tensor(block_table, "block_table", device, torch.int32, 2)
    _check_tensor(lengths, "lengths", device, torch.int32, 1)
    sequences = block_table.shape[0]
    if lengths.shape[0] != sequences:
        raise ValueError(f"lengths has {lengths.shape[0]} entries, block_table {sequences} rows")
    if q_starts is None:
        if tokens != sequences:
            raise ValueError(f"without q_starts every sequence has one token: q has {tokens} rows, "
                             f"block_table {sequences}")
    else:
        _check_tensor(q_starts, "q_starts", device, torch.int32, 1)
        if q_starts.shape[0] != sequences + 1:
            raise ValueError(f"q_starts has {q_starts.shape[0]} entries, expected {sequences + 1}")
        q_starts = q_starts.contiguous()
    scale = 1.0 / math.sqrt(shape.head_dim) if scale is None else float(scale)
    if not math.isfinite(scale):
        raise ValueError(f"scale must be finite, got {scale}")
    _on_gpu(device)
    out = torch.empty(q.shape, dtype=q.dtype, device=device)
    lse = torch.empty((tokens, heads), dtype=torch.float32, device=device) if return_lse else None
    if tokens == 0:
        return (out, lse) if return_lse else out
    q, block_table, lengths = _unit(q), _unit(block_table), lengths.contiguous()
    lib = _lib.load()
    with torch.cuda.device(device):
        index = device.index if device.index is not None else torch.cuda.current_device()
        size = lib.velograd_mx_cache_attention_workspace_bytes(
            tokens, sequences, heads, shape.kv_heads, shape.head_dim, block_table.shape[1],
            shape.page_size, 0 if q_starts is None else 1, code, shape.fmt, index)
        ws = torch.empty(size, dtype=torch.uint8, device=device) if size else None
        rc = lib.velograd_mx_cache_attention(
            q.data_ptr(), *(t.data_ptr() for t in cache), block_table.data_ptr(), lengths.data_ptr(),
            None if q_starts is None else q_starts.data_ptr(), out.data_ptr(),
            None if lse is None else lse.data_ptr(), None if ws is None else ws.data_ptr(), size, tokens,
            sequences, heads, shape.kv_heads, shape.head_dim, q.stride(0), q.stride(1),
            block_table.stride(0), block_table.shape[1], shape.pages, shape.page_size, scale,
            1 if causal else 0, code, shape.fmt, _stream(device))
    _lib.check(rc, "velograd_mx_cache_attention")
    return (out, lse) if return_lse else out

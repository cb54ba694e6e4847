"""Rows held in 4 bits: the K/V cache of a decode, attention over it, and linears with 4-bit weights.

A row is cut into groups of 64 channels.  ``z`` is the least value of a group and ``s = bf16((most - least) / 15)``; a
channel is the code ``n`` (0 to 15) nearest to ``(x - z) / s``, of two equally near ones the even one, and stands for
``s n + z``.  A group without spread (or with one whose ``s`` is below the least normal bf16) has ``s = 0`` and reads back
as ``z``; a group with a NaN or an infinity, or with a spread beyond fp32, reads back as NaN throughout.  Inputs count as
bf16: wider ones are rounded to it first.

:class:`Q4Rows` holds rows of ``K`` channels at the width ``W`` = 64 for ``K <= 64``, else ``K`` rounded up to a multiple of
128 (padding has ``s = z = 0``): ``codes`` uint8 ``[..., W / 2]`` and ``affine`` bf16 ``[..., W / 64, 2]`` = ``(s, z)``, 36
bytes for 64 channels.  Eight channels make a 32-bit word, channel ``i`` of the eight at nibble ``i // 2 + 4 * (i % 2)``;
words of a block of 128 alternate between its two groups (word ``2 g + h``: channels ``64 h + 8 g ..``).

Nothing here has a gradient: a call that would record one, of rows, queries or the pairs of 4-bit rows, or that would carry a
forward-mode tangent, is refused.  :func:`quantize_rows_q4` makes plain data, also of what requires a gradient.  On a CUDA
device bf16 tensors go to the kernels of ``csrc/quant4.cu``, ``csrc/decode_q4.cu`` and ``csrc/linear_q4.cu``; on the CPU the
restatements below run, in any dtype.
"""

from __future__ import annotations

import functools
import math
from contextlib import nullcontext
from typing import NamedTuple

import torch
import torch.nn.functional as F
from torch.autograd import forward_ad

from research_b200.errors import KernelError
from research_b200.ops import native

GROUP = 64


class _CodesAndPairs(NamedTuple):
    codes: torch.Tensor
    affine: torch.Tensor


class Q4Rows(_CodesAndPairs):
    """Rows in 4 bits: ``codes`` uint8 ``[..., W / 2]``, ``affine`` bf16 ``[..., W / 64, 2]`` (scale, least value).

    ``channels`` is how many of the W a row has, where that is known: :func:`quantize_rows_q4` and :func:`empty_rows` say so,
    and a call with rows of another number is refused.  Rows that are put together from tensors without it (None) are only
    held against their width."""

    channels: int | None = None

    def __new__(cls, codes: torch.Tensor, affine: torch.Tensor, channels: int | None = None):
        self = tuple.__new__(cls, (codes, affine))
        if channels is not None:
            self.channels = channels
        return self


def row_width(channels: int) -> int:
    """Channels that a row of ``channels`` is stored as."""

    return GROUP if channels <= GROUP else -(-channels // (2 * GROUP)) * 2 * GROUP


def empty_rows(*shape: int, channels: int, device=None) -> Q4Rows:
    """``Q4Rows`` of zeros: ``shape`` rows of ``channels`` channels (a cache: ``[B, pages, Hkv, page_rows]`` rows of D)."""

    width = row_width(channels)
    return Q4Rows(torch.zeros(*shape, width // 2, dtype=torch.uint8, device=device),
                  torch.zeros(*shape, width // GROUP, 2, dtype=torch.bfloat16, device=device), channels)


# --------------------------------------------------------------------------------------------------
# plain restatements
# --------------------------------------------------------------------------------------------------
_NIBBLE = tuple(i // 2 + 4 * (i % 2) for i in range(8))


def quantize_rows_reference(x: torch.Tensor) -> Q4Rows:
    channels, width = x.shape[-1], row_width(x.shape[-1])
    groups = F.pad(x.to(torch.bfloat16), (0, width - channels)).unflatten(-1, (-1, GROUP)).double()
    real = (torch.arange(width, device=x.device) < channels).view(-1, GROUP)
    some = real[:, :1]
    z = torch.where(some, groups.masked_fill(~real, math.inf).amin(-1, keepdim=True), 0.0)
    spread = torch.where(some, groups.masked_fill(~real, -math.inf).amax(-1, keepdim=True), 0.0) - z
    s = torch.where(spread <= torch.finfo(torch.float32).max, spread / 15.0, math.nan).to(torch.bfloat16).double()
    s = torch.where(s < torch.finfo(torch.bfloat16).tiny, 0.0, s)
    coded = real & (s > 0)
    step = torch.where(s > 0, s, 1.0)
    d = groups - z
    k = torch.floor(d / step)
    k = torch.where((k + 1.5) * step <= d, k + 1, torch.where((k - 0.5) * step > d, k - 1, k))
    above = d - (k + 0.5) * step                        # exact next to 0; what d itself lost decides where it is 0
    back = d - groups
    lost = (groups - (d - back)) - (z + back)
    up = (above > 0) | ((above == 0) & ((lost > 0) | ((lost == 0) & (k % 2 == 1))))
    n = torch.where(coded, (k + up).clamp(0, 15), 0.0).to(torch.uint8)
    pair = 2 if width > GROUP else 1
    words = n.unflatten(-2, (-1, pair)).unflatten(-1, (8, 8)).transpose(-3, -2)
    nibbles = words[..., [_NIBBLE.index(k) for k in range(8)]]
    return Q4Rows((nibbles[..., 0::2] | (nibbles[..., 1::2] << 4)).flatten(-4),
                  torch.cat([s, z], dim=-1).to(torch.bfloat16), channels)


def dequantize_rows_reference(rows: Q4Rows, channels: int, dtype: torch.dtype = torch.float32) -> torch.Tensor:
    width = rows.codes.shape[-1] * 2
    b = rows.codes.unflatten(-1, (-1, 8, 2 if width > GROUP else 1, 4))
    nibbles = torch.stack([b & 15, b >> 4], dim=-1).flatten(-2)
    n = nibbles[..., list(_NIBBLE)].transpose(-3, -2).flatten(-2).flatten(-3, -2)              # [..., groups, 64]
    a = rows.affine.float()
    return (n.float() * a[..., :1] + a[..., 1:]).flatten(-2)[..., :channels].to(dtype)


def _pool_index(pool: Q4Rows, T: int, start: torch.Tensor | None):
    """Page and row in it of positions ``start[b] + t``, and which of them the cache has."""

    B, pages, _, page_rows, _ = pool.codes.shape
    at = torch.arange(T, device=pool.codes.device).expand(B, T)
    if start is not None:
        at = at + start.to(at.device).long()[:, None]
    inside = (at >= 0) & (at < pages * page_rows)
    return at, inside


def kv_write_paged_q4_reference(k, v, k_pool: Q4Rows, v_pool: Q4Rows, start=None) -> None:
    at, inside = _pool_index(k_pool, k.shape[1], start)
    b = torch.arange(k.shape[0], device=at.device)[:, None].expand_as(at)[inside]
    at, page_rows = at[inside], k_pool.codes.shape[3]
    for x, pool in ((k, k_pool), (v, v_pool)):
        held = quantize_rows_reference(x)
        pool.codes[b, at // page_rows, :, at % page_rows] = held.codes[inside]
        pool.affine[b, at // page_rows, :, at % page_rows] = held.affine[inside]


def kv_read_paged_q4_reference(k_pool: Q4Rows, v_pool: Q4Rows, rows: int, start=None, *, channels: int,
                               dtype: torch.dtype = torch.bfloat16):
    at, inside = _pool_index(k_pool, rows, start)
    b = torch.arange(at.shape[0], device=at.device)[:, None].expand_as(at)
    _, pages, heads, page_rows, _ = k_pool.codes.shape
    if pages * page_rows == 0:
        return tuple(torch.zeros(*at.shape, heads, channels, dtype=dtype, device=at.device) for _ in range(2))
    at = at.clamp(0, pages * page_rows - 1)
    out = []
    for pool in (k_pool, v_pool):
        held = Q4Rows(*(t[b, at // page_rows, :, at % page_rows] for t in pool))
        out.append(dequantize_rows_reference(held, channels, dtype).masked_fill(~inside[:, :, None, None], 0.0))
    return tuple(out)


def decode_attention_paged_q4_reference(q: torch.Tensor, k_pool: Q4Rows, v_pool: Q4Rows, lengths: torch.Tensor,
                                        lo: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    B, Hq, D = q.shape
    k, v = (dequantize_rows_reference(pool, D).permute(0, 2, 1, 3, 4).flatten(2, 3) for pool in (k_pool, v_pool))
    Hkv = k.shape[1]
    s = torch.einsum("bhgd,bhrd->bhgr", q.float().view(B, Hkv, Hq // Hkv, D), k) * (D ** -0.5 if scale is None else scale)
    at = torch.arange(k.shape[2], device=q.device)
    seen = at < lengths.long()[:, None]
    if lo is not None:
        seen = seen & (at >= lo.long()[:, None])
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    none = ~seen.any(-1)
    p = torch.softmax(s.masked_fill(none[:, None, None, None], 0.0), dim=-1)
    # what a masked row holds counts for nothing, whatever it is; a row of probability 0 counts
    o = torch.einsum("bhgr,bhrd->bhgd", p, v.masked_fill(~seen[:, None, :, None], 0.0))
    return o.masked_fill(none[:, None, None, None], 0.0).reshape(B, Hq * D).to(q.dtype)


def linear_q4_reference(x: torch.Tensor, w: Q4Rows) -> torch.Tensor:
    _check_channels("linear_q4", w, x.shape[-1])
    return F.linear(x.float(), dequantize_rows_reference(w, x.shape[-1])).to(x.dtype)


# --------------------------------------------------------------------------------------------------
# argument checks
# --------------------------------------------------------------------------------------------------
def _no_gradient(what: str, *tensors: torch.Tensor) -> None:
    if torch.is_grad_enabled():
        for t in tensors:
            if t.requires_grad:
                raise KernelError(f"{what} has no gradient: call it under torch.no_grad() or on detached tensors")
    if forward_ad._current_level >= 0:                  # which torch.no_grad() does not end
        for t in tensors:
            if forward_ad.unpack_dual(t).tangent is not None:
                raise KernelError(f"{what} has no forward-mode derivative: call it on primal tensors")


def _same_device(what: str, first: torch.Tensor, *others: torch.Tensor | None) -> None:
    at = first.get_device()                             # -1: the CPU
    for t in others:
        if t is not None and t.get_device() != at:
            raise KernelError(f"{what}: all tensors have to be on {first.device}, got one on {t.device}")


_SAME = nullcontext()


def _on(t: torch.Tensor):
    """Launches go to the current stream of the tensors' own device."""

    return _SAME if t.get_device() == torch._C._cuda_getDevice() else torch.cuda.device(t.device)


def _check_channels(what: str, rows: Q4Rows, channels: int) -> None:
    if rows.channels is not None and rows.channels != channels:
        raise KernelError(f"{what}: rows of {channels} channels do not go with 4-bit rows of {rows.channels} channels")


def _check_rows(what: str, rows: Q4Rows, channels: int) -> None:
    _check_channels(what, rows, channels)
    _check_width(what, rows, channels)


def _check_width(what: str, rows: Q4Rows, channels: int) -> None:
    width = row_width(channels)
    codes, affine = rows
    *shape, half = codes.shape
    if (half * 2 == width and affine.shape == (*shape, width // GROUP, 2) and codes.dtype is torch.uint8
            and affine.dtype is torch.bfloat16 and codes.is_contiguous() and affine.is_contiguous()
            and codes.get_device() == affine.get_device()):
        return
    if codes.dtype != torch.uint8 or affine.dtype != torch.bfloat16:
        raise KernelError(f"{what}: 4-bit rows are uint8 codes and bf16 pairs, got {codes.dtype} and {affine.dtype}")
    if codes.shape[-1] * 2 != width or affine.shape != (*codes.shape[:-1], width // GROUP, 2):
        raise KernelError(f"{what}: rows of {channels} channels are codes [..., {width // 2}] with pairs [..., "
                          f"{width // GROUP}, 2], got {tuple(codes.shape)} and {tuple(affine.shape)}")
    if not codes.is_contiguous() or not affine.is_contiguous():
        raise KernelError(f"{what}: codes and pairs have to be contiguous")
    _same_device(what, codes, affine)


def _check_pools(what: str, k_pool: Q4Rows, v_pool: Q4Rows, B: int, Hkv: int | None, D: int) -> tuple[int, int, int]:
    (kc, ka), (vc, va) = k_pool, v_pool
    shape, pairs, width, at = kc.shape, ka.shape, row_width(D), kc.get_device()
    if not (len(shape) == 5 and shape[4] * 2 == width and pairs == (*shape[:4], width // GROUP, 2) and vc.shape == shape
            and va.shape == pairs and kc.dtype is vc.dtype is torch.uint8 and ka.dtype is va.dtype is torch.bfloat16
            and kc.is_contiguous() and ka.is_contiguous() and vc.is_contiguous() and va.is_contiguous()
            and at == ka.get_device() == vc.get_device() == va.get_device()):
        for pool in (k_pool, v_pool):                   # says what is wrong
            if pool.codes.dim() != 5:
                raise KernelError(f"{what}: a cache has codes [B, pages, Hkv, page_rows, D / 2], got "
                                  f"{tuple(pool.codes.shape)}")
            _check_width(what, pool, D)
        if shape != vc.shape:
            raise KernelError(f"{what}: the K and the V cache must have one shape, got {tuple(shape)} and {tuple(vc.shape)}")
        _same_device(what, kc, vc)
    seqs, pages, heads, page_rows, _ = shape
    if seqs != B or (Hkv is not None and heads != Hkv):
        raise KernelError(f"{what}: a cache {tuple(shape)} does not hold {B} sequences"
                          + ("" if Hkv is None else f" of {Hkv} heads"))
    if pages * page_rows > 2 ** 31 - 1:
        raise KernelError(f"{what}: a sequence has at most 2^31 - 1 rows, got {pages} pages of {page_rows}")
    return pages, heads, page_rows


def _per_sequence(what: str, name: str, t: torch.Tensor | None, B: int, like: torch.Tensor) -> torch.Tensor | None:
    if t is None or (t.dtype is torch.int32 and t.dim() == 1 and t.shape[0] == B and t.is_contiguous()
                     and t.get_device() == like.get_device()):
        return t
    if t.dim() != 1 or t.shape[0] != B or t.dtype not in (torch.int32, torch.int64):
        raise KernelError(f"{what}: {name} is an int32 or int64 tensor [{B}], got {tuple(t.shape)} {t.dtype}")
    if t.get_device() != like.get_device():
        _same_device(what, like, t)
    return t.clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32) if t.dtype == torch.int64 else t.contiguous()


def _head_dim(what: str, D: int) -> None:
    if D not in (64, 128):
        raise KernelError(f"{what} supports head_dim 64 and 128 on a CUDA device, got {D}")


# --------------------------------------------------------------------------------------------------
# whole rows
# --------------------------------------------------------------------------------------------------
@torch.no_grad()
def quantize_rows_q4(x: torch.Tensor) -> Q4Rows:
    """4-bit form of the rows of ``x [..., K]`` (for weights, once; fp32 values are rounded to bf16 first)."""

    if x.dim() < 1 or x.shape[-1] < 1 or not x.is_floating_point():
        raise KernelError(f"quantize_rows_q4 needs rows of floating point numbers, got {tuple(x.shape)} {x.dtype}")
    _no_gradient("quantize_rows_q4", x)
    if not x.is_cuda:
        return quantize_rows_reference(x)
    x2 = x.to(torch.bfloat16).reshape(-1, x.shape[-1])
    if x2.stride(1) != 1:
        x2 = x2.contiguous()
    width = row_width(x.shape[-1])
    codes = torch.empty(*x.shape[:-1], width // 2, dtype=torch.uint8, device=x.device)
    affine = torch.empty(*x.shape[:-1], width // GROUP, 2, dtype=torch.bfloat16, device=x.device)
    if x2.shape[0]:
        with _on(x):
            native._check((native._lib or native.load()).b200_q4_quantize_rows(
                x2.data_ptr(), x2.stride(0), codes.data_ptr(), affine.data_ptr(), x2.shape[0], x2.shape[1],
                native._stream()), "b200_q4_quantize_rows")
    return Q4Rows(codes, affine, x.shape[-1])


def dequantize_rows_q4(rows: Q4Rows, channels: int, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """Values ``[..., channels]`` of 4-bit rows, rounded once to ``dtype`` (bf16 on a CUDA device)."""

    _check_rows("dequantize_rows_q4", rows, channels)
    _no_gradient("dequantize_rows_q4", rows.affine)
    if not rows.codes.is_cuda:
        return dequantize_rows_reference(rows, channels, dtype)
    if dtype != torch.bfloat16:
        raise KernelError(f"dequantize_rows_q4 writes bf16 on a CUDA device, got {dtype}")
    return _expand(rows)[..., :channels]


def _expand(rows: Q4Rows) -> torch.Tensor:
    width = rows.codes.shape[-1] * 2
    out = torch.empty(*rows.codes.shape[:-1], width, dtype=torch.bfloat16, device=rows.codes.device)
    if out.numel():
        with _on(out):
            native._check((native._lib or native.load()).b200_q4_dequantize_rows(
                rows.codes.data_ptr(), rows.affine.data_ptr(), out.data_ptr(), out.numel() // width, width,
                native._stream()), "b200_q4_dequantize_rows")
    return out


# --------------------------------------------------------------------------------------------------
# cache
# --------------------------------------------------------------------------------------------------
def _copied(t: torch.Tensor) -> torch.Tensor:
    """A dense copy on an address of its own, also of what is dense already."""

    return t.clone(memory_format=torch.contiguous_format)


def _heads_apart(t: torch.Tensor, Hkv: int, D: int) -> tuple[torch.Tensor, int, int]:
    """``t [B, T, Hkv, D]`` as the kernel reads it (a copy where heads are not D apart or rows off 16 bytes), with the strides
    of rows and sequences."""

    batch, row, head, one = t.stride()
    if one == 1 and head == D and row % 8 == 0 and batch % 8 == 0 and t.data_ptr() % 16 == 0:
        return t, row, batch
    return _copied(t), Hkv * D, t.shape[1] * Hkv * D


def kv_write_paged_q4(k: torch.Tensor, v: torch.Tensor, k_pool: Q4Rows, v_pool: Q4Rows,
                      start: torch.Tensor | None = None) -> None:
    """Quantise ``k`` / ``v`` ``[B, T, Hkv, D]`` into rows ``start[b] .. start[b] + T - 1`` of head-major paged caches of 4-bit
    rows ``[B, pages, Hkv, page_rows, D]`` (``start`` int32 or int64 ``[B]``; None: rows ``0 .. T - 1``, which then have to
    fit).  One token per sequence is ``T = 1`` with ``start`` the positions.  Rows that the cache does not have are left
    out; all others keep what they held."""

    what = "kv_write_paged_q4"
    if k.dim() != 4 or k.shape != v.shape or k.dtype != v.dtype or not k.is_floating_point():
        raise KernelError(f"{what}: k and v are [B, T, Hkv, D] of one shape and type, got {tuple(k.shape)} {k.dtype} and "
                          f"{tuple(v.shape)} {v.dtype}")
    B, T, Hkv, D = k.shape
    _check_channels(what, k_pool, D)
    _check_channels(what, v_pool, D)
    pages, _, page_rows = _check_pools(what, k_pool, v_pool, B, Hkv, D)
    _same_device(what, k, v, k_pool.codes)
    start = _per_sequence(what, "start", start, B, k)
    if start is None and T > pages * page_rows:
        raise KernelError(f"{what}: {T} rows do not fit a cache of {pages} pages of {page_rows}")
    _no_gradient(what, k, v, k_pool.affine, v_pool.affine)
    if k.numel() == 0:
        return
    (k_codes, k_affine), (v_codes, v_affine) = k_pool, v_pool
    k_codes_at, k_affine_at, v_codes_at, v_affine_at = (k_codes.data_ptr(), k_affine.data_ptr(), v_codes.data_ptr(),
                                                        v_affine.data_ptr())
    # both are written at once
    if abs(k_codes_at - v_codes_at) < k_codes.numel() or abs(k_affine_at - v_affine_at) < 2 * k_affine.numel():
        raise KernelError(f"{what}: the K and the V cache share memory")
    if not k.is_cuda:
        return kv_write_paged_q4_reference(k, v, k_pool, v_pool, start)
    _head_dim(what, D)
    if k.dtype != torch.bfloat16:
        raise KernelError(f"{what} quantises bf16 rows on a CUDA device, got {k.dtype}")
    k, k_row, k_batch = _heads_apart(k, Hkv, D)
    v, v_row, v_batch = _heads_apart(v, Hkv, D)
    with _on(k):
        native._check((native._lib or native.load()).b200_q4_kv_write(
            k.data_ptr(), v.data_ptr(), k_row, k_batch, v_row, v_batch, k_codes_at, k_affine_at, v_codes_at, v_affine_at,
            native._ptr(start), B, T, Hkv, D, pages, page_rows, native._stream()), "b200_q4_kv_write")


def kv_read_paged_q4(k_pool: Q4Rows, v_pool: Q4Rows, rows: int, start: torch.Tensor | None = None, *,
                     head_dim: int | None = None, dtype: torch.dtype = torch.bfloat16):
    """Rows ``start[b] .. start[b] + rows - 1`` (None: from 0) of both caches as dense ``(k, v)`` ``[B, rows, Hkv, D]`` bf16.
    Rows that the cache does not have read as zeros.  ``head_dim`` is D where it is not the stored width, ``dtype`` another
    result type (both on the CPU only)."""

    what = "kv_read_paged_q4"
    D = k_pool.codes.shape[-1] * 2 if head_dim is None else head_dim
    if head_dim is not None:                            # else all that is stored, padding too
        _check_channels(what, k_pool, D)
        _check_channels(what, v_pool, D)
    B = k_pool.codes.shape[0]
    pages, Hkv, page_rows = _check_pools(what, k_pool, v_pool, B, None, D)
    start = _per_sequence(what, "start", start, B, k_pool.codes)
    if rows < 0:
        raise KernelError(f"{what}: rows must not be negative, got {rows}")
    _no_gradient(what, k_pool.affine, v_pool.affine)
    if not k_pool.codes.is_cuda:
        return kv_read_paged_q4_reference(k_pool, v_pool, rows, start, channels=D, dtype=dtype)
    _head_dim(what, D)
    if dtype != torch.bfloat16:
        raise KernelError(f"{what} writes bf16 on a CUDA device, got {dtype}")
    k, v = k_pool.affine.new_empty(B, rows, Hkv, D), v_pool.affine.new_empty(B, rows, Hkv, D)
    if k.numel() and pages * page_rows:
        with _on(k):
            native._check((native._lib or native.load()).b200_q4_kv_read(
                k.data_ptr(), v.data_ptr(), k_pool.codes.data_ptr(), k_pool.affine.data_ptr(),
                v_pool.codes.data_ptr(), v_pool.affine.data_ptr(), native._ptr(start), B, rows, Hkv, D, pages,
                page_rows, native._stream()), "b200_q4_kv_read")
    else:
        k.zero_(), v.zero_()
    return k, v


def decode_attention_paged_q4(q: torch.Tensor, k_pool: Q4Rows, v_pool: Q4Rows, lengths: torch.Tensor,
                              lo: torch.Tensor | None = None, scale: float | None = None) -> torch.Tensor:
    """Attention of one query token per sequence, ``q [B, Hq, D]``, over rows ``lo[b] <= r < lengths[b]`` of caches of 4-bit
    rows ``[B, pages, Hkv, page_rows, D]`` (``lengths``, ``lo`` int32 or int64 ``[B]``; rows beyond the cache do not count, a
    sequence without a row gets zeros).  Up to 8 query heads share a K/V head.  Returns ``[B, Hq * D]`` in q's type.  On a CUDA
    device weights of up to 2^8 times values are added up in fp32 before the division: V of up to 2^95 in size cannot overflow
    it in a cache of 2^24 rows."""

    what = "decode_attention_paged_q4"
    if q.dim() != 3 or not q.is_floating_point():
        raise KernelError(f"{what}: q is [B, Hq, D], got {tuple(q.shape)} {q.dtype}")
    B, Hq, D = q.shape
    _check_channels(what, k_pool, D)
    _check_channels(what, v_pool, D)
    pages, Hkv, page_rows = _check_pools(what, k_pool, v_pool, B, None, D)
    if Hkv == 0 or Hq % Hkv:
        raise KernelError(f"{what}: {Hq} query heads do not share {Hkv} K/V heads evenly")
    _same_device(what, q, k_pool.codes)
    lengths, lo = _per_sequence(what, "lengths", lengths, B, q), _per_sequence(what, "lo", lo, B, q)
    if lengths is None:
        raise KernelError(f"{what} needs the lengths of the sequences")
    scale = float(D ** -0.5 if scale is None else scale)
    if not math.isfinite(scale):
        raise KernelError(f"{what}: the scale is a finite number, got {scale}")
    _no_gradient(what, q, k_pool.affine, v_pool.affine)
    if not q.is_cuda:
        return decode_attention_paged_q4_reference(q, k_pool, v_pool, lengths, lo, scale)
    _head_dim(what, D)
    if q.dtype != torch.bfloat16 or Hq // Hkv > 8:
        raise KernelError(f"{what} supports bf16 queries and up to 8 query heads to a K/V head on a CUDA device, got "
                          f"{q.dtype}, Hq={Hq}, Hkv={Hkv}")
    per_row, per_head, one = q.stride()
    if one != 1 or per_head != D or per_row % 8 or q.data_ptr() % 16:
        q, per_row = _copied(q), Hq * D
    out = q.new_empty(B, Hq * D)
    if out.numel() == 0:
        return out
    if pages * page_rows == 0:
        return out.zero_()
    lib = native._lib or native.load()
    with _on(q):
        runs = _attention_runs(B, Hkv, pages * page_rows, q.get_device())
        slots = (runs + B * Hkv) * (Hq // Hkv)
        parts = q.new_empty(slots * (D + 2), dtype=torch.float32)
        native._check(lib.b200_q4_decode_attn(
            q.data_ptr(), per_row, k_pool.codes.data_ptr(), k_pool.affine.data_ptr(), v_pool.codes.data_ptr(),
            v_pool.affine.data_ptr(), lengths.data_ptr(), native._ptr(lo), out.data_ptr(), parts.data_ptr(),
            parts.data_ptr() + 4 * slots * D, B, Hq, Hkv, D, pages, page_rows, runs,
            scale, native._stream()), "b200_q4_decode_attn")
    native.LAUNCHES += 1                                # _check counts one launch; joining the runs is the second
    return out


@functools.lru_cache(maxsize=4096)
def _attention_runs(B: int, Hkv: int, rows: int, device: int) -> int:
    return native.load().b200_q4_decode_attn_runs(B, Hkv, rows)


# --------------------------------------------------------------------------------------------------
# linear
# --------------------------------------------------------------------------------------------------
def linear_q4(x: torch.Tensor, w: Q4Rows) -> torch.Tensor:
    """``y = x W^T`` for ``x [..., K]`` and weights ``w`` of ``N`` 4-bit rows of K channels; ``y [..., N]`` in x's type.  Up to
    8 or 16 rows of x (:func:`few_rows`) the weights count as they are; for more rows each counts as a
    bf16.  An infinity or a NaN in a row of x leaves no number in its results."""

    what = "linear_q4"
    if x.dim() < 1 or not x.is_floating_point() or x.shape[-1] < 1:
        raise KernelError(f"{what}: x is [..., K], got {tuple(x.shape)} {x.dtype}")
    K = x.shape[-1]
    if w.codes.dim() != 2:
        raise KernelError(f"{what}: weights are [N, K] as 4-bit rows, got codes {tuple(w.codes.shape)}")
    _check_rows(what, w, K)
    _same_device(what, x, w.codes)
    _no_gradient(what, x, w.affine)
    if not x.is_cuda:
        return linear_q4_reference(x, w)
    if x.dtype != torch.bfloat16:
        raise KernelError(f"{what} takes bf16 rows on a CUDA device, got {x.dtype}")
    N = w.codes.shape[0]
    x2 = x if x.dim() == 2 else x.reshape(-1, K)
    rows = x2.shape[0]
    if rows == 0 or N == 0:
        return torch.empty(*x.shape[:-1], N, dtype=x.dtype, device=x.device)
    with _on(x):
        slices = linear_slices(rows, N, K)
        out = _coded_linear(x2, w, rows, N, K, slices) if slices else _expanded_linear(x2, w)
    return out if x2 is x else out.view(*x.shape[:-1], N)


def _coded_linear(x: torch.Tensor, w: Q4Rows, rows: int, N: int, K: int, slices: int) -> torch.Tensor:
    few = rows <= few_rows(N, K)
    if not few:
        x = _rows_on_16_bytes(x)
    ld, one = x.stride()
    if one != 1:
        x, ld = x.contiguous(), K
    out = x.new_empty(rows, N)
    native._check((native._lib or native.load()).b200_q4_linear(
        x.data_ptr(), ld, w.codes.data_ptr(), w.affine.data_ptr(), out.data_ptr(), N, rows, N, K, 0 if few else slices,
        native.status_word(x.device).data_ptr(), native._stream()), "b200_q4_linear")
    return out


def few_rows(n: int, k: int) -> int:
    """Rows of x up to which a linear of ``n`` x ``k`` weights multiplies the codes themselves; more rows have bf16 weights,
    expanded on their way or before.

    A cluster of up to 8 blocks has registers for 8 rows of 32768 channels or 16 of 16384; more than 8 rows are better off
    there where they need no cluster or have few weights: 16 rows of 11264 x 2048 take 8.4 us against 10 to 12, of 2048 x 5632
    7.3 against 9.0, of 28672 x 4096 35 against 27, of 4096 x 14336 27 against 17."""

    if k <= GROUP:
        return 64
    if k <= 2048 or (k <= 16384 and n * k <= 2 ** 24):
        return 16
    return 8 if k <= 32768 else 0


def _rows_on_16_bytes(x: torch.Tensor) -> torch.Tensor:
    """``x [rows, K]`` as tensor maps take it: dense rows that start on 16 bytes (a copy where they do not)."""

    if x.stride(1) == 1 and x.stride(0) % 8 == 0 and x.stride(0) >= x.shape[1] and x.data_ptr() % 16 == 0:
        return x
    return F.pad(x, (0, -x.shape[1] % 8))[:, :x.shape[1]] if x.shape[1] % 8 else _copied(x)


@functools.lru_cache(maxsize=4096)
def linear_slices(rows: int, n: int, k: int, sms: int = 148) -> int:
    """Slices of K (1, 2, 4 or 8 blocks of a cluster) for a product of more than :func:`few_rows` rows with 4-bit weights: the
    count of least estimated time, or 0 where that is to expand the weights first.

    A step of 128 channels takes a tile of 128 weights and 64 rows 0.34 us (0.36 with 128 rows) by itself, twice that in
    pairs on an SM (up to 64 rows), and clusters of 4 and 8 find no room on some of the SMs.  Expanding first takes 1.5 us and
    0.48 us a million weights, and the GEMM then 0.4 us per 64 channels of its tiles of 128 x 256.  Measured 1 / 2 / 4 / 8 slices,
    expanded: 32 rows, 2048 x 2048 9.4 / 7.2 / 5.9 / 11.0 us, 11264 x 2048 9.8 / 10.8 / 13.1 / 21.1 us, 28672 x 4096 27.7 / 32.4 /
    38.7 / 59.7 us; 128 rows, 2048 x 2048 11.1 / 8.7 / 7.5 / 16.5, 17.6 us; 777 rows, 2048 x 5632 22.8 / 29.8 / 44.7 / 80.6, 38.2 us; 1024
    rows, 4096 x 4096 36.9 / 52.3 / 81.1 / 172.9, 36.2 us; 2048 rows, 2048 x 2048 23.9 / 38.7 / 66.3 / 156.5, 19.0 us."""

    if rows <= few_rows(n, k):
        return 1
    if k <= GROUP:
        return 0
    stages = -(-k // 256)
    best, best_cost = 1, float("inf")
    for s, exchange, full in ((1, 0.0, 1.0), (2, 0.3, 1.0), (4, 0.5, 0.9), (8, 1.2, 0.75)):
        if s > 1 and stages < s:
            break
        per, blocks = -(-stages // s), -(-n // 128) * -(-rows // (64 if rows <= 64 else 128)) * s
        if rows <= 64 and blocks > sms:
            waves = math.ceil(blocks / (2 * sms))
            cost = 4.4 + 1.36 * per * waves + (waves - 1) * 6.0 + exchange
        else:
            waves = math.ceil(blocks / (sms * full))
            cost = (4.6 + 0.68 * per if rows <= 64 else 5.0 + 0.72 * per) * waves + exchange + (1.7 if rows > 64 else 0.0)
        if cost < best_cost:
            best, best_cost = s, cost
    if rows <= 64:
        return best
    waves = math.ceil(-(-n // 256) * -(-rows // 128) / sms)
    return best if best_cost < 3.5 + 0.48e-6 * n * k + waves * (2.0 + 0.4 * -(-k // 64)) else 0


def _expanded_linear(x: torch.Tensor, w: Q4Rows) -> torch.Tensor:
    (rows, K), N = x.shape, w.codes.shape[0]
    full = _expand(w)[:, :K]
    ld = -(-N // 8) * 8
    out = torch.empty(rows, ld, dtype=torch.bfloat16, device=x.device)
    native.gemm(_rows_on_16_bytes(x), full, out=out[:, :N])
    return out if ld == N else out[:, :N].contiguous()

"""Paged key / value cache for serving with PoPE, and attention over it.

A cache holds the rows of many sequences in pages of ``page_size`` slots; a page table says which pages a sequence has,
in order, so sequences grow without copies and may share pages (a common prompt).  Keys are stored transformed,
K_hat = [softplus(k) cos t, softplus(k) sin t, pass-through dims] with t = freqs + bias: a token's softplus, sine and
cosine are computed once, when it is written, and positions may be anything, since attention needs the new rows'
angles only.  ``quantized`` caches hold e4m3 codes times a power of two per (token, head) instead of 16-bit values.

  paged_cache_write            new k, v rows into their slots
  paged_cache_read             rows out of their slots: k_hat as ``apply_pope_to_qk`` gives it, and v
  paged_flash_attn_with_pope   attention of new rows (a single token, a chunk, a whole prompt) over all that their
                               sequences have cached, the new rows included

New rows are (batch, heads, n, dim), or (batch, n, heads, dim) with ``head_dimension_at_first=False``: sequence b's
are batch entry b.  Packed calls have batch 1 and ``cu_seqlens`` (batch + 1 ascending numbers; of rows that numbers
which descend leave out or count twice nothing is said): rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1 belong to sequence b.
``lengths`` counts a sequence's tokens with the new ones; row i of n stands at position lengths - n + i, and
``pos_emb`` has one row of angles per new row, ``pope(positions)``.  Lengths beyond the slots of a page table's row
count as those slots: the new rows then take the last ones.  A serving step is a write and an attention call with the
same page table, lengths and cu_seqlens.

Rows without a slot (negative positions, packed rows outside every sequence, page numbers outside the cache) are not
written, read as zeros and never seen; rows that see no key, or none with a score above -inf, give 0.  Nothing
synchronises or reads lengths on the host, so a captured graph replays with new page tables and lengths in the same
tensors.  There is no gradient.

No counterpart in the reference, whose decoding caches plain k and transforms all of it for every token
(PoPE_pytorch/attention.py:75-145).  GPU caches run the HIP kernels (csrc/paged_*.hip), CPU caches the torch
computation below, on the same page layout.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F
from torch import Tensor
from torch.autograd import forward_ad

from . import _lib

_DTYPES = (torch.bfloat16, torch.float16)
_BLOCK = 32   # slots per block of a page


def exists(v):
    return v is not None


def _unit(t: Tensor) -> Tensor:
    """The tensor with unit stride in its last dim (contiguous() keeps odd strides of extents of 1)."""
    return t if t.stride(-1) == 1 else t.clone(memory_format=torch.contiguous_format)


def _v_tiles(D: int) -> int:
    """Value columns held, in tiles of 16: 32, 64, 96, 128 or 256."""
    return next(t for t, most in ((2, 32), (4, 64), (6, 96), (8, 128), (16, 256)) if D <= most)


def _k_steps(D: int, R: int) -> int:
    """Key columns held, in steps of 32: enough for D + R out of 1, 3/2 and 2 times the value columns."""
    tiles = _v_tiles(D)
    need = (D + R + 31) // 32
    return next(s for s in (tiles // 2, (3 * tiles + 3) // 4, tiles) if need <= s)


class PagedPoPECache:
    """Pages of expanded key rows and value rows of ``heads`` kv heads.

    ``dim`` 1 to 256, ``rotate_dim`` 0 (plain attention) to ``dim``, ``page_size`` a power of two from 32 to 1024,
    ``dtype`` bf16 or fp16 (of k, v, q and the outputs).  ``quantized``: e4m3 codes times a power of two per row, half
    the memory; values that are not finite are held as NaN.  ``k_pages``, ``v_pages`` and ``scales`` are the pages, in the kernels' operand order."""

    def __init__(self, num_pages: int, *, heads: int, dim: int, rotate_dim: int = 0, page_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16, quantized: bool = False, device=None):
        if num_pages < 1 or heads < 1:
            raise ValueError(f"num_pages and heads must be at least 1, got {num_pages} and {heads}")
        if not 1 <= dim <= 256:
            raise ValueError(f"dim must be 1 to 256, got {dim}")
        if not 0 <= rotate_dim <= dim:
            raise ValueError(f"rotate_dim must be 0 to dim {dim}, got {rotate_dim}")
        if page_size < 32 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"page_size must be a power of two from 32 to 1024, got {page_size}")
        if dtype not in _DTYPES:
            raise TypeError(f"dtype must be bfloat16 or float16, got {dtype}")
        self.num_pages, self.heads, self.dim, self.rotate_dim = num_pages, heads, dim, rotate_dim
        self.page_size, self.dtype, self.quantized = page_size, dtype, bool(quantized)
        blocks = page_size // _BLOCK
        held = torch.uint8 if quantized else dtype
        self.k_pages = torch.zeros(num_pages, heads, blocks, _BLOCK * 32 * _k_steps(dim, rotate_dim), dtype=held, device=device)
        self.v_pages = torch.zeros(num_pages, heads, blocks, _BLOCK * 16 * _v_tiles(dim), dtype=held, device=device)
        self.scales = torch.zeros((num_pages, heads, blocks, 2 * _BLOCK) if quantized else (0,), dtype=torch.uint8, device=device)

    @property
    def device(self) -> torch.device:
        return self.k_pages.device

    @property
    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.k_pages, self.v_pages, self.scales))

    def __repr__(self):
        return (f"PagedPoPECache(num_pages={self.num_pages}, heads={self.heads}, dim={self.dim}, rotate_dim={self.rotate_dim}, "
                f"page_size={self.page_size}, dtype={self.dtype}, quantized={self.quantized}, device='{self.device}')")


# ---------------------------------------------------------------- arguments

def _check_seqs(cache: PagedPoPECache, page_table: Tensor, lengths: Tensor, cu_seqlens: Optional[Tensor]):
    if page_table.ndim != 2 or page_table.shape[0] < 1 or page_table.shape[1] < 1:
        raise ValueError(f"page_table must be (batch, pages) with at least one of each, got {tuple(page_table.shape)}")
    B = page_table.shape[0]
    if tuple(lengths.shape) != (B,):
        raise ValueError(f"lengths {tuple(lengths.shape)} must be (batch,) = ({B},)")
    if exists(cu_seqlens) and tuple(cu_seqlens.shape) != (B + 1,):
        raise ValueError(f"cu_seqlens {tuple(cu_seqlens.shape)} must be (batch + 1,) = ({B + 1},)")
    out = []
    for t, name in ((page_table, "page_table"), (lengths, "lengths"), (cu_seqlens, "cu_seqlens")):
        if exists(t):
            if t.dtype not in (torch.int32, torch.int64):
                raise TypeError(f"{name} must be int32 or int64, got {t.dtype}")
            if t.device != cache.device:
                raise RuntimeError(f"pope_amd paged cache: {name} on {t.device}, the cache on {cache.device}")
            if t.dtype != torch.int32:
                # out of range is no slot, never another one: what int32 cannot hold stays out of range
                t = t.clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32)
            t = _unit(t)
        out.append(t)
    return out


def _check_rows(cache: PagedPoPECache, t: Tensor, name: str, B: int, heads: Optional[int], packed: bool):
    if t.ndim != 4:
        raise ValueError(f"{name} must be 4-D, got {tuple(t.shape)}")
    if t.dtype != cache.dtype:
        raise TypeError(f"{name} of dtype {t.dtype}, the cache has {cache.dtype}")
    if t.device != cache.device:
        raise RuntimeError(f"pope_amd paged cache: {name} on {t.device}, the cache on {cache.device}")
    if t.shape[0] != (1 if packed else B):
        raise ValueError(f"{name} {tuple(t.shape)} must have batch {1 if packed else B}" + (" (cu_seqlens: packed rows)" if packed else ""))
    if t.shape[3] != cache.dim or (heads is not None and t.shape[1] != heads):
        raise ValueError(f"{name} {tuple(t.shape)} (batch, heads, n, dim) does not fit a cache of {cache.heads} heads of dim {cache.dim}")
    return _unit(t)


def _check_pos_emb(cache: PagedPoPECache, pos_emb, batch: int, n: int):
    """freqs as (1 or batch, n, R) fp32 with unit feature stride, bias as (1 or heads, R); None, None without rotation."""
    R = cache.rotate_dim
    if R == 0:
        if exists(pos_emb):
            raise ValueError("pos_emb given, but the cache has rotate_dim 0")
        return None, None
    if not exists(pos_emb):
        raise ValueError(f"the cache has rotate_dim {R}: pos_emb is needed")
    freqs, bias = pos_emb
    if freqs.ndim == 2:
        freqs = freqs.unsqueeze(0)
    if freqs.ndim != 3 or freqs.shape[2] != R or freqs.shape[1] != n or freqs.shape[0] not in (1, batch):
        raise ValueError(f"freqs {tuple(pos_emb[0].shape)} must have one row of {R} per new row: ({n}, {R}) or ({batch}, {n}, {R})")
    if exists(bias):
        if bias.ndim == 1:
            bias = bias.unsqueeze(0)
        if bias.ndim != 2 or bias.shape[1] != R or bias.shape[0] not in (1, cache.heads):
            raise ValueError(f"bias {tuple(pos_emb[1].shape)} must be (1 or {cache.heads}, {R})")
    out = []
    for t, name in ((freqs, "freqs"), (bias, "bias")):
        if exists(t):
            if t.device != cache.device:
                raise RuntimeError(f"pope_amd paged cache: {name} on {t.device}, the cache on {cache.device}")
            t = _unit(t.float())
        out.append(t)
    return out


def _no_grad(*ts):
    ts = [t for t in ts if exists(t)]
    if (torch.is_grad_enabled() and any(t.requires_grad for t in ts)) or (
            not torch.compiler.is_compiling() and any(exists(forward_ad.unpack_dual(t).tangent) for t in ts)):
        raise RuntimeError("pope_amd paged cache: no gradient is defined; call it under torch.no_grad() or on detached tensors")


# ---------------------------------------------------------------- ops (tracing); eager calls take the same native calls

@torch.library.custom_op("pope_amd::paged_write", mutates_args=("k_pages", "v_pages", "scales"), device_types="cuda")
def paged_write_op(k: Tensor, v: Tensor, freqs: Optional[Tensor], bias: Optional[Tensor], k_pages: Tensor, v_pages: Tensor,
                   scales: Tensor, page_table: Tensor, lengths: Tensor, cu_seqlens: Optional[Tensor], page_size: int) -> None:
    _lib.host().paged_write(k, v, freqs, bias, k_pages, v_pages, scales, page_table, lengths, cu_seqlens, page_size)


@paged_write_op.register_fake
def _(k, v, freqs, bias, k_pages, v_pages, scales, page_table, lengths, cu_seqlens, page_size):
    return None


@torch.library.custom_op("pope_amd::paged_read", mutates_args=(), device_types="cuda")
def paged_read_op(k_pages: Tensor, v_pages: Tensor, scales: Tensor, page_table: Tensor, lengths: Tensor, cu_seqlens: Optional[Tensor],
                  n: int, dim: int, rotate_dim: int, page_size: int, half: bool, head_first: bool) -> tuple[Tensor, Tensor]:
    return _lib.host().paged_read(k_pages, v_pages, scales, page_table, lengths, cu_seqlens, n, dim, rotate_dim, page_size, half, head_first)


@paged_read_op.register_fake
def _(k_pages, v_pages, scales, page_table, lengths, cu_seqlens, n, dim, rotate_dim, page_size, half, head_first):
    B, H = 1 if exists(cu_seqlens) else page_table.shape[0], k_pages.shape[1]
    dt = torch.float16 if half else torch.bfloat16
    if head_first:
        return tuple(k_pages.new_empty((B, H, n, c), dtype=dt) for c in (dim + rotate_dim, dim))
    return tuple(k_pages.new_empty((B, n, H, c), dtype=dt).transpose(1, 2) for c in (dim + rotate_dim, dim))


@torch.library.custom_op("pope_amd::paged_attn", mutates_args=(), device_types="cuda")
def paged_attn_op(q: Tensor, freqs: Optional[Tensor], k_pages: Tensor, v_pages: Tensor, scales: Tensor, page_table: Tensor,
                  lengths: Tensor, cu_seqlens: Optional[Tensor], page_size: int, causal: bool, softmax_scale: float,
                  with_lse: bool) -> tuple[Tensor, Tensor]:
    return _lib.host().paged_attn(q, freqs, k_pages, v_pages, scales, page_table, lengths, cu_seqlens, page_size, causal, softmax_scale, with_lse)


@paged_attn_op.register_fake
def _(q, freqs, k_pages, v_pages, scales, page_table, lengths, cu_seqlens, page_size, causal, softmax_scale, with_lse):
    o = torch.empty_like(q)
    o = o if o.stride(-1) == 1 else q.new_empty(q.shape)   # rows_like of csrc_torch/pope_host.cpp
    return o, q.new_empty(q.shape[:3] if with_lse else (0,), dtype=torch.float32)


# ---------------------------------------------------------------- public calls

def paged_cache_write(cache: PagedPoPECache, k: Tensor, v: Tensor, pos_emb, page_table: Tensor, lengths: Tensor, *,
                      cu_seqlens: Optional[Tensor] = None, head_dimension_at_first: bool = True) -> None:
    """Writes the new rows k, v (batch, heads, n, dim) into their slots (see the module's text).

    ``pos_emb``: (freqs, bias) of the new rows, ``pope(positions)``, or None for a cache without rotated dims.
    ``page_table`` (sequences, pages), ``lengths`` (sequences,) with the new rows counted.  Slots of other tokens are
    not touched.  Two rows must not share a slot."""
    on_gpu = cache.k_pages.is_cuda
    freqs, bias = pos_emb if exists(pos_emb) else (None, None)
    eager = on_gpu and _lib.eager(k, v, freqs, bias, cache.k_pages, page_table, lengths, cu_seqlens)
    if eager and _lib.host().paged_write_eager(k, v, freqs, bias, cache.k_pages, cache.v_pages, cache.scales, page_table, lengths, cu_seqlens,
                                               cache.page_size, cache.dim, cache.rotate_dim, cache.dtype == torch.float16, head_dimension_at_first):
        return
    # conversions, what is wrong with the call, tracing
    if not head_dimension_at_first:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    packed = exists(cu_seqlens)
    page_table, lengths, cu_seqlens = _check_seqs(cache, page_table, lengths, cu_seqlens)
    B = page_table.shape[0]
    k = _check_rows(cache, k, "k", B, cache.heads, packed)
    v = _check_rows(cache, v, "v", B, cache.heads, packed)
    if v.shape != k.shape:
        raise ValueError(f"v {tuple(v.shape)} must match k {tuple(k.shape)}")
    freqs, bias = _check_pos_emb(cache, pos_emb, k.shape[0], k.shape[2])
    if exists(freqs) and not exists(bias):
        raise ValueError("pos_emb needs its bias: keys are stored with it")
    _no_grad(k, v, freqs, bias)
    if not on_gpu:
        return _write_torch(cache, k, v, freqs, bias, page_table, lengths, cu_seqlens)
    args = (k, v, freqs, bias, cache.k_pages, cache.v_pages, cache.scales, page_table, lengths, cu_seqlens, cache.page_size)
    if eager:
        _lib.host().paged_write(*args)
    else:
        paged_write_op(*args)


def paged_cache_read(cache: PagedPoPECache, page_table: Tensor, lengths: Tensor, n: int, *, cu_seqlens: Optional[Tensor] = None,
                     head_dimension_at_first: bool = True) -> tuple[Tensor, Tensor]:
    """The last n cached rows of every sequence, (k_hat, v) of (batch, heads, n, dim + rotate_dim) and (.., dim) in the
    cache's dtype; packed: n rows in all, of sequence b its last cu_seqlens[b + 1] - cu_seqlens[b].  k_hat has the
    column order of ``apply_pope_to_qk``.  Rows without a slot are zeros."""
    on_gpu = cache.k_pages.is_cuda
    eager = on_gpu and _lib.eager(cache.k_pages, page_table, lengths, cu_seqlens)
    if eager:
        r = _lib.host().paged_read_eager(cache.k_pages, cache.v_pages, cache.scales, page_table, lengths, cu_seqlens, n, cache.dim, cache.rotate_dim,
                                         cache.page_size, cache.dtype == torch.float16, head_dimension_at_first)
        if exists(r):
            return r
    page_table, lengths, cu_seqlens = _check_seqs(cache, page_table, lengths, cu_seqlens)
    if n < 0:
        raise ValueError(f"n must not be negative, got {n}")
    if not on_gpu:
        k, v = _read_torch(cache, page_table, lengths, cu_seqlens, n)
    else:
        args = (cache.k_pages, cache.v_pages, cache.scales, page_table, lengths, cu_seqlens, n, cache.dim, cache.rotate_dim,
                cache.page_size, cache.dtype == torch.float16, head_dimension_at_first)
        k, v = _lib.host().paged_read(*args) if eager else paged_read_op(*args)
    return (k, v) if head_dimension_at_first else (k.transpose(1, 2), v.transpose(1, 2))


def paged_flash_attn_with_pope(q: Tensor, cache: PagedPoPECache, pos_emb, page_table: Tensor, lengths: Tensor, *,
                               cu_seqlens: Optional[Tensor] = None, causal: bool = True, softmax_scale: Optional[float] = None,
                               return_lse: bool = False, head_dimension_at_first: bool = True):
    """Attention of the new rows q (batch, query heads, n, dim) over their sequences' cached rows, the new ones included
    (they are written before).  Query head h reads kv head h % heads.  ``causal``: a row sees positions up to its own
    (bottom-right aligned: the last row sees everything), otherwise all of its sequence.  ``pos_emb``: the new rows'
    (freqs, bias); bias is not read.  ``return_lse``: also the scores' log-sum-exp, fp32 (batch, query heads, n).  Sums are
    fp32: a row's values times their keys' number stay below 2^119."""
    on_gpu = cache.k_pages.is_cuda
    scale = cache.dim ** -0.5 if softmax_scale is None else float(softmax_scale)
    freqs = pos_emb[0] if exists(pos_emb) else None
    eager = on_gpu and _lib.eager(q, freqs, cache.k_pages, page_table, lengths, cu_seqlens)
    if eager:
        r = _lib.host().paged_attn_eager(q, freqs, cache.k_pages, cache.v_pages, cache.scales, page_table, lengths, cu_seqlens, cache.page_size,
                                         cache.dim, cache.rotate_dim, cache.dtype == torch.float16, head_dimension_at_first, causal, scale, return_lse)
        if exists(r):
            return r if return_lse else r[0]
    if not head_dimension_at_first:
        q = q.transpose(1, 2)
    packed = exists(cu_seqlens)
    page_table, lengths, cu_seqlens = _check_seqs(cache, page_table, lengths, cu_seqlens)
    q = _check_rows(cache, q, "q", page_table.shape[0], None, packed)
    if q.shape[1] < 1 or q.shape[1] % cache.heads:
        raise ValueError(f"{q.shape[1]} query heads must be a multiple of the cache's {cache.heads}")
    freqs, _ = _check_pos_emb(cache, pos_emb, q.shape[0], q.shape[2])
    _no_grad(q, freqs)
    if not on_gpu:
        o, lse = _attend_torch(cache, q, freqs, page_table, lengths, cu_seqlens, causal, scale)
    else:
        args = (q, freqs, cache.k_pages, cache.v_pages, cache.scales, page_table, lengths, cu_seqlens, cache.page_size, bool(causal),
                scale, bool(return_lse))
        o, lse = _lib.host().paged_attn(*args) if eager else paged_attn_op(*args)
    if not head_dimension_at_first:
        o = o.transpose(1, 2)
    return (o, lse) if return_lse else o


# ---------------------------------------------------------------- CPU caches: the same pages, torch operators

def _segments(B: int, lengths: Tensor, cu_seqlens: Optional[Tensor], n: int, capacity: int):
    """(sequence, batch entry, first row, rows, length) of every sequence."""
    lens = [min(max(int(x), 0), capacity) for x in lengths]
    if not exists(cu_seqlens):
        return [(b, b, 0, n, lens[b]) for b in range(B)]
    cu = [min(max(int(x), 0), n) for x in cu_seqlens]
    return [(b, 0, cu[b], max(cu[b + 1] - cu[b], 0), lens[b]) for b in range(B)]


def _k_offsets(q8: bool, cols: int) -> Tensor:
    """(32, cols) element offsets of a block's key rows (paged_k_off of csrc/paged_index.hpp)."""
    t, e = torch.arange(_BLOCK)[:, None], torch.arange(cols)[None, :]
    step, half, lane, j = e // 32, t // 16, t % 16 + 16 * (e % 32 // 8), e % 8
    return ((step * 64 + lane) * 2 + half) * 8 + j if q8 else ((step * 2 + half) * 64 + lane) * 8 + j


def _v_offsets(q8: bool, cols: int) -> Tensor:
    t, d = torch.arange(_BLOCK)[:, None], torch.arange(cols)[None, :]
    tile, lane, j = d // 16, d % 16 + 16 * (t % 16 // 4), 4 * (t // 16) + t % 4
    return ((tile // 2 * 64 + lane) * 2 + tile % 2) * 8 + j if q8 else (tile * 64 + lane) * 8 + j


def _slots(cache: PagedPoPECache, table_row: Tensor, pos: Tensor):
    """Block number (over all pages' blocks of one head), slot in it, and whether there is one."""
    page = table_row[(pos // cache.page_size).clamp(0, table_row.numel() - 1)].long()
    ok = (pos >= 0) & (page >= 0) & (page < cache.num_pages)
    return page.clamp(0, cache.num_pages - 1), (pos.clamp_min(0) % cache.page_size) // _BLOCK, pos.clamp_min(0) % _BLOCK, ok


def _row_index(cache: PagedPoPECache, slots, offsets: Tensor, per_block: int) -> Tensor:
    """(heads, rows, columns) flat element indexes."""
    page, blk, t, _ = slots
    h = torch.arange(cache.heads)[:, None]
    block = (page * cache.heads + h) * (cache.page_size // _BLOCK) + blk
    return block[..., None] * per_block + offsets[t][None]


def _quantize(x: Tensor):
    """e4m3 codes and exponent bytes of rows."""
    finite = x.isfinite()
    amax = torch.where(finite, x.abs(), 0.0).amax(-1)
    mant, e = torch.frexp(amax)
    e = torch.where(mant <= 0.875, e - 9, e - 8).clamp(-126, 126)
    e = torch.where(amax == 0, -126, e)
    y = torch.where(finite, x * ((127 - e).int() << 23).view(torch.float32)[..., None], float("nan"))
    return y.to(torch.float8_e4m3fn).view(torch.uint8), (e + 127).to(torch.uint8)


def _write_torch(cache, k, v, freqs, bias, page_table, lengths, cu_seqlens):
    R, q8 = cache.rotate_dim, cache.quantized
    ko, vo = _k_offsets(q8, 32 * _k_steps(cache.dim, R)), _v_offsets(q8, 16 * _v_tiles(cache.dim))
    for b, batch, row0, n, length in _segments(len(page_table), lengths, cu_seqlens, k.shape[2], page_table.shape[1] * cache.page_size):
        pos = length - n + torch.arange(n)
        *slots, ok = _slots(cache, page_table[b], pos)
        slots = [s[ok] for s in slots] + [None]
        kr, vr = (t[batch, :, row0:row0 + n][:, ok].float() for t in (k, v))
        if R:
            f = freqs[batch if freqs.shape[0] > 1 else 0, row0:row0 + n][ok].double()
            angle = f + bias.double()[:, None, :]
            m = F.softplus(kr[..., :R])
            kr = torch.cat((m * angle.cos().float(), m * angle.sin().float(), kr[..., R:]), -1)
        kr, vr = F.pad(kr, (0, ko.shape[1] - kr.shape[-1])), F.pad(vr, (0, vo.shape[1] - vr.shape[-1]))
        ki, vi = _row_index(cache, slots, ko, ko.numel()), _row_index(cache, slots, vo, vo.numel())
        if q8:
            st = torch.arange(_BLOCK)
            si = _row_index(cache, slots, torch.stack((st // 4 * 8 + st % 4, st // 4 * 8 + 4 + st % 4), -1), 2 * _BLOCK)
            kr, ke = _quantize(kr)
            vr, ve = _quantize(vr)
            cache.scales.view(-1)[si] = torch.stack((ke, ve), -1)
        cache.k_pages.view(-1)[ki] = kr.to(cache.k_pages.dtype)
        cache.v_pages.view(-1)[vi] = vr.to(cache.v_pages.dtype)


def _load_torch(cache, table_row, pos):
    """K_hat (columns [cos | sin | rest]) and V rows at positions pos, (heads, rows, columns) fp32, zeros without a slot."""
    q8, E = cache.quantized, cache.dim + cache.rotate_dim
    slots = _slots(cache, table_row, pos)
    ko, vo = _k_offsets(q8, 32 * _k_steps(cache.dim, cache.rotate_dim)), _v_offsets(q8, 16 * _v_tiles(cache.dim))
    k = cache.k_pages.view(-1)[_row_index(cache, slots, ko[:, :E], ko.numel())]
    v = cache.v_pages.view(-1)[_row_index(cache, slots, vo[:, :cache.dim], vo.numel())]
    if q8:
        st = torch.arange(_BLOCK)
        si = _row_index(cache, slots, torch.stack((st // 4 * 8 + st % 4, st // 4 * 8 + 4 + st % 4), -1), 2 * _BLOCK)
        e = cache.scales.view(-1)[si].double() - 127
        k, v = (t.view(torch.float8_e4m3fn).float() * torch.exp2(e[..., i, None]).float() for i, t in enumerate((k, v)))
    ok = slots[3][None, :, None]
    return k.float().where(ok, 0.0), v.float().where(ok, 0.0), slots[3]


def _interleave(k: Tensor, R: int) -> Tensor:
    return torch.cat((torch.stack((k[..., :R], k[..., R:2 * R]), -1).flatten(-2), k[..., 2 * R:]), -1)


def _read_torch(cache, page_table, lengths, cu_seqlens, n):
    batch = 1 if exists(cu_seqlens) else len(page_table)
    k = torch.zeros(batch, cache.heads, n, cache.dim + cache.rotate_dim, dtype=cache.dtype)
    v = torch.zeros(batch, cache.heads, n, cache.dim, dtype=cache.dtype)
    most = torch.finfo(cache.dtype).max
    for b, at, row0, m, length in _segments(len(page_table), lengths, cu_seqlens, n, page_table.shape[1] * cache.page_size):
        kr, vr, _ = _load_torch(cache, page_table[b], length - m + torch.arange(m))
        for out, rows in ((k, _interleave(kr, cache.rotate_dim)), (v, vr)):
            # a 16-bit page has nothing beyond its type, and an 8-bit one no infinity: its codes may round up past the largest
            rows = rows.clamp(-most, most) if cache.quantized else rows
            out[at, :, row0:row0 + m] = rows.to(cache.dtype)
    return k, v


def _attend_torch(cache, q, freqs, page_table, lengths, cu_seqlens, causal, scale):
    R, Hk = cache.rotate_dim, cache.heads
    G, N = q.shape[1] // Hk, q.shape[2]
    o = torch.zeros_like(q)
    lse = torch.full(q.shape[:3], float("-inf"))
    for b, at, row0, n, length in _segments(len(page_table), lengths, cu_seqlens, N, page_table.shape[1] * cache.page_size):
        if n == 0 or length == 0:
            continue
        kr, vr, ok = _load_torch(cache, page_table[b], torch.arange(length))
        x = q[at, :, row0:row0 + n].float()
        if R:
            f = freqs[at if freqs.shape[0] > 1 else 0, row0:row0 + n].double()
            m = F.softplus(x[..., :R])
            x = torch.cat((m * f.cos().float(), m * f.sin().float(), x[..., R:]), -1)
        sc = torch.matmul(x.view(G, Hk, n, -1), kr.transpose(1, 2).contiguous()) * scale       # (G, Hk, n, length)
        keep = ok.expand(n, length)
        if causal:
            keep = keep & (torch.arange(length) <= (length - n + torch.arange(n))[:, None])
        sc = sc.masked_fill(~keep, float("-inf"))
        row_any = (sc != float("-inf")).any(-1, keepdim=True)
        p = torch.softmax(sc.masked_fill(~row_any, 0.0), -1).masked_fill(~keep | ~row_any, 0.0)
        bad = ~vr.isfinite()
        out = torch.matmul(p, vr.masked_fill(bad, 0.0))
        for j in bad.any(-1).any(0).nonzero().flatten().tolist():   # values that are not finite count where they are seen
            extra = torch.where(bad[:, j], vr[:, j], 0.0)
            out += torch.where(keep[:, j, None] & bad[:, j][None, :, None, :], p[..., j, None] * extra[:, None, :], 0.0)
        if o.dtype == torch.float16:   # averages of values that were finite; 8-bit ones may stand for 65536
            out = torch.where(out.isfinite(), out.clamp(-65504.0, 65504.0), out)
        o[at, :, row0:row0 + n] = out.reshape(G * Hk, n, -1).to(o.dtype)
        lse[at, :, row0:row0 + n] = torch.logsumexp(sc, -1).reshape(G * Hk, n)
    return o, lse

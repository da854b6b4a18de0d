"""Linear attention of PoPE rows with a decay for each head, its single-token step, and the gated norm behind it.

With q_hat, k_hat the rows of ``apply_pope_to_qk``, g = exp(log_decay) of a kv head and S its state, a matrix of
(dim + rotate_dim, value dim) in fp32 whose rows have the column order of ``apply_pope_to_qk``:

  S_i = g S_(i-1) + k_hat_i v_i^T        o_i = scale S_i^T q_hat_i

that is o_i = scale sum_{j <= i} g^(i - j) (q_hat_i . k_hat_j) v_j plus what the state before carries in: attention without a
softmax, whose cost grows linearly with the length and whose cache is one state.  Always causal.  Query head h reads kv
head h % heads, as in the softmax attention here.

  linear_attn_with_pope        prompts and training, with autograd: q, k, v, pos_emb, the initial state, gate and norm weight
  linear_attn_step_with_pope   one token of each sequence against its state, states in slots
  gated_head_norm              y = x / sqrt(mean x^2 + eps) * weight * silu(gate) over each head's row: no softmax bounds the
                               outputs, so layers of this kind norm and gate them; both calls above take ``gate``

Rows are bf16, fp16 or fp32, (batch, heads, n, dim) or (batch, n, heads, dim) with ``head_dimension_at_first=False``; dim and the value
dim go up to 256, of any size.  A sequence goes on from a state with any split of its rows over calls: positions come from
``pos_emb``, ``pope(positions)``, one row of angles per row.

Precision on the GPU.  States, sums, powers of g and the norm are fp32; softplus, sine and cosine are off by up to 1e-6, whatever their
value.  A step is fp32 throughout, from rows as they are.  Prompts and training run on bf16 matrix instructions.  bf16 rows are one
bf16 part: q_hat (times the scale), k_hat, the weighted q_hat . k_hat (backward: dO . v) and a state on its way into a product are each
rounded to bf16, which leaves outputs and gradients off by 0.003 to 0.004 in the 2-norm; their own rounding is 0.0017 of that.  fp16 and fp32
rows are the sum of two bf16 parts, as are bf16 rows under a gate and calls of up to 32 bf16 rows a sequence (packed: in all): 16 significant
bits, fp32 rows too, the product of the second parts left out; outputs are off by 1e-5, and by their own rounding.  The states that a call returns
have keys of two parts whatever the rows.  How rows are cut into segments depends on the call's batch, heads and length, and with that the last
bits of a sequence's results; the same call gives the same bits.

No counterpart in the reference, whose attention is the softmax's (PoPE_pytorch/attention.py:75-145).  GPU tensors run the HIP
kernels (csrc/linear_*.hip, csrc/gated_norm.hip), CPU tensors the torch computation below.  Calls do not synchronise or read
lengths on the host, and can be captured into graphs (a backward pass while no eager autograd graph of the same leaves
lives); gradients are summed in a fixed order.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn.functional as F
from torch import Tensor
from torch.autograd import forward_ad

from . import _lib

_DTYPES = (torch.bfloat16, torch.float16, torch.float32)
_MAX_DIM, _MAX_NORM = 256, 512
_NORM_DOWN = 2.0 ** -100   # kNormDown of csrc/linear_dev.hpp
_CHUNK = 128   # rows that the CPU computation takes at once


def exists(v):
    return v is not None


def _tracked(t: Optional[Tensor]) -> bool:
    return exists(t) and ((torch.is_grad_enabled() and t.requires_grad)
                          or (not torch.compiler.is_compiling() and exists(forward_ad.unpack_dual(t).tangent)))


# ---------------------------------------------------------------- arguments

def _check_device(q: Tensor, **ts):
    for name, t in ts.items():
        if exists(t) and t.device != q.device:
            raise RuntimeError(f"pope_amd linear attention: {name} on {t.device}, q on {q.device}")


def _check_rows(q: Tensor, k: Tensor, v: Tensor):
    """Head-first rows."""
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        if t.ndim != 4:
            raise ValueError(f"{name} must be 4-D, got {tuple(t.shape)}")
        if t.dtype not in _DTYPES or t.dtype != q.dtype:
            raise TypeError(f"q, k, v must be all bfloat16, all float16 or all float32, got {name} of dtype {t.dtype}")
    if k.shape[0] != q.shape[0] or k.shape[2] != q.shape[2] or k.shape[3] != q.shape[3] or v.shape[:3] != k.shape[:3]:
        raise ValueError(f"incompatible q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} (batch, heads, n, dim)")
    if k.shape[1] < 1 or q.shape[1] < 1 or q.shape[1] % k.shape[1]:
        raise ValueError(f"{q.shape[1]} query heads must be a multiple of {k.shape[1]} kv heads")
    if not 1 <= q.shape[3] <= _MAX_DIM or not 1 <= v.shape[3] <= _MAX_DIM:
        raise ValueError(f"dim and value dim must be 1 to {_MAX_DIM}, got {q.shape[3]} and {v.shape[3]}")


def _default_scale(q: Tensor) -> float:
    dim = q.shape[-1] if q.ndim else 0
    return dim ** -0.5 if dim else 1.0   # no dim: refused with the rows


def _check_pos_emb(pos_emb, q: Tensor, heads: int):
    """freqs (n, R) or (1 or batch, n, R) and bias (1 or heads, R); None, None without rotation."""
    if not exists(pos_emb):
        return None, None
    freqs, bias = pos_emb
    R = freqs.shape[-1] if exists(freqs) else 0
    if R == 0:
        return None, None
    if not exists(bias):
        raise ValueError("pos_emb needs its bias: keys carry it")
    if R > q.shape[3]:
        raise ValueError(f"rotate dim {R} exceeds the head dim {q.shape[3]}")
    B, n = q.shape[0], q.shape[2]
    if freqs.ndim not in (2, 3) or freqs.shape[-2] != n or (freqs.ndim == 3 and freqs.shape[0] not in (1, B)):
        raise ValueError(f"freqs {tuple(freqs.shape)} must have one row of angles per row: ({n}, {R}) or ({B}, {n}, {R})")
    if bias.ndim == 1:
        bias = bias.unsqueeze(0)
    if bias.ndim != 2 or bias.shape[1] != R or bias.shape[0] not in (1, heads):
        raise ValueError(f"bias {tuple(bias.shape)} must be (1 or {heads}, {R})")
    _check_device(q, freqs=freqs, bias=bias)
    return freqs.float(), bias if bias.dtype in _DTYPES else bias.float()


def _check_decay(log_decay: Optional[Tensor], q: Tensor, heads: int):
    if not exists(log_decay):
        return None
    if tuple(log_decay.shape) != (heads,):
        raise ValueError(f"log_decay {tuple(log_decay.shape)} must be (kv heads,) = ({heads},)")
    if not log_decay.is_floating_point():
        raise TypeError(f"log_decay must be floating, got {log_decay.dtype}")
    if _tracked(log_decay):
        raise RuntimeError("pope_amd linear attention: no gradient is defined for log_decay; pass it detached")
    _check_device(q, log_decay=log_decay)
    return log_decay.float().contiguous()


def _check_state(name: str, state: Tensor, want: tuple, q: Tensor):
    if tuple(state.shape) != want:
        raise ValueError(f"{name} {tuple(state.shape)} must be (sequences, kv heads, dim + rotate dim, value dim) = {want}")
    if not state.is_floating_point():
        raise TypeError(f"{name} must be floating, got {state.dtype}")
    _check_device(q, **{name: state})


def _ints(name: str, t: Tensor, q: Tensor, n: int):
    if tuple(t.shape) != (n,):
        raise ValueError(f"{name} {tuple(t.shape)} must be ({n},)")
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be int32 or int64, got {t.dtype}")
    _check_device(q, **{name: t})
    if t.dtype != torch.int32:   # what int32 cannot hold stays out of range
        t = t.clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32)
    return t.contiguous()


def _check_norm(x: Tensor, gate: Tensor, weight: Optional[Tensor], heads: int):
    if x.ndim != 4:
        raise ValueError(f"x must be 4-D, got {tuple(x.shape)}")
    if gate.dtype not in _DTYPES or x.dtype not in (gate.dtype, torch.float32):
        raise TypeError(f"gate must be bfloat16, float16 or float32, and x of its dtype or float32, got {gate.dtype} and {x.dtype}")
    if gate.shape != x.shape:
        raise ValueError(f"gate {tuple(gate.shape)} must match x {tuple(x.shape)}")
    _check_device(x, gate=gate, weight=weight)
    if not 1 <= x.shape[3] <= _MAX_NORM:
        raise ValueError(f"rows must have 1 to {_MAX_NORM} values, got {x.shape[3]}")
    if heads < 1:
        raise ValueError(f"x {tuple(x.shape)} has no heads")
    if exists(weight):
        if weight.ndim not in (1, 2) or weight.shape[-1] != x.shape[3] or (weight.ndim == 2 and weight.shape[0] not in (1, heads)):
            raise ValueError(f"weight {tuple(weight.shape)} must be ({x.shape[3]},) or (1 or {heads}, {x.shape[3]})")
        if weight.dtype not in (gate.dtype, torch.float32):
            raise TypeError(f"weight must be {gate.dtype} or float32, got {weight.dtype}")


# ---------------------------------------------------------------- ops (tracing); eager calls take the same native calls
# Rows are head-first; what an op does not return is empty.

@torch.library.custom_op("pope_amd::linear_fwd", mutates_args=(), device_types="cuda")
def linear_fwd_op(q: Tensor, k: Tensor, v: Tensor, freqs: Optional[Tensor], bias: Optional[Tensor], log_decay: Optional[Tensor], mask: Optional[Tensor],
                  cu_seqlens: Optional[Tensor], initial: Optional[Tensor], scale: float, with_state: bool, o_f32: bool) -> tuple[Tensor, Tensor, Tensor]:
    return _lib.host().linear_fwd(q, k, v, freqs, bias, log_decay, mask, cu_seqlens, initial, scale, with_state, o_f32)


def _linear_state_shape(q, k, v, freqs, cu_seqlens):
    return (q.shape[0] if cu_seqlens is None else cu_seqlens.shape[0] - 1, k.shape[1], q.shape[3] + (0 if freqs is None else freqs.shape[-1]), v.shape[3])


@linear_fwd_op.register_fake
def _(q, k, v, freqs, bias, log_decay, mask, cu_seqlens, initial, scale, with_state, o_f32):
    o = q.new_empty((*q.shape[:3], v.shape[3]), dtype=torch.float32 if o_f32 else q.dtype)
    last = q.new_empty(_linear_state_shape(q, k, v, freqs, cu_seqlens) if with_state else (0,), dtype=torch.float32)
    # what the backward reads: as many bytes as the library says
    n = torch.library.get_ctx().new_dynamic_size()
    return o, last, q.new_empty((n,), dtype=torch.uint8)


@torch.library.custom_op("pope_amd::linear_bwd", mutates_args=(), device_types="cuda")
def linear_bwd_op(dout: Tensor, dlast: Optional[Tensor], q: Tensor, k: Tensor, v: Tensor, freqs: Optional[Tensor], bias: Optional[Tensor],
                  log_decay: Optional[Tensor], mask: Optional[Tensor], cu_seqlens: Optional[Tensor], initial: Optional[Tensor], kept: Optional[Tensor],
                  scale: float, o_f32: bool, need_dfreqs: bool, need_dbias: bool, need_dinitial: bool) -> tuple[Tensor, Tensor, Tensor, Tensor, Tensor, Tensor]:
    return _lib.host().linear_bwd(dout, dlast, q, k, v, freqs, bias, log_decay, mask, cu_seqlens, initial, kept, scale, o_f32, need_dfreqs,
                                  need_dbias, need_dinitial)


@linear_bwd_op.register_fake
def _(dout, dlast, q, k, v, freqs, bias, log_decay, mask, cu_seqlens, initial, kept, scale, o_f32, need_dfreqs, need_dbias, need_dinitial):
    some = lambda shape, want: q.new_empty(shape if want else (0,), dtype=torch.float32)
    return (q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape), some(freqs.shape if need_dfreqs else (0,), need_dfreqs),
            q.new_empty(bias.shape, dtype=bias.dtype) if need_dbias else some((0,), False), some(_linear_state_shape(q, k, v, freqs, cu_seqlens), need_dinitial))


def _linear_setup(ctx, inputs, output):
    q, k, v, freqs, bias, log_decay, mask, cu_seqlens, initial, ctx.scale, ctx.with_state, ctx.o_f32 = inputs
    ctx.save_for_backward(q, k, v, freqs, bias, log_decay, mask, cu_seqlens, initial, output[2])
    ctx.set_materialize_grads(False)


def _linear_backward(ctx, dout, dlast, dkept):
    q, k, v, freqs, bias, log_decay, mask, cu_seqlens, initial, kept = ctx.saved_tensors
    need = ctx.needs_input_grad
    if dout is None:
        dout = q.new_zeros((*q.shape[:3], v.shape[3]), dtype=torch.float32 if ctx.o_f32 else q.dtype)
    dq, dk, dv, df, db, d0 = linear_bwd_op(dout, dlast if ctx.with_state else None, q, k, v, freqs, bias, log_decay, mask, cu_seqlens, initial, kept,
                                           ctx.scale, ctx.o_f32, need[3], need[4], need[8])
    return dq, dk, dv, df if need[3] else None, db if need[4] else None, None, None, None, d0 if need[8] else None, None, None, None


linear_fwd_op.register_autograd(_linear_backward, setup_context=_linear_setup)


@torch.library.custom_op("pope_amd::linear_step", mutates_args=("state",), device_types="cuda")
def linear_step_op(q: Tensor, k: Tensor, v: Tensor, freqs: Optional[Tensor], bias: Optional[Tensor], log_decay: Optional[Tensor], state: Tensor,
                   state_index: Optional[Tensor], new_index: Optional[Tensor], gate: Optional[Tensor], norm_weight: Optional[Tensor], norm_eps: float,
                   scale: float) -> Tensor:
    return _lib.host().linear_step(q, k, v, freqs, bias, log_decay, state, state_index, new_index, gate, norm_weight, norm_eps, scale)


@linear_step_op.register_fake
def _(q, k, v, freqs, bias, log_decay, state, state_index, new_index, gate, norm_weight, norm_eps, scale):
    return q.new_empty((*q.shape[:3], v.shape[3]))


@torch.library.custom_op("pope_amd::gated_norm_fwd", mutates_args=(), device_types="cuda")
def gated_norm_fwd_op(x: Tensor, gate: Tensor, weight: Optional[Tensor], eps: float, head_first: bool) -> Tensor:
    return _lib.host().gated_norm_fwd(x, gate, weight, eps, head_first)


def _rows_like(x, dtype=None):   # rows_like of csrc_torch/pope_host.cpp
    y = torch.empty_like(x, dtype=dtype)
    return y if y.stride(-1) == 1 else x.new_empty(x.shape, dtype=dtype)


@gated_norm_fwd_op.register_fake
def _(x, gate, weight, eps, head_first):
    return _rows_like(x if x.stride(-1) == 1 else x.contiguous(), gate.dtype)


@torch.library.custom_op("pope_amd::gated_norm_bwd", mutates_args=(), device_types="cuda")
def gated_norm_bwd_op(dy: Tensor, x: Tensor, gate: Tensor, weight: Optional[Tensor], eps: float, head_first: bool, need_dweight: bool) -> tuple[Tensor, Tensor, Tensor]:
    return _lib.host().gated_norm_bwd(dy, x, gate, weight, eps, head_first, need_dweight)


@gated_norm_bwd_op.register_fake
def _(dy, x, gate, weight, eps, head_first, need_dweight):
    unit = lambda t: t if t.stride(-1) == 1 else t.contiguous()
    return _rows_like(unit(x)), _rows_like(unit(gate)), torch.empty_like(weight) if need_dweight else x.new_empty((0,), dtype=torch.float32)


def _norm_setup(ctx, inputs, output):
    x, gate, weight, ctx.eps, ctx.head_first = inputs
    ctx.save_for_backward(x, gate, weight)


def _norm_backward(ctx, dy):
    x, gate, weight = ctx.saved_tensors
    need = ctx.needs_input_grad[2]
    dx, dg, dw = gated_norm_bwd_op(dy, x, gate, weight, ctx.eps, ctx.head_first, need)
    return dx, dg, dw if need else None, None, None


gated_norm_fwd_op.register_autograd(_norm_backward, setup_context=_norm_setup)


# ---------------------------------------------------------------- public calls

def gated_head_norm(x: Tensor, gate: Tensor, weight: Optional[Tensor] = None, *, eps: float = 1e-5, head_dimension_at_first: bool = True) -> Tensor:
    """x / sqrt(mean x^2 + eps) * weight * silu(gate) over the last dim of x (batch, heads, n, dim), dim 1 to 512, with autograd.

    ``gate`` is shaped as x and has the result's dtype; x has that dtype or is fp32; ``weight`` (dim,) or (1 or heads, dim), of gate's
    dtype or fp32, or None.  Arithmetic is fp32, rounded once.  ``head_dimension_at_first`` says which dim a weight of several heads goes with."""
    if x.is_cuda and _lib.eager(x, gate, weight):
        y = _lib.host().gated_norm_eager(x, gate, weight, eps, head_dimension_at_first)
        if exists(y):
            return y
    _check_norm(x, gate, weight, x.shape[1 if head_dimension_at_first else 2] if x.ndim == 4 else 1)
    if exists(weight) and weight.stride(-1) != 1:
        weight = weight.contiguous()
    if not x.is_cuda:
        return _norm_torch(x, gate, weight, eps, head_dimension_at_first)
    _lib.refuse_tangents("gated norm", x, gate, weight)
    return gated_norm_fwd_op(x, gate, weight, float(eps), bool(head_dimension_at_first))


def linear_attn_with_pope(q: Tensor, k: Tensor, v: Tensor, log_decay: Optional[Tensor] = None, pos_emb=None, mask: Optional[Tensor] = None, *,
                          scale: Optional[float] = None, initial_state: Optional[Tensor] = None, return_state: bool = False,
                          cu_seqlens: Optional[Tensor] = None, gate: Optional[Tensor] = None, norm_weight: Optional[Tensor] = None, norm_eps: float = 1e-5,
                          head_dimension_at_first: bool = True):
    """Causal linear attention (see the module's text) of q (batch, query heads, n, dim) over k (batch, kv heads, n, dim) and
    v (batch, kv heads, n, value dim): o (batch, query heads, n, value dim), or (o, state) with ``return_state``.

    ``log_decay`` (kv heads,): log g, 0 or less in use (above 0 states grow), None for no decay; no gradient.  ``pos_emb``:
    (freqs, bias), ``pope(positions)``, or None for no rotated dims; freqs (n, rotate dim) or (batch, n, rotate dim).  ``mask``
    (batch, n): rows that are False have no key and no value; time passes for the state all the same.  ``scale``: dim^-1/2 by default.

    ``initial_state`` (sequences, kv heads, dim + rotate dim, value dim): the states to go on from, zeros by default; states are
    fp32.  Packed calls have batch 1 and ``cu_seqlens`` (sequences + 1 ascending numbers): rows cu_seqlens[b] .. cu_seqlens[b + 1] - 1
    belong to sequence b; rows outside every sequence give 0.

    ``gate`` (shaped as o; bf16, fp16 or fp32, which the result then has): o is ``gated_head_norm(o, gate, norm_weight, eps=norm_eps)``.

    A value that is not finite reaches the rows from its own on, where sums through a state may turn infinities into NaN; on the GPU,
    finite fp32 values above 3.3895e38, the largest bf16, count as that.  GPU calls
    that would need 2^22 workgroups (about one for each 64 rows or more of each head) raise."""
    args = (log_decay, mask, cu_seqlens, initial_state)
    freqs, bias = pos_emb if exists(pos_emb) else (None, None)
    scale = _default_scale(q) if scale is None else float(scale)
    hf = bool(head_dimension_at_first)
    if exists(norm_weight) and not exists(gate):
        raise ValueError("norm_weight given without a gate")
    if exists(gate) and q.ndim == 4 and v.ndim == 4:   # before anything is launched
        want = (*q.shape[:3], v.shape[3])
        if tuple(gate.shape) != want:
            raise ValueError(f"gate {tuple(gate.shape)} must match the output {want}")
        _check_device(q, gate=gate)
        _check_norm(gate, gate, norm_weight, q.shape[1 if hf else 2])
    # the norm divides by the size of a row, and a short row's own rounding would come out as large as that row is small: its
    # input, and the gradient that comes back, are fp32
    o_f32 = exists(gate)
    out = None
    if q.is_cuda and _lib.eager(q, k, v, freqs, bias, *args):
        out = _lib.host().linear_eager(q, k, v, freqs, bias, *args, scale, return_state, hf, o_f32)
    if exists(out):
        o, last = out
    else:
        if not hf:
            q, k, v = (t.transpose(1, 2) if t.ndim == 4 else t for t in (q, k, v))
        _check_rows(q, k, v)
        _check_device(q, k=k, v=v, mask=mask)
        B, n, Hk = q.shape[0], q.shape[2], k.shape[1]
        log_decay = _check_decay(log_decay, q, Hk)
        freqs, bias = _check_pos_emb(pos_emb, q, Hk)
        if exists(mask):
            if tuple(mask.shape) != (B, n):
                raise ValueError(f"mask {tuple(mask.shape)} must be (batch, n) = ({B}, {n})")
            mask = mask.bool()
        if exists(cu_seqlens):
            if B != 1:
                raise ValueError(f"packed rows (cu_seqlens) need a batch of 1, got {B}")
            if cu_seqlens.ndim != 1 or cu_seqlens.shape[0] < 2:
                raise ValueError(f"cu_seqlens {tuple(cu_seqlens.shape)} must be (sequences + 1,)")
            cu_seqlens = _ints("cu_seqlens", cu_seqlens, q, cu_seqlens.shape[0])
        shape = _linear_state_shape(q, k, v, freqs, cu_seqlens)
        if exists(initial_state):
            _check_state("initial_state", initial_state, shape, q)
            initial_state = initial_state.float()
        if n == 0 or B == 0:
            o = q.new_zeros((*q.shape[:3], v.shape[3]), dtype=torch.float32 if o_f32 else q.dtype)
            last = initial_state.clone() if exists(initial_state) else torch.zeros(shape, device=q.device)
        elif not q.is_cuda:
            o, last = _linear_torch(q, k, v, freqs, bias, log_decay, mask, cu_seqlens, initial_state, scale, shape, torch.float32 if o_f32 else q.dtype)
        else:
            _lib.refuse_tangents("linear attention", q, k, v, freqs, bias, initial_state)
            o, last, _ = linear_fwd_op(q, k, v, freqs, bias, log_decay, mask, cu_seqlens, initial_state, scale, bool(return_state), o_f32)
        if not o.requires_grad and (n == 0 or B == 0 or not q.is_cuda):
            for t in (q, k, v, freqs, bias):   # gradients of zeros, for a batch without rows, or with rows of no sequence
                if _tracked(t):
                    none = t.flatten()[:0].sum(dtype=torch.float32)
                    o, last = o + none.to(o.dtype), last + none
        if not hf:
            o = o.transpose(1, 2)
    if exists(gate):
        o = gated_head_norm(o, gate, norm_weight, eps=norm_eps, head_dimension_at_first=hf)
    return (o, last) if return_state else o


def linear_attn_step_with_pope(q: Tensor, k: Tensor, v: Tensor, log_decay: Optional[Tensor], pos_emb, state: Tensor, *,
                               state_index: Optional[Tensor] = None, new_index: Optional[Tensor] = None, scale: Optional[float] = None,
                               gate: Optional[Tensor] = None, norm_weight: Optional[Tensor] = None, norm_eps: float = 1e-5,
                               head_dimension_at_first: bool = True) -> Tensor:
    """One new row of each sequence, q (batch, query heads, 1, dim), against its state: o (batch, query heads, 1, value dim).

    ``state`` (slots, kv heads, dim + rotate dim, value dim) fp32 is updated in place; slots may be spaced, a slot is contiguous.
    Sequence b reads slot ``state_index[b]`` (by default b) and writes slot ``new_index[b]`` (by default where it read), so sequences
    can go on from a prompt that they share.  No slot may be written by two sequences of a call, or written by one and read by
    another: what they then hold is unspecified.  A sequence whose ``state_index`` is no slot has no token: its output is 0 and nothing
    is written; a ``new_index`` that is no slot is not written.  ``pos_emb``: (freqs, bias) of the new rows, freqs (1, rotate dim) or (batch,
    1, rotate dim); ``gate`` has the rows' dtype; the other arguments as in ``linear_attn_with_pope``.  No gradient is defined."""
    freqs, bias = pos_emb if exists(pos_emb) else (None, None)
    scale = _default_scale(q) if scale is None else float(scale)
    hf = bool(head_dimension_at_first)
    if q.is_cuda and _lib.eager(q, k, v, freqs, bias, log_decay, state, state_index, new_index, gate, norm_weight):
        o = _lib.host().linear_step_eager(q, k, v, freqs, bias, log_decay, state, state_index, new_index, gate, norm_weight, norm_eps, scale, hf)
        if exists(o):
            return o
    if not hf:
        q, k, v, gate = (t.transpose(1, 2) if exists(t) and t.ndim == 4 else t for t in (q, k, v, gate))
    _check_rows(q, k, v)
    if q.shape[2] != 1:
        raise ValueError(f"a step takes one row for each sequence, got {q.shape[2]}")
    _check_device(q, k=k, v=v)
    B, Hk, Dv = q.shape[0], k.shape[1], v.shape[3]
    log_decay = _check_decay(log_decay, q, Hk)
    freqs, bias = _check_pos_emb(pos_emb, q, Hk)
    want = (state.shape[0] if state.ndim == 4 else 1, *_linear_state_shape(q, k, v, freqs, None)[1:])
    _check_state("state", state, want, q)
    if state.dtype != torch.float32:
        raise TypeError(f"state must be float32, got {state.dtype}")
    if state.shape[0] < 1 or state.stride(3) != 1 or state.stride(2) != Dv or state.stride(1) != want[2] * Dv or (
            state.shape[0] > 1 and state.stride(0) < want[1] * want[2] * Dv):
        raise ValueError("state must have at least one slot, and its slots must be contiguous and apart")
    if not exists(state_index) and B > state.shape[0]:
        raise ValueError(f"{B} sequences, {state.shape[0]} slots")
    state_index, new_index = (_ints(n, t, q, B) if exists(t) else None for n, t in (("state_index", state_index), ("new_index", new_index)))
    if exists(norm_weight) and not exists(gate):
        raise ValueError("norm_weight given without a gate")
    if exists(gate):
        if tuple(gate.shape) != (B, q.shape[1], 1, Dv):
            raise ValueError(f"gate {tuple(gate.shape)} must match the output {(B, q.shape[1], 1, Dv)}")
        _check_norm(gate, gate, norm_weight, q.shape[1])
        if gate.dtype != q.dtype:
            raise TypeError(f"gate of dtype {gate.dtype}, the rows have {q.dtype}")
        _check_device(q, gate=gate)
        gate = gate if gate.stride(-1) == 1 else gate.contiguous()
        if exists(norm_weight) and norm_weight.stride(-1) != 1:
            norm_weight = norm_weight.contiguous()
    if any(_tracked(t) for t in (q, k, v, freqs, bias, state, gate, norm_weight)):
        raise RuntimeError("pope_amd linear attention step: no gradient is defined; call it under torch.no_grad() or on detached tensors")
    if B == 0:
        o = q.new_zeros((0, q.shape[1], 1, Dv))
    elif not q.is_cuda:
        o = _step_torch(q, k, v, freqs, bias, log_decay, state, state_index, new_index, scale)
        if exists(gate):
            o = _norm_torch(o, gate, norm_weight, norm_eps, True)
        o = o.to(q.dtype)
    else:
        o = linear_step_op(q, k, v, freqs, bias, log_decay, state, state_index, new_index, gate, norm_weight, float(norm_eps), scale)
    return o if hf else o.transpose(1, 2)


# ---------------------------------------------------------------- CPU tensors: torch operators, fp32

def _norm_torch(x, gate, weight, eps, head_first):
    y = x.float()
    with torch.no_grad():   # rows whose squares pass fp32's range, at a smaller scale
        scale = torch.where(y.square().sum(-1, keepdim=True).isfinite(), 1.0, _NORM_DOWN)
    y = y * scale
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + eps * scale * scale)
    if exists(weight):
        y = y * (weight.float()[:, None, :] if weight.ndim == 2 and head_first else weight.float())
    return (y * F.silu(gate.float())).to(gate.dtype)


def _expand(x: Tensor, freqs: Optional[Tensor], bias: Optional[Tensor]) -> Tensor:
    """Rows of apply_pope_to_qk in fp32, angles in fp64: x head-first."""
    x = x.float()
    if not exists(freqs):
        return x
    R = freqs.shape[-1]
    angle = (freqs if freqs.ndim == 2 else freqs.unsqueeze(1)).double()
    if exists(bias):
        angle = angle + bias.double()[:, None, :]
    m = F.softplus(x[..., :R])
    pairs = torch.stack((m * angle.cos().float(), m * angle.sin().float()), -1).flatten(-2)
    return torch.cat((pairs, x[..., R:]), -1)


def _linear_torch(q, k, v, freqs, bias, log_decay, mask, cu_seqlens, initial, scale, shape, dtype):
    G, Hk, n = q.shape[1] // k.shape[1], k.shape[1], q.shape[2]
    gone = ~mask[:, None, :, None] if exists(mask) else None
    if exists(gone):   # before the expansion: its derivatives of what is not finite would make a gradient of 0 NaN
        k, v = k.masked_fill(gone, 0.0), v.masked_fill(gone, 0.0)
    qh, kh, vf = _expand(q, freqs, None) * scale, _expand(k, freqs, bias), v.float()
    if exists(gone):   # and behind it: the magnitude of 0 is log 2
        kh = kh.masked_fill(gone, 0.0)
    ld = log_decay.double() if exists(log_decay) else torch.zeros(Hk, dtype=torch.float64)
    # g^p; g^0 is 1 whatever g is
    power = lambda p: torch.where(p == 0, 1.0, (ld.view(-1, *([1] * p.ndim)) * p.clamp_min(1)).exp()).float()
    if exists(cu_seqlens):
        cu = [min(max(int(x), 0), n) for x in cu_seqlens]
        parts = [(0, cu[b], max(cu[b + 1], cu[b])) for b in range(len(cu) - 1)]
    else:
        parts = [(b, 0, n) for b in range(q.shape[0])]
    o = q.new_zeros((*q.shape[:3], v.shape[3]), dtype=dtype)
    last, pieces = [], []
    for s, (b, lo, hi) in enumerate(parts):
        S = initial[s] if exists(initial) else torch.zeros(shape[1:])
        for a in range(lo, hi, _CHUNK):
            z = min(a + _CHUNK, hi)
            i = torch.arange(z - a)
            qc, kc, vc = qh[b, :, a:z].unflatten(0, (G, Hk)), kh[b, :, a:z], vf[b, :, a:z]
            d = i[:, None] - i
            w = (qc @ kc.transpose(1, 2)) * power(d.clamp_min(0))
            # a row behind counts for nothing, also where it is not finite
            out = (qc @ S) * power(i + 1)[..., None]
            if bool(vc.isfinite().all()):
                out = out + w.masked_fill(d < 0, 0.0) @ vc
            else:
                terms = (w[..., None] * vc[:, None]).masked_fill((d < 0)[..., None], 0.0)
                out = out + terms.sum(-2)
            pieces.append((b, a, out.flatten(0, 1).to(o.dtype)))
            left = z - a - 1 - i
            S = power(torch.tensor(z - a)).view(-1, 1, 1) * S + (kc * power(left)[..., None]).transpose(1, 2) @ vc
        last.append(S)
    for b, a, rows in pieces:
        o[b, :, a:a + rows.shape[1]] = rows
    return o, torch.stack(last)


def _step_torch(q, k, v, freqs, bias, log_decay, state, state_index, new_index, scale):
    """o in fp32; the states in place."""
    B, Hk = q.shape[0], k.shape[1]
    G, slots = q.shape[1] // Hk, state.shape[0]
    src = (state_index if exists(state_index) else torch.arange(B)).long()
    dst = (new_index if exists(new_index) else src).long()
    some = (src >= 0) & (src < slots)
    qh, kh = _expand(q, freqs, None) * scale, _expand(k, freqs, bias)
    g = log_decay.double().exp().float() if exists(log_decay) else torch.ones(Hk)
    S = state[src.clamp(0, slots - 1)] * g[:, None, None] + kh.transpose(2, 3) * v.float()
    o = (qh.unflatten(1, (G, Hk)) @ S[:, None]).flatten(1, 2)
    put = some & (dst >= 0) & (dst < slots)
    state[dst[put]] = S[put]
    return o.masked_fill(~some[:, None, None, None], 0.0)

"""Linear attention, its step and the gated norm on CPU tensors against 64-bit formulas, what the calls refuse, and the C ABI's host
checks of them."""
import ctypes
import math

import pytest
import torch
import torch.nn.functional as F

import linear_common as L
import pope_amd
from linear_common import Case, check, run
from pope_amd import _lib, gated_head_norm, linear_attn_step_with_pope, linear_attn_with_pope

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
INF, NAN = math.inf, math.nan
CPU = torch.device("cpu")


def bound(case, name, value, tol):
    """fp32 arithmetic on rows as they are, as in linear_common, and each output's own rounding."""
    own = L.half(case.dtype) if name in ("o", "d_q", "d_k", "d_v") else 2.0 ** -24
    return 2e-5 * tol * (1 + own) + own * value.abs() + (2.0 ** -25 if case.dtype == F16 else 1e-30)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("shape", [
    dict(N=1, D=16, R=16, Dv=16, initial=True), dict(B=2, N=63, mask="random"), dict(B=2, N=65, mask="empty", initial=True, batch_freqs=True),
    dict(B=2, Hq=6, Hk=2, N=300, D=24, R=10, Dv=9, mask="random", initial=True), dict(Hq=3, Hk=1, N=130, D=20, R=0, Dv=7), dict(N=3, D=1, R=1, Dv=1, bias_heads=1),
    dict(lens=[0, 1, 129, 0, 30], lead=2, tail=5, D=12, R=6, Dv=10, initial=True), dict(N=140, D=8, R=8, Dv=8, decay=[-INF, 0.0], initial=True),
    dict(N=140, D=8, R=8, Dv=8, decay=None)])
def test_rows(shape, dtype):
    for head_first in (True, False):
        case = Case(CPU, dtype=dtype, **shape)
        got = run(pope_amd, case, head_first=head_first)
        val, tol = case.exact()
        for n in val:
            # gradients of 16-bit rows go through autograd in fp32 and are rounded once
            check(got[n], val[n], bound(case, n, val[n], tol[n]), n)


def test_formula_against_differences():
    """The 64-bit formula's gradients, which all others are compared with."""
    case = Case(CPU, N=5, D=4, R=2, Dv=3, Hq=2, Hk=1, initial=True, mask="random", dtype=F32)
    x = [case.leaves()[n].double().requires_grad_() for n in ("q", "k", "v", "freqs", "bias", "s0")]

    def f(q, k, v, freqs, bias, s0):
        return L.attend64(L.expand64(q, freqs, None, 2), L.expand64(k, freqs, bias, 2), v, case.decay64(), case.scale, case.mask, s0, case.seqs)

    assert torch.autograd.gradcheck(f, x)
    y = [torch.randn(1, 2, 3, 4, dtype=torch.float64, requires_grad=True) for _ in range(2)] + [torch.randn(2, 4, dtype=torch.float64, requires_grad=True)]
    assert torch.autograd.gradcheck(lambda a, b, w: L.norm64(a, b, w, 1e-5), y)


@pytest.mark.parametrize("value", [INF, NAN])
def test_not_finite(value):
    case = Case(CPU, B=2, N=150, mask="empty", initial=True)
    clean = run(pope_amd, case)
    keep = case.k, case.v
    case.k, case.v = (t.masked_fill(~case.mask[:, None, :, None], value) for t in keep)
    got = run(pope_amd, case, grads=False)
    for n in got:
        assert torch.equal(got[n], clean[n]), n
    case.k, case.v = keep
    case.mask = None
    clean = run(pope_amd, case, grads=False)["o"]
    case.v = case.v.clone()
    case.v[0, 1, 140] = value
    o = run(pope_amd, case, grads=False)["o"]
    assert torch.allclose(o[0, :, :140].float(), clean[0, :, :140].float(), rtol=1e-2) and not o[0, 1, 140:].isfinite().any() and torch.equal(o[1], clean[1])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_pieces_then_steps_are_one_prompt(dtype):
    case = Case(CPU, B=2, Hq=4, Hk=2, N=150, D=24, R=12, Dv=20, dtype=dtype)
    gate, w = torch.randn_like(case.do), torch.rand(4, 20) + 0.5
    kw = dict(norm_weight=w)
    whole, last = linear_attn_with_pope(case.q, case.k, case.v, case.ld, case.emb(), gate=gate, return_state=True, **kw)
    o, state = linear_attn_with_pope(*(t[:, :, :140] for t in (case.q, case.k, case.v)), case.ld, (case.freqs[:140], case.bias), gate=gate[:, :, :140], return_state=True, **kw)
    parts = [o]
    for i in range(140, 150):
        parts.append(linear_attn_step_with_pope(*(t[:, :, i:i + 1] for t in (case.q, case.k, case.v)), case.ld, (case.freqs[i:i + 1], case.bias), state, gate=gate[:, :, i:i + 1], **kw))
    val, tol = case.exact(False)
    e, rms = 2e-5 * tol["o"], (val["o"].square().mean(-1, keepdim=True) + 1e-5).sqrt()
    y = L.norm64(val["o"], gate, w, 1e-5)
    limit = 2 * (e / rms * (w[:, None, :] * F.silu(gate.float())).abs() + y.abs() * e.square().mean(-1, keepdim=True).sqrt() / rms) + 1.01 * L.half(dtype) * y.abs() + 1e-6
    for got in (whole, torch.cat(parts, 2)):
        check(got, y, limit, "gated o")
    check(state, val["states"], 2e-5 * tol["states"], "states")


def test_step_slots():
    case = Case(CPU, B=4, N=1, initial=True)
    plain_state = case.s0.clone()
    plain = linear_attn_step_with_pope(case.q, case.k, case.v, case.ld, case.emb(), plain_state)
    val, tol = case.exact(False)
    check(plain_state, val["states"], 2e-5 * tol["states"], "states")
    state = case.s0.clone()
    o = linear_attn_step_with_pope(case.q, case.k, case.v, case.ld, case.emb(), state, state_index=torch.tensor([0, -1, 2 ** 40, 3]), new_index=torch.tensor([0, 1, 2, 9]))
    assert torch.equal(o[0], plain[0]) and torch.equal(o[3], plain[3]) and not o[1:3].any()
    assert torch.equal(state[0], plain_state[0]) and torch.equal(state[1:], case.s0[1:])


def test_norm():
    for dtype in (BF16, F16, F32):
        for wide in (False, True):
            x, gate, w = torch.randn(2, 3, 9, 33), torch.randn(2, 3, 9, 33).to(dtype), torch.randn(3, 33)
            x = x if wide else x.to(dtype)
            y = gated_head_norm(x, gate, w)
            want = L.norm64(x, gate, w, 1e-5)
            assert y.dtype == dtype
            check(y, want, (L.half(dtype) + 1e-5) * want.abs() + 2.0 ** -25 + 1e-7, "y")
            t = lambda z: z.transpose(1, 2)
            assert torch.equal(t(gated_head_norm(t(x), t(gate), w, head_dimension_at_first=False)), y)


def test_no_rows():
    q, kv = torch.empty(2, 4, 0, 8), torch.empty(2, 2, 0, 8)
    s0 = torch.randn(2, 2, 8, 5)
    o, last = linear_attn_with_pope(q, kv, kv.new_empty(2, 2, 0, 5), initial_state=s0, return_state=True)
    assert o.shape == (2, 4, 0, 5) and torch.equal(last, s0)
    o, last = linear_attn_with_pope(q, kv, kv, return_state=True)
    assert last.shape == (2, 2, 8, 8) and not last.any()
    assert gated_head_norm(q, q).shape == q.shape
    assert linear_attn_with_pope(q, kv, kv, gate=q).shape == q.shape


def test_refusals():
    case = Case(CPU, N=6, D=8, R=4, Dv=5, initial=True)
    q, k, v, ld, emb = case.q, case.k, case.v, case.ld, case.emb()
    call = linear_attn_with_pope

    def refuses(kind, match, f, *a, **kw):
        with pytest.raises(kind, match=match):
            f(*a, **kw)

    refuses(ValueError, "4-D", call, q[0], k, v)
    refuses(TypeError, "q, k, v must be all", call, q, k.float(), v)
    refuses(TypeError, "q, k, v must be all", call, q.double(), k.double(), v.double())
    refuses(ValueError, "incompatible", call, q, k[:, :, :5], v)
    refuses(ValueError, "incompatible", call, q, k, v[:, :1])
    refuses(ValueError, "multiple", call, q.expand(1, 2, 6, 8)[:, :1].repeat(1, 3, 1, 1), k, v)
    refuses(ValueError, "1 to 256", call, *(torch.zeros(1, 1, 2, 257) for _ in range(3)))
    refuses(ValueError, "rows? of angles|one row", call, q, k, v, ld, (emb[0][:5], emb[1]))
    refuses(ValueError, "bias", call, q, k, v, ld, (emb[0], emb[1].repeat(2, 1)))
    refuses(ValueError, "needs its bias", call, q, k, v, ld, (emb[0], None))
    refuses(ValueError, "exceeds", call, q, k, v, ld, (torch.zeros(6, 9), torch.zeros(2, 9)))
    refuses(ValueError, "log_decay", call, q, k, v, ld[:1], emb)
    refuses(TypeError, "log_decay", call, q, k, v, torch.zeros(2, dtype=torch.int32), emb)
    refuses(RuntimeError, "no gradient is defined", call, q, k, v, ld.clone().requires_grad_(), emb)
    refuses(ValueError, "mask", call, q, k, v, ld, emb, torch.ones(1, 5, dtype=torch.bool))
    refuses(ValueError, "initial_state", call, q, k, v, ld, emb, initial_state=case.s0[:, :, :8])
    refuses(TypeError, "initial_state", call, q, k, v, ld, emb, initial_state=case.s0.int())
    refuses(ValueError, "batch of 1", call, q.repeat(2, 1, 1, 1), k.repeat(2, 1, 1, 1), v.repeat(2, 1, 1, 1), ld, emb, cu_seqlens=torch.tensor([0, 6]))
    refuses(ValueError, "cu_seqlens", call, q, k, v, ld, emb, cu_seqlens=torch.tensor([0]))
    refuses(TypeError, "cu_seqlens", call, q, k, v, ld, emb, cu_seqlens=torch.tensor([0., 6.]))
    refuses(ValueError, "without a gate", call, q, k, v, ld, emb, norm_weight=torch.ones(5))
    refuses(ValueError, "gate", call, q, k, v, ld, emb, gate=torch.zeros(1, 2, 6, 4, dtype=BF16))
    refuses(ValueError, "weight", call, q, k, v, ld, emb, gate=torch.zeros(1, 2, 6, 5, dtype=BF16), norm_weight=torch.ones(4))

    step = linear_attn_step_with_pope
    one, e1 = [t[:, :, :1] for t in (q, k, v)], (emb[0][:1], emb[1])
    refuses(ValueError, "one row", step, q, k, v, ld, emb, case.s0)
    refuses(TypeError, "float32", step, *one, ld, e1, case.s0.double())
    refuses(ValueError, "state", step, *one, ld, e1, case.s0[..., :4])
    refuses(ValueError, "contiguous and apart", step, *one, ld, e1, case.s0.transpose(2, 3).contiguous().transpose(2, 3))
    refuses(ValueError, "contiguous and apart", step, *one, ld, e1, case.s0.expand(2, -1, -1, -1))
    refuses(ValueError, "slots", step, *(t.repeat(2, 1, 1, 1) for t in one), ld, e1, case.s0)
    refuses(ValueError, "state_index", step, *one, ld, e1, case.s0, state_index=torch.tensor([0, 0]))
    refuses(TypeError, "new_index", step, *one, ld, e1, case.s0, new_index=torch.tensor([0.]))
    refuses(ValueError, "gate", step, *one, ld, e1, case.s0, gate=torch.zeros(1, 2, 1, 4, dtype=BF16))
    refuses(TypeError, "gate", step, *one, ld, e1, case.s0, gate=torch.zeros(1, 2, 1, 5))
    refuses(ValueError, "without a gate", step, *one, ld, e1, case.s0, norm_weight=torch.ones(5))
    refuses(RuntimeError, "no gradient is defined", step, one[0].clone().requires_grad_(), *one[1:], ld, e1, case.s0)
    refuses(RuntimeError, "no gradient is defined", step, *one, ld, e1, case.s0.clone().requires_grad_())

    x = torch.zeros(1, 2, 3, 8)
    refuses(ValueError, "4-D", gated_head_norm, x[0], x[0])
    refuses(ValueError, "must match", gated_head_norm, x, x[:, :1])
    refuses(TypeError, "gate", gated_head_norm, x.half(), x)
    refuses(TypeError, "weight", gated_head_norm, x, x, torch.ones(8, dtype=F16))
    refuses(ValueError, "weight", gated_head_norm, x, x, torch.ones(3, 8))
    refuses(ValueError, "1 to 512", gated_head_norm, torch.zeros(1, 1, 1, 513), torch.zeros(1, 1, 1, 513))


# ---------------------------------------------------------------- the C ABI's host checks: none of these launches anything

def _desc(**kw):
    d = _lib.PopeLinear(B=2, N=100, Hq=4, Hk=2, D=64, R=32, Dv=48, dtype=2, scale=1.0)
    for n, cols, heads in (("q_s", 64, 4), ("k_s", 64, 2), ("v_s", 48, 2), ("o_s", 48, 4), ("do_s", 48, 4), ("dq_s", 64, 4), ("dk_s", 64, 2), ("dv_s", 48, 2)):
        getattr(d, n)[:] = [heads * 100 * cols, 100 * cols, cols]
    d.f_s[:] = [0, 32]
    d.bias_sh = 32
    for n, v in kw.items():
        if isinstance(v, tuple):
            getattr(d, n)[:] = v
        else:
            setattr(d, n, v)
    return d


def _error():
    buf = ctypes.create_string_buffer(256)
    _lib.lib().pope_last_error(buf, 256)
    return buf.value


def test_abi_refuses():
    lib = _lib.lib()
    size = (ctypes.c_size_t * 2)()
    assert lib.pope_linear_bytes(ctypes.byref(_desc()), 0, 1, 1, size) == 0 and size[0] > 0 and size[1] > 0
    for bad in (dict(B=0), dict(N=-1), dict(Hq=3), dict(Hk=0), dict(D=0), dict(D=257), dict(Dv=0), dict(Dv=300), dict(R=65), dict(R=-1), dict(dtype=7), dict(Hq=1 << 17),
                dict(q_s=(0, 0, 1 << 22)), dict(k_s=(-1, 0, 0)), dict(bias_sh=-1), dict(f_s=(0, 1 << 22))):
        assert lib.pope_linear_bytes(ctypes.byref(_desc(**bad)), 0, 1, 1, size) != 0, bad
        assert _error()
    assert lib.pope_linear_bytes(None, 0, 0, 0, size) != 0 and lib.pope_linear_bytes(ctypes.byref(_desc()), 0, 0, 0, None) != 0
    null, some = None, ctypes.c_void_p(4096)
    d = ctypes.byref(_desc())
    fwd = lambda q=some, f=some, o=some, last=null, ws=some, n=1 << 40, desc=d: lib.pope_linear_fwd(desc, q, some, some, f, some, null, null, null, null, o, last, ws, n, null)
    assert fwd(q=null) and fwd(f=null) and fwd(o=null) and fwd(ws=null) and fwd(n=16) and fwd(ws=ctypes.c_void_p(4100))
    empty = ctypes.byref(_desc(N=0))
    assert fwd(desc=empty) == 0 and fwd(desc=empty, last=some) != 0
    bwd = lambda dout=some, kept=some, kn=1 << 40, dq=some, ws=some, n=1 << 40: lib.pope_linear_bwd(
        d, dout, null, some, some, some, some, some, null, null, null, null, kept, kn, dq, some, some, null, null, null, ws, n, null)
    assert bwd(dout=null) and bwd(kept=null) and bwd(kn=8) and bwd(dq=null) and bwd(ws=null) and bwd(n=8)
    one = _desc(N=1)
    step = lambda desc=one, state=some, slots=2, slot=2 * 96 * 48, o=some, norm=null, gate=null: lib.pope_linear_step(
        ctypes.byref(desc), some, some, some, some, some, null, state, slots, slot, null, null, norm, gate, null, o, null)
    assert step(desc=_desc()) and step(state=null) and step(slots=0) and step(slots=1) and step(slot=2 * 96 * 48 - 1) and step(o=null) and step(gate=some)
    norm = _lib.PopeGatedNorm(B=2, H=4, N=1, cols=47, dtype=2, weight_rows=1, eps=1e-5)
    assert step(norm=ctypes.byref(norm), gate=some)

    g = lambda **kw: _lib.PopeGatedNorm(**{**dict(B=2, H=4, N=3, cols=48, dtype=2, weight_rows=1, eps=1e-5), **kw})
    n = ctypes.c_size_t()
    assert lib.pope_gated_norm_bytes(ctypes.byref(g()), ctypes.byref(n)) == 0 and n.value > 0
    for bad in (dict(B=-1), dict(H=0), dict(cols=0), dict(cols=513), dict(dtype=5), dict(weight_rows=2), dict(weight_sh=-1)):
        assert lib.pope_gated_norm_bytes(ctypes.byref(g(**bad)), ctypes.byref(n)) != 0, bad
    assert lib.pope_gated_norm_fwd(ctypes.byref(g()), null, some, null, some, null) != 0
    assert lib.pope_gated_norm_fwd(ctypes.byref(g(B=0)), null, null, null, null, null) == 0
    assert lib.pope_gated_norm_bwd(ctypes.byref(g()), some, some, some, null, some, some, some, some, 1 << 40, null) != 0    # a weight's gradient without one
    assert lib.pope_gated_norm_bwd(ctypes.byref(g()), some, some, some, some, some, some, some, some, 8, null) != 0

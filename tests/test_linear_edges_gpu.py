"""Inputs of the linear attention, its step and the gated norm that few calls have, against 64-bit formulas (bounds: linear_common)."""
import math

import pytest
import torch
import torch.nn.functional as F

import linear_common as L
import pope_amd
from linear_common import Case, check, half, run
from pope_amd import gated_head_norm, linear_attn_step_with_pope, linear_attn_with_pope

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "fp16", "fp32"])


# ---------------------------------------------------------------- broadcast inputs

@pytest.mark.parametrize("bias_dtype", [F32, BF16])
def test_gradients_of_expanded_angles_and_biases(cuda, bias_dtype):
    """One bias for all heads and one table for all batches, as views that repeat them: a gradient row for each row of the views."""
    case = Case(cuda, B=3, Hq=6, Hk=3, N=150, D=32, R=16, Dv=24, dtype=F16, bias_heads=1)
    one_bias, table = case.bias.to(bias_dtype), case.freqs
    case.freqs = table.expand(3, -1, -1)
    case.bias = one_bias.float().expand(3, -1)
    val, tol = case.exact()
    case.bias = one_bias.expand(3, -1)
    got = run(pope_amd, case)
    for n in val:
        own = half(bias_dtype) * val[n].abs() if n == "d_bias" and bias_dtype != F32 else 0.0
        check(got[n], val[n], case.bound(n, val[n], tol[n]) + own, n)
    # through the expand: the rows' sum
    b = one_bias.clone().requires_grad_()
    o, last = linear_attn_with_pope(case.q, case.k, case.v, case.ld, (table, b.expand(3, -1)), return_state=True)
    g, = torch.autograd.grad([o, last], b, [case.do, case.ds])
    own = 0.0 if bias_dtype == F32 else 2 * half(bias_dtype) * val["d_bias"].abs().sum(0, keepdim=True) * 1.01
    check(g, val["d_bias"].sum(0, keepdim=True), case.bound("d_bias", val["d_bias"].sum(0, keepdim=True), tol["d_bias"].sum(0, keepdim=True)) + own, "bias")
    # the op, as traced programs call it
    x = {n: t.detach().requires_grad_() for n, t in case.leaves().items()}
    o, last, _ = torch.ops.pope_amd.linear_fwd(x["q"], x["k"], x["v"], x["freqs"], x["bias"], case.ld, None, None, None, case.scale, True, False)
    g = dict(zip(x, torch.autograd.grad([o, last], list(x.values()), [case.do, case.ds])))
    for n in x:
        assert torch.equal(g[n], got["d_" + n]), n


# ---------------------------------------------------------------- one row, at any stride

@TYPES
def test_one_row_of_any_stride(cuda, dtype):
    """The row dim of one row may have any stride: nothing reads or writes by it."""
    for gated in (False, True):
        case = Case(cuda, B=2, Hq=4, Hk=2, N=1, D=48, R=16, Dv=40, dtype=dtype, initial=True)
        gate = torch.randn(2, 4, 1, 40, generator=torch.Generator().manual_seed(2)).to(cuda, dtype)

        def call(turn):
            x = {n: turn(t).detach().requires_grad_() for n, t in dict(case.leaves(), gate=gate).items()}
            o, last = linear_attn_with_pope(x["q"], x["k"], x["v"], case.ld, (x["freqs"], x["bias"]), initial_state=x["s0"], return_state=True, gate=x["gate"] if gated else None)
            used = [t for n, t in x.items() if gated or n != "gate"]
            return [o, last, *torch.autograd.grad([o, last], used, [turn(case.do.to(o.dtype)), case.ds])]

        far = lambda t: t.as_strided(t.shape, (*t.stride()[:2], 2 ** 33 + 1, t.stride(3)), t.storage_offset()) if t.ndim == 4 and t.shape[2] == 1 else t
        assert far(case.do).stride(2) > 2 ** 33
        for a, b in zip(call(lambda t: t), call(far)):
            assert torch.equal(a, b)


# ---------------------------------------------------------------- values next to the largest

@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("name,column", [("q", 20), ("q", 3), ("k", 20), ("k", 3), ("v", 20), ("do", 20)])
def test_fp32_values_next_to_the_largest(cuda, name, column, sign):
    """The largest fp32 value in a row: every output is finite and the formula's of the largest bf16, as which it counts (2^-8 below); the
    bounds of rows that do not depend on it are as small as ever.  The other operands are small, so that the formula is finite."""
    most = torch.finfo(BF16).max
    for at in (0, 37, 140, 209):
        case = Case(cuda, B=2, N=210, D=32, R=16, Dv=40, dtype=F32, seed=at)
        for n in ("q", "k", "v", "do"):
            if n != name:
                setattr(case, n, getattr(case, n) * 2.0 ** -8)
        case.ds = case.ds * 2.0 ** -8
        t = getattr(case, name)
        t[0, 0, at, column] = sign * most
        val, tol = case.exact()
        t[0, 0, at, column] = sign * torch.finfo(F32).max
        got = run(pope_amd, case)
        for n in val:
            assert val[n].isfinite().all() and got[n].isfinite().all(), (n, at)
            check(got[n], val[n], case.bound(n, val[n], tol[n]), f"{n} {at}")


@pytest.mark.parametrize("size", [1e18, 1e20, 1e30, 1e37])
@pytest.mark.parametrize("dim", [7, 64, 200, 512])
@pytest.mark.parametrize("x_dtype,dtype", [(F32, F32), (F32, BF16), (F32, F16), (BF16, BF16)])
def test_norm_of_large_rows(cuda, dim, size, x_dtype, dtype):
    """Rows whose squares pass fp32's range, among ordinary ones: fp32 arithmetic and one rounding, as for all (512 2^-24 of the sum of
    squares), above 2^-126, where fp32 and bf16 lose bits."""
    g = torch.Generator().manual_seed(dim)
    x, gate, dy = (torch.randn(2, 3, 9, dim, generator=g).to(cuda) for _ in range(3))
    x[:, :, ::2] *= size
    x[0, 0, 1, :3] = torch.finfo(BF16).max
    x, gate, dy = x.to(x_dtype), gate.to(dtype), dy.to(dtype)
    w = torch.randn(3, dim, generator=g).to(cuda)
    leaves = [t.requires_grad_() for t in (x, gate, w)]
    y = gated_head_norm(x, gate, w)
    got = torch.autograd.grad(y, leaves, dy)
    e = [t.detach().double().requires_grad_() for t in leaves]
    want = L.norm64(*e, 1e-5)
    grads = torch.autograd.grad(want, e, dy.double())
    u, small = half(dtype), 2.0 ** -126 + (2.0 ** -25 if dtype == F16 else 0)
    check(y.detach(), want.detach(), (u + 1e-4) * want.detach().abs() + small, "y")
    with torch.no_grad():
        a = (dy.double() * e[2][:, None, :] * F.silu(e[1])).abs()
        rms = (e[0].square().mean(-1, keepdim=True) + 1e-5).sqrt()
        mags = [(a + e[0].abs() / rms * (a * e[0].abs() / rms).mean(-1, keepdim=True)) / rms, (dy.double() * e[2][:, None, :] * e[0] / rms).abs() * 1.1,
                (dy.double() * e[0] / rms * F.silu(e[1])).abs().sum((0, 2))]
    for n, t, got_t, want_t, mag in zip(("dx", "dgate", "dweight"), leaves, got, grads, mags):
        assert got_t.dtype == t.dtype
        check(got_t, want_t, half(t.dtype) * want_t.abs() + 1e-4 * mag + small, n)


@TYPES
def test_gated_step_of_large_states(cuda, dtype):
    case = Case(cuda, B=3, Hq=4, Hk=2, N=1, D=40, R=16, Dv=72, dtype=dtype, initial=True)
    gate, w = torch.randn(3, 4, 1, 72, device=cuda).to(dtype), torch.rand(72, device=cuda) + 0.5
    for size in (1.0, 2.0 ** 66, 2.0 ** 110):
        state = case.s0 * size
        y = linear_attn_step_with_pope(case.q, case.k, case.v, case.ld, case.emb(), state.clone(), gate=gate, norm_weight=w)
        o, _ = L.attend64(L.expand64(case.q, case.freqs, None, 16), L.expand64(case.k, case.freqs, case.bias, 16), case.v.double(), case.decay64(), case.scale, None,
                          state.double(), case.seqs)
        a, _ = L.attend64(L.expand64(case.q, case.freqs, None, 16).abs() + 0.05, L.expand64(case.k, case.freqs, case.bias, 16).abs() + 0.05, case.v.double().abs(),
                          case.decay64(), case.scale, None, state.double().abs(), case.seqs)
        # fp32 sums (2e-5 of absolute values, as in linear_common), relative to a row's size, and the output's rounding
        rms = (o.square().mean(-1, keepdim=True) + 1e-5).sqrt()
        want = L.norm64(o, gate, w, 1e-5)
        e = 2e-5 * a / rms
        check(y, want, 2 * (e * (w * F.silu(gate.double())).abs() + want.abs() * e.square().mean(-1, keepdim=True).sqrt()) + (half(dtype) + 1e-4) * want.abs() + 2.0 ** -25, size)


def test_no_rows_have_gradients(cuda):
    from test_linear_edges_cpu import no_rows_have_gradients
    no_rows_have_gradients(cuda)


# ---------------------------------------------------------------- buffers that are mostly empty

@TYPES
@pytest.mark.parametrize("lens,lead,tail", [([60, 40], 1500, 3400), ([0, 0], 0, 4097), ([1], 4100, 0), ([3] * 70, 5, 1), ([2500], 700, 900)])
def test_rows_of_no_sequence_are_zeros(cuda, lens, lead, tail, dtype):
    """Every output and gradient row outside every sequence is written, over memory that held NaN, with shared and single heads, wide and odd rows."""
    for kw in (dict(Hq=4, Hk=2, D=40, R=20, Dv=48), dict(Hq=1, Hk=1, D=130, R=65, Dv=250), dict(Hq=6, Hk=2, D=9, R=3, Dv=7)):
        case = Case(cuda, lens=lens, lead=lead, tail=tail, dtype=dtype, initial=True, **kw)
        stale = [torch.full((n,), math.nan, device=cuda) for n in (1 << 16, 1 << 18, 1 << 20, 1 << 22) for _ in range(4)]
        del stale
        got = run(pope_amd, case, head_first=False)
        outside = torch.ones(case.q.shape[2], dtype=torch.bool, device=cuda)
        outside[lead:lead + sum(lens)] = False
        for n in ("o", "d_q", "d_k", "d_v"):
            assert torch.equal(got[n][:, :, outside], torch.zeros_like(got[n][:, :, outside])), n
        assert not got["d_freqs"][outside].any()
        L.compare(got, case)


# ---------------------------------------------------------------- forward-mode derivatives

def test_tangents_are_refused_under_transforms(cuda):
    """There is no forward-mode derivative: torch's would be 0, without a word."""
    case = Case(cuda, B=2, N=70, initial=True, dtype=F32)
    ones = {n: torch.ones_like(t) for n, t in case.leaves().items()}
    for name in case.leaves():
        def f(t):
            x = dict(case.leaves(), **{name: t})
            return linear_attn_with_pope(x["q"], x["k"], x["v"], case.ld, (x["freqs"], x["bias"]), initial_state=x["s0"])
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            torch.func.jvp(f, (case.leaves()[name],), (ones[name],))
        assert torch.equal(torch.func.vmap(f, in_dims=0)(case.leaves()[name][None])[0], f(case.leaves()[name]))   # other transforms are as they were
    gate, w = torch.randn_like(case.do), torch.rand(64, device=cuda)
    for i in range(3):
        args = [case.do, gate, w]
        f = lambda t: gated_head_norm(*args[:i], t, *args[i + 1:])
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            torch.func.jvp(f, (args[i],), (torch.ones_like(args[i]),))

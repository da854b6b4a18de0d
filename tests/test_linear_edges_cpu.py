"""Inputs of the linear attention, its step and the gated norm that few calls have, on CPU tensors, and the kernels' addresses on the host."""
import math
import os
import subprocess

import pytest
import torch

import pope_amd
from linear_common import Case, check, norm64, run

CPU = torch.device("cpu")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_row_addresses(tmp_path):
    exe = str(tmp_path / "check")
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", os.path.join(ROOT, "pope-pytorch_amd", "csrc"), os.path.join(ROOT, "tests", "linear_rows_check.cpp"),
                    "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout


@pytest.mark.parametrize("value", [math.inf, -math.inf, math.nan, "lowest"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_masked_rows_reach_no_gradient(dtype, value):
    case = Case(CPU, B=2, N=150, mask="empty", dtype=dtype, initial=True)
    clean = run(pope_amd, case)
    x = torch.finfo(dtype).min if value == "lowest" else value
    case.k, case.v = (t.masked_fill(~case.mask[:, None, :, None], x) for t in (case.k, case.v))
    got = run(pope_amd, case)
    for n in clean:
        assert torch.equal(got[n], clean[n]), n
    assert not got["d_k"][0].any() and not got["d_v"][0].any()


@pytest.mark.parametrize("size", [1.0, 1e20, 1e37])
def test_norm_of_large_rows(size):
    """Rows whose squares pass fp32's range: fp32 arithmetic on them all the same."""
    g = torch.Generator().manual_seed(3)
    x, gate, dy = (torch.randn(2, 3, 5, 33, generator=g) for _ in range(3))
    x[:, :, ::2] *= size
    w = torch.randn(3, 33, generator=g)
    leaves = [t.requires_grad_() for t in (x, gate, w)]
    y = pope_amd.gated_head_norm(x, gate, w)
    e = [t.detach().double().requires_grad_() for t in leaves]
    want = norm64(*e, 1e-5)
    check(y.detach(), want.detach(), 1e-5 * want.detach().abs() + 1e-7, "y")
    for n, a, b in zip(("dx", "dgate", "dweight"), torch.autograd.grad(y, leaves, dy), torch.autograd.grad(want, e, dy.double())):
        scale = b.abs().amax(-1, keepdim=True) if n == "dx" else 1.0
        check(a, b, 1e-4 * scale + 1e-5 * b.abs(), n)


def no_rows_have_gradients(device):
    for shape, cu in (((2, 4, 0), None), ((0, 4, 5), None), ((1, 4, 0), (0, 0)), ((1, 4, 3), (2, 2))):   # the last: rows of no sequence
        cu = None if cu is None else torch.tensor(cu, dtype=torch.int32, device=device)
        x = {n: torch.randn(*s, device=device).requires_grad_() for n, s in dict(q=(*shape, 8), k=(shape[0], 2, shape[2], 8), v=(shape[0], 2, shape[2], 5), freqs=(shape[2], 4), bias=(2, 4),
                                                                                 s0=(shape[0], 2, 12, 5), gate=(*shape, 5), w=(5,)).items()}
        for gated in (False, True):
            o, last = pope_amd.linear_attn_with_pope(x["q"], x["k"], x["v"], None, (x["freqs"], x["bias"]), initial_state=x["s0"], return_state=True, cu_seqlens=cu,
                                                     gate=x["gate"] if gated else None, norm_weight=x["w"] if gated else None)
            used = list(x) if gated else list(x)[:6]
            g = dict(zip(used, torch.autograd.grad([o.sum() + last.sum()], [x[n] for n in used])))
            for n in used:
                assert g[n].shape == x[n].shape and g[n].dtype == x[n].dtype and bool((g[n] == (1 if n == "s0" else 0)).all()), n


def test_no_rows_have_gradients():
    no_rows_have_gradients(CPU)


def test_gates_are_refused_before_the_attention(monkeypatch):
    case = Case(CPU, N=6, D=8, R=4, Dv=5)
    call = lambda **kw: pope_amd.linear_attn_with_pope(case.q, case.k, case.v, case.ld, case.emb(), **kw)
    gate = torch.randn(1, 2, 6, 5)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):   # of any of the types, whatever the rows'
        assert call(gate=gate.to(dtype), norm_weight=torch.ones(5)).dtype == dtype

    def computed(*a):
        raise AssertionError("the attention ran")

    monkeypatch.setattr(pope_amd.linear, "_linear_torch", computed)
    with pytest.raises(AssertionError):
        call(gate=gate)
    for kind, match, kw in ((ValueError, "gate", dict(gate=gate[..., :4])), (ValueError, "gate", dict(gate=gate.transpose(1, 2))), (ValueError, "gate", dict(gate=gate[0])),
                            (TypeError, "gate", dict(gate=gate.double())), (ValueError, "weight", dict(gate=gate, norm_weight=torch.ones(4))),
                            (TypeError, "weight", dict(gate=gate, norm_weight=torch.ones(5, dtype=torch.float16))),
                            (RuntimeError, "meta", dict(gate=gate.to("meta"))), (RuntimeError, "meta", dict(gate=gate, norm_weight=torch.ones(5, device="meta")))):
        with pytest.raises(kind, match=match):
            call(**kw)


def test_rows_without_a_dim_are_refused():
    for call in (lambda *a: pope_amd.linear_attn_with_pope(*a), lambda *a: pope_amd.linear_attn_step_with_pope(*a, None, None, torch.zeros(1, 2, 1, 1))):
        with pytest.raises(ValueError, match="1 to 256"):
            call(*(torch.zeros(1, 2, 1, 0) for _ in range(3)))
        with pytest.raises(ValueError, match="4-D"):
            call(*(torch.zeros(()) for _ in range(3)))


def test_exact_operands_give_the_formula():
    """linear_rounded without roundings is the formula of linear_common; with those of one part it is off by what bf16 takes."""
    from linear_rounded import outputs
    for shape in (dict(B=2, N=70, mask="random", batch_freqs=True), dict(Hq=4, Hk=2, N=50, D=24, R=10, Dv=9, initial=True, bias_heads=1), dict(N=40, D=12, R=0, Dv=8)):
        case = Case(CPU, dtype=torch.bfloat16, **shape)
        val, _ = case.exact()
        for n, y in outputs(case, 0, own=False).items():
            assert (y - val[n]).norm() <= 1e-12 * val[n].norm(), n
        for n, y in outputs(case, 1).items():
            assert 1e-3 * val[n].norm() <= (y - val[n]).norm() <= 6e-3 * val[n].norm(), n


def test_abi_refuses_rows_beyond_its_counts():
    """Their bytes and segments would pass the integers that hold them: a query answered with what was left of those."""
    import ctypes

    from pope_amd import _lib
    from test_linear_cpu import _desc
    size = (ctypes.c_size_t * 2)()
    ask = lambda packed, **kw: _lib.lib().pope_linear_bytes(ctypes.byref(_desc(**kw)), packed, 1, 1, size)
    assert ask(0, B=1 << 20, N=1 << 28, Hq=32768, Hk=32768) != 0
    assert ask(0, B=1 << 20, N=1 << 20, Hq=2, Hk=1) != 0
    assert ask(0, B=1 << 20, N=1 << 19, Hq=2, Hk=1) == 0 and size[0] >= 3 * (1 << 39) * 96 * 2
    assert ask(1, B=1 << 16, N=1 << 20, Hq=64, Hk=64) == 0   # sequences of packed rows are not rows
    assert ask(1, B=1, N=1 << 28, Hq=4, Hk=4) == 0 and size[0] >= 8 * (1 << 28) * 96 * 2

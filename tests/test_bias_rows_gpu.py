"""Gradients of biases whose rows are views, one row for all heads or part of wider rows: the same bits as those of a copy with rows side
by side, in deterministic mode, and what a copy's row gradients sum to."""
import pytest
import torch

from pope_amd import apply_pope_to_qk
from pope_amd.attention import flash_attn_with_pope
from pope_amd.hip_pope import hip_compute_qk_similarity

pytestmark = pytest.mark.gpu

VIEWS = {"repeated": lambda t: t[:1].expand(4, -1), "of_wider_rows": lambda t: torch.cat((t, t, t), 1)[:, t.shape[1]:2 * t.shape[1]]}


@pytest.fixture(autouse=True)
def deterministic():
    torch.use_deterministic_algorithms(True, warn_only=True)
    yield
    torch.use_deterministic_algorithms(False)


def _inputs(cuda, dtype, D, R, Hq=8, N=170):
    g = torch.Generator().manual_seed(D + R)
    q, k, v = (torch.randn(2, h, N, D, generator=g).to(cuda, dtype) for h in (Hq, 4, 4))
    freqs = (torch.arange(N).float()[:, None] * 10000 ** -(torch.arange(R).float() / R)).to(cuda)
    return q, k, v, freqs, (-2 * torch.rand(4, R, generator=g)).to(cuda)


CALLS = {
    "flash": (torch.bfloat16, lambda q, k, v, f, b: flash_attn_with_pope(q, k, v, (f, b))),
    "flash_causal_fp32": (torch.float32, lambda q, k, v, f, b: flash_attn_with_pope(q, k, v, (f, b), causal=True)),
    "similarity": (torch.float32, lambda q, k, v, f, b: hip_compute_qk_similarity(q, k, f, b)),
    "polar": (torch.float16, lambda q, k, v, f, b: torch.cat([t.flatten() for t in apply_pope_to_qk((f, b), q, k)])),
}


@pytest.mark.parametrize("view", VIEWS)
@pytest.mark.parametrize("dims", [(64, 32), (40, 20), (192, 64)])
@pytest.mark.parametrize("call", CALLS)
def test_gradient_rows(cuda, call, dims, view):
    dtype, f = CALLS[call]
    q, k, v, freqs, bias = _inputs(cuda, dtype, *dims)
    rows = VIEWS[view](bias)
    copy = rows.clone(memory_format=torch.contiguous_format).requires_grad_()
    rows = rows.detach().requires_grad_()
    out = f(q, k, v, freqs, copy)
    up = torch.randn(out.shape, generator=torch.Generator(device=cuda).manual_seed(1), device=cuda).to(out.dtype)
    want, = torch.autograd.grad(out, copy, up)
    for seen in (rows, VIEWS[view](bias).detach().requires_grad_()):
        got, = torch.autograd.grad(f(q, k, v, freqs, seen), seen, up)
        assert got.shape == want.shape and torch.equal(got, want)
    assert want.abs().amin(1).gt(0).all()   # every row has one


@pytest.mark.parametrize("view", VIEWS)
def test_gradient_rows_of_the_ops(cuda, view):
    """The ops, as traced programs call them, through their own autograd."""
    ops = torch.ops.pope_amd
    q, k, v, freqs, bias = _inputs(cuda, torch.bfloat16, 64, 32)
    calls = {"flash": lambda b: ops.flash_fwd(q, k, v, freqs, b, None, False, 0.125)[0],
             "similarity": lambda b: ops.sim_fwd(q.float(), k.float(), freqs, b, False),
             "polar": lambda b: torch.cat([t.flatten() for t in ops.polar_fwd(q, k, freqs, b, False)])}
    for name, f in calls.items():
        rows = VIEWS[view](bias)
        copy = rows.clone(memory_format=torch.contiguous_format).requires_grad_()
        rows = rows.detach().requires_grad_()
        out = f(copy)
        up = torch.randn(out.shape, generator=torch.Generator(device=cuda).manual_seed(1), device=cuda).to(out.dtype)
        assert torch.equal(torch.autograd.grad(f(rows), rows, up)[0], torch.autograd.grad(out, copy, up)[0]), name

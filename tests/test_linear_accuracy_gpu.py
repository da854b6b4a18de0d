"""How far the linear attention is from its formula, in 2-norms: no further than the roundings that it says it makes (linear_rounded).  The
bounds of linear_common hold value by value, for roundings that all add up; sums that all but cancel, as a bias's gradient, are far
smaller than those."""
import pytest
import torch

import linear_common as L
import pope_amd
from linear_common import Case, check, half, run
from linear_rounded import check_norms
from pope_amd import linear_attn_with_pope

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "fp16", "fp32"])

SHAPES = {   # of more than 32 rows, and enough of them for their roundings to even out
    "one_chunk": dict(B=2, N=64),
    "chunk_and_a_row": dict(B=2, N=65, batch_freqs=True),
    "masked": dict(B=2, N=300, mask="random"),
    "one_bias": dict(B=2, N=150, Hq=6, Hk=3, bias_heads=1, mask="random"),
    "segments": dict(Hq=1, Hk=1, N=1000, R=64, initial=True),
    "grouped": dict(B=2, Hq=6, Hk=2, N=300, D=48, R=24, Dv=33, mask="random", initial=True),
    "heads_share_rows": dict(B=3, Hq=24, Hk=8, N=200, D=32, R=16, Dv=32, mask="random"),
    "wide": dict(N=140, D=256, R=256, Dv=256, Hq=1, Hk=1, initial=True),
    "wide_values": dict(N=170, D=20, R=20, Dv=250, initial=True, past=5000),
    "wide_rows": dict(N=100, D=200, R=101, Dv=19, Hq=2, Hk=1),
    "no_rotation": dict(Hq=3, Hk=1, N=200, D=100, R=0, Dv=7),
    "long": dict(Hq=4, Hk=4, N=2500, mask="random"),
    "no_decay": dict(Hq=2, Hk=2, N=700, decay=None),
}


@TYPES
@pytest.mark.parametrize("shape", SHAPES)
def test_norms(cuda, shape, dtype):
    case = Case(cuda, dtype=dtype, **SHAPES[shape])
    check_norms(run(pope_amd, case), case, 1 if dtype == BF16 else 2, *case.exact())


@pytest.mark.parametrize("heads", [1, 2])
@pytest.mark.parametrize("bias_dtype", [BF16, F16], ids=["bias_bf16", "bias_fp16"])
@TYPES
def test_biases_of_16_bits(cuda, dtype, bias_dtype, heads):
    """A bias is read, and its gradient written, in its own type."""
    case = Case(cuda, B=2, Hq=4, Hk=2, N=180, D=48, R=32, Dv=40, dtype=dtype, bias_heads=heads, mask="random")
    case.bias = case.bias.to(bias_dtype)
    got = run(pope_amd, case)
    val, tol = case.exact()
    assert got["d_bias"].dtype == bias_dtype
    for n in val:
        own = half(bias_dtype) * val[n].abs() * 1.01 if n == "d_bias" else 0.0
        check(got[n], val[n], case.bound(n, val[n], tol[n]) + own, n)
    check_norms(got, case, 1 if dtype == BF16 else 2, val, tol)


@pytest.mark.parametrize("rows", [1, 5, 31, 32])
@pytest.mark.parametrize("packed", [False, True])
def test_few_bf16_rows_in_two_parts(cuda, rows, packed):
    """Up to 32 bf16 rows are as exact as fp16 ones: two parts, 6 2^-16 of absolute values, and the outputs' rounding."""
    kw = dict(lens=[rows // 2, rows - rows // 2], D=40, R=20, Dv=48) if packed else dict(B=3, N=rows, mask="random" if rows > 1 else None)
    case = Case(cuda, Hq=4, Hk=2, dtype=BF16, initial=True, **kw)
    got = run(pope_amd, case)
    val, tol = case.exact()
    for n in val:
        rel = 3 * 2.0 ** -16 if n in ("states", "d_s0") else 6 * 2.0 ** -16
        own = half(BF16) if n in ("o", "d_q", "d_k", "d_v") else 2.0 ** -24
        check(got[n], val[n], (rel + 2e-5) * tol[n] * (1 + own) + own * val[n].abs() + 1e-30, n)


@pytest.mark.parametrize("shape", [dict(B=40, Hq=8, Hk=8), dict(B=9, Hq=64, Hk=32, D=24, R=8, Dv=20)])
def test_few_bf16_rows_are_as_exact_in_large_batches(cuda, shape):
    case = Case(cuda, N=17, dtype=BF16, **shape)
    got = run(pope_amd, case)
    val, tol = case.exact()
    for n in ("o", "d_q", "d_k", "d_v"):
        own = half(BF16)
        check(got[n], val[n], (6 * 2.0 ** -16 + 2e-5) * tol[n] * (1 + own) + own * val[n].abs() + 1e-30, n)


def test_gated_bf16_gradients_in_two_parts(cuda):
    """bf16 rows under a gate: what gradients are off by beyond their own rounding.  Operands of two parts leave 6e-6 of the sums' norms;
    the norm behind them raises that in rows that are short beside their terms, by 100 in the worst one: 1e-3 over all allows
    more than that, and operands of one part leave twice as much, 2e-3, before the norm raises it."""
    case = Case(cuda, B=2, Hq=4, Hk=2, N=170, D=48, R=16, Dv=40, dtype=BF16, mask="random", initial=True)
    gate, w = torch.randn_like(case.do), (torch.rand(4, 40, device=cuda) + 0.5)
    x = {n: t.clone().requires_grad_() for n, t in {**case.leaves(), "gate": gate, "w": w}.items()}
    y, last = linear_attn_with_pope(x["q"], x["k"], x["v"], case.ld, (x["freqs"], x["bias"]), gate=x["gate"], norm_weight=x["w"], return_state=True,
                                    **dict(case.kw(), initial_state=x["s0"]))
    got = torch.autograd.grad([y, last], list(x.values()), [case.do, case.ds])
    e = {n: t.detach().double().requires_grad_() for n, t in x.items()}
    o, last = L.attend64(L.expand64(e["q"], e["freqs"], None, case.R), L.expand64(e["k"], e["freqs"], e["bias"], case.R), e["v"], case.decay64(), case.scale, case.mask,
                         e["s0"], case.seqs)
    y64 = L.norm64(o, e["gate"], e["w"], 1e-5)
    want = torch.autograd.grad([y64, last], list(e.values()), [case.do.double(), case.ds.double()])
    for n, a, b in (("y", y.detach(), y64.detach()), *zip(x, got, want)):
        rounding = (b.to(a.dtype).double() - b).norm()
        beyond = ((a.double() - b).norm() ** 2 - rounding ** 2).clamp_min(0.0).sqrt()
        assert beyond <= 1e-3 * b.norm(), (n, (beyond / b.norm()).item())

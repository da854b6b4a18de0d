"""Linear attention with head decays, its step and the gated norm on the GPU, against 64-bit formulas (bounds: linear_common)."""
import math

import pytest
import torch
import torch.nn.functional as F

import linear_common as L
import pope_amd
from linear_common import Case, check, compare, half, run
from pope_amd import gated_head_norm, linear_attn_step_with_pope, linear_attn_with_pope

pytestmark = pytest.mark.gpu

BF16, F16, F32, I32 = torch.bfloat16, torch.float16, torch.float32, torch.int32
INF, NAN = math.inf, math.nan
TYPES = pytest.mark.parametrize("dtype", [BF16, F16, F32], ids=["bf16", "fp16", "fp32"])

SHAPES = {
    "one_row": dict(N=1, D=16, R=16, Dv=16, initial=True),
    "one_column": dict(N=70, D=1, R=1, Dv=1, initial=True),
    "63_rows": dict(B=2, N=63, mask="random"),
    "64_rows": dict(B=2, N=64, bias_heads=1),
    "65_rows_empty": dict(B=2, N=65, mask="empty", initial=True, batch_freqs=True),
    "grouped_odd": dict(B=2, Hq=6, Hk=2, N=300, D=48, R=10, Dv=33, mask="random", initial=True),
    "no_rotation": dict(Hq=3, Hk=1, N=200, D=100, R=0, Dv=7),
    "96_columns": dict(Hq=4, Hk=2, N=129, D=96, R=24, Dv=96, batch_freqs=True, B=2),
    "wide": dict(N=140, D=256, R=256, Dv=256, Hq=1, Hk=1, initial=True),
    "wide_values": dict(N=70, D=20, R=12, Dv=250, initial=True, past=5000),
    "wide_rows": dict(N=100, D=200, R=101, Dv=19, Hq=2, Hk=1),
    "many_segments": dict(Hq=1, Hk=1, N=1000, R=64, initial=True),
    "longer_segments": dict(B=2, Hq=16, Hk=16, N=1100, D=32, R=16, Dv=32),
    "heads_share_wide_rows": dict(B=40, Hq=24, Hk=8, N=64, D=130, R=6, Dv=20),
    "heads_share_rows": dict(B=9, Hq=24, Hk=8, N=500, D=32, R=16, Dv=32, mask="random"),
}


@TYPES
@pytest.mark.parametrize("shape", SHAPES)
def test_rows(cuda, shape, dtype):
    case = Case(cuda, dtype=dtype, **SHAPES[shape])
    compare(run(pope_amd, case), case)


@TYPES
@pytest.mark.parametrize("lens,lead,tail", [([0, 1, 64, 65, 0, 130], 0, 0), ([5, 200, 0], 3, 9), ([1], 0, 0), ([0, 0], 2, 0), ([1] * 40, 0, 1), ([700, 30, 640], 0, 64)])
def test_packed(cuda, lens, lead, tail, dtype):
    case = Case(cuda, lens=lens, lead=lead, tail=tail, D=40, R=20, Dv=48, Hq=4, Hk=2, dtype=dtype, initial=True)
    got = run(pope_amd, case, head_first=False)
    compare(got, case)
    outside = torch.ones(case.q.shape[2], dtype=torch.bool, device=cuda)
    outside[lead:lead + sum(lens)] = False
    for n in ("o", "d_q", "d_k", "d_v"):
        assert not got[n][:, :, outside].any(), n
    assert not got["d_freqs"][outside].any()


@TYPES
def test_packed_with_a_mask(cuda, dtype):
    case = Case(cuda, lens=[100, 3, 0, 61], lead=1, tail=2, Hq=4, Hk=2, dtype=dtype, initial=True, mask="random")
    case.mask[0, 101:104] = False   # nothing is left of the second sequence
    compare(run(pope_amd, case), case)


def test_decreasing_bounds_stay_in_range(cuda):
    case = Case(cuda, lens=[30, 40, 50], tail=5)
    for bad in ([0, 90, 20, 125], [-7, 10, 400, 125], [125, 0, 0, 0], [2 ** 31 - 1, -2 ** 31, 5, 9]):
        case.cu = torch.tensor(bad, dtype=I32, device=cuda)
        run(pope_amd, case)
    torch.cuda.synchronize()


@TYPES
@pytest.mark.parametrize("decay", [None, [0.0, 0.0], [-INF, -1e-8], [-30.0, -1e-3], [0.001, -5e-7]])
def test_decays(cuda, decay, dtype):
    case = Case(cuda, N=260, decay=decay, dtype=dtype, initial=True)
    compare(run(pope_amd, case), case)


@pytest.mark.parametrize("head_first", [True, False])
@TYPES
def test_strides(cuda, dtype, head_first):
    case = Case(cuda, B=2, N=150, D=40, R=24, Dv=40, dtype=dtype, mask="random")
    want = run(pope_amd, case)
    # slices of one buffer of q, k, v, starting at an odd element
    B, H, N, D = case.q.shape
    buf = torch.zeros(B, N, 3 * H * D + 1, dtype=dtype, device=cuda)
    views = {n: buf[..., 1 + j * H * D:1 + (j + 1) * H * D].unflatten(-1, (H, D)).transpose(1, 2) for j, n in enumerate("qkv")}
    # feature stride of 2
    spread = {n: torch.stack((case.leaves()[n],) * 2, -1).flatten(-2)[..., ::2] for n in "qkv"}
    for x in (views, spread):
        for n in "qkv":
            if x is views:
                x[n].copy_(case.leaves()[n])
        got = run(pope_amd, case, leaves=x, head_first=head_first)
        for n in want:
            assert torch.equal(got[n], want[n]), n
    # one head's keys for all, without copies; rows far apart
    shared = Case(cuda, B=2, N=150, D=40, R=24, Dv=40, dtype=dtype)
    shared.k, shared.v = (t[:1, :1].expand(2, 2, -1, -1) for t in (shared.k, shared.v))
    compare(run(pope_amd, shared), shared)


def test_rows_far_apart(cuda):
    case = Case(cuda, N=3, D=16, R=8, Dv=16)
    want = run(pope_amd, case)
    buf = torch.empty(3, 1 << 23, dtype=BF16, device=cuda)
    q = buf[:, :32].unflatten(1, (2, 16)).permute(1, 0, 2)[None]
    q.copy_(case.q)
    got = run(pope_amd, case, leaves={"q": q})
    for n in want:
        assert torch.equal(got[n], want[n]), n


def test_offsets_beyond_32_bits(cuda):
    case = Case(cuda, B=2, N=130, D=64, R=32, Dv=64, initial=True)
    want = run(pope_amd, case, grads=False)
    buf = torch.empty((1 << 32) + (1 << 20), dtype=BF16, device=cuda)
    far = {}
    for j, n in enumerate("qkv"):
        t = case.leaves()[n]
        far[n] = buf[j * t[0].numel():].as_strided(t.shape, (1 << 32, *t.stride()[1:]))
        far[n].copy_(t)
    got = run(pope_amd, case, grads=False, leaves=far)
    for n in want:
        assert torch.equal(got[n], want[n]), n
    del buf, far
    slots = torch.empty((1 << 31) + (1 << 20), device=cuda).as_strided((3, 2, 96, 64), (1 << 30, 96 * 64, 64, 1))
    near = case.s0[[0, 1, 1]].clone()
    slots.copy_(near)
    with torch.no_grad():
        args = [t[:, :, :1] for t in (case.q, case.k, case.v)]
        index = torch.tensor([2, 0], dtype=I32, device=cuda)
        o = [linear_attn_step_with_pope(*args, case.ld, (case.freqs[:1], case.bias), s, state_index=index) for s in (slots, near)]
    assert torch.equal(o[0], o[1]) and torch.equal(slots, near)


@TYPES
def test_what_is_not_finite_reaches_no_row_before_it(cuda, dtype):
    """Rows before it are as without it (their sums may be in another order), other heads and sequences are the same bits."""
    case = Case(cuda, B=2, N=210, D=32, R=16, Dv=40, dtype=dtype)
    clean = run(pope_amd, case, grads=False)
    val, tol = case.exact(False)
    bound = case.bound("o", val["o"], tol["o"])
    for at in (0, 37, 64, 140, 209):
        for name in "qkv":
            for x in (INF, -INF, NAN):
                t = case.leaves()[name].clone()
                t[0, 0, at, 20] = x
                o = run(pope_amd, case, grads=False, leaves={name: t})["o"]
                check(o[0, :, :at], val["o"][0, :, :at], bound[0, :, :at], f"{name} {at} {x}")
                assert torch.equal(o[1], clean["o"][1]) and torch.equal(o[:, 1], clean["o"][:, 1]), (name, at, x)
                assert not o[0, 0, at].isfinite().all(), (name, at, x)
                if name == "q":
                    assert torch.equal(o[0, 0, at + 1:], clean["o"][0, 0, at + 1:]), (at, x)
    # nor, in gradients, a row behind it
    val, tol = case.exact()
    bound = {n: case.bound(n, val[n], tol[n]) for n in val}
    do = case.do.clone()
    for at in (63, 100, 128):
        case.do = do.clone()
        case.do[0, 0, at, 3] = NAN
        got = run(pope_amd, case)
        for n in ("d_k", "d_v"):
            check(got[n][0, :, at + 1:], val[n][0, :, at + 1:], bound[n][0, :, at + 1:], f"{n} {at}")
            assert got[n][0, 0, at].isnan().any(), (n, at)
        rest = torch.arange(210, device=cuda) != at
        check(got["d_q"][0, :, rest], val["d_q"][0, :, rest], bound["d_q"][0, :, rest], f"d_q {at}")
        assert got["d_q"][0, 0, at].isnan().any(), at


@TYPES
@pytest.mark.parametrize("value", [INF, NAN, "lowest"])
def test_masked_rows_are_not_seen(cuda, dtype, value):
    case = Case(cuda, B=2, N=150, mask="empty", dtype=dtype, initial=True)
    clean = run(pope_amd, case)
    v = torch.finfo(dtype).min if value == "lowest" else value
    case.k, case.v = (t.masked_fill(~case.mask[:, None, :, None], v) for t in (case.k, case.v))
    got = run(pope_amd, case)
    for n in clean:
        assert torch.equal(got[n], clean[n]), n
    assert not got["d_k"][0].any() and not got["d_v"][0].any()


def test_runs_are_the_same_bits(cuda):
    case = Case(cuda, B=2, Hq=8, Hk=4, N=700, mask="random", initial=True)
    a, b = run(pope_amd, case), run(pope_amd, case)
    for n in a:
        assert torch.equal(a[n], b[n]), n


def test_gradients_against_differences(cuda):
    """A central difference of the call and its gradient differ by the formula's own difference error, which 64 bits give, and by the
    outputs' errors over the step (bounds of o and the states against |do| and |ds|), and by the gradients' bounds."""
    case = Case(cuda, N=90, D=16, R=8, Dv=16, dtype=F32, initial=True, seed=5)
    got = run(pope_amd, case)
    val, tol = case.exact()
    g = torch.Generator(device=cuda).manual_seed(1)
    for n, h in (("q", 2 ** -5), ("k", 2 ** -5), ("v", 1.0), ("freqs", 2 ** -6), ("bias", 2 ** -6), ("s0", 1.0)):
        t = case.leaves()[n]
        u = torch.randint(0, 2, t.shape, generator=g, device=cuda).float() * 2 - 1
        own, exact, noise = 0.0, 0.0, 0.0
        for sign in (1, -1):
            moved = t + sign * h * u
            setattr(case, n, moved)
            r = run(pope_amd, case, grads=False)
            e, a = case.exact(False)
            setattr(case, n, t)
            loss = lambda x: (x["o"].double() * case.do.double()).sum() + (x["states"].double() * case.ds.double()).sum()
            own, exact = own + sign * loss(r) / (2 * h), exact + sign * loss(e) / (2 * h)
            for out, up in (("o", case.do), ("states", case.ds)):
                noise = noise + (case.bound(out, e[out], a[out]) * up.double().abs()).sum() / (2 * h)
        direct = (got["d_" + n].double() * u).sum()
        bound = noise + (exact - (val["d_" + n] * u).sum()).abs() + case.bound("d_" + n, val["d_" + n], tol["d_" + n]).sum()
        assert (own - direct).abs() <= bound, (n, own.item(), direct.item(), bound.item())
        assert (own - direct).abs() <= 0.02 * (val["d_" + n].abs().sum()), n


# ---------------------------------------------------------------- through states

@TYPES
def test_pieces_then_steps_are_one_prompt(cuda, dtype):
    """A gated layer over a prompt in pieces, then token by token, beside the whole prompt at once."""
    case = Case(cuda, B=2, Hq=4, Hk=2, N=200, D=48, R=24, Dv=40, dtype=dtype)
    gate, w = torch.randn_like(case.do), torch.rand(4, 40, device=cuda) + 0.5
    kw = dict(norm_weight=w, norm_eps=1e-4)
    with torch.no_grad():
        whole, last = linear_attn_with_pope(case.q, case.k, case.v, case.ld, case.emb(), gate=gate, return_state=True, **kw)
        state, parts = None, []
        for a, z in ((0, 1), (1, 100), (100, 190)):
            o, state = linear_attn_with_pope(*(t[:, :, a:z] for t in (case.q, case.k, case.v)), case.ld, (case.freqs[a:z], case.bias), gate=gate[:, :, a:z],
                                             initial_state=state, return_state=True, **kw)
            parts.append(o)
        for i in range(190, 200):
            parts.append(linear_attn_step_with_pope(*(t[:, :, i:i + 1] for t in (case.q, case.k, case.v)), case.ld, (case.freqs[i:i + 1], case.bias), state,
                                                    gate=gate[:, :, i:i + 1], **kw))
    val, tol = case.exact(False)
    # the norm of o + e is off by |e| / rms, and by |y| times the row's e relative to its rms
    e = (6 * 2.0 ** -16 + 2e-5) * tol["o"]
    rms = (val["o"].square().mean(-1, keepdim=True) + 1e-4).sqrt()
    y = L.norm64(val["o"], gate, w, 1e-4)
    bound = 2 * (e / rms * (w[:, None, :] * F.silu(gate.float())).abs() + y.abs() * (e.square().mean(-1, keepdim=True)).sqrt() / rms) + 2 * half(dtype) * y.abs() + 1e-6
    for got in (whole, torch.cat(parts, 2)):
        check(got, y, bound, "gated o")
    for s in (last, state):
        check(s, val["states"], case.bound("states", val["states"], tol["states"]), "states")


@TYPES
def test_gated_gradients(cuda, dtype):
    """The norm's gradient at o, whose bound is 6 2^-16 of the sums of absolute values: rows here are at least a hundredth of those, so
    dO is off by 1e-2 at most in the worst row and by far less over all; with two-part products and the gradients' rounding
    (half a step) the 2-norms differ by no more than half a step and 2e-3."""
    case = Case(cuda, B=2, Hq=4, Hk=2, N=170, D=48, R=16, Dv=40, dtype=dtype, mask="random", initial=True)
    gate, w = torch.randn_like(case.do), (torch.rand(4, 40, device=cuda) + 0.5)
    x = {n: t.clone().requires_grad_() for n, t in {**case.leaves(), "gate": gate, "w": w}.items()}
    args = dict(case.kw(), initial_state=x["s0"])
    y, last = linear_attn_with_pope(x["q"], x["k"], x["v"], case.ld, (x["freqs"], x["bias"]), gate=x["gate"], norm_weight=x["w"], return_state=True, **args)
    got = torch.autograd.grad([y, last], list(x.values()), [case.do, case.ds])
    e = {n: t.detach().double().requires_grad_() for n, t in x.items()}
    o, last = L.attend64(L.expand64(e["q"], e["freqs"], None, case.R), L.expand64(e["k"], e["freqs"], e["bias"], case.R), e["v"], case.decay64(), case.scale, case.mask,
                         e["s0"], case.seqs)
    want = torch.autograd.grad([L.norm64(o, e["gate"], e["w"], 1e-5), last], list(e.values()), [case.do.double(), case.ds.double()])
    for n, a, b in zip(x, got, want):
        own = half(dtype) if a.dtype == dtype else 0.0
        assert a.dtype == x[n].dtype and (a.double() - b).norm() <= (own + 2e-3) * b.norm(), (n, ((a.double() - b).norm() / b.norm()).item())


@pytest.mark.parametrize("dtype", [BF16, F16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("lens", [None, [1] * 9])
def test_gated_gradients_of_rows_alone(cuda, dtype, lens):
    """Of a sequence of one row o is a multiple of v, and the norm's gradient at right angles to it but for eps: what is left of
    dO . v is `small` of its terms.  dO and the sum are fp32 (16 roundings of 2^-24 together), so d_q and d_k, multiples of it, are off by
    2^-20 / small, and by half a step; a row's k_hat and q_hat are expanded to 2^-16."""
    case = Case(cuda, B=1 if lens else 3, N=1, lens=lens, Hq=4, Hk=2, D=16, R=8, Dv=16, dtype=dtype)
    gate = torch.randn_like(case.do)
    x = {n: t.clone().requires_grad_() for n, t in {**{n: case.leaves()[n] for n in "qkv"}, "gate": gate}.items()}
    y = linear_attn_with_pope(x["q"], x["k"], x["v"], case.ld, case.emb(), gate=x["gate"], **case.kw())
    got = torch.autograd.grad(y, list(x.values()), case.do)
    e = {n: t.detach().double().requires_grad_() for n, t in x.items()}
    o, _ = L.attend64(L.expand64(e["q"], case.freqs, None, case.R), L.expand64(e["k"], case.freqs, case.bias, case.R), e["v"], case.decay64(), case.scale, None, case.zero, case.seqs)
    o.retain_grad()
    (L.norm64(o, e["gate"], None, 1e-5) * case.do.double()).sum().backward()
    dov = o.grad.unflatten(1, (2, 2)) * e["v"][:, None]
    small = (dov.sum(-1).abs() / dov.abs().sum(-1)).flatten(1, 2)[..., None]   # (batch, query heads, n, 1)
    of = {"q": small, "k": small.unflatten(1, (2, 2)).amin(1)}
    for n, t in zip(x, got):
        want, own = e[n].grad, half(dtype)
        if n in of:
            err, lim = (t.double() - want).abs(), own + 2.0 ** -14 + 2.0 ** -20 / of[n]
            size = want.norm(dim=-1, keepdim=True) if n == "q" else want.norm(dim=-1, keepdim=True) * 4
            assert (err <= lim * size + 2.0 ** -24).all(), (n, (err / (lim * size + 2.0 ** -24)).max().item())
        else:
            assert ((t.double() - want).norm() <= (own + 1e-4) * want.norm()), n


# ---------------------------------------------------------------- single tokens

STEPS = {
    "plain": dict(B=3),
    "one_sequence": dict(B=1, Hq=8, Hk=8),
    "grouped": dict(B=5, Hq=6, Hk=2, D=100, R=33, Dv=72),
    "many_queries": dict(B=2, Hq=16, Hk=1, D=64, R=0, Dv=130),
    "wide": dict(B=2, Hq=4, Hk=1, D=256, R=256, Dv=256),
    "one_column": dict(B=2, D=1, R=1, Dv=1),
    "many_sequences": dict(B=130, Hq=8, Hk=4, D=32, R=32, Dv=17),
}


@TYPES
@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("shape", STEPS)
def test_step(cuda, shape, gated, dtype):
    case = Case(cuda, N=1, dtype=dtype, initial=True, batch_freqs=True, past=7000, **STEPS[shape])
    B, Hq, Dv = case.q.shape[0], case.q.shape[1], case.v.shape[3]
    gate = torch.randn(B, Hq, 1, Dv, device=cuda).to(dtype) if gated else None
    w = torch.rand(Hq, Dv, device=cuda) if gated else None
    val, tol = case.exact(False)
    # spaced slots, more of them than sequences, read from the odd ones and written to the even ones
    slots = torch.full((2 * B + 1, case.s0[0].numel() + 8), NAN, device=cuda)[:, :-8].unflatten(1, case.s0.shape[1:])
    slots[1::2] = case.s0
    keep = slots.clone()
    read = torch.arange(1, 2 * B, 2, device=cuda, dtype=I32)
    o = linear_attn_step_with_pope(case.q, case.k, case.v, case.ld, case.emb(), slots, state_index=read, new_index=read - 1, gate=gate, norm_weight=w)
    check(slots[0:-1:2], val["states"], 2e-5 * tol["states"] + 1e-30, "states")   # fp32 arithmetic
    assert torch.equal(slots[1::2], keep[1::2]) and slots[-1].isnan().all()
    e = 2e-5 * tol["o"]
    if not gated:
        check(o, val["o"], e + half(dtype) * val["o"].abs() + 2.0 ** -25, "o")
        return
    rms = (val["o"].square().mean(-1, keepdim=True) + 1e-5).sqrt()
    y = L.norm64(val["o"], gate, w, 1e-5)
    bound = 2 * (e / rms * (w[:, None, :] * F.silu(gate.float())).abs() + y.abs() * e.square().mean(-1, keepdim=True).sqrt() / rms) + 1.01 * half(dtype) * y.abs() + 1e-6
    check(o, y, bound, "gated o")


def test_step_slots(cuda):
    case = Case(cuda, B=6, N=1, initial=True)
    call = lambda state, **kw: linear_attn_step_with_pope(case.q, case.k, case.v, case.ld, case.emb(), state, **kw)
    ints = lambda *x, dtype=I32: torch.tensor(x, dtype=dtype, device=cuda)
    base = case.s0.clone()
    plain = call(base)
    # out of range: output 0 and nothing written; a target that is none is not written
    state = case.s0.clone()
    read, write = ints(0, -1, 6, 2 ** 31 - 1, -2 ** 31, 5), ints(0, 1, 2, 3, 4, 6)
    o = call(state, state_index=read, new_index=write)
    assert torch.equal(o[0], plain[0]) and torch.equal(o[5], plain[5]) and not o[1:5].any()
    assert torch.equal(state[0], base[0]) and torch.equal(state[1:], case.s0[1:])
    # what int32 cannot hold
    o = call(case.s0.clone(), state_index=ints(0, 2 ** 32, 2 ** 32 + 1, -2 ** 40, 4, 5, dtype=torch.int64))
    assert torch.equal(o[[0, 4, 5]], plain[[0, 4, 5]]) and not o[1:4].any()
    # all from one slot, to their own
    state = case.s0.clone()
    o = call(state, state_index=ints(*[5] * 5, 5), new_index=ints(0, 1, 2, 3, 4, 6))
    assert torch.equal(o[5], plain[5]) and torch.equal(state[5], case.s0[5])
    g = case.ld.exp()[:, None, None]
    row = L.expand64(case.k, case.freqs, case.bias, case.R).transpose(2, 3) * case.v.double()
    want = case.s0[5].double() * g.double() + row[:5]
    assert (state[:5].double() - want).abs().max() <= 2e-5 * (case.s0[5].abs().max() + row.abs().max())
    # a version that autograd sees
    before = state._version
    call(state)
    assert state._version > before


def test_step_in_the_other_layout(cuda):
    case = Case(cuda, B=3, Hq=4, Hk=2, N=1, D=30, R=7, Dv=21, initial=True)
    a, b = case.s0.clone(), case.s0.clone()
    gate = torch.randn(3, 1, 4, 21, device=cuda).to(BF16)
    t = lambda x: x.transpose(1, 2)
    o = linear_attn_step_with_pope(case.q, case.k, case.v, case.ld, case.emb(), a, gate=t(gate))
    p = linear_attn_step_with_pope(t(case.q), t(case.k), t(case.v), case.ld, case.emb(), b, gate=gate, head_dimension_at_first=False)
    assert torch.equal(o, t(p)) and torch.equal(a, b)


# ---------------------------------------------------------------- the gated norm

@TYPES
@pytest.mark.parametrize("dim", [1, 7, 12, 64, 100, 256, 300, 511, 512])
@pytest.mark.parametrize("weight", [None, "row", "heads", "heads32"])
def test_norm(cuda, dim, weight, dtype):
    """fp32 arithmetic over up to 512 values and one rounding: a sum of squares is off by 512 2^-24 at most, its root by half that;
    the weight's gradient sums up to B n rows in fp32 and is rounded to the weight's type."""
    B, H, N, eps = 2, 3, 37, 1e-5
    g = torch.Generator().manual_seed(dim)
    for wide in (False, True):
        for head_first in (True, False):
            shape = (B, H, N, dim) if head_first else (B, N, H, dim)
            x, gate, dy = (torch.randn(shape, generator=g).to(cuda) for _ in range(3))
            x, gate, dy = (x if wide else x.to(dtype)), gate.to(dtype), dy.to(dtype)
            w = None if weight is None else torch.randn(*((dim,) if weight == "row" else (H, dim)), generator=g).to(cuda, F32 if weight == "heads32" else dtype)
            x[0, 0, 0] = 0
            gate[0, 0, 1] = 100.
            gate[0, 0, 2] = -100.
            leaves = [t.requires_grad_() for t in (x, gate, w) if t is not None]
            y = gated_head_norm(x, gate, w, eps=eps, head_dimension_at_first=head_first)
            got = torch.autograd.grad(y, leaves, dy)
            e = [t.detach().double().requires_grad_() for t in leaves]
            want = L.norm64(e[0], e[1], e[2] if w is not None else None, eps, head_first)
            u = half(dtype)
            check(y.detach(), want.detach(), (u + 1e-4) * want.detach().abs() + 2.0 ** -25 + 1e-6, "y")
            grads = torch.autograd.grad(want, e, dy.double())
            # dx = (a - x mean(a x) / (mean x^2 + eps)) / rms, a = dy w silu(gate): of absolute values
            with torch.no_grad():
                wf = 1.0 if w is None else (e[2][:, None, :] if w.ndim == 2 and head_first else e[2])
                rms = (e[0].square().mean(-1, keepdim=True) + eps).sqrt()
                a = (dy.double() * wf * F.silu(e[1])).abs()
                mags = [(a + e[0].abs() * (a * e[0].abs()).mean(-1, keepdim=True) / rms ** 2) / rms,
                        (dy.double() * wf * e[0] / rms).abs() * 1.1]
                if w is not None:
                    m = (dy.double() * e[0] / rms * F.silu(e[1])).abs()
                    m = m if head_first else m.transpose(1, 2)
                    mags.append(m.sum((0, 2)) if w.ndim == 2 else m.sum((0, 1, 2)))
            for t, got_t, want_t, mag in zip(leaves, got, grads, mags):
                own = half(got_t.dtype)
                assert got_t.dtype == t.dtype
                check(got_t, want_t, own * want_t.abs() + 1e-4 * mag + 2.0 ** -25 + 1e-6, "gradient")


def test_norm_strides_and_empty(cuda):
    base = torch.randn(2, 3, 40, 2 * 64 + 3, device=cuda).to(BF16)
    x, gate = base[..., 1:65], base[..., 67:131]
    want = gated_head_norm(x.contiguous(), gate.contiguous())
    assert torch.equal(gated_head_norm(x, gate), want)
    assert torch.equal(gated_head_norm(x.mT.contiguous().mT, gate.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)), want)
    assert torch.equal(gated_head_norm(x[:1, :1].expand(2, 3, -1, -1), gate), gated_head_norm(x[:1, :1].expand(2, 3, -1, -1).contiguous(), gate))
    for shape in ((0, 3, 5, 64), (2, 3, 0, 64)):
        x, w = torch.empty(shape, device=cuda, dtype=BF16, requires_grad=True), torch.ones(64, device=cuda, requires_grad=True)
        y = gated_head_norm(x, x.detach(), w)
        assert y.shape == shape
        dx, dw = torch.autograd.grad(y.sum(), (x, w))
        assert dx.shape == shape and not dw.any()


def test_norm_many_rows(cuda):
    """The weight's gradient over many workgroups; twice the same bits."""
    x, gate, dy = (torch.randn(2, 4, 5000, 64, device=cuda) for _ in range(3))
    w = torch.randn(4, 64, device=cuda, requires_grad=True)
    a, b = (torch.autograd.grad(gated_head_norm(x, gate, w), w, dy)[0] for _ in range(2))
    assert torch.equal(a, b)
    m = dy.double() * x.double() * torch.rsqrt(x.double().square().mean(-1, keepdim=True) + 1e-5) * F.silu(gate.double())
    assert ((a.double() - m.sum((0, 2))).abs() <= 1e-5 * m.abs().sum((0, 2))).all()


# ---------------------------------------------------------------- calls

def test_no_rows(cuda):
    q = torch.empty(2, 4, 0, 32, device=cuda, dtype=BF16)
    kv = torch.empty(2, 2, 0, 32, device=cuda, dtype=BF16)
    s0 = torch.randn(2, 2, 32, 32, device=cuda, requires_grad=True)
    o, last = linear_attn_with_pope(q, kv, kv, initial_state=s0, return_state=True)
    assert o.shape == q.shape and torch.equal(last, s0)
    last.sum().backward()
    assert (s0.grad == 1).all()
    assert linear_attn_step_with_pope(q[:0, :, :].new_empty(0, 4, 1, 32), kv.new_empty(0, 2, 1, 32), kv.new_empty(0, 2, 1, 32), None, None, s0.detach()).shape == (0, 4, 1, 32)
    none = torch.zeros(3, dtype=I32, device=cuda)
    o, last = linear_attn_with_pope(q[:1], kv[:1], kv[:1], initial_state=s0, return_state=True, cu_seqlens=none)
    assert o.shape[2] == 0 and torch.equal(last, s0)


def test_types_that_are_converted(cuda):
    case = Case(cuda, N=70, initial=True)
    want = run(pope_amd, case, grads=False)
    o, s = linear_attn_with_pope(case.q, case.k, case.v, case.ld.double(), (case.freqs.double(), case.bias.double()), case.kw()["mask"],
                                 initial_state=case.s0.double(), return_state=True)
    assert torch.equal(o, want["o"]) and torch.equal(s, want["states"])
    # a bias of one row, and float gradients for the parameters' own types
    b = case.bias[0].to(BF16).requires_grad_()
    s0 = case.s0.to(BF16).requires_grad_()
    o = linear_attn_with_pope(case.q, case.k, case.v, case.ld, (case.freqs, b), initial_state=s0)
    o.sum().backward()
    assert b.grad.dtype == BF16 and b.grad.shape == b.shape and s0.grad.dtype == BF16
    packed = Case(cuda, lens=[20, 30])
    want = run(pope_amd, packed, grads=False)["o"]
    packed.cu = packed.cu.long()
    assert torch.equal(run(pope_amd, packed, grads=False)["o"], want)


def test_only_some_gradients(cuda):
    """The states' pass of the backward holds queries more exactly where the initial states' gradient is wanted, so other gradients
    are within their bounds, not the same bits."""
    case = Case(cuda, B=2, N=100, initial=True)
    val, tol = case.exact()
    for n in case.leaves():
        x = {m: t.detach().requires_grad_(m == n) for m, t in case.leaves().items()}
        o, last = linear_attn_with_pope(x["q"], x["k"], x["v"], case.ld, (x["freqs"], x["bias"]), initial_state=x["s0"], return_state=True)
        g, = torch.autograd.grad([o, last], [x[n]], [case.do, case.ds])
        check(g, val["d_" + n], case.bound("d_" + n, val["d_" + n], tol["d_" + n]), n)
    # of o alone, and of the states alone
    for which in ("o", "states"):
        x = {m: t.detach().requires_grad_() for m, t in case.leaves().items()}
        o, last = linear_attn_with_pope(x["q"], x["k"], x["v"], case.ld, (x["freqs"], x["bias"]), initial_state=x["s0"], return_state=True)
        g = torch.autograd.grad(o if which == "o" else last, list(x.values()), case.do if which == "o" else case.ds)
        other = Case(cuda, B=2, N=100, initial=True)
        if which == "o":
            other.ds = torch.zeros_like(other.ds)
        else:
            other.do = torch.zeros_like(other.do)
        for (m, _), t, w in zip(x.items(), g, [run(pope_amd, other)["d_" + m] for m in x]):
            assert torch.equal(t, w), (which, m)


def test_refusals(cuda):
    case = Case(cuda, N=20, initial=True)
    ld = case.ld.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="no gradient is defined for log_decay"):
        linear_attn_with_pope(case.q, case.k, case.v, ld, case.emb())
    with pytest.raises(RuntimeError, match="cpu"):
        linear_attn_with_pope(case.q, case.k.cpu(), case.v, case.ld, case.emb())
    with pytest.raises(RuntimeError, match="cpu"):
        linear_attn_with_pope(case.q, case.k, case.v, case.ld, case.emb(), torch.ones(1, 20, dtype=torch.bool))
    x = case.q.clone().requires_grad_()
    o = linear_attn_with_pope(x, case.k, case.v, case.ld, case.emb())
    g, = torch.autograd.grad(o.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()
    with pytest.raises(RuntimeError, match="no gradient is defined"):
        linear_attn_step_with_pope(x[:, :, :1], case.k[:, :, :1], case.v[:, :, :1], case.ld, (case.freqs[:1], case.bias), case.s0.clone())
    with torch.autograd.forward_ad.dual_level(), pytest.raises((RuntimeError, NotImplementedError)):
        linear_attn_with_pope(torch.autograd.forward_ad.make_dual(case.q, torch.ones_like(case.q)), case.k, case.v, case.ld, case.emb())
    gate = torch.randn_like(case.do).requires_grad_()
    y = gated_head_norm(case.do, gate)
    g, = torch.autograd.grad(y.float().square().sum(), gate, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()


def test_on_another_stream(cuda):
    case = Case(cuda, B=2, N=300, initial=True)
    want = run(pope_amd, case)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = run(pope_amd, case)
    s.synchronize()
    for n in want:
        assert torch.equal(got[n], want[n]), n


def test_captured_training_step(cuda):
    case = Case(cuda, B=2, N=300, mask="random", initial=True)
    x = {n: t.detach().clone().requires_grad_() for n, t in case.leaves().items()}
    gate = torch.randn_like(case.do).requires_grad_()
    w = torch.rand(64, device=cuda).requires_grad_()
    leaves = [*x.values(), gate, w]

    def step():
        o, last = linear_attn_with_pope(x["q"], x["k"], x["v"], case.ld, (x["freqs"], x["bias"]), case.mask, initial_state=x["s0"], return_state=True,
                                        gate=gate, norm_weight=w)
        return [o.detach(), last.detach(), *torch.autograd.grad([o, last], leaves, [case.do, case.ds])]

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for _ in range(2):   # two graphs of the same pool
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=graphs[0].pool() if graphs else None):
            outs.append(step())
        graphs.append(g)
    for it in range(3):
        with torch.no_grad():
            for t in (x["q"], x["v"], gate):
                t.copy_(torch.randn_like(t))
        want = [t.clone() for t in step()]
        torch.cuda.synchronize()
        for j in range(2):
            graphs[j].replay()
            torch.cuda.synchronize()
            for a, b in zip(outs[j], want):
                assert torch.equal(a, b), (it, j)


def test_captured_step(cuda):
    case = Case(cuda, B=4, N=12, Hq=4, Hk=2, initial=True)
    state, eager = case.s0.clone(), case.s0.clone()
    gate = torch.randn_like(case.do)
    args = [t[:, :, :1].clone() for t in (case.q, case.k, case.v, gate)]
    freqs = case.freqs[:1].clone()
    call = lambda s: linear_attn_step_with_pope(*args[:3], case.ld, (freqs, case.bias), s, gate=args[3])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call(case.s0.clone())
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = call(state)
    for i in range(12):
        for t, x in zip(args, (case.q, case.k, case.v, gate)):
            t.copy_(x[:, :, i:i + 1])
        freqs.copy_(case.freqs[i:i + 1])
        want = call(eager)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want) and torch.equal(state, eager), i


def test_compiled(cuda):
    case = Case(cuda, B=2, N=90, mask="random", initial=True)
    gate = torch.randn_like(case.do)

    def f(q, k, v, bias, s0, gate):
        y, last = linear_attn_with_pope(q, k, v, case.ld, (case.freqs, bias), case.mask, initial_state=s0, return_state=True, gate=gate)
        return y.float().square().sum() + last.square().sum()

    def grads(fn):
        x = [t.detach().clone().requires_grad_() for t in (case.q, case.k, case.v, case.bias, case.s0, gate)]
        return torch.autograd.grad(fn(*x), x)

    for a, b in zip(grads(f), grads(torch.compile(f, backend="aot_eager", fullgraph=True))):
        assert torch.equal(a, b)

    def steps(q, k, v, state):
        o = linear_attn_step_with_pope(q, k, v, case.ld, (case.freqs[:1], case.bias), state)
        return o + linear_attn_step_with_pope(q, k, v, case.ld, (case.freqs[1:2], case.bias), state)

    args = [t[:, :, :1].contiguous() for t in (case.q, case.k, case.v)]
    a, b = case.s0.clone(), case.s0.clone()
    with torch.no_grad():
        o, p = steps(*args, a), torch.compile(steps, backend="aot_eager", fullgraph=True)(*args, b)
    assert torch.equal(o, p) and torch.equal(a, b)


def test_ops(cuda):
    case = Case(cuda, B=2, N=70, initial=True)
    checks = ("test_schema", "test_autograd_registration", "test_faketensor")
    req = lambda t: t.detach().clone().requires_grad_()
    torch.library.opcheck(torch.ops.pope_amd.linear_fwd, (req(case.q), req(case.k), req(case.v), req(case.freqs), req(case.bias), case.ld, None, None, req(case.s0), 0.1, True, False),
                          test_utils=checks[:2])
    one = [t[:, :, :1].contiguous() for t in (case.q, case.k, case.v)]
    torch.library.opcheck(torch.ops.pope_amd.linear_step, (*one, case.freqs[:1], case.bias, case.ld, case.s0.clone(), None, None, None, None, 1e-5, 0.1), test_utils=checks)
    torch.library.opcheck(torch.ops.pope_amd.gated_norm_fwd, (req(case.do), req(case.do), None, 1e-5, True), test_utils=checks)


def test_autocast_parameters(cuda):
    """bf16 rows with fp32 angles, bias and norm weight, as under autocast."""
    pope = pope_amd.PoPE(64, heads=2).to(cuda)
    q, k, v = (torch.randn(2, 2, 80, 64, device=cuda, requires_grad=True) for _ in range(3))
    w = torch.ones(64, device=cuda, requires_grad=True)
    with torch.autocast("cuda", dtype=BF16):
        emb = pope(80)
        y = linear_attn_with_pope(q.to(BF16), k.to(BF16), v.to(BF16), None, emb, gate=torch.ones(2, 2, 80, 64, device=cuda, dtype=BF16), norm_weight=w)
    y.float().square().sum().backward()
    assert all(t.grad is not None and t.grad.isfinite().all() for t in (q, k, v, w, *pope.parameters()))

"""The linear attention, its step and the gated norm in 64 bits, and how far from them the calls may be.

A product of two operands held as sums of bf16 parts is off by what each holds less than its value (one part: half a step, 2^-8; two:
2^-16 relative, and 2^-16 for the product of the second parts, which is left out).  An output is a sum of products
x_ie y_je z_j, of which at most x, y, z, the weighted x . y and the state are rounded, three of them on any path where z is
held exactly (16-bit values) and four otherwise, so with A the same sum over absolute values it is off by at most
  one part    (3 2^-8 + second orders) A: 4 2^-8 A
  two parts   (4 2^-16 + 2 2^-16 for left-out products) A: 6 2^-16 A
  states      two parts, one product: 3 2^-16 A
and for all of them 2e-5 A more: fp32 sums of up to 256 + 64 terms and n / 32 updates of a state (2^-24 each), powers of g
(|p log g| 2^-24, and g^p is 0 where that passes 2e-5), the sine, cosine, exp and log of the hardware (1e-6 together).  Then the
output's own rounding.  Gradients are the same sums with other operands; those of rows are turned from expanded columns to q and k by
(cos, sin) sigmoid(x), exact to 1e-6.  A itself comes from the same formulas, on absolute values; the 1e-6 of a sine or cosine is absolute,
whatever its value, so A is taken with |cos| + 0.05: 2e-5 of that is 1e-6.
"""
import math

import torch
import torch.nn.functional as F

F64 = torch.float64


def angles(pos, R):
    return pos[..., None].float() * 10000 ** -(torch.arange(R, device=pos.device).float() / max(R, 1))


def half(t):
    return torch.finfo(t).eps / 2


def expand64(x, freqs, bias, R):
    """Interleaved pairs, then the other columns, in 64 bits; differentiable."""
    x = x.double()
    if not R:
        return x
    th = (freqs if freqs.ndim == 2 else freqs.unsqueeze(1)).double()
    if bias is not None:
        th = th + bias.double()[:, None, :]
    m = F.softplus(x[..., :R])
    return torch.cat((torch.stack((m * th.cos(), m * th.sin()), -1).flatten(-2), x[..., R:]), -1)


def attend64(qh, kh, v, ld, scale, mask, s0, seqs):
    """o and the final states of expanded rows in 64 bits: qh (B, Hq, N, E).  seqs: (batch entry, first row, last + 1)."""
    Hk = kh.shape[1]
    G = qh.shape[1] // Hk
    if mask is not None:
        kh, v = (t.masked_fill(~mask[:, None, :, None], 0.0) for t in (kh, v))
    power = lambda p: torch.where(p == 0, 1.0, (ld.double().view(-1, *([1] * p.ndim)) * p.clamp_min(1)).exp())
    o, last = qh.new_zeros((*qh.shape[:3], v.shape[3])), []
    for s, (b, lo, hi) in enumerate(seqs):
        S, n = s0[s], hi - lo
        if n:
            i = torch.arange(n, device=qh.device)
            d = i[:, None] - i
            q, k, x = qh[b, :, lo:hi].unflatten(0, (G, Hk)), kh[b, :, lo:hi], v[b, :, lo:hi]
            w = (q @ k.transpose(1, 2)) * power(d.clamp_min(0)).masked_fill(d < 0, 0.0)
            out = (w @ x + (q @ S) * power(i + 1)[..., None]) * scale
            o = torch.cat((o[:b], torch.cat((o[b, :, :lo], out.flatten(0, 1), o[b, :, hi:]), 1)[None], o[b + 1:]))
            S = S * power(torch.tensor(n, device=qh.device)).view(-1, 1, 1) + (k * power(n - 1 - i)[..., None]).transpose(1, 2) @ x
        last.append(S)
    return o, torch.stack(last)


class Case:
    """Inputs of a call, head-first; `args()` what the call is given."""

    def __init__(self, device, *, B=1, Hq=2, Hk=2, N=65, D=64, R=32, Dv=64, dtype=torch.bfloat16, mask=None, initial=False, lens=None, lead=0, tail=0,
                 past=0, bias_heads=None, batch_freqs=False, decay="memory", seed=0):
        g = torch.Generator().manual_seed(seed)
        rand = lambda *s: torch.randn(*s, generator=g)
        self.dtype, self.R, self.lens = dtype, R, lens
        self.cu = None
        if lens is not None:
            B, N = 1, lead + sum(lens) + tail
            cu = [lead]
            for n in lens:
                cu.append(cu[-1] + n)
            self.cu = torch.tensor(cu, dtype=torch.int32, device=device)
            self.seqs = [(0, cu[b], cu[b + 1]) for b in range(len(lens))]
        else:
            self.seqs = [(b, 0, N) for b in range(B)]
        self.q, self.k, self.v = (rand(B, h, N, d).to(device, dtype) for h, d in ((Hq, D), (Hk, D), (Hk, Dv)))
        pos = torch.arange(N) + past
        if batch_freqs:
            pos = pos + 3 * torch.arange(B)[:, None]
        self.freqs = angles(pos, R).to(device) if R else None
        self.bias = (-2 * math.pi * torch.rand(bias_heads or Hk, R, generator=g)).to(device) if R else None
        if decay == "memory":
            self.ld = torch.log1p(-1 / torch.logspace(1, 2.5, Hk)).to(device)
        else:
            self.ld = decay if decay is None else torch.tensor(decay, device=device)
        self.mask = None
        if mask == "random":
            self.mask = torch.rand(B, N, generator=g).lt(0.7).to(device)
        elif mask == "empty":     # nothing is left of the first sequence
            self.mask = torch.rand(B, N, generator=g).lt(0.7).to(device)
            self.mask[0] = False
        self.s0 = rand(len(self.seqs), Hk, D + R, Dv).to(device) if initial else None
        self.zero = torch.zeros(len(self.seqs), Hk, D + R, Dv, dtype=F64, device=device)
        self.scale = D ** -0.5
        self.do, self.ds = rand(B, Hq, N, Dv).to(device, dtype), rand(len(self.seqs), Hk, D + R, Dv).to(device)

    def emb(self):
        return (self.freqs, self.bias) if self.R else None

    def kw(self):
        return dict(mask=self.mask, initial_state=self.s0, cu_seqlens=self.cu)

    def leaves(self):
        return {n: getattr(self, n) for n in ("q", "k", "v", "freqs", "bias", "s0") if getattr(self, n) is not None}

    def decay64(self):
        return torch.zeros(self.k.shape[1], dtype=F64, device=self.q.device) if self.ld is None else self.ld.double()

    def exact(self, grads=True):
        """{name: value}, {name: A} in 64 bits; with the gradients of sum(o do) + sum(states ds)."""
        x = {n: t.double().requires_grad_(grads) for n, t in self.leaves().items()}
        qh, kh = expand64(x["q"], x.get("freqs"), None, self.R), expand64(x["k"], x.get("freqs"), x.get("bias"), self.R)
        s0 = x.get("s0", self.zero)
        o, last = attend64(qh, kh, x["v"], self.decay64(), self.scale, self.mask, s0, self.seqs)
        if grads:   # nothing may reach an output where no sequence has rows
            o = o + 0.0 * (qh.sum() + kh.sum() + x["v"].sum())
        near = lambda h, r: h.detach().abs() + F.pad((0.05 * F.softplus(r.detach()[..., :self.R])).repeat_interleave(2, -1), (0, r.shape[-1] - self.R))
        a = {"qh": near(qh, x["q"]), "kh": near(kh, x["k"]), "v": x["v"].detach().abs(), "s0": s0.detach().abs()}
        a = {n: t.requires_grad_(grads) for n, t in a.items()}
        ao, alast = attend64(a["qh"], a["kh"], a["v"], self.decay64(), self.scale, self.mask, a["s0"], self.seqs)
        if grads:
            ao = ao + 0.0 * (a["qh"].sum() + a["kh"].sum() + a["v"].sum())
        val, tol = {"o": o.detach(), "states": last.detach()}, {"o": ao.detach(), "states": alast.detach()}
        if not grads:
            return val, tol
        g = torch.autograd.grad([o, last], list(x.values()), [self.do.double(), self.ds.double()])
        val.update({"d_" + n: t for n, t in zip(x, g)})
        ga = dict(zip(a, torch.autograd.grad([ao, alast], list(a.values()), [self.do.double().abs(), self.ds.double().abs()])))
        tol["d_v"] = ga["v"]
        if self.s0 is not None:
            tol["d_s0"] = ga["s0"]
        phase = {}
        for n, h in (("q", "qh"), ("k", "kh")):
            R, raw = self.R, x[n].detach()
            gh = ga[h]
            if not R:
                tol["d_" + n] = gh
                continue
            th = (self.freqs if self.freqs.ndim == 2 else self.freqs.unsqueeze(1)).double()
            if n == "k":
                th = th + self.bias.double()[:, None, :]
            c, s = th.cos().abs() + 0.05, th.sin().abs() + 0.05
            gc, gs = gh[..., 0:2 * R:2], gh[..., 1:2 * R:2]
            tol["d_" + n] = torch.cat(((gc * c + gs * s) * torch.sigmoid(raw[..., :R]), gh[..., 2 * R:]), -1)
            phase[n] = (gc * s + gs * c) * F.softplus(raw[..., :R])
        if self.R:
            t = phase["k"].sum((0, 2))
            tol["d_bias"] = t if self.bias.shape[0] > 1 else t.sum(0, keepdim=True)
            t = phase["q"].sum(1) + phase["k"].sum(1)
            tol["d_freqs"] = t if self.freqs.ndim == 3 else t.sum(0)
        return val, tol

    def bound(self, name, value, tol):
        parts16 = self.dtype == torch.bfloat16
        rel = 3 * 2.0 ** -16 if name in ("states", "d_s0") else 4 * 2.0 ** -8 if parts16 else 6 * 2.0 ** -16
        own = half(self.dtype) if name in ("o", "d_q", "d_k", "d_v") else 2.0 ** -24
        return (rel + 2e-5) * tol * (1 + own) + own * value.abs() + (2.0 ** -25 if self.dtype == torch.float16 else 1e-30)


def check(got, want, bound, what):
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)}, want {tuple(want.shape)}"
    err = (got.double() - want).abs()
    over = ~(err <= bound)
    if over.any():
        at = tuple(over.nonzero()[0].tolist())
        raise AssertionError(f"{what}: {int(over.sum())} of {over.numel()} off, first {at}: {got[at].item()} for {want[at].item()}, bound {bound[at].item():.3g}; "
                             f"worst {(err / bound).max().item():.3g} bounds")


def run(pope_amd, case, *, grads=True, head_first=True, leaves=None, **kw):
    """The call and its gradients as {name: tensor}, head-first."""
    turn = (lambda t: t) if head_first else (lambda t: t.transpose(1, 2))
    x = {n: (leaves or {}).get(n, t).detach().requires_grad_(grads) for n, t in case.leaves().items()}
    args = dict(case.kw(), **kw)
    if "s0" in x:
        args["initial_state"] = x["s0"]
    o, last = pope_amd.linear_attn_with_pope(turn(x["q"]), turn(x["k"]), turn(x["v"]), case.ld, (x["freqs"], x["bias"]) if case.R else None,
                                             return_state=True, head_dimension_at_first=head_first, **args)
    out = {"o": turn(o).detach(), "states": last.detach()}
    if grads:
        g = torch.autograd.grad([turn(o), last], list(x.values()), [case.do.to(o.dtype), case.ds])
        out.update({"d_" + n: t for n, t in zip(x, g)})
    return out


def compare(got, case, grads=True):
    val, tol = case.exact(grads)
    for n in val:
        check(got[n], val[n], case.bound(n, val[n], tol[n]), n)


def norm64(x, gate, weight, eps, head_first=True):
    x, gate = x.double(), gate.double()
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    if weight is not None:
        w = weight.double()
        y = y * (w[:, None, :] if w.ndim == 2 and head_first else w)
    return y * F.silu(gate)

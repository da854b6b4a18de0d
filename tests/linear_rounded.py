"""What roundings of operands alone do to the linear attention: its outputs and gradients in 64 bits, from operands held as one bf16 part or as
the sum of two (their second parts' product left out), as the kernels hold them.

Held so are q_hat (times the scale), k_hat, v and dO, the weighted x . y of rows, the initial states and the final states' gradient; each kernel
holds at most one operand more on any path (a state between chunks, and z weighted on its way into it, in place of the weighted x . y).
Each such rounding is as likely up as down and as large as any other, so the errors' 2-norms add up as squares: with five roundings
on a path where this has four an error is sqrt(5 / 4) of this one's, at most sqrt(2) where those that differ are the larger ones.
Twice this one's error is asked for; three times for the bias's gradient, a few tens of sums, whose own norms scatter.
"""
import torch
import torch.nn.functional as F

from linear_common import expand64, half


def parts(x, n):
    """x as (first part, second part); n 0: exact."""
    if n == 0:
        return x, torch.zeros_like(x)
    a = x.float().bfloat16().double()
    return a, (x - a).float().bfloat16().double() if n == 2 else torch.zeros_like(x)


def product(x, y):
    return (x[0] + x[1]) @ (y[0] + y[1]) - x[1] @ y[1]


def t(x):
    return x[0].mT, x[1].mT


def outputs(case, n, *, own=True):
    """{name: value} of a padded case with operands of n parts; own: with the outputs' rounding to the rows' type."""
    B, Hq, N, D = case.q.shape
    Hk, R = case.k.shape[1], case.R
    G = Hq // Hk
    S0 = (case.s0 if case.s0 is not None else case.zero).double()[:, None]
    dS, dO = case.ds.double()[:, None], case.do.double().unflatten(1, (G, Hk))
    qh = expand64(case.q, case.freqs, None, R).unflatten(1, (G, Hk)) * case.scale
    kh, v = expand64(case.k, case.freqs, case.bias, R), case.v.double()
    if case.mask is not None:
        kh, v = (x.masked_fill(~case.mask[:, None, :, None], 0.0) for x in (kh, v))
    i = torch.arange(N, device=qh.device)
    ld = case.decay64().view(-1, 1)
    power = lambda p: torch.where(p == 0, 1.0, (ld.view(-1, *([1] * p.ndim)) * p.clamp_min(1)).exp())
    D_ = power((i[:, None] - i).clamp_min(0)).masked_fill(i[:, None] < i, 0.0)
    first, later = power(i + 1)[..., None], power(N - 1 - i)[..., None]
    q, k, x, g, s, ds = (parts(y, n) for y in (qh, kh[:, None], v[:, None], dO, S0, dS))
    a, b = parts(product(q, t(k)) * D_, n), parts(product(g, t(x)) * D_, n)
    o = product(a, x) + product(q, s) * first
    dqh = (product(b, k) + product(g, t(s)) * first) * case.scale
    dkh = (product(t(b), q) + (product(x, t(ds)) * later) / G).sum(1)
    dv = (product(t(a), g) + (product(k, ds) * later) / G).sum(1)
    if case.mask is not None:
        dkh, dv = (y.masked_fill(~case.mask[:, None, :, None], 0.0) for y in (dkh, dv))
    out = {"o": o.flatten(1, 2), "d_v": dv}
    phase = {}
    for name, raw, d, bias in (("q", case.q, dqh.flatten(1, 2), None), ("k", case.k, dkh, case.bias)):
        if not R:
            out["d_" + name] = d
            continue
        th = (case.freqs if case.freqs.ndim == 2 else case.freqs.unsqueeze(1)).double()
        th = th if bias is None else th + bias.double()[:, None, :]
        y, dc, dsn = raw.double()[..., :R], d[..., 0:2 * R:2], d[..., 1:2 * R:2]
        out["d_" + name] = torch.cat(((dc * th.cos() + dsn * th.sin()) * torch.sigmoid(y), d[..., 2 * R:]), -1)
        phase[name] = F.softplus(y) * (dsn * th.cos() - dc * th.sin())
    if own:
        out = {m: y.to(case.dtype).double() for m, y in out.items()}
    if R:
        y = phase["k"].sum((0, 2))
        out["d_bias"] = y if case.bias.shape[0] > 1 else y.sum(0, keepdim=True)
        y = phase["q"].sum(1) + phase["k"].sum(1)
        out["d_freqs"] = y if case.freqs.ndim == 3 else y.sum(0)
    return out


def check_norms(got, case, n, val, tol):
    """Errors' 2-norms against those of operands of n parts.  fp32 sums, sines and exponentials: 2e-6 of absolute values, in the
    2-norm (2^-24 of each of some hundred terms, as likely up as down, and 1e-6)."""
    model = outputs(case, n)
    for m, y in model.items():
        exact = val[m]
        err, lim = (got[m].double() - exact).norm(), (3 if m == "d_bias" else 2) * (y - exact).norm() + 2e-6 * tol[m].norm()
        if m == "d_bias" and got[m].dtype != torch.float32:
            lim = lim + half(got[m].dtype) * exact.norm()
        assert err <= lim, f"{m}: off by {(err / exact.norm()).item():.2e} of its norm, allowed {(lim / exact.norm()).item():.2e}"

"""The paged key / value cache of PoPE rows and the attention over it, as measurable cases.

Kinds, one operator each (attention in its two forms):

  write    ``paged_cache_write`` of new tokens, then ``paged_cache_read`` of the rows they got: what the cache holds for
           them (a program that scores a prompt on the values its cache will answer from does both)
  read     ``paged_cache_read`` of contexts: handing sequences on as plain rows
  chunk    ``paged_flash_attn_with_pope``, several new tokens per sequence against all that is cached
  decode   the same for one new token per sequence

New tokens come as a padded batch (batch, heads, n, dim), or packed: a batch of one whose rows belong to the sequences
that ``cu_seqlens`` delimits.  Row i of the n new ones of a sequence of length L (the new ones included) stands at
position L - n + i.  A cached key row is [softplus(k) cos, softplus(k) sin] of the angle freqs + bias for the rotated
dims and k itself for the others; it is rounded once, to the 16-bit type, or (``q8``) to e4m3 times the smallest power
of two that brings the row's largest magnitude to at most 448, and so is the value row.  Query head h reads key head
h % Hk.  Inputs are N(0, 1), biases uniform in [-2 pi, 0], pages in random order.
"""
from __future__ import annotations

import math
import os
import random
import sys

import torch
import torch.nn.functional as F

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
_DEFAULTS = dict(kind="decode", B=1, Hq=8, Hk=8, N=1, past=0, least=0, D=64, R=32, dtype="bf16", q8=False, packed=False,
                 causal=True, page=64, head_first=True)


def _case(name=None, **kw):
    """N: new tokens per sequence (packed: on average); past: cached before them, drawn from [least, past]."""
    c = dict(_DEFAULTS, **kw)
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one generated token for each of 16 sequences enters the cache: launches and host time count
        _case("write_step", kind="write", B=16, N=1, past=4096, least=100),
        # four prompts of 2048 tokens on average, ragged, into an 8-bit cache with 128-wide heads
        _case("write_prompt_8bit", kind="write", B=4, N=2048, past=0, D=128, R=64, q8=True, packed=True),
        # a prompt of 256-wide heads, fully rotated, in fp16 and (batch, seq, heads, dim)
        _case("write_wide", kind="write", B=1, N=2047, past=1000, D=256, R=256, dtype="fp16", head_first=False),
        # long contexts leave the cache: eight of 8192 tokens on average
        _case("read_long", kind="read", B=8, Hk=16, Hq=16, N=8192, D=64, R=64, packed=True),
        # the last 500 rows of 8 short contexts of an 8-bit cache, a head dim that is no multiple of 16
        _case("read_8bit", kind="read", B=8, N=500, past=777, least=0, D=72, R=40, q8=True, page=32),
        # a block of a prompt against what is cached already
        _case("chunk_cache", kind="chunk", B=1, N=130, past=15870, least=13870, D=64, R=64),
        # whole prompts of 4096 tokens, nothing cached before them
        _case("chunk_prompt", kind="chunk", B=2, N=4096, past=0, D=64, R=32),
        # ragged pieces of four prompts, grouped heads, 8-bit cache
        _case("chunk_gqa_8bit", kind="chunk", B=4, Hq=16, Hk=4, N=300, past=8000, least=500, D=128, R=64, q8=True, packed=True),
        # five proposed tokens of each of 16 sequences checked at once, grouped heads, fp16
        _case("chunk_verify", kind="chunk", B=16, Hq=32, Hk=8, N=5, past=4096, least=500, D=128, R=64, dtype="fp16", page=128),
        # generation for eight sequences of 4096 to 32768 cached tokens
        _case("decode_batch", kind="decode", B=8, Hq=16, Hk=16, past=32767, least=4095, D=64, R=64),
        # generation for one sequence, grouped heads
        _case("decode_single", kind="decode", B=1, Hq=32, Hk=8, past=4000, least=3001, D=128, R=64),
        # generation for 32 sequences on an 8-bit cache, grouped heads, packed
        _case("decode_8bit", kind="decode", B=32, Hq=32, Hk=8, past=16383, least=1000, D=128, R=64, q8=True, packed=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    kind = rng.choice(["write", "read", "chunk", "chunk", "decode", "decode"])
    D = rng.choice([32, 48, 64, 64, 64, 72, 80, 96, 100, 112, 128, 128, 128, 160, 192, 256])
    Hk = rng.choice([1, 2, 4, 8, 8, 16])
    G = rng.choice([g for g in (1, 1, 2, 3, 4, 4, 8) if g * Hk <= 32])
    R = rng.choice([D, D, D // 2, D // 2, D // 4, rng.randint(1, D), 0])
    N = 1 if kind == "decode" else _log_int(rng, 1, 8192) if kind in ("write", "read") else _log_int(rng, 2, 2048)
    past = _log_int(rng, 1, 32768) if kind != "read" else rng.choice([0, _log_int(rng, 1, 4096)])
    return _case(kind=kind, B=rng.choice([1, 1, 2, 3, 4, 8, 16, 32]), Hq=Hk * G, Hk=Hk, N=N, past=past,
                 least=rng.choice([past, past // 8, 0]), D=D, R=R, dtype=rng.choice(["bf16", "bf16", "fp16"]),
                 q8=rng.random() < 0.35, packed=rng.random() < 0.5, causal=rng.random() < 0.8,
                 page=rng.choice([32, 64, 64, 128, 256]), head_first=rng.random() < 0.7)


def draw(rng):
    while True:
        c = _draw(rng)
        w = work(c)
        n = c["N"] * (1 + math.log(c["B"])) if c["packed"] and c["kind"] != "decode" else c["N"]   # the longest, about
        held = c["B"] * (c["past"] + c["N"]) * c["Hk"] * (2 * c["D"] + c["R"])
        scores = c["B"] * c["Hq"] * n * (n + c["past"]) if c["kind"] == "chunk" else 0
        if w["bytes"] <= 6e8 and w["flops"] <= 5e10 and held <= 6e8 and scores <= 2.7e8:
            return c


def work(case):
    c = case
    B, Hq, Hk, N, D, R = (c[n] for n in ("B", "Hq", "Hk", "N", "D", "R"))
    row = (2 * D + R) * (1 if c["q8"] else 2) + (2 if c["q8"] else 0)   # a cached key and value row of one head
    mean = (c["past"] + c["least"]) / 2
    if c["kind"] == "write":
        # k, v and the angles read, rows written; read again, and the answer written
        return {"bytes": B * N * (Hk * (4 * D + 2 * row + 2 * (2 * D + R)) + 4 * R), "flops": B * N * Hk * (20 * R + 2 * D)}
    if c["kind"] == "read":
        return {"bytes": B * N * Hk * (row + 2 * (2 * D + R)), "flops": B * N * Hk * (2 * D + R)}
    pairs = B * Hq * N * (mean + (N + 1) / 2 if c["causal"] else mean + N)
    return {"bytes": B * (mean + N) * Hk * row + B * N * (4 * Hq * D + 4 * R), "flops": 2 * (2 * D + R) * pairs}


# ---------------------------------------------------------------- inputs

def _lengths(c, seed):
    """New tokens and total length of each sequence, as lists."""
    rng = random.Random(seed)
    B, N = c["B"], c["N"]
    new = [N] * B
    if c["packed"] and c["kind"] != "decode":
        cuts = sorted(rng.randint(0, B * N) for _ in range(B - 1))
        new = [b - a for a, b in zip([0] + cuts, cuts + [B * N])]
    return new, [n + rng.randint(c["least"], c["past"]) for n in new]


def _inv_freqs(R):
    return 10000 ** -(torch.arange(R, device="cuda").float() / R)


def _rows(c, g, H, N):
    """N(0, 1) rows of the new tokens in the case's layout."""
    B, N = (1, c["B"] * N) if c["packed"] else (c["B"], N)
    shape = (B, H, N, c["D"]) if c["head_first"] else (B, N, H, c["D"])
    return torch.randn(shape, generator=g, device="cuda").to(_DTYPES[c["dtype"]])


def _inputs(c, seed):
    """All that a case is made from; nothing here depends on how the cache holds it."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    new, total = _lengths(c, seed)
    B, D, R, PS = c["B"], c["D"], c["R"], c["page"]
    s = {"case": c, "most_new": max(new)}
    i32 = dict(dtype=torch.int32, device="cuda")
    s["lengths"] = torch.tensor(total, **i32)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    s["cu"] = torch.tensor(cu, **i32) if c["packed"] else None
    # pages of the sequences in random order, a few to spare
    need = [-(-t // PS) for t in total]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(B, max(1, max(need)), **i32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    s["table"], s["pages"] = table, pages
    s["bias"] = torch.rand(c["Hk"], R, generator=g, device="cuda") * (-2 * math.pi)
    # positions of the new rows
    nw, tt = torch.tensor(new, device="cuda"), torch.tensor(total, device="cuda")
    if c["packed"]:
        owner = torch.repeat_interleave(torch.arange(B, device="cuda"), nw)
        i = torch.arange(cu[-1], device="cuda") - (torch.cumsum(nw, 0) - nw)[owner]
        pos = (tt - nw)[owner] + i
        s["owner"], s["nth"] = owner, i
    else:
        pos = (tt - nw)[:, None] + torch.arange(c["N"], device="cuda")
    s["pos"] = pos
    s["freqs"] = pos[..., None].float() * _inv_freqs(R)
    if c["kind"] == "write":
        s["k"], s["v"] = _rows(c, g, c["Hk"], c["N"]), _rows(c, g, c["Hk"], c["N"])
        return s
    if c["kind"] != "read":
        s["q"] = _rows(c, g, c["Hq"], c["N"])
    # the whole contexts, packed and head-first, for filling the cache
    T = sum(total)
    s["ctx_cu"] = torch.tensor([0] + torch.tensor(total).cumsum(0).tolist(), **i32)
    s["ctx_owner"] = torch.repeat_interleave(torch.arange(B, device="cuda"), tt)
    s["ctx_pos"] = torch.arange(T, device="cuda") - (torch.cumsum(tt, 0) - tt)[s["ctx_owner"]]
    s["ctx_freqs"] = s["ctx_pos"][:, None].float() * _inv_freqs(R)
    ctx = lambda: torch.randn((1, c["Hk"], T, D), generator=g, device="cuda").to(_DTYPES[c["dtype"]])
    s["ctx_k"], s["ctx_v"] = ctx(), ctx()
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    c = case
    if own:
        sys.path.insert(0, os.path.abspath("pope-pytorch_amd"))
        import pope_amd
        s["pope_amd"] = pope_amd
        s["cache"] = pope_amd.PagedPoPECache(s["pages"], heads=c["Hk"], dim=c["D"], rotate_dim=c["R"], page_size=c["page"],
                                             dtype=_DTYPES[c["dtype"]], quantized=c["q8"], device="cuda")
        if c["kind"] != "write":
            pope_amd.paged_cache_write(s["cache"], s["ctx_k"], s["ctx_v"], (s["ctx_freqs"], s["bias"]) if c["R"] else None,
                                       s["table"], s["lengths"], cu_seqlens=s["ctx_cu"])
    else:
        s["pool"] = _pool(c, s["pages"])
        if c["kind"] != "write":
            _store(s["pool"], c, s["table"][s["ctx_owner"], s["ctx_pos"] // c["page"]].long(), s["ctx_pos"] % c["page"],
                   s["ctx_k"][0].transpose(0, 1), s["ctx_v"][0].transpose(0, 1), s["ctx_freqs"], s["bias"])
    for n in ("ctx_k", "ctx_v", "ctx_freqs"):
        s.pop(n, None)
    return s


def run(state):
    s, c = state, state["case"]
    if own:
        P, hf = s["pope_amd"], c["head_first"]
        emb = (s["freqs"], s["bias"]) if c["R"] else None
        if c["kind"] == "write":
            P.paged_cache_write(s["cache"], s["k"], s["v"], emb, s["table"], s["lengths"], cu_seqlens=s["cu"], head_dimension_at_first=hf)
        if c["kind"] in ("write", "read"):
            n = c["B"] * c["N"] if c["packed"] else c["N"]
            k_hat, v = P.paged_cache_read(s["cache"], s["table"], s["lengths"], n, cu_seqlens=s["cu"], head_dimension_at_first=hf)
            return {"k_hat": k_hat, "v": v}
        return {"o": P.paged_flash_attn_with_pope(s["q"], s["cache"], emb, s["table"], s["lengths"], cu_seqlens=s["cu"],
                                                  causal=c["causal"], head_dimension_at_first=hf)}
    if c["kind"] == "write":
        return _plain_write(s, c)
    if c["kind"] == "read":
        return _plain_read(s, c)
    return _plain_attend(s, c)


# ---------------------------------------------------------------- plain forms

def _pool(c, pages):
    """Pages of (slot, head, column) rows; 8 bits as the codes' bytes with a scale per row."""
    dt = torch.uint8 if c["q8"] else _DTYPES[c["dtype"]]
    shape = (pages, c["page"], c["Hk"])
    pool = {"k": torch.zeros(shape + (c["D"] + c["R"],), dtype=dt, device="cuda"),
            "v": torch.zeros(shape + (c["D"],), dtype=dt, device="cuda")}
    if c["q8"]:
        pool["k_scale"], pool["v_scale"] = torch.ones(shape, device="cuda"), torch.ones(shape, device="cuda")
    return pool


def _expand(x, angle, R):
    """[softplus cos, softplus sin] pairs of the first R columns, then the others; angles in 64 bits, the rest in 32."""
    m = F.softplus(x[..., :R].float())
    pairs = torch.stack((m * angle.cos().float(), m * angle.sin().float()), -1).flatten(-2)
    return torch.cat((pairs, x[..., R:].float()), -1)


def _to_8bit(x):
    """e4m3 codes and the power of two they stand in: the smallest with |x| <= 448 of it."""
    amax = x.abs().amax(-1)
    mant, e = torch.frexp(amax)                 # amax = mant 2^e, mant in [1/2, 1)
    e = torch.where(mant <= 0.875, e - 9, e - 8).clamp(-126, 126)
    scale = ((e.int() + 127) << 23).view(torch.float32)   # 2^e, by its bits: a power function may be an ulp off
    return (x / scale[..., None]).to(torch.float8_e4m3fn).view(torch.uint8), scale


def _store(pool, c, page, off, k, v, freqs, bias):
    """Rows (tokens, heads, D) into their slots."""
    kh = _expand(k, freqs.double()[:, None, :] + bias.double(), c["R"])
    if c["q8"]:
        pool["k"][page, off], pool["k_scale"][page, off] = _to_8bit(kh)
        pool["v"][page, off], pool["v_scale"][page, off] = _to_8bit(v.float())
    else:
        pool["k"][page, off] = kh.to(pool["k"].dtype)
        pool["v"][page, off] = v


def _load(pool, c, index):
    """Rows at `index` in 32 bits."""
    if not c["q8"]:
        return pool["k"][index].float(), pool["v"][index].float()
    value = lambda n: pool[n][index].view(torch.float8_e4m3fn).float() * pool[n + "_scale"][index][..., None]
    return value("k"), value("v")


def _slots(s, c):
    """Page and offset of each new row, (tokens) or (B, N)."""
    pos = s["pos"]
    b = s["owner"] if c["packed"] else torch.arange(c["B"], device="cuda")[:, None]
    return s["table"][b, pos // c["page"]].long(), pos % c["page"]


def _plain_read(s, c):
    k, v = (t.to(_DTYPES[c["dtype"]]) for t in _load(s["pool"], c, _slots(s, c)))   # (.., heads, columns)
    if c["packed"]:
        k, v = k[None], v[None]
    if c["head_first"]:
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    return {"k_hat": k, "v": v}


def _plain_write(s, c):
    k, v = (t.transpose(1, 2) if c["head_first"] else t for t in (s["k"], s["v"]))
    page, off = _slots(s, c)
    _store(s["pool"], c, page.reshape(-1), off.reshape(-1), k.flatten(0, 1), v.flatten(0, 1), s["freqs"].reshape(page.numel(), c["R"]), s["bias"])
    return _plain_read(s, c)


def _plain_attend(s, c):
    B, Hq, Hk, D, R = (c[n] for n in ("B", "Hq", "Hk", "D", "R"))
    G = Hq // Hk
    q = s["q"].transpose(1, 2) if c["head_first"] else s["q"]              # (.., rows, heads, D)
    qh = _expand(q, s["freqs"].double().unsqueeze(-2), R)
    n = s["most_new"]
    if c["packed"]:   # one padded row block per sequence
        padded = torch.zeros((B, n, Hq, D + R), device="cuda")
        padded[s["owner"], s["nth"]] = qh[0]
        qh = padded
        first = s["lengths"] - (s["cu"][1:] - s["cu"][:-1])
    else:
        first = s["lengths"] - n
    k, v = _load(s["pool"], c, s["table"].long())                         # (B, pages, slots, heads, columns)
    k, v = (t.flatten(1, 2).transpose(1, 2) for t in (k, v))              # (B, Hk, L, columns)
    qh = qh.view(B, n, G, Hk, D + R).permute(0, 3, 2, 1, 4).reshape(B, Hk, G * n, D + R)
    sc = torch.matmul(qh, k.transpose(2, 3).contiguous()) * D ** -0.5
    del k
    j = torch.arange(sc.shape[-1], device="cuda")
    keep = j < s["lengths"][:, None, None]
    if c["causal"]:
        keep = keep & (j <= (first[:, None] + torch.arange(n, device="cuda"))[..., None])
    sc = sc.view(B, Hk, G, n, -1).masked_fill_(~keep[:, None, None], float("-inf"))
    sc = sc - sc.amax(-1, keepdim=True).clamp_min(-1e30)
    p = sc.exp_()
    norm = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, Hk, G * n, -1), v).view(B, Hk, G, n, D) / norm.clamp_min(1e-30)
    o = o.permute(0, 3, 2, 1, 4).reshape(B, n, Hq, D)                     # head g Hk + hk
    if c["packed"]:
        o = o[s["owner"], s["nth"]][None]
    o = o.to(_DTYPES[c["dtype"]])
    return {"o": o.transpose(1, 2) if c["head_first"] else o}


# ---------------------------------------------------------------- the definition in 64 bits

def _exact_rows(c, k, v, freqs, bias):
    """What the cache holds for key and value rows (heads, tokens, D), in 64 bits: a row at a head."""
    R, dt = c["R"], _DTYPES[c["dtype"]]
    x, w = k.double(), v.double()
    th = freqs.double() + bias.double()[:, None, :]
    m = torch.log1p(torch.exp(-x[..., :R].abs())) + x[..., :R].clamp_min(0)
    kh = torch.empty(x.shape[:-1] + (x.shape[-1] + R,), dtype=torch.float64, device=x.device)
    kh[..., 0:2 * R:2], kh[..., 1:2 * R:2], kh[..., 2 * R:] = m * th.cos(), m * th.sin(), x[..., R:]
    if not c["q8"]:
        return kh.to(dt).double(), w

    power = lambda e: ((e.long() + 1023) << 52).view(torch.float64)             # 2^e exactly

    def eight(t):
        top = t.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -100)
        unit = power(torch.ceil(torch.log2(top / 448)))
        unit = torch.where(top > 448 * unit, unit * 2, torch.where(top <= 224 * unit, unit / 2, unit))
        y = (t / unit).abs()
        step = power(torch.floor(torch.log2(y.clamp_min(2.0 ** -6))) - 3)      # spacing of e4m3 at y
        return torch.sign(t) * torch.round(y / step) * step * unit

    return eight(kh), eight(w)


def exact(case, seed):
    c, s = case, _inputs(case, seed)
    B, Hq, Hk, D, R, hf = (c[n] for n in ("B", "Hq", "Hk", "D", "R", "head_first"))
    new, total = _lengths(c, seed)
    f64 = dict(dtype=torch.float64, device="cuda")
    if c["kind"] == "write":
        k, v = (t if hf else t.transpose(1, 2) for t in (s["k"], s["v"]))
        got = [_exact_rows(c, k[b], v[b], s["freqs"] if c["packed"] else s["freqs"][b], s["bias"]) for b in range(k.shape[0])]
        kh, vv = (torch.stack(t) for t in zip(*got))
    else:
        ends = torch.tensor(total).cumsum(0).tolist()
        H, rows, cols = (Hk, c["N"], D + R) if c["kind"] == "read" else (Hq, c["N"], D)
        shape = (1, H, B * rows) if c["packed"] else (B, H, rows)
        kh, vv = torch.zeros(shape + (cols,), **f64), torch.zeros(shape + (D,), **f64)
        at = 0
        for b in range(B):
            lo, L, n = ends[b] - total[b], total[b], new[b]
            out = (0, slice(None), slice(at, at + n)) if c["packed"] else (b,)
            at += n
            if n == 0:
                continue
            hk, hv = _exact_rows(c, s["ctx_k"][0, :, lo:lo + L], s["ctx_v"][0, :, lo:lo + L], s["ctx_freqs"][lo:lo + L], s["bias"])
            if c["kind"] == "read":
                kh[out], vv[out] = hk[:, L - n:], hv[:, L - n:]
                continue
            q = (s["q"] if hf else s["q"].transpose(1, 2))[out]               # (Hq, n, D)
            fr = s["freqs"][at - n:at] if c["packed"] else s["freqs"][b]
            x, th = q.double(), fr.double()
            m = torch.log1p(torch.exp(-x[..., :R].abs())) + x[..., :R].clamp_min(0)
            qh = torch.empty((Hq, n, D + R), **f64)
            qh[..., 0:2 * R:2], qh[..., 1:2 * R:2], qh[..., 2 * R:] = m * th.cos(), m * th.sin(), x[..., R:]
            sees = torch.arange(L, device="cuda") <= (torch.arange(n, device="cuda") + L - n)[:, None] if c["causal"] else None
            for h in range(Hq):
                sc = torch.mm(qh[h], hk[h % Hk].t().contiguous()) * D ** -0.5
                if sees is not None:
                    sc = sc.masked_fill(~sees, float("-inf"))
                kh[out][h] = torch.mm(torch.softmax(sc, -1), hv[h % Hk])
    if not hf:
        kh, vv = kh.transpose(1, 2), vv.transpose(1, 2)
    return {"k_hat": kh, "v": vv} if c["kind"] in ("write", "read") else {"o": kh}

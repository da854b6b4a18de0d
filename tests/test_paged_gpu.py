"""The paged cache's kernels against 64-bit formulas, and against the CPU cache's page bytes.

Tolerances, element by element, for attention over the rows the cache holds (they are read back):
  output's own rounding             u |o|,              u = eps / 2 of the type
  rounding of P                     u sum_j p_j |v_j|   (and 2^-25 sum_j |v_j| / l where fp16 P is subnormal, l >= 1)
  scores: Q_hat as two 16-bit parts leaves u^2 of each product (fp16's second part is subnormal below: 2^-25 |k|), fp32
  accumulation E 2^-24, the hardware sine, cosine, exp2 and log2 together 1e-6, all relative to A = scale sum_e |q_e k_e|; a score
  off by x changes p by x, numerator and denominator: 2 max_j x sum_j p_j |v_j|
  fp32 sums and rescaling           2e-5 sum_j p_j |v_j|
"""
import math

import pytest
import torch
import torch.nn.functional as F

import pope_amd
from pope_amd import PagedPoPECache, PoPE, paged_cache_read, paged_cache_write, paged_flash_attn_with_pope

pytestmark = pytest.mark.gpu

I32 = torch.int32
INF, NAN = math.inf, math.nan


def angles(pos, R):
    return pos[..., None].float() * 10000 ** -(torch.arange(R, device=pos.device).float() / max(R, 1))


def rows64(k, freqs, bias, R):
    """K_hat (interleaved pairs) in 64 bits: k (heads, n, D), freqs (n, R), bias (heads or 1, R)."""
    x, th = k.double(), freqs.double() + bias.double()[:, None, :]
    m = F.softplus(x[..., :R])
    return torch.cat((torch.stack((m * th.cos(), m * th.sin()), -1).flatten(-2), x[..., R:]), -1)


def held(x, dtype, q8):
    """Half a step of what the cache holds of 64-bit rows x, and what fp32 arithmetic before the rounding adds."""
    slack = 1e-6 * (1 + x.abs())
    if not q8:
        return x.abs() * torch.finfo(dtype).eps / 2 + 2.0 ** -25 + slack
    unit = torch.exp2(torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True).clamp_min(1e-30) / 448)))
    return torch.maximum(x.abs(), unit * 2.0 ** -6) * 2.0 ** -4 + slack


class Batch:
    """Sequences with pages in random order, their whole contexts written in one packed call."""

    def __init__(self, total, *, heads, G=1, D=64, R=32, page=64, dtype=torch.bfloat16, q8=False, seed=0, spare=2):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.g, self.total, self.heads, self.G, self.D, self.R, self.dtype, self.q8 = g, total, heads, G, D, R, dtype, q8
        need = [-(-t // page) for t in total]
        n = sum(need) + spare
        self.cache = PagedPoPECache(n, heads=heads, dim=D, rotate_dim=R, page_size=page, dtype=dtype, quantized=q8, device="cuda")
        order = torch.randperm(n, generator=g, device="cuda").to(I32)
        self.table = torch.full((len(total), max(1, max(need))), -1, dtype=I32, device="cuda")
        at = 0
        for b, m in enumerate(need):
            self.table[b, :m] = order[at:at + m]
            at += m
        self.lengths = torch.tensor(total, dtype=I32, device="cuda")
        self.bias = -torch.rand(heads, R, generator=g, device="cuda") * 2 * math.pi
        self.cu = torch.tensor([0, *torch.tensor(total).cumsum(0)], dtype=I32, device="cuda")
        T = sum(total)
        self.pos = torch.cat([torch.arange(t, device="cuda") for t in total]) if T else torch.zeros(0, dtype=torch.long, device="cuda")
        self.k, self.v = self.rand(1, heads, T, D), self.rand(1, heads, T, D)
        paged_cache_write(self.cache, self.k, self.v, self.emb(self.pos), self.table, self.lengths, cu_seqlens=self.cu)

    def rand(self, *shape):
        return torch.randn(shape, generator=self.g, device="cuda").to(self.dtype)

    def emb(self, pos):
        return (angles(pos, self.R), self.bias) if self.R else None

    def rows(self, b):
        """Held rows of sequence b, (heads, length, columns) in 64 bits."""
        k, v = paged_cache_read(self.cache, self.table[b:b + 1], self.lengths[b:b + 1], self.total[b])
        return k[0].double(), v[0].double()


def reference(q, freqs, k, v, R, scale, causal, dtype):
    """64-bit attention of q (Hq, n, D) at the last n positions over held rows, its lse, and the kernel's error bound."""
    Hq, n, L, G = q.shape[0], q.shape[1], k.shape[1], q.shape[0] // k.shape[0]
    qh = rows64(q, freqs, torch.zeros(1, R, device="cuda"), R)
    k, v = k.repeat(G, 1, 1), v.repeat(G, 1, 1)
    sc = torch.bmm(qh, k.transpose(1, 2).contiguous()) * scale
    A = torch.bmm(qh.abs(), k.abs().transpose(1, 2).contiguous()) * abs(scale)
    see = torch.arange(L, device="cuda") <= (L - n + torch.arange(n, device="cuda"))[:, None] if causal else torch.ones(n, L, dtype=torch.bool, device="cuda")
    sc, A = sc.masked_fill(~see, -INF), A.masked_fill(~see, 0.0)
    p = torch.softmax(sc, -1).nan_to_num(0.0)
    o, pv = torch.bmm(p, v), torch.bmm(p, v.abs())
    u, f16 = torch.finfo(dtype).eps / 2, dtype == torch.float16
    x = (u * u + k.shape[-1] * 2.0 ** -24 + 1e-6) * A.amax(-1, keepdim=True) if L else torch.zeros(Hq, n, 1, device="cuda")
    if f16 and L:
        x = x + 2.0 ** -25 * k.abs().sum(-1).amax(-1)[:, None, None] * abs(scale)
    tol = u * o.abs() + (u + 2 * x + 2e-5) * pv + 2.0 ** -25
    if f16:
        tol = tol + 2.0 ** -25 * v.abs().sum(1, keepdim=True)
    return o, torch.logsumexp(sc, -1), tol, x[..., 0] + 1e-5


def attend_and_check(B, new, *, packed, causal=True, scale=None, gap=0, head_first=True):
    """New rows' queries of every sequence against the reference; `gap` packed rows behind the last sequence."""
    Hq, D, R = B.heads * B.G, B.D, B.R
    scale = D ** -0.5 if scale is None else scale
    if packed:
        cu = [0, *torch.tensor(new).cumsum(0).tolist()]
        N = cu[-1] + gap
        pos = torch.zeros(N, dtype=torch.long, device="cuda")
        for b, n in enumerate(new):
            pos[cu[b]:cu[b + 1]] = torch.arange(B.total[b] - n, B.total[b], device="cuda")
        q, cu_t = B.rand(1, Hq, N, D), torch.tensor(cu, dtype=I32, device="cuda")
        part = [(0, slice(cu[b], cu[b + 1])) for b in range(len(new))]
    else:
        N = new[0]
        assert all(n == N for n in new)
        pos = B.lengths[:, None].long() - N + torch.arange(N, device="cuda")
        q, cu_t = B.rand(len(new), Hq, N, D), None
        part = [(b, slice(0, N)) for b in range(len(new))]
    emb = B.emb(pos)
    arg = q if head_first else q.transpose(1, 2)
    o, lse = paged_flash_attn_with_pope(arg, B.cache, emb, B.table, B.lengths, cu_seqlens=cu_t, causal=causal, softmax_scale=scale,
                                        return_lse=True, head_dimension_at_first=head_first)
    o = o if head_first else o.transpose(1, 2)
    assert o.shape == q.shape and o.dtype == B.dtype
    if packed and gap:
        assert not o[:, :, -gap:].any() and (lse[:, :, -gap:] == -INF).all()
    worst = 0.0
    for b, n in enumerate(new):
        if not n:
            continue
        i, s = part[b]
        k, v = B.rows(b)
        f = angles(pos[s] if packed else pos[b], R)
        want, wl, tol, ltol = reference(q[i, :, s], f, k, v, R, scale, causal, B.dtype)
        err = (o[i, :, s].double() - want).abs()
        assert not o[i, :, s].isnan().any()
        assert (err <= tol).all(), f"sequence {b}: {(err / tol).max().item():.2f} of the bound"
        worst = max(worst, (err / tol).max().item() if err.numel() else 0.0)
        got = lse[i, :, s].double()
        assert torch.equal(got == -INF, wl == -INF)
        fin = wl != -INF
        assert ((got - wl).abs()[fin] <= (ltol + 1e-6 * wl.abs())[fin]).all()
    return worst


# ---------------------------------------------------------------- write and read

SHAPES = [(16, 8), (32, 32), (1, 1), (48, 0), (64, 32), (64, 64), (80, 10), (72, 40), (96, 96), (128, 0), (128, 64), (100, 99),
          (160, 31), (192, 192), (250, 100)]


@pytest.mark.parametrize("D,R", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("q8", [False, True], ids=["16bit", "8bit"])
def test_write_and_read(cuda, D, R, dtype, q8):
    """Rows read back are the rounded exact ones; the pages are those of the CPU cache, and other slots keep their bytes."""
    total = [70, 1, 0, 131, 33]
    B = Batch(total, heads=3, D=D, R=R, dtype=dtype, q8=q8, page=32 if D < 100 else 64)
    for b, t in enumerate(total):
        k, v = B.rows(b)
        s = slice(int(B.cu[b]), int(B.cu[b + 1]))
        want = rows64(B.k[0, :, s], angles(B.pos[s], R), B.bias, R)
        assert ((k - want).abs() <= held(want, dtype, q8)).all()
        wv = B.v[0, :, s].double()
        assert ((v - wv).abs() <= held(wv, dtype, q8)).all()
        assert q8 or torch.equal(v, wv)
    C = PagedPoPECache(B.cache.num_pages, heads=3, dim=D, rotate_dim=R, page_size=B.cache.page_size, dtype=dtype, quantized=q8)
    emb = B.emb(B.pos)
    paged_cache_write(C, B.k.cpu(), B.v.cpu(), tuple(t.cpu() for t in emb) if R else None, B.table.cpu(), B.lengths.cpu(), cu_seqlens=B.cu.cpu())
    assert torch.equal(C.v_pages, B.cache.v_pages.cpu())
    gk, ck = B.cache.k_pages.cpu().float(), C.k_pages.float()
    # a key value next to a rounding border may fall on either side of it (fp32 functions, an ulp apart)
    assert (gk != ck).float().mean() <= 2e-4
    # what no row was written to is as it was: fill, write one row, compare
    for t in (B.cache.k_pages, B.cache.v_pages, B.cache.scales):
        t.view(torch.uint8).fill_(0x3a)
    for t in (C.k_pages, C.v_pages, C.scales):
        t.view(torch.uint8).fill_(0x3a)
    n, lens = 3, torch.tensor([66, 1, 0, 97, 33], dtype=I32, device="cuda")   # row 0 of sequence 1: positions -2, -1, 0
    pos = lens[:, None].long() - n + torch.arange(n, device="cuda")
    k, v = B.rand(5, 3, n, D), B.rand(5, 3, n, D)
    emb = B.emb(pos)
    paged_cache_write(B.cache, k, v, emb, B.table, lens)
    paged_cache_write(C, k.cpu(), v.cpu(), tuple(t.cpu() for t in emb) if R else None, B.table.cpu(), lens.cpu())
    assert torch.equal(C.v_pages.view(torch.uint8), B.cache.v_pages.view(torch.uint8).cpu())
    same = C.k_pages.view(torch.uint8) == B.cache.k_pages.view(torch.uint8).cpu()
    assert (~same).float().mean() <= 2e-4 and (C.scales != B.cache.scales.cpu()).sum() <= 2e-3 * C.scales.numel()


def test_far_positions_and_wide_ranges(cuda):
    """Angles at positions of 2^20 (fp32 F + bias would be off by 0.06), 8-bit rows of very large, tiny and zero values."""
    cache = PagedPoPECache(2, heads=2, dim=32, rotate_dim=32, page_size=32, dtype=torch.float16, device="cuda")
    k, bias = torch.randn(1, 2, 32, 32, device="cuda").half(), -torch.rand(2, 32, device="cuda") * 6
    freqs = angles(torch.arange(2 ** 20 - 32, 2 ** 20, device="cuda"), 32)
    table, lens = torch.tensor([[1]], dtype=I32, device="cuda"), torch.tensor([32], dtype=I32, device="cuda")
    paged_cache_write(cache, k, k, (freqs, bias), table, lens)
    got = paged_cache_read(cache, table, lens, 32)[0][0].double()
    want = rows64(k[0], freqs, bias, 32)
    assert ((got - want).abs() <= held(want, torch.float16, False)).all()
    cache = PagedPoPECache(2, heads=1, dim=8, page_size=32, quantized=True, device="cuda")
    k = torch.zeros(1, 1, 6, 8, device="cuda").bfloat16()
    k[0, 0, 0], k[0, 0, 1], k[0, 0, 2] = 3e38, 1e-38, 2.0 ** -130
    k[0, 0, 3, 0], k[0, 0, 3, 1], k[0, 0, 3, 2], k[0, 0, 4] = INF, NAN, 3.0, 448.0
    lens = torch.tensor([6], dtype=I32, device="cuda")
    paged_cache_write(cache, k, k, None, table, lens)
    for got in paged_cache_read(cache, table, lens, 6):
        got = got[0, 0].double()
        assert ((got[0] - 3e38).abs() <= 3e38 / 16).all() and ((got[1] - 1e-38).abs() <= 1e-38 / 16).all()
        assert (got[2] <= 2.0 ** -129).all() and (got[4] == 448).all() and not got[5].any()
        assert got[3, :2].isnan().all() and got[3, 2] == 3.0 and not got[3, 3:].any()


def test_read_windows(cuda):
    B = Batch([100, 40, 0], heads=2, q8=True)
    full = [B.rows(b) for b in range(3)]
    k, v = paged_cache_read(B.cache, B.table, B.lengths, 60)
    for b, t in enumerate(B.total):
        m = min(t, 60)
        for got, want in zip((k, v), full[b]):
            assert torch.equal(got[b, :, 60 - m:].double(), want[:, t - m:]) and not got[b, :, :60 - m].any()
    cu = torch.tensor([2, 35, 35, 36], dtype=I32, device="cuda")   # rows before the first sequence and behind the last
    k, v = paged_cache_read(B.cache, B.table, B.lengths, 40, cu_seqlens=cu, head_dimension_at_first=False)
    assert k.shape == (1, 40, 2, 96) and k.is_contiguous()
    assert torch.equal(k[0, 2:35].transpose(0, 1).double(), full[0][0][:, 67:]) and torch.equal(v[0, 2:35].transpose(0, 1).double(), full[0][1][:, 67:])
    assert not k[0, :2].any() and not k[0, 35:].any() and not v[0, 35:].any()
    assert paged_cache_read(B.cache, B.table, B.lengths, 0)[0].shape == (3, 2, 0, 96)


# ---------------------------------------------------------------- attention

@pytest.mark.parametrize("D,R", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("q8", [False, True], ids=["16bit", "8bit"])
def test_attention_shapes(cuda, D, R, dtype, q8):
    """Every instance: single tokens, a few rows, many rows."""
    B = Batch([300, 33, 65, 1], heads=2, G=2, D=D, R=R, dtype=dtype, q8=q8)
    print(D, R, [f"{x:.2f}" for x in (attend_and_check(B, [1] * 4, packed=False), attend_and_check(B, [17, 1, 5, 0], packed=True, gap=1),
                                      attend_and_check(B, [299, 33, 64, 1], packed=True))], flush=True)


LENGTHS = [([1], 1), ([31], 1), ([32], 2), ([33], 33), ([5], 9), ([64, 96], 64), ([2000, 17, 0, 900], 1), ([2000, 17, 0, 900], 16), ([0, 0], 3),
           ([4097], 1), ([4097], 130), ([700, 650], 500), ([9000, 1], 1)]


@pytest.mark.parametrize("total,n", LENGTHS)
@pytest.mark.parametrize("heads,G", [(1, 1), (2, 3), (2, 8), (1, 20)])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "all"])
def test_attention_lengths(cuda, total, n, heads, G, causal):
    """Lengths of zero and one, at and around block and page borders, rows at negative positions (n above a length)."""
    B = Batch(total, heads=heads, G=G, D=32, R=16, page=32, seed=n)
    attend_and_check(B, [n] * len(total), packed=False, causal=causal)


@pytest.mark.parametrize("page", [32, 128, 1024])
@pytest.mark.parametrize("q8", [False, True], ids=["16bit", "8bit"])
def test_attention_ragged(cuda, page, q8):
    total = [1500, 3, 64, 0, 2048, 31, 129] + [40] * 70   # more sequences than a wave has lanes
    B = Batch(total, heads=2, G=2, page=page, q8=q8)
    attend_and_check(B, [1] * len(total), packed=True)
    attend_and_check(B, [700, 0, 64, 0, 1, 31, 100] + [0, 3] * 35, packed=True, gap=5, head_first=False)
    attend_and_check(B, [0] * 4 + [2048] + [0] * 72, packed=True, causal=False)


@pytest.mark.parametrize("D,R", [(64, 32), (128, 64), (200, 40)])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "all"])
def test_prompts_in_parts(cuda, D, R, causal):
    """More row tiles than the join has workgroups for, their keys in parts, the first tiles of a prompt in one."""
    attend_and_check(Batch([2300], heads=8, D=D, R=R, dtype=torch.float16), [2300], packed=False, causal=causal)


def test_shared_pages_in_parts(cuda):
    """One page table row for all sequences, of different lengths, single tokens, in parts of the key axis."""
    B = Batch([2500], heads=16, D=32, R=16)
    k, v = B.rows(0)
    lens = torch.arange(2500, 2500 - 40 * 60, -60, dtype=I32, device="cuda")
    pos = lens[:, None].long() - 1
    q = B.rand(40, 16, 1, 32)
    o = paged_flash_attn_with_pope(q, B.cache, B.emb(pos), B.table.expand(40, -1), lens)
    for b, L in enumerate(lens.tolist()):
        want, _, tol, _ = reference(q[b], angles(pos[b], 16), k[:, :L], v[:, :L], 16, 32 ** -0.5, True, B.dtype)
        assert ((o[b].double() - want).abs() <= tol).all(), L


@pytest.mark.parametrize("q8", [False, True], ids=["16bit", "8bit"])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "all"])
def test_parts_by_length(cuda, q8, causal):
    """Long sequences between short and empty ones, their keys in parts; packed with empty segments and rows behind."""
    B = Batch([1900, 40, 0, 1200] * 5, heads=2, G=4, D=96, R=48, page=32, q8=q8)
    attend_and_check(B, [30] * 20, packed=False, causal=causal)
    attend_and_check(B, [70, 33, 0, 5, 300, 0, 0, 100, 1, 40, 0, 0] + [9, 8, 0, 64] * 2, packed=True, causal=causal, gap=150)


@pytest.mark.parametrize("n", [1, 70])
def test_wide_page_tables(cuda, n):
    """A page table far wider than the sequences are long: within the same bounds, behind them bad page numbers."""
    B = Batch([300, 77], heads=2, G=2)
    table = torch.full((2, 5000), 2 ** 31 - 1, dtype=I32, device="cuda")
    table[:, :B.table.shape[1]] = B.table
    B.table = table
    attend_and_check(B, [n, n], packed=False)
    attend_and_check(B, [n, min(n, 50)], packed=True, gap=3)


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0, 40.0])
def test_softmax_scales(cuda, scale):
    for dtype in (torch.bfloat16, torch.float16):
        B = Batch([200, 64], heads=2, dtype=dtype)
        attend_and_check(B, [3, 3], packed=False, scale=scale)


@pytest.mark.parametrize("size", [1e-6, 1e-3, 60.0, 2e4])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("q8", [False, True], ids=["16bit", "8bit"])
def test_values_far_from_one(cuda, size, dtype, q8):
    """Tiny and large values: the second product's operands carry the 8-bit values' scales.  Keys are small, so that every
    key counts."""
    B = Batch([700, 64], heads=2, dtype=dtype, q8=q8)
    B.k, B.v = B.k * 0.25, (B.v.float() * size).clamp(-65000, 65000).to(dtype)
    paged_cache_write(B.cache, B.k, B.v, B.emb(B.pos), B.table, B.lengths, cu_seqlens=B.cu)
    for new in ([1, 1], [64, 64]):
        q = B.rand(1, 2, sum(new), 64)
        cu = torch.tensor([0, new[0], sum(new)], dtype=I32, device="cuda")
        pos = torch.cat([torch.arange(t - n, t, device="cuda") for t, n in zip(B.total, new)])
        o = paged_flash_attn_with_pope(q, B.cache, B.emb(pos), B.table, B.lengths, cu_seqlens=cu)
        for b in range(2):
            s = slice(int(cu[b]), int(cu[b + 1]))
            k, v = B.rows(b)
            want, _, tol, _ = reference(q[0, :, s], angles(pos[s], 32), k, v, 32, 0.125, True, dtype)
            # the reference's absolute term is for values of about 1; outputs below fp16's normal range have its spacing
            tol = tol - 2.0 ** -25 + (2.0 ** -25 if dtype == torch.float16 else 0.0)
            assert ((o[0, :, s].double() - want).abs() <= tol).all()


def test_layouts_and_strides(cuda):
    """Views with any strides and odd offsets, broadcast angles and one bias row, int64 tables: the same bits."""
    B = Batch([90, 90], heads=2, G=2, D=40, R=20)
    n, Hq, D = 7, 4, 40
    pos = torch.arange(83, 90, device="cuda")
    q, k, v = (B.rand(2, h, n, D) for h in (Hq, 2, 2))
    freqs = angles(pos, 20)
    bias = B.bias[:1]
    lens = torch.tensor([90, 90], device="cuda")

    def run(q, k, v, emb, table, lens, hf=True):
        c = PagedPoPECache(B.cache.num_pages, heads=2, dim=D, rotate_dim=20, device="cuda")
        c.k_pages.copy_(B.cache.k_pages), c.v_pages.copy_(B.cache.v_pages)
        paged_cache_write(c, k, v, emb, table, lens, head_dimension_at_first=hf)
        o = paged_flash_attn_with_pope(q, c, emb, table, lens, head_dimension_at_first=hf)
        r = paged_cache_read(c, table, lens, n, head_dimension_at_first=hf)
        return [t if hf else t.transpose(1, 2) for t in (o, *r)]

    want = run(q, k, v, (freqs, bias), B.table, lens.int())

    def odd(t):   # rows 3 elements into a buffer, row stride D + 5
        buf = torch.zeros(t.numel() // D * (D + 5) + 3, dtype=t.dtype, device="cuda")
        out = buf[3:].view(*t.shape[:-1], D + 5)[..., :D]
        out.copy_(t)
        return out

    tr = lambda t: t.transpose(1, 2).contiguous()
    slow = lambda t: torch.stack((t, t), -1)[..., 0]   # feature stride 2
    wide = torch.zeros(2, B.table.shape[1] + 3, dtype=torch.int64, device="cuda")
    wide[:, 1:-2] = B.table
    for got in (run(odd(q), odd(k), odd(v), (freqs, bias), B.table, lens), run(tr(q), tr(k), tr(v), (freqs, bias.expand(2, 20)), B.table, lens, False),
                run(slow(q), slow(k), slow(v), (freqs.expand(2, n, 20), bias[0]), wide[:, 1:-2], lens),
                run(q, k, v, (slow(freqs), bias.double()), B.table, torch.stack((lens, lens), 1)[:, 0])):
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_pages_outside_the_cache(cuda):
    """Bad page numbers: skipped by writes, zeros to reads, not seen by attention; lengths out of range."""
    for q8 in (False, True):
        B = Batch([200, 150], heads=2, page=32, q8=q8)
        clean = [B.rows(b) for b in range(2)]
        good = B.table.clone()
        for bad in (-1, B.cache.num_pages, 2 ** 31 - 1, -2 ** 31):
            B.table.copy_(good)
            B.table[0, 2] = bad
            k, v = (t[0].double() for t in paged_cache_read(B.cache, B.table[:1], B.lengths[:1], 200))
            gone = slice(64, 96)
            assert not k[:, gone].any() and not v[:, gone].any() and torch.equal(k[:, 96:], clean[0][0][:, 96:])
            before = [t.clone() for t in (B.cache.k_pages, B.cache.v_pages, B.cache.scales)]
            lens = torch.tensor([96, 150], dtype=I32, device="cuda")
            paged_cache_write(B.cache, B.rand(1, 2, 32, 64), B.rand(1, 2, 32, 64), B.emb(torch.arange(64, 96, device="cuda")), B.table[:1], lens[:1])
            assert all(torch.equal(a, b) for a, b in zip(before, (B.cache.k_pages, B.cache.v_pages, B.cache.scales)))
            q = B.rand(1, 2, 3, 64)
            pos = torch.arange(197, 200, device="cuda")
            for n in (3, 1):
                o = paged_flash_attn_with_pope(q[:, :, -n:], B.cache, B.emb(pos[-n:]), B.table[:1], B.lengths[:1], causal=False)
                keep = torch.ones(200, dtype=torch.bool, device="cuda")
                keep[gone] = False
                want, _, tol, _ = reference(q[0, :, -n:], angles(pos[-n:], 32), k[:, keep], v[:, keep], 32, 0.125, False, B.dtype)
                assert ((o[0].double() - want).abs() <= tol).all()
        B.table.copy_(good)
        cap = good.shape[1] * 32
        q = B.rand(2, 2, 2, 64)
        f = B.emb(torch.zeros(2, dtype=torch.long, device="cuda"))
        big = paged_flash_attn_with_pope(q, B.cache, f, B.table, torch.tensor([2 ** 31 - 1, cap + 1], dtype=I32, device="cuda"))
        assert torch.equal(big, paged_flash_attn_with_pope(q, B.cache, f, B.table, torch.tensor([cap, cap], dtype=I32, device="cuda")))
        assert not paged_flash_attn_with_pope(q, B.cache, f, B.table, torch.tensor([-2 ** 31, 0], dtype=I32, device="cuda")).any()


@pytest.mark.parametrize("q8", [False, True], ids=["16bit", "8bit"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 200])
def test_not_finite_where_masked(cuda, q8, dtype, D):
    """Stale slots behind the sequence and keys later than a row hold infinities and NaN: nothing changes."""
    for n, G in ((1, 1), (40, 1), (20, 2), (150, 2)):
        B = Batch([150, 70, 201], heads=2, G=G, D=D, R=32, dtype=dtype, q8=q8, page=128)
        pos = B.lengths[:, None].long() - n + torch.arange(n, device="cuda")
        q = B.rand(3, 2 * G, n, D)
        call = lambda: paged_flash_attn_with_pope(q, B.cache, B.emb(pos), B.table, B.lengths)
        clean = call()
        # rows behind the end: written by a longer sequence that had these pages before
        longer = B.lengths + 20
        junk = torch.full((3, 2, 20, D), NAN, device="cuda").to(dtype)
        junk[:, :, ::2] = INF
        paged_cache_write(B.cache, junk, junk, B.emb(torch.zeros(20, dtype=torch.long, device="cuda")), B.table, longer)
        assert torch.equal(call(), clean)
        if n == 1:
            continue
        # the last new key and value of each sequence: only the last row sees them
        k = torch.full((3, 2, 1, D), NAN, device="cuda").to(dtype)
        v = B.rand(3, 2, 1, D)
        v[:, :, 0, 5], v[:, :, 0, 6] = INF, NAN
        paged_cache_write(B.cache, k, v, B.emb(pos[:, -1:]), B.table, B.lengths)
        o = call()
        # rows at negative positions see nothing
        assert torch.equal(o[:, :, :-1], clean[:, :, :-1]) and o[:, :, -1].isnan().all()
        k = B.rand(3, 2, 1, D) * 0.5
        paged_cache_write(B.cache, k, v, B.emb(pos[:, -1:]), B.table, B.lengths)
        o = call()
        assert torch.equal(o[:, :, :-1], clean[:, :, :-1]) and o[:, :, -1, 6].isnan().all()
        # 8 bits have no infinity: the value is stored as NaN
        assert o[:, :, -1, 5].isnan().all() if q8 else (o[:, :, -1, 5] == INF).all()
        assert o[:, :, -1, 7:].isfinite().all()


def test_not_finite_queries_and_values_seen(cuda):
    B = Batch([300, 90], heads=2, G=2)
    pos = B.lengths[:, None].long() - 4 + torch.arange(4, device="cuda")
    q = B.rand(2, 4, 4, 64)
    clean = paged_flash_attn_with_pope(q, B.cache, B.emb(pos), B.table, B.lengths)
    q[0, 1, 2, 40] = NAN
    q[1, 3, 0, 3] = INF
    o = paged_flash_attn_with_pope(q, B.cache, B.emb(pos), B.table, B.lengths)
    bad = torch.zeros(2, 4, 4, dtype=torch.bool, device="cuda")
    bad[0, 1, 2] = bad[1, 3, 0] = True
    assert o[bad].isnan().all() and torch.equal(o[~bad], clean[~bad])
    # every score of a split NaN: the row is NaN, not skipped
    B = Batch([8000], heads=1)
    k = torch.full((1, 1, 32, 64), NAN, device="cuda").bfloat16()
    paged_cache_write(B.cache, k, B.rand(1, 1, 32, 64), B.emb(torch.arange(7968, 8000, device="cuda")), B.table, B.lengths)
    o, lse = paged_flash_attn_with_pope(B.rand(1, 1, 1, 64), B.cache, B.emb(torch.tensor([7999], device="cuda")), B.table, B.lengths, return_lse=True)
    assert o.isnan().all() and lse.isnan().all()


def test_offsets_beyond_32_bits(cuda):
    """A cache whose pages lie beyond 2^32 bytes and 2^31 elements, 16- and 8-bit."""
    for q8, pages in ((False, 300000), (True, 600000)):
        c = PagedPoPECache(pages, heads=2, dim=64, rotate_dim=64, page_size=32, quantized=q8, device="cuda")
        assert c.k_pages.numel() > 2 ** 31
        table = torch.tensor([[pages - 1, 5, pages - 7]], dtype=I32, device="cuda")
        small = torch.tensor([[2, 0, 1]], dtype=I32, device="cuda")
        d = PagedPoPECache(3, heads=2, dim=64, rotate_dim=64, page_size=32, quantized=q8, device="cuda")
        n = torch.tensor([90], dtype=I32, device="cuda")
        k, v, q = (torch.randn(1, 2, 90, 64, device="cuda").bfloat16() for _ in range(3))
        emb = (angles(torch.arange(90, device="cuda"), 64), torch.zeros(2, 64, device="cuda"))
        for cache, t in ((c, table), (d, small)):
            paged_cache_write(cache, k, v, emb, t, n)
        for a, b in zip(paged_cache_read(c, table, n, 90), paged_cache_read(d, small, n, 90)):
            assert torch.equal(a, b) and a.any()
        assert torch.equal(paged_flash_attn_with_pope(q, c, emb, table, n), paged_flash_attn_with_pope(q, d, emb, small, n))
        assert not c.k_pages[6:1000].any()
        del c
        torch.cuda.empty_cache()


# ---------------------------------------------------------------- a run together, streams, graphs, tracing

@pytest.mark.parametrize("q8", [False, True], ids=["16bit", "8bit"])
def test_serving_run(cuda, q8):
    """Two prompts in chunks, then single tokens, against the framework's attention over the whole sequences.

    The contiguous path rounds K_hat to bf16 as the cache does, with the bias on the query's side: each rounds Q_hat or
    K_hat differently, and each output to bf16.  Bound: 2e-2 absolute, the contract of the bf16 flash forward; 8-bit
    caches are held to the same path fed with what they hold."""
    pope = PoPE(32, heads=2, bias_uniform_init=True).cuda()
    Hq, D, page = 4, 64, 32
    cache = PagedPoPECache(20, heads=2, dim=D, rotate_dim=32, page_size=page, quantized=q8, device="cuda")
    table = torch.randperm(20, device="cuda").to(I32).view(2, 10)
    total = [200, 170]
    q, k, v = (torch.randn(2, h, 200, D, device="cuda").bfloat16() for h in (Hq, 2, 2))
    got = torch.zeros_like(q)
    done = [0, 0]
    with torch.no_grad():
        for new in ([64, 100], [90, 60], [40, 4]) + ([1, 1],) * 6:
            cu = torch.tensor([0, new[0], sum(new)], dtype=I32, device="cuda")
            part = [slice(d, d + n) for d, n in zip(done, new)]
            done = [d + n for d, n in zip(done, new)]
            pos = torch.cat([torch.arange(s.start, s.stop, device="cuda") for s in part])
            pack = lambda t: torch.cat([t[b, :, s] for b, s in enumerate(part)], 1)[None]
            lens = torch.tensor(done, dtype=I32, device="cuda")
            paged_cache_write(cache, pack(k), pack(v), pope(pos), table, lens, cu_seqlens=cu)
            o = paged_flash_attn_with_pope(pack(q), cache, pope(pos), table, lens, cu_seqlens=cu)
            for b, s in enumerate(part):
                got[b, :, s] = o[0, :, cu[b]:cu[b + 1]]
        assert done == [200, 170]
        for b, L in enumerate(total):
            if q8:
                kh, vh = (t.double() for t in paged_cache_read(cache, table[b:b + 1], torch.tensor([L], dtype=I32, device="cuda"), L))
                freqs, _ = pope(L)
                want, _, tol, _ = reference(q[b, :, :L], freqs, kh[0], vh[0], 32, D ** -0.5, True, torch.bfloat16)
                assert ((got[b, :, :L].double() - want).abs() <= tol).all()
            else:
                want = pope_amd.flash_attn_with_pope(q[b:b + 1, :, :L], k[b:b + 1, :, :L], v[b:b + 1, :, :L], pos_emb=pope(L), causal=True)
                assert (got[b, :, :L].float() - want[0].float()).abs().max() <= 2e-2


def test_streams_and_repeats(cuda):
    """The current stream is used, repeated calls give the same bits, and calls at once on two streams do not mix."""
    B = Batch([5000, 300], heads=2, G=2)
    q = [B.rand(2, 4, 1, 64) for _ in range(2)]
    emb = B.emb(B.lengths[:, None].long() - 1)
    want = [paged_flash_attn_with_pope(x, B.cache, emb, B.table, B.lengths) for x in q]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                outs[i].append(paged_flash_attn_with_pope(q[i], B.cache, emb, B.table, B.lengths))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in outs[i])


def test_graph_of_a_serving_step(cuda):
    """A captured write + attention step replays with new rows, lengths and pages; two graphs do not share scratch."""
    B = Batch([3000, 900], heads=2, G=2)
    k, v, q = (B.rand(2, h, 1, 64) for h in (2, 2, 4))
    pos = (B.lengths.long() - 1)[:, None]
    freqs, bias = B.emb(pos)

    def step():
        paged_cache_write(B.cache, k, v, (freqs, bias), B.table, B.lengths)
        return paged_flash_attn_with_pope(q, B.cache, (freqs, bias), B.table, B.lengths)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for g in graphs:
        with torch.cuda.graph(g):
            outs.append(step())
    for n in range(4):
        for t in (k, v, q):
            t.copy_(B.rand(*t.shape))
        B.lengths.copy_(torch.tensor([2900 + 7 * n, 800 + n], dtype=I32, device="cuda"))
        freqs.copy_(angles((B.lengths.long() - 1)[:, None], 32))
        if n == 2:
            B.table[1, 3] = B.table[0, 0]   # a shared page
        want = step()
        for t in outs:
            t.zero_()
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want) and torch.equal(outs[1], want)
        assert want.any()


def test_graph_of_packed_chunks(cuda):
    """A captured call of packed chunks replays with other bounds, lengths and pages."""
    B = Batch([2100, 700, 64], heads=2, G=2)
    q = B.rand(1, 4, 150, 64)
    cu = torch.tensor([0, 90, 140, 150], dtype=I32, device="cuda")
    freqs = B.emb(torch.zeros(150, device="cuda"))[0]
    run = lambda: paged_flash_attn_with_pope(q, B.cache, (freqs, B.bias), B.table, B.lengths, cu_seqlens=cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        run()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = run()
    for bounds, lens in (([0, 90, 140, 150], [2100, 700, 64]), ([0, 0, 150, 150], [5, 690, 0]), ([20, 100, 100, 130], [2000, 64, 40]), ([0, 1, 2, 3], [2100, 1, 64])):
        cu.copy_(torch.tensor(bounds, dtype=I32, device="cuda"))
        B.lengths.copy_(torch.tensor(lens, dtype=I32, device="cuda"))
        q.copy_(B.rand(*q.shape))
        freqs.copy_(angles(torch.randint(0, 2100, (150,), generator=B.g, device="cuda"), 32))
        B.table.copy_(B.table[[0, 1, 2]].roll(1, 1).where(torch.tensor([[True], [False], [True]], device="cuda"), B.table))
        want = run()
        out.fill_(NAN)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and want.any()


def test_ops_trace(cuda):
    from pope_amd import paged as m
    B = Batch([70, 40], heads=2, G=2, q8=True)
    c = B.cache
    q, k, v = (B.rand(2, h, 3, 64) for h in (4, 2, 2))
    freqs, bias = B.emb(B.lengths[:, None].long() - 3 + torch.arange(3, device="cuda"))
    tests = ("test_schema", "test_faketensor")
    torch.library.opcheck(m.paged_write_op, (k, v, freqs, bias, c.k_pages, c.v_pages, c.scales, B.table, B.lengths, None, 64), test_utils=tests)
    torch.library.opcheck(m.paged_read_op, (c.k_pages, c.v_pages, c.scales, B.table, B.lengths, None, 5, 64, 32, 64, False, False), test_utils=tests)
    torch.library.opcheck(m.paged_attn_op, (q, freqs, c.k_pages, c.v_pages, c.scales, B.table, B.lengths, None, 64, True, 0.125, True), test_utils=tests)

    def step(q, k, v, freqs, bias, table, lengths):
        paged_cache_write(c, k, v, (freqs, bias), table, lengths)
        return paged_flash_attn_with_pope(q, c, (freqs, bias), table, lengths) * 1

    want = step(q, k, v, freqs, bias, B.table, B.lengths)
    pages = c.k_pages.clone()
    c.k_pages.zero_()
    paged_cache_write(c, B.k, B.v, B.emb(B.pos), B.table, B.lengths, cu_seqlens=B.cu)
    got = torch.compile(step, backend="aot_eager", fullgraph=True)(q, k, v, freqs, bias, B.table, B.lengths)
    assert torch.equal(got, want) and torch.equal(c.k_pages, pages)


def test_extents_of_one(cuda):
    """Dims of extent 1 may have any stride: one page, one sequence, one column, one rotated dim."""
    c = PagedPoPECache(2, heads=1, dim=1, rotate_dim=1, page_size=32, device="cuda")
    odd = lambda t: t.as_strided(t.shape, [7 if n == 1 else s for n, s in zip(t.shape, t.stride())])
    table, lens = torch.ones(1, 1, dtype=I32, device="cuda"), torch.full((1,), 3, dtype=I32, device="cuda")
    k = torch.randn(1, 1, 3, 1, device="cuda").bfloat16()
    emb = (torch.rand(3, 1, device="cuda"), torch.zeros(1, 1, device="cuda"))
    paged_cache_write(c, k, k, emb, table, lens)
    want = paged_flash_attn_with_pope(k, c, emb, table, lens), *paged_cache_read(c, table, lens, 3)
    c.k_pages.zero_(), c.v_pages.zero_()
    emb = tuple(odd(t) for t in emb)
    paged_cache_write(c, odd(k), odd(k), emb, odd(table), odd(lens))
    got = paged_flash_attn_with_pope(odd(k), c, emb, odd(table), odd(lens)), *paged_cache_read(c, odd(table), odd(lens), 3)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and got[1].any()


def test_refusals_on_the_gpu(cuda):
    B = Batch([70], heads=2)
    q = B.rand(1, 2, 1, 64)
    emb = B.emb(torch.tensor([69], device="cuda"))
    for bad in (lambda: paged_flash_attn_with_pope(q, B.cache, emb, B.table.cpu(), B.lengths), lambda: paged_flash_attn_with_pope(q.cpu(), B.cache, emb, B.table, B.lengths),
                lambda: paged_flash_attn_with_pope(q, B.cache, (emb[0].cpu(), emb[1]), B.table, B.lengths)):
        with pytest.raises(RuntimeError):
            bad()
    c = PagedPoPECache(2, heads=2, dim=64, rotate_dim=32, device="cuda")
    c.v_pages = c.v_pages[:1]
    with pytest.raises(ValueError, match="do not fit"):
        paged_flash_attn_with_pope(q, c, emb, B.table, B.lengths)


@pytest.mark.parametrize("causal", [True, False], ids=["causal", "all"])
def test_segments_that_overlap(cuda, causal):
    """Bounds that descend: nothing is said of these rows' values, but the call stays within its buffers (host test of the
    plan), and the rows of the calls behind it are right."""
    total = [4096 if causal else 1024] * 5
    B = Batch(total, heads=1, D=32, R=16)
    cu = torch.tensor([0, 1280, 0, 1280, 0, 1280], dtype=I32, device="cuda")
    q = B.rand(1, 1, 1280, 32)
    f = B.emb(torch.zeros(1280, dtype=torch.long, device="cuda"))
    o = paged_flash_attn_with_pope(q, B.cache, f, B.table, B.lengths, cu_seqlens=cu, causal=causal)
    torch.cuda.synchronize()
    assert o.shape == q.shape
    attend_and_check(B, [1280, 0, 3, 200, 1], packed=True, causal=causal)


@pytest.mark.parametrize("gap", [0, 3, 150])
@pytest.mark.parametrize("causal", [True, False], ids=["causal", "all"])
def test_rows_without_keys_next_to_parts(cuda, causal, gap):
    """Rows behind the last sequence and rows of sequences of length zero, several tiles of each, next to sequences whose keys
    are cut into parts that the first workgroups get."""
    B = Batch([1900, 40, 0, 1200] * 5, heads=2, G=4, D=96, R=48, page=32)
    attend_and_check(B, [70, 33, 100, 5, 300, 0, 100, 100, 1, 40, 0, 0] + [9, 8, 0, 64] * 2, packed=True, causal=causal, gap=gap)


def with_infinities(q, freqs, k, v, R, scale, causal, dtype):
    """`reference` where held rows have infinities and NaN: the formula in 64 bits, an infinite value counting where its key
    is seen.  The bounds are `reference`'s, with the formula's own weights (a key of score -inf has none, so it must not
    share in sum_j p_j |v_j|, as it does where its infinity is taken for 0) and the finite elements of keys and values: an
    infinity that counts leaves nothing to round."""
    n, L, G = q.shape[1], k.shape[1], q.shape[0] // k.shape[0]
    fin = lambda t: torch.where(t.isfinite(), t, 0.0)
    qh = rows64(q, freqs, torch.zeros(1, R, device="cuda"), R).cpu()
    k, v = k.repeat(G, 1, 1).cpu(), v.repeat(G, 1, 1).cpu()
    see = torch.arange(L) <= (L - n + torch.arange(n))[:, None] if causal else torch.ones(n, L, dtype=torch.bool)
    sc = (torch.bmm(qh, k.transpose(1, 2).contiguous()) * scale).masked_fill(~see, -INF)
    p = torch.softmax(sc.masked_fill(~see.any(-1)[:, None], 0.0), -1).masked_fill(~see, 0.0)
    o, pv = torch.bmm(p, fin(v)), torch.bmm(p, fin(v).abs())
    A = (torch.bmm(qh.abs(), fin(k).abs().transpose(1, 2).contiguous()) * abs(scale)).masked_fill(sc == -INF, 0.0)
    u, f16 = torch.finfo(dtype).eps / 2, dtype == torch.float16
    x = (u * u + k.shape[-1] * 2.0 ** -24 + 1e-6) * A.amax(-1, keepdim=True)
    if f16:
        x = x + 2.0 ** -25 * fin(k).abs().sum(-1).amax(-1)[:, None, None] * abs(scale)
    tol = u * o.abs() + (u + 2 * x + 2e-5) * pv + 2.0 ** -25
    if f16:
        tol = tol + 2.0 ** -25 * fin(v).abs().sum(1, keepdim=True)
    for j in (~v.isfinite()).any(-1).any(0).nonzero().flatten().tolist():
        o += torch.where(see[:, j, None] & ~v[:, j].isfinite()[:, None, :], p[..., j, None] * torch.where(v[:, j].isfinite(), 0.0, v[:, j])[:, None, :], 0.0)
    return o.cuda(), torch.logsumexp(sc, -1).cuda(), tol.cuda(), x[..., 0].cuda() + 1e-5


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("D", [64, 128, 200])
@pytest.mark.parametrize("n,G", [(1, 1), (3, 4), (40, 1), (150, 2)])
@pytest.mark.parametrize("where", ["values", "keys", "both"])
def test_infinities_seen(cuda, dtype, D, n, G, where):
    """Infinite keys and values that rows see, in every block: a key's infinity against a column of the other sign has weight 0,
    an infinite value makes its column of the output infinite."""
    total = [2500, 700, 151, 33]
    B = Batch(total, heads=2, G=G, D=D, R=32, dtype=dtype)
    for b, t in enumerate(total):
        at = int(B.cu[b])
        if where != "keys":
            for pos, col, x in ((3, 5, INF), (31, 6, -INF), (t // 2, 7, INF), (t // 2 + 1, 7, -INF), (t - 1, 8, INF), (t // 3, D - 1, -INF)):
                B.v[0, :, at + pos, col] = x
        if where != "values":
            for pos, col, x in ((2, 40, INF), (t // 2, 41, -INF), (t - 1, 40, INF)):
                B.k[0, :, at + pos, col] = x
    paged_cache_write(B.cache, B.k, B.v, B.emb(B.pos), B.table, B.lengths, cu_seqlens=B.cu)
    pos = B.lengths[:, None].long() - n + torch.arange(n, device="cuda")
    q = B.rand(4, 2 * G, n, D)
    q[:, ::2, :, 40].abs_().neg_()   # half of the heads give the infinite keys no weight, where their rows' signs are such
    q[:, ::2, :, 41].abs_()
    for causal in (True, False):
        o, lse = paged_flash_attn_with_pope(q, B.cache, B.emb(pos), B.table, B.lengths, causal=causal, return_lse=True)
        for b in range(4):
            k, v = B.rows(b)
            want, wl, tol, ltol = with_infinities(q[b], angles(pos[b], 32), k, v, 32, D ** -0.5, causal, dtype)
            got = o[b].double()
            assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf()) and torch.equal(got[got.isinf()], want[want.isinf()])
            fin = want.isfinite()
            assert ((got - want).abs()[fin] <= tol[fin]).all(), ((got - want).abs() / tol)[fin].max().item()
            assert fin.any()
            gl = lse[b].double()
            assert torch.equal(gl.isnan(), wl.isnan() | (wl == INF))   # a score of +inf: no weights, and no sum of them
            fin = wl.isfinite()
            assert torch.equal(gl.isfinite(), fin) and ((gl - wl).abs()[fin] <= (ltol + 1e-6 * wl.abs())[fin]).all()


@pytest.mark.parametrize("n,G", [(1, 1), (40, 1)])
@pytest.mark.parametrize("D", [64, 128])
def test_infinities_next_to_bad_pages(cuda, n, G, D):
    """Infinities seen where pages of the same sequence lie outside the cache: as the CPU cache has it."""
    B = Batch([1500, 90], heads=2, G=G, D=D, R=32, page=32)
    B.v[0, :, 10, 4], B.v[0, :, 700, 5], B.k[0, :, 300, 40] = INF, -INF, INF
    B.v[0, :, 1500 + 33, 6] = -INF
    paged_cache_write(B.cache, B.k, B.v, B.emb(B.pos), B.table, B.lengths, cu_seqlens=B.cu)
    B.table[0, 3], B.table[0, 20], B.table[1, 0] = -1, 2 ** 31 - 1, B.cache.num_pages
    C = PagedPoPECache(B.cache.num_pages, heads=2, dim=D, rotate_dim=32, page_size=32)
    C.k_pages.copy_(B.cache.k_pages), C.v_pages.copy_(B.cache.v_pages)
    pos = B.lengths[:, None].long() - n + torch.arange(n, device="cuda")
    q = B.rand(2, 2 * G, n, D)
    q[:, ::2, :, 40].abs_().neg_()
    emb = B.emb(pos)
    for causal in (True, False):
        got = paged_flash_attn_with_pope(q, B.cache, emb, B.table, B.lengths, causal=causal).float().cpu()
        want = paged_flash_attn_with_pope(q.cpu(), C, tuple(t.cpu() for t in emb), B.table.cpu(), B.lengths.cpu(), causal=causal).float()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf()) and torch.equal(got[got.isinf()], want[got.isinf()])
        fin = want.isfinite()
        assert fin.any() and want.isinf().any()
        # both fp32 arithmetic over the same rows: a rounding each, and P's in the many-row kernel, of outputs below 4
        assert ((got - want).abs()[fin] <= 4 * 2.0 ** -8 * 3).all()


@pytest.mark.parametrize("q8", [False, True], ids=["16bit", "8bit"])
@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("D", [64, 200])
def test_values_at_the_end_of_fp16(cuda, q8, n, D):
    """Averages of values next to fp16's largest stay finite: an 8-bit code may stand for 65536 (65000 does), and P's rounding
    may carry an average past the values'.  The true average is 65504 (what reads give), P is off by 2^-11, a sum by less."""
    B = Batch([1, 70, 3000], heads=2, D=D, dtype=torch.float16, q8=q8)
    B.v = torch.full_like(B.v, 65000.0 if q8 else 65504.0)
    B.v[..., 1::2] *= -1
    paged_cache_write(B.cache, B.k, B.v, B.emb(B.pos), B.table, B.lengths, cu_seqlens=B.cu)
    assert (B.rows(2)[1].abs() == 65504).all()
    pos = (B.lengths[:, None].long() - n + torch.arange(n, device="cuda")).clamp_min(0)
    o = paged_flash_attn_with_pope(B.rand(3, 2, n, D), B.cache, B.emb(pos), B.table, B.lengths, causal=False).double()
    assert o.isfinite().all() and (o.abs() >= 65504 * (1 - 3 * 2.0 ** -11)).all() and (o[..., 0] > 0).all() and (o[..., 1] < 0).all()


def test_rounded_weights_at_the_end_of_fp16(cuda):
    """Many rows: a weight of 2^7.00073 = 128.0648 (against 1 three blocks before) is 128.125 in fp16 and itself in their sum: the
    average would be 65504 (1 + 0.0602 / 129.06) = 65534, which rounds to infinity."""
    c = PagedPoPECache(4, heads=1, dim=32, page_size=32, dtype=torch.float16, device="cuda")
    k = torch.zeros(1, 1, 128, 32, device="cuda").half()
    k[..., 0] = -60
    k[0, 0, 3, 0], k[0, 0, 100, 0] = 0, 7
    v, q = torch.full_like(k, 65504.0), torch.zeros_like(k[:, :, :40])
    q[..., 0] = 1
    table, lens = torch.tensor([[1, 0, 3, 2]], dtype=I32, device="cuda"), torch.tensor([128], dtype=I32, device="cuda")
    paged_cache_write(c, k, v, None, table, lens)
    o = paged_flash_attn_with_pope(q, c, None, table, lens, causal=False, softmax_scale=7.00073 / 7 * math.log(2))
    assert (o == 65504).all()


def test_8_bit_rows_at_the_end_of_bf16(cuda):
    """3.39e38 has a code that stands for 2^128: it is read as bf16's largest, as fp16's are."""
    c = PagedPoPECache(1, heads=1, dim=8, page_size=32, quantized=True, device="cuda")
    k = torch.full((1, 1, 2, 8), torch.finfo(torch.bfloat16).max, device="cuda").bfloat16()
    k[..., 1::2] *= -1
    table, lens = torch.zeros(1, 1, dtype=I32, device="cuda"), torch.tensor([2], dtype=I32, device="cuda")
    paged_cache_write(c, k, k, None, table, lens)
    for got in paged_cache_read(c, table, lens, 2):
        assert torch.equal(got, k)


def test_forward_mode_tangents_are_refused(cuda):
    import torch.autograd.forward_ad as fwd
    B = Batch([70], heads=2)
    q, emb = B.rand(1, 2, 1, 64), B.emb(torch.tensor([69], device="cuda"))
    one = lambda t: fwd.make_dual(t, torch.ones_like(t))
    with fwd.dual_level(), torch.no_grad():
        for call in (lambda: paged_flash_attn_with_pope(one(q), B.cache, emb, B.table, B.lengths),
                     lambda: paged_flash_attn_with_pope(q, B.cache, (one(emb[0]), emb[1]), B.table, B.lengths),
                     lambda: paged_cache_write(B.cache, one(q), q, emb, B.table, B.lengths), lambda: paged_cache_write(B.cache, q, one(q), emb, B.table, B.lengths),
                     lambda: paged_cache_write(B.cache, q, q, (emb[0], one(emb[1])), B.table, B.lengths)):
            with pytest.raises(RuntimeError, match="gradient"):
                call()


@pytest.mark.parametrize("n", [1, 3, 70])
def test_rows_that_overlap(cuda, n):
    """Windows that slide by one element: two dims of stride 1, of which the features stay the output's last."""
    from pope_amd import paged as m
    B = Batch([90, 75], heads=2, D=32, R=16)
    flat = B.rand(2, 2, n + 31)
    q = flat.unfold(2, 32, 1)
    assert q.shape == (2, 2, n, 32) and q.stride(2) == q.stride(3) == 1
    emb = B.emb(B.lengths[:, None].long() - n + torch.arange(n, device="cuda"))
    want = paged_flash_attn_with_pope(q.contiguous(), B.cache, emb, B.table, B.lengths)
    got = paged_flash_attn_with_pope(q, B.cache, emb, B.table, B.lengths)
    assert got.stride(-1) == 1 and torch.equal(got, want)
    c = B.cache
    args = (q, emb[0], c.k_pages, c.v_pages, c.scales, B.table, B.lengths, None, 64, True, 32 ** -0.5, False)
    assert torch.equal(m.paged_attn_op(*args)[0], want)
    torch.library.opcheck(m.paged_attn_op, args, test_utils=("test_faketensor",))
    paged_cache_write(c, q, q, emb, B.table, B.lengths)   # read rows may overlap too
    a = [t.clone() for t in (c.k_pages, c.v_pages)]
    paged_cache_write(c, q.contiguous(), q.contiguous(), emb, B.table, B.lengths)
    assert torch.equal(a[0], c.k_pages) and torch.equal(a[1], c.v_pages)


@pytest.mark.parametrize("n,total", [(1, 5), (3, 2500), (40, 70), (40, 2500)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_rows_whose_keys_all_have_weight_zero(cuda, n, total, dtype):
    """Every visible score -inf: as with no key to see, 0 and a log-sum-exp of -inf, as CPU caches have it."""
    c = PagedPoPECache(-(-total // 32), heads=2, dim=48, page_size=32, dtype=dtype, device="cuda")
    k, v, q = (torch.randn(1, 2, m, 48, device="cuda").to(dtype) for m in (total, total, n))
    k[..., 2], q[:, 0, :, 2], q[:, 1, :, 2] = -INF, 1.0, -1.0
    table, lens = torch.arange(c.num_pages, device="cuda").to(I32)[None], torch.tensor([total], dtype=I32, device="cuda")
    paged_cache_write(c, k, v, None, table, lens)
    for causal in (True, False):
        o, lse = paged_flash_attn_with_pope(q, c, None, table, lens, causal=causal, return_lse=True)
        assert not o[0, 0].any() and (lse[0, 0] == -INF).all()
        assert o[0, 1].isnan().all()   # scores of +inf


@pytest.mark.parametrize("n", [2, 40])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
def test_softmax_scale_zero_keeps_nan(cuda, n, dtype):
    """0 x inf is NaN, in queries and keys, as the formula and CPU caches have it; finite rows average the values."""
    B = Batch([100], heads=2, dtype=dtype)
    pos = torch.arange(100 - n, 100, device="cuda")
    q = B.rand(1, 2, n, 64)
    q[0, 0, 0, 3], q[0, 0, 1, 40], q[0, 1, 0, 50] = NAN, INF, -INF
    bad = ~q.isfinite().all(-1)
    run = lambda: paged_flash_attn_with_pope(q, B.cache, B.emb(pos), B.table, B.lengths, softmax_scale=0.0, causal=False)
    o = run()
    assert o[bad].isnan().all() and o[~bad].isfinite().all()
    mean = B.v[0].double().mean(1, keepdim=True)
    err = (o[0].double() - mean).abs()[~bad[0]]
    assert (err <= 2e-2).all()   # an average of 100 values: P is exact, 2^-9 of a mean below 1 and fp32 sums
    B.k[0, 0, 9, 45] = INF
    paged_cache_write(B.cache, B.k, B.v, B.emb(B.pos), B.table, B.lengths, cu_seqlens=B.cu)
    o = run()
    assert o[0, 0].isnan().all() and torch.equal(o[0, 1].isnan().all(-1), bad[0, 1])


@pytest.mark.parametrize("n,G", [(2, 8), (90, 1)])
@pytest.mark.parametrize("q8", [False, True], ids=["16bit", "8bit"])
def test_infinities_beyond_64_pages(cuda, n, G, q8):
    """Page numbers are held 64 at a time: more pages than that, infinities in the first and the last ones."""
    B = Batch([2500, 5000], heads=2, G=G, D=64, R=32, page=32, q8=q8)
    clean = B.rows(1)[1]
    for b, t in enumerate(B.total):
        B.v[0, :, int(B.cu[b]) + 40, 5], B.v[0, :, int(B.cu[b]) + t - 300, 6] = INF, -INF
    paged_cache_write(B.cache, B.k, B.v, B.emb(B.pos), B.table, B.lengths, cu_seqlens=B.cu)
    pos = B.lengths[:, None].long() - n + torch.arange(n, device="cuda")
    q = B.rand(2, 2 * G, n, 64)
    o = paged_flash_attn_with_pope(q, B.cache, B.emb(pos), B.table, B.lengths)
    for b in range(2):
        k, v = B.rows(b)
        want, _, tol, _ = with_infinities(q[b], angles(pos[b], 32), k, v, 32, 0.125, True, B.dtype)
        got = o[b].double()
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf()) and torch.equal(got[got.isinf()], want[want.isinf()])
        fin = want.isfinite()
        assert ((got - want).abs()[fin] <= tol[fin]).all() and fin.any()
        # 8 bits have no infinity: the values are stored as NaN
        assert o[b, ..., 5].isnan().all() if q8 else (o[b, ..., 5] == INF).all() and (o[b, ..., 6] == -INF).all()
    assert clean.isfinite().all()


@pytest.mark.parametrize("D,R", [(256, 256), (200, 190)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16], ids=["bf16", "fp16"])
@pytest.mark.parametrize("q8", [False, True], ids=["16bit", "8bit"])
def test_widest_rows(cuda, D, R, dtype, q8):
    """More than 384 columns of K_hat: written, read, and attended by single tokens, a few rows, many rows, in parts too."""
    B = Batch([300, 33, 65, 1, 1700], heads=2, G=2, D=D, R=R, dtype=dtype, q8=q8)
    k, v = B.rows(0)
    s = slice(0, 300)
    want = rows64(B.k[0, :, s], angles(B.pos[s], R), B.bias, R)
    assert ((k - want).abs() <= held(want, dtype, q8)).all() and ((v - B.v[0, :, s].double()).abs() <= held(B.v[0, :, s].double(), dtype, q8)).all()
    for causal in (True, False):
        attend_and_check(B, [1] * 5, packed=False, causal=causal)
        attend_and_check(B, [7] * 5, packed=False, causal=causal, head_first=False)
        attend_and_check(B, [17, 1, 5, 0, 3], packed=True, gap=1, causal=causal)
        attend_and_check(B, [299, 33, 64, 1, 200], packed=True, causal=causal)
    if q8:
        return
    B.v[0, :, 60, 3], B.v[0, :, 61, D - 1], B.k[0, :, 100, R - 1] = INF, -INF, -INF   # softplus(-inf) is 0
    paged_cache_write(B.cache, B.k, B.v, B.emb(B.pos), B.table, B.lengths, cu_seqlens=B.cu)
    for n in (1, 40):
        pos = B.lengths[:1, None].long() - n + torch.arange(n, device="cuda")
        q = B.rand(1, 4, n, D)
        o = paged_flash_attn_with_pope(q, B.cache, B.emb(pos), B.table[:1], B.lengths[:1])[0].double()
        k, v = B.rows(0)
        want, _, tol, _ = with_infinities(q[0], angles(pos[0], R), k, v, R, D ** -0.5, True, dtype)
        assert torch.equal(o.isnan(), want.isnan()) and torch.equal(o.isinf(), want.isinf()) and (o[..., 3] == INF).all() and (o[..., D - 1] == -INF).all()
        fin = want.isfinite()
        assert ((o - want).abs()[fin] <= tol[fin]).all() and fin.any()

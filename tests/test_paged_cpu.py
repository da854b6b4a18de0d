"""The paged cache on the CPU: index arithmetic, argument checks, the C ABI's refusals, and the torch computation of
CPU caches against plain 64-bit formulas.

Tolerances: a stored 16-bit value is the rounding of one that fp32 holds to a few ulp (at most 1e-6 relative to the
magnitude softplus(k)), so half a step of the type and that; e4m3 likewise, half a step of the value or of the smallest
normal (2^-6 in units of the row's power of two).  Attention on CPU caches is fp32 arithmetic rounded once.
"""
import ctypes
import math
import os
import subprocess

import pytest
import torch
import torch.nn.functional as F

import pope_amd
from pope_amd import PagedPoPECache, PoPE, _lib, paged, paged_cache_read, paged_cache_write, paged_flash_attn_with_pope

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
I32 = torch.int32


def test_index_arithmetic(tmp_path):
    exe = str(tmp_path / "check")
    subprocess.run(["g++", "-O1", "-std=c++17", "-include", "algorithm", "-I", os.path.join(ROOT, "pope-pytorch_amd", "csrc"),
                    os.path.join(ROOT, "tests", "paged_index_check.cpp"), "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout


def test_plan_of_many_rows(tmp_path):
    """The plan's workgroups on the host: also with descending bounds every part that the join reads has been written."""
    exe = str(tmp_path / "plan")
    subprocess.run(["g++", "-O2", "-std=c++17", "-I", os.path.join(ROOT, "pope-pytorch_amd", "csrc"), os.path.join(ROOT, "tests", "paged_plan_check.cpp"),
                    "-o", exe], check=True)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout


# ---------------------------------------------------------------- C ABI

def _desc(**kw):
    d = _lib.PopePaged()
    base = dict(pages=4, page_size=64, Hk=2, D=64, R=32, dtype=_lib.POPE_BF16, quantized=0, B=2, N=3, table_cols=2, Hq=4, causal=1,
                softmax_scale=0.125, table_sb=2, bias_sh=32)
    for n, v in {**base, **kw}.items():
        setattr(d, n, v)
    return d


@pytest.mark.parametrize("D,R", [(1, 0), (1, 1), (32, 17), (33, 0), (64, 32), (72, 40), (96, 96), (128, 64), (129, 3), (256, 256)])
@pytest.mark.parametrize("q8", [False, True])
def test_cache_bytes(D, R, q8):
    d = _desc(D=D, R=R, quantized=int(q8), pages=3, page_size=128)
    n = (ctypes.c_size_t * 3)()
    assert _lib.lib().pope_paged_cache_bytes(ctypes.byref(d), n) == 0
    c = PagedPoPECache(3, heads=2, dim=D, rotate_dim=R, page_size=128, quantized=q8)
    assert [t.numel() * t.element_size() for t in (c.k_pages, c.v_pages, c.scales)] == list(n)
    assert c.nbytes == sum(n)


_BUF = ctypes.create_string_buffer(1 << 16)
_A = ctypes.c_void_p((ctypes.addressof(_BUF) + 255) // 256 * 256)


@pytest.mark.parametrize("change,needle", [
    (dict(pages=0), "pages"), (dict(Hk=0), "Hk"), (dict(page_size=48), "page size"), (dict(page_size=16), "page size"),
    (dict(page_size=2048), "page size"), (dict(D=0), "head dims"), (dict(D=257), "head dims"), (dict(R=65), "rotate dim"),
    (dict(R=-1), "rotate dim"), (dict(dtype=_lib.POPE_F32), "fp16 or bf16"), (dict(B=0), "B, table_cols"), (dict(N=-1), "N >= 0"),
    (dict(table_cols=0), "table_cols"), (dict(table_cols=1 << 25), "32-bit positions"), (dict(table_sb=-1), "negative"),
    (dict(bias_sh=-1), "negative"),
])
def test_abi_refuses(change, needle):
    L, d = _lib.lib(), _desc(**change)
    for rc in (L.pope_paged_write(ctypes.byref(d), _A, _A, _A, _A, _A, _A, None, _A, _A, None, None),
               L.pope_paged_read(ctypes.byref(d), _A, _A, None, _A, _A, None, _A, _A, None),
               L.pope_paged_attn(ctypes.byref(d), _A, _A, _A, _A, None, _A, _A, None, _A, None, _A, 1 << 14, None)):
        assert rc in (1, 2) and needle in _lib.last_error()


def test_abi_refuses_pointers_strides_and_workspace():
    L, d, B = _lib.lib(), _desc(), ctypes.byref
    off = ctypes.c_void_p(_A.value + 2)
    write = lambda d, **o: L.pope_paged_write(B(d), *[o.get(n, _A) for n in ("k", "v", "freqs", "bias", "kp", "vp", "sc", "table", "len")], None, None)
    for name in ("k", "v", "freqs", "bias", "kp", "vp", "table", "len"):
        assert write(d, **{name: None}) == 1
    assert write(d, kp=off) == 1 and "16-byte" in _lib.last_error()
    assert write(_desc(quantized=1), sc=None) == 1 and "scales" in _lib.last_error()
    d.k_s[1] = -8
    assert write(d) == 1 and "negative" in _lib.last_error()
    d = _desc(Hq=3)
    attn = lambda d, ws=_A, n=1 << 14: L.pope_paged_attn(B(d), _A, _A, _A, _A, None, _A, _A, None, _A, None, ws, n, None)
    assert attn(d) == 1 and "multiple of kv heads" in _lib.last_error()
    d, n = _desc(N=1, table_cols=400), ctypes.c_size_t()
    assert L.pope_paged_workspace_bytes(B(d), 0, B(n)) == 0 and n.value > 1 << 14   # a long cache, few rows: split
    assert attn(d) == 3 and attn(d, None, 0) == 3 and "workspace" in _lib.last_error()
    # no rows: nothing to do, nothing to point at
    d = _desc(N=0)
    assert write(d, k=None, v=None) == 0 and attn(d, None, 0) == 0


@pytest.mark.parametrize("change", [dict(B=1 << 24, N=1), dict(B=1 << 23, N=2, Hk=2, Hq=40), dict(B=1, N=1 << 30, Hq=1, Hk=1)])
def test_abi_refuses_grids_beyond_a_launch(change):
    """A launch has fewer than 2^32 threads, and a tile's first row is a 32-bit number."""
    L, d = _lib.lib(), _desc(**change)
    n = ctypes.c_size_t()
    calls = [lambda: L.pope_paged_write(ctypes.byref(d), _A, _A, _A, _A, _A, _A, None, _A, _A, None, None),
             lambda: L.pope_paged_read(ctypes.byref(d), _A, _A, None, _A, _A, None, _A, _A, None)]
    if d.N < 1 << 30:
        calls += [lambda: L.pope_paged_workspace_bytes(ctypes.byref(d), 0, ctypes.byref(n)), lambda: L.pope_paged_workspace_bytes(ctypes.byref(d), 1, ctypes.byref(n)),
                  lambda: L.pope_paged_attn(ctypes.byref(d), _A, _A, _A, _A, None, _A, _A, None, _A, None, _A, 1 << 14, None)]
    for call in calls:
        assert call() == 2 and "too many workgroups" in _lib.last_error(), _lib.last_error()


# ---------------------------------------------------------------- Python checks

def _call(**kw):
    c = kw.pop("cache", None) or PagedPoPECache(4, heads=2, dim=16, rotate_dim=8, page_size=32)
    a = dict(k=torch.randn(2, 2, 3, 16).bfloat16(), v=torch.randn(2, 2, 3, 16).bfloat16(), q=torch.randn(2, 4, 3, 16).bfloat16(),
             pos_emb=(torch.rand(3, 8), torch.zeros(2, 8)), page_table=torch.tensor([[0, 1], [2, 3]], dtype=I32),
             lengths=torch.tensor([3, 10], dtype=I32), cu_seqlens=None)
    a.update(kw)
    return c, a


def _write(c, a, **kw):
    paged_cache_write(c, a["k"], a["v"], a["pos_emb"], a["page_table"], a["lengths"], cu_seqlens=a["cu_seqlens"], **kw)


def _attend(c, a, **kw):
    return paged_flash_attn_with_pope(a["q"], c, a["pos_emb"], a["page_table"], a["lengths"], cu_seqlens=a["cu_seqlens"], **kw)


@pytest.mark.parametrize("kw", [dict(num_pages=0), dict(heads=0), dict(dim=0), dict(dim=257), dict(rotate_dim=17), dict(rotate_dim=-1),
                                dict(page_size=48), dict(page_size=16), dict(page_size=2048)])
def test_cache_refuses(kw):
    a = dict(num_pages=2, heads=1, dim=16, rotate_dim=0)
    a.update(kw)
    with pytest.raises(ValueError):
        PagedPoPECache(a.pop("num_pages"), **a)
    with pytest.raises(TypeError):
        PagedPoPECache(2, heads=1, dim=16, dtype=torch.float32)


@pytest.mark.parametrize("change,error", [
    (dict(k=torch.zeros(2, 2, 3, 16)), TypeError), (dict(v=torch.zeros(2, 2, 3, 16).half()), TypeError),
    (dict(k=torch.zeros(2, 3, 3, 16).bfloat16()), ValueError), (dict(k=torch.zeros(2, 2, 3, 8).bfloat16()), ValueError),
    (dict(k=torch.zeros(1, 2, 3, 16).bfloat16()), ValueError), (dict(v=torch.zeros(2, 2, 4, 16).bfloat16()), ValueError),
    (dict(k=torch.zeros(2, 2, 16).bfloat16()), ValueError), (dict(pos_emb=None), ValueError),
    (dict(pos_emb=(torch.rand(4, 8), torch.zeros(2, 8))), ValueError), (dict(pos_emb=(torch.rand(3, 6), torch.zeros(2, 6))), ValueError),
    (dict(pos_emb=(torch.rand(3, 3, 8), torch.zeros(2, 8))), ValueError), (dict(pos_emb=(torch.rand(1, 2, 3, 8), torch.zeros(2, 8))), ValueError),
    (dict(pos_emb=(torch.rand(3, 8), torch.zeros(3, 8))), ValueError), (dict(pos_emb=(torch.rand(3, 8), None)), ValueError),
    (dict(page_table=torch.zeros(4, dtype=I32)), ValueError), (dict(page_table=torch.zeros(2, 0, dtype=I32)), ValueError),
    (dict(page_table=torch.zeros(2, 2)), TypeError), (dict(lengths=torch.zeros(3, dtype=I32)), ValueError),
    (dict(lengths=torch.zeros(2)), TypeError), (dict(cu_seqlens=torch.zeros(2, dtype=I32)), ValueError),
    (dict(cu_seqlens=torch.zeros(3, dtype=I32)), ValueError),   # packed rows have batch 1
])
def test_write_refuses(change, error):
    c, a = _call(**change)
    with pytest.raises(error):
        _write(c, a)
    assert not c.k_pages.any() and not c.v_pages.any()


def test_attention_and_read_refuse():
    for change in (dict(q=torch.zeros(2, 3, 3, 16).bfloat16()), dict(q=torch.zeros(2, 4, 3, 8).bfloat16()), dict(q=torch.zeros(3, 4, 3, 16).bfloat16())):
        c, a = _call(**change)
        with pytest.raises(ValueError):
            _attend(c, a)
    c, a = _call()
    with pytest.raises(ValueError):
        paged_cache_read(c, a["page_table"], a["lengths"], -1)
    a["q"].requires_grad_(True)
    with pytest.raises(RuntimeError, match="gradient"):
        _attend(c, a)
    with torch.no_grad():
        _attend(c, a)
    c, a = _call(cache=PagedPoPECache(4, heads=2, dim=16, page_size=32))
    with pytest.raises(ValueError, match="rotate_dim 0"):
        _attend(c, a)


# ---------------------------------------------------------------- the torch computation

def rows64(k, v, freqs, bias, R):
    """K_hat with interleaved pairs, and V, in 64 bits: k, v (heads, n, D), freqs (n, R)."""
    x = k.double()
    th = freqs.double() + bias.double()[:, None, :]
    m = F.softplus(x[..., :R])
    return torch.cat((torch.stack((m * th.cos(), m * th.sin()), -1).flatten(-2), x[..., R:]), -1), v.double()


def held(x, dtype, q8):
    """Half-step bound of what the cache holds of 64-bit rows x."""
    if not q8:
        return x.abs() * torch.finfo(dtype).eps / 2 + 2.0 ** -25
    unit = torch.exp2(torch.ceil(torch.log2(x.abs().amax(-1, keepdim=True).clamp_min(1e-30) / 448)))
    return torch.maximum(x.abs(), unit * 2.0 ** -6) * 2.0 ** -4


CASES = [  # heads, G, D, R, page, dtype, q8
    (2, 1, 16, 8, 32, torch.bfloat16, False), (1, 4, 33, 33, 64, torch.float16, False), (3, 2, 72, 40, 32, torch.bfloat16, True),
    (2, 2, 20, 0, 128, torch.float16, True), (1, 1, 160, 31, 64, torch.bfloat16, False),
]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(x).replace("torch.", "") for x in c))
@pytest.mark.parametrize("packed", [False, True])
def test_cpu_cache_against_formulas(case, packed):
    Hk, G, D, R, page, dtype, q8 = case
    g = torch.Generator().manual_seed(5)
    rnd = lambda *s: torch.randn(*s, generator=g)
    cache = PagedPoPECache(12, heads=Hk, dim=D, rotate_dim=R, page_size=page, dtype=dtype, quantized=q8)
    table = torch.tensor([[7, 2, 9], [4, 11, 0], [3, 5, 1]], dtype=I32)
    bias = -torch.rand(Hk, R, generator=g) * 6
    pope = lambda pos: pos[..., None].float() * 100 ** -(torch.arange(R).float() / max(R, 1))
    total = [0, 0, 0]
    hist = [[], [], []]   # (k_hat, v) pieces in 64 bits, per sequence
    for new in ([5, 40, 0], [30, 1, 2], [1, 1, 1]):
        total = [t + n for t, n in zip(total, new)]
        if packed:
            cu = torch.tensor([0, *torch.tensor(new).cumsum(0)], dtype=I32)
            T = int(cu[-1]) + 2   # two rows behind the last sequence
            pos = torch.zeros(T, dtype=torch.long)
            for b in range(3):
                pos[cu[b]:cu[b + 1]] = torch.arange(total[b] - new[b], total[b])
            at = [(0, slice(int(cu[b]), int(cu[b + 1]))) for b in range(3)]
            N, batch = T, 1
        else:
            N, batch, cu = max(new), 3, None
            pos = torch.tensor(total)[:, None] - N + torch.arange(N)   # shorter sequences: leading rows repeat what they have
            at = [(b, slice(N - new[b], N)) for b in range(3)]
        k, v, q = (rnd(batch, h, N, D).to(dtype) for h in (Hk, Hk, Hk * G))
        freqs = pope(pos)
        if not packed:
            lens = torch.tensor(total, dtype=I32)
            for b in range(3):   # one sequence at a time: a padded call with exactly its rows
                if new[b]:
                    s = at[b][1]
                    paged_cache_write(cache, k[b:b + 1, :, s], v[b:b + 1, :, s], (freqs[b:b + 1, s], bias) if R else None, table[b:b + 1], lens[b:b + 1])
        else:
            lens = torch.tensor(total, dtype=I32)
            paged_cache_write(cache, k, v, (freqs, bias) if R else None, table, lens, cu_seqlens=cu)
        for b in range(3):
            i, s = at[b]
            hist[b].append(rows64(k[i, :, s], v[i, :, s], (freqs[0] if freqs.ndim == 3 and packed else freqs if packed else freqs[b])[s], bias, R))
        # read back
        for b in range(3):
            kh, vv = paged_cache_read(cache, table[b:b + 1], lens[b:b + 1], total[b] + 3)
            assert not kh[0, :, :3].any() and not vv[0, :, :3].any()   # before the first position
            for got, want in ((kh, torch.cat([h[0] for h in hist[b]], 1)), (vv, torch.cat([h[1] for h in hist[b]], 1))):
                assert ((got[0, :, 3:].double() - want).abs() <= held(want, dtype, q8) + 2e-6 * (1 + want.abs())).all()
        # attention over what is held
        for causal in (True, False):
            o, lse = paged_flash_attn_with_pope(q, cache, (freqs, bias) if R else None, table, lens, cu_seqlens=cu, causal=causal,
                                                return_lse=True, softmax_scale=0.3)
            if packed:
                assert not o[:, :, -2:].any() and (lse[:, :, -2:] == -math.inf).all()
            for b in range(3):
                kh, vv = (t[0].double() for t in paged_cache_read(cache, table[b:b + 1], lens[b:b + 1], total[b]))
                i, s = at[b] if packed else (b, slice(0, N))
                n = (s.stop - s.start)
                if n == 0 or total[b] == 0:
                    continue
                f = (freqs if packed else freqs[b])[s] if freqs.ndim == 2 or not packed else freqs[0, s]
                qh, _ = rows64(q[i, :, s], q[i, :, s], f, torch.zeros(1, R), R)
                sc = qh @ kh.repeat(G, 1, 1).transpose(1, 2) * 0.3
                see = torch.arange(total[b]) <= (total[b] - n + torch.arange(n))[:, None] if causal else torch.ones(n, total[b], dtype=torch.bool)
                sc = sc.masked_fill(~see, -math.inf)
                p = torch.softmax(sc, -1).nan_to_num(0.0)
                want = p @ vv.repeat(G, 1, 1)
                err = (o[i, :, s].double() - want).abs()
                assert (err <= torch.finfo(dtype).eps / 2 * want.abs() + 1e-5 + 2.0 ** -25).all()
                assert torch.allclose(lse[i, :, s].double(), torch.logsumexp(sc, -1), atol=1e-4)


def test_bad_pages_and_lengths_on_the_cpu():
    cache = PagedPoPECache(3, heads=1, dim=16, page_size=32)
    k = torch.randn(1, 1, 96, 16).bfloat16()
    table = torch.tensor([[0, -5, 2]], dtype=I32)
    full = torch.tensor([96], dtype=I32)
    paged_cache_write(cache, k, k, None, table, full)
    kh, v = paged_cache_read(cache, table, full, 96)
    assert torch.equal(kh[:, :, :32], k[:, :, :32]) and torch.equal(v[:, :, 64:], k[:, :, 64:]) and not kh[:, :, 32:64].any()
    for bad in ([[0, 3, 2]], [[0, 2 ** 31 - 1, 2]]):
        assert torch.equal(paged_cache_read(cache, torch.tensor(bad, dtype=I32), full, 96)[0], kh)
    assert torch.equal(paged_cache_read(cache, torch.tensor([[0, 2 ** 40, 2]]), full, 96)[0], kh)   # int64, beyond 32 bits
    # keys on the bad page are not seen
    q = torch.randn(1, 1, 1, 16).bfloat16()
    o = paged_flash_attn_with_pope(q, cache, None, table, full)
    seen = torch.cat((k[0, 0, :32], k[0, 0, 64:])).double()
    want = torch.softmax(q[0, 0].double() @ seen.T / 4, -1) @ seen
    assert (o[0, 0].double() - want).abs().max() <= 2e-2
    # lengths beyond the table row are cut to it, negative ones are empty
    assert torch.equal(paged_flash_attn_with_pope(q, cache, None, table, torch.tensor([500], dtype=I32)), o)
    o = paged_flash_attn_with_pope(q, cache, None, table, torch.tensor([-7], dtype=I32), return_lse=True)
    assert not o[0].any() and o[1].item() == -math.inf


def test_rows_not_finite_in_masked_places_on_the_cpu():
    cache = PagedPoPECache(2, heads=1, dim=16, page_size=32)
    k, v = torch.randn(1, 1, 5, 16).bfloat16(), torch.randn(1, 1, 5, 16).bfloat16()
    table, lens = torch.tensor([[1]], dtype=I32), torch.tensor([5], dtype=I32)
    paged_cache_write(cache, k, v, None, table, lens)
    q = torch.randn(1, 1, 5, 16).bfloat16()
    clean = paged_flash_attn_with_pope(q, cache, None, table, lens)
    v[0, 0, 3, 2], k[0, 0, 4, 1] = math.inf, math.nan
    paged_cache_write(cache, k, v, None, table, lens)
    o = paged_flash_attn_with_pope(q, cache, None, table, lens)
    assert torch.equal(o[0, 0, :3], clean[0, 0, :3]) and o[0, 0, 3, 2] == math.inf and o[0, 0, 4].isnan().all()
    assert torch.equal(o[0, 0, 3, 3:], clean[0, 0, 3, 3:])


def test_module_positions_feed_the_cache():
    """pope(positions) of the new rows gives what the whole context's table gives."""
    pope = PoPE(8, heads=2)
    table = torch.tensor([[0, 1]], dtype=I32)
    k, v, q = (torch.randn(1, 2, 40, 16).bfloat16() for _ in range(3))
    a, b = (PagedPoPECache(2, heads=2, dim=16, rotate_dim=8, page_size=32) for _ in range(2))
    with torch.no_grad():
        paged_cache_write(a, k, v, pope(40), table, torch.tensor([40], dtype=I32))
        for lo, hi in ((0, 33), (33, 34), (34, 40)):
            paged_cache_write(b, k[:, :, lo:hi], v[:, :, lo:hi], pope(torch.arange(lo, hi)), table, torch.tensor([hi]))
        assert torch.equal(a.k_pages, b.k_pages) and torch.equal(a.v_pages, b.v_pages)
        o = paged_flash_attn_with_pope(q, a, pope(40), table, torch.tensor([40], dtype=I32))
        ref = pope_amd.flash_attn_with_pope(q.float(), k.float(), v.float(), pos_emb=pope(40), causal=True)
    # a cached key is off by half a bf16 step (2^-9), so scores by about 2^-9 of sum |q k| / 4, the output by twice that
    assert (o.float() - ref).abs().max() <= 6e-2


def test_8_bit_rows_at_the_end_of_their_type_on_the_cpu():
    """e4m3 may round a row's largest values past the type's range; they are read, and averaged, as its largest."""
    for dtype, x in ((torch.float16, 65000.0), (torch.bfloat16, torch.finfo(torch.bfloat16).max)):
        most = torch.finfo(dtype).max
        cache = PagedPoPECache(1, heads=1, dim=8, page_size=32, dtype=dtype, quantized=True)
        v = torch.full((1, 1, 3, 8), x, dtype=dtype)
        v[..., 1::2] *= -1
        table, lens = torch.tensor([[0]], dtype=I32), torch.tensor([3], dtype=I32)
        paged_cache_write(cache, torch.zeros_like(v), v, None, table, lens)
        assert (paged_cache_read(cache, table, lens, 3)[1].abs() == most).all()
        if dtype == torch.float16:
            o = paged_flash_attn_with_pope(torch.zeros_like(v), cache, None, table, lens)
            assert (o.abs() == most).all()


def test_forward_mode_tangents_are_refused():
    import torch.autograd.forward_ad as fwd
    c, a = _call()
    for name in ("q", "k", "v"):
        with fwd.dual_level():
            b = dict(a, **{name: fwd.make_dual(a[name], torch.ones_like(a[name]))})
            for grad in (torch.enable_grad, torch.no_grad):   # no_grad is no word on tangents
                with grad(), pytest.raises(RuntimeError, match="gradient"):
                    (_attend if name == "q" else _write)(c, b)
    with fwd.dual_level():
        f = fwd.make_dual(a["pos_emb"][0], torch.ones(3, 8))
        for call in (_attend, _write):
            with pytest.raises(RuntimeError, match="gradient"):
                call(c, dict(a, pos_emb=(f, a["pos_emb"][1])))
    with pytest.raises(RuntimeError, match="gradient"):
        torch.func.jvp(lambda q: _attend(c, dict(a, q=q)), (a["q"],), (torch.ones_like(a["q"]),))
    with pytest.raises(RuntimeError, match="gradient"):
        torch.func.grad(lambda q: _attend(c, dict(a, q=q)).float().sum())(a["q"])


def test_the_output_of_rows_that_overlap_has_unit_feature_stride():
    """Shapes and strides alone (the kernels write rows of unit feature stride): windows that slide by one element."""
    from torch._subclasses import FakeTensorMode
    c, a = _call()
    q = torch.zeros(2, 4, 3 + 15, dtype=torch.bfloat16).unfold(2, 16, 1)
    assert q.shape == (2, 4, 3, 16) and torch.empty_like(q).stride(-1) != 1
    freqs = a["pos_emb"][0][None]
    with FakeTensorMode() as mode:
        f = lambda t: mode.from_tensor(t).to("cuda") if t is not None else None
        o, _ = paged.paged_attn_op(f(q), f(freqs), f(c.k_pages), f(c.v_pages), f(c.scales), f(a["page_table"]), f(a["lengths"]), None, 32, True, 0.25, False)
    assert o.shape == q.shape and o.stride() == (4 * 3 * 16, 3 * 16, 16, 1)


@pytest.mark.parametrize("causal", [True, False])
def test_rows_whose_keys_all_have_weight_zero_on_the_cpu(causal):
    """Every visible score -inf: as with no key to see, 0 and a log-sum-exp of -inf; a NaN score stays NaN."""
    cache = PagedPoPECache(2, heads=1, dim=16, page_size=32)
    k, v, q = (torch.randn(1, 1, 5, 16).bfloat16() for _ in range(3))
    k[..., 2], q[..., 2] = -math.inf, 1.0
    q[0, 0, 3, 5] = math.nan
    table, lens = torch.tensor([[1]], dtype=I32), torch.tensor([5], dtype=I32)
    paged_cache_write(cache, k, v, None, table, lens)
    o, lse = paged_flash_attn_with_pope(q, cache, None, table, lens, causal=causal, return_lse=True)
    good = torch.tensor([0, 1, 2, 4])
    assert not o[0, 0, good].any() and (lse[0, 0, good] == -math.inf).all() and o[0, 0, 3].isnan().all() and lse[0, 0, 3].isnan()

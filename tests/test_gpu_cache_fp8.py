"""The 8-bit paged cache and the windowed cache with first tokens that stay visible: writing, reading back, attention.

Attention is compared with the definition in 64 bits.  The tolerance is a bound, element by element:

* one rounding of the output: ``u_out |o|`` with u = 2^-8 (bf16) or 2^-11 (fp16);
* the probabilities are rounded to fp16 over 8-bit K/V (u_p = 2^-11) and to the inputs' type otherwise; each of them
  moves the output by at most ``u_p p_j |v_j|``, together ``u_p A`` with ``A = sum_j softmax_j |v_j|``.  fp16 is
  absolute below 2^-14: 2^-25 a key, ``n 2^-25 max|v|``;
* a score is a sum of D products in fp32; with 2^-22 for each term and operation it is off by at most
  ``ds = (D + 8) 2^-22 scale sum_d |q_d| |k_d|``, which changes the output by at most ``2 ds A``;
* exponentials, sums, divisions and the joining of splits in fp32: 2^-16 A.
"""
import math
from types import SimpleNamespace

import pytest
import torch

from flaggems_b200 import _lib, fused, patches

pytestmark = pytest.mark.gpu
DEV = "cuda"
E4M3, E5M2 = torch.float8_e4m3fn, torch.float8_e5m2
NAME = {E4M3: "fp8_e4m3", E5M2: "fp8_e5m2"}
TOP = {E4M3: 448.0, E5M2: 57344.0}
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def quantise(x, s, cache):
    """The definition, with torch's own division and conversion; `s` broadcasts."""
    return (x.float() / s).clamp(-TOP[cache], TOP[cache]).to(cache)


def same(a, b):
    """Equal values; NaN equals NaN."""
    a, b = a.double(), b.double()
    return bool(((a == b) | (a.isnan() & b.isnan())).all())


# ------------------------------------------------------------------------------------------------------ write
@pytest.mark.parametrize("cache", [E4M3, E5M2])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens, heads, dim, page, per_head, layout", [
    (1, 1, 16, 16, False, "dense"), (42, 8, 128, 16, True, "dense"), (42, 8, 128, 16, True, "fused"),
    (7, 3, 80, 8, True, "fused"), (5, 2, 64, 32, False, "uint8"), (9, 3, 24, 5, True, "dense"),
    (11, 2, 72, 16, False, "odd"), (300, 4, 256, 64, True, "hnd"), (13, 2, 128, 1, True, "dense")])
def test_write_is_the_definition(fg, dtype, cache, tokens, heads, dim, page, per_head, layout):
    g = gen(tokens * dim)
    if layout == "fused":
        qkv = randn(g, tokens, 5, heads, dim).to(dtype)
        key, value = qkv[:, 3], qkv[:, 4]
    elif layout == "odd":           # rows that start on no 16-byte boundary
        flat = randn(g, 2, tokens * heads * dim + 1).to(dtype)
        key, value = (flat[i, 1:].view(tokens, heads, dim) for i in range(2))
    else:
        key, value = randn(g, tokens, heads, dim).to(dtype), randn(g, tokens, heads, dim).to(dtype)
    blocks = (2 * tokens + page - 1) // page + 1
    if layout == "hnd":             # [blocks, heads, page, dim] memory, seen as [blocks, page, heads, dim]
        caches = [randn(g, blocks, heads, page, dim).to(cache).permute(0, 2, 1, 3) for _ in range(2)]
    else:
        caches = [randn(g, blocks, page, heads, dim).to(cache) for _ in range(2)]
    n = heads if per_head else 1
    ks, vs = (0.01 + 0.1 * torch.rand(n, generator=g, device=DEV) for _ in range(2))
    slots = torch.randperm(blocks * page, generator=g, device=DEV)[:tokens]
    if tokens > 5:
        slots[2], slots[4], slots[5] = -1, blocks * page, 2 ** 40     # padding, and behind the cache
    want = []
    for x, c, s in ((key, caches[0], ks), (value, caches[1], vs)):
        w = c.double().reshape(-1, heads, dim)
        ok = (slots >= 0) & (slots < blocks * page)
        w[slots[ok]] = quantise(x[ok], s.view(-1, 1), cache).double()
        want.append(w.view(blocks, page, heads, dim))
    given = [c.view(torch.uint8) for c in caches] if layout == "uint8" else caches
    slot_arg = slots.to(torch.int32) if tokens <= 5 else slots
    assert fg.reshape_and_cache_flash(key, value, *given, slot_arg, NAME[cache], ks, vs) is None
    assert same(caches[0], want[0]) and same(caches[1], want[1])


@pytest.mark.parametrize("cache", [E4M3, E5M2])
@pytest.mark.parametrize("dim", [16, 8])          # the packet kernel and the one for single elements
def test_write_every_bf16_value(fg, cache, dim):
    x = torch.arange(65536, dtype=torch.int32, device=DEV).to(torch.int16).view(torch.bfloat16).view(-1, 1, dim)
    slots = torch.arange(x.shape[0], device=DEV)
    for s in (1.0, 0.5, 0.0133, 3.0, 1 / 448, 0.9999999, 1.1754944e-38, 1e-30, 2.0 ** -60, 1e-18, 1e18, 1e30, 3e38, 0.0,
              -0.25, math.inf, math.nan):
        scale = torch.tensor([s], device=DEV)
        kc, vc = (torch.zeros((x.shape[0], 1, 1, dim), dtype=cache, device=DEV) for _ in range(2))
        fg.reshape_and_cache_flash(x, x, kc, vc, slots, NAME[cache], scale, None)
        assert same(kc.view(-1), quantise(x, scale, cache).view(-1)), s
        assert same(vc.view(-1), quantise(x, 1.0, cache).view(-1)), s


@pytest.mark.parametrize("cache", [E4M3, E5M2])
def test_write_quotients_next_to_a_border(fg, cache):
    """fp32 rows at and around the halfway points between neighbouring 8-bit values, for many scales."""
    g = gen(5)
    grid = torch.arange(256, dtype=torch.int32, device=DEV).to(torch.uint8).view(cache).float()
    grid = grid[grid.isfinite()].unique()
    half = ((grid[1:].double() + grid[:-1].double()) / 2).float()
    for _ in range(40):
        s = (torch.rand(1, generator=g, device=DEV) * 4 - 2).exp2() * 10.0 ** (torch.rand(1, generator=g, device=DEV) * 8 - 4)
        x = (half.double() * s.double()).float()
        around = torch.cat([x, torch.nextafter(x, x + 1), torch.nextafter(x, x - 1)])
        n = around.numel() // 16 * 16
        rows = around[:n].view(-1, 1, 16).contiguous()
        kc, vc = (torch.zeros((rows.shape[0], 1, 1, 16), dtype=cache, device=DEV) for _ in range(2))
        fg.reshape_and_cache_flash(rows, rows, kc, vc, torch.arange(rows.shape[0], device=DEV), NAME[cache], s, s)
        assert same(kc.view(-1), quantise(rows, s, cache).view(-1)) and same(vc.view(-1), kc.view(-1))


def test_write_keeps_what_it_did_before(fg):
    """Caches of the rows' own dtype are copied into, whatever the cache dtype's name says."""
    g = gen(1)
    for dtype in (torch.bfloat16, torch.float32):
        key, value = randn(g, 5, 2, 32).to(dtype), randn(g, 5, 2, 32).to(dtype)
        kc, vc = (torch.zeros((4, 8, 2, 32), dtype=dtype, device=DEV) for _ in range(2))
        slots = torch.tensor([3, 9, -1, 30, 0], device=DEV)
        fg.reshape_and_cache_flash(key, value, kc, vc, slots, "fp8", torch.ones(1, device=DEV), None)
        for i, s in enumerate(slots.tolist()):
            if s >= 0:
                assert torch.equal(kc[s // 8, s % 8], key[i]) and torch.equal(vc[s // 8, s % 8], value[i])
    with pytest.raises(RuntimeError, match="share a dtype"):
        fg.reshape_and_cache_flash(key, value, kc.to(E4M3), vc.to(E4M3), slots, "auto", None, None)


def test_write_refusals(fg):
    key = torch.zeros((4, 2, 32), dtype=torch.bfloat16, device=DEV)
    kc = torch.zeros((4, 8, 2, 32), dtype=E4M3, device=DEV)
    slots = torch.arange(4, device=DEV)
    one = torch.ones(1, device=DEV)

    def call(key=key, value=key, kc=kc, vc=None, slots=slots, name="fp8", ks=one, vs=one):
        fg.reshape_and_cache_flash(key, value, kc, kc if vc is None else vc, slots, name, ks, vs)

    for match, kw in [
            ("needs caches of", dict(name="fp8_e5m2")), ("needs caches of", dict(kc=kc.view(torch.int8))),
            ("share a dtype", dict(name="fp8_inc")), ("float32", dict(ks=one.double())),
            ("one for each", dict(vs=torch.ones(3, device=DEV))), ("one for each", dict(ks=torch.ones((2, 2), device=DEV))),
            ("is on cpu", dict(ks=torch.ones(1))), ("do not fit", dict(kc=kc[:, :, :1])),
            ("no more entries", dict(slots=torch.arange(5, device=DEV))),
            ("equal strides", dict(vc=torch.zeros((4, 8, 4, 32), dtype=E4M3, device=DEV)[:, :, ::2])),
            ("densely packed", dict(key=torch.zeros((4, 2, 64), dtype=torch.bfloat16, device=DEV)[..., ::2])),
            ("of one dtype", dict(value=key.half())), ("unsupported dtype", dict(key=key.double(), value=key.double()))]:
        with pytest.raises(RuntimeError, match=match):
            call(**kw)


# ------------------------------------------------------------------------------------------------------ gather
def paged(g, lens, page, heads, dim, cache, scale_k=None, scale_v=None, spare=3):
    """Caches and a table whose pages are in no order; unused pages and the rows behind a sequence's end hold NaN."""
    pages = [(n + page - 1) // page for n in lens]
    total = sum(pages) + spare
    order = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    table = torch.full((len(lens), max(max(pages), 1)), int(order[-1]), dtype=torch.int32, device=DEV)
    caches = [torch.full((total, page, heads, dim), math.nan, device=DEV).to(cache) for _ in range(2)]
    rows = []
    at = 0
    for i, n in enumerate(lens):
        table[i, :pages[i]] = order[at:at + pages[i]]
        at += pages[i]
        pos = torch.arange(n, device=DEV)
        where = (table[i, pos // page].long(), pos % page)
        pair = []
        for c, s in zip(caches, (scale_k, scale_v)):
            x = randn(g, n, heads, dim)
            x = x.to(cache) if s is None else quantise(x, s.view(-1, 1), cache)
            if c.element_size() == 1:
                c.view(torch.uint8)[where] = x.view(torch.uint8)
            else:
                c[where] = x
            pair.append(x)
        rows.append(pair)
    return caches[0], caches[1], table, rows


@pytest.mark.parametrize("cache", [E4M3, E5M2, None])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("lens, heads, dim, page, per_head", [
    ([1], 1, 16, 16, False), ([5, 0, 130, 16, 17, 0], 8, 128, 16, True), ([33, 1, 64], 3, 72, 8, True),
    ([0, 40], 2, 64, 5, False), ([700, 3], 2, 256, 64, True)])
def test_gather(fg, dtype, cache, lens, heads, dim, page, per_head):
    g = gen(sum(lens))
    n = heads if per_head else 1
    ks, vs = ((0.01 + 0.1 * torch.rand(n, generator=g, device=DEV)) if cache else None for _ in range(2))
    kc, vc, table, rows = paged(g, lens, page, heads, dim, cache or dtype, ks, vs)
    behind, before = 5, 2
    for starts in (None, [n // 3 for n in lens]):
        got_lens = [m - (starts[i] if starts else 0) for i, m in enumerate(lens)]
        cu = torch.tensor([before] + got_lens, dtype=torch.int32, device=DEV).cumsum(0, dtype=torch.int32)
        key, value = (torch.full((sum(got_lens) + before + behind, heads, dim), 7.0, dtype=dtype, device=DEV) for _ in range(2))
        st = torch.tensor(starts, dtype=torch.int32, device=DEV) if starts else None
        out = fg.gather_cache_flash(kc, vc, key, value, table, cu, NAME[cache] if cache else "auto", ks, vs, st)
        assert out[0] is key and out[1] is value
        for t, which, s in ((key, 0, ks), (value, 1, vs)):
            assert (t[:before] == 7.0).all() and (t[before + sum(got_lens):] == 7.0).all()
            for b, m in enumerate(got_lens):
                want = rows[b][which][lens[b] - m:]
                if cache:
                    want = (want.float() * s.view(-1, 1)).to(dtype)
                assert torch.equal(t[cu[b]:cu[b + 1]], want)


def test_gather_strided_outputs_and_bad_pages(fg):
    g = gen(3)
    one = torch.ones(1, device=DEV)
    kc, vc, table, rows = paged(g, [50, 20], 16, 2, 32, E4M3, one, one)
    cu = torch.tensor([0, 50, 70], dtype=torch.int32, device=DEV)
    both = torch.full((70, 2, 2, 32), 7.0, dtype=torch.bfloat16, device=DEV)
    fg.gather_cache_flash(kc, vc, both[:, 0], both[:, 1], table, cu, "fp8")
    for which in range(2):
        assert torch.equal(both[:, which], torch.cat([r[which].to(torch.bfloat16) for r in rows]))
    # page numbers outside the cache, and rows behind the table's last page, read some page of the cache and fault nothing
    bad = table.clone()
    bad[0, 1], bad[1, 0] = 10 ** 6, -5
    key, value = (torch.zeros((300, 2, 32), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    far = torch.tensor([0, 200, 300], dtype=torch.int32, device=DEV)
    fg.gather_cache_flash(kc, vc, key, value, bad, far, "fp8", seq_starts=torch.tensor([-7, 10 ** 9], dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()


def test_gather_refusals(fg):
    kc = torch.zeros((4, 8, 2, 32), dtype=E4M3, device=DEV)
    key = torch.zeros((10, 2, 32), dtype=torch.bfloat16, device=DEV)
    table = torch.zeros((1, 4), dtype=torch.int32, device=DEV)
    cu = torch.tensor([0, 10], dtype=torch.int32, device=DEV)

    def call(kc=kc, key=key, value=None, table=table, cu=cu, name="fp8", **kw):
        fg.gather_cache_flash(kc, kc, key, key.clone() if value is None else value, table, cu, name, **kw)

    call()
    for match, kw in [
            ("unknown kv_cache_dtype", dict(name="int8")), ("needs caches of", dict(name="fp8_e5m2")),
            ("share a dtype", dict(name="auto")), ("do not fit", dict(key=key[:, :1], value=key[:, :1])),
            ("block_table", dict(table=table.long())), ("cu_seqlens", dict(cu=cu.long())), ("cu_seqlens", dict(cu=cu[:1])),
            ("seq_starts", dict(seq_starts=cu)), ("overlap", dict(key=key[:1].expand(10, 2, 32))),
            ("k_scale", dict(k_scale=torch.ones(3, device=DEV))), ("unsupported dtype", dict(key=key.double(), value=key.double()))]:
        with pytest.raises(RuntimeError, match=match):
            call(**kw)


# ------------------------------------------------------------------------------------------------------ attention
def attention(q_lens, k_lens, q, rows, ks, vs, scale, causal, window, sinks, softcap, dtype, cache):
    """Definition in 64 bits over each sequence's own rows: (out, lse, and the largest error allowed of each)."""
    total, heads, dim = q.shape
    out = torch.zeros((total, heads, dim), dtype=torch.float64, device=DEV)
    tol = torch.zeros_like(out)
    lse = torch.full((heads, total), math.inf, dtype=torch.float64, device=DEV)
    lse_tol = torch.zeros_like(lse)
    at = 0
    u_p = 2.0 ** -11 if cache in TOP else U[dtype]
    for b, (n, m) in enumerate(zip(q_lens, k_lens)):
        if n == 0 or m == 0:
            at += n
            continue
        hk = rows[b][0].shape[1]
        k, v = rows[b][0].double() * ks[b].view(-1, 1), rows[b][1].double() * vs[b].view(-1, 1)
        p = torch.arange(n, device=DEV).view(-1, 1) + m - n
        j = torch.arange(m, device=DEV).view(1, -1)
        seen = torch.ones((n, m), dtype=torch.bool, device=DEV)
        if causal:
            seen &= j <= p
        elif window[1] >= 0:
            seen &= j <= p + window[1]
        if window[0] >= 0:
            seen &= (j >= p - window[0]) | (j < sinks)
        for h in range(heads):
            kk, vv = k[:, h // (heads // hk)], v[:, h // (heads // hk)]
            qq = q[at:at + n, h].double()
            a = qq @ kk.T * scale
            if softcap:
                a = softcap * torch.tanh(a / softcap)
            a = a.masked_fill(~seen, -math.inf)
            some = seen.any(-1)
            w = torch.softmax(a[some], -1)
            ref = w @ vv
            size = w @ vv.abs()
            ds = (dim + 8) * 2.0 ** -22 * scale * (qq[some].abs() @ kk.abs().T).masked_fill(~seen[some], 0).amax(-1)
            rows_at = torch.nonzero(some).flatten() + at
            out[rows_at, h] = ref
            few = m * 2.0 ** -25 * (vv.abs().max() if m else 0)
            tol[rows_at, h] = U[dtype] * ref.abs() + (u_p + 2 * ds.view(-1, 1) + 2.0 ** -16) * size + few + 1e-30
            lse[h, rows_at] = torch.logsumexp(a[some], -1)
            lse_tol[h, rows_at] = 2 * ds + 2.0 ** -16 * (1 + lse[h, rows_at].abs())
        at += n
    return out, lse, tol, lse_tol


def check(fg, q_lens, k_lens, heads, hk, dim, page, dtype, cache, causal=True, window=(-1, -1), sinks=0, softcap=0.0,
          scale_shape="one", seed=0, behind=3, contiguous=False, spread=1.0, bound=0):
    """`bound`: max_seqlen_k that the call is given, where it is not the longest sequence."""
    bound = bound or max(k_lens)
    g = gen(seed + sum(k_lens) + dim)
    eight = cache in TOP
    batch = len(k_lens)
    ks = vs = None
    if eight:
        n = 1 if scale_shape == "one" else hk
        ks, vs = ((4.5 / TOP[cache]) * (0.5 + torch.rand(n, generator=g, device=DEV)) for _ in range(2))
    if contiguous:
        rows = [[(quantise(randn(g, m, hk, dim), s.view(-1, 1), cache) if eight else randn(g, m, hk, dim).to(cache))
                 for s in (ks, vs)] for m in k_lens]
        kc, vc = (torch.cat([r[i].view(torch.uint8) if eight else r[i] for r in rows]).view(cache) for i in range(2))
        where = dict(cu_seqlens_k=torch.tensor([0] + k_lens, device=DEV).cumsum(0, dtype=torch.int32))
    else:
        kc, vc, table, rows = paged(g, k_lens, page, hk, dim, cache, ks, vs)
        where = dict(seqused_k=torch.tensor(k_lens, dtype=torch.int32, device=DEV), block_table=table)
        if window[0] >= 0:      # pages and rows that no query sees hold anything: here NaN
            for b, (n, m) in enumerate(zip(q_lens, k_lens)):
                j = torch.arange(min(sinks, m), max(min(sinks, m), m - n - window[0]), device=DEV)
                for c in (kc, vc):
                    c = c.view(torch.uint8) if eight else c
                    c[table[b, j // page].long(), j % page] = 0x7f if eight else math.nan
    total = sum(q_lens)
    q = (spread * randn(g, total + behind, heads, dim)).to(dtype)
    cu = torch.tensor([0] + q_lens, device=DEV).cumsum(0, dtype=torch.int32)
    descale = {}
    if eight:
        wide = (lambda s: s.view(1, -1).expand(batch, hk)) if scale_shape == "batch" else (lambda s: s)
        descale = dict(k_descale=wide(ks), v_descale=wide(vs))
    out = torch.full((total + behind, heads, dim), 7.0, dtype=dtype, device=DEV)
    got, lse = fg.flash_attn_varlen_func(
        q, kc, vc, max(q_lens), cu, bound, softmax_scale=dim ** -0.5, causal=causal, window_size=window,
        softcap=softcap, sink_tokens=sinks, out=out, return_softmax_lse=True, **where, **descale)
    assert got is out and (out[total:] == 7.0).all()
    one = torch.ones(1, device=DEV)
    want, wlse, tol, lse_tol = attention(
        q_lens, k_lens, q[:total], rows, [ks if eight else one] * batch, [vs if eight else one] * batch, dim ** -0.5,
        causal, window, sinks, softcap, dtype, cache)
    err = (out[:total].double() - want).abs()
    worst = (err / tol.clamp(min=1e-30)).max().item()
    assert out[:total].isfinite().all() and worst <= 1.0, f"error {worst:.3g} of the bound"
    lse = lse[:, :total].double()
    empty = wlse == math.inf
    assert (lse[empty] == math.inf).all()
    assert ((lse[~empty] - wlse[~empty]).abs() <= lse_tol[~empty]).all()
    again = fg.flash_attn_varlen_func(
        q, kc, vc, max(q_lens), cu, bound, softmax_scale=dim ** -0.5, causal=causal, window_size=window,
        softcap=softcap, sink_tokens=sinks, out=torch.full_like(out, 7.0), **where, **descale)
    assert torch.equal(again, out)          # the same inputs, the same bits


HEADS = [(4, 4), (8, 2), (7, 1), (32, 8), (48, 2)]


@pytest.mark.parametrize("dtype, cache", [(torch.bfloat16, E4M3), (torch.float16, E4M3), (torch.bfloat16, E5M2),
                                          (torch.float16, E5M2)])
@pytest.mark.parametrize("dim", [64, 128, 256, 96, 40])
@pytest.mark.parametrize("heads, hk", HEADS)
def test_fp8_decode(fg, dtype, cache, dim, heads, hk):
    check(fg, [1] * 6, [1, 17, 64, 463, 1328, 129], heads, hk, dim, 16, dtype, cache, scale_shape="heads")


@pytest.mark.parametrize("cache", [E4M3, torch.bfloat16])
@pytest.mark.parametrize("heads, hk, tokens", [(7, 1, 1), (16, 1, 1), (4, 1, 4), (4, 4, 1), (4, 1, 40)])
def test_many_long_sequences(fg, cache, heads, hk, tokens):
    """Runs of tiles that are cut in the middle of sequences, with waits long enough to look at the abort flag."""
    lens = [2000 + (i * 997) % 3000 for i in range(48)]
    window = (-1, -1) if cache in TOP else (4500, 0)
    check(fg, [tokens] * 48, lens, heads, hk, 128, 16, torch.bfloat16, cache, window=window, sinks=4, scale_shape="heads")


@pytest.mark.parametrize("dtype, cache", [(torch.bfloat16, E4M3), (torch.float16, E5M2)])
@pytest.mark.parametrize("dim", [64, 128, 256, 72])
@pytest.mark.parametrize("heads, hk", HEADS)
def test_fp8_chunk(fg, dtype, cache, dim, heads, hk):
    check(fg, [1, 5, 129, 64, 3, 33], [1328, 18, 463, 64, 3, 700], heads, hk, dim, 16, dtype, cache, scale_shape="batch")


@pytest.mark.parametrize("page", [1, 8, 16, 24, 64, 128, 256])
@pytest.mark.parametrize("q_lens", [[1, 1, 1], [40, 7, 130], [2, 3, 4]])
def test_fp8_page_sizes(fg, page, q_lens):
    check(fg, q_lens, [300, 77, 515], 8, 2, 128, page, torch.bfloat16, E4M3)


@pytest.mark.parametrize("cache", [torch.bfloat16, E4M3])
@pytest.mark.parametrize("window, sinks", [((0, 0), 1), ((5, 0), 4), ((63, 0), 4), ((64, 0), 64), ((100, 0), 130),
                                           ((1000, 0), 4), ((31, 0), 0)])
@pytest.mark.parametrize("q_lens, k_lens", [
    ([1, 1, 1, 1], [1, 64, 700, 2100]), ([3, 4, 1, 2], [3, 500, 900, 66]), ([200, 70, 1, 300], [200, 500, 900, 1500])])
@pytest.mark.parametrize("dim", [128, 64])
def test_window_with_first_tokens(fg, cache, window, sinks, q_lens, k_lens, dim):
    if cache == torch.bfloat16 and sinks == 0:
        pytest.skip("a window alone over a 16-bit cache is covered elsewhere")
    check(fg, q_lens, k_lens, 8, 2, dim, 16, torch.bfloat16, cache, window=window, sinks=sinks)


@pytest.mark.parametrize("cache", [torch.float16, E5M2])
@pytest.mark.parametrize("kw", [
    dict(causal=False), dict(causal=False, window=(20, 15), sinks=6), dict(causal=False, window=(-1, 3)),
    dict(softcap=20.0, window=(90, 0), sinks=3), dict(causal=True, window=(40, 0), sinks=5, contiguous=True),
    dict(contiguous=True, causal=True, window=(2000, 0), sinks=1)])
@pytest.mark.parametrize("q_lens", [[1, 1, 1], [65, 130, 2]])
def test_other_masks_and_layouts(fg, cache, kw, q_lens):
    if cache == torch.float16 and not (kw.get("sinks") and kw.get("window", (-1,))[0] >= 0):
        pytest.skip("not this path")
    check(fg, q_lens, [300, 130, 515], 4, 2, 128, 16, torch.float16, cache, **kw)


@pytest.mark.parametrize("dim", [128, 64])
def test_rows_that_see_nothing_and_empty_sequences(fg, dim):
    # more new tokens than keys: the first rows see no key; sequences without keys or without new tokens
    check(fg, [9, 0, 4, 1, 140], [3, 50, 0, 0, 100], 8, 2, dim, 16, torch.bfloat16, E4M3)
    check(fg, [1, 0, 1, 1], [3, 50, 0, 700], 8, 2, dim, 16, torch.bfloat16, E4M3)
    check(fg, [9, 0, 4, 1, 140], [3, 50, 0, 0, 100], 8, 2, dim, 16, torch.bfloat16, torch.bfloat16, window=(7, 0), sinks=2)


@pytest.mark.parametrize("spread", [1e-30, 1e-4, 1e3])
def test_query_magnitudes(fg, spread):
    """bf16 queries beyond fp16's range: the power of two taken out of each row brings them there and back."""
    for q_lens in ([1, 1], [130, 3]):
        check(fg, q_lens, [200, 90], 8, 2, 128, 16, torch.bfloat16, E4M3, spread=spread)


@pytest.mark.parametrize("bound", [190, 10 ** 6])
def test_long_context_offsets(fg, bound):
    """A cache of more than 2^32 bytes: the last pages are used."""
    page, hk, dim = 64, 8, 128
    blocks = (2 ** 32 + 2 ** 28) // (page * hk * dim)
    g = gen(2)
    kc, vc = (torch.zeros((blocks, page, hk, dim), dtype=E4M3, device=DEV) for _ in range(2))
    lens = [190, 70]
    table = torch.tensor([[blocks - 1, 5, blocks - 3], [blocks - 2, blocks - 4, 0]], dtype=torch.int32, device=DEV)
    scale = torch.tensor([0.01], device=DEV)
    rows = []
    for b, n in enumerate(lens):
        x = [randn(g, n, hk, dim).to(torch.bfloat16) for _ in range(2)]
        pos = torch.arange(n, device=DEV)
        slots = table[b, pos // page].long() * page + pos % page
        fg.reshape_and_cache_flash(*x, kc, vc, slots, "fp8", scale, scale)
        rows.append([quantise(t, scale, E4M3) for t in x])
    key, value = (torch.empty((sum(lens), hk, dim), device=DEV) for _ in range(2))
    cu_k = torch.tensor([0, 190, 260], dtype=torch.int32, device=DEV)
    fg.gather_cache_flash(kc, vc, key, value, table, cu_k, "fp8", scale, scale)
    assert torch.equal(key, torch.cat([r[0].float() * scale for r in rows]))
    assert torch.equal(value, torch.cat([r[1].float() * scale for r in rows]))
    for q_lens in ([1, 1], [100, 3]):
        q = randn(g, sum(q_lens), 32, dim).to(torch.bfloat16)
        cu = torch.tensor([0] + q_lens, device=DEV).cumsum(0, dtype=torch.int32)
        out = fg.flash_attn_varlen_func(
            q, kc, vc, max(q_lens), cu, bound, seqused_k=torch.tensor(lens, dtype=torch.int32, device=DEV), causal=True,
            block_table=table, k_descale=scale, v_descale=scale)
        want, _, tol, _ = attention(q_lens, lens, q, rows, [scale] * 2, [scale] * 2, dim ** -0.5, True, (-1, -1), 0, 0.0,
                                    torch.bfloat16, E4M3)
        assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("bound", [100, 10 ** 6])
def test_nan_that_a_query_sees_reaches_its_row(fg, bound):
    page, hk, dim = 16, 2, 128
    g = gen(4)
    one = torch.ones(1, device=DEV)
    for q_lens in ([1, 1], [70, 20]):
        kc, vc, table, rows = paged(g, [100, 60], page, hk, dim, E4M3, one, one)
        kc.view(torch.uint8)[table[0, 0].long(), 3, 0] = 0x7f          # a key of sequence 0, head 0
        cu = torch.tensor([0] + q_lens, device=DEV).cumsum(0, dtype=torch.int32)
        q = randn(g, sum(q_lens), 4, dim).to(torch.bfloat16)
        out, lse = fg.flash_attn_varlen_func(
            q, kc, vc, max(q_lens), cu, bound, seqused_k=torch.tensor([100, 60], dtype=torch.int32, device=DEV), causal=True,
            block_table=table, return_softmax_lse=True)
        n = q_lens[0]
        assert out[:n, :2].isnan().all() and out[:n, 2:].isfinite().all() and out[n:].isfinite().all()
        assert lse[:2, :n].isnan().all() and lse[2:].isfinite().all()


def test_strided_tensors_and_out_views(fg):
    """q and out as slices of wider buffers, a block table with spare columns, caches interleaved as one tensor."""
    g = gen(6)
    page, hk, heads, dim = 16, 2, 8, 128
    lens, q_lens = [200, 45], [1, 1]
    scale = torch.tensor([0.01], device=DEV)
    kc0, vc0, table, rows = paged(g, lens, page, hk, dim, E4M3, scale, scale)
    both = torch.stack([kc0.view(torch.uint8), vc0.view(torch.uint8)], 1).view(E4M3)     # [blocks, 2, page, hk, dim]
    wide = torch.zeros((2, table.shape[1] + 5), dtype=torch.int32, device=DEV)
    wide[:, :table.shape[1]] = table
    for q_lens in ([1, 1], [100, 30]):
        qkv = randn(g, sum(q_lens), heads + 4, dim).to(torch.bfloat16)
        hold = torch.full((sum(q_lens), heads + 2, dim), 7.0, dtype=torch.bfloat16, device=DEV)
        cu = torch.tensor([0] + q_lens, device=DEV).cumsum(0, dtype=torch.int32)
        fg.flash_attn_varlen_func(
            qkv[:, 2:2 + heads], both[:, 0], both[:, 1], max(q_lens), cu, 200, causal=True, out=hold[:, 1:-1],
            seqused_k=torch.tensor(lens, dtype=torch.int32, device=DEV), block_table=wide[:, :table.shape[1]],
            k_descale=scale, v_descale=scale)
        want, _, tol, _ = attention(q_lens, lens, qkv[:, 2:2 + heads], rows, [scale] * 2, [scale] * 2, dim ** -0.5, True,
                                    (-1, -1), 0, 0.0, torch.bfloat16, E4M3)
        assert ((hold[:, 1:-1].double() - want).abs() <= tol).all()
        assert (hold[:, 0] == 7.0).all() and (hold[:, -1] == 7.0).all()


@pytest.mark.parametrize("bound", [2000, 10 ** 6])
def test_two_captured_graphs_and_another_stream(fg, bound):
    """Write, attend and read back captured in two graphs, replayed at the same time on two streams."""
    g = gen(7)
    page, hk, heads, dim, batch = 16, 8, 32, 128, 6
    lens = [1500, 40, 900, 2000, 17, 640]
    scale = torch.tensor([0.012], device=DEV)
    runs = []
    for seed in range(2):
        kc, vc, table, rows = paged(g, lens, page, hk, dim, E4M3, scale, scale)
        s = dict(kc=kc, vc=vc, table=table, q=randn(g, batch, heads, dim).to(torch.bfloat16),
                 new=randn(g, batch, 2, hk, dim).to(torch.bfloat16), cu=torch.arange(batch + 1, dtype=torch.int32, device=DEV),
                 lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
        last = torch.tensor(lens, device=DEV) - 1
        s["slots"] = table[torch.arange(batch, device=DEV), last // page].long() * page + last % page
        s["cu_k"] = torch.tensor([0] + lens, device=DEV).cumsum(0, dtype=torch.int32)
        s["rows"] = [torch.zeros((sum(lens), hk, dim), dtype=torch.bfloat16, device=DEV) for _ in range(2)]
        runs.append(s)

    def step(s):
        fg.reshape_and_cache_flash(s["new"][:, 0], s["new"][:, 1], s["kc"], s["vc"], s["slots"], "fp8", scale, scale)
        fg.gather_cache_flash(s["kc"], s["vc"], *s["rows"], s["table"], s["cu_k"], "fp8", scale, scale)
        return fg.flash_attn_varlen_func(s["q"], s["kc"], s["vc"], 1, s["cu"], bound, seqused_k=s["lens"], causal=True,
                                         block_table=s["table"], k_descale=scale, v_descale=scale)

    eager = [step(s).clone() for s in runs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in runs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(s))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for o in outs:
            o.fill_(7.0)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for o, e in zip(outs, eager):
            assert torch.equal(o, e)
    # and without a graph, on another stream than the one that made the tensors
    with torch.cuda.stream(streams[0]):
        out = step(runs[0])
    torch.cuda.synchronize()
    assert torch.equal(out, eager[0])
    for s in runs:        # a run of them together: what was written is what is read back
        for i, which in enumerate((0, 1)):
            want = (quantise(s["new"][:, which], scale, E4M3).float() * scale).to(torch.bfloat16)
            assert torch.equal(s["rows"][i][s["cu_k"][1:].long() - 1], want)


@pytest.mark.parametrize("dtype, cache", [(torch.bfloat16, E4M3), (torch.float16, E4M3), (torch.bfloat16, E5M2), (torch.float16, E5M2)])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads, hk, tokens", [(4, 4, 1), (8, 2, 1), (7, 1, 1), (4, 1, 4), (48, 3, 1)])
def test_fp8_decode_with_a_large_bound(fg, dtype, cache, dim, heads, hk, tokens):
    """Enough keys, by max_seqlen_k, for the kernels that walk long contexts."""
    check(fg, [tokens] * 6, [tokens, 17, 64, 463, 1328, 129], heads, hk, dim, 16, dtype, cache, scale_shape="batch", bound=200000)
    check(fg, [tokens, 0, tokens, 1], [3, 50, 0, 700], heads, hk, dim, 64, dtype, cache, causal=False, window=(-1, 3), bound=400000)


@pytest.mark.parametrize("page", [8, 16, 32, 64, 128, 256])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_decode_with_a_large_bound_by_page_size(fg, page, dim):
    check(fg, [1, 1, 1], [300, 77, 515], 8, 2, dim, page, torch.bfloat16, E4M3, bound=10 ** 6)
    check(fg, [1, 1, 0], [300, 77, 515], 16, 1, dim, page, torch.float16, E5M2, bound=10 ** 6, contiguous=True)
    check(fg, [2, 1], [300, 1], 8, 2, dim, page, torch.bfloat16, E4M3, bound=10 ** 6, spread=1e-30)


@pytest.mark.parametrize("dtype, cache", [(torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16), (torch.bfloat16, E4M3),
                                          (torch.float16, E5M2)])
@pytest.mark.parametrize("dim", [64, 256])
@pytest.mark.parametrize("window, sinks", [((100, 0), 130), ((1000, 0), 4), ((30, 0), 1)])
def test_windowed_chunks_at_other_head_dims(fg, dtype, cache, dim, window, sinks):
    check(fg, [200, 70, 1, 300], [200, 500, 900, 1500], 16, 4, dim, 16, dtype, cache, window=window, sinks=sinks)
    check(fg, [20, 7, 9], [2000, 500, 9], 4, 4, dim, 64, dtype, cache, window=window, sinks=sinks)


@pytest.mark.parametrize("cache", [torch.bfloat16, torch.float16, E4M3])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("window, sinks", [((100, 0), 130), ((31, 0), 4), ((0, 0), 1)])
@pytest.mark.parametrize("heads, hk, batch", [(16, 4, 64), (56, 8, 64), (48, 3, 270)])
def test_windowed_decode_of_many_sequences(fg, cache, dim, window, sinks, heads, hk, batch):
    if (dim, cache) in ((256, torch.bfloat16), (256, torch.float16)) or (batch == 270 and (window[0] != 100 or dim == 64)):
        pytest.skip("not this kernel")
    dtype = torch.bfloat16 if cache == E4M3 else cache
    check(fg, [1] * batch, [1 + (i * 61) % 900 for i in range(batch)], heads, hk, dim, 16, dtype, cache, window=window, sinks=sinks)


def test_large_groups_many_sequences_and_nothing_cached(fg):
    # more heads of a group than a tile of the general kernel has rows, and than one of the tensor-core kernel has
    check(fg, [3, 1, 40], [90, 5, 300], 72, 1, 128, 16, torch.bfloat16, E4M3)
    check(fg, [2, 1], [90, 5], 160, 1, 128, 16, torch.bfloat16, E4M3)
    check(fg, [3, 1], [90, 5], 80, 1, 64, 16, torch.float16, E4M3)
    # more sequences than a block has threads
    lens = [1 + (i * 37) % 150 for i in range(600)]
    check(fg, [1] * 600, lens, 4, 2, 128, 16, torch.bfloat16, E4M3)
    check(fg, [i % 3 + (i == 7) * 30 for i in range(600)], lens, 4, 2, 128, 16, torch.bfloat16, torch.bfloat16, window=(60, 0), sinks=4)
    # nothing cached at all
    for cache, dim in ((E4M3, 128), (torch.bfloat16, 128), (E4M3, 64)):
        for q_lens in ([1, 1], [30, 200]):
            check(fg, q_lens, [0, 0], 4, 2, dim, 16, torch.bfloat16, cache, window=(9, 0), sinks=2)


@pytest.mark.parametrize("window", [(-1, -1), (200, 0)])
@pytest.mark.parametrize("contiguous", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_long_chunks_over_an_8_bit_store(fg, dtype, contiguous, window):
    """Chunks that are long enough for the store to be widened ahead of the attention."""
    check(fg, [600, 1, 0, 130], [900, 700, 33, 130], 8, 4, 128, 16, dtype, E4M3, window=window, sinks=3, contiguous=contiguous,
          scale_shape="one" if contiguous else "batch")


@pytest.mark.parametrize("cache", [E4M3, torch.bfloat16])
@pytest.mark.parametrize("q_lens", [[1, 1, 1], [40, 3, 130]])
def test_without_a_workspace(fg, monkeypatch, cache, q_lens):
    monkeypatch.setattr(_lib.load(), "fg_flash_attn_cache_workspace_bytes", lambda params: 0)
    for dim in (128, 64):
        check(fg, q_lens, [3000, 77, 515], 8, 2, dim, 16, torch.bfloat16, cache, window=(2500, 0), sinks=4)


@pytest.mark.parametrize("paged_store", [True, False])
@pytest.mark.parametrize("dim", [128, 64])
@pytest.mark.parametrize("q_len", [1, 40])
def test_lengths_that_contradict_the_call_are_cut(fg, q_len, dim, paged_store):
    """More keys than max_seqlen_k, and rows behind q or K/V: the results are those of the lengths cut to what there is."""
    g = gen(11)
    heads, hk = 8, 2
    q = randn(g, 2 * q_len, heads, dim).to(torch.bfloat16)
    cu = torch.tensor([0, q_len, 2 * q_len], dtype=torch.int32, device=DEV)
    kc, vc, table, _ = paged(g, [200, 150], 16, hk, dim, E4M3, torch.ones(1, device=DEV), torch.ones(1, device=DEV))
    flat = [torch.randint(0, 100, (350, hk, dim), generator=g, device=DEV, dtype=torch.uint8).view(E4M3) for _ in range(2)]

    def run(cu_q, lens, max_k):
        lens = torch.tensor(lens, dtype=torch.int32, device=DEV)
        out = torch.full_like(q, 7.0)
        if paged_store:
            return fg.flash_attn_varlen_func(q, kc, vc, q_len, cu_q, max_k, seqused_k=lens, causal=True, block_table=table, out=out)
        cu_k = torch.cat([lens.new_zeros(1), lens.cumsum(0, dtype=torch.int32)])
        return fg.flash_attn_varlen_func(q, *flat, q_len, cu_q, max_k, cu_seqlens_k=cu_k, causal=True, out=out)

    assert torch.equal(run(cu, [200, 10 ** 8], 200)[:q_len], run(cu, [200, 150], 200)[:q_len])
    far = torch.tensor([0, q_len, 10 ** 9], dtype=torch.int32, device=DEV)
    assert torch.equal(run(far, [200, 150], 200)[:q_len], run(cu, [200, 150], 200)[:q_len])
    run(torch.tensor([0, 10 ** 8, 2 * 10 ** 8], dtype=torch.int32, device=DEV), [2 * 10 ** 9, 50], 200)
    run(torch.tensor([-5, 10, 3], dtype=torch.int32, device=DEV), [-4, 50], 200)
    torch.cuda.synchronize()


@pytest.mark.parametrize("form", ["short", "long", "windowed"])
def test_chunks_in_two_captured_graphs(fg, form):
    g = gen(12)
    page, hk, heads, dim = 16, 2, 8, 128
    cache = torch.bfloat16 if form == "windowed" else E4M3
    q_lens, lens = ([400, 3], [1500, 900]) if form == "long" else ([30, 3], [1500, 900])
    scale = torch.tensor([0.012], device=DEV)
    kw = dict(window_size=(300, 0), sink_tokens=4) if form == "windowed" else dict(k_descale=scale, v_descale=scale)
    eight = None if form == "windowed" else scale
    runs = []
    for _ in range(2):
        kc, vc, table, _ = paged(g, lens, page, hk, dim, cache, eight, eight)
        runs.append((randn(g, sum(q_lens), heads, dim).to(torch.bfloat16), kc, vc, max(q_lens),
                     torch.tensor([0] + q_lens, device=DEV).cumsum(0, dtype=torch.int32), max(lens), table,
                     torch.tensor(lens, dtype=torch.int32, device=DEV)))

    def step(r):
        return fg.flash_attn_varlen_func(*r[:6], seqused_k=r[7], causal=True, block_table=r[6], **kw)

    eager = [step(r).clone() for r in runs]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for r in runs:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(r))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for o in outs:
            o.fill_(7.0)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for o, e in zip(outs, eager):
            assert torch.equal(o, e)


def test_attention_refusals(fg):
    kc = torch.zeros((4, 16, 2, 64), dtype=E4M3, device=DEV)
    q = torch.zeros((2, 4, 64), dtype=torch.bfloat16, device=DEV)
    cu = torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV)
    lens = torch.tensor([5, 6], dtype=torch.int32, device=DEV)
    table = torch.zeros((2, 1), dtype=torch.int32, device=DEV)
    one = torch.ones(1, device=DEV)

    def call(q=q, kc=kc, vc=None, cu=cu, lens=lens, table=table, **kw):
        return fg.flash_attn_varlen_func(q, kc, kc if vc is None else vc, 1, cu, 6, seqused_k=lens, causal=True,
                                         block_table=table, **kw)

    call()
    for match, kw in [
            ("float32", dict(k_descale=one.half())), ("one element or the shape", dict(v_descale=torch.ones(3, device=DEV))),
            ("ALiBi", dict(alibi_slopes=torch.ones(4, device=DEV))), ("must not be negative", dict(sink_tokens=-1)),
            ("ALiBi", dict(kc=kc.bfloat16(), vc=kc.bfloat16(), sink_tokens=2, window_size=(3, 0),
                           alibi_slopes=torch.ones(4, device=DEV))),
            ("is on cpu", dict(k_descale=torch.ones(1))), ("softcap", dict(softcap=-1.0)),
            ("CUDA tensors only", dict(q=q.cpu()))]:
        with pytest.raises(RuntimeError, match=match):
            call(**kw)
    for kw in [dict(q=q.float()), dict(vc=kc.view(torch.uint8).view(E5M2)), dict(lens=lens.long()), dict(table=table.long()),
               dict(table=torch.zeros((3, 1), dtype=torch.int32, device=DEV)), dict(cu=cu.long()),
               dict(q=torch.zeros((2, 3, 64), dtype=torch.bfloat16, device=DEV)), dict(out=q.half()),
               dict(q=q[:, :, :40], kc=kc[..., :36], vc=kc[..., :36])]:
        with pytest.raises((AssertionError, RuntimeError)):
            call(**kw)


def test_sixteen_bit_calls_ignore_the_new_arguments(fg):
    g = gen(8)
    kc, vc, table, rows = paged(g, [100, 33], 16, 2, 64, torch.bfloat16)
    q = randn(g, 2, 4, 64).to(torch.bfloat16)
    args = (q, kc, vc, 1, torch.tensor([0, 1, 2], dtype=torch.int32, device=DEV), 100)
    kw = dict(seqused_k=torch.tensor([100, 33], dtype=torch.int32, device=DEV), causal=True, block_table=table)
    plain = fg.flash_attn_varlen_func(*args, **kw)
    half = torch.full((1,), 0.5, device=DEV)
    assert torch.equal(plain, fg.flash_attn_varlen_func(*args, k_descale=half, v_descale=half, **kw))
    assert torch.equal(plain, fg.flash_attn_varlen_func(*args, sink_tokens=4, **kw))     # no window: every key is visible
    assert torch.equal(plain, fg.flash_attn_varlen_func(*args, sink_tokens=4, window_size=(-1, 0), **kw))


# ------------------------------------------------------------------------------------------------------ callers
@pytest.mark.parametrize("name, cache", [("fp8", E4M3), ("fp8_e4m3", E4M3), ("fp8_e5m2", E5M2)])
def test_patched_attention_layer_with_an_8_bit_cache(fg, name, cache):
    g = gen(9)
    heads, hk, dim, page = 8, 2, 128, 16
    seqs = [(1, 1328), (5, 18), (129, 463), (1, 77), (200, 200)]
    q_lens, k_lens = [a for a, _ in seqs], [b for _, b in seqs]
    ks, vs = (torch.tensor(s, device=DEV) for s in (0.011, 0.017))        # vLLM's scales have no dimension
    kc, vc, table, rows = paged(g, k_lens, page, hk, dim, cache, ks, vs)
    total, pad = sum(q_lens), 4
    key, value = randn(g, total + pad, hk, dim).to(torch.bfloat16), randn(g, total + pad, hk, dim).to(torch.bfloat16)
    slots, at = [], 0
    for b, (n, m) in enumerate(seqs):
        slots += [int(table[b, t // page]) * page + t % page for t in range(m - n, m)]
        for i, (x, s) in enumerate(((key, ks), (value, vs))):
            rows[b][i] = torch.cat([rows[b][i][:m - n].view(torch.uint8), quantise(x[at:at + n], s, cache).view(torch.uint8)]).view(cache)
        at += n
    md = SimpleNamespace(
        num_actual_tokens=total, slot_mapping=torch.tensor(slots + [-1] * pad, device=DEV),
        query_start_loc=torch.tensor([0] + q_lens, device=DEV).cumsum(0, dtype=torch.int32),
        seq_lens=torch.tensor(k_lens, dtype=torch.int32, device=DEV), max_query_len=max(q_lens), max_seq_len=max(k_lens),
        block_table=table, use_cascade=False)
    impl = SimpleNamespace(kv_cache_dtype=name, scale=dim ** -0.5, alibi_slopes=None, sliding_window=(-1, -1),
                           logits_soft_cap=0.0, use_irope=False)
    layer = SimpleNamespace(_k_scale=ks, _v_scale=vs)
    kv_cache = torch.stack([kc.view(torch.uint8), vc.view(torch.uint8)])
    query = randn(g, total + pad, heads, dim).to(torch.bfloat16)
    output = torch.full((total + pad, heads, dim), 7.0, dtype=torch.bfloat16, device=DEV)
    ret = patches.custom_gems_flash_attention_impl_forward(impl, layer, query, key, value, kv_cache, md, output=output)
    assert ret is output and (output[total:] == 7.0).all()
    want, _, tol, _ = attention(q_lens, k_lens, query[:total], rows, [ks] * 5, [vs] * 5, dim ** -0.5, True, (-1, -1), 0, 0.0,
                                torch.bfloat16, cache)
    assert ((output[:total].double() - want).abs() <= tol).all()
    impl.kv_cache_dtype = "fp8_inc"
    with pytest.raises(NotImplementedError, match="fp8_inc"):
        patches.custom_gems_flash_attention_impl_forward(impl, layer, query, key, value, kv_cache, md, output=output)


def test_custom_ops(fg):
    g = gen(10)
    scale = torch.tensor([0.01], device=DEV)
    kc, vc, table, rows = paged(g, [30], 16, 2, 64, E4M3, scale, scale)
    x = randn(g, 1, 2, 64).to(torch.bfloat16)
    slot = (table[0, 1:2].long() * 16 + 13)
    torch.ops.flag_gems.reshape_and_cache_flash(x, x, kc, vc, slot, "fp8", scale, scale)
    key, value = (torch.zeros((30, 2, 64), dtype=torch.bfloat16, device=DEV) for _ in range(2))
    cu = torch.tensor([0, 30], dtype=torch.int32, device=DEV)
    torch.ops.flag_gems.gather_cache_flash(kc, vc, key, value, table, cu, "fp8", scale, scale)
    assert torch.equal(key[29], (quantise(x, scale, E4M3).float() * scale).to(torch.bfloat16)[0])
    assert torch.equal(value[:29], (rows[0][1].float() * scale).to(torch.bfloat16)[:29])
    q = randn(g, 1, 4, 64).to(torch.bfloat16)
    cu_q, used = torch.tensor([0, 1], dtype=torch.int32, device=DEV), torch.tensor([30], dtype=torch.int32, device=DEV)
    out, lse = torch.ops.flag_gems.flash_attn_varlen_func(q, kc, vc, 1, cu_q, 30, None, used, causal=True, block_table=table,
                                                          k_descale=scale, v_descale=scale)
    want = fg.flash_attn_varlen_func(q, kc, vc, 1, cu_q, 30, seqused_k=used, causal=True, block_table=table, k_descale=scale,
                                     v_descale=scale)
    assert torch.equal(out, want) and lse.shape == (4, 1)

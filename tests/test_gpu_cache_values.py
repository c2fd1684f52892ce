"""Attention over an 8-bit or windowed cache where values are uneven: rows of Q with outlying channels, keys whose
probabilities are tiny beside one key's, infinities that a query sees.

Every kernel family is asked: the one for few keys and the one for many (a large ``bound``) where there are few query
rows, chunks, long chunks over a widened store, and the general form.  The definition in 64 bits and the bounds are those
of ``test_gpu_cache_fp8``, which hold a score to the rounding of a sum in 32 bits whatever the rows hold.
"""
import math

import pytest
import torch

from test_gpu_cache_fp8 import DEV, E4M3, E5M2, TOP, U, attention, check, gen, quantise, randn

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
PAGE = 16
# (tokens of each sequence, max_seqlen_k or 0 for the longest): few and many keys, chunks, long chunks
FORMS = [([1, 1, 1], 0), ([1, 1, 1], 10 ** 6), ([40, 3, 7], 0), ([300, 1, 20], 0)]
LENS = [700, 333, 90]


def store(g, rows, cache):
    """Paged caches that hold `rows` (pairs of K and V), the pages in no order, and their table."""
    pages = [(r[0].shape[0] + PAGE - 1) // PAGE for r in rows]
    order = torch.randperm(sum(pages) + 2, generator=g, device=DEV).to(torch.int32)
    table = torch.zeros((len(rows), max(pages)), dtype=torch.int32, device=DEV)
    shape = (sum(pages) + 2, PAGE, *rows[0][0].shape[1:])
    view = (lambda t: t.view(torch.uint8)) if cache in TOP else (lambda t: t)
    caches = [torch.zeros(shape, dtype=cache, device=DEV) for _ in range(2)]
    at = 0
    for i, pair in enumerate(rows):
        table[i, :pages[i]] = order[at:at + pages[i]]
        at += pages[i]
        pos = torch.arange(pair[0].shape[0], device=DEV)
        for c, x in zip(caches, pair):
            view(c)[table[i, pos // PAGE].long(), pos % PAGE] = view(x)
    return *caches, table


def call(fg, q_lens, bound, q, rows, cache, table=None, window=(-1, -1), sinks=0, scale=None):
    kc, vc, table = store(gen(1), rows, cache)
    cu = torch.tensor([0] + q_lens, device=DEV).cumsum(0, dtype=torch.int32)
    lens = torch.tensor([r[0].shape[0] for r in rows], dtype=torch.int32, device=DEV)
    return fg.flash_attn_varlen_func(
        q, kc, vc, max(q_lens), cu, bound or int(lens.max()), seqused_k=lens, block_table=table, causal=True,
        softmax_scale=q.shape[-1] ** -0.5, window_size=window, sink_tokens=sinks, k_descale=scale, v_descale=scale,
        return_softmax_lse=True)


def random_rows(g, hk, dim, cache, scale):
    if cache in TOP:
        return [[quantise(randn(g, n, hk, dim), scale, cache) for _ in range(2)] for n in LENS]
    return [[randn(g, n, hk, dim).to(cache) for _ in range(2)] for n in LENS]


def poke(x, index, value):
    """x[index] = value for 8-bit types too."""
    if x.dtype in TOP:
        x.view(torch.uint8)[index] = torch.tensor(value, device=DEV).to(x.dtype).view(torch.uint8)
    else:
        x[index] = value


@pytest.mark.parametrize("q_lens, bound", FORMS)
@pytest.mark.parametrize("factor", [16.0, 64.0, 1024.0])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("heads, hk", [(8, 2), (7, 1), (16, 1)])
@pytest.mark.parametrize("dtype, cache", [(BF16, E4M3), (FP16, E4M3), (BF16, E5M2), (FP16, E5M2)])
def test_outlying_channels_of_q(fg, dtype, cache, heads, hk, dim, factor, q_lens, bound):
    """One channel of each query row far above the others, where the keys hold next to nothing: the scores come from the
    small channels.  The kernels may lose 2^-27 of a row's largest value in each channel, 2^-17 at a factor of 1024;
    the bound of a score's sum allows (dim + 8) 2^-22 >= 2^-15.9 of each channel's product."""
    g = gen(int(factor) + dim + heads)
    scale = torch.tensor([4.5 / TOP[cache]], device=DEV)
    rows = random_rows(g, hk, dim, cache, scale)
    q = randn(g, sum(q_lens), heads, dim)
    for channel in (3, dim - 10):
        q[:, :, channel] = factor * (1 + torch.rand(q.shape[:2], generator=g, device=DEV))
        for k, _ in rows:
            poke(k, (slice(None), slice(None), channel), 0.0)
    q = q.to(dtype)
    out, lse = call(fg, q_lens, bound, q, rows, cache, scale=scale)
    want, wlse, tol, lse_tol = attention(q_lens, LENS, q, rows, [scale] * 3, [scale] * 3, dim ** -0.5, True, (-1, -1), 0, 0.0,
                                         dtype, cache)
    worst = ((out.double() - want).abs() / tol).max().item()
    assert worst <= 1.0, f"error {worst:.3g} of the bound"
    assert ((lse.double() - wlse).abs() <= lse_tol).all()


def test_outlying_channels_give_the_same_in_every_form(fg):
    """The form for many keys against the one for few, score by score: both hold Q to well below a bf16 step."""
    g = gen(5)
    scale = torch.tensor([0.01], device=DEV)
    rows = random_rows(g, 2, 128, E4M3, scale)
    q = randn(g, 3, 8, 128)
    q[:, :, 7] = 4096.0
    for k, _ in rows:
        poke(k, (slice(None), slice(None), 7), 0.0)
    q = q.to(BF16)
    few, many = (call(fg, [1, 1, 1], bound, q, rows, E4M3, scale=scale)[1] for bound in (0, 10 ** 6))
    # 2^-27 of 4096 in 128 channels, with keys of 4.5 standard deviations at most; beside it the sums' own roundings
    assert ((few - many).abs() <= 128 * 2.0 ** -15 * 4.5 * 128 ** -0.5 + 1e-4).all()


@pytest.mark.parametrize("q_lens, bound", FORMS)
@pytest.mark.parametrize("dim", [64, 128, 256, 72])
@pytest.mark.parametrize("dtype, cache", [(BF16, E5M2), (FP16, E5M2), (BF16, BF16), (FP16, FP16)])
def test_infinite_values_that_every_query_sees(fg, dtype, cache, dim, q_lens, bound):
    """An infinity among the V values of a channel is that channel's output, two of opposite signs or a NaN are a NaN, and the
    other channels are what they are."""
    g = gen(dim)
    window, sinks = ((-1, -1), 0) if cache in TOP else ((10 ** 5, 0), 4)
    if bound == 0 and cache not in TOP:
        window = (600, 0)         # shorter than the longest sequence, longer than every chunk
    scale = torch.tensor([0.01 if cache in TOP else 1.0], device=DEV)
    rows = random_rows(g, 2, dim, cache, scale)
    clean = [[t.clone() for t in pair] for pair in rows]
    for b, (_, v) in enumerate(rows):     # keys 0 to 3 and the first new token's own are seen by every query
        last = LENS[b] - q_lens[b]
        poke(v, (1, 0, 5), math.inf)
        poke(v, (last, 0, 9), -math.inf)
        poke(v, (2, 1, 11), math.inf)
        poke(v, (3, 1, 11), math.inf)
        poke(v, (2, 1, 20), math.inf)
        poke(v, (last, 1, 20), -math.inf)
        poke(v, (0, 1, 21), math.nan)
    q = randn(g, sum(q_lens), 8, dim).to(dtype)
    out, lse = call(fg, q_lens, bound, q, rows, cache, window=window, sinks=sinks, scale=scale if cache in TOP else None)
    want, wlse, tol, lse_tol = attention(q_lens, LENS, q, clean, [scale] * 3, [scale] * 3, dim ** -0.5, True, window, sinks, 0.0,
                                         dtype, cache)
    odd = torch.zeros((8, dim), dtype=torch.float64, device=DEV)
    odd[:4, 5], odd[:4, 9], odd[4:, 11] = math.inf, -math.inf, math.inf
    odd[4:, 20:22] = math.nan
    want = want + odd
    ok = odd == 0
    assert torch.equal(out[:, ~ok].nan_to_num(7.0), want[:, ~ok].to(dtype).nan_to_num(7.0))
    assert ((out[:, ok].double() - want[:, ok]).abs() <= tol[:, ok]).all()
    assert ((lse.double() - wlse).abs() <= lse_tol).all()


@pytest.mark.parametrize("q_lens, bound", FORMS)
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_infinite_keys(fg, dtype, dim, q_lens, bound):
    """A score of -inf takes its key out; +inf, or both in one product, leave no number."""
    g = gen(dim + 1)
    scale = torch.tensor([0.01], device=DEV)
    rows = random_rows(g, 2, dim, E5M2, scale)
    q = randn(g, sum(q_lens), 8, dim)
    q[:, :, 5] = q[:, :, 5].abs() + 0.1
    q[:, :, 6] = -q[:, :, 6].abs() - 0.1
    q = q.to(dtype)
    clean = [[t.clone() for t in pair] for pair in rows]
    for b, (k, v) in enumerate(rows):
        for j, channel, value in ((2, 5, -math.inf), (30, 6, math.inf), (LENS[b] - q_lens[b], 5, -math.inf)):
            poke(k, (j, 0, channel), value)
            # in the definition: a key so small that its probability is below any rounding
            poke(clean[b][0], (j, 0, channel), -57344.0 if channel == 5 else 57344.0)
        poke(k, (1, 1, 6), -math.inf)
    out, lse = call(fg, q_lens, bound, q, rows, E5M2, scale=scale)
    ends = torch.tensor(q_lens).cumsum(0).tolist()
    at = 0
    for b, end in enumerate(ends):
        # keys far below, with their part of the sum's rounding error left out of the bound
        k, v = clean[b][0].double() * 0.01, clean[b][1].double() * 0.01
        k, v = k[:, 0], v[:, 0]
        p = torch.arange(end - at, device=DEV).view(-1, 1) + LENS[b] - (end - at)
        for h in range(4):
            qq = q[at:end, h].double()
            a = (qq @ k.T * dim ** -0.5).masked_fill(torch.arange(LENS[b], device=DEV) > p, -math.inf)
            keep = k.abs().amax(-1) < 500
            a[:, ~keep] = -math.inf
            w = torch.softmax(a, -1)
            size = w @ v.abs()
            ds = (dim + 8) * 2.0 ** -22 * dim ** -0.5 * (qq.abs() @ k[keep].abs().T).amax(-1, keepdim=True)
            tol = U[dtype] * (w @ v).abs() + (2.0 ** -11 + 2 * ds + 2.0 ** -16) * size + LENS[b] * 2.0 ** -25 * v.abs().max()
            assert ((out[at:end, h].double() - w @ v).abs() <= tol).all()
            assert ((lse[h, at:end].double() - torch.logsumexp(a, -1)).abs() <= 2 * ds[:, 0] + 2.0 ** -12).all()
        at = end
    assert out[:, 4:].isnan().all() and lse[4:].isnan().all()


@pytest.mark.parametrize("q_lens, bound", FORMS)
@pytest.mark.parametrize("gap", [16.0, 18.0])
@pytest.mark.parametrize("dim", [64, 128, 256, 72])
@pytest.mark.parametrize("dtype, cache", [(BF16, E4M3), (FP16, E5M2), (FP16, FP16)])
def test_small_probabilities_beside_a_first_token(fg, dtype, cache, dim, gap, q_lens, bound):
    """The first token draws nearly all attention and its value is zero, as trained models have it: the output is the sum of many
    probabilities of about e^-gap.  A probability may be off by 2^-11 of itself or 2^-32 of the row's largest."""
    g = gen(int(gap) + dim)
    eight = cache in TOP
    window, sinks = ((-1, -1), 0) if eight else ((600, 0), 4)
    scale = torch.tensor([2.0 ** -6 if eight else 1.0], device=DEV)
    rows = random_rows(g, 2, dim, cache, scale)
    u = torch.zeros(dim, device=DEV)
    u[:8] = 1.0                        # the first token's direction: eight channels that the other keys leave alone
    for k, v in rows:
        poke(k, (slice(1, None), slice(None), slice(0, 8)), 0.0)
        poke(k, 0, 0.0)
        poke(v, 0, 0.0)
        k0 = 4.0 / scale.item()
        poke(k, (0, slice(None), slice(0, 8)), k0)
    q = 0.5 * randn(g, sum(q_lens), 8, dim)
    q[:, :, :8] = gap * dim ** 0.5 / (8 * 4.0)
    q = q.to(dtype)
    out, lse = call(fg, q_lens, bound, q, rows, cache, window=window, sinks=sinks, scale=scale if eight else None)
    want, wlse, tol, lse_tol = attention(q_lens, LENS, q, rows, [scale] * 3, [scale] * 3, dim ** -0.5, True, window, sinks, 0.0,
                                         dtype, cache)
    # The outputs are about 2^-18.  fp16 values below 2^-14 are multiples of 2^-24: rounding one to them moves it by up to 2^-25,
    # whatever its size, which the share of the value in the bound does not hold.
    tol += 2.0 ** -25 if dtype == FP16 else 0.0
    at = 0
    for b, n in enumerate(q_lens):     # the bound of test_gpu_cache_fp8 takes 2^-25 a key; here it is 2^-32
        top = (rows[b][1].double() * scale.double()).abs().max()
        tol[at:at + n] -= LENS[b] * (2.0 ** -25 - 2.0 ** -32) * top
        at += n
    worst = ((out.double() - want).abs() / tol).max().item()
    assert worst <= 1.0, f"error {worst:.3g} of the bound"
    assert ((lse.double() - wlse).abs() <= lse_tol).all()


@pytest.mark.parametrize("kw", [dict(dim=128, softcap=30.0), dict(dim=96), dict(dim=256, cache=BF16, window=(10 ** 5, 0), sinks=4)])
def test_long_ranges_of_a_large_bound(fg, kw):
    """So many rows that the ranges of the keys grow with the bound: sequences shorter than one, longer, and as long as several."""
    kw = {"cache": E4M3, **kw}
    lens = [1 + (i * 977) % 3000 for i in range(44)] + [40000, 16384, 16385, 0]
    check(fg, [1] * 48, lens, 32, 8, page=16, dtype=BF16, bound=10 ** 6, **kw)


@pytest.mark.parametrize("limit", [0, 96 << 20])
@pytest.mark.parametrize("q_lens, dim", [([600, 1, 0, 130], 128), ([600, 1, 0, 130], 64), ([300, 1, 20, 7], 256), ([1, 1, 1, 1], 128)])
def test_calls_that_find_no_memory_for_their_workspace(fg, monkeypatch, q_lens, dim, limit):
    """The allocator is out of memory beyond `limit` bytes: the same results from the forms that need less."""
    real, refused = torch.empty, []

    def empty(*args, **kw):
        if kw.get("dtype") == torch.uint8 and args[0] > limit:
            refused.append(args[0])
            raise torch.OutOfMemoryError("no memory")
        return real(*args, **kw)

    monkeypatch.setattr(torch, "empty", empty)
    check(fg, q_lens, [900, 700, 33, 130], 8, 4, dim, 16, BF16, E4M3, bound=40000)
    assert refused or (limit and max(q_lens) == 1)


@pytest.mark.parametrize("cache", [BF16, E4M3])
@pytest.mark.parametrize("q_lens", [[1, 1, 1], [40, 3, 7]])
def test_the_custom_op_takes_first_tokens(fg, cache, q_lens):
    g = gen(3)
    scale = torch.tensor([0.01], device=DEV) if cache in TOP else None
    kc, vc, table = store(g, random_rows(g, 2, 128, cache, scale), cache)
    cu = torch.tensor([0] + q_lens, device=DEV).cumsum(0, dtype=torch.int32)
    lens = torch.tensor(LENS, dtype=torch.int32, device=DEV)
    q = randn(g, sum(q_lens), 8, 128).to(BF16)
    args, kw = (q, kc, vc, max(q_lens), cu, max(LENS)), dict(seqused_k=lens, causal=True, window_size=[50, 0], block_table=table,
                                                            k_descale=scale, v_descale=scale)
    out, lse = torch.ops.flag_gems.flash_attn_varlen_func(*args, sink_tokens=5, **kw)
    want, want_lse = fg.flash_attn_varlen_func(*args, sink_tokens=5, return_softmax_lse=True, **kw)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
    without = torch.ops.flag_gems.flash_attn_varlen_func(*args, **kw)[0]
    assert not torch.equal(out, without)


@pytest.mark.parametrize("heads, hk", [(32, 32), (40, 40), (17, 17), (64, 32)])
@pytest.mark.parametrize("cache, kw", [
    (E4M3, {}), (E4M3, dict(bound=10 ** 6)), (BF16, dict(window=(2500, 0), sinks=4)), (E5M2, dict(dim=256, bound=10 ** 5))])
def test_more_kv_heads_than_a_team_of_ctas(fg, heads, hk, cache, kw):
    """Decode walks KV heads in teams of CTAs, in rounds where there are more heads than a team has; unequal long sequences are cut
    in later rounds and joined, short ones are whole."""
    kw = {"dim": 128, **kw}
    lens = [3000, 17, 5000, 129, 2900, 1, 4100, 640]
    check(fg, [1] * 8, lens, heads, hk, page=16, dtype=BF16, cache=cache, scale_shape="heads", **kw)
    check(fg, [1] * 8, [1 + n % 700 for n in lens], heads, hk, page=16, dtype=BF16, cache=cache, scale_shape="heads", **kw)


@pytest.mark.parametrize("kw", [dict(dim=96), dict(dim=128, softcap=30.0), dict(dim=200, cache=E5M2), dict(dim=72, cache=BF16,
                                                                                             window=(900, 0), sinks=4)])
@pytest.mark.parametrize("q_lens", [[1, 1, 1, 1], [20, 3, 0, 1], [200, 1, 64, 65]])
def test_many_rows_behind_the_sequences(fg, kw, q_lens):
    """A q padded far beyond its sequences: the rows behind them are left as they were, and take no room."""
    check(fg, q_lens, [4000, 1300, 77, 700], 8, 2, page=16, dtype=BF16, behind=9000, **{"cache": E4M3, **kw})


@pytest.mark.parametrize("dim", [64, 128, 256, 96])
@pytest.mark.parametrize("cache", [E4M3, BF16])
@pytest.mark.parametrize("window", [(0, 100), (1023, 5), (3, 20), (8, 12), (2, 1)])
@pytest.mark.parametrize("q_lens, bound", [([102, 25, 3], 0), ([102, 25, 3], 2000), ([4, 3, 1], 0), ([4, 3, 1], 10 ** 6)])
def test_right_windows_over_fewer_keys_than_new_tokens(fg, q_lens, bound, window, cache, dim):
    """Without the causal mask, the first of many new tokens are at negative positions: a right window longer than the sequence
    still hides keys from them."""
    check(fg, q_lens, [5, 9, 2], 8, 2, dim, 16, BF16, cache, causal=False, window=window, sinks=4, bound=bound)


@pytest.mark.parametrize("scale", [None, 0.3, 114.0, 1e-20])
@pytest.mark.parametrize("dim", [128, 40])
@pytest.mark.parametrize("cache", [E4M3, E5M2])
@pytest.mark.parametrize("dtype", [BF16, FP16, torch.float32])
def test_write_keeps_the_sign_of_zero(fg, dtype, cache, dim, scale):
    """Zeros, and quotients that round to zero, keep their sign as in a division, and come back with it."""
    key = torch.zeros((4, 2, dim), device=DEV)
    key[1] = -0.0
    key[2], key[3] = 1e-7 * (scale or 1.0), -1e-7 * (scale or 1.0)      # below half of the smallest value of either type
    key = key.to(dtype)
    caches = [torch.full((1, 4, 2, dim), 0x55, dtype=torch.uint8, device=DEV).view(cache) for _ in range(2)]
    s = None if scale is None else torch.tensor([scale], device=DEV)
    name = "fp8_e4m3" if cache == E4M3 else "fp8_e5m2"
    fg.reshape_and_cache_flash(key, -key, *caches, torch.arange(4, device=DEV), name, s, s)
    for c, x in zip(caches, (key, -key)):
        assert torch.equal(c.view(torch.uint8)[0], torch.signbit(x).to(torch.uint8) * 0x80)
    k, v = torch.empty_like(key), torch.empty_like(key)
    table, cu = torch.zeros((1, 1), dtype=torch.int32, device=DEV), torch.tensor([0, 4], dtype=torch.int32, device=DEV)
    fg.gather_cache_flash(*caches, k, v, table, cu, name, s, s)
    assert (k == 0).all() and torch.equal(torch.signbit(k), torch.signbit(key)) and torch.equal(torch.signbit(v), torch.signbit(-key))

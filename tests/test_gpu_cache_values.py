"""Attention over an 8-bit or windowed cache where values are uneven: rows of Q with outlying channels, keys whose
probabilities are tiny beside one key's, infinities that a query sees.

Every kernel family is asked: the one for few keys and the one for many (a large ``bound``) where there are few query
rows, chunks, long chunks over a widened store, and the general form.  The definition in 64 bits and the bounds are those
of ``test_gpu_cache_fp8``, which hold a score to the rounding of a sum in 32 bits whatever the rows hold.
"""
import math

import pytest
import torch

from test_gpu_cache_fp8 import DEV, E4M3, E5M2, TOP, U, attention, gen, quantise, randn

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

"""Host side of the 8-bit and windowed cache: structure layout, refusals before any CUDA call, path and workspace rules,
and a restatement of the tile runs that the attention kernels walk."""
import ctypes
import re
import subprocess
import sys
from pathlib import Path

import pytest
import torch

from flaggems_b200 import _lib, fused


def params(**kw):
    p = _lib.AttnCacheParams()
    b = p.base
    b.q = b.k = b.v = b.out = b.cu_seqlens_q = b.seqused_k = b.block_table = 0x10000
    b.q_row_stride, b.q_head_stride, b.o_row_stride, b.o_head_stride = 1024, 128, 1024, 128
    b.k_block_stride = b.v_block_stride = 16 * 256
    b.k_row_stride = b.v_row_stride = 256
    b.k_head_stride = b.v_head_stride = 128
    b.total_q, b.batch, b.num_heads, b.num_heads_k, b.head_dim = 4, 4, 8, 2, 128
    b.max_seqlen_q, b.max_seqlen_k, b.block_size, b.num_blocks = 1, 1000, 16, 100
    b.window_left = b.window_right = -1
    b.softmax_scale, b.causal, b.dtype = 0.1, 1, _lib.FG_BF16
    p.block_table_cols, p.cache_dtype = 63, _lib.FG_E4M3
    for name, v in kw.items():
        setattr(p if hasattr(p, name) else b, name, v)
    return p


def test_parameter_blocks():
    """The packed blocks have the header's layout: every field of the attention block lands where the Structure has it."""
    assert ctypes.sizeof(_lib.AttnCacheParams) == ctypes.sizeof(_lib.AttnParams) + 2 * 8 + 6 * 8 + 2 * 4
    assert _lib.ATTN_CACHE.size == ctypes.sizeof(_lib.AttnCacheParams)
    values = [i + 1 for i in range(40)] + [0.5, 0.25] + list(range(43, 47)) + list(range(47, 57))
    p = _lib.AttnCacheParams.from_buffer_copy(_lib.ATTN_CACHE.pack(*values))
    got = [getattr(p.base, n) for n, _ in _lib.AttnParams._fields_] + [getattr(p, n) for n, _ in p._fields_[1:]]
    assert got == values
    for fmt, name in ((_lib.CACHE_WRITE, "fg_cache_write_params"), (_lib.CACHE_GATHER, "fg_cache_gather_params")):
        header = (Path(__file__).resolve().parent.parent / "include" / "flaggems_b200.h").read_text()
        body = re.search(r"typedef struct \{([^}]*)\} " + name, header).group(1)
        body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
        kinds = [("Q" if "*" in d else "i" if "int32_t" in d else "q") * (d.count(",") + 1) for d in body.split(";") if d.strip()]
        assert "".join(kinds) == "".join(c * int(n or 1) for n, c in re.findall(r"(\d*)([Qqi])", fmt.format))


@pytest.mark.parametrize("match, kw", [
    ("fp16 and bf16", dict(dtype=_lib.FG_F32)), ("8-bit type", dict(cache_dtype=_lib.FG_F16)), ("8-bit type", dict(cache_dtype=9)),
    ("scales belong", dict(cache_dtype=_lib.FG_BF16, k_scale=0x10000)), ("negative size", dict(batch=-1)),
    ("must divide", dict(num_heads=7)), ("at most 256", dict(head_dim=264)), ("multiple of 8", dict(head_dim=124)),
    ("sink_tokens", dict(sink_tokens=-1)), ("ALiBi", dict(alibi_slopes=0x10000)), ("batch strides", dict(q_batch_stride=8)),
    ("softcap", dict(softcap=-1.0)), ("65535", dict(batch=70000, total_q=70000)), ("null tensor", dict(k=None)),
    ("cu_seqlens_q", dict(cu_seqlens_q=None)), ("seqused_k", dict(seqused_k=None)), ("block_size", dict(block_size=0)),
    ("no columns", dict(block_table_cols=0)), ("16-byte", dict(q=0x10008)), ("multiples of 8", dict(k_row_stride=252)),
    ("too long", dict(max_seqlen_k=2 ** 31)), ("cu_seqlens_k", dict(block_table=None)), ("positive", dict(num_heads_k=0))])
def test_attention_refuses_on_the_host(match, kw):
    lib = _lib.load()
    rc = lib.fg_flash_attn_cache(ctypes.byref(params(**kw)), None)
    assert rc < 0
    with pytest.raises(RuntimeError, match=match):
        _lib.check(rc)


def test_nothing_to_do_is_no_call():
    lib = _lib.load()
    for kw in (dict(batch=0), dict(total_q=0), dict(max_seqlen_q=0)):
        assert lib.fg_flash_attn_cache(ctypes.byref(params(**kw)), None) == 0


def test_small_workspace_is_refused():
    lib = _lib.load()
    p = params(max_seqlen_k=60000, batch=1, total_q=1, head_dim=80)
    need = lib.fg_flash_attn_cache_workspace_bytes(ctypes.byref(p))
    assert need > 0 and need % (8 * 81 * 4) == 0
    p.base.workspace, p.base.workspace_bytes = 0x10000, need - 4
    with pytest.raises(RuntimeError, match="workspace of"):
        _lib.check(lib.fg_flash_attn_cache(ctypes.byref(p), None))
    p.base.workspace, p.base.workspace_bytes = 0x10004, need
    with pytest.raises(RuntimeError, match="aligned"):
        _lib.check(lib.fg_flash_attn_cache(ctypes.byref(p), None))


def test_workspace_goes_by_what_is_visible():
    """A window bounds the keys that are split, however long the context."""
    need = lambda **kw: _lib.load().fg_flash_attn_cache_workspace_bytes(ctypes.byref(params(**kw)))
    for size in (dict(head_dim=80), dict(head_dim=248, max_seqlen_q=30, total_q=100)):
        long, windowed = need(max_seqlen_k=10 ** 6, **size), need(max_seqlen_k=10 ** 6, window_left=2047, sink_tokens=4, **size)
        assert 0 < windowed < long and windowed == need(max_seqlen_k=10 ** 5, window_left=2047, sink_tokens=4, **size)
    chunk = dict(max_seqlen_q=30, total_q=100)
    assert need(max_seqlen_k=10 ** 6, **chunk) == need(max_seqlen_k=10 ** 4, **chunk) > need(max_seqlen_k=10 ** 4) > 0
    assert need(max_seqlen_k=100, **chunk) == need(max_seqlen_k=100) == 0      # short contexts are not cut
    # a long chunk: the 16-bit copy of an 8-bit store comes on top, until it would be larger than 1 GiB
    long = dict(max_seqlen_q=256, total_q=1000)
    copy = need(max_seqlen_k=6400, **long) - need(max_seqlen_k=6400, cache_dtype=_lib.FG_BF16, **long)
    assert copy == 2 * 4 * 6400 * 2 * 128 * 2
    assert need(max_seqlen_k=10 ** 6, **long) == need(max_seqlen_k=10 ** 6, cache_dtype=_lib.FG_BF16, **long)
    assert need(max_seqlen_k=10 ** 6) == need(max_seqlen_k=10 ** 4)        # head parts and tail parts of a fixed number of CTAs
    # chunks whose 8-bit store is widened ahead of the attention: the copy holds what is visible
    for size in (dict(head_dim=256, max_seqlen_q=30, total_q=100), dict(max_seqlen_q=600, total_q=1000)):
        long, windowed = need(max_seqlen_k=10 ** 5, **size), need(max_seqlen_k=10 ** 5, window_left=2047, sink_tokens=4, **size)
        assert 0 < windowed < long // 5 and windowed == need(max_seqlen_k=10 ** 6, window_left=2047, sink_tokens=4, **size)


def test_long_chunks_without_the_widened_copy():
    need = lambda **kw: _lib.load().fg_flash_attn_cache_workspace_bytes(ctypes.byref(params(**kw)))
    path = lambda **kw: _lib.load().fg_flash_attn_cache_path(ctypes.byref(params(**kw)))
    long = dict(max_seqlen_q=256, total_q=1000, max_seqlen_k=6400)
    assert need(flags=1, **long) == need(cache_dtype=_lib.FG_BF16, **long) < need(**long) and path(flags=1, **long) == 1
    long["head_dim"] = 64
    assert path(**long) == 1 and path(flags=1, **long) == 0 and need(flags=1, **long) < need(**long)
    with pytest.raises(RuntimeError, match="unknown flags"):
        _lib.check(_lib.load().fg_flash_attn_cache(ctypes.byref(params(flags=6)), None))


def test_no_memory_for_the_workspace(monkeypatch):
    """What the call gets when the allocation fails: the form without the copy, then none."""
    from flaggems_b200 import ops
    lib = _lib.load()
    block = bytes(params(max_seqlen_q=256, total_q=1000, max_seqlen_k=6400))
    full = lib.fg_flash_attn_cache_workspace_bytes(block)
    asked, limit = [], [0]
    real = torch.empty

    def empty(n, dtype, device):
        asked.append(n)
        if n > limit[0]:
            raise torch.OutOfMemoryError("no memory")
        return real(n, dtype=dtype, device="cpu")

    monkeypatch.setattr(torch, "empty", empty)
    for limit[0], sizes in ((full, 1), (full - 1, 2), (0, 2)):
        asked.clear()
        ws, got = ops._cache_workspace(lib, block, full, "cuda")
        p = _lib.AttnCacheParams.from_buffer_copy(got)
        assert len(asked) == sizes and asked[0] == full and p.flags == sizes - 1
        small = lib.fg_flash_attn_cache_workspace_bytes(block[:-4] + _lib.CACHE_NO_COPY)
        assert small < full and asked[1:] == [small][:sizes - 1]
        if limit[0] == 0:
            assert ws is None and not p.base.workspace and p.base.workspace_bytes == 0
        else:
            assert p.base.workspace == ws.data_ptr() and p.base.workspace_bytes == ws.numel() == asked[-1]
        assert got[:80] == block[:80] and got[96:-4] == block[96:-4]


def test_workspace_of_the_split_decode_form_is_bounded():
    """Soft-capping and odd head dims split by max_seqlen_k: large batches with a bound far above their contexts stay small."""
    need = lambda **kw: _lib.load().fg_flash_attn_cache_workspace_bytes(ctypes.byref(params(**kw)))
    path = lambda **kw: _lib.load().fg_flash_attn_cache_path(ctypes.byref(params(**kw)))
    for batch in (1, 4, 64, 256, 4096):
        for heads, heads_k in ((8, 2), (32, 8), (128, 8)):
            for form in (dict(softcap=50.0), dict(head_dim=96), dict(head_dim=256, cache_dtype=_lib.FG_BF16, window_left=10 ** 5)):
                for bound in (1000, 131072, 10 ** 6, 10 ** 7):
                    size = dict(batch=batch, total_q=batch, num_heads=heads, num_heads_k=heads_k, max_seqlen_k=bound, **form)
                    assert path(**size) == 2 and need(**size) <= 64 * 2 ** 20
                    small = dict(size, max_seqlen_k=min(bound, 8000))
                    assert need(**size) > 0 or need(**small) == 0 or batch * heads >= 4096   # few rows are split all the same
    assert need(total_q=0, softcap=50.0, max_seqlen_k=10 ** 6) == 0


def test_rows_behind_the_sequences_take_no_workspace():
    """A padded q: the split forms' partial results go by the tokens that the sequences can have, not by the rows of q."""
    need = lambda **kw: _lib.load().fg_flash_attn_cache_workspace_bytes(ctypes.byref(params(**kw)))
    for form in (dict(head_dim=96), dict(head_dim=200, softcap=30.0)):
        for batch, max_q in ((1, 20), (3, 100), (2, 1), (64, 1)):
            size = dict(batch=batch, max_seqlen_q=max_q, num_heads=32, num_heads_k=8, max_seqlen_k=16384, **form)
            assert 0 < need(total_q=batch * max_q, **size) == need(total_q=65536, **size) <= 64 * 2 ** 20
            assert need(total_q=batch * max_q - 1, **size) <= need(total_q=65536, **size)


def test_sizes_of_nothing_and_out_of_range():
    """The size queries come before any check of the call: no division by a size of zero, nor by a product that wrapped."""
    need = lambda **kw: _lib.load().fg_flash_attn_cache_workspace_bytes(ctypes.byref(params(**kw)))
    for form in (dict(), dict(head_dim=96), dict(softcap=3.0), dict(head_dim=64, max_seqlen_q=30), dict(max_seqlen_q=300)):
        for kw in (dict(batch=0), dict(max_seqlen_q=0), dict(total_q=0), dict(max_seqlen_k=0), dict(batch=0, total_q=0)):
            assert need(**{**form, **kw}) >= 0
        for kw in (dict(total_q=2 ** 62), dict(batch=2 ** 40, total_q=2 ** 40), dict(num_heads=2 ** 40, num_heads_k=2 ** 40),
                   dict(total_q=2 ** 31 - 1, num_heads=2 ** 20, num_heads_k=2 ** 10)):
            assert need(**{**form, **kw}) == 0
            with pytest.raises(RuntimeError, match="too long, or too many rows"):
                _lib.check(_lib.load().fg_flash_attn_cache(ctypes.byref(params(**{**form, **kw})), None))


def test_path_by_sizes():
    path = lambda **kw: _lib.load().fg_flash_attn_cache_path(ctypes.byref(params(**{"max_seqlen_k": 10 ** 5, **kw})))
    assert path(max_seqlen_k=1000) == 2      # too few tiles of keys
    assert path() == 3 and path(max_seqlen_q=4, total_q=16) == 3      # 4 tokens of a group of 4: 16 rows
    assert path(max_seqlen_q=5, total_q=20) == 1 and path(max_seqlen_q=3000, total_q=9000) == 1
    assert path(head_dim=64) == path(head_dim=256) == 3 and path(head_dim=80) == path(head_dim=256, cache_dtype=_lib.FG_BF16) == 2
    assert path(softcap=5.0) == 2 and path(head_dim=72, max_seqlen_q=5, total_q=20) == 0
    assert path(head_dim=64, max_seqlen_q=1000, total_q=4000) == path(head_dim=256, max_seqlen_q=5, total_q=20) == 1
    assert path(head_dim=64, max_seqlen_q=5, total_q=20, max_seqlen_k=600) == 0       # too few tiles for a widened copy
    assert path(block_size=24) == 0 and path(block_size=4) == 0 and path(k_row_stride=264) == 0   # pages or strides TMA cannot take
    assert path(cache_dtype=_lib.FG_BF16, k_row_stride=264, sink_tokens=1, window_left=70000) == 3    # 528 bytes are fine
    assert path(num_heads=400, num_heads_k=2) == 0                    # a group of 200


@pytest.mark.parametrize("match, kw", [("no 8-bit", dict(cache_dtype=_lib.FG_F16)), ("negative", dict(num_tokens=-1)),
                                       ("block_size", dict(block_size=0)), ("null pointer", dict(key=None)),
                                       ("unknown dtype", dict(dtype=7))])
def test_write_refuses_on_the_host(match, kw):
    a = dict(key=0x10000, value=0x10000, kc=0x10000, vc=0x10000, slots=0x10000, ks=None, vs=None, ksh=0, vsh=0, num_tokens=2,
             heads=2, dim=64, block_size=16, blocks=4, kst=128, vst=128, cb=2048, cr=128, ch=64, dtype=_lib.FG_BF16,
             cache_dtype=_lib.FG_E4M3)
    a.update(kw)
    a = [0 if v is None else v for v in a.values()]
    with pytest.raises(RuntimeError, match=match):
        _lib.check(_lib.load().fg_reshape_and_cache_flash_fp8(_lib.CACHE_WRITE.pack(*a), None))


@pytest.mark.parametrize("match, kw", [("hold the type", dict(cache_dtype=_lib.FG_F16)), ("negative", dict(rows=-1)),
                                       ("empty cache", dict(blocks=0)), ("no columns", dict(cols=0)), ("null pointer", dict(cu=None)),
                                       ("unknown dtype", dict(dtype=7, cache_dtype=_lib.FG_E5M2))])
def test_gather_refuses_on_the_host(match, kw):
    a = dict(kc=0x10000, vc=0x10000, key=0x10000, value=0x10000, table=0x10000, cu=0x10000, starts=None, ks=None, vs=None, ksh=0,
             vsh=0, rows=2, batch=1, heads=2, dim=64, block_size=16, blocks=4, tst=4, cols=4, kst=128, vst=128, cb=2048, cr=128,
             ch=64, dtype=_lib.FG_BF16, cache_dtype=_lib.FG_E4M3)
    a.update(kw)
    a = [0 if v is None else v for v in a.values()]
    with pytest.raises(RuntimeError, match=match):
        _lib.check(_lib.load().fg_gather_cache_flash(_lib.CACHE_GATHER.pack(*a), None))


def test_cpu_tensors_are_refused():
    kc = torch.zeros((2, 8, 1, 16), dtype=torch.float8_e4m3fn)
    x = torch.zeros((2, 1, 16), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        fused.reshape_and_cache_flash(x, x, kc, kc, torch.arange(2), "fp8", None, None)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        fused.gather_cache_flash(kc, kc, x, x, torch.zeros((1, 1), dtype=torch.int32), torch.zeros(2, dtype=torch.int32), "fp8")


def span(k_len, p_first, p_last, wl, wr, sinks, bn):
    """The tile runs of attn_cache_common.cuh, restated: tile numbers in the order they are walked."""
    hi = min(k_len, p_last + wr + 1) if wr >= 0 else k_len
    if hi <= 0:
        return []
    lo = max(0, min(hi, p_first - wl)) if wl >= 0 else 0
    win = lo // bn
    sink = min(-(-min(sinks, hi) // bn), win)
    n = sink + -(-hi // bn) - win
    return [i if i < sink else win + i - sink for i in range(n)]


@pytest.mark.parametrize("bn", [4, 8])
def test_tile_runs_cover_what_is_visible_once(bn):
    for k_len in (0, 1, 3, 8, 9, 23, 40):
        for q_len in (1, 2, 7, 12):
            for wl in (-1, 0, 2, 9, 30):
                for wr in (-1, 0, 3):
                    for sinks in (0, 1, 5, 17, 50):
                        first, last = k_len - q_len, k_len - 1
                        tiles = span(k_len, first, last, wl, wr, sinks if wl >= 0 else 0, bn)
                        assert len(set(tiles)) == len(tiles) and all(0 <= t < -(-k_len // bn) for t in tiles)
                        seen = {j // bn for p in range(first, last + 1) for j in range(k_len)
                                if (wr < 0 or j <= p + wr) and (wl < 0 or j >= p - wl or j < sinks)}
                        assert seen <= set(tiles)
                        if wl >= 0:   # no tile outside the window's and the first tokens' own runs
                            assert all(t * bn < sinks or t >= max(0, first - wl) // bn for t in tiles)


def gathered_row(row, cu, starts, table, page, num_blocks):
    """(block, row of the block) that packed row `row` is read from, as the gather kernel finds it; None: not in a sequence."""
    batch, cols = len(table), len(table[0])
    if row < cu[0] or row >= cu[batch]:
        return None
    lo, hi = 0, batch
    while hi - lo > 1:
        mid = (lo + hi) // 2
        lo, hi = (mid, hi) if cu[mid] <= row else (lo, mid)
    pos = max(0, row - cu[lo] + (starts[lo] if starts else 0))
    pg = pos // page
    return min(max(table[lo][min(pg, cols - 1)], 0), num_blocks - 1), pos - pg * page


def test_gather_stays_inside_the_cache():
    """Page numbers outside the cache, positions behind the table and before the sequence, decreasing starts."""
    for cu in ([0, 200, 300], [3, 3, 300], [0, 250, 100], [5, 0, 300]):
        for starts in (None, [-7, 10 ** 9]):
            for row in range(310):
                got = gathered_row(row, cu, starts, [[0, 10 ** 6, 2], [-5, 1, 3]], 16, 4)
                assert got is None or (0 <= got[0] < 4 and 0 <= got[1] < 16)
    assert gathered_row(21, [0, 5, 40], [0, 3], [[9, 9], [2, 1]], 16, 4) == (1, 3)
    assert gathered_row(4, [0, 5, 5, 40], None, [[1], [2], [3]], 16, 4) == (1, 4)


def test_import_without_the_private_stream_binding():
    """A torch build without it still imports the package, and the stream comes from the public call."""
    code = ("import torch; del torch._C._cuda_getCurrentRawStream\n"
            "import flaggems_b200._lib as lib\n"
            "torch.cuda.current_stream = lambda index: type('Stream', (), {'cuda_stream': 40 + index})\n"
            "assert lib.raw_stream(2) == 42")
    root = Path(__file__).resolve().parent.parent
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr

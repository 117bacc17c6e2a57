"""CPU tests of the 4-bit cache: refusals of the C ABI and of the Python functions, the
packed format's arithmetic, and what the attention kernels were compiled to.
"""
from __future__ import annotations

import ctypes
import os
import re
import subprocess

import pytest
import torch

import _kv4_ref as R

A = 1 << 12   # an aligned address that is never followed


def _kv(**over):
    from w4a16 import _lib

    v = dict(pool=A, table=A, pages=8, rows=4, max_pages=4, heads=2, head_dim=128, group_size=64,
             page_size=64)
    v.update(over)
    return _lib.KV4(**v)


def _query(**over):
    from w4a16 import _lib

    v = dict(q=A, q_token=512, q_head=128, out=A, lse=None, lens=A, q_starts=None, seqs=None,
             tokens=4, batch=4, max_q=1, max_context=256, q_heads=4, window=0, scale=0.1, flags=4)
    v.update(over)
    return _lib.KV4Query(**v)


def _rope(**over):
    from w4a16 import _lib

    v = dict(q=A, k=A, v=A, q_token=512, q_head=128, k_token=256, k_head=128, v_token=256,
             v_head=128, q_out=A, k_out=A, cos=A, sin=A, token_position=A, q_weight=None,
             k_weight=None, tokens=3, positions=100, q_heads=4, kv_heads=2, head_dim=128,
             rot_dim=128, eps=1e-6, flags=0)
    v.update(over)
    return _lib.Rope(**v)


def _book(**over):
    from w4a16 import _lib

    v = dict(table=A, lens=A, refs=A, rows=4, max_pages=4, pages=8, page_size=64)
    v.update(over)
    return _lib.KV4Book(**v)


@pytest.mark.parametrize("D,G,P,want", [
    (128, 64, 64, 64 * (32 + 4)), (128, 128, 32, 32 * (32 + 2)), (64, 32, 256, 256 * (16 + 4)),
    (256, 64, 128, 128 * (64 + 8)),
    (96, 32, 64, -2), (128, 16, 64, -3), (128, 256, 64, -3), (256, 32, 64, -3), (128, 48, 64, -3),
    (128, 64, 16, -2), (128, 64, 48, -2), (128, 64, 512, -2),
])
def test_words_of_a_block(lib, D, G, P, want):
    assert lib.w4a16_kv4_words(D, G, P) == want


@pytest.mark.parametrize("kv,q,code", [
    ({}, dict(tokens=0, batch=0), 0),
    ({}, dict(q=None), -1), ({}, dict(out=None), -1), ({}, dict(lens=None), -1),
    (dict(pool=None), {}, -1), (dict(table=None), {}, -1),
    (dict(head_dim=80), {}, -2), (dict(group_size=16), {}, -3), (dict(page_size=33), {}, -2),
    (dict(heads=3), {}, -2),                      # 4 query heads over 3
    (dict(heads=0), {}, -2), (dict(pages=-1), {}, -2), (dict(rows=2**31), {}, -2),
    (dict(heads=60000, page_size=256, head_dim=256), dict(q_heads=60000), -2),   # a page over 4 GiB
    (dict(pool=A + 8), {}, -5), ({}, dict(out=A + 2), -5), ({}, dict(flags=8), -5),
    ({}, dict(batch=3), -2),                      # one token a sequence, without starts
    ({}, dict(tokens=-1), -2), ({}, dict(window=-1), -2), ({}, dict(q_heads=0), -2),
    ({}, dict(scale=0.0), -2), ({}, dict(scale=-1.0), -2), ({}, dict(scale=float("nan")), -2),
    ({}, dict(scale=float("inf")), -2), ({}, dict(max_context=-5), -2),
    (dict(max_pages=1000, heads=1), dict(max_context=60000), -4),   # splits need a workspace
])
def test_attention_refuses(lib, kv, q, code):
    got = lib.w4a16_kv4_attention(ctypes.byref(_kv(**kv)), ctypes.byref(_query(**q)), None, 0, None)
    assert got == code


def test_attention_workspace(lib):
    """Bytes for the splits that a launch makes; none for short contexts; never more
    splits than the join takes."""
    def need(kv, q):
        return lib.w4a16_kv4_attention_workspace_bytes(ctypes.byref(_kv(**kv)),
                                                       ctypes.byref(_query(**q)))

    assert need(dict(max_pages=1), dict(max_context=64)) == 0
    assert need(dict(heads=0), {}) == 0              # a refused call needs none
    one = dict(tokens=1, batch=1, q_heads=1)
    for ctx in (600, 5000, 100000, 2**30):
        b = need(dict(max_pages=2**25, heads=1), dict(max_context=ctx, **one))
        splits, rest = divmod(b, (128 + 2) * 4)
        assert rest == 0 and 2 <= splits <= 256, (ctx, splits)
    ws = need(dict(max_pages=1000, heads=1), dict(max_context=60000))
    k, q = _kv(max_pages=1000, heads=1), _query(max_context=60000)
    assert lib.w4a16_kv4_attention(ctypes.byref(k), ctypes.byref(q), A, ws - 1, None) == -4
    assert lib.w4a16_kv4_attention(ctypes.byref(k), ctypes.byref(q), A + 16, ws, None) == -5


@pytest.mark.parametrize("over,code", [
    (dict(tokens=0), 0), (dict(q=None), -1), (dict(k=None), -1), (dict(cos=None), -1),
    (dict(token_position=None), -1), (dict(q_out=None), -1),
    (dict(head_dim=96), -2), (dict(rot_dim=24), -2), (dict(rot_dim=144), -2), (dict(tokens=-1), -2),
    (dict(tokens=2**30), -2), (dict(q_heads=-1), -2), (dict(flags=4), -5), (dict(q_out=A + 8), -5),
])
def test_rope_refuses(lib, over, code):
    r = _rope(**over)
    more = _rope(**{**over, "k_out": None})
    assert lib.w4a16_qk_norm_rope(ctypes.byref(r), None) == code
    assert lib.w4a16_kv4_append(ctypes.byref(more), ctypes.byref(_kv()), None, None) == code


def test_append_and_read_refuse(lib):
    call = lib.w4a16_kv4_append
    assert call(ctypes.byref(_rope(v=None)), ctypes.byref(_kv()), None, None) == -1
    assert call(ctypes.byref(_rope(kv_heads=1)), ctypes.byref(_kv()), None, None) == -2
    assert call(ctypes.byref(_rope()), ctypes.byref(_kv(head_dim=64, group_size=32)), None, None) == -2
    assert call(None, ctypes.byref(_kv()), None, None) == -1
    assert lib.w4a16_qk_norm_rope(ctypes.byref(_rope(k_out=None)), None) == -1
    read = lib.w4a16_kv4_read
    assert read(ctypes.byref(_kv()), A, None, 0, None, None, 0, None) == 0
    assert read(ctypes.byref(_kv()), None, None, 2, A, A, 0, None) == -1
    assert read(ctypes.byref(_kv()), A, None, 2, A, None, 0, None) == -1
    assert read(ctypes.byref(_kv()), A, None, 2**31, A, A, 0, None) == -2
    assert read(ctypes.byref(_kv()), A, None, 2, A + 8, A, 0, None) == -5
    assert read(ctypes.byref(_kv()), A, None, 2, A, A, 2, None) == -5
    assert read(None, A, None, 2, A, A, 0, None) == -1


def test_page_calls_refuse(lib):
    b = ctypes.byref
    words = 2 * 2304
    assert lib.w4a16_kv4_copy_pages(A, 1, 8, words, A, A, 0, None) == 0
    assert lib.w4a16_kv4_copy_pages(A, 1, 8, words, None, A, 1, None) == -1
    assert lib.w4a16_kv4_copy_pages(None, 1, 8, words, A, A, 1, None) == -1
    assert lib.w4a16_kv4_copy_pages(A, 1, 8, words + 2, A, A, 1, None) == -2
    assert lib.w4a16_kv4_copy_pages(A, 1, 8, words, A, A, -1, None) == -2
    assert lib.w4a16_kv4_copy_pages(A, 1, 8, words, A, A, 2**21, None) == -2
    assert lib.w4a16_kv4_copy_pages(A + 4, 1, 8, words, A, A, 1, None) == -5
    assert lib.w4a16_kv4_extend(b(_book()), A, A, 0, A, None) == 0
    assert lib.w4a16_kv4_extend(b(_book()), A, A, 1, None, None) == -1
    assert lib.w4a16_kv4_extend(b(_book(page_size=40)), A, A, 1, A, None) == -2
    assert lib.w4a16_kv4_extend(b(_book(lens=None)), A, A, 1, A, None) == -1
    assert lib.w4a16_kv4_extend(None, A, A, 1, A, None) == -1
    assert lib.w4a16_kv4_free(b(_book()), None, 1, None) == -1
    assert lib.w4a16_kv4_free(b(_book(refs=None)), A, 1, None) == -1
    assert lib.w4a16_kv4_free(b(_book()), A, 0, None) == 0
    need = lib.w4a16_kv4_fork_workspace_bytes(3)
    assert need >= 3 * 8 and lib.w4a16_kv4_fork_workspace_bytes(0) == 0
    fork = lib.w4a16_kv4_fork
    assert fork(A, 1, words, b(_book()), A, A, 0, A, None, 0, None) == 0
    assert fork(A, 1, words, b(_book()), A, A, 3, A, A, need - 1, None) == -4
    assert fork(A, 1, words, b(_book()), A, A, 3, A, None, need, None) == -4
    assert fork(A, 1, words, b(_book()), A, None, 3, A, A, need, None) == -1
    assert fork(A, -1, words, b(_book()), A, A, 3, A, A, need, None) == -2
    need = lib.w4a16_kv4_compact_workspace_bytes(8)
    compact = lib.w4a16_kv4_compact
    assert compact(A, 1, words, b(_book()), 2 * A, 2 * A, A, A, need - 1, None) == -4
    assert compact(A, 1, words, b(_book()), A, 2 * A, A, A, need, None) == -5     # in place
    assert compact(A, 1, words, b(_book()), 2 * A, A, A, A, need, None) == -5
    assert compact(A, 1, words, b(_book()), None, 2 * A, A, A, need, None) == -1
    assert compact(A, 1, words, b(_book(pages=0)), 2 * A, 2 * A, A, A, need, None) == -2


def test_python_functions_check_their_arguments():
    """AssertionError before any device work."""
    import w4a16 as w

    q = torch.zeros(2, 4, 128, dtype=torch.float16)
    pool = torch.zeros(3, 2, 64 * 36, dtype=torch.int32)
    i32 = torch.zeros(2, dtype=torch.int32)
    table = torch.zeros(2, 2, dtype=torch.int32)
    cos = torch.zeros(8, 64)
    calls = [
        lambda: w.kv4_attention(q, pool, table, i32),
        lambda: w.qk_norm_rope(q, q, cos, cos, i32),
        lambda: w.kv4_append(q, q, q, cos, cos, i32, pool, table),
        lambda: w.kv4_read(pool, table, i32, head_dim=128),
        lambda: w.kv4_copy_pages(pool, i32, i32),
        lambda: w.kv4_extend(table, i32, i32, i32, i32, page_size=64),
        lambda: w.kv4_fork(pool, table, i32, i32, i32, i32, page_size=64),
        lambda: w.kv4_free(table, i32, i32, i32),
        lambda: w.kv4_compact(pool, table, i32),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(AssertionError):
            call()
    for bad in ((96, 32, 64), (128, 16, 64), (128, 64, 48)):
        with pytest.raises(AssertionError):
            w.kv4_words(*bad)
        with pytest.raises(AssertionError):
            w.KV4Cache(1, 1, 1, bad[0], sequences=1, max_pages=1, group_size=bad[1],
                       page_size=bad[2], device="cpu")
    assert w.kv4_words(128, 64, 64) == R.words(128, 64, 64)
    with pytest.raises(ValueError):
        w.W4A16Attention(256, 3, 2, 64)


def test_the_format_round_trips():
    """Packing by code and group, then reading back by the word's formulas."""
    g = torch.Generator().manual_seed(0)
    for D, G, P in ((64, 32, 32), (128, 64, 32)):
        x = torch.randn(2, P, D, generator=g)
        parts = [R.quantise(t, G) for t in x]
        block = R.pack(*parts[0], *parts[1], D, G, P)
        assert block.numel() == R.words(D, G, P)
        for t, got, (c, s, z) in zip(x, R.unpack(block, D, G, P), parts):
            s, z = (v.double().repeat_interleave(G, -1) for v in (s, z))
            assert torch.equal(got, (c - 8) * s + z)
            assert ((got - t).abs() <= 0.52 * s + 2.0**-10 * z.abs()).all()


def test_attention_kernels_do_not_spill(tmp_path):
    """The loop's counted waits take every vector memory load for one of its own: a
    spill to memory would be counted with them."""
    from w4a16 import _build

    try:
        hipcc = _build.hipcc()
    except RuntimeError:
        pytest.skip("hipcc not available")
    seen = 0
    for src in ("kv4_attn_tokens1.hip", "kv4_attn_tokens2.hip", "kv4_attn_rows.hip"):
        out = str(tmp_path / (src + ".s"))
        r = subprocess.run([hipcc, *_build.COMMON_FLAGS, *_build.SOURCE_FLAGS.get(src, []),
                            "--cuda-device-only", "-S", "-x", "hip",
                            os.path.join(_build.CSRC, src), "-o", out],
                           capture_output=True, text=True)
        assert r.returncode == 0, r.stderr
        text = open(out).read()
        sizes = re.findall(r"\.private_segment_fixed_size:\s+(\d+)", text)
        assert sizes and set(sizes) == {"0"}, (src, sizes)
        assert "scratch_" not in re.sub(r";.*", "", text).replace(".amdhsa", ""), src
        seen += len(sizes)
    assert seen >= 8 + 5 + 8

"""GPU tests of the 4-bit paged cache: storing, reading, attending, paging.

Storing is held to its definition bit for bit (an fp32 evaluation in the defined
order) and to the formulas in 64 bits; attention to fp64 within a bound derived
from the one rounding it makes (weights of the values to fp16), its fp32 scores and
the output's own rounding; page calls exactly.
"""
from __future__ import annotations

import math

import pytest
import torch

import _kv4_ref as R
from _helpers import DEV, log

pytestmark = pytest.mark.gpu

ULP = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}   # half an ulp, relative


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _tables(rows, max_pages, pages, lens, P, seed):
    """A table over shuffled pages, -1 beyond."""
    order = torch.randperm(pages, generator=_gen(seed)).to(torch.int32)
    table = torch.full((rows, max_pages), -1, dtype=torch.int32)
    at = 0
    for r, n in enumerate(lens):
        held = -(-n // P)
        table[r, :held] = order[at:at + held]
        at += held
    assert at <= pages
    return table


def _rotation(positions, R_, seed=0):
    half = R_ // 2
    a = torch.arange(positions, dtype=torch.float64)[:, None] * \
        10000.0 ** (-torch.arange(half, dtype=torch.float64) / half)
    return a.cos().float(), a.sin().float()


# ---- storing ---------------------------------------------------------------------

ROPE = [
    # D, G, P, Hq, Hkv, rot, norm, interleaved, dtype
    (128, 64, 64, 8, 2, 128, True, False, torch.float16),
    (128, 32, 32, 4, 4, 64, True, True, torch.bfloat16),
    (128, 128, 128, 4, 1, 96, False, False, torch.float16),
    (64, 32, 32, 6, 3, 64, True, False, torch.bfloat16),
    (64, 64, 256, 2, 2, 16, True, True, torch.float16),
    (256, 64, 64, 4, 1, 256, True, False, torch.float16),
    (256, 256, 32, 2, 1, 128, False, True, torch.bfloat16),
]


def _qkv(T, Hq, Hkv, D, dtype, seed, layout):
    g = _gen(seed)
    x = torch.randn(T, Hq + 2 * Hkv, D, generator=g) * torch.exp(
        torch.randn(1, Hq + 2 * Hkv, D, generator=g))
    x = x.to(dtype)
    if layout == "fused":            # slices of a fused projection
        x = x.to(DEV)
    elif layout == "odd":            # rows off 16 bytes
        wide = torch.zeros(T, (Hq + 2 * Hkv) * D + 3, dtype=dtype, device=DEV)
        wide[:, 1:-2] = x.to(DEV).view(T, -1)
        x = wide[:, 1:-2].unflatten(1, (-1, D))
    else:                            # heads outermost
        x = x.transpose(0, 1).contiguous().to(DEV).transpose(0, 1)
    return x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]


@pytest.mark.parametrize("layout", ["fused", "odd", "heads"])
@pytest.mark.parametrize("case", ROPE, ids=lambda c: "-".join(map(str, c)))
def test_append_stores_the_defined_bits(case, layout):
    from w4a16 import kv4_append, kv4_read, qk_norm_rope

    D, G, P, Hq, Hkv, rot, norm, inter, dtype = case
    log(f"append {case} {layout}")
    # prompts from the start and from inside an octet, single tokens, a skipped one
    spans = [(0, 0, 70), (1, 3, 9), (2, 40, 41), (3, P - 1, P + 2)]
    tok = [(r, p) for r, a, b in spans for p in range(a, b)]
    lens = [b for _, _, b in spans]
    T = len(tok) + 2
    rows = torch.tensor([r for r, _ in tok] + [2, 77], dtype=torch.int32)
    pos = torch.tensor([p for _, p in tok] + [-1, 5], dtype=torch.int32)   # neither is stored
    q, k, v = _qkv(T, Hq, Hkv, D, dtype, 5, layout)
    cos, sin = _rotation(300, rot)
    wq, wk = ((torch.rand(D, generator=_gen(6)) + 0.5).to(dtype) if norm else None
              for _ in range(2))
    pages = 24
    table = _tables(4, 9, pages, lens, P, 7)
    g = _gen(8)
    before = torch.randint(-2**31, 2**31 - 1, (pages, Hkv, R.words(D, G, P)), generator=g,
                           dtype=torch.int32)
    pool = before.to(DEV)
    dev = dict(cos=cos.to(DEV), sin=sin.to(DEV), positions=pos.to(DEV))
    how = dict(q_weight=None if wq is None else wq.to(DEV),
               k_weight=None if wk is None else wk.to(DEV), eps=1e-5, interleaved=inter)
    qo = kv4_append(q, k, v, dev["cos"], dev["sin"], dev["positions"], pool, table.to(DEV),
                    rows=rows.to(DEV), group_size=G, **how)
    qd, kd = qk_norm_rope(q, k, dev["cos"], dev["sin"], dev["positions"], **how)
    rk, rv = kv4_read(pool, table.to(DEV), dev["positions"], rows=rows.to(DEV), head_dim=D,
                      group_size=G, dtype=dtype)
    torch.cuda.synchronize()
    args = (cos, sin, pos.clamp(min=0), 1e-5, inter)
    q32, k32 = (R.norm_rotate32(x.cpu(), w, *args) for x, w in ((q, wq), (k, wk)))
    good = pos >= 0
    assert torch.equal(qo.cpu()[good], q32.to(dtype)[good])
    assert torch.isnan(qo.cpu()[~good].float()).all()
    assert torch.equal(qd.cpu()[good], q32.to(dtype)[good])
    assert torch.equal(kd.cpu()[good], k32.to(dtype)[good])
    q64 = R.norm_rotate64(q.cpu(), wq, *args)
    off = (qo.cpu().double() - q64)[good].abs()
    assert (off <= 1.01 * ULP[dtype] * q64[good].abs() + 2e-6 * q64[good].abs().max()).all()
    # the pool: stored tokens by the definition, everything else as it was
    (kc, ks, kz), (vc, vs, vz) = R.quantise(k32, G), R.quantise(v.cpu(), G)
    after = pool.cpu()
    want_k, want_v = torch.zeros(2, T, Hkv, D, dtype=torch.float64)
    for page in range(pages):
        for h in range(Hkv):
            got, old = (R.unpack(x[page, h], D, G, P, parts=True) for x in (after, before))
            mine = [(i, int(pos[i]) % P) for i in range(T - 2)
                    if table[rows[i], pos[i] // P] == page]
            for side, (codes, s, c) in enumerate(((kc, ks, kz), (vc, vs, vz))):
                want = [x.clone() for x in old[side]]
                for i, t in mine:
                    want[0][t] = codes[i, h]
                    want[1][t] = s[i, h].double().repeat_interleave(G)
                    want[2][t] = c[i, h].double().repeat_interleave(G)
                for x, y, name in zip(got[side], want, ("codes", "scales", "centres")):
                    assert torch.equal(torch.nan_to_num(x), torch.nan_to_num(y)), \
                        (page, h, side, name)
                for i, t in mine:
                    (want_k, want_v)[side][i, h] = (want[0][t] - 8) * want[1][t] + want[2][t]
    assert torch.equal(rk.cpu(), want_k.float().to(dtype))   # (product and sum are exact in fp32
    assert torch.equal(rv.cpu(), want_v.float().to(dtype))   # but for one rounding)
    # and the stored values are within half a step of the formula's
    for got, x, s in ((want_k, R.norm_rotate64(k.cpu(), wk, *args), ks), (want_v, v.cpu().double(), vs)):
        step = s.double().repeat_interleave(G, -1)
        n = T - 2
        c = (kz if got is want_k else vz).double().repeat_interleave(G, -1)
        assert ((got - x)[:n].abs() <= (0.52 * step + 2.0**-10 * c.abs() + 1e-6 * x.abs())[:n]).all()


def test_append_one_token_or_all_together():
    """The same tokens stored one call each, out of order, leave the same pool."""
    from w4a16 import kv4_append

    D, G, P, H, T = 128, 64, 32, 2, 45
    q, k, v = _qkv(T, 4, H, D, torch.float16, 3, "fused")
    cos, sin = (x.to(DEV) for x in _rotation(64, D))
    w = torch.rand(D, generator=_gen(1)).half().to(DEV)
    table = torch.tensor([[3, 1]], dtype=torch.int32, device=DEV)
    pos = torch.arange(T, dtype=torch.int32, device=DEV)
    row = torch.zeros(T, dtype=torch.int32, device=DEV)
    pools = [torch.zeros(4, H, R.words(D, G, P), dtype=torch.int32, device=DEV) for _ in range(3)]
    how = dict(q_weight=w, k_weight=w)
    outs = [kv4_append(q, k, v, cos, sin, pos, pools[0], table, rows=row, **how)]
    one = torch.empty_like(outs[0])
    for i in torch.randperm(T, generator=_gen(2)).tolist():
        s = slice(i, i + 1)
        one[s] = kv4_append(q[s], k[s], v[s], cos, sin, pos[s], pools[1], table, rows=row[s], **how)
    mix = torch.randperm(T, generator=_gen(4)).to(DEV)
    kv4_append(q[mix], k[mix], v[mix], cos, sin, pos[mix], pools[2], table, rows=row, **how)
    assert torch.equal(outs[0], one)
    assert torch.equal(pools[0], pools[1]) and torch.equal(pools[0], pools[2])


@pytest.mark.parametrize("T", [700, 2500])
def test_append_long_prompts(T):
    """Both chunk lengths of the value workgroups, over many pages and heads."""
    from w4a16 import kv4_append, kv4_read

    D, G, P, H = 64, 32, 64, 8
    q, k, v = _qkv(T, 8, H, D, torch.float16, 3, "fused")
    cos, sin = (x.to(DEV) for x in _rotation(T + 5, D))
    pages = T // P + 2
    table = torch.randperm(pages, generator=_gen(5)).to(torch.int32)[None].to(DEV)
    pos = torch.arange(5, T + 5, dtype=torch.int32, device=DEV)
    row = torch.zeros(T, dtype=torch.int32, device=DEV)
    pool = torch.full((pages, H, R.words(D, G, P)), -1, dtype=torch.int32, device=DEV)
    kv4_append(q, k, v, cos, sin, pos, pool, table, rows=row, group_size=G)
    rk, rv = kv4_read(pool, table, pos, rows=row, head_dim=D, group_size=G)
    kf = R.norm_rotate32(k.cpu(), None, cos.cpu(), sin.cpu(), pos.cpu(), 1e-6, False)
    for got, x in ((rk, kf), (rv, v.cpu())):
        c, s, z = R.quantise(x, G)
        want = (c - 8).float() * s.float().repeat_interleave(G, -1) + \
            z.float().repeat_interleave(G, -1)
        assert torch.equal(got.cpu(), want.half())


def test_append_special_values():
    """Constant, zero and non-finite groups; other groups and tokens keep their values."""
    from w4a16 import kv4_append, kv4_read

    D, G, P = 64, 32, 32
    x = torch.randn(6, 1, D, generator=_gen(1)).half()
    x[0] = 0.0
    x[1, 0, :G] = 3.25
    x[2, 0, 5] = float("nan")
    x[3, 0, 40] = float("inf")
    x[4, 0, :G] = 6e-8          # a range that fp16 scales cannot tell from none
    x[5, 0, :G] = torch.linspace(-65504, 65504, G).half()
    x = x.to(DEV)
    cos, sin = torch.ones(8, D // 2, device=DEV), torch.zeros(8, D // 2, device=DEV)
    pool = torch.zeros(1, 1, R.words(D, G, P), dtype=torch.int32, device=DEV)
    table = torch.zeros(1, 1, dtype=torch.int32, device=DEV)
    pos = torch.arange(6, dtype=torch.int32, device=DEV)
    row = torch.zeros(6, dtype=torch.int32, device=DEV)
    kv4_append(x, x, x, cos, sin, pos, pool, table, rows=row, group_size=G)
    k, v = kv4_read(pool, table, pos, rows=row, head_dim=D, group_size=G)
    # (a rotation by nothing still multiplies a partner by 0: keys spread NaN to it)
    turned = R.norm_rotate32(x.cpu(), None, cos.cpu(), sin.cpu(), pos.cpu(), 1e-6, False)
    for got, src in ((k, turned), (v, x.cpu().float())):
        c, s, z = R.quantise(src, G)
        want = ((c - 8).float() * s.float().repeat_interleave(G, -1)
                + z.float().repeat_interleave(G, -1)).half()
        assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
        assert torch.equal(torch.nan_to_num(got.cpu()), torch.nan_to_num(want))
    assert (k[0] == 0).all() and (v[0] == 0).all() and (v[1, 0, :G] == 3.25).all()
    assert torch.isnan(v[2, 0, :G]).all() and torch.isfinite(v[2, 0, G:]).all()
    assert torch.isnan(v[3, 0, G:]).all() and torch.isfinite(v[3, 0, :G]).all()


def test_append_outside_the_rotation_tables():
    """A position that the cos / sin tables do not hold gives NaN, loudly."""
    from w4a16 import qk_norm_rope

    q = torch.ones(3, 2, 64, dtype=torch.float16, device=DEV)
    cos, sin = (x.to(DEV) for x in _rotation(4, 32))
    pos = torch.tensor([3, 4, -1], dtype=torch.int32, device=DEV)
    for inter in (False, True):
        a, b = qk_norm_rope(q, q[:, :1], cos, sin, pos, interleaved=inter)
        assert torch.isfinite(a[0]).all() and torch.isnan(a[1:]).all()
        assert torch.isfinite(b[0]).all() and torch.isnan(b[1:]).all()


# ---- attention ---------------------------------------------------------------------

def _random_pool(pages, H, D, G, P, seed, wide=False):
    g = _gen(seed)
    pool = torch.randint(-2**31, 2**31 - 1, (pages, H, R.words(D, G, P)), generator=g,
                         dtype=torch.int32)
    NG, a, c = D // G, P * D // 8, P * D // 4 + (D // G) * P
    for at, size in ((a, 0.15), (c, 0.3)):
        s = torch.rand(pages, H, NG * P, generator=g) * size + 0.01
        if wide:   # scales of very unlike size from token to token
            s = s * torch.exp(4 * torch.randn(pages, H, NG * P, generator=g)).clamp(1e-4, 300)
        z = torch.randn(pages, H, NG * P, generator=g) * 0.5
        w = torch.stack((s, z), -1).half().view(torch.int32).squeeze(-1)
        pool[:, :, at:at + NG * P] = w
    return pool


def _check_attention(q, pool, table, lens, D, G, P, out, lse=None, starts=None, seqs=None,
                     scale=None, causal=True, window=0, what=""):
    dtype = q.dtype
    H, Hq = pool.shape[1], q.shape[1]
    scale = 1 / math.sqrt(D) if scale is None else scale
    batch = len(starts) - 1 if starts is not None else q.shape[0]
    out, q = out.cpu().double(), q.cpu()
    for b in range(batch):
        row = b if seqs is None else seqs[b]
        lo, hi = (starts[b], starts[b + 1]) if starts is not None else (b, b + 1)
        n = lens[row]
        held = [int(p) for p in table[row, :-(-n // P)]]
        for h in range(H):
            parts = [R.unpack(pool[p, h], D, G, P, parts=True) for p in held]
            mine = slice(h * (Hq // H), (h + 1) * (Hq // H))
            if parts:
                (kc, ks, kz), (vc, vs, vz) = (
                    [torch.cat([x[side][j] for x in parts])[:n] for j in range(3)]
                    for side in range(2))
                k, v = (kc - 8) * ks + kz, (vc - 8) * vs + vz
                res, sizes = ((vc - 8) * vs).abs(), 8 * ks + kz.abs()
            else:
                k = v = res = sizes = torch.zeros(0, D, dtype=torch.float64)
            ref, rl, err = R.attention(q[lo:hi, mine], k, v, res, n, scale, causal, window, sizes)
            got = out[lo:hi, mine]
            bound = 1.01 * (ULP[dtype] * (ref.abs() + err) + err) + 1e-7
            bad = ~((got - ref).abs() <= bound)
            assert not bad.any(), (what, b, h, int(bad.sum()), float((got - ref).abs().max()),
                                   float(((got - ref).abs() / bound).max()))
            if lse is not None:
                gl = lse[lo:hi, mine].cpu().double()
                assert torch.equal(torch.isinf(gl), torch.isinf(rl)), (what, b, h)
                fin = torch.isfinite(rl)
                assert ((gl - rl)[fin].abs() <= 1e-4 + 1e-5 * rl[fin].abs()).all(), (what, b, h)


SHAPES = [
    # D, G, P, Hq, H, dtype
    (128, 64, 64, 8, 2, torch.float16),
    (128, 128, 32, 16, 1, torch.bfloat16),
    (128, 32, 128, 3, 3, torch.float16),
    (64, 64, 32, 8, 1, torch.float16),
    (64, 32, 256, 4, 2, torch.bfloat16),
    (256, 64, 64, 4, 1, torch.float16),
    (256, 128, 32, 2, 2, torch.bfloat16),
    (256, 256, 32, 20, 1, torch.float16),
]


@pytest.mark.parametrize("shape", SHAPES, ids=lambda c: "-".join(map(str, c)))
def test_attention_single_tokens(shape):
    """One token a sequence: every length from none to a few pages, lse, seqs, window."""
    from w4a16 import kv4_attention

    D, G, P, Hq, H, dtype = shape
    lens = [0, 1, 31, 32, 33, P, P + 1, 2 * P + 17, 700]
    pages = sum(-(-n // P) for n in lens) + 1
    table = _tables(len(lens), -(-700 // P) + 1, pages, lens, P, 1)
    pool = _random_pool(pages, H, D, G, P, 2)
    q = (torch.randn(len(lens), Hq, D, generator=_gen(3)) * 2).to(dtype)
    dev = [x.to(DEV) for x in (q, pool, table, torch.tensor(lens, dtype=torch.int32))]
    log(f"attention {shape}")
    out, lse = kv4_attention(*dev, group_size=G, return_lse=True)
    _check_attention(q, pool, table, lens, D, G, P, out, lse, what="plain")
    assert (out[0] == 0).all() and torch.isinf(lse[0]).all()
    for window in (1, 40):
        out = kv4_attention(*dev, group_size=G, window=window, max_context=64)
        _check_attention(q, pool, table, lens, D, G, P, out, window=window, what=f"window {window}")
    seqs = [8, 2, 2, 0]
    out = kv4_attention(dev[0][:4], *dev[1:], group_size=G, scale=0.01,
                        seqs=torch.tensor(seqs, dtype=torch.int32, device=DEV))
    _check_attention(q[:4], pool, table, lens, D, G, P, out, seqs=seqs, scale=0.01, what="seqs")


@pytest.mark.parametrize("causal,window", [(True, 0), (True, 19), (False, 0), (False, 33)])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda c: "-".join(map(str, c)))
def test_attention_many_tokens(shape, causal, window):
    """Ragged numbers of new tokens: drafts, prompts, more than the context holds."""
    from w4a16 import kv4_attention

    D, G, P, Hq, H, dtype = shape
    nq = [5, 0, 1, 70, 9, 3]
    lens = [45, 20, 333, 100, 4, 0]      # rows 4 and 5: some or all queries see nothing
    starts = [0]
    for a in nq:
        starts.append(starts[-1] + a)
    pages = sum(-(-n // P) for n in lens) + 1
    table = _tables(6, -(-333 // P), pages, lens, P, 4)
    pool = _random_pool(pages, H, D, G, P, 5)
    q = (torch.randn(starts[-1], Hq, D, generator=_gen(6)) * 2).to(dtype)
    dev = [x.to(DEV) for x in (q, pool, table, torch.tensor(lens, dtype=torch.int32))]
    st = torch.tensor(starts, dtype=torch.int32, device=DEV)
    log(f"attention tokens {shape} {causal} {window}")
    out, lse = kv4_attention(*dev, q_starts=st, group_size=G, causal=causal, window=window,
                             return_lse=True)
    _check_attention(q, pool, table, lens, D, G, P, out, lse, starts, causal=causal, window=window,
                     what="all")
    # only the short ones, so that few rows a head take the forms for few rows
    few = [0, 2, 5]
    st2 = torch.tensor([0, 5, 6, 9], dtype=torch.int32, device=DEV)
    q2 = torch.cat([q[starts[i]:starts[i + 1]] for i in few])
    for max_q in (5, None):
        out = kv4_attention(q2.to(DEV), *dev[1:], q_starts=st2, group_size=G, causal=causal,
                            window=window, max_q=max_q, max_context=333,
                            seqs=torch.tensor(few, dtype=torch.int32, device=DEV))
        _check_attention(q2, pool, table, lens, D, G, P, out, starts=[0, 5, 6, 9], seqs=few,
                         causal=causal, window=window, what=f"few {max_q}")


@pytest.mark.parametrize("nq", [1, 4])
@pytest.mark.parametrize("D,G,dtype", [(128, 128, torch.float16), (128, 64, torch.bfloat16),
                                       (128, 32, torch.float16), (64, 64, torch.bfloat16),
                                       (64, 32, torch.float16)])
def test_attention_few_blocks_for_eight_waves(D, G, dtype, nq):
    """Contexts of 17 blocks and a few more, which one workgroup takes whole, and rows
    shorter and longer than was said."""
    from w4a16 import kv4_attention

    P, Hq, H = 64, 8, 2
    said = 560 if D == 128 else 1100
    lens = [said, 4, 33, 257, said + 300, 512]
    pages = sum(-(-n // P) for n in lens)
    table = _tables(len(lens), max(-(-n // P) for n in lens), pages, lens, P, 41)
    pool = _random_pool(pages, H, D, G, P, 42)
    T = nq * len(lens)
    q = (torch.randn(T, Hq, D, generator=_gen(43)) * 2).to(dtype)
    starts = list(range(0, T + 1, nq))
    dev = [x.to(DEV) for x in (q, pool, table, torch.tensor(lens, dtype=torch.int32))]
    how = dict(q_starts=torch.tensor(starts, dtype=torch.int32, device=DEV), max_q=nq) if nq > 1 else {}
    for window in (0, 530):
        out, lse = kv4_attention(*dev, group_size=G, max_context=said, window=window,
                                 return_lse=True, **how)
        _check_attention(q, pool, table, lens, D, G, P, out, lse, starts, window=window,
                         what=f"window {window}")
        again = kv4_attention(*dev, group_size=G, max_context=said, window=window, **how)
        assert torch.equal(out, again)


@pytest.mark.parametrize("D,G,Hq,H,nq", [(128, 64, 4, 1, 1), (64, 64, 2, 2, 40), (256, 64, 6, 2, 5)])
def test_attention_long_and_split(D, G, Hq, H, nq):
    """A context over which the work is split, value scales of very unlike sizes."""
    from w4a16 import kv4_attention

    P, n = 64, 9000
    pages = -(-n // P)
    table = _tables(1, pages + 2, pages, [n], P, 7)
    pool = _random_pool(pages, H, D, G, P, 8, wide=True)
    q = torch.randn(nq, Hq, D, generator=_gen(9)).half()
    st = [0, nq]
    out, lse = kv4_attention(q.to(DEV), pool.to(DEV), table.to(DEV),
                             torch.tensor([n], dtype=torch.int32, device=DEV),
                             q_starts=torch.tensor(st, dtype=torch.int32, device=DEV),
                             group_size=G, return_lse=True, scale=0.02)
    _check_attention(q, pool, table, [n], D, G, P, out, lse, st, scale=0.02, what="long")


def test_attention_one_token_holds_all_the_weight():
    """Small value scales at the token that counts, large ones where nothing does:
    weights keep their precision over the whole range of fp16 scales."""
    from w4a16 import kv4_attention

    D = G = 64
    P, n = 32, 64
    kc = torch.full((n, D), 8)
    kc[17] = 15
    vc = torch.randint(0, 16, (n, D), generator=_gen(1))
    ks = torch.ones(n, 1)
    vs = torch.full((n, 1), 1000.0)
    vs[17] = 1e-3
    zero = torch.zeros(n, 1)
    pool = torch.stack([R.pack(kc[i:i + P], ks[i:i + P], zero[i:i + P], vc[i:i + P], vs[i:i + P],
                               zero[i:i + P], D, G, P) for i in (0, P)])[:, None]
    q = torch.full((1, 1, D), 3.0).half()      # score of token 17: 21 * 64 / 8 = 168
    table = torch.tensor([[0, 1]], dtype=torch.int32)
    out = kv4_attention(q.to(DEV), pool.to(DEV), table.to(DEV),
                        torch.tensor([n], dtype=torch.int32, device=DEV), group_size=G)
    _check_attention(q, pool, table, [n], D, G, P, out, what="one token")


@pytest.mark.parametrize("size", [2.0**-24, 1e-6, 1.0, 6e4])
def test_attention_any_size_of_query(size):
    """Queries from subnormal to the largest keep their precision."""
    from w4a16 import kv4_attention

    D, G, P, n = 128, 64, 32, 77
    pool = _random_pool(3, 1, D, G, P, 8)
    q = (torch.randn(1, 4, D, generator=_gen(9)).clamp(-1, 1) * size).half()
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32)
    scale = min(0.3 / size, 1e6)
    out = kv4_attention(q.to(DEV), pool.to(DEV), table.to(DEV),
                        torch.tensor([n], dtype=torch.int32, device=DEV), group_size=G, scale=scale)
    _check_attention(q, pool, table, [n], D, G, P, out, scale=scale, what=str(size))


@pytest.mark.parametrize("shape", SHAPES[:4], ids=lambda c: "-".join(map(str, c)))
def test_attention_one_large_query_value(shape):
    """A query value far above the others leaves the others' products their precision:
    scores of single tokens (lse) and of many."""
    from w4a16 import kv4_attention

    D, G, P, Hq, H, dtype = shape
    lens = [1] * 40 + [500]
    pages = 41 + -(-500 // P)
    table = _tables(len(lens), -(-500 // P), pages, lens, P, 31)
    pool = _random_pool(pages, H, D, G, P, 32)
    q = torch.randn(len(lens), Hq, D, generator=_gen(33))
    q[:, :, 5::32] = 64.0
    q = q.to(dtype)
    out, lse = kv4_attention(q.to(DEV), pool.to(DEV), table.to(DEV),
                             torch.tensor(lens, dtype=torch.int32, device=DEV), group_size=G,
                             return_lse=True)
    _check_attention(q, pool, table, lens, D, G, P, out, lse, what="one large")


def _nan_meta(pool, D, G, P, page, tokens):
    """NaN and infinite scales and centres at tokens of a page (all heads)."""
    NG, a, c = D // G, P * D // 8, P * D // 4 + (D // G) * P
    for at in (a, c):
        for g in range(NG):
            for i, t in enumerate(tokens):
                pool[page, :, at + g * P + t] = (0x7E007E00, 0x7C007C00, -0x03FF0400)[i % 3]


@pytest.mark.parametrize("nq", [1, 20, 90])
def test_attention_garbage_in_hidden_places(nq):
    """NaN and infinities behind the last token, before the window and after a
    query's own position reach nobody."""
    from w4a16 import kv4_attention

    D, G, P, H, Hq, n, window = 128, 64, 64, 2, 4, 150, 30
    lens = [n]
    pool = _random_pool(4, H, D, G, P, 11)
    table = torch.tensor([[3, 0, 2, -1]], dtype=torch.int32)
    q = torch.randn(nq, Hq, D, generator=_gen(12)).half()
    st = torch.tensor([0, nq], dtype=torch.int32, device=DEV)
    ln = torch.tensor(lens, dtype=torch.int32, device=DEV)

    def run(p):
        return kv4_attention(q.to(DEV), p.to(DEV), table.to(DEV), ln, q_starts=st, group_size=G,
                             window=window)

    want = run(pool)
    _check_attention(q, pool, table, lens, D, G, P, want, starts=[0, nq], window=window, what="clean")
    dirty = pool.clone()
    _nan_meta(dirty, D, G, P, 2, range(n - 2 * P, P))              # behind the end
    _nan_meta(dirty, D, G, P, 3, range(0, max(0, min(P, n - nq - window + 1))))
    _nan_meta(dirty, D, G, P, 1, range(P))                        # a page of nobody
    assert torch.equal(run(dirty), want)
    if nq > 1:
        # the last token hidden from every query but the last
        _nan_meta(dirty, D, G, P, 2, [n - 1 - 2 * P])
        got = run(dirty)
        assert torch.equal(got[:-1], want[:-1]) and torch.isnan(got[-1]).any()


def test_attention_missing_pages_are_hidden():
    from w4a16 import kv4_attention

    D, G, P = 64, 64, 32
    pool = _random_pool(3, 1, D, G, P, 1).to(DEV)
    q = torch.randn(1, 2, D, generator=_gen(2)).half().to(DEV)
    ln = torch.tensor([96], dtype=torch.int32, device=DEV)
    a = kv4_attention(q, pool, torch.tensor([[0, -1, 2]], dtype=torch.int32, device=DEV), ln,
                      group_size=G)
    b = kv4_attention(q, pool, torch.tensor([[0, 99, 2]], dtype=torch.int32, device=DEV), ln,
                      group_size=G)
    c = kv4_attention(q, pool, torch.tensor([[0, 2, 1]], dtype=torch.int32, device=DEV),
                      torch.tensor([64], dtype=torch.int32, device=DEV), group_size=G)
    assert torch.equal(a, b)
    assert (a.double() - c.double()).abs().max() <= 2.0**-10 * c.abs().max().double()


def test_attention_strided_and_unaligned_queries():
    from w4a16 import kv4_attention

    D, G, P = 128, 64, 32
    pool = _random_pool(3, 2, D, G, P, 1).to(DEV)
    table = torch.tensor([[0, 1, 2]], dtype=torch.int32, device=DEV)
    ln = torch.tensor([80], dtype=torch.int32, device=DEV)
    q = torch.randn(1, 4, D, generator=_gen(2)).half().to(DEV)
    want = kv4_attention(q, pool, table, ln, group_size=G)
    wide = torch.zeros(1, 4, D + 5, dtype=torch.float16, device=DEV)
    wide[:, :, 3:-2] = q
    assert torch.equal(kv4_attention(wide[:, :, 3:-2], pool, table, ln, group_size=G), want)
    out = torch.empty_like(want)
    assert kv4_attention(q, pool, table, ln, group_size=G, out=out) is out
    assert torch.equal(out, want)


def test_attention_pool_beyond_32_bits():
    """Pages beyond 2^31 words from the pool's start."""
    from w4a16 import kv4_append, kv4_attention, kv4_read

    D, G, P, H = 128, 32, 256, 16
    words = R.words(D, G, P)
    pages = (2**31 + 2**27) // (H * words)
    pool = torch.empty(pages, H, words, dtype=torch.int32, device=DEV)
    small = torch.zeros(2, H, words, dtype=torch.int32, device=DEV)
    T = 300
    q, k, v = _qkv(T, H, H, D, torch.float16, 3, "fused")
    cos, sin = (x.to(DEV) for x in _rotation(T, D))
    pos = torch.arange(T, dtype=torch.int32, device=DEV)
    row = torch.zeros(T, dtype=torch.int32, device=DEV)
    far = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32, device=DEV)
    near = torch.tensor([[0, 1]], dtype=torch.int32, device=DEV)
    ln = torch.tensor([T], dtype=torch.int32, device=DEV)
    res = []
    for p, t in ((pool, far), (small, near)):
        x = kv4_append(q, k, v, cos, sin, pos, p, t, rows=row, group_size=G)
        res.append((x, *kv4_read(p, t, pos, rows=row, head_dim=D, group_size=G),
                    kv4_attention(x[-1:], p, t, ln, group_size=G)))
    for a, b in zip(*res):
        assert torch.equal(a, b)


def test_attention_on_another_stream_and_in_a_graph():
    """A captured step of append and attention replays to the eager results; a side
    stream gives the same."""
    from w4a16 import kv4_append, kv4_attention

    D, G, P, H, Hq, B, n = 128, 64, 64, 2, 8, 3, 2000
    pages = B * (-(-n // P))
    table = _tables(B, -(-n // P), pages, [n] * B, P, 1).to(DEV)
    pool0 = _random_pool(pages, H, D, G, P, 2).to(DEV)
    cos, sin = (x.to(DEV) for x in _rotation(n, D))
    pos = torch.full((B,), n - 1, dtype=torch.int32, device=DEV)
    ln = torch.full((B,), n, dtype=torch.int32, device=DEV)
    qkv = torch.empty(B, Hq + 2 * H, D, dtype=torch.float16, device=DEV)
    pool = pool0.clone()

    def step():
        q = kv4_append(qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:], cos, sin, pos, pool, table,
                       group_size=G)
        return kv4_attention(q, pool, table, ln, group_size=G)

    inputs = [torch.randn(B, Hq + 2 * H, D, generator=_gen(20 + i)).half().to(DEV) for i in range(4)]
    want = []
    for x in inputs:
        qkv.copy_(x)
        want.append(step().clone())
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        qkv.copy_(inputs[1])
        assert torch.equal(step(), want[1])
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = step()
    for i in (2, 0, 3, 1):
        qkv.copy_(inputs[i])
        g.replay()
        assert torch.equal(y, want[i])
        torch.cuda.synchronize()
        qkv.copy_(inputs[3 - i])
        assert torch.equal(step(), want[3 - i])


# ---- pages ---------------------------------------------------------------------

def _book(rows, max_pages, pages, P, lens, seed):
    table = _tables(rows, max_pages, pages, lens, P, seed)
    refs = torch.zeros(pages, dtype=torch.int32)
    refs[table[table >= 0].long()] = 1
    full = torch.zeros(rows, dtype=torch.int32)
    full[:len(lens)] = torch.tensor(lens, dtype=torch.int32)
    return table, full, refs


@pytest.mark.parametrize("pages", [40, 5000])
def test_extend_takes_the_lowest_free_pages(pages):
    from w4a16 import KV4Cache, kv4_extend

    P, rows, most = 32, 9, 20
    table, lens, refs = _book(rows, most, pages, P, [40, 0, 64, 33], 1)
    refs[:7] += 1 - refs[:7].clamp(max=1)    # the first pages held by someone
    seqs, counts = [3, 1, 0, 5, 2], [31, 100, 24, 1, 0]
    d = [x.to(DEV) for x in (table, lens, refs)]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)   # noqa: E731
    status = kv4_extend(*d, i32(seqs), i32(counts), page_size=P)
    for r, c in zip(seqs, counts):
        have, want = -(-int(lens[r]) // P), -(-(int(lens[r]) + c) // P)
        for k in range(have, want):
            page = int((refs == 0).nonzero()[0])
            table[r, k], refs[page] = page, 1
        lens[r] += c
    for got, want in zip(d, (table, lens, refs)):
        assert torch.equal(got.cpu(), want)
    assert int(status) == 0
    # a full row, a row that is none, a pool that runs out: those rows stay
    big = [most * P, 1, 2]
    status = kv4_extend(*d, i32([0, 77, 4]), i32(big), page_size=P)
    assert int(status) == KV4Cache.ROW_FULL | KV4Cache.BAD_ROW
    page = int((refs == 0).nonzero()[0])
    table[4, 0], refs[page], lens[4] = page, 1, 2
    for got, want in zip(d, (table, lens, refs)):
        assert torch.equal(got.cpu(), want)
    d[2].fill_(1)
    d[2][3] = 0                                # one page left, two asked for
    status = kv4_extend(*d, i32([6, 7]), i32([33, 5]), page_size=P)
    assert int(status) == KV4Cache.NO_PAGES
    assert torch.equal(d[0].cpu(), table) and torch.equal(d[1].cpu(), lens)
    assert int((d[2] == 0).sum()) == 1


def test_extend_many_rows():
    """More rows than the counting workgroup has threads."""
    from w4a16 import kv4_extend

    P, rows, pages = 32, 2500, 9000
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)   # noqa: E731
    table = torch.full((rows, 4), -1, dtype=torch.int32, device=DEV)
    lens, refs = torch.zeros(rows, dtype=torch.int32, device=DEV), torch.zeros(pages, dtype=torch.int32, device=DEV)
    counts = [(i * 37) % 129 for i in range(rows)]
    status = kv4_extend(table, lens, refs, i32(list(range(rows))), i32(counts), page_size=P)
    need = [-(-c // P) for c in counts]
    flat = table[table >= 0].cpu()
    assert int(status) == 0 and torch.equal(flat, torch.arange(sum(need), dtype=torch.int32))
    assert (table >= 0).sum(1).cpu().tolist() == need and lens.cpu().tolist() == counts
    assert torch.equal(refs.cpu(), (torch.arange(pages) < sum(need)).int())


@pytest.mark.parametrize("layers", [1, 3])
def test_fork_shares_whole_pages_and_copies_the_last(layers):
    from w4a16 import KV4Cache, kv4_attention, kv4_fork, kv4_free

    P, D, G, H, pages, rows, most = 32, 64, 64, 2, 24, 8, 6
    lens = [70, 64, 0, 5]
    table, ln, refs = _book(rows, most, pages, P, lens, 2)
    pool = torch.stack([_random_pool(pages, H, D, G, P, 30 + i) for i in range(layers)])
    parents, children = [0, 1, 0, 2, 3], [4, 5, 6, 7, 3]      # the last child is in use
    d = [x.to(DEV) for x in (pool if layers > 1 else pool[0], table, ln, refs)]
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)   # noqa: E731
    status = kv4_fork(*d, i32(parents), i32(children), page_size=P)
    assert int(status) == KV4Cache.BAD_ROW
    for p, c in list(zip(parents, children))[:-1]:
        whole = lens[p] // P
        table[c, :whole] = table[p, :whole]
        refs[table[c, :whole].long()] += 1
        if lens[p] % P:
            page = int((refs == 0).nonzero()[0])
            table[c, whole], refs[page] = page, 1
            pool[:, page] = pool[:, table[p, whole]]
        ln[c] = lens[p]
    got = [x.cpu() for x in d]
    assert torch.equal(got[0].view(pool.shape), pool)
    for x, want in zip(got[1:], (table, ln, refs)):
        assert torch.equal(x, want)
    q = torch.randn(rows, 4, D, generator=_gen(3)).half().to(DEV)
    q[4:7] = q[[0, 1, 0]]
    y = kv4_attention(q, d[0] if layers == 1 else d[0][0], *d[1:3], group_size=G)
    assert torch.equal(y[4:7], y[[0, 1, 0]])
    # freeing the parents leaves the children whole; a row named twice counts once
    kv4_free(*d[1:], i32([0, 1, 0, 99, -1, 2]))
    for r in (0, 1):
        for p in table[r][table[r] >= 0].tolist():
            refs[p] -= 1
        table[r], ln[r] = -1, 0
    for x, want in zip([x.cpu() for x in d[1:]], (table, ln, refs)):
        assert torch.equal(x, want)
    z = kv4_attention(q, d[0] if layers == 1 else d[0][0], *d[1:3], group_size=G)
    assert torch.equal(z[4:7], y[4:7]) and (z[:3] == 0).all()
    # no free page: the child stays empty
    d[3].fill_(1)
    status = kv4_fork(*d, i32([4]), i32([0]), page_size=P)
    assert int(status) == KV4Cache.NO_PAGES and int(d[2][0]) == 0 and (d[1][0] == -1).all()


@pytest.mark.parametrize("pages,share", [(1, 1.0), (33, 0.5), (2500, 0.3), (2500, 0.9), (64, 0.0)])
def test_compact_moves_pages_to_the_front(pages, share):
    from w4a16 import kv4_compact

    rows, most = 5, pages
    g = _gen(pages)
    refs = (torch.rand(pages, generator=g) < share).int() * torch.randint(1, 4, (pages,), generator=g).int()
    used = refs.nonzero().flatten()
    table = torch.full((rows, most), -1, dtype=torch.int32)
    for i, p in enumerate(used.tolist()):
        table[i % rows, i // rows] = p
    pool = torch.randint(-2**31, 2**31 - 1, (2, pages, 3, 256), generator=g, dtype=torch.int32)
    dp = pool.to(DEV)
    t, r, live = kv4_compact(dp, table.to(DEV), refs.to(DEV))
    n = len(used)
    src = [p for p in used.tolist() if p >= n]
    dst = [p for p in range(n) if refs[p] == 0]
    to = torch.arange(pages, dtype=torch.int32)
    want_r = torch.where(torch.arange(pages) < n, refs, 0)
    for a, b in zip(src, dst):
        pool[:, b], to[a], want_r[b] = pool[:, a], b, refs[a]
    assert int(live) == n and torch.equal(r.cpu(), want_r)
    assert torch.equal(t.cpu(), torch.where(table >= 0, to[table.clamp(min=0).long()], -1))
    assert torch.equal(dp.cpu(), pool)


def test_copy_pages():
    from w4a16 import kv4_copy_pages

    pool = torch.randint(-2**31, 2**31 - 1, (3, 20, 5, 1028), generator=_gen(1), dtype=torch.int32)
    d = pool.to(DEV)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)   # noqa: E731
    kv4_copy_pages(d, i32([3, 3, 7, -1, 20, 2]), i32([5, 0, 19, 4, 1, 20]))
    for a, b in ((3, 5), (3, 0), (7, 19)):
        pool[:, b] = pool[:, a]
    assert torch.equal(d.cpu(), pool)
    kv4_copy_pages(d[1], i32([]), i32([]))
    kv4_copy_pages(d[1], i32([2]), i32([9]))
    pool[1, 9] = pool[1, 2]
    assert torch.equal(d.cpu(), pool)


# ---- together --------------------------------------------------------------------

def test_layer_prefill_decode_fork_compact():
    """W4A16Attention over a KV4Cache: prompts, decode steps, a fork and a compaction
    give what a dense evaluation of the same stored tokens gives."""
    from w4a16 import KV4Cache, W4A16Attention, kv4_read

    torch.manual_seed(0)
    hidden, Hq, H, D, P = 512, 4, 2, 128, 32
    lin = [torch.nn.Linear(hidden, (Hq + 2 * H) * D, bias=False).half().to(DEV),
           torch.nn.Linear(Hq * D, hidden, bias=False).half().to(DEV)]
    from w4a16 import W4A16Linear

    layer = W4A16Attention(hidden, Hq, H, D, device=DEV)
    layer.qkv, layer.out = (W4A16Linear.from_linear(x) for x in lin)
    layer.q_norm.mul_(1.5)
    cache = KV4Cache(1, 40, H, D, sequences=6, max_pages=8, page_size=P, device=DEV)
    cos, sin = (x.to(DEV) for x in _rotation(256, D))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)   # noqa: E731

    def step(rows, counts, seed, lens):
        """lens: tokens before."""
        T = sum(counts)
        x = torch.randn(T, hidden, generator=_gen(seed)).half().to(DEV)
        pos = i32([lens[r] + j for r, c in zip(rows, counts) for j in range(c)])
        of = i32([r for r, c in zip(rows, counts) for _ in range(c)])
        starts = [0]
        for c in counts:
            starts.append(starts[-1] + c)
        cache.extend(i32(rows), i32(counts))
        y = layer(x, cache, pos, cos, sin, rows=of, q_starts=i32(starts), seqs=i32(rows),
                  max_q=max(counts))
        for r, c in zip(rows, counts):
            lens[r] += c
        cache.check()
        assert cache.lens.cpu().tolist() == [lens.get(r, 0) for r in range(6)]
        # the same from the stored tokens, dense, in fp64
        qkv = layer.qkv(x).view(T, Hq + 2 * H, D)
        q = R.norm_rotate32(qkv[:, :Hq].cpu(), layer.q_norm.cpu(), cos.cpu(), sin.cpu(), pos.cpu(),
                            layer.eps, False).half()
        att = torch.zeros(T, Hq, D, dtype=torch.float64)
        for b, r in enumerate(rows):
            n = lens[r]
            at = i32(range(n))
            k, v = kv4_read(cache.pool[0], cache.table, at, rows=torch.full_like(at, r), head_dim=D,
                            dtype=torch.float16)
            for h in range(H):
                kk, vv = k[:, h].cpu().double(), v[:, h].cpu().double()
                att[starts[b]:starts[b + 1], 2 * h:2 * h + 2] = R.attention(
                    q[starts[b]:starts[b + 1], 2 * h:2 * h + 2], kk, vv, vv.abs(), n,
                    1 / math.sqrt(D), True, 0, kk.abs())[0]
        want = layer.out(att.half().to(DEV).view(T, -1))
        off = (y.double() - want.double()).norm() / want.double().norm()
        # the read values are rounded to fp16 (2^-11 each, keys and values), the
        # attention's output twice, its weights once
        assert off < 5 * 2.0**-11, float(off)
        return y

    lens: dict[int, int] = {}
    lens.update({0: 0, 1: 0, 2: 0})
    step([0, 1, 2], [70, 33, 5], 1, lens)
    step([2, 0, 1], [1, 1, 1], 2, lens)
    cache.fork(i32([0, 0]), i32([3, 4]))
    lens[3] = lens[4] = lens[0]
    step([0, 3, 4], [1, 1, 1], 3, lens)
    cache.free(i32([1, 0]))
    lens[0] = lens[1] = 0
    live = int(cache.compact())
    used = cache.table[cache.table >= 0]
    assert live == len(used.unique()) and int(used.max()) == live - 1
    step([3, 2, 4, 0], [2, 1, 1, 40], 4, lens)


def test_decode_step_in_a_graph():
    """Extending, storing and attending captured once and replayed, with eager work in
    between, fill a cache as eager steps do; pages are taken as they are needed."""
    from w4a16 import KV4Cache

    H, Hq, D, P, B = 2, 4, 64, 32, 3
    cos, sin = (x.to(DEV) for x in _rotation(256, D))
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)   # noqa: E731
    rows = i32([4, 0, 2])
    ones = i32([1] * B)
    qkv = torch.empty(B, Hq + 2 * H, D, dtype=torch.float16, device=DEV)
    inputs = [torch.randn(qkv.shape, generator=_gen(i)).half().to(DEV) for i in range(40)]

    def make():
        c = KV4Cache(2, 12, H, D, sequences=5, max_pages=4, page_size=P, group_size=32, device=DEV)
        return c, torch.zeros(B, dtype=torch.int32, device=DEV)

    def step(c, pos):
        c.extend(rows, ones)
        y = None
        for layer in range(2):
            q = c.append(layer, qkv[:, :Hq], qkv[:, Hq:Hq + H], qkv[:, Hq + H:], cos, sin, pos, rows)
            y = c.attend(layer, q, seqs=rows, max_context=128)
        pos += 1
        return y

    eager, pos = make()
    want = []
    for x in inputs:
        qkv.copy_(x)
        want.append(step(eager, pos).clone())
    cache, pos = make()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = step(cache, pos)
    for i, x in enumerate(inputs):
        qkv.copy_(x)
        g.replay()
        assert torch.equal(y, want[i]), i
        if i % 7 == 0:
            torch.cuda.synchronize()
            eager.attend(0, qkv[:, :Hq], seqs=rows)
    cache.check()
    for a, b in ((cache.pool, eager.pool), (cache.table, eager.table), (cache.lens, eager.lens),
                 (cache.refs, eager.refs)):
        assert torch.equal(a, b)


def test_python_and_native_calls_agree():
    """A given output takes the Python path, none the native one: the same bits."""
    from w4a16 import kv4_append, kv4_attention, qk_norm_rope

    D, G, P, H, Hq, T = 128, 32, 32, 2, 6, 11
    q, k, v = _qkv(T, Hq, H, D, torch.bfloat16, 3, "heads")
    cos, sin = (x.to(DEV) for x in _rotation(64, 64))
    w = torch.rand(D, generator=_gen(1)).bfloat16().to(DEV)
    pos = torch.arange(T, dtype=torch.int32, device=DEV)
    row = torch.zeros(T, dtype=torch.int32, device=DEV)
    table = torch.tensor([[1, 0]], dtype=torch.int32, device=DEV)
    pools = [torch.zeros(2, H, R.words(D, G, P), dtype=torch.int32, device=DEV) for _ in range(2)]
    how = dict(q_weight=w, k_weight=w, interleaved=True)
    a = qk_norm_rope(q, k, cos, sin, pos, **how)
    b = qk_norm_rope(q, k, cos, sin, pos, out=tuple(torch.empty_like(x) for x in a), **how)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    qa = kv4_append(q, k, v, cos, sin, pos, pools[0], table, rows=row, group_size=G, **how)
    qb = kv4_append(q, k, v, cos, sin, pos, pools[1], table, rows=row, group_size=G,
                    out=torch.empty_like(qa), **how)
    assert torch.equal(qa, qb) and torch.equal(*pools)
    ln = torch.tensor([T], dtype=torch.int32, device=DEV)
    st = torch.tensor([0, T], dtype=torch.int32, device=DEV)
    for n in (dict(q_starts=st), dict(q_starts=st, window=3, causal=False, scale=0.2)):
        ya = kv4_attention(qa, pools[0], table, ln, group_size=G, **n)
        yb = kv4_attention(qa, pools[0], table, ln, group_size=G, out=torch.empty_like(qa), **n)
        assert torch.equal(ya, yb)


def test_refusals_on_the_device():
    """What the kernels do not take is refused before anything is launched."""
    import w4a16 as w

    D, P = 128, 32
    q = torch.zeros(2, 4, D, dtype=torch.float16, device=DEV)
    k = torch.zeros(2, 2, D, dtype=torch.float16, device=DEV)
    pool = torch.zeros(3, 2, R.words(D, 64, P), dtype=torch.int32, device=DEV)
    table = torch.zeros(2, 3, dtype=torch.int32, device=DEV)
    i32 = torch.zeros(2, dtype=torch.int32, device=DEV)
    cos = torch.zeros(8, 32, device=DEV)
    status = torch.zeros(1, dtype=torch.int32, device=DEV)
    refs = torch.zeros(3, dtype=torch.int32, device=DEV)
    long = i32.long()
    bad = [
        lambda: w.kv4_attention(q.float(), pool, table, i32),
        lambda: w.kv4_attention(q[:, :3], pool, table, i32),               # heads
        lambda: w.kv4_attention(q, pool, table, i32, group_size=32),       # another pool
        lambda: w.kv4_attention(q, pool, table.long(), i32),
        lambda: w.kv4_attention(q, pool, table, long),
        lambda: w.kv4_attention(q, pool, table, i32[:1]),
        lambda: w.kv4_attention(q, pool, table, i32, window=-1),
        lambda: w.kv4_attention(q, pool, table, i32, scale=0.0),
        lambda: w.kv4_attention(q, pool, table, i32, seqs=i32[:1]),
        lambda: w.kv4_attention(torch.cat((q, q)), pool, table, i32),      # rows
        lambda: w.kv4_attention(q.transpose(1, 2), pool, table, i32),
        lambda: w.kv4_attention(q, pool, table, i32, out=q.float()),
        lambda: w.kv4_attention(q, pool.cpu(), table, i32),
        lambda: w.kv4_append(q, k, k[:, :1], cos, cos, i32, pool, table),
        lambda: w.kv4_append(q, k.bfloat16(), k, cos, cos, i32, pool, table),
        lambda: w.kv4_append(q, k, k, cos, cos[:4], i32, pool, table),
        lambda: w.kv4_append(q, k, k, cos.half(), cos, i32, pool, table),
        lambda: w.kv4_append(q, k, k, cos, cos, long, pool, table),
        lambda: w.kv4_append(q, k, k, cos, cos, i32, pool[:, :1].contiguous(), table),
        lambda: w.kv4_append(q, k, k, cos, cos, i32, pool, table, rows=i32[:1]),
        lambda: w.kv4_append(q, k, k, cos, cos, i32, pool, table, q_weight=cos[0]),
        lambda: w.qk_norm_rope(q, k, cos[:, :5].contiguous(), cos[:, :5].contiguous(), i32),
        lambda: w.kv4_read(pool, table, i32, head_dim=D, dtype=torch.float32),
        lambda: w.kv4_read(pool, table, i32, head_dim=256),
        lambda: w.kv4_fork(pool, table, i32, refs[:2], i32, i32, page_size=P, status=status),
        lambda: w.kv4_fork(pool, table, i32, refs, i32, i32[:1], page_size=P, status=status),
        lambda: w.kv4_fork(pool, table, i32, refs, i32, i32, page_size=P, status=long[:1]),
        lambda: w.kv4_extend(table, i32, refs, i32, i32, page_size=48, status=status),
        lambda: w.kv4_free(table, i32, refs, long),
        lambda: w.kv4_compact(pool, table, refs[:2]),
        lambda: w.kv4_copy_pages(pool[:, :, :-4], i32, i32),
        lambda: w.kv4_copy_pages(pool, i32, i32[:1]),
    ]
    for i, call in enumerate(bad):
        with pytest.raises((AssertionError, RuntimeError)):
            call()
            print("not refused:", i)
    # nothing of no tokens or no sequences is an error
    none = q[:0]
    assert w.kv4_attention(none, pool, table, i32).shape == (0, 4, D)
    assert w.kv4_append(none, k[:0], k[:0], cos, cos, i32[:0], pool, table).shape == (0, 4, D)
    assert w.kv4_read(pool, table, i32[:0], head_dim=D)[0].shape == (0, 2, D)
    w.kv4_free(table, i32, refs, i32[:0])
    w.kv4_copy_pages(pool, i32[:0], i32[:0])

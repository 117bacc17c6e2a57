"""The operators around a 4-bit paged key / value cache, as measurable cases.

Imported with the repository's root as the working folder.  A case is a dict of
plain values; ``prepare`` makes what a serving program holds before the call,
``run`` is one pass (in elementary torch operations, or through ``w4a16`` where
``own`` is true), ``exact`` the same result in 64 bits, ``work`` the bytes and
operations of one pass.

Case fields:
  op      "append"  rotate and norm new queries and keys, store keys and values
                    in 4 bits (kv4_append), and read the stored tokens back
                    (kv4_read)
          "rotate"  norm and rotate queries and keys, no cache (qk_norm_rope)
          "attend"  attention over the stored tokens (kv4_attention)
          "fork"    drop the rows of dead beams, fork live ones into them
                    (kv4_free, kv4_fork)
          "compact" move the live pages of a pool to its front (kv4_compact)
  B       sequences; pad: how many more rows of the batch are empty
  q       new tokens of the longest sequence; ctx: its length, those included
          (shorter ones follow a fixed spread, see _spread)
  Hq, Hkv query and key / value heads; D values a head; G values a quantised
          group; P tokens a page
  dtype   "fp16" or "bf16", of queries, keys and values
  norm    whether heads are normed; R: rotated values of a head; inter: whether
          neighbours rotate together (else halves)
  window  how many of the last positions a query sees (0: all)
  L       layers whose pages move together; pages: pages of the pool

Format of a pool, int32 [layers, pages, Hkv, words], one block of words for a
page and head: key codes, key groups, value codes, value groups.
  value of a code: (code - 8) * scale + centre, per token and group of G
  group word:  [D / G, P], scale in the low 16 bits, centre in the high (fp16)
  key codes:   [P, D / 8]: values 8o..8o+7 in the word (D / 32) * (o % 4) + o // 4
  value codes: [P / 8, D]: eight tokens of value d in the word 64 * (d // 64)
               + 4 * (d % 16) + d // 16 % 4
  the i-th of eight codes in a word lies in bits [4n, 4n + 4), n = i // 2 + 4 * (i % 2)
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_DEVICE = "cuda:0"
_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-6
_HEADS = dict(Hq=32, Hkv=8, D=128, G=64, P=64)


def _package():
    pkg = os.path.join(os.getcwd(), "w4a16-dequant-fused-matmul-kernel_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import w4a16

    return w4a16


def listed() -> list[dict]:
    """Twelve cases: storing, rotating, attending and moving pages."""
    return [
        # one new token of one sequence: all launch and latency (the heads of a
        # 4096 x 6144 fused projection)
        dict(name="append_token", op="append", B=1, q=1, ctx=1001, **_HEADS, R=128, norm=True,
             inter=False, dtype="fp16"),
        # a decode step of many sequences, other rotation and type
        dict(name="append_batch", op="append", B=96, q=1, ctx=16384, Hq=32, Hkv=8, D=128, G=32,
             P=32, R=128, norm=True, inter=True, dtype="bf16"),
        # prompts packed into one batch, one of them continued from the middle
        # of a page
        dict(name="append_prompt", op="append", B=3, q=4097, ctx=5003, Hq=64, Hkv=8, D=128, G=64,
             P=64, R=128, norm=True, inter=False, dtype="fp16"),
        # a prompt's queries and keys for attention that keeps no cache, half
        # of each head rotated
        dict(name="rotate_prompt", op="rotate", B=1, q=4095, ctx=4095, Hq=32, Hkv=32, D=64, R=32,
             norm=False, inter=False, dtype="bf16"),
        # one token of one sequence over a short cache
        dict(name="attend_token", op="attend", B=1, pad=0, q=1, ctx=1000, **_HEADS, window=0,
             dtype="fp16"),
        # a decode step of a served batch, its last rows empty
        dict(name="attend_batch", op="attend", B=46, pad=2, q=1, ctx=8192, **_HEADS, window=0,
             dtype="fp16"),
        # few long contexts: the cache no longer fits any on-chip memory
        dict(name="attend_long", op="attend", B=3, pad=0, q=1, ctx=131071, Hq=64, Hkv=8, D=128,
             G=128, P=128, window=0, dtype="bf16"),
        # drafted tokens checked together, a window over their context, as many
        # key heads as query heads
        dict(name="attend_draft", op="attend", B=16, pad=0, q=7, ctx=4099, Hq=16, Hkv=16, D=64,
             G=32, P=32, window=1000, dtype="fp16"),
        # prompts on top of a cached part
        dict(name="attend_prompt", op="attend", B=2, pad=0, q=2048, ctx=4000, **_HEADS, window=0,
             dtype="fp16"),
        # one sequence forked: all launch and latency
        dict(name="fork_one", op="fork", B=1, q=1, ctx=333, L=2, pages=64, Hkv=8, D=128, G=64,
             P=64),
        # a beam step over a whole model: half the rows dropped, half forked
        dict(name="fork_beams", op="fork", B=32, q=32, ctx=2049, L=32, pages=2100, Hkv=8, D=128,
             G=64, P=64),
        # half of a pool's pages freed all over it, the rest moved together
        dict(name="compact_pool", op="compact", B=24, q=0, ctx=2000, L=32, pages=1000, Hkv=8,
             D=128, G=64, P=64),
    ]


def _log(rng, lo: float, hi: float) -> int:
    return max(int(lo), min(int(hi), round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _draw_one(rng) -> dict:
    op = rng.choice(("append", "append", "rotate", "attend", "attend", "attend", "attend", "fork",
                     "compact"))
    D = rng.choice((64, 128, 128, 128, 256))
    heads = dict(D=D, G=rng.choice([g for g in (32, 64, 128) if g <= D <= 4 * g]),
                 P=rng.choice((32, 64, 128)))
    Hkv = rng.choice((1, 2, 4, 8, 8, 16))
    Hq = Hkv * rng.choice((1, 2, 4, 4, 8))
    dtype = rng.choice(("fp16", "fp16", "bf16"))
    if op in ("fork", "compact"):
        B = _log(rng, 1, 48)
        ctx = _log(rng, 40, 6000)
        case = dict(op=op, B=B, q=rng.randint(1, B) if op == "fork" else 0, ctx=ctx,
                    L=_log(rng, 1, 40), pages=0, Hkv=Hkv, **heads)
        need = sum(-(-n // case["P"]) for n in _spread(B, ctx))
        case["pages"] = int(need * rng.uniform(1.1, 2.5)) + 2 * B + 1
        return case
    kind = rng.choice(("token", "batch", "batch", "draft", "prompt"))
    B = {"token": 1, "batch": _log(rng, 2, 128), "draft": _log(rng, 1, 32),
         "prompt": rng.randint(1, 4)}[kind]
    q = {"token": 1, "batch": 1, "draft": rng.randint(2, 8), "prompt": _log(rng, 9, 4097)}[kind]
    ctx = q + _log(rng, 1, 131070 if B <= 4 and q < 9 else 8191)
    if op == "attend":
        return dict(op=op, B=B, pad=rng.choice((0, 0, 1)), q=q, ctx=ctx, Hq=Hq, Hkv=Hkv, **heads,
                    window=rng.choice((0, 0, 0, _log(rng, 16, 4096))), dtype=dtype)
    more = dict(R=rng.choice((D, D, D // 2)), norm=rng.random() < 0.7, inter=rng.random() < 0.3,
                dtype=dtype)
    if op == "rotate":
        return dict(op=op, B=1, q=q * B, ctx=q * B + rng.randint(0, 1000), Hq=Hq, Hkv=Hkv, D=D,
                    **more)
    return dict(op=op, B=B, q=q, ctx=ctx, Hq=Hq, Hkv=Hkv, **heads, **more)


def draw(rng) -> dict:
    """One more case of the listed ones' ranges: every operator, 1 to 128
    sequences, 1 to 4097 new tokens, contexts to 131071, and no more work than
    the largest listed case of its operator."""
    most = {}
    for c in listed():
        w, m = work(c), most.setdefault(c["op"], dict(bytes=0, flops=0))
        most[c["op"]] = {k: max(w[k], m[k]) for k in w}
    while True:
        case = _draw_one(rng)
        w = work(case)
        if all(w[k] <= most[case["op"]][k] for k in w):
            # the scores that the plain form holds at once, in 32 bits
            if case["op"] != "attend" or (case["B"] + case["pad"]) * case["Hq"] * case["q"] \
                    * case["ctx"] <= 1 << 30:
                return case


# ---- lengths ---------------------------------------------------------------

def _spread(n: int, top: int, low: int = 1) -> list[int]:
    """n lengths in [low, top], the first of them top: steps of the golden ratio."""
    return [top if i == 0 else low + int((top - low) * ((i * 0.6180339887498949) % 1.0))
            for i in range(n)]


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """(new tokens, length with them) of every sequence, empty rows last."""
    q = _spread(case["B"], case["q"])
    if case["op"] == "append" and case["q"] > 8:
        # whole prompts but the first
        n = [case["ctx"] if i == 0 else t for i, t in enumerate(q)]
    else:
        n = [max(a, b) for a, b in zip(_spread(case["B"], case["ctx"]), q)]
    pad = case.get("pad", 0)
    return q + [1] * pad, n + [0] * pad


def _live_pages(case: dict) -> list[int]:
    return [-(-n // case["P"]) for n in _spread(case["B"], case["ctx"])]


def _page_words(case: dict) -> int:
    """Words of one page in one layer."""
    D, G = case["D"], case["G"]
    return case["Hkv"] * case["P"] * (D // 4 + 2 * (D // G))


def work(case: dict) -> dict:
    op = case["op"]
    if op == "fork":
        # partial pages copied: read and written
        copies = sum(n % case["P"] != 0 for n in _forked(case)[2])
        return dict(bytes=8 * case["L"] * _page_words(case) * copies + 8 * case["pages"], flops=0)
    if op == "compact":
        # each moved page read and written; as many pages lie beyond the live
        # ones as the share of the pool that is free
        live = sum(_live_pages(case))
        moved = live * (case["pages"] - live) // case["pages"]
        return dict(bytes=8 * case["L"] * _page_words(case) * moved + 8 * case["pages"], flops=0)
    q, n = _lengths(case)
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    T = sum(q)
    if op == "rotate":
        return dict(bytes=4 * T * (Hq + Hkv) * D + 4 * T * case["R"], flops=8 * T * (Hq + Hkv) * D)
    token = 2 * Hkv * (D // 2 + 4 * (D // case["G"]))   # bytes of one stored token
    if op == "append":
        return dict(bytes=2 * T * (Hq + 2 * Hkv) * D + 2 * T * Hq * D + T * token
                    + 4 * T * Hkv * D + 4 * T * case["R"], flops=20 * T * (Hq + 2 * Hkv) * D)
    pairs = read = 0
    for a, b in zip(q, n):
        if not b:
            continue
        w = case["window"] or b
        read += min(b, a + w - 1)
        first = b - a + 1                    # keys that the first new token sees
        if first >= w:
            pairs += a * w
        else:
            whole = min(a, w - first)        # queries that see less than the window
            pairs += whole * first + whole * (whole - 1) // 2 + (a - whole) * w
    return dict(bytes=read * token + 4 * T * Hq * D, flops=4 * pairs * Hq * D)


# ---- the packed format ------------------------------------------------------

def _groups(x: torch.Tensor, G: int):
    """(codes, scales, centres) of x [..., D] fp32, in groups of G along D."""
    g = x.reshape(*x.shape[:-1], -1, G)
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    s = ((hi - lo) / 15.0).to(torch.float16).float()
    c = (lo + 8.0 * s).to(torch.float16).float()
    inv = 1.0 / s
    ok = torch.isfinite(inv) & torch.isfinite(c) & (s < math.inf)
    code = torch.where(ok, ((g - c) * inv).round().clamp(-8, 7), torch.zeros_like(g)) + 8
    return (code.reshape(x.shape).to(torch.int32), s.squeeze(-1).to(torch.float16),
            c.squeeze(-1).to(torch.float16))


_NIBBLE = [4 * (i // 2 + 4 * (i % 2)) for i in range(8)]   # first bit of the i-th code


def _words(codes: torch.Tensor) -> torch.Tensor:
    """int32 codes [..., 8] to words [...]."""
    shift = torch.tensor(_NIBBLE, dtype=torch.int32, device=codes.device)
    return (codes << shift).sum(-1, dtype=torch.int32)


def _octet_order(D: int, device) -> torch.Tensor:
    """Which octet of a key lies in each word of its row."""
    w = torch.arange(D // 8, device=device)
    return (w % (D // 32)) * 4 + w // (D // 32)


def _value_order(D: int, device) -> torch.Tensor:
    """In which word of its row each value lies."""
    d = torch.arange(D, device=device)
    return 64 * (d // 64) + 4 * (d % 16) + d // 16 % 4


def _group_words(s: torch.Tensor, c: torch.Tensor) -> torch.Tensor:
    return torch.stack((s, c), -1).view(torch.int32).squeeze(-1)


def _pack(k: torch.Tensor, v: torch.Tensor, G: int) -> torch.Tensor:
    """Pages of keys and values fp32 [pages, Hkv, P, D] to [pages, Hkv, words]."""
    n, H, P, D = k.shape
    kc, ks, kz = _groups(k, G)
    vc, vs, vz = _groups(v, G)
    kw = _words(kc.view(n, H, P, D // 8, 8))[..., _octet_order(D, k.device)]
    vw = _words(vc.view(n, H, P // 8, 8, D).transpose(-1, -2))
    vw = vw[..., torch.argsort(_value_order(D, k.device))]
    parts = (kw, _group_words(ks, kz).transpose(-1, -2), vw, _group_words(vs, vz).transpose(-1, -2))
    return torch.cat([p.reshape(n, H, -1) for p in parts], -1)


def _bounds(case: dict) -> tuple[int, int, int, int]:
    """Where the four parts of a block begin, the first at 0, and its words."""
    P, D, NG = case["P"], case["D"], case["D"] // case["G"]
    return P * D // 8, P * D // 8 + NG * P, P * D // 4 + NG * P, P * D // 4 + 2 * NG * P


def _unwords(w: torch.Tensor) -> torch.Tensor:
    shift = torch.tensor(_NIBBLE, dtype=torch.int32, device=w.device)
    return (w[..., None] >> shift) & 15


def _ungroup(code: torch.Tensor, meta: torch.Tensor, G: int) -> torch.Tensor:
    """Values of codes [..., D] with group words [..., D / G]."""
    s, c = meta.contiguous().view(torch.float16).view(*meta.shape, 2).float().unbind(-1)
    x = (code - 8).float().view(*meta.shape, G)
    return (x * s[..., None] + c[..., None]).view(code.shape)


def _unpack(blocks: torch.Tensor, case: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """Blocks [..., words] to keys and values fp32 [..., P, D]."""
    P, D, G = case["P"], case["D"], case["G"]
    a, b, c, d = _bounds(case)
    lead = blocks.shape[:-1]
    kw = blocks[..., :a].reshape(*lead, P, D // 8)
    kw = kw[..., torch.argsort(_octet_order(D, blocks.device))]
    kc = _unwords(kw).reshape(*lead, P, D)
    vw = blocks[..., b:c].reshape(*lead, P // 8, D)[..., _value_order(D, blocks.device)]
    vc = _unwords(vw).transpose(-1, -2)
    vc = vc.reshape(*lead, P, D)
    k = _ungroup(kc, blocks[..., a:b].reshape(*lead, D // G, P).transpose(-1, -2), G)
    v = _ungroup(vc, blocks[..., c:d].reshape(*lead, D // G, P).transpose(-1, -2), G)
    return k, v


# ---- what a program has in hand ---------------------------------------------

def _gen(seed: int, stream: int) -> torch.Generator:
    return torch.Generator(device=_DEVICE).manual_seed(seed * 64 + stream)


def _randn(shape, seed: int, stream: int) -> torch.Tensor:
    return torch.randn(shape, generator=_gen(seed, stream), device=_DEVICE)


def _ints(values) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=_DEVICE)


def _table(case: dict, lens: list[int], seed: int) -> tuple[torch.Tensor, int]:
    """Page tables int32 [rows, most pages] over pages in a shuffled order; a few
    pages more than the rows hold."""
    P = case["P"]
    held = [-(-n // P) for n in lens]
    pages = sum(held) + 3
    order = torch.randperm(pages, generator=_gen(seed, 1), device=_DEVICE).to(torch.int32)
    held_t = torch.tensor(held, device=_DEVICE)
    first = held_t.cumsum(0) - held_t
    at = torch.arange(max(held), device=_DEVICE)
    idx = (first[:, None] + at).clamp(max=pages - 1)
    return torch.where(at < held_t[:, None], order[idx], -1), pages


def _heads(case: dict, T: int, seed: int) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Queries, keys and values as slices of one fused projection's output."""
    Hq, Hkv, D = case["Hq"], case["Hkv"], case["D"]
    qkv = _randn((T, (Hq + 2 * Hkv) * D), seed, 2)
    # a few channels of every head are wider than the others, in a trained model
    qkv *= 1.0 + 3.0 * (_randn((Hq + 2 * Hkv) * D, seed, 3) > 2.0)
    qkv = qkv.to(_DTYPES[case["dtype"]]).view(T, Hq + 2 * Hkv, D)
    return qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]


def _rotation(case: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """cos and sin fp32 [positions, R / 2]."""
    half = case["R"] // 2
    freq = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=_DEVICE) / half)
    angle = torch.arange(case["ctx"], dtype=torch.float64, device=_DEVICE)[:, None] * freq
    return angle.cos().float(), angle.sin().float()


def _weights(case: dict, seed: int):
    if not case["norm"]:
        return None, None
    dt = _DTYPES[case["dtype"]]
    return tuple((1.0 + 0.2 * _randn(case["D"], seed, k)).to(dt) for k in (4, 5))


def _tokens(case: dict) -> tuple[torch.Tensor, torch.Tensor]:
    """(position, table row) of every new token."""
    q, n = _lengths(case)
    q, n = torch.tensor(q, device=_DEVICE), torch.tensor(n, device=_DEVICE)
    rows = torch.repeat_interleave(torch.arange(len(q), device=_DEVICE), q)
    first = (n - q - (q.cumsum(0) - q))[rows]
    return ((first + torch.arange(len(rows), device=_DEVICE)).to(torch.int32),
            rows.to(torch.int32))


def _forked(case: dict) -> tuple[list[int], list[int], list[int]]:
    """(parents, children, the parents' lengths) of a beam step: children are
    rows B .. B + q - 1."""
    lens = _spread(case["B"], case["ctx"])
    parents = [(3 * i + 1) % case["B"] for i in range(case["q"])]
    return parents, [case["B"] + i for i in range(case["q"])], [lens[p] for p in parents]


def _pool_state(case: dict, seed: int) -> dict:
    """A pool of random words; B live rows over shuffled pages (and, for a fork,
    q rows of beams that the step drops, each holding one page of its own)."""
    P, pages, B = case["P"], case["pages"], case["B"]
    words = _page_words(case) // case["Hkv"]
    pool = torch.randint(-2**31, 2**31 - 1, (case["L"], pages, case["Hkv"], words),
                         generator=_gen(seed, 6), device=_DEVICE, dtype=torch.int32)
    lens = _spread(B, case["ctx"]) + [1] * case["q"]
    held = torch.tensor([-(-n // P) for n in lens], device=_DEVICE)
    order = torch.randperm(pages, generator=_gen(seed, 1), device=_DEVICE).to(torch.int32)
    at = torch.arange(-(-case["ctx"] // P) + 2, device=_DEVICE)
    idx = (held.cumsum(0) - held)[:, None] + at
    table = torch.where(at < held[:, None], order[idx.clamp(max=pages - 1)], -1)
    refs = torch.zeros(pages, dtype=torch.int32, device=_DEVICE)
    refs[order[:int(held.sum())].long()] = 1
    return dict(pool=pool, table=table, lens=_ints(lens), refs=refs)


def prepare(case: dict, seed: int) -> dict:
    op = case["op"]
    state = dict(case=dict(case))
    if op in ("fork", "compact"):
        state |= _pool_state(case, seed)
        if op == "fork":
            parents, children, _ = _forked(case)
            state |= dict(parents=_ints(parents), children=_ints(children),
                          status=torch.zeros(1, dtype=torch.int32, device=_DEVICE))
        return state
    qs, ns = _lengths(case)
    if op in ("append", "rotate"):
        state["q"], state["k"], state["v"] = _heads(case, sum(qs), seed)
        state["cos"], state["sin"] = _rotation(case)
        state["wq"], state["wk"] = _weights(case, seed)
        state["positions"], state["rows"] = _tokens(case)
        if op == "append":
            state["table"], pages = _table(case, ns, seed)
            words = _page_words(case) // case["Hkv"]
            state["pool"] = torch.zeros((pages, case["Hkv"], words), dtype=torch.int32,
                                        device=_DEVICE)
        return state
    D, H, P = case["D"], case["Hkv"], case["P"]
    state["table"], pages = _table(case, ns, seed)
    # keys of a normed head have channels of different widths; values do not
    wide = 1.0 + 3.0 * (_randn((H, 1, D), seed, 7) > 2.0)
    pool = torch.empty((pages, H, _page_words(case) // H), dtype=torch.int32, device=_DEVICE)
    step = max(1, (1 << 26) // (H * P * D))
    for k, i in enumerate(range(0, pages, step)):
        n = min(step, pages - i)
        kv = _randn((2, n, H, P, D), seed * 4096 + k, 8)
        pool[i:i + n] = _pack(kv[0] * wide, kv[1], case["G"])
    state["pool"] = pool
    state["lens"] = _ints(ns)
    starts = [0]
    for a in qs:
        starts.append(starts[-1] + a)
    state["starts"] = _ints(starts) if case["q"] > 1 else None
    # scores of a trained head spread over a few units
    q = _randn((sum(qs), case["Hq"], D), seed, 9) * 1.5 / wide.mean()
    state["q"] = q.to(_DTYPES[case["dtype"]])
    return state


# ---- the plain forms ----------------------------------------------------------

def _rotate(x: torch.Tensor, w, state: dict) -> torch.Tensor:
    """Norm and rotation of x [T, H, D], fp32; the squares are summed in a fixed
    tree, so that the sum is the same to the bit wherever it is made."""
    case = state["case"]
    x = x.float()
    if w is not None:
        D = x.shape[-1]
        t = (x * x).view(*x.shape[:-1], D // 8, 8)
        t = t[..., :4] + t[..., 4:]
        t = t[..., :2] + t[..., 2:]
        t = t[..., 0] + t[..., 1]
        while t.shape[-1] > 1:
            t = t[..., :t.shape[-1] // 2] + t[..., t.shape[-1] // 2:]
        # (torch's fp32 square root is not rounded correctly; by way of fp64 it is)
        root = (t * (1.0 / D) + _EPS).double().sqrt().float()
        x = x * (1.0 / root) * w.float()
    R, pos = case["R"], state["positions"].long()
    c, s = state["cos"][pos][:, None], state["sin"][pos][:, None]
    if case["inter"]:
        a, b = x[..., 0:R:2], x[..., 1:R:2]
        r = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    else:
        a, b = x[..., :R // 2], x[..., R // 2:R]
        r = torch.cat((a * c - b * s, b * c + a * s), -1)
    return torch.cat((r, x[..., R:]), -1)


def _append_plain(state: dict):
    case = state["case"]
    P, D, G, H = case["P"], case["D"], case["G"], case["Hkv"]
    dt = _DTYPES[case["dtype"]]
    q = _rotate(state["q"], state["wq"], state).to(dt)
    kc, ks, kz = _groups(_rotate(state["k"], state["wk"], state), G)
    vc, vs, vz = _groups(state["v"].float(), G)
    pos = state["positions"].long()
    page = state["table"][state["rows"].long(), pos // P].long()
    tok = (pos % P)[:, None, None]
    pool = state["pool"]
    a, b, c, _ = _bounds(case)
    at = (page[:, None] * H + torch.arange(H, device=_DEVICE))[..., None] * pool.shape[-1]
    flat = pool.view(-1)
    T = len(pos)
    kw = _words(kc.view(T, H, D // 8, 8))[..., _octet_order(D, _DEVICE)]
    flat[at + tok * (D // 8) + torch.arange(D // 8, device=_DEVICE)] = kw
    groups = torch.arange(D // G, device=_DEVICE) * P
    flat[at + a + groups + tok] = _group_words(ks, kz)
    flat[at + c + groups + tok] = _group_words(vs, vz)
    # eight tokens share a word: every token adds its own change to it
    word = at + b + tok // 8 * D + _value_order(D, _DEVICE)
    i = tok % 8
    shift = (4 * (i // 2 + 4 * (i % 2))).to(torch.int32)
    old = (flat[word] >> shift) & 15
    flat.index_add_(0, word.view(-1), ((vc - old) << shift).view(-1))
    k, v = _read_plain(state)
    return q, k.to(dt), v.to(dt)


def _read_plain(state: dict):
    """Stored tokens [T, H, D] fp32."""
    case = state["case"]
    P, D, G, H = case["P"], case["D"], case["G"], case["Hkv"]
    pos = state["positions"].long()
    page = state["table"][state["rows"].long(), pos // P].long()
    tok = (pos % P)[:, None, None]
    flat = state["pool"].view(-1)
    a, b, c, _ = _bounds(case)
    at = (page[:, None] * H + torch.arange(H, device=_DEVICE))[..., None] * state["pool"].shape[-1]
    order = torch.argsort(_octet_order(D, _DEVICE))
    kc = _unwords(flat[at + tok * (D // 8) + order]).flatten(-2)
    i = tok % 8
    shift = (4 * (i // 2 + 4 * (i % 2))).to(torch.int32)
    vc = (flat[at + b + tok // 8 * D + _value_order(D, _DEVICE)] >> shift) & 15
    groups = torch.arange(D // G, device=_DEVICE) * P
    return (_ungroup(kc, flat[at + a + groups + tok], G),
            _ungroup(vc, flat[at + c + groups + tok], G))


def _attend_plain(state: dict):
    case = state["case"]
    D, H, Hq, G = case["D"], case["Hkv"], case["Hq"], case["G"]
    table, lens, q = state["table"], state["lens"].long(), state["q"]
    B, most = table.shape
    k, v = _unpack(state["pool"][table.clamp(min=0).long()], case)   # [B, pages, H, P, D]
    N = most * case["P"]
    k = k.transpose(1, 2).reshape(B, H, N, D)
    v = v.transpose(1, 2).reshape(B, H, N, D)
    if state["starts"] is None:
        nq = torch.ones_like(lens)
        top, first = 1, torch.arange(B, device=_DEVICE)
    else:
        starts = state["starts"].long()
        nq, first = starts[1:] - starts[:-1], starts[:-1]
        top = case["q"]
    i = torch.arange(top, device=_DEVICE)
    have = i < nq[:, None]                                            # [B, top]
    idx = torch.where(have, first[:, None] + i, 0)
    x = q[idx].float().view(B, top, H, Hq // H, D).permute(0, 2, 3, 1, 4)
    x = x.reshape(B, H, Hq // H * top, D)
    s = torch.matmul(x, k.transpose(-1, -2).contiguous()) * (1.0 / math.sqrt(D))
    pos = (lens - nq)[:, None] + i                                    # [B, top]
    t = torch.arange(N, device=_DEVICE)
    see = (t <= pos[..., None]) & (t < lens[:, None, None]) & have[..., None]
    if case["window"]:
        see &= t > pos[..., None] - case["window"]
    see = see[:, None, None].expand(B, H, Hq // H, top, N).reshape(s.shape)
    s = torch.where(see, s, -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m > -math.inf, m, 0.0))
    l = p.sum(-1, keepdim=True)
    seen = (t < lens[:, None])[:, None, :, None]
    o = torch.matmul(p, torch.where(seen, v, 0.0))
    o = torch.where(l > 0, o / l, 0.0)
    o = o.view(B, H, Hq // H, top, D).permute(0, 3, 1, 2, 4).reshape(B, top, Hq, D)
    return o[have].to(q.dtype)


def _free_first(refs: torch.Tensor) -> torch.Tensor:
    """Pages in the order in which they are taken: free ones first, lowest first."""
    return torch.sort((refs != 0).to(torch.int32), stable=True)[1]


def _fork_plain(state: dict):
    case = state["case"]
    P = case["P"]
    pool, table, lens, refs = state["pool"], state["table"], state["lens"], state["refs"]
    par, chi = state["parents"].long(), state["children"].long()
    # drop what the children's rows hold
    old = table[chi]
    refs.index_add_(0, old.clamp(min=0).flatten().long(), -(old >= 0).flatten().to(torch.int32))
    table[chi] = -1
    lens[chi] = 0
    # share the whole pages, copy the partial ones
    n = lens[par]
    at = torch.arange(table.shape[1], device=_DEVICE)
    part = n % P != 0
    # (the others' turns come after theirs, and end where they began)
    turn = torch.sort((~part).to(torch.int32), stable=True)[1].argsort()
    fresh = _free_first(refs)[turn].to(torch.int32)
    rows = table[par]
    last = (at == (n // P)[:, None]) & part[:, None]
    src = torch.where(part, rows.gather(1, (n // P)[:, None].long().clamp(
        max=table.shape[1] - 1)).squeeze(1), fresh)
    pool[:, fresh.long()] = torch.where(part[None, :, None, None], pool[:, src.long()],
                                        pool[:, fresh.long()])
    new = torch.where(last, fresh[:, None], rows)
    refs.index_add_(0, new.clamp(min=0).flatten().long(), (new >= 0).flatten().to(torch.int32))
    table[chi] = new
    lens[chi] = n
    return pool, table, lens, refs


def _compact_plain(state: dict):
    pool, table, refs = state["pool"], state["table"], state["refs"]
    n = refs.numel()
    used = refs > 0
    live = used.sum()
    at = torch.arange(n, device=_DEVICE)
    moves, hole = used & (at >= live), ~used & (at < live)
    # the k-th page that moves goes to the k-th hole
    src, dst = moves.nonzero().flatten(), hole.nonzero().flatten()
    to = at.index_put((src,), dst)
    pool[:, dst] = pool[:, src]
    new_refs = torch.zeros_like(refs).index_add_(0, to, refs)
    new_table = torch.where(table >= 0, to[table.clamp(min=0).long()].to(torch.int32), -1)
    return pool, new_table, new_refs, live.to(torch.int32).view(1)


# ---- one pass ------------------------------------------------------------------

def run(state: dict):
    return _run_own(state) if own else _run_plain(state)


def _run_plain(state: dict):
    op = state["case"]["op"]
    if op == "append":
        return _append_plain(state)
    if op == "rotate":
        dt = state["q"].dtype
        return (_rotate(state["q"], state["wq"], state).to(dt),
                _rotate(state["k"], state["wk"], state).to(dt))
    if op == "attend":
        return _attend_plain(state)
    return _fork_plain(state) if op == "fork" else _compact_plain(state)


def _run_own(state: dict):
    w, case = _package(), state["case"]
    op = case["op"]
    if op in ("append", "rotate"):
        turn = dict(q_weight=state["wq"], k_weight=state["wk"], eps=_EPS,
                    interleaved=case["inter"])
        if op == "rotate":
            return w.qk_norm_rope(state["q"], state["k"], state["cos"], state["sin"],
                                  state["positions"], **turn)
        q = w.kv4_append(state["q"], state["k"], state["v"], state["cos"], state["sin"],
                         state["positions"], state["pool"], state["table"], rows=state["rows"],
                         group_size=case["G"], **turn)
        k, v = w.kv4_read(state["pool"], state["table"], state["positions"], rows=state["rows"],
                          head_dim=case["D"], group_size=case["G"], dtype=q.dtype)
        return q, k, v
    if op == "attend":
        return w.kv4_attention(state["q"], state["pool"], state["table"], state["lens"],
                               q_starts=state["starts"], max_q=case["q"],
                               max_context=case["ctx"], window=case["window"],
                               group_size=case["G"])
    if op == "fork":
        w.kv4_free(state["table"], state["lens"], state["refs"], state["children"])
        w.kv4_fork(state["pool"], state["table"], state["lens"], state["refs"], state["parents"],
                   state["children"], page_size=case["P"], status=state["status"])
        return state["pool"], state["table"], state["lens"], state["refs"]
    table, refs, live = w.kv4_compact(state["pool"], state["table"], state["refs"])
    return state["pool"], table, refs, live


# ---- the definition in 64 bits ----------------------------------------------------

def _code(words: torch.Tensor, i: torch.Tensor) -> torch.Tensor:
    """The i-th code of each word."""
    bit = (i >> 1) * 4 + (i & 1) * 16
    return ((words.long() & 0xFFFFFFFF) >> bit) & 15


def _half(bits: torch.Tensor) -> torch.Tensor:
    """fp16 numbers in the low 16 bits, as fp64."""
    b = bits.long() & 0xFFFF
    return torch.where(b > 32767, b - 65536, b).to(torch.int16).view(torch.float16).double()


def _stored(pool: torch.Tensor, pages: torch.Tensor, head: int, case: dict):
    """Keys and values fp64 [len(pages) * P, D] of one head, by the format's words."""
    P, D, G = case["P"], case["D"], case["G"]
    block = pool[pages.long(), head]
    d = torch.arange(D, device=_DEVICE)
    t = torch.arange(P, device=_DEVICE)[:, None]
    kword = t * (D // 8) + (D // 32) * (d // 8 % 4) + d // 32
    k = _code(block[:, kword], (d % 8).expand(P, D)).double() - 8
    at = P * D // 8
    meta = block[:, at + d // G * P + t]
    k = k * _half(meta) + _half(meta >> 16)
    at += P * (D // G)
    vword = d - d % 64 + d % 16 * 4 + d % 64 // 16
    v = _code(block[:, at + t // 8 * D + vword], (t % 8).expand(P, D)).double() - 8
    at += P * D // 8
    meta = block[:, at + d // G * P + t]
    v = v * _half(meta) + _half(meta >> 16)
    return k.reshape(-1, D), v.reshape(-1, D)


def _turned(x: torch.Tensor, w, case: dict) -> torch.Tensor:
    """Norm and rotation as complex factors, fp64."""
    x = x.double()
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + _EPS).sqrt() * w.double()
    pos, _ = _tokens(case)
    half = case["R"] // 2
    # the tables are inputs, and fp32
    cos, sin = _rotation(case)
    turn = torch.complex(cos.double(), sin.double())[pos.long()][:, None]
    head, rest = x[..., :case["R"]], x[..., case["R"]:]
    pair = head.unflatten(-1, (half, 2)) if case["inter"] else \
        head.unflatten(-1, (2, half)).transpose(-1, -2)
    z = torch.view_as_real(torch.view_as_complex(pair.contiguous()) * turn)
    z = z if case["inter"] else z.transpose(-1, -2)
    return torch.cat((z.reshape(head.shape), rest), -1)


def _rounded(x: torch.Tensor, G: int) -> torch.Tensor:
    """What 4 bits keep of x: 16 steps a group, scale and centre in fp16."""
    g = x.unflatten(-1, (-1, G))
    lo = g.min(-1, keepdim=True)[0]
    step = ((g.max(-1, keepdim=True)[0] - lo) / 15).half().double()
    mid = (lo + 8 * step).half().double()
    n = torch.where(step > 0, ((g - mid) / step).round().clamp(-8, 7), 0.0)
    return (n * step + mid).view(x.shape)


def exact(case: dict, seed: int):
    op = case["op"]
    if op in ("fork", "compact"):
        return None                      # whole numbers only
    state = prepare(case, seed)
    if op in ("append", "rotate"):
        q = _turned(state["q"], state["wq"], case)
        k = _turned(state["k"], state["wk"], case)
        if op == "rotate":
            return q, k
        return q, _rounded(k, case["G"]), _rounded(state["v"].double(), case["G"])
    D, H, Hq = case["D"], case["Hkv"], case["Hq"]
    qs, ns = _lengths(case)
    out = torch.zeros((sum(qs), Hq, D), dtype=torch.float64, device=_DEVICE)
    at = 0
    for b, (a, n) in enumerate(zip(qs, ns)):
        pages = state["table"][b, :-(-n // case["P"])]
        for h in range(H if n else 0):
            k, v = _stored(state["pool"], pages, h, case)
            mine = slice(h * (Hq // H), (h + 1) * (Hq // H))
            x = state["q"][at:at + a, mine].double()                  # [a, heads, D]
            s = (x.reshape(-1, D) @ k[:n].t().contiguous()).view(a, Hq // H, n) / math.sqrt(D)
            p = n - a + torch.arange(a, device=_DEVICE)[:, None, None]
            t = torch.arange(n, device=_DEVICE)
            hidden = t > p
            if case["window"]:
                hidden = hidden | (t <= p - case["window"])
            s = s.masked_fill(hidden, -math.inf).softmax(-1)
            out[at:at + a, mine] = (s.view(-1, n) @ v[:n]).view(a, Hq // H, D)
        at += a
    return out

"""Measured calls of the operators around the 8-bit key/value cache: rotary positions, append, attention, pages.

Between the projections that the engine has (q, k, v in, o out) a decoder rotates queries and keys, keeps keys and values, and
attends to them. Five kinds of work, over the sizes, types and masks that programs use:

- ``rope``: ``rope_into``, rotary positions with one or several axes (text; time, height and width of images and video).
- ``append``: ``KvCache.append`` of a step's keys and values (rotated on the way, as the queries are), and the blocks that it
  touched as ``KvCache.read`` gives them back.
- ``attend``: ``KvCache.attend`` of the last ``tokens`` tokens of every sequence to all that its mask lets it see.
- ``beam``: sequences forked into beams that share their pages, one token appended to each (which copies the partly filled
  pages), its page read back, the beams freed.
- ``compact``: half of the sequences copied page by page, the originals freed, the pool compacted, the copies renamed.

The cache holds int8 codes with a 32-bit scale for every block of 16 tokens and head, for keys and values each. A block's
first tokens set its scale to their largest magnitude / 127 (at least 2^-64); a later token that does not fit doubles it
as often as it takes, and the codes in place are divided by as much and rounded to even, once. A code is the value times the scale's
reciprocal, rounded to even, all in 32 bits.

A query at position p of its sequence sees the tokens j <= p with j > p - window (window 0: all of them) or j < sinks.
"""
from __future__ import annotations

import numpy as np
import torch

own = False

_DEV = "cuda:0"
_BLOCK = 16
_TINY = 2.0 ** -64
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}


def listed():
    return [
        # the q and k heads of one request's token: a call of a few microseconds
        dict(name="rope_t1_h40_d128", kind="rope", tokens=1, heads=40, dim=128, rot=128, axes=1, interleaved=True, type="f32"),
        # patches of a video in a vision tower: three axes, bf16, a size that divides by nothing
        dict(name="rope_video_t16381_h16_d80", kind="rope", tokens=16381, heads=16, dim=80, rot=80, axes=3, interleaved=False, type="bf16"),
        # a decode step of many requests: one token each, at places all over their blocks
        dict(name="append_b64_t1", kind="append", n=64, len=2000, tokens=1, layers=4, kv_heads=8, group=4, dim=128, page=16, rot=128, axes=1,
             interleaved=True, type="f32"),
        # a prompt of no round length, whose first tokens end a block that others began
        dict(name="append_b1_t2043", kind="append", n=1, len=2057, tokens=2043, layers=4, kv_heads=8, group=4, dim=128, page=64, rot=64, axes=3,
             interleaved=False, type="f32"),
        # one request that has just begun
        dict(name="attend_b1_t1_l293", kind="attend", n=1, len=293, tokens=1, layers=4, kv_heads=8, group=4, dim=128, page=16, window=0, sinks=0,
             qtype="f32", otype="f32"),
        # many requests of all lengths decoded together
        dict(name="attend_b64_t1_l8191", kind="attend", n=64, len=8191, tokens=1, layers=2, kv_heads=8, group=4, dim=128, page=16, window=0, sinks=0,
             qtype="f32", otype="f32"),
        # one request with a very long context
        dict(name="attend_b1_t1_l131071", kind="attend", n=1, len=131071, tokens=1, layers=2, kv_heads=8, group=4, dim=128, page=64, window=0, sinks=0,
             qtype="f32", otype="f32"),
        # long conversations through a sliding window and four first tokens, heads of 64
        dict(name="attend_b32_t1_l20000_w1024", kind="attend", n=32, len=20000, tokens=1, layers=2, kv_heads=8, group=8, dim=64, page=32, window=1024,
             sinks=4, qtype="bf16", otype="bf16"),
        # a prompt, whole
        dict(name="attend_b1_t8192", kind="attend", n=1, len=8192, tokens=8192, layers=1, kv_heads=8, group=4, dim=128, page=64, window=0, sinks=0,
             qtype="f32", otype="bf16"),
        # chunks of several prompts onto what is there, windowed
        dict(name="attend_b4_t509_l9001_w4096", kind="attend", n=4, len=9001, tokens=509, layers=1, kv_heads=4, group=7, dim=128, page=32, window=4096,
             sinks=4, qtype="f32", otype="bf16"),
        # a step of a beam search
        dict(name="beam_b8_x4_l1000", kind="beam", n=8, beams=4, len=1000, layers=8, kv_heads=8, dim=128, page=16),
        # a pool tidied up after requests of all lengths have come and gone
        dict(name="compact_b16_l3000", kind="compact", n=16, len=3000, layers=4, kv_heads=8, dim=128, page=64),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["rope", "append", "attend", "attend", "attend", "beam", "compact"])
    kv_heads, dim, page = rng.choice([1, 2, 4, 8]), rng.choice([64, 96, 128, 128, 192, 256]), rng.choice([16, 32, 64])
    if kind == "rope":
        dim = rng.choice([64, 80, 96, 128, 256])
        axes = rng.choice([1, 2, 3])
        return dict(kind=kind, tokens=_log(rng, 1, 16000), heads=rng.randint(1, 40), dim=dim, rot=rng.choice([dim, dim // 2]), axes=axes,
                    interleaved=rng.random() < 0.5, type=rng.choice(["f32", "bf16"]))
    if kind == "append":
        n = _log(rng, 1, 64)
        tokens = rng.choice([1, rng.randint(2, 8), _log(rng, 1, max(1, 2048 // n))])
        return dict(kind=kind, n=n, len=tokens + _log(rng, 1, 2000), tokens=tokens, layers=rng.choice([1, 2, 4]), kv_heads=kv_heads,
                    group=rng.choice([1, 2, 4, 7]), dim=dim, page=page, rot=rng.choice([dim, dim // 2]), axes=rng.choice([1, 3]),
                    interleaved=rng.random() < 0.5, type=rng.choice(["f32", "f32", "bf16"]))
    if kind == "attend":
        group, window = rng.choice([1, 2, 3, 4, 5, 7, 8]), rng.choice([0, 0, _log(rng, 100, 4096)])
        sinks = rng.choice([0, 4, rng.randint(1, 100)]) if window else 0
        types = dict(qtype=rng.choice(["f32", "f32", "bf16"]), otype=rng.choice(["f32", "bf16"]))
        if rng.random() < 0.6:  # decoding, a token or a few to be verified
            n = _log(rng, 1, 64)
            tokens = rng.choice([1, 1, 1, rng.randint(2, 5)])
            return dict(kind=kind, n=n, len=max(tokens, _log(rng, 30, min(65536, 400000 // n))), tokens=tokens, layers=rng.choice([1, 2]),
                        kv_heads=kv_heads, group=group, dim=dim, page=page, window=window, sinks=sinks, **types)
        n = _log(rng, 1, 4)
        tokens = _log(rng, 9, 4096 // n)
        return dict(kind=kind, n=n, len=tokens + rng.choice([0, _log(rng, 10, 8000 // n)]), tokens=tokens, layers=1, kv_heads=min(4, kv_heads),
                    group=group, dim=dim, page=page, window=window, sinks=sinks, qtype="f32", otype=rng.choice(["bf16", "bf16", "f32"]))
    if kind == "beam":
        n = _log(rng, 1, 16)
        return dict(kind=kind, n=n, beams=rng.randint(2, 6), len=_log(rng, 20, 2000), layers=rng.choice([2, 4, 8]), kv_heads=kv_heads, dim=dim, page=page)
    return dict(kind=kind, n=_log(rng, 2, 16), len=_log(rng, 100, 3000), layers=rng.choice([1, 2, 4]), kv_heads=kv_heads, dim=dim, page=page)


# ---- inputs ----------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=_DEV).manual_seed(seed)


def _lens(case):
    """The sequences' lengths: the longest first, down to about a quarter of it, nowhere round."""
    n, most, least = case["n"], case["len"], case.get("tokens", 1)
    return [max(least, most - (i * most * 3) // (4 * n)) for i in range(n)]


def _heads_like(g, *shape):
    """Keys or queries of a head: N(0, 1), and a few channels several times larger."""
    x = torch.randn(shape, generator=g, device=_DEV)
    big = torch.rand(shape[-1:], generator=g, device=_DEV) < 0.02
    return torch.where(big, 4 * x, x)


def _rope_tables(rows, rot):
    pair = torch.arange(rot // 2, device=_DEV, dtype=torch.float64)
    angle = torch.arange(rows, device=_DEV, dtype=torch.float64)[:, None] * 10000.0 ** (-2 * pair / rot)
    return angle.cos().float(), angle.sin().float()


def _sections(rot, axes):
    """Pairs of each axis: as many for each, the first one the rest."""
    p = rot // 2
    return [p - (axes - 1) * (p // axes)] + [p // axes] * (axes - 1)


def _rope_inputs(case, g, tokens, positions):
    """Tables and the positions [axes, tokens] (time first; the other axes inside a frame)."""
    cos, sin = _rope_tables(int(positions.max()) + 257, case["rot"])
    more = torch.randint(0, 256, (case["axes"] - 1, tokens), generator=g, device=_DEV, dtype=torch.int32)
    sections = _sections(case["rot"], case["axes"])
    axis = torch.repeat_interleave(torch.arange(case["axes"], device=_DEV), torch.tensor(sections, device=_DEV))
    return dict(cos=cos, sin=sin, positions=torch.cat([positions.to(torch.int32).reshape(1, -1), more]).contiguous(), sections=sections,
                axis=axis)


def _dense(case, seed):
    """The case's inputs, without the cache: {name: tensor}, a list over layers where there is one per layer."""
    g, kind = _gen(seed), case["kind"]
    d = {}
    if kind == "rope":
        d["x"] = _heads_like(g, case["tokens"], case["heads"], case["dim"]).to(_TYPES[case["type"]])
        d["rope"] = _rope_inputs(case, g, case["tokens"], torch.randint(0, 8192, (case["tokens"],), generator=g, device=_DEV))
        return d
    n, h, dim, layers = case["n"], case["kv_heads"], case["dim"], case["layers"]
    lens = _lens(case)
    padded = -(-max(lens) // _BLOCK) * _BLOCK
    t = case.get("tokens", 0)
    # what the sequences hold before the step, [n, padded, heads, dim], and the step's keys and values, [n * tokens, heads, dim]
    d["k"] = [_heads_like(g, n, padded, h, dim) for _ in range(layers)]
    d["v"] = [torch.randn((n, padded, h, dim), generator=g, device=_DEV) for _ in range(layers)]
    if kind == "append":
        typ, rows = _TYPES[case["type"]], n * t
        d["new_k"] = [_heads_like(g, rows, h, dim).mul_(1.1).to(typ) for _ in range(layers)]
        d["new_v"] = [torch.randn((rows, h, dim), generator=g, device=_DEV).mul_(1.1).to(typ) for _ in range(layers)]
        d["q"] = [_heads_like(g, rows, h * case["group"], dim).to(typ) for _ in range(layers)]
        place = torch.cat([torch.arange(l - t, l) for l in lens]).to(_DEV)
        d["rope"] = _rope_inputs(case, g, rows, place)
    if kind == "attend":
        d["q"] = [_heads_like(g, n * t, h * case["group"], dim).to(_TYPES[case["qtype"]]) for _ in range(layers)]
    if kind == "beam":
        m = n * case["beams"]
        d["new_k"] = [_heads_like(g, m, h, dim) for _ in range(layers)]
        d["new_v"] = [torch.randn((m, h, dim), generator=g, device=_DEV) for _ in range(layers)]
    return d


# ---- the framework's side --------------------------------------------------------------------


def _prepare_own(s, case, d):
    from jax4j_amd import DType, KvCache, Mi355xBackend, Rope

    s.be = Mi355xBackend()
    s.types = {"f32": DType.F32, "bf16": DType.BF16}
    if "rope" in d:
        r = d["rope"]
        s.rope = Rope(r["cos"].data_ptr(), r["sin"].data_ptr(), r["cos"].shape[0], case["rot"], positions=r["positions"].data_ptr(),
                      sections=r["sections"], interleaved=case["interleaved"])
    if case["kind"] == "rope":
        s.y = torch.empty_like(d["x"])
        torch.cuda.synchronize()
        return s
    kind, n, page = case["kind"], case["n"], case["page"]
    lens, seqs = _lens(case), list(range(case["n"]))
    t = case.get("tokens", 0)
    per = [-(-(l + 1) // page) for l in lens]
    slots = n * (1 + case["beams"]) if kind == "beam" else 2 * n
    pages = sum(per) + (n * case["beams"] if kind == "beam" else sum(per) if kind == "compact" else 0)
    s.kv = KvCache(s.be, layers=case["layers"], kv_heads=case["kv_heads"], head_dim=case["dim"], pages=pages, page_tokens=page, sequences=slots,
                   sequence_pages=max(per))
    held = [l - t for l in lens] if kind == "append" else lens
    at = [0] * n
    step = 16 * 1024 if kind in ("beam", "compact") else 512  # pages of long sequences lie between each other's
    while any(a < l for a, l in zip(at, held)):
        who = [i for i in seqs if at[i] < held[i]]
        part = [min(step, held[i] - at[i]) for i in who]
        s.kv.extend(who, part)
        for l in range(case["layers"]):
            rows_k = torch.cat([d["k"][l][i, at[i]:at[i] + c] for i, c in zip(who, part)])
            rows_v = torch.cat([d["v"][l][i, at[i]:at[i] + c] for i, c in zip(who, part)])
            torch.cuda.synchronize()
            s.kv.append(l, rows_k.data_ptr(), rows_v.data_ptr())
            s.be.sync()
        for i, c in zip(who, part):
            at[i] += c
    dense = dict(device=_DEV, dtype=torch.float32)
    if kind == "append":
        s.kv.extend(seqs, [t] * n)
        s.first, s.count = [(l - t) // _BLOCK * _BLOCK for l in lens], _window(t)
        s.q_out = [torch.empty_like(q) for q in d["q"]]
    elif kind == "attend":  # the step is the last tokens of every sequence, which the cache holds
        s.kv.begin(seqs, [t] * n)
        s.out = [torch.empty(q.shape, device=_DEV, dtype=_TYPES[case["otype"]]) for q in d["q"]]
    elif kind == "beam":
        m = n * case["beams"]
        s.src = [i for i in range(n) for _ in range(case["beams"])]
        s.dst = list(range(n, n + m))
        s.first, s.count = [lens[i] // page * page for i in s.src], page
    else:
        s.half = seqs[::2]
        s.copies = [n + i for i in s.half]
        s.first, s.count = [0] * len(s.half), max(lens)
    if kind != "attend":
        m = {"append": n, "beam": n * case.get("beams", 0), "compact": (n + 1) // 2}[kind]
        shape = (m, s.count, case["kv_heads"], case["dim"])
        s.read_k = [torch.empty(shape, **dense) for _ in range(case["layers"])]
        s.read_v = [torch.empty(shape, **dense) for _ in range(case["layers"])]
    torch.cuda.synchronize()
    return s


def _run_own(s):
    case, d = s.case, s.d
    kind, layers = case["kind"], case.get("layers", 1)
    if kind == "rope":
        s.be.rope_into(d["x"].data_ptr(), s.y.data_ptr(), case["tokens"], case["heads"], case["dim"], s.rope, s.types[case["type"]])
        return s.y
    if kind == "attend":
        heads, q, o = case["kv_heads"] * case["group"], s.types[case["qtype"]], s.types[case["otype"]]
        for l in range(layers):
            s.kv.attend(l, d["q"][l].data_ptr(), s.out[l].data_ptr(), heads, q_type=q, out_type=o, window=case["window"], sinks=case["sinks"])
        return s.out
    if kind == "append":
        heads = case["kv_heads"] * case["group"]
        for l in range(layers):
            s.kv.append(l, d["new_k"][l].data_ptr(), d["new_v"][l].data_ptr(), s.types[case["type"]], rope=s.rope, q_ptr=d["q"][l].data_ptr(),
                        q_out_ptr=s.q_out[l].data_ptr(), heads=heads)
        for l in range(layers):
            s.kv.read(l, range(case["n"]), s.first, s.count, s.read_k[l].data_ptr(), s.read_v[l].data_ptr())
        return {"q": s.q_out, "k": s.read_k, "v": s.read_v}
    if kind == "beam":
        s.kv.fork(s.src, s.dst)
        s.kv.extend(s.dst, [1] * len(s.dst))
        for l in range(layers):
            s.kv.append(l, d["new_k"][l].data_ptr(), d["new_v"][l].data_ptr())
        for l in range(layers):
            s.kv.read(l, s.dst, s.first, s.count, s.read_k[l].data_ptr(), s.read_v[l].data_ptr())
        tables = s.kv.tables(s.dst)
        s.kv.truncate(s.dst, [0] * len(s.dst))
        return {"k": s.read_k, "v": s.read_v, "tables": tables}
    s.kv.fork(s.half, s.copies, share=False)
    s.kv.truncate(s.half, [0] * len(s.half))
    s.kv.compact()
    s.kv.fork(s.copies, s.half)
    s.kv.truncate(s.copies, [0] * len(s.half))
    for l in range(layers):
        s.kv.read(l, s.half, s.first, s.count, s.read_k[l].data_ptr(), s.read_v[l].data_ptr())
    return {"k": s.read_k, "v": s.read_v, "tables": s.kv.tables(range(case["n"]))}


# ---- the plain form --------------------------------------------------------------------------


def _window(tokens):
    """Tokens of the blocks that `tokens` new ones can touch, wherever they begin."""
    return -(-(_BLOCK - 1 + tokens) // _BLOCK) * _BLOCK


def _rotate(x, r, interleaved):
    """Rotary positions of x [tokens, heads, dim] in 32 bits."""
    pairs = r["cos"].shape[1]
    at = r["positions"].long()[r["axis"]]  # [pairs, tokens]
    pair = torch.arange(pairs, device=_DEV)[:, None]
    c, sn = r["cos"][at, pair].t()[:, None], r["sin"][at, pair].t()[:, None]
    y = x.float().clone()
    one, two = (y[..., 0:2 * pairs:2], y[..., 1:2 * pairs:2]) if interleaved else (y[..., :pairs], y[..., pairs:2 * pairs])
    a, b = one * c - two * sn, two * c + one * sn
    one.copy_(a)
    two.copy_(b)
    return y


def _quantize(x):
    """Codes and scales [n, blocks, heads] of whole blocks x [n, tokens, heads, dim] that nothing was in."""
    n, t, h, dim = x.shape
    b = x.reshape(n, t // _BLOCK, _BLOCK, h, dim)
    amax = b.abs().amax((2, 4))
    scale = (amax / torch.full_like(amax, 127.0)).clamp_min(_TINY)  # a tensor: division by a number multiplies by its reciprocal
    return torch.round(b * (1.0 / scale)[:, :, None, :, None]).to(torch.int8).reshape(x.shape), scale


def _power(k):
    """2 to whole numbers k, in 32 bits."""
    return ((k.int() + 127) << 23).view(torch.float32)


def _append_plain(codes, scale, offset, new):
    """New tokens [n, tokens, heads, dim] at `offset` [n] of blocks codes [n, 16 * blocks, heads, dim] and scale [n, blocks, heads]."""
    n, w, h, dim = codes.shape
    at = (offset[:, None] + torch.arange(new.shape[1], device=_DEV))[:, :, None, None].expand(-1, -1, h, dim)
    x = torch.zeros(codes.shape, device=_DEV).scatter_(1, at, new)
    fresh = torch.zeros(codes.shape, device=_DEV, dtype=torch.bool).scatter_(1, at, True)
    amax = x.reshape(n, w // _BLOCK, _BLOCK, h, dim).abs().amax((2, 4))
    first = (amax / torch.full_like(amax, 127.0)).clamp_min(_TINY)
    block = torch.arange(w // _BLOCK, device=_DEV)[None, :, None]
    begun = (block * _BLOCK < offset[:, None, None]) & (scale > _TINY)
    kept = torch.where(begun, scale, torch.ones_like(scale))
    part, power = torch.frexp(amax * (1.0 / kept))
    steps = torch.where(begun, (power - 7 + (part >= 127.5 / 128).int()).clamp_min(0), torch.zeros_like(power))
    new_scale = torch.where(begun, kept * _power(steps), first)
    rows = lambda v: v.repeat_interleave(_BLOCK, 1)[..., None]  # noqa: E731
    old = torch.round(codes.float() * rows(_power(-steps)))
    return torch.where(fresh, torch.round(x * rows(1.0 / new_scale)), old).to(torch.int8), new_scale


def _values(codes, scale):
    return codes.float() * scale.repeat_interleave(_BLOCK, 1)[..., None]


def _gather(pool, table):
    """Tokens [n, pages * page, heads, dim] (or blocks) of a pool [pages, page, heads, dim] in a table's order."""
    return pool[table].flatten(1, 2)


def _prepare_plain(s, case, d):
    if case["kind"] == "rope":
        return s
    kind, n, h, dim, page, layers = case["kind"], case["n"], case["kv_heads"], case["dim"], case["page"], case["layers"]
    lens = _lens(case)
    t = case.get("tokens", 0)
    s.lens = torch.tensor(lens, device=_DEV)
    held = s.lens - t if kind == "append" else s.lens
    per = -(-(max(lens) + _window(t) + 1) // page)  # pages of a sequence in the table, some behind its end
    if kind in ("beam", "compact"):  # in the order in which they were taken
        used = np.array([-(-l // page) for l in lens])
        base = np.cumsum(used) - used
        s.used, s.base = used, base
        table = torch.from_numpy(np.minimum(base[:, None] + np.arange(per), used.sum() - 1)).to(_DEV)
        pages = int(used.sum()) + (n * case["beams"] if kind == "beam" else int(used.sum()))
        real = torch.from_numpy(np.arange(per)[None] < used[:, None]).to(_DEV)
    else:
        table = torch.randperm(n * per, generator=_gen(1), device=_DEV).reshape(n, per)
        pages, real = n * per, torch.ones((n, per), device=_DEV, dtype=torch.bool)
    s.table = table
    s.pool = {}
    for name in ("k", "v"):
        s.pool[name] = torch.zeros((layers, pages, page, h, dim), device=_DEV, dtype=torch.int8)
        s.pool[name + "s"] = torch.full((layers, pages, page // _BLOCK, h), _TINY, device=_DEV)
        for l in range(layers):
            x = torch.zeros((n, per * page, h, dim), device=_DEV)
            x[:, :d[name][l].shape[1]] = d[name][l][:, :per * page]
            x *= (torch.arange(per * page, device=_DEV) < held[:, None])[..., None, None]
            codes, scale = _quantize(x)
            s.pool[name][l][table[real]] = codes.reshape(n, per, page, h, dim)[real]
            s.pool[name + "s"][l][table[real]] = scale.reshape(n, per, page // _BLOCK, h)[real]
    return s


def _attend_plain(q, k, v, lens, case):
    """q [n, tokens, heads, dim] to k, v [n, places, kv heads, dim]."""
    n, t, heads, dim = q.shape
    h, g = case["kv_heads"], case["group"]
    q = q.float().reshape(n, t, h, g, dim).permute(0, 2, 3, 1, 4).reshape(n, h, g * t, dim)
    scores = torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) * dim ** -0.5
    at = (lens[:, None] - t + torch.arange(t, device=_DEV))[:, :, None]
    key = torch.arange(k.shape[1], device=_DEV)
    seen = key <= at
    if case["window"]:
        seen &= (key > at - case["window"]) | (key < case["sinks"])
    scores = scores.reshape(n, h, g, t, -1).masked_fill_(~seen[:, None, None], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(n, h, g * t, -1), v.transpose(1, 2).contiguous()).reshape(n, h, g, t, dim)
    return torch.where(total > 0, o / total, torch.zeros_like(o)).permute(0, 3, 1, 2, 4).reshape(n * t, heads, dim)


def _run_plain(s):
    case, d = s.case, s.d
    kind = case["kind"]
    if kind == "rope":
        return _rotate(d["x"], d["rope"], case["interleaved"]).to(d["x"].dtype)
    n, h, dim, page, layers = case["n"], case["kv_heads"], case["dim"], case["page"], case["layers"]
    pool = s.pool
    if kind == "attend":
        out = []
        for l in range(layers):
            k = _values(_gather(pool["k"][l], s.table), _gather(pool["ks"][l], s.table))
            v = _values(_gather(pool["v"][l], s.table), _gather(pool["vs"][l], s.table))
            q = d["q"][l].reshape(n, case["tokens"], -1, dim)
            out.append(_attend_plain(q, k, v, s.lens, case).to(_TYPES[case["otype"]]))
        return out
    if kind == "append":
        t = case["tokens"]
        start, w = s.lens - t, _window(t)
        first = start // _BLOCK * _BLOCK
        at = first[:, None] + torch.arange(w, device=_DEV)
        blocks = at[:, ::_BLOCK]
        tok, blk = (torch.gather(s.table, 1, at // page), at % page), (torch.gather(s.table, 1, blocks // page), blocks % page // _BLOCK)
        live = (at < s.lens[:, None])[..., None, None]
        got = {"q": [], "k": [], "v": []}
        for l in range(layers):
            got["q"].append(_rotate(d["q"][l], d["rope"], case["interleaved"]).to(d["q"][l].dtype))
            for name, x in (("k", _rotate(d["new_k"][l], d["rope"], case["interleaved"])), ("v", d["new_v"][l].float())):
                codes, scale = _append_plain(pool[name][l][tok], pool[name + "s"][l][blk], start - first, x.reshape(n, t, h, dim))
                pool[name][l][tok], pool[name + "s"][l][blk] = codes, scale
                got[name].append(torch.where(live, _values(codes, scale), torch.zeros((), device=_DEV)))
        return got
    if kind == "beam":
        m = n * case["beams"]
        src = np.repeat(np.arange(n), case["beams"])
        lens = np.array(_lens(case))[src]
        last = lens // page  # the page of the new token
        tables = np.full((m, max(-(-(l + 1) // page) for l in _lens(case))), -1, np.int32)
        place = np.arange(tables.shape[1])[None]
        tables = np.where(place < last[:, None], s.base[src][:, None] + place, tables).astype(np.int32)
        tables[np.arange(m), last] = s.used.sum() + np.arange(m)
        new = torch.arange(m, device=_DEV) + int(s.used.sum())
        old = torch.from_numpy(np.minimum(s.base[src] + last, s.base[src] + s.used[src] - 1)).to(_DEV)
        for name in ("k", "ks", "v", "vs"):  # the pages that others hold too are copied before they are written
            pool[name][:, new] = pool[name][:, old]
        offset = torch.from_numpy(lens % page).to(_DEV)
        live = (torch.arange(page, device=_DEV) <= offset[:, None])[..., None, None]
        got = {"k": [], "v": [], "tables": tables}
        for l in range(layers):
            for name in ("k", "v"):
                block = (offset // _BLOCK)[:, None]
                at = block * _BLOCK + torch.arange(_BLOCK, device=_DEV)
                codes, scale = _append_plain(pool[name][l][new[:, None], at], pool[name + "s"][l][new[:, None], block], offset % _BLOCK,
                                             d["new_" + name][l][:, None])
                pool[name][l][new[:, None], at], pool[name + "s"][l][new[:, None], block] = codes, scale
                got[name].append(torch.where(live, _values(pool[name][l][new], pool[name + "s"][l][new]), torch.zeros((), device=_DEV)))
        return got
    lens, per = np.array(_lens(case)), int(s.used.max())
    place = np.arange(per)[None]
    tables = np.where(place < s.used[:, None], s.base[:, None] + place, -1).astype(np.int32)
    half = np.arange(0, n, 2)
    src = torch.from_numpy(tables[half][tables[half] >= 0].astype(np.int64)).to(_DEV)
    dst = torch.arange(src.numel(), device=_DEV) + int(s.used.sum())
    for name in ("k", "ks", "v", "vs"):
        pool[name][:, dst] = pool[name][:, src]
    for name in ("k", "ks", "v", "vs"):  # the freed pages are the lowest
        pool[name][:, src] = pool[name][:, dst]
    count = int(lens.max())
    table = torch.from_numpy(np.maximum(tables[half], 0).astype(np.int64)).to(_DEV)
    live = (torch.arange(count, device=_DEV) < s.lens[::2, None])[..., None, None]
    got = {"k": [], "v": [], "tables": np.pad(tables, ((0, 0), (0, max(-(-(l + 1) // page) for l in lens) - per)), constant_values=-1)}
    for l in range(layers):
        for name in ("k", "v"):
            x = _values(_gather(pool[name][l], table), _gather(pool[name + "s"][l], table))[:, :count]
            got[name].append(torch.where(live, x, torch.zeros((), device=_DEV)))
    return got


# ---- what is measured ------------------------------------------------------------------------


class _State:
    """What a program holds between calls; gives the engine's cache back when it goes."""

    kv = None

    def __del__(self):
        if self.kv is not None:
            torch.cuda.synchronize()
            self.kv.destroy()


def prepare(case, seed):
    s = _State()
    s.case, s.d = case, _dense(case, seed)
    s = _prepare_own(s, case, s.d) if own else _prepare_plain(s, case, s.d)
    for name in ("k", "v"):  # in the cache now
        s.d.pop(name, None)
    torch.cuda.synchronize()
    return s


def run(s):
    return _run_own(s) if own else _run_plain(s)


def _seen(case):
    """Tokens that the step's queries see: any of them (read once), and summed over the queries."""
    any_, pairs, t = 0, 0, case["tokens"]
    w, sinks = case["window"], case["sinks"]
    for l in _lens(case):
        p = np.arange(l - t, l, dtype=np.int64)
        low = np.maximum(0, p - w + 1) if w else np.zeros_like(p)
        pairs += int((p + 1 - low + np.minimum(sinks, low)).sum())
        any_ += int(l - low[0] + min(sinks, low[0]))
    return any_, pairs


def work(case):
    kind = case["kind"]
    if kind == "rope":
        e = 4 if case["type"] == "f32" else 2
        values = case["tokens"] * case["heads"] * case["dim"]
        return {"bytes": 2 * e * values + 4 * case["tokens"] * case["axes"], "flops": 3 * case["tokens"] * case["heads"] * case["rot"]}
    n, h, dim, layers = case["n"], case["kv_heads"], case["dim"], case["layers"]
    token = 2 * h * dim + 2 * h * 4 / _BLOCK  # bytes that the cache holds of a token in a layer
    if kind == "attend":
        any_, pairs = _seen(case)
        e = sum(4 if case[k] == "f32" else 2 for k in ("qtype", "otype"))
        rows = n * case["tokens"] * h * case["group"]
        return {"bytes": layers * (any_ * token + e * rows * dim), "flops": layers * 4 * pairs * h * case["group"] * dim}
    if kind == "append":
        e, t = (4 if case["type"] == "f32" else 2), n * case["tokens"]
        back = n * case["tokens"] * (token + 2 * 4 * h * dim)
        return {"bytes": layers * (t * dim * e * (2 * h + 2 * h * case["group"]) + t * token + back),
                "flops": layers * t * dim * (3 * h * (1 + case["group"]) + 4 * h)}
    page = case["page"]
    if kind == "beam":
        m = n * case["beams"]
        return {"bytes": layers * m * (2 * page * token + 2 * 4 * h * dim + page // 2 * (token + 2 * 4 * h * dim)), "flops": layers * m * 4 * h * dim}
    tokens = sum(_lens(case)[::2])
    return {"bytes": layers * tokens * (4 * token + token + 2 * 4 * h * dim), "flops": layers * tokens * 2 * h * dim}


# ---- the definition in 64 bits ---------------------------------------------------------------


def _block64(codes, scale, place, rows):
    """A block's codes [16, heads, dim] and scales [heads] after rows [r, heads, dim] at `place`; the stored codes' rule in 32 bits, as numpy has it."""
    top = np.abs(rows).max((0, 2))
    one, most = np.float32(1), np.float32(127)
    for j in range(rows.shape[1]):
        if place == 0 or scale[j] <= np.float32(_TINY):
            scale[j] = max(top[j] / most, np.float32(_TINY))
        else:
            was = scale[j]
            while top[j] * (one / scale[j]) >= np.float32(127.5):
                scale[j] = scale[j] * np.float32(2)
            codes[:, j] = np.rint(codes[:, j] * (was / scale[j]))
        codes[place:place + rows.shape[0], j] = np.rint(rows[:, j] * (one / scale[j]))


def _fresh64(x):
    """The values in 64 bits that the cache holds of rows x [tokens, heads, dim] written from a block's first place on."""
    t, h, dim = x.shape
    b = torch.cat([x, x.new_zeros((-t % _BLOCK, h, dim))]).unflatten(0, (-1, _BLOCK))
    top = b.abs().amax((1, 3), keepdim=True)
    s = torch.maximum(top / torch.full_like(top, 127.0), torch.full_like(top, _TINY))
    return ((b * torch.reciprocal(s)).round().double() * s.double()).flatten(0, 1)[:t]


def _rope_pairs(x, r, interleaved, dtype):
    """Rotary positions pair by pair, in 64 bits or, for what is stored then, in 32."""
    x = x.to(dtype, copy=True)
    at, pair = r["positions"].long(), 0
    half = r["cos"].shape[1]
    for a, count in enumerate(r["sections"]):
        for i in range(pair, pair + count):
            c, s = r["cos"][at[a], i].to(dtype)[:, None], r["sin"][at[a], i].to(dtype)[:, None]
            i1, i2 = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
            u, w = x[..., i1].clone(), x[..., i2].clone()
            x[..., i1], x[..., i2] = u * c - w * s, w * c + u * s
        pair += count
    return x


def _read64(x, first, count):
    """Tokens [first, first + count) of x [tokens, heads, dim], zeros behind its end."""
    part = x[first:first + count]
    return torch.cat([part, part.new_zeros((count - part.shape[0], *part.shape[1:]))])


def exact(case, seed):
    d, kind = _dense(case, seed), case["kind"]
    if kind == "rope":
        return _rope_pairs(d["x"], d["rope"], case["interleaved"], torch.float64)
    lens, layers, n = _lens(case), case["layers"], case["n"]
    if kind == "compact":
        return {name: [torch.stack([_read64(_fresh64(d[name][l][i, :lens[i]]), 0, max(lens)) for i in range(0, n, 2)]) for l in range(layers)]
                for name in ("k", "v")} | {"tables": None}
    if kind == "beam":
        page, got = case["page"], {"k": [], "v": [], "tables": None}
        for l in range(layers):
            for name in ("k", "v"):
                rows = []
                for i in range(n * case["beams"]):
                    p = i // case["beams"]
                    length = lens[p]
                    at, first = length // _BLOCK * _BLOCK, length // page * page
                    rows.append(_read64(_appended64(d[name][l][p, :length], d["new_" + name][l][i][None], at), first, page))
                got[name].append(torch.stack(rows))
        return got
    if kind == "append":
        t, got = case["tokens"], {"q": [], "k": [], "v": []}
        w = _window(t)
        for l in range(layers):
            got["q"].append(_rope_pairs(d["q"][l], d["rope"], case["interleaved"], torch.float64))
            # the keys are rotated in 32 bits before they are stored
            for name, x in (("k", _rope_pairs(d["new_k"][l], d["rope"], case["interleaved"], torch.float32)), ("v", d["new_v"][l].float())):
                rows = []
                for i in range(n):
                    start = lens[i] - t
                    first = start // _BLOCK * _BLOCK
                    rows.append(_read64(_appended64(d[name][l][i, :start], x[i * t:(i + 1) * t], first), first, w))
                got[name].append(torch.stack(rows))
        return got
    out, t, h, g, dim = [], case["tokens"], case["kv_heads"], case["group"], case["dim"]
    for l in range(layers):
        rows = []
        for i, length in enumerate(lens):
            k, v = (_fresh64(d[name][l][i, :length]).transpose(0, 1) for name in ("k", "v"))
            q = d["q"][l][i * t:(i + 1) * t].double().unflatten(1, (h, g)).permute(1, 2, 0, 3)
            part = torch.empty((h, g, t, dim), device=_DEV, dtype=torch.float64)
            j = torch.arange(length, device=_DEV)
            for at in range(0, t, 1024):
                p = torch.arange(at, min(t, at + 1024), device=_DEV)[:, None] + (length - t)
                hidden = j > p
                if case["window"]:
                    hidden |= (j <= p - case["window"]) & (j >= case["sinks"])
                for head in range(h):
                    sc = (q[head, :, at:at + 1024].reshape(-1, dim) @ k[head].t()) / dim ** 0.5
                    sc = sc.unflatten(0, (g, -1)) + torch.zeros(hidden.shape, device=_DEV, dtype=torch.float64).masked_fill(hidden, -torch.inf)
                    part[head, :, at:at + 1024] = torch.softmax(sc, -1) @ v[head]
            rows.append(part.permute(2, 0, 1, 3).reshape(t, h * g, dim))
        out.append(torch.cat(rows))
    return out


def _appended64(held, new, first):
    """Values [tokens, heads, dim] from token `first` (a block's first) on, behind zeros: held [held tokens, ...] and then the new rows."""
    codes = np.zeros((_BLOCK, *new.shape[1:]), np.float32)
    scale = np.full(new.shape[1], _TINY, np.float32)
    begun = held.shape[0] - first
    rows = new.cpu().numpy()
    if begun:
        _block64(codes, scale, 0, held[first:].cpu().numpy())
    values, at = [], begun
    while rows.shape[0]:
        take = min(_BLOCK - at, rows.shape[0])
        _block64(codes, scale, at, rows[:take])
        values.append(codes.astype(np.float64) * scale.astype(np.float64)[:, None])
        rows, at = rows[take:], 0
        if rows.shape[0]:
            codes[:] = 0
    tail = torch.from_numpy(np.concatenate(values)[:held.shape[0] - first + new.shape[0]]).to(_DEV)
    before = _fresh64(held[:first]) if first else tail.new_zeros((0, *tail.shape[1:]))
    return torch.cat([before, tail])

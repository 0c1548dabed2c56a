"""Measured calls of the operators of a block of experts: routing, the experts' products, the norms around a block.

Three kinds of work, over the sizes and types that programs use:

- ``route``: ``Mi355xBackend.route_into``, logits of a router to the experts of each token and their weights.
- ``experts``: ``Experts.apply``, y = sum over a token's experts of weight * down . (act(gate . x) * (up . x)), over GGUF blocks.
- ``norm``: ``Mi355xBackend.norm_into``, h' = h + scale * gate * after(block) and before(h'), with root-mean-square or layer norms.

Routing: an expert's score is softmax(logits) or sigmoid(logit). Chosen are the largest logits, or with a bias the largest score + bias,
of equals the one with the lowest index; with groups only among the experts of the groups whose best one or two have the largest sum. A
logit of minus infinity or NaN is never chosen; where too few are left, the slot's expert is -1 and its weight 0. The weights are the
scores without the bias, divided by their sum if so asked, times a factor.
"""
from __future__ import annotations

import numpy as np
import torch

own = False

_DEV = "cuda:0"
_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
# GGUF blocks: elements, bytes
_BLOCKS = {"Q8_0": (32, 34), "Q4_0": (32, 18), "Q4_K": (256, 144), "Q6_K": (256, 210)}


def listed():
    return [
        # the router of one request's token: a call of a few microseconds
        dict(name="route_t1_e64", kind="route", tokens=1, experts=64, top=8, score="softmax", bias=False, groups=1, top_groups=1, best=1,
             norm=True, type="f32", masked=False),
        # a decode step of many requests, experts in groups with a bias that balances them
        dict(name="route_t61_e256_g8", kind="route", tokens=61, experts=256, top=8, score="sigmoid", bias=True, groups=8, top_groups=4, best=2,
             norm=True, type="f32", masked=False),
        # long prompts together, bf16 logits (so that equal ones are common), some experts masked
        dict(name="route_t16381_e128", kind="route", tokens=16381, experts=128, top=8, score="softmax", bias=False, groups=1, top_groups=1,
             best=1, norm=True, type="bf16", masked=True),
        # one request's token through many small experts
        dict(name="experts_t1_e64_d2048", kind="experts", tokens=1, experts=64, top=8, dim=2048, ffn=1024, up="Q4_K", down="Q6_K", act="silu",
             type="f32", absent=False),
        # drafted tokens of one request through a few large experts
        dict(name="experts_t5_e8_d4096", kind="experts", tokens=5, experts=8, top=2, dim=4096, ffn=14336, up="Q4_K", down="Q6_K", act="silu",
             type="f32", absent=False),
        # a decode step of many requests, bf16
        dict(name="experts_t48_e64_d2048", kind="experts", tokens=48, experts=64, top=6, dim=2048, ffn=1408, up="Q8_0", down="Q8_0", act="silu",
             type="bf16", absent=False),
        # a short prompt in 32 bits; some of the chosen experts are held elsewhere
        dict(name="experts_t509_e32_f32", kind="experts", tokens=509, experts=32, top=4, dim=2048, ffn=1408, up="Q4_0", down="Q4_0", act="gelu",
             type="f32", absent=True),
        # prompts of several requests, many small experts
        dict(name="experts_t4093_e64_d2048", kind="experts", tokens=4093, experts=64, top=8, dim=2048, ffn=1024, up="Q4_K", down="Q6_K",
             act="silu", type="bf16", absent=False),
        # a prompt through a few large experts
        dict(name="experts_t2043_e8_d4096", kind="experts", tokens=2043, experts=8, top=2, dim=4096, ffn=14336, up="Q4_K", down="Q6_K",
             act="silu", type="bf16", absent=False),
        # one request's token: residual and the next block's norm
        dict(name="norm_t1_d4096", kind="norm", tokens=1, dim=4096, after="none", before="rms", gate="none", scale=1.0, block="f32",
             residual="f32", out="f32"),
        # images' patches with a gate for each image, layer norms, no round sizes
        dict(name="norm_t1021_d1152", kind="norm", tokens=1021, dim=1152, after="layer", before="layer", gate="rows", scale=1.0, block="bf16",
             residual="f32", out="bf16"),
        # long prompts, a norm behind the block too
        dict(name="norm_t16381_d4096", kind="norm", tokens=16381, dim=4096, after="rms", before="rms", gate="channels", scale=0.25, block="bf16",
             residual="f32", out="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["route", "experts", "experts", "experts", "norm"])
    if kind == "route":
        experts = rng.choice([8, 16, 32, 60, 64, 96, 128, 160, 256, 384])
        groups = rng.choice([1, 1, 2, 4, 8]) if experts % 8 == 0 and experts > 8 else 1
        top_groups = rng.randint(1, groups)
        return dict(kind=kind, tokens=_log(rng, 1, 16384), experts=experts, top=rng.randint(1, min(10, experts // groups * top_groups)),
                    score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.5, groups=groups, top_groups=top_groups, best=rng.choice([1, 2]),
                    norm=rng.random() < 0.7, type=rng.choice(["f32", "f32", "bf16"]), masked=rng.random() < 0.3)
    if kind == "experts":
        experts, few = rng.choice([4, 8, 16, 32, 60, 64]), rng.random() < 0.5
        up, down = rng.choice([("Q4_K", "Q6_K"), ("Q4_K", "Q4_K"), ("Q6_K", "Q6_K"), ("Q8_0", "Q8_0"), ("Q4_0", "Q4_0"), ("Q4_0", "Q8_0")])
        small = up in ("Q8_0", "Q4_0")
        dim = rng.choice([512, 1024, 1536, 2048, 2560, 4096]) if not small else rng.choice([640, 1024, 1920, 2048, 2560])
        ffn = rng.choice([256, 512, 768, 1024, 1536, 2048]) if not small else rng.choice([384, 640, 768, 896, 1408, 2048])
        return dict(kind=kind, tokens=_log(rng, 1, 64) if few else _log(rng, 65, 2048), experts=experts, top=rng.randint(1, min(8, experts)), dim=dim,
                    ffn=ffn, up=up, down=down, act=rng.choice(["silu", "silu", "gelu", "relu"]),
                    type=rng.choice(["f32", "bf16"]) if few else rng.choice(["f32", "bf16", "bf16", "bf16"]), absent=rng.random() < 0.3)
    dim = rng.choice([64, 1000, 1152, 2048, 2560, 4096, 5120, rng.randint(65, 8192)])
    return dict(kind=kind, tokens=_log(rng, 1, 16000 * 4096 // max(dim, 4096)), dim=dim, after=rng.choice(["none", "none", "rms", "layer"]),
                before=rng.choice(["rms", "rms", "layer"]), gate=rng.choice(["none", "channels", "rows"]), scale=rng.choice([1.0, 0.25, 1.5]),
                block=rng.choice(["f32", "bf16"]), residual=rng.choice(["f32", "f32", "bf16"]), out=rng.choice(["f32", "bf16"]))


# ---- inputs ----------------------------------------------------------------------------------


def _gen(seed):
    return torch.Generator(device=_DEV).manual_seed(seed)


def _blocks(g, kind, experts, rows, cols):
    """GGUF blocks, uint8 [experts, rows, blocks of a row, bytes], of weights about 1 / sqrt(cols) large around 0."""
    elements, size = _BLOCKS[kind]
    shape = (experts, rows, cols // elements)
    b = torch.randint(0, 256, (*shape, size), generator=g, device=_DEV, dtype=torch.uint8)

    def put(at, scale):  # fp16 scales from half of to one and a half times `scale`
        d = (scale * (0.5 + torch.rand(shape, generator=g, device=_DEV))).half()
        b[..., at:at + 2] = d[..., None].view(torch.uint8)

    unit = cols ** -0.5
    if kind == "Q8_0":
        put(0, unit / 74)
    elif kind == "Q4_0":
        put(0, unit / 4.6)
    elif kind == "Q6_K":
        b[..., 192:208] = torch.randint(24, 96, (*shape, 16), generator=g, device=_DEV, dtype=torch.uint8)  # scales of 16 each
        put(208, unit / (18.5 * 60))
    else:
        # scales and minima of 32 each, 6 bits from 20 to 51: the minima lie where half of the codes are, so that the weights lie around 0
        sc = torch.randint(20, 52, (2, *shape, 8), generator=g, device=_DEV, dtype=torch.uint8)
        sc[1] = ((3 * sc[0].int() + sc[1].int()) // 4).to(torch.uint8)
        low, high = sc[..., :4], sc[..., 4:]
        b[..., 4:8] = low[0] | (high[0] >> 4) << 6
        b[..., 8:12] = low[1] | (high[1] >> 4) << 6
        b[..., 12:16] = (high[0] & 15) | (high[1] & 15) << 4
        put(0, unit / (4.6 * 35.5))
        b[..., 2:4] = (b[..., 0:2].contiguous().view(torch.float16).float() * 7.5).half().view(torch.uint8)
    return b


def _activations(g, tokens, dim):
    """Rows of a residual stream behind a norm: N(0, 1), and a few channels several times larger."""
    x = torch.randn((tokens, dim), generator=g, device=_DEV)
    return torch.where(torch.rand((dim,), generator=g, device=_DEV) < 0.01, 6 * x, x)


def _inputs(case, seed):
    g, kind, t = _gen(seed), case["kind"], case["tokens"]
    d = {}
    if kind == "route":
        e = case["experts"]
        x = 2 * torch.randn((t, e), generator=g, device=_DEV) + 0.5 * torch.randn((e,), generator=g, device=_DEV)
        if case["masked"]:  # a twentieth of all, and whole rows but for a few
            hidden = torch.rand((t, e), generator=g, device=_DEV) < 0.05
            hidden |= (torch.arange(t, device=_DEV)[:, None] % 97 == 5) & (torch.arange(e, device=_DEV) > 2)
            x = x.masked_fill(hidden, float("-inf"))
        d["logits"] = x.to(_TYPES[case["type"]])
        d["bias"] = 0.2 * torch.randn((e,), generator=g, device=_DEV)
    elif kind == "experts":
        e, k, dim, ffn = case["experts"], case["top"], case["dim"], case["ffn"]
        d["x"] = _activations(g, t, dim).to(_TYPES[case["type"]])
        # some experts are chosen more often than others
        logits = torch.randn((t, e), generator=g, device=_DEV) + 0.5 * torch.randn((e,), generator=g, device=_DEV)
        top, ids = torch.topk(torch.softmax(logits, -1), k)
        if case["absent"]:
            ids = ids.masked_fill(torch.rand((t, k), generator=g, device=_DEV) < 0.2, -1)
        d["ids"], d["weights"] = ids.int(), (top / top.sum(-1, keepdim=True)).contiguous()
        d["gate"], d["up"] = (_blocks(g, case["up"], e, ffn, dim) for _ in range(2))
        d["down"] = _blocks(g, case["down"], e, dim, ffn)
    else:
        dim = case["dim"]
        d["block"] = _activations(g, t, dim).to(_TYPES[case["block"]])
        d["residual"] = (3 * _activations(g, t, dim) + 0.3).to(_TYPES[case["residual"]])
        for name in ("after", "before"):
            d[name] = 1 + 0.2 * torch.randn((dim,), generator=g, device=_DEV)
            d[name + "_bias"] = 0.1 * torch.randn((dim,), generator=g, device=_DEV)
        every = _every(case)
        d["gate"] = 0.5 + torch.rand((-(-t // every) if case["gate"] == "rows" else 1, dim), generator=g, device=_DEV)
    return d


def _every(case):
    """Rows that share a gate where there are several: an image's, say."""
    return max(1, case["tokens"] // 4)


# ---- the framework's side --------------------------------------------------------------------


def _prepare_own(s, case, d):
    from jax4j_amd import DType, Experts, Mi355xBackend, Norm, QuantType

    s.be = Mi355xBackend()
    s.types = {"f32": DType.F32, "bf16": DType.BF16}
    kind, t = case["kind"], case["tokens"]
    if kind == "route":
        s.ids = torch.empty((t, case["top"]), device=_DEV, dtype=torch.int32)
        s.weights = torch.empty((t, case["top"]), device=_DEV)
    elif kind == "experts":
        s.kept = []
        for name, typ in (("gate", "up"), ("up", "up"), ("down", "down")):
            b = d[name]
            e, rows, per, _ = b.shape
            torch.cuda.synchronize()
            s.kept.append(s.be.upload_quantized_device(b.data_ptr(), b.numel(), QuantType[case[typ]], (e * rows, per * _BLOCKS[case[typ]][0])))
        s.experts = Experts(s.be, *s.kept, experts=case["experts"], activation=case["act"])
        s.out = torch.empty_like(d["x"])
    else:
        s.out = torch.empty(d["block"].shape, device=_DEV, dtype=_TYPES[case["out"]])
        s.h = torch.empty_like(d["residual"])
        s.norms = {}
        for name in ("after", "before"):
            if case[name] != "none":
                s.norms[name] = Norm(d[name].data_ptr(), case[name], bias_ptr=d[name + "_bias"].data_ptr() if case[name] == "layer" else 0, eps=1e-6)
    return s


def _run_own(s):
    case, d, kind = s.case, s.d, s.case["kind"]
    if kind == "route":
        s.be.route_into(d["logits"].data_ptr(), s.ids.data_ptr(), s.weights.data_ptr(), case["tokens"], case["experts"], case["top"],
                        dtype=s.types[case["type"]], score=case["score"], bias_ptr=d["bias"].data_ptr() if case["bias"] else 0, groups=case["groups"],
                        top_groups=case["top_groups"], group_best=case["best"], renormalize=case["norm"], scale=1.5)
        return {"ids": s.ids, "weights": s.weights}
    if kind == "experts":
        s.experts.apply(d["x"].data_ptr(), d["ids"].data_ptr(), d["weights"].data_ptr(), s.out.data_ptr(), case["tokens"], case["top"],
                        s.types[case["type"]])
        return s.out
    gated = case["gate"] != "none"
    s.be.norm_into(d["residual"].data_ptr(), s.out.data_ptr(), case["tokens"], case["dim"], s.norms["before"],
                   residual_type=s.types[case["residual"]], out_type=s.types[case["out"]], block_ptr=d["block"].data_ptr(),
                   block_type=s.types[case["block"]], after=s.norms.get("after"), gate_ptr=d["gate"].data_ptr() if gated else 0,
                   gate_every=_every(case) if case["gate"] == "rows" else 0, scale=case["scale"], residual_out_ptr=s.h.data_ptr())
    return {"h": s.h, "y": s.out}


# ---- the plain form --------------------------------------------------------------------------


def _route_plain(case, d):
    x, e, k = d["logits"].double(), case["experts"], case["top"]
    low = torch.full((), float("-inf"), device=_DEV, dtype=torch.float64)
    x = torch.where(torch.isnan(x), low, x)
    if case["score"] == "softmax":
        top = x.amax(-1, keepdim=True)
        p = torch.exp(x - torch.where(torch.isinf(top), torch.zeros_like(top), top))
        score = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    else:
        score = 1 / (1 + torch.exp(-x))
    key = torch.where(x > low, score + d["bias"].double(), low) if case["bias"] else x
    if case["groups"] > 1:
        inside = key.unflatten(1, (case["groups"], -1))
        best = torch.sort(inside, dim=-1, descending=True, stable=True).values[..., :case["best"]]
        some = best[..., 0] > low
        rank = torch.where(best > low, best, torch.zeros_like(best)).sum(-1)
        rank = torch.where(some, rank, low)
        keep = torch.sort(rank, dim=-1, descending=True, stable=True).indices[:, :case["top_groups"]]
        kept = torch.zeros_like(some).scatter_(1, keep, True) & some
        key = torch.where(kept[..., None], inside, low).flatten(1)
    key, ids = torch.sort(key, dim=-1, descending=True, stable=True)
    key, ids = key[:, :k], ids[:, :k]
    none = key == low
    w = torch.where(none, torch.zeros_like(key), torch.gather(score, 1, ids))
    if case["norm"]:
        w = w / w.sum(-1, keepdim=True).clamp_min(1e-300)
    return {"ids": torch.where(none, torch.full_like(ids, -1), ids).int(), "weights": (1.5 * w).float()}


def _half(b):
    return b.contiguous().view(torch.float16).float()


def _weights(b, kind):
    """fp32 weights [experts, rows, cols] of GGUF blocks."""
    e, rows = b.shape[:2]
    if kind == "Q8_0":
        w = b[..., 2:].contiguous().view(torch.int8).float() * _half(b[..., :2])
    elif kind == "Q4_0":
        q = b[..., 2:]
        w = (torch.cat([q & 15, q >> 4], -1).float() - 8) * _half(b[..., :2])
    elif kind == "Q4_K":
        s = b[..., 4:16]
        scale = torch.cat([s[..., :4] & 63, (s[..., 8:] & 15) | (s[..., :4] >> 6) << 4], -1).float() * _half(b[..., :2])
        low = torch.cat([s[..., 4:8] & 63, (s[..., 8:] >> 4) | (s[..., 4:8] >> 6) << 4], -1).float() * _half(b[..., 2:4])
        q = b[..., 16:].unflatten(-1, (4, 32))
        q = torch.stack([q & 15, q >> 4], -2).flatten(-3, -2).float()  # 8 sub-blocks of 32
        w = (q * scale[..., None] - low[..., None]).flatten(-2)
    else:
        ql, qh = b[..., :128].unflatten(-1, (2, 2, 32)), b[..., 128:192].unflatten(-1, (2, 32))
        low = torch.stack([ql[..., 0, :] & 15, ql[..., 1, :] & 15, ql[..., 0, :] >> 4, ql[..., 1, :] >> 4], -2)
        high = torch.stack([qh & 3, qh >> 2 & 3, qh >> 4 & 3, qh >> 6], -2)
        q = (low | high << 4).flatten(-3).unflatten(-1, (16, 16)).float() - 32
        scale = b[..., 192:208].contiguous().view(torch.int8).float() * _half(b[..., 208:210])
        w = (q * scale[..., None]).flatten(-2)
    return w.reshape(e, rows, -1)


def _act(x, name):
    if name == "relu":
        return x.clamp_min(0)
    if name == "gelu":
        return 0.5 * x * (1 + torch.tanh(0.7978845608028654 * (x + 0.044715 * x * x * x)))
    return x / (1 + torch.exp(-x))


def _experts_plain(case, d):
    ids, w = d["ids"].long().reshape(-1), torch.where(d["ids"] >= 0, d["weights"], torch.zeros_like(d["weights"])).reshape(-1)
    k = case["top"]
    used, at = torch.unique(ids.clamp_min(0), return_inverse=True)  # the experts that tokens have chosen, and each pair's place among them
    order = torch.argsort(at, stable=True)
    count = torch.bincount(at, minlength=used.numel())
    place = torch.empty_like(at)
    place[order] = torch.arange(at.numel(), device=_DEV) - (torch.cumsum(count, 0) - count)[at[order]]
    x = torch.zeros((used.numel(), case["dim"], int(count.max())), device=_DEV)
    x[at, :, place] = d["x"].float().repeat_interleave(k, 0)
    h = _act(torch.bmm(_weights(d["gate"][used], case["up"]), x), case["act"]) * torch.bmm(_weights(d["up"][used], case["up"]), x)
    y = torch.bmm(_weights(d["down"][used], case["down"]), h)[at, :, place]
    return (y * w[:, None]).unflatten(0, (-1, k)).sum(1).to(_TYPES[case["type"]])


def _normed(x, kind, weight, bias):
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    y = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * weight
    return y + bias if kind == "layer" else y


def _norm_plain(case, d):
    b = d["block"].float()
    if case["after"] != "none":
        b = _normed(b, case["after"], d["after"], d["after_bias"])
    if case["gate"] == "channels":
        b = b * d["gate"]
    elif case["gate"] == "rows":
        b = b * d["gate"].repeat_interleave(_every(case), 0)[:b.shape[0]]
    h = d["residual"].float() + case["scale"] * b
    return {"h": h.to(d["residual"].dtype), "y": _normed(h, case["before"], d["before"], d["before_bias"]).to(_TYPES[case["out"]])}


# ---- what is measured ------------------------------------------------------------------------


class _State:
    """What a program holds between calls; gives the engine's memory back when it goes."""

    experts, kept = None, ()

    def __del__(self):
        if self.experts is not None:
            torch.cuda.synchronize()
            self.experts.destroy()
        for w in self.kept:
            self.be.release(w)


def prepare(case, seed):
    s = _State()
    s.case, s.d = case, _inputs(case, seed)
    if own:
        s = _prepare_own(s, case, s.d)
        for name in ("gate", "up", "down") if case["kind"] == "experts" else ():  # in the engine now
            s.d.pop(name)
    torch.cuda.synchronize()
    return s


def run(s):
    if own:
        return _run_own(s)
    return {"route": _route_plain, "experts": _experts_plain, "norm": _norm_plain}[s.case["kind"]](s.case, s.d)


def work(case):
    kind, t = case["kind"], case["tokens"]
    if kind == "route":
        e, k = case["experts"], case["top"]
        return {"bytes": t * e * (4 if case["type"] == "f32" else 2) + 8 * t * k, "flops": 4 * t * e}
    if kind == "norm":
        size = {"f32": 4, "bf16": 2}
        gate = {"none": 0, "channels": 4 * case["dim"], "rows": 4 * case["dim"] * -(-t // _every(case))}[case["gate"]]
        return {"bytes": t * case["dim"] * (size[case["block"]] + 2 * size[case["residual"]] + size[case["out"]]) + gate, "flops": 10 * t * case["dim"]}
    e, k, dim, ffn = case["experts"], case["top"], case["dim"], case["ffn"]
    touched = e * (1 - (1 - k / e) ** t)  # experts that some token chooses, were all as likely

    def of(name):
        elements, size = _BLOCKS[case[name]]
        return size / elements

    weights = touched * dim * ffn * (2 * of("up") + of("down"))
    return {"bytes": weights + 2 * t * dim * (4 if case["type"] == "f32" else 2) + 8 * t * k, "flops": 6 * t * k * dim * ffn * (0.8 if case["absent"] else 1)}


# ---- the definition in 64 bits ---------------------------------------------------------------


def _route64(case, d):
    """Token by token: the weights in the order of the choice."""
    x, k = d["logits"].double().cpu().numpy(), case["top"]
    bias, groups = d["bias"].double().cpu().numpy(), case["groups"]
    e = x.shape[1]
    out = np.zeros((x.shape[0], k))
    index = np.arange(e)
    for r in range(x.shape[0]):
        row = x[r]
        live = row > -np.inf
        score = np.zeros(e)
        if case["score"] == "softmax":
            if live.any():
                score[live] = np.exp(row[live] - row[live].max())
                score /= score.sum()
        else:
            score[live] = 1 / (1 + np.exp(-row[live]))
        key = score + bias if case["bias"] else row
        live = live.copy()
        if groups > 1:
            size = e // groups
            rank = []
            for j in range(groups):
                inside = np.sort(key[j * size:(j + 1) * size][live[j * size:(j + 1) * size]])[::-1][:case["best"]]
                rank.append(inside.sum() if inside.size else -np.inf)
            chosen = sorted(range(groups), key=lambda j: (-rank[j], j))[:case["top_groups"]]
            live &= np.isin(index // size, chosen)
        at = index[live]
        best = at[np.lexsort((at, -key[at]))][:k]
        w = score[best]
        out[r, :best.size] = 1.5 * (w / w.sum() if case["norm"] and best.size else w)
    return {"ids": None, "weights": torch.from_numpy(out)}


def _weights64(b, kind):
    """Weights [rows, cols] in 64 bits of one expert's blocks, element by element of a block."""
    b = b.to(torch.int32)
    half = lambda at: (b[..., at] | b[..., at + 1] << 8).to(torch.int16).view(torch.float16).double()  # noqa: E731
    signed = lambda v: torch.where(v > 127, v - 256, v)  # noqa: E731
    out = []
    elements = _BLOCKS[kind][0]
    for i in range(elements):
        if kind == "Q8_0":
            out.append(half(0) * signed(b[..., 2 + i]))
        elif kind == "Q4_0":
            out.append(half(0) * ((b[..., 2 + i % 16] >> 4 * (i // 16) & 15) - 8))
        elif kind == "Q4_K":
            j = i // 32  # sub-block
            if j < 4:
                sc, mn = b[..., 4 + j] & 63, b[..., 8 + j] & 63
            else:
                sc, mn = b[..., 8 + j] & 15 | b[..., j] >> 6 << 4, b[..., 8 + j] >> 4 | b[..., 4 + j] >> 6 << 4
            out.append(half(0) * sc * (b[..., 16 + 32 * (j // 2) + i % 32] >> 4 * (j % 2) & 15) - half(2) * mn)
        else:
            part, r = i // 128, i % 128
            q = b[..., 64 * part + r % 64] >> 4 * (r // 64) & 15 | (b[..., 128 + 32 * part + r % 32] >> 2 * (r // 32) & 3) << 4
            out.append(half(208) * signed(b[..., 192 + i // 16]) * (q - 32))
    return torch.stack(out, -1).flatten(-2)


def _experts64(case, d):
    x, ids, w = d["x"].double(), d["ids"].long(), d["weights"].double()
    y = torch.zeros_like(x)
    for e in range(case["experts"]):
        token, slot = torch.where(ids == e)
        if not token.numel():
            continue
        g, u = x[token] @ _weights64(d["gate"][e], case["up"]).t(), x[token] @ _weights64(d["up"][e], case["up"]).t()
        if case["act"] == "relu":
            a = torch.relu(g)
        elif case["act"] == "gelu":
            a = g / 2 * (1 + torch.tanh((2 / np.pi) ** 0.5 * (g + 0.044715 * g ** 3)))
        else:
            a = g * torch.sigmoid(g)
        y.index_add_(0, token, w[token, slot][:, None] * ((a * u) @ _weights64(d["down"][e], case["down"]).t()))
    return y


def _norm64(case, d):
    def norm(x, name):
        if case[name] == "none":
            return x
        if case[name] == "layer":
            return (x - x.mean(1)[:, None]) / torch.sqrt(x.var(1, unbiased=False) + 1e-6)[:, None] * d[name].double() + d[name + "_bias"].double()
        return x / torch.sqrt((x ** 2).mean(1) + 1e-6)[:, None] * d[name].double()

    b = norm(d["block"].double(), "after")
    if case["gate"] != "none":
        row = torch.arange(b.shape[0], device=_DEV) // _every(case) if case["gate"] == "rows" else torch.zeros(b.shape[0], device=_DEV, dtype=torch.long)
        b = b * d["gate"].double()[row]
    h = d["residual"].double() + case["scale"] * b
    return {"h": h, "y": norm(h, "before")}


def exact(case, seed):
    d = _inputs(case, seed)
    return {"route": _route64, "experts": _experts64, "norm": _norm64}[case["kind"]](case, d)

"""The operators of a decoding step over a long context as measured cases: rotary positions scaled for long
contexts, the cache held in 8 bits, the attention over it, and sampling from the logits on the device.

A program of this framework enqueues a step's operators in one open sequence of its context and waits once, at
the sequence's end; a pass here is one operator's share of that.  The device memory is the caller's (torch
tensors), seen through wrapped buffers, which `prepare` makes.

The cache's layout, one layer: K codes [kv head][position][dim], V codes [kv head][block of 32][dim][position in
the block], both int8 with positions rounded up to whole blocks, and float32 scales [kv head][block].
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda"
BLOCK = 32  # positions that share a scale
NONE, LINEAR, YARN, BANDS = 0, 1, 2, 3
_context = []


def _own_context():
    """The package and the process's context, its sequence open."""
    if not _context:
        sys.path.insert(0, os.path.join(os.getcwd(), "ziggy-llm_amd"))
        from zhip import hip
        ctx = hip.Context(0)
        ctx.begin()
        _context.extend((hip, ctx))
    return _context


# ---- cases ----

def _rope(name, rows, heads, hd, rd, style, scaling, base, factor, orig, low, high, first, spread, factors):
    return dict(name=name, op="rope", rows=rows, heads=heads, hd=hd, rd=rd, style=style, scaling=scaling, base=base,
                factor=factor, orig=orig, low=low, high=high, magnitude=1.0 + 0.125 * (scaling == YARN), first=first,
                spread=spread, factors=factors)


def _store(name, rows, kvh, hd, position, layer):
    return dict(name=name, op="store", rows=rows, kvh=kvh, hd=hd, position=position, layer=layer)


def _attend(name, queries, heads, kvh, hd, position, window, layer):
    return dict(name=name, op="attend", queries=queries, heads=heads, kvh=kvh, hd=hd, position=position,
                window=window, layer=layer)


def _sample(name, rows, vocab, temperature, top_k, top_p, min_p, penalty, recent):
    return dict(name=name, op="sample", rows=rows, vocab=vocab, temperature=temperature, top_k=top_k, top_p=top_p,
                min_p=min_p, penalty=penalty, recent=recent)


def listed():
    return [
        # a decoding step's query and key heads of one token, frequencies in bands
        _rope("rope_step", 1, 40, 128, 128, 0, BANDS, 500000.0, 8.0, 8192, 1.0, 4.0, 100000, False, False),
        # half of each head of an odd number of rows at positions in no order, with factors per pair
        _rope("rope_partial", 333, 9, 96, 48, 1, LINEAR, 10000.0, 4.0, 0, 0.0, 0.0, 7, True, True),
        # a prompt's query and key heads
        _rope("rope_prompt", 4096, 40, 128, 128, 1, YARN, 1000000.0, 4.0, 32768, 1.0, 32.0, 65536, False, False),
        # a decoding step's key and value, inside a block
        _store("store_step", 1, 8, 128, 4113, 1),
        # a prompt's keys and values after 1000 cached rows
        _store("store_prompt", 4095, 8, 128, 1000, 0),
        # one step after a short chat, small heads
        _attend("attend_chat", 1, 32, 4, 64, 150, 0, 3),
        # decoding at 4k and at the end of a long context
        _attend("attend_4k", 1, 32, 8, 128, 4112, 0, 2),
        _attend("attend_128k", 1, 32, 8, 128, 131070, 0, 0),
        # a verify pass: the pending token and 8 drafts
        _attend("attend_verify", 9, 32, 8, 128, 16389, 0, 0),
        # the second half of a prompt
        _attend("attend_prompt", 2048, 32, 8, 128, 14336, 0, 0),
        # a chat's next token from the 40 best, with a repeat penalty
        _sample("sample_top40", 1, 128256, 0.8, 40, 0.9, 0.0, 1.1, 512),
        # a nucleus of the whole vocabulary for the rows of a verify pass
        _sample("sample_nucleus", 16, 151936, 1.0, 0, 0.95, 0.02, 1.0, 0),
    ]


def _log(rng, lo, hi):
    return min(hi, int(lo * math.exp(rng.random() * math.log((hi + 1) / lo))))


def draw(rng):
    op = rng.choice(["rope", "store", "attend", "attend", "sample"])
    if op == "rope":
        hd = rng.choice([64, 80, 96, 128, 256])
        rows, heads = _log(rng, 1, 4096), _log(rng, 1, 40 * 128 // hd)
        scaling = rng.choice([NONE, LINEAR, YARN, BANDS])
        c = _rope("", rows, heads, hd, hd if rng.random() < 0.6 else 2 * rng.randint(1, hd // 2), rng.choice([0, 1]),
                  scaling, rng.choice([10000.0, 500000.0, 1000000.0]), 1.0 + rng.randint(1, 64) / 4.0,
                  rng.choice([4096, 8192, 32768]), 1.0, float(rng.choice([4, 32])), _log(rng, 1, 1000000),
                  rng.random() < 0.5, rng.random() < 0.3)
    elif op == "store":
        hd = rng.choice([64, 96, 128, 256])
        c = _store("", _log(rng, 1, 4095 * 128 // max(hd, 128)), _log(rng, 1, 8), hd, _log(rng, 1, 8192) - 1,
                   rng.choice([0, 1]))
    elif op == "attend":
        hd = rng.choice([64, 96, 128, 256])
        kvh = _log(rng, 1, 8)
        heads = kvh * rng.randint(1, 4 * 128 // max(hd, 128))
        if rng.random() < 0.6:  # single tokens and verify passes, over caches of any length
            queries, position = rng.choice([1, 1, 1, rng.randint(2, 16)]), _log(rng, 1, 100000) - 1
        else:
            queries, position = _log(rng, 17, 2048), _log(rng, 1, 14000) - 1
        c = _attend("", queries, heads, kvh, hd, position, rng.choice([0, 0, 0, _log(rng, 16, 4096)]), rng.choice([0, 1]))
    else:
        limited = rng.random() < 0.5
        penalised = rng.random() < 0.5
        c = _sample("", _log(rng, 1, 16), _log(rng, 1000, 151936), round(0.3 + 1.2 * rng.random(), 2),
                    _log(rng, 1, 1000) if limited else 0, rng.choice([1.0, round(0.3 + 0.69 * rng.random(), 2)]),
                    rng.choice([0.0, 0.0, round(0.2 * rng.random(), 3)]), 1.15 if penalised else 1.0,
                    _log(rng, 16, 2048) if penalised else 0)
    del c["name"]
    return c


# ---- inputs ----

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _f32(x):
    return float(torch.tensor(x, dtype=torch.float32))


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _uniform(g, *shape):
    return torch.rand(shape, generator=g, device=DEV)


def _blocks(n):
    return -(-n // BLOCK)


def _cache(g, layers, kvh, hd, positions):
    """Codes as rows of a normal distribution give them, scales that give values near 1."""
    nb = _blocks(positions)

    def codes(*shape):
        out = torch.empty(shape, dtype=torch.int8, device=DEV)
        for layer in range(shape[0]):
            out[layer] = (32 * _randn(g, *shape[1:])).round_().clamp_(-127, 127).to(torch.int8)
        return out

    def scales():
        return (0.75 + 0.5 * _uniform(g, layers, kvh, nb)) / 32

    return dict(kc=codes(layers, kvh, nb * BLOCK, hd), vc=codes(layers, kvh, nb, hd, BLOCK), ks=scales(), vs=scales())


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = dict(case=c)
    if c["op"] == "rope":
        # rows as a fused projection leaves them: the rotated heads, then values that stay
        s["x"] = _randn(g, c["rows"], (c["heads"] + 2) * c["hd"])
        s["y"] = torch.zeros(c["rows"], c["heads"] * c["hd"], device=DEV)
        at = torch.arange(c["rows"], device=DEV, dtype=torch.int32) + c["first"]
        s["at"] = at[torch.randperm(c["rows"], generator=g, device=DEV)].contiguous() if c["spread"] else at
        s["factors"] = 1.0 + 3.0 * _uniform(g, c["rd"] // 2) if c["factors"] else None
    elif c["op"] == "store":
        s["n"] = c["position"] + c["rows"] + 5
        s.update(_cache(g, c["layer"] + 1, c["kvh"], c["hd"], s["n"]))
        # keys and values beside the queries of a fused projection; a few large channels, as keys have
        s["x"] = _randn(g, c["rows"], 4, c["kvh"] * c["hd"])
        s["x"][:, :, ::37] *= 4
        s["from"] = c["position"] // BLOCK * BLOCK
        n = c["position"] + c["rows"] - s["from"]
        s["k"], s["v"] = (torch.zeros(n, c["kvh"] * c["hd"], device=DEV) for _ in range(2))
    elif c["op"] == "attend":
        s["n"] = c["position"] + c["queries"]
        s.update(_cache(g, c["layer"] + 1, c["kvh"], c["hd"], s["n"]))
        s["q"] = 1.5 * _randn(g, c["queries"], c["heads"] * c["hd"])
        s["y"] = torch.zeros_like(s["q"])
    else:
        # a model's logits: a broad body, and the few tokens that it is sure of
        s["x"] = 2.0 * _randn(g, c["rows"], c["vocab"])
        best = torch.randint(0, c["vocab"], (c["rows"], 24), generator=g, device=DEV)
        s["x"].scatter_(1, best, 6.0 + 4.0 * _randn(g, c["rows"], 24))
        s["u"] = torch.rand(c["rows"], generator=g, device=DEV, dtype=torch.float64)
        s["recent"] = None
        if c["recent"]:  # tokens so far, the likely ones among them
            s["recent"] = torch.randint(0, c["vocab"], (c["rows"], c["recent"]), generator=g, device=DEV, dtype=torch.int32)
            s["recent"][:, :8] = best[:, :8].to(torch.int32)
        s["y"] = torch.zeros(c["rows"], dtype=torch.int32, device=DEV)
    if own:
        hip, ctx = _own_context()
        s["ctx"] = ctx
        s["own"] = {k: ctx.wrap(v.data_ptr(), v.numel() * v.element_size())
                    for k, v in s.items() if isinstance(v, torch.Tensor)}
        if c["op"] == "rope":
            s["desc"] = hip.RopeDesc(head_dim=c["hd"], rope_dim=c["rd"], style=c["style"], base=c["base"],
                                     scaling=c["scaling"], factor=c["factor"], original_context=c["orig"],
                                     low=c["low"], high=c["high"], magnitude=c["magnitude"])
        elif c["op"] in ("store", "attend"):
            b = s["own"]
            s["cache"] = hip.Kv8Cache(b["kc"], b["ks"], b["vc"], b["vs"], layers=c["layer"] + 1, heads_kv=c["kvh"],
                                      head_dim=c["hd"], context=s["n"])
        else:
            s["options"] = hip.SamplingOptions(temperature=c["temperature"], repeat_penalty=c["penalty"],
                                               top_k=c["top_k"], top_p=c["top_p"], min_p=c["min_p"])
        torch.cuda.synchronize()  # the context's stream is another than the one that made the inputs
    return s


# ---- the operators in their plain form ----

def _frequencies(c):
    """Radians a position, in 64 bits."""
    d = c["rd"]
    i = torch.arange(d // 2, device=DEV, dtype=torch.float64)
    f = torch.exp(i * (-2.0 / d * math.log(c["base"])))
    if c["scaling"] == LINEAR:
        return f / c["factor"]
    if c["scaling"] == YARN:
        def pair_of(turns):
            return d * math.log(c["orig"] / (2 * math.pi * turns)) / (2 * math.log(c["base"]))

        lo, hi = max(0, math.floor(pair_of(c["high"]))), min(d - 1, math.ceil(pair_of(c["low"])))
        keep = 1 - ((i - lo) / max(0.001, hi - lo)).clamp(0, 1)
        return f / c["factor"] * (1 - keep) + f * keep
    if c["scaling"] == BANDS:
        turns = c["orig"] * f / (2 * math.pi)
        keep = ((turns - c["low"]) / (c["high"] - c["low"])).clamp(0, 1)
        return f / c["factor"] * (1 - keep) + f * keep
    return f


def _plain_rope(s):
    c = s["case"]
    f = _frequencies(c)
    if s["factors"] is not None:
        f = f / s["factors"].double()
    angle = torch.remainder(s["at"].double()[:, None] * f, 2 * math.pi)
    cos, sin = ((m(angle) * _f32(c["magnitude"])).float()[:, None, :] for m in (torch.cos, torch.sin))
    x = s["x"][:, :c["heads"] * c["hd"]].reshape(c["rows"], c["heads"], c["hd"])
    y, half = x.clone(), c["rd"] // 2
    a, b = (slice(0, half), slice(half, c["rd"])) if c["style"] else (slice(0, c["rd"], 2), slice(1, c["rd"], 2))
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., a] * sin + x[..., b] * cos
    return y.reshape(c["rows"], -1)


def _plain_store(s):
    c = s["case"]
    first, end = s["from"] // BLOCK, _blocks(c["position"] + c["rows"])
    back = c["position"] - s["from"]  # rows of the first block that are there already
    at = torch.arange(first * BLOCK, end * BLOCK, device=DEV)
    new = ((at >= c["position"]) & (at < c["position"] + c["rows"])).reshape(1, -1, BLOCK, 1)
    out = []
    for codes, scales, part in ((s["kc"], s["ks"], 2), (s["vc"], s["vs"], 3)):
        held = codes[c["layer"]].reshape(c["kvh"], -1, BLOCK, c["hd"]) if part == 2 else codes[c["layer"]].transpose(2, 3)
        held, scale = held[:, first:end], scales[c["layer"], :, first:end]
        x = torch.zeros(end * BLOCK - s["from"], c["kvh"], c["hd"], device=DEV)
        x[back:back + c["rows"]] = s["x"][:, part].reshape(c["rows"], c["kvh"], c["hd"])
        x = x.permute(1, 0, 2).reshape(c["kvh"], -1, BLOCK, c["hd"])
        was = torch.zeros_like(scale)
        if back:
            was[:, 0] = scale[:, 0]
        now = torch.maximum(was, x.abs().amax(dim=(2, 3)) / 127)
        wide = now.double()[:, :, None, None]
        old = held.double() * was.double()[:, :, None, None]
        kept = at.reshape(1, -1, BLOCK, 1) < c["position"]
        q = torch.where(new, x.double(), torch.where(kept, old, torch.zeros_like(old))) / wide
        q = q.nan_to_num(0.0).round().clamp(-127, 127).to(torch.int8)
        q = torch.where(new | kept, q, held)
        scale.copy_(now)
        held.copy_(q)
        rows = (q.float() * now[:, :, None, None]).reshape(c["kvh"], -1, c["hd"])[:, :back + c["rows"]]
        out.append(rows.permute(1, 0, 2).reshape(back + c["rows"], -1).contiguous())
    return out


def _plain_attend(s):
    c = s["case"]
    group, nb = c["heads"] // c["kvh"], _blocks(s["n"])
    k = s["kc"][c["layer"]].reshape(c["kvh"], nb, BLOCK, -1).float() * s["ks"][c["layer"]][:, :, None, None]
    v = s["vc"][c["layer"]].float() * s["vs"][c["layer"]][:, :, None, None]
    k = k.reshape(c["kvh"], nb * BLOCK, -1)[:, :s["n"]].transpose(1, 2).contiguous()
    v = v.transpose(2, 3).reshape(c["kvh"], nb * BLOCK, -1)[:, :s["n"]].contiguous()
    q = s["q"].reshape(c["queries"], c["kvh"], group, -1).permute(1, 2, 0, 3).reshape(c["kvh"], group * c["queries"], -1)
    p = torch.matmul(q.contiguous(), k).mul_(_f32(c["hd"] ** -0.5)).reshape(c["kvh"], group, c["queries"], -1)
    at = torch.arange(s["n"], device=DEV)
    of = torch.arange(c["queries"], device=DEV)[:, None] + c["position"]
    hidden = at > of
    if c["window"]:
        hidden = hidden | (at <= of - c["window"])
    p.masked_fill_(hidden, -math.inf)
    p = p.sub_(p.amax(dim=-1, keepdim=True)).exp_()
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.reshape(c["kvh"], group * c["queries"], -1), v).reshape(c["kvh"], group, c["queries"], -1) / total
    return o.permute(2, 0, 1, 3).reshape(c["queries"], -1).contiguous()


def _plain_sample(s):
    c, x = s["case"], s["x"]
    a = x
    if s["recent"] is not None:
        seen = torch.zeros(x.shape, dtype=torch.bool, device=DEV).scatter_(1, s["recent"].long(), True)
        p = torch.tensor(c["penalty"], dtype=torch.float32, device=DEV)
        a = torch.where(seen, torch.where(x < 0, x * p, x / p), x)
    order = None
    if 0 < c["top_k"] < c["vocab"]:
        order = torch.argsort(x, dim=1, descending=True, stable=True)[:, :c["top_k"]]
        a = a.gather(1, order)
    w = torch.exp((a.double() - a.amax(dim=1, keepdim=True).double()) / _f32(c["temperature"]))
    if c["min_p"] > 0:
        w = torch.where(w >= _f32(c["min_p"]), w, torch.zeros_like(w))
    if c["top_p"] < 1:
        by = torch.argsort(w, dim=1, descending=True, stable=True)
        w = w.gather(1, by)
        order = by if order is None else order.gather(1, by)
        share = w.cumsum(1) / w.sum(1, keepdim=True)
        before = (share < _f32(c["top_p"])).to(torch.int32).cumsum(1)  # a token stays if the share before it is below top_p
        rank = torch.arange(w.shape[1], device=DEV)
        w = torch.where(before >= rank, w, torch.zeros_like(w))
    reached = (w.cumsum(1) >= s["u"][:, None] * w.sum(1, keepdim=True)) & (w > 0)
    at = reached.to(torch.int32).argmax(dim=1, keepdim=True)
    return (at if order is None else order.gather(1, at))[:, 0].to(torch.int32)


# ---- one pass ----

def run(state):
    s, c = state, state["case"]
    if own:
        ctx, b = s["ctx"], s["own"]
        if c["op"] == "rope":
            ctx.rope_rows(s["desc"], b["x"], b["y"], c["rows"], c["heads"], positions=b["at"],
                          src_stride=(c["heads"] + 2) * c["hd"], freq_factors=b.get("factors"))
            return s["y"]
        if c["op"] == "store":
            w = c["kvh"] * c["hd"]
            ctx.kv8_store(s["cache"], b["x"], b["x"], c["layer"], c["position"], c["rows"], row_stride=4 * w,
                          k_off=8 * w, v_off=12 * w)
            ctx.kv8_load(s["cache"], b["k"], b["v"], c["layer"], s["from"], s["k"].shape[0])
            return [s["k"], s["v"]]
        if c["op"] == "attend":
            ctx.kv8_attention(s["cache"], b["q"], b["y"], c["heads"], c["layer"], c["position"], c["queries"],
                              window=c["window"])
            return s["y"]
        ctx.sample_rows(b["x"], b["y"], b["u"], s["options"], c["rows"], c["vocab"], recent=b.get("recent"),
                        recent_count=c["recent"])
        return s["y"]
    return {"rope": _plain_rope, "store": _plain_store, "attend": _plain_attend, "sample": _plain_sample}[c["op"]](s)


def _pairs(c):
    """(query, position) pairs that the mask leaves."""
    n = 0
    for i in range(c["queries"]):
        n += min(c["position"] + i + 1, c["window"] or c["position"] + i + 1)
    return n


def work(case):
    c = case
    if c["op"] == "rope":
        return {"bytes": 8 * c["rows"] * c["heads"] * c["hd"] + 4 * c["rows"], "flops": 3 * c["rows"] * c["heads"] * c["rd"]}
    if c["op"] == "store":  # rows in and codes out, and the read-back: codes in and rows out
        n = 2 * c["rows"] * c["kvh"] * c["hd"]
        return {"bytes": (4 + 1 + 1 + 4) * n, "flops": 4 * n}
    if c["op"] == "attend":
        seen = c["position"] + c["queries"]
        if c["window"]:
            seen = min(seen, c["window"] + c["queries"] - 1)
        cache = 2 * c["kvh"] * (seen * c["hd"] + 4 * _blocks(seen))
        return {"bytes": cache + 8 * c["queries"] * c["heads"] * c["hd"], "flops": 4 * c["heads"] * c["hd"] * _pairs(c)}
    return {"bytes": 4 * c["rows"] * (c["vocab"] + c["recent"]), "flops": 8 * c["rows"] * (c["top_k"] or c["vocab"])}


# ---- the definitions in 64 bits ----

def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "rope":
        d, out = c["rd"], s["x"][:, :c["heads"] * c["hd"]].double().reshape(c["rows"], c["heads"], c["hd"]).clone()
        x = out.clone()
        for i in range(d // 2):
            f = c["base"] ** (-2.0 * i / d)
            g = 1.0
            if c["scaling"] == LINEAR:
                g = 0.0
            elif c["scaling"] == YARN:
                first, last = (d / 2 * math.log(c["orig"] / (2 * math.pi * t), c["base"]) for t in (c["high"], c["low"]))
                first, last = max(math.floor(first), 0), min(math.ceil(last), d - 1)
                g = 1 - min(1.0, max(0.0, (i - first) / max(last - first, 0.001)))
            elif c["scaling"] == BANDS:
                wave = 2 * math.pi / f
                g = min(1.0, max(0.0, (c["orig"] / wave - c["low"]) / (c["high"] - c["low"])))
            f *= g + (1 - g) / c["factor"]
            if s["factors"] is not None:
                f /= float(s["factors"][i])
            turn = torch.polar(torch.full((c["rows"],), _f32(c["magnitude"]), dtype=torch.float64, device=DEV),
                               s["at"].double() * f)
            a, b = (i, i + d // 2) if c["style"] else (2 * i, 2 * i + 1)
            z = torch.complex(x[:, :, a], x[:, :, b]) * turn[:, None]
            out[:, :, a], out[:, :, b] = z.real, z.imag
        return out.reshape(c["rows"], -1)
    if c["op"] == "store":
        got = []
        for part in (2, 3):
            codes, scales = (s["kc"], s["ks"]) if part == 2 else (s["vc"], s["vs"])
            rows = torch.zeros(c["position"] + c["rows"] - s["from"], c["kvh"], c["hd"], dtype=torch.float64, device=DEV)
            x = s["x"][:, part].double().reshape(c["rows"], c["kvh"], c["hd"])
            for b in range(s["from"], c["position"] + c["rows"], BLOCK):
                lo, hi = max(b, c["position"]), min(b + BLOCK, c["position"] + c["rows"])
                part_x = x[lo - c["position"]:hi - c["position"]]
                scale = (part_x.abs().amax(dim=(0, 2)) / 127).float()
                if lo > b:
                    was = scales[c["layer"], :, b // BLOCK]
                    scale = torch.maximum(scale, was)
                    kept = codes[c["layer"], :, b:lo] if part == 2 else codes[c["layer"], :, b // BLOCK, :, :lo - b].transpose(1, 2)
                    step = scale.double()[:, None, None]
                    rows[b - s["from"]:lo - s["from"]] = (torch.round(kept.double() * was.double()[:, None, None] / step) * step).transpose(0, 1)
                step = scale.double()[None, :, None]
                rows[lo - s["from"]:hi - s["from"]] = torch.round(part_x / step) * step
            got.append(rows.reshape(rows.shape[0], -1))
        return got
    if c["op"] == "attend":
        group, out = c["heads"] // c["kvh"], torch.zeros(c["queries"], c["heads"], c["hd"], dtype=torch.float64, device=DEV)
        q = s["q"].double().reshape(c["queries"], c["heads"], c["hd"])
        at = torch.arange(s["n"], device=DEV)
        for h in range(c["kvh"]):
            ks = s["ks"][c["layer"], h].double().repeat_interleave(BLOCK)[:s["n"]]
            vs = s["vs"][c["layer"], h].double().repeat_interleave(BLOCK)[:s["n"]]
            kt = s["kc"][c["layer"], h, :s["n"]].double().t().contiguous()
            v = s["vc"][c["layer"], h].double().permute(0, 2, 1).reshape(-1, c["hd"])[:s["n"]].contiguous()
            for j in range(h * group, (h + 1) * group):
                for lo in range(0, c["queries"], 512):
                    of = torch.arange(lo, min(lo + 512, c["queries"]), device=DEV)[:, None] + c["position"]
                    seen = (at <= of) & ((at > of - c["window"]) if c["window"] else (at >= 0))
                    z = (q[lo:lo + 512, j].contiguous() @ kt) * ks * _f32(c["hd"] ** -0.5)
                    z = torch.where(seen, z, torch.full_like(z, -math.inf))
                    e = torch.exp(z - z.max(dim=1, keepdim=True).values)
                    out[lo:lo + 512, j] = ((e * vs) @ v) / e.sum(dim=1, keepdim=True)
        return out.reshape(c["queries"], -1)
    return None  # tokens: whole numbers, held to be equal

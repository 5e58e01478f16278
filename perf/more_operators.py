"""The operators of a step that serves several sequences from one pool of pages, as measured cases: norms of the query
and key heads with the position rotation in the same pass, keys and values appended to a paged cache held in 4 bits,
the attention over it, and log probabilities of given tokens.

A program of this framework enqueues a step's operators in one open sequence of its context and waits once, at
the sequence's end; a pass here is one operator's share of that.  The device memory is the caller's (torch
tensors), seen through wrapped buffers, which `prepare` makes.

A batch: row_starts [sequences + 1] says which rows are whose, lengths [sequences] how many positions each sequence
has with these rows, which are its last ones; page_table [sequences][pages of a sequence] where its pages of 64
positions lie in the pool (-1 behind the last).

The cache's layout, bytes of one layer, G = head dim / 32:
  K codes  [page][kv head][position 64][g 4][t G][4]: dims 32 t + 8 g .. + 7, the lower half of a byte first
  V codes  [page][kv head][half 2][g 4][d 16][j 8][t G]: dims 32 t + d (lower half) and 32 t + 16 + d of position
           32 half + 8 g + j
  scales   [page][kv head][position 64][t G]: 2^(byte - 127)
A code is a sign and one of 0, .5, 1, 1.5, 2, 3, 4, 6; a scale the least power of two, from 2^-96 to 2^92, that is at
least a seventh of the largest of its 32 values.
"""
import math
import os
import random
import sys

import torch

own = False
DEV = "cuda"
PAGE = 64
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
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

def _turns(hd, rd, style, scaling, base, norm, offset):
    return dict(hd=hd, rd=rd, style=style, scaling=scaling, base=base, factor=8.0 if scaling else 1.0, orig=8192,
                low=1.0, high=4.0 if scaling == BANDS else 32.0, magnitude=1.0, norm=norm, offset=offset, eps=1e-6)


def _heads(name, rows, heads, kvh, first, spread, turns):
    return dict(name=name, op="heads", rows=rows, heads=heads, kvh=kvh, first=first, spread=spread, **turns)


def _append(name, sequences, rows, length, mix, heads, kvh, layer, turns):
    return dict(name=name, op="append", sequences=sequences, rows=rows, length=length, mix=mix, heads=heads, kvh=kvh,
                layer=layer, **turns)


def _attend(name, sequences, rows, length, mix, heads, kvh, hd, window, layer):
    return dict(name=name, op="attend", sequences=sequences, rows=rows, length=length, mix=mix, heads=heads, kvh=kvh,
                hd=hd, window=window, layer=layer)


def _logprobs(name, rows, vocab, top):
    return dict(name=name, op="logprobs", rows=rows, vocab=vocab, top=top)


def listed():
    normed = _turns(128, 128, 1, NONE, 1000000.0, True, 0.0)
    return [
        # a decoding step of one sequence: its query and key heads
        _heads("heads_step", 1, 32, 8, 5000, False, normed),
        # a prompt's query and key heads
        _heads("heads_prompt", 4095, 32, 8, 1000, False, normed),
        # a decoding step of 32 chats of different lengths
        _append("append_step", 32, 1, 8192, 5, 32, 8, 1, normed),
        # chunks of four prompts, keys as a model without norms has them, frequencies in bands
        _append("append_prompts", 4, 1500, 6000, 7, 32, 8, 0, _turns(128, 128, 0, BANDS, 500000.0, False, 0.0)),
        # one chat at 4k, and one at the end of a long context
        _attend("attend_4k", 1, 1, 4113, 0, 32, 8, 128, 0, 1),
        _attend("attend_128k", 1, 1, 131071, 0, 32, 8, 128, 0, 0),
        # a decoding step of 48 sequences of different lengths
        _attend("attend_batch", 48, 1, 16384, 3, 32, 8, 128, 0, 0),
        # verify passes of up to five tokens, small heads
        _attend("attend_verify", 7, 5, 2000, 4, 32, 4, 64, 0, 2),
        # the last chunk of a prompt
        _attend("attend_prompt", 1, 2048, 16384, 0, 32, 8, 128, 0, 0),
        # the token just drawn, with its alternatives
        _logprobs("logprobs_one", 1, 151936, 5),
        # the same for a batch
        _logprobs("logprobs_batch", 33, 128256, 20),
        # a prompt's own tokens, as for its perplexity
        _logprobs("logprobs_prompt", 511, 151936, 0),
    ]


def _log(rng, lo, hi):
    return min(hi, int(lo * math.exp(rng.random() * math.log((hi + 1) / lo))))


def draw(rng):
    op = rng.choice(["heads", "append", "attend", "attend", "logprobs"])
    hd = rng.choice([64, 96, 128, 256])
    kvh = _log(rng, 1, 8 * 128 // max(hd, 128))
    heads = kvh * rng.randint(1, 4)
    if op in ("heads", "append"):
        turns = _turns(hd, hd if rng.random() < 0.6 else 2 * rng.randint(1, hd // 2), rng.choice([0, 1]),
                       rng.choice([NONE, LINEAR, YARN, BANDS]), rng.choice([10000.0, 500000.0, 1000000.0]),
                       rng.random() < 0.6, rng.choice([0.0, 1.0]))
    if op == "heads":
        c = _heads("", _log(rng, 1, 4095), heads, kvh, _log(rng, 1, 1000000), rng.random() < 0.5, turns)
    elif op == "append":
        sequences = _log(rng, 1, 64)
        rows = 1 if rng.random() < 0.4 else _log(rng, 1, 4000 // sequences)
        c = _append("", sequences, rows, max(rows, _log(rng, 1, 8192)), rng.choice([0, rng.randint(1, 1 << 20)]), heads, kvh,
                    rng.choice([0, 1]), turns)
    elif op == "attend":
        sequences = _log(rng, 1, 64)
        length = _log(rng, 1, 120000 // sequences)
        if rng.random() < 0.7:  # single tokens and verify passes
            rows = rng.choice([1, 1, 1, rng.randint(2, 12)])
        else:
            sequences, length = min(sequences, 6), min(length, 14000)
            rows = _log(rng, 13, 1800 // sequences)
        c = _attend("", sequences, min(rows, length), length, rng.choice([0, rng.randint(1, 1 << 20)]), heads, kvh, hd,
                    rng.choice([0, 0, 0, _log(rng, 16, 4096)]), rng.choice([0, 1]))
    else:
        rows = _log(rng, 1, 400)
        c = _logprobs("", rows, _log(rng, 1000, 151936), rng.choice([0, 1, 5, 20, rng.randint(1, 64)]))
    del c["name"]
    return c


def _batch(c):
    """Each sequence's rows and length.  Mixed: the first has the case's own, the others have fewer rows, some none, and
    shorter contexts."""
    rng, rows, lengths = random.Random(c["mix"]), [c["rows"]], [c["length"]]
    for _ in range(1, c["sequences"]):
        r = rng.randint(1, c["rows"]) if c["mix"] else c["rows"]
        n = max(r, _log(rng, max(1, c["length"] // 16), c["length"])) if c["mix"] else c["length"]
        rows.append(0 if c["mix"] and rng.random() < 0.06 else r)
        lengths.append(n)
    return rows, lengths


def _pages(n):
    return -(-n // PAGE)


# ---- inputs ----

def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def _f32(x):
    return float(torch.tensor(x, dtype=torch.float32))


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _bytes(g, lo, hi, *shape):
    return torch.randint(lo, hi, shape, generator=g, device=DEV, dtype=torch.uint8)


def _paged(s, c, g):
    """The batch's tables, and a pool of pages with the cached positions in no order, as they come free."""
    rows, lengths = _batch(c)
    used = [_pages(n) for n in lengths]
    pool = sum(used) + 3
    free = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    table = torch.full((c["sequences"], max(used) + 1), -1, dtype=torch.int32, device=DEV)
    owner = torch.repeat_interleave(torch.arange(c["sequences"]), torch.tensor(used))
    first = torch.tensor([0] + used).cumsum(0)
    place = torch.arange(sum(used)) - first[owner]
    table[owner.to(DEV), place.to(DEV)] = free[:sum(used)]
    s["table"] = table
    s["starts"] = torch.tensor([0] + rows).cumsum(0).to(device=DEV, dtype=torch.int32)
    s["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=DEV)
    s["n"], s["longest"], s["pool"] = sum(rows), max(lengths), pool
    # each row's sequence and place in it
    s["owner"] = torch.repeat_interleave(torch.arange(c["sequences"]), torch.tensor(rows)).to(DEV)
    s["place"] = torch.arange(s["n"], device=DEV) - s["starts"][s["owner"]]
    each = (c["layer"] + 1, pool, c["kvh"], PAGE)
    s["kc"], s["vc"] = (_bytes(g, 0, 256, *each, c["hd"] // 2) for _ in range(2))
    s["ks"], s["vs"] = (_bytes(g, 125, 128, *each, c["hd"] // 32) for _ in range(2))  # values of .25 to 6


def _norms(s, c, g):
    s["q_norm"], s["k_norm"] = (1.0 - c["offset"] + 0.1 * _randn(g, c["hd"]) if c["norm"] else None for _ in range(2))


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = dict(case=c)
    if c["op"] == "heads":
        # rows as a fused projection leaves them: queries, keys, then values, which stay
        s["x"] = _randn(g, c["rows"], (c["heads"] + 2 * c["kvh"]) * c["hd"])
        s["y"] = torch.zeros(c["rows"], (c["heads"] + c["kvh"]) * c["hd"], device=DEV)
        at = torch.arange(c["rows"], device=DEV, dtype=torch.int32) + c["first"]
        s["at"] = at[torch.randperm(c["rows"], generator=g, device=DEV)].contiguous() if c["spread"] else at
        _norms(s, c, g)
    elif c["op"] == "append":
        _paged(s, c, g)
        s["x"] = _randn(g, s["n"], (c["heads"] + 2 * c["kvh"]) * c["hd"])
        s["x"][:, ::37] *= 4  # a few large channels, as keys have
        s["q"] = torch.zeros(s["n"], c["heads"] * c["hd"], device=DEV)
        s["k"], s["v"] = (torch.zeros(s["n"], c["kvh"] * c["hd"], device=DEV) for _ in range(2))
        _norms(s, c, g)
    elif c["op"] == "attend":
        _paged(s, c, g)
        s["q"] = 0.6 * _randn(g, s["n"], c["heads"] * c["hd"])
        s["y"] = torch.zeros_like(s["q"])
    else:
        # a model's logits: a broad body, and the few tokens that it is sure of
        s["x"] = 2.0 * _randn(g, c["rows"], c["vocab"])
        best = torch.randint(0, c["vocab"], (c["rows"], 24), generator=g, device=DEV)
        s["x"].scatter_(1, best, 6.0 + 4.0 * _randn(g, c["rows"], 24))
        any_one = torch.randint(0, c["vocab"], (c["rows"],), generator=g, device=DEV)
        likely = torch.rand(c["rows"], generator=g, device=DEV) < 0.7
        s["tokens"] = torch.where(likely, best[:, 0], any_one).to(torch.int32)
        s["y"], s["entropy"] = (torch.zeros(c["rows"], device=DEV) for _ in range(2))
        s["top"] = torch.zeros(c["rows"], c["top"], device=DEV) if c["top"] else None
        s["top_tokens"] = torch.zeros(c["rows"], c["top"], device=DEV, dtype=torch.int32) if c["top"] else None
    if own:
        hip, ctx = _own_context()
        s["ctx"] = ctx
        b = s["own"] = {k: ctx.wrap(v.data_ptr(), v.numel() * v.element_size())
                        for k, v in s.items() if isinstance(v, torch.Tensor)}
        if c["op"] in ("heads", "append"):
            rope = hip.RopeDesc(head_dim=c["hd"], rope_dim=c["rd"], style=c["style"], base=c["base"], scaling=c["scaling"],
                                factor=c["factor"], original_context=c["orig"], low=c["low"], high=c["high"],
                                magnitude=c["magnitude"])
            s["heads"] = hip.Heads(rope, q_norm=b.get("q_norm"), k_norm=b.get("k_norm"), eps=c["eps"],
                                   weight_offset=c["offset"])
        if c["op"] in ("append", "attend"):
            s["cache"] = hip.Kv4Cache(b["kc"], b["ks"], b["vc"], b["vs"], layers=c["layer"] + 1, heads_kv=c["kvh"],
                                      head_dim=c["hd"], pages=s["pool"])
            s["batch"] = hip.Batch(b["table"], b["starts"], b["lengths"], sequences=c["sequences"],
                                   pages_per_sequence=s["table"].shape[1], rows=s["n"], max_rows=c["rows"],
                                   max_length=s["longest"])
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


def _plain_heads(c, x, at, weights):
    """x [rows][heads][hd] normalised by `weights` (or not at all) and turned, in x's own type."""
    if weights is not None:
        mean = x.square().mean(dim=-1, keepdim=True)
        x = x * (weights + c["offset"]).to(x.dtype) / (mean + _f32(c["eps"])).sqrt()
    angle = torch.remainder(at.double()[:, None] * _frequencies(c), 2 * math.pi)
    cos, sin = ((m(angle) * _f32(c["magnitude"])).to(x.dtype)[:, None, :] for m in (torch.cos, torch.sin))
    y, half = x.clone(), c["rd"] // 2
    a, b = (slice(0, half), slice(half, c["rd"])) if c["style"] else (slice(0, c["rd"], 2), slice(1, c["rd"], 2))
    y[..., a] = x[..., a] * cos - x[..., b] * sin
    y[..., b] = x[..., a] * sin + x[..., b] * cos
    return y


def _fused_parts(c, x):
    n, qw, kw = x.shape[0], c["heads"] * c["hd"], c["kvh"] * c["hd"]
    return (x[:, :qw].reshape(n, c["heads"], -1), x[:, qw:qw + kw].reshape(n, c["kvh"], -1),
            x[:, qw + kw:].reshape(n, c["kvh"], -1))


def _run_plain_heads(s):
    c = s["case"]
    q, k, _ = _fused_parts(c, s["x"])
    y = [_plain_heads(c, x, s["at"], w) for x, w in ((q, s["q_norm"]), (k, s["k_norm"]))]
    return torch.cat(y, dim=1).reshape(c["rows"], -1)


def _in_four_bits(x):
    """(codes, scale bytes) of float32 rows, 32 values a scale."""
    x = x.reshape(*x.shape[:-1], -1, 32)
    part, power = torch.frexp(x.abs().amax(dim=-1, keepdim=True))  # largest = part * 2^power, part in [.5, 1)
    power = torch.where(part <= 0.875, power - 3, power - 2).clamp(-96, 92)
    power = torch.where(part > 0, power, torch.full_like(power, -96))
    a = torch.ldexp(x.double().abs(), -power)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (torch.round(a / step) * step).clamp(max=6)
    code = torch.bucketize(a, torch.tensor(VALUES, dtype=torch.float64, device=DEV))
    return torch.where(torch.signbit(x), code + 8, code).to(torch.uint8), (power + 127).to(torch.uint8).squeeze(-1)


def _plain_append(s):
    c = s["case"]
    q, k, v = _fused_parts(c, s["x"])
    at = (s["lengths"] - s["starts"].diff())[s["owner"]] + s["place"]
    q = _plain_heads(c, q, at, s["q_norm"])
    k = _plain_heads(c, k.double(), at, s["k_norm"]).float()  # next to a tie of the codes 32 bits would decide otherwise
    page = s["table"][s["owner"], at // PAGE].long()
    slot, g = at % PAGE, c["hd"] // 32
    codes, scales = _in_four_bits(k)  # [row][head][t][32]
    packed = codes[..., 0::2] | codes[..., 1::2] << 4  # [row][head][t][16]
    s["kc"][c["layer"]].reshape(-1, c["kvh"], PAGE, c["hd"] // 2)[page, :, slot] = (
        packed.reshape(*packed.shape[:2], g, 4, 4).transpose(2, 3).reshape(*packed.shape[:2], -1))
    s["ks"][c["layer"]][page, :, slot] = scales
    k = _of_four_bits(codes, scales)
    codes, scales = _in_four_bits(v)
    packed = (codes[..., :16] | codes[..., 16:] << 4).transpose(2, 3)  # [row][head][d][t]
    s["vc"][c["layer"]].reshape(-1, c["kvh"], 8, 16, 8, g)[page, :, slot // 8, :, slot % 8] = packed
    s["vs"][c["layer"]][page, :, slot] = scales
    return {"q": q.reshape(s["n"], -1), "k": k.reshape(s["n"], -1), "v": _of_four_bits(codes, scales).reshape(s["n"], -1)}


def _of_four_bits(codes, scales):
    values = torch.tensor(VALUES + tuple(-v for v in VALUES), device=DEV)
    return (values[codes.int()] * torch.ldexp(torch.ones((), device=DEV), scales.int() - 127)[..., None]).flatten(-2)


def _cached(s):
    """The sequences' keys and values, [sequence][kv head][position][dim] float32."""
    c, layer = s["case"], s["case"]["layer"]
    table = s["table"].clamp(min=0).long()
    count, pages = table.shape
    g = c["hd"] // 32

    def halves(codes):
        return torch.stack((codes & 15, codes >> 4), dim=-1)

    k = halves(s["kc"][layer][table].reshape(count, pages, c["kvh"], PAGE, 4, g, 4)).flatten(-2)  # .. position, g, t, 8
    k = k.transpose(-2, -3).reshape(count, pages, c["kvh"], PAGE, g, 32)
    v = halves(s["vc"][layer][table].reshape(count, pages, c["kvh"], 8, 16, 8, g))  # .. position / 8, d, position % 8, t, half
    v = v.permute(0, 1, 2, 3, 5, 6, 7, 4).reshape(count, pages, c["kvh"], PAGE, g, 32)
    return [_of_four_bits(x, y[layer][table]).transpose(1, 2).reshape(count, c["kvh"], pages * PAGE, c["hd"])[:, :, :s["longest"]]
            for x, y in ((k, s["ks"]), (v, s["vs"]))]


def _plain_attend(s):
    c = s["case"]
    count, most, group = c["sequences"], c["rows"], c["heads"] // c["kvh"]
    k, v = _cached(s)
    q = torch.zeros(count, most, c["heads"], c["hd"], device=DEV)
    q[s["owner"], s["place"]] = s["q"].reshape(s["n"], c["heads"], c["hd"])
    q = q.reshape(count, most, c["kvh"], group, c["hd"]).permute(0, 2, 3, 1, 4).reshape(count, c["kvh"], group * most, c["hd"])
    p = torch.matmul(q.contiguous(), k.transpose(2, 3).contiguous()).mul_(_f32(c["hd"] ** -0.5))
    p = p.reshape(count, c["kvh"], group, most, -1)
    at = torch.arange(s["longest"], device=DEV)
    of = (s["lengths"] - s["starts"].diff())[:, None, None] + torch.arange(most, device=DEV)[:, None]
    hidden = at > of
    if c["window"]:
        hidden = hidden | (at <= of - c["window"])
    p.masked_fill_(hidden[:, None, None], -math.inf)
    p = p.sub_(p.amax(dim=-1, keepdim=True)).exp_()
    total = p.sum(dim=-1, keepdim=True)
    o = torch.matmul(p.reshape(count, c["kvh"], group * most, -1), v).reshape(count, c["kvh"], group, most, -1) / total
    return o.permute(0, 3, 1, 2, 4)[s["owner"], s["place"]].reshape(s["n"], -1)


def _plain_logprobs(s):
    c, x = s["case"], s["x"]
    d = x - x.amax(dim=1, keepdim=True)
    e = torch.exp(d).double()
    total = e.sum(dim=1, keepdim=True)
    log = d.double() - total.log()
    out = {"logprob": log.gather(1, s["tokens"].long()[:, None])[:, 0].float(),
           "entropy": (total.log()[:, 0] - (e * d).sum(dim=1) / total[:, 0]).float()}
    if c["top"]:
        by = torch.argsort(x, dim=1, descending=True, stable=True)[:, :c["top"]]
        out["top_tokens"], out["top"] = by.to(torch.int32), log.gather(1, by).float()
    return out


# ---- one pass ----

def run(state):
    s, c = state, state["case"]
    if own:
        ctx, b = s["ctx"], s["own"]
        if c["op"] == "heads":
            ctx.norm_rope_rows(s["heads"], b["x"], b["y"], c["rows"], c["heads"], c["kvh"], positions=b["at"],
                               src_stride=(c["heads"] + 2 * c["kvh"]) * c["hd"])
            return s["y"]
        if c["op"] == "append":
            at = 4 * c["heads"] * c["hd"]
            ctx.kv4_append(s["cache"], c["layer"], s["batch"], s["heads"], b["x"], k_off=at, v_off=at + 4 * c["kvh"] * c["hd"],
                           row_stride=(c["heads"] + 2 * c["kvh"]) * c["hd"], q_heads=c["heads"], q_out=b["q"])
            ctx.kv4_load(s["cache"], c["layer"], s["batch"], b["k"], b["v"])
            return {"q": s["q"], "k": s["k"], "v": s["v"]}
        if c["op"] == "attend":
            ctx.kv4_attention(s["cache"], c["layer"], s["batch"], b["q"], b["y"], c["heads"], window=c["window"])
            return s["y"]
        ctx.token_logprobs(b["x"], b["tokens"], b["y"], c["rows"], c["vocab"], entropy=b["entropy"], top=c["top"],
                           top_tokens=b.get("top_tokens"), top_logprobs=b.get("top"))
        out = {"logprob": s["y"], "entropy": s["entropy"]}
        return {**out, "top_tokens": s["top_tokens"], "top": s["top"]} if c["top"] else out
    return {"heads": _run_plain_heads, "append": _plain_append, "attend": _plain_attend, "logprobs": _plain_logprobs}[c["op"]](s)


def work(case):
    c = case
    if c["op"] == "heads":
        n = c["rows"] * (c["heads"] + c["kvh"]) * c["hd"]
        return {"bytes": 8 * n + 4 * c["rows"], "flops": (3 + 4 * c["norm"]) * n}
    if c["op"] == "logprobs":
        n = c["rows"] * c["vocab"]
        return {"bytes": 4 * n + c["rows"] * (12 + 8 * c["top"]), "flops": 5 * n}
    rows, lengths = _batch(c)
    if c["op"] == "append":  # rows in, queries and codes out, and the read-back: codes in and rows out
        q, kv = sum(rows) * c["heads"] * c["hd"], 2 * sum(rows) * c["kvh"] * c["hd"]
        return {"bytes": 8 * q + (4 + 17 / 32 + 17 / 32 + 4) * kv, "flops": (3 + 4 * c["norm"]) * (q + kv // 2) + 4 * kv}
    read = pairs = 0
    for r, n in zip(rows, lengths):
        w = c["window"] or n
        read += min(n, w + r - 1) if r else 0
        seen = min(r, max(0, w - (n - r)))  # rows that see all before them
        pairs += seen * (n - r) + seen * (seen + 1) // 2 + (r - seen) * w
    kv = 2 * read * c["kvh"] * c["hd"]
    return {"bytes": kv * 17 / 32 + 8 * sum(rows) * c["heads"] * c["hd"], "flops": 4 * c["heads"] * c["hd"] * pairs}


# ---- the definitions in 64 bits ----

def _exact_heads(c, x, at, weights):
    x = x.double()
    if weights is not None:
        w = weights.double() + c["offset"]
        x = x * w * torch.rsqrt((x * x).sum(dim=-1, keepdim=True) / c["hd"] + _f32(c["eps"]))
    d, out = c["rd"], x.clone()
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
        turn = torch.polar(torch.full((at.numel(),), _f32(c["magnitude"]), dtype=torch.float64, device=DEV), at.double() * f)
        a, b = (i, i + d // 2) if c["style"] else (2 * i, 2 * i + 1)
        z = torch.complex(x[:, :, a], x[:, :, b]) * turn[:, None]
        out[:, :, a], out[:, :, b] = z.real, z.imag
    return out


def _exact_four_bits(x):
    """Each value of 32 that share a scale as the nearest one that 4 bits hold."""
    x = x.float().double().reshape(*x.shape[:-1], -1, 32)
    scale = torch.exp2(torch.ceil(torch.log2(x.abs().amax(dim=-1, keepdim=True).clamp(min=2.0 ** -126) / 7)).clamp(-96, 92))
    near, best = torch.full_like(x, math.inf), torch.zeros_like(x)
    for code in (0, 2, 4, 6, 1, 3, 5, 7):  # even ones first: they win ties
        off = (x.abs() - VALUES[code] * scale).abs()
        best = torch.where(off < near, VALUES[code] * scale, best)
        near = torch.minimum(off, near)
    return (best * torch.where(x < 0, -1.0, 1.0)).flatten(-2)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["op"] == "heads":
        q, k, _ = _fused_parts(c, s["x"])
        return torch.cat([_exact_heads(c, x, s["at"], w) for x, w in ((q, s["q_norm"]), (k, s["k_norm"]))], dim=1).flatten(1)
    if c["op"] == "logprobs":
        y, h, top, at = [], [], [], []
        for r in range(c["rows"]):
            x = s["x"][r].double()
            log = x - torch.logsumexp(x, 0)
            y.append(log[s["tokens"][r].long()])
            h.append(-(log.exp() * log).sum())
            if c["top"]:
                best = torch.sort(x, descending=True, stable=True).indices[:c["top"]]
                at.append(best.to(torch.int32))
                top.append(log[best])
        out = {"logprob": torch.stack(y), "entropy": torch.stack(h)}
        return {**out, "top_tokens": torch.stack(at), "top": torch.stack(top)} if c["top"] else out
    rows, lengths = _batch(c)
    if c["op"] == "append":
        at = torch.tensor([n - r + i for r, n in zip(rows, lengths) for i in range(r)], device=DEV)
        q, k, v = _fused_parts(c, s["x"])
        return {"q": _exact_heads(c, q, at, s["q_norm"]).flatten(1),
                "k": _exact_four_bits(_exact_heads(c, k, at, s["k_norm"])).flatten(1), "v": _exact_four_bits(v).flatten(1)}
    group, g, row = c["heads"] // c["kvh"], c["hd"] // 32, 0
    out = torch.zeros(s["n"], c["heads"], c["hd"], dtype=torch.float64, device=DEV)
    values = torch.tensor(VALUES + tuple(-v for v in VALUES), dtype=torch.float64, device=DEV)
    q = s["q"].double().reshape(s["n"], c["heads"], c["hd"])
    dim = torch.arange(c["hd"], device=DEV)
    k_byte, k_high = dim % 32 // 8 * 4 * g + dim // 32 * 4 + dim % 8 // 2, dim % 2
    v_byte, v_high = dim % 16 * 8 * g + dim // 32, dim % 32 // 16
    for i, (r, n) in enumerate(zip(rows, lengths)):
        at = torch.arange(n, device=DEV)
        page, slot = s["table"][i].long()[at // PAGE], at % PAGE
        for h in range(c["kvh"] if r else 0):
            kb = s["kc"][c["layer"], page, h, slot][:, k_byte].int()
            vb = s["vc"][c["layer"], :, h].reshape(s["pool"], -1)
            vb = vb[page[:, None], (slot // 8 * (128 * g) + slot % 8 * g)[:, None] + v_byte].int()
            ks, vs = (torch.exp2(x[c["layer"], page, h, slot].double() - 127).repeat_interleave(32, dim=1) for x in (s["ks"], s["vs"]))
            kt = (values[torch.where(k_high > 0, kb >> 4, kb & 15)] * ks).t().contiguous()
            v = values[torch.where(v_high > 0, vb >> 4, vb & 15)] * vs
            for j in range(h * group, (h + 1) * group):
                for lo in range(0, r, 512):
                    of = torch.arange(lo, min(lo + 512, r), device=DEV)[:, None] + n - r
                    seen = (at <= of) & ((at > of - c["window"]) if c["window"] else (at >= 0))
                    z = q[row + lo:row + min(lo + 512, r), j].contiguous() @ kt * _f32(c["hd"] ** -0.5)
                    z = torch.where(seen, z, torch.full_like(z, -math.inf))
                    e = torch.exp(z - z.max(dim=1, keepdim=True).values)
                    out[row + lo:row + min(lo + 512, r), j] = (e @ v) / e.sum(dim=1, keepdim=True)
        row += r
    return out.reshape(s["n"], -1)

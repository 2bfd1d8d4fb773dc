"""Softmax attention over a paged cache and what feeds it, as timed cases.

  rotary  the rotation of heads by their positions: both layouts, whole heads or a part of them,
          frequencies stretched for long contexts
  append  the new keys and values of a batch of sequences written into the pages of a cache, the
          keys, and the queries beside them, rotated on the way
  attn    attention of the new rows over the pages: prompts, chunks behind a long past, single
          tokens, and batches that mix them

The plain forms below are torch products, sums and exponentials. With `own` set, the same inputs go
through the package's binding of the C ABI on one asynchronous context, as a serving loop does.
"""
from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import torch

own = False

DEV = torch.device("cuda", 0)
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16}

# Heads of width 128, as the layers have them whose projections the package holds; a few key heads
# for many query heads. Pages of 64 tokens.
QUERY_HEADS, KEY_HEADS, WIDTH, PAGE = 16, 2, 128, 64
ORIGINAL, FACTOR = 32768, 8.0  # the context that stretched frequencies come from, and by how much


def _rotary(name, tokens, heads=QUERY_HEADS, width=WIDTH, dims=WIDTH, pairs=False, scaled=False,
            first=0):
    c = {"kind": "rotary", "tokens": tokens, "heads": heads, "width": width, "dims": dims,
         "pairs": pairs, "scaled": scaled, "first": first}
    return {"name": name, **c} if name else c


def _append(name, tokens, seqs, past, step=False, hq=QUERY_HEADS, hk=KEY_HEADS, width=WIDTH,
            page=PAGE, type="f16", dims=WIDTH, pairs=False, layout=0):
    c = {"kind": "append", "tokens": tokens, "seqs": seqs, "past": past, "step": step, "hq": hq,
         "hk": hk, "width": width, "page": page, "type": type, "dims": dims, "pairs": pairs,
         "scaled": False, "layout": layout}
    return {"name": name, **c} if name else c


def _attn(name, tokens, seqs, past, step=False, hq=QUERY_HEADS, hk=KEY_HEADS, width=WIDTH,
          page=PAGE, type="f16", window=0, sinks=False, gate=False, causal=True, layout=0):
    c = {"kind": "attn", "tokens": tokens, "seqs": seqs, "past": past, "step": step, "hq": hq,
         "hk": hk, "width": width, "page": page, "type": type, "window": window, "sinks": sinks,
         "gate": gate, "causal": causal, "layout": layout}
    return {"name": name, **c} if name else c


def listed():
    return [
        # the query heads of one token
        _rotary("rotary_1", 1, first=1023),
        # a long document's rows, a part of each head, frequencies stretched for its length
        _rotary("rotary_part_8191", 8191, heads=24, dims=64, pairs=True, scaled=True,
                first=1 << 18),
        # one sequence decoding: its key, value and query
        _append("append_step_1", 1, 1, 8191, step=True),
        # 61 sequences decoding together
        _append("append_step_61", 61, 61, 16384, step=True, layout=3),
        # a batch of prompts, some of which go on from what the cache holds
        _append("append_prompt_4099", 4099, 7, 2048, hq=32, hk=8, layout=5),
        # one sequence decoding, a short context
        _attn("attn_step_1", 1, 1, 512, step=True),
        # and the longest one: all of the device reads one sequence's pages
        _attn("attn_step_1_long", 1, 1, 130001, step=True),
        # 61 sequences decoding, contexts of 500 to 32,000 tokens
        _attn("attn_step_61", 61, 61, 32000, step=True, layout=11),
        # a prompt of 8192 tokens, nothing before it
        _attn("attn_prompt_8192", 8192, 1, 0),
        # a chunk of a very long prompt over all that came before
        _attn("attn_chunk_509_past_65000", 509, 1, 65000),
        # prompts and decoding sequences in one call: a window of 1024, a logit for each head that
        # takes weight from the rest, outputs gated; small pages of bf16
        _attn("attn_ragged_2003", 2003, 19, 3500, hq=24, hk=8, width=64, page=16, type="bf16",
              window=1024, sinks=True, gate=True, layout=7),
        # wide heads in bf16, a prompt behind a cached beginning
        _attn("attn_wide_2049", 2049, 1, 1000, hq=16, hk=4, width=256, type="bf16", gate=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choice(("attn", "attn", "attn", "append", "rotary"))
    layout = rng.randint(1, 1 << 20)
    if kind == "rotary":
        width = rng.choice((64, 80, 96, 128, 256))
        return _rotary("", _log_int(rng, 1, 8191), rng.randint(1, 24), width,
                       rng.choice((width, width, width // 2, width // 2 - 6)),
                       rng.random() < 0.5, rng.random() < 0.5,
                       rng.choice((0, 0, 1000, 1 << 18, 1 << 20)))
    hk, per = rng.choice((1, 2, 3, 4, 8)), rng.choice((1, 2, 3, 4, 6, 8))
    more = {"hq": hk * per, "hk": hk, "page": rng.choice((16, 32, 64, 128, 256)),
            "type": rng.choice(("f16", "bf16")), "layout": layout}
    step = rng.random() < 0.5
    if kind == "append":
        width = rng.choice((64, 128, 256))
        tokens = _log_int(rng, 1, 256) if step else _log_int(rng, 2, 2500)
        return _append("", tokens, tokens if step else _log_int(rng, 1, min(16, tokens)),
                       _log_int(rng, 64, 16384 if tokens < 32 else 2048), step, width=width,
                       dims=rng.choice((width, width // 2)), pairs=rng.random() < 0.5, **more)
    more |= {"width": rng.choice((64, 128, 128, 256)), "sinks": rng.random() < 0.25,
             "gate": rng.random() < 0.25, "causal": rng.random() < 0.85}
    if rng.random() < 0.25:
        more["window"] = _log_int(rng, 16, 2048)
    if step:
        seqs = _log_int(rng, 1, 64)
        return _attn("", seqs, seqs, _log_int(rng, 1, min(131072, 1 << 20 // seqs.bit_length())),
                     True, **more)
    if rng.random() < 0.5:
        return _attn("", _log_int(rng, 2, 2048), 1, _log_int(rng, 1, 16384), **more)
    tokens = _log_int(rng, 32, 1500)
    return _attn("", tokens, _log_int(rng, 2, 16), _log_int(rng, 1, 4000), **more)


# ------------------------------------------------------------------ inputs


def _lengths(case):
    """The sequences' new rows and what the cache holds of them before: about a third of a mixed
    batch are single tokens; a decoding sequence has a past, a prompt less often."""
    n, s, past = case["tokens"], case["seqs"], case["past"]
    if s == 1:
        return [n], [past]
    r = random.Random(case["layout"])
    if case["step"]:
        pasts = [max(1, round(past * (1 / 64) ** r.random())) for _ in range(s)]
        pasts[r.randrange(s)] = past
        return [1] * s, pasts
    rest = n - s  # one token at least for each
    share = [0.0 if r.random() < 0.33 else r.random() + 0.2 for _ in range(s)]
    share[r.randrange(s)] += 0.5
    total = sum(share)
    more = [int(rest * x / total) for x in share]
    more[max(range(s), key=lambda i: share[i])] += rest - sum(more)
    rows = [1 + m for m in more]
    return rows, [r.randrange(past + 1) if m == 1 or r.random() < 0.4 else 0 for m in rows]


def _frequencies(case):
    """Radians a position for each rotated pair, in 64 bits: powers of a base, and for a context
    FACTOR times the original one the slow ones divided by that factor, those that turn more than
    32 times in the original context kept, a straight line between. Returns them with the factor
    of cos and sin that goes with it."""
    dims = case["dims"]
    f = 1.0e6 ** (-torch.arange(0, dims, 2, dtype=torch.float64) / dims)
    if not case["scaled"]:
        return f.to(DEV), 1.0
    at = lambda turns: (dims * math.log(ORIGINAL / (turns * 2 * math.pi)) /  # noqa: E731
                        (2 * math.log(1.0e6)))
    low, high = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), dims - 1)
    i = torch.arange(dims // 2, dtype=torch.float64)
    slow = torch.clamp((i - low) / max(high - low, 0.001), 0.0, 1.0)
    return (f * (1 - slow) + f / FACTOR * slow).to(DEV), 0.1 * math.log(FACTOR) + 1.0


def _inputs(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    s, n = {}, case["tokens"]
    if case["kind"] != "attn":
        s["frequencies"], s["magnitude"] = _frequencies(case)
    if case["kind"] == "rotary":
        s["positions"] = torch.arange(case["first"], case["first"] + n, dtype=torch.int32,
                                      device=DEV)
        s["x"] = normal(n, case["heads"] * case["width"])
        return s
    hq, hk, width, page = case["hq"], case["hk"], case["width"], case["page"]
    rows, past = _lengths(case)
    seqs = len(rows)
    slots_all = seqs + seqs // 4
    slots = torch.randperm(slots_all, generator=g, device=DEV)[:seqs]
    s["rows"], s["past"] = rows, past
    s["slots"] = slots.to(torch.int32)
    begin = torch.cumsum(torch.tensor([0] + rows), 0)
    s["offsets"] = begin.to(torch.int32).to(DEV)
    # pages in the order in which a pool that has been in use hands them out
    held = torch.tensor([-(-(a + b) // page) for a, b in zip(past, rows)])
    pages = int(held.sum()) + 3
    width_pages = int(held.max()) + 1
    order = torch.randperm(pages, generator=g, device=DEV)
    lines = torch.arange(width_pages)[None, :]
    first = (torch.cumsum(held, 0) - held)[:, None]
    mine = (lines < held[:, None]).to(DEV)
    table = torch.full((slots_all, width_pages), -1, dtype=torch.int32, device=DEV)
    table[slots] = torch.where(mine, order[torch.clamp(first + lines, max=pages - 1).to(DEV)],
                               -1).to(torch.int32)
    lengths = torch.zeros(slots_all, dtype=torch.int32, device=DEV)
    lengths[slots] = torch.tensor(past, dtype=torch.int32, device=DEV)
    s["table"], s["lengths"] = table, lengths
    # what the pool holds behind a sequence's end is of others before it
    pool = lambda: normal(pages, hk, page, width).to(TYPES[case["type"]])  # noqa: E731
    s["keys"], s["values"] = pool(), pool()
    s["q"] = normal(n, hq * width)
    if case["kind"] == "append":
        s["kv"] = normal(n, 2 * hk * width)  # one projection's rows: the keys, then the values
        return s
    if case["sinks"]:
        s["sinks"] = normal(hq)
    if case["gate"]:
        s["gate"] = normal(n, hq * width)
    return s


def prepare(case, seed):
    """The inputs, and the buffers that a serving loop keeps for the results."""
    s = {"case": case, **_inputs(case, seed)}
    if case["kind"] == "rotary":
        s["y"] = torch.zeros_like(s["x"])
    else:
        rows = torch.tensor(s["rows"], device=DEV)
        # for the plain forms: the sequence, the place and the position of each row
        s["seq_of"] = torch.repeat_interleave(torch.arange(len(s["rows"]), device=DEV), rows)
        s["place"] = torch.arange(case["tokens"], device=DEV) - s["offsets"].long()[s["seq_of"]]
        s["position"] = torch.tensor(s["past"], device=DEV)[s["seq_of"]] + s["place"]
        s["most_rows"] = max(s["rows"])
        s["most_keys"] = max(a + b for a, b in zip(s["rows"], s["past"]))
        s["y"] = torch.zeros_like(s["q"])
    torch.cuda.synchronize()  # the library's stream is not torch's
    return s


# ------------------------------------------------------- the package's calls

_context = None


def _ctx():
    global _context
    if _context is None:
        root = str(Path(__file__).resolve().parents[1] / "kestrel-q_amd")
        if root not in sys.path:
            sys.path.insert(0, root)
        import kq_hip
        _context = kq_hip.Context(0)
        _context.set_async(True)
    return _context


def _own_plan(s):
    """The descriptions of the call that a program makes once and keeps."""
    ctx = _ctx()
    import kq_hip
    case = s["case"]
    p = {"ctx": ctx}
    ptr = lambda k: s[k].data_ptr() if k in s else None  # noqa: E731
    if case["kind"] != "attn":
        p["rotary"] = kq_hip.rotary(case["dims"], ptr("frequencies"),
                                    layout="pairs" if case["pairs"] else "halves",
                                    magnitude=s["magnitude"])
    if case["kind"] == "rotary":
        return p
    hq, hk, width = case["hq"], case["hk"], case["width"]
    p["seqs"] = kq_hip.sequences(case["tokens"], len(s["rows"]), s["lengths"].numel(),
                                 None if case["step"] else ptr("offsets"), ptr("slots"))
    type_id = kq_hip.TYPE_F16 if case["type"] == "f16" else kq_hip.TYPE_BF16
    p["cache"] = kq_hip.paged_cache(type_id, hk, width, case["page"], s["keys"].shape[0],
                                    s["table"].shape[1], ptr("keys"), ptr("values"), ptr("table"),
                                    ptr("lengths"))
    if case["kind"] == "append":
        kv, row = ptr("kv"), 2 * hk * width
        p["in"] = kq_hip.cache_rows(kv, row, kv + 4 * hk * width, row, hq, ptr("q"), hq * width,
                                    ptr("y"), hq * width)
        return p
    p["attn"] = kq_hip.paged_attention(hq, width ** -0.5, causal=case["causal"],
                                       window=case["window"], sinks=ptr("sinks"),
                                       gate="sigmoid" if case["gate"] else "none")
    p["bytes"] = kq_hip.paged_attention_scratch_bytes(p["attn"], p["cache"], p["seqs"])
    p["scratch"] = torch.empty(max(p["bytes"], 1), dtype=torch.uint8, device=DEV)
    torch.cuda.synchronize()
    return p


def _run_own(s):
    p = s.get("own")
    if p is None:
        p = s["own"] = _own_plan(s)
    case, ctx = s["case"], p["ctx"]
    ptr = lambda k: s[k].data_ptr() if k in s else None  # noqa: E731
    if case["kind"] == "rotary":
        w = case["heads"] * case["width"]
        ctx.rotary(p["rotary"], case["heads"], case["width"], case["tokens"], ptr("positions"),
                   ptr("x"), w, ptr("y"), w)
        return s["y"]
    w = case["hq"] * case["width"]
    if case["kind"] == "append":
        ctx.cache_append(p["cache"], p["seqs"], p["in"], p["rotary"])
        return {"q": s["y"], "keys": s["keys"], "values": s["values"]}
    ctx.paged_attention(p["attn"], p["cache"], p["seqs"], ptr("q"), w, ptr("gate"), w, ptr("y"), w,
                        p["scratch"].data_ptr(), p["bytes"])
    return s["y"]


# ------------------------------------------------------------- plain forms


def _turn(x, positions, frequencies, magnitude, pairs):
    """x [rows][heads][width]; the angles are formed in 64 bits."""
    angle = positions.double()[:, None] * frequencies
    cos = (torch.cos(angle) * magnitude).float()[:, None, :]
    sin = (torch.sin(angle) * magnitude).float()[:, None, :]
    half = frequencies.numel()
    y = x.clone()
    if pairs:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
        y[..., 0:2 * half:2] = a * cos - b * sin
        y[..., 1:2 * half:2] = a * sin + b * cos
    else:
        a, b = x[..., :half], x[..., half:2 * half]
        y[..., :half] = a * cos - b * sin
        y[..., half:2 * half] = a * sin + b * cos
    return y


def _rotary_plain(s):
    case = s["case"]
    x = s["x"].view(case["tokens"], case["heads"], case["width"])
    return _turn(x, s["positions"], s["frequencies"], s["magnitude"],
                 case["pairs"]).view_as(s["x"])


def _append_plain(s):
    case = s["case"]
    n, hk, width, page = case["tokens"], case["hk"], case["width"], case["page"]
    k, v = s["kv"].view(n, 2, hk, width).unbind(1)
    turn = lambda x: _turn(x, s["position"], s["frequencies"], s["magnitude"],  # noqa: E731
                           case["pairs"])
    where = s["table"][s["slots"].long()[s["seq_of"]], s["position"] // page].long()
    off = s["position"] % page
    s["keys"][where, :, off] = turn(k).to(s["keys"].dtype)
    s["values"][where, :, off] = v.to(s["values"].dtype)
    return {"q": turn(s["q"].view(n, -1, width)).view_as(s["q"]), "keys": s["keys"],
            "values": s["values"]}


def _attn_plain(s):
    """Every sequence padded to the longest: its keys and values gathered out of the pages, one
    product for the scores, the softmax, one product for the outputs."""
    case = s["case"]
    n, hq, hk, width, page = case["tokens"], case["hq"], case["hk"], case["width"], case["page"]
    per, most, keys = hq // hk, s["most_rows"], s["most_keys"]
    at = torch.arange(keys, device=DEV)
    where = torch.clamp(s["table"][s["slots"].long()][:, at // page], min=0).long()
    k = s["keys"][where, :, at % page].float()           # [sequences][keys][heads][width]
    v = s["values"][where, :, at % page].float()
    k = k.permute(0, 2, 3, 1).contiguous()
    v = v.permute(0, 2, 1, 3).contiguous()
    begin, end = s["offsets"][:-1].long(), s["offsets"][1:].long()
    place = torch.arange(most, device=DEV)
    row = torch.clamp(begin[:, None] + place, max=n - 1)  # [sequences][rows]
    q = s["q"].view(n, hk, per, width)[row].permute(0, 2, 3, 1, 4)
    q = (q * width ** -0.5).reshape(len(s["rows"]), hk, per * most, width)
    score = (q @ k).view(len(s["rows"]), hk, per, most, keys)
    past = s["lengths"].long()[s["slots"].long()]
    position = past[:, None] + place
    last = position if case["causal"] else (past + end - begin - 1)[:, None].expand_as(position)
    seen = at <= last[:, :, None]
    if case["window"]:
        seen = seen & (at > position[:, :, None] - case["window"])
    score = torch.where(seen[:, None, None], score, -math.inf)
    top = score.amax(-1, keepdim=True)
    if case["sinks"]:
        sink = s["sinks"].view(1, hk, per, 1, 1)
        top = torch.maximum(top, sink)
    top = torch.clamp(top, min=-1.0e30)  # places behind a sequence's rows may see nothing
    p = torch.exp(score - top)
    total = p.sum(-1, keepdim=True)
    if case["sinks"]:
        total = total + torch.exp(sink - top)
    y = (p.view(len(s["rows"]), hk, per * most, keys) @ v).view(*p.shape[:-1], width) / total
    y = y.permute(0, 3, 1, 2, 4)[s["seq_of"], s["place"]].reshape(n, hq * width)
    return y * torch.sigmoid(s["gate"]) if case["gate"] else y


def run(s):
    if own:
        return _run_own(s)
    return {"rotary": _rotary_plain, "append": _append_plain, "attn": _attn_plain}[
        s["case"]["kind"]](s)


# ------------------------------------------------------------ what it costs


def work(case):
    n = case["tokens"]
    if case["kind"] == "rotary":
        w, turned = case["heads"] * case["width"], case["heads"] * case["dims"]
        return {"bytes": 4 * (2 * n * w + n) + 4 * case["dims"], "flops": 3 * n * turned}
    hq, hk, width = case["hq"], case["hk"], case["width"]
    if case["kind"] == "append":
        return {"bytes": n * width * (4 * (2 * hq + 2 * hk) + 2 * 2 * hk) + 4 * case["dims"],
                "flops": 3 * n * (hq + hk) * case["dims"]}
    held = scores = 0
    for m, past in zip(*_lengths(case)):
        window = case["window"] or past + m
        held += past + m - max(0, past + 1 - window)
        if not case["causal"]:
            scores += sum(past + m - max(0, past + j + 1 - window) for j in range(m))
        else:
            scores += sum(min(past + j + 1, window) for j in range(m))
    return {"bytes": 4 * n * hq * width * (2 + case["gate"]) + 2 * 2 * held * hk * width,
            "flops": 4 * scores * hq * width}


# ---------------------------------------------- the definitions in 64 bits


def _exact_turn(x, positions, frequencies, magnitude, pairs):
    """Each pair as a complex number, times e^(i position frequency)."""
    half = frequencies.numel()
    head, rest = x[..., :2 * half], x[..., 2 * half:]
    z = (torch.view_as_complex(head.unflatten(-1, (half, 2)).contiguous()) if pairs
         else torch.complex(head[..., :half].contiguous(), head[..., half:].contiguous()))
    angle = positions.double()[:, None, None] * frequencies
    z = z * torch.polar(torch.full_like(angle, magnitude), angle)
    head = (torch.view_as_real(z).flatten(-2) if pairs else torch.cat((z.real, z.imag), -1))
    return torch.cat((head, rest), -1)


def _exact_attn(case, t):
    """One sequence and one key head after the other."""
    n, hq, hk, width, page = case["tokens"], case["hq"], case["hk"], case["width"], case["page"]
    per = hq // hk
    y = torch.zeros(n, hk, per, width, dtype=torch.float64, device=DEV)
    q = t["q"].double().view(n, hk, per, width)
    a = 0
    for slot, m, past in zip(t["slots"].tolist(), t["rows"], t["past"]):
        pages = t["table"][slot][:-(-(past + m) // page)].long()
        at = torch.arange(past + m, device=DEV)
        mine = torch.arange(past, past + m, device=DEV)[:, None]
        hidden = at > (mine if case["causal"] else mine * 0 + past + m)
        if case["window"]:
            hidden = hidden | (at <= mine - case["window"])
        for h in range(hk):
            k = t["keys"][pages, h].reshape(-1, width)[:past + m].double()
            v = t["values"][pages, h].reshape(-1, width)[:past + m].double()
            e = (q[a:a + m, h].reshape(m * per, width) @ k.T.contiguous()).view(m, per, past + m)
            e /= math.sqrt(width)
            e.masked_fill_(hidden[:, None], -math.inf)
            if case["sinks"]:
                sink = t["sinks"].double().view(hk, per)[h].expand(m, per)[..., None]
                e = torch.cat((e, sink), -1)
            w = torch.softmax(e, -1)[..., :past + m].reshape(m * per, past + m)
            y[a:a + m, h] = (w @ v).view(m, per, width)
        a += m
    y = y.view(n, hq * width)
    return y / (1 + torch.exp(-t["gate"].double())) if case["gate"] else y


def exact(case, seed):
    t = _inputs(case, seed)
    if case["kind"] == "attn":
        return _exact_attn(case, t)
    turn = lambda x, at: _exact_turn(x.double(), at, t["frequencies"],  # noqa: E731
                                     t["magnitude"], case["pairs"])
    if case["kind"] == "rotary":
        x = t["x"].view(case["tokens"], case["heads"], case["width"])
        return turn(x, t["positions"]).view_as(t["x"])
    n, hk, width, page = case["tokens"], case["hk"], case["width"], case["page"]
    keys, values = t["keys"].double(), t["values"].double()
    kv = t["kv"].view(n, 2, hk, width)
    q = torch.zeros(n, case["hq"], width, dtype=torch.float64, device=DEV)
    a = 0
    for slot, m, past in zip(t["slots"].tolist(), t["rows"], t["past"]):
        at = torch.arange(past, past + m, device=DEV)
        pages = t["table"][slot].long()[at // page]
        keys[pages, :, at % page] = turn(kv[a:a + m, 0], at)
        values[pages, :, at % page] = kv[a:a + m, 1].double()
        q[a:a + m] = turn(t["q"][a:a + m].view(m, -1, width), at)
        a += m
    return {"q": q.view(n, -1), "keys": keys, "values": values}

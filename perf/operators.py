"""The operators between a GDN layer's projections and its residual, as timed cases.

  conv    the causal depthwise convolution over the projected q, k, v channels, with its SiLU
          and its state of the last taps - 1 inputs
  attn    linear attention with a decay for each head, with the delta correction or without:
          prompts, batches of sequences of different lengths, and single tokens
  norm    the RMS norm of each head, times its weight and its gate
  join    the end of a block: norm and gate of its output, its addition to the residual branches,
          and the norm of the branches before the next block

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
CHUNK = 64      # tokens that the plain form of the attention takes at a time
EPS = 1.0e-6

# The layer whose projections the package holds: 16 key heads and 48 value heads of width 128, a
# convolution of 4 taps over q, k and v (10240 channels), 4 residual branches of 2560.
KEY_HEADS, VALUE_HEADS, WIDTH, TAPS = 16, 48, 128, 4
CHANNELS = 2 * KEY_HEADS * WIDTH + VALUE_HEADS * WIDTH
BRANCHES, HIDDEN = 4, 2560


def _attn(name, tokens, seqs, step=False, hk=KEY_HEADS, hv=VALUE_HEADS, dk=WIDTH, dv=WIDTH,
          delta=True, alpha=True, layout=0):
    c = {"kind": "attn", "tokens": tokens, "seqs": seqs, "step": step, "hk": hk, "hv": hv,
         "dk": dk, "dv": dv, "delta": delta, "alpha": alpha, "layout": layout}
    return {"name": name, **c} if name else c


def listed():
    return [
        # one sequence decoding: the state of 48 heads read, updated and written
        _attn("attn_step_1", 1, 1, step=True),
        # 61 sequences decoding together, their states in slots of a larger pool
        _attn("attn_step_61", 61, 61, step=True),
        # a short prompt, of an odd length
        _attn("attn_prompt_513", 513, 1),
        # the longest prompt: chunk after chunk of one sequence
        _attn("attn_prompt_16384", 16384, 1),
        # prompts of different lengths with single tokens between them, in one call
        _attn("attn_ragged_6001", 6001, 23, layout=7),
        # plain linear attention with a constant decay, narrower heads
        _attn("attn_decay_64_4099", 4099, 3, hk=8, hv=8, dk=64, dv=64, delta=False, alpha=False,
              layout=3),
        # the convolution of 32 sequences decoding together
        {"name": "conv_step_32", "kind": "conv", "tokens": 32, "seqs": 32, "step": True,
         "channels": CHANNELS, "taps": TAPS, "layout": 0},
        # and of a batch of prompts
        {"name": "conv_prompt_4097", "kind": "conv", "tokens": 4097, "seqs": 5, "step": False,
         "channels": CHANNELS, "taps": TAPS, "layout": 5},
        # the heads of one token behind the attention: norm and SiLU gate
        {"name": "norm_heads_1", "kind": "norm", "tokens": 1, "groups": VALUE_HEADS,
         "width": WIDTH, "gate": "silu"},
        # and of a prompt
        {"name": "norm_heads_4099", "kind": "norm", "tokens": 4099, "groups": VALUE_HEADS,
         "width": WIDTH, "gate": "silu"},
        # the end of a block for one token, four branches, with the next block's norm
        {"name": "join_1", "kind": "join", "tokens": 1, "branches": BRANCHES, "hidden": HIDDEN,
         "gate": "none", "post": True, "pre": True},
        # and for a long prompt
        {"name": "join_2499", "kind": "join", "tokens": 2499, "branches": BRANCHES,
         "hidden": HIDDEN, "gate": "sigmoid", "post": True, "pre": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, round(lo * (hi / lo) ** rng.random())))


def draw(rng):
    kind = rng.choice(("attn", "attn", "attn", "conv", "norm", "join"))
    layout = rng.randint(1, 1 << 20)
    if kind == "attn":
        step = rng.random() < 0.4
        tokens = _log_int(rng, 1, 64) if step else _log_int(rng, 2, 8192)
        hk, per = rng.choice((4, 8, 16)), rng.choice((1, 2, 3))
        return _attn("", tokens, tokens if step else _log_int(rng, 1, min(32, tokens)), step,
                     hk, hk * per, rng.choice((64, 128)), rng.choice((64, 128)),
                     rng.random() < 0.75, rng.random() < 0.75, layout)
    if kind == "conv":
        step = rng.random() < 0.4
        tokens = _log_int(rng, 1, 256) if step else _log_int(rng, 2, 4096)
        return {"kind": kind, "tokens": tokens,
                "seqs": tokens if step else _log_int(rng, 1, min(32, tokens)), "step": step,
                "channels": _log_int(rng, 64, CHANNELS), "taps": rng.randint(2, 6),
                "layout": layout}
    if kind == "norm":
        return {"kind": kind, "tokens": _log_int(rng, 1, 4099), "groups": rng.randint(1, 48),
                "width": rng.choice((64, 96, 128, 131, 256)),
                "gate": rng.choice(("none", "sigmoid", "silu"))}
    return {"kind": kind, "tokens": _log_int(rng, 1, 2499), "branches": rng.randint(1, 4),
            "hidden": rng.choice((640, 1001, 2048, 2560)),
            "gate": rng.choice(("none", "sigmoid", "silu")), "post": rng.random() < 0.7,
            "pre": rng.random() < 0.7}


# ------------------------------------------------------------------ inputs


def _lengths(case):
    """The sequences' lengths: about a third of a mixed batch are single tokens, as where prompts
    and decoding share a call."""
    n, s = case["tokens"], case["seqs"]
    if case["step"] or s == 1:
        return [1] * s if case["step"] else [n]
    r = random.Random(case["layout"])
    rest = n - s  # one token at least for each
    share = [0.0 if r.random() < 0.33 else r.random() ** 2 + 0.01 for _ in range(s)]
    share[r.randrange(s)] += 0.5
    total = sum(share)
    more = [int(rest * x / total) for x in share]
    more[max(range(s), key=lambda i: share[i])] += rest - sum(more)
    return [1 + m for m in more]


def _sequences(case, g, r):
    lengths = _lengths(case)
    offsets = [0]
    for n in lengths:
        offsets.append(offsets[-1] + n)
    seqs = len(lengths)
    pool = seqs + seqs // 4
    slots = torch.randperm(pool, generator=g, device=DEV)[:seqs].to(torch.int32)
    # a prompt begins with no state more often than not; a decoding sequence has one
    fresh = [0 if n == 1 or r.random() < 0.3 else 1 for n in lengths]
    return {"lengths": lengths, "pool": pool, "slots": slots,
            "offsets": torch.tensor(offsets, dtype=torch.int32, device=DEV),
            "fresh": torch.tensor(fresh, dtype=torch.int32, device=DEV)}


def _inputs(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    normal = lambda *s: torch.randn(s, generator=g, device=DEV)  # noqa: E731
    uniform = lambda lo, hi, *s: torch.rand(s, generator=g, device=DEV) * (hi - lo) + lo  # noqa: E731
    s = {}
    n = case["tokens"]
    if case["kind"] in ("attn", "conv"):
        s["seq"] = _sequences(case, g, random.Random(seed))
        pool = s["seq"]["pool"]
    if case["kind"] == "conv":
        c, taps = case["channels"], case["taps"]
        s["x"] = normal(n, c)
        s["w"] = normal(c, taps) * (1.0 / math.sqrt(taps))
        s["state"] = normal(pool, taps - 1, c)
    elif case["kind"] == "attn":
        hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
        # q, k and v lie side by side in a row, as the convolution leaves them
        x = normal(n, 2 * hk * dk + hv * dv)
        s["qkv"] = x * torch.sigmoid(x)
        s["state"] = normal(pool, hv, dk, dv) * 0.1
        if case["alpha"]:
            # decays as a trained layer has them: rates of 1 to 16, steps of 0.001 to 0.1
            s["rate"] = -uniform(1.0, 16.0, hv)
            step = torch.exp(uniform(math.log(0.001), math.log(0.1), hv))
            s["bias"] = torch.log(torch.expm1(step))
            s["alpha"] = normal(n, hv)
        else:
            # constant decays: memories of 32 to 1024 tokens
            s["rate"] = torch.log1p(-torch.exp2(-uniform(5.0, 10.0, hv)))
        if case["delta"]:
            s["beta"] = normal(n, hv)
    elif case["kind"] == "norm":
        w = case["groups"] * case["width"]
        s["x"] = normal(n, w) * 0.3
        s["w"] = 1.0 + 0.1 * normal(case["width"])
        if case["gate"] != "none":
            s["gate"] = normal(n, w)
    else:
        h, b = case["hidden"], case["branches"]
        s["x"] = normal(n, h)
        if case["gate"] != "none":
            s["gate"] = normal(n, h)
        s["residual"] = normal(n, b, h)
        s["write"] = 2.0 * torch.sigmoid(normal(n, b))
        if case["post"]:
            s["post"] = 0.1 * normal(h)
        if case["pre"]:
            s["pre"] = 0.1 * normal(b, h)
    return s


def prepare(case, seed):
    """The inputs, and the buffers that a serving loop keeps for the results."""
    s = {"case": case, **_inputs(case, seed)}
    zeros = lambda *shape: torch.zeros(shape, device=DEV)  # noqa: E731
    n = case["tokens"]
    if case["kind"] in ("attn", "conv"):
        s["plan"] = _plan(s["seq"]["lengths"])
        s["state_out"] = torch.zeros_like(s["state"])
        s["y"] = zeros(n, case["channels"] if case["kind"] == "conv"
                       else case["hv"] * case["dv"])
    elif case["kind"] == "norm":
        s["y"] = torch.zeros_like(s["x"])
    else:
        s["residual_out"] = torch.zeros_like(s["residual"])
        if case["pre"]:
            s["normalized"] = torch.zeros_like(s["residual"])
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
    if "seq" in s:
        q = s["seq"]
        p["seqs"] = kq_hip.sequences(case["tokens"], case["seqs"], q["pool"],
                                     None if case["step"] else q["offsets"].data_ptr(),
                                     q["slots"].data_ptr(), q["fresh"].data_ptr())
    if case["kind"] == "conv":
        p["conv"] = kq_hip.causal_conv(case["channels"], case["taps"], s["w"].data_ptr(),
                                       activation="silu")
    elif case["kind"] == "attn":
        ptr = lambda k: s[k].data_ptr() if k in s else None  # noqa: E731
        hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
        p["attn"] = kq_hip.linear_attention(hk, hv, dk, dv, dk ** -0.5, ptr("rate"), ptr("bias"),
                                            normalize=True, epsilon=EPS)
        row, qkv = 2 * hk * dk + hv * dv, s["qkv"].data_ptr()
        p["in"] = kq_hip.linear_attention_inputs(qkv, row, qkv + 4 * hk * dk, row,
                                                 qkv + 8 * hk * dk, row, ptr("alpha"), hv,
                                                 ptr("beta"), hv)
        p["bytes"] = kq_hip.linear_attention_scratch_bytes(p["attn"], p["seqs"])
        p["scratch"] = torch.empty(max(p["bytes"], 1), dtype=torch.uint8, device=DEV)
    elif case["kind"] == "norm":
        p["norm"] = kq_hip.gated_norm(case["groups"], case["width"], EPS, s["w"].data_ptr(),
                                      gate=case["gate"])
    else:
        ptr = lambda k: s[k].data_ptr() if k in s else None  # noqa: E731
        p["join"] = kq_hip.block_join(case["branches"], case["hidden"], EPS,
                                      post=ptr("post"), post_offset=1.0, gate=case["gate"],
                                      scale=0.5, pre=ptr("pre"), pre_offset=1.0)
    torch.cuda.synchronize()
    return p


def _run_own(s):
    p = s.get("own")
    if p is None:
        p = s["own"] = _own_plan(s)
    case, ctx = s["case"], p["ctx"]
    ptr = lambda k: s[k].data_ptr() if k in s else None  # noqa: E731
    if case["kind"] == "conv":
        c = case["channels"]
        ctx.causal_conv(p["conv"], p["seqs"], ptr("x"), c, ptr("state"), ptr("state_out"),
                        ptr("y"), c)
        return {"y": s["y"], "state": s["state_out"]}
    if case["kind"] == "attn":
        ctx.linear_attention(p["attn"], p["seqs"], p["in"], ptr("state"), ptr("state_out"),
                             ptr("y"), case["hv"] * case["dv"], p["scratch"].data_ptr(),
                             p["bytes"])
        return {"y": s["y"], "state": s["state_out"]}
    if case["kind"] == "norm":
        w = case["groups"] * case["width"]
        ctx.gated_norm(p["norm"], case["tokens"], ptr("x"), w, ptr("gate"), w, ptr("y"), w)
        return s["y"]
    ctx.block_join(p["join"], case["tokens"], ptr("x"), ptr("gate"), ptr("residual"),
                   ptr("write"), ptr("residual_out"), ptr("normalized"))
    return ({"residual": s["residual_out"], "normalized": s["normalized"]} if case["pre"]
            else s["residual_out"])


# ------------------------------------------------------------- plain forms


def _plan(lengths):
    """Index tables of the chunked plain form: the tokens of each chunk, and for each step the
    sequences that have a chunk there. A row that no token has points behind the last token."""
    n, starts, at = sum(lengths), [], 0
    for m in lengths:
        starts.append(at)
        at += m
    counts = [-(-m // CHUNK) for m in lengths]
    base = [sum(counts[:i]) for i in range(len(counts))]
    first = torch.tensor([starts[i] + CHUNK * c for i in range(len(lengths))
                          for c in range(counts[i])], dtype=torch.long)
    last = torch.tensor([starts[i] + lengths[i] for i in range(len(lengths))
                         for c in range(counts[i])], dtype=torch.long)
    rows = first[:, None] + torch.arange(CHUNK)
    rows = torch.where(rows < last[:, None], rows, n)
    steps = []
    for c in range(max(counts)):
        who = [i for i in range(len(lengths)) if counts[i] > c]
        steps.append((torch.tensor(who, device=DEV), torch.tensor([base[i] + c for i in who],
                                                                  device=DEV)))
    return {"rows": rows.to(DEV), "steps": steps,
            "starts": torch.tensor(starts, device=DEV),
            "seq_of": torch.tensor([i for i, m in enumerate(lengths) for _ in range(m)],
                                   device=DEV)}


def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-torch.abs(x)))


def _gate(kind, g):
    return torch.sigmoid(g) if kind == "sigmoid" else g * torch.sigmoid(g)


def _rms(x):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)


def _start_states(s):
    q = s["seq"]
    got = s["state"][q["slots"].long()]
    return torch.where(q["fresh"].view(-1, *[1] * (got.dim() - 1)) != 0, torch.zeros_like(got),
                       got)


def _end_states(s, states):
    out = torch.zeros_like(s["state"])
    out[s["seq"]["slots"].long()] = states
    return out


def _conv(s):
    x, w, taps = s["x"], s["w"], s["case"]["taps"]
    plan, start = s["plan"], _start_states(s)
    at = torch.arange(x.shape[0], device=DEV)
    seq = plan["seq_of"]
    y = torch.zeros_like(x)
    for j in range(taps):  # tap j reads the input taps - 1 - j tokens before
        back = taps - 1 - j
        from_start = at - plan["starts"][seq] - back
        before = start[seq, torch.clamp(from_start + taps - 1, max=taps - 2)]
        here = torch.where((from_start >= 0)[:, None], x[torch.clamp(at - back, min=0)], before)
        y = y + w[:, j] * here
    lengths = s["seq"]["offsets"][1:].long() - s["seq"]["offsets"][:-1].long()
    old = torch.arange(taps - 1, device=DEV) + lengths[:, None]  # in [state, inputs]
    inside = torch.clamp(plan["starts"][:, None] + old - (taps - 1), 0, x.shape[0] - 1)
    end = torch.where((old >= taps - 1)[:, :, None], x[inside],
                      torch.gather(start, 1, torch.clamp(old, max=taps - 2)[:, :, None]
                                   .expand(-1, -1, x.shape[1])))
    return {"y": y * torch.sigmoid(y), "state": _end_states(s, end)}


def _rows(s):
    """Normalized q (scaled) and k [tokens][key heads][dk], v, log decay in 64 bits, beta."""
    case, n = s["case"], s["case"]["tokens"]
    hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
    q, k, v = s["qkv"].split((hk * dk, hk * dk, hv * dv), 1)
    unit = lambda x: x * torch.rsqrt(x.square().sum(-1, keepdim=True) + EPS)  # noqa: E731
    q = unit(q.reshape(n, hk, dk)) * dk ** -0.5
    k = unit(k.reshape(n, hk, dk))
    decay = s["rate"].double().expand(n, hv)
    if case["alpha"]:
        decay = decay * _softplus(s["alpha"].double() + s["bias"].double())
    beta = torch.sigmoid(s["beta"]) if case["delta"] else None
    return q, k, v.reshape(n, hv, dv), decay, beta


def _attn_step(s):
    q, k, v, decay, beta = _rows(s)
    per = s["case"]["hv"] // s["case"]["hk"]
    q, k = q.repeat_interleave(per, 1), k.repeat_interleave(per, 1)
    state = _start_states(s) * torch.exp(decay).float()[:, :, None, None]
    d = v
    if beta is not None:
        d = beta[:, :, None] * (v - (k[:, :, None, :] @ state)[:, :, 0])
    state = state + k[:, :, :, None] * d[:, :, None, :]
    y = (q[:, :, None, :] @ state)[:, :, 0]
    return {"y": y.reshape(y.shape[0], -1), "state": _end_states(s, state)}


def _attn_chunks(s):
    case = s["case"]
    per, dv = case["hv"] // case["hk"], case["dv"]
    q, k, v, decay, beta = _rows(s)
    rows = s["plan"]["rows"]
    nc = rows.shape[0]
    pad = lambda x: torch.cat((x, torch.zeros_like(x[:1])))[rows].transpose(1, 2)  # noqa: E731
    q, k, v = pad(q).contiguous(), pad(k).contiguous(), pad(v).contiguous()
    total = torch.cumsum(pad(decay[:, :, None])[..., 0], 2)       # [chunks][hv][64], 64 bits
    tri = torch.tril(torch.ones(CHUNK, CHUNK, device=DEV))
    fall = torch.exp(torch.clamp(total[..., :, None] - total[..., None, :], max=0)).float() * tri
    kt = k.transpose(2, 3).contiguous()
    mix = (q @ kt).repeat_interleave(per, 1) * fall               # what token i takes from j
    q, k = q.repeat_interleave(per, 1), k.repeat_interleave(per, 1)
    from_start = torch.exp(total).float()[..., None]
    to_end = torch.exp(total[..., -1:] - total).float()[..., None]
    whole = from_start[..., -1:, :]
    if beta is not None:
        b = pad(beta[:, :, None])
        low = (b * (k @ k.transpose(2, 3).contiguous()) * fall) * torch.tril(tri, -1)
        solve = torch.zeros_like(low)
        for i in range(CHUNK):  # (1 + low) solve = diag(beta), row by row
            solve[..., i, :] = -(low[..., i:i + 1, :] @ solve)[..., 0, :]
            solve[..., i, i] += b[..., i, 0]
    states = _start_states(s).clone()
    y = torch.zeros(case["tokens"] + 1, case["hv"], dv, device=DEV)
    for who, chunk in s["plan"]["steps"]:
        st, kc, d = states[who], k[chunk], v[chunk]
        if beta is not None:
            d = solve[chunk] @ (d - from_start[chunk] * (kc @ st))
        o = from_start[chunk] * (q[chunk] @ st) + mix[chunk] @ d
        y[rows[chunk]] = o.transpose(1, 2)
        kd = (kc * to_end[chunk]).transpose(2, 3).contiguous()
        states[who] = whole[chunk] * st + kd @ d
    return {"y": y[:-1].reshape(case["tokens"], -1), "state": _end_states(s, states)}


def _norm(s):
    case = s["case"]
    x = s["x"].view(-1, case["groups"], case["width"])
    y = _rms(x) * s["w"]
    if case["gate"] != "none":
        y = y * _gate(case["gate"], s["gate"].view_as(x))
    return y.reshape(s["x"].shape)


def _join(s):
    case, y = s["case"], s["x"]
    if case["post"]:
        y = _rms(y) * (1.0 + s["post"])
    if case["gate"] != "none":
        y = y * _gate(case["gate"], s["gate"])
    r = s["residual"] + (0.5 * s["write"])[:, :, None] * y[:, None, :]
    if not case["pre"]:
        return r
    return {"residual": r, "normalized": _rms(r) * (1.0 + s["pre"])}


def run(s):
    if own:
        return _run_own(s)
    kind = s["case"]["kind"]
    if kind == "attn":
        return _attn_step(s) if s["case"]["step"] else _attn_chunks(s)
    return {"conv": _conv, "norm": _norm, "join": _join}[kind](s)


# ------------------------------------------------------------ what it costs


def work(case):
    n = case["tokens"]
    if case["kind"] == "conv":
        c, taps, seqs = case["channels"], case["taps"], case["seqs"]
        return {"bytes": 4 * (2 * n * c + c * taps + 2 * seqs * (taps - 1) * c),
                "flops": n * c * (2 * taps + 4)}
    if case["kind"] == "attn":
        hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
        row = 2 * hk * dk + 2 * hv * dv + hv * (int(case["alpha"]) + int(case["delta"]))
        return {"bytes": 4 * (n * row + 2 * case["seqs"] * hv * dk * dv),
                "flops": n * hv * dk * dv * (7 if case["delta"] else 5)}
    if case["kind"] == "norm":
        w, gate = case["groups"] * case["width"], case["gate"] != "none"
        return {"bytes": 4 * (n * w * (2 + gate) + case["width"]), "flops": n * w * (4 + 4 * gate)}
    h, b, gate = case["hidden"], case["branches"], case["gate"] != "none"
    return {"bytes": 4 * (n * h * (1 + gate + b * (2 + case["pre"])) + n * b +
                          h * (case["post"] + b * case["pre"])),
            "flops": n * h * (4 * case["post"] + 4 * gate + b * (2 + 4 * case["pre"]))}


# ---------------------------------------------- the definitions in 64 bits


def _exact_attn(case, t):
    """Token after token, every sequence that still has one at a time."""
    seq, n = t["seq"], case["tokens"]
    hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
    at = t["qkv"].double()
    head = torch.arange(hv, device=DEV) // (hv // hk)
    query = at[:, :hk * dk].view(n, hk, dk)
    key = at[:, hk * dk:2 * hk * dk].view(n, hk, dk)
    value = at[:, 2 * hk * dk:].view(n, hv, dv)
    query = query / (query.pow(2).sum(2, keepdim=True) + EPS).sqrt() / math.sqrt(dk)
    key = key / (key.pow(2).sum(2, keepdim=True) + EPS).sqrt()
    rate = t["rate"].double()
    keep = torch.exp(rate * torch.log(1 + torch.exp(t["alpha"].double() + t["bias"].double()))
                     if case["alpha"] else rate.expand(n, hv))
    part = 1 / (1 + torch.exp(-t["beta"].double())) if case["delta"] else None
    states = t["state"].double()[seq["slots"].long()]
    states[seq["fresh"] != 0] = 0
    y = torch.zeros(n, hv, dv, dtype=torch.float64, device=DEV)
    lengths = torch.tensor(seq["lengths"], device=DEV)
    begin = seq["offsets"][:-1].long()
    order = torch.argsort(lengths, descending=True)
    counts = sorted(seq["lengths"], reverse=True)
    states, begin = states[order], begin[order]
    live = len(counts)
    for i in range(counts[0]):
        while counts[live - 1] <= i:
            live -= 1
        rows = begin[:live] + i
        k, q, v = key[rows][:, head], query[rows][:, head], value[rows]
        st = states[:live]
        st *= keep[rows][:, :, None, None]
        if part is not None:
            v = part[rows][:, :, None] * (v - (st * k[:, :, :, None]).sum(2))
        st += k[:, :, :, None] * v[:, :, None, :]
        y[rows] = (st * q[:, :, :, None]).sum(2)
    out = torch.zeros(t["state"].shape, dtype=torch.float64, device=DEV)
    out[seq["slots"].long()[order]] = states
    return {"y": y.view(n, -1), "state": out}


def _exact_conv(case, t):
    seq, taps, w = t["seq"], case["taps"], t["w"].double()
    out = torch.zeros(t["state"].shape, dtype=torch.float64, device=DEV)
    parts, at = [], 0
    slots, fresh = seq["slots"].tolist(), seq["fresh"].tolist()
    for i, m in enumerate(seq["lengths"]):
        st = t["state"][slots[i]].double()
        line = torch.cat((st * 0 if fresh[i] else st, t["x"][at:at + m].double()))
        y = sum(line[j:j + m] * w[:, j] for j in range(taps))
        parts.append(y / (1 + torch.exp(-y)))
        out[slots[i]] = line[m:]
        at += m
    return {"y": torch.cat(parts), "state": out}


def _exact_rms(x):
    return x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt()


def _exact_gate(kind, g):
    p = 1 / (1 + torch.exp(-g.double()))
    return p if kind == "sigmoid" else g.double() * p


def exact(case, seed):
    t = _inputs(case, seed)
    if case["kind"] == "attn":
        return _exact_attn(case, t)
    if case["kind"] == "conv":
        return _exact_conv(case, t)
    if case["kind"] == "norm":
        x = t["x"].double().view(case["tokens"], case["groups"], case["width"])
        y = (_exact_rms(x) * t["w"].double()).view(case["tokens"], -1)
        return y if case["gate"] == "none" else y * _exact_gate(case["gate"], t["gate"])
    y = t["x"].double()
    if case["post"]:
        y = _exact_rms(y) * (1 + t["post"].double())
    if case["gate"] != "none":
        y = y * _exact_gate(case["gate"], t["gate"])
    r = t["residual"].double() + t["write"].double()[:, :, None] * y[:, None, :] / 2
    if not case["pre"]:
        return r
    return {"residual": r, "normalized": _exact_rms(r) * (1 + t["pre"].double())}

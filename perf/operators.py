"""The decoding operators and their measured cases.

Five calls of `B200Session` carry a generation loop over a key/value cache:

  kv_cache_write      new keys and values go into the cache, quantised to int8 where the cache is int8
  kv_cache_read       the values a range of the cache stands for
  kv_cache_attention  attention of one token, or of a chain or tree of drafted tokens, over the cache
  beam_select         the best continuations of a group of beams over the vocabulary
  beam_reorder        caches, histories and other per-beam state rearranged to follow the selected beams

With `own` false, `run` computes them in elementary torch operations in 32 bits (64 where a rounding decides a whole
number); with `own` true it makes the framework's calls on the same data.

A cache is [slots, heads, capacity, head size]; an int8 cache holds codes c and one 32-bit scale s per slot, head and
position, and stands for c * s.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "int8": torch.int8}
_session = None


def _open():
    """The session that a program keeps for its lifetime."""
    global _session
    if _session is None:
        from sheaf_b200.session import B200Session
        _session = B200Session(device=torch.cuda.current_device())
    return _session


# --------------------------------------------------------------------------- cases

def listed():
    return [
        # one decoding step of the nanoGPT shape, one sequence: six heads of one token into the cache (latency)
        {"name": "write_step", "op": "write", "slots": 1, "tokens": 1, "heads": 6, "dim": 64, "capacity": 256,
         "input": "f32", "cache": "int8"},
        # the prompts of a GPT-2-small batch: 8 x 1024 tokens of one layer
        {"name": "write_prompt", "op": "write", "slots": 8, "tokens": 1024, "heads": 12, "dim": 64, "capacity": 1024,
         "input": "f32", "cache": "int8"},
        # a ragged batch's cache read back as the values it stands for
        {"name": "read_ragged", "op": "read", "slots": 24, "heads": 12, "dim": 64, "capacity": 4096, "cache": "int8",
         "output": "f32"},
        # one decoding step of the nanoGPT shape: one token over a 256-position cache (latency)
        {"name": "attention_step", "op": "attention", "slots": 1, "tokens": 1, "q_heads": 6, "heads": 6, "dim": 64,
         "capacity": 256, "input": "f32", "cache": "f32", "tree": False, "low": 0.5, "high": 0.95},
        # one decoding step of a ragged batch of the GPT-2-small shape over int8 caches
        {"name": "attention_batch", "op": "attention", "slots": 64, "tokens": 1, "q_heads": 12, "heads": 12, "dim": 64,
         "capacity": 1024, "input": "f32", "cache": "int8", "tree": False, "low": 0.05, "high": 0.95},
        # one decoding step over long bf16 caches whose heads are shared by four query heads each
        {"name": "attention_long", "op": "attention", "slots": 4, "tokens": 1, "q_heads": 32, "heads": 8, "dim": 128,
         "capacity": 32768, "input": "bf16", "cache": "bf16", "tree": False, "low": 0.8, "high": 0.999},
        # a tree of 63 drafted tokens of the GPT-2-small shape, queries in 32 bits
        {"name": "attention_tree", "op": "attention", "slots": 8, "tokens": 63, "q_heads": 12, "heads": 12, "dim": 64,
         "capacity": 1024, "input": "f32", "cache": "bf16", "tree": True, "low": 0.3, "high": 0.9},
        # a tree of 32 drafted tokens over long int8 caches, eight query heads to a cache head
        {"name": "attention_tree_long", "op": "attention", "slots": 8, "tokens": 32, "q_heads": 32, "heads": 4,
         "dim": 128, "capacity": 16384, "input": "bf16", "cache": "int8", "tree": True, "low": 0.5, "high": 0.95},
        # beam search of one sequence over the nanoGPT vocabulary (latency)
        {"name": "select_small", "op": "select", "groups": 1, "beams": 4, "vocab": 65, "input": "f32", "eos": -1},
        # 32 sequences of 8 beams over the GPT-2-small vocabulary, some beams finished
        {"name": "select_vocab", "op": "select", "groups": 32, "beams": 8, "vocab": 50304, "input": "f32",
         "eos": 50256},
        # the nanoGPT caches of four beams, all layers
        {"name": "reorder_small", "op": "reorder", "groups": 1, "beams": 4, "layers": 6, "heads": 6, "dim": 64,
         "capacity": 256, "cache": "f32", "low": 0.5, "high": 0.9},
        # the GPT-2-small caches of eight sequences of eight beams, all layers
        {"name": "reorder_batch", "op": "reorder", "groups": 8, "beams": 8, "layers": 12, "heads": 12, "dim": 64,
         "capacity": 1024, "cache": "bf16", "low": 0.3, "high": 0.9},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["write", "read", "attention", "attention", "attention", "select", "reorder"])
    if op == "write":
        heads, dim = rng.randint(1, 16), rng.choice([32, 64, 80, 128, 256])
        slots = _log(rng, 1, 96)
        tokens = min(_log(rng, 1, 1024), max(1, 8 * 1024 * 12 * 64 // (slots * heads * dim)))
        return {"op": op, "slots": slots, "tokens": tokens, "heads": heads, "dim": dim,
                "capacity": tokens + rng.randint(0, 300), "input": rng.choice(["f32", "bf16"]),
                "cache": rng.choice(["f32", "bf16", "int8", "int8"])}
    if op == "read":
        heads, dim = rng.randint(1, 16), rng.choice([32, 64, 80, 128, 256])
        slots = _log(rng, 1, 48)
        capacity = min(_log(rng, 1, 8192), max(1, 24 * 4096 * 12 * 64 // (slots * heads * dim)))
        return {"op": op, "slots": slots, "heads": heads, "dim": dim, "capacity": capacity,
                "cache": rng.choice(["f32", "bf16", "int8", "int8"]), "output": rng.choice(["f32", "bf16"])}
    if op == "attention":
        tokens = rng.choice([1, 1, 1, _log(rng, 2, 64), _log(rng, 2, 64)])
        group = rng.choice([1, 1, 2, 3, 4, 8])
        heads, dim = rng.randint(1, 12), rng.choice([32, 64, 64, 80, 128, 128, 256])
        slots = _log(rng, 1, 48)
        most = 1 << 23 if tokens == 1 else 1 << 21
        capacity = tokens + min(_log(rng, 1, 24000), max(1, most // (slots * heads * group)))
        capacity = min(capacity, max(tokens, (1 << 28) // (slots * heads * dim)))
        kind = rng.choice(["f32", "bf16"])
        return {"op": op, "slots": slots, "tokens": tokens, "q_heads": heads * group, "heads": heads, "dim": dim,
                "capacity": capacity, "input": kind,
                "cache": rng.choice(["f32", "bf16", "int8"] if kind == "f32" else ["bf16", "int8"]),
                "tree": tokens > 1 and rng.random() < 0.7, "low": round(rng.uniform(0.0, 0.6), 3),
                "high": round(rng.uniform(0.6, 1.0), 3)}
    if op == "select":
        beams, vocab = rng.randint(1, 16), _log(rng, 2, 60000)
        groups = min(_log(rng, 1, 64), max(1, 32 * 8 * 50304 // (beams * vocab)))
        return {"op": op, "groups": groups, "beams": beams, "vocab": vocab, "input": rng.choice(["f32", "bf16"]),
                "eos": rng.choice([-1, rng.randrange(vocab)])}
    heads, dim = rng.randint(1, 12), rng.choice([32, 64, 80, 128])
    beams, layers = rng.randint(2, 16), rng.randint(1, 12)
    groups = _log(rng, 1, 8)
    kind = rng.choice(["f32", "bf16"])
    most = 64 * 12 * 12 * 1024 * 64 // (groups * beams * layers * heads * dim * _bytes(kind))
    capacity = min(_log(rng, 8, 2048), max(2, most))
    return {"op": op, "groups": groups, "beams": beams, "layers": layers, "heads": heads, "dim": dim,
            "capacity": capacity, "cache": kind, "low": round(rng.uniform(0.0, 0.6), 3),
            "high": round(rng.uniform(0.6, 1.0), 3)}


# --------------------------------------------------------------------------- inputs

def _spread(count, low, high, gen):
    """`count` whole numbers spread evenly over [low, high], in an order that the seed gives."""
    v = torch.linspace(float(low), float(high), count, device="cuda", dtype=torch.float64).round().to(torch.int32)
    return v[torch.randperm(count, generator=gen, device="cuda")].contiguous()


def _lengths(c):
    return int(c["low"] * (c["capacity"] - c.get("tokens", 0))), int(c["high"] * (c["capacity"] - c.get("tokens", 0)))


def _randn(shape, gen, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda", dtype=dtype)


def _keys(shape, gen, dtype):
    """Keys or values [..., head size]: most channels near 1, a few large ones, as in trained models."""
    x = _randn(shape, gen, dtype)
    x[..., ::16] *= 6
    return x


def _cache(shape, kind, gen):
    """A filled cache and its scales."""
    if kind != "int8":
        return _keys(shape, gen, _TYPES[kind]), None
    codes = torch.randint(-127, 128, shape, generator=gen, device="cuda", dtype=torch.int8)
    scale = torch.rand(shape[:-1], generator=gen, device="cuda") * 0.02 + 0.005
    return codes, scale


def prepare(case, seed):
    c, gen = case, torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": c}
    if c["op"] == "write":
        n, t, h, d = c["slots"], c["tokens"], c["heads"], c["dim"]
        shape = (n, h, c["capacity"], d)
        s["k"], s["v"] = (_keys((n, t, h, d), gen, _TYPES[c["input"]]) for _ in range(2))
        s["positions"] = _spread(n, 0, c["capacity"] - t, gen)
        s["k_cache"], s["v_cache"] = (torch.zeros(shape, device="cuda", dtype=_TYPES[c["cache"]]) for _ in range(2))
        s["k_scale"], s["v_scale"] = (torch.zeros(shape[:3], device="cuda") if c["cache"] == "int8" else None
                                      for _ in range(2))
        s["k_out"], s["v_out"] = (torch.zeros((n, h, t, d), device="cuda") for _ in range(2))
    elif c["op"] == "read":
        shape = (c["slots"], c["heads"], c["capacity"], c["dim"])
        s["k_cache"], s["k_scale"] = _cache(shape, c["cache"], gen)
        s["v_cache"], s["v_scale"] = _cache(shape, c["cache"], gen)
        s["counts"] = _spread(c["slots"], c["capacity"] // 8, c["capacity"], gen)
        s["k_out"], s["v_out"] = (torch.zeros(shape, device="cuda", dtype=_TYPES[c["output"]]) for _ in range(2))
    elif c["op"] == "attention":
        n, t = c["slots"], c["tokens"]
        shape = (n, c["heads"], c["capacity"], c["dim"])
        s["k_cache"], s["k_scale"] = _cache(shape, c["cache"], gen)
        s["v_cache"], s["v_scale"] = _cache(shape, c["cache"], gen)
        s["q"] = _randn((n, t, c["q_heads"], c["dim"]), gen).to(_TYPES[c["input"]])
        s["positions"] = _spread(n, *_lengths(c), gen)
        s["parents"] = None
        if c["tree"]:  # token i continues one of the up to eight tokens before it, or (-1) the sequence itself
            i = torch.arange(t, device="cuda", dtype=torch.float32)
            back = torch.rand((n, t), generator=gen, device="cuda") * torch.clamp(i + 1, max=8)
            s["parents"] = (i - 1 - back.floor()).to(torch.int32).contiguous()
        s["out"] = torch.zeros_like(s["q"])
    elif c["op"] == "select":
        g, w, v = c["groups"], c["beams"], c["vocab"]
        s["logits"] = (_randn((g * w, v), gen) * 2.5).to(_TYPES[c["input"]])
        s["scores"] = (-20 * torch.rand((g, w), generator=gen, device="cuda")).sort(1, descending=True)[0].contiguous()
        s["finished"] = (torch.rand((g, w), generator=gen, device="cuda") < 0.15).to(torch.int32)
        s["out_scores"] = torch.zeros((g, w), device="cuda")
        s["out_parents"], s["out_tokens"], s["out_finished"] = (
            torch.zeros((g, w), device="cuda", dtype=torch.int32) for _ in range(3))
    else:
        n = c["groups"] * c["beams"]
        shape = (n, c["heads"], c["capacity"], c["dim"])
        s["states"] = [_randn(shape, gen, _TYPES[c["cache"]]) for _ in range(2 * c["layers"])]
        s["states"].append(torch.randint(0, 50000, (n, c["capacity"]), generator=gen, device="cuda",
                                         dtype=torch.int32))
        s["axes"] = [2] * (2 * c["layers"]) + [1]
        s["parents"] = torch.randint(0, c["beams"], (c["groups"], c["beams"]), generator=gen, device="cuda",
                                     dtype=torch.int32)
        s["lengths"] = _spread(c["groups"], *_lengths(c), gen).repeat_interleave(c["beams"]).contiguous()
    if own:
        _wrap(s)
    return s


def _wrap(s):
    """The handles of the same memory that a program of the framework holds."""
    from sheaf_b200.session import KVCache
    b = _open()
    h = {k: b.wrap_torch(v) for k, v in s.items() if isinstance(v, torch.Tensor)}
    if "k_cache" in h:
        h["cache"] = KVCache(h["k_cache"], h["v_cache"], h.get("k_scale"), h.get("v_scale"))
    if "states" in s:
        h["states"] = [b.wrap_torch(x) for x in s["states"]]
    torch.cuda.synchronize()  # the session's stream is its own: the inputs are there before its first call
    s["handles"] = h


# --------------------------------------------------------------------------- one pass

def run(s):
    op = s["case"]["op"]
    if own:
        return {"write": _own_write, "read": _own_read, "attention": _own_attention, "select": _own_select,
                "reorder": _own_reorder}[op](s)
    return {"write": _write, "read": _read, "attention": _attention, "select": _select, "reorder": _reorder}[op](s)


def _own_write(s):
    h = s["handles"]
    _open().kv_cache_write(h["cache"], h["positions"], h["k"], h["v"])
    _open().kv_cache_read(h["cache"], h["k_out"], h["v_out"], starts=h["positions"])
    return s["k_out"], s["v_out"]


def _own_read(s):
    h = s["handles"]
    _open().kv_cache_read(h["cache"], h["k_out"], h["v_out"], counts=h["counts"])
    return s["k_out"], s["v_out"]


def _own_attention(s):
    h = s["handles"]
    _open().kv_cache_attention(h["cache"], h["positions"], h["q"], h["out"], parents=h.get("parents"))
    return s["out"]


def _own_select(s):
    h, eos = s["handles"], s["case"]["eos"]
    if eos < 0:
        _open().beam_select(h["logits"], h["scores"], h["out_scores"], h["out_parents"], h["out_tokens"])
    else:
        _open().beam_select(h["logits"], h["scores"], h["out_scores"], h["out_parents"], h["out_tokens"],
                            finished=h["finished"], out_finished=h["out_finished"], eos=eos)
    return s["out_scores"], s["out_parents"], s["out_tokens"], s["out_finished"]


def _own_reorder(s):
    h = s["handles"]
    _open().beam_reorder(h["states"], h["parents"], time_axes=s["axes"], lengths=h["lengths"])
    return s["states"]


def _codes(x):
    """int8 codes and scales of rows [..., head size]: the scale is the largest magnitude / 127."""
    scale = (x.double().abs().amax(-1) / 127).float()
    ratio = x.double() / scale.double()[..., None]
    codes = torch.where(scale[..., None] > 0, ratio.round(), torch.zeros_like(ratio))
    return codes.clamp(-127, 127).to(torch.int8), scale


def _put(x, cache, scale, slot, place):
    if scale is None:
        cache[slot, :, place] = x.to(cache.dtype)
    else:
        codes, step = _codes(x)
        cache[slot, :, place] = codes
        scale[slot, :, place] = step


def _values(cache, scale):
    return cache.float() if scale is None else cache.float() * scale[..., None]


def _write(s):
    n, t = s["k"].shape[:2]
    slot = torch.arange(n, device="cuda")[:, None]
    place = s["positions"].long()[:, None] + torch.arange(t, device="cuda")
    _put(s["k"], s["k_cache"], s["k_scale"], slot, place)
    _put(s["v"], s["v_cache"], s["v_scale"], slot, place)
    got = [_values(c[slot, :, place], None if z is None else z[slot, :, place]).transpose(1, 2).contiguous()
           for c, z in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"]))]
    return got[0], got[1]


def _read(s):
    live = torch.arange(s["case"]["capacity"], device="cuda") < s["counts"][:, None]
    live = live[:, None, :, None]
    for out, cache, scale in ((s["k_out"], s["k_cache"], s["k_scale"]), (s["v_out"], s["v_cache"], s["v_scale"])):
        out.copy_(torch.where(live, _values(cache, scale).to(out.dtype), out))
    return s["k_out"], s["v_out"]


def _visible(s):
    """[slots, tokens, capacity]: which positions a token attends to: those before the drafted tokens, its
    ancestors among the drafted tokens, and itself."""
    c = s["case"]
    t, pos = c["tokens"], s["positions"].long()
    if s["parents"] is None:
        seen = torch.ones((t, t), device="cuda").tril().expand(c["slots"], t, t)
    else:  # with P the parents as a 0/1 matrix, (1 + P)^64 is positive exactly at ancestors and selves
        step = (s["parents"][..., None] == torch.arange(t, device="cuda")).double() + torch.eye(t, device="cuda")
        two = step @ step
        four = two @ two
        sixteen = (four @ four) @ (four @ four)
        seen = (sixteen @ sixteen) @ (sixteen @ sixteen)
    at = torch.arange(c["capacity"], device="cuda")[None, None]
    behind = (at - pos[:, None, None]).clamp(0, t - 1).expand(c["slots"], t, c["capacity"])
    drafted = (at >= pos[:, None, None]) & (at < pos[:, None, None] + t)
    return (at < pos[:, None, None]) | (drafted & (seen.gather(2, behind) > 0))


def _attention(s):
    c = s["case"]
    n, t, h, d = c["slots"], c["tokens"], c["heads"], c["dim"]
    g = c["q_heads"] // h
    q = s["q"].float().view(n, t, h, g, d).permute(0, 2, 3, 1, 4).reshape(n, h, g * t, d)
    score = (q * (1 / math.sqrt(d))) @ _values(s["k_cache"], s["k_scale"]).transpose(-1, -2)
    score = score.view(n, h, g, t, c["capacity"])
    score = torch.where(_visible(s)[:, None, None], score, -math.inf)
    p = (score - score.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    out = p.view(n, h, g * t, c["capacity"]) @ _values(s["v_cache"], s["v_scale"])
    return out.view(n, h, g, t, d).permute(0, 3, 1, 2, 4).reshape(n, t, h * g, d).to(s["q"].dtype)


def _select(s):
    c = s["case"]
    g, w, v = c["groups"], c["beams"], c["vocab"]
    z = s["logits"].float()
    # the best of each beam by logit, the lowest token first among equals: one whole number orders both
    bits = (z + 0.0).view(torch.int32).long()
    order = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF)) * (1 << 32) - torch.arange(v, device="cuda")
    token = -(order.topk(min(w, v), dim=1)[0] % -(1 << 32))
    z = z.double()
    top = z.amax(1, keepdim=True)
    total = top + (z - top).exp().sum(1, keepdim=True).log()
    cand = s["scores"].view(-1, 1).double() + (z.gather(1, token) - total)
    done = torch.zeros_like(s["finished"])
    if c["eos"] >= 0:  # a finished beam goes on with the end token alone, at its score
        done = s["finished"]
        over = (done != 0).view(-1, 1)
        first = torch.arange(token.shape[1], device="cuda") == 0
        cand = torch.where(over, torch.where(first, s["scores"].view(-1, 1).double(), -math.inf), cand)
        token = torch.where(over, c["eos"], token)
    cand, token = cand.view(g, -1), token.view(g, -1)
    flat = torch.arange(w, device="cuda").repeat_interleave(cand.shape[1] // w) * v + token
    by = flat.sort(dim=1, stable=True)[1]
    cand, token, flat = cand.gather(1, by), token.gather(1, by), flat.gather(1, by)
    pick = cand.sort(dim=1, descending=True, stable=True)[1][:, :w]
    parent = flat.gather(1, pick).div(v, rounding_mode="floor")
    token = token.gather(1, pick)
    if c["eos"] >= 0:
        done = (done.gather(1, parent) != 0) | (token == c["eos"])
    return cand.gather(1, pick).float(), parent.int(), token.int(), done.int()


def _reorder(s):
    c = s["case"]
    first = torch.arange(c["groups"], device="cuda")[:, None] * c["beams"]
    source = (first + s["parents"]).view(-1)
    live = torch.arange(c["capacity"], device="cuda") < s["lengths"][source][:, None]
    shape = {1: (-1, c["capacity"]), 2: (-1, 1, c["capacity"], 1)}
    return [x.copy_(torch.where(live.view(shape[a]), x[source], x)) for x, a in zip(s["states"], s["axes"])]


# --------------------------------------------------------------------------- what a pass cannot do without

def _bytes(kind):
    return {"f32": 4, "bf16": 2, "int8": 1}[kind]


def work(c):
    if c["op"] == "write":  # rows in, rows into the cache, rows read back as values
        rows = 2 * c["slots"] * c["tokens"] * c["heads"]
        kept = c["dim"] * _bytes(c["cache"]) + (4 if c["cache"] == "int8" else 0)
        return {"bytes": rows * (c["dim"] * _bytes(c["input"]) + 2 * kept + 4 * c["dim"]), "flops": 0}
    if c["op"] == "read":
        rows = 2 * c["slots"] * c["heads"] * (c["capacity"] // 8 + c["capacity"]) / 2
        kept = c["dim"] * _bytes(c["cache"]) + (4 if c["cache"] == "int8" else 0)
        return {"bytes": rows * (kept + c["dim"] * _bytes(c["output"])), "flops": 0}
    if c["op"] == "attention":
        rows = c["slots"] * (sum(_lengths(c)) / 2 + c["tokens"])
        kept = c["dim"] * _bytes(c["cache"]) + (4 if c["cache"] == "int8" else 0)
        q = c["slots"] * c["tokens"] * c["q_heads"] * c["dim"]
        return {"bytes": 2 * rows * c["heads"] * kept + 2 * q * _bytes(c["input"]),
                "flops": 4 * rows * c["q_heads"] * c["dim"] * c["tokens"]}
    if c["op"] == "select":
        n = c["groups"] * c["beams"]
        return {"bytes": n * c["vocab"] * _bytes(c["input"]) + 28 * n, "flops": 4 * n * c["vocab"]}
    # of w beams with parents drawn alike, 1 - 1/w move; what they come from is read once
    w = c["beams"]
    moved, sources = w - 1, w * (1 - (1 - 1 / w) ** (w - 1))
    row = 2 * c["layers"] * c["heads"] * c["dim"] * _bytes(c["cache"]) + 4
    return {"bytes": c["groups"] * (moved + sources) * row * sum(_lengths(c)) / 2, "flops": 0}


# --------------------------------------------------------------------------- the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "write":
        return tuple(_exact_kept(s[x], c["cache"]) for x in ("k", "v"))
    if c["op"] == "read":
        got = []
        for x in ("k", "v"):
            out = s[x + "_out"].double()
            for i, n in enumerate(s["counts"].tolist()):
                live = s[x + "_cache"][i, :, :n].double()
                out[i, :, :n] = live if s[x + "_scale"] is None else live * s[x + "_scale"][i, :, :n, None].double()
            got.append(out)
        return tuple(got)
    if c["op"] == "attention":
        return _exact_attention(s)
    if c["op"] == "select":
        return _exact_select(s)
    keep = [x.clone() for x in s["states"]]
    parents, lengths = s["parents"].tolist(), s["lengths"].tolist()
    for g, row in enumerate(parents):
        for j, p in enumerate(row):
            to, of = g * c["beams"] + j, g * c["beams"] + p
            for x, y, axis in zip(s["states"], keep, s["axes"]):
                x[to].narrow(axis - 1, 0, lengths[of]).copy_(y[of].narrow(axis - 1, 0, lengths[of]))
    return [x.double() if x.is_floating_point() else x for x in s["states"]]


def _exact_kept(x, kind):
    x = x.double().transpose(1, 2)
    if kind == "f32":
        return x.contiguous()
    if kind == "bf16":
        return x.float().bfloat16().double().contiguous()
    step = (x.abs().amax(-1, keepdim=True) / 127).float().double()
    return torch.where(step > 0, torch.round(x / step.clamp(min=1e-300)), 0.0).clamp(-127, 127) * step


def _exact_attention(s):
    c = s["case"]
    out = torch.zeros_like(s["q"], dtype=torch.float64)
    g, t = c["q_heads"] // c["heads"], c["tokens"]
    for i, length in enumerate(s["positions"].tolist()):
        chain = list(range(-1, t - 1)) if s["parents"] is None else s["parents"][i].tolist()
        mask = torch.zeros((t, length + t), dtype=torch.bool)
        mask[:, :length] = True
        for r in range(t):
            j = r
            while j >= 0:
                mask[r, length + j] = True
                j = chain[j]
        mask = mask.cuda()[None]
        k, v = (s[x + "_cache"][i, :, : length + t].double() for x in ("k", "v"))
        if s["k_scale"] is not None:
            k = k * s["k_scale"][i, :, : length + t, None].double()
            v = v * s["v_scale"][i, :, : length + t, None].double()
        for j in range(g):
            q = s["q"][i, :, j::g].double().transpose(0, 1)
            z = torch.einsum("htd,hld->htl", q, k) / math.sqrt(c["dim"])
            z = z.masked_fill(~mask, -math.inf)
            out[i, :, j::g] = torch.einsum("htl,hld->thd", torch.softmax(z, -1), v)
    return out


def _exact_select(s):
    c = s["case"]
    w, v = c["beams"], c["vocab"]
    logp = torch.log_softmax(s["logits"].double(), 1).view(c["groups"], w, v)
    scores, parents, tokens, ends = [], [], [], []
    for i in range(c["groups"]):
        cand = s["scores"][i].double()[:, None] + logp[i]
        over = s["finished"][i].tolist() if c["eos"] >= 0 else [0] * w
        for j in range(w):
            if over[j]:
                cand[j] = -math.inf
                cand[j, c["eos"]] = s["scores"][i, j].double()
        best, at = cand.view(-1).sort(descending=True, stable=True)
        at = at[:w].tolist()
        scores.append(best[:w])
        parents.append([a // v for a in at])
        tokens.append([a % v for a in at])
        ends.append([int(c["eos"] >= 0 and (over[a // v] or a % v == c["eos"])) for a in at])
    whole = [torch.tensor(x, dtype=torch.int32) for x in (parents, tokens, ends)]
    return torch.stack(scores), whole[0], whole[1], whole[2]

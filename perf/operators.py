"""Performance cases: softmax attention in training and over prompts, and from a key/value cache held in 8 bits.

Kinds, each through the entry point that a program uses for it:

* ``train``: ``ops.attention`` and its backward pass: output and gradients of queries, keys and values.
* ``prompt``: ``ops.attention`` without gradients; ``prefix`` keys stand before the queries' own (a later portion of a prompt).
* ``append``: ``ops.kv8_append`` of a prompt's keys and values into the 8-bit cache, and ``ops.kv8_expand``, which gives them back
  in 16 bits (the hand-over of a session).
* ``decode``: ``ops.kv8_attention`` with new tokens: they go into the cache and attend to all of it. ``tokens`` is 1 for a decoding
  step, a few for the verification of drafted tokens, many for a later portion of a prompt.

Queries are [batch, tokens, heads, head_dim], keys and values [batch, tokens, kv_heads, head_dim], bfloat16. The cache holds blocks of
64 tokens as codes times one scale per block and head (``int8``: largest magnitude / 127; ``e4m3``: / 448) and the last 128 tokens
as they came; the block that is not full yet is read from those. Widths are those of the model presets: 6 to 30 heads of 64, 8 to 24
heads of 128, and the shared key/value heads of the dense models (16 query heads on 4).
"""

import math

import torch

own = False

BLOCK, RING = 64, 128
TOP = {"int8": 127.0, "e4m3": 448.0}
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
MOST_PAIRS = 16 * 8192.0 * 8192.0  # heads x queries x keys of the largest training case
MOST_CACHE = 32 * 8 * 8192.0 * 128  # elements of the largest cache


def _attention(kind, name, batch, tokens, heads, kv_heads, head_dim, prefix=0, window=0, ragged=False):
    return {"name": name, "kind": kind, "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim,
            "prefix": prefix, "window": window, "ragged": ragged}


def _cached(kind, name, code, batch, tokens, length, heads, kv_heads, head_dim, ragged=False):
    return {"name": name, "kind": kind, "code": code, "batch": batch, "tokens": tokens, "length": length, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "ragged": ragged}


def listed():
    return [
        # a few short rows of a fine-tuning set on a small model: the latency of the launches
        _attention("train", "train 2x37 4x64", 2, 37, 4, 4, 64),
        # a training batch of the 90M benchmark model (16 x 2048 tokens, 6 heads of 64)
        _attention("train", "train 16x2048 6x64", 16, 2048, 6, 6, 64),
        # long documents on a dense model with shared key/value heads
        _attention("train", "train 1x8192 16/4x128", 1, 8192, 16, 4, 128),
        # a padded batch of odd length, a sliding window, a head size between the tiles'
        _attention("train", "train 4x1001 12x80 window", 4, 1001, 12, 12, 80, window=300, ragged=True),
        # a later portion of a long prompt, as the generation loop sends it
        _attention("prompt", "prompt 1x1024+15360 16/4x128", 1, 1024, 16, 4, 128, prefix=15360),
        # a prompt of the serving benchmark's batch goes into the cache
        _cached("append", "append int8 4x4096 8x128", "int8", 4, 4096, 0, 16, 8, 128),
        # a short odd prompt after an earlier turn
        _cached("append", "append e4m3 1x201 4x64", "e4m3", 1, 201, 320, 4, 4, 64),
        # one request to a small model: the latency of a step
        _cached("decode", "decode int8 1x301 6x64", "int8", 1, 1, 301, 6, 6, 64),
        # a batch of requests of different lengths
        _cached("decode", "decode int8 32x8191 16/8x128", "int8", 32, 1, 8191, 16, 8, 128, ragged=True),
        # one request with a very long context
        _cached("decode", "decode e4m3 1x131000 16/4x128", "e4m3", 1, 1, 131000, 16, 4, 128),
        # drafted tokens are verified, four at a time
        _cached("decode", "verify int8 8x2047 30x64", "int8", 8, 4, 2047, 30, 30, 64, ragged=True),
        # a later portion of a prompt on the cache
        _cached("decode", "portion e4m3 1x512+7680 16/4x128", "e4m3", 1, 512, 7680, 16, 4, 128),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("train", "train", "prompt", "append", "decode", "decode", "decode"))
    head_dim = rng.choice((64, 64, 80, 128, 128))
    kv_heads = rng.choice((1, 2, 4, 6, 8))
    heads = kv_heads * rng.choice((1, 2, 3, 4))
    if kind in ("train", "prompt"):
        tokens = _between(rng, 1, 8192)
        prefix = _between(rng, 1, 16384) if kind == "prompt" else 0
        if heads * tokens * (tokens + prefix) > MOST_PAIRS:
            prefix = int(MOST_PAIRS / (heads * tokens)) - tokens
            if prefix < 0:
                prefix, tokens = 0, int(math.sqrt(MOST_PAIRS / heads))
        most = max(1, min(16, int(MOST_PAIRS / (heads * tokens * (tokens + prefix)))))
        window = rng.choice((0, 0, _between(rng, 1, 2048)))
        case = _attention(kind, "", _between(rng, 1, most), tokens, heads, kv_heads, head_dim, prefix, window, rng.random() < 0.4)
        del case["name"]
        return case
    code = rng.choice(("int8", "e4m3"))
    if kind == "append":
        length, tokens = BLOCK * _between(rng, 1, 64) - BLOCK, _between(rng, 1, 8192)
    else:
        length = _between(rng, 1, 65536)
        tokens = rng.choice((1, 1, 1, 2, 3, 5, 8, 200))
        if tokens > BLOCK:
            length = max(BLOCK, length // BLOCK * BLOCK)
    most = max(1, min(32, int(MOST_CACHE / 4 / (kv_heads * 128 * (length + tokens)))))
    batch = _between(rng, 1, most)
    case = _cached(kind, "", code, batch, tokens, length, heads, kv_heads, head_dim, kind == "decode" and tokens <= BLOCK and rng.random() < 0.5)
    del case["name"]
    return case


# ---------------------------------------------------------------------------------------------------- what a program has in hand
def _lengths(case):
    """Keys of each sequence before the call, or cached tokens: from the length given down to half of it where they are ragged."""
    n = case["tokens"] + case["prefix"] if "prefix" in case else case["length"]
    if not case["ragged"]:
        return [n] * case["batch"]
    return [max(1, n - (n // 2) * b // max(1, case["batch"] - 1)) for b in range(case["batch"])]


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(torch.bfloat16)


def _coded(x, code):
    """[..., 64 n, D] -> (codes, scales [..., n]) of the blocks of 64 rows, in 32 bits."""
    blocks = x.float().unflatten(-2, (-1, BLOCK))
    scale = blocks.abs().amax((-1, -2)) / torch.full((), TOP[code], device=x.device)
    units = blocks / torch.where(scale > 0, scale, torch.ones_like(scale))[..., None, None]
    codes = units.round().to(torch.int8) if code == "int8" else units.to(torch.float8_e4m3fn)
    return codes.flatten(-3, -2), scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    B, T, H, G, D = (case[n] for n in ("batch", "tokens", "heads", "kv_heads", "head_dim"))
    s = {"case": case, "lengths": None}
    if case["kind"] in ("train", "prompt"):
        train = case["kind"] == "train"
        s["q"] = _normal(gen, B, T, H, D).requires_grad_(train)
        s["k"] = _normal(gen, B, T + case["prefix"], G, D).requires_grad_(train)
        s["v"] = _normal(gen, B, T + case["prefix"], G, D).requires_grad_(train)
        if train:
            s["grad"] = _normal(gen, B, T, H, D)
        if case["ragged"]:
            s["lengths"] = torch.tensor(_lengths(case), device="cuda")
        return s
    # a cache that already holds the earlier tokens; a key has some channels that are larger than the others
    loud = 1.0 + 3.0 * (torch.rand(G, 1, D, generator=gen, device="cuda") > 0.95)
    pitch = 64 if D <= 64 else 128
    n, room = case["length"], -(-(case["length"] + T) // BLOCK) * BLOCK
    before = torch.tensor(_lengths(case), device="cuda")
    cache = {}
    for name, factor in (("k", loud), ("v", None)):
        x = torch.zeros(B, G, room, pitch, dtype=torch.bfloat16, device="cuda")
        y = _normal(gen, B, G, n, D)
        x[:, :, :n, :D] = y if factor is None else (y * factor).to(torch.bfloat16)
        cache[name + "8"], cache[name + "s"] = _coded(x, case["code"])
        slot = torch.arange(RING, device="cuda")
        held = before[:, None] - 1 - (before[:, None] - 1 - slot) % RING  # the newest token whose place this is
        rows = x.gather(2, held.clamp_min(0)[:, None, :, None].expand(B, G, RING, pitch))
        cache[name + "t"] = torch.where((held >= 0)[:, None, :, None], rows, torch.zeros_like(rows))
    s["cache"] = cache
    s["q"] = _normal(gen, B, T, H, D)
    s["k"] = (_normal(gen, B, T, G, D) * loud.transpose(0, 1)).to(torch.bfloat16)
    s["v"] = _normal(gen, B, T, G, D)
    s["pos"] = before if case["ragged"] else n
    return s


# ---------------------------------------------------------------------------------------------------- the plain form
def _grouped(x, G):
    """[B, T, H, D] -> [B, G, H / G, T, D] in 32 bits."""
    return x.detach().float().unflatten(2, (G, -1)).permute(0, 2, 3, 1, 4)


def _plain_attention(s):
    case, train = s["case"], "grad" in s
    G, T, S, D = case["kv_heads"], case["tokens"], case["tokens"] + case["prefix"], case["head_dim"]
    q, scale = _grouped(s["q"], G), case["head_dim"] ** -0.5
    k, v = (_grouped(s[n], G) for n in ("k", "v"))  # [B, G, 1, S, D]
    at, key = torch.arange(S - T, S, device="cuda")[:, None], torch.arange(S, device="cuda")
    seen = key <= at
    if case["window"]:
        seen = seen & (key > at - case["window"])
    seen = seen.expand(1, T, S) if s["lengths"] is None else seen & (key < s["lengths"][:, None, None])
    seen = seen[:, None, None]
    x = (q @ k.transpose(-1, -2)).mul_(scale).masked_fill_(~seen, float("-inf"))
    top = x.amax(-1, keepdim=True).clamp_min(-3e38)  # a row without a visible key: nothing is left of it
    p = x.sub_(top).exp_()
    p = p.div_(p.sum(-1, keepdim=True).clamp_min(1e-30))
    o = p @ v
    flat = lambda y: y.permute(0, 3, 1, 2, 4).flatten(2, 3).to(torch.bfloat16)  # noqa: E731
    if not train:
        return flat(o)
    g = _grouped(s["grad"], G)
    dv = (p.transpose(-1, -2) @ g).sum(2, keepdim=True)
    ds = (g @ v.transpose(-1, -2)).sub_((g * o).sum(-1, keepdim=True)).mul_(p)
    dq, dk = (ds @ k).mul_(scale), (ds.transpose(-1, -2) @ q).sum(2, keepdim=True).mul_(scale)
    return tuple(flat(y) for y in (o, dq, dk, dv))


def _plain_append(s):
    """New tokens into the cache: the ring, and the codes of the blocks that are full now."""
    case, cache, T = s["case"], s["cache"], s["case"]["tokens"]
    pos = torch.as_tensor(s["pos"], device="cuda").expand(case["batch"])
    for name in ("k", "v"):
        codes, scales, ring = cache[name + "8"], cache[name + "s"], cache[name + "t"]
        new = torch.zeros(*ring.shape[:2], T, ring.shape[3], dtype=ring.dtype, device="cuda")
        new[..., : case["head_dim"]] = s[name].transpose(1, 2)
        keep = min(T, RING)
        slot = (pos[:, None] + torch.arange(T - keep, T, device="cuda")) % RING
        ring.scatter_(2, slot[:, None, :, None].expand(-1, ring.shape[1], -1, ring.shape[3]), new[:, :, T - keep :])
        if T > BLOCK or not case["ragged"] and case["kind"] == "append":  # from the start of a block on
            full, first = T // BLOCK, s["pos"] // BLOCK
            done, scale = _coded(new[:, :, : full * BLOCK], case["code"])
            codes.view(torch.uint8)[:, :, first * BLOCK : (first + full) * BLOCK] = done.view(torch.uint8)
            scales[:, :, first : first + full] = scale
        else:  # one block at most is full now
            block = pos // BLOCK
            full = (block + 1) * BLOCK <= pos + T
            at = (block[:, None] * BLOCK + torch.arange(BLOCK, device="cuda"))[:, None, :, None].expand(-1, ring.shape[1], -1, ring.shape[3])
            done, scale = _coded(ring.gather(2, at % RING), case["code"])
            held = codes.view(torch.uint8)
            held.scatter_(2, at, torch.where(full[:, None, None, None], done.view(torch.uint8), held.gather(2, at)))
            at = block[:, None, None].expand(-1, ring.shape[1], 1)
            scales.scatter_(2, at, torch.where(full[:, None, None], scale, scales.gather(2, at)))


def _plain_values(codes, scales):
    return (codes.float().unflatten(2, (-1, BLOCK)) * scales[..., None, None]).flatten(2, 3)


def _plain_expand(s):
    case, cache = s["case"], s["cache"]
    n = case["length"] + case["tokens"]
    full, D = n // BLOCK * BLOCK, case["head_dim"]
    slot = torch.arange(full, n, device="cuda") % RING
    return [torch.cat((_plain_values(cache[x + "8"][:, :, :full], cache[x + "s"][:, :, : full // BLOCK]), cache[x + "t"][:, :, slot].float()), 2)
            [..., :D].transpose(1, 2).to(torch.bfloat16) for x in ("k", "v")]


def _plain_decode(s):
    case, cache = s["case"], s["cache"]
    B, T, G, D = (case[n] for n in ("batch", "tokens", "kv_heads", "head_dim"))
    pos = torch.as_tensor(s["pos"], device="cuda").expand(B)
    full = (pos + T) // BLOCK * BLOCK
    keys, slots = torch.arange(case["length"] + T, device="cuda"), torch.arange(RING, device="cuda")
    held = (pos + T)[:, None] - 1 - ((pos + T)[:, None] - 1 - slots) % RING  # the token in each place of the ring
    at = (pos[:, None] + torch.arange(T, device="cuda"))[:, :, None]
    seen = torch.cat((((keys < full[:, None])[:, None] & (keys <= at)), (held >= full[:, None])[:, None] & (held[:, None] <= at)), -1)[:, None, None]
    n = -(-keys.numel() // BLOCK)
    k, v = (torch.cat((_plain_values(cache[x + "8"][:, :, : n * BLOCK], cache[x + "s"][:, :, :n])[:, :, : keys.numel()], cache[x + "t"].float()), 2)
            [:, :, None, :, :D] for x in ("k", "v"))
    x = (_grouped(s["q"], G) @ k.transpose(-1, -2)).mul_(D ** -0.5).masked_fill_(~seen, float("-inf"))
    p = x.sub_(x.amax(-1, keepdim=True)).exp_()
    o = (p @ v).div_(p.sum(-1, keepdim=True))
    return o.permute(0, 3, 1, 2, 4).flatten(2, 3).to(torch.bfloat16)


def run(state):
    case, cache = state["case"], state.get("cache")
    if own:
        from triune_b200 import ops

        if cache is None:
            more = {"window": case["window"] or None, "key_lengths": state["lengths"]}
            if case["kind"] == "prompt":
                with torch.no_grad():
                    return ops.attention(state["q"], state["k"], state["v"], **more)
            inputs = (state["q"], state["k"], state["v"])
            out = ops.attention(*inputs, **more)
            return (out.detach(), *torch.autograd.grad(out, inputs, state["grad"]))
        if case["kind"] == "append":
            ops.kv8_append(cache, state["k"], state["v"], state["pos"])
            out = ops.kv8_expand(cache, case["length"] + case["tokens"], case["head_dim"])
        else:
            out = ops.kv8_attention(state["q"], cache, state["pos"], state["k"], state["v"])
    elif cache is None:
        return _plain_attention(state)
    else:
        _plain_append(state)
        out = _plain_expand(state) if case["kind"] == "append" else _plain_decode(state)
    if case["kind"] == "append":  # the scales of the blocks that are full
        full = (case["length"] + case["tokens"]) // BLOCK
        return (*out, cache["ks"][:, :, :full], cache["vs"][:, :, :full])
    return out, cache["kt"], cache["vt"]


# ---------------------------------------------------------------------------------------------------- what a pass cannot do without
def _pairs(case):
    """(query, key) pairs of one head that see each other, over the batch."""
    T = case["tokens"]
    if "prefix" not in case:
        return sum(T * n + T * (T + 1) // 2 for n in _lengths(case))
    total, first = 0, case["prefix"]
    for n in _lengths(case):
        at = torch.arange(first, first + T)
        low = (at - case["window"] + 1).clamp_min(0) if case["window"] else torch.zeros_like(at)
        total += int((torch.minimum(at + 1, torch.tensor(n)) - low).clamp_min(0).sum())
    return total


def work(case):
    B, T, H, G, D = (case[n] for n in ("batch", "tokens", "heads", "kv_heads", "head_dim"))
    pairs = _pairs(case)
    if case["kind"] in ("train", "prompt"):
        S = T + case["prefix"]
        rows, keys = 2 * B * T * H * D, 2 * B * S * G * D
        if case["kind"] == "prompt":
            return {"bytes": 2 * rows + 2 * keys, "flops": 4 * D * H * pairs}
        return {"bytes": 2 * (2 * rows + 2 * keys), "flops": 14 * D * H * pairs}
    n = case["length"] + T
    if case["kind"] == "append":  # 16 bits in, codes and scales out, codes in, 16 bits out
        tokens = 2 * B * G * D
        return {"bytes": tokens * (2 * T + T + n + 2 * n) + 16 * B * G * (n // BLOCK), "flops": tokens * (2 * T + n)}
    cached = sum(2 * G * D * m + 8 * G * (m // BLOCK) for m in _lengths(case))
    return {"bytes": cached + 4 * B * T * H * D + 4 * B * T * G * D * 2, "flops": 4 * D * H * pairs}


# ---------------------------------------------------------------------------------------------------- the definition, in 64 bits
def _softmax_rows(q, k, seen, scale):
    """Probabilities [rows, keys] of one head; rows without a visible key are zero."""
    x = torch.where(seen, scale * (q @ k.T), torch.full((), -math.inf, device=q.device, dtype=q.dtype))
    p = torch.exp(x - torch.nan_to_num(x.max(-1, keepdim=True).values, neginf=0.0))
    return p / p.sum(-1, keepdim=True).clamp_min(1e-300)


def _exact_attention(s):
    case = s["case"]
    B, T, H, G, D = (case[n] for n in ("batch", "tokens", "heads", "kv_heads", "head_dim"))
    S, rep, scale = T + case["prefix"], H // G, D ** -0.5
    q, k, v = (s[n].detach().double() for n in ("q", "k", "v"))
    o, dq = torch.zeros_like(q), torch.zeros_like(q)
    dk, dv = torch.zeros_like(k), torch.zeros_like(v)
    lengths, keys = _lengths(case), torch.arange(S, device="cuda")
    for b in range(B):
        for h in range(H):
            g = h // rep
            for t0 in range(0, T, 4096):
                t = slice(t0, min(T, t0 + 4096))
                i = torch.arange(case["prefix"] + t.start, case["prefix"] + t.stop, device="cuda")[:, None]
                seen = (keys <= i) & (keys < lengths[b])
                if case["window"]:
                    seen &= i - keys < case["window"]
                p = _softmax_rows(q[b, t, h], k[b, :, g], seen, scale)
                o[b, t, h] = p @ v[b, :, g]
                if "grad" in s:
                    do = s["grad"][b, t, h].double()
                    dv[b, :, g] += p.T @ do
                    dp = do @ v[b, :, g].T
                    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
                    dq[b, t, h] = ds @ k[b, :, g]
                    dk[b, :, g] += ds.T @ q[b, t, h]
    return (o, dq, dk, dv) if "grad" in s else o


def _exact_cache(s, name):
    """(values [B, G, n, D] as the cache gives them after the call, scales of its full blocks, ring)."""
    case, cache, new = s["case"], s["cache"], s[name].double().transpose(1, 2)
    B, T, D, top = case["batch"], case["tokens"], case["head_dim"], TOP[case["code"]]
    n = case["length"] + T
    ring = cache[name + "t"].double()
    values = torch.zeros(*ring.shape[:2], n, D, device="cuda", dtype=torch.float64)
    scales = torch.zeros(*ring.shape[:2], n // BLOCK, device="cuda", dtype=torch.float64)
    for b, before in enumerate(_lengths(case)):
        old, full = before // BLOCK, (before + T) // BLOCK
        raw = torch.cat((ring[b][:, torch.arange(old * BLOCK, before, device="cuda") % RING, :D], new[b]), 1)  # from the open block on
        for i in range(T):
            ring[b, :, (before + i) % RING, :D] = new[b, :, i]
        held = cache[name + "8"][b, :, : old * BLOCK, :D].double()
        scale = cache[name + "s"][b, :, :old].double()
        values[b, :, : old * BLOCK] = held * scale.repeat_interleave(BLOCK, -1)[..., None]
        values[b, :, old * BLOCK : before + T] = raw
        scales[b, :, :old] = scale
        for m in range(old, full):
            x = raw[:, (m - old) * BLOCK : (m - old + 1) * BLOCK]
            unit = x.abs().amax((1, 2)) / top
            y = x / unit.clamp_min(1e-300)[:, None, None]
            y = y.round() if case["code"] == "int8" else y.float().to(torch.float8_e4m3fn).double()
            values[b, :, m * BLOCK : (m + 1) * BLOCK] = y * unit[:, None, None]
            scales[b, :, m] = unit
    return values, scales, ring


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("train", "prompt"):
        return _exact_attention(s)
    (k, ks, kt), (v, vs, vt) = _exact_cache(s, "k"), _exact_cache(s, "v")
    if case["kind"] == "append":
        return k.transpose(1, 2), v.transpose(1, 2), ks, vs
    B, T, H, G, D = (case[n] for n in ("batch", "tokens", "heads", "kv_heads", "head_dim"))
    o = torch.zeros(B, T, H, D, device="cuda", dtype=torch.float64)
    for b, before in enumerate(_lengths(case)):
        seen = torch.arange(before + T, device="cuda") <= before + torch.arange(T, device="cuda")[:, None]
        for h in range(H):
            g = h // (H // G)
            o[b, :, h] = _softmax_rows(s["q"][b, :, h].double(), k[b, g, : before + T], seen, D ** -0.5) @ v[b, g, : before + T]
    return o, kt, vt

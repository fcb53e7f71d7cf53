"""Softmax attention and the 8-bit cache in 64 bits, written from the definitions, with bounds of what rounding may do to results."""

import torch

STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}  # half a step of a type, relative to the value
BLOCK, RING = 64, 128


def visible(T, S, causal, window, length, start, device="cpu"):
    at, key = torch.arange(start, start + T, device=device)[:, None], torch.arange(S, device=device)
    see = (key < length).expand(T, S)
    if causal:
        see = see & (key <= at)
    if window:
        see = see & (at - key < window)
    return see


def attention64(q, k, v, causal=True, window=None, lengths=None, starts=None, scale=None, grad=None):
    """-> {"o": (value, bound), and with ``grad`` "dq", "dk", "dv"}. Bounds: weights and dS rounded to bf16 (2^-8 of each), results rounded to
    the queries' type, o rounded before it enters delta; 3e-5 of the sums' magnitudes for fp32 arithmetic (scores of up to 30
    times log2(e), off by a few 2^-24 of themselves, exponentials, sums of a few thousand terms)."""
    B, T, H, D = q.shape
    S, G = k.shape[1], k.shape[2]
    step, slack = STEP[torch.bfloat16], 3e-5
    scale = D ** -0.5 if scale is None else scale
    x = {n: t.detach().double() for n, t in (("q", q), ("k", k), ("v", v))}
    g = None if grad is None else grad.double()
    like = {"o": x["q"], "dq": x["q"], "dk": x["k"], "dv": x["v"]}
    out = {n: [torch.zeros_like(t), torch.zeros_like(t)] for n, t in like.items() if n == "o" or g is not None}
    for b in range(B):
        see = visible(T, S, causal, window, S if lengths is None else int(lengths[b]), S - T if starts is None else int(starts[b]), q.device)
        some = see.any(-1, keepdim=True)
        for h in range(H):
            r = h // (H // G)
            Q, K, V = x["q"][b, :, h], x["k"][b, :, r], x["v"][b, :, r]
            s = (scale * Q @ K.T).masked_fill(~see, float("-inf"))
            p = torch.where(some, torch.softmax(torch.where(some, s, torch.zeros_like(s)), -1), torch.zeros_like(s))
            o = p @ V
            off = (step + slack) * (o.abs() + p @ V.abs())
            out["o"][0][b, :, h], out["o"][1][b, :, h] = o, off
            if g is None:
                continue
            dO = g[b, :, h]
            dP, delta = dO @ V.T, (dO * o).sum(-1, keepdim=True)
            ds = p * (dP - delta)
            d_off = (dO.abs() * off).sum(-1, keepdim=True)  # of delta, by the rounding of o
            loose = p * slack * (dO.abs() @ V.abs().T + (dO * o).abs().sum(-1, keepdim=True))  # fp32 sums of dP and delta
            s_off = step * ds.abs() + p * d_off + loose + slack * ds.abs()
            for n, value, bound in (("dq", scale * ds @ K, scale * s_off @ K.abs()), ("dk", scale * ds.T @ Q, scale * s_off.T @ Q.abs()),
                                    ("dv", p.T @ dO, (step + slack) * (p.T @ dO.abs()))):
                at = (b, slice(None), h if n == "dq" else r)
                out[n][0][at] += value
                out[n][1][at] += bound
    for n in out:
        if n != "o":
            out[n][1] += step * (out[n][0].abs() + out[n][1])
    return {n: tuple(y) for n, y in out.items()}


def near(got, want, what=""):
    value, bound = want
    off = (got.double() - value).abs()
    worst = (off - bound).max() if off.numel() else torch.zeros(())
    assert torch.isfinite(got).all() and bool((off <= bound + 1e-30).all()), f"{what}: {float(worst):.3g} past its bound, off by {float(off.max()):.3g}"


def coded64(x, kind):
    """[..., 64, D] bf16 -> (values, scales) of blocks with one scale, as fp32 forms them: the scale is max|x| / 127 (/ 448) rounded
    to fp32, a code the nearest one (ties to even) to the fp32 quotient."""
    x = x.double()
    top = 127.0 if kind == "int8" else 448.0
    scale = (x.abs().amax((-1, -2)) / top).float().double()
    y = (x / scale.masked_fill(scale == 0, 1.0)[..., None, None]).float()  # both are fp32 numbers: one rounding, as of a division in fp32
    y = (y.round() if kind == "int8" else y.to(torch.float8_e4m3fn).float()).double()
    return y * scale[..., None, None], scale


def cache64(tokens, kind, n):
    """Tokens [G, >= n, D] (bf16) of one sequence -> [G, n, D]: the values that a cache of n of them stands for."""
    full = n // BLOCK * BLOCK
    held = tokens[:, :n].double().clone()
    if full:
        held[:, :full] = coded64(tokens[:, :full].unflatten(1, (-1, BLOCK)), kind)[0].flatten(1, 2)
    return held


def kv8_attention64(q, k, v, kind, pos, scale=None):
    """q [T, H, D] at pos .., k, v [G, >= pos + T, D] of one sequence -> (value, bound): results rounded to bf16, weights to fp16 (2^-11 of
    each, and 2^-24 of the largest value where they are small), 3e-5 of the sums for fp32 arithmetic."""
    T, H, D = q.shape
    G, n = k.shape[0], pos + T
    K, V = cache64(k, kind, n), cache64(v, kind, n)
    see = torch.arange(n, device=q.device) <= torch.arange(pos, n, device=q.device)[:, None]
    value, bound = (torch.zeros(T, H, D, dtype=torch.float64, device=q.device) for _ in "ab")
    for h in range(H):
        g = h // (H // G)
        s = (D ** -0.5 if scale is None else scale) * q[:, h].double() @ K[g].T
        p = torch.softmax(s.masked_fill(~see, float("-inf")), -1)
        o = p @ V[g]
        value[:, h] = o
        small = (2.0 ** -24 / p.amax(-1, keepdim=True).clamp_min(1e-30)).clamp_max(1.0) * p.amax(-1, keepdim=True) * V[g].abs().sum(0)
        bound[:, h] = STEP[torch.bfloat16] * o.abs() + (1 + STEP[torch.bfloat16]) * ((2.0 ** -11 + 3e-5) * (p @ V[g].abs()) + small)
    return value, bound

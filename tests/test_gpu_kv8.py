"""The 8-bit key/value cache and attention from it, on the GPU, against the definition in 64 bits."""

import pytest
import torch

from attention_cases import BLOCK, RING, attention64, cache64, coded64, kv8_attention64, near
from triune_b200 import ops
from triune_b200.ops import reference

pytestmark = pytest.mark.gpu
KINDS = ["int8", "e4m3"]


def rows(B, T, G, D, seed=0, loud=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(B, T, G, D, generator=gen, device="cuda")
    if loud:
        x[..., 3] *= 9.0  # a channel that is larger than the others
    return x.bfloat16()


def filled(B, G, D, n, kind, seed=0, capacity=None, chunk=None):
    """-> (cache of n tokens, keys and values [B, n, G, D])"""
    cache = ops.kv8_cache(B, G, capacity or n, D, kind, device="cuda")
    k, v = rows(B, n, G, D, seed), rows(B, n, G, D, seed + 1, False)
    chunk = chunk or n
    for p in range(0, n, max(1, chunk)):
        ops.kv8_append(cache, k[:, p : p + chunk], v[:, p : p + chunk], p)
    return cache, k, v


def bits(cache):
    return {n: t.view(torch.uint8) for n, t in cache.items()}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 63, 64, 65, 128, 200, 1000])
@pytest.mark.parametrize("G,D", [(1, 64), (3, 128), (2, 8), (2, 80)])
def test_what_the_cache_holds(kind, n, G, D):
    cache, k, v = filled(2, G, D, n, kind)
    full = n // BLOCK
    got = ops.kv8_expand(cache, n, D)
    for x, y, name in zip(got, (k, v), ("k", "v")):
        for b in range(2):
            held = cache64(y[b].transpose(0, 1), kind, n)  # codes times scale in fp32, rounded to bf16: twice on the way
            assert torch.equal(x[b].transpose(0, 1), held.float().bfloat16())
            scale = coded64(y[b, : full * BLOCK].transpose(0, 1).unflatten(1, (full, BLOCK)), kind)[1] if full else cache[name + "s"][b, :, :0]
            assert torch.equal(cache[name + "s"][b, :, :full].double(), scale.double())
        slots = torch.arange(max(0, n - RING), n, device="cuda")
        assert torch.equal(cache[name + "t"][:, :, slots % RING, :D].transpose(1, 2), y[:, slots])
        assert not cache[name + "t"][..., D:].any() and not cache[name + "8"].view(torch.uint8)[..., D:].any()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128])
def test_contents_do_not_depend_on_the_portions(kind, D):
    n = 500
    whole, k, v = filled(2, 2, D, n, kind)
    for chunk in (1, 7, 64, 65, 100, 190, 333):
        assert all(torch.equal(a, bits(whole)[x]) for x, a in bits(filled(2, 2, D, n, kind, chunk=chunk)[0]).items()), chunk
    # up to 64 tokens are taken back and others come in their place
    for back in (1, 30, 64):
        new_k, new_v = rows(2, back + 40, 2, D, 77), rows(2, back + 40, 2, D, 78)
        cache = filled(2, 2, D, n, kind, capacity=640)[0]
        ops.kv8_append(cache, new_k, new_v, n - back)
        k2, v2 = torch.cat((k[:, : n - back], new_k), 1), torch.cat((v[:, : n - back], new_v), 1)
        fresh = ops.kv8_cache(2, 2, 640, D, kind, device="cuda")
        ops.kv8_append(fresh, k2, v2, 0)
        m = k2.shape[1]
        assert all(torch.equal(a, b) for a, b in zip(ops.kv8_expand(cache, m, D), ops.kv8_expand(fresh, m, D)))
        assert torch.equal(cache["kt"], fresh["kt"])


def attend(B, G, rep, D, T, starts, kind, seed=0, chunk=None, on_device=True, append=True):
    """Decodes T tokens per sequence after ``starts`` ones, together, and compares every sequence."""
    longest = max(max(starts), 0) + T
    cache, k, v = filled(B, G, D, longest, kind, seed, capacity=longest + 70)
    for b, n in enumerate(starts):  # each sequence as it was before its new tokens
        if n >= 0:
            one = ops.kv8_cache(1, G, longest + 70, D, kind, device="cuda")
            if n:
                ops.kv8_append(one, k[b : b + 1, :n], v[b : b + 1, :n], 0)
            for x in cache:
                cache[x].view(torch.uint8)[b] = one[x].view(torch.uint8)[0]
    pos = torch.tensor(starts, device="cuda") if on_device else starts[0]
    q = rows(B, T, G * rep, D, seed + 5, False)
    at = lambda x: torch.stack([x[b, max(n, 0) : max(n, 0) + T] for b, n in enumerate(starts)])  # noqa: E731
    if append:
        out = ops.kv8_attention(q, cache, pos, at(k), at(v))
    else:
        ops.kv8_append(cache, at(k), at(v), pos)
        out = ops.kv8_attention(q, cache, pos)
    for b, n in enumerate(starts):
        if n < 0:
            assert not out[b].any()
            continue
        near(out[b], kv8_attention64(q[b], k[b].transpose(0, 1), v[b].transpose(0, 1), kind, n), f"sequence {b}")
    return out


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [8, 64, 72, 128])
@pytest.mark.parametrize("T,rep", [(1, 1), (1, 4), (1, 8), (4, 1), (3, 5), (9, 2), (20, 3)])
def test_steps_and_drafted_tokens(kind, D, T, rep):
    attend(5, 2, rep, D, T, [0, 1, 63, 200, 517], kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [5000, 40000])
def test_long_caches(kind, n):
    attend(1, 2, 4, 128, 1, [n], kind, on_device=False)
    attend(2, 1, 2, 64, 2, [n, 3], kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [64, 100, 300])
def test_portions_of_prompts(kind, T):
    """Many queries at once go over codes on the tensor cores: weights, times a block's scale, are rounded to bf16 (2^-8 of each) there."""
    for on_device, starts in ((False, [130]), (True, [0, 130, -1, 77])):
        B, G, rep, D = len(starts), 2, 2, 64
        longest = max(starts) + T
        cache, k, v = filled(B, G, D, longest, kind, capacity=longest)
        q = rows(B, T, G * rep, D, 5, False) * 0.25
        pos = torch.tensor(starts, device="cuda") if on_device else starts[0]
        at = lambda x: torch.stack([x[b, max(n, 0) : max(n, 0) + T] for b, n in enumerate(starts)])  # noqa: E731
        for b, n in enumerate(starts):
            one = ops.kv8_cache(1, G, longest, D, kind, device="cuda")
            ops.kv8_append(one, k[b : b + 1, : max(n, 0)], v[b : b + 1, : max(n, 0)], 0)
            for x in cache:
                cache[x].view(torch.uint8)[b] = one[x].view(torch.uint8)[0]
        out = ops.kv8_attention(q, cache, pos, at(k), at(v))
        for b, n in enumerate(starts):
            if n < 0:
                assert not out[b].any()
                continue
            K, V = (cache64(x[b].transpose(0, 1), kind, n + T).transpose(0, 1)[None] for x in (k, v))
            near(out[b : b + 1], attention64(q[b : b + 1], K, V)["o"], f"sequence {b}")


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [40, 64, 72, 128])
@pytest.mark.parametrize("starts", [[0, 130, -1, 77, 400, 63, 64, 65, 1, 250], [300]])
def test_portions_of_many_sequences_and_of_one(kind, D, starts):
    """More tiles of queries than SMs, and fewer (keys are split then); sums over the blocks as above."""
    B, G, rep, T = len(starts), 4, 4, 130
    longest = max(starts) + T
    _, k, v = filled(B, G, D, longest, kind)
    cache = ops.kv8_cache(B, G, longest + 40, D, kind, device="cuda")
    for b, n in enumerate(starts):
        one = ops.kv8_cache(1, G, longest + 40, D, kind, device="cuda")
        ops.kv8_append(one, k[b : b + 1, : max(n, 0)], v[b : b + 1, : max(n, 0)], 0)
        for x in cache:
            cache[x].view(torch.uint8)[b] = one[x].view(torch.uint8)[0]
    q = rows(B, T, G * rep, D, 5, False) * 0.25
    at = lambda x: torch.stack([x[b, max(n, 0) : max(n, 0) + T] for b, n in enumerate(starts)])  # noqa: E731
    out = ops.kv8_attention(q, cache, torch.tensor(starts, device="cuda"), at(k), at(v))
    for b, n in enumerate(starts):
        if n < 0:
            assert not out[b].any()
            continue
        K, V = (cache64(x[b].transpose(0, 1), kind, n + T).transpose(0, 1)[None] for x in (k, v))
        near(out[b : b + 1], attention64(q[b : b + 1], K, V)["o"], f"sequence {b}")


def test_appending_first_is_the_same_and_scale_and_bound_are_the_callers():
    a = attend(3, 2, 2, 64, 3, [10, 61, 300], "int8")
    assert torch.equal(a, attend(3, 2, 2, 64, 3, [10, 61, 300], "int8", append=False))
    cache, k, v = filled(1, 2, 64, 3000, "int8", capacity=4096)
    q = rows(1, 1, 4, 64, 3, False)
    for most in (None, 3000, 100000):
        out = ops.kv8_attention(q, cache, torch.tensor([2999], device="cuda"), scale=0.3, most=most)
        near(out[0], kv8_attention64(q[0], k[0].transpose(0, 1), v[0].transpose(0, 1), "int8", 2999, 0.3))


def test_queries_of_any_size_and_keys_far_from_one():
    for factor in (1e-30, 1e-5, 3e4, 1e15):
        cache = ops.kv8_cache(1, 1, 300, 64, "int8", device="cuda")
        k, v = rows(1, 200, 1, 64, 1, False), rows(1, 200, 1, 64, 2, False)
        k, v = (k.float() / factor).bfloat16(), (v.float() * factor).bfloat16()
        q = (rows(1, 1, 2, 64, 3, False).float() * factor).bfloat16()
        ops.kv8_append(cache, k, v, 0)
        out = ops.kv8_attention(q, cache, 199)
        near(out[0], kv8_attention64(q[0], k[0].transpose(0, 1), v[0].transpose(0, 1), "int8", 199))


def test_blocks_whose_scales_differ_and_blocks_of_zeros():
    cache = ops.kv8_cache(1, 1, 400, 64, "int8", device="cuda")
    k, v = rows(1, 330, 1, 64, 1, False), rows(1, 330, 1, 64, 2, False)
    for m, f in enumerate((0.0, 1e-6, 1.0, 1e6, 0.0)):
        v[:, 64 * m : 64 * m + 64] *= f
    k[:, 64:128] = 0
    ops.kv8_append(cache, k, v, 0)
    q = rows(1, 1, 3, 64, 3, False)
    near(ops.kv8_attention(q, cache, 329)[0], kv8_attention64(q[0], k[0].transpose(0, 1), v[0].transpose(0, 1), "int8", 329))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("exponent", [0, 1, 4, 9, 127, 200, 254])  # of the largest number of a block, from subnormal ones on
def test_codes_of_every_number_at_every_scale(kind, exponent):
    """A block for each of the 128 fractions of its largest number; the others are numbers of all kinds not above it."""
    gen = torch.Generator(device="cuda").manual_seed(exponent)
    top = torch.arange(128, device="cuda") + 128 * exponent
    x = (torch.rand(1, 128, BLOCK * 128, generator=gen, device="cuda") * 26 * 128).long()  # bf16 numbers' bits, 26 powers of two of them
    x = (top[None, :, None] - x).clamp(min=0)
    x[..., 0] = top
    x = x | (torch.rand(x.shape, generator=gen, device="cuda") < 0.5).long() << 15
    x = x.int().short().view(torch.bfloat16).view(1, 128 * BLOCK, 1, 128)
    cache = ops.kv8_cache(1, 1, x.shape[1], 128, kind, device="cuda")
    ops.kv8_append(cache, x, -x, 0)
    blocks = x.view(128, BLOCK, 128)
    codes, scale = reference.kv8_codes(blocks, cache["k8"].dtype)
    assert torch.equal(cache["ks"].flatten(), scale.flatten()) and torch.equal(cache["vs"].flatten(), scale.flatten())
    assert torch.equal(bits(cache)["k8"].view(-1), codes.view(torch.uint8).view(-1))
    assert torch.equal(bits(cache)["v8"].view(-1), reference.kv8_codes(-blocks, cache["k8"].dtype)[0].view(torch.uint8).view(-1))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [1, 5, 100])
def test_idle_sequences_and_tokens_past_the_capacity_leave_the_rest_alone(kind, T):
    B, G, D, C = 3, 2, 64, 128
    cache, k, v = filled(B, G, D, 100, kind, capacity=C)
    before = {n: t.clone() for n, t in bits(cache).items()}
    q, nk, nv = rows(B, T, 4, D, 3, False), rows(B, T, G, D, 4), rows(B, T, G, D, 5)
    out = ops.kv8_attention(q, cache, torch.tensor([-1, C, -5], device="cuda"), nk, nv)
    assert all(torch.equal(before[n], t) for n, t in bits(cache).items())
    assert not out[0].any() and not out[2].any() and bool(torch.isnan(out[1]).all())
    out = ops.kv8_attention(q, cache, torch.tensor([100, C - 2, -1], device="cuda"), nk, nv)
    assert bool(torch.isnan(out[1, 2:]).all()) and not torch.isnan(out[1, :2]).any() and not torch.isnan(out[0, : C - 100]).any()
    assert all(torch.equal(before[n][2], t[2]) for n, t in bits(cache).items())


@pytest.mark.parametrize("T", [1, 5, 100])
def test_idle_by_a_number_and_bounds_beyond_what_is_held(T):
    cache, k, v = filled(2, 2, 64, 100, "int8", capacity=512)
    before = {n: t.clone() for n, t in bits(cache).items()}
    q, nk, nv = rows(2, T, 4, 64, 3, False), rows(2, T, 2, 64, 4), rows(2, T, 2, 64, 5)
    assert not ops.kv8_attention(q, cache, -3, nk, nv).any() and all(torch.equal(before[n], t) for n, t in bits(cache).items())
    pad = torch.zeros(2, T, 4, 136, device="cuda", dtype=torch.bfloat16)  # rows whose addresses are no multiples of 16 bytes: copied
    copies = [pad[:, :, : x.shape[2], 3:67].copy_(x) for x in (nk,)] + [nv.clone()]
    out = ops.kv8_attention(q, {n: t.clone() for n, t in cache.items()}, 100, *copies, most=512)
    assert torch.equal(out, ops.kv8_attention(q, cache, 100, nk, nv))


@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_tokens_that_are_no_numbers(what):
    for T in (4, 100):
        cache, k, v = filled(1, 1, 64, 70, "int8", capacity=256)
        q, nk, nv = rows(1, T, 2, 64, 3, False), rows(1, T, 1, 64, 4), rows(1, T, 1, 64, 5)
        clean = ops.kv8_attention(q, {n: t.clone() for n, t in cache.items()}, 70, nk, nv)
        nv[0, 2, 0, 7] = what
        out = ops.kv8_attention(q, cache, 70, nk, nv)
        assert torch.equal(out[:, :2], clean[:, :2]) if T == 4 else True  # 70 + 100 fill the block, which reads as NaN throughout
        assert bool(torch.isnan(out[:, 2:, :, 7]).all()) or what == float("inf") and not torch.isfinite(out[:, 2:, :, 7]).any()
    cache, k, v = filled(1, 1, 64, 200, "int8")
    assert torch.isfinite(ops.kv8_attention(q[:, :1], cache, 199)).all()
    v[0, 70, 0, 1] = what
    ops.kv8_append(cache, k, v, 0)
    got = ops.kv8_expand(cache, 200, 64)[1][0, :, 0]
    assert bool(torch.isnan(got[64:128]).all()) and torch.isfinite(got[:64]).all() and torch.isfinite(got[128:]).all()
    assert bool(torch.isnan(ops.kv8_attention(q[:, :1], cache, 199)).all())


def test_offsets_past_32_bits():
    """5 sequences of 2^17 tokens, 32 heads of 128: codes of 2.7 GB, the last of them past 2^31."""
    B, G, D, C = 5, 32, 128, 1 << 17
    cache = ops.kv8_cache(B, G, C, D, "int8", device="cuda")
    assert cache["k8"].numel() > 2 ** 31
    k, v = rows(B, 200, G, D, 1), rows(B, 200, G, D, 2, False)
    pos = torch.tensor([-1, -1, -1, -1, C - 200], device="cuda")
    ops.kv8_append(cache, k, v, pos)  # block by block: C - 200 is 56 past a block's start, so this block holds older (zero) tokens too
    full = torch.zeros(G, C, D, device="cuda", dtype=torch.bfloat16)
    full[:, C - 200 :] = v[4].transpose(0, 1)
    got = ops.kv8_expand(cache, torch.tensor([0, 0, 0, 0, C], device="cuda"), D)[1]
    assert torch.equal(got[4, C - 256 :].transpose(0, 1), cache64(full[:, C - 256 :], "int8", 256).float().bfloat16())
    q = rows(B, 1, G, D, 3, False)
    out = ops.kv8_attention(q, cache, torch.tensor([-1, -1, -1, -1, C - 1], device="cuda"))
    keys = torch.zeros(1, C, D, device="cuda", dtype=torch.bfloat16)
    keys[:, C - 200 :] = k[4, :, 31:].transpose(0, 1)
    near(out[4, :, 31:], kv8_attention64(q[4, :, 31:], keys, full[31:], "int8", C - 1))


@pytest.mark.parametrize("T", [1, 3, 80])
def test_captured_steps_follow_positions_on_the_device(T):
    B, G, D = 2, 2, 64
    n, steps = 100, 6
    k, v, q = (rows(B, n + T * steps, h, D, s, False) for h, s in ((G, 1), (G, 2), (4, 3)))

    def fresh():
        cache = ops.kv8_cache(B, G, n + T * steps, D, "e4m3", device="cuda")
        ops.kv8_append(cache, k[:, :n], v[:, :n], 0)
        return cache

    want, cache = [], fresh()
    for i in range(steps):
        at = slice(n + T * i, n + T * i + T)
        want.append(ops.kv8_attention(q[:, at], cache, torch.tensor([n + T * i], device="cuda"), k[:, at], v[:, at]))
    caches = [fresh(), fresh()]
    graphs = []
    for c in caches:  # two captures, replayed in turn
        pos = torch.tensor([n, n], device="cuda")
        at = [x[:, n : n + T].clone() for x in (q, k, v)]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.kv8_attention(at[0], c, pos, at[1], at[2])
            pos += T
        pos.fill_(n)
        graphs.append((g, at, out, pos))  # the captured steps read and move the positions
    for i in range(steps):
        for g, at, out, _ in graphs:
            for x, y in zip(at, (q, k, v)):
                x.copy_(y[:, n + T * i : n + T * i + T])
            g.replay()
            assert torch.equal(out, want[i])
    assert all(torch.equal(a, bits(caches[0])[x]) for x, a in bits(cache).items())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [128, 300])
@pytest.mark.parametrize("starts", [[0], [64, 130, -1, 0]])
@pytest.mark.parametrize("what", [float("nan"), -float("inf")])
def test_queries_before_a_block_that_reads_as_none_do_not_see_it(kind, D, T, starts, what):
    """A token of the portion is no number, and so its whole block once it is full. Queries before the block (before the token, where
    the block is open) are, bit for bit, what they are without it; the others are no numbers in all columns of a full block."""
    B, G, rep, longest = len(starts), 2, 2, max(starts) + T
    _, k, v = filled(B, G, D, longest, kind)
    q = rows(B, T, G * rep, D, 5, False) * 0.25
    at = lambda x: torch.stack([x[b, max(n, 0) : max(n, 0) + T] for b, n in enumerate(starts)])  # noqa: E731

    def call(new_k, new_v, on_device):
        cache = ops.kv8_cache(B, G, longest, D, kind, device="cuda")
        for b, n in enumerate(starts):  # each sequence as it was before its new tokens
            one = ops.kv8_cache(1, G, longest, D, kind, device="cuda")
            ops.kv8_append(one, k[b : b + 1, : max(n, 0)], v[b : b + 1, : max(n, 0)], 0)
            for x in cache:
                cache[x].view(torch.uint8)[b] = one[x].view(torch.uint8)[0]
        return ops.kv8_attention(q, cache, torch.tensor(starts, device="cuda") if on_device else starts[0], new_k, new_v)

    for on_device in (True, False)[: 1 + (B == 1)]:
        clean = call(at(k), at(v), on_device)
        for side in range(2):
            for token in (T // 2 + 36, T - 1):
                new = [at(k), at(v)]
                new[side][:, token, :, 7] = what
                out = call(*new, on_device)
                for b, n in enumerate(starts):
                    if n < 0:
                        assert not out[b].any()
                        continue
                    block = (n + token) // BLOCK * BLOCK
                    full = block + BLOCK <= n + T
                    first = max(0, block - n) if full else token
                    assert torch.equal(out[b, :first], clean[b, :first]), (b, side, token)
                    if full:
                        assert bool(torch.isnan(out[b, first:]).all())
                    elif side:
                        assert not torch.isfinite(out[b, first:, :, 7]).any()


def by_contributions(q, k, v, kind, pos):
    """As ``kv8_attention64``, but weights that are small are off by what half a step of fp16's smallest is next to the largest
    CONTRIBUTION (weight times the block's scale): a power of two of at most twice that is the unit of the weights times scales,
    which are rounded to fp16, 2^-25 at most below 2^-14."""
    T, H, D = q.shape
    G, n = k.shape[0], pos + T
    full = n // BLOCK
    K, V = cache64(k, kind, n), cache64(v, kind, n)
    value, bound = (torch.zeros(T, H, D, dtype=torch.float64, device=q.device) for _ in "ab")
    see = torch.arange(n, device=q.device) <= torch.arange(pos, n, device=q.device)[:, None]
    for h in range(H):
        g = h // (H // G)
        scale = coded64(v[g, : full * BLOCK].unflatten(0, (full, BLOCK)), kind)[1].repeat_interleave(BLOCK)
        p = torch.softmax((D ** -0.5 * q[:, h].double() @ K[g].T).masked_fill(~see, float("-inf")), -1)
        value[:, h] = p @ V[g]
        codes = (V[g, : full * BLOCK] / scale.masked_fill(scale == 0, 1.0)[:, None]).abs().sum(0)
        largest = (p[:, : full * BLOCK] * scale).amax(-1, keepdim=True)
        off = (2.0 ** -11 + 3e-5) * (p @ V[g].abs()) + 2.0 ** -24 * largest * codes
        bound[:, h] = 2.0 ** -8 * value[:, h].abs() + (1 + 2.0 ** -8) * off
    return value, bound


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D,T,n", [(64, 1, 2047), (128, 1, 2060), (64, 4, 2100), (128, 12, 20000)])
@pytest.mark.parametrize("factor", [1e3, 1e5, 1e8, 1e20, 1e34])
def test_a_loud_block_that_hardly_counts_leaves_the_others_their_digits(kind, D, T, n, factor):
    """Values of one block are larger by a factor than all others, and its scores lower by so much that its weight next to nothing is: what the
    other blocks give has its digits all the same. With the largest factor it outweighs them, and they are what is lost."""
    B, G, H = 1, 1, 2
    q, k, v = rows(B, T, H, D, 3, False), rows(B, n + T, G, D, 1, False), rows(B, n + T, G, D, 2, False)
    q[:] = q[:, :1, :1]  # one direction, which the loud keys point away from
    loud = slice(BLOCK * 5, BLOCK * 6)
    x = q[0, 0, 0].float()
    k[0, loud, 0] = (-60 * D ** 0.5 * x / (x @ x)).bfloat16()
    v[0, loud] = (v[0, loud].float() * factor).bfloat16()
    cache = ops.kv8_cache(B, G, n + T, D, kind, device="cuda")
    ops.kv8_append(cache, k[:, :n], v[:, :n], 0)
    out = ops.kv8_attention(q, cache, n, k[:, n:], v[:, n:])
    near(out[0], by_contributions(q[0], k[0].transpose(0, 1), v[0].transpose(0, 1), kind, n))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("order", [(1e-36, 1.0, 1e30, 0.0, 1e-20), (1e30, 1e-36, 0.0, 1.0, 1e-38), (0.0, 0.0, 1e-38, 1e-39, 0.0), (1e36, 1e-30, 1e36, 0.0, 1e-36)])
def test_scales_from_the_smallest_to_the_largest(kind, order):
    q, k, v = rows(1, 1, 3, 64, 3, False), rows(1, 330, 1, 64, 1, False), rows(1, 330, 1, 64, 2, False)
    for m, f in enumerate(order):
        v[:, 64 * m : 64 * m + 64] = (v[:, 64 * m : 64 * m + 64].double() * f).bfloat16()
    v[:, 320:] = 0
    cache = ops.kv8_cache(1, 1, 400, 64, kind, device="cuda")
    ops.kv8_append(cache, k, v, 0)
    value, bound = by_contributions(q[0], k[0].transpose(0, 1), v[0].transpose(0, 1), kind, 329)
    # numbers below the least normal one (2^-126) are off by half a step of the subnormal ones, 2^-134 in bf16, or flushed
    near(ops.kv8_attention(q, cache, 329)[0], (value, bound + 2.0 ** -125))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,low", [(270, 256), (6000, 3000)])
@pytest.mark.parametrize("T", [1, 3])
def test_a_block_that_is_no_number_reaches_queries_whose_weight_for_it_is_zero(kind, n, low, T):
    """Scores so much lower than others that the weights are zero in 32 bits: zero times what is no number is none."""
    q, k, v = rows(1, T, 2, 64, 3, False), rows(1, n + T, 1, 64, 1, False), rows(1, n + T, 1, 64, 2, False)
    q[:] = q[:, :1, :1]
    x = q[0, 0, 0].float()
    k[0, :low, 0] = (-300 * 8.0 * x / (x @ x)).bfloat16()
    v[0, 70, 0, 5] = float("inf")
    cache = ops.kv8_cache(1, 1, n + T, 64, kind, device="cuda")
    ops.kv8_append(cache, k[:, :n], v[:, :n], 0)
    assert bool(torch.isnan(ops.kv8_attention(q, cache, n, k[:, n:], v[:, n:])).all())


@pytest.mark.parametrize("T", [1, 3, 100])
def test_positions_at_the_ends_of_64_bits(T):
    cache, k, v = filled(3, 2, 64, 100, "int8", capacity=128)
    before = {n: t.clone() for n, t in bits(cache).items()}
    q, nk, nv = rows(3, T, 4, 64, 3, False), rows(3, T, 2, 64, 4), rows(3, T, 2, 64, 5)
    far = torch.tensor([2 ** 63 - 1, -(2 ** 63), 2 ** 63 - 50], device="cuda")
    out = ops.kv8_attention(q, cache, far, nk, nv)
    assert bool(torch.isnan(out[0]).all()) and not out[1].any() and bool(torch.isnan(out[2]).all())
    assert all(torch.equal(before[n], t) for n, t in bits(cache).items())
    got = ops.kv8_expand(cache, torch.tensor([2 ** 63 - 1, -(2 ** 63), 100], device="cuda"), 64, 100)
    assert torch.equal(got[0][2], ops.kv8_expand(cache, 100, 64)[0][2]) and not got[0][1].any()


@pytest.mark.parametrize("T", [1, 3, 100])
def test_caches_without_room(T):
    q, nk, nv = rows(3, T, 4, 64, 3, False), rows(3, T, 2, 64, 4), rows(3, T, 2, 64, 5)
    empty = ops.kv8_cache(3, 2, 0, 64, "int8", device="cuda")
    out = ops.kv8_attention(q, empty, torch.tensor([0, -1, 5], device="cuda"), nk, nv)
    assert bool(torch.isnan(out[0]).all()) and not out[1].any() and bool(torch.isnan(out[2]).all())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [40, 64, 128])
@pytest.mark.parametrize("T", [1, 3, 64, 130, 300])
@pytest.mark.parametrize("starts", [[0], [130], [0, 130, -1, 77, 64, 63, 200, 1]])
def test_new_tokens_as_given(kind, D, T, starts):
    """Earlier full blocks are codes, the open block and the call's own tokens as they came; the cache is the same afterwards."""
    B, G, rep = len(starts), 2, 2
    longest = max(starts) + T
    _, k, v = filled(B, G, D, longest, kind)
    caches = [ops.kv8_cache(B, G, longest + 70, D, kind, device="cuda") for _ in range(2)]
    for b, n in enumerate(starts):
        one = ops.kv8_cache(1, G, longest + 70, D, kind, device="cuda")
        ops.kv8_append(one, k[b : b + 1, : max(n, 0)], v[b : b + 1, : max(n, 0)], 0)
        for c in caches:
            for x in c:
                c[x].view(torch.uint8)[b] = one[x].view(torch.uint8)[0]
    q = rows(B, T, G * rep, D, 5, False) * 0.25
    at = lambda x: torch.stack([x[b, max(n, 0) : max(n, 0) + T] for b, n in enumerate(starts)])  # noqa: E731
    for pos in (torch.tensor(starts, device="cuda"), starts[0])[: 1 + (B == 1)]:
        cache = {x: t.clone() for x, t in caches[0].items()}
        out = ops.kv8_attention(q, cache, pos, at(k), at(v), as_given=True)
        for b, n in enumerate(starts):
            if n < 0:
                assert not out[b].any()
                continue
            K, V = (torch.cat((cache64(x[b].transpose(0, 1), kind, n), x[b, n : n + T].double().transpose(0, 1)), 1).transpose(0, 1)[None] for x in (k, v))
            near(out[b : b + 1], attention64(q[b : b + 1], K, V)["o"], f"sequence {b}")
    ops.kv8_append(caches[1], at(k), at(v), pos)
    assert all(torch.equal(t, bits(caches[1])[x]) for x, t in bits(cache).items())


def test_new_tokens_as_given_at_the_edges():
    cache, k, v = filled(3, 2, 64, 100, "int8", capacity=128)
    q, nk, nv = rows(3, 100, 4, 64, 3, False), rows(3, 100, 2, 64, 4), rows(3, 100, 2, 64, 5)
    before = {n: t.clone() for n, t in bits(cache).items()}
    out = ops.kv8_attention(q, cache, torch.tensor([100, 2 ** 63 - 1, -7], device="cuda"), nk, nv, as_given=True)
    assert torch.isfinite(out[0, :28]).all() and bool(torch.isnan(out[0, 28:]).all()) and bool(torch.isnan(out[1]).all()) and not out[2].any()
    assert all(torch.equal(before[n][1:], t[1:]) for n, t in bits(cache).items())
    assert not ops.kv8_attention(q, cache, -3, nk, nv, as_given=True).any()
    cache = filled(1, 2, 64, 100, "int8", capacity=512)[0]  # what is no number reaches the queries that see it, and no others
    same = {n: t.clone() for n, t in cache.items()}
    clean = ops.kv8_attention(q[:1], same, 100, nk[:1], nv[:1], as_given=True)
    nv[0, 20, 1, 5] = float("inf")
    out = ops.kv8_attention(q[:1], cache, 100, nk[:1], nv[:1], as_given=True)
    assert torch.equal(out[:, :20], clean[:, :20]) and torch.equal(out[:, :, :2], clean[:, :, :2]) and not torch.isfinite(out[:, 20:, 2:, 5]).any()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("T", [2, 64])
def test_what_a_full_cache_gives_for_fewer_tokens(kind, T):
    """Multiples of a block, and up to 64 tokens back."""
    cache, k, v = filled(1, 2, 64, 300, kind)
    q = rows(1, T, 4, 64, 3, False)
    for n in (64, 128, 192, 236, 237, 255, 256, 299):
        fresh = ops.kv8_cache(1, 2, 320, 64, kind, device="cuda")
        ops.kv8_append(fresh, k[:, :n], v[:, :n], 0)
        assert all(torch.equal(a, b) for a, b in zip(ops.kv8_expand(cache, n, 64), ops.kv8_expand(fresh, n, 64))), n
        assert torch.equal(ops.kv8_attention(q, cache, n - T), ops.kv8_attention(q, fresh, n - T)), n


@pytest.mark.parametrize("T", [3, 80])
def test_new_tokens_as_given_in_a_graph_on_a_stream_and_in_other_layouts(T):
    n, steps = 100, 4
    k, v, q = (rows(2, n + T * steps, h, 64, s, False) for h, s in ((2, 1), (2, 2), (4, 3)))

    def fresh():
        cache = ops.kv8_cache(2, 2, n + T * steps, 64, "int8", device="cuda")
        ops.kv8_append(cache, k[:, :n], v[:, :n], 0)
        return cache

    def at_device(i):  # as captured: keys are split by the capacity then, not by the tokens that there are
        return torch.tensor([n + T * i], device="cuda")

    want, cache = [], fresh()
    for i in range(steps):
        at = slice(n + T * i, n + T * i + T)
        want.append(ops.kv8_attention(q[:, at], cache, at_device(i), k[:, at], v[:, at], as_given=True))
    graphs = []
    for _ in range(2):  # two captures, replayed in turn
        c, pos = fresh(), torch.tensor([n], device="cuda")
        new = [x[:, n : n + T].clone() for x in (q, k, v)]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.kv8_attention(new[0], c, pos, new[1], new[2], as_given=True)
        graphs.append((g, new, out, pos, c))
    for i in range(steps):
        for g, new, out, pos, _ in graphs:
            pos.fill_(n + T * i)
            for x, y in zip(new, (q, k, v)):
                x.copy_(y[:, n + T * i : n + T * i + T])
            g.replay()
            assert torch.equal(out, want[i])
    assert all(torch.equal(a, bits(graphs[0][4])[x]) for x, a in bits(cache).items())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = fresh()
        for i in range(steps):  # heads first, and rows whose addresses are no multiples of 16 bytes: copied
            new = [x[:, n + T * i : n + T * i + T] for x in (q, k, v)]
            new[1] = new[1].transpose(1, 2).contiguous().transpose(1, 2)
            new[2] = torch.zeros(2, T, 2, 72, device="cuda", dtype=torch.bfloat16)[..., 3:67].copy_(new[2])
            assert torch.equal(ops.kv8_attention(new[0], other, at_device(i), new[1], new[2], as_given=True), want[i])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, bits(other)[x]) for x, a in bits(cache).items())

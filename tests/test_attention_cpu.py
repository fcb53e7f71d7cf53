"""Softmax attention and the 8-bit key/value cache on the CPU: the PyTorch statements against the definition, refusals, the layers and
models that use them."""

import pytest
import torch

from attention_cases import attention64, cache64, kv8_attention64
from triune_b200 import ops
from triune_b200.config import ModelConfig
from triune_b200.inference import GraphedGreedyDecoder, generate_tokens
from triune_b200.models import SoftmaxAttention, kv8_state
from triune_b200.models.layer_state import LayerState
from triune_b200.models.universal import DenseTransformerBlock, UniversalDenseTransformer
from triune_b200.serve.srsm import _pack, _unpack

KINDS = ["int8", "e4m3"]


def rand(*shape, seed=0, dtype=torch.float32):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed), dtype=dtype)


@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1, 8), (2, 7, 7, 4, 2, 16), (3, 5, 20, 3, 1, 8), (2, 9, 4, 2, 2, 8)])
@pytest.mark.parametrize("how", [{}, {"causal": False}, {"window": 3}, {"scale": 0.3}])
def test_attention_and_its_gradients(shape, how):
    B, T, S, H, G, D = shape
    q, k, v = rand(B, T, H, D, dtype=torch.float64), rand(B, S, G, D, seed=1, dtype=torch.float64), rand(B, S, G, D, seed=2, dtype=torch.float64)
    inputs = [x.requires_grad_() for x in (q, k, v)]
    lengths, grad = [S, 0, 1][:B], rand(B, T, H, D, seed=3, dtype=torch.float64)
    for n in (None, lengths):
        out = ops.attention(*inputs, key_lengths=None if n is None else torch.tensor(n), **how)
        want = attention64(*inputs, how.get("causal", True), how.get("window"), n, None, how.get("scale"), grad)
        for got, name in zip((out, *torch.autograd.grad(out, inputs, grad)), ("o", "dq", "dk", "dv")):
            assert torch.allclose(got, want[name][0], rtol=1e-10, atol=1e-12), name


def test_gradients_against_differences():
    q, k, v = (rand(1, n, h, 4, seed=h, dtype=torch.float64).requires_grad_() for n, h in ((3, 4), (5, 2), (5, 2)))
    assert torch.autograd.gradcheck(lambda *x: ops.attention(*x, window=3, key_lengths=torch.tensor([4])), (q, k, v))


def test_positions_and_what_masked_places_hold():
    q, k, v = rand(2, 4, 2, 8), rand(2, 10, 1, 8, seed=1), rand(2, 10, 1, 8, seed=2)
    starts = torch.tensor([3, 6])
    out = ops.attention(q, k, v, query_start=starts)
    for b in range(2):
        assert torch.allclose(out[b : b + 1], ops.attention(q[b : b + 1], k[b : b + 1], v[b : b + 1], query_start=int(starts[b])), atol=1e-6)
    clean = ops.attention(q, k, v, key_lengths=torch.tensor([7, 7]), causal=False)
    k[:, 7:], v[:, 7:] = float("nan"), float("inf")
    assert torch.equal(ops.attention(q, k, v, key_lengths=torch.tensor([7, 7]), causal=False), clean)
    out = ops.attention(q, k[:, :8].nan_to_num(0.0), v[:, :8], query_start=4)
    assert torch.isfinite(out[:, :3]).all() and not torch.isfinite(out[:, 3:]).any()


@pytest.mark.parametrize("bad", [
    dict(q=(2, 3, 4)), dict(q=(1, 3, 3, 8)), dict(q=(2, 3, 4, 8)), dict(q=(1, 3, 4, 16)), dict(v=(1, 4, 2, 8)), dict(k=(1, 5, 0, 8), v=(1, 5, 0, 8)),
    dict(dtype=torch.float64), dict(how={"window": 0}), dict(how={"window": 2.5}), dict(how={"window": 3, "causal": False}), dict(how={"scale": 0.0}),
    dict(how={"scale": float("nan")}), dict(how={"key_lengths": torch.tensor([1.0])}), dict(how={"key_lengths": torch.tensor([1, 2])}),
    dict(how={"query_start": torch.tensor([1, 2, 3])}),
])
def test_attention_refuses(bad):
    q, k, v = rand(*bad.get("q", (1, 3, 4, 8))), rand(*bad.get("k", (1, 5, 2, 8))), rand(*bad.get("v", (1, 5, 2, 8)))
    with pytest.raises(ValueError):
        ops.attention(q.to(bad.get("dtype", q.dtype)), k, v, **bad.get("how", {}))


@pytest.mark.parametrize("scale", [1e-40, 1e38, float("inf")])
def test_scales_that_are_no_numbers_in_32_bits_are_refused(scale):
    q = rand(1, 3, 2, 8)
    with pytest.raises(ValueError, match="scale"):
        ops.attention(q, q, q, scale=scale)
    with pytest.raises(ValueError, match="scale"):
        ops.kv8_attention(q.bfloat16(), ops.kv8_cache(1, 2, 64, 8), 0, scale=scale)


def rows(*shape, seed=0):
    x = rand(*shape, seed=seed)
    x[..., 1] *= 7.0
    return x.bfloat16()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("D", [8, 64, 80])
def test_the_cache_and_attention_from_it(kind, D):
    B, G, H, n = 3, 2, 4, 150
    k, v, q = rows(B, n + 80, G, D), rows(B, n + 80, G, D, seed=1), rand(B, 5, H, D, seed=2).bfloat16()
    cache = ops.kv8_cache(B, G, 256, D, kind)
    ops.kv8_append(cache, k[:, :n], v[:, :n], 0)
    for x, y in zip(ops.kv8_expand(cache, n, D), (k, v)):
        for b in range(B):
            assert torch.equal(x[b].transpose(0, 1), cache64(y[b].transpose(0, 1), kind, n).float().bfloat16())
    starts = torch.tensor([n, -1, 100])  # the third sequence goes back by 50 tokens
    at = torch.stack([torch.arange(max(0, s), max(0, s) + 5) for s in starts.tolist()])
    new = [torch.stack([x[b, at[b]] for b in range(B)]) for x in (k, v)]
    before = {name: t.clone() for name, t in cache.items()}
    out = ops.kv8_attention(q, cache, starts, *new)
    assert not out[1].any() and all(torch.equal(before[name][1].view(torch.uint8), t[1].view(torch.uint8)) for name, t in cache.items())
    value, bound = kv8_attention64(q[0], k[0].transpose(0, 1), v[0].transpose(0, 1), kind, n)
    assert bool(((out[0].double() - value).abs() <= bound).all())
    past = ops.kv8_attention(q, cache, torch.tensor([254, 256, -3]), *new)
    assert bool(torch.isnan(past[0, 2:]).all()) and not torch.isnan(past[0, :2]).any() and bool(torch.isnan(past[1]).all()) and not past[2].any()


@pytest.mark.parametrize("kind", KINDS)
def test_contents_do_not_depend_on_the_portions(kind):
    k, v = rows(2, 300, 2, 64), rows(2, 300, 2, 64, seed=1)
    whole = ops.kv8_cache(2, 2, 300, 64, kind)
    ops.kv8_append(whole, k, v, 0)
    for chunk in (1, 50, 64, 129):
        cache = ops.kv8_cache(2, 2, 300, 64, kind)
        for p in range(0, 300, chunk):
            ops.kv8_append(cache, k[:, p : p + chunk], v[:, p : p + chunk], torch.tensor([p, p]))
        assert all(torch.equal(cache[n].view(torch.uint8), whole[n].view(torch.uint8)) for n in whole)


def test_a_block_with_what_is_no_number_reads_as_none():
    cache = ops.kv8_cache(1, 1, 128, 8)
    k, v = rows(1, 128, 1, 8), rows(1, 128, 1, 8)
    v[0, 70, 0, 0] = float("inf")
    ops.kv8_append(cache, k, v, 0)
    got = ops.kv8_expand(cache, 128, 8)[1][0, :, 0]
    assert torch.isfinite(got[:64]).all() and bool(torch.isnan(got[64:]).all())


def test_the_cache_refuses():
    cache, k = ops.kv8_cache(2, 2, 100, 64), rows(2, 3, 2, 64)
    q = rows(2, 3, 4, 64)
    assert cache["k8"].shape == (2, 2, 128, 64) and ops.kv8_cache(1, 1, 1, 72)["k8"].shape[3] == 128
    for bad in (dict(kind="int4"), dict(head_dim=136), dict(head_dim=12), dict(kv_heads=0), dict(capacity=-1)):
        with pytest.raises(ValueError):
            ops.kv8_cache(**{**dict(batch=1, kv_heads=1, capacity=64, head_dim=64), **bad})
    for call in (lambda: ops.kv8_append(cache, k.float(), k.float(), 0), lambda: ops.kv8_append(cache, k, k[:, :2], 0), lambda: ops.kv8_append(cache, k[:1], k[:1], 0),
                 lambda: ops.kv8_append(cache, k, k, 126), lambda: ops.kv8_append(cache, k, k, torch.tensor([1.0])), lambda: ops.kv8_append(cache, k, k, torch.tensor([1, 2, 3])),
                 lambda: ops.kv8_attention(q[:, :, :3], cache, 0), lambda: ops.kv8_attention(q.float(), cache, 0), lambda: ops.kv8_attention(q, cache, 0, k),
                 lambda: ops.kv8_attention(q, cache, 0, k[:, :2], k[:, :2]), lambda: ops.kv8_attention(q, cache, 0, scale=-1.0),
                 lambda: ops.kv8_expand(cache, 10, 60), lambda: ops.kv8_expand(cache, 129, 64), lambda: ops.kv8_expand(cache, 10, 64, 200)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(RuntimeError, match="no gradients"):
        ops.kv8_attention(q.requires_grad_(), cache, 0, k, k)


# ---------------------------------------------------------------------------------------------------- layers and models
def model(kv_cache=None, **kw):
    torch.manual_seed(0)
    cfg = ModelConfig(family="universal", vocab_size=61, hidden_dim=32, num_layers=2, num_heads=4, head_dim=8, num_kv_heads=2, mixer="sdpa",
                      ffn="swiglu", dense_hidden=48, kv_cache=kv_cache, **kw).validate()
    return UniversalDenseTransformer.from_config(cfg).eval()


@pytest.mark.parametrize("kind", KINDS)
@torch.no_grad()
def test_a_layer_serves_from_8_bits_near_what_it_serves_from_16(kind):
    """Keys and values of the full blocks are off by half a code of their block's scale: 1 / 254 (int8) of the block's largest, or 2^-4 of
    themselves (e4m3); outputs are averages of values, so they stay within a few per cent of their size."""
    torch.manual_seed(1)
    layer = SoftmaxAttention(64, 8, 8, 2)
    x = rand(2, 200, 64)
    wide, cache = (None, 0), (kv8_state(2, 2, 8, kind), 0)
    for part in x.split((130, 1, 1, 60, 1, 7), 1):
        a, wide = layer(part, cache=wide)
        b, cache = layer(part, cache=cache)
        assert float((a - b).norm() / a.norm()) < (0.03 if kind == "int8" else 0.1)
    assert cache[1] == 200 and isinstance(cache[0], LayerState) and cache[0].capacity >= 200


@pytest.mark.parametrize("kind", KINDS)
def test_generation_does_not_depend_on_the_portions_of_the_prompt(kind):
    m = model(kind)
    ids = torch.randint(0, 61, (1, 150), generator=torch.Generator().manual_seed(3))
    outs = [generate_tokens(m, ids, 20, temperature=0.0, repetition_penalty=1.0, count_penalty=0.0, prefill_chunk=150)[0] for _ in range(2)]
    assert outs[0] == outs[1] and len(outs[0]) == 20
    decoder = GraphedGreedyDecoder(m, 1)
    for _ in range(2):  # a second request in the same buffers
        assert decoder.generate(ids, 20)[0, 150:].tolist() == outs[0]


def test_sessions_are_parked_and_come_back():
    m = model("int8")
    ids = torch.randint(0, 61, (1, 100), generator=torch.Generator().manual_seed(4))
    with torch.no_grad():
        _, cache = m(ids, cache=m.init_cache(1))
        back = _unpack(*_pack(cache))
        assert all(b[0].capacity == 128 and b[1] == 100 for b in back)
        step = torch.tensor([[5]])
        a, _ = m(step, cache=[(c[0].clone(), c[1]) for c in cache])
        b, after = m(step, cache=back)
    assert torch.equal(a, b) and after[0][1] == 101


def test_growing_keeps_what_is_held():
    state = kv8_state(1, 2, 8, "e4m3")
    k, v = rows(1, 200, 2, 8), rows(1, 200, 2, 8, seed=1)
    ops.kv8_append(state, k, v, 0)
    want = ops.kv8_expand(state, 200, 8)
    assert state.reserve(1000) and state.capacity == 1024 and state["ks"].shape[2] == 16 and not state.reserve(1024)
    assert all(torch.equal(a, b) for a, b in zip(ops.kv8_expand(state, 200, 8), want))


def test_configurations_without_such_a_cache_are_refused():
    for bad in (dict(kv_cache="int4"), dict(kv_cache="int8", mixer="gla"), dict(kv_cache="int8", family="triune")):
        with pytest.raises(ValueError):
            ModelConfig(**{**dict(family="universal", hidden_dim=32, num_heads=4, head_dim=8, num_layers=8, mixer="sdpa"), **bad}).validate()
    assert ModelConfig.from_dict(model("e4m3").cfg.to_dict()).kv_cache == "e4m3"


def test_training_a_model_with_shared_heads():
    m = model().train()
    ids = torch.randint(0, 61, (2, 40), generator=torch.Generator().manual_seed(5))
    m.forward_loss(ids[:, :-1], ids[:, 1:]).backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in m.parameters())
    block = DenseTransformerBlock(32, 4, num_kv_heads=2)
    y, state = block(rand(1, 5, 32), state=(None, 0))
    assert y.shape == (1, 5, 32) and state[0][0].shape == (1, 5, 2, 8)


def test_the_status_word_is_no_inference_tensor():
    from triune_b200.ops import hybrid

    kept = dict(hybrid._STATUS)
    hybrid._STATUS.clear()
    try:
        with torch.inference_mode():
            assert not hybrid.status_word("cpu").is_inference()
    finally:
        hybrid._STATUS.clear()
        hybrid._STATUS.update(kept)


@pytest.mark.parametrize("mixer", ["sdpa", "gla"])
def test_a_model_evaluated_in_inference_mode_can_be_trained_afterwards(mixer):
    torch.manual_seed(0)
    m = UniversalDenseTransformer.from_config(ModelConfig(family="universal", vocab_size=61, hidden_dim=32, num_layers=2, num_heads=4, head_dim=8,
                                                          mixer=mixer, ffn="swiglu", dense_hidden=48).validate())
    ids = torch.randint(0, 61, (2, 40), generator=torch.Generator().manual_seed(5))
    with torch.inference_mode():
        m.eval()(ids)
    m.train().forward_loss(ids[:, :-1], ids[:, 1:]).backward()
    assert all(torch.isfinite(p.grad).all() for p in m.parameters())


def one_by_one(layer, x, kind):
    cache, out = (kv8_state(x.shape[0], layer.kv_heads, layer.head_dim, kind), 0), []
    for t in range(x.shape[1]):
        y, cache = layer(x[:, t : t + 1], cache=cache)
        out.append(y)
    return torch.cat(out, 1), cache


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("first", [0, 1, 61, 63, 64, 127])
@torch.no_grad()
def test_drafted_tokens_that_cross_the_end_of_a_block_are_single_steps(kind, first):
    """Outputs of the attention are rounded to bf16 (2^-8 of themselves at most), from sums in another order, before the layer's last product."""
    torch.manual_seed(2)
    layer = SoftmaxAttention(64, 8, 8, 2)
    for n in (2, 5, 40, 64):
        x = rand(2, first + n, 64, seed=n)
        want, held = one_by_one(layer, x, kind)
        _, cache = one_by_one(layer, x[:, :first], kind) if first else (None, (kv8_state(2, 2, 8, kind), 0))
        got, cache = layer(x[:, first:], cache=cache)
        assert float((got - want[:, first:]).norm() / want[:, first:].norm()) < 2.0 ** -8
        assert cache[1] == first + n and all(cache[0][name].shape == t.shape for name, t in held[0].tensors.items())


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("first,n", [(0, 64), (0, 200), (3, 61), (40, 100), (63, 2), (130, 130)])
@torch.no_grad()
def test_outputs_do_not_depend_on_later_tokens(kind, first, n):
    """The last token of a call is another, and much larger: the others' outputs stay."""
    torch.manual_seed(3)
    layer = SoftmaxAttention(64, 8, 8, 2)
    x = rand(1, first + n, 64)
    y = x.clone()
    y[:, -1] *= -1000.0
    outs = []
    for z in (x, y):
        cache = (kv8_state(1, 2, 8, kind), 0)
        if first:
            _, cache = layer(z[:, :first], cache=cache)
        outs.append(layer(z[:, first:], cache=cache)[0])
    assert torch.equal(outs[0][:, :-1], outs[1][:, :-1]) and not torch.equal(outs[0][:, -1], outs[1][:, -1])


@pytest.mark.parametrize("kind,limit", [("int8", 0.02), ("e4m3", 0.08)])
@torch.no_grad()
def test_portions_of_a_prompt_of_several_sizes(kind, limit):
    """The first layer's cache is the same whatever the portions, but for the few numbers that a product of another shape rounds otherwise; logits, and later layers' caches, differ by what codes round off (1 / 254 of a
    block's largest, or 2^-4 of each number) in averages over what is seen."""
    m = model(kind)
    ids = torch.randint(0, 61, (1, 150), generator=torch.Generator().manual_seed(3))
    want, held = m(ids, cache=m.init_cache(1))
    for chunk in (50, 64, 65, 7, 1):
        cache, out = m.init_cache(1), []
        for part in ids.split(chunk, 1):
            y, cache = m(part, cache=cache)
            out.append(y)
        assert float((torch.cat(out, 1) - want).norm() / want.norm()) < limit, chunk
        n = 150 // ops.KV8_BLOCK
        for name in ("k8", "v8"):
            a, b = (c[0][0][name][:, :, : n * ops.KV8_BLOCK].float() for c in (cache, held))
            assert float((a != b).float().mean()) < 1e-2, (chunk, name)


@pytest.mark.parametrize("kind", KINDS)
def test_new_tokens_as_given(kind):
    B, G, H, D, n, T = 3, 2, 4, 64, 100, 150
    k, v, q = rows(B, n + T, G, D), rows(B, n + T, G, D, seed=1), rand(B, T, H, D, seed=2).bfloat16()
    cache, same = (ops.kv8_cache(B, G, 256, D, kind) for _ in range(2))
    for c in (cache, same):
        ops.kv8_append(c, k[:, :n], v[:, :n], 0)
    starts = torch.tensor([n, -1, 64])  # the third sequence goes back
    new = [torch.stack([x[b, max(0, s) : max(0, s) + T] for b, s in enumerate(starts.tolist())]) for x in (k, v)]
    out = ops.kv8_attention(q, cache, starts, *new, as_given=True)
    ops.kv8_append(same, *new, starts)
    assert all(torch.equal(cache[x].view(torch.uint8), same[x].view(torch.uint8)) for x in cache) and not out[1].any()
    for b in (0, 2):
        p = int(starts[b])
        K, V = (torch.cat((cache64(x[b].transpose(0, 1), kind, p), y[b].double().transpose(0, 1)), 1).transpose(0, 1)[None] for x, y in zip((k, v), new))
        value, bound = attention64(q[b : b + 1], K, V)["o"]
        assert bool(((out[b : b + 1].double() - value).abs() <= bound).all())
    with pytest.raises(ValueError, match="as_given"):
        ops.kv8_attention(q, cache, 0, as_given=True)


def test_a_loss_that_is_no_number_because_a_wait_expired_says_so():
    """Attention gives NaN where a kernel's wait expired; what trains raises with that reason. The status word is set here, on the host."""
    from triune_b200.models.universal import TriuneUniversalEngine
    from triune_b200.ops import hybrid
    from triune_b200.trainer.trainer import Trainer

    m = model()
    ids = torch.randint(0, 61, (2, 20), generator=torch.Generator().manual_seed(5))
    calls = [lambda e=TriuneUniversalEngine(m, optimizer=torch.optim.SGD(m.parameters(), lr=0.0)): e.train_step(ids)]
    t = Trainer(m, {"optimizer": "adamw", "mode": "cortex"}, optimizer=torch.optim.SGD(m.parameters(), lr=0.0), device="cpu")
    t.step_on_device = lambda *a: m.forward_loss(a[0], a[1]).detach()
    calls.append(lambda: t.train_step(ids[:, :-1], ids[:, 1:]))
    kept, weight = dict(hybrid._STATUS), m.norm.weight.detach().clone()
    try:
        word = hybrid.status_word("cpu")
        for broken in (False, True):
            with torch.no_grad():
                m.norm.weight.copy_(weight * (float("nan") if broken else 1.0))
            for status in (0, 3):
                word.fill_(status)
                for call in calls:
                    if broken and status:
                        with pytest.raises(RuntimeError, match="bounded wait expired"):
                            call()
                    else:
                        assert torch.isfinite(torch.tensor(call())) != broken
    finally:
        word.zero_()
        hybrid._STATUS.clear()
        hybrid._STATUS.update(kept)


@pytest.mark.parametrize("kind", KINDS)
def test_what_a_full_cache_gives_for_fewer_tokens(kind):
    """Multiples of a block, and up to 64 tokens back."""
    k, v = rows(1, 300, 2, 64), rows(1, 300, 2, 64, seed=1)
    cache = ops.kv8_cache(1, 2, 320, 64, kind)
    ops.kv8_append(cache, k, v, 0)
    q = rand(1, 2, 4, 64, seed=2).bfloat16()
    for n in (64, 128, 192, 236, 237, 255, 256, 299):
        fresh = ops.kv8_cache(1, 2, 320, 64, kind)
        ops.kv8_append(fresh, k[:, :n], v[:, :n], 0)
        assert all(torch.equal(a, b) for a, b in zip(ops.kv8_expand(cache, n, 64), ops.kv8_expand(fresh, n, 64))), n
        assert torch.equal(ops.kv8_attention(q, cache, n - 2), ops.kv8_attention(q, fresh, n - 2)), n

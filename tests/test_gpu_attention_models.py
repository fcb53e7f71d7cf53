"""Layers and models over the softmax attention kernels, and over the 8-bit cache: trained, prompted, decoded in graphs."""

import pytest
import torch

from triune_b200 import _ext, ops
from triune_b200.config import ModelConfig
from triune_b200.inference import GraphedGreedyDecoder, advance, generate_tokens
from triune_b200.models import SoftmaxAttention, kv8_state
from triune_b200.models.universal import UniversalDenseTransformer
from triune_b200.utils import place_model

pytestmark = pytest.mark.gpu


def layer(heads=8, kv_heads=2, head_dim=64, seed=0):
    torch.manual_seed(seed)
    return SoftmaxAttention(heads * head_dim, heads, head_dim, kv_heads).cuda().bfloat16()


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("kv_heads,head_dim,prefix", [(2, 64, 0), (8, 64, 77), (2, 128, 300), (1, 80, 5)])
def test_a_layer_follows_its_plain_form(kv_heads, head_dim, prefix):
    """Against the layer in fp32 with the same weights: projections, rotations and outputs are rounded to bf16 (2^-8 at most, some
    2^-9.3 on average), five of them on the way to an output and twice as many to a gradient, errors of which are independent."""
    m = layer(8, kv_heads, head_dim)
    plain = SoftmaxAttention(m.dim, 8, head_dim, kv_heads).cuda()
    plain.load_state_dict(m.state_dict())
    x = torch.randn(2, 150, m.dim, device="cuda").bfloat16().requires_grad_()
    y = x.detach().float().requires_grad_()
    past = [torch.randn(2, prefix, kv_heads, head_dim, device="cuda").bfloat16() for _ in "kv"]
    before = ops.launch_count()
    a, state = m(x, cache=((past[0], past[1]), prefix) if prefix else None)
    assert ops.launch_count() > before
    _ext.set_reference_ops(True)
    try:
        b, _ = plain(y, cache=((past[0].float(), past[1].float()), prefix) if prefix else None)
        g = torch.randn_like(a)
        want = torch.autograd.grad(b, [y, *plain.parameters()], g.float())
    finally:
        _ext.set_reference_ops(False)
    assert rel(a, b) < 2e-2
    got = torch.autograd.grad(a, [x, *m.parameters()], g)
    assert all(rel(p, q) < 4e-2 for p, q in zip(got, want))
    assert state is None or state[0][0].shape[1] == prefix + 150


def model(kv_cache, head_dim=64, seed=1):
    torch.manual_seed(seed)
    cfg = ModelConfig(family="universal", vocab_size=512, hidden_dim=8 * head_dim, num_layers=3, num_heads=8, head_dim=head_dim, num_kv_heads=2,
                      mixer="sdpa", ffn="swiglu", dense_hidden=768, kv_cache=kv_cache).validate()
    return place_model(UniversalDenseTransformer.from_config(cfg), "cuda", torch.bfloat16).eval()


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
def test_decoding_in_a_graph_is_decoding_step_by_step(kind):
    m = model(kind)
    ids = torch.randint(0, 512, (1, 200), device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    decoder = GraphedGreedyDecoder(m, 1)
    for n in (200, 90, 150):  # the second and third request find the buffers and the capture of the first
        want = generate_tokens(m, ids[:, :n], 140, temperature=0.0, repetition_penalty=1.0, count_penalty=0.0, prefill_chunk=4096)[0]
        assert decoder.generate(ids[:, :n], 140)[0, n:].tolist() == want


@pytest.mark.parametrize("kind,limit", [("int8", 0.05), ("e4m3", 0.15)])
@torch.no_grad()
def test_logits_from_8_bits_are_near_those_from_16(kind, limit):
    narrow, wide = model(kind), model(None)
    ids = torch.randint(0, 512, (2, 300), device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    caches = [m.init_cache(2) for m in (narrow, wide)]
    for part in ids.split((200, 3, 1, 96), 1):
        (a, caches[0]), (b, caches[1]) = (advance(m, part, c) for m, c in zip((narrow, wide), caches))
        assert rel(a, b) < limit


@torch.no_grad()
def test_a_cache_on_another_stream_and_one_that_grows():
    m = layer()
    x = torch.randn(1, 700, m.dim, device="cuda").bfloat16()
    outs = []
    for side in (False, True):
        stream = torch.cuda.Stream() if side else torch.cuda.current_stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            cache = (kv8_state(1, 2, 64, "int8", "cuda"), 0)
            out = []
            for part in x.split((1, 255, 2, 300, 142), 1):
                y, cache = m(part, cache=cache)
                out.append(y)
            outs.append(torch.cat(out, 1))
        torch.cuda.current_stream().wait_stream(stream)
        assert cache[1] == 700 and cache[0].capacity >= 700
    assert torch.equal(*outs)


@pytest.mark.parametrize("kind", ["int8", "e4m3"])
@pytest.mark.parametrize("heads,kv_heads,head_dim", [(8, 2, 64), (4, 4, 128), (16, 1, 72)])
@pytest.mark.parametrize("first,n", [(0, 64), (0, 200), (3, 61), (40, 100), (317, 5), (63, 2), (1000, 700)])
@torch.no_grad()
def test_outputs_on_an_8_bit_cache_do_not_depend_on_later_tokens(kind, heads, kv_heads, head_dim, first, n):
    """The last token of a call is another, and much larger: the others' outputs stay, bit for bit."""
    m = layer(heads, kv_heads, head_dim, seed=4)
    x = torch.randn(1, first + n, m.dim, device="cuda").bfloat16()
    y = x.clone()
    y[:, -1] *= -1000.0
    outs = []
    for z in (x, y):
        cache = (kv8_state(1, kv_heads, head_dim, kind, "cuda"), 0)
        if first:
            _, cache = m(z[:, :first], cache=cache)
        outs.append(m(z[:, first:], cache=cache)[0])
    assert torch.equal(outs[0][:, :-1], outs[1][:, :-1]) and not torch.equal(outs[0][:, -1], outs[1][:, -1])


@torch.no_grad()
def test_a_prompt_at_once_and_in_portions_is_near_the_prompt_in_16_bits():
    """Outputs against the layer without a cache: codes are off by 1 / 254 of a block's largest (some 3.5 times a value's size), and bf16 on the way."""
    m = layer(8, 2, 128, seed=5)
    x = torch.randn(2, 900, m.dim, device="cuda").bfloat16()
    want, _ = m(x)
    for chunk in (900, 256, 100, 64, 3):
        cache, out = (kv8_state(2, 2, 128, "int8", "cuda"), 0), []
        for part in x.split(chunk, 1):
            y, cache = m(part, cache=cache)
            out.append(y)
        assert rel(torch.cat(out, 1), want) < 3e-2, chunk
        assert cache[1] == 900


@pytest.mark.parametrize("shape", [(2, 37, 8, 2, 64), (1, 700, 8, 2, 128), (1, 2500, 16, 4, 64), (3, 2048, 8, 2, 80), (1, 2048, 6, 1, 128)])
@pytest.mark.parametrize("train", [True, False])
def test_prompts_with_shared_heads_of_any_size(shape, train):
    """Small and large prompts run on different attention; both follow the definition: outputs are rounded to bf16, weights on the way (2^-8 each), and
    so are the gradients of shared heads, on the library's way before they are added up."""
    from triune_b200.models.attention import _causal, _own_kernels

    B, T, H, G, D = shape
    q, k, v = (torch.randn(B, T, h, D, device="cuda", generator=torch.Generator("cuda").manual_seed(h)).bfloat16().requires_grad_(train) for h in (H, G, G + 1))
    v = v[:, :, :G]
    assert _own_kernels(q, k, v) == (B * H * T * T * D <= (1 << 32 if train else 1 << 27))
    out = _causal(q, k, v)
    kk, vv = (x.detach().double().repeat_interleave(H // G, 2).transpose(1, 2).requires_grad_() for x in (k, v))
    qq = q.detach().double().transpose(1, 2).requires_grad_()
    s = (qq @ kk.transpose(-1, -2)) * D ** -0.5
    want = s.masked_fill(torch.ones(T, T, dtype=torch.bool, device="cuda").triu(1), float("-inf")).softmax(-1) @ vv
    assert rel(out, want.transpose(1, 2)) < 2.0 ** -7
    if train:
        g = torch.randn_like(out)
        got = torch.autograd.grad(out, (q, k, v), g)
        dq, dk, dv = torch.autograd.grad(want, (qq, kk, vv), g.double().transpose(1, 2))
        for a, b in zip(got, (dq.transpose(1, 2), *(x.transpose(1, 2).unflatten(2, (G, H // G)).sum(3) for x in (dk, dv)))):
            assert rel(a, b) < 3 * 2.0 ** -7

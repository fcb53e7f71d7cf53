"""Softmax attention kernels (forward, backward) against the definition in 64 bits."""

import pytest
import torch

from attention_cases import attention64, near
from triune_b200 import ops
from triune_b200.ops.hybrid import check_status

pytestmark = pytest.mark.gpu


def make(B, T, S, H, G, D, seed=0, grad=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    new = lambda *s: torch.randn(*s, generator=gen, device="cuda").bfloat16()  # noqa: E731
    q, k, v = new(B, T, H, D), new(B, S, G, D), new(B, S, G, D)
    return [x.requires_grad_(grad) for x in (q, k, v)], new(B, T, H, D)


def check(qkv, grad, lengths=None, start=None, **how):
    """Outputs and gradients of one call, and the outputs of the same call without gradients."""
    q, k, v = qkv
    key_lengths = None if lengths is None else torch.tensor(lengths, device="cuda")
    out = ops.attention(q, k, v, key_lengths=key_lengths, query_start=start, **how)
    got = dict(zip(("dq", "dk", "dv"), torch.autograd.grad(out, (q, k, v), grad)), o=out.detach())
    starts = None if start is None else start.expand(q.shape[0]).tolist() if torch.is_tensor(start) else [start] * q.shape[0]
    want = attention64(q, k, v, how.get("causal", True), how.get("window"), lengths, starts, how.get("scale"), grad)
    for n in ("o", "dv", "dq", "dk"):
        near(got[n], want[n], n)
    with torch.no_grad():
        assert torch.equal(ops.attention(q, k, v, key_lengths=key_lengths, query_start=start, **how), got["o"])
    check_status(q.device)
    return got


SHAPES = [
    # B, T, S, H, G, D
    (1, 1, 1, 1, 1, 64), (1, 1, 1, 1, 1, 8), (2, 37, 37, 4, 4, 64), (1, 128, 128, 2, 1, 64), (2, 129, 129, 2, 2, 128), (1, 127, 127, 6, 2, 72),
    (1, 256, 256, 3, 1, 80), (3, 300, 300, 2, 2, 128), (1, 513, 513, 4, 1, 128), (2, 700, 700, 30, 10, 64), (1, 1500, 1500, 16, 4, 128),
    (1, 5, 200, 4, 2, 64), (2, 130, 1000, 4, 2, 128), (1, 200, 100, 2, 1, 64), (1, 3, 5000, 2, 1, 128), (40, 260, 260, 4, 4, 64),
]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("causal", [True, False])
def test_attention_follows_its_definition(shape, causal):
    check(*make(*shape), causal=causal)


@pytest.mark.parametrize("window", [1, 5, 64, 128, 129, 1000])
@pytest.mark.parametrize("shape", [(1, 300, 300, 2, 1, 64), (2, 257, 600, 4, 2, 128), (40, 400, 400, 4, 4, 64)])
def test_windows(shape, window):
    check(*make(*shape, seed=1), window=window)


@pytest.mark.parametrize("causal,window", [(True, None), (False, None), (True, 40)])
def test_padded_batches_and_sequences_without_keys(causal, window):
    qkv, grad = make(6, 260, 260, 4, 2, 80, seed=2)
    got = check(qkv, grad, lengths=[260, 0, 1, 128, 129, 255], causal=causal, window=window)
    assert not got["o"][1].any() and not any(got[n][1].any() for n in ("dq", "dk", "dv"))
    assert not got["dk"][4, 129:].any() and not got["dv"][2, 1:].any()


@pytest.mark.parametrize("start", [0, 3, 130, -2, 1000, 2 ** 40])
def test_positions_given_as_numbers_and_on_the_device(start):
    qkv, grad = make(2, 70, 200, 2, 1, 64, seed=3)
    a = check(qkv, grad, start=min(start, 10 ** 6))
    b = ops.attention(*qkv, query_start=torch.tensor([start], device="cuda", dtype=torch.int64))
    assert torch.equal(a["o"], b)
    if start < 200:
        check(qkv, grad, start=torch.tensor([start, start // 2], device="cuda"), window=31)


@pytest.mark.parametrize("window", [2 ** 31 - 1000, 2 ** 31 - 100, 2 ** 31 + 50, 2 ** 40, 2 ** 62])
def test_windows_as_far_as_positions(window):
    qkv, grad = make(2, 70, 200, 2, 1, 64, seed=3)
    got = check(qkv, grad, start=torch.tensor([2 ** 31, 2 ** 31 + 7], device="cuda"), window=window)
    assert got["o"].any() == (window > 2 ** 31 - 200)  # the first query sees the keys j > 2^31 - window, of 200


def test_scale_is_the_callers():
    check(*make(1, 150, 150, 2, 2, 64, seed=4), scale=0.7)


@pytest.mark.parametrize("T", [100, 400])
def test_large_scores_stay_in_range(T):
    (q, k, v), grad = make(1, T, T, 2, 2, 64, seed=5, grad=False)
    qkv = [(q * 12).requires_grad_(), k.requires_grad_(), v.requires_grad_()]
    out = ops.attention(*qkv, scale=4.0)  # scores of several hundred: rows are almost one-hot, sums are rescaled many times
    s = 4.0 * torch.einsum("bthd,bshd->bhts", qkv[0].double(), k.double())
    p = s.masked_fill(torch.ones(T, T, dtype=torch.bool, device="cuda").triu(1), float("-inf")).softmax(-1)
    want = torch.einsum("bhts,bshd->bthd", p, v.double())
    # fp32 scores of up to 4 * 12 * 64 * 4 = 12288, off by 64 * 2^-24 of themselves at most, move weights by 5 %: of neighbours in rank only
    assert float((out.double() - want).norm() / want.norm()) < 2e-2
    assert all(torch.isfinite(g).all() for g in torch.autograd.grad(out, qkv, grad))


@pytest.mark.parametrize("D", [64, 80, 128])
def test_layouts_in_place_and_copied(D):
    B, T, H, G = 2, 140, 4, 2
    gen = torch.Generator(device="cuda").manual_seed(6)
    wide = torch.randn(B, T, (H + 2 * G) * D + 8, generator=gen, device="cuda").bfloat16()
    rows = [wide[..., : H * D].unflatten(-1, (H, D)), wide[..., H * D : (H + G) * D].unflatten(-1, (G, D)), wide[..., (H + G) * D : (H + 2 * G) * D].unflatten(-1, (G, D))]
    grad = torch.randn(B, T, H, D, generator=gen, device="cuda").bfloat16()
    check([x.detach().requires_grad_() for x in rows], grad)
    heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2).requires_grad_() for x in rows]
    check(heads_first, grad.transpose(1, 2).contiguous().transpose(1, 2))
    odd = [torch.empty(x.numel() + 3, device="cuda", dtype=x.dtype)[3:].view(x.shape).copy_(x).requires_grad_() for x in rows]  # 6 bytes off
    check(odd, torch.empty(B, T, H, D + 1, device="cuda", dtype=grad.dtype)[..., :D].copy_(grad))


def test_expanded_inputs_sum_their_gradients():
    (q, k, v), _ = make(1, 100, 100, 4, 1, 64, seed=7)
    grad = torch.randn(3, 100, 4, 64, device="cuda").bfloat16()
    qq, kk, vv = (x.expand(3, -1, -1, -1) for x in (q, k, v))
    out = ops.attention(qq, kk, vv)
    want = attention64(qq, kk, vv, grad=grad)
    near(out, want["o"], "o")
    for got, n in zip(torch.autograd.grad(out, (q, k, v), grad), ("dq", "dk", "dv")):
        value, bound = (x.sum(0, keepdim=True) for x in want[n])
        near(got, (value, bound + 3 * 2.0 ** -8 * want[n][0].abs().sum(0, keepdim=True)), n)  # and the sums of bf16 gradients
    one = torch.ones((), device="cuda", dtype=torch.bfloat16)
    for g in torch.autograd.grad(ops.attention(q, k, v).sum(), (q, k, v), one):  # a gradient that is expanded itself
        assert torch.isfinite(g).all()


@pytest.mark.parametrize("T,S,H", [(300, 300, 2), (300, 300, 200), (5, 1000, 2)])
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
def test_values_that_are_no_numbers_reach_the_queries_that_see_them(T, S, H, what):
    (q, k, v), _ = make(1, T, S, H, 1, 64, seed=8, grad=False)
    at = S - T + T // 2  # seen by the second half of the queries
    clean = ops.attention(q, k, v)
    v[0, at, 0, 5] = what
    out = ops.attention(q, k, v)
    assert torch.equal(out[:, : T // 2], clean[:, : T // 2])
    assert torch.equal(out[:, T // 2 :, :, 5], torch.full_like(out[:, T // 2 :, :, 5], what)) or what != what and bool(torch.isnan(out[:, T // 2 :, :, 5]).all())
    keep = torch.arange(64, device="cuda") != 5
    assert torch.equal(out[..., keep], clean[..., keep])
    k[0, at] = what
    out = ops.attention(q, k, v)
    assert torch.equal(out[:, : T // 2], clean[:, : T // 2])


@pytest.mark.parametrize("what", [float("nan"), float("inf"), 3e38])
def test_padding_may_hold_anything(what):
    (q, k, v), grad = make(2, 200, 200, 2, 1, 128, seed=9)
    lengths = torch.tensor([130, 77], device="cuda")
    clean = ops.attention(q, k, v, key_lengths=lengths, causal=False)
    want = torch.autograd.grad(clean, (q, k, v), grad)
    with torch.no_grad():
        for b, n in enumerate(lengths.tolist()):
            k[b, n:] = what
            v[b, n:] = what
    out = ops.attention(q, k, v, key_lengths=lengths, causal=False)
    assert torch.equal(out, clean)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, (q, k, v), grad), want))


@pytest.mark.parametrize("D", [40, 64])
@pytest.mark.parametrize("causal,window", [(True, None), (False, None), (True, 70)])
def test_many_short_sequences_that_end_anywhere(D, causal, window):
    """More tiles of heads of up to 64 than twice the SMs, of sequences that end at, before and behind the tiles' ends."""
    lengths = [0, 1, 2, 31, 63, 64, 65, 100, 127, 128, 129, 191, 192, 193, 255, 256, 257, 298, 299, 300]
    qkv, grad = make(20, 300, 300, 8, 8, D, seed=13)
    got = check(qkv, grad, lengths=lengths, causal=causal, window=window)
    assert not got["o"][0].any() and not any(got["d" + n][0].any() for n in "qkv")
    with torch.no_grad():
        for b, n in enumerate(lengths):
            qkv[1][b, n:] = float("nan")
            qkv[2][b, n:] = float("inf")
    out = ops.attention(*qkv, key_lengths=torch.tensor(lengths, device="cuda"), causal=causal, window=window)
    assert torch.equal(out, got["o"])
    for n, x in zip("qkv", torch.autograd.grad(out, qkv, grad)):
        assert torch.equal(x, got["d" + n])


@pytest.mark.parametrize("shape", [(1, 520, 520, 16, 2, 64), (2, 400, 400, 10, 2, 40), (1, 1100, 1100, 16, 2, 128), (2, 300, 700, 24, 3, 72), (1, 1025, 129, 1, 1, 64)])
@pytest.mark.parametrize("causal", [True, False])
def test_keys_whose_queries_are_walked_by_two_blocks(shape, causal):
    """Fewer tiles of keys than half of the SMs, and eight tiles of queries or more of all heads that share them; some keys are seen by none."""
    qkv, grad = make(*shape, seed=14)
    got = check(qkv, grad, causal=causal)
    for _ in range(10):
        again = torch.autograd.grad(ops.attention(*qkv, causal=causal), qkv, grad)
        assert all(torch.equal(x, got["d" + n]) for n, x in zip("qkv", again))
    check(qkv, grad, lengths=[shape[2] - 130 if shape[2] > 130 else 1] * shape[0], causal=causal)
    if causal:
        check(qkv, grad, causal=True, window=shape[2])
        check(qkv, grad, causal=True, start=-3 if shape[1] < 1000 else 1)


def test_gradients_against_differences():
    (q, k, v), grad = make(1, 140, 140, 2, 1, 64, seed=10)
    out = ops.attention(q, k, v)
    grads = torch.autograd.grad(out, (q, k, v), grad)
    for i, g in enumerate(grads):
        step = torch.randn(g.shape, device="cuda", dtype=torch.float64)
        moved = []
        for sign in (1, -1):
            x = [t.detach().double() for t in (q, k, v)]
            x[i] = x[i] + sign * 1e-5 * step
            moved.append((attention64(*x)["o"][0] * grad.double()).sum())
        want = (moved[0] - moved[1]) / 2e-5
        bound = (attention64(q, k, v, grad=grad)[("dq", "dk", "dv")[i]][1] * step.abs()).sum()
        assert abs(float((g.double() * step).sum() - want)) <= float(bound) + 1e-6 * abs(float(want))


def test_the_same_bits_every_time_on_another_stream_and_in_a_graph():
    (q, k, v), grad = make(2, 300, 300, 4, 2, 128, seed=11)
    call = lambda: (lambda o: (o.detach(), *torch.autograd.grad(o, (q, k, v), grad)))(ops.attention(q, k, v))  # noqa: E731
    first = call()
    assert all(torch.equal(a, b) for a, b in zip(first, call()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = call()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, other))
    graphs = []
    for _ in range(2):  # two captures, replayed in turn
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = call()
        graphs.append((g, got))
    for _ in range(2):
        for g, got in graphs:
            for x in got:
                x.zero_()
            g.replay()
            assert all(torch.equal(a, b) for a, b in zip(first, got))
    with torch.no_grad():
        q.mul_(0.5)
    for g, got in graphs:
        g.replay()
    assert all(torch.equal(a, b) for a, b in zip(graphs[0][1], call()))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window", [5, 64, None])
def test_the_same_bits_however_warps_run_ahead(D, window):
    """Many short walks over keys, most of whose tiles are masked for some rows: warps that differ in speed."""
    (q, k, v), grad = make(40, 512, 512, 4, 4, D, seed=12)
    out = ops.attention(q, k, v, window=window)
    first = torch.autograd.grad(out, (q, k, v), grad, retain_graph=True)
    assert all(torch.isfinite(x).all() for x in first)
    for _ in range(60):
        again = torch.autograd.grad(out, (q, k, v), grad, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("shape", [(0, 4, 4, 2, 1, 64), (2, 0, 5, 2, 1, 64), (2, 5, 0, 2, 1, 64)])
def test_nothing_to_attend(shape):
    qkv, grad = make(*shape)
    out = ops.attention(*qkv)
    assert out.shape == qkv[0].shape and not out.any()
    assert all(not g.any() and g.shape == x.shape for g, x in zip(torch.autograd.grad(out, qkv, grad), qkv))


def test_only_some_inputs_want_gradients():
    (q, k, v), grad = make(1, 50, 50, 2, 1, 64)
    full = torch.autograd.grad(ops.attention(q, k, v), (q, k, v), grad)
    for i in range(3):
        x = [t if j == i else t.detach() for j, t in enumerate((q, k, v))]
        assert torch.equal(torch.autograd.grad(ops.attention(*x), x[i], grad)[0], full[i])


def test_second_derivatives_and_tangents_are_refused():
    (q, k, v), _ = make(1, 20, 20, 2, 1, 64)
    (g,) = torch.autograd.grad(ops.attention(q, k, v).float().square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()
    import torch.autograd.forward_ad as fw

    with fw.dual_level(), pytest.raises(NotImplementedError):
        ops.attention(fw.make_dual(q.detach(), torch.ones_like(q)), k.detach(), v.detach())


def test_training_after_a_first_call_in_inference_mode():
    """The word that a kernel's expired wait sets is made by whichever call comes first, also one that keeps nothing for a backward pass."""
    from triune_b200.ops import hybrid

    (q, k, v), grad = make(1, 50, 50, 2, 1, 64)
    want = torch.autograd.grad(ops.attention(q, k, v), (q, k, v), grad)
    kept = dict(hybrid._STATUS)
    hybrid._STATUS.clear()
    try:
        with torch.inference_mode():
            ops.attention(q, k, v)
        out = ops.attention(q, k, v)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, (q, k, v), grad), want))
        out = ops.attention(q, k, v)
        for word in hybrid._STATUS.values():  # what looks at it may write it between the passes
            word.zero_()
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, (q, k, v), grad), want))
    finally:
        hybrid._STATUS.update(kept)


@pytest.mark.parametrize("T,S,H", [(1, 4096, 1), (3, 9000, 2), (200, 200, 200)])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
def test_values_that_are_no_numbers_reach_queries_whose_weight_for_them_is_zero(T, S, H, what):
    """Where keys are split over blocks, a part whose scores are far below the others' counts for nothing, unless its sums are no numbers."""
    (q, k, v), _ = make(1, T, S, H, 1, 64, seed=15, grad=False)
    q[:] = q[:, :1, :1]
    x = q[0, 0, 0].float()
    k[0, : S // 2, 0] = (-300 * 8.0 * x / (x @ x)).bfloat16()
    v[0, 10, 0, 5] = what
    out = ops.attention(q, k, v, query_start=S)
    assert not torch.isfinite(out[..., 5]).any()
    keep = torch.arange(64, device="cuda") != 5
    assert torch.isfinite(out[..., keep]).all()

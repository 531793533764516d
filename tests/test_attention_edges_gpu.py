"""packed_attention on the GPU where it can go wrong."""
import math

import pytest
import torch

from powersgd_b200.ops.attention import packed_attention

pytestmark = pytest.mark.gpu


def _offsets(lengths, first=0):
    return torch.tensor([first + sum(lengths[:i]) for i in range(len(lengths) + 1)], device="cuda", dtype=torch.int32)


def _inputs(tokens, heads, groups, size, dtype, seed=0, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda n: (torch.randn(tokens, n, size, generator=gen, device="cuda") * scale).to(dtype)  # noqa: E731
    return make(heads), make(groups), make(groups), make(heads)


def test_offsets_that_go_down_again_and_again():
    """2^24 and more sequences of 128 tiles each over the same rows: their tiles, more than 2^31, are counted without overflow, and what the grid
    has no room for is left. What such offsets give is not defined, but nothing is written elsewhere."""
    tokens, turns = 2**14, 2**24 + 2**21
    offsets = torch.zeros(2 * turns, device="cuda", dtype=torch.int32)
    offsets[1::2] = tokens
    whole = torch.zeros(3, tokens, 1, 16, device="cuda", dtype=torch.bfloat16)
    q, k, v = whole.unbind(0)
    guard = torch.full((2**26,), 7, device="cuda", dtype=torch.int32)
    packed_attention(q, k, v, offsets)
    torch.cuda.synchronize()
    assert (guard == 7).all() and (whole == 0).all()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("size", [64, 128])
def test_scores_that_are_no_numbers(size, bad, causal):
    """One key of a sequence: positions that see a score of NaN (or +inf, whose softmax is none) give NaN, as the form in torch operations does,
    wherever in a tile the key lies."""
    for place in (0, 1, 2, 16, 17, 40, 123, 124, 127, 128, 130, 250):
        q, k, v, _ = _inputs(300, 2, 1, size, torch.bfloat16, seed=place)
        k[20 + place] = bad if math.isnan(bad) else k[20 + place]
        if math.isinf(bad):
            k[20 + place, 0, 3] = bad
        offsets = torch.tensor([0, 20, 280, 300], device="cuda", dtype=torch.int32)
        got = packed_attention(q, k, v, offsets, causal=causal)
        want = packed_attention(*(x.cpu().float() for x in (q, k, v)), offsets.cpu(), causal=causal)
        assert torch.equal(got.isnan().cpu(), want.isnan()), place
        fine = ~want.isnan()
        assert want.isnan().any() and fine.any()
        # a weight is off by 2^-8 of itself and 2^-12 (its score), the output by half a step, 2^-8
        assert ((got.cpu().float() - want)[fine].abs() <= (2.0**-7 + 2.0**-11) * v.abs().max().item()).all()


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("size", [64, 128])
@pytest.mark.parametrize("until", [128, 150, 256, 300])
def test_scores_of_minus_infinity_come_first(until, size, causal):
    """Keys whose scores are -inf have no weight, also where whole tiles of them come before all others."""
    q, k, v, _ = _inputs(500, 2, 1, size, torch.bfloat16, seed=until)
    q[..., 3] = q[..., 3].abs() + 0.25
    k[:until, :, 3] = -math.inf
    got = packed_attention(q, k, v, _offsets([500]), causal=causal)
    want = packed_attention(*(x.cpu().float() for x in (q, k, v)), _offsets([500]).cpu(), causal=causal)
    assert torch.equal(got.isnan().cpu(), want.isnan()) and want[until:].isfinite().all()
    assert ((got.cpu().float() - want)[until:].abs() <= (2.0**-7 + 2.0**-11) * v.abs().max().item()).all()


def _half_precision(q, k, v, g, offsets, causal=True):
    """float16 gradients against 64 bits. With u = 2^-11 and weights off by E = 2^-12 (test_attention_gpu.py): dS is rounded after it was multiplied with a
    power of two that keeps 2 |dO_i| |V_j| below 2^14, the lengths taken up to twice as long, or with 2^14: its smallest step is
    2^-24 max(|dO_i| |V_j| 2^-11, 2^-14). Roundings of one sum are independent: their squares add up, which is asked of all elements of a head together.
    delta is off by (u + E) P |V| in each element of the output, and moves a whole row of dS."""
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    got = torch.autograd.grad(packed_attention(*leaves, offsets, causal=causal), leaves, g)
    heads, groups, size = q.shape[1], k.shape[1], q.shape[2]
    u, E, c = 2.0**-11, 2.0**-12, 1 / math.sqrt(size)
    ends = offsets.tolist()
    for lo, hi in zip(ends, ends[1:]):
        s = slice(lo, hi)
        for kh in range(groups if hi > lo else 0):
            K, V = k[s, kh].double(), v[s, kh].double()
            of = range(kh * heads // groups, (kh + 1) * heads // groups)
            longest = max(g[s, h].double().norm(dim=1).max().item() for h in of) * V.norm(dim=1).max().item()
            dk, dk2, dv, dv2 = (torch.zeros_like(K) for _ in range(4))
            for h in of:
                Q, G = q[s, h].double(), g[s, h].double()
                S = Q @ K.T * c
                if causal:
                    S = S.masked_fill(torch.ones_like(S, dtype=torch.bool).triu(1), -math.inf)
                P = torch.softmax(S, 1)
                O = P @ V
                dS = P * (G @ V.T - (G * O).sum(1, keepdim=True))
                delta = (G.abs() * ((u + E) * (P @ V.abs()) + 2.0**-25)).sum(1, keepdim=True)
                smooth = E * dS.abs() + 2.0**-17 * P * (G.abs() @ V.abs().T)
                step = lambda length: 2.0**-25 * (length * 2.0**-11).clamp_min(2.0**-14)  # noqa: E731
                w = dS @ K * c
                rounded = (u * dS.abs() + step(G.norm(dim=1, keepdim=True) * V.norm(dim=1).max())) * (P > 0)
                off2 = (rounded**2 + smooth**2) @ (K * c) ** 2 + ((delta * P) @ K.abs() * c) ** 2 + (u * w.abs() + 2.0**-25) ** 2
                _within("dq", got[0][s, h], w, off2)
                dk += dS.T @ Q * c
                rounded = (u * dS.abs() + step(torch.tensor(longest, device=q.device))) * (P > 0)
                dk2 += (rounded**2 + smooth**2).T @ (Q * c) ** 2 + ((delta * P).T ** 2) @ (Q * c) ** 2
                dv += P.T @ G
                dv2 += (((u + E) * P + 2.0**-25) ** 2).T @ G**2
            _within("dk", got[1][s, kh], dk, dk2 + (u * dk.abs() + 2.0**-25) ** 2)
            _within("dv", got[2][s, kh], dv, dv2 + (u * dv.abs() + 2.0**-25) ** 2)
    return got


def _within(name, got, want, off2):
    inside = want.abs() < 2.0**15      # float16 ends at 65504: what lies beyond becomes infinite, as it should
    got, want, off2 = got[inside], want[inside], off2[inside]
    assert got.isfinite().all(), name
    off = ((got.double() - want) ** 2).sum().sqrt().item()
    assert off <= off2.sum().sqrt().item(), (name, off / off2.sum().sqrt().item(), off / want.norm().item())


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("heads, groups, size", [(1, 1, 64), (4, 1, 128), (6, 2, 40)])
@pytest.mark.parametrize("gradients, values", [(2.0**-20, 1.0), (2.0**-14, 1.0), (2.0**-10, 1.0), (1.0, 1.0), (2.0**-10, 2.0**-6), (2.0**8, 2.0**7), (2.0**-14, 2.0**7)])
def test_half_precision_gradients_of_any_size(gradients, values, heads, groups, size, causal):
    """Scores as always, but keys (for dQ) or queries (for dK) of a size that brings the results into float16's range."""
    lengths = [2048, 129, 0, 70, 1, 300]
    times = 2.0 ** max(min(-round(math.log2(gradients * values)), 8), -8)
    for of_k in (times, 1 / times):
        q, k, v, g = _inputs(sum(lengths), heads, groups, size, torch.float16, seed=size)
        _half_precision((q / of_k).half(), (k * of_k).half(), (v * values).half(), (g * gradients).half(), _offsets(lengths), causal)


def test_half_precision_gradients_of_different_sizes():
    """Rows of a gradient that differ by 2^12, and a sequence of zeros: each row of dQ has a power of its own."""
    lengths = [600, 100, 64]
    q, k, v, g = _inputs(sum(lengths), 2, 2, 64, torch.float16)
    g[500] *= 2.0**12
    g[650] *= 2.0**-12
    g[700:] = 0
    got = _half_precision(q, k, v, g, _offsets(lengths))
    assert all((x[700:] == 0).all() for x in got)
    rows = slice(0, 500)      # which do not see the large one
    leaves = [x.detach()[rows].requires_grad_() for x in (q, k, v)]
    want, = torch.autograd.grad(packed_attention(*leaves, _offsets([500])), leaves[:1], g[rows])
    u = 2.0**-11
    size = want.abs().max().item()
    assert ((got[0][rows] - want).abs() <= 64 * u * size).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_half_precision_rows_that_are_no_numbers(bad):
    """They have no say in the powers: queries before them have the gradients that they have without them."""
    q, k, v, g = _inputs(800, 2, 1, 64, torch.float16)
    g *= 2.0**-12
    offsets = _offsets([700, 100])

    def dq():
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        return torch.autograd.grad(packed_attention(*leaves, offsets), leaves[:1], g)[0]

    want = dq()
    g[600] = bad
    v[650] = bad
    got = dq()
    assert torch.equal(got[:512], want[:512]) and torch.equal(got[700:], want[700:])     # (tiles of 128 queries, see the call's notes)


@pytest.mark.parametrize("size, heads, groups", [(16, 1, 1), (128, 2, 1)])
@pytest.mark.parametrize("length, gradients", [(3 * 2**16 + 5, 64.0), (20000, 64.0), (20000, 0.001), (5, 64.0)])
def test_half_precision_weights_of_long_sequences(length, gradients, size, heads, groups):
    """Queries of zeros: all weights are 1 / length, dV is the mean of the gradients. A weight and the result are rounded, 2^-11 each; scores add 2^-12. The
    tensor cores add 16 terms at a time to a sum in 32 bits and may cut what does not fit, 2^-23 of it. All terms are equal and all cuts go one way: n / 16 of
    them, of a sum that is half of the last one on average, make n 2^-28 (twice 196613 terms are 2^-9.4)."""
    q, k, v, _ = _inputs(length, heads, groups, size, torch.float16)
    q.zero_()
    g = torch.full_like(q, gradients)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = packed_attention(*leaves, _offsets([length]), causal=False)
    dv, = torch.autograd.grad(out, leaves[2:], g)
    want = g[0, 0, 0].double() * heads / groups
    off = 2.0**-10 + 2.0**-12 + length * heads / groups * 2.0**-28
    assert ((dv.double() - want).abs() <= off * want).all(), ((dv.double() - want).abs().max() / want).item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths, heads, groups, size", [([700, 300, 24], 4, 2, 64), ([700, 300, 24], 8, 1, 128), ([20] * 40 + [224], 4, 4, 64), ([64] * 16, 2, 1, 16)])
def test_graphs_and_repeats(lengths, heads, groups, size, dtype):
    """The same bits in every run, beside other calls on another stream, and from a graph whose offsets change."""
    q, k, v, g = _inputs(1024, heads, groups, size, dtype)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    offsets = _offsets(lengths)

    def call():
        out = packed_attention(*leaves, offsets)
        return (out.detach(), *torch.autograd.grad(out, leaves, g))

    want = [x.clone() for x in call()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    others = []
    for _ in range(30):
        with torch.cuda.stream(side):
            others.append(call())
        got = call()
        assert all(torch.equal(a, b) for a, b in zip(want, got))
    side.synchronize()
    assert all(torch.equal(a, b) for other in others for a, b in zip(want, other))
    del others, got
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    reverse = _offsets(lengths[::-1])
    offsets.copy_(reverse)
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(call(), got))


def test_half_precision_more_elements_than_thirty_two_bits_count():
    """Rows that begin behind 2^31 elements: the same as those rows by themselves."""
    tokens = 2**20 + 5000
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, g, k, v = (torch.empty(tokens, 16, 128, device="cuda", dtype=torch.float16).normal_(generator=gen) for _ in range(4))
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = packed_attention(*leaves, _offsets([128] * (2**13) + [3000, 2000]))
    got = (out, *torch.autograd.grad(out, leaves, g))
    last = [x.detach()[-5000:].clone().requires_grad_() for x in (q, k, v)]
    want = packed_attention(*last, _offsets([3000, 2000]))
    for a, b in zip(got, (want, *torch.autograd.grad(want, last, g[-5000:]))):
        assert torch.equal(a.detach()[-5000:], b.detach())

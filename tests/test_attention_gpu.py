"""packed_attention on the tensor cores against float64, element by element. Bounds, with u half a step of the 16-bit type:
a score has at most 2^-13 of error (float32 sums of up to 128 products, |s| < 2^6), so a weight is off by 2^-12 of itself, and by u
where it is rounded as an operand; delta takes the rounded output; dS is rounded once; results are rounded once."""
import math

import pytest
import torch

from powersgd_b200.ops.attention import packed_attention

pytestmark = pytest.mark.gpu

E = 2.0**-12


def _offsets(lengths, first=0):
    return torch.tensor([first + sum(lengths[:i]) for i in range(len(lengths) + 1)], device="cuda", dtype=torch.int32)


def _inputs(tokens, heads, groups, size, dtype, seed=0, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    make = lambda n: (torch.randn(tokens, n, size, generator=gen, device="cuda") * scale).to(dtype)  # noqa: E731
    return make(heads), make(groups), make(groups), make(heads)


def _check(q, k, v, g, offsets, causal=True, scale=None, backward=True):
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = packed_attention(*leaves, offsets, causal=causal, scale=scale)
    got = [out.detach(), *(torch.autograd.grad(out, leaves, g) if backward else ())]
    assert [x.dtype for x in got] == [q.dtype] * len(got)
    heads, groups, size = q.shape[1], k.shape[1], q.shape[2]
    c = 1 / math.sqrt(size) if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    least = 0.0 if q.dtype == torch.bfloat16 else 2.0**-25      # float16: half of the smallest step
    want = [torch.zeros(x.shape, dtype=torch.float64, device="cuda") for x in (q, k, v)]
    want.insert(0, torch.zeros(q.shape, dtype=torch.float64, device="cuda"))
    bound = [torch.zeros_like(x) for x in want]
    ends = offsets.tolist()
    for lo, hi in zip(ends, ends[1:]):
        for h in range(heads):
            if hi == lo:
                continue
            s, kh = slice(lo, hi), h // (heads // groups)
            Q, K, V, G = q[s, h].double(), k[s, kh].double(), v[s, kh].double(), g[s, h].double()
            S = Q @ K.T * c
            if causal:
                S = S.masked_fill(torch.ones_like(S, dtype=torch.bool).triu(1), -math.inf)
            P = torch.softmax(S, 1)
            O = P @ V
            off_o = (u + E) * (P @ V.abs()) + u * O.abs()
            want[0][s, h], bound[0][s, h] = O, off_o
            if not backward:
                continue
            dP = G @ V.T
            dS = P * (dP - (G * O).sum(1, keepdim=True))
            off_delta = (G.abs() * off_o).sum(1, keepdim=True) + 2.0**-17 * (G.abs() * O.abs()).sum(1, keepdim=True)
            off_ds = (u + E) * dS.abs() + P * (off_delta + 2.0**-17 * (G.abs() @ V.abs().T)) + least
            want[3][s, kh] += P.T @ G
            bound[3][s, kh] += (u + E) * (P.T @ G.abs())
            want[1][s, h] = dS @ K * c
            bound[1][s, h] = off_ds @ K.abs() * c
            want[2][s, kh] += dS.T @ Q * c
            bound[2][s, kh] += off_ds.T @ Q.abs() * c
    for name, x, w, b in zip(("out", "dq", "dk", "dv"), got, want, bound):
        b = b + (u + E * u) * w.abs() + least + 1e-30
        off = (x.double() - w).abs()
        assert x.isfinite().all(), name
        assert (off <= b).all(), (name, (off / b).max().item(), (off / b).flatten().argmax().item())
    return got


@pytest.mark.parametrize("lengths", [[128], [1], [64], [129], [256], [257], [100, 28], [300, 0, 5, 1]])
@pytest.mark.parametrize("size", [64, 128])
def test_forward(lengths, size):
    q, k, v, g = _inputs(sum(lengths), 2, 2, size, torch.bfloat16)
    _check(q, k, v, g, _offsets(lengths), backward=False)


@pytest.mark.parametrize("lengths", [[128], [1], [64], [129], [256], [257], [100, 28], [300, 0, 5, 1]])
@pytest.mark.parametrize("size", [64, 128])
def test_backward(lengths, size):
    q, k, v, g = _inputs(sum(lengths), 2, 2, size, torch.bfloat16)
    _check(q, k, v, g, _offsets(lengths))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads, groups", [(1, 1), (4, 4), (6, 2), (8, 1)])
@pytest.mark.parametrize("size", [8, 16, 24, 40, 64, 72, 80, 96, 128])
def test_sizes_and_heads(size, heads, groups, dtype):
    lengths = [130, 3, 0, 260, 64]
    q, k, v, g = _inputs(sum(lengths), heads, groups, size, dtype, seed=size)
    _check(q, k, v, g, _offsets(lengths))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("size", [64, 112])
def test_long_and_many(causal, size):
    for lengths in ([1500], [1, 2, 3] * 40, [513, 0, 0, 700, 127, 385], [7] * 100 + [400]):
        q, k, v, g = _inputs(sum(lengths), 4, 2, size, torch.bfloat16, seed=3)
        _check(q, k, v, g, _offsets(lengths), causal=causal, scale=0.2)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("size", [32, 128])
def test_more_sequences_than_lanes(size, causal):
    """Their order is written down first."""
    gen = torch.Generator().manual_seed(5)
    for lengths in ([1] * 33, [0] * 40 + [129] + [5] * 20, torch.randint(0, 400, (70,), generator=gen).tolist(), torch.randint(0, 6, (900,), generator=gen).tolist()):
        q, k, v, g = _inputs(sum(lengths) + 3, 2, 1, size, torch.bfloat16, seed=4)
        got = _check(q, k, v, g, _offsets(lengths), causal=causal)
        assert all((x[sum(lengths):] == 0).all() for x in got)
    q, k, v, _ = _inputs(300, 2, 1, size, torch.bfloat16)
    bad = torch.tensor([0, 250, 20, 300] * 20, device="cuda", dtype=torch.int32)     # overlapping: not defined, but inside
    packed_attention(q, k, v, bad)
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_large_scores(dtype):
    q, k, v, g = _inputs(700, 2, 1, 64, dtype, scale=0.5)
    ramp = torch.linspace(0, 6, 700, device="cuda")[:, None, None]       # maxima that move on from tile to tile
    _check((q + ramp).to(dtype), (k + 0.5 * ramp).to(dtype), v, g, _offsets([500, 200]), scale=1 / 8, backward=False)
    _check((q + ramp.flip(0)).to(dtype), k, v, g, _offsets([700]))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("size", [64, 128])
def test_scores_far_below_zero(size, causal):
    """Weights relative to a row's own sum would be infinite for a score of zero, which a key that does not exist has."""
    for lengths in ([70, 200], [129, 1, 300]):
        q, k, v, g = _inputs(sum(lengths), 2, 1, size, torch.bfloat16, scale=0.25)
        q[..., 0] = 32.0
        k[..., 0] = -32.0
        _check(q, k, v, g, _offsets(lengths), causal=causal, scale=0.5)


def test_views_of_one_projection():
    lengths = [200, 31, 150]
    qkv = torch.randn(sum(lengths), 3, 4, 64, device="cuda").bfloat16()
    g = torch.randn(sum(lengths), 4, 64, device="cuda").bfloat16()
    q, k, v = qkv.unbind(1)
    _check(q, k, v, g, _offsets(lengths))
    leaf = qkv.detach().requires_grad_()
    out = packed_attention(*leaf.unbind(1), _offsets(lengths))
    grad, = torch.autograd.grad(out, leaf, g)
    a, b, c = (x.detach().requires_grad_() for x in (q, k, v))
    want = torch.autograd.grad(packed_attention(a, b, c, _offsets(lengths)), (a, b, c), g)
    assert torch.equal(grad, torch.stack(want, 1))
    # by heads first, odd places, and elements that lie apart: copied
    flip = lambda x: x.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    odd = torch.empty(sum(lengths) * 4 * 64 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(sum(lengths), 4, 64).copy_(k)
    apart = v.repeat_interleave(2, 2)[..., ::2]
    got = _check(flip(q), odd, apart, g.transpose(0, 1).contiguous().transpose(0, 1), _offsets(lengths))
    assert all(torch.equal(x, y) for x, y in zip(got[1:], want))
    one = torch.randn(231, 1, 64, device="cuda").bfloat16()
    _check(one.expand(231, 4, 64), one, one, torch.randn(231, 4, 64, device="cuda").bfloat16(), _offsets([200, 31]))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_rows_outside_may_hold_anything(bad, causal):
    lengths, first = [100, 130, 7, 129], 20
    tokens = first + sum(lengths) + 50
    q, k, v, g = _inputs(tokens, 4, 2, 64, torch.bfloat16)
    offsets = _offsets(lengths, first)
    want = _check(q, k, v, g, offsets, causal=causal)
    for x in (q, k, v, g):
        x[:first] = bad
        x[first + sum(lengths):] = bad
    leaves = [x.detach().requires_grad_() for x in (q, k, v)]
    out = packed_attention(*leaves, offsets, causal=causal)
    got = [out.detach(), *torch.autograd.grad(out, leaves, g)]
    for a, b in zip(want, got):
        assert torch.equal(a, b) and (b[:first] == 0).all() and (b[first + sum(lengths):] == 0).all()
    # another sequence's rows neither
    for x in (q, k, v, g):
        x[first + 100 : first + 230] = bad
    out = packed_attention(*leaves, offsets, causal=causal)
    got = [out.detach(), *torch.autograd.grad(out, leaves, g)]
    for a, b in zip(want, got):
        for lo, hi in ((first, first + 100), (first + 230, first + 366)):
            assert torch.equal(a[lo:hi], b[lo:hi])


def test_bad_offsets_stay_inside():
    q, k, v, g = _inputs(300, 2, 2, 64, torch.bfloat16)
    for bad in ([-5, 100, 9000], [0, 250, 20, 300], [400, 500], [300, 0]):
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        out = packed_attention(*leaves, torch.tensor(bad, device="cuda", dtype=torch.int32))
        torch.autograd.grad(out, leaves, g)
    torch.cuda.synchronize()
    clamped = packed_attention(q, k, v, torch.tensor([-5, 100, 9000], device="cuda", dtype=torch.int32))
    assert torch.equal(clamped, packed_attention(q, k, v, torch.tensor([0, 100, 300], device="cuda", dtype=torch.int32)))


def test_streams_graphs_and_repeats():
    lengths = [700, 300, 24]
    q, k, v, g = _inputs(1024, 4, 2, 64, torch.bfloat16)
    leaves = [x.requires_grad_() for x in (q, k, v)]
    offsets = _offsets(lengths)

    def call():
        out = packed_attention(*leaves, offsets)
        return (out, *torch.autograd.grad(out, leaves, g))

    want = [x.detach().clone() for x in call()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            got = [x.detach() for x in call()]
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    offsets.copy_(_offsets([24, 1000, 0]))       # other lengths: the kernels read them
    graph.replay()
    want = [x.detach().clone() for x in call()]
    assert all(torch.equal(a, b.detach()) for a, b in zip(want, got))


def test_refusals():
    q, k, v, _ = _inputs(10, 2, 2, 64, torch.float32)
    with pytest.raises(TypeError, match="bfloat16"):
        packed_attention(q, k, v, _offsets([10]))
    q, k, v, _ = _inputs(10, 2, 2, 64, torch.bfloat16)
    with pytest.raises(ValueError, match="tensors on"):
        packed_attention(q, k, v, _offsets([10]).cpu())


@pytest.mark.parametrize("heads, size", [(16, 128), (32, 64)])
def test_more_elements_than_thirty_two_bits_count(heads, size):
    """Rows that begin behind 2^31 elements: the same as those rows by themselves."""
    tokens = 2**20 + 5000
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, g = (torch.empty(tokens, heads, size, device="cuda", dtype=torch.bfloat16).normal_(generator=gen) for _ in range(2))
    k, v = (torch.empty(tokens, heads, size, device="cuda", dtype=torch.bfloat16).normal_(generator=gen) for _ in range(2))
    lengths = [128] * (2**13) + [3000, 2000]
    leaves = [x.requires_grad_() for x in (q, k, v)]
    out = packed_attention(*leaves, _offsets(lengths))
    got = (out, *torch.autograd.grad(out, leaves, g))
    last = [x.detach()[-5000:].clone().requires_grad_() for x in (q, k, v)]
    want = packed_attention(*last, _offsets([3000, 2000]))
    for a, b in zip(got, (want, *torch.autograd.grad(want, last, g[-5000:]))):
        assert torch.equal(a.detach()[-5000:], b.detach())


@pytest.mark.parametrize("scale", [2.0**-100, 2.0**-60, 2.0**-12])
def test_small_scales(scale):
    """Scores that hardly differ: the output is near the mean of the values, dV near that of the gradients."""
    q, k, v, g = _inputs(200, 2, 1, 64, torch.bfloat16)
    _check(q, k, v, g, _offsets([200]), False, scale=scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("length, size", [(2, 16), (64, 16), (128, 64), (128, 80), (16, 128)])
def test_short_sequences_lose_little(length, size, dtype):
    """With queries (or keys) of zeros and a power of two of keys the weights are exact: what is left is one rounding of dQ (of dK) and that of dS in
    two 16-bit parts, u^2 < 2^-15 of it (float16: what is lost below its smallest step, 2^-25, besides)."""
    u = torch.finfo(dtype).eps / 2
    heads, tokens = 2, 4 * length
    offsets = _offsets([length] * 4)
    for zero in ("q", "k"):
        q, k, v, g = _inputs(tokens, heads, heads, size, dtype, seed=length)
        (q if zero == "q" else k).zero_()
        leaves = [x.requires_grad_() for x in (q, k, v)]
        got = torch.autograd.grad(packed_attention(*leaves, offsets, causal=False), leaves, g)[0 if zero == "q" else 1]
        Q, K, V, G, got = (x.detach().double().view(4, length, heads, size).transpose(1, 2) for x in (q, k, v, g, got))
        O = V.mean(2, keepdim=True)
        dP = G @ V.transpose(2, 3)
        dS = (dP - (G * O).sum(3, keepdim=True)) / length
        off = 2.0**-15 * dS.abs() + (2.0**-15 * (G.abs() * O.abs()).sum(3, keepdim=True) + 2.0**-17 * (G.abs() @ V.abs().transpose(2, 3))) / length
        off = off + (2.0**-25 if dtype == torch.float16 else 0.0)
        c = 1 / math.sqrt(size)
        if zero == "q":
            want, bound = dS @ K * c, off @ K.abs() * c
        else:
            want, bound = dS.transpose(2, 3) @ Q * c, off.transpose(2, 3) @ Q.abs() * c
        bound = bound + u * (want.abs() + bound) + (2.0**-25 if dtype == torch.float16 else 0.0)
        assert ((got - want).abs() <= bound).all()

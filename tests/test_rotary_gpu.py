"""Heads normed and turned by position on the GPU, through the extension and through Python, and GPT-2 that uses them with clipping and AdamW. Bounds: see
test_rotary_cpu.py."""
import copy
import math

import pytest
import torch
from test_packed_training_cpu import _by_document, _documents
from test_rotary_cpu import (check, check_no_rows_and_no_values, check_offsets, check_one_weight, check_sizes_at_the_border, check_small, check_some_gradients, exact,
                             places, refused, tangents, values)

from powersgd_b200 import AdamW, Config, PowerSGD, clip_grad_norm, optimizer_step
from powersgd_b200.models import GPT2, GPT2Config
from powersgd_b200.ops import host, rotary
from powersgd_b200.ops.attention import packed_attention
from powersgd_b200.ops.rotary import rotate_heads, rotate_projection

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(params=["extension", "python"])
def form(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(rotary, "operators", None)
    else:
        assert host.operators is not None
    return request.param


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("size, rotated", [(8, 8), (16, 16), (24, 8), (32, 32), (40, 40), (64, 64), (64, 32), (64, 0), (72, 40), (80, 80), (96, 48), (128, 128), (136, 136), (256, 256), (256, 64)])
def test_against_64_bits(size, rotated, interleaved, dtype):
    check(values(70, 8, size, dtype, "cuda"), 4, 2, lengths=[33, 0, 31, 1], rotated=rotated, interleaved=interleaved)
    check(values(20, 7, size, dtype, "cuda"), 7, 0, position=torch.randint(-1000, 2**20, (20,), device="cuda"), rotated=rotated, interleaved=interleaved, weight_type=dtype)
    check(values(20, 3, size, dtype, "cuda"), 3, 0, lengths=[20], eps=None, rotated=rotated, interleaved=interleaved)


@pytest.mark.parametrize("heads, keys, values_", [(1, 1, 1), (16, 16, 16), (32, 8, 8), (12, 4, 4), (40, 1, 2), (5, 5, 0), (3, 7, 1)])
@pytest.mark.parametrize("rows", [1, 8, 300])
def test_heads_and_rows(form, rows, heads, keys, values_):
    for dtype, size in ((torch.bfloat16, 64), (torch.float32, 128), (torch.float16, 80)):
        check(values(rows, heads + keys + values_, size, dtype, "cuda"), heads, keys, position=torch.randint(0, 2**20, (rows,), device="cuda", dtype=torch.int32))
        check(values(rows, heads + keys + values_, size, dtype, "cuda"), heads, keys, lengths=[rows // 2, rows - rows // 2], weights=False, rotated=size // 16 * 8)


@pytest.mark.parametrize("rows", [20000])
def test_many_rows(rows):
    """More rows than warps, many to a warp; weights' gradients add up many terms."""
    lengths = [1] * 5000 + [0] * 700 + [17, 983, 7000] + [2] * 3000
    check(values(rows, 6, 64, torch.bfloat16, "cuda"), 3, 2, lengths=lengths)


@pytest.mark.parametrize("heads, keys, values_, size", [(4095, 1, 0, 8), (1, 4000, 95, 256), (2048, 2048, 0, 72)])
@pytest.mark.parametrize("rows", [1, 3, 700])
def test_many_heads(rows, heads, keys, values_, size):
    """Rows that hundreds of warps share."""
    rows = rows if size < 256 or rows < 100 else 70
    check(values(rows, heads + keys + values_, size, torch.float32 if size == 256 else torch.bfloat16, "cuda"), heads, keys, lengths=[rows])


@pytest.mark.parametrize("sequences", [1, 31, 32, 33, 1023, 1024, 1025, 33000])
def test_where_sequences_begin(sequences):
    """Positions by themselves: a pair (1, 0) turned once around in 2^20 positions gives them back."""
    gen = torch.Generator().manual_seed(sequences)
    lengths = torch.where(torch.rand(sequences, generator=gen) < 0.3, 0, torch.randint(0, 8, (sequences,), generator=gen))
    rows = int(lengths.sum()) + 50
    start = 13      # rows before the first
    offsets = torch.cat((torch.zeros(1, dtype=torch.int64), lengths.cumsum(0))) + start
    position = torch.full((rows,), -1)
    for lo, n in zip(offsets.tolist(), lengths.tolist()):
        position[lo : lo + n] = torch.arange(n)
    x = torch.zeros(rows, 1, 8, device="cuda")
    x[:, :, 0] = 1
    z = rotate_heads(x, offsets=offsets.int().cuda(), eps=None, rotated=8)[:, 0].cpu()
    got = torch.where((z == 0).all(1), -1, torch.atan2(z[:, 4], z[:, 0]).round().long() % 7)     # (a radian per position: lengths are below 2 pi + 1)
    want = torch.where(position < 0, -1, torch.atan2(position.double().sin(), position.double().cos()).round().long() % 7)
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", TYPES)
def test_offsets(form, dtype):
    check_offsets("cuda", dtype)


def test_sizes_at_the_border(form):
    check_sizes_at_the_border("cuda")


def test_small(form):
    check_small("cuda")


def test_no_rows_no_values_one_weight(form):
    check_no_rows_and_no_values("cuda")
    check_one_weight("cuda")


@pytest.mark.parametrize("dtype", TYPES)
def test_some_gradients(form, dtype):
    check_some_gradients("cuda", dtype)


def test_positions_far_out():
    far = torch.tensor([0, 1, -1, 2**31 - 1, -(2**31), 2**40 + 12345, 10**15 + 7], device="cuda")
    check(values(7, 2, 64, torch.float32, "cuda"), 2, 0, position=far)
    check(values(7, 2, 64, torch.float32, "cuda"), 2, 0, position=far[:5].int().repeat(2)[:7])


def test_refusals(form):
    for call, error in refused("cuda"):
        with pytest.raises(error):
            call()
    x = torch.randn(6, 4, 16, device="cuda")
    for call in (lambda: rotate_heads(x, positions=torch.arange(6)), lambda: rotate_heads(x, positions=torch.arange(6, device="cuda"), weight=torch.ones(16))):
        with pytest.raises(ValueError, match="tensors on"):
            call()
    with pytest.raises(TypeError, match="float64"):
        rotate_heads(x.double(), positions=torch.arange(6, device="cuda"))
    with pytest.raises(NotImplementedError, match="jit.trace"):
        torch.jit.trace(lambda x, p: rotate_heads(x, positions=p), (x, torch.arange(6, device="cuda")))
    for call in tangents("cuda"):
        with pytest.raises((NotImplementedError, RuntimeError), match="forward-mode"):
            call()
    x.requires_grad_()
    g, = torch.autograd.grad(rotate_heads(x, positions=torch.arange(6, device="cuda")).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.sum().backward()


def test_views_and_layouts(form):
    """Rows and heads that lie elsewhere, elements that are not side by side, tensors that only say that they are negated; gradients of the kind."""
    base = values(30, 12, 64, torch.bfloat16, "cuda")
    at = torch.arange(30, device="cuda")
    want = rotate_heads(base, positions=at)
    wide = torch.zeros(30, 2, 13, 64, device="cuda", dtype=torch.bfloat16)
    wide[:, 1, :12] = base
    odd = torch.zeros(30 * 12 * 64 + 1, device="cuda", dtype=torch.bfloat16)[1:]
    odd.copy_(base.flatten())
    for x in (wide[:, 1, :12], base.transpose(0, 1).contiguous().transpose(0, 1), odd.view(30, 12, 64), base.transpose(1, 2).contiguous().transpose(1, 2), torch._neg_view(-base)):
        assert torch.equal(rotate_heads(x, positions=at), want)
        leaf = x.detach().requires_grad_()
        grad = torch.randn(12, 30, 64, device="cuda").bfloat16().transpose(0, 1)
        got, = torch.autograd.grad(rotate_heads(leaf, positions=at), leaf, grad)
        plain = base.clone().requires_grad_()
        expected, = torch.autograd.grad(rotate_heads(plain, positions=at), plain, grad.contiguous())
        assert torch.equal(got, expected) and got.shape == x.shape
    leaf = base.clone().requires_grad_()
    zeros, = torch.autograd.grad(rotate_heads(leaf, positions=at), leaf, torch._efficientzerotensor(leaf.shape, device="cuda", dtype=torch.bfloat16))
    assert (zeros == 0).all()
    sums, = torch.autograd.grad(rotate_heads(leaf, positions=at).sum(), leaf)       # a gradient whose elements share memory
    assert sums.isfinite().all() and (sums != 0).any()
    strided = torch.stack((at, at + 1), 1)[:, 0]
    assert torch.equal(rotate_heads(base, positions=strided), want)
    weight = torch.stack((torch.ones(64), torch.zeros(64)), 1).cuda()[:, 0]
    assert torch.equal(rotate_heads(base, positions=at, weight=weight), want)


def test_values_are_a_view(form):
    x = values(5, 6, 16, torch.bfloat16, "cuda").requires_grad_()
    v = rotate_projection(x * 1, 2, 2, positions=torch.arange(5, device="cuda"))[2]
    with pytest.raises(RuntimeError, match="view"):
        v.add_(1)
    y = x * 1
    q, k, v = rotate_projection(y, 2, 2, positions=torch.arange(5, device="cuda"))
    with torch.no_grad():
        y.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        q.sum().backward()


def test_the_same_bits_in_every_run():
    x, grad = values(9000, 6, 64, torch.bfloat16, "cuda"), values(9000, 4, 64, torch.bfloat16, "cuda", seed=1)
    results = []
    for _ in range(3):
        leaf, w = x.clone().requires_grad_(), torch.linspace(0.5, 2, 64, device="cuda").requires_grad_()
        q, k, _ = rotate_projection(leaf, 3, 1, offsets=torch.tensor([0, 4000, 8999], dtype=torch.int32, device="cuda"), q_weight=w, k_weight=w)
        results.append((q, k, *torch.autograd.grad((q, k), (leaf, w), (grad[:, :3], grad[:, 3:]))))
    assert all(torch.equal(a, b) for r in results[1:] for a, b in zip(results[0], r))


@pytest.mark.parametrize("which", ["offsets", "positions"])
def test_recorded(form, which):
    """Lengths and positions change between replays; two graphs share nothing."""
    x, grad = values(40, 6, 64, torch.bfloat16, "cuda"), [values(40, 2, 64, torch.bfloat16, "cuda", seed=s) for s in range(3)]
    w = [torch.linspace(0.5, 2, 64, device="cuda"), torch.linspace(2, 0.5, 64, device="cuda")]
    place = {"offsets": torch.tensor([0, 10, 40], dtype=torch.int32, device="cuda"), "positions": torch.arange(40, device="cuda")}[which]

    def step(x, *w):
        leaves = [t.detach().requires_grad_() for t in (x, *w)]
        out = rotate_projection(leaves[0], 2, 2, q_weight=leaves[1], k_weight=leaves[2], **{which: place})
        return [*[t.detach() for t in out], *torch.autograd.grad(out, leaves, grad)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x, *w)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, step(x, *w)))
    for new in ([3, 20, 20], [0, 0, 40], [5, 6, 7]):
        place.copy_(torch.tensor(new) if which == "offsets" else torch.arange(40) * new[1] - new[0])
        x.copy_(values(40, 6, 64, torch.bfloat16, "cuda", seed=sum(new)))
        want = step(x, *w)
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream() for _ in graphs]
        for stream, (graph, _) in zip(streams, graphs):      # at once
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, got in graphs:
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_another_stream(form):
    x, at = values(3000, 24, 64, torch.bfloat16, "cuda"), torch.arange(3000, device="cuda")
    want = rotate_heads(x, positions=at)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device="cuda")
        for _ in range(20):
            big = (big @ big).clamp(-1, 1)
        y = x * 1 + big[0, 0].bfloat16() * 0
        got = rotate_heads(y, positions=at)
    side.synchronize()
    assert torch.equal(got, want)


def test_more_elements_than_31_bits():
    rows = 2**31 // (17 * 128) + 3
    x = torch.zeros(rows, 17, 128, dtype=torch.bfloat16, device="cuda")
    assert x.numel() > 2**31
    pick = [0, 1, rows // 2, rows - 2, rows - 1]
    x[pick] = values(5, 17, 128, torch.bfloat16, "cuda")
    leaf = x.requires_grad_()
    offsets = torch.tensor([0, rows // 3, rows], dtype=torch.int32, device="cuda")
    q, k, v = rotate_projection(leaf, 15, 1, offsets=offsets)
    position = torch.tensor([0, 1, rows // 2 - rows // 3, rows - 2 - rows // 3, rows - 1 - rows // 3], device="cuda")
    small = x.detach()[pick].clone().requires_grad_()
    q2, k2, v2 = rotate_projection(small, 15, 1, positions=position)
    assert torch.equal(q[pick], q2) and torch.equal(k[pick], k2) and torch.equal(v[pick], v2)
    dq, dk, dv = torch.randn_like(q2), torch.randn_like(k2), torch.randn_like(v2)
    want, = torch.autograd.grad((q2, k2, v2), small, (dq, dk, dv))
    grads = []
    for t, g in ((q, dq), (k, dk), (v, dv)):
        full = torch.zeros(t.shape, dtype=t.dtype, device="cuda")
        full[pick] = g
        grads.append(full)
    got, = torch.autograd.grad((q, k, v), leaf, grads)
    assert torch.equal(got[pick], want) and (got[2] == 0).all()


# ---- in a model --------------------------------------------------------------------------------
CONFIG = GPT2Config(vocab_size=1003, n_positions=512, n_embd=128, n_layer=2, n_head=2, rotary=True, qk_norm=True)


def _on_gpu(lengths, rows):
    return [x.cuda() for x in _documents(lengths, rows)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rotary, qk_norm", [(True, True), (True, False), (False, True)])
def test_gpt2_gradients_as_near_to_float32_as_document_by_document(rotary, qk_norm, dtype):
    torch.manual_seed(0)
    model = GPT2(GPT2Config(vocab_size=1003, n_positions=512, n_embd=128, n_layer=2, n_head=2, rotary=rotary, qk_norm=qk_norm)).cuda()
    params = list(model.parameters())
    tokens, targets, offsets = _on_gpu([300, 0, 1, 128, 77], 511)
    want = torch.autograd.grad(_by_document(model, tokens, targets, offsets), params)
    found = {}
    for name, loss in (("packed", lambda: model.loss(tokens, targets, offsets)), ("by document", lambda: _by_document(model, tokens, targets, offsets))):
        with torch.autocast("cuda", dtype):
            value = loss()
        found[name] = torch.autograd.grad(value * 256, params)      # (float16: gradients of means are small)
    for w, a, b in zip(want, found["packed"], found["by document"]):
        off, other = (a / 256 - w).norm(), (b / 256 - w).norm()
        assert off <= 2 * other + 1e-3 * w.norm() + 1e-7      # the same roundings to 16 bits in other places


def test_projection_into_attention_and_back():
    """Rows behind the last sequence hold what is no number, and spoil nothing."""
    lengths, rows = [100, 0, 28, 1], 150
    offsets, position, held = places(lengths, rows, "cuda")
    qkv = values(rows, 12, 64, torch.bfloat16, "cuda")
    w = [torch.linspace(0.8, 1.2, 64, device="cuda").requires_grad_() for _ in range(2)]
    outs = []
    for fill in (0.0, math.nan):
        x = qkv.clone()
        x[~held] = fill
        x.requires_grad_()
        q, k, v = rotate_projection(x, 8, 2, offsets=offsets, q_weight=w[0], k_weight=w[1])
        out = packed_attention(q, k, v, offsets)
        outs.append((out, *torch.autograd.grad(out, (x, *w), torch.ones_like(out))))
    for a, b in zip(*outs):
        assert torch.equal(a, b) and a.isfinite().all()
    wide = exact(qkv[:, :8].double(), position, held, w[0].double(), 1e-6, 10000.0, 64, False)
    assert wide.shape == (rows, 8, 64) and (outs[0][1][~held] == 0).all()


@pytest.mark.parametrize("bits", [8, 32])
def test_recorded_steps_with_clipping_and_adamw(bits):
    """Rotary GPT-2, token log probabilities, clipping, PowerSGD and AdamW as one graph; lengths and tokens change between replays."""
    torch.manual_seed(0)
    first = GPT2(CONFIG).cuda()
    twin = copy.deepcopy(first)
    tokens, targets, offsets = _on_gpu([300, 0, 1, 128, 77], 512)
    batches = [_on_gpu(lengths, 512) for lengths in ([100, 200, 50, 1, 160], [512, 0, 0, 0, 0], [1, 1, 1, 1, 1])]

    def make(model):
        params = list(model.parameters())
        agg = PowerSGD(params, Config(rank=2, min_compression_rate=2, num_iters_per_step=2, start_compressing_after_num_steps=0))
        return params, AdamW(params, lr=torch.tensor(1e-3, device="cuda"), state_bits=bits), agg

    def step(model, params, opt, agg, batch):
        with torch.autocast("cuda", torch.bfloat16, cache_enabled=False):
            loss = model.loss(*batch)
        loss.backward()
        norm = clip_grad_norm(params, 0.05)
        optimizer_step(opt, agg)
        return loss.detach(), norm

    a, b = make(first), make(twin)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for made, model in ((a, first), (b, twin)):
            for _ in range(2):
                step(model, *made, (tokens, targets, offsets))
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded, norm = step(first, *a, (tokens, targets, offsets))
    for batch in batches:
        for x, y in zip((tokens, targets, offsets), batch):
            x.copy_(y)
        graph.replay()
        loss, want = step(twin, *b, batch)
        torch.testing.assert_close(recorded, loss, rtol=1e-2, atol=1e-2)      # bfloat16, sums of embeddings' gradients in another order
        torch.testing.assert_close(norm, want, rtol=5e-2, atol=1e-6)
    torch.cuda.synchronize()
    for p, q in zip(a[0], b[0]):
        assert p.isfinite().all() and (p - q).norm() <= 0.1 * 5e-3 * p.numel() ** 0.5      # a tenth of what five steps can move

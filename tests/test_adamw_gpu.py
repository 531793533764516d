"""AdamW's kernels against the formula in 64 bits. Bounds: m and v have three roundings (2^-24 each) of their terms; an
update has some twelve, two of them in the bias corrections, so 2^-20 of itself; p half a step of its type and one of
float32 besides."""
import copy
import math

import pytest
import torch

from powersgd_b200 import AdamW, Config, PowerSGD, optimizer_step
from powersgd_b200.ops import adamw

pytestmark = pytest.mark.gpu

LR, B1, B2, EPS, WD = 3e-3, 0.9, 0.99, 1e-8, 0.1


def _make(shapes, dtype, bits, device="cuda", seed=0, **more):
    gen = torch.Generator().manual_seed(seed)
    params = [torch.nn.Parameter(torch.randn(s, generator=gen).to(dtype).to(device)) for s in shapes]
    return params, AdamW(params, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=bits, seed=77, **more)


def _grads(params, step, scale=1.0):
    gen = torch.Generator().manual_seed(1000 + step)
    for p in params:
        p.grad = (torch.randn(p.shape, generator=gen) * torch.exp(2 * torch.randn(p.shape, generator=gen)) * scale).to(p.dtype).to(p.device)


def _moments64(opt, p, bits):
    s = opt.state.get(p, {})
    if not s:
        return torch.zeros(p.numel(), dtype=torch.float64, device=p.device), torch.zeros(p.numel(), dtype=torch.float64, device=p.device)
    flat = lambda t: t.as_strided((t.numel(),), (1,)).double()  # noqa: E731
    if bits == 32:
        return flat(s["exp_avg"]).clone(), flat(s["exp_avg_sq"]).clone()
    spread = lambda scale: scale.double().repeat_interleave(256)[: p.numel()]  # noqa: E731
    return flat(s["exp_avg"]) * spread(s["exp_avg_scale"]), (flat(s["exp_avg_sq_root"]) * spread(s["exp_avg_sq_root_scale"])) ** 2


def _one_step(params, opt, step, bits, scale=1.0):
    """A step, and what 64 bits make of the same state."""
    _grads(params, step, scale)
    flat = lambda t: t.detach().as_strided((t.numel(),), (1,)).double()  # noqa: E731
    before = [(flat(p), flat(p.grad), *_moments64(opt, p, bits)) for p in params]
    opt.step()
    t = step + 1
    first = 0
    for p, (old, g, m, v) in zip(params, before):
        mm, vv = B1 * m + (1 - B1) * g, B2 * v + (1 - B2) * g * g
        update = LR / (1 - B1**t) * mm / ((vv / (1 - B2**t)).sqrt() + EPS)
        want = old * (1 - LR * WD) - update
        tiny = torch.finfo(torch.float32).tiny
        m_off = 2.0**-22 * (m.abs() + g.abs()) + tiny
        # (beta2 and 1 - beta2 themselves are float32 numbers)
        update_off = update.abs() * 2.0**-20 + LR / (1 - B1**t) * m_off / ((vv / (1 - B2**t)).sqrt() + EPS)
        # a root below float32's normal range
        update_off = torch.where(vv < 2.0**-120, update.abs() + update_off, update_off)
        got = flat(p)
        off = (got - want).abs()
        # below the smallest normal number half a step is eps / 2 of that (float16: 2^-25)
        bound = want.abs().clamp_min(torch.finfo(p.dtype).smallest_normal) * torch.finfo(p.dtype).eps / 2 + old.abs() * 2.0**-22 + update_off
        assert (off <= bound).all(), ((off / bound).max().item(), p.shape)
        state = opt.state[p]
        assert state["step"].item() == t
        if bits == 32:
            assert ((flat(state["exp_avg"]) - mm).abs() <= m_off).all()
            assert ((flat(state["exp_avg_sq"]) - vv).abs() <= vv * 2.0**-21 + tiny).all()
        elif p.numel():
            blocks = adamw.blocks_of(p.numel())
            words = adamw.random_words(blocks, first, t, 77, p.device)
            for key, x, random, least in (("exp_avg", mm, words & 0xFFFF, False), ("exp_avg_sq_root", vv.sqrt(), words >> 16, True)):
                codes, scale_of = adamw.quantize(adamw._in_blocks(x.float()), random, least)
                got_codes = adamw._in_blocks(state[key].as_strided((p.numel(),), (1,)).float())
                # float32 sums differ in their last bits from 64: a value next to a random border goes the other way, once in 2^12
                differ = got_codes != codes.float()
                assert differ.float().mean() <= 2.0**-10 + 3 / got_codes.numel(), (key, differ.float().mean().item())
                a, b = got_codes[differ], codes.float()[differ]
                assert ((a - b).abs() <= torch.maximum(a.abs(), b.abs()) * 2.0**-2.9 + 2.0**-8.9).all()
                torch.testing.assert_close(state[key + "_scale"], scale_of, rtol=2.0**-21, atol=0)
        first += adamw.blocks_of(p.numel())


SHAPES = [(1,), (255,), (256,), (257,), (3, 5), (64, 64), (4096,), (4097,), (1000, 13), (7, 1023), (0,), (2, 3, 4, 5), (12289,)]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_steps(dtype, bits):
    params, opt = _make(SHAPES, dtype, bits)
    for step in range(4):
        _one_step(params, opt, step, bits, scale=1.0 if step != 2 else 1e-3)


@pytest.mark.parametrize("bits", [32, 8])
def test_long_lists(bits):
    params, opt = _make([(i % 37 + 1, i % 11 + 1) for i in range(900)], torch.float32, bits)   # three launches
    for step in range(2):
        _one_step(params, opt, step, bits)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_views_and_layouts(dtype, bits):
    buffer = torch.randn(20000, device="cuda").to(dtype)
    params = [torch.nn.Parameter(buffer[1:5001].view(50, 100)), torch.nn.Parameter(buffer[5003:9003]), torch.nn.Parameter(buffer[10000:15000].view(100, 50).t()),
              torch.nn.Parameter(torch.randn(8, 6, 3, 3, device="cuda").to(dtype).contiguous(memory_format=torch.channels_last))]
    edges = buffer[[0, 5001, 5002, 9003, 9999, 15000]].clone()
    opt = AdamW(params, lr=LR, betas=(B1, B2), eps=EPS, weight_decay=WD, state_bits=bits, seed=77)
    for step in range(2):
        gen = torch.Generator(device="cuda").manual_seed(step)
        _grads(params, step)
        for p in params:     # gradients laid out like their parameters, and one that is not on a 16-byte boundary
            p.grad = torch.empty_like(p, memory_format=torch.preserve_format).copy_(p.grad)
        old = [p.detach().double().clone() for p in params]
        moments = [[x.view(-1) for x in _moments64(opt, p, bits)] for p in params]
        opt.step()
        for p, o, (m, v) in zip(params, old, moments):
            order = lambda t: t.as_strided((t.numel(),), (1,)).double()  # noqa: E731
            g = order(p.grad)
            mm, vv = B1 * m + (1 - B1) * g, B2 * v + (1 - B2) * g * g
            t = step + 1
            update = LR / (1 - B1**t) * mm / ((vv / (1 - B2**t)).sqrt() + EPS)
            # `o` was cloned with the parameter's strides
            want = order(o) * (1 - LR * WD) - update
            assert ((order(p.detach()) - want).abs() <= want.abs() * torch.finfo(dtype).eps / 2 + order(o).abs() * 2.0**-22 + update.abs() * 2.0**-15 + 1e-9).all()
    assert torch.equal(edges, buffer[[0, 5001, 5002, 9003, 9999, 15000]])
    p = torch.nn.Parameter(torch.zeros(3, 4, device="cuda"))
    p.grad = torch.arange(12.0, device="cuda").view(4, 3).t()      # another order than the parameter's: copied
    opt = AdamW([p], state_bits=bits)
    opt.step()
    assert p[0, 1] != 0 and p[0, 0] == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_mixed_groups_and_missing_gradients(bits):
    a = torch.nn.Parameter(torch.ones(300, device="cuda"))
    b = torch.nn.Parameter(torch.ones(300, device="cuda", dtype=torch.bfloat16))
    c = torch.nn.Parameter(torch.ones(300))
    d = torch.nn.Parameter(torch.ones(300, device="cuda"))
    opt = AdamW([dict(params=[a, b, c]), dict(params=[d], lr=0.0)], lr=0.1, weight_decay=0.0, state_bits=bits)
    for p in (a, b, d):
        p.grad = torch.ones_like(p)
    opt.step()
    c.grad = torch.ones(300)
    opt.step()
    torch.testing.assert_close(a.detach(), torch.full_like(a, 0.8), atol=1e-5 if bits == 32 else 0.04, rtol=0)
    assert (c == 0.9).all() or torch.allclose(c, torch.full((300,), 0.9))
    assert (d == 1).all() and opt.state[c]["step"] == 1 and opt.state[a]["step"] == 2
    torch.testing.assert_close(b.detach().float(), a.detach(), atol=0.01 + (0 if bits == 32 else 0.04), rtol=0)


@pytest.mark.parametrize("bits", [32, 8])
def test_recorded_steps_count_on(bits):
    shapes = [(100, 70), (333,), (5000,)]
    params, opt = _make(shapes, torch.float32, bits)
    twins, plain = _make(shapes, torch.float32, bits)
    lr = torch.tensor(LR, device="cuda")
    opt.param_groups[0]["lr"] = lr
    grads = [torch.zeros_like(p) for p in params]
    for p, g in zip(params, grads):
        p.grad = g
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()            # nothing runs yet: moments and counters are made beside the recording
    for step in range(4):
        _grads(twins, step)
        for g, q in zip(grads, twins):
            g.copy_(q.grad)
        rate = LR * (1 + step)
        lr.fill_(rate)
        plain.param_groups[0]["lr"] = rate
        graph.replay()
        plain.step()
    torch.cuda.synchronize()
    assert opt.state[params[0]]["step"] == 4
    assert all(torch.equal(p, q) for p, q in zip(params, twins))
    assert all(torch.equal(a, b) for p, q in zip(params, twins) for a, b in zip((x.reshape(-1).view(torch.uint8) for x in opt.state[p].values()), (x.reshape(-1).view(torch.uint8) for x in plain.state[q].values())))
    before = [p.detach().clone() for p in params]
    opt.load_state_dict(copy.deepcopy(plain.state_dict()))    # what the graph refers to is kept
    graph.replay()
    torch.cuda.synchronize()
    assert not torch.equal(before[0], params[0]) and params[0].isfinite().all()


def test_same_as_the_cpu_and_repeatable():
    runs = []
    for device in ("cuda", "cuda", "cpu"):
        params, opt = _make([(50, 60), (777,)], torch.float32, 8, device=device)
        for step in range(5):
            _grads(params, step)
            opt.step()
        runs.append([p.detach().cpu() for p in params])
    assert all(torch.equal(a, b) for a, b in zip(runs[0], runs[1]))
    for a, b in zip(runs[0], runs[2]):
        assert ((a - b).abs() > 1e-5).float().mean() < 0.01      # a code that goes the other way moves its element


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_moments_are_those_of_torch_operations_bit_for_bit(dtype, bits):
    """Products and sums rounded one by one: otherwise a code now and then goes the other way, and takes its element with it."""
    p, opt = _make([(300, 1000)], dtype, bits)
    p = p[0]
    q, state = p.detach().clone(), adamw.new_state(p, bits)
    names = adamw.state_names(bits)
    for step in range(3):
        _grads([p], step)
        adamw._step_torch(q, p.grad, [state[n] for n in names], state["step"], bits, LR, B1, B2, EPS, WD, 77, 0)
        opt.step()
        for name in names:
            assert torch.equal(state[name].view(torch.uint8), opt.state[p][name].view(torch.uint8)), name
        assert (p.double() - q.double()).norm() <= 2.0**-20 * q.double().norm() if dtype == torch.float32 else (p != q).float().mean() < 1e-3


def test_infinite_gradients_stay_in_their_block():
    p = torch.nn.Parameter(torch.ones(1024, device="cuda"))
    p.grad = torch.ones(1024, device="cuda")
    p.grad[300] = math.inf
    p.grad[800] = math.nan
    opt = AdamW([p], state_bits=8)
    opt.step()
    p.grad = torch.ones(1024, device="cuda")
    opt.step()
    bad = p.isfinite().logical_not().view(4, 256).any(1)
    assert bad.tolist() == [False, True, False, True]


def test_on_another_stream_and_behind_powersgd():
    torch.manual_seed(0)
    params, opt = _make([(256, 128), (128,), (64, 96)], torch.float32, 32)
    agg = PowerSGD(params, Config(rank=2, min_compression_rate=2, num_iters_per_step=2, start_compressing_after_num_steps=0))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for step in range(3):
            gen = torch.Generator(device="cuda").manual_seed(step)
            for p in params:
                fresh = torch.randn(p.shape, generator=gen, device="cuda")
                p.grad = fresh if p.grad is None else p.grad + fresh
            old = [p.detach().clone() for p in params]
            optimizer_step(opt, agg)
    side.synchronize()
    assert all(opt.state[p]["step"] == 3 for p in params)
    assert all((p - o).abs().max() <= 1.7 * LR for p, o in zip(params, old))   # |m / sqrt(v)| of three steps, decay
    assert params[0].grad.norm() > 0 and params[1].grad.norm() == 0            # residuals


def test_refusals():
    p = torch.nn.Parameter(torch.zeros(8, device="cuda"))
    p.grad = torch.ones(8, device="cuda")
    for lr in (torch.zeros((), device="cuda", dtype=torch.float64),):
        with pytest.raises(ValueError):
            AdamW([p], lr=lr).step()
    opt = AdamW([p])
    opt.step()
    opt.state[p]["exp_avg"] = torch.zeros(9, device="cuda")
    with pytest.raises(ValueError, match="exp_avg"):
        opt.step()
    with pytest.raises(ValueError, match="ticket"):
        adamw.adamw_step([p], [p.grad], [[torch.zeros(8, device="cuda")], [torch.zeros(8, device="cuda")]], [torch.zeros((), device="cuda")], bits=32, lr=0.1,
                         beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0)


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_between_forward_and_backward_is_noticed(bits):
    """The first step goes one by one through Python, the second by the list."""
    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    opt = AdamW([p], state_bits=bits)
    for _ in range(2):
        p.grad = torch.ones_like(p)
        loss = p.square().sum()
        opt.step()
        with pytest.raises(RuntimeError, match="modified by an inplace"):
            loss.backward()


def test_a_recorded_step_keeps_its_learning_rate():
    """A group's learning rate is replaced by another one: the recorded step goes on with the tensor that it was recorded with."""
    p = torch.nn.Parameter(torch.ones(300, device="cuda"))
    opt = AdamW([p], lr=torch.tensor(LR, device="cuda"), weight_decay=0.0)
    p.grad = torch.ones_like(p)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    opt.param_groups[0]["lr"] = 0.5
    others = [torch.full((), 7.0, device="cuda") for _ in range(64)]     # (would take the place of a tensor that is gone)
    graph.replay()
    torch.cuda.synchronize()
    assert (p.detach() - (1 - LR)).abs().max() < 1e-6 and len(others) == 64   # first step: lr m / sqrt(v), both corrected; 1e-8 / |g| less


def test_more_elements_than_thirty_two_bits_count():
    """A tensor of more than 2^31 elements: its end is stepped as the same elements by themselves are."""
    n, tail = 2**31 + 5000, 4096 + 904      # the tail begins a block of 256
    whole = torch.nn.Parameter(torch.empty(n, device="cuda", dtype=torch.bfloat16).normal_())
    part = torch.nn.Parameter(whole.detach()[-tail:].clone())
    gradient = torch.empty(n, device="cuda", dtype=torch.bfloat16).normal_()
    for p in (whole, part):
        p.grad = gradient[-p.numel():].clone() if p is part else gradient
        AdamW([p], lr=LR).step()
    assert torch.equal(whole.detach()[-tail:], part.detach())
    before = whole.detach()[:10].clone()
    AdamW([whole], lr=LR, state_bits=8).step()
    AdamW([part], lr=LR, state_bits=8).step()      # first step: the update uses the moments before they are rounded
    assert torch.equal(whole.detach()[-tail:], part.detach()) and not torch.equal(before, whole.detach()[:10])


@pytest.mark.parametrize("device", ["cuda", "cpu"])
@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_without_elements_make_steps(bits, device):
    params = [torch.nn.Parameter(torch.zeros(0, 4, device=device)) for _ in range(2)]
    opt = AdamW(params, state_bits=bits)
    for _ in range(3):
        for p in params:
            p.grad = torch.zeros_like(p)
        opt.step()
    assert [float(opt.state[p]["step"]) for p in params] == [3, 3]

"""The norm of many gradients and clipping on the GPU, through the extension and through Python. Bounds: see test_grad_norm_cpu.py."""
import math

import pytest
import torch
from test_grad_norm_cpu import SHAPES, TYPES, check, check_counted_twice, check_refusals, exact, layouts, make

from powersgd_b200 import AdamW, AllReduce, Config, PowerSGD, clip_grad_norm, grad_norm, optimizer_step
from powersgd_b200.engine import TrainStep
from powersgd_b200.ops import grad_norm as module
from powersgd_b200.ops import host

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["extension", "python"])
def form(request, monkeypatch):
    if request.param == "python":
        monkeypatch.setattr(module, "operators", None)
    else:
        assert host.operators is not None
    return request.param


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("dtypes", [[t] for t in TYPES] + [TYPES])
@pytest.mark.parametrize("max_norm", [0.0, 0.4, 1e9, math.inf])
def test_against_64_bits(form, dtypes, max_norm, norm_type):
    check(make(SHAPES, dtypes, "cuda"), max_norm, norm_type)


@pytest.mark.parametrize("dtypes", [[t] for t in TYPES] + [TYPES])
@pytest.mark.parametrize("count", [39, 40, 41, 1200, 1201, 2500])
def test_long_lists(count, dtypes):
    check(make([(i % 37, i % 11 + 1) for i in range(count)], dtypes, "cuda"), 0.4)


@pytest.mark.parametrize("full, empty", [(40, 3), (1200, 1), (1200, 1300), (2400, 1), (3, 1300)])
@pytest.mark.parametrize("behind", [True, False])
def test_tensors_without_elements(full, empty, behind):
    shapes = [[(0,)] * empty, [(70, 100)] * full]
    check(make(sum(shapes[::-1] if behind else shapes, []), [torch.float32], "cuda"), 0.4)


@pytest.mark.parametrize("dtype", TYPES)
def test_ends_of_pieces(dtype):
    """Tensors that end around a piece's end, begin anywhere and lie right behind one another; what is between them stays."""
    piece = 16384 // dtype.itemsize
    sizes = [piece - 1, piece, piece + 1, 2 * piece, 2 * piece + 3, 5, 1, piece // 2, 17, 40 * piece + 7, 3]
    gen = torch.Generator(device="cuda").manual_seed(1)
    buffer = torch.randn(sum(sizes) + len(sizes) * 2 + 9, generator=gen, device="cuda").to(dtype)
    before, params, at, gaps = buffer.clone(), [], 1, [0]
    for i, n in enumerate(sizes):
        p = torch.nn.Parameter(torch.zeros(n, dtype=dtype, device="cuda"))
        p.grad = buffer[at : at + n]
        params.append(p)
        at += n
        if i % 2:
            gaps.append(at)
            at += 1
    gaps += list(range(at, buffer.numel()))
    check(params, 0.4)
    assert torch.equal(buffer[gaps], before[gaps]) and not torch.equal(buffer, before)


def test_layouts(form):
    check(layouts("cuda"), 0.4)


def test_refusals(form):
    check_refusals("cuda")
    check_counted_twice("cuda")


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("dtype", TYPES)
def test_what_is_not_finite(dtype, norm_type):
    for bad, place in ((math.nan, 3), (math.inf, 70001), (-math.inf, 0), (-math.nan, 70001)):
        params = make([(70003,), (5, 5)], [dtype], "cuda")
        params[0].grad[place] = bad
        before = [p.grad.clone() for p in params]
        with pytest.raises(RuntimeError, match="norm of the gradients"):
            clip_grad_norm(params, 1.0, norm_type, error_if_nonfinite=True)
        norm = grad_norm(params, norm_type)
        assert all(torch.equal(p.grad.nan_to_num(5.0), b.nan_to_num(5.0)) for p, b in zip(params, before))
        got = clip_grad_norm(params, 1.0, norm_type)
        if math.isnan(bad):
            assert norm.isnan() and got.isnan() and all(p.grad.isnan().all() for p in params)
        else:
            assert norm == math.inf and got == math.inf and params[0].grad[place].isnan()
            assert sum((p.grad == 0).sum() for p in params) == 70003 + 25 - 1


def test_large_and_small_gradients():
    for scale, dtype in ((1e30, torch.float32), (1e-30, torch.float32), (1e30, torch.bfloat16), (1e-30, torch.bfloat16), (1e-7, torch.float16), (1e200, torch.float64)):
        params = make([(5000,), (33, 3)], [dtype], "cuda", scale=scale if dtype != torch.float64 else 1e100)
        norm = exact(params, 2)
        assert abs(grad_norm(params).item() - norm) <= norm * 2.0**-23
        if scale > 1:
            check(params, 0.5 * norm)


def test_the_same_bits_in_every_run():
    results = []
    for _ in range(3):
        params = make([(3000, 1000), (777,)], [torch.float32], "cuda")
        results.append((clip_grad_norm(params, 0.3), *[p.grad for p in params]))
    assert all(torch.equal(a, b) for r in results[1:] for a, b in zip(results[0], r))


def test_more_elements_than_31_bits():
    g = torch.zeros(2**31 + 5, dtype=torch.bfloat16, device="cuda")
    g[[0, 2**30, 2**31 - 1, 2**31, 2**31 + 4]] = 2.0
    p = torch.nn.Parameter(torch.empty(0, dtype=torch.bfloat16, device="cuda"))
    p.data = g.view(-1)
    p.grad = g
    assert clip_grad_norm([p], math.sqrt(5.0)).item() == pytest.approx(math.sqrt(20.0), rel=1e-6)
    assert (g != 0).sum() == 5 and (g[[0, 2**30, 2**31 - 1, 2**31, 2**31 + 4]] == 1).all()


def test_recorded(form):
    """Replays read what lies there now; two graphs recorded from the same gradients share nothing else."""
    params = make(SHAPES, [torch.float32, torch.bfloat16], "cuda")
    fresh = [make(SHAPES, [torch.float32, torch.bfloat16], "cuda", seed=s) for s in range(4)]
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        clip_grad_norm(params, 0.4)
    torch.cuda.synchronize()
    graphs, norms = [], []
    for max_norm in (0.4, 0.1):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norms.append(clip_grad_norm(params, max_norm))
            with pytest.raises(RuntimeError, match="recorded"):
                clip_grad_norm(params, max_norm, error_if_nonfinite=True)
        graphs.append(graph)
    for twin in fresh:
        for graph, norm, max_norm in zip(graphs, norms, (0.4, 0.1)):
            for p, q in zip(params, twin):
                p.grad.copy_(q.grad)
            want = [q.grad.clone() for q in twin]
            for q, w in zip(twin, want):
                q.grad = w.clone()
            expected = clip_grad_norm(twin, max_norm)
            graph.replay()
            assert torch.equal(norm, expected) and all(torch.equal(p.grad, q.grad) for p, q in zip(params, twin))
            for q, w in zip(twin, want):
                q.grad = w


def test_two_streams_at_once(form):
    lists = [make([(2000, 1500), (777,), (33, 3)], [torch.float32], "cuda", seed=s) for s in range(4)]
    want = [exact(params, 2) for params in lists]
    torch.cuda.synchronize()
    streams, norms = [torch.cuda.Stream() for _ in lists], []
    for _ in range(5):
        for stream, params in zip(streams, lists):
            with torch.cuda.stream(stream):
                norms.append(clip_grad_norm(params, 1e9))
    torch.cuda.synchronize()
    assert all(abs(n.item() - want[i % 4]) <= want[i % 4] * 2.0**-23 for i, n in enumerate(norms))


def test_autograd_knows(form):
    p = make([(4,)], TYPES[:1], "cuda")[0]
    x = torch.ones(4, device="cuda", requires_grad=True)
    loss = (x * p.grad).sum()
    grad_norm([p])
    clip_grad_norm([p], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


@pytest.mark.parametrize("graph", [True, False])
def test_train_step_clips(graph):
    """Recorded and eager steps, against the same loop with the library's clipping."""
    def run(own):
        torch.manual_seed(0)
        model = torch.nn.Sequential(torch.nn.Linear(64, 256), torch.nn.Tanh(), torch.nn.Linear(256, 10)).cuda()
        params = list(model.parameters())
        optimizer = torch.optim.SGD(params, lr=0.1, momentum=0.9)
        agg = PowerSGD(params, Config(rank=2, min_compression_rate=2, num_iters_per_step=2, start_compressing_after_num_steps=1))
        gen = torch.Generator(device="cuda").manual_seed(3)
        step = TrainStep(model, torch.nn.functional.cross_entropy, optimizer, agg, cuda_graph=graph, grad_clip=0.05) if own else None
        for _ in range(8):
            x, y = torch.randn(32, 64, device="cuda", generator=gen), torch.randint(0, 10, (32,), device="cuda", generator=gen)
            if own:
                step(x, y)
            else:
                torch.nn.functional.cross_entropy(model(x), y).backward()
                torch.nn.utils.clip_grad_norm_(params, 0.05)
                optimizer_step(optimizer, agg)
        if own and graph:
            assert step._graphs
        return params

    for p, q in zip(run(True), run(False)):
        torch.testing.assert_close(p, q, rtol=1e-4, atol=1e-5)   # float32 sums in other orders through eight steps


def test_lists_that_are_refused_are_clipped_by_the_library():
    from powersgd_b200.ops.grad_norm import clip_for_step

    def lists():
        complex_, cpu = torch.nn.Parameter(torch.zeros(4, dtype=torch.complex64, device="cuda")), make([(4, 6)], TYPES[:1])[0]
        complex_.grad = torch.ones(4, dtype=torch.complex64, device="cuda")
        return [*make([(4, 6)], TYPES[:1], "cuda"), cpu], [*make([(4, 6)], TYPES[:1], "cuda"), complex_], [cpu]

    for ours, theirs in zip(lists(), lists()):
        assert torch.equal(clip_for_step(iter(ours), 0.1), torch.nn.utils.clip_grad_norm_(theirs, 0.1))
        assert all(torch.equal(p.grad, q.grad) for p, q in zip(ours, theirs))


@pytest.mark.parametrize("bits", [8, 32])
def test_with_adamw_behind_an_aggregator(bits):
    torch.manual_seed(0)
    model = torch.nn.Linear(64, 64).cuda()
    params = list(model.parameters())
    optimizer, agg = AdamW(params, lr=1e-2, state_bits=bits), AllReduce()
    for _ in range(3):
        optimizer.zero_grad()
        (100 * model(torch.randn(8, 64, device="cuda")).square().sum()).backward()
        norm = clip_grad_norm(params, 1.0)
        assert norm > 1 and abs(grad_norm(params).item() - 1) <= 1e-5
        optimizer_step(optimizer, agg)
    assert all(p.isfinite().all() for p in params)

"""GPT-2 on packed documents, token log probabilities and AdamW together on the GPU: against document by document through the library's
attention and loss, eagerly and recorded."""
import copy

import pytest
import torch

from powersgd_b200 import AdamW, AllReduce, Config, PowerSGD, optimizer_step
from powersgd_b200.models import GPT2, GPT2Config
from tests.test_packed_training_cpu import _by_document, _documents

pytestmark = pytest.mark.gpu

CONFIG = GPT2Config(vocab_size=1003, n_positions=512, n_embd=128, n_layer=2, n_head=2)


def _on_gpu(lengths, rows):
    return [x.cuda() for x in _documents(lengths, rows)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("config", [GPT2Config.tiny(), CONFIG])
def test_gradients_as_near_to_float32_as_document_by_document(config, dtype):
    torch.manual_seed(0)
    lengths = [9, 0, 1, 60, 17] if config.n_positions == 64 else [300, 0, 1, 128, 77]
    model = GPT2(config).cuda()
    params = list(model.parameters())
    tokens, targets, offsets = _on_gpu(lengths, sum(lengths) + 5)
    want = torch.autograd.grad(_by_document(model, tokens, targets, offsets), params)
    found = {}
    for name, loss in (("packed", lambda: model.loss(tokens, targets, offsets)), ("by document", lambda: _by_document(model, tokens, targets, offsets))):
        with torch.autocast("cuda", dtype):
            value = loss()
        found[name] = torch.autograd.grad(value * 256, params)      # (float16: gradients of means are small)
    for w, a, b in zip(want, found["packed"], found["by document"]):
        off, other = (a / 256 - w).norm(), (b / 256 - w).norm()
        assert off <= 2 * other + 1e-3 * w.norm() + 1e-7      # the same roundings to 16 bits in other places


@pytest.mark.parametrize("bits", [8, 32])
def test_steps_behind_powersgd(bits):
    torch.manual_seed(0)
    model = GPT2(CONFIG).cuda()
    params = list(model.parameters())
    opt = AdamW(params, lr=1e-3, state_bits=bits)
    agg = PowerSGD(params, Config(rank=2, min_compression_rate=2, num_iters_per_step=2, start_compressing_after_num_steps=1))
    for step in range(4):
        tokens, targets, offsets = _on_gpu([300 - 50 * step, 0, 1, 128, 77], 512)
        with torch.autocast("cuda", torch.bfloat16):
            loss = model.loss(tokens, targets, offsets)
        loss.backward()
        optimizer_step(opt, agg)
    assert loss.isfinite() and all(p.isfinite().all() for p in params) and all(opt.state[p]["step"] == 4 for p in params)


@pytest.mark.parametrize("aggregator", ["none", "powersgd"])
@pytest.mark.parametrize("bits", [8, 32])
def test_recorded_steps_with_other_lengths(bits, aggregator):
    """The whole step as one graph; lengths, tokens and learning rate change between replays."""
    torch.manual_seed(0)
    first = GPT2(CONFIG).cuda()
    twin = copy.deepcopy(first)
    tokens, targets, offsets = _on_gpu([300, 0, 1, 128, 77], 512)
    batches = [_on_gpu(lengths, 512) for lengths in ([100, 200, 50, 1, 160], [512, 0, 0, 0, 0], [1, 1, 1, 1, 1])]

    def make(model):
        params = list(model.parameters())
        agg = AllReduce() if aggregator == "none" else PowerSGD(params, Config(rank=2, min_compression_rate=2, num_iters_per_step=2, start_compressing_after_num_steps=0))
        return params, AdamW(params, lr=torch.tensor(1e-3, device="cuda"), state_bits=bits), agg

    def step(model, params, opt, agg, batch):
        if aggregator == "none":
            opt.zero_grad()
        with torch.autocast("cuda", torch.bfloat16, cache_enabled=False):
            loss = model.loss(*batch)
        loss.backward()
        optimizer_step(opt, agg)
        return loss.detach()

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
        recorded = step(first, *a, (tokens, targets, offsets))
    for batch in batches:
        for x, y in zip((tokens, targets, offsets), batch):
            x.copy_(y)
        graph.replay()
        loss = step(twin, *b, batch)
        torch.testing.assert_close(recorded, loss, rtol=1e-2, atol=1e-2)      # bfloat16, sums of embeddings' gradients in another order
    torch.cuda.synchronize()
    assert all(a[1].state[p]["step"] == 5 for p in a[0])
    for p, q in zip(a[0], b[0]):
        assert p.isfinite().all() and (p - q).norm() <= 0.1 * 5e-3 * p.numel() ** 0.5      # a tenth of what five steps can move

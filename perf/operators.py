"""Operators of a language model's training step, as cases that can be timed and checked.

  tokens     `token_log_probs(logits, targets, ...)`: log probabilities of given tokens, with entropy and the
             top alternatives where asked; `train` adds the gradient with respect to the logits
  adamw      `AdamW.step()` over a list of tensors, with moments in 32 bits or in 8
  attention  `packed_attention(q, k, v, offsets)`: causal attention over packed sequences of different lengths,
             grouped heads; `train` adds the gradients of q, k and v

`own` chooses between the package's operators and their plain form in elementary torch operations.
Tensors of an optimizer case live in a few flat buffers, each tensor on a multiple of 256 elements, so that
results can be handed over whole and blocks of 256 of a tensor are blocks of the buffer.

All figures are for one GPU.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 256           # elements that share a scale of an 8-bit moment
LR, BETA1, BETA2, EPS, DECAY, SEED = 1e-3, 0.9, 0.999, 1e-8, 0.01, 1234
MOST_LOGITS = 8192 * 50257
MOST_PARAMS = 355_000_000
MOST_SCORES = 2 * 32 * 8192 * 8192      # of the padded score matrix, all heads
MOST_PAIRS = 32 * (8192**2 + 6144**2) * 128   # sum over heads of length^2 x head size


# ---- the cases -------------------------------------------------------------------------------
def listed():
    return [
        # one decoding step of eight streams: sampled tokens' log probabilities, eight alternatives each
        dict(name="tokens-step", kind="tokens", rows=8, vocab=50257, dtype="bf16", top=8, entropy=True, train=False, temperature=1.0, dead=0, ignored=0.0),
        # perplexity of a window of the recurrent language model: 30 steps x 64 columns
        dict(name="tokens-eval-lstm", kind="tokens", rows=1920, vocab=33278, dtype="f32", top=0, entropy=False, train=False, temperature=1.0, dead=0, ignored=0.0),
        # the loss of GPT-2's training step and its gradient: batch 8 x 1024 positions
        dict(name="tokens-train-gpt2", kind="tokens", rows=8192, vocab=50257, dtype="bf16", top=0, entropy=False, train=True, temperature=1.0, dead=0, ignored=0.0),
        # policy gradients with an entropy bonus: ragged rows, padded vocabulary, temperature, prompt rows ignored
        dict(name="tokens-policy", kind="tokens", rows=1023, vocab=33281, dtype="f16", top=20, entropy=True, train=True, temperature=0.7, dead=3, ignored=0.25),
        # the smallest program: two-layer perceptron, four tensors
        dict(name="adamw-mlp", kind="adamw", shapes="784x256 256 256x10 10", dtype="f32", bits=32, step=3),
        # the recurrent language model: tied embedding, three layers, rows of 650
        dict(name="adamw-lstm", kind="adamw", shapes="lstm", dtype="f32", bits=32, step=1000),
        # moments in 8 bits: odd sizes, parameters in 16 bits
        dict(name="adamw8-odd", kind="adamw", shapes="4*1001x777 3*515x2049 333 1 255 257", dtype="bf16", bits=8, step=17),
        # the largest: 355 M parameters, moments in 8 bits
        dict(name="adamw8-gpt2-medium", kind="adamw", shapes="gpt2-medium", dtype="f32", bits=8, step=250),
        # a few short documents through a small model, one of them empty
        dict(name="attention-short", kind="attention", lengths="1 7 33 64 0 20 3", heads=4, groups=4, size=16, dtype="bf16", train=True),
        # GPT-2 medium's training step with documents packed to 8 x 1024 positions
        dict(name="attention-gpt2-packed", kind="attention", lengths="1024 811 213 1024 640 384 1000 24 1024 77 947 512 512", heads=16, groups=16, size=64, dtype="bf16", train=True),
        # grouped heads, odd lengths, a head size between two tiles
        dict(name="attention-grouped-odd", kind="attention", lengths="333 1 0 1999 129 128 127 640", heads=12, groups=4, size=80, dtype="f16", train=True),
        # two long prompts, four query heads to a key head
        dict(name="attention-long-prompts", kind="attention", lengths="8192 6144", heads=32, groups=8, size=128, dtype="bf16", train=False),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw_tokens(rng):
    vocab = _log(rng, 300, 131072)
    rows = _log(rng, 1, max(2, min(16384, MOST_LOGITS // (2 * vocab))))
    train = rng.random() < 0.6
    return dict(kind="tokens", rows=rows, vocab=vocab, dtype=rng.choice(["f32", "bf16", "bf16", "f16"]), top=rng.choice([0, 0, 0, 1, 5, 8, 20, 32]),
                entropy=rng.random() < 0.5, train=train, temperature=rng.choice([1.0, 1.0, 0.7, 1.3]), dead=rng.choice([0, 0, 1, 40]),
                ignored=rng.choice([0.0, 0.0, 0.3]) if train else 0.0)


def _draw_adamw(rng):
    words, left = [], _log(rng, 20_000, 120_000_000)
    for _ in range(rng.randint(1, 6)):
        n, m = _log(rng, 8, 34000), _log(rng, 8, 5000)
        if rng.random() < 0.5:
            n, m = -(-n // 16) * 16, -(-m // 16) * 16
        count = rng.randint(1, 6)
        while count > 1 and count * n * m > left:
            count -= 1
        if count * n * m > left:
            continue
        left -= count * n * m
        words.append(f"{count}*{n}x{m}")
    words.append(f"{rng.randint(1, 40)}*{_log(rng, 1, 4000)}")
    return dict(kind="adamw", shapes=" ".join(words), dtype=rng.choice(["f32", "f32", "bf16", "f16"]), bits=rng.choice([32, 8]), step=_log(rng, 1, 20000) - 1)


def _draw_attention(rng):
    group = rng.choice([1, 1, 2, 3, 4, 8])
    groups = rng.choice([1, 2, 4, 8])
    heads, size = group * groups, rng.choice([16, 32, 40, 64, 64, 64, 80, 96, 128, 128])
    train = rng.random() < 0.6
    longest = min(_log(rng, 16, 8192), int(math.sqrt(MOST_PAIRS / (heads * size * (4 if train else 1)))))
    scores = pairs = 0
    lengths = []
    for _ in range(rng.randint(1, 24)):
        n = rng.choice([longest, rng.randint(0, longest), rng.randint(0, longest), rng.randint(0, 300)])
        top = max([n] + lengths)
        scores, pairs = heads * (len(lengths) + 1) * top * top, pairs + heads * n * n * size * (4 if train else 1)
        if lengths and (scores > MOST_SCORES // 2 or pairs > MOST_PAIRS):
            break
        lengths.append(n)
    if sum(lengths) == 0:
        lengths.append(rng.randint(1, 100))
    return dict(kind="attention", lengths=" ".join(map(str, lengths)), heads=heads, groups=groups, size=size, dtype=rng.choice(["bf16", "bf16", "f16"]), train=train)


def draw(rng):
    return rng.choice([_draw_tokens, _draw_adamw, _draw_attention])(rng)


# ---- shapes ----------------------------------------------------------------------------------
def _shapes(text):
    if text == "lstm":
        return [(33278, 650)] + 3 * [(2600, 650), (2600, 650), (2600,), (2600,)] + [(33278,)]
    if text == "gpt2-medium":
        w = 1024
        block = [(w,), (w,), (3 * w, w), (3 * w,), (w, w), (w,), (w,), (w,), (4 * w, w), (4 * w,), (w, 4 * w), (w,)]
        return [(50257, w), (1024, w)] + 24 * block + [(w,), (w,)]
    out = []
    for word in text.split():
        count, _, dims = word.rpartition("*")
        out += [tuple(int(d) for d in dims.split("x"))] * int(count or 1)
    return out


def _total(shapes):
    return sum(-(-math.prod(s) // BLOCK) * BLOCK for s in shapes)


def _views(flat, shapes, per=1):
    """The tensors in a flat buffer; `per` = 256: their stretches of a buffer with a value for each block."""
    out, at = [], 0
    for s in shapes:
        n = math.prod(s)
        out.append(flat[at // per : at // per + n].view(s) if per == 1 else flat[at // per : (at + -(-n // BLOCK) * BLOCK) // per])
        at += -(-n // BLOCK) * BLOCK
    return out


def _lengths(case):
    return [int(n) for n in case["lengths"].split()]


# ---- inputs ----------------------------------------------------------------------------------
def _prepare_tokens(case, gen):
    rows, vocab, dtype = case["rows"], case["vocab"], DTYPES[case["dtype"]]
    live = vocab - case["dead"]
    # a few likely words and a long tail, as a trained model's output has
    bias = -torch.log(torch.arange(1, vocab + 1, device="cuda", dtype=torch.float32))
    logits = torch.empty(rows, vocab, device="cuda", dtype=dtype)
    for lo in range(0, rows, 1024):
        part = logits[lo : lo + 1024]
        part.copy_(torch.randn(part.shape, generator=gen, device="cuda") * 2.0 + bias)
    logits[:, live:] = -math.inf   # words that a padded vocabulary does not have
    targets = torch.randint(0, live, (rows,), generator=gen, device="cuda")
    if case["ignored"]:
        targets[torch.rand(rows, generator=gen, device="cuda") < case["ignored"]] = -100
    state = dict(logits=logits, targets=targets)
    if case["train"]:
        logits.requires_grad_()
        state["grad"] = torch.randn(rows, generator=gen, device="cuda") / rows
        state["grad_entropy"] = torch.randn(rows, generator=gen, device="cuda") * (0.01 / rows) if case["entropy"] else None
    return state


def _fp8_blocks(x):
    """Blocks of 256 in 8 bits (nearest), as an earlier step left them: values and scales."""
    blocks = x.view(-1, BLOCK)
    scale = blocks.abs().amax(1) / 448.0
    codes = (blocks / scale.clamp_min(1e-30)[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return codes.view(-1), scale


def _prepare_adamw(case, gen):
    shapes, dtype = _shapes(case["shapes"]), DTYPES[case["dtype"]]
    n = _total(shapes)
    live = torch.zeros(n, device="cuda")
    for view in _views(live, shapes):
        view.fill_(1.0)
    randn = lambda scale: torch.randn(n, generator=gen, device="cuda").mul_(live).mul_(scale)  # noqa: E731
    width = torch.exp(randn(1.0))      # how large an element's gradients usually are
    params, grads = randn(0.02).to(dtype), (randn(1e-3) * width).to(dtype)
    avg, avg_sq = randn(3e-4) * width, (randn(1e-3) * width).square_() * 0.5 + (1e-3 * width).square_() * live * 0.5
    state = dict(shapes=shapes, params=params, grads=grads, bits=case["bits"], step=torch.tensor(float(case["step"]), device="cuda"))
    if case["bits"] == 32:
        state.update(exp_avg=avg, exp_avg_sq=avg_sq)
    else:
        state["exp_avg"], state["exp_avg_scale"] = _fp8_blocks(avg)
        state["exp_avg_sq_root"], state["exp_avg_sq_root_scale"] = _fp8_blocks(avg_sq.sqrt_())
    if own:   # the optimizer that a program keeps, in the middle of a run
        state["optimizer"] = _optimizer(state)
    return state


def _moments(bits):
    return (("exp_avg", 1), ("exp_avg_sq", 1)) if bits == 32 else (("exp_avg", 1), ("exp_avg_scale", BLOCK), ("exp_avg_sq_root", 1), ("exp_avg_sq_root_scale", BLOCK))


def _optimizer(state):
    from powersgd_b200 import AdamW

    params = [torch.nn.Parameter(v) for v in _views(state["params"], state["shapes"])]
    for p, g in zip(params, _views(state["grads"], state["shapes"])):
        p.grad = g
    optimizer = AdamW(params, lr=LR, betas=(BETA1, BETA2), eps=EPS, weight_decay=DECAY, state_bits=state["bits"], seed=SEED)
    for key, per in _moments(state["bits"]):
        for p, v in zip(params, _views(state[key], state["shapes"], per)):
            optimizer.state[p][key] = v
    for p in params:
        optimizer.state[p]["step"] = state["step"].clone()
    return optimizer


def _prepare_attention(case, gen):
    lengths, dtype = _lengths(case), DTYPES[case["dtype"]]
    total, heads, groups, size = sum(lengths), case["heads"], case["groups"], case["size"]
    # one projection gives all three, as a model's does: q, k and v are parts of each row of it
    qkv = torch.randn(total, heads + 2 * groups, size, generator=gen, device="cuda").to(dtype)
    q, k, v = (x.detach() for x in qkv.split([heads, groups, groups], dim=1))
    offsets = torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], device="cuda", dtype=torch.int32)
    state = dict(q=q, k=k, v=v, offsets=offsets, lengths=lengths)
    if case["train"]:
        for x in (q, k, v):
            x.requires_grad_()
        state["grad"] = torch.randn(total, heads, size, generator=gen, device="cuda").to(dtype)
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    state = {"tokens": _prepare_tokens, "adamw": _prepare_adamw, "attention": _prepare_attention}[case["kind"]](case, gen)
    state["case"] = case
    return state


# ---- one pass --------------------------------------------------------------------------------
def _tokens_own(state):
    from powersgd_b200.ops.tokens import token_log_probs

    case = state["case"]
    r = token_log_probs(state["logits"], state["targets"], top=case["top"], entropy=case["entropy"], temperature=case["temperature"])
    out = dict(log_probs=r.log_probs.detach(), entropy=None if r.entropy is None else r.entropy.detach(),
               top_log_probs=None if r.top_log_probs is None else r.top_log_probs.detach(), top_tokens=r.top_tokens)
    if case["train"]:
        outs = [r.log_probs] + ([r.entropy] if case["entropy"] else [])
        out["grad_logits"], = torch.autograd.grad(outs, state["logits"], [state["grad"]] + ([state["grad_entropy"]] if case["entropy"] else []))
    return out


@torch.no_grad()
def _tokens_plain(state):
    case, targets = state["case"], state["targets"]
    z = state["logits"].float()
    top = z.amax(1, keepdim=True)
    d = (z - top) / case["temperature"]
    log_p = d - torch.log(torch.exp(d).sum(1, keepdim=True))
    p = torch.exp(log_p)
    held = targets != -100
    at = targets.clamp_min(0)[:, None]
    out = dict(log_probs=torch.where(held, log_p.gather(1, at)[:, 0], torch.zeros_like(log_p[:, 0])), entropy=None, top_log_probs=None, top_tokens=None)
    if case["entropy"]:
        p_log_p = torch.where(p > 0, p * log_p, torch.zeros_like(p))
        out["entropy"] = -p_log_p.sum(1)
    if case["top"]:
        bits = z.view(torch.int32).to(torch.int64)
        order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)       # as integers, in the order of the numbers
        order = order * 2**20 + (2**20 - 1 - torch.arange(z.shape[1], device=z.device))   # equal ones: the lowest index first
        _, out["top_tokens"] = torch.topk(order, case["top"], dim=1)
        out["top_log_probs"] = log_p.gather(1, out["top_tokens"])
    if case["train"]:
        grad = torch.where(held, state["grad"], torch.zeros_like(state["grad"]))[:, None]
        dz = -p * grad
        dz.scatter_add_(1, at, grad)
        if case["entropy"]:
            dz -= state["grad_entropy"][:, None] * (p_log_p + p * out["entropy"][:, None])
        out["grad_logits"] = (dz / case["temperature"]).to(state["logits"].dtype)
    return out


def _mix(x):
    """The finalizer of MurmurHash3 (32 bits), in integers of 64."""
    x = x ^ (x >> 16)
    x = (x * 0x85EBCA6B) & 0xFFFFFFFF
    x = x ^ (x >> 13)
    x = (x * 0xC2B2AE35) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _random_words(n, step):
    """32 random bits for each element of the flat buffer at this step."""
    key = _mix(SEED ^ _mix(step.to(torch.int64)))
    block = _mix(key ^ torch.arange(n // BLOCK, device=step.device))
    return _mix((block[:, None] + torch.arange(BLOCK, device=step.device)) & 0xFFFFFFFF)


def _round_to_8(x, random, least):
    """Blocks of 256 in e4m3 with a scale each; rounded up with the probability that keeps the mean. What is not
    zero stays above it where `least` says so."""
    most = x.abs().amax(1, keepdim=True)
    live = most >= 2.0**-100
    y = x.abs() * torch.where(live, 448.0 / most, torch.zeros_like(most))
    low = y < 2.0**-6
    t = torch.where(low, y + 2.0**-6, y)      # the steps below 2^-6 are those right above it
    t = ((t.view(torch.int32) + (random * 16 + 8).to(torch.int32)) & ~0xFFFFF).view(torch.float32)
    t = torch.where(low, t - 2.0**-6, t).clamp_max(448.0)
    if least:
        t = torch.where(y > 0, t.clamp_min(2.0**-9), t)
    return torch.copysign(t, x).to(torch.float8_e4m3fn).view(-1), torch.where(live, most / 448.0, torch.zeros_like(most))[:, 0]


@torch.no_grad()
def _adamw_plain(state):
    step = state["step"] + 1
    state["step"].copy_(step)
    g = state["grads"].float()
    if state["bits"] == 32:
        m, v = state["exp_avg"], state["exp_avg_sq"]
    else:
        m = (state["exp_avg"].float().view(-1, BLOCK) * state["exp_avg_scale"][:, None]).view(-1)
        v = (state["exp_avg_sq_root"].float().view(-1, BLOCK) * state["exp_avg_sq_root_scale"][:, None]).view(-1).square()
    m = m * BETA1 + g * (1 - BETA1)
    v = v * BETA2 + g * g * (1 - BETA2)
    first, second = 1 - BETA1 ** step.double(), 1 - BETA2 ** step.double()
    update = m / (v.sqrt() / second.sqrt().float() + EPS) * (LR / first).float()
    state["params"].copy_(state["params"].float() * (1 - LR * DECAY) - update)
    if state["bits"] == 32:
        state["exp_avg"].copy_(m)
        state["exp_avg_sq"].copy_(v)
    else:
        words = _random_words(m.numel(), step)
        for key, x, random, least in (("exp_avg", m, words & 0xFFFF, False), ("exp_avg_sq_root", v.sqrt(), words >> 16, True)):
            codes, scale = _round_to_8(x.view(-1, BLOCK), random, least)
            state[key].copy_(codes)
            state[key + "_scale"].copy_(scale)
    return _adamw_out(state, state["step"])


def _adamw_out(state, step):
    return dict({key: state[key] for key, _ in _moments(state["bits"])}, params=state["params"], step=step)


def _adamw_own(state):
    optimizer = state["optimizer"]
    optimizer.step()
    return _adamw_out(state, optimizer.state[optimizer.param_groups[0]["params"][-1]]["step"])


def _attention_own(state):
    from powersgd_b200.ops.attention import packed_attention

    out = packed_attention(state["q"], state["k"], state["v"], state["offsets"])
    if "grad" not in state:
        return dict(out=out)
    dq, dk, dv = torch.autograd.grad(out, (state["q"], state["k"], state["v"]), state["grad"])
    return dict(out=out.detach(), dq=dq, dk=dk, dv=dv)


@torch.no_grad()
def _attention_plain(state):
    """Sequences padded to the longest, one product for all of them."""
    lengths, offsets, dtype = state["lengths"], state["offsets"], state["q"].dtype
    longest, heads, groups = max(lengths), state["q"].shape[1], state["k"].shape[1]
    place = torch.arange(longest, device="cuda")
    count = (offsets[1:] - offsets[:-1])[:, None]
    held = place < count                                                           # [sequences, longest]
    row = torch.where(held, offsets[:-1, None] + place, torch.zeros_like(place)).to(torch.int64)

    def padded(x, split):   # [sequences, key heads, queries' heads to each, longest, size]
        x = torch.where(held[:, :, None, None], x.float()[row], torch.zeros((), device="cuda"))
        return x.view(*x.shape[:2], groups, split, x.shape[-1]).permute(0, 2, 3, 1, 4)

    def packed(x):
        return x.permute(0, 3, 1, 2, 4).reshape(len(lengths), longest, -1, x.shape[-1])[held].to(dtype)

    q, k, v = padded(state["q"], heads // groups), padded(state["k"], 1), padded(state["v"], 1)
    scale = 1 / math.sqrt(q.shape[-1])
    p = (q * scale) @ k.transpose(-1, -2)
    p.masked_fill_(place > place[:, None], -math.inf)
    p.sub_(p.amax(-1, keepdim=True)).exp_()
    p.div_(p.sum(-1, keepdim=True))
    out = p @ v
    if "grad" not in state:
        return dict(out=packed(out))
    grad = padded(state["grad"], heads // groups)
    dv = (p.transpose(-1, -2) @ grad).sum(2, keepdim=True)
    ds = grad @ v.transpose(-1, -2)
    ds.sub_((grad * out).sum(-1, keepdim=True)).mul_(p)
    dq = ds @ k * scale
    dk = (ds.transpose(-1, -2) @ q).sum(2, keepdim=True) * scale
    return dict(out=packed(out), dq=packed(dq), dk=packed(dk), dv=packed(dv))


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"tokens": _tokens_own, "adamw": _adamw_own, "attention": _attention_own}[kind](state)
    return {"tokens": _tokens_plain, "adamw": _adamw_plain, "attention": _attention_plain}[kind](state)


# ---- what a pass cannot do without -----------------------------------------------------------
def work(case):
    width = {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    if case["kind"] == "tokens":
        n = case["rows"] * case["vocab"]
        passes = 2 if case["train"] else 1           # logits read; their gradient written
        return {"bytes": n * width * passes + case["rows"] * (12 + 12 * case["top"]), "flops": n * (5 + 2 * case["entropy"] + 6 * case["train"])}
    if case["kind"] == "adamw":
        n = sum(math.prod(s) for s in _shapes(case["shapes"]))
        moments = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
        return {"bytes": n * (3 * width + moments), "flops": n * (14 if case["bits"] == 32 else 40)}
    lengths = _lengths(case)
    pairs = sum(n * (n + 1) // 2 for n in lengths) * case["heads"]
    rows = sum(lengths) * case["size"] * width
    once = case["heads"] + 2 * case["groups"]
    if not case["train"]:
        return {"bytes": rows * (once + case["heads"]), "flops": 4 * pairs * case["size"]}
    return {"bytes": rows * (2 * once + 2 * case["heads"]), "flops": 14 * pairs * case["size"]}


# ---- the definition in 64 bits ---------------------------------------------------------------
def _exact_tokens(case, state):
    logits, targets = state["logits"].detach(), state["targets"]
    parts = []
    for lo in range(0, case["rows"], 512):
        z = logits[lo : lo + 512].double()
        t = targets[lo : lo + 512]
        lse = torch.logsumexp(z / case["temperature"], 1, keepdim=True)
        log_p = z / case["temperature"] - lse
        p = log_p.exp()
        keep = t != -100
        one = torch.zeros_like(z)
        one[torch.arange(len(t), device="cuda")[keep], t[keep]] = 1.0
        entropy = torch.special.entr(p).sum(1)
        part = dict(log_probs=torch.where(one > 0, log_p, 0.0).sum(1))
        if case["entropy"]:
            part["entropy"] = entropy
        if case["top"]:
            ranked = torch.sort(z, dim=1, descending=True, stable=True).indices[:, : case["top"]]
            part["top_tokens"], part["top_log_probs"] = ranked, log_p.gather(1, ranked)
        if case["train"]:
            dz = state["grad"][lo : lo + 512, None].double() * (one - p * keep[:, None])
            if case["entropy"]:
                dz = dz + state["grad_entropy"][lo : lo + 512, None].double() * (torch.special.entr(p) - p * entropy[:, None])
            part["grad_logits"] = dz / case["temperature"]
        parts.append(part)
    out = dict(log_probs=None, entropy=None, top_log_probs=None, top_tokens=None)
    out.update({key: torch.cat([part[key] for part in parts]) for key in parts[0]})
    return out


def _exact_round(x, random, least):
    most = x.abs().amax(1, keepdim=True)
    y = torch.where(most > 0, x.abs() / most.clamp_min(1e-300) * 448.0, 0.0)
    spacing = torch.exp2(torch.floor(torch.log2(y.clamp_min(2.0**-6))) - 3)
    code = (torch.floor(y / spacing + (random + 0.5) / 65536) * spacing).clamp_max(448.0)
    if least:
        code = torch.where((y > 0) & (code == 0), 2.0**-9, code)
    return (torch.sign(x) * code).reshape(-1), most[:, 0] / 448.0


def _exact_adamw(case, state):
    t = case["step"] + 1
    g, p = state["grads"].double(), state["params"].double()
    if case["bits"] == 32:
        m, v = state["exp_avg"].double(), state["exp_avg_sq"].double()
    else:
        m = state["exp_avg"].double() * state["exp_avg_scale"].double().repeat_interleave(BLOCK)
        v = (state["exp_avg_sq_root"].double() * state["exp_avg_sq_root_scale"].double().repeat_interleave(BLOCK)) ** 2
    m, v = BETA1 * m + (1 - BETA1) * g, BETA2 * v + (1 - BETA2) * g**2
    p = p - LR * DECAY * p - LR * (m / (1 - BETA1**t)) / ((v / (1 - BETA2**t)).sqrt() + EPS)
    out = dict(params=p, step=torch.tensor(float(t), dtype=torch.float64))
    if case["bits"] == 32:
        return dict(out, exp_avg=m, exp_avg_sq=v)
    words = _random_words(p.numel(), torch.tensor(t, device="cuda"))   # random numbers are inputs
    out["exp_avg"], out["exp_avg_scale"] = _exact_round(m.view(-1, BLOCK), words & 0xFFFF, False)
    out["exp_avg_sq_root"], out["exp_avg_sq_root_scale"] = _exact_round(v.sqrt().view(-1, BLOCK), words >> 16, True)
    return out


def _exact_attention(case, state):
    q, k, v = (state[x].detach().double() for x in "qkv")
    group = case["heads"] // case["groups"]
    out = dict(out=torch.zeros_like(q))
    if case["train"]:
        out.update(dq=torch.zeros_like(q), dk=torch.zeros_like(k), dv=torch.zeros_like(v))
    at = 0
    for n in _lengths(case):
        mask = torch.ones(n, n, dtype=torch.bool, device="cuda").tril()
        for h in range(case["heads"] if n else 0):
            rows, kv = slice(at, at + n), h // group
            s = (q[rows, h] @ k[rows, kv].T / math.sqrt(case["size"])).masked_fill(~mask, -math.inf)
            p = torch.softmax(s, 1)
            o = out["out"][rows, h] = p @ v[rows, kv]
            if case["train"]:
                do = state["grad"][rows, h].double()
                ds = p * (do @ v[rows, kv].T - (do * o).sum(1, keepdim=True)) / math.sqrt(case["size"])
                out["dv"][rows, kv] += p.T @ do
                out["dq"][rows, h] = ds @ k[rows, kv]
                out["dk"][rows, kv] += ds.T @ q[rows, h]
        at += n
    return out


@torch.no_grad()
def exact(case, seed):
    return {"tokens": _exact_tokens, "adamw": _exact_adamw, "attention": _exact_attention}[case["kind"]](case, prepare(case, seed))

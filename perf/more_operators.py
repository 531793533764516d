"""More operators of a language model's training step, as cases that can be timed and checked.

  clip     `clip_grad_norm(parameters, max_norm)`: the norm of all gradients together, and each of them scaled where it is
           too large; with `share` zero `grad_norm(parameters)`, the norm alone
  rotate   `rotate_projection(qkv, heads, key_heads, ...)`: queries and keys of one projection, each head normed and turned by its
           position; `rotate_heads(x, ...)` the same for one tensor of heads; `train` adds the gradients

`own` chooses between the package's operators and their plain form in elementary torch operations.
Gradients of a clip case live in a flat buffer of each type, each on a multiple of 256 elements or, where `packed`, one right
behind another as a communication buffer has them. A program's next call finds other gradients; here the threshold falls by a hundredth from call to call,
so that each has something to scale.

All figures are for one GPU.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
WIDTHS = {"f32": 4, "bf16": 2, "f16": 2}
APART = 256           # elements that gradients begin on multiples of, where they are not packed
USUAL = 1e-3          # magnitude of a gradient
FALL = 0.99           # of the threshold from call to call
EPS, BASE = 1e-6, 10000.0
MOST_HEADS = 14336 * 40 * 128     # elements of queries and keys


# ---- the cases -------------------------------------------------------------------------------
def listed():
    return [
        # the smallest program: two-layer perceptron, four tensors
        dict(name="clip-mlp", kind="clip", shapes="784x256 256 256x10 10", dtype="f32", packed=False, share=0.4, norm=2.0),
        # the recurrent language model, whose task clips at every step: tied embedding, three layers, rows of 650
        dict(name="clip-lstm", kind="clip", shapes="lstm", dtype="f32", packed=False, share=0.4, norm=2.0),
        # gradients in 16 bits that lie one right behind another: odd sizes, odd starts
        dict(name="clip-odd", kind="clip", shapes="4*1001x777 3*515x2049 333 1 255 257", dtype="bf16", packed=True, share=0.4, norm=2.0),
        # matrices in 16 bits beside norms and biases in 32, by their largest element
        dict(name="clip-mixed", kind="clip", shapes="24*1024x1024 24*4096x1024 48*1024 24*4096", dtype="mixed", packed=False, share=0.4, norm=math.inf),
        # the largest: GPT-2 medium
        dict(name="clip-gpt2-medium", kind="clip", shapes="gpt2-medium", dtype="f32", packed=False, share=0.4, norm=2.0),
        # one decoding step of eight streams, far into their documents
        dict(name="rotate-step", kind="rotate", lengths="", rows=8, heads=16, groups=16, size=64, rotated=64, interleaved=False, norm=True, dtype="bf16", train=False, tail=0),
        # GPT-2 medium's training step with documents packed to 8 x 1024 positions
        dict(name="rotate-gpt2-packed", kind="rotate", lengths="1024 811 213 1024 640 384 1000 24 1024 77 947 512 512", rows=0, heads=16, groups=16, size=64, rotated=64,
             interleaved=False, norm=True, dtype="bf16", train=True, tail=0),
        # grouped heads, odd lengths, a part of each head turned in neighbouring pairs, rows behind the last document
        dict(name="rotate-grouped-odd", kind="rotate", lengths="333 1 0 1999 129 128 127 640", rows=0, heads=12, groups=4, size=80, rotated=40, interleaved=True, norm=True,
             dtype="f16", train=True, tail=27),
        # queries of a projection of their own, not normed, in 32 bits: heads alone
        dict(name="rotate-queries", kind="rotate", lengths="511 2048 1000 1", rows=0, heads=12, groups=0, size=64, rotated=64, interleaved=False, norm=False, dtype="f32", train=True, tail=0),
        # two long prompts, four query heads to a key head
        dict(name="rotate-long-prompts", kind="rotate", lengths="8192 6144", rows=0, heads=32, groups=8, size=128, rotated=128, interleaved=False, norm=True, dtype="bf16", train=False, tail=0),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _draw_clip(rng):
    words, left = [], _log(rng, 20_000, 250_000_000)
    for _ in range(rng.randint(1, 8)):
        n, m = _log(rng, 8, 34000), _log(rng, 8, 5000)
        if rng.random() < 0.5:
            n, m = -(-n // 16) * 16, -(-m // 16) * 16
        count = rng.randint(1, 12)
        while count > 1 and count * n * m > left:
            count -= 1
        if count * n * m > left:
            continue
        left -= count * n * m
        words.append(f"{count}*{n}x{m}")
    words.append(f"{rng.randint(1, 200)}*{_log(rng, 1, 4000)}")
    return dict(kind="clip", shapes=" ".join(words), dtype=rng.choice(["f32", "f32", "bf16", "f16", "mixed"]), packed=rng.random() < 0.3,
                share=rng.choice([0.4, 0.4, 0.7, 0.0]), norm=rng.choice([2.0, 2.0, 2.0, math.inf]))


def _draw_rotate(rng):
    group = rng.choice([1, 1, 2, 3, 4, 8])
    groups = rng.choice([0, 1, 2, 4, 8, 12, 16])
    heads = group * groups or rng.randint(1, 40)
    size = rng.choice([16, 32, 40, 64, 64, 64, 72, 80, 96, 128, 128, 128, 256])
    rotated = rng.choice([size, size, size // 16 * 8, size // 4 // 8 * 8])
    train = rng.random() < 0.6
    case = dict(kind="rotate", lengths="", rows=0, heads=heads, groups=groups, size=size, rotated=rotated, interleaved=rng.random() < 0.3, norm=not rotated or rng.random() < 0.8,
                dtype=rng.choice(["bf16", "bf16", "f16", "f32"]), train=train, tail=rng.choice([0, 0, 5, 64]))
    most = MOST_HEADS // ((heads + groups) * size * (4 if train else 1) * WIDTHS[case["dtype"]] // 2)
    if rng.random() < 0.3:
        return dict(case, rows=_log(rng, 1, min(most, 4096)), tail=0)
    longest, lengths = _log(rng, 1, min(most, 8192)), []
    for _ in range(rng.choice([1, 4, 24, 100])):
        n = rng.choice([longest, rng.randint(0, longest), rng.randint(0, longest), rng.randint(0, 300)])
        if sum(lengths) + n + case["tail"] > most:
            break
        lengths.append(n)
    if sum(lengths) == 0:
        lengths.append(1)
    return dict(case, lengths=" ".join(map(str, lengths)))


def draw(rng):
    return rng.choice([_draw_clip, _draw_rotate])(rng)


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


def _layout(case):
    """Of each tensor its shape, its type and where it begins in the flat buffer of that type; and how long these are."""
    out, ends = [], {}
    for shape in _shapes(case["shapes"]):
        dtype = case["dtype"] if case["dtype"] != "mixed" else "f32" if len(shape) == 1 else "bf16"
        at = ends.get(dtype, 0)
        out.append((shape, dtype, at))
        n = math.prod(shape)
        ends[dtype] = at + (n if case["packed"] else -(-n // APART) * APART)
    return out, ends


def _threshold(case):
    """Below the norm of gradients as `_prepare_clip` makes them, at which a program clips."""
    n = sum(math.prod(s) for s in _shapes(case["shapes"]))
    return case["share"] * USUAL * (math.sqrt(n) if case["norm"] == 2.0 else 1.0)


def _lengths(case):
    return [int(n) for n in case["lengths"].split()]


def _rows(case):
    return case["rows"] or sum(_lengths(case)) + case["tail"]


# ---- inputs ----------------------------------------------------------------------------------
def _prepare_clip(case, gen):
    layout, ends = _layout(case)
    flats = {}
    for dtype, n in ends.items():     # most are small, a few are not
        flats[dtype] = torch.randn(n, generator=gen, device="cuda").mul_(torch.exp(torch.randn(n, generator=gen, device="cuda"))).mul_(USUAL).to(DTYPES[dtype])
    views = [flats[dtype][at : at + math.prod(shape)].view(shape) for shape, dtype, at in layout]
    if not case["packed"]:            # what lies between two tensors is nobody's
        for (shape, dtype, at) in layout:
            flats[dtype][at + math.prod(shape) : at + -(-math.prod(shape) // APART) * APART] = 0
    params = []
    for view in views:
        p = torch.nn.Parameter(torch.zeros_like(view))
        p.grad = view
        params.append(p)
    return dict(params=params, views=views, flats=flats, threshold=_threshold(case))


def _prepare_rotate(case, gen):
    rows, heads, groups, size, dtype = _rows(case), case["heads"], case["groups"], case["size"], DTYPES[case["dtype"]]
    values = groups     # as many values as keys
    x = torch.randn(rows, heads + groups + values, size, generator=gen, device="cuda").to(dtype)
    state = dict(x=x, offsets=None, positions=None, q_weight=None, k_weight=None)
    if case["lengths"]:
        lengths = _lengths(case)
        state["offsets"] = torch.tensor([sum(lengths[:i]) for i in range(len(lengths) + 1)], device="cuda", dtype=torch.int32)
    else:
        state["positions"] = torch.randint(0, 2**20, (rows,), generator=gen, device="cuda")
    if case["norm"]:    # parameters of the model, in 32 bits
        for name in ("q_weight", "k_weight") if groups else ("q_weight",):
            state[name] = 1 + 0.2 * torch.randn(size, generator=gen, device="cuda")
    if case["train"]:
        for t in (x, state["q_weight"], state["k_weight"]):
            if t is not None:
                t.requires_grad_()
        # as the attention behind it hands them back
        state["grads"] = [torch.randn(rows, n, size, generator=gen, device="cuda").to(dtype) for n in ((heads, groups, values) if groups else (heads,))]
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    state = {"clip": _prepare_clip, "rotate": _prepare_rotate}[case["kind"]](case, gen)
    state["case"] = case
    return state


# ---- one pass --------------------------------------------------------------------------------
def _clip_own(state):
    case = state["case"]
    if not case["share"]:
        from powersgd_b200 import grad_norm

        return dict(norm=grad_norm(state["params"], norm_type=case["norm"]))
    from powersgd_b200 import clip_grad_norm

    norm = clip_grad_norm(state["params"], state["threshold"], norm_type=case["norm"])
    state["threshold"] *= FALL
    return dict(norm=norm, **state["flats"])


@torch.no_grad()
def _clip_plain(state):
    case = state["case"]
    if case["norm"] == 2.0:
        norm = torch.stack([g.float().square().sum(dtype=torch.float64) for g in state["views"]]).sum().sqrt().float()
    else:
        norm = torch.stack([g.abs().amax().float() for g in state["views"]]).amax()
    if not case["share"]:
        return dict(norm=norm)
    factor = (state["threshold"] / (norm + 1e-6)).clamp(max=1.0)
    for g in state["views"]:
        g.copy_(g.float() * factor)
    state["threshold"] *= FALL
    return dict(norm=norm, **state["flats"])


def _rotate_own(state):
    from powersgd_b200.ops.rotary import rotate_heads, rotate_projection

    case = state["case"]
    options = dict(offsets=state["offsets"], positions=state["positions"], eps=EPS if case["norm"] else None, base=BASE, rotated=case["rotated"], interleaved=case["interleaved"])
    if case["groups"]:
        outs = rotate_projection(state["x"], case["heads"], case["groups"], q_weight=state["q_weight"], k_weight=state["k_weight"], **options)
    else:
        outs = (rotate_heads(state["x"], weight=state["q_weight"], **options),)
    result = {name: t.detach() for name, t in zip("qkv", outs)}
    if case["train"]:
        leaves = {name: t for name, t in (("dx", state["x"]), ("dq_weight", state["q_weight"]), ("dk_weight", state["k_weight"])) if t is not None}
        result.update(zip(leaves, torch.autograd.grad(outs, list(leaves.values()), state["grads"])))
    return result


def _where(state):
    """Positions of the rows and whether they belong to a sequence."""
    if state["offsets"] is None:
        return state["positions"], torch.ones_like(state["positions"], dtype=torch.bool)
    row, offsets = torch.arange(state["x"].shape[0], device="cuda"), state["offsets"].long()
    sequence = (row[:, None] >= offsets).sum(1)          # the first that begins behind the row
    held = (sequence > 0) & (row < offsets[-1])
    return torch.where(held, row - offsets[sequence - 1], torch.zeros_like(row)), held


def _turned(y, cos, sin, rotated, interleaved):
    """The first `rotated` elements of each head turned, pair by pair."""
    if not rotated:
        return y
    part = y[..., :rotated]
    a, b = (part[..., 0::2], part[..., 1::2]) if interleaved else part.chunk(2, dim=-1)
    c, d = a * cos - b * sin, b * cos + a * sin
    part = torch.stack((c, d), -1).flatten(-2) if interleaved else torch.cat((c, d), -1)
    return torch.cat((part, y[..., rotated:]), -1)


@torch.no_grad()
def _rotate_plain(state):
    case = state["case"]
    x, heads, groups, rotated, interleaved = state["x"], case["heads"], case["groups"], case["rotated"], case["interleaved"]
    position, held = _where(state)
    angle = position.double()[:, None] * BASE ** (-torch.arange(0, rotated, 2, device="cuda", dtype=torch.float64) / max(rotated, 1))
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    held = held[:, None, None]
    zero = torch.zeros((), device="cuda")
    result, grads = {}, []
    for i, (name, lo, n, weight) in enumerate((("q", 0, heads, state["q_weight"]), ("k", heads, groups, state["k_weight"]))[: 2 if groups else 1]):
        part = x[:, lo : lo + n].float()
        r = torch.rsqrt(part.square().mean(-1, keepdim=True) + EPS) if case["norm"] else torch.ones((), device="cuda")
        normed = part * r
        y = normed if weight is None else normed * weight
        result[name] = torch.where(held, _turned(y, cos, sin, rotated, interleaved), zero).to(x.dtype)
        if case["train"]:
            dy = torch.where(held, _turned(state["grads"][i].float(), cos, -sin, rotated, interleaved), zero)
            if weight is not None:
                result[f"d{name}_weight"] = (dy * torch.where(held, normed, zero)).sum((0, 1), dtype=torch.float64).to(weight.dtype)
                dy = dy * weight
            if case["norm"]:
                dy = torch.where(held, r * (dy - normed * (dy * normed).mean(-1, keepdim=True)), zero)
            grads.append(dy.to(x.dtype))
    if groups:
        result["v"] = x[:, heads + groups :].detach()
    if case["train"]:
        result["dx"] = torch.cat(grads + state["grads"][2:], 1)
    return result


def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"clip": _clip_own, "rotate": _rotate_own}[kind](state)
    return {"clip": _clip_plain, "rotate": _rotate_plain}[kind](state)


# ---- what a pass cannot do without -----------------------------------------------------------
def work(case):
    if case["kind"] == "clip":
        layout, _ = _layout(case)
        bytes_ = sum(math.prod(shape) * WIDTHS[dtype] for shape, dtype, _ in layout)
        n = sum(math.prod(shape) for shape, _, _ in layout)
        return {"bytes": bytes_ * (2 if case["share"] else 1), "flops": n * (3 if case["share"] else 2)}
    turned, values = case["heads"] + case["groups"], case["groups"]
    n, width = _rows(case) * case["size"], WIDTHS[case["dtype"]]
    if not case["train"]:
        return {"bytes": 2 * n * turned * width, "flops": n * turned * 8}
    # queries and keys in and out; gradients of all three in, that of the projection out
    return {"bytes": n * width * (2 * turned + 2 * (turned + values)), "flops": n * turned * 22}


# ---- the definition in 64 bits ---------------------------------------------------------------
def _exact_clip(case, state):
    parts = [g.flatten().double() for g in state["views"]]
    norm = math.sqrt(math.fsum(float(p @ p) for p in parts)) if case["norm"] == 2.0 else max(float(p.abs().max()) for p in parts)
    out = dict(norm=torch.tensor(norm, dtype=torch.float64))
    if case["share"]:
        factor = min(1.0, state["threshold"] / (norm + 1e-6))
        del parts
        for dtype, flat in state["flats"].items():
            out[dtype] = flat.double() * factor
    return out


def _exact_rotate(case, state):
    """Pairs as complex numbers; gradients by differentiating in 64 bits."""
    heads, groups, size, rotated = case["heads"], case["groups"], case["size"], case["rotated"]
    leaves = {"dx": state["x"]}
    leaves.update((name, state[key]) for name, key in (("dq_weight", "q_weight"), ("dk_weight", "k_weight")) if state[key] is not None)
    leaves = {name: t.detach().double().requires_grad_(case["train"]) for name, t in leaves.items()}
    x, rows = leaves["dx"], _rows(case)
    place, live = torch.zeros(rows, dtype=torch.float64), torch.zeros(rows, dtype=torch.float64)
    if case["lengths"]:
        at = 0
        for n in _lengths(case):
            place[at : at + n], live[at : at + n] = torch.arange(n, dtype=torch.float64), 1.0
            at += n
    else:
        place, live = state["positions"].double(), live + 1.0
    place, live = place.cuda(), live.cuda().view(-1, 1, 1)
    frequency = torch.exp(torch.arange(rotated // 2, dtype=torch.float64, device="cuda") * (-2 / max(rotated, 1) * math.log(BASE)))
    unit = torch.polar(torch.ones(rows, 1, rotated // 2, dtype=torch.float64, device="cuda"), (place[:, None] * frequency)[:, None])
    outs = {}
    with torch.enable_grad():
        for name, lo, n in (("q", 0, heads), ("k", heads, groups)):
            if not n:
                continue
            y = x[:, lo : lo + n]
            if case["norm"]:
                y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / size + EPS) * leaves[f"d{name}_weight"]
            if rotated:
                head = y[..., :rotated]
                pairs = head.unflatten(-1, (-1, 2)) if case["interleaved"] else head.unflatten(-1, (2, -1)).transpose(-1, -2)
                turned = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * unit)
                turned = turned.flatten(-2) if case["interleaved"] else turned.transpose(-1, -2).flatten(-2)
                y = torch.cat((turned, y[..., rotated:]), -1)
            outs[name] = y * live
        if groups:
            outs["v"] = x[:, heads + groups :] * 1.0
        result = {name: t.detach() for name, t in outs.items()}
        if case["train"]:
            result.update(zip(leaves, torch.autograd.grad(list(outs.values()), list(leaves.values()), [g.double() for g in state["grads"]])))
    return result


@torch.no_grad()
def exact(case, seed):
    return {"clip": _exact_clip, "rotate": _exact_rotate}[case["kind"]](case, prepare(case, seed))

"""The operators of a layer around attention, as cases to time: the residual sum with the norm in front of a block
(``residual_norm``), the norm behind it with its gate (``norm_gate``), rotary positions on jagged queries and keys (``rotary``)
and both projections of a gated feed-forward block with activation and product (``gated_linear``); the trained ones with their
backward pass.

The plain forms compute the same from elementary torch operations in 32 bits, gradients by their formulas; ``exact`` takes the
definitions in 64 bits and lets autograd differentiate them.

A case is a dict of plain values.  ``rows`` tokens; ``train`` adds the gradients of every differentiable input, for gradients of
the outputs that ``prepare`` makes.
"""

import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZES = {"bf16": 2, "fp16": 2, "fp32": 4}
_DEVICE = "cuda:0"
_EPSILON = 1e-5

_DEFAULTS = dict(kind="gated_linear", dtype="bf16", train=False, rows=20292, cols=512, inner=2048, bias=True, activation="silu", stream="bf16",
                 scale=False, beta=True, rms=False, groups=1, gate=True, silu=False, residual=False, batch=32, heads=4, heads_k=4, dim=128,
                 rotary=128, interleaved=False, far=0, stretch=1.0)  # fmt: skip


def _case(**values):
    return dict(_DEFAULTS, **values)


def listed():
    return [
        # ---- gated feed-forward: hidden = act(x Wg^T + bg) * (x Wu^T + bu) ----
        # the next token of one user through a small layer: latency
        _case(name="gated-one", rows=1, cols=512, inner=2048, bias=False),
        # the next tokens of a batch of users through a wide layer: bound by the bytes of the weights
        _case(name="gated-batch", dtype="fp16", rows=48, cols=2048, inner=5632, activation="gelu"),
        # histories of a batch read in one call, wide layer: bound by the matrix products
        _case(name="gated-prefill", rows=8191, cols=2048, inner=5632, bias=False),
        # a training step at the token count of the headline batch, with the gradients of x, weights and bias
        _case(name="gated-train", rows=20292, cols=512, inner=2048, train=True),
        # ---- residual sum and norm in front of a block ----
        # one step of decoding for a batch of users
        _case(name="residual-norm-one", kind="residual_norm", rows=64, cols=512),
        # training: the stream in 32 bits, a learnt scale on the block's output
        _case(name="residual-norm-train", kind="residual_norm", rows=20292, cols=512, stream="fp32", scale=True, train=True),
        # inference over odd widths, root mean square
        _case(name="residual-norm-odd", kind="residual_norm", dtype="fp16", stream="fp16", rows=30011, cols=1002, rms=True, beta=False),
        # ---- norm and gate behind attention ----
        # training: a norm per head, the gate not activated yet
        _case(name="norm-gate-heads-train", kind="norm_gate", rows=20292, cols=512, groups=4, silu=True, train=True),
        # inference over long histories: gate, scale and residual in one pass
        _case(name="norm-gate-residual", kind="norm_gate", dtype="fp16", stream="fp16", rows=65536, cols=1024, rms=True, beta=False, residual=True),
        # ---- rotary positions ----
        # single new tokens of users with long histories: latency, and angles far out
        _case(name="rotary-one", kind="rotary", rows=64, batch=64, far=120011),
        # training on the headline batch: queries and keys there, their gradients back
        _case(name="rotary-train", kind="rotary", rows=20292, batch=32, train=True),
        # long chunks in 32 bits: pairs side by side, part of the head, shared keys, stretched positions
        _case(name="rotary-long", kind="rotary", dtype="fp32", rows=65521, batch=8, heads=8, heads_k=2, dim=96, rotary=64, interleaved=True, far=30011,
              stretch=8.0),
    ]  # fmt: skip


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["gated_linear", "gated_linear", "residual_norm", "norm_gate", "rotary"])
    dtype = rng.choice(["bf16", "bf16", "fp16"] if kind == "gated_linear" else ["bf16", "bf16", "fp16", "fp32"])
    case = _case(kind=kind, dtype=dtype, train=rng.random() < 0.4, rows=_log_int(rng, 1, 65536))
    if kind == "gated_linear":
        case.update(cols=8 * _log_int(rng, 8, 512), inner=8 * _log_int(rng, 8, 1024), bias=rng.random() < 0.5,
                    activation=rng.choice(["silu", "silu", "gelu", "sigmoid"]))  # fmt: skip
        while work(case)["flops"] > 3.6e11 or work(case)["bytes"] > 5.2e8:
            case["rows"] = max(1, case["rows"] // 2)
    elif kind == "rotary":
        case["heads_k"] = rng.choice([1, 2, 4, 8])
        case["heads"] = min(16, case["heads_k"] * rng.choice([1, 1, 2, 4]))
        case["dim"] = rng.choice([32, 50, 64, 64, 96, 128, 128, 192, 256])
        case["rotary"] = rng.choice([case["dim"], case["dim"], 2 * rng.randint(1, case["dim"] // 2)])
        case.update(batch=rng.randint(1, max(1, min(256, case["rows"]))), interleaved=rng.random() < 0.5, far=rng.choice([0, _log_int(rng, 100, 1000000)]),
                    stretch=rng.choice([1.0, 1.0, rng.uniform(1.5, 16.0)]))  # fmt: skip
    else:
        case.update(cols=rng.choice([8 * _log_int(rng, 4, 512), _log_int(rng, 30, 4096)]), stream=rng.choice([dtype, "fp32"]),
                    rms=rng.random() < 0.5, beta=rng.random() < 0.5)  # fmt: skip
        if kind == "residual_norm":
            case["scale"] = rng.random() < 0.5
        else:
            case.update(residual=rng.random() < 0.5, gate=rng.random() < 0.85, silu=rng.random() < 0.5)
            case["groups"] = rng.choice([1, 1, rng.choice([g for g in (2, 3, 4, 5, 7, 8, 16) if case["cols"] % g == 0 and case["cols"] > 8 * g] or [1])])
    while work(case)["bytes"] > 5.2e8:
        case["rows"] = max(1, case["rows"] // 2)
    case["batch"] = min(case["batch"], case["rows"])
    return case


# ------------------------------------------------------------------------------------------------------- inputs ----


def _lengths(rng, rows, batch):
    """``rows`` tokens over ``batch`` sequences of one to four parts each, every one with a row at least."""
    parts = [rng.uniform(1.0, 4.0) for _ in range(batch)]
    ends = [0]
    for p in parts:
        ends.append(ends[-1] + p)
    at = [round(e / ends[-1] * (rows - batch)) for e in ends]
    return [b - a + 1 for a, b in zip(at, at[1:])]


def prepare(case, seed):
    rng = random.Random(seed)
    gen = torch.Generator(_DEVICE).manual_seed(seed)
    dtype, stream = _DTYPES[case["dtype"]], _DTYPES[case["stream"]]
    rows, cols, inner, kind = case["rows"], case["cols"], case["inner"], case["kind"]

    def randn(*shape, std=1.0, mean=0.0, to=dtype):
        return torch.randn(*shape, generator=gen, device=_DEVICE).mul_(std).add_(mean).to(to)

    state = dict(case=case)
    if kind == "gated_linear":
        inputs = dict(x=randn(rows, cols), weight=randn(2 * inner, cols, std=cols**-0.5), bias=randn(2 * inner, std=0.1) if case["bias"] else None)
        state["grads"] = [randn(rows, inner)] if case["train"] else []
    elif kind == "residual_norm":
        # a stream grows over the layers, and some of its channels more than others
        size = torch.rand(cols, generator=gen, device=_DEVICE).mul_(3.0).add_(0.5)
        inputs = dict(x=randn(rows, cols), residual=(torch.randn(rows, cols, generator=gen, device=_DEVICE) * size + 0.2).to(stream),
                      gamma=randn(cols, std=0.2, mean=1.0, to=torch.float32), beta=randn(cols, std=0.1, to=torch.float32) if case["beta"] else None,
                      scale=randn(cols, std=0.1, mean=0.5, to=torch.float32) if case["scale"] else None)  # fmt: skip
        state["grads"] = [randn(rows, cols), randn(rows, cols, to=stream)] if case["train"] else []
    elif kind == "norm_gate":
        # what attention without a softmax returns: small, of another size in every row
        size = torch.rand(rows, 1, generator=gen, device=_DEVICE).mul_(0.2).add_(0.05)
        inputs = dict(x=(torch.randn(rows, cols, generator=gen, device=_DEVICE) * size).to(dtype), gate=randn(rows, cols) if case["gate"] else None,
                      gamma=randn(cols, std=0.2, mean=1.0, to=torch.float32), beta=randn(cols, std=0.1, to=torch.float32) if case["beta"] else None,
                      residual=randn(rows, cols, std=2.0, to=stream) if case["residual"] else None)  # fmt: skip
        state["grads"] = [randn(rows, cols, to=stream if case["residual"] else dtype)] if case["train"] else []
    else:
        lengths = _lengths(rng, rows, case["batch"])
        offsets = [0]
        for n in lengths:
            offsets.append(offsets[-1] + n)
        j = torch.arange(case["rotary"] // 2, dtype=torch.float64)
        state.update(frequencies=(10000.0 ** (-2.0 * j / case["rotary"]) / case["stretch"]).to(_DEVICE),
                     seq_offset=torch.tensor(offsets, dtype=torch.int32, device=_DEVICE),
                     start=torch.tensor([rng.randint(0, case["far"]) for _ in lengths], dtype=torch.int32, device=_DEVICE) if case["far"] else None,
                     magnitude=1.0 + 0.1 * math.log(case["stretch"]))  # fmt: skip
        inputs = dict(q=randn(rows, case["heads"], case["dim"]), k=randn(rows, case["heads_k"], case["dim"]))
        state["grads"] = [randn(rows, case["heads"], case["dim"]), randn(rows, case["heads_k"], case["dim"])] if case["train"] else []
    for t in inputs.values():
        if t is not None:
            t.requires_grad_(case["train"])
    state["inputs"] = inputs
    return state


# -------------------------------------------------------------------------------------------------- plain forms ----


def _activation(name, z):
    """An activation and its derivative; gelu by its tanh form."""
    if name == "gelu":
        c = math.sqrt(2.0 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * z * (1 + t), 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    s = torch.sigmoid(z)
    return (s, s * (1 - s)) if name == "sigmoid" else (z * s, s * (1 + z * (1 - s)))


def _float(t):
    return None if t is None else t.detach().float()


def _plain_gated(case, given, grads):
    x, weight, bias = (_float(t) for t in given.values())
    mixed = torch.matmul(x, weight.t())
    if bias is not None:
        mixed = mixed + bias
    g, u = mixed[:, : case["inner"]], mixed[:, case["inner"] :]
    a, slope = _activation(case["activation"], g)
    dtype = given["x"].dtype
    out = [(a * u).to(dtype)]
    if grads:
        dh = grads[0].float()
        d_mixed = torch.cat([dh * u * slope, dh * a], dim=1)
        out += [torch.matmul(d_mixed, weight).to(dtype), torch.matmul(d_mixed.t(), x).to(dtype)]
        if bias is not None:
            out.append(d_mixed.sum(0).to(dtype))
    return out


def _statistics(s, rms):
    """Rows centred and divided by their size, and one over it."""
    if not rms:
        s = s - s.mean(-1, keepdim=True)
    rstd = torch.rsqrt((s * s).mean(-1, keepdim=True) + _EPSILON)
    return s * rstd, rstd


def _norm_gradient(g, n, rstd, rms):
    inner = (g * n).mean(-1, keepdim=True)
    return rstd * (g - n * inner - (0.0 if rms else g.mean(-1, keepdim=True)))


def _plain_residual_norm(case, given, grads):
    x, residual, gamma, beta, scale = (_float(t) for t in given.values())
    s = residual + (x if scale is None else scale * x)
    n, rstd = _statistics(s, case["rms"])
    y = n * gamma
    if beta is not None:
        y = y + beta
    dtype, stream = given["x"].dtype, given["residual"].dtype
    out = [y.to(dtype), s.to(stream)]
    if grads:
        dy, dr = (_float(t) for t in grads)
        ds = dr + _norm_gradient(dy * gamma, n, rstd, case["rms"])
        out += [(ds if scale is None else scale * ds).to(dtype), ds.to(stream), (dy * n).sum(0)]
        if beta is not None:
            out.append(dy.sum(0))
        if scale is not None:
            out.append((ds * x).sum(0))
    return out


def _plain_norm_gate(case, given, grads):
    x, gate, gamma, beta, residual = (_float(t) for t in given.values())
    rows, groups, factor = case["rows"], case["groups"], _factor(case)
    n, rstd = _statistics(x.view(rows, groups, -1), case["rms"])
    flat = n.view(rows, -1)
    m = flat * gamma
    if beta is not None:
        m = m + beta
    a, slope = (None, None) if gate is None else (gate, 1.0) if not case["silu"] else _activation("silu", gate)
    z = m if a is None else m * a
    dtype = given["x"].dtype
    out = [z.to(dtype) if residual is None else (residual + factor * z).to(given["residual"].dtype)]
    if grads:
        d = grads[0].float()
        dz = d if residual is None else factor * d
        dm = dz if a is None else dz * a
        dx = _norm_gradient((dm * gamma).view(rows, groups, -1), n, rstd, case["rms"]).view(rows, -1)
        out.append(dx.to(dtype))
        if gate is not None:
            out.append((dz * m * slope).to(dtype))
        out.append((dm * flat).sum(0))
        if beta is not None:
            out.append(dm.sum(0))
        if residual is not None:
            out.append(grads[0])
    return out


def _factor(case):
    return 0.25 if case["residual"] else 1.0


def _plain_positions(s):
    """The position of every row, in 64 bits."""
    offsets = s["seq_offset"].long()
    row = torch.arange(s["case"]["rows"], device=_DEVICE)
    b = torch.bucketize(row, offsets[1:], right=True)
    position = row - offsets[b]
    return (position if s["start"] is None else position + s["start"].long()[b]).double()


def _plain_rotary(s, tensors, sign):
    case = s["case"]
    angle = _plain_positions(s)[:, None, None] * s["frequencies"]
    cos, sin = (torch.cos(angle) * s["magnitude"]).float(), (torch.sin(angle) * (sign * s["magnitude"])).float()
    out = []
    for t in tensors:
        w = t.detach().float()
        turned, rest = w[..., : case["rotary"]], w[..., case["rotary"] :]
        if case["interleaved"]:
            a, b = turned[..., 0::2], turned[..., 1::2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
        else:
            a, b = turned.chunk(2, dim=-1)
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
        out.append(torch.cat([turned, rest], dim=-1).to(t.dtype))
    return out


def _plain(s):
    case, given, grads = s["case"], s["inputs"], s["grads"]
    if case["kind"] == "rotary":
        return _plain_rotary(s, given.values(), 1.0) + (_plain_rotary(s, grads, -1.0) if grads else [])
    form = {"gated_linear": _plain_gated, "residual_norm": _plain_residual_norm, "norm_gate": _plain_norm_gate}[case["kind"]]
    return form(case, given, grads)


# -------------------------------------------------------------------------------------------------------- calls ----


def _package():
    if "ops_rec" not in sys.modules:
        sys.path.insert(0, os.path.join(os.getcwd(), "ops-rec_amd"))
        import ops_rec  # noqa: F401
    return sys.modules["ops_rec"].ascendc


def _own(s):
    case, g = s["case"], s["inputs"]
    ops = _package()
    if case["kind"] == "gated_linear":
        # (the projections are kept for the backward pass where there is one)
        out = ops.activation.gated_linear(g["x"], g["weight"], g["bias"], case["activation"], case["train"])[:1]
    elif case["kind"] == "residual_norm":
        out = ops.activation.residual_norm(g["x"], g["residual"], g["gamma"], g["beta"], g["scale"], _EPSILON, case["rms"])
    elif case["kind"] == "norm_gate":
        out = [ops.activation.norm_gate(g["x"], g["gate"], g["gamma"], g["beta"], g["residual"], _factor(case), case["groups"], _EPSILON, case["rms"],
                                        case["silu"])]  # fmt: skip
    else:
        out = ops.attention.rotary(g["q"], g["k"], s["frequencies"], s["seq_offset"], s["start"], None, case["interleaved"], s["magnitude"])
    out = list(out)
    if case["train"]:
        wanted = [t for t in g.values() if t is not None]
        out += torch.autograd.grad(out, wanted, s["grads"])
    return [t.detach() for t in out]


def run(state):
    return _own(state) if own else _plain(state)


# --------------------------------------------------------------------------------------------------------- work ----


def work(case):
    rows, cols, inner, size, stream = case["rows"], case["cols"], case["inner"], _SIZES[case["dtype"]], _SIZES[case["stream"]]
    train, kind = case["train"], case["kind"]
    if kind == "gated_linear":
        weights = 2 * inner * (cols + (1 if case["bias"] else 0))
        moved = rows * (cols + inner) + weights
        if train:  # the gradient of hidden in, of x, weights and bias out
            moved += rows * (cols + inner) + weights
        return {"bytes": float(moved * size), "flops": 4.0 * rows * inner * cols * (3 if train else 1)}
    if kind == "rotary":
        moved = rows * (case["heads"] + case["heads_k"]) * case["dim"]
        turned = rows * (case["heads"] + case["heads_k"]) * case["rotary"]
        return {"bytes": 2.0 * moved * size * (2 if train else 1), "flops": 3.0 * turned * (2 if train else 1)}
    vectors = 4 * cols * (1 + case["beta"] + (case["scale"] if kind == "residual_norm" else 0)) * (2 if train else 1)
    if kind == "residual_norm":
        each = 2 * size + 2 * stream  # x, residual in; y, r out
        if train:  # their gradients
            each *= 2
        return {"bytes": float(rows * cols * each + vectors), "flops": 10.0 * rows * cols * (3 if train else 1)}
    tensors = size * (1 + case["gate"])
    each = tensors + (2 * stream if case["residual"] else size)
    if train:  # the gradient of the output in, those of x and gate out; that of the residual is the output's own
        each += tensors + (stream if case["residual"] else size)
    return {"bytes": float(rows * cols * each + vectors), "flops": 12.0 * rows * cols * (3 if train else 1)}


# -------------------------------------------------------------------------------------------------------- exact ----


def exact(case, seed):
    s = prepare(case, seed)
    given = {name: None if t is None else t.detach().double().requires_grad_(case["train"]) for name, t in s["inputs"].items()}
    with torch.enable_grad():
        if case["kind"] == "gated_linear":
            projections = torch.nn.functional.linear(given["x"], given["weight"], given["bias"]).view(case["rows"], 2, case["inner"])
            gate = projections[:, 0]
            if case["activation"] == "gelu":
                gate = gate * torch.sigmoid(math.sqrt(8.0 / math.pi) * (gate + 0.044715 * gate**3))  # (1 + tanh(x)) / 2 = sigmoid(2 x)
            else:
                gate = gate.sigmoid() * (gate if case["activation"] == "silu" else 1.0)
            out = [gate * projections[:, 1]]
        elif case["kind"] == "residual_norm":
            scale = 1.0 if given["scale"] is None else given["scale"]
            r = given["x"] * scale + given["residual"]
            out = [_exact_norm(r, case["rms"]) * given["gamma"] + (0.0 if given["beta"] is None else given["beta"]), r]
        elif case["kind"] == "norm_gate":
            parts = given["x"].unflatten(1, (case["groups"], case["cols"] // case["groups"]))
            z = _exact_norm(parts, case["rms"]).flatten(1) * given["gamma"] + (0.0 if given["beta"] is None else given["beta"])
            if given["gate"] is not None:
                z = z * given["gate"] / (1.0 + torch.exp(-given["gate"])) if case["silu"] else z * given["gate"]
            out = [z if given["residual"] is None else given["residual"] + _factor(case) * z]
        else:
            out = [_exact_rotary(s, t) for t in given.values()]
        if case["train"]:
            wanted = [t for t in given.values() if t is not None]
            out += torch.autograd.grad(out, wanted, [t.double() for t in s["grads"]])
    return [t.detach() for t in out]


def _exact_norm(t, rms):
    if rms:
        return t / (t.square().mean(-1, keepdim=True) + _EPSILON).sqrt()
    return (t - t.mean(-1, keepdim=True)) / (t.var(-1, unbiased=False, keepdim=True) + _EPSILON).sqrt()


def _exact_rotary(s, t):
    """Pairs as complex numbers, turned by e^(i position frequency), sequence by sequence."""
    case, half = s["case"], s["case"]["rotary"] // 2
    offsets = s["seq_offset"].tolist()
    starts = [0] * case["batch"] if s["start"] is None else s["start"].tolist()
    place = torch.cat([torch.arange(b - a, device=_DEVICE, dtype=torch.float64) + p for a, b, p in zip(offsets, offsets[1:], starts)])
    turn = torch.polar(torch.full((case["rows"], 1, half), s["magnitude"], dtype=torch.float64, device=_DEVICE),
                       (place[:, None] * s["frequencies"])[:, None])  # fmt: skip
    front, rest = t.split([case["rotary"], case["dim"] - case["rotary"]], dim=-1)
    pairs = front.unflatten(-1, (half, 2)) if case["interleaved"] else front.unflatten(-1, (2, half)).transpose(-1, -2)
    turned = torch.view_as_real(torch.complex(pairs[..., 0], pairs[..., 1]) * turn)
    turned = turned.flatten(-2) if case["interleaved"] else turned.transpose(-1, -2).flatten(-2)
    return torch.cat([turned, rest], dim=-1)

"""A dense layer as one product and the optimiser step behind it: what they are measured on.

``linear``  ``residual + dropout(act(x @ weight.T + bias))`` over the nodes' features, forward, or forward and backward
            (gradients of the features, the weight and the bias; a residual's gradient is the incoming one).
``adamw``   one AdamW step over all of a model's tensors, the moments held in 32 bits, or in 8 with a scale for each block
            of 256 elements and stochastic rounding; with or without clipping by the norm of all gradients.

``run`` computes them with elementary torch operations, or with the package's own operators where ``own`` is set.
A training case of ``linear`` has no ReLU: the gradient of one jumps at its border, where 32 and 64 bits may fall on
either side.
"""
import math

import torch

own = False

NODES = 325557         # nodes of the benchmark's web graph
MANY_NODES = 2450000   # nodes of the benchmark's cluster workload
CLASSES = 47           # classes of the benchmark's models
BETAS = (0.9, 0.999)
EPS = 1e-8
DECAY = 0.01
RATE = 1e-3
BLOCK = 256            # elements that share a scale
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LOW = 0xFFFFFFFF       # the low 32 bits of a word
TENSOR_KEY = 0x9E3779B97F4A7C15  # what the key of a tensor's random words moves on by from tensor to tensor,
STEP_KEY = 0xD1342543DE82EF95    # and from step to step


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _linear(rows, inner, outer, dtype, train=False, relu=False, p=0.0, residual=False):
    return {"op": "linear", "rows": rows, "in": inner, "out": outer, "dtype": dtype, "train": train, "relu": relu, "p": p,
            "residual": residual}


def _adamw(shapes, dtype, bits, clip, done):
    """``shapes``: the tensors, as "65x7 7"; ``done``: steps taken before this one."""
    return {"op": "adamw", "shapes": shapes, "dtype": dtype, "bits": bits, "clip": clip, "done": done}


def _gcn(features, hidden, classes, layers):
    """The tensors of a GCN with layer normalisation."""
    dims = [features] + [hidden] * (layers - 1) + [classes]
    of_layers = [f"{b}x{a} {b}" + (f" {b} {b}" if i + 2 < len(dims) else "") for i, (a, b) in enumerate(zip(dims, dims[1:]))]
    return " ".join(of_layers)


def listed():
    cases = {
        # class scores of the two-layer model on the citation-sized graph: latency
        "linear_small_infer": _linear(2708, 64, CLASSES, "f32"),
        # its hidden layer in training: latency
        "linear_small_train": _linear(2708, 128, 64, "f32", train=True, p=0.3),
        # a hidden layer of a residual model on the web graph, evaluated
        "linear_web_infer": _linear(NODES, 256, 256, "f32", relu=True, residual=True),
        # the benchmark's hidden layer on the web graph in training
        "linear_web_train": _linear(NODES, 256, 128, "f32", train=True, p=0.3),
        # the linear map of the benchmark's cluster workload on all of its nodes, in 16 bits
        "linear_many_train": _linear(MANY_NODES, 128, 256, "bf16", train=True),
        # a wide encoder in front of the graph layers: the largest product
        "linear_wide_infer": _linear(16384, 4096, 4096, "bf16", relu=True),
        # widths that no vector divides
        "linear_odd_train": _linear(50001, 301, 173, "f16", train=True, p=0.1, residual=True),
        # the tensors of a five-layer model with normalisation: latency
        "adamw_model": _adamw(_gcn(256, 128, CLASSES, 5), "f32", 32, 1.0, 10),
        # a learned embedding of every node in front of a model, the moments in 32 bits
        "adamw_table": _adamw(f"{MANY_NODES}x64 128x64 128", "f32", 32, 0.0, 100),
        # the same with moments in 8 bits, which make room for a table of twice the nodes
        "adamw_table_8bit": _adamw(f"{MANY_NODES}x64 128x64 128", "f32", 8, 0.0, 100),
        # a wide encoder in 16 bits, clipped
        "adamw_encoder": _adamw("4096x4096 4096 " * 6, "bf16", 32, 1.0, 1000),
        # tensors of odd sizes, the last blocks of their scales cut short
        "adamw_odd_8bit": _adamw("50001x301 173x301 173 47x173 47 1", "f16", 8, 0.0, 0),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _spread(rng, least, most):
    """A whole number of [least, most], even over its logarithm."""
    return max(least, min(most, int(round(math.exp(rng.uniform(math.log(least), math.log(most)))))))


def draw(rng):
    dtype = rng.choice(("f32", "f32", "bf16", "f16"))
    if rng.random() < 0.6:
        train = rng.random() < 0.6
        inner, outer = _spread(rng, 1, 4096), _spread(rng, 1, 4096)
        if rng.random() < 0.5:
            inner, outer = (inner + 7) // 8 * 8, (outer + 7) // 8 * 8
        room = min(MANY_NODES, 900_000_000 // (inner + outer), (60_000_000_000 if train else 180_000_000_000) // (inner * outer))
        return _linear(_spread(rng, 1, room), inner, outer, dtype, train, not train and rng.random() < 0.5,
                       rng.choice((0.0, 0.0, 0.1, 0.3, 0.5)), rng.random() < 0.4)
    shapes, left = [], 150_000_000
    for _ in range(_spread(rng, 1, 11)):
        if left >= 8:
            width = _spread(rng, 1, 4096)
            rows = _spread(rng, 1, max(1, min(left // width, MANY_NODES)))
            shapes.append(f"{rows}x{width}" if rng.random() < 0.7 else f"{width}")
            left -= rows * width
    bits = rng.choice((32, 8))
    return _adamw(" ".join(shapes), dtype, bits, 1.0 if bits == 32 and rng.random() < 0.5 else 0.0, rng.choice((0, 1, 10, 1000)))


def _shapes(case):
    return [tuple(int(n) for n in shape.split("x")) for shape in case["shapes"].split()]


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = TYPES[case["dtype"]]

    def normal(*shape, scale=1.0):
        return torch.randn(*shape, device="cuda", generator=gen).mul_(scale)

    key = int(torch.randint(0, 2**62, (1,), device="cuda", generator=gen))
    state = {"case": case, "key": key}
    if case["op"] == "linear":
        rows, inner, outer = case["rows"], case["in"], case["out"]
        # what a propagation or a normalisation hands on: columns of different offsets, values of order one
        state["x"] = normal(rows, inner).add_(normal(inner, scale=0.5)).to(dtype)
        state["weight"] = normal(outer, inner, scale=inner**-0.5).to(dtype)
        state["bias"] = normal(outer, scale=0.1).to(dtype)
        if case["residual"]:
            state["residual"] = normal(rows, outer).to(dtype)
        if case["train"]:
            state["grad"] = normal(rows, outer, scale=0.1).to(dtype)
            for name in ("x", "weight", "bias", "residual"):
                if name in state:
                    state[name].requires_grad_()
        return state
    shapes = _shapes(case)
    state["params"] = [normal(*s, scale=0.1).to(dtype) for s in shapes]
    state["grads"] = [normal(*s, scale=0.01).to(dtype) for s in shapes]
    started = 1.0 if case["done"] else 0.0
    first = [normal(*s, scale=0.003 * started) for s in shapes]
    # (the second moment's root, from tenths of a gradient to a few)
    root = [normal(*s).mul_(0.5).exp_().mul_(0.01 * started) for s in shapes]
    state["steps"] = torch.full((len(shapes),), case["done"], dtype=torch.int64, device="cuda")
    state["step_of"] = list(state["steps"].unbind())
    if case["bits"] == 8:
        for name, values in (("first", first), ("root", root)):
            packed = [_nearest_e4m3(v) for v in values]
            state[name], state[name + "_scale"] = [list(part) for part in zip(*packed)]
    else:
        state["first"], state["second"] = first, [r.square_() for r in root]
    return state


def _nearest_e4m3(values):
    """Values as e4m3 numbers and, for each block, the power of two that they are multiplied by."""
    flat = values.reshape(-1)
    blocks = torch.nn.functional.pad(flat, (0, -flat.numel() % BLOCK)).view(-1, BLOCK)
    scale = torch.exp2(torch.ceil(torch.log2(blocks.amax(1).abs().maximum(blocks.amin(1).abs()).div(448.0).clamp(min=2.0**-117))))
    codes = (blocks / scale[:, None]).to(torch.float8_e4m3fn).view(-1)[:flat.numel()].clone()
    return codes.view(values.shape), scale


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return _plain_linear(state) if state["case"]["op"] == "linear" else _plain_adamw(state)


def _run_own(state):
    from compressgnn_b200 import runtime
    case = state["case"]
    if case["op"] == "adamw":
        eight = case["bits"] == 8
        norm = runtime.adamw_step(state["params"], state["grads"], state["first"], state["root" if eight else "second"],
                                  state["step_of"], lr=RATE, betas=BETAS, eps=EPS, weight_decay=DECAY,
                                  max_norm=case["clip"] or None, exp_avg_scales=state["first_scale"] if eight else None,
                                  exp_avg_sq_scales=state["root_scale"] if eight else None, seed=state["key"])
        return _updated(state, norm)
    x, weight, bias = state["x"], state["weight"], state["bias"]
    y = runtime.linear(x, weight, bias, activation="relu" if case["relu"] else None, dropout=case["p"],
                       residual=state.get("residual"), seed=state["key"])
    if not case["train"]:
        return {"y": y}
    dx, dweight, dbias = torch.autograd.grad(y, (x, weight, bias), state["grad"])
    return {"y": y.detach(), "dx": dx, "dweight": dweight, "dbias": dbias}


def _updated(state, norm):
    """What a step leaves: 8-bit moments are e4m3 numbers beside the scales of their blocks."""
    names = ("params", "first", "second", "root", "first_scale", "root_scale", "steps")
    out = {name: state[name] for name in names if name in state}
    return dict(out, norm=norm) if state["case"]["clip"] else out


def _round(c0, c1, c2, c3, key, i):
    """Round i of Philox4x32 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011)."""
    p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # 64-bit products; their bits do not depend on the sign
    k0, k1 = ((key & LOW) + i * 0x9E3779B9) & LOW, ((key >> 32) + i * 0xBB67AE85) & LOW
    return (p1 >> 32 & LOW) ^ c1 ^ k0, p1 & LOW, (p0 >> 32 & LOW) ^ c3 ^ k1, p0 & LOW


def _random_words(like, key):
    """A word of 32 random bits for each element: element e has word e % 4 of the block of four that counter e // 4 gives
    under the key after seven rounds."""
    n = like.numel()
    block = torch.arange((n + 3) // 4, device=like.device)
    c = block & LOW, block >> 32, torch.full_like(block, 0x243F6A88), torch.full_like(block, 0x85A308D3)
    c = _round(*_round(*_round(*c, key, 0), key, 1), key, 2)
    c = _round(*_round(*_round(*_round(*c, key, 3), key, 4), key, 5), key, 6)
    return torch.stack(c, 1).view(-1)[:n].view(like.shape)


def _plain_linear(state):
    case, x, weight = state["case"], state["x"], state["weight"]
    dtype = x.dtype
    wide, w = x.float(), weight.float()
    y = wide @ w.t() + state["bias"].float()
    if case["relu"]:
        y = torch.where(y < 0, 0.0, y)
    keep = scale = None
    if case["p"]:
        keep, scale = _random_words(y, state["key"]) >= int(case["p"] * 2**32), 1.0 / (1.0 - case["p"])
        y = torch.where(keep, y * scale, 0.0)
    if case["residual"]:
        y = y + state["residual"].float()
    if not case["train"]:
        return {"y": y.to(dtype)}
    g = state["grad"].float()
    if keep is not None:
        g = torch.where(keep, g * scale, 0.0)
    # (sums over all nodes: 64 bits where there is one for each column only)
    return {"y": y.to(dtype), "dx": (g @ w).to(dtype), "dweight": (g.t() @ wide).to(dtype),
            "dbias": g.sum(0, dtype=torch.float64).to(dtype)}


def _e4m3_with_scale(values, bits16, floor_to_least):
    """Stochastic rounding of each block's values to e4m3 times the least power of two that takes its largest in."""
    n, shape = values.numel(), values.shape
    blocks = torch.nn.functional.pad(values.reshape(-1), (0, -n % BLOCK)).view(-1, BLOCK)
    fraction, exponent = torch.frexp(blocks.abs().amax(1, keepdim=True))
    exponent = (exponent - 9 + (fraction > 0.875)).clamp(min=-117)
    exponent = torch.where(fraction == 0, -117, exponent)
    size = torch.ldexp(blocks.abs(), -exponent).view(-1)[:n]
    bits16 = bits16.reshape(-1)
    upper = ((size.view(torch.int32) + (bits16 << 4).int()) & -0x100000).view(torch.float32)
    lower = (size * 512 + bits16.float() * 2.0**-16).floor() * 2.0**-9  # below the least normal number: steps of 2^-9
    rounded = torch.where(size >= 2.0**-6, upper, lower)
    if floor_to_least:
        rounded = torch.where(size > 0, rounded.clamp(min=2.0**-9), rounded)
    rounded = torch.where(values.reshape(-1) < 0, -rounded, rounded)
    return rounded.view(shape).to(torch.float8_e4m3fn), torch.exp2(exponent.view(-1).float())


def _spread_scale(codes, scale):
    return codes.float().reshape(-1).mul(scale.repeat_interleave(BLOCK)[:codes.numel()]).view(codes.shape)


def _plain_adamw(state):
    case, (b1, b2), eight = state["case"], BETAS, state["case"]["bits"] == 8
    done, norm, clip = case["done"], None, None
    if case["clip"]:
        norm = torch.stack([g.double().square().sum() for g in state["grads"]]).sum().sqrt().float()
        clip = (case["clip"] / (norm.double() + 1e-6)).clamp(max=1.0).float()
    # (the counts on the device say how often this state has been stepped already)
    counts = state["steps"].add_(1)
    rate_of = -RATE / (1 - b1 ** counts.double())
    root_of = (1 - b2 ** counts.double()).sqrt()
    for i, (p, g) in enumerate(zip(state["params"], state["grads"])):
        g = g.float()
        if clip is not None:
            g = g * clip
        first = _spread_scale(state["first"][i], state["first_scale"][i]) if eight else state["first"][i]
        second = _spread_scale(state["root"][i], state["root_scale"][i]).square() if eight else state["second"][i]
        first = first * b1 + g * (1 - b1)
        second = second * b2 + g * g * (1 - b2)
        root = second.sqrt()
        q = p.float() * (1 - RATE * DECAY)
        p.copy_(q + rate_of[i].float() * (first / (root / root_of[i].float() + EPS)))
        if eight:
            count = done + state.get("passes", 0)
            key = (state["key"] + i * TENSOR_KEY + count * STEP_KEY) % 2**64
            words = _random_words(p, key)
            for name, values, bits in (("first", first, words & 0xFFFF), ("root", root, words >> 16)):
                codes, scale = _e4m3_with_scale(values, bits, name == "root")
                state[name][i].copy_(codes)
                state[name + "_scale"][i].copy_(scale)
        else:
            state["first"][i].copy_(first)
            state["second"][i].copy_(second)
    state["passes"] = state.get("passes", 0) + 1
    return _updated(state, norm)


# ---------------------------------------------------------------------------------------------
# the same from the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------
def _high_half(a, b):
    """The upper 32 bits of a * b for whole numbers below 2^32, from 16-bit halves."""
    al, ah, bl, bh = a % 65536, a // 65536, b % 65536, b // 65536
    cross = ah * bl + (al * bl) // 65536
    return ah * bh + cross // 65536 + (al * bh + cross % 65536) // 65536


def _words(first, count, key):
    """The random words of elements first .. first + count."""
    e = torch.arange(first, first + count, device="cuda")
    c = [(e // 4) % 2**32, (e // 4) // 2**32, torch.zeros_like(e) + 0x243F6A88, torch.zeros_like(e) + 0x85A308D3]
    low, high = key % 2**32, key // 2**32
    for _ in range(7):
        upper0, upper2 = _high_half(c[0], 0xD2511F53), _high_half(c[2], 0xCD9E8D57)
        lower0, lower2 = (c[0] * 0xD2511F53) % 2**32, (c[2] * 0xCD9E8D57) % 2**32
        c = [upper2 ^ c[1] ^ low, lower2, upper0 ^ c[3] ^ high, lower0]
        low, high = (low + 0x9E3779B9) % 2**32, (high + 0xBB67AE85) % 2**32
    which = e % 4
    return sum(torch.where(which == k, c[k], 0) for k in range(4))


def _in_parts(n):
    step = 1 << 24
    return ((first, min(step, n - first)) for first in range(0, n, step))


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return _exact_linear(state) if case["op"] == "linear" else _exact_adamw(state)


def _exact_linear(state):
    case = state["case"]
    x, weight = state["x"].double(), state["weight"].double()
    y = torch.addmm(state["bias"].double(), x, weight.t())
    if case["relu"]:
        y.clamp_(min=0)
    factor = None
    if case["p"]:
        factor = torch.empty_like(y)
        flat = factor.view(-1)
        for first, count in _in_parts(flat.numel()):
            kept = _words(first, count, state["key"]) >= math.floor(case["p"] * 2**32)
            flat[first:first + count] = kept.double().div_(1 - case["p"])
        y.mul_(factor)
    if case["residual"]:
        y.add_(state["residual"].double())
    if not case["train"]:
        return {"y": y}
    g = state["grad"].double()
    if factor is not None:
        g.mul_(factor)
    return {"y": y, "dx": torch.mm(g, weight), "dweight": torch.einsum("no,ni->oi", g, x), "dbias": torch.einsum("no->o", g)}


def _exact_adamw(state):
    case, t = state["case"], state["case"]["done"] + 1
    eight = case["bits"] == 8
    out = {"params": [], "first": [], "root" if eight else "second": [], "steps": [t] * len(state["params"])}
    out["steps"] = torch.tensor(out["steps"], device="cuda")
    if eight:
        out.update(first_scale=[], root_scale=[])
    shrink = 1.0
    if case["clip"]:
        out["norm"] = torch.sqrt(sum(torch.linalg.vector_norm(g, dtype=torch.float64).square() for g in state["grads"]))
        shrink = min(1.0, case["clip"] / (float(out["norm"]) + 1e-6))
    for i, p in enumerate(state["params"]):
        g, theta = state["grads"][i].double() * shrink, p.double()
        if eight:
            where = torch.arange(p.numel(), device="cuda").div(BLOCK, rounding_mode="floor").view(p.shape)
            m = state["first"][i].double() * state["first_scale"][i].double()[where]
            v = (state["root"][i].double() * state["root_scale"][i].double()[where]).pow(2)
        else:
            m, v = state["first"][i].double(), state["second"][i].double()
        m = torch.lerp(g, m, BETAS[0])
        v = torch.lerp(g.pow(2), v, BETAS[1])
        m_hat, v_hat = m / (1 - BETAS[0] ** t), v / (1 - BETAS[1] ** t)
        out["params"].append(theta - RATE * DECAY * theta - RATE * m_hat / (torch.sqrt(v_hat) + EPS))
        if not eight:
            out["first"].append(m)
            out["second"].append(v)
            continue
        key = (state["key"] + i * TENSOR_KEY + case["done"] * STEP_KEY) % 2**64
        words = torch.cat([_words(first, count, key) for first, count in _in_parts(p.numel())]).view(p.shape)
        for name, values, part in (("first", m, words % 65536), ("root", v.sqrt(), words // 65536)):
            largest = torch.zeros(where.max() + 1, dtype=torch.float64, device="cuda")
            largest.scatter_reduce_(0, where.view(-1), values.abs().view(-1), "amax")
            scale = torch.exp2(torch.ceil(torch.log2(torch.clamp(largest / 448, min=2.0**-117))))
            size = values.abs() / scale[where]
            step = torch.exp2(torch.clamp(torch.floor(torch.log2(torch.clamp(size, min=2.0**-30))), min=-6) - 3)
            code = torch.floor(size / step + part.double() / 65536) * step
            if name == "root":
                code = torch.where((size > 0) & (code == 0), 2.0**-9, code)
            out[name].append(torch.copysign(code, values))
            out[name + "_scale"].append(scale)
    return out


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    item = TYPES[case["dtype"]].itemsize
    if case["op"] == "linear":
        rows, inner, outer = case["rows"], case["in"], case["out"]
        passed = rows * (inner + outer) + inner * outer + outer
        if case["residual"]:
            passed += rows * outer
        if case["train"]:  # the incoming gradient, and those of x, the weight and the bias
            passed += rows * outer + rows * inner + inner * outer + outer
        return {"bytes": passed * item, "flops": (6 if case["train"] else 2) * rows * inner * outer}
    n = sum(math.prod(shape) for shape in _shapes(case))
    moments = 4 + 4 if case["bits"] == 32 else 2 + 2 * 4 / BLOCK
    return {"bytes": n * (3 * item + 2 * moments), "flops": n * (16 if case["bits"] == 32 else 60)}

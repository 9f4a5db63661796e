"""The operators of a training step that stand between and behind the propagations: what they are measured on.

``norm``     layer normalisation of node features with the ReLU and the dropout that follow it in a hidden layer,
             forward, or forward and backward (gradients of the features, the weight and the bias).
``drop``     dropout from a counter-based generator, alone or added to a residual stream, forward, or both ways.
``loss``     softmax cross entropy of class scores over the labelled nodes, with the gradient of the scores or without.

``run`` computes them with elementary torch operations, or with the package's own operators where ``own`` is set.
A training case of ``norm`` has no ReLU: the gradient of one jumps at its border, where 32 and 64 bits may fall on
either side.
"""
import math

import torch

own = False

NODES = 325557         # nodes of the benchmark's web graph
MANY_NODES = 2450000   # nodes of the benchmark's cluster workload
CLASSES = 47           # classes of the benchmark's models
EPS = 1e-5
IGNORED = -100         # the label of a node outside the training set
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
LOW = 0xFFFFFFFF       # the low 32 bits of a word


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _norm(rows, width, dtype, weights, train, p, relu):
    return {"op": "norm", "rows": rows, "width": width, "dtype": dtype, "weights": weights, "train": train, "p": p,
            "relu": relu}


def _drop(rows, width, dtype, train, p, residual):
    return {"op": "drop", "rows": rows, "width": width, "dtype": dtype, "train": train, "p": p, "residual": residual}


def _loss(rows, classes, dtype, train, labelled, reduction, scale):
    return {"op": "loss", "rows": rows, "classes": classes, "dtype": dtype, "train": train, "labelled": labelled,
            "reduction": reduction, "scale": scale}


def listed():
    cases = {
        # inference and training of the two-layer model's hidden layer on the citation-sized graph: latency
        "norm_small_infer": _norm(2708, 64, "f32", "f32", False, 0.0, True),
        "norm_small_train": _norm(2708, 64, "f32", "f32", True, 0.3, False),
        # the hidden layer of the benchmark's model on the web graph
        "norm_web_train": _norm(NODES, 128, "f32", "f32", True, 0.3, False),
        # the largest node set of the benchmark at its feature width
        "norm_many_train": _norm(MANY_NODES, 128, "f32", "f32", True, 0.5, False),
        # wide rows in 16 bits: the activations of a wide encoder in front of the graph layers
        "norm_wide_infer": _norm(16384, 4096, "bf16", "f32", False, 0.1, True),
        # a width that no vector divides
        "norm_odd_train": _norm(50001, 301, "f16", "f16", True, 0.0, False),
        # a mini-batch of seed nodes with their features: latency
        "drop_small": _drop(1024, 128, "f32", False, 0.3, False),
        # the residual connection of a hidden layer on the web graph, both ways
        "drop_web_train": _drop(NODES, 256, "f32", True, 0.3, True),
        # the loss of the citation-sized model: seven classes, a few labelled nodes
        "loss_small_train": _loss(2708, 7, "f32", True, 0.3, "mean", 1.0),
        # the loss of the benchmark's model on its largest node set
        "loss_many_train": _loss(MANY_NODES, CLASSES, "f32", True, 0.6, "mean", 1.0),
        # the loss of each node, for hard-example mining or evaluation
        "loss_web_rows": _loss(NODES, CLASSES, "f32", False, 1.0, "none", 1.0),
        # scores over a vocabulary of entities, an odd number of them
        "loss_wide_train": _loss(8192, 50001, "bf16", True, 0.9, "mean", 1.0),
    }
    return [dict(case, name=name) for name, case in cases.items()]


def _spread(rng, least, most):
    """A whole number of [least, most], even over its logarithm."""
    return max(least, min(most, int(round(math.exp(rng.uniform(math.log(least), math.log(most)))))))


def draw(rng):
    op = rng.choice(("norm", "norm", "drop", "loss", "loss"))
    dtype = rng.choice(("f32", "f32", "bf16", "f16"))
    train = rng.random() < 0.6
    p = rng.choice((0.0, 0.1, 0.3, 0.5))
    if op == "norm":
        width = _spread(rng, 4, 8192)
        if rng.random() < 0.5:
            width = max(4, width // 8 * 8)
        rows = _spread(rng, 1, min(MANY_NODES, 120_000_000 // width))
        return _norm(rows, width, dtype, rng.choice((dtype, "f32")), train, p, not train and rng.random() < 0.5)
    if op == "drop":
        width = _spread(rng, 1, 4096)
        rows = _spread(rng, 1, min(MANY_NODES, 80_000_000 // width))
        return _drop(rows, width, dtype, train, max(p, 0.1), rng.random() < 0.5)
    classes = _spread(rng, 2, 50257)
    rows = _spread(rng, 1, min(MANY_NODES, 100_000_000 // classes))
    return _loss(rows, classes, dtype, train, rng.choice((0.1, 0.6, 1.0)), rng.choice(("mean", "sum", "none")),
                 1024.0 if dtype == "f16" else 1.0)


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    dtype = TYPES[case["dtype"]]

    def normal(*shape, kind=dtype):
        return torch.randn(*shape, device="cuda", generator=gen).to(kind)

    if case["op"] == "loss":
        rows, classes = case["rows"], case["classes"]
        logits = torch.randn(rows, classes, device="cuda", generator=gen).mul_(3.0).to(dtype)
        target = torch.randint(0, classes, (rows,), device="cuda", generator=gen)
        unlabelled = torch.rand(rows, device="cuda", generator=gen) >= case["labelled"]
        unlabelled[0] = False
        target[unlabelled] = IGNORED
        state = {"case": case, "logits": logits, "target": target}
        if case["train"]:
            logits.requires_grad_()
            shape = (rows,) if case["reduction"] == "none" else ()
            state["upstream"] = torch.full(shape, case["scale"], device="cuda")
            if shape:
                state["upstream"] *= torch.rand(rows, device="cuda", generator=gen)
        return state
    rows, width = case["rows"], case["width"]
    # what a propagation and a linear map hand on: columns of different offsets, values of order one
    x = (torch.randn(rows, width, device="cuda", generator=gen) +
         torch.randn(width, device="cuda", generator=gen).mul_(0.5)).to(dtype)
    key = int(torch.randint(0, 2**62, (1,), device="cuda", generator=gen))
    state = {"case": case, "x": x, "key": key}
    if case["op"] == "norm":
        kind = TYPES[case["weights"]]
        state["weight"] = normal(width).float().mul_(0.2).add_(1.0).to(kind)
        state["bias"] = normal(width).float().mul_(0.2).to(kind)
    elif case["residual"]:
        state["residual"] = normal(rows, width)
    if case["train"]:
        state["grad"] = normal(rows, width)
        for name in ("x", "weight", "bias", "residual"):
            if name in state:
                state[name].requires_grad_()
    return state


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"norm": _plain_norm, "drop": _plain_drop, "loss": _plain_loss}[state["case"]["op"]](state)


def _run_own(state):
    from compressgnn_b200 import runtime
    case = state["case"]
    if case["op"] == "loss":
        logits = state["logits"]
        loss = runtime.cross_entropy(logits, state["target"], ignore_index=IGNORED, reduction=case["reduction"])
        if not case["train"]:
            return {"loss": loss}
        dlogits, = torch.autograd.grad(loss, logits, state["upstream"])
        return {"loss": loss.detach(), "dlogits": dlogits}
    if case["op"] == "drop":
        x, residual = state["x"], state.get("residual")
        y = runtime.dropout(x, case["p"], residual=residual, seed=state["key"])
        if not case["train"]:
            return {"y": y}
        # (a residual's gradient is the incoming one: there is nothing to compute for it)
        dx, = torch.autograd.grad(y, x, state["grad"])
        return {"y": y.detach(), "dx": dx}
    x, weight, bias = state["x"], state["weight"], state["bias"]
    y = runtime.layer_norm(x, weight, bias, eps=EPS, activation="relu" if case["relu"] else None, dropout=case["p"],
                           seed=state["key"])
    if not case["train"]:
        return {"y": y}
    dx, dweight, dbias = torch.autograd.grad(y, (x, weight, bias), state["grad"])
    return {"y": y.detach(), "dx": dx, "dweight": dweight, "dbias": dbias}


def _round(c0, c1, c2, c3, key, i):
    """Round i of Philox4x32 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011)."""
    p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # 64-bit products; their bits do not depend on the sign
    k0, k1 = ((key & LOW) + i * 0x9E3779B9) & LOW, ((key >> 32) + i * 0xBB67AE85) & LOW
    return (p1 >> 32 & LOW) ^ c1 ^ k0, p1 & LOW, (p0 >> 32 & LOW) ^ c3 ^ k1, p0 & LOW


def _kept(like, p, key):
    """Which elements stay: element e takes word e % 4 of the block of four that counter e // 4 gives under the key
    after seven rounds, and is dropped where that is below p * 2^32."""
    n = like.numel()
    block = torch.arange((n + 3) // 4, device=like.device)
    c = block & LOW, block >> 32, torch.full_like(block, 0x243F6A88), torch.full_like(block, 0x85A308D3)
    c = _round(*_round(*_round(*c, key, 0), key, 1), key, 2)
    c = _round(*_round(*_round(*_round(*c, key, 3), key, 4), key, 5), key, 6)
    return (torch.stack(c, 1).view(-1)[:n] >= int(p * 2**32)).view(like.shape)


def _plain_drop(state):
    case, x = state["case"], state["x"]
    keep, scale = _kept(x, case["p"], state["key"]), 1.0 / (1.0 - case["p"])
    y = torch.where(keep, x.float() * scale, 0.0)
    if case["residual"]:
        y = y + state["residual"].float()
    if not case["train"]:
        return {"y": y.to(x.dtype)}
    return {"y": y.to(x.dtype), "dx": torch.where(keep, state["grad"].float() * scale, 0.0).to(x.dtype)}


def _plain_norm(state):
    case, x = state["case"], state["x"]
    weight, bias = state["weight"].float(), state["bias"].float()
    keep = _kept(x, case["p"], state["key"]) if case["p"] else None
    scale = 1.0 / (1.0 - case["p"])
    wide = x.float()
    off = wide - wide.mean(1, keepdim=True)
    rstd = (off.square().mean(1, keepdim=True) + EPS).rsqrt()
    hat = off * rstd
    y = hat * weight + bias
    if case["relu"]:
        y = torch.where(y < 0, 0.0, y)
    if keep is not None:
        y = torch.where(keep, y * scale, 0.0)
    y = y.to(x.dtype)
    if not case["train"]:
        return {"y": y}
    g = state["grad"].float()
    if keep is not None:
        g = torch.where(keep, g * scale, 0.0)
    gw = g * weight
    dx = rstd * (gw - gw.mean(1, keepdim=True) - hat * (gw * hat).mean(1, keepdim=True))
    # (sums over all nodes: 64 bits)
    return {"y": y, "dx": dx.to(x.dtype), "dweight": (g * hat).sum(0, dtype=torch.float64).to(state["weight"].dtype),
            "dbias": g.sum(0, dtype=torch.float64).to(state["bias"].dtype)}


def _plain_loss(state):
    case, logits, target = state["case"], state["logits"], state["target"]
    labelled = target != IGNORED
    place = torch.where(labelled, target, 0)[:, None]
    z = logits.float()
    z = z - z.max(1, keepdim=True).values
    e = z.exp()
    total = e.sum(1, keepdim=True)
    rows = torch.where(labelled, (total.log() - z.gather(1, place)).view(-1), 0.0)
    if case["reduction"] == "none":
        loss = rows
    else:
        loss = rows.sum(dtype=torch.float64)
        if case["reduction"] == "mean":
            loss = loss / labelled.sum()
        loss = loss.float()
    if not case["train"]:
        return {"loss": loss}
    # (a mean's share of each node is exact to 32 bits before it meets the probabilities)
    share = state["upstream"].double()
    if case["reduction"] == "mean":
        share = share / labelled.sum()
    share = torch.where(labelled, share.float(), 0.0)[:, None]
    grad = e / total
    grad.scatter_add_(1, place, torch.full_like(place, -1, dtype=torch.float32))
    return {"loss": loss, "dlogits": (grad * share).to(logits.dtype)}


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


def _factors(shape, p, key):
    """What dropout multiplies each element by, in 64 bits, for a matrix of that shape."""
    n = shape[0] * shape[1]
    out = torch.ones(n, dtype=torch.float64, device="cuda")
    if p:
        step = 1 << 25
        for first in range(0, n, step):
            part = out[first:first + step]
            part.copy_((_words(first, part.numel(), key) >= math.floor(p * 2**32)).double().div_(1 - p))
    return out.view(shape)


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "loss":
            return _exact_loss(state)
        x = state["x"].double()
        factor = _factors(x.shape, case["p"], state["key"])
        if case["op"] == "drop":
            y = x.mul_(factor)
            if case["residual"]:
                y += state["residual"].double()
            return {"y": y, "dx": factor.mul_(state["grad"].double())} if case["train"] else {"y": y}
        return _exact_norm(state, x, factor)


def _exact_norm(state, x, factor):
    case, width = state["case"], x.size(1)
    weight, bias = state["weight"].double(), state["bias"].double()
    variance, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    deviation = torch.sqrt(variance + EPS)
    hat = x.sub_(mean).div_(deviation)
    y = torch.addcmul(bias, hat, weight)
    if case["relu"]:
        y.clamp_(min=0)
    y.mul_(factor)
    if not case["train"]:
        return {"y": y}
    g = factor.mul_(state["grad"].double())
    dweight, dbias = torch.einsum("nd,nd->d", g, hat), g.sum(0)
    g.mul_(weight)
    along, across = torch.einsum("nd,nd->n", g, hat) / width, g.sum(1) / width
    dx = g.sub_(across[:, None]).sub_(hat.mul_(along[:, None])).div_(deviation)
    return {"y": y, "dx": dx, "dweight": dweight, "dbias": dbias}


def _exact_loss(state):
    case, target = state["case"], state["target"]
    z = state["logits"].double()
    labelled = (target != IGNORED).nonzero().view(-1)
    at = target[labelled]
    rest = torch.logsumexp(z, 1)
    rows = torch.zeros(target.numel(), dtype=torch.float64, device="cuda")
    rows[labelled] = rest[labelled] - z[labelled, at]
    share = {"mean": 1.0 / labelled.numel(), "sum": 1.0, "none": 1.0}[case["reduction"]]
    loss = rows if case["reduction"] == "none" else rows.sum() * share
    if not case["train"]:
        return {"loss": loss}
    up = torch.zeros(target.numel(), dtype=torch.float64, device="cuda")
    up[labelled] = (state["upstream"].double().expand(target.numel()) * share)[labelled]
    z.sub_(rest[:, None]).exp_()
    z[labelled, at] -= 1.0
    z.mul_(up[:, None])
    return {"loss": loss, "dlogits": z}


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    item = TYPES[case["dtype"]].itemsize
    if case["op"] == "loss":
        rows, n = case["rows"], case["rows"] * case["classes"]
        read = case["labelled"] * n * item + 8 * rows  # the scores of a node without a label are not needed
        write = (n * item if case["train"] else 0) + (4 * rows if case["reduction"] == "none" else 4)
        return {"bytes": read + write, "flops": case["labelled"] * n * (6 if case["train"] else 4)}
    n = case["rows"] * case["width"]
    both = 2 if case["train"] else 1
    if case["op"] == "drop":
        return {"bytes": (2 * both + (1 if case["residual"] else 0)) * n * item, "flops": 2 * both * n}
    weights = 2 * case["width"] * TYPES[case["weights"]].itemsize
    return {"bytes": 2 * both * n * item + both * weights, "flops": (20 if case["train"] else 8) * n}

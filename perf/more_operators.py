"""A training step's heavy operators around a dense model, as cases that can be timed and whose results can be compared.  `op`:
  * "gated":      h = f(x @ gate_weight.T + gate_bias) * (x @ up_weight.T + up_bias), the first half of a gated feed-forward block
  * "gated_grad": its gradient, from the two products that the forward pass saved: those of x, of both weights and both biases
  * "loss":       softmax cross entropy of x @ weight.T + bias over many items, one target a row, without a matrix of logits
  * "loss_grad":  its gradient: those of x, of weight and of bias
  * "norm":       the 2-norm of many gradients together
  * "clip":       that, and the gradients scaled by min(1, max_norm / norm) into the buffers that an optimiser or a collective takes
`act` is the type of activations and weights (of gradients, for the last two), `bias` that of the biases ("none": there are none).
`saved`: the forward pass returns both products, or the rows' log of the sum of exponentials, as training needs them.  `pad`: the
rows of activations lie that many values apart, as slices of wider matrices do.  `ignored`: the share of rows whose target
is -100, which take no part.  The gradients of the last two are those of `layers` blocks of three matrices of `width` x `hidden`
values and two float vectors of `width`, and of `rows` rows of 128 floats that a table pulled.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZES = {"f32": 4, "bf16": 2, "f16": 2}
_IGNORED = -100
_DEFAULTS = {
    "gated": {"op": "gated", "rows": 1, "width": 4096, "hidden": 16384, "act": "bf16", "bias": "none", "f": "silu", "saved": False, "pad": 0},
    "loss": {"op": "loss", "rows": 1, "width": 128, "items": 1000, "act": "bf16", "bias": "none", "saved": False, "pad": 0, "ignored": 0.0},
    "clip": {"op": "clip", "layers": 1, "width": 128, "hidden": 512, "rows": 0, "act": "bf16", "max_norm": 1.0},
}
_KIND = {"gated": "gated", "gated_grad": "gated", "loss": "loss", "loss_grad": "loss", "norm": "clip", "clip": "clip"}


def _case(name=None, **options):
    defaults = _DEFAULTS[_KIND[options["op"]]]
    case = dict(defaults, **options)
    assert set(case) == set(defaults)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # serving: one token of a wide model
        _case("gated_one_token", op="gated"),
        # decoding 64 tokens, weights in half precision, with biases
        _case("gated_64", op="gated", rows=64, width=8192, hidden=8192, act="f16", bias="act", f="gelu"),
        # the first layer of a click model: the large batch of 65536 samples, 26 fields of 128 values side by side
        _case("gated_click_train", op="gated", rows=65536, width=26 * 128, hidden=512, bias="f32", saved=True),
        # training, a block of a sequence model: 8192 tokens
        _case("gated_train", op="gated", rows=8192, saved=True),
        _case("gated_train_grad", op="gated_grad", rows=8192),
        # sizes nobody rounds: 39 fields of 37 floats, a ragged batch, all of it in 32 bits
        _case("gated_odd_grad", op="gated_grad", rows=5003, width=39 * 37, hidden=1001, act="f32", bias="f32", f="relu"),
        # scoring: the likelihood of 32 tokens in a large vocabulary
        _case("loss_few", op="loss", rows=32, width=4096, items=131072),
        # the next item among a million rows of a table, a batch of 4096 histories
        _case("loss_items", op="loss", rows=4096, items=1_000_000, bias="f32", saved=True),
        _case("loss_items_grad", op="loss_grad", rows=4096, items=1_000_000, bias="f32"),
        # training a sequence model: padded sequences, a vocabulary nobody rounds
        _case("loss_train_grad", op="loss_grad", rows=8192, width=4096, items=65537, ignored=0.25),
        # the gradients of a small click model and of the rows of its batch, 2048 samples of 26 fields
        _case("clip_click", op="clip", layers=2, rows=2048 * 26, act="f32"),
        # of eight wide blocks, and of the rows of the large batch
        _case("clip_model", op="clip", layers=8, width=4096, hidden=16384, rows=65536 * 26),
    ]


_MOST_FLOPS = 6 * 8192 * 4096 * 65537      # of a pass, in the largest listed case
_MOST_LOGITS = 4096 * 1_000_000
_MOST_VALUES = 8 * 3 * 4096 * 16384        # of the blocks' gradients


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """Any, a multiple of 8 or a power of two"""
    n = _log_uniform(rng, lo, hi)
    return rng.choice([n, max(8, n // 8 * 8), 1 << (n.bit_length() - 1)])


def draw(rng):
    op = rng.choice(["gated", "gated", "gated_grad", "gated_grad", "loss", "loss_grad", "loss_grad", "norm", "clip"])
    kind, act = _KIND[op], rng.choice(["f32", "bf16", "bf16", "f16"])
    case = _case(op=op, act=act, width=_size(rng, 16, 4096 if kind == "clip" else 8192))
    if kind == "clip":
        case.update(layers=_log_uniform(rng, 1, 100), hidden=_size(rng, 16, 16384), rows=rng.choice([0, _log_uniform(rng, 100, 2_000_000)]),
                    max_norm=rng.choice([0.1, 1.0, 1e6]))
        case["layers"] = max(1, min(case["layers"], _MOST_VALUES // (3 * case["width"] * case["hidden"])))
        return case
    case.update(bias=rng.choice(["none", "none", "act", "f32"]), pad=rng.choice([0, 0, 0, 5, 64]))
    if op in ("gated", "loss"):
        case["saved"] = rng.random() < 0.6
    rows = rng.choice([_log_uniform(rng, 1, 64), _log_uniform(rng, 1, 16384), _log_uniform(rng, 64, 65536)])
    if kind == "gated":
        case.update(hidden=_size(rng, 16, 16384), f=rng.choice(["silu", "gelu", "relu", "sigmoid"]))
        most = _MOST_VALUES // max(case["width"], case["hidden"])
    else:
        case.update(items=_size(rng, 100, 1_000_000), ignored=rng.choice([0.0, 0.0, 0.25, 0.6]))
        most = _MOST_LOGITS // case["items"]
    # (a product in 32 bits costs more than one in 16)
    share = 8 if act == "f32" else 1
    case["rows"] = max(1, min(rows, most))
    case["rows"] = max(1, min(case["rows"], int(case["rows"] * _MOST_FLOPS / share / work(case)["flops"])))
    return case


# ---- inputs -----------------------------------------------------------------------------------------------------------
def _shapes(case):
    """(shape, type) of each gradient of "norm" and "clip"."""
    width, hidden, act = case["width"], case["hidden"], _TYPES[case["act"]]
    block = [((hidden, width), act), ((hidden, width), act), ((width, hidden), act), ((width,), torch.float32), ((width,), torch.float32)]
    return ([((case["rows"], 128), torch.float32)] if case["rows"] else []) + block * case["layers"]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    act = _TYPES[case["act"]]

    def values(shape, std, dtype=act):
        return torch.empty(shape, device="cuda").normal_(0.0, std, generator=gen).to(dtype)

    def activations(columns, std):
        return values((case["rows"], columns + case["pad"]), std)[:, :columns]

    def bias(columns):
        return None if case["bias"] == "none" else values(columns, 0.1, torch.float32 if case["bias"] == "f32" else act)

    state = {"case": case}
    kind, op = _KIND[case["op"]], case["op"]
    if kind == "clip":
        # later layers have smaller gradients
        state["gradients"] = [values(shape, 1e-3 / (1 + i % 7), dtype) for i, (shape, dtype) in enumerate(_shapes(case))]
        if op == "clip":
            state["into"] = [torch.empty_like(g) for g in state["gradients"]]
    elif kind == "gated":
        state["x"] = activations(case["width"], 1.0)
        state["weights"] = [values((case["hidden"], case["width"]), case["width"] ** -0.5) for _ in range(2)]
        state["biases"] = [bias(case["hidden"]) for _ in range(2)]
        if op == "gated_grad":
            state["dh"] = activations(case["hidden"], 1e-3)
            state["gate"], state["up"] = (p.to(act) for p in _products(state))
    else:
        state["x"] = activations(case["width"], 1.0)
        state["weight"] = values((case["items"], case["width"]), 2 * case["width"] ** -0.5)
        state["bias"] = bias(case["items"])
        target = torch.randint(0, case["items"], (case["rows"],), device="cuda", generator=gen)
        left = torch.rand(case["rows"], device="cuda", generator=gen) < case["ignored"]
        state["target"] = torch.where(left, _IGNORED, target)
        if op == "loss_grad":
            # of a mean over the rows that take part
            state["dloss"] = torch.ones(case["rows"], device="cuda") / (state["target"] != _IGNORED).sum().clamp_min(1)
            state["lse"] = torch.where(left, 0.0, torch.logsumexp(_logits(state), 1))
    torch.cuda.synchronize()
    return state


# ---- the plain forms --------------------------------------------------------------------------------------------------
_F = {"silu": lambda v: v / (1 + torch.exp(-v)), "gelu": lambda v: 0.5 * v * (1 + torch.erf(v * 0.5 ** 0.5)),
      "relu": lambda v: torch.where(v > 0, v, 0.0), "sigmoid": lambda v: 1 / (1 + torch.exp(-v))}


def _slope(f, v):
    if f == "relu":
        return (v > 0).to(v.dtype)
    if f == "gelu":
        return 0.5 * (1 + torch.erf(v * 0.5 ** 0.5)) + v * torch.exp(-0.5 * v * v) * (2 * math.pi) ** -0.5
    s = 1 / (1 + torch.exp(-v))
    return s * (1 - s) * v + s if f == "silu" else s * (1 - s)


def _products(state):
    x = state["x"].float()
    out = [x @ w.float().T for w in state["weights"]]
    return [p if b is None else p + b.float() for p, b in zip(out, state["biases"])]


def _logits(state):
    out = state["x"].float() @ state["weight"].float().T
    return out if state["bias"] is None else out + state["bias"].float()


def _plain_gated(state, case, act):
    gate, up = _products(state)
    h = (_F[case["f"]](gate) * up).to(act)
    return (h, gate.to(act), up.to(act)) if case["saved"] else h


def _plain_gated_grad(state, case, act):
    dh, x, gate, up = (state[k].float() for k in ("dh", "x", "gate", "up"))
    dgate, dup = dh * up * _slope(case["f"], gate), dh * _F[case["f"]](gate)
    dx = dgate @ state["weights"][0].float() + dup @ state["weights"][1].float()
    dbiases = [None if b is None else d.sum(0).to(b.dtype) for d, b in zip((dgate, dup), state["biases"])]
    return (dx.to(act), (dgate.T @ x).to(act), (dup.T @ x).to(act), *dbiases)


def _plain_loss(state, case):
    logits, target = _logits(state), state["target"]
    most = logits.amax(1)
    lse = most + torch.log(torch.exp(logits - most[:, None]).sum(1))
    there = target != _IGNORED
    loss = torch.where(there, lse - logits.gather(1, target.clamp_min(0)[:, None])[:, 0], 0.0)
    return (loss, torch.where(there, lse, 0.0)) if case["saved"] else loss


def _plain_loss_grad(state, act):
    target, there = state["target"], state["target"] != _IGNORED
    d = torch.exp(_logits(state) - state["lse"][:, None])
    d.scatter_add_(1, target.clamp_min(0)[:, None], torch.full_like(d[:, :1], -1.0))
    d = torch.where(there[:, None], d * state["dloss"][:, None], 0.0)
    dbias = None if state["bias"] is None else d.sum(0).to(state["bias"].dtype)
    return (d @ state["weight"].float()).to(act), (d.T @ state["x"].float()).to(act), dbias


def _plain_norm(gradients):
    return torch.sqrt(torch.stack([(g.float() * g.float()).sum() for g in gradients]).sum())


def _plain(state):
    case, act = state["case"], _TYPES[state["case"]["act"]]
    op = case["op"]
    if op == "gated":
        return _plain_gated(state, case, act)
    if op == "gated_grad":
        return _plain_gated_grad(state, case, act)
    if op == "loss":
        return _plain_loss(state, case)
    if op == "loss_grad":
        return _plain_loss_grad(state, act)
    norm = _plain_norm(state["gradients"])
    if op == "norm":
        return norm
    scale = torch.clamp(case["max_norm"] / norm, max=1.0)
    return (norm, *[into.copy_(g.float() * scale) for g, into in zip(state["gradients"], state["into"])])


# ---- one pass -----------------------------------------------------------------------------------------------------------
def run(state):
    if not own:
        return _plain(state)
    from hetuctr_amd import nn
    case = state["case"]
    op = case["op"]
    if op == "gated":
        return nn.gated_linear(state["x"], *state["weights"], *state["biases"], activation=case["f"], saved=case["saved"])
    if op == "gated_grad":
        return nn.gated_linear_backward(state["dh"], state["x"], state["gate"], state["up"], *state["weights"], *state["biases"],
                                        activation=case["f"])
    if op == "loss":
        return nn.linear_cross_entropy(state["x"], state["weight"], state["target"], state["bias"], ignore_index=_IGNORED, stats=case["saved"])
    if op == "loss_grad":
        return nn.linear_cross_entropy_backward(state["dloss"], state["x"], state["weight"], state["target"], state["lse"], state["bias"],
                                                ignore_index=_IGNORED)
    if op == "norm":
        return nn.gradient_norm(state["gradients"])
    return (nn.clip_gradients(state["gradients"], case["max_norm"], into=state["into"]), *state["into"])


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------
def work(case):
    op, act = case["op"], _SIZES[case["act"]]
    if _KIND[op] == "clip":
        values = [(math.prod(shape), dtype.itemsize) for shape, dtype in _shapes(case)]
        count = sum(n for n, _ in values)
        # each value is read once, and written once
        passes = 2 if op == "clip" else 1
        return {"bytes": passes * sum(n * size for n, size in values), "flops": (passes + 1) * count}
    rows, width = case["rows"], case["width"]
    bias = {"none": 0, "act": act, "f32": 4}[case["bias"]]
    if _KIND[op] == "gated":
        hidden = case["hidden"]
        matrices, product = 2 * hidden * width * act, 2 * rows * 2 * hidden * width
        if op == "gated":
            return {"bytes": matrices + rows * (width + hidden * (3 if case["saved"] else 1)) * act + 2 * hidden * bias, "flops": product}
        # read: dh, gate, up, x and the weights; written: dx, the weights' and the biases' gradients
        return {"bytes": 2 * matrices + rows * (2 * width + 3 * hidden) * act + 2 * hidden * bias, "flops": 2 * product}
    items = case["items"]
    # the rows that take part, as they are on average
    product = 2 * rows * (1 - case["ignored"]) * items * width
    small = rows * 8 + items * bias
    if op == "loss":
        return {"bytes": (items + rows) * width * act + small + rows * (8 if case["saved"] else 4), "flops": product}
    return {"bytes": 2 * (items + rows) * width * act + small + items * bias + rows * 8, "flops": 3 * product}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------
def _exact_f(f, v):
    """f(v) and its derivative"""
    if f == "relu":
        return v.clamp_min(0), torch.heaviside(v, torch.zeros((), dtype=v.dtype, device=v.device))
    if f == "gelu":
        phi = torch.special.ndtr(v)
        return v * phi, phi + v * torch.exp(v.square() / -2) / math.sqrt(2 * math.pi)
    s = torch.special.expit(v)
    return (s, s - s.square()) if f == "sigmoid" else (v * s, s + v * (s - s.square()))


def _exact_gated(state, case):
    x, (wg, wu) = state["x"].double(), [w.double() for w in state["weights"]]
    bg, bu = [0.0 if b is None else b.double() for b in state["biases"]]
    if case["op"] == "gated":
        gate, up = torch.matmul(x, wg.t()).add_(bg), torch.matmul(x, wu.t()).add_(bu)
        h = _exact_f(case["f"], gate)[0] * up
        return (h, gate, up) if case["saved"] else h
    value, slope = _exact_f(case["f"], state["gate"].double())
    dh = state["dh"].double()
    dup, dgate = dh * value, dh * slope * state["up"].double()
    none = case["bias"] == "none"
    return (torch.addmm(torch.mm(dup, wu), dgate, wg), torch.mm(dgate.t(), x), torch.mm(dup.t(), x), None if none else dgate.sum(0),
            None if none else dup.sum(0))


def _exact_loss(state, case, piece=65536):
    x, weight, target = state["x"].double(), state["weight"], state["target"]
    live = (target != _IGNORED).nonzero()[:, 0]
    rows, items, width = case["rows"], case["items"], case["width"]
    x, aim = x[live], target[live]
    pieces = [slice(i, min(i + piece, items)) for i in range(0, items, piece)]

    def logits(at):
        out = torch.mm(x, weight[at].double().t())
        return out if state["bias"] is None else out + state["bias"][at].double()

    def spread(v, *shape):
        return torch.zeros((rows, *shape), dtype=torch.float64, device="cuda").index_copy_(0, live, v)

    if case["op"] == "loss":
        lse = torch.stack([torch.logsumexp(logits(at), 1) for at in pieces]).logsumexp(0)
        hit = (x * weight[aim].double()).sum(1) + (0.0 if state["bias"] is None else state["bias"][aim].double())
        return (spread(lse - hit), spread(lse)) if case["saved"] else spread(lse - hit)
    lse, scale = state["lse"][live].double()[:, None], state["dloss"][live].double()[:, None]
    dx, dweight, dbias = torch.zeros_like(x), [], []
    for at in pieces:
        d = logits(at).sub_(lse).exp_()
        inside = ((aim >= at.start) & (aim < at.stop)).nonzero()[:, 0]
        d[inside, aim[inside] - at.start] -= 1
        d *= scale
        dx += torch.mm(d, weight[at].double())
        dweight.append(torch.mm(d.t(), x))
        dbias.append(d.sum(0))
    return spread(dx, width), torch.cat(dweight), None if state["bias"] is None else torch.cat(dbias)


def exact(case, seed):
    state = prepare(case, seed)
    if _KIND[case["op"]] == "gated":
        return _exact_gated(state, case)
    if _KIND[case["op"]] == "loss":
        return _exact_loss(state, case)
    norm = math.sqrt(math.fsum(torch.linalg.vector_norm(g.flatten(), dtype=torch.float64).item() ** 2 for g in state["gradients"]))
    total = torch.tensor(norm, dtype=torch.float64, device="cuda")
    if case["op"] == "norm":
        return total
    scale = case["max_norm"] / norm if norm > case["max_norm"] else 1.0
    return (total, *[g.double() * scale for g in state["gradients"]])

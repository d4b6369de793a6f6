"""The operators between the table's rows and a dense model, as cases that can be timed and whose results can be compared.

A matrix of `rows` x `width` values is dropped out, normalised over its rows, or both; `op` says which:
  * "dropout":       y = drop(x)
  * "norm":          y = drop(layer_norm(x)), as the rows that a table's pull returned are made the input of a dense model
  * "norm_grad":     its gradient, which becomes the gradient of the rows for the table's push, and those of weight and bias
  * "add_norm":      s = residual + drop(x), y = layer_norm(s): the step between two layers of a dense model
  * "add_norm_grad": its gradient
`act` is the type of the activations (x and y of dropout and add_norm, y of norm), `stream` that of what is normalised (x of
norm, residual and s of add_norm), `affine` that of weight and bias ("none": there are none).  `p` is the probability of
dropping a value, 0: no dropout.  `stats`: the forward pass returns the rows' mean and 1 / deviation, as training needs them.
`joined`: s goes on beside y, and has a gradient of its own.  `pad`: the rows of every input lie that many values apart, as
slices of wider matrices do.

Dropout keeps the value in row r, column c if a 32-bit word is at least p * 2^32, and multiplies it by 1 / (1 - p).  The word
is number c % 4 of Philox4x32 with 7 rounds (Salmon, Moraes, Dror, Shaw: Parallel random numbers: as easy as 1, 2, 3; SC 2011),
with the counter (r * ceil(width / 4) + c // 4, step), two 64-bit numbers, low words first, and the seed as key.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
_SIZES = {"f32": 4, "bf16": 2, "f16": 2}
_EPS = 1e-5
_DEFAULTS = {"op": "norm", "rows": 1, "width": 128, "stream": "f32", "act": "bf16", "affine": "f32", "p": 0.0, "stats": True,
             "joined": True, "pad": 0}


def _case(name=None, **options):
    case = dict(_DEFAULTS, **options)
    assert set(case) == set(_DEFAULTS)
    if name:
        case["name"] = name
    return case


def listed():
    return [
        # serving: the rows of a request of 128 samples of 26 fields, normalised for a dense model in bfloat16
        _case("norm_serve_128", rows=128 * 26, stats=False),
        # serving: one token of a wide model
        _case("norm_one_row", rows=1, width=8192, stream="bf16", affine="act", stats=False),
        # training, the rows of the large batch (65536 samples of 26 fields): normalised and dropped, and the gradient that the
        # table's next push takes
        _case("norm_rows_65536", rows=65536 * 26, p=0.1),
        _case("norm_rows_65536_grad", op="norm_grad", rows=65536 * 26, p=0.1),
        # sizes nobody rounds: 39 fields of 37 floats, a ragged batch, all of it in 32 bits
        _case("norm_odd_grad", op="norm_grad", rows=5003 * 39, width=37, act="f32"),
        # a hidden layer in 16 bits, weights included
        _case("norm_hidden_grad", op="norm_grad", rows=4096, width=8192, stream="f16", act="f16", affine="act"),
        # decoding: the step between two layers for 64 tokens
        _case("add_norm_64", op="add_norm", rows=64, width=4096, stream="bf16", affine="act", stats=False),
        # training: the step between two layers, the sum kept in 32 bits beside activations in 16
        _case("add_norm_train", op="add_norm", rows=16384, width=4096, p=0.1),
        _case("add_norm_train_grad", op="add_norm_grad", rows=16384, width=4096, p=0.1),
        # dropout of the pulled rows of the reference's own batch, 2048 samples of 26 fields
        _case("dropout_2048", op="dropout", rows=2048 * 26, act="f32", p=0.1),
        # of ragged rows: 39 fields of 37 values side by side
        _case("dropout_odd", op="dropout", rows=5003, width=39 * 37, act="f16", p=0.25),
        # of the large batch, its 26 fields of 128 values side by side
        _case("dropout_65536", op="dropout", rows=65536, width=26 * 128, p=0.5),
    ]


_MOST_VALUES = 65536 * 26 * 128        # of a matrix, in the largest listed cases
_MOST_BYTES = _MOST_VALUES * 10        # that a pass moves, in the largest listed case


def _log_uniform(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["dropout", "norm", "norm", "norm_grad", "norm_grad", "add_norm", "add_norm_grad"])
    stream, act = rng.choice([("f32", "f32"), ("f32", "bf16"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")])
    case = _case(op=op, stream=stream, act=act, affine=rng.choice(["f32", "act", "act", "none"]),
                 p=rng.choice([0.0, 0.1, 0.1, 0.25, 0.5]), stats=rng.random() < 0.7, joined=rng.random() < 0.7,
                 pad=rng.choice([0, 0, 0, 5, 64]))
    if op == "dropout":
        case["p"] = case["p"] or 0.2
    width = rng.choice([16, 32, 64, 128, 1024, 4096, _log_uniform(rng, 8, 16384), _log_uniform(rng, 8, 16384)])
    case["width"] = width
    case["rows"] = max(1, min(_log_uniform(rng, 1, 2_000_000), _MOST_VALUES // (width + case["pad"])))
    case["rows"] = max(1, min(case["rows"], case["rows"] * _MOST_BYTES // work(case)["bytes"]))
    return case


# ---- inputs -----------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    rows, width, act, stream = case["rows"], case["width"], _TYPES[case["act"]], _TYPES[case["stream"]]

    def values(dtype, std, mean=0.0):
        wide = torch.empty((rows, width + case["pad"]), device="cuda").normal_(mean, std, generator=gen)
        return wide.to(dtype)[:, :width]

    def per_column(std, mean):
        if case["affine"] == "none":
            return None
        dtype = torch.float32 if case["affine"] == "f32" else act
        return torch.empty(width, device="cuda").normal_(mean, std, generator=gen).to(dtype)

    # the dropout of one layer (the seed) in one training step
    state = {"case": case, "drop": (case["p"], seed * 2 + 1, 1000 + seed % 977) if case["p"] else None}
    if case["op"] == "dropout":
        state["x"] = values(act, 1.0)
        return state
    state["weight"], state["bias"] = per_column(0.1, 1.0), per_column(0.1, 0.0)
    if case["op"] == "norm":
        state["x"] = values(stream, 0.1, 0.02)            # rows of a table that started as Normal(0, 0.1)
    elif case["op"] == "add_norm":
        state["x"], state["residual"] = values(act, 1.0), values(stream, 2.0, 0.3)
    else:
        # the gradient of a mean over many samples, and what the forward pass left
        state["dy"] = values(act, 1e-3)
        if case["op"] == "norm_grad":
            state["x"] = normed = values(stream, 0.1, 0.02)
        else:
            state["s"] = normed = values(stream, 2.0, 0.3)
            state["ds"] = values(stream, 1e-3) if case["joined"] else None
        _, state["mean"], state["rstd"] = _normalise(normed)
    torch.cuda.synchronize()
    return state


# ---- the plain forms --------------------------------------------------------------------------------------------------
def _kept(drop, rows, width):
    """Truth values [rows, width]: which values dropout keeps."""
    p, seed, step = drop
    low = 0xFFFFFFFF
    quads = (width + 3) // 4
    at = torch.arange(rows * quads, device="cuda")
    c0, c1, c2, c3 = at & low, at >> 32, torch.full_like(at, step & low), torch.full_like(at, step >> 32)
    k0, k1 = seed & low, seed >> 32
    for _ in range(7):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57         # modulo 2^64
        c0, c1, c2, c3 = (b >> 32 & low) ^ c1 ^ k0, b & low, (a >> 32 & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    words = torch.stack((c0, c1, c2, c3), dim=1).view(rows, quads * 4)[:, :width]
    return words >= round(p * 2 ** 32)


def _dropped(v, drop):
    if drop is None:
        return v
    return torch.where(_kept(drop, *v.shape), v * (1 / (1 - drop[0])), 0.0)


def _normalise(x):
    x = x.float()
    mean = x.mean(1)
    off = x - mean[:, None]
    rstd = 1 / torch.sqrt((off * off).mean(1) + _EPS)
    return off * rstd[:, None], mean, rstd


def _scaled(normed, state):
    if state["weight"] is None:
        return normed
    return normed * state["weight"].float() + state["bias"].float()


def _norm_gradient(g, x, state):
    """The gradients of x, weight and bias from that of weight * normalised + bias."""
    normed = (x.float() - state["mean"][:, None]) * state["rstd"][:, None]
    dweight = dbias = None
    if state["weight"] is not None:
        dtype = state["weight"].dtype
        dweight, dbias = (g * normed).sum(0).to(dtype), g.sum(0).to(dtype)
        g = g * state["weight"].float()
    dx = state["rstd"][:, None] * (g - g.mean(1, keepdim=True) - normed * (g * normed).mean(1, keepdim=True))
    return dx, dweight, dbias


def _plain(state):
    case, drop = state["case"], state["drop"]
    act, stream = _TYPES[case["act"]], _TYPES[case["stream"]]
    if case["op"] == "dropout":
        return _dropped(state["x"].float(), drop).to(act)
    if case["op"] == "norm":
        normed, mean, rstd = _normalise(state["x"])
        y = _dropped(_scaled(normed, state), drop).to(act)
        return (y, mean, rstd) if case["stats"] else y
    if case["op"] == "add_norm":
        s = state["residual"].float() + _dropped(state["x"].float(), drop)
        normed, mean, rstd = _normalise(s)
        y = _scaled(normed, state).to(act)
        return (y, s.to(stream), mean, rstd) if case["stats"] else (y, s.to(stream))
    if case["op"] == "norm_grad":
        dx, dweight, dbias = _norm_gradient(_dropped(state["dy"].float(), drop), state["x"], state)
        return dx.to(stream), dweight, dbias
    ds, dweight, dbias = _norm_gradient(state["dy"].float(), state["s"], state)
    if state["ds"] is not None:
        ds = ds + state["ds"].float()
    return _dropped(ds, drop).to(act), ds.to(stream), dweight, dbias


# ---- one pass -----------------------------------------------------------------------------------------------------------
def run(state):
    if not own:
        return _plain(state)
    from hetuctr_amd import nn
    case = state["case"]
    drop = nn.Drop(*state["drop"]) if state["drop"] else None
    if case["op"] == "dropout":
        return nn.dropout(state["x"], drop)
    weight, bias = state["weight"], state["bias"]
    if case["op"] == "norm":
        return nn.layer_norm(state["x"], weight, bias, _EPS, drop=drop, dtype=_TYPES[case["act"]], stats=case["stats"])
    if case["op"] == "add_norm":
        return nn.dropout_add_layer_norm(state["x"], state["residual"], weight, bias, _EPS, drop=drop, stats=case["stats"])
    if case["op"] == "norm_grad":
        return nn.layer_norm_backward(state["dy"], state["x"], state["mean"], state["rstd"], weight, bias, drop=drop)
    return nn.dropout_add_layer_norm_backward(state["dy"], state["ds"], state["s"], state["mean"], state["rstd"], weight, bias,
                                              drop=drop)


# ---- what a pass cannot do without ----------------------------------------------------------------------------------------
def work(case):
    rows, width, act, stream = case["rows"], case["width"], _SIZES[case["act"]], _SIZES[case["stream"]]
    n, op, dropped = rows * width, case["op"], 2 if case["p"] else 0      # a comparison and a product
    # weight and bias, or their gradients
    columns = 0 if case["affine"] == "none" else 2 * width * (4 if case["affine"] == "f32" else act)
    stats = 8 * rows if case["stats"] or op.endswith("grad") else 0
    if op == "dropout":
        return {"bytes": 2 * n * act, "flops": 2 * n}
    # forward: the mean, the variance (2 and a subtraction), the product with 1 / deviation, weight and bias
    if op == "norm":
        return {"bytes": n * (stream + act) + stats + columns, "flops": n * (7 + dropped)}
    if op == "add_norm":
        return {"bytes": n * 2 * (act + stream) + stats + columns, "flops": n * (8 + dropped)}
    # gradient: the normalised value (2), the weight, two sums over the row (3), two over the column (3), the result (4); the
    # weight is read, the gradients of weight and bias are written
    columns += columns // 2
    if op == "norm_grad":
        return {"bytes": n * (act + 2 * stream) + stats + columns, "flops": n * (13 + dropped)}
    read = act + stream * (2 if case["joined"] else 1)
    # without dropout and in the same type the gradients of x and residual are one
    written = stream + (act if case["p"] or act != stream else 0)
    return {"bytes": n * (read + written) + stats + columns, "flops": n * (13 + dropped + case["joined"])}


# ---- the definitions in 64 bits -------------------------------------------------------------------------------------------
def _high_word(a, m):
    """The upper 32 bits of the products of 32-bit numbers, from halves of 16 bits."""
    al, ah, ml, mh = a % 65536, a // 65536, m % 65536, m // 65536
    middle = ah * ml + al * ml // 65536
    return ah * mh + middle // 65536 + (al * mh + middle % 65536) // 65536


def _low_word(a, m):
    return ((a // 65536 * m % 65536) * 65536 + a % 65536 * m) % 2 ** 32


def _exact_factors(drop, rows, width):
    """What dropout multiplies each value by."""
    if drop is None:
        return torch.ones((), device="cuda", dtype=torch.float64)
    p, seed, step = drop
    column = torch.arange(width, device="cuda") // 4
    counter = torch.arange(rows, device="cuda")[:, None] * -(-width // 4) + column[None, ::4]
    x = [counter % 2 ** 32, counter // 2 ** 32, torch.full_like(counter, step % 2 ** 32), torch.full_like(counter, step // 2 ** 32)]
    for r in range(7):
        key0, key1 = (seed + r * 0x9E3779B9) % 2 ** 32, (seed // 2 ** 32 + r * 0xBB67AE85) % 2 ** 32
        x = [_high_word(x[2], 0xCD9E8D57) ^ x[1] ^ key0, _low_word(x[2], 0xCD9E8D57),
             _high_word(x[0], 0xD2511F53) ^ x[3] ^ key1, _low_word(x[0], 0xD2511F53)]
    out = torch.empty((rows, width), device="cuda", dtype=torch.float64)
    for word in range(4):
        kept = (x[word] >= round(p * 2 ** 32)).double() / (1 - p)
        out[:, word::4] = kept[:, :out[:, word::4].shape[1]]
    return out


def exact(case, seed):
    state = prepare(case, seed)
    wide = {k: v.double() for k, v in state.items() if isinstance(v, torch.Tensor)}
    op, rows, width = case["op"], case["rows"], case["width"]
    factors = _exact_factors(state["drop"], rows, width)
    if op == "dropout":
        return wide["x"] * factors
    weight, bias = wide.get("weight"), wide.get("bias")
    if op in ("norm", "add_norm"):
        v = wide["x"] if op == "norm" else wide["residual"] + factors * wide["x"]
        var, mean = torch.var_mean(v, dim=1, correction=0)
        rstd = (var + _EPS).rsqrt()
        y = (v - mean.unsqueeze(1)).mul_(rstd.unsqueeze(1))
        if weight is not None:
            y = torch.addcmul(bias, y, weight)
        outs = [y * factors] if op == "norm" else [y, v]
        outs += [mean, rstd] if case["stats"] else []
        return tuple(outs) if len(outs) > 1 else outs[0]
    # the gradient, with the rows' statistics as the forward pass gave them
    v = wide["x" if op == "norm_grad" else "s"]
    hat = v.sub_(wide["mean"].unsqueeze(1)).mul_(wide["rstd"].unsqueeze(1))
    dy = wide["dy"] * factors if op == "norm_grad" else wide["dy"]
    dbias = dy.sum(0) if weight is not None else None
    dweight = torch.mul(dy, hat).sum(0) if weight is not None else None
    dhat = dy * weight if weight is not None else dy
    along = torch.mul(dhat, hat).sum(1) / width
    dv = (dhat - (dhat.sum(1) / width).unsqueeze(1) - hat * along.unsqueeze(1)) * wide["rstd"].unsqueeze(1)
    if op == "norm_grad":
        return dv, dweight, dbias
    if "ds" in wide:
        dv = dv + wide["ds"]
    return dv * factors, dv, dweight, dbias

"""The operators between the table's rows and a dense model (hetuctr_amd.nn, hctr_dropout, hctr_layer_norm, ..) against their
definitions in 64 bits.

Tolerances.  A result is rounded once to its type: UNIT * |value| (half a step of the smallest normal value below it).  Before
that it is off by some units of 2^-24 of the magnitudes that its sums and differences are made of.  A sum of n terms that a
lane adds one by one and the lanes join in pairs is off by at most (terms per lane + 2 * log2(lanes) + 2) units; a lane has at most
32 columns of a row, and of the rows below at most some hundred of a column: ROW and COLUMN units allow for that.
"""
import numpy as np
import pytest
import torch

from hetuctr_amd import capi, nn
from tests import dense_reference as ref

gpu = pytest.mark.gpu
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CODES = {"f32": capi.F32, "bf16": capi.BF16, "f16": capi.F16}
PAIRS = [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f16")]
ROW, COLUMN = 64 * 2.0 ** -24, 256 * 2.0 ** -24
EPS = 1e-5


def name_of(dtype):
    return next(k for k, v in TYPES.items() if v == dtype)


def wide(t):
    return None if t is None else t.detach().cpu().double().numpy()


def values(shape, kind, seed, std=1.0, mean=0.0):
    gen = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=gen) * std + mean).to(TYPES[kind]).cuda()


def check(got, want, size, units, what=""):
    """|got - want| <= one rounding to got's type + `units` * size"""
    kind = name_of(got.dtype)
    got = wide(got).reshape(want.shape)
    off = units * size
    allowed = off + ref.UNIT[kind] * np.maximum(np.abs(want) + off, ref.TINY[kind])
    bad = ~(np.abs(got - want) <= allowed)
    assert not bad.any(), "%s: %d of %d values, worst %.3g of what is allowed" % (
        what, bad.sum(), bad.size, np.nanmax(np.abs(got - want) / allowed))


# ---- dropout ------------------------------------------------------------------------------------------------------------
def test_reference_generator_gives_the_published_words():
    # the known answers that accompany the paper's generator: all bits clear, all bits set, digits of pi
    ones, pi = 0xFFFFFFFF, (0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344, 0xA4093822, 0x299F31D0)
    for rounds, counter, key, words in [
            (7, (0, 0, 0, 0), (0, 0), (0x5F6FB709, 0x0D893F64, 0x4F121F81, 0x4F730A48)),
            (7, (ones,) * 4, (ones,) * 2, (0x5207DDC2, 0x45165E59, 0x4D8EE751, 0x8C52F662)),
            (7, pi[:4], pi[4:], (0x4DFCCABA, 0x190A87F0, 0xC47362BA, 0xB6B5242A)),
            (10, (0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
            (10, pi[:4], pi[4:], (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))]:
        assert tuple(int(w) for w in ref.philox(counter, key, rounds)) == words


def dropped(x, drop):
    """What dropout of the GPU tensor x gives, bit for bit: one product in 32 bits, one rounding."""
    keep = torch.from_numpy(ref.kept(x.shape[0], x.shape[1], *drop)) if drop[0] < 1 else torch.zeros(x.shape, dtype=torch.bool)
    scale = np.float32(1 / (1 - drop[0])) if drop[0] < 1 else np.float32(0)
    return torch.where(keep, (x.cpu().float() * float(scale)).to(x.dtype), torch.zeros((), dtype=x.dtype))


SHAPES = [(1, 1), (7, 1), (3, 3), (5, 4), (9, 7), (300, 8), (64, 12), (17, 37), (1000, 16), (33, 128), (5, 1443), (6, 3328), (2, 16385),
          (1, 70001)]


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_dropout_is_the_function_of_position_seed_and_step(shape, kind):
    x = values(shape, kind, 1)
    for drop in [(0.1, 5, 0), (0.5, -3, 2 ** 40 + 1), (0.999, 2 ** 63 + 12345, 7), (1.0, 1, 1), (2.0 ** -40, 1, 1), (0.0, 1, 1)]:
        want = dropped(x, drop) if drop[0] > 2.0 ** -33 else x.cpu()
        got = nn.dropout(x, nn.Drop(*drop)).cpu()
        assert got.dtype == x.dtype and torch.equal(got, want), drop
    assert torch.equal(nn.dropout(x, None), x)


@gpu
def test_dropout_keeps_as_many_as_it_says():
    n = 1 << 20
    x = torch.ones((1024, 1024), device="cuda")
    for p in (0.1, 0.5, 0.9):
        share = (nn.dropout(x, nn.Drop(p, 11, 3)) == 0).sum().item() / n
        assert abs(share - p) < 5 * (p * (1 - p) / n) ** 0.5
    # neither another step nor another seed drops the same values, nor do they shift them
    a = nn.dropout(x, nn.Drop(0.5, 11, 3)) != 0
    for other in (nn.Drop(0.5, 11, 4), nn.Drop(0.5, 12, 3)):
        b = nn.dropout(x, other) != 0
        for shift in (0, 1, 4, 1024):
            both = (a.flatten()[shift:] == b.flatten()[:n - shift]).float().mean().item()
            assert abs(both - 0.5) < 5 * 0.5 / n ** 0.5


@gpu
@pytest.mark.parametrize("kind", TYPES)
def test_what_is_dropped_may_be_anything(kind):
    drop = (0.5, 9, 9)
    keep = torch.from_numpy(ref.kept(40, 100, *drop)).cuda()
    x = values((40, 100), kind, 2)
    for odd in (float("nan"), float("inf"), -float("inf"), torch.finfo(TYPES[kind]).min):
        bad = torch.where(keep, x, torch.full_like(x, odd))
        got = nn.dropout(bad, nn.Drop(*drop))
        assert torch.equal(got, nn.dropout(torch.where(keep, x, torch.zeros_like(x)), nn.Drop(*drop)))
        assert (got[~keep] == 0).all()


def layouts(x):
    """The values of the [rows, width] tensor x in other places of memory."""
    rows, width = x.shape
    apart = torch.full((rows, width + 3), float("nan"), dtype=x.dtype, device="cuda")
    apart[:, 1:width + 1] = x
    yield "a slice of wider rows", apart[:, 1:width + 1]
    every = torch.full((2 * rows, width), float("nan"), dtype=x.dtype, device="cuda")
    every[::2] = x
    yield "every other row", every[::2]
    yield "columns apart", x.t().contiguous().t()
    block = torch.full((rows * width + 1,), float("nan"), dtype=x.dtype, device="cuda")
    block[1:] = x.flatten()
    yield "behind one element", block[1:].view(rows, width)


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("width", [5, 64, 200])
def test_dropout_of_any_layout(kind, width):
    x = values((30, width), kind, 3)
    drop = nn.Drop(0.3, 4, 4)
    want = nn.dropout(x, drop)
    for what, other in layouts(x):
        assert torch.equal(other, x), what
        assert torch.equal(nn.dropout(other, drop), want), what
    assert torch.equal(nn.dropout(x.view(5, 6, width), drop), want.view(5, 6, width))
    assert torch.equal(nn.dropout(x.view(5, 6, width).transpose(0, 1), drop), nn.dropout(x.view(5, 6, width).transpose(0, 1).contiguous(), drop))
    same = x[:1].expand(30, width)                 # rows that are one and the same are dropped apart
    assert torch.equal(nn.dropout(same, drop), nn.dropout(same.contiguous(), drop))
    assert torch.equal(nn.dropout(x[0], drop), want[0])


@gpu
def test_dropout_in_place_and_of_rows_far_apart():
    width, far = 24, 2 ** 31 + 5                   # elements between rows: the third lies beyond 2^32
    block = torch.empty(2 * far + width, dtype=torch.float16, device="cuda")
    x = torch.as_strided(block, (3, width), (far, 1))
    x.copy_(values((3, width), "f16", 5))
    near = x.clone()
    drop = (0.4, 8, 2)
    want = nn.dropout(near, nn.Drop(*drop))
    assert torch.equal(nn.dropout(x, nn.Drop(*drop)), want)
    stream = torch.cuda.current_stream().cuda_stream
    for t, stride in ((x, far), (near, width)):
        at = (t.data_ptr(), stride)
        capi.dropout(3, width, at, at, drop + (0,), capi.F16, stream)
        assert torch.equal(t, want)


@gpu
@pytest.mark.parametrize("kind", TYPES)
@pytest.mark.parametrize("rows, width", [(50, 3), (40, 37), (7, 1443), (300, 12), (1, 1001)])
def test_dropout_in_place_of_ragged_rows(rows, width, kind):
    x = values((rows, width + 2), kind, 7)[:, :width]
    drop = (0.4, 8, 2)
    want = nn.dropout(x, nn.Drop(*drop))
    at = (x.data_ptr(), width + 2)
    capi.dropout(rows, width, at, at, drop + (0,), CODES[kind], torch.cuda.current_stream().cuda_stream)
    assert torch.equal(x, want)


@gpu
def test_counters_beyond_32_bits():
    # 2^34 values and some: their quads, and with them the counter's low word, pass 2^32 in the last rows
    width, rows = 1024, 2 ** 24 + 3
    drop, quads = (0.3, 77, 5), width // 4
    at = np.arange((rows - 4) * quads, rows * quads, dtype=np.uint64)
    words = ref.philox([at & np.uint64(0xFFFFFFFF), at >> np.uint64(32), np.uint64(5), np.uint64(0)], (77, 0), 7)
    keep = torch.from_numpy(words.T.reshape(4, width) >= np.uint64(round(0.3 * 2 ** 32)))
    assert (at >> np.uint64(32)).max() == 1 and (at >> np.uint64(32)).min() == 0
    want = torch.where(keep, torch.tensor(1 / 0.7, dtype=torch.float32).half(), torch.tensor(0.0).half())
    x = torch.ones((rows, width), dtype=torch.float16, device="cuda")
    place = (x.data_ptr(), width)
    capi.dropout(rows, width, place, place, drop + (0,), capi.F16, torch.cuda.current_stream().cuda_stream)
    assert torch.equal(x[-4:].cpu(), want)
    # rows without spread become their bias, which is dropped likewise
    x.zero_()
    y = nn.layer_norm(x, None, torch.ones(width, dtype=torch.float16, device="cuda"), drop=nn.Drop(*drop))
    assert torch.equal(y[-4:].cpu(), want)
    del x, y
    torch.cuda.empty_cache()


@gpu
def test_step_tensor_is_added_to_the_step():
    x = values((20, 40), "f32", 6)
    for base, more in ((3, 4), (0, 2 ** 40), (2 ** 64 - 1, 2)):
        step = torch.tensor([more], device="cuda")
        assert torch.equal(nn.dropout(x, nn.Drop(0.5, 1, base, step)), nn.dropout(x, nn.Drop(0.5, 1, (base + more) % 2 ** 64)))


# ---- layer normalisation --------------------------------------------------------------------------------------------------
WIDTHS = [1, 2, 3, 4, 5, 8, 12, 16, 17, 31, 32, 36, 37, 64, 65, 100, 128, 129, 200, 256, 260, 500, 512, 513, 1000, 1024, 1025, 1443, 2048,
          2056, 3328, 4096, 4100, 8192, 8200, 16384, 16388, 20001]


def row_count(width):
    return max(2, min(77, 60000 // width)) + 1


def affine(kind, width, act):
    if kind == "none":
        return None, None
    kind = "f32" if kind == "f32" else act
    return values(width, kind, 21, 0.2, 1.0), values(width, kind, 22, 0.2)


def forward_size(x, weight, mean, rstd):
    """what the rounding errors of a normalised row scale with"""
    off = (np.abs(x) + np.abs(mean)[:, None] + np.abs(x).mean(1, keepdims=True)) * rstd[:, None]
    # the variance's own error, relative, moves every value of the row
    h = np.abs(x - mean[:, None]) * rstd[:, None]
    off = off + h * (1 + (off * h).mean(1, keepdims=True))
    return off if weight is None else off * np.abs(weight)


def check_norm(x, weight, bias, drop, got, eps=EPS):
    y, mean, rstd = got
    v, w, b = wide(x), wide(weight), wide(bias)
    want_mean, want_rstd = ref.statistics(v, eps)
    f = ref.factors(v.shape[0], v.shape[1], drop)
    size = forward_size(v, w, want_mean, want_rstd) + (0 if b is None else np.abs(b))
    check(y, ref.normalise(v, w, b, eps) * f, size * f, ROW, "y")
    check(mean, want_mean, np.abs(v).mean(1), ROW, "mean")
    h = (v - want_mean[:, None]) * want_rstd[:, None]
    spread = 1 + (np.abs(h) * (np.abs(v) + np.abs(want_mean)[:, None]) * want_rstd[:, None]).mean(1)
    check(rstd, want_rstd, want_rstd * spread, ROW, "rstd")


@gpu
@pytest.mark.parametrize("stream, act", PAIRS)
@pytest.mark.parametrize("width", WIDTHS)
def test_layer_norm(width, stream, act):
    rows = row_count(width)
    x = values((rows, width), stream, width, 0.5, 0.1)
    for kind, drop in (("f32", None), ("act", (0.25, 3, width)), ("none", None)):
        weight, bias = affine(kind, width, act)
        got = nn.layer_norm(x, weight, bias, EPS, drop=drop and nn.Drop(*drop), dtype=TYPES[act], stats=True)
        assert got[0].dtype == TYPES[act] and got[0].shape == x.shape
        check_norm(x, weight, bias, drop, got)
        alone = nn.layer_norm(x, weight, bias, EPS, drop=drop and nn.Drop(*drop), dtype=TYPES[act])
        assert torch.equal(alone, got[0])


@gpu
@pytest.mark.parametrize("stream, act", PAIRS)
@pytest.mark.parametrize("width", WIDTHS)
def test_dropout_add_layer_norm(width, stream, act):
    rows = row_count(width)
    x, residual = values((rows, width), act, width), values((rows, width), stream, width + 1, 2.0, 0.3)
    for kind, drop in (("act", None), ("f32", (0.25, 3, width)), ("none", (0.1, 4, width))):
        weight, bias = affine(kind, width, act)
        y, s, mean, rstd = nn.dropout_add_layer_norm(x, residual, weight, bias, EPS, drop=drop and nn.Drop(*drop), stats=True)
        assert s.dtype == TYPES[stream] and y.dtype == TYPES[act]
        branch = wide(x) * ref.factors(rows, width, drop)
        total = wide(residual) + branch
        check(s, total, np.abs(branch) + np.abs(total), 2 * 2.0 ** -24, "s")
        # the statistics of a sum that carries its own rounding of 2^-24: within what ROW allows for
        v, w, b = total, wide(weight), wide(bias)
        want_mean, want_rstd = ref.statistics(v, EPS)
        size = forward_size(np.abs(wide(residual)) + np.abs(branch), w, want_mean, want_rstd) + forward_size(v, w, want_mean, want_rstd)
        check(y, ref.normalise(v, w, b, EPS), size + (0 if b is None else np.abs(b)), ROW, "y")
        check(mean, want_mean, (np.abs(wide(residual)) + np.abs(branch)).mean(1), ROW, "mean")
        h = (v - want_mean[:, None]) * want_rstd[:, None]
        sizes = np.abs(wide(residual)) + np.abs(branch) + np.abs(want_mean)[:, None]
        check(rstd, want_rstd, want_rstd * (1 + (np.abs(h) * sizes * want_rstd[:, None]).mean(1)), ROW, "rstd")
        alone = nn.dropout_add_layer_norm(x, residual, weight, bias, EPS, drop=drop and nn.Drop(*drop))
        assert torch.equal(alone[0], y) and torch.equal(alone[1], s)


@gpu
@pytest.mark.parametrize("stream, act", PAIRS)
@pytest.mark.parametrize("width", WIDTHS)
def test_layer_norm_gradient(width, stream, act):
    rows = row_count(width)
    x, dy = values((rows, width), stream, width, 0.5, 0.1), values((rows, width), act, width + 2, 0.01)
    mean, rstd = (torch.from_numpy(t).float().cuda() for t in ref.statistics(wide(x), EPS))
    for kind, drop in (("f32", None), ("act", (0.25, 3, width)), ("none", (0.5, 1, 1))):
        weight, bias = affine(kind, width, act)
        dx, dweight, dbias = nn.layer_norm_backward(dy, x, mean, rstd, weight, bias, drop=drop and nn.Drop(*drop))
        g = wide(dy) * ref.factors(rows, width, drop)
        want, size = ref.gradient(g, wide(x), wide(mean), wide(rstd), wide(weight))
        assert dx.dtype == x.dtype
        check(dx, want[0], size[0], ROW, "dx")
        if weight is None:
            assert dweight is None and dbias is None
        else:
            assert dweight.dtype == weight.dtype and dbias.dtype == bias.dtype
            check(dweight, want[1], size[1], COLUMN, "dweight")
            check(dbias, want[2], size[2], COLUMN, "dbias")


@gpu
@pytest.mark.parametrize("stream, act", PAIRS)
@pytest.mark.parametrize("width", WIDTHS)
def test_dropout_add_layer_norm_gradient(width, stream, act):
    rows = row_count(width)
    s, dy = values((rows, width), stream, width, 2.0, 0.3), values((rows, width), act, width + 2, 0.01)
    ds = values((rows, width), stream, width + 3, 0.01)
    mean, rstd = (torch.from_numpy(t).float().cuda() for t in ref.statistics(wide(s), EPS))
    for kind, drop, more in (("f32", (0.25, 3, width), ds), ("act", None, None), ("none", (0.5, 1, 1), None), ("act", None, ds)):
        weight, bias = affine(kind, width, act)
        dx, dresidual, dweight, dbias = nn.dropout_add_layer_norm_backward(dy, more, s, mean, rstd, weight, bias,
                                                                           drop=drop and nn.Drop(*drop))
        want, size = ref.gradient(wide(dy), wide(s), wide(mean), wide(rstd), wide(weight))
        total = want[0] + (0 if more is None else wide(more))
        sizes = size[0] + np.abs(total)
        assert dx.dtype == dy.dtype and dresidual.dtype == s.dtype
        check(dresidual, total, sizes, ROW, "dresidual")
        f = ref.factors(rows, width, drop)
        check(dx, total * f, sizes * f, ROW, "dx")
        if weight is not None:
            check(dweight, want[1], size[1], COLUMN, "dweight")
            check(dbias, want[2], size[2], COLUMN, "dbias")


@gpu
@pytest.mark.parametrize("rows, width", [(1, 1), (1, 128), (2, 37), (1, 8192), (4097, 16), (20000, 37), (3000, 128), (1300, 1024), (600, 4096)])
def test_weight_gradient_over_many_rows_or_few(rows, width):
    # a lane adds up to rows / (rows a launch works on at once) terms one by one: at most some tens here, as COLUMN allows
    x, dy = values((rows, width), "f32", 1, 0.5, 0.1), values((rows, width), "bf16", 2, 0.01)
    weight, bias = affine("f32", width, "bf16")
    y, mean, rstd = nn.layer_norm(x, weight, bias, EPS, dtype=torch.bfloat16, stats=True)
    dx, dweight, dbias = nn.layer_norm_backward(dy, x, mean, rstd, weight, bias)
    want, size = ref.gradient(wide(dy), wide(x), wide(mean), wide(rstd), wide(weight))
    for got, w, z, units in zip((dx, dweight, dbias), want, size, (ROW, COLUMN, COLUMN)):
        check(got, w, z, units)
    # one of the two alone, and neither: the same bits
    again = nn.layer_norm_backward(dy, x, mean, rstd, weight, None)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dweight) and again[2] is None
    last = nn.layer_norm_backward(dy, x, mean, rstd, None, bias)
    assert last[1] is None and torch.equal(last[2], dbias)


@gpu
@pytest.mark.parametrize("stream, act", PAIRS)
@pytest.mark.parametrize("rows, width", [(513, 3), (900, 12), (2000, 37), (1500, 64), (700, 333), (600, 1000), (530, 1443), (520, 2056),
                                         (140, 4100), (100, 8192), (66, 16388)])
def test_gradients_of_more_rows_than_one_launch_takes(rows, width, stream, act):
    x, dy = values((rows, width), stream, 1, 0.5, 0.1), values((rows, width), act, 2, 0.01)
    mean, rstd = (torch.from_numpy(t).float().cuda() for t in ref.statistics(wide(x), EPS))
    weight, bias = affine("act", width, act)
    drop = (0.25, 3, width)
    f = ref.factors(rows, width, drop)
    for g, got in ((wide(dy) * f, nn.layer_norm_backward(dy, x, mean, rstd, weight, bias, drop=nn.Drop(*drop))),
                   (wide(dy), nn.dropout_add_layer_norm_backward(dy, x, x, mean, rstd, weight, bias, drop=nn.Drop(*drop))[1:])):
        want, size = ref.gradient(g, wide(x), wide(mean), wide(rstd), wide(weight))
        more = 0 if g.shape == f.shape and np.array_equal(g, wide(dy) * f) else wide(x)
        check(got[0], want[0] + more, size[0] + np.abs(want[0] + more), ROW, "rows")
        check(got[1], want[1], size[1], COLUMN, "dweight")
        check(got[2], want[2], size[2], COLUMN, "dbias")


# ---- gradients against differences ------------------------------------------------------------------------------------------
def test_reference_gradient_against_differences():
    rng = np.random.default_rng(3)
    x, dy, w, b = rng.normal(0.2, 0.7, (5, 23)), rng.normal(size=(5, 23)), rng.normal(1, 0.2, 23), rng.normal(size=23)
    (dx, dw, db), _ = ref.gradient(dy, x, *ref.statistics(x, EPS), w)
    loss = lambda x, w, b: (ref.normalise(x, w, b, EPS) * dy).sum()
    for at, grad in ((0, dx), (1, dw), (2, db)):
        args = [x, w, b]
        along = rng.normal(size=args[at].shape)
        h = 1e-5
        up, down = list(args), list(args)
        up[at], down[at] = args[at] + h * along, args[at] - h * along
        slope = (loss(*up) - loss(*down)) / (2 * h)
        # the error of the difference: h^2 / 6 times the third derivative, and 2^-52 |loss| / h
        assert abs(slope - (grad * along).sum()) < 1e-6 * max(1, abs(slope))


@gpu
@pytest.mark.parametrize("width", [5, 37, 128, 1000])
def test_gradients_against_differences(width):
    # Slopes of sum(y * c) + sum(s * e) along a direction, from the results of the forward calls in 32 bits.  h = 2^-6: the
    # difference is off by the third derivative times h^2 / 6 (some 1e-4 of the slope's terms) and by the roundings of y, 2^-24 *
    # |y| / h = 4e-6 of each term.  The slope's terms are of size |c| |along| sqrt(values); 1e-2 of that allows for both.
    drop, h = nn.Drop(0.2, 5, 6), 2.0 ** -6
    x, r, c, e = (values((6, width), "f32", i) for i in range(4))
    w, b = values(width, "f32", 8, 0.2, 1.0), values(width, "f32", 9)

    def results(x, r, w, b):
        y, s = nn.dropout_add_layer_norm(x, r, w, b, EPS, drop=drop)
        z = nn.layer_norm(r, w, b, EPS, drop=drop)
        return wide(y), wide(s), wide(z)

    y, s, mean, rstd = nn.dropout_add_layer_norm(x, r, w, b, EPS, drop=drop, stats=True)
    added = nn.dropout_add_layer_norm_backward(c, e, s, mean, rstd, w, b, drop=drop)
    _, mean, rstd = nn.layer_norm(r, w, b, EPS, drop=drop, stats=True)
    plain = (None,) + nn.layer_norm_backward(c, r, mean, rstd, w, b, drop=drop)
    args = [x, r, w, b]
    for at in range(4):
        along = values(args[at].shape, "f32", 30 + at)
        up, down = list(args), list(args)
        up[at], down[at] = args[at] + h * along, args[at] - h * along
        (y1, s1, z1), (y0, s0, z0) = results(*up), results(*down)
        span = wide(up[at]) - wide(down[at])                       # as it was rounded
        sloped = ((y1 - y0) * wide(c) + (s1 - s0) * wide(e)).sum()
        assert abs(sloped - (wide(added[at]) * span).sum()) < 1e-2 * 2 * h * 2 * (6 * width) ** 0.5
        if at:
            assert abs(((z1 - z0) * wide(c)).sum() - (wide(plain[at]) * span).sum()) < 1e-2 * 2 * h * 2 * (6 * width) ** 0.5


# ---- hard rows ------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("width", [1, 16, 37, 128, 1024, 3328, 20001])
def test_rows_without_spread_and_far_from_zero(width):
    # every value the same: the variance is 0, up to the rounding of the mean; y = bias up to that rounding / sqrt(eps)
    x = torch.full((5, width), 3.7, device="cuda")
    w, b = affine("f32", width, "f32")
    check_norm(x, w, b, None, nn.layer_norm(x, w, b, EPS, stats=True))
    # values that differ in their last digits only: a mean 1000 times the deviation
    x = values((9, width), "f32", 1, 1.0, 1000.0)
    check_norm(x, w, b, None, nn.layer_norm(x, w, b, EPS, stats=True))
    # one value far from all others
    x = values((9, width), "f32", 1)
    x[:, 0] = 1e4
    check_norm(x, w, b, None, nn.layer_norm(x, w, b, EPS, stats=True))
    if width > 1:
        z = nn.layer_norm(torch.zeros((2, width), device="cuda"), None, None, 0.0)
        assert torch.isnan(z).all()                # 0 / 0, as the definition says


@gpu
@pytest.mark.parametrize("width", [5, 37, 64, 128, 1000, 4096, 20001])
def test_a_row_that_is_not_finite_stays_alone(width):
    x, dy = values((12, width), "f32", 1), values((12, width), "f32", 2)
    w, b = affine("f32", width, "f32")
    good = nn.layer_norm(x, w, b, stats=True)
    grad = nn.layer_norm_backward(dy, x, good[1], good[2], w, b)[0]
    for odd in (float("nan"), float("inf")):
        bad = x.clone()
        bad[4, width // 2] = odd
        got = nn.layer_norm(bad, w, b, stats=True)
        others = [r for r in range(12) if r != 4]
        for a, g in zip(got, good):
            assert torch.equal(a[others], g[others])
        assert not torch.isfinite(got[0][4]).any()
        got = nn.layer_norm_backward(dy, bad, got[1], got[2], w, b)[0]
        assert torch.equal(got[others], grad[others]) and not torch.isfinite(got[4]).any()
        # where dropout takes the value away it is gone
        drop = next(d for d in (nn.Drop(0.5, 1, i) for i in range(200)) if not ref.kept(12, width, *d[:3])[4, width // 2])
        y, s = nn.dropout_add_layer_norm(bad, x, w, b, drop=drop)
        assert torch.isfinite(y).all() and torch.isfinite(s).all()


@gpu
def test_no_rows_and_no_columns():
    w, b = affine("f32", 16, "f32")
    x = torch.empty((0, 16), device="cuda")
    none = torch.empty(0, device="cuda")
    assert nn.dropout(x, nn.Drop(0.5, 1)).shape == (0, 16)
    y, mean, rstd = nn.layer_norm(x, w, b, stats=True)
    assert y.shape == (0, 16) and mean.shape == rstd.shape == (0,)
    assert [t.shape for t in nn.dropout_add_layer_norm(x, x, w, b)] == [(0, 16), (0, 16)]
    # sums over no rows are zero, not what lay in memory
    dx, dweight, dbias = nn.layer_norm_backward(x, x, none, none, w, b)
    assert dx.shape == (0, 16) and (dweight == 0).all() and (dbias == 0).all()
    with pytest.raises(RuntimeError, match="width"):
        nn.layer_norm(torch.empty((3, 0), device="cuda"))
    with pytest.raises(RuntimeError, match="width"):
        nn.dropout(torch.empty((3, 0), device="cuda"), nn.Drop(0.5, 1))


@gpu
@pytest.mark.parametrize("stream, act", [("f32", "bf16"), ("bf16", "bf16"), ("f32", "f32")])
@pytest.mark.parametrize("width", [7, 64, 128, 1030])
def test_norms_of_any_layout(width, stream, act):
    rows = 30
    x, r, dy = values((rows, width), act, 1), values((rows, width), stream, 2), values((rows, width), act, 3)
    w, b = affine("f32", width, act)
    drop = nn.Drop(0.3, 4, 4)
    want = nn.layer_norm(r, w, b, drop=drop, dtype=TYPES[act], stats=True)
    grads = nn.layer_norm_backward(dy, r, want[1], want[2], w, b, drop=drop)
    both = nn.dropout_add_layer_norm(x, r, w, b, drop=drop, stats=True)
    back = nn.dropout_add_layer_norm_backward(dy, r, both[1], both[2], both[3], w, b, drop=drop)
    for (what, xx), (_, rr), (_, gg), (_, ss) in zip(layouts(x), layouts(r), layouts(dy), layouts(both[1])):
        for a, g in zip(nn.layer_norm(rr, w, b, drop=drop, dtype=TYPES[act], stats=True), want):
            assert torch.equal(a, g), what
        for a, g in zip(nn.layer_norm_backward(gg, rr, want[1], want[2], w, b, drop=drop), grads):
            assert torch.equal(a, g), what
        for a, g in zip(nn.dropout_add_layer_norm(xx, rr, w, b, drop=drop, stats=True), both):
            assert torch.equal(a, g), what
        for a, g in zip(nn.dropout_add_layer_norm_backward(gg, rr, ss, both[2], both[3], w, b, drop=drop), back):
            assert torch.equal(a, g), what
    more = nn.layer_norm(r.view(5, 6, width), w, b, drop=drop, dtype=TYPES[act], stats=True)
    assert torch.equal(more[0], want[0].view(5, 6, width)) and more[1].shape == (30,)
    even = torch.empty(2 * width, device="cuda")[::2]              # weights apart
    even.copy_(w)
    assert torch.equal(nn.layer_norm(r, even, b, drop=drop, dtype=TYPES[act]), want[0])
    # results of the C entry point that are columns of a wider matrix leave the rest of it alone
    wider = torch.full((rows, width + 5), 7.0, dtype=TYPES[act], device="cuda")
    capi.layer_norm(rows, width, (r.data_ptr(), width), (wider[:, 2:].data_ptr(), width + 5), w.data_ptr(), b.data_ptr(), 0, 0,
                    (0.3, 4, 4, 0), 1e-5, (CODES[stream], CODES[act], capi.F32), torch.cuda.current_stream().cuda_stream)
    assert torch.equal(wider[:, 2:width + 2], want[0]) and (wider[:, :2] == 7).all() and (wider[:, width + 2:] == 7).all()


@gpu
def test_norm_of_rows_far_apart():
    width, far = 40, 2 ** 31 + 5                                   # the third row lies beyond 2^32 elements
    block = torch.empty(2 * far + width, dtype=torch.bfloat16, device="cuda")
    x = torch.as_strided(block, (3, width), (far, 1))
    x.copy_(values((3, width), "bf16", 5))
    near, dy = x.clone(), values((3, width), "bf16", 6)
    y, mean, rstd = nn.layer_norm(x, stats=True)
    assert all(torch.equal(a, b) for a, b in zip((y, mean, rstd), nn.layer_norm(near, stats=True)))
    assert torch.equal(nn.layer_norm_backward(dy, x, mean, rstd)[0], nn.layer_norm_backward(dy, near, mean, rstd)[0])


# ---- programs ---------------------------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("stream, act", PAIRS)
def test_autograd_gives_the_gradients(stream, act):
    x, r, dy, ds = (values((4, 7, 48), k, i) for i, k in enumerate((act, stream, act, stream)))
    w, b = affine("f32", 48, act)
    drop = nn.Drop(0.3, 4, 4)
    y, s, mean, rstd = nn.dropout_add_layer_norm(x, r, w, b, drop=drop, stats=True)
    want = nn.dropout_add_layer_norm_backward(dy, ds, s, mean, rstd, w, b, drop=drop)
    leaves = [t.clone().requires_grad_() for t in (x, r, w, b)]
    out = nn.dropout_add_layer_norm(*leaves, drop=drop)
    assert torch.equal(out[0], y) and torch.equal(out[1], s)
    for leaf, g in zip(leaves, torch.autograd.grad(out, leaves, (dy, ds))):
        assert torch.equal(g, want[[leaf is t for t in leaves].index(True)])
    out = nn.dropout_add_layer_norm(*leaves, drop=drop)            # the sum alone
    gx, gr = torch.autograd.grad(out[1], leaves[:2], ds)
    assert torch.equal(gr, ds) and torch.equal(gx, nn.dropout(ds, drop).to(x.dtype))
    out = nn.dropout_add_layer_norm(*leaves, drop=drop)            # y alone
    alone = nn.dropout_add_layer_norm_backward(dy, None, s, mean, rstd, w, b, drop=drop)
    assert all(torch.equal(a, g) for a, g in zip(torch.autograd.grad(out[0], leaves, dy), alone))

    y, mean, rstd = nn.layer_norm(r, w, b, drop=drop, dtype=x.dtype, stats=True)
    want = nn.layer_norm_backward(dy, r, mean, rstd, w, b, drop=drop)
    out = nn.layer_norm(*leaves[1:], drop=drop, dtype=x.dtype)
    assert torch.equal(out, y)
    assert all(torch.equal(a, g) for a, g in zip(torch.autograd.grad(out, leaves[1:], dy), want))
    out = nn.layer_norm(leaves[1], w, b, dtype=x.dtype)            # the rows' gradient alone, of a sum: one value for all
    assert torch.equal(torch.autograd.grad(out.sum(), leaves[1])[0], nn.layer_norm_backward(
        torch.ones_like(out), r, *nn.layer_norm(r, w, b, dtype=x.dtype, stats=True)[1:], w, b)[0])
    assert torch.equal(torch.autograd.grad(nn.dropout(leaves[0], drop), leaves[0], dy)[0], nn.dropout(dy, drop))


@gpu
@pytest.mark.parametrize("wanted", [(0,), (1,), (2,), (3,), (0, 3), (1, 2)])
def test_autograd_of_some_of_the_inputs(wanted):
    x, r, dy = (values((700, 48), "f32", i) for i in range(3))
    w, b = affine("f32", 48, "f32")
    drop = nn.Drop(0.3, 4, 4)
    y, s, mean, rstd = nn.dropout_add_layer_norm(x, r, w, b, drop=drop, stats=True)
    want = nn.dropout_add_layer_norm_backward(dy, None, s, mean, rstd, w, b, drop=drop)
    _, mean, rstd = nn.layer_norm(r, w, b, drop=drop, stats=True)
    plain = (None,) + nn.layer_norm_backward(dy, r, mean, rstd, w, b, drop=drop)
    inputs = [t.clone().requires_grad_(i in wanted) for i, t in enumerate((x, r, w, b))]
    leaves = [inputs[i] for i in wanted]
    out = nn.dropout_add_layer_norm(*inputs, drop=drop)[0]
    for i, g in zip(wanted, torch.autograd.grad(out, leaves, dy)):
        assert torch.equal(g, want[i])
    if 0 not in wanted:
        out, mean, rstd = nn.layer_norm(*inputs[1:], drop=drop, stats=True)
        assert not mean.requires_grad and not rstd.requires_grad
        for i, g in zip(wanted, torch.autograd.grad(out, leaves, dy)):
            assert torch.equal(g, plain[i])
    with torch.no_grad():
        assert not nn.layer_norm(*inputs[1:]).requires_grad


@gpu
def test_a_step_that_changed_before_its_gradient_is_an_error():
    x = values((4, 16), "f32", 1).requires_grad_()
    step = torch.zeros(1, dtype=torch.int64, device="cuda")
    for f in (lambda d: nn.dropout(x, d), lambda d: nn.layer_norm(x, drop=d), lambda d: nn.dropout_add_layer_norm(x, x, drop=d)[0]):
        y = f(nn.Drop(0.5, 1, 0, step))
        step.add_(1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            y.sum().backward()


@gpu
def test_graphs_and_streams():
    x, r, dy = values((300, 96), "bf16", 1), values((300, 96), "f32", 2), values((300, 96), "bf16", 3)
    w, b = affine("f32", 96, "bf16")
    step = torch.zeros(1, dtype=torch.int64, device="cuda")

    def work(drop):
        y, s, mean, rstd = nn.dropout_add_layer_norm(x, r, w, b, drop=drop, stats=True)
        grads = nn.dropout_add_layer_norm_backward(dy, s, s, mean, rstd, w, b, drop=drop)
        z, mean, rstd = nn.layer_norm(s, w, b, drop=drop, dtype=torch.bfloat16, stats=True)
        return (y, s, *grads, z, *nn.layer_norm_backward(dy, s, mean, rstd, w, b, drop=drop), nn.dropout(x, drop))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        work(nn.Drop(0.2, 7, 5, step))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = work(nn.Drop(0.2, 7, 5, step))
        step.add_(1)
    for i in range(4):
        step.fill_(i * 3)
        x.copy_(values((300, 96), "bf16", 10 + i))
        graph.replay()
        torch.cuda.synchronize()
        assert step.item() == i * 3 + 1
        for a, g in zip(work(nn.Drop(0.2, 7, 5 + i * 3)), outs):
            assert torch.equal(a, g)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):                              # the same bits from another stream
            for a, g in zip(work(nn.Drop(0.2, 7, 5 + i * 3)), outs):
                assert torch.equal(a, g)
        torch.cuda.current_stream().wait_stream(side)


@gpu
def test_rows_of_a_table_through_the_norm_and_back():
    # preprocess, push_pull, norm and dropout, gradient, push: the next pull returns rows that moved by -lr * gradient
    rows, width, n, lr = 500, 32, 64, 0.1
    rng = np.random.default_rng(1)
    capi.seed(1)
    t = capi.Table(0, 1, 0, "127.0.0.1", 30999, rows, width, 0, 0, np.zeros(rows, np.uint8), np.arange(rows, dtype=np.int64),
                   ("Normal", 0.0, 0.1), lr, 0)
    keys = np.ascontiguousarray(rng.permutation(rows)[:n].astype(np.int64))
    pulled, after = torch.empty((n, width), device="cuda"), torch.empty((n, width), device="cuda")
    w, b = affine("f32", width, "bf16")
    t.preprocess(keys.ctypes.data, n)
    t.push_pull(0, pulled.data_ptr())
    pulled.requires_grad_()
    y = nn.layer_norm(pulled, w, b, drop=nn.Drop(0.1, 1, 0), dtype=torch.bfloat16)
    y.backward(values((n, width), "bf16", 5))
    assert pulled.grad.dtype == torch.float32
    t.preprocess(keys.ctypes.data, n)
    t.push_pull(pulled.grad.data_ptr(), after.data_ptr())
    want = wide(pulled) - lr * wide(pulled.grad)
    check(after, want, np.abs(wide(pulled)) + np.abs(want), 4 * 2.0 ** -24)
    t.close()


@gpu
def test_the_example_learns():
    # the labels are a function of the ids: a model that gets the table's rows, and sends it their gradients, learns them; one that
    # could not would stay at log 2
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "examples", "train_dense.py")
    spec = importlib.util.spec_from_file_location("train_dense", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    losses = example.train(steps=60, samples=1024)
    assert np.isfinite(losses).all()
    assert np.mean(losses[-10:]) < 0.9 * np.log(2) < np.mean(losses[:3])


# ---- refusals ---------------------------------------------------------------------------------------------------------------

def test_the_c_entry_points_refuse_what_they_cannot_do():
    # refused before anything is launched: no GPU is needed
    m, none, drop = (4096, 8), capi.NO_MATRIX, capi.NO_DROP
    f32, bf16, f16 = capi.F32, capi.BF16, capi.F16
    for args, match in [
            ((2, 0, m, m, drop, f32), "width"), ((2, 2 ** 31, m, m, drop, f32), "width"), ((2, 8, m, m, drop, 3), "type"),
            ((2, 8, none, m, drop, f32), "null"), ((2, 8, m, none, drop, f32), "null"), ((2, 8, m, (4096, 7), drop, f32), "overlap"),
            ((2, 8, m, m, (-0.1, 0, 0, 0), f32), "probability"), ((2, 8, m, m, (1.5, 0, 0, 0), f32), "probability"),
            ((2, 8, m, m, (float("nan"), 0, 0, 0), f32), "probability")]:
        with pytest.raises(RuntimeError, match=match):
            capi.dropout(*args)
    types = (f32, f32, f32)
    for args, match in [
            ((2, 0, m, m, 0, 0, 0, 0, drop, EPS, types), "width"), ((2, 8, none, m, 0, 0, 0, 0, drop, EPS, types), "null"),
            ((2, 8, m, (4096, 0), 0, 0, 0, 0, drop, EPS, types), "overlap"), ((2, 8, m, m, 0, 0, 0, 0, drop, -1.0, types), "eps"),
            ((2, 8, m, m, 0, 0, 0, 0, drop, float("nan"), types), "eps"), ((2, 8, m, m, 0, 0, 0, 0, drop, EPS, (bf16, f32, f32)), "normalised"),
            ((2, 8, m, m, 0, 0, 0, 0, drop, EPS, (bf16, f16, f32)), "normalised"), ((2, 8, m, m, 0, 0, 0, 0, drop, EPS, (7, 7, f32)), "type"),
            ((2, 8, m, m, 4096, 0, 0, 0, drop, EPS, (f32, bf16, f16)), "weight and bias"),
            ((2, 8, m, m, 0, 0, 0, 0, (2.0, 0, 0, 0), EPS, types), "probability")]:
        with pytest.raises(RuntimeError, match=match):
            capi.layer_norm(*args)
    for residual, total in ((none, m), (m, none), (m, (4096, 1))):
        with pytest.raises(RuntimeError, match="null|overlap"):
            capi.dropout_add_layer_norm(2, 8, m, residual, total, m, 0, 0, 0, 0, drop, EPS, types)
    rows = 100_000                                  # few rows need no workspace
    need = capi.layer_norm_workspace(rows, 8)
    assert need >= 2 * 8 * 4
    for args, match in [
            ((2, 8, none, m, m, 0, 0, 0, 16, 16, 0, 0, drop, types), "null"), ((2, 8, m, m, m, 0, 0, 0, 0, 16, 0, 0, drop, types), "mean and rstd"),
            ((rows, 8, m, m, m, 0, 4096, 0, 16, 16, 0, 0, drop, types), "workspace"),
            ((rows, 8, m, m, m, 0, 4096, 0, 16, 16, 4096, need - 1, drop, types), "workspace"),
            ((rows, 8, m, m, m, 0, 4096, 0, 16, 16, 4100, need, drop, types), "workspace"),
            ((2, 8, m, m, (4096, 2), 0, 0, 0, 16, 16, 0, 0, drop, types), "overlap"),
            ((2, 8, m, m, m, 4096, 0, 0, 16, 16, 0, 0, drop, (f32, f32, bf16)), "weight and bias")]:
        with pytest.raises(RuntimeError, match=match):
            capi.layer_norm_backward(*args)
    with pytest.raises(RuntimeError, match="null argument"):
        capi._check(capi.lib().hctr_dropout(None))


def test_tensors_that_are_not_on_the_gpu_are_refused():
    x = torch.zeros((2, 8))
    for f in (lambda: nn.dropout(x, nn.Drop(0.5, 1)), lambda: nn.layer_norm(x), lambda: nn.dropout_add_layer_norm(x, x),
              lambda: nn.layer_norm_backward(x, x, x[:, 0], x[:, 0])):
        with pytest.raises(RuntimeError, match="on the GPU"):
            f()


@gpu
def test_the_functions_refuse_what_does_not_fit():
    x, h = torch.zeros((2, 8), device="cuda"), torch.zeros((2, 8), device="cuda", dtype=torch.bfloat16)
    w, stat = torch.zeros(8, device="cuda"), torch.zeros(2, device="cuda")
    for f, match in [
            (lambda: nn.dropout(x.double(), nn.Drop(0.5, 1)), "float32, bfloat16 or float16"),
            (lambda: nn.dropout(x, nn.Drop(0.5, 1, 0, stat)), "step tensor"), (lambda: nn.dropout(x, nn.Drop(2, 1)), "probability"),
            (lambda: nn.dropout(x[0, 0], nn.Drop(0.5, 1)), "dimension"), (lambda: nn.layer_norm(x, w[:4]), "weight"),
            (lambda: nn.layer_norm(x, w, w.half()), "bias"), (lambda: nn.layer_norm(h, w, w.bfloat16()), "one type"),
            (lambda: nn.layer_norm(x, w.cpu()), "weight"), (lambda: nn.layer_norm(h, dtype=torch.float32), "normalised"),
            (lambda: nn.layer_norm(x, eps=-1.0), "eps"), (lambda: nn.dropout_add_layer_norm(x, x[:1]), "residual"),
            (lambda: nn.dropout_add_layer_norm(x, h), "normalised"), (lambda: nn.layer_norm_backward(x[:, :4], x, stat, stat), "dy"),
            (lambda: nn.layer_norm_backward(x, x, stat[:1], stat), "mean"), (lambda: nn.layer_norm_backward(x, x, stat, stat.double()), "rstd"),
            (lambda: nn.dropout_add_layer_norm_backward(h, h, x, stat, stat), "ds")]:
        with pytest.raises(RuntimeError, match=match):
            f()

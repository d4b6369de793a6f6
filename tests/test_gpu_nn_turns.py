"""The dense operators where a kernel's loops go round more than once: more rows than a launch works on at a time.  Every row is
compared with the definition in 64 bits.

Tolerances, in units of 2^-24 of the magnitudes that dense_reference64.py gives.  A sum whose lanes add n terms one by one and are
joined in pairs, 2 * log2(lanes) + 2 steps at most, is off by n + 2 * log2(lanes) + 2 units, and what is made of it by some
roundings more, for which 8 are allowed.
  A row of up to 16384 columns has at most 16 of them in a lane and at most 1024 lanes.  Of a longer row a lane adds V (4 of 32 bits, 8 of
16) of every 256 V columns (forward), or of every 1024 V (gradient).
  A column of the gradient of weight and bias has a term in every turn of a block, then one of each of the up to 128 groups of lanes of the
block; of the blocks' sums, at most 2048, a thread adds 64 at most, and 64 threads' at most are added: turns + 256 units.
The result is rounded once more, to its type."""
import math

import numpy as np
import pytest
import torch

from hetuctr_amd import capi, nn
from tests import dense_reference as ref
from tests import dense_reference64 as ref64
from tests.test_gpu_nn import CODES, EPS, PAIRS, TYPES

gpu = pytest.mark.gpu
SIZES = {"f32": 4, "bf16": 2, "f16": 2}


def per_vector(kind):
    return 16 // SIZES[kind]


def row_units(width, kind, threads):
    terms, lanes = (16, 1024) if width <= 16384 else (per_vector(kind) * math.ceil(width / (threads * per_vector(kind))), threads)
    return (terms + 2 * math.log2(lanes) + 2 + 8) * 2.0 ** -24


def groups(width, kind):
    """rows that a block of the kernels holds at a time"""
    lanes = 2
    while lanes < 64 and lanes * per_vector(kind) < width:
        lanes *= 2
    return 256 // lanes if width <= 1024 else 1


def values(shape, kind, seed, std=1.0, mean=0.0):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    return torch.empty(shape, device="cuda").normal_(mean, std, generator=gen).to(TYPES[kind])


def wide(t):
    return None if t is None else t.double()


def check(got, want, size, units, what):
    kind = next(k for k, v in TYPES.items() if v == got.dtype)
    got = got.double().view(want.shape)
    off = units * size
    allowed = off + ref.UNIT[kind] * (want.abs() + off).clamp_min(ref.TINY[kind])
    bad = ~((got - want).abs() <= allowed)
    if bad.any():
        at = bad.nonzero()
        raise AssertionError("%s: %d of %d values, first at %s, last at %s, worst %.3g of what is allowed" % (
            what, len(at), bad.numel(), at[0].tolist(), at[-1].tolist(), ((got - want).abs() / allowed).nan_to_num(1e30).max().item()))


@pytest.mark.parametrize("width", [1, 5, 37, 64])
def test_the_two_references_agree(width):
    rng = np.random.default_rng(width)
    x, dy, w, b = rng.normal(0.3, 2, (9, width)), rng.normal(size=(9, width)), rng.normal(1, 0.2, width), rng.normal(size=width)
    tensor = torch.from_numpy
    for drop in (None, (0.3, 2 ** 63 + 5, 2 ** 40 + 3), (0.5, 7, 9)):
        assert np.array_equal(np.broadcast_to(ref64.factors(9, width, drop, "cpu").numpy(), (9, width)), ref.factors(9, width, drop))
    assert np.array_equal(ref64.kept(2, width, 0.3, 1, 2, "cpu", first=7).numpy(), ref.kept(9, width, 0.3, 1, 2)[7:])
    near = lambda a, b: np.allclose(np.asarray(a).reshape(np.shape(b)), b, rtol=1e-11, atol=1e-11)
    (y, mean, rstd), _ = ref64.forward(tensor(x), tensor(w), tensor(b), EPS)
    assert near(y, ref.normalise(x, w, b, EPS)) and near(mean, ref.statistics(x, EPS)[0]) and near(rstd, ref.statistics(x, EPS)[1])
    got = ref64.gradient(tensor(dy), tensor(x), mean, rstd, tensor(w))
    want = ref.gradient(dy, x, *ref.statistics(x, EPS), w)
    for g, h in zip(got, want):
        assert all(near(a, c) for a, c in zip(g, h))


def affine(width, kind):
    return values(width, kind, 21, 0.2, 1.0), values(width, kind, 22, 0.2)


# Blocks that stay for several rows, of every number of lanes and pieces, even and ragged: at most 16 blocks a CU.
FORWARD_WIDTHS = [600, 601, 1000, 1024, 1032, 1443, 2048, 2056, 4093, 4096, 4100, 8192, 11381, 16384]


def forward_rows(width, kind):
    return 2 * 256 * 16 * (groups(width, kind) if width <= 1024 else 1) + 5 if width <= 8192 else 3 * 256 + 5


@gpu
@pytest.mark.parametrize("stream, act", PAIRS)
@pytest.mark.parametrize("width", FORWARD_WIDTHS)
def test_layer_norm_of_many_rows(width, stream, act):
    rows = forward_rows(width, stream)
    x = values((rows, width), stream, width, 0.5, 0.1)
    weight, bias = affine(width, act)
    (y, mean, rstd), (size, mean_size, rstd_size) = ref64.forward(wide(x), wide(weight), wide(bias), EPS)
    units = row_units(width, stream, 256)
    for drop in (None, (0.25, 3, width)):
        got = nn.layer_norm(x, weight, bias, EPS, drop=drop and nn.Drop(*drop), dtype=TYPES[act], stats=True)
        f = ref64.factors(rows, width, drop, "cuda")
        check(got[1], mean, mean_size, units, "mean")
        check(got[2], rstd, rstd_size, units, "rstd")
        check(got[0], y * f, size * f, units, "y")


@gpu
@pytest.mark.parametrize("stream, act", PAIRS)
@pytest.mark.parametrize("width", FORWARD_WIDTHS)
def test_dropout_add_layer_norm_of_many_rows(width, stream, act):
    rows = forward_rows(width, stream) // 4             # (forms with a branch added have at most four blocks a CU)
    x, residual = values((rows, width), act, width), values((rows, width), stream, width + 1, 2.0, 0.3)
    weight, bias = affine(width, "f32")
    units = row_units(width, stream, 256)
    for drop in (None, (0.25, 3, width)):
        got = nn.dropout_add_layer_norm(x, residual, weight, bias, EPS, drop=drop and nn.Drop(*drop), stats=True)
        branch = wide(x) * ref64.factors(rows, width, drop, "cuda")
        total = wide(residual) + branch
        check(got[1], total, branch.abs() + total.abs(), 2 * 2.0 ** -24, "s")
        (y, mean, rstd), sizes = ref64.forward(total, wide(weight), wide(bias), EPS)
        # the sum carries two roundings of its own, of the branch and of the total: they add to every magnitude
        extra = branch.abs() + total.abs()
        moved = (extra + extra.mean(1, keepdim=True)) * rstd
        h = (total - mean) * rstd
        moved = moved + h.abs() * (moved * h.abs()).mean(1, keepdim=True)
        check(got[0], y, sizes[0] + moved * wide(weight).abs(), units, "y")
        check(got[2], mean, sizes[1] + extra.mean(1, keepdim=True), units, "mean")
        check(got[3], rstd, sizes[2] + rstd * (h.abs() * extra * rstd).mean(1, keepdim=True), units, "rstd")


# Of every number of lanes and pieces, even and ragged: the gradient's blocks stay, whatever the width.
GRADIENT_WIDTHS = [1, 3, 8, 12, 16, 17, 37, 64, 100, 130, 256, 333, 512, 600, 1000, 1024, 1443, 2048, 2056, 4096, 4100, 8192, 8200, 11381, 16384,
                   16388, 20001]


def gradient_rows(width, kind):
    # at most 8 blocks a CU, as many as fetch 17 KiB at a time, of 4 bytes a column at least: more than two turns
    each = groups(width, kind)
    return 2 * 256 * each * min(8, 17 * 1024 // (each * width * 4) + 1) + each + 3


@gpu
@pytest.mark.parametrize("stream, act", PAIRS)
@pytest.mark.parametrize("width", GRADIENT_WIDTHS)
def test_layer_norm_gradient_of_many_rows(width, stream, act):
    rows = gradient_rows(width, stream)
    x, dy = values((rows, width), stream, width, 0.5, 0.1), values((rows, width), act, width + 2, 0.01)
    mean, rstd = (t.float() for t in ref64.statistics(wide(x), EPS))
    weight, bias = affine(width, act)
    units, columns = row_units(width, stream, 1024), (math.ceil(rows / (256 * groups(width, stream))) + 256) * 2.0 ** -24
    for drop in (None, (0.25, 3, width)):
        dx, dweight, dbias = nn.layer_norm_backward(dy, x, mean, rstd, weight, bias, drop=drop and nn.Drop(*drop))
        want, size = ref64.gradient(wide(dy) * ref64.factors(rows, width, drop, "cuda"), wide(x), wide(mean), wide(rstd), wide(weight))
        check(dx, want[0], size[0], units, "dx")
        check(dweight, want[1], size[1], columns, "dweight")
        check(dbias, want[2], size[2], columns, "dbias")


@gpu
@pytest.mark.parametrize("stream, act", PAIRS)
@pytest.mark.parametrize("width", GRADIENT_WIDTHS)
def test_dropout_add_layer_norm_gradient_of_many_rows(width, stream, act):
    rows = gradient_rows(width, stream)
    s, dy = values((rows, width), stream, width, 2.0, 0.3), values((rows, width), act, width + 2, 0.01)
    ds = values((rows, width), stream, width + 3, 0.01)
    mean, rstd = (t.float() for t in ref64.statistics(wide(s), EPS))
    weight, bias = affine(width, "f32")
    units, columns = row_units(width, stream, 1024), (math.ceil(rows / (256 * groups(width, stream))) + 256) * 2.0 ** -24
    want, size = ref64.gradient(wide(dy), wide(s), wide(mean), wide(rstd), wide(weight))
    for drop, more in ((None, None), (None, ds), ((0.25, 3, width), None), ((0.25, 3, width), ds)):
        dx, dresidual, dweight, dbias = nn.dropout_add_layer_norm_backward(dy, more, s, mean, rstd, weight, bias,
                                                                           drop=drop and nn.Drop(*drop))
        total = want[0] if more is None else want[0] + wide(more)
        sizes = size[0] + total.abs()
        f = ref64.factors(rows, width, drop, "cuda")
        check(dresidual, total, sizes, units, "dresidual")
        check(dx, total * f, sizes * f, units, "dx")
        check(dweight, want[1], size[1], columns, "dweight")
        check(dbias, want[2], size[2], columns, "dbias")


# ---- more blocks than a launch has ------------------------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize("width, rows, kind", [(260, 2 ** 25 + 5, "f32"), (16388, 2 ** 20 + 3, "bf16")])
def test_layer_norm_of_more_rows_than_blocks(width, rows, kind):
    # one row, read again and again: its results are the same in every row
    x = values((1, width), kind, 5)
    weight, bias = affine(width, "bf16")
    one = nn.layer_norm(x, weight, bias, dtype=torch.bfloat16, stats=True)
    many = nn.layer_norm(x.expand(rows, width), weight, bias, dtype=torch.bfloat16, stats=True)
    for a, b in zip(many, one):
        assert (a == b).all()
    del many, a
    torch.cuda.empty_cache()


@gpu
@pytest.mark.parametrize("width, rows", [(1024, 2 ** 23 + 5), (5, 2 ** 30 + 3)])
def test_dropout_of_more_values_than_blocks(width, rows):
    x = torch.ones((rows, width), device="cuda")
    place = (x.data_ptr(), width)
    capi.dropout(rows, width, place, place, (0.3, 77, 5, 0), CODES["f32"], torch.cuda.current_stream().cuda_stream)
    scale = torch.tensor(1 / 0.7, dtype=torch.float32, device="cuda")
    for first in (0, rows // 2, rows - 8):
        keep = ref64.kept(8, width, 0.3, 77, 5, "cuda", first=first)
        assert torch.equal(x[first:first + 8], torch.where(keep, scale, torch.zeros_like(scale)))
    del x
    torch.cuda.empty_cache()
